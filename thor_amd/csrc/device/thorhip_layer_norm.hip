// Layer norm over the last axis, forward and backward.
//
// Forward, one row: mean = sum x / C, rstd = 1 / sqrt(sum (x - mean)^2 / C + epsilon), y = (x - mean) * rstd * weight + bias.  A row is
// read once and stays in registers between the two sums and the output; the squares are those of differences from the mean, and where the
// mean's rounding could be seen in h the sum of these differences makes up for it.  Everything is fp32, rounded once where it is stored.
//
// Backward, one row, with h = (x - mean) * rstd and g = dy * weight:
//   dx = rstd * (g - sum(g) / C - h * sum(g * h) / C),  weight gradient = sum over rows of dy * h,  bias gradient = sum over rows of dy.
// A block keeps its columns' share of both parameter gradients in registers while it takes row after row, so that x and dy are read once
// for all three results; a second kernel adds the blocks' shares in a fixed order.
//
// Both are streams (4 bytes per element forward and 6 backward for 16-bit types): what bounds them is the bytes they move.  A copy of
// large tensors by the library runs at 5.4 TB/s on this card; the times at the kernels are to be read against that.
#include "thorhip_rows.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {

using namespace thor;

struct ForwardArgs {
    RowsOf input, output;
    const void* weight;
    const void* bias;
    float* mean;
    float* rstd;
    u8* codes;
    float* scales;
    Extent extent;
    u32 columns, innerRows, blocksPerRow;
    int parametersAreFloat, format;
    float epsilon, inverse;  // 1 / columns
};

struct BackwardArgs {
    RowsOf error, input, gradient;
    const void* weight;
    const float* mean;
    const float* rstd;
    const u8* codes;
    const float* scales;
    float* partials;  // [blocks][2][columns], or null: no parameter gradient is asked for, or the kernel writes them itself
    void* weightGradient;
    void* biasGradient;
    Extent extent;
    u32 columns, innerRows, blocksPerRow;
    u32 sharesOfBlock;  // of the partials: one for each kRowsOfShare rows of a team
    int parametersAreFloat, format;
    float inverse;  // 1 / columns
};

// Rows that a lane adds up for a parameter gradient one after the other, at most.  A block that takes more of them begins another share,
// and the sums over shares are compensated, so that a gradient over millions of rows has the error of one over some thousands.
constexpr u32 kRowsOfShare = 128;

template <typename T>
__device__ __forceinline__ void loadParameters(const void* p, int isFloat, float missing, u32 column, bool has, float (&v)[kVec<T>]) {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) v[i] = missing;
    if (p == nullptr || !has) return;
    if (isFloat) {
        loadShared<kVec<T>>(static_cast<const float*>(p) + column, v);
    } else {
        loadShared<kVec<T>>(static_cast<const T*>(p) + column, v);
    }
}
template <typename T>
__device__ __forceinline__ float loadParameter(const void* p, int isFloat, float missing, u32 column, bool has) {
    if (p == nullptr || !has) return missing;
    return isFloat ? static_cast<const float*>(p)[column] : widen(static_cast<const T*>(p)[column]);
}

// sum / columns with the bits of a division but for a last one: one product, put right by what is left over.  A wavefront's row waits for
// each of these, and a division is four times as long a chain (bf16 65536 x 512 forward: 25.0 us with divisions and a square root, 23.8
// with this and the hardware's reciprocal root; 8192 x 8192 backward from codes 58.9 and 57.5).
__device__ __forceinline__ float average(float sum, u32 columns, float inverse) {
    const float q = sum * inverse, left = __builtin_fmaf(-q, (float)columns, sum);
    return __builtin_fmaf(__builtin_fminf(left, 3.40282347e38f), inverse, q);  // an infinite sum leaves no number
}
// Whether a row's mean is refined by the sum of the differences from it.  A mean rounds to its own last bits, which are many of the
// deviation's where it is large against that: fp32 rows around 4096 with a deviation of one have an h that is off by 4e-4 without, 5e-7
// with it.  16-bit rows do without as long as sums of equal elements are exact, 8 bits each of bf16 and 11 of up to 6144 of fp16: a row
// of one value is zero then, and where the elements differ, their own last bits are 2^13 times the mean's at least.  There it would cost
// time (16380 x 4097 61.0 us, without 55.8; 262144 x 96 18.2 and 17.0; 8192 x 8192 46.6 and 44.7), while fp32 takes the same either way
// (32768 x 1024 43.9 us, 16380 x 4097 106, 8192 x 8192 99).
template <typename T, int LANES>
constexpr bool kRefined = sizeof(T) == 4 || (std::is_same<T, f16>::value && LANES >= 512);

// A row's mean and 1 / sqrt(variance + epsilon) (the hardware's reciprocal root, one unit off at most where its argument is a normal
// number, which epsilon sees to), from a value near the mean, the sum of the squares of the differences from it, and the sum of these.
struct Moments {
    float mean, rstd, shift;
    __device__ __forceinline__ float normalised(float difference) const { return __builtin_fmaf(difference, rstd, shift); }
};
__device__ __forceinline__ Moments momentsOf(float near, const float (&sums)[1], const ForwardArgs& a) {
    return {near, __builtin_amdgcn_rsqf(__builtin_fmaf(sums[0], a.inverse, a.epsilon)), 0.0f};
}
__device__ __forceinline__ Moments momentsOf(float near, const float (&sums)[2], const ForwardArgs& a) {
    constexpr float kMost = 3.40282347e38f;
    // of a row with an infinity the differences are no numbers, but its mean is one; squares that overflow, or are no numbers, stay
    const float left = __builtin_amdgcn_fmed3f(sums[1] * a.inverse, -kMost, kMost);
    const float squares = sums[0] < __builtin_inff() ? __builtin_fmaxf(__builtin_fmaf(-left, sums[1], sums[0]), 0.0f) : sums[0];
    const float rstd = __builtin_amdgcn_rsqf(__builtin_fmaf(squares, a.inverse, a.epsilon));
    return {near + left, rstd, -left * rstd};
}

// The team of a block that a lane is in; the compiler is told that it is the same for a wavefront.
template <int LANES>
__device__ __forceinline__ u32 teamOfBlock() {
    if constexpr (LANES >= 64) return __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
    return threadIdx.x / LANES;
}
// Threads of a forward block: several teams where a team is one wavefront at most and none waits for another.
template <int LANES>
constexpr int kForwardThreads = LANES < 128 ? 256 : LANES;
// Threads of a backward block: whole teams of eight or twelve wavefronts in all.
template <int LANES>
constexpr int kBackwardThreads = LANES % 3 == 0 ? 768 : LANES < 512 ? 512 : LANES;

// The sum over the four rows of 16 lanes of a wavefront, lane by lane, in each of them.
__device__ __forceinline__ float sumRowsOfWave(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(f32Bits(x), f32Bits(x), false, false);
    x = bitsF32(r[0]) + bitsF32(r[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(f32Bits(x), f32Bits(x), false, false);
    return bitsF32(h[0]) + bitsF32(h[1]);
}

// Waits for every load so far.  A loop that loads the next row while it works on this one is entered with nothing on its way: the
// compiler would otherwise let each turn begin with the wait that only the first one needs, and have the next row's loads waited for at once.
__device__ __forceinline__ void loadsArrived() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0), no other counter

// Rows of at most LANES * K chunks, a team of LANES lanes per row.  The blocks stay, keep weight and bias in registers and take every
// gridDim-th row; a row is loaded while the one before it is worked on.
// fp32 32768 x 1024 takes 43.7 us (6.1 TB/s), bf16 16384 x 4096 44.6 us (6.0 TB/s), bf16 8192 x 8192 with e4m3 codes 58.2 us (5.8 TB/s).
template <typename T, int LANES, int K, bool CHECKPOINT, Fit FIT>
__global__ __launch_bounds__(kForwardThreads<LANES>) void layerNormForward(ForwardArgs a) {
    constexpr int VEC = kVec<T>, TEAMS = kForwardThreads<LANES> / LANES;
    constexpr bool REFINED = kRefined<T, LANES>;
    __shared__ float shared[LANES / 64 + 1][1], sharedOfDifferences[LANES / 64 + 1][REFINED ? 2 : 1];
    const RowLayout<T, LANES, FIT> at(a.columns, threadIdx.x % LANES);
    // a lane without a chunk works on another's where the whole block of codes does; elsewhere the block's scale would not be the same
    const auto works = [&](int k) { return FIT == Fit::Blocks || at.has(k); };
    const auto source = [&](int k) { return FIT == Fit::Blocks ? at.source(k) : at.column(k); };
    const u32 rows = rowsInUse(a.extent), step = gridDim.x * TEAMS;
    u32 row = blockIdx.x * TEAMS + teamOfBlock<LANES>();
    struct Loaded {
        Words4 words[K];
        T tail;  // as it was loaded: to widen it is to wait for it
    } now, next;
    const auto load = [&](u32 of, Loaded& to) {
        const T* in = rowPointer<const T>(a.input, of, a.innerRows);
#pragma unroll
        for (int k = 0; k < K; ++k) to.words[k] = works(k) ? loadWords(in + source(k)) : Words4{};
        to.tail = narrow<T>(0.0f);
        if (at.tail) to.tail = in[at.tailColumn];
    };
    if (row < rows) load(row, now);
    float weight[K][VEC], bias[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        loadParameters<T>(a.weight, a.parametersAreFloat, 1.0f, source(k), works(k), weight[k]);
        loadParameters<T>(a.bias, a.parametersAreFloat, 0.0f, source(k), works(k), bias[k]);
    }
    const float tailWeight = loadParameter<T>(a.weight, a.parametersAreFloat, 1.0f, at.tailColumn, at.tail);
    const float tailBias = loadParameter<T>(a.bias, a.parametersAreFloat, 0.0f, at.tailColumn, at.tail);
    loadsArrived();
    for (; row < rows; row += step) {
        if (row + step < rows) load(row + step, next);
        float x[K][VEC], tail = widen(now.tail);
        float sum[1] = {tail};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            unpack<T>(now.words[k], x[k]);
            float ofChunk = 0.0f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) ofChunk += x[k][i];
            sum[0] += at.has(k) ? ofChunk : 0.0f;
        }
        sumTeam<LANES>(sum, shared);
        const float near = average(sum[0], a.columns, a.inverse);
        tail -= near;
        float sums[REFINED ? 2 : 1];
        sums[0] = at.tail ? tail * tail : 0.0f;
        if constexpr (REFINED) sums[1] = at.tail ? tail : 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float ofChunk[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                x[k][i] -= near;
                ofChunk[0] += x[k][i] * x[k][i];
                if constexpr (REFINED) ofChunk[1] += x[k][i];
            }
            sums[0] += at.has(k) ? ofChunk[0] : 0.0f;
            if constexpr (REFINED) sums[1] += at.has(k) ? ofChunk[1] : 0.0f;
        }
        sumTeam<LANES>(sums, sharedOfDifferences);
        const Moments m = momentsOf(near, sums, a);
        if (at.lane == 0) {
            a.mean[row] = m.mean;
            a.rstd[row] = m.rstd;
        }
        T* out = rowPointer<T>(a.output, row, a.innerRows);
        u8* codes = a.codes + (i64)row * a.columns;
        float* scales = a.scales + (i64)row * a.blocksPerRow;
        tail = REFINED ? m.normalised(tail) : tail * m.rstd;
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[k][i] = REFINED ? m.normalised(x[k][i]) : x[k][i] * m.rstd;
            if constexpr (CHECKPOINT) {
                const bool hasTail = at.tail && k == at.tailChunk;
                const BlockScale scale = scaleOfLanes<VEC>(x[k], works(k), tail, hasTail, a.format);
                if (works(k)) storeCodes<VEC>(codes + source(k), encodeChunk<VEC>(x[k], scale, a.format));
                if (hasTail) codes[at.tailColumn] = encodeOne(tail, scale, a.format);
                if (at.column(k) % kCheckpointBlock == 0 && at.column(k) < a.columns) scales[at.column(k) / kCheckpointBlock] = scale.scale;
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[k][i] = x[k][i] * weight[k][i] + bias[k][i];
            if (works(k)) storeChunk(out + source(k), x[k]);
        }
        if (at.tail) out[at.tailColumn] = narrow<T>(tail * tailWeight + tailBias);
        now = next;
    }
}

// A sum of any length with the error of a short one: what an addition loses is given to the next.
struct LongSum {
    float sum = 0.0f, lost = 0.0f;
    __device__ __forceinline__ void add(float x) {
        const float y = x - lost, t = sum + y;
        lost = __builtin_fabsf(t) < __builtin_inff() ? (t - sum) - y : 0.0f;  // an infinity stays one
        sum = t;
    }
};

// Rows of any length: a block of 1024 lanes per row, which reads it three times (the second and third time from the caches).  bf16
// 4096 x 20000 takes 112 us (2.9 TB/s), with e4m3 codes 189 us: a wavefront has a chunk on its way at a time, and folds between the readings.
template <typename T, bool CHECKPOINT>
__global__ __launch_bounds__(1024) void layerNormForwardLong(ForwardArgs a) {
    constexpr int VEC = kVec<T>, LANES = 1024;
    __shared__ float shared[LANES / 64][1], sharedOfDifferences[LANES / 64][2];
    const RowLayout<T, LANES, Fit::Any> at(a.columns, threadIdx.x);
    const u32 rows = rowsInUse(a.extent);
    for (u32 row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* in = rowPointer<const T>(a.input, row, a.innerRows);
        float x[VEC], tail = at.tail ? widen(in[at.tailColumn]) : 0.0f;
        LongSum ofLane;
        for (int k = 0; at.has(k); ++k) {
            loadChunk(in + at.column(k), x);
            float ofChunk = 0.0f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) ofChunk += x[i];
            ofLane.add(ofChunk);
        }
        float sum[1] = {ofLane.sum + tail};
        sumTeam<LANES>(sum, shared);
        const float near = average(sum[0], a.columns, a.inverse);
        tail -= near;
        LongSum squaresOfLane, differencesOfLane;
        for (int k = 0; at.has(k); ++k) {
            loadChunk(in + at.column(k), x);
            float ofChunk[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                ofChunk[0] += (x[i] - near) * (x[i] - near);
                ofChunk[1] += x[i] - near;
            }
            squaresOfLane.add(ofChunk[0]);
            differencesOfLane.add(ofChunk[1]);
        }
        float sums[2] = {squaresOfLane.sum + (at.tail ? tail * tail : 0.0f), differencesOfLane.sum + (at.tail ? tail : 0.0f)};
        sumTeam<LANES>(sums, sharedOfDifferences);
        const Moments m = momentsOf(near, sums, a);
        if (threadIdx.x == 0) {
            a.mean[row] = m.mean;
            a.rstd[row] = m.rstd;
        }
        T* out = rowPointer<T>(a.output, row, a.innerRows);
        u8* codes = a.codes + (i64)row * a.columns;
        float* scales = a.scales + (i64)row * a.blocksPerRow;
        tail = m.normalised(tail);
        const int steps = (a.columns + LANES * VEC - 1) / (LANES * VEC);  // the same for all lanes of a block of codes
        for (int k = 0; k < steps; ++k) {
            const bool has = at.has(k);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[i] = 0.0f;
            if (has) {
                loadChunk(in + at.column(k), x);
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[i] = m.normalised(x[i] - near);
            }
            if constexpr (CHECKPOINT) {
                const bool hasTail = at.tail && k == at.tailChunk;
                const BlockScale scale = scaleOfLanes<VEC>(x, has, tail, hasTail, a.format);
                if (has) storeCodes<VEC>(codes + at.column(k), encodeChunk<VEC>(x, scale, a.format));
                if (hasTail) codes[at.tailColumn] = encodeOne(tail, scale, a.format);
                if (at.column(k) % kCheckpointBlock == 0 && at.column(k) < a.columns) scales[at.column(k) / kCheckpointBlock] = scale.scale;
            }
            if (has) {
                float weight[VEC], bias[VEC];
                loadParameters<T>(a.weight, a.parametersAreFloat, 1.0f, at.column(k), true, weight);
                loadParameters<T>(a.bias, a.parametersAreFloat, 0.0f, at.column(k), true, bias);
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[i] = x[i] * weight[i] + bias[i];
                storeChunk(out + at.column(k), x);
            }
        }
        if (at.tail) {
            out[at.tailColumn] = narrow<T>(tail * loadParameter<T>(a.weight, a.parametersAreFloat, 1.0f, at.tailColumn, true) +
                                           loadParameter<T>(a.bias, a.parametersAreFloat, 0.0f, at.tailColumn, true));
        }
    }
}

// What a lane needs of a row, as it was loaded.
template <typename T, int K, bool CODES>
struct RowLoaded {
    Words4 error[K];
    Words4 input[CODES ? 1 : K];
    Codes<kVec<T>> codes[CODES ? K : 1];
    float scale[CODES ? K : 1];
    float mean, rstd;
    T tailError, tailInput;
    u32 tailCode;
    float tailScale;

    template <int LANES, Fit FIT>
    __device__ __forceinline__ void load(const BackwardArgs& a, const RowLayout<T, LANES, FIT>& at, u32 row) {
        constexpr int VEC = kVec<T>;
        const T* dy = rowPointer<const T>(a.error, row, a.innerRows);
        const T* x = CODES ? nullptr : rowPointer<const T>(a.input, row, a.innerRows);
        const u8* code = a.codes + (i64)row * a.columns;
        const float* scales = a.scales + (i64)row * a.blocksPerRow;
        mean = CODES ? 0.0f : a.mean[row];
        rstd = a.rstd[row];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const u32 from = at.source(k);
            error[k] = at.works(k) ? loadWords(dy + from) : Words4{};
            if constexpr (CODES) {
                codes[k] = at.works(k) ? loadCodes<VEC>(code + from) : Codes<VEC>{};
                scale[k] = at.works(k) ? scales[from / kCheckpointBlock] : 0.0f;
            } else {
                input[k] = at.works(k) ? loadWords(x + from) : Words4{};
            }
        }
        tailError = tailInput = narrow<T>(0.0f);
        tailCode = 0;
        tailScale = 0.0f;
        if (at.tail) {
            tailError = dy[at.tailColumn];
            if constexpr (CODES) {
                tailCode = code[at.tailColumn];
                tailScale = scales[at.tailColumn / kCheckpointBlock];
            } else {
                tailInput = x[at.tailColumn];
            }
        }
    }

    // dy and h of chunk k; zeros for dy where the lane has none.
    __device__ __forceinline__ void chunk(const BackwardArgs& a, int k, float (&dy)[kVec<T>], float (&h)[kVec<T>]) const {
        unpack<T>(error[k], dy);
        if constexpr (CODES) {
            decode<kVec<T>>(codes[k], a.format, scale[k], h);
        } else {
            unpack<T>(input[k], h);
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i) h[i] = (h[i] - mean) * rstd;
        }
    }
    __device__ __forceinline__ float tailRow(const BackwardArgs& a) const {
        return CODES ? decodeOne(tailCode, a.format, tailScale) : (widen(tailInput) - mean) * rstd;
    }
};

// Four of a lane's sums.
template <int K, int VEC>
__device__ __forceinline__ Elements<float> quarter(const float (&v)[K][VEC], int q) {
    return {{v[q * 4 / VEC][q * 4 % VEC], v[q * 4 / VEC][q * 4 % VEC + 1], v[q * 4 / VEC][q * 4 % VEC + 2], v[q * 4 / VEC][q * 4 % VEC + 3]}};
}

// Rows of at most LANES * K chunks, a team of LANES lanes per row.  The blocks stay and take every gridDim-th row; a row is loaded while
// the one before it is worked on, where the lanes have the registers for both.
// bf16 16384 x 4096 takes 69.6 us (5.9 TB/s with the shares), 8192 x 8192 from e4m3 codes 58.3 us (6.1 TB/s).
template <typename T, int LANES, int K, bool CODES, Fit FIT>
__global__ __launch_bounds__(kBackwardThreads<LANES>) void layerNormBackward(BackwardArgs a) {
    constexpr int VEC = kVec<T>, THREADS = kBackwardThreads<LANES>, TEAMS = THREADS / LANES;
    constexpr bool AHEAD = LANES < 1024;  // of 128 registers per lane this row takes 112 to 128
    __shared__ float shared[2][THREADS / 64][2];
    const RowLayout<T, LANES, FIT> at(a.columns, threadIdx.x % LANES);
    const u32 team = teamOfBlock<LANES>(), rows = rowsInUse(a.extent), step = gridDim.x * TEAMS;
    u32 row = blockIdx.x * TEAMS + team;
    RowLoaded<T, K, CODES> now, next;
    if (AHEAD && row < rows) now.load(a, at, row);
    float weightSum[K][VEC] = {}, errorSum[K][VEC] = {}, weight[K][VEC];
#pragma unroll
    for (int k = 0; AHEAD && k < K; ++k) loadParameters<T>(a.weight, a.parametersAreFloat, 1.0f, at.source(k), at.works(k), weight[k]);
    const float tailWeight = loadParameter<T>(a.weight, a.parametersAreFloat, 1.0f, at.tailColumn, at.tail);
    float tailWeightSum = 0.0f, tailErrorSum = 0.0f;
    loadsArrived();
    int turn = 0;
    u32 first = blockIdx.x * TEAMS;
    for (u32 share = 0; share < a.sharesOfBlock; ++share) {
        // The teams of a block take their turns together: those of several wavefronts synchronise.
        for (u32 turns = a.sharesOfBlock == 1 ? ~0u : kRowsOfShare; first < rows && turns != 0; first += step, row += step, --turns) {
            const bool mine = row < rows;
            float h[K][VEC], g[K][VEC], tail = 0.0f, tailRow = 0.0f;
            float sums[2] = {0.0f, 0.0f};
            if (mine) {
                if constexpr (AHEAD) {
                    if (row + step < rows) next.load(a, at, row + step);
                } else {
                    now.load(a, at, row);
                }
                tail = widen(now.tailError);
                tailRow = now.tailRow(a);
                // where a lane has no element, h is 0 - mean times rstd, which may be no number
                tailWeightSum += at.tail ? tail * tailRow : 0.0f;
                tailErrorSum += tail;
                tail *= tailWeight;
                sums[0] = tail;
                sums[1] = at.tail ? tail * tailRow : 0.0f;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    now.chunk(a, k, g[k], h[k]);
                    if constexpr (!AHEAD) loadParameters<T>(a.weight, a.parametersAreFloat, 1.0f, at.source(k), at.works(k), weight[k]);
                    float ofChunk[2] = {0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        weightSum[k][i] += g[k][i] * h[k][i];
                        errorSum[k][i] += g[k][i];
                        g[k][i] *= weight[k][i];
                        ofChunk[0] += g[k][i];
                        ofChunk[1] += g[k][i] * h[k][i];
                    }
                    sums[0] += at.has(k) ? ofChunk[0] : 0.0f;
                    sums[1] += at.has(k) ? ofChunk[1] : 0.0f;
                }
            }
            sumTeam<LANES>(sums, shared[turn]);
            turn ^= 1;
            if (mine) {
                const float ofError = average(sums[0], a.columns, a.inverse), ofProduct = average(sums[1], a.columns, a.inverse);
                T* out = rowPointer<T>(a.gradient, row, a.innerRows);
#pragma unroll
                for (int k = 0; k < K; ++k) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) g[k][i] = now.rstd * (g[k][i] - ofError - h[k][i] * ofProduct);
                    if (at.works(k)) storeChunk(out + at.source(k), g[k]);
                }
                if (at.tail) out[at.tailColumn] = narrow<T>(now.rstd * (tail - ofError - tailRow * ofProduct));
                if constexpr (AHEAD) {
                    __builtin_amdgcn_sched_barrier(0);  // the stores first: what is copied here has to have arrived
                    now = next;
                }
            }
        }
        if (a.partials == nullptr) return;
        float* mine = a.partials + ((i64)share * gridDim.x + blockIdx.x) * 2 * a.columns;
        if constexpr (TEAMS > 1) {
            // The upper half of the teams gives its sums to the lower half until one team has them all; the block stores them together, 16
            // adjacent bytes per lane.
            constexpr u32 PARTS = K * VEC / 4, ROW = LANES * VEC / 4;
            __shared__ Words4 given[TEAMS / 2][2][PARTS][LANES];
            __shared__ float givenTail[TEAMS / 2][2][FIT == Fit::Any ? LANES : 1];
            u32 thread = threadIdx.x;
            asm volatile("" : "+v"(thread));  // what follows from it is worked out here and takes no registers from the rows
            const u32 lane = thread % LANES;
            const auto give = [&](u32 to) {
#pragma unroll
                for (u32 q = 0; q < PARTS; ++q) {
                    given[to][0][q][lane] = __builtin_bit_cast(Words4, quarter(weightSum, q));
                    given[to][1][q][lane] = __builtin_bit_cast(Words4, quarter(errorSum, q));
                }
            };
#pragma unroll
            for (u32 half = TEAMS / 2; half >= 1; half /= 2) {
                if (team >= half && team < 2 * half) {
                    give(team - half);
                    if constexpr (FIT == Fit::Any) {
                        givenTail[team - half][0][lane] = tailWeightSum;
                        givenTail[team - half][1][lane] = tailErrorSum;
                    }
                }
                __syncthreads();
                if (team < half) {
#pragma unroll
                    for (u32 q = 0; q < PARTS; ++q) {
                        const Elements<float> w = __builtin_bit_cast(Elements<float>, given[team][0][q][lane]);
                        const Elements<float> e = __builtin_bit_cast(Elements<float>, given[team][1][q][lane]);
#pragma unroll
                        for (u32 i = 0; i < 4; ++i) {
                            weightSum[q * 4 / VEC][q * 4 % VEC + i] += w.e[i];
                            errorSum[q * 4 / VEC][q * 4 % VEC + i] += e.e[i];
                        }
                    }
                    if constexpr (FIT == Fit::Any) {
                        tailWeightSum += givenTail[team][0][lane];
                        tailErrorSum += givenTail[team][1][lane];
                    }
                    if (half == 1) give(0);
                }
                __syncthreads();
            }
            for (u32 t = thread; t < 2 * K * ROW; t += THREADS) {
                const u32 which = t / (K * ROW), k = t / ROW % K, of = t % ROW / (VEC / 4), q = k * (VEC / 4) + t % (VEC / 4);
                const u32 column = t % (K * ROW) * 4;
                if (column < at.whole) *reinterpret_cast<Words4OfFloats*>(mine + which * a.columns + column) = given[0][which][q][of];
            }
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!at.has(k)) continue;
                storeFloats<VEC>(mine + at.column(k), weightSum[k]);
                storeFloats<VEC>(mine + a.columns + at.column(k), errorSum[k]);
            }
        }
        if (at.tail && team == 0) {
            mine[at.tailColumn] = tailWeightSum;
            mine[a.columns + at.tailColumn] = tailErrorSum;
        }
        if (share + 1 == a.sharesOfBlock) return;
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) weightSum[k][i] = errorSum[k][i] = 0.0f;
        }
        tailWeightSum = tailErrorSum = 0.0f;
        if constexpr (TEAMS > 1) __syncthreads();  // what the teams gave each other has been read
    }
}

// Rows of any length: the input's gradient, a block of 1024 lanes per row that reads it twice ...
template <typename T, bool CODES>
__device__ __forceinline__ void longRow(const BackwardArgs& a, u32 row, float (*shared)[2]) {
    constexpr int VEC = kVec<T>, LANES = 1024;
    const RowLayout<T, LANES, Fit::Any> at(a.columns, threadIdx.x);
    const float mean = CODES ? 0.0f : a.mean[row], rstd = a.rstd[row];
    const T* error = rowPointer<const T>(a.error, row, a.innerRows);
    const T* input = CODES ? nullptr : rowPointer<const T>(a.input, row, a.innerRows);
    const u8* codes = a.codes + (i64)row * a.columns;
    const float* scales = a.scales + (i64)row * a.blocksPerRow;
    const auto chunk = [&](int k, float(&g)[VEC], float(&h)[VEC]) {
        const u32 column = at.column(k);
        float weight[VEC];
        loadChunk(error + column, g);
        if constexpr (CODES) {
            decode<VEC>(loadCodes<VEC>(codes + column), a.format, scales[column / kCheckpointBlock], h);
        } else {
            loadChunk(input + column, h);
#pragma unroll
            for (int i = 0; i < VEC; ++i) h[i] = (h[i] - mean) * rstd;
        }
        loadParameters<T>(a.weight, a.parametersAreFloat, 1.0f, column, true, weight);
#pragma unroll
        for (int i = 0; i < VEC; ++i) g[i] *= weight[i];
    };
    float tail = 0.0f, tailRow = 0.0f;
    if (at.tail) {
        tail = widen(error[at.tailColumn]) * loadParameter<T>(a.weight, a.parametersAreFloat, 1.0f, at.tailColumn, true);
        tailRow = CODES ? decodeOne(codes[at.tailColumn], a.format, scales[at.tailColumn / kCheckpointBlock]) : (widen(input[at.tailColumn]) - mean) * rstd;
    }
    float h[VEC], g[VEC];
    LongSum errorOfLane, productOfLane;
    for (int k = 0; at.has(k); ++k) {
        chunk(k, g, h);
        float ofChunk[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            ofChunk[0] += g[i];
            ofChunk[1] += g[i] * h[i];
        }
        errorOfLane.add(ofChunk[0]);
        productOfLane.add(ofChunk[1]);
    }
    float sums[2] = {errorOfLane.sum + tail, productOfLane.sum + tail * tailRow};
    sumTeam<LANES>(sums, shared);
    const float ofError = average(sums[0], a.columns, a.inverse), ofProduct = average(sums[1], a.columns, a.inverse);
    T* out = rowPointer<T>(a.gradient, row, a.innerRows);
    for (int k = 0; at.has(k); ++k) {
        chunk(k, g, h);
#pragma unroll
        for (int i = 0; i < VEC; ++i) g[i] = rstd * (g[i] - ofError - h[i] * ofProduct);
        storeChunk(out + at.column(k), g);
    }
    if (at.tail) out[at.tailColumn] = narrow<T>(rstd * (tail - ofError - tailRow * ofProduct));
}

template <typename T, bool CODES>
__global__ __launch_bounds__(1024) void layerNormBackwardLong(BackwardArgs a) {
    __shared__ float shared[2][16][2];
    const u32 rows = rowsInUse(a.extent);
    int turn = 0;
    for (u32 row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) longRow<T, CODES>(a, row, shared[turn]);
}

// (bf16 4096 x 20000: 214 us in all, 2.3 TB/s) ... and the parameter gradients: LANES chunks of columns per block (one element of the tail
// for the lanes behind the last whole chunk) by THREADS / LANES rows at a time, every shares-th group of them.  They need nothing that the
// rows' sums give, so a single share is the result.
// Chunks of columns that a block takes for the parameter gradients: a cache line of 128 bytes, so that a block of 1024 lanes takes 128 rows
// at a time (bf16 512 x 1024 in one launch: 6.9 us, with 16 chunks 9.4); twice that where there are over a thousand chunks, and blocks
// enough (fp32 200 x 8192: 7.4 us, with 8 chunks 9.1).
constexpr int columnLanes(int chunks) { return chunks > 1024 ? 16 : 8; }
constexpr int kManyChunks = 1 << 20;  // of rows of any length
template <typename T, bool CODES, int THREADS, int LANES>
__device__ __forceinline__ void columnGradients(const BackwardArgs& a, u32 block, u32 share, u32 shares) {
    constexpr int VEC = kVec<T>, GROUPS = THREADS / LANES, WAVES = THREADS / 64, WIDTH = LANES * VEC;
    __shared__ float added[2][WAVES][WIDTH];
    const u32 lane = threadIdx.x % LANES, group = threadIdx.x / LANES, rows = rowsInUse(a.extent);
    const u32 chunks = a.columns / VEC;
    const auto columnOf = [&](u32 l) {
        const u32 at = block * LANES + l;
        return at < chunks ? at * VEC : chunks * VEC + (at - chunks);
    };
    const auto countOf = [&](u32 l) { return columnOf(l) >= a.columns ? 0u : block * LANES + l < chunks ? (u32)VEC : 1u; };
    const u32 column = columnOf(lane), count = countOf(lane);
    float sums[2][VEC] = {};
    if (count != 0) {
#pragma unroll 2
        for (u32 row = share * GROUPS + group; row < rows; row += shares * GROUPS) {
            const T* error = rowPointer<const T>(a.error, row, a.innerRows) + column;
            const T* input = CODES ? nullptr : rowPointer<const T>(a.input, row, a.innerRows) + column;
            const u8* codes = a.codes + (i64)row * a.columns + column;
            const float* scale = a.scales + (i64)row * a.blocksPerRow + column / kCheckpointBlock;
            const float mean = CODES ? 0.0f : a.mean[row], rstd = CODES ? 0.0f : a.rstd[row];
            float h[VEC] = {}, g[VEC] = {};
            if (count == VEC) {
                loadChunk(error, g);
                if constexpr (CODES) {
                    decode<VEC>(loadCodes<VEC>(codes), a.format, *scale, h);
                } else {
                    loadChunk(input, h);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) h[i] = (h[i] - mean) * rstd;
                }
            } else {
                g[0] = widen(*error);
                h[0] = CODES ? decodeOne(*codes, a.format, *scale) : (widen(*input) - mean) * rstd;
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                sums[0][i] += g[i] * h[i];
                sums[1][i] += g[i];
            }
        }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if (LANES == 8) sums[p][i] += bitsF32(rotated<0x128>(f32Bits(sums[p][i])));  // two rows in 16 lanes
            const float sum = sumRowsOfWave(sums[p][i]);
            if (threadIdx.x % 64 < LANES) added[p][threadIdx.x / 64][lane * VEC + i] = sum;
        }
    }
    __syncthreads();
    for (u32 t = threadIdx.x; t < 2 * WIDTH; t += THREADS) {
        const u32 p = t / WIDTH, c = t % WIDTH;
        if (c % VEC >= countOf(c / VEC)) continue;
        const u32 to = columnOf(c / VEC) + c % VEC;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) sum += added[p][w][c];
        if (a.partials != nullptr) {
            a.partials[((i64)share * 2 + p) * a.columns + to] = sum;
        } else if (void* out = p == 0 ? a.weightGradient : a.biasGradient; out != nullptr) {
            if (a.parametersAreFloat) {
                static_cast<float*>(out)[to] = sum;
            } else {
                static_cast<T*>(out)[to] = narrow<T>(sum);
            }
        }
    }
}
template <typename T, bool CODES>
__global__ __launch_bounds__(256) void layerNormColumns(BackwardArgs a) {
    columnGradients<T, CODES, 256, columnLanes(kManyChunks)>(a, blockIdx.x, blockIdx.y, gridDim.y);
}

// A few rows in one launch: the first blocks do columns, the others one row per team.  Everything is read twice, which costs less than
// a second launch while there is little of it (fp16 37 x 513 from int8 codes: 5.1 us, a launch's time and two trips to memory).
template <typename T, int LANES, int K, bool CODES>
__global__ __launch_bounds__(1024) void layerNormBackwardFew(BackwardArgs a, u32 columnBlocks) {
    constexpr int VEC = kVec<T>, THREADS = 1024, TEAMS = THREADS / LANES;
    if (blockIdx.x < columnBlocks) return columnGradients<T, CODES, THREADS, columnLanes(LANES * K)>(a, blockIdx.x, 0, 1);
    __shared__ float shared[THREADS / 64][2];
    const RowLayout<T, LANES, Fit::Any> at(a.columns, threadIdx.x % LANES);
    const u32 row = (blockIdx.x - columnBlocks) * TEAMS + teamOfBlock<LANES>();
    const bool mine = row < rowsInUse(a.extent);
    RowLoaded<T, K, CODES> now;
    float h[K][VEC], g[K][VEC], weight[K][VEC], tail = 0.0f, tailRow = 0.0f;
    float sums[2] = {0.0f, 0.0f};
    if (mine) {
        now.load(a, at, row);
        // every load is on its way before the first result is waited for
#pragma unroll
        for (int k = 0; k < K; ++k) loadParameters<T>(a.weight, a.parametersAreFloat, 1.0f, at.column(k), at.has(k), weight[k]);
        const float tailWeight = loadParameter<T>(a.weight, a.parametersAreFloat, 1.0f, at.tailColumn, at.tail);
        tail = widen(now.tailError) * tailWeight;
        tailRow = now.tailRow(a);
        sums[0] = tail;
        sums[1] = at.tail ? tail * tailRow : 0.0f;  // where a lane has no element, h is 0 - mean times rstd, which may be no number
#pragma unroll
        for (int k = 0; k < K; ++k) {
            now.chunk(a, k, g[k], h[k]);
            float ofChunk[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                g[k][i] *= weight[k][i];
                ofChunk[0] += g[k][i];
                ofChunk[1] += g[k][i] * h[k][i];
            }
            sums[0] += ofChunk[0];
            sums[1] += at.has(k) ? ofChunk[1] : 0.0f;
        }
    }
    sumTeam<LANES>(sums, shared);
    if (!mine) return;
    const float ofError = average(sums[0], a.columns, a.inverse), ofProduct = average(sums[1], a.columns, a.inverse);
    T* out = rowPointer<T>(a.gradient, row, a.innerRows);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) g[k][i] = now.rstd * (g[k][i] - ofError - h[k][i] * ofProduct);
        if (at.has(k)) storeChunk(out + at.column(k), g[k]);
    }
    if (at.tail) out[at.tailColumn] = narrow<T>(now.rstd * (tail - ofError - tailRow * ofProduct));
}
template <typename T, bool CODES>
__global__ __launch_bounds__(1024) void layerNormBackwardFewLong(BackwardArgs a, u32 columnBlocks) {
    if (blockIdx.x < columnBlocks) return columnGradients<T, CODES, 1024, columnLanes(kManyChunks)>(a, blockIdx.x, 0, 1);
    __shared__ float shared[16][2];
    if (blockIdx.x - columnBlocks < rowsInUse(a.extent)) longRow<T, CODES>(a, blockIdx.x - columnBlocks, shared);
}

// The sum of `shares` shares [2][columns] of one of the parameter gradients (blockIdx.y: 0 weight, 1 bias): 32 columns by 128 shares at a
// time, 4 columns per lane, so that a lane has few additions to wait for.  256 shares of 4096 columns take 4.6 us, half of that a
// launch's own time.
template <typename W>
__global__ __launch_bounds__(1024) void addShares(const float* partials, u32 shares, u32 columns, W* weightGradient, W* biasGradient) {
    __shared__ float added[16][32];
    const u32 column = blockIdx.x * 32 + threadIdx.x % 8 * 4, wave = threadIdx.x / 64;
    W* out = blockIdx.y == 0 ? weightGradient : biasGradient;
    if (out == nullptr) return;
    LongSum sums[4];
    if (column + 4 <= columns) {
#pragma unroll 4
        for (u32 s = threadIdx.x / 8; s < shares; s += 128) {
            const Elements<float> x = __builtin_bit_cast(Elements<float>, *reinterpret_cast<const Words4OfFloats*>(partials + ((i64)s * 2 + blockIdx.y) * columns + column));
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[i].add(x.e[i]);
        }
    } else {
        for (u32 s = threadIdx.x / 8; s < shares; s += 128) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (column + i < columns) sums[i].add(partials[((i64)s * 2 + blockIdx.y) * columns + column + i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // the eight shares of a wavefront
        const float sum = sumRowsOfWave(sums[i].sum + bitsF32(rotated<0x128>(f32Bits(sums[i].sum))));
        if (threadIdx.x % 64 < 8) added[wave][threadIdx.x % 8 * 4 + i] = sum;
    }
    __syncthreads();
    const u32 mine = blockIdx.x * 32 + threadIdx.x;
    if (threadIdx.x >= 32 || mine >= columns) return;
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) total += added[w][threadIdx.x];
    out[mine] = narrow<W>(total);
}

// ---- which kernel ------------------------------------------------------------------------------------------------------------------------

typedef void (*Forward)(ForwardArgs);
typedef void (*Backward)(BackwardArgs);
typedef void (*BackwardFew)(BackwardArgs, u32);

// Lanes of a team and chunks of a lane; lanes 0: rows of any length.
struct Shape {
    int lanes, chunks;
};

// The smallest team that holds a row with 16 elements per lane (8 in rows of at most 512, 16 bytes in rows of at most 256).  More
// elements per lane need registers that the next row's loads are worth more in, fewer leave the folds more of the time: bf16 rows of 8192
// backward take 58 us with 512 lanes of 16 elements and 64 us with 1024 of 8 (8192 rows, from a checkpoint), rows of 4096 forward 47 us
// with 256 lanes of 16 and 52 us with 512 of 8 (16384 rows).  Teams of 3, 6 and 12 wavefronts beside the powers of two keep at least two
// thirds of the lanes busy; `powers` asks for powers of two, of which any divides a block of 1024.
Shape shapeOf(uint32_t columns, int vec, bool powers) {
    if (columns <= kCheckpointBlock) return {kCheckpointBlock / vec, 1};
    if (columns <= 2 * kCheckpointBlock) return {2 * kCheckpointBlock / vec, 1};
    if (columns <= 512) return {64, 8 / vec};
    for (int lanes : {64, 128, 192, 256, 384, 512, 768, 1024})
        if (columns <= 16u * lanes && !(powers && lanes % 3 == 0)) return {lanes, 16 / vec};
    return {0, 0};
}
bool isFull(Shape s, uint32_t columns, int vec) { return s.lanes >= 64 && columns == (uint32_t)(s.lanes * s.chunks * vec); }
bool isWhole(Shape s, uint32_t columns, int vec) { return s.lanes >= 64 && columns % vec == 0; }

template <typename T, bool CHECKPOINT, Fit FIT>
Forward forwardOf(Shape s) {
    constexpr int VEC = kVec<T>, K = 16 / VEC;
    switch (s.lanes) {
        case 0: return layerNormForwardLong<T, CHECKPOINT>;
        case 64:
            if (s.chunks == K) return layerNormForward<T, 64, K, CHECKPOINT, FIT>;
            if (s.chunks == 8 / VEC) return layerNormForward<T, 64, 8 / VEC, CHECKPOINT, FIT>;
            return layerNormForward<T, 64, 1, CHECKPOINT, FIT>;
        case 128: return layerNormForward<T, 128, K, CHECKPOINT, FIT>;
        case 192: return layerNormForward<T, 192, K, CHECKPOINT, FIT>;
        case 256: return layerNormForward<T, 256, K, CHECKPOINT, FIT>;
        case 384: return layerNormForward<T, 384, K, CHECKPOINT, FIT>;
        case 512: return layerNormForward<T, 512, K, CHECKPOINT, FIT == Fit::Whole ? Fit::Blocks : FIT>;
        case 768: return layerNormForward<T, 768, K, CHECKPOINT, FIT == Fit::Whole ? Fit::Blocks : FIT>;
        case 1024: return layerNormForward<T, 1024, K, CHECKPOINT, FIT == Fit::Whole ? Fit::Blocks : FIT>;
        case 32: return layerNormForward<T, 32, 1, CHECKPOINT, Fit::Any>;
        default:
            if constexpr (VEC == 8) return layerNormForward<T, 16, 1, CHECKPOINT, Fit::Any>;
            return nullptr;
    }
}
// Full rows gain: bf16 8192 x 8192 with a checkpoint takes 61.2 us, as any row 63.2.  Whole ones of 16-bit elements do without the tail's
// registers: 13107 x 5120 with a checkpoint 64.7 us and 68.3.  From 512 lanes on they are rows of whole blocks instead, whose loads have no
// branches: 6096 x 11008 46.0 us, as any row 55.8, with a checkpoint 59.7 and 78.4 (smaller teams gain nothing by that, and 52428 x 1280
// loses: 52.0 and 47.6).  fp32 gains by neither.
bool isWholeForward(Shape s, uint32_t columns, int vec) { return vec == 8 && s.lanes >= 64 && columns % (s.lanes >= 512 ? kCheckpointBlock : vec) == 0; }
template <typename T, bool CHECKPOINT>
Forward forwardOf(Shape s, bool whole, bool full) {
    if (full) return forwardOf<T, CHECKPOINT, Fit::Full>(s);
    if constexpr (sizeof(T) == 2) {
        if (whole) return forwardOf<T, CHECKPOINT, Fit::Whole>(s);
    }
    return forwardOf<T, CHECKPOINT, Fit::Any>(s);
}
template <typename T>
Forward forwardOf(Shape s, bool checkpoint, bool whole, bool full) {
    return checkpoint ? forwardOf<T, true>(s, whole, full) : forwardOf<T, false>(s, whole, full);
}
// Forward blocks per CU, by the wavefronts that keep memory busy; more of them only compete.  Eight where a lane has 64 bytes of a row or
// every lane has 32 (fp32 20000 x 1537 with a checkpoint 57.5 us, with sixteen 64.5; bf16 16384 x 4096 59.4 and 64.0), twelve where two
// thirds of the lanes have 32 and there are no codes to work out (18724 x 3584 45.4 and 49.7, 87381 x 768 47.4 and 50.5), else sixteen
// (52428 x 1280 47.6 us, with twelve 56.0; 65536 x 512 23.7 and 25.0).  Teams of six wavefronts: two of them, three for whole rows with a
// checkpoint (10922 x 5888 61.0 and 65.5), whose registers allow it.
uint32_t forwardBlocks(Shape s, uint32_t columns, int vec, uint32_t threads, bool checkpoint, bool whole, bool full) {
    if (threads == 384) return whole && !full && checkpoint ? 3 : 2;
    uint32_t waves = 16;
    if (s.chunks == 4 || (s.chunks == 2 && full)) {
        waves = 8;
    } else if (s.chunks == 2 && !checkpoint && s.lanes <= 256 && columns * 3 >= (uint32_t)(s.lanes * s.chunks * vec) * 2) {
        waves = 12;
    }
    return std::max(1u, (waves * 64 + threads / 2) / threads);
}
// The team of a backward row.  Blocks of 768 lanes have registers for fp32 rows where those are full, from codes whole ones too, and in
// teams of all 768 any whole ones; other rows take the next power of two (from the input 13107 x 2560 67.7 us, with 192 lanes 85.5; 6552 x
// 5121 74.7 and 93.8; 3048 x 11008 83.6 with 1024 lanes, as whole rows of 768 73.8; forward and backward from codes 16360 x 2051 124.5 us,
// with 192 lanes 132.2; 5462 x 6143 122.3 and 126.8; 3727 x 9001 137.0 and 141.4, but 8190 x 4097 127.9 and 126.7).
Shape backwardShapeOf(uint32_t columns, int vec, bool codes) {
    const Shape s = shapeOf(columns, vec, false);
    const bool room = vec == 8 || s.lanes % 3 != 0 || isFull(s, columns, vec) || ((codes || s.lanes == 768) && isWhole(s, columns, vec));
    return room ? s : shapeOf(columns, vec, true);
}
template <typename T, int LANES, bool CODES, Fit FIT>
Backward backwardOfThree() {
    constexpr bool ROOM = sizeof(T) == 2 || FIT == Fit::Full || ((CODES || LANES == 768) && FIT == Fit::Whole);
    if constexpr (ROOM) return layerNormBackward<T, LANES, 16 / kVec<T>, CODES, FIT>;
    return nullptr;
}
template <typename T, bool CODES, Fit FIT>
Backward backwardOf(Shape s) {
    constexpr int VEC = kVec<T>, K = 16 / VEC;
    switch (s.lanes) {
        case 0: return layerNormBackwardLong<T, CODES>;
        case 64:
            if (s.chunks == K) return layerNormBackward<T, 64, K, CODES, FIT>;
            if (s.chunks == 8 / VEC) return layerNormBackward<T, 64, 8 / VEC, CODES, FIT>;
            return layerNormBackward<T, 64, 1, CODES, FIT>;
        case 128: return layerNormBackward<T, 128, K, CODES, FIT>;
        case 192: return backwardOfThree<T, 192, CODES, FIT>();
        case 256: return layerNormBackward<T, 256, K, CODES, FIT>;
        case 384: return backwardOfThree<T, 384, CODES, FIT>();
        case 512: return layerNormBackward<T, 512, K, CODES, FIT>;
        case 768: return backwardOfThree<T, 768, CODES, FIT>();
        case 1024: return layerNormBackward<T, 1024, K, CODES, FIT>;
        case 32: return layerNormBackward<T, 32, 1, CODES, Fit::Any>;
        default:
            if constexpr (VEC == 8) return layerNormBackward<T, 16, 1, CODES, Fit::Any>;
            return nullptr;
    }
}
// Full rows gain most (bf16 from codes 16384 x 4096: 57.4 us, as any row 67.6; from the input 67.9 and 71.1).  From codes, whose three
// loads per chunk are in branches otherwise, other rows that end with a whole chunk gain too (8192 x 7168 67.1 -> 63.9 us, 32768 x 768
// forward and backward 58.7 -> 49.0); from the input they lose (16384 x 2560 43.6 -> 46.2).
template <typename T>
Backward backwardOf(Shape s, bool codes, bool whole, bool full) {
    if (!codes) {
        if constexpr (sizeof(T) == 4) {
            if (whole && !full && s.lanes == 768) return backwardOfThree<T, 768, false, Fit::Whole>();
        }
        return full ? backwardOf<T, false, Fit::Full>(s) : backwardOf<T, false, Fit::Any>(s);
    }
    return full ? backwardOf<T, true, Fit::Full>(s) : whole ? backwardOf<T, true, Fit::Whole>(s) : backwardOf<T, true, Fit::Any>(s);
}
template <typename T, bool CODES>
BackwardFew fewOf(Shape s) {
    constexpr int VEC = kVec<T>, K = 16 / VEC;
    switch (s.lanes) {
        case 0: return layerNormBackwardFewLong<T, CODES>;
        case 64:
            if (s.chunks == K) return layerNormBackwardFew<T, 64, K, CODES>;
            if (s.chunks == 8 / VEC) return layerNormBackwardFew<T, 64, 8 / VEC, CODES>;
            return layerNormBackwardFew<T, 64, 1, CODES>;
        case 128: return layerNormBackwardFew<T, 128, K, CODES>;
        case 256: return layerNormBackwardFew<T, 256, K, CODES>;
        case 512: return layerNormBackwardFew<T, 512, K, CODES>;
        case 1024: return layerNormBackwardFew<T, 1024, K, CODES>;
        case 32: return layerNormBackwardFew<T, 32, 1, CODES>;
        default:
            if constexpr (VEC == 8) return layerNormBackwardFew<T, 16, 1, CODES>;
            return nullptr;
    }
}
template <typename T>
BackwardFew fewOf(Shape s, bool codes) {
    return codes ? fewOf<T, true>(s) : fewOf<T, false>(s);
}
template <typename T>
Backward columnsOf(bool codes) {
    return codes ? layerNormColumns<T, true> : layerNormColumns<T, false>;
}

// Rows up to which one launch that reads everything twice is faster than two: bf16 512 x 1024 takes 6.9 us against 7.5, 512 x 4096 7.8
// against 11.3, 768 x 1024 8.9 against 7.6; short rows 384 x 300 6.8 against 6.9, 512 x 300 8.1 against 6.9.
uint32_t fewRows(uint32_t columns) { return columns <= 512 ? 384 : 512; }

RowsOf rowsOf(const thorhip_rows& r) { return {static_cast<char*>(r.data), r.outer, r.inner}; }

uint32_t ceilDiv(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

int computeUnits() {
    int device = 0, units = 0;
    if (hipGetDevice(&device) != hipSuccess || hipDeviceGetAttribute(&units, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess) return 256;
    return units;
}

int load(const void* kernel) {  // a first launch under stream capture must not have to
    hipFuncAttributes attributes;
    THORHIP_TRY(hipFuncGetAttributes(&attributes, kernel));
    return 0;
}

bool knownType(int dtype) { return dtype == THORHIP_FP32 || dtype == THORHIP_FP16 || dtype == THORHIP_BF16; }
bool knownFormat(int dtype) { return dtype == THORHIP_FP8_E4M3 || dtype == THORHIP_FP8_E5M2 || dtype == THORHIP_INT8; }

}  // namespace

extern "C" {

int thorhip_layer_norm_forward(const thorhip_layer_norm* call, void* stream, int launch, char* variant, size_t variant_capacity) {
    THORHIP_REQUIRE(call != nullptr, "thorhip_layer_norm_forward: no call");
    const thorhip_layer_norm& c = *call;
    THORHIP_REQUIRE(knownType(c.dtype), "thorhip_layer_norm_forward: dtype %d", c.dtype);
    THORHIP_REQUIRE(c.parameter_dtype == THORHIP_FP32 || c.parameter_dtype == c.dtype, "thorhip_layer_norm_forward: parameter dtype %d", c.parameter_dtype);
    THORHIP_REQUIRE(c.checkpoint_dtype == 0 || knownFormat(c.checkpoint_dtype), "thorhip_layer_norm_forward: checkpoint dtype %d", c.checkpoint_dtype);
    THORHIP_REQUIRE(c.rows > 0 && c.columns > 0 && c.rows < (1u << 31) && c.columns < (1u << 24), "thorhip_layer_norm_forward: %u rows of %u columns", c.rows,
                    c.columns);
    THORHIP_REQUIRE(c.epsilon > 0.0f && std::isnormal(c.epsilon), "thorhip_layer_norm_forward: epsilon %g", c.epsilon);
    THORHIP_REQUIRE(c.input.data != nullptr && c.output.data != nullptr && c.mean != nullptr && c.rstd != nullptr, "thorhip_layer_norm_forward: NULL tensor");
    THORHIP_REQUIRE(c.checkpoint_dtype == 0 || (c.codes != nullptr && c.scales != nullptr), "thorhip_layer_norm_forward: no checkpoint");
    ForwardArgs a{};
    a.input = rowsOf(c.input);
    a.output = rowsOf(c.output);
    a.weight = c.weight;
    a.bias = c.bias;
    a.mean = c.mean;
    a.rstd = c.rstd;
    a.codes = static_cast<u8*>(c.codes);
    a.scales = c.scales;
    a.extent = {c.extent, c.extent_is_64, c.rows};
    a.columns = c.columns;
    a.innerRows = c.inner_rows;
    a.blocksPerRow = ceilDiv(c.columns, kCheckpointBlock);
    a.parametersAreFloat = c.parameter_dtype == THORHIP_FP32;
    a.format = c.checkpoint_dtype;
    a.epsilon = c.epsilon;
    a.inverse = 1.0f / (float)c.columns;
    const int vec = 16 / thorhip_dtype_size(c.dtype);
    const Shape shape = shapeOf(c.columns, vec, false);
    const bool checkpoint = c.checkpoint_dtype != 0, whole = isWholeForward(shape, c.columns, vec), full = isFull(shape, c.columns, vec);
    const Forward kernel = c.dtype == THORHIP_FP32   ? forwardOf<float>(shape, checkpoint, whole, full)
                           : c.dtype == THORHIP_FP16 ? forwardOf<f16>(shape, checkpoint, whole, full)
                                                     : forwardOf<bf16>(shape, checkpoint, whole, full);
    const uint32_t threads = shape.lanes == 0 ? 1024 : shape.lanes < 128 ? 256 : shape.lanes, teams = shape.lanes == 0 ? 1 : threads / shape.lanes;  // kForwardThreads
    const uint32_t grid = std::min(ceilDiv(c.rows, teams), (uint32_t)computeUnits() * (shape.lanes == 0 ? 2 : forwardBlocks(shape, c.columns, vec, threads, checkpoint, whole, full)));
    if (variant != nullptr && variant_capacity > 0) {
        snprintf(variant, variant_capacity, "layer_norm_forward(lanes=%d,chunks=%d,threads=%u,grid=%u%s)", shape.lanes, shape.chunks, threads, grid,
                 checkpoint ? ",checkpoint" : "");
    }
    if (!launch) return load(reinterpret_cast<const void*>(kernel));
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, (hipStream_t)stream, a);
    THORHIP_TRY(hipGetLastError());
    return 0;
}

int thorhip_layer_norm_backward(const thorhip_layer_norm_gradient* call, void* stream, int launch, size_t* needed_workspace, char* variant,
                                size_t variant_capacity) {
    THORHIP_REQUIRE(call != nullptr, "thorhip_layer_norm_backward: no call");
    const thorhip_layer_norm_gradient& c = *call;
    THORHIP_REQUIRE(knownType(c.dtype), "thorhip_layer_norm_backward: dtype %d", c.dtype);
    THORHIP_REQUIRE(c.parameter_dtype == THORHIP_FP32 || c.parameter_dtype == c.dtype, "thorhip_layer_norm_backward: parameter dtype %d", c.parameter_dtype);
    THORHIP_REQUIRE(c.checkpoint_dtype == 0 || knownFormat(c.checkpoint_dtype), "thorhip_layer_norm_backward: checkpoint dtype %d", c.checkpoint_dtype);
    THORHIP_REQUIRE(c.rows > 0 && c.columns > 0 && c.rows < (1u << 31) && c.columns < (1u << 24), "thorhip_layer_norm_backward: %u rows of %u columns", c.rows,
                    c.columns);
    THORHIP_REQUIRE(c.error.data != nullptr && c.input_gradient.data != nullptr && c.rstd != nullptr, "thorhip_layer_norm_backward: NULL tensor");
    const bool codes = c.checkpoint_dtype != 0;
    THORHIP_REQUIRE(codes ? c.codes != nullptr && c.scales != nullptr : c.input.data != nullptr && c.mean != nullptr, "thorhip_layer_norm_backward: nothing saved");
    BackwardArgs a{};
    a.error = rowsOf(c.error);
    a.input = rowsOf(c.input);
    a.gradient = rowsOf(c.input_gradient);
    a.weight = c.weight;
    a.mean = c.mean;
    a.rstd = c.rstd;
    a.codes = static_cast<const u8*>(c.codes);
    a.scales = c.scales;
    a.extent = {c.extent, c.extent_is_64, c.rows};
    a.columns = c.columns;
    a.innerRows = c.inner_rows;
    a.blocksPerRow = ceilDiv(c.columns, kCheckpointBlock);
    a.parametersAreFloat = c.parameter_dtype == THORHIP_FP32;
    a.format = c.checkpoint_dtype;
    a.inverse = 1.0f / (float)c.columns;
    a.sharesOfBlock = 1;
    const bool parameters = c.weight_gradient != nullptr || c.bias_gradient != nullptr;
    const int vec = 16 / thorhip_dtype_size(c.dtype);
    a.weightGradient = c.weight_gradient;
    a.biasGradient = c.bias_gradient;
    const uint32_t units = (uint32_t)computeUnits();
    const auto columnBlocksOf = [&](const Shape& s) { return ceilDiv(c.columns / vec + c.columns % vec, columnLanes(s.lanes == 0 ? kManyChunks : s.lanes * s.chunks)); };
    if (parameters && c.rows <= fewRows(c.columns)) {
        const Shape shape = shapeOf(c.columns, vec, true);
        const BackwardFew few = c.dtype == THORHIP_FP32 ? fewOf<float>(shape, codes) : c.dtype == THORHIP_FP16 ? fewOf<f16>(shape, codes) : fewOf<bf16>(shape, codes);
        const uint32_t columnBlocks = columnBlocksOf(shape), rowBlocks = ceilDiv(c.rows, shape.lanes == 0 ? 1 : 1024 / shape.lanes);
        if (needed_workspace != nullptr) *needed_workspace = 0;
        if (variant != nullptr && variant_capacity > 0) {
            snprintf(variant, variant_capacity, "layer_norm_backward_few(lanes=%d,chunks=%d,threads=1024,grid=%u+%u%s)", shape.lanes, shape.chunks, columnBlocks,
                     rowBlocks, codes ? ",checkpoint" : "");
        }
        if (!launch) return load(reinterpret_cast<const void*>(few));
        hipLaunchKernelGGL(few, dim3(columnBlocks + rowBlocks), dim3(1024), 0, (hipStream_t)stream, a, columnBlocks);
        THORHIP_TRY(hipGetLastError());
        return 0;
    }
    const Shape shape = backwardShapeOf(c.columns, vec, codes);
    const bool whole = isWhole(shape, c.columns, vec), full = isFull(shape, c.columns, vec);
    const Backward kernel = c.dtype == THORHIP_FP32   ? backwardOf<float>(shape, codes, whole, full)
                            : c.dtype == THORHIP_FP16 ? backwardOf<f16>(shape, codes, whole, full)
                                                      : backwardOf<bf16>(shape, codes, whole, full);
    const uint32_t threads = shape.lanes == 0 ? 1024 : shape.lanes % 3 == 0 ? 768 : std::max(512, shape.lanes), teams = shape.lanes == 0 ? 1 : threads / shape.lanes;  // kBackwardThreads
    uint32_t grid = std::min(c.rows, 2 * units), shares = 0;
    Backward columnsKernel = nullptr;
    dim3 columnsGrid(1, 1);
    if (shape.lanes != 0) {
        // One block of eight wavefronts or more per CU stays, two where a lane has 16 bytes of 16-bit elements and registers to spare: more
        // blocks have more shares to write and to add (bf16 16384 x 4096: 71.4 us with 256 blocks, 74.4 with 512; 65536 x 512: 44.4, 37.3).
        grid = std::min(ceilDiv(c.rows, teams), units * (shape.chunks * vec < 16 ? 2 : 1));
        if (parameters) a.sharesOfBlock = ceilDiv(ceilDiv(c.rows, teams * grid), kRowsOfShare);
        shares = parameters ? grid * a.sharesOfBlock : 0;
    } else if (parameters) {
        columnsKernel = c.dtype == THORHIP_FP32 ? columnsOf<float>(codes) : c.dtype == THORHIP_FP16 ? columnsOf<f16>(codes) : columnsOf<bf16>(codes);
        columnsGrid.x = columnBlocksOf(shape);
        constexpr uint32_t kGroups = 256 / columnLanes(kManyChunks);  // of rows at a time
        columnsGrid.y = std::min(ceilDiv(c.rows, kGroups), std::max(1u, 8 * units / columnsGrid.x));
        columnsGrid.y = std::min(std::max(columnsGrid.y, ceilDiv(c.rows, kGroups * kRowsOfShare)), 65535u);
        shares = columnsGrid.y > 1 ? columnsGrid.y : 0;
    }
    const size_t workspace = (size_t)shares * 2 * c.columns * sizeof(float);
    if (needed_workspace != nullptr) *needed_workspace = workspace;
    const void* finish = c.parameter_dtype == THORHIP_FP32   ? reinterpret_cast<const void*>(addShares<float>)
                         : c.parameter_dtype == THORHIP_FP16 ? reinterpret_cast<const void*>(addShares<f16>)
                                                             : reinterpret_cast<const void*>(addShares<bf16>);
    if (variant != nullptr && variant_capacity > 0) {
        snprintf(variant, variant_capacity, "layer_norm_backward(lanes=%d,chunks=%d,threads=%u,grid=%u,shares=%u%s)", shape.lanes, shape.chunks, threads, grid,
                 shares, codes ? ",checkpoint" : "");
    }
    if (!launch) {
        if (const int rc = load(reinterpret_cast<const void*>(kernel))) return rc;
        if (columnsKernel != nullptr)
            if (const int rc = load(reinterpret_cast<const void*>(columnsKernel))) return rc;
        return shares != 0 ? load(finish) : 0;
    }
    THORHIP_REQUIRE(workspace == 0 || (c.workspace != nullptr && c.workspace_bytes >= workspace), "thorhip_layer_norm_backward: %zu bytes of workspace, %zu are needed",
                    c.workspace_bytes, workspace);
    a.partials = shares != 0 ? c.workspace : nullptr;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, (hipStream_t)stream, a);
    THORHIP_TRY(hipGetLastError());
    if (columnsKernel != nullptr) {
        hipLaunchKernelGGL(columnsKernel, columnsGrid, dim3(256), 0, (hipStream_t)stream, a);
        THORHIP_TRY(hipGetLastError());
    }
    if (shares != 0) {
        const dim3 finishGrid(ceilDiv(c.columns, 32), 2);
        const float* partials = c.workspace;
        u32 count = shares, columns = c.columns;
        void* weightGradient = c.weight_gradient;
        void* biasGradient = c.bias_gradient;
        void* args[] = {&partials, &count, &columns, &weightGradient, &biasGradient};
        THORHIP_TRY(hipLaunchKernel(finish, finishGrid, dim3(1024), args, 0, (hipStream_t)stream));
    }
    return 0;
}

}  // extern "C"
