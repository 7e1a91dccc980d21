// 8-bit checkpoints of activations, and the activations that keep their input as one.
//
// A block of 128 elements of a row lies in 16 adjacent lanes (32 for fp32), 16 bytes of it each: one load, a fold of the largest
// magnitude within a row of lanes, one rounding per element, one store of 8 or 4 bytes.  Nothing is read twice and no element depends
// on another block, so every kernel here is a stream: what bounds it is the bytes it moves; a copy of
// large tensors by the library runs at 5.4 TB/s on this card.  Only gelu has the vector units work as long as the memory.
#include "thorhip_rows.h"

#include <algorithm>

namespace {

using namespace thor;

constexpr int kThreads = 256;

// Groups of kThreads lanes' blocks that a block of threads loads before it works on the first.  Two in flight are faster where there is
// nothing but a checkpoint to save or to restore (bf16 16384 x 4096: 37.1 -> 36.0 us and 36.0 -> 34.2), and slower where fp32 is restored,
// 4 bytes of codes for 16 bytes of it (8192 x 8192: 60.8 -> 63.6 us), and with an activation, which has more streams (gelu backward bf16
// 16384 x 8192: 102.8 -> 105.4 us, swish forward 104.5 -> 106.0, gated swish 8192 x 8192 forward 85.0 -> 91.4).
template <typename T, int KIND, bool BACKWARD>
constexpr int kTurns = KIND != THORHIP_IDENTITY || (BACKWARD && sizeof(T) == 4) ? 1 : 2;

struct CheckpointedArgs {
    RowsOf first, second, third;  // forward: input, multiplier, output; backward: error, multiplier gradient, input gradient
    u8* codes;
    float* scales;
    u8* multiplierCodes;
    float* multiplierScales;
    Extent extent;
    i64 columns;       // of a row as the kernel walks it: dense rows of whole blocks are walked as one row
    u32 innerRows;
    u32 blocksPerRow;  // of a row as the kernel walks it
    u32 blocksPerUse;  // of a row as the extent counts it
    u32 blocks, firstBlock;  // the launch's first
    int format;
};

// Consecutive workgroups are dealt to the eight XCDs in turn.  With this numbering each XCD walks runs of 16 adjacent blocks of threads
// (a bijection where the grid is a multiple of 128, else nothing changes): 2 to 4 % more bandwidth on every large case.
__device__ __forceinline__ u32 numberOfBlock() {
    constexpr u32 kXcds = 8, kRun = 16;
    if (gridDim.x % (kXcds * kRun) != 0) return blockIdx.x;
    const u32 within = blockIdx.x % (kXcds * kRun);
    return blockIdx.x - within + within % kXcds * kRun + within / kXcds;
}

// The VEC elements of a lane, or, in the block that a row ends in, one element of the columns % VEC behind its last whole chunk.
struct Place {
    bool there;
    bool first;       // lane of its block
    bool has, tail;   // a whole chunk, an element of the tail
    u32 block, row;
    i64 column, tailColumn;
};
template <int VEC>
__device__ __forceinline__ Place placeOf(const CheckpointedArgs& a, u32 number) {
    constexpr u32 kLanes = kCheckpointBlock / VEC;
    const u32 lane = threadIdx.x % kLanes;
    Place p;
    p.block = a.firstBlock + number * (kThreads / kLanes) + threadIdx.x / kLanes;
    const u64 used = a.extent.end == nullptr ? a.blocks : (u64)rowsInUse(a.extent) * a.blocksPerUse;
    p.there = p.block < a.blocks && p.block < used;
    p.row = a.blocksPerRow == a.blocks ? 0 : p.block / a.blocksPerRow;
    const u32 inRow = p.block - p.row * a.blocksPerRow;
    p.column = (i64)inRow * kCheckpointBlock + lane * VEC;
    p.first = lane == 0;
    const u32 count = (u32)(a.columns % VEC);
    p.has = p.column + VEC <= a.columns;
    p.tailColumn = a.columns - count + lane;
    p.tail = lane < count && inRow + 1 == a.blocksPerRow;
    return p;
}

// Phi(-a) = H(a) exp(-a^2 / 2) for a >= 0.  H falls slowly from 1/2 like 0.4 / a, so a polynomial in t = 1 / (1 + 0.3 a) follows it:
// t P(t) with the P that is nearest in relative terms on [0, 14.5] (beyond, 16-bit results are zero).  It shares the exponential with the
// density, where the library's erfc has one of its own and a division.
//
// fp32: degree 9 (off by 3.5e-9), t from the sum 1 + 0.3 a as it is before its rounding.
// 16 bits: degree 7 (off by 1.7e-7) at the hardware's reciprocal, some eight units of 2^-24, and H / 2^11 for bellTimes2To11().
template <typename T>
__device__ __forceinline__ float tailFactor(float a) {
    const float d = __builtin_fmaf(a, 0.3f, 1.0f);
    float t = __builtin_amdgcn_rcpf(d);
    if constexpr (sizeof(T) == 4) {
        const float lost = __builtin_fmaf(a, 0.3f, 1.0f - d);
        t = __builtin_fmaf(t, __builtin_fmaf(-lost, t, __builtin_fmaf(-d, t, 1.0f)), t);
        float p = -0.020624879747629166f;
        p = __builtin_fmaf(p, t, 0.11244352906942368f);
        p = __builtin_fmaf(p, t, -0.22823289036750793f);
        p = __builtin_fmaf(p, t, 0.19181127846240997f);
        p = __builtin_fmaf(p, t, -0.07944672554731369f);
        p = __builtin_fmaf(p, t, 0.09616988152265549f);
        p = __builtin_fmaf(p, t, 0.07838491350412369f);
        p = __builtin_fmaf(p, t, 0.11023649573326111f);
        p = __builtin_fmaf(p, t, 0.11957168579101562f);
        p = __builtin_fmaf(p, t, 0.11968670040369034f);
        return p * t;
    }
    constexpr float k = 0x1p-11f;
    float p = 0.03542373867332211f * k;
    p = __builtin_fmaf(p, t, -0.1561584693838267f * k);
    p = __builtin_fmaf(p, t, 0.20455683389817478f * k);
    p = __builtin_fmaf(p, t, -0.05203407264399261f * k);
    p = __builtin_fmaf(p, t, 0.12769180626590437f * k);
    p = __builtin_fmaf(p, t, 0.10017593626445624f * k);
    p = __builtin_fmaf(p, t, 0.1207121381245411f * k);
    p = __builtin_fmaf(p, t, 0.1196320071032971f * k);
    return p * t;
}

// Results of 16 bits: 2^11 exp(-x^2 / 2) and 2^15 sigmoid(x), through the hardware's power of two and reciprocal.  Those know no numbers
// below 2^-126, which a bf16 result can be made of: the factors bring everything that the types can hold into their range.  The exponents
// are rounded to fp32, which costs x^2 or |x| units of 2^-24 in the tails, 1.2e-5 at most, and up to 3.4e-7 near zero, where larger
// factors would cost more; a result rounds by 2^-9 or 2^-12.
__device__ __forceinline__ float bellTimes2To11(float x) { return __builtin_amdgcn_exp2f(__builtin_fmaf(x * x, -0.72134752044448170f, 11.0f)); }
__device__ __forceinline__ float sigmoidTimes2To15(float x) {
    return __builtin_amdgcn_rcpf(0x1p-15f + __builtin_amdgcn_exp2f(__builtin_fmaf(x, -1.4426950408889634f, -15.0f)));
}

// Results of fp32: a power of two as factor * 2^exponent, of an argument hi + lo with |lo| far below one, so that its rounding does not
// grow with it and no result is below the numbers that the hardware's power knows.
struct Power {
    float factor;
    int exponent;
    __device__ __forceinline__ float times(float x) const { return __builtin_ldexpf(x, exponent); }  // 2^exponent x
    __device__ __forceinline__ float value() const { return times(factor); }
};
__device__ __forceinline__ Power powerOfTwo(float hi, float lo) {
#pragma clang fp contract(off)  // a fused hi - whole would bring what lo holds a second time
    const float whole = __builtin_rintf(hi);
    return {__builtin_amdgcn_exp2f(hi - whole + lo), (int)whole};
}
// exp(-a) for a in [0, 200], exp(-a^2 / 2) for a in [0, 100]: log2(e) in two parts, and what the products lose.
__device__ __forceinline__ Power exponential(float a) {
#pragma clang fp contract(off)
    const float hi = a * -1.44269502f;
    return powerOfTwo(hi, __builtin_fmaf(a, -1.92596303e-8f, __builtin_fmaf(a, -1.44269502f, -hi)));
}
__device__ __forceinline__ Power exactBell(float a) {
#pragma clang fp contract(off)
    const float square = a * a, hi = square * -0.721347511f;
    float lo = __builtin_fmaf(square, -0.721347511f, -hi);
    lo = __builtin_fmaf(square, -9.62981517e-9f, lo);
    return powerOfTwo(hi, __builtin_fmaf(__builtin_fmaf(a, a, -square), -0.721347511f, lo));
}

// What the activations are made of at one x, in fp32 to some six units of 2^-24 (nine at most) down to the least number, in fewer
// instructions for 16-bit results: f(x) of a finite x, f(x) of any x, and f'(x).
template <typename T, int KIND>
struct Activated;

template <typename T>
struct Activated<T, THORHIP_RELU> {
    float x;
    __device__ __forceinline__ explicit Activated(float x) : x(x) {}
    __device__ __forceinline__ float finite() const { return any(); }
    __device__ __forceinline__ float any() const { return x < 0.0f ? 0.0f : x; }  // a NaN stays one
    __device__ __forceinline__ float slope() const { return x > 0.0f ? 1.0f : x != x ? x : 0.0f; }
};

// 16 bits: f = x s, f' = s + f (1 - s).
template <typename T>
struct Activated<T, THORHIP_SWISH> {
    float x, s;
    __device__ __forceinline__ explicit Activated(float x) : x(x), s(sigmoidTimes2To15(x) * 0x1p-15f) {}
    __device__ __forceinline__ float finite() const { return any(); }
    __device__ __forceinline__ float any() const { return x * s; }
    __device__ __forceinline__ float slope() const { return __builtin_fmaf(any(), 1.0f - s, s); }
};
// fp32: with e = exp(-|x|) and r = 1 / (1 + e) the sigmoid is e r below zero and r above, and one less it is the other of the two.
template <>
struct Activated<float, THORHIP_SWISH> {
    float x, within, s, rest;  // within: x where the product with s, which is without its power of two, is finite
    int exponent;
    __device__ __forceinline__ explicit Activated(float x) : x(x), within(x < -200.0f ? -200.0f : x) {
        const Power e = exponential(__builtin_amdgcn_fmed3f(__builtin_fabsf(x), 0.0f, 200.0f));
        const float value = e.value(), r = __builtin_amdgcn_rcpf(1.0f + value);
        s = x < 0.0f ? e.factor * r : r;
        rest = x < 0.0f ? r : value * r;
        exponent = x < 0.0f ? e.exponent : 0;
    }
    __device__ __forceinline__ float finite() const { return __builtin_ldexpf(within * s, exponent); }
    __device__ __forceinline__ float any() const { return x * __builtin_ldexpf(s, exponent); }
    __device__ __forceinline__ float slope() const { return __builtin_ldexpf(__builtin_fmaf(within * s, rest, s), exponent); }
};

// 16 bits: f = max(x, 0) - |x| Phi(-|x|), two instructions less than by cases (bf16 16384 x 8192 forward 126 -> 121 us: the one kernel
// here that the vector units bound); f' = exp(-x^2 / 2) (H(|x|) - |x| / sqrt(2 pi)) below zero, and that from one above.
template <typename T>
struct Activated<T, THORHIP_GELU> {
    float x, h, e;  // h / 2^11, 2^11 e
    __device__ __forceinline__ explicit Activated(float x) : x(x), h(tailFactor<T>(__builtin_fabsf(x))), e(bellTimes2To11(x)) {}
    __device__ __forceinline__ float finite() const { return __builtin_fmaf(-__builtin_fabsf(x), h * e, __builtin_fmaxf(x, 0.0f)); }
    __device__ __forceinline__ float any() const { return x * phi(); }
    __device__ __forceinline__ float phi() const { return x < 0.0f ? h * e : 1.0f - h * e; }
    __device__ __forceinline__ float slope() const {
        const float below = e * __builtin_fmaf(__builtin_fabsf(x), -0.39894228040143268f * 0x1p-11f, h);
        return x < 0.0f ? below : 1.0f - below;
    }
};
template <>
struct Activated<float, THORHIP_GELU> {
    float x, h;
    Power e;
    __device__ __forceinline__ explicit Activated(float x) : x(x) {
        const float a = __builtin_amdgcn_fmed3f(__builtin_fabsf(x), 0.0f, 100.0f);
        h = tailFactor<float>(a);
        e = exactBell(a);
    }
    __device__ __forceinline__ float finite() const {
        return __builtin_fmaxf(x, 0.0f) + e.times(-__builtin_fabsf(x) * (h * e.factor));
    }
    __device__ __forceinline__ float any() const { return x * phi(); }
    __device__ __forceinline__ float phi() const {
        const float below = e.times(h * e.factor);
        return x < 0.0f ? below : 1.0f - below;
    }
    __device__ __forceinline__ float slope() const {
        const float below = e.times(e.factor * __builtin_fmaf(__builtin_fabsf(x), -0.39894228040143268f, h));
        return x < 0.0f ? below : 1.0f - below;
    }
};

// One operand of the forward pass: its elements, and their codes.
template <typename T>
struct Kept {
    float v[kVec<T>] = {}, tail = 0.0f;
    __device__ __forceinline__ void load(const RowsOf& rows, const CheckpointedArgs& a, const Place& p) {
        const T* in = rowPointer<const T>(rows, p.row, a.innerRows);
        if (p.has) loadChunk(in + p.column, v);
        if (p.tail) tail = widen(in[p.tailColumn]);
    }
    __device__ __forceinline__ BlockScale keep(u8* codes, float* scales, const CheckpointedArgs& a, const Place& p) const {
        constexpr int VEC = kVec<T>;
        const BlockScale scale = scaleOfLanes<VEC>(v, p.has, tail, p.tail, a.format);
        const i64 row = (i64)p.row * a.columns;
        if (p.has) storeCodes<VEC>(codes + row + p.column, encodeChunk<VEC>(v, scale, a.format));
        if (p.tail) codes[row + p.tailColumn] = encodeOne(tail, scale, a.format);
        if (p.first) scales[p.block] = scale.scale;
        return scale;
    }
};

// Saving bf16 16384 x 4096 as e4m3 takes 34.6 us (5.9 TB/s), gated swish bf16 8192 x 8192 85.7 us (6.3 TB/s).
template <typename T, int KIND, bool MULTIPLIED>
__global__ __launch_bounds__(kThreads) void checkpointedForward(CheckpointedArgs a) {
    constexpr int VEC = kVec<T>, TURNS = kTurns<T, KIND, false>;
    Place p[TURNS];
    Kept<T> x[TURNS], z[TURNS];
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
        p[u] = placeOf<VEC>(a, numberOfBlock() * TURNS + u);
        if (!p[u].there) continue;
        x[u].load(a.first, a, p[u]);
        if constexpr (MULTIPLIED) z[u].load(a.second, a, p[u]);
    }
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
        if (!p[u].there) return;  // the same for all lanes of a block
        const BlockScale scale = x[u].keep(a.codes, a.scales, a, p[u]);
        if constexpr (MULTIPLIED) z[u].keep(a.multiplierCodes, a.multiplierScales, a, p[u]);
        if constexpr (KIND != THORHIP_IDENTITY) {
            T* out = rowPointer<T>(a.third, p[u].row, a.innerRows);
            if (p[u].has) {
                if (scale.times != 0.0f) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) x[u].v[i] = Activated<T, KIND>(x[u].v[i]).finite();
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) x[u].v[i] = Activated<T, KIND>(x[u].v[i]).any();
                }
                if constexpr (MULTIPLIED) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) x[u].v[i] *= z[u].v[i];
                }
                storeChunk(out + p[u].column, x[u].v);
            }
            if (p[u].tail) {
                const Activated<T, KIND> f(x[u].tail);
                out[p[u].tailColumn] = narrow<T>((scale.times != 0.0f ? f.finite() : f.any()) * (MULTIPLIED ? z[u].tail : 1.0f));
            }
        }
    }
}

// The largest finite value of a type: a code can stand for a little more than the largest magnitude of its block, and a finite value is
// not brought back as an infinity.
template <typename T>
constexpr float kLargest = 3.40282347e38f;
template <>
constexpr float kLargest<f16> = 65504.0f;
template <>
constexpr float kLargest<bf16> = 3.38953139e38f;

template <typename T>
__device__ __forceinline__ float finite(float x) {
    return x == x ? __builtin_fminf(__builtin_fmaxf(x, -kLargest<T>), kLargest<T>) : x;
}

// gelu's slope, and Phi where there is a multiplier, at every value that a code of the two floating point formats can stand for.  Their
// scales are powers of two, so such a value has a sign, an exponent and at most three bits more; the slope and Phi are 1/2 to the last
// bit below 2^-26, and 0 or 1 to the last bit from 15 on.  That leaves 480 values, which a block of threads works out into shared memory
// while its loads are on their way.  Without the table the kernel is bound by its vector instructions, some 28 slots per element in 16
// bits and 45 in fp32 with the exponential and the reciprocal at a quarter of the rate: bf16 16384 x 8192 124.4 us, with it 103.0; with a
// multiplier 8192 x 8192 90.3 and 84.8; fp32 8192 x 8192 103.5 and 96.4.  fp32 with a multiplier takes 159 either way and goes without,
// as fp32's Phi has lost bits where x Phi has not; so do int8 codes, whose scales are any number.
template <typename T, bool PAIRS>
struct GeluTable {
    static constexpr u32 kFirst = (127 - 26) << 3, kLast = (127 + 3) << 3 | 7, kEntries = 2 * (kLast - kFirst + 1);
    static constexpr u32 kWidth = PAIRS ? 2 : 1, kFloats = kEntries * kWidth;
    __device__ static __forceinline__ void fill(float* table) {
        for (u32 i = threadIdx.x; i < kEntries; i += kThreads) {
            const float a = bitsF32((kFirst + i / 2) << 20);
            const Activated<T, THORHIP_GELU> f(i % 2 != 0 ? -a : a);
            table[i * kWidth] = f.slope();
            if constexpr (PAIRS) table[i * kWidth + 1] = f.phi();
        }
    }
    __device__ static __forceinline__ const float* at(const float* table, float x) {
        const u32 bits = f32Bits(x), entry = bits >> 20 & 0x7ff;
        const u32 within = entry < kFirst ? kFirst : entry > kLast ? kLast : entry;
        return table + ((within << 1 | bits >> 31) - 2 * kFirst) * kWidth;
    }
};

// One element of the backward pass.
template <typename T, int KIND, bool MULTIPLIED>
__device__ __forceinline__ void backward(float dy, float& x, float& z) {
    if constexpr (KIND == THORHIP_IDENTITY) {
        x = finite<T>(x);
    } else {
        const Activated<T, KIND> f(x);
        x = MULTIPLIED ? dy * (z * f.slope()) : dy * f.slope();  // a slope of zero before error times multiplier can overflow
        z = dy * f.finite();
    }
}
template <typename T, bool MULTIPLIED>
__device__ __forceinline__ void backwardOfTable(const float* table, float dy, float& x, float& z) {
    const float* entry = GeluTable<T, MULTIPLIED>::at(table, x);
    if constexpr (MULTIPLIED) {
        const float f = x * entry[1];
        x = dy * (z * entry[0]);
        z = dy * f;
    } else {
        x = dy * entry[0];
    }
}

// Whether a chunk is of finite values; its infinities (of e5m2's codes, or of a product near fp32's largest) are made finite where not:
// no formula above makes a slope of them.
template <int VEC>
__device__ __forceinline__ bool keepFinite(float (&v)[VEC]) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum += v[i];
    if (__builtin_fabsf(sum) < __builtin_inff()) return true;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = finite<float>(v[i]);
    return false;
}

// What a lane needs of a block in the backward pass, as it was loaded.
template <typename T, int KIND, bool MULTIPLIED>
struct Saved {
    Words4 error;
    Codes<kVec<T>> x, z;
    float xScale, zScale;
    T tailError;
    u32 xTail, zTail;
    __device__ __forceinline__ void load(const CheckpointedArgs& a, const Place& p) {
        const i64 row = (i64)p.row * a.columns;
        const T* dy = KIND == THORHIP_IDENTITY ? nullptr : rowPointer<const T>(a.first, p.row, a.innerRows);
        xScale = a.scales[p.block];
        if constexpr (MULTIPLIED) zScale = a.multiplierScales[p.block];
        if (p.has) {
            if constexpr (KIND != THORHIP_IDENTITY) error = loadWords(dy + p.column);
            x = loadCodes<kVec<T>>(a.codes + row + p.column);
            if constexpr (MULTIPLIED) z = loadCodes<kVec<T>>(a.multiplierCodes + row + p.column);
        }
        if (p.tail) {
            if constexpr (KIND != THORHIP_IDENTITY) tailError = dy[p.tailColumn];
            xTail = a.codes[row + p.tailColumn];
            if constexpr (MULTIPLIED) zTail = a.multiplierCodes[row + p.tailColumn];
        }
    }
};

// Restoring bf16 16384 x 4096 from e4m3 takes 34.0 us (6.0 TB/s), gelu's gradient bf16 16384 x 8192 102.0 us (6.6 TB/s).
template <typename T, int KIND, bool MULTIPLIED>
__global__ __launch_bounds__(kThreads) void checkpointedBackward(CheckpointedArgs a) {
    constexpr int VEC = kVec<T>, TURNS = kTurns<T, KIND, true>;
    Place p[TURNS];
    Saved<T, KIND, MULTIPLIED> saved[TURNS];
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
        p[u] = placeOf<VEC>(a, numberOfBlock() * TURNS + u);
        if (p[u].there) saved[u].load(a, p[u]);
    }
    constexpr bool kTabled = KIND == THORHIP_GELU && (sizeof(T) == 2 || !MULTIPLIED);
    __shared__ __attribute__((aligned(8))) float table[kTabled ? GeluTable<T, MULTIPLIED>::kFloats : 1];
    const bool tabled = kTabled && a.format != THORHIP_INT8;
    if (tabled) {
        GeluTable<T, MULTIPLIED>::fill(table);
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < TURNS; ++u) {
        if (!p[u].there) return;
        const Saved<T, KIND, MULTIPLIED>& s = saved[u];
        T* zOut = MULTIPLIED ? rowPointer<T>(a.second, p[u].row, a.innerRows) : nullptr;
        T* xOut = rowPointer<T>(a.third, p[u].row, a.innerRows);
        if (p[u].has) {
            float dy[VEC], x[VEC], z[VEC];
            if constexpr (KIND != THORHIP_IDENTITY) unpack<T>(s.error, dy);
            decode<VEC>(s.x, a.format, s.xScale, x);
            if constexpr (MULTIPLIED) decode<VEC>(s.z, a.format, s.zScale, z);
            bool byTable = tabled && (f32Bits(s.xScale) & 0x7fffff) == 0;  // a power of two, as it is if the checkpoint was saved here
            if constexpr (KIND != THORHIP_IDENTITY) byTable = keepFinite(x) && byTable;
            if constexpr (MULTIPLIED) keepFinite(z);
            if (byTable) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) backwardOfTable<T, MULTIPLIED>(table, dy[i], x[i], z[i]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) backward<T, KIND, MULTIPLIED>(dy[i], x[i], z[i]);
            }
            storeChunk(xOut + p[u].column, x);
            if constexpr (MULTIPLIED) storeChunk(zOut + p[u].column, z);
        }
        if (p[u].tail) {
            const float dy = KIND == THORHIP_IDENTITY ? 0.0f : widen(s.tailError);
            float x = decodeOne(s.xTail, a.format, s.xScale), z = MULTIPLIED ? finite<float>(decodeOne(s.zTail, a.format, s.zScale)) : 0.0f;
            if constexpr (KIND != THORHIP_IDENTITY) x = finite<float>(x);
            backward<T, KIND, MULTIPLIED>(dy, x, z);
            xOut[p[u].tailColumn] = narrow<T>(x);
            if constexpr (MULTIPLIED) zOut[p[u].tailColumn] = narrow<T>(z);
        }
    }
}

struct Kernel {
    void (*function)(CheckpointedArgs);
    int turns;
};

template <typename T, int KIND>
Kernel kernelOf(bool backward, bool multiplied) {
    if constexpr (KIND != THORHIP_IDENTITY) {
        if (multiplied) {
            return backward ? Kernel{checkpointedBackward<T, KIND, true>, kTurns<T, KIND, true>} : Kernel{checkpointedForward<T, KIND, true>, kTurns<T, KIND, false>};
        }
    }
    return backward ? Kernel{checkpointedBackward<T, KIND, false>, kTurns<T, KIND, true>} : Kernel{checkpointedForward<T, KIND, false>, kTurns<T, KIND, false>};
}
template <typename T>
Kernel kernelOf(int activation, bool backward, bool multiplied) {
    switch (activation) {
        case THORHIP_RELU: return kernelOf<T, THORHIP_RELU>(backward, multiplied);
        case THORHIP_GELU: return kernelOf<T, THORHIP_GELU>(backward, multiplied);
        case THORHIP_SWISH: return kernelOf<T, THORHIP_SWISH>(backward, multiplied);
        default: return kernelOf<T, THORHIP_IDENTITY>(backward, false);
    }
}

RowsOf rowsOf(const thorhip_rows& r) { return {static_cast<char*>(r.data), r.outer, r.inner}; }

int checkpointed(const thorhip_checkpointed* call, bool backward, void* stream, int launch, char* variant, size_t variant_capacity) {
    const char* who = backward ? "thorhip_checkpointed_backward" : "thorhip_checkpointed_forward";
    THORHIP_REQUIRE(call != nullptr, "%s: no call", who);
    const thorhip_checkpointed& c = *call;
    THORHIP_REQUIRE(c.dtype == THORHIP_FP32 || c.dtype == THORHIP_FP16 || c.dtype == THORHIP_BF16, "%s: dtype %d", who, c.dtype);
    THORHIP_REQUIRE(c.checkpoint_dtype == THORHIP_FP8_E4M3 || c.checkpoint_dtype == THORHIP_FP8_E5M2 || c.checkpoint_dtype == THORHIP_INT8,
                    "%s: checkpoint dtype %d", who, c.checkpoint_dtype);
    THORHIP_REQUIRE(c.activation >= THORHIP_IDENTITY && c.activation <= THORHIP_SWISH, "%s: activation %d", who, c.activation);
    THORHIP_REQUIRE(c.rows > 0 && c.columns > 0 && c.rows < (1u << 31) && c.columns < (1u << 31), "%s: %u rows of %u columns", who, c.rows, c.columns);
    const bool identity = c.activation == THORHIP_IDENTITY;
    const bool multiplied = backward ? c.multiplier_gradient.data != nullptr : c.multiplier.data != nullptr;
    THORHIP_REQUIRE(!(identity && multiplied), "%s: a multiplier without an activation", who);
    THORHIP_REQUIRE(c.codes != nullptr && c.scales != nullptr, "%s: no checkpoint", who);
    THORHIP_REQUIRE(!multiplied || (c.multiplier_codes != nullptr && c.multiplier_scales != nullptr), "%s: no checkpoint of the multiplier", who);
    CheckpointedArgs a{};
    a.first = rowsOf(backward ? c.error : c.input);
    a.second = rowsOf(backward ? c.multiplier_gradient : c.multiplier);
    a.third = rowsOf(backward ? c.input_gradient : c.output);
    THORHIP_REQUIRE(a.first.data != nullptr || (backward && identity), "%s: nothing to read", who);
    THORHIP_REQUIRE(a.third.data != nullptr || (!backward && identity), "%s: nothing to write to", who);
    a.codes = static_cast<u8*>(c.codes);
    a.scales = c.scales;
    a.multiplierCodes = static_cast<u8*>(c.multiplier_codes);
    a.multiplierScales = c.multiplier_scales;
    a.extent = {c.extent, c.extent_is_64, c.rows};
    a.format = c.checkpoint_dtype;
    a.columns = c.columns;
    a.innerRows = c.inner_rows;
    const uint64_t perRow = (c.columns + (uint64_t)kCheckpointBlock - 1) / kCheckpointBlock;
    const uint64_t blocks = perRow * c.rows;
    const uint32_t lanes = kCheckpointBlock * thorhip_dtype_size(c.dtype) / 16;
    THORHIP_REQUIRE(blocks < (1ull << 31), "%s: %llu blocks of %d elements are over 2^31", who, (unsigned long long)blocks, kCheckpointBlock);
    a.blocks = (u32)blocks;
    a.blocksPerUse = (u32)perRow;
    a.blocksPerRow = (u32)perRow;
    // dense rows of whole blocks are one row: no division per block
    const auto dense = [&](const RowsOf& r) { return r.data == nullptr || (c.inner_rows == 0 && (r.inner == (int64_t)c.columns || c.rows == 1)); };
    const bool one = c.columns % kCheckpointBlock == 0 && dense(a.first) && dense(a.second) && dense(a.third);
    if (one) {
        a.columns = (i64)c.rows * c.columns;
        a.blocksPerRow = a.blocks;
    }
    const Kernel kernel = c.dtype == THORHIP_FP32   ? kernelOf<float>(c.activation, backward, multiplied)
                          : c.dtype == THORHIP_FP16 ? kernelOf<f16>(c.activation, backward, multiplied)
                                                    : kernelOf<bf16>(c.activation, backward, multiplied);
    // a grid has fewer than 2^32 threads: tensors of over 2^33 elements take several launches
    constexpr uint32_t kMost = 1u << 26;
    const uint32_t perBlock = kThreads / lanes * kernel.turns, grid = (std::min(a.blocks, kMost) + perBlock - 1) / perBlock;
    if (variant != nullptr && variant_capacity > 0) {
        snprintf(variant, variant_capacity, "%s(grid=%u,%s)", backward ? "checkpointed_backward" : "checkpointed_forward", grid, one ? "one_row" : "rows");
    }
    if (!launch) {  // loads the kernel: a first launch under stream capture must not have to
        hipFuncAttributes attributes;
        THORHIP_TRY(hipFuncGetAttributes(&attributes, reinterpret_cast<const void*>(kernel.function)));
        return 0;
    }
    for (; a.firstBlock < a.blocks; a.firstBlock += kMost) {
        hipLaunchKernelGGL(kernel.function, dim3((std::min(a.blocks - a.firstBlock, kMost) + perBlock - 1) / perBlock), dim3(kThreads), 0, (hipStream_t)stream, a);
        THORHIP_TRY(hipGetLastError());
    }
    return 0;
}

}  // namespace

extern "C" {

int thorhip_checkpointed_forward(const thorhip_checkpointed* call, void* stream, int launch, char* variant, size_t variant_capacity) {
    return checkpointed(call, false, stream, launch, variant, variant_capacity);
}

int thorhip_checkpointed_backward(const thorhip_checkpointed* call, void* stream, int launch, char* variant, size_t variant_capacity) {
    return checkpointed(call, true, stream, launch, variant, variant_capacity);
}

}  // extern "C"
