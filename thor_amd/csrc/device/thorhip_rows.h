// What the row kernels (layer norm, 8-bit checkpoints, checkpointed activations) share: 16-byte chunks of a row, folds over teams of
// lanes, the addresses of rows, and the 8-bit code of a block of 128 elements.
#pragma once

#include <hip/hip_runtime.h>

#include "thorhip.h"
#include "thorhip_internal.h"
#include "thorhip_numeric.h"

namespace thor {

// ---- rows ----------------------------------------------------------------------------------------------------------------------------

// A kernel's view of a tensor [rows, columns] with adjacent columns; strides in elements.  Row r = q * innerRows + i starts at
// q * outer + i * inner (innerRows == 0: r * inner), which covers leading axes in another order than their storage's.
struct RowsOf {
    char* data;
    i64 outer, inner;
};

template <typename T>
__device__ __forceinline__ T* rowPointer(const RowsOf& t, u32 row, u32 innerRows) {
    i64 offset;
    if (innerRows == 0) {
        offset = (i64)row * t.inner;
    } else {
        const u32 q = row / innerRows;
        offset = (i64)q * t.outer + (i64)(row - q * innerRows) * t.inner;
    }
    return reinterpret_cast<T*>(t.data) + offset;
}

// Rows in use of a packed ragged batch: everything before the end of the last segment.  Without offsets all of them.
struct Extent {
    const void* end;  // the last element of the offsets tensor, or null
    int is64;
    u32 rows;
};
__device__ __forceinline__ u32 rowsInUse(const Extent& e) {
    if (e.end == nullptr) return e.rows;
    const u64 n = e.is64 ? *static_cast<const u64*>(e.end) : (u64)*static_cast<const u32*>(e.end);
    return n < e.rows ? (u32)n : e.rows;
}

// Elements of a row that share a scale, and elements of a type in 16 bytes.
constexpr int kCheckpointBlock = 128;
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// What is known of a row when its kernel is compiled.  Any: nothing.  Whole: it ends with a whole chunk and has one, so there is no tail; a
// lane without a chunk of its own can work on the row's last one as that chunk's lane does (source(), works()), reading and writing the
// same bits, so that loads and stores need no branches and the compiler can count what is on its way.  The backward pass does; the forward
// pass does not, where a block of codes would get another scale by it, and has the registers of the tail from it.  Blocks: a row of whole
// blocks of codes, where the lanes of a block work on the last block as its own lanes do, so that its codes and scale come out the same
// too; the forward pass does that.  Full: every lane has all of its chunks.
enum class Fit { Any, Whole, Blocks, Full };

// How a team of LANES lanes holds a row: whole chunks of VEC elements, chunk k of lane l at column (k * LANES + l) * VEC, and the
// columns % VEC elements behind the last whole chunk as a tail, one element each in the first lanes of those that have the tail's block
// of codes.  So every access is a whole chunk or one element, and a block of codes never leaves its GROUP adjacent lanes.
template <typename T, int LANES, Fit FIT>
struct RowLayout {
    static constexpr u32 VEC = kVec<T>, GROUP = kCheckpointBlock / VEC;
    u32 lane, whole;      // columns in whole chunks
    u32 tailColumn;
    int tailChunk;        // the k of the chunks that have the tail's block; -1: no tail
    bool tail;            // this lane has an element of it

    __device__ __forceinline__ RowLayout(u32 columns, u32 lane) : lane(lane) {
        const u32 count = FIT == Fit::Any ? columns % VEC : 0, first = (columns - 1) / kCheckpointBlock * GROUP;  // of the last block's lanes
        whole = columns - count;
        const u32 at = lane - first % LANES;
        tail = FIT == Fit::Any && at < count;
        tailColumn = whole + at;
        tailChunk = count != 0 ? (int)(first / LANES) : -1;
    }
    __device__ __forceinline__ u32 column(int k) const { return ((u32)k * LANES + lane) * VEC; }
    __device__ __forceinline__ bool has(int k) const { return FIT == Fit::Full || column(k) < whole; }
    // The chunk that the lane works on, and whether it works on any.
    __device__ __forceinline__ u32 source(int k) const {
        if (FIT == Fit::Any || FIT == Fit::Full || column(k) < whole) return column(k);
        return FIT == Fit::Whole ? whole - VEC : whole - kCheckpointBlock + lane % GROUP * VEC;
    }
    __device__ __forceinline__ bool works(int k) const { return FIT != Fit::Any || column(k) < whole; }
};

// ---- chunks: 16 bytes of a row per lane ------------------------------------------------------------------------------------------------

typedef u32 Words2 __attribute__((ext_vector_type(2)));
typedef u32 Words4 __attribute__((ext_vector_type(4)));
// The same at any address that is aligned to an element: global memory takes it, at the price of one more cache line.
typedef Words4 Words4OfElements __attribute__((aligned(2)));
typedef Words4 Words4OfFloats __attribute__((aligned(4)));
typedef Words2 Words2OfElements __attribute__((aligned(2)));
typedef Words2 Words2OfBytes __attribute__((aligned(1)));
typedef u32 WordOfBytes __attribute__((aligned(1)));

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(f16 x) { return (float)__builtin_bit_cast(_Float16, x.bits); }
__device__ __forceinline__ float widen(bf16 x) { return toFloat(x); }

template <typename T>
__device__ __forceinline__ T narrow(float x);
template <>
__device__ __forceinline__ float narrow<float>(float x) { return x; }
template <>
__device__ __forceinline__ f16 narrow<f16>(float x) { return toF16(x); }
template <>
__device__ __forceinline__ bf16 narrow<bf16>(float x) { return toBf16(x); }

template <typename T>
struct Elements {
    T e[kVec<T>];
};
template <typename T>
__device__ __forceinline__ Words4 loadWords(const T* p) {
    return __builtin_nontemporal_load(reinterpret_cast<const Words4OfElements*>(p));
}
template <typename T>
__device__ __forceinline__ void unpack(const Words4& w, float (&v)[kVec<T>]) {
    const Elements<T> x = __builtin_bit_cast(Elements<T>, w);
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) v[i] = widen(x.e[i]);
}
template <typename T>
__device__ __forceinline__ void loadChunk(const T* p, float (&v)[kVec<T>]) {
    unpack<T>(loadWords(p), v);
}
template <typename T>
__device__ __forceinline__ void storeChunk(T* p, const float (&v)[kVec<T>]) {
    Elements<T> x;
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) x.e[i] = narrow<T>(v[i]);
    __builtin_nontemporal_store(__builtin_bit_cast(Words4, x), reinterpret_cast<Words4OfElements*>(p));
}
// VEC elements that many rows share (weights), through the caches.
template <int VEC, typename W>
__device__ __forceinline__ void loadShared(const W* p, float (&v)[VEC]) {
    constexpr int kPart = 16 / (int)sizeof(W) < VEC ? 16 / (int)sizeof(W) : VEC;
    struct Part {
        W e[kPart];
    };
#pragma unroll
    for (int j = 0; j < VEC; j += kPart) {
        Part x;
        if constexpr (sizeof(Part) == 16) {
            x = __builtin_bit_cast(Part, *reinterpret_cast<const Words4OfElements*>(p + j));
        } else {
            static_assert(sizeof(Part) == 8, "chunks of 8 or 16 bytes");
            x = __builtin_bit_cast(Part, *reinterpret_cast<const Words2OfElements*>(p + j));
        }
#pragma unroll
        for (int i = 0; i < kPart; ++i) v[j + i] = widen(x.e[i]);
    }
}
// fp32 results that another kernel reads.
template <int VEC>
__device__ __forceinline__ void storeFloats(float* p, const float (&v)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; j += 4) {
        const Elements<float> x = {{v[j], v[j + 1], v[j + 2], v[j + 3]}};
        *reinterpret_cast<Words4OfFloats*>(p + j) = __builtin_bit_cast(Words4, x);
    }
}

// ---- folds over 16, 32 or 64 adjacent lanes, the result in each of them ------------------------------------------------------------------

template <int CTRL>
__device__ __forceinline__ u32 rotated(u32 x) {
    return (u32)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
}
struct AddF {
    __device__ __forceinline__ u32 operator()(u32 a, u32 b) const { return f32Bits(bitsF32(a) + bitsF32(b)); }
};
struct MaxU {
    __device__ __forceinline__ u32 operator()(u32 a, u32 b) const { return a > b ? a : b; }
};
// Four rotations within a row of 16 lanes, then exchanges of whole rows.  All lanes of the team take part.
template <int LANES, typename Op>
__device__ __forceinline__ u32 foldLanes(u32 x, Op op) {
    static_assert(LANES == 16 || LANES == 32 || LANES == 64, "teams of 16, 32 or 64 lanes");
    x = op(x, rotated<0x128>(x));  // row_ror:8
    x = op(x, rotated<0x124>(x));
    x = op(x, rotated<0x122>(x));
    x = op(x, rotated<0x121>(x));
    if constexpr (LANES >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        x = op(s[0], s[1]);
    }
    if constexpr (LANES >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        x = op(s[0], s[1]);
    }
    return x;
}
template <int LANES>
__device__ __forceinline__ float sumLanes(float x) { return bitsF32(foldLanes<LANES>(f32Bits(x), AddF())); }

// Sums of N values over a team of LANES lanes.  Teams of more than one wavefront meet in `shared` (N floats per wavefront of the block),
// at a barrier of the whole block; `shared` may be used again after one more barrier, which callers get by taking turns between two arrays.
template <int LANES, int N>
__device__ __forceinline__ void sumTeam(float (&v)[N], float (*shared)[N]) {
    constexpr int kWave = LANES < 64 ? LANES : 64;
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = sumLanes<kWave>(v[n]);
    if constexpr (LANES > 64) {
        constexpr int kWaves = LANES / 64;
        if (threadIdx.x % 64 == 0) {
#pragma unroll
            for (int n = 0; n < N; ++n) shared[threadIdx.x / 64][n] = v[n];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) s += shared[threadIdx.x / LANES * kWaves + w][n];
            v[n] = s;
        }
    }
}

// ---- 8-bit codes of a block ----------------------------------------------------------------------------------------------------------------

// scale: what a code is multiplied with; times: what a value is multiplied with before it is rounded to a code.
struct BlockScale {
    float scale, times;
};

// From the largest magnitude bits of a block.  Two formats are floating point: their scale is the smallest power of two (2^-126 at
// least) that brings the magnitude within the largest code, which is 1.75 * 2^8 or 1.75 * 2^15, so that the products are exact and a
// code is one rounding of its value.  int8 divides the largest magnitude by 127.  A block with a NaN or an infinity has a NaN for its
// scale: what is restored from it is NaN throughout.
__device__ __forceinline__ BlockScale scaleOfBlock(u32 magnitude, int format) {
    BlockScale s;
    if (magnitude >= 0x7f800000u) {
        s.scale = bitsF32(0x7fc00000u);
        s.times = 0.0f;
    } else if (format == THORHIP_INT8) {
        const float m = __builtin_fmaxf(bitsF32(magnitude), 0x1p-100f);
        s.scale = m / 127.0f;
        s.times = 127.0f / m;
    } else {
        int e = (int)((magnitude + 0x1fffffu) >> 23) - (format == THORHIP_FP8_E4M3 ? 8 : 15);
        e = e < 1 ? 1 : e;
        s.scale = bitsF32((u32)e << 23);
        s.times = bitsF32((u32)(254 - e) << 23);
    }
    return s;
}

// Four values, already multiplied, to four codes.  The hardware's conversions round to nearest even; nothing here is out of range.
__device__ __forceinline__ u32 encode4(float a, float b, float c, float d, int format) {
    if (format == THORHIP_FP8_E4M3) {
        return (u32)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
    }
    if (format == THORHIP_FP8_E5M2) {
        return (u32)__builtin_amdgcn_cvt_pk_bf8_f32(c, d, __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false), true);
    }
    const u32 x = (u32)(int)__builtin_rintf(a) & 0xffu, y = (u32)(int)__builtin_rintf(b) & 0xffu;
    const u32 z = (u32)(int)__builtin_rintf(c) & 0xffu, w = (u32)(int)__builtin_rintf(d);
    return x | (y << 8) | (z << 16) | (w << 24);
}
__device__ __forceinline__ void decode4(u32 codes, int format, float* v) {
    if (format == THORHIP_FP8_E4M3) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
        v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
    } else if (format == THORHIP_FP8_E5M2) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_bf8((int)codes, false), hi = __builtin_amdgcn_cvt_pk_f32_bf8((int)codes, true);
        v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (float)((int)(codes << (24 - 8 * i)) >> 24);
    }
}

// Codes of VEC (4 or 8) elements of a row, at any address.
template <int VEC>
struct Codes {
    u32 w[VEC / 4];
};
template <int VEC>
__device__ __forceinline__ Codes<VEC> loadCodes(const u8* p) {
    Codes<VEC> c;
    if constexpr (VEC == 8) {
        const Words2 w = __builtin_nontemporal_load(reinterpret_cast<const Words2OfBytes*>(p));
        c.w[0] = w[0], c.w[1] = w[1];
    } else {
        c.w[0] = __builtin_nontemporal_load(reinterpret_cast<const WordOfBytes*>(p));
    }
    return c;
}
template <int VEC>
__device__ __forceinline__ void storeCodes(u8* p, const Codes<VEC>& c) {
    if constexpr (VEC == 8) {
        Words2 w;
        w[0] = c.w[0], w[1] = c.w[1];
        __builtin_nontemporal_store(w, reinterpret_cast<Words2OfBytes*>(p));
    } else {
        __builtin_nontemporal_store(c.w[0], reinterpret_cast<WordOfBytes*>(p));
    }
}
template <int VEC>
__device__ __forceinline__ void decode(const Codes<VEC>& c, int format, float scale, float (&v)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC / 4; ++j) decode4(c.w[j], format, v + 4 * j);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] *= scale;
}
// One code, of a tail.
__device__ __forceinline__ float decodeOne(u32 code, int format, float scale) {
    float v[4];
    decode4(code, format, v);
    return v[0] * scale;
}
__device__ __forceinline__ u8 encodeOne(float x, const BlockScale& s, int format) {
    return s.times == 0.0f ? 0 : (u8)encode4(x * s.times, 0.0f, 0.0f, 0.0f, format);
}

// The scale of a block that lies in kCheckpointBlock / VEC adjacent lanes: VEC elements in those that have a chunk of it, one more in
// those that have an element of the tail.  Every lane of the block takes part.
template <int VEC>
__device__ __forceinline__ BlockScale scaleOfLanes(const float (&v)[VEC], bool has, float tail, bool hasTail, int format) {
    u32 magnitude = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) magnitude = MaxU()(magnitude, f32Bits(v[i]) & 0x7fffffffu);
    magnitude = has ? magnitude : 0;
    magnitude = MaxU()(magnitude, hasTail ? f32Bits(tail) & 0x7fffffffu : 0);
    return scaleOfBlock(foldLanes<kCheckpointBlock / VEC>(magnitude, MaxU()), format);
}
template <int VEC>
__device__ __forceinline__ Codes<VEC> encodeChunk(const float (&v)[VEC], const BlockScale& s, int format) {
    Codes<VEC> c;
#pragma unroll
    for (int j = 0; j < VEC / 4; ++j) {
        c.w[j] = encode4(v[4 * j] * s.times, v[4 * j + 1] * s.times, v[4 * j + 2] * s.times, v[4 * j + 3] * s.times, format);
    }
    if (s.times == 0.0f) {  // infinity * 0 is no zero
#pragma unroll
        for (int j = 0; j < VEC / 4; ++j) c.w[j] = 0;
    }
    return c;
}

}  // namespace thor
