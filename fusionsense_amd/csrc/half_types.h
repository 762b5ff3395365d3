// The three element types of the semantic-head operators (fp32 / bf16 / fp16) and their matrix instructions.
#pragma once
#include <type_traits>

#include "common.h"

namespace fsgs {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// A chunk is 16 bytes of a row: what a lane loads, stores and feeds to the matrix pipe at a time.
struct alignas(16) Chunk {
    uint32_t u[4];
};

template <typename T>
constexpr int kChunk = 16 / (int)sizeof(T);

// `p` is aligned to its element only (rows of odd length start anywhere): gfx950 takes vector accesses at any byte address,
// so the compiler keeps these as one access.
template <typename T>
__device__ __forceinline__ Chunk load_chunk(const T *p) {
    Chunk c;
    __builtin_memcpy(&c, p, sizeof(Chunk));
    return c;
}

// The first `n` elements (n <= 0: none), the others zero; nothing behind the n-th is touched.
template <typename T>
__device__ __forceinline__ Chunk load_chunk_n(const T *p, int n) {
    if (n >= kChunk<T>) return load_chunk(p);
    T v[kChunk<T>];
#pragma unroll
    for (int i = 0; i < kChunk<T>; ++i) v[i] = i < n ? p[i] : (T)0.f;
    Chunk c;
    __builtin_memcpy(&c, v, sizeof(Chunk));
    return c;
}

// Rows of a matrix read in chunks that need not end with the row: raw() reads 16 bytes wherever they start (held back only at
// the matrix' last element, so nothing outside it is read; a matrix of less than 16 bytes is read from its start) and has no
// branch, so it can be under way long before it is used; fix() then moves what was held back to its place and zeroes what lies behind `valid` elements.
template <typename T>
struct RowReader {
    const T *p;
    int64_t pitch, lim;  // lim: the last element a chunk may start at
    __device__ RowReader(const void *base, int64_t rows, int64_t pitch_, int width)
        : p((const T *)base), pitch(pitch_), lim(max((rows - 1) * pitch_ + width - kChunk<T>, (int64_t)0)) {}
    __device__ __forceinline__ Chunk raw(int64_t at) const { return load_chunk(p + min(at, lim)); }
    // A chunk known to lie inside: `from` (the same for the whole wave) plus a byte offset, no address arithmetic per lane.
    __device__ __forceinline__ Chunk inside(int64_t from, uint32_t offset) const {
        Chunk c;
        __builtin_memcpy(&c, (const char *)(p + from) + offset, sizeof(Chunk));
        return c;
    }
    // may_end: some lane's chunk may reach the matrix' end (the same for the whole wave)
    __device__ __forceinline__ void fix(Chunk &c, int64_t at, int valid, bool may_end) const {
        constexpr int CE = kChunk<T>;
        if (may_end) {
            const int s = at > lim ? (int)min(at - lim, (int64_t)(CE - 1)) : 0;
            if (s & (CE / 2)) c.u[0] = c.u[2], c.u[1] = c.u[3], c.u[2] = c.u[3] = 0;
            if (s & (CE / 4)) c.u[0] = c.u[1], c.u[1] = c.u[2], c.u[2] = c.u[3], c.u[3] = 0;
            if (sizeof(T) == 2 && (s & 1)) {
                c.u[0] = c.u[0] >> 16 | c.u[1] << 16, c.u[1] = c.u[1] >> 16 | c.u[2] << 16;
                c.u[2] = c.u[2] >> 16 | c.u[3] << 16, c.u[3] >>= 16;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int left = valid - i * (CE / 4);
            if constexpr (sizeof(T) == 2) c.u[i] = left >= 2 ? c.u[i] : left == 1 ? c.u[i] & 0xffffu : 0;
            else c.u[i] = left >= 1 ? c.u[i] : 0;
        }
    }
};
// kChunk floats rounded (to nearest, ties to even) to a chunk: two per instruction in the half-width types.
template <typename T>
__device__ __forceinline__ Chunk pack_chunk(const float *v) {
    Chunk c;
    if constexpr (sizeof(T) == 4) {
        __builtin_memcpy(&c, v, sizeof(Chunk));
    } else {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        typedef T tx2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x2 p = {v[2 * i], v[2 * i + 1]};
            c.u[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, tx2));
        }
    }
    return c;
}

template <typename T>
__device__ __forceinline__ void unpack_chunk(const Chunk &c, float *v) {
    T t[kChunk<T>];
    __builtin_memcpy(t, &c, sizeof(Chunk));
#pragma unroll
    for (int e = 0; e < kChunk<T>; ++e) v[e] = (float)t[e];
}

// kChunk floats as the sum of two chunks of a half-width type: hi the rounded values, lo what that left, rounded.  Together 16 bits
// of a value (bf16) or 22 (fp16, down to the absolute 2^-25 that half of its least number is).  Values of up to twice fp16's
// largest number are held too; infinities lie in hi alone.
template <typename T>
__device__ __forceinline__ Chunk split_chunk(const float *v, Chunk &lo) {
    static_assert(sizeof(T) == 2);
    constexpr float kMax = std::is_same_v<T, _Float16> ? 65504.f : 0x1.fep127f;
    float r[8], m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[e]));
    Chunk hi = pack_chunk<T>(v);
    unpack_chunk<T>(hi, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = v[e] - r[e];
    if (__any(m > kMax)) {
        float h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool finite = fabsf(v[e]) < INFINITY;
            h[e] = finite ? __builtin_amdgcn_fmed3f(v[e], -kMax, kMax) : v[e];
            r[e] = finite ? v[e] - (float)(T)h[e] : 0.f;
        }
        hi = pack_chunk<T>(h);
    }
    lo = pack_chunk<T>(r);
    return hi;
}

// Past the caches: for outputs that no kernel reads while they could still be there.  16-byte aligned.
__device__ __forceinline__ void store_streaming(void *p, const Chunk &c) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, c), (u32x4 *)p);
}

// acc += A B for one 16x16 tile: lane l holds row (l & 15) of A and column (l & 15) of B; its 16 bytes cover the same part
// of the summed axis in both, so their order along that axis does not matter.  Result: column l & 15, rows 4 (l >> 4) .. + 3.
template <typename T>
__device__ __forceinline__ void mma_chunk(f32x4 &acc, const Chunk &a, const Chunk &b);
template <>
__device__ __forceinline__ void mma_chunk<__bf16>(f32x4 &acc, const Chunk &a, const Chunk &b) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
}
template <>
__device__ __forceinline__ void mma_chunk<_Float16>(f32x4 &acc, const Chunk &a, const Chunk &b) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
}
template <>
__device__ __forceinline__ void mma_chunk<float>(f32x4 &acc, const Chunk &a, const Chunk &b) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, a.u[i]), __builtin_bit_cast(float, b.u[i]), acc,
                                                   0, 0, 0);
}

// The operand of mma_chunk whose 16 rows are columns of a matrix that lies row by row in LDS (`pitch` bytes apart).
// Half width: gfx950's transposing LDS read (16 lanes read 4 rows x 16 columns, lane i leaves with column i); the lanes of
// group lg get the rows lo .. lo + 3 and hi .. hi + 3, columns by `col` (lane j of a group points at 4 neighbouring ones of row
// j / 4).  fp32: plain reads, rows lo .. lo + 3.
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
template <typename T>
__device__ __forceinline__ Chunk load_columns(const char *lds, int pitch, int lo, int hi, int col) {
    Chunk c;
    if constexpr (sizeof(T) == 2) {
        const int j = threadIdx.x & 15;
        const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(lds + (lo + (j >> 2)) * pitch + col * 2));
        const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)(lds + (hi + (j >> 2)) * pitch + col * 2));
        __builtin_memcpy(c.u, &a, 8);
        __builtin_memcpy(c.u + 2, &b, 8);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) c.u[e] = *(const uint32_t *)(lds + (lo + e) * pitch + col * 4);
    }
    return c;
}

// A workgroup barrier for LDS alone: __syncthreads also waits for every global load under way, which is what a kernel that
// reads ahead must not do.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

inline bool known_dtype(int d) { return d == FSGS_F32 || d == FSGS_BF16 || d == FSGS_F16; }

}  // namespace fsgs
