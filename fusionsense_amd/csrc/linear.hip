// One layer of the semantic head: y = act(x W^T + b) + r and its backward pass.
//
//   forward    z = x W^T + b, y = act(z) + r                       x [M,K], W [N,K], y [M,N]
//   backward   dz = dy * act'(z) (z formed again from x: M*K values are read instead of M*N kept), dx = dz W,
//              dW = dz^T x, db = sum_m dz, dr = dy
//
// Products run on the matrix cores in the tensors' own type, sums are fp32 throughout (fp32 tensors use the fp32 matrix
// instructions: no reduced-precision product).
#include "half_types.h"

namespace fsgs {

namespace {

constexpr int kSlabBytes = 128;  // one step along the summed axis of the general tile: 64 half-width or 32 fp32 values

struct LinArgs {
    const void *x, *w, *bias, *res, *dy;
    void *y;
    int64_t rows, xp, rp, dyp, yp;
    int K, N, act;
    int stream;     // general tile: store past the caches
    float *part_b;  // dz kernels: partial column sums of dz, or null
    int lo;         // dz kernels: dz as two values, the second this many columns on; 0: one value
};

// The normal distribution's tail h = P(t) exp(-z^2 / 2) at |z|, t = 1 / (1 + c |z|), P a polynomial without a constant term
// fitted here to erfc over rounded coefficients; P and the exponential apart.  The fit is off by 1.3e-9 at most (h is a half at
// zero), a fiftieth of half an fp32 step at 1; its evaluation in fp32 adds 1.5e-7, two and a half of those.  The slopes of every type and
// fp32's forward use it.
__device__ __forceinline__ float normal_tail(float z, float &e) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.32f, fabsf(z), 1.f));
    e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
    float p = fmaf(0.04611215f, t, -0.24249351f);
    p = fmaf(p, t, 0.41171595f);
    p = fmaf(p, t, -0.16985106f);
    p = fmaf(p, t, 0.22053833f);
    p = fmaf(p, t, 0.104102224f);
    p = fmaf(p, t, 0.12987591f);
    return p * t;
}

// The tail at |z| for the half-width types' forward as one exponential: 2^Q(|z|), Q a polynomial fitted here to log2 of the tail.
// bf16: degree 9 on [0, 13.2]; relative errors below 5e-6 at |z| < 1, 3.1e-5 < 2, 1e-4 everywhere, a twentieth of an output's
// half step or less.  fp16: degree 7 on [0, 6], behind which outputs are zero; 5.6e-6 (1e-5 with fp32's roundings, a
// twenty-fifth).  Both fall on behind their ranges.  (640 000 rows, 64 -> 128: bf16 61 us, fp16 59; by the form above, with its reciprocal, 65 and 72.)
template <typename T>
__device__ __forceinline__ float normal_tail_half(float z) {
    const float a = fabsf(z);
    float q;
    if constexpr (std::is_same_v<T, __bf16>) {
        q = fmaf(-1.56790725e-09f, a, 1.2192244e-07f);
        q = fmaf(q, a, -4.12213922e-06f);
        q = fmaf(q, a, 8.01530987e-05f);
        q = fmaf(q, a, -0.00100325886f);
        q = fmaf(q, a, 0.00863550697f);
        q = fmaf(q, a, -0.0540182889f);
        q = fmaf(q, a, -0.458512872f);
        q = fmaf(q, a, -1.15121996f);
        q = fmaf(q, a, -0.999997079f);
    } else {
        q = fmaf(-1.8348113e-06f, a, 6.159829e-05f);
        q = fmaf(q, a, -0.00093052484f);
        q = fmaf(q, a, 0.008507891f);
        q = fmaf(q, a, -0.05396007f);
        q = fmaf(q, a, -0.45846438f);
        q = fmaf(q, a, -1.1512511f);
        q = fmaf(q, a, -0.9999953f);
    }
    return __builtin_amdgcn_exp2f(q);
}

// Half of the type's least number: what is not above it rounds to zero.  (fp32: nothing is rounded.)
template <typename T>
constexpr float kRoundsToZero = std::is_same_v<T, _Float16> ? 0x1p-25f : sizeof(T) == 2 ? 0x1p-134f : 0.f;

// z -> act(z) for N values (one uniform branch for all of them).  relu: a positive value that the type rounds to zero leaves as
// -0, so that the output's bits tell the backward of a wide layer where the slope is one.
template <typename T, int N>
__device__ __forceinline__ void act_fwd(float (&z)[N], int act) {
    if (act == FSGS_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i)  // (NaN stays)
            z[i] = z[i] <= kRoundsToZero<T> ? (sizeof(T) == 2 && z[i] > 0.f ? -0.f : 0.f) : z[i];
    } else if (act == FSGS_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float h;
            if constexpr (sizeof(T) == 2) {
                h = normal_tail_half<T>(z[i]);
            } else {
                float e;
                h = normal_tail(z[i], e);
                h *= e;
            }
            // z >= 0: z - z h; z < 0: -|z| h  (+inf, where h is zero, stays; -inf and NaN give NaN, as z Phi(z) does)
            z[i] = fmaf(-fabsf(fminf(z[i], 1e30f)), h, fmaxf(z[i], 0.f));
        }
    } else if (act == FSGS_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            z[i] *= __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z[i] * -1.4426950408889634f));
    }
}

// z -> dz = d act'(z) for N values.  (relu takes d or nothing: an infinite or NaN gradient of a value that it cut off is gone.)
template <typename T, int N>
__device__ __forceinline__ void act_bwd(float (&z)[N], const float (&d)[N], int act) {
    if (act == FSGS_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = z[i] > 0.f ? d[i] : 0.f;
    } else if (act == FSGS_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float e;
            const float p = normal_tail(z[i], e), r = e * fmaf(-0.39894228040143268f, fabsf(z[i]), p);
            z[i] = d[i] * (z[i] < 0.f ? r : 1.f - r);  // z < 0: h + z density; z >= 0: 1 - h + z density
        }
    } else if (act == FSGS_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z[i] * -1.4426950408889634f));
            z[i] = d[i] * (s * fmaf(z[i], 1.f - s, 1.f));
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = d[i];
    }
}

// A chunk that starts inside a row reaches behind the matrix only in its last 8 rows (rows at least one element apart) or
// where all rows are one.
constexpr int kEndRows = 8;

enum { kModeFwd = 0, kModeDz = 1 };

// A lane's 8 columns (of 32) of fp32 dz, summed over the 16 lanes that hold different rows.
__device__ __forceinline__ void sum_rows(float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        v[e] += dpp_f<0xB1>(v[e]);
        v[e] += dpp_f<0x4E>(v[e]);
        v[e] += dpp_f<0x141>(v[e]);
        v[e] += dpp_f<0x140>(v[e]);
    }
}
// ... and the column of each among the 32.
template <typename T>
__device__ __forceinline__ int held_column(int lg, int e) {
    return sizeof(T) == 2 ? lg * 8 + e : (e >> 2) * 16 + lg * 4 + (e & 3);
}

// Workgroups in dispatch order go round the 8 XCDs, each with an L2 of its own: neighbouring tiles, which share rows of x, are
// given to one XCD.
__device__ __forceinline__ int64_t xcd_tile(int64_t id, int64_t n) {
    const int64_t per = (n + 7) / 8, t = (id & 7) * per + (id >> 3);
    return t < n && (id >> 3) < per ? t : -1;
}

// Columns go by groups of 32 (two A tiles): in the half-width types tile t holds the rows of W with
// column = 8 (r / 4) + 4 t + r % 4 of the group, so that a lane ends with 8 neighbouring columns of one row, 16 bytes.
template <typename T>
__device__ __forceinline__ int group_column(int t, int r) {
    return sizeof(T) == 2 ? (r >> 2) * 8 + t * 4 + (r & 3) : t * 16 + r;
}

// The first n (at least one) elements of a chunk.  The two branches end apart (two empty instructions that differ).  Left to join
// them, the compiler gave both one last store, `n == 3 ? element 2 : element 3` of an fp32 chunk, and moved element 2 into the
// register of element 3 for every lane where the branches meet, before the lanes of whole chunks had stored theirs (read in the
// assembly of the store to LDS: v_mov_b32 v19, v18 behind s_or_b64 exec, then ds_write_b32 of v19 in either branch).
template <typename T>
__device__ __forceinline__ void put_chunk(T *to, const Chunk &c, int n, bool stream) {
    if (n >= kChunk<T>) {
        if (stream) store_streaming(to, c);
        else __builtin_memcpy(to, &c, sizeof(Chunk));
        asm volatile("; whole chunk" ::: "memory");
    } else {
        T t[kChunk<T>];
        __builtin_memcpy(t, &c, sizeof(Chunk));
#pragma unroll
        for (int e = 0; e < kChunk<T>; ++e)
            if (e < n) to[e] = t[e];
        asm volatile("; part of a chunk" ::: "memory");
    }
}

// A lane's values of a row of the output.
template <typename T, int MODE>
__device__ __forceinline__ void put_values(T *to, const float *v, int n, bool stream, int lo) {
    if constexpr (MODE == kModeDz && sizeof(T) == 2) {
        if (lo) {
            Chunk rest;
            put_chunk(to, split_chunk<T>(v, rest), n, stream);
            put_chunk(to + lo, rest, n, stream);
            return;
        }
    }
    put_chunk(to, pack_chunk<T>(v), n, stream);
}

// ---- general tile: 32 MT rows x BN columns, four waves of 16 MT x BN/2 ---------------------------------------------------
// Both operands go through LDS in 128-byte slabs of the summed axis (the next slab is under way in registers); W is the A
// operand, so that a lane ends with neighbouring columns of one row.  Slab rows are two to the 64 banks: chunk c of row r lies
// at c ^ key(r), with a key that gives the 16 rows of either operand 16 different bank quads.
// 128 x 128 x 100 003 rows, fp16: 512 -> 768 113 us, 694 TFLOP/s (the library's bare product: 102 us); 513 -> 768, whose rows
// start at any element, 172 (162); 8192 rows, 4096 -> 4096 310 (185).  Bound by the two barriers and the LDS reads between its
// matrix instructions; tiles of 256 rows were no faster (155 us against 158 at 513 -> 768, without the epilogue).
template <typename T, int MODE, int BN, int MT>
__global__ __launch_bounds__(256, 3) void linear_tile_kernel(LinArgs a) {
    constexpr int CE = kChunk<T>, BK = kSlabBytes / (int)sizeof(T), BM = 32 * MT;
    constexpr int NT = BN / 32;
    constexpr int XL = BM * 8 / 256, WL = BN * 8 / 256;  // chunks per thread and slab
    constexpr int CPG = sizeof(T) == 2 ? 1 : 2;          // 16-byte pieces of a row that a lane holds of 32 columns
    __shared__ Chunk xs[BM * 8], ws[BN * 8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int ntiles_n = (a.N + BN - 1) / BN;
    const int64_t tile = xcd_tile(blockIdx.x, (a.rows + BM - 1) / BM * ntiles_n);
    if (tile < 0) return;
    const int64_t m0 = tile / ntiles_n * BM;
    const int n0 = (int)(tile % ntiles_n) * BN;
    const int wm = (wave & 1) * 16 * MT, wn = (wave >> 1) * (BN / 2);
    const int li = lane & 15, lg = lane >> 4;
    // (keys depend on the row modulo 32: one per thread for its stores, one per lane and operand for its reads)
    auto xkey = [](int r) { return (r >> 1) & 7; };
    auto wkey = [](int r) { return sizeof(T) == 2 ? ((r >> 3) & 3) << 1 | ((r >> 1) & 1) : (r >> 1) & 7; };
    const int trow = tid >> 3, ck = (tid & 7) * CE;
    Chunk *const xput = xs + trow * 8 + ((tid & 7) ^ xkey(trow)), *const wput = ws + trow * 8 + ((tid & 7) ^ wkey(trow));
    const int xr0 = wm + li, wr0 = wn + group_column<T>(0, li);

    const RowReader<T> xr(a.x, a.rows, a.xp, a.K), wr(a.w, a.N, a.K, a.K);
    f32x4 acc[NT][MT] = {};
    Chunk xc[XL], wc[WL];
    auto xrow = [&](int i) { return (int)min((int64_t)(trow + i * 32), a.rows - 1 - m0); };  // (rows behind the last repeat it,
    auto wrow = [&](int i) { return min(trow + i * 32, a.N - 1 - n0); };                     //  unstored)
    auto stage = [&] {
        lds_barrier();
#pragma unroll
        for (int i = 0; i < XL; ++i) xput[i * 256] = xc[i];
#pragma unroll
        for (int i = 0; i < WL; ++i) wput[i * 256] = wc[i];
        lds_barrier();
    };
    // (a last tile of few columns, and the last slab of the summed axis, leave out what holds nothing: N = 513 has a fifth tile
    // of one column, K = 513 a ninth slab of one)
    const int nt = min(NT, (a.N - n0 - wn + 31) / 32 * 2);
    auto multiply = [&](int left) {
        const Chunk *xg[2], *wg[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            xg[s] = xs + xr0 * 8 + ((s * 4 + lg) ^ xkey(xr0));
            wg[s] = ws + wr0 * 8 + ((s * 4 + lg) ^ wkey(wr0));
        }
        auto wat = [](int i) { return (i >> 1) * 256 + (i & 1) * (sizeof(T) == 2 ? 32 : 128); };
        if (nt == NT && left > BK / 2) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                Chunk xf[MT], wf[NT];
#pragma unroll
                for (int i = 0; i < NT; ++i) wf[i] = wg[s][wat(i)];
#pragma unroll
                for (int i = 0; i < MT; ++i) xf[i] = xg[s][i * 128];
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int j = 0; j < MT; ++j) mma_chunk<T>(acc[i][j], wf[i], xf[j]);
            }
        } else if (nt > 0) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                if (s * (BK / 2) >= left) break;
                Chunk xf[MT];
#pragma unroll
                for (int i = 0; i < MT; ++i) xf[i] = xg[s][i * 128];
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    if (i >= nt) break;
                    const Chunk wf = wg[s][wat(i)];
#pragma unroll
                    for (int j = 0; j < MT; ++j) mma_chunk<T>(acc[i][j], wf, xf[j]);
                }
            }
        }
    };
    // whole slabs, byte offsets inside the tile in 32 bits; then what is left of the summed axis (or all of it, where rows lie
    // too far apart for that)
    const int kfull = a.xp * BM * (int64_t)sizeof(T) > UINT32_MAX ? 0 : a.K / BK * BK;
    if (kfull > 0) {
        uint32_t xo[XL], wo[WL];
#pragma unroll
        for (int i = 0; i < XL; ++i) xo[i] = (uint32_t)((xrow(i) * a.xp + ck) * sizeof(T));
#pragma unroll
        for (int i = 0; i < WL; ++i) wo[i] = (uint32_t)((wrow(i) * (int64_t)a.K + ck) * sizeof(T));
        auto fetch = [&](int k0) {
#pragma unroll
            for (int i = 0; i < XL; ++i) xc[i] = xr.inside(m0 * a.xp + k0, xo[i]);
#pragma unroll
            for (int i = 0; i < WL; ++i) wc[i] = wr.inside((int64_t)n0 * a.K + k0, wo[i]);
        };
        fetch(0);
        for (int k0 = 0; k0 < kfull; k0 += BK) {
            stage();
            fetch(min(k0 + BK, kfull - BK));
            multiply(BK);
        }
    }
    for (int k0 = kfull; k0 < a.K; k0 += BK) {
        const bool end = m0 + BM + kEndRows >= a.rows || n0 + BN + kEndRows >= a.N || a.xp == 0;
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            const int64_t at = (m0 + xrow(i)) * a.xp + k0 + ck;
            xc[i] = xr.raw(at);
            xr.fix(xc[i], at, a.K - k0 - ck, end);
        }
#pragma unroll
        for (int i = 0; i < WL; ++i) {
            const int64_t at = (int64_t)(n0 + wrow(i)) * a.K + k0 + ck;
            wc[i] = wr.raw(at);
            wr.fix(wc[i], at, a.K - k0 - ck, end);
        }
        stage();
        multiply(a.K - k0);
    }

    const T *bias = (const T *)a.bias;
    const T *side = (const T *)(MODE == kModeDz ? a.dy : a.res);
    const int64_t sp = MODE == kModeDz ? a.dyp : a.rp;
    const bool stream = a.stream;
#pragma unroll
    for (int i = 0; i < NT / 2; ++i) {
        float b[8], colsum[8] = {};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int n = n0 + wn + i * 32 + held_column<T>(lg, e);
            b[e] = bias && n < a.N ? (float)bias[n] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const int64_t m = m0 + wm + j * 16 + li;
            if (m >= a.rows) continue;
            float z[8], sv[8];
#pragma unroll
            for (int q = 0; q < CPG; ++q) {
                const int n = n0 + wn + i * 32 + (CPG == 1 ? lg * 8 : q * 16 + lg * 4);
                if (side) unpack_chunk<T>(load_chunk_n(side + m * sp + n, a.N - n), sv + q * CE);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = acc[2 * i + (e >> 2)][j][e & 3] + b[e];
            if constexpr (MODE == kModeDz) {
                act_bwd<T>(z, sv, a.act);
            } else {
                act_fwd<T>(z, a.act);
                if (side)
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[e] += sv[e];
            }
            if constexpr (MODE == kModeDz)
#pragma unroll
                for (int e = 0; e < 8; ++e) colsum[e] += z[e];
#pragma unroll
            for (int q = 0; q < CPG; ++q) {
                const int n = n0 + wn + i * 32 + (CPG == 1 ? lg * 8 : q * 16 + lg * 4);
                if (n < a.N) put_values<T, MODE>((T *)a.y + m * a.yp + n, z + q * CE, a.N - n, stream, a.lo);
            }
        }
        if constexpr (MODE == kModeDz)
            if (a.part_b) {
                sum_rows(colsum);
                float *to = a.part_b + (m0 / (16 * MT) + (wave & 1)) * a.N;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int n = n0 + wn + i * 32 + held_column<T>(lg, e);
                    if (li == 0 && n < a.N) to[n] = colsum[e];
                }
            }
    }
}

// ---- few rows, long summed axis: 16 rows x 32 columns per workgroup, the summed axis over its eight waves --------------------
// A wave takes every eighth 64-byte step of x and W straight from memory (four steps under way), the waves' sums meet in LDS.
constexpr int kFewWaves = 8;

// Bound by the latency of its loads: 16 rows, 1024 -> 1500, 5.3 us in bf16 and 8.3 in fp32 (by tiles 14.7 and 73).
template <typename T, int MODE>
__global__ __launch_bounds__(64 * kFewWaves) void linear_few_kernel(LinArgs a) {
    constexpr int CE = kChunk<T>, CPG = sizeof(T) == 2 ? 1 : 2, U = 4;
    __shared__ f32x4 part[kFewWaves][2][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, lg = lane >> 4;
    const int64_t m0 = (int64_t)blockIdx.y * 16, m = m0 + li;
    const int n0 = blockIdx.x * 32;
    const RowReader<T> xr(a.x, a.rows, a.xp, a.K), wr(a.w, a.N, a.K, a.K);
    const int64_t xa = min(m, a.rows - 1) * a.xp;  // (rows behind the last repeat it, unstored)
    const int64_t wa[2] = {(int64_t)min(n0 + group_column<T>(0, li), a.N - 1) * a.K,
                           (int64_t)min(n0 + group_column<T>(1, li), a.N - 1) * a.K};
    const int steps = (a.K + 4 * CE - 1) / (4 * CE);
    f32x4 acc[2] = {};
    for (int s0 = wave; s0 < steps; s0 += kFewWaves * U) {
        Chunk xc[U], wc[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = ((s0 + u * kFewWaves) * 4 + lg) * CE;
            xc[u] = xr.raw(xa + k);
            wc[u][0] = wr.raw(wa[0] + k), wc[u][1] = wr.raw(wa[1] + k);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + u * kFewWaves, k = (s * 4 + lg) * CE;
            if (s >= steps) break;
            if ((s + 1) * 4 * CE > a.K) {
                xr.fix(xc[u], xa + k, a.K - k, true);
                wr.fix(wc[u][0], wa[0] + k, a.K - k, true);
                wr.fix(wc[u][1], wa[1] + k, a.K - k, true);
            }
            mma_chunk<T>(acc[0], wc[u][0], xc[u]);
            mma_chunk<T>(acc[1], wc[u][1], xc[u]);
        }
    }
    part[wave][0][lane] = acc[0], part[wave][1][lane] = acc[1];
    __syncthreads();
    if (wave != 0) return;
    float z[8], c[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f32x4 v = part[0][i][lane];
        for (int w = 1; w < kFewWaves; ++w) v += part[w][i][lane];
#pragma unroll
        for (int q = 0; q < 4; ++q) z[i * 4 + q] = v[q];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int n = n0 + held_column<T>(lg, e);
        if (a.bias && n < a.N) z[e] += (float)((const T *)a.bias)[n];
    }
    const T *side = (const T *)(MODE == kModeDz ? a.dy : a.res);
    const int64_t sp = MODE == kModeDz ? a.dyp : a.rp;
    const bool here = m < a.rows;
    float sv[8];
    if (side)
#pragma unroll
        for (int q = 0; q < CPG; ++q) {
            const int n = n0 + (CPG == 1 ? lg * 8 : q * 16 + lg * 4);
            unpack_chunk<T>(load_chunk_n(side + (here ? m : 0) * sp + n, a.N - n), sv + q * CE);
        }
    if constexpr (MODE == kModeDz) {
        act_bwd<T>(z, sv, a.act);
    } else {
        act_fwd<T>(z, a.act);
        if (side)
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] += sv[e];
    }
#pragma unroll
    for (int q = 0; q < CPG; ++q) {
        const int n = n0 + (CPG == 1 ? lg * 8 : q * 16 + lg * 4);
        if (here && n < a.N) put_values<T, MODE>((T *)a.y + m * a.yp + n, z + q * CE, a.N - n, false, a.lo);
    }
    if (MODE == kModeDz && a.part_b) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = here ? z[e] : 0.f;
        sum_rows(c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int n = n0 + held_column<T>(lg, e);
            if (li == 0 && n < a.N) a.part_b[(int64_t)blockIdx.y * a.N + n] = c[e];
        }
    }
}

// ---- short summed axis: rows go straight from memory to the matrix pipe ------------------------------------------------
// One wave takes 16 rows at a time and all columns of its workgroup's range.  W (its range) lies in LDS for the life of the
// workgroup, a row of x is read once, 16 bytes per lane, directly in the layout of the B operand: no barrier and no staging
// in the loop.
//
// How y is stored (640 000 rows, 64 -> 128 bf16: plain 77 us, streaming 49; 32 -> 150 fp32: plain 190, streaming 463):
//   kStorePlain   through the caches: small outputs, which the next kernel finds there
//   kStoreStream  past the caches; rows must start at 64-byte boundaries, which a store instruction then covers whole
//   kStoreTile    the wave's 16 rows (neighbours in y) are put together in LDS and leave it as aligned streaming stores
// Bound by memory where the activation is cheap (921 600 rows, 64 -> 64 fp32, silu and a residual: 139 us, 708 MB at 5.1 TB/s;
// a 4 GiB copy reaches 4.8), by gelu's vector instructions at 640 000 rows, 64 -> 128 bf16 (60 us, 48 without it), and with
// fp32 class scores (640 000 rows, 32 -> 150: 130 us, 466 MB at 3.6 TB/s) by what overlaps between twelve waves a CU.
enum { kStorePlain = 0, kStoreStream = 1, kStoreTile = 2 };

struct RowsArgs {
    LinArgs l;
    int range;      // columns per workgroup (a multiple of 32)
    int transpose;  // W is given as [transpose,N], its element (n,k) at k * N + n; a longer K runs through it once more
};

template <typename T, int KC>
constexpr int rows_pitch() { return KC * 4 + 1; }  // chunks between two rows of W in LDS: 16 rows then lie in 16 bank quads

template <typename T>
constexpr int tile_bytes(int N) { return (16 * N * (int)sizeof(T) + 31) / 16 * 16; }  // (with an offset of up to a chunk)

// W's rows [n0, n0 + range) into LDS, zero behind N and K.
template <typename T, int KC>
__device__ __forceinline__ void fill_weights(Chunk *wl, const T *w, int n0, int range, int N, int K, int transpose) {
    constexpr int CE = kChunk<T>, P = rows_pitch<T, KC>();
    if (!transpose) {
        for (int c = threadIdx.x; c < range * KC * 4; c += blockDim.x) {
            const int n = c / (KC * 4), k = (c % (KC * 4)) * CE;
            wl[n * P + c % (KC * 4)] = load_chunk_n(w + (int64_t)(n0 + n) * K + k, n0 + n < N ? K - k : 0);
        }
    } else {
        for (int c = threadIdx.x; c < range * KC * 4 * CE; c += blockDim.x) {
            const int k = c / range, n = c % range;
            ((T *)(wl + n * P))[k] = n0 + n < N && k < K ? w[(int64_t)(k < transpose ? k : k - transpose) * N + n0 + n] : (T)0.f;
        }
    }
}

// Waves of a workgroup: with output tiles six, two workgroups a CU (640 000 rows, 32 -> 150 fp32: 127 us; with four, also two:
// 133).
constexpr int rows_waves(int store) { return store == kStoreTile ? 6 : 4; }

template <typename T, int MODE, int KC, int STORE>
__global__ __launch_bounds__(64 * rows_waves(STORE)) void linear_rows_kernel(RowsArgs ra) {
    constexpr int WAVES = rows_waves(STORE);
    constexpr int CE = kChunk<T>, P = rows_pitch<T, KC>();
    extern __shared__ Chunk lds[];
    const LinArgs &a = ra.l;
    T *y = (T *)a.y;
    Chunk *wl = lds;
    float *bl = (float *)(lds + ra.range * P);
    const int n0 = blockIdx.y * ra.range, ncols = min(ra.range, a.N - n0);
    fill_weights<T, KC>(wl, (const T *)a.w, n0, ra.range, a.N, a.K, ra.transpose);
    for (int n = threadIdx.x; n < ra.range; n += 64 * WAVES)
        bl[n] = a.bias && n < ncols ? (float)((const T *)a.bias)[n0 + n] : 0.f;
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, lg = lane >> 4;
    float *dbl = bl + ra.range + wave * ra.range;                      // (kModeDz with part_b: this wave's column sums)
    char *mine = (char *)(bl + ra.range) + wave * tile_bytes<T>(a.N);  // (kStoreTile)
    if (MODE == kModeDz && a.part_b)
        for (int n = lane; n < ra.range; n += 64) dbl[n] = 0.f;
    constexpr int CPG = sizeof(T) == 2 ? 1 : 2;  // 16-byte pieces of a row that a lane holds of a group
    const RowReader<T> xr(a.x, a.rows, a.xp, a.K);
    const bool has_side = MODE == kModeDz || a.res;
    const RowReader<T> sr(MODE == kModeDz ? a.dy : a.res, a.rows, MODE == kModeDz ? a.dyp : a.rp, a.N);
    const bool ragged_x = a.K != KC * 4 * CE, ragged_n = ncols % 32 != 0;
    const int64_t tiles = (a.rows + 15) / 16, step = (int64_t)gridDim.x * WAVES;
    auto column = [&](int g, int q) { return g * 32 + (CPG == 1 ? lg * 8 : q * 16 + lg * 4); };
    auto load_x = [&](Chunk (&f)[KC], int64_t row) {
#pragma unroll
        for (int c = 0; c < KC; ++c) f[c] = xr.raw(row * a.xp + (c * 4 + lg) * CE);
    };
    auto load_side = [&](Chunk (&f)[CPG], int64_t row, int g) {
#pragma unroll
        for (int q = 0; q < CPG; ++q) f[q] = sr.raw(row * sr.pitch + n0 + column(g, q));
    };
    int64_t t = (int64_t)blockIdx.x * WAVES + wave;
    // the next tile's rows, and of the side input the next group, are under way while this one is worked on
    Chunk xn[KC], sn[CPG];
    if (t < tiles) {
        load_x(xn, min(t * 16 + li, a.rows - 1));
        if (has_side) load_side(sn, min(t * 16 + li, a.rows - 1), 0);
    }
    for (; t < tiles; t += step) {
        const int64_t m = t * 16 + li, mr = min(m, a.rows - 1);  // (lanes behind the last row repeat it and store nothing)
        const int64_t mn = min((t + step) * 16 + li, a.rows - 1);
        const bool end = (t + 1) * 16 + kEndRows >= a.rows;
        Chunk xf[KC];
#pragma unroll
        for (int c = 0; c < KC; ++c) xf[c] = xn[c];
        load_x(xn, mn);
        if (ragged_x)
#pragma unroll
            for (int c = 0; c < KC; ++c) xr.fix(xf[c], mr * a.xp + (c * 4 + lg) * CE, a.K - (c * 4 + lg) * CE, end || a.xp == 0);
        T *to = y + t * 16 * a.yp;  // (kStoreTile: yp == N, one range)
        const int off = (int)(((uintptr_t)to & 15) / sizeof(T));
        for (int g = 0; g * 32 < ncols; ++g) {
            Chunk sc[CPG];
#pragma unroll
            for (int q = 0; q < CPG; ++q) sc[q] = sn[q];
            if (has_side) {
                const bool more = (g + 1) * 32 < ncols;
                load_side(sn, more ? mr : mn, more ? g + 1 : 0);
            }
            f32x4 acc[2] = {};
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    mma_chunk<T>(acc[i], wl[(g * 32 + group_column<T>(i, li)) * P + c * 4 + lg], xf[c]);
            float z[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = acc[e >> 2][e & 3] + bl[g * 32 + held_column<T>(lg, e)];
            if constexpr (MODE == kModeFwd) act_fwd<T>(z, a.act);
            if (has_side) {
                float sv[8];
#pragma unroll
                for (int q = 0; q < CPG; ++q) {
                    if (ragged_n) sr.fix(sc[q], mr * sr.pitch + n0 + column(g, q), ncols - column(g, q), end || sr.pitch == 0);
                    unpack_chunk<T>(sc[q], sv + q * CE);
                }
                if constexpr (MODE == kModeDz) {
                    act_bwd<T>(z, sv, a.act);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[e] += sv[e];
                }
            }
            if (MODE == kModeDz && a.part_b) {
                float c[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) c[e] = m < a.rows ? z[e] : 0.f;
                sum_rows(c);
                if (li == 0)
#pragma unroll
                    for (int e = 0; e < 8; ++e) dbl[g * 32 + held_column<T>(lg, e)] += c[e];
            }
#pragma unroll
            for (int q = 0; q < CPG; ++q) {
                const int n = column(g, q);
                if (m < a.rows && n < ncols) {
                    if constexpr (STORE == kStoreTile) put_values<T, MODE>((T *)mine + off + li * a.N + n, z + q * CE, ncols - n, false, 0);
                    else put_values<T, MODE>(y + m * a.yp + n0 + n, z + q * CE, ncols - n, STORE == kStoreStream, a.lo);
                }
            }
        }
        if constexpr (STORE == kStoreTile) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (LDS runs in the wave's order: no barrier)
            const int n = off + (int)min((int64_t)16, a.rows - t * 16) * a.N;
            const T *from = (const T *)mine;
            T *dst = to - off;
            for (int e0 = lane * CE; e0 < n; e0 += kWave * CE) {
                if (e0 >= off && e0 + CE <= n) store_streaming(dst + e0, *(const Chunk *)(from + e0));
                else
#pragma unroll
                    for (int e = 0; e < CE; ++e)
                        if (e0 + e >= off && e0 + e < n) dst[e0 + e] = from[e0 + e];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
    if (MODE == kModeDz && a.part_b) {
        __syncthreads();
        float *to = a.part_b + (int64_t)blockIdx.x * a.N + n0;
        const float *all = bl + ra.range;
        for (int n = threadIdx.x; n < ncols; n += 64 * WAVES)
            to[n] = (all[n] + all[ra.range + n]) + (all[2 * ra.range + n] + all[3 * ra.range + n]);
    }
}

// ---- backward of a layer whose two axes are both short: one pass over x and dy -----------------------------------------
// A workgroup of eight waves takes 128 rows at a time, a wave 16 of them.  Per 32 columns: z from W (LDS) and the wave's rows of
// x, dz = dy act'(z) in fp32 registers (db is summed from these), put into T and used twice: as it stands it is the B
// operand of dx^T = W^T dz^T, and through LDS it meets x again in dW = dz^T x, whose whole [N,K] lies in the workgroup's
// registers for the life of the workgroup.  x and dy are read once, dx is written once; W is held once, read along its rows for
// z and along its columns for dx.
// 640 000 rows: fp32 32 -> 150 201 us (its three products alone 120 at the rate of a large fp32 product, its bytes 110), bf16
// 128 -> 128 with gelu 257 us (bytes 98; 174 with dz rounded to one value).  Bound by what two waves a SIMD overlap: one workgroup
// a CU, whose waves meet twice per 128 rows.  LDS holds no second one (126 and 148 KB, of which dz 84 and 74), and a wave takes
// 230 to 256 registers for the rows of x and dy under way, dz, dx and db (dW's tiles are 12 and 32 of them).  (The two layers'
// training calls went from 0.92 to 0.38 and, with dz rounded, from 0.71 to 0.36 ms when this kernel took the place of one each
// for dz, dx and dW.)
struct BwdRowsArgs {
    const void *x, *w, *bias, *dy;
    void *dx;
    float *part_w, *part_b;  // [workgroups][N*K], [workgroups][N]
    int64_t rows, xp, dyp;
    int K, N, act, stream;
};

constexpr int kBwdWaves = 8, kBwdRows = 16 * kBwdWaves;

constexpr int bwd_wave_cols(int kt) { return kt >= 2 ? 2 : 1; }

// LDS: W [32 ceil(N/32)][K], dz [128][N], x [128][K], bias; pitches that keep 16 or 32 lanes on different banks.
template <typename T>
struct BwdRowsLds {
    int pk, pn, w, dz, x, bias, bytes, lo, fine_bytes;  // (lo: what dz's rounding left, where that is kept)
    __host__ __device__ BwdRowsLds(int KC, int N) {
        const int cols = (N + 31) / 32 * 32, pad = sizeof(T) == 2 ? 32 : 16;
        pk = KC * 64 + pad, pn = cols * (int)sizeof(T) + pad;
        w = 0, dz = w + cols * pk, x = dz + kBwdRows * pn, bias = x + kBwdRows * pk, bytes = bias + cols * 4;
        lo = bytes, fine_bytes = lo + kBwdRows * pn;
    }
};

// NG: groups of 32 columns that the registers provide for.  FINE: dz goes into its products as the sum of two values of T, the
// rounded one and what that left (split_chunk).
template <typename T, int KC, int NG, bool FINE>
__global__ __launch_bounds__(64 * kBwdWaves, 2) void linear_bwd_rows_kernel(BwdRowsArgs a) {
    constexpr int CE = kChunk<T>, CPG = sizeof(T) == 2 ? 1 : 2;
    constexpr int KT = KC * 4 / (int)sizeof(T);  // 16-column tiles of K
    // dW's tiles over the waves: 4 x 2 (fewer operands to fetch than 8 x 1, and 10 x 2 tiles come out as 3, not 4, per wave)
    constexpr int WK = bwd_wave_cols(KT), WN = kBwdWaves / WK, NTW = (2 * NG + WN - 1) / WN, KTW = KT / WK;
    extern __shared__ Chunk lds[];
    char *const mem = (char *)lds;
    const BwdRowsLds<T> lay(KC, a.N);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, lg = lane >> 4;
    const int cols = (a.N + 31) / 32 * 32, ng = cols / 32;
    float *bl = (float *)(mem + lay.bias);
    for (int c = threadIdx.x; c < cols * KC * 4; c += 64 * kBwdWaves) {
        const int n = c / (KC * 4), k = c % (KC * 4);
        *(Chunk *)(mem + lay.w + n * lay.pk + k * 16) =
            load_chunk_n((const T *)a.w + (int64_t)n * a.K + k * CE, n < a.N ? a.K - k * CE : 0);
    }
    for (int n = threadIdx.x; n < cols; n += 64 * kBwdWaves) bl[n] = a.bias && n < a.N ? (float)((const T *)a.bias)[n] : 0.f;
    __syncthreads();

    const RowReader<T> xr(a.x, a.rows, a.xp, a.K), gr(a.dy, a.rows, a.dyp, a.N);
    const bool ragged_x = a.K != KC * 4 * CE, ragged_n = a.N % 32 != 0;
    auto column = [&](int g, int q) { return g * 32 + (CPG == 1 ? lg * 8 : q * 16 + lg * 4); };
    auto load_x = [&](Chunk (&f)[KC], int64_t row) {
#pragma unroll
        for (int c = 0; c < KC; ++c) f[c] = xr.raw(row * a.xp + (c * 4 + lg) * CE);
    };
    auto load_dy = [&](Chunk (&f)[CPG], int64_t row, int g) {
#pragma unroll
        for (int q = 0; q < CPG; ++q) f[q] = gr.raw(row * a.dyp + column(g, q));
    };
    const int wn = wave / WK, wk = wave % WK;
    f32x4 accw[NTW][KTW] = {};
    constexpr bool kRegDb = sizeof(T) == 2;
    float db[kRegDb ? NG : 1][8] = {};
    float accb[kRegDb ? 1 : NTW] = {};
    const bool tiles = a.part_w || (!kRegDb && a.part_b);
    Chunk xf[KC], dyc[NG][CPG];
    const int64_t blocks = (a.rows + kBwdRows - 1) / kBwdRows;
    int64_t m = (int64_t)blockIdx.x * kBwdRows + wave * 16 + li;
    load_x(xf, min(m, a.rows - 1));
#pragma unroll
    for (int g = 0; g < NG; ++g)
        if (g < ng) load_dy(dyc[g], min(m, a.rows - 1), g);
    for (int64_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
        const int64_t next = m + (int64_t)gridDim.x * kBwdRows;
        const int row = wave * 16 + li;
        const int64_t mr = min(m, a.rows - 1), nr = min(next, a.rows - 1);
        const bool end = (blk + 1) * kBwdRows + kEndRows >= a.rows;
        const int held = (int)min((int64_t)kBwdRows, a.rows - blk * kBwdRows);  // rows of this block
        constexpr int STEP = 4 * CE;  // rows per matrix instruction of dW: 32, or 16 by four instructions
        const bool idle = wave * 16 >= (held + STEP - 1) / STEP * STEP;  // (a whole wave without rows, in the last block)
        if (!idle) {
            if (ragged_x || end)
#pragma unroll
                for (int c = 0; c < KC; ++c)
                    xr.fix(xf[c], mr * a.xp + (c * 4 + lg) * CE, m < a.rows ? a.K - (c * 4 + lg) * CE : 0, end || a.xp == 0);
            // dx^T tiles: rows k of a pair of tiles are 8 neighbours per lane in half width, 4 of one tile in fp32
            auto add_dx = [&](f32x4 &acc, int kt, int g, const Chunk (&dz)[CPG], const Chunk (&lo)[CPG]) {
                const int col = CPG == 1 ? (kt >> 1) * 32 + (li & 3) * 8 + (kt & 1) * 4 : kt * 16 + li;
#pragma unroll
                for (int q = 0; q < CPG; ++q) {
                    const int n = column(g, q);
                    const Chunk wc = load_columns<T>(mem + lay.w, lay.pk, n, n + 4, col);
                    mma_chunk<T>(acc, wc, dz[q]);
                    if constexpr (FINE) mma_chunk<T>(acc, wc, lo[q]);
                }
            };
            auto store_dx = [&](int kt, const f32x4 *acc) {
                const int k = kt * 16 + lg * CE;
                float v[CE];
#pragma unroll
                for (int e = 0; e < CE; ++e) v[e] = acc[e >> 2][e & 3];
                if (m < a.rows && k < a.K) put_chunk((T *)a.dx + m * a.K + k, pack_chunk<T>(v), a.K - k, a.stream);
            };
            // whichever holds fewer registers meanwhile: dx summed group by group, or the groups' dz kept and dx done at the end
            constexpr bool kKeepDz = KT > NG * CPG * (FINE ? 2 : 1);
            f32x4 accx[kKeepDz ? 1 : KT] = {};
            Chunk dzc[kKeepDz ? NG : 1][CPG], loc[FINE && kKeepDz ? NG : 1][CPG];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if (g >= ng) break;
                float z[8], d[8];
                if (a.act != FSGS_ACT_NONE) {
                    f32x4 acc[2] = {};
#pragma unroll
                    for (int c = 0; c < KC; ++c)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            mma_chunk<T>(acc[i], *(const Chunk *)(mem + lay.w + (g * 32 + group_column<T>(i, li)) * lay.pk + (c * 4 + lg) * 16),
                                         xf[c]);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        z[e] = acc[e >> 2][e & 3] + bl[g * 32 + held_column<T>(lg, e)];
                }
                if (ragged_n || end)
#pragma unroll
                    for (int q = 0; q < CPG; ++q)
                        gr.fix(dyc[g][q], mr * a.dyp + column(g, q), m < a.rows ? a.N - column(g, q) : 0, end || a.dyp == 0);
#pragma unroll
                for (int q = 0; q < CPG; ++q) unpack_chunk<T>(dyc[g][q], d + q * CE);
                load_dy(dyc[g], nr, g);
                if (a.act != FSGS_ACT_NONE) {
                    act_bwd<T>(z, d, a.act);
#pragma unroll
                    for (int e = 0; e < 8; ++e) d[e] = z[e];
                }
                if constexpr (kRegDb)
#pragma unroll
                    for (int e = 0; e < 8; ++e) db[g][e] += d[e];
                Chunk (&dz)[CPG] = dzc[kKeepDz ? g : 0], (&lo)[CPG] = loc[FINE && kKeepDz ? g : 0];
#pragma unroll
                for (int q = 0; q < CPG; ++q) {
                    char *const to = mem + lay.dz + row * lay.pn + column(g, q) * (int)sizeof(T);
                    if constexpr (FINE) {
                        dz[q] = split_chunk<T>(d + q * CE, lo[q]);
                        *(Chunk *)(to + (lay.lo - lay.dz)) = lo[q];
                    } else {
                        dz[q] = pack_chunk<T>(d + q * CE);
                    }
                    *(Chunk *)to = dz[q];
                }
                if constexpr (!kKeepDz)
                    if (a.dx)
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt) add_dx(accx[kt], kt, g, dz, lo);
            }
            if (a.dx) {
                if constexpr (!kKeepDz) {
#pragma unroll
                    for (int kt = 0; kt < KT; kt += 3 - CPG) store_dx(kt, accx + kt);
                } else {
#pragma unroll
                    for (int kt = 0; kt < KT; kt += 3 - CPG) {
                        f32x4 acc[3 - CPG] = {};
#pragma unroll
                        for (int g = 0; g < NG; ++g)
                            if (g < ng)
#pragma unroll
                                for (int i = 0; i < 3 - CPG; ++i) add_dx(acc[i], kt + i, g, dzc[g], loc[FINE ? g : 0]);
                        store_dx(kt, acc);
                    }
                }
            }
            if (a.part_w) {
#pragma unroll
                for (int c = 0; c < KC; ++c) *(Chunk *)(mem + lay.x + row * lay.pk + (c * 4 + lg) * 16) = xf[c];
            }
        }
        m = next;
        load_x(xf, nr);
        if (tiles) {
            lds_barrier();
            // (the wave's number of tiles compiled in: no branch between the steps)
            auto add_dw = [&](auto tiles_of_wave, auto all_rows) {
#pragma unroll
                for (int s = 0; s < kBwdRows / STEP; ++s) {
                    if (!decltype(all_rows)::value && s * STEP >= held) break;
                    const int lo = s * STEP + lg * 4, hi = lo + 16;
                    Chunk xc[KTW];
#pragma unroll
                    for (int j = 0; j < KTW; ++j)
                        xc[j] = load_columns<T>(mem + lay.x, lay.pk, lo, hi, (wk * KTW + j) * 16 + (CPG == 1 ? (li & 3) * 4 : li));
#pragma unroll
                    for (int i = 0; i < decltype(tiles_of_wave)::value; ++i) {
                        const int n = (i * WN + wn) * 16;
                        if (!decltype(all_rows)::value && n >= cols) break;
                        const Chunk zc = load_columns<T>(mem + lay.dz, lay.pn, lo, hi, n + (CPG == 1 ? (li & 3) * 4 : li));
                        if constexpr (!kRegDb) {
                            float v[4];
                            __builtin_memcpy(v, &zc, sizeof(v));
                            accb[i] += (v[0] + v[1]) + (v[2] + v[3]);
                        }
#pragma unroll
                        for (int j = 0; j < KTW; ++j) mma_chunk<T>(accw[i][j], zc, xc[j]);
                        if constexpr (FINE) {
                            const Chunk lc = load_columns<T>(mem + lay.lo, lay.pn, lo, hi, n + (li & 3) * 4);
#pragma unroll
                            for (int j = 0; j < KTW; ++j) mma_chunk<T>(accw[i][j], lc, xc[j]);
                        }
                    }
                }
            };
            const int mine = (cols / 16 - wn + WN - 1) / WN;
            const std::true_type all;
            if (held < kBwdRows) add_dw(std::integral_constant<int, NTW>(), std::false_type());  // (the last block: branches)
            else if (mine >= NTW) add_dw(std::integral_constant<int, NTW>(), all);
            else if (NTW > 1 && mine == NTW - 1) add_dw(std::integral_constant<int, (NTW > 1 ? NTW - 1 : 0)>(), all);
            else if (NTW > 2 && mine == NTW - 2) add_dw(std::integral_constant<int, (NTW > 2 ? NTW - 2 : 0)>(), all);
            else if (NTW > 3 && mine == NTW - 3) add_dw(std::integral_constant<int, (NTW > 3 ? NTW - 3 : 0)>(), all);
            lds_barrier();
        }
    }
    if (a.part_w) {
        float *pw = a.part_w + (int64_t)blockIdx.x * a.N * a.K;
#pragma unroll
        for (int i = 0; i < NTW; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int n = (i * WN + wn) * 16 + lg * 4 + q;
#pragma unroll
                for (int j = 0; j < KTW; ++j) {
                    const int k = (wk * KTW + j) * 16 + li;
                    if (n < a.N && k < a.K) pw[(int64_t)n * a.K + k] = accw[i][j][q];
                }
            }
    }
    if constexpr (!kRegDb) {
        if (a.part_b)
#pragma unroll
            for (int i = 0; i < NTW; ++i) {
                float v = accb[i];  // column li of the tile, rows of this lane group
                v += __shfl_xor(v, 16);
                v += __shfl_xor(v, 32);
                const int n = (i * WN + wn) * 16 + li;
                if (lg == 0 && wk == 0 && n < a.N) a.part_b[(int64_t)blockIdx.x * a.N + n] = v;
            }
    } else if (a.part_b) {
        float *wb = (float *)(mem + lay.dz) + wave * cols;  // (the tiles are done with: every wave is behind its last barrier)
        __syncthreads();
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            if (g >= ng) break;
            sum_rows(db[g]);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (li == 0) wb[g * 32 + held_column<T>(lg, e)] = db[g][e];
        }
        __syncthreads();
        const float *all = (const float *)(mem + lay.dz);
        for (int n = threadIdx.x; n < a.N; n += 64 * kBwdWaves) {
            float v = 0.f;
            for (int w = 0; w < kBwdWaves; ++w) v += all[w * cols + n];
            a.part_b[(int64_t)blockIdx.x * a.N + n] = v;
        }
    }
}

// ---- backward of a few rows and outputs, half width: one launch ------------------------------------------------------------
// Every workgroup forms all of dz (rows x N) by itself in fp32 LDS and takes 32 columns of dW and dx.  Bound by latency: 16
// rows, 64 -> 20 bf16 gelu 6.5 us; one row, 64 -> 150 11.4, where four rows take 18 in the one-pass kernel and its sum over slices; one row,
// 512 -> 512 48.
constexpr int kSmallDz = 512, kSmallCols = 32, kSmallWaves = 8;
constexpr int64_t kSmallWeights = 1 << 18;  // every workgroup reads all of W: up to half a megabyte

bool small_bwd(int64_t rows, int K, int N, size_t e) {
    return e == 2 && rows * N <= kSmallDz && (int64_t)K * N <= kSmallWeights;
}

struct SmallArgs {
    const void *x, *w, *bias, *dy;
    void *dx, *dw, *db;
    int64_t xp, dyp;
    int rows, K, N, act;
};

template <typename T>
__global__ __launch_bounds__(64 * kSmallWaves) void linear_bwd_small_kernel(SmallArgs a) {
    constexpr int CE = kChunk<T>, U = 4, THREADS = 64 * kSmallWaves;
    __shared__ float dz[kSmallDz], part[THREADS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, lg = lane >> 4;
    const T *x = (const T *)a.x, *w = (const T *)a.w, *bias = (const T *)a.bias, *dy = (const T *)a.dy;
    const RowReader<T> xr(a.x, a.rows, a.xp, a.K), wr(a.w, a.N, a.K, a.K);
    const bool tiny = a.N * a.K < CE;  // (of x the caller has 16 bytes to read, not of W)
    const int nts = (a.N + 15) / 16, tiles = (a.rows + 15) / 16 * nts, steps = (a.K + 4 * CE - 1) / (4 * CE);
    for (int t = wave; t < tiles; t += kSmallWaves) {  // a wave: 16 rows x 16 columns of z
        const int m = t / nts * 16 + li, n0 = t % nts * 16;
        float z[4] = {};
        if (a.act != FSGS_ACT_NONE) {
            const int64_t xa = min(m, a.rows - 1) * a.xp, wa = (int64_t)min(n0 + li, a.N - 1) * a.K;
            f32x4 acc = {};
            for (int s0 = 0; s0 < steps; s0 += U) {
                Chunk xc[U], wc[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int k = ((s0 + u) * 4 + lg) * CE;
                    xc[u] = xr.raw(xa + k);
                    if (tiny) wc[u] = load_chunk_n(w + wa + k, a.K - k);
                    else wc[u] = wr.raw(wa + k);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int k = ((s0 + u) * 4 + lg) * CE;
                    xr.fix(xc[u], xa + k, a.K - k, true);
                    if (!tiny) wr.fix(wc[u], wa + k, a.K - k, true);
                    mma_chunk<T>(acc, wc[u], xc[u]);
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) z[q] = acc[q] + (bias && n0 + lg * 4 + q < a.N ? (float)bias[n0 + lg * 4 + q] : 0.f);
        }
        float d[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) d[q] = m < a.rows && n0 + lg * 4 + q < a.N ? (float)dy[m * a.dyp + n0 + lg * 4 + q] : 0.f;
        act_bwd<T>(z, d, a.act);
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (m < a.rows && n0 + lg * 4 + q < a.N) dz[m * a.N + n0 + lg * 4 + q] = z[q];
    }
    __syncthreads();
    const int k0 = blockIdx.x * kSmallCols, cols = min(kSmallCols, a.K - k0);
    // out[o][k] = sum over j < len of dz value (o, j) times other's (j, k); where there are threads to spare each takes every S-th j
    auto product = [&](T *out, int outer, int len, int dzo, int dzj, const T *other, int64_t pitch) {
        const int items = outer * kSmallCols;
        int split = 1;
        while (split < len && items * split * 2 <= THREADS) split *= 2;
        auto sum = [&](int i, int j0, int step) {
            const int o = i / kSmallCols, k = i % kSmallCols;
            float v = 0.f;
            if (k < cols)
#pragma unroll 8
                for (int j = j0; j < len; j += step) v = fmaf(dz[o * dzo + j * dzj], (float)other[j * pitch + k0 + k], v);
            return v;
        };
        auto put = [&](int i, float v) {
            const int o = i / kSmallCols, k = i % kSmallCols;
            if (k < cols) out[(int64_t)o * a.K + k0 + k] = (T)v;
        };
        if (split == 1) {
            for (int i = tid; i < items; i += THREADS) put(i, sum(i, 0, 1));
            return;
        }
        if (tid < items * split) part[tid] = sum(tid % items, tid / items, split);
        __syncthreads();
        if (tid < items) {
            float v = part[tid];
            for (int p = 1; p < split; ++p) v += part[tid + p * items];
            put(tid, v);
        }
        __syncthreads();
    };
    if (a.dw) product((T *)a.dw, a.N, a.rows, 1, a.N, x, a.xp);
    if (a.dx) product((T *)a.dx, a.rows, a.N, a.N, 1, w, a.K);
    if (a.db && blockIdx.x == 0 && tid < a.N) {
        float v = 0.f;
        for (int m = 0; m < a.rows; ++m) v += dz[m * a.N + tid];
        ((T *)a.db)[tid] = (T)v;
    }
}

// dz of a relu layer from its output: dy where y > 0 or y is -0 (act_fwd), exact and without a product.
// Rows of `width` elements; y and dz without gaps.  Bound by memory: 100 003 x 768 fp16 76 us, 461 MB at 6.1 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void relu_dz_kernel(const T *__restrict__ dy, int64_t dyp, const T *__restrict__ y,
                                                      T *__restrict__ dz, int64_t rows, int64_t width) {
    constexpr int CE = kChunk<T>;
    const int64_t chunks = (width + CE - 1) / CE, total = rows * chunks;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = rows == 1 ? 0 : i / chunks, c = (i - r * chunks) * CE;
        const int n = (int)min(width - c, (int64_t)CE);
        const Chunk yc = load_chunk_n(y + r * width + c, n);
        Chunk g = load_chunk_n(dy + r * dyp + c, n);
        float yv[CE];
        unpack_chunk<T>(yc, yv);
        T gv[CE];
        __builtin_memcpy(gv, &g, sizeof(Chunk));
        auto minus_zero = [&](int e) {
            return sizeof(T) == 2 ? (yc.u[e >> 1] >> (e & 1) * 16 & 0xffffu) == 0x8000u : yc.u[e] == 0x80000000u;
        };
#pragma unroll
        for (int e = 0; e < CE; ++e) gv[e] = yv[e] > 0.f || minus_zero(e) ? gv[e] : (T)0.f;
        __builtin_memcpy(&g, gv, sizeof(Chunk));
        put_chunk(dz + r * width + c, g, n, false);
    }
}

// W [N,K] -> W^T [K,N], `parts` times side by side: the operand of dx = dz W with its summed axis contiguous (768 x 513 fp16:
// 5 us).
template <typename T>
__global__ __launch_bounds__(256) void transpose_kernel(const T *__restrict__ w, T *__restrict__ wt, int N, int K, int parts) {
    __shared__ T t[32][33];
    const int k0 = blockIdx.x * 32, n0 = blockIdx.y * 32;
    const int c = threadIdx.x & 31, r = threadIdx.x >> 5;
    for (int i = r; i < 32; i += 8)
        if (n0 + i < N && k0 + c < K) t[i][c] = w[(int64_t)(n0 + i) * K + k0 + c];
    __syncthreads();
    for (int i = r; i < 32; i += 8)
        if (k0 + i < K && n0 + c < N)
            for (int p = 0; p < parts; ++p) wt[((int64_t)(k0 + i) * parts + p) * N + n0 + c] = t[c][i];
}

struct DwArgs {
    const void *dz, *x;
    float *part_w, *part_b;  // [slices][N*K], [slices][N]; each may be null
    void *dw, *db;           // where `direct`: the outputs themselves, in place of the partial sums
    int64_t rows, dzp, xp, slice_rows;
    int K, N, slices, direct;
};

// dW tile over one slice of the rows: WN x WK waves (four) of 64 columns of dz x 64 columns of x.  Slabs of 64 (fp32: 32)
// rows of both lie in LDS as they come and are read by columns; the next slab is under way in registers.  db beside it, where
// dz is dy as it stands (tiles of k = 0: dz against ones).  Tiles of one slice, which share rows, go to one XCD.
// 100 003 rows, fp16: 512 x 768 124-151 us (640-520 TFLOP/s), 513 x 768 182: a fifth tile of one column is loaded like the
// others.  Bound by the barriers and column reads between its matrix instructions, two workgroups a CU.
template <typename T, int WN, int WK>
__global__ __launch_bounds__(256, 2) void linear_dw_kernel(DwArgs a) {
    static_assert(WN * WK == 4, "four waves");
    constexpr int CE = kChunk<T>, ROWS = 128 / (int)sizeof(T), STEP = 4 * CE, BN = 64 * WN, BK = 64 * WK;
    constexpr int DCPR = BN / CE, XCPR = BK / CE, DL = ROWS * DCPR / 256, XLD = ROWS * XCPR / 256;  // chunks a row, a thread
    constexpr int PAD = sizeof(T) == 2 ? 32 : 16, DP = BN * (int)sizeof(T) + PAD, XP = BK * (int)sizeof(T) + PAD;
    __shared__ Chunk ds[ROWS * DP / 16], xs[ROWS * XP / 16];
    char *const dm = (char *)ds, *const xm = (char *)xs;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, lg = lane >> 4;
    const int kts = a.part_w ? (a.K + BK - 1) / BK : 1, nts = (a.N + BN - 1) / BN;
    const int64_t id = xcd_tile(blockIdx.x, (int64_t)a.slices * kts * nts);
    if (id < 0) return;
    const int slice = (int)(id / (kts * nts)), tile = (int)(id % (kts * nts));
    const int k0 = tile % kts * BK, n0 = tile / kts * BN;
    const int wn = wave / WK * 64, wk = wave % WK * 64;
    const int nt = min(4, (a.N - n0 - wn + 15) / 16), kt = a.part_w ? min(4, (a.K - k0 - wk + 15) / 16) : 0;  // (may be < 1)
    const int64_t mb = slice * a.slice_rows, me = min(a.rows, mb + a.slice_rows);
    const bool want_b = a.part_b && k0 == 0 && wk == 0;

    const RowReader<T> dr(a.dz, a.rows, a.dzp, a.N), xr(a.x, a.rows, a.xp, a.K);
    const int drow = tid / DCPR, dcol = tid % DCPR * CE, xrow = tid / XCPR, xcol = tid % XCPR * CE;  // first chunks of a slab
    constexpr int DSTEP = 256 / DCPR, XSTEP = 256 / XCPR;
    Chunk dc[DL], xc[XLD];
    f32x4 acc[4][4] = {}, accb[4] = {};
    T one[CE];
#pragma unroll
    for (int e = 0; e < CE; ++e) one[e] = (T)1.f;
    Chunk ones;
    __builtin_memcpy(&ones, one, sizeof(Chunk));
    auto stage = [&] {
        lds_barrier();
#pragma unroll
        for (int i = 0; i < DL; ++i) *(Chunk *)(dm + (drow + i * DSTEP) * DP + dcol * (int)sizeof(T)) = dc[i];
#pragma unroll
        for (int i = 0; i < XLD; ++i) *(Chunk *)(xm + (xrow + i * XSTEP) * XP + xcol * (int)sizeof(T)) = xc[i];
        lds_barrier();
    };
    auto multiply = [&] {
        const int lc = sizeof(T) == 2 ? (li & 3) * 4 : li;
        if (nt == 4 && kt == 4 && !want_b) {
#pragma unroll
            for (int s = 0; s < ROWS / STEP; ++s) {
                const int lo = s * STEP + lg * 4, hi = lo + 16;
                Chunk df[4], xf[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    df[i] = load_columns<T>(dm, DP, lo, hi, wn + i * 16 + lc);
                    xf[i] = load_columns<T>(xm, XP, lo, hi, wk + i * 16 + lc);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) mma_chunk<T>(acc[i][j], df[i], xf[j]);
            }
        } else {
            for (int s = 0; s < ROWS / STEP; ++s) {
                const int lo = s * STEP + lg * 4, hi = lo + 16;
                Chunk xf[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < kt) xf[j] = load_columns<T>(xm, XP, lo, hi, wk + j * 16 + lc);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < nt && (kt > 0 || want_b)) {
                        const Chunk df = load_columns<T>(dm, DP, lo, hi, wn + i * 16 + lc);
                        if (want_b) mma_chunk<T>(accb[i], df, ones);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (j < kt) mma_chunk<T>(acc[i][j], df, xf[j]);
                    }
            }
        }
    };
    // Columns behind N or K read what follows the row; their sums are not stored.  So whole slabs need no care as long as that
    // still lies in the matrix; the others (the last ones, or all, where rows lie too far apart for 32-bit offsets) do.
    auto whole = [&](int64_t m1) {  // the slab that ends before row m1
        return (m1 - 1) * a.dzp + n0 + BN <= dr.lim + CE && (m1 - 1) * a.xp + k0 + BK <= xr.lim + CE;
    };
    int64_t mfull = mb + (me - mb) / ROWS * ROWS;
    if (me <= mb || max(a.dzp, a.xp) * ROWS * (int64_t)sizeof(T) > UINT32_MAX) mfull = mb;
    while (mfull > mb && !whole(mfull)) mfull -= ROWS;
    if (mfull > mb) {
        uint32_t dof[DL], xof[XLD];
#pragma unroll
        for (int i = 0; i < DL; ++i) dof[i] = (uint32_t)(((drow + i * DSTEP) * a.dzp + dcol) * sizeof(T));
#pragma unroll
        for (int i = 0; i < XLD; ++i) xof[i] = (uint32_t)(((xrow + i * XSTEP) * a.xp + xcol) * sizeof(T));
        auto fetch = [&](int64_t m0) {
#pragma unroll
            for (int i = 0; i < DL; ++i) dc[i] = dr.inside(m0 * a.dzp + n0, dof[i]);
#pragma unroll
            for (int i = 0; i < XLD; ++i) xc[i] = xr.inside(m0 * a.xp + k0, xof[i]);
        };
        fetch(mb);
        for (int64_t m0 = mb; m0 < mfull; m0 += ROWS) {
            stage();
            fetch(min(m0 + ROWS, mfull - ROWS));
            multiply();
        }
    }
    for (int64_t m0 = mfull; m0 < me; m0 += ROWS) {
        auto fetch = [&](const RowReader<T> &r, Chunk &c, int64_t mi, int at, int width) {
            const int64_t e = min(mi, a.rows - 1) * r.pitch + at;
            c = r.raw(e);
            r.fix(c, e, mi < me ? width - at : 0, true);
        };
#pragma unroll
        for (int i = 0; i < DL; ++i) fetch(dr, dc[i], m0 + drow + i * DSTEP, n0 + dcol, a.N);
#pragma unroll
        for (int i = 0; i < XLD; ++i) fetch(xr, xc[i], m0 + xrow + i * XSTEP, k0 + xcol, a.K);
        stage();
        multiply();
    }
    float *pw = a.part_w ? a.part_w + (int64_t)slice * a.N * a.K : nullptr;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int n = n0 + wn + i * 16 + lg * 4 + q;
            if (n >= a.N) continue;
            if (pw)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int k = k0 + wk + j * 16 + li;
                    if (k >= a.K) continue;
                    if (a.direct) ((T *)a.dw)[(int64_t)n * a.K + k] = (T)acc[i][j][q];
                    else pw[(int64_t)n * a.K + k] = acc[i][j][q];
                }
            if (want_b && li == 0) {
                if (a.direct) ((T *)a.db)[n] = (T)accb[i][q];
                else a.part_b[(int64_t)slice * a.N + n] = accb[i][q];
            }
        }
}

// Sum of partial gradients over their slices: C neighbouring values per workgroup, R threads take every R-th slice of a value
// (eight loads under way), in an order that the sizes alone fix.  Values behind n1 are those of a second array of n2.
template <typename T, int C, int R>
__global__ __launch_bounds__(C * R) void reduce_slices_kernel(const float *__restrict__ p1, int64_t n1, T *__restrict__ out1,
                                                              const float *__restrict__ p2, int64_t n2, T *__restrict__ out2,
                                                              int slices) {
    __shared__ float part[R][C];
    const int c = threadIdx.x % C, r = threadIdx.x / C;
    for (int64_t base = (int64_t)blockIdx.x * C; base < n1 + n2; base += (int64_t)gridDim.x * C) {
        const int64_t i = base + c;
        const bool first = i < n1, second = !first && i < n1 + n2;
        const float *from = first ? p1 + i : p2 + (i - n1);
        const int64_t pitch = first ? n1 : n2;
        float s = 0.f;
        if (first || second) {
            int t = r;
            for (; t + 7 * R < slices; t += 8 * R) {
                float v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] = from[(t + u * R) * pitch];
#pragma unroll
                for (int u = 0; u < 8; ++u) s += v[u];
            }
            for (; t < slices; t += R) s += from[t * pitch];
        }
        if constexpr (R > 1) {
            part[r][c] = s;
            __syncthreads();
            if (r == 0)
                for (int t = 1; t < R; ++t) s += part[t][c];
            __syncthreads();
        }
        if (r == 0 && first) out1[i] = (T)s;
        if (r == 0 && second) out2[i - n1] = (T)s;
    }
}

constexpr int kSlicesOfOneThread = 32;

// One or two arrays with the same number of slices.  Few values with many slices (db of a long layer: 1024 x 256) take 64 threads
// each: 5.9 us.  (16 threads each over 4096 slices, a row per wave of the kernel before it, took 110 us.)  Few slices take
// one thread a value (by sixteen: 4096 x 4096 values of two slices 41 us (399), 600 x 600 of 8 to 32 slices 4.8 (13.1), 128 x 128 of
// as many 3.6 (3.5)).
template <typename T>
int launch_reduce(const float *p1, int64_t n1, void *out1, const float *p2, int64_t n2, void *out2, int slices, hipStream_t s) {
    if (!out1) p1 = p2, n1 = n2, out1 = out2, n2 = 0;
    if (!out2) n2 = 0;
    const int64_t n = n1 + n2;
    T *const o1 = (T *)out1, *const o2 = (T *)out2;
    auto blocks = [&](int c) { return (unsigned)min((n + c - 1) / c, (int64_t)1 << 20); };  // (a grid holds at most 2^32 threads)
    if (slices > 512) reduce_slices_kernel<T, 16, 64><<<blocks(16), 1024, 0, s>>>(p1, n1, o1, p2, n2, o2, slices);
    else if (slices > kSlicesOfOneThread) reduce_slices_kernel<T, 64, 16><<<blocks(64), 1024, 0, s>>>(p1, n1, o1, p2, n2, o2, slices);
    else reduce_slices_kernel<T, 256, 1><<<blocks(256), 256, 0, s>>>(p1, n1, o1, p2, n2, o2, slices);
    return check_launch();
}

// LDS of a workgroup of the rows kernel: weights up to 40 KB, four workgroups per CU; with the waves' output tiles up to 80 KB.
constexpr int kRowsLds = 40 * 1024;
constexpr int64_t kStreamBytes = 32 << 20;  // outputs from here on are stored past the caches

unsigned rows_blocks(int64_t rows) { return (unsigned)((rows + 63) / 64 < 1024 ? (rows + 63) / 64 : 1024); }

// How the rows kernel would take a product.
struct RowsPlan {
    int kc, range, store;
    size_t bytes;
};

template <typename T, int MODE>
RowsPlan rows_plan(const LinArgs &a) {
    const int row = a.K * (int)sizeof(T);
    RowsPlan p;
    p.kc = row <= 64 ? 1 : row <= 128 ? 2 : row <= 256 ? 4 : 8;
    const int row_bytes = (p.kc * 4 + 1) * 16 + 4;  // (rows_pitch, and a bias)
    const int fit = kRowsLds / row_bytes / 32 * 32, need = (a.N + 31) / 32 * 32;
    p.range = need < fit ? need : fit;
    // few rows: more, narrower ranges, whose weights are fetched side by side (one row, 64 -> 150 fp32: 7.0 -> 4.9 us)
    while (p.range > 32 && (int64_t)rows_blocks(a.rows) * ((a.N + p.range - 1) / p.range) < 256)
        p.range = (p.range / 2 + 31) / 32 * 32;
    const bool sums = MODE == kModeDz && a.part_b;
    p.bytes = (size_t)p.range * (row_bytes + (sums ? 16 : 0));
    p.store = kStorePlain;
    if (a.rows * a.N * (int64_t)sizeof(T) >= kStreamBytes) {
        const size_t tiled = p.bytes + rows_waves(kStoreTile) * (size_t)tile_bytes<T>(a.N);
        if (a.N * sizeof(T) % 64 == 0 && (uintptr_t)a.y % 64 == 0) p.store = kStoreStream;
        else if (!sums && p.range >= a.N && a.yp == a.N && tiled <= 2 * kRowsLds) p.store = kStoreTile, p.bytes = tiled;
    }
    return p;
}

template <typename T, int MODE, int KC>
int launch_rows_kc(const RowsArgs &r, const RowsPlan &p, hipStream_t s) {
    const dim3 grid(rows_blocks(r.l.rows), (r.l.N + p.range - 1) / p.range);
    if (p.store == kStoreTile) {
        const int rc = ensure_dynamic_lds<linear_rows_kernel<T, MODE, KC, kStoreTile>>(p.bytes);
        if (rc != FSGS_OK) return rc;
        constexpr unsigned rows_tile_blocks = 512;  // (what the card holds at once; such an output is long enough for all)
        linear_rows_kernel<T, MODE, KC, kStoreTile><<<rows_tile_blocks, 64 * rows_waves(kStoreTile), p.bytes, s>>>(r);
    } else if (p.store == kStoreStream) {
        linear_rows_kernel<T, MODE, KC, kStoreStream><<<grid, 256, p.bytes, s>>>(r);
    } else {
        linear_rows_kernel<T, MODE, KC, kStorePlain><<<grid, 256, p.bytes, s>>>(r);
    }
    return check_launch();
}

template <typename T, int MODE>
int launch_rows(const LinArgs &a, int transpose, hipStream_t s) {
    const RowsPlan p = rows_plan<T, MODE>(a);
    RowsArgs r;
    r.l = a, r.range = p.range, r.transpose = transpose;
    switch (p.kc) {
        case 1: return launch_rows_kc<T, MODE, 1>(r, p, s);
        case 2: return launch_rows_kc<T, MODE, 2>(r, p, s);
        case 4: return launch_rows_kc<T, MODE, 4>(r, p, s);
        default:
            if constexpr (sizeof(T) == 4) return launch_rows_kc<T, MODE, 8>(r, p, s);
            return FSGS_EINVAL;  // (product_kind sends no such product here)
    }
}

// Which kernel a product takes (times in us; "small" is a tile of 64 x 64, "tile" of 128 x 128).
//
// Rows: a wave reads all of W from LDS for its 16 rows, a tile's waves an 8th or a 16th of that, but there x goes through LDS
// too.  It pays for short rows as long as its stores leave in whole lines, or are few (rows / small / tile):
//   640 000 rows  bf16 64 -> 128 48/60/54 | gelu 68/80/74     bf16 32 -> 150 48/92/95     fp32 32 -> 128 105/114/120 (gelu)
//   ... where they cannot  bf16 128 -> 150 227/161/142    fp32 64 -> 150 296/231/264
//   120 000 rows, outputs below kStreamBytes  bf16 64 -> 128 28/16/19    fp32 32 -> 64 21/17/17    bf16 64 -> 21 9/10/10
//   16 384 rows  fp32 32 -> 64 5.6/4.4/5.7    bf16 32 -> 64 4.3/4.4/5.3   4096 rows  bf16 32 -> 64 3.4/4.3/5.1
//   300 001 rows, longer  bf16 256 -> 1024 452/-/255    fp32 128 -> 128 109/-/115
// Few: the summed axis over a workgroup's waves, for long sums with few tiles (few / small / tile):
//   bf16 1024 -> 256  512 rows 5.5/7.6/16, 1024 9.1/7.6/16     bf16 512 -> 256  512 rows 5.4/5.2/10
//   fp32 512 -> 256  1024 rows (16 tiles) 9.9/13.9/41, 2500 (40) 23/14/42
// Small: until there are tiles enough for the card (small / tile):
//   bf16 192 -> 256  20 000 rows (314 tiles) 7.7/9.2, 40 000 (626) 13.7/13.7, 80 000 (1250) 23/19; 4096 -> 512  8000 rows 64/54
//   fp32 192 -> 256  40 000 rows (626) 46/48, 160 000 (2500) 162/152; 1024 -> 256  40 000 rows 205/211, 80 000 (1250) 400/346
enum { kByRows, kByFew, kBySmall, kByTiles };
constexpr int64_t kFewBytes = 4 << 20;
constexpr int kFewTiles = 16;  // tiles of 128 x 128 up to which the few-rows kernel is asked

template <typename T, int MODE>
int product_kind(const LinArgs &a) {
    constexpr bool half = sizeof(T) == 2;
    const int64_t out = a.rows * a.N * (int64_t)sizeof(T), tiles = (a.rows + 127) / 128 * ((a.N + 127) / 128);
    if (a.K * sizeof(T) <= (half ? 256 : 512) && (a.N <= 32 || out < kFewBytes || rows_plan<T, MODE>(a).store != kStorePlain))
        return kByRows;
    if (half ? a.K > 512 && tiles <= kFewTiles / 2 : tiles <= kFewTiles) return kByFew;
    if (half ? a.K <= 2048 && tiles <= 512 : tiles <= 1024) return kBySmall;
    return kByTiles;
}

// Rows of partial column sums that a dz kernel leaves in part_b.
int64_t sum_rows_of(int kind, int64_t rows) {
    switch (kind) {
        case kByRows: return rows_blocks(rows);
        case kByFew: return (rows + 15) / 16;
        case kBySmall: return (rows + 63) / 64 * 2;
        default: return (rows + 127) / 128 * 2;
    }
}

template <typename T, int MODE, int BN, int MT>
int launch_tiles(const LinArgs &a, hipStream_t s) {
    const int64_t tiles = (a.rows + 32 * MT - 1) / (32 * MT) * ((a.N + BN - 1) / BN), blocks = (tiles + 7) / 8 * 8;
    if (blocks > (int64_t)UINT32_MAX / 256) return FSGS_EINVAL;  // (a grid holds at most 2^32 threads)
    LinArgs b = a;
    b.stream = a.rows * a.N * (int64_t)sizeof(T) >= kStreamBytes && a.yp * sizeof(T) % 64 == 0 && (uintptr_t)a.y % 64 == 0;
    linear_tile_kernel<T, MODE, BN, MT><<<(unsigned)blocks, 256, 0, s>>>(b);
    return check_launch();
}

template <typename T, int MODE>
int launch_product(const LinArgs &a, int kind, hipStream_t s) {
    switch (kind) {
        case kByRows: return launch_rows<T, MODE>(a, 0, s);
        case kByFew:
            linear_few_kernel<T, MODE><<<dim3((a.N + 31) / 32, (unsigned)((a.rows + 15) / 16)), 64 * kFewWaves, 0, s>>>(a);
            return check_launch();
        case kBySmall: return launch_tiles<T, MODE, 64, 2>(a, s);
        default: return a.N > 64 ? launch_tiles<T, MODE, 128, 4>(a, s) : launch_tiles<T, MODE, 64, 4>(a, s);
    }
}

// dW's tiles: 128 x 128, or 256 along the other axis where one has 64 columns at most (320 000 rows, 64 -> 192 fp32: half of the
// waves of a square tile would be idle).
struct DwShape {
    int wn, wk, tiles;  // waves along N and K; tiles of [N,K]
    int64_t slices;
};

DwShape dw_shape(int64_t rows, int K, int N, bool weights) {
    DwShape p;
    p.wk = K <= 64 ? 1 : N <= 64 ? 4 : 2, p.wn = 4 / p.wk;
    p.tiles = (weights ? (K + 64 * p.wk - 1) / (64 * p.wk) : 1) * ((N + 64 * p.wn - 1) / (64 * p.wn));
    // slices of the rows: as many workgroups as the card holds (two per CU), but 256 rows each at least
    const int64_t want = 512 / p.tiles, most = (rows + 255) / 256;
    p.slices = want < most ? want : most;
    if (p.slices < 1) p.slices = 1;
    return p;
}

template <typename T>
int launch_dw(const DwArgs &d, const DwShape &p, hipStream_t s) {
    const unsigned blocks = (unsigned)((p.slices * p.tiles + 7) / 8 * 8);
    if (p.wk == 1) linear_dw_kernel<T, 4, 1><<<blocks, 256, 0, s>>>(d);
    else if (p.wk == 4) linear_dw_kernel<T, 1, 4><<<blocks, 256, 0, s>>>(d);
    else linear_dw_kernel<T, 2, 2><<<blocks, 256, 0, s>>>(d);
    return check_launch();
}

// The one-pass backward takes a layer whose weights, and the tiles of 128 rows, fit LDS, and whose accumulators (dW, dx, db)
// and rows under way fit 256 registers with something left for the work on them.
struct BwdRowsPlan {
    int kc, ng, bytes, blocks;  // kc == 0: the layer is too wide
    bool fine;  // dz as two values (FINE)
};

// gelu and silu in half width: dz is no number of the type.  (none and relu: it is dy's, or zero.)  Rounded to one it would add
// two fifths to the error of the gradients' own rounding (128 -> 128 bf16: 2.35e-3 against 1.66e-3), so its products take two
// values of it: 640 000 rows, 128 -> 128 bf16 gelu, forward and backward, 324 us against 266; 64 -> 64 87 against 69 (backward);
// 100 003 rows, 513 -> 768 fp16 gelu 980 against 640 (backward: dz 317, dx 258, dW 370).
bool two_values(int act, size_t e) { return e == 2 && (act == FSGS_ACT_GELU || act == FSGS_ACT_SILU); }

template <typename T>
constexpr bool bwd_rows_fits(int kc, int ng) {
    const int kt = kc * 4 / (int)sizeof(T), wk = bwd_wave_cols(kt), wn = kBwdWaves / wk, ntw = (2 * ng + wn - 1) / wn;
    return ntw * (kt / wk) * 4 + kt * 4 + ng * (sizeof(T) == 2 ? 12 : 8) + kc * 4 <= 144;
}

template <typename T>
BwdRowsPlan bwd_rows_plan(int64_t rows, int K, int N, int act) {
    BwdRowsPlan p = {};
    const int row = K * (int)sizeof(T);
    if (row > 512 || N > 256) return p;
    const int kc = row <= 64 ? 1 : row <= 128 ? 2 : row <= 256 ? 4 : 8, ng = (N + 63) / 64 * 2;
    const BwdRowsLds<T> lay(kc, N);
    p.fine = two_values(act, sizeof(T));
    p.bytes = p.fine ? lay.fine_bytes : lay.bytes;
    if (!bwd_rows_fits<T>(kc, ng) || p.bytes > 160 * 1024) return p;
    p.kc = kc, p.ng = ng;
    const int64_t want = (rows + kBwdRows - 1) / kBwdRows;
    p.blocks = (int)(want < 256 ? want : 256);
    return p;
}

BwdRowsPlan bwd_rows_plan(int64_t rows, int K, int N, int act, size_t e) {
    return e == 4 ? bwd_rows_plan<float>(rows, K, N, act) : bwd_rows_plan<__bf16>(rows, K, N, act);
}

template <typename T, int KC, int NG, bool FINE>
int launch_bwd_rows_as(const BwdRowsArgs &a, const BwdRowsPlan &p, hipStream_t s) {
    const int rc = ensure_dynamic_lds<linear_bwd_rows_kernel<T, KC, NG, FINE>>(p.bytes);
    if (rc != FSGS_OK) return rc;
    linear_bwd_rows_kernel<T, KC, NG, FINE><<<p.blocks, 64 * kBwdWaves, p.bytes, s>>>(a);
    return check_launch();
}

template <typename T, int KC, int NG>
int launch_bwd_rows(const BwdRowsArgs &a, const BwdRowsPlan &p, hipStream_t s) {
    if constexpr (bwd_rows_fits<T>(KC, NG)) {
        if constexpr (sizeof(T) == 2)
            if (p.fine) return launch_bwd_rows_as<T, KC, NG, true>(a, p, s);
        return launch_bwd_rows_as<T, KC, NG, false>(a, p, s);
    } else {
        return FSGS_EINVAL;
    }
}

template <typename T, int KC>
int launch_bwd_rows_n(const BwdRowsArgs &a, const BwdRowsPlan &p, hipStream_t s) {
    switch (p.ng) {
        case 2: return launch_bwd_rows<T, KC, 2>(a, p, s);
        case 4: return launch_bwd_rows<T, KC, 4>(a, p, s);
        case 6: return launch_bwd_rows<T, KC, 6>(a, p, s);
        default: return launch_bwd_rows<T, KC, 8>(a, p, s);
    }
}

template <typename T>
int launch_bwd_rows_k(const BwdRowsArgs &a, const BwdRowsPlan &p, hipStream_t s) {
    switch (p.kc) {
        case 1: return launch_bwd_rows_n<T, 1>(a, p, s);
        case 2: return launch_bwd_rows_n<T, 2>(a, p, s);
        case 4: return launch_bwd_rows_n<T, 4>(a, p, s);
        default: return launch_bwd_rows_n<T, 8>(a, p, s);
    }
}

struct BwdScratch {
    size_t dz, wt, part_w, part_b, total;
    int64_t sums;  // rows of partial column sums that part_b holds
};

// Room for the partial column sums of dz, whichever kernel forms it (that depends on where the workspace lies too).  The tile
// kernels leave two rows per tile, also for a single row of dz.
int64_t most_sum_rows(int64_t rows, int N) {
    const int64_t tiles = (rows + 127) / 128 * ((N + 127) / 128);
    int64_t most = max(max(sum_rows_of(kByRows, rows), sum_rows_of(kBySmall, rows)), sum_rows_of(kByTiles, rows));
    if (tiles <= kFewTiles) most = max(most, sum_rows_of(kByFew, rows));
    return most;
}

BwdScratch bwd_layout(int64_t rows, int K, int N, size_t e, int act, bool dx, bool dw, bool db) {
    auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    BwdScratch l;
    const BwdRowsPlan p = bwd_rows_plan(rows, K, N, act, e);
    if (p.kc) {
        l.dz = l.wt = l.part_w = 0, l.sums = p.blocks;
        l.part_b = dw ? up((size_t)p.blocks * K * N * 4) : 0;
        l.total = l.part_b + (db ? up((size_t)p.blocks * N * 4) : 0);
        return l;
    }
    const int cols = two_values(act, e) ? 2 * N : N;  // of dz
    const size_t s = (size_t)dw_shape(rows, K, cols, dw).slices;
    l.dz = 0;
    l.wt = l.dz + (act != FSGS_ACT_NONE ? up((size_t)rows * cols * e) : 0);
    l.part_w = l.wt + (dx ? up((size_t)K * cols * e) : 0);
    l.part_b = l.part_w + (dw ? up(s * (size_t)K * cols * 4) : 0);
    l.sums = act != FSGS_ACT_NONE ? max(most_sum_rows(rows, N), (int64_t)s) : (int64_t)s;
    l.total = l.part_b + (db ? up((size_t)l.sums * (size_t)N * 4) : 0);
    return l;
}

template <typename T>
int run_bwd(LinArgs a, const void *y, void *dx, void *dw, void *db, char *scratch, const BwdScratch &l, hipStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (small_bwd(a.rows, a.K, a.N, sizeof(T))) {  // (needs no workspace)
            SmallArgs b = {};
            b.x = a.x, b.xp = a.xp, b.w = a.w, b.bias = a.bias, b.dy = a.dy, b.dyp = a.dyp, b.dx = dx, b.dw = dw, b.db = db;
            b.rows = (int)a.rows, b.K = a.K, b.N = a.N, b.act = a.act;
            const int blocks = dx || dw ? (a.K + kSmallCols - 1) / kSmallCols : 1;
            linear_bwd_small_kernel<T><<<blocks, 64 * kSmallWaves, 0, s>>>(b);
            return check_launch();
        }
    const BwdRowsPlan p = bwd_rows_plan<T>(a.rows, a.K, a.N, a.act);
    if (p.kc) {
        BwdRowsArgs b = {};
        b.x = a.x, b.xp = a.xp, b.w = a.w, b.bias = a.bias, b.dy = a.dy, b.dyp = a.dyp, b.dx = dx;
        b.rows = a.rows, b.K = a.K, b.N = a.N, b.act = a.act;
        b.part_w = dw ? (float *)(scratch + l.part_w) : nullptr;
        b.part_b = db ? (float *)(scratch + l.part_b) : nullptr;
        b.stream = a.rows * a.K * (int64_t)sizeof(T) >= kStreamBytes && a.K * sizeof(T) % 64 == 0 && (uintptr_t)dx % 64 == 0;
        const int rc = launch_bwd_rows_k<T>(b, p, s);
        if (rc != FSGS_OK || (!dw && !db)) return rc;
        return launch_reduce<T>(b.part_w, (int64_t)a.N * a.K, dw, b.part_b, a.N, db, p.blocks, s);
    }
    // dz as two values: [rows, 2N], so that dx sums over twice the columns, against W twice, and dW's second half adds to its first
    const int parts = two_values(a.act, sizeof(T)) ? 2 : 1, cols = parts * a.N;
    const void *dz = a.dy;
    int64_t dzp = a.dyp;
    float *part_w = dw ? (float *)(scratch + l.part_w) : nullptr, *part_b = db ? (float *)(scratch + l.part_b) : nullptr;
    int rc = FSGS_OK, sum_rows = 0;
    if (a.act == FSGS_ACT_RELU && y) {
        const bool flat = a.dyp == a.N;
        const int64_t rows = flat ? 1 : a.rows, width = flat ? a.rows * a.N : a.N;
        const int64_t blocks = (rows * ((width + kChunk<T> - 1) / kChunk<T>) + 255) / 256;
        T *to = (T *)(scratch + l.dz);
        relu_dz_kernel<T><<<(unsigned)(blocks < 8192 ? blocks : 8192), 256, 0, s>>>((const T *)a.dy, a.dyp, (const T *)y, to, rows,
                                                                                   width);
        rc = check_launch();
        if (rc != FSGS_OK) return rc;
        dz = to, dzp = a.N;
    } else if (a.act != FSGS_ACT_NONE) {
        // (the sums of db are taken here, before dz is rounded to T)
        LinArgs z = a;
        z.y = scratch + l.dz, z.yp = cols, z.part_b = part_b, z.lo = cols - a.N;
        const int kind = product_kind<T, kModeDz>(z);
        if (part_b && sum_rows_of(kind, a.rows) > l.sums) return FSGS_ESCRATCH;
        rc = launch_product<T, kModeDz>(z, kind, s);
        if (rc != FSGS_OK) return rc;
        dz = z.y, dzp = cols, sum_rows = (int)sum_rows_of(kind, a.rows);
    }
    if (dx) {
        LinArgs g = {};
        g.x = dz, g.xp = dzp, g.y = dx, g.yp = a.K, g.rows = a.rows, g.K = cols, g.N = a.K;
        const int kind = product_kind<T, kModeFwd>(g);
        if (kind == kByRows) {
            g.w = a.w;
            rc = launch_rows<T, kModeFwd>(g, a.N, s);
        } else {
            T *wt = (T *)(scratch + l.wt);
            transpose_kernel<T><<<dim3((a.K + 31) / 32, (a.N + 31) / 32), 256, 0, s>>>((const T *)a.w, wt, a.N, a.K, parts);
            rc = check_launch();
            if (rc != FSGS_OK) return rc;
            g.w = wt;
            rc = launch_product<T, kModeFwd>(g, kind, s);
        }
        if (rc != FSGS_OK) return rc;
    }
    if (!dw && !db) return FSGS_OK;
    const DwShape shape = dw_shape(a.rows, a.K, cols, dw);
    const int slices = (int)shape.slices, sums = slices * parts;
    if (dw || !sum_rows) {
        DwArgs d = {};
        d.dz = dz, d.dzp = dzp, d.x = a.x, d.xp = a.xp, d.rows = a.rows, d.K = a.K, d.N = cols, d.slices = slices, d.direct = sums == 1;
        d.part_w = part_w, d.part_b = sum_rows ? nullptr : part_b, d.dw = dw, d.db = db;
        d.slice_rows = ((a.rows + slices - 1) / slices + 63) / 64 * 64;
        rc = launch_dw<T>(d, shape, s);
        if (rc != FSGS_OK) return rc;
    }
    const int64_t nk = (int64_t)a.N * a.K;
    if (sum_rows && db) {
        rc = launch_reduce<T>(part_b, a.N, db, nullptr, 0, nullptr, sum_rows, s);
        if (rc != FSGS_OK) return rc;
        db = nullptr;
    }
    if (sums == 1 || (!dw && !db)) return FSGS_OK;
    return launch_reduce<T>(part_w, nk, dw, part_b, a.N, db, sums, s);
}

bool bad_sizes(int64_t rows, int K, int N, int dtype, int act) {
    return rows < 0 || rows > INT32_MAX || K < 1 || N < 1 || K > FSGS_LINEAR_MAX_DIM || N > FSGS_LINEAR_MAX_DIM ||
           !known_dtype(dtype) || act < FSGS_ACT_NONE || act > FSGS_ACT_SILU;
}

}  // namespace
}  // namespace fsgs

using namespace fsgs;

extern "C" int fsgs_linear_fwd(int64_t rows, int in_dim, int out_dim, int dtype, const void *x, int64_t x_pitch, const void *w,
                               const void *bias, int act, const void *residual, int64_t res_pitch, void *y,
                               fsgs_stream_t stream) {
    if (bad_sizes(rows, in_dim, out_dim, dtype, act)) return FSGS_EINVAL;
    if (rows == 0) return FSGS_OK;
    if (!x || !w || !y || x_pitch < 0 || res_pitch < 0) return FSGS_EINVAL;
    LinArgs a = {};
    a.x = x, a.xp = x_pitch, a.w = w, a.bias = bias, a.res = residual, a.rp = res_pitch, a.y = y, a.yp = out_dim;
    a.rows = rows, a.K = in_dim, a.N = out_dim, a.act = act;
    switch (dtype) {
        case FSGS_F32: return launch_product<float, kModeFwd>(a, product_kind<float, kModeFwd>(a), as_stream(stream));
        case FSGS_BF16: return launch_product<__bf16, kModeFwd>(a, product_kind<__bf16, kModeFwd>(a), as_stream(stream));
        default: return launch_product<_Float16, kModeFwd>(a, product_kind<_Float16, kModeFwd>(a), as_stream(stream));
    }
}

extern "C" int fsgs_linear_bwd_uses_output(int64_t rows, int in_dim, int out_dim, int dtype, int act) {
    if (bad_sizes(rows, in_dim, out_dim, dtype, act)) return FSGS_EINVAL;
    const size_t e = dtype == FSGS_F32 ? 4 : 2;
    return act == FSGS_ACT_RELU && bwd_rows_plan(rows, in_dim, out_dim, act, e).kc == 0 && !small_bwd(rows, in_dim, out_dim, e);
}

extern "C" int64_t fsgs_linear_bwd_scratch_bytes(int64_t rows, int in_dim, int out_dim, int dtype, int act, int want_dx,
                                                 int want_dw, int want_db) {
    if (bad_sizes(rows, in_dim, out_dim, dtype, act)) return FSGS_EINVAL;
    return (int64_t)bwd_layout(rows, in_dim, out_dim, dtype == FSGS_F32 ? 4 : 2, act, want_dx, want_dw, want_db).total;
}

extern "C" int fsgs_linear_bwd(int64_t rows, int in_dim, int out_dim, int dtype, const void *x, int64_t x_pitch, const void *w,
                               const void *bias, int act, const void *y, const void *dy, int64_t dy_pitch, void *dx, void *dw,
                               void *db, void *scratch, int64_t scratch_bytes, fsgs_stream_t stream) {
    if (bad_sizes(rows, in_dim, out_dim, dtype, act)) return FSGS_EINVAL;
    if (rows == 0 || (!dx && !dw && !db)) return FSGS_OK;
    if (!x || !w || !dy || x_pitch < 0 || dy_pitch < 0) return FSGS_EINVAL;
    const BwdScratch l = bwd_layout(rows, in_dim, out_dim, dtype == FSGS_F32 ? 4 : 2, act, dx, dw, db);
    if (l.total > 0 && (!scratch || scratch_bytes < (int64_t)l.total)) return FSGS_ESCRATCH;
    LinArgs a = {};
    a.x = x, a.xp = x_pitch, a.w = w, a.bias = bias, a.dy = dy, a.dyp = dy_pitch;
    a.rows = rows, a.K = in_dim, a.N = out_dim, a.act = act;
    switch (dtype) {
        case FSGS_F32: return run_bwd<float>(a, y, dx, dw, db, (char *)scratch, l, as_stream(stream));
        case FSGS_BF16: return run_bwd<__bf16>(a, y, dx, dw, db, (char *)scratch, l, as_stream(stream));
        default: return run_bwd<_Float16>(a, y, dx, dw, db, (char *)scratch, l, as_stream(stream));
    }
}
