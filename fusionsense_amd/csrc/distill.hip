// Distillation from a teacher's top-K scores: row losses, their (weighted) reduction, and the gradient of the student's scores.
//
//   p = softmax over the row's entries of u / T,  q = softmax over all V classes of s / T
//   L = T^2 sum_k p_k (log p_k - log q_{t_k}),    dL/ds_j = T (q_j - sum_{k: t_k = j} p_k)
//
// An entry whose class lies outside [0, V) is no entry; a row without entries (or whose entries are all -inf) and a row of
// weight zero have loss 0 and gradient 0, whatever their scores hold.  Softmax statistics and sums are fp32, the sums over
// rows fp64; every sum runs in a fixed order.
#include "half_types.h"

namespace fsgs {

namespace {

constexpr int kRowBlocks = 1536;   // workgroups that go round the rows: the 6 per CU that are resident at once
constexpr int kMaxBlocks = 4096;   // ... where a row fills a workgroup: handed out as they finish
constexpr int kWideRow = 256;      // lanes of a row that has a workgroup to itself

struct DistillArgs {
    const void *s, *idx, *u;
    const float *weight;
    int64_t rows, sp, ip, up;
    int V, K, tdtype, idx64;
    float T, scale2, loss_scale;  // log2(e) / T, T^2 ln 2
    float *row_loss;      // fwd, reduction none: [rows]
    float4 *stat;         // [rows] max s, 1 / sum_j exp, max u, 1 / sum_k exp (0: the row counts for nothing)
    double2 *partial;     // [workgroups] sum of w L, sum of w
    const float *g;       // bwd: upstream gradient (one value, or one per row)
    const float *inv_w;   // bwd: 1 / sum of weights, or null
    int g_per_row;
    void *ds;             // [rows, V]
};

__device__ __forceinline__ float teacher_at(const void *u, int64_t i, int dtype) {
    if (dtype == FSGS_F32) return ((const float *)u)[i];
    if (dtype == FSGS_BF16) return (float)((const __bf16 *)u)[i];
    return (float)((const _Float16 *)u)[i];
}

__device__ __forceinline__ int class_at(const void *idx, int64_t i, int idx64, int V) {
    const int64_t c = idx64 ? ((const int64_t *)idx)[i] : (int64_t)((const int32_t *)idx)[i];
    return c >= 0 && c < V ? (int)c : -1;
}

// ---- reductions over the L lanes (neighbours, L a power of two) of a row ----
struct MaxOp {
    __device__ static float f(float a, float b) { return fmaxf(a, b); }
};
struct AddOp {
    __device__ static float f(float a, float b) { return a + b; }
};
template <int L, class Op>
__device__ __forceinline__ float lanes_reduce(float v) {
    if constexpr (L >= 2) v = Op::f(v, dpp_f<0xB1>(v));    // quad_perm [1,0,3,2]
    if constexpr (L >= 4) v = Op::f(v, dpp_f<0x4E>(v));    // quad_perm [2,3,0,1]
    if constexpr (L >= 8) v = Op::f(v, dpp_f<0x141>(v));   // row_half_mirror
    if constexpr (L >= 16) v = Op::f(v, dpp_f<0x140>(v));  // row_mirror
    if constexpr (L >= 32) v = Op::f(v, __shfl_xor(v, 16));
    if constexpr (L >= 64) v = Op::f(v, __shfl_xor(v, 32));
    return v;
}
// three at once: a row that fills a workgroup joins its waves behind one barrier
template <int L, class Op>
__device__ __forceinline__ void row_reduce(float &x, float &y, float &z) {
    x = lanes_reduce<L, Op>(x), y = lanes_reduce<L, Op>(y), z = lanes_reduce<L, Op>(z);
    if constexpr (L == kWideRow) {
        __shared__ float part[3][4];
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            const int w = threadIdx.x >> 6;
            part[0][w] = x, part[1][w] = y, part[2][w] = z;
        }
        __syncthreads();
        auto all = [](const float *p) { return Op::f(Op::f(p[0], p[1]), Op::f(p[2], p[3])); };
        x = all(part[0]), y = all(part[1]), z = all(part[2]);
    }
}
template <int L>
__device__ __forceinline__ bool lanes_any(bool b) {
    const uint64_t m = __ballot(b);
    if constexpr (L == 64) return m != 0;
    const int first = (threadIdx.x & 63) & ~(L - 1);
    return (m >> first) & ((1ull << (L & 63)) - 1);
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// A row is read in chunks of 16 bytes, chunk c by lane c mod L, kStep chunks per lane at a time (all of a row that has at most
// kStep * L chunks: lanes_per_row).  Rows start at any element.  The last chunk of a row that does not end on one is read
// shifted back to end with the row, its doubled elements masked: no element-wise reads, nothing behind the row.
constexpr int kStep = 5;
constexpr int kFullSteps = 2;  // with several lanes per row every row has more than kStep / 2 chunks a lane
template <int STEPS>
constexpr int kHeldOf = STEPS == kStep ? 2 : 4;  // entries per lane kept in registers; further ones are read again where needed

template <typename T, int L, int STEPS>
__device__ __forceinline__ void load_step(Chunk (&c)[STEPS], const T *s, int c0, int V) {
    constexpr int CE = kChunk<T>;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int j = (c0 + i * L) * CE;
        if (V < CE) c[i] = load_chunk_n(s, j < V ? V : 0);
        else c[i] = load_chunk(s + min(j, V - CE));
    }
}

// -inf in place of what other chunks count, or of what lies behind the row, in the chunk at element j.
template <typename T>
__device__ __forceinline__ void mask_chunk(Chunk &c, int j, int V) {
    constexpr int CE = kChunk<T>;
    if (j + CE <= V) return;
    const int from = V < CE ? 0 : j - (V - CE), to = j >= V ? 0 : (V < CE ? V : CE);
    T t[CE];
    __builtin_memcpy(t, &c, sizeof(Chunk));
#pragma unroll
    for (int e = 0; e < CE; ++e) t[e] = e >= from && e < to ? t[e] : (T)-INFINITY;
    __builtin_memcpy(&c, t, sizeof(Chunk));
}

// The compiler must not keep a chunk's floats from one pass over it to the next (8 registers against 4).
__device__ __forceinline__ void forget(Chunk &c) {
    asm volatile("" : "+v"(c.u[0]), "+v"(c.u[1]), "+v"(c.u[2]), "+v"(c.u[3]));
}

typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// Maximum of a lane's chunks.  Half-width types: two elements per instruction on their bits.  As signed integers non-negative
// floats order as they should and lie above all negative ones; if there is none, the largest negative float has the smallest
// unsigned bits.  (A NaN is either the largest of all, and then the maximum, or ignored: it reaches the sum either way.)
template <typename T, int STEPS>
__device__ __forceinline__ float chunks_max(const Chunk (&c)[STEPS]) {
    if constexpr (sizeof(T) == 4) {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) m = fmaxf(m, __builtin_bit_cast(float, c[i].u[e]));
        return m;
    } else {
        i16x2 hi = __builtin_bit_cast(i16x2, c[0].u[0]);
        u16x2 lo = __builtin_bit_cast(u16x2, c[0].u[0]);
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                hi = __builtin_elementwise_max(hi, __builtin_bit_cast(i16x2, c[i].u[e]));
                lo = __builtin_elementwise_min(lo, __builtin_bit_cast(u16x2, c[i].u[e]));
            }
        const int h = max((int)hi.x, (int)hi.y), l = min((int)lo.x, (int)lo.y);
        return (float)__builtin_bit_cast(T, (unsigned short)(h >= 0 ? h : l));
    }
}

// Exponents of a row against its maximum m, in base 2.  A row that its lanes hold whole: one multiply-add per score, v scale2 -
// round(m scale2).  The shift's rounding is the same for every score of the row and cancels in the softmax, as all of its parts
// use this form.  It is 2^-9 at most: from a shift of 2^16 on the difference is taken first (from 2^32 on half a step of the
// shift alone would leave the exponential's range: a row of nothing but -1e10, or scores of 12 345 at T = 1e-6).
// A row that fills a workgroup always takes the difference first: its lanes sum against maxima of their own, whose shifts'
// roundings would stay in the sum (4e-6 of it at an offset of 1000, 4e-5 at 1e4).  It costs nothing there (V = 32 003: 200 us
// either way, forward and backward); held rows would pay for it (800x800 x 150 fp32: 264 against 292).
template <int L>
struct RowExp {
    float m, scale2, shift;
    bool far;
    __device__ RowExp(float m_, float s)
        : m(m_ == -INFINITY ? 0.f : m_), scale2(s), shift(m * s), far(L == kWideRow || !(fabsf(shift) < 65536.f)) {}
    __device__ __forceinline__ float of(float v) const { return far ? (v - m) * scale2 : fmaf(v, scale2, -shift); }
};

// L lanes per row, the row in their registers (a row that fills a workgroup: step by step, the next step's loads under way).
// Bound by memory up to some thousand classes: 640 000 x 150 fp32 with K = 16 102 us, 445 MB at 4.4 TB/s; 230 400 x 1203 bf16 with
// K = 32 155 us, 630 MB at 4.1.  4099 x 32 003 fp16 95 us, 262 MB at 2.8 TB/s: four steps a row beside its joins; more workgroups
// a CU would spill (5: 120 us, 6: 150).  2 073 600 x 21 bf16 with K = 4 51 us: a lane per row, by its entries' dependent loads.
template <typename T, int L, int STEPS>
__global__ __launch_bounds__(256, L == kWideRow ? 4 : 6) void distill_fwd_kernel(DistillArgs a) {
    constexpr int CE = kChunk<T>, ROWS = 256 / L, kHeld = kHeldOf<STEPS>;
    const int sub = threadIdx.x & (L - 1);
    const int chunks = (a.V + CE - 1) / CE;
    double sum_l = 0.0, sum_w = 0.0;
    for (int64_t base = (int64_t)blockIdx.x * ROWS; base < a.rows; base += (int64_t)gridDim.x * ROWS) {
        const int64_t slot = base + threadIdx.x / L;
        const bool here = slot < a.rows;
        const int64_t row = here ? slot : a.rows - 1;  // (lanes behind the last row repeat it and store nothing)
        const T *s = (const T *)a.s + row * a.sp;
        Chunk c[STEPS];
        load_step<T, L>(c, s, sub, a.V);
        int cls[kHeld];
        float u[kHeld], sv[kHeld];
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int k = i * L + sub;
            cls[i] = -1;
            if (i * L < a.K && k < a.K) cls[i] = class_at(a.idx, row * a.ip + k, a.idx64, a.V);
        }
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            u[i] = sv[i] = -INFINITY;
            if (i * L < a.K && cls[i] >= 0) {
                u[i] = teacher_at(a.u, row * a.up + i * L + sub, a.tdtype);
                sv[i] = (float)s[cls[i]];
            }
        }
        const float w = a.weight ? a.weight[row] : 1.f;

        float um = -INFINITY, any = 0.f;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            um = fmaxf(um, u[i]);
            any = u[i] != -INFINITY ? 1.f : any;  // (NaN counts: it reaches the loss)
        }
        for (int k = kHeld * L + sub; k < a.K; k += L)
            if (class_at(a.idx, row * a.ip + k, a.idx64, a.V) >= 0) {
                const float uk = teacher_at(a.u, row * a.up + k, a.tdtype);
                um = fmaxf(um, uk);
                any = uk != -INFINITY ? 1.f : any;
            }

        // maximum and sum of the row: held whole, or step by step with a lane's sum rescaled to its new maximum
        float m = -INFINITY, sum = 0.f;
        for (int c0 = sub;;) {
            const bool more = L == kWideRow && c0 - sub + STEPS * L < chunks;
            Chunk ahead[STEPS];
            if (more) load_step<T, L>(ahead, s, c0 + STEPS * L, a.V);
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
                if (!(L > 1 && L < kWideRow && i < kFullSteps)) mask_chunk<T>(c[i], (c0 + i * L) * CE, a.V);
            const float before = m;
            m = fmaxf(m, chunks_max<T>(c));
            if constexpr (L != kWideRow) row_reduce<L, MaxOp>(m, um, any);
            const RowExp<L> x(m, a.scale2);
            if constexpr (L == kWideRow) sum *= exp2_hw(x.of(before));
            auto add = [&](auto exponent) {
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    float v[CE];
                    if constexpr (sizeof(T) == 2) forget(c[i]);
                    unpack_chunk<T>(c[i], v);
#pragma unroll
                    for (int e = 0; e < CE; ++e) sum += exp2_hw(exponent(v[e]));
                }
            };
            if (__any(x.far)) add([&](float v) { return x.of(v); });
            else add([&](float v) { return fmaf(v, x.scale2, -x.shift); });
            if (!more) break;
            c0 += STEPS * L;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) c[i] = ahead[i];
        }
        if constexpr (L == kWideRow) {
            const float lane_m = m;
            row_reduce<L, MaxOp>(m, um, any);
            sum *= exp2_hw(RowExp<L>(m, a.scale2).of(lane_m));
        }
        const RowExp<L> x(m, a.scale2);
        const bool alive = any != 0.f && w != 0.f;
        // sum_k p_k (log p_k - log q_k) = (sum_k e_k y_k) / Z - log Z + log S with e_k = exp((u_k - um) / T), Z their sum,
        // y_k = (u_k - um) / T - (s_k - m) / T; exponents and logarithms in base 2, ln 2 at the end
        float z = 0.f, ex = 0.f;
        auto entry = [&](float uk, float sk) {
            const float lu = (uk - um) * a.scale2, e = exp2_hw(lu);
            z += e;
            if (e != 0.f) ex += e * (lu - x.of(sk));
        };
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (i * L < a.K && cls[i] >= 0) entry(u[i], sv[i]);
        for (int k = kHeld * L + sub; k < a.K; k += L) {
            const int ck = class_at(a.idx, row * a.ip + k, a.idx64, a.V);
            if (ck >= 0) entry(teacher_at(a.u, row * a.up + k, a.tdtype), (float)s[ck]);
        }
        row_reduce<L, AddOp>(sum, z, ex);
        if (m == -INFINITY) sum = NAN;  // (a row of -inf only has no softmax)
        if (sub == 0 && here) {
            const float inv_z = __builtin_amdgcn_rcpf(z);
            const float loss = (ex * inv_z + (__builtin_amdgcn_logf(sum) - __builtin_amdgcn_logf(z))) * a.loss_scale;
            const float wl = alive ? w * loss : 0.f;
            if (a.row_loss) a.row_loss[row] = wl;
            if (a.stat) a.stat[row] = make_float4(m, __builtin_amdgcn_rcpf(sum), um, alive ? inv_z : 0.f);
            if (alive) sum_l += (double)wl, sum_w += (double)w;
        }
    }
    if (a.partial) {
        __shared__ double2 part[256];
        part[threadIdx.x] = make_double2(sum_l, sum_w);
        __syncthreads();
        for (int o = 128; o; o >>= 1) {
            if ((int)threadIdx.x < o) {
                part[threadIdx.x].x += part[threadIdx.x + o].x;
                part[threadIdx.x].y += part[threadIdx.x + o].y;
            }
            __syncthreads();
        }
        if (threadIdx.x == 0) a.partial[blockIdx.x] = part[0];
    }
}

// loss = sum w L (/ sum w), in a fixed order (one workgroup: 4-5 us for 1536 partial sums); inv_w is what the gradient is
// scaled by.  All weights zero: loss 0, no gradient.
__global__ __launch_bounds__(256) void distill_reduce_kernel(const double2 *__restrict__ partial, int n, int mean, float *loss,
                                                             float *inv_w) {
    __shared__ double2 part[256];
    double2 t = make_double2(0.0, 0.0);
    for (int i = threadIdx.x; i < n; i += 256) t.x += partial[i].x, t.y += partial[i].y;
    part[threadIdx.x] = t;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if ((int)threadIdx.x < o) {
            part[threadIdx.x].x += part[threadIdx.x + o].x;
            part[threadIdx.x].y += part[threadIdx.x + o].y;
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const double w = part[0].y;
        const double inv = mean ? (w != 0.0 ? 1.0 / w : 0.0) : 1.0;
        *loss = (float)(part[0].x * inv);
        if (inv_w) *inv_w = (float)inv;
    }
}

// LDS of one wave of the backward: its rows' gradients behind up to one chunk of offset, then a bit per class and row.
template <typename T, int L>
struct BwdLds {
    int words, bits_at, bytes;
    __host__ __device__ explicit BwdLds(int V) {
        words = (V + 31) / 32;
        bits_at = ((kWave / L) * V * (int)sizeof(T) + 31) / 16 * 16;
        bytes = bits_at + ((kWave / L) * words * 4 + 15) / 16 * 16;
    }
};

// Bound by memory: 640 000 x 150 fp32 162 us, 845 MB at 5.2 TB/s; 230 400 x 1203 bf16 297 us, 1.19 GB at 4.0 TB/s.
// A wave's rows (64 / L of them, neighbours in the gradient) are put together in LDS and leave it as aligned 16-byte
// streaming stores: rows start at any element, and the line that two stores share would otherwise be written twice.  q of every
// class goes first, then the teacher's classes once more with their mass taken off.  A class may stand in several entries: its
// first entry carries their sum, taken in the entries' order; whether a row has such a class at all is found with one bit per
// class.  A row's lanes are one wave's, and LDS runs in a wave's order: no barrier.
template <typename T, int L, int STEPS>
__global__ __launch_bounds__(256, 5) void distill_bwd_kernel(DistillArgs a) {
    constexpr int CE = kChunk<T>, ROWS = kWave / L, kHeld = kHeldOf<STEPS>;
    extern __shared__ Chunk lds[];
    const int lane = threadIdx.x & 63, sub = lane & (L - 1), group = lane / L;
    const BwdLds<T, L> lay(a.V);
    char *mine = (char *)lds + (threadIdx.x >> 6) * lay.bytes;
    uint32_t *bits = (uint32_t *)(mine + lay.bits_at) + group * lay.words;
    const float up = a.g_per_row ? 0.f : a.g[0];
    const float inv_w = a.inv_w ? *a.inv_w : 1.f;
    const int64_t waves = (int64_t)gridDim.x * 4;
    for (int64_t base = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * ROWS; base < a.rows; base += waves * ROWS) {
        const int64_t slot = base + group;
        const bool here = slot < a.rows;
        const int64_t row = here ? slot : a.rows - 1;
        const T *s = (const T *)a.s + row * a.sp;
        Chunk c[STEPS];
        load_step<T, L>(c, s, sub, a.V);
        const float4 st = a.stat[row];
        const bool dead = st.w == 0.f || !here;
        const float coef = a.T * (a.weight ? a.weight[row] : 1.f) * (a.g_per_row ? a.g[row] : up) * inv_w;
        const RowExp<L> x(st.x, a.scale2);
        const float cq = dead ? 0.f : coef * st.y, cp = coef * st.w;
        auto class_of = [&](int k) { return class_at(a.idx, row * a.ip + k, a.idx64, a.V); };
        auto mass_of = [&](int k) { return cp * exp2_hw((teacher_at(a.u, row * a.up + k, a.tdtype) - st.z) * a.scale2); };
        int cls[kHeld];
        float p[kHeld], sv[kHeld];
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int k = i * L + sub;
            cls[i] = i * L < a.K && k < a.K && !dead ? class_of(k) : -1;
        }
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (i * L < a.K && cls[i] >= 0) {
                p[i] = mass_of(i * L + sub);
                sv[i] = (float)s[cls[i]];
                bits[cls[i] >> 5] = 0;
            }
        if (!dead)
            for (int k = kHeld * L + sub; k < a.K; k += L) {
                const int ck = class_of(k);
                if (ck >= 0) bits[ck >> 5] = 0;
            }
        // the wave's part of the gradient, at the offset that its start has from a 16-byte boundary
        T *to = (T *)a.ds + base * a.V;
        const int off = (int)(((uintptr_t)to & 15) / sizeof(T));
        T *tile = (T *)mine + off, *out_row = tile + group * a.V;
        auto put = [&](auto exponent) {
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const int j = (sub + i * L) * CE;
                if (j >= a.V || !here) break;
                float v[CE];
                unpack_chunk<T>(c[i], v);
#pragma unroll
                for (int e = 0; e < CE; ++e) v[e] = cq * exp2_hw(exponent(v[e]));
                if (a.V < CE) {
#pragma unroll
                    for (int e = 0; e < CE; ++e)
                        if (e < a.V) out_row[e] = (T)v[e];
                } else {
                    // (the last chunk of a row stores the elements before it a second time, with the same values)
                    const Chunk out = pack_chunk<T>(v);
                    __builtin_memcpy(out_row + min(j, a.V - CE), &out, sizeof(Chunk));
                }
            }
        };
        // (a row that counts for nothing gives zeros, whatever it holds)
        if (__any(x.far || dead)) put([&](float v) { return dead ? -INFINITY : x.of(v); });
        else put([&](float v) { return fmaf(v, x.scale2, -x.shift); });
        bool again = false;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (another lane may have cleared the word)
        auto mark = [&](int ck) { again |= (atomicOr(&bits[ck >> 5], 1u << (ck & 31)) >> (ck & 31)) & 1u; };
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (i * L < a.K && cls[i] >= 0) mark(cls[i]);
        if (!dead)
            for (int k = kHeld * L + sub; k < a.K; k += L) {
                const int ck = class_of(k);
                if (ck >= 0) mark(ck);
            }
        again = lanes_any<L>(again);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        auto fix = [&](int k, int ck, float pk, float sk) {
            if (again) {
                pk = 0.f;
                bool first = true;
                for (int t = 0; t < a.K; ++t)
                    if (class_of(t) == ck) pk += mass_of(t), first &= t >= k;
                if (!first) return;
            }
            out_row[ck] = (T)fmaf(cq, exp2_hw(x.of(sk)), -pk);
        };
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (i * L < a.K && cls[i] >= 0) fix(i * L + sub, cls[i], p[i], sv[i]);
        if (!dead)
            for (int k = kHeld * L + sub; k < a.K; k += L) {
                const int ck = class_of(k);
                if (ck >= 0) fix(k, ck, mass_of(k), (float)s[ck]);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int n = off + (int)min((int64_t)ROWS, a.rows - base) * a.V;  // elements [off, n) of the wave's LDS
        T *from = (T *)mine, *dst = to - off;
        for (int e0 = lane * CE; e0 < n; e0 += kWave * CE) {
            if (e0 >= off && e0 + CE <= n) {
                store_streaming(dst + e0, *(const Chunk *)(from + e0));
            } else {
#pragma unroll
                for (int e = 0; e < CE; ++e)
                    if (e0 + e >= off && e0 + e < n) dst[e0 + e] = from[e0 + e];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// One row per workgroup, too long for a float per class in LDS: q for every class first, then the teacher's classes once more
// with their mass taken off.  One bit per class finds a class that stands in several entries.  Bound by memory:
// 4099 x 32 003 fp16 103 us, 525 MB at 5.1 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void distill_bwd_wide_kernel(DistillArgs a) {
    constexpr int CE = kChunk<T>, L = kWideRow;
    extern __shared__ uint32_t seen[];
    const int sub = threadIdx.x;
    const int chunks = (a.V + CE - 1) / CE;
    const float up = a.g_per_row ? 0.f : a.g[0];
    const float inv_w = a.inv_w ? *a.inv_w : 1.f;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *s = (const T *)a.s + row * a.sp;
        T *ds = (T *)a.ds + row * a.V;
        Chunk c[kStep];
        load_step<T, L>(c, s, sub, a.V);
        const float4 st = a.stat[row];
        const bool dead = st.w == 0.f;
        const float coef = a.T * (a.weight ? a.weight[row] : 1.f) * (a.g_per_row ? a.g[row] : up) * inv_w;
        const RowExp<L> x(st.x, a.scale2);
        const float cq = coef * st.y, cp = coef * st.w;
        // (at most one entry per lane: K <= 256)
        const int cls = sub < a.K && !dead ? class_at(a.idx, row * a.ip + sub, a.idx64, a.V) : -1;
        auto mass_of = [&](int k) { return cp * exp2_hw((teacher_at(a.u, row * a.up + k, a.tdtype) - st.z) * a.scale2); };
        float q = 0.f, mass = 0.f;
        if (cls >= 0) {
            q = cq * exp2_hw(x.of((float)s[cls]));
            mass = mass_of(sub);
            seen[cls >> 5] = 0;
        }
        for (int c0 = sub;;) {
#pragma unroll
            for (int i = 0; i < kStep; ++i) {
                const int j = (c0 + i * L) * CE;
                if (j >= a.V) break;
                float v[CE];
                unpack_chunk<T>(c[i], v);
#pragma unroll
                for (int e = 0; e < CE; ++e) v[e] = dead ? 0.f : cq * exp2_hw(x.of(v[e]));
                const Chunk out = pack_chunk<T>(v);
                __builtin_memcpy(ds + min(j, a.V - CE), &out, sizeof(Chunk));
            }
            c0 += kStep * L;
            if (c0 - sub >= chunks) break;
            load_step<T, L>(c, s, c0, a.V);
        }
        // every store above has landed before a lane writes over one of them
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        const bool taken = cls >= 0 && ((atomicOr(&seen[cls >> 5], 1u << (cls & 31)) >> (cls & 31)) & 1u);
        bool first = cls >= 0;
        if (__syncthreads_or(taken) && cls >= 0) {
            mass = 0.f;
            for (int t = 0; t < a.K; ++t)
                if (class_at(a.idx, row * a.ip + t, a.idx64, a.V) == cls) mass += mass_of(t), first &= t >= sub;
        }
        if (first) ds[cls] = (T)(q - mass);
        __syncthreads();
    }
}

// Lanes per row: the fewest that hold the row in kStep chunks each (a wave then has many rows in flight and the joins over
// lanes stay short); a row that 64 lanes cannot hold gets a workgroup.
int lanes_per_row(int V, int dtype) {
    const int ce = dtype == FSGS_F32 ? 4 : 8, chunks = (V + ce - 1) / ce;
    int l = 1;
    while (l <= 64 && chunks > kStep * l) l *= 2;
    return l <= 64 ? l : kWideRow;
}

int row_blocks(int64_t rows, int lanes) {
    const int64_t per = 256 / lanes, b = (rows + per - 1) / per, most = lanes == kWideRow ? kMaxBlocks : kRowBlocks;
    return (int)(b < most ? b : most);
}

template <typename T, int L, int STEPS>
void launch_rows(const DistillArgs &a, bool bwd, hipStream_t st) {
    const int blocks = row_blocks(a.rows, L);
    if constexpr (L == kWideRow) {
        if (bwd) return distill_bwd_wide_kernel<T><<<blocks, 256, (size_t)((a.V + 31) / 32) * 4, st>>>(a);
    } else {
        if (bwd) return distill_bwd_kernel<T, L, STEPS><<<blocks, 256, 4 * BwdLds<T, L>(a.V).bytes, st>>>(a);
    }
    distill_fwd_kernel<T, L, STEPS><<<blocks, 256, 0, st>>>(a);
}

template <typename T, int L>
void launch_steps(const DistillArgs &a, bool bwd, hipStream_t st) {
    // (a row of three steps does not carry the registers and the idle steps of five: 1080p, V = 21: 67 -> 58 us)
    if (a.V <= 3 * L * kChunk<T>) launch_rows<T, L, 3>(a, bwd, st);
    else launch_rows<T, L, kStep>(a, bwd, st);
}

template <typename T>
void launch_lanes(const DistillArgs &a, int lanes, bool bwd, hipStream_t st) {
    switch (lanes) {
        case 1: return launch_steps<T, 1>(a, bwd, st);
        case 2: return launch_steps<T, 2>(a, bwd, st);
        case 4: return launch_steps<T, 4>(a, bwd, st);
        case 8: return launch_steps<T, 8>(a, bwd, st);
        case 16: return launch_steps<T, 16>(a, bwd, st);
        case 32: return launch_steps<T, 32>(a, bwd, st);
        case 64: return launch_steps<T, 64>(a, bwd, st);
        default: return launch_rows<T, kWideRow, kStep>(a, bwd, st);
    }
}

int launch(const DistillArgs &a, int dtype, bool bwd, hipStream_t st) {
    const int lanes = lanes_per_row(a.V, dtype);
    switch (dtype) {
        case FSGS_F32: launch_lanes<float>(a, lanes, bwd, st); break;
        case FSGS_BF16: launch_lanes<__bf16>(a, lanes, bwd, st); break;
        default: launch_lanes<_Float16>(a, lanes, bwd, st); break;
    }
    return check_launch();
}

bool bad_args(int64_t rows, int V, int K, int dtype, int tdtype, int idx_bits, float T) {
    return rows < 0 || rows > INT32_MAX || V < 1 || V > FSGS_DISTILL_MAX_CLASSES || K < 1 || K > FSGS_DISTILL_MAX_K ||
           !known_dtype(dtype) || !known_dtype(tdtype) || (idx_bits != 32 && idx_bits != 64) || !(T >= FSGS_DISTILL_MIN_T) || !(T <= FSGS_DISTILL_MAX_T);
}

}  // namespace
}  // namespace fsgs

using namespace fsgs;

extern "C" int64_t fsgs_distill_scratch_bytes(void) { return (int64_t)kMaxBlocks * sizeof(double2); }

extern "C" int fsgs_distill_fwd(int64_t rows, int classes, int top_k, int dtype, const void *logits, int64_t pitch,
                                int idx_bits, const void *idx, int64_t idx_pitch, int teacher_dtype, const void *teacher,
                                int64_t teacher_pitch, const float *weight, float temperature, int reduction, float *loss,
                                float *stat, float *inv_weight, void *scratch, int64_t scratch_bytes, fsgs_stream_t stream) {
    if (bad_args(rows, classes, top_k, dtype, teacher_dtype, idx_bits, temperature)) return FSGS_EINVAL;
    if (reduction < FSGS_REDUCE_NONE || reduction > FSGS_REDUCE_MEAN || pitch < 0 || idx_pitch < 0 || teacher_pitch < 0)
        return FSGS_EINVAL;
    if (rows == 0 && reduction == FSGS_REDUCE_NONE) return FSGS_OK;
    if (!loss || (rows > 0 && (!logits || !idx || !teacher))) return FSGS_EINVAL;
    if (reduction != FSGS_REDUCE_NONE && (!scratch || scratch_bytes < fsgs_distill_scratch_bytes())) return FSGS_ESCRATCH;
    DistillArgs a = {};
    a.s = logits, a.sp = pitch, a.idx = idx, a.ip = idx_pitch, a.u = teacher, a.up = teacher_pitch, a.weight = weight;
    a.rows = rows, a.V = classes, a.K = top_k, a.tdtype = teacher_dtype, a.idx64 = idx_bits == 64;
    a.T = temperature, a.scale2 = (float)(1.4426950408889634 / (double)temperature);
    a.loss_scale = (float)((double)temperature * temperature * 0.69314718055994531);
    a.stat = (float4 *)stat;
    if (reduction == FSGS_REDUCE_NONE) a.row_loss = loss;
    else a.partial = (double2 *)scratch;
    hipStream_t st = as_stream(stream);
    if (rows > 0) {
        const int rc = launch(a, dtype, false, st);
        if (rc != FSGS_OK) return rc;
    }
    if (reduction == FSGS_REDUCE_NONE) return FSGS_OK;
    const int blocks = rows > 0 ? row_blocks(rows, lanes_per_row(classes, dtype)) : 0;
    distill_reduce_kernel<<<1, 256, 0, st>>>((const double2 *)scratch, blocks, reduction == FSGS_REDUCE_MEAN, loss, inv_weight);
    return check_launch();
}

extern "C" int fsgs_distill_bwd(int64_t rows, int classes, int top_k, int dtype, const void *logits, int64_t pitch,
                                int idx_bits, const void *idx, int64_t idx_pitch, int teacher_dtype, const void *teacher,
                                int64_t teacher_pitch, const float *weight, float temperature, const float *stat,
                                const float *inv_weight, const float *grad_loss, int grad_per_row, void *grad_logits,
                                fsgs_stream_t stream) {
    if (bad_args(rows, classes, top_k, dtype, teacher_dtype, idx_bits, temperature)) return FSGS_EINVAL;
    if (rows == 0) return FSGS_OK;
    if (!logits || !idx || !teacher || !stat || !grad_loss || !grad_logits || pitch < 0 || idx_pitch < 0 || teacher_pitch < 0)
        return FSGS_EINVAL;
    DistillArgs a = {};
    a.s = logits, a.sp = pitch, a.idx = idx, a.ip = idx_pitch, a.u = teacher, a.up = teacher_pitch, a.weight = weight;
    a.rows = rows, a.V = classes, a.K = top_k, a.tdtype = teacher_dtype, a.idx64 = idx_bits == 64;
    a.T = temperature, a.scale2 = (float)(1.4426950408889634 / (double)temperature);
    a.loss_scale = (float)((double)temperature * temperature * 0.69314718055994531);
    a.stat = (float4 *)const_cast<float *>(stat);
    a.g = grad_loss, a.g_per_row = grad_per_row, a.inv_w = inv_weight, a.ds = grad_logits;
    return launch(a, dtype, true, as_stream(stream));
}
