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

constexpr int kRowBlocks = 2048;   // workgroups of the row kernels: 8 per CU, the rows go round them
constexpr int kWideRow = 256;      // lanes of a row that has a workgroup to itself

struct DistillArgs {
    const void *s, *idx, *u;
    const float *weight;
    int64_t rows, sp, ip, up;
    int V, K, tdtype, idx64;
    float T, invT, scale2;  // scale2 = log2(e) / T
    float *row_loss;      // fwd, reduction none: [rows]
    float4 *stat;         // [rows] max s, 1 / sum_j exp, max u, 1 / sum_k exp (0: the row counts for nothing)
    double2 *partial;     // [kRowBlocks] sum of w L, sum of w
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
__device__ __forceinline__ float row_reduce(float v) {
    if constexpr (L >= 2) v = Op::f(v, dpp_f<0xB1>(v));    // quad_perm [1,0,3,2]
    if constexpr (L >= 4) v = Op::f(v, dpp_f<0x4E>(v));    // quad_perm [2,3,0,1]
    if constexpr (L >= 8) v = Op::f(v, dpp_f<0x141>(v));   // row_half_mirror
    if constexpr (L >= 16) v = Op::f(v, dpp_f<0x140>(v));  // row_mirror
    if constexpr (L >= 32) v = Op::f(v, __shfl_xor(v, 16));
    if constexpr (L >= 64) v = Op::f(v, __shfl_xor(v, 32));
    if constexpr (L == kWideRow) {
        __shared__ float part[4];
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = Op::f(Op::f(part[0], part[1]), Op::f(part[2], part[3]));
    }
    return v;
}
template <int L>
__device__ __forceinline__ bool row_any(bool b) {
    if constexpr (L == kWideRow) return __syncthreads_or(b);
    const uint64_t m = __ballot(b);
    if constexpr (L == 64) return m != 0;
    const int first = (threadIdx.x & 63) & ~(L - 1);
    return (m >> first) & ((1ull << (L & 63)) - 1);
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// exp of a score against a maximum of -inf (no finite score) must not turn -inf - -inf into NaN
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

template <typename T>
__device__ __forceinline__ void unpack(const Chunk &c, float *v) {
    T t[kChunk<T>];
    __builtin_memcpy(t, &c, sizeof(Chunk));
#pragma unroll
    for (int e = 0; e < kChunk<T>; ++e) v[e] = (float)t[e];
}

// A row is read in chunks of 16 bytes, chunk c by lane c mod L, kStep chunks per lane at a time (all of a row that has at most
// kStep * L chunks: lanes_per_row).  Rows start at any element.  The last chunk of a row that does not end on one is read
// shifted back to end with the row, its doubled elements masked: no element-wise reads, nothing behind the row.
constexpr int kStep = 5;
constexpr int kHeld = 4;  // entries per lane kept in registers; further ones are read again where they are needed

template <typename T, int L>
__device__ __forceinline__ void load_step(Chunk (&c)[kStep], const T *s, int c0, int V) {
    constexpr int CE = kChunk<T>;
#pragma unroll
    for (int i = 0; i < kStep; ++i) {
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

template <typename T, int L>
__global__ __launch_bounds__(256) void distill_fwd_kernel(DistillArgs a) {
    constexpr int CE = kChunk<T>, ROWS = 256 / L;
    const int sub = threadIdx.x & (L - 1);
    const int chunks = (a.V + CE - 1) / CE;
    double sum_l = 0.0, sum_w = 0.0;
    for (int64_t base = (int64_t)blockIdx.x * ROWS; base < a.rows; base += (int64_t)gridDim.x * ROWS) {
        const int64_t slot = base + threadIdx.x / L;
        const bool here = slot < a.rows;
        const int64_t row = here ? slot : a.rows - 1;  // (lanes behind the last row repeat it and store nothing)
        const T *s = (const T *)a.s + row * a.sp;
        Chunk c[kStep];
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

        // maximum and sum of the row: held whole, or step by step with the sum rescaled to each step's maximum
        float m = -INFINITY, sum = 0.f;
        for (int c0 = sub;;) {
            float mn = m;
#pragma unroll
            for (int i = 0; i < kStep; ++i) {
                float v[CE];
                mask_chunk<T>(c[i], (c0 + i * L) * CE, a.V);
                unpack<T>(c[i], v);
#pragma unroll
                for (int e = 0; e < CE; ++e) mn = fmaxf(mn, v[e]);
            }
            const float mf = finite_max(mn);
            sum *= exp2_hw((m - mf) * a.scale2);
            m = mn;
#pragma unroll
            for (int i = 0; i < kStep; ++i) {
                float v[CE];
                if constexpr (sizeof(T) == 2) forget(c[i]);
                unpack<T>(c[i], v);
#pragma unroll
                for (int e = 0; e < CE; ++e) sum += exp2_hw((v[e] - mf) * a.scale2);
            }
            if constexpr (L != kWideRow) break;
            c0 += kStep * L;
            if (c0 - sub >= chunks) break;
            load_step<T, L>(c, s, c0, a.V);
        }
        const float lane_m = m;
        m = row_reduce<L, MaxOp>(m);
        sum = row_reduce<L, AddOp>(sum * exp2_hw((lane_m - finite_max(m)) * a.scale2));
        // (a row of -inf only: sum 0, and the -inf - -inf below are the NaN that its softmax is)

        float um = -INFINITY;
        bool any = false;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            um = fmaxf(um, u[i]);
            any |= u[i] != -INFINITY;  // (NaN counts: it reaches the loss)
        }
        for (int k = kHeld * L + sub; k < a.K; k += L)
            if (class_at(a.idx, row * a.ip + k, a.idx64, a.V) >= 0) {
                const float uk = teacher_at(a.u, row * a.up + k, a.tdtype);
                um = fmaxf(um, uk);
                any |= uk != -INFINITY;
            }
        um = row_reduce<L, MaxOp>(um);
        const bool alive = row_any<L>(any) && w != 0.f;
        // sum_k p_k (log p_k - log q_k) = (sum_k e_k x_k) / Z - log Z + log S with e_k = exp((u_k - um) / T), Z their sum,
        // x_k = (u_k - um) / T - (s_k - m) / T
        float z = 0.f, ex = 0.f;
        auto entry = [&](float uk, float sk) {
            const float lu = uk - um, e = exp2_hw(lu * a.scale2);
            z += e;
            if (e != 0.f) ex += e * ((lu - (sk - m)) * a.invT);
        };
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (i * L < a.K && cls[i] >= 0) entry(u[i], sv[i]);
        for (int k = kHeld * L + sub; k < a.K; k += L) {
            const int ck = class_at(a.idx, row * a.ip + k, a.idx64, a.V);
            if (ck >= 0) entry(teacher_at(a.u, row * a.up + k, a.tdtype), (float)s[ck]);
        }
        z = row_reduce<L, AddOp>(z);
        ex = row_reduce<L, AddOp>(ex);
        if (sub == 0 && here) {
            const float inv_z = 1.f / z;
            const float loss = (ex * inv_z + (logf(sum) - logf(z))) * (a.T * a.T);
            const float wl = alive ? w * loss : 0.f;
            if (a.row_loss) a.row_loss[row] = wl;
            if (a.stat) a.stat[row] = make_float4(m, 1.f / sum, um, alive ? inv_z : 0.f);
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

// loss = sum w L (/ sum w); inv_w is what the gradient is scaled by.  All weights zero: loss 0, no gradient.
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

// q for every class, then the teacher's classes once more with their mass taken off.  A class may stand in several entries:
// its first entry carries their sum, taken in the entries' order.  Whether a row has such a class at all is found with one bit
// per class in LDS; only then are its entries compared pair by pair.
template <typename T, int L>
__global__ __launch_bounds__(256) void distill_bwd_kernel(DistillArgs a) {
    constexpr int CE = kChunk<T>, ROWS = 256 / L;
    extern __shared__ uint32_t seen[];  // [ROWS][words]
    const int sub = threadIdx.x & (L - 1), group = threadIdx.x / L;
    const int chunks = (a.V + CE - 1) / CE, words = (a.V + 31) / 32;
    uint32_t *bits = seen + group * words;
    const float up = a.g_per_row ? 0.f : a.g[0];
    const float inv_w = a.inv_w ? *a.inv_w : 1.f;
    for (int64_t base = (int64_t)blockIdx.x * ROWS; base < a.rows; base += (int64_t)gridDim.x * ROWS) {
        const int64_t slot = base + group;
        const bool here = slot < a.rows;
        const int64_t row = here ? slot : a.rows - 1;
        const T *s = (const T *)a.s + row * a.sp;
        T *ds = (T *)a.ds + row * a.V;
        Chunk c[kStep];
        load_step<T, L>(c, s, sub, a.V);
        const float4 st = a.stat[row];
        const float m = st.x, um = st.z;
        const bool dead = st.w == 0.f;
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
            u[i] = sv[i] = 0.f;
            if (i * L < a.K && cls[i] >= 0) {
                u[i] = teacher_at(a.u, row * a.up + i * L + sub, a.tdtype);
                sv[i] = (float)s[cls[i]];
                bits[cls[i] >> 5] = 0;
            }
        }
        for (int k = kHeld * L + sub; k < a.K; k += L) {
            const int ck = class_at(a.idx, row * a.ip + k, a.idx64, a.V);
            if (ck >= 0) bits[ck >> 5] = 0;
        }
        const float coef = a.T * (a.weight ? a.weight[row] : 1.f) * (a.g_per_row ? a.g[row] : up) * inv_w;
        const float cq = coef * st.y;
        for (int c0 = sub;;) {
#pragma unroll
            for (int i = 0; i < kStep; ++i) {
                const int j = (c0 + i * L) * CE;
                if (j >= a.V || !here) break;
                float v[CE];
                unpack<T>(c[i], v);
                T out[CE];
#pragma unroll
                for (int e = 0; e < CE; ++e) out[e] = (T)(dead ? 0.f : cq * exp2_hw((v[e] - m) * a.scale2));
                if (a.V < CE) {
#pragma unroll
                    for (int e = 0; e < CE; ++e)
                        if (e < a.V) ds[e] = out[e];
                } else {
                    // (the last chunk of a row stores the elements before it a second time, with the same values)
                    __builtin_memcpy(ds + min(j, a.V - CE), out, sizeof(Chunk));
                }
            }
            if constexpr (L != kWideRow) break;
            c0 += kStep * L;
            if (c0 - sub >= chunks) break;
            load_step<T, L>(c, s, c0, a.V);
        }
        if constexpr (L == kWideRow) __syncthreads();
        bool again = false;
        auto mark = [&](int ck) { again |= (atomicOr(&bits[ck >> 5], 1u << (ck & 31)) >> (ck & 31)) & 1u; };
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (i * L < a.K && cls[i] >= 0) mark(cls[i]);
        for (int k = kHeld * L + sub; k < a.K; k += L) {
            const int ck = class_at(a.idx, row * a.ip + k, a.idx64, a.V);
            if (ck >= 0) mark(ck);
        }
        again = row_any<L>(again);
        // every store above has landed before a lane writes over one of them
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if constexpr (L == kWideRow) __syncthreads();
        auto fix = [&](int k, int ck, float uk, float sk) {
            float mass = exp2_hw((uk - um) * a.scale2);
            if (again) {
                mass = 0.f;
                bool first = true;
                for (int t = 0; t < a.K; ++t)
                    if (class_at(a.idx, row * a.ip + t, a.idx64, a.V) == ck) {
                        mass += exp2_hw((teacher_at(a.u, row * a.up + t, a.tdtype) - um) * a.scale2);
                        first &= t >= k;
                    }
                if (!first) return;
            }
            ds[ck] = (T)(coef * (exp2_hw((sk - m) * a.scale2) * st.y - mass * st.w));
        };
        if (here && !dead) {
#pragma unroll
            for (int i = 0; i < kHeld; ++i)
                if (i * L < a.K && cls[i] >= 0) fix(i * L + sub, cls[i], u[i], sv[i]);
            for (int k = kHeld * L + sub; k < a.K; k += L) {
                const int ck = class_at(a.idx, row * a.ip + k, a.idx64, a.V);
                if (ck >= 0) fix(k, ck, teacher_at(a.u, row * a.up + k, a.tdtype), (float)s[ck]);
            }
        }
        if constexpr (L == kWideRow) __syncthreads();
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
    const int64_t per = 256 / lanes, b = (rows + per - 1) / per;
    return (int)(b < kRowBlocks ? b : kRowBlocks);
}

template <typename T, int L>
void launch_rows(const DistillArgs &a, bool bwd, hipStream_t st) {
    const int blocks = row_blocks(a.rows, L);
    if (bwd) distill_bwd_kernel<T, L><<<blocks, 256, (256 / L) * (size_t)((a.V + 31) / 32) * 4, st>>>(a);
    else distill_fwd_kernel<T, L><<<blocks, 256, 0, st>>>(a);
}

template <typename T>
void launch_lanes(const DistillArgs &a, int lanes, bool bwd, hipStream_t st) {
    switch (lanes) {
        case 1: return launch_rows<T, 1>(a, bwd, st);
        case 2: return launch_rows<T, 2>(a, bwd, st);
        case 4: return launch_rows<T, 4>(a, bwd, st);
        case 8: return launch_rows<T, 8>(a, bwd, st);
        case 16: return launch_rows<T, 16>(a, bwd, st);
        case 32: return launch_rows<T, 32>(a, bwd, st);
        case 64: return launch_rows<T, 64>(a, bwd, st);
        default: return launch_rows<T, kWideRow>(a, bwd, st);
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
    return rows < 0 || rows > INT32_MAX || V < 1 || V > FSGS_DISTILL_MAX_CLASSES || K < 1 || K > FSGS_DISTILL_MAX_K || !known_dtype(dtype) || !known_dtype(tdtype) ||
           (idx_bits != 32 && idx_bits != 64) || !(T >= FSGS_DISTILL_MIN_T) || !(T <= FSGS_DISTILL_MAX_T);
}

}  // namespace
}  // namespace fsgs

using namespace fsgs;

extern "C" int64_t fsgs_distill_scratch_bytes(void) { return (int64_t)kRowBlocks * sizeof(double2); }

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
    a.T = temperature, a.invT = 1.f / temperature, a.scale2 = (float)(1.4426950408889634 / (double)temperature);
    a.stat = (float4 *)stat;
    if (reduction == FSGS_REDUCE_NONE) a.row_loss = loss;
    else a.partial = (double2 *)scratch;
    hipStream_t st = as_stream(stream);
    if (rows > 0) {
        const int rc = launch(a, dtype, false, st);
        if (rc != FSGS_OK) return rc;
    }
    if (reduction == FSGS_REDUCE_NONE) return FSGS_OK;
    distill_reduce_kernel<<<1, 256, 0, st>>>((const double2 *)scratch, rows > 0 ? row_blocks(rows, lanes_per_row(classes, dtype)) : 0, reduction == FSGS_REDUCE_MEAN,
                                             loss, inv_weight);
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
    a.T = temperature, a.invT = 1.f / temperature, a.scale2 = (float)(1.4426950408889634 / (double)temperature);
    a.stat = (float4 *)const_cast<float *>(stat);
    a.g = grad_loss, a.g_per_row = grad_per_row, a.inv_w = inv_weight, a.ds = grad_logits;
    return launch(a, dtype, true, as_stream(stream));
}
