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

constexpr int kRowBlocks = 2048;  // workgroups of the row kernels: 8 per CU

struct DistillArgs {
    const void *s, *idx, *u;
    const float *weight;
    int64_t rows, sp, ip, up;
    int V, K, tdtype, idx64;
    float T, invT;
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

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

constexpr int kMaxPerLane = FSGS_DISTILL_MAX_K / kWave;

// One wave per row.
template <typename T>
__global__ __launch_bounds__(256) void distill_fwd_kernel(DistillArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double sum_l = 0.0, sum_w = 0.0;
    for (int64_t row = (int64_t)blockIdx.x * 4 + wave; row < a.rows; row += (int64_t)gridDim.x * 4) {
        const T *s = (const T *)a.s + row * a.sp;
        float m = -INFINITY;
        for (int j = lane; j < a.V; j += 64) m = fmaxf(m, (float)s[j]);
        m = wave_max(m);
        float sum = 0.f;
        for (int j = lane; j < a.V; j += 64) sum += expf(((float)s[j] - m) * a.invT);
        sum = wave_add(sum);
        const float log_sum = logf(sum);

        int cls[kMaxPerLane];
        float u[kMaxPerLane];
        float um = -INFINITY;
        bool any = false;
#pragma unroll
        for (int i = 0; i < kMaxPerLane; ++i) {
            const int k = i * 64 + lane;
            cls[i] = k < a.K ? class_at(a.idx, row * a.ip + k, a.idx64, a.V) : -1;
            u[i] = cls[i] >= 0 ? teacher_at(a.u, row * a.up + k, a.tdtype) : -INFINITY;
            um = fmaxf(um, u[i]);
            any |= u[i] != -INFINITY;  // (NaN counts: it reaches the loss)
        }
        um = wave_max(um);
        const float w = a.weight ? a.weight[row] : 1.f;
        const bool alive = __any(any) && w != 0.f;
        float z = 0.f, loss = 0.f;
#pragma unroll
        for (int i = 0; i < kMaxPerLane; ++i)
            if (cls[i] >= 0) z += expf((u[i] - um) * a.invT);
        z = wave_add(z);
        const float inv_z = 1.f / z, log_z = logf(z);
#pragma unroll
        for (int i = 0; i < kMaxPerLane; ++i)
            if (cls[i] >= 0) {
                const float lu = (u[i] - um) * a.invT, p = expf(lu) * inv_z;
                const float lq = ((float)s[cls[i]] - m) * a.invT - log_sum;
                if (p != 0.f) loss += p * (lu - log_z - lq);
            }
        loss = wave_add(loss) * a.T * a.T;
        if (lane == 0) {
            const float wl = alive ? w * loss : 0.f;
            if (a.row_loss) a.row_loss[row] = wl;
            if (a.stat) a.stat[row] = make_float4(m, 1.f / sum, um, alive ? inv_z : 0.f);
            if (alive) sum_l += (double)wl, sum_w += (double)w;
        }
    }
    if (a.partial) {
        __shared__ double2 part[4];
        if (lane == 0) part[wave] = make_double2(sum_l, sum_w);
        __syncthreads();
        if (threadIdx.x == 0) {
            double2 t = part[0];
            for (int i = 1; i < 4; ++i) t.x += part[i].x, t.y += part[i].y;
            a.partial[blockIdx.x] = t;
        }
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

// One wave per row: q for every class, then the teacher's classes once more with their mass taken off.
template <typename T>
__global__ __launch_bounds__(256) void distill_bwd_kernel(DistillArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t row = (int64_t)blockIdx.x * 4 + wave; row < a.rows; row += (int64_t)gridDim.x * 4) {
        const T *s = (const T *)a.s + row * a.sp;
        T *ds = (T *)a.ds + row * a.V;
        const float4 st = a.stat[row];
        if (st.w == 0.f) {
            for (int j = lane; j < a.V; j += 64) ds[j] = (T)0.f;
            continue;
        }
        const float coef = a.T * (a.weight ? a.weight[row] : 1.f) * a.g[a.g_per_row ? row : 0] * (a.inv_w ? *a.inv_w : 1.f);
        for (int j = lane; j < a.V; j += 64) ds[j] = (T)(coef * (expf(((float)s[j] - st.x) * a.invT) * st.y));
        // the same class may stand in several entries: its first entry carries the sum
        int cls[kMaxPerLane];
        float p[kMaxPerLane];
#pragma unroll
        for (int i = 0; i < kMaxPerLane; ++i) {
            const int k = i * 64 + lane;
            cls[i] = k < a.K ? class_at(a.idx, row * a.ip + k, a.idx64, a.V) : -1;
            p[i] = cls[i] >= 0 ? expf((teacher_at(a.u, row * a.up + k, a.tdtype) - st.z) * a.invT) * st.w : 0.f;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __builtin_amdgcn_s_waitcnt(0);  // the q stores have landed before any lane writes over them
#pragma unroll
        for (int i = 0; i < kMaxPerLane; ++i) {
            float mass = 0.f;
            bool first = cls[i] >= 0;
#pragma unroll
            for (int t = 0; t < kMaxPerLane; ++t)
                if (t * 64 < a.K)
                    for (int l = 0; l < 64; ++l) {
                        const int oc = __shfl(cls[t], l);
                        const float op = __shfl(p[t], l);
                        const bool same = oc == cls[i];
                        if (same) mass += op;
                        if (same && t * 64 + l < i * 64 + lane) first = false;
                    }
            if (first) ds[cls[i]] = (T)(coef * (expf(((float)s[cls[i]] - st.x) * a.invT) * st.y - mass));
        }
    }
}

int row_blocks(int64_t rows) {
    const int64_t b = (rows + 3) / 4;
    return (int)(b < kRowBlocks ? b : kRowBlocks);
}

bool bad_args(int64_t rows, int V, int K, int dtype, int tdtype, int idx_bits, float T) {
    return rows < 0 || rows > INT32_MAX || V < 1 || K < 1 || K > FSGS_DISTILL_MAX_K || !known_dtype(dtype) || !known_dtype(tdtype) ||
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
    a.T = temperature, a.invT = 1.f / temperature;
    a.stat = (float4 *)stat;
    if (reduction == FSGS_REDUCE_NONE) a.row_loss = loss;
    else a.partial = (double2 *)scratch;
    const int blocks = row_blocks(rows);
    hipStream_t st = as_stream(stream);
    if (rows > 0) {
        switch (dtype) {
            case FSGS_F32: distill_fwd_kernel<float><<<blocks, 256, 0, st>>>(a); break;
            case FSGS_BF16: distill_fwd_kernel<__bf16><<<blocks, 256, 0, st>>>(a); break;
            default: distill_fwd_kernel<_Float16><<<blocks, 256, 0, st>>>(a); break;
        }
        const int rc = check_launch();
        if (rc != FSGS_OK) return rc;
    }
    if (reduction == FSGS_REDUCE_NONE) return FSGS_OK;
    distill_reduce_kernel<<<1, 256, 0, st>>>((const double2 *)scratch, rows > 0 ? blocks : 0, reduction == FSGS_REDUCE_MEAN,
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
    a.T = temperature, a.invT = 1.f / temperature;
    a.stat = (float4 *)const_cast<float *>(stat);
    a.g = grad_loss, a.g_per_row = grad_per_row, a.inv_w = inv_weight, a.ds = grad_logits;
    hipStream_t st = as_stream(stream);
    const int blocks = row_blocks(rows);
    switch (dtype) {
        case FSGS_F32: distill_bwd_kernel<float><<<blocks, 256, 0, st>>>(a); break;
        case FSGS_BF16: distill_bwd_kernel<__bf16><<<blocks, 256, 0, st>>>(a); break;
        default: distill_bwd_kernel<_Float16><<<blocks, 256, 0, st>>>(a); break;
    }
    return check_launch();
}
