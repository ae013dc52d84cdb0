// Label fields' losses and answers over logits [rows, labels]:
//
//   x_v = z_v / T,  p = softmax(x) = e^{x_v - m} / S,  m = max x,  S = sum e^{x_v - m}
//
// distillation from a teacher's best few logits t_k at labels j_k
// (q = softmax of t / T over a row's valid entries):
//   loss = u T^2 sum_k q_k (log q_k - log p_{j_k})
//   dz_v = g u T (p_v - sum_{k : j_k = v} q_k)
// log probability of a label y, the entropy and the best labels:
//   lp = log p_y,  H = log S - (1/S) sum (x_v - m) e^{x_v - m}
//   dz_v = (1/T) (g_lp (1_{v = y} - p_v) - g_H p_v (log p_v + H))
//
// All statistics and sums are fp32 whatever the logits' type; gradients are
// rounded to it once.  A logit of -inf is a label masked out; a row of nothing
// else has no distribution, and no loss, no entropy and no gradient.
#include "label_device.h"

using namespace sdfoam_hip;
using namespace sdfoam_hip::label;

namespace {

constexpr uint32_t kMaxTeacher = 1024; // teacher's entries a row
constexpr uint32_t kMaxTop = 64;       // best labels returned a row
constexpr float kLog2e = 1.44269504088896341f;

__device__ __forceinline__ float block_max(float x, float *shared) {
    x = wave_max(x);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) shared[threadIdx.x >> 6] = x;
    __syncthreads();
    for (uint32_t k = 0; k < blockDim.x / 64u; ++k) x = fmaxf(x, shared[k]);
    return x;
}
__device__ __forceinline__ float block_sum(float x, float *shared) {
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) shared[threadIdx.x >> 6] = x;
    __syncthreads();
    float s = 0.0f;
    for (uint32_t k = 0; k < blockDim.x / 64u; ++k) s += shared[k];
    return s;
}

// The largest logit of a row (0 for a row of nothing but -inf, so that
// differences from it stay defined) and S.  NaN reaches S.
struct RowStats {
    float m, s;
};

template <typename T>
__device__ RowStats row_stats(const T *z, uint32_t labels, float c, float *shared) {
    float m = -INFINITY;
    for (uint32_t v = threadIdx.x; v < labels; v += blockDim.x) m = fmaxf(m, (float)z[v]);
    m = block_max(m, shared);
    if (m == -INFINITY) m = 0.0f;
    float s = 0.0f;
    for (uint32_t v = threadIdx.x; v < labels; v += blockDim.x)
        s += __builtin_amdgcn_exp2f(((float)z[v] - m) * c);
    return {m, block_sum(s, shared)};
}

struct DistillArgs {
    const void *logits;
    uint64_t stride; // elements from row to row
    uint32_t labels;
    int id_type;
    const void *teacher_labels;
    int teacher_type;
    const void *teacher_logits;
    uint32_t top;
    float temperature;
    const float *row_weight;   // NULL: 1
    const float *loss_grad;    // NULL: 1
    uint32_t loss_grad_stride; // 0: one for all rows
    float reduce;              // what a row's loss counts in the result
    float *loss;               // [rows]; NULL: not written
    float2 *stats;             // [rows] {m, S}; read where `have_stats`, else written unless NULL
    void *logits_grad;         // [rows, labels]; NULL: not written
};

__device__ __forceinline__ float teacher_logit(const DistillArgs &a, uint64_t i) {
    if (a.teacher_type == SDF_TYPE_F16) return (float)static_cast<const half_t *>(a.teacher_logits)[i];
    if (a.teacher_type == SDF_TYPE_BF16) return (float)static_cast<const bf16_t *>(a.teacher_logits)[i];
    return static_cast<const float *>(a.teacher_logits)[i];
}

template <typename T, bool have_stats>
__global__ __launch_bounds__(256) void distill_kernel(DistillArgs a) {
    __shared__ float shared[4];
    __shared__ float q[kMaxTeacher];
    __shared__ int32_t id[kMaxTeacher];
    const uint64_t r = blockIdx.x;
    const T *z = static_cast<const T *>(a.logits) + r * a.stride;
    T *dz = a.logits_grad ? static_cast<T *>(a.logits_grad) + r * a.labels : nullptr;
    const float inv_t = 1.0f / a.temperature, c = inv_t * kLog2e;
    const float u = a.row_weight ? a.row_weight[r] : 1.0f;

    float tm = -INFINITY;
    for (uint32_t k = threadIdx.x; k < a.top; k += 256u) {
        const int32_t j = load_id(a.teacher_labels, a.id_type, r * a.top + k, a.labels);
        const float t = j < 0 ? -INFINITY : teacher_logit(a, r * a.top + k);
        id[k] = t == -INFINITY ? -1 : j;
        q[k] = t;
        tm = fmaxf(tm, t);
    }
    tm = block_max(tm, shared);
    if (tm == -INFINITY) tm = 0.0f;
    float ts = 0.0f;
    for (uint32_t k = threadIdx.x; k < a.top; k += 256u)
        ts += __builtin_amdgcn_exp2f((q[k] - tm) * c);
    ts = block_sum(ts, shared);

    RowStats st = {0.0f, 0.0f};
    const bool counts = !(u == 0.0f) && !(ts == 0.0f);
    if (counts) {
        if (have_stats) {
            const float2 h = a.stats[r];
            st = {h.x, h.y};
        } else {
            st = row_stats(z, a.labels, c, shared);
        }
    }
    const bool live = counts && !(st.s == 0.0f);
    if (!have_stats && a.stats && threadIdx.x == 0) a.stats[r] = make_float2(st.m, st.s);
    if (!live) {
        if (threadIdx.x == 0 && a.loss) a.loss[r] = 0.0f;
        if (dz)
            for (uint32_t v = threadIdx.x; v < a.labels; v += 256u) dz[v] = (T)0.0f;
        return;
    }

    float sum = 0.0f;
    const float log_s = logf(st.s), log_ts = logf(ts);
    for (uint32_t k = threadIdx.x; k < a.top; k += 256u) {
        const float d = (q[k] - tm) * inv_t;
        const float qk = __builtin_amdgcn_exp2f((q[k] - tm) * c) / ts;
        // an entry of no mass adds nothing, whatever its label's probability
        if (a.loss && !(qk == 0.0f))
            sum += qk * (d - log_ts - (((float)z[id[k]] - st.m) * inv_t - log_s));
        q[k] = qk;
    }
    if (a.loss) {
        sum = block_sum(sum, shared);
        if (threadIdx.x == 0) a.loss[r] = u * a.temperature * a.temperature * sum;
    }
    if (!dz) return;
    const float g = a.loss_grad ? a.loss_grad[r * a.loss_grad_stride] : 1.0f;
    const float coef = g * a.reduce * u * a.temperature, share = coef / st.s;
    for (uint32_t v = threadIdx.x; v < a.labels; v += 256u)
        dz[v] = (T)(share * __builtin_amdgcn_exp2f(((float)z[v] - st.m) * c));
    __syncthreads(); // the teacher's labels are written over what stands there
    for (uint32_t k = threadIdx.x; k < a.top; k += 256u) {
        const int32_t j = id[k];
        if (j < 0) continue;
        float mass = 0.0f; // a label that the teacher names twice has both shares
        for (uint32_t o = 0; o < a.top; ++o) mass += id[o] == j ? q[o] : 0.0f;
        const float p = __builtin_amdgcn_exp2f(((float)z[j] - st.m) * c) / st.s;
        dz[j] = (T)(coef * (p - mass));
    }
}

// The rows' losses in one sum, always in the same order.
__global__ __launch_bounds__(1024) void loss_sum_kernel(const float *__restrict__ loss,
                                                        uint64_t rows, float scale,
                                                        float *__restrict__ out) {
    __shared__ double part[16];
    double s = 0.0;
    for (uint64_t r = threadIdx.x; r < rows; r += 1024u) s += (double)loss[r];
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63u) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x != 0) return;
    s = 0.0;
    for (int k = 0; k < 16; ++k) s += part[k];
    *out = (float)(s * (double)scale);
}

struct AnswerArgs {
    const void *logits;
    uint64_t stride;
    uint32_t labels;
    int id_type;
    const void *label_ids;
    uint32_t top;
    float temperature;
    float *log_prob, *entropy; // [rows]
    float *top_log_probs;      // [rows, top]
    int64_t *top_labels;       // [rows, top]
    float2 *stats;             // [rows] {m, S}; NULL: not written
    const float *log_prob_grad, *entropy_grad; // backward, either may be NULL
    void *logits_grad;
};

// A whole number that orders logits as their values do (-0 and 0 alike), 0
// for -inf and NaN, which are never among the best.
__device__ __forceinline__ uint32_t logit_order(float z) {
    if (!(z > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(z + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename T> __global__ __launch_bounds__(256) void answer_kernel(AnswerArgs a) {
    __shared__ float shared[4];
    __shared__ uint64_t best[4];
    const uint64_t r = blockIdx.x;
    const T *z = static_cast<const T *>(a.logits) + r * a.stride;
    const float inv_t = 1.0f / a.temperature, c = inv_t * kLog2e;
    const RowStats st = row_stats(z, a.labels, c, shared);
    float w = 0.0f;
    for (uint32_t v = threadIdx.x; v < a.labels; v += 256u) {
        const float d = ((float)z[v] - st.m) * c;
        // fmaxf: 0, not NaN, where the exponential has underflowed
        w += fmaxf(d, -200.0f) * __builtin_amdgcn_exp2f(d);
    }
    w = block_sum(w, shared);
    const float log_s = logf(st.s);
    const bool empty = st.s == 0.0f;
    if (threadIdx.x == 0) {
        const int32_t y = load_id(a.label_ids, a.id_type, r, a.labels);
        float lp = 0.0f;
        if (y >= 0) lp = empty ? -INFINITY : ((float)z[y] - st.m) * inv_t - log_s;
        a.log_prob[r] = lp;
        a.entropy[r] = empty ? 0.0f : log_s - w / (st.s * kLog2e);
        if (a.stats) a.stats[r] = make_float2(st.m, st.s);
    }
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < a.top; ++k) {
        uint64_t key = 0;
        for (uint32_t v = threadIdx.x; v < a.labels; v += 256u) {
            const uint64_t o = logit_order((float)z[v]);
            const uint64_t x = o << 32 | (0xffffffffu - v);
            if (o != 0 && x < last && x > key) key = x;
        }
        for (int d = 32; d > 0; d >>= 1) {
            const uint64_t o = __shfl_xor((unsigned long long)key, d);
            key = o > key ? o : key;
        }
        __syncthreads();
        if ((threadIdx.x & 63u) == 0) best[threadIdx.x >> 6] = key;
        __syncthreads();
        for (int i = 0; i < 4; ++i) key = best[i] > key ? best[i] : key;
        if (threadIdx.x == 0) {
            const uint32_t v = 0xffffffffu - (uint32_t)key;
            a.top_labels[r * a.top + k] = key ? (int64_t)v : -1;
            a.top_log_probs[r * a.top + k] = key ? ((float)z[v] - st.m) * inv_t - log_s : -INFINITY;
        }
        last = key;
    }
}

template <typename T> __global__ __launch_bounds__(256) void answer_grad_kernel(AnswerArgs a) {
    const uint64_t r = blockIdx.x;
    const T *z = static_cast<const T *>(a.logits) + r * a.stride;
    T *dz = static_cast<T *>(a.logits_grad) + r * a.labels;
    const float inv_t = 1.0f / a.temperature, c = inv_t * kLog2e;
    const float2 st = a.stats[r];
    const int32_t y = load_id(a.label_ids, a.id_type, r, a.labels);
    const float glp = a.log_prob_grad && y >= 0 ? a.log_prob_grad[r] : 0.0f;
    const float gh = a.entropy_grad ? a.entropy_grad[r] : 0.0f;
    const float log_s = logf(st.y), h = a.entropy[r];
    for (uint32_t v = threadIdx.x; v < a.labels; v += 256u) {
        float o = 0.0f;
        if (!(st.y == 0.0f)) {
            const float d = ((float)z[v] - st.x) * c;
            const float p = __builtin_amdgcn_exp2f(d) / st.y;
            const float log_p = fmaxf(d, -200.0f) / kLog2e - log_s;
            o = -p * (glp + gh * (log_p + h));
            if ((int32_t)v == y) o += glp;
        }
        dz[v] = (T)(o * inv_t);
    }
}

int check_logits(const char *what, int type, const void *logits, uint64_t rows, uint64_t labels,
                 uint64_t stride, int id_type, float temperature) {
    if (!known_type(type)) return fail(SDF_E_INVALID, "%s: unknown element type %d", what, type);
    if (!known_id_type(id_type)) return fail(SDF_E_INVALID, "%s: unknown id type %d", what, id_type);
    if (labels == 0 || labels >= (1ull << 31))
        return fail(SDF_E_INVALID, "%s takes 1 to 2^31 - 1 labels", what);
    if (rows >= (1ull << 31)) return fail(SDF_E_INVALID, "%s takes fewer than 2^31 rows", what);
    if (!(temperature > 0.0f) || temperature > 3.0e38f)
        return fail(SDF_E_INVALID, "%s: temperature must be positive and finite", what);
    if (rows > 0 && !logits) return fail(SDF_E_INVALID, "NULL pointer argument");
    (void)stride;
    if ((reinterpret_cast<uintptr_t>(logits) & (type_bytes(type) - 1)) != 0)
        return fail(SDF_E_INVALID, "%s: logits must be aligned to their elements", what);
    return SDF_OK;
}

int check_distill(const char *what, int type, const void *logits, uint64_t rows, uint64_t labels,
                  uint64_t stride, int id_type, const void *teacher_labels, int teacher_type,
                  const void *teacher_logits, uint32_t top, float temperature, int reduction) {
    const int rc = check_logits(what, type, logits, rows, labels, stride, id_type, temperature);
    if (rc != SDF_OK) return rc;
    if (!known_type(teacher_type))
        return fail(SDF_E_INVALID, "%s: unknown element type %d", what, teacher_type);
    if (top > kMaxTeacher)
        return fail(SDF_E_INVALID, "%s takes at most %u teacher logits a row", what, kMaxTeacher);
    if (rows > 0 && top > 0 && (!teacher_labels || !teacher_logits))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    if (reduction < SDF_REDUCE_NONE || reduction > SDF_REDUCE_MEAN)
        return fail(SDF_E_INVALID, "%s: unknown reduction %d", what, reduction);
    return SDF_OK;
}

} // namespace

extern "C" {

size_t sdf_distill_scratch_bytes(uint64_t rows, uint64_t labels) {
    (void)labels;
    return 4 * rows + 256;
}

int sdf_distill(int type, const void *logits, uint64_t rows, uint64_t labels, uint64_t stride,
                int id_type, const void *teacher_labels, int teacher_type,
                const void *teacher_logits, uint32_t top, float temperature,
                const float *row_weight, int reduction, const float *loss_grad, float *loss,
                float *stats, void *logits_grad, void *scratch, size_t scratch_bytes,
                void *stream) {
    const int rc = check_distill("distill", type, logits, rows, labels, stride, id_type,
                                 teacher_labels, teacher_type, teacher_logits, top, temperature,
                                 reduction);
    if (rc != SDF_OK) return rc;
    if (!loss && (rows > 0 || reduction != SDF_REDUCE_NONE))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    const size_t need = sdf_distill_scratch_bytes(rows, labels);
    if (!scratch || scratch_bytes < need)
        return fail(SDF_E_INVALID, "scratch must hold %zu bytes (got %zu)", need, scratch_bytes);
    if ((reinterpret_cast<uintptr_t>(scratch) & 255u) != 0)
        return fail(SDF_E_INVALID, "scratch must be 256-byte aligned");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool none = reduction == SDF_REDUCE_NONE;
    const float reduce = reduction == SDF_REDUCE_MEAN ? (float)(1.0 / (double)rows) : 1.0f;
    DistillArgs a = {logits, stride, (uint32_t)labels, id_type, teacher_labels, teacher_type,
                     teacher_logits, top, temperature, row_weight, loss_grad, none ? 1u : 0u,
                     reduce, none ? loss : static_cast<float *>(scratch),
                     reinterpret_cast<float2 *>(stats), logits_grad};
    if (rows > 0)
        with_type(type, [&](auto t) {
            hipLaunchKernelGGL((distill_kernel<decltype(t), false>), dim3((unsigned)rows), dim3(256),
                               0, s, a);
        });
    if (!none)
        hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, s, a.loss, rows, reduce, loss);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SDF_OK : hip_fail(e, "distill");
}

int sdf_distill_backward(int type, const void *logits, uint64_t rows, uint64_t labels,
                         uint64_t stride, int id_type, const void *teacher_labels,
                         int teacher_type, const void *teacher_logits, uint32_t top,
                         float temperature, const float *row_weight, int reduction,
                         const float *loss_grad, const float *stats, void *logits_grad,
                         void *stream) {
    const int rc = check_distill("distill_backward", type, logits, rows, labels, stride, id_type,
                                 teacher_labels, teacher_type, teacher_logits, top, temperature,
                                 reduction);
    if (rc != SDF_OK) return rc;
    if (rows == 0) return SDF_OK;
    if (!loss_grad || !stats || !logits_grad) return fail(SDF_E_INVALID, "NULL pointer argument");
    const float reduce = reduction == SDF_REDUCE_MEAN ? (float)(1.0 / (double)rows) : 1.0f;
    DistillArgs a = {logits, stride, (uint32_t)labels, id_type, teacher_labels, teacher_type,
                     teacher_logits, top, temperature, row_weight, loss_grad,
                     reduction == SDF_REDUCE_NONE ? 1u : 0u, reduce, nullptr,
                     reinterpret_cast<float2 *>(const_cast<float *>(stats)), logits_grad};
    with_type(type, [&](auto t) {
        hipLaunchKernelGGL((distill_kernel<decltype(t), true>), dim3((unsigned)rows), dim3(256), 0,
                           static_cast<hipStream_t>(stream), a);
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SDF_OK : hip_fail(e, "distill_backward");
}

size_t sdf_label_log_probs_scratch_bytes(uint64_t rows, uint64_t labels, uint32_t top) {
    (void)rows;
    (void)labels;
    (void)top;
    return 256;
}

int sdf_label_log_probs(int type, const void *logits, uint64_t rows, uint64_t labels,
                        uint64_t stride, int id_type, const void *label_ids, uint32_t top,
                        float temperature, float *log_prob, float *entropy, float *top_log_probs,
                        int64_t *top_labels, float *stats, void *scratch, size_t scratch_bytes,
                        void *stream) {
    const int rc = check_logits("label_log_probs", type, logits, rows, labels, stride, id_type,
                                temperature);
    if (rc != SDF_OK) return rc;
    if (top > kMaxTop)
        return fail(SDF_E_INVALID, "label_log_probs returns at most %u best labels", kMaxTop);
    if (rows == 0) return SDF_OK;
    if (!label_ids || !log_prob || !entropy || (top > 0 && (!top_log_probs || !top_labels)))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    const size_t need = sdf_label_log_probs_scratch_bytes(rows, labels, top);
    if (!scratch || scratch_bytes < need)
        return fail(SDF_E_INVALID, "scratch must hold %zu bytes (got %zu)", need, scratch_bytes);
    if ((reinterpret_cast<uintptr_t>(scratch) & 255u) != 0)
        return fail(SDF_E_INVALID, "scratch must be 256-byte aligned");
    AnswerArgs a = {logits, stride, (uint32_t)labels, id_type, label_ids, top, temperature,
                    log_prob, entropy, top_log_probs, top_labels,
                    reinterpret_cast<float2 *>(stats), nullptr, nullptr, nullptr};
    with_type(type, [&](auto t) {
        hipLaunchKernelGGL(answer_kernel<decltype(t)>, dim3((unsigned)rows), dim3(256), 0,
                           static_cast<hipStream_t>(stream), a);
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SDF_OK : hip_fail(e, "label_log_probs");
}

int sdf_label_log_probs_backward(int type, const void *logits, uint64_t rows, uint64_t labels,
                                 uint64_t stride, int id_type, const void *label_ids,
                                 float temperature, const float *entropy, const float *stats,
                                 const float *log_prob_grad, const float *entropy_grad,
                                 void *logits_grad, void *stream) {
    const int rc = check_logits("label_log_probs_backward", type, logits, rows, labels, stride,
                                id_type, temperature);
    if (rc != SDF_OK) return rc;
    if (rows == 0) return SDF_OK;
    if (!label_ids || !entropy || !stats || !logits_grad)
        return fail(SDF_E_INVALID, "NULL pointer argument");
    AnswerArgs a = {logits, stride, (uint32_t)labels, id_type, label_ids, 0, temperature, nullptr,
                    const_cast<float *>(entropy), nullptr, nullptr,
                    reinterpret_cast<float2 *>(const_cast<float *>(stats)), log_prob_grad,
                    entropy_grad, logits_grad};
    with_type(type, [&](auto t) {
        hipLaunchKernelGGL(answer_grad_kernel<decltype(t)>, dim3((unsigned)rows), dim3(256), 0,
                           static_cast<hipStream_t>(stream), a);
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SDF_OK : hip_fail(e, "label_log_probs_backward");
}

} // extern "C"
