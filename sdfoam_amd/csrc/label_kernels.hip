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

// Softmax statistics of the labels seen so far: the largest logit, and relative
// to it S and W = sum d e, d = (z - m) c, e = 2^d, c = log2(e) / T (the logits
// are scaled to base 2 once, so that an exponential is one instruction).
// Nothing but -inf seen: m = -inf, S = 0.  A NaN reaches S, and so does +inf.
struct Part {
    float m, s, w;
};
// m >= p.m.  Where p.m is -inf, S is 0 and stays so; the bound on d keeps
// 0 * inf out of W.
template <bool kEntropy> __device__ __forceinline__ void rebase(Part &p, float m, float c) {
    const float d = p.m == m ? 0.0f : (p.m - m) * c;
    const float f = __builtin_amdgcn_exp2f(d);
    if (kEntropy) p.w = (p.w + fmaxf(d, -200.0f) * p.s) * f;
    p.s *= f;
    p.m = m;
}
// The elements of kU chunks into p: for kGroup chunks at a time one change of
// base, then a subtraction, a product, an exponential and a sum for each.
// (A group's elements are unpacked at once: 8 held chunks of 8 in one group
// take 138 VGPRs and leave one block of 512 threads a CU.)  The largest of them.
template <bool kEntropy, int kGroup, typename T, int kU>
__device__ __forceinline__ float absorb(Part &p, const Chunk<T> (&ch)[kU], float c) {
    float largest = -INFINITY;
#pragma unroll
    for (int i0 = 0; i0 < kU; i0 += kGroup) {
        float m = -INFINITY;
#pragma unroll
        for (int i = i0; i < kU && i < i0 + kGroup; ++i)
#pragma unroll
            for (int e = 0; e < Chunk<T>::kN; ++e) m = fmaxf(m, ch[i][e]);
        largest = fmaxf(largest, m);
        m = fmaxf(m, p.m);
        rebase<kEntropy>(p, m, c);
        const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int i = i0; i < kU && i < i0 + kGroup; ++i)
#pragma unroll
            for (int e = 0; e < Chunk<T>::kN; ++e) {
                const float d = (ch[i][e] - base) * c;
                const float x = __builtin_amdgcn_exp2f(d);
                p.s += x;
                if (kEntropy) p.w = fmaf(fmaxf(d, -200.0f), x, p.w);
            }
    }
    return largest;
}
// One Part of the kLanes neighbouring lanes' (in all of them).
template <int kLanes, bool kEntropy> __device__ __forceinline__ void merge_lanes(Part &p, float c) {
    rebase<kEntropy>(p, group_max<kLanes>(p.m), c);
    p.s = group_sum<kLanes>(p.s);
    if (kEntropy) p.w = group_sum<kLanes>(p.w);
}
// One Part of n others.
template <bool kEntropy> __device__ __forceinline__ Part merge_parts(const Part *parts, uint32_t n, float c) {
    Part all = {-INFINITY, 0.0f, 0.0f};
    for (uint32_t k = 0; k < n; ++k) all.m = fmaxf(all.m, parts[k].m);
    for (uint32_t k = 0; k < n; ++k) {
        Part p = parts[k];
        rebase<kEntropy>(p, all.m, c);
        all.s += p.s;
        if (kEntropy) all.w += p.w;
    }
    return all;
}
// One Part of the block's threads; `parts` holds one per wavefront.  Leaves a
// barrier behind it that orders the threads' earlier writes to LDS.
template <bool kEntropy> __device__ __forceinline__ Part merge_block(Part p, Part *parts, float c) {
    merge_lanes<64, kEntropy>(p, c);
    if ((threadIdx.x & 63u) == 0) parts[threadIdx.x >> 6] = p;
    __syncthreads();
    return merge_parts<kEntropy>(parts, blockDim.x >> 6, c);
}

// f(chunks, at) over a span, kU chunks of each of kThreads threads at a time,
// chunk i at `at` + i kThreads kN, and one by one where the span's end leaves
// fewer; what is not a chunk's own is -inf where kMask, else as it was read.
// kOnce: past the caches, for what is not read again (8,192 rows of 65,536: 190
// -> 164 us, 6.6 TB/s).  Only the steps that begin in [first, last).
template <int kThreads, int kU, bool kMask, bool kOnce, typename T, typename F>
__device__ __forceinline__ void for_steps(const Span<T> &z, uint32_t first, uint32_t last, F f) {
    constexpr uint32_t kStep = kThreads * Chunk<T>::kN;
    uint32_t at = first + threadIdx.x % kThreads * Chunk<T>::kN;
    for (; first < last && first + kStep * kU <= z.last(); first += kStep * kU, at += kStep * kU) {
        Chunk<T> ch[kU];
        if (z.plain_step(first, kStep * kU)) {
            const T *p = z.row + (at - z.skew);
#pragma unroll
            for (int i = 0; i < kU; ++i) ch[i] = load_chunk_if<kOnce>(p + i * kStep);
        } else {
#pragma unroll
            for (int i = 0; i < kU; ++i)
                ch[i] = z.template load<kOnce>(at + i * kStep, (T)-INFINITY);
            if (kMask) {
#pragma unroll
                for (int i = 0; i < kU; ++i) z.mask(ch[i], at + i * kStep, (T)-INFINITY);
            }
        }
        f(ch, at);
    }
    if (first >= last) return;
    for (; at < z.last(); at += kStep) {
        Chunk<T> ch[1] = {z.template load<kOnce>(at, (T)-INFINITY)};
        if (kMask) z.mask(ch[0], at, (T)-INFINITY);
        f(ch, at);
    }
}
template <int kThreads, int kU, bool kMask, bool kOnce, typename T, typename F>
__device__ __forceinline__ void for_chunks(const Span<T> &z, F f) {
    for_steps<kThreads, kU, kMask, kOnce>(z, z.begin, z.last(), f);
}
// to[i] = f(z[i]) over a span, chunk by chunk, z read for the last time
template <int kThreads, int kU, bool kPast, typename T, typename F>
__device__ __forceinline__ void map_chunks(const Span<T> &z, T *to, F f) {
    constexpr uint32_t kStep = kThreads * Chunk<T>::kN;
    for_chunks<kThreads, kU, false, true>(z, [&](const auto &ch, uint32_t at) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(ch) / 16); ++i)
            if (at + i * kStep < z.last()) {
                const uint32_t from = z.place(at + i * kStep);
                const Chunk<T> o = f(ch[i], from);
                // two threads may write one element, and then the same value
                if (z.whole) store_chunk_if<kPast>(to + from, o);
                else z.store_own(to, from, o);
            }
    });
}

constexpr int kStream = 256; // threads a block where rows are streamed
constexpr int kUnroll = 4;   // chunks in flight per thread

template <bool kEntropy, int kThreads, typename T>
__device__ __forceinline__ void stream_part(Part &p, const Span<T> &z, float c) {
    for_chunks<kThreads, kUnroll, true, false>(
        z, [&](const auto &ch, uint32_t) { absorb<kEntropy, kUnroll>(p, ch, c); });
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
    float temperature, c; // T, log2(e) / T
    const float *row_weight;   // NULL: 1
    const float *loss_grad;    // NULL: 1
    uint32_t loss_grad_stride; // 0: one for all rows
    float reduce;              // what a row's loss counts in the result
    float *loss;               // [rows]; NULL: not written
    float2 *stats;             // [rows] {m, S}: the backward's input, else written unless NULL
    void *logits_grad;         // [rows, labels]; NULL: not written
};

__device__ __forceinline__ float teacher_logit(const DistillArgs &a, uint64_t i) {
    if (a.teacher_type == SDF_TYPE_F16) return (float)static_cast<const half_t *>(a.teacher_logits)[i];
    if (a.teacher_type == SDF_TYPE_BF16) return (float)static_cast<const bf16_t *>(a.teacher_logits)[i];
    return static_cast<const float *>(a.teacher_logits)[i];
}

// A row's teacher in LDS: each entry's logit (later its share q), label (-1:
// does not count) and the row's own logit there.  Read from memory once, on
// their way while the row itself is.
struct Entries {
    float *q, *z;
    int32_t *id;
};
constexpr uint32_t kEntryBytes = 12;
__device__ __forceinline__ Entries entries_at(void *shared, uint32_t top) {
    float *q = static_cast<float *>(shared);
    return {q, q + top, reinterpret_cast<int32_t *>(q + 2 * top)};
}
__device__ __forceinline__ float entry(const DistillArgs &a, uint64_t r, uint32_t k, int32_t &j) {
    j = load_id(a.teacher_labels, a.id_type, r * a.top + k, a.labels);
    const float t = j < 0 ? -INFINITY : teacher_logit(a, r * a.top + k);
    if (t == -INFINITY) j = -1;
    return t;
}
template <typename T>
__device__ __forceinline__ void put_entry(const Entries &e, uint32_t k, int32_t j, float t, const T *z) {
    e.q[k] = t;
    e.id[k] = j;
    e.z[k] = j < 0 ? 0.0f : (float)z[j];
}
// Entries `first`, `first` + step, ... from memory.
template <typename T>
__device__ __forceinline__ void load_entries(const DistillArgs &a, uint64_t r, const T *z,
                                             const Entries &e, uint32_t first, uint32_t step) {
    for (uint32_t k = first; k < a.top; k += step) {
        int32_t j;
        const float t = entry(a, r, k, j);
        put_entry(e, k, j, t, z);
    }
}
// The softmax of the counting entries, by every group of kLanes lanes for
// itself.  s = 0: none counts.
struct Teacher {
    float m, s;
};
template <int kLanes>
__device__ __forceinline__ Teacher teacher_of(const DistillArgs &a, const Entries &e) {
    const uint32_t l = threadIdx.x & (kLanes - 1);
    Teacher t = {-INFINITY, 0.0f};
    for (uint32_t k = l; k < a.top; k += kLanes) t.m = fmaxf(t.m, e.q[k]);
    t.m = group_max<kLanes>(t.m);
    if (t.m == -INFINITY) t.m = 0.0f;
    for (uint32_t k = l; k < a.top; k += kLanes)
        t.s += __builtin_amdgcn_exp2f((e.q[k] - t.m) * a.c);
    t.s = group_sum<kLanes>(t.s);
    return t;
}
// The entries' logits become their shares, by the kLanes lanes of one group
// (when every other has read them), and T sum q (log q - log p) over them, the
// row's loss over u T.  (The T goes into the sum: what it multiplies is a
// difference of logits over T, and T^2 by itself is 0 or infinite in fp32 for
// temperatures below 1e-23 and above 1e19.)
template <int kLanes>
__device__ __forceinline__ float shares(const DistillArgs &a, const Entries &e, const Teacher &t,
                                        const Part &st) {
    const float log_s = logf(st.s), log_ts = logf(t.s);
    float sum = 0.0f;
    for (uint32_t k = threadIdx.x & (kLanes - 1); k < a.top; k += kLanes) {
        const float d = e.q[k] - t.m, q = __builtin_amdgcn_exp2f(d * a.c) / t.s;
        // an entry of no mass adds nothing, whatever its label's probability
        if (e.id[k] >= 0 && !(q == 0.0f))
            sum += q * (d - (e.z[k] - st.m) + a.temperature * (log_s - log_ts));
        e.q[k] = q;
    }
    return group_sum<kLanes>(sum);
}
// The row's gradient at the teacher's labels in [begin, end), over what stands
// there: entries `first`, `first` + `step`, ...
template <typename T>
__device__ __forceinline__ void write_shares(const DistillArgs &a, T *dz, const Entries &x,
                                             const Part &st, float coef, uint32_t first,
                                             uint32_t step, uint32_t begin, uint32_t end) {
    for (uint32_t k = first; k < a.top; k += step) {
        const int32_t j = x.id[k];
        if (j < 0 || (uint32_t)j < begin || (uint32_t)j >= end) continue;
        // A label that the teacher names twice has both shares.  Labels are compared four
        // at a time and a share is read where one is equal (one by one, with its share:
        // 4,096 rows of 32,768 bfloat16, 64 entries 124 -> 113 us, 1,024 737 -> 482).
        float mass = 0.0f;
        uint32_t o = 0;
        for (; o + 4 <= a.top; o += 4) {
            int32_t id[4];
            __builtin_memcpy(id, x.id + o, sizeof(id));
            if (id[0] != j && id[1] != j && id[2] != j && id[3] != j) continue;
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) mass += id[u] == j ? x.q[o + u] : 0.0f;
        }
        for (; o < a.top; ++o) mass += x.id[o] == j ? x.q[o] : 0.0f;
        const float p = __builtin_amdgcn_exp2f((x.z[k] - st.m) * a.c) / st.s;
        dz[j] = (T)(coef * (p - mass));
    }
}
__device__ __forceinline__ float row_coef(const DistillArgs &a, uint64_t r, float u) {
    const float g = a.loss_grad ? a.loss_grad[r * a.loss_grad_stride] : 1.0f;
    return g * a.reduce * u * a.temperature;
}
__device__ __forceinline__ float row_weight(const DistillArgs &a, uint64_t r) {
    return a.row_weight ? a.row_weight[r] : 1.0f;
}
// share * e of a chunk's logits
template <typename T>
__device__ __forceinline__ Chunk<T> grad_chunk(const Chunk<T> &ch, float m, float c, float share) {
    Chunk<T> o = {};
#pragma unroll
    for (int e = 0; e < Chunk<T>::kN; ++e)
        o.set(e, (T)(share * __builtin_amdgcn_exp2f((ch[e] - m) * c)));
    return o;
}
template <int kThreads, bool kPast, typename T>
__device__ __forceinline__ void write_zeros(T *dz, uint32_t begin, uint32_t end) {
    const Span<T> z(dz, begin, end);
    for (uint32_t at = begin + threadIdx.x * z.kN; at < z.last(); at += kThreads * z.kN)
        z.template store_own<kPast>(dz, at, {});
}

// A block per row.  With kHeld > 0 (the gradient is wanted): the row's first
// kThreads * kHeld chunks stay in registers between the statistics and the
// gradient, so they are read once; the rest is read again.  kHeld = 0: loss and
// statistics alone, streamed.  kPast: the gradient is written past the caches,
// or, with kHeld = 0, no backward will read the logits again.
// Bound by memory.  bfloat16, loss alone: 8,192 rows of 65,536 in 164 us (6.5
// TB/s).  With the gradient: 16,384 of 32,768 in 415 us (5.2 TB/s), 8,192 of
// 65,536 in 433 (5.0; blocks of 1,024 threads, one a CU: 749), 2,048 of 262,144,
// three quarters of a row read twice, in 456 (4.7 of the bytes needed).
template <typename T, int kThreads, int kHeld, bool kPast>
__global__ __launch_bounds__(kThreads)
    __attribute__((amdgpu_waves_per_eu(kHeld > 8 ? 4 : kHeld > 4 ? 6 : 7))) void
    distill_kernel(DistillArgs a) {
    constexpr uint32_t kN = Chunk<T>::kN;
    extern __shared__ float shared[];
    __shared__ Part parts[kThreads / 64];
    const Entries e = entries_at(shared, a.top);
    const uint64_t r = blockIdx.x;
    const Span<T> z(static_cast<const T *>(a.logits) + r * a.stride, 0u, a.labels);
    T *dz = static_cast<T *>(a.logits_grad) + r * a.labels;
    constexpr uint32_t kRest = kThreads * kN * kHeld;
    const float u = row_weight(a, r);
    Teacher t = {0.0f, 0.0f};
    Part st = {0.0f, 0.0f, 0.0f};
    Chunk<T> held[kHeld ? kHeld : 1];
    if (!(u == 0.0f)) { // the same in every thread
        int32_t j = -1;
        float logit = -INFINITY;
        if (threadIdx.x < a.top) logit = entry(a, r, threadIdx.x, j);
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            held[i] = z.template load<true>((threadIdx.x + i * kThreads) * kN, (T)-INFINITY);
        if (threadIdx.x < a.top) put_entry(e, threadIdx.x, j, logit, z.row);
        load_entries(a, r, z.row, e, threadIdx.x + kThreads, kThreads);
        __syncthreads();
        t = teacher_of<64>(a, e);
        if (!(t.s == 0.0f)) { // and this
            Part p = {-INFINITY, 0.0f, 0.0f};
            if constexpr (kHeld > 0) {
                if (!z.plain_step(0u, kRest)) {
#pragma unroll
                    for (int i = 0; i < kHeld; ++i)
                        z.mask(held[i], (threadIdx.x + i * kThreads) * kN, (T)-INFINITY);
                }
                absorb<false, 2>(p, held, a.c);
            }
            for_steps<kThreads, kUnroll, true, kHeld == 0 && kPast>(
                z, kRest, z.last(),
                [&](const auto &ch, uint32_t) { absorb<false, kUnroll>(p, ch, a.c); });
            st = merge_block<false>(p, parts, a.c);
            if (st.m == -INFINITY) st.m = 0.0f;
        }
    }
    const bool live = !(st.s == 0.0f);
    if (a.stats && threadIdx.x == 0) a.stats[r] = make_float2(st.m, st.s);
    if (threadIdx.x < 64u) {
        const float loss = live ? u * a.temperature * shares<64>(a, e, t, st) : 0.0f;
        if (threadIdx.x == 0) a.loss[r] = loss;
    }
    if constexpr (kHeld > 0) {
        if (!live) {
            write_zeros<kThreads, kPast>(dz, 0, a.labels);
            return;
        }
        const float coef = row_coef(a, r, u), share = coef / st.s;
        for_steps<kThreads, kUnroll, true, true>(z, kRest, z.last(), [&](const auto &ch, uint32_t at) {
#pragma unroll
            for (int i = 0; i < (int)(sizeof(ch) / 16); ++i)
                z.template store_own<kPast>(dz, at + i * kThreads * kN,
                                            grad_chunk(ch[i], st.m, a.c, share));
        });
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const uint32_t at = (threadIdx.x + i * kThreads) * kN;
            if (at < z.last())
                z.template store_own<kPast>(dz, at, grad_chunk(held[i], st.m, a.c, share));
        }
        __syncthreads(); // the teacher's labels are written over what stands there
        write_shares(a, dz, e, st, coef, threadIdx.x, kThreads, 0u, a.labels);
    }
}

// Few long rows: the statistics of a slice of a row per block.  64 rows of
// 100,003 with their gradient: 21 us with finish_kernel, as long as the call.
template <typename T>
__global__ __launch_bounds__(kStream) void part_kernel(DistillArgs a, uint32_t slices,
                                                       uint32_t slice, Part *out) {
    __shared__ Part parts[kStream / 64];
    const uint64_t r = blockIdx.x / slices;
    const uint32_t k = blockIdx.x % slices, begin = k * slice;
    const T *z = static_cast<const T *>(a.logits) + r * a.stride;
    const float c = a.c;
    if (a.row_weight && a.row_weight[r] == 0.0f) return; // not read, here or later
    Part p = {-INFINITY, 0.0f, 0.0f};
    stream_part<false, kStream>(p, Span<T>(z, begin, min(a.labels, begin + slice)), c);
    p = merge_block<false>(p, parts, c);
    if (threadIdx.x == 0) out[r * slices + k] = p;
}

// The loss, and the gradient of a slice of a row per block, from the row's
// statistics: `parts` of its slices, or a.stats where `parts` is NULL.  As the
// backward of a loss through autograd bound by memory: 4,096 rows of 32,768
// bfloat16, a third of them masked, 85 us (5.6 TB/s), 2,048 of 262,147 354.
template <typename T, bool kPast>
__global__ __launch_bounds__(kStream) void finish_kernel(DistillArgs a, uint32_t tiles,
                                                         uint32_t tile, const Part *parts,
                                                         uint32_t slices) {
    extern __shared__ float shared[];
    const Entries e = entries_at(shared, a.top);
    const uint64_t r = blockIdx.x / tiles;
    const uint32_t begin = (uint32_t)(blockIdx.x % tiles) * tile;
    const uint32_t end = min(a.labels, begin + tile);
    const T *z = static_cast<const T *>(a.logits) + r * a.stride;
    T *dz = static_cast<T *>(a.logits_grad) + r * a.labels;
    const float u = row_weight(a, r);
    Teacher t = {0.0f, 0.0f};
    Part st = {0.0f, 0.0f, 0.0f};
    if (!(u == 0.0f)) {
        load_entries(a, r, z, e, threadIdx.x, kStream);
        if (parts) {
            st = merge_parts<false>(parts + r * slices, slices, a.c);
            if (st.m == -INFINITY) st.m = 0.0f;
        } else {
            const float2 h = a.stats[r];
            st = {h.x, h.y, 0.0f};
        }
        __syncthreads();
        t = teacher_of<64>(a, e);
        if (t.s == 0.0f) st.s = 0.0f;
        __syncthreads(); // before the shares take the logits' place
    }
    const bool live = !(st.s == 0.0f);
    if (threadIdx.x < 64u) {
        const float loss = live ? u * a.temperature * shares<64>(a, e, t, st) : 0.0f;
        if (parts && begin == 0 && threadIdx.x == 0) {
            a.loss[r] = loss;
            if (a.stats) a.stats[r] = make_float2(live ? st.m : 0.0f, st.s);
        }
    }
    if (!a.logits_grad) return;
    if (!live) {
        write_zeros<kStream, kPast>(dz, begin, end);
        return;
    }
    const float coef = row_coef(a, r, u), share = coef / st.s;
    map_chunks<kStream, kUnroll, kPast>(Span<T>(z, begin, end), dz, [&](const Chunk<T> &ch, uint32_t) {
        return grad_chunk(ch, st.m, a.c, share);
    });
    __syncthreads();
    write_shares(a, dz, e, st, coef, threadIdx.x, kStream, begin, end);
}

// Short rows: kLanes lanes a row, the whole row in their registers (kHeld
// chunks each), 256 / kLanes rows a block or fewer where the teacher's entries
// fill LDS.  4,096 rows of 201 floats with their gradient: 6 us.
template <typename T, int kLanes, int kHeld, bool kHaveStats>
__global__ __launch_bounds__(256) void distill_short_kernel(DistillArgs a, uint64_t rows) {
    constexpr uint32_t kN = Chunk<T>::kN;
    extern __shared__ float shared[];
    const uint32_t g = threadIdx.x / kLanes, l = threadIdx.x % kLanes;
    const uint64_t r = (uint64_t)blockIdx.x * (blockDim.x / kLanes) + g;
    const bool in = r < rows;
    const Entries e = entries_at(shared + (size_t)g * 3 * a.top, a.top);
    const T *z = static_cast<const T *>(a.logits) + r * a.stride;
    T *dz = static_cast<T *>(a.logits_grad) + r * a.labels;
    const Span<T> span(z, 0u, a.labels);
    const float u = in ? row_weight(a, r) : 0.0f;
    Teacher t = {0.0f, 0.0f};
    Part st = {0.0f, 0.0f, 0.0f};
    Chunk<T> held[kHeld];
    if (!(u == 0.0f)) {
        int32_t j = -1;
        float logit = -INFINITY;
        if (l < a.top) logit = entry(a, r, l, j);
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            held[i] = span.load((l + i * kLanes) * kN, (T)-INFINITY);
        if (l < a.top) put_entry(e, l, j, logit, z);
        load_entries(a, r, z, e, l + kLanes, kLanes);
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            span.mask(held[i], (l + i * kLanes) * kN, (T)-INFINITY);
        if (kHaveStats) {
            const float2 h = a.stats[r];
            st = {h.x, h.y, 0.0f};
        } else {
            st = {-INFINITY, 0.0f, 0.0f};
            absorb<false, 2>(st, held, a.c);
            merge_lanes<kLanes, false>(st, a.c);
            if (st.m == -INFINITY) st.m = 0.0f;
        }
    }
    wave_sync(); // a group's lanes are of one wavefront
    if (!(u == 0.0f)) {
        t = teacher_of<kLanes>(a, e);
        if (t.s == 0.0f) st.s = 0.0f;
    }
    wave_sync();
    const bool live = !(st.s == 0.0f);
    if (live) {
        const float sum = shares<kLanes>(a, e, t, st);
        if (!kHaveStats && l == 0) a.loss[r] = u * a.temperature * sum;
    } else if (!kHaveStats && in && l == 0) {
        a.loss[r] = 0.0f;
    }
    if (!kHaveStats && a.stats && in && l == 0) a.stats[r] = make_float2(live ? st.m : 0.0f, st.s);
    if (!a.logits_grad) return;
    const float coef = live ? row_coef(a, r, u) : 0.0f, share = coef / st.s;
    if (in) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const uint32_t at = (l + i * kLanes) * kN;
            if (at >= span.last()) continue;
            Chunk<T> o = {};
            if (live) o = grad_chunk(held[i], st.m, a.c, share);
            span.store_own(dz, at, o);
        }
    }
    __syncthreads();
    if (live) write_shares(a, dz, e, st, coef, l, kLanes, 0u, a.labels);
}

// The rows' losses in one sum, always in the same order: each block a share of
// them, 32 in flight per thread; one block where they are few, else the blocks'
// sums are added by a second launch of one (160,000 rows: 7 us, 44 with one load
// at a time in one block).
constexpr uint64_t kSumRows = 1 << 15; // of a block
template <typename V>
__global__ __launch_bounds__(1024) void loss_sum_kernel(const V *__restrict__ loss, uint64_t rows,
                                                        uint64_t each, float scale,
                                                        double *__restrict__ partial,
                                                        float *__restrict__ out) {
    __shared__ double part[16];
    const uint64_t begin = blockIdx.x * each, end = begin + each < rows ? begin + each : rows;
    double s = 0.0;
    for (uint64_t r = begin + threadIdx.x; r < end; r += 1024u * 32u) {
        V x[32];
#pragma unroll
        for (uint32_t k = 0; k < 32u; ++k) // no branches: all of them on their way at once
            x[k] = loss[r + k * 1024u < end ? r + k * 1024u : end - 1];
#pragma unroll
        for (uint32_t k = 0; k < 32u; ++k) s += r + k * 1024u < end ? (double)x[k] : 0.0;
    }
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63u) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x != 0) return;
    s = 0.0;
    for (int k = 0; k < 16; ++k) s += part[k];
    if (out) *out = (float)(s * (double)scale);
    else partial[blockIdx.x] = s;
}
uint64_t sum_blocks(uint64_t rows) { return (rows + kSumRows - 1) / kSumRows; }
void launch_loss_sum(const float *loss, uint64_t rows, float scale, double *partial, float *out,
                     hipStream_t s) {
    const uint64_t blocks = sum_blocks(rows);
    if (blocks <= 1) {
        hipLaunchKernelGGL(loss_sum_kernel<float>, dim3(1), dim3(1024), 0, s, loss, rows, rows, scale,
                           partial, out);
        return;
    }
    hipLaunchKernelGGL(loss_sum_kernel<float>, dim3((unsigned)blocks), dim3(1024), 0, s, loss, rows,
                       kSumRows, scale, partial, static_cast<float *>(nullptr));
    hipLaunchKernelGGL(loss_sum_kernel<double>, dim3(1), dim3(1024), 0, s, partial, blocks, blocks,
                       scale, partial, out);
}

struct AnswerArgs {
    const void *logits;
    uint64_t stride;
    uint32_t labels;
    int id_type;
    const void *label_ids;
    uint32_t top;
    float inv_t, c; // 1 / T, log2(e) / T
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

__device__ __forceinline__ float order_logit(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
// The same in 16 bits for two 16-bit elements side by side: sign and magnitude
// become a two's complement number (so -0 and 0 are one) moved to be unsigned.
// NaN of either sign and -inf are not taken out: -inf and negative NaN lie below
// kLeast, positive NaN above +inf.
__device__ __forceinline__ uint32_t half_orders(uint32_t w) {
    typedef short Two __attribute__((ext_vector_type(2)));
    const Two sign = __builtin_bit_cast(Two, w) >> 15;
    const Two magnitude = __builtin_bit_cast(Two, w & 0x7fff7fffu);
    return __builtin_bit_cast(uint32_t, (Two)((magnitude ^ sign) - sign)) ^ 0x80008000u;
}
template <typename T> struct HalfOrder {
    static constexpr uint32_t kInf = __is_same(T, bf16_t) ? 0x7f80u : 0x7c00u;
    static constexpr uint32_t kLeast = 0x8000u - kInf + 1u; // of the lowest finite value
    static constexpr uint32_t kMost = 0x8000u + kInf;       // of +inf
    static __device__ __forceinline__ float value(uint32_t o) {
        const uint16_t bits = (uint16_t)(o >= 0x8000u ? o - 0x8000u : 0x8000u + (0x8000u - o));
        return (float)__builtin_bit_cast(T, bits);
    }
};
// Largest first.
template <int kCount> __device__ __forceinline__ void sort_falling(uint32_t (&x)[kCount]) {
    // Batcher's odd-even merge sort
#pragma unroll
    for (int p = 1; p < kCount; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < kCount; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < kCount && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const uint32_t a = x[i + j], b = x[i + j + k];
                        x[i + j] = max(a, b);
                        x[i + j + k] = min(a, b);
                    }
}
// Keys order labels by falling logit, then by rising label; 0 is no label.
__device__ __forceinline__ uint64_t key_of(uint32_t order, uint32_t label) {
    return (uint64_t)order << 32 | (0xffffffffu - label);
}

constexpr uint32_t kCandidates = 512;

// A bound from below on the k-th largest of the wavefront's 64 kEach orders, bit
// by bit: its upper half, which is all of it for bfloat16.  At least that of the
// lowest finite logit.
template <int kEach>
__device__ __forceinline__ uint32_t bound_of_wave(const uint32_t (&x)[kEach], uint32_t k) {
    uint32_t t = 0;
    for (int b = 31; b >= 16; --b) {
        const uint32_t with = t | 1u << b;
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) n += (uint32_t)__popcll(__ballot(x[i] >= with));
        if (n >= k) t = with;
    }
    return max(t, 0x00800000u);
}

__device__ __forceinline__ void write_answer(const AnswerArgs &a, uint64_t r, float z_label,
                                             bool named, const Part &st, float inv_t, float log_s) {
    const bool empty = st.s == 0.0f;
    float lp = 0.0f;
    if (named) lp = empty ? -INFINITY : (z_label - st.m) * inv_t - log_s;
    a.log_prob[r] = lp;
    a.entropy[r] = empty ? 0.0f : log_s - st.w * __builtin_amdgcn_rcpf(st.s * kLog2e);
    if (a.stats) a.stats[r] = make_float2(empty ? 0.0f : st.m, st.s);
}
__device__ __forceinline__ void write_best(const AnswerArgs &a, uint64_t r, uint32_t k, bool any,
                                           float z, uint32_t label, const Part &st, float inv_t,
                                           float log_s) {
    a.top_labels[r * a.top + k] = any ? (int64_t)label : -1;
    a.top_log_probs[r * a.top + k] =
        any ? (z - st.m) * inv_t - log_s : (st.s != st.s ? st.s : -INFINITY);
}
__device__ __forceinline__ void write_best(const AnswerArgs &a, uint64_t r, uint32_t k, uint64_t key,
                                           const Part &st, float inv_t, float log_s) {
    write_best(a, r, k, key != 0, order_logit((uint32_t)(key >> 32)), 0xffffffffu - (uint32_t)key, st,
               inv_t, log_s);
}

// A block per row, or per slice of one where rows are few; one pass over the
// logits for the softmax, its entropy and each thread's largest logit.
// The best labels: the top-th largest of the threads' largest logits bounds the
// top-th best label from below (the threads are more than `top`).  Only threads
// whose largest logit reaches the bound (about `top`) look at theirs again, and
// only at the one or two steps that hold it where no third does; what reaches
// it is ranked by counting.
// Bound by memory, then by VALU issue (11 lane-operations a label): 8,192 rows of
// 100,003 bfloat16, 8 best: 276 us (5.9 TB/s); 2,048 of 50,021 floats: 74.
// slices > 1: Part and keys of each slice, for join_kernel.  kOnce: no backward
// will read the logits again (2,048 rows of 50,021 floats with their gradient:
// 221 us past the caches, 207 through them).
template <typename T, bool kOnce>
__global__ __launch_bounds__(kStream) void answer_kernel(AnswerArgs a, uint32_t slices,
                                                         uint32_t slice, Part *out,
                                                         uint64_t *out_keys) {
    __shared__ Part parts[kStream / 64];
    constexpr int kEach = kStream / 64;
    __shared__ uint32_t bests[kStream];
    __shared__ uint64_t keys[kCandidates];
    __shared__ uint32_t found;
    const uint64_t r = blockIdx.x / slices;
    const uint32_t part = blockIdx.x % slices, begin = part * slice;
    const uint32_t end = min(a.labels, begin + slice);
    const T *z = static_cast<const T *>(a.logits) + r * a.stride;
    const float inv_t = a.inv_t, c = a.c;
    const Span<T> span(z, begin, end);
    // beside its largest logit, where the thread met it, the next largest step's
    // and where, and the largest of its other steps
    Part mine = {-INFINITY, 0.0f, 0.0f};
    float second = -INFINITY, third = -INFINITY;
    uint32_t where = begin, where_second = begin;
    for_chunks<kStream, kUnroll, true, kOnce>(span, [&](const auto &ch, uint32_t at) {
        const float first = mine.m, m = absorb<true, kUnroll>(mine, ch, c);
        const bool leads = m > first, follows = m > second;
        third = fmaxf(third, fminf(m, second));
        where_second = leads ? where : follows ? at : where_second;
        second = fmaxf(second, fminf(m, first));
        where = leads ? at : where;
    });
    const uint32_t best = logit_order(mine.m);
    bests[threadIdx.x] = best;
    if (threadIdx.x == 0) found = 0;
    Part st = merge_block<true>(mine, parts, c);
    if (slices == 1 && st.m == -INFINITY) st.m = 0.0f;
    if (threadIdx.x == 0) {
        if (slices > 1) {
            out[r * slices + part] = st;
        } else {
            const int32_t y = load_id(a.label_ids, a.id_type, r, a.labels);
            write_answer(a, r, y < 0 ? 0.0f : (float)z[y], y >= 0, st, inv_t, logf(st.s));
        }
    }
    if (!a.top) return;
    const float log_s = logf(st.s);
    const auto emit = [&](uint32_t k, uint64_t key) {
        if (slices > 1) out_keys[(r * slices + part) * a.top + k] = key;
        else write_best(a, r, k, key, st, inv_t, log_s);
    };
    uint32_t of_threads[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) of_threads[k] = bests[k * 64u + (threadIdx.x & 63u)];
    const uint32_t bound = bound_of_wave(of_threads, a.top);
    const float least = order_logit(bound);
    if (best >= bound) {
        const auto collect = [&](const auto &ch, uint32_t at) {
#pragma unroll
            for (int i = 0; i < (int)(sizeof(ch) / 16); ++i)
#pragma unroll
                for (uint32_t e = 0; e < (uint32_t)Chunk<T>::kN; ++e) {
                    if (!(ch[i][e] >= least)) continue;
                    const uint32_t o = logit_order(ch[i][e]);
                    const uint32_t k = atomicAdd(&found, 1u);
                    const uint32_t from = span.place(at + i * kStream * Chunk<T>::kN);
                    if (k < kCandidates) keys[k] = key_of(o, from + e);
                }
        };
        if (logit_order(third) < bound) {
            constexpr uint32_t kStep = kStream * Chunk<T>::kN;
            const uint32_t own = threadIdx.x * Chunk<T>::kN;
            const uint32_t steps = logit_order(second) < bound ? 1 : 2;
            for (uint32_t k = 0; k < steps; ++k) {
                const uint32_t at = k ? where_second : where, first = at - own;
                if (first + kStep * kUnroll <= span.last()) {
                    for_steps<kStream, kUnroll, true, false>(span, first, first + 1, collect);
                } else {
                    Chunk<T> ch[1] = {span.load(at, (T)-INFINITY)};
                    span.mask(ch[0], at, (T)-INFINITY);
                    collect(ch, at);
                }
            }
        } else {
            for_chunks<kStream, kUnroll, true, false>(span, collect);
        }
    }
    __syncthreads();
    const uint32_t n = found;
    if (n <= kCandidates) {
        for (uint32_t i = threadIdx.x; i < n; i += kStream) {
            const uint64_t key = keys[i];
            uint32_t rank = 0;
            for (uint32_t o = 0; o < n; ++o) rank += keys[o] > key;
            if (rank < a.top) emit(rank, key);
        }
        if (threadIdx.x >= n && threadIdx.x < a.top) emit(threadIdx.x, 0);
        return;
    }
    // More labels reach the bound than there is room for.  Where `top` threads and
    // more have the row's largest logit, as in a row of one value, the first
    // `top` labels that have it are the answer: in order, counted as they come.
    uint32_t peak = 0, equal = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) peak = max(peak, of_threads[k]);
    peak = group_all<64>(peak, [](uint32_t x, uint32_t y) { return max(x, y); });
#pragma unroll
    for (int k = 0; k < kEach; ++k) equal += (uint32_t)__popcll(__ballot(of_threads[k] == peak));
    if (equal >= a.top) {
        const float largest = order_logit(peak);
        uint32_t *counts = reinterpret_cast<uint32_t *>(keys); // [2][wavefronts]
        uint32_t have = 0, turn = 0;
        for (uint32_t first = begin; have < a.top && first < span.last();
             first += kStream * Chunk<T>::kN, turn ^= kStream / 64) {
            const uint32_t at = first + threadIdx.x * Chunk<T>::kN;
            uint32_t bits = 0;
            if (at < span.last()) {
                Chunk<T> ch = span.load(at, (T)-INFINITY);
                span.mask(ch, at, (T)-INFINITY);
#pragma unroll
                for (int e = 0; e < Chunk<T>::kN; ++e) bits |= (ch[e] == largest ? 1u : 0u) << e;
            }
            uint32_t upto = __popc(bits);
            for (uint32_t d = 1; d < 64u; d <<= 1) {
                const uint32_t o = __shfl_up(upto, d);
                if ((threadIdx.x & 63u) >= d) upto += o;
            }
            if ((threadIdx.x & 63u) == 63u) counts[turn + (threadIdx.x >> 6)] = upto;
            __syncthreads();
            uint32_t rank = have + upto - __popc(bits);
            for (uint32_t w = 0; w < kStream / 64u; ++w) {
                if (w < threadIdx.x >> 6) rank += counts[turn + w];
                have += counts[turn + w];
            }
            for (; bits != 0 && rank < a.top; bits &= bits - 1u, ++rank)
                emit(rank, key_of(peak, span.place(at) + __ffs(bits) - 1));
        }
        return;
    }
    // Else one pass for each.
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < a.top; ++k) {
        uint64_t key = 0;
        for_chunks<kStream, 1, true, false>(span, [&](const Chunk<T>(&ch)[1], uint32_t at) {
#pragma unroll
            for (uint32_t e = 0; e < (uint32_t)Chunk<T>::kN; ++e) {
                const uint32_t o = logit_order(ch[0][e]);
                const uint64_t x = key_of(o, span.place(at) + e);
                if (o != 0 && x < last && x > key) key = x;
            }
        });
        for (int d = 32; d > 0; d >>= 1) {
            const uint64_t o = __shfl_xor((unsigned long long)key, d);
            key = o > key ? o : key;
        }
        __syncthreads();
        if ((threadIdx.x & 63u) == 0) keys[threadIdx.x >> 6] = key;
        __syncthreads();
        for (int i = 0; i < kStream / 64; ++i) key = keys[i] > key ? keys[i] : key;
        if (threadIdx.x == 0) emit(k, key);
        last = key;
    }
}

constexpr uint32_t kMaxSlices = 32; // of a row of answers

// One row of its slices: their Parts merged, and the best of their best.  With
// q = top / slices rounded up, the m-th largest of the slices' q-th keys has at
// least m q keys at or above it: for m q >= top it bounds the top-th best label
// from below.  What reaches it (about `top`) is ranked by counting.  32 slices of
// 20: 3.5 us (39 with the rank of every key found by halving).
template <typename T>
__global__ __launch_bounds__(kStream) void join_kernel(AnswerArgs a, uint32_t slices,
                                                       const Part *parts, const uint64_t *keys) {
    constexpr uint32_t kEach = kMaxSlices * kMaxTop / kStream;
    __shared__ uint64_t all[kMaxSlices * kMaxTop];
    __shared__ uint32_t found;
    const uint64_t r = blockIdx.x;
    const float inv_t = a.inv_t, c = a.c;
    const uint32_t lane = threadIdx.x & 63u, n = slices * a.top;
    if (threadIdx.x == 0) found = 0;
    const int32_t y = load_id(a.label_ids, a.id_type, r, a.labels);
    const float zy = y < 0 ? 0.0f : (float)(static_cast<const T *>(a.logits) + r * a.stride)[y];
    // every wavefront merges the Parts for itself, a lane each
    Part st = {-INFINITY, 0.0f, 0.0f};
    if (lane < slices) st = parts[r * slices + lane];
    uint64_t mine[kEach];
    uint32_t bound = 0;
    if (a.top) {
#pragma unroll
        for (uint32_t k = 0; k < kEach; ++k) {
            const uint32_t i = k * kStream + threadIdx.x;
            mine[k] = i < n ? keys[r * n + i] : 0;
        }
        const uint32_t q = (a.top + slices - 1) / slices;
        const uint32_t of_slices[1] = {
            lane < slices ? (uint32_t)(keys[r * n + lane * a.top + q - 1] >> 32) : 0u};
        bound = bound_of_wave(of_slices, (a.top + q - 1) / q);
    }
    merge_lanes<64, true>(st, c);
    if (st.m == -INFINITY) st.m = 0.0f;
    if (threadIdx.x == 0) write_answer(a, r, zy, y >= 0, st, inv_t, logf(st.s));
    if (!a.top) return;
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < kEach; ++k)
        if ((uint32_t)(mine[k] >> 32) >= bound) all[atomicAdd(&found, 1u)] = mine[k];
    __syncthreads();
    const uint32_t some = found;
    const float log_s = logf(st.s);
    for (uint32_t i = threadIdx.x; i < some; i += kStream) {
        const uint64_t key = all[i];
        uint32_t rank = 0;
        for (uint32_t o = 0; o < some; ++o) rank += all[o] > key;
        if (rank < a.top) write_best(a, r, rank, key, st, inv_t, log_s);
    }
    // fewer labels than asked for
    if (threadIdx.x >= some && threadIdx.x < a.top)
        write_best(a, r, threadIdx.x, 0, st, inv_t, log_s);
}

// Short rows: kLanes lanes a row, in their registers.  The best labels one
// after the other: the largest of the lanes' largest logits, then the lowest
// label that has it.  160,000 rows of 121 halves, 5 best: 24 us, bound by VALU
// issue (about 370 instructions for four rows).
template <typename T, int kLanes, int kHeld>
__global__ __launch_bounds__(256) void answer_short_kernel(AnswerArgs a, uint64_t rows) {
    constexpr uint32_t kN = Chunk<T>::kN;
    const uint32_t l = threadIdx.x % kLanes;
    const uint64_t r = ((uint64_t)blockIdx.x * 256u + threadIdx.x) / kLanes;
    if (r >= rows) return; // a whole group
    const T *z = static_cast<const T *>(a.logits) + r * a.stride;
    const float inv_t = a.inv_t, c = a.c;
    const Span<T> span(z, 0u, a.labels);
    Chunk<T> held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = span.load((l + i * kLanes) * kN, (T)-INFINITY);
    // (no branch: the row is on its way, and this load with the arithmetic)
    const int32_t y = load_id(a.label_ids, a.id_type, r, a.labels);
    const T zy = z[max(y, 0)];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) span.mask(held[i], (l + i * kLanes) * kN, (T)-INFINITY);
    Part st = {-INFINITY, 0.0f, 0.0f};
    absorb<true, 2>(st, held, c);
    merge_lanes<kLanes, true>(st, c);
    if (st.m == -INFINITY) st.m = 0.0f;
    const float log_s = logf(st.s);
    // (the rest is written last: a wait for a load waits for earlier stores too)
    const auto done = [&]() {
        if (l == 0) write_answer(a, r, (float)zy, y >= 0, st, inv_t, log_s);
    };
    if (!a.top) return done();
    // lane k % kLanes keeps the k-th best until every lane has one to write
    const auto flush = [&](uint32_t k, bool any, float best, uint32_t label) {
        const uint32_t last = k % kLanes;
        if (l <= last) write_best(a, r, k - last + l, any, best, label, st, inv_t, log_s);
    };
    const auto greater = [](uint32_t x, uint32_t w) { return max(x, w); };
    constexpr uint32_t kOwn = kHeld * kN;
    if constexpr (sizeof(T) == 2) {
        // order and label fit 32 bits (the label from the end: ties to the lowest)
        using Order = HalfOrder<T>;
        uint32_t key[kOwn], kept = 0;
#pragma unroll
        for (uint32_t i = 0; i < kOwn; i += 2) {
            const uint32_t label = 0xffffu - span.place((l + i / kN * kLanes) * kN) - i % kN;
            const uint32_t o = half_orders(held[i / kN].w[i % kN / 2]);
            key[i] = o << 16 | label;
            key[i + 1] = (o & 0xffff0000u) | (label - 1u);
        }
        if (st.s != st.s) { // of a row that may hold NaN: those are never the best
#pragma unroll
            for (uint32_t i = 0; i < kOwn; ++i) key[i] = key[i] >> 16 > Order::kMost ? 0u : key[i];
        }
        constexpr bool kSorted = kOwn <= 8; // else taking out the best is less work
        if constexpr (kSorted) sort_falling(key);
        for (uint32_t k = 0; k < a.top; ++k) {
            uint32_t best = key[0];
            if constexpr (!kSorted) {
#pragma unroll
                for (uint32_t i = 1; i < kOwn; ++i) best = max(best, key[i]);
            }
            best = group_all<kLanes>(best, greater);
            if constexpr (kSorted) {
                if (key[0] == best) {
#pragma unroll
                    for (uint32_t i = 0; i + 1 < kOwn; ++i) key[i] = key[i + 1];
                    key[kOwn - 1] = 0u;
                }
            } else {
#pragma unroll
                for (uint32_t i = 0; i < kOwn; ++i) key[i] = key[i] == best ? 0u : key[i];
            }
            kept = l == k % kLanes ? best : kept;
            if (k % kLanes == kLanes - 1 || k + 1 == a.top)
                flush(k, kept >> 16 >= Order::kLeast, Order::value(kept >> 16),
                      0xffffu - (kept & 0xffffu));
        }
    } else {
        uint32_t o[kOwn], kept = 0, kept_label = 0;
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) o[i] = logit_order(held[i / kN][i % kN]);
        for (uint32_t k = 0; k < a.top; ++k) {
            uint32_t best = 0, at = 0;
#pragma unroll
            for (uint32_t i = 0; i < kOwn; ++i)
                if (o[i] > best) {
                    best = o[i];
                    at = i;
                }
            const uint32_t top = group_all<kLanes>(best, greater);
            const uint32_t label = span.place((l + at / kN * kLanes) * kN) + at % kN;
            const uint32_t lowest =
                group_all<kLanes>(best == top ? label : 0xffffffffu,
                                  [](uint32_t x, uint32_t w) { return min(x, w); });
            if (label == lowest) {
#pragma unroll
                for (uint32_t i = 0; i < kOwn; ++i) o[i] = i == at ? 0u : o[i];
            }
            kept = l == k % kLanes ? top : kept;
            kept_label = l == k % kLanes ? lowest : kept_label;
            if (k % kLanes == kLanes - 1 || k + 1 == a.top)
                flush(k, kept != 0, order_logit(kept), kept_label);
        }
    }
    done();
}

// kLanes lanes a row (256: a block, or a tile of a row per block).  Bound by
// memory: 2,048 rows of 50,021 floats in 125 us (6.5 TB/s, part of the logits
// still in the caches from the forward).
template <typename T, int kLanes, bool kPast>
__global__ __launch_bounds__(256) void answer_grad_kernel(AnswerArgs a, uint64_t rows,
                                                          uint32_t tiles, uint32_t tile) {
    const uint64_t r = kLanes == 256 ? blockIdx.x / tiles
                                     : ((uint64_t)blockIdx.x * 256u + threadIdx.x) / kLanes;
    if (r >= rows) return;
    const uint32_t begin = kLanes == 256 ? (uint32_t)(blockIdx.x % tiles) * tile : 0u;
    const uint32_t end = min(a.labels, begin + tile);
    const T *z = static_cast<const T *>(a.logits) + r * a.stride;
    T *dz = static_cast<T *>(a.logits_grad) + r * a.labels;
    const float inv_t = a.inv_t, c = a.c;
    const float2 st = a.stats[r];
    const int32_t y = load_id(a.label_ids, a.id_type, r, a.labels);
    const bool live = !(st.y == 0.0f);
    const float glp = live && a.log_prob_grad && y >= 0 ? a.log_prob_grad[r] * inv_t : 0.0f;
    const float gh = live && a.entropy_grad ? a.entropy_grad[r] * inv_t : 0.0f;
    // -p (glp + gh (log p + H)) = -e / S (gh ln2 d + glp + gh (H - log S))
    const float slope = gh / kLog2e, level = glp + gh * (a.entropy[r] - logf(st.y));
    const float inv_s = live ? -1.0f / st.y : 0.0f;
    map_chunks<kLanes, kUnroll, kPast>(Span<T>(z, begin, end), dz, [&](const Chunk<T> &ch, uint32_t at) {
        Chunk<T> o = {};
#pragma unroll
        for (int e = 0; e < Chunk<T>::kN; ++e) {
            const float d = (ch[e] - st.x) * c;
            const float p = __builtin_amdgcn_exp2f(d) * inv_s;
            float g = live ? p * fmaf(slope, fmaxf(d, -200.0f), level) : 0.0f;
            if ((int32_t)(at + e) == y) g += glp;
            o.set(e, (T)g);
        }
        return o;
    });
}

// ---- which kernel --------------------------------------------------------------

// f(first row, rows) for windows of rows: a launch holds fewer than 2^32 threads.
template <typename F> void for_windows(uint64_t rows, F f) {
    constexpr uint64_t kWindow = 1ull << 22;
    for (uint64_t r = 0; r < rows; r += kWindow) f(r, rows - r < kWindow ? rows - r : kWindow);
}
template <typename P> P *advance(P *p, uint64_t bytes) {
    return p ? (P *)((uintptr_t)p + bytes) : p;
}
size_t id_bytes(int id_type) { return id_type == SDF_ID_I64 ? 8 : 4; }

DistillArgs from_row(DistillArgs a, int type, uint64_t r) {
    a.logits = advance(a.logits, r * a.stride * type_bytes(type));
    a.teacher_labels = advance(a.teacher_labels, r * a.top * id_bytes(a.id_type));
    a.teacher_logits = advance(a.teacher_logits, r * a.top * type_bytes(a.teacher_type));
    a.row_weight = advance(a.row_weight, 4 * r);
    a.loss_grad = advance(a.loss_grad, 4 * r * a.loss_grad_stride);
    a.loss = advance(a.loss, 4 * r);
    a.stats = advance(a.stats, 8 * r);
    a.logits_grad = advance(a.logits_grad, r * a.labels * type_bytes(type));
    return a;
}
AnswerArgs from_row(AnswerArgs a, int type, uint64_t r) {
    a.logits = advance(a.logits, r * a.stride * type_bytes(type));
    a.label_ids = advance(a.label_ids, r * id_bytes(a.id_type));
    a.log_prob = advance(a.log_prob, 4 * r);
    a.entropy = advance(a.entropy, 4 * r);
    a.top_log_probs = advance(a.top_log_probs, 4 * r * a.top);
    a.top_labels = advance(a.top_labels, 8 * r * a.top);
    a.stats = advance(a.stats, 8 * r);
    a.log_prob_grad = advance(a.log_prob_grad, 4 * r);
    a.entropy_grad = advance(a.entropy_grad, 4 * r);
    a.logits_grad = advance(a.logits_grad, r * a.labels * type_bytes(type));
    return a;
}

// Slices for rows that are too few to fill the chip: enough blocks of at least
// 4,096 labels each; a multiple of a chunk long.  Made once of all rows of a
// call, as the size of the scratch is: a window's own rows may be few where the
// call's are many, and have no room for its Parts then.
struct Slices {
    uint32_t count, length;
};
Slices slices_of(uint64_t rows, uint64_t labels, uint32_t most) {
    uint64_t n = 1;
    if (rows < 512) n = 1024 / (rows ? rows : 1);
    n = n < labels / 4096 ? n : labels / 4096;
    n = n < most ? n : most;
    if (n < 2) return {1, (uint32_t)labels};
    const uint64_t length = ((labels + n - 1) / n + 7) / 8 * 8;
    return {(uint32_t)((labels + length - 1) / length), (uint32_t)length};
}
constexpr uint32_t kDistillSlices = 64;
constexpr uint32_t kShort = 64 * 4; // chunks of a row that a wavefront holds

// Chunks of a row at most: one more where rows begin between 16-byte boundaries.
template <typename T> uint64_t chunks_of(const void *logits, uint64_t stride, uint64_t labels) {
    const bool aligned = (reinterpret_cast<uintptr_t>(logits) & 15u) == 0 &&
                         stride * sizeof(T) % 16 == 0;
    return (labels + (aligned ? 0 : Chunk<T>::kN - 1) + Chunk<T>::kN - 1) / Chunk<T>::kN;
}
// Gradients that no cache would keep for their reader are written past them
// (1 GB, 2,048 rows of 262,144 bfloat16: 553 -> 475 us, 16,384 of 32,768: 454 ->
// 412; 256 MiB, 4,096 of 32,768, a third of the rows masked: 97 -> 104).
template <typename T> bool past_caches(uint64_t rows, uint64_t labels) {
    return rows * labels * sizeof(T) > 256ull << 20;
}
// f(lanes, chunks held by each) of a short row, as types
template <int kV> struct Int {
    static constexpr int v = kV;
};
template <typename F> void with_short(uint64_t chunks, F f) {
    if (chunks <= 8) f(Int<8>(), Int<1>());
    else if (chunks <= 16) f(Int<16>(), Int<1>());
    else if (chunks <= 32) f(Int<16>(), Int<2>());
    else if (chunks <= 64) f(Int<32>(), Int<2>());
    else if (chunks <= 128) f(Int<64>(), Int<2>());
    else f(Int<64>(), Int<4>());
}

constexpr size_t kEntriesLds = 32768; // of a block of short rows

template <typename T, bool kHaveStats>
void launch_short(const DistillArgs &a, uint64_t rows, hipStream_t s) {
    const size_t row_bytes = kEntryBytes * (size_t)a.top;
    // At least as many lanes a row as leave a wavefront's rows that room for their
    // teacher's entries: 8 up to 341 of them, 16 up to 682, then 32 (20,000 rows of 20
    // floats at 8 lanes: 400 entries 186 -> 124 us, 700 550 -> 171, 1,024 1,470 -> 332).
    uint64_t chunks = chunks_of<T>(a.logits, a.stride, a.labels);
    if (64 / 16 * row_bytes > kEntriesLds) chunks = chunks > 33 ? chunks : 33;
    else if (64 / 8 * row_bytes > kEntriesLds) chunks = chunks > 9 ? chunks : 9;
    with_short(chunks, [&](auto lanes, auto held) {
        constexpr uint32_t kLanes = decltype(lanes)::v;
        uint32_t threads = 256; // fewer where the teacher's entries fill LDS
        while (threads > 64 && threads / kLanes * row_bytes > kEntriesLds) threads /= 2;
        const uint64_t per = threads / kLanes;
        hipLaunchKernelGGL((distill_short_kernel<T, kLanes, decltype(held)::v, kHaveStats>),
                           dim3((unsigned)((rows + per - 1) / per)), dim3(threads),
                           (unsigned)(per * row_bytes), s, a, rows);
    });
}

constexpr uint32_t kTile = 32768; // labels of a block of finish_kernel

template <typename T>
void launch_finish(const DistillArgs &a, uint64_t rows, const Part *parts, uint32_t slices,
                   hipStream_t s) {
    // where rows are few, as many blocks as the statistics had
    const uint32_t tile = slices > 1 ? ((a.labels + slices - 1) / slices + 7) / 8 * 8 : kTile;
    const uint32_t tiles = a.logits_grad ? (a.labels + tile - 1) / tile : 1;
    const auto kernel = past_caches<T>(rows, a.labels) ? finish_kernel<T, true> : finish_kernel<T, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(rows * tiles)), dim3(kStream), kEntryBytes * a.top, s,
                       a, tiles, a.logits_grad ? tile : a.labels, parts, slices);
}

template <typename T>
void launch_distill(const DistillArgs &a, uint64_t rows, const Slices &sl, Part *parts,
                    hipStream_t s) {
    const uint64_t chunks = chunks_of<T>(a.logits, a.stride, a.labels);
    if (chunks <= kShort) return launch_short<T, false>(a, rows, s);
    if (sl.count > 1) {
        hipLaunchKernelGGL(part_kernel<T>, dim3((unsigned)(rows * sl.count)), dim3(kStream), 0, s,
                           a, sl.count, sl.length, parts);
        return launch_finish<T>(a, rows, parts, sl.count, s);
    }
    const auto launch = [&](auto threads, auto held, auto past) {
        constexpr int kThreads = decltype(threads)::v;
        hipLaunchKernelGGL((distill_kernel<T, kThreads, decltype(held)::v, decltype(past)::v != 0>),
                           dim3((unsigned)rows), dim3(kThreads), kEntryBytes * a.top, s, a);
    };
    if (!a.logits_grad) {
        if (a.stats) return launch(Int<kStream>(), Int<0>(), Int<0>());
        return launch(Int<kStream>(), Int<0>(), Int<1>());
    }
    // The fewest held chunks that leave little to read again.
    const auto launch_held = [&](auto past) {
        if (chunks <= 256 * 4) launch(Int<256>(), Int<4>(), past);
        else if (chunks <= 512 * 4) launch(Int<512>(), Int<4>(), past);
        else if (chunks <= 512 * 9) launch(Int<512>(), Int<8>(), past);
        else if (chunks <= 512 * 13) launch(Int<512>(), Int<12>(), past);
        else launch(Int<512>(), Int<16>(), past);
    };
    if (past_caches<T>(rows, a.labels)) launch_held(Int<1>());
    else launch_held(Int<0>());
}

template <typename T>
void launch_answer(const AnswerArgs &a, uint64_t rows, const Slices &sl, void *scratch,
                   hipStream_t s) {
    const uint64_t chunks = chunks_of<T>(a.logits, a.stride, a.labels);
    if (chunks <= kShort) {
        with_short(chunks_of<T>(a.logits, a.stride, a.labels), [&](auto lanes, auto held) {
            constexpr uint32_t kLanes = decltype(lanes)::v;
            hipLaunchKernelGGL((answer_short_kernel<T, kLanes, decltype(held)::v>),
                               dim3((unsigned)((rows * kLanes + 255) / 256)), dim3(256), 0, s, a,
                               rows);
        });
        return;
    }
    uint64_t *keys = static_cast<uint64_t *>(scratch);
    Part *parts = reinterpret_cast<Part *>(keys + rows * sl.count * a.top);
    const auto kernel = a.stats ? answer_kernel<T, false> : answer_kernel<T, true>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(rows * sl.count)), dim3(kStream), 0, s, a, sl.count,
                       sl.length, parts, keys);
    if (sl.count > 1)
        hipLaunchKernelGGL(join_kernel<T>, dim3((unsigned)rows), dim3(kStream), 0, s, a, sl.count,
                           parts, keys);
}

template <typename T> void launch_answer_grad(const AnswerArgs &a, uint64_t rows, hipStream_t s) {
    const uint64_t chunks = chunks_of<T>(a.logits, a.stride, a.labels);
    const auto launch = [&](auto lanes) {
        constexpr uint32_t kLanes = decltype(lanes)::v;
        const uint32_t tile = kLanes == 256 ? 256 * Chunk<T>::kN * kUnroll : a.labels;
        const uint32_t tiles = (a.labels + tile - 1) / tile;
        const auto kernel = past_caches<T>(rows, a.labels) ? answer_grad_kernel<T, kLanes, true>
                                                           : answer_grad_kernel<T, kLanes, false>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((rows * tiles * kLanes + 255) / 256)), dim3(256),
                           0, s, a, rows, tiles, tile);
    };
    if (chunks <= 8 * kUnroll) launch(Int<8>());
    else if (chunks <= 64 * kUnroll) launch(Int<64>());
    else launch(Int<256>());
}

size_t align256(size_t x) { return (x + 255u) & ~(size_t)255u; }
size_t sum_bytes(uint64_t rows) {
    return align256(4 * rows) + (sum_blocks(rows) > 1 ? align256(8 * sum_blocks(rows)) : 0);
}

int check_logits(const char *what, int type, const void *logits, uint64_t rows, uint64_t labels,
                 int id_type, float temperature) {
    if (!known_type(type)) return fail(SDF_E_INVALID, "%s: unknown element type %d", what, type);
    if (!known_id_type(id_type)) return fail(SDF_E_INVALID, "%s: unknown id type %d", what, id_type);
    if (labels == 0 || labels >= (1ull << 31))
        return fail(SDF_E_INVALID, "%s takes 1 to 2^31 - 1 labels", what);
    if (rows >= (1ull << 31)) return fail(SDF_E_INVALID, "%s takes fewer than 2^31 rows", what);
    if (!(temperature >= 1.0e-38f) || temperature > 3.0e38f) // (1 / T is formed)
        return fail(SDF_E_INVALID, "%s: temperature must be positive and finite, as its reciprocal",
                    what);
    if (rows > 0 && !logits) return fail(SDF_E_INVALID, "NULL pointer argument");
    if ((reinterpret_cast<uintptr_t>(logits) & (type_bytes(type) - 1)) != 0)
        return fail(SDF_E_INVALID, "%s: logits must be aligned to their elements", what);
    return SDF_OK;
}

int check_distill(const char *what, int type, const void *logits, uint64_t rows, uint64_t labels,
                  int id_type, const void *teacher_labels, int teacher_type,
                  const void *teacher_logits, uint32_t top, float temperature, int reduction) {
    const int rc = check_logits(what, type, logits, rows, labels, id_type, temperature);
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

// the rows' losses and their blocks' sums where they are added up, and the Parts
// of slices
size_t sdf_distill_scratch_bytes(uint64_t rows, uint64_t labels, int reduction) {
    const Slices sl = slices_of(rows, labels, kDistillSlices);
    return (reduction == SDF_REDUCE_NONE ? 0 : sum_bytes(rows)) +
           (sl.count > 1 ? align256(rows * sl.count * sizeof(Part)) : 0);
}

int sdf_distill(int type, const void *logits, uint64_t rows, uint64_t labels, uint64_t stride,
                int id_type, const void *teacher_labels, int teacher_type,
                const void *teacher_logits, uint32_t top, float temperature,
                const float *row_weight, int reduction, const float *loss_grad, float *loss,
                float *stats, void *logits_grad, void *scratch, size_t scratch_bytes,
                void *stream) {
    const int rc = check_distill("distill", type, logits, rows, labels, id_type,
                                 teacher_labels, teacher_type, teacher_logits, top, temperature,
                                 reduction);
    if (rc != SDF_OK) return rc;
    if (!loss && (rows > 0 || reduction != SDF_REDUCE_NONE))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    const size_t need = sdf_distill_scratch_bytes(rows, labels, reduction);
    if (scratch_bytes < need || (need > 0 && !scratch))
        return fail(SDF_E_INVALID, "scratch must hold %zu bytes (got %zu)", need, scratch_bytes);
    if ((reinterpret_cast<uintptr_t>(scratch) & 255u) != 0)
        return fail(SDF_E_INVALID, "scratch must be 256-byte aligned");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool none = reduction == SDF_REDUCE_NONE;
    const float reduce = reduction == SDF_REDUCE_MEAN ? (float)(1.0 / (double)rows) : 1.0f;
    DistillArgs a = {logits, stride, (uint32_t)labels, id_type, teacher_labels, teacher_type,
                     teacher_logits, top, temperature, 1.0f / temperature * kLog2e, row_weight,
                     loss_grad, none ? 1u : 0u,
                     reduce, none ? loss : static_cast<float *>(scratch),
                     reinterpret_cast<float2 *>(stats), logits_grad};
    Part *parts = reinterpret_cast<Part *>(static_cast<char *>(scratch) +
                                           (none ? 0 : sum_bytes(rows)));
    const Slices sl = slices_of(rows, labels, kDistillSlices);
    with_type(type, [&](auto t) {
        for_windows(rows, [&](uint64_t r, uint64_t n) {
            launch_distill<decltype(t)>(from_row(a, type, r), n, sl, parts, s);
        });
    });
    if (!none)
        launch_loss_sum(a.loss, rows, reduce,
                        reinterpret_cast<double *>(static_cast<char *>(scratch) + align256(4 * rows)),
                        loss, s);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SDF_OK : hip_fail(e, "distill");
}

int sdf_distill_backward(int type, const void *logits, uint64_t rows, uint64_t labels,
                         uint64_t stride, int id_type, const void *teacher_labels,
                         int teacher_type, const void *teacher_logits, uint32_t top,
                         float temperature, const float *row_weight, int reduction,
                         const float *loss_grad, const float *stats, void *logits_grad,
                         void *stream) {
    const int rc = check_distill("distill_backward", type, logits, rows, labels, id_type,
                                 teacher_labels, teacher_type, teacher_logits, top, temperature,
                                 reduction);
    if (rc != SDF_OK) return rc;
    if (rows == 0) return SDF_OK;
    if (!loss_grad || !stats || !logits_grad) return fail(SDF_E_INVALID, "NULL pointer argument");
    const float reduce = reduction == SDF_REDUCE_MEAN ? (float)(1.0 / (double)rows) : 1.0f;
    DistillArgs a = {logits, stride, (uint32_t)labels, id_type, teacher_labels, teacher_type,
                     teacher_logits, top, temperature, 1.0f / temperature * kLog2e, row_weight,
                     loss_grad,
                     reduction == SDF_REDUCE_NONE ? 1u : 0u, reduce, nullptr,
                     reinterpret_cast<float2 *>(const_cast<float *>(stats)), logits_grad};
    with_type(type, [&](auto t) {
        using T = decltype(t);
        hipStream_t s = static_cast<hipStream_t>(stream);
        const bool is_short = chunks_of<T>(logits, stride, labels) <= kShort;
        for_windows(rows, [&](uint64_t r, uint64_t n) {
            const DistillArgs w = from_row(a, type, r);
            if (is_short) launch_short<T, true>(w, n, s);
            else launch_finish<T>(w, n, nullptr, 0, s);
        });
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SDF_OK : hip_fail(e, "distill_backward");
}

size_t sdf_label_log_probs_scratch_bytes(uint64_t rows, uint64_t labels, uint32_t top) {
    const Slices sl = slices_of(rows, labels, kMaxSlices);
    return sl.count > 1 ? align256(rows * sl.count * (sizeof(Part) + 8 * (size_t)top)) : 256;
}

int sdf_label_log_probs(int type, const void *logits, uint64_t rows, uint64_t labels,
                        uint64_t stride, int id_type, const void *label_ids, uint32_t top,
                        float temperature, float *log_prob, float *entropy, float *top_log_probs,
                        int64_t *top_labels, float *stats, void *scratch, size_t scratch_bytes,
                        void *stream) {
    const int rc = check_logits("label_log_probs", type, logits, rows, labels, id_type, temperature);
    if (rc != SDF_OK) return rc;
    if (top > kMaxTop)
        return fail(SDF_E_INVALID, "label_log_probs returns at most %u best labels", kMaxTop);
    if (rows == 0) return SDF_OK;
    if (!label_ids || !log_prob || !entropy || (top > 0 && (!top_log_probs || !top_labels)))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    const size_t need = sdf_label_log_probs_scratch_bytes(rows, labels, top);
    if (scratch_bytes < need || (need > 0 && !scratch))
        return fail(SDF_E_INVALID, "scratch must hold %zu bytes (got %zu)", need, scratch_bytes);
    if ((reinterpret_cast<uintptr_t>(scratch) & 255u) != 0)
        return fail(SDF_E_INVALID, "scratch must be 256-byte aligned");
    AnswerArgs a = {logits, stride, (uint32_t)labels, id_type, label_ids, top,
                    1.0f / temperature, 1.0f / temperature * kLog2e,
                    log_prob, entropy, top_log_probs, top_labels,
                    reinterpret_cast<float2 *>(stats), nullptr, nullptr, nullptr};
    with_type(type, [&](auto t) {
        const Slices sl = slices_of(rows, labels, kMaxSlices);
        for_windows(rows, [&](uint64_t r, uint64_t n) {
            launch_answer<decltype(t)>(from_row(a, type, r), n, sl, scratch,
                                       static_cast<hipStream_t>(stream));
        });
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SDF_OK : hip_fail(e, "label_log_probs");
}

int sdf_label_log_probs_backward(int type, const void *logits, uint64_t rows, uint64_t labels,
                                 uint64_t stride, int id_type, const void *label_ids,
                                 float temperature, const float *entropy, const float *stats,
                                 const float *log_prob_grad, const float *entropy_grad,
                                 void *logits_grad, void *stream) {
    const int rc = check_logits("label_log_probs_backward", type, logits, rows, labels, id_type,
                                temperature);
    if (rc != SDF_OK) return rc;
    if (rows == 0) return SDF_OK;
    if (!label_ids || !entropy || !stats || !logits_grad)
        return fail(SDF_E_INVALID, "NULL pointer argument");
    AnswerArgs a = {logits, stride, (uint32_t)labels, id_type, label_ids, 0,
                    1.0f / temperature, 1.0f / temperature * kLog2e, nullptr,
                    const_cast<float *>(entropy), nullptr, nullptr,
                    reinterpret_cast<float2 *>(const_cast<float *>(stats)), log_prob_grad,
                    entropy_grad, logits_grad};
    with_type(type, [&](auto t) {
        for_windows(rows, [&](uint64_t r, uint64_t n) {
            launch_answer_grad<decltype(t)>(from_row(a, type, r), n,
                                            static_cast<hipStream_t>(stream));
        });
    });
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? SDF_OK : hip_fail(e, "label_log_probs_backward");
}

} // extern "C"
