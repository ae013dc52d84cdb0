// Device pieces shared by the label-field kernels (cell_rows.hip,
// label_kernels.hip): element and id types, 16-byte pieces of rows, and sums over
// neighbouring lanes.
#pragma once

#include <cstddef>
#include <cstdint>

#include <hip/hip_runtime.h>

#include "../../include/sdfoam_hip.h"

namespace sdfoam_hip {

// sdf_last_error()'s message and `code` (capi.hip)
int fail(int code, const char *fmt, ...);
int hip_fail(hipError_t e, const char *where);

namespace label {

typedef _Float16 half_t;
typedef __bf16 bf16_t;

// f(a value of the element type) for SDF_TYPE_*; the caller has checked `type`
template <typename F> inline auto with_type(int type, F f) {
    if (type == SDF_TYPE_F16) return f(half_t());
    if (type == SDF_TYPE_BF16) return f(bf16_t());
    return f(float());
}

inline size_t type_bytes(int type) { return type == SDF_TYPE_F32 ? 4 : 2; }
inline bool known_type(int type) { return type >= SDF_TYPE_F32 && type <= SDF_TYPE_BF16; }
inline bool known_id_type(int type) { return type >= SDF_ID_U32 && type <= SDF_ID_I64; }

// The i-th id, or -1 where it does not lie in [0, limit) (limit < 2^31): no
// cell, no label.
__device__ __forceinline__ int32_t load_id(const void *ids, int id_type, uint64_t i,
                                           uint32_t limit) {
    if (id_type == SDF_ID_I64) {
        const uint64_t v = static_cast<const uint64_t *>(ids)[i];
        return v < limit ? (int32_t)v : -1;
    }
    const uint32_t v = static_cast<const uint32_t *>(ids)[i];
    return v < limit ? (int32_t)v : -1;
}

// 16 bytes of a row: kN elements, at any address that the element type allows
// (the hardware takes 16-byte accesses at element alignment).  Kept as it is in
// memory: as separate values, 16-bit elements would take a register each.
template <typename T> struct Chunk {
    static constexpr int kN = 16 / (int)sizeof(T);
    uint32_t w[4];
    __device__ __forceinline__ float operator[](int e) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
        else if constexpr (__is_same(T, bf16_t))
            return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
        else return (float)__builtin_bit_cast(half_t, bits(e));
    }
    __device__ __forceinline__ uint16_t bits(int e) const { // of a 16-bit element
        return (uint16_t)(e & 1 ? w[e / 2] >> 16 : w[e / 2]);
    }
    __device__ __forceinline__ T value(int e) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[e]);
        else return __builtin_bit_cast(T, bits(e));
    }
    __device__ __forceinline__ void set(int e, T x) {
        if constexpr (sizeof(T) == 4) w[e] = __float_as_uint(x);
        else {
            const uint32_t b = __builtin_bit_cast(uint16_t, x);
            w[e / 2] = e & 1 ? (w[e / 2] & 0xffffu) | b << 16 : (w[e / 2] & 0xffff0000u) | b;
        }
    }
};
template <typename T> __device__ __forceinline__ Chunk<T> load_chunk(const T *p) {
    Chunk<T> c;
    __builtin_memcpy(&c, p, 16);
    return c;
}
template <typename T> __device__ __forceinline__ void store_chunk(T *p, const Chunk<T> &c) {
    __builtin_memcpy(p, &c, 16);
}

// 16 bytes that are read or written once, past the caches, at the alignment of
// an element of kElement bytes.
template <int kElement> struct Past;
template <> struct Past<2> {
    typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
};
template <> struct Past<4> {
    typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(4)));
};
template <int kElement, typename V> __device__ __forceinline__ void store_past(void *p, const V &v) {
    static_assert(sizeof(V) == 16, "16 bytes");
    typename Past<kElement>::Words w;
    __builtin_memcpy(&w, &v, 16);
    __builtin_nontemporal_store(w, static_cast<typename Past<kElement>::Words *>(p));
}
template <typename V, int kElement> __device__ __forceinline__ V load_past(const void *p) {
    static_assert(sizeof(V) == 16, "16 bytes");
    const auto w =
        __builtin_nontemporal_load(static_cast<const typename Past<kElement>::Words *>(p));
    V v;
    __builtin_memcpy(&v, &w, 16);
    return v;
}

template <bool kOnce, typename T> __device__ __forceinline__ Chunk<T> load_chunk_if(const T *p) {
    if constexpr (kOnce) return load_past<Chunk<T>, sizeof(T)>(p);
    else return load_chunk(p);
}
template <bool kPast, typename T>
__device__ __forceinline__ void store_chunk_if(T *p, const Chunk<T> &c) {
    if constexpr (kPast) store_past<sizeof(T)>(p, c);
    else store_chunk(p, c);
}

// Elements [begin, end) of a row, cut into chunks at 16-byte boundaries: chunk
// `at` (begin, begin + kN, ...) has the elements [at, at + kN) moved down by
// `skew`, as far as they lie in the range.  (Rows of an odd number of 16-bit
// elements read at element alignment take 1.2 times as long.)  Memory is read
// and written in whole chunks inside the range: the first and the last begin
// where the range begins, or end where it ends (place()), and so share elements
// with their neighbours, which mask_chunk sets to `fill`.  A range shorter than
// two chunks goes element by element, unskewed.
template <typename T> struct Span {
    static constexpr uint32_t kN = Chunk<T>::kN;
    const T *row;
    uint32_t begin, end, skew;
    bool whole;
    // begin: a multiple of kN
    __device__ __forceinline__ Span(const T *r, uint32_t b, uint32_t e)
        : row(r), begin(b), end(e), whole(e - b >= 2 * kN) {
        skew = whole ? (uint32_t)(reinterpret_cast<uintptr_t>(r) & 15u) / (uint32_t)sizeof(T) : 0u;
    }
    __device__ __forceinline__ uint32_t last() const { return end + skew; } // chunks lie before it
    __device__ __forceinline__ uint32_t first_own(uint32_t at) const {
        return at == begin ? begin : at - skew;
    }
    __device__ __forceinline__ uint32_t end_own(uint32_t at) const {
        return min(at + kN - skew, end);
    }
    __device__ __forceinline__ uint32_t place(uint32_t at) const {
        return whole ? min(first_own(at), end - kN) : at;
    }
    // f(element of the chunk, element of the row) for the chunk's own elements
    template <typename F> __device__ __forceinline__ void each_own(uint32_t at, F f) const {
        const uint32_t from = place(at), lo = first_own(at), hi = end_own(at);
#pragma unroll
        for (uint32_t e = 0; e < kN; ++e)
            if (from + e >= lo && from + e < hi) f(e, from + e);
    }
    __device__ __forceinline__ bool plain(uint32_t at) const { // nothing shared with a neighbour
        return first_own(at) + kN <= end && (at != begin || skew == 0);
    }
    // steps of `count` chunk positions, all of them plain
    __device__ __forceinline__ bool plain_step(uint32_t first, uint32_t elements) const {
        return first + elements - skew <= end && (first != begin || skew == 0) && whole;
    }
    // unmasked; kOnce: past the caches
    template <bool kOnce = false>
    __device__ __forceinline__ Chunk<T> load(uint32_t at, T fill) const {
        if (whole) return load_chunk_if<kOnce>(row + place(at));
        Chunk<T> c = {};
#pragma unroll
        for (uint32_t e = 0; e < kN; ++e) c.set(e, at + e < end ? row[at + e] : fill);
        return c;
    }
    __device__ __forceinline__ void mask(Chunk<T> &c, uint32_t at, T fill) const {
        if (plain(at)) return;
        // elements [lo, hi) of the chunk are its own (lo >= hi: none)
        const uint32_t from = place(at);
        const uint32_t lo = min(first_own(at) - from, kN), hi = max(end_own(at), from) - from;
        const uint32_t own = hi > lo ? (1u << hi) - (1u << lo) : 0u; // hi <= kN
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (uint32_t e = 0; e < kN; ++e) c.w[e] = own >> e & 1u ? c.w[e] : __builtin_bit_cast(uint32_t, fill);
        } else {
            const uint32_t both = __builtin_bit_cast(uint16_t, fill) * 0x10001u;
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q) { // two elements' bits, as two masks of 16
                const uint32_t bits = own >> (2 * q);
                const uint32_t m = (bits & 1u ? 0xffffu : 0u) | (bits & 2u ? 0xffff0000u : 0u);
                c.w[q] = (c.w[q] & m) | (both & ~m);
            }
        }
    }
    // the chunk's own elements into another row
    template <bool kPast = false>
    __device__ __forceinline__ void store_own(T *to, uint32_t at, const Chunk<T> &c) const {
        if (plain(at)) store_chunk_if<kPast>(to + place(at), c);
        else each_own(at, [&](uint32_t e, uint32_t i) { to[i] = c.value(e); });
    }
};

// What a wavefront's lanes wrote to LDS before it, all of them see after it.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// x of the lane across: lanes of 2, 4, 8 and 16 meet through the VALU's own
// crossbar (quads by xor; eights and sixteens mirrored, which pairs up equal
// values once the smaller steps are done), 32 and 64 through LDS's.
template <int kStep> __device__ __forceinline__ uint32_t across(uint32_t x) {
    if constexpr (kStep == 1) return __builtin_amdgcn_update_dpp(0, x, 0xb1, 0xf, 0xf, true);
    else if constexpr (kStep == 2) return __builtin_amdgcn_update_dpp(0, x, 0x4e, 0xf, 0xf, true);
    else if constexpr (kStep == 4) return __builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, true);
    else if constexpr (kStep == 8) return __builtin_amdgcn_update_dpp(0, x, 0x140, 0xf, 0xf, true);
    else return (uint32_t)__shfl_xor((int)x, kStep);
}
template <int kStep> __device__ __forceinline__ float across(float x) {
    return __uint_as_float(across<kStep>(__float_as_uint(x)));
}

// op over the kLanes neighbouring lanes (a power of two), in every one of
// them; op must not depend on the order of its arguments.
template <int kLanes, typename V, typename F> __device__ __forceinline__ V group_all(V x, F op) {
    if constexpr (kLanes > 1) x = op(x, across<1>(x));
    if constexpr (kLanes > 2) x = op(x, across<2>(x));
    if constexpr (kLanes > 4) x = op(x, across<4>(x));
    if constexpr (kLanes > 8) x = op(x, across<8>(x));
    if constexpr (kLanes > 16) x = op(x, across<16>(x));
    if constexpr (kLanes > 32) x = op(x, across<32>(x));
    return x;
}
template <int kLanes> __device__ __forceinline__ float group_max(float x) {
    return group_all<kLanes>(x, [](float a, float b) { return fmaxf(a, b); });
}
template <int kLanes> __device__ __forceinline__ float group_sum(float x) {
    return group_all<kLanes>(x, [](float a, float b) { return a + b; });
}

} // namespace label
} // namespace sdfoam_hip
