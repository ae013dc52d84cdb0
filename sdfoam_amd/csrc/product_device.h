// Tiles of matrix products for rows in groups: what products.hip and adapters.hip run.
//
// Two forms, over 128 bytes of the inner dimension at a time (64 elements of 16 bits, 32
// floats), fp32 accumulators in the matrix units:
//
//   rows:     out[m, n] = sum_k a[m, k] b_g[n, k]   for the rows m of group g
//   weights:  out_g[m, n] = sum over rows k of group g of a[k, m] b[k, n]
//
// Either operand may lie with k along its rows or across them.  Large tiles keep it in LDS
// as memory has it and turn it when they read (Feed, Fragments); the narrow tiles of the
// adapters' ranks turn it on its way there (Along, Across).
#pragma once

#include "head_device.h"

namespace sdfoam_hip {
namespace head {

using namespace label;

typedef float F16x __attribute__((ext_vector_type(16)));
typedef float F4x __attribute__((ext_vector_type(4)));
typedef half_t H8 __attribute__((ext_vector_type(8)));
typedef bf16_t B8 __attribute__((ext_vector_type(8)));

// D[i][j] += sum over k of a's row i times b's row j, from 16 bytes a lane of each.  32x32:
// lane l has row l % 32 and chunk l / 32 of two; 16x16: row l % 16, chunk l / 16 of four.
// Element e of a lane's chunk meets element e of the other's, so it does not matter which
// k of the operands the chunks are, as long as both have the same.  Lane l gets column
// j = l % 32 (l % 16) and rows 8 (v / 4) + 4 (l / 32) + v % 4 (4 (l / 16) + v).
template <typename T> __device__ __forceinline__ void mma32(F16x &d, const Chunk<T> &a, const Chunk<T> &b) {
    if constexpr (__is_same(T, half_t))
        d = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), d, 0, 0, 0);
    else if constexpr (__is_same(T, bf16_t))
        d = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(B8, a), __builtin_bit_cast(B8, b), d, 0, 0, 0);
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) d = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], d, 0, 0, 0);
}
template <typename T> __device__ __forceinline__ void mma16(F4x &d, const Chunk<T> &a, const Chunk<T> &b) {
    if constexpr (__is_same(T, half_t))
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), d, 0, 0, 0);
    else if constexpr (__is_same(T, bf16_t))
        d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(B8, a), __builtin_bit_cast(B8, b), d, 0, 0, 0);
    else
#pragma unroll
        for (int e = 0; e < 4; ++e) d = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], d, 0, 0, 0);
}

// kN elements as they lie in memory, at any address that the element type allows.
template <typename T, int kN> struct Few {
    T v[kN];
};
template <typename T, int kN> __device__ __forceinline__ Few<T, kN> load_few(const T *p) {
    Few<T, kN> c;
    __builtin_memcpy(&c, p, sizeof(c));
    return c;
}
// the elements [0, have) of them, the others 0
template <typename T, int kN>
__device__ __forceinline__ Few<T, kN> load_some(const T *p, uint32_t have) {
    if (have >= kN) return load_few<T, kN>(p);
    Few<T, kN> c;
#pragma unroll
    for (uint32_t e = 0; e < kN; ++e) c.v[e] = e < have ? p[e] : (T)0.0f;
    return c;
}
template <typename T, int kN>
__device__ __forceinline__ void store_some(T *p, const Few<T, kN> &c, uint32_t have) {
    if (have >= kN) __builtin_memcpy(p, &c, sizeof(c));
    else
#pragma unroll
        for (uint32_t e = 0; e < kN - 1; ++e)
            if (e < have) p[e] = c.v[e];
}

// Rows of group g: [offsets[g], offsets[g + 1]); those behind the last group's are a group
// of their own, `groups`, whose rows of the result are 0.  offsets NULL: one group has all.
struct Groups {
    const int32_t *offsets;
    uint32_t groups;
    uint32_t total; // rows
    __device__ __forceinline__ uint32_t at(uint32_t g) const {
        const int32_t v = offsets[g]; // whatever the caller's array holds stays in range
        return v < 0 ? 0u : min((uint32_t)v, total);
    }
    __device__ __forceinline__ uint32_t begin(uint32_t g) const { return offsets ? at(g) : 0u; }
    __device__ __forceinline__ uint32_t end(uint32_t g) const {
        return !offsets || g == groups ? total : at(g + 1);
    }
};

struct TileOfRows {
    uint32_t group, first, rows; // rows [first, first + rows); group `groups`: none of them
};

// Tiles of kRows rows, counted group by group.  count(): of all groups; find(): the
// `tile`-th one.  Every thread of the block calls both; `lds` has room for 20 words.
template <int kRows, int kThreads> struct TilesOfRows {
    const Groups &g;
    uint32_t *lds;
    uint32_t lo, hi, before, sum; // a run of groups a thread, and the tiles before and in it
    __device__ __forceinline__ static uint32_t tiles(uint32_t b, uint32_t e) {
        return e > b ? (e - b + kRows - 1) / kRows : 0u;
    }
    __device__ __forceinline__ TilesOfRows(const Groups &groups, uint32_t *words)
        : g(groups), lds(words) {}
    __device__ __forceinline__ uint32_t count() {
        if (!g.offsets) return tiles(0, g.total);
        const uint32_t keys = g.groups + 1, each = (keys + kThreads - 1) / kThreads;
        lo = min(threadIdx.x * each, keys);
        hi = min(lo + each, keys);
        sum = 0;
        for (uint32_t k = lo; k < hi; ++k) sum += tiles(g.begin(k), g.end(k));
        const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        uint32_t run = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t v = __shfl_up(run, d);
            if ((int)lane >= d) run += v;
        }
        if (lane == 63) lds[wave] = run;
        __syncthreads();
        uint32_t all = 0;
        for (uint32_t w = 0; w < kThreads / 64; ++w) {
            if (w == wave) before = all + run - sum;
            all += lds[w];
        }
        return __builtin_amdgcn_readfirstlane(all); // the same in every lane
    }
    __device__ __forceinline__ TileOfRows find(uint32_t tile) {
        TileOfRows t;
        if (!g.offsets) {
            t.group = 0;
            t.first = tile * kRows;
            t.rows = min((uint32_t)kRows, g.total - t.first);
            return t;
        }
        if (tile >= before && tile - before < sum) {
            uint32_t left = tile - before;
            for (uint32_t k = lo; k < hi; ++k) {
                const uint32_t b = g.begin(k), e = g.end(k), n = tiles(b, e);
                if (left < n) {
                    lds[16] = k;
                    lds[17] = b + left * kRows;
                    lds[18] = min((uint32_t)kRows, e - (b + left * kRows));
                    break;
                }
                left -= n;
            }
        }
        __syncthreads();
        t.group = __builtin_amdgcn_readfirstlane(lds[16]);
        t.first = __builtin_amdgcn_readfirstlane(lds[17]);
        t.rows = __builtin_amdgcn_readfirstlane(lds[18]);
        return t;
    }
};
// no more tiles than this
inline uint64_t tiles_of_rows(uint64_t rows, uint32_t groups, bool grouped, uint32_t tile) {
    const uint64_t most = (rows + tile - 1) / tile;
    const uint64_t some = rows < (uint64_t)groups + 1 ? rows : (uint64_t)groups + 1;
    return grouped ? most + some : most;
}

struct Operand {
    const void *base;
    uint64_t stride;       // between rows
    uint64_t group_stride; // between the groups' matrices; 0: one for all
    const int32_t *index;  // the row at a place; NULL: the place itself
};

// What a row's adapter adds to its product: sum_r inner[place, r] outer_g[n, r], g the
// row's group (adapters.hip).
struct Beside {
    const float *inner; // [places][pitch]; NULL: nothing beside
    uint32_t rank, pitch;
    const void *outer; // [groups] of [n][rank], or across: [rank][n]
    uint64_t group_stride, stride;
    const int32_t *group_of; // of a place, -1: none
};

struct ProductArgs {
    Operand a, b;
    Groups groups;
    uint32_t m, n; // rows form: n alone; weights form: both
    uint32_t n_out; // narrow rows: columns written, those past n as 0 (at most as many tiles); 0: n
    uint32_t k;    // rows form
    uint32_t splits, k_each; // of the inner dimension; k_each: a multiple of 64
    bool parts;              // the sums go to `partial` and are joined from there
    void *out;
    uint64_t out_stride;
    const int32_t *out_index; // rows form: the row of the result for a place; NULL: itself
    float *partial;           // [split][rows or group m][n], unscaled
    float scale;              // narrow tiles and their joining; 1 for all others
    Beside beside;
    uint32_t tiles_n;
    uint32_t first; // tile of the launch
};

// ---- large tiles: LDS as memory has it ----------------------------------------------------
//
// kRows rows (along) or columns (across) of 128 bytes of k: as many bytes either way.  Each
// wave brings 1 KB at a time, 16 bytes a lane, straight into LDS where 16-byte pieces line
// up (kDirect), through registers where they do not.  LDS takes a wave's 16 bytes a lane in
// the order of the lanes, so the swizzle is in which piece a lane fetches:
//
//   along:  [row][128 bytes], piece c of row r at c ^ (r / 2 & 7): 16 rows' same piece on
//           all banks
//   across: [k][kRows], 16 bits: piece c of row k at c ^ 2 ((k & 3) + 4 (k / 8 & 1)), which
//           keeps the 8 rows that a transposing read takes at a time off each other's banks;
//           floats: at c ^ 8 (k / 4 & 1), for the two that a read of 64 words takes

__device__ const uint32_t kZeros[4] = {0, 0, 0, 0}; // what pieces past the end are read from

template <typename T> struct TileOf {
    static constexpr int kK = 128 / sizeof(T); // elements of k
    static constexpr int kC = 16 / sizeof(T);  // of a piece
};

// A wave's 16 bytes a lane to LDS from `at` (the same in every lane) on, on their way until
// the wave waits for its loads (landed()).  As an instruction of its own: were it a builtin,
// the compiler would wait for it before every read of LDS that it cannot tell apart.
__device__ __forceinline__ void to_lds(const void *from, uint32_t at) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "{m0}"(at), "v"(from) : "memory");
}
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }
__device__ __forceinline__ uint32_t lds_address(const char *p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)p;
}

template <typename T, bool kAcross, int kRows, int kWaves, bool kDirect> struct Feed {
    static constexpr int kPer = kRows / 8 / kWaves; // pieces a lane
    static constexpr int kC = TileOf<T>::kC, kK = TileOf<T>::kK;
    static constexpr int kRowBytes = kAcross ? kRows * (int)sizeof(T) : 128;
    const T *p[kPer];
    uint64_t stride;
    uint32_t columns; // across: from the tile's first column on
    bool tiny;        // rows of less than a piece
    Chunk<T> c[kDirect ? 1 : kPer];

    // where in the tile the lane's j-th piece lies: its row of LDS and its place there
    __device__ __forceinline__ static uint32_t wave() {
        return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    }
    __device__ __forceinline__ static uint32_t lds_row(int j) {
        return ((wave() * kPer + j) * 1024u + (threadIdx.x & 63u) * 16u) / kRowBytes;
    }
    __device__ __forceinline__ static uint32_t swizzle(uint32_t row) {
        if constexpr (!kAcross) return row >> 1 & 7u;
        else if constexpr (sizeof(T) == 2) return ((row & 3u) | (row >> 3 & 1u) << 2) << 1;
        else return (row >> 2 & 1u) << 3;
    }
    __device__ __forceinline__ static uint32_t piece(int j) {
        return (((threadIdx.x & 63u) * 16u) % kRowBytes / 16u) ^ swizzle(lds_row(j));
    }

    // along: rows [first, first + rows), by the operand's index; across: columns from `first`
    // of `rows` in all.  length: elements of a row.
    __device__ __forceinline__ void begin(const Operand &o, uint64_t group, uint32_t first,
                                          uint32_t rows, uint32_t k0, uint32_t length) {
        const T *base = static_cast<const T *>(o.base) + group * o.group_stride;
        stride = o.stride;
        columns = kAcross ? rows - first : rows;
        tiny = length < kC;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if constexpr (!kAcross) {
                const uint32_t r = first + min(lds_row(j), rows - 1);
                p[j] = base + (uint64_t)(o.index ? (uint32_t)o.index[r] : r) * stride + k0 + piece(j) * kC;
            } else {
                p[j] = base + (uint64_t)(k0 + lds_row(j)) * stride + first + piece(j) * kC;
            }
        }
    }

    // how many elements of the lane's j-th piece of the tile at k there are, or more
    __device__ __forceinline__ uint32_t there(int j, uint32_t k, uint32_t end) const {
        if constexpr (!kAcross) {
            const uint32_t at = k + piece(j) * kC;
            return end > at ? end - at : 0u;
        } else {
            const uint32_t at = k + lds_row(j), n = piece(j) * kC;
            return at < end && n < columns ? columns - n : 0u;
        }
    }

    // of the tile at k, the lane's pieces; k0 as in begin().  A piece that the row's end cuts
    // is read where it ends there and moved down (store()): every piece is one read, without a
    // branch (element by element, the waits of the cut pieces held up all others: TN of 8,192
    // rows of 1,000 x 5,003 bf16 182 TFLOP/s).
    __device__ __forceinline__ void load(char *lds, uint32_t k, uint32_t k0, uint32_t end) {
        const uint64_t on = kAcross ? (uint64_t)(k - k0) * stride : k - k0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const T *from = p[j] + on;
            const uint32_t have = there(j, k, end);
            if constexpr (kDirect) {
                to_lds(have ? static_cast<const void *>(from) : kZeros,
                       lds_address(lds) + (wave() * kPer + j) * 1024u);
            } else if (tiny) {
                c[j] = __builtin_bit_cast(Chunk<T>, load_some<T, kC>(from, have));
            } else {
                const void *at = have >= kC ? from : have ? from - (kC - have) : static_cast<const void *>(kZeros);
                __builtin_memcpy(&c[j], at, 16);
            }
        }
    }
    __device__ __forceinline__ void store(char *lds, uint32_t k, uint32_t end) {
        if constexpr (!kDirect)
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const uint32_t have = there(j, k, end);
                const bool cut = !tiny && have > 0 && have < kC;
                if (__ballot(cut)) { // the piece ends with the elements that there are: down with them
                    typedef unsigned __int128 U128;
                    const U128 all = __builtin_bit_cast(U128, c[j]);
                    if (cut) c[j] = __builtin_bit_cast(Chunk<T>, all >> ((kC - have) * 8 * sizeof(T)));
                }
                *reinterpret_cast<uint4 *>(lds + (wave() * kPer + j) * 1024u + (threadIdx.x & 63u) * 16u) =
                    __builtin_bit_cast(uint4, c[j]);
            }
    }
};

// Fragments of 32 rows (columns) from `first` (a multiple of 64; of 128 for more than two)
// on, of the 32 bytes of k at step kk.  What the swizzle changes with i or kk are bits that
// nothing else has: one address each.
template <typename T, bool kAcross, int kRows, int kFragments> struct Fragments {
    static constexpr int kRowBytes = kAcross ? kRows * (int)sizeof(T) : 128;
    static constexpr int kAt = kAcross ? kFragments : 4;
    uint32_t at[kAt];
    __device__ __forceinline__ explicit Fragments(uint32_t first) {
        const uint32_t lane = threadIdx.x & 63u, half = lane >> 5, q = lane & 15u;
#pragma unroll
        for (uint32_t i = 0; i < kAt; ++i) {
            if constexpr (!kAcross) {
                at[i] = (first + (lane & 31u)) * 128u + (((2u * i + half) ^ (lane >> 1 & 7u)) << 4);
            } else if constexpr (sizeof(T) == 2) {
                // 16 lanes read 4 rows k of 16 columns; each gets its column's 4
                const uint32_t n = first + i * 32u + (lane >> 4 & 1u) * 16u + (q & 3u) * 4u;
                at[i] = (half * 8u + (q >> 2)) * kRowBytes +
                        (((n >> 3) ^ (((q >> 2) | half << 2) << 1)) << 4) + (n & 7u) * 2u;
            } else {
                const uint32_t n = first + i * 32u + (lane & 31u);
                at[i] = half * 4u * kRowBytes + (((n >> 2) ^ half << 3) << 4) + (n & 3u) * 4u;
            }
        }
    }
    __device__ __forceinline__ Chunk<T> read(const char *lds, int i, int kk) const {
        Chunk<T> c;
        if constexpr (!kAcross) {
            c = __builtin_bit_cast(Chunk<T>, *reinterpret_cast<const uint4 *>(lds + at[kk] + i * 4096u));
        } else if constexpr (sizeof(T) == 2) {
            typedef short S4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) S4 LdsS4;
            S4 v[2];
#pragma unroll
            for (int s = 0; s < 2; ++s)
                v[s] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (LdsS4 *)(lds + at[i] + (kk * 16 + s * 4) * kRowBytes));
            __builtin_memcpy(&c, v, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                c.w[e] = *reinterpret_cast<const uint32_t *>(lds + at[i] + (kk * 8 + e) * kRowBytes);
        }
        return c;
    }
};

// ---- narrow tiles: turned on their way to LDS ---------------------------------------------
//
// The tile in LDS always has k along its rows, so that every wave reads its fragments as 16
// bytes a lane.  Chunk c of row r lies at c ^ ((r ^ r >> 3) & 7), which keeps reads (32 rows,
// the same chunk) and turned writes (every 4th or 8th row) off each other's banks.
__device__ __forceinline__ uint32_t place_in_lds(uint32_t row, uint32_t chunk) {
    return row * 128u + ((chunk ^ ((row ^ row >> 3) & 7u)) << 4);
}

// kRows rows with k along them: 8 threads a row.  Rows past the end repeat the last (what
// becomes of them is not stored).
template <typename T, int kRows, int kThreads> struct Along {
    static constexpr int kPer = kRows * 8 / kThreads;
    const T *row[kPer];
    Chunk<T> c[kPer];
    __device__ __forceinline__ void begin(const Operand &o, uint64_t group, uint32_t first,
                                          uint32_t rows) {
        const T *base = static_cast<const T *>(o.base) + group * o.group_stride;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const uint32_t r = first + min(threadIdx.x / 8 + j * (kThreads / 8), rows - 1);
            row[j] = base + (uint64_t)(o.index ? (uint32_t)o.index[r] : r) * o.stride;
        }
    }
    __device__ __forceinline__ void load(uint32_t k0, uint32_t end) {
        const uint32_t k = k0 + (threadIdx.x & 7u) * TileOf<T>::kC;
        if (k0 + TileOf<T>::kK <= end) {
#pragma unroll
            for (int j = 0; j < kPer; ++j) c[j] = load_chunk(row[j] + k);
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                c[j] = __builtin_bit_cast(Chunk<T>, load_some<T, TileOf<T>::kC>(
                                                        row[j] + k, end > k ? end - k : 0u));
        }
    }
    __device__ __forceinline__ void store(char *lds) const {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            *reinterpret_cast<uint4 *>(
                lds + place_in_lds(threadIdx.x / 8 + j * (kThreads / 8), threadIdx.x & 7u)) =
                __builtin_bit_cast(uint4, c[j]);
    }
};

// kRows columns of rows k of type S: a thread has 4 rows k by as many columns as 16 bytes
// hold of the wider type, and turns them.  Rows and columns past the end are 0.
template <typename T, typename S, int kRows, int kThreads> struct Across {
    static constexpr int kN = TileOf<T>::kC;      // columns a thread
    static constexpr int kAcross = kRows / kN;    // threads across
    static constexpr int kTasks = kAcross * (TileOf<T>::kK / 4);
    static constexpr int kPer = (kTasks + kThreads - 1) / kThreads;
    const S *base;
    uint64_t stride;
    const int32_t *index;
    uint32_t columns, first;
    Few<S, kN> c[kPer][4];
    __device__ __forceinline__ void begin(const Operand &o, uint64_t group, uint32_t first_column,
                                          uint32_t all_columns) {
        base = static_cast<const S *>(o.base) + group * o.group_stride;
        stride = o.stride;
        index = o.index;
        first = first_column;
        columns = all_columns;
    }
    __device__ __forceinline__ void load(uint32_t k0, uint32_t end) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const uint32_t task = threadIdx.x + j * kThreads;
            if (kTasks % kThreads && task >= kTasks) break;
            const uint32_t n = first + task % kAcross * kN, k = k0 + task / kAcross * 4;
            const uint32_t have = n < columns ? columns - n : 0u;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                if (k + i < end && have) {
                    const uint64_t r = index ? (uint32_t)index[k + i] : k + i;
                    c[j][i] = load_some<S, kN>(base + r * stride + n, have);
                } else {
                    c[j][i] = {};
                }
            }
        }
    }
    __device__ __forceinline__ void store(char *lds) const {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const uint32_t task = threadIdx.x + j * kThreads;
            if (kTasks % kThreads && task >= kTasks) break;
            const uint32_t n = task % kAcross * kN, k = task / kAcross * 4;
#pragma unroll
            for (uint32_t e = 0; e < kN; ++e) {
                Few<T, 4> t;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (__is_same(T, S)) t.v[i] = c[j][i].v[e];
                    else t.v[i] = (T)(float)c[j][i].v[e];
                }
                *reinterpret_cast<Few<T, 4> *>(lds + place_in_lds(n + e, k * sizeof(T) / 16) +
                                               k * sizeof(T) % 16) = t;
            }
        }
    }
};

} // namespace head
} // namespace sdfoam_hip
