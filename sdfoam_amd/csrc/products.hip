// Products of rows in groups with the groups' matrices, and their gradients:
//
//   out[p, :]     = rows[p, :] weight_g^T          for the places p of group g
//   rows_grad     = out_grad[p, :] weight_g
//   weight_grad_g = sum over p of group g of out_grad[p, :]^T rows[p, :]
//
// and the same for low-rank adapters beside a shared matrix (adapters.hip).  Accumulators
// are fp32 in the matrix units (16-bit operands by 32x32x16, floats by 32x32x2), rounded to
// the output's type once.
#include "products.h"

using namespace sdfoam_hip;
using namespace sdfoam_hip::label;
using namespace sdfoam_hip::head;

namespace {

template <bool kAcross, typename T, typename S, int kRows, int kThreads> struct LoaderOf {
    typedef Along<T, kRows, kThreads> type;
};
template <typename T, typename S, int kRows, int kThreads>
struct LoaderOf<true, T, S, kRows, kThreads> {
    typedef Across<T, S, kRows, kThreads> type;
};

// What the rows' adapters add to 32 rows of kTn x 32 columns from n0 on, in one of two ways:
// by the matrix units, one adapter of the 32 rows' after the other, where they have few
// (add_beside; a lane has row m0 + mi, as the accumulators do), and for each row by itself
// where they have many (beside_of_rows).  One after the other, each waits for its values: 200
// rows, an adapter each, of 2,048 -> 32,768 bf16 and rank 16 took 247 us, 48 without them.
// Microseconds by the matrix units and row by row, 4,096 rows of 512 -> 2,048 bf16 in order,
// with 1, 3, 4 and 8 adapters in 32 rows: rank 8 37 and 70, 45 and 71, 52 and 77, 66 and 83;
// rank 64 49 and 637, 81 and 639, 106 and 649, 213 and 690.  At these sizes the two meet at
// more adapters than the limit.
constexpr uint32_t kFewAdapters = 3;
__device__ __forceinline__ bool few_adapters(int32_t mine) {
    uint64_t left = __ballot(mine >= 0);
#pragma unroll
    for (uint32_t k = 0; k < kFewAdapters; ++k)
        if (left) left &= ~__ballot(mine == __builtin_amdgcn_readlane(mine, __ffsll((long long)left) - 1));
    return left == 0;
}

// Column n of kRows rows from `place` on (the last of `rows` again where there are fewer),
// their values on their way together; the rows are the same in every lane, `groups` has
// theirs from lane `from` on.  Every lane of the wave calls it.
template <typename S, bool kAcross, int kRows>
__device__ __forceinline__ void beside_of_rows(const ProductArgs &p, uint32_t place, uint32_t rows,
                                               int32_t groups, uint32_t from, uint32_t n, float *sum) {
    const S *outer[kRows];
    const float *inner[kRows];
    bool some[kRows];
#pragma unroll
    for (uint32_t i = 0; i < kRows; ++i) {
        const uint32_t at = place + min(i, rows - 1);
        const int32_t g = __builtin_amdgcn_readlane(groups, from + min(i, rows - 1));
        some[i] = g >= 0;
        outer[i] = static_cast<const S *>(p.beside.outer) + (uint64_t)max(g, 0) * p.beside.group_stride +
                   (kAcross ? n : (uint64_t)n * p.beside.stride);
        inner[i] = p.beside.inner + (uint64_t)at * p.beside.pitch;
        sum[i] = 0.0f;
    }
    constexpr uint32_t kE = 8;
    for (uint32_t r = 0; r < p.beside.rank; r += kE) { // inner is 0 past the rank
        const uint32_t have = p.beside.rank - r;
        Few<S, kE> o[kRows];
#pragma unroll
        for (uint32_t i = 0; i < kRows; ++i) {
            if constexpr (kAcross) {
#pragma unroll
                for (uint32_t e = 0; e < kE; ++e)
                    o[i].v[e] = e < have ? outer[i][(uint64_t)(r + e) * p.beside.stride] : (S)0.0f;
            } else {
                o[i] = load_some<S, kE>(outer[i] + r, have);
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kRows; ++i)
#pragma unroll
            for (uint32_t e = 0; e < kE; ++e) sum[i] = fmaf((float)o[i].v[e], inner[i][r + e], sum[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < kRows; ++i)
        if (!some[i]) sum[i] = 0.0f;
}

template <typename S, bool kAcross, int kTn>
__device__ __forceinline__ void add_beside(const ProductArgs &p, uint32_t m0, uint32_t rows,
                                           uint32_t mi, int32_t mine, uint32_t n0, F16x *acc) {
    const uint32_t lane = threadIdx.x & 63u, l32 = lane & 31u, half = lane >> 5;
    const uint32_t place = m0 + min(mi, rows - 1);
    uint64_t left = __ballot(mine >= 0);
    const float *inner = p.beside.inner + (uint64_t)place * p.beside.pitch + half * 4;
    while (left) {
        const int32_t g = __builtin_amdgcn_readlane(mine, __ffsll((long long)left) - 1);
        left &= ~__ballot(mine == g);
        const S *outer = static_cast<const S *>(p.beside.outer) + (uint64_t)g * p.beside.group_stride;
        F16x extra[kTn] = {};
        for (uint32_t r = 0; r < p.beside.rank; r += 8) {
            const uint32_t r0 = r + half * 4;
            const uint32_t have = p.beside.rank > r0 ? p.beside.rank - r0 : 0u;
            const Few<float, 4> h = load_few<float, 4>(inner + r);
#pragma unroll
            for (int j = 0; j < kTn; ++j) {
                const uint32_t n = n0 + j * 32 + l32;
                Few<S, 4> o = {};
                if (n < p.n) {
                    if constexpr (kAcross) {
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e)
                            if (e < have) o.v[e] = outer[(uint64_t)(r0 + e) * p.beside.stride + n];
                    } else {
                        o = load_some<S, 4>(outer + (uint64_t)n * p.beside.stride + r0, have);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    extra[j] = __builtin_amdgcn_mfma_f32_32x32x2f32((float)o.v[e], h.v[e], extra[j], 0, 0, 0);
            }
        }
        // its own rows alone: another adapter's values, NaN among them, stay out
        if (mine == g)
#pragma unroll
            for (int j = 0; j < kTn; ++j) acc[j] += extra[j];
    }
}

// A wave's 32 rows of kTn x 32 columns from n0 on, turned in LDS of its own (a lane has one
// row, l32, and runs of 4 columns) to be written in pieces of 16 bytes side by side.  Rows
// [0, rows) are written, the l32-th to row_at(to_row of lane l32).
template <int kTn> constexpr uint32_t turn_bytes() { return 32 * (kTn * 32 * 4 + 16); }

template <typename O, int kTn, typename RowAt>
__device__ __forceinline__ void write_rows(const ProductArgs &p, char *turn, const F16x *sums, uint32_t rows,
                                           uint32_t n0, int32_t to_row, RowAt row_at) {
    constexpr uint32_t kE = 16 / sizeof(O), kPieces = kTn * 32 / kE;
    constexpr uint32_t kBytes = kTn * 32 * sizeof(O) + 16;
    const uint32_t lane = threadIdx.x & 63u, l32 = lane & 31u, half = lane >> 5;
    wave_sync();
#pragma unroll
    for (int j = 0; j < kTn; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t n = j * 32 + q * 8 + half * 4;
            Few<O, 4> o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o.v[e] = (O)sums[j][q * 4 + e];
            *reinterpret_cast<Few<O, 4> *>(turn + l32 * kBytes + n * sizeof(O)) = o;
        }
    wave_sync();
#pragma unroll
    for (uint32_t t = 0; t < kPieces / 2; ++t) {
        const uint32_t at = t * 64 + lane, r = at / kPieces, n = at % kPieces * kE;
        const O *from = reinterpret_cast<const O *>(turn + r * kBytes) + n;
        const int32_t row = __shfl(to_row, r);
        if (r >= rows || n0 + n >= p.n) continue;
        O *to = row_at(row) + n0 + n;
        const uint32_t have = p.n - (n0 + n);
        if (have >= kE) __builtin_memcpy(to, from, 16);
        else
#pragma unroll 1
            for (uint32_t e = 0; e < have; ++e) to[e] = from[e];
    }
}

// The same with the rows' adapters added one by one; a lane has a column.  The first row is
// at `place`, lane l32 has the l32-th row's adapter.  Lanes past the last column stay to the
// end, with that column's values: the rows that the others write to are read from them.
template <typename S, bool kAcross, typename O, int kTn, typename RowAt>
__device__ __forceinline__ void write_by_row(const ProductArgs &p, char *turn, const F16x *sums, uint32_t place,
                                             uint32_t rows, uint32_t n0, int32_t to_row, int32_t adapters,
                                             RowAt row_at) {
    static_assert(kTn * 32 == 64, "a lane for each column");
    constexpr uint32_t kFloats = kTn * 32 + 4;
    const uint32_t lane = threadIdx.x & 63u, l32 = lane & 31u, half = lane >> 5;
    float *turned = reinterpret_cast<float *>(turn);
    wave_sync();
#pragma unroll
    for (int j = 0; j < kTn; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            Few<float, 4> o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o.v[e] = sums[j][q * 4 + e];
            *reinterpret_cast<Few<float, 4> *>(turned + l32 * kFloats + j * 32 + q * 8 + half * 4) = o;
        }
    wave_sync();
    if (n0 >= p.n) return; // all lanes of the wave
    const uint32_t n = n0 + lane;
    constexpr uint32_t kBatch = 4;
    for (uint32_t r = 0; r < rows; r += kBatch) {
        float extra[kBatch];
        beside_of_rows<S, kAcross, kBatch>(p, place + r, rows - r, adapters, r, min(n, p.n - 1), extra);
#pragma unroll
        for (uint32_t i = 0; i < kBatch; ++i) {
            if (r + i >= rows) break;
            const int32_t row = __builtin_amdgcn_readlane(to_row, r + i);
            if (n < p.n) row_at(row)[n] = (O)(turned[(r + i) * kFloats + lane] + extra[i]);
        }
    }
}

constexpr uint32_t kXcds = 8;
// Blocks go to the XCDs in turn; of `tiles_m` x tiles_n tiles each XCD takes a run, kGroup
// tiles of rows by all of the columns at a time, so that its L2 holds what its blocks share.
__device__ __forceinline__ void tile_of_block(uint32_t block, uint32_t tiles_m, uint32_t tiles_n,
                                              uint32_t &tile_m, uint32_t &tile_n) {
    constexpr uint32_t kGroup = 4;
    const uint32_t each = tiles_m * tiles_n / kXcds;
    const uint32_t at = block < each * kXcds ? (block % kXcds) * each + block / kXcds : block;
    const uint32_t group = at / (kGroup * tiles_n);
    const uint32_t rows = min(kGroup, tiles_m - group * kGroup), in = at - group * kGroup * tiles_n;
    tile_m = group * kGroup + in % rows;
    tile_n = in / rows;
}

// One tile of kM x kN, kWavesM x kWavesN waves: two tiles of the inner dimension in LDS,
// one multiplied while the other is brought.  Bound by the matrix units: 8,192^3 bf16 in
// tiles of 256 x 256 at 1,145 TFLOP/s with both operands along k, 1,164 with b across, 1,125
// with both (a large library product: 1,390, 1,310, 1,150), in tiles of 128 x 128 at 854;
// 4,096^3 floats at 140 (131).  At rows that do not line up a third to a half of that.  Read
// in pairs of words for want of alignment, LDS alone took as long: 550.
template <typename T, bool kWeights, bool kAcrossB, int kM, int kN, int kWavesM, int kWavesN, bool kDirect>
__global__ __launch_bounds__(64 * kWavesM * kWavesN, 2) void tile_kernel(ProductArgs p) {
    constexpr int kWaves = kWavesM * kWavesN, kBlock = 64 * kWaves;
    constexpr int kTm = kM / kWavesM / 32, kTn = kN / kWavesN / 32, kK = TileOf<T>::kK;
    constexpr uint32_t kTile = (kM + kN) * 128;
    constexpr uint32_t kTurn = turn_bytes<kTn>();
    __shared__ __attribute__((aligned(16))) char lds[2 * kTile];
    __shared__ uint32_t found[20];
    Feed<T, kWeights, kM, kWaves, kDirect> a;
    Feed<T, kWeights || kAcrossB, kN, kWaves, kDirect> b;

    uint32_t tile_m, tile_n;
    const uint32_t split = blockIdx.y, block = p.first + blockIdx.x;
    uint32_t k_begin = 0, k_end = p.k, group, m0, rows_m, n0;
    if constexpr (kWeights) {
        const uint32_t tiles_m = (p.m + kM - 1) / kM;
        // every XCD has a share of each group, whose rows differ in number
        group = block / (tiles_m * p.tiles_n);
        tile_of_block(block - group * tiles_m * p.tiles_n, tiles_m, p.tiles_n, tile_m, tile_n);
        n0 = tile_n * kN;
        m0 = tile_m * kM;
        rows_m = min((uint32_t)kM, p.m - m0);
        k_begin = __builtin_amdgcn_readfirstlane(p.groups.begin(group));
        k_end = __builtin_amdgcn_readfirstlane(max(p.groups.end(group), k_begin));
        // each split a share of the group's rows
        const uint32_t each = ((k_end - k_begin + p.splits - 1) / p.splits + 63u) & ~63u;
        const uint32_t from = min(k_begin + split * each, k_end);
        k_end = min(from + each, k_end);
        k_begin = from;
        a.begin(p.a, 0, m0, p.m, k_begin, p.m);
        b.begin(p.b, 0, n0, p.n, k_begin, p.n);
    } else {
        TilesOfRows<kM, kBlock> tiles(p.groups, found);
        const uint32_t tiles_m = tiles.count();
        if (block >= tiles_m * p.tiles_n) return; // left over
        tile_of_block(block, tiles_m, p.tiles_n, tile_m, tile_n);
        const TileOfRows t = tiles.find(tile_m);
        n0 = tile_n * kN;
        group = t.group;
        m0 = t.first;
        rows_m = t.rows;
        if (p.groups.offsets && group == p.groups.groups) { // rows of no group: zeros
            group = 0;
            k_end = 0;
        } else if (p.splits > 1) {
            k_begin = min(split * p.k_each, p.k);
            k_end = min(k_begin + p.k_each, p.k);
        }
        const uint64_t which = p.b.group_stride ? group : 0;
        a.begin(p.a, 0, m0, rows_m, k_begin, p.k);
        b.begin(p.b, which, n0, kAcrossB ? p.n : min((uint32_t)kN, p.n - n0), k_begin, kAcrossB ? p.n : p.k);
    }

    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t wm = wave % kWavesM * (kTm * 32), wn = wave / kWavesM * (kTn * 32);
    const uint32_t l32 = lane & 31u;
    F16x acc[kTm][kTn] = {};
    // what the end needs of the rows, on its way meanwhile: where each goes, its adapter
    int32_t groups[kTm], goes_to[kTm];
    if constexpr (!kWeights)
#pragma unroll
        for (int i = 0; i < kTm; ++i) {
            const uint32_t mi = wm + i * 32 + l32, place = m0 + min(mi, rows_m - 1);
            groups[i] = p.beside.inner && split == 0 && mi < rows_m ? p.beside.group_of[place] : -1;
            goes_to[i] = p.out_index && !p.parts ? p.out_index[place] : (int32_t)place;
        }
    const Fragments<T, kWeights, kM, kTm> of_a(wm);
    const Fragments<T, kWeights || kAcrossB, kN, kTn> of_b(wn);
    if (k_begin < k_end) {
        const auto bring = [&](char *to, uint32_t k) {
            a.load(to, k, k_begin, k_end);
            b.load(to + kM * 128, k, k_begin, k_end);
        };
        const auto brought = [&](char *to, uint32_t k) {
            a.store(to, k, k_end);
            b.store(to + kM * 128, k, k_end);
            if (kDirect) landed();
            __syncthreads();
        };
        bring(lds, k_begin);
        brought(lds, k_begin);
        uint32_t now = 0;
        for (uint32_t k = k_begin; k < k_end; k += kK) {
            const bool more = k + kK < k_end;
            if (more) bring(lds + (now ^ kTile), k + kK);
            const char *from = lds + now;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                Chunk<T> fa[kTm], fb[kTn];
#pragma unroll
                for (int j = 0; j < kTn; ++j) fb[j] = of_b.read(from + kM * 128, j, kk);
#pragma unroll
                for (int i = 0; i < kTm; ++i) fa[i] = of_a.read(from, i, kk);
#pragma unroll
                for (int i = 0; i < kTm; ++i)
#pragma unroll
                    for (int j = 0; j < kTn; ++j) mma32<T>(acc[i][j], fb[j], fa[i]);
            }
            now ^= kTile;
            if (more) brought(lds + now, k + kK);
        }
        __syncthreads();
    }

    static_assert(kWaves * kTurn <= sizeof(lds), "room for each wave");
    char *turn = lds + wave * kTurn;
    const uint64_t rows = kWeights ? (uint64_t)p.groups.groups * p.m : p.groups.total;
    uint32_t by_row = 0; // bit i: its rows' adapters are added row by row
    if constexpr (!kWeights)
        if (p.beside.inner && split == 0)
#pragma unroll
            for (int i = 0; i < kTm; ++i) {
                if (few_adapters(groups[i]))
                    add_beside<T, kAcrossB, kTn>(p, m0, rows_m, wm + i * 32 + l32, groups[i], n0 + wn, acc[i]);
                else by_row |= 1u << i;
            }
#pragma unroll
    for (int i = 0; i < kTm; ++i) {
        const uint32_t first = wm + i * 32;
        int32_t to_row = (int32_t)(m0 + first + l32), adapters = -1; // of the lane's row
        if constexpr (!kWeights) to_row = goes_to[i], adapters = groups[i];
        const uint32_t left = first < rows_m ? min(32u, rows_m - first) : 0u; // of the 32 rows
        if (p.parts) {
            const auto row_at = [&](int32_t row) {
                return p.partial + (split * rows + (kWeights ? (uint64_t)group * p.m : 0) + (uint32_t)row) * p.n;
            };
            if (!kWeights && (by_row >> i & 1u))
                write_by_row<T, kAcrossB, float, kTn>(p, turn, acc[i], m0 + first, left, n0 + wn, to_row, adapters, row_at);
            else write_rows<float, kTn>(p, turn, acc[i], left, n0 + wn, to_row, row_at);
        } else {
            const auto row_at = [&](int32_t row) {
                return static_cast<T *>(p.out) + ((kWeights ? (uint64_t)group * p.m : 0) + (uint32_t)row) * p.out_stride;
            };
            if (!kWeights && (by_row >> i & 1u))
                write_by_row<T, kAcrossB, T, kTn>(p, turn, acc[i], m0 + first, left, n0 + wn, to_row, adapters, row_at);
            else write_rows<T, kTn>(p, turn, acc[i], left, n0 + wn, to_row, row_at);
        }
    }
}

constexpr int kThreads = 256;

// ---- narrow tiles: the adapters' ranks ---------------------------------------------------
//
// One tile of kM x kN of the result, kWavesM x kWavesN waves; operands of other types than T
// are converted on their way.  Two tiles of the inner dimension in LDS: while one is
// multiplied, the next is on its way to registers.  Bound by the waits for the long operand:
// h of 160,000 rows of 64 fp16 13 us, b of 8,192 rows of 5,003 36, up's gradient 77.
//
// kWeights: the weights form (both operands across, k the rows of a group); else the rows
// form, b across for gradients.
template <typename T, typename SA, typename SB, bool kWeights, bool kAcrossB, int kM, int kN,
          int kWavesM, int kWavesN, typename O>
__global__ __launch_bounds__(kThreads) void product_kernel(ProductArgs p) {
    constexpr int kTm = kM / kWavesM / 32, kTn = kN / kWavesN / 32;
    __shared__ __attribute__((aligned(16))) char lds[2][(kM + kN) * 128];
    __shared__ uint32_t found[20];
    typename LoaderOf<kWeights, T, SA, kM, kThreads>::type a;
    typename LoaderOf<kWeights || kAcrossB, T, SB, kN, kThreads>::type b;

    const uint32_t block = p.first + blockIdx.x, split = blockIdx.y;
    const uint32_t tile_n = block % p.tiles_n, tile_m = block / p.tiles_n;
    const uint32_t n0 = tile_n * kN;
    uint32_t k_begin = 0, k_end = p.k, group, m0, rows_m;
    if constexpr (kWeights) {
        const uint32_t tiles_m = (p.m + kM - 1) / kM;
        group = tile_m / tiles_m;
        m0 = tile_m % tiles_m * kM;
        rows_m = min((uint32_t)kM, p.m - m0);
        k_begin = __builtin_amdgcn_readfirstlane(p.groups.begin(group));
        k_end = __builtin_amdgcn_readfirstlane(max(p.groups.end(group), k_begin));
        // each split a share of the group's rows
        const uint32_t each = ((k_end - k_begin + p.splits - 1) / p.splits + 63u) & ~63u;
        const uint32_t from = min(k_begin + split * each, k_end);
        k_end = min(from + each, k_end);
        k_begin = from;
        a.begin(p.a, 0, m0, p.m);
        b.begin(p.b, 0, n0, p.n);
    } else {
        TilesOfRows<kM, kThreads> tiles(p.groups, found);
        if (tile_m >= tiles.count()) return;
        const TileOfRows t = tiles.find(tile_m);
        group = t.group;
        m0 = t.first;
        rows_m = t.rows;
        if (p.groups.offsets && group == p.groups.groups) { // rows of no group: zeros
            group = 0;
            k_end = 0;
        } else if (p.splits > 1) {
            k_begin = min(split * p.k_each, p.k);
            k_end = min(k_begin + p.k_each, p.k);
        }
        const uint64_t which = p.b.group_stride ? group : 0;
        a.begin(p.a, 0, m0, rows_m);
        if constexpr (kAcrossB) b.begin(p.b, which, n0, p.n);
        else b.begin(p.b, which, n0, min((uint32_t)kN, p.n - n0));
    }

    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t wm = wave % kWavesM * (kTm * 32), wn = wave / kWavesM * (kTn * 32);
    const uint32_t l32 = lane & 31u, half = lane >> 5;
    F16x acc[kTm][kTn] = {};
    if (k_begin < k_end) {
        a.load(k_begin, k_end);
        b.load(k_begin, k_end);
        a.store(lds[0]);
        b.store(lds[0] + kM * 128);
        __syncthreads();
        int at = 0;
        for (uint32_t k = k_begin; k < k_end; k += TileOf<T>::kK) {
            const bool more = k + TileOf<T>::kK < k_end;
            if (more) {
                a.load(k + TileOf<T>::kK, k_end);
                b.load(k + TileOf<T>::kK, k_end);
            }
            const char *la = lds[at], *lb = lds[at] + kM * 128;
#pragma unroll
            for (uint32_t c = 0; c < 8; c += 2) {
                Chunk<T> fa[kTm], fb[kTn];
#pragma unroll
                for (int i = 0; i < kTm; ++i)
                    fa[i] = __builtin_bit_cast(Chunk<T>, *reinterpret_cast<const uint4 *>(la + place_in_lds(wm + i * 32 + l32, c + half)));
#pragma unroll
                for (int j = 0; j < kTn; ++j)
                    fb[j] = __builtin_bit_cast(Chunk<T>, *reinterpret_cast<const uint4 *>(lb + place_in_lds(wn + j * 32 + l32, c + half)));
#pragma unroll
                for (int i = 0; i < kTm; ++i)
#pragma unroll
                    for (int j = 0; j < kTn; ++j) mma32<T>(acc[i][j], fb[j], fa[i]);
            }
            if (more) {
                at ^= 1;
                a.store(lds[at]);
                b.store(lds[at] + kM * 128);
                __syncthreads();
            }
        }
    }

    // a lane has one row of the result (l32) and runs of 4 columns of it
#pragma unroll
    for (int i = 0; i < kTm; ++i) {
        const uint32_t mi = wm + i * 32 + l32;
        if (mi >= rows_m) continue;
        const uint64_t row = kWeights ? (uint64_t)group * p.m + m0 + mi : m0 + mi;
#pragma unroll
        for (int j = 0; j < kTn; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t n = n0 + wn + j * 32 + q * 8 + half * 4;
                if (n >= p.n_out) continue;
                if (p.parts) {
                    Few<float, 4> sum;
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum.v[e] = acc[i][j][q * 4 + e];
                    const uint64_t rows = kWeights ? (uint64_t)p.groups.groups * p.m : p.groups.total;
                    store_some<float, 4>(p.partial + (split * rows + row) * p.n_out + n, sum, p.n_out - n);
                } else {
                    Few<O, 4> o; // 0 past n, at any scale
#pragma unroll
                    for (int e = 0; e < 4; ++e) o.v[e] = (O)(n + e < p.n ? p.scale * acc[i][j][q * 4 + e] : 0.0f);
                    store_some<O, 4>(static_cast<O *>(p.out) + (p.out_index ? (uint32_t)p.out_index[row] : row) * p.out_stride + n,
                                     o, p.n_out - n);
                }
            }
    }
}

// The parts' sums in order.  rows x n floats a part; four columns a thread.
template <typename O> __global__ __launch_bounds__(256) void join_kernel(ProductArgs p, uint64_t rows) {
    const uint32_t quads = (p.n_out + 3) / 4;
    const uint64_t t = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint64_t row = t / quads;
    if (row >= rows) return;
    const uint32_t n = (uint32_t)(t % quads) * 4, have = p.n_out - n;
    float sum[4] = {};
    for (uint32_t s = 0; s < p.splits; ++s) {
        const Few<float, 4> v = load_some<float, 4>(p.partial + (s * rows + row) * p.n_out + n, have);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += v.v[e];
    }
    O *to = static_cast<O *>(p.out) + (p.out_index ? (uint32_t)p.out_index[row] : row) * p.out_stride + n;
    Few<O, 4> o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o.v[e] = (O)(n + e < p.n ? p.scale * sum[e] : 0.0f);
    store_some<O, 4>(to, o, have);
}

// The same with what the rows' adapters add, where the tiles left that out (Plan::late): a
// column a thread, so that neighbours read neighbouring values (four columns a thread, 128
// bytes from one lane to the next: 152 us for 200 rows of 32,768 and rank 16).
template <typename O, bool kAcross> __global__ __launch_bounds__(256) void join_late_kernel(ProductArgs p) {
    const uint32_t row = blockIdx.y, n = blockIdx.x * 256 + threadIdx.x;
    if (n >= p.n) return;
    float sum = 0.0f, extra = 0.0f;
    for (uint32_t s = 0; s < p.splits; ++s) sum += p.partial[((uint64_t)s * gridDim.y + row) * p.n + n];
    const int32_t g = p.beside.group_of[row];
    if (g >= 0) {
        const O *outer = static_cast<const O *>(p.beside.outer) + (uint64_t)g * p.beside.group_stride;
        const float *inner = p.beside.inner + (uint64_t)row * p.beside.pitch;
        if constexpr (kAcross) {
#pragma unroll 16
            for (uint32_t r = 0; r < p.beside.rank; ++r)
                extra = fmaf((float)outer[(uint64_t)r * p.beside.stride + n], inner[r], extra);
        } else {
            constexpr uint32_t kE = 8;
#pragma unroll 4
            for (uint32_t r = 0; r < p.beside.rank; r += kE) { // inner is 0 past the rank
                const Few<O, kE> o = load_some<O, kE>(outer + (uint64_t)n * p.beside.stride + r, p.beside.rank - r);
#pragma unroll
                for (uint32_t e = 0; e < kE; ++e) extra = fmaf((float)o.v[e], inner[r + e], extra);
            }
        }
    }
    static_cast<O *>(p.out)[(p.out_index ? (uint32_t)p.out_index[row] : row) * p.out_stride + n] = (O)(sum + extra);
}

// ---- a short inner dimension -------------------------------------------------------------
//
// At most 128 bytes of it: a wave keeps 32 rows in registers and goes over the columns, 64 at
// a time, their fragments from the caches while the 64 before are written, without LDS but to
// turn what it writes and without waiting for another wave.  Bound by the waits for columns
// and the VALU's share of conversions and addresses (160,000 rows of 64 -> 512 fp16, other
// rows each time: 63 us, with adapters 79; tiles, which wait in turn for rows, columns and
// each other, 76 and 88).  Microseconds on the same rows again and again, tiles after: 10^6
// rows of 64 -> 512 fp16 323 and 391, of 32 -> 64 floats 113 and 162; 160,000 of 16 -> 64 fp16
// 14 and 17; but where the caches hold the result and it is wider, 64 -> 512 67 and 57, 64 ->
// 256 39 and 30, of 32 -> 201 floats 65 and 57.
constexpr uint32_t kShortWaves = 4, kShortRows = 32 * kShortWaves;

template <typename T> __global__ __launch_bounds__(64 * kShortWaves, 3) void short_kernel(ProductArgs p, uint32_t columns) {
    constexpr uint32_t kC = TileOf<T>::kC, kPieces = 4;
    __shared__ __attribute__((aligned(16))) char turns[kShortWaves * turn_bytes<2>()];
    __shared__ uint32_t found[20];
    TilesOfRows<kShortRows, 64 * kShortWaves> tiles(p.groups, found);
    const uint32_t block = p.first + blockIdx.x;
    if (block >= tiles.count()) return;
    const TileOfRows t = tiles.find(block);
    const bool none = p.groups.offsets && t.group == p.groups.groups; // rows of no group: zeros
    const uint32_t lane = threadIdx.x & 63u, l32 = lane & 31u, half = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (wave * 32 >= t.rows) return;
    const uint32_t m0 = t.first + wave * 32, rows = min(32u, t.rows - wave * 32), k_all = none ? 0u : p.k;
    char *turn = turns + wave * turn_bytes<2>();
    const uint32_t place = m0 + min(l32, rows - 1);
    // pieces 2 kk + half of a row, of zeros past the end
    const auto pieces = [&](const T *row, Chunk<T> *c) {
#pragma unroll
        for (uint32_t kk = 0; kk < kPieces; ++kk) {
            const uint32_t at = (2 * kk + half) * kC;
            c[kk] = __builtin_bit_cast(Chunk<T>, load_some<T, kC>(row + at, k_all > at ? k_all - at : 0u));
        }
    };
    const T *w = static_cast<const T *>(p.b.base) + (none ? 0u : t.group) * p.b.group_stride;
    const uint32_t from = blockIdx.y * columns, to = min(from + columns, p.n);
    Chunk<T> fa[kPieces], fb[2][kPieces];
    pieces(static_cast<const T *>(p.a.base) + (uint64_t)(p.a.index ? (uint32_t)p.a.index[place] : place) * p.a.stride, fa);
    const auto bring = [&](uint32_t n0) {
#pragma unroll
        for (int j = 0; j < 2; ++j) pieces(w + (uint64_t)min(n0 + j * 32 + l32, p.n - 1) * p.b.stride, fb[j]);
    };
    bring(from);
    const int32_t group = p.beside.inner && l32 < rows ? p.beside.group_of[place] : -1;
    const int32_t goes_to = p.out_index ? p.out_index[place] : (int32_t)place;
    const bool few = few_adapters(group);
    for (uint32_t n0 = from; n0 < to; n0 += 64) {
        F16x acc[2] = {};
#pragma unroll
        for (uint32_t kk = 0; kk < kPieces; ++kk)
#pragma unroll
            for (int j = 0; j < 2; ++j) mma32<T>(acc[j], fb[j][kk], fa[kk]);
        if (n0 + 64 < to) bring(n0 + 64);
        const auto row_at = [&](int32_t row) { return static_cast<T *>(p.out) + (uint32_t)row * p.out_stride; };
        if (few) {
            if (p.beside.inner) add_beside<T, false, 2>(p, m0, rows, l32, group, n0, acc);
            write_rows<T, 2>(p, turn, acc, rows, n0, goes_to, row_at);
        } else {
            write_by_row<T, false, T, 2>(p, turn, acc, m0, rows, n0, goes_to, group, row_at);
        }
    }
}

// ---- few rows a group --------------------------------------------------------------------
//
// 16 kMt rows by 16 kNt columns a block; each of four waves has a quarter of the inner
// dimension and reads its operands straight into registers, 128 bytes of a row at a time,
// since no other wave of the block needs them.  Bound by the bytes of the matrices; the
// rows come from L2, as often as there are tiles of columns (64 rows of 2,048 -> 32,768: 60 us,
// tiles 44; 32 rows: 44 both; 16: 37; the 64 entries of 16 rows over 64 experts of 1,024 ->
// 2,048 bf16, 171 MB: 30 us, 5.6 TB/s).
constexpr int kThinWaves = 4;

template <typename T, int kMt, int kNt>
__global__ __launch_bounds__(64 * kThinWaves) void thin_kernel(ProductArgs p) {
    constexpr uint32_t kC = TileOf<T>::kC, kStep = TileOf<T>::kK; // a lane has two pieces a step
    // steps asked for together; of their loads the compiler keeps some in flight: 16 bits,
    // tiles of 16 x 16 eight, of 16 x 32 three, of 32 x 32 four; floats two to four
    constexpr int kAhead = kMt * kNt <= 2 ? 4 : 2;
    __shared__ F4x sums[kThinWaves][kMt * kNt][64];
    __shared__ uint32_t found[20];
    const uint32_t block = p.first + blockIdx.x, tile_n = block % p.tiles_n, tile_m = block / p.tiles_n;
    TilesOfRows<16 * kMt, 64 * kThinWaves> tiles(p.groups, found);
    if (tile_m >= tiles.count()) return;
    const TileOfRows t = tiles.find(tile_m);
    const bool none = p.groups.offsets && t.group == p.groups.groups; // rows of no group: zeros
    const uint32_t k_all = none ? 0u : p.k, n0 = tile_n * (16 * kNt);
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, l16 = lane & 15u, q = lane >> 4;
    const T *x[kMt], *w[kNt];
#pragma unroll
    for (int i = 0; i < kMt; ++i) {
        const uint32_t r = t.first + min(i * 16 + l16, t.rows - 1);
        x[i] = static_cast<const T *>(p.a.base) + (uint64_t)(p.a.index ? (uint32_t)p.a.index[r] : r) * p.a.stride;
    }
#pragma unroll
    for (int j = 0; j < kNt; ++j)
        w[j] = static_cast<const T *>(p.b.base) + (none ? 0u : t.group) * p.b.group_stride +
               (uint64_t)min(n0 + j * 16 + l16, p.n - 1) * p.b.stride;
    const uint32_t steps = (k_all + kStep - 1) / kStep, each = (steps + kThinWaves - 1) / kThinWaves;
    const uint32_t k_begin = min(wave * each * kStep, k_all), k_end = min(k_begin + each * kStep, k_all);
    F4x acc[kMt][kNt] = {};
    uint32_t k = k_begin;
    for (; k + kAhead * kStep <= k_end; k += kAhead * kStep) {
        Chunk<T> fx[kAhead][kMt][2], fw[kAhead][kNt][2];
#pragma unroll
        for (int s = 0; s < kAhead; ++s)
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                const uint32_t at = k + s * kStep + (q * 2 + h) * kC;
#pragma unroll
                for (int j = 0; j < kNt; ++j) fw[s][j][h] = load_chunk(w[j] + at);
#pragma unroll
                for (int i = 0; i < kMt; ++i) fx[s][i][h] = load_chunk(x[i] + at);
            }
#pragma unroll
        for (int s = 0; s < kAhead; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < kMt; ++i)
#pragma unroll
                    for (int j = 0; j < kNt; ++j) mma16<T>(acc[i][j], fw[s][j][h], fx[s][i][h]);
    }
    for (; k < k_end; k += kStep)
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            const uint32_t at = k + (q * 2 + h) * kC, have = k_end > at ? k_end - at : 0u;
            Chunk<T> fx[kMt], fw[kNt];
#pragma unroll
            for (int j = 0; j < kNt; ++j) fw[j] = __builtin_bit_cast(Chunk<T>, load_some<T, kC>(w[j] + at, have));
#pragma unroll
            for (int i = 0; i < kMt; ++i) fx[i] = __builtin_bit_cast(Chunk<T>, load_some<T, kC>(x[i] + at, have));
#pragma unroll
            for (int i = 0; i < kMt; ++i)
#pragma unroll
                for (int j = 0; j < kNt; ++j) mma16<T>(acc[i][j], fw[j], fx[i]);
        }
#pragma unroll
    for (int i = 0; i < kMt; ++i)
#pragma unroll
        for (int j = 0; j < kNt; ++j) sums[wave][i * kNt + j][lane] = acc[i][j];
    __syncthreads();
    // an element of the result a thread, its row's adapter read for it alone: of few rows
    // each has its own, as often as not
#pragma unroll 4
    for (uint32_t c = 0; c < kMt * kNt; ++c) {
        const uint32_t at = c * 256 + threadIdx.x, m = at / (16 * kNt), nn = at % (16 * kNt), n = n0 + nn;
        if (m >= t.rows || n >= p.n) continue;
        const uint32_t place = t.first + m;
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < kThinWaves; ++v)
            sum += sums[v][m / 16 * kNt + nn / 16][m % 16 + nn % 16 / 4 * 16][nn % 4];
        const int32_t g = p.beside.inner ? p.beside.group_of[place] : -1;
        if (g >= 0) {
            const T *outer = static_cast<const T *>(p.beside.outer) + (uint64_t)g * p.beside.group_stride +
                             (uint64_t)n * p.beside.stride;
            const float *h = p.beside.inner + (uint64_t)place * p.beside.pitch;
            float extra = 0.0f;
#pragma unroll 2
            for (uint32_t r = 0; r < p.beside.rank; r += kC) { // h is 0 past the rank
                const Few<T, kC> o = load_some<T, kC>(outer + r, p.beside.rank - r);
                const Few<float, kC> hr = load_few<float, kC>(h + r);
#pragma unroll
                for (uint32_t e = 0; e < kC; ++e) extra = fmaf((float)o.v[e], hr.v[e], extra);
            }
            sum += extra;
        }
        const uint64_t row = p.out_index ? (uint32_t)p.out_index[place] : place;
        static_cast<T *>(p.out)[row * p.out_stride + n] = (T)sum;
    }
}

constexpr uint64_t kMaxTiles = 1ull << 31; // 32 bits count them

// f(p, tiles) for windows of the tiles: a launch holds fewer than 2^32 threads
template <typename F> void each_window(ProductArgs p, uint64_t tiles, F f) {
    constexpr uint64_t kWindow = 1ull << 22;
    for (uint64_t t = 0; t < tiles; t += kWindow) {
        p.first = (uint32_t)t;
        f(p, (uint32_t)(tiles - t < kWindow ? tiles - t : kWindow));
    }
}

// whether rows of n elements are whole pieces of 16 bytes wherever one begins
bool lines_up(const Operand &o, int type, uint32_t n) {
    const size_t e = type_bytes(type);
    return reinterpret_cast<uintptr_t>(o.base) % 16 == 0 && o.stride * e % 16 == 0 &&
           o.group_stride * e % 16 == 0 && n * e % 16 == 0;
}

template <typename T, bool kWeights, bool kAcross, bool kDirect>
void launch_tiles_as(const ProductArgs &args, const Plan &plan, hipStream_t s) {
    each_window(args, plan.tiles, [&](const ProductArgs &p, uint32_t tiles) {
        const dim3 grid(tiles, plan.splits);
        if (plan.large) tile_kernel<T, kWeights, kAcross, 256, 256, 2, 4, kDirect><<<grid, 512, 0, s>>>(p);
        else tile_kernel<T, kWeights, kAcross, 128, 128, 2, 2, kDirect><<<grid, 256, 0, s>>>(p);
    });
}
template <typename T, bool kWeights, bool kAcross>
void launch_tiles(const ProductArgs &p, const Plan &plan, bool direct, hipStream_t s) {
    if (direct) launch_tiles_as<T, kWeights, kAcross, true>(p, plan, s);
    else launch_tiles_as<T, kWeights, kAcross, false>(p, plan, s);
}

template <typename T> void launch_thin(const ProductArgs &args, const Plan &plan, hipStream_t s) {
    const uint32_t block = 64 * kThinWaves;
    each_window(args, plan.tiles, [&](const ProductArgs &p, uint32_t tiles) {
        switch (plan.thin_m * 8 + plan.thin_n) {
        case 9: thin_kernel<T, 1, 1><<<tiles, block, 0, s>>>(p); break;
        case 10: thin_kernel<T, 1, 2><<<tiles, block, 0, s>>>(p); break;
        case 17: thin_kernel<T, 2, 1><<<tiles, block, 0, s>>>(p); break;
        default: thin_kernel<T, 2, 2><<<tiles, block, 0, s>>>(p); break;
        }
    });
}

// a wave keeps its rows; a share of the columns each, so many that the chip has waves enough
template <typename T> void launch_short(const ProductArgs &args, hipStream_t s) {
    const uint64_t all =
        tiles_of_rows(args.groups.total, args.groups.groups, args.groups.offsets != nullptr, kShortRows);
    const uint64_t shares = 2048 / all + 1, steps = (args.n + 63) / 64;
    const uint32_t columns = 64 * (uint32_t)((steps + shares - 1) / shares);
    each_window(args, all, [&](const ProductArgs &p, uint32_t tiles) {
        const dim3 grid(tiles, (p.n + columns - 1) / columns);
        short_kernel<T><<<grid, 64 * kShortWaves, 0, s>>>(p, columns);
    });
}

// tiles of the adapters' ranks: kM x kN
template <typename T, typename SA, typename SB, bool kWeights, bool kAcross, int kM, int kN, int kWavesM,
          int kWavesN, typename O>
void launch_narrow(const ProductArgs &args, const Plan &plan, hipStream_t s) {
    each_window(args, plan.tiles, [&](const ProductArgs &p, uint32_t tiles) {
        product_kernel<T, SA, SB, kWeights, kAcross, kM, kN, kWavesM, kWavesN, O>
            <<<dim3(tiles, plan.splits), kThreads, 0, s>>>(p);
    });
}

template <typename O> hipError_t join(const ProductArgs &p, uint64_t rows, hipStream_t s) {
    const uint64_t threads = rows * ((p.n_out + 3) / 4);
    join_kernel<O><<<(uint32_t)((threads + 255) / 256), 256, 0, s>>>(p, rows);
    return hipGetLastError();
}

} // namespace

namespace sdfoam_hip {
namespace head {

// Whether tiles of 256 x 256, one a CU, take less time than tiles of 128 x 128, two a CU:
// a round of the small ones takes two thirds of one of the large (bf16 8,192^3 by large
// tiles 1,095 TFLOP/s, by small ones 854; 8,192 x 2,112 x 8,192 642 and 639).
bool take_large(uint64_t large, uint64_t small) {
    return 3 * ((large + 255) / 256) <= 2 * ((small + 511) / 512);
}

Plan plan_rows(uint64_t rows, uint32_t groups, bool grouped, uint32_t n, uint32_t k, bool across,
               bool skinny) {
    Plan plan = {};
    const uint64_t each = grouped && groups > 0 ? (rows + groups - 1) / groups : rows;
    // Microseconds of thin and of large tiles, 4,096 -> 4,096: 16 rows bf16 12 and 19, floats 24
    // and 64; 32 rows 20 and 20, 38 and 66.  8 rows each of 16 experts, 1,024 -> 2,048 bf16 16 and
    // 17, 32 rows each 21 and 18 (floats 37 and 73); 32 rows of 2,048 -> 32,768 bf16 35 and 29, 48
    // rows 57 and 29.
    if (!skinny && !across && each <= 32) {
        plan.thin_m = each <= 16 ? 1 : 2;
        const uint64_t tiles_m = tiles_of_rows(rows, groups, grouped, 16 * plan.thin_m);
        // Wider where there are columns enough for every CU: the rows are read less often.
        // Microseconds at 32 columns and at 16, bf16: 16 rows of 4,096 -> 32,768 54 and 63, 64
        // entries over 64 experts of 1,024 -> 2,048 43 and 45, one row of 4,096 -> 4,096 13 and 9;
        // 32 rows of 4,096 -> 4,096 20 and 16 (128 tiles of 32), -> 6,144 20 and 26, -> 8,192 20
        // and 26 (256 tiles).
        plan.thin_n = plan.thin_m;
        if (plan.thin_n < 2 && tiles_m * (n / 32) >= 1024) plan.thin_n = 2;
        while (plan.thin_n > 1 && tiles_m * ((n + 16 * plan.thin_n - 1) / (16 * plan.thin_n)) < 256)
            plan.thin_n /= 2;
        plan.tiles_n = (n + 16 * plan.thin_n - 1) / (16 * plan.thin_n);
        plan.tiles = tiles_m * plan.tiles_n;
        plan.splits = 1;
        return plan;
    }
    // as many as there are on average: a group's last tile is half full
    const auto tiles = [&](uint64_t tile) {
        const uint64_t halves = grouped ? 2 * ((rows + tile - 1) / tile) + (rows < groups ? rows : groups) - 1
                                        : 2 * ((rows + tile - 1) / tile);
        return halves / 2 * ((n + tile - 1) / tile);
    };
    // not at a short inner dimension, where they gain little: 4,096 rows of 320 -> 4,096 bf16
    // take 21 us by large tiles and 24 by small ones, of 256 20 and 22, of 128 16 and 18
    plan.large = !skinny && k > 256 && rows > 0 && take_large(tiles(256), tiles(128));
    const uint32_t km = plan.large ? 256 : 128, kn = skinny ? 32 : km;
    plan.tiles_n = (n + kn - 1) / kn;
    plan.tiles = tiles_of_rows(rows, groups, grouped, km) * plan.tiles_n;
    // Few tiles: the inner dimension in several parts, of 512 elements at least, until the
    // chip has a block for each of its places.  Microseconds in parts and whole, 128 rows of
    // 4,096 -> 4,096: bf16 22 and 46, floats 67 and 265; with 256 and 1,024 blocks bf16 31 and 24,
    // floats 141 and 82.  512 rows bf16 41 and 47; 1,024 rows (256 tiles) whole 50, in parts 63.
    // Parts of 256, 512 and 1,024 elements, 64 rows of 2,048 -> 2,048: bf16 15, 15 and 18, floats
    // 29, 43 and 74.  Skinny ones wait for memory, in shorter parts: the gradients of 64 adapters
    // of rank 16, 1,024 rows of 2,048 -> 2,048 bf16, take 53, with b and h whole 96, in parts of
    // 128 62, of 512 57.
    plan.splits = 1;
    if (plan.tiles > 0 && !plan.large && plan.tiles < (skinny ? 768 : 256)) {
        const uint64_t want = (skinny ? 1536 : 512) / plan.tiles, most = k / (skinny ? 256 : 512);
        plan.splits = (uint32_t)(want < most ? want : most);
        if (plan.splits < 1) plan.splits = 1;
    }
    plan.k_each = ((k + plan.splits - 1) / plan.splits + 63) / 64 * 64;
    plan.bytes = plan.splits > 1 ? round_up(plan.splits * rows * n * 4) : 0;
    return plan;
}

Plan plan_weights(uint64_t rows, uint32_t groups, uint32_t m, uint32_t n, bool narrow_m, bool narrow_n) {
    Plan plan = {};
    plan.large = !narrow_m && !narrow_n &&
                 take_large((uint64_t)groups * ((m + 255) / 256) * ((n + 255) / 256),
                            (uint64_t)groups * ((m + 127) / 128) * ((n + 127) / 128));
    const uint32_t km = narrow_m ? 32 : plan.large ? 256 : 128, kn = narrow_n ? 32 : plan.large ? 256 : 128;
    plan.tiles_n = (n + kn - 1) / kn;
    plan.tiles = (uint64_t)groups * ((m + km - 1) / km) * plan.tiles_n;
    plan.splits = 1;
    // Parts of 512 rows at least, and blocks for two rounds of places.  Microseconds in parts
    // and whole, 65,536 rows of 512 x 512: bf16 93 and 657 (512 blocks 83, 2,048 132), floats 293
    // and 4,171; 8 experts of 1,024 rows, 1,024 x 1,024 bf16 (512 tiles) in parts 48, whole 25.
    // Narrow ones wait for memory more than they multiply: more blocks, shorter parts.  The
    // gradients of 12 adapters of rank 8, 8,192 rows of 1,000 -> 5,003 bf16, take 175 us; with
    // the narrow products whole 256, in parts of 192 rows at least 190, of 48 178, in half as
    // many blocks 189; 8 of rank 16, 4,096 -> 4,096, 217, whole 324, 192 rows 187.
    const bool narrow = narrow_m || narrow_n;
    if (plan.tiles > 0 && !plan.large && plan.tiles < (narrow ? 768 : 400)) {
        const uint64_t want = (narrow ? 1536 : 1024) / plan.tiles, most = rows / groups / (narrow ? 96 : 512);
        plan.splits = (uint32_t)(want < most ? want : most);
        if (plan.splits < 1) plan.splits = 1;
    }
    plan.bytes = plan.splits > 1 ? round_up((uint64_t)plan.splits * groups * m * n * 4) : 0;
    return plan;
}

Plan late(Plan plan, uint64_t rows, uint32_t n) {
    if (plan.thin_m || plan.late) return plan;
    plan.late = true;
    plan.bytes = round_up(plan.splits * rows * n * 4);
    return plan;
}

hipError_t product_rows(int type, const ProductArgs &args, const Plan &plan, bool across, bool skinny,
                        bool out_float, hipStream_t s) {
    if (plan.tiles == 0) return hipSuccess;
    ProductArgs p = args;
    p.parts = plan.splits > 1 || plan.late;
    if (p.parts && !p.partial) return hipErrorInvalidValue; // the caller's layout
    p.tiles_n = plan.tiles_n;
    if (p.n_out == 0) p.n_out = p.n;
    p.splits = plan.splits;
    p.k_each = plan.k_each;
    if (plan.late) p.beside.inner = nullptr;
    return with_type(type, [&](auto t) {
        typedef decltype(t) T;
        if (plan.thin_m) {
            launch_thin<T>(p, plan, s);
        } else if (!skinny && !across && !p.parts && p.k <= TileOf<T>::kK) {
            launch_short<T>(p, s);
        } else if (skinny) {
            if (across) launch_narrow<T, T, T, false, true, 128, 32, 4, 1, float>(p, plan, s);
            else launch_narrow<T, T, T, false, false, 128, 32, 4, 1, float>(p, plan, s);
        } else {
            const bool direct = lines_up(p.a, type, p.k) && lines_up(p.b, type, across ? p.n : p.k);
            if (across) launch_tiles<T, false, true>(p, plan, direct, s);
            else launch_tiles<T, false, false>(p, plan, direct, s);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || !p.parts) return e;
        if (plan.late && args.beside.inner) {
            p.beside = args.beside;
            const dim3 blocks((p.n + 255) / 256, p.groups.total); // at most 1,024 rows
            if (across) join_late_kernel<T, true><<<blocks, 256, 0, s>>>(p);
            else join_late_kernel<T, false><<<blocks, 256, 0, s>>>(p);
            return hipGetLastError();
        }
        return out_float ? join<float>(p, p.groups.total, s) : join<T>(p, p.groups.total, s);
    });
}

hipError_t product_weights(int type, ProductArgs p, const Plan &plan, bool narrow_m, bool narrow_n,
                           hipStream_t s) {
    if (plan.tiles == 0) return hipSuccess;
    p.parts = plan.splits > 1;
    if (p.parts && !p.partial) return hipErrorInvalidValue; // the caller's layout
    p.tiles_n = plan.tiles_n;
    if (p.n_out == 0) p.n_out = p.n;
    p.splits = plan.splits;
    return with_type(type, [&](auto t) {
        typedef decltype(t) T;
        if (narrow_m) launch_narrow<float, float, T, true, true, 32, 128, 1, 4, T>(p, plan, s);
        else if (narrow_n) launch_narrow<float, T, float, true, true, 128, 32, 4, 1, T>(p, plan, s);
        else launch_tiles<T, true, true>(p, plan, lines_up(p.a, type, p.m) && lines_up(p.b, type, p.n), s);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess || plan.splits == 1) return e;
        return join<T>(p, (uint64_t)p.groups.groups * p.m, s);
    });
}

int check_blocks(const char *call, const Plan &plan) {
    if (plan.tiles >= kMaxTiles) return fail(SDF_E_INVALID, "%s: too many tiles of the result", call);
    return SDF_OK;
}

} // namespace head
} // namespace sdfoam_hip

namespace {

int check_linear(const char *call, int type, uint64_t rows, uint32_t experts, uint32_t width, uint32_t out) {
    if (!known_type(type)) return fail(SDF_E_INVALID, "%s: type must be SDF_TYPE_*", call);
    if (experts > SDF_MAX_EXPERTS)
        return fail(SDF_E_INVALID, "at most %u experts (got %u)", SDF_MAX_EXPERTS, experts);
    if (rows >= 1ull << 31) return fail(SDF_E_INVALID, "%s takes fewer than 2^31 rows", call);
    if (width > 1u << 18 || out > 1u << 18)
        return fail(SDF_E_INVALID, "%s takes rows of at most 2^18 elements", call);
    return SDF_OK;
}

} // namespace

extern "C" {

size_t sdf_expert_linear_scratch_bytes(uint64_t count, uint32_t num_experts, uint32_t width,
                                       uint32_t out_width) {
    if (count >= 1ull << 31 || num_experts > SDF_MAX_EXPERTS) return 0;
    return plan_rows(count, num_experts, true, out_width, width, false, false).bytes;
}

int sdf_expert_linear(int type, const void *rows, uint64_t rows_stride, uint64_t count,
                      uint32_t num_experts, uint32_t width, uint32_t out_width,
                      const void *weight, const int32_t *offsets, void *out, void *scratch,
                      size_t scratch_bytes, void *stream) {
    int rc = check_linear("sdf_expert_linear", type, count, num_experts, width, out_width);
    if (rc != SDF_OK) return rc;
    if (count == 0 || out_width == 0) return SDF_OK;
    if (!offsets || !out || (width > 0 && (!rows || (num_experts > 0 && !weight))))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    const Plan plan = plan_rows(count, num_experts, true, out_width, width, false, false);
    if ((rc = check_scratch(scratch, scratch_bytes, plan.bytes)) != SDF_OK) return rc;
    if ((rc = check_blocks("sdf_expert_linear", plan)) != SDF_OK) return rc;
    ProductArgs p = {};
    p.a = {rows, rows_stride, 0, nullptr};
    p.b = {weight, width, (uint64_t)out_width * width, nullptr};
    p.groups = {offsets, num_experts, (uint32_t)count};
    p.n = out_width;
    p.k = width;
    p.out = out;
    p.out_stride = out_width;
    p.partial = static_cast<float *>(scratch);
    p.scale = 1.0f;
    const hipError_t e = product_rows(type, p, plan, false, false, false, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? SDF_OK : hip_fail(e, "expert_linear");
}

size_t sdf_expert_linear_backward_scratch_bytes(uint64_t count, uint32_t num_experts,
                                                uint32_t width, uint32_t out_width) {
    if (count >= 1ull << 31 || num_experts > SDF_MAX_EXPERTS) return 0;
    const size_t a = plan_rows(count, num_experts, true, width, out_width, true, false).bytes;
    const size_t b = plan_weights(count, num_experts, out_width, width, false, false).bytes;
    return a > b ? a : b; // one after the other
}

int sdf_expert_linear_backward(int type, const void *out_grad, uint64_t out_grad_stride,
                               const void *rows, uint64_t rows_stride, uint64_t count,
                               uint32_t num_experts, uint32_t width, uint32_t out_width,
                               const void *weight, const int32_t *offsets, void *rows_grad,
                               void *weight_grad, void *scratch, size_t scratch_bytes,
                               void *stream) {
    int rc = check_linear("sdf_expert_linear_backward", type, count, num_experts, width, out_width);
    if (rc != SDF_OK) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const bool want_rows = rows_grad && count > 0 && width > 0;
    const bool want_weight = weight_grad && num_experts > 0 && width > 0 && out_width > 0;
    if (!want_rows && !want_weight) return SDF_OK;
    if (!offsets || (count > 0 && out_width > 0 &&
                     (!out_grad || (want_rows && num_experts > 0 && !weight) || (want_weight && !rows))))
        return fail(SDF_E_INVALID, "NULL pointer argument");
    rc = check_scratch(scratch, scratch_bytes,
                       sdf_expert_linear_backward_scratch_bytes(count, num_experts, width, out_width));
    if (rc != SDF_OK) return rc;
    const Plan rows_plan = plan_rows(count, num_experts, true, width, out_width, true, false);
    const Plan weight_plan = plan_weights(count, num_experts, out_width, width, false, false);
    if ((want_rows && (rc = check_blocks("sdf_expert_linear_backward", rows_plan)) != SDF_OK) ||
        (want_weight && (rc = check_blocks("sdf_expert_linear_backward", weight_plan)) != SDF_OK))
        return rc;
    ProductArgs p = {};
    p.groups = {offsets, num_experts, (uint32_t)count};
    p.partial = static_cast<float *>(scratch);
    p.scale = 1.0f;
    if (want_rows) {
        p.a = {out_grad, out_grad_stride, 0, nullptr};
        p.b = {weight, width, (uint64_t)out_width * width, nullptr};
        p.n = width;
        p.k = out_width;
        p.out = rows_grad;
        p.out_stride = width;
        const hipError_t e = product_rows(type, p, rows_plan, true, false, false, s);
        if (e != hipSuccess) return hip_fail(e, "expert_linear_backward");
    }
    if (want_weight) {
        p.a = {out_grad, out_grad_stride, 0, nullptr};
        p.b = {rows, rows_stride, 0, nullptr};
        p.m = out_width;
        p.n = width;
        p.out = weight_grad;
        p.out_stride = width;
        const hipError_t e = product_weights(type, p, weight_plan, false, false, s);
        if (e != hipSuccess) return hip_fail(e, "expert_linear_backward");
    }
    return SDF_OK;
}

} // extern "C"
