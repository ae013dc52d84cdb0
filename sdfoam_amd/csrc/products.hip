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

// What the rows' adapters add to 32 rows of kTn x 32 columns from n0 on: a lane has row m0 +
// mi.  One adapter of the 32 rows' after the other, floats in the matrix units.
template <typename S, bool kAcross, int kTn>
__device__ __forceinline__ void add_beside(const ProductArgs &p, uint32_t m0, uint32_t rows,
                                           uint32_t mi, uint32_t n0, F16x *acc) {
    const uint32_t lane = threadIdx.x & 63u, l32 = lane & 31u, half = lane >> 5;
    const uint32_t place = m0 + min(mi, rows - 1);
    const int32_t mine = mi < rows ? p.beside.group_of[place] : -1;
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
// one multiplied while the other is brought.
template <typename T, bool kWeights, bool kAcrossB, int kM, int kN, int kWavesM, int kWavesN, bool kDirect>
__global__ __launch_bounds__(64 * kWavesM * kWavesN, 2) void tile_kernel(ProductArgs p) {
    constexpr int kWaves = kWavesM * kWavesN, kBlock = 64 * kWaves;
    constexpr int kTm = kM / kWavesM / 32, kTn = kN / kWavesN / 32, kK = TileOf<T>::kK;
    constexpr uint32_t kTile = (kM + kN) * 128;
    __shared__ __attribute__((aligned(16))) char lds[2 * kTile];
    __shared__ uint32_t found[20];
    Feed<T, kWeights, kM, kWaves, kDirect> a;
    Feed<T, kWeights || kAcrossB, kN, kWaves, kDirect> b;

    uint32_t tile_m, tile_n;
    const uint32_t split = blockIdx.y;
    uint32_t k_begin = 0, k_end = p.k, group, m0, rows_m, n0;
    if constexpr (kWeights) {
        const uint32_t tiles_m = (p.m + kM - 1) / kM;
        // every XCD has a share of each group, whose rows differ in number
        group = blockIdx.x / (tiles_m * p.tiles_n);
        tile_of_block(blockIdx.x - group * tiles_m * p.tiles_n, tiles_m, p.tiles_n, tile_m, tile_n);
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
        a.begin(p.a, 0, m0, p.m, k_begin);
        b.begin(p.b, 0, n0, p.n, k_begin);
    } else {
        TilesOfRows<kM, kBlock> tiles(p.groups, found);
        const uint32_t tiles_m = tiles.count();
        if (blockIdx.x >= tiles_m * p.tiles_n) return; // left over
        tile_of_block(blockIdx.x, tiles_m, p.tiles_n, tile_m, tile_n);
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
        a.begin(p.a, 0, m0, rows_m, k_begin);
        b.begin(p.b, which, n0, kAcrossB ? p.n : min((uint32_t)kN, p.n - n0), k_begin);
    }

    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t wm = wave % kWavesM * (kTm * 32), wn = wave / kWavesM * (kTn * 32);
    const uint32_t l32 = lane & 31u, half = lane >> 5;
    F16x acc[kTm][kTn] = {};
    const Fragments<T, kWeights, kM, kTm> of_a(wm);
    const Fragments<T, kWeights || kAcrossB, kN, kTn> of_b(wn);
    if (k_begin < k_end) {
        const auto bring = [&](char *to, uint32_t k) {
            a.load(to, k, k_begin, k_end);
            b.load(to + kM * 128, k, k_begin, k_end);
        };
        const auto brought = [&](char *to) {
            a.store(to);
            b.store(to + kM * 128);
            if (kDirect) landed();
            __syncthreads();
        };
        bring(lds, k_begin);
        brought(lds);
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
            if (more) brought(lds + now);
        }
        __syncthreads();
    }

    // a lane has one row of the result (l32) and runs of 4 columns of it; a wave turns 32
    // rows at a time in LDS of its own, to write each in pieces of 16 bytes side by side
    constexpr uint32_t kTurn = 32 * (kTn * 32 * 4 + 16);
    static_assert(kWaves * kTurn <= sizeof(lds), "room for each wave");
    char *turn = lds + wave * kTurn;
    const uint64_t rows = kWeights ? (uint64_t)p.groups.groups * p.m : p.groups.total;
    const uint64_t row0 = kWeights ? (uint64_t)group * p.m + m0 : m0;
    if constexpr (!kWeights)
        if (p.beside.inner && split == 0)
#pragma unroll
            for (int i = 0; i < kTm; ++i)
                add_beside<T, kAcrossB, kTn>(p, m0, rows_m, wm + i * 32 + l32, n0 + wn, acc[i]);
    const auto write = [&](auto t, const F16x *sums, uint32_t first, auto row_at, float scale) {
        typedef decltype(t) O;
        constexpr uint32_t kE = 16 / sizeof(O), kPieces = kTn * 32 / kE;
        constexpr uint32_t kBytes = kTn * 32 * sizeof(O) + 16;
        wave_sync();
#pragma unroll
        for (int j = 0; j < kTn; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t n = j * 32 + q * 8 + half * 4;
                Few<O, 4> o;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    o.v[e] = n0 + wn + n + e < p.n ? (O)(scale * sums[j][q * 4 + e]) : (O)0.0f;
                *reinterpret_cast<Few<O, 4> *>(turn + l32 * kBytes + n * sizeof(O)) = o;
            }
        wave_sync();
#pragma unroll
        for (uint32_t t = 0; t < kPieces / 2; ++t) {
            const uint32_t at = t * 64 + lane, r = at / kPieces, n = at % kPieces * kE;
            const uint32_t m = first + r;
            const O *from = reinterpret_cast<const O *>(turn + r * kBytes) + n;
            if (m >= rows_m || n0 + wn + n >= p.n_out) continue;
            O *to = row_at(row0 + m) + n0 + wn + n;
            const uint32_t have = p.n_out - (n0 + wn + n);
            if (have >= kE) __builtin_memcpy(to, from, 16);
            else
#pragma unroll 1
                for (uint32_t e = 0; e < have; ++e) to[e] = from[e];
        }
    };
    if (p.splits > 1) {
#pragma unroll
        for (int i = 0; i < kTm; ++i)
            write(0.0f, acc[i], wm + i * 32,
                  [&](uint64_t row) { return p.partial + (split * rows + row) * p.n_out; }, 1.0f);
    } else {
#pragma unroll
        for (int i = 0; i < kTm; ++i)
            write(T(), acc[i], wm + i * 32, [&](uint64_t row) {
                return static_cast<T *>(p.out) + (p.out_index ? (uint32_t)p.out_index[row] : row) * p.out_stride;
            }, p.scale);
    }
}

constexpr int kThreads = 256;

// One tile of kM x kN of the result, kWavesM x kWavesN waves.  Two tiles of the inner
// dimension in LDS: while one is multiplied, the next is on its way to registers.
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

    const uint32_t tile_n = blockIdx.x % p.tiles_n, tile_m = blockIdx.x / p.tiles_n;
    const uint32_t split = blockIdx.y;
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
        if constexpr (!kWeights)
            if (p.beside.inner && split == 0)
                add_beside<SB, kAcrossB, kTn>(p, m0, rows_m, mi, n0 + wn, acc[i]);
        if (mi >= rows_m) continue;
        const uint64_t row = kWeights ? (uint64_t)group * p.m + m0 + mi : m0 + mi;
#pragma unroll
        for (int j = 0; j < kTn; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t n = n0 + wn + j * 32 + q * 8 + half * 4;
                if (n >= p.n_out) continue;
                Few<float, 4> sum;
#pragma unroll
                for (int e = 0; e < 4; ++e) sum.v[e] = n + e < p.n ? acc[i][j][q * 4 + e] : 0.0f;
                if (p.splits > 1) {
                    const uint64_t rows = kWeights ? (uint64_t)p.groups.groups * p.m : p.groups.total;
                    store_some<float, 4>(p.partial + (split * rows + row) * p.n_out + n, sum, p.n_out - n);
                } else {
                    Few<O, 4> o;
#pragma unroll
                    for (int e = 0; e < 4; ++e) o.v[e] = (O)(p.scale * sum.v[e]);
                    store_some<O, 4>(static_cast<O *>(p.out) + (p.out_index ? (uint32_t)p.out_index[row] : row) * p.out_stride + n,
                                     o, p.n_out - n);
                }
            }
    }
}

// The splits' sums in order.  rows x n floats a split; four columns a thread.
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
    for (int e = 0; e < 4; ++e) o.v[e] = (O)(p.scale * sum[e]);
    store_some<O, 4>(to, o, have);
}

constexpr uint64_t kMaxBlocks = 1ull << 23;

// whether rows of n elements are whole pieces of 16 bytes wherever one begins
bool lines_up(const Operand &o, int type, uint32_t n) {
    const size_t e = type_bytes(type);
    return reinterpret_cast<uintptr_t>(o.base) % 16 == 0 && o.stride * e % 16 == 0 &&
           o.group_stride * e % 16 == 0 && n * e % 16 == 0;
}

template <typename T, bool kWeights, bool kAcross, bool kDirect>
void launch_tiles_as(const ProductArgs &p, const Plan &plan, hipStream_t s) {
    const dim3 grid((uint32_t)plan.tiles, plan.splits);
    if (plan.large) tile_kernel<T, kWeights, kAcross, 256, 256, 2, 4, kDirect><<<grid, 512, 0, s>>>(p);
    else tile_kernel<T, kWeights, kAcross, 128, 128, 2, 2, kDirect><<<grid, 256, 0, s>>>(p);
}
template <typename T, bool kWeights, bool kAcross>
void launch_tiles(const ProductArgs &p, const Plan &plan, bool direct, hipStream_t s) {
    if (direct) launch_tiles_as<T, kWeights, kAcross, true>(p, plan, s);
    else launch_tiles_as<T, kWeights, kAcross, false>(p, plan, s);
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

Plan plan_rows(uint64_t rows, uint32_t groups, bool grouped, uint32_t n, uint32_t k, bool skinny) {
    Plan plan = {};
    plan.large = !skinny && take_large(tiles_of_rows(rows, groups, grouped, 256) * ((n + 255) / 256),
                                       tiles_of_rows(rows, groups, grouped, 128) * ((n + 127) / 128));
    const uint32_t km = plan.large ? 256 : 128, kn = skinny ? 32 : km;
    plan.tiles_n = (n + kn - 1) / kn;
    plan.tiles = tiles_of_rows(rows, groups, grouped, km) * plan.tiles_n;
    // few tiles: the inner dimension in several parts, of 512 elements at least, until the
    // chip has a block for each of its places
    plan.splits = 1;
    if (plan.tiles > 0 && !plan.large && plan.tiles < 256) {
        const uint64_t want = 512 / plan.tiles, most = k / 512;
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
    if (plan.tiles > 0 && !plan.large && plan.tiles < 256) {
        const uint64_t want = 512 / plan.tiles, most = rows / groups / 256;
        plan.splits = (uint32_t)(want < most ? want : most);
        if (plan.splits < 1) plan.splits = 1;
    }
    plan.bytes = plan.splits > 1 ? round_up((uint64_t)plan.splits * groups * m * n * 4) : 0;
    return plan;
}

hipError_t product_rows(int type, ProductArgs p, const Plan &plan, bool across, bool skinny,
                        bool out_float, hipStream_t s) {
    if (plan.tiles == 0) return hipSuccess;
    p.tiles_n = plan.tiles_n;
    if (p.n_out == 0) p.n_out = p.n;
    p.splits = plan.splits;
    p.k_each = plan.k_each;
    const dim3 grid((uint32_t)plan.tiles, plan.splits);
    return with_type(type, [&](auto t) {
        typedef decltype(t) T;
        if (skinny) {
            if (across) product_kernel<T, T, T, false, true, 128, 32, 4, 1, float><<<grid, kThreads, 0, s>>>(p);
            else product_kernel<T, T, T, false, false, 128, 32, 4, 1, float><<<grid, kThreads, 0, s>>>(p);
        } else {
            const bool direct = lines_up(p.a, type, p.k) && lines_up(p.b, type, across ? p.n : p.k);
            if (across) launch_tiles<T, false, true>(p, plan, direct, s);
            else launch_tiles<T, false, false>(p, plan, direct, s);
        }
        hipError_t e = hipGetLastError();
        if (e != hipSuccess || plan.splits == 1) return e;
        return out_float ? join<float>(p, p.groups.total, s) : join<T>(p, p.groups.total, s);
    });
}

hipError_t product_weights(int type, ProductArgs p, const Plan &plan, bool narrow_m, bool narrow_n,
                           hipStream_t s) {
    if (plan.tiles == 0) return hipSuccess;
    p.tiles_n = plan.tiles_n;
    if (p.n_out == 0) p.n_out = p.n;
    p.splits = plan.splits;
    const dim3 grid((uint32_t)plan.tiles, plan.splits);
    return with_type(type, [&](auto t) {
        typedef decltype(t) T;
        if (narrow_m) product_kernel<float, float, T, true, true, 32, 128, 1, 4, T><<<grid, kThreads, 0, s>>>(p);
        else if (narrow_n) product_kernel<float, T, float, true, true, 128, 32, 4, 1, T><<<grid, kThreads, 0, s>>>(p);
        else launch_tiles<T, true, true>(p, plan, lines_up(p.a, type, p.m) && lines_up(p.b, type, p.n), s);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess || plan.splits == 1) return e;
        return join<T>(p, (uint64_t)p.groups.groups * p.m, s);
    });
}

int check_blocks(const char *call, const Plan &plan) {
    if (plan.tiles > kMaxBlocks) return fail(SDF_E_INVALID, "%s: too many tiles of the result", call);
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
    return plan_rows(count, num_experts, true, out_width, width, false).bytes;
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
    const Plan plan = plan_rows(count, num_experts, true, out_width, width, false);
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
    if (count >= 1ull << 31 || num_experts > SDF_MAX_EXPERTS || num_experts == 0) return 0;
    const size_t a = plan_rows(count, num_experts, true, width, out_width, false).bytes;
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
    ProductArgs p = {};
    p.groups = {offsets, num_experts, (uint32_t)count};
    p.partial = static_cast<float *>(scratch);
    p.scale = 1.0f;
    if (want_rows) {
        const Plan plan = plan_rows(count, num_experts, true, width, out_width, false);
        if ((rc = check_blocks("sdf_expert_linear_backward", plan)) != SDF_OK) return rc;
        p.a = {out_grad, out_grad_stride, 0, nullptr};
        p.b = {weight, width, (uint64_t)out_width * width, nullptr};
        p.n = width;
        p.k = out_width;
        p.out = rows_grad;
        p.out_stride = width;
        const hipError_t e = product_rows(type, p, plan, true, false, false, s);
        if (e != hipSuccess) return hip_fail(e, "expert_linear_backward");
    }
    if (want_weight) {
        const Plan plan = plan_weights(count, num_experts, out_width, width, false, false);
        if ((rc = check_blocks("sdf_expert_linear_backward", plan)) != SDF_OK) return rc;
        p.a = {out_grad, out_grad_stride, 0, nullptr};
        p.b = {rows, rows_stride, 0, nullptr};
        p.m = out_width;
        p.n = width;
        p.out = weight_grad;
        p.out_stride = width;
        const hipError_t e = product_weights(type, p, plan, false, false, s);
        if (e != hipSuccess) return hip_fail(e, "expert_linear_backward");
    }
    return SDF_OK;
}

} // extern "C"
