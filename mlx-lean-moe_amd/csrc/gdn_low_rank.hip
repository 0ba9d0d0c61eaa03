// Low-rank adapters of many requests at once, added to a projection's output:
// for row i with adapter a, and each block j of the output's columns,
//   t = c x_i A_a^T (all blocks' ranks side by side),   out_j[i] += t_j B_aj^T.
// The rows come sorted by adapter and cut into tiles of one adapter (a plan that
// the caller keeps for all projections of a step), so each product is a plain
// one on the matrix cores, with float32 sums. The first leaves t for the second: in
// float32, which the second cuts into three bfloat16 pieces where B is bfloat16 (exact, at
// Ranks), or in float16 as two pieces of that type, the second what the first leaves, 22
// bits: t need not fit the type, so there 16 ranks of a row come times a power of two of
// their own, and their product goes back by it.
//
// A, B and t lie in memory in the order in which a wave's lanes take them: a load of
// 16 bytes a lane is 1 KB in one piece (8192 rows, 2048 -> 4096, rank 64: rows of them
// instead, 32 to 128 bytes a row and load, 25.0 + 50.3 us, so 18.9 + 39.4).
//
// Every kernel adds in the same order: K's steps w, w + 8, ... in wave w, the waves
// in turn, then 16 ranks after each other. So a row's result has the same bits
// whichever rows and projections it comes with.
#include <type_traits>

#include "gdn_common.h"
#include "gdn_host.h"
#include "gdn_low_rank_plan.h"

namespace gdn {
namespace {

constexpr int kDepth = 2;  // steps of K under way at once (3, 4 and 6: the same within 2 %)

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

struct AdapterBlock {
    int64_t b;      // first element of B: 16 ranks after each other, all columns of each
    int32_t a_row;  // first rank in A
    int32_t rank;   // without padding to 16; 0: no adapter here
    float scale;
    int32_t t_col;  // first column of t
};

struct LowRankArgs {
    const void *x, *A, *B;
    const AdapterBlock* table;     // (S, blocks)
    const int32_t *order, *tiles;  // rows by adapter; {adapter, first place in order, rows} a tile
    uint8_t* t;                    // (16 rows of a tile, 16 ranks) after each other, kBlockOfT bytes each
    void* out[kLowRankBlocks];
    int64_t out_stride[kLowRankBlocks];
    int width[kLowRankBlocks], group_end[kLowRankBlocks];
    int64_t x_stride;
    int S, blocks, rank_total, M, K, steps;
    int tile_count, parts, rows;   // parts of `rows` rows a tile
    int columns;                   // of a block a workgroup takes (both products in one launch)
};

GDN_DEV int pad16(int r) { return (r + 15) & ~15; }

struct Tile {
    int adapter, start, count;
    int64_t block;  // of t: its first 16 rows
};

// Part i of the plan's tiles; count 0 or less where it holds none, or what no plan
// holds.
GDN_DEV Tile part_of(const LowRankArgs& p, int i) {
    const int at = i / p.parts, from = i % p.parts * p.rows;
    Tile t{p.tiles[3 * at], p.tiles[3 * at + 1], p.tiles[3 * at + 2], (int64_t(at) * p.parts * p.rows + from) / 16};
    if (uint32_t(t.adapter) >= uint32_t(p.S) || t.start < 0 || t.count < 0 || t.start > p.M - t.count) t.count = 0;
    t.start += from;
    t.count = min(t.count - from, p.rows);
    return t;
}

GDN_DEV f32x4 mfma_bf16(const uint4& a, const uint4& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// A product of 16 x 16 results over a 16-byte piece of both operands a lane (which
// of the k they are does not matter as long as both sides agree).
template <class Act>
GDN_DEV f32x4 mfma_pieces(const uint4& a, const uint4& b, f32x4 c) {
    if constexpr (Act::code == GDN_BF16) {
        return mfma_bf16(a, b, c);
    } else if constexpr (Act::code == GDN_F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    } else {
        const f32x4 u = __builtin_bit_cast(f32x4, a), v = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(u[e], v[e], c, 0, 0, 0);
        return c;
    }
}

// 16 bytes from any element; beyond `count` elements zeros.
template <class S>
GDN_DEV uint4 piece_of(const S* p, int count) {
    constexpr int kCount = 16 / sizeof(S);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (count >= kCount) {
        __builtin_memcpy(&v, p, 16);
    } else {
        S e[kCount] = {};
#pragma unroll
        for (int i = 0; i < kCount; ++i)
            if (i < count) e[i] = p[i];
        __builtin_memcpy(&v, e, 16);
    }
    return v;
}

GDN_DEV void two_f16(float v, uint16_t& high, uint16_t& low) {
    high = f32_to_f16_bits(v);
    low = (high & 0x7C00) == 0x7C00 ? 0 : f32_to_f16_bits(v - f16_bits_to_f32(high));
}

// Bytes of t for 16 rows and 16 ranks: 16 a lane of the second product, and in float16
// a float a row.
template <class Act>
constexpr int kBlockOfT = Act::code == GDN_F16 ? 1024 + 64 : 1024;

// 16 rows' sums over 16 ranks, four ranks of a row a lane, as the second product's
// operand. Of the ranks the first `rank` exist (what is padding is 0, also 0 times what
// is not finite). float16: a row's largest is brought to between 2^13 and 2^14, so that
// both pieces are normal numbers of the type.
template <class Act>
GDN_DEV void store_t(uint8_t* to, f32x4 v, int rank, float scale) {
    const int g = (threadIdx.x & 63) >> 4, lr = threadIdx.x & 15;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = 4 * g + e < rank ? v[e] * scale : 0.f;
    if constexpr (Act::code != GDN_F16) {
        *reinterpret_cast<f32x4*>(to + lr * 16 + 256 * g) = v;
    } else {  // quarters of 1 KB: ranks 0 to 7 and 8 to 15 high, then low
        uint16_t high[4], low[4];
        float most = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        const int up = int(__float_as_uint(most) >> 23) - 127;  // 2^up <= most < 2^(up + 1)
        const bool usable = most > 0x1p-100f && most <= 0x1.fffffep127f;
        const float fit = usable ? __uint_as_float(uint32_t(127 + 13 - up) << 23) : 1.f;
        if (g == 0) *reinterpret_cast<float*>(to + 1024 + lr * 4) = usable ? __uint_as_float(uint32_t(127 - 13 + up) << 23) : 1.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) two_f16(v[e] * fit, high[e], low[e]);
        to += lr * 16 + g / 2 * 256 + g % 2 * 8;
        __builtin_memcpy(__builtin_assume_aligned(to, 8), high, 8);
        __builtin_memcpy(__builtin_assume_aligned(to + 512, 8), low, 8);
    }
}

// 16 ranks of one operand of B (16 columns), as a lane of the second product has them.
template <class Act>
using PartOfB = std::conditional_t<Act::code == GDN_BF16, uint2, uint4>;

// t of 16 rows and 16 ranks, as a lane of the second product has it. add: sum + B t for
// the four operands of a wave's 64 columns.
template <class Act>
struct Ranks {  // float32
    f32x4 v;
    GDN_DEV void load(const uint8_t* block) { v = *reinterpret_cast<const f32x4*>(block + (threadIdx.x & 63) * 16); }
    GDN_DEV void cut() {}
    GDN_DEV void add(const uint4 (&b)[4], f32x4 (&sum)[4]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] = mfma_pieces<Act>(b[j], __builtin_bit_cast(uint4, v), sum[j]);
    }
};

// bfloat16: t's float32 value as three pieces, each the upper 8 bits of what those before
// it leave (cut off, so exact; rounded up, the largest would overflow), in three products
// of 16 ranks. Two pieces in one product of 32 would lose 2^-16 of t: both launches, us,
// 8192 rows of rank 64 53.5 and with two 50.5, 4096 packed ones 54.4 and 53.3. The pieces
// made by the first product instead: half as many bytes of t again, 59.4 and 57.3; two of
// the three in one product, B's ranks held twice: 54.0 and 55.6.
template <>
struct Ranks<ActBF16> {
    f32x4 v;
    uint2 p[3];
    GDN_DEV void load(const uint8_t* block) { v = *reinterpret_cast<const f32x4*>(block + (threadIdx.x & 63) * 16); }
    static GDN_DEV float upper(float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u); }
    static GDN_DEV uint2 upper_halves(const f32x4& x) {
        const uint4 u = __builtin_bit_cast(uint4, x);
        return make_uint2(__builtin_amdgcn_perm(u.y, u.x, 0x07060302u), __builtin_amdgcn_perm(u.w, u.z, 0x07060302u));
    }
    GDN_DEV void cut() {
        f32x4 rest, last;
#pragma unroll
        for (int e = 0; e < 4; ++e) rest[e] = v[e] - upper(v[e]);
        const float most = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
        if (__builtin_expect(most > 0x1.fffffep127f, 0)) {  // what is infinite has no rest
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (fabsf(v[e]) > 0x1.fffffep127f) rest[e] = 0.f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) last[e] = rest[e] - upper(rest[e]);
        p[0] = upper_halves(v);
        p[1] = upper_halves(rest);
        p[2] = upper_halves(last);
    }
    GDN_DEV void add(const uint2 (&b)[4], f32x4 (&sum)[4]) const {
#pragma unroll
        for (int i = 2; i >= 0; --i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                sum[j] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4, b[j]), __builtin_bit_cast(i16x4, p[i]),
                                                                   sum[j], 0, 0, 0);
    }
};

template <>
struct Ranks<ActF16> {
    uint4 v;
    float back;
    GDN_DEV void load(const uint8_t* block) {
        v = *reinterpret_cast<const uint4*>(block + (threadIdx.x & 63) * 16);
        back = *reinterpret_cast<const float*>(block + 1024 + (threadIdx.x & 15) * 4);
    }
    GDN_DEV void cut() {}
    GDN_DEV void add(const uint4 (&b)[4], f32x4 (&sum)[4]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x4 p = mfma_pieces<ActF16>(b[j], v, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[j][e] = __builtin_fmaf(p[e], back, sum[j][e]);
        }
    }
};

// t for kRF x 16 rows of a tile and kNR x 16 of its adapter's ranks. Ranks are the
// left operand, so a lane ends with four ranks of one row. The waves share out K and
// add their sums in LDS; kDepth steps' loads are under way at once.
//
// One round of workgroups, bound by its chain of waits (tile, row numbers, x, LDS) and
// by x's way from memory: 8192 rows of 2048, rank 64, 14.0 us (33.5 MB), rank 16 10.8;
// 9.0 at 2112 values a row, which do not lie a power of two apart (a part of K in one
// piece a wave, to read at eight places far apart, took as long in all). A is read by each
// workgroup: of 4096 packed rows 59 MB pass the vector caches for 17 MB of x.
template <class Act, int kRF, int kNR>
__global__ __launch_bounds__(64 * kLowRankDownWaves) void low_rank_down_kernel(LowRankArgs p) {
    using S = typename Act::storage;
    constexpr int kStep = 128 / sizeof(S), kPiece = 16 / sizeof(S);
    __shared__ f32x4 sums[kLowRankDownWaves][kRF * kNR][64];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, lr = lane & 15;
    const Tile tile = part_of(p, blockIdx.x);
    if (tile.count <= 0) return;
    const AdapterBlock* ab = p.table + int64_t(tile.adapter) * p.blocks;
    const int total = min(ab[p.blocks - 1].t_col + pad16(ab[p.blocks - 1].rank), p.rank_total), r0 = blockIdx.y * 16 * kNR;
    if (r0 >= total) return;
    const S* xr[kRF];
#pragma unroll
    for (int i = 0; i < kRF; ++i) {
        const int row = p.order[tile.start + min(16 * i + lr, tile.count - 1)];
        xr[i] = static_cast<const S*>(p.x) + int64_t(min(max(row, 0), p.M - 1)) * p.x_stride + g * kPiece;
    }
    const uint8_t* ar[kNR];
#pragma unroll
    for (int j = 0; j < kNR; ++j)
        ar[j] = static_cast<const uint8_t*>(p.A) + int64_t(ab[0].a_row + min(r0 + 16 * j, total - 16)) * (p.steps * 128) + lane * 16;
    f32x4 acc[kRF][kNR];
#pragma unroll
    for (int i = 0; i < kRF; ++i)
#pragma unroll
        for (int j = 0; j < kNR; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const auto load = [&](int s, uint4 (&xv)[kRF][2], uint4 (&av)[kNR][2]) {
        const int k = s * kStep;
#pragma unroll
        for (int j = 0; j < kNR; ++j) {
            av[j][0] = *reinterpret_cast<const uint4*>(ar[j] + s * 2048);
            av[j][1] = *reinterpret_cast<const uint4*>(ar[j] + s * 2048 + 1024);
        }
        if (k + kStep <= p.K) {
#pragma unroll
            for (int i = 0; i < kRF; ++i) {
                __builtin_memcpy(&xv[i][0], xr[i] + k, 16);
                __builtin_memcpy(&xv[i][1], xr[i] + k + kStep / 2, 16);
            }
        } else {  // the last step of a K that is no multiple of it
            const int left = p.K - k - g * kPiece;
#pragma unroll
            for (int i = 0; i < kRF; ++i) {
                xv[i][0] = piece_of(xr[i] + k, left);
                xv[i][1] = piece_of(xr[i] + k + kStep / 2, left - kStep / 2);
            }
        }
    };
    const auto multiply = [&](const uint4 (&xv)[kRF][2], const uint4 (&av)[kNR][2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < kRF; ++i)
#pragma unroll
                for (int j = 0; j < kNR; ++j) acc[i][j] = mfma_pieces<Act>(av[j][h], xv[i][h], acc[i][j]);
    };
    uint4 xv[kDepth][kRF][2], av[kDepth][kNR][2];
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
        if (wave + d * kLowRankDownWaves < p.steps) load(wave + d * kLowRankDownWaves, xv[d], av[d]);
    for (int s0 = wave; s0 < p.steps; s0 += kDepth * kLowRankDownWaves)
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            const int s = s0 + d * kLowRankDownWaves;
            if (s >= p.steps) break;
            multiply(xv[d], av[d]);
            if (s + kDepth * kLowRankDownWaves < p.steps) load(s + kDepth * kLowRankDownWaves, xv[d], av[d]);
        }
#pragma unroll
    for (int i = 0; i < kRF; ++i)
#pragma unroll
        for (int j = 0; j < kNR; ++j) sums[wave][i * kNR + j][lane] = acc[i][j];
    __syncthreads();
    static_assert(kRF * kNR <= kLowRankDownWaves, "a wave for each 16 x 16 of t");
    const int r = r0 + wave % kNR * 16, rows = wave / kNR * 16;  // of the 16 x 16 that this wave finishes
    if (wave >= kRF * kNR || r >= total || rows >= tile.count) return;
    f32x4 v = sums[0][wave][lane];
#pragma unroll
    for (int w = 1; w < kLowRankDownWaves; ++w) v += sums[w][wave][lane];
    int block = 0;
    while (r >= ab[block].t_col + pad16(ab[block].rank)) ++block;
    store_t<Act>(p.t + ((tile.block + rows / 16) * (p.rank_total / 16) + r / 16) * kBlockOfT<Act>, v,
                 ab[block].t_col + ab[block].rank - r, ab[block].scale);
}

// A wave's 64 columns: the lane's 16 values of a row in 16-byte pieces, the four lanes
// of a row beside each other in each. acc[j] holds four columns from quad_at(g, j).
template <class Act>
struct Columns {
    using S = typename Act::storage;
    static constexpr int kY = sizeof(S), kCount = 16 / kY;
    static GDN_DEV int quad_at(int q, int j) { return j / (4 / kY) * 4 * kCount + q * kCount + j % (4 / kY) * 4; }
    static GDN_DEV void load(const S* y, uint4 (&v)[kY]) {
#pragma unroll
        for (int k = 0; k < kY; ++k) __builtin_memcpy(&v[k], y + k * 4 * kCount, 16);
    }
    // y (read into v if the wave's columns are `whole`) + acc; else the `left` columns
    // that there are from y on
    static GDN_DEV void add(S* y, const uint4 (&v)[kY], const f32x4 (&acc)[4], bool whole, int left) {
        if (whole) {
            S e[16];
            __builtin_memcpy(e, v, sizeof(e));
#pragma unroll
            for (int j = 0; j < 16; ++j) Act::store(e, j, acc[j / 4][j % 4] + Act::load(e, j));
#pragma unroll
            for (int k = 0; k < kY; ++k) __builtin_memcpy(y + k * 4 * kCount, e + k * kCount, 16);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int at = quad_at(0, j / 4) + j % 4;
                if (at < left) Act::store(y, at, acc[j / 4][j % 4] + Act::load(y, at));
            }
        }
    }
    // B: for each 16 ranks and 64 columns four operands, of 512 bytes in 16 bits: float16's
    // two pieces of t meet the same, in bfloat16 a lane has four ranks, half of 16 bytes
    static constexpr int kB = Act::code == GDN_F32 ? 1024 : 512;
    static GDN_DEV const uint8_t* operands(const LowRankArgs& p, const AdapterBlock& ab, int n0) {
        const int lane = threadIdx.x & 63;
        return static_cast<const uint8_t*>(p.B) + ab.b * kY + int64_t(n0 / 64) * (4 * kB) +
               (Act::code == GDN_BF16 ? lane / 32 * 256 + lane % 16 * 16 + lane / 16 % 2 * 8 : lane * 16 % kB);
    }
    static GDN_DEV int64_t next_ranks(int width) { return int64_t((width + 63) / 64) * (4 * kB); }
};

// out += t B^T for a part of a tile and 256 columns of one block, 64 a wave, 16
// rows at a time. B is the left operand and its rows are dealt out so that a lane
// ends with 16-byte pieces of one row's output, the four lanes of a row beside each
// other in each piece (32 bytes a lane instead: 45 us for 34 at rank 16). The 32 values
// of k of a float16 product are 16 ranks of t's high piece and the same of its low one, B
// the same for both. A wave keeps its part of B (kHeld pieces of 16 ranks; 0: more ranks
// than that, read again for each 16 rows) and streams the rows: the next ones' output
// and t are under way while these are multiplied and stored.
//
// Bound by the output's way through memory and back: 8192 x 4096, rank 16 about 30 us
// (134 MB, 4.5 TB/s), rank 64 42; 4096 x 12288, rank up to 32, 45 (201 MB, 4.4 TB/s).
// Past rank 64 by B, which is read for each 16 rows with nothing under way behind it: 4096 x
// 4096, rank 100, 32 us (225 MB of reads at the vector caches, 67 MB of output).
// At rank 64 t is twice the output's bytes at the vector caches, and cutting it is more of
// the arithmetic than the output's sums. Four waves a SIMD there in bfloat16 (120
// registers; left alone 132 and three: 8192 rows 53.5 us and 54.1, 2048 20.2 and 20.6).
template <class Act, int kHeld>
__global__ __launch_bounds__(64 * kLowRankUpWaves, Act::code == GDN_BF16 && kHeld == 4 ? 4 : 1) void low_rank_up_kernel(LowRankArgs p) {
    using S = typename Act::storage;
    using Own = Columns<Act>;
    constexpr int kT = kHeld ? kHeld : 1;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, lr = lane & 15;
    // neighbours take neighbouring columns: workgroups that run at once cover whole
    // rows, not one window of columns at strides that fall on few memory channels
    const int groups = p.group_end[p.blocks - 1], group = blockIdx.x % groups;
    const Tile tile = part_of(p, blockIdx.x / groups);
    if (tile.count <= 0) return;
    int block = 0;
    while (group >= p.group_end[block]) ++block;
    const AdapterBlock ab = p.table[int64_t(tile.adapter) * p.blocks + block];
    if (ab.rank <= 0) return;
    const int pieces = (ab.rank + 15) / 16, width = p.width[block];
    if (ab.t_col < 0 || ab.t_col + 16 * pieces > p.rank_total) return;  // (not what a table of these sizes holds)
    const int n0 = (group - (block ? p.group_end[block - 1] : 0)) * kLowRankColumns + wave * 64;
    // the rows' numbers, all at first: a number fetched among the rows' output would
    // be there only after the output before it
    __shared__ int rows[kLowRankTile];
    if (tid < p.rows) rows[tid] = tid < tile.count ? p.order[tile.start + tid] : -1;
    __syncthreads();
    if (n0 >= width) return;
    const int n = n0 + Own::kCount * g;
    const bool whole = n0 + 64 <= width;  // (of the wave: one branch)
    const uint8_t* br = Own::operands(p, ab, n0);
    const int64_t b_stride = Own::next_ranks(width);
    using Part = PartOfB<Act>;
    Part b[kT][4];
    const auto load_b = [&](int i, Part (&v)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const Part*>(br + i * b_stride + j * Own::kB);
    };
    if constexpr (kHeld != 0) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (i < pieces) load_b(i, b[i]);
    }
    S* out = static_cast<S*>(p.out[block]) + n;
    const int64_t stride = p.out_stride[block];
    constexpr int kBlock = kBlockOfT<Act>;
    const int64_t t_stride = int64_t(p.rank_total / 16) * kBlock;
    const uint8_t* t = p.t + tile.block * t_stride + int64_t(ab.t_col / 16) * kBlock;
    const int steps = (tile.count + 15) / 16;

    struct Rows {
        S* y;  // null: no row
        uint4 yv[Own::kY];
        Ranks<Act> tv[kT];
    };
    const auto fetch = [&](Rows& r, int s) {
        const int row = rows[16 * s + lr];
        r.y = uint32_t(row) < uint32_t(p.M) ? out + row * stride : nullptr;
        if (r.y && whole) Own::load(r.y, r.yv);
        if constexpr (kHeld != 0) {
#pragma unroll
            for (int i = 0; i < kHeld; ++i)
                if (i < pieces) r.tv[i].load(t + s * t_stride + kBlock * i);
        }
    };
    const auto finish = [&](Rows& r, int s) {
        f32x4 acc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (kHeld != 0) {
#pragma unroll
            for (int i = 0; i < kHeld; ++i)
                if (i < pieces) {
                    r.tv[i].cut();
                    r.tv[i].add(b[i], acc);
                }
        } else {
            for (int i = 0; i < pieces; ++i) {
                load_b(i, b[0]);
                Ranks<Act> v;
                v.load(t + s * t_stride + int64_t(kBlock) * i);
                v.cut();
                v.add(b[0], acc);
            }
        }
        if (r.y) Own::add(r.y, r.yv, acc, whole, width - n);
    };
    Rows even, odd;
    fetch(even, 0);
    for (int s = 0; s < steps; s += 2) {
        if (s + 1 < steps) fetch(odd, s + 1);
        finish(even, s);
        if (s + 1 >= steps) break;
        if (s + 2 < steps) fetch(even, s + 2);
        finish(odd, s + 1);
    }
}

// Both products in one launch, for few rows: 16 rows of a tile and p.columns columns of
// one block a workgroup, which forms their t itself, its waves sharing out K, while the
// first of its output and B are on their way. Then each wave takes every eighth 64
// columns, t from LDS; the next ones' output is under way while these are multiplied,
// their B while these are stored. Every workgroup of a block reads the same rows of
// A: low_rank_plan says where that is too much. Bound by its chain of waits: 1 row,
// 2048 -> 8192 | 4096, rank 16, 5.3 us; 64 rows of 27 adapters 9.2 (17.6 MB).
template <class Act, int kNR>
__global__ __launch_bounds__(64 * kLowRankDownWaves) void low_rank_whole_kernel(LowRankArgs p) {
    using S = typename Act::storage;
    using Own = Columns<Act>;
    constexpr int kStep = 128 / sizeof(S), kPiece = 16 / sizeof(S);
    __shared__ f32x4 sums[kLowRankDownWaves][kNR][64];
    __shared__ __attribute__((aligned(16))) uint8_t t[kNR * kBlockOfT<Act>];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, lr = lane & 15;
    const int groups = p.group_end[p.blocks - 1], group = blockIdx.x % groups;
    const Tile tile = part_of(p, blockIdx.x / groups);
    if (tile.count <= 0) return;
    int block = 0;
    while (group >= p.group_end[block]) ++block;
    const AdapterBlock ab = p.table[int64_t(tile.adapter) * p.blocks + block];
    if (ab.rank <= 0) return;
    const int pieces = (ab.rank + 15) / 16, width = p.width[block];
    const int row = p.order[tile.start + min(lr, tile.count - 1)];
    const S* xr = static_cast<const S*>(p.x) + int64_t(min(max(row, 0), p.M - 1)) * p.x_stride + g * kPiece;
    const uint8_t* ar = static_cast<const uint8_t*>(p.A) + int64_t(ab.a_row) * (p.steps * 128) + lane * 16;
    const int64_t a_stride = int64_t(p.steps) * 2048;
    const auto load = [&](int s, uint4 (&xv)[2], uint4 (&av)[kNR][2]) {
        const int k = s * kStep;
#pragma unroll
        for (int j = 0; j < kNR; ++j) {
            const uint8_t* a = ar + min(j, pieces - 1) * a_stride + s * 2048;
            av[j][0] = *reinterpret_cast<const uint4*>(a);
            av[j][1] = *reinterpret_cast<const uint4*>(a + 1024);
        }
        if (k + kStep <= p.K) {
            __builtin_memcpy(&xv[0], xr + k, 16);
            __builtin_memcpy(&xv[1], xr + k + kStep / 2, 16);
        } else {  // the last step of a K that is no multiple of it
            const int left = p.K - k - g * kPiece;
            xv[0] = piece_of(xr + k, left);
            xv[1] = piece_of(xr + k + kStep / 2, left - kStep / 2);
        }
    };

    int n0 = (group - (block ? p.group_end[block - 1] : 0)) * p.columns;
    const int n_end = min(width, n0 + p.columns);
    n0 += wave * 64;
    S* yr = lr < tile.count && uint32_t(row) < uint32_t(p.M)  // (null: no row)
                ? static_cast<S*>(p.out[block]) + int64_t(row) * p.out_stride[block] + Own::kCount * g : nullptr;
    const uint8_t* br = Own::operands(p, ab, 0);
    const int64_t b_stride = Own::next_ranks(width);
    using Part = PartOfB<Act>;
    Part raw[kNR][4];
    const auto load_b = [&](int n) {
#pragma unroll
        for (int i = 0; i < kNR; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                raw[i][j] = *reinterpret_cast<const Part*>(br + min(i, pieces - 1) * b_stride + (n / 64 * 4 + j) * Own::kB);
    };
    const auto load_y = [&](int n, uint4 (&v)[Own::kY]) {
        if (yr && n + 64 <= width) Own::load(yr + n, v);  // (else read where it is written)
    };
    uint4 even[Own::kY], odd[Own::kY];
    {
        f32x4 acc[kNR];
#pragma unroll
        for (int j = 0; j < kNR; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        uint4 xv[kDepth][2], av[kDepth][kNR][2];
#pragma unroll
        for (int d = 0; d < kDepth; ++d)
            if (wave + d * kLowRankDownWaves < p.steps) load(wave + d * kLowRankDownWaves, xv[d], av[d]);
        if (n0 < n_end) {
            load_y(n0, even);
            load_b(n0);
        }
        for (int s0 = wave; s0 < p.steps; s0 += kDepth * kLowRankDownWaves)
#pragma unroll
            for (int d = 0; d < kDepth; ++d) {
                const int s = s0 + d * kLowRankDownWaves;
                if (s >= p.steps) break;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < kNR; ++j) acc[j] = mfma_pieces<Act>(av[d][j][h], xv[d][h], acc[j]);
                if (s + kDepth * kLowRankDownWaves < p.steps) load(s + kDepth * kLowRankDownWaves, xv[d], av[d]);
            }
#pragma unroll
        for (int j = 0; j < kNR; ++j) sums[wave][j][lane] = acc[j];
    }
    __syncthreads();
    if (wave < kNR) {
        f32x4 v = sums[0][wave][lane];
#pragma unroll
        for (int w = 1; w < kLowRankDownWaves; ++w) v += sums[w][wave][lane];
        store_t<Act>(t + wave * kBlockOfT<Act>, v, ab.rank - wave * 16, ab.scale);
    }
    __syncthreads();

    const auto step = [&](int n, uint4 (&now)[Own::kY], uint4 (&next)[Own::kY]) {
        const int n2 = n + 64 * kLowRankDownWaves;
        if (n2 < n_end) load_y(n2, next);
        f32x4 sum[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kNR; ++c)
            if (c < pieces) {
                Ranks<Act> v;
                v.load(t + c * kBlockOfT<Act>);
                v.cut();
                v.add(raw[c], sum);
            }
        if (n2 < n_end) load_b(n2);
        if (yr) Own::add(yr + n, now, sum, n + 64 <= width, width - n - Own::kCount * g);
    };
    for (; n0 < n_end; n0 += 2 * 64 * kLowRankDownWaves) {
        step(n0, even, odd);
        if (n0 + 64 * kLowRankDownWaves >= n_end) break;
        step(n0 + 64 * kLowRankDownWaves, odd, even);
    }
}

bool low_rank_sizes_ok(int tiles, int tile_rows, int rank_total, int M, int K) {
    return tiles >= 0 && tile_rows >= 16 && tile_rows <= kLowRankTile && (tile_rows & (tile_rows - 1)) == 0 && rank_total > 0 && rank_total % 16 == 0 &&
           rank_total <= (1 << 16) && M >= 0 && M <= INT32_MAX - 512 && K > 0 && K <= (1 << 24);
}

}  // namespace
}  // namespace gdn

using namespace gdn;

namespace {

int64_t t_bytes(int dtype, int tiles, int tile_rows, int rank_total) {
    return int64_t(tiles) * (tile_rows / 16) * (rank_total / 16) * (dtype == GDN_F16 ? kBlockOfT<ActF16> : 1024);
}

LowRankPlan plan_of(int dtype, int rank_total, int rank_block, const int* widths, int blocks, int tiles, int tile_rows, int K) {
    return low_rank_plan(tiles, tile_rows, rank_total, rank_block, K, dtype_size(dtype), widths, blocks);
}

}  // namespace

extern "C" int64_t gdn_add_low_rank_workspace_size(int dtype, int blocks, int rank_total, int rank_block, const int* widths,
                                                   int tile_count, int tile_rows, int K) {
    if (!valid_dtype(dtype) || !low_rank_sizes_ok(tile_count, tile_rows, rank_total, 0, K) || blocks < 1 ||
        blocks > kLowRankBlocks || !widths)
        return 0;
    const LowRankPlan plan = plan_of(dtype, rank_total, rank_block, widths, blocks, tile_count, tile_rows, K);
    return plan.columns ? 0 : t_bytes(dtype, tile_count, tile_rows, rank_total);
}

extern "C" int gdn_add_low_rank(const void* x, int64_t x_stride, int dtype, const void* A, const void* B, const void* table,
                                int adapters, int blocks, int rank_total, int rank_block, void* const* outs,
                                const int64_t* out_strides, const int* widths, const int32_t* order, const int32_t* tiles,
                                int tile_count, int tile_rows, int M, int K, void* workspace, int64_t workspace_bytes,
                                void* stream) {
    GDN_REQUIRE(low_rank_sizes_ok(tile_count, tile_rows, rank_total, M, K) && adapters > 0 && rank_block > 0 &&
                    rank_block <= rank_total,
                "gdn_add_low_rank: bad sizes M=%d K=%d ranks %d of %d, tiles %d of %d, %d adapters", M, K, rank_block,
                rank_total, tile_count, tile_rows, adapters);
    GDN_REQUIRE(blocks >= 1 && blocks <= kLowRankBlocks, "gdn_add_low_rank: %d blocks of columns, 1 to %d", blocks,
                kLowRankBlocks);
    GDN_REQUIRE(valid_dtype(dtype), "gdn_add_low_rank: bad dtype");
    if (M == 0 || tile_count == 0) return 0;
    GDN_REQUIRE(x && A && B && table && outs && out_strides && widths && order && tiles, "gdn_add_low_rank: null pointer");
    GDN_REQUIRE(x_stride >= K || M == 1, "gdn_add_low_rank: rows of x closer than their width");
    GDN_REQUIRE((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B) | reinterpret_cast<uintptr_t>(table) |
                 reinterpret_cast<uintptr_t>(workspace)) % 16 == 0,
                "gdn_add_low_rank: A, B, table and workspace must be 16-byte aligned");
    LowRankArgs p{x, A, B, static_cast<const AdapterBlock*>(table), order, tiles, static_cast<uint8_t*>(workspace)};
    for (int j = 0; j < blocks; ++j) {
        GDN_REQUIRE(widths[j] >= 0 && widths[j] <= kLowRankMostColumns && (widths[j] == 0 || (outs[j] && (out_strides[j] >= widths[j] || M == 1))),
                    "gdn_add_low_rank: block %d of %d columns, rows %lld apart", j, widths[j], (long long)out_strides[j]);
        p.out[j] = outs[j];
        p.out_stride[j] = out_strides[j];
        p.width[j] = widths[j];
    }
    const int64_t groups = column_groups(widths, blocks, kLowRankColumns, p.group_end);
    if (groups == 0) return 0;
    const LowRankPlan plan = plan_of(dtype, rank_total, rank_block, widths, blocks, tile_count, tile_rows, K);
    const int64_t need = plan.columns ? 0 : t_bytes(dtype, tile_count, tile_rows, rank_total);
    GDN_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "gdn_add_low_rank: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)need);
    const int64_t down_parts = tile_rows / plan.down_rows, up_parts = tile_rows / plan.up_rows;
    GDN_REQUIRE(one_grid_row(tile_count * down_parts, 64 * kLowRankDownWaves) &&
                    one_grid_row(groups * tile_count * up_parts, 64 * kLowRankUpWaves),
                "gdn_add_low_rank: too many rows and columns");
    p.x_stride = x_stride;
    p.S = adapters;
    p.blocks = blocks;
    p.rank_total = rank_total;
    p.M = M;
    p.K = K;
    p.steps = plan.steps;
    p.tile_count = tile_count;
    hipStream_t s = as_stream(stream);
    const auto typed = [&](auto act) {
        using Act = decltype(act);
        if (plan.columns) {
            const auto whole = [&](auto kernel) {
                p.parts = tile_rows / 16;
                p.rows = 16;
                p.columns = plan.columns;
                const int64_t all = column_groups(widths, blocks, plan.columns, p.group_end);
                hipLaunchKernelGGL(kernel, dim3(unsigned(all * tile_count * p.parts)), dim3(64 * kLowRankDownWaves), 0, s, p);
            };
            if (plan.held == 1) whole(low_rank_whole_kernel<Act, 1>);
            else whole(low_rank_whole_kernel<Act, 2>);
            return;
        }
        const auto down = [&](auto kernel) {
            p.parts = int(down_parts);
            p.rows = plan.down_rows;
            hipLaunchKernelGGL(kernel, dim3(unsigned(tile_count * down_parts), unsigned((rank_total + plan.ranks - 1) / plan.ranks)),
                               dim3(64 * kLowRankDownWaves), 0, s, p);
        };
        const auto up = [&](auto kernel) {
            p.parts = int(up_parts);
            p.rows = plan.up_rows;
            hipLaunchKernelGGL(kernel, dim3(unsigned(groups * tile_count * up_parts)), dim3(64 * kLowRankUpWaves), 0, s, p);
        };
        if (plan.down_rows == 32) {
            if (plan.ranks == 16) down(low_rank_down_kernel<Act, 2, 1>);
            else if (plan.ranks == 32) down(low_rank_down_kernel<Act, 2, 2>);
            else down(low_rank_down_kernel<Act, 2, 4>);
        } else {
            if (plan.ranks == 16) down(low_rank_down_kernel<Act, 1, 1>);
            else if (plan.ranks == 32) down(low_rank_down_kernel<Act, 1, 2>);
            else down(low_rank_down_kernel<Act, 1, 4>);
        }
        if (plan.held == 1) up(low_rank_up_kernel<Act, 1>);
        else if (plan.held == 2) up(low_rank_up_kernel<Act, 2>);
        else if (plan.held == 4) up(low_rank_up_kernel<Act, 4>);
        else up(low_rank_up_kernel<Act, 0>);
    };
    if (dtype == GDN_F32) typed(ActF32{});
    else if (dtype == GDN_BF16) typed(ActBF16{});
    else typed(ActF16{});
    return check_launch("gdn_add_low_rank");
}
