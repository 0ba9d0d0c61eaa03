// Low-rank adapters of many requests at once, added to a projection's output:
// for row i with adapter a, and each block j of the output's columns,
//   t = x_i A_a^T (all blocks' ranks side by side),   out_j[i] += c t_j B_aj^T.
// The rows come sorted by adapter and cut into tiles of one adapter (a plan that
// the caller keeps for all projections of a step), so each product is a plain
// one: the first gives t in float32, K split over waves and workgroups, the second
// reads B once a tile and the output once. Both run on the matrix cores; 16-bit
// adapters take t as two pieces of their type, which keeps 16 bits of it.
#include <type_traits>

#include "gdn_common.h"
#include "gdn_host.h"
#include "gdn_low_rank_plan.h"

namespace gdn {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct AdapterBlock {
    int64_t b;      // first element of B (width, padded rank)
    int32_t a_row;  // first row of A
    int32_t rank;   // without padding to 16; 0: no adapter here
    float scale;
    int32_t t_col;  // first column of t
};

struct LowRankArgs {
    const void *x, *A, *B;
    const AdapterBlock* table;    // (S, blocks)
    const int32_t *order, *tiles; // rows by adapter; {adapter, first place in order, rows} a tile
    float* t;                     // (splits, M, rank_total)
    void* out[kLowRankBlocks];
    int64_t out_stride[kLowRankBlocks];
    int width[kLowRankBlocks], group_end[kLowRankBlocks];
    int64_t x_stride;
    int S, blocks, rank_total, M, K, Kp, tile_count, splits, per_wave, steps;
};

GDN_DEV int pad16(int r) { return (r + 15) & ~15; }

struct Tile {
    int adapter, start, count;
};

// A tile of the plan; count 0 where it holds none, or what no plan holds.
template <int kRows>
GDN_DEV Tile tile_of(const LowRankArgs& p, int i) {
    Tile t{p.tiles[3 * i], p.tiles[3 * i + 1], min(p.tiles[3 * i + 2], kRows)};
    if (uint32_t(t.adapter) >= uint32_t(p.S) || t.start < 0 || t.start > p.M - t.count) t.count = 0;
    return t;
}

// One wave's product of a 16 x 16 tile over 128 bytes of both operands' rows, two
// 16-byte pieces a lane (which of the k they are does not matter as long as
// both sides agree).
template <class Act>
GDN_DEV f32x4 mfma_pieces(const uint4& a, const uint4& b, f32x4 c) {
    if constexpr (Act::code == GDN_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
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

// t for a tile of kRF x 16 rows and kNR x 16 of its adapter's ranks. Ranks are the
// left operand, so a lane ends with four ranks of one row.
template <class Act, int kRF, int kNR>
__global__ __launch_bounds__(64 * kLowRankWaves) void low_rank_down_kernel(LowRankArgs p) {
    using S = typename Act::storage;
    constexpr int kStep = 128 / sizeof(S), kPiece = 16 / sizeof(S);
    __shared__ f32x4 sums[kLowRankWaves][kRF * kNR][64];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, lr = lane & 15;
    const Tile tile = tile_of<16 * kRF>(p, blockIdx.x);
    if (tile.count <= 0) return;
    const AdapterBlock* ab = p.table + int64_t(tile.adapter) * p.blocks;
    const int total = ab[p.blocks - 1].t_col + pad16(ab[p.blocks - 1].rank), r0 = blockIdx.y * 16 * kNR;
    if (r0 >= total) return;
    const S* xr[kRF];
    const S* ar[kNR];
#pragma unroll
    for (int i = 0; i < kRF; ++i) {
        const int row = p.order[tile.start + min(16 * i + lr, tile.count - 1)];
        xr[i] = static_cast<const S*>(p.x) + int64_t(min(max(row, 0), p.M - 1)) * p.x_stride + g * 2 * kPiece;
    }
#pragma unroll
    for (int j = 0; j < kNR; ++j)
        ar[j] = static_cast<const S*>(p.A) + int64_t(ab[0].a_row + min(r0 + 16 * j + lr, total - 1)) * p.Kp + g * 2 * kPiece;
    f32x4 acc[kRF][kNR];
#pragma unroll
    for (int i = 0; i < kRF; ++i)
#pragma unroll
        for (int j = 0; j < kNR; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int s0 = (blockIdx.z * kLowRankWaves + wave) * p.per_wave, s1 = min(p.steps, s0 + p.per_wave);
    const auto multiply = [&](const uint4 (&xv)[kRF][2], const uint4 (&av)[kNR][2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < kRF; ++i)
#pragma unroll
                for (int j = 0; j < kNR; ++j) acc[i][j] = mfma_pieces<Act>(av[j][h], xv[i][h], acc[i][j]);
    };
    const auto load_a = [&](int k, uint4 (&av)[kNR][2]) {
#pragma unroll
        for (int j = 0; j < kNR; ++j) {
            av[j][0] = *reinterpret_cast<const uint4*>(ar[j] + k);
            av[j][1] = *reinterpret_cast<const uint4*>(ar[j] + k + kPiece);
        }
    };
    const int whole = min(s1, p.K / kStep);
    for (int s = s0; s < whole; ++s) {
        uint4 xv[kRF][2], av[kNR][2];
        load_a(s * kStep, av);
#pragma unroll
        for (int i = 0; i < kRF; ++i) {
            __builtin_memcpy(&xv[i][0], xr[i] + s * kStep, 16);
            __builtin_memcpy(&xv[i][1], xr[i] + s * kStep + kPiece, 16);
        }
        multiply(xv, av);
    }
    if (s1 > whole && s1 > s0) {  // the last step of a K that is no multiple of it
        uint4 xv[kRF][2], av[kNR][2];
        const int k = (s1 - 1) * kStep, left = p.K - k - g * 2 * kPiece;
        load_a(k, av);
#pragma unroll
        for (int i = 0; i < kRF; ++i) {
            xv[i][0] = piece_of(xr[i] + k, left);
            xv[i][1] = piece_of(xr[i] + k + kPiece, left - kPiece);
        }
        multiply(xv, av);
    }
#pragma unroll
    for (int i = 0; i < kRF; ++i)
#pragma unroll
        for (int j = 0; j < kNR; ++j) sums[wave][i * kNR + j][lane] = acc[i][j];
    __syncthreads();
    for (int u = wave; u < kRF * kNR; u += kLowRankWaves) {
        f32x4 v = sums[0][u][lane];
#pragma unroll
        for (int w = 1; w < kLowRankWaves; ++w) v += sums[w][u][lane];
        const int row = u / kNR * 16 + lr, r = r0 + u % kNR * 16;
        if (row < tile.count && r < total)
            *reinterpret_cast<f32x4*>(p.t + (int64_t(blockIdx.z) * p.M + tile.start + row) * p.rank_total + r + 4 * g) = v;
    }
}

// Eight ranks of t (summed over the shares of K, times the adapter's scale) as the
// second product's operand: float32 as they are; 16 bits as two pieces, `low`
// 32 bytes behind `high`. bfloat16: the upper 8 bits and what they leave (16
// bits in all, and no overflow by rounding up); float16: t times `fit`, a power of
// two that brings the row's largest to between 2^13 and 2^14, so that both pieces
// are within the type. What is not finite has no rest.
template <class Act>
GDN_DEV void store_pieces(uint8_t* at, const float (&t)[8], float fit) {
    if constexpr (Act::code == GDN_F32) {
        *reinterpret_cast<float4*>(at) = make_float4(t[0], t[1], t[2], t[3]);
        *reinterpret_cast<float4*>(at + 16) = make_float4(t[4], t[5], t[6], t[7]);
    } else {
        uint16_t high[8], low[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (Act::code == GDN_BF16) {
                high[e] = uint16_t(__float_as_uint(t[e]) >> 16);
                const float rest = t[e] - bf16_bits_to_f32(high[e]);
                low[e] = (high[e] & 0x7F80) == 0x7F80 ? 0 : f32_to_bf16_bits(rest);
                if (t[e] != t[e]) high[e] = 0x7FC0;
            } else {
                const float v = t[e] * fit;
                high[e] = f32_to_f16_bits(v);
                low[e] = (high[e] & 0x7C00) == 0x7C00 ? 0 : f32_to_f16_bits(v - f16_bits_to_f32(high[e]));
            }
        }
        __builtin_memcpy(__builtin_assume_aligned(at, 16), high, 16);
        __builtin_memcpy(__builtin_assume_aligned(at + 32, 16), low, 16);
    }
}

// out += c t B^T for a tile of kRF x 16 rows and 256 columns of one block, 64 a
// wave. B is the left operand and its rows are dealt out so that a lane ends with
// 16 consecutive columns of one row. The 32 values of k of a 16-bit product are 16
// ranks of t's high piece and the same of its low one, B the same for both.
template <class Act, int kRF>
__global__ __launch_bounds__(64 * kLowRankWaves) void low_rank_up_kernel(LowRankArgs p) {
    using S = typename Act::storage;
    constexpr int kRows = 16 * kRF, kChunk = 64, kLine = kChunk / 16 * 64 + 16;  // (rows 16 bytes apart in the banks)
    constexpr int kPer = 64 * kLowRankWaves / kRows;                              // threads a row
    __shared__ __attribute__((aligned(16))) uint8_t pieces[kRows * kLine];
    __shared__ float fits[kRows];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, lr = lane & 15;
    const int group = blockIdx.x / p.tile_count;
    const Tile tile = tile_of<kRows>(p, blockIdx.x % p.tile_count);
    if (tile.count <= 0) return;
    int block = 0;
    while (group >= p.group_end[block]) ++block;
    const AdapterBlock ab = p.table[int64_t(tile.adapter) * p.blocks + block];
    if (ab.rank <= 0) return;
    const int R = pad16(ab.rank), width = p.width[block];
    const int n0 = (group - (block ? p.group_end[block - 1] : 0)) * kLowRankColumns + wave * 64;

    const int own = tid / kPer;  // the row whose ranks this thread brings in
    const float* t = p.t + (int64_t(tile.start) + min(own, tile.count - 1)) * p.rank_total + ab.t_col;
    const int64_t share = int64_t(p.M) * p.rank_total;
    const bool there = own < tile.count;
    const auto ranks8 = [&](int r, float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
        if (!there || r >= R) return;
        for (int s = 0; s < p.splits; ++s) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(t + s * share + r);
            const f32x4 b = *reinterpret_cast<const f32x4*>(t + s * share + r + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += a[e], v[4 + e] += b[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = r + e < ab.rank ? v[e] * ab.scale : 0.f;  // (padding: 0 times what is not finite)
    };
    float fit = 1.f;
    if constexpr (Act::code == GDN_F16) {
        float most = 0.f;
        for (int r = tid % kPer * 8; r < R; r += kPer * 8) {
            float v[8];
            ranks8(r, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));
        }
#pragma unroll
        for (int o = 1; o < kPer; o *= 2) most = fmaxf(most, __shfl_xor(most, o));
        const int up = int(__float_as_uint(most) >> 23) - 127;  // 2^up <= most < 2^(up + 1)
        const bool usable = most > 0x1p-100f && most < 0x1p100f;
        fit = usable ? __uint_as_float(uint32_t(127 + 13 - up) << 23) : 1.f;
        if (tid % kPer == 0) fits[own] = usable ? __uint_as_float(uint32_t(127 - 13 + up) << 23) : 1.f;
    }

    const S* br[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = n0 + lr / 4 * 16 + 4 * i + lr % 4;
        br[i] = static_cast<const S*>(p.B) + ab.b + int64_t(min(n, width - 1)) * R + (Act::code == GDN_F32 ? 4 * g : 8 * (g & 1));
    }
    f32x4 acc[kRF][4];
#pragma unroll
    for (int i = 0; i < kRF; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int r0 = 0; r0 < R; r0 += kChunk) {
        if (r0) __syncthreads();
        for (int r = tid % kPer * 8; r < min(kChunk, R - r0); r += kPer * 8) {
            float v[8];
            ranks8(r0 + r, v);
            store_pieces<Act>(pieces + own * kLine + r / 16 * 64 + r % 16 * (Act::code == GDN_F32 ? 4 : 2), v, fit);
        }
        __syncthreads();
        for (int c = 0; c < min(kChunk, R - r0); c += 16) {
            uint4 b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const uint4*>(br[j] + r0 + c);
#pragma unroll
            for (int i = 0; i < kRF; ++i) {
                const uint4 v = *reinterpret_cast<const uint4*>(pieces + (16 * i + lr) * kLine + c * 4 + g * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = mfma_pieces<Act>(b[j], v, acc[i][j]);
            }
        }
    }
    const int n = n0 + 16 * g;
    if (n >= width) return;
#pragma unroll
    for (int i = 0; i < kRF; ++i) {
        if (16 * i + lr >= tile.count) continue;
        const int row = p.order[tile.start + 16 * i + lr];
        if (uint32_t(row) >= uint32_t(p.M)) continue;
        S* y = static_cast<S*>(p.out[block]) + int64_t(row) * p.out_stride[block] + n;
        const float back = Act::code == GDN_F16 ? fits[16 * i + lr] : 1.f;
        if (n + 16 <= width) {
            S e[16];
            __builtin_memcpy(e, y, sizeof(e));
#pragma unroll
            for (int j = 0; j < 16; ++j) Act::store(e, j, __builtin_fmaf(acc[i][j / 4][j % 4], back, Act::load(e, j)));
            __builtin_memcpy(y, e, sizeof(e));
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (n + j < width) Act::store(y, j, __builtin_fmaf(acc[i][j / 4][j % 4], back, Act::load(y, j)));
        }
    }
}

int ranks_per_group(int rank_total) { return rank_total <= 16 ? 16 : rank_total <= 32 ? 32 : 64; }

bool low_rank_sizes_ok(int tiles, int tile_rows, int rank_total, int M, int K) {
    return tiles >= 0 && (tile_rows == 16 || tile_rows == 64) && rank_total > 0 && rank_total % 16 == 0 &&
           rank_total <= (1 << 16) && M >= 0 && M <= INT32_MAX - 256 && K > 0 && K <= (1 << 28);
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int64_t gdn_add_low_rank_workspace_size(int dtype, int tiles, int tile_rows, int rank_total, int M, int K) {
    if (!valid_dtype(dtype) || !low_rank_sizes_ok(tiles, tile_rows, rank_total, M, K)) return 0;
    const LowRankPlan plan = low_rank_plan(tiles, rank_total, K, dtype_size(dtype), ranks_per_group(rank_total));
    return int64_t(plan.splits) * M * rank_total * 4;
}

extern "C" int gdn_add_low_rank(const void* x, int64_t x_stride, int dtype, const void* A, const void* B, const void* table,
                                int adapters, int blocks, int rank_total, void* const* outs, const int64_t* out_strides,
                                const int* widths, const int32_t* order, const int32_t* tiles, int tile_count, int tile_rows,
                                int M, int K, void* workspace, int64_t workspace_bytes, void* stream) {
    GDN_REQUIRE(low_rank_sizes_ok(tile_count, tile_rows, rank_total, M, K) && adapters > 0,
                "gdn_add_low_rank: bad sizes M=%d K=%d rank_total=%d tiles=%d of %d, %d adapters", M, K, rank_total, tile_count,
                tile_rows, adapters);
    GDN_REQUIRE(blocks >= 1 && blocks <= kLowRankBlocks, "gdn_add_low_rank: %d blocks of columns, 1 to %d", blocks,
                kLowRankBlocks);
    GDN_REQUIRE(valid_dtype(dtype), "gdn_add_low_rank: bad dtype");
    if (M == 0 || tile_count == 0) return 0;
    GDN_REQUIRE(x && A && B && table && outs && out_strides && widths && order && tiles, "gdn_add_low_rank: null pointer");
    GDN_REQUIRE(x_stride >= K || M == 1, "gdn_add_low_rank: rows of x closer than their width");
    const int es = dtype_size(dtype), per = ranks_per_group(rank_total);
    const LowRankPlan plan = low_rank_plan(tile_count, rank_total, K, es, per);
    const int64_t need = int64_t(plan.splits) * M * rank_total * 4;
    GDN_REQUIRE(workspace && workspace_bytes >= need, "gdn_add_low_rank: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)need);
    GDN_REQUIRE((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B) | reinterpret_cast<uintptr_t>(table) |
                 reinterpret_cast<uintptr_t>(workspace)) % 16 == 0,
                "gdn_add_low_rank: A, B, table and workspace must be 16-byte aligned");
    LowRankArgs p{x, A, B, static_cast<const AdapterBlock*>(table), order, tiles, static_cast<float*>(workspace)};
    int64_t groups = 0;
    for (int j = 0; j < blocks; ++j) {
        GDN_REQUIRE(widths[j] >= 0 && (widths[j] == 0 || (outs[j] && (out_strides[j] >= widths[j] || M == 1))),
                    "gdn_add_low_rank: block %d of %d columns, rows %lld apart", j, widths[j], (long long)out_strides[j]);
        p.out[j] = outs[j];
        p.out_stride[j] = out_strides[j];
        p.width[j] = widths[j];
        groups += (int64_t(widths[j]) + kLowRankColumns - 1) / kLowRankColumns;
        GDN_REQUIRE(groups * tile_count <= INT32_MAX, "gdn_add_low_rank: too many rows and columns");
        p.group_end[j] = int(groups);
    }
    if (groups == 0) return 0;
    GDN_REQUIRE(one_grid_row(groups * tile_count, 256), "gdn_add_low_rank: too many rows and columns");
    p.x_stride = x_stride;
    p.S = adapters;
    p.blocks = blocks;
    p.rank_total = rank_total;
    p.M = M;
    p.K = K;
    p.Kp = plan.steps * (128 / es);
    p.tile_count = tile_count;
    p.splits = plan.splits;
    p.per_wave = plan.per_wave;
    p.steps = plan.steps;
    hipStream_t s = as_stream(stream);
    const auto go = [&](auto act, auto rf) {
        using Act = decltype(act);
        constexpr int RF = decltype(rf)::value;
        const dim3 down(unsigned(tile_count), unsigned((rank_total + per - 1) / per), unsigned(plan.splits));
        const dim3 threads(64 * kLowRankWaves);
        if (per == 16) hipLaunchKernelGGL((low_rank_down_kernel<Act, RF, 1>), down, threads, 0, s, p);
        else if (per == 32) hipLaunchKernelGGL((low_rank_down_kernel<Act, RF, 2>), down, threads, 0, s, p);
        else hipLaunchKernelGGL((low_rank_down_kernel<Act, RF, 4>), down, threads, 0, s, p);
        hipLaunchKernelGGL((low_rank_up_kernel<Act, RF>), dim3(unsigned(groups * tile_count)), threads, 0, s, p);
    };
    const auto typed = [&](auto act) {
        if (tile_rows == 64) go(act, std::integral_constant<int, 4>{});
        else go(act, std::integral_constant<int, 1>{});
    };
    if (dtype == GDN_F32) typed(ActF32{});
    else if (dtype == GDN_BF16) typed(ActBF16{});
    else typed(ActF16{});
    return check_launch("gdn_add_low_rank");
}
