// The causal depthwise conv of a state-space layer with its bias and SiLU, for
// packed runs: out[t, c] = silu(bias[c] + sum_j w[c, j] x[t - K + 1 + j, c]),
// the rows before a run taken from its conv state; the new state is the last
// K - 1 rows of state and run together. float32 throughout, one rounding.
//
// It reads and writes each element once: memory-bound, with the vector units
// close behind (about 70 cycles of a SIMD per 64 elements, exp2 and reciprocal
// half of them). A lane owns V neighbouring channels (16 bytes where the layout
// allows) over a tile of tokens and slides the K - 1 previous rows through
// registers; the rows of a tile come kConvAhead at a time, the next while these
// are used. A workgroup's four waves hold the same channels of four tiles that
// follow each other, so the taps (4 V K bytes a lane, as much as a tile of 16-bit
// values) and the K - 1 rows before a tile come from the CU's own cache.
//
// Measured, 6144 channels, over 1.6 GB of different inputs in turn, so that none
// are in a cache: 4096 bf16 tokens 27.2 us (3.7 TB/s; a copy of the same bytes
// 21.5), 16384 88 (4.6 TB/s; 78), 512 8.1 (4.3), 41 6.2 (2.0); 4096 float32 tokens
// 41.1 (4.9 TB/s; 39.6). On one input over and over, which the last-level cache
// holds in part: 21.9, 85, 6.4, 5.5 and 33.0.
#include "gdn_host.h"
#include "gdn_ssm.h"

namespace gdn {
namespace {

constexpr int kConvWaves = 4, kConvThreads = kConvWaves * kWave;
constexpr int kConvAhead = 4;

template <class Act, int V>
GDN_DEV void conv_raw(const typename Act::storage* p, typename Act::storage (&x)[V]) {
    if constexpr (V == 1) {
        x[0] = p[0];
    } else {
        typedef typename Act::storage vec __attribute__((ext_vector_type(V)));
        const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = v[e];
    }
}

template <class Act, int V>
GDN_DEV void conv_load(const typename Act::storage* p, float (&x)[V]) {
    typename Act::storage raw[V];
    conv_raw<Act, V>(p, raw);
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = Act::load(raw, e);
}

template <class Act, int V>
GDN_DEV void conv_store(typename Act::storage* p, const float (&x)[V]) {
    typename Act::storage s[V];
    if constexpr (Act::code == GDN_BF16 && V % 2 == 0) {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            const uint32_t two = pack_bf16x2(x[e], x[e + 1]);
            s[e] = uint16_t(two);
            s[e + 1] = uint16_t(two >> 16);
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) Act::store(s, e, x[e]);
    }
    if constexpr (V == 1) {
        p[0] = s[0];
    } else {
        typedef typename Act::storage vec __attribute__((ext_vector_type(V)));
        vec v;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = s[e];
        *reinterpret_cast<vec*>(p) = v;
    }
}

// Waves y < token_tiles take tokens; the others each write one run's state.
template <class Act, int V, int K, int kConvTile>
__global__ __launch_bounds__(kConvThreads) void conv_silu_kernel(
    const typename Act::storage* __restrict__ x, int64_t x_stride,
    const typename Act::storage* __restrict__ cs_in, typename Act::storage* __restrict__ cs_out,
    const float* __restrict__ w, const float* __restrict__ bias, const int32_t* __restrict__ cu, int N, int64_t L,
    int64_t T, int64_t token_tiles, typename Act::storage* __restrict__ out, int C) {
    const int c = (blockIdx.x * kWave + threadIdx.x % kWave) * V;
    if (c >= C) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t end = cu ? min(T, int64_t(cu[N])) : T;  // rows behind the last run are left as they are
    const int64_t rows = token_tiles + N, step = int64_t(gridDim.y) * kConvWaves;
    for (int64_t by = int64_t(blockIdx.y) * kConvWaves + wave; by < rows; by += step) {
        if (by >= token_tiles) {
            const int r = int(by - token_tiles);
            const int64_t b = run_start(cu, L, r), e = run_start(cu, L, r + 1);
#pragma unroll
            for (int j = 0; j < K - 1; ++j) {
                const int64_t t = e - (K - 1) + j;
                float v[V];
                if (t >= b) conv_load<Act, V>(x + t * x_stride + c, v);
                else conv_load<Act, V>(cs_in + (int64_t(r) * (K - 1) + (t - b) + (K - 1)) * C + c, v);
                conv_store<Act, V>(cs_out + (int64_t(r) * (K - 1) + j) * C + c, v);
            }
            continue;
        }
        float wr[V][K], bv[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
#pragma unroll
            for (int j = 0; j < K; ++j) wr[e][j] = w[int64_t(c + e) * K + j];
            bv[e] = bias ? bias[c + e] : 0.f;
        }
        const int64_t t0 = by * kConvTile, t1 = min(t0 + kConvTile, end);
        if (t0 >= end) continue;
        int r = cu ? find_run(cu, N, t0) : int(t0 / L);
        int64_t b = run_start(cu, L, r), e1 = run_start(cu, L, r + 1);
        float win[K - 1][V];
        const auto fill = [&](int64_t t) {  // the K - 1 rows before token t of run r
#pragma unroll
            for (int j = 0; j < K - 1; ++j) {
                const int64_t s = t - (K - 1) + j;
                if (s >= b) conv_load<Act, V>(x + s * x_stride + c, win[j]);
                else conv_load<Act, V>(cs_in + (int64_t(r) * (K - 1) + (s - b) + (K - 1)) * C + c, win[j]);
            }
        };
        const auto token = [&](int64_t t, const float (&xv)[V]) {
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float a = bv[e];
#pragma unroll
                for (int j = 0; j < K - 1; ++j) a = __builtin_fmaf(wr[e][j], win[j][e], a);
                o[e] = __builtin_fmaf(wr[e][K - 1], xv[e], a);
#pragma unroll
                for (int j = 0; j + 1 < K - 1; ++j) win[j][e] = win[j + 1][e];
                win[K - 2][e] = xv[e];
            }
            silu_all<Act::code>(o);
            conv_store<Act, V>(out + t * C + c, o);
        };
        if (t1 - t0 == kConvTile && e1 >= t1) {
            typename Act::storage raw[2][kConvAhead][V];
            const auto fetch = [&](int64_t t, typename Act::storage (&v)[kConvAhead][V]) {
#pragma unroll
                for (int i = 0; i < kConvAhead; ++i) conv_raw<Act, V>(x + (t + i) * x_stride + c, v[i]);
            };
            fetch(t0, raw[0]);
            fill(t0);
#pragma unroll
            for (int i = 0; i < kConvTile / kConvAhead; ++i) {
                if ((i + 1) * kConvAhead < kConvTile) fetch(t0 + (i + 1) * kConvAhead, raw[(i + 1) & 1]);
#pragma unroll
                for (int k = 0; k < kConvAhead; ++k) {
                    float xv[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) xv[e] = Act::load(raw[i & 1][k], e);
                    token(t0 + i * kConvAhead + k, xv);
                }
            }
            continue;
        }
        fill(t0);
        for (int64_t t = t0; t < t1; ++t) {
            if (t >= e1) {
                do {
                    ++r;
                    b = e1;
                    e1 = run_start(cu, L, r + 1);
                } while (t >= e1);
                fill(t);
            }
            float xv[V];
            conv_load<Act, V>(x + t * x_stride + c, xv);
            token(t, xv);
        }
    }
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_conv_silu(const void* x, int64_t x_stride, const void* conv_state_in, void* conv_state_out,
                             const float* weight, const float* bias, const int32_t* cu_seqlens, int N,
                             int64_t T_total, void* out, int C, int K, int act_dtype, void* stream) {
    GDN_REQUIRE(N >= 1 && T_total >= 0 && C > 0, "gdn_conv_silu: bad sizes N=%d T=%lld C=%d", N,
                (long long)T_total, C);
    GDN_REQUIRE(valid_dtype(act_dtype), "gdn_conv_silu: bad dtype");
    if (K < 2 || K > 4) return fail(GDN_EUNSUPPORTED, "gdn_conv_silu: 2 to 4 taps (got %d)", K);
    GDN_REQUIRE(cu_seqlens || T_total % N == 0, "gdn_conv_silu: %lld tokens are not divisible into %d runs",
                (long long)T_total, N);
    GDN_REQUIRE(T_total < (int64_t(1) << 31), "gdn_conv_silu: too many tokens");
    GDN_REQUIRE(x_stride >= C, "gdn_conv_silu: x_stride %lld below C=%d", (long long)x_stride, C);
    GDN_REQUIRE(conv_state_in && conv_state_out && weight && (T_total == 0 || (x && out)),
                "gdn_conv_silu: null pointer");
    const int es = dtype_size(act_dtype);
    const int64_t state_bytes = int64_t(N) * (K - 1) * C * es;
    GDN_REQUIRE(!overlaps(conv_state_in, state_bytes, conv_state_out, state_bytes),
                "gdn_conv_silu: conv_state_out overlaps conv_state_in");
    const int64_t L = T_total / N;
    const auto fits = [&](int v) {  // v channels in one aligned access everywhere
        const auto at = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(conv_state_in) |
                        reinterpret_cast<uintptr_t>(conv_state_out) | reinterpret_cast<uintptr_t>(out);
        return C % v == 0 && x_stride % v == 0 && at % (uintptr_t(v) * es) == 0;
    };
    const auto launch = [&](auto act, auto vec, auto tile) {
        using Act = decltype(act);
        constexpr int V = decltype(vec)::value, kTile = decltype(tile)::value;
        const int64_t token_tiles = (T_total + kTile - 1) / kTile, rows = (token_tiles + N + kConvWaves - 1) / kConvWaves;
        const dim3 grid(unsigned((C + kWave * V - 1) / (kWave * V)), unsigned(rows < 65535 ? rows : 65535));
        const auto kern = K == 4   ? conv_silu_kernel<Act, V, 4, kTile>
                          : K == 3 ? conv_silu_kernel<Act, V, 3, kTile>
                                   : conv_silu_kernel<Act, V, 2, kTile>;
        hipLaunchKernelGGL(kern, grid, dim3(kConvThreads), 0, as_stream(stream),
                           static_cast<const typename Act::storage*>(x), x_stride,
                           static_cast<const typename Act::storage*>(conv_state_in),
                           static_cast<typename Act::storage*>(conv_state_out), weight, bias, cu_seqlens, N, L,
                           T_total, token_tiles, static_cast<typename Act::storage*>(out), C);
    };
    // Tiles of 8 tokens; of 16 where lanes hold 8 channels, there are 8 waves of
    // them a CU and runs have 64 tokens on average. us with 8 and 16, bf16, 6144
    // channels, inputs from memory: 41 tokens 5.5, 6.8; 512 6.8, 8.5; 4096 28.5, 26.4; 16384 91, 83;
    // 256 runs of 8 17.4, 24.8 (a tile that runs share goes row by row). 4096
    // float32 tokens 39.7, 42.1.
    const auto tiled = [&](auto act, auto vec) {
        if constexpr (decltype(vec)::value == 8)
            if (T_total / 16 * (C / (kWave * 8)) >= 2048 && L >= 64)
                return launch(act, vec, std::integral_constant<int, 16>{});
        launch(act, vec, std::integral_constant<int, 8>{});
    };
    const auto pick = [&](auto act, auto wide, auto narrow) {
        if (fits(decltype(wide)::value)) tiled(act, wide);
        else if (fits(decltype(narrow)::value)) tiled(act, narrow);
        else tiled(act, std::integral_constant<int, 1>{});
    };
    using I2 = std::integral_constant<int, 2>;
    using I4 = std::integral_constant<int, 4>;
    using I8 = std::integral_constant<int, 8>;
    if (act_dtype == GDN_F32) pick(ActF32{}, I4{}, I2{});
    else if (act_dtype == GDN_BF16) pick(ActBF16{}, I8{}, I2{});
    else pick(ActF16{}, I8{}, I2{});
    return check_launch("gdn_conv_silu");
}
