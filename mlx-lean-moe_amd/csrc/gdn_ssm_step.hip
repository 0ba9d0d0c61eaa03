// One token of a state-space layer for B sequences: conv + SiLU over the
// token's channels with the conv state rolled on, the step d = softplus(dt +
// dt_bias), and per head
//   S <- exp(-exp(A_log) d) S + (d x) B^T,   y = S C + D x.
//
// The float32 head_dim x state_dim state is the only large operand: it is read
// once and written once, so the kernel is bound by memory, and below a few
// hundred workgroups by latency. A workgroup takes a head (or, of few heads, a
// share of its rows), kPass x kRows rows at a time; a state row lies across
// kLanes lanes, four values each, so a wave reads 1 KB in one piece. Every head of a group needs
// the group's B and C channels after the conv: each workgroup computes them
// itself (2 state_dim channels from cached rows) instead of a launch of its
// own, and the group's first workgroup rolls their conv state. What does not
// depend on the slot is loaded before the slot is known, and a thread's
// channels all at once: a chain of loads is what one sequence's token costs. So is the
// counter: the shares of a row's workgroups meet in one place, 10 ns each,
// hence few large workgroups for few heads (64 heads, one sequence: 13.2 us as
// 512 workgroups of 256 threads, 6.0 as 64 of 1024).
//
// 256 sequences, 64 heads of 64 x 128 (1.07 GB): 200 us, 5.4 TB/s. 512 threads against
// 256 (us): 8 sequences 12.2 and 15.3, 32 31.0 and 37.1, 256 200 and 200;
// two passes' loads in flight or several heads a workgroup were no faster.
#include <type_traits>

#include "gdn_host.h"
#include "gdn_ssm.h"

namespace gdn {
namespace {

constexpr int kStepCounter = 1 << 16;  // what a step adds to a slot's counter, over all its workgroups
constexpr int kMaxState = 256, kMaxHead = 256;

struct StepArgs {
    const void* xbc;
    int64_t xbc_stride;
    const void* dt;
    int64_t dt_stride;
    const void* cs_in;
    void* cs_out;
    const float *w, *bias, *A_log, *dt_bias, *D, *S_in;
    float* S_out;
    void* y;
    int y_dtype, G, H, P, N, K;
    int split;  // workgroups of a head
    int B;
    const int32_t* slots;
    int pool;
    const int32_t* half;
    int32_t* arrivals;
};

// kPass: rows of state a thread holds at a time
template <class Act, int kLanes, int kStepThreads, int kPass>
__global__ __launch_bounds__(kStepThreads) void step_kernel(StepArgs a) {
    constexpr int kRows = kStepThreads / kLanes;  // rows side by side
    constexpr int kItems = (kMaxHead + 2 * kMaxState + kStepThreads - 1) / kStepThreads;  // channels of a thread
    __shared__ __attribute__((aligned(16))) float Bs[kMaxState], Cs[kMaxState], xs[kMaxHead];
    __shared__ float gates[2];
    using S = typename Act::storage;
    const int P = a.P, N = a.N, H = a.H, K1 = a.K - 1, tid = threadIdx.x;
    const int per = H / a.G, blocks = H * a.split;  // of a row
    const unsigned id = blockIdx.y * gridDim.x + blockIdx.x;
    const int b = int(id / unsigned(blocks)), block = int(id % unsigned(blocks));
    if (b >= a.B) return;  // (the last row of the grid may be short)
    const int h = block / a.split, part = block % a.split, grp = h / per;
    const int share = (P + a.split - 1) / a.split;
    const int p_lo = min(P, part * share), rows = min(P, p_lo + share) - p_lo;
    const int C = H * P + 2 * a.G * N;

    // this thread's channels: the head's x rows, then B, then C
    const int count = rows + 2 * N;
    const S* x = static_cast<const S*>(a.xbc) + b * a.xbc_stride;
    int ch[kItems];
    float now[kItems], bias[kItems], w[kItems][4];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int at = tid + kStepThreads * i, k = at - rows;
        ch[i] = at >= count ? 0 : k < 0 ? h * P + p_lo + at
                : H * P + (k < N ? grp * N + k : (a.G + grp) * N + (k - N));
        if (kStepThreads * i < count) {
            now[i] = Act::load(x, ch[i]);
            bias[i] = a.bias ? a.bias[ch[i]] : 0.f;
            const float* wc = a.w + int64_t(ch[i]) * a.K;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i][j] = j < a.K ? wc[j] : 0.f;
        }
    }
    float dt = 0.f, A = 0.f;
    if (tid == 0) {
        dt = Act::load(static_cast<const S*>(a.dt), b * a.dt_stride + h) + a.dt_bias[h];
        A = a.A_log[h];
    }

    const int sl = a.slots ? a.slots[b] : b;
    if (unsigned(sl) >= unsigned(a.pool)) {  // a slot outside the pool: touch no state
        for (int i = tid; i < rows; i += kStepThreads)
            store_any(a.y, (int64_t(b) * H + h) * P + p_lo + i, a.y_dtype, __builtin_nanf(""));
        return;
    }
    int64_t ci = sl, co = b;
    if (a.half) {
        const int hb = (a.half[sl] ^ (a.arrivals ? a.arrivals[sl] >> 16 : 0)) & 1;
        ci = sl + int64_t(a.pool) * hb;
        co = sl + int64_t(a.pool) * (1 - hb);
    }
    const S* from = static_cast<const S*>(a.cs_in) + ci * K1 * C;
    float taps[kItems][3];
#pragma unroll
    for (int i = 0; i < kItems; ++i)
        if (kStepThreads * i < count)
#pragma unroll
            for (int j = 0; j < 3; ++j) taps[i][j] = j < K1 ? Act::load(from, int64_t(j) * C + ch[i]) : 0.f;

    const int lane = tid % kLanes, row = tid / kLanes, n0 = 4 * lane;
    const bool cols = n0 < N;
    const int64_t tile = ((int64_t(sl) * H + h) * P + p_lo) * N + n0;
    f32x4 s[kPass];
    const auto load_pass = [&](int p0) {
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
            const int p = p0 + i * kRows + row;
            s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (cols && p < rows)
                s[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(a.S_in + tile + int64_t(p) * N));
        }
    };
    load_pass(0);

    float u[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        u[i] = 0.f;
        if (kStepThreads * i < count) {
            // the last of K taps is the current token
            u[i] = bias[i];
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (j < K1) u[i] = __builtin_fmaf(w[i][j], taps[i][j], u[i]);
            u[i] = __builtin_fmaf(K1 == 3 ? w[i][3] : K1 == 2 ? w[i][2] : w[i][1], now[i], u[i]);
        }
    }
    silu_all<GDN_F32>(u);
    S* to = static_cast<S*>(a.cs_out) + co * K1 * C;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int at = tid + kStepThreads * i, k = at - rows;
        if (at < count) {
            (k < 0 ? xs[at] : k < N ? Bs[k] : Cs[k - N]) = u[i];
            if (k < 0 || (h % per == 0 && part == 0)) {
                if (K1 > 1) Act::store(to, ch[i], taps[i][1]);
                if (K1 > 2) Act::store(to, int64_t(C) + ch[i], taps[i][2]);
                Act::store(to, int64_t(K1 - 1) * C + ch[i], now[i]);
            }
        }
    }
    if (tid == 0) {
        const float d = softplus(dt);
        gates[0] = d;
        gates[1] = expf(-expf(A) * d);
    }
    __syncthreads();
    // Every thread has read the slot's half: this workgroup's share of the
    // step's 2^16. The shares add up to it exactly, so bit 16 flips with the
    // last of them.
    if (a.arrivals && tid == 0) {
        const int mine = int(uint32_t(kStepCounter) * uint32_t(block + 1) / uint32_t(blocks) -
                             uint32_t(kStepCounter) * uint32_t(block) / uint32_t(blocks));
        __hip_atomic_fetch_add(&a.arrivals[sl], mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    f32x4 Bv = {0.f, 0.f, 0.f, 0.f}, Cv = Bv;
    if (cols) {
        Bv = *reinterpret_cast<const f32x4*>(Bs + n0);
        Cv = *reinterpret_cast<const f32x4*>(Cs + n0);
    }
    const float d = gates[0], g = gates[1], skip = a.D ? a.D[h] : 0.f;
    for (int p0 = 0; p0 < rows; p0 += kPass * kRows) {
        if (p0) load_pass(p0);
        float dot[kPass], xr[kPass];
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
            const int p = p0 + i * kRows + row;
            xr[i] = p < rows ? xs[p] : 0.f;
            dot[i] = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[i][e] = __builtin_fmaf(g, s[i][e], d * xr[i] * Bv[e]);
                dot[i] = __builtin_fmaf(s[i][e], Cv[e], dot[i]);
            }
            if (cols && p < rows)
                __builtin_nontemporal_store(s[i], reinterpret_cast<f32x4*>(a.S_out + tile + int64_t(p) * N));
        }
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
            const float y = group_sum<kLanes>(dot[i]);
            const int p = p0 + i * kRows + row;
            if (lane == 0 && p < rows)
                store_any(a.y, (int64_t(b) * H + h) * P + p_lo + p, a.y_dtype, a.D ? __builtin_fmaf(skip, xr[i], y) : y);
        }
    }
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_selective_step(const void* xbc, int64_t xbc_stride, const void* dt, int64_t dt_stride,
                                  const void* conv_state_in, void* conv_state_out, const float* conv_weight,
                                  const float* conv_bias, const float* A_log, const float* dt_bias, const float* D,
                                  const float* state_in, float* state_out, void* y, int y_dtype, int B, int G, int H,
                                  int P, int N, int K, int act_dtype, const int32_t* slots, int pool,
                                  const int32_t* conv_half, int32_t* conv_arrivals, void* stream) {
    GDN_REQUIRE(B >= 0 && G > 0 && H > 0 && H % G == 0 && P > 0 && N > 0,
                "gdn_selective_step: bad sizes B=%d G=%d H=%d P=%d N=%d", B, G, H, P, N);
    GDN_REQUIRE(valid_dtype(act_dtype) && valid_dtype(y_dtype), "gdn_selective_step: bad dtype");
    if (N % 8 || N > kMaxState || P > kMaxHead || K < 2 || K > 4)
        return fail(GDN_EUNSUPPORTED,
                    "gdn_selective_step: state_dim a multiple of 8 up to %d, head_dim up to %d, 2 to 4 taps "
                    "(got %d, %d, %d)", kMaxState, kMaxHead, N, P, K);
    if (B == 0) return 0;
    GDN_REQUIRE(xbc && dt && conv_state_in && conv_state_out && conv_weight && A_log && dt_bias && state_in &&
                    state_out && y,
                "gdn_selective_step: null pointer");
    if (!slots) pool = B;
    GDN_REQUIRE(pool >= 1, "gdn_selective_step: bad pool size %d", pool);
    GDN_REQUIRE(!conv_half || slots, "gdn_selective_step: conv_half needs slots");
    GDN_REQUIRE(!conv_arrivals || conv_half, "gdn_selective_step: conv_arrivals needs conv_half");
    const int64_t C = int64_t(H) * P + 2 * int64_t(G) * N;
    GDN_REQUIRE(C <= INT32_MAX, "gdn_selective_step: too many channels");
    GDN_REQUIRE(xbc_stride >= C && dt_stride >= H, "gdn_selective_step: row strides %lld, %lld below %lld, %d",
                (long long)xbc_stride, (long long)dt_stride, (long long)C, H);
    const int64_t row_bytes = (K - 1) * C * dtype_size(act_dtype);
    if (conv_half)
        GDN_REQUIRE(conv_state_in == conv_state_out,
                    "gdn_selective_step: with conv_half, conv_state_in and conv_state_out are one array");
    else
        GDN_REQUIRE(!overlaps(conv_state_in, int64_t(pool) * row_bytes, conv_state_out, int64_t(B) * row_bytes),
                    "gdn_selective_step: conv_state_out overlaps conv_state_in");
    const int64_t state_bytes = int64_t(pool) * H * P * N * 4;
    GDN_REQUIRE(state_in == state_out || !overlaps(state_in, state_bytes, state_out, state_bytes),
                "gdn_selective_step: state_out partially overlaps state_in");
    GDN_REQUIRE((reinterpret_cast<uintptr_t>(state_in) | reinterpret_cast<uintptr_t>(state_out)) % 16 == 0,
                "gdn_selective_step: states must be 16-byte aligned");
    int lanes = 2;
    while (4 * lanes < N) lanes *= 2;
    const int64_t heads = int64_t(B) * H;
    int split = 1;
    while (heads * split < 64 && P / (split * 2) >= 16) split *= 2;
    GDN_REQUIRE(heads * split <= INT32_MAX && int64_t(H) * split < kStepCounter, "gdn_selective_step: B * H too large");
    const StepArgs args{xbc, xbc_stride, dt, dt_stride, conv_state_in, conv_state_out, conv_weight, conv_bias,
                        A_log, dt_bias, D, state_in, state_out, y, y_dtype, G, H, P, N, K, split, B, slots, pool,
                        conv_half, conv_arrivals};
    const auto launch = [&](auto act, auto threads, auto pass) {
        using Act = decltype(act);
        constexpr int T = decltype(threads)::value, R = decltype(pass)::value;
        const auto kern = lanes == 2 ? step_kernel<Act, 2, T, R> : lanes == 4 ? step_kernel<Act, 4, T, R>
                          : lanes == 8 ? step_kernel<Act, 8, T, R> : lanes == 16 ? step_kernel<Act, 16, T, R>
                          : lanes == 32 ? step_kernel<Act, 32, T, R> : step_kernel<Act, 64, T, R>;
        hipLaunchKernelGGL(kern, rows_of_blocks(heads * split), dim3(T), 0, as_stream(stream), args);
    };
    const auto sized = [&](auto act) {
        using std::integral_constant;
        if (heads <= 256) launch(act, integral_constant<int, 1024>{}, integral_constant<int, 2>{});
        else launch(act, integral_constant<int, 512>{}, integral_constant<int, 4>{});
    };
    if (act_dtype == GDN_F32) sized(ActF32{});
    else if (act_dtype == GDN_BF16) sized(ActBF16{});
    else sized(ActF16{});
    return check_launch("gdn_selective_step");
}
