// One token of a state-space layer for B sequences: conv + SiLU over the
// token's channels with the conv state rolled on, the step d = softplus(dt +
// dt_bias), and per head
//   S <- exp(-exp(A_log) d) S + (d x) B^T,   y = S C + D x.
//
// The float32 head_dim x state_dim state is the only large operand: it is read
// once and written once, so the kernel is bound by memory, and below a few
// hundred workgroups by latency. A workgroup takes kRows-row passes over (a
// share of) one head's state; a state row lies across kLanes lanes, four
// values each, so a wave reads 1 KB in one piece. The state's loads are issued
// first and the front-end's arithmetic runs under them. Every head of a group
// needs the group's B and C channels after the conv: each workgroup computes
// them itself (2 state_dim channels from cached rows) instead of a launch of
// its own, and the group's first workgroup rolls their conv state.
#include "gdn_host.h"
#include "gdn_ssm.h"

namespace gdn {
namespace {

constexpr int kStepThreads = 256;
constexpr int kStepCounter = 1 << 16;  // what a step adds to a slot's counter, over all its workgroups
constexpr int kPass = 8;               // rows of state a thread holds at a time
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
    int y_dtype, G, H, P, N, K, split;
    const int32_t* slots;
    int pool;
    const int32_t* half;
    int32_t* arrivals;
};

template <class Act, int kLanes>
__global__ __launch_bounds__(kStepThreads) void step_kernel(StepArgs a) {
    constexpr int kRows = kStepThreads / kLanes;  // rows of one pass
    __shared__ __attribute__((aligned(16))) float Bs[kMaxState], Cs[kMaxState], xs[kMaxHead];
    __shared__ float gate[2];
    const int P = a.P, N = a.N, H = a.H, tid = threadIdx.x;
    const int part = blockIdx.x % a.split;
    const int bh = blockIdx.x / a.split, b = bh / H, h = bh % H;
    const int per = H / a.G, grp = h / per;
    const int rows_per = (P + a.split - 1) / a.split;
    const int p_lo = min(P, part * rows_per), p_hi = min(P, p_lo + rows_per);
    const int C = H * P + 2 * a.G * N, K1 = a.K - 1;
    using S = typename Act::storage;
    const int sl = a.slots ? a.slots[b] : b;
    if (unsigned(sl) >= unsigned(a.pool)) {  // a slot outside the pool: touch no state
        for (int p = p_lo + tid; p < p_hi; p += kStepThreads)
            store_any(a.y, int64_t(bh) * P + p, a.y_dtype, __builtin_nanf(""));
        return;
    }
    int64_t ci = sl, co = b;
    if (a.half) {
        const int hb = (a.half[sl] ^ (a.arrivals ? a.arrivals[sl] >> 16 : 0)) & 1;
        ci = sl + int64_t(a.pool) * hb;
        co = sl + int64_t(a.pool) * (1 - hb);
    }
    const int lane = tid % kLanes, row = tid / kLanes, n0 = 4 * lane;
    const bool cols = n0 < N;
    const int64_t sbase = (int64_t(sl) * H + h) * P;
    const auto at = [&](int p) { return (sbase + p) * N + n0; };
    f32x4 s[kPass];
    const auto load_pass = [&](int p0) {
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
            const int p = p0 + i * kRows + row;
            s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (cols && p < p_hi)
                s[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(a.S_in + at(p)));
        }
    };
    load_pass(p_lo);

    // the conv of this head's x channels and its group's B and C channels
    const S* x = static_cast<const S*>(a.xbc) + b * a.xbc_stride;
    const S* ci_p = static_cast<const S*>(a.cs_in) + ci * K1 * C;
    S* co_p = static_cast<S*>(a.cs_out) + co * K1 * C;
    for (int i = tid; i < (p_hi - p_lo) + 2 * N; i += kStepThreads) {
        const int np = p_hi - p_lo;
        const int k = i - np;  // channel of B (below N), of C (from N on)
        const int c = k < 0 ? h * P + p_lo + i
                            : H * P + (k < N ? grp * N + k : (a.G + grp) * N + (k - N));
        const bool roll = k < 0 || (h % per == 0 && part == 0);
        float taps[3], acc = a.bias ? a.bias[c] : 0.f;
        const float now = Act::load(x, c);
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < K1) taps[j] = Act::load(ci_p, int64_t(j) * C + c);
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < K1) acc = __builtin_fmaf(a.w[int64_t(c) * a.K + j], taps[j], acc);
        float v[1] = {__builtin_fmaf(a.w[int64_t(c) * a.K + K1], now, acc)};
        silu_all<GDN_F32>(v);
        (k < 0 ? xs[i] : k < N ? Bs[k] : Cs[k - N]) = v[0];
        if (roll) {
#pragma unroll
            for (int j = 0; j + 1 < 3; ++j)
                if (j + 1 < K1) Act::store(co_p, int64_t(j) * C + c, taps[j + 1]);
            Act::store(co_p, int64_t(K1 - 1) * C + c, now);
        }
    }
    if (tid == 0) {
        const float d = softplus(Act::load(static_cast<const S*>(a.dt), b * a.dt_stride + h) + a.dt_bias[h]);
        gate[0] = d;
        gate[1] = expf(-expf(a.A_log[h]) * d);
    }
    __syncthreads();
    // Every thread has read the slot's half: this workgroup's share of the
    // step's 2^16. The shares add up to it exactly, so bit 16 flips with the
    // last of them.
    if (a.arrivals && tid == 0) {
        const int64_t n = int64_t(H) * a.split, i = int64_t(h) * a.split + part;
        const int share = int(kStepCounter * (i + 1) / n - kStepCounter * i / n);
        __hip_atomic_fetch_add(&a.arrivals[sl], share, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    const float d = gate[0], g = gate[1], skip = a.D ? a.D[h] : 0.f;
    f32x4 Bv = {0.f, 0.f, 0.f, 0.f}, Cv = Bv;
    if (cols) {
        Bv = *reinterpret_cast<const f32x4*>(Bs + n0);
        Cv = *reinterpret_cast<const f32x4*>(Cs + n0);
    }
    for (int p0 = p_lo; p0 < p_hi; p0 += kPass * kRows) {
        if (p0 != p_lo) load_pass(p0);
        float dot[kPass];
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
            const int p = p0 + i * kRows + row;
            const float dx = p < p_hi ? d * xs[p - p_lo] : 0.f;
            dot[i] = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[i][e] = __builtin_fmaf(g, s[i][e], dx * Bv[e]);
                dot[i] = __builtin_fmaf(s[i][e], Cv[e], dot[i]);
            }
            if (cols && p < p_hi)
                __builtin_nontemporal_store(s[i], reinterpret_cast<f32x4*>(a.S_out + at(p)));
        }
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
            const float y = group_sum<kLanes>(dot[i]);
            const int p = p0 + i * kRows + row;
            if (lane == 0 && p < p_hi)
                store_any(a.y, int64_t(bh) * P + p, a.y_dtype, a.D ? __builtin_fmaf(skip, xs[p - p_lo], y) : y);
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
    while (heads * split < 512 && P / (split * 2) >= 8) split *= 2;
    GDN_REQUIRE(heads * split <= INT32_MAX && int64_t(H) * split <= kStepCounter, "gdn_selective_step: B * H too large");
    const StepArgs args{xbc, xbc_stride, dt, dt_stride, conv_state_in, conv_state_out, conv_weight, conv_bias,
                        A_log, dt_bias, D, state_in, state_out, y, y_dtype, G, H, P, N, K, split, slots, pool,
                        conv_half, conv_arrivals};
    const auto launch = [&](auto act) {
        using Act = decltype(act);
        const auto kern = lanes == 2 ? step_kernel<Act, 2> : lanes == 4 ? step_kernel<Act, 4>
                          : lanes == 8 ? step_kernel<Act, 8> : lanes == 16 ? step_kernel<Act, 16>
                          : lanes == 32 ? step_kernel<Act, 32> : step_kernel<Act, 64>;
        hipLaunchKernelGGL(kern, dim3(unsigned(heads * split)), dim3(kStepThreads), 0, as_stream(stream), args);
    };
    if (act_dtype == GDN_F32) launch(ActF32{});
    else if (act_dtype == GDN_BF16) launch(ActBF16{});
    else launch(ActF16{});
    return check_launch("gdn_selective_step");
}
