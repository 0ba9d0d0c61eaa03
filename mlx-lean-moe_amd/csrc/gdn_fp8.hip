// y = x W^T for W in e4m3 codes with one float32 scale per 128 x 128 block, x
// quantized on the way in: each row's 128-column group b to e4m3 codes q under
// its own scale s = max(amax |x| / 448, 2^-126), q = e4m3(x / s) (both float32
// divisions, then one rounding to nearest even). Then
//   y[m, n] = sum_b s[m, b] sw[n / 128, b] sum_{k in b} q[m, k] w[n, k],
// the inner sums on the 8-bit matrix cores (one 16x16x128 product per block, so
// scales meet float32 sums only), the outer one in float32.
#include "gdn_host.h"
#include "gdn_common.h"
#include "gdn_ssm.h"

namespace gdn {
namespace {

constexpr int kB = 128;  // block of the scales, both ways
constexpr float kE4m3Max = 448.f;

typedef int i32x8 __attribute__((ext_vector_type(8)));

// The largest |x| of 16 lanes as float bits, NaN above all.
GDN_DEV uint32_t row16_max(uint32_t v) {
#define GDN_DPP_MAX(CTRL) \
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 0xF, 0xF, false)))
    GDN_DPP_MAX(0xB1);
    GDN_DPP_MAX(0x4E);
    GDN_DPP_MAX(0x141);
    GDN_DPP_MAX(0x140);
#undef GDN_DPP_MAX
    return v;
}

GDN_DEV float scale_of(uint32_t amax_bits) {
    const float s = __uint_as_float(amax_bits) / kE4m3Max;
    return s < 0x1p-126f ? 0x1p-126f : s;
}

// Codes of four values.
GDN_DEV uint32_t codes4(float a, float b, float c, float d) {
    int r = 0;
    r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
}

// Rows' codes (M x kb * 128, columns past K zero) and scales (kb x M): 16 lanes
// a group of 128, 8 values a lane.
template <class Act>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(const typename Act::storage* __restrict__ x, int M, int K,
                                                           int kb, uint8_t* __restrict__ codes,
                                                           float* __restrict__ scales) {
    const int64_t groups = int64_t(M) * kb;
    const int64_t first = int64_t(blockIdx.x) * 16 + threadIdx.x / 16;
    const int64_t gi = first < groups ? first : groups - 1;
    const int m = int(gi / kb), b = int(gi % kb), k = b * kB + (threadIdx.x & 15) * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (k < K) load8f<Act>(x + int64_t(m) * K + k, v);
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    const float s = scale_of(row16_max(top));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] / s;
    if (first >= groups) return;
    *reinterpret_cast<uint2*>(codes + int64_t(m) * kb * kB + k) =
        make_uint2(codes4(v[0], v[1], v[2], v[3]), codes4(v[4], v[5], v[6], v[7]));
    if ((threadIdx.x & 15) == 0) scales[int64_t(b) * M + m] = s;
}

struct Fp8Args {
    const uint8_t *q, *w;
    const float *sx, *sw;
    const void* residual;
    void* y;
    int y_dtype, M, N, K, kb;
};

GDN_DEV f32x4 mfma_fp8(uint4 a0, uint4 a1, uint4 b0, uint4 b1) {
    const i32x8 a = {int(a0.x), int(a0.y), int(a0.z), int(a0.w), int(a1.x), int(a1.y), int(a1.z), int(a1.w)};
    const i32x8 b = {int(b0.x), int(b0.y), int(b0.z), int(b0.w), int(b1.x), int(b1.y), int(b1.z), int(b1.w)};
    // both operands e4m3 (format 0), block exponents of 127: factors of one
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0x7F7F7F7F, 0,
                                                            0x7F7F7F7F);
}

// Eight codes as bfloat16, exactly.
GDN_DEV bf16x8 widen8(uint32_t lo, uint32_t hi) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The same block's product with float32 sums to the last bits: the 8-bit
// matrix cores add a block's products on a common exponent with about 13 bits
// below the largest (measured against 64 bits: 1.3e-5 of the result's norm for
// normal operands, 5.4e-5 for ones of wide range), which 16-bit results do not
// show and float32 ones do. So those take the codes widened to bfloat16.
GDN_DEV f32x4 mfma_widened(uint4 a0, uint4 a1, uint4 b0, uint4 b1) {
    f32x4 c = {0.f, 0.f, 0.f, 0.f};
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(a0.x, a0.y), widen8(b0.x, b0.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(a0.z, a0.w), widen8(b0.z, b0.w), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(a1.x, a1.y), widen8(b1.x, b1.y), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(a1.z, a1.w), widen8(b1.z, b1.w), c, 0, 0, 0);
}

// Four results of row m, columns n .. n + 3: the product rounded to y's type,
// then the residual added and rounded again.
GDN_DEV void store4(const Fp8Args& a, int m, int n, f32x4 v) {
    if (m >= a.M) return;
    const int64_t at = int64_t(m) * a.N + n;
    if (a.N % 4 == 0 && n + 3 < a.N) {
        if (a.residual) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = round_to(v[i], a.y_dtype) + load_any(a.residual, at + i, a.y_dtype);
        }
        if (a.y_dtype == GDN_F32) {
            *reinterpret_cast<f32x4*>(static_cast<float*>(a.y) + at) = v;
        } else if (a.y_dtype == GDN_BF16) {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.y) + at) =
                make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        } else {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.y) + at) =
                make_uint2(f32_to_f16_bits(v[0]) | uint32_t(f32_to_f16_bits(v[1])) << 16,
                           f32_to_f16_bits(v[2]) | uint32_t(f32_to_f16_bits(v[3])) << 16);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < a.N) {
            float o = v[i];
            if (a.residual) o = round_to(o, a.y_dtype) + load_any(a.residual, at + i, a.y_dtype);
            store_any(a.y, at + i, a.y_dtype, o);
        }
}

// One wave per 16 rows of W and 16 rows of x, operands straight from memory.
template <bool kExact>
__global__ __launch_bounds__(64) void fp8_simple_kernel(Fp8Args a) {
    const int lane = threadIdx.x, g = lane >> 4, lr = lane & 15;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
    const int n = min(n0 + lr, a.N - 1), m = min(m0 + lr, a.M - 1);
    const uint8_t* wr = a.w + int64_t(n) * a.K;
    const uint8_t* qr = a.q + int64_t(m) * a.kb * kB;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int b = 0; b < a.kb; ++b) {
        const int k = b * kB + 32 * g;
        const uint4 w0 = k < a.K ? *reinterpret_cast<const uint4*>(wr + k) : zero;
        const uint4 w1 = k + 16 < a.K ? *reinterpret_cast<const uint4*>(wr + k + 16) : zero;
        const uint4 q0 = *reinterpret_cast<const uint4*>(qr + k), q1 = *reinterpret_cast<const uint4*>(qr + k + 16);
        const f32x4 p = kExact ? mfma_widened(w0, w1, q0, q1) : mfma_fp8(w0, w1, q0, q1);
        const float s = a.sx[int64_t(b) * a.M + m] * a.sw[int64_t(n0 / kB) * a.kb + b];
        acc += s * p;
    }
    store4(a, m0 + lr, n0 + 4 * g, acc);
}

// The dense weights: code times its block's scale, one rounding. 16 codes a
// thread.
__global__ __launch_bounds__(256) void fp8_dequantize_kernel(const uint8_t* __restrict__ w,
                                                             const float* __restrict__ sw, void* __restrict__ out,
                                                             int out_dtype, int N, int K, int kb) {
    const int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 16;
    if (i >= int64_t(N) * K) return;
    const int n = int(i / K), k = int(i % K);
    const uint4 c = *reinterpret_cast<const uint4*>(w + i);
    const float s = sw[int64_t(n / kB) * kb + k / kB];
    const uint32_t d[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        store_any(out, i + 4 * j, out_dtype, s * __builtin_amdgcn_cvt_f32_fp8(int(d[j]), 0));
        store_any(out, i + 4 * j + 1, out_dtype, s * __builtin_amdgcn_cvt_f32_fp8(int(d[j]), 1));
        store_any(out, i + 4 * j + 2, out_dtype, s * __builtin_amdgcn_cvt_f32_fp8(int(d[j]), 2));
        store_any(out, i + 4 * j + 3, out_dtype, s * __builtin_amdgcn_cvt_f32_fp8(int(d[j]), 3));
    }
}

int64_t codes_bytes(int M, int K) { return (int64_t(M) * ((K + kB - 1) / kB) * kB + 255) / 256 * 256; }

bool fp8_sizes_ok(int M, int N, int K) {
    return M >= 0 && N > 0 && K > 0 && K % 16 == 0 && K <= INT32_MAX - kB && N <= INT32_MAX - 256 && M <= INT32_MAX - 256;
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int64_t gdn_fp8_matmul_workspace_size(int M, int N, int K) {
    if (!fp8_sizes_ok(M, N, K)) return 0;
    return codes_bytes(M, K) + int64_t(M) * ((K + kB - 1) / kB) * 4;
}

extern "C" int gdn_fp8_matmul(const void* x, int x_dtype, const void* w, const float* scales, void* y, int y_dtype,
                              const void* residual, int M, int N, int K, void* workspace, int64_t workspace_bytes,
                              void* stream) {
    GDN_REQUIRE(fp8_sizes_ok(M, N, K), "gdn_fp8_matmul: bad sizes M=%d N=%d K=%d (K a multiple of 16)", M, N, K);
    GDN_REQUIRE(valid_dtype(x_dtype) && valid_dtype(y_dtype), "gdn_fp8_matmul: bad dtype");
    if (M == 0) return 0;
    GDN_REQUIRE(x && w && scales && y, "gdn_fp8_matmul: null pointer");
    GDN_REQUIRE((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(y) |
                 reinterpret_cast<uintptr_t>(workspace)) % 16 == 0,
                "gdn_fp8_matmul: x, w, y and workspace must be 16-byte aligned");
    const int64_t need = gdn_fp8_matmul_workspace_size(M, N, K);
    GDN_REQUIRE(workspace && workspace_bytes >= need, "gdn_fp8_matmul: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)need);
    const int kb = (K + kB - 1) / kB;
    const int64_t blocks = (int64_t(M) * kb + 15) / 16;
    GDN_REQUIRE(blocks <= INT32_MAX && (M + 15) / 16 <= 65535, "gdn_fp8_matmul: too many rows");
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    float* sx = reinterpret_cast<float*>(codes + codes_bytes(M, K));
    hipStream_t s = as_stream(stream);
    const auto quantize = [&](auto act) {
        using Act = decltype(act);
        hipLaunchKernelGGL(fp8_quantize_kernel<Act>, dim3(unsigned(blocks)), dim3(256), 0, s,
                           static_cast<const typename Act::storage*>(x), M, K, kb, codes, sx);
    };
    if (x_dtype == GDN_F32) quantize(ActF32{});
    else if (x_dtype == GDN_BF16) quantize(ActBF16{});
    else quantize(ActF16{});
    const Fp8Args a{codes, static_cast<const uint8_t*>(w), sx, scales, residual, y, y_dtype, M, N, K, kb};
    hipLaunchKernelGGL(y_dtype == GDN_F32 ? fp8_simple_kernel<true> : fp8_simple_kernel<false>, dim3(unsigned((N + 15) / 16), unsigned((M + 15) / 16)), dim3(64), 0, s, a);
    return check_launch("gdn_fp8_matmul");
}

extern "C" int gdn_fp8_dequantize(const void* w, const float* scales, void* out, int out_dtype, int N, int K,
                                  void* stream) {
    GDN_REQUIRE(fp8_sizes_ok(0, N, K), "gdn_fp8_dequantize: bad sizes N=%d K=%d (K a multiple of 16)", N, K);
    GDN_REQUIRE(valid_dtype(out_dtype), "gdn_fp8_dequantize: bad dtype");
    GDN_REQUIRE(w && scales && out, "gdn_fp8_dequantize: null pointer");
    GDN_REQUIRE(reinterpret_cast<uintptr_t>(w) % 16 == 0, "gdn_fp8_dequantize: w must be 16-byte aligned");
    const int64_t blocks = (int64_t(N) * K / 16 + 255) / 256;
    GDN_REQUIRE(blocks <= INT32_MAX, "gdn_fp8_dequantize: too many weights");
    hipLaunchKernelGGL(fp8_dequantize_kernel, dim3(unsigned(blocks)), dim3(256), 0, as_stream(stream),
                       static_cast<const uint8_t*>(w), scales, out, out_dtype, N, K, (K + kB - 1) / kB);
    return check_launch("gdn_fp8_dequantize");
}
