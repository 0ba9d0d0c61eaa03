// RMS norm over rows, with the residual's addition in front of it and, if asked,
// the result in e4m3 codes:
//   s = T(x + r),   y = T(s w / sqrt(mean(s^2) + eps)),
//   per 128 columns: scale = max(amax |y| / 448, 2^-126), code = e4m3(y / scale),
// T the rounding to the rows' type. y is formed in 64 bits and rounded to float32 and
// then to T: sums are held in 64 bits (a square of a float32 value is exact there), and so
// is each product that falls near a border of T. That is within 2^-48 of the exact value
// for rows of up to 16384 (at most 38 roundings a sum, of which the root leaves half,
// and six more), so y is the exact value's rounding but where that lies so near a border.
// A row's sum is added in an order of K alone: its y and codes do not depend on
// the rows beside it, and the codes are those that gdn_fp8_matmul makes of y.
#include <type_traits>

#include "gdn_common.h"
#include "gdn_fp8.h"
#include "gdn_host.h"

namespace gdn {
namespace {

struct NormArgs {
    const void *x, *residual;
    void *sum, *out;
    const float* w;
    uint8_t* codes;
    float* scales;
    int64_t x_stride, r_stride, s_stride, rows;
    int K, kb, ldx;
    double eps;
};

// kN consecutive values at any alignment of their own type (global memory takes
// 16-byte accesses at any address); beyond `count` of them zeros, or left alone.
template <class A, int kN>
GDN_DEV void load_some(const typename A::storage* p, int count, float* v) {
    if (count >= kN) {
        typename A::storage raw[kN];
        __builtin_memcpy(raw, p, sizeof(raw));
#pragma unroll
        for (int e = 0; e < kN; ++e) v[e] = A::load(raw, e);
        return;
    }
#pragma unroll
    for (int e = 0; e < kN; ++e) v[e] = e < count ? A::load(p, e) : 0.f;
}

template <class A, int kN>
GDN_DEV void store_some(typename A::storage* p, int count, const float* v) {
    if (count >= kN) {
        typename A::storage raw[kN];
#pragma unroll
        for (int e = 0; e < kN; ++e) A::store(raw, e, v[e]);
        __builtin_memcpy(p, raw, sizeof(raw));
        return;
    }
#pragma unroll
    for (int e = 0; e < kN; ++e)
        if (e < count) A::store(p, e, v[e]);
}

// A thread's eight columns, number c of a row's: rows of 16 bits eight beside each
// other, 16 bytes; float32 rows four and the four 64 further on, so that a load of 16
// bytes a lane leaves no holes between lanes (1531 rows of 2501: 10.0 us with 32 bytes a
// lane, 9.6 so). Sixteen threads have 128 columns either way.
template <class Act>
struct Eight {
    static constexpr int kN = Act::code == GDN_F32 ? 4 : 8;
    static GDN_DEV int first(int c) { return kN == 8 ? c * 8 : c / 16 * 128 + c % 16 * 4; }
    template <class A>  // (the weights are float32 whatever the rows are)
    static GDN_DEV void load(const typename A::storage* row, int c, int K, float (&v)[8]) {
#pragma unroll
        for (int h = 0; h < 8 / kN; ++h) load_some<A, kN>(row + first(c) + 64 * h, K - first(c) - 64 * h, v + kN * h);
    }
    static GDN_DEV void store(typename Act::storage* row, int c, int K, const float (&v)[8]) {
#pragma unroll
        for (int h = 0; h < 8 / kN; ++h) store_some<Act, kN>(row + first(c) + 64 * h, K - first(c) - 64 * h, v + kN * h);
    }
};

// y of eight values, rounded to the rows' type. In 16 bits the float32 product
// of three factors, each rounding at most half a last place, lies within 3 last
// places of the exact value: further than 4 from a border of the type (a tie of
// the dropped bits) both round alike, else the eight go through 64 bits, as do
// values near the type's or float32's smallest, and rows (`wild`) whose factor
// float32 does not hold well.
template <class Act>
GDN_DEV void scaled8(const float (&v)[8], double r, float r32, bool wild, const float (&w)[8], float (&y)[8]) {
    if constexpr (Act::code != GDN_F32) {
        constexpr uint32_t kMask = Act::code == GDN_BF16 ? 0xFFFFu : 0x1FFFu, kTie = (kMask + 1) / 2;
        constexpr float kSmall = Act::code == GDN_BF16 ? 0x1p-100f : 0x1p-14f;
        bool close = wild;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float t = v[e] * r32, f = t * w[e];
            const uint32_t low = __float_as_uint(f) & kMask;
            close |= low - (kTie - 4) <= 8u || (fminf(fabsf(t), fabsf(f)) < kSmall && v[e] != 0.f);
            y[e] = f;
        }
        if (close) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = float(double(v[e]) * r * double(w[e]));
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = Act::round(y[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = float(double(v[e]) * r * double(w[e]));
    }
}

// Eight columns of a row: the stream's values (kept or read again).
template <class Act>
GDN_DEV void stream8(const NormArgs& a, int64_t row, int c, bool live, float (&v)[8]) {
    using S = typename Act::storage;
    Eight<Act>::template load<Act>(static_cast<const S*>(a.x) + row * a.x_stride, c, a.K, v);
    if (!a.residual) return;
    float r[8];
    Eight<Act>::template load<Act>(static_cast<const S*>(a.residual) + row * a.r_stride, c, a.K, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = Act::round(v[e] + r[e]);
    if (live) Eight<Act>::store(static_cast<S*>(a.sum) + row * a.s_stride, c, a.K, v);
}

GDN_DEV double squares8(const float (&v)[8], double acc) {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = __builtin_fma(double(v[e]), double(v[e]), acc);
    return acc;
}

struct Factor {
    double r;
    float r32;
    bool wild;
};

GDN_DEV Factor factor_of(double sum, int K, double eps) {
    Factor f;
    f.r = 1.0 / sqrt(sum / double(K) + eps);
    f.r32 = float(f.r);
    f.wild = !(f.r32 > 0x1p-60f && f.r32 < 0x1p60f);
    return f;
}

// y of eight columns, stored as it is asked for. With codes, sixteen consecutive
// lanes hold the columns of one scale.
template <class Act, bool kCodes>
GDN_DEV void finish8(const NormArgs& a, int64_t row, int c, bool live, const float (&v)[8], const Factor& f) {
    using E = Eight<Act>;
    float w[8], y[8];
    if (a.w) {
        E::template load<ActF32>(a.w, c, a.K, w);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = 1.f;
    }
    scaled8<Act>(v, f.r, f.r32, f.wild, w, y);
    if (a.out && live) E::store(static_cast<typename Act::storage*>(a.out) + row * a.K, c, a.K, y);
    if constexpr (kCodes) {
        const int k = E::first(c);
#pragma unroll
        for (int e = 0; e < 8; ++e)  // (behind the last column: zeros, also in a row of NaN)
            if (k + e / E::kN * 64 >= a.K) y[e] = 0.f;
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(y[e]) & 0x7FFFFFFFu);
        const float s = scale_of(row16_max(top));
        divide_all(y, s);
        if (live && k < a.kb * kB) {
            uint8_t* to = a.codes + row * (int64_t(a.kb) * kB) + k;
            const uint32_t low = codes4(y[0], y[1], y[2], y[3]), high = codes4(y[4], y[5], y[6], y[7]);
            if constexpr (E::kN == 8) {
                *reinterpret_cast<uint2*>(to) = make_uint2(low, high);
            } else {
                *reinterpret_cast<uint32_t*>(to) = low;
                *reinterpret_cast<uint32_t*>(to + 64) = high;
            }
            if (c % 16 == 0) a.scales[int64_t(c / 16) * a.ldx + row] = s;
        }
    }
}

// The sum over a row's threads, in all of them: kLanes of a wave, or (0) the whole
// workgroup.
template <int kLanes>
GDN_DEV double row_sum(double v) {
    if constexpr (kLanes != 0) {
        return group_sum<kLanes>(v);
    } else {
        __shared__ double part[1024 / kWave];
        const int waves = blockDim.x / kWave;
        v = group_sum<kWave>(v);
        if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
        __syncthreads();
        v = part[0];
        for (int i = 1; i < waves; ++i) v += part[i];
        return v;
    }
}

// A row's columns stay in the registers of its threads, kVec times eight in each:
// memory is read once and written once, and that is what bounds it. kLanes threads
// of a wave a row, or (0) a workgroup of as many waves as the row's columns take.
// Measured, with the residual, bf16, calls one after the other: 4096 rows of 2048 13.8 us
// (67 MB, 4.9 TB/s; a large copy 5.1), 8192 to codes 26.3 (118 MB); 1 row 3.0 by
// itself, a launch and its waits.
template <class Act, int kLanes, int kVec, bool kCodes>
__global__ __launch_bounds__(kLanes ? 256 : 1024) void rms_norm_kernel(NormArgs a) {
    const int lanes = kLanes ? kLanes : blockDim.x, per = kLanes ? 256 / kLanes : 1;
    const int64_t id = int64_t(blockIdx.y) * gridDim.x + blockIdx.x;
    const int64_t mine = id * per + (kLanes ? int(threadIdx.x) / lanes : 0);
    if (id * per >= a.rows) return;  // (the last row of the grid may be short)
    const bool live = mine < a.rows;
    const int64_t row = live ? mine : a.rows - 1;
    const int lane = kLanes ? threadIdx.x % lanes : threadIdx.x;
    float v[kVec][8];
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
        stream8<Act>(a, row, j * lanes + lane, live, v[j]);
        sum = squares8(v[j], sum);
    }
    const Factor f = factor_of(row_sum<kLanes>(sum), a.K, a.eps);
#pragma unroll
    for (int j = 0; j < kVec; ++j) finish8<Act, kCodes>(a, row, j * lanes + lane, live, v[j], f);
}

// Rows longer than registers hold: the stream is read again for the second pass
// (from `sum` where there is a residual: each thread reads what it wrote).
template <class Act, bool kCodes>
__global__ __launch_bounds__(1024) void rms_norm_long_kernel(NormArgs a) {
    const int64_t row = int64_t(blockIdx.y) * gridDim.x + blockIdx.x;
    if (row >= a.rows) return;
    const int end = (a.K + 8191) / 8192 * 1024;
    float v[8];
    double sum = 0.0;
    for (int c = threadIdx.x; c < end; c += 1024) {
        stream8<Act>(a, row, c, true, v);
        sum = squares8(v, sum);
    }
    const Factor f = factor_of(row_sum<0>(sum), a.K, a.eps);
    NormArgs again = a;
    if (a.residual) again.x = a.sum, again.x_stride = a.s_stride, again.residual = nullptr;
    for (int c = threadIdx.x; c < end; c += 1024) {
        stream8<Act>(again, row, c, true, v);
        finish8<Act, kCodes>(a, row, c, true, v, f);
    }
}

template <class Act, bool kCodes>
void launch_norm(const NormArgs& a, hipStream_t s) {
    const auto rows = [&](auto kernel, int per, int threads) {
        hipLaunchKernelGGL(kernel, rows_of_blocks((a.rows + per - 1) / per), dim3(threads), 0, s, a);
    };
    // One eight a thread up to 4096 columns, two beyond (us, one and two: 1 x 4096 to
    // codes 4.0 and 4.9, 4096 x 4096 25.7 and 26.2, to codes without a residual 21.0 and
    // 19.9; 8 x 8192 4.8 and 5.4, 1000 x 5120 to codes 10.4 and 9.3, 2048 x 8192 28.6 and
    // 27.4). Rows of up to 512 columns share a workgroup.
    const int waves = (a.K + 511) / 512;  // of eight columns a thread
    if (a.K <= 128) rows(rms_norm_kernel<Act, 16, 1, kCodes>, 16, 256);
    else if (a.K <= 512) rows(rms_norm_kernel<Act, 64, 1, kCodes>, 4, 256);
    else if (waves <= 8) rows(rms_norm_kernel<Act, 0, 1, kCodes>, 1, waves * kWave);
    else if (waves <= 32) rows(rms_norm_kernel<Act, 0, 2, kCodes>, 1, (waves + 1) / 2 * kWave);
    else rows(rms_norm_long_kernel<Act, kCodes>, 1, 1024);
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int gdn_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, void* sum,
                            int64_t sum_stride, const float* w, double eps, int dtype, void* out, void* codes,
                            float* scales, int scale_stride, int64_t rows, int K, void* stream) {
    GDN_REQUIRE(rows >= 0 && K > 0 && K <= INT32_MAX - 8192, "gdn_rms_norm: bad sizes rows=%lld K=%d", (long long)rows, K);
    GDN_REQUIRE(valid_dtype(dtype), "gdn_rms_norm: bad dtype");
    if (rows == 0) return 0;
    GDN_REQUIRE(x && (out || codes), "gdn_rms_norm: null pointer");
    GDN_REQUIRE(!residual == !sum, "gdn_rms_norm: a residual goes with a sum");
    GDN_REQUIRE(x_stride >= K && (!residual || (residual_stride >= K && sum_stride >= K)),
                "gdn_rms_norm: rows closer than their width of %d", K);
    if (residual) {  // in place in either input, or apart from both
        const int es = dtype_size(dtype);
        const auto span = [&](int64_t stride) { return ((rows - 1) * stride + K) * es; };
        const auto apart = [&](const void* in, int64_t stride) {
            if ((sum == in && (sum_stride == stride || rows == 1)) || !overlaps(sum, span(sum_stride), in, span(stride))) return true;
            if (sum_stride != stride || rows == 1) return false;
            // columns of one buffer beside each other
            const int64_t row = stride * es, off = (reinterpret_cast<intptr_t>(in) - reinterpret_cast<intptr_t>(sum)) % row;
            const int64_t at = off < 0 ? off + row : off, width = int64_t(K) * es;
            return at >= width && at <= row - width;
        };
        GDN_REQUIRE(apart(x, x_stride), "gdn_rms_norm: sum overlaps x");
        GDN_REQUIRE(apart(residual, residual_stride), "gdn_rms_norm: sum overlaps residual");
    }
    const int kb = (K + kB - 1) / kB;
    if (codes) {
        GDN_REQUIRE(scales && K % 16 == 0, "gdn_rms_norm: codes need scales and K a multiple of 16, got %d", K);
        GDN_REQUIRE(rows <= INT32_MAX - 256 && scale_stride >= rows, "gdn_rms_norm: scales %d apart for %lld rows",
                    scale_stride, (long long)rows);
        GDN_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16 == 0, "gdn_rms_norm: codes must be 16-byte aligned");
    }
    const NormArgs a{x, residual, sum, out, w, static_cast<uint8_t*>(codes), scales, x_stride, residual_stride,
                     sum_stride, rows, K, kb, scale_stride, eps};
    const auto go = [&](auto act) {
        using Act = decltype(act);
        if (codes) launch_norm<Act, true>(a, as_stream(stream));
        else launch_norm<Act, false>(a, as_stream(stream));
    };
    if (dtype == GDN_F32) go(ActF32{});
    else if (dtype == GDN_BF16) go(ActBF16{});
    else go(ActF16{});
    return check_launch("gdn_rms_norm");
}
