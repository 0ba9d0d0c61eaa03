// Shared pieces of the state-space operators: the run and segment layout of
// packed prompts, SiLU, and eight values as floats.
#pragma once

#include "gdn_common.h"

namespace gdn {

// A packed batch is cut into segments of 2^shift tokens, counted from each run's
// first token. Run r's segments take the slots (cu[r] >> shift) + r and on:
// distinct for all runs whatever their lengths (a run of len tokens has at most
// (cu[r + 1] >> shift) - (cu[r] >> shift) + 1 of them), one slot at least for an
// empty run, and (T >> shift) + N in all, which the host knows without the
// offsets. With shift 31 run r has slot r alone.
struct Segment {
    int run;          // -1: no run has this slot
    int64_t t0, t1;   // its tokens
};

GDN_DEV int64_t run_start(const int32_t* cu, int64_t L, int r) { return cu ? int64_t(cu[r]) : r * L; }

// The slot's run is the last whose first slot is not past it: found 64 runs at
// a time, one load each step (a binary search waits for six).
GDN_DEV Segment segment_of(const int32_t* cu, int N, int64_t L, int shift, int slot) {
    const int lane = threadIdx.x % kWave;
    int lo = 0, count = N;
    while (count > 1) {
        const int step = (count + kWave - 1) / kWave, at = lane * step;
        const bool before = at < count && int(run_start(cu, L, lo + at) >> shift) + lo + at <= slot;
        const int last = __popcll(__ballot(before)) - 1;  // (lane 0's always is)
        lo += last * step;
        count = min(step, count - last * step);
    }
    const int64_t b = run_start(cu, L, lo), e = run_start(cu, L, lo + 1);
    const int k = slot - int(b >> shift) - lo;
    Segment s;
    s.t0 = b + (int64_t(k) << shift);
    s.t1 = min(e, s.t0 + (int64_t(1) << shift));
    s.run = k == 0 || s.t0 < e ? lo : -1;
    return s;
}

// SiLU of N float32 values, within a few float32 ulps: e^-x from the hardware's
// exp2 with the argument's rounding (up to |x| ulps of the result) put back to
// first order, and the reciprocal after one Newton step. kDt 16 bits: without
// either, within about |x| + 4 ulps. Below -80, where e^-x leaves float32, the
// form x e^x / (1 + e^x); a wave takes that only if one of its values is there.
template <int kDt, int N>
GDN_DEV void silu_all(float (&x)[N]) {
#pragma clang fp contract(off)
    constexpr float kL = 1.44269504088896341f, kLLow = 1.92596299112661746e-8f, kLn2 = 0.693147180559945309f;
    float least = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) least = fminf(least, x[i]);
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (kDt == GDN_F32) {
            const float c = fminf(x[i], 80.f);
            const float h = c * kL;
            const float l = __builtin_fmaf(c, kLLow, __builtin_fmaf(c, kL, -h));
            const float e = __builtin_amdgcn_exp2f(-h);
            const float d = 1.f + __builtin_fmaf(e, l * -kLn2, e);
            const float r = __builtin_amdgcn_rcpf(d);
            y[i] = x[i] * __builtin_fmaf(__builtin_fmaf(-d, r, 1.f), r, r);
        } else {
            y[i] = x[i] * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-x[i] * kL));
        }
    }
    if (__builtin_amdgcn_ballot_w64(least < -80.f) != 0) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (x[i] < -80.f) {
                const float e = expf(x[i]);
                y[i] = x[i] * (e / (1.f + e));
            }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = y[i];
}

// Eight values of 16 bits in 16 bytes, or of float32 in 32, as floats.
template <class Act, class V, int n>
GDN_DEV void raw8(const V (&raw)[n], float (&x)[8]) {
    static_assert(n == int(sizeof(typename Act::storage)) / 2, "eight values");
    if constexpr (Act::code == GDN_F32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(raw[e / 4][e % 4]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t d = raw[0][i];
            if constexpr (Act::code == GDN_BF16) {
                x[2 * i] = __uint_as_float(d << 16);
                x[2 * i + 1] = __uint_as_float(d & 0xFFFF0000u);
            } else {
                x[2 * i] = f16_bits_to_f32(uint16_t(d & 0xFFFF));
                x[2 * i + 1] = f16_bits_to_f32(uint16_t(d >> 16));
            }
        }
    }
}

// Eight consecutive 16-bit or float32 values as floats, from an address
// aligned to 16 bytes.
template <class Act>
GDN_DEV void load8f(const typename Act::storage* p, float (&x)[8]) {
    if constexpr (Act::code == GDN_F32) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = v[e];
    } else if constexpr (Act::code == GDN_BF16) {
        unpack8(*reinterpret_cast<const uint4*>(p), x);
    } else {
        const uint4 r = *reinterpret_cast<const uint4*>(p);
        const uint32_t d[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = f16_bits_to_f32(uint16_t(d[i] & 0xFFFF));
            x[2 * i + 1] = f16_bits_to_f32(uint16_t(d[i] >> 16));
        }
    }
}

}  // namespace gdn
