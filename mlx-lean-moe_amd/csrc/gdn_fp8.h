// Values put in e4m3 codes under one scale for 128 of them: what the fp8_block
// product and the norm with 8-bit output share.
#pragma once

#include "gdn_common.h"

namespace gdn {

constexpr int kB = 128;  // block of the scales, both ways
constexpr float kE4m3Max = 448.f;

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

// x / s to the last bit for the lane's values, s one group's scale: two
// Newton corrections of x times the rounded reciprocal, each remainder exact
// (the second starts within one ulp and so ends correctly rounded). Remainders
// of the smallest scales would leave float32: divisions there.
template <int N>
GDN_DEV void divide_all(float (&x)[N], float s) {
    if (s < 0x1p-80f) {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = x[e] / s;
        return;
    }
    const float inv = 1.f / s;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        float r = x[e] * inv;
        r = __builtin_fmaf(__builtin_fmaf(-r, s, x[e]), inv, r);
        x[e] = __builtin_fmaf(__builtin_fmaf(-r, s, x[e]), inv, r);
    }
}

// Codes of four values.
GDN_DEV uint32_t codes4(float a, float b, float c, float d) {
    int r = 0;
    r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
}

// Columns of the (blocks, rows) array of the rows' scales: a tile's 256 scales are
// one aligned kilobyte.
inline int scale_columns(int M) { return (M + 255) / 256 * 256; }

}  // namespace gdn
