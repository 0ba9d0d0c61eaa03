// The selective state-space scan over packed runs. Per head, with
// d_t = softplus(dt_t + dt_bias) and l_t = -exp(A_log) d_t,
//   S_t = exp(l_t) S_{t-1} + (d_t x_t) B_t^T,   y_t = S_t C_t + D x_t,
// S head_dim x state_dim, B and C shared by the heads of a group.
//
// Within a chunk of Q tokens, with c_t = l_1 + .. + l_t of the chunk and S the
// state before it, that is
//   y_t = exp(c_t) S C_t + sum_{s <= t} (C_t . B_s) exp(c_t - c_s) d_s x_s + D x_t
//   S'  = exp(c_Q) S + sum_s exp(c_Q - c_s) d_s x_s B_s^T,
// four matrix products: C B^T (Q x Q, one for all heads of a group), the
// masked and decayed scores times x, S C^T, and x'^T B. They run on the matrix
// cores; the chain over chunks is only S' in accumulator registers.
//
// A long run on few heads leaves most CUs idle, so runs are cut into segments:
// a first pass forms each segment's own sum of x'^T B (the state after it from
// an empty one) and its decay, a second one chains these, elementwise, into the
// state before each segment, and the last one computes y from there. The first
// pass costs one of the four products again.
#include <type_traits>

#include "gdn_host.h"
#include "gdn_ssm.h"
#include "gdn_ssm_plan.h"

namespace gdn {
namespace {

constexpr int kScanThreads = 256;
constexpr int kMaxGridY = 65535;
constexpr double kLog2e = 1.4426950408889634;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

struct ScanArgs {
    const void *x, *B, *C, *dt;
    int64_t x_stride, B_stride, C_stride, dt_stride;
    int dt_dtype;
    const float *A_log, *dt_bias, *D, *S_in;
    float* S_out;
    void* y;
    int y_dtype;
    const int32_t* cu;
    int runs;
    int64_t L;
    int shift;  // segments of 2^shift tokens
    int G, H, P, N;
    float *part, *decay;  // per (slot, head): a segment's own sum, then the state before it; its decay
    int segmented, slots;
};

// The running sum over the wave's lanes (DPP moves: rows of 16, then the rows'
// ends handed on).
template <int kCtrl, int kRows>
GDN_DEV double dpp_add(double c) {
    const int64_t u = __double_as_longlong(c);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, int(u), kCtrl, kRows, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, int(u >> 32), kCtrl, kRows, 0xF, false);
    return c + __longlong_as_double(int64_t(lo | uint64_t(hi) << 32));
}

GDN_DEV double running_sum(double c) {
    c = dpp_add<0x111, 0xF>(c);  // row_shr 1, 2, 4, 8
    c = dpp_add<0x112, 0xF>(c);
    c = dpp_add<0x114, 0xF>(c);
    c = dpp_add<0x118, 0xF>(c);
    c = dpp_add<0x142, 0xA>(c);  // row_bcast 15, 31
    return dpp_add<0x143, 0xC>(c);
}

GDN_DEV double lane_value(double c, int lane) {
    const int64_t u = __double_as_longlong(c);
    const uint32_t lo = __builtin_amdgcn_readlane(int(u), lane), hi = __builtin_amdgcn_readlane(int(u >> 32), lane);
    return __longlong_as_double(int64_t(lo | uint64_t(hi) << 32));
}

// The exponent of a token's decay, a power of two. At -256 and below the decay is
// zero in float32, and so is every product with it: the exponent stays at -256
// there, so that one such token does not take the bits of the sum that the decays
// between later tokens are differences of (a step of 1000 at a rate of 8000 is an
// exponent of 1e7, which leaves 24 bits of a tile's sum no digit behind the
// point). NaN stays NaN.
GDN_DEV double exponent(float d, float rate) {
    const double l = double(d) * double(rate) * kLog2e;
    return l < -256.0 ? -256.0 : l;
}

// The decays of one chunk, per token (all in powers of two): c_t as the sum of
// two floats, d_t, exp(c_t), and d_t exp(c_Q - c_t). The running sum is in
// double: what counts are differences of its terms, and a chunk's sum reaches
// thousands where single terms are 1e-3. (These are read 16 bytes at a time, and
// stand in arrays.)
template <int Q>
struct alignas(16) Decays {
    float hi[Q], lo[Q], d[Q], e[Q], w[Q], end;
};

template <int Q>
GDN_DEV double chunk_decays(Decays<Q>& o, int lane, float d, float rate) {
    const double c = running_sum(exponent(d, rate)), end = lane_value(c, Q - 1);
    if (lane < Q) {
        const float hi = float(c);
        o.hi[lane] = hi;
        o.lo[lane] = float(c - double(hi));
        o.d[lane] = d;
        o.e[lane] = __builtin_amdgcn_exp2f(hi);
        o.w[lane] = d * __builtin_amdgcn_exp2f(float(end - c));
    }
    if (lane == 0) o.end = __builtin_amdgcn_exp2f(float(end));
    return end;
}

// For scores rounded to bfloat16, tile by tile of 16 tokens: with r the sum up
// to the tile t lies in, exp(c_t - c_s) is exp(c_t - r) exp(r - c_s) for every s
// before the tile, neither above one; only a tile's own pairs take an
// exponential each. (Near is c - r, at most 16 x 256: its 24 bits leave a decay
// 2^-12, the score keeps 2^-8.)
struct alignas(16) TileDecays {
    float near[64], d[64], from[64], e[64], w[64], to[3][64], end;
};

GDN_DEV double tile_decays(TileDecays& o, int lane, float d, float rate) {
    const double c = running_sum(exponent(d, rate)), end = lane_value(c, 63);
    const double r1 = lane_value(c, 15), r2 = lane_value(c, 31), r3 = lane_value(c, 47);
    const float near = float(c - (lane < 16 ? 0.0 : lane < 32 ? r1 : lane < 48 ? r2 : r3));
    o.near[lane] = near;
    o.d[lane] = d;
    o.from[lane] = __builtin_amdgcn_exp2f(near);
    o.e[lane] = __builtin_amdgcn_exp2f(float(c));
    o.w[lane] = d * __builtin_amdgcn_exp2f(float(end - c));
    o.to[0][lane] = lane < 16 ? d * __builtin_amdgcn_exp2f(float(r1 - c)) : 0.f;
    o.to[1][lane] = lane < 32 ? d * __builtin_amdgcn_exp2f(float(r2 - c)) : 0.f;
    o.to[2][lane] = lane < 48 ? d * __builtin_amdgcn_exp2f(float(r3 - c)) : 0.f;
    if (lane == 0) o.end = __builtin_amdgcn_exp2f(float(end));
    return end;
}

// Memory from `p` on as a buffer for 31-bit byte offsets. A lane with nothing
// to fetch (a token past the segment, a column past the row) asks for kNowhere,
// beyond the buffer: it reads zero and stores nothing, without a branch.
constexpr int kNowhere = 0x7FFFFF00;

GDN_DEV __amdgpu_buffer_rsrc_t buffer_at(const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, p ? kNowhere : 0, 0x00027000);
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

GDN_DEV u32x4 load16(__amdgpu_buffer_rsrc_t r, int at, int more) {
    return __builtin_amdgcn_raw_buffer_load_b128(r, at, more, 0);
}

GDN_DEV f32x4 mfma_bf16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

GDN_DEV bf16x8 frag(uint4 v) { return __builtin_bit_cast(bf16x8, v); }

// Operand of 16 columns of a row-major LDS tile, rows r0 .. r0 + 7, by
// transposing reads: within each 16-lane group, lane i receives element i % 4
// of source lane i / 4 + 4 k, k = 0 .. 3. The 16 columns are four groups of
// four from col on, kApart apart.
template <int kApart>
GDN_DEV bf16x8 column_frag(const uint16_t* tile, int stride, int r0, int col, int sl) {
    const uint16_t* a = tile + (r0 + (sl >> 2)) * stride + col + kApart * (sl & 3);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + 4 * stride));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// bfloat16 inputs and output, 64-token chunks, four waves. A workgroup covers
// kHeads heads of one group and 64 kTiles / kHeads head_dim rows of each; a
// wave owns 16 kTiles rows of one head: its S^T (state_dim x rows) in
// accumulators, which are at once the left operand of S C^T, so the state
// never passes through LDS. kNP: state_dim rounded up to 32, 64, 128 or 256.
//
// Roundings to bfloat16: the decayed scores and, as the operand of S C^T, a
// copy of the state; both only enter y, which is bfloat16 itself (error against
// 64 bits 1.9e-3, 1.7e-3 of it y's own rounding; nearly all of the difference is
// the scores': the state in two pieces gave 1.9e-3 too and cost 4 %, and scores in
// two pieces would leave LDS room for one workgroup a CU). The state's own update
// takes x' = d exp(c_Q - c) x in three bfloat16 pieces, all 24 bits (two left 2.7e-6
// of the state behind, and took 0.85 of the time).
//
// Bound by the chain of chunks: two workgroups a CU leave the matrix cores 19 %,
// the vector units 36 % and LDS 40 % busy (12 of them bank conflicts), 6.2 us a
// chunk. Eight waves a workgroup, 128 registers each, spilled and took twice as
// long; LDS rows with their pieces permuted or spaced apart were no faster.
// Measured, state_dim 128: 41 tokens of 32 heads of 64 9.5 us; 4096 of 64 heads in
// segments of 256 26.7 for their sums, 12.5 for the chain, 44.2 for y (87 MB
// without the segments' states: 1.0 TB/s).
template <int kNP, int kHeads, int kTiles, bool kStateOnly>
__global__ __launch_bounds__(kScanThreads, kNP <= 128 ? 2 : 1) void scan_bf16_kernel(ScanArgs a) {
    constexpr int Q = 64, NS = kNP + 8, PW = 64 * kTiles, PH = PW / kHeads, XS = PW + 8, WS = Q + 8;
    constexpr int kRowsN = kNP / 8;                     // 16-byte pieces of a B or C row
    constexpr int kLoadN = Q * kRowsN / kScanThreads, kLoadX = Q * (PW / 8) / kScanThreads;
    constexpr int NT = kNP / 16, KS = kNP / 32;
    __shared__ __attribute__((aligned(16))) uint16_t Bs[Q * NS], Cs[kStateOnly ? 8 : Q * NS], Xs[Q * XS],
        Ws[kStateOnly ? 8 : kHeads * Q * WS];
    __shared__ __attribute__((aligned(16))) TileDecays decays[2][kHeads];

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, lr = lane & 15;
    const int P = a.P, N = a.N, H = a.H;
    const int tiles = (P + PH - 1) / PH;
    const int unit = blockIdx.x, slot = blockIdx.y + blockIdx.z * kMaxGridY;
    if (slot >= a.slots) return;
    const int pair = tiles == 1 ? unit : unit / tiles;
    const int h0 = pair * kHeads, p0 = tiles == 1 ? 0 : (unit - pair * tiles) * PH;
    const int grp = a.G == 1 ? 0 : h0 / (H / a.G);
    const Segment sg = segment_of(a.cu, a.runs, a.L, a.shift, slot);
    if (sg.run < 0) return;
    const int hb = wave * kHeads / 4, h = h0 + hb;
    const int pw = wave * 16 * kTiles;   // the wave's first row in the workgroup's, and in its head's
    const int pl = p0 + pw - hb * PH;

    // What a thread fetches of a chunk: the same 16-byte piece of every
    // 256 / kRowsN-th row of B and C, and of every 2048 / PW-th row of x
    constexpr int kStepN = kScanThreads / kRowsN, kStepX = kScanThreads * 8 / PW;
    const int row_n = tid / kRowsN, n_at = tid % kRowsN * 8, row_x = tid / (PW / 8), col_x = tid % (PW / 8) * 8;
    const int at_b = n_at < N ? int(row_n * a.B_stride + n_at) * 2 : kNowhere;
    const int at_c = n_at < N ? int(row_n * a.C_stride + n_at) * 2 : kNowhere;
    const int p_x = p0 + col_x % PH;
    const int at_x = p_x < P ? int(row_x * a.x_stride + (col_x / PH) * P + p_x) * 2 : kNowhere;
    u32x4 rb[kLoadN], rc[kStateOnly ? 1 : kLoadN], rx[kLoadX];
    float rdt = 0.f;
    const auto fetch = [&](int64_t t0) {
        const int left = int(min(sg.t1 - t0, int64_t(Q)));
        if (wave < kHeads && lane < left)  // (first: waited for first)
            rdt = load_any(a.dt, (t0 + lane) * a.dt_stride + h0 + wave, a.dt_dtype);
        const auto br = buffer_at(static_cast<const uint16_t*>(a.B) + t0 * a.B_stride + grp * N);
        const auto cr = buffer_at(static_cast<const uint16_t*>(a.C) + t0 * a.C_stride + grp * N);
        const auto xr = buffer_at(static_cast<const uint16_t*>(a.x) + t0 * a.x_stride + int64_t(h0) * P);
#pragma unroll
        for (int i = 0; i < kLoadN; ++i) {
            const bool in = row_n + i * kStepN < left;
            rb[i] = load16(br, in ? at_b : kNowhere, int(i * kStepN * a.B_stride * 2));
            if constexpr (!kStateOnly) rc[i] = load16(cr, in ? at_c : kNowhere, int(i * kStepN * a.C_stride * 2));
        }
#pragma unroll
        for (int i = 0; i < kLoadX; ++i)
            rx[i] = load16(xr, row_x + i * kStepX < left ? at_x : kNowhere, int(i * kStepX * a.x_stride * 2));
    };

    const float rate = wave < kHeads ? -expf(a.A_log[h0 + wave]) : 0.f;
    const float dtb = wave < kHeads ? a.dt_bias[h0 + wave] : 0.f;
    const float skip = !kStateOnly && a.D ? a.D[h] : 0.f;
    double total = 0.0;

    const auto form_decays = [&](TileDecays* dec, int64_t t0) {
        if (wave < kHeads) total += tile_decays(dec[wave], lane, t0 + lane < sg.t1 ? softplus(rdt + dtb) : 0.f, rate);
    };
    // the state before the segment: tiles 2 k and 2 k + 1 of the wave's S^T hold
    // columns p = lr and rows n = 32 k + 8 g + i and + 4 + i, so that the pair is
    // an operand over n in order
    f32x4 S[kTiles][NT];
    const int64_t slot_state = (int64_t(slot) * H + h) * P, run_state = (int64_t(sg.run) * H + h) * P;
    const auto from = buffer_at(kStateOnly ? nullptr : a.segmented ? a.part + slot_state * N
                                             : a.S_in ? a.S_in + run_state * N : nullptr);
    const auto state_at = [&](int pt, int j) {  // bytes; four values of row n of column p
        const int p = pl + 16 * pt + lr, n = 32 * (j / 2) + 8 * g + 4 * (j & 1);
        return p < P && n < N ? (p * N + n) * 4 : kNowhere;
    };
    // (the first chunk's loads go out before the state's, which it needs last)
    if (sg.t0 < sg.t1) fetch(sg.t0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int pt = 0; pt < kTiles; ++pt)
#pragma unroll
        for (int j = 0; j < NT; ++j) S[pt][j] = __builtin_bit_cast(f32x4, load16(from, state_at(pt, j), 0));
    __builtin_amdgcn_sched_barrier(0);
    if (sg.t0 < sg.t1) form_decays(decays[0], sg.t0);
    int at_decays = 0;
    for (int64_t t0 = sg.t0; t0 < sg.t1; t0 += Q, at_decays ^= 1) {
        const TileDecays* dec = decays[at_decays];
#pragma unroll
        for (int i = 0; i < kLoadN; ++i) {
            const int o = (row_n + i * kStepN) * NS + n_at;
            *reinterpret_cast<u32x4*>(Bs + o) = rb[i];
            if constexpr (!kStateOnly) *reinterpret_cast<u32x4*>(Cs + o) = rc[i];
        }
#pragma unroll
        for (int i = 0; i < kLoadX; ++i) *reinterpret_cast<u32x4*>(Xs + (row_x + i * kStepX) * XS + col_x) = rx[i];
        __syncthreads();
        if (t0 + Q < sg.t1) fetch(t0 + Q);

        if constexpr (!kStateOnly) {
            // the wave's 16 tokens' scores against all tokens up to them, as
            // columns (D: rows s, column t), decayed per head
            const int t = 16 * wave + lr;
            bf16x8 cf[KS];
#pragma unroll
            for (int k = 0; k < KS; ++k) cf[k] = frag(*reinterpret_cast<const uint4*>(Cs + t * NS + 32 * k + 8 * g));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j > (wave | 1)) break;
                f32x4 sc = {0.f, 0.f, 0.f, 0.f};
                if (j <= wave) {
#pragma unroll
                    for (int k = 0; k < KS; ++k)
                        sc = mfma_bf16(frag(*reinterpret_cast<const uint4*>(Bs + (16 * j + lr) * NS + 32 * k + 8 * g)),
                                       cf[k], sc);
                }
                const int s0 = 16 * j + 4 * g;
#pragma unroll
                for (int hh = 0; hh < kHeads; ++hh) {
                    float v[4] = {0.f, 0.f, 0.f, 0.f};
                    if (j < wave) {
                        const f32x4 to = *reinterpret_cast<const f32x4*>(dec[hh].to[wave - 1] + s0);
                        const float from = dec[hh].from[t];
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = sc[i] * (to[i] * from);
                    } else if (j == wave) {
                        const f32x4 near = *reinterpret_cast<const f32x4*>(dec[hh].near + s0);
                        const f32x4 sd = *reinterpret_cast<const f32x4*>(dec[hh].d + s0);
                        const float tn = dec[hh].near[t];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            v[i] = s0 + i <= t ? sc[i] * (sd[i] * __builtin_amdgcn_exp2f(tn - near[i])) : 0.f;
                    }
                    *reinterpret_cast<uint2*>(Ws + (hh * Q + t) * WS + s0) =
                        make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
                }
            }
            __syncthreads();
        }
        // the next chunk's decays, in the other buffer: the first waves, which
        // have the fewest scores before their tokens
        if (t0 + Q < sg.t1) form_decays(decays[at_decays ^ 1], t0 + Q);

        // x^T of the wave's rows: tokens 32 q + 8 g + 0 .. 7 per lane
        bf16x8 xf[kTiles][2];
#pragma unroll
        for (int pt = 0; pt < kTiles; ++pt)
#pragma unroll
            for (int q = 0; q < 2; ++q)
                xf[pt][q] = column_frag<4>(Xs, XS, 32 * q + 8 * g, pw + 16 * pt, lr);

        // Scores of pairs that are none are zero, and zero times a value that is
        // not finite is NaN at tokens before it: such values of x leave the
        // product (for zeros) and are added to their own and later tokens alone.
        bool apart = false;
        if constexpr (!kStateOnly) {
            u16x8 top = {};
#pragma unroll
            for (int pt = 0; pt < kTiles; ++pt)
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x8, xf[pt][q]) & uint16_t(0x7FFF));
            bool any = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) any |= top[e] >= 0x7F80;
            apart = __builtin_amdgcn_ballot_w64(any) != 0;
            if (apart) {
#pragma unroll
                for (int pt = 0; pt < kTiles; ++pt)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        u16x8 v = __builtin_bit_cast(u16x8, xf[pt][q]);
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = (v[e] & 0x7F80) == 0x7F80 ? 0 : v[e];
                        xf[pt][q] = __builtin_bit_cast(bf16x8, v);
                    }
            }
        }

        if constexpr (!kStateOnly) {
            const int left = int(min(sg.t1 - t0, int64_t(Q)));
            const auto yr = buffer_at(static_cast<uint16_t*>(a.y) + (t0 * H + h) * P);
            f32x4 y[kTiles][4];
#pragma unroll
            for (int pt = 0; pt < kTiles; ++pt)
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) y[pt][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                bf16x8 sf[kTiles];
#pragma unroll
                for (int pt = 0; pt < kTiles; ++pt) {
                    const f32x4 u = S[pt][2 * k], v = S[pt][2 * k + 1];
                    sf[pt] = frag(make_uint4(pack_bf16x2(u[0], u[1]), pack_bf16x2(u[2], u[3]),
                                             pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])));
                }
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) {
                    const bf16x8 cf = frag(*reinterpret_cast<const uint4*>(Cs + (16 * tt + lr) * NS + 32 * k + 8 * g));
#pragma unroll
                    for (int pt = 0; pt < kTiles; ++pt) y[pt][tt] = mfma_bf16(sf[pt], cf, y[pt][tt]);
                }
            }
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) {
                const int t = 16 * tt + lr;
                const float e = dec[hb].e[t];
#pragma unroll
                for (int pt = 0; pt < kTiles; ++pt) y[pt][tt] *= e;
#pragma unroll
                for (int q = 0; q <= tt / 2; ++q) {
                    const bf16x8 wf = frag(*reinterpret_cast<const uint4*>(Ws + (hb * Q + t) * WS + 32 * q + 8 * g));
#pragma unroll
                    for (int pt = 0; pt < kTiles; ++pt) y[pt][tt] = mfma_bf16(xf[pt][q], wf, y[pt][tt]);
                }
#pragma unroll
                for (int pt = 0; pt < kTiles; ++pt) {
                    const int p = pl + 16 * pt + 4 * g;
                    f32x4 o = y[pt][tt];
                    if (apart)
#pragma clang loop unroll(disable)
                        for (int r = 0; r <= t; ++r) {
                            const float w = bf16_bits_to_f32(Ws[(hb * Q + t) * WS + r]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint16_t v = Xs[r * XS + pw + 16 * pt + 4 * g + i];
                                if ((v & 0x7F80) == 0x7F80) o[i] = __builtin_fmaf(w, bf16_bits_to_f32(v), o[i]);
                            }
                        }
                    if (a.D) {
                        const uint2 xv = *reinterpret_cast<const uint2*>(Xs + t * XS + pw + 16 * pt + 4 * g);
                        o[0] = __builtin_fmaf(skip, __uint_as_float(xv.x << 16), o[0]);
                        o[1] = __builtin_fmaf(skip, __uint_as_float(xv.x & 0xFFFF0000u), o[1]);
                        o[2] = __builtin_fmaf(skip, __uint_as_float(xv.y << 16), o[2]);
                        o[3] = __builtin_fmaf(skip, __uint_as_float(xv.y & 0xFFFF0000u), o[3]);
                    }
                    __builtin_amdgcn_raw_buffer_store_b64(u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])}, yr,
                                                          t < left && p < P ? (t * H * P + p) * 2 : kNowhere, 0, 0);
                }
            }
        }

        if (kStateOnly || !a.segmented || t0 + Q < sg.t1) {
            if (apart) {
#pragma unroll
                for (int pt = 0; pt < kTiles; ++pt)
#pragma unroll
                    for (int q = 0; q < 2; ++q)
                        xf[pt][q] = column_frag<4>(Xs, XS, 32 * q + 8 * g, pw + 16 * pt, lr);
            }
            const float end = dec[hb].end;
#pragma unroll
            for (int pt = 0; pt < kTiles; ++pt)
#pragma unroll
                for (int j = 0; j < NT; ++j) S[pt][j] *= end;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const f32x4 w0 = *reinterpret_cast<const f32x4*>(dec[hb].w + 32 * q + 8 * g);
                const f32x4 w1 = *reinterpret_cast<const f32x4*>(dec[hb].w + 32 * q + 8 * g + 4);
                // three pieces: the upper 16 bits as they are, twice, and the rest
                bf16x8 xw[3][kTiles];
#pragma unroll
                for (int pt = 0; pt < kTiles; ++pt) {
                    float v[8];
                    unpack8(__builtin_bit_cast(uint4, xf[pt][q]), v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] *= e < 4 ? w0[e & 3] : w1[e & 3];
#pragma unroll
                    for (int c = 0; c < 3; ++c) {
                        uint32_t up[4];
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            up[e / 2] = __builtin_amdgcn_perm(__float_as_uint(v[e + 1]), __float_as_uint(v[e]), 0x07060302u);
                            v[e] -= __uint_as_float(__float_as_uint(v[e]) & 0xFFFF0000u);
                            v[e + 1] -= __uint_as_float(__float_as_uint(v[e + 1]) & 0xFFFF0000u);
                        }
                        xw[c][pt] = frag(make_uint4(up[0], up[1], up[2], up[3]));
                    }
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const bf16x8 bf = column_frag<8>(Bs, NS, 32 * q + 8 * g, 32 * (j / 2) + 4 * (j & 1), lr);
#pragma unroll
                    for (int c = 2; c >= 0; --c)
#pragma unroll
                        for (int pt = 0; pt < kTiles; ++pt) S[pt][j] = mfma_bf16(bf, xw[c][pt], S[pt][j]);
                }
            }
        }
        __syncthreads();
    }

    if (kStateOnly || !a.segmented) {
        const auto to = buffer_at(kStateOnly ? a.part + slot_state * N : a.S_out + run_state * N);
#pragma unroll
        for (int pt = 0; pt < kTiles; ++pt)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, S[pt][j]), to, state_at(pt, j), 0, 0);
        if (kStateOnly && wave < kHeads && lane == 0 && p0 == 0)
            a.decay[int64_t(slot) * H + h0 + wave] = exp2f(float(total));
    }
}

// The same in float32 on the float32 matrix cores, 32-token chunks: inputs of
// any float type, every operand in full. k of a 16x16x4 product is the lane's
// quarter g, so step (j, i) takes element 16 j + 4 g + i: a lane's four i are
// one 16-byte read of a row, and the state's accumulators are again an operand
// as they lie.
//
// Bound by the float32 matrix cores' rate and the LDS reads of their operands
// (each 16-byte read feeds four steps). Measured, float32, 1531 tokens of 32
// heads of 128, state_dim 128: 34.6 us for the segments' sums, 10.2 for the
// chain, 54.7 for y (with four waves a workgroup the three took 115, with eight
// 93). float16 and bfloat16 with float32 y run here too, 4096 tokens of 64 heads of
// 64 170 us (bfloat16 y on the kernel above 84).
template <class Act, int kNP, int kHeads, int kWaves, bool kStateOnly>
__global__ __launch_bounds__(64 * kWaves, kNP <= 128 ? kWaves / 2 : kWaves / 4) void scan_f32_kernel(ScanArgs a) {
    constexpr int Q = 32, kThreads = 64 * kWaves, NS = kNP + 4, PW = 16 * kWaves, PH = PW / kHeads, XS = PW + 4, WS = Q + 4;
    constexpr int kRowsN = kNP / 8;
    constexpr int kLoadN = Q * kRowsN / kThreads > 0 ? Q * kRowsN / kThreads : 1;
    constexpr int kLoadX = Q * (PW / 8) / kThreads;
    constexpr int NT = kNP / 16;
    __shared__ __attribute__((aligned(16))) float Bs[Q * NS], Cs[kStateOnly ? 4 : Q * NS], Xs[Q * XS],
        Ws[kStateOnly ? 4 : kHeads * Q * WS];
    __shared__ __attribute__((aligned(16))) Decays<Q> dec[kHeads];
    using St = typename Act::storage;

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, lr = lane & 15;
    const int P = a.P, N = a.N, H = a.H;
    const int tiles = (P + PH - 1) / PH;
    const int unit = blockIdx.x, slot = blockIdx.y + blockIdx.z * kMaxGridY;
    if (slot >= a.slots) return;
    const int pair = tiles == 1 ? unit : unit / tiles;
    const int h0 = pair * kHeads, p0 = tiles == 1 ? 0 : (unit - pair * tiles) * PH;
    const int grp = a.G == 1 ? 0 : h0 / (H / a.G);
    const Segment sg = segment_of(a.cu, a.runs, a.L, a.shift, slot);
    if (sg.run < 0) return;
    const int hb = wave * kHeads / kWaves, h = h0 + hb;
    const int pw = wave * 16;
    const int pl = p0 + pw - hb * PH;

    constexpr int es = sizeof(St), kStepN = kThreads / kRowsN, kStepX = kThreads * 8 / PW;
    const int row_n = tid / kRowsN, n_at = tid % kRowsN * 8, row_x = tid / (PW / 8), col_x = tid % (PW / 8) * 8;
    const int at_b = n_at < N && row_n < Q ? int(row_n * a.B_stride + n_at) * es : kNowhere;
    const int at_c = n_at < N && row_n < Q ? int(row_n * a.C_stride + n_at) * es : kNowhere;
    const int p_x = p0 + col_x % PH;
    const int at_x = p_x < P ? int(row_x * a.x_stride + (col_x / PH) * P + p_x) * es : kNowhere;
    constexpr int kRaw = es / 2;  // 16-byte loads of eight values
    u32x4 rb[kLoadN][kRaw], rc[kStateOnly ? 1 : kLoadN][kRaw], rx[kLoadX][kRaw];
    float rdt = 0.f;
    const auto get = [&](__amdgpu_buffer_rsrc_t r, int at, int more, u32x4 (&v)[kRaw]) {
#pragma unroll
        for (int e = 0; e < kRaw; ++e) v[e] = load16(r, at, more + 16 * e);
    };
    const auto fetch = [&](int64_t t0) {
        const int left = int(min(sg.t1 - t0, int64_t(Q)));
        const auto br = buffer_at(static_cast<const St*>(a.B) + t0 * a.B_stride + grp * N);
        const auto cr = buffer_at(static_cast<const St*>(a.C) + t0 * a.C_stride + grp * N);
        const auto xr = buffer_at(static_cast<const St*>(a.x) + t0 * a.x_stride + int64_t(h0) * P);
#pragma unroll
        for (int i = 0; i < kLoadN; ++i) {
            const bool in = row_n + i * kStepN < left;
            get(br, in ? at_b : kNowhere, int(i * kStepN * a.B_stride * es), rb[i]);
            if constexpr (!kStateOnly) get(cr, in ? at_c : kNowhere, int(i * kStepN * a.C_stride * es), rc[i]);
        }
#pragma unroll
        for (int i = 0; i < kLoadX; ++i)
            get(xr, row_x + i * kStepX < left ? at_x : kNowhere, int(i * kStepX * a.x_stride * es), rx[i]);
        if (wave < kHeads && lane < left)
            rdt = load_any(a.dt, (t0 + lane) * a.dt_stride + h0 + wave, a.dt_dtype);
    };
    const auto put = [](float* p, const u32x4 (&raw)[kRaw]) {
        float v[8];
        raw8<Act>(raw, v);
        *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
    };

    const float rate = wave < kHeads ? -expf(a.A_log[h0 + wave]) : 0.f;
    const float dtb = wave < kHeads ? a.dt_bias[h0 + wave] : 0.f;
    const float skip = !kStateOnly && a.D ? a.D[h] : 0.f;
    double total = 0.0;

    f32x4 S[NT];
    const int64_t slot_state = (int64_t(slot) * H + h) * P, run_state = (int64_t(sg.run) * H + h) * P;
    const auto from = buffer_at(kStateOnly ? nullptr : a.segmented ? a.part + slot_state * N
                                             : a.S_in ? a.S_in + run_state * N : nullptr);
    const auto state_at = [&](int j) {
        const int p = pl + lr, n = 16 * j + 4 * g;
        return p < P && n < N ? (p * N + n) * 4 : kNowhere;
    };
    if (sg.t0 < sg.t1) fetch(sg.t0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NT; ++j) S[j] = __builtin_bit_cast(f32x4, load16(from, state_at(j), 0));
    __builtin_amdgcn_sched_barrier(0);
    for (int64_t t0 = sg.t0; t0 < sg.t1; t0 += Q) {
#pragma unroll
        for (int i = 0; i < kLoadN; ++i) {
            const int o = (row_n + i * kStepN) * NS + n_at;
            if (kLoadN * kStepN <= Q || row_n < Q) {
                put(Bs + o, rb[i]);
                if constexpr (!kStateOnly) put(Cs + o, rc[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kLoadX; ++i) put(Xs + (row_x + i * kStepX) * XS + col_x, rx[i]);
        if (wave < kHeads) {
            const float d = lane < Q && t0 + lane < sg.t1 ? softplus(rdt + dtb) : 0.f;
            total += chunk_decays<Q>(dec[wave], lane, d, rate);
        }
        __syncthreads();
        if (t0 + Q < sg.t1) fetch(t0 + Q);

        if constexpr (!kStateOnly) {
            // tile (tt, j) of the scores per wave: (0, 0), none, (1, 0), (1, 1);
            // of eight waves the upper four take the second head's, if any
            const int tt = (wave >> 1) & 1, j = wave & 1, part = wave >> 2;
            const int t = 16 * tt + lr, s0 = 16 * j + 4 * g;
            f32x4 sc = {0.f, 0.f, 0.f, 0.f};
            if (j <= tt && part < kHeads) {
#pragma unroll
                for (int k = 0; k < NT; ++k) {
                    const f32x4 bv = *reinterpret_cast<const f32x4*>(Bs + (16 * j + lr) * NS + 16 * k + 4 * g);
                    const f32x4 cv = *reinterpret_cast<const f32x4*>(Cs + t * NS + 16 * k + 4 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[i], cv[i], sc, 0, 0, 0);
                }
#pragma unroll
                for (int hi = 0; hi < (kWaves == 8 ? 1 : kHeads); ++hi) {
                    const int hh = kWaves == 8 ? part : hi;
                    const float thi = dec[hh].hi[t], tlo = dec[hh].lo[t];
                    f32x4 v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float diff = (thi - dec[hh].hi[s0 + i]) + (tlo - dec[hh].lo[s0 + i]);
                        v[i] = s0 + i <= t ? sc[i] * (dec[hh].d[s0 + i] * __builtin_amdgcn_exp2f(diff)) : 0.f;
                    }
                    *reinterpret_cast<f32x4*>(Ws + (hh * Q + t) * WS + s0) = v;
                }
            }
            __syncthreads();
        }

        float xf[Q / 16][4];  // x[16 j + 4 g + i] of the lane's row
#pragma unroll
        for (int j = 0; j < Q / 16; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) xf[j][i] = Xs[(16 * j + 4 * g + i) * XS + pw + lr];
        bool apart = false;  // (as in the bfloat16 kernel)
        if constexpr (!kStateOnly) {
            bool any = false;
#pragma unroll
            for (int j = 0; j < Q / 16; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) any |= !__builtin_isfinite(xf[j][i]);
            apart = __builtin_amdgcn_ballot_w64(any) != 0;
            if (apart) {
#pragma unroll
                for (int j = 0; j < Q / 16; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) xf[j][i] = __builtin_isfinite(xf[j][i]) ? xf[j][i] : 0.f;
            }
        }

        if constexpr (!kStateOnly) {
            const int left = int(min(sg.t1 - t0, int64_t(Q)));
            const auto yr = buffer_at(static_cast<char*>(a.y) + ((t0 * H + h) * P) * (a.y_dtype == GDN_F32 ? 4 : 2));
            f32x4 y[Q / 16];
#pragma unroll
            for (int tt = 0; tt < Q / 16; ++tt) y[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < NT; ++k)
#pragma unroll
                for (int tt = 0; tt < Q / 16; ++tt) {
                    const f32x4 cv = *reinterpret_cast<const f32x4*>(Cs + (16 * tt + lr) * NS + 16 * k + 4 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        y[tt] = __builtin_amdgcn_mfma_f32_16x16x4f32(S[k][i], cv[i], y[tt], 0, 0, 0);
                }
#pragma unroll
            for (int tt = 0; tt < Q / 16; ++tt) {
                const int t = 16 * tt + lr, p = pl + 4 * g;
                y[tt] *= dec[hb].e[t];
#pragma unroll
                for (int j = 0; j <= tt; ++j) {
                    const f32x4 wv = *reinterpret_cast<const f32x4*>(Ws + (hb * Q + t) * WS + 16 * j + 4 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        y[tt] = __builtin_amdgcn_mfma_f32_16x16x4f32(xf[j][i], wv[i], y[tt], 0, 0, 0);
                }
                f32x4 o = y[tt];
                if (apart)
#pragma clang loop unroll(disable)
                    for (int r = 0; r <= t; ++r) {
                        const float w = Ws[(hb * Q + t) * WS + r];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float v = Xs[r * XS + pw + 4 * g + i];
                            if (!__builtin_isfinite(v)) o[i] = __builtin_fmaf(w, v, o[i]);
                        }
                    }
                if (a.D) {
                    const f32x4 xv = *reinterpret_cast<const f32x4*>(Xs + t * XS + pw + 4 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(skip, xv[i], o[i]);
                }
                const bool in = t < left && p < P;
                const int at = (t * H * P + p) * (a.y_dtype == GDN_F32 ? 4 : 2);
                if (a.y_dtype == GDN_F32) {
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), yr, in ? at : kNowhere, 0, 0);
                } else {
                    uint16_t b[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        b[i] = a.y_dtype == GDN_BF16 ? f32_to_bf16_bits(o[i]) : f32_to_f16_bits(o[i]);
                    __builtin_amdgcn_raw_buffer_store_b64(u32x2{b[0] | uint32_t(b[1]) << 16, b[2] | uint32_t(b[3]) << 16},
                                                          yr, in ? at : kNowhere, 0, 0);
                }
            }
        }

        if (kStateOnly || !a.segmented || t0 + Q < sg.t1) {
            if (apart) {
#pragma unroll
                for (int j = 0; j < Q / 16; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) xf[j][i] = Xs[(16 * j + 4 * g + i) * XS + pw + lr];
            }
            const float end = dec[hb].end;
#pragma unroll
            for (int j = 0; j < NT; ++j) S[j] *= end;
#pragma unroll
            for (int q = 0; q < Q / 16; ++q) {
                const f32x4 w = *reinterpret_cast<const f32x4*>(dec[hb].w + 16 * q + 4 * g);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float xw = xf[q][i] * w[i];
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        S[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(Bs[(16 * q + 4 * g + i) * NS + 16 * j + lr], xw, S[j],
                                                                    0, 0, 0);
                }
            }
        }
        __syncthreads();
    }

    if (kStateOnly || !a.segmented) {
        const auto to = buffer_at(kStateOnly ? a.part + slot_state * N : a.S_out + run_state * N);
#pragma unroll
        for (int j = 0; j < NT; ++j)
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, S[j]), to, state_at(j), 0, 0);
        if (kStateOnly && wave < kHeads && lane == 0 && p0 == 0)
            a.decay[int64_t(slot) * H + h0 + wave] = exp2f(float(total));
    }
}

// Chains the segments' own sums into the state before each of them, in place,
// and the state after the run: four values of a run's state per thread, the
// next kAhead segments' sums in flight. Memory-bound: 16 segments of 64 heads of
// 64 x 128, read and written, 12.7 us (5.3 TB/s).
__global__ __launch_bounds__(kScanThreads) void scan_chain_kernel(ScanArgs a) {
    constexpr int kAhead = 8;
    const int64_t per = int64_t(a.H) * a.P * a.N / 4;
    const int64_t i = int64_t(blockIdx.x) * kScanThreads + threadIdx.x;
    const int r = blockIdx.y + blockIdx.z * kMaxGridY;
    if (i >= per || r >= a.runs) return;
    const int h = int(uint32_t(i) / uint32_t(a.P * a.N / 4));
    const int64_t b = run_start(a.cu, a.L, r), e = run_start(a.cu, a.L, r + 1);
    const int64_t first = (b >> a.shift) + r;
    const int n = int((e - b + (int64_t(1) << a.shift) - 1) >> a.shift);
    f32x4 S = {0.f, 0.f, 0.f, 0.f};
    if (a.S_in) S = reinterpret_cast<const f32x4*>(a.S_in)[r * per + i];
    f32x4* part = reinterpret_cast<f32x4*>(a.part) + first * per + i;
    const float* decay = a.decay + first * a.H + h;
    for (int k0 = 0; k0 < n; k0 += kAhead) {
        f32x4 own[kAhead];
        float d[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (k0 + k < n) {
                own[k] = part[(k0 + k) * per];
                d[k] = decay[int64_t(k0 + k) * a.H];
            }
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (k0 + k < n) {
                part[(k0 + k) * per] = S;
                S = S * d[k] + own[k];
            }
    }
    reinterpret_cast<f32x4*>(a.S_out)[r * per + i] = S;
}

template <int kNP, int kHeads, int kWaves>
void launch_scan(const ScanArgs& a, int act_dtype, bool bf16, bool state_only, dim3 grid, hipStream_t s) {
    // (kWaves of 16 head_dim rows, or in bfloat16 four of up to 32)
    const auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(bf16 ? kScanThreads : 64 * kWaves), 0, s, a); };
    if (bf16) {
        if (state_only) go(scan_bf16_kernel<kNP, kHeads, kWaves / 4, true>);
        else go(scan_bf16_kernel<kNP, kHeads, kWaves / 4, false>);
        return;
    }
    const auto f32 = [&](auto act) {
        using Act = decltype(act);
        if (state_only) go(scan_f32_kernel<Act, kNP, kHeads, kWaves, true>);
        else go(scan_f32_kernel<Act, kNP, kHeads, kWaves, false>);
    };
    if (act_dtype == GDN_F32) f32(ActF32{});
    else if (act_dtype == GDN_F16) f32(ActF16{});
    else f32(ActBF16{});
}

template <int kNP>
void launch_scan_shape(const ScanPlan& p, const ScanArgs& a, int act_dtype, bool bf16, bool state_only, dim3 grid,
                       hipStream_t s) {
    if (p.heads == 2 && p.waves == 8) launch_scan<kNP, 2, 8>(a, act_dtype, bf16, state_only, grid, s);
    else if (p.heads == 2) launch_scan<kNP, 2, 4>(a, act_dtype, bf16, state_only, grid, s);
    else if (p.waves == 8) launch_scan<kNP, 1, 8>(a, act_dtype, bf16, state_only, grid, s);
    else launch_scan<kNP, 1, 4>(a, act_dtype, bf16, state_only, grid, s);
}

bool scan_sizes_ok(int N, int64_t T, int G, int H, int P, int S) {
    return N >= 1 && T >= 0 && T < (int64_t(1) << 31) && G > 0 && H > 0 && H % G == 0 && P > 0 && S > 0;
}

bool on_bf16(int act_dtype, int y_dtype) { return act_dtype == GDN_BF16 && y_dtype == GDN_BF16; }

bool scan_shape_taken(int P, int S) { return P % 8 == 0 && S % 8 == 0 && S <= 256; }

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int64_t gdn_selective_scan_workspace_size(int act_dtype, int y_dtype, int N, int64_t T_total,
                                                     int64_t longest_run, int G, int H, int P, int S) {
    if (!scan_sizes_ok(N, T_total, G, H, P, S) || !scan_shape_taken(P, S) || !valid_dtype(act_dtype) ||
        !valid_dtype(y_dtype))
        return 0;
    return scan_plan(on_bf16(act_dtype, y_dtype), N, T_total, longest_run, G, H, P, S).bytes;
}

extern "C" int gdn_selective_scan(const void* x, int64_t x_stride, const void* B, int64_t B_stride, const void* C,
                                  int64_t C_stride, int act_dtype, const void* dt, int64_t dt_stride, int dt_dtype,
                                  const float* A_log, const float* dt_bias, const float* D, const float* state_in,
                                  float* state_out, void* y, int y_dtype, const int32_t* cu_seqlens, int N,
                                  int64_t T_total, int64_t longest_run, int G, int H, int P, int S, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
    GDN_REQUIRE(scan_sizes_ok(N, T_total, G, H, P, S), "gdn_selective_scan: bad sizes N=%d T=%lld G=%d H=%d P=%d S=%d",
                N, (long long)T_total, G, H, P, S);
    GDN_REQUIRE(valid_dtype(act_dtype) && valid_dtype(dt_dtype) && valid_dtype(y_dtype),
                "gdn_selective_scan: bad dtype");
    if (!scan_shape_taken(P, S))
        return fail(GDN_EUNSUPPORTED,
                    "gdn_selective_scan: head_dim and state_dim are multiples of 8, state_dim at most 256 (got %d, %d)",
                    P, S);
    GDN_REQUIRE(cu_seqlens || T_total % N == 0, "gdn_selective_scan: %lld tokens are not divisible into %d runs",
                (long long)T_total, N);
    GDN_REQUIRE(state_out && A_log && dt_bias && (T_total == 0 || (x && B && C && dt && y)),
                "gdn_selective_scan: null pointer");
    GDN_REQUIRE(x_stride >= int64_t(H) * P && B_stride >= int64_t(G) * S && C_stride >= int64_t(G) * S && dt_stride >= H,
                "gdn_selective_scan: a row stride is below its row");
    // (a chunk's rows are addressed in 31 bits)
    GDN_REQUIRE(x_stride <= (1 << 22) && B_stride <= (1 << 22) && C_stride <= (1 << 22) && int64_t(P) * S <= (1 << 28),
                "gdn_selective_scan: rows or states too wide");
    const int es = dtype_size(act_dtype);
    const auto at = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(B) | reinterpret_cast<uintptr_t>(C) |
                    reinterpret_cast<uintptr_t>(state_in) | reinterpret_cast<uintptr_t>(state_out) |
                    reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(workspace);
    GDN_REQUIRE(at % 16 == 0 && (x_stride | B_stride | C_stride) * es % 16 == 0,
                "gdn_selective_scan: x, B, C (rows too), y, states and workspace must be 16-byte aligned");
    const int64_t state_bytes = int64_t(N) * H * P * S * 4;
    GDN_REQUIRE(!state_in || state_in == state_out || !overlaps(state_in, state_bytes, state_out, state_bytes),
                "gdn_selective_scan: state_out partially overlaps state_in");
    const bool bf16 = on_bf16(act_dtype, y_dtype);
    const ScanPlan p = scan_plan(bf16, N, T_total, longest_run, G, H, P, S);
    GDN_REQUIRE(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes),
                "gdn_selective_scan: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                (long long)p.bytes);
    GDN_REQUIRE(p.slots <= INT32_MAX && p.units <= INT32_MAX && int64_t(H) * P * S / 4 <= INT32_MAX,
                "gdn_selective_scan: too many runs or heads");
    float* part = static_cast<float*>(workspace);
    ScanArgs a{x, B, C, dt, x_stride, B_stride, C_stride, dt_stride, dt_dtype, A_log, dt_bias, D, state_in,
               state_out, y, y_dtype, cu_seqlens, N, T_total / N, p.shift, G, H, P, S, part,
               part ? part + p.slots * H * int64_t(P) * S : nullptr, p.segmented, int(p.slots)};
    hipStream_t s = as_stream(stream);
    const auto tall = [](int64_t x, int64_t n) {
        return dim3(unsigned(x), unsigned(n < kMaxGridY ? n : kMaxGridY), unsigned((n + kMaxGridY - 1) / kMaxGridY));
    };
    const dim3 grid = tall(p.units, p.slots);
    const auto pass = [&](bool state_only) {
        if (S <= 32) launch_scan_shape<32>(p, a, act_dtype, bf16, state_only, grid, s);
        else if (S <= 64) launch_scan_shape<64>(p, a, act_dtype, bf16, state_only, grid, s);
        else if (S <= 128) launch_scan_shape<128>(p, a, act_dtype, bf16, state_only, grid, s);
        else launch_scan_shape<256>(p, a, act_dtype, bf16, state_only, grid, s);
    };
    if (p.segmented) {
        pass(true);
        const int64_t per = int64_t(H) * P * S / 4;
        hipLaunchKernelGGL(scan_chain_kernel, tall((per + kScanThreads - 1) / kScanThreads, N), dim3(kScanThreads), 0, s, a);
    }
    pass(false);
    return check_launch("gdn_selective_scan");
}
