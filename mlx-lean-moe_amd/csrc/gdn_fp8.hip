// y = x W^T for W in e4m3 codes with one float32 scale per 128 x 128 block, x
// quantized on the way in: each row's 128-column group b to e4m3 codes q under
// its own scale s = max(amax |x| / 448, 2^-126), q = e4m3(x / s) (both float32
// divisions, then one rounding to nearest even). Then
//   y[m, n] = sum_b s[m, b] sw[n / 128, b] sum_{k in b} q[m, k] w[n, k],
// the inner sums on the 8-bit matrix cores (one 16x16x128 product per block, so
// scales meet float32 sums only), the outer one in float32. float32 results take
// the codes widened to bfloat16 instead (at mfma_widened). Rows may come in such codes
// already, from the norm in front of the product (gdn_fp8_matmul_codes), which saves
// the launch that makes them: 2048 -> 12352, 64 rows 11.6 us and 8.1 by codes, 4096 118 and
// 110, the weights in the caches; 16 weights in turn, so from memory, 16 rows 12.0 and
// 10.3, 64 19.3 and 16.6, 200 23.5 and 20.8, 4096 137 and 127.
#include <type_traits>

#include "gdn_common.h"
#include "gdn_fp8.h"
#include "gdn_fp8_plan.h"
#include "gdn_host.h"
#include "gdn_ssm.h"

namespace gdn {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// Rows' codes (M x kb * 128, columns past K zero) and scales (kb x ldx): 16 lanes
// a group of 128, 8 values a lane. A workgroup takes one block of 16 rows, whose
// scales are one 64-byte line (the groups of one row, whose scales lie far apart:
// the same within 5 %). Measured, bf16: 200 rows of 4096 3.5 us, 4096 of 2048
// 10.9 (2.3 TB/s; the fastest of 23 calls 9.5, with four groups a lane 10.6).
template <class Act>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(const typename Act::storage* __restrict__ x, int M, int K,
                                                           int kb, uint8_t* __restrict__ codes,
                                                           float* __restrict__ scales, int ldx) {
    const unsigned id = blockIdx.y * gridDim.x + blockIdx.x;
    const int b = int(id % unsigned(kb));
    const int64_t row = int64_t(id / unsigned(kb)) * 16 + threadIdx.x / 16;
    const int m = int(min(row, int64_t(M - 1))), k = b * kB + (threadIdx.x & 15) * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (k < K) load8f<Act>(x + int64_t(m) * K + k, v);
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    const float s = scale_of(row16_max(top));
    divide_all(v, s);
    if (row >= M) return;
    *reinterpret_cast<uint2*>(codes + int64_t(m) * kb * kB + k) =
        make_uint2(codes4(v[0], v[1], v[2], v[3]), codes4(v[4], v[5], v[6], v[7]));
    if ((threadIdx.x & 15) == 0) scales[int64_t(b) * ldx + m] = s;
}

struct Fp8Args {
    const uint8_t *q, *w;
    const float *sx, *sw;
    const void* residual;
    void* y;
    int y_dtype, M, N, K, kb;
    int ldx;      // columns of sx, a multiple of 256
    int steps;    // blocks of K a workgroup takes
    float* part;  // split K: (splits, M, N4) float32, else null
    int N4;       // N rounded up to 4
    int ldy;      // columns of y's rows (N, or more where these N columns are a part)
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

// Whether rows of y start on multiples of `count` elements, and this launch's
// columns end on one: both, since rows lie ldy apart whatever part of their
// columns the launch takes.
GDN_DEV bool whole_pieces(const Fp8Args& a, int count) { return ((a.N | a.ldy) & (count - 1)) == 0; }

// Four results of row m, columns n .. n + 3: the product rounded to y's type,
// then the residual added and rounded again.
GDN_DEV void store4(const Fp8Args& a, int m, int n, f32x4 v) {
    if (m >= a.M) return;
    const int64_t at = int64_t(m) * a.ldy + n;
    if (whole_pieces(a, 4) && n + 3 < a.N) {
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

typedef __attribute__((address_space(3))) void lds_void;

// `rows` rows of `width` bytes as a buffer; what lies beyond reads as zero.
GDN_DEV __amdgpu_buffer_rsrc_t byte_rows(const uint8_t* base, int rows, int width) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, rows * width, 0x00027000);
}

// A tile of TN rows of W by TM rows of x, kWN x kWM waves, one 128-column block
// of both a step. The blocks go from memory to LDS without passing registers,
// into one of two buffers while the other is multiplied. A row's 128 bytes are
// eight 16-byte pieces, piece c of row r at place c ^ (r % 8): the DMA writes
// places in order, so a lane fetches the piece that belongs at its place, and
// the 16 rows of an operand read fall on all banks. Which columns a lane holds
// does not matter inside a block as long as both operands agree: pieces g and
// g + 4 of its row.
//
// W is the left operand, so a lane's column is one row of x: its scale is one
// value per 16 rows, times W's scale once a step, and each product of a block
// costs four multiply-adds to add.
//
// Bound by the matrix cores and those multiply-adds, which share the issue
// slots: 256 x 256 tiles of 4096 x 12288 x 2048 117 us (1.76 PFLOP/s; the vendor's
// product with one scale for each operand reached 2.7 at 8192^3). Small tiles are
// bound by the latency of a block's loads; rows and outputs too few for a tile a
// CU split K. float32 results, 4096 x 12352 x 2048: 252 us in all, 200 rows 27. A
// residual is read two bytes at a time: 4096 rows 4096 -> 2048 62 us with, 52
// without.
template <int TN, int TM, int kWN, int kWM, bool kExact>
__global__ __launch_bounds__(64 * kWN * kWM) void fp8_tile_kernel(Fp8Args a) {
    constexpr int kWaves = kWN * kWM, RN = TN / (16 * kWN), RM = TM / (16 * kWM);
    constexpr int kScales = (TN + TM) * kB, kBytes = kScales + 1024, kLoadsW = TN / 8 / kWaves, kLoadsQ = TM / 8 / kWaves;
    static_assert(TN % (8 * kWaves) == 0 && TM % (8 * kWaves) == 0 && (TN % kB == 0 || kB % TN == 0) && kB % (16 * RN) == 0, "tile");
    __shared__ __attribute__((aligned(1024))) uint8_t buf0[kBytes], buf1[kBytes];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, lr = lane & 15;
    const int wn = wave / kWM * (16 * RN), wm = wave % kWM * (16 * RM);

    // consecutive workgroups go to the 8 dies in turn: each die takes a
    // contiguous share of the tiles, in which neighbours share rows of W
    const int tiles_m = (a.M + TM - 1) / TM, tiles = tiles_m * ((a.N + TN - 1) / TN);
    const int share = tiles / 8, rest = tiles % 8, die = blockIdx.x % 8;
    const int tile = die * share + min(die, rest) + blockIdx.x / 8;
    const int n0 = tile / tiles_m * TN, m0 = tile % tiles_m * TM;
    const int b0 = blockIdx.y * a.steps, b1 = min(a.kb, b0 + a.steps);

    const int Kq = a.kb * kB;
    const auto wr = byte_rows(a.w + int64_t(n0) * a.K, min(TN, a.N - n0), a.K);
    const auto qr = byte_rows(a.q + int64_t(m0) * Kq, min(TM, a.M - m0), Kq);
    const auto xr = byte_rows(reinterpret_cast<const uint8_t*>(a.sx + m0), 1, a.kb * a.ldx * 4 - m0 * 4);
    // The lane's piece of a matrix's first 8 rows of this wave's share; 8 rows
    // on it is the same piece (r % 8 is the lane's). Rows past the last repeat it.
    const int r8 = lane >> 3, c16 = ((lane & 7) ^ r8) * 16;
    const int w_at = (wave * kLoadsW * 8 + r8) * a.K + c16, w_last = (min(TN, a.N - n0) - 1) * a.K + c16;
    const int q_at = (wave * kLoadsQ * 8 + r8) * Kq + c16, q_last = (min(TM, a.M - m0) - 1) * Kq + c16;
    const auto fetch = [&](uint8_t* buf, int b) {
        // W's last block may be short: pieces beyond it are placed past the
        // buffer's end, which reads as zero (q's rows are padded)
        const int past = b * kB + c16 >= a.K ? 0x7FFFFF00 : 0;
        int wa = w_at, qa = q_at;
        asm volatile("" : "+v"(wa), "+v"(qa));  // (places formed here, not kept in registers across steps)
#pragma unroll
        for (int i = 0; i < kLoadsW; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (lds_void*)(buf + (wave * kLoadsW + i) * 1024), 16,
                                                     max(min(wa + i * 8 * a.K, w_last), past), b * kB, 0, 0);
#pragma unroll
        for (int i = 0; i < kLoadsQ; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(qr, (lds_void*)(buf + TN * kB + (wave * kLoadsQ + i) * 1024), 16,
                                                     min(qa + i * 8 * Kq, q_last), b * kB, 0, 0);
        if (wave == 0)  // the rows' scales of this block
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_void*)(buf + kScales), 16, lane * 16, b * a.ldx * 4, 0, 0);
    };
    const float* sw = a.sw + int64_t(min(n0 + wn, a.N - 1) / kB) * a.kb;

    f32x4 acc[RN][RM];
#pragma unroll
    for (int i = 0; i < RN; ++i)
#pragma unroll
        for (int j = 0; j < RM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // the lane's two pieces of a row r with r % 16 = lr
    const int at0 = lr * kB + ((g ^ (lr & 7)) << 4), at1 = at0 ^ 64;
    const auto multiply = [&](const uint8_t* buf, float sn) {
        const uint8_t* wb = buf + wn * kB;
        const uint8_t* qb = buf + (TN + wm) * kB;
        uint4 q[RM][2], w[2][2];
        float s[RM];
        w[0][0] = *reinterpret_cast<const uint4*>(wb + at0);
        w[0][1] = *reinterpret_cast<const uint4*>(wb + at1);
#pragma unroll
        for (int j = 0; j < RM; ++j) {
            q[j][0] = *reinterpret_cast<const uint4*>(qb + 16 * j * kB + at0);
            q[j][1] = *reinterpret_cast<const uint4*>(qb + 16 * j * kB + at1);
            s[j] = sn * *reinterpret_cast<const float*>(buf + kScales + (wm + 16 * j + lr) * 4);
        }
#pragma unroll
        for (int i = 0; i < RN; ++i) {
            if (i + 1 < RN) {  // the next rows of W, while these are multiplied
                w[(i + 1) & 1][0] = *reinterpret_cast<const uint4*>(wb + 16 * (i + 1) * kB + at0);
                w[(i + 1) & 1][1] = *reinterpret_cast<const uint4*>(wb + 16 * (i + 1) * kB + at1);
            }
            f32x4 p[RM];
#pragma unroll
            for (int j = 0; j < RM; ++j)
                p[j] = kExact ? mfma_widened(w[i & 1][0], w[i & 1][1], q[j][0], q[j][1])
                              : mfma_fp8(w[i & 1][0], w[i & 1][1], q[j][0], q[j][1]);
#pragma unroll
            for (int j = 0; j < RM; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(s[j], p[j][e], acc[i][j][e]);
            // products and sums stay here and the later rows' reads below: no
            // more rows of W in registers than two
#pragma unroll
            for (int j = 0; j < RM; ++j) asm volatile("" : "+v"(acc[i][j])::"memory");
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const auto step = [&](uint8_t* cur, uint8_t* next, int b) {
        const float sn = sw[b];
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's pieces are in LDS
        __syncthreads();
        if (b + 1 < b1) fetch(next, b + 1);
        multiply(cur, sn);
    };
    fetch(buf0, b0);
    for (int b = b0; b < b1; b += 2) {
        step(buf0, buf1, b);
        if (b + 1 < b1) step(buf1, buf0, b + 1);
    }
    if (kExact || a.part) {
#pragma unroll
        for (int i = 0; i < RN; ++i)
#pragma unroll
            for (int j = 0; j < RM; ++j) {
                const int n = n0 + wn + 16 * i + 4 * g, m = m0 + wm + 16 * j + lr;
                if (!a.part)
                    store4(a, m, n, acc[i][j]);
                else if (m < a.M && n < a.N4)
                    *reinterpret_cast<f32x4*>(a.part + (int64_t(blockIdx.y) * a.M + m) * a.N4 + n) = acc[i][j];
            }
        return;
    }
    // 16-bit results: a wave's rows of x lie 16 apart in its lanes, four columns
    // each, and stored like that would write 32 bytes of a line at a time. They
    // are turned round through the wave's share of LDS (8 values a piece, piece
    // c of row m at place c ^ m) and leave as whole rows.
    constexpr int kPieces = 2 * RN, kShare = 512 * RN * RM;
    static_assert(kShare * kWaves / 2 <= kBytes || kWaves == 1, "a wave's results fit its share of LDS");
    __syncthreads();
    uint8_t* own = (wave < kWaves / 2 ? buf0 : buf1) + wave % (kWaves / 2) * kShare;
#pragma unroll
    for (int i = 0; i < RN; ++i)
#pragma unroll
        for (int j = 0; j < RM; ++j) {
            const int m = 16 * j + lr, c = (2 * i + (g >> 1)) ^ (m & (kPieces - 1));
            const f32x4 v = acc[i][j];
            const uint2 o = a.y_dtype == GDN_BF16
                                ? make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]))
                                : make_uint2(f32_to_f16_bits(v[0]) | uint32_t(f32_to_f16_bits(v[1])) << 16,
                                             f32_to_f16_bits(v[2]) | uint32_t(f32_to_f16_bits(v[3])) << 16);
            *reinterpret_cast<uint2*>(own + (m * kPieces + c) * 16 + (g & 1) * 8) = o;
        }
    const bool whole = whole_pieces(a, 8);
    // (a wave reads only what it wrote itself: no barrier)
    for (int p = lane; p < 16 * RM * kPieces; p += 64) {
        const int row = p / kPieces, c = p % kPieces;
        const int m = m0 + wm + row, n = n0 + wn + 8 * c;
        uint4 v = *reinterpret_cast<const uint4*>(own + (row * kPieces + (c ^ (row & (kPieces - 1)))) * 16);
        if (m >= a.M || n >= a.N) continue;
        const int64_t at = int64_t(m) * a.ldy + n;
        uint16_t* y = static_cast<uint16_t*>(a.y) + at;
        if (whole && !a.residual) {
            *reinterpret_cast<uint4*>(y) = v;
            continue;
        }
        uint16_t e[8];
        __builtin_memcpy(e, &v, 16);
        const int count = min(8, a.N - n);
        if (a.residual) {
            const uint16_t* r = static_cast<const uint16_t*>(a.residual) + at;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < count) {
                    const float sum = a.y_dtype == GDN_BF16 ? bf16_bits_to_f32(e[k]) + bf16_bits_to_f32(r[k])
                                                            : f16_bits_to_f32(e[k]) + f16_bits_to_f32(r[k]);
                    e[k] = a.y_dtype == GDN_BF16 ? f32_to_bf16_bits(sum) : f32_to_f16_bits(sum);
                }
        }
        if (whole) {
            __builtin_memcpy(&v, e, 16);
            *reinterpret_cast<uint4*>(y) = v;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < count) y[k] = e[k];
        }
    }
}

// Up to 16 rows of x, in one launch: each workgroup quantizes them itself (or copies
// their codes) into
// LDS (codes and scales, K whole), while its first blocks of W are on their
// way, then its 16 waves take kNs x 16 rows of W and every (16 / kNs)-th block
// of K each, straight from memory into the left operand, and add their sums in
// LDS. No wave waits for another until then. W is read once, and that is what
// bounds it; the launches that the tiles need (rows' codes, product, sum of the
// split) cost more than the product at these sizes. Every workgroup quantizes the
// same rows, so there is an end to it: kSkinnyGroups groups of 128 values.
// Measured, us, this against the launches of the tiles: 2048 -> 12352 1 row 7.8
// (3.3 TB/s), 12.7; 16 rows 11.7, 16.2; 4096 -> 2048 1 row 5.3, 11.1; 12 rows (384
// groups) 10.6, 11.7; 16 rows (512) 12.7, 11.9; 8192 -> 8192 4 rows (256) 18.3,
// 21.0; 8 rows (512) 23.8, 21.7.
constexpr int kSkinnyWaves = 16;
constexpr int kAhead = 4;  // blocks of W in flight a wave

// Rows that are in codes already (Fp8Args' q and sx) instead of an activation type.
struct InCodes {
    using storage = uint8_t;
    static constexpr int code = -1;
};

template <class Act, int kNs, bool kExact>
__global__ __launch_bounds__(64 * kSkinnyWaves) void fp8_skinny_kernel(Fp8Args a, const typename Act::storage* x) {
    constexpr int kGroups = kSkinnyWaves / kNs;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, lr = lane & 15;
    const int Kq = a.kb * kB, stride = Kq + 16;  // (rows 16 bytes apart in the banks)
    uint8_t* codes = lds;
    float* sx = reinterpret_cast<float*>(lds + a.M * stride);

    const int sub = wave % kNs, group = wave / kNs;
    const unsigned id = blockIdx.y * gridDim.x + blockIdx.x;
    if (int64_t(id) * (16 * kNs) >= a.N) return;  // (the last row of the grid may be short)
    const int n0 = (int(id) * kNs + sub) * 16;
    const uint8_t* wr = a.w + int64_t(min(n0 + lr, a.N - 1)) * a.K + 32 * g;
    const float* sw = a.sw + int64_t(min(n0, a.N - 1) / kB) * a.kb;
    uint4 w[kAhead][2];
    float sn[kAhead];
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const auto fetch = [&](int b, uint4 (&v)[2], float& s) {
        const int k = b * kB + 32 * g;
        v[0] = v[1] = zero;
        s = 0.f;
        if (b < a.kb) {
            s = sw[b];
            if (k < a.K) v[0] = *reinterpret_cast<const uint4*>(wr + b * kB);
            if (k + 16 < a.K) v[1] = *reinterpret_cast<const uint4*>(wr + b * kB + 16);
        }
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch(group + i * kGroups, w[i], sn[i]);

    for (int at = tid / 16; at < a.M * a.kb; at += 4 * kSkinnyWaves) {
        const int m = at / a.kb, b = at % a.kb, k = b * kB + (tid & 15) * 8;
        if constexpr (Act::code == InCodes::code) {
            *reinterpret_cast<uint2*>(codes + m * stride + k) = *reinterpret_cast<const uint2*>(a.q + m * Kq + k);
            if ((tid & 15) == 0) sx[m * a.kb + b] = a.sx[int64_t(b) * a.ldx + m];
        } else {
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (k < a.K) load8f<Act>(x + int64_t(m) * a.K + k, v);
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
            const float s = scale_of(row16_max(top));
            divide_all(v, s);
            *reinterpret_cast<uint2*>(codes + m * stride + k) =
                make_uint2(codes4(v[0], v[1], v[2], v[3]), codes4(v[4], v[5], v[6], v[7]));
            if ((tid & 15) == 0) sx[m * a.kb + b] = s;
        }
    }
    __syncthreads();

    const int m = min(lr, a.M - 1);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int b0 = group; b0 < a.kb; b0 += kAhead * kGroups)
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int b = b0 + i * kGroups;
            if (b >= a.kb) break;
            const uint8_t* q = codes + m * stride + b * kB + 32 * g;
            const uint4 q0 = *reinterpret_cast<const uint4*>(q), q1 = *reinterpret_cast<const uint4*>(q + 16);
            const f32x4 p = kExact ? mfma_widened(w[i][0], w[i][1], q0, q1) : mfma_fp8(w[i][0], w[i][1], q0, q1);
            const float s = sx[m * a.kb + b] * sn[i];
            fetch(b + kAhead * kGroups, w[i], sn[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = __builtin_fmaf(s, p[e], acc[e]);
        }
    __syncthreads();
    f32x4* sums = reinterpret_cast<f32x4*>(lds);  // over the codes
    sums[wave * 64 + lane] = acc;
    __syncthreads();
    if (group == 0) {
#pragma unroll
        for (int i = 1; i < kGroups; ++i) acc += sums[(i * kNs + sub) * 64 + lane];
        store4(a, lr, n0 + 4 * g, acc);
    }
}

// LDS of a skinny product: codes and scales, and at least the 16 waves' sums.
int64_t skinny_bytes(int M, int kb) {
    const int64_t need = int64_t(M) * (kb * kB + 16 + kb * 4);
    return need > kSkinnyWaves * 1024 ? need : kSkinnyWaves * 1024;
}

// Adds the shares of a split product in their order: four columns a thread.
__global__ __launch_bounds__(256) void fp8_sum_kernel(Fp8Args a, int splits) {
    const int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) * 4, per = int64_t(a.M) * a.N4;
    if (i >= per) return;
    f32x4 v = *reinterpret_cast<const f32x4*>(a.part + i);
    for (int s = 1; s < splits; ++s) v += *reinterpret_cast<const f32x4*>(a.part + s * per + i);
    store4(a, int(i / a.N4), int(i % a.N4), v);
}

// The dense weights: code times its block's scale, one rounding. 16 codes a
// thread, stored one by one, 32 bytes from lane to lane, which bounds it: 12352 x
// 2048 to bfloat16 64 us (1.2 TB/s), to float32 115.
__global__ __launch_bounds__(256) void fp8_dequantize_kernel(const uint8_t* __restrict__ w,
                                                             const float* __restrict__ sw, void* __restrict__ out,
                                                             int out_dtype, int N, int K, int kb) {
    const int64_t i = ((int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * 256 + threadIdx.x) * 16;
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

template <int TN, int TM, int kWN, int kWM, bool kExact>
void launch_tiles(const Fp8Args& a, int splits, hipStream_t s) {
    const dim3 grid(unsigned(((a.N + TN - 1) / TN) * ((a.M + TM - 1) / TM)), unsigned(splits));
    hipLaunchKernelGGL((fp8_tile_kernel<TN, TM, kWN, kWM, kExact>), grid, dim3(64 * kWN * kWM), 0, s, a);
}

void launch_product(const Fp8Plan& p, const Fp8Args& a, hipStream_t s) {
    if (a.y_dtype == GDN_F32) {
        if (p.kind == 0) launch_tiles<64, 32, 2, 2, true>(a, p.splits, s);
        else if (p.kind == 1) launch_tiles<64, 64, 2, 2, true>(a, p.splits, s);
        else launch_tiles<128, 128, 2, 2, true>(a, p.splits, s);
    } else {
        if (p.kind == 0) launch_tiles<64, 32, 2, 2, false>(a, p.splits, s);
        else if (p.kind == 1) launch_tiles<64, 64, 2, 2, false>(a, p.splits, s);
        else if (p.kind == 2) launch_tiles<128, 256, 2, 4, false>(a, p.splits, s);
        else launch_tiles<256, 256, 2, 4, false>(a, p.splits, s);
    }
    if (a.part)
        hipLaunchKernelGGL(fp8_sum_kernel, dim3(unsigned((int64_t(a.M) * a.N4 / 4 + 255) / 256)), dim3(256), 0, s, a,
                           p.splits);
}

// Few rows: one launch of whichever x the rows come as.
template <class Act>
void launch_skinny(const Fp8Args& a, const void* x, hipStream_t s) {
    const unsigned bytes = unsigned(skinny_bytes(a.M, a.kb));
    // 64 rows of W a workgroup, 32 or 16: as many as still give most CUs one
    // (1 row, us, 16, 32 and 64: 12352 outputs 9.8, 8.0, 7.8; 8192 5.2, 4.9, 5.1;
    // 2048 5.3, 7.0, 10.5)
    const auto go = [&](auto exact) {
        constexpr bool E = decltype(exact)::value;
        const auto launch = [&](auto kernel, int rows) {
            hipLaunchKernelGGL(kernel, rows_of_blocks((int64_t(a.N) + rows - 1) / rows), dim3(64 * kSkinnyWaves), bytes, s,
                               a, static_cast<const typename Act::storage*>(x));
        };
        if (a.N > 64 * 190) launch(fp8_skinny_kernel<Act, 4, E>, 64);
        else if (a.N > 32 * 190) launch(fp8_skinny_kernel<Act, 2, E>, 32);
        else launch(fp8_skinny_kernel<Act, 1, E>, 16);
    };
    if (a.y_dtype == GDN_F32) go(std::true_type{});
    else go(std::false_type{});
}

// The product of rows in codes: `a` as for all columns, cut as planned, the
// shares of a split K in `part`.
void launch_cut(const Fp8Cut& cut, const Fp8Args& a, float* part, hipStream_t s) {
    const int ys = dtype_size(a.y_dtype);
    const auto product = [&](const Fp8Plan& p, int n0, int cols) {
        Fp8Args b = a;
        b.w += int64_t(n0) * a.K;
        b.sw += int64_t(n0 / kB) * a.kb;
        if (a.residual) b.residual = static_cast<const char*>(a.residual) + int64_t(n0) * ys;
        b.y = static_cast<char*>(a.y) + int64_t(n0) * ys;
        b.N = cols;
        b.steps = p.steps;
        b.part = p.splits > 1 ? part : nullptr;
        b.N4 = (cols + 3) / 4 * 4;
        launch_product(p, b, s);
    };
    product(cut.first, 0, cut.n0);
    if (cut.n0 < a.N) product(cut.rest, cut.n0, a.N - cut.n0);
}

int64_t codes_bytes(int M, int K) { return (int64_t(M) * ((K + kB - 1) / kB) * kB + 255) / 256 * 256; }

// (K: a tile's rows are addressed in 31 bits)
bool fp8_sizes_ok(int M, int N, int K) {
    return M >= 0 && N > 0 && K > 0 && K % 16 == 0 && K <= (1 << 22) && N <= INT32_MAX - 256 && M <= INT32_MAX - 256;
}

}  // namespace
}  // namespace gdn

using namespace gdn;

extern "C" int64_t gdn_fp8_matmul_workspace_size(int y_dtype, int M, int N, int K) {
    if (!fp8_sizes_ok(M, N, K) || !valid_dtype(y_dtype)) return 0;
    const int kb = (K + kB - 1) / kB;
    if (skinny(M, kb)) return 0;
    return codes_bytes(M, K) + int64_t(scale_columns(M)) * kb * 4 + fp8_cut(y_dtype == GDN_F32, M, N, kb).part_bytes();
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
    const int kb = (K + kB - 1) / kB, ldx = scale_columns(M);
    hipStream_t s = as_stream(stream);
    if (skinny(M, kb)) {
        const Fp8Args a{nullptr, static_cast<const uint8_t*>(w), nullptr, scales, residual, y, y_dtype, M, N, K, kb, 0, kb,
                        nullptr, 0, N};
        if (x_dtype == GDN_F32) launch_skinny<ActF32>(a, x, s);
        else if (x_dtype == GDN_BF16) launch_skinny<ActBF16>(a, x, s);
        else launch_skinny<ActF16>(a, x, s);
        return check_launch("gdn_fp8_matmul");
    }
    const Fp8Cut cut = fp8_cut(y_dtype == GDN_F32, M, N, kb);
    const int64_t need = codes_bytes(M, K) + int64_t(ldx) * kb * 4 + cut.part_bytes();
    GDN_REQUIRE(workspace && workspace_bytes >= need, "gdn_fp8_matmul: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes, (long long)need);
    const int64_t blocks = (int64_t(M) + 15) / 16 * kb;
    GDN_REQUIRE(blocks <= INT32_MAX && int64_t(ldx) * kb <= INT32_MAX / 4, "gdn_fp8_matmul: too many rows");
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    float* sx = reinterpret_cast<float*>(codes + codes_bytes(M, K));
    const auto quantize = [&](auto act) {
        using Act = decltype(act);
        hipLaunchKernelGGL(fp8_quantize_kernel<Act>, rows_of_blocks(blocks), dim3(256), 0, s,
                           static_cast<const typename Act::storage*>(x), M, K, kb, codes, sx, ldx);
    };
    if (x_dtype == GDN_F32) quantize(ActF32{});
    else if (x_dtype == GDN_BF16) quantize(ActBF16{});
    else quantize(ActF16{});
    launch_cut(cut, {codes, static_cast<const uint8_t*>(w), sx, scales, residual, y, y_dtype, M, N, K, kb, ldx, 0, nullptr,
                     0, N}, sx + int64_t(ldx) * kb, s);
    return check_launch("gdn_fp8_matmul");
}

extern "C" int64_t gdn_fp8_matmul_codes_workspace_size(int y_dtype, int M, int N, int K) {
    if (!fp8_sizes_ok(M, N, K) || !valid_dtype(y_dtype)) return 0;
    const int kb = (K + kB - 1) / kB;
    return skinny(M, kb) ? 0 : fp8_cut(y_dtype == GDN_F32, M, N, kb).part_bytes();
}

extern "C" int gdn_fp8_matmul_codes(const void* codes, const float* row_scales, int scale_stride, const void* w,
                                    const float* scales, void* y, int y_dtype, const void* residual, int M, int N, int K,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
    GDN_REQUIRE(fp8_sizes_ok(M, N, K), "gdn_fp8_matmul_codes: bad sizes M=%d N=%d K=%d (K a multiple of 16)", M, N, K);
    GDN_REQUIRE(valid_dtype(y_dtype), "gdn_fp8_matmul_codes: bad dtype");
    if (M == 0) return 0;
    GDN_REQUIRE(codes && row_scales && w && scales && y, "gdn_fp8_matmul_codes: null pointer");
    GDN_REQUIRE((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(row_scales) |
                 reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(y) |
                 reinterpret_cast<uintptr_t>(workspace)) % 16 == 0,
                "gdn_fp8_matmul_codes: codes, their scales, w, y and workspace must be 16-byte aligned");
    GDN_REQUIRE(scale_stride >= M && scale_stride % 256 == 0,
                "gdn_fp8_matmul_codes: scales %d apart for %d rows (a multiple of 256)", scale_stride, M);
    const int kb = (K + kB - 1) / kB;
    hipStream_t s = as_stream(stream);
    const Fp8Args a{static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(w), row_scales, scales, residual, y,
                    y_dtype, M, N, K, kb, scale_stride, kb, nullptr, 0, N};
    if (skinny(M, kb)) {
        launch_skinny<InCodes>(a, codes, s);
        return check_launch("gdn_fp8_matmul_codes");
    }
    const Fp8Cut cut = fp8_cut(y_dtype == GDN_F32, M, N, kb);
    GDN_REQUIRE(cut.part_bytes() == 0 || (workspace && workspace_bytes >= cut.part_bytes()),
                "gdn_fp8_matmul_codes: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                (long long)cut.part_bytes());
    GDN_REQUIRE(int64_t(scale_stride) * kb <= INT32_MAX / 4, "gdn_fp8_matmul_codes: too many rows");
    launch_cut(cut, a, static_cast<float*>(workspace), s);
    return check_launch("gdn_fp8_matmul_codes");
}

extern "C" int gdn_fp8_dequantize(const void* w, const float* scales, void* out, int out_dtype, int N, int K,
                                  void* stream) {
    GDN_REQUIRE(fp8_sizes_ok(0, N, K), "gdn_fp8_dequantize: bad sizes N=%d K=%d (K a multiple of 16)", N, K);
    GDN_REQUIRE(valid_dtype(out_dtype), "gdn_fp8_dequantize: bad dtype");
    GDN_REQUIRE(w && scales && out, "gdn_fp8_dequantize: null pointer");
    GDN_REQUIRE(reinterpret_cast<uintptr_t>(w) % 16 == 0, "gdn_fp8_dequantize: w must be 16-byte aligned");
    const int64_t blocks = (int64_t(N) * K / 16 + 255) / 256;
    GDN_REQUIRE(blocks <= INT32_MAX, "gdn_fp8_dequantize: too many weights");
    hipLaunchKernelGGL(fp8_dequantize_kernel, rows_of_blocks(blocks), dim3(256), 0, as_stream(stream),
                       static_cast<const uint8_t*>(w), scales, out, out_dtype, N, K, (K + kB - 1) / kB);
    return check_launch("gdn_fp8_dequantize");
}
