// gfx950 kernels that write the 8-bit input of a projection, codes and scales:
//   - add_rms_norm_quant: the RMSNorm in front of it, with the residual's
//     addition:  h = round(x + residual),  y = h r w,  r = 1/sqrt(mean(h^2) + eps);
//   - silu_mul_quant: the gated activation of a feed-forward block, of rows
//     gate | up:  y = g / (1 + exp(-g)) * u.
// int8 codes have one scale per row (for int8_scaled_mm), e4m3fn codes one per
// 128 columns (for fp8_einsum):
//   a = max |y| under the scale,  s = a / q  (q = 127 or 448),  code = RNE(q y / a).
//
// The codes are those of this definition in 64 bits, every one.  In the norm r
// cancels, so a code is the rounded quotient q h w / max |h w| and needs no
// sum.  The fast path works on v = h w (exact in binary32 for 16-bit weights,
// rounded once for float32 ones) or v = y within a relative 2^-21: t = v * (q / a)
// in binary32 is off by less than 2^-20.2 relative (in units of 2^-24: 8 of v, 4 of
// q / a, 1 of the product), so a code can be wrong only
// where t lies that close to the border between two codes.  Those elements, one
// in some thousand, are computed again in binary64 (with a correctly rounded
// division) and their bytes overwritten.  The largest magnitude is settled the
// same way: of float32 weights by the products' rounding errors, which an FMA
// gives exactly, of the activation by computing every element within 2^-19 of
// the binary32 maximum again.  Where the binary32 values leave the range in which
// these bounds hold (a row of zeros, of values below 2^-60 or above 2^120,
// gates or up values above 2^20, NaN, infinities), all elements under the scale go that way.
//
// Bound by memory: 7 bytes per element with a residual (x, residual, hidden,
// code), 3 without, 5 for the activation.  A row is read once and held in
// registers; a thread holds P pieces of 8 elements, piece j at element
// 8 (t + LANES j), so a wave's loads are 1 KiB contiguous, and 16 consecutive
// threads hold the 128 columns of an e4m3fn scale.  Loads and stores assume no
// alignment beyond the element's own, so rows of any stride and width take the
// same code.
#include "fgv_device.h"
#include "fgv_host.h"

namespace fgv {
namespace {

enum Op { kNorm = 0, kSilu = 1 };
constexpr int kGroup = 128;       // columns under one e4m3fn scale
constexpr int kMaxCols = 65536;   // 1024 threads x 8 pieces x 8 elements

struct QuantArgs {
    const uint16_t* x;         // norm: x[rows, cols]; silu: gate | up [rows, 2 cols]
    int64_t x_stride;
    const uint16_t* residual;  // or null
    int64_t r_stride;
    const void* w;             // norm weights
    uint16_t* hidden;          // with a residual
    int64_t h_stride;
    uint8_t* codes;
    int64_t c_stride;
    float* scales;
    int64_t s_stride;
    int64_t rows;
    int32_t cols;
    double eps;
};

typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_a1 __attribute__((ext_vector_type(2), aligned(1)));

// ---- 16-bit elements ----

template <bool F16>
__device__ __forceinline__ float elem(uint16_t bits) {
    if constexpr (F16)
        return (float)__builtin_bit_cast(_Float16, bits);
    else
        return __uint_as_float((uint32_t)bits << 16);
}
template <bool F16>
__device__ __forceinline__ float lo_of(uint32_t w) {
    return F16 ? elem<true>((uint16_t)w) : bf16_lo(w);
}
template <bool F16>
__device__ __forceinline__ float hi_of(uint32_t w) {
    return F16 ? elem<true>((uint16_t)(w >> 16)) : bf16_hi(w);
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (F16) {
        const uint32_t l = __builtin_bit_cast(uint16_t, (_Float16)a), h = __builtin_bit_cast(uint16_t, (_Float16)b);
        return l | (h << 16);
    } else {
        return pack_bf16x2(a, b);
    }
}

// Eight elements from e0 on of a row that ends at cols (zeros behind it).
__device__ __forceinline__ u32x4_t load_piece(const uint16_t* row, int e0, int cols) {
    if (e0 + 8 <= cols)
        return __builtin_nontemporal_load(reinterpret_cast<const u32x4_a2*>(row + e0));
    u32x4_t v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (e0 + i < cols)
            v[i >> 1] |= (uint32_t)row[e0 + i] << (16 * (i & 1));
    return v;
}
__device__ __forceinline__ void store_piece(uint16_t* row, int e0, int cols, u32x4_t v) {
    if (e0 + 8 <= cols) {
        __builtin_nontemporal_store(v, reinterpret_cast<u32x4_a2*>(row + e0));
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (e0 + i < cols)
            row[e0 + i] = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
}
__device__ __forceinline__ void store_codes(uint8_t* row, int e0, int cols, uint32_t lo, uint32_t hi) {
    if (e0 + 8 <= cols) {
        const u32x2_t v = {lo, hi};
        *reinterpret_cast<u32x2_a1*>(row + e0) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (e0 + i < cols)
            row[e0 + i] = (uint8_t)((i < 4 ? lo : hi) >> (8 * (i & 3)));
}

// ---- the value that is quantised ----

// silu(g) u in binary32, within a relative 2^-21 (units of 2^-24: v_exp_f32 and
// v_rcp_f32 2 each, the exponent's fraction 1/3, 1 + e and two products 1 each).
// The exponent g log2(e) is split into an integer and a fraction known to 2^-25,
// so that v_exp_f32's argument keeps its low bits (one rounding of g log2(e)
// alone would cost 2^-17 at g = -88).  The exponent stops at g = +-86, where the
// sigmoid is 1 or below 2^-124: further out on the negative side the product is
// too large, by no more than |g u| 2^-124.  With both factors within kWide that is
// 2^-84, under 2^-15 of a code's unit where the largest magnitude is kLeast or more
// (448 * 2^-84 / 2^-60), so the code is 0 as it should be.
__device__ __forceinline__ float silu_mul32(float g, float u) {
    constexpr float kLog2e = 0x1.715476p0f, kLog2eLo = 0x1.4ae0cp-26f;  // log2(e) = their sum to 2^-49
    constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: the sum's low bits are the rounded value's
    const float x = __builtin_amdgcn_fmed3f(-g, -86.f, 86.f);
    const float s = fmaf(x, kLog2e, kMagic), n = s - kMagic;
    const float f = fmaf(x, kLog2eLo, fmaf(x, kLog2e, -n));
    const float e = __uint_as_float(__float_as_uint(__builtin_amdgcn_exp2f(f)) + (__float_as_uint(s) << 23));
    return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}

__device__ __forceinline__ double silu_mul64(double g, double u) { return g / (1.0 + exp(-g)) * u; }

// Element e of the row in binary64.  h is read back from hidden where there
// is a residual (this thread wrote it).
template <int OP, bool F16, bool WF32>
__device__ __forceinline__ double value64(const QuantArgs& a, int64_t row, int e) {
    if constexpr (OP == kSilu) {
        const uint16_t* x = a.x + row * a.x_stride;
        return silu_mul64(elem<F16>(x[e]), elem<F16>(x[a.cols + e]));
    } else {
        const double h = elem<F16>(a.residual ? a.hidden[row * a.h_stride + e] : a.x[row * a.x_stride + e]);
        const double w = WF32 ? reinterpret_cast<const float*>(a.w)[e]
                              : elem<F16>(reinterpret_cast<const uint16_t*>(a.w)[e]);
        return h * w;
    }
}

// Element i of a piece, where reading it again would cost another memory latency.
template <bool F16>
__device__ __forceinline__ float elem_of(u32x4_t p, int i) {
    const uint32_t w = i & 4 ? (i & 2 ? p[3] : p[2]) : (i & 2 ? p[1] : p[0]);
    return i & 1 ? hi_of<F16>(w) : lo_of<F16>(w);
}

// The int8 code of v under the largest magnitude `most` (0 for a row of zeros
// or one that is not finite).
__device__ __forceinline__ uint8_t code64_i8(double v, double most) {
    if (!(most > 0.0 && most < HUGE_VAL))
        return 0;
    return (uint8_t)(int8_t)(int)rint(v * 127.0 / most);
}
// The e4m3fn code: the quotient is rounded to binary32 towards zero with the
// lost part kept in the last bit (to odd), so that the second rounding, to
// e4m3fn, is the only one that counts.
__device__ __forceinline__ uint8_t code64_fp8(double v, double most) {
    if (!(most > 0.0 && most < HUGE_VAL))
        return 0;
    const double q = v * 448.0 / most;
    const float f = (float)q;
    const double left = q - (double)f;
    uint32_t bits = __float_as_uint(f);
    if (left != 0.0) {
        if ((left > 0.0) != (q > 0.0))
            --bits;  // |f| > |q|
        bits |= 1u;
    }
    return (uint8_t)(pack_fp8x4(__uint_as_float(bits), 0.f, 0.f, 0.f) & 0xffu);
}

// ---- reductions over the LANES threads of a row ----

__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
template <int CTRL>
__device__ __forceinline__ uint64_t dpp_u64(uint64_t v) {
    return (uint64_t)dpp_u32<CTRL>((uint32_t)v) | ((uint64_t)dpp_u32<CTRL>((uint32_t)(v >> 32)) << 32);
}
__device__ __forceinline__ uint64_t row16_max64(uint64_t v) {
    v = max64(v, dpp_u64<kDppQuadXor1>(v));
    v = max64(v, dpp_u64<kDppQuadXor2>(v));
    v = max64(v, dpp_u64<kDppHalfMirror>(v));
    v = max64(v, dpp_u64<kDppMirror>(v));
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
    v = row16_sum(v);
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = row16_max(v);
    v = max(v, (uint32_t)__shfl_xor((int)v, 16));
    return max(v, (uint32_t)__shfl_xor((int)v, 32));
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
    v = row16_max64(v);
    v = max64(v, (uint64_t)__shfl_xor((unsigned long long)v, 16));
    return max64(v, (uint64_t)__shfl_xor((unsigned long long)v, 32));
}

// The larger of m, |a| and |b|; NaN if any is.
__device__ __forceinline__ float max3_abs(float m, float a, float b) {
    return __builtin_elementwise_maximum(m, __builtin_elementwise_maximum(fabsf(a), fabsf(b)));
}

// binary32 magnitudes between these (as bits) keep the fast path's bounds
constexpr uint32_t kLeast = (127 - 60) << 23, kMost = (127 + 120) << 23;
constexpr float kNearMost = 1.0f - 0x1p-19f;  // nearer to the maximum than this: settled in binary64
// Gates and up values above this go the 64-bit way: an up value could bring a product
// back from below binary32's range, a gate outweigh the least sigmoid.
constexpr float kWide = 0x1p20f;
// Distance from the nearest code at which an element counts as beside a border.
// int8: 0.5 - 2^-13 of a step (127 * 2^-20.2 < 2^-13); e4m3fn: half a step times
// 1 - 2^-14 (the step is at least 2^-4 of the value: 16 * 2^-20.2 < 2^-15).
constexpr float kBorderI8 = 0.5f - 0x1p-13f, kBorderFp8 = 0x1p-4f * (1.0f - 0x1p-14f);

// Eight weights from e0 on (zeros behind cols).
template <bool F16, bool WF32>
__device__ __forceinline__ void load_weights(const void* weights, int e0, int cols, float w[8]) {
    if constexpr (WF32) {
        const float* wp = reinterpret_cast<const float*>(weights) + e0;
        if (e0 + 8 <= cols) {
            const f32x4_a4 lo = *reinterpret_cast<const f32x4_a4*>(wp);
            const f32x4_a4 hi = *reinterpret_cast<const f32x4_a4*>(wp + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = lo[i];
                w[4 + i] = hi[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                w[i] = e0 + i < cols ? wp[i] : 0.f;
        }
    } else {
        const uint16_t* wp = reinterpret_cast<const uint16_t*>(weights);
        u32x4_t v = {0, 0, 0, 0};
        if (e0 + 8 <= cols)
            v = *reinterpret_cast<const u32x4_a2*>(wp + e0);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (e0 + i < cols)
                    v[i >> 1] |= (uint32_t)wp[e0 + i] << (16 * (i & 1));
#pragma unroll
        for (int i = 0; i < 8; ++i)
            w[i] = i & 1 ? hi_of<F16>(v[i >> 1]) : lo_of<F16>(v[i >> 1]);
    }
}

// One row per LANES threads (64: four rows to a workgroup; else one).  The
// e4m3fn activation, whose groups of 128 columns need nothing of each other,
// gives a wave 512 columns of a row and a second grid dimension the rest of it.
// It is bound by the vector instructions (some 370 for a wave's 512 elements,
// among them one evaluation in 64 bits that settles the groups' maxima), so the
// elements for that come out of registers, not out of memory again: 8192 rows of
// 16384 columns 159 us (256 threads to 2048 columns, a division for the row and
// loads again 168), 65536 rows of 512 44 (60), 256 rows of 2048 4.0 (4.5), but
// 2048 rows of 8192 25.0 (24.1).  Sixteen elements per thread, half the 64-bit
// evaluations, took 170.
template <int OP, bool F16, bool WF32, bool FP8, int LANES, int P>
__global__ void __launch_bounds__(LANES == 64 ? 256 : LANES) act_quant_kernel(QuantArgs a) {
    constexpr int kBlock = LANES == 64 ? 256 : LANES, kWaves = LANES / 64;
    constexpr bool kRowScale = !FP8;              // one scale per row, else per 16 threads and piece
    constexpr bool kAlone = OP == kSilu && FP8;  // a wave by itself
    // The piece stays in registers for its 64-bit evaluations (int8, 4096 rows of 2048 columns: 13.6 us, read again
    // 14.3; but with four rows to a workgroup, 65536 of 512, the selection costs more than the wait: 43.7 and 41.1).
    constexpr bool kKeep = OP == kSilu && P == 1 && (FP8 || LANES > 64);
    constexpr bool kExact32 = OP == kNorm && !WF32;  // v is exact
    constexpr bool kWithLost = OP == kNorm && WF32;  // v's rounding error is kept
    __shared__ double sum_of[kWaves];
    __shared__ uint32_t max_of[kWaves];
    __shared__ unsigned long long best_of;

    int64_t row = (int64_t)blockIdx.x * (kBlock / LANES) + threadIdx.x / LANES;
    int t = threadIdx.x % LANES;
    if constexpr (kAlone) {
        static_assert(LANES == 64 && P == 1);
        row = (int64_t)blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
        t += (int)blockIdx.x * 64;
    }
    if (row >= a.rows)
        return;  // (only where waves are rows: no barrier below)
    const int cols = a.cols;
    const uint16_t* xrow = a.x + row * a.x_stride;
    uint8_t* crow = a.codes + row * a.c_stride;

    // ---- one pass over the row: v, the sum of squares, the largest magnitude ----
    float v[P][8], lost[kWithLost ? P : 1][8];
    double ss = 0.0;
    float most32[P];
    u32x4_t kept0 = {}, kept1 = {};
    {
        u32x4_t p0[P], p1[P];
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int e0 = 8 * (t + LANES * j);
            p0[j] = load_piece(xrow, e0, cols);
            if constexpr (OP == kSilu)
                p1[j] = load_piece(xrow + cols, e0, cols);
            else if (a.residual)
                p1[j] = load_piece(a.residual + row * a.r_stride, e0, cols);
        }
        if constexpr (kKeep) {
            kept0 = p0[0];
            kept1 = p1[0];
        }
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int e0 = 8 * (t + LANES * j);
            float most = 0.f;
            if constexpr (OP == kSilu) {
                float widest = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float g0 = lo_of<F16>(p0[j][i >> 1]), g1 = hi_of<F16>(p0[j][i >> 1]);
                    const float u0 = lo_of<F16>(p1[j][i >> 1]), u1 = hi_of<F16>(p1[j][i >> 1]);
                    v[j][i] = silu_mul32(g0, u0);
                    v[j][i + 1] = silu_mul32(g1, u1);
                    most = max3_abs(most, v[j][i], v[j][i + 1]);
                    if constexpr (!F16) {  // (fp16 ends at 65504, and its infinities reach the product)
                        widest = max3_abs(widest, u0, u1);
                        widest = max3_abs(widest, g0, g1);
                    }
                }
                if (!F16 && !(widest <= kWide))
                    most = __builtin_nanf("");
            } else {
                float w[8];
                load_weights<F16, WF32>(a.w, e0, cols, w);
                if (a.residual) {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        p0[j][q] = pack2<F16>(lo_of<F16>(p0[j][q]) + lo_of<F16>(p1[j][q]),
                                              hi_of<F16>(p0[j][q]) + hi_of<F16>(p1[j][q]));
                    store_piece(a.hidden + row * a.h_stride, e0, cols, p0[j]);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float h = i & 1 ? hi_of<F16>(p0[j][i >> 1]) : lo_of<F16>(p0[j][i >> 1]);
                    ss = fma((double)h, (double)h, ss);  // (the square is exact)
                    v[j][i] = h * w[i];
                    if constexpr (kWithLost)
                        lost[j][i] = fmaf(h, w[i], -v[j][i]);
                    if (i & 1)
                        most = max3_abs(most, v[j][i - 1], v[j][i]);
                }
            }
            most32[j] = most;
        }
    }

    // ---- the row's sum, and its largest magnitude where it has one scale ----
    uint32_t mx = 0;  // (bits: a NaN is above all)
    if constexpr (OP == kNorm || kRowScale) {
#pragma unroll
        for (int j = 0; j < P; ++j)
            mx = max(mx, __float_as_uint(most32[j]) & 0x7fffffffu);
        if constexpr (OP == kNorm)
            ss = wave_sum(ss);
        if constexpr (kRowScale)
            mx = wave_max(mx);
        if constexpr (kWaves > 1) {
            if ((threadIdx.x & 63) == 0) {
                sum_of[threadIdx.x >> 6] = ss;
                max_of[threadIdx.x >> 6] = mx;
            }
            if (threadIdx.x == 0)
                best_of = 0;
            __syncthreads();
            ss = sum_of[0];
            mx = max_of[0];
#pragma unroll
            for (int i = 1; i < kWaves; ++i) {
                ss += sum_of[i];
                mx = max(mx, max_of[i]);
            }
        }
    }
    auto value_at = [&](int j, int i) __attribute__((always_inline)) {  // element i of piece j in 64 bits
        if constexpr (kKeep)
            return silu_mul64(elem_of<F16>(kept0, i), elem_of<F16>(kept1, i));
        else
            return value64<OP, F16, WF32>(a, row, 8 * (t + LANES * j) + i);
    };
    // the factor of the scales: the norm's r (NaN for a row that holds a NaN or an infinity) over q
    auto factor = [&](double q) __attribute__((always_inline)) {
        if constexpr (OP == kNorm)
            return ss < HUGE_VAL ? rsqrt(ss / cols + a.eps) * (1.0 / q) : __builtin_nan("");
        else
            return 1.0 / q;
    };

    if constexpr (kRowScale) {
        // ---- int8: one scale per row ----
        const bool odd = !(mx >= kLeast && mx <= kMost);  // (the same in all threads of the row)
        const float top = __uint_as_float(mx);
        double most = top;
        if (!kExact32 || odd) {
            uint64_t best = 0;
            if (kWithLost && !odd) {
                // |h w| = top + what its rounding lost, of the elements that reach top
                float more = -top;
#pragma unroll
                for (int j = 0; j < P; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (fabsf(v[j][i]) == top)
                            more = fmaxf(more, copysignf(1.f, v[j][i]) * lost[j][i]);
                best = __builtin_bit_cast(uint64_t, (double)top + (double)more);  // (not negative)
            } else {
                const float from = odd ? -1.f : top * kNearMost;
                uint64_t mask = 0;
#pragma unroll
                for (int j = 0; j < P; ++j)
                    if (odd || most32[j] >= from) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (8 * (t + LANES * j) + i < cols && (odd || fabsf(v[j][i]) >= from))
                                mask |= 1ull << (8 * j + i);
                    }
                while (mask) {
                    const int at = __builtin_ctzll(mask);
                    mask &= mask - 1;
                    const double y = fabs(value_at(at >> 3, at & 7));
                    best = max64(best, __builtin_bit_cast(uint64_t, y));  // (a NaN is above all)
                }
            }
            best = wave_max64(best);
            if constexpr (kWaves > 1) {
                if ((threadIdx.x & 63) == 0 && best)
                    atomicMax(&best_of, (unsigned long long)best);
                __syncthreads();
                best = best_of;
            }
            most = __builtin_bit_cast(double, best);
        }
        const float inv = 127.f * __builtin_amdgcn_rcpf((float)most);
        uint64_t near = 0;
#pragma unroll
        for (int j = 0; j < P; ++j) {
            constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: the sum's low byte is the rounded value's
            const int e0 = 8 * (t + LANES * j);
            uint32_t m[8];
            float off[8], worst = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float s = fmaf(v[j][i], inv, kMagic);
                m[i] = __float_as_uint(s);
                off[i] = fmaf(v[j][i], inv, -(s - kMagic));
                if (i & 1)
                    worst = max3_abs(worst, off[i - 1], off[i]);
            }
            const uint32_t lo = __builtin_amdgcn_perm(__builtin_amdgcn_perm(m[3], m[2], 0x0c0c0400u),
                                                      __builtin_amdgcn_perm(m[1], m[0], 0x0c0c0400u), 0x05040100u);
            const uint32_t hi = __builtin_amdgcn_perm(__builtin_amdgcn_perm(m[7], m[6], 0x0c0c0400u),
                                                      __builtin_amdgcn_perm(m[5], m[4], 0x0c0c0400u), 0x05040100u);
            store_codes(crow, e0, cols, lo, hi);
            if (odd || worst > kBorderI8) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (e0 + i < cols && (odd || fabsf(off[i]) > kBorderI8))
                        near |= 1ull << (8 * j + i);
            }
        }
        while (near) {
            const int at = __builtin_ctzll(near);
            near &= near - 1;
            const int e = 8 * (t + LANES * (at >> 3)) + (at & 7);
            crow[e] = code64_i8(value_at(at >> 3, at & 7), most);
        }
        if (t == 0)
            a.scales[row * a.s_stride] = most < HUGE_VAL ? (float)(most * factor(127.0)) : __builtin_nanf("");
    } else {
        // ---- e4m3fn: one scale per 16 threads and piece (cols a multiple of 128: a group is whole or absent) ----
        const double each = factor(448.0);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int e0 = 8 * (t + LANES * j);
            if (e0 >= cols)
                continue;
            const uint32_t m = row16_max(__float_as_uint(most32[j]) & 0x7fffffffu);
            const bool odd = !(m >= kLeast && m <= kMost);  // (the same in the 16 threads)
            const float top = __uint_as_float(m);
            double most = top;
            if (!kExact32 || odd) {
                uint64_t best = 0;
                if (kWithLost && !odd) {
                    float more = -top;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (fabsf(v[j][i]) == top)
                            more = fmaxf(more, copysignf(1.f, v[j][i]) * lost[kWithLost ? j : 0][i]);
                    best = __builtin_bit_cast(uint64_t, (double)top + (double)more);
                } else {
                    const float from = odd ? -1.f : top * kNearMost;
                    uint32_t mask = 0;
                    if (odd || most32[j] >= from) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            mask |= odd || fabsf(v[j][i]) >= from ? 1u << i : 0u;
                    }
                    while (mask) {
                        const int at = __builtin_ctz(mask);
                        mask &= mask - 1;
                        best = max64(best, __builtin_bit_cast(uint64_t, fabs(value_at(j, at))));
                    }
                }
                most = __builtin_bit_cast(double, row16_max64(best));
            }
            const float inv = 448.f * __builtin_amdgcn_rcpf((float)most);
            float q[8], over[8], worst = -1.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                q[i] = v[j][i] * inv;
            const uint32_t lo = pack_fp8x4(q[0], q[1], q[2], q[3]), hi = pack_fp8x4(q[4], q[5], q[6], q[7]);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const auto r = i & 2 ? __builtin_amdgcn_cvt_pk_f32_fp8(i < 4 ? lo : hi, true)
                                     : __builtin_amdgcn_cvt_pk_f32_fp8(i < 4 ? lo : hi, false);
#pragma unroll
                for (int k = i; k < i + 2; ++k) {
                    // half a step of e4m3fn at this magnitude: 2^-4 of its power of two, 2^-10 below 2^-6
                    const float binade = fmaxf(__uint_as_float(__float_as_uint(q[k]) & 0x7f800000u), 0x1p-6f);
                    over[k] = fmaf(binade, -kBorderFp8, fabsf(q[k] - r[k - i]));
                }
                worst = __builtin_elementwise_maximum(worst, __builtin_elementwise_maximum(over[i], over[i + 1]));
            }
            store_codes(crow, e0, cols, lo, hi);
            if (odd || worst > 0.f) {
                uint32_t near = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    near |= odd || over[i] > 0.f ? 1u << i : 0u;
                while (near) {
                    const int at = __builtin_ctz(near);
                    near &= near - 1;
                    crow[e0 + at] = code64_fp8(value_at(j, at), most);
                }
            }
            if ((t & 15) == 0)
                a.scales[row * a.s_stride + e0 / kGroup] = most < HUGE_VAL ? (float)(most * each) : __builtin_nanf("");
        }
    }
}

// A launch has fewer than 2^32 threads and 2^16 workgroups in its second dimension: more rows go in several.
constexpr int64_t kLaunchThreads = 1LL << 31;
QuantArgs rows_from(QuantArgs a, int64_t first, int64_t rows) {
    a.x += first * a.x_stride;
    if (a.residual) {
        a.residual += first * a.r_stride;
        a.hidden += first * a.h_stride;
    }
    a.codes += first * a.c_stride;
    a.scales += first * a.s_stride;
    a.rows = rows;
    return a;
}

template <int OP, bool F16, bool WF32, bool FP8, int LANES, int P>
void launch(const QuantArgs& a, hipStream_t st) {
    constexpr int kRows = LANES == 64 ? 4 : 1;
    constexpr bool kAlone = OP == kSilu && FP8;
    const int64_t most = kAlone ? 65535 * kRows : kLaunchThreads / LANES;
    for (int64_t r = 0; r < a.rows; r += most) {
        const QuantArgs s = rows_from(a, r, a.rows - r < most ? a.rows - r : most);
        const unsigned groups = (unsigned)((s.rows + kRows - 1) / kRows);
        hipLaunchKernelGGL((act_quant_kernel<OP, F16, WF32, FP8, LANES, P>),
                           kAlone ? dim3((unsigned)(a.cols + 511) / 512, groups) : dim3(groups), dim3(kRows * LANES),
                           0, st, s);
    }
}

template <int OP, bool F16, bool WF32, bool FP8>
int launch_cols(const QuantArgs& a, hipStream_t st) {
    const int pieces = (a.cols + 7) / 8;
    if constexpr (OP == kSilu && FP8) {
        launch<kSilu, F16, WF32, true, 64, 1>(a, st);
        return launch_status();
    } else {
        // As few idle lanes as may be, and 256 threads to a workgroup while there
        // are rows enough: 8192 rows of 4096, 7168, 16384 columns: 256 x 2 46.1
        // us (512 x 1 50.6), 256 x 4 75.0 (512 x 2 77.4, 1024 x 1 85.8), of the
        // activation 256 x 8 121 (512 x 4 149); with two rows to a CU or less the
        // shortest way through a row counts: one row of 7168 1024 x 1 3.7 (256 x 4
        // 5.7), 512 rows 9.1 (10.3), but 1024 rows 15.3 (15.2); up to eight rows
        // to a CU of 4096 512 x 1: 2047 rows 14.9 (256 x 2 16.0).
        const bool few = a.rows <= 2 * cu_count();
        if (pieces <= 64)
            launch<OP, F16, WF32, FP8, 64, 1>(a, st);
        else if (pieces <= 128)
            launch<OP, F16, WF32, FP8, 128, 1>(a, st);
        else if (pieces <= 256)
            launch<OP, F16, WF32, FP8, 256, 1>(a, st);
        else if (pieces <= 512 && a.rows <= 8 * cu_count())
            launch<OP, F16, WF32, FP8, 512, 1>(a, st);
        else if (pieces <= 512)
            launch<OP, F16, WF32, FP8, 256, 2>(a, st);
        else if (pieces <= 1024 && few)
            launch<OP, F16, WF32, FP8, 1024, 1>(a, st);
        else if (pieces <= 768)
            launch<OP, F16, WF32, FP8, 256, 3>(a, st);
        else if (pieces <= 1024)
            launch<OP, F16, WF32, FP8, 256, 4>(a, st);
        else if (pieces <= 2048 && few)
            launch<OP, F16, WF32, FP8, 1024, 2>(a, st);
        else if (pieces <= 1536)
            launch<OP, F16, WF32, FP8, 512, 3>(a, st);
        else if (pieces <= 2048)
            launch<OP, F16, WF32, FP8, OP == kSilu ? 256 : 512, OP == kSilu ? 8 : 4>(a, st);
        else if (pieces <= 4096)
            launch<OP, F16, WF32, FP8, 1024, 4>(a, st);
        else
            launch<OP, F16, WF32, FP8, 1024, 8>(a, st);
        return launch_status();
    }
}

// (before cols goes into 32 bits)
int check_size(int64_t rows, int64_t cols) {
    if (rows < 0 || cols <= 0)
        return fail(FGV_E_BAD_SHAPE, "rows must not be negative and cols positive");
    if (rows > 0x7fffffffLL || cols > kMaxCols)
        return fail(FGV_E_TOO_LARGE, "at most 2^31 - 1 rows of 65536 columns");
    return FGV_OK;
}

int check_types(const QuantArgs& a, int x_dtype, int code_dtype) {
    if ((x_dtype != 0 && x_dtype != 1) || (code_dtype != 0 && code_dtype != 1))
        return fail(FGV_E_BAD_SHAPE, "x_dtype must be 0 (bf16) or 1 (fp16), code_dtype 0 (int8) or 1 (e4m3fn)");
    if (code_dtype == 1 && a.cols % kGroup)
        return fail(FGV_E_BAD_SHAPE, "e4m3fn codes need cols to be a multiple of 128");
    return FGV_OK;
}

}  // namespace
}  // namespace fgv

extern "C" int fgv_add_rms_norm_quant(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                                      const void* weight, int32_t weight_is_fp32, void* hidden, int64_t hidden_stride,
                                      void* codes, int64_t codes_stride, float* scales, int64_t scales_stride,
                                      int64_t rows, int64_t cols, double eps, int32_t x_dtype, int32_t code_dtype,
                                      void* stream) {
    using namespace fgv;
    if (const int rc = check_size(rows, cols))
        return rc;
    const QuantArgs a{static_cast<const uint16_t*>(x), x_stride, static_cast<const uint16_t*>(residual), residual_stride,
                      weight, static_cast<uint16_t*>(hidden), hidden_stride, static_cast<uint8_t*>(codes), codes_stride,
                      scales, scales_stride, rows, (int32_t)cols, eps};
    if (const int rc = check_types(a, x_dtype, code_dtype))
        return rc;
    if (!(eps > 0.0 && eps < HUGE_VAL))
        return fail(FGV_E_BAD_SHAPE, "eps must be positive and finite");
    if (rows == 0)
        return FGV_OK;
    if (!x || !weight || !codes || !scales || (residual && !hidden))
        return fail(FGV_E_NULL_POINTER, "null tensor");
    if (!aligned(x, 2) || !aligned(residual, 2) || !aligned(hidden, 2) || !aligned(weight, weight_is_fp32 ? 4 : 2) ||
        !aligned(scales, 4))
        return fail(FGV_E_MISALIGNED, "tensors must be aligned to their element size");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (x_dtype == 0) {
        if (code_dtype == 0)
            return weight_is_fp32 ? launch_cols<kNorm, false, true, false>(a, st)
                                  : launch_cols<kNorm, false, false, false>(a, st);
        return weight_is_fp32 ? launch_cols<kNorm, false, true, true>(a, st)
                              : launch_cols<kNorm, false, false, true>(a, st);
    }
    if (code_dtype == 0)
        return weight_is_fp32 ? launch_cols<kNorm, true, true, false>(a, st)
                              : launch_cols<kNorm, true, false, false>(a, st);
    return weight_is_fp32 ? launch_cols<kNorm, true, true, true>(a, st) : launch_cols<kNorm, true, false, true>(a, st);
}

extern "C" int fgv_silu_mul_quant(const void* x, int64_t x_stride, void* codes, int64_t codes_stride, float* scales,
                                  int64_t scales_stride, int64_t rows, int64_t cols, int32_t x_dtype,
                                  int32_t code_dtype, void* stream) {
    using namespace fgv;
    if (const int rc = check_size(rows, cols))
        return rc;
    const QuantArgs a{static_cast<const uint16_t*>(x), x_stride, nullptr, 0, nullptr, nullptr, 0,
                      static_cast<uint8_t*>(codes), codes_stride, scales, scales_stride, rows, (int32_t)cols, 0.0};
    if (const int rc = check_types(a, x_dtype, code_dtype))
        return rc;
    if (rows == 0)
        return FGV_OK;
    if (!x || !codes || !scales)
        return fail(FGV_E_NULL_POINTER, "null tensor");
    if (!aligned(x, 2) || !aligned(scales, 4))
        return fail(FGV_E_MISALIGNED, "tensors must be aligned to their element size");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (x_dtype == 0)
        return code_dtype == 0 ? launch_cols<kSilu, false, false, false>(a, st)
                               : launch_cols<kSilu, false, false, true>(a, st);
    return code_dtype == 0 ? launch_cols<kSilu, true, false, false>(a, st)
                           : launch_cols<kSilu, true, false, true>(a, st);
}
