// gfx950 product of int8 codes with a scale per token and per channel:
//   out[m, n] = scale_a[m] * scale_b[n] * sum_k a[m, k] b[n, k]  (+ bias[n]),
// a [M, K] and b [N, K] int8 with contiguous rows, out bf16, fp16 or fp32.
// The sum is an exact int32 (K <= 131071: at most 2^14 per product), so the
// result does not depend on how K is cut; the scales are applied in binary32,
// (sum * scale_a) * scale_b + bias, and the output rounded once.
//
// v_mfma_i32_16x16x64_i8 register images: lane (c, g) = (l % 16, l / 16) holds
// operand row c, bytes 16 g .. 16 g + 15 of the 64; the accumulator holds rows
// 4 g .. 4 g + 3 of the first operand against row c of the second.  b is the
// first operand, so a lane holds four neighbouring channels of one token.
#include "fgv_device.h"
#include "fgv_host.h"

namespace fgv {
namespace {

typedef int v4i_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef v4i_t v4i_a1 __attribute__((aligned(1)));

enum OutType { kOutBf16 = 0, kOutF16 = 1, kOutF32 = 2 };
constexpr int kBlockK = 128;
constexpr int64_t kMaxK = 131071;  // K * 2^14 fits int32

struct MmArgs {
    const int8_t* a;  // a[m, k], rows a_s bytes apart
    int64_t a_s;
    const int8_t* b;  // b[n, k]
    int64_t b_s;
    const float* sa;  // scale_a[m * sa_s] (0: one scale)
    int64_t sa_s;
    const float* sb;
    int64_t sb_s;
    const void* bias;  // bias[n] in bias_type, or null
    int32_t bias_type;
    void* out;  // out[m, n], rows o_s elements apart
    int64_t o_s;
    int32_t m, n, k;
};

__device__ __forceinline__ v4i_t mfma_i8(v4i_t a, v4i_t b, v4i_t c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float bias_at(const MmArgs& p, int n) {
    if (!p.bias)
        return 0.f;
    if (p.bias_type == kOutF32)
        return reinterpret_cast<const float*>(p.bias)[n];
    const uint16_t v = reinterpret_cast<const uint16_t*>(p.bias)[n];
    return p.bias_type == kOutF16 ? (float)__builtin_bit_cast(_Float16, v) : __uint_as_float((uint32_t)v << 16);
}

// Four channels n .. n + 3 of one token (those below p.n).
template <int OUT>
__device__ __forceinline__ void store4(const MmArgs& p, int64_t m, int n, const float v[4]) {
    if constexpr (OUT == kOutF32) {
        float* o = reinterpret_cast<float*>(p.out) + m * p.o_s + n;
        if (n + 4 <= p.n) {
            const f32x4_a4 w = {v[0], v[1], v[2], v[3]};
            *reinterpret_cast<f32x4_a4*>(o) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < p.n)
                    o[i] = v[i];
        }
    } else {
        uint16_t* o = reinterpret_cast<uint16_t*>(p.out) + m * p.o_s + n;
        u32x2_a2 w;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (OUT == kOutBf16)
                w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
            else
                w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i]) |
                       ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i + 1]) << 16);
        }
        if (n + 4 <= p.n) {
            *reinterpret_cast<u32x2_a2*>(o) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < p.n)
                    o[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        }
    }
}

// ---- few rows: fragments straight from memory ----
// Tokens m0 .. m0 + 16 MT, channels n0 .. n0 + 16 NW of a workgroup; its KS
// waves take the 128-byte K blocks in turn and add their sums up in LDS.

__device__ __forceinline__ v4i_t load_frag(const int8_t* row, int k) {
    return *reinterpret_cast<const v4i_a1*>(row + k);
}
// ... of the last, short block: bytes from K on as 0
__device__ __forceinline__ v4i_t load_frag_end(const int8_t* row, int k, int end) {
    if (k + 16 <= end)
        return load_frag(row, k);
    v4i_t v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (k + i < end)
            v[i >> 2] |= (int)((uint32_t)(uint8_t)row[k + i] << (8 * (i & 3)));
    return v;
}

template <int MT, int NW, int KS, int OUT>
__global__ void __launch_bounds__(64 * KS) int8_mm_rows_kernel(MmArgs p) {
    __shared__ v4i_t part[KS - 1][MT * NW][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int c = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16 * NW, m0 = blockIdx.y * 16 * MT;
    // rows past the end read the last one: they only feed outputs that are not stored
    const int8_t* arow[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
        arow[i] = p.a + (int64_t)min(m0 + 16 * i + c, p.m - 1) * p.a_s;
    const int8_t* brow[NW];
#pragma unroll
    for (int j = 0; j < NW; ++j)
        brow[j] = p.b + (int64_t)min(n0 + 16 * j + c, p.n - 1) * p.b_s;

    v4i_t acc[MT][NW];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NW; ++j)
            acc[i][j] = v4i_t{0, 0, 0, 0};
    const int nkb = p.k / kBlockK;
    for (int kb = w; kb < nkb; kb += KS) {
        const int k0 = kb * kBlockK + 16 * g;
        v4i_t A[MT][2], B[NW][2];
#pragma unroll
        for (int j = 0; j < NW; ++j) {
            B[j][0] = load_frag(brow[j], k0);
            B[j][1] = load_frag(brow[j], k0 + 64);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            A[i][0] = load_frag(arow[i], k0);
            A[i][1] = load_frag(arow[i], k0 + 64);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NW; ++j)
                    acc[i][j] = mfma_i8(B[j][h], A[i][h], acc[i][j]);
    }
    if (nkb * kBlockK < p.k && w == nkb % KS) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k0 = nkb * kBlockK + 64 * h + 16 * g;
            v4i_t A[MT], B[NW];
#pragma unroll
            for (int j = 0; j < NW; ++j)
                B[j] = load_frag_end(brow[j], k0, p.k);
#pragma unroll
            for (int i = 0; i < MT; ++i)
                A[i] = load_frag_end(arow[i], k0, p.k);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NW; ++j)
                    acc[i][j] = mfma_i8(B[j], A[i], acc[i][j]);
        }
    }

    if (w > 0) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NW; ++j)
                part[w - 1][i * NW + j][lane] = acc[i][j];
    }
    __syncthreads();
    if (w != 0)
        return;
#pragma unroll
    for (int v = 0; v < KS - 1; ++v)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NW; ++j)
                acc[i][j] += part[v][i * NW + j][lane];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int m = m0 + 16 * i + c;
        if (m >= p.m)
            continue;
        const float sa = p.sa[m * p.sa_s];
#pragma unroll
        for (int j = 0; j < NW; ++j) {
            const int n = n0 + 16 * j + 4 * g;
            float v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int nq = min(n + q, p.n - 1);
                v[q] = (float)acc[i][j][q] * sa * p.sb[nq * p.sb_s] + bias_at(p, nq);
            }
            store4<OUT>(p, m, n, v);
        }
    }
}

template <int MT, int NW, int KS, int OUT>
void launch_rows(const MmArgs& p, hipStream_t st) {
    const dim3 grid((unsigned)((p.n + 16 * NW - 1) / (16 * NW)), (unsigned)((p.m + 16 * MT - 1) / (16 * MT)));
    hipLaunchKernelGGL((int8_mm_rows_kernel<MT, NW, KS, OUT>), grid, dim3(64 * KS), 0, st, p);
}

template <int OUT>
int launch_mm(const MmArgs& p, hipStream_t st) {
    if (p.m <= 16)
        launch_rows<1, 2, 8, OUT>(p, st);
    else
        launch_rows<2, 2, 8, OUT>(p, st);
    return launch_status();
}

}  // namespace
}  // namespace fgv

extern "C" int fgv_int8_scaled_mm(const int8_t* a, int64_t a_stride, const int8_t* b, int64_t b_stride,
                                  const float* scale_a, int64_t scale_a_stride, const float* scale_b,
                                  int64_t scale_b_stride, const void* bias, int32_t bias_dtype, void* out,
                                  int64_t out_stride, int64_t m, int64_t n, int64_t k, int32_t out_dtype,
                                  void* stream) {
    using namespace fgv;
    if (m < 0 || n < 0 || k < 0)
        return fail(FGV_E_BAD_SHAPE, "negative size");
    if (out_dtype < kOutBf16 || out_dtype > kOutF32 || (bias && (bias_dtype < kOutBf16 || bias_dtype > kOutF32)))
        return fail(FGV_E_BAD_SHAPE, "out_dtype and bias_dtype must be 0 (bf16), 1 (fp16) or 2 (fp32)");
    if (k > kMaxK)
        return fail(FGV_E_TOO_LARGE, "k above 131071: the int32 sum could overflow");
    if (m > 0x7fffff00LL || n > 0x7fffff00LL || m > (1LL << 20))
        return fail(FGV_E_TOO_LARGE, "m at most 2^20, n below 2^31");
    if (m == 0 || n == 0)
        return FGV_OK;
    if (!out || !scale_a || !scale_b || (k > 0 && (!a || !b)))
        return fail(FGV_E_NULL_POINTER, "null tensor");
    if (!aligned(out, out_dtype == kOutF32 ? 4 : 2) || !aligned(scale_a, 4) || !aligned(scale_b, 4) ||
        (bias && !aligned(bias, bias_dtype == kOutF32 ? 4 : 2)))
        return fail(FGV_E_MISALIGNED, "out, scales and bias must be aligned to their element size");
    const MmArgs p{a,    a_stride,   b,   b_stride,   scale_a,    scale_a_stride, scale_b, scale_b_stride,
                   bias, bias_dtype, out, out_stride, (int32_t)m, (int32_t)n,     (int32_t)k};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    switch (out_dtype) {
    case kOutBf16:
        return launch_mm<kOutBf16>(p, st);
    case kOutF16:
        return launch_mm<kOutF16>(p, st);
    default:
        return launch_mm<kOutF32>(p, st);
    }
}
