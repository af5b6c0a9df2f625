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

// ---- many rows: tiles through LDS ----
// Output tiles of 32 TM tokens x 32 TN channels, four waves of 16 TM x 16 TN
// each.  The 128-byte K blocks of a's and b's rows stream through a ring of NS
// LDS stages by LDS DMA; rows are stored unpadded, 16-byte chunk q of row r at
// q ^ ((r >> 1) & 7), so that the 16 rows of a fragment read hit all 64 banks.
// A block is two slices of 64 bytes (one MFMA each); a slice's operands are read
// into registers under the MFMAs of the slice before it, in a second register
// set, so the matrix unit only waits at the barrier that hands a block over:
// once per block, between its two slices, when every wave holds the second
// slice in registers, the block's stage is free for block kb + NS and block
// kb + 1 has landed.
__device__ __forceinline__ int swz(int row, int chunk) { return chunk ^ ((row >> 1) & 7); }

// s_waitcnt operand: vector memory operations outstanding <= n (expcnt and
// lgkmcnt not waited for; gfx9 encoding vmcnt bits 3:0 and 15:14).
constexpr int wait_vm(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8); }

// Workgroup barrier over LDS work only (__syncthreads would wait for every DMA).
__device__ __forceinline__ void lds_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));  // lgkmcnt(0): this wave's LDS accesses done
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// LDS DMA of 16 bytes per lane from row + off (row a scalar result, not a
// v_readlane's) to lds + 16 lane, by all lanes (`lanes` ~0) or none (0: what a
// step past the last block sends).  Counted by vmcnt.
__device__ __forceinline__ void dma16_if(const void* row, uint32_t off, uint32_t lds, uint32_t lanes) {
    asm volatile("s_mov_b32 m0, %2\n\ts_mov_b32 exec_lo, %3\n\ts_mov_b32 exec_hi, %3\n\tglobal_load_lds_dwordx4 %1, %0\n\ts_mov_b64 exec, -1" ::"s"(row),
                 "v"(off), "s"(lds), "s"(lanes)
                 : "memory", "m0");
}

// The tile kernels' MFMA as inline assembly, its accumulator tied in place: left
// to itself the compiler gives the result other registers and copies the
// 256 accumulators around (150 copies to 128 MFMAs).  It knows of no
// wait states inside assembly: operands come from LDS or memory (whose waits it
// does insert); where the VALU may have written them `kAfterValu` waits, and
// mfma_done() stands before the accumulators are read.
template <bool kAfterValu = false>
__device__ __forceinline__ void mfma_in_place(v4i_t& acc, v4i_t a, v4i_t b) {
    if constexpr (kAfterValu)
        asm volatile("s_nop 4\n\tv_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
    else
        asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mfma_done() { asm volatile("s_nop 15\n\ts_nop 7" ::: "memory"); }

constexpr int kXcds = 8;

// Tile of workgroup `at`: workgroups go to the XCDs in turn, and each XCD, with
// an L2 of its own, takes a run of tiles in which kGroupM tiles along m share
// their b rows and neighbouring n share the a rows.
constexpr int kGroupM = 4;
__device__ __forceinline__ void tile_of(int at, int mtiles, int ntiles, int& mt, int& nt) {
    const int total = mtiles * ntiles, xcd = at % kXcds, each = total / kXcds, more = total % kXcds;
    const int t = xcd * each + min(xcd, more) + at / kXcds;
    const int per_group = kGroupM * ntiles, group = t / per_group, first = group * kGroupM;
    const int height = min(kGroupM, mtiles - first), in = t - group * per_group;
    mt = first + in % height;
    nt = in / height;
}

template <int TM, int TN, int NS, int OUT>
__global__ void __launch_bounds__(256, 1) int8_mm_tile_kernel(MmArgs p, int32_t mtiles, int32_t ntiles) {
    constexpr int kBM = 32 * TM, kBN = 32 * TN, kABytes = kBM * kBlockK;
    constexpr int kStage = (kBM + kBN) * kBlockK, kPer = TM + TN;  // DMAs per wave and block
    __shared__ __attribute__((aligned(1024))) uint8_t st[NS][kStage];

    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int c = lane & 15, g = lane >> 4, wm = wave >> 1, wn = wave & 1;
    int mt, nt;
    tile_of(blockIdx.x, mtiles, ntiles, mt, nt);
    const int m0 = mt * kBM, n0 = nt * kBN;

    // This lane's DMA sources, relative to the tile's first row: instruction j of
    // the wave covers tile rows 8 (wave T + j) + lane / 8, physical chunk lane % 8.
    // Rows past the end read the last one: they only feed outputs that are not stored.
    const int8_t* const abase = p.a + (int64_t)m0 * p.a_s;
    const int8_t* const bbase = p.b + (int64_t)n0 * p.b_s;
    uint32_t src[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const bool is_a = j < TM;
        const int row = 8 * (is_a ? wave * TM + j : wave * TN + j - TM) + (lane >> 3);
        const int r = is_a ? min(row, p.m - 1 - m0) : min(row, p.n - 1 - n0);
        src[j] = (uint32_t)r * (uint32_t)(is_a ? p.a_s : p.b_s) + 16 * swz(row, lane & 7);
    }
    const int nkb = p.k / kBlockK;  // whole blocks; what is left of K comes last, straight from memory
    auto issue = [&](int kb, uint32_t base, int j, uint32_t lanes) __attribute__((always_inline)) {
        const int8_t* row = (j < TM ? abase : bbase) + (int64_t)kb * kBlockK;
        const uint32_t to = base + (j < TM ? 1024 * (wave * TM + j) : kABytes + 1024 * (wave * TN + j - TM));
        dma16_if(row, src[j], to, lanes);
    };

    auto sending = [&](int kb) __attribute__((always_inline)) {
        return (uint32_t)__builtin_amdgcn_readfirstlane((kb - nkb) >> 31);  // ~0 below nkb
    };

    v4i_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
            acc[i][j] = v4i_t{0, 0, 0, 0};

    v4i_t A[2][TM], B[2][TN];
    const uint32_t lane_off = c * kBlockK + 16 * swz(c, g);
    const uint32_t aoff = wm * 16 * TM * kBlockK + lane_off, boff = kABytes + wn * 16 * TN * kBlockK + lane_off;
    // fragment u of slice s: a's, then b's (slice 1 is chunk ^ 4)
    auto read = [&](const uint8_t* stage, int s, int u) __attribute__((always_inline)) {
        if (u < TM)
            A[s][u] = *reinterpret_cast<const v4i_t*>(stage + (aoff ^ (64 * s)) + 16 * u * kBlockK);
        else
            B[s][u - TM] = *reinterpret_cast<const v4i_t*>(stage + (boff ^ (64 * s)) + 16 * (u - TM) * kBlockK);
    };

#pragma unroll
    for (int b = 0; b < NS; ++b)
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            issue(b, lds_addr(st[b]), j, sending(b));
    if (NS <= nkb)
        __builtin_amdgcn_s_waitcnt(wait_vm((NS - 1) * kPer));
    else
        __builtin_amdgcn_s_waitcnt(wait_vm(0));
    lds_barrier();
    constexpr int kMfmas = TM * TN;
    static_assert(kMfmas >= 3 * kPer - 1, "every read finds its MFMA");
    if (nkb > 0) {
#pragma unroll
        for (int u = 0; u < kPer; ++u)
            read(st[0], 0, u);
    }
    int at = 0;
    for (int kb = 0; kb < nkb; ++kb) {
        const uint8_t* cur = st[at];
        at = at + 1 < NS ? at + 1 : 0;
        const uint8_t* nxt = st[at];
        const uint32_t dst = lds_addr(cur);
#pragma unroll
        for (int u = 0; u < kMfmas; ++u) {
            const int i = u / TN, j = u % TN;
            mfma_in_place(acc[i][j], B[0][j], A[0][i]);
            if (u % 2 == 0 && u / 2 < kPer)
                read(cur, 1, u / 2);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (NS > 2 && kb + NS - 1 < nkb)
            __builtin_amdgcn_s_waitcnt(wait_vm((NS - 2) * kPer));
        else
            __builtin_amdgcn_s_waitcnt(wait_vm(0));
        lds_barrier();
        const uint32_t lanes = sending(kb + NS);
#pragma unroll
        for (int u = 0; u < kMfmas; ++u) {
            const int i = u / TN, j = u % TN;
            mfma_in_place(acc[i][j], B[1][j], A[1][i]);
            if (u < kPer)
                issue(kb + NS, dst, u, lanes);
            // (behind the last block this reads a stage that nothing uses)
            if (u >= kPer && u - kPer < 2 * kPer && (u - kPer) % 2 == 0)
                read(nxt, 0, (u - kPer) / 2);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (nkb * kBlockK < p.k) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int k0 = nkb * kBlockK + 64 * s + 16 * g;
            v4i_t b[TN];
#pragma unroll
            for (int j = 0; j < TN; ++j)
                b[j] = load_frag_end(p.b + (int64_t)min(n0 + wn * 16 * TN + 16 * j + c, p.n - 1) * p.b_s, k0, p.k);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const v4i_t a =
                    load_frag_end(p.a + (int64_t)min(m0 + wm * 16 * TM + 16 * i + c, p.m - 1) * p.a_s, k0, p.k);
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    mfma_in_place<true>(acc[i][j], b[j], a);
            }
        }
    }
    mfma_done();

    // ---- scales, bias, store ----
    const int nb = n0 + wn * 16 * TN + 4 * g;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int m = m0 + wm * 16 * TM + 16 * i + c;
        if (m >= p.m)
            continue;
        const float sa = p.sa[m * p.sa_s];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int n = nb + 16 * j;
            float v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int nq = min(n + q, p.n - 1);
                v[q] = (float)acc[i][j][q] * sa * p.sb[nq * p.sb_s] + bias_at(p, nq);
            }
            if (n < p.n)
                store4<OUT>(p, m, n, v);
        }
    }
}

template <int TM, int TN, int NS, int OUT>
void launch_tiles(const MmArgs& p, hipStream_t st) {
    const int32_t mtiles = (p.m + 32 * TM - 1) / (32 * TM), ntiles = (p.n + 32 * TN - 1) / (32 * TN);
    hipLaunchKernelGGL((int8_mm_tile_kernel<TM, TN, NS, OUT>), dim3((unsigned)(mtiles * ntiles)), dim3(256), 0, st, p,
                       mtiles, ntiles);
}

template <int MT, int NW, int KS, int OUT>
void launch_rows(const MmArgs& p, hipStream_t st) {
    const dim3 grid((unsigned)((p.n + 16 * NW - 1) / (16 * NW)), (unsigned)((p.m + 16 * MT - 1) / (16 * MT)));
    hipLaunchKernelGGL((int8_mm_rows_kernel<MT, NW, KS, OUT>), grid, dim3(64 * KS), 0, st, p);
}

template <int OUT>
int launch_mm(const MmArgs& p, hipStream_t st) {
    const bool al = aligned(p.a, 16) && aligned(p.b, 16) && p.a_s % 16 == 0 && p.b_s % 16 == 0 &&
                    p.a_s < (1 << 23) && p.b_s < (1 << 23);
    if (p.m <= 16)
        launch_rows<1, 2, 8, OUT>(p, st);
    else if (al && p.k > 0 && p.m > 64)
        launch_tiles<8, 8, 2, OUT>(p, st);
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
