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
#include <algorithm>
#include <type_traits>

#include "fgv_device.h"
#include "fgv_host.h"

namespace fgv {
namespace {

typedef int v4i_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef v4i_t v4i_a1 __attribute__((aligned(1)));
typedef v4i_t v4i_a4 __attribute__((aligned(4)));

enum OutType { kOutBf16 = 0, kOutF16 = 1, kOutF32 = 2 };
constexpr int kBlockK = 128;
constexpr int64_t kMaxK = 131071;  // K * 2^14 fits int32
constexpr int64_t kMaxM = 1 << 20, kMaxN = 1 << 24;

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

// The bias of four channels from n on (the last one's past the end); without one -0, which leaves every sum as it
// is, also the sign of a zero.  One choice of type for all four, so that their loads are under way together.
__device__ __forceinline__ void bias4(const MmArgs& p, int n, float v[4]) {
    if (!p.bias) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            v[q] = -0.f;
    } else if (p.bias_type == kOutF32) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            v[q] = reinterpret_cast<const float*>(p.bias)[min(n + q, p.n - 1)];
    } else {
        uint16_t raw[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            raw[q] = reinterpret_cast<const uint16_t*>(p.bias)[min(n + q, p.n - 1)];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            v[q] = p.bias_type == kOutF16 ? (float)__builtin_bit_cast(_Float16, raw[q])
                                          : __uint_as_float((uint32_t)raw[q] << 16);
    }
}

// Two outputs in one word.
template <int OUT>
__device__ __forceinline__ uint32_t pack_out(float lo, float hi) {
    if constexpr (OUT == kOutBf16)
        return pack_bf16x2(lo, hi);
    // (kept apart from the product before it: the compiler would round both at
    // once in one kernel and not in another, and results would depend on the schedule)
    asm("" : "+v"(lo), "+v"(hi));
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) |
           ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16);
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
        for (int i = 0; i < 2; ++i)
            w[i] = pack_out<OUT>(v[2 * i], v[2 * i + 1]);
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

// ---- few rows, or few tiles: fragments straight from memory ----
// Tokens m0 .. m0 + 16 MT, channels n0 .. n0 + 16 NW of a workgroup; its KS
// waves take the 128-byte K blocks in turn and add their sums up in LDS.

__device__ __forceinline__ v4i_t load_frag(const int8_t* row, int k) {
    return *reinterpret_cast<const v4i_a1*>(row + k);
}
// 32 bytes from row + k of a row that starts at any byte, out of whole words
// (loads across words keep the address path busy: 8 x 4096 x 4111 15.7 us, so
// 8.4): `words` is the row rounded down to a word, `past` the bytes that dropped.
// No word is read that holds none of the 32 bytes.
__device__ __forceinline__ void load_frags_by_words(const int8_t* words, uint32_t past, int k, v4i_t& lo, v4i_t& hi) {
    const v4i_t w0 = *reinterpret_cast<const v4i_a4*>(words + k), w1 = *reinterpret_cast<const v4i_a4*>(words + k + 16);
    const int w2 = *reinterpret_cast<const int*>(words + k + (past ? 32 : 28));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lo[i] = (int)__builtin_amdgcn_alignbyte((uint32_t)(i < 3 ? w0[i + 1] : w1[0]), (uint32_t)w0[i], past);
        hi[i] = (int)__builtin_amdgcn_alignbyte((uint32_t)(i < 3 ? w1[i + 1] : w2), (uint32_t)w1[i], past);
    }
}
// ... of the last, short block: bytes from `end` on as 0.  The chunk that the row
// ends in is cut out of the row's last 16 bytes (a row of fewer byte by byte).
__device__ __forceinline__ v4i_t load_frag_end(const int8_t* row, int k, int end) {
    if (k + 16 <= end)
        return load_frag(row, k);
    v4i_t v = {0, 0, 0, 0};
    if (k >= end)
        return v;
    if (end >= 16) {
        const v4i_t w = load_frag(row, end - 16);
        const int past = 8 * (k + 16 - end);  // bits to drop, 8 .. 120
        uint64_t lo = (uint32_t)w[0] | ((uint64_t)(uint32_t)w[1] << 32), hi = (uint32_t)w[2] | ((uint64_t)(uint32_t)w[3] << 32);
        lo = past < 64 ? (lo >> past) | (hi << (64 - past)) : hi >> (past - 64);
        hi = past < 64 ? hi >> past : 0;
        return v4i_t{(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
    }
#pragma unroll
    for (int i = 0; i < 15; ++i)
        if (k + i < end)
            v[i >> 2] |= (int)((uint32_t)(uint8_t)row[k + i] << (8 * (i & 3)));
    return v;
}

template <int MT, int NW, int KS, int OUT, bool SHIFT>
__global__ void __launch_bounds__(64 * KS) int8_mm_rows_kernel(MmArgs p) {
    __shared__ v4i_t part[KS - 1][MT * NW][64];
    // K blocks whose loads go together: two where a wave has two column tiles (16 x 7168 x 7168 14.5 us, one 15.4);
    // with one, more in flight slows the stream of b down (1 x 7168 x 7168 11.0 us, two 11.5, four 11.8)
    constexpr int kBatch = MT * NW == 1 ? 1 : 2;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
    // scales and bias, for wave 0 at the end: on their way before the K blocks, so that nothing waits for them
    float sa[MT], sb[NW][4], bias[NW][4];
    if (w == 0) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
            sa[i] = p.sa[min(m0 + 16 * i + c, p.m - 1) * p.sa_s];
#pragma unroll
        for (int j = 0; j < NW; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                sb[j][q] = p.sb[min(n0 + 16 * j + 4 * g + q, p.n - 1) * p.sb_s];
#pragma unroll
        for (int j = 0; j < NW; ++j)
            bias4(p, n0 + 16 * j + 4 * g, bias[j]);
    }

    const int nkb = p.k / kBlockK;
    int kb = w;
    auto blocks = [&](auto count) __attribute__((always_inline)) {
        constexpr int kCount = decltype(count)::value;
        v4i_t A[kCount][MT][2], B[kCount][NW][2];
#pragma unroll
        for (int u = 0; u < kCount; ++u) {
            const int k0 = (kb + KS * u) * kBlockK;
            // (which 16 bytes of the block a lane group takes does not matter, as long as a's and b's agree)
            auto load = [&](const int8_t* row, v4i_t to[2]) __attribute__((always_inline)) {
                if constexpr (SHIFT) {
                    const uint32_t past = (uint32_t)reinterpret_cast<uintptr_t>(row) & 3;
                    load_frags_by_words(row - past, past, k0 + 32 * g, to[0], to[1]);
                } else {
                    to[0] = load_frag(row, k0 + 16 * g);
                    to[1] = load_frag(row, k0 + 16 * g + 64);
                }
            };
#pragma unroll
            for (int j = 0; j < NW; ++j)
                load(brow[j], B[u][j]);
#pragma unroll
            for (int i = 0; i < MT; ++i)
                load(arow[i], A[u][i]);
        }
#pragma unroll
        for (int u = 0; u < kCount; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NW; ++j)
                        acc[i][j] = mfma_i8(B[u][j][h], A[u][i][h], acc[i][j]);
        kb += KS * kCount;
    };
    while (kb + KS * (kBatch - 1) < nkb)
        blocks(std::integral_constant<int, kBatch>{});
    if (kBatch > 1 && kb < nkb)
        blocks(std::integral_constant<int, 1>{});
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
#pragma unroll
        for (int j = 0; j < NW; ++j) {
            const int n = n0 + 16 * j + 4 * g;
            float v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
                v[q] = (float)acc[i][j][q] * sa[i] * sb[j][q] + bias[j][q];
            store4<OUT>(p, m, n, v);
        }
    }
}

// ---- many rows: tiles through LDS ----
// Output tiles of 16 TM WM tokens x 16 TN WN channels, WM x WN waves of
// 16 TM x 16 TN each.  The 128-byte K blocks of a's and b's rows stream through
// a ring of NS LDS stages by LDS DMA; rows are stored unpadded, 16-byte chunk q
// of row r at q ^ ((r >> 1) & 7), so that a fragment read meets no bank conflict.
// A block is two slices of 64 bytes (one MFMA each); a slice's operands are read
// into registers under the MFMAs of the slice before it, in a second register
// set.  Between a block's two slices stands the barrier that hands blocks over:
// every wave holds the second slice in registers, so the stage is free for block
// kb + NS, and block kb + 1 has landed.
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

// A value that is the same in all lanes, in a scalar register (the builtin is
// dropped where the compiler knows that much, and the value may stay in a vector
// register, which the "s" operands below then get).  The VALU may have written v
// just before: a v_readfirstlane must not follow within a wait state, which the
// compiler does not see to inside assembly.
__device__ __forceinline__ uint32_t scalar(uint32_t v) {
    uint32_t r;
    asm volatile("s_nop 1\n\tv_readfirstlane_b32 %0, %1" : "=s"(r) : "v"(v));
    return r;
}

// LDS DMA of 16 bytes per lane from row + off to lds + 16 lane, by all lanes (`lanes` ~0) or none (0: what a
// step past the last block sends).  Counted by vmcnt.  (The row may come from a
// v_readfirstlane: a vector memory instruction must not read it within five wait
// states, and the compiler does not look for that inside assembly.)
__device__ __forceinline__ void dma16_if(const void* row, uint32_t off, uint32_t lds, uint32_t lanes) {
    asm volatile("s_mov_b32 m0, %2\n\ts_mov_b32 exec_lo, %3\n\ts_mov_b32 exec_hi, %3\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %1, %0\n\ts_mov_b64 exec, -1" ::"s"(row),
                 "v"(off), "s"(lds), "s"(lanes)
                 : "memory", "m0");
}

// The tile kernels' MFMA as inline assembly, its accumulator tied in place: left
// to itself the compiler gives the result other registers and copies the
// 256 accumulators around (150 copies to 128 MFMAs).  It knows of no
// wait states inside assembly: the operands come from LDS (whose waits it does
// insert), never from the VALU, and mfma_done() stands before the accumulators
// are read.
__device__ __forceinline__ void mfma_in_place(v4i_t& acc, v4i_t a, v4i_t b) {
    asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mfma_done() { asm volatile("s_nop 15\n\ts_nop 7" ::: "memory"); }

constexpr int kXcds = 8;

// Tile of workgroup `at`: workgroups go to the XCDs in turn, and each XCD, with
// an L2 of its own, takes a run of tiles in which group_m tiles along m share
// their b rows and neighbouring n share the a rows: so many that the 32 tiles its
// CUs work on together read as few different rows as may be, g bm = 32 / g bn.
// (256 x 256 tiles, us, g = 2, 4, 6, 8, 16: 8192 x 7168 x 7168 341, 346, 332, 344,
// 355; 8192^3 413, 407, 395, 407, 419.)
constexpr int group_m(int bm, int bn) {
    int g = 1;
    while ((2 * g + 1) * (2 * g + 1) * bm <= 4 * 32 * bn)
        ++g;
    return g;
}
template <int kGroupM>
__device__ __forceinline__ void tile_of(int at, int mtiles, int ntiles, int& mt, int& nt) {
    const int total = mtiles * ntiles, xcd = at % kXcds, each = total / kXcds, more = total % kXcds;
    const int t = xcd * each + min(xcd, more) + at / kXcds;
    const int per_group = kGroupM * ntiles, group = t / per_group, first = group * kGroupM;
    const int height = min(kGroupM, mtiles - first), in = t - group * per_group;
    mt = first + in % height;
    nt = in / height;
}

// Split K: with gridDim.y = S > 1, workgroup y takes its part of the K blocks
// and writes its int32 tile to partial y of `part` ([S][m][part_pitch(n)]);
// int8_mm_sum_kernel adds the partials and scales.  The sums are whole numbers,
// so the result is the unsplit one, bit for bit.
__host__ __device__ constexpr int64_t part_pitch(int64_t n) { return (n + 3) / 4 * 4; }

template <int WM, int WN, int TM, int TN, int NS, int OUT, bool SPLIT>
__global__ void __launch_bounds__(64 * WM * WN, 1) int8_mm_tile_kernel(MmArgs p, int32_t mtiles, int32_t ntiles,
                                                                       int32_t* part) {
    constexpr int kWaves = WM * WN, kBM = 16 * TM * WM, kBN = 16 * TN * WN, kABytes = kBM * kBlockK;
    constexpr int kStage = (kBM + kBN) * kBlockK;
    constexpr int kA = kBM / 8 / kWaves, kB = kBN / 8 / kWaves, kPer = kA + kB;  // DMAs per wave and block
    static_assert(kBM % (8 * kWaves) == 0 && kBN % (8 * kWaves) == 0, "tile shape");
    using Elem = std::conditional_t<OUT == kOutF32, float, uint16_t>;
    constexpr int kRowBytes = 16 * TN * sizeof(Elem) + 16, kCornerRows = OUT == kOutF32 ? 8 : 16;
    constexpr int kSa = (kBM + 63) / 64 * 64, kScales = kSa + (kBN + 63) / 64 * 64;
    __shared__ __attribute__((aligned(1024))) uint8_t st[NS][kStage];
    __shared__ __attribute__((aligned(16))) float scales[SPLIT ? 4 : kScales];

    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int c = lane & 15, g = lane >> 4, wm = wave / WN, wn = wave % WN;
    // the workgroup's K blocks: all, or the part blockIdx.y of them; at least one (K is a multiple of 128 here,
    // and no 0)
    const int all = p.k / kBlockK;
    const int kb_lo = SPLIT ? (int)((int64_t)all * blockIdx.y / gridDim.y) : 0;
    const int nkb = SPLIT ? (int)((int64_t)all * (blockIdx.y + 1) / gridDim.y) - kb_lo : all;

    int mt, nt;
    tile_of<group_m(kBM, kBN)>(blockIdx.x, mtiles, ntiles, mt, nt);
    const int m0 = mt * kBM, n0 = nt * kBN;

    // This lane's DMA sources, relative to the tile's first row: instruction j of
    // the wave covers 8 tile rows, lane / 8 of them, physical chunk lane % 8.
    // Rows past the end read the last one: they only feed outputs that are not stored.
    const int8_t* const abase = p.a + (int64_t)m0 * p.a_s + (int64_t)kb_lo * kBlockK;
    const int8_t* const bbase = p.b + (int64_t)n0 * p.b_s + (int64_t)kb_lo * kBlockK;
    uint32_t src[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const bool is_a = j < kA;
        const int row = 8 * (is_a ? wave * kA + j : wave * kB + j - kA) + (lane >> 3);
        const int r = is_a ? min(row, p.m - 1 - m0) : min(row, p.n - 1 - n0);
        src[j] = (uint32_t)r * (uint32_t)(is_a ? p.a_s : p.b_s) + 16 * swz(row, lane & 7);
    }
    auto issue = [&](int kb, uint32_t base, int j, uint32_t lanes) __attribute__((always_inline)) {
        const int8_t* row = (j < kA ? abase : bbase) + (int64_t)kb * kBlockK;
        dma16_if(row, src[j], base + (j < kA ? 1024 * (wave * kA + j) : kABytes + 1024 * (wave * kB + j - kA)), lanes);
    };
    auto sending = [&](int kb) __attribute__((always_inline)) {
        return scalar((kb - nkb) >> 31);  // ~0 below nkb
    };

    // A slice's operands: b's and a's last row in two register sets, a's other
    // rows in one (row i is reloaded behind its own MFMAs).
    v4i_t acc[TM][TN];
    v4i_t A[TM - 1], last[2], B[2][TN];
    const uint32_t lane_off = c * kBlockK + 16 * swz(c, g);
    const uint32_t aoff = wm * 16 * TM * kBlockK + lane_off, boff = kABytes + wn * 16 * TN * kBlockK + lane_off;
    // (slice 1 is chunk ^ 4)
    auto read_b = [&](const uint8_t* stage, int s, int j) __attribute__((always_inline)) {
        B[s][j] = *reinterpret_cast<const v4i_t*>(stage + (boff ^ (64 * s)) + 16 * j * kBlockK);
    };
    auto read_a = [&](const uint8_t* stage, int s, int i) __attribute__((always_inline)) {
        (i < TM - 1 ? A[i] : last[s]) =
            *reinterpret_cast<const v4i_t*>(stage + (aoff ^ (64 * s)) + 16 * i * kBlockK);
    };
    constexpr int kMfmas = TM * TN;
    constexpr int kSendEvery = kMfmas >= 4 * kPer ? 4 : kMfmas >= 2 * kPer ? 2 : 1;
    static_assert(kMfmas >= 2 * TN && kMfmas >= kPer * kSendEvery, "every read and DMA finds its MFMA");
    // MFMA u of slice s, and behind it what it lets go of of slice s ^ 1, which is in `stage`
    auto mfma_and_read = [&](int u, int s, const uint8_t* stage) __attribute__((always_inline)) {
        const int i = u / TN, j = u % TN;
        mfma_in_place(acc[i][j], B[s][j], i < TM - 1 ? A[i] : last[s]);
        if (u == 1)
            read_a(stage, s ^ 1, TM - 1);
        if (u % 2 == 0 && u / 2 < TN)
            read_b(stage, s ^ 1, u / 2);
        if (j == TN - 1 && i < TM - 1)
            read_a(stage, s ^ 1, i);
    };

    // the tile's scales, then its first NS blocks
    if constexpr (!SPLIT) {
#pragma unroll
        for (int i = 0; i < (kScales / 64 + kWaves - 1) / kWaves; ++i) {
            const int to = 64 * (wave + kWaves * i);
            if (to < kScales)
                dma4(to < kSa ? p.sa + min(m0 + to + lane, p.m - 1) * p.sa_s
                              : p.sb + min(n0 + to - kSa + lane, p.n - 1) * p.sb_s,
                     lds_addr(scales) + 4 * to);
        }
    }
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
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
            acc[i][j] = v4i_t{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < TN; ++j)
        read_b(st[0], 0, j);
#pragma unroll
    for (int i = 0; i < TM; ++i)
        read_a(st[0], 0, i);
    int at = 0, kb = 0;
    do {  // (there is a block: no way around the loop on which the accumulators would have to be moved)
        const uint8_t* cur = st[at];
        at = at + 1 < NS ? at + 1 : 0;
        const uint8_t* nxt = st[at];
        const uint32_t dst = lds_addr(cur);
#pragma unroll
        for (int u = 0; u < kMfmas; ++u) {
            mfma_and_read(u, 0, cur);
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
            // (behind the last block this reads a stage that nothing uses)
            mfma_and_read(u, 1, nxt);
            if (u % kSendEvery == 0 && u / kSendEvery < kPer)
                issue(kb + NS, dst, u / kSendEvery, lanes);
            __builtin_amdgcn_sched_barrier(0);
        }
    } while (++kb < nkb);
    mfma_done();
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
            asm volatile("" : "+a"(acc[i][j]));  // (no read of it moves in front of the wait)

    const int nb = n0 + wn * 16 * TN, mb = m0 + wm * 16 * TM;
    if constexpr (SPLIT) {
        const int64_t pitch = part_pitch(p.n);
        int32_t* to = part + (int64_t)blockIdx.y * p.m * pitch;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int m = mb + 16 * i + c;
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int n = nb + 16 * j + 4 * g;
                if (m < p.m && n < p.n)
                    *reinterpret_cast<v4i_t*>(to + m * pitch + n) = acc[i][j];
            }
        }
    } else {
        // ---- scales, bias, store ----
        // 16 tokens at a time through a corner of the stages of the wave's own (no
        // DMA is in flight, no wave reads a stage for use any more), so that a
        // store instruction writes whole runs of a row.  Rows 16 bytes apart
        // from a multiple of 256 keep the writes free of bank conflicts.
        constexpr int kVec = 16 / sizeof(Elem), kRowLanes = 16 * TN / kVec;
        constexpr int kRowsPer = kRowLanes <= 4 ? 16 : kRowLanes <= 8 ? 8 : kRowLanes <= 16 ? 4 : 2;
        static_assert(kRowLanes <= 32 && kWaves * kCornerRows * kRowBytes <= NS * kStage, "epilogue shape");
        using Put = std::conditional_t<OUT == kOutF32, float4, uint2>;
        uint8_t* const corner = &st[0][0] + wave * kCornerRows * kRowBytes;
        const float* const sas = scales + wm * 16 * TM + c;
        const float* const sbs = scales + kSa + wn * 16 * TN + 4 * g;
        const int my_row = lane / kRowLanes, my_col = lane % kRowLanes * kVec;
        const int rows = p.m - mb - my_row, cols = p.n - nb - my_col;  // still in range from this lane's on
        Elem* to = reinterpret_cast<Elem*>(p.out) + (int64_t)(mb + my_row) * p.o_s + nb + my_col;
        auto finish = [&](auto with_bias) __attribute__((always_inline)) {
            float bias[TN][4];
            if constexpr (decltype(with_bias)::value) {
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    bias4(p, nb + 16 * j + 4 * g, bias[j]);
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const float sa = sas[16 * i];
                Put put[TN];
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    const float4 sb = *reinterpret_cast<const float4*>(sbs + 16 * j);
                    float v[4] = {(float)acc[i][j][0] * sa * sb.x, (float)acc[i][j][1] * sa * sb.y,
                                  (float)acc[i][j][2] * sa * sb.z, (float)acc[i][j][3] * sa * sb.w};
                    if constexpr (decltype(with_bias)::value) {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            v[q] += bias[j][q];
                    }
                    if constexpr (OUT == kOutF32)
                        put[j] = make_float4(v[0], v[1], v[2], v[3]);
                    else
                        put[j] = make_uint2(pack_out<OUT>(v[0], v[1]), pack_out<OUT>(v[2], v[3]));
                }
#pragma unroll
                for (int h = 0; h < 16; h += kCornerRows) {
                    if (kCornerRows == 16 || (c & 8) == h) {
#pragma unroll
                        for (int j = 0; j < TN; ++j)
                            *reinterpret_cast<Put*>(corner + c % kCornerRows * kRowBytes +
                                                    (16 * j + 4 * g) * sizeof(Elem)) = put[j];
                    }
                    asm volatile("" ::: "memory");
#pragma unroll
                    for (int r = 0; r < kCornerRows; r += kRowsPer) {
                        if (my_row < kRowsPer && 16 * i + h + r < rows) {
                            const uint8_t* from = corner + (r + my_row) * kRowBytes + my_col * sizeof(Elem);
                            if (cols >= kVec) {
                                *reinterpret_cast<u32x4_a2*>(to) = *reinterpret_cast<const u32x4_t*>(from);
                            } else {
#pragma unroll 1
                                for (int e = 0; e < cols; ++e)
                                    to[e] = reinterpret_cast<const Elem*>(from)[e];
                            }
                        }
                        to += kRowsPer * p.o_s;
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    asm volatile("" ::: "memory");
                }
            }
        };
        if (p.bias)
            finish(std::true_type{});
        else
            finish(std::false_type{});
    }
}

// out = the sum of the partials, scaled: four channels of a token per thread.
template <int OUT>
__global__ void __launch_bounds__(256) int8_mm_sum_kernel(MmArgs p, const int32_t* part, int32_t splits) {
    const int64_t pitch = part_pitch(p.n), fours = pitch / 4, slot = p.m * pitch;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < p.m * fours; u += (int64_t)gridDim.x * 256) {
        const int64_t m = u / fours;
        const int n = (int)(u - m * fours) * 4;
        const float sa = p.sa[m * p.sa_s];
        float sb[4], bias[4], v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            sb[q] = p.sb[min(n + q, p.n - 1) * p.sb_s];
        bias4(p, n, bias);
        const v4i_t* from = reinterpret_cast<const v4i_t*>(part + 4 * u);
        v4i_t sum = from[0];
        for (int z = 1; z < splits; ++z)
            sum += from[z * (slot / 4)];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            v[q] = (float)sum[q] * sa * sb[q] + bias[q];
        store4<OUT>(p, m, n, v);
    }
}

// ---- rows that the tiles cannot take as they are ----
// Rows whose start or stride is no multiple of 16 bytes, or whose K is none of
// 128, are copied to rows of a whole number of K blocks, zeros behind K (which
// add nothing to a sum): a row per wave, a's rows, then b's.
struct PackArgs {
    const int8_t* from[2];
    int64_t from_s[2];
    int8_t* to[2];
    int64_t rows[2];
    int32_t k, pitch;  // pitch: K rounded up to 128
};

__global__ void __launch_bounds__(256) int8_mm_pack_kernel(PackArgs p) {
    int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;  // a wave takes a row
    const int which = row < p.rows[0] ? 0 : 1;
    row -= which * p.rows[0];
    if (row >= p.rows[which])
        return;
    const int8_t* from = p.from[which] + row * p.from_s[which];
    int8_t* to = p.to[which] + row * p.pitch;
    for (int k0 = 16 * (threadIdx.x % 64); k0 < p.pitch; k0 += 4096) {
        v4i_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)  // all four in flight
            v[i] = k0 + 1024 * i + 16 <= p.k ? load_frag(from, k0 + 1024 * i) : v4i_t{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = k0 + 1024 * i;
            if (k < p.k && k + 16 > p.k)
                v[i] = load_frag_end(from, k, p.k);
            if (k < p.pitch)
                *reinterpret_cast<v4i_t*>(to + k) = v[i];
        }
    }
}

// ---- schedules ----

// The tiles, by what a K block costs a CU that works on one of them (measured
// at K 7168 with a tile for nearly every CU, us: 64 x 64 21.2, 128 x 64 28.8,
// 128 x 128 36.9, 256 x 128 52.2, 192 x 256 79, 256 x 256 94 in all, about 3 of
// them before and behind the K loop; 128 x 192 25.1 at K 4096).  Sizes between
// the powers of two are there for the last turn: 6144 x 6144 x 6144 takes 193 us
// in tiles of 256 x 192, 211 in 256 x 256; 1024 x 4224 x 4096 25 in 128 x 192, 35
// in 128 x 128.  Below 256 x 192, which the matrix units bound (and at
// full size the power limit), the loads of the operands' rows do: 52-56 GB/s
// into a CU, however many blocks are in flight (NS 3, 4 and 5 alike).
struct TileKind {
    int bm, bn;
    float us_per_block;
};
constexpr TileKind kTiles[] = {{64, 64, 0.31f},   {128, 64, 0.43f},  {128, 128, 0.60f}, {128, 192, 0.69f},
                               {192, 128, 0.69f}, {256, 128, 0.85f}, {192, 256, 1.38f}, {256, 192, 1.38f}, {256, 256, 1.5f}};
constexpr int kTileKinds = 9;
constexpr float kTileFixedUs = 3.f;

struct Plan {
    bool rows;  // straight from memory
    int tile, splits;
    int64_t a_bytes, b_bytes, part_bytes;  // workspace: packed a, packed b, partials
    int64_t bytes() const { return a_bytes + b_bytes + part_bytes; }
};

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Where an operand's rows lie.
struct Rows {
    const int8_t* p;
    int64_t stride;
    // every row starts at a multiple of 16 bytes
    bool chunks() const { return aligned(p, 16) && stride % 16 == 0; }
    // the tiles' DMAs can read the rows as they are (32-bit offsets over the 256 rows of a tile)
    bool direct(int64_t k) const { return chunks() && stride >= 0 && stride < (1 << 23) && k % kBlockK == 0; }
};

// Workgroups of mt x nt tiles of 16 x 16.
int64_t row_groups(int64_t m, int64_t n, int mt, int nt) {
    return (m + 16 * mt - 1) / (16 * mt) * ((n + 16 * nt - 1) / (16 * nt));
}

// Rows straight from memory while
// - one pass of 16-row workgroups takes all tokens, or
// - workgroups of 16 x 16 have a CU each (256 x 256 x 7168 8.6 us, in split tiles 12), or
// - workgroups of 16 x 32 have, and the sum is not long enough for split tiles to catch up (us, and in tiles: 24 x
//   4096 x 4096 8.1, 9.4; 128 x 1024 x 1024 3.5, 4.6; 300 x 300 x 5120 9.3, 9.3; 48 x 2048 x 7168 11.7, 10.8), or tiles
//   would need the rows packed first (100 x 600 x 1000 4.8, 7.6; 64 x 1031 x 8001 17.4, 17.7; but 100 x 600 x 8001
//   17.6, 15.9), or
// - tiles would need that and workgroups of 32 x 32 have a CU each (64 x 4096 x 4111 11.6, 21.9), or
// - tiles would need b packed, two reads of it and a write, and one row of workgroups of 32 x 32 reads it once, however
//   many there are: with rows that are 16-byte aligned (17 x 16384 x 2880 10.9, 27.2; 32 x 28672 x 7008 69, 108; 32 x
//   8224 x 16016 72.9, 72.7), at any byte while the sum is short (32 x 16384 x 2879 18.7, 26.8; but 32 x 8224 x 6001
//   32.8, 29.7).  Beyond 32 tokens it depends (us, and packed: 64 x 8224 x 2880 14.9, 21.7; 64 x 8224 x 16016 90, 73;
//   64 x 7168 x 7001 38.7, 31.8); those are packed.
// Else the tile that takes the least time, counted as whole turns of the CUs; where even the smallest tiles leave more
// than half the CUs idle they are split along K, at least eight blocks each (128 x 2048 x 7168: 15.1 us, in four parts
// 11.3).
Plan plan_mm(int64_t m, int64_t n, int64_t k, const Rows& a, const Rows& b) {
    const bool a_direct = a.direct(k), b_direct = b.direct(k);
    Plan plan{true, 0, 1, 0, 0, 0};
    const int64_t cus = cu_count(), nkb = (k + kBlockK - 1) / kBlockK;
    const bool direct = a_direct && b_direct;
    if (k == 0 || m <= 16 || row_groups(m, n, 1, 1) <= cus)
        return plan;
    if (row_groups(m, n, 1, 2) <= cus && (nkb < 40 || !direct))
        return plan;
    if (!direct && row_groups(m, n, 2, 2) <= cus)
        return plan;
    if (!b_direct && m <= 32 && (nkb <= 32 || (a.chunks() && b.chunks())))
        return plan;
    plan.rows = false;
    float least = 0.f;
    for (int i = 0; i < kTileKinds; ++i) {
        const int64_t tiles = (m + kTiles[i].bm - 1) / kTiles[i].bm * ((n + kTiles[i].bn - 1) / kTiles[i].bn);
        const float us = (float)((tiles + cus - 1) / cus) * (kTileFixedUs + (float)nkb * kTiles[i].us_per_block);
        if (i == 0 || us < least) {
            least = us;
            plan.tile = i;
        }
    }
    if (plan.tile == 0) {
        const int64_t tiles = (m + 63) / 64 * ((n + 63) / 64);
        plan.splits = (int)std::max<int64_t>(1, std::min(cus / tiles, nkb / 8));
        if (plan.splits > 1)
            plan.part_bytes = up(plan.splits * m * part_pitch(n) * 4, 256);
    }
    if (!a_direct)
        plan.a_bytes = up(m * up(k, kBlockK), 256);
    if (!b_direct)
        plan.b_bytes = up(n * up(k, kBlockK), 256);
    return plan;
}

template <int WM, int WN, int TM, int TN, int NS, int OUT>
void launch_tiles(const MmArgs& p, hipStream_t st) {
    constexpr int kBM = 16 * TM * WM, kBN = 16 * TN * WN;
    const int32_t mtiles = (p.m + kBM - 1) / kBM, ntiles = (p.n + kBN - 1) / kBN;
    hipLaunchKernelGGL((int8_mm_tile_kernel<WM, WN, TM, TN, NS, OUT, false>), dim3((unsigned)(mtiles * ntiles)),
                       dim3(64 * WM * WN), 0, st, p, mtiles, ntiles, (int32_t*)nullptr);
}

template <int OUT>
void launch_split_tiles(const MmArgs& p, int splits, int32_t* part, hipStream_t st) {
    const int32_t mtiles = (p.m + 63) / 64, ntiles = (p.n + 63) / 64;
    hipLaunchKernelGGL((int8_mm_tile_kernel<2, 2, 2, 2, 4, kOutF32, true>), dim3((unsigned)(mtiles * ntiles), splits),
                       dim3(256), 0, st, p, mtiles, ntiles, part);
    const int64_t blocks = (p.m * (part_pitch(p.n) / 4) + 255) / 256;
    hipLaunchKernelGGL(int8_mm_sum_kernel<OUT>, dim3((unsigned)std::min<int64_t>(blocks, 65536)), dim3(256), 0, st, p,
                       (const int32_t*)part, (int32_t)splits);
}

template <int MT, int NW, int KS, int OUT>
void launch_rows(const MmArgs& p, hipStream_t st) {
    const dim3 grid((unsigned)((p.n + 16 * NW - 1) / (16 * NW)), (unsigned)((p.m + 16 * MT - 1) / (16 * MT)));
    const bool words = aligned(p.a, 4) && aligned(p.b, 4) && p.a_s % 4 == 0 && p.b_s % 4 == 0;
    if (words)
        hipLaunchKernelGGL((int8_mm_rows_kernel<MT, NW, KS, OUT, false>), grid, dim3(64 * KS), 0, st, p);
    else
        hipLaunchKernelGGL((int8_mm_rows_kernel<MT, NW, KS, OUT, true>), grid, dim3(64 * KS), 0, st, p);
}

template <int OUT>
int launch_mm(MmArgs p, void* workspace, int64_t workspace_bytes, hipStream_t st) {
    const Rows a{p.a, p.a_s}, b{p.b, p.b_s};
    const bool a_direct = a.direct(p.k), b_direct = b.direct(p.k);
    const Plan plan = plan_mm(p.m, p.n, p.k, a, b);
    const bool room = plan.bytes() == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= plan.bytes());
    if (plan.rows || !room) {
        // One tile of 16 x 16 to a workgroup while each has a CU of its own (256 x 256 x 7168 8.6 us, 2 x 2 of them to a
        // workgroup 15.2; 64 x 1024 x 4096 6.0 and 9.9); beyond, two along n halve the reads of a's rows (16 x 7168 x
        // 7168 16.5, one 18.7; one row of 16384 x 16384 loses), and where those have no CU each, two along m with them
        // those of b's (32 x 7168 x 7001 28.7, one 35.9).
        const bool alone = row_groups(p.m, p.n, 1, 1) <= cu_count();
        if (p.m > 16 && row_groups(p.m, p.n, 1, 2) > cu_count())
            launch_rows<2, 2, 8, OUT>(p, st);
        else if (p.m > 2 && !alone)
            launch_rows<1, 2, 8, OUT>(p, st);
        else if (p.k >= 16 * kBlockK)
            launch_rows<1, 1, 8, OUT>(p, st);
        else
            launch_rows<1, 1, 4, OUT>(p, st);
        return launch_status();
    }
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if (!a_direct || !b_direct) {
        const int32_t pitch = (int32_t)up(p.k, kBlockK);
        const PackArgs pack{{p.a, p.b},
                            {p.a_s, p.b_s},
                            {(int8_t*)ws, (int8_t*)ws + plan.a_bytes},
                            {a_direct ? 0 : p.m, b_direct ? 0 : p.n},
                            p.k,
                            pitch};
        hipLaunchKernelGGL(int8_mm_pack_kernel, dim3((unsigned)((pack.rows[0] + pack.rows[1] + 3) / 4)), dim3(256), 0, st,
                           pack);
        if (!a_direct) {
            p.a = pack.to[0];
            p.a_s = pitch;
        }
        if (!b_direct) {
            p.b = pack.to[1];
            p.b_s = pitch;
        }
        p.k = pitch;
    }
    if (plan.splits > 1) {
        launch_split_tiles<OUT>(p, plan.splits, reinterpret_cast<int32_t*>(ws + plan.a_bytes + plan.b_bytes), st);
        return launch_status();
    }
    switch (plan.tile) {
    case 0:
        launch_tiles<2, 2, 2, 2, 4, OUT>(p, st);
        break;
    case 1:
        launch_tiles<4, 2, 2, 2, 3, OUT>(p, st);
        break;
    case 2:
        launch_tiles<2, 4, 4, 2, 3, OUT>(p, st);
        break;
    case 3:
        launch_tiles<2, 4, 4, 3, 3, OUT>(p, st);
        break;
    case 4:
        launch_tiles<4, 2, 3, 4, 3, OUT>(p, st);
        break;
    case 5:
        launch_tiles<4, 2, 4, 4, 3, OUT>(p, st);
        break;
    case 6:
        launch_tiles<2, 4, 6, 4, 2, OUT>(p, st);
        break;
    case 7:
        launch_tiles<4, 2, 4, 6, 2, OUT>(p, st);
        break;
    default:
        launch_tiles<2, 4, 8, 4, 2, OUT>(p, st);
        break;
    }
    return launch_status();
}

}  // namespace
}  // namespace fgv

extern "C" int64_t fgv_int8_scaled_mm_workspace_bytes(const int8_t* a, int64_t a_stride, const int8_t* b,
                                                      int64_t b_stride, int64_t m, int64_t n, int64_t k) {
    using namespace fgv;
    if (m <= 0 || n <= 0 || k <= 0 || k > kMaxK || m > kMaxM || n > kMaxN)
        return 0;
    return plan_mm(m, n, k, Rows{a, a_stride}, Rows{b, b_stride}).bytes();
}

extern "C" int fgv_int8_scaled_mm(const int8_t* a, int64_t a_stride, const int8_t* b, int64_t b_stride,
                                  const float* scale_a, int64_t scale_a_stride, const float* scale_b,
                                  int64_t scale_b_stride, const void* bias, int32_t bias_dtype, void* out,
                                  int64_t out_stride, int64_t m, int64_t n, int64_t k, int32_t out_dtype,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace fgv;
    if (m < 0 || n < 0 || k < 0)
        return fail(FGV_E_BAD_SHAPE, "negative size");
    if (out_dtype < kOutBf16 || out_dtype > kOutF32 || (bias && (bias_dtype < kOutBf16 || bias_dtype > kOutF32)))
        return fail(FGV_E_BAD_SHAPE, "out_dtype and bias_dtype must be 0 (bf16), 1 (fp16) or 2 (fp32)");
    if (k > kMaxK)
        return fail(FGV_E_TOO_LARGE, "k above 131071: the int32 sum could overflow");
    if (m > kMaxM || n > kMaxN)
        return fail(FGV_E_TOO_LARGE, "m at most 2^20, n at most 2^24");
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
        return launch_mm<kOutBf16>(p, workspace, workspace_bytes, st);
    case kOutF16:
        return launch_mm<kOutF16>(p, workspace, workspace_bytes, st);
    default:
        return launch_mm<kOutF32>(p, workspace, workspace_bytes, st);
    }
}
