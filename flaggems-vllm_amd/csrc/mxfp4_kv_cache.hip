// gfx950 kernel that quantises a step's keys and values to MXFP4 and writes
// them into the paged cache (layout: mxfp4_cache.h).
//
// Per 32 values x of a head's row, a = max |x|:
//   e = clamp(ceil(log2(a / 6)), -126, 125), byte e + 127,
//   code = E2M1 value nearest to x 2^-e, ties to the even code, the sign kept;
// so the largest magnitude lands in (3, 6] and nothing is cut off (but above
// 6 * 2^125, in bf16 alone).  -126 is what zeros and values below 1.5 * 2^-124
// get.  A block that holds a NaN or an infinity gets byte 255, which stands for
// NaN, and codes 0.
//
// A thread takes 8 values of the key and the 8 at the same place of the value:
// the two share the slot and all of their addresses but a constant.  A block
// is a lane quad, its maximum two DPP steps; the codes come from
// v_cvt_scalef32_pk_fp4_{bf16,f16}, which divide by the scale and round as
// above.  A row's scale bytes are put together over its lanes and leave in one
// store.  The op moves 4 bytes in and 1.06 out per value pair and is bound by
// memory.  Consecutive workgroups stay on one XCD: a prefill's tokens fill pages
// in order, and the parts of a 128-byte line that several workgroups write
// then meet in one L2.
#include "fgv_device.h"
#include "fgv_host.h"
#include "mxfp4_cache.h"

namespace fgv {
namespace {

constexpr int kInsThreads = 256;
// Threads of a launch: one of 2^32 and more is cut to the low 32 bits without an error.
constexpr int64_t kInsMostThreads = 1LL << 31;

struct InsertArgs {
    const void* k;
    const void* v;
    int64_t k_st, k_sh, v_st, v_sh;  // elements
    uint8_t* cache;
    int64_t block_stride, num_slots;  // num_slots at most 2^32
    const int64_t* slots;
    uint32_t num_rows, kv_heads, page;  // rows: num_tokens * kv_heads
    uint32_t blocks_per_xcd;  // 0: in the launch's order
};

typedef __bf16 ins_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 ins_f16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short ins_u16x2 __attribute__((ext_vector_type(2)));

// ceil(log2(a / 6)) from a's bits, within [-126, 125] (a / 6 never rounds across a power of two).
__device__ __forceinline__ int mx_exponent(uint32_t amax_bits) {
    const uint32_t a = max(amax_bits, 0x01C00000u);  // 6 * 2^-126
    return min((int)(a >> 23) - 127 - 2 + ((a & 0x7fffffu) > 0x400000u ? 1 : 0), 125);
}

// Codes of 8 values (w: packed 16-bit pairs) and the scale byte of their quad.
template <bool kHalf>
__device__ __forceinline__ uint32_t mx_codes(const uint32_t (&w)[4], uint32_t& byte) {
    // magnitudes of 16-bit floats compare as integers
    ins_u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        m = __builtin_elementwise_max(m, __builtin_bit_cast(ins_u16x2, w[i] & 0x7fff7fffu));
    uint32_t most = m.x > m.y ? m.x : m.y;
    most = max(most, dpp_u32<kDppQuadXor1>(most));
    most = max(most, dpp_u32<kDppQuadXor2>(most));
    const bool bad = most >= (kHalf ? 0x7c00u : 0x7f80u);
    uint32_t bits;
    if constexpr (kHalf)
        bits = __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)most));
    else
        bits = most << 16;
    const int e = mx_exponent(bits);
    const float scale = __uint_as_float((uint32_t)(e + 127) << 23);
    uint32_t r = 0;
    if constexpr (kHalf) {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(ins_f16x2, w[0]), scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(ins_f16x2, w[1]), scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(ins_f16x2, w[2]), scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(ins_f16x2, w[3]), scale, 3);
    } else {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(ins_bf16x2, w[0]), scale, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(ins_bf16x2, w[1]), scale, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(ins_bf16x2, w[2]), scale, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(ins_bf16x2, w[3]), scale, 3);
    }
    byte = bad ? 255u : (uint32_t)(e + 127);
    return bad ? 0u : r;
}

template <bool kWide>
__device__ __forceinline__ void load8(const void* p, int64_t at, uint32_t (&w)[4]) {
    const uint16_t* s = static_cast<const uint16_t*>(p) + at;
    if constexpr (kWide) {
        const uint4 x = load16(s);
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = (uint32_t)s[2 * i] | (uint32_t)s[2 * i + 1] << 16;
    }
}

// The bytes of a row of D / 8 lanes (2, 4 or 8, from its quads) stored by its first lane.
template <int D>
__device__ __forceinline__ void store_scales(uint8_t* at, uint32_t byte, int piece) {
    if constexpr (D == 64) {
        const uint32_t two = byte | (dpp_u32<kDppRowRor12>(byte) << 8);
        if (piece == 0)
            *reinterpret_cast<uint16_t*>(at) = (uint16_t)two;
    } else {
        // lane i of a row of 16 reads the lanes 4, 8 and 12 places on
        const uint32_t four = byte | dpp_u32<kDppRowRor12>(byte) << 8 | dpp_u32<kDppRowRor8>(byte) << 16 |
                              dpp_u32<kDppRowRor4>(byte) << 24;
        if ((piece & 15) == 0)
            *reinterpret_cast<uint32_t*>(at + piece / 4) = four;
    }
}

template <int D, bool kHalf, bool kWide>
__global__ void __launch_bounds__(kInsThreads) mxfp4_insert_kernel(InsertArgs a) {
    constexpr int kPieces = D / 8;
    uint32_t wg = blockIdx.x;
    if (a.blocks_per_xcd)
        wg = (wg & 7) * a.blocks_per_xcd + (wg >> 3);
    const int piece = threadIdx.x % kPieces;
    const uint32_t row = wg * (kInsThreads / kPieces) + threadIdx.x / kPieces;
    if (row >= a.num_rows)
        return;  // whole rows of lanes: the DPP steps of the others stay inside theirs
    const uint32_t t = row / a.kv_heads, h = row - t * a.kv_heads;
    uint32_t kw[4], vw[4];
    load8<kWide>(a.k, t * a.k_st + (int64_t)h * a.k_sh + 8 * piece, kw);
    load8<kWide>(a.v, t * a.v_st + (int64_t)h * a.v_sh + 8 * piece, vw);
    const int64_t slot = a.slots[t];
    uint32_t kb, vb;
    const uint32_t kc = mx_codes<kHalf>(kw, kb);
    const uint32_t vc = mx_codes<kHalf>(vw, vb);
    if (slot < 0 || slot >= a.num_slots)
        return;
    // 32 bits: the 64-bit divisions of slot and row took more instructions than all the rest
    const uint32_t block = (uint32_t)slot / a.page;
    const int64_t page = a.page, place = (uint32_t)slot - block * a.page;
    uint8_t* head = a.cache + block * a.block_stride + h * page * mx_token_bytes(D);
    *reinterpret_cast<uint32_t*>(head + mx_part(0, page, D) + place * (D / 2) + 4 * piece) = kc;
    *reinterpret_cast<uint32_t*>(head + mx_part(1, page, D) + place * (D / 2) + 4 * piece) = vc;
    store_scales<D>(head + mx_part(2, page, D) + place * (D / kMxBlock), kb, piece);
    store_scales<D>(head + mx_part(3, page, D) + place * (D / kMxBlock), vb, piece);
}

template <int D>
void launch_insert(bool half, bool wide, hipStream_t st, InsertArgs a) {
    const int64_t groups = (a.num_rows + kInsThreads / (D / 8) - 1) / (kInsThreads / (D / 8));
    // a multiple of 8 workgroups, each XCD's a consecutive range (more than the grid's end: threads past the tokens leave)
    a.blocks_per_xcd = groups >= 64 ? (uint32_t)((groups + 7) / 8) : 0;
    const dim3 g(a.blocks_per_xcd ? 8 * a.blocks_per_xcd : (unsigned)groups), b(kInsThreads);
    if (half && wide)
        hipLaunchKernelGGL((mxfp4_insert_kernel<D, true, true>), g, b, 0, st, a);
    else if (half)
        hipLaunchKernelGGL((mxfp4_insert_kernel<D, true, false>), g, b, 0, st, a);
    else if (wide)
        hipLaunchKernelGGL((mxfp4_insert_kernel<D, false, true>), g, b, 0, st, a);
    else
        hipLaunchKernelGGL((mxfp4_insert_kernel<D, false, false>), g, b, 0, st, a);
}

}  // namespace
}  // namespace fgv

extern "C" int fgv_mxfp4_kv_quant_and_cache(const void* k, int64_t k_stride_token, int64_t k_stride_head, const void* v,
                                            int64_t v_stride_token, int64_t v_stride_head, int32_t dtype,
                                            int64_t num_tokens, int64_t num_kv_heads, int64_t head_dim, uint8_t* kv_cache,
                                            int64_t cache_block_stride, int64_t num_blocks, int64_t block_size,
                                            const int64_t* slot_mapping, void* stream) {
    using namespace fgv;
    if (num_tokens < 0 || num_kv_heads < 0 || num_blocks < 0)
        return fail(FGV_E_BAD_SHAPE, "negative size");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return fail(FGV_E_BAD_SHAPE, "head_dim must be 64, 128 or 256");
    if (dtype != 0 && dtype != 1)
        return fail(FGV_E_BAD_SHAPE, "dtype must be 0 (bf16) or 1 (fp16)");
    if (block_size <= 0 || block_size % 16 != 0)
        return fail(FGV_E_BAD_SHAPE, "block_size must be a positive multiple of 16");
    if (num_tokens == 0 || num_kv_heads == 0 || num_blocks == 0)
        return FGV_OK;
    if (num_kv_heads > 65536 || block_size > 4096)
        return fail(FGV_E_TOO_LARGE, "at most 65536 heads and 4096 tokens per block");
    const int64_t threads_per_token = num_kv_heads * (head_dim / 8);
    if (num_tokens > 0x7fffffffLL / num_kv_heads)
        return fail(FGV_E_TOO_LARGE, "num_tokens * num_kv_heads must be below 2^31");
    if (num_blocks > 0x100000000LL / block_size)
        return fail(FGV_E_TOO_LARGE, "the cache may hold at most 2^32 tokens");
    if (!k || !v || !kv_cache || !slot_mapping)
        return fail(FGV_E_NULL_POINTER, "null pointer argument");
    if (cache_block_stride < num_kv_heads * block_size * mx_token_bytes((int)head_dim) || cache_block_stride % 16 != 0)
        return fail(FGV_E_BAD_STRIDE, "cache_block_stride must hold a block and be a multiple of 16");
    if (!aligned(kv_cache, 16) || !aligned(slot_mapping, 8) || !aligned(k, 2) || !aligned(v, 2))
        return fail(FGV_E_MISALIGNED, "kv_cache must be 16-byte aligned, slot_mapping 8, k and v by element");
    InsertArgs a;
    a.k_st = k_stride_token;
    a.k_sh = k_stride_head;
    a.v_st = v_stride_token;
    a.v_sh = v_stride_head;
    a.cache = kv_cache;
    a.block_stride = cache_block_stride;
    a.num_slots = num_blocks * block_size;
    a.kv_heads = (uint32_t)num_kv_heads;
    a.page = (uint32_t)block_size;
    const bool wide = aligned(k, 16) && aligned(v, 16) &&
                      ((k_stride_token | k_stride_head | v_stride_token | v_stride_head) & 7) == 0;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t most = kInsMostThreads / threads_per_token;  // 2^10 tokens at least
    for (int64_t first = 0; first < num_tokens; first += most) {
        a.k = static_cast<const uint16_t*>(k) + first * k_stride_token;
        a.v = static_cast<const uint16_t*>(v) + first * v_stride_token;
        a.slots = slot_mapping + first;
        a.num_rows = (uint32_t)((num_tokens - first < most ? num_tokens - first : most) * num_kv_heads);
        switch (head_dim) {
            case 64: launch_insert<64>(dtype == 1, wide, st, a); break;
            case 128: launch_insert<128>(dtype == 1, wide, st, a); break;
            default: launch_insert<256>(dtype == 1, wide, st, a); break;
        }
    }
    return launch_status();
}
