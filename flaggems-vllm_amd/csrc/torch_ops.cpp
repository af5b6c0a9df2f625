// Host-side torch bindings of the path's ops:
//   fused_deepseek_v4_qnorm_rope_kv_rope_quant_insert  (reference wrapper
//     src/flaggems_vllm/ops/fused_deepseek_v4_qnorm_rope_kv_rope_quant_insert.py:289-351)
//   fused_inv_rope_fp8_quant                            (reference wrapper
//     src/flaggems_vllm/ops/fused_inv_rope_fp8_quant.py:157-256)
// and of the five ops beside them (fused_q_kv_rmsnorm,
// dequantize_and_gather_k_cache, fused_indexer_q_rope_quant,
// compute_slot_mapping_parallel, indexer_k_quant_and_cache) and the 8-bit
// linear ops around the layer (fused_add_rms_norm_quant,
// fused_silu_mul_quant, int8_scaled_mm) and the ops of the 4-bit paged cache
// (build_block_tables, mxfp4_kv_quant_and_cache, mxfp4_paged_attention), which
// have no counterpart there.
//
// The argument checks, the output allocation and the launch run here in C++,
// so an eager call costs a few microseconds of host time instead of the
// Python asserts plus a ctypes call of some twenty arguments.  The main op and
// the sibling are reachable two ways, both ending in the same function:
//   - the module functions (pybind11), which the Python drop-ins call.  They
//     return a status: 0, kAssertFailed (a reference assertion failed: the
//     Python side raises AssertionError with assert_message()), or the C ABI's
//     code (negative: argument error, positive: hipError_t);
//   - the dispatcher ops torch.ops.flaggems_vllm.<name> (TORCH_LIBRARY_FRAGMENT;
//     schemas mark q and k_cache written), for torch.compile and graph capture.
//     These raise RuntimeError on any failure, as vLLM's own compiled op does.
// The others are module functions only; their torch.ops registrations
// call the Python wrappers.
// Launches go on torch's current HIP stream of the tensors' device; nothing
// synchronises and nothing is read back from the device.
#include <cmath>

#include <torch/extension.h>
#include <torch/library.h>

#include <c10/core/DeviceGuard.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPStream.h>

#include <optional>
#include <string>
#include <tuple>
#include <utility>

#include "flaggems_vllm_amd.h"

namespace {

constexpr int kAssertFailed = -1000;
constexpr int64_t kHeadDim = 512;
constexpr int64_t kRopeDim = 64;

thread_local std::string g_assert_message;

int assert_failed(const char* msg) {
    g_assert_message = msg;
    return kAssertFailed;
}

#define FGV_ASSERT(cond, msg)              \
    do {                                   \
        if (!(cond))                       \
            return assert_failed(msg);     \
    } while (0)

void* current_stream(const at::Tensor& t) {
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// Whether each block t[i] is contiguous bytes: the dims after the first are
// dense in row-major order (dims of size 1 may have any stride), the test
// Tensor.is_contiguous() makes on t[0].
bool blocks_contiguous(const at::Tensor& t) {
    int64_t expected = 1;
    for (int64_t d = t.dim() - 1; d >= 1; --d) {
        const int64_t n = t.size(d);
        if (n != 1 && t.stride(d) != expected)
            return false;
        expected *= n;
    }
    return true;
}

// The reference's assertions (same conditions, same order), the extensions
// documented in the Python drop-in (strided q and kv, cos_sin row stride, a
// 1-D cache as one block), then one C-ABI launch.
int qnorm_rope_kv_insert(const at::Tensor& q, const at::Tensor& kv, const at::Tensor& k_cache,
                         const at::Tensor& slot_mapping, const at::Tensor& position_ids,
                         const at::Tensor& cos_sin_cache, double eps, int64_t cache_block_size) {
    FGV_ASSERT(q.dim() == 3 && kv.dim() == 2, "q must be 3-D and kv 2-D");
    FGV_ASSERT(q.stride(2) == 1 && kv.stride(1) == 1, "q and kv need a unit last stride");
    const int64_t num_tokens = q.size(0), num_heads = q.size(1);
    FGV_ASSERT(q.size(2) == kHeadDim, "q's head_dim must be 512");
    FGV_ASSERT(kv.size(0) == num_tokens && kv.size(1) == kHeadDim, "kv must be [num_tokens, 512]");
    FGV_ASSERT(q.scalar_type() == at::kBFloat16 && kv.scalar_type() == at::kBFloat16,
               "q and kv must be bfloat16");
    FGV_ASSERT(k_cache.scalar_type() == at::kByte, "k_cache must be uint8");
    FGV_ASSERT(slot_mapping.dim() == 1, "slot_mapping must be 1-D");
    const int64_t num_tokens_insert = slot_mapping.size(0);
    FGV_ASSERT(num_tokens_insert <= num_tokens, "slot_mapping is longer than the number of tokens");
    FGV_ASSERT(slot_mapping.scalar_type() == at::kLong, "slot_mapping must be int64");
    FGV_ASSERT(position_ids.dim() == 1 && position_ids.size(0) == num_tokens,
               "position_ids must be [num_tokens]");
    FGV_ASSERT(position_ids.scalar_type() == at::kLong, "position_ids must be int64");
    FGV_ASSERT(cos_sin_cache.dim() == 2 && cos_sin_cache.size(1) == kRopeDim,
               "cos_sin_cache must be [max_pos, 64]");
    FGV_ASSERT(cos_sin_cache.scalar_type() == at::kFloat, "cos_sin_cache must be float32");
    FGV_ASSERT(cos_sin_cache.stride(1) == 1, "cos_sin_cache rows must be contiguous");
    FGV_ASSERT(slot_mapping.stride(0) == 1 || num_tokens_insert <= 1, "slot_mapping must be contiguous");
    FGV_ASSERT(position_ids.stride(0) == 1 || num_tokens <= 1, "position_ids must be contiguous");
    FGV_ASSERT(k_cache.dim() >= 1 && blocks_contiguous(k_cache), "each k_cache block must be contiguous bytes");
    const c10::Device dev = q.device();
    FGV_ASSERT(kv.device() == dev && k_cache.device() == dev && slot_mapping.device() == dev &&
                   position_ids.device() == dev && cos_sin_cache.device() == dev,
               "all tensors must be on q's device");
    FGV_ASSERT(dev.is_cuda(), "flaggems_vllm runs on the GPU (HIP) only");

    if (num_tokens == 0)
        return 0;
    // A [num_blocks, block_bytes] cache (or more dims) has size(0) blocks,
    // stride(0) bytes apart; a 1-D cache is one block of numel bytes.
    const bool one_block = k_cache.dim() == 1;
    const int64_t num_blocks = one_block ? 1 : k_cache.size(0);
    const int64_t block_stride = one_block ? k_cache.numel() : k_cache.stride(0);
    const c10::DeviceGuard guard(dev);
    return fgv_qnorm_rope_kv_rope_quant_insert(
        q.data_ptr(), q.stride(0), q.stride(1), kv.data_ptr(), kv.stride(0), k_cache.data_ptr(), block_stride,
        num_blocks, slot_mapping.data_ptr<int64_t>(), num_tokens_insert, position_ids.data_ptr<int64_t>(),
        cos_sin_cache.data_ptr<float>(), cos_sin_cache.stride(0), cos_sin_cache.size(0), num_tokens, num_heads,
        static_cast<float>(eps), cache_block_size, current_stream(q));
}

using SiblingOut = std::tuple<at::Tensor, at::Tensor>;

// The reference's assertions in its order (:184-205, plus this build's
// geometry limits), its output allocation (:207-227): codes [G, T, hpg * D]
// e4m3fn and scales stored (G, K, Tpad4) token-fastest, returned transposed to
// [T, G, d] and [T, G, K]; then one C-ABI launch.
int inv_rope_fp8_quant(const at::Tensor& o, const at::Tensor& positions_in, const at::Tensor& cos_sin_cache,
                       int64_t n_groups, int64_t heads_per_group, int64_t nope_dim, int64_t rope_dim,
                       int64_t quant_group_size, double eps, bool fp8_e4m3fn, bool tma_aligned_scales,
                       SiblingOut* out) {
    FGV_ASSERT(fp8_e4m3fn, "only torch.float8_e4m3fn is supported");
    FGV_ASSERT(o.dim() == 3, "`o` must be [num_tokens, num_heads, head_dim]");
    FGV_ASSERT(positions_in.dim() == 1, "`positions` must be 1D");
    FGV_ASSERT(cos_sin_cache.dim() == 2, "`cos_sin_cache` must be 2D");
    FGV_ASSERT(o.stride(2) == 1, "head_dim must be contiguous");
    FGV_ASSERT(positions_in.size(0) == o.size(0), "positions and o token count mismatch");
    const int64_t num_tokens = o.size(0), num_heads = o.size(1), head_dim = o.size(2);
    FGV_ASSERT(num_heads == n_groups * heads_per_group, "num_heads must be n_groups * heads_per_group");
    FGV_ASSERT(head_dim == nope_dim + rope_dim, "head_dim must be nope_dim + rope_dim");
    FGV_ASSERT(quant_group_size > 0 && head_dim % quant_group_size == 0,
               "head_dim must be a multiple of quant_group_size");
    FGV_ASSERT(nope_dim % quant_group_size == quant_group_size - rope_dim,
               "nope_dim % quant_group_size must be quant_group_size - rope_dim");
    FGV_ASSERT(rope_dim % 2 == 0, "rope_dim must be even");
    FGV_ASSERT(cos_sin_cache.size(1) == rope_dim, "cos_sin_cache's last dim must be rope_dim");
    FGV_ASSERT(cos_sin_cache.scalar_type() == at::kFloat, "cos_sin_cache must be float32");
    FGV_ASSERT((head_dim & (head_dim - 1)) == 0 && head_dim >= 8 && head_dim <= 512 &&
                   (quant_group_size & (quant_group_size - 1)) == 0 && quant_group_size >= 8,
               "this build takes head_dim a power of two in [8, 512] and quant_group_size a power of two >= 8");
    FGV_ASSERT(o.scalar_type() == at::kBFloat16, "`o` must be bfloat16");
    FGV_ASSERT(cos_sin_cache.stride(1) == 1, "cos_sin_cache rows must be contiguous");
    const c10::Device dev = o.device();
    FGV_ASSERT(dev.is_cuda(), "flaggems_vllm runs on the GPU (HIP) only");
    FGV_ASSERT(positions_in.device() == dev && cos_sin_cache.device() == dev, "all tensors must be on o's device");
    const int64_t chunks_per_head = head_dim / quant_group_size;
    if (tma_aligned_scales) {
        FGV_ASSERT(chunks_per_head <= 4, "packed UE8M0 path currently expects at most 4 scale blocks per head");
        // the reference's packed tensor holds (hpg * chunks + 3) / 4 words per
        // (group, token) and its kernel writes one per head: below four chunks
        // that is past the tensor unless there is one head per group
        FGV_ASSERT(chunks_per_head == 4 || heads_per_group == 1,
                   "packed scales with fewer than 4 scale blocks per head need heads_per_group 1");
    }

    const at::Tensor positions = (positions_in.scalar_type() != at::kLong || positions_in.stride(0) != 1)
                                     ? positions_in.to(at::kLong).contiguous()
                                     : positions_in;
    const int64_t d = heads_per_group * head_dim;
    const int64_t num_scale_blocks = d / quant_group_size;
    const int64_t tpad = (num_tokens + 3) / 4 * 4;
    const int64_t scale_inner = tma_aligned_scales ? (num_scale_blocks + 3) / 4 : num_scale_blocks;
    const auto opts = o.options();
    // both outputs allocated straight in the returned layouts (no transposed
    // views to make): codes [T, G, d] over storage [G][T][d]; scales
    // [T, G, K] over storage [G][K][Tpad] (all Tpad columns: the kernel writes
    // the padding tokens' zero scales)
    at::Tensor fp8 = at::empty_strided({num_tokens, n_groups, d}, {d, num_tokens * d, 1},
                                       opts.dtype(at::kFloat8_e4m3fn));
    at::Tensor scale = at::empty({n_groups * scale_inner * tpad}, opts.dtype(tma_aligned_scales ? at::kInt : at::kFloat))
                           .as_strided({num_tokens, n_groups, scale_inner}, {1, scale_inner * tpad, tpad});
    int rc = 0;
    if (tpad > 0) {
        const c10::DeviceGuard guard(dev);
        rc = fgv_inv_rope_fp8_quant(o.data_ptr(), o.stride(0), o.stride(1), positions.data_ptr<int64_t>(),
                                    cos_sin_cache.data_ptr<float>(), cos_sin_cache.stride(0), cos_sin_cache.size(0),
                                    num_tokens, n_groups, heads_per_group, nope_dim, rope_dim, quant_group_size,
                                    fp8.data_ptr(), fp8.stride(1),
                                    fp8.stride(0), scale.data_ptr(), scale.stride(1), scale.stride(2), tpad,
                                    static_cast<float>(eps), tma_aligned_scales ? 1 : 0, current_stream(o));
    }
    *out = SiblingOut(fp8, scale);
    return rc;
}

// ---- the ops beside the path: checks, allocation and launch of their Python drop-ins ----

using TensorPair = std::tuple<at::Tensor, at::Tensor>;

int32_t* i32_ptr(const at::Tensor& t) { return t.data_ptr<int32_t>(); }

at::Tensor to_i32(const at::Tensor& t) { return t.scalar_type() == at::kInt ? t : t.to(at::kInt); }

// fused_q_kv_rmsnorm (reference wrapper
// src/flaggems_vllm/ops/deepseek_v4_attention_fused_q_kv_rmsnorm.py:65-103):
// outputs like qr and kv, one C-ABI launch.
int q_kv_rmsnorm(const at::Tensor& qr, const at::Tensor& kv, const at::Tensor& q_weight, const at::Tensor& kv_weight,
                 double eps, TensorPair* out) {
    FGV_ASSERT(qr.dim() == 2 && kv.dim() == 2, "qr and kv must be 2D [num_tokens, size]");
    FGV_ASSERT(qr.size(0) == kv.size(0), "qr and kv token count mismatch");
    FGV_ASSERT(qr.stride(-1) == 1 && kv.stride(-1) == 1, "qr and kv rows must be contiguous");
    FGV_ASSERT(q_weight.is_contiguous() && kv_weight.is_contiguous(), "weights must be contiguous");
    const int64_t q_size = qr.size(1), kv_size = kv.size(1), num_tokens = qr.size(0);
    at::Tensor qr_out = at::empty_like(qr), kv_out = at::empty_like(kv);
    *out = TensorPair(qr_out, kv_out);
    if (num_tokens == 0)
        return 0;
    FGV_ASSERT(qr.scalar_type() == at::kBFloat16 && kv.scalar_type() == at::kBFloat16, "bf16 activations");
    FGV_ASSERT(q_weight.scalar_type() == kv_weight.scalar_type() &&
                   (q_weight.scalar_type() == at::kBFloat16 || q_weight.scalar_type() == at::kFloat),
               "weights must be both bf16 or both float32");
    FGV_ASSERT(q_weight.numel() == q_size && kv_weight.numel() == kv_size, "weight sizes must match the row sizes");
    const c10::Device dev = qr.device();
    FGV_ASSERT(dev.is_cuda(), "flaggems_vllm runs on the GPU (HIP) only");
    FGV_ASSERT(kv.device() == dev && q_weight.device() == dev && kv_weight.device() == dev,
               "all tensors must be on qr's device");
    const c10::DeviceGuard guard(dev);
    return fgv_fused_q_kv_rmsnorm(qr.data_ptr(), qr.stride(0), qr_out.data_ptr(), qr_out.stride(0),
                                  q_weight.data_ptr(), q_size, kv.data_ptr(), kv.stride(0), kv_out.data_ptr(),
                                  kv_out.stride(0), kv_weight.data_ptr(), kv_size, num_tokens,
                                  static_cast<float>(eps), q_weight.scalar_type() == at::kFloat ? 1 : 0,
                                  current_stream(qr));
}

// dequantize_and_gather_k_cache (reference wrapper
// src/flaggems_vllm/ops/deepseek_v4_attention_dequantize_and_gather_k_cache.py:123-172):
// out written in place; int64 index tensors converted to int32.
int dequantize_gather(const at::Tensor& out, const at::Tensor& k_cache, const at::Tensor& seq_lens_in,
                      const std::optional<at::Tensor>& gather_lens_in, const at::Tensor& block_table_in,
                      int64_t block_size, int64_t offset, int64_t rope_dim, std::optional<int64_t> nope_dim_in,
                      std::optional<int64_t> scale_slots_in) {
    FGV_ASSERT(out.dim() == 3 && out.scalar_type() == at::kBFloat16, "out must be 3D bfloat16");
    FGV_ASSERT(seq_lens_in.dim() == 1 && block_table_in.dim() == 2, "seq_lens must be 1D and block_table 2D");
    FGV_ASSERT(seq_lens_in.size(0) == block_table_in.size(0) && block_table_in.size(0) <= out.size(0),
               "seq_lens, block_table and out must agree on the request count");
    const int64_t nope_dim = nope_dim_in.has_value() ? *nope_dim_in : out.size(2) - rope_dim;
    const int64_t scale_slots =
        scale_slots_in.has_value() ? *scale_slots_in : (nope_dim + 63) / 64 + (nope_dim % 64 == 0 ? 1 : 0);
    FGV_ASSERT(nope_dim + rope_dim <= out.size(2), "nope_dim + rope_dim must fit out's last dim");
    FGV_ASSERT(k_cache.dim() == 2 || k_cache.dim() == 3, "k_cache must be 2D or 3D");
    FGV_ASSERT(out.stride(2) == 1, "out rows must be contiguous");
    FGV_ASSERT(blocks_contiguous(k_cache), "each k_cache block must be contiguous bytes");
    FGV_ASSERT(block_table_in.stride(1) == 1, "block_table rows must be contiguous");
    const c10::Device dev = out.device();
    FGV_ASSERT(dev.is_cuda(), "flaggems_vllm runs on the GPU (HIP) only");
    FGV_ASSERT(k_cache.device() == dev && seq_lens_in.device() == dev && block_table_in.device() == dev &&
                   (!gather_lens_in.has_value() || gather_lens_in->device() == dev),
               "all tensors must be on out's device");
    const at::Tensor seq_lens = to_i32(seq_lens_in).contiguous();
    const at::Tensor gather_lens =
        gather_lens_in.has_value() ? to_i32(*gather_lens_in).contiguous() : at::Tensor();
    const at::Tensor block_table = to_i32(block_table_in);
    const int64_t num_reqs = seq_lens.size(0);
    if (num_reqs == 0)
        return 0;
    const c10::DeviceGuard guard(dev);
    return fgv_dequantize_and_gather_k_cache(
        out.data_ptr(), out.stride(0), out.stride(1), out.size(1), k_cache.data_ptr(), k_cache.stride(0),
        k_cache.size(0), i32_ptr(seq_lens), gather_lens.defined() ? i32_ptr(gather_lens) : nullptr,
        i32_ptr(block_table), block_table.stride(0), block_table.size(1), num_reqs, block_size, offset, nope_dim,
        rope_dim, scale_slots, current_stream(out));
}

using IndexerOut = std::tuple<at::Tensor, at::Tensor, at::Tensor>;

// fused_indexer_q_rope_quant (reference wrapper
// src/flaggems_vllm/ops/fused_indexer_q_rope_quant.py:285-410): returns
// (q codes, the UE8M0 scale bytes viewed as int32 [T, H, D/128] and squeezed
// to [T, H] for D = 128 (MXFP4), or an undefined tensor (FP8), folded weights).
int indexer_q_rope_quant(const at::Tensor& positions_in, const at::Tensor& index_q, const at::Tensor& cos_sin,
                         const at::Tensor& weights, double softmax_scale, double head_scale, bool use_fp4,
                         IndexerOut* out) {
    FGV_ASSERT(positions_in.dim() == 1, "positions must be 1D");
    FGV_ASSERT(index_q.dim() == 3, "index_q must be [num_tokens, num_heads, head_dim]");
    FGV_ASSERT(cos_sin.dim() == 2, "index_q_cos_sin_cache must be 2D");
    const int64_t num_tokens = positions_in.size(0), num_heads = index_q.size(1), head_dim = index_q.size(2);
    at::Tensor weights_out = at::empty_like(weights, weights.options().dtype(at::kFloat));
    FGV_ASSERT(index_q.scalar_type() == at::kBFloat16 && index_q.stride(2) == 1,
               "index_q must be bfloat16 with contiguous rows");
    FGV_ASSERT(index_q.size(0) >= num_tokens, "index_q has fewer rows than positions");
    FGV_ASSERT(cos_sin.size(-1) == 64, "rope dim 64");
    FGV_ASSERT(cos_sin.scalar_type() == at::kFloat || cos_sin.scalar_type() == at::kBFloat16,
               "index_q_cos_sin_cache must be float32 or bfloat16");
    FGV_ASSERT(cos_sin.stride(-1) == 1, "index_q_cos_sin_cache rows must be contiguous");
    FGV_ASSERT(weights.scalar_type() == at::kBFloat16 || weights.scalar_type() == at::kFloat,
               "index_weights must be bfloat16 or float32");
    FGV_ASSERT(weights.dim() == 2 && weights.stride(-1) == 1, "index_weights must be 2D with contiguous rows");
    FGV_ASSERT(weights.size(0) >= num_tokens && weights.size(1) == num_heads,
               "index_weights must be [>= num_tokens, num_heads]");
    FGV_ASSERT(head_dim == 128 || head_dim == 256 || head_dim == 512, "head_dim 128, 256 or 512");
    const c10::Device dev = index_q.device();
    FGV_ASSERT(dev.is_cuda(), "flaggems_vllm runs on the GPU (HIP) only");
    FGV_ASSERT(positions_in.device() == dev && cos_sin.device() == dev && weights.device() == dev,
               "all tensors must be on index_q's device");
    const at::Tensor positions = (positions_in.scalar_type() != at::kLong || positions_in.stride(0) != 1)
                                     ? positions_in.to(at::kLong).contiguous()
                                     : positions_in;
    at::Tensor q_out, scale;
    if (use_fp4) {
        q_out = at::empty({num_tokens, num_heads, head_dim / 2}, index_q.options().dtype(at::kByte));
        scale = at::empty({num_tokens, num_heads, head_dim / 32}, index_q.options().dtype(at::kByte));
    } else {
        // as the reference allocates it: index_q's shape and layout
        q_out = at::empty_like(index_q, index_q.options().dtype(at::kFloat8_e4m3fn));
        FGV_ASSERT(q_out.stride(2) == 1, "q codes must have contiguous rows");
    }
    *out = IndexerOut(q_out, scale.defined() ? scale.view(at::kInt).squeeze(-1) : scale, weights_out);
    const c10::DeviceGuard guard(dev);
    return fgv_fused_indexer_q_rope_quant(
        positions.data_ptr<int64_t>(), num_tokens, index_q.data_ptr(), index_q.stride(0), index_q.stride(1),
        num_heads, head_dim, cos_sin.data_ptr(), cos_sin.stride(0), cos_sin.size(0),
        cos_sin.scalar_type() == at::kBFloat16 ? 1 : 0, weights.data_ptr(), weights.stride(0),
        weights.scalar_type() == at::kFloat ? 1 : 0, static_cast<float>(softmax_scale),
        static_cast<float>(head_scale), weights_out.data_ptr<float>(), weights_out.stride(0), use_fp4 ? 1 : 0,
        q_out.data_ptr(), q_out.stride(0), q_out.stride(1), scale.defined() ? scale.data_ptr() : nullptr,
        scale.defined() ? scale.stride(0) : 0, scale.defined() ? scale.stride(1) : 0, current_stream(index_q));
}

// indexer_k_quant_and_cache's checks (the ValueError on head_dim stays with
// the Python drop-in) and launch.  kv_cache[0] and slot_mapping.shape[0]
// raise IndexError where they do not exist, as there.
int indexer_k_quant(const at::Tensor& k, const at::Tensor& kv_cache, const at::Tensor& slot_mapping,
                    int64_t quant_block_size, bool use_ue8m0) {
    TORCH_CHECK_INDEX(slot_mapping.dim() > 0, "slot_mapping must have a dimension");
    const int64_t num_tokens = slot_mapping.size(0), head_dim = k.size(-1);
    FGV_ASSERT(k.scalar_type() == at::kBFloat16 || k.scalar_type() == at::kHalf, "k must be bfloat16 or float16");
    FGV_ASSERT(kv_cache.dim() == 3 && kv_cache.element_size() == 1,
               "kv_cache must be [num_blocks, block_size, bytes per token] of a 1-byte type");
    TORCH_CHECK_INDEX(kv_cache.size(0) > 0, "kv_cache has no block");
    FGV_ASSERT(blocks_contiguous(kv_cache), "each kv_cache block must be contiguous bytes");
    FGV_ASSERT(slot_mapping.dim() == 1 && slot_mapping.scalar_type() == at::kLong, "slot_mapping must be 1-D int64");
    FGV_ASSERT(slot_mapping.stride(0) == 1 || num_tokens <= 1, "slot_mapping must be contiguous");
    const at::Tensor k2 = k.dim() != 2 ? k.reshape({-1, head_dim}) : k;
    FGV_ASSERT(k2.size(0) >= num_tokens, "k has fewer rows than slot_mapping");
    FGV_ASSERT(k2.stride(-1) == 1, "k rows must be contiguous");
    FGV_ASSERT(kv_cache.device() == k.device() && slot_mapping.device() == k.device(),
               "all tensors must be on k's device");
    FGV_ASSERT(k.is_cuda(), "flaggems_vllm runs on the GPU (HIP) only");
    if (num_tokens == 0)
        return 0;
    const c10::DeviceGuard guard(k.device());
    return fgv_indexer_k_quant_and_cache(k2.data_ptr(), k2.stride(0), k.scalar_type() == at::kHalf ? 1 : 0, num_tokens,
                                         head_dim, quant_block_size, kv_cache.data_ptr(), kv_cache.stride(0),
                                         kv_cache.size(0), kv_cache.size(1), slot_mapping.data_ptr<int64_t>(),
                                         use_ue8m0 ? 1 : 0, current_stream(k));
}


// compute_slot_mapping_parallel (reference
// src/flaggems_vllm/runtime/backend/_ascend/ops/slot_mapping.py:109-144):
// slot_mapping written in place.
int slot_mapping(int64_t num_tokens, int64_t max_num_tokens, const at::Tensor& query_start_loc_in, int64_t num_reqs,
                 const at::Tensor& positions, const at::Tensor& block_table, const at::Tensor& slot_mapping_out,
                 int64_t block_size, int64_t cp_world_size, int64_t cp_rank, int64_t cp_interleave, int64_t pad_id) {
    FGV_ASSERT(slot_mapping_out.scalar_type() == at::kLong && slot_mapping_out.stride(-1) == 1,
               "slot_mapping must be contiguous int64");
    FGV_ASSERT(slot_mapping_out.numel() >= max_num_tokens, "slot_mapping holds fewer than max_num_tokens entries");
    FGV_ASSERT(query_start_loc_in.scalar_type() == at::kInt && query_start_loc_in.numel() >= num_reqs + 1,
               "query_start_loc must be int32 with num_reqs + 1 entries");
    FGV_ASSERT((positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong) &&
                   positions.stride(-1) == 1,
               "positions must be contiguous int32 or int64");
    FGV_ASSERT(block_table.scalar_type() == at::kInt && block_table.dim() == 2, "block_table must be 2D int32");
    FGV_ASSERT(block_table.stride(-1) == 1, "block_table rows must be contiguous");
    const c10::Device dev = slot_mapping_out.device();
    FGV_ASSERT(dev.is_cuda(), "flaggems_vllm runs on the GPU (HIP) only");
    FGV_ASSERT(query_start_loc_in.device() == dev && positions.device() == dev && block_table.device() == dev,
               "all tensors must be on slot_mapping's device");
    const at::Tensor query_start_loc = query_start_loc_in.contiguous();
    const c10::DeviceGuard guard(dev);
    return fgv_compute_slot_mapping(num_tokens, max_num_tokens, i32_ptr(query_start_loc), num_reqs,
                                    positions.data_ptr(), positions.scalar_type() == at::kLong ? 1 : 0,
                                    i32_ptr(block_table), block_table.stride(0), block_table.size(1),
                                    slot_mapping_out.data_ptr<int64_t>(), block_size, cp_world_size, cp_rank,
                                    cp_interleave, pad_id, current_stream(slot_mapping_out));
}

// ---- the 8-bit linear ops: norm or activation to codes and scales, int8 product ----

// Whether autograd expects a derivative of t: backward, or the tangent of a
// forward-mode dual tensor (which is carried on without grad mode, too).
bool takes_grad(const at::Tensor& t) {
    return (t.requires_grad() && at::GradMode::is_enabled()) ||
           (t._fw_grad(/*level=*/0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode());
}

// Why t's values are not what a kernel would read at its address, or null.  A
// lazily negated view (the imaginary part of a conjugate) has them with the other
// sign; fake tensors and tensors whose storage was freed have no memory, and a
// view into them has an address that is neither null nor valid.
const char* not_readable(const at::Tensor& t) {
    if (t.is_neg())
        return "no tensor may be a lazily negated view (resolve_neg() gives its values)";
    const at::Storage& s = t.unsafeGetTensorImpl()->unsafe_storage();
    if (t.numel() > 0 && (!s || s.unsafeGetStorageImpl()->data_ptr().get() == nullptr))
        return "every tensor must have memory (no fake tensors, no freed storage)";
    return nullptr;
}
const char* not_readable(const std::optional<at::Tensor>& t) { return t ? not_readable(*t) : nullptr; }

// The first reason among several tensors.
template <class... Tensors>
const char* any_not_readable(const Tensors&... tensors) {
    const char* why = nullptr;
    ((why = why ? why : not_readable(tensors)), ...);
    return why;
}

bool unit_rows(const at::Tensor& t) { return t.size(1) <= 1 || t.stride(1) == 1; }

// Bytes [first, last) that a tensor of at least one element spans.
std::pair<uintptr_t, uintptr_t> span_of(const at::Tensor& t) {
    const auto first = reinterpret_cast<uintptr_t>(t.data_ptr());
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d)
        last += (t.size(d) - 1) * t.stride(d);
    return {first, first + (last + 1) * t.element_size()};
}

bool spans_meet(const at::Tensor& a, const at::Tensor& b) {
    if (a.numel() == 0 || b.numel() == 0)
        return false;
    const auto x = span_of(a), y = span_of(b);
    return x.first < y.second && y.first < x.second;
}

// Whether rows of `to` (2-D, the shape and type of `from`) may be written while
// those of `from` are read row by row: the same rows, rows side by side in one
// wider buffer, or other memory.
bool rows_apart_or_same(const at::Tensor& to, const at::Tensor& from) {
    if (!spans_meet(to, from))
        return true;
    const int64_t rows = to.size(0), cols = to.size(1);
    if (to.data_ptr() == from.data_ptr())
        return rows <= 1 || to.stride(0) == from.stride(0);
    if (rows <= 1 || to.stride(0) != from.stride(0))
        return false;
    const int64_t size = to.element_size(), step = to.stride(0) * size;
    int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(to.data_ptr()) -
                                       reinterpret_cast<uintptr_t>(from.data_ptr())) % step;
    if (off < 0)
        off += step;
    return off >= cols * size && step - off >= cols * size;
}

constexpr int64_t kQuantGroup = 128;
constexpr int64_t kQuantMaxCols = 65536;

// A new tensor on the GPU, past the dispatcher (three at::empty cost a short
// call about 2 us of host time, these half of it).
at::Tensor new_on(const c10::Device& dev, at::IntArrayRef sizes, at::ScalarType type) {
    return at::detail::empty_cuda(sizes, type, dev, std::nullopt);
}

// Checks that both producers share, and their outputs: codes [rows, cols] and
// scales [rows, 1] (int8) or [rows, cols / 128] (e4m3fn).
int quant_outputs(const at::Tensor& x, int64_t cols, bool int8, at::Tensor* codes, at::Tensor* scales) {
    FGV_ASSERT(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "x must be bfloat16 or float16");
    FGV_ASSERT(cols >= 1 && cols <= kQuantMaxCols, "rows must have 1 to 65536 columns to quantise");
    FGV_ASSERT(int8 || cols % kQuantGroup == 0, "float8_e4m3fn codes need a multiple of 128 columns");
    FGV_ASSERT(unit_rows(x), "x's rows must be contiguous");
    FGV_ASSERT(x.is_cuda(), "flaggems_vllm runs on the GPU (HIP) only");
    const int64_t rows = x.size(0);
    *codes = new_on(x.device(), {rows, cols}, int8 ? at::kChar : at::kFloat8_e4m3fn);
    *scales = new_on(x.device(), {rows, int8 ? 1 : cols / kQuantGroup}, at::kFloat);
    return 0;
}

using NormQuantOut = std::tuple<at::Tensor, at::Tensor, at::Tensor>;

int add_rms_norm_quant(const at::Tensor& x, const std::optional<at::Tensor>& residual, const at::Tensor& weight,
                       double eps, bool int8, const std::optional<at::Tensor>& hidden_out, NormQuantOut* out) {
    FGV_ASSERT(x.dim() == 2, "x must be 2D [num_tokens, size]");
    FGV_ASSERT(!takes_grad(x) && !takes_grad(weight) && !(residual && takes_grad(*residual)),
               "inference only: no input may require a gradient or carry a tangent");
    const int64_t rows = x.size(0), cols = x.size(1);
    FGV_ASSERT(weight.dim() == 1 && weight.size(0) == cols && weight.is_contiguous(),
               "weight must be [size] and contiguous");
    FGV_ASSERT(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat,
               "weight must have x's type or float32");
    FGV_ASSERT(eps > 0.0 && std::isfinite(eps), "eps must be positive and finite");
    FGV_ASSERT(residual || !hidden_out, "hidden_out needs a residual");
    if (const char* why = any_not_readable(x, residual, weight, hidden_out))
        return assert_failed(why);
    FGV_ASSERT(weight.device() == x.device(), "all tensors must be on x's device");
    if (residual) {
        FGV_ASSERT(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(),
                   "residual must have x's shape and type");
        FGV_ASSERT(unit_rows(*residual), "residual's rows must be contiguous");
        FGV_ASSERT(residual->device() == x.device(), "all tensors must be on x's device");
    }
    if (hidden_out) {
        const at::Tensor& h = *hidden_out;
        FGV_ASSERT(h.sizes() == x.sizes() && h.scalar_type() == x.scalar_type() && h.device() == x.device(),
                   "hidden_out must have x's shape, type and device");
        FGV_ASSERT(!takes_grad(h), "inference only: no output may require a gradient or carry a tangent");
        FGV_ASSERT(unit_rows(h) && (rows <= 1 || h.stride(0) >= cols),
                   "hidden_out's rows must be contiguous and apart");
        FGV_ASSERT(rows_apart_or_same(h, x) && rows_apart_or_same(h, *residual) && !spans_meet(h, weight),
                   "hidden_out must be x or residual itself, or apart from every input");
    }
    at::Tensor codes, scales;
    if (const int rc = quant_outputs(x, cols, int8, &codes, &scales))
        return rc;
    const at::Tensor hidden =
        hidden_out ? *hidden_out : residual ? new_on(x.device(), {rows, cols}, x.scalar_type()) : x;
    *out = NormQuantOut(codes, scales, hidden);
    const c10::DeviceGuard guard(x.device());
    return fgv_add_rms_norm_quant(x.data_ptr(), x.stride(0), residual ? residual->data_ptr() : nullptr,
                                  residual ? residual->stride(0) : 0, weight.data_ptr(),
                                  weight.scalar_type() == at::kFloat ? 1 : 0, residual ? hidden.data_ptr() : nullptr,
                                  residual ? hidden.stride(0) : 0, codes.data_ptr(), codes.stride(0),
                                  scales.data_ptr<float>(), scales.stride(0), rows, cols, eps,
                                  x.scalar_type() == at::kHalf ? 1 : 0, int8 ? 0 : 1, current_stream(x));
}

int silu_mul_quant(const at::Tensor& x, bool int8, TensorPair* out) {
    FGV_ASSERT(x.dim() == 2 && x.size(1) % 2 == 0, "x must be 2D [num_tokens, 2 * size], gate beside up");
    if (const char* why = not_readable(x))
        return assert_failed(why);
    FGV_ASSERT(!takes_grad(x), "inference only: no input may require a gradient or carry a tangent");
    const int64_t cols = x.size(1) / 2;
    at::Tensor codes, scales;
    if (const int rc = quant_outputs(x, cols, int8, &codes, &scales))
        return rc;
    *out = TensorPair(codes, scales);
    const c10::DeviceGuard guard(x.device());
    return fgv_silu_mul_quant(x.data_ptr(), x.stride(0), codes.data_ptr(), codes.stride(0), scales.data_ptr<float>(),
                              scales.stride(0), x.size(0), cols, x.scalar_type() == at::kHalf ? 1 : 0, int8 ? 0 : 1,
                              current_stream(x));
}

int out_code(at::ScalarType t) { return t == at::kBFloat16 ? 0 : t == at::kHalf ? 1 : t == at::kFloat ? 2 : -1; }

// The stride of n scales given as [n], [n, 1], [1, n] or one scale for all (0); -1: none of these.
int64_t scale_stride(const at::Tensor& s, int64_t n) {
    if (s.dim() > 2 || s.scalar_type() != at::kFloat)
        return -1;
    if (s.numel() == 1)
        return 0;
    if (s.numel() != n)
        return -1;
    if (s.dim() == 1)
        return s.stride(0);
    return s.size(0) == n ? s.stride(0) : s.size(1) == n ? s.stride(1) : -1;
}

int int8_mm(const at::Tensor& a, const at::Tensor& b, const at::Tensor& scale_a, const at::Tensor& scale_b,
            const std::optional<at::Tensor>& bias, at::ScalarType out_dtype, const std::optional<at::Tensor>& out_in,
            at::Tensor* result) {
    FGV_ASSERT(a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(1), "a must be [M, K] and b [N, K]");
    FGV_ASSERT(a.scalar_type() == at::kChar && b.scalar_type() == at::kChar, "a and b must be int8");
    const int64_t m = a.size(0), n = b.size(0), k = a.size(1);
    FGV_ASSERT(unit_rows(a) && unit_rows(b), "a's and b's rows must be contiguous");
    if (const char* why = any_not_readable(a, b, scale_a, scale_b, bias, out_in))
        return assert_failed(why);
    const int64_t sa = scale_stride(scale_a, m), sb = scale_stride(scale_b, n);
    FGV_ASSERT(sa >= 0 && (scale_a.numel() == 1 || scale_a.dim() == 1 || scale_a.size(0) == m),
               "scale_a must be float32: [M], [M, 1] or one scale");
    FGV_ASSERT(sb >= 0, "scale_b must be float32: [N], [N, 1], [1, N] or one scale");
    FGV_ASSERT(out_code(out_dtype) >= 0, "out_dtype must be bfloat16, float16 or float32");
    FGV_ASSERT(!takes_grad(scale_a) && !takes_grad(scale_b) && !(bias && takes_grad(*bias)),
               "inference only: no input may require a gradient or carry a tangent");
    const c10::Device dev = a.device();
    FGV_ASSERT(b.device() == dev && scale_a.device() == dev && scale_b.device() == dev &&
                   (!bias || bias->device() == dev) && (!out_in || out_in->device() == dev),
               "all tensors must be on a's device");
    if (bias) {
        FGV_ASSERT(bias->dim() == 1 && bias->size(0) == n && bias->is_contiguous(), "bias must be [N] and contiguous");
        FGV_ASSERT(bias->scalar_type() == at::kFloat || bias->scalar_type() == out_dtype,
                   "bias must be float32 or have the output's type");
    }
    if (out_in) {
        const at::Tensor& o = *out_in;
        FGV_ASSERT(o.dim() == 2 && o.size(0) == m && o.size(1) == n && o.scalar_type() == out_dtype,
                   "out must be [M, N] of out_dtype");
        FGV_ASSERT(!takes_grad(o), "inference only: no output may require a gradient or carry a tangent");
        FGV_ASSERT(unit_rows(o) && (m <= 1 || o.stride(0) >= n), "out's rows must be contiguous and apart");
        FGV_ASSERT(!spans_meet(o, a) && !spans_meet(o, b) && !spans_meet(o, scale_a) && !spans_meet(o, scale_b) &&
                       !(bias && spans_meet(o, *bias)),
                   "out must not overlap an input");
    }
    FGV_ASSERT(dev.is_cuda(), "flaggems_vllm runs on the GPU (HIP) only");
    const at::Tensor out = out_in ? *out_in : new_on(dev, {m, n}, out_dtype);
    *result = out;
    const c10::DeviceGuard guard(dev);
    // from torch's caching allocator, in the order of the current stream
    const int64_t ws_bytes = fgv_int8_scaled_mm_workspace_bytes(a.data_ptr<int8_t>(), a.stride(0),
                                                                b.data_ptr<int8_t>(), b.stride(0), m, n, k);
    const at::Tensor ws = ws_bytes > 0 ? new_on(dev, {ws_bytes}, at::kByte) : at::Tensor();
    return fgv_int8_scaled_mm(a.data_ptr<int8_t>(), a.stride(0), b.data_ptr<int8_t>(), b.stride(0),
                              scale_a.data_ptr<float>(), sa, scale_b.data_ptr<float>(), sb,
                              bias ? bias->data_ptr() : nullptr, bias ? out_code(bias->scalar_type()) : 0,
                              out.data_ptr(), out.stride(0), m, n, k, out_code(out_dtype),
                              ws.defined() ? ws.data_ptr() : nullptr, ws_bytes, current_stream(a));
}

// ---- serving from the 4-bit paged cache: block tables, insert, attention ----

bool is_i32_vector(const at::Tensor& t, int64_t n) {
    return t.dim() == 1 && t.size(0) == n && t.scalar_type() == at::kInt && (n <= 1 || t.stride(0) == 1);
}

using TablesOut = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

int build_block_tables(const at::Tensor& context_lens, const at::Tensor& query_lens, const at::Tensor& block_table,
                       const at::Tensor& free_blocks, const at::Tensor& num_free, int64_t block_size,
                       int64_t max_num_tokens, int64_t pad_id, TablesOut* out) {
    FGV_ASSERT(context_lens.dim() == 1, "context_lens must be 1-D");
    const int64_t reqs = context_lens.size(0);
    FGV_ASSERT(is_i32_vector(context_lens, reqs) && is_i32_vector(query_lens, reqs),
               "context_lens and query_lens must be contiguous int32 [num_reqs]");
    FGV_ASSERT(block_table.dim() == 2 && block_table.size(0) == reqs && block_table.scalar_type() == at::kInt,
               "block_table must be int32 [num_reqs, max blocks]");
    FGV_ASSERT(unit_rows(block_table) && (reqs <= 1 || block_table.stride(0) >= block_table.size(1)),
               "block_table's rows must be contiguous and apart");
    FGV_ASSERT(free_blocks.dim() == 1 && is_i32_vector(free_blocks, free_blocks.size(0)),
               "free_blocks must be contiguous 1-D int32");
    FGV_ASSERT(num_free.numel() == 1 && num_free.scalar_type() == at::kInt, "num_free must be one int32");
    FGV_ASSERT(block_size > 0, "block_size must be positive");
    FGV_ASSERT(max_num_tokens >= 0, "max_num_tokens must not be negative");
    if (const char* why = any_not_readable(context_lens, query_lens, block_table, free_blocks, num_free))
        return assert_failed(why);
    FGV_ASSERT(!spans_meet(block_table, context_lens) && !spans_meet(block_table, query_lens) &&
                   !spans_meet(block_table, free_blocks) && !spans_meet(block_table, num_free),
               "block_table must not overlap an input");
    const c10::Device dev = block_table.device();
    FGV_ASSERT(dev.is_cuda(), "flaggems_vllm runs on the GPU (HIP) only");
    FGV_ASSERT(context_lens.device() == dev && query_lens.device() == dev && free_blocks.device() == dev &&
                   num_free.device() == dev,
               "all tensors must be on block_table's device");
    const c10::DeviceGuard guard(dev);
    const at::Tensor qsl = new_on(dev, {reqs + 1}, at::kInt), lens = new_on(dev, {reqs}, at::kInt);
    const at::Tensor positions = new_on(dev, {max_num_tokens}, at::kLong);
    const at::Tensor slots = new_on(dev, {max_num_tokens}, at::kLong), left = new_on(dev, {1}, at::kInt);
    *out = TablesOut(qsl, lens, positions, slots, left);
    return fgv_build_block_tables(i32_ptr(context_lens), i32_ptr(query_lens), reqs, i32_ptr(block_table),
                                  block_table.stride(0), block_table.size(1), i32_ptr(free_blocks), free_blocks.size(0),
                                  i32_ptr(num_free), block_size, max_num_tokens, pad_id, i32_ptr(qsl), i32_ptr(lens),
                                  positions.data_ptr<int64_t>(), slots.data_ptr<int64_t>(), i32_ptr(left),
                                  current_stream(block_table));
}

// The head dim of an MXFP4 cache [blocks, kv heads, block size, D + D / 16]; 0: it is none.
int64_t mx_head_dim(const at::Tensor& cache) {
    if (cache.dim() != 4 || cache.scalar_type() != at::kByte)
        return 0;
    const int64_t width = cache.size(3);
    return width == 68 ? 64 : width == 136 ? 128 : width == 272 ? 256 : 0;
}

constexpr const char* kMxCache =
    "kv_cache must be uint8 [num_blocks, num_kv_heads, block_size, D + D / 16], D 64, 128 or 256";

int mxfp4_insert(const at::Tensor& k, const at::Tensor& v, const at::Tensor& cache, const at::Tensor& slots) {
    const int64_t dim = mx_head_dim(cache);
    FGV_ASSERT(dim > 0, kMxCache);
    FGV_ASSERT(blocks_contiguous(cache), "each kv_cache block must be contiguous bytes");
    FGV_ASSERT(cache.size(2) > 0 && cache.size(2) % 16 == 0 && cache.size(2) <= 4096,
               "block_size must be a multiple of 16 of at most 4096");
    FGV_ASSERT(k.dim() == 3 && v.sizes() == k.sizes() && k.size(1) == cache.size(1) && k.size(2) == dim,
               "k and v must be [num_tokens, num_kv_heads, D]");
    FGV_ASSERT((k.scalar_type() == at::kBFloat16 || k.scalar_type() == at::kHalf) && v.scalar_type() == k.scalar_type(),
               "k and v must both be bfloat16 or float16");
    FGV_ASSERT(k.stride(2) == 1 && v.stride(2) == 1, "k's and v's rows must be contiguous");
    FGV_ASSERT(slots.dim() == 1 && slots.scalar_type() == at::kLong && (slots.size(0) <= 1 || slots.stride(0) == 1),
               "slot_mapping must be contiguous 1-D int64");
    FGV_ASSERT(slots.size(0) <= k.size(0), "slot_mapping is longer than the number of tokens");
    FGV_ASSERT(!takes_grad(k) && !takes_grad(v), "inference only: no input may require a gradient or carry a tangent");
    if (const char* why = any_not_readable(k, v, cache, slots))
        return assert_failed(why);
    FGV_ASSERT(!spans_meet(cache, k) && !spans_meet(cache, v) && !spans_meet(cache, slots),
               "kv_cache must not overlap an input");
    const c10::Device dev = cache.device();
    FGV_ASSERT(dev.is_cuda(), "flaggems_vllm runs on the GPU (HIP) only");
    FGV_ASSERT(k.device() == dev && v.device() == dev && slots.device() == dev,
               "all tensors must be on kv_cache's device");
    const c10::DeviceGuard guard(dev);
    return fgv_mxfp4_kv_quant_and_cache(k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                                        k.scalar_type() == at::kHalf ? 1 : 0, slots.size(0), k.size(1), dim,
                                        cache.data_ptr<uint8_t>(), cache.stride(0), cache.size(0), cache.size(2),
                                        slots.data_ptr<int64_t>(), current_stream(cache));
}

int mxfp4_attention(const at::Tensor& q, const at::Tensor& cache, const at::Tensor& block_table,
                    const at::Tensor& seq_lens, double scale, const std::optional<at::Tensor>& query_start_loc,
                    std::optional<int64_t> max_query_len, std::optional<int64_t> max_seq_len,
                    std::optional<int64_t> window, const std::optional<at::Tensor>& sink,
                    const std::optional<at::Tensor>& out_in, TensorPair* result) {
    const int64_t dim = mx_head_dim(cache);
    FGV_ASSERT(dim > 0, kMxCache);
    FGV_ASSERT(blocks_contiguous(cache), "each kv_cache block must be contiguous bytes");
    const int64_t page = cache.size(2), kv_heads = cache.size(1);
    FGV_ASSERT(page > 0 && page % 16 == 0 && page <= 4096, "block_size must be a multiple of 16 of at most 4096");
    FGV_ASSERT(q.dim() == 3 && q.size(2) == dim, "q must be [num_tokens, num_heads, D]");
    FGV_ASSERT(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, "q must be bfloat16 or float16");
    FGV_ASSERT(q.stride(2) == 1, "q's rows must be contiguous");
    const int64_t tokens = q.size(0), heads = q.size(1);
    FGV_ASSERT(kv_heads > 0 && heads % kv_heads == 0, "num_heads must be a multiple of num_kv_heads");
    FGV_ASSERT(seq_lens.dim() == 1, "seq_lens must be 1-D");
    const int64_t reqs = seq_lens.size(0);
    FGV_ASSERT(is_i32_vector(seq_lens, reqs), "seq_lens must be contiguous int32 [num_reqs]");
    FGV_ASSERT(block_table.dim() == 2 && block_table.size(0) == reqs && block_table.scalar_type() == at::kInt,
               "block_table must be int32 [num_reqs, max blocks]");
    FGV_ASSERT(unit_rows(block_table), "block_table's rows must be contiguous");
    if (query_start_loc)
        FGV_ASSERT(is_i32_vector(*query_start_loc, reqs + 1), "query_start_loc must be contiguous int32 [num_reqs + 1]");
    else
        FGV_ASSERT(tokens == reqs, "without query_start_loc there is one token per request");
    FGV_ASSERT(std::isfinite(scale) && std::fabs(scale) <= 1e30, "softmax_scale must be finite");
    FGV_ASSERT(!window || *window >= 1, "window_size must be at least 1");
    FGV_ASSERT((!max_query_len || *max_query_len >= 0) && (!max_seq_len || *max_seq_len >= 0),
               "max_query_len and max_seq_len must not be negative");
    if (sink)
        FGV_ASSERT(sink->dim() == 1 && sink->size(0) == heads && sink->scalar_type() == at::kFloat &&
                       (heads <= 1 || sink->stride(0) == 1),
                   "attn_sink must be contiguous float32 [num_heads]");
    FGV_ASSERT(!takes_grad(q) && !(sink && takes_grad(*sink)),
               "inference only: no input may require a gradient or carry a tangent");
    if (const char* why = any_not_readable(q, cache, block_table, seq_lens, query_start_loc, sink, out_in))
        return assert_failed(why);
    const c10::Device dev = q.device();
    FGV_ASSERT(cache.device() == dev && block_table.device() == dev && seq_lens.device() == dev &&
                   (!query_start_loc || query_start_loc->device() == dev) && (!sink || sink->device() == dev) &&
                   (!out_in || out_in->device() == dev),
               "all tensors must be on q's device");
    if (out_in) {
        const at::Tensor& o = *out_in;
        FGV_ASSERT(o.sizes() == q.sizes() && o.scalar_type() == q.scalar_type(), "out must have q's shape and type");
        FGV_ASSERT(!takes_grad(o), "inference only: no output may require a gradient or carry a tangent");
        FGV_ASSERT(o.stride(2) == 1 && (heads <= 1 || o.stride(1) >= dim) &&
                       (tokens <= 1 || o.stride(0) >= (heads - 1) * o.stride(1) + dim),
                   "out's rows must be contiguous and apart, heads within tokens");
        FGV_ASSERT(!spans_meet(o, q) && !spans_meet(o, cache) && !spans_meet(o, block_table) &&
                       !spans_meet(o, seq_lens) && !(query_start_loc && spans_meet(o, *query_start_loc)) &&
                       !(sink && spans_meet(o, *sink)),
                   "out must not overlap an input");
    }
    FGV_ASSERT(dev.is_cuda(), "flaggems_vllm runs on the GPU (HIP) only");
    const c10::DeviceGuard guard(dev);
    const at::Tensor out = out_in ? *out_in : new_on(dev, {tokens, heads, dim}, q.scalar_type());
    const at::Tensor lse = new_on(dev, {tokens, heads}, at::kFloat);
    *result = TensorPair(out, lse);
    const int64_t most_q = max_query_len ? *max_query_len : query_start_loc ? tokens : 1;
    const int64_t most_s = max_seq_len ? *max_seq_len : block_table.size(1) * page;
    // from torch's caching allocator, in the order of the current stream
    const int64_t ws_bytes =
        fgv_mxfp4_paged_attention_workspace_bytes(tokens, heads, kv_heads, dim, reqs, most_q, most_s);
    const at::Tensor ws = ws_bytes > 0 ? new_on(dev, {ws_bytes}, at::kByte) : at::Tensor();
    return fgv_mxfp4_paged_attention(
        q.data_ptr(), q.stride(0), q.stride(1), q.scalar_type() == at::kHalf ? 1 : 0, tokens, heads, kv_heads, dim,
        cache.data_ptr<uint8_t>(), cache.stride(0), cache.size(0), page, i32_ptr(block_table), block_table.stride(0),
        block_table.size(1), i32_ptr(seq_lens), query_start_loc ? i32_ptr(*query_start_loc) : nullptr, reqs, most_q,
        most_s, scale, window ? *window : 0, sink ? sink->data_ptr<float>() : nullptr, out.data_ptr(), out.stride(0),
        out.stride(1), lse.data_ptr<float>(), lse.stride(0), ws.defined() ? ws.data_ptr() : nullptr, ws_bytes,
        current_stream(q));
}

// ---- dispatcher ops: the same functions, failures raised as RuntimeError ----

void raise_on_status(int rc, const char* op) {
    if (rc == 0)
        return;
    if (rc == kAssertFailed)
        TORCH_CHECK(false, op, ": ", g_assert_message);
    if (rc < 0)
        TORCH_CHECK(false, op, ": ", fgv_last_error(), " (code ", rc, ")");
    TORCH_CHECK(false, op, ": HIP launch failed with hipError_t ", rc);
}

void qnorm_rope_kv_insert_op(at::Tensor& q, const at::Tensor& kv, at::Tensor& k_cache,
                             const at::Tensor& slot_mapping, const at::Tensor& position_ids,
                             const at::Tensor& cos_sin_cache, double eps, int64_t cache_block_size) {
    raise_on_status(qnorm_rope_kv_insert(q, kv, k_cache, slot_mapping, position_ids, cos_sin_cache, eps,
                                         cache_block_size),
                    "fused_deepseek_v4_qnorm_rope_kv_rope_quant_insert");
}

SiblingOut inv_rope_fp8_quant_op(const at::Tensor& o, const at::Tensor& positions, const at::Tensor& cos_sin_cache,
                                 int64_t n_groups, int64_t heads_per_group, int64_t nope_dim, int64_t rope_dim,
                                 int64_t quant_group_size, double eps, bool tma_aligned_scales) {
    SiblingOut out;
    raise_on_status(inv_rope_fp8_quant(o, positions, cos_sin_cache, n_groups, heads_per_group, nope_dim, rope_dim,
                                       quant_group_size, eps, true, tma_aligned_scales, &out),
                    "fused_inv_rope_fp8_quant");
    return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(flaggems_vllm, m) {
    // positional order of vLLM's torch.ops._C op of the same name
    m.def("fused_deepseek_v4_qnorm_rope_kv_rope_quant_insert(Tensor(a0!) q, Tensor kv, Tensor(a2!) k_cache, "
          "Tensor slot_mapping, Tensor position_ids, Tensor cos_sin_cache, float eps, int cache_block_size) -> ()");
    m.def("fused_inv_rope_fp8_quant(Tensor o, Tensor positions, Tensor cos_sin_cache, int n_groups, "
          "int heads_per_group, int nope_dim=448, int rope_dim=64, int quant_group_size=128, float eps=1e-10, "
          "bool tma_aligned_scales=False) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(flaggems_vllm, CUDA, m) {
    m.impl("fused_deepseek_v4_qnorm_rope_kv_rope_quant_insert", &qnorm_rope_kv_insert_op);
    m.impl("fused_inv_rope_fp8_quant", &inv_rope_fp8_quant_op);
}

PYBIND11_MODULE(_fgv_torch, m) {
    m.doc() = "C++ checks and launches of fused_deepseek_v4_qnorm_rope_kv_rope_quant_insert, "
              "fused_inv_rope_fp8_quant, the five ops beside them, the 8-bit linear ops and those of the 4-bit "
              "paged cache (status-returning; the "
              "Python wrappers map the status)";
    m.attr("ASSERT_FAILED") = kAssertFailed;
    m.def("qnorm_rope_kv_insert", &qnorm_rope_kv_insert);
    m.def("inv_rope_fp8_quant",
          [](const at::Tensor& o, const at::Tensor& positions, const at::Tensor& cos_sin_cache, int64_t n_groups,
             int64_t heads_per_group, int64_t nope_dim, int64_t rope_dim, int64_t quant_group_size, double eps,
             bool fp8_e4m3fn, bool tma_aligned_scales) {
              SiblingOut out;
              const int rc = inv_rope_fp8_quant(o, positions, cos_sin_cache, n_groups, heads_per_group, nope_dim,
                                                rope_dim, quant_group_size, eps, fp8_e4m3fn, tma_aligned_scales,
                                                &out);
              return std::make_tuple(rc, std::get<0>(out), std::get<1>(out));
          });
    m.def("q_kv_rmsnorm",
          [](const at::Tensor& qr, const at::Tensor& kv, const at::Tensor& q_weight, const at::Tensor& kv_weight,
             double eps) {
              TensorPair out;
              const int rc = q_kv_rmsnorm(qr, kv, q_weight, kv_weight, eps, &out);
              return std::make_tuple(rc, std::get<0>(out), std::get<1>(out));
          });
    m.def("dequantize_gather", &dequantize_gather);
    m.def("indexer_q_rope_quant",
          [](const at::Tensor& positions, const at::Tensor& index_q, const at::Tensor& cos_sin,
             const at::Tensor& weights, double softmax_scale, double head_scale, bool use_fp4) {
              IndexerOut out;
              const int rc = indexer_q_rope_quant(positions, index_q, cos_sin, weights, softmax_scale, head_scale,
                                                  use_fp4, &out);
              return std::make_tuple(rc, std::get<0>(out), std::get<1>(out), std::get<2>(out));
          });
    m.def("slot_mapping", &slot_mapping);
    m.def("indexer_k_quant", &indexer_k_quant);
    m.def("add_rms_norm_quant",
          [](const at::Tensor& x, const std::optional<at::Tensor>& residual, const at::Tensor& weight, double eps,
             bool int8, const std::optional<at::Tensor>& hidden_out) {
              NormQuantOut out;
              const int rc = add_rms_norm_quant(x, residual, weight, eps, int8, hidden_out, &out);
              return std::make_tuple(rc, std::get<0>(out), std::get<1>(out), std::get<2>(out));
          });
    m.def("silu_mul_quant", [](const at::Tensor& x, bool int8) {
        TensorPair out;
        const int rc = silu_mul_quant(x, int8, &out);
        return std::make_tuple(rc, std::get<0>(out), std::get<1>(out));
    });
    m.def("int8_mm", [](const at::Tensor& a, const at::Tensor& b, const at::Tensor& scale_a, const at::Tensor& scale_b,
                        const std::optional<at::Tensor>& bias, at::ScalarType out_dtype,
                        const std::optional<at::Tensor>& out_in) {
        at::Tensor out;
        const int rc = int8_mm(a, b, scale_a, scale_b, bias, out_dtype, out_in, &out);
        return std::make_tuple(rc, out);
    });
    m.def("build_block_tables",
          [](const at::Tensor& context_lens, const at::Tensor& query_lens, const at::Tensor& block_table,
             const at::Tensor& free_blocks, const at::Tensor& num_free, int64_t block_size, int64_t max_num_tokens,
             int64_t pad_id) {
              TablesOut out;
              const int rc = build_block_tables(context_lens, query_lens, block_table, free_blocks, num_free,
                                                block_size, max_num_tokens, pad_id, &out);
              return std::make_tuple(rc, out);
          });
    m.def("mxfp4_insert", &mxfp4_insert);
    m.def("mxfp4_attention",
          [](const at::Tensor& q, const at::Tensor& cache, const at::Tensor& block_table, const at::Tensor& seq_lens,
             double scale, const std::optional<at::Tensor>& query_start_loc, std::optional<int64_t> max_query_len,
             std::optional<int64_t> max_seq_len, std::optional<int64_t> window, const std::optional<at::Tensor>& sink,
             const std::optional<at::Tensor>& out_in) {
              TensorPair out;
              const int rc = mxfp4_attention(q, cache, block_table, seq_lens, scale, query_start_loc, max_query_len,
                                             max_seq_len, window, sink, out_in, &out);
              return std::make_tuple(rc, std::get<0>(out), std::get<1>(out));
          });
    m.def("assert_message", []() { return g_assert_message; });
}
