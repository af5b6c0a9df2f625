// gfx950 kernel that turns a step's request lengths into what the paged-cache
// ops read: block tables (new blocks taken off a stack of free ones),
// query_start_loc, sequence lengths, positions and cache slots.
//
// With page tokens to a block and W table columns, request b brings query_b
// new tokens behind its ctx_b cached ones:
//   start_b = min(sum_{b' < b} query_b', max_tokens), q_b = start_{b+1} - start_b
//   held_b  = min(ceil(ctx_b / page), W)
//   all_b   = min(ceil((ctx_b + q_b) / page), W)
//   its new columns held_b .. all_b - 1 get the blocks free[num_free - 1 - n],
//   n counted over the requests in order, and -1 once the stack is empty;
//   token i: pos = ctx_b + i, slot = table[b, pos / page] * page + pos % page.
//
// One launch, and no workgroup waits for another: each scans the lengths for
// itself (they stay in the cache: 512 requests are 4 KB) and keeps in LDS the
// requests that its 256 tokens fall into, at most 256 that are not empty.
// Each new block has exactly one token at its first place, since new columns
// begin at or behind the context's end: the thread of that token takes the
// block off the stack and enters it.  The other tokens of a new block work out
// the same id from the stack, so nothing that is written here is read here.
// Workgroup 0 writes what there is per request.  A call is bound by its latency:
// launch, one read of the lengths, two scans, one read of the stack or the table.
#include "fgv_device.h"
#include "fgv_host.h"

namespace fgv {
namespace {

constexpr int kTbThreads = 256;   // tokens per workgroup, one a thread
constexpr int kTbPer = 4;         // consecutive requests a thread scans at a time
constexpr int kTbWaves = kTbThreads / 64;
constexpr int kTbSlots = 2 * kTbThreads;  // LDS places: the requests of 256 tokens have consecutive ranks

struct TablesArgs {
    const int32_t* context_lens;
    const int32_t* query_lens;
    int32_t* block_table;
    int64_t bt_stride;
    const int32_t* free_blocks;
    const int32_t* num_free;
    int32_t* query_start_loc;
    int32_t* seq_lens;
    int64_t* positions;
    int64_t* slot_mapping;
    int32_t* num_free_out;
    int64_t pad_id;
    int32_t num_reqs, width, stack_size, page, max_tokens;
};

// Exclusive prefix sum over the workgroup's threads; total gets the sum.  `part`
// holds a value per wave and is free again after the caller's next barrier.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t (&part)[kTbWaves], int64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t o = __shfl_up(s, d);
        if (lane >= d)
            s += o;
    }
    if (lane == 63)
        part[wave] = s;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kTbWaves; ++w) {
        before += w < wave ? part[w] : 0;
        total += part[w];
    }
    return before + s - v;
}

__device__ __forceinline__ int32_t blocks_of(int32_t tokens, int32_t page, int32_t width) {
    const int32_t n = tokens / page + (tokens % page != 0);
    return n < width ? n : width;
}

__global__ void __launch_bounds__(kTbThreads) block_tables_kernel(TablesArgs a) {
    __shared__ int64_t part_q[kTbWaves], part_n[kTbWaves];
    __shared__ int32_t s_start[kTbSlots], s_req[kTbSlots], s_ctx[kTbSlots], s_held[kTbSlots];
    __shared__ int64_t s_nth[kTbSlots];
    __shared__ int32_t s_first, s_count;
    const int32_t t0 = (int32_t)blockIdx.x * kTbThreads;
    const int32_t t1 = min(t0 + kTbThreads, a.max_tokens);  // max_tokens fits
    const int64_t most = a.max_tokens;
    if (threadIdx.x == 0) {
        s_first = 0;
        s_count = 0;
    }
    int64_t tokens = 0, blocks = 0;  // of the requests before this turn's
    int32_t ranks = 0;               // of those with tokens
    for (int32_t base = 0; base < a.num_reqs; base += kTbThreads * kTbPer) {
        int32_t ctx[kTbPer], start[kTbPer], q[kTbPer], held[kTbPer], all[kTbPer];
        const int32_t b0 = base + (int32_t)threadIdx.x * kTbPer;
        int64_t sum = 0;
#pragma unroll
        for (int i = 0; i < kTbPer; ++i) {
            const bool in = b0 + i < a.num_reqs;
            ctx[i] = in ? max(a.context_lens[b0 + i], 0) : 0;
            q[i] = in ? max(a.query_lens[b0 + i], 0) : 0;
            sum += q[i];
        }
        int64_t all_q, all_n, at = tokens + block_scan(sum, part_q, all_q);
        int64_t packed = 0;  // new blocks, and in the upper half requests with tokens
#pragma unroll
        for (int i = 0; i < kTbPer; ++i) {
            start[i] = (int32_t)min(at, most);
            at += q[i];
            q[i] = (int32_t)min(at, most) - start[i];
            const int32_t end = (int32_t)min((int64_t)ctx[i] + q[i], (int64_t)0x7fffffff);  // lengths end there
            held[i] = blocks_of(ctx[i], a.page, a.width);
            all[i] = blocks_of(end, a.page, a.width);
            packed += all[i] - held[i] + ((int64_t)(q[i] > 0) << 40);
            if (blockIdx.x == 0 && b0 + i < a.num_reqs) {
                a.query_start_loc[b0 + i] = start[i];
                a.seq_lens[b0 + i] = end;
            }
        }
        const int64_t before = block_scan(packed, part_n, all_n);
        int64_t nth = blocks + (before & ((1LL << 40) - 1));
        int32_t rank = ranks + (int32_t)(before >> 40);
#pragma unroll
        for (int i = 0; i < kTbPer; ++i) {
            if (q[i] > 0 && start[i] < t1 && start[i] + q[i] > t0) {
                const int32_t at_slot = rank & (kTbSlots - 1);
                s_start[at_slot] = start[i];
                s_req[at_slot] = b0 + i;
                s_ctx[at_slot] = ctx[i];
                s_held[at_slot] = held[i];
                s_nth[at_slot] = nth;
                if (start[i] <= t0)
                    s_first = rank;
                atomicAdd(&s_count, 1);
            }
            rank += q[i] > 0;
            nth += all[i] - held[i];
        }
        tokens += all_q;
        blocks += all_n & ((1LL << 40) - 1);
        ranks += (int32_t)(all_n >> 40);
        // every workgroup but the first may stop behind its last token
        if (blockIdx.x != 0 && tokens >= t1)
            break;
    }
    __syncthreads();
    const int32_t avail = min(max(*a.num_free, 0), a.stack_size);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.query_start_loc[a.num_reqs] = (int32_t)min(tokens, most);
        const int64_t left = (int64_t)avail - blocks;
        *a.num_free_out = (int32_t)max(left, (int64_t)-0x7fffffff);
    }
    const int32_t t = t0 + (int32_t)threadIdx.x;
    if (t >= t1)
        return;
    if (t >= tokens) {  // tokens up to t1 were counted
        a.positions[t] = 0;
        a.slot_mapping[t] = a.pad_id;
        return;
    }
    // the last of the kept requests that starts at or before t
    int32_t lo = 0, hi = s_count - 1;
    while (lo < hi) {
        const int32_t mid = (lo + hi + 1) >> 1;
        if (s_start[(s_first + mid) & (kTbSlots - 1)] <= t)
            lo = mid;
        else
            hi = mid - 1;
    }
    const int32_t e = (s_first + lo) & (kTbSlots - 1);
    const int64_t pos = (int64_t)s_ctx[e] + (t - s_start[e]);
    a.positions[t] = pos;
    const int64_t column = pos / a.page;
    const int32_t place = (int32_t)(pos - column * a.page);
    int64_t slot = a.pad_id;
    if (column < a.width) {
        int32_t* entry = a.block_table + (int64_t)s_req[e] * a.bt_stride + column;
        int32_t block;
        if (column < s_held[e]) {
            block = *entry;
        } else {
            const int64_t n = s_nth[e] + (column - s_held[e]);
            block = n < avail ? a.free_blocks[avail - 1 - n] : -1;
            if (place == 0)
                *entry = block;
        }
        if (block >= 0)
            slot = (int64_t)block * a.page + place;
    }
    a.slot_mapping[t] = slot;
}

}  // namespace
}  // namespace fgv

extern "C" int fgv_build_block_tables(const int32_t* context_lens, const int32_t* query_lens, int64_t num_reqs,
                                      int32_t* block_table, int64_t block_table_stride, int64_t max_blocks_per_req,
                                      const int32_t* free_blocks, int64_t free_blocks_size, const int32_t* num_free,
                                      int64_t block_size, int64_t max_num_tokens, int64_t pad_id,
                                      int32_t* query_start_loc, int32_t* seq_lens, int64_t* positions,
                                      int64_t* slot_mapping, int32_t* num_free_out, void* stream) {
    using namespace fgv;
    if (num_reqs < 0 || max_num_tokens < 0 || max_blocks_per_req < 0 || free_blocks_size < 0)
        return fail(FGV_E_BAD_SHAPE, "negative size");
    if (num_reqs > 0x3fffffffLL || max_num_tokens > 0x3fffffffLL || max_blocks_per_req > 0x7fffffffLL ||
        free_blocks_size > 0x7fffffffLL)
        return fail(FGV_E_TOO_LARGE, "at most 2^30 - 1 requests and tokens, 2^31 - 1 table columns and free blocks");
    if (block_size <= 0 || block_size > 0x7fffffffLL)
        return fail(FGV_E_BAD_SHAPE, "block_size must be positive and fit in int32");
    if (!num_free || !query_start_loc || !num_free_out ||
        (num_reqs > 0 && (!context_lens || !query_lens || !seq_lens || (max_blocks_per_req > 0 && !block_table))) ||
        (max_num_tokens > 0 && (!positions || !slot_mapping)) || (free_blocks_size > 0 && !free_blocks))
        return fail(FGV_E_NULL_POINTER, "null pointer argument");
    if (num_reqs > 1 && block_table_stride < max_blocks_per_req)
        return fail(FGV_E_BAD_STRIDE, "block_table rows must not overlap");
    if (!aligned(positions, 8) || !aligned(slot_mapping, 8))
        return fail(FGV_E_MISALIGNED, "positions and slot_mapping must be 8-byte aligned");
    TablesArgs a;
    a.context_lens = context_lens;
    a.query_lens = query_lens;
    a.block_table = block_table;
    a.bt_stride = block_table_stride;
    a.free_blocks = free_blocks;
    a.num_free = num_free;
    a.query_start_loc = query_start_loc;
    a.seq_lens = seq_lens;
    a.positions = positions;
    a.slot_mapping = slot_mapping;
    a.num_free_out = num_free_out;
    a.pad_id = pad_id;
    a.num_reqs = (int32_t)num_reqs;
    a.width = (int32_t)max_blocks_per_req;
    a.stack_size = (int32_t)free_blocks_size;
    a.page = (int32_t)block_size;
    a.max_tokens = (int32_t)max_num_tokens;
    const unsigned grid = (unsigned)((max_num_tokens + kTbThreads - 1) / kTbThreads);
    hipLaunchKernelGGL(block_tables_kernel, dim3(grid ? grid : 1), dim3(kTbThreads), 0,
                       static_cast<hipStream_t>(stream), a);
    return launch_status();
}
