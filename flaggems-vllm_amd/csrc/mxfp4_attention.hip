// gfx950 kernels for attention over the paged MXFP4 key/value cache
// (layout: mxfp4_cache.h).
//
// Query token i of request b (query_start_loc[b] <= i < query_start_loc[b+1],
// or i = b with one token each) stands at position
//   pos = seq_lens[b] - (tokens of b) + (i - query_start_loc[b])
// and sees the keys j with pos - window < j <= pos.  Query head h reads the
// key/value head h / G, G = Hq / Hkv:
//   s_j = scale * q . k_j,  lse = ln sum_j exp(s_j),
//   out = sum_j exp(s_j) v_j / (sum_j exp(s_j) + exp(sink_h)).
// A token that sees nothing gets out 0 and lse +inf.
//
// The rows of a tile are (token, head of the group) pairs of one key/value
// head, so that a key is read once for all of them.  Everything runs
// transposed, S^T = K q^T and O^T = V^T P^T: a lane then holds one query row,
// whose maximum and sum are a scalar in it, and S^T's accumulator layout is the
// second operand's of PV without a move between lanes.
//
// QK: the matrix instruction reads the cache's own format.  K's codes go from
// memory into the A registers of v_mfma_scale_f32_16x16x128_f8f6f4, the UE8M0
// bytes are its scales, and nothing is dequantised.  The query is the B
// operand in e4m3: divided by a power of two per row that puts the row's
// maximum into [128, 256), its 8 (bf16) or 11 (fp16) bits split into 2 or 3
// e4m3 pieces of 4, each under a scale 2^-4 smaller.  Values near their row's
// maximum are held whole; what values far below it lose is under 2^-16 (2^-20) of
// that maximum.  With the products that the instruction cuts (take_piece) that
// leaves scores of normal queries and keys an error of 1e-6 to 5e-6 rms (fp16: 1e-7 to
// 4e-7; D = 256 to 64), which lse carries: up to 2.2e-4 of 5 to 8 in 128 windows of
// 1000 keys, heads of 64; 3e-5 in 64 requests, heads of 128.  Register
// images (measured; the tests pin them through the results): lane (r, g) =
// (l % 16, l / 16) holds of A k = 32g..32g+31 of key r, of B k = 16g..16g+15
// and 64+16g..64+16g+15 of row r; scales apply to k = 32g..32g+31; D holds
// keys 4g..4g+3 of row r.
//
// PV: v_cvt_scalef32_pk_bf16_fp4 gives V in bf16 exactly (codes have two
// bits), token by token; LDS turns it, written by tokens and read by
// ds_read_b64_tr_b16.  P goes in as two bf16 pieces (16 bits): one alone would
// put its own 2^-9 beside the output's.  A value block under byte 255 (NaN) makes
// the outputs of those rows NaN that see it, and so do 253 and 254, whose values
// bf16 does not hold (their infinities would make any row NaN in whose tile they lie).
//
// Two kernels: 16-row tiles, whose waves share out the keys (here; single tokens,
// a few of them, and D = 256), and 128-row tiles, whose waves share out the rows
// (mxfp4_attend_wide.h).  Single tokens are bound by the cache's bytes, once there
// are many: 64 requests of up to 8191 keys, 199 MB, 51 us, of it 4 to 5 for joining
// cuts; 1 x 131072 keys, 143 MB, 38.4 us, of it 5 to 6.  In front of the bytes stand some 6 us
// of latency (1 x 16 keys takes 6.2 us in all, 64 requests of 16 keys, with the plan,
// 7.9): launch, lengths, block table and first keys each wait for the one before.
#include <math.h>

#include "fgv_device.h"
#include "fgv_host.h"
#include "mxfp4_cache.h"

namespace fgv {
namespace {

typedef int v8i_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) short4_t lds_short4_t;

constexpr int kAttThreads = 256;
constexpr int kAttWaves = kAttThreads / 64;
constexpr int kTileKeys = 64;  // keys of every tile begin at a multiple of this
constexpr int kRows = 16;      // query rows of a workgroup
constexpr int kMostWorkers = 1024;  // per head
// Work is dealt out in units, a turn of the workgroup's waves over 128 keys, about 1 us.
// Beginning and ending a tile (block table, query, joining the waves) costs as
// much as this many more, so that a worker of many short tiles gets fewer units.
constexpr int kTileCost = 4;
constexpr int kLeastCost = kTileCost + 1;  // what a worker takes at least
// Tiles of no more units than this are not cut: joining cuts takes a launch, 4 us.  Cut and whole, D = 128, 4 query heads
// to a key head: 8 tiles of 8 units 14.0 and 11.9 us, of 10 14.0 and 13.7, of 12 14.0 and 15.4; 64 tiles of 10 14.8 and
// 15.0, of 12 14.9 and 16.7; 512 tiles of 10 23.4 and 21.2, of 16 35.3 and 32.9.  D = 64: 8 tiles of 10 13.1 and 12.3, of 12
// 13.2 and 14.1.  D = 256: 8 tiles of 8 20.5 and 19.5, of 10 20.5 and 22.0; 128 tiles of 10 25.9 and 23.1.  128 windows of
// 1000 keys, 1024 tiles of 9, D = 64: 30.4 and 27.8.  (Few tiles of D = 256 would be cut from 9 units on, many of any D later.)
constexpr int kWholeUnits = 10;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// A row's reference is raised when a score exceeds it, and then to this much
// above the score (base 2), so that most tiles rescale nothing.  P is at most 1.
constexpr float kAhead = 4.0f;
// The last scale byte of values: above it they are NaN.
constexpr uint32_t kMostByte = 252;
// Sums of P v over 2^30 keys stay finite with P at most 1 for values under bytes up to kLargeByte
// (6 * 2^89).  Once a wave meets larger ones, up to 6 * 2^125, P and its sums are taken under a
// reference that is large_margin higher: by as many binades as a sum over the `keys` that a row
// may see could pass 6 * 2^125 by.  (Nothing is P below 2^-126: 2^-122 of the row's largest, and so much more there.)
constexpr uint32_t kLargeByte = 216;
__device__ __forceinline__ float large_margin(int32_t keys, uint32_t byte) {
    return (float)max(32 - __builtin_clz((uint32_t)keys | 1u) + (int)byte - (int)kMostByte, 0);
}
// The wave's largest byte, some being past kLargeByte (step by step: such tiles are rare, and what
// moves between lanes would take registers in all of them).
__device__ __forceinline__ uint32_t wave_largest(uint32_t v) {
    uint32_t most = kMostByte;
    while (most > kLargeByte && !__any(v >= most))
        --most;
    return most;
}
// References farther from 0 are rounded by more than the one below which a score that is not
// rounded may lie: there both are.
constexpr float kFar = 1 << 20;

// 16-key subtiles that a wave takes at a time: two such tiles have to fit its registers.
__host__ __device__ constexpr int key_subtiles(int) { return 2; }
// Workgroups that a CU holds at a time.
__host__ __device__ constexpr int groups_per_cu(int dim) { return dim == 64 ? 3 : 2; }
// Keys of a turn of the workgroup's waves, in which keys are dealt out.
__host__ __device__ constexpr int unit_keys(int dim) { return kAttWaves * 16 * key_subtiles(dim); }

struct AttArgs {
    const void* q;
    int64_t q_st, q_sh;
    const uint8_t* cache;
    int64_t block_stride, num_blocks;
    const int32_t* block_table;
    int64_t bt_stride;
    const int32_t* seq_lens;
    const int32_t* query_start_loc;  // or null: one token per request
    const float* sink;               // or null
    void* out;
    int64_t o_st, o_sh;
    float* lse;
    int64_t lse_st;
    float scale_f;    // softmax scale * log2(e) = scale_sign * scale_f * 2^scale_e, scale_f in [1, 2), sign 1, 0 or -1
    int32_t scale_e;
    float scale_sign;
    int32_t num_reqs, num_tokens, kv_heads, group, page, table_keys, window;
    int32_t first_worker;        // of this launch
    int32_t rows_from, rows_to;  // requests of other numbers of rows are another launch's
    // Stream mode (workers > 0): workers per head, and the workspace's parts.
    int32_t workers, per_cu, tile_cost;
    int32_t q_wide, o_wide;
    float* partials;
    struct CutTile* cut_tiles;
};

// A row tile whose keys are cut between workers: `count` of them from the first one on.
struct CutTile {
    int32_t first_token, first_row, rows, count;
};

// Longer requests are taken as this long: twice a table's keys, which windows are below.
constexpr int32_t kLongest = 0x7ff00000;

// A request's query tokens [first, first + count) and lengths.
struct Request {
    int32_t first, count, len;
};

__device__ __forceinline__ Request request_of(const AttArgs& a, int32_t b) {
    Request r;
    if (a.query_start_loc) {
        const int32_t lo = min(max(a.query_start_loc[b], 0), a.num_tokens);
        const int32_t hi = min(max(a.query_start_loc[b + 1], 0), a.num_tokens);
        r.first = lo;
        r.count = max(hi - lo, 0);
    } else {
        r.first = b;
        r.count = 1;
    }
    r.len = min(max(a.seq_lens[b], 0), kLongest);
    return r;
}

// The first tile boundary in front of what a row at position `pos` sees.
__device__ __forceinline__ int32_t keys_begin(const AttArgs& a, int32_t pos) {
    int32_t begin = 0;
    if (a.window > 0) {
        asm volatile("");  // a branch: without a window nothing waits for the request's length here
        begin = max(pos - a.window + 1, 0) & ~(kTileKeys - 1);
    }
    return begin;
}

// The most keys that a row of a request sees.
__device__ __forceinline__ int32_t keys_seen(const AttArgs& a, const Request& r) {
    const int32_t keys = min(r.len, a.table_keys);
    return a.window > 0 ? min(keys, a.window) : keys;
}

// A request and its tiles of rows, `units` units of keys each, dealt out as `cost`.
struct Tiles {
    Request req;
    int32_t count, units;
    __device__ int32_t cost(const AttArgs& a) const { return a.tile_cost + units; }
};

__device__ __forceinline__ Tiles tiles_of(const AttArgs& a, int32_t b, int32_t rows_per_tile, int32_t unit_keys) {
    Tiles t;
    t.req = request_of(a, b);
    const int32_t rows = t.req.count * a.group;  // fits: they are rows of q
    t.count = rows >= a.rows_from && rows <= a.rows_to ? (rows + rows_per_tile - 1) / rows_per_tile : 0;
    t.units = 1;
    if (a.workers > 0) {
        // the same for all tiles, as many as the longest can have: all keys from its first row's on, or what
        // its rows' windows cover
        int32_t keys = min(t.req.len, a.table_keys) - keys_begin(a, t.req.len - t.req.count);
        if (a.window > 0)
            keys = min(keys, a.window + (rows_per_tile + a.group - 2) / a.group + kTileKeys);
        t.units = max((keys + unit_keys - 1) / unit_keys, 1);
    }
    return t;
}

// Where a workgroup begins: `at` into the cost of tile `tile` of request b; it takes
// `take` of cost, through tiles and requests in order.  `each` is what workers take.
struct Start {
    Tiles tiles;
    int32_t b, tile, at;
    int32_t take, each;
};

// Sum of v over the lanes up to this one; sums stay at 2^32 - 1.
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v = add_sat(v, __builtin_amdgcn_update_dpp(0u, v, 0x111, 0xF, 0xF, false));  // row_shr:1, 2, 4, 8
    v = add_sat(v, __builtin_amdgcn_update_dpp(0u, v, 0x112, 0xF, 0xF, false));
    v = add_sat(v, __builtin_amdgcn_update_dpp(0u, v, 0x114, 0xF, 0xF, false));
    v = add_sat(v, __builtin_amdgcn_update_dpp(0u, v, 0x118, 0xF, 0xF, false));
    v = add_sat(v, __builtin_amdgcn_update_dpp(0u, v, 0x142, 0xA, 0xF, false));  // row_bcast:15 into rows 1 and 3
    v = add_sat(v, __builtin_amdgcn_update_dpp(0u, v, 0x143, 0xC, 0xF, false));  // row_bcast:31 into rows 2 and 3
    return v;
}

// The start of worker `index`; false if there is nothing for it.  Every workgroup
// works out the plan for itself: lengths are known on the device only, and a
// launch to do it would cost more than the scan.  In stream mode the cost of
// all tiles, one after the other, is dealt out evenly, so that workgroups have
// the same to do whatever the lengths are; a tile that is longer than the
// rest of its worker's share goes on with the next.  Otherwise a worker is a tile.
// (The host sees to it that the cost fits 31 bits, and that whole tiles have a
// workgroup each, for requests whose rows are their own.  Of requests that share rows
// the cost may be more: past 31 bits nothing is computed, nor are more tiles than there are workgroups.)
__device__ __forceinline__ bool find_start(const AttArgs& a, uint32_t index, int32_t rows_per_tile, int32_t unit_keys,
                                           Start& start) {
    if (a.workers == 0 && (a.num_reqs == 1 || !a.query_start_loc)) {
        // requests of equally many tiles need no scan (1 x 518 keys, 32 heads: 10.0 us with it, 9.3 without)
        const uint32_t each = (uint32_t)(a.group + rows_per_tile - 1) / (uint32_t)rows_per_tile;
        start.b = a.num_reqs == 1 ? 0 : (int32_t)(index / each);
        if (start.b >= a.num_reqs)
            return false;
        start.tiles = tiles_of(a, start.b, rows_per_tile, unit_keys);
        start.tile = start.tiles.count - 1 - (int32_t)(index - start.b * each);
        start.at = 0;
        start.take = start.each = 1;
        return start.tile >= 0;
    }
    __shared__ uint32_t part[kAttWaves];
    __shared__ int32_t found[8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Tiles mine = {};
    uint32_t at = 0, n = 0;  // cost in front of this thread's request of the turn, and its own
    auto scan_turn = [&](int32_t base, uint32_t& before) {
        const int32_t b = base + (int32_t)threadIdx.x;
        n = 0;
        if (b < a.num_reqs) {
            mine = tiles_of(a, b, rows_per_tile, unit_keys);
            n = __umulhi(mine.count, mine.cost(a)) ? ~0u : (uint32_t)mine.count * mine.cost(a);
        }
        const uint32_t s = wave_scan(n);
        if (lane == 63)
            part[wave] = s;
        __syncthreads();
        at = add_sat(before, s - n);
#pragma unroll
        for (int w = 0; w < kAttWaves; ++w) {
            at = add_sat(at, w < wave ? part[w] : 0);
            before = add_sat(before, part[w]);
        }
    };
    uint32_t total = 0;
    for (int32_t base = 0; base < a.num_reqs; base += kAttThreads) {
        if (base > 0)
            __syncthreads();  // the last turn's sums were read
        scan_turn(base, total);
    }
    uint32_t each = 1;
    if (a.workers > 0) {
        // as many workgroups to every CU, and fewer rather than with less than kLeastCost to do (24 requests of up to
        // 20000 keys, D = 256: 285 workgroups with 7 each 27.5 us, 333 with 6 32.5, as most CUs had one and some two)
        uint32_t to = (uint32_t)a.workers;
        for (int32_t k = a.per_cu - 1; k > 0; --k)
            to = total < to * (uint32_t)kLeastCost ? (uint32_t)max(a.workers * k / a.per_cu, 1) : to;
        each = max((total + to - 1) / to, (uint32_t)kLeastCost);
    }
    uint64_t first = (uint64_t)each * index;
    if (first >= total || total > 0x7fffffffu)
        return false;
    if (a.workers == 0)
        first = total - 1 - first;  // from the end: of a prompt's tiles the last have the most keys
    uint32_t before = 0;
    for (int32_t base = 0; base < a.num_reqs; base += kAttThreads) {
        if (a.num_reqs > kAttThreads) {
            __syncthreads();
            scan_turn(base, before);
        }
        if (first >= at && first - at < n) {
            const uint32_t in = (uint32_t)first - at, cost = mine.cost(a);
            const uint32_t tile = in / cost;
            found[0] = base + (int32_t)threadIdx.x;
            found[1] = (int32_t)tile;
            found[2] = (int32_t)(in - tile * cost);
            found[3] = mine.req.first;
            found[4] = mine.req.count;
            found[5] = mine.req.len;
            found[6] = mine.count;
            found[7] = mine.units;
        }
    }
    __syncthreads();
    start.b = __builtin_amdgcn_readfirstlane(found[0]);
    start.tile = __builtin_amdgcn_readfirstlane(found[1]);
    start.at = __builtin_amdgcn_readfirstlane(found[2]);
    start.tiles.req.first = __builtin_amdgcn_readfirstlane(found[3]);
    start.tiles.req.count = __builtin_amdgcn_readfirstlane(found[4]);
    start.tiles.req.len = __builtin_amdgcn_readfirstlane(found[5]);
    start.tiles.count = __builtin_amdgcn_readfirstlane(found[6]);
    start.tiles.units = __builtin_amdgcn_readfirstlane(found[7]);
    start.each = __builtin_amdgcn_readfirstlane((int32_t)each);
    start.take = __builtin_amdgcn_readfirstlane((int32_t)(total - first < each ? total - first : each));
    return true;
}

// How the dims of a head meet the matrix instruction's k of 128: kChunks
// instructions' worth of codes, 16 bytes of them a lane each; kSteps
// instructions for one 16 x 16 tile of scores with `kPieces` pieces of the query.
template <int D, int kPieces>
struct Shape {
    static constexpr int kChunks = D < 128 ? 1 : D / 128;
    // at D = 64 two pieces share an instruction, the keys' codes standing there twice
    static constexpr int kSteps = D < 128 ? (kPieces + 1) / 2 : kChunks * kPieces;
    static constexpr int kVPitch = 2 * D + 32;  // bytes between tokens of the turned V: the reads' banks differ
    static constexpr int kVBytes = 16 * key_subtiles(D) * kVPitch;
    static constexpr int kOPitch = 4 * D + 16;
    static_assert(kRows * kOPitch <= kVBytes, "a wave's O fits its V buffer");
};

// The query rows as the instruction's B operand.
template <int D, int kPieces>
struct Query {
    v8i_t q[Shape<D, kPieces>::kSteps];
    int scale[Shape<D, kPieces>::kSteps];
};

// N consecutive 16-bit values, two to a word; 0 where not valid.
template <int N>
__device__ __forceinline__ void load_words(const void* base, int64_t at, bool wide, bool valid, uint32_t (&w)[N / 2]) {
    const uint16_t* s = static_cast<const uint16_t*>(base) + at;
    if (!valid) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i)
            w[i] = 0;
    } else if (wide) {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(s + 8 * i);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i)
            w[i] = (uint32_t)s[2 * i] | (uint32_t)s[2 * i + 1] << 16;
    }
}

template <bool kHalf, int N>
__device__ __forceinline__ void to_floats(const uint32_t (&w)[N / 2], float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        if constexpr (kHalf) {
            x[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] & 0xffffu));
            x[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
        } else {
            x[2 * i] = bf16_lo(w[i]);
            x[2 * i + 1] = bf16_hi(w[i]);
        }
    }
}

// Four floats of magnitude below 448 to e4m3 codes; x keeps 16 times what they
// leave.  The first piece takes whole multiples of 1/8 only: the instruction
// cuts a product's bits below 2^-13 of the largest one that is added with it,
// and so those of small values, which the pieces behind then hold as well
// (scores of normal queries, error rms: 1.3e-5 without, 4.8e-6 with it in two
// pieces, 3.4e-7 in three; multiples of 1/4 and 1/16 lie between).
template <bool kFirst>
__device__ __forceinline__ uint32_t take_piece(float* x) {
    constexpr float kWhole = 1.5f * (float)(1 << 20);  // adding it and taking it away rounds to multiples of 1/8
    uint32_t w;
    if constexpr (kFirst)
        w = pack_fp8x4((x[0] + kWhole) - kWhole, (x[1] + kWhole) - kWhole, (x[2] + kWhole) - kWhole,
                       (x[3] + kWhole) - kWhole);
    else
        w = pack_fp8x4(x[0], x[1], x[2], x[3]);
    x[0] = (x[0] - __builtin_amdgcn_cvt_f32_fp8((int)w, 0)) * 16.0f;
    x[1] = (x[1] - __builtin_amdgcn_cvt_f32_fp8((int)w, 1)) * 16.0f;
    x[2] = (x[2] - __builtin_amdgcn_cvt_f32_fp8((int)w, 2)) * 16.0f;
    x[3] = (x[3] - __builtin_amdgcn_cvt_f32_fp8((int)w, 3)) * 16.0f;
    return w;
}

// A lane's part of a query row: dims 16g..16g+15 of each 64.
template <int D>
struct RawQuery {
    uint32_t w[D / 64][8];
};

template <int D>
__device__ __forceinline__ void load_query(const AttArgs& a, int64_t at, bool valid, int g, RawQuery<D>& raw) {
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
        load_words<16>(a.q, at + 64 * c + 16 * g, a.q_wide, valid, raw.w[c]);
}

// How a row with largest magnitude `most` (its bits) enters: q 2^scale_e = x 2^e,
// x = q * down with its maximum in [128, 256).  The softmax scale's power of two
// goes in here, so that scores leave binary32's range only where scaled ones
// would.  -118 leaves room for the pieces' smaller scales: rows whose largest value is below
// 2^-111 under the scale lose bits, which only keys of 2^100 and more would show.
struct QueryScale {
    bool bad;  // not finite, or not under the scale (2^135 and more): the scale says NaN
    int byte;
    float down;
};

__device__ __forceinline__ QueryScale query_scale(const AttArgs& a, uint32_t most) {
    const int exact = (int)(most >> 23) - 127 - 7 + a.scale_e, e = min(max(exact, -118), 127);
    QueryScale q;
    q.bad = most >= 0x7f800000u || exact > 127;
    q.byte = e + 127;
    q.down = __uint_as_float((uint32_t)min(max(127 - e + a.scale_e, 1), 254) << 23) * a.scale_sign;
    return q;
}

// Row r of lane (r, g) as the matrix instruction's operand.
template <int D, int kPieces, bool kHalf>
__device__ __forceinline__ void split_query(const AttArgs& a, const RawQuery<D>& raw, Query<D, kPieces>& out, int g) {
    constexpr int kRuns = D / 64;  // runs of 16 dims per lane
    float x[kRuns][16];
    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < kRuns; ++c) {
        to_floats<kHalf, 16>(raw.w[c], x[c]);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            most = max(most, __float_as_uint(x[c][i]) & 0x7fffffffu);
    }
    // over the row's four lanes
    most = max(most, (uint32_t)__shfl_xor((int)most, 16));
    most = max(most, (uint32_t)__shfl_xor((int)most, 32));
    const QueryScale q = query_scale(a, most);
#pragma unroll
    for (int c = 0; c < kRuns; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            x[c][i] = q.bad ? 0.f : x[c][i] * q.down;
    if constexpr (D == 64) {
#pragma unroll
        for (int s = 0; s < Shape<D, kPieces>::kSteps; ++s) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    out.q[s][4 * half + i] = 2 * s + half >= kPieces ? 0
                                             : (int)(s + half == 0 ? take_piece<true>(&x[0][4 * i])
                                                                   : take_piece<false>(&x[0][4 * i]));
            // (a piece that is not there, zeros, takes the last one's scale: one more step down might be no byte, or NaN's)
            out.scale[s] = q.bad ? 255 : q.byte - 4 * min(2 * s + (g >> 1), kPieces - 1);
        }
    } else {
#pragma unroll
        for (int p = 0; p < kPieces; ++p)
#pragma unroll
            for (int c = 0; c < Shape<D, kPieces>::kChunks; ++c) {
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        out.q[p * Shape<D, kPieces>::kChunks + c][4 * half + i] =
                            (int)(p == 0 ? take_piece<true>(&x[2 * c + half][4 * i])
                                         : take_piece<false>(&x[2 * c + half][4 * i]));
                out.scale[p * Shape<D, kPieces>::kChunks + c] = q.bad ? 255 : q.byte - 4 * p;
            }
    }
}

// A wave's keys as they stand in the cache, kSub subtiles of 16: lane (r, g) has
// dims 32g..32g+31 of each chunk of token 16t + r.
template <int kSub, int kChunks>
struct RawTile {
    uint4 k[kSub][kChunks], v[kSub][kChunks];
    uint32_t ks[kSub][kChunks], vs[kSub][kChunks];
    int32_t place[kSub];  // of its first token in the block, negative: there is none
};

// Where a wave's next 64 subtiles below `end` lie (entries are read up to `limit`): lane kSub i + t has subtile t of the i-th
// tile, the head's block at `base` and the first of its tokens at `place`
// (negative: no block).  Tiles of a wave are `stride` keys apart.
struct Places {
    int64_t base;
    int32_t place;
};

template <int kSub>
__device__ __forceinline__ Places find_places(const AttArgs& a, int32_t b, int32_t h, int32_t token_bytes, int32_t key0,
                                              int32_t stride, int32_t limit, int32_t end, int lane) {
    const int64_t key = (int64_t)key0 + (int64_t)(lane / kSub) * stride + 16 * (lane % kSub);
    Places p = {0, -1};
    if (key < limit) {
        const int32_t column = (int32_t)key / a.page;
        const int32_t id = a.block_table[(int64_t)b * a.bt_stride + column];
        if (id >= 0 && id < a.num_blocks && key < end) {
            p.base = (int64_t)id * a.block_stride + (int64_t)h * a.page * token_bytes;
            p.place = (int32_t)key - column * a.page;
        }
    }
    return p;
}

template <int D, int kSub>
__device__ __forceinline__ void load_tile(const AttArgs& a, const Places& p, int tile, int lane,
                                          RawTile<kSub, D < 128 ? 1 : D / 128>& raw) {
    constexpr int kChunks = D < 128 ? 1 : D / 128;
    const int r = lane & 15, g = D < 128 ? (lane >> 4) & 1 : lane >> 4;
#pragma unroll
    for (int t = 0; t < kSub; ++t) {
        const int from = tile % (64 / kSub) * kSub + t;
        const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)p.base, from);
        const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)((uint64_t)p.base >> 32), from);
        raw.place[t] = __builtin_amdgcn_readlane(p.place, from);
        // a subtile without a block reads the cache's first one, whose values nobody sees
        const int32_t first = max(raw.place[t], 0);
        const uint8_t* head = a.cache + (int64_t)((uint64_t)hi << 32 | lo);
        const uint8_t* kc = head + (int64_t)first * (D / 2);
        const uint8_t* vc = kc + mx_part(1, a.page, D);
        const uint8_t* ks = head + mx_part(2, a.page, D) + (int64_t)first * (D / kMxBlock);
        const uint8_t* vs = ks + (int64_t)a.page * (D / kMxBlock);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            raw.k[t][c] = *reinterpret_cast<const uint4*>(kc + (uint32_t)(r * (D / 2) + 64 * c + 16 * g));
            raw.ks[t][c] = ks[(uint32_t)(r * (D / kMxBlock) + 4 * c + g)];
            raw.v[t][c] = *reinterpret_cast<const uint4*>(vc + (uint32_t)(r * (D / 2) + 64 * c + 16 * g));
            raw.vs[t][c] = vs[(uint32_t)(r * (D / kMxBlock) + 4 * c + g)];
        }
    }
}

// 8 codes times 2^(byte - 127) in bf16, exact up to byte kMostByte; byte 255 gives NaN.
__device__ __forceinline__ uint4 values_of(uint32_t codes, float scale) {
    return make_uint4(
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3)));
}

__device__ __forceinline__ uint2 read_turned(const uint8_t* at) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (lds_short4_t*)(__attribute__((address_space(3))) uint8_t*)at));
}

__device__ __forceinline__ v8i_t key_operand(uint4 k) {
    const v8i_t v = {(int)k.x, (int)k.y, (int)k.z, (int)k.w, 0, 0, 0, 0};
    return v;
}

// What a lane knows of its row: the `count` keys from `first` on are seen.
struct Seen {
    int32_t first;
    uint32_t count;
    __device__ bool operator()(int32_t key) const { return (uint32_t)(key - first) < count; }
};
constexpr int32_t kNoKey = 0x7ff80000;  // seen by nobody: behind the longest request's last position

// Attends the tile's keys, from key0 on, for the wave's 16 rows.  `plain`: all of
// them are seen by all rows; otherwise, and where values are large or NaN, some may be
// hidden, hold anything or be NaN.  (One body for both: with two, the compiler keeps two sets of sums.)
//
// `margin` is large_margin of the largest values so far and `most_keys`, which a row sees at
// most; sums are under the reference m_run + margin.
//
// `refill` loads the next tile into `raw` as soon as this one has left it, for
// the matrix instruction and for LDS.
template <int D, int kPieces, int kSub, class Refill>
__device__ __forceinline__ void attend(RawTile<kSub, Shape<D, kPieces>::kChunks>& raw, int32_t key0, bool plain,
                                       Seen any, Seen seen, float scale_f, const Query<D, kPieces>& query,
                                       uint8_t* turned, int lane, f32x4_t (&acc)[D / 16], float& m_run, float& l_run,
                                       float& margin, int32_t most_keys, Refill refill) {
    using S = Shape<D, kPieces>;
    const int r = lane & 15, g = lane >> 4;
    f32x4_t s[kSub];
#pragma unroll
    for (int t = 0; t < kSub; ++t)
        s[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i)
#pragma unroll
        for (int t = 0; t < kSub; ++t) {
            const int c = i % S::kChunks;
            s[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(key_operand(raw.k[t][c]), query.q[i], s[t], 4, 0, 0,
                                                                    (int)raw.ks[t][c], 0, query.scale[i]);
        }

    uint64_t nan[kSub][S::kChunks];  // which value blocks are NaN, bit by lane
    int32_t key_of[kSub];            // each subtile's first key
    bool any_nan = false;
    uint32_t largest = 0;
#pragma unroll
    for (int t = 0; t < kSub; ++t)
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c)
            largest = max(largest, raw.vs[t][c]);
    plain = plain & !__any(largest > kLargeByte);
    if (!plain) {
        largest = 0;
#pragma unroll
        for (int t = 0; t < kSub; ++t) {
            key_of[t] = raw.place[t] >= 0 ? key0 + 16 * t : kNoKey;
#pragma unroll
            for (int c = 0; c < S::kChunks; ++c) {
                // a token that no row sees may hold anything; a NaN that some rows see is dealt with at the end
                const uint32_t byte = any(key_of[t] + r) ? raw.vs[t][c] : 0;
                nan[t][c] = __ballot(byte > kMostByte);
                any_nan |= nan[t][c] != 0;
                raw.vs[t][c] = byte > kMostByte ? 0 : byte;
                largest = max(largest, raw.vs[t][c]);
            }
        }
        if (__any(largest > kLargeByte)) {
            const float more = large_margin(most_keys, wave_largest(largest));
            if (more > margin) {
                const float down = __builtin_amdgcn_exp2f(margin - more);
                margin = more;
                l_run *= down;
#pragma unroll
                for (int d = 0; d < D / 16; ++d)
                    acc[d] *= down;
            }
        }
    }

    // V into LDS while the scores are on their way
    asm volatile("" ::: "memory");
#pragma unroll
    for (int t = 0; t < kSub; ++t)
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
            const float scale = __uint_as_float(raw.vs[t][c] << 23);
            if (D >= 128 || g < 2) {
                uint4* to = reinterpret_cast<uint4*>(turned + (16 * t + r) * S::kVPitch + 256 * c + 64 * g);
                to[0] = values_of(raw.v[t][c].x, scale);
                to[1] = values_of(raw.v[t][c].y, scale);
                to[2] = values_of(raw.v[t][c].z, scale);
                to[3] = values_of(raw.v[t][c].w, scale);
            }
            // (the scheduler would convert the whole tile first, into registers that there are not)
            __builtin_amdgcn_sched_barrier(0);
        }
    asm volatile("" ::: "memory");

    if (!plain) {
#pragma unroll
        for (int t = 0; t < kSub; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                s[t][i] = seen(key_of[t] + 4 * g + i) ? s[t][i] : -INFINITY;
    }
    float most = -INFINITY;
#pragma unroll
    for (int t = 0; t < kSub; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            most = fmaxf(most, s[t][i]);
    most = group4_max(most) * scale_f;
    if (__any(most > m_run)) {
        const float m_new = most > m_run ? most + kAhead : m_run;
        const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
            acc[d] *= alpha;
        m_run = m_new;
    }
    // (here, not earlier: behind the branch above the products above have left K's registers)
    refill();
    const float m_use = (m_run == -INFINITY ? 0.f : m_run) + margin;
    float p[4 * kSub];
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < kSub; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            p[4 * t + i] = __builtin_fmaf(s[t][i], scale_f, -m_use);
    if (__any(fabsf(m_use) > kFar)) {
#pragma unroll
        for (int t = 0; t < kSub; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                p[4 * t + i] = s[t][i] * scale_f - m_use;
    }
#pragma unroll
    for (int i = 0; i < 4 * kSub; ++i) {
        p[i] = __builtin_amdgcn_exp2f(p[i]);
        sum += p[i];
    }
    l_run += sum;  // this lane's keys; the row's four lanes are added up at the end

    // lane j of group g reads 4 dims of row 4g + j / 4 and gets dim j of rows 4g..4g+3
    const uint8_t* from = turned + (4 * g + (r >> 2)) * S::kVPitch + 8 * (r & 3);
    constexpr int kAtOnce = 4;  // 16-dim tiles whose reads are in flight together
#pragma unroll
    for (int half = 0; half < kSub / 2; ++half) {
        // k = 8g + i of this product is key 4g + i, or 16 + 4g + i - 4
        const float* ph = p + 8 * half;
        const uint4 hi = make_uint4(pack_bf16x2(ph[0], ph[1]), pack_bf16x2(ph[2], ph[3]), pack_bf16x2(ph[4], ph[5]),
                                    pack_bf16x2(ph[6], ph[7]));
        const uint4 lo = make_uint4(pack_bf16x2(ph[0] - bf16_lo(hi.x), ph[1] - bf16_hi(hi.x)),
                                    pack_bf16x2(ph[2] - bf16_lo(hi.y), ph[3] - bf16_hi(hi.y)),
                                    pack_bf16x2(ph[4] - bf16_lo(hi.z), ph[5] - bf16_hi(hi.z)),
                                    pack_bf16x2(ph[6] - bf16_lo(hi.w), ph[7] - bf16_hi(hi.w)));
#pragma unroll
        for (int d0 = 0; d0 < D / 16; d0 += kAtOnce) {
            bf16x8_t v[kAtOnce];
#pragma unroll
            for (int d = 0; d < kAtOnce; ++d) {
                const uint8_t* at = from + 32 * half * S::kVPitch + 32 * (d0 + d);
                const uint2 x = read_turned(at), y = read_turned(at + 16 * S::kVPitch);
                v[d] = __builtin_bit_cast(bf16x8_t, make_uint4(x.x, x.y, y.x, y.y));
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 0; d < kAtOnce; ++d)
                acc[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[d], __builtin_bit_cast(bf16x8_t, hi), acc[d0 + d], 0,
                                                                      0, 0);
#pragma unroll
            for (int d = 0; d < kAtOnce; ++d)
                acc[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[d], __builtin_bit_cast(bf16x8_t, lo), acc[d0 + d], 0,
                                                                      0, 0);
        }
    }

    // value blocks that are NaN, for the rows that see them
    if (any_nan) {
#pragma unroll
        for (int t = 0; t < kSub; ++t)
#pragma unroll
            for (int c = 0; c < S::kChunks; ++c)
#pragma unroll
                for (int b = 0; b < (D < 128 ? 2 : 4); ++b) {
                    float add = 0.f;
                    for (uint32_t bits = (uint32_t)(nan[t][c] >> (16 * b)) & 0xffffu; bits; bits &= bits - 1)
                        add = seen(key_of[t] + __builtin_ctz(bits)) ? NAN : add;
                    acc[8 * c + 2 * b] += add;
                    acc[8 * c + 2 * b + 1] += add;
                }
    }
}

// kN consecutive outputs of a row times inv, in its type.
template <bool kHalf, int kN>
__device__ __forceinline__ void store_out(uint16_t* to, const float* o, float inv, bool wide) {
    uint32_t w[kN / 2];
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
        const float x = o[2 * i] * inv, y = o[2 * i + 1] * inv;
        if constexpr (kHalf)
            w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x) |
                   (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)y) << 16;
        else
            w[i] = pack_bf16x2(x, y);
    }
    if (wide) {
#pragma unroll
        for (int i = 0; i < kN / 2; i += 2)
            *reinterpret_cast<uint2*>(to + 2 * i) = make_uint2(w[i], w[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < kN / 2; ++i) {
            to[2 * i] = (uint16_t)w[i];
            to[2 * i + 1] = (uint16_t)(w[i] >> 16);
        }
    }
}

// What a row's sums under reference m (base 2) come to: the factor of O and the lse.
struct RowEnd {
    float inv, lse;
};

__device__ __forceinline__ RowEnd finish_row(const AttArgs& a, int32_t head, float m, float l) {
    const float m_use = m == -INFINITY ? 0.f : m;
    RowEnd e;
    if (m == -INFINITY && l == 0.f) {  // nothing was seen
        e.inv = 0.f;
        e.lse = INFINITY;
        return e;
    }
    float below = l;
    if (a.sink)
        below += __builtin_amdgcn_exp2f(a.sink[head] * kLog2e - m_use);
    e.inv = 1.0f / below;
    e.lse = kLn2 * (m_use + __builtin_amdgcn_logf(l));
    return e;
}

// Floats of a slot of partial results: O of the tile's rows, their references and sums.
constexpr int slot_floats(int dim, int rows) { return rows * (dim + 2); }

// A worker has two slots of each head: for a tile that began before it (or is all
// cut through it), and for one that begins in it and goes on.
__device__ __forceinline__ int64_t slot_of(const AttArgs& a, int32_t h, int32_t worker, bool begins) {
    return 2 * ((int64_t)h * a.workers + worker) + (begins ? 1 : 0);
}

// A worker's tiles of 16 rows: four waves take a tile of keys each in turn,
// loaded one tile ahead, and their sums meet in LDS.
template <int D, int kPieces>
__global__ void __launch_bounds__(kAttThreads, groups_per_cu(D)) mxfp4_attend_kernel(AttArgs a) {
    using S = Shape<D, kPieces>;
    constexpr bool kHalf = kPieces == 3;
    constexpr int kSub = key_subtiles(D);
    constexpr int kKeys = 16 * kSub, kUnit = unit_keys(D), kBatch = 64 / kSub;
    constexpr int kDepth = D == 256 ? 1 : 2;  // tiles in registers
    __shared__ __align__(16) uint8_t turned[kAttWaves][S::kVBytes];
    __shared__ float wave_m[kAttWaves][kRows], wave_l[kAttWaves][kRows];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = (int)blockIdx.x % a.kv_heads;
    const int32_t worker = a.first_worker + (int32_t)(blockIdx.x / a.kv_heads);
    const int r = lane & 15, g = lane >> 4;
    const int orow = threadIdx.x >> 4, part = threadIdx.x & 15;  // of the end: 16 threads per row
    Start w;
    const bool busy = find_start(a, worker, kRows, kUnit, w);
    CutTile cut = {0, 0, 0, 0};  // the tile that begins here and goes on with the next workers
    int32_t left = busy ? w.take : 0;
    while (left > 0) {
        const Request req = w.tiles.req;
        // of the tile's cost a.tile_cost stands before its first unit
        const int32_t cost = min(left, w.tiles.cost(a) - w.at);
        const int32_t unit = max(w.at - a.tile_cost, 0);
        const int32_t units = max(w.at + cost - a.tile_cost, 0) - unit;
        if (units == 0)
            break;  // the tile begins with the next worker
        const bool whole = units == w.tiles.units;
        const int32_t rows = req.count * a.group;  // fits: count * group rows are rows of q
        const int32_t row = w.tile * kRows + r;
        const bool valid = row < rows;
        const int32_t token = (valid ? row : 0) / a.group;
        const int32_t head = h * a.group + (valid ? row - token * a.group : 0);
        const int32_t pos0 = req.len - req.count;
        const int32_t last_row = min(w.tile * kRows + kRows, rows) - 1;
        const int32_t first_pos = pos0 + w.tile * kRows / a.group, last_pos = pos0 + last_row / a.group;
        // keys seen by a row, and by any of them
        Seen seen, any;
        seen.first = a.window > 0 ? pos0 + token - a.window + 1 : 0;
        seen.count = valid ? (uint32_t)max(pos0 + token - seen.first + 1, 0) : 0;
        any.first = a.window > 0 ? first_pos - a.window + 1 : 0;
        any.count = (uint32_t)max(last_pos - any.first + 1, 0);
        int32_t begin = keys_begin(a, first_pos), end = min(min(req.len, a.table_keys), last_pos + 1);
        if (!whole) {
            begin += unit * kUnit;
            end = min(end, begin + units * kUnit);
        }

        const int32_t key0 = begin + wave * kKeys;
        const int32_t tiles = end > key0 ? (end - key0 + kUnit - 1) / kUnit : 0;
        // in the order in which they are waited for (without cuts the length is not known yet: the table has its columns
        // whatever it is, so that one does not wait for the other): the query's values are split while the first tiles come
        RawQuery<D> raw_query;
        load_query<D>(a, (req.first + token) * a.q_st + head * a.q_sh, valid, g, raw_query);
        Places places = find_places<kSub>(a, w.b, h, mx_token_bytes(D), key0, kUnit,
                                           a.workers > 0 ? end : a.table_keys, end, lane);
        // kDepth tiles are on their way: a tile's registers take another as soon as they are free
        RawTile<kSub, S::kChunks> raw[kDepth];
#pragma unroll
        for (int i = 0; i < kDepth; ++i)
            if (i < tiles)
                load_tile<D, kSub>(a, places, i, lane, raw[i]);

        Query<D, kPieces> query;
        split_query<D, kPieces, kHalf>(a, raw_query, query, g);
        f32x4_t acc[D / 16];
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
            acc[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        float m_run = -INFINITY, l_run = 0.f;
        float margin = 0.f;

        auto step = [&](int32_t i, RawTile<kSub, S::kChunks>& now) {
            auto refill = [&]() {
                const int32_t next = i + kDepth;
                if (next < tiles) {
                    if (next % kBatch == 0)
                        places = find_places<kSub>(a, w.b, h, mx_token_bytes(D), key0 + next * kUnit, kUnit, end, end, lane);
                    load_tile<D, kSub>(a, places, next, lane, now);
                }
            };
            const int32_t key = key0 + i * kUnit;
            bool plain = (key + kKeys - 1 <= min(first_pos, end - 1)) & ((a.window == 0) | (key > last_pos - a.window));
#pragma unroll
            for (int t = 0; t < kSub; ++t)
                plain = plain & (now.place[t] >= 0);
            attend<D, kPieces, kSub>(now, key, plain, any, seen, a.scale_f, query, turned[wave], lane, acc, m_run, l_run,
                                     margin, keys_seen(a, req), refill);
        };
        for (int32_t i = 0; i < tiles; i += kDepth) {
#pragma unroll
            for (int u = 0; u < kDepth; ++u)
                if (i + u < tiles)
                    step(i + u, raw[u]);
        }
        l_run = group4_sum(l_run);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
            *reinterpret_cast<f32x4_t*>(turned[wave] + r * S::kOPitch + 64 * d + 16 * g) = acc[d];
        if (g == 0) {
            wave_m[wave][r] = m_run + margin;
            wave_l[wave][r] = l_run;
        }
        __syncthreads();

        constexpr int kDims = D / 16;
        const int32_t mine = w.tile * kRows + orow;
        if (mine < rows) {
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < kAttWaves; ++i)
                m = fmaxf(m, wave_m[i][orow]);
            const float m_use = m == -INFINITY ? 0.f : m;
            float l = 0.f, o[kDims];
#pragma unroll
            for (int i = 0; i < kDims; ++i)
                o[i] = 0.f;
#pragma unroll
            for (int i = 0; i < kAttWaves; ++i) {
                const float f = __builtin_amdgcn_exp2f(wave_m[i][orow] - m_use);
                l += f * wave_l[i][orow];
                const float* from = reinterpret_cast<const float*>(turned[i] + orow * S::kOPitch) + part * kDims;
#pragma unroll
                for (int d = 0; d < kDims; d += 4) {
                    const f32x4_t v = *reinterpret_cast<const f32x4_t*>(from + d);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        o[d + j] += f * v[j];
                }
            }
            if (whole) {
                const int32_t otoken = mine / a.group, ohead = h * a.group + mine - otoken * a.group;
                const int64_t t = req.first + otoken;
                const RowEnd e = finish_row(a, ohead, m, l);
                store_out<kHalf, kDims>(static_cast<uint16_t*>(a.out) + t * a.o_st + ohead * a.o_sh + part * kDims, o,
                                        e.inv, a.o_wide);
                if (part == 0)
                    a.lse[t * a.lse_st + ohead] = e.lse;
            } else {
                // a worker's first slot holds the tile that came from the one before, its second the one that goes on
                float* slot = a.partials + slot_of(a, h, worker, unit == 0) * slot_floats(D, kRows);
#pragma unroll
                for (int i = 0; i < kDims; i += 4)
                    *reinterpret_cast<f32x4_t*>(slot + orow * D + part * kDims + i) =
                        f32x4_t{o[i], o[i + 1], o[i + 2], o[i + 3]};
                if (part == 0) {
                    slot[kRows * D + orow] = m;
                    slot[kRows * D + kRows + orow] = l;
                }
            }
        }
        left -= cost;
        if (!whole && unit == 0) {
            cut.first_token = req.first;
            cut.first_row = w.tile * kRows;
            cut.rows = rows;
            // the units behind this worker's, dealt out to the next ones
            cut.count = 1 + (w.tiles.units - units + w.each - 1) / w.each;
        }
        if (left > 0) {
            w.at = 0;
            if (++w.tile == w.tiles.count) {
                w.tile = 0;
                do
                    w.tiles = tiles_of(a, ++w.b, kRows, kUnit);  // there is one: cost is left
                while (w.tiles.count == 0);
            }
            __syncthreads();  // the joined sums were read
        }
    }
    if (a.workers > 0 && h == 0 && threadIdx.x == 0)
        a.cut_tiles[worker] = cut;
}

}  // namespace
}  // namespace fgv

#include "mxfp4_attend_wide.h"

namespace fgv {
namespace {

// Writes a joined row: kLanes lanes from `part` 0 on hold four dims each.
template <int D, bool kHalf>
__device__ __forceinline__ void write_row(const AttArgs& a, const CutTile& tile, int32_t r, int32_t h, int part, f32x4_t o,
                                          float m, float l) {
    const int32_t row = tile.first_row + r;
    const int32_t token = row / a.group, head = h * a.group + row - token * a.group;
    const int64_t t = tile.first_token + token;
    const RowEnd e = finish_row(a, head, m, l);
    const float out[4] = {o[0], o[1], o[2], o[3]};
    store_out<kHalf, 4>(static_cast<uint16_t*>(a.out) + t * a.o_st + head * a.o_sh + 4 * part, out, e.inv, a.o_wide);
    if (part == 0)
        a.lse[t * a.lse_st + head] = e.lse;
}

// The worker in which the index-th of the cut tiles begins (in some order); -1: there
// are fewer.
__device__ __forceinline__ int32_t find_cut(const AttArgs& a, int32_t index) {
    __shared__ int32_t found, in_front[kAttWaves];
    const int wave = threadIdx.x >> 6;
    if (threadIdx.x == 0)
        found = -1;
    for (int32_t base = 0; base < a.workers; base += kAttThreads) {
        const int32_t worker = base + (int32_t)threadIdx.x;
        const bool cut = worker < a.workers && a.cut_tiles[worker].count > 0;
        const uint64_t cuts = __ballot(cut);
        if (base > 0)
            __syncthreads();  // the last turn's counts were read
        in_front[wave] = __popcll(cuts);
        __syncthreads();
        int32_t rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(cuts >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)cuts, 0));
        int32_t all = 0;
#pragma unroll
        for (int w = 0; w < kAttWaves; ++w) {
            rank += w < wave ? in_front[w] : 0;
            all += in_front[w];
        }
        if (cut && rank == index)
            found = worker;
        index -= all;
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(found);
}

// Joins the cuts of a tile, for one head (both blockIdx.x) and the rows of blockIdx.y.
// kWide: a workgroup per row, its waves share out the cuts (few rows, of many
// cuts); otherwise a wave per row.  (The grid has as many rows as the host was told
// of; there may be more.)  Workgroups are launched for tiles, which the host knows
// better than how many workers there will be (875 rows of one request, 2 heads: 5.4 us;
// for each worker, most of them with nothing to join, 8.4).
template <int D, bool kHalf, int kTileRows, bool kWide>
__global__ void __launch_bounds__(kAttThreads) mxfp4_combine_kernel(AttArgs a) {
    constexpr int kLanes = D / 4, kGroups = 64 / kLanes;  // lanes per row, cuts that a wave takes at a time
    constexpr int kRowsAtOnce = kWide ? 1 : kAttWaves;
    __shared__ f32x4_t sums[kWide ? kAttWaves : 1][kLanes];
    __shared__ float factors[kAttWaves][64];
    const int32_t h = (int32_t)(blockIdx.x % a.kv_heads), worker = find_cut(a, (int32_t)(blockIdx.x / a.kv_heads));
    if (worker < 0)
        return;
    const CutTile tile = a.cut_tiles[worker];
    const int32_t rows = min(tile.rows - tile.first_row, kTileRows);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = lane % kLanes, group = lane / kLanes;
    // the cuts are this worker's second slot and the next ones' first
    auto slot_at = [&](int32_t i) {
        return a.partials + slot_of(a, h, worker + i, i == 0) * slot_floats(D, kTileRows);
    };
    for (int32_t r = (int32_t)blockIdx.y * kRowsAtOnce + (kWide ? 0 : wave); r < rows;
         r += (int32_t)gridDim.y * kRowsAtOnce) {
        // the first sums are asked for before their factors are known
        constexpr int kEarly = 4, kStep = kWide ? kAttWaves * kGroups : kGroups;
        const int32_t mine = kWide ? wave * kGroups + group : group;
        f32x4_t early[kEarly];
#pragma unroll
        for (int e = 0; e < kEarly; ++e)
            early[e] = *reinterpret_cast<const f32x4_t*>(slot_at(min(mine + e * kStep, tile.count - 1)) + r * D + 4 * part);
        // every wave finds the reference for itself
        float m_first = -INFINITY, l_first = 0.f;  // of the cut with this lane's number
        if (lane < tile.count) {
            m_first = slot_at(lane)[kTileRows * D + r];
            l_first = slot_at(lane)[kTileRows * D + kTileRows + r];
        }
        float m = m_first;
        for (int32_t i = lane + 64; i < tile.count; i += 64)
            m = fmaxf(m, slot_at(i)[kTileRows * D + r]);
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1)
            m = fmaxf(m, __shfl_xor(m, d));
        const float m_use = m == -INFINITY ? 0.f : m;
        float l = 0.f;
        f32x4_t o = {0.f, 0.f, 0.f, 0.f};
        for (int32_t base = 0; base < tile.count; base += 64) {
            float f = 0.f;
            if (base == 0) {
                f = __builtin_amdgcn_exp2f(m_first - m_use);
                l = f * l_first;
            } else if (base + lane < tile.count) {
                const float* slot = slot_at(base + lane) + kTileRows * D + r;
                f = __builtin_amdgcn_exp2f(slot[0] - m_use);
                l += f * slot[kTileRows];
            }
            const int32_t n = min(tile.count - base, 64);
            factors[wave][lane] = f;  // read by this wave alone
            int32_t i = mine;
            if (base == 0) {
#pragma unroll
                for (int e = 0; e < kEarly; ++e) {
                    if (i < n)
                        o += factors[wave][i] * early[e];
                    i += kStep;
                }
            }
#pragma unroll 8
            for (; i < n; i += kStep)
                o += factors[wave][i] * *reinterpret_cast<const f32x4_t*>(slot_at(base + i) + r * D + 4 * part);
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1)
            l += __shfl_xor(l, d);
#pragma unroll
        for (int d = kLanes; d < 64; d <<= 1)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                o[j] += __shfl_xor(o[j], d);
        if constexpr (kWide) {
            if (group == 0)
                sums[wave][part] = o;
            __syncthreads();
            if (wave == 0 && group == 0) {
#pragma unroll
                for (int i = 1; i < kAttWaves; ++i)
                    o += sums[i][part];
                write_row<D, kHalf>(a, tile, r, h, part, o, m, l);
            }
            __syncthreads();  // before the next row's sums
        } else {
            if (group == 0)
                write_row<D, kHalf>(a, tile, r, h, part, o, m, l);
        }
    }
}

// How a launch is dealt out, from what the host knows.
struct Dealing {
    int64_t tiles;    // row tiles at most
    int32_t rows;     // of a tile, as far as the host knows
    int32_t workers;  // per head; 0: a workgroup per tile
    int64_t cut_tiles_at, bytes;  // of the workspace
};

// One launch takes all requests, or two share them by their rows: 16-row tiles for
// up to kFewRows, 128-row tiles (whose waves would have nothing to do: 56 rows
// 49 us with the first, 68 with the others) for more, where D is at most 128 (D =
// 256 leaves 128-row tiles one workgroup to a CU; they took 842 us where the others
// take 735, 2048 tokens behind 8192 keys).
constexpr int kFewRows = 64;

struct Call {
    int64_t tokens, heads, kv_heads, dim, reqs, max_query;
    int64_t max_keys;  // of a tile's rows
    bool wide() const { return dim <= 128 && max_query * (heads / kv_heads) > kFewRows; }
    // Short requests, if they are a few, are better off in the others' tiles than in two launches more, whether there
    // are any or not (6 prompts 109 us with the launches, 104 without).
    bool few() const {
        return !wide() || (reqs > 1 && (max_keys > kWholeUnits * unit_keys((int)dim) || reqs * kv_heads > cu_count() / 4));
    }
};

Call call_of(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t reqs, int64_t max_query,
             int64_t max_seq, int64_t window) {
    // (a window's tile: its rows' tokens apart, and the boundary before its first key)
    const int64_t most = window > 0 && window < max_seq ? window + kTileKeys + 128 * kv_heads / heads : max_seq;
    return {tokens, heads, kv_heads, dim, reqs, max_query < tokens ? max_query : tokens, most < max_seq ? most : max_seq};
}

int per_cu(int dim, bool wide) { return wide ? 2 : groups_per_cu(dim); }

Dealing dealing_of(const Call& c, bool wide) {
    const int64_t group = c.heads / c.kv_heads, tile_rows = wide ? kWideRows : kRows;
    const int64_t slots = per_cu((int)c.dim, wide) * cu_count();
    const int64_t unit = wide ? kWideKeys : unit_keys((int)c.dim);
    Dealing d = {};
    const int64_t rows = group * (c.max_query < 1 ? 1 : c.max_query < tile_rows ? c.max_query : tile_rows);
    d.rows = (int32_t)(rows < tile_rows ? rows : tile_rows);
    // no request has more tiles than its rows' share, rounded up
    d.tiles = c.reqs == 1 ? (c.tokens * group + tile_rows - 1) / tile_rows : c.tokens * group / tile_rows + c.reqs;
    int64_t workers = slots / c.kv_heads;
    workers = workers > kMostWorkers ? kMostWorkers : workers;
    // Nothing to cut; or two 128-row tiles a workgroup and more.  Their partial results are 66 KB at D = 128: prompts
    // of 1140 tiles on 512 workgroups took 151 us with cuts, which leave no workgroup idle, and 108 without.
    if (workers < 2 || c.max_keys <= kWholeUnits * unit || (wide && (d.tiles - c.reqs) * c.kv_heads >= 2 * slots))
        return d;
    // One request's tiles, much alike, in (nearly) whole turns of the chip, the longest first.  Dealt out and whole, 32 heads
    // of 128, 512 workgroups: behind 14336 keys 512 tiles (2048 tokens) 500 and 483 us, 488 tiles 511 and 472, 472 tiles 491
    // and 461, 384 tiles 394 and 437, 520 tiles 545 and 726, 960 tiles 1038 and 953.  Behind 2048 keys whole is ahead at any
    // number (256 tiles 79 and 76, 384 119 and 92, 512 128 and 112, 576 183 and 165), which this rule does not know.
    const int64_t turns = (d.tiles * c.kv_heads + slots - 1) / slots;
    if (wide && c.reqs == 1 && 20 * d.tiles * c.kv_heads >= 19 * turns * slots)
        return d;
    d.workers = (int32_t)workers;
    d.cut_tiles_at = 2 * workers * c.kv_heads * (int64_t)slot_floats((int)c.dim, (int)tile_rows) * 4;
    d.bytes = (d.cut_tiles_at + workers * (int64_t)sizeof(CutTile) + 255) / 256 * 256;
    return d;
}

// Workgroups of a launch: one of 2^32 threads and more is cut to the low 32 bits without an error.
constexpr int64_t kMostGroups = (1LL << 31) / kAttThreads;

template <int D, int kPieces, int kTileRows>
void launch_part(const Dealing& d, uint8_t* workspace, int64_t unit, hipStream_t st, AttArgs a) {
    // (the cost of all tiles has to fit 31 bits: with more of it there is nothing to gain either)
    const bool stream = workspace && d.workers > 0 && d.tiles * (kTileCost + 1 + a.table_keys / unit) <= 0x7fffffffLL;
    a.workers = stream ? d.workers : 0;
    a.tile_cost = stream ? kTileCost : 0;
    a.per_cu = per_cu(D, kTileRows == kWideRows);
    a.partials = reinterpret_cast<float*>(workspace);
    a.cut_tiles = reinterpret_cast<CutTile*>(workspace + d.cut_tiles_at);
    const int64_t workers = stream ? d.workers : d.tiles, most = kMostGroups / a.kv_heads;
    for (int64_t first = 0; first < workers; first += most) {
        a.first_worker = (int32_t)first;
        const unsigned grid = (unsigned)((workers - first < most ? workers - first : most) * a.kv_heads);
        if constexpr (kTileRows == kRows)
            hipLaunchKernelGGL((mxfp4_attend_kernel<D, kPieces>), dim3(grid), dim3(kAttThreads), 0, st, a);
        else
            hipLaunchKernelGGL((mxfp4_attend_wide_kernel<D, kPieces>), dim3(grid), dim3(kAttThreads), 0, st, a);
    }
    if (!stream)
        return;
    // a wave per row where that fills the chip (4 x 256 rows)
    const int64_t cut_tiles = (d.tiles < a.workers ? d.tiles : a.workers) * a.kv_heads;
    if (cut_tiles * d.rows >= 1024) {
        // (4096 workgroups at most, if each has a tile: they take more rows then)
        const int64_t share = 4096 / cut_tiles, rows = (d.rows + 3) / 4;
        hipLaunchKernelGGL((mxfp4_combine_kernel<D, kPieces == 3, kTileRows, false>),
                           dim3((unsigned)cut_tiles, (unsigned)(share < 1 ? 1 : share < rows ? share : rows)),
                           dim3(kAttThreads), 0, st, a);
    } else {
        hipLaunchKernelGGL((mxfp4_combine_kernel<D, kPieces == 3, kTileRows, true>), dim3((unsigned)cut_tiles, d.rows),
                           dim3(kAttThreads), 0, st, a);
    }
}

template <int D, int kPieces>
void launch_attend(const Call& c, uint8_t* workspace, hipStream_t st, AttArgs a) {
    a.rows_from = 0;
    a.rows_to = 0x7fffffff;
    if constexpr (D <= 128) {
        if (c.wide()) {
            const Dealing d = dealing_of(c, true);
            a.rows_from = c.few() ? kFewRows + 1 : 0;
            launch_part<D, kPieces, kWideRows>(d, workspace, kWideKeys, st, a);
            workspace = workspace ? workspace + d.bytes : nullptr;
            a.rows_from = 0;
            a.rows_to = kFewRows;
        }
    }
    if (c.few())
        launch_part<D, kPieces, kRows>(dealing_of(c, false), workspace, unit_keys(D), st, a);
}

template <int D>
void launch_attend(bool half, const Call& c, uint8_t* workspace, hipStream_t st, const AttArgs& a) {
    half ? launch_attend<D, 3>(c, workspace, st, a) : launch_attend<D, 2>(c, workspace, st, a);
}

int64_t workspace_of(const Call& c) {
    return (c.wide() ? dealing_of(c, true).bytes : 0) + (c.few() ? dealing_of(c, false).bytes : 0);
}

}  // namespace
}  // namespace fgv

extern "C" int fgv_mxfp4_paged_attention(const void* q, int64_t q_stride_token, int64_t q_stride_head, int32_t dtype,
                                         int64_t num_tokens, int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                                         const uint8_t* kv_cache, int64_t cache_block_stride, int64_t num_blocks,
                                         int64_t block_size, const int32_t* block_table, int64_t block_table_stride,
                                         int64_t max_blocks_per_req, const int32_t* seq_lens,
                                         const int32_t* query_start_loc, int64_t num_reqs, int64_t max_query_len,
                                         int64_t max_seq_len, double softmax_scale, int64_t window_size,
                                         const float* attn_sink, void* out, int64_t out_stride_token,
                                         int64_t out_stride_head, float* lse, int64_t lse_stride_token, void* workspace,
                                         int64_t workspace_bytes, void* stream) {
    using namespace fgv;
    if (num_tokens < 0 || num_heads < 0 || num_kv_heads < 0 || num_blocks < 0 || num_reqs < 0 || max_blocks_per_req < 0 ||
        max_query_len < 0 || max_seq_len < 0 || window_size < 0)
        return fail(FGV_E_BAD_SHAPE, "negative size");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return fail(FGV_E_BAD_SHAPE, "head_dim must be 64, 128 or 256");
    if (dtype != 0 && dtype != 1)
        return fail(FGV_E_BAD_SHAPE, "dtype must be 0 (bf16) or 1 (fp16)");
    if (block_size <= 0 || block_size % 16 != 0)
        return fail(FGV_E_BAD_SHAPE, "block_size must be a positive multiple of 16");
    if (num_tokens == 0 || num_heads == 0 || num_reqs == 0)
        return FGV_OK;
    if (num_kv_heads == 0 || num_heads % num_kv_heads != 0)
        return fail(FGV_E_BAD_SHAPE, "num_heads must be a multiple of num_kv_heads");
    if (!query_start_loc && num_tokens != num_reqs)
        return fail(FGV_E_BAD_SHAPE, "without query_start_loc there is one token per request");
    if (!(softmax_scale >= -1e30 && softmax_scale <= 1e30))
        return fail(FGV_E_BAD_SHAPE, "softmax_scale must be finite");
    if (num_heads > 65536 || block_size > 4096 || num_reqs > 0x3fffffffLL || num_blocks > 0x7fffffffLL ||
        num_tokens > 0x3fffffffLL / num_heads || max_blocks_per_req > (0x3fffffffLL / block_size))
        return fail(FGV_E_TOO_LARGE, "at most 65536 heads, 4096 tokens per block, 2^30 - 1 query rows and table keys");
    if (!q || !out || !lse || !seq_lens || (max_blocks_per_req > 0 && !block_table) || (num_blocks > 0 && !kv_cache))
        return fail(FGV_E_NULL_POINTER, "null pointer argument");
    if (num_blocks > 0 && (cache_block_stride < num_kv_heads * block_size * mx_token_bytes((int)head_dim) ||
                           cache_block_stride % 16 != 0))
        return fail(FGV_E_BAD_STRIDE, "cache_block_stride must hold a block and be a multiple of 16");
    if (!aligned(kv_cache, 16) || !aligned(q, 2) || !aligned(out, 2) || !aligned(lse, 4))
        return fail(FGV_E_MISALIGNED, "kv_cache must be 16-byte aligned, q, out and lse by element");
    AttArgs a;
    a.q = q;
    a.q_st = q_stride_token;
    a.q_sh = q_stride_head;
    a.cache = kv_cache;
    a.block_stride = cache_block_stride;
    a.num_blocks = num_blocks;
    a.block_table = block_table;
    a.bt_stride = block_table_stride;
    a.seq_lens = seq_lens;
    a.query_start_loc = query_start_loc;
    a.sink = attn_sink;
    a.out = out;
    a.o_st = out_stride_token;
    a.o_sh = out_stride_head;
    a.lse = lse;
    a.lse_st = lse_stride_token;
    const double scale_log2 = softmax_scale * 1.4426950408889634;
    int e = 0;
    frexp(scale_log2, &e);
    a.scale_e = scale_log2 == 0.0 ? 0 : e - 1 < -100 ? -100 : e - 1;
    a.scale_f = scale_log2 == 0.0 ? 1.0f : (float)ldexp(fabs(scale_log2), -a.scale_e);
    a.scale_sign = scale_log2 > 0.0 ? 1.0f : scale_log2 < 0.0 ? -1.0f : 0.0f;
    a.num_reqs = (int32_t)num_reqs;
    a.num_tokens = (int32_t)num_tokens;
    a.kv_heads = (int32_t)num_kv_heads;
    a.group = (int32_t)(num_heads / num_kv_heads);
    a.page = (int32_t)block_size;
    // without a block nothing is seen
    a.table_keys = num_blocks > 0 ? (int32_t)(max_blocks_per_req * block_size) : 0;
    a.window = (int32_t)(window_size < 0x3fffffffLL ? window_size : 0);
    a.q_wide = aligned(q, 16) && ((q_stride_token | q_stride_head) & 7) == 0;
    a.o_wide = aligned(out, 8) && ((out_stride_token | out_stride_head) & 3) == 0;
    const Call call = call_of(num_tokens, num_heads, num_kv_heads, head_dim, num_reqs, max_query_len, max_seq_len,
                              window_size);
    if ((num_tokens * a.group / kRows + num_reqs) * num_kv_heads > 0x7fffffffLL)
        return fail(FGV_E_TOO_LARGE, "too many row tiles");
    const int64_t bytes = workspace_of(call);
    uint8_t* const ws = bytes > 0 && workspace_bytes >= bytes ? static_cast<uint8_t*>(workspace) : nullptr;
    if (ws && !aligned(ws, 16))
        return fail(FGV_E_MISALIGNED, "workspace must be 16-byte aligned");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    switch (head_dim) {
        case 64: launch_attend<64>(dtype == 1, call, ws, st, a); break;
        case 128: launch_attend<128>(dtype == 1, call, ws, st, a); break;
        default: launch_attend<256>(dtype == 1, call, ws, st, a); break;
    }
    return launch_status();
}

extern "C" int64_t fgv_mxfp4_paged_attention_workspace_bytes(int64_t num_tokens, int64_t num_heads,
                                                             int64_t num_kv_heads, int64_t head_dim, int64_t num_reqs,
                                                             int64_t max_query_len, int64_t max_seq_len) {
    if (num_tokens <= 0 || num_reqs <= 0 || num_kv_heads <= 0 || num_heads < num_kv_heads || num_heads > 65536 ||
        num_tokens > 0x3fffffffLL / num_heads || num_reqs > 0x3fffffffLL)
        return 0;
    return fgv::workspace_of(
        fgv::call_of(num_tokens, num_heads, num_kv_heads, head_dim, num_reqs, max_query_len, max_seq_len, 0));
}
