// Attention over the paged MXFP4 cache for requests of many query rows: tiles of
// 128 rows, included by mxfp4_attention.hip behind the parts that it shares
// with the kernel for few rows.
//
// A workgroup's four waves hold 32 rows each and go through the same keys, 64 at
// a time.  QK takes K's codes and scale bytes from memory straight into
// v_mfma_scale_f32_32x32x64_f8f6f4 (every wave for itself: a tile of K is 4 KB,
// which the CU's cache holds).  V is converted once per workgroup, 16 keys by
// each wave, into LDS, from where all waves read it turned; two buffers, and
// one barrier per tile.  Registers (as measured): lane (n, h) = (l % 32, l / 32)
// holds of A (K) dims 32h..32h+31 of key n, of B (q) dims 16h..16h+15 and
// 32+16h..32+16h+15 of row n, of S^T keys 8 (i / 4) + 4h + i % 4 of row n, i < 16.
//
// P goes in as one fp16 piece (bf16 calls; two in fp16 calls), V as fp16 values:
// bf16's 8 bits of P would put as large an error beside the output's rounding
// again, and a second piece another half of PV's time.  Value blocks beyond
// fp16's range (half_holds) are left to a second loop in bf16 with two pieces,
// which the first one enters at the first 64 keys that hold one, for all keys
// behind them: a single block among 16384 keys takes the call below from 487 us to
// 660 if it stands in the middle, and to 854 at the first key.
//
// A wave's matrix instructions of a tile take 1026 cycles (D = 128, bf16 calls), its
// vector instructions 1180 (exp2 among them), and the two overlap only where other
// instructions stand between them in the stream: so V's conversion goes between
// QK's, the second half's exponentials between PV's for the first, loads are asked
// for a tile (V: two) ahead.  2048 tokens behind 14336 keys, 32 heads of 128: 475 to 495 us
// (by the card), 515 GFLOP at 1040 to 1085 TFLOP/s, matrix units busy half of the time, vector
// issue somewhat more; QK, softmax and PV one after the other took 610, 16-row tiles 1083.
#pragma once

namespace fgv {
namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

constexpr int kWideRows = 128;  // query rows of a workgroup
constexpr int kWideKeys = 64;   // keys of a tile, and of a unit

// P times 2^7 and V times 2^-7 use fp16's range better than P, at most 1, and V
// would: P is held to 2^-32.  2^-7 * 0.5 * 2^(111 - 127) is fp16's least value,
// and 2^-7 * 6 * 2^(147 - 127) below its largest.
constexpr int kHalfShift = 7;
__device__ __forceinline__ bool half_holds(uint32_t byte, u32x4_t codes) {
    const bool zeros = ((codes.x | codes.y | codes.z | codes.w) & 0x77777777u) == 0;
    return (byte - (104u + kHalfShift) <= 36u) | (zeros & (byte <= kMostByte));
}

template <int D, int kPieces>
struct WideShape {
    static constexpr int kChunks = D / 64;                // of 64 dims: one QK instruction per piece
    static constexpr int kVPitch = D == 64 ? 192 : 2 * D + 64;  // four rows of 64 bytes meet no bank twice
    static constexpr int kVBytes = kWideKeys * kVPitch;
    static constexpr int kOPitch = 2 * D + 16;
    static_assert(kAttWaves * 32 * kOPitch <= 2 * kVBytes, "the outputs fit the V buffers");
};

template <int D>
struct WideKeyTile {
    u32x4_t k[2][D / 64];
    uint32_t ks[2];  // the key's scales
};

template <int D>
struct WideValueTile {
    u32x4_t v;    // 32 dims of a token
    uint32_t vs;  // the token's scales; `look` takes this lane's
    int32_t key;  // of the first of the wave's 16 tokens, kNoKey: no block
};

// Where the wave's next 64 subtiles lie, one a lane: the K codes and K scales of
// their first token.  One without a block is taken from the cache's first block,
// whose values nobody sees.
struct WidePlaces {
    uint64_t codes, scales;
    uint64_t live;  // the lanes that have a block
};

template <int D>
__device__ __forceinline__ WidePlaces find_wide_places(const AttArgs& a, int32_t b, int32_t h, int32_t key, int32_t end,
                                                       int lane) {
    const Places p = find_places<4>(a, b, h, mx_token_bytes(D), key, kWideKeys, end, end, lane);
    const uint64_t head = (uint64_t)a.cache + (uint64_t)p.base;
    const uint32_t first = (uint32_t)max(p.place, 0);
    WidePlaces w;
    w.codes = head + first * (D / 2);
    w.scales = head + (uint64_t)mx_part(2, a.page, D) + first * (D / kMxBlock);
    w.live = __ballot(p.place >= 0);
    return w;
}

__device__ __forceinline__ uint64_t from_lane(uint64_t v, int lane) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * lane, (int)(uint32_t)v);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * lane, (int)(uint32_t)(v >> 32));
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t from_uniform(uint64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), lane);
    return (uint64_t)hi << 32 | lo;
}

// (told to be global memory: a flat load would count as LDS work, which barriers wait for)
template <typename T>
__device__ __forceinline__ const __attribute__((address_space(1))) T* global(uint64_t at) {
    return reinterpret_cast<const __attribute__((address_space(1))) T*>(at);
}

template <int D>
__device__ __forceinline__ uint32_t scales_of(uint64_t at) {
    return D == 64 ? *global<uint16_t>(at) : *global<uint32_t>(at);
}

// Where the subtiles lie that hold this lane's keys of a tile: l % 32 of its halves.
struct WideKeyAt {
    uint64_t codes[2], scales[2];
};

template <int D>
__device__ __forceinline__ WideKeyAt find_keys(const WidePlaces& p, int tile, int lane) {
    const int upper = lane >> 4 & 1;
    WideKeyAt at;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int from = (tile & 15) * 4 + 2 * t + upper;
        at.codes[t] = from_lane(p.codes, from);
        at.scales[t] = from_lane(p.scales, from);
    }
    return at;
}

template <int D>
__device__ __forceinline__ void load_keys(const WideKeyAt& at, int lane, WideKeyTile<D>& out) {
    const int r = lane & 15, h = lane >> 5;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const uint64_t codes = at.codes[t] + (uint32_t)(r * (D / 2) + 16 * h);
        const uint64_t scales = at.scales[t] + (uint32_t)(r * (D / kMxBlock));
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
            out.k[t][i] = *global<u32x4_t>(codes + 32 * i);
        out.ks[t] = scales_of<D>(scales);
    }
}

template <int D>
__device__ __forceinline__ void load_values(const AttArgs& a, const WidePlaces& p, int tile, int wave, int lane, int32_t key0,
                                            WideValueTile<D>& out) {
    const int r = lane & 15, g = D < 128 ? (lane >> 4) & 1 : lane >> 4;
    const int from = (tile & 15) * 4 + wave;
    const uint64_t codes = from_uniform(p.codes, from) + (uint64_t)mx_part(1, a.page, D);
    const uint64_t scales = from_uniform(p.scales, from) + (uint64_t)a.page * (D / kMxBlock);
    out.key = p.live >> from & 1 ? key0 + 16 * wave : kNoKey;
    out.v = *global<u32x4_t>(codes + (uint32_t)(r * (D / 2) + 16 * g));
    out.vs = scales_of<D>(scales + (uint32_t)(r * (D / kMxBlock)));
}

// The query rows as the B operand: piece p of 64 dims c in step p * kChunks + c.
// The first kHeld pieces stay in registers; the others, of fp16 calls, which would
// be too many for them, in LDS.
template <int D, int kPieces>
struct WideQuery {
    static constexpr int kHeld = 2;
    static constexpr int kInLds = (kPieces - kHeld) * D / 32;  // 16 bytes of each lane
    v8i_t q[D / 64 * kHeld];
    int scale;  // of the first piece
};

// A lane's part of a query row: dims 16h..16h+15 of each 32.
template <int D>
struct RawWideQuery {
    uint32_t w[D / 32][8];
};

template <int D>
__device__ __forceinline__ void load_wide_query(const AttArgs& a, int64_t at, bool valid, int h, RawWideQuery<D>& raw) {
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
        load_words<16>(a.q, at + 32 * c + 16 * h, a.q_wide, valid, raw.w[c]);
}

constexpr int kBadScale = 0x10000;

// The scale byte of piece p: each is 2^-4 of the one before.
__device__ __forceinline__ int piece_scale(int scale, int p) { return scale == kBadScale ? 255 : scale - 4 * p; }

template <int D, int kPieces, bool kHalf>
__device__ __forceinline__ void split_wide_query(const AttArgs& a, const RawWideQuery<D>& raw, WideQuery<D, kPieces>& out,
                                                 uint4* in_lds, int lane) {
    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        float x[16];
        to_floats<kHalf, 16>(raw.w[c], x);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
    }
    most = max(most, (uint32_t)__shfl_xor((int)most, 32));  // over the row's two lanes
    const QueryScale q = query_scale(a, most);
    out.scale = q.bad ? kBadScale : q.byte;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        float x[16];
        to_floats<kHalf, 16>(raw.w[c], x);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            x[i] = q.bad ? 0.f : x[i] * q.down;
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
            uint32_t piece[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                piece[i] = p == 0 ? take_piece<true>(x + 4 * i) : take_piece<false>(x + 4 * i);
                if (p < out.kHeld)
                    out.q[p * (D / 64) + c / 2][4 * (c & 1) + i] = (int)piece[i];
            }
            if (p >= out.kHeld)
                in_lds[64 * ((p - out.kHeld) * (D / 32) + c) + lane] = make_uint4(piece[0], piece[1], piece[2], piece[3]);
        }
    }
}

// Over the two lanes of a row.
__device__ __forceinline__ float pair_max(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto x = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}

// Barrier over LDS work only: loads of the next tiles stay on their way.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));  // lgkmcnt(0) alone
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <bool kHalf>
__device__ __forceinline__ uint4 wide_values(uint32_t codes, float scale) {
    if constexpr (kHalf)
        return make_uint4(
            __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0)),
            __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1)),
            __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2)),
            __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3)));
    else
        return values_of(codes, scale);
}

template <bool kHalf>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    if constexpr (kHalf) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), f16x2_t));
    } else {
        return pack_bf16x2(lo, hi);
    }
}
template <bool kHalf>
__device__ __forceinline__ float first_of(uint32_t w) {
    return kHalf ? (float)__builtin_bit_cast(f16x2_t, w)[0] : bf16_lo(w);
}
template <bool kHalf>
__device__ __forceinline__ float second_of(uint32_t w) {
    return kHalf ? (float)__builtin_bit_cast(f16x2_t, w)[1] : bf16_hi(w);
}

template <bool kHalf>
__device__ __forceinline__ f32x16_t wide_product(uint4 v, uint4 p, f32x16_t acc) {
    if constexpr (kHalf)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, v), __builtin_bit_cast(f16x8_t, p), acc,
                                                      0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, v),
                                                       __builtin_bit_cast(bf16x8_t, p), acc, 0, 0, 0);
}

constexpr int kLdsRead = 0x100;  // what sched_barrier lets pass

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

template <int D, int kPieces>
__global__ void __launch_bounds__(kAttThreads, 2) mxfp4_attend_wide_kernel(AttArgs a) {
    using S = WideShape<D, kPieces>;
    constexpr bool kHalf = kPieces == 3;
    __shared__ __align__(16) uint8_t turned[2][S::kVBytes];
    __shared__ __align__(16) uint32_t held_by[2][kAttWaves];  // whether fp16 holds each wave's values
    __shared__ uint64_t nan_of[2][kAttWaves];                 // which of its value blocks are NaN, bit by lane
    __shared__ __align__(16) uint32_t large_of[2][kAttWaves];  // their largest byte, if it is past kLargeByte
    using Rows = WideQuery<D, kPieces>;
    __shared__ uint4 more_query[kAttWaves][Rows::kInLds ? 64 * Rows::kInLds : 1];  // the pieces not in registers
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, hh = lane >> 5, r = lane & 15, g = lane >> 4;
    const int h = (int)blockIdx.x % a.kv_heads;
    const int32_t worker = a.first_worker + (int32_t)(blockIdx.x / a.kv_heads);
    // Where this lane writes its first 16-byte piece of V, and reads V turned: piece i of a 64-byte run
    // lies at i ^ (row / 4 % 4), so that neither the lanes of a write nor of a read meet a bank twice.
    static_assert(S::kVPitch % 64 == 0 && S::kVBytes % 64 == 0, "pieces are found by xor");
    const uint32_t write_at = (uint32_t)((16 * wave + r) * S::kVPitch + 64 * (D < 128 ? g & 1 : g) + 16 * (r >> 2));
    const uint32_t read_at = (uint32_t)((4 * hh + (r >> 2)) * S::kVPitch +
                                        16 * ((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ hh) + 8 * (lane & 1));

    Start w;
    const bool busy = find_start(a, worker, kWideRows, kWideKeys, w);
    CutTile cut = {0, 0, 0, 0};  // the tile that begins here and goes on with the next workers
    int32_t left = busy ? w.take : 0;
    while (left > 0) {
        const Request req = w.tiles.req;
        const int32_t cost = min(left, w.tiles.cost(a) - w.at);
        const int32_t unit = max(w.at - a.tile_cost, 0);
        const int32_t units = max(w.at + cost - a.tile_cost, 0) - unit;
        if (units == 0)
            break;  // the tile begins with the next worker
        const bool whole = units == w.tiles.units;
        const int32_t rows = req.count * a.group;  // fits: count * group rows are rows of q
        const int32_t row0 = w.tile * kWideRows, wave_row0 = row0 + 32 * wave;
        const int32_t row = wave_row0 + n;
        const bool valid = row < rows;
        const int32_t token = (valid ? row : 0) / a.group;
        const int32_t head = h * a.group + (valid ? row - token * a.group : 0);
        const int32_t pos0 = req.len - req.count;
        const int32_t first_pos = pos0 + row0 / a.group, last_pos = pos0 + (min(row0 + kWideRows, rows) - 1) / a.group;
        // positions of this wave's rows; a wave without rows sees nothing
        const bool idle = wave_row0 >= rows;
        const int32_t wave_first = pos0 + wave_row0 / a.group;
        const int32_t wave_last = idle ? -1 : pos0 + (min(wave_row0 + 32, rows) - 1) / a.group;
        Seen seen, any;
        seen.first = a.window > 0 ? pos0 + token - a.window + 1 : 0;
        seen.count = valid ? (uint32_t)max(pos0 + token - seen.first + 1, 0) : 0;
        any.first = a.window > 0 ? first_pos - a.window + 1 : 0;
        any.count = (uint32_t)max(last_pos - any.first + 1, 0);
        int32_t begin = keys_begin(a, first_pos), end = min(min(req.len, a.table_keys), last_pos + 1);
        if (!whole) {
            begin += unit * kWideKeys;
            end = min(end, begin + units * kWideKeys);
        }
        const int32_t tiles = end > begin ? (end - begin + kWideKeys - 1) / kWideKeys : 0;

        RawWideQuery<D> raw_query;
        load_wide_query<D>(a, (req.first + token) * a.q_st + head * a.q_sh, valid, hh, raw_query);
        WidePlaces places = find_wide_places<D>(a, w.b, h, begin, end, lane);
        WideKeyTile<D> keys;
        WideValueTile<D> now, next;
        if (tiles > 0) {
            load_keys<D>(find_keys<D>(places, 0, lane), lane, keys);
            load_values<D>(a, places, 0, wave, lane, begin, now);
            load_values<D>(a, places, min(1, tiles - 1), wave, lane, begin + kWideKeys, next);
        }
        Rows query;
        split_wide_query<D, kPieces, kHalf>(a, raw_query, query, more_query[wave], lane);
        f32x16_t acc[D / 32];
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                acc[d][i] = 0.f;
        float m_run = -INFINITY, l_run = 0.f;
        float margin = 0.f;  // as in attend(): from the first large values on, which only the second loop meets

        // A token that no row sees may hold anything: its values are taken as finite.
        auto look = [&](WideValueTile<D>& t, int buffer) {
            t.vs = any(t.key + r) ? t.vs >> (8 * (D < 128 ? g & 1 : g)) & 255u : 127;
            held_by[buffer][wave] = __all(half_holds(t.vs, t.v));
        };
        uint32_t live_next = (uint32_t)places.live & 15u;  // which of the next tile's subtiles have a block
        bool all_held = false;  // by fp16, the next tile's values
        auto read_held = [&](int buffer) { return *reinterpret_cast<const uint4*>(held_by[buffer]); };
        auto set_held = [&](uint4 f) { all_held = __builtin_amdgcn_readfirstlane(f.x & f.y & f.z & f.w) != 0; };

        // This wave's 16 tokens into LDS: the scale they are converted with, and their 8-dim parts 0..3.
        auto scale_values = [&](auto kind, int buffer) {
            uint32_t byte = now.vs;
            if constexpr (decltype(kind)::value) {
                byte = max(byte, (uint32_t)kHalfShift) - kHalfShift;
            } else {
                nan_of[buffer][wave] = __ballot(byte > kMostByte);
                byte = byte > kMostByte ? 0 : byte;
                large_of[buffer][wave] = __any(byte > kLargeByte) ? wave_largest(byte) : 0;
            }
            return __uint_as_float(byte << 23);
        };
        auto put_values = [&](auto kind, int buffer, int part, float scale) {
            // (D = 64: both halves of the wave write the same)
            *reinterpret_cast<uint4*>(turned[0] + (((uint32_t)(buffer * S::kVBytes) + write_at) ^ (16 * part))) =
                wide_values<decltype(kind)::value>(now.v[part], scale);
        };
        auto find_ahead = [&](int32_t i) {
            if (i + 2 < tiles && ((i + 2) & 15) == 0)
                places = find_wide_places<D>(a, w.b, h, begin + (i + 2) * kWideKeys, end, lane);
        };
        auto load_ahead = [&](int32_t i) {
            load_values<D>(a, places, min(i + 2, tiles - 1), wave, lane, begin + (i + 2) * kWideKeys, next);
        };

        // A wave without rows has its part in V only.
        auto idle_step = [&](auto kind, int32_t i) {
            find_ahead(i);
            const float scale = scale_values(kind, i & 1);
#pragma unroll
            for (int part = 0; part < 4; ++part)
                put_values(kind, i & 1, part, scale);
            now = next;
            look(now, (i & 1) ^ 1);
            load_ahead(i);
            lds_barrier();
            set_held(read_held((i & 1) ^ 1));
        };

        auto step = [&](auto kind, int32_t i) {
            constexpr bool kFast = decltype(kind)::value;
            constexpr int kPPieces = kFast && kPieces == 2 ? 1 : 2;
            const int buffer = i & 1;
            const int32_t key = begin + i * kWideKeys;
            const WideKeyAt next_keys = find_keys<D>(places, min(i + 1, tiles - 1), lane);
            const uint32_t live = live_next;
            live_next = (uint32_t)(places.live >> (4 * ((i + 1) & 15))) & 15u;
            find_ahead(i);
            // ---- scores; between the matrix instructions this tile's V into LDS
            __builtin_amdgcn_s_setprio(1);
            f32x16_t s[2];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    s[t][j] = 0.f;
            const float v_scale = scale_values(kind, buffer);
#pragma unroll
            for (int q = 0; q < S::kChunks * kPieces; ++q) {
                const int c = q % S::kChunks, piece = q / S::kChunks;
                v8i_t rows_q;
                if (piece >= Rows::kHeld) {
                    const uint4* at = more_query[wave] + 128 * (q - Rows::kHeld * S::kChunks) + lane;
                    const uint4 x = at[0], y = at[64];
                    rows_q = v8i_t{(int)x.x, (int)x.y, (int)x.z, (int)x.w, (int)y.x, (int)y.y, (int)y.z, (int)y.w};
                } else {
                    rows_q = query.q[q];
                }
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const v8i_t k = key_operand(__builtin_bit_cast(uint4, keys.k[t][c]));
                    const int scales = (int)(keys.ks[t] >> 8 * hh), q_scale = piece_scale(query.scale, piece);
                    s[t] = c & 1 ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, rows_q, s[t], 4, 0, 2, scales, 0, q_scale)
                                 : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(k, rows_q, s[t], 4, 0, 0, scales, 0, q_scale);
                    if (2 * q + t < 4)
                        put_values(kind, buffer, 2 * q + t, v_scale);
                    __builtin_amdgcn_sched_barrier(kLdsRead);
                }
            }
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            now = next;
            look(now, buffer ^ 1);
            // ---- the next tile of K, and the one after it of V
            load_keys<D>(next_keys, lane, keys);
            load_ahead(i);
            lds_barrier();
            const uint4 held = read_held(buffer ^ 1);

            const bool plain = (key + kWideKeys - 1 <= min(wave_first, end - 1)) &
                               ((a.window == 0) | (key > wave_last - a.window)) & (live == 15u);
            if (!plain) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        int32_t base = (live >> (2 * t + u) & 1 ? key + 32 * t + 16 * u : kNoKey) + 4 * hh;
                        asm("" : "+v"(base));  // one register in all, not one for each key
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            s[t][8 * u + j] = seen(base + 8 * (j / 4) + j % 4) ? s[t][8 * u + j] : -INFINITY;
                    }
            }
            float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                most[j & 1] = fmaxf(most[j & 1], s[0][j]);
                most[2 + (j & 1)] = fmaxf(most[2 + (j & 1)], s[1][j]);
            }
            const float top = pair_max(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]))) * a.scale_f;
            if constexpr (!kFast) {
                const uint4 large = *reinterpret_cast<const uint4*>(large_of[buffer]);
                const uint32_t largest = __builtin_amdgcn_readfirstlane(max(max(large.x, large.y), max(large.z, large.w)));
                const float more = largest > 0 ? large_margin(keys_seen(a, req), largest) : 0.f;
                if (more > margin) {
                    const float down = __builtin_amdgcn_exp2f(margin - more);
                    margin = more;
                    l_run *= down;
#pragma unroll
                    for (int d = 0; d < D / 32; ++d)
                        acc[d] *= down;
                }
            }
            if (__any(top > m_run)) {
                const float m_new = top > m_run ? top + kAhead : m_run;
                const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
                l_run *= alpha;
#pragma unroll
                for (int d = 0; d < D / 32; ++d)
                    acc[d] *= alpha;
                m_run = m_new;
            }
            float m_use = (m_run == -INFINITY ? 0.f : m_run) + (kFast ? -(float)kHalfShift : margin);
            float times = a.scale_f;
            if (__any(fabsf(m_use) > kFar)) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        s[t][j] = s[t][j] * a.scale_f - m_use;
                times = 1.f;
                m_use = 0.f;
            }
            // Products of the first 32 keys' values go between the second's exponentials, and those
            // between the sums; operands are read kFetch products ahead.
            constexpr int kOps = 2 * (D / 32), kFetch = D == 128 && kPPieces == 1 ? 3 : 2;
            const uint32_t from0 = (uint32_t)(buffer * S::kVBytes) + read_at;
            const uint32_t from1 = (from0 + 8 * S::kVPitch) ^ 32;
            float p[32];
            uint4 pw[2][kPPieces][2];  // by 16 keys: keys 4h..4h+3 and 8+4h..8+4h+3 of them
            uint4 v[2 * kOps];
            auto fetch = [&](int q) {
                if (q < 2 * kOps) {
                    const uint8_t* at = turned[0] + 16 * (q / (D / 32)) * S::kVPitch + 64 * (q % (D / 32));
                    const uint2 x = read_turned(at + from0), y = read_turned(at + from1);
                    v[q] = make_uint4(x.x, x.y, y.x, y.y);
                }
            };
            auto weigh = [&](int j) {
                p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j / 16][j % 16], times, -m_use));
                if (j & 1) {
                    const uint32_t hi = pack_pair<kFast>(p[j - 1], p[j]);
                    uint32_t* to = &pw[j / 16][0][j / 8 % 2].x;
                    to[j / 2 % 4] = hi;
                    if constexpr (kPPieces == 2)
                        (&pw[j / 16][1][j / 8 % 2].x)[j / 2 % 4] =
                            pack_pair<kFast>(p[j - 1] - first_of<kFast>(hi), p[j] - second_of<kFast>(hi));
                }
            };
            auto product = [&](int q) {
                const int t = q / kOps, u = q / (D / 32) % 2, d = q % (D / 32);
#pragma unroll
                for (int piece = 0; piece < kPPieces; ++piece)
                    acc[d] = wide_product<kFast>(v[q], pw[t][piece][u], acc[d]);
            };
#pragma unroll
            for (int q = 0; q < kFetch; ++q)
                fetch(q);
#pragma unroll
            for (int j = 0; j < 16; ++j)
                weigh(j);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int q = 0; q < kOps; ++q) {
                fetch(q + kFetch);
                product(q);
#pragma unroll
                for (int j = 16 + q * 16 / kOps; j < 16 + (q + 1) * 16 / kOps; ++j)
                    weigh(j);
                __builtin_amdgcn_sched_barrier(0);
            }
            float sum = 0.f;
#pragma unroll
            for (int q = kOps; q < 2 * kOps; ++q) {
                fetch(q + kFetch);
                product(q);
#pragma unroll
                for (int j = (q - kOps) * 32 / kOps; j < (q + 1 - kOps) * 32 / kOps; ++j)
                    sum += p[j];
                __builtin_amdgcn_sched_barrier(0);
            }
            l_run += kFast ? sum * (1.0f / (1 << kHalfShift)) : sum;
            if constexpr (!kFast) {
                // value blocks that are NaN, for the rows that see them
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint64_t nan = nan_of[buffer][u];
                    const uint32_t half[2] = {(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)nan),
                                              (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(nan >> 32))};
#pragma unroll
                    for (int b = 0; b < D / 32; ++b) {
                        float add = 0.f;
                        for (uint32_t bits = half[b / 2] >> (16 * (b & 1)) & 0xffffu; bits; bits &= bits - 1)
                            add = seen(key + 16 * u + __builtin_ctz(bits)) ? NAN : add;
                        acc[b] += add;
                    }
                }
            }
            set_held(held);
        };

        if (tiles > 0) {
            look(now, 0);
            lds_barrier();
            set_held(read_held(0));
            int32_t i = 0;
            if (idle) {
                for (; i < tiles && all_held; ++i)
                    idle_step(Yes{}, i);
                for (; i < tiles; ++i)
                    idle_step(No{}, i);
            } else {
                for (; i < tiles && all_held; ++i)
                    step(Yes{}, i);
                for (; i < tiles; ++i)
                    step(No{}, i);
            }
        }

        l_run += __shfl_xor(l_run, 32);
        m_run += margin;
        lds_barrier();  // V was read
        int lane_again = lane;
        asm("" : "+v"(lane_again));  // what follows from it takes no registers in the loops
        const int end_n = lane_again & 31, end_hh = lane_again >> 5;
        const int32_t end_row = wave_row0 + end_n;
        const bool end_valid = end_row < rows;
        const int32_t end_token = (end_valid ? end_row : 0) / a.group;
        const int32_t end_head = h * a.group + (end_valid ? end_row - end_token * a.group : 0);
        if (whole) {
            const RowEnd e = finish_row(a, end_head, m_run, l_run);
            if (end_valid && end_hh == 0)
                a.lse[(req.first + end_token) * a.lse_st + end_head] = e.lse;
            // through LDS, so that whole rows are written: the wave's 32 rows in its own quarter
            uint8_t* stage = &turned[0][0] + wave * 32 * S::kOPitch;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float x0 = acc[d][4 * q] * e.inv, x1 = acc[d][4 * q + 1] * e.inv;
                    const float x2 = acc[d][4 * q + 2] * e.inv, x3 = acc[d][4 * q + 3] * e.inv;
                    *reinterpret_cast<uint2*>(stage + end_n * S::kOPitch + 2 * (32 * d + 8 * q + 4 * end_hh)) =
                        make_uint2(pack_pair<kHalf>(x0, x1), pack_pair<kHalf>(x2, x3));
                }
            asm volatile("" ::: "memory");
            constexpr int kPieceLanes = D / 8;  // lanes of 16 bytes a row
#pragma unroll 2
            for (int base = 0; base < 32; base += 64 / kPieceLanes) {
                const int mine = base + lane_again / kPieceLanes, piece = lane_again % kPieceLanes;
                const int32_t out_row = wave_row0 + mine;
                const uint4 x = *reinterpret_cast<const uint4*>(stage + mine * S::kOPitch + 16 * piece);
                if (out_row < rows) {
                    const int32_t t = out_row / a.group;
                    uint16_t* to = static_cast<uint16_t*>(a.out) + (req.first + t) * a.o_st +
                                   (h * a.group + out_row - t * a.group) * a.o_sh + 8 * piece;
                    if (a.o_wide) {
                        *reinterpret_cast<uint2*>(to) = make_uint2(x.x, x.y);
                        *reinterpret_cast<uint2*>(to + 4) = make_uint2(x.z, x.w);
                    } else {
                        const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            to[2 * j] = (uint16_t)u[j];
                            to[2 * j + 1] = (uint16_t)(u[j] >> 16);
                        }
                    }
                }
            }
        } else if (end_valid) {
            // a worker's first slot holds the tile that came from the one before, its second the one that goes on
            float* slot = a.partials + slot_of(a, h, worker, unit == 0) * slot_floats(D, kWideRows);
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<f32x4_t*>(slot + (32 * wave + end_n) * D + 32 * d + 8 * q + 4 * end_hh) =
                        f32x4_t{acc[d][4 * q], acc[d][4 * q + 1], acc[d][4 * q + 2], acc[d][4 * q + 3]};
            if (end_hh == 0) {
                slot[kWideRows * D + 32 * wave + end_n] = m_run;
                slot[kWideRows * D + kWideRows + 32 * wave + end_n] = l_run;
            }
        }
        left -= cost;
        if (!whole && unit == 0) {
            cut.first_token = req.first;
            cut.first_row = row0;
            cut.rows = rows;
            // the units behind this worker's, dealt out to the next ones
            cut.count = 1 + (w.tiles.units - units + w.each - 1) / w.each;
        }
        if (left > 0) {
            w.at = 0;
            if (++w.tile == w.tiles.count) {
                w.tile = 0;
                do
                    w.tiles = tiles_of(a, ++w.b, kWideRows, kWideKeys);  // there is one: cost is left
                while (w.tiles.count == 0);
            }
            lds_barrier();  // the outputs have left LDS
        }
    }
    if (a.workers > 0 && h == 0 && threadIdx.x == 0)
        a.cut_tiles[worker] = cut;
}

}  // namespace
}  // namespace fgv
