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
// which the first one enters at the first tile that holds one.
#pragma once

namespace fgv {
namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

constexpr int kWideRows = 128;  // query rows of a workgroup
constexpr int kWideKeys = 64;   // keys of a tile, and of a unit

// P times 2^7 and V times 2^-7 use fp16's range better than P, at most 1, and V
// would: P is held to 2^-32.  2^-7 * 0.5 * 2^(111 - 127) is fp16's least value,
// and 2^-7 * 6 * 2^(147 - 127) below its largest.
constexpr int kHalfShift = 7;
__device__ __forceinline__ bool half_holds(uint32_t byte, uint4 codes) {
    const bool zeros = ((codes.x | codes.y | codes.z | codes.w) & 0x77777777u) == 0;
    return (byte - (104u + kHalfShift) <= 36u) | (zeros & (byte != 255u));
}

template <int D, int kPieces>
struct WideShape {
    static constexpr int kChunks = D / 64;                // of 64 dims: one QK instruction per piece
    static constexpr int kVChunks = D < 128 ? 1 : D / 128;  // of 128 dims: 16 bytes of codes a lane
    static constexpr int kVPitch = D == 64 ? 192 : 2 * D + 64;  // four rows of 64 bytes meet no bank twice
    static constexpr int kVBytes = kWideKeys * kVPitch;
    static constexpr int kOPitch = 2 * D + 16;
    static_assert(kAttWaves * 32 * kOPitch <= 2 * kVBytes, "the outputs fit the V buffers");
};

template <int D>
struct WideKeyTile {
    uint4 k[2][D / 64];
    uint32_t ks[2][D / 64];
    uint32_t live;  // which of the four subtiles have a block, bit by bit
};

template <int D>
struct WideValueTile {
    uint4 v[D < 128 ? 1 : D / 128];
    uint32_t vs[D < 128 ? 1 : D / 128];
    int32_t key;  // of the first of the wave's 16 tokens, kNoKey: no block
};

// Codes and scales of the head's subtile `from` of `p`, at its first token.
template <int D>
__device__ __forceinline__ const uint8_t* subtile_at(const AttArgs& a, const Places& p, int from, int32_t& place,
                                                     const uint8_t*& scales) {
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)p.base, from);
    const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)((uint64_t)p.base >> 32), from);
    place = __builtin_amdgcn_readlane(p.place, from);
    // one without a block reads the cache's first one, whose values nobody sees
    const int32_t first = max(place, 0);
    const uint8_t* head = a.cache + (int64_t)((uint64_t)hi << 32 | lo);
    scales = head + mx_part(2, a.page, D) + (int64_t)first * (D / kMxBlock);
    return head + (int64_t)first * (D / 2);
}

template <int D>
__device__ __forceinline__ void load_keys(const AttArgs& a, const Places& p, int tile, int lane, WideKeyTile<D>& out) {
    const int r = lane & 15, h = lane >> 5;
    const bool upper = lane & 16;
    out.live = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const uint8_t *codes[2], *scales[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            int32_t place;
            codes[u] = subtile_at<D>(a, p, (tile & 15) * 4 + 2 * t + u, place, scales[u]);
            out.live |= place >= 0 ? 1u << (2 * t + u) : 0;
        }
        const uint8_t* c = (upper ? codes[1] : codes[0]) + (uint32_t)(r * (D / 2) + 16 * h);
        const uint8_t* s = (upper ? scales[1] : scales[0]) + (uint32_t)(r * (D / kMxBlock) + h);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            out.k[t][i] = *reinterpret_cast<const uint4*>(c + 32 * i);
            out.ks[t][i] = s[2 * i];
        }
    }
}

template <int D>
__device__ __forceinline__ void load_values(const AttArgs& a, const Places& p, int tile, int wave, int lane, int32_t key0,
                                            WideValueTile<D>& out) {
    const int r = lane & 15, g = D < 128 ? (lane >> 4) & 1 : lane >> 4;
    int32_t place;
    const uint8_t* scales;
    const uint8_t* codes = subtile_at<D>(a, p, (tile & 15) * 4 + wave, place, scales);
    out.key = place >= 0 ? key0 + 16 * wave : kNoKey;
    codes += mx_part(1, a.page, D);
    scales += (int64_t)a.page * (D / kMxBlock);
#pragma unroll
    for (int c = 0; c < (D < 128 ? 1 : D / 128); ++c) {
        out.v[c] = *reinterpret_cast<const uint4*>(codes + (uint32_t)(r * (D / 2) + 64 * c + 16 * g));
        out.vs[c] = scales[(uint32_t)(r * (D / kMxBlock) + 4 * c + g)];
    }
}

// The query rows as the B operand: piece p of 64 dims c in step p * kChunks + c.
// The first kHeld pieces stay in registers; the others, of fp16 calls, which would
// be too many for them, in LDS.
template <int D, int kPieces>
struct WideQuery {
    static constexpr int kHeld = kPieces == 2 ? 2 : D == 256 ? 1 : 2;
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

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

template <int D, int kPieces>
__global__ void __launch_bounds__(kAttThreads, D == 256 ? 1 : 2) mxfp4_attend_wide_kernel(AttArgs a) {
    using S = WideShape<D, kPieces>;
    constexpr bool kHalf = kPieces == 3;
    __shared__ __align__(16) uint8_t turned[2][S::kVBytes];
    __shared__ __align__(16) uint32_t held_by[2][kAttWaves];  // whether fp16 holds each wave's values
    __shared__ uint64_t nan_of[2][kAttWaves][S::kVChunks];    // which of its value blocks are NaN, bit by lane
    using Rows = WideQuery<D, kPieces>;
    __shared__ uint4 more_query[kAttWaves][Rows::kInLds ? 64 * Rows::kInLds : 1];  // the pieces not in registers
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, hh = lane >> 5, r = lane & 15, g = lane >> 4;
    const int h = (int)blockIdx.x % a.kv_heads;
    const int32_t worker = (int32_t)(blockIdx.x / a.kv_heads);
    const int32_t tile_cost = a.workers > 0 ? kTileCost : 0;
    // where this lane writes its 16-byte pieces of V, rotated so that the lanes of a write meet
    // no bank twice, and where it reads them turned
    const int turn = r >> 2;
    uint32_t write_at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        write_at[i] = (uint32_t)((16 * wave + r) * S::kVPitch + 64 * g + 16 * ((i + turn) & 3));
    const uint32_t read_at = (uint32_t)((4 * hh + (r >> 2)) * S::kVPitch + 32 * ((lane >> 4) & 1) + 8 * (lane & 3));

    Start w;
    const bool busy = find_start(a, worker, kWideRows, kWideKeys, w);
    CutTile cut = {0, 0, 0, 0};  // the tile that begins here and goes on with the next workers
    int32_t left = busy ? w.take : 0;
    while (left > 0) {
        const Request req = w.tiles.req;
        const int32_t cost = min(left, w.tiles.cost(a) - w.at);
        const int32_t unit = max(w.at - tile_cost, 0);
        const int32_t units = a.workers > 0 ? max(w.at + cost - tile_cost, 0) - unit : 1;
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
        int32_t begin, end;
        key_range(a, req, begin, end);
        if (!whole) {
            begin += unit * kWideKeys;  // below the request's end
            end = units <= (end - begin) / kWideKeys ? begin + units * kWideKeys : end;
        }
        end = min(end, last_pos + 1);
        begin = max(begin, max(any.first, 0) & ~(kTileKeys - 1));
        const int32_t tiles = end > begin ? (end - begin + kWideKeys - 1) / kWideKeys : 0;

        RawWideQuery<D> raw_query;
        load_wide_query<D>(a, (req.first + token) * a.q_st + head * a.q_sh, valid, hh, raw_query);
        Places places = find_places<4>(a, w.b, h, mx_token_bytes(D), begin, kWideKeys, end, lane);
        WideKeyTile<D> keys;
        WideValueTile<D> now, next;
        keys.live = 0;
        if (tiles > 0) {
            load_keys<D>(a, places, 0, lane, keys);
            load_values<D>(a, places, 0, wave, lane, begin, now);
            next = now;
            if (tiles > 1)
                load_values<D>(a, places, 1, wave, lane, begin + kWideKeys, next);
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

        // A token that no row sees may hold anything: its values are taken as finite.
        auto look = [&](WideValueTile<D>& t, int buffer) {
            bool held = true;
#pragma unroll
            for (int c = 0; c < S::kVChunks; ++c) {
                t.vs[c] = any(t.key + r) ? t.vs[c] : 127;
                held = held & half_holds(t.vs[c], t.v[c]);
            }
            const bool all = __all(held);
            if (lane == 0)
                held_by[buffer][wave] = all;
        };
        auto all_held = [&](int buffer) {
            const uint4 f = *reinterpret_cast<const uint4*>(held_by[buffer]);
            return __builtin_amdgcn_readfirstlane(f.x & f.y & f.z & f.w) != 0;
        };

        auto step = [&](auto kind, int32_t i) {
            constexpr bool kFast = decltype(kind)::value;
            constexpr int kPPieces = kFast && kPieces == 2 ? 1 : 2;
            const int buffer = i & 1;
            const int32_t key = begin + i * kWideKeys;
            // ---- this tile's V into LDS; whether the next one's can go as fp16
            asm volatile("" ::: "memory");
#pragma unroll
            for (int c = 0; c < S::kVChunks; ++c) {
                uint32_t byte = now.vs[c];
                if constexpr (kFast) {
                    byte = max(byte, (uint32_t)kHalfShift) - kHalfShift;
                } else {
                    const uint64_t nan = __ballot(byte == 255u);
                    if (lane == 0)
                        nan_of[buffer][wave][c] = nan;
                    byte = byte == 255u ? 0 : byte;
                }
                const float scale = __uint_as_float(byte << 23);
                uint4 q = now.v[c];
                q = turn & 1 ? make_uint4(q.y, q.z, q.w, q.x) : q;
                q = turn & 2 ? make_uint4(q.z, q.w, q.x, q.y) : q;
                if (D >= 128 || g < 2) {
                    uint8_t* to = turned[buffer] + 256 * c;
                    *reinterpret_cast<uint4*>(to + write_at[0]) = wide_values<kFast>(q.x, scale);
                    *reinterpret_cast<uint4*>(to + write_at[1]) = wide_values<kFast>(q.y, scale);
                    *reinterpret_cast<uint4*>(to + write_at[2]) = wide_values<kFast>(q.z, scale);
                    *reinterpret_cast<uint4*>(to + write_at[3]) = wide_values<kFast>(q.w, scale);
                }
            }
            now = next;
            look(now, buffer ^ 1);
            asm volatile("" ::: "memory");

            // ---- scores
            const bool active = (key <= wave_last) & ((a.window == 0) | (key + kWideKeys > wave_first - a.window + 1));
            f32x16_t s[2];
            if (active) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        s[t][j] = 0.f;
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
                    for (int t = 0; t < 2; ++t)
                        s[t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(key_operand(keys.k[t][c]), rows_q, s[t], 4,
                                                                               0, 0, (int)keys.ks[t][c], 0,
                                                                               piece_scale(query.scale, piece));
                }
                const bool plain = (key + kWideKeys - 1 <= min(wave_first, end - 1)) &
                                   ((a.window == 0) | (key > wave_last - a.window)) & (keys.live == 15u);
                if (!plain) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const int32_t base = keys.live >> (2 * t + u) & 1 ? key + 32 * t + 16 * u : kNoKey;
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                s[t][8 * u + j] =
                                    seen(base + 8 * (j / 4) + 4 * hh + j % 4) ? s[t][8 * u + j] : -INFINITY;
                        }
                }
                float most = -INFINITY;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        most = fmaxf(most, s[t][j]);
                most = pair_max(most) * a.scale_f;
                if (__any(most > m_run)) {
                    const float m_new = most > m_run ? most + kAhead : m_run;
                    const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
                    l_run *= alpha;
#pragma unroll
                    for (int d = 0; d < D / 32; ++d)
                        acc[d] *= alpha;
                    m_run = m_new;
                }
            }
            // ---- the next tile of K, and the one after it of V
            if (i + 1 < tiles)
                load_keys<D>(a, places, i + 1, lane, keys);
            if (i + 2 < tiles) {
                if (((i + 2) & 15) == 0)
                    places = find_places<4>(a, w.b, h, mx_token_bytes(D), key + 2 * kWideKeys, kWideKeys, end, lane);
                load_values<D>(a, places, i + 2, wave, lane, key + 2 * kWideKeys, next);
            }
            uint4 pw[kPPieces][4];  // by 16 keys: keys 4h..4h+3 and 8+4h..8+4h+3 of them
            if (active) {
                const float m_use = (m_run == -INFINITY ? 0.f : m_run) - (kFast ? (float)kHalfShift : 0.f);
                const bool far = __any(fabsf(m_use) > kFar);
                float sum = 0.f;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    float p[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        p[j] = __builtin_fmaf(s[t][j], a.scale_f, -m_use);
                    if (far) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            p[j] = s[t][j] * a.scale_f - m_use;
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        p[j] = __builtin_amdgcn_exp2f(p[j]);
                        sum += p[j];
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const float* x = p + 8 * u;
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            hi[j] = pack_pair<kFast>(x[2 * j], x[2 * j + 1]);
                            lo[j] = kPPieces == 2 ? pack_pair<kFast>(x[2 * j] - first_of<kFast>(hi[j]),
                                                                     x[2 * j + 1] - second_of<kFast>(hi[j]))
                                                  : 0;
                        }
                        pw[0][2 * t + u] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        if constexpr (kPPieces == 2)
                            pw[1][2 * t + u] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                }
                l_run += kFast ? sum * (1.0f / (1 << kHalfShift)) : sum;
            }
            lds_barrier();
            if (active) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint8_t* from = turned[buffer] + read_at + 16 * u * S::kVPitch;
                    uint4 v[D / 32];
#pragma unroll
                    for (int d = 0; d < D / 32; ++d) {
                        const uint2 x = read_turned(from + 64 * d), y = read_turned(from + 8 * S::kVPitch + 64 * d);
                        v[d] = make_uint4(x.x, x.y, y.x, y.y);
                    }
#pragma unroll
                    for (int q = 0; q < kPPieces; ++q)
#pragma unroll
                        for (int d = 0; d < D / 32; ++d)
                            acc[d] = wide_product<kFast>(v[d], pw[q][u], acc[d]);
                }
                if constexpr (!kFast) {
                    // value blocks that are NaN, for the rows that see them
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int c = 0; c < S::kVChunks; ++c) {
                            const uint64_t nan = nan_of[buffer][u][c];
                            const uint32_t half[2] = {(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)nan),
                                                      (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(nan >> 32))};
#pragma unroll
                            for (int b = 0; b < (D < 128 ? 2 : 4); ++b) {
                                float add = 0.f;
                                for (uint32_t bits = half[b / 2] >> (16 * (b & 1)) & 0xffffu; bits; bits &= bits - 1)
                                    add = seen(key + 16 * u + __builtin_ctz(bits)) ? NAN : add;
                                acc[4 * c + b] += add;
                            }
                        }
                }
            }
        };

        if (tiles > 0) {
            look(now, 0);
            lds_barrier();
            int32_t i = 0;
            for (; i < tiles && all_held(i & 1); ++i)
                step(Yes{}, i);
            for (; i < tiles; ++i)
                step(No{}, i);
        }

        l_run += __shfl_xor(l_run, 32);
        lds_barrier();  // V was read
        if (whole) {
            const RowEnd e = finish_row(a, head, m_run, l_run);
            if (valid && hh == 0)
                a.lse[(req.first + token) * a.lse_st + head] = e.lse;
            // through LDS, so that whole rows are written: the wave's 32 rows in its own quarter
            uint8_t* stage = &turned[0][0] + wave * 32 * S::kOPitch;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float x0 = acc[d][4 * q] * e.inv, x1 = acc[d][4 * q + 1] * e.inv;
                    const float x2 = acc[d][4 * q + 2] * e.inv, x3 = acc[d][4 * q + 3] * e.inv;
                    *reinterpret_cast<uint2*>(stage + n * S::kOPitch + 2 * (32 * d + 8 * q + 4 * hh)) =
                        make_uint2(pack_pair<kHalf>(x0, x1), pack_pair<kHalf>(x2, x3));
                }
            asm volatile("" ::: "memory");
            constexpr int kPieceLanes = D / 8;  // lanes of 16 bytes a row
#pragma unroll 2
            for (int base = 0; base < 32; base += 64 / kPieceLanes) {
                const int mine = base + lane / kPieceLanes, piece = lane % kPieceLanes;
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
        } else if (valid) {
            // a worker's first slot holds the tile that came from the one before, its second the one that goes on
            float* slot = a.partials + slot_of(a, h, worker, unit == 0) * slot_floats(D, kWideRows);
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<f32x4_t*>(slot + (32 * wave + n) * D + 32 * d + 8 * q + 4 * hh) =
                        f32x4_t{acc[d][4 * q], acc[d][4 * q + 1], acc[d][4 * q + 2], acc[d][4 * q + 3]};
            if (hh == 0) {
                slot[kWideRows * D + 32 * wave + n] = m_run;
                slot[kWideRows * D + kWideRows + 32 * wave + n] = l_run;
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
