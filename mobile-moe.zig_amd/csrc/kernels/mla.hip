// Attention of single tokens over the paged latent cache (mlaAttention's
// cached part, inference.zig:539-660) on gfx950: for every token and head,
// out = sum_p softmax_p(scale (q . c_p + q_pe . k_p)) c_p over the rows (c, k)
// that the token's page table names. One pass over the rows with the running
// maximum and sum of the softmax; all heads of a token share the read rows.
//
// A row of 512 + 64 values is 1152 B in f16 (612 B in Q8_0) and costs 2 x 20 x
// 1088 operations. The matrix work is more than that: the f32 operand of each
// product enters as two f16 parts (all 24 bits; the cached values are exact in
// f16), and heads come in tiles of 16. From 17 to 24 heads the second tile holds
// up to 8 heads' high parts in its first half and their low parts in the other,
// one product in place of two (kPacked; at 20 heads against two full tiles: 64
// ragged contexts in Q8_0 56 us against 59, a chunk of 256 tokens 161 against
// 168, f16 contexts alike).
//
// What bounds it: with long contexts in f16, HBM (131072 positions of one token
// 38 us, 4.0 TB/s, and 13 for the join of its pieces; 64 times 4096 73 us, 4.1
// TB/s). Otherwise a wave's chain through a tile, about 5000 cycles with two
// workgroups on a CU: 64 ragged contexts up to 16384 in Q8_0 43 to 55 us by their
// lengths, 256 tokens over the same 4096 positions in f16 162 to 168 us, in Q8_0 223
// (f16: matrix cores busy 31% of the time, LDS 42%). One short context: two
// launches, 16 us.
//
// A workgroup is four waves and takes tiles of 32 positions. Wave w owns the
// latent columns 128 w .. 128 w + 127 and 16 of the rotary ones, both as keys
// and as values, so cached data never crosses waves: a wave stages its slice
// of the next tile in registers while it works on the current one, and keeps
// it in its own part of LDS, from which it is read as keys in rows and as
// values transposed (ds_read_b64_tr_b16). Per tile:
//   S^T partial = K Q^T over the wave's columns     (rows are positions)
//   exchange: the four partials are added, each wave takes a quarter of the
//             heads through the softmax and leaves P
//   O^T += V^T P^T for the wave's columns           (rows are columns)
// with two barriers. S^T leaves the matrix cores with four consecutive
// positions per lane, and P is stored in the order in which O^T's operand takes
// positions, so both are 16-byte accesses.
//
// Q8_0: codes become f16 integers on their way to LDS. A score is summed block
// by block, each block's product times the position's block scale. In O the
// values are scaled: d * code has 19 bits, its f16 rounding and the rest (an
// FMA away) are both exact, one vector instruction per value for both. (The
// rest times P's lower part, 2^-24 of the product at most, is left out. The
// scale folded into P instead costs three per head tile and value.) From scales
// of 2^9 on d * code can pass f16's range. Such blocks count as 0 in these
// products and are taken in a second round, only by tiles that have any, with
// 2^-9 d, which is as exact; so no scale costs another block or position any bits.
//
// Work is cut evenly, whatever the lengths: the tiles of all tokens and head
// tiles form one list, of which every workgroup takes an equal run, two
// workgroups per CU (one: 64 ragged contexts in Q8_0 69 us instead of 57). A run
// may end inside a token; such pieces leave their sums in the workspace and
// mla_join_kernel adds them in the list's order.
#include "device_common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"

namespace mmhip {

namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

constexpr int kMlaThreads = 256, kMlaWaves = 4;
constexpr uint32_t kMlaTile = 32;       // positions per tile
constexpr uint32_t kMlaCols = 128;      // latent columns per wave
constexpr uint32_t kMlaPe = 16;         // rotary columns per wave
constexpr uint32_t kSpLd = 36;          // floats between rows of the score partials (16-byte rows)
constexpr float kPScale = 32768.0f;     // P in [0, 1] uses f16's upper range: parts down to 2^-39 survive
constexpr int kJoinThreads = 1024;

// A begun and unfinished item of a workgroup: the item, and how many pieces it
// has (this workgroup's and the first ones of the following); pieces 0: none.
struct MlaSplit {
    uint32_t item, pieces;
};

// Heads per head tile: one product tile of 16, two, or one and a packed one.
enum MlaMode : int { kOne = 0, kTwo = 1, kPacked = 2 };
constexpr int mode_tiles(int mode) { return mode == kOne ? 1 : 2; }
constexpr uint32_t mode_rows(int mode) { return mode == kOne ? 16 : mode == kTwo ? 32 : 24; }

template <bool Q8, int MODE>
struct MlaLds {
    static constexpr int NT = mode_tiles(MODE);
    uint8_t kv[kMlaWaves][kMlaTile * 256];  // f16 [position][128], 16-byte chunks swizzled by the position
    uint8_t pe[kMlaWaves][kMlaTile * 32];   // f16 [position][16]
    float sp[kMlaWaves][mode_rows(MODE)][kSpLd];  // score partials
    // P: f16 in rows of 40 (per tile high parts, low parts; packed as it is)
    uint32_t p[(MODE == kTwo ? 4 : MODE == kPacked ? 3 : 2) * 16 * 20];
    float ds[Q8 ? kMlaWaves : 1][5][kMlaTile];  // block scales of the keys
    uint16_t dv[Q8 ? kMlaWaves : 1][4][kMlaTile];  // of the values, in f16: those below 2^9,
    uint16_t db[Q8 ? kMlaWaves : 1][4][kMlaTile];  // and the others times 2^-9
    float alpha[16 * NT], factor[16 * NT], qmax[kMlaWaves][16 * NT];
    float2 ml[16 * NT];
    uint64_t scan[kMlaWaves];
    uint64_t start_off;
    uint32_t start_token, start_row, start_len;
};

__device__ __forceinline__ uint32_t tiles_of(uint32_t len) { return (uint32_t)(((uint64_t)len + kMlaTile - 1) / kMlaTile); }
// An item's slots of the list that is cut evenly: its tiles, behind slots that
// stand for its queries' conversion and its result. (64 ragged contexts 57 us
// instead of 71. Equal lengths lose: 64 times 4096, whose pieces ended with the
// sequences before, 76 instead of 71, and one token at 131072 positions has runs
// of 9 tiles where 8 would do.)
constexpr uint32_t kItemSlots = 3;
__device__ __forceinline__ uint32_t slots_of(uint32_t len) { return len ? tiles_of(len) + kItemSlots : 0; }

__device__ __forceinline__ uint32_t seen(const MlaArgs& a, uint32_t t, uint32_t& row, uint32_t& bad) {
    row = a.table_of ? a.table_of[t] : t;
    return paged_seen(a.geom, a.lens[t], row, a.n_tables, a.table_pages, bad);
}

// Two codes (bytes i, i + 1 of u = code + 128) as f16 integers: 0x6400 | u is
// 1024 + u.
__device__ __forceinline__ uint32_t codes2(uint32_t u, uint32_t sel) {
    const uint32_t h = __builtin_amdgcn_perm(0x64646464u, u, sel);
    const v2h v = __builtin_bit_cast(v2h, h) - (v2h){(_Float16)1152.0f, (_Float16)1152.0f};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint4 codes8(uint32_t a, uint32_t b) {
    const uint32_t x = a ^ 0x80808080u, y = b ^ 0x80808080u;
    return make_uint4(codes2(x, 0x04010400u), codes2(x, 0x04030402u), codes2(y, 0x04010400u), codes2(y, 0x04030402u));
}

// Two values as f16 parts, both rounded to nearest: what hi leaves is at most
// half a step of 11 bits, with a sign, on the grid of 24, so lo holds it and
// hi + lo is the value, down to f16's smallest step (2^-24; half of one is lost).
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const v2h h = __builtin_convertvector((v2f){a, b}, v2h);
    const v2h l = __builtin_convertvector((v2f){a - (float)h[0], b - (float)h[1]}, v2h);
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}

__device__ __forceinline__ v8h half8(const uint4& v) { return __builtin_bit_cast(v8h, v); }

// A value that is the same in all lanes, in scalar registers from here on.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t uniform(uint64_t v) {
    return (uint64_t)uniform((uint32_t)(v >> 32)) << 32 | uniform((uint32_t)v);
}

// A lane-dependent value that the compiler takes as new here: what follows
// from it is computed again where it is used, not kept in registers over the
// loop around (registers that run out would go to scratch memory, whose loads
// wait for every row load in flight).
__device__ __forceinline__ uint32_t afresh(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}

// 2^e, e within f32's normal exponents.
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <bool Q8, int MODE, bool FULL, int POL>
__global__ __launch_bounds__(kMlaThreads, 2) void mla_split_kernel(MlaArgs a, MlaPlan pl) {
    constexpr int NT = mode_tiles(MODE);       // product tiles of 16 columns
    constexpr uint32_t kHeads = mode_rows(MODE);
    __shared__ __align__(256) MlaLds<Q8, MODE> s;
    const PagedGeom g = a.geom;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t wg = blockIdx.x;
    MlaSplit* const splits = reinterpret_cast<MlaSplit*>(pl.splits);

    // ---- this workgroup's run of the list ----
    uint64_t f, end, total, off;
    uint64_t chunk;
    uint32_t token, row, len;
    const auto cut = [&] {
        // (a 64-bit division is some 150 instructions)
        chunk = total < 0x80000000u ? ((uint32_t)total + pl.groups - 1) / pl.groups : (total + pl.groups - 1) / pl.groups;
        // Up to three slots, one workgroup per CU is enough: fewer pieces to join.
        // (One token at 12288 positions 21.7 us instead of 27.2, at 24576 25.3
        // instead of 30.0, four at 4096 22.2 instead of 24.0; with four slots
        // eight at 4096 take 31.0 instead of 30.2.)
        const uint64_t least = total <= pl.groups / 2 ? 1 : total <= pl.groups ? 2 : 3;
        if (chunk < least) chunk = least;
        f = wg * chunk;
        end = f + chunk < total ? f + chunk : total;
    };
    if (a.n_tokens <= 64) {
        // Every wave finds it for itself.
        uint32_t bad, my_row = 0, my_len = 0;
        if (lane < a.n_tokens) my_len = seen(a, lane, my_row, bad);
        const uint64_t mine = (uint64_t)slots_of(my_len) * pl.head_tiles, incl = wave_scan(mine);
        total = lane_value(incl, 63);
        cut();
        const uint64_t here = __ballot(incl - mine <= f && f < incl);
        token = here ? __builtin_ctzll(here) : a.n_tokens;
        const uint32_t at = here ? token : 0;
        row = __builtin_amdgcn_readlane(my_row, at);
        len = __builtin_amdgcn_readlane(my_len, at);
        off = f - lane_value(incl - mine, at);
    } else {
        const uint32_t per = (a.n_tokens + kMlaThreads - 1) / kMlaThreads;
        const uint64_t t0 = (uint64_t)tid * per;
        uint64_t mine = 0;
        uint32_t last_row = 0, last_len = 0;
        for (uint64_t t = t0; t < t0 + per && t < a.n_tokens; ++t) {
            uint32_t bad;
            last_len = seen(a, (uint32_t)t, last_row, bad);
            mine += slots_of(last_len);
        }
        mine *= pl.head_tiles;
        uint64_t incl = wave_scan(mine);
        if (lane == 63) s.scan[wave] = incl;
        __syncthreads();
        total = 0;
        uint64_t before = 0;
#pragma unroll
        for (uint32_t w = 0; w < kMlaWaves; ++w) {
            if (w < wave) before += s.scan[w];
            total += s.scan[w];
        }
        incl += before;
        total = uniform(total);
        cut();
        if (f < end && incl - mine <= f && f < incl) {
            uint64_t at = incl - mine;
            uint32_t t = (uint32_t)t0, row = last_row, len = last_len;
            if (per > 1) {
                uint32_t bad;
                for (;; ++t) {
                    len = seen(a, t, row, bad);
                    const uint64_t n = (uint64_t)slots_of(len) * pl.head_tiles;
                    if (f < at + n || t + 1 >= a.n_tokens) break;
                    at += n;
                }
            }
            s.start_token = t;
            s.start_row = row;
            s.start_len = len;
            s.start_off = f - at;
        }
        __syncthreads();
        token = uniform(s.start_token);
        row = uniform(s.start_row);
        len = uniform(s.start_len);
        off = uniform(s.start_off);
    }
    MlaSplit begun{0, 0};

    const uint32_t row_bytes = Q8 ? g.width : 2 * g.width, at_mask = (1u << g.page_shift) - 1;
    const uint32_t blocks = FULL ? 4u : (g.rank / 32 > 4 * wave ? min(g.rank / 32 - 4 * wave, 4u) : 0u);
    const bool has_pe = FULL || kMlaPe * wave < g.width - g.rank;

    uint32_t of_token = token;
    while (f < end && token < a.n_tokens) {
        if (token != of_token) {
            uint32_t bad;
            len = seen(a, token, row, bad);
            of_token = token;
        }
        len = uniform(len);
        row = uniform(row);
        const uint32_t n_tiles = tiles_of(len);
        if (n_tiles == 0) {
            ++token;
            continue;
        }
        const uint32_t n_slots = n_tiles + kItemSlots;
        const uint32_t ht_index = pl.head_tiles == 1 ? 0u : (uint32_t)(off / n_slots);
        const uint32_t slot0 = (uint32_t)(off - (uint64_t)ht_index * n_slots);
        const uint32_t span = (uint32_t)(end - f < n_slots - slot0 ? end - f : n_slots - slot0);
        const uint32_t tile0 = max(slot0, kItemSlots) - kItemSlots;
        const uint32_t count = max(slot0 + span, kItemSlots) - kItemSlots - tile0;
        const auto advance = [&] {
            f += span;
            off += span;
            if (off == (uint64_t)n_slots * pl.head_tiles) {
                off = 0;
                ++token;
            }
        };
        if (count == 0) {
            advance();
            continue;
        }
        const uint32_t head0 = ht_index * kHeads;
        const int32_t* table = a.tables + (uint64_t)row * a.table_stride;

        // ---- loads of a tile: page numbers one tile before its rows ----
        // None stands under a branch, past the piece's last tile neither: where
        // a register is loaded on one way and kept on the other, the ways'
        // meeting point waits for the load. Rows that are not wanted have an
        // empty resource (no memory is touched); the few other bytes are read.
        int32_t id[2];
        auto load_ids = [&](uint32_t tile) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t p = min(tile, n_tiles - 1) * kMlaTile | 16 * h;
                id[h] = table[min(p, len - 1) >> g.page_shift];
            }
        };
        uint4 pre[Q8 ? 4 : 8], pre_pe;
        uint2 pre_d;
        uint32_t pre_dpe = 0, live = 0;
        bool lost = false;  // a page that the pool does not have
        pre_pe = make_uint4(0, 0, 0, 0);
        pre_d = make_uint2(0, 0);
        auto load_rows = [&](uint32_t tile, bool wanted) {
            const uint32_t lane = afresh(tid & 63), n16 = lane & 15, grp = lane >> 4;
            BufRsrc rows[2];
            const uint8_t *base[2], *base_d[2];
            live = 0;
            const uint32_t p0 = tile * kMlaTile;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int32_t page = (int32_t)uniform((uint32_t)id[h]);
                const uint32_t p = p0 + 16 * h;
                const bool want = p < len, ok = want && paged_has(g, page);
                live |= ok ? 0xFFFFu >> (16 - min(len - p, 16u)) << (16 * h) : 0;
                lost |= want && !ok;
                // 16 rows from p on. A page that is not there is read as page 0
                // and left out.
                base[h] = a.pool + paged_row(g, ok ? (uint32_t)page : 0u, p & at_mask);
                rows[h] = make_rsrc(base[h], wanted ? 16 * row_bytes : 0);
                if constexpr (Q8) base_d[h] = a.pool + paged_scales(g, ok ? (uint32_t)page : 0u, p & at_mask);
            }
            if (FULL || blocks) {
                // A lane's 16 bytes of the wave's columns (past the columns
                // there are: the last ones again).
                const uint32_t at_rows = Q8 ? (lane >> 3) * row_bytes + wave * kMlaCols + 16 * (FULL ? lane & 7 : min(lane & 7, 2 * blocks - 1))
                                            : grp * row_bytes + wave * (2 * kMlaCols) + 16 * (FULL ? n16 : min(n16, 4 * blocks - 1));
#pragma unroll
                for (int j = 0; j < (Q8 ? 4 : 8); ++j) {
                    if constexpr (Q8) pre[j] = buf_load_b128<POL>(rows[j >> 1], at_rows, 8 * (j & 1) * row_bytes);
                    else pre[j] = buf_load_b128<POL>(rows[j >> 2], at_rows, 4 * (j & 3) * row_bytes);
                }
            }
            if constexpr (Q8) {
                // A position per lane, twice over.
                const uint8_t* d = (lane & 16 ? base_d[1] : base_d[0]) + n16 * (g.width / 32 * 2);
                if constexpr (FULL) {
                    pre_d.x = reinterpret_cast<const uint32_t*>(d + wave * 8)[0];
                    pre_d.y = reinterpret_cast<const uint32_t*>(d + wave * 8)[1];
                } else if (blocks) {
                    uint32_t v[4];
#pragma unroll
                    for (uint32_t b = 0; b < 4; ++b) v[b] = reinterpret_cast<const uint16_t*>(d + wave * 8)[min(b, blocks - 1)];
                    pre_d = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
                }
                if (has_pe) {
                    pre_pe = *reinterpret_cast<const uint4*>((lane & 16 ? base[1] : base[0]) + n16 * row_bytes + g.rank + wave * kMlaPe);
                    // Two blocks' scales in a word, picked from when they are
                    // used: widening a 16-bit load waits for it right here.
                    if constexpr (FULL) pre_dpe = *reinterpret_cast<const uint32_t*>(d + 32);
                    else pre_dpe = *reinterpret_cast<const uint16_t*>(d + (g.rank / 32 + wave / 2) * 2);
                }
            } else if (has_pe) {
                pre_pe = *reinterpret_cast<const uint4*>((lane & 32 ? base[1] : base[0]) + ((lane >> 1) & 15) * row_bytes +
                                                         2 * g.rank + wave * (2 * kMlaPe) + (lane & 1) * 16);
            }
        };

        // The wave's slice of the tile in registers -> LDS, in f16. Positions
        // that count for nothing (past the length, on a page that is not
        // there) become zeros: their bytes may be anything.
        uint8_t* const kv = s.kv[wave];
        uint32_t mask = 0;
        v4f o[8][NT];
        uint32_t big = 0;  // Q8_0: positions with block scales of 2^9 and more, NaN among them
        auto stage = [&]() {
            const uint32_t lane = afresh(tid & 63);
            mask = live;
            if constexpr (Q8) {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {  // row 8 j + lane / 8
                    uint8_t* dst = kv + 2048 * j;
                    const uint32_t at = (lane >> 3) * 256 + (((lane >> 3) ^ 2 * (lane & 7)) << 4) ^ (j & 1) << 7;
                    *reinterpret_cast<uint4*>(dst + at) = codes8(pre[j].x, pre[j].y);
                    *reinterpret_cast<uint4*>(dst + (at ^ 16)) = codes8(pre[j].z, pre[j].w);
                }
                const uint32_t p = lane & 31;
                float d[5];
                d[0] = f16_scale((uint16_t)(pre_d.x & 0xFFFFu));
                d[1] = f16_scale((uint16_t)(pre_d.x >> 16));
                d[2] = f16_scale((uint16_t)(pre_d.y & 0xFFFFu));
                d[3] = f16_scale((uint16_t)(pre_d.y >> 16));
                d[4] = f16_scale((uint16_t)(FULL ? pre_dpe >> (wave / 2 * 16) : pre_dpe));
                // (the two highest bits of the exponent)
                uint32_t d01 = pre_d.x, d23 = pre_d.y;
                const uint32_t b01 = d01 & d01 << 1 & 0x40004000u, b23 = d23 & d23 << 1 & 0x40004000u;
                big = uniform((uint32_t)__ballot(b01 | b23) & mask);
                if (big) {
                    const uint32_t m01 = (b01 >> 14) * 0xFFFFu, m23 = (b23 >> 14) * 0xFFFFu;
                    const v2h f = {(_Float16)0x1p-9f, (_Float16)0x1p-9f};
                    const uint32_t s01 = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, d01 & m01) * f);
                    const uint32_t s23 = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, d23 & m23) * f);
                    d01 &= ~m01;
                    d23 &= ~m23;
                    if (lane < 32) {
                        s.db[wave][0][p] = (uint16_t)(s01 & 0xFFFFu);
                        s.db[wave][1][p] = (uint16_t)(s01 >> 16);
                        s.db[wave][2][p] = (uint16_t)(s23 & 0xFFFFu);
                        s.db[wave][3][p] = (uint16_t)(s23 >> 16);
                    }
                }
                if (lane < 32) {
#pragma unroll
                    for (int b = 0; b < 5; ++b) s.ds[wave][b][p] = d[b];
                    s.dv[wave][0][p] = (uint16_t)(d01 & 0xFFFFu);
                    s.dv[wave][1][p] = (uint16_t)(d01 >> 16);
                    s.dv[wave][2][p] = (uint16_t)(d23 & 0xFFFFu);
                    s.dv[wave][3][p] = (uint16_t)(d23 >> 16);
                    *reinterpret_cast<uint4*>(s.pe[wave] + p * 32) = codes8(pre_pe.x, pre_pe.y);
                    *reinterpret_cast<uint4*>(s.pe[wave] + p * 32 + 16) = codes8(pre_pe.z, pre_pe.w);
                }
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {  // row 4 j + lane / 16
                    const uint32_t at = (lane >> 4) * 256 + (((lane >> 4) ^ (lane & 15)) << 4) ^ (j & 3) << 6;
                    *reinterpret_cast<uint4*>(kv + 1024 * j + at) = pre[j];
                }
                *reinterpret_cast<uint4*>(s.pe[wave] + lane * 16) = pre_pe;
            }
            // The slice is read back through other types, by this wave alone.
            asm volatile("" ::: "memory");
            if (mask != 0xFFFFFFFFu) {  // two lanes clear a row
                const uint32_t p = lane >> 1;
                if (!((mask >> p) & 1)) {
                    const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(kv + p * 256 + (lane & 1) * 128 + 16 * j) = zero;
                    *reinterpret_cast<uint4*>(s.pe[wave] + lane * 16) = zero;
                    if constexpr (Q8) {
#pragma unroll
                        for (int b = 0; b < 5; ++b) {
                            s.ds[wave][b][p] = 0.0f;
                            if (b < 4) s.dv[wave][b][p] = s.db[wave][b][p] = 0;
                        }
                    }
                }
                asm volatile("" ::: "memory");
            }
        };

        load_ids(tile0);
        load_rows(tile0, true);
        load_ids(tile0 + 1);

        // ---- the queries, scaled by a power of two per head, in two parts ----
        // (packed tile: each lane has the part of its half)
        v8h qh[NT][4], ql[MODE == kTwo ? 2 : 1][4];
        // The 16 rotary columns fill one product of 32: their keys stand twice,
        // against the high parts and the low parts. (Products of 16 and of 32
        // on one accumulator, one right after the other, lost the earlier sum.)
        v8h pe2[NT];
        {
            // Every load is issued whether its head exists or not (the last
            // head's again, zeroed below): a load under a branch would be
            // waited for at the branch's end, together with the rows.
            float q[NT][4][8], pe[NT][8];
            const float *src[NT], *src_pe[NT];
            // The head (of the head tile) behind column n16 of product tile t; in
            // a packed tile column 8 + k has head k's low parts.
            const uint32_t ln = afresh(lane), n16 = ln & 15, grp = ln >> 4;
            const bool low_half = n16 >= 8;
            const auto head_of = [&](int t) { return MODE == kPacked && t == 1 ? 16 + (n16 & 7) : 16 * t + n16; };
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint32_t h = min(head0 + head_of(t), a.n_heads - 1);
                src[t] = a.q + (uint64_t)token * a.q_token_stride + (uint64_t)h * a.q_head_stride + wave * kMlaCols + 8 * grp;
                src_pe[t] = a.q_pe + (uint64_t)token * a.q_pe_token_stride + (uint64_t)h * a.q_pe_head_stride + wave * kMlaPe + 8 * (grp & 1);
                if (!FULL) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) pe[t][e] = 0.0f;
#pragma unroll
                    for (int b = 0; b < 4; ++b)
#pragma unroll
                        for (int e = 0; e < 8; ++e) q[t][b][e] = 0.0f;
                }
            }
            if (pl.vec_q) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (uint32_t b = 0; b < 4; ++b) {
                        if (!FULL && b >= blocks) continue;
                        const float4 x = *reinterpret_cast<const float4*>(src[t] + 32 * b);
                        const float4 y = *reinterpret_cast<const float4*>(src[t] + 32 * b + 4);
                        q[t][b][0] = x.x, q[t][b][1] = x.y, q[t][b][2] = x.z, q[t][b][3] = x.w;
                        q[t][b][4] = y.x, q[t][b][5] = y.y, q[t][b][6] = y.z, q[t][b][7] = y.w;
                    }
                    if (has_pe) {
                        const float4 x = *reinterpret_cast<const float4*>(src_pe[t]);
                        const float4 y = *reinterpret_cast<const float4*>(src_pe[t] + 4);
                        pe[t][0] = x.x, pe[t][1] = x.y, pe[t][2] = x.z, pe[t][3] = x.w;
                        pe[t][4] = y.x, pe[t][5] = y.y, pe[t][6] = y.z, pe[t][7] = y.w;
                    }
                }
            } else {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (uint32_t b = 0; b < 4; ++b) {
                        if (!FULL && b >= blocks) continue;
#pragma unroll
                        for (int e = 0; e < 8; ++e) q[t][b][e] = src[t][32 * b + e];
                    }
                    if (has_pe) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) pe[t][e] = src_pe[t][e];
                    }
                }
            }
            // The first tile goes to LDS and the second is asked for before
            // the queries are waited for.
            stage();
            load_rows(tile0 + 1, count > 1);
            load_ids(tile0 + 2);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const bool there = head0 + head_of(t) < a.n_heads;
                float top = 0.0f;
#pragma unroll
                for (int b = 0; b < 4; ++b)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        q[t][b][e] = there ? q[t][b][e] : 0.0f;
                        top = fmaxf(top, fabsf(q[t][b][e]));
                    }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    pe[t][e] = there ? pe[t][e] : 0.0f;
                    top = fmaxf(top, fabsf(pe[t][e]));
                }
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                if (grp == 0) s.qmax[wave][t * 16 + n16] = top;
            }
            lds_barrier();
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const uint32_t r = t * 16 + n16;
                const float m = fmaxf(fmaxf(s.qmax[0][r], s.qmax[1][r]), fmaxf(s.qmax[2][r], s.qmax[3][r]));
                // m 2^e in [2^13, 2^14) for m within f32's middle range
                const int e = m > 0.0f ? min(max(140 - (int)(__float_as_uint(m) >> 23), -115), 115) : 0;
                const float sc = pow2(e);
                if (wave == 0 && grp == 0) s.factor[head_of(t)] = a.scale * 1.44269504088896f * pow2(-e);
                const bool packed = MODE == kPacked && t == 1;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    uint32_t h[4], l[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        split2(q[t][b][2 * i] * sc, q[t][b][2 * i + 1] * sc, h[i], l[i]);
                        if (packed && low_half) h[i] = l[i];
                    }
                    qh[t][b] = half8(make_uint4(h[0], h[1], h[2], h[3]));
                    if (!packed) ql[packed ? 0 : t][b] = half8(make_uint4(l[0], l[1], l[2], l[3]));
                }
                // (packed tile: both parts in the columns of the high ones)
                uint32_t h[4], l[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    split2(pe[t][2 * i] * sc, pe[t][2 * i + 1] * sc, h[i], l[i]);
                    if (grp >= 2) h[i] = l[i];
                    if (packed && low_half) h[i] = 0;
                }
                pe2[t] = half8(make_uint4(h[0], h[1], h[2], h[3]));
            }
        }

#pragma unroll
        for (int c = 0; c < 8; ++c)
#pragma unroll
            for (int t = 0; t < NT; ++t) o[c][t] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
        // Softmax state: this wave's heads, kPer positions per lane.
        constexpr uint32_t kPer = MODE == kOne ? 2 : 4, kLanes = kMlaTile / kPer;
        const bool softmax = MODE != kPacked || wave < 3;  // 24 heads: three waves' rows
        float m_run = -INFINITY, l_run = 0.0f;

        for (uint32_t i = 0;;) {
            const uint32_t ln = afresh(lane), n16 = ln & 15, grp = ln >> 4;
            const bool low_half = n16 >= 8;
            const auto head_of = [&](int t) { return MODE == kPacked && t == 1 ? 16 + (n16 & 7) : 16 * t + n16; };
            // Where a lane reads its keys (row n16 of 16 positions, chunk grp of
            // a block) and values (transposed: rows 4 grp + n16 / 4, 8 bytes of
            // 16 columns); blocks and columns are further bits to flip.
            const uint32_t k_at = n16 * 256 + ((grp ^ n16) << 4);
            const auto value_place = [](uint32_t ln) {
                const uint32_t n16 = ln & 15, row = 4 * (ln >> 4) + (n16 >> 2);
                return row * 256 + ((((n16 >> 1) & 1) ^ row) << 4) + (n16 & 1) * 8;
            };
            const uint32_t v_at = value_place(ln);
            const uint32_t srow = wave * (64 / kLanes) + ln / kLanes, spos = (ln % kLanes) * kPer;
            // Two workgroups share a CU: the one between its barriers goes first
            // (1 to 4%).
            __builtin_amdgcn_s_setprio(1);
            // ---- S^T partial ----
            // The keys of the first 16 positions, then each block's products with
            // the same block of the other 16 requested behind them: no wait on
            // LDS but the first. (The scheduling barriers keep that order; left
            // alone, each read is placed and waited for right before its use.)
            {
                const auto key = [&](int pt, uint32_t b) {
                    return half8(b < 4 ? *reinterpret_cast<const uint4*>(kv + pt * 4096 + (k_at ^ (b << 6)))
                                       : *reinterpret_cast<const uint4*>(s.pe[wave] + pt * 512 + n16 * 32 + 16 * (grp & 1)));
                };
                const auto there = [&](uint32_t b) { return b < 4 ? FULL || b < blocks : has_pe; };
                v8h k[5];
                v4f sc[2][NT], x[2][NT], d[2];
#pragma unroll
                for (uint32_t b = 0; b < 5; ++b) k[b] = key(0, b);
                if constexpr (Q8) d[0] = *reinterpret_cast<const v4f*>(&s.ds[wave][0][4 * grp]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int pt = 0; pt < 2; ++pt)
#pragma unroll
                    for (int t = 0; t < NT; ++t) sc[pt][t] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
                // Step i: block i % 5 (4: the rotary columns) of half i / 5.
#pragma unroll
                for (uint32_t i = 0; i <= (Q8 ? 10 : 9); ++i) {
                    const uint32_t pt = i / 5, b = i % 5;
                    if (i < 10 && there(b)) {
                        v4f(&acc)[NT] = Q8 ? x[i & 1] : sc[pt & 1];
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            if (Q8) acc[t] = (v4f){0.0f, 0.0f, 0.0f, 0.0f};
                            if (b < 4 && !(MODE == kPacked && t == 1))
                                acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[b], ql[t % (MODE == kTwo ? 2 : 1)][b & 3], acc[t], 0, 0, 0);
                        }
#pragma unroll
                        for (int t = NT - 1; t >= 0; --t)
                            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[b], b < 4 ? qh[t][b & 3] : pe2[t], acc[t], 0, 0, 0);
                    }
                    if (i < 5) k[b] = key(1, b);
                    if constexpr (Q8) {
                        // The block before, while this one's products run.
                        if (i > 0 && there((i - 1) % 5)) {
#pragma unroll
                            for (int t = 0; t < NT; ++t)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    sc[(i - 1) / 5][t][e] = fmaf(d[(i - 1) & 1][e], x[(i - 1) & 1][t][e], sc[(i - 1) / 5][t][e]);
                        }
                        if (i < 9) d[(i + 1) & 1] = *reinterpret_cast<const v4f*>(&s.ds[wave][(i + 1) % 5][(i + 1) / 5 * 16 + 4 * grp]);
                    }
                    if (!Q8 && i < 5) __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int pt = 0; pt < 2; ++pt) {
                    if constexpr (MODE == kPacked) {  // high and low parts' products, half a row of lanes apart
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[pt][1][e] += permuted<kRotate8>(sc[pt][1][e]);
                    }
                    *reinterpret_cast<v4f*>(&s.sp[wave][n16][pt * 16 + 4 * grp]) = sc[pt][0];
                    if (MODE == kTwo || (MODE == kPacked && !low_half))
                        *reinterpret_cast<v4f*>(&s.sp[wave][16 + n16][pt * 16 + 4 * grp]) = sc[pt][NT - 1];
                }
            }
            lds_barrier();

            // ---- softmax of this wave's heads ----
            // Half of the values' operands (16 columns, all 32 positions each)
            // are read behind the scores and arrive meanwhile.
            typedef float vper __attribute__((ext_vector_type(kPer)));
            vper part[kMlaWaves];
            const uint32_t from = min(srow, kHeads - 1);  // (a wave without heads reads along)
            const float fac = s.factor[from];
#pragma unroll
            for (uint32_t w = 0; w < kMlaWaves; ++w) part[w] = *reinterpret_cast<const vper*>(&s.sp[w][from][spos]);
            v8h val[8];
            const auto values = [&](uint32_t c, uint32_t at) {
                const v4s t0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(kv + (at ^ (c << 5))));
                const v4s t1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(kv + 4096 + (at ^ (c << 5))));
                const uint2 x = __builtin_bit_cast(uint2, t0), y = __builtin_bit_cast(uint2, t1);
                return half8(make_uint4(x.x, x.y, y.x, y.y));
            };
            const auto read_values = [&](uint32_t c) { val[c] = values(c, v_at); };
#pragma unroll
            for (uint32_t c = 0; c < 4; ++c) read_values(c);
            __builtin_amdgcn_sched_barrier(0);
            if (softmax) {
                const uint32_t lv = mask >> spos;
                const float m_was = m_run, l_was = l_run;
                // Scores to probabilities; the lane's own sum.
                const auto weigh = [&](vper x) {
                    float top = -INFINITY;
#pragma unroll
                    for (uint32_t e = 0; e < kPer; ++e) {
                        x[e] = (lv >> e) & 1 ? x[e] : -INFINITY;
                        top = fmaxf(top, x[e]);
                    }
                    top = group_max<kLanes>(top);
                    const float m_new = fmaxf(m_was, top), base = m_new == -INFINITY ? 0.0f : m_new;
                    const float al = __builtin_amdgcn_exp2f(m_was - base);
                    float own = 0.0f;
#pragma unroll
                    for (uint32_t e = 0; e < kPer; ++e) {
                        x[e] = __builtin_amdgcn_exp2f(x[e] - base);
                        own += x[e];
                    }
                    l_run = l_was * al + group_sum<kLanes>(own);
                    m_run = m_new;
                    if (ln % kLanes == 0) s.alpha[srow] = al;
                    // position 16 h + 4 g + e is O^T's operand element 4 h + e of group g;
                    // rows: high parts of both tiles, low parts of both; packed: high 16, packed 16, low 16
                    const uint32_t at = ((spos >> 2) & 3) * 8 + (spos >> 4) * 4 + (spos & 3);
                    const bool packed = MODE == kPacked && wave == 2;
                    uint32_t* hi = s.p + srow * 20 + at / 2;
                    uint32_t* lo = hi + (packed ? 8 : 16 * NT) * 20;
                    uint32_t h[kPer / 2], l[kPer / 2];
#pragma unroll
                    for (uint32_t e = 0; e < kPer; e += 2) split2(x[e] * kPScale, x[e + 1] * kPScale, h[e / 2], l[e / 2]);
                    if constexpr (kPer == 4) {
                        *reinterpret_cast<uint2*>(hi) = make_uint2(h[0], h[1]);
                        *reinterpret_cast<uint2*>(lo) = make_uint2(l[0], l[1]);
                    } else {
                        *hi = h[0];
                        *lo = l[0];
                    }
                    return own;
                };
                const float own = weigh((((part[0] + part[1]) + part[2]) + part[3]) * fac);
                // NaN: an infinite cached value met a part of the query that is 0
                // or of the other sign, where the formula has an infinity, or the
                // formula has NaN too. Such scores again, a head's lanes sharing the
                // columns of all waves' slices; the terms that are not finite
                // decide. (A query that is not finite gives NaN.)
                if (__builtin_expect(__any(own != own), 0)) {
                    if (__builtin_expect(group_max<kLanes>(own != own ? 1.0f : 0.0f) > 0.0f, 0)) {  // alike for a head's lanes
                        const uint32_t h = min(head0 + from, a.n_heads - 1), t = afresh(token), c0 = ln % kLanes;
                        const float* q = a.q + (uint64_t)t * a.q_token_stride + (uint64_t)h * a.q_head_stride;
                        const float* q_pe = a.q_pe + (uint64_t)t * a.q_pe_token_stride + (uint64_t)h * a.q_pe_head_stride;
                        const auto query = [&](uint32_t c) { return c < g.rank ? q[c] : q_pe[c - g.rank]; };
                        float none = 0.0f;
#pragma unroll 4
                        for (uint32_t c = c0; c < g.width; c += kLanes) none += query(c) - query(c);
                        none = group_sum<kLanes>(none);
#pragma unroll 1
                        for (uint32_t p = 0; p < kMlaTile; ++p) {
                            float score = (((s.sp[0][from][p] + s.sp[1][from][p]) + s.sp[2][from][p]) + s.sp[3][from][p]) * fac;
                            if (score != score && none == 0.0f) {
                                score = 0.0f;
#pragma unroll 1
                                for (uint32_t c = c0; c < g.width; c += kLanes) {
                                    const bool pe = c >= g.rank;
                                    const uint32_t i = pe ? c - g.rank : c, w = pe ? i / kMlaPe : i / kMlaCols;
                                    const uint32_t j = pe ? i % kMlaPe : i % kMlaCols;
                                    const uint8_t* at = pe ? s.pe[w] + p * 32 + 2 * j : s.kv[w] + p * 256 + (((j >> 3) ^ (p & 15)) << 4) + 2 * (j & 7);
                                    float k = (float)*reinterpret_cast<const _Float16*>(at);
                                    if constexpr (Q8) k *= s.ds[w][pe ? 4 : j / 32][p];
                                    if (!(fabsf(k) < INFINITY)) score += query(c) * k;
                                }
                                score = group_sum<kLanes>(score) * a.scale;
                            }
                            if (c0 == 0) s.sp[0][from][p] = score;
                        }
                        (void)weigh(*reinterpret_cast<const vper*>(&s.sp[0][from][spos]));
                    }
                }
            }
            lds_barrier();

            // ---- O^T += V^T P^T ----
            __builtin_amdgcn_s_setprio(0);
            {
                float al[NT];
                bool same = true;
                v8h ph[NT], plo[MODE == kTwo ? 2 : 1];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    al[t] = s.alpha[head_of(t)];
                    const uint32_t* src = s.p + (t * 16 + n16) * 20 + grp * 4;
                    ph[t] = half8(*reinterpret_cast<const uint4*>(src));
                    if (!(MODE == kPacked && t == 1)) plo[t % (MODE == kTwo ? 2 : 1)] = half8(*reinterpret_cast<const uint4*>(src + 16 * NT * 20));
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    same = same && al[t] == 1.0f;
                }
                if (!__all(same)) {
#pragma unroll
                    for (int c = 0; c < 8; ++c)
#pragma unroll
                        for (int t = 0; t < NT; ++t) o[c][t] *= al[t];
                }
#pragma unroll
                for (uint32_t c = 4; c < 8; ++c) read_values(c);
                // Two column tiles at a time, so that a product's sum is not
                // asked for by the next one. (Q8_0: the next two tiles' values
                // are scaled between this one's products.)
                v8h v[2], rest[2];
                const auto scale = [&](uint32_t b, v8h (&to)[2], v8h (&left)[2]) {
                    if constexpr (Q8) {
                        const uint2 d0 = *reinterpret_cast<const uint2*>(&s.dv[wave][b][4 * grp]);
                        const uint2 d1 = *reinterpret_cast<const uint2*>(&s.dv[wave][b][16 + 4 * grp]);
                        const v8h d = half8(make_uint4(d0.x, d0.y, d1.x, d1.y));
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            to[c] = val[2 * b + c] * d;
                            left[c] = __builtin_elementwise_fma(val[2 * b + c], d, -to[c]);
                        }
                    } else {
                        to[0] = val[2 * b];
                        to[1] = val[2 * b + 1];
                    }
                };
                scale(0, v, rest);
#pragma unroll
                for (uint32_t b = 0; b < 4; ++b) {
                    if (!FULL && b >= blocks) continue;
                    v8h nv[2], nrest[2];
#pragma unroll
                    for (int part = 0; part < 3; ++part) {
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                v4f& acc = o[2 * b + c][t];
                                if (part == 0 && !(MODE == kPacked && t == 1))
                                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[c], plo[t % (MODE == kTwo ? 2 : 1)], acc, 0, 0, 0);
                                if (part == 1 && Q8) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(rest[c], ph[t], acc, 0, 0, 0);
                                if (part == 2) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[c], ph[t], acc, 0, 0, 0);
                            }
                        if (part == 0 && b < 3) scale(b + 1, nv, nrest);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    if (b < 3) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) v[c] = nv[c], rest[c] = nrest[c];
                    }
                }
                // The blocks of large scales, into sums 2^-9 as large. (Places are
                // formed anew: kept from above they would cost the general kernels
                // 8 more spilled registers and a tenth of their speed.)
                if (Q8 && __builtin_expect(big != 0, 0)) {
                    const uint32_t ln = afresh(lane), at = value_place(ln), d_at = 4 * (ln >> 4);
#pragma unroll
                    for (uint32_t c = 0; c < 8; ++c) {
                        const uint2 d0 = *reinterpret_cast<const uint2*>(&s.db[wave][c / 2][d_at]);
                        const uint2 d1 = *reinterpret_cast<const uint2*>(&s.db[wave][c / 2][16 + d_at]);
                        const v8h d = half8(make_uint4(d0.x, d0.y, d1.x, d1.y));
                        const v8h code = values(c, at), high = code * d, left = __builtin_elementwise_fma(code, d, -high);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            v4f& acc = o[c][t];
                            acc *= 0x1p-9f;
                            if (!(MODE == kPacked && t == 1))
                                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(high, plo[t % (MODE == kTwo ? 2 : 1)], acc, 0, 0, 0);
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(left, ph[t], acc, 0, 0, 0);
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(high, ph[t], acc, 0, 0, 0);
                            acc *= 0x1p9f;
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            if (++i >= count) break;
            stage();
            load_rows(tile0 + i + 1, i + 1 < count);
            load_ids(tile0 + i + 2);
        }

        // ---- the piece's result ----
        if (lost && tid == 0) report(a.status, kBadPage);
        if (softmax && lane % kLanes == 0) s.ml[wave * (64 / kLanes) + lane / kLanes] = make_float2(m_run, l_run);
        lds_barrier();
        const uint32_t ln = afresh(lane), n16 = ln & 15, grp = ln >> 4;
        const bool low_half = n16 >= 8;
        const auto head_of = [&](int t) { return MODE == kPacked && t == 1 ? 16 + (n16 & 7) : 16 * t + n16; };
        const bool first = tile0 == 0, whole = first && count == n_tiles;
        const float back = 1.0f / kPScale;
        const uint64_t slot = (uint64_t)wg * 2 + (first ? 1 : 0);
        if constexpr (MODE == kPacked) {  // both parts' sums
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[c][1][e] += permuted<kRotate8>(o[c][1][e]);
        }
        // Through the wave's slice of LDS, so that a store writes two heads'
        // whole runs of 512 bytes and not 64 bytes of 16 heads each.
        float* const dst = (whole ? a.out + (uint64_t)token * a.out_token_stride + (uint64_t)head0 * a.out_head_stride
                                  : pl.parts + slot * pl.part_rows * g.rank) + wave * kMlaCols + 4 * (ln & 31);
        const uint64_t head_step = whole ? a.out_head_stride : g.rank;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint32_t r = head_of(t), h = head0 + r;
            const float2 ml = s.ml[r];
            const float f2 = !whole ? back : ml.y == 0.0f ? 0.0f : back / ml.y;
            if (wave == 0 && grp == 0 && h < a.n_heads && !(MODE == kPacked && t == 1 && low_half)) {
                if (!whole) pl.part_ml[slot * kHeads + r] = ml;
                else if (a.lse)
                    a.lse[(uint64_t)token * a.n_heads + h] =
                        ml.y == 0.0f ? -INFINITY : 0.69314718055995f * (ml.x + __builtin_amdgcn_logf(ml.y));
            }
#pragma unroll
            for (uint32_t c = 0; c < 8; ++c) *reinterpret_cast<v4f*>(kv + n16 * 512 + (((4 * c + grp) ^ n16) << 4)) = o[c][t] * f2;
            asm volatile("" ::: "memory");
#pragma unroll
            for (uint32_t j = 0; j < (MODE == kPacked && t == 1 ? 4 : 8); ++j) {
                const uint32_t n = 2 * j + (ln >> 5);
                const v4f v = *reinterpret_cast<const v4f*>(kv + n * 512 + (((ln & 31) ^ n) << 4));
                if (head0 + 16 * t + n >= a.n_heads || (!FULL && (ln & 31) >= 8 * blocks)) continue;
                float* to = dst + (16 * t + n) * head_step;
                if (!whole || pl.vec_out) {
                    // Written through: the next launch reads them on other XCDs,
                    // and lines left in L2 would be flushed at this one's end.
                    __builtin_nontemporal_store(v, reinterpret_cast<v4f*>(to));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) to[e] = v[e];
                }
            }
            asm volatile("" ::: "memory");
        }
        if (first && !whole) {
            begun.item = token * pl.head_tiles + ht_index;
            const uint64_t last = f + (n_slots - slot0) - 1;
            begun.pieces = (last < 0x80000000u ? (uint32_t)last / (uint32_t)chunk : (uint32_t)(last / chunk)) - wg + 1;
        }
        advance();
        lds_barrier();
    }
    if (tid == 0) splits[wg] = begun;

    // ---- tokens that see nothing, 256 at a time ----
    for (uint64_t t0 = (uint64_t)wg * kMlaThreads; t0 < a.n_tokens; t0 += (uint64_t)pl.groups * kMlaThreads) {
        uint32_t row, bad = 0;
        bool none = false;
        if (t0 + tid < a.n_tokens) none = seen(a, (uint32_t)(t0 + tid), row, bad) == 0;
        if (bad) report(a.status, bad == 1 ? kBadTableRow : kBadLength);
        for (uint64_t todo = __ballot(none); todo; todo &= todo - 1) {
            const uint64_t t = t0 + wave * 64 + __builtin_ctzll(todo);
            for (uint32_t h = 0; h < a.n_heads; ++h) {
                float* dst = a.out + t * a.out_token_stride + (uint64_t)h * a.out_head_stride;
                for (uint32_t c = lane; c < g.rank; c += 64) dst[c] = 0.0f;
                if (a.lse && lane == 0) a.lse[t * a.n_heads + h] = -INFINITY;
            }
        }
    }
}

// Joins the pieces of split items, in order: out = sum_k w_k O_k / sum_k w_k l_k
// with w_k = 2^(m_k - max m). A team of 8 lanes takes 32 columns of a head (16
// bytes per lane), so that one item reaches the whole chip (teams of 32 lanes:
// one token at 131072 positions in Q8_0 58 us instead of 56, the others alike).
// Teams share an item's pieces, up to four each, and add their sums through LDS.
constexpr uint32_t kTeam = 8, kJoinTeams = kJoinThreads / kTeam;
struct JoinShape {
    uint32_t share;  // teams per head and column part
    __device__ explicit JoinShape(uint32_t pieces) {
        share = 1;
        while (share < kJoinTeams && share * 4 < pieces) share *= 2;
    }
    __device__ static uint32_t parts(uint32_t rank) { return rank / (4 * kTeam); }
    __device__ uint32_t per_job() const { return kJoinTeams / share; }  // heads x parts
};

// (64 registers, so that two workgroups fit a CU: with 66 the join of 512 pieces
// took 17 us instead of 13)
__global__ __launch_bounds__(kJoinThreads, 8) void mla_join_kernel(MlaArgs a, MlaPlan pl) {
    __shared__ __align__(16) float sums[kJoinThreads * 4];
    // A job's heads times the item's pieces: at most 128 / share heads of 4 share
    // pieces, or one of kMlaMostGroups.
    __shared__ float weights[kMlaMostGroups];
    __shared__ float2 row_ml[32];
    __shared__ uint32_t scan[kJoinThreads / 64];
    __shared__ uint32_t cur[4];
    const uint32_t tid = threadIdx.x, wave = tid >> 6;
    const uint32_t rank = a.geom.rank;
    // Thread g knows the item that workgroup g began and did not finish, and
    // which of the call's jobs are that item's.
    MlaSplit sp{0, 0};
    if (tid < pl.groups) sp = reinterpret_cast<const MlaSplit*>(pl.splits)[tid];
    uint32_t my_jobs = 0;
    if (sp.pieces) {
        const JoinShape j(sp.pieces);
        const uint32_t heads = min(pl.rows, a.n_heads - (sp.item % pl.head_tiles) * pl.rows);
        my_jobs = (heads * j.parts(rank) + j.per_job() - 1) / j.per_job();
    }
    uint32_t end = (uint32_t)wave_scan(my_jobs);
    if ((tid & 63) == 63) scan[wave] = end;
    __syncthreads();
    uint32_t total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kJoinThreads / 64; ++w) {
        if (w < wave) end += scan[w];
        total += scan[w];
    }
    for (uint32_t all_job = blockIdx.x; all_job < total; all_job += gridDim.x) {
        __syncthreads();
        if (all_job < end && all_job >= end - my_jobs) {
            cur[0] = tid;
            cur[1] = sp.item;
            cur[2] = sp.pieces;
            cur[3] = all_job - (end - my_jobs);
        }
        __syncthreads();
        const uint32_t g0 = cur[0], item = cur[1], pieces = cur[2], job = cur[3];
        const JoinShape j(pieces);
        const uint32_t token = item / pl.head_tiles, head0 = (item % pl.head_tiles) * pl.rows;
        const uint32_t heads = min(pl.rows, a.n_heads - head0);
        const uint32_t parts = j.parts(rank), units = heads * parts, per_job = j.per_job();
        const uint32_t team = tid / kTeam, in_team = tid % kTeam;
        const uint32_t unit = job * per_job + team / j.share, mine = team % j.share;
        const bool on = unit < units;
        const uint32_t r0 = job * per_job / parts, r1 = min((job + 1) * per_job - 1, units - 1) / parts;
        const uint32_t r = on ? unit / parts : r0, c = ((on ? unit % parts : 0) * kTeam + in_team) * 4;
        // A thread's first four pieces are read while the weights are found (the
        // last piece again where there are fewer).
        const float* src = pl.parts + ((uint64_t)g0 * 2 * pl.part_rows + r) * rank + c;
        const uint64_t step = 2ull * pl.part_rows * rank, own = (uint64_t)pl.part_rows * rank;
        v4f early[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            const uint32_t p = min(mine + k * j.share, pieces - 1);
            early[k] = *reinterpret_cast<const v4f*>(src + p * step + (p == 0 ? own : 0));
        }
        // The weights of this job's heads: every maximum and sum by a thread of
        // its own, then 32 lanes per head.
        for (uint32_t i = tid; i < (r1 - r0 + 1) * pieces; i += kJoinThreads) {
            const uint32_t q = i % pieces, h = r0 + i / pieces;
            const float2 ml = pl.part_ml[((uint64_t)(g0 + q) * 2 + (q == 0)) * pl.rows + h];
            weights[i] = ml.x;
            sums[i] = ml.y;
        }
        __syncthreads();
        for (uint32_t i = tid / 32; i <= r1 - r0; i += kJoinThreads / 32) {
            const uint32_t l32 = tid & 31;
            float* w = weights + i * pieces;
            float top = -INFINITY, l = 0.0f;
            for (uint32_t q = l32; q < pieces; q += 32) top = fmaxf(top, w[q]);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
            const float base = top == -INFINITY ? 0.0f : top;
            for (uint32_t q = l32; q < pieces; q += 32) {
                w[q] = __builtin_amdgcn_exp2f(w[q] - base);
                l += w[q] * sums[i * pieces + q];
            }
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) l += __shfl_xor(l, d, 64);
            if (l32 == 0) row_ml[i] = make_float2(top, l);
        }
        __syncthreads();
        v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
        if (on) {
            const float* w = weights + (r - r0) * pieces;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                if (mine + k * j.share < pieces) acc += early[k] * w[mine + k * j.share];
            for (uint32_t p = mine + 4 * j.share; p < pieces; p += j.share)
                acc += *reinterpret_cast<const v4f*>(src + p * step + (p == 0 ? own : 0)) * w[p];
        }
        const float top = row_ml[r - r0].x, l = row_ml[r - r0].y;
        // A unit's teams: those of a wave by shuffles, the waves through LDS.
        const uint32_t in_wave = min(j.share, 64 / kTeam);
        for (uint32_t n = 1; n < in_wave; n *= 2)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += n == 1 ? permuted<kRotate8>(acc[e]) : __shfl_xor(acc[e], n * kTeam, 64);
        if (j.share > in_wave) {
            const uint32_t waves = j.share / in_wave;
            __syncthreads();
            if ((tid & 63) < kTeam) *reinterpret_cast<v4f*>(&sums[(wave * kTeam + in_team) * 4]) = acc;
            __syncthreads();
            if (mine == 0) {
                for (uint32_t n = 1; n < waves; ++n) acc += *reinterpret_cast<const v4f*>(&sums[((wave + n) * kTeam + in_team) * 4]);
            }
        }
        if (mine == 0 && on) {
            const v4f v = l == 0.0f ? (v4f){0.0f, 0.0f, 0.0f, 0.0f} : acc / l;
            float* dst = a.out + (uint64_t)token * a.out_token_stride + (uint64_t)(head0 + r) * a.out_head_stride + c;
            if (pl.vec_out) {
                *reinterpret_cast<v4f*>(dst) = v;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) dst[e] = v[e];
            }
            if (a.lse && c == 0)
                a.lse[(uint64_t)token * a.n_heads + head0 + r] =
                    l == 0.0f ? -INFINITY : 0.69314718055995f * (top + __builtin_amdgcn_logf(l));
        }
    }
}

// Two workgroups per CU, whatever the call: its lengths are known on the
// device alone.
uint32_t mla_groups(int num_cu) { return num_cu * 2 < (int)kMlaMostGroups ? (uint32_t)num_cu * 2 : kMlaMostGroups; }
uint64_t up256(uint64_t v) { return (v + 255) / 256 * 256; }

struct MlaLayout {
    int mode;
    uint32_t groups, rows, head_tiles, part_rows;
    uint64_t parts, ml, splits, bytes;
};
MlaLayout mla_layout(uint32_t n_heads, uint32_t rank, int num_cu) {
    MlaLayout w;
    w.groups = mla_groups(num_cu);
    w.mode = n_heads <= 16 ? kOne : n_heads <= 24 && rank == kKvMaxRank ? kPacked : kTwo;
    w.rows = mode_rows(w.mode);
    w.head_tiles = (n_heads + w.rows - 1) / w.rows;
    w.part_rows = n_heads < w.rows ? n_heads : w.rows;
    w.parts = 0;
    w.ml = up256(2ull * w.groups * w.part_rows * rank * 4);
    w.splits = w.ml + up256(2ull * w.groups * w.rows * 8);
    w.bytes = w.splits + up256(w.groups * sizeof(MlaSplit));
    return w;
}

template <bool Q8, int MODE, int POL>
void launch_mode(const MlaArgs& a, const MlaPlan& p, hipStream_t s) {
    // Every block and rotary column there is: no test of either in the loops.
    const bool full = a.geom.rank == kKvMaxRank && a.geom.width == kKvMaxRank + kKvMaxRope;
    if (full) mla_split_kernel<Q8, MODE, true, POL><<<p.groups, kMlaThreads, 0, s>>>(a, p);
    else mla_split_kernel<Q8, MODE, false, POL><<<p.groups, kMlaThreads, 0, s>>>(a, p);
}
template <bool Q8, int POL>
void launch_split(const MlaArgs& a, const MlaPlan& p, int mode, hipStream_t s) {
    if (mode == kOne) launch_mode<Q8, kOne, POL>(a, p, s);
    else if (mode == kPacked) launch_mode<Q8, kPacked, POL>(a, p, s);
    else launch_mode<Q8, kTwo, POL>(a, p, s);
}

}  // namespace

uint64_t mla_workspace_bytes(uint32_t n_tokens, uint32_t n_heads, uint32_t rank, int num_cu) {
    if (n_tokens == 0 || n_heads == 0 || rank == 0) return 0;
    return mla_layout(n_heads, rank, num_cu).bytes;
}

hipError_t launch_mla(const MlaArgs& a, hipStream_t s) {
    if (a.n_tokens == 0 || a.n_heads == 0) return hipSuccess;
    const MlaLayout w = mla_layout(a.n_heads, a.geom.rank, a.num_cu);
    char* base = static_cast<char*>(a.work);
    MlaPlan p{};
    p.groups = w.groups;
    p.rows = w.rows;
    p.head_tiles = w.head_tiles;
    p.part_rows = w.part_rows;
    p.parts = reinterpret_cast<float*>(base + w.parts);
    p.part_ml = reinterpret_cast<float2*>(base + w.ml);
    p.splits = base + w.splits;
    const auto aligned = [](const void* q, uint64_t s0, uint64_t s1) {
        return (reinterpret_cast<uintptr_t>(q) & 15u) == 0 && s0 % 4 == 0 && s1 % 4 == 0;
    };
    p.vec_q = aligned(a.q, a.q_token_stride, a.q_head_stride) &&
              (a.geom.width == a.geom.rank || aligned(a.q_pe, a.q_pe_token_stride, a.q_pe_head_stride));
    p.vec_out = aligned(a.out, a.out_token_stride, a.out_head_stride);
    // Rows that several tokens read (more tokens than tables: a prompt's chunk)
    // stay in the caches, f16 rows read once pass them by: 256 tokens at 4096
    // positions 171 us against 193, one token at 131072 positions 56 against
    // 53 and 64 tokens at 4096 positions 81 against 71. Q8_0 rows stay either
    // way: 241 against 247, 54.5 against 55.7 and 79.3 against 79.5.
    if (a.geom.q8) launch_split<true, kCacheNormal>(a, p, w.mode, s);
    else if (a.n_tokens > a.n_tables) launch_split<false, kCacheNormal>(a, p, w.mode, s);
    else launch_split<false, kCacheStream>(a, p, w.mode, s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    mla_join_kernel<<<2 * a.num_cu, kJoinThreads, 0, s>>>(a, p);
    return hipGetLastError();
}

}  // namespace mmhip
