// Attention of new tokens over a paged cache: what every build of it shares. The tokens of a sequence that read one of the
// cache's heads, `group` = heads / kv_heads queries' heads each, are its rows: row r is head r % group of token r / group, so
// that a page read once serves them all.
//
// Sequences of few rows or short ones (attend_few.h, fp32 in attend_f32.h): a group takes a tile of 16 rows of a sequence and
// cache head and a part of its keys, and finds out by itself which (af_share). The others (attend_tile.h): a group takes a
// unit, a tile of 128 rows and a run of its keys, of every head; of up to 1024 tiles it finds out by itself which (at_share),
// of more attend_plan makes a list. Where keys are split, attend_join puts the parts together.
//
// Constants: 0 q 2 q stride 4 out 6 out stride 8 k 10 v 12 page stride 14 head stride 16 token stride (bytes) 18 table 20 table
// stride 22 lengths 24 starts (0: `longest` tokens each) 26 few rows' parts 28 tiles of 128 rows of the longest sequence 29
// group 30 D 31 kv heads 32 sequences 33 longest 34 tokens 35 pages 36 page size 37 table width 38 flags (1 causal, 2 32 bits
// span the cache) 39 window 40 scale times log2(e) 41 groups that few rows' keys are split for (0: they are not) 42 tiles of
// few rows per sequence 43 type 44 keys of a tile 45 tiles that make a part 46 rows of a sequence that units take it from (0:
// none) 47 groups of attend_join for the few rows 48 units' list (0: none) 50 units' parts 52 logarithm of the page size,
// rounded up, and 59 its reciprocal 53 units that the list holds 54 parts that the workspace holds, per head 55 keys of a tile
// of units 56 rows that attend_join takes of a few rows' tile 57 tiles of keys up to which few rows' are not split 58 tiles
// that make a unit

#pragma once
#include "rows.h"

// What a group that shares its rows' keys keeps in the workspace: the maximum and the sum of each row, then the rows.
__device__ __forceinline__ uint64_t at_part_bytes(const GdArgs &a, uint32_t rows) { return (uint64_t)(rows * 4u) * (a.c[30] + 2u); }

// Of few rows: AF_ROWS a group.
#define AF_ROWS 16u
__device__ __forceinline__ uint64_t af_part(const GdArgs &a, uint32_t slot, uint32_t head) {
    return gd_addr(a, 26) + ((uint64_t)slot * a.c[31] + head) * at_part_bytes(a, AF_ROWS);
}

// Of many rows: AT_ROWS a group. The list of units that attend_plan makes.
#define AT_ROWS 128u
#define AT_SPLITS 1024u
struct AtUnit {
    uint32_t seq, tile, from, to;       // tile of rows, tiles of keys
    uint32_t slot, part, parts, none;  // parts of one tile of rows have neighbouring slots
};
struct AtPlan {
    uint32_t units, splits, none[62];
    uint32_t split[AT_SPLITS];  // units that are the first of several parts
};
__device__ __forceinline__ gd_gptr<AtPlan> at_plan(const GdArgs &a) { return gd_at<AtPlan>(gd_addr(a, 48)); }
__device__ __forceinline__ gd_gptr<AtUnit> at_units(const GdArgs &a) { return gd_at<AtUnit>(gd_addr(a, 48) + sizeof(AtPlan)); }
__device__ __forceinline__ uint64_t at_slot(const GdArgs &a, uint32_t slot, uint32_t head) {
    return gd_addr(a, 50) + ((uint64_t)slot * a.c[31] + head) * at_part_bytes(a, AT_ROWS);
}

// A tile of rows of a sequence and cache head, and the keys that any of them sees.
struct AtItem {
    uint32_t seq, head, token0, ql, rows, row0;  // rows: of the sequence and head; row0: the tile's first
    int32_t kl, first, end;      // keys first .. end - 1 are seen by some row of the tile,
    int32_t all_first, all_end;  // all_first .. all_end - 1 by each
};

// A sequence's tokens and keys, as the tables say and the call's bounds allow.
__device__ __forceinline__ void at_sequence(const GdArgs &a, uint32_t seq, AtItem &o) {
    const uint32_t longest = a.c[33], n = a.c[34];
    const int32_t most = (int32_t)(a.c[37] * a.c[36]);
    o.seq = seq;
    o.kl = min(max(gd_at<const int32_t>(gd_addr(a, 22))[seq], 0), most);
    if (gd_addr(a, 24)) {
        const gd_gptr<const int32_t> starts = gd_at<const int32_t>(gd_addr(a, 24)) + seq;
        const int32_t from = min(max(starts[0], 0), (int32_t)n), to = min(max(starts[1], from), (int32_t)n);
        o.token0 = from;
        o.ql = to - from;
    } else {
        o.token0 = seq * longest;
        o.ql = longest;
    }
    o.rows = o.ql * a.c[29];
}
// The keys that rows row0 .. row0 + rows - 1 (as far as there are) of a sequence see.
__device__ __forceinline__ void at_keys(const GdArgs &a, uint32_t row0, uint32_t rows, AtItem &o) {
    const uint32_t group = a.c[29];
    const int32_t window = (int32_t)a.c[39];
    const bool causal = a.c[38] & 1u;
    o.row0 = row0;
    // Positions of the tile's first and last token.
    const int32_t base = o.kl - (int32_t)o.ql, p0 = base + (int32_t)(row0 / group),
                  p1 = base + (int32_t)((min(row0 + rows, o.rows) - 1u) / group);
    o.first = window ? max(0, p0 - window + 1) : 0;
    o.end = causal ? max(0, p1 + 1) : o.kl;
    o.all_first = window ? max(0, p1 - window + 1) : 0;
    o.all_end = causal ? p0 + 1 : o.kl;
}
// Tiles of `keys` keys of an item and the first's number.
__device__ __forceinline__ uint32_t at_tiles(const AtItem &o, uint32_t keys, uint32_t &tile0) {
    tile0 = (uint32_t)o.first / keys;
    return o.end > o.first ? ((uint32_t)o.end + keys - 1u) / keys - tile0 : 0u;
}

// The page of key j of a sequence, and the key's offset in the cache, in bytes; -1: on a page outside it (or past `end`). Apart,
// so that the page's load can be far ahead of its use. No load is conditional: the compiler counts the loads that are on their
// way, and would wait for all of them where it is not certain of their number.
// i / page size, of i < 2^29: the size's reciprocal in 29 bits and its logarithm.
__device__ __forceinline__ uint32_t at_slot_of(const GdArgs &a, uint32_t i) { return __umulhi(i << 3, a.c[59]) >> a.c[52]; }
__device__ __forceinline__ uint32_t at_page(const GdArgs &a, uint32_t seq, int32_t j, int32_t end) {
    return (uint32_t)gd_at<const int32_t>(gd_addr(a, 18))[seq * gd_addr(a, 20) + at_slot_of(a, j < end ? (uint32_t)j : 0u)];
}
__device__ __forceinline__ int64_t at_key(const GdArgs &a, uint32_t page, uint32_t head, int32_t j, int32_t end) {
    const uint32_t place = (uint32_t)j - at_slot_of(a, (uint32_t)j) * a.c[36];
    const int64_t at = page * gd_addr(a, 12) + place * gd_addr(a, 16) + head * gd_addr(a, 14);
    return (j < end) & (page < a.c[35]) ? at : -1;
}

// As at_key, of a cache that 32 bits span, without the head (its offset is the wave's).
__device__ __forceinline__ uint32_t at_key_small(const GdArgs &a, uint32_t page, int32_t j, int32_t end, bool &there) {
    const uint32_t place = (uint32_t)j - at_slot_of(a, (uint32_t)j) * a.c[36];
    there = (j < end) & (page < a.c[35]);
    return there ? page * a.c[12] + place * a.c[16] : 0u;
}

// The larger of a value and lane ^ 32's.
__device__ __forceinline__ float at_max_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(gd_f32_bits(v), gd_f32_bits(v), false, false);
    return fmaxf(gd_bits_f32(r[0]), gd_bits_f32(r[1]));
}
__device__ __forceinline__ float at_sum_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(gd_f32_bits(v), gd_f32_bits(v), false, false);
    return gd_bits_f32(r[0]) + gd_bits_f32(r[1]);
}
__device__ __forceinline__ float at_exp2(float v) { return __builtin_amdgcn_exp2f(v); }

// Four values of a row from d on, times `by`; zeros where nothing was seen.
typedef gd_u32x2 at_u32x2_any __attribute__((aligned(2)));
template <uint32_t TYPE>
__device__ __forceinline__ void at_store4(uint64_t row, uint32_t d, gd_f32x4 x, float by, bool none) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = none ? 0.f : x[i] * by;
    if constexpr (TYPE == ROW_F32)
        *gd_at<gd_f32x4_any>(row + 4ull * d) = x;
    else
        *gd_at<at_u32x2_any>(row + 2ull * d) = gd_u32x2{row_bits16(x[0], TYPE) | row_bits16(x[1], TYPE) << 16,
                                                        row_bits16(x[2], TYPE) | row_bits16(x[3], TYPE) << 16};
}

// Where maxima begin: no finite score is below it, and the difference of two such is zero, not NaN.
#define AT_LOWEST -3.402823466e38f

// A weight is exp2(s scale - top), in one fused step. top is a product of that kind as well, but rounded: off by up to half a
// unit of its last place, by which all of a row's weights are too large or small alike. From 2^20 on that is 2^-5 and more, and
// with no bound: of scores of 10^10 all weights were zero, or infinite. Rows with such a top take both products rounded, so
// that the largest score's weight is one.
#define AT_FAR 1048576.f
__device__ __forceinline__ bool at_far(float top) { return (fabsf(top) >= AT_FAR) & (top > AT_LOWEST); }
__device__ __forceinline__ float at_from_top(float s, float scale, float top) {
    float product = s * scale;
    asm volatile("" : "+v"(product));  // (not to be fused)
    return at_far(top) ? product - top : fmaf(s, scale, -top);
}

// Few rows (attend_few.h, attend_f32.h).

// The larger (the sum) of the four lanes that hold a row's keys, 16 lanes apart.
__device__ __forceinline__ float af_max(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(gd_f32_bits(v), gd_f32_bits(v), false, false);
    return at_max_halves(fmaxf(gd_bits_f32(r[0]), gd_bits_f32(r[1])));
}
__device__ __forceinline__ float af_sum(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(gd_f32_bits(v), gd_f32_bits(v), false, false);
    return at_sum_halves(gd_bits_f32(r[0]) + gd_bits_f32(r[1]));
}

// How the few rows' keys are shared out: entry e is tile e % tiles of sequence e / tiles. One of more tiles of keys than a
// constant is split into as many parts as leave none more than `share` tiles, a fair part of all entries' and heads' among the
// groups. The split entries' parts come first, then the whole ones. Every wave works this out by itself, 64 entries at a time.
struct AfEntry {
    uint32_t rows, keys;  // of the sequence (0: none for this launch), tiles of keys
};
__device__ __forceinline__ AfEntry af_entry(const GdArgs &a, uint32_t e, AtItem &o, uint32_t &tile0) {
    const uint32_t tiles = a.c[42], seq = tiles == 1u ? e : e / tiles, row0 = (e - seq * tiles) * AF_ROWS;
    o.rows = 0u;
    if (seq >= a.c[32]) return {0u, 0u};
    at_sequence(a, seq, o);
    if (row0 >= o.rows || (a.c[46] && o.rows >= a.c[46])) {
        o.rows = 0u;
        return {0u, 0u};
    }
    at_keys(a, row0, AF_ROWS, o);
    return {o.rows, at_tiles(o, a.c[44], tile0)};
}
__device__ __forceinline__ uint32_t af_last(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, 63); }

struct AfShare {
    AfEntry first;  // the lane's of the first 64
    uint32_t share;
};
__device__ __forceinline__ AfEntry af_mine(const GdArgs &a, const AfShare &s, uint32_t e0) {
    AtItem o;
    uint32_t tile0;
    return e0 ? af_entry(a, e0 + (threadIdx.x & 63u), o, tile0) : s.first;
}
__device__ __forceinline__ AfShare af_share(const GdArgs &a) {
    const uint32_t entries = a.c[32] * a.c[42];
    AfShare s;
    AtItem o;
    uint32_t tile0;
    s.first = af_entry(a, threadIdx.x & 63u, o, tile0);
    uint64_t all = 0;
    for (uint32_t e0 = 0; e0 < entries; e0 += 64u) all += af_last(gd_wave_scan_u32(af_mine(a, s, e0).keys));  // at most 2^25 each
    s.share = (uint32_t)max((uint64_t)a.c[45], (all * a.c[31] + a.c[41] - 1u) / a.c[41]);
    return s;
}
// The entry of number `wanted` among the split ones, counting parts (or entries), or the whole ones; false: there are fewer.
// `wanted` becomes the part's number in it, `slot` the number of its first part among all split ones'.
enum { AF_PARTS, AF_SPLITS, AF_WHOLE };
template <int WHAT>
__device__ __forceinline__ bool af_find(const GdArgs &a, const AfShare &s, uint32_t &wanted, uint32_t &entry, uint32_t &parts, uint32_t &slot) {
    const uint32_t entries = a.c[32] * a.c[42];
    slot = 0;
    for (uint32_t e0 = 0; e0 < entries; e0 += 64u) {
        const AfEntry mine = af_mine(a, s, e0);
        const uint32_t split = mine.keys > max(s.share, a.c[57]) ? (mine.keys + s.share - 1u) / s.share : 0u;
        const uint32_t count = WHAT == AF_PARTS ? split : WHAT == AF_SPLITS ? (split ? 1u : 0u) : mine.rows && !split ? 1u : 0u;
        const uint32_t upto = gd_wave_scan_u32(count), total = af_last(upto), slots = gd_wave_scan_u32(split);
        if (wanted < total) {
            const uint32_t at = (uint32_t)__builtin_ctzll(__ballot(upto > wanted));  // the first lane past it
            auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)at); };
            entry = e0 + at;
            parts = max(1u, of(split));
            slot += of(slots) - of(split);
            wanted -= of(upto) - of(count);
            return true;
        }
        wanted -= total;
        slot += af_last(slots);
    }
    return false;
}

// A group's tile, its part of the keys' tiles, and what a lane knows of its row: lane l has row l % 16 (rows past the last are
// the last again), and of the scores the keys 4 (l / 16) + i.
struct AfWork {
    AtItem o;
    uint32_t slot, parts, from, to;
    uint64_t q;           // offset of the row in q, in values
    int32_t first, last;  // keys that the row sees
};
__device__ __forceinline__ bool af_work(const GdArgs &a, AfWork &w) {
    const uint32_t id = blockIdx.y * gridDim.x + blockIdx.x, group = a.c[29], KVH = a.c[31], unit = id / KVH;
    uint32_t part = 0, entry = unit, tile0;
    w.parts = 1;
    w.slot = 0;
    if (a.c[41]) {
        const AfShare share = af_share(a);
        part = unit;
        if (!af_find<AF_PARTS>(a, share, part, entry, w.parts, w.slot)) {
            uint32_t none;
            if (!af_find<AF_WHOLE>(a, share, part, entry, w.parts, none)) return false;
        }
    }
    const AfEntry own = af_entry(a, entry, w.o, tile0);
    const uint32_t tiles = own.keys;
    if (!own.rows) return false;
    w.o.head = id - unit * KVH;
    w.slot += part;
    w.from = tile0 + (uint32_t)((uint64_t)tiles * part / w.parts);
    w.to = tile0 + (uint32_t)((uint64_t)tiles * (part + 1u) / w.parts);
    const uint32_t row = min(w.o.row0 + (threadIdx.x & 15u), w.o.rows - 1u), token = row / group;
    w.q = (uint64_t)(w.o.token0 + token) * gd_addr(a, 2) + (uint64_t)(w.o.head * group + row - token * group) * a.c[30];
    const int32_t p = w.o.kl - (int32_t)w.o.ql + (int32_t)token, window = (int32_t)a.c[39];
    w.last = a.c[38] & 1u ? p : w.o.kl - 1;
    w.first = window ? p - window + 1 : 0;
    return true;
}

// Joins the waves' parts and writes the rows, or the group's part of them. The waves have put their rows into LDS, DT + 4 values
// each, EACH values a wave.
template <uint32_t TYPE, uint32_t DT, uint32_t EACH, uint32_t WAVES>
__device__ __forceinline__ void af_finish(const GdArgs &a, const AfWork &k, float top, float sum, float *lds) {
    constexpr uint32_t WIDE = DT + 4u;
    static_assert(EACH >= AF_ROWS * WIDE, "a wave's rows");
    __shared__ float stats[WAVES][2][AF_ROWS];
    const AtItem &o = k.o;
    const uint32_t lane = threadIdx.x & 63u, col = lane & 15u, wave = threadIdx.x >> 6, D = a.c[30], group = a.c[29];
    sum = af_sum(sum);
    if (lane < 16u) {
        stats[wave][0][col] = top;
        stats[wave][1][col] = sum;
    }
    __syncthreads();
    constexpr uint32_t THREADS = 4u * WAVES;  // of a row
    const uint32_t r = threadIdx.x / THREADS, c = threadIdx.x % THREADS;
    if (o.row0 + r >= o.rows) return;
    float most = stats[0][0][r], total = 0.f, shrink[WAVES];
#pragma unroll
    for (uint32_t w = 1; w < WAVES; ++w) most = fmaxf(most, stats[w][0][r]);
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) {
        shrink[w] = at_exp2(stats[w][0][r] - most);
        total += stats[w][1][r] * shrink[w];
    }
    const bool alone = k.parts == 1u;
    const uint64_t to_part = af_part(a, k.slot, o.head);
    if (!alone && c == 0u) {
        gd_at<float>(to_part)[r] = most;
        gd_at<float>(to_part)[AF_ROWS + r] = total;
    }
    const uint32_t token = (o.row0 + r) / group;
    const uint64_t out = gd_addr(a, 4) + (((uint64_t)(o.token0 + token) * gd_addr(a, 6) + (uint64_t)(o.head * group + o.row0 + r - token * group) * D)
                                          << row_shift(TYPE));
    const float by = 1.f / total;
#pragma unroll
    for (uint32_t e = 0; e < (DT + 4u * THREADS - 1u) / (4u * THREADS); ++e) {
        const uint32_t d = 4u * THREADS * e + 4u * c;
        if (d >= D) continue;
        gd_f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (uint32_t w = 0; w < WAVES; ++w) {
            const gd_f32x4 y = *reinterpret_cast<const gd_f32x4 *>(lds + w * EACH + r * WIDE + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] += y[i] * shrink[w];
        }
        if (alone) at_store4<TYPE>(out, d, x, by, total == 0.f);
        else *gd_at<gd_f32x4>(to_part + 8u * AF_ROWS + ((uint64_t)r * D + d) * 4u) = x;
    }
}

// The tiles of keys that a unit has at most, of so many that all tiles of rows have: a 512th of every head's (two groups for each
// compute unit) and an eighth more, so that tiles a little larger than that are not split into units that fill a second round
// by half (40 tiles of 250 and 22 small ones, four heads: 4 parts each 288 us, 3 parts 230).
__device__ __forceinline__ uint32_t at_fair(const GdArgs &a, uint64_t all) {
    return (uint32_t)min(max((uint64_t)a.c[58], (all * a.c[31] * 9u + 4095u) / 4096u), (uint64_t)~0u);
}

// How the many rows' keys are shared out without a list: entry e is tile tiles - 1 - e / sequences of sequence e % sequences, the
// tiles that see most keys first. Its keys are split as attend_plan splits them. Units of half a share or more come first (the
// parts of split entries among them, which makes their numbers slots), then the others. The 256 threads of a group work this out
// together, four entries each at most. Every group comes to the same numbers, those of the split entries among them.
#define AT_HELD 4u
struct AtShare {
    uint32_t sums[AT_HELD][4], split[AT_SPLITS];  // a wave's counts; split entries: first slot << 16 | entry
    uint32_t entry, part, parts, splits, found;
    uint64_t all;
};
// The unit of number `wanted` (found 0: there is none), or the split entries, in `s`.
__device__ __forceinline__ void at_share(const GdArgs &a, AtShare &s, uint32_t wanted, bool list) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, S = a.c[32], tiles = a.c[28], entries = S * tiles;
    if (tid == 0u) {
        s.all = 0;
        s.found = 0u;
    }
    uint32_t keys[AT_HELD], rows[AT_HELD], own = 0;
#pragma unroll
    for (uint32_t k = 0; k < AT_HELD; ++k) {
        const uint32_t e = 256u * k + tid;
        keys[k] = rows[k] = 0u;
        if (256u * k < entries && e < entries) {
            AtItem o;
            uint32_t tile0;
            const uint32_t back = e / S, row0 = (tiles - 1u - back) * AT_ROWS;
            at_sequence(a, e - back * S, o);
            if (row0 < o.rows && o.rows >= a.c[46]) {
                at_keys(a, row0, AT_ROWS, o);
                keys[k] = at_tiles(o, a.c[55], tile0);
                rows[k] = 1u;
            }
        }
        own += min(keys[k], 0xffffffu);  // of 2^24 at most; 64 lanes' 4 in 32 bits
    }
    __syncthreads();
    const uint32_t of_wave = (uint32_t)__builtin_amdgcn_readlane((int)gd_wave_scan_u32(own), 63);
    if (lane == 0u && of_wave) atomicAdd((unsigned long long *)&s.all, (unsigned long long)of_wave);
    __syncthreads();
    const uint32_t share = at_fair(a, s.all);
    // In 11 bits each, units of the first kind and of the second, of which there are fewer than 1024 + 456 and 1025; then split
    // entries, each of more than 9 / 4096 of all keys.
    uint32_t parts[AT_HELD], count[AT_HELD], upto[AT_HELD];
#pragma unroll
    for (uint32_t k = 0; k < AT_HELD; ++k) {
        parts[k] = max(1u, (keys[k] + share - 1u) / share);
        count[k] = !rows[k] ? 0u : 2u * (keys[k] / parts[k]) >= share ? parts[k] | (parts[k] > 1u ? 1u << 22 : 0u) : 1u << 11;
        upto[k] = gd_wave_scan_u32(count[k]);
        if (lane == 63u) s.sums[k][wave] = upto[k];
    }
    __syncthreads();
    uint32_t before = 0, total = 0;
#pragma unroll
    for (uint32_t k = 0; k < AT_HELD; ++k)
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w) total += s.sums[k][w];
    if (tid == 0u) s.splits = total >> 22;
#pragma unroll
    for (uint32_t k = 0; k < AT_HELD; ++k) {
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w) {
            if (w == wave) upto[k] += before - count[k];  // units before the thread's
            before += s.sums[k][w];
        }
        const uint32_t first = upto[k] & 2047u, small = (total & 2047u) + (upto[k] >> 11 & 2047u);
        const bool one = count[k] == 1u << 11;
        if (list) {
            if (parts[k] > 1u && upto[k] >> 22 < AT_SPLITS) s.split[upto[k] >> 22] = first << 16 | (256u * k + tid);
        } else if (rows[k] && (one ? wanted == small : wanted - first < parts[k])) {
            s.entry = 256u * k + tid;
            s.part = one ? 0u : wanted - first;
            s.parts = one ? 1u : parts[k];
            s.found = 1u;
        }
    }
    __syncthreads();
}
