// Rotary positions, the paged cache's appending and the attention over it (gm_rotary, gm_cache_append, gm_attention): argument
// checks, the choice of a build, its constants and grid, as row_ops.h has them for the other operators. Their kernels are
// csrc/kernels/rotary.h and attend*.h.
#pragma once
#include "gyro_attention.h"
#include "row_ops.h"

namespace gyro {

// Launches of the same constants, one after another.
struct Launches {
    Constants c;
    struct Step {
        const char *kernel;
        uint32_t x, y;
    } step[4] = {};
    int count = 0;
    // A grid of at least `groups` groups (a kernel's own check drops the others).
    void add(const char *kernel, uint64_t groups) {
        const uint32_t x = (uint32_t)std::min<uint64_t>(groups, 65535);
        step[count++] = {kernel, x, (uint32_t)((groups + x - 1) / x)};
    }
};

struct Rotary {
    Buffer table;  // per pair the fraction of a turn of one position, of 2^64
    uint32_t pairs = 0, layout = 0;
    float scale = 1;
};

class AttentionOps {
  public:
    std::vector<Rotary> rotaries;

    // ---- rotary positions ----

    // The fraction of a turn, of 2^64, by which a frequency below 2^31 turns, rounded: m 2^-down (m of 53 bits) times 1 / (2
    // pi) in 128 bits, before rounding exact to 2^-21 of the last place, however many whole turns there are.
    static uint64_t fraction(double frequency) {
        constexpr uint64_t high = 0x28be60db9391054aull, low = 0x7f09d5f47d4d3770ull;  // 2^128 / (2 pi)
        int e;
        const uint64_t m = (uint64_t)std::ldexp(std::frexp(std::fabs(frequency), &e), 53);
        const uint32_t down = (uint32_t)(53 - e);  // at least 22
        // m / (2 pi) in units of 2^-64, of which the last place is 2^22 or more.
        const unsigned __int128 turns = (unsigned __int128)m * high + (uint64_t)((unsigned __int128)m * low >> 64);
        if (down > 128) return 0;
        const uint64_t whole = down < 128 ? (uint64_t)(turns >> down) : 0, f = whole + (uint64_t)(turns >> (down - 1) & 1);
        return frequency < 0 ? 0 - f : f;
    }

    static Rotary describe(const double *frequencies, uint32_t pairs, uint32_t layout, float scale, std::vector<uint64_t> &table) {
        require(frequencies && pairs && pairs <= 512, "a rotary has 1 to 512 pairs");
        require(layout <= GM_ROTARY_INTERLEAVED, "unknown rotary layout");
        require(std::isfinite(scale), "a rotary's scale is finite");
        table.resize(pairs);
        for (uint32_t i = 0; i < pairs; ++i) {
            require(std::fabs(frequencies[i]) < 2147483648.0, "a rotary's frequencies are below 2^31 in magnitude");
            table[i] = fraction(frequencies[i]);
        }
        Rotary r;
        r.pairs = pairs;
        r.layout = layout;
        r.scale = scale;
        return r;
    }
    const Rotary &rotary(uint32_t i) const {
        require(i < rotaries.size() && rotaries[i].table.handle, "no such rotary");
        return rotaries[i];
    }
    uint32_t keep(Rotary &&r) {
        for (uint32_t i = 0; i < rotaries.size(); ++i)
            if (!rotaries[i].table.handle) {
                rotaries[i] = std::move(r);
                return i;
            }
        rotaries.push_back(std::move(r));
        return (uint32_t)rotaries.size() - 1;
    }

    // Rows of `heads` heads and what becomes of them: in place, of one type and stride.
    static void check_pair(const gm_rows &x, const gm_rows &y, uint32_t n, uint32_t values, const char *what) {
        RowOps::check_rows(x, n, values, false, what);
        RowOps::check_rows(y, n, values, true, what);
        require(x.data != y.data || (x.type == y.type && (n == 1 || x.stride == y.stride)), what);
    }

    // The launch of queries (heads of them), keys and values (kv_heads of each) of n tokens, D values a head.
    static void turn(Launch &l, const Rotary *r, const gm_rows *q, const gm_rows *q_out, uint32_t heads, const gm_rows *k, const gm_rows *v,
                     uint32_t kv_heads, uint32_t D, uint32_t n) {
        Constants &c = l.c;
        const gm_rows &x = q ? *q : *k;
        if (q) {
            c.set(0, q->data);
            c.set64(2, q->stride);
            c.set(4, q_out->data);
            c.set64(6, q_out->stride);
        }
        if (k) {
            c.set(8, k->data);
            c.set64(10, k->stride);
            c.set(12, v->data);
            c.set64(14, v->stride);
        }
        const uint32_t pairs = r ? r->pairs : 0, all = heads + 2 * kv_heads;
        if (r) {
            c.set64(26, r->table.gpu);
            c.set(39, r->scale);
        }
        c.set(32, D);
        c.set(33, pairs);
        c.set(34, heads);
        c.set(35, kv_heads);
        c.set(36, n);
        const uint32_t units = std::max((pairs + 7) / 8 + (D - 2 * pairs + 15) / 16, (D + 15) / 16);
        // A group's 256 threads take at_once heads together, two a thread and turn. Of few tokens a group takes one turn of a
        // token, so that all are on their way at once; of many (256 compute units hold eight groups each) up to eight turns of
        // it, or, where eight turns of a wave cover the heads, four tokens, one a wave (us, 4096 tokens of 128 values: one head
        // 20 and 9.5, 8 heads 13.0 and 7.2, 24 14.8 and 12.4; 32 and 8 + 8 into a cache 26.8 and 24.8; replayed, 2048 tokens of
        // 8 heads 6.7 and 4.3, of 32 and 8 + 8 13.2 and 12.2, 1023 tokens 4.6 and 3.8, 8.1 and 9.9).
        const bool narrow = n > 2048 && units <= 64 && 16 * (64 / units) >= all && pairs <= 128;
        const uint32_t at_once = (narrow ? 64 : 256) / units, all_turns = (all + 2 * at_once - 1) / (2 * at_once);
        const uint32_t turns = (uint64_t)n * all_turns > 2048 ? std::min(all_turns, 8u) : 1u, sharers = (all_turns + turns - 1) / turns;
        c.set(45, narrow ? 1u : 0u);
        c.set(42, sharers);
        c.set(43, units);
        c.set(44, turns);
        const uint64_t blocks = narrow ? ((uint64_t)n + 3) / 4 : (uint64_t)n * sharers;
        l.kernel = x.type == GM_F32 ? "rotary_f" : x.type == GM_BF16 ? "rotary_b" : "rotary_h";
        l.x = (uint32_t)std::min<uint64_t>(blocks, 65535);
        l.y = (uint32_t)((blocks + 65534) / 65535);
    }

    Launch turned(const gm_rotary_desc &d, uint32_t n) const {
        Launch l;
        const Rotary &r = rotary(d.rotary);
        if (!n) return l;  // of no rows there may be no memory
        require(d.heads && d.head_dim && d.head_dim <= 1024 && 2 * r.pairs <= d.head_dim, "gm_rotary: heads of up to 1024 values, all pairs in them");
        require((uint64_t)n * d.heads < 1u << 31 && d.heads <= 1u << 20, "gm_rotary: n * heads is below 2^31");
        check_pair(d.x, d.y, n, d.heads * d.head_dim, "gm_rotary: x and y");
        require(d.positions && (uintptr_t)d.positions % (d.positions_64 ? 8 : 4) == 0, "gm_rotary: positions");
        turn(l, &r, &d.x, &d.y, d.heads, nullptr, nullptr, 0, d.head_dim, n);
        l.c.set(28, d.positions);
        l.c.set(37, d.y.type);
        l.c.set(38, (r.layout == GM_ROTARY_INTERLEAVED ? 1u : 0u) | (d.positions_64 ? 2u : 0u) | (d.x.data == d.y.data ? 8u : 0u));
        return l;
    }

    // ---- the cache ----

    static void check_cache(const gm_cache &c, const char *what) {
        require(c.k && c.v && c.type <= GM_F16, what);
        const uint64_t size = c.type == GM_F32 ? 4 : 2;
        require((uintptr_t)c.k % size == 0 && (uintptr_t)c.v % size == 0, what);
        require(c.pages && c.page_size && (uint64_t)c.pages * c.page_size < 1u << 31, what);
        require(c.kv_heads && c.kv_heads <= 1u << 20 && c.head_dim, what);
        const uint64_t most = uint64_t(1) << 40;
        require(c.page_stride <= most && c.head_stride <= most && c.token_stride <= most, what);
    }
    // Strides in bytes, at constant `at`.
    static void set_cache(Constants &c, const gm_cache &cache, int at) {
        const uint64_t size = cache.type == GM_F32 ? 4 : 2;
        c.set64(at, cache.page_stride * size);
        c.set64(at + 2, cache.head_stride * size);
        c.set64(at + 4, cache.token_stride * size);
    }

    Launch append(const gm_cache_append_desc &d, uint32_t n) const {
        Launch l;
        const Rotary *const r = d.rotary == GM_NO_ROTARY ? nullptr : &rotary(d.rotary);
        if (!n) return l;  // of no rows there may be no memory
        const uint32_t D = d.cache.head_dim, G = d.cache.kv_heads;
        check_cache(d.cache, "gm_cache_append: cache");
        require(D <= 1024 && (!r || 2 * r->pairs <= D), "gm_cache_append: heads of up to 1024 values, all pairs in them");
        require(d.heads <= 1u << 20 && (uint64_t)n * (d.heads + 2ull * G) < 1u << 31, "gm_cache_append: n times the heads is below 2^31");
        RowOps::check_rows(d.k, n, G * D, false, "gm_cache_append: k");
        RowOps::check_rows(d.v, n, G * D, false, "gm_cache_append: v");
        require(d.k.type == d.v.type, "gm_cache_append: k and v have one type");
        require(!d.heads == !d.q.data && !d.heads == !d.q_out.data, "gm_cache_append: q, q_out and its heads go together");
        if (d.heads) {
            check_pair(d.q, d.q_out, n, d.heads * D, "gm_cache_append: q and q_out");
            require(d.q.type == d.k.type, "gm_cache_append: q has the type of k");
        }
        require(d.slots && (uintptr_t)d.slots % (d.slots_64 ? 8 : 4) == 0, "gm_cache_append: slots");
        require(!r || (d.positions && (uintptr_t)d.positions % (d.positions_64 ? 8 : 4) == 0), "gm_cache_append: positions");
        // No two (page, head, token) may share an element: of two dimensions one's stride spans the other's extent. (Whether
        // keys and values lie apart is the caller's to know; one array for both is told.)
        check_apart(d.cache);
        require(d.cache.k != d.cache.v, "gm_cache_append: the cache's keys and values are one array");
        turn(l, r, d.heads ? &d.q : nullptr, &d.q_out, d.heads, &d.k, &d.v, G, D, n);
        Constants &c = l.c;
        c.set(16, d.cache.k);
        c.set(18, d.cache.v);
        set_cache(c, d.cache, 20);
        if (r) c.set(28, d.positions);
        c.set(30, d.slots);
        c.set(37, (d.heads ? d.q_out.type : 0u) | d.cache.type << 4);
        c.set(38, (r && r->layout == GM_ROTARY_INTERLEAVED ? 1u : 0u) | (d.positions_64 ? 2u : 0u) | (d.slots_64 ? 4u : 0u) |
                      (d.q.data == d.q_out.data ? 8u : 0u));
        c.set(40, d.cache.page_size);
        c.set(41, d.cache.pages * d.cache.page_size);
        return l;
    }
    static void check_apart(const gm_cache &c) {
        struct Dim {
            uint64_t stride, count;
        } dims[3] = {{c.page_stride, c.pages}, {c.head_stride, c.kv_heads}, {c.token_stride, c.page_size}};
        std::sort(dims, dims + 3, [](const Dim &a, const Dim &b) { return a.stride < b.stride; });
        uint64_t extent = c.head_dim;
        for (const Dim &d : dims) {
            if (d.count == 1) continue;
            require(d.stride >= extent, "gm_cache_append: the cache's heads overlap");
            extent = d.stride * (d.count - 1) + extent;
        }
    }

    // ---- attention ----

    // Few rows: groups that their keys are split for, the workspace holds twice as many parts (an entry of more than a fair part
    // is split into less than twice as many), and entries whose shares every group works out. Many: parts of 128 rows that the
    // workspace holds (attend_plan splits tiles of more than a 512th of all keys: twice 512 at most), and units.
    static constexpr uint32_t kGroups = 1024, kEntries = 1024, kSlots = 1024, kUnits = 1u << 18, kPlanBytes = 256 + 4 * 1024, kUnitBytes = 32;
    static constexpr uint32_t kFewRows = 16, kTileRows = 128;
    static uint64_t part_bytes(uint32_t rows, uint32_t D) { return (uint64_t)rows * 4 * (D + 2); }
    // The workspace: the few rows' parts, the plan with its units, the units' parts.
    static uint64_t plan_at(uint32_t D) { return 2 * kGroups * part_bytes(kFewRows, D); }
    static uint64_t slots_at(uint32_t D) { return plan_at(D) + kPlanBytes + (uint64_t)kUnits * kUnitBytes; }
    static uint64_t workspace(uint32_t heads, uint32_t kv_heads, uint32_t D) {
        if (!heads || !kv_heads || heads % kv_heads || !D || D > 256) return 0;
        return slots_at(D) + kSlots * part_bytes(kTileRows, D);
    }

    static Launches attention(const gm_attention_desc &d, uint32_t n) {
        Launches l;
        if (!n) return l;  // of no rows there may be no memory
        const uint32_t D = d.cache.head_dim, G = d.cache.kv_heads, H = d.heads;
        check_cache(d.cache, "gm_attention: cache");
        require(D % 8 == 0 && D <= 256, "gm_attention takes heads of a multiple of 8 values up to 256");
        require(H && H % G == 0 && H <= 1u << 20, "gm_attention: heads are a multiple of kv_heads");
        require((uint64_t)n * H <= 1u << 30, "gm_attention: n * heads is at most 2^30");
        RowOps::check_rows(d.q, n, H * D, false, "gm_attention: q");
        RowOps::check_rows(d.out, n, H * D, true, "gm_attention: out");
        require(d.q.type == d.cache.type && d.out.type == d.cache.type, "gm_attention: q, out and the cache have one type");
        require(d.q.data != d.out.data || n == 1 || d.q.stride == d.out.stride, "gm_attention: rows in place have one stride");
        require(d.sequences && d.longest && d.longest <= n, "gm_attention: sequences, longest");
        require(d.starts || (uint64_t)d.sequences * d.longest == n, "gm_attention: without starts n is sequences * longest");
        require(d.lengths && (uintptr_t)d.lengths % 4 == 0 && (uintptr_t)d.starts % 4 == 0, "gm_attention: lengths and starts");
        require(d.table && (uintptr_t)d.table % 4 == 0 && d.table_width && d.table_stride <= uint64_t(1) << 40, "gm_attention: table");
        const uint64_t capacity = (uint64_t)d.table_width * d.cache.page_size;
        require(capacity < 1u << 29, "gm_attention: table_width * page_size is below 2^29");  // 2^25 tiles of 16 keys, 64 of them in 32 bits
        require(d.causal || !d.window, "gm_attention: a window without the causal mask");
        require(d.scale > 0 && std::isfinite(d.scale * 1.44269504088896341f), "gm_attention: scale");  // (times log2 e in the kernels)
        const bool wide = d.cache.type == GM_F32;
        const uint32_t group = H / G;
        const uint64_t rows = (uint64_t)d.longest * group;
        // Tiles of 16 rows of all sequences and cache heads. Rows past 16 of a sequence go to attend_tile if these tiles are
        // more than 512 or have more keys to read (as far as the table tells) than 2^18: below that the kernels of few rows,
        // which read a sequence's keys once for every 16 rows but start faster, are ahead (us, 8 cache heads: 64 rows of 4000
        // keys 18 against 24, of 16000 32 against 31; 256 rows of 2000 24 against 27, of 4000 40 against 29; 512 pairs of 300
        // keys 16 against 25, 1024 32 against 27). attend_tile loads straight to LDS, which wants addresses that are multiples
        // of four bytes (4096 tokens of 32 heads over 8 160 us, over a cache off by two bytes 2360; 256 tokens 14 and 26).
        const uint64_t row_tiles = (rows + kFewRows - 1) / kFewRows;
        const unsigned __int128 pairs = (unsigned __int128)row_tiles * d.sequences * G;
        const bool direct = !wide && !(((uintptr_t)d.cache.k | (uintptr_t)d.cache.v | (d.cache.pages > 1 ? 2 * d.cache.page_stride : 0) |
                                        (G > 1 ? 2 * d.cache.head_stride : 0) | (d.cache.page_size > 1 ? 2 * d.cache.token_stride : 0)) & 3);
        const bool many = direct && rows > kFewRows && (pairs > kFewPairs || pairs * capacity > kFewKeys), few = !many || d.starts;
        Constants &c = l.c;
        c.set(0, d.q.data);
        c.set64(2, d.q.stride);
        c.set(4, d.out.data);
        c.set64(6, d.out.stride);
        c.set(8, d.cache.k);
        c.set(10, d.cache.v);
        set_cache(c, d.cache, 12);
        c.set(18, d.table);
        c.set64(20, d.table_stride);
        c.set(22, d.lengths);
        c.set(24, d.starts);
        c.set(29, group);
        c.set(30, D);
        c.set(31, G);
        c.set(32, d.sequences);
        c.set(33, d.longest);
        c.set(34, n);
        c.set(35, d.cache.pages);
        c.set(36, d.cache.page_size);
        c.set(37, d.table_width);
        c.set(39, std::min(d.window, 1u << 30));
        c.set(40, d.scale * 1.44269504088896341f);
        c.set(43, d.cache.type);
        // Whether 32 bits span the cache: keys' offsets take half the work then.
        const auto reach = [](uint32_t count, uint64_t stride) { return count > 1 ? (unsigned __int128)(count - 1) * stride : 0; };
        const auto span = reach(d.cache.pages, d.cache.page_stride) + reach(G, d.cache.head_stride) + reach(d.cache.page_size, d.cache.token_stride) + D;
        c.set(38, (d.causal ? 1u : 0u) | (span <= (uint64_t(1) << 32) / (wide ? 4 : 2) ? 2u : 0u));
        c.set(46, many ? kFewRows + 1 : 0u);
        // Division of key numbers below 2^29 by the page size: with 2^(s-1) < size <= 2^s the reciprocal 2^(29+s) / size, rounded
        // up by less than one, is off by less than i / 2^(29+s) < 1 / size in i times it.
        uint32_t shift = 0;
        while ((uint64_t(1) << shift) < d.cache.page_size) ++shift;
        c.set(52, shift);
        c.set(59, (uint32_t)(((uint64_t(1) << (29 + shift)) + d.cache.page_size - 1) / d.cache.page_size));
        const int size = D <= 64 ? 0 : D <= 128 ? 1 : 2, type = d.cache.type;
        uint64_t need = 0, join = 0, groups = 0;
        bool short_keys = false;
        if (few) {
            const uint32_t keys = wide && D > 64 ? 16 : 32, tiles = many ? 1 : (uint32_t)row_tiles;
            const uint64_t entries = (uint64_t)d.sequences * tiles;
            require(entries * G < 1u << 31, "gm_attention: too many sequences");
            groups = entries * G;
            c.set(42, tiles);
            c.set(44, keys);
            // Where one group's waves (eight, but for heads above 128 values) take all keys of 16 rows as fast as several and a
            // join, by the pairs of row tiles and cache heads that there are to fill the GPU.
            const uint64_t few_pairs = entries * G;
            const uint32_t alone = wide ? (few_pairs >= kWidePairs ? 4096 : 512)
                                        : (uint32_t)std::min<uint64_t>(D > 128 ? 1024 : 2048, std::max<uint64_t>(896, 16 * few_pairs));
            short_keys = capacity <= alone;
            const uint32_t resident = (wide ? 256 : kResident[size]) * (!wide && few_pairs >= kResident[size] / 2 ? kPerGroup : 1);
            if (entries <= kEntries && entries * G < 2 * resident && !short_keys) {
                groups += resident;
                c.set(41, resident);
                c.set(45, (wide ? 2 * kLeast : kLeast) / keys);
                c.set(57, (wide ? alone : kLeast) / keys);
                need = plan_at(D);
                const uint32_t most = (uint32_t)std::min<uint64_t>(kFewRows, rows);
                c.set(56, most);
                join = std::min<uint64_t>(entries, resident / G) * G * most;
            }
        }
        c.set(47, (uint32_t)join);
        uint64_t units = 0;
        if (many) {
            // Tiles of rows: of every sequence as many as of the longest, or by their tokens, one more each; and what splits add.
            const uint64_t tiles = (rows + kTileRows - 1) / kTileRows, entries = tiles * d.sequences;
            units = (uint64_t)n * group / kTileRows + std::min<uint64_t>(d.sequences, (uint64_t)n * group / (kFewRows + 1));
            units = std::min(units, entries) + 512 / G + 1;
            require(units <= kUnits && units * G < 1u << 31, "gm_attention: n * heads / kv_heads / 128 + sequences is at most 2^18 - 1024");
            need = workspace(H, G, D);
            c.set64(50, (uint64_t)(uintptr_t)d.workspace + slots_at(D));
            c.set(54, kSlots / G);
            c.set(55, D > 128 ? 32u : 64u);
            c.set(58, entries * G >= kTilePairs ? 16u : 4u);
            if (entries <= kEntries) {
                c.set(28, (uint32_t)tiles);
            } else {
                c.set64(48, (uint64_t)(uintptr_t)d.workspace + plan_at(D));
                c.set(53, (uint32_t)units);
                l.add("attend_plan", 1);
            }
            join += 1024;
        }
        require(!need || (d.workspace && d.workspace_bytes >= need && (uintptr_t)d.workspace % 256 == 0), "gm_attention: workspace");
        c.set(26, d.workspace);
        static const char *const few_names[3][3] = {{"attend_f32_64", "attend_f32_128", "attend_f32_256"},
                                                    {"attend_few_b64", "attend_few_b128", "attend_few_b256"},
                                                    {"attend_few_h64", "attend_few_h128", "attend_few_h256"}};
        static const char *const tile_names[3][3] = {{}, {"attend_tile_b64", "attend_tile_b128", "attend_tile_b256"},
                                                     {"attend_tile_h64", "attend_tile_h128", "attend_tile_h256"}};
        static const char *const short_names[3][3] = {{"attend_f32_64", "attend_f32_128", "attend_f32_256"},
                                                      {"attend_short_b64", "attend_short_b128", "attend_few_b256"},
                                                      {"attend_short_h64", "attend_short_h128", "attend_few_h256"}};
        if (few) l.add((short_keys ? short_names : few_names)[type][size], groups);
        if (many) l.add(tile_names[type][size], units * G);
        if (join) l.add("attend_join", join);
        return l;
    }
    // Few rows' keys: groups that the GPU holds, by the heads' size, and parts for each of them where row tiles and heads (half
    // as many or more) differ in keys (us: 64 sequences of 91 to 8192 keys 110 with one part, 98 with two, of 4000 each 198 and
    // 207; 4 of 4000 each 19.5 and 23).
    static constexpr uint32_t kResident[3] = {512, 512, 256}, kPerGroup = 2;
    // Keys that make a part (twice as many in fp32). 1500 keys of one sequence: 11.1 us with 128, 12.0 with 256, 14.0 with 512.
    static constexpr uint32_t kLeast = 128;
    // Keys of one group alone against several and a join, us, replayed (outside a graph the second launch costs its caller 2
    // more), 8 heads of 128 values: one sequence of 640 keys 10.9 and 10.8, of 1024 14.0 and 10.9; 8 of 1024 15.1 and 15.4, of
    // 2048 24.6 and 19.5; 16 of 2048 26 and 31, of 4000 71 and 59; 32 of 2048 42 and 49. Heads of 256, 16 of 1024 31 and 38, of
    // 1536 55 and 52. fp32: 8 tiles of 512 keys 11.9 and 13.0, of 1024 18 and 13; 112 of 1024 20 and 27, of 4096 58 and 65.
    static constexpr uint32_t kWidePairs = 96;
    static constexpr uint32_t kFewKeys = 1u << 18, kFewPairs = 512;
    // Many rows: tiles of rows and heads from which on a part has 16 tiles of keys at least, otherwise 4 (us: 1023 tokens of 32
    // heads alone, 256 such tiles, 44.5 with 4 and 34.6 with 16; 64 tokens of 4096 keys, 16 tiles, 28.4 and 36.5).
    static constexpr uint32_t kTilePairs = 128;
};

}  // namespace gyro
