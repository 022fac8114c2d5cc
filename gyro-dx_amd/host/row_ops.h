// The operators around the MoE layers (gm_linear, gm_block_norm, gm_logprobs): argument checks, the choice of a
// build, its constants and grid. The engine launches what they return. Their kernels (csrc/kernels/q4.h, block_norm.h,
// logprobs.h) take every address in the launch's constants, so a call needs no table entry and may be captured.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstring>
#include <functional>
#include <map>
#include <string>
#include <vector>

#include "device.h"
#include "gyro_ops.h"

namespace gyro {

inline void require(bool ok, const char *what) {
    if (!ok) throw NativeError((gd_result)0x80070057u, what);  // E_INVALIDARG
}

// The constants of a launch, set by position.
struct Constants {
    uint32_t w[60] = {};
    void set(int i, uint32_t v) { w[i] = v; }
    void set64(int i, uint64_t v) {
        w[i] = (uint32_t)v;
        w[i + 1] = (uint32_t)(v >> 32);
    }
    void set(int i, const void *p) { set64(i, (uint64_t)(uintptr_t)p); }
    void set(int i, float v) { std::memcpy(&w[i], &v, 4); }
};

// A launch: the kernel, its constants and grid (x 0: nothing to do), and one of the same constants after it.
struct Launch {
    const char *kernel = nullptr, *next = nullptr;
    Constants c;
    uint32_t x = 0, y = 0, next_x = 0, next_y = 0;
};

struct Matrix {
    Buffer data;  // quants, scales, minima (q4_repack)
    uint32_t rows = 0, cols = 0, lg = 0, tiles = 0, chunks = 0;
    bool gated = false, mins = false;
    uint64_t scales = 0, minima = 0;  // byte offsets
};

class RowOps {
  public:
    std::map<std::string, std::string, std::less<>> files;  // kernels not loaded yet
    std::map<std::string, gd_pipeline *, std::less<>> pipes;
    std::vector<Matrix> matrices;

    static bool owns(const std::string &kernel) {
        for (const char *prefix : {"mv_q4", "mm_q4", "q4_repack", "block_norm", "logprobs"})
            if (kernel.rfind(prefix, 0) == 0) return true;
        return false;
    }
    using Loader = std::function<gd_pipeline *(const std::string &file)>;
    Loader loader;
    void load(const std::string &prefix) {
        for (auto it = files.begin(); it != files.end();) {
            if (it->first.rfind(prefix, 0) != 0) {
                ++it;
                continue;
            }
            pipes[it->first] = loader(it->second);
            it = files.erase(it);
        }
    }

    // ---- linear ----

    static uint64_t layout(Matrix &m) {
        const uint64_t units = (uint64_t)m.tiles * m.chunks, per = 128u >> m.lg;
        m.scales = units * 1024;
        m.minima = m.scales + units * 16 * per * 2;
        return m.mins ? m.minima + units * 16 * per * 2 : m.minima;
    }
    // Source bytes of a matrix's quants, and of its scales or minima (format GM_MATRIX_Q4).
    static uint64_t quant_bytes(const gm_matrix_desc &d) {
        const uint64_t n = (uint64_t)d.rows * d.cols;
        return d.format == GM_MATRIX_Q4_0 ? n / 32 * 18 : d.format == GM_MATRIX_Q4_1 ? n / 32 * 20 : n / 2;
    }
    static uint64_t scale_bytes(const gm_matrix_desc &d) { return (uint64_t)d.rows * (d.cols / d.group) * 2; }

    static Matrix describe(const gm_matrix_desc &d) {
        require(d.format <= GM_MATRIX_Q4, "unknown matrix format");
        require(d.group == 32 || (d.format == GM_MATRIX_Q4 && (d.group == 64 || d.group == 128)),
                "a matrix's group is 32, or 64 or 128 in the format of separate scales");
        require(d.rows && d.cols && d.cols % d.group == 0, "a matrix has rows, and columns in whole groups");
        require(d.rows <= 1u << 26 && d.cols <= 1u << 20, "a matrix has at most 2^26 rows and 2^20 columns");
        const bool arrays = d.format == GM_MATRIX_Q4;
        require(d.quants && (!arrays || d.scales), "a matrix needs its quants and scales");
        require(arrays || (!d.scales && !d.mins && !d.up_scales && !d.up_mins), "GGUF blocks hold their own scales");
        require(d.up_quants ? (!arrays || d.up_scales) && !d.mins == !d.up_mins : !d.up_scales && !d.up_mins,
                "a gated pair's matrices have one format");
        Matrix m;
        m.rows = d.rows;
        m.cols = d.cols;
        m.lg = d.group == 32 ? 5 : d.group == 64 ? 6 : 7;
        m.gated = d.up_quants != nullptr;
        m.mins = d.format == GM_MATRIX_Q4_1 || (arrays && d.mins);
        m.tiles = (d.rows + 15) / 16 * (m.gated ? 2u : 1u);
        m.chunks = (d.cols + 127) / 128;
        const uint64_t limit = uint64_t(4) << 30;
        require(layout(m) <= limit && quant_bytes(d) <= limit, "a matrix takes at most 4 GiB");
        return m;
    }

    const Matrix &matrix(uint32_t i) const {
        require(i < matrices.size() && matrices[i].data.handle, "no such matrix");
        return matrices[i];
    }
    uint32_t keep(Matrix &&m) {
        for (uint32_t i = 0; i < matrices.size(); ++i)
            if (!matrices[i].data.handle) {
                matrices[i] = std::move(m);
                return i;
            }
        matrices.push_back(std::move(m));
        return (uint32_t)matrices.size() - 1;
    }

    static void check_rows(const gm_rows &r, uint32_t n, uint32_t cols, bool output, const char *what) {
        require(r.data != nullptr && r.type <= GM_F16, what);
        const uint64_t size = r.type == GM_F32 ? 4 : 2;
        require((uintptr_t)r.data % size == 0, what);
        require(r.stride <= uint64_t(1) << 40, what);
        require(!output || n <= 1 || r.stride >= cols, what);
    }

    static Launch linear(const Matrix &m, uint32_t cus, const gm_rows &x, uint32_t n, const gm_rows &y, uint32_t act,
                         uint32_t accumulate, float scale) {
        Launch l;
        if (!n) return l;  // of no rows there may be no memory
        check_rows(x, n, m.cols, false, "gm_linear: x");
        check_rows(y, n, m.rows, true, "gm_linear: y");
        require(n == 1 || x.stride <= 1u << 24, "gm_linear: x's rows are at most 2^24 values apart");
        require(act <= GM_ACT_SIGMOID && (!m.gated || act == GM_ACT_NONE), "gm_linear: act");
        require(n <= 1u << 18, "gm_linear takes at most 2^18 tokens");
        Constants &c = l.c;
        c.set64(0, m.data.gpu);
        c.set64(2, m.data.gpu + m.scales);
        c.set64(4, m.mins ? m.data.gpu + m.minima : 0);
        c.set(6, m.tiles);
        c.set(7, m.chunks);
        c.set(8, m.lg);
        c.set(9, m.cols);
        c.set(10, m.rows);
        c.set(11, m.gated ? 1u : 0u);
        c.set(12, x.data);
        c.set64(14, x.stride);
        c.set(16, x.type);
        c.set(17, n);
        c.set(18, y.data);
        c.set64(20, y.stride);
        c.set(22, y.type);
        c.set(23, act);
        c.set(24, accumulate ? 1u : 0u);
        c.set(25, scale);
        // Tokens that share a pass of mv_q4 over the weights.
        const uint32_t per = x.type == GM_F32 ? 5u : x.type == GM_F16 ? 8u : 16u, passes = (n + per - 1) / per;
        // mm_q4's few large groups take 1.1 to 1.4 us a chunk however little there is to do; mv_q4's time grows with tiles
        // and passes. They meet near (fp32, bf16, binary16) 12, 7 and 8 tile passes per compute unit. us at 2048
        // columns, mv / mm: 2048 rows of 64, 128 and 512 fp32 tokens 16.6 / 23.4, 28.1 / 23.6 and 90.3 / 25.3; 8192 rows of
        // 17 and 32 16.3 / 23.4 and 26.8 / 23.6; of 32 and 64 bf16 tokens 12.2 / 18.6 and 21.4 / 19.2, binary16 18.4 / 18.9
        // and 33.5 / 19.4. Measured at 512 to 32768 rows of 2048 columns and 2048 rows of 512, on 6 to 512 tokens; the worst
        // choice there is mm_q4 for 32768 rows and 6 fp32 tokens (21.8 / 23.8). Longer rows were not measured.
        // (The grid of more than 2^20 tiles would be too wide for mm_q4.)
        static const uint32_t meet[] = {12, 7, 8};
        const uint32_t blocks = (m.tiles + 15) / 16;
        if (passes > 1 && blocks <= 65535 && (uint64_t)m.tiles * passes > (uint64_t)meet[x.type] * cus) {
            static const char *const names[3][3] = {{"mm_q4_f32", "mm_q4_f64", "mm_q4_f128"},
                                                    {"mm_q4_b32", "mm_q4_b64", "mm_q4_b128"},
                                                    {"mm_q4_h32", "mm_q4_h64", "mm_q4_h128"}};
            // 16 T tokens to a group: the fewest rounds of two groups per unit, by a step's vector instructions.
            uint32_t tokens = 16;
            uint64_t cost = ~0ull;
            const uint32_t most = x.type != GM_F32 ? 4 : m.lg == 5 ? 2 : 3;  // mm_q4_body's
            for (uint32_t t = 1; t <= most; ++t) {
                const uint64_t groups = (uint64_t)blocks * ((n + 16 * t - 1) / (16 * t));
                const uint64_t k = (groups + 2 * cus - 1) / (2 * cus) * (28 + 16 * t);
                if (k <= cost) {
                    cost = k;
                    tokens = 16 * t;
                }
            }
            c.set(26, tokens / 16);
            l.kernel = names[x.type][m.lg - 5];
            l.x = blocks;
            l.y = (n + tokens - 1) / tokens;
            return l;
        }
        // Waves that share a tile's columns: two, or as few as leave every unit its 16 waves (one fp32 token at 2048 columns,
        // us at 1 / 2 / 4 / 8: 131072 rows 35.8 / 35.0 / 35.6 / 41.7, 32768 rows 18.2 / 12.3 / 11.3 / 12.9, 2048 rows 14.9 /
        // 9.6 / 7.0 / 6.2).
        uint32_t wk = m.chunks > 1 ? 2 : 1;
        while (wk < 8 && wk * 2 <= m.chunks && m.tiles / 2 * wk < 16 * cus) wk *= 2;
        c.set(26, wk);
        const uint32_t run = 2 * (8 / wk), runs = (m.tiles + run - 1) / run;
        l.kernel = m.mins ? "mv_q4_m" : "mv_q4";
        l.x = std::min(runs, 2 * cus);
        l.y = passes;
        return l;
    }

    // ---- block norm ----

    static Launch block_norm(const gm_block_norm_desc &d, uint32_t n) {
        Launch l;
        if (!n) return l;  // of no rows there may be no memory
        require(d.E && d.E <= 16384, "gm_block_norm takes rows of 1 to 16384 values");
        require(d.out.data || d.normed.data, "gm_block_norm: no output");
        check_rows(d.x, n, d.E, false, "gm_block_norm: x");
        if (d.h.data) check_rows(d.h, n, d.E, false, "gm_block_norm: h");
        if (d.out.data) check_rows(d.out, n, d.E, true, "gm_block_norm: out");
        if (d.normed.data) check_rows(d.normed, n, d.E, true, "gm_block_norm: normed");
        // In place a thread writes where it has read; rows of another layout would reach into its neighbours'.
        for (const gm_rows *in : {&d.x, &d.h})
            for (const gm_rows *to : {&d.out, &d.normed})
                require(!in->data || in->data != to->data || (in->type == to->type && (n == 1 || in->stride == to->stride)),
                        "gm_block_norm: rows in place have one type and stride");
        require(d.gate_kind <= GM_GATE_VALUE && (d.gate_act == GM_ACT_NONE || d.gate_act == GM_ACT_SIGMOID), "gm_block_norm: gate");
        const bool gate = d.gate_kind != GM_GATE_NONE;
        require(d.h.data || (!gate && !d.post), "gm_block_norm: a gate or a post norm without h");
        if (gate) check_rows(d.gate, n, d.E, false, "gm_block_norm: gate");
        require(d.post || !d.post_weight, "gm_block_norm: a post weight without the post norm");
        require((uintptr_t)d.post_weight % 4 == 0 && (uintptr_t)d.pre_weight % 4 == 0, "gm_block_norm: weights");
        require(d.post_eps >= 0 && d.pre_eps >= 0, "gm_block_norm: eps");
        Constants &c = l.c;
        c.set(0, d.h.data);
        c.set64(2, d.h.stride);
        c.set(4, d.x.data);
        c.set64(6, d.x.stride);
        c.set(8, d.out.data);
        c.set64(10, d.out.stride);
        c.set(12, d.normed.data);
        c.set64(14, d.normed.stride);
        c.set(16, d.post_weight);
        c.set(18, d.pre_weight);
        if (gate) c.set(20, d.gate.data);
        c.set64(22, d.gate_kind == GM_GATE_CHANNEL ? 0 : d.gate.stride);
        c.set(24, d.gate_kind >= GM_GATE_CHANNEL ? 1u : 0u);
        c.set(25, d.h.type | d.x.type << 4 | d.out.type << 8 | d.normed.type << 12 | d.gate.type << 16);
        c.set(26, (d.post ? 1u : 0u) | (d.gate_act == GM_ACT_SIGMOID ? 2u : 0u));
        c.set(27, d.E);
        c.set(28, d.post_eps);
        c.set(29, d.pre_eps);
        c.set(30, d.scale);
        c.set(31, n);
        l.kernel = d.E <= 2048 ? "block_norm_s" : d.E <= 4096 ? "block_norm" : "block_norm_l";
        l.x = std::min(n, 65535u);
        l.y = (uint32_t)(((uint64_t)n + 65534) / 65535);
        return l;
    }

    // ---- log probabilities ----

    // Groups that share a row: four for each of 256 compute units, each of a group's four waves with a batch of 1024 logits
    // at least. Fewer leave units idle, more pay for their lists twice (131072 logits, top 5, us at 1 / 2 / 4 / 8 / 16 groups
    // a row: one row 37 / 25 / 17 / 13 / 11, 128 rows 45 / 31 / 25 / 22 / 25, 512 rows 61 / 57 / 62 / 63 / 73).
    static uint32_t logprobs_parts(uint32_t n, uint32_t V) {
        const uint32_t batches = (V + 1023) / 1024;
        return std::max(1u, std::min({32u, (batches + 3) / 4, 1024 / std::max(1u, n)}));
    }
    static uint64_t logprobs_part_bytes(uint32_t top) { return 16 + 8ull * ((top + 1) & ~1u); }
    // Bytes that every call of up to n rows finds enough: the most parts of any such call, p to each of the most rows that
    // are split into p (so at most 1024 parts).
    static uint64_t logprobs_workspace(uint32_t n, uint32_t V, uint32_t top) {
        uint64_t most = 0;
        for (uint32_t p = logprobs_parts(1, V); p > 1; --p) most = std::max(most, (uint64_t)p * std::min(n, 1024 / p));
        return most * logprobs_part_bytes(top);
    }

    static Launch logprobs(const gm_logprobs_desc &d, uint32_t n) {
        Launch l;
        if (!n) return l;  // of no rows there may be no memory
        require(d.V && d.V < 1u << 31, "gm_logprobs: V");
        check_rows(d.logits, n, d.V, false, "gm_logprobs: logits");
        require(d.scale > 0 && std::isfinite(d.scale), "gm_logprobs: scale");
        require(d.given <= 64 && d.top <= 64 && d.top <= d.V, "gm_logprobs: given, top");
        require(!d.given || (d.tokens && d.logprobs && (uintptr_t)d.tokens % (d.tokens_64 ? 8 : 4) == 0 &&
                             (uintptr_t)d.logprobs % 4 == 0 && (n <= 1 || d.logprobs_stride >= d.given)),
                "gm_logprobs: tokens and logprobs");
        require(!d.top || (d.top_ids && d.top_logprobs && (uintptr_t)d.top_ids % 4 == 0 &&
                           (uintptr_t)d.top_logprobs % 4 == 0 && (n <= 1 || d.top_stride >= d.top)),
                "gm_logprobs: top_ids and top_logprobs");
        require((uintptr_t)d.entropy % 4 == 0 && (d.given || d.entropy || d.top), "gm_logprobs: no output");
        const uint32_t parts = logprobs_parts(n, d.V);
        const uint64_t need = parts == 1 ? 0 : (uint64_t)n * parts * logprobs_part_bytes(d.top);
        require(!need || (d.workspace && d.workspace_bytes >= need && (uintptr_t)d.workspace % 256 == 0),
                "gm_logprobs: workspace");
        Constants &c = l.c;
        c.set(0, d.logits.data);
        c.set64(2, d.logits.stride);
        c.set(4, d.logits.type);
        c.set(5, d.V);
        c.set(6, d.scale);
        c.set(7, d.top);
        c.set(8, d.tokens);
        c.set64(10, d.tokens_stride);
        c.set(12, d.given);
        c.set(13, d.tokens_64 ? 1u : 0u);
        c.set(14, d.logprobs);
        c.set64(16, d.logprobs_stride);
        c.set(18, d.entropy);
        c.set(20, d.top_ids);
        c.set(22, d.top_logprobs);
        c.set64(24, d.top_stride);
        c.set(26, n);
        c.set(27, parts);
        c.set(28, d.workspace);
        l.kernel = d.logits.type == GM_F32 ? "logprobs" : d.logits.type == GM_BF16 ? "logprobs_b" : "logprobs_h";
        l.x = std::min(n, 65535u);
        l.y = (uint32_t)(((uint64_t)n + 65534) / 65535) * parts;
        if (parts > 1) {
            l.next = "logprobs_join";
            l.next_x = l.x;
            l.next_y = l.y / parts;
        }
        return l;
    }
};

}  // namespace gyro
