// Rows of logits to the log probabilities of given tokens, the entropy and the top alternatives: with m = max x,
// d = scale (x - m) (the difference first: the scale may not take the type's lowest value out of range),
// S = sum exp(d), T = sum d exp(d):
//   logprob[j] = d[token j] - log S,   entropy = log S - T / S,   the `top` largest x, equal ones by id.
// One group per row. S and T are running sums: a larger maximum rescales them.
// Constants: 0 x 2 x stride 4 type 5 V 6 scale (fp32 bits) 7 top 8 tokens 10 tokens' stride 12 given 13 token type
// (0 int32, 1 int64) 14 logprob 16 logprob stride 18 entropy (0: none) 20 ids 22 top logprobs 24 top stride 26 n.
#include "rows.h"

struct LpState {
    float m, s, t;
};
__device__ __forceinline__ LpState lp_join(const LpState &p, const LpState &q, float scale) {
    LpState o;
    o.m = fmaxf(p.m, q.m);
    // At least -1e30, so that a term of exp 0 stays 0 and no NaN.
    auto diff = [&](const LpState &r) {
        const float d = scale * (r.m - o.m);
        return r.s == 0.f ? 0.f : d < -1e30f ? -1e30f : d;
    };
    const float dp = diff(p), dq = diff(q);
    const float ep = __expf(dp), eq = __expf(dq);
    o.s = p.s * ep + q.s * eq;
    o.t = ep * (p.t + p.s * dp) + eq * (q.t + q.s * dq);
    return o;
}
// Value i's place in the order: falling values, NaNs first, equal ones by index. Never 0, and below the start ~0.
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t i) {
    uint32_t u = gd_f32_bits(x + 0.0f);
    u = x != x ? 0xfffffffeu : u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t)u << 32 | (uint32_t)~i;
}

GD_PIPELINE_NAMED(logprobs, 256) {
    __shared__ LpState st[4];
    __shared__ uint64_t best[4];
    const uint32_t V = a.c[5], type = a.c[4], top = a.c[7], lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint64_t row = (uint64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (row >= a.c[26]) return;
    const float scale = gd_bits_f32(a.c[6]);
    const uint64_t X = gd_addr(a, 0) + ((row * gd_addr(a, 2)) << row_shift(type));
    LpState p = {-INFINITY, 0.f, 0.f};
    for (uint32_t i = threadIdx.x; i < V; i += 256u) {
        const float x = row_load(X, i, type);
        if (x == -INFINITY) continue;
        p = lp_join(p, LpState{x, 1.f, 0.f}, scale);
    }
    for (int o = 32; o > 0; o >>= 1) {
        const LpState q = {__shfl_xor(p.m, o, 64), __shfl_xor(p.s, o, 64), __shfl_xor(p.t, o, 64)};
        p = lp_join(p, q, scale);
    }
    if (lane == 0) st[wave] = p;
    __syncthreads();
    p = lp_join(lp_join(st[0], st[1], scale), lp_join(st[2], st[3], scale), scale);
    const bool none = p.s == 0.f;
    const float logs = none ? 0.f : logf(p.s);
    auto logprob = [&](float x) { return none ? -INFINITY : scale * (x - p.m) - logs; };
    if (threadIdx.x == 0 && gd_addr(a, 18)) gd_at<float>(gd_addr(a, 18))[row] = none ? 0.f : logs - p.t / p.s;
    if (threadIdx.x < a.c[12]) {
        const uint64_t at = row * gd_addr(a, 10) + threadIdx.x;
        const int64_t token = a.c[13] ? gd_at<const int64_t>(gd_addr(a, 8))[at] : gd_at<const int32_t>(gd_addr(a, 8))[at];
        float v = token < 0 ? 0.f : __builtin_nanf("");
        if (token >= 0 && token < (int64_t)V) v = logprob(row_load(X, (uint64_t)token, type));
        gd_at<float>(gd_addr(a, 14))[row * gd_addr(a, 16) + threadIdx.x] = v;
    }
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < top; ++k) {
        uint64_t b = 0;
        for (uint32_t i = threadIdx.x; i < V; i += 256u) {
            const uint64_t key = lp_key(row_load(X, i, type), i);
            if (key < last && key > b) b = key;
        }
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t q = (uint64_t)__shfl_xor((long long)b, o, 64);
            b = q > b ? q : b;
        }
        __syncthreads();
        if (lane == 0) best[wave] = b;
        __syncthreads();
        for (int w = 0; w < 4; ++w) b = best[w] > b ? best[w] : b;
        last = b;
        if (threadIdx.x == 0) {
            const uint32_t id = min(~(uint32_t)b, V - 1u);
            gd_at<uint32_t>(gd_addr(a, 20))[row * gd_addr(a, 24) + k] = id;
            gd_at<float>(gd_addr(a, 22))[row * gd_addr(a, 24) + k] = logprob(row_load(X, id, type));
        }
    }
}
