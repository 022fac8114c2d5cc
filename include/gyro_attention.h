/*
 * gyro_attention: positions, a paged cache and the attention over it, beside the operators of gyro_ops.h and on the same
 * terms: rows in device memory, launches queued on the caller's stream, nothing allocated, waited for or copied by a call
 * (gm_add_rotary and gm_release_rotary aside), captures, errors and serialised calls as that header states them.
 *
 * What the reference's GPU path has as rope_neox, store_f16, attn_chunk and attn_merge (shaders/engine/attn.hlsl:14-340) for
 * one sequence, one layout and a contiguous cache.
 */
#ifndef GYRO_ATTENTION_H
#define GYRO_ATTENTION_H

#include "gyro_ops.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rotary positions: of a head's first 2 `pairs` values, pair j turns by position * frequencies[j] (radians, host memory, of
 * magnitude below 2^31), and is multiplied by `scale`:
 *   (y1, y2) = scale (x1 cos a - x2 sin a, x1 sin a + x2 cos a)
 * GM_ROTARY_HALF: x1 = x[j], x2 = x[pairs + j]; GM_ROTARY_INTERLEAVED: x1 = x[2 j], x2 = x[2 j + 1]. The values behind
 * them are copied. Angles are exact to 2^-27 of a turn for positions below 2^36 in magnitude (64-bit fixed point, modulo whole
 * turns). */
enum { GM_ROTARY_HALF = 0, GM_ROTARY_INTERLEAVED = 1 };
/* Uploads frequencies (1 to 512 pairs) and returns their index. */
GM_API int gm_add_rotary(gm_engine *e, const double *frequencies, uint32_t pairs, uint32_t layout, float scale,
                         uint32_t *out_index);
/* Frees them once the device's work is done; the index may come again. A graph captured with them may not be replayed. */
GM_API int gm_release_rotary(gm_engine *e, uint32_t rotary);

/* Rows of `heads` heads of `head_dim` <= 1024 neighbouring values: y[t] is x[t] turned by positions[t] (int32, or int64 with
 * positions_64), in fp32 and rounded once. y may be x's rows, of the same type and stride; it overlaps x in no other way.
 * n * heads is below 2^31. */
typedef struct gm_rotary_desc {
    uint32_t rotary, heads, head_dim, positions_64;
    gm_rows x, y;
    const void *positions;
} gm_rotary_desc;
GM_API int gm_rotary(gm_engine *e, const gm_rotary_desc *desc, uint32_t n, void *stream);

/* Keys and values in `pages` pages of `page_size` tokens each: the key of token i of page p and head g starts at
 * k + p page_stride + g head_stride + i token_stride (values; at most 2^40 each), its head_dim values are neighbours;
 * values likewise at v. k and v are aligned to their type. (Attention of prompts over a 16-bit cache takes up to 15 times as
 * long where k, v or a stride is no multiple of four bytes.) pages * page_size is below 2^31. */
typedef struct gm_cache {
    void *k, *v;
    uint32_t type; /* GM_F32, GM_BF16, GM_F16 */
    uint32_t pages, page_size, kv_heads, head_dim, reserved;
    uint64_t page_stride, head_stride, token_stride;
} gm_cache;

/* New tokens' keys and values, rows of kv_heads heads, into the cache: k turned by its position (rotary GM_NO_ROTARY: as it
 * is) and v go to slot slots[t] = page * page_size + place, rounded once to the cache's type. A slot outside the cache
 * (negative: a padded token) is skipped. Of two tokens with one slot either's values may stay, value by value. With q (rows
 * of `heads` heads, of every token) also q_out = q turned: q_out may be q's rows, as gm_rotary's y. k, v and q have one type.
 * slots int32, or int64 with slots_64; positions (absent without a rotary) alike. head_dim is at most 1024, n times the
 * heads of all three below 2^31; the cache's elements must be apart for different (page, head, token), its keys from its
 * values, and both from all inputs. */
#define GM_NO_ROTARY 0xffffffffu
typedef struct gm_cache_append_desc {
    gm_cache cache;
    uint32_t rotary, heads, slots_64, positions_64;
    gm_rows k, v, q, q_out;
    const void *slots, *positions;
} gm_cache_append_desc;
GM_API int gm_cache_append(gm_engine *e, const gm_cache_append_desc *desc, uint32_t n, void *stream);

/* Attention of new tokens over a paged cache that already holds theirs. q and out: rows of `heads` heads (a multiple of
 * kv_heads; head h reads the cache's head h / (heads / kv_heads)) of head_dim values, a multiple of 8 up to 256, of the
 * cache's type. Sequence b has the tokens starts[b] .. starts[b + 1] - 1 of q (int32 [sequences + 1], not falling), or,
 * with starts NULL, `longest` tokens from b * longest on (then n = sequences * longest); `longest`, at most n, is at least
 * every sequence's count of tokens (of more, the first `longest` are certain to be computed, the rest may be left). Its keys
 * are the first lengths[b] places (int32, the new tokens' own among them) of the pages table[b * table_stride + i],
 * i < table_width (int32; cut to table_width * page_size, which is below 2^29).
 * Token i of q tokens stands at p = lengths[b] - q + i and sees the keys j <= p with `causal`, else all of its sequence's;
 * with a window w > 0 (and causal) only j > p - w. A key on a page outside the cache is seen by no token.
 *   out = sum_j softmax_j(scale q . k_j) v_j   (0 < scale < 2^127)
 * A token that sees no key, or only keys whose score is -infinity (in fp32, times log2 e), has zeros. What is not seen does
 * not count, NaNs and infinities among it. Rows of q behind the last sequence's are left in out as they were. Products of
 * 16-bit types are exact and summed in fp32, as are the softmax's statistics; its weights may be rounded to the type before
 * they meet v, in binary16, which has no smaller ones, by up to 2^-36 of a row's largest; an infinite value times a weight that
 * is zero then is NaN. out may be q's rows, of the same stride; it overlaps nothing else. n * heads is at most 2^30, and
 * n * heads / kv_heads / 128 + sequences at most 2^18 - 1024; sequences * kv_heads, in fp32 and over caches not aligned to
 * four bytes times the tiles of 16 rows in longest * heads / kv_heads, is below 2^31.
 * The workspace (256-byte aligned, of gm_attention_workspace(heads, kv_heads, head_dim) bytes, which serve every call of that
 * shape) holds nothing between calls; calls that may overlap, replayed graphs among them, take one each. */
typedef struct gm_attention_desc {
    gm_cache cache;
    gm_rows q, out;
    uint32_t heads, sequences, longest, causal, window;
    float scale;
    const int32_t *table;
    uint64_t table_stride;
    const int32_t *lengths, *starts;
    uint32_t table_width, reserved;
    void *workspace;
    uint64_t workspace_bytes;
} gm_attention_desc;
GM_API uint64_t gm_attention_workspace(uint32_t heads, uint32_t kv_heads, uint32_t head_dim);
GM_API int gm_attention(gm_engine *e, const gm_attention_desc *desc, uint32_t n, void *stream);

#ifdef __cplusplus
}
#endif
#endif
