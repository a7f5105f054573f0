/*
 * arclight_paged.h - C ABI of a paged f16 KV cache: appending a batch's keys
 * and values to it, attention of each sequence's new tokens over it, and cells
 * moved and copied in it.
 *
 * The ring of arclight_kv.h gives a sequence one range of cells, as the
 * reference's llm_kv_cache does. A server of many requests keeps their cells
 * in pages of a pool instead: cell c of sequence s lies in page
 * table[s][c / P] of the pool, at cell c % P of the page. These operators
 * have no counterpart in the reference. What they compute is what
 * al_attn_inputs_f32 and al_fattn_f16 compute over a ring (the node run of
 * models/qwen3.cpp:211-227), with the tables and lengths read by the kernels,
 * so that a step captured into a HIP graph can be replayed while sequences
 * grow, come and go.
 *
 * The pools (one of K and one of V for each layer):
 *   f16 ne = [128, P, Hkv, n_pages], nb0 = 2, the other strides free
 *   multiples of 16 bytes, data 16-byte aligned. P is a multiple of 8, at most
 *   2^20, max_pages P at most 2^30 and max_pages P^2 below 2^38.
 *   A pool of [page][cell][head][128] is the layout of the ring: a sequence
 *   whose pages follow one another is a ring view for al_fattn_f16.
 * The table: i32 ne = [max_pages, n_seq], device, nb0 = 4. Entries behind a
 *   sequence's last page are not read and may hold anything. Pages may be
 *   shared by sequences that only read them.
 *
 * All data pointers are device pointers of the current device; no pointer is
 * kept after a call returns. Error convention as arclight_fattn.h. Calls
 * enqueue on `stream` without synchronizing. What a kernel finds wrong when
 * it runs (a page outside the pool, a length or position beyond the table, a
 * sequence index beyond n_seq) it does not access: it records it, and
 * al_device_errors() returns AL_ERR_INVALID after the stream completes.
 */
#ifndef ARCLIGHT_PAGED_H
#define ARCLIGHT_PAGED_H

#include <stdint.h>

#include "arclight_fattn.h"
#include "arclight_prologue.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Arguments of al_paged_append_f32. Row t of q, k and v is one token: the
 * one at position pos[t] of sequence seq[t]. Its key and value go to cell
 * pos[t] of that sequence.
 *   q      f32 [128, Hq, T]   (data NULL: no queries, q_out is not used)
 *   k, v   f32 [128, Hkv, T]
 *   q_w, k_w  f32 [128], the norm weights (data NULL: none)
 *   pos    i32 [T], device
 *   seq    i32 [T], device; negative: the row belongs to no sequence (a
 *          slot of a padded batch), and nothing is written for it
 *   q_out  f32 [128, Hq, T]
 *   norm   non-zero: q and k rows are RMS-normalised (eps) and weighted
 *          before the rotation; zero: rotated as they are (q_w and k_w have
 *          to be NULL)
 *   rope   NULL for no rotation
 * nb0 = 4 everywhere; rows of q, k, v and q_out at multiples of 4 bytes. T is
 * at most 2^24, Hq 4096. q_out may be q; it may not overlap it otherwise, nor
 * k or v.
 * q_out rows and cached keys have the bits that al_attn_inputs_f32 gives.
 * Two rows of one call that name the same cell leave one of the two there,
 * or parts of both.
 */
typedef struct al_paged_append_args {
    al_tensor q;
    al_tensor q_w;
    al_tensor k;
    al_tensor k_w;
    al_tensor v;
    al_tensor pos;
    al_tensor seq;
    al_tensor q_out;
    al_tensor k_pool;
    al_tensor v_pool;
    al_tensor table;
    float     eps;
    int32_t   norm;
    const al_rope_params * rope;
    void *    stream;
} al_paged_append_args;

int al_paged_append_f32(const al_paged_append_args * args);

/*
 * Arguments of al_paged_fattn_f16: attention of up to T new tokens of each of
 * n_seq sequences, the last ones of their cells.
 *   q       f32 ne = [128, T, Hq, n_seq], nb0 = 4, rows 16-byte aligned
 *   dst     f32 ne = [128, Hq, T, n_seq], nb0 = 4, rows 16-byte aligned
 *   lens    i32 [n_seq], device: cells of each sequence, the new tokens'
 *           among them
 *   counts  i32 [n_seq], device: new tokens of each sequence, 0 to T (data
 *           NULL: T each)
 *   sinks   f32 [Hq], or data NULL
 * Token t < counts[s] sees cells c < lens[s] - counts[s] + 1 + t. Rows of
 * tokens t >= counts[s] are left as they were (counts[s] = 0: an empty slot
 * of the batch, whose length is not looked at; a negative count is recorded
 * as an error, and the slot is empty too). A row that sees no cell is zero, with or without a sink
 * (al_fattn_f16 gives NaN without one). The logits are scale * q . k, or
 * logit_softcap * tanh(scale * q . k / logit_softcap) when logit_softcap is
 * not 0. What cells that a row does not see hold, NaN and infinities too,
 * does not reach it.
 * Hq is a multiple of Hkv, G = Hq / Hkv. T is at most 2^16, Hq 4096, T Hq
 * 2^22, n_seq 65535, T G / 64 Hkv 65535; T G^2 is below 2^32, n_seq max_pages
 * P / 32 below 2^31 (AL_ERR_UNSUPPORTED otherwise). dst may not overlap q.
 * T decides how the launch shares out the card, for every sequence: single
 * tokens beside a prompt are right, but slow. They belong in two calls over the
 * same buffers, one with T = 1 (views with ne = 1 there), each with a count of 0
 * for the other's sequences. 63 sequences of 4000 cells with one token and a
 * prompt of 2048, 32 heads over 8: 6.7 ms in one call, 0.2 + 0.2 ms in two.
 * Queries and probabilities are carried as pairs of f16, so that results are
 * those of f32 arithmetic (relative error about 1e-6), unlike al_fattn_f16's,
 * for finite operands: a row that sees a key which is not finite, and the dim
 * of a value which is not, may be NaN where f32 arithmetic gives an infinity
 * or the cell no weight. (al_paged_append_f32 stores what lies beyond f16's
 * range, 65504, as an infinity.)
 * A sequence whose length or count is recorded as an error has NaN rows, and
 * so have all rows that see a cell of a page outside the pool (others of that
 * sequence, which a wave or a workgroup takes with them, may be NaN too).
 * workspace: device scratch (al_paged_fattn_workspace_bytes), NULL: the
 * library's own for (current device, stream), as al_fattn_f16: then one
 * eager call of the same shapes has to come before a capture. Calls and
 * replays that share a workspace must be ordered on one stream. A workspace
 * needs no initial value; its first 256 KiB are not touched, so that it may
 * also be al_fattn_f16's, whose counters those are.
 */
typedef struct al_paged_fattn_args {
    al_tensor q;
    al_tensor k_pool;
    al_tensor v_pool;
    al_tensor table;
    al_tensor lens;
    al_tensor counts;
    al_tensor sinks;
    al_tensor dst;
    float     scale;
    float     logit_softcap;
    void *    stream;
    void *    workspace;
    uint64_t  workspace_bytes;
} al_paged_fattn_args;

int al_paged_fattn_f16(const al_paged_fattn_args * args);

/* Bytes of a caller's workspace for these arguments; 0 for refused ones. */
uint64_t al_paged_fattn_workspace_bytes(const al_paged_fattn_args * args);

/*
 * Which cells a token sees, where that is not all before it: layers with a
 * window, and trees of drafted tokens.
 *   window  positions that a token sees, its own among them (0: all)
 *   first   cells at the beginning that stay visible behind a window
 *   bits    i32 ne = [words, T, n_seq], nb0 = 4: bit u % 32 of word u / 32 of
 *           token t is set where t sees new token u (its own is u = t); words
 *           is (T + 31) / 32 or more, bits from counts[s] on are not looked at
 *           (data NULL: those up to and with itself)
 *   pos     i32 ne = [T, n_seq], nb0 = 4: the new tokens' positions (data NULL:
 *           the cells that they lie in). With bits and a window they are
 *           required, without bits refused.
 * With n = lens[s], b = n - counts[s] and p the token's position (pos[t][s],
 * without positions b + t), token t sees cell c of those before the new ones
 * (c < b) if c > p - window or c < first, and new token u (cell b + u) if its
 * bit is set (without bits: u <= t) and its position is above p - window or
 * below first. Positions have to lie in b to n - 1 where a window needs them:
 * the rows of others are recorded as errors and NaN.
 * Pages are looked up for every new cell, for the first cells, and from the
 * first window's beginning on: the lowest of the tokens', with bits that of a
 * token at position b. What the table says of other pages is not looked at, so
 * that they may have been freed.
 */
typedef struct al_paged_sees {
    int32_t   window;
    int32_t   first;
    al_tensor bits;
    al_tensor pos;
} al_paged_sees;

/* al_paged_fattn_f16 of what `sees` says instead of all cells before a token.
 * Its cost goes by the cells that are seen, not by the sequences' lengths. (For
 * small calls of several query rows the table's width, max_pages, is what the
 * kernel is chosen by.) */
int al_paged_fattn_sees_f16(const al_paged_fattn_args * args, const al_paged_sees * sees);

/* Bytes of a caller's workspace for these arguments; 0 for refused ones. */
uint64_t al_paged_fattn_sees_workspace_bytes(const al_paged_fattn_args * args, const al_paged_sees * sees);

/*
 * al_paged_append_f32 of rows whose cells are not their positions, as those of
 * a drafted tree are not: row t goes to cell cells[t] (i32 [T], device) of its
 * sequence, rotated by pos[t], which may be any value then.
 */
int al_paged_append_cells_f32(const al_paged_append_args * args, const al_tensor * cells);

/*
 * Pools of all layers, for calls that move cells in every layer at once:
 * k and v are host arrays of n_layers device pointers, each a pool of the
 * shape and strides of k_pool and v_pool (whose own data is not used). The
 * arrays are read before the call returns. n_layers is at most 65535.
 */
typedef struct al_paged_layers {
    al_tensor k_pool;
    al_tensor v_pool;
    void * const * k;
    void * const * v;
    int32_t n_layers;
} al_paged_layers;

/*
 * Arguments of al_paged_keep_f16: of the last counts[s] cells of each sequence
 * those of an accepted path are kept, in the path's order, behind the cells
 * before them: cell b + path[i] goes to cell b + i for i < kept[s], with
 * b = lens[s] - counts[s].
 *   table     i32 [max_pages, n_seq]
 *   lens      i32 [n_seq], counts i32 [n_seq] (data NULL: T each)
 *   path      i32 ne = [T, n_seq], nb0 = 4: rising, path[i] >= i
 *   kept      i32 [n_seq], 0 to counts[s]
 *   lens_out  i32 [n_seq], the new lengths b + kept[s] (data NULL: none). May
 *             not overlap the other operands.
 * A path[i] below i or at counts[s] or more, or a page outside the pool, is
 * recorded as an error and the cell is not moved; a sequence whose length
 * (0 to max_pages P), count (0 to T and the length) or kept is wrong is recorded,
 * and its cells and length stay as they are. Pages that hold moved cells may not be
 * shared with another sequence. T is at most 2^16, n_seq 65535.
 */
typedef struct al_paged_keep_args {
    al_paged_layers layers;
    al_tensor table;
    al_tensor lens;
    al_tensor counts;
    al_tensor path;
    al_tensor kept;
    al_tensor lens_out;
    void *    stream;
} al_paged_keep_args;

int al_paged_keep_f16(const al_paged_keep_args * args);

/*
 * Arguments of al_paged_copy_f16: page src[i] copied into page dst[i], or its
 * first cells[i] cells, for n pairs: the last, partly filled page of a
 * sequence that is forked, or pages brought together.
 *   src, dst  i32 [n], device; a pair with a negative src or dst is left out
 *   cells     i32 [n], device, 0 to P (data NULL: P)
 * No page may be the dst of two pairs, nor dst of one and src of another (a
 * page copied into itself is left alone). A page outside the pool and a count
 * of cells that does not fit are recorded as errors, and the pair is left out.
 * n is at most 65535.
 */
typedef struct al_paged_copy_args {
    al_paged_layers layers;
    al_tensor src;
    al_tensor dst;
    al_tensor cells;
    void *    stream;
} al_paged_copy_args;

int al_paged_copy_f16(const al_paged_copy_args * args);

#ifdef __cplusplus
}
#endif

#endif /* ARCLIGHT_PAGED_H */
