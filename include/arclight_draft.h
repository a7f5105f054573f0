/*
 * arclight_draft.h - C ABI of trees of drafted tokens: what a step of many
 * sequences needs before attention, and their verification after it.
 *
 * The reference's speculative decoder (al-spec) drafts one chain of tokens for
 * one sequence and verifies it on the host. Here each sequence of a batch brings
 * a tree: node 0 is the last token that was accepted, whose keys are not in the
 * cache yet, the others are drafts. parents[t] is the node that node t follows, a
 * smaller one; of node 0 it is negative. A chain is parents[t] = t - 1.
 * al_draft_tree_i32 makes of the parents what the paged cache's append and
 * attention take (arclight_paged.h), al_draft_verify_f32 takes the target's
 * probabilities for the nodes and gives the accepted path, which
 * al_paged_keep_f16 takes. No operand passes through the host, so that a step
 * can be captured into a HIP graph and replayed.
 *
 * All data pointers are device pointers of the current device; no pointer is
 * kept after a call returns. Error convention as arclight_fattn.h. Calls
 * enqueue on `stream` without synchronizing. What a kernel finds wrong when it
 * runs it does not follow: it records it, and al_device_errors() returns
 * AL_ERR_INVALID after the stream completes.
 */
#ifndef ARCLIGHT_DRAFT_H
#define ARCLIGHT_DRAFT_H

#include <stdint.h>

#include "arclight_fattn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Arguments of al_draft_tree_i32, for n_seq trees of up to T nodes:
 *   parents  i32 ne = [T, n_seq], nb0 = 4
 *   lens     i32 [n_seq]: cells of each sequence, the nodes' among them
 *   counts   i32 [n_seq]: nodes of each sequence, 0 to T (data NULL: T each)
 *   pos      i32 ne = [T, n_seq], nb0 = 4: each node's position, b + its depth
 *            (the root's is 0), with b = lens[s] - counts[s]
 *   cells    the same: the node's cell, b + t
 *   seq      the same: the node's sequence, s
 *   bits     i32 ne = [words, T, n_seq], nb0 = 4, words at least (T + 31) / 32:
 *            bit u % 32 of word u / 32 is set where node u is node t or above
 *            it; further words are 0
 * Each of the outputs may be left out (data NULL); none may overlap another
 * operand. For t >= counts[s] pos and cells are 0, seq is -1 and no bit is set.
 * A node with a negative parent is a root. One whose parent is t or more is
 * recorded as an error and taken for a root; a count that is not 0 to T, or
 * above the length, is recorded and the sequence has no nodes.
 * T is at most 1024 (AL_ERR_UNSUPPORTED otherwise), n_seq 65535.
 */
typedef struct al_draft_tree_args {
    al_tensor parents;
    al_tensor lens;
    al_tensor counts;
    al_tensor pos;
    al_tensor cells;
    al_tensor seq;
    al_tensor bits;
    void *    stream;
} al_draft_tree_args;

int al_draft_tree_i32(const al_draft_tree_args * args);

/*
 * Arguments of al_draft_verify_f32:
 *   target   f32 ne = [V, T, n_seq], nb0 = 4: row t holds the target's
 *            probabilities of the token that follows node t
 *   draft    the same of the draft: row t holds the probabilities that the
 *            children of node t were drawn from, each by itself (data NULL:
 *            they were chosen, not drawn)
 *   tokens   i32 ne = [T, n_seq], nb0 = 4: the nodes' tokens (of node 0: not
 *            looked at)
 *   parents  i32 ne = [T, n_seq], nb0 = 4 (data NULL: chains)
 *   counts   i32 [n_seq]: nodes of each sequence, 0 to T (data NULL: T each)
 *   accept   f32 ne = [T, n_seq], nb0 = 4: a random number in [0, 1) for each node
 *   sample   f32 [n_seq]: one for the token that follows
 *   path     i32 ne = [T, n_seq], nb0 = 4: the accepted nodes from the root
 *            on, -1 behind them
 *   kept     i32 [n_seq]: how many they are, the root among them
 *   next     i32 [n_seq]: the token that follows the last of them
 * path, kept and next may not overlap one another or another operand.
 * From node v = 0 on, with p = p_0 = target row v: the children of v are tried in
 * their order. Child u of token x is accepted if accept[u] q(x) < p_i(x) and
 * p_i(x) > 0, and becomes v; else the next one is tried with p_(i+1). Without a
 * draft q = 1 and p_i is p without the tokens that were rejected, over 1 - the
 * sum of their p. With one q is draft row v and p_(i+1) = max(p_i - q, 0) over its
 * sum. Where no child is accepted, next is drawn from what is left of p:
 * without a draft p without the rejected tokens, with one the last max(p_i - q,
 * 0), p where there are no children. It is the first token y with w(y) > 0 at
 * which the sum of the w up to it is above sample times the sum of all. Where
 * nothing is left p itself is taken. All of this in 64 bits.
 * With a draft, a child that is rejected before another one of its node costs a
 * pass over both rows by one workgroup (128000 tokens: 34 us for a node's first, 60
 * for a later one), and the workspace holds 8 V bytes for a sequence (T > 2, with
 * parents).
 * Values that are not above 0, NaN among them, count as 0. Probabilities need
 * not sum to 1 for next. A row whose sum is 0 or not finite gives next = -1 and
 * is recorded as an error. A node t > 0 with a negative parent is nobody's
 * child, and neither is one whose parent is t or more or whose token is not 0 to
 * V - 1, which is recorded. A count that is not 0 to T is recorded, and the
 * sequence has no nodes: kept = 0, next = -1.
 * V is at most 2^24, T 1024 (AL_ERR_UNSUPPORTED otherwise), n_seq 65535. Rows may
 * begin at any multiple of 4 bytes.
 * workspace: device scratch (al_draft_verify_workspace_bytes), NULL: the
 * library's own for (current device, stream), as al_fattn_f16: then one eager
 * call of the same shapes has to come before a capture. Calls and replays that
 * share a workspace must be ordered on one stream. It needs no initial value;
 * its first 256 KiB are not touched, so that it may also be al_fattn_f16's.
 */
typedef struct al_draft_verify_args {
    al_tensor target;
    al_tensor draft;
    al_tensor tokens;
    al_tensor parents;
    al_tensor counts;
    al_tensor accept;
    al_tensor sample;
    al_tensor path;
    al_tensor kept;
    al_tensor next;
    void *    stream;
    void *    workspace;
    uint64_t  workspace_bytes;
} al_draft_verify_args;

int al_draft_verify_f32(const al_draft_verify_args * args);

/* Bytes of a caller's workspace for these arguments; 0 for refused ones. */
uint64_t al_draft_verify_workspace_bytes(const al_draft_verify_args * args);

#ifdef __cplusplus
}
#endif

#endif /* ARCLIGHT_DRAFT_H */
