/*
 * lum_tree.h — operators of speculative decoding as single calls (included by lum_b200.h, whose conventions hold: a status per call,
 * lum_last_error(NULL) for the message, plain device pointers, `stream` a cudaStream_t).  No counterpart in the reference, whose loop decodes
 * one token per step (examples/llama/src/main.rs:82-118).
 *
 * A step verifies, for every sequence of a batch, a TREE of drafted tokens in one pass of the model: node 0 is the token that decoding stands
 * at, other nodes are guesses of what follows their parent.  The nodes' keys and values are written behind the sequence's cached rows — node i
 * at cache row prefix + i, with the angles of its own place, prefix + depth(i) — and then
 *   lum_op_attn_tree     attends from every node to the cached rows and to its own ancestors,
 *   lum_op_tree_accept   walks from node 0 along the nodes that the model itself would have produced,
 *   lum_op_kv_compact    moves the rows of those nodes up behind the cached rows, in every layer,
 *   lum_op_kv_copy       copies spans of rows in every layer (forks of a sequence, pages shared until written).
 *
 * Nothing is allocated, so the calls can be captured into graphs; all arrays named `device` are read by the kernels, not by the call.  What a
 * kernel finds wrong in them — a parent that is not an earlier node, a row or page outside the cache, more nodes or cached rows than the call
 * named — is left out and reported by the next lum_op_status as LUM_E_DEVICE: the sequence or span it belongs to keeps its outputs as they were
 * (every sequence of a batch whose row_start decreases may), a parent counts as none, the rows of an unknown page as zeros.  The pointers must belong to the current device (LUM_E_INVALID otherwise).  Calls may run at the
 * same time on several streams, each with a workspace of its own.
 */
#ifndef LUM_TREE_H
#define LUM_TREE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define LUM_TREE_MAX_NODES 256      /* nodes of one tree */

/* The trees of a batch.  Sequence s has the batch's rows row_start[s] .. row_start[s + 1] - 1 (row_start[0] need not be 0; rows outside every
 * sequence are left alone; a sequence may have none). */
typedef struct lum_draft_tree {
    const int32_t* row_start;  /* device [n_seq + 1] */
    const int32_t* prefix;     /* device [n_seq]: cached rows before the tree */
    const int32_t* parent;     /* device [n_rows]: an earlier node of the same tree (counted from its node 0), or -1 */
    const int32_t* slot;       /* device [n_seq]: the sequence's cache slot / row of the page table; NULL: s */
    int32_t n_seq;
    int32_t n_rows;            /* rows of the batch */
    int32_t max_rows;          /* no tree has more nodes (1 .. LUM_TREE_MAX_NODES) */
    int32_t max_prefix;        /* no sequence has more cached rows */
} lum_draft_tree;

/* Where the cached rows of a slot are.  page_rows 0: rows [slot * max_seq, (slot + 1) * max_seq) of the cache.  Otherwise a pool of pages of
 * page_rows rows (a power of two >= 16); page_table[slot * pages_per_seq + row / page_rows] names the page.  Entries of pages that hold none
 * of a sequence's rows are not read. */
typedef struct lum_kv_map {
    const int32_t* page_table; /* device, or NULL */
    int64_t rows;              /* rows of the cache (of the pool) */
    int32_t slots;
    int32_t max_seq;           /* rows a slot can hold */
    int32_t page_rows;
    int32_t pages_per_seq;
} lum_kv_map;

/* Attention of the nodes: out = sum_j w_j v_j, w = softmax over the visible keys of scale * q . k_j.  A node sees the cached rows, its ancestors and
 * itself; with `window` > 0 only what is fewer than `window` places before its own.  q and out: [n_rows][n_q_heads][head_dim], rows q_stride /
 * out_stride elements apart; k and v: rows kv_stride elements apart, each [n_kv_heads][head_dim]; query head h reads K/V head
 * h / (n_q_heads / n_kv_heads).  sinks (device [n_q_heads], or NULL): a logit per head that joins the softmax's denominator.  A row all of whose
 * visible scores are -inf is 0 / 0 and comes out as NaN (as 0 with a sink above -inf); so is one that sees a score that is NaN or +inf.  A sink of -inf is none, one of +inf leaves zeros.
 * out must not overlap q. */
typedef struct lum_tree_attn {
    uint32_t q_dtype;          /* LUM_BF16 or LUM_F32, of q and out */
    uint32_t kv_dtype;         /* LUM_BF16, or LUM_F32 with queries in f32 */
    int32_t n_q_heads, n_kv_heads;
    int32_t head_dim;          /* 64 or 128 */
    int32_t window;            /* 0: none */
    float scale;               /* 0: 1 / sqrt(head_dim) */
    int32_t reserved;
    int64_t q_stride, kv_stride, out_stride;     /* elements; 0: rows follow each other */
} lum_tree_attn;

/* Device scratch of such a call, in bytes (0: none needed); (size_t)-1 when the call would be refused. */
size_t lum_op_attn_tree_workspace(const lum_tree_attn* desc, const lum_draft_tree* tree, const lum_kv_map* map);
int32_t lum_op_attn_tree(const lum_tree_attn* desc, const lum_draft_tree* tree, const lum_kv_map* map, const void* q_dev, const void* k_dev, const void* v_dev,
                         const float* sinks_dev, void* out_dev, void* workspace_dev, size_t workspace_bytes, void* stream);

/* The nodes that stand.  Node 0 stands; the token picked at a node is the arg-max of its row of logits (last maximum wins, NaN counting as -inf: the
 * greedy sample) or picks[row] (what a sampler drew there); the first child of the node that carries the picked token stands next.
 * logits_dev [n_rows][vocab] f32, rows logits_stride elements apart (0: vocab), or NULL with picks_dev [n_rows].  tokens_dev [n_rows]: the nodes'
 * tokens (node 0's is not read).  path_dev [n_seq][path_len]: the nodes that stand, in order, -1 behind them (path_len >= max_rows);
 * n_accepted_dev [n_seq]: how many; next_dev [n_seq]: the token picked at the last of them.  A sequence without rows: none, 0 and -1. */
size_t lum_op_tree_accept_workspace(const lum_draft_tree* tree, int32_t vocab);
int32_t lum_op_tree_accept(const lum_draft_tree* tree, const int32_t* tokens_dev, const float* logits_dev, int32_t vocab, int64_t logits_stride,
                           const int32_t* picks_dev, int32_t* path_dev, int32_t path_len, int32_t* n_accepted_dev, int32_t* next_dev, void* workspace_dev,
                           size_t workspace_bytes, void* stream);

/* One plane of cache rows (K or V of one layer): rows of row_bytes bytes (a multiple of 16), one behind the other, 16-byte aligned.  A plane that
 * is not is left out and reported by lum_op_status. */
typedef struct lum_kv_plane {
    void* rows;
    uint64_t row_bytes;
} lum_kv_plane;

/* Every plane's row prefix + path[s][i] becomes row prefix + i, for i < n_accepted[s] (as lum_op_tree_accept leaves them: path is increasing).  The
 * rows moved must not share pages with another sequence, nor two sequences a slot.  planes_dev: device [n_planes]. */
int32_t lum_op_kv_compact(const lum_kv_plane* planes_dev, int32_t n_planes, const lum_kv_map* map, const lum_draft_tree* tree, const int32_t* path_dev,
                          int32_t path_len, const int32_t* n_accepted_dev, void* stream);
/* spans_dev: device [n_spans][3] of {first source row, first destination row, rows}; every plane (of `rows` rows) has rows src .. src + n - 1 copied
 * to dst .. dst + n - 1.  Destinations overlap neither each other nor any source.  max_rows: no span has more rows. */
int32_t lum_op_kv_copy(const lum_kv_plane* planes_dev, int32_t n_planes, int64_t rows, const int32_t* spans_dev, int32_t n_spans, int32_t max_rows, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* LUM_TREE_H */
