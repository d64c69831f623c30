// Argument blocks and launchers of the operators of speculative decoding (include/lum_tree.h): attention of drafted trees (lum_tree_attn.cu), the
// walk that accepts drafted tokens and the moves of cache rows (lum_tree.cu).
#pragma once
#include "lum_kernels.cuh"

namespace lum {

constexpr int kTreeMax = 256;                        // nodes of one tree
constexpr int kTreeWords = kTreeMax / 32;

struct TreeBatch {                                   // lum_draft_tree
    const int *row_start, *prefix, *parent, *slot;
    int n_seq, n_rows, max_rows, max_prefix;
};
struct TreeMap {                                     // lum_kv_map; lg < 0: contiguous slots
    const int* table;
    long long rows;
    int slots, max_seq, lg, pages_per_seq;
};
struct TreeAttnArgs {
    TreeBatch t;
    TreeMap m;
    const void *q, *k, *v;
    const float* sinks;
    void* out;
    long long q_stride, kv_stride, out_stride;       // elements
    int n_q, n_kv, hd, q_bf16, kv_bf16, window;
    float scale;
    void* ws; size_t ws_bytes;
    uint32_t* status;
};
struct TreeAcceptArgs {
    TreeBatch t;
    const int* tokens;
    const float* logits; int vocab; long long ld;
    const int* picks;
    int* path; int path_len;
    int *n_accepted, *next;
    void* ws; size_t ws_bytes;
    uint32_t* status;
};
struct KvPlane { void* rows; uint64_t row_bytes; };

// Sequence s of a batch, as far as it can be trusted: its numbers, and false (and a status bit) where they do not fit what the call named.
struct TreeSeq { int r0, n, prefix, slot; };
__device__ __forceinline__ TreeSeq tree_seq_load(const TreeBatch& t, int s) {
    TreeSeq o;
    o.r0 = __ldg(t.row_start + s);
    o.n = __ldg(t.row_start + s + 1);
    o.prefix = __ldg(t.prefix + s);
    o.slot = t.slot ? __ldg(t.slot + s) : s;
    return o;
}
__device__ __forceinline__ bool tree_seq_ok(const TreeBatch& t, const TreeMap* m, TreeSeq* o, uint32_t* status) {      // once, behind tree_seq_load: n becomes a count
    const long long n = (long long)o->n - o->r0;
    const bool ok = o->r0 >= 0 && n >= 0 && n <= t.max_rows && o->n <= t.n_rows && o->prefix >= 0 && o->prefix <= t.max_prefix &&
                    (!m || (o->slot >= 0 && o->slot < m->slots && o->prefix <= m->max_seq - n));
    o->n = (int)n;
    if (!ok && status) atomicOr(status, LUM_ST_BAD_POS);
    return ok;
}
__device__ __forceinline__ bool tree_seq(const TreeBatch& t, const TreeMap* m, int s, TreeSeq* o, uint32_t* status) {
    *o = tree_seq_load(t, s);
    return tree_seq_ok(t, m, o, status);
}
// Physical row of a slot's row, -1 (and a status bit) where the page table or the cache does not hold it.
__device__ __forceinline__ long long tree_row(const TreeMap& m, int slot, int row, uint32_t* status) {
    long long at;
    if (m.lg < 0) at = (long long)slot * m.max_seq + row;
    else {
        const int lp = row >> m.lg, e = lp < m.pages_per_seq ? __ldg(m.table + (size_t)slot * m.pages_per_seq + lp) : -1;
        at = e < 0 ? -1 : ((long long)e << m.lg) + (row & ((1 << m.lg) - 1));
    }
    if (at >= 0 && at < m.rows) return at;
    if (status) atomicOr(status, LUM_ST_BAD_PAGE);
    return -1;
}

bool tree_attn_supported(const TreeAttnArgs& a);     // heads per K/V head, and sizes that can be counted
size_t tree_attn_workspace(const TreeAttnArgs& a, int sm_count);
cudaError_t launch_tree_attn(const TreeAttnArgs& a, int sm_count, cudaStream_t st);
size_t tree_accept_workspace(const TreeBatch& t, int vocab, int sm_count);
cudaError_t launch_tree_accept(const TreeAcceptArgs& a, int sm_count, cudaStream_t st);
cudaError_t launch_kv_compact(const KvPlane* planes, int n_planes, const TreeMap& m, const TreeBatch& t, const int* path, int path_len, const int* n_accepted, uint32_t* status,
                              cudaStream_t st);
cudaError_t launch_kv_copy(const KvPlane* planes, int n_planes, long long rows, const int* spans, int n_spans, int max_rows, uint32_t* status, int sm_count, cudaStream_t st);

}  // namespace lum
