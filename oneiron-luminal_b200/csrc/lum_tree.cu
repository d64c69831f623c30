// Operators of speculative decoding around the attention of drafted trees (include/lum_tree.h): the walk along the nodes that stand, the moves of cache
// rows, and the C entries.
#include <string>

#include "../../include/lum_b200.h"
#include "lum_tree.cuh"

namespace lum {

void set_op_error(const char* msg);                  // lum_runtime.cu

namespace {

__device__ uint32_t g_tree_status;                   // status word of these operators: part of the library, so that no call allocates

// ---------------------------------------------------------------------------------------------------- accepted nodes
// pick(i) = arg-max of the logits of node i (the last maximum); node 0 stands, and the first child of a node that carries its pick stands next.  What it costs is
// reading logits.  Two ways:
//   tree_picks, tree_follow   every row's arg-max at once, spread over all SMs, then the walk through numbers;
//   tree_walk                 row by row along the path: rows of nodes that do not stand are not read, but each one waits for the one before.  A cluster per
//                             sequence shares a row and exchanges its maxima through distributed shared memory, one barrier a step.
// Both use 16-byte loads and as many of them in flight as a thread has.

// A pick as a key: order-preserving bits of the logit, then its index, so that the largest key is the last maximum (-0 as 0).
__device__ __forceinline__ unsigned long long pick_key(float v, int i) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return ((unsigned long long)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32) | (uint32_t)i;
}
__device__ __forceinline__ unsigned long long key_max(unsigned long long a, unsigned long long b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned long long warp_key(unsigned long long k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) k = key_max(k, __shfl_xor_sync(0xffffffffu, k, o));
    return k;
}
// The best of row[i0 .. i1) among `threads` threads (every thread its own; 0: it has none).  NaN counts as -inf.
__device__ __forceinline__ unsigned long long pick_range(const float* row, int i0, int i1, int tid, int threads) {
    float v[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    int at[4] = {-1, -1, -1, -1};
    auto take = [&](int u, float x, int i) {
        x = fmaxf(x, -INFINITY);
        if (x >= v[u]) { v[u] = x; at[u] = i; }      // (a thread's indices grow)
    };
    const int head = min(i1 - i0, (int)(-((uintptr_t)(row + i0) >> 2) & 3)), n4 = (i1 - i0 - head) >> 2, tail = i0 + head + 4 * n4;
    if (tid < head) take(0, __ldcg(row + i0 + tid), i0 + tid);
    const float4* p = (const float4*)(row + i0 + head);
    constexpr int U = 8;
    for (int x0 = tid; x0 < n4; x0 += threads * U) {
        float4 y[U];
#pragma unroll
        for (int u = 0; u < U; u++) if (x0 + u * threads < n4) y[u] = __ldcg(p + x0 + u * threads);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (x0 + u * threads < n4) {
                const int i = i0 + head + 4 * (x0 + u * threads);
                take(0, y[u].x, i); take(1, y[u].y, i + 1); take(2, y[u].z, i + 2); take(3, y[u].w, i + 3);
            }
    }
    if (tid < i1 - tail) take(0, __ldcg(row + tail + tid), tail + tid);
    unsigned long long k = 0ull;
#pragma unroll
    for (int u = 0; u < 4; u++) if (at[u] >= 0) k = key_max(k, pick_key(v[u], at[u]));
    return k;
}

// The tree of a sequence in shared memory; parents that are no earlier node count as none.
struct WalkTree { int token[kTreeMax]; short parent[kTreeMax]; };
__device__ __forceinline__ void walk_load(WalkTree& w, const TreeAcceptArgs& a, const TreeSeq& q, int tid, int threads, bool report) {
    for (int i = tid; i < q.n; i += threads) {
        w.token[i] = a.tokens[q.r0 + i];
        int p = __ldg(a.t.parent + q.r0 + i);
        if (p < -1 || p >= i) { p = -1; if (report) atomicOr(a.status, LUM_ST_BAD_TREE); }
        w.parent[i] = (short)p;
    }
}
// The first child of `node` that carries `pick`, by a warp (kTreeMax: none).
__device__ __forceinline__ int walk_child(const WalkTree& w, int n, int node, int pick, int lane) {
    for (int i0 = node + 1; i0 < n; i0 += 32) {
        const unsigned int m = __ballot_sync(0xffffffffu, i0 + lane < n && w.parent[i0 + lane] == node && w.token[i0 + lane] == pick);
        if (m) return i0 + __ffs(m) - 1;
    }
    return kTreeMax;
}

constexpr int kPickThreads = 256;
__global__ void __launch_bounds__(kPickThreads) tree_picks(const TreeAcceptArgs a, int chunks, unsigned long long* keys) {
    __shared__ unsigned long long s_key[kPickThreads / 32];
    pdl_launch_dependents();
    const int row = blockIdx.x / chunks, c = blockIdx.x - row * chunks, per = (a.vocab + chunks - 1) / chunks, i0 = min(a.vocab, c * per), i1 = min(a.vocab, i0 + per);
    unsigned long long k = warp_key(pick_range(a.logits + (size_t)row * a.ld, i0, i1, threadIdx.x, kPickThreads));
    if ((threadIdx.x & 31) == 0) s_key[threadIdx.x >> 5] = k;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 1; i < kPickThreads / 32; i++) k = key_max(k, s_key[i]);
        keys[blockIdx.x] = k;
    }
}
// One CTA per sequence: the picks of its rows (from their chunks' keys, or given), then the walk by one warp.
__global__ void __launch_bounds__(256) tree_follow(const TreeAcceptArgs a, int chunks, const unsigned long long* keys) {
    __shared__ WalkTree w;
    __shared__ int s_pick[kTreeMax];
    const int s = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    TreeSeq q;
    const bool ok = tree_seq(a.t, nullptr, s, &q, a.status);
    int* path = a.path + (size_t)s * a.path_len;
    if (ok) {
        walk_load(w, a, q, tid, 256, true);
        if (!keys) for (int i = tid; i < q.n; i += 256) s_pick[i] = a.picks[q.r0 + i];
    }
    pdl_grid_wait();                                 // (what comes before does not depend on the kernel before)
    if (!ok) return;
    if (keys)
        for (int i = warp; i < q.n; i += 8) {
            unsigned long long k = 0ull;
            for (int c = lane; c < chunks; c += 32) k = key_max(k, __ldcg(keys + (size_t)(q.r0 + i) * chunks + c));
            k = warp_key(k);
            if (lane == 0) s_pick[i] = (int)(uint32_t)k;
        }
    __syncthreads();
    if (warp == 0) {
        int node = q.n > 0 ? 0 : kTreeMax, count = 0, pick = -1;
        while (node < kTreeMax) {
            if (lane == 0) path[count] = node;
            count++;
            pick = s_pick[node];
            node = walk_child(w, q.n, node, pick, lane);
        }
        for (int i = count + lane; i < a.path_len; i += 32) path[i] = -1;
        if (lane == 0) { a.n_accepted[s] = count; a.next[s] = pick; }
    }
}

constexpr int kWalkThreads = 512, kWalkMax = 8;      // CTAs of a (portable) cluster
__global__ void __launch_bounds__(kWalkThreads) tree_walk(const TreeAcceptArgs a) {
    __shared__ WalkTree w;
    __shared__ unsigned long long s_key[kWalkThreads / 32], s_all[2][kWalkMax];
    const int C = gridDim.x, c = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    TreeSeq q;
    if (!tree_seq(a.t, nullptr, s, &q, a.status)) return;                      // (the whole cluster)
    walk_load(w, a, q, tid, kWalkThreads, c == 0);
    int* path = a.path + (size_t)s * a.path_len;
    const int per = ((a.vocab + C - 1) / C + 3) & ~3, i0 = min(a.vocab, c * per), i1 = min(a.vocab, i0 + per);
    int node = q.n > 0 ? 0 : kTreeMax, count = 0, pick = -1;
    cluster_arrive_release();                        // nobody writes into a CTA that has not begun
    cluster_wait_acquire();
    while (node < kTreeMax) {
        if (c == 0 && tid == 0) path[count] = node;
        unsigned long long k = warp_key(pick_range(a.logits + (size_t)(q.r0 + node) * a.ld, i0, i1, tid, kWalkThreads));
        if (lane == 0) s_key[warp] = k;
        __syncthreads();                             // (also: the tree is there)
        if (warp == 0) {
            k = warp_key(lane < kWalkThreads / 32 ? s_key[lane] : 0ull);
            if (lane < C) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_map(smem_u32(&s_all[count & 1][c]), (uint32_t)lane)), "l"(k) : "memory");
        }
        cluster_arrive_release();
        cluster_wait_acquire();
        k = warp_key(lane < C ? s_all[count & 1][lane] : 0ull);
        pick = (int)(uint32_t)k;
        node = walk_child(w, q.n, node, pick, lane);
        count++;
    }
    if (c == 0) {
        for (int i = count + tid; i < a.path_len; i += kWalkThreads) path[i] = -1;
        if (tid == 0) { a.n_accepted[s] = count; a.next[s] = pick; }
    }
}

// ---------------------------------------------------------------------------------------------------- cache rows
__device__ __forceinline__ bool plane_ok(const KvPlane& p, uint32_t* status) {
    if (!((p.row_bytes | (uint64_t)(uintptr_t)p.rows) & 15)) return true;
    if (threadIdx.x == 0) atomicOr(status, LUM_ST_BAD_PAGE);
    return false;
}
// The rows that stand, one CTA per (plane, sequence).  A thread has a 16-byte column of the rows: it reads eight rows and then writes them.  Rows go up only and
// in order (path[i] >= i, increasing), so nothing that is still to be read has been written, whatever the rows' places in memory.  32 layers of rows of 2 KB: one tree of 8
// nodes, 4 of which stand, 3.2 us (a launch and three dependent loads); 32 trees, up to 8 of up to 64 nodes, 7.1 us (24 MB, 3.4 TB/s, mostly from L2).
__global__ void __launch_bounds__(128) kv_compact(const KvPlane* planes, const TreeMap m, const TreeBatch t, const int* path, int path_len, const int* n_accepted, uint32_t* status) {
    __shared__ long long s_src[kTreeMax], s_dst[kTreeMax];
    __shared__ int s_bad;
    const int tid = threadIdx.x, s = blockIdx.y;
    TreeSeq q;
    if (!tree_seq(t, &m, s, &q, status)) return;
    const int n = n_accepted[s];
    if (tid == 0) s_bad = n < 0 || n > q.n || n > path_len;
    __syncthreads();
    if (!s_bad)
        for (int i = tid; i < n; i += 128) {
            const int at = path[(size_t)s * path_len + i], before = i ? path[(size_t)s * path_len + i - 1] : -1;
            if (at <= before || at >= q.n) s_bad = 1;
            else if (at != i) {
                s_src[i] = tree_row(m, q.slot, q.prefix + at, status);
                s_dst[i] = tree_row(m, q.slot, q.prefix + i, status);
                if (s_src[i] < 0 || s_dst[i] < 0) s_bad = 2;
            } else s_src[i] = s_dst[i] = -1;
        }
    __syncthreads();
    if (s_bad) {
        if (tid == 0 && s_bad == 1) atomicOr(status, LUM_ST_BAD_TREE);
        return;
    }
    const KvPlane p = planes[blockIdx.x];
    if (!plane_ok(p, status)) return;
    const long long cols = (long long)(p.row_bytes >> 4);
    uint4* rows = (uint4*)p.rows;
    for (long long c = tid; c < cols; c += 128) {
        for (int i0 = 0; i0 < n; i0 += 8) {
            uint4 v[8];
#pragma unroll
            for (int u = 0; u < 8; u++) if (i0 + u < n && s_src[i0 + u] >= 0) v[u] = rows[s_src[i0 + u] * cols + c];
#pragma unroll
            for (int u = 0; u < 8; u++) if (i0 + u < n && s_src[i0 + u] >= 0) rows[s_dst[i0 + u] * cols + c] = v[u];
        }
    }
}

// Spans of rows, `per` CTAs for each (plane, span); a span's rows follow each other in memory, so it is one run of 16-byte pieces, eight of a thread on their way.  Bound by HBM:
// two spans of 4001 and 3998 rows of 2 KB in 64 planes (2.1 GB) 334 us, 6.3 TB/s; eight of up to 37 rows 8.8 us, from L2.
constexpr int kCopyThreads = 256, kCopyPieces = 8;
__global__ void __launch_bounds__(kCopyThreads) kv_copy(const KvPlane* planes, long long rows, const int* spans, int n_spans, int max_rows, int per, uint32_t* status) {
    const int part = blockIdx.x % per, item = blockIdx.x / per, span = item % n_spans;
    const long long src = spans[3 * (size_t)span], dst = spans[3 * (size_t)span + 1], n = spans[3 * (size_t)span + 2];
    if (n < 0 || n > max_rows || src < 0 || dst < 0 || src > rows - n || dst > rows - n) {
        if (threadIdx.x == 0) atomicOr(status, LUM_ST_BAD_PAGE);
        return;
    }
    const KvPlane p = planes[item / n_spans];
    if (!plane_ok(p, status)) return;
    const long long cols = (long long)(p.row_bytes >> 4), total = n * cols, step = (long long)kCopyThreads * kCopyPieces;
    const uint4* from = (const uint4*)p.rows + src * cols;
    uint4* to = (uint4*)p.rows + dst * cols;
    for (long long i0 = part * step + threadIdx.x; i0 < total; i0 += per * step) {
        uint4 v[kCopyPieces];
#pragma unroll
        for (int u = 0; u < kCopyPieces; u++) if (i0 + u * kCopyThreads < total) v[u] = __ldcs(from + i0 + u * kCopyThreads);
#pragma unroll
        for (int u = 0; u < kCopyPieces; u++) if (i0 + u * kCopyThreads < total) __stcs(to + i0 + u * kCopyThreads, v[u]);
    }
}

}  // namespace

// Every row at once where that is little to read, else along the paths.  Measured from HBM, us, all rows / along paths of 4 nodes, vocabulary 128256: 1 x 8 nodes (4 MB)
// 11.4 / 18.5, 4 x 16 (33 MB) 18.2 / 19.1, 1 x 64 (33 MB) 21.3 / 18.1, 8 x 16 (66 MB) 27.0 / 20.2, 32 x 64 (1051 MB) 180 / 26.8.
static bool picks_all(const TreeBatch& t, int vocab) { return (long long)t.n_rows * vocab <= (8ll << 20); }
static int pick_chunks(const TreeBatch& t, int vocab, int sm_count) {          // four CTAs per SM, each with at least a load per thread
    const long long want = (4ll * sm_count + t.n_rows - 1) / t.n_rows, most = (vocab + 4 * kPickThreads - 1) / (4 * kPickThreads);
    return (int)(want < most ? want : most);
}
size_t tree_accept_workspace(const TreeBatch& t, int vocab, int sm_count) { return picks_all(t, vocab) ? (size_t)t.n_rows * pick_chunks(t, vocab, sm_count) * 8 : 0; }

cudaError_t launch_tree_accept(const TreeAcceptArgs& a, int sm_count, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    cfg.stream = st;
    cfg.attrs = at;
    if (a.logits && !picks_all(a.t, a.vocab)) {
        // two CTAs per SM in all, at least one per sequence
        int C = 1;
        while (C < kWalkMax && 2 * C * a.t.n_seq <= 2 * sm_count) C *= 2;
        cfg.gridDim = dim3(C, a.t.n_seq);
        cfg.blockDim = dim3(kWalkThreads);
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = (unsigned)C; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, tree_walk, a);
    }
    int chunks = 0;
    unsigned long long* keys = nullptr;
    if (a.logits) {
        chunks = pick_chunks(a.t, a.vocab, sm_count);
        keys = (unsigned long long*)a.ws;
        tree_picks<<<(unsigned)(a.t.n_rows * chunks), kPickThreads, 0, st>>>(a, chunks, keys);
        if (const cudaError_t e = cudaGetLastError()) return e;
    }
    cfg.gridDim = dim3(a.t.n_seq);
    cfg.blockDim = dim3(256);
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = a.logits ? 1 : 0;                 // (without tree_picks before it, it waits for whatever wrote the picks)
    return cudaLaunchKernelEx(&cfg, tree_follow, a, chunks, (const unsigned long long*)keys);
}
cudaError_t launch_kv_compact(const KvPlane* planes, int n_planes, const TreeMap& m, const TreeBatch& t, const int* path, int path_len, const int* n_accepted, uint32_t* status,
                              cudaStream_t st) {
    kv_compact<<<dim3(n_planes, t.n_seq), 128, 0, st>>>(planes, m, t, path, path_len, n_accepted, status);
    return cudaGetLastError();
}
cudaError_t launch_kv_copy(const KvPlane* planes, int n_planes, long long rows, const int* spans, int n_spans, int max_rows, uint32_t* status, int sm_count, cudaStream_t st) {
    const long long items = (long long)n_planes * n_spans;
    // the rows' bytes are known on the device only: enough CTAs for eight on every SM, no more than a row for each
    long long per = (8ll * sm_count + items - 1) / items;
    if (per > max_rows) per = max_rows;
    if (items * per > 0x7fffffff) return cudaErrorInvalidValue;
    kv_copy<<<(unsigned)(items * per), kCopyThreads, 0, st>>>(planes, rows, spans, n_spans, max_rows, (int)per, status);
    return cudaGetLastError();
}

}  // namespace lum

// =================================================================================== C entries

using namespace lum;

// the status word of the current device (null: it cannot be had); lum_op_status reads it too
uint32_t* lum_tree_status_word() {
    static std::atomic<void*> known[64] = {};        // its address per device: asking takes longer than a launch
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return nullptr;
    void* p = dev >= 0 && dev < 64 ? known[dev].load(std::memory_order_acquire) : nullptr;
    if (!p) {
        if (cudaGetSymbolAddress(&p, g_tree_status) != cudaSuccess) return nullptr;
        if (dev >= 0 && dev < 64) known[dev].store(p, std::memory_order_release);
    }
    return (uint32_t*)p;
}

namespace {

int32_t refuse(const char* op, const std::string& why, int32_t code = LUM_E_INVALID) { set_op_error((std::string(op) + ": " + why).c_str()); return code; }
int32_t cuda_failed(const char* op, cudaError_t e) { return refuse(op, cudaGetErrorString(e), LUM_E_CUDA); }

struct Device { int id, sms; };
int32_t device_of(const char* op, Device* d) {
    cudaError_t e = cudaGetDevice(&d->id);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&d->sms, cudaDevAttrMultiProcessorCount, d->id);
    return e == cudaSuccess ? 0 : cuda_failed(op, e);
}
// device memory that kernels of device `dev` may be given
int32_t on_device(const char* op, const char* name, const void* p, int dev) {
    cudaPointerAttributes at;
    const cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) { cudaGetLastError(); return refuse(op, std::string(name) + " is no device pointer"); }
    if (at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeDevice && at.device == dev)) return 0;
    return refuse(op, std::string(name) + (at.type == cudaMemoryTypeDevice ? " belongs to another device than the current one" : " is no device pointer"));
}
#define NEED(expr) do { if (const int32_t r_ = (expr)) return r_; } while (0)

int32_t check_tree(const char* op, const lum_draft_tree* t, TreeBatch* o) {
    if (!t) return refuse(op, "no tree");
    if (t->n_seq < 0 || t->n_seq > 65535 || t->n_rows < 0 || t->max_rows < 1 || t->max_rows > LUM_TREE_MAX_NODES || t->max_prefix < 0 || t->max_prefix > 0x7fffffff - LUM_TREE_MAX_NODES)
        return refuse(op, "sequences 0 .. 65535, rows of the batch, nodes of a tree 1 .. " + std::to_string(LUM_TREE_MAX_NODES) + " and cached rows: got " + std::to_string(t->n_seq) + ", " +
                              std::to_string(t->n_rows) + ", " + std::to_string(t->max_rows) + ", " + std::to_string(t->max_prefix));
    if (t->n_seq > 0 && t->n_rows > 0 && (!t->row_start || !t->prefix || !t->parent)) return refuse(op, "a null array in the tree");
    *o = {t->row_start, t->prefix, t->parent, t->slot, t->n_seq, t->n_rows, t->max_rows, t->max_prefix};
    return 0;
}
int32_t tree_on_device(const char* op, const TreeBatch& t, int dev) {
    NEED(on_device(op, "row_start", t.row_start, dev));
    NEED(on_device(op, "prefix", t.prefix, dev));
    NEED(on_device(op, "parent", t.parent, dev));
    return t.slot ? on_device(op, "slot", t.slot, dev) : 0;
}
int32_t check_map(const char* op, const lum_kv_map* m, TreeMap* o) {
    if (!m) return refuse(op, "no cache map");
    if (m->rows < 1 || m->rows > 0x7fffffffll || m->slots < 1 || m->max_seq < 1) return refuse(op, "a cache of 1 .. 2^31 - 1 rows, slots and rows per slot of at least one");
    int lg = -1;
    if (m->page_rows) {
        if (m->page_rows < 16 || (m->page_rows & (m->page_rows - 1))) return refuse(op, "page_rows must be a power of two of at least 16");
        if (!m->page_table || m->pages_per_seq < 1) return refuse(op, "pages without a page table");
        lg = __builtin_ctz((unsigned)m->page_rows);
    } else if ((int64_t)m->slots * m->max_seq > m->rows) return refuse(op, "the cache holds fewer rows than its slots");
    *o = {m->page_rows ? m->page_table : nullptr, (long long)m->rows, m->slots, m->max_seq, lg, m->pages_per_seq};
    return 0;
}

// everything that needs no device
int32_t check_attn(const lum_tree_attn* d, const lum_draft_tree* tree, const lum_kv_map* map, TreeAttnArgs* a) {
    const char* op = "attn_tree";
    if (!d) return refuse(op, "no description");
    NEED(check_tree(op, tree, &a->t));
    NEED(check_map(op, map, &a->m));
    if (d->head_dim != 64 && d->head_dim != 128) return refuse(op, "heads of 64 or 128, got " + std::to_string(d->head_dim), LUM_E_UNSUPPORTED);
    if (d->n_kv_heads < 1 || d->n_q_heads < 1 || d->n_q_heads % d->n_kv_heads || d->n_q_heads > 1024) return refuse(op, "query heads must be a multiple of the K/V heads (at most 1024)");
    const bool qb = d->q_dtype == LUM_BF16, kb = d->kv_dtype == LUM_BF16;
    if ((!qb && d->q_dtype != LUM_F32) || (!kb && d->kv_dtype != LUM_F32) || (qb && !kb)) return refuse(op, "queries in bf16 or f32 over a bf16 cache, or in f32 over an f32 cache", LUM_E_UNSUPPORTED);
    if (d->window < 0 || !(d->scale >= 0.0f) || !(d->scale < __builtin_inff())) return refuse(op, "window and scale must not be negative");
    const long long qw = (long long)d->n_q_heads * d->head_dim, kw = (long long)d->n_kv_heads * d->head_dim;
    a->q_stride = d->q_stride ? d->q_stride : qw; a->out_stride = d->out_stride ? d->out_stride : qw; a->kv_stride = d->kv_stride ? d->kv_stride : kw;
    if (a->q_stride < qw || a->out_stride < qw || a->kv_stride < kw) return refuse(op, "a row stride shorter than a row");
    const int qe = qb ? 2 : 4, ke = kb ? 2 : 4;
    if (a->q_stride * qe % 16 || a->out_stride * qe % 16 || a->kv_stride * ke % 16) return refuse(op, "row strides must be multiples of 16 bytes");
    // a window that reaches over everything is none
    a->n_q = d->n_q_heads; a->n_kv = d->n_kv_heads; a->hd = d->head_dim; a->q_bf16 = qb; a->kv_bf16 = kb; a->window = (long long)d->window < (long long)a->t.max_prefix + a->t.max_rows ? d->window : 0;
    a->scale = d->scale != 0.0f ? d->scale : 1.0f / __builtin_sqrtf((float)d->head_dim);
    if (a->t.n_seq && a->t.n_rows && !tree_attn_supported(*a)) return refuse(op, "more than 128 query heads per K/V head, or a batch of 2^31 tiles of 64 keys (sequences x heads x cached rows) or 2^34 rows of heads", LUM_E_UNSUPPORTED);
    return 0;
}

int32_t check_planes(const char* op, const lum_kv_plane* planes, int32_t n) {
    if (n < 1 || n > 65535 || !planes) return refuse(op, "1 .. 65535 planes");
    return 0;
}

}  // namespace

extern "C" {

size_t lum_op_attn_tree_workspace(const lum_tree_attn* desc, const lum_draft_tree* tree, const lum_kv_map* map) {
    TreeAttnArgs a{};
    Device d;
    if (check_attn(desc, tree, map, &a) || device_of("attn_tree", &d)) return (size_t)-1;
    return a.t.n_seq && a.t.n_rows ? tree_attn_workspace(a, d.sms) : 0;
}

int32_t lum_op_attn_tree(const lum_tree_attn* desc, const lum_draft_tree* tree, const lum_kv_map* map, const void* q, const void* k, const void* v, const float* sinks, void* out,
                         void* workspace, size_t workspace_bytes, void* stream) {
    const char* op = "attn_tree";
    TreeAttnArgs a{};
    Device d;
    NEED(check_attn(desc, tree, map, &a));
    if (!a.t.n_seq || !a.t.n_rows) return 0;
    if (!q || !k || !v || !out || out == q) return refuse(op, "null q, k, v or out, or out in the place of q");
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)workspace) & 15) return refuse(op, "q, k, v, out and the workspace must be 16-byte aligned");
    NEED(device_of(op, &d));
    const size_t need = tree_attn_workspace(a, d.sms);
    if (need && (!workspace || workspace_bytes < need)) return refuse(op, "the workspace needs " + std::to_string(need) + " bytes, got " + std::to_string(workspace ? workspace_bytes : 0));
    NEED(tree_on_device(op, a.t, d.id));
    NEED(on_device(op, "q", q, d.id));
    NEED(on_device(op, "k", k, d.id));
    NEED(on_device(op, "v", v, d.id));
    NEED(on_device(op, "out", out, d.id));
    if (a.m.table) NEED(on_device(op, "page_table", a.m.table, d.id));
    if (sinks) NEED(on_device(op, "sinks", sinks, d.id));
    if (need) NEED(on_device(op, "workspace", workspace, d.id));
    a.q = q; a.k = k; a.v = v; a.sinks = sinks; a.out = out; a.ws = workspace; a.ws_bytes = need;
    a.status = lum_tree_status_word();
    if (!a.status) return refuse(op, "no status word", LUM_E_CUDA);
    const cudaError_t e = launch_tree_attn(a, d.sms, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : cuda_failed(op, e);
}

size_t lum_op_tree_accept_workspace(const lum_draft_tree* tree, int32_t vocab) {
    TreeBatch t{};
    Device d;
    if (check_tree("tree_accept", tree, &t)) return (size_t)-1;
    if (vocab < 1 || vocab > (1 << 30)) { refuse("tree_accept", "a vocabulary of 1 .. 2^30, got " + std::to_string(vocab)); return (size_t)-1; }
    if (device_of("tree_accept", &d)) return (size_t)-1;
    return t.n_seq && t.n_rows ? tree_accept_workspace(t, vocab, d.sms) : 0;
}

int32_t lum_op_tree_accept(const lum_draft_tree* tree, const int32_t* tokens, const float* logits, int32_t vocab, int64_t logits_stride, const int32_t* picks, int32_t* path,
                           int32_t path_len, int32_t* n_accepted, int32_t* next, void* workspace, size_t workspace_bytes, void* stream) {
    const char* op = "tree_accept";
    TreeAcceptArgs a{};
    Device d;
    NEED(check_tree(op, tree, &a.t));
    if (!a.t.n_seq) return 0;
    if (!path || !n_accepted || !next) return refuse(op, "null output");
    if (path_len < a.t.max_rows) return refuse(op, "paths of " + std::to_string(path_len) + " nodes cannot hold a tree of " + std::to_string(a.t.max_rows));
    if (a.t.n_rows && (!tokens || (logits != nullptr) == (picks != nullptr))) return refuse(op, "tokens, and either logits or picks");
    if (logits && (vocab < 1 || vocab > (1 << 30) || (logits_stride && logits_stride < vocab) || ((uintptr_t)logits & 3)))
        return refuse(op, "a vocabulary of 1 .. 2^30, rows of logits that do not overlap, 4-byte aligned");
    NEED(device_of(op, &d));
    if (!a.t.n_rows) {                               // every sequence is empty
        NEED(on_device(op, "path", path, d.id));
        NEED(on_device(op, "n_accepted", n_accepted, d.id));
        NEED(on_device(op, "next", next, d.id));
        cudaError_t e = cudaMemsetAsync(path, 0xff, (size_t)a.t.n_seq * path_len * 4, (cudaStream_t)stream);
        if (e == cudaSuccess) e = cudaMemsetAsync(n_accepted, 0, (size_t)a.t.n_seq * 4, (cudaStream_t)stream);
        if (e == cudaSuccess) e = cudaMemsetAsync(next, 0xff, (size_t)a.t.n_seq * 4, (cudaStream_t)stream);
        return e == cudaSuccess ? 0 : cuda_failed(op, e);
    }
    const size_t need = logits ? tree_accept_workspace(a.t, vocab, d.sms) : 0;
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
        return refuse(op, "the workspace needs " + std::to_string(need) + " bytes, 16-byte aligned, got " + std::to_string(workspace ? workspace_bytes : 0));
    NEED(tree_on_device(op, a.t, d.id));
    NEED(on_device(op, "tokens", tokens, d.id));
    NEED(on_device(op, "logits or picks", logits ? (const void*)logits : picks, d.id));
    NEED(on_device(op, "path", path, d.id));
    NEED(on_device(op, "n_accepted", n_accepted, d.id));
    NEED(on_device(op, "next", next, d.id));
    if (need) NEED(on_device(op, "workspace", workspace, d.id));
    a.tokens = tokens; a.logits = logits; a.vocab = vocab; a.ld = logits_stride ? logits_stride : vocab; a.picks = picks; a.path = path; a.path_len = path_len;
    a.n_accepted = n_accepted; a.next = next; a.ws = workspace; a.ws_bytes = need;
    a.status = lum_tree_status_word();
    if (!a.status) return refuse(op, "no status word", LUM_E_CUDA);
    const cudaError_t e = launch_tree_accept(a, d.sms, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : cuda_failed(op, e);
}

int32_t lum_op_kv_compact(const lum_kv_plane* planes, int32_t n_planes, const lum_kv_map* map, const lum_draft_tree* tree, const int32_t* path, int32_t path_len,
                          const int32_t* n_accepted, void* stream) {
    const char* op = "kv_compact";
    TreeBatch t{};
    TreeMap m{};
    Device d;
    NEED(check_planes(op, planes, n_planes));
    NEED(check_tree(op, tree, &t));
    NEED(check_map(op, map, &m));
    if (!t.n_seq || !t.n_rows) return 0;
    if (!path || !n_accepted || path_len < 1) return refuse(op, "null or empty path");
    NEED(device_of(op, &d));
    NEED(tree_on_device(op, t, d.id));
    NEED(on_device(op, "planes", planes, d.id));
    NEED(on_device(op, "path", path, d.id));
    NEED(on_device(op, "n_accepted", n_accepted, d.id));
    if (m.table) NEED(on_device(op, "page_table", m.table, d.id));
    uint32_t* status = lum_tree_status_word();
    if (!status) return refuse(op, "no status word", LUM_E_CUDA);
    const cudaError_t e = launch_kv_compact((const KvPlane*)planes, n_planes, m, t, path, path_len, n_accepted, status, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : cuda_failed(op, e);
}

int32_t lum_op_kv_copy(const lum_kv_plane* planes, int32_t n_planes, int64_t rows, const int32_t* spans, int32_t n_spans, int32_t max_rows, void* stream) {
    const char* op = "kv_copy";
    Device d;
    NEED(check_planes(op, planes, n_planes));
    if (rows < 1 || rows > 0x7fffffffll || n_spans < 0 || max_rows < 0 || (long long)n_planes * n_spans > 0x7fffffffll) return refuse(op, "rows 1 .. 2^31 - 1, spans and their rows not negative, at most 2^31 - 1 planes x spans");
    if (!n_spans || !max_rows) return 0;
    if (!spans) return refuse(op, "null spans");
    NEED(device_of(op, &d));
    NEED(on_device(op, "planes", planes, d.id));
    NEED(on_device(op, "spans", spans, d.id));
    uint32_t* status = lum_tree_status_word();
    if (!status) return refuse(op, "no status word", LUM_E_CUDA);
    const cudaError_t e = launch_kv_copy((const KvPlane*)planes, n_planes, rows, spans, n_spans, max_rows, status, d.sms, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : cuda_failed(op, e);
}

}  // extern "C"
