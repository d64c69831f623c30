// Attention of drafted trees over a K/V cache (lum_op_attn_tree): node i of sequence s, with p = prefix[s], sees the cached rows j < p, its ancestors a
// (row p + a) and itself:
//     o_i = sum_j w_ij v_j,   w_ij = exp(x_ij) / (sum_j exp(x_ij) + exp(sink)),   x_ij = scale q_i . k_j
// One pass over the keys with the running maximum and sum of the softmax.  All nodes of a tree and the G query heads of a K/V head share every key: row
// f = node * G + head of a K/V head's query rows.  The keys of a sequence are cut into chunks, one CTA each; where there are several, every chunk leaves its
// (maximum, sum, outputs) in the workspace and tree_combine joins them.
#include "lum_tree.cuh"

namespace lum {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTileKeys = 64;                        // chunks are whole tiles of so many cache rows, from the first visible one's tile on

struct TreeWork {                                    // the keys of a sequence that any node sees: rows low .. n_keys - 1, tiles t_lo .. t_lo + n_tiles - 1
    int low, n_keys, t_lo, n_tiles;
};
__host__ __device__ inline TreeWork tree_work(int prefix, int n, int window) {
    TreeWork w;
    w.low = window > 0 && prefix + 1 > window ? prefix + 1 - window : 0;      // node 0 may stand at place `prefix`
    w.n_keys = prefix + n;
    w.t_lo = w.low / kTileKeys;
    w.n_tiles = (w.n_keys + kTileKeys - 1) / kTileKeys - w.t_lo;
    return w;
}

// The tree in shared memory: depths and, as bits, ancestors (the node itself included).  All threads of the CTA; synchronise before and after.
struct TreeNodes { unsigned int anc[kTreeMax][kTreeWords]; short depth[kTreeMax]; short parent[kTreeMax]; };
__device__ __forceinline__ void tree_load(TreeNodes& s, const TreeBatch& t, const TreeSeq& q, int tid, int threads, uint32_t* status) {
    for (int i = tid; i < q.n; i += threads) {
        int p = __ldg(t.parent + q.r0 + i);
        if (p < -1 || p >= i) { p = -1; if (status) atomicOr(status, LUM_ST_BAD_TREE); }
        s.parent[i] = (short)p;
    }
    __syncthreads();
    for (int i = tid; i < q.n; i += threads) {
        unsigned int w[kTreeWords];
#pragma unroll
        for (int k = 0; k < kTreeWords; k++) w[k] = 0u;
        int depth = -1;
        for (int a = i; a >= 0; a = s.parent[a], depth++)
#pragma unroll
            for (int k = 0; k < kTreeWords; k++) if (k == a >> 5) w[k] |= 1u << (a & 31);
#pragma unroll
        for (int k = 0; k < kTreeWords; k++) s.anc[i][k] = w[k];
        s.depth[i] = (short)depth;
    }
}
// whether node i sees cache row j of its sequence (j < n_keys)
__device__ __forceinline__ bool tree_sees(const TreeNodes& s, const TreeSeq& q, int window, int i, int j) {
    const int a = j - q.prefix;
    if (a < 0) return window <= 0 || q.prefix + s.depth[i] - j < window;
    return (s.anc[i][a >> 5] >> (a & 31) & 1u) && (window <= 0 || s.depth[i] - s.depth[a] < window);
}

struct Part {                                        // where chunk c leaves its share of (row, head); out is used where there is one chunk
    float *o, *ml;                                   // [chunk][row][head][hd], [chunk][row][head][2]
    int chunks, tiles;                               // chunks of the longest sequence, tiles of a chunk
};
__device__ __forceinline__ size_t part_at(const TreeAttnArgs& a, int c, int row, int h) { return ((size_t)c * a.t.n_rows + row) * a.n_q + h; }

template <typename T> __device__ __forceinline__ float4 load4(const T* p);
template <> __device__ __forceinline__ float4 load4<float>(const float* p) { return *(const float4*)p; }
template <> __device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* p) {
    const uint2 v = *(const uint2*)p;
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ T out_of(float x);
template <> __device__ __forceinline__ float out_of<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 out_of<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }      // the one rounding of the result

// ---- products on CUDA cores, in 32 bits: an f32 cache
// CTA = chunk x (K/V head, 32 query rows) x sequence; 8 warps of 4 query rows.  32 keys at a time lie in shared memory as f32: a lane multiplies its key with
// the warp's four rows, and then four (two) dimensions of the values with their weights.
constexpr int kRowsTile = 32, kRowsKeys = 32;
template <int HD>
constexpr int rows_smem() { return (kRowsTile * HD + kRowsKeys * (HD + 4) + kRowsKeys * HD + kRowsTile * kRowsKeys) * 4 + (int)sizeof(TreeNodes); }

template <int HD, typename TQ, typename TK>
__global__ void __launch_bounds__(256) attn_tree_rows(const TreeAttnArgs a, const Part part) {
    extern __shared__ __align__(16) unsigned char smem[];
    float* s_q = (float*)smem;                       // [32][HD]
    float* s_k = s_q + kRowsTile * HD;               // [32][HD + 4]
    float* s_v = s_k + kRowsKeys * (HD + 4);         // [32][HD]
    float* s_p = s_v + kRowsKeys * HD;               // [32 rows][32 keys]
    TreeNodes& tree = *(TreeNodes*)(s_p + kRowsTile * kRowsKeys);
    constexpr int DPL = HD / 32;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, chunk = blockIdx.x, s = blockIdx.z, G = a.n_q / a.n_kv;
    const int kvh = blockIdx.y % a.n_kv, f0 = blockIdx.y / a.n_kv * kRowsTile;
    TreeSeq q;
    if (!tree_seq(a.t, &a.m, s, &q, a.status) || f0 >= q.n * G) return;
    const TreeWork w = tree_work(q.prefix, q.n, a.window);
    if (chunk * part.tiles >= w.n_tiles) return;
    tree_load(tree, a.t, q, tid, 256, a.status);
    for (int x = tid; x < kRowsTile * HD / 4; x += 256) {
        const int r = x / (HD / 4), c = x % (HD / 4) * 4, f = f0 + r;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (f < q.n * G) v = load4((const TQ*)a.q + (size_t)(q.r0 + f / G) * a.q_stride + ((size_t)kvh * G + f % G) * HD + c);
        *(float4*)(s_q + r * HD + c) = v;
    }
    const float scale = a.scale * kLog2e;
    float o[4][DPL], mx[4], l[4];
    int node[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        mx[r] = -INFINITY; l[r] = 0.0f;
        const int f = f0 + warp * 4 + r;
        node[r] = f < q.n * G ? f / G : -1;
#pragma unroll
        for (int i = 0; i < DPL; i++) o[r][i] = 0.0f;
    }
    const int j_first = (w.t_lo + chunk * part.tiles) * kTileKeys, j_end = min(w.n_keys, j_first + part.tiles * kTileKeys);
#pragma unroll 1
    for (int j0 = j_first; j0 < j_end; j0 += kRowsKeys) {
        __syncthreads();                             // (the tree and the queries are there; the tile before has been read)
        for (int x = tid; x < kRowsKeys * HD / 4; x += 256) {
            const int r = x / (HD / 4), c = x % (HD / 4) * 4, j = j0 + r;
            float4 kf = make_float4(0.0f, 0.0f, 0.0f, 0.0f), vf = kf;
            const long long at = j >= w.low && j < j_end ? tree_row(a.m, q.slot, j, a.status) : -1;
            if (at >= 0) {
                const size_t off = (size_t)at * a.kv_stride + (size_t)kvh * HD + c;
                kf = load4((const TK*)a.k + off);
                vf = load4((const TK*)a.v + off);
            }
            *(float4*)(s_k + r * (HD + 4) + c) = kf;
            *(float4*)(s_v + r * HD + c) = vf;
        }
        __syncthreads();
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const float* qr = s_q + warp * 4 * HD;
#pragma unroll 8
        for (int c = 0; c < HD; c += 4) {
            const float4 k4 = *(const float4*)(s_k + lane * (HD + 4) + c);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float4 q4 = *(const float4*)(qr + r * HD + c);
                x[r] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, x[r]))));
            }
        }
        const int j = j0 + lane;
        const bool live = j >= w.low && j < j_end;
        unsigned int vis[4], all = 0xffffffffu;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const bool see = live && node[r] >= 0 && tree_sees(tree, q, a.window, node[r], j);
            vis[r] = __ballot_sync(0xffffffffu, see);
            all &= vis[r];
            const float y = see ? x[r] * scale : -INFINITY;
            float top = y;
#pragma unroll
            for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
            const float mn = fmaxf(mx[r], top);
            const float p = see ? exp2f(y - (mn == -INFINITY ? 0.0f : mn)) : 0.0f;
            const float corr = mx[r] == mn ? 1.0f : exp2f(mx[r] - mn);
            l[r] = l[r] * corr + p;
            mx[r] = mn;
#pragma unroll
            for (int i = 0; i < DPL; i++) o[r][i] *= corr;
            s_p[(warp * 4 + r) * kRowsKeys + lane] = p;
        }
        __syncwarp();
        // a key that a row does not see adds nothing to it, whatever its value holds (0 times infinity is no zero)
#pragma unroll 4
        for (int key = 0; key < kRowsKeys; key++) {
            float v[DPL];
#pragma unroll
            for (int i = 0; i < DPL; i++) v[i] = s_v[key * HD + lane * DPL + i];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                if (all == 0xffffffffu || (vis[r] >> key & 1u)) {
                    const float p = s_p[(warp * 4 + r) * kRowsKeys + key];
#pragma unroll
                    for (int i = 0; i < DPL; i++) o[r][i] = fmaf(p, v[i], o[r][i]);
                }
            }
        }
        __syncwarp();
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        if (node[r] < 0) continue;
        const int f = f0 + warp * 4 + r, row = q.r0 + node[r], h = kvh * G + f % G;
        float sum = warp_sum(l[r]);
        if (part.chunks == 1) {
            float top = mx[r], c = 1.0f;
            if (a.sinks) {
                const float sink = a.sinks[h] * kLog2e;
                top = fmaxf(top, sink);
                c = mx[r] == -INFINITY ? 0.0f : exp2f(mx[r] - top);
                sum = sum * c + exp2f(sink - top);
            }
            const float inv = sum > 0.0f ? c / sum : sum;      // (undefined stays undefined)
            TQ* dst = (TQ*)a.out + (size_t)row * a.out_stride + (size_t)h * HD + lane * DPL;
#pragma unroll
            for (int i = 0; i < DPL; i++) dst[i] = out_of<TQ>(o[r][i] * inv);
        } else {
            const size_t at = part_at(a, chunk, row, h);
#pragma unroll
            for (int i = 0; i < DPL; i++) part.o[at * HD + lane * DPL + i] = o[r][i];
            if (lane == 0) { part.ml[2 * at] = mx[r]; part.ml[2 * at + 1] = sum; }
        }
    }
}

// ---- joins the chunks: a warp per (row, head); o = sum_c 2^(m_c - M) o_c / (sum_c 2^(m_c - M) l_c + 2^(sink - M))
template <int HD, typename TQ>
__global__ void __launch_bounds__(256) tree_combine(const TreeAttnArgs a, const Part part) {
    constexpr int DPL = HD / 32;
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= (long long)a.t.n_rows * a.n_q) return;
    const int row = (int)(item / a.n_q), h = (int)(item % a.n_q);
    // the row's sequence: the last one that starts at or before it
    int lo = 0, hi = a.t.n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(a.t.row_start + mid) <= row) lo = mid; else hi = mid - 1;
    }
    TreeSeq q;
    if (!tree_seq(a.t, &a.m, lo, &q, nullptr) || row < q.r0 || row >= q.r0 + q.n) return;
    const int n_tiles = tree_work(q.prefix, q.n, a.window).n_tiles, chunks = (n_tiles + part.tiles - 1) / part.tiles;
    float top = a.sinks ? a.sinks[h] * kLog2e : -INFINITY;
    for (int c = lane; c < chunks; c += 32) top = fmaxf(top, part.ml[2 * part_at(a, c, row, h)]);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
    float sum = a.sinks ? exp2f(a.sinks[h] * kLog2e - top) : 0.0f, o[DPL];
#pragma unroll
    for (int i = 0; i < DPL; i++) o[i] = 0.0f;
    for (int c = 0; c < chunks; c++) {
        const size_t at = part_at(a, c, row, h);
        const float m = part.ml[2 * at], l = part.ml[2 * at + 1];
        if (m == -INFINITY && l == 0.0f) continue;   // the chunk holds no key that this row sees
        const float f = m == top ? 1.0f : exp2f(m - top);
        sum = fmaf(l, f, sum);
#pragma unroll
        for (int i = 0; i < DPL; i++) o[i] = fmaf(part.o[at * HD + lane * DPL + i], f, o[i]);
    }
    const float inv = sum > 0.0f ? 1.0f / sum : sum;
    TQ* dst = (TQ*)a.out + (size_t)row * a.out_stride + (size_t)h * HD + lane * DPL;
#pragma unroll
    for (int i = 0; i < DPL; i++) dst[i] = out_of<TQ>(o[i] * inv);
}

// Chunks of keys: as many as give every SM work, from what the call knows on the host (the longest sequence).
Part plan(const TreeAttnArgs& a, int sm_count, int rows_tile, int per_sm) {
    Part p{};
    const int G = a.n_q / a.n_kv;
    int tiles = (int)(((long long)a.t.max_prefix + a.t.max_rows + kTileKeys - 1) / kTileKeys);
    if (a.window > 0) {
        const long long seen = ((long long)a.window + a.t.max_rows) / kTileKeys + 2;
        if (seen < tiles) tiles = (int)seen;
    }
    const long long units = (long long)a.t.n_seq * a.n_kv * ((a.t.max_rows * G + rows_tile - 1) / rows_tile), slots = (long long)sm_count * per_sm;
    long long want = (slots + units - 1) / units;
    if (want > tiles) want = tiles;
    if (want < 1) want = 1;
    p.tiles = (int)((tiles + want - 1) / want);
    p.chunks = (tiles + p.tiles - 1) / p.tiles;
    return p;
}
size_t part_bytes(const TreeAttnArgs& a, const Part& p) { return p.chunks > 1 ? (size_t)p.chunks * a.t.n_rows * a.n_q * (a.hd + 2) * 4 : 0; }

Part plan_of(const TreeAttnArgs& a, int sm_count) { return plan(a, sm_count, kRowsTile, 2); }

template <int HD, typename TQ>
cudaError_t combine(const TreeAttnArgs& a, const Part& p, cudaStream_t st) {
    const long long items = (long long)a.t.n_rows * a.n_q;
    tree_combine<HD, TQ><<<(unsigned)((items + 7) / 8), 256, 0, st>>>(a, p);
    return cudaGetLastError();
}
template <int HD, typename TQ, typename TK>
cudaError_t rows_launch(const TreeAttnArgs& a, const Part& p, cudaStream_t st) {
    static std::atomic<uint64_t> raised{0};
    if (const cudaError_t e = allow_smem(raised, (const void*)attn_tree_rows<HD, TQ, TK>, rows_smem<HD>())) return e;
    const int G = a.n_q / a.n_kv;
    attn_tree_rows<HD, TQ, TK><<<dim3(p.chunks, a.n_kv * ((a.t.max_rows * G + kRowsTile - 1) / kRowsTile), a.t.n_seq), 256, rows_smem<HD>(), st>>>(a, p);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess || p.chunks == 1 ? e : combine<HD, TQ>(a, p, st);
}

}  // namespace

size_t tree_attn_workspace(const TreeAttnArgs& a, int sm_count) { return part_bytes(a, plan_of(a, sm_count)); }

cudaError_t launch_tree_attn(const TreeAttnArgs& a, int sm_count, cudaStream_t st) {
    Part p = plan_of(a, sm_count);
    if (part_bytes(a, p) > a.ws_bytes) return cudaErrorInvalidValue;
    p.o = (float*)a.ws;
    p.ml = p.o + (size_t)p.chunks * a.t.n_rows * a.n_q * a.hd;
    using bf = __nv_bfloat16;
    if (a.hd == 128) return a.q_bf16 ? rows_launch<128, bf, bf>(a, p, st) : a.kv_bf16 ? rows_launch<128, float, bf>(a, p, st) : rows_launch<128, float, float>(a, p, st);
    return a.q_bf16 ? rows_launch<64, bf, bf>(a, p, st) : a.kv_bf16 ? rows_launch<64, float, bf>(a, p, st) : rows_launch<64, float, float>(a, p, st);
}

}  // namespace lum
