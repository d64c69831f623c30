// Attention of drafted trees over a K/V cache (lum_op_attn_tree): node i of sequence s, with p = prefix[s], sees the cached rows j < p, its ancestors a
// (row p + a) and itself:
//     o_i = sum_j w_ij v_j,   w_ij = exp(x_ij) / (sum_j exp(x_ij) + exp(sink)),   x_ij = scale q_i . k_j
// One pass over the keys with the running maximum and sum of the softmax.  All nodes of a tree and the G query heads of a K/V head share every key: row
// f = node * G + head of a K/V head's query rows.  The keys of a sequence are cut into chunks, one CTA each; where there are several, every chunk leaves its
// (maximum, sum, outputs) in the workspace and tree_combine joins them.
#include <cuda.h>
#include <type_traits>

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

// The tree in shared memory: depths and, as bits, the nodes that a node sees (itself and its ancestors, fewer than `window` places before it).  By
// `threads` threads that share barrier `id` (0: the whole CTA); synchronise afterwards.
struct TreeNodes { unsigned int anc[kTreeMax][kTreeWords]; short depth[kTreeMax]; short parent[kTreeMax]; };
__device__ __forceinline__ void tree_load(TreeNodes& s, const TreeBatch& t, const TreeSeq& q, int window, int tid, int threads, int id, uint32_t* status) {
    for (int i = tid; i < q.n; i += threads) {
        int p = __ldg(t.parent + q.r0 + i);
        if (p < -1 || p >= i) { p = -1; if (status) atomicOr(status, LUM_ST_BAD_TREE); }
        s.parent[i] = (short)p;
    }
    named_sync(id, threads);
    for (int i = tid; i < q.n; i += threads) {
        unsigned int w[kTreeWords];
#pragma unroll
        for (int k = 0; k < kTreeWords; k++) w[k] = 0u;
        int depth = -1;
        for (int a = i; a >= 0; a = s.parent[a]) {
            depth++;
            if (window > 0 && depth >= window) continue;
#pragma unroll
            for (int k = 0; k < kTreeWords; k++) if (k == a >> 5) w[k] |= 1u << (a & 31);
        }
#pragma unroll
        for (int k = 0; k < kTreeWords; k++) s.anc[i][k] = w[k];
        s.depth[i] = (short)depth;
    }
}
// whether node i sees cache row j of its sequence (j < n_keys)
__device__ __forceinline__ bool tree_sees(const TreeNodes& s, const TreeSeq& q, int window, int i, int j) {
    const int a = j - q.prefix;
    if (a < 0) return window <= 0 || q.prefix + s.depth[i] - j < window;
    return s.anc[i][a >> 5] >> (a & 31) & 1u;
}

struct Part {                                        // where chunk c leaves its share of (row, head); out is used where there is one chunk
    float *o, *ml;                                   // [chunk][row][head][hd], [chunk][row][head][2]
    int chunks, tiles;                               // chunks of the longest sequence, tiles of a chunk
};
__device__ __forceinline__ size_t part_at(const TreeAttnArgs& a, int c, int row, int h) { return ((size_t)c * a.t.n_rows + row) * a.n_q + h; }

template <typename T> __device__ __forceinline__ T out_of(float x);
template <> __device__ __forceinline__ float out_of<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 out_of<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }      // the one rounding of the result

// ---- products on CUDA cores, in 32 bits: an f32 cache
// CTA = chunk x (K/V head, 32 query rows) x sequence; 8 warps of 4 query rows.  32 keys at a time lie in shared memory as f32: a lane multiplies its key with
// the warp's four rows, and then four (two) dimensions of the values with their weights.
constexpr int kRowsTile = 32, kRowsKeys = 32;
template <int HD>
constexpr int rows_smem() { return (kRowsTile * HD + kRowsKeys * (HD + 4) + kRowsKeys * HD + kRowsTile * kRowsKeys) * 4 + (int)sizeof(TreeNodes); }

template <int HD>
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
    tree_load(tree, a.t, q, a.window, tid, 256, 0, a.status);
    for (int x = tid; x < kRowsTile * HD / 4; x += 256) {
        const int r = x / (HD / 4), c = x % (HD / 4) * 4, f = f0 + r;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (f < q.n * G) v = *(const float4*)((const float*)a.q + (size_t)(q.r0 + f / G) * a.q_stride + ((size_t)kvh * G + f % G) * HD + c);
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
                kf = *(const float4*)((const float*)a.k + off);
                vf = *(const float4*)((const float*)a.v + off);
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
            float* dst = (float*)a.out + (size_t)row * a.out_stride + (size_t)h * HD + lane * DPL;
#pragma unroll
            for (int i = 0; i < DPL; i++) dst[i] = o[r][i] * inv;
        } else {
            const size_t at = part_at(a, chunk, row, h);
#pragma unroll
            for (int i = 0; i < DPL; i++) part.o[at * HD + lane * DPL + i] = o[r][i];
            if (lane == 0) { part.ml[2 * at] = mx[r]; part.ml[2 * at + 1] = sum; }
        }
    }
}

// ---- products on the tensor core (tcgen05): a bf16 cache
// CTA = chunk x (K/V head, 128 query rows) x sequence: four softmax warps, a thread per query row; one warp that asks for keys, one for
// values, one that issues the products.  Per tile of 64 cache rows:
//     S = Q K^T             M 128, N 64; Q in shared memory, one bf16 term (bf16 queries) or three (f32 queries, 24 bits)
//     p = 2^(S - m)         a thread reads its row's 64 scores, masks, exponentiates, and stores the weights' terms over them
//     O (+)= P V            M 128, N head_dim; P from tensor memory, V as stored (MN-major)
// Tiles arrive by one tensor-map copy each for K and V (a box per page where pages are smaller than a tile), two tiles ahead; rows that the call must not
// read (before the window, behind the last node, pages outside the pool) are asked for outside the tensor and read as zeros.  S(t + 1) is computed while tile t
// is exponentiated.
//   bf16 results: O stays in tensor memory.  m is the maximum of some tile before: it follows a row's true maximum only when that has grown by 8 (weights up to
//     2^8 lose nothing in f32), so O is rescaled a few times per chunk at most.  Weights enter as two bf16 terms: one would add an error as large as the rounding of
//     the result (2^-9 each).
//   f32 results: three terms of the weights, and a tile's O is added up in registers: the tensor core's accumulator cuts every addition to 24 bits, and over
//     thousands of keys the cuts add up.  Low terms go first.
// A key that a row does not see has weight 0, but 0 times infinity is no zero: rows of V behind the last node or before the window are zeroed, and a row whose
// result is not finite is computed again by tree_row_plain, key by key.
constexpr int kTcThreads = 224;                     // four softmax warps, K, products, V
constexpr int kTcGroup = 128 * 16 + 16;              // Q: 16-byte column groups of 128 rows, the next one 16 bytes further on (banks)
template <int HD, bool F32>
struct TcShape {
    static constexpr int q_terms = F32 ? 3 : 1, p_terms = F32 ? 3 : 2;
    static constexpr int tile = kTileKeys * HD * 2;  // bytes of K (or V)
    static constexpr int q_bytes = HD / 8 * kTcGroup;
    static constexpr int off_k = 0, off_v = 2 * tile, off_q = 4 * tile, off_misc = off_q + q_terms * q_bytes, off_tree = off_misc + 128 + 32 * 4;
    static constexpr int smem = off_tree + (int)sizeof(TreeNodes);
    static constexpr int ctas = F32 && HD == 128 ? 1 : 2;                 // per SM
    static constexpr int cols = F32 && HD == 128 ? 512 : 256;             // tensor memory: scores 2 x 64, O, third terms 2 x 32
    static constexpr int col_o = 128, col_x = 128 + HD;
};
__host__ __device__ constexpr uint32_t tc_idesc(int n, bool b_mn) { return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24); }
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ uint64_t tc_desc_sw128(uint32_t addr, uint32_t lbo, uint32_t sbo) { return umma_smem_desc(addr, lbo, sbo) | (2ull << 61); }
__device__ __forceinline__ void tc_ld32(uint32_t at, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                   "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
                   "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(at) : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t at, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
                 "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
                 "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]) : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t at, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float tc_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// two at a time: the softmax warps are bound by what they issue (beside their exponentials)
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// (x0, x1) as packed bf16, rounded; what is left of them goes back
__device__ __forceinline__ uint32_t tc_term(float* x0, float* x1) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(*x0, *x1);
    const uint32_t b = *(const uint32_t*)&h;
    const float2 r = fma2(make_float2(__uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u)), make_float2(-1.0f, -1.0f), make_float2(*x0, *x1));
    *x0 = r.x; *x1 = r.y;
    return b;
}
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int row, int col, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(0), "r"(row), "r"(col), "r"(bar) : "memory");
}

// One query row (f of its K/V head) over cache rows [j0, j1) by a warp, in f32 and key by key: (m, l) in every lane, out[i] = dimension lane * HD / 32 + i.
template <int HD, typename TQ>
__device__ __noinline__ void tree_row_plain(const TreeAttnArgs& a, const TreeNodes& tree, const TreeSeq& q, int kvh, int f, int j0, int j1, int lane, float* m, float* l, float* out) {
    constexpr int DPL = HD / 32;
    const int G = a.n_q / a.n_kv, node = f / G;
    const float scale = a.scale * kLog2e;
    const TQ* src = (const TQ*)a.q + (size_t)(q.r0 + node) * a.q_stride + ((size_t)kvh * G + f % G) * HD + lane * DPL;
    float x[DPL], o[DPL], mx = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < DPL; i++) { x[i] = (float)src[i]; o[i] = 0.0f; }
    for (int j = j0; j < j1; j++) {
        if (!tree_sees(tree, q, a.window, node, j)) continue;
        const long long at = tree_row(a.m, q.slot, j, nullptr);
        if (at < 0) continue;
        const size_t off = (size_t)at * a.kv_stride + (size_t)kvh * HD + lane * DPL;
        float d = 0.0f;
#pragma unroll
        for (int i = 0; i < DPL; i++) d = fmaf(x[i], __bfloat162float(((const __nv_bfloat16*)a.k)[off + i]), d);
        d = warp_sum(d) * scale;
        const float mn = fmaxf(mx, d), c = mx == mn ? 1.0f : exp2f(mx - mn), p = exp2f(d - (mn == -INFINITY ? 0.0f : mn));
        sum = sum * c + p;
#pragma unroll
        for (int i = 0; i < DPL; i++) o[i] = fmaf(p, __bfloat162float(((const __nv_bfloat16*)a.v)[off + i]), o[i] * c);
        mx = mn;
    }
    *m = mx; *l = sum;
#pragma unroll
    for (int i = 0; i < DPL; i++) out[i] = o[i];
}
// A finished row of a call with one chunk: 1 / l and the sink's share.
__device__ __forceinline__ float tree_inverse(const TreeAttnArgs& a, int h, float m, float l) {
    if (!a.sinks) return l > 0.0f ? 1.0f / l : l;    // (undefined stays undefined)
    const float sink = a.sinks[h] * kLog2e, top = fmaxf(m, sink), c = m == -INFINITY ? 0.0f : exp2f(m - top);
    const float sum = l * c + exp2f(sink - top);
    return sum > 0.0f ? c / sum : sum;
}

template <int HD, bool F32>
__global__ void __launch_bounds__(kTcThreads, TcShape<HD, F32>::ctas) attn_tree_tc(const __grid_constant__ TreeAttnArgs a, const Part part, const __grid_constant__ CUtensorMap map_k,
                                                                                   const __grid_constant__ CUtensorMap map_v, int box_rows) {
    using S = TcShape<HD, F32>;
    using TQ = typename std::conditional<F32, float, __nv_bfloat16>::type;
    extern __shared__ __align__(1024) unsigned char tc_smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, chunk = blockIdx.x, s = blockIdx.z, G = a.n_q / a.n_kv;
    const int kvh = blockIdx.y % a.n_kv, f0 = blockIdx.y / a.n_kv * 128;
    const uint32_t base = smem_u32(tc_smem), misc = base + S::off_misc;
    const uint32_t bar_k = misc, bar_v = misc + 16, bar_s = misc + 32, bar_p = misc + 48, bar_o = misc + 64;      // two of each: tile t uses number t % 2
    volatile int* gave_up = (volatile int*)(tc_smem + S::off_misc + 88);
    unsigned int* s_odd = (unsigned int*)(tc_smem + S::off_misc + 96);       // [4]: rows whose result is not finite
    TreeNodes& tree = *(TreeNodes*)(tc_smem + S::off_tree);
    if (part.chunks > 1) pdl_launch_dependents();    // (tree_combine waits for this kernel's end)
    TreeSeq q = tree_seq_load(a.t, s);               // on its way while the CTA sets itself up
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(bar_k + 8 * i, 1);             // K(t) has landed
            mbar_init(bar_v + 8 * i, 1);             // V(t)
            mbar_init(bar_s + 8 * i, 1);             // S(t) is there, K(t) is no longer read
            mbar_init(bar_p + 8 * i, 4);             // P(t) is stored, O may be added to
            mbar_init(bar_o + 8 * i, 1);             // O holds tile t, V(t) is no longer read
        }
        mbar_fence_init();
        *gave_up = 0;
    }
    if (tid < 4) s_odd[tid] = 0u;
    if (warp == 5) tmem_alloc(misc + 80, S::cols);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *(volatile uint32_t*)(tc_smem + S::off_misc + 80);
    const bool ok = tree_seq_ok(a.t, &a.m, &q, a.status);
    const TreeWork w = tree_work(q.prefix, q.n, a.window);
    const int t_first = w.t_lo + chunk * part.tiles, n_tiles = min(part.tiles, w.t_lo + w.n_tiles - t_first);
    if (!ok || f0 >= q.n * G || n_tiles <= 0) {
        if (warp == 5) tmem_dealloc(tmem, S::cols);
        return;
    }
    const int live_rows = min(128, q.n * G - f0);
    const uint32_t magic = 0xffffffffu / (uint32_t)G + 1u;               // f / G = f magic / 2^32 for f < 2^18, 2 <= G <= 2^10
    auto node_of = [&](int f) { return G == 1 ? f : (int)__umulhi((uint32_t)f, magic); };

    // A wait that runs out of its budget is remembered; what follows hardly waits and multiplies no more, but meets every barrier.
    auto wait = [&](uint32_t bar, int t) {
        const uint32_t at = bar + 8u * (t & 1), parity = (uint32_t)(t >> 1) & 1u;
        if (mbar_try_wait(at, parity)) return;
        if (!mbar_wait_abortable(at, parity, gave_up)) *gave_up = 1;
    };
    constexpr int kHalves = HD / 64;
    // Where this lane's box of tile t starts in the cache (a lane per box); one page-table entry on its way while the tile before is waited for.
    auto box_row = [&](int t) {
        const int j = (t_first + t) * kTileKeys + lane * box_rows;
        if (t >= n_tiles || lane >= kTileKeys / box_rows || j >= w.n_keys || j + box_rows <= w.low) return (int)a.m.rows;     // outside the tensor: zeros
        const long long row = tree_row(a.m, q.slot, j, a.status);
        return (int)(row < 0 ? a.m.rows : row);
    };
    auto load = [&](const CUtensorMap* map, int t, int row, uint32_t dst, uint32_t full) {
        const uint32_t bar = full + 8u * (t & 1);
        dst += (uint32_t)(t & 1) * S::tile;
        if (lane == 0) mbar_arrive_expect_tx(bar, S::tile);
        __syncwarp();
        // a box holds its halves of 64 dimensions one behind the other; a whole tile's are kTileKeys rows apart
        if (box_rows == kTileKeys) { if (elect_one()) tma_box(dst, map, row, kvh * kHalves, bar); }
        else if (lane < kTileKeys / box_rows)
#pragma unroll
            for (int h = 0; h < kHalves; h++) tma_box(dst + h * (kTileKeys * 128) + lane * box_rows * 128, map, row, kvh * kHalves + h, bar);
    };
    const bool loads_k = warp == 4, loads = loads_k || warp == 6;
    int next_row = 0;
    if (loads) {
        const int first = box_row(0);
        const int second = box_row(1);
        next_row = box_row(2);
        load(loads_k ? &map_k : &map_v, 0, first, base + (loads_k ? S::off_k : S::off_v), loads_k ? bar_k : bar_v);
        if (n_tiles > 1) load(loads_k ? &map_k : &map_v, 1, second, base + (loads_k ? S::off_k : S::off_v), loads_k ? bar_k : bar_v);
    }
    // ---- the tree, by the warps that then only issue; the queries, by the others
    if (loads) {
        tree_load(tree, a.t, q, a.window, (warp == 6 ? 32 : 0) + lane, 64, 1, a.status);
        named_arrive(3, 192);
    } else if (warp < 4) {
        // (rows beyond the last query are left as they are: nobody reads what they make)
        constexpr int kPieces = HD / 8, kStep = 128 / kPieces, kAhead = F32 ? 2 : 4;
        const int c = tid % kPieces;
        for (int r0 = tid / kPieces; r0 < live_rows; r0 += kStep * kAhead) {
            uint4 raw[kAhead][F32 ? 2 : 1];
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                const int f = f0 + min(r0 + u * kStep, live_rows - 1), node = node_of(f);
                const uint4* src = (const uint4*)((const TQ*)a.q + (size_t)(q.r0 + node) * a.q_stride + ((size_t)kvh * G + f - node * G) * HD + c * 8);
#pragma unroll
                for (int e = 0; e < (F32 ? 2 : 1); e++) raw[u][e] = src[e];
            }
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                const int r = r0 + u * kStep;
                if (r >= live_rows) break;
                unsigned char* dst = tc_smem + S::off_q + c * kTcGroup + r * 16;
                if constexpr (F32) {
                    float* y = (float*)raw[u];
#pragma unroll
                    for (int e = 0; e < 3; e++) *(uint4*)(dst + e * S::q_bytes) = make_uint4(tc_term(y, y + 1), tc_term(y + 2, y + 3), tc_term(y + 4, y + 5), tc_term(y + 6, y + 7));
                } else *(uint4*)dst = raw[u][0];
            }
        }
        fence_proxy_async_smem();
        named_arrive(2, 160);
    } else named_sync(2, 160);                       // (the queries are there)

    float m_run = -INFINITY, l_run = 0.0f;
    float o[F32 ? HD : 1];
    const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int row = warp * 32 + lane, f = f0 + row, node = row < live_rows && warp < 4 ? node_of(f) : -1;
    if (loads) {
        // K(t + 2) goes out when S(t) is there, V(t + 2) when O holds tile t
        const CUtensorMap* map = loads_k ? &map_k : &map_v;
        const uint32_t dst = base + (loads_k ? S::off_k : S::off_v), full = loads_k ? bar_k : bar_v, used = loads_k ? bar_s : bar_o;
        int last = min(n_tiles, 2) - 1;
        for (int t = 2; t < n_tiles; t++) {
            const int row = next_row;
            next_row = box_row(t + 1);
            wait(used, t - 2);
            if (__any_sync(0xffffffffu, *gave_up)) break;
            load(map, last = t, row, dst, full);
        }
        // no copy is on its way when the CTA ends (they have landed long ago, unless a wait was given up)
        for (int t = max(last - 1, 0); t <= last; t++) mbar_wait(full + 8u * (t & 1), (uint32_t)(t >> 1) & 1u);
    } else if (warp == 5) {
        constexpr uint32_t id_s = tc_idesc(kTileKeys, false), id_o = tc_idesc(HD, true);
        if (elect_one()) {
#pragma unroll 1
            for (int t = 0; t <= n_tiles; t++) {
                if (t < n_tiles) {
                    wait(bar_k, t);
                    if (*gave_up) break;
                    tc_fence_after_sync();
                    const uint32_t kb = base + S::off_k + (t & 1) * S::tile, d = tmem + (uint32_t)(t & 1) * 64u;
#pragma unroll
                    for (int e = S::q_terms - 1; e >= 0; e--)
#pragma unroll
                        for (int ks = 0; ks < HD / 16; ks++)
                            tc_mma(d, umma_smem_desc(base + S::off_q + e * S::q_bytes + ks * 2 * kTcGroup, kTcGroup, 128), tc_desc_sw128(kb + (ks >> 2) * (kTileKeys * 128) + (ks & 3) * 32, 16, 1024),
                                   id_s, e != S::q_terms - 1 || ks ? 1u : 0u);
                    umma_commit(bar_s + 8u * (t & 1));
                }
                if (t > 0) {
                    const int u = t - 1;
                    wait(bar_v, u);
                    wait(bar_p, u);
                    if (*gave_up) break;
                    tc_fence_after_sync();
                    const uint32_t vb = base + S::off_v + (u & 1) * S::tile, p = tmem + (uint32_t)(u & 1) * 64u, px = tmem + S::col_x + (uint32_t)(u & 1) * 32u, d = tmem + S::col_o;
#pragma unroll
                    for (int e = S::p_terms - 1; e >= 0; e--)
#pragma unroll
                        for (int ks = 0; ks < kTileKeys / 16; ks++)
                            tc_mma_ts(d, (e == 2 ? px : p + e * 32u) + ks * 8u, tc_desc_sw128(vb + ks * 2048, kTileKeys * 128, 1024), id_o, (!F32 && u) || e != S::p_terms - 1 || ks ? 1u : 0u);
                    umma_commit(bar_o + 8u * (u & 1));
                }
            }
        }
        __syncwarp();
    } else {
        if constexpr (F32)
#pragma unroll
            for (int i = 0; i < HD; i++) o[i] = 0.0f;
        const float scale = a.scale * kLog2e;
        auto zero_v = [&](int t) {                   // rows of V(t) that no query row may see
            const int j0 = (t_first + t) * kTileKeys;
            if (j0 >= w.low && j0 + kTileKeys <= w.n_keys) return;
            wait(bar_v, t);
            unsigned char* vb = tc_smem + S::off_v + (t & 1) * S::tile;
            for (int x = tid; x < kTileKeys * (HD / 8); x += 128) {
                const int j = x / (HD / 8), c = x % (HD / 8);
                if (j0 + j < w.low || j0 + j >= w.n_keys) *(uint4*)(vb + (c >> 3) * (kTileKeys * 128) + j * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();
        };
#pragma unroll 1
        for (int t = 0; t < n_tiles; t++) {
            if (t > 1) wait(bar_o, t - 2);           // (long there: every phase of bar_o is seen, and V(t - 2) has been used)
            zero_v(t);
            wait(bar_s, t);
            tc_fence_after_sync();
            if (t == 0) named_sync(3, 192);          // (the tree is there)
            if (warp * 32 < live_rows) {             // (a warp without live rows leaves its rows of P as they are: nobody reads what they make)
                const uint32_t sc = mine + (uint32_t)(t & 1) * 64u;
                float v[64];
                tc_ld32(sc, (uint32_t*)v);
                tc_ld32(sc + 32u, (uint32_t*)v + 32);
                tmem_ld_wait();
                const int j0 = (t_first + t) * kTileKeys;
                if (j0 + kTileKeys > q.prefix || a.window > 0) {         // some key may be out of some row's sight
                    unsigned long long see = 0ull;
                    if (node >= 0) {
                        const int cached = q.prefix - j0;                // keys of the tile before the tree
                        see = cached >= 64 ? ~0ull : cached > 0 ? (1ull << cached) - 1 : 0ull;
                        const int first = q.prefix + tree.depth[node] - a.window + 1 - j0;
                        if (a.window > 0 && first > 0) see = first >= 64 ? 0ull : see & (~0ull << first);
#pragma unroll
                        for (int k = 0; k < kTreeWords; k++) {           // nodes 32 k .. 32 k + 31 are the keys from 32 k + cached on
                            const int at = 32 * k + cached;
                            if (32 * k < q.n && at < 64 && at > -32) see |= at >= 0 ? (unsigned long long)tree.anc[node][k] << at : (unsigned long long)(tree.anc[node][k] >> -at);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        if (!((uint32_t)see >> i & 1u)) v[i] = -INFINITY;
                        if (!((uint32_t)(see >> 32) >> i & 1u)) v[32 + i] = -INFINITY;
                    }
                }
                float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                for (int i = 4; i < 60; i += 8)
#pragma unroll
                    for (int e = 0; e < 4; e++) top[e] = fmaxf(top[e], fmaxf(v[i + e], v[i + 4 + e]));
#pragma unroll
                for (int e = 0; e < 4; e++) top[e] = fmaxf(top[e], v[60 + e]);
                const float tm = node >= 0 ? fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale : -INFINITY;
                // the reference of the exponents: kept while nothing is more than 2^8 times it
                const bool grows = tm > m_run + (F32 ? 0.0f : 8.0f) || m_run == -INFINITY;
                const float m_new = grows ? fmaxf(tm, m_run) : m_run;
                const float alpha = m_new == m_run ? 1.0f : tc_ex2(m_run - m_new);
                m_run = m_new;
                const float off = m_new == -INFINITY ? 0.0f : -m_new;
                float2 sum[2] = {};
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                    const float2 x = fma2(make_float2(v[i], v[i + 1]), make_float2(scale, scale), make_float2(off, off));
                    v[i] = tc_ex2(x.x); v[i + 1] = tc_ex2(x.y);
                    sum[i >> 1 & 1] = add2(sum[i >> 1 & 1], make_float2(v[i], v[i + 1]));
                }
                l_run = l_run * alpha + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
                if constexpr (F32) {
                    uint32_t pk[16];
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int e = 0; e < 3; e++) {
#pragma unroll
                            for (int i = 0; i < 16; i++) pk[i] = tc_term(&v[h * 32 + 2 * i], &v[h * 32 + 2 * i + 1]);
                            tc_st16(e == 2 ? mine + S::col_x + (uint32_t)(t & 1) * 32u + h * 16u : sc + e * 32u + h * 16u, pk);
                        }
                } else {
                    uint32_t pk[32];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
#pragma unroll
                        for (int i = 0; i < 32; i++) pk[i] = tc_term(&v[2 * i], &v[2 * i + 1]);
                        tc_st32(sc + e * 32u, pk);
                    }
                }
                if (t > 0) {
                    if constexpr (F32) {             // O(t - 1) comes out before O(t) is made
                        wait(bar_o, t - 1);
                        tc_fence_after_sync();
#pragma unroll
                        for (int c = 0; c < HD / 32; c++) {
                            uint32_t y[32];
                            tc_ld32(mine + S::col_o + c * 32u, y);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; i++) o[c * 32 + i] = (o[c * 32 + i] + __uint_as_float(y[i])) * alpha;
                        }
                    } else if (__any_sync(0xffffffffu, alpha != 1.0f)) {
                        wait(bar_o, t - 1);
                        tc_fence_after_sync();
#pragma unroll 1
                        for (int c = 0; c < HD / 32; c++) {
                            uint32_t y[32];
                            tc_ld32(mine + S::col_o + c * 32u, y);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; i++) y[i] = __float_as_uint(__uint_as_float(y[i]) * alpha);
                            tc_st32(mine + S::col_o + c * 32u, y);
                        }
                    }
                }
                tc_st_wait();
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_p + 8u * (t & 1));
        }
        if (n_tiles > 1) wait(bar_o, n_tiles - 2);
        wait(bar_o, n_tiles - 1);
        tc_fence_after_sync();
        // ---- out = O / l, or this chunk's share
        if (warp * 32 < live_rows) {
            const int h = kvh * G + (node >= 0 ? f - node * G : 0), out_row = q.r0 + max(node, 0);
            const float inv = part.chunks == 1 && node >= 0 ? tree_inverse(a, h, m_run, l_run) : 1.0f;
            float odd = l_run * 0.0f;                // 0, or NaN where something is not finite
            const size_t at = part_at(a, chunk, out_row, h);
#pragma unroll
            for (int c = 0; c < HD / 32; c++) {
                uint32_t y[32];
                tc_ld32(mine + S::col_o + c * 32u, y);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    float x = __uint_as_float(y[i]);
                    if constexpr (F32) x += o[c * 32 + i];
                    odd = fmaf(x, 0.0f, odd);
                    y[i] = __float_as_uint(x * inv);
                }
                if (node >= 0) {
                    if (part.chunks > 1) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) *(uint4*)(part.o + at * HD + c * 32 + i) = make_uint4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                    } else {
                        TQ* dst = (TQ*)a.out + (size_t)out_row * a.out_stride + (size_t)h * HD + c * 32;
                        if constexpr (F32) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4) *(uint4*)(dst + i) = make_uint4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i += 8) {
                                uint32_t b[4];
#pragma unroll
                                for (int e = 0; e < 4; e++) {            // the one rounding of the result
                                    const __nv_bfloat162 r = __floats2bfloat162_rn(__uint_as_float(y[i + 2 * e]), __uint_as_float(y[i + 2 * e + 1]));
                                    b[e] = *(const uint32_t*)&r;
                                }
                                *(uint4*)(dst + i) = make_uint4(b[0], b[1], b[2], b[3]);
                            }
                        }
                    }
                }
            }
            if (part.chunks > 1 && node >= 0) { part.ml[2 * at] = m_run; part.ml[2 * at + 1] = l_run; }
            const unsigned int bad = __ballot_sync(0xffffffffu, node >= 0 && odd != 0.0f);
            if (lane == 0) s_odd[warp] = bad;
        }
        tc_fence_before_sync();
    }
    __syncthreads();
    if (warp == 5) tmem_dealloc(tmem, S::cols);
    if (*gave_up) {
        if (tid == 0) atomicOr(a.status, LUM_ST_WAIT_TMEM);
        return;
    }
    // rows that are not finite, once more and key by key
    const int j_first = max(t_first * kTileKeys, w.low), j_end = min(w.n_keys, (t_first + n_tiles) * kTileKeys);
    for (int r = warp; r < live_rows; r += kTcThreads / 32) {
        if (!(s_odd[r >> 5] >> (r & 31) & 1u)) continue;
        const int fr = f0 + r, h = kvh * G + fr % G, out_row = q.r0 + fr / G;
        float m, l, x[HD / 32];
        tree_row_plain<HD, TQ>(a, tree, q, kvh, fr, j_first, j_end, lane, &m, &l, x);
        if (part.chunks > 1) {
            const size_t at = part_at(a, chunk, out_row, h);
            for (int i = 0; i < HD / 32; i++) part.o[at * HD + lane * (HD / 32) + i] = x[i];
            if (lane == 0) { part.ml[2 * at] = m; part.ml[2 * at + 1] = l; }
        } else {
            const float inv = tree_inverse(a, h, m, l);
            TQ* dst = (TQ*)a.out + (size_t)out_row * a.out_stride + (size_t)h * HD + lane * (HD / 32);
            for (int i = 0; i < HD / 32; i++) dst[i] = out_of<TQ>(x[i] * inv);
        }
    }
}

// ---- joins the chunks: a warp per (row, head); o = sum_c 2^(m_c - M) o_c / (sum_c 2^(m_c - M) l_c + 2^(sink - M))
template <int HD, typename TQ>
__global__ void __launch_bounds__(256) tree_combine(const TreeAttnArgs a, const Part part) {
    constexpr int DPL = HD / 32;
    pdl_grid_wait();
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

Part plan_of(const TreeAttnArgs& a, int sm_count) { return a.kv_bf16 ? plan(a, sm_count, 128, !a.q_bf16 && a.hd == 128 ? 1 : 2) : plan(a, sm_count, kRowsTile, 2); }

// A cache as a tensor [dimension groups of 64][row][64]: one copy brings both halves of a head of 128.
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
cudaError_t tensor_map(CUtensorMap* map, const TreeAttnArgs& a, const void* cache, int box_rows) {
    static std::atomic<EncodeTiled> found{nullptr};
    EncodeTiled encode = found.load(std::memory_order_acquire);
    if (!encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult res;
        if (const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &res)) return e;
        if (!fn || res != cudaDriverEntryPointSuccess) return cudaErrorNotSupported;
        encode = (EncodeTiled)fn;
        found.store(encode, std::memory_order_release);
    }
    const cuuint64_t dims[3] = {64, (cuuint64_t)a.m.rows, (cuuint64_t)a.n_kv * a.hd / 64}, strides[2] = {(cuuint64_t)a.kv_stride * 2, 128};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, box_rows == kTileKeys ? (cuuint32_t)a.hd / 64 : 1u}, step[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(cache), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <int HD, typename TQ>
cudaError_t combine(const TreeAttnArgs& a, const Part& p, cudaStream_t st) {
    const long long items = (long long)a.t.n_rows * a.n_q;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((items + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // its CTAs are there when the last chunk ends
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, tree_combine<HD, TQ>, a, p);
}
template <int HD>
cudaError_t rows_launch(const TreeAttnArgs& a, const Part& p, cudaStream_t st) {
    static std::atomic<uint64_t> raised{0};
    if (const cudaError_t e = allow_smem(raised, (const void*)attn_tree_rows<HD>, rows_smem<HD>())) return e;
    const int G = a.n_q / a.n_kv;
    attn_tree_rows<HD><<<dim3(p.chunks, a.n_kv * ((a.t.max_rows * G + kRowsTile - 1) / kRowsTile), a.t.n_seq), 256, rows_smem<HD>(), st>>>(a, p);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess || p.chunks == 1 ? e : combine<HD, float>(a, p, st);
}

template <int HD, bool F32>
cudaError_t tc_launch(const TreeAttnArgs& a, const Part& p, cudaStream_t st) {
    using S = TcShape<HD, F32>;
    static std::atomic<uint64_t> raised{0};
    if (const cudaError_t e = allow_smem(raised, (const void*)attn_tree_tc<HD, F32>, S::smem, true)) return e;
    const int G = a.n_q / a.n_kv, box_rows = a.m.lg >= 0 && 1 << a.m.lg < kTileKeys ? 1 << a.m.lg : kTileKeys;
    CUtensorMap map_k, map_v;
    if (const cudaError_t e = tensor_map(&map_k, a, a.k, box_rows)) return e;
    if (const cudaError_t e = tensor_map(&map_v, a, a.v, box_rows)) return e;
    attn_tree_tc<HD, F32><<<dim3(p.chunks, a.n_kv * ((a.t.max_rows * G + 127) / 128), a.t.n_seq), kTcThreads, S::smem, st>>>(a, p, map_k, map_v, box_rows);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess || p.chunks == 1 ? e : combine<HD, typename std::conditional<F32, float, __nv_bfloat16>::type>(a, p, st);
}

}  // namespace

size_t tree_attn_workspace(const TreeAttnArgs& a, int sm_count) { return part_bytes(a, plan_of(a, sm_count)); }

cudaError_t launch_tree_attn(const TreeAttnArgs& a, int sm_count, cudaStream_t st) {
    Part p = plan_of(a, sm_count);
    if (part_bytes(a, p) > a.ws_bytes) return cudaErrorInvalidValue;
    p.o = (float*)a.ws;
    p.ml = p.o + (size_t)p.chunks * a.t.n_rows * a.n_q * a.hd;
    if (!a.kv_bf16) return a.hd == 128 ? rows_launch<128>(a, p, st) : rows_launch<64>(a, p, st);
    if (a.hd == 128) return a.q_bf16 ? tc_launch<128, false>(a, p, st) : tc_launch<128, true>(a, p, st);
    return a.q_bf16 ? tc_launch<64, false>(a, p, st) : tc_launch<64, true>(a, p, st);
}

}  // namespace lum
