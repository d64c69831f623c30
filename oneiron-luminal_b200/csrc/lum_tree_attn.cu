// Attention of drafted trees over a K/V cache (lum_op_attn_tree): node i of sequence s, with p = prefix[s], sees the cached rows j < p, its ancestors a
// (row p + a) and itself:
//     o_i = sum_j w_ij v_j,   w_ij = exp(x_ij) / (sum_j exp(x_ij) + exp(sink)),   x_ij = scale q_i . k_j
// One pass over the keys with the running maximum and sum of the softmax.  All nodes of a tree and the G query heads of a K/V head share every key: row
// f = node * G + head of a K/V head's query rows.
#include <cuda.h>
#include <algorithm>
#include <type_traits>
#include <utility>

#include "lum_tree.cuh"

namespace lum {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kJoinCtas = 5;                         // CTAs of tree_combine per SM
constexpr int kClusterMax = 8;                       // CTAs of a (portable) cluster
constexpr int kTileKeys = 64;                        // tiles of so many cache rows, from the first visible one's tile on

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

// How the work is shared out.  A unit is a (sequence, K/V head, tile of query rows); it may be cut into equal pieces of its tiles of keys, one CTA per piece.  How
// long a piece may be is chosen on the device, where the lengths are.  A whole unit is finished by its CTA; a unit in pieces leaves a share (maximum, sum,
// outputs) of each in the workspace, and tree_combine joins them.  Or, where the call knows that units are few, every unit has a cluster of CTAs, which join their shares
// themselves (cluster_of says when).
constexpr int kNoCut = 1 << 30;                       // as the longest piece: longer than any unit
struct Share {
    int* plan;                                       // [0] tiles of a piece at most, [1 + s] the first share of sequence s; written by CTA 0 for tree_combine
    float *ml, *o;                                   // [share][rows][2], [share][rows][hd]
    int grid, shares, slots;                         // CTAs launched, shares there is room for, CTAs that run at once
    int copies, rows, tile_rows;                     // copies of a query row in a tile, query rows of a share, of a unit
    int cluster, row_tiles, sms;                     // > 1: a cluster of so many CTAs per unit; units of a K/V head there may be; the card's SMs
};
__device__ __forceinline__ size_t share_at(const Share& p, int share, int r) { return (size_t)share * p.rows + r; }

struct alignas(16) Piece {
    TreeSeq q;
    TreeWork w;
    int s, kvh, f0, tile, tiles, share;              // sequence, K/V head, first query row, tiles [tile, tile + tiles) of the unit's; share -1: none
};
struct SeqWork { TreeSeq q; int units, tiles; };       // units of a sequence (0: none, or its numbers are wrong), tiles of keys of each
__device__ __forceinline__ int pieces_of(int tiles, int per) { return (tiles + per - 1) / per; }
__device__ __forceinline__ int warp_scan(int x, int lane) {                    // inclusive
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, i); if (lane >= i) x += y; }
    return x;
}
// The CTA's piece, by one warp (x->s -1: none); CTA 0 writes the plan down.
// A piece is at most `per` tiles long.  Where there are fewer units than CTAs that run at once, the pieces should be as many as those, nearly: the even share of all
// tiles, longer by what rounding up makes of it.  (Pieces are at most units + tiles / per, so the last choice always fits.)  But a piece costs tree_combine about a third
// of a tile's time (a 48th, of a tile on CUDA cores): n tiles in pieces of p take p + n / (3 p) tiles' time, least at p = sqrt(n / 3).  Measured with this bound /
// without, us: 1 K/V head of 4 query heads, a tree of 8 over 32000 rows 25 / 60, 2 of them over 40000 28 / 47.  Where there are more units, only one longer than twice the even
// share is cut.  Pieces twice to six times as many (for SMs that are faster than others) gained nothing: 284 to 345 us for 16 trees of 32 over up to 32768 rows, 268 so; nor
// did an order that puts long and short pieces together on an SM (271 / 272).  Short code: every CTA runs it once, cold.
__device__ __forceinline__ void piece_find(const TreeAttnArgs& a, const Share& p, int lane, Piece* x) {
    auto work = [&](int s) {
        SeqWork y{{}, 0, 1};
        if (s < a.t.n_seq && tree_seq(a.t, &a.m, s, &y.q, a.status)) {
            y.units = a.n_kv * ((y.q.n * (a.n_q / a.n_kv) + p.tile_rows - 1) / p.tile_rows);
            y.tiles = tree_work(y.q.prefix, y.q.n, a.window).n_tiles;
        }
        return y;
    };
    const SeqWork mine = work(lane);                 // (batches of up to 32 sequences: all there is)
    int units = mine.units, total = mine.units * mine.tiles, longest = mine.units ? mine.tiles : 0;             // (the call bounds them)
#pragma unroll 1
    for (int s0 = 32; s0 < a.t.n_seq; s0 += 32) { const SeqWork y = work(s0 + lane); units += y.units; total += y.units * y.tiles; longest = max(longest, y.units ? y.tiles : 0); }
    units = __reduce_add_sync(0xffffffffu, units);
    total = __reduce_add_sync(0xffffffffu, total);
    longest = __reduce_max_sync(0xffffffffu, longest);
    const int slots = p.slots;
    const float even = (float)total / (float)slots;
    int per = p.shares ? (int)(2.0f * even) + 2 : kNoCut;
    if (p.shares && units < slots) {
        per = max((int)even + 1, (int)sqrtf((float)longest * (a.kv_bf16 ? 1.0f / 3.0f : 1.0f / 48.0f)) + 1);
#pragma unroll 1
        for (int i = 0; i < 4; i++) {
            int n = mine.units * pieces_of(mine.tiles, per);
#pragma unroll 1
            for (int s0 = 32; s0 < a.t.n_seq; s0 += 32) { const SeqWork y = work(s0 + lane); n += y.units * pieces_of(y.tiles, per); }
            n = __reduce_add_sync(0xffffffffu, n);
            if (n <= slots) break;
            per = i == 3 ? total / (slots - units) + 1 : (int)((float)per * (float)n / (float)slots) + 1;
        }
    }
    const bool plans = blockIdx.x == 0 && p.shares;  // (without shares nobody reads it)
    if (lane == 0) x->s = -1;
    __syncwarp();
    int before = 0, shares = 0;
#pragma unroll 1
    for (int s0 = 0; s0 < a.t.n_seq; s0 += 32) {
        const SeqWork y = s0 ? work(s0 + lane) : mine;
        const int k = pieces_of(y.tiles, per), n = y.units * k, sum = warp_scan(n, lane), cut = k > 1 ? n : 0, cuts = warp_scan(cut, lane);
        if (plans && s0 + lane < a.t.n_seq) p.plan[1 + s0 + lane] = shares + cuts - cut;
        const int at = (int)blockIdx.x - before - (sum - n);
        if (at >= 0 && at < n) {                     // (of all lanes and rounds, one)
            const int unit = at / k, i = at - unit * k, per_head = y.units / a.n_kv, least = y.tiles / k, more = y.tiles - least * k;
            x->q = y.q;
            x->w = tree_work(y.q.prefix, y.q.n, a.window);
            x->s = s0 + lane;
            x->kvh = unit / per_head;                // a K/V head's row tiles follow each other: their keys are in L2
            x->f0 = (unit - x->kvh * per_head) * p.tile_rows;
            x->tile = i * least + min(i, more);
            x->tiles = least + (i < more ? 1 : 0);
            x->share = k > 1 ? shares + cuts - cut + at : -1;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
        shares += __shfl_sync(0xffffffffu, cuts, 31);
        if (blockIdx.x && (int)blockIdx.x < before) break;
    }
    if (plans && lane == 0) p.plan[0] = shares ? per : kNoCut;
}

// The piece of a CTA of a cluster: its part of the unit's tiles (perhaps none).  By one thread.
__device__ __forceinline__ void piece_of_cluster(const TreeAttnArgs& a, const Share& p, Piece* x) {
    const int unit = (int)blockIdx.x / p.cluster, i = (int)blockIdx.x - unit * p.cluster, u = unit / p.row_tiles, s = u / a.n_kv, f0 = (unit - u * p.row_tiles) * p.tile_rows;
    const bool live = tree_seq(a.t, &a.m, s, &x->q, a.status) && f0 < x->q.n * (a.n_q / a.n_kv);
    x->w = tree_work(x->q.prefix, live ? x->q.n : 0, a.window);
    x->s = live ? s : -1;
    x->kvh = u - s * a.n_kv;
    x->f0 = f0;
    const int least = x->w.n_tiles / p.cluster, more = x->w.n_tiles - least * p.cluster;
    x->tile = i * least + min(i, more);
    x->tiles = least + (i < more ? 1 : 0);
    x->share = -1;
}

template <typename T> __device__ __forceinline__ T out_of(float x);
template <> __device__ __forceinline__ float out_of<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 out_of<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }      // the one rounding of the result

// x / sum; a sum that is not positive is undefined: a row all of whose visible scores are -inf is 0 / 0 (a finite score adds 1 to its row's sum, or a share that is
// scaled against one that has)
__device__ __forceinline__ float tree_ratio(float x, float sum) { return sum > 0.0f ? x / sum : __int_as_float(0x7fffffff); }
// What a share (maximum m, sum l) of a row weighs against the row's maximum; a share with no score above -inf weighs nothing, undefined sums stay undefined.
__device__ __forceinline__ float share_factor(float m, float l, float top) { return l != l ? 1.0f : m == -INFINITY ? 0.0f : m == top ? 1.0f : exp2f(m - top); }
// What a sink adds to the sum against the maximum `top`, which is not below it: nothing where it is -inf, 1 where it is the maximum (+inf leaves nothing to the keys).
__device__ __forceinline__ float sink_part(float sink, float top) { return sink == -INFINITY ? 0.0f : sink == top ? 1.0f : exp2f(sink - top); }
// The factor of a finished row: out = o / l, with the sink's part in l.
__device__ __forceinline__ float tree_inverse(const TreeAttnArgs& a, int h, float m, float l) {
    if (!a.sinks) return tree_ratio(1.0f, l);
    const float sink = a.sinks[h] * kLog2e, top = fmaxf(m, sink), c = share_factor(m, l, top);
    return tree_ratio(c, fmaf(l, c, sink_part(sink, top)));
}

__device__ __forceinline__ float2 cluster_ld2(uint32_t at) { float2 v; asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory"); return v; }
__device__ __forceinline__ float4 cluster_ld4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}
// The unit's rows are shared out among the warps of the cluster, which join the CTAs' shares of them: o_at(r) and ml_at(r) are where a CTA has its outputs and (maximum, sum).
template <int HD, typename TQ, typename At, typename MlAt>
__device__ __forceinline__ void join_cluster(const TreeAttnArgs& a, const Share& p, const Piece& x, int live_rows, int warp, int warps, int lane, At o_at, MlAt ml_at) {
    using V = typename std::conditional<HD == 128, float4, float2>::type;
    const int C = p.cluster, rank = (int)blockIdx.x % C, G = a.n_q / a.n_kv;
    __syncwarp();
    cluster_arrive_release();
    cluster_wait_acquire();
    for (int r = rank + C * warp; r < live_rows; r += C * warps) {
        const int node = (x.f0 + r) / G, h = x.kvh * G + (x.f0 + r) - node * G;
        float2 ml[kClusterMax];
        V y[kClusterMax];
#pragma unroll
        for (int c = 0; c < kClusterMax; c++) {                      // all on their way at once
            ml[c] = make_float2(-INFINITY, 0.0f);
            if (c < C) {
                ml[c] = cluster_ld2(cluster_map(ml_at(r), (uint32_t)c));
                const uint32_t from = cluster_map(o_at(r) + (uint32_t)(lane * (HD / 32)) * 4u, (uint32_t)c);
                if constexpr (HD == 128) y[c] = cluster_ld4(from); else y[c] = cluster_ld2(from);
            }
        }
        const float sink = a.sinks ? a.sinks[h] * kLog2e : -INFINITY;
        float top = sink, z[HD / 32];
#pragma unroll
        for (int c = 0; c < kClusterMax; c++) top = fmaxf(top, ml[c].x);
        float sum = sink_part(sink, top);
#pragma unroll
        for (int i = 0; i < HD / 32; i++) z[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < kClusterMax; c++) {
            if (c >= C) continue;
            const float f = share_factor(ml[c].x, ml[c].y, top);
            const float* part_of = (const float*)&y[c];
            sum = fmaf(ml[c].y, f, sum);
#pragma unroll
            for (int i = 0; i < HD / 32; i++) z[i] = fmaf(part_of[i], f, z[i]);
        }
        const float inv = tree_ratio(1.0f, sum);
        TQ* dst = (TQ*)a.out + (size_t)(x.q.r0 + node) * a.out_stride + (size_t)h * HD + lane * (HD / 32);
#pragma unroll
        for (int i = 0; i < HD / 32; i++) dst[i] = out_of<TQ>(z[i] * inv);
    }
    __syncwarp();
    cluster_arrive_release();                        // nobody leaves while another may read its shares
    cluster_wait_acquire();
}

// Pairs of floats in 64-bit registers, whose operations issue once for two.
using F2 = unsigned long long;
__device__ __forceinline__ F2 pack2(float a, float b) { F2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float2 unpack2(F2 x) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x)); return r; }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) { F2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ F2 add2(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

// ---- products on CUDA cores, in 32 bits: an f32 cache
// A unit has 32 query rows; 8 warps of 4 query rows.  A tile of 64 keys lies in shared memory as f32: a lane multiplies two keys with the warp's four rows, and then four
// (two) dimensions of the values with their weights.  Bound by what is read from shared memory: every warp reads all keys and values.  8 trees of 8 nodes over 4000 rows, 8 K/V
// heads of 4 query heads of 128 (8.4 GFLOP): 208 us, 40 TFLOP/s; with one key a lane and no pairs 291.  4 trees of 47 over 7030 rows, 2 K/V heads of 7 query heads (9.5 GFLOP): 442 us, 21
// TFLOP/s.  Shared memory's data pipe is 63 to 70 % busy, issue 40 %.
constexpr int kRowsTile = 32, kRowsKeys = kTileKeys;
template <int HD>
constexpr int rows_smem() { return (kRowsTile * HD + kRowsKeys * (HD + 4) + kRowsKeys * HD + 2 * kRowsTile * kRowsKeys) * 4 + (int)sizeof(Piece) + (int)sizeof(TreeNodes); }

template <int HD>
__global__ void __launch_bounds__(256, 2) attn_tree_rows(const TreeAttnArgs a, const Share part) {
    extern __shared__ __align__(16) unsigned char smem[];
    float* s_q = (float*)smem;                       // [32][HD]
    float* s_k = s_q + kRowsTile * HD;               // [64][HD + 4]
    float* s_v = s_k + kRowsKeys * (HD + 4);         // [64][HD]
    float* s_p = s_v + kRowsKeys * HD;               // [8 warps][64 keys][4 rows], each weight twice
    Piece* s_piece = (Piece*)(s_p + 2 * kRowsTile * kRowsKeys);
    TreeNodes& tree = *(TreeNodes*)(s_piece + 1);
    constexpr int DPL = HD / 32, PPL = DPL / 2;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = a.n_q / a.n_kv;
    if (part.cluster > 1) { if (tid == 0) piece_of_cluster(a, part, s_piece); }
    else if (warp == 0) piece_find(a, part, lane, s_piece);
    __syncthreads();
    if (s_piece->s < 0) return;
    const Piece x = *s_piece;
    const bool clustered = part.cluster > 1;
    const float scale = a.scale * kLog2e;
    {
        const TreeSeq& q = x.q;
        const TreeWork& w = x.w;
        tree_load(tree, a.t, q, a.window, tid, 256, 0, a.status);
        for (int e = tid; e < kRowsTile * HD / 4; e += 256) {
            const int r = e / (HD / 4), c = e % (HD / 4) * 4, f = x.f0 + r;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (f < q.n * G) v = *(const float4*)((const float*)a.q + (size_t)(q.r0 + f / G) * a.q_stride + ((size_t)x.kvh * G + f % G) * HD + c);
            *(float4*)(s_q + r * HD + c) = v;
        }
        F2 o[4][PPL];
        float mx[4], l[4];
        int node[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            mx[r] = -INFINITY; l[r] = 0.0f;
            const int f = x.f0 + warp * 4 + r;
            node[r] = f < q.n * G ? f / G : -1;
#pragma unroll
            for (int i = 0; i < PPL; i++) o[r][i] = 0ull;
        }
        const int j_first = (w.t_lo + x.tile) * kTileKeys, j_end = min(w.n_keys, j_first + x.tiles * kTileKeys);
#pragma unroll 1
        for (int j0 = j_first; j0 < j_end; j0 += kRowsKeys) {
            __syncthreads();                         // (the tree and the queries are there; the tile before has been read)
            constexpr int kStep = 256 / (HD / 4), kBatch = 4;        // a thread has one column of every kStep-th row
            const int col = tid % (HD / 4) * 4;
            float odd = 0.0f;                        // 0, or NaN where a value is not finite
#pragma unroll 1
            for (int r0 = tid / (HD / 4); r0 < kRowsKeys; r0 += kStep * kBatch) {
                float4 kf[kBatch], vf[kBatch];
#pragma unroll
                for (int u = 0; u < kBatch; u++) {
                    const int j = j0 + r0 + u * kStep;
                    const long long at = j >= w.low && j < j_end ? tree_row(a.m, q.slot, j, a.status) : -1;
                    kf[u] = vf[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (at >= 0) {
                        const size_t off = (size_t)at * a.kv_stride + (size_t)x.kvh * HD + col;
                        kf[u] = *(const float4*)((const float*)a.k + off);
                        vf[u] = *(const float4*)((const float*)a.v + off);
                    }
                }
#pragma unroll
                for (int u = 0; u < kBatch; u++) {
                    *(float4*)(s_k + (r0 + u * kStep) * (HD + 4) + col) = kf[u];
                    *(float4*)(s_v + (r0 + u * kStep) * HD + col) = vf[u];
                    odd = fmaf(vf[u].x, 0.0f, fmaf(vf[u].y, 0.0f, fmaf(vf[u].z, 0.0f, fmaf(vf[u].w, 0.0f, odd))));
                }
            }
            const bool finite = !__syncthreads_or(odd != 0.0f);
            F2 y[2][4];
#pragma unroll
            for (int r = 0; r < 4; r++) y[0][r] = y[1][r] = 0ull;
            const float* qr = s_q + warp * 4 * HD;
#pragma unroll 4
            for (int c = 0; c < HD; c += 4) {
                const ulonglong2 ka = *(const ulonglong2*)(s_k + lane * (HD + 4) + c), kb = *(const ulonglong2*)(s_k + (lane + 32) * (HD + 4) + c);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const ulonglong2 q4 = *(const ulonglong2*)(qr + r * HD + c);
                    y[0][r] = fma2(q4.y, ka.y, fma2(q4.x, ka.x, y[0][r]));
                    y[1][r] = fma2(q4.y, kb.y, fma2(q4.x, kb.x, y[1][r]));
                }
            }
            unsigned int vis[2][4], all = 0xffffffffu;
            float pr[2][4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float z[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int j = j0 + lane + 32 * h;
                    const bool see = j >= w.low && j < j_end && node[r] >= 0 && tree_sees(tree, q, a.window, node[r], j);
                    vis[h][r] = __ballot_sync(0xffffffffu, see);
                    all &= vis[h][r];
                    const float2 t = unpack2(y[h][r]);
                    z[h] = see ? (t.x + t.y) * scale : -INFINITY;
                }
                float top = fmaxf(z[0], z[1]);
#pragma unroll
                for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
                const float mn = fmaxf(mx[r], top), off = mn == -INFINITY ? 0.0f : mn;
#pragma unroll
                for (int h = 0; h < 2; h++) pr[h][r] = vis[h][r] >> lane & 1u ? exp2f(z[h] - off) : 0.0f;
                const float corr = mx[r] == mn ? 1.0f : exp2f(mx[r] - mn);
                l[r] = l[r] * corr + (pr[0][r] + pr[1][r]);
                mx[r] = mn;
                const F2 corr2 = pack2(corr, corr);
#pragma unroll
                for (int i = 0; i < PPL; i++) o[r][i] = mul2(o[r][i], corr2);
            }
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int r = 0; r < 4; r += 2)
                    *(float4*)(s_p + ((warp * kRowsKeys + lane + 32 * h) * 4 + r) * 2) = make_float4(pr[h][r], pr[h][r], pr[h][r + 1], pr[h][r + 1]);
            __syncwarp();
            using V = typename std::conditional<HD == 128, ulonglong2, F2>::type;
            const float *pw = s_p + warp * kRowsKeys * 8, *vl = s_v + lane * DPL;
            if (finite || all == 0xffffffffu) {      // (keys that a row does not see have weight 0)
#pragma unroll 8
                for (int key = 0; key < kRowsKeys; key++) {
                    const V v = *(const V*)(vl + key * HD);
                    const ulonglong2 p01 = *(const ulonglong2*)(pw + key * 8), p23 = *(const ulonglong2*)(pw + key * 8 + 4);
                    const F2 p2[4] = {p01.x, p01.y, p23.x, p23.y};
#pragma unroll
                    for (int r = 0; r < 4; r++)
#pragma unroll
                        for (int i = 0; i < PPL; i++) o[r][i] = fma2(p2[r], ((const F2*)&v)[i], o[r][i]);
                }
            } else {
                // but 0 times infinity is no zero
#pragma unroll 1
                for (int key = 0; key < kRowsKeys; key++) {
                    const V v = *(const V*)(vl + key * HD);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        if ((key < 32 ? vis[0][r] : vis[1][r]) >> (key & 31) & 1u) {
                            const F2 p2 = *(const F2*)(pw + key * 8 + 2 * r);
#pragma unroll
                            for (int i = 0; i < PPL; i++) o[r][i] = fma2(p2, ((const F2*)&v)[i], o[r][i]);
                        }
                    }
                }
            }
            __syncwarp();
        }
        float out[4][DPL];
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int i = 0; i < PPL; i++) { const float2 t = unpack2(o[r][i]); out[r][2 * i] = t.x; out[r][2 * i + 1] = t.y; }
        if (clustered) __syncthreads();              // (a CTA without a tile: the queries are there, which a share takes the place of)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if (node[r] < 0) continue;
            const int row = q.r0 + node[r], h = x.kvh * G + (x.f0 + warp * 4 + r) % G;
            const float sum = warp_sum(l[r]);
            if (clustered || x.share >= 0) {
                const size_t at = share_at(part, max(x.share, 0), warp * 4 + r);
                float *o_to = clustered ? s_q + (warp * 4 + r) * HD : part.o + at * HD, *ml_to = clustered ? s_p + (warp * kRowsKeys * 4 + r) * 2 : part.ml + 2 * at;      // (this warp's own)
#pragma unroll
                for (int i = 0; i < DPL; i++) o_to[lane * DPL + i] = out[r][i];
                if (lane == 0) { ml_to[0] = mx[r]; ml_to[1] = sum; }
            } else {
                const float inv = tree_inverse(a, h, mx[r], sum);
                float* dst = (float*)a.out + (size_t)row * a.out_stride + (size_t)h * HD + lane * DPL;
#pragma unroll
                for (int i = 0; i < DPL; i++) dst[i] = out[r][i] * inv;
            }
        }
        if (clustered)
            join_cluster<HD, float>(a, part, x, min(kRowsTile, q.n * G - x.f0), warp, 8, lane, [&](int r) { return smem_u32(s_q + r * HD); },
                                    [&](int r) { return smem_u32(s_p + ((r >> 2) * kRowsKeys * 4 + (r & 3)) * 2); });
    }
}

// ---- products on the tensor core (tcgen05): a bf16 cache
// Four softmax warps, a thread per query row; one warp that asks for keys, one for values, one that issues the products (and asks for bf16 queries: a copy per 64
// dimensions brings a unit's rows as the operand wants them).  Per tile of 64 cache rows:
//     S = Q K^T             M 128, N 64; Q in shared memory, one bf16 term (bf16 queries) or three (f32 queries, 24 bits)
//     p = 2^(S - m)         a thread reads its row's 64 scores, masks, exponentiates, and stores the weights' terms over them
//     O (+)= P V            M 128, N head_dim; P from tensor memory, V as stored (MN-major)
// Up to 64 (32) query rows lie in the operand two (four) times: copy c takes the softmax of every tile's c-th half (quarter) of the keys, with zeros as the weights of the
// others, and the copies are joined at the end, so that all four warps have work whatever the rows.
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
// What bounds it, and what it measured (20 passes in a graph over the same data, SM clock 1.9 GHz): 16 trees of 32 nodes over up to 32768 rows in pages of 16, 8 K/V heads of 4 query
// heads of 128 (1.28 GB): 268 us, 4.8 TB/s; with more products per byte than HBM alone would let them wait for, it slows down with the SMs' clock: 327 us, 3.9 TB/s, in calls that
// go on for a second, which are held to 1.1 - 1.4 GHz.  8 trees of 64 over 4096 rows, 8 query heads of 64 per K/V head (34.6 GFLOP): 82 us, 420 TFLOP/s; bound by the softmax warps (ALU and exponentials busy half of the
// time each, issue 46 %).  32 trees of up to 16 over up to 2048 rows (0.18 GB): 50 us, 3.6 TB/s (56 where nothing is in L2), of which launch, first tiles and joining are 15.
// f32 queries, whose terms leave room for one CTA an SM with heads of 128 and whose outputs pass through registers every tile: 8 trees of 64 over 4096 rows, 4 query heads of 128 per
// K/V head 108 us where bf16 queries take 63 (tensor pipe 43 %, issue 35 %), 32 of up to 16 over up to 2048 88 / 50, 16 of 32 over up to 32768 581 / 268.  Tried without gain: two
// threads per query row (104 us to 107 where this came to 104), weights by the maximum of the tile before with a second try where it grew (112), room for four tiles
// (n_seq 1 .. 8 with 4000 .. 16000 rows: 13.9 / 14.1, 27.8 / 29.7, 36.4 / 32.2, 25.1 / 37.0: with that much shared memory clusters no longer fit beside one another).
constexpr int kTcGroup = 128 * 16 + 16;              // f32 queries' terms: 16-byte column groups of 128 rows, the next one 16 bytes further on (banks)
constexpr int kTcThreads = 224;                     // four softmax warps, keys, products, values
template <int HD, bool F32>
struct TcShape {
    static constexpr int q_terms = F32 ? 3 : 1, p_terms = F32 ? 3 : 2;
    static constexpr int tile = kTileKeys * HD * 2;  // bytes of K (or V)
    static constexpr int q_bytes = F32 ? HD / 8 * kTcGroup : 128 * HD * 2;
    static constexpr int off_k = 0, off_v = 2 * tile, off_q = 4 * tile, off_misc = off_q + q_terms * q_bytes, off_tree = off_misc + 112 + (int)sizeof(Piece);
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
// N consecutive 32-bit columns of this thread's lane of tensor memory, by a whole warp
template <int N> __device__ __forceinline__ void tc_ld(uint32_t at, uint32_t* v);
template <int N> __device__ __forceinline__ void tc_st(uint32_t at, const uint32_t* v);
template <> __device__ __forceinline__ void tc_ld<16>(uint32_t at, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(at) : "memory");
}
template <> __device__ __forceinline__ void tc_ld<32>(uint32_t at, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(at) : "memory");
}
template <> __device__ __forceinline__ void tc_st<8>(uint32_t at, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
template <> __device__ __forceinline__ void tc_st<32>(uint32_t at, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
                 : "memory");
}
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// (passes over NaN as fmaxf does)
__device__ __forceinline__ float max3(float a, float b, float c) { float r; asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
__device__ __forceinline__ float tc_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// x as packed bf16, rounded; what is left of it goes back, by additions that take a bf16 operand as it is (8 trees of 64 nodes over 4096 rows 81.8 us; with the terms made f32
// again 84.3)
__device__ __forceinline__ uint32_t tc_term(float* x0, float* x1) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(*x0, *x1);
    const uint32_t b = *(const uint32_t*)&h;
    asm("{\n\t.reg .b16 lo, hi, m;\n\tmov.b32 {lo, hi}, %2;\n\tmov.b16 m, 0xBF80;\n\tfma.rn.f32.bf16 %0, lo, m, %0;\n\tfma.rn.f32.bf16 %1, hi, m, %1;\n\t}" : "+f"(*x0), "+f"(*x1) : "r"(b));      // m: -1
    return b;
}
__device__ __forceinline__ uint32_t tc_term(F2* x) {
    float2 y = unpack2(*x);
    const uint32_t b = tc_term(&y.x, &y.y);
    *x = pack2(y.x, y.y);
    return b;
}
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int row, int col, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(0), "r"(row), "r"(col), "r"(bar) : "memory");
}

__device__ __forceinline__ void tma_queries(uint32_t dst, const CUtensorMap* map, int head, int row, int half, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map), "r"(0), "r"(head), "r"(row), "r"(half),
                 "r"(bar) : "memory");
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
        const size_t off = (size_t)max(at, 0ll) * a.kv_stride + (size_t)kvh * HD + lane * DPL;
        float d = 0.0f, v[DPL];
#pragma unroll
        for (int i = 0; i < DPL; i++) {                              // (the rows of an unknown page are zeros)
            d = fmaf(x[i], at >= 0 ? __bfloat162float(((const __nv_bfloat16*)a.k)[off + i]) : 0.0f, d);
            v[i] = at >= 0 ? __bfloat162float(((const __nv_bfloat16*)a.v)[off + i]) : 0.0f;
        }
        d = warp_sum(d) * scale;
        const float mn = fmaxf(mx, d), c = mx == mn ? 1.0f : exp2f(mx - mn), p = exp2f(d - (mn == -INFINITY ? 0.0f : mn));
        sum = sum * c + p;
#pragma unroll
        for (int i = 0; i < DPL; i++) o[i] = fmaf(p, v[i], o[i] * c);
        mx = mn;
    }
    *m = mx; *l = sum;
#pragma unroll
    for (int i = 0; i < DPL; i++) out[i] = o[i];
}
template <int HD, bool F32, int DUP>
__global__ void __launch_bounds__(kTcThreads, TcShape<HD, F32>::ctas) attn_tree_tc(const __grid_constant__ TreeAttnArgs a, const __grid_constant__ Share part, const __grid_constant__ CUtensorMap map_q,
                                                                                   const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, int box_rows) {
    using S = TcShape<HD, F32>;
    using TQ = typename std::conditional<F32, float, __nv_bfloat16>::type;
    extern __shared__ __align__(1024) unsigned char tc_smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = a.n_q / a.n_kv;
    const uint32_t base = smem_u32(tc_smem), misc = base + S::off_misc;
    const uint32_t bar_k = misc, bar_v = misc + 16, bar_s = misc + 32, bar_p = misc + 48, bar_o = misc + 64, bar_q = misc + 80;      // two of each (queries: one): tile t uses number t % 2
    volatile int* gave_up = (volatile int*)(tc_smem + S::off_misc + 104);
    Piece* s_piece = (Piece*)(tc_smem + S::off_misc + 112);
    TreeNodes& tree = *(TreeNodes*)(tc_smem + S::off_tree);
    pdl_launch_dependents();                         // (tree_combine waits for this kernel's end)
    if (tid == 32) {
        for (int i = 0; i < 2; i++) {
            mbar_init(bar_k + 8 * i, 1);             // K(t) has landed
            mbar_init(bar_v + 8 * i, 1);             // V(t)
            mbar_init(bar_s + 8 * i, 1);             // S(t) is there, K(t) is no longer read
            mbar_init(bar_p + 8 * i, 4);             // P(t) is stored, O may be added to
            mbar_init(bar_o + 8 * i, 1);             // O holds tile t, V(t) is no longer read
        }
        mbar_init(bar_q, F32 ? 4 : 1);               // the queries are there
        mbar_fence_init();
        *gave_up = 0;
    }
    if (part.cluster > 1) { if (tid == 0) piece_of_cluster(a, part, s_piece); }
    else if (warp == 0) piece_find(a, part, lane, s_piece);
    if (warp == 5) tmem_alloc(misc + 96, S::cols);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *(volatile uint32_t*)(tc_smem + S::off_misc + 96);
    if (s_piece->s < 0) {
        if (warp == 5) tmem_dealloc(tmem, S::cols);
        return;
    }
    const Piece x = *s_piece;
    const TreeSeq q = x.q;
    const TreeWork w = x.w;
    const int t_first = w.t_lo + x.tile, n_tiles = x.tiles, kvh = x.kvh, f0 = x.f0, live_rows = min(part.tile_rows, q.n * G - f0);
    const bool clustered = part.cluster > 1;
    // Room of the tiles and queries behind the last product: copies' outputs and (maximum, sum), then a cluster's
    constexpr int kLd = HD + 4, kCopyRows = 128 / DUP;
    constexpr int off_copy_ml = (DUP - 1) * kCopyRows * kLd * 4, off_share = DUP > 1 ? off_copy_ml + 1024 : 0, off_share_ml = off_share + kCopyRows * kLd * 4;
    static_assert(off_share_ml + kCopyRows * 8 <= S::off_misc, "fits");
    float *c_o = (float*)(tc_smem + off_share), *c_ml = (float*)(tc_smem + off_share_ml);      // [row][kLd], [row][2]

    // A wait that runs out of its budget is remembered; what follows hardly waits and multiplies no more, but meets every barrier.
    auto wait = [&](uint32_t bar, int t) {
        const uint32_t at = bar + 8u * (t & 1), parity = (uint32_t)(t >> 1) & 1u;
        if (mbar_try_wait(at, parity)) return;
        if (!mbar_wait_abortable(at, parity, gave_up)) *gave_up = 1;
    };
    constexpr int kHalves = HD / 64;
    if (warp == 4 || warp == 6) {
        // ---- keys (warp 4) or values (warp 6): K(t + 2) goes out when S(t) is there, V(t + 2) when O holds tile t
        const bool keys = warp == 4;
        const CUtensorMap* map = keys ? &map_k : &map_v;
        const uint32_t dst0 = base + (keys ? S::off_k : S::off_v), full = keys ? bar_k : bar_v, used = keys ? bar_s : bar_o;
        int last = -1;
        // Where this lane's box of tile t starts in the cache (a lane per box; a box of a whole tile is every lane's, whichever is elected to ask for it); a
        // page-table entry is on its way while the tile before is waited for.
        const int boxes = kTileKeys / box_rows, box = boxes == 1 ? 0 : lane;
        auto box_row = [&](int t) {
            const int j = (t_first + t) * kTileKeys + box * box_rows;
            if (t >= n_tiles || box >= boxes || j >= w.n_keys || j + box_rows <= w.low) return (int)a.m.rows;     // outside the tensor: zeros
            const long long row = tree_row(a.m, q.slot, j, a.status);
            return (int)(row < 0 ? a.m.rows : row);
        };
        int next = box_row(0);
        for (int t = 0; t < n_tiles; t++) {
            const int row = next;
            next = box_row(t + 1);
            if (t > 1) wait(used, t - 2);
            if (__any_sync(0xffffffffu, *gave_up)) break;
            const uint32_t bar = full + 8u * (t & 1), dst = dst0 + (uint32_t)(t & 1) * S::tile;
            if (lane == 0) mbar_arrive_expect_tx(bar, S::tile);
            __syncwarp();
            // a box holds its halves of 64 dimensions one behind the other; a whole tile's are kTileKeys rows apart
            if (box_rows == kTileKeys) { if (elect_one()) tma_box(dst, map, row, kvh * kHalves, bar); }
            else if (lane < boxes)
#pragma unroll
                for (int h = 0; h < kHalves; h++) tma_box(dst + h * (kTileKeys * 128) + lane * box_rows * 128, map, row, kvh * kHalves + h, bar);
            last = t;
        }
        // no copy is on its way when the CTA ends (they have landed long ago, unless a wait was given up)
        for (int t = max(last - 1, 0); t <= last; t++) mbar_wait(full + 8u * (t & 1), (uint32_t)(t >> 1) & 1u);
    } else if (warp == 5) {
        // ---- the products (and the copy of bf16 queries: the unit's nodes, their heads of this K/V head, in the order of the operand's rows)
        constexpr uint32_t id_s = tc_idesc(kTileKeys, false), id_o = tc_idesc(HD, true);
        if (elect_one()) {
            if constexpr (!F32) {
                mbar_arrive_expect_tx(bar_q, (uint32_t)part.tile_rows * 128u * kHalves * DUP);
#pragma unroll
                for (int h = 0; h < kHalves; h++)
#pragma unroll
                    for (int d = 0; d < DUP; d++) tma_queries(base + S::off_q + h * (128 * 128) + d * (128 / DUP * 128), &map_q, kvh * G, q.r0 + f0 / G, h, bar_q);
            }
            wait(bar_q, 0);
#pragma unroll 1
            for (int t = 0; t <= n_tiles; t++) {
                if (t < n_tiles) {
                    const int b = t & 1;
                    wait(bar_k, t);
                    if (*gave_up) break;
                    tc_fence_after_sync();
                    const uint32_t kb = base + S::off_k + b * S::tile, d = tmem + (uint32_t)b * 64u;
#pragma unroll
                    for (int e = S::q_terms - 1; e >= 0; e--)
#pragma unroll
                        for (int ks = 0; ks < HD / 16; ks++)
                            tc_mma(d, F32 ? umma_smem_desc(base + S::off_q + e * S::q_bytes + ks * 2 * kTcGroup, kTcGroup, 128) : tc_desc_sw128(base + S::off_q + (ks >> 2) * (128 * 128) + (ks & 3) * 32, 16, 1024),
                                   tc_desc_sw128(kb + (ks >> 2) * (kTileKeys * 128) + (ks & 3) * 32, 16, 1024), id_s, e != S::q_terms - 1 || ks ? 1u : 0u);
                    umma_commit(bar_s + 8u * b);
                }
                if (t > 0) {
                    const int u = t - 1, b = u & 1;
                    wait(bar_v, u);
                    wait(bar_p, u);
                    if (*gave_up) break;
                    tc_fence_after_sync();
                    const uint32_t vb = base + S::off_v + b * S::tile, p = tmem + (uint32_t)b * 64u, px = tmem + S::col_x + (uint32_t)b * 32u, d = tmem + S::col_o;
#pragma unroll
                    for (int e = S::p_terms - 1; e >= 0; e--)
#pragma unroll
                        for (int ks = 0; ks < kTileKeys / 16; ks++)
                            tc_mma_ts(d, (e == 2 ? px : p + e * 32u) + ks * 8u, tc_desc_sw128(vb + ks * 2048, kTileKeys * 128, 1024), id_o, (!F32 && u) || e != S::p_terms - 1 || ks ? 1u : 0u);
                    umma_commit(bar_o + 8u * b);
                }
            }
            if constexpr (!F32) mbar_wait(bar_q, 0);     // (landed long ago, unless a wait was given up)
        }
        __syncwarp();
    } else {
        // ---- softmax
        constexpr int KPT = kTileKeys / DUP;         // keys per thread and tile
        const float scale = a.scale * kLog2e;
        const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
        const uint32_t magic = 0xffffffffu / (uint32_t)G + 1u;           // f / G = f magic / 2^32 for f < 2^18, 2 <= G <= 2^10
        auto node_of = [&](int f) { return G == 1 ? f : (int)__umulhi((uint32_t)f, magic); };
        if constexpr (F32) {                         // three terms of the queries (rows beyond the last one are left as they are: nobody reads what they make)
            constexpr int kPieces = HD / 8, kStep = 128 / kPieces, kAhead = 4;
            const int c = tid % kPieces;
            for (int r0 = tid / kPieces; r0 < live_rows; r0 += kStep * kAhead) {
                uint4 raw[kAhead][2];
#pragma unroll
                for (int u = 0; u < kAhead; u++) {
                    const int f = f0 + min(r0 + u * kStep, live_rows - 1), node = node_of(f);
                    const uint4* src = (const uint4*)((const float*)a.q + (size_t)(q.r0 + node) * a.q_stride + ((size_t)kvh * G + f - node * G) * HD + c * 8);
                    raw[u][0] = src[0]; raw[u][1] = src[1];
                }
#pragma unroll
                for (int u = 0; u < kAhead; u++) {
                    const int r = r0 + u * kStep;
                    if (r >= live_rows) break;
                    float* y = (float*)raw[u];
#pragma unroll
                    for (int e = 0; e < 3; e++) {
                        const uint4 t = make_uint4(tc_term(y, y + 1), tc_term(y + 2, y + 3), tc_term(y + 4, y + 5), tc_term(y + 6, y + 7));
#pragma unroll
                        for (int d = 0; d < DUP; d++) *(uint4*)(tc_smem + S::off_q + e * S::q_bytes + c * kTcGroup + (d * (128 / DUP) + r) * 16) = t;
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_q);
        }
        // the tree, where the piece reaches it (with a window every tile may be cut)
        if (a.window > 0 || (t_first + n_tiles) * kTileKeys > q.prefix) {
            tree_load(tree, a.t, q, a.window, tid, 128, 1, a.status);
            named_sync(1, 128);
        }
        const int grp = DUP == 1 ? 0 : warp / (4 / DUP), warp_row = warp % (4 / DUP) * 32, col = grp * KPT, row = warp_row + lane, f = f0 + row, node = row < live_rows ? node_of(f) : -1;
        const bool live = warp_row < live_rows;      // a warp without live rows leaves its rows of P as they are: nobody reads what they make
        float m_run = -INFINITY, l_run = 0.0f;
        float o[F32 ? HD : 1];
        if constexpr (F32)
#pragma unroll
            for (int i = 0; i < HD; i++) o[i] = 0.0f;
#pragma unroll 1
        for (int t = 0; t < n_tiles; t++) {
            const int b = t & 1, j0 = (t_first + t) * kTileKeys;
            if (t > 1) wait(bar_o, t - 2);           // (long there: every phase of bar_o is seen, and V(t - 2) has been used)
            if (j0 < w.low || j0 + kTileKeys > w.n_keys) {           // rows of V that no query row may see
                wait(bar_v, t);
                unsigned char* vb = tc_smem + S::off_v + b * S::tile;
                for (int e = tid; e < kTileKeys * (HD / 8); e += 128) {
                    const int j = e / (HD / 8), c = e % (HD / 8);
                    if (j0 + j < w.low || j0 + j >= w.n_keys) *(uint4*)(vb + (c >> 3) * (kTileKeys * 128) + j * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async_smem();
            }
            wait(bar_s, t);
            tc_fence_after_sync();
            if (live) {
                const uint32_t sc = mine + (uint32_t)b * 64u;
                float v[KPT];
#pragma unroll
                for (int c = 0; c < KPT; c += KPT < 32 ? KPT : 32) tc_ld<(KPT < 32 ? KPT : 32)>(sc + col + c, (uint32_t*)v + c);
                tmem_ld_wait();
                if (j0 + kTileKeys > q.prefix || a.window > 0) {     // some key may be out of some row's sight
                    unsigned long long see = 0ull;
                    if (node >= 0) {
                        const int cached = q.prefix - j0;            // keys of the tile before the tree
                        see = cached >= 64 ? ~0ull : cached > 0 ? (1ull << cached) - 1 : 0ull;
                        const int first = q.prefix + tree.depth[node] - a.window + 1 - j0;
                        if (a.window > 0 && first > 0) see = first >= 64 ? 0ull : see & (~0ull << first);
#pragma unroll
                        for (int k = 0; k < kTreeWords; k++) {       // nodes 32 k .. 32 k + 31 are the keys from 32 k + cached on
                            const int at = 32 * k + cached;
                            if (32 * k < q.n && at < 64 && at > -32) see |= at >= 0 ? (unsigned long long)tree.anc[node][k] << at : (unsigned long long)(tree.anc[node][k] >> -at);
                        }
                    }
                    see >>= col;
#pragma unroll
                    for (int i = 0; i < KPT; i++)
                        if (!((i < 32 ? (uint32_t)see : (uint32_t)(see >> 32)) >> (i & 31) & 1u)) v[i] = -INFINITY;
                }
                float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                for (int i = 4; i < KPT; i += 2) top[i >> 1 & 3] = max3(top[i >> 1 & 3], v[i], v[i + 1]);
                const float tm = node >= 0 ? fmaxf(max3(top[0], top[1], top[2]), top[3]) * scale : -INFINITY;
                // the reference of the exponents: kept while nothing is more than 2^8 times it
                const bool grows = tm > m_run + (F32 ? 0.0f : 8.0f) || m_run == -INFINITY;
                const float m_new = grows ? fmaxf(tm, m_run) : m_run;
                const float alpha = m_new == m_run ? 1.0f : tc_ex2(m_run - m_new);
                m_run = m_new;
                const float off = m_new == -INFINITY ? 0.0f : -m_new;
                // 16 keys at a time: their exponentials (one pipe) beside the terms of the 16 before (another), which go over the scores (the third one beside
                // them), zeros where the keys are another row's
                constexpr int kStep = 16, kCols = kStep / 2;
                F2 w2[2][kCols], sum[2] = {0ull, 0ull};
                const F2 scale2 = pack2(scale, scale), off2 = pack2(off, off);
#pragma unroll
                for (int c = 0; c <= KPT / kStep; c++) {
                    if (c < KPT / kStep) {
#pragma unroll
                        for (int i = 0; i < kCols; i++) {
                            const float2 y = unpack2(fma2(pack2(v[c * kStep + 2 * i], v[c * kStep + 2 * i + 1]), scale2, off2));
                            w2[c & 1][i] = pack2(tc_ex2(y.x), tc_ex2(y.y));
                        }
                    }
                    if (c > 0) {
#pragma unroll
                        for (int i = 0; i < kCols; i++) sum[i & 1] = add2(sum[i & 1], w2[(c - 1) & 1][i]);
#pragma unroll
                        for (int e = 0; e < S::p_terms; e++) {
                            uint32_t pk[kCols];
#pragma unroll
                            for (int i = 0; i < kCols; i++) pk[i] = tc_term(&w2[(c - 1) & 1][i]);
                            const uint32_t to = (e == 2 ? mine + S::col_x + (uint32_t)b * 32u : sc + e * 32u) + (c - 1) * kCols;
#pragma unroll
                            for (int d = 0; d < DUP; d++) {
                                uint32_t out[kCols];
#pragma unroll
                                for (int i = 0; i < kCols; i++) out[i] = DUP == 1 || d == grp ? pk[i] : 0u;
                                tc_st<kCols>(to + d * (KPT / 2), out);
                            }
                        }
                    }
                }
                const float2 sums = unpack2(add2(sum[0], sum[1]));
                l_run = l_run * alpha + (sums.x + sums.y);
                if (t > 0) {
                    if constexpr (F32) {         // O(t - 1) comes out before O(t) is made
                        wait(bar_o, t - 1);
                        tc_fence_after_sync();
#pragma unroll
                        for (int c = 0; c < HD / 32; c++) {
                            uint32_t y[32];
                            tc_ld<32>(mine + S::col_o + c * 32u, y);
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
                            tc_ld<32>(mine + S::col_o + c * 32u, y);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; i++) y[i] = __float_as_uint(__uint_as_float(y[i]) * alpha);
                            tc_st<32>(mine + S::col_o + c * 32u, y);
                        }
                    }
                }
                tc_st_wait();
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_p + 8u * b);
        }
        if (n_tiles > 1) wait(bar_o, n_tiles - 2);
        if (n_tiles > 0) wait(bar_o, n_tiles - 1);
        else wait(bar_q, 0);                         // (a cluster's CTA without a tile: the queries are there, nothing else comes)
        tc_fence_after_sync();
        auto outputs = [&](int c, uint32_t* y) {     // columns 32 c .. 32 c + 31 of this thread's row
            if (n_tiles > 0) {
                tc_ld<32>(mine + S::col_o + c * 32u, y);
                tmem_ld_wait();
            } else
#pragma unroll
                for (int i = 0; i < 32; i++) y[i] = 0u;
        };
        // ---- the row's other copies: (maximum, sum, outputs) of their keys, through the room of the tiles (all of them have been used)
        float *s_o = (float*)tc_smem, *s_ml = (float*)(tc_smem + off_copy_ml);         // [copy - 1][row][kLd], [copy][row][2]
        float f_own = 1.0f, f_other[DUP > 1 ? DUP - 1 : 1];
        if constexpr (DUP > 1) {
            if (live && grp > 0) {
                s_ml[2 * (grp * (128 / DUP) + row)] = m_run; s_ml[2 * (grp * (128 / DUP) + row) + 1] = l_run;
#pragma unroll (F32 ? HD / 32 : 1)
                for (int c = 0; c < HD / 32; c++) {
                    uint32_t y[32];
                    outputs(c, y);
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        float4 z = make_float4(__uint_as_float(y[i]), __uint_as_float(y[i + 1]), __uint_as_float(y[i + 2]), __uint_as_float(y[i + 3]));
                        if constexpr (F32) { z.x += o[c * 32 + i]; z.y += o[c * 32 + i + 1]; z.z += o[c * 32 + i + 2]; z.w += o[c * 32 + i + 3]; }
                        *(float4*)(s_o + ((grp - 1) * (128 / DUP) + row) * kLd + c * 32 + i) = z;
                    }
                }
            }
            named_sync(1, 128);
            if (live && grp == 0) {
                float top = m_run, m_g[DUP - 1], l_g[DUP - 1];
#pragma unroll
                for (int g = 0; g < DUP - 1; g++) {
                    m_g[g] = s_ml[2 * ((g + 1) * (128 / DUP) + row)]; l_g[g] = s_ml[2 * ((g + 1) * (128 / DUP) + row) + 1];
                    top = fmaxf(top, m_g[g]);
                }
                f_own = m_run == top ? 1.0f : exp2f(m_run - top);
                l_run *= f_own;
#pragma unroll
                for (int g = 0; g < DUP - 1; g++) { f_other[g] = m_g[g] == top ? 1.0f : exp2f(m_g[g] - top); l_run = fmaf(l_g[g], f_other[g], l_run); }
                m_run = top;
            }
        }
        // ---- out = O / l, or this piece's share
        const bool share = x.share >= 0;
        if (live && grp == 0) {
            const int h = kvh * G + (node >= 0 ? f - node * G : 0), out_row = q.r0 + max(node, 0);
            const float inv = !share && !clustered && node >= 0 ? tree_inverse(a, h, m_run, l_run) : 1.0f;
            float odd = l_run * 0.0f;            // 0, or NaN where something is not finite
            const size_t at = share_at(part, max(x.share, 0), row);
#pragma unroll (F32 ? HD / 32 : 1)                   // (code that runs once is fetched as it runs: short code is fast code)
            for (int c = 0; c < HD / 32; c++) {
                uint32_t y[32];
                outputs(c, y);
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    float z = __uint_as_float(y[i]);
                    if constexpr (F32) z += o[c * 32 + i];
                    if constexpr (DUP > 1) {
                        z *= f_own;
#pragma unroll
                        for (int g = 0; g < DUP - 1; g++) z = fmaf(s_o[(g * (128 / DUP) + row) * kLd + c * 32 + i], f_other[g], z);
                    }
                    odd = fmaf(z, 0.0f, odd);
                    y[i] = __float_as_uint(z * inv);
                }
                if (node >= 0) {
                    if (share || clustered) {
                        float* to = clustered ? c_o + row * kLd : part.o + at * HD;
#pragma unroll
                        for (int i = 0; i < 32; i += 4) *(uint4*)(to + c * 32 + i) = make_uint4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                    } else {
                        TQ* dst = (TQ*)a.out + (size_t)out_row * a.out_stride + (size_t)h * HD + c * 32;
                        if constexpr (F32) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4) *(uint4*)(dst + i) = make_uint4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i += 8) {
                                uint32_t r[4];
#pragma unroll
                                for (int e = 0; e < 4; e++) {        // the one rounding of the result
                                    const __nv_bfloat162 z = __floats2bfloat162_rn(__uint_as_float(y[i + 2 * e]), __uint_as_float(y[i + 2 * e + 1]));
                                    r[e] = *(const uint32_t*)&z;
                                }
                                *(uint4*)(dst + i) = make_uint4(r[0], r[1], r[2], r[3]);
                            }
                        }
                    }
                }
            }
            if ((share || clustered) && node >= 0) *(float2*)(clustered ? c_ml + 2 * row : part.ml + 2 * at) = make_float2(m_run, l_run);
            __syncwarp();                            // (before another lane writes a row's share once more)
            // rows that are not finite, once more and key by key
            unsigned int bad = __ballot_sync(0xffffffffu, node >= 0 && odd != 0.0f && !*gave_up);
            const int j_first = max(t_first * kTileKeys, w.low), j_end = min(w.n_keys, (t_first + n_tiles) * kTileKeys);
            for (; bad; bad &= bad - 1) {
                const int r = warp_row + __ffs(bad) - 1, fr = f0 + r, nr = node_of(fr), hr = kvh * G + fr - nr * G;
                float m, l, z[HD / 32];
                tree_row_plain<HD, TQ>(a, tree, q, kvh, fr, j_first, j_end, lane, &m, &l, z);
                if (share || clustered) {
                    const size_t to = share_at(part, max(x.share, 0), r);
                    float* z_to = clustered ? c_o + r * kLd : part.o + to * HD;
                    for (int i = 0; i < HD / 32; i++) z_to[lane * (HD / 32) + i] = z[i];
                    if (lane == 0) *(float2*)(clustered ? c_ml + 2 * r : part.ml + 2 * to) = make_float2(m, l);
                } else {
                    const float c = tree_inverse(a, hr, m, l);
                    TQ* dst = (TQ*)a.out + (size_t)(q.r0 + nr) * a.out_stride + (size_t)hr * HD + lane * (HD / 32);
                    for (int i = 0; i < HD / 32; i++) dst[i] = out_of<TQ>(z[i] * c);
                }
            }
        }
        tc_fence_before_sync();
    }
    if (clustered)
        join_cluster<HD, TQ>(a, part, x, live_rows, warp, kTcThreads / 32, lane, [&](int r) { return smem_u32(c_o + r * kLd); }, [&](int r) { return smem_u32(c_ml + 2 * r); });
    __syncthreads();
    if (warp == 5) tmem_dealloc(tmem, S::cols);
    if (tid == 0 && *gave_up) atomicOr(a.status, LUM_ST_WAIT_TMEM);
}

// ---- joins the shares of units that were cut: a warp per (row, head); o = sum_c 2^(m_c - M) o_c / (sum_c 2^(m_c - M) l_c + 2^(sink - M)).  Most warps of a batch find
// that their unit was not cut, so what counts is how soon they know: no more than two rounds of CTAs, which end at once where nothing was cut
// (8 trees of 64 nodes over 4096 rows, none cut, 84 us, with a CTA for every eight results 89; 64 of 32 over 1000, 71 and 83).
template <int HD, typename TQ>
__global__ void __launch_bounds__(256, kJoinCtas) tree_combine(const TreeAttnArgs a, const Share part) {
    constexpr int DPL = HD / 32;
    const int lane = threadIdx.x & 31, G = a.n_q / a.n_kv, blocks = (a.n_q + 7) >> 3;
    const unsigned int items = (unsigned)a.t.n_rows * (unsigned)blocks;      // (below 2^31)
    int per = 0;
#pragma unroll 1
    for (unsigned int item = blockIdx.x; item < items; item += gridDim.x) {
        const int row = (int)(item / (unsigned)blocks), h = ((int)item - row * blocks) * 8 + (threadIdx.x >> 5);
        // the row's sequence: the last one that starts at or before it, 32 at a time
        int s = 0;
        for (int len = a.t.n_seq; len > 1;) {
            const int step = (len + 31) >> 5, at = lane * step;
            const unsigned int m = __ballot_sync(0xffffffffu, at < len && __ldg(a.t.row_start + s + min(at, len - 1)) <= row);
            const int k = m ? 31 - __clz(m) : 0;
            s += k * step;
            len = min(step, len - k * step);
        }
        TreeSeq q;
        const bool mine = h < a.n_q && tree_seq(a.t, &a.m, s, &q, nullptr) && row >= q.r0 && row < q.r0 + q.n;
        if (!per) pdl_grid_wait();                   // (what comes before does not depend on the kernel before; every warp waits, so that this kernel ends behind that one)
        per = __ldcg(part.plan);
        const int first_of_seq = __ldcg(part.plan + 1 + s);
        if (per == kNoCut) return;
        if (!mine) continue;
        const int shares = pieces_of(tree_work(q.prefix, q.n, a.window).n_tiles, per);
        if (shares == 1) continue;                       // finished by its CTA
        const int f = (row - q.r0) * G + h % G, R = part.tile_rows, first = first_of_seq + (h / G * ((q.n * G + R - 1) / R) + f / R) * shares, r = f % R;
        const float sink = a.sinks ? a.sinks[h] * kLog2e : -INFINITY;
        float top = sink, sum = sink_part(sink, sink), o[DPL];
#pragma unroll
        for (int i = 0; i < DPL; i++) o[i] = 0.0f;
        // 32 shares at a time: a lane has the factor of one, all have their dimensions of each, four on their way
        for (int c0 = 0; c0 < shares; c0 += 32) {
            float m = -INFINITY, l = 0.0f;
            if (c0 + lane < shares) {
                const float2 v = __ldcg((const float2*)part.ml + share_at(part, first + c0 + lane, r));
                m = v.x; l = v.y;
            }
            const int n = min(32, shares - c0);
            using V = typename std::conditional<DPL == 4, float4, float2>::type;
            V y[4];
            auto fetch = [&](int c) {
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (c + u < n) y[u] = __ldcg((const V*)(part.o + share_at(part, first + c0 + c + u, r) * HD) + lane);
            };
            fetch(0);
            float t = fmaxf(top, m);
#pragma unroll
            for (int i = 16; i > 0; i >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, i));
            const float before = top == t ? 1.0f : exp2f(top - t);
            const float factor = share_factor(m, l, t);
            sum = sum * before + warp_sum(l * factor);
            top = t;
#pragma unroll
            for (int i = 0; i < DPL; i++) o[i] *= before;
            for (int c = 0; c < n; c += 4) {
                if (c) fetch(c);
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const float g = __shfl_sync(0xffffffffu, factor, min(c + u, 31));
                    if (c + u < n) {
                        const float* z = (const float*)&y[u];
#pragma unroll
                        for (int i = 0; i < DPL; i++) o[i] = fmaf(z[i], g, o[i]);
                    }
                }
            }
        }
        const float inv = tree_ratio(1.0f, sum);
        TQ* dst = (TQ*)a.out + (size_t)row * a.out_stride + (size_t)h * HD + lane * DPL;
#pragma unroll
        for (int i = 0; i < DPL; i++) dst[i] = out_of<TQ>(o[i] * inv);
    }
}

// Copies of the query rows in a tile of 128 (see attn_tree_tc): as many as there is room for, since the lengths, which tell who waits for HBM, are on the device.  Two of the pairs
// below lose 5 % by it, the others gain 9 to 18.  Measured with / without, us: 32 trees of 16 nodes of 4 query heads (2 copies) 53 / 65
// when they came in, 10 trees of 8 over 850 rows (4) 20.3 / 22.2, 16 of 16 over 16000 (2) 212 / 241, 16 of 8 over 16000 (4; bound by HBM) 185 / 177, one of 8 over 500 10.0 / 9.5.
int copies_of(const TreeAttnArgs& a) {
    const int rows = a.t.max_rows * (a.n_q / a.n_kv);
    return rows <= 32 ? 4 : rows <= 64 ? 2 : 1;
}
// What the call knows on the host: the CTAs that run at once, and bounds of the units and pieces the batch can have.
struct Bounds { long long units, tiles; };
Bounds bounds_of(const TreeAttnArgs& a, int tile_rows) {
    const int G = a.n_q / a.n_kv;
    long long tiles = ((long long)a.t.max_prefix + a.t.max_rows + kTileKeys - 1) / kTileKeys;
    if (a.window > 0) tiles = std::min(tiles, ((long long)a.window + a.t.max_rows) / kTileKeys + 2);
    return {(long long)a.t.n_seq * a.n_kv * ((a.t.max_rows * G + tile_rows - 1) / tile_rows), tiles};
}
// Few units of not too many tiles (as the call's bounds have it: a graph captured with large ones keeps to pieces): a cluster for each, whose CTAs share its tiles evenly and join their shares through distributed shared memory.  One launch, no scratch, and
// no search for pieces.  Measured against pieces and tree_combine (or, below 9 tiles, whole units), us in a graph, 8 K/V heads of 4 query heads of 128 in bf16, trees of 8:
// 1 x 4 tiles 10.1 / 10.6 (of 32 nodes 13.7 / 12.6: more rows to join), 1 x 8 9.9 / 13.0, 1 x 63 13.7 / 17.5, 4 x 63 19.9 / 24.6, 1 x 251 27.6 / 34.7, 2 x 251 41.9 / 40.7, 1 x 501
// 55.0 / 45.1 (8 CTAs a unit are too few).  From an f32 cache, whose tiles take CUDA cores 7 us, only one tile a CTA: 1 x 4 17.8 / 18.9, 1 x 8 19.1 / 20.5,
// but 1 x 16 in 8 CTAs 26.0 / 22.0.  Clusters of 16 gain 1 us at most and lose up to 10 where an SM holds one CTA.
// A second CTA on an SM pays from six tiles each on: 16 x 16 tiles (8 a CTA) 19.4 in 256 CTAs / 23.5, but 4 x 8 (1 a CTA) 12.3 / 11.1.  Where lengths differ, pieces find the long
// sequence more CTAs (one of 63 tiles and 7 of 2: 16.8, in 4 CTAs a unit 19.7, in 2 28.4; with 15 of 2 18.4, in 2 29.1), so batches get fewer
// tiles a CTA: one of 63 and 3 of 2 (8 CTAs a unit) 14.8 / 16.6.
int cluster_of(const TreeAttnArgs& a, const Bounds& b, int sm_count, int slots) {
    int C = 1;
    while (C < kClusterMax && 2 * C <= b.tiles && (2 * C * b.units <= sm_count || (2 * C * b.units <= slots && 12 * C <= b.tiles))) C *= 2;
    const int most = !a.kv_bf16 ? 1 : a.t.n_seq == 1 ? 32 : 8 + C;             // tiles of a CTA
    return b.tiles > (a.kv_bf16 ? 4 : 1) && b.tiles <= (long long)C * most ? C : 1;
}
Share share_of(const TreeAttnArgs& a, int sm_count) {
    Share p{};
    const int G = a.n_q / a.n_kv;
    p.copies = a.kv_bf16 ? copies_of(a) : 1;
    p.tile_rows = a.kv_bf16 ? 128 / p.copies / G * G : kRowsTile;
    p.rows = std::min(p.tile_rows, a.t.max_rows * G);
    p.slots = sm_count * (a.kv_bf16 && !a.q_bf16 && a.hd == 128 ? 1 : 2);
    const Bounds b = bounds_of(a, p.tile_rows);
    p.sms = sm_count;
    p.cluster = cluster_of(a, b, sm_count, p.slots);
    p.row_tiles = (a.t.max_rows * G + p.tile_rows - 1) / p.tile_rows;
    if (p.cluster > 1) { p.grid = (int)b.units * p.cluster; return p; }
    // Few tiles: nothing is cut, and tree_combine (2 to 3 us, and as much of the caller's time) need not run.  Measured, us, whole / cut: 16 trees of 8 nodes over 508 rows in
    // bf16 (8 tiles, 128 units) 14.4 / 16.8, 64 of them 39.6 / 44.6; over f32 caches of 208 rows (4 tiles) 8 trees (64 units) 37.9 / 25.2, 16 37.7 / 39.3, 32 57.0 / 60.5.
    if (b.tiles <= (a.kv_bf16 ? 8 : 2 * b.units >= sm_count ? 4 : 1)) { p.grid = (int)b.units; return p; }
    // Pieces, as piece_find cuts them: at most `slots` where there are fewer units, else at most units + tiles / (2 tiles / slots).  Shares: the pieces of units that are cut, at
    // most `slots` in both cases.
    p.grid = (int)std::min(b.units * b.tiles, b.units < p.slots ? (long long)p.slots : b.units + p.slots / 2);
    p.shares = std::min(p.grid, p.slots);
    return p;
}
size_t plan_bytes(const TreeAttnArgs& a) { return ((size_t)a.t.n_seq + 1 + 3) / 4 * 16; }
size_t share_bytes(const TreeAttnArgs& a, const Share& p) { return !p.shares ? 0 : plan_bytes(a) + (size_t)p.shares * p.rows * (a.hd + 2) * 4; }

template <int HD, typename TQ>
cudaError_t combine(const TreeAttnArgs& a, const Share& p, cudaStream_t st) {
    if (!p.shares) return cudaSuccess;               // nothing is cut
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)std::min<long long>((long long)a.t.n_rows * ((a.n_q + 7) / 8), 2ll * p.sms * kJoinCtas));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // its CTAs are there when the last share is
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, tree_combine<HD, TQ>, a, p);
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
cudaError_t encode_bf16(CUtensorMap* map, const void* p, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
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
    const cuuint32_t step[4] = {1, 1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}
// A cache as a tensor [groups of 64 dimensions][row][64]: one copy brings both halves of a head of 128.
cudaError_t map_cache(CUtensorMap* map, const TreeAttnArgs& a, const void* cache, int box_rows) {
    const cuuint64_t dims[3] = {64, (cuuint64_t)a.m.rows, (cuuint64_t)a.n_kv * a.hd / 64}, strides[2] = {(cuuint64_t)a.kv_stride * 2, 128};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, box_rows == kTileKeys ? (cuuint32_t)a.hd / 64 : 1u};
    return encode_bf16(map, cache, 3, dims, strides, box);
}
// The queries as a tensor [half][row][head][64]: a box is the heads of a K/V head for the nodes of a unit.
cudaError_t map_queries(CUtensorMap* map, const TreeAttnArgs& a, int tile_rows) {
    const int G = a.n_q / a.n_kv;
    const cuuint64_t dims[4] = {64, (cuuint64_t)a.n_q, (cuuint64_t)a.t.n_rows, (cuuint64_t)a.hd / 64}, strides[3] = {(cuuint64_t)a.hd * 2, (cuuint64_t)a.q_stride * 2, 128};
    const cuuint32_t box[4] = {64, (cuuint32_t)G, (cuuint32_t)(tile_rows / G), 1};
    return encode_bf16(map, a.q, 4, dims, strides, box);
}
template <typename... Params, typename... Args>
cudaError_t launch_pieces(const Share& p, int threads, int smem, cudaStream_t st, void (*kernel)(Params...), Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)p.cluster; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = p.cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}
template <int HD>
cudaError_t rows_launch(const TreeAttnArgs& a, const Share& p, cudaStream_t st) {
    static std::atomic<uint64_t> raised{0};
    if (const cudaError_t e = allow_smem(raised, (const void*)attn_tree_rows<HD>, rows_smem<HD>())) return e;
    const cudaError_t e = launch_pieces(p, 256, rows_smem<HD>(), st, attn_tree_rows<HD>, a, p);
    return e != cudaSuccess ? e : combine<HD, float>(a, p, st);
}
template <int HD, bool F32, int DUP>
cudaError_t tc_launch_copies(const TreeAttnArgs& a, const Share& p, cudaStream_t st) {
    using S = TcShape<HD, F32>;
    static std::atomic<uint64_t> raised{0};
    if (const cudaError_t e = allow_smem(raised, (const void*)attn_tree_tc<HD, F32, DUP>, S::smem, true)) return e;
    const int box_rows = a.m.lg >= 0 && 1 << a.m.lg < kTileKeys ? 1 << a.m.lg : kTileKeys;
    CUtensorMap map_q{}, map_k, map_v;
    if constexpr (!F32) if (const cudaError_t e = map_queries(&map_q, a, p.tile_rows)) return e;
    if (const cudaError_t e = map_cache(&map_k, a, a.k, box_rows)) return e;
    if (const cudaError_t e = map_cache(&map_v, a, a.v, box_rows)) return e;
    const cudaError_t e = launch_pieces(p, kTcThreads, S::smem, st, attn_tree_tc<HD, F32, DUP>, a, p, map_q, map_k, map_v, box_rows);
    return e != cudaSuccess ? e : combine<HD, typename std::conditional<F32, float, __nv_bfloat16>::type>(a, p, st);
}
template <int HD, bool F32>
cudaError_t tc_launch(const TreeAttnArgs& a, const Share& p, cudaStream_t st) {
    return p.copies == 4 ? tc_launch_copies<HD, F32, 4>(a, p, st) : p.copies == 2 ? tc_launch_copies<HD, F32, 2>(a, p, st) : tc_launch_copies<HD, F32, 1>(a, p, st);
}

}  // namespace

bool tree_attn_supported(const TreeAttnArgs& a) {
    if (a.kv_bf16 && a.n_q / a.n_kv > 128) return false;
    const Bounds b = bounds_of(a, a.kv_bf16 ? 128 / copies_of(a) / (a.n_q / a.n_kv) * (a.n_q / a.n_kv) : kRowsTile);
    // tiles are counted in 32 bits, and so are tree_combine's items of eight (row, head)
    return b.units < 0x40000000ll && b.units * b.tiles < 0x7fffffffll && (long long)a.t.n_rows * ((a.n_q + 7) / 8) < 0x7fffffffll;
}
size_t tree_attn_workspace(const TreeAttnArgs& a, int sm_count) { return share_bytes(a, share_of(a, sm_count)); }

cudaError_t launch_tree_attn(const TreeAttnArgs& a, int sm_count, cudaStream_t st) {
    Share p = share_of(a, sm_count);
    if (share_bytes(a, p) > a.ws_bytes) return cudaErrorInvalidValue;
    p.plan = (int*)a.ws;
    p.o = (float*)((char*)a.ws + plan_bytes(a));
    p.ml = p.o + (size_t)p.shares * p.rows * a.hd;
    if (!a.kv_bf16) return a.hd == 128 ? rows_launch<128>(a, p, st) : rows_launch<64>(a, p, st);
    if (a.hd == 128) return a.q_bf16 ? tc_launch<128, false>(a, p, st) : tc_launch<128, true>(a, p, st);
    return a.q_bf16 ? tc_launch<64, false>(a, p, st) : tc_launch<64, true>(a, p, st);
}

}  // namespace lum
