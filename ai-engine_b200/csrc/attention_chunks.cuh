// Attention of a few new tokens a request over its paged cache, with the lengths on the device alone: how the work is shared out,
// and how shared results are joined.  Included by the kernels' files.
//
// Token i of request r stands at position ctx_len[r] + i, its query head h reads key head h / G (G = H / K).  The queries of one key head
// are rows: row = i * G + g.  An item is (request, key head, tile of M rows); it walks key tiles of KT keys, from the one that holds the
// first key any of its rows sees to the one of its last row's own key.
//
// All items' key tiles stand in one line, in the order of requests, key heads and row tiles; block c of C takes those from c * per to
// (c + 1) * per - 1, per = ceil(all / C), so every block has the same number of tiles whatever the requests' lengths.  Every
// block works out the line from the lengths by itself (two passes of sums over the requests), so nothing comes from the host and a
// captured call follows the lengths.  An item that a block does not finish is left as a part: sums of exp2(x - m) v without
// division, m and l, in a place of the block's own (one for an item that it began, one for an item that it continued), and a second,
// small kernel joins the parts of every item in their order.  The split depends on all requests' lengths: the sums of a token
// are taken in another order in another batch.
#pragma once
#include "common.cuh"

struct ChArgs {
    const void* q;                    // [T, H, d], elements q_token / q_head apart
    const void* k_pages;              // [num_pages, K, P, d]
    const void* v_pages;
    void* out;                        // [T, H, d]
    const int *q_start, *q_len, *ctx_len, *table;
    float* part_o;                    // [2 * C][M][D]
    float* part_ml;                   // [2 * C][M][2]
    int4* meta;                       // [C] (request, key head, row tile, parts) of the item that block c began and did not finish
    long long q_token, q_head;
    int R, W, T, num_pages, P, H, K, G, d, window;
    float scale2;                     // scale * log2 e: exponentials are powers of two
    unsigned* err;
};

struct ChReq { int n, c; };           // tokens it brings (0: none, or lengths that do not fit), tokens it has
__device__ __forceinline__ ChReq ch_req(const ChArgs& a, int r, unsigned* bad = nullptr) {
    const int n = a.q_len[r], c = a.ctx_len[r], s = a.q_start[r];
    const bool fits = n >= 0 && c >= 0 && s >= 0 && s <= a.T && n <= a.T - s && ((long long)c + n + a.P - 1) / a.P <= a.W;
    if (!fits && bad) *bad |= AIE_DEV_SLOT_OOB;
    return {fits ? n : 0, c};
}

struct ChTile { int row0, rows, i0, i1, first, tiles; };      // rows of the tile, its first and last token, first key tile, key tiles
template <int M, int KT> __device__ __forceinline__ ChTile ch_tile(const ChArgs& a, const ChReq& q, int m) {
    ChTile t;
    t.row0 = m * M;
    t.rows = min(M, q.n * a.G - t.row0);
    t.i0 = t.row0 / a.G;
    t.i1 = (t.row0 + t.rows - 1) / a.G;
    const int lo = a.window > 0 ? max(0, q.c + t.i0 - a.window + 1) : 0;
    t.first = lo / KT;
    t.tiles = (q.c + t.i1) / KT - t.first + 1;
    return t;
}
template <int M, int KT> __device__ __forceinline__ long long ch_tiles(const ChArgs& a, const ChReq& q) {      // of one key head
    long long s = 0;
    for (int m = 0; m * M < q.n * a.G; ++m) s += ch_tile<M, KT>(a, q, m).tiles;
    return s;
}

// Where a block is in the line.
struct ChWalk {
    long long at, end;       // next key tile of the line, end of this block's share
    int r, kh, m, k;         // item, and key tile within it
    ChReq req;
    ChTile tile;
};
struct ChShared { long long sums[32]; long long all; long long off; int r; };

// Adds up `v` over the block in the order of threads; the result is what comes before this thread's, `all` the sum.
template <int THREADS> __device__ __forceinline__ long long ch_scan(long long v, ChShared* s, long long* all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) s->sums[warp] = x;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w == warp) before = total;
        total += s->sums[w];
    }
    *all = total;
    return before + x - v;
}

// This block's share of the line; false: none.  All threads of the block call it.
template <int THREADS, int M, int KT, int MIN_TILES>
__device__ __forceinline__ bool ch_begin(const ChArgs& a, int c, int C, ChShared* s, ChWalk& w) {
    const int tid = threadIdx.x;
    long long all = 0, mine = 0, before = 0;
    for (int base = 0; base < a.R; base += THREADS) {
        const int r = base + tid;
        unsigned bad = 0;
        mine = 0;
        if (r < a.R) {
            const ChReq q = ch_req(a, r, &bad);
            mine = a.K * ch_tiles<M, KT>(a, q);
            if (bad && c == 0) atomicOr(a.err, bad);
        }
        long long sum;
        before = all + ch_scan<THREADS>(mine, s, &sum);
        all += sum;
    }
    long long per = (all + C - 1) / C;
    if (per < MIN_TILES) per = MIN_TILES;
    w.at = c * per;
    w.end = min(all, w.at + per);
    if (w.at >= all) return false;
    if (a.R <= THREADS) {
        if (w.at >= before && w.at < before + mine) { s->r = tid; s->off = w.at - before; }
    } else {
        long long upto = 0;
        for (int base = 0; base < a.R; base += THREADS) {
            const int r = base + tid;
            const long long here = r < a.R ? a.K * ch_tiles<M, KT>(a, ch_req(a, r)) : 0;
            long long sum;
            const long long b = upto + ch_scan<THREADS>(here, s, &sum);
            if (w.at >= b && w.at < b + here) { s->r = r; s->off = w.at - b; }
            upto += sum;
        }
    }
    __syncthreads();
    w.r = s->r;
    w.req = ch_req(a, w.r);
    const long long one = ch_tiles<M, KT>(a, w.req);
    w.kh = (int)(s->off / one);
    long long k = s->off % one;
    for (w.m = 0;; ++w.m) {
        w.tile = ch_tile<M, KT>(a, w.req, w.m);
        if (k < w.tile.tiles) break;
        k -= w.tile.tiles;
    }
    w.k = (int)k;
    return true;
}
// ... the next item after `n` tiles of this one; false: the share is done
template <int M, int KT> __device__ __forceinline__ bool ch_next(const ChArgs& a, ChWalk& w, int n) {
    w.at += n;
    if (w.at >= w.end) return false;
    w.k = 0;
    ++w.m;
    if (w.m * M >= w.req.n * a.G) {
        w.m = 0;
        if (++w.kh == a.K) {
            w.kh = 0;
            do { w.req = ch_req(a, ++w.r); } while (w.req.n == 0);
        }
    }
    w.tile = ch_tile<M, KT>(a, w.req, w.m);
    return true;
}
__device__ __forceinline__ int ch_share(const ChWalk& w) {      // key tiles of the item that are this block's
    return (int)min((long long)(w.tile.tiles - w.k), w.end - w.at);
}
// Blocks that have a part of the item which block `c` begins and leaves at `w` (its last `n` tiles of the share).
__device__ __forceinline__ int ch_parts(const ChWalk& w, int n, long long per) {
    const long long rest = w.tile.tiles - w.k - n;
    return 1 + (int)((rest + per - 1) / per);
}

// Joins the parts of the item that block c began: out = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p.  A thread has four columns of a row.
template <typename T, int M, int D>
__global__ void __launch_bounds__(256) chunk_join_kernel(const ChArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int c = blockIdx.x;
    const int4 it = a.meta[c];
    if (it.w == 0) return;
    const int r = it.x, n = a.q_len[r];
    const int rows = min(M, n * a.G - it.z * M);
    constexpr int CH = D / 4;
    for (int i = blockIdx.y * 256 + threadIdx.x; i < rows * CH; i += gridDim.y * 256) {
        const int row = i / CH, e = (i - row * CH) * 4;
        if (e >= a.d) continue;
        auto place = [&](int p) { return (size_t)(p == 0 ? 2 * c + 1 : 2 * (c + p)) * M + row; };
        float m = -INFINITY;
        for (int p = 0; p < it.w; ++p) m = fmaxf(m, a.part_ml[place(p) * 2]);
        float l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p = 0; p < it.w; ++p) {
            const size_t at = place(p);
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
            const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - m);
            const float4 x = *reinterpret_cast<const float4*>(a.part_o + at * D + e);
            l += f * ml.y;
            o.x += f * x.x, o.y += f * x.y, o.z += f * x.z, o.w += f * x.w;
        }
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        const int full = it.z * M + row, i_tok = full / a.G, h = it.y * a.G + full - i_tok * a.G;
        store4<T>(reinterpret_cast<T*>(a.out) + ((size_t)(a.q_start[r] + i_tok) * a.H + h) * a.d + e,
                  make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    }
}
