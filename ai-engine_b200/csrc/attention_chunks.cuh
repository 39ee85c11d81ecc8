// Attention of a few new tokens a request over its paged cache, with the lengths on the device alone: how the work is shared out,
// and how shared results are joined.  Included by the kernels' files.
//
// Token i of request r stands at position ctx_len[r] + i, its query head h reads key head h / G (G = H / K).  The queries of one key head
// are rows: row = i * G + g.  An item is (request, key head, tile of M rows); it walks key tiles of KT keys, from the one that holds the
// first key any of its rows sees to the one of its last row's own key.
//
// All items' key tiles stand in one line, in the order of requests, key heads and row tiles, each as long as it takes (a weight by the
// item's rows); block c of C takes those that begin in [c * per, (c + 1) * per), per = ceil(all / C), so every block has the same work
// whatever the requests' lengths.  Every block works out the line from the lengths by itself (sums over the requests), so nothing comes from
// the host and a captured call follows the lengths.  An item that a block does not finish is left as a part: sums of exp2(x - m) v without
// division, m and l, in a place of the block's own (one for an item that it began, one for an item that it continued), and a second,
// small kernel joins the parts of every item in their order.  The split depends on all requests' lengths: the sums of a token
// are taken in another order in another batch.
#pragma once
#include "common.cuh"
#include "division.cuh"
#include "draft_args.h"

struct ChArgs : ChCall {
    FastDiv by_g, by_p;
};

// Checks a call and completes it; M, KT, weight: rows of an item, keys of a tile and its largest weight in the kernel that takes it; line: whether
// blocks share it (what they leave has to have its place, and an item's parts are counted in 15 bits).
static inline int ch_args(const ChCall* call, int M, int KT, int weight, bool line, ChArgs* a) {
    *static_cast<ChCall*>(a) = *call;
    if (a->W <= 0 || a->num_pages <= 0 || a->P <= 0 || a->K <= 0 || a->H <= 0 || a->H % a->K || a->G != a->H / a->K) return AIE_BAD_ARG;
    if (line && (a->blocks <= 0 || a->blocks > 0x7fff || !a->part_o || !a->part_ml || !a->meta)) return AIE_BAD_ARG;
    // the line's length has to fit 31 bits: every request at least one row tile a key head, each over all the table's keys (where
    // requests name the same rows more than once, ch_begin finds what this does not)
    const double items = (double)a->T * a->H / M + (double)a->R * a->K, keys = (double)a->W * a->P / KT + 2;
    if (items * keys * weight > 2147000000.0) return -3;
    a->by_g = fast_div((unsigned)a->G);
    a->by_p = fast_div((unsigned)a->P);
    return 0;
}

struct ChReq { int n, c; };           // tokens it brings (0: none, or lengths that do not fit), tokens it has
__device__ __forceinline__ ChReq ch_req(const ChArgs& a, int r, unsigned* bad = nullptr) {
    const int n = a.q_len[r], c = a.ctx_len[r], s = a.q_start[r];
    // W * P fits 31 bits
    const bool fits = n >= 0 && c >= 0 && s >= 0 && s <= a.T && n <= a.T - s && c <= a.W * a.P && n <= a.W * a.P - c;
    if (!fits && bad) *bad |= AIE_DEV_SLOT_OOB;
    return {fits ? n : 0, c};
}

// A kernel's shape Sh: M rows of an item, KT keys of a tile, weight(rows) of a key tile (at most MAX_WEIGHT).
struct ChTile { int row0, rows, i0, i1, first, tiles; };      // rows of the tile, its first and last token, first key tile, key tiles
template <typename Sh> __device__ __forceinline__ ChTile ch_tile(const ChArgs& a, const ChReq& q, int m) {
    ChTile t;
    t.row0 = m * Sh::M;
    t.rows = min(Sh::M, q.n * a.G - t.row0);
    t.i0 = fast_over(t.row0, a.by_g);
    t.i1 = fast_over(t.row0 + t.rows - 1, a.by_g);
    const int lo = a.window > 0 ? max(0, q.c + t.i0 - a.window + 1) : 0;
    t.first = lo / Sh::KT;
    t.tiles = (q.c + t.i1) / Sh::KT - t.first + 1;
    return t;
}
template <typename Sh> __device__ __forceinline__ int ch_length(const ChArgs& a, const ChReq& q) {      // of the line of one key head
    int s = 0;
    for (int m = 0; m * Sh::M < q.n * a.G; ++m) {
        const ChTile t = ch_tile<Sh>(a, q, m);
        s += t.tiles * Sh::weight(t.rows);
    }
    return s;
}

// Where a block is in the line.
struct ChWalk {
    int left, per;           // of the line, from the beginning of tile k to the end of this block's share; length of a share
    int r, kh, m, k, s0;     // item, key tile within it, the request's first token
    ChReq req;
    ChTile tile;
};
struct ChShared {
    long long sums[16];     // of a block's warps
    int r, off, n, c, s0;    // request in which the share begins, how far behind the request's first tile, its lengths
};

// Adds up `v` over the block in the order of threads; the result is what comes before this thread's, `all` the sum.
template <int THREADS> __device__ __forceinline__ long long ch_scan(int v, ChShared* s, long long* all) {
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

// ... on to the next item; false: there is none
template <typename Sh> __device__ __forceinline__ bool ch_item(const ChArgs& a, ChWalk& w) {
    w.k = 0;
    ++w.m;
    if (w.m * Sh::M >= w.req.n * a.G) {
        w.m = 0;
        if (++w.kh == a.K) {
            w.kh = 0;
            do {
                if (++w.r >= a.R) return false;
                w.req = ch_req(a, w.r);
            } while (w.req.n == 0);
            w.s0 = a.q_start[w.r];
        }
    }
    w.tile = ch_tile<Sh>(a, w.req, w.m);
    return true;
}
// This block's share of the line; false: none.  All threads of the block call it.
template <int THREADS, typename Sh>
__device__ __forceinline__ bool ch_begin(const ChArgs& a, int c, int C, ChShared* s, ChWalk& w) {
    const int tid = threadIdx.x;
    int mine = 0;
    long long all = 0, before = 0;
    ChReq q = {0, 0};
    for (int base = 0; base < a.R; base += THREADS) {
        const int r = base + tid;
        unsigned bad = 0;
        mine = 0;
        if (r < a.R) {
            q = ch_req(a, r, &bad);
            mine = a.K * ch_length<Sh>(a, q);
            if (bad && c == 0) atomicOr(a.err, bad);
        }
        long long sum;
        before = all + ch_scan<THREADS>(mine, s, &sum);
        all += sum;
    }
    if (all > 0x7fffffff) {          // only where requests name the same rows again and again: their lengths do not fit q together
        if (c == 0 && tid == 0) atomicOr(a.err, AIE_DEV_SLOT_OOB);
        return false;
    }
    // at least the weight of a tile: a tile then begins in every share that lies within one item
    w.per = max((int)(((unsigned)all + C - 1) / (unsigned)C), Sh::MAX_WEIGHT);
    const long long first = (long long)c * w.per;
    if (first >= all) return false;
    const int at = (int)first;
    auto leave = [&](int r, const ChReq& x, int off) {
        s->r = r;
        s->off = off;
        s->n = x.n;
        s->c = x.c;
        s->s0 = a.q_start[r];
    };
    if (a.R <= THREADS) {
        if (at >= before && at < before + mine) leave(tid, q, (int)(at - before));
    } else {
        long long upto = 0;
        for (int base = 0; base < a.R; base += THREADS) {
            const int r = base + tid;
            q = r < a.R ? ch_req(a, r) : ChReq{0, 0};
            const int here = r < a.R ? a.K * ch_length<Sh>(a, q) : 0;
            long long sum;
            const long long b = upto + ch_scan<THREADS>(here, s, &sum);
            if (at >= b && at < b + here) leave(r, q, (int)(at - b));
            upto += sum;
        }
    }
    __syncthreads();
    w.r = s->r;
    w.s0 = s->s0;
    w.req = {s->n, s->c};
    const unsigned one = (unsigned)ch_length<Sh>(a, w.req), off = (unsigned)s->off;
    w.kh = (int)(off / one);
    int rest = (int)(off - w.kh * one), weight;
    for (w.m = 0;; ++w.m) {
        w.tile = ch_tile<Sh>(a, w.req, w.m);
        weight = Sh::weight(w.tile.rows);
        if (rest < w.tile.tiles * weight) break;
        rest -= w.tile.tiles * weight;
    }
    w.k = (rest + weight - 1) / weight;                  // the first tile that begins in the share
    w.left = w.per - (w.k * weight - rest);
    if (w.k == w.tile.tiles) return w.left > 0 && ch_item<Sh>(a, w);
    return w.left > 0;
}
template <typename Sh> __device__ __forceinline__ int ch_share(const ChWalk& w) {      // key tiles of the item that are this block's
    const int weight = Sh::weight(w.tile.rows);
    return min(w.tile.tiles - w.k, (w.left + weight - 1) / weight);
}
// ... the next item behind the `n` tiles of this one; false: the share is done
template <typename Sh> __device__ __forceinline__ bool ch_next(const ChArgs& a, ChWalk& w, int n) {
    w.left -= n * Sh::weight(w.tile.rows);
    return w.left > 0 && ch_item<Sh>(a, w);
}
// A value that is not finite belongs to the rows that see its key and to no others, but a probability of 0 times it is NaN.  Where every row of an
// item sees every key of a step that is as it should be; on the other steps, which touch the diagonal or a window's edge, the kernels take
// such values out of the product and add them to the outputs of the rows that see them (whatever the weight: it is above 0).
__device__ __forceinline__ bool ch_sees(int pos, int key, int window) { return key <= pos && (window <= 0 || key > pos - window); }
// of two pairs of bfloat16, each the one that is larger in size, NaN where one of them is (the sign means nothing)
__device__ __forceinline__ unsigned ch_larger(unsigned a, unsigned b) {
    unsigned r;
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// two bfloat16: bits 15 and 31 where the lower, the upper one is not finite
__device__ __forceinline__ unsigned ch_unfinite(unsigned v) { return ((v & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }
__device__ __forceinline__ unsigned ch_without(unsigned v, unsigned unfinite) { return v & ~((unfinite >> 15) * 0xffffu); }

// A row's maximum for those who join its parts: maxima pass over what is not a number, a sum that is none has to come along.
__device__ __forceinline__ float2 ch_left(float m, float l) { return make_float2(l == l ? m : l, l); }

// What the joining kernel has to know of the item that block c begins here and does not finish.
template <typename Sh> __device__ __forceinline__ void ch_leave(const ChArgs& a, const ChWalk& w, int c) {
    const int last = (w.tile.tiles - 1) * Sh::weight(w.tile.rows);      // where its last tile begins, from the item's beginning
    const int parts = last < w.left ? 1 : 2 + (last - w.left) / w.per;      // at most as many as there are blocks
    a.meta[c] = make_int4(w.kh, w.tile.row0, w.tile.rows | parts << 16, w.s0);
}
__device__ __forceinline__ float ch_inverse(float l) { return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); }      // of a row's sum; a row that sees nothing is zero

// Joins the parts of the items that blocks c .. c + PER - 1 began: out = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p, four columns of a row a
// thread.  What bounds it is the way to memory, twice: what there is to join, then its parts.  Four parts' loads are under way together:
// 60 registers, so that four blocks stay on an SM (eight parts and 80: 300 to 500 new tokens of four requests behind 6,000 to 9,000 228 us in
// all instead of 223, calls of 20 to 100 us 6 % more).  Items of 256 rows take 32 blocks, so that one in sixty parts does not take eight
// of them 30 us, and a block looks at two of them (at four or at one: 2 and 4 % more; a list of the items with parts, made by every block, cost 4 us).
template <typename T, int M, int D, int PER>
__global__ void __launch_bounds__(256) chunk_join_kernel(const ChArgs a, int C) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int CH = D / 4, AT = 4;
    int4 its[PER];
#pragma unroll
    for (int x = 0; x < PER; ++x) its[x] = blockIdx.x * PER + x < C ? a.meta[blockIdx.x * PER + x] : make_int4(0, 0, 0, 0);
#pragma unroll 1
    for (int x = 0; x < PER; ++x) {
        int4 it = its[0];
#pragma unroll
        for (int y = 1; y < PER; ++y)
            if (y == x) it = its[y];
        const int c = blockIdx.x * PER + x, rows = it.z & 0xffff, parts = it.z >> 16;
        if (parts == 0) continue;
        for (int i = blockIdx.y * 256 + threadIdx.x; i < rows * CH; i += gridDim.y * 256) {
            const int row = i / CH, e = (i - row * CH) * 4;
            if (e >= a.d) continue;
            // part 0 lies in block c's place for items begun, part p in block c + p's for items continued
            const float* ml = a.part_ml + ((size_t)2 * c * M + row) * 2;
            const float* po = a.part_o + ((size_t)2 * c * M + row) * D + e;
            float m = -INFINITY, l = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int p0 = 0; p0 < parts; p0 += AT) {
                float2 g[AT];
                float4 z[AT];
#pragma unroll
                for (int p = 0; p < AT; ++p) {
                    const bool there = p0 + p < parts;
                    const size_t place = there ? (p0 + p == 0 ? 1 : 2 * (p0 + p)) : 1;
                    g[p] = there ? *reinterpret_cast<const float2*>(ml + place * (M * 2)) : make_float2(-INFINITY, 0.f);
                    if (there) z[p] = *reinterpret_cast<const float4*>(po + place * ((size_t)M * D));
                }
                float top = m;
#pragma unroll
                for (int p = 0; p < AT; ++p) top = fmaxf(top, g[p].x);
                const float was = m == -INFINITY ? 0.f : exp2f(m - top);
                l *= was;
                o.x *= was, o.y *= was, o.z *= was, o.w *= was;
#pragma unroll
                for (int p = 0; p < AT; ++p) {
                    if (g[p].x == -INFINITY) continue;
                    const float f = exp2f(g[p].x - top);
                    l += f * g[p].y;
                    o.x += f * z[p].x, o.y += f * z[p].y, o.z += f * z[p].z, o.w += f * z[p].w;
                }
                m = top;
            }
            const float inv = ch_inverse(l);
            const int full = it.y + row, tok = fast_over(full, a.by_g), h = it.x * a.G + full - tok * a.G;
            store4<T>(reinterpret_cast<T*>(a.out) + ((size_t)(it.w + tok) * a.H + h) * a.d + e,
                      make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
        }
    }
}
// What a kernel is told once on each device: the shared memory it takes (0: none), and that it wants as much of it an SM as there is.
template <typename F> static void ch_prepare(F kern, int bytes, unsigned long long* done) {
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && dev < 64 && (*done >> dev & 1)) return;
    if (bytes) cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (dev < 64) *done |= 1ull << dev;
}
// ... with as much shared memory an SM as the kernel before it, which would otherwise have to leave the SM before it changes
template <typename T, int M, int D> static int launch_chunk_join(const ChArgs& a, int C, cudaStream_t st) {
    constexpr int PER = M > 32 ? 2 : 1;
    auto kern = chunk_join_kernel<T, M, D, PER>;
    static unsigned long long done = 0;
    ch_prepare(kern, 0, &done);
    return (int)launch_pdl(kern, dim3((C + PER - 1) / PER, M * D / 4 / 256), dim3(256), 0, st, a, C);
}
