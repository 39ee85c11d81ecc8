// Attention of new tokens over a paged cache (see attention_chunks.cuh) in bfloat16, heads of 64 and 128, for items of 32 rows:
// a few drafted tokens of a request times the query heads of a key head; any page size.
//   o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),   x_j = (q . k_j) * scale * log2 e
//
// Products go through mma.sync, whose tiles of 16 rows fit 4 tokens of 4 heads.  A block has four groups of two warps; of every key
// tile each group takes CK keys of its own through a ring of its own (cp.async, stages of 8 KB), and each warp of a group has 16 rows of
// the item and reads the group's keys and values.  Groups meet only at an item's end, where their outputs are added up in shared memory.
// What bounds it: reading keys and values once, and 10 us of a small call's chain of waits (lengths, pages, rows, outputs that meet).  One
// warp for 32 rows (255 registers, eight warps an SM) waited for its own instructions, 5.3 cycles each, at half of the memory's rate
// (56 requests of heads of 64: 84 us, now 73); items of 16 rows or of 64 were at most a twentieth better anywhere.
// Scores, maxima and sums are float32, a row's reference maximum moves by more than 8 (log2 units) or not at all; probabilities are rounded
// to bfloat16 for the product with the values, as the values are (a product in two terms would be half as many instructions again); sums take them unrounded.
// An error of 0.0021 to 0.0023 of the result's norm, of which the result's own rounding is 0.0017.
//
// Two ways to share the work out.  The line of attention_chunks.cuh balances any lengths, at the price of a second kernel.  For few requests
// with few keys that is a third of the call, so there a cluster of S blocks takes a (request, key head), each block a part of every item's
// key tiles, and the parts are joined in the cluster's shared memory (one request of 5 tokens behind 1,000, 32 heads of 128: 10.3 us
// by the line, 7.3 by clusters of eight; eight requests behind 500 to 2,000: 20.5, and 18.7 by clusters of four).
#include <cooperative_groups.h>

#include "attention_chunks.cuh"

namespace cg = cooperative_groups;

#define CB_GROUPS 4
#define CB_GW 2                // warps of a group
#define CB_RESCALE_STEP 8.0f

template <int D> struct CbShape {
    static constexpr int GW = CB_GW;
    static constexpr int M = 16 * GW;                 // rows of an item
    static constexpr int threads = CB_GROUPS * GW * 32;
    static constexpr int CK = D == 64 ? 32 : 16;      // keys of a group's stage
    static constexpr int KT = CB_GROUPS * CK;         // keys of a tile
    static constexpr int MAX_WEIGHT = 1;
    static __device__ __forceinline__ int weight(int) { return 1; }
    static constexpr int NST = 3;
    static constexpr int stage = 2 * CK * D;          // elements: keys, then values
    static constexpr int TPK = 32 * GW / CK;          // threads that copy a key
    static constexpr int ring_bytes = CB_GROUPS * NST * stage * 2;
    static constexpr int blocks = 2;                  // an SM: 16 warps of 128 registers
    static constexpr int o_bytes = CB_GROUPS * M * D * 4;      // the groups' outputs meet in the ring's memory
    static constexpr int q_off = ring_bytes > o_bytes ? ring_bytes : o_bytes, ml_off = q_off + M * D * 2;
    static constexpr int block_ml_off = ml_off + CB_GROUPS * M * 2 * 4, bytes = block_ml_off + M * 2 * 4;      // the block's own maxima and sums, for its cluster
};

__device__ __forceinline__ void cb_fetch(unsigned dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(there ? 16 : 0));
}
__device__ __forceinline__ void cb_ldsm(unsigned (&r)[4], unsigned p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p));
}
__device__ __forceinline__ void cb_ldsm_t(unsigned (&r)[4], unsigned p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p));
}
__device__ __forceinline__ unsigned cb_load(unsigned p) {
    unsigned v;
    asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(v) : "r"(p) : "memory");
    return v;
}
__device__ __forceinline__ void cb_mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned cb_pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<unsigned*>(&v);
}
__device__ __forceinline__ float cb_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// whether any of `STAGE / 2` elements at `p` is not finite, for a whole warp
template <int STAGE> __device__ __forceinline__ bool cb_unfinite(unsigned p, int lane) {
    unsigned m[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < STAGE / 512; ++i) {
        unsigned v[4];
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(p + (i * 32 + lane) * 16) : "memory");
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = ch_larger(m[e], v[e]);
    }
    return __any_sync(0xffffffffu, ch_unfinite(ch_larger(ch_larger(m[0], m[1]), ch_larger(m[2], m[3]))) != 0);
}
// byte offset of row r, 16-byte piece c of rows of D elements: pieces are permuted so that eight rows' pieces lie in different banks
template <int D> __device__ __forceinline__ unsigned cb_at(int row, int piece) { return (unsigned)(row * (D * 2) + ((piece ^ (row & 7)) << 4)); }

// The walk of a block in a cluster: its part of the tiles of row tile `m` (maybe none).
template <typename Sh> __device__ __forceinline__ void cb_part(const ChArgs& a, ChWalk& w, int m, int rank, int S) {
    w.m = m;
    w.tile = ch_tile<Sh>(a, w.req, m);
    w.per = (w.tile.tiles + S - 1) / S;
    w.k = rank * w.per;
    w.left = max(0, min(w.per, w.tile.tiles - w.k));
}

template <int D, bool CLUSTER>
__global__ void __launch_bounds__(CbShape<D>::threads, CbShape<D>::blocks) chunk_bf16_kernel(const ChArgs a, int S_blocks) {
    using S = CbShape<D>;
    constexpr int GW = CB_GW, M = S::M, KT = S::KT, CK = S::CK, PC = D / 8, NST = S::NST, THREADS = S::threads, TPK = S::TPK;
    extern __shared__ __align__(128) unsigned char cb_smem[];
    __shared__ ChShared sh;
    __shared__ ChWalk place_in_line;      // while the registers hold rows' outputs
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = warp / GW, mt = warp % GW, gt = mt * 32 + lane;
    const int rank = CLUSTER ? blockIdx.x % S_blocks : 0;
    ChWalk w;
    if constexpr (CLUSTER) {
        const int item = blockIdx.x / S_blocks;
        unsigned bad_lengths = 0;
        w.r = item / a.K;
        w.kh = item - w.r * a.K;
        w.req = ch_req(a, w.r, &bad_lengths);
        w.s0 = a.q_start[w.r];
        if (bad_lengths && tid == 0 && rank == 0 && w.kh == 0) atomicOr(a.err, bad_lengths);
        if (w.req.n == 0) return;                 // the whole cluster
        cb_part<S>(a, w, 0, rank, S_blocks);
    } else {
        if (tid == 0) a.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
        if (!ch_begin<THREADS, S>(a, blockIdx.x, gridDim.x, &sh, w)) return;
    }
    const unsigned smem = (unsigned)__cvta_generic_to_shared(cb_smem);
    const unsigned ring = smem + group * NST * S::stage * 2, q_s = smem + S::q_off;
    float* ml = reinterpret_cast<float*>(cb_smem + S::ml_off);      // [groups][M][2]
    const bf16* kp = reinterpret_cast<const bf16*>(a.k_pages);
    const bf16* vp = reinterpret_cast<const bf16*>(a.v_pages);
    const int r0 = lane >> 2, col = (lane & 3) * 2;      // of a 16 x 8 accumulator: rows r0 and r0 + 8, columns col and col + 1
    const int lm = lane >> 3, l8 = lane & 7;             // ldmatrix: matrix and row that this lane points at
    const bool plain = a.scale2 > 0.f;                   // else scores are scaled before they are masked
    const float sl2 = plain ? a.scale2 : 1.f;
    unsigned bad = 0;

    for (;;) {
        const int n = CLUSTER ? w.left : ch_share<S>(w);
        const ChTile tl = w.tile;
        const int c0 = w.req.c, s0 = w.s0, hi = c0 + tl.i1 + 1;
        const int* bt = a.table + (size_t)w.r * a.W;
        const int kt0 = tl.first + w.k;
        const int low_all = a.window > 0 ? c0 + tl.i0 - a.window + 1 : 0;      // first key that any row sees

        // this thread copies every TPK-th piece of its key of the stage; the pages of the next two stages' keys are read ahead
        auto key_of = [&](int i) { return (kt0 + i) * KT + group * CK + gt / TPK; };
        auto page_of = [&](int i) {
            const int key = key_of(i);
            return i < n && key < hi && key >= low_all ? bt[fast_over(key, a.by_p)] : -1;
        };
        int page = page_of(0), page_next = page_of(1);
        // queries of the item: they land with the first stage
        for (int i = tid; i < M * PC; i += THREADS) {
            const int row = i / PC, pc = i % PC;
            const bool there = row < tl.rows;
            const int full = tl.row0 + (there ? row : 0), t = fast_over(full, a.by_g), g = full - t * a.G;
            cb_fetch(q_s + cb_at<D>(row, pc), reinterpret_cast<const bf16*>(a.q) + (s0 + t) * a.q_token + (long long)(w.kh * a.G + g) * a.q_head + pc * 8, there);
        }
        auto issue = [&](int i, int slot) {
            if (i < n) {
                const unsigned st = ring + slot * S::stage * 2;
                const int key = key_of(i);
                bool there = key < hi && key >= low_all;
                if (there && (page < 0 || page >= a.num_pages)) {
                    bad |= AIE_DEV_PAGE_OOB;
                    there = false;
                }
                const size_t off = there ? (((size_t)page * a.K + w.kh) * a.P + (key - fast_over(key, a.by_p) * a.P)) * D + gt % TPK * 8 : 0;
#pragma unroll
                for (int y = 0; y < PC / TPK; ++y) {
                    const unsigned to = st + cb_at<D>(gt / TPK, gt % TPK + y * TPK);
                    cb_fetch(to, kp + off + y * TPK * 8, there);
                    cb_fetch(to + CK * D * 2, vp + off + y * TPK * 8, there);
                }
                page = page_next;
                page_next = page_of(i + 2);
            }
            asm volatile("cp.async.commit_group;\n" ::);
        };
#pragma unroll
        for (int i = 0; i < NST - 1; ++i) issue(i, i);

        asm volatile("cp.async.wait_group %0;\n" ::"n"(NST - 2));
        __syncthreads();

        const bool live = mt * 16 < tl.rows;             // any row of this warp
        float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f}, o[D / 8][4];
        const int pos0 = c0 + fast_over(tl.row0 + mt * 16 + r0, a.by_g), pos1 = c0 + fast_over(tl.row0 + mt * 16 + r0 + 8, a.by_g);
#pragma unroll
        for (int x = 0; x < D / 8; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[x][e] = 0.f;
        const int last_low = a.window > 0 ? c0 + tl.i1 - a.window + 1 : 0;      // first key that the last row sees

        if (tid == 0) place_in_line = w;
        int slot = 0;
        for (int i = 0; i < n; ++i) {
            asm volatile("cp.async.wait_group %0;\n" ::"n"(NST - 2));
            // the stage is there for the whole group, and the group has read the one that the next copies go to
            asm volatile("bar.sync %0, %1;\n" ::"r"(1 + group), "n"(32 * GW) : "memory");
            issue(i + NST - 1, slot == 0 ? NST - 1 : slot - 1);
            const unsigned ks = ring + slot * S::stage * 2, vs = ks + CK * D * 2;
            slot = slot + 1 == NST ? 0 : slot + 1;
            const int k_at = (kt0 + i) * KT + group * CK;
            if (k_at >= hi || !live) continue;
            const bool edge = k_at + CK - 1 > c0 + tl.i0 || k_at < last_low;      // some rows do not see some of these keys
            float s[CK / 8][4];
#pragma unroll
            for (int x = 0; x < CK / 8; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[x][e] = 0.f;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                unsigned qa[4];
                cb_ldsm(qa, q_s + cb_at<D>(mt * 16 + (lm & 1) * 8 + l8, kk * 2 + (lm >> 1)));
#pragma unroll
                for (int x = 0; x < CK / 16; ++x) {
                    unsigned b[4];
                    cb_ldsm(b, ks + cb_at<D>(x * 16 + (lm >> 1) * 8 + l8, kk * 2 + (lm & 1)));
                    cb_mma(s[2 * x], qa, b[0], b[1]);
                    cb_mma(s[2 * x + 1], qa, b[2], b[3]);
                }
            }
            if (__builtin_expect(!plain, 0)) {
#pragma unroll
                for (int x = 0; x < CK / 8; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[x][e] *= a.scale2;
            }
            if (edge) {
#pragma unroll
                for (int x = 0; x < CK / 8; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = k_at + x * 8 + col + (e & 1), q = e < 2 ? pos0 : pos1;
                        if (key > q || (a.window > 0 && key <= q - a.window)) s[x][e] = -INFINITY;
                    }
                if (__builtin_expect(cb_unfinite<S::stage>(vs, lane), 0)) {
#pragma unroll 1
                    for (int kk = 0; kk < CK; ++kk) {
                        const bool sees0 = ch_sees(pos0, k_at + kk, a.window), sees1 = ch_sees(pos1, k_at + kk, a.window);
#pragma unroll
                        for (int x = 0; x < D / 8; ++x) {
                            const unsigned v = cb_load(vs + cb_at<D>(kk, x) + col * 2), u = ch_unfinite(v);
                            const float v0 = __uint_as_float(v << 16), v1 = __uint_as_float(v & 0xffff0000u);
                            if (sees0 && (u & 0x8000u)) o[x][0] += v0;
                            if (sees0 && (u >> 31)) o[x][1] += v1;
                            if (sees1 && (u & 0x8000u)) o[x][2] += v0;
                            if (sees1 && (u >> 31)) o[x][3] += v1;
                        }
                    }
                    // all warps that read the stage have added them: now they are taken out of it
                    const bool both = tl.rows > 16;
                    if (both) asm volatile("bar.sync %0, %1;\n" ::"r"(1 + group), "n"(32 * GW) : "memory");
                    else __syncwarp();
#pragma unroll 1
                    for (int i = lane; i < CK * D / 2; i += 32) {
                        const unsigned v = cb_load(vs + i * 4);
                        asm volatile("st.shared.u32 [%0], %1;\n" ::"r"(vs + i * 4), "r"(ch_without(v, ch_unfinite(v))) : "memory");
                    }
                    if (both) asm volatile("bar.sync %0, %1;\n" ::"r"(1 + group), "n"(32 * GW) : "memory");
                    else __syncwarp();
                }
            }
            float top[2] = {-INFINITY, -INFINITY}, corr[2] = {1.f, 1.f}, use[2];
#pragma unroll
            for (int x = 0; x < CK / 8; ++x) {
                top[0] = fmaxf(top[0], fmaxf(s[x][0], s[x][1]));
                top[1] = fmaxf(top[1], fmaxf(s[x][2], s[x][3]));
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2)) * sl2;
                if (top[e] > m_run[e] + CB_RESCALE_STEP) {
                    corr[e] = m_run[e] == -INFINITY ? 1.f : cb_exp2(m_run[e] - top[e]);      // (1: all is 0 yet, but for infinite values)
                    m_run[e] = top[e];
                }
                use[e] = m_run[e] == -INFINITY ? 0.f : m_run[e];
            }
            if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
                l_run[0] *= corr[0];
                l_run[1] *= corr[1];
#pragma unroll
                for (int x = 0; x < D / 8; ++x) {
                    o[x][0] *= corr[0], o[x][1] *= corr[0];
                    o[x][2] *= corr[1], o[x][3] *= corr[1];
                }
            }
#pragma unroll
            for (int y = 0; y < CK / 16; ++y) {
                unsigned p[4];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float f[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) f[e] = cb_exp2(fmaf(s[2 * y + x][e], sl2, -use[e >> 1]));
                    l_run[0] += f[0] + f[1];          // of this lane's keys
                    l_run[1] += f[2] + f[3];
                    p[2 * x] = cb_pack(f[0], f[1]);
                    p[2 * x + 1] = cb_pack(f[2], f[3]);
                }
#pragma unroll
                for (int x = 0; x < D / 16; ++x) {
                    unsigned b[4];
                    cb_ldsm_t(b, vs + cb_at<D>(y * 16 + (lm & 1) * 8 + l8, x * 2 + (lm >> 1)));
                    cb_mma(o[2 * x], p, b[0], b[1]);
                    cb_mma(o[2 * x + 1], p, b[2], b[3]);
                }
            }
        }
        asm volatile("cp.async.wait_group 0;\n" ::);
        __syncthreads();

        // the groups meet
        float* o_s = reinterpret_cast<float*>(cb_smem);      // [groups][M][D]
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = mt * 16 + r0 + 8 * e;
            float l = l_run[e];
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            if ((lane & 3) == 0) *reinterpret_cast<float2*>(ml + (group * M + row) * 2) = ch_left(m_run[e], l);
            if (row < place_in_line.tile.rows)
#pragma unroll
                for (int x = 0; x < D / 8; ++x)
                    *reinterpret_cast<float2*>(o_s + (group * M + row) * D + ((x * 8 + col) ^ ((row & 3) << 3))) = make_float2(o[x][2 * e], o[x][2 * e + 1]);
        }
        __syncthreads();
        w = place_in_line;
        const bool begins = w.k == 0, ends = w.k + n == w.tile.tiles;
        const size_t place = (size_t)2 * blockIdx.x + (begins ? 1 : 0);
        for (int i = tid; i < w.tile.rows * (D / 4); i += THREADS) {
            const int row = i / (D / 4), e = (i % (D / 4)) * 4;
            float2 g[CB_GROUPS];
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int x = 0; x < CB_GROUPS; ++x) {
                g[x] = *reinterpret_cast<const float2*>(ml + (x * M + row) * 2);
                m = fmaxf(m, g[x].x);
            }
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int x = 0; x < CB_GROUPS; ++x) {
                const float f = g[x].x == -INFINITY ? 0.f : cb_exp2(g[x].x - m);
                const float4 z = *reinterpret_cast<const float4*>(o_s + (x * M + row) * D + (e ^ ((row & 3) << 3)));
                l += f * g[x].y;
                y.x += f * z.x, y.y += f * z.y, y.z += f * z.z, y.w += f * z.w;
            }
            if constexpr (CLUSTER) {              // for the other blocks, where group 0's outputs were (this thread's alone to read)
                *reinterpret_cast<float4*>(o_s + row * D + (e ^ ((row & 3) << 3))) = y;
                if (e == 0) *reinterpret_cast<float2*>(cb_smem + S::block_ml_off + row * 8) = ch_left(m, l);
            } else if (begins && ends) {
                const float inv = ch_inverse(l);
                const int full = w.tile.row0 + row, t = fast_over(full, a.by_g), h = w.kh * a.G + full - t * a.G;
                store4<bf16>(reinterpret_cast<bf16*>(a.out) + ((size_t)(w.s0 + t) * a.H + h) * D + e,
                             make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
            } else {
                *reinterpret_cast<float4*>(a.part_o + (place * M + row) * D + e) = y;
                if (e == 0) *reinterpret_cast<float2*>(a.part_ml + (place * M + row) * 2) = ch_left(m, l);
            }
        }
        if constexpr (CLUSTER) {
            cg::cluster_group cluster = cg::this_cluster();
            cluster.sync();
            for (int i = rank * THREADS + tid; i < w.tile.rows * (D / 4); i += S_blocks * THREADS) {
                const int row = i / (D / 4), e = (i % (D / 4)) * 4;
                float m = -INFINITY, l = 0.f;
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                for (int b0 = 0; b0 < S_blocks; b0 += 4) {      // four blocks at a time, so that their reads are under way together
                    float2 g[4];
                    float4 z[4];
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const unsigned char* at = cluster.map_shared_rank(cb_smem, min(b0 + b, S_blocks - 1));
                        g[b] = *reinterpret_cast<const float2*>(at + S::block_ml_off + row * 8);
                        z[b] = *reinterpret_cast<const float4*>(at + (row * D + (e ^ ((row & 3) << 3))) * 4);
                        if (b0 + b >= S_blocks) g[b].x = -INFINITY;
                    }
                    const float top = fmaxf(m, fmaxf(fmaxf(g[0].x, g[1].x), fmaxf(g[2].x, g[3].x)));
                    const float was = m == -INFINITY ? 0.f : cb_exp2(m - top);
                    l *= was;
                    y.x *= was, y.y *= was, y.z *= was, y.w *= was;
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        if (g[b].x != -INFINITY) {
                            const float f = cb_exp2(g[b].x - top);
                            l += f * g[b].y;
                            y.x += f * z[b].x, y.y += f * z[b].y, y.z += f * z[b].z, y.w += f * z[b].w;
                        }
                    m = top;
                }
                const float inv = ch_inverse(l);
                const int full = w.tile.row0 + row, t = fast_over(full, a.by_g), h = w.kh * a.G + full - t * a.G;
                store4<bf16>(reinterpret_cast<bf16*>(a.out) + ((size_t)(w.s0 + t) * a.H + h) * D + e,
                             make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
            }
            cluster.sync();                   // the others have read this block's memory
            if ((w.m + 1) * M >= w.req.n * a.G) break;
            cb_part<S>(a, w, w.m + 1, rank, S_blocks);
        } else {
            if (begins && !ends && tid == 0) ch_leave<S>(a, w, blockIdx.x);
            if (!ch_next<S>(a, w, n)) break;
            __syncthreads();                  // the ring's memory is the next item's
        }
    }
    if (bad) atomicOr(a.err, bad);
}

template <int D> static int launch_chunk_bf16(const ChArgs& a, cudaStream_t st) {
    using S = CbShape<D>;
    auto kern = chunk_bf16_kernel<D, false>;
    const int C = a.blocks;
    static unsigned long long done = 0;
    ch_prepare(kern, S::bytes, &done);
    const int rc = (int)launch_pdl(kern, dim3(C), dim3(S::threads), S::bytes, st, a, 1);
    if (rc) return rc;
    return launch_chunk_join<bf16, S::M, D>(a, C, st);
}

template <int D> static int launch_chunk_clusters(const ChArgs& a, int blocks, cudaStream_t st) {
    using S = CbShape<D>;
    auto kern = chunk_bf16_kernel<D, true>;
    static unsigned long long done = 0;
    ch_prepare(kern, S::bytes, &done);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.R * a.K * blocks));
    cfg.blockDim = dim3(S::threads);
    cfg.dynamicSmemBytes = S::bytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)blocks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, kern, a, blocks);
}

// clusters 0: by the line, as many blocks as the call says (the host: two an SM).  clusters 2 .. 8: blocks of a cluster for every request and
// key head, no scratch.
extern "C" int aie_attention_chunks_bf16(const ChCall* call, int clusters, cudaStream_t stream) {
    if (call->R <= 0 || call->T <= 0) return 0;
    ChArgs a;
    const int rc = ch_args(call, 32, 64, 1, !clusters, &a);
    if (rc) return rc;
    if (a.d != 64 && a.d != 128) return AIE_UNSUPPORTED;
    if (!clusters) return a.d == 64 ? launch_chunk_bf16<64>(a, stream) : launch_chunk_bf16<128>(a, stream);
    if (clusters < 2 || clusters > 8 || (long long)a.R * a.K * clusters > 0x7fffffff) return AIE_UNSUPPORTED;
    return a.d == 64 ? launch_chunk_clusters<64>(a, clusters, stream) : launch_chunk_clusters<128>(a, clusters, stream);
}
