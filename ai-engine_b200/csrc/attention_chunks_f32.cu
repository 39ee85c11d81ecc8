// Attention of new tokens over a paged cache (see attention_chunks.cuh) in true float32: float32 caches, and bfloat16
// ones whose head size the tensor-core kernels do not take.
//   o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),   x_j = (q . k_j) * scale * log2 e,   keys j <= position (and > position - window)
//
// A block has NG groups of four warps; of every key tile each group takes sixteen keys of its own through a ring of its own (cp.async), and
// each warp of a group has eight of the item's rows.  Groups meet only at an item's end.
// Scores: a 16-byte read of shared memory takes four cycles of the SM whatever lanes share, so a lane multiplies 4 keys x 4 rows: the lanes
// are 4 (keys) x 2 (rows) x 4 (parts of the head).  The parts' sums are then exchanged so that every lane ends with one key and four rows:
// its i-th key is the (i ^ part)-th of its four, and what a lane gives away lies in the same registers in all lanes.  (Two keys x two
// rows a lane: 512 cycles of reads a warp's step against 128 of multiply-adds, 47 us for the case below.)
// Outputs: a lane has D / 32 columns of the warp's rows, two rows an instruction (fma.rn.f32x2).
// What bounds it: these reads, twice what the packed multiply-adds beside them take: full items reach 30 TFLOP/s of 74.  3 to 7 tokens x 4
// heads behind 500 to 3,000 keys, 8 requests: 37.2 us, 14.5 TFLOP/s (their multiply-adds and their bytes take 9 each): items of 12 to 28 of 32 rows.
#include "attention_chunks.cuh"

typedef unsigned long long u64;

__device__ __forceinline__ u64 cf_fma2(u64 a, u64 b, u64 c) {
    u64 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ u64 cf_mul2(u64 a, u64 b) {
    u64 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float cf_exp2(float x) {      // 2^-22 relative; below 2^-126: 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float cf_larger(float a, float b) {      // in size; NaN where one of them is (the sign means nothing)
    float r;
    asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ u64 cf_pack(float lo, float hi) {
    u64 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 cf_both(u64 v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}

#define CF_ROWS 32      // of an item: four warps' eight

template <int D> struct CfShape {
    static constexpr int M = CF_ROWS;
    static constexpr int NG = D > 128 ? 2 : 4;       // groups of four warps
    static constexpr int threads = NG * 128;
    static constexpr int NST = D > 128 ? 2 : D > 64 ? 3 : 4;      // stages of a group's ring: 16 keys and their values each
    static constexpr int KT = NG * 16;               // keys of a tile
    // a tile takes as long as its warps with rows, and a part that does not depend on them
    static constexpr int MAX_WEIGHT = 8;
    static __device__ __forceinline__ int weight(int rows) { return 4 + (rows + 7) / 8; }
    static constexpr int KS = D + 4;                 // distance of two rows of keys or queries: eight of them lie in different banks
    static constexpr int stage = 16 * KS + 16 * D;   // floats
    static constexpr int PS = 12;                    // distance of two keys' probabilities
    static constexpr int q_off = NG * NST * stage, p_off = q_off + M * KS, ml_off = p_off + NG * 4 * 16 * PS, end = ml_off + NG * M * 2;
    static constexpr int bytes = end * 4;
    static_assert(NG * M * D <= NG * NST * stage && bytes <= 227 * 1024 - 256, "the groups' outputs meet in the ring's memory");
};

// four floats of a row at dst: asynchronously out of a float32 pool, by way of registers out of a bfloat16 one
__device__ __forceinline__ void cf_fetch(float* dst, const float* src, bool there) {
    const unsigned d = (unsigned)__cvta_generic_to_shared(dst);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(d), "l"(src), "r"(there ? 16 : 0));
}
__device__ __forceinline__ void cf_fetch(float* dst, const bf16* src, bool there) {
    *reinterpret_cast<float4*>(dst) = there ? load4<bf16>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
}

template <typename T, int D>
__global__ void __launch_bounds__(CfShape<D>::threads, 1) chunk_f32_kernel(const ChArgs a) {
    using S = CfShape<D>;
    constexpr int M = S::M, NG = S::NG, NST = S::NST, KT = S::KT, CH = D / 4, CL = D / 32, THREADS = S::threads;      // CL: columns of a lane
    extern __shared__ __align__(16) float cf_smem[];
    __shared__ ChShared sh;
    __shared__ ChWalk place_in_line;              // while the registers hold rows' outputs
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = warp % NG, mt = warp / NG, gt = mt * 32 + lane;      // mt: which eight rows
    const int c = blockIdx.x, C = gridDim.x;
    if (tid == 0) a.meta[c] = make_int4(0, 0, 0, 0);
    ChWalk w;
    if (!ch_begin<THREADS, S>(a, c, C, &sh, w)) return;
    float* ring = cf_smem + group * NST * S::stage;
    float* q_s = cf_smem + S::q_off;              // [M][KS]
    float* p_s = cf_smem + S::p_off + warp * 16 * S::PS;      // this warp's [16 keys][8]
    float* ml = cf_smem + S::ml_off;              // [NG][M][2]
    const T* kp = reinterpret_cast<const T*>(a.k_pages);
    const T* vp = reinterpret_cast<const T*>(a.v_pages);
    const int kq = lane & 3, rq = (lane >> 2) & 1, ds = lane >> 3;      // for the scores: keys kq + 4 i, rows 4 rq + r of the warp, part of the head
    const int key = kq + 4 * ds;                  // the one that this lane has in the end
    unsigned bad = 0;

    for (;;) {
        const int n = ch_share<S>(w);
        const int c0 = w.req.c, hi = c0 + w.tile.i1 + 1, low_all = a.window > 0 ? c0 + w.tile.i0 - a.window + 1 : 0;
        const int rows = w.tile.rows, row0 = w.tile.row0, kt0 = w.tile.first + w.k, kh = w.kh;
        const int* bt = a.table + (size_t)w.r * a.W;

        // eight threads copy a key: each every eighth piece; the pages of the next two stages' keys are read ahead
        const int my_key = group * 16 + (gt >> 3);
        auto page_of = [&](int i) {
            const int k_at = (kt0 + i) * KT + my_key;
            return i < n && k_at < hi && k_at >= low_all ? bt[fast_over(k_at, a.by_p)] : -1;
        };
        int page = page_of(0), page_next = page_of(1);
        // queries of the item: they land with the first stage
        for (int i = tid; i < M * CH; i += THREADS) {
            const int row = i / CH, ch = i - row * CH, e = ch * 4;
            const bool there = row < rows && e < a.d;
            const int full = row0 + (there ? row : 0), t = fast_over(full, a.by_g), g = full - t * a.G;
            cf_fetch(q_s + row * S::KS + e, reinterpret_cast<const T*>(a.q) + (w.s0 + t) * a.q_token + (long long)(kh * a.G + g) * a.q_head + (there ? e : 0), there);
        }
        auto issue = [&](int i, int slot) {
            if (i < n) {
                const int k_at = (kt0 + i) * KT + my_key;
                bool there = k_at < hi && k_at >= low_all;
                if (there && (page < 0 || page >= a.num_pages)) {
                    bad |= AIE_DEV_PAGE_OOB;
                    there = false;
                }
                const size_t row_at = there ? (((size_t)page * a.K + kh) * a.P + (k_at - fast_over(k_at, a.by_p) * a.P)) * a.d : 0;
                float* to = ring + slot * S::stage;
#pragma unroll
                for (int y = 0; y < CH / 8; ++y) {
                    const int ch = (gt & 7) + 8 * y;
                    const bool in = there && ch * 4 < a.d;
                    const size_t off = in ? row_at + ch * 4 : 0;
                    cf_fetch(to + (gt >> 3) * S::KS + ch * 4, kp + off, in);
                    cf_fetch(to + 16 * S::KS + (gt >> 3) * D + ch * 4, vp + off, in);
                }
                page = page_next;
                page_next = page_of(i + 2);
            }
            asm volatile("cp.async.commit_group;\n" ::);
        };
#pragma unroll
        for (int i = 0; i < NST - 1; ++i) issue(i, i);
        if (tid == 0) place_in_line = w;
        asm volatile("cp.async.wait_group %0;\n" ::"n"(NST - 2));
        __syncthreads();

        const bool live = mt * 8 < rows;          // any row of this warp
        float m_run[4], l_run[4];                 // of rows 8 mt + 4 rq + r
        int lim[4];                               // last key that a row sees (a row that is not there: the last one's)
        u64 o[2][2][CL];                          // rows 8 mt + 4 j + 2 e and the next, columns CL lane .. (128 further from the fifth on)
        const int reach = a.window > 0 ? a.window : 0x7fffffff;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            m_run[r] = -INFINITY;
            l_run[r] = 0.f;
            const int row = mt * 8 + rq * 4 + r;
            lim[r] = c0 + fast_over(row0 + min(row, rows - 1), a.by_g);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int x = 0; x < CL; ++x) o[j][0][x] = o[j][1][x] = 0ull;

        int slot = 0;
        for (int i = 0; i < n; ++i) {
            asm volatile("cp.async.wait_group %0;\n" ::"n"(NST - 2));
            // the stage is there for the whole group, and the group has read the one that the next copies go to
            asm volatile("bar.sync %0, 128;\n" ::"r"(1 + group) : "memory");
            issue(i + NST - 1, slot == 0 ? NST - 1 : slot - 1);
            const float* ks = ring + slot * S::stage;
            const float* vs = ks + 16 * S::KS;
            slot = slot + 1 == NST ? 0 : slot + 1;
            const int k_at = (kt0 + i) * KT + group * 16;
            if (k_at >= hi || !live) continue;
            float x[4];
            {
                u64 s2[4][4];
#pragma unroll
                for (int y = 0; y < 4; ++y)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s2[y][r] = 0ull;
                const float *k0 = ks + (kq + 4 * ds) * S::KS + ds * 4, *k1 = ks + (kq + 4 * (ds ^ 1)) * S::KS + ds * 4;
                const float *k2 = ks + (kq + 4 * (ds ^ 2)) * S::KS + ds * 4, *k3 = ks + (kq + 4 * (ds ^ 3)) * S::KS + ds * 4;
                const float* q0 = q_s + (mt * 8 + rq * 4) * S::KS + ds * 4;
#pragma unroll 2
                for (int ch = 0; ch < CH / 4; ++ch) {
                    const ulonglong2 kv[4] = {*reinterpret_cast<const ulonglong2*>(k0 + ch * 16), *reinterpret_cast<const ulonglong2*>(k1 + ch * 16),
                                              *reinterpret_cast<const ulonglong2*>(k2 + ch * 16), *reinterpret_cast<const ulonglong2*>(k3 + ch * 16)};
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const ulonglong2 q2 = *reinterpret_cast<const ulonglong2*>(q0 + r * S::KS + ch * 16);
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            s2[y][r] = cf_fma2(kv[y].x, q2.x, s2[y][r]);
                            s2[y][r] = cf_fma2(kv[y].y, q2.y, s2[y][r]);
                        }
                    }
                }
                float f[4][4];
#pragma unroll
                for (int y = 0; y < 4; ++y)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float2 t = cf_both(s2[y][r]);
                        f[y][r] = t.x + t.y;
                    }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    f[0][r] += __shfl_xor_sync(0xffffffffu, f[2][r], 16);
                    f[1][r] += __shfl_xor_sync(0xffffffffu, f[3][r], 16);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = f[0][r] + __shfl_xor_sync(0xffffffffu, f[1][r], 8);
            }
            const int at = k_at + key;
            float top[4], corr[4];
            bool edge = false;                    // some rows do not see some of these keys
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool sees = at <= lim[r] && lim[r] - at < reach;
                top[r] = x[r] = sees ? x[r] * a.scale2 : -INFINITY;
                edge = edge || !sees;
            }
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], b < 2 ? 1 << b : 2 << b));
            bool moved = false;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                // the reference moves by more than 8 or not at all: weights stay below 2^8, outputs are rarely rescaled
                corr[r] = 1.f;
                if (top[r] > m_run[r] + 8.f) {
                    corr[r] = m_run[r] == -INFINITY ? 0.f : cf_exp2(m_run[r] - top[r]);
                    m_run[r] = top[r];
                    moved = true;
                }
                x[r] = x[r] == -INFINITY ? 0.f : cf_exp2(x[r] - m_run[r]);
                l_run[r] = l_run[r] * corr[r] + x[r];          // of this lane's keys
            }
            *reinterpret_cast<float4*>(p_s + key * S::PS + rq * 4) = make_float4(x[0], x[1], x[2], x[3]);
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float f0 = __shfl_sync(0xffffffffu, corr[2 * e], 4 * j), f1 = __shfl_sync(0xffffffffu, corr[2 * e + 1], 4 * j);
                        const u64 ff = cf_pack(f0, f1);
#pragma unroll
                        for (int y = 0; y < CL; ++y) o[j][e][y] = cf_mul2(o[j][e][y], ff);
                    }
            }
            __syncwarp();
            auto values = [&](float (&v)[CL], int kk) {      // this lane's columns of key kk
                if constexpr (CL == 2) {
                    const float2 t = *reinterpret_cast<const float2*>(vs + kk * D + lane * 2);
                    v[0] = t.x, v[1] = t.y;
                } else {
#pragma unroll
                    for (int y = 0; y < CL / 4; ++y) {
                        const float4 t = *reinterpret_cast<const float4*>(vs + kk * D + (lane + 32 * y) * 4);
                        v[4 * y] = t.x, v[4 * y + 1] = t.y, v[4 * y + 2] = t.z, v[4 * y + 3] = t.w;
                    }
                }
            };
            auto product = [&](const float (&v)[CL], int kk) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const ulonglong2 p2 = *reinterpret_cast<const ulonglong2*>(p_s + kk * S::PS + j * 4);
#pragma unroll
                    for (int y = 0; y < CL; ++y) {
                        const u64 vv = cf_pack(v[y], v[y]);
                        o[j][0][y] = cf_fma2(p2.x, vv, o[j][0][y]);
                        o[j][1][y] = cf_fma2(p2.y, vv, o[j][1][y]);
                    }
                }
            };
            float v[CL];
            bool unfinite = false;
            if (__any_sync(0xffffffffu, edge)) {
                float most = 0.f;
#pragma unroll 4
                for (int kk = 0; kk < 16; ++kk) {
                    values(v, kk);
#pragma unroll
                    for (int y = 0; y < CL; ++y) most = cf_larger(most, v[y]);
                }
                unfinite = __any_sync(0xffffffffu, !isfinite(most));
            }
            if (__builtin_expect(!unfinite, 1)) {
#pragma unroll 4
                for (int kk = 0; kk < 16; ++kk) {
                    values(v, kk);
                    product(v, kk);
                }
            } else {
#pragma unroll 1
                for (int kk = 0; kk < 16; ++kk) {
                    values(v, kk);
                    float some[CL];
#pragma unroll
                    for (int y = 0; y < CL; ++y) some[y] = isfinite(v[y]) ? v[y] : 0.f;
                    product(some, kk);
#pragma unroll
                    for (int row = 0; row < 8; ++row) {
                        const int pos = place_in_line.req.c + fast_over(place_in_line.tile.row0 + mt * 8 + row, a.by_g);
                        if (!ch_sees(pos, k_at + kk, a.window)) continue;
#pragma unroll
                        for (int y = 0; y < CL; ++y) {
                            float2 t = cf_both(o[row >> 2][(row & 3) >> 1][y]);
                            if (!isfinite(v[y])) (row & 1 ? t.y : t.x) += v[y];
                            o[row >> 2][(row & 3) >> 1][y] = cf_pack(t.x, t.y);
                        }
                    }
                }
            }
            __syncwarp();
        }
        asm volatile("cp.async.wait_group 0;\n" ::);

        // the groups meet: every row's maximum, then outputs and sums
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float l = l_run[r];
#pragma unroll
            for (int b = 0; b < 4; ++b) l += __shfl_xor_sync(0xffffffffu, l, b < 2 ? 1 << b : 2 << b);
            if (key == 0) *reinterpret_cast<float2*>(ml + (group * M + mt * 8 + rq * 4 + r) * 2) = ch_left(m_run[r], l);
        }
        __syncthreads();
        w = place_in_line;
        float* o_s = cf_smem;                     // [NG][M][D]
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = mt * 8 + j * 4 + e;
                if (row >= w.tile.rows) continue;
                float f[CL];
#pragma unroll
                for (int x = 0; x < CL; ++x) f[x] = (e & 1) ? cf_both(o[j][e >> 1][x]).y : cf_both(o[j][e >> 1][x]).x;
                float* to = o_s + (group * M + row) * D;
                if constexpr (CL == 2) {
                    *reinterpret_cast<float2*>(to + lane * 2) = make_float2(f[0], f[1]);
                } else {
#pragma unroll
                    for (int x = 0; x < CL / 4; ++x)
                        *reinterpret_cast<float4*>(to + (lane + 32 * x) * 4) = make_float4(f[4 * x], f[4 * x + 1], f[4 * x + 2], f[4 * x + 3]);
                }
            }
        __syncthreads();
        const bool begins = w.k == 0, ends = w.k + n == w.tile.tiles;
        const size_t place = (size_t)2 * c + (begins ? 1 : 0);
        for (int i = tid; i < w.tile.rows * CH; i += THREADS) {
            const int row = i / CH, e = (i - row * CH) * 4;
            float m = -INFINITY, l = 0.f;
            float2 g[NG];
#pragma unroll
            for (int x = 0; x < NG; ++x) {
                g[x] = *reinterpret_cast<const float2*>(ml + (x * M + row) * 2);
                m = fmaxf(m, g[x].x);
            }
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int x = 0; x < NG; ++x) {
                const float f = g[x].x == -INFINITY ? 0.f : exp2f(g[x].x - m);
                const float4 z = *reinterpret_cast<const float4*>(o_s + (x * M + row) * D + e);
                l += f * g[x].y;
                y.x += f * z.x, y.y += f * z.y, y.z += f * z.z, y.w += f * z.w;
            }
            if (begins && ends) {
                const float inv = ch_inverse(l);
                const int full = w.tile.row0 + row, t = fast_over(full, a.by_g), h = w.kh * a.G + full - t * a.G;
                if (e < a.d)
                    store4<T>(reinterpret_cast<T*>(a.out) + ((size_t)(w.s0 + t) * a.H + h) * a.d + e,
                              make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
            } else {
                *reinterpret_cast<float4*>(a.part_o + (place * M + row) * D + e) = y;
                if (e == 0) *reinterpret_cast<float2*>(a.part_ml + (place * M + row) * 2) = ch_left(m, l);
            }
        }
        if (begins && !ends && tid == 0) ch_leave<S>(a, w, c);
        if (!ch_next<S>(a, w, n)) break;
        __syncthreads();                          // the ring's memory is the next item's
    }
    if (bad) atomicOr(a.err, bad);
}

template <typename T, int D> static int launch_chunk_f32(const ChArgs& a, cudaStream_t st) {
    using S = CfShape<D>;
    auto kern = chunk_f32_kernel<T, D>;
    const int C = a.blocks;
    static unsigned long long done = 0;
    ch_prepare(kern, S::bytes, &done);
    const int rc = (int)launch_pdl(kern, dim3(C), dim3(S::threads), S::bytes, st, a);
    if (rc) return rc;
    return launch_chunk_join<T, S::M, D>(a, C, st);
}

// The scratch is for items of 32 rows and a head size D rounded up to 64, 128 or 256; the host gives it a block an SM.
extern "C" int aie_attention_chunks_f32(const ChCall* call, int dtype, cudaStream_t stream) {
    if (call->R <= 0 || call->T <= 0) return 0;
    if (call->d <= 0 || call->d > 256 || call->d % 8) return AIE_UNSUPPORTED;
    ChArgs a;
    const int rc = ch_args(call, 32, 32, 8, true, &a);
    if (rc) return rc;
    const int w = a.d <= 64 ? 0 : a.d <= 128 ? 1 : 2;
    if (dtype == AIE_F32) return w == 0 ? launch_chunk_f32<float, 64>(a, stream) : w == 1 ? launch_chunk_f32<float, 128>(a, stream) : launch_chunk_f32<float, 256>(a, stream);
    if (dtype == AIE_BF16) return w == 0 ? launch_chunk_f32<bf16, 64>(a, stream) : w == 1 ? launch_chunk_f32<bf16, 128>(a, stream) : launch_chunk_f32<bf16, 256>(a, stream);
    return AIE_BAD_ARG;
}
