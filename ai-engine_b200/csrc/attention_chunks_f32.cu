// Attention of new tokens over a paged cache (see attention_chunks.cuh) in true float32: float32 caches, and bfloat16
// ones whose head size or pages the tensor-core kernels do not take.
//   o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),   x_j = (q . k_j) * scale * log2 e,   keys j <= position (and > position - window)
//
// A block has NW warps; of every key tile each warp takes eight keys of its own and keeps a running maximum, sum and output of all M rows
// for them, so that warps meet only at an item's end.  The loop over key tiles exists for 8, 16, 24 and 32 rows.  A warp's keys and values come through a ring of its own (cp.async, three stages).
// Scores: a lane has one key and every fourth row, products and sums two at a time (fma.rn.f32x2) along the head; outputs: a lane has
// D / 32 columns of all rows.  Operands are 16-byte reads of shared memory, most of them the same for many lanes:
// at 32 rows and heads of 128, 9 reads a step of 32 multiply-adds for the scores and 12 for 128 for the outputs.
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

template <int N> struct CfInt { static constexpr int value = N; };

template <int D> struct CfShape {
    static constexpr int M = D > 128 ? 16 : 32;      // rows of an item: M * D / 32 floats of output a lane
    static constexpr int NW = D > 128 ? 4 : 8;       // warps
    static constexpr int NST = D > 64 ? 3 : 2;       // stages of a warp's ring: 8 keys and their values each (two blocks an SM at 64)
    static constexpr int KT = NW * 8;                // keys of a tile
    static constexpr int stage = 2 * 8 * D;          // floats
    static constexpr int q_off = NW * NST * stage, p_off = q_off + M * D, ml_off = p_off + NW * 8 * M, end = ml_off + NW * M * 2;
    static constexpr int bytes = end * 4;
    static_assert(NW * M * D <= NW * NST * stage, "the warps' outputs meet in the ring's memory");
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
__global__ void __launch_bounds__(CfShape<D>::NW * 32) chunk_f32_kernel(const ChArgs a) {
    using S = CfShape<D>;
    constexpr int M = S::M, NW = S::NW, NST = S::NST, KT = S::KT, CH = D / 4, RJ = M / 4, CP = D / 64;      // CP: packed pairs of columns a lane
    extern __shared__ __align__(16) float cf_smem[];
    __shared__ ChShared sh;
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c = blockIdx.x, C = gridDim.x;
    if (tid == 0) a.meta[2 * c] = make_int4(0, 0, 0, 0);
    ChWalk w;
    if (!ch_begin<NW * 32, M, KT>(a, c, C, &sh, w)) return;
    float* ring = cf_smem + warp * NST * S::stage;
    float* q_s = cf_smem + S::q_off;              // [M][D], 16-byte pieces at (piece ^ row & 7)
    float* p_s = cf_smem + S::p_off + warp * 8 * M;      // this warp's [8 keys][M]
    float* ml = cf_smem + S::ml_off;              // [NW][M][2]
    const T* kp = reinterpret_cast<const T*>(a.k_pages);
    const T* vp = reinterpret_cast<const T*>(a.v_pages);
    const int key = lane & 7, rg = lane >> 3;     // for the scores: this lane's key, and its rows rg, rg + 4, ..
    unsigned bad = 0;

    for (;;) {
        const int n = ch_share(w);
        const ChTile tl = w.tile;
        const int c0 = w.req.c, s0 = w.s0, hi = c0 + tl.i1 + 1;
        // queries of the item
        for (int i = tid; i < M * CH; i += NW * 32) {
            const int row = i / CH, ch = i - row * CH, e = ch * 4;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row < tl.rows && e < a.d) {
                const int full = tl.row0 + row, t = ch_over(full, a.by_g), g = full - t * a.G;
                x = load4<T>(reinterpret_cast<const T*>(a.q) + (s0 + t) * a.q_token + (long long)(w.kh * a.G + g) * a.q_head + e);
            }
            *reinterpret_cast<float4*>(q_s + row * D + ((ch ^ (row & 7)) << 2)) = x;
        }
        __syncthreads();
        const int* bt = a.table + (size_t)w.r * a.W;
        const int kt0 = tl.first + w.k;

        auto issue = [&](int i) {
            if (i < n) {
                float* ks = ring + (i % NST) * S::stage;
                const int k_at = (kt0 + i) * KT + warp * 8 + (lane & 7);
                long long row_at = -1;
                if (k_at < hi && (a.window <= 0 || k_at > c0 + tl.i0 - a.window)) {
                    const int pi = ch_over(k_at, a.by_p), page = bt[pi];
                    if (page >= 0 && page < a.num_pages) row_at = ((long long)page * a.K + w.kh) * a.P + (k_at - pi * a.P);
                    else bad |= AIE_DEV_PAGE_OOB;
                }
                for (int x = lane; x < 8 * CH; x += 32) {
                    const int kk = x / CH, ch = x - kk * CH;
                    const long long ra = __shfl_sync(0xffffffffu, row_at, kk);
                    const bool there = ra >= 0 && ch * 4 < a.d;
                    const long long off = there ? ra * a.d + ch * 4 : 0;
                    const int to = kk * D + ((ch ^ kk) << 2);
                    cf_fetch(ks + to, kp + off, there);
                    cf_fetch(ks + 8 * D + to, vp + off, there);
                }
            }
            asm volatile("cp.async.commit_group;\n" ::);
        };

        float m_run[RJ], l_run[RJ];
        int lim[RJ], low[RJ];                     // a row sees the keys from low + 1 to lim
        u64 o[M][CP];
#pragma unroll
        for (int j = 0; j < RJ; ++j) {
            m_run[j] = -INFINITY;
            l_run[j] = 0.f;
            const int row = j * 4 + rg, pos = c0 + ch_over(tl.row0 + row, a.by_g);
            lim[j] = row < tl.rows ? pos : -1;
            low[j] = a.window > 0 ? pos - a.window : -1;
        }
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
            for (int x = 0; x < CP; ++x) o[i][x] = 0ull;

#pragma unroll
        for (int i = 0; i < NST - 1; ++i) issue(i);
        // fours of rows that are there, rounded up to eights: a loop for each number, without branches between its loads
        auto walk = [&](auto fours) {
            constexpr int JN = decltype(fours)::value;
            for (int i = 0; i < n; ++i) {
                issue(i + NST - 1);
                asm volatile("cp.async.wait_group %0;\n" ::"n"(NST - 1));
                __syncwarp();
                const float* ks = ring + (i % NST) * S::stage;
                const float* vs = ks + 8 * D;
                u64 s2[JN];
#pragma unroll
                for (int j = 0; j < JN; ++j) s2[j] = 0ull;
#pragma unroll 4
                for (int ch = 0; ch < CH; ++ch) {
                    const ulonglong2 k2 = *reinterpret_cast<const ulonglong2*>(ks + key * D + ((ch ^ key) << 2));
#pragma unroll
                    for (int j = 0; j < JN; ++j) {
                            const int row = j * 4 + rg;
                            const ulonglong2 q2 = *reinterpret_cast<const ulonglong2*>(q_s + row * D + ((ch ^ (row & 7)) << 2));
                            s2[j] = cf_fma2(k2.x, q2.x, s2[j]);
                            s2[j] = cf_fma2(k2.y, q2.y, s2[j]);
                        }
                }
                const int k_at = (kt0 + i) * KT + warp * 8 + key;
                float top[JN];
#pragma unroll
                for (int j = 0; j < JN; ++j) {
                    const float2 f = cf_both(s2[j]);
                    top[j] = k_at <= lim[j] && k_at > low[j] ? (f.x + f.y) * a.scale2 : -INFINITY;
                    s2[j] = cf_pack(top[j], 0.f);
                }
#pragma unroll
                for (int b = 1; b < 8; b <<= 1)
#pragma unroll
                    for (int j = 0; j < JN; ++j) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], b));
                float corr[JN];
                bool moved = false;
#pragma unroll
                for (int j = 0; j < JN; ++j) {
                    // the reference moves by more than 8 or not at all: weights stay below 2^8, outputs are rarely rescaled
                    corr[j] = 1.f;
                    if (top[j] > m_run[j] + 8.f) {
                        corr[j] = m_run[j] == -INFINITY ? 0.f : exp2f(m_run[j] - top[j]);
                        m_run[j] = top[j];
                        moved = true;
                    }
                    const float x = cf_both(s2[j]).x, p = x == -INFINITY ? 0.f : exp2f(x - m_run[j]);
                    l_run[j] = l_run[j] * corr[j] + p;          // of this lane's keys
                    p_s[key * M + j * 4 + rg] = p;
                }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int i2 = 0; i2 < 4 * JN; ++i2) {
                        const float f = __shfl_sync(0xffffffffu, corr[i2 >> 2], (i2 & 3) * 8);
                        const u64 ff = cf_pack(f, f);
#pragma unroll
                        for (int x = 0; x < CP; ++x) o[i2][x] = cf_mul2(o[i2][x], ff);
                    }
                }
                __syncwarp();
#pragma unroll 2
                for (int kk = 0; kk < 8; ++kk) {
                    u64 v2[CP];
                    if constexpr (CP == 1) {
                        v2[0] = *reinterpret_cast<const u64*>(vs + kk * D + (((lane >> 1) ^ kk) << 2) + (lane & 1) * 2);
                    } else {
#pragma unroll
                        for (int x = 0; x < CP / 2; ++x) {
                            const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(vs + kk * D + (((lane + 32 * x) ^ kk) << 2));
                            v2[2 * x] = t.x;
                            v2[2 * x + 1] = t.y;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < JN; ++j) {
                            const float4 p4 = *reinterpret_cast<const float4*>(p_s + kk * M + j * 4);
                            const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const u64 pp = cf_pack(p[e], p[e]);
#pragma unroll
                                for (int x = 0; x < CP; ++x) o[j * 4 + e][x] = cf_fma2(pp, v2[x], o[j * 4 + e][x]);
                            }
                        }
                }
                __syncwarp();
            }
        };
        if (tl.rows <= 8) walk(CfInt<2>());
        else if (tl.rows <= 16 || RJ == 4) walk(CfInt<4>());
        else if (tl.rows <= 24) walk(CfInt<RJ < 6 ? RJ : 6>());
        else walk(CfInt<RJ>());
        asm volatile("cp.async.wait_group 0;\n" ::);

        // the warps meet: every row's maximum, then outputs and sums
#pragma unroll
        for (int j = 0; j < RJ; ++j) {
            float l = l_run[j];
#pragma unroll
            for (int b = 1; b < 8; b <<= 1) l += __shfl_xor_sync(0xffffffffu, l, b);
            if (key == 0) {
                ml[(warp * M + j * 4 + rg) * 2] = m_run[j];
                ml[(warp * M + j * 4 + rg) * 2 + 1] = l;
            }
        }
        __syncthreads();
        float* o_s = cf_smem;                     // [NW][M][D]
#pragma unroll
        for (int i = 0; i < M; ++i)
            if (i < tl.rows) {
                if constexpr (CP == 1) {
                    *reinterpret_cast<u64*>(o_s + (warp * M + i) * D + lane * 2) = o[i][0];
                } else {
#pragma unroll
                    for (int x = 0; x < CP / 2; ++x)
                        *reinterpret_cast<ulonglong2*>(o_s + (warp * M + i) * D + (lane + 32 * x) * 4) = make_ulonglong2(o[i][2 * x], o[i][2 * x + 1]);
                }
            }
        __syncthreads();
        const bool begins = w.k == 0, ends = w.k + n == tl.tiles;
        const size_t slot = (size_t)2 * c + (begins ? 1 : 0);
        for (int i = tid; i < tl.rows * CH; i += NW * 32) {
            const int row = i / CH, e = (i - row * CH) * 4;
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int x = 0; x < NW; ++x) m = fmaxf(m, ml[(x * M + row) * 2]);
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int x = 0; x < NW; ++x) {
                const float mx = ml[(x * M + row) * 2], f = mx == -INFINITY ? 0.f : exp2f(mx - m);
                const float4 z = *reinterpret_cast<const float4*>(o_s + (x * M + row) * D + e);
                l += f * ml[(x * M + row) * 2 + 1];
                y.x += f * z.x, y.y += f * z.y, y.z += f * z.z, y.w += f * z.w;
            }
            if (begins && ends) {
                const float inv = ch_inverse(l);
                const int full = tl.row0 + row, t = ch_over(full, a.by_g), h = w.kh * a.G + full - t * a.G;
                if (e < a.d)
                    store4<T>(reinterpret_cast<T*>(a.out) + ((size_t)(s0 + t) * a.H + h) * a.d + e,
                              make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
            } else {
                *reinterpret_cast<float4*>(a.part_o + (slot * M + row) * D + e) = y;
                if (e == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * M + row) * 2) = make_float2(m, l);
            }
        }
        if (begins && !ends && tid == 0) ch_leave(a, w, c, n);
        if (!ch_next<M, KT>(a, w, n)) break;
        __syncthreads();                          // the ring's memory is the next item's
    }
    if (bad) atomicOr(a.err, bad);
}

template <typename T, int D> static int launch_chunk_f32(const ChArgs& a, int C, cudaStream_t st) {
    using S = CfShape<D>;
    auto kern = chunk_f32_kernel<T, D>;
    static unsigned long long done = 0;
    ch_prepare(kern, S::bytes, &done);
    const int rc = (int)launch_pdl(kern, dim3(C), dim3(S::NW * 32), S::bytes, st, a);
    if (rc) return rc;
    return launch_chunk_join<T, S::M, D>(a, C, st);
}

// Rows of an item, and blocks of the kernel.  The scratch is [2 * blocks * rows * (D + 2)] floats and [2 * blocks] int4, D the head size
// rounded up to 64, 128 or 256.
extern "C" int aie_attention_chunks_f32_rows(int d) { return d > 128 ? CfShape<256>::M : CfShape<128>::M; }
extern "C" int aie_attention_chunks_f32_blocks(int d) { return aie_sm_count() * (d <= 64 ? 2 : 1); }

extern "C" int aie_attention_chunks_f32(const ChCall* call, int dtype, cudaStream_t stream) {
    if (call->R <= 0 || call->T <= 0) return 0;
    if (call->d <= 0 || call->d > 256 || call->d % 8) return AIE_UNSUPPORTED;
    ChArgs a;
    const int rc = ch_args(call, 16, 32, &a);
    if (rc) return rc;
    const int C = aie_attention_chunks_f32_blocks(a.d), w = a.d <= 64 ? 0 : a.d <= 128 ? 1 : 2;
    if (dtype == AIE_F32) return w == 0 ? launch_chunk_f32<float, 64>(a, C, stream) : w == 1 ? launch_chunk_f32<float, 128>(a, C, stream) : launch_chunk_f32<float, 256>(a, C, stream);
    if (dtype == AIE_BF16) return w == 0 ? launch_chunk_f32<bf16, 64>(a, C, stream) : w == 1 ? launch_chunk_f32<bf16, 128>(a, C, stream) : launch_chunk_f32<bf16, 256>(a, C, stream);
    return AIE_BAD_ARG;
}
