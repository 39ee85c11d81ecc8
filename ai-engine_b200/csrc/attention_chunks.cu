// Attention of new tokens over a paged cache (see attention_chunks.cuh) in bfloat16, heads of 64 and 128, for items of up to 32 rows:
// a few drafted tokens of a request times the query heads of a key head.
//   o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),   x_j = (q . k_j) * scale * log2 e
//
// What bounds it: reading keys and values once.  Products go through mma.sync, whose tiles of 16 rows fit 4 tokens of 4 heads: at 16 rows they
// need a fifth of the time that the bytes take.  A block has four warps; of every key tile each warp takes CK keys of its own through a ring
// of its own (cp.async, stages of 8 KB), so that warps meet only at an item's end, where their outputs are added up in shared memory.
// Queries are read as fragments out of shared memory.  Scores, maxima and sums are float32; probabilities are rounded to bfloat16 for the
// product with the values, as the values are, which the result's own rounding hides (2^-9 each on average).
#include "attention_chunks.cuh"

#define CB_WARPS 4
#define CB_STAGES 3

template <int D, int MT> struct CbShape {
    static constexpr int M = 16 * MT;                 // rows of an item
    static constexpr int CK = D == 64 ? 32 : 16;      // keys of a warp's stage
    static constexpr int KT = CB_WARPS * CK;          // keys of a tile
    static constexpr int stage = 2 * CK * D;          // elements: keys, then values
    static constexpr int ring_bytes = CB_WARPS * CB_STAGES * stage * 2;
    static constexpr int q_off = ring_bytes, ml_off = q_off + M * D * 2, bytes = ml_off + CB_WARPS * M * 2 * 4;
    static_assert(CB_WARPS * M * D * 4 <= ring_bytes, "the warps' outputs meet in the ring's memory");
};

__device__ __forceinline__ void cb_fetch(void* dst, const void* src, bool there) {
    const unsigned d = (unsigned)__cvta_generic_to_shared(dst);
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;\n" ::"r"(d), "l"(src), "r"(there ? 16 : 0));
}
__device__ __forceinline__ void cb_ldsm(unsigned (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"((unsigned)__cvta_generic_to_shared(p)));
}
__device__ __forceinline__ void cb_ldsm_t(unsigned (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"((unsigned)__cvta_generic_to_shared(p)));
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
// row r, 16-byte piece c of rows of D elements: pieces are permuted so that eight rows' pieces lie in different banks
template <int D> __device__ __forceinline__ bf16* cb_at(bf16* base, int row, int piece) { return base + row * D + ((piece ^ (row & 7)) << 3); }

template <int D, int MT>
__global__ void __launch_bounds__(CB_WARPS * 32, 2) chunk_bf16_kernel(const ChArgs a) {
    using S = CbShape<D, MT>;
    constexpr int M = S::M, KT = S::KT, CK = S::CK, PC = D / 8, NST = CB_STAGES;
    extern __shared__ __align__(128) unsigned char cb_smem[];
    __shared__ ChShared sh;
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c = blockIdx.x, C = gridDim.x;
    if (tid == 0) a.meta[2 * c] = make_int4(0, 0, 0, 0);
    ChWalk w;
    if (!ch_begin<CB_WARPS * 32, M, KT>(a, c, C, &sh, w)) return;
    bf16* ring = reinterpret_cast<bf16*>(cb_smem) + warp * NST * S::stage;
    bf16* q_s = reinterpret_cast<bf16*>(cb_smem + S::q_off);
    float* ml = reinterpret_cast<float*>(cb_smem + S::ml_off);      // [warps][M][2]
    const bf16* kp = reinterpret_cast<const bf16*>(a.k_pages);
    const bf16* vp = reinterpret_cast<const bf16*>(a.v_pages);
    const int r0 = lane >> 2, col = (lane & 3) * 2;      // of a 16 x 8 accumulator: rows r0 and r0 + 8, columns col and col + 1
    const int lm = lane >> 3, l8 = lane & 7;             // ldmatrix: matrix and row that this lane points at
    unsigned bad = 0;

    for (;;) {
        const int n = ch_share(w);
        const ChTile tl = w.tile;
        const int c0 = w.req.c, s0 = w.s0, hi = c0 + tl.i1 + 1;
        const int* bt = a.table + (size_t)w.r * a.W;
        const int kt0 = tl.first + w.k;
        const int low_all = a.window > 0 ? c0 + tl.i0 - a.window + 1 : 0;      // first key that any row sees

        auto issue = [&](int i) {
            if (i < n) {
                bf16* ks = ring + (i % NST) * S::stage;
                bf16* vs = ks + CK * D;
                const int k_at = (kt0 + i) * KT + warp * CK + (lane & (CK - 1));
                long long row_at = -1;
                if (k_at < hi && k_at >= low_all) {
                    const int pi = ch_over(k_at, a.by_p), page = __ldg(bt + pi);
                    if (page >= 0 && page < a.num_pages) row_at = ((long long)page * a.K + w.kh) * a.P + (k_at - pi * a.P);
                    else bad |= AIE_DEV_PAGE_OOB;
                }
#pragma unroll
                for (int x = 0; x < CK * PC / 32; ++x) {
                    const int kk = (lane + 32 * x) / PC, pc = (lane + 32 * x) % PC;
                    const long long ra = __shfl_sync(0xffffffffu, row_at, kk);
                    const size_t off = ra >= 0 ? (size_t)ra * D + pc * 8 : 0;
                    cb_fetch(cb_at<D>(ks, kk, pc), kp + off, ra >= 0);
                    cb_fetch(cb_at<D>(vs, kk, pc), vp + off, ra >= 0);
                }
            }
            asm volatile("cp.async.commit_group;\n" ::);
        };
#pragma unroll
        for (int i = 0; i < NST - 1; ++i) issue(i);

        // queries of the item
        for (int i = tid; i < M * PC; i += CB_WARPS * 32) {
            const int row = i / PC, pc = i % PC;
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (row < tl.rows) {
                const int full = tl.row0 + row, t = ch_over(full, a.by_g), g = full - t * a.G;
                x = *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(a.q) + (s0 + t) * a.q_token +
                                                    (long long)(w.kh * a.G + g) * a.q_head + pc * 8);
            }
            *reinterpret_cast<uint4*>(cb_at<D>(q_s, row, pc)) = x;
        }
        __syncthreads();

        float m_run[MT][2], l_run[MT][2], o[MT][D / 8][4];
        int pos[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m_run[mt][e] = -INFINITY;
                l_run[mt][e] = 0.f;
                pos[mt][e] = c0 + ch_over(tl.row0 + mt * 16 + r0 + 8 * e, a.by_g);
            }
#pragma unroll
            for (int x = 0; x < D / 8; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[mt][x][e] = 0.f;
        }
        const int last_low = a.window > 0 ? c0 + tl.i1 - a.window + 1 : 0;      // first key that the last row sees

        for (int i = 0; i < n; ++i) {
            issue(i + NST - 1);
            asm volatile("cp.async.wait_group %0;\n" ::"n"(NST - 1));
            __syncwarp();
            bf16* ks = ring + (i % NST) * S::stage;
            bf16* vs = ks + CK * D;
            const int k_at = (kt0 + i) * KT + warp * CK;
            if (k_at < hi) {
                float s[MT][CK / 8][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int x = 0; x < CK / 8; ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[mt][x][e] = 0.f;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    unsigned qa[MT][4];
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) cb_ldsm(qa[mt], cb_at<D>(q_s, mt * 16 + (lm & 1) * 8 + l8, kk * 2 + (lm >> 1)));
#pragma unroll
                    for (int x = 0; x < CK / 16; ++x) {
                        unsigned b[4];
                        cb_ldsm(b, cb_at<D>(ks, x * 16 + (lm >> 1) * 8 + l8, kk * 2 + (lm & 1)));
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            cb_mma(s[mt][2 * x], qa[mt], b[0], b[1]);
                            cb_mma(s[mt][2 * x + 1], qa[mt], b[2], b[3]);
                        }
                    }
                }
                const bool masked = k_at + CK - 1 > c0 + tl.i0 || k_at < last_low;
                unsigned p[MT][CK / 16][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int x = 0; x < CK / 8; ++x)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float v = s[mt][x][e] * a.scale2;
                            if (masked) {
                                const int key = k_at + x * 8 + col + (e & 1), q = pos[mt][e >> 1];
                                if (key > q || (a.window > 0 && key <= q - a.window)) v = -INFINITY;
                            }
                            s[mt][x][e] = v;
                            top[e >> 1] = fmaxf(top[e >> 1], v);
                        }
                    float corr[2], use[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
                        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
                        const float m_new = fmaxf(m_run[mt][e], top[e]);
                        use[e] = m_new == -INFINITY ? 0.f : m_new;
                        corr[e] = m_run[mt][e] == m_new ? 1.f : cb_exp2(m_run[mt][e] - use[e]);
                        m_run[mt][e] = m_new;
                        l_run[mt][e] *= corr[e];
                    }
#pragma unroll
                    for (int x = 0; x < CK / 8; ++x) {
                        float f[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) f[e] = cb_exp2(s[mt][x][e] - use[e >> 1]);
                        l_run[mt][0] += f[0] + f[1];          // of this lane's keys
                        l_run[mt][1] += f[2] + f[3];
                        p[mt][x >> 1][(x & 1) * 2] = cb_pack(f[0], f[1]);
                        p[mt][x >> 1][(x & 1) * 2 + 1] = cb_pack(f[2], f[3]);
                    }
                    if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
                        for (int x = 0; x < D / 8; ++x) {
                            o[mt][x][0] *= corr[0], o[mt][x][1] *= corr[0];
                            o[mt][x][2] *= corr[1], o[mt][x][3] *= corr[1];
                        }
                    }
                }
#pragma unroll
                for (int y = 0; y < CK / 16; ++y)
#pragma unroll
                    for (int x = 0; x < D / 16; ++x) {
                        unsigned b[4];
                        cb_ldsm_t(b, cb_at<D>(vs, y * 16 + (lm & 1) * 8 + l8, x * 2 + (lm >> 1)));
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            cb_mma(o[mt][2 * x], p[mt][y], b[0], b[1]);
                            cb_mma(o[mt][2 * x + 1], p[mt][y], b[2], b[3]);
                        }
                    }
            }
            __syncwarp();      // the stage is free again
        }
        asm volatile("cp.async.wait_group 0;\n" ::);
        __syncthreads();

        // the warps meet
        float* o_s = reinterpret_cast<float*>(cb_smem);      // [warps][M][D]
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = mt * 16 + r0 + 8 * e;
                float l = l_run[mt][e];
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                if ((lane & 3) == 0) *reinterpret_cast<float2*>(ml + (warp * M + row) * 2) = make_float2(m_run[mt][e], l);
                if (row < tl.rows)
#pragma unroll
                    for (int x = 0; x < D / 8; ++x)
                        *reinterpret_cast<float2*>(o_s + (warp * M + row) * D + x * 8 + col) = make_float2(o[mt][x][2 * e], o[mt][x][2 * e + 1]);
            }
        __syncthreads();
        const bool begins = w.k == 0, ends = w.k + n == tl.tiles;
        const size_t slot = (size_t)2 * c + (begins ? 1 : 0);
        for (int i = tid; i < tl.rows * (D / 4); i += CB_WARPS * 32) {
            const int row = i / (D / 4), e = (i % (D / 4)) * 4;
            float2 g[CB_WARPS];
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int x = 0; x < CB_WARPS; ++x) {
                g[x] = *reinterpret_cast<const float2*>(ml + (x * M + row) * 2);
                m = fmaxf(m, g[x].x);
            }
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int x = 0; x < CB_WARPS; ++x) {
                const float f = g[x].x == -INFINITY ? 0.f : cb_exp2(g[x].x - m);
                const float4 z = *reinterpret_cast<const float4*>(o_s + (x * M + row) * D + e);
                l += f * g[x].y;
                y.x += f * z.x, y.y += f * z.y, y.z += f * z.z, y.w += f * z.w;
            }
            if (begins && ends) {
                const float inv = ch_inverse(l);
                const int full = tl.row0 + row, t = ch_over(full, a.by_g), h = w.kh * a.G + full - t * a.G;
                store4<bf16>(reinterpret_cast<bf16*>(a.out) + ((size_t)(s0 + t) * a.H + h) * D + e,
                             make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
            } else {
                *reinterpret_cast<float4*>(a.part_o + (slot * M + row) * D + e) = y;
                if (e == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * M + row) * 2) = make_float2(m, l);
            }
        }
        if (begins && !ends && tid == 0) ch_leave(a, w, c, n);
        if (!ch_next<M, KT>(a, w, n)) break;
        __syncthreads();                      // the ring's memory is the next item's
    }
    if (bad) atomicOr(a.err, bad);
}

template <int D, int MT> static int launch_chunk_bf16(const ChArgs& a, int C, cudaStream_t st) {
    using S = CbShape<D, MT>;
    auto kern = chunk_bf16_kernel<D, MT>;
    static unsigned long long done = 0;
    ch_prepare(kern, S::bytes, &done);
    const int rc = (int)launch_pdl(kern, dim3(C), dim3(CB_WARPS * 32), S::bytes, st, a);
    if (rc) return rc;
    return launch_chunk_join<bf16, S::M, D>(a, C, st);
}

// Blocks of the kernels: two an SM.  The scratch is [2 * blocks * rows * (d + 2)] floats and [2 * blocks] int4.
extern "C" int aie_attention_chunks_bf16_blocks() { return 2 * aie_sm_count(); }

// rows: 16 or 32 of an item
extern "C" int aie_attention_chunks_bf16(const ChCall* call, int rows, cudaStream_t stream) {
    if (call->R <= 0 || call->T <= 0) return 0;
    ChArgs a;
    const int rc = ch_args(call, 16, 64, &a);
    if (rc) return rc;
    const int C = aie_attention_chunks_bf16_blocks();
    if (a.d == 64 && rows == 16) return launch_chunk_bf16<64, 1>(a, C, stream);
    if (a.d == 64 && rows == 32) return launch_chunk_bf16<64, 2>(a, C, stream);
    if (a.d == 128 && rows == 16) return launch_chunk_bf16<128, 1>(a, C, stream);
    if (a.d == 128 && rows == 32) return launch_chunk_bf16<128, 2>(a, C, stream);
    return AIE_UNSUPPORTED;
}
