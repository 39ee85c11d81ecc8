// Attention of new tokens over a paged cache (see attention_chunks.cuh) in bfloat16 on the fifth-generation tensor cores: heads of 64 and
// 128, items of up to 256 rows, for chunks of tokens whose rows fill the tiles of tcgen05.mma.
//   o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),   x_j = (q . k_j) * scale * log2 e
//
// A block stays on its SM and walks its share of the line of items.  Two streams of work run half a period apart on one tensor pipe, so that
// one's products run while the other's softmax does.  An item of more than 128 rows has a stream for each half of its rows, both over
// all key tiles; an item of 128 rows or fewer lets the streams take turns at the key tiles (its streams' outputs are added up at the end).
// Roles:
//   warps 0-3, 4-7   softmax of stream 0 / 1, a thread a row: the row of S in registers (tcgen05.ld), masked on tiles that
//                    touch the diagonal or a window's edge; its reference maximum moves by more than 8 (log2 units) or not at all, so that
//                    outputs are rarely rescaled; probabilities go as bfloat16 pairs over the scores in tensor memory;
//   warps 8, 10      keys, values by TMA: a box a page (128 keys of a larger page), in the order in which the products read them, into
//                    one ring of 128-key tiles of both that runs on from item to item.  A page that is not there has a box past the pool's
//                    end, which arrives as zeros.  (One warp for both spent 2,000 cycles a tile of eight pages on asking, more than
//                    the tile's bytes take at heads of 64.)
//   warp 9           issues the products: S = Q K^T and O += P V of a step of a stream, P from tensor memory, V as the MN-major
//                    operand; zeroes the values past a request's last key, since a probability of 0 must not meet what an unwritten slot
//                    holds, and what is not finite among those of keys that some rows do not see;
//   warp 11          queries: rows = (token, head of the group) gathered by cp.async into the swizzled tile that TMA would write (tokens
//                    and heads may lie any distance apart), ahead of the item that uses them where a place is free.
// Tensor memory: scores of stream t at columns 128 t (P over the first 64), outputs at 256 + 128 t.
// What bounds it: long chunks the exponentials (16 a cycle and SM: 2,048 cycles for two rows' tiles of 128 keys, against 2,048 of
// products; four requests of 300 to 500 tokens behind 6,000 to 9,000, 32 heads of 128: 226 to 229 us, 913 to 925 TFLOP/s, tensor pipe
// 0.51 busy; 273 us back to back under the power limit), few rows behind many keys the reading of those (four requests of 6 to 9 tokens
// behind 30,000: 92.5 us, 5.6 TB/s).  A call of any size takes 12 to 16 us more than its tiles: the start, the queries, the first tiles, the join.
// Probabilities are rounded to bfloat16 for the product with the values, as the values are; sums take them unrounded.
#include "attention_chunks.cuh"
#include "tc_rows.cuh"

#define CT_M 128
#define CT_KT 128
#define CT_THREADS 384
// named barriers: the probabilities of a step of stream t are in tensor memory.  Its steps take turns at two (t + 1 and t + 3): scores are asked
// for behind the step before, so a warp that has seen those of a step knows that the barrier of the step before that is over.
#define CT_BAR_P 1
#define CT_BARS 2
#define CT_BAR_MEET 5          // 5, 6: the two streams of an item of few rows
#define CT_RESCALE_STEP 8.0f

#ifndef CT_STRAY               // tile of values whose barrier waits for more bytes than come: for the test of a wait that runs out
#define CT_STRAY (-1)
#endif

template <int D> struct CtShape {
    static constexpr int M = 2 * CT_M, KT = CT_KT;     // rows of an item, keys of a tile
    // both streams take every key tile of an item of more than 128 rows, one of them that of a smaller one
    static constexpr int MAX_WEIGHT = 2;
    static __device__ __forceinline__ int weight(int rows) { return rows > CT_M ? 2 : 1; }
    static constexpr int tile = 128 * D * 2;           // bytes of 128 rows
    static constexpr int NS = D == 128 ? 5 : 10;       // tiles of keys or values in the ring
    // [3 KB: barriers, what the walk and the streams tell one another | queries x 2 | ring], 227 KB at heads of 128: nothing is left
    // for aligning the start, which the runtime puts on 1 KB as long as there is no other shared memory
    static constexpr int walk_off = 256, warps_off = 480, meet_off = 1024, q_off = 3 * 1024, kv_off = q_off + 2 * tile, bytes = kv_off + NS * tile;
};

// Adds to 32 columns of a row's outputs, from column c0 on, what is not finite among the values that the row sees of keys that not all of the
// item's rows see, in this block's share (n tiles from w.k on); they are read out of the pages again.
__device__ __forceinline__ void ct_add_unfinite(const ChArgs& a, const ChWalk& w, int n, int pos, int c0, unsigned (&ov)[32]) {
    const int first_pos = w.req.c + w.tile.i0, last_low = a.window > 0 ? w.req.c + w.tile.i1 - a.window + 1 : 0;
    const int k0 = (w.tile.first + w.k) * CT_KT, k1 = min(k0 + n * CT_KT, pos + 1);
#pragma unroll 1
    for (int key = k0; key < k1; ++key) {
        if (key >= last_low && key <= first_pos) {      // on to the keys that the first row does not see
            key = first_pos;
            continue;
        }
        const int in = fast_over(key, a.by_p), page = ch_sees(pos, key, a.window) ? a.table[(size_t)w.r * a.W + in] : -1;
        if (page < 0 || page >= a.num_pages) continue;
        const uint4* row = reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(a.v_pages) +
                                                          (((size_t)page * a.K + w.kh) * a.P + (key - in * a.P)) * a.d + c0);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const uint4 v4 = row[x];
            const unsigned v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned u = ch_unfinite(v[e]);
                const int i = x * 8 + e * 2;
                if (u & 0x8000u) ov[i] = __float_as_uint(__uint_as_float(ov[i]) + __uint_as_float(v[e] << 16));
                if (u >> 31) ov[i + 1] = __float_as_uint(__uint_as_float(ov[i + 1]) + __uint_as_float(v[e] & 0xffff0000u));
            }
        }
    }
}

// The order in which an item's tiles of keys (K) and values (V) pass through the ring: `ahead` tiles of keys, then V(j), K(j + ahead).
__device__ __forceinline__ int ct_ahead(const ChTile& t) { return t.rows > CT_M ? 1 : 2; }

template <int D>
__global__ void __launch_bounds__(CT_THREADS, 1)
chunk_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const ChArgs a, int end_group) {
    using S = CtShape<D>;
    static_assert(CT_BARS == 2, "whose turn it is is a bit a stream");
    constexpr int M = S::M, NS = S::NS, TILE = S::tile, HV = D / 64, GROUP = HV * 1024, PC = D / 8;
    extern __shared__ __align__(1024) unsigned char sm[];
    ChShared* sh = reinterpret_cast<ChShared*>(sm + S::walk_off);
    ChWalk* walks = reinterpret_cast<ChWalk*>(sm + S::warps_off);      // [8] where a softmax warp is, while its registers hold a row
    static_assert(sizeof(ChShared) <= S::warps_off - S::walk_off && 8 * sizeof(ChWalk) <= S::meet_off - S::warps_off, "places");
    float2(*meet)[CT_M] = reinterpret_cast<float2(*)[CT_M]>(sm + S::meet_off);      // [2] (m, l) of a row's two streams
    unsigned long long* full = reinterpret_cast<unsigned long long*>(sm);      // [NS]
    unsigned long long* empty = full + NS;          // [NS]
    unsigned long long* q_full = empty + NS;        // [2]
    unsigned long long* q_empty = q_full + 2;       // [2]
    unsigned long long* s_full = q_empty + 2;       // [2] the scores of a stream's step (and its products before them) are done
    unsigned long long* o_done = s_full + 2;        // [2] the last product of an item's stream is done
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(o_done + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    unsigned* unfinite = tmem_slot + 6;             // not 0: on some step of this block that not all rows see wholly, a value was not finite
    unsigned* armed = tmem_slot + 2;                // [2][2] tiles of the ring that the loaders asked for last, and of what phase (a bit each)
    unsigned char* q_s = sm + S::q_off;
    unsigned char* kv_s = sm + S::kv_off;

    // what needs nothing from the kernel before this one
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c = blockIdx.x, C = gridDim.x;
    if (tid == 0) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&q_full[t], 1);
            mbar_init(&q_empty[t], 1);
            mbar_init(&s_full[t], 1);
            mbar_init(&o_done[t], 1);
        }
        *abort_flag = 0;
        *unfinite = 0u;
        for (int i = 0; i < 4; ++i) armed[i] = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        tma_prefetch_map(&map_k);
        tma_prefetch_map(&map_v);
    }
    pdl_wait();
    if (tid == 0) a.meta[c] = make_int4(0, 0, 0, 0);
    if (tc_smem(sm) & 1023u) {                      // swizzled tiles would not be where the products look for them
        if (tid == 0) atomicOr(a.err, AIE_DEV_WAIT_TIMEOUT);
        return;
    }
    ChWalk w;
    if (!ch_begin<CT_THREADS, S>(a, c, C, sh, w)) return;
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc_smem(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    const unsigned tmem_base = *tmem_slot;

    // registers: the launch allots 168 to each of the 384 threads; the third warpgroup keeps 88 and the softmax warpgroups take 208
    // each, 88 + 2 x 208 = 3 x 168 (an increase waits for what a decrease has released)
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;\n");
        if (warp == 8 || warp == 10) {
            // keys / values.  In the ring an item's first L tiles of keys come first, then V(0), K(L), V(1), K(L + 1), .. and
            // the last tiles of values: the order in which the products read them
            const bool values = warp == 10;
            const CUtensorMap* map = values ? &map_v : &map_k;
            const int BP = min(a.P, CT_KT), boxes = CT_KT / BP;      // rows of a box; lane i asks for box i of a tile
            asm volatile("fence.proxy.async.global;\n" ::: "memory");      // the pages were written through the other proxy, by the kernels before
            int slot = 0, ph = 1;
            unsigned bad = 0, mine = 0, phase = 0;
            bool ok = true;
            auto skip = [&](int n) {                                 // n < NS
                slot += n;
                if (slot >= NS) {
                    slot -= NS;
                    ph ^= 1;
                }
            };
            for (;;) {
                const int n = ch_share<S>(w), L = min(ct_ahead(w.tile), n), kt0 = w.tile.first + w.k;
                const int hi = w.req.c + w.tile.i1 + 1, low = a.window > 0 ? w.req.c + w.tile.i0 - a.window + 1 : 0;
                const int* bt = a.table + (size_t)w.r * a.W;
                // the page of this lane's box of tile j (read some tiles ahead of its use), and its first group of 8 rows
                auto wanted = [&](int j) {
                    const int key = (kt0 + j) * CT_KT + lane * BP;
                    return j < n && lane < boxes && key < hi && key + BP > low;
                };
                auto page_of = [&](int j) { return wanted(j) ? bt[fast_over((kt0 + j) * CT_KT + lane * BP, a.by_p)] : -1; };
                auto group_of = [&](int j, int page) {
                    if (!wanted(j)) return end_group;
                    if (page >= 0 && page < a.num_pages) {
                        const int key = (kt0 + j) * CT_KT + lane * BP, in = key - fast_over(key, a.by_p) * a.P;
                        return (int)((((long long)page * a.K + w.kh) * a.P + in) >> 3);
                    }
                    bad |= AIE_DEV_PAGE_OOB;
                    return end_group;
                };
                int p1 = page_of(0), p2 = page_of(1);
                if (values) skip(L);
                for (int j = 0; j < n; ++j) {
                    const int p3 = page_of(j + 2), group = group_of(j, p1);
                    if (lane == 0 && ok) {
                        ok = mbar_wait(&empty[slot], (unsigned)ph, abort_flag, a.err);
                        if (ok) mbar_expect_tx(&full[slot], TILE + (values && j == CT_STRAY ? 16 : 0));
                    }
                    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                    if (!ok) break;
                    if (lane < boxes) tma_load_4d(kv_s + slot * TILE + lane * BP * (D * 2), map, &full[slot], 0, 0, 0, group);
                    mine |= 1u << slot;
                    phase = (phase & ~(1u << slot)) | (ph ? 0u : 1u << slot);
                    __syncwarp();
                    p1 = p2;
                    p2 = p3;
                    // to the next one: K(j) has a tile of values before it from K(L) on, V(j) one of keys behind it up to V(n - L - 1)
                    skip(values ? (j < n - L ? 2 : 1) : (j < L - 1 || j == n - 1 ? 1 : 2));
                }
                if (!ok) break;
                if (!values) skip(L);
                if (!ch_next<S>(a, w, n)) break;
            }
            if (lane == 0) {
                armed[2 * values] = mine;
                armed[2 * values + 1] = phase;
            }
            if (bad) atomicOr(a.err, bad);
        } else if (warp == 9) {
            // the whole warp walks the steps (it meets the softmax warps at named barriers); one lane issues
            const unsigned idesc_s = umma_idesc(CT_KT), idesc_o = umma_idesc(D, true);
            const unsigned long long dq0 = umma_desc(q_s), dk0 = umma_desc(kv_s, GROUP), dv0 = umma_desc_mn(kv_s, 1024, GROUP);
            const bool lead = tc_elect();
            bool ok = true;                 // that lane's; once false, the warp only keeps its appointments at the barriers
            int slot = 0, ph = 0, nq = 0;   // next tile of the ring, tiles of queries used so far
            unsigned turn = 0;              // bit t: at which of its barriers stream t hands over next
            auto scores = [&](int t, int qs, int ks_) {
                const unsigned long long dq = dq0 + (unsigned long long)((qs * TILE) >> 4), dk = dk0 + (unsigned long long)((ks_ * TILE) >> 4);
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    umma(tmem_base + (unsigned)(t * CT_KT), dq + (unsigned long long)((((ks >> 2) * 16384) >> 4) + 2 * (ks & 3)),
                         dk + (unsigned long long)((((ks >> 2) * 1024) >> 4) + 2 * (ks & 3)), idesc_s, ks > 0 ? 1u : 0u);
                umma_commit(&s_full[t]);      // covers the P V before: the softmax may rescale O once it sees it
            };
            auto outputs = [&](int t, int vs_, bool first) {
                const unsigned long long dv = dv0 + (unsigned long long)((vs_ * TILE) >> 4);
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)
                    umma_a_tmem(tmem_base + 256u + (unsigned)(t * 128), tmem_base + (unsigned)(t * CT_KT + ks * 8),
                                dv + (unsigned long long)((ks * 2 * GROUP) >> 4), idesc_o, (!first || ks > 0) ? 1u : 0u);
            };
            auto step = [&](int& s_, int& p_) {
                if (++s_ == NS) {
                    s_ = 0;
                    p_ ^= 1;
                }
            };
            for (;;) {
                const int n = ch_share<S>(w), L = ct_ahead(w.tile);
                const bool pair = L == 1, ends = w.k + n == w.tile.tiles;
                const int past = w.req.c + w.tile.i1 + 1 - (w.tile.first + w.tile.tiles - 1) * CT_KT;      // keys of the item's last tile
                const int first_pos = w.req.c + w.tile.i0, last_low = a.window > 0 ? w.req.c + w.tile.i1 - a.window + 1 : 0;
                const int kt0 = w.tile.first + w.k;
                const int q0 = nq & 1, q1 = pair ? q0 ^ 1 : q0, qp0 = (nq >> 1) & 1, qp1 = ((nq + 1) >> 1) & 1;
                if (lead && ok) {
                    ok = mbar_wait(&q_full[q0], (unsigned)qp0, abort_flag, a.err);
                    if (ok && pair) ok = mbar_wait(&q_full[q1], (unsigned)qp1, abort_flag, a.err);
                }
                nq += pair ? 2 : 1;
                for (int t = 0; t < L && t < n; ++t) {
                    if (lead && ok) {
                        ok = mbar_wait(&full[slot], (unsigned)ph, abort_flag, a.err);
                        if (ok) {
                            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                            scores(t, q0, slot);
                            if (pair) scores(1, q1, slot);
                            umma_commit(&empty[slot]);
                        }
                    }
                    step(slot, ph);
                }
                if (lead && ok && n <= L) {
                    umma_commit(&q_empty[q0]);
                    if (pair) umma_commit(&q_empty[q1]);
                }
                for (int j = 0; j < n; ++j) {
                    const int sv = slot, pv = ph;
                    const bool more = j + L < n;
                    step(slot, ph);
                    const int sk = slot, pk = ph;
                    if (more) step(slot, ph);
                    // operands first: as a rule they landed long ago, and nothing but the probabilities then stands
                    // between the end of a softmax and its products
                    if (lead && ok) {
                        ok = mbar_wait(&full[sv], (unsigned)pv, abort_flag, a.err);
                        if (ok && more) ok = mbar_wait(&full[sk], (unsigned)pk, abort_flag, a.err);
                    }
                    const int kbase = (kt0 + j) * CT_KT;
                    if (kbase + CT_KT - 1 > first_pos || kbase < last_low) {
                        // the keys past the request's end get zeros for values, and so does what is not finite among those of keys that
                        // some rows do not see: a probability of 0 must not meet it (the softmax warps add it to the rows that see it)
                        if (__ballot_sync(0xffffffffu, lead && ok)) {
                            const int keys = ends && j == n - 1 ? min(past, CT_KT) : CT_KT;
                            const int upto = max(0, min(last_low - kbase, keys)), from = max(upto, min(first_pos + 1 - kbase, keys));
                            auto piece = [&](int row) {      // of this lane, which looks at every 32 / PC-th row
                                const int x = lane % PC;
                                return reinterpret_cast<uint4*>(kv_s + sv * TILE + (row >> 3) * GROUP + (x >> 3) * 1024 + (row & 7) * 128 + (x & 7) * 16);
                            };
                            unsigned most = 0u;
#pragma unroll 1
                            for (int half = 0; half < 2; ++half)      // the first keys, the last ones
                                for (int row = (half ? from : 0) + lane / PC; row < (half ? keys : upto); row += 32 / PC) {
                                    const uint4 v = *piece(row);
                                    most = ch_larger(most, ch_larger(ch_larger(v.x, v.y), ch_larger(v.z, v.w)));
                                }
                            for (int row = keys + lane / PC; row < CT_KT; row += 32 / PC) *piece(row) = make_uint4(0, 0, 0, 0);
                            if (__any_sync(0xffffffffu, ch_unfinite(most) != 0)) {
#pragma unroll 1
                                for (int half = 0; half < 2; ++half)
#pragma unroll 1
                                    for (int row = (half ? from : 0) + lane / PC; row < (half ? keys : upto); row += 32 / PC) {
                                        const uint4 v = *piece(row);
                                        *piece(row) = make_uint4(ch_without(v.x, ch_unfinite(v.x)), ch_without(v.y, ch_unfinite(v.y)),
                                                                 ch_without(v.z, ch_unfinite(v.z)), ch_without(v.w, ch_unfinite(v.w)));
                                    }
                                if (lane == 0) atomicOr(unfinite, 1u);
                                __threadfence_block();
                            }
                            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                        }
                        __syncwarp();
                    }
                    for (int t = pair ? 0 : j & 1; t < 2; t += pair ? 1 : 2) {
                        // the softmax threads of a stream arrive, this warp waits: a hardware barrier, since an mbarrier test costs
                        // the issuing thread some hundred cycles while the tensor pipe reads shared memory
                        asm volatile("bar.sync %0, %1;\n" ::"r"(CT_BAR_P + t + 2 * (turn >> t & 1)), "r"(CT_M + 32) : "memory");
                        turn ^= 1u << t;
                        if (!lead || !ok) continue;
                        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                        outputs(t, sv, j < L);
                        if (more) scores(t, t == 0 ? q0 : q1, sk);
                        else umma_commit(&o_done[t]);
                    }
                    if (lead && ok) {
                        umma_commit(&empty[sv]);
                        if (more) {
                            umma_commit(&empty[sk]);
                            if (j + L == n - 1) {
                                umma_commit(&q_empty[q0]);
                                if (pair) umma_commit(&q_empty[q1]);
                            }
                        }
                    }
                }
                if (!ch_next<S>(a, w, n)) break;
            }
        } else {
            // queries: every lane has four rows (token, head) of an item's tile; rows beyond the item's are zeros
            int nq = 0;
            bool ok = true;
            for (; ok;) {
                const int n = ch_share<S>(w), tiles = w.tile.rows > CT_M ? 2 : 1;
                for (int t = 0; t < tiles && ok; ++t, ++nq) {
                    if (lane == 0) ok = mbar_wait(&q_empty[nq & 1], (unsigned)(((nq >> 1) & 1) ^ 1), abort_flag, a.err);
                    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                    if (!ok) break;
#pragma unroll
                    for (int x4 = 0; x4 < 4; ++x4) {
                        const int row = x4 * 32 + lane, at = t * CT_M + row;
                        const bool there = at < w.tile.rows;
                        const int fl = w.tile.row0 + (there ? at : 0), tok = fast_over(fl, a.by_g), g = fl - tok * a.G;
                        const bf16* src = reinterpret_cast<const bf16*>(a.q) + (w.s0 + tok) * a.q_token + (long long)(w.kh * a.G + g) * a.q_head;
                        // [halves of 64 columns][128 rows][128 bytes], 16-byte pieces permuted by row & 7
                        const unsigned d = tc_smem(q_s + (nq & 1) * TILE + row * 128);
#pragma unroll
                        for (int x = 0; x < PC; ++x)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n"
                                         ::"r"(d + (x >> 3) * 16384 + (((x & 7) ^ (row & 7)) << 4)), "l"(src + x * 8), "r"(there ? 16 : 0));
                    }
                    asm volatile("cp.async.wait_all;\n" ::: "memory");
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive_plain(&q_full[nq & 1]);
                }
                if (!ok || !ch_next<S>(a, w, n)) break;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;\n");
        const int t = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const unsigned lane_addr = (unsigned)(quarter * 32) << 16;
        const unsigned tmem_s = tmem_base + (unsigned)(t * CT_KT) + lane_addr, tmem_o = tmem_base + 256u + lane_addr;
        const bool plain = a.scale2 > 0.f;                             // else scores are scaled before they are masked
        const float sl2 = plain ? a.scale2 : 1.f;
        unsigned s_ph = 0, o_ph = 0;
        bool ok = true;
        for (;;) {
            const int n = ch_share<S>(w), kt0 = w.tile.first + w.k;
            const bool pair = w.tile.rows > CT_M;
            const int at = pair ? t * CT_M + row : row;                // row of the item
            const bool live = at - lane < w.tile.rows;                 // any row of this warp
            const int qpos = w.req.c + fast_over(w.tile.row0 + at, a.by_g);
            const int p_min = w.req.c + fast_over(w.tile.row0 + (pair ? t * CT_M : 0), a.by_g);
            const int low = a.window > 0 ? qpos - a.window + 1 : 0, low_last = a.window > 0 ? w.req.c + w.tile.i1 - a.window + 1 : 0;
            float m_run = -INFINITY, l_run = 0.f;
            bool first = true;
            if (lane == 0) walks[warp] = w;
            for (int j = pair ? 0 : t; j < n; j += pair ? 1 : 2, first = false) {
                // (a warp that gave up still comes to the barrier of every step: the issuing warp waits there without a limit)
                if (ok) {
                    if (lane == 0) ok = mbar_wait(&s_full[t], s_ph, abort_flag, a.err);
                    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                }
                s_ph ^= 1u;
                if (ok && live) {
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                    const int kbase = (kt0 + j) * CT_KT;
                    unsigned sv[128];
                    AT_LD32((sv + 0), tmem_s + 0u);
                    AT_LD32((sv + 32), tmem_s + 32u);
                    AT_LD32((sv + 64), tmem_s + 64u);
                    AT_LD32((sv + 96), tmem_s + 96u);
                    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
                    if (__builtin_expect(!plain, 0)) {
#pragma unroll
                        for (int i = 0; i < 128; ++i) sv[i] = __float_as_uint(__uint_as_float(sv[i]) * a.scale2);
                    }
                    if (kbase + CT_KT - 1 > p_min || kbase < low_last) {
#pragma unroll
                        for (int i = 0; i < 128; ++i)
                            if (kbase + i > qpos || kbase + i < low) sv[i] = 0xff800000u;
                    }
                    float x0 = -INFINITY, x1 = -INFINITY, x2 = -INFINITY, x3 = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 128; i += 8) {
                        x0 = at_max3(x0, __uint_as_float(sv[i]), __uint_as_float(sv[i + 1]));
                        x1 = at_max3(x1, __uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3]));
                        x2 = at_max3(x2, __uint_as_float(sv[i + 4]), __uint_as_float(sv[i + 5]));
                        x3 = at_max3(x3, __uint_as_float(sv[i + 6]), __uint_as_float(sv[i + 7]));
                    }
                    const float top = fmaxf(at_max3(x0, x1, x2), x3) * sl2;
                    float corr = 1.0f;
                    if (top > m_run + CT_RESCALE_STEP) {
                        corr = m_run == -INFINITY ? 0.f : exp2f(m_run - top);
                        m_run = top;
                    }
                    const float m_use = m_run == -INFINITY ? 0.f : m_run;
                    // (the product before has landed: the commit that announced these scores was issued after it)
                    if (!first && __any_sync(0xffffffffu, corr != 1.0f)) {
#pragma unroll
                        for (int c0 = 0; c0 < D; c0 += 32) {
                            unsigned ov[32];
                            AT_LD32(ov, tmem_o + (unsigned)(t * 128 + c0));
                            asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * corr);
                            AT_ST32(ov, tmem_o + (unsigned)(t * 128 + c0));
                        }
                    }
                    const unsigned long long sl2_2 = at_pack2(sl2, sl2), negm_2 = at_pack2(-m_use, -m_use);
                    unsigned long long sum_a = 0ull, sum_b = 0ull;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        unsigned pk[16];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            unsigned long long xx;
                            asm("fma.rn.f32x2 %0, %1, %2, %3;"
                                : "=l"(xx) : "l"(at_pack2(__uint_as_float(sv[32 * q + i]), __uint_as_float(sv[32 * q + i + 1]))), "l"(sl2_2), "l"(negm_2));
                            float e0, e1;
                            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(at_lo(xx)));
                            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(at_hi(xx)));
                            if (i & 2) asm("add.rn.f32x2 %0, %1, %2;" : "=l"(sum_b) : "l"(sum_b), "l"(at_pack2(e0, e1)));
                            else asm("add.rn.f32x2 %0, %1, %2;" : "=l"(sum_a) : "l"(sum_a), "l"(at_pack2(e0, e1)));
                            __nv_bfloat162 bb = __floats2bfloat162_rn(e0, e1);
                            pk[i >> 1] = *reinterpret_cast<unsigned*>(&bb);
                        }
                        AT_ST16(pk, tmem_s + (unsigned)(16 * q));
                    }
                    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(sum_a) : "l"(sum_a), "l"(sum_b));
                    l_run = l_run * corr + (at_lo(sum_a) + at_hi(sum_a));
                    asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
                }
                tc_hand_over(CT_BAR_P + t + 2 * (s_ph ^ 1u), CT_M + 32, ok);
            }
            // the item's end
            __syncwarp();
            w = walks[warp];
            if (!first) {
                if (ok) {
                    if (lane == 0) ok = mbar_wait(&o_done[t], o_ph, abort_flag, a.err);
                    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                }
                o_ph ^= 1u;
            }
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            const bool begins = w.k == 0, ends = w.k + n == w.tile.tiles, whole = begins && ends, there = ok && at < w.tile.rows;
            const int fl = w.tile.row0 + at, tok = fast_over(fl, a.by_g), h = w.kh * a.G + fl - tok * a.G;
            const size_t place = ((size_t)2 * c + (begins ? 1 : 0)) * M + at;
            bf16* dst = reinterpret_cast<bf16*>(a.out) + ((size_t)(w.s0 + tok) * a.H + h) * D;
            float f0 = 1.f, f1 = 0.f;                                  // of this stream's outputs, of the other's
            m_run = ch_left(m_run, l_run).x;
            if (!pair) {
                // both streams have read the same rows: each puts together half of the columns
                meet[t][row] = make_float2(m_run, l_run);
                asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
                asm volatile("bar.sync %0, %1;\n" ::"r"(CT_BAR_MEET), "r"(2 * CT_M) : "memory");
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                const float2 y = meet[t ^ 1][row];
                const float m = l_run == l_run && y.y == y.y ? fmaxf(m_run, y.x) : NAN;
                f0 = m_run == -INFINITY ? 0.f : exp2f(m_run - m);
                f1 = y.x == -INFINITY ? 0.f : exp2f(y.x - m);
                l_run = f0 * l_run + f1 * y.y;
                m_run = m;
            }
            // (set before the products whose end was waited for, by this stream or by the one that it met)
            const bool some_unfinite = *reinterpret_cast<volatile unsigned*>(unfinite) != 0u;
            if (live && ok) {
                const float inv = whole ? ch_inverse(l_run) : 1.f;
                f0 *= inv;
                f1 *= inv;
                const int from = pair ? 0 : t * (D / 2), to = pair ? D : from + D / 2;
#pragma unroll 1
                for (int c0 = from; c0 < to; c0 += 32) {
                    unsigned ov[32];
                    AT_LD32(ov, tmem_o + (unsigned)(t * 128 + c0));
                    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                    for (int i = 0; i < 32; ++i) ov[i] = f0 == 0.f ? 0u : __float_as_uint(__uint_as_float(ov[i]) * f0);
                    if (!pair) {
                        unsigned ow[32];
                        AT_LD32(ow, tmem_o + (unsigned)((t ^ 1) * 128 + c0));
                        asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
                        if (f1 != 0.f) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) + __uint_as_float(ow[i]) * f1);
                        }
                    }
                    if (__builtin_expect(some_unfinite, 0) && there) ct_add_unfinite(a, w, n, w.req.c + tok, c0, ov);
                    if (there && whole) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            unsigned pk[4];
#pragma unroll
                            for (int e = 0; e < 8; e += 2) {
                                __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(ov[i + e]), __uint_as_float(ov[i + e + 1]));
                                pk[e >> 1] = *reinterpret_cast<unsigned*>(&b);
                            }
                            *reinterpret_cast<uint4*>(dst + c0 + i) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                        }
                    } else if (there) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<uint4*>(a.part_o + place * D + c0 + i) = make_uint4(ov[i], ov[i + 1], ov[i + 2], ov[i + 3]);
                    }
                }
                if (there && !whole && (pair || t == 0)) *reinterpret_cast<float2*>(a.part_ml + place * 2) = make_float2(m_run, l_run);
            }
            if (begins && !ends && tid == 0 && ok) ch_leave<S>(a, w, c);
            asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            if (!pair) asm volatile("bar.sync %0, %1;\n" ::"r"(CT_BAR_MEET + 1), "r"(2 * CT_M) : "memory");      // both have read the outputs
            if (!ch_next<S>(a, w, n)) break;
        }
    }

    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    if (*abort_flag && tid < 2) {                   // copies that are still in flight are given a bounded time to land
        for (int s = 0; s < NS; ++s)
            if (armed[2 * tid] >> s & 1u)
                for (unsigned i = 0; i < TC_DRAIN_LIMIT && !mbar_try_wait(&full[s], armed[2 * tid + 1] >> s & 1u); ++i) {}
    }
    __syncthreads();
    if (warp == 9) {
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(512));
    }
}

template <int D> static int launch_chunk_tc(const ChArgs& a, cudaStream_t st) {
    const int C = a.blocks;
    using S = CtShape<D>;
    CUtensorMap mk, mv;
    const unsigned long long rows = (unsigned long long)a.num_pages * a.K * a.P;
    const int box = (a.P < CT_KT ? a.P : CT_KT) / 8;
    int rc = tc_make_map_rows8(&mk, a.k_pages, rows, D / 64, box);
    if (rc == 0) rc = tc_make_map_rows8(&mv, a.v_pages, rows, D / 64, box);
    if (rc) return rc;
    auto kern = chunk_tc_kernel<D>;
    static unsigned long long done = 0;
    ch_prepare(kern, S::bytes, &done);
    rc = (int)launch_pdl(kern, dim3(C), dim3(CT_THREADS), S::bytes, st, mk, mv, a, (int)(rows / 8));
    if (rc) return rc;
    return launch_chunk_join<bf16, S::M, D>(a, C, st);
}

// Scratch for items of 256 rows; the host gives it a block an SM.  Pages of 8 .. 128 keys that divide 128, or of a multiple of 128; up
// to 2^31 - 1 groups of 8 rows in a pool.
extern "C" int aie_attention_chunks_tc(const ChCall* call, cudaStream_t stream) {
    if (call->R <= 0 || call->T <= 0) return 0;
    ChArgs a;
    const int rc = ch_args(call, 128, CT_KT, 2, true, &a);
    if (rc) return rc;
    if (a.P % 8 || (CT_KT % a.P && a.P % CT_KT) || (long long)a.num_pages * a.K * a.P / 8 > 0x7ffffffe) return AIE_UNSUPPORTED;
    if (a.d == 64) return launch_chunk_tc<64>(a, stream);
    if (a.d == 128) return launch_chunk_tc<128>(a, stream);
    return AIE_UNSUPPORTED;
}
