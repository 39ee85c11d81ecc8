// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Request r drafted n = draft_len[r] tokens x_0 .. x_(n-1) out of distributions q_0 .. q_(n-1) (null: each was certain of its
// token); rows q_start[r] .. q_start[r] + n of `target` are the target's distributions p_0 .. p_n at the same places.  Draft i is
// kept while u_i q_i(x_i) < p_i(x_i), u_i in [0, 1) (the product of two floats is exact in 64 bits, so nothing is rounded here).
// Behind the k kept ones one token is drawn, by v in [0, 1), from the weights
//     w = max(p_k - q_k, 0)   where draft k was refused,        w = p_n   where all were kept:
// the first token whose cumulative weight is above floor(v W), W the sum of all.  If every w is 0 (p_k nowhere above q_k: possible only
// by the rounding of their sums) the weights are p_k.  Which tokens come out then follows the target's distribution as far as the
// draws tell shares apart: u and v are float32, as a rule multiples of 2^-24, so a draft is kept, and a token drawn, with a probability that is off
// by up to 2^-24, and a token whose interval lies between two such multiples is never drawn; p_k - q_k is rounded to float32.
// Weights are integers, w clipped to 1 in units of 2^-48 rounded to nearest: 2^-49 is off at most, a float below 2^-25 of
// the largest mass, and sums are exact, the same whatever their order.  A drafted token outside the vocabulary is refused and takes nothing off p.
//
// What bounds it: one row of p and one of q a request (64 requests of 128,256 tokens: 14.3 us, 4.0 TB/s), and the chain of waits around
// them: lengths, the drafts' probabilities, the blocks' sums, a segment again (one request: 7.3 us).  A cluster of eight blocks shares a
// request's row: every warp adds up segments of 512 tokens (eight 16-byte loads a lane under way), the segments' sums stay in shared
// memory, the blocks' sums meet in everyone's shared memory, and the block that holds the wanted one looks for its segment and reads that
// once more.  Eight blocks because a row of 128,256 floats twice is 128 KB for each, about 2 us of what an SM can load.  At 64 registers a
// thread an SM holds one block of 1,024 threads or four of 256: up to 16 requests (two clusters of eight fit each of eight groups of SMs)
// take 1,024, which read their part of a row in one go, 17 to 32 take 512, more take 256, whose clusters are then all there at once.
#include <cooperative_groups.h>

#include "common.cuh"
#include "draft_args.h"

namespace cg = cooperative_groups;
typedef unsigned long long u64;

#define VD_CLUSTER 8
#define VD_SEGMENT 512          // tokens a warp adds up at a time: four of 16 bytes a lane, of each row
#define VD_MAX_SEGMENTS 256     // a block's: 1,048,576 tokens of vocabulary
#define VD_TOO_MUCH (~0ull)     // a sum that does not fit

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() {
    __syncwarp();                           // .aligned: a warp's threads come together, which what stands before may not have left them
    asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory");
}

// in units of 2^-48; NaN and what is negative weigh nothing
__device__ __forceinline__ u64 vd_fixed(float w) { return w > 0.f ? __float2ull_rn(fminf(w, 1.f) * 281474976710656.f) : 0ull; }

__device__ __forceinline__ u64 vd_warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// what is taken off p: nothing, the draft's row, or everything at one token
struct VdMinus {
    const float* row;
    int token;
};

// weights of the four tokens t .. t + 3; tokens from `V` on weigh nothing
template <bool VEC> __device__ __forceinline__ void vd_load(float (&x)[4], const float* row, int t, int V) {
    if (VEC && t + 4 <= V) {
        const float4 a = *reinterpret_cast<const float4*>(row + t);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = t + k < V ? row[t + k] : 0.f;
    }
}
// the weights of a warp's segment: lane l has tokens 128 j + 4 l .. + 3 of it
template <bool VEC> __device__ __forceinline__ void vd_segment(u64 (&w)[4][4], const float* p, const VdMinus& m, int t0, int V, int lane) {
    float a[4][4], b[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) vd_load<VEC>(a[j], p, t0 + 128 * j + 4 * lane, V);
    if (m.row)
#pragma unroll
        for (int j = 0; j < 4; ++j) vd_load<VEC>(b[j], m.row, t0 + 128 * j + 4 * lane, V);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float x = m.row ? a[j][k] - b[j][k] : a[j][k];
            w[j][k] = t0 + 128 * j + 4 * lane + k == m.token ? 0ull : vd_fixed(x);
        }
}

template <bool VEC, int VD_THREADS>
__global__ void __cluster_dims__(VD_CLUSTER, 1, 1) __launch_bounds__(VD_THREADS, 1024 / VD_THREADS)
verify_drafts_kernel(const float* target, long long target_row, int T, int V, const int* q_start,
                     const int* draft_tokens, const int* draft_len, const float* draft_probs,
                     long long draft_req, long long draft_place, int N, const float* accept_draws,
                     const float* token_draws, int* tokens, int* emitted, unsigned* err) {
    __shared__ u64 seg_sum[VD_MAX_SEGMENTS];
    __shared__ u64 warp_sum[VD_THREADS / 32];
    __shared__ u64 sums[2][VD_CLUSTER];     // of every block: of w, of p alone
    __shared__ int s_kept, s_token;         // drafts kept; the refused one's token, -1: all were kept, or it is outside the vocabulary
    cg::cluster_group cluster = cg::this_cluster();
    pdl_launch_dependents();
    pdl_wait();
    cluster_arrive();                       // (waited for before the first write to another block's memory: that it has started)
    const int r = blockIdx.x / VD_CLUSTER, rank = blockIdx.x % VD_CLUSTER;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // what the first decision needs, all asked for at once
    const int start = q_start[r];
    const int n = draft_len ? draft_len[r] : N;
    int x0 = 0;
    float u0 = 0.f;
    if (warp == 0 && lane < N) {
        x0 = draft_tokens[(size_t)r * N + lane];
        u0 = accept_draws[(size_t)r * N + lane];
    }
    const float v0 = token_draws[r];
    int* out = tokens + (size_t)r * (N + 1);
    const bool bad = n > N || (n >= 0 && (start < 0 || start > T - 1 - n));
    if (n < 0 || bad) {                     // an idle request, or rows that are not there: the same in all blocks of the cluster
        if (rank == 0) {
            for (int i = tid; i <= N; i += VD_THREADS) out[i] = -1;
            if (tid == 0) {
                emitted[r] = 0;
                if (bad) atomicOr(err, AIE_DEV_SLOT_OOB);
            }
        }
        cluster_wait();
        return;
    }

    // how many drafts are kept: a warp looks at 32 places at a time
    if (warp == 0) {
        int kept = n, token = -1;
        for (int base = 0; base < n; base += 32) {
            const int i = base + lane;
            bool refused = false;
            if (base > 0 && i < n) {
                x0 = draft_tokens[(size_t)r * N + i];
                u0 = accept_draws[(size_t)r * N + i];
            }
            if (i < n) {
                refused = true;
                if (x0 >= 0 && x0 < V) {
                    const float p = target[(start + i) * target_row + x0];
                    const float q = draft_probs ? draft_probs[r * draft_req + i * draft_place + x0] : 1.f;
                    refused = !((double)u0 * (double)q < (double)p);
                } else if (rank == 0) {
                    atomicOr(err, AIE_DEV_TOKEN_OOB);
                }
            }
            const unsigned any = __ballot_sync(0xffffffffu, refused);
            if (any) {
                kept = base + __ffs(any) - 1;
                token = __shfl_sync(0xffffffffu, x0, __ffs(any) - 1);
                if (token >= V) token = -1;
                break;
            }
        }
        if (lane == 0) {
            s_kept = kept;
            s_token = token;
        }
    }
    __syncthreads();
    const int kept = s_kept;
    const float* p = target + (start + kept) * target_row;
    VdMinus minus = {nullptr, -1};
    if (s_token >= 0) {                     // (a token outside the vocabulary came out of no distribution: nothing is taken off for it)
        if (draft_probs) minus.row = draft_probs + r * draft_req + kept * draft_place;
        else minus.token = s_token;
    }

    const int segments = (V + VD_SEGMENT - 1) / VD_SEGMENT, per = (segments + VD_CLUSTER - 1) / VD_CLUSTER;
    const int s0 = rank * per, mine = max(0, min(per, segments - s0));
    u64 before = 0, total = 0;
    int round = 0;
    for (;; ++round) {      // a second round only where something was taken off p and nothing is left: p by itself
        u64 sum = 0;
        for (int s = warp; s < mine; s += VD_THREADS / 32) {
            u64 w[4][4], a = 0;
            vd_segment<VEC>(w, p, minus, (s0 + s) * VD_SEGMENT, V, lane);
#pragma unroll
            for (int j = 0; j < 4; ++j) a += (w[j][0] + w[j][1]) + (w[j][2] + w[j][3]);
            a = vd_warp_sum(a);
            if (lane == 0) seg_sum[s] = a;
            sum += a;
        }
        if (lane == 0) warp_sum[warp] = sum;
        __syncthreads();
        if (round == 0) cluster_wait();
        if (tid < VD_CLUSTER) {                    // to block `tid`
            // a warp's sum is below 2^62; a block's from 2^60 on is that of no distribution, and would not fit when the blocks' are added
            u64 a = 0, high = 0;
#pragma unroll
            for (int w = 0; w < VD_THREADS / 32; ++w) {
                a += warp_sum[w];
                high += warp_sum[w] >> 32;
            }
            *cluster.map_shared_rank(&sums[round][rank], tid) = high >> 28 ? VD_TOO_MUCH : a;
        }
        cluster.sync();
        before = total = 0;
        bool fits = true;
#pragma unroll
        for (int b = 0; b < VD_CLUSTER; ++b) {
            const u64 a = sums[round][b];
            if (b < rank) before += a;
            total += a;
            fits = fits && a != VD_TOO_MUCH;
        }
        if (!fits) total = 0;
        if (total > 0 || round == 1 || s_token < 0) break;      // the same in all blocks
        minus.row = nullptr;
        minus.token = -1;
    }

    if (rank == 0) {
        for (int i = tid; i <= N; i += VD_THREADS)
            if (i != kept) out[i] = i < kept ? draft_tokens[(size_t)r * N + i] : -1;
        if (tid == 0) {
            emitted[r] = kept + 1;
            if (total == 0) {                      // a row of zeros, or of no probabilities: no token can be drawn from it
                out[kept] = 0;
                atomicOr(err, AIE_DEV_NO_MASS);
            }
        }
    }
    if (total > 0) {
        // total is below 2^53 for anything that sums to about 1, so the product is rounded once
        const double v = (double)v0;
        u64 goal = v > 0.0 ? (u64)(v * (double)total) : 0ull;
        if (goal > total - 1) goal = total - 1;
        const u64 here = sums[round][rank];
        if (warp == 0 && goal >= before && goal - before < here) {
            goal -= before;
            int s = 0;                             // the segment: 32 sums at a time
            for (int base = 0; base < mine; base += 32) {
                u64 a = base + lane < mine ? seg_sum[base + lane] : 0ull;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 b = __shfl_up_sync(0xffffffffu, a, o);
                    if (lane >= o) a += b;
                }
                const unsigned above = __ballot_sync(0xffffffffu, a > goal);
                if (above) {
                    const int at = __ffs(above) - 1;
                    const u64 prev = __shfl_sync(0xffffffffu, a, at > 0 ? at - 1 : 0);
                    if (at > 0) goal -= prev;
                    s = base + at;
                    break;
                }
                goal -= __shfl_sync(0xffffffffu, a, 31);
            }
            u64 w[4][4];
            const int t0 = (s0 + s) * VD_SEGMENT;
            vd_segment<VEC>(w, p, minus, t0, V, lane);
            bool found = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u64 a = (w[j][0] + w[j][1]) + (w[j][2] + w[j][3]);
                const u64 own = a;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const u64 b = __shfl_up_sync(0xffffffffu, a, o);
                    if (lane >= o) a += b;
                }
                const unsigned above = __ballot_sync(0xffffffffu, a > goal);
                if (!found && above) {
                    found = true;
                    if (lane == __ffs(above) - 1) {
                        u64 c = a - own;
                        int k = 0;
                        while (k < 3 && c + w[j][k] <= goal) c += w[j][k++];
                        out[kept] = t0 + 128 * j + 4 * lane + k;
                    }
                }
                if (!found) goal -= __shfl_sync(0xffffffffu, a, 31);
            }
        }
    }
}

extern "C" int aie_verify_drafts(const VdArgs* args, cudaStream_t stream) {
    const VdArgs& a = *args;
    if (a.R <= 0) return 0;
    if (a.V <= 0 || a.N < 0 || a.T < 0) return AIE_BAD_ARG;
    if (a.V > VD_CLUSTER * VD_MAX_SEGMENTS * VD_SEGMENT || a.R > 0x7fffffff / VD_CLUSTER) return -3;
    const bool vec = ((size_t)a.target | (size_t)a.draft_probs) % 16 == 0 && (a.target_row | a.draft_req | a.draft_place) % 4 == 0;
    const int threads = a.R <= 16 ? 1024 : a.R <= 32 ? 512 : 256;
    auto kern = threads == 1024 ? (vec ? verify_drafts_kernel<true, 1024> : verify_drafts_kernel<false, 1024>)
                : threads == 512 ? (vec ? verify_drafts_kernel<true, 512> : verify_drafts_kernel<false, 512>)
                                 : (vec ? verify_drafts_kernel<true, 256> : verify_drafts_kernel<false, 256>);
    return (int)launch_pdl(kern, dim3(a.R * VD_CLUSTER), dim3(threads), 0, stream,
                           a.target, a.target_row, a.T, a.V, a.q_start, a.draft_tokens, a.draft_len, a.draft_probs, a.draft_req,
                           a.draft_place, a.N, a.accept_draws, a.token_draws, a.tokens, a.emitted, a.err);
}
