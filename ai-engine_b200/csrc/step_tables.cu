// The lists of a step, made on the device from the requests' lengths: pages handed out, block tables, first tokens,
// positions, requests and cache slots of the tokens.
//
// Request r holds cached[r] tokens in held[r] pages and brings counts[r] more.  In the order of the requests
//   need[r]    = max(ceil((cached[r] + counts[r]) / P) - held[r], 0)         pages it is short of
//   q_start[r] = counts[0] + .. + counts[r - 1],   upto[r] = need[0] + .. + need[r]
//   granted[r] = need[r] == 0 or upto[r] <= free_count
// (a request that has to wait for pages makes those behind it that need some wait too).  A granted request takes
// its pages from the end of the free list, the first of them free_pages[free_count - 1 - (upto[r] - need[r])].
//
// What bounds it: nothing but the launch and two rounds to memory for small steps (8 requests: 3.6 us), writing the table for large ones
// (512 requests of 2,048 entries, 15,700 tokens: 6.7 us; bytes 1.0).  So that one launch does it, every block adds up the lengths of all
// requests by itself (512 at a time; 12 bytes a request out of L2) and keeps what its tokens and table rows ask of them in shared memory;
// then the grid shares out the table, a warp taking pieces of 512 entries of a row (four 16-byte loads a lane under way), and the tokens,
// which find their request by bisection.
#include "common.cuh"
#include "draft_args.h"

#define ST_THREADS 512
#define ST_MAX_REQUESTS 4096      // 16 bytes of shared memory each

struct StRow {       // what a block keeps of a request
    int q_start;     // its first token, INT_MAX where that is beyond 32 bits
    int held;        // pages it came with
    int first;       // place in the free list of the first page that it takes
    int now;         // pages it has after the step, or ~held where it has to wait
};

__device__ __forceinline__ long long st_shfl_up(long long v, int o) { return __shfl_up_sync(0xffffffffu, v, o); }

template <bool VEC>
__global__ void __launch_bounds__(ST_THREADS, 2)
step_tables_kernel(const int* cached, const int* counts, const int* held_in,
                   const int* tables_in, const int* free_pages, const int* free_count, int R, int W,
                   int F, int P, int num_pages, int capacity, int table_blocks, int* tables, int* held,
                   int* free_left, int* q_start, int* q_len, int* positions,
                   int* token_req, int* slots, unsigned* err) {
    extern __shared__ StRow rows[];
    __shared__ long long w_tokens[ST_THREADS / 32], w_pages[ST_THREADS / 32];
    __shared__ long long s_taken;
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned bad = 0;
    if (tid == 0) s_taken = 0;
    int avail = *free_count;
    if (avail < 0 || avail > F) { bad |= AIE_DEV_SLOT_OOB; avail = avail < 0 ? 0 : F; }

    long long tokens_before = 0, pages_before = 0;      // of all requests before them
    for (int base = 0; base < R; base += ST_THREADS) {
        const int r = base + tid;
        long long n = 0, need = 0;
        int h = 0, c = 0;
        bool fits = true;
        if (r < R) {
            n = counts[r];
            h = held_in[r];
            c = cached[r];
            if (n < 0 || c < 0 || h < 0 || h > W || c + n > 0x7fffffffll) {      // (n is 64 bits wide)
                bad |= AIE_DEV_SLOT_OOB;
                n = 0;
                c = 0;
                h = h < 0 ? 0 : min(h, W);
            }
            if (n > 0) need = ((long long)c + n + P - 1) / P - h;
            if (need < 0) need = 0;
            if (h + need > W) { bad |= AIE_DEV_SLOT_OOB; fits = false; need = 0; }
        }
        long long tok = n, pag = need;       // inclusive sums over these requests
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long a = st_shfl_up(tok, o), b = st_shfl_up(pag, o);
            if (lane >= o) { tok += a; pag += b; }
        }
        __syncthreads();          // the pass before has read the warps' sums
        if (lane == 31) { w_tokens[warp] = tok; w_pages[warp] = pag; }
        __syncthreads();
        long long all_tok = 0, all_pag = 0;
#pragma unroll
        for (int w = 0; w < ST_THREADS / 32; ++w) {
            if (w == warp) { tok += all_tok; pag += all_pag; }
            all_tok += w_tokens[w];
            all_pag += w_pages[w];
        }
        tok += tokens_before;
        pag += pages_before;
        tokens_before += all_tok;
        pages_before += all_pag;
        if (r < R) {
            if (n > 0 && tok > capacity) { bad |= AIE_DEV_SLOT_OOB; fits = false; }
            const bool granted = fits && (need == 0 || pag <= avail);
            const long long at = tok - n;
            StRow s;
            s.q_start = (int)(at < 0x7fffffff ? at : 0x7fffffff);
            s.held = h;
            s.first = granted ? (int)(avail - 1 - (pag - need)) : 0;
            s.now = granted ? h + (int)need : ~h;
            rows[r] = s;
            // requests that take pages come before all that wait for some: the largest sum of a granted one is what is taken
            if (granted && need > 0) atomicMax(&s_taken, pag);
            if (blockIdx.x == 0) {
                q_start[r] = s.q_start;
                q_len[r] = granted ? (int)n : 0;
                held[r] = h + (granted ? (int)need : 0);
            }
        }
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) *free_left = avail - (int)s_taken;
    const int total = (int)(tokens_before < capacity ? tokens_before : capacity);

    if ((int)blockIdx.x < table_blocks) {
        // entry w of row r: what it held, then the pages it takes, then -1
        constexpr int V = VEC ? 4 : 1, U = 4, PIECE = 32 * V * U;
        const unsigned pieces = (W + PIECE - 1) / PIECE, tasks = R * pieces;
        for (unsigned i = blockIdx.x * (ST_THREADS / 32) + warp; i < tasks; i += table_blocks * (ST_THREADS / 32)) {
            const unsigned r = i / pieces;
            const int w0 = (int)(i - r * pieces) * PIECE + lane * V;
            const StRow s = rows[r];
            const int now = s.now < 0 ? ~s.now : s.now;
            const int* from = tables_in + (size_t)r * W;
            int* to = tables + (size_t)r * W;
            int4 e[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int w = w0 + u * 32 * V;
                e[u] = make_int4(-1, -1, -1, -1);
                if (VEC ? w + V <= s.held : w < s.held) {
                    if (VEC) e[u] = *reinterpret_cast<const int4*>(from + w);
                    else e[u].x = from[w];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int w = w0 + u * 32 * V;
                if (w >= W) continue;
                if (w + V > s.held && w < now) {      // the rows' ends
                    int* x = reinterpret_cast<int*>(&e[u]);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        if (w + k < s.held) x[k] = from[w + k];
                        else if (w + k < now) {
                            x[k] = free_pages[s.first - (w + k - s.held)];
                            if (x[k] < 0 || x[k] >= num_pages) bad |= AIE_DEV_PAGE_OOB;
                        }
                    }
                }
                if (VEC) *reinterpret_cast<int4*>(to + w) = e[u];
                else to[w] = e[u].x;
            }
        }
    } else {
        const int stride = (gridDim.x - table_blocks) * ST_THREADS;
        for (int t = (blockIdx.x - table_blocks) * ST_THREADS + tid; t < capacity; t += stride) {
            int pos = -1, req = -1, slot = -1;
            if (t < total) {
                int lo = 0, hi = R - 1;      // the last request whose first token is at or before t
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (rows[mid].q_start <= t) lo = mid;
                    else hi = mid - 1;
                }
                const StRow s = rows[lo];
                const long long p = (long long)cached[lo] + t - s.q_start;
                req = lo;
                pos = (int)(p < 0x7fffffff ? p : 0x7fffffff);
                if (s.now >= 0) {
                    const int w = pos / P;      // below now: the request's tokens fit its pages
                    const int page = w < s.held ? tables_in[(size_t)lo * W + w] : free_pages[s.first - (w - s.held)];
                    if (page >= 0 && page < num_pages) slot = page * P + (pos - w * P);
                    else bad |= AIE_DEV_PAGE_OOB;
                }
            }
            positions[t] = pos;
            token_req[t] = req;
            slots[t] = slot;
        }
    }
    if (bad) atomicOr(err, bad);
}

extern "C" int aie_step_tables(const StArgs* args, cudaStream_t stream) {
    const StArgs& a = *args;
    const int R = a.R, W = a.W, capacity = a.capacity;
    if (R <= 0 || W <= 0 || a.F < 0 || a.P <= 0 || a.num_pages < 0 || capacity < 0) return AIE_BAD_ARG;
    if (R > ST_MAX_REQUESTS) return -3;
    int* held = a.out + (size_t)R * W;
    int *free_left = held + R, *q_start = free_left + 1, *q_len = q_start + R, *positions = q_len + R, *token_req = positions + capacity,
        *slots = token_req + capacity;
    const bool vec = W % 4 == 0 && ((size_t)a.tables_in | (size_t)a.out) % 16 == 0;
    const int most = 2 * aie_sm_count();
    const int piece = vec ? 512 : 128, warps = ST_THREADS / 32;
    const long long tb = ((long long)R * ((W + piece - 1) / piece) + warps - 1) / warps, kb = (capacity + ST_THREADS - 1) / ST_THREADS;
    const int table_blocks = (int)(tb < most ? tb : most), token_blocks = (int)(kb < most ? kb : most);
    auto kern = vec ? step_tables_kernel<true> : step_tables_kernel<false>;
    // more than 48 KB with what the kernel has besides; told once on each device
    static unsigned long long done[2] = {0, 0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= 64 || !(done[vec] >> dev & 1))) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, ST_MAX_REQUESTS * (int)sizeof(StRow));
        if (e == cudaSuccess && dev < 64) done[vec] |= 1ull << dev;
    }
    if (e != cudaSuccess) return (int)e;
    const size_t smem = (size_t)R * sizeof(StRow);
    return (int)launch_pdl(kern, dim3(table_blocks + token_blocks), dim3(ST_THREADS), smem, stream, a.cached, a.counts, a.held_in, a.tables_in,
                           a.free_pages, a.free_count, R, W, a.F, a.P, a.num_pages, capacity, table_blocks, a.out, held, free_left, q_start,
                           q_len, positions, token_req, slots, a.err);
}
