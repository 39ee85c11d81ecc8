// Keys and values of a step's tokens written to their cache slots: row t of k and v goes to page slots[t] / P, place
// slots[t] % P of a layer's pool [pages][kv heads][P][d].  Rows may be columns of a fused projection (any distance between
// tokens and between heads) and are rounded once where the cache holds fewer bits.  A negative slot leaves its row out.
//
// What bounds it: memory (8,191 tokens of 8 heads of 128 in bfloat16: 12.7 us, 5.3 TB/s; 40 tokens: 2.2 us).  A thread moves units of eight
// consecutive elements of one head (16 bytes of bfloat16), four of them under way, the loads of its rows asked for before the slots are
// known.
#include "common.cuh"
#include "division.cuh"
#include "draft_args.h"

#define CW_THREADS 256
#define CW_UNITS 4      // units of a thread under way

template <typename T, int V> struct CwVec { T e[V]; };

// V consecutive elements: 16-byte accesses when V is 8, single ones when it is 1
template <typename T, int V> __device__ __forceinline__ void cw_load(CwVec<T, V>& v, const T* p) {
    if constexpr (V == 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(v.e)[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    } else {
        v.e[0] = *p;
    }
}

template <typename I, typename C, int V>
__global__ void __launch_bounds__(CW_THREADS)
write_kv_slots_kernel(const I* k, const I* v, long long k_token, long long k_head, long long v_token,
                      long long v_head, C* k_pages, C* v_pages, const int* slots,
                      unsigned total, unsigned per_plane, FastDiv by_token, FastDiv by_head, FastDiv by_p, int P, int K, int d, int n_slots,
                      unsigned* err) {
    pdl_launch_dependents();
    pdl_wait();
    const unsigned first = blockIdx.x * (CW_THREADS * CW_UNITS) + threadIdx.x, per_head = d / V;
    alignas(16) CwVec<I, V> x[CW_UNITS];
    int slot[CW_UNITS], head[CW_UNITS], at[CW_UNITS];      // head: K and more for values; at: element of the head
#pragma unroll
    for (int u = 0; u < CW_UNITS; ++u) {
        const unsigned i = first + u * CW_THREADS;
        slot[u] = -1;
        if (i < total) {
            const unsigned t = fast_over(i, by_token), unit = i - t * (2 * per_plane), h = fast_over(unit, by_head);
            head[u] = (int)h;
            at[u] = (int)(unit - h * per_head) * V;
            const bool is_v = (int)h >= K;
            slot[u] = slots[t];
            cw_load<I, V>(x[u], is_v ? v + t * v_token + (long long)(h - K) * v_head + at[u] : k + t * k_token + (long long)h * k_head + at[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < CW_UNITS; ++u) {
        if (slot[u] < 0) continue;
        if (slot[u] >= n_slots) { atomicOr(err, AIE_DEV_PAGE_OOB); continue; }
        const bool is_v = head[u] >= K;
        const int page = (int)fast_over((unsigned)slot[u], by_p);
        C* to = (is_v ? v_pages : k_pages) + (((size_t)page * K + (is_v ? head[u] - K : head[u])) * P + (slot[u] - page * P)) * d + at[u];
        if constexpr (V == 8) {
            alignas(16) CwVec<C, V> y;
#pragma unroll
            for (int j = 0; j < V; ++j) y.e[j] = from_f32<C>(to_f32<I>(x[u].e[j]));
#pragma unroll
            for (int j = 0; j < (int)sizeof(C) / 2; ++j) reinterpret_cast<uint4*>(to)[j] = reinterpret_cast<const uint4*>(y.e)[j];
        } else {
            *to = from_f32<C>(to_f32<I>(x[u].e[0]));
        }
    }
}

template <typename I, typename C, int V>
static int launch_write(const void* k, const void* v, long long kt, long long kh, long long vt, long long vh, void* kp, void* vp,
                        const int* slots, int T, int num_pages, int P, int K, int d, unsigned* err, cudaStream_t st) {
    const long long total = (long long)T * 2 * K * (d / V);
    if (total > 0x7ffffc00) return -3;
    const unsigned blocks = (unsigned)((total + CW_THREADS * CW_UNITS - 1) / (CW_THREADS * CW_UNITS)), per_plane = (unsigned)(K * (d / V));
    return (int)launch_pdl(write_kv_slots_kernel<I, C, V>, dim3(blocks), dim3(CW_THREADS), 0, st, (const I*)k, (const I*)v, kt, kh, vt, vh,
                           (C*)kp, (C*)vp, slots, (unsigned)total, per_plane, fast_div(2 * per_plane), fast_div((unsigned)(d / V)),
                           fast_div((unsigned)P), P, K, d, num_pages * P, err);
}

template <typename I, typename C>
static int launch_write_rows(bool wide, const void* k, const void* v, long long kt, long long kh, long long vt, long long vh, void* kp,
                             void* vp, const int* slots, int T, int num_pages, int P, int K, int d, unsigned* err, cudaStream_t st) {
    return wide ? launch_write<I, C, 8>(k, v, kt, kh, vt, vh, kp, vp, slots, T, num_pages, P, K, d, err, st)
                : launch_write<I, C, 1>(k, v, kt, kh, vt, vh, kp, vp, slots, T, num_pages, P, K, d, err, st);
}

extern "C" int aie_write_kv_slots(const CwArgs* args, cudaStream_t stream) {
    const CwArgs& a = *args;
    if (a.T <= 0) return 0;
    if (a.P <= 0 || a.K <= 0 || a.d <= 0 || a.num_pages < 0) return AIE_BAD_ARG;
    const long long step = a.row_dtype == AIE_BF16 ? 8 : 4;      // elements in 16 bytes
    const bool wide = a.d % 8 == 0 && (a.k_token | a.k_head | a.v_token | a.v_head) % step == 0 &&
                      ((size_t)a.k | (size_t)a.v | (size_t)a.k_pages | (size_t)a.v_pages) % 16 == 0;
#define CW_ARGS wide, a.k, a.v, a.k_token, a.k_head, a.v_token, a.v_head, a.k_pages, a.v_pages, a.slots, a.T, a.num_pages, a.P, a.K, a.d, a.err, stream
    if (a.row_dtype == AIE_BF16 && a.cache_dtype == AIE_BF16) return launch_write_rows<bf16, bf16>(CW_ARGS);
    if (a.row_dtype == AIE_F32 && a.cache_dtype == AIE_BF16) return launch_write_rows<float, bf16>(CW_ARGS);
    if (a.row_dtype == AIE_F32 && a.cache_dtype == AIE_F32) return launch_write_rows<float, float>(CW_ARGS);
    if (a.row_dtype == AIE_BF16 && a.cache_dtype == AIE_F32) return launch_write_rows<bf16, float>(CW_ARGS);
    return AIE_BAD_ARG;
#undef CW_ARGS
}
