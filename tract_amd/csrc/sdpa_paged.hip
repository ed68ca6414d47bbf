// Attention over pages of keys and values: o = softmax(scale q k^T) v for one or a few new tokens of every sequence, whose keys lie in
// pages anywhere, found through a table, and whose lengths are read from device memory.  f16 and f32.
#include <hip/hip_fp16.h>
#include <math.h>
#include <algorithm>
#include "common.h"
#include "fast_div.h"

namespace trocm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct PagedDev {
    const char *q, *k, *v;
    char *out;
    const int *table, *lens;
    int64_t table_width, stride_page, stride_h, stride_t;   // strides: bytes
    int B, Hq, Hkv, Sq, G, D, n_pages, most;                // most: tokens that a row of the table has pages for
    float scale;
    int causal;
    FastDiv by_page;
};

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(_Float16 x) { return (float)x; }

// ---- any head size, page size and alignment: a workgroup per query row ----------------------------------------------------

constexpr int kAnyThreads = 256, kAnyWaves = kAnyThreads / 64;

template <typename T>
__global__ __launch_bounds__(kAnyThreads) void sdpa_paged_any_kernel(PagedDev p) {
    __shared__ float lds_q[kRowsMaxD], lds_o[kRowsMaxD], lds_p[kAnyThreads], lds_red[2 * kAnyWaves];
    __shared__ int64_t lds_at[kAnyThreads];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, D = p.D;
    const int qh = blockIdx.x % p.Hq, i = blockIdx.x / p.Hq, kvh = qh / p.G;
    for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
        const int64_t row = ((int64_t)b * p.Hq + qh) * p.Sq + i;
        const T *q = reinterpret_cast<const T *>(p.q) + row * D;
        const int len = min(max(p.lens[b], 0), p.most), n = p.causal ? min(len - p.Sq + i + 1, len) : len;
        const int *pages = p.table + b * p.table_width;
        for (int d = tid; d < D; d += kAnyThreads) lds_q[d] = widen(q[d]), lds_o[d] = 0.0f;   // (lds_o: a thread's own features)
        __syncthreads();
        float m_run = -INFINITY, l_run = 0.0f;
        for (int j0 = 0; j0 < n; j0 += kAnyThreads) {
            const int j = j0 + tid;
            float s = -INFINITY;
            bool sees = false;
            if (j < n) {
                const int pi = p.by_page.by(j), id = pages[pi];
                sees = (unsigned)id < (unsigned)p.n_pages;
                if (sees) {
                    const int64_t at = id * p.stride_page + kvh * p.stride_h + (j - pi * (int)p.by_page.d) * p.stride_t;
                    lds_at[tid] = at;
                    const T *k = reinterpret_cast<const T *>(p.k + at);
                    float dot = 0.0f;
#pragma unroll 1
                    for (int d = 0; d < D; d++) dot = __builtin_fmaf(lds_q[d], widen(k[d]), dot);
                    s = dot * (p.scale * kLog2e);
                }
            }
            float m = s;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
            if (lane == 0) lds_red[w] = m;
            __syncthreads();
            m = fmaxf(fmaxf(lds_red[0], lds_red[1]), fmaxf(lds_red[2], lds_red[3]));
            const float m_new = fmaxf(m_run, m), ref = m_new == -INFINITY ? 0.0f : m_new;
            const float keep = __builtin_amdgcn_exp2f(m_run - ref), e = sees ? __builtin_amdgcn_exp2f(s - ref) : 0.0f;
            float l = e;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d, 64);
            if (lane == 0) lds_red[kAnyWaves + w] = l;
            lds_p[tid] = sees ? e : -1.0f;   // (what is hidden is not read: it may hold anything; a weight of NaN is not hidden)
            __syncthreads();
            l_run = l_run * keep + (lds_red[kAnyWaves] + lds_red[kAnyWaves + 1] + lds_red[kAnyWaves + 2] + lds_red[kAnyWaves + 3]);
            m_run = m_new;
            const int cnt = min(kAnyThreads, n - j0);
#pragma unroll 1
            for (int d = tid; d < D; d += kAnyThreads) {
                float acc = lds_o[d] * keep;
#pragma unroll 1
                for (int x = 0; x < cnt; x++)
                    if (!(lds_p[x] < 0.0f)) acc = __builtin_fmaf(lds_p[x], widen(reinterpret_cast<const T *>(p.v + lds_at[x])[d]), acc);
                lds_o[d] = acc;
            }
            __syncthreads();
        }
        T *out = reinterpret_cast<T *>(p.out) + row * D;
        for (int d = tid; d < D; d += kAnyThreads) out[d] = (T)(l_run == 0.0f ? 0.0f : lds_o[d] / l_run);
        __syncthreads();
    }
}

}  // namespace

size_t sdpa_paged_workspace_bytes(int64_t, int64_t, int64_t, int64_t, int64_t) { return kWsCounterBytes; }

int launch_sdpa_paged(const SdpaPagedArgs &a, hipStream_t s) {
    if (a.B == 0 || a.Hq == 0 || a.Sq == 0 || a.D == 0) return 0;
    const int64_t es = (int64_t)elem_bytes(a.dtype);
    PagedDev p;
    p.q = (const char *)a.q, p.k = (const char *)a.k, p.v = (const char *)a.v, p.out = (char *)a.out;
    p.table = a.table, p.lens = a.lens, p.table_width = a.table_width;
    p.stride_page = a.stride_page * es, p.stride_h = a.stride_h * es, p.stride_t = a.stride_t * es;
    p.B = (int)a.B, p.Hq = (int)a.Hq, p.Hkv = (int)a.Hkv, p.Sq = (int)a.Sq, p.G = (int)(a.Hq / a.Hkv), p.D = (int)a.D;
    p.n_pages = (int)a.n_pages, p.most = (int)std::min<int64_t>(a.table_width * a.page_size, 1 << 30);
    p.scale = a.scale, p.causal = a.causal, p.by_page = fast_div(a.page_size);
    TROCM_REQUIRE(a.D <= kRowsMaxD, "sdpa_paged: head_dim %lld is more than %d", (long long)a.D, kRowsMaxD);
    const dim3 grid((unsigned)(a.Hq * a.Sq), (unsigned)std::min<int64_t>(a.B, 32768));
    if (a.dtype == TROCM_F16) sdpa_paged_any_kernel<_Float16><<<grid, kAnyThreads, 0, s>>>(p);
    else sdpa_paged_any_kernel<float><<<grid, kAnyThreads, 0, s>>>(p);
    TROCM_HIP(hipGetLastError());
    return 0;
}

}  // namespace trocm
