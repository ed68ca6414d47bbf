// RMS norm of every query and key head, scaled by a weight per feature, and the rotation by position, in one pass:
//   y = x * rsqrt(mean(x^2) + eps) * w,   out = y * cos + RotateHalf(y) * sin      (RotateHalf: apply_rope.rs:58-76)
// in f32 from the first square to the last sum, rounded once to the tensor's type.  (ApplyRope on its own rounds every
// product, as the CPU op does; here nothing stands between the norm and the rotation that a graph could observe.)
//
// HBM-bound: a row is read and written once (2 x 4096 tokens of 32 + 8 heads of 128 features in f16: 36.3 us, of which a plain copy of
// as many bytes takes 33; a token of a decoding step, 5 us, is the launch's latency).  A lane holds VW consecutive pairs (i, i + D/2) as two 16-byte pieces, so a
// row takes D / (2 VW) lanes, whose squares are summed by shuffles; rows of the same token that a lane takes one after
// the other (HPC heads) share its cos and sin pieces, which would otherwise cost as many load instructions as the rows.
#include <hip/hip_fp16.h>
#include <string.h>
#include "common.h"

namespace trocm {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Rows of which at least this much is read and written go past the caches (non-temporal loads and stores): 168 MB of
// f16 at 128 features 36.3 us (4.75 TB/s) against 41.1 through them, 82 MB 20.1 against 20.2, 61 MB 15.2 against 12.5, 20 MB 7.0 against 6.0.
constexpr int64_t kStreamBytes = 80ll << 20;

struct NormRope {
    const void *x[2];        // q, k
    const void *w[2];        // [D] each, NULL: ones
    void *y[2];              // dense [B, H, n, D]
    int64_t xs[2][3];        // element strides of batch, head, token
    int H[2];
    int q_chunks;            // workgroups in y that take query heads
    const void *cos, *sin;
    int64_t cs_stride_b;
    int64_t n_tok;           // B * n
    int n, D;
    float eps, inv_d;
};

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(_Float16 x) { return (float)x; }

template <bool STREAM, typename P>
__device__ __forceinline__ P load16(const void *a) {
    if (!STREAM) return *reinterpret_cast<const P *>(a);
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(a));
    return __builtin_bit_cast(P, v);
}

template <bool STREAM, typename P>
__device__ __forceinline__ void store16(void *a, const P &v) {
    if (STREAM) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<u32x4 *>(a));
    else *reinterpret_cast<P *>(a) = v;
}

template <typename T, int LPR, int HPC, bool STREAM>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(NormRope p) {
    constexpr int VW = 16 / sizeof(T), HALF = LPR * VW, D = 2 * HALF;
    struct alignas(16) Piece { T e[VW]; };
    const int64_t tok = (int64_t)blockIdx.x * (blockDim.x / LPR) + threadIdx.x / LPR;
    const int i = (threadIdx.x % LPR) * VW;
    const bool live = tok < p.n_tok;
    const int64_t t0 = live ? tok : p.n_tok - 1;   // (no lane leaves before the shuffles)
    const int64_t b = t0 / p.n, t = t0 - b * p.n;
    const int which = (int)blockIdx.y >= p.q_chunks;
    const int h0 = ((int)blockIdx.y - (which ? p.q_chunks : 0)) * HPC, H = p.H[which];
    const T *x = reinterpret_cast<const T *>(p.x[which]) + b * p.xs[which][0] + t * p.xs[which][2] + i;
    T *y = reinterpret_cast<T *>(p.y[which]) + (b * H * p.n + t) * D + i;
    Piece a[HPC], c[HPC];
#pragma unroll
    for (int j = 0; j < HPC; j++) {
        const T *row = x + (int64_t)min(h0 + j, H - 1) * p.xs[which][1];
        a[j] = load16<STREAM, Piece>(row);
        c[j] = load16<STREAM, Piece>(row + HALF);
    }
    const int64_t cs = b * p.cs_stride_b + t * D + i;
    const T *cos = reinterpret_cast<const T *>(p.cos) + cs, *sin = reinterpret_cast<const T *>(p.sin) + cs;
    const Piece c0 = *reinterpret_cast<const Piece *>(cos), c1 = *reinterpret_cast<const Piece *>(cos + HALF);
    const Piece s0 = *reinterpret_cast<const Piece *>(sin), s1 = *reinterpret_cast<const Piece *>(sin + HALF);
    float wa[VW], wc[VW];
    if (p.w[which]) {
        const T *w = reinterpret_cast<const T *>(p.w[which]) + i;
        const Piece w0 = *reinterpret_cast<const Piece *>(w), w1 = *reinterpret_cast<const Piece *>(w + HALF);
#pragma unroll
        for (int e = 0; e < VW; e++) wa[e] = widen(w0.e[e]), wc[e] = widen(w1.e[e]);
    } else {
#pragma unroll
        for (int e = 0; e < VW; e++) wa[e] = wc[e] = 1.0f;
    }
#pragma unroll
    for (int j = 0; j < HPC; j++) {
        float sq = 0.0f;
#pragma unroll
        for (int e = 0; e < VW; e++) {
            const float u = widen(a[j].e[e]), v = widen(c[j].e[e]);
            sq = __builtin_fmaf(u, u, __builtin_fmaf(v, v, sq));
        }
#pragma unroll
        for (int d = 1; d < LPR; d <<= 1) sq += __shfl_xor(sq, d, 64);
        const float r = 1.0f / sqrtf(__builtin_fmaf(sq, p.inv_d, p.eps));
        Piece lo, hi;
#pragma unroll
        for (int e = 0; e < VW; e++) {
            const float u = widen(a[j].e[e]) * r * wa[e], v = widen(c[j].e[e]) * r * wc[e];
            lo.e[e] = (T)(u * widen(c0.e[e]) - v * widen(s0.e[e]));
            hi.e[e] = (T)(v * widen(c1.e[e]) + u * widen(s1.e[e]));
        }
        if (live && h0 + j < H) {
            T *row = y + (int64_t)(h0 + j) * p.n * D;
            store16<STREAM>(row, lo);
            store16<STREAM>(row + HALF, hi);
        }
    }
}

// Any even head size, any alignment: a wave per row, a pair per lane at a time.
template <typename T>
__global__ __launch_bounds__(64) void qk_norm_rope_any_kernel(NormRope p) {
    const int which = (int)blockIdx.y >= p.H[0];
    const int h = (int)blockIdx.y - (which ? p.H[0] : 0), lane = threadIdx.x, half = p.D / 2;
    const int64_t b = (int64_t)blockIdx.x / p.n, t = (int64_t)blockIdx.x - b * p.n;
    const T *x = reinterpret_cast<const T *>(p.x[which]) + b * p.xs[which][0] + h * p.xs[which][1] + t * p.xs[which][2];
    T *y = reinterpret_cast<T *>(p.y[which]) + ((b * p.H[which] + h) * p.n + t) * p.D;
    const T *cos = reinterpret_cast<const T *>(p.cos) + b * p.cs_stride_b + t * p.D, *sin = reinterpret_cast<const T *>(p.sin) + b * p.cs_stride_b + t * p.D;
    const T *w = reinterpret_cast<const T *>(p.w[which]);
    float sq = 0.0f;
    for (int i = lane; i < p.D; i += 64) {
        const float u = widen(x[i]);
        sq = __builtin_fmaf(u, u, sq);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sq += __shfl_xor(sq, d, 64);
    const float r = 1.0f / sqrtf(__builtin_fmaf(sq, p.inv_d, p.eps));
    for (int i = lane; i < half; i += 64) {   // (a pair is read before it is written, by one lane: y may be x)
        const float u = widen(x[i]) * r * (w ? widen(w[i]) : 1.0f), v = widen(x[i + half]) * r * (w ? widen(w[i + half]) : 1.0f);
        y[i] = (T)(u * widen(cos[i]) - v * widen(sin[i]));
        y[i + half] = (T)(v * widen(cos[i + half]) + u * widen(sin[i + half]));
    }
}

template <typename T, int LPR, int HPC, bool STREAM>
void launch_vec(NormRope p, hipStream_t s) {
    p.q_chunks = (p.H[0] + HPC - 1) / HPC;
    const int threads = p.n_tok * LPR <= 64 ? 64 : 256;   // (a whole number of rows either way)
    const int64_t blocks = (p.n_tok * LPR + threads - 1) / threads;
    hipLaunchKernelGGL((qk_norm_rope_kernel<T, LPR, HPC, STREAM>), dim3((unsigned)blocks, (unsigned)(p.q_chunks + (p.H[1] + HPC - 1) / HPC)), dim3(threads), 0, s, p);
}

template <typename T, int LPR>
void launch_heads(const NormRope &p, hipStream_t s) {
    // a lane takes two heads where that leaves four workgroups per compute unit: 168 MB of f16 41.1 us, against 44.9 with one head a
    // lane, 40.9 with four and 42.3 with eight (past the caches 36.3, 36.5 with four, 37.7 with eight); 1000 tokens 5.9 to 6.0 with each
    const int64_t rows = (p.n_tok * LPR + 255) / 256 * (p.H[0] + p.H[1]), enough = (int64_t)num_compute_units() * 4;
    const int64_t bytes = 2 * p.n_tok * (p.H[0] + p.H[1]) * p.D * (int64_t)sizeof(T);
    if (bytes > kStreamBytes) launch_vec<T, LPR, 2, true>(p, s);
    else if (rows >= 2 * enough) launch_vec<T, LPR, 2, false>(p, s);
    else launch_vec<T, LPR, 1, false>(p, s);
}

}  // namespace

int launch_qk_norm_rope(const QkNormRopeArgs &a, hipStream_t s) {
    if (a.B == 0 || a.n == 0 || a.D == 0) return 0;
    NormRope p;
    memset(&p, 0, sizeof(p));
    p.n = (int)a.n, p.D = (int)a.D, p.n_tok = a.B * a.n;
    p.eps = a.eps, p.inv_d = 1.0f / (float)a.D;
    p.cos = a.cos, p.sin = a.sin, p.cs_stride_b = a.cs_stride_b;
    const size_t es = elem_bytes(a.dtype);
    const int64_t vw = 16 / es;
    bool vec = (uintptr_t)a.cos % 16 == 0 && (uintptr_t)a.sin % 16 == 0 && a.cs_stride_b % vw == 0;
    for (int i = 0; i < 2; i++) {
        p.x[i] = a.x[i], p.w[i] = a.w[i], p.y[i] = a.y[i], p.H[i] = (int)a.H[i];
        for (int d = 0; d < 3; d++) {
            p.xs[i][d] = a.xs[i][d];
            vec = vec && a.xs[i][d] % vw == 0;
        }
        vec = vec && (uintptr_t)a.x[i] % 16 == 0 && (uintptr_t)a.w[i] % 16 == 0 && (uintptr_t)a.y[i] % 16 == 0;
    }
    const int64_t lanes = vec && a.D % (2 * vw) == 0 ? a.D / (2 * vw) : 0;
    if (a.dtype == TROCM_F16 && lanes == 4) launch_heads<_Float16, 4>(p, s);
    else if (a.dtype == TROCM_F16 && lanes == 8) launch_heads<_Float16, 8>(p, s);
    else if (a.dtype == TROCM_F16 && lanes == 16) launch_heads<_Float16, 16>(p, s);
    else if (a.dtype == TROCM_F32 && lanes == 8) launch_heads<float, 8>(p, s);
    else if (a.dtype == TROCM_F32 && lanes == 16) launch_heads<float, 16>(p, s);
    else if (a.dtype == TROCM_F32 && lanes == 32) launch_heads<float, 32>(p, s);
    else if (a.dtype == TROCM_F16)
        hipLaunchKernelGGL((qk_norm_rope_any_kernel<_Float16>), dim3((unsigned)p.n_tok, (unsigned)(a.H[0] + a.H[1])), dim3(64), 0, s, p);
    else
        hipLaunchKernelGGL((qk_norm_rope_any_kernel<float>), dim3((unsigned)p.n_tok, (unsigned)(a.H[0] + a.H[1])), dim3(64), 0, s, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail("qk_norm_rope launch failed: %s", hipGetErrorString(e));
    return 0;
}

}  // namespace trocm
