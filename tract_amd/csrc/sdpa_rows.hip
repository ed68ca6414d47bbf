// Attention of a few or many query rows over streamed keys: over a prefix that a batch shares, kept once, followed by
// the sequences' own keys; and over keys whose scores are capped, biased by distance or cut into documents.  f16 and f32.
//
// All query rows that read the same keys are rows of one matrix product.  Row r of a kv head is (b, i, g) =
// (r / (Sq G), r / G % Sq, r % G): sequence, query, head of the group.  Over a sequence's own keys a tile takes rows of one
// sequence; over the shared prefix it takes rows of any, so that the prefix is read once for as many sequences as a tile
// has rows.  The formulation is the transposed one of the other MFMA kernels, S^T = K Q^T and O^T = V^T P^T: every softmax
// scalar of a row sits in one lane.
//
// Work item = (kv head, tile of 32 RB rows, range of keys); a workgroup of 4 waves takes one.  The waves take the range's
// tiles of 32 keys in turn, each with a private K and V tile in LDS and the next one in flight in registers: no barrier in
// the loop.  Waves are joined through LDS, ranges through the workspace (partial rows of f32: unnormalised O, maximum, sum).
#include <hip/hip_fp16.h>
#include <limits.h>
#include <stddef.h>
#include <string.h>
#include <type_traits>
#include "common.h"

namespace trocm {
namespace {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef float float16_t __attribute__((ext_vector_type(16)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef int int4_a4 __attribute__((ext_vector_type(4), aligned(4)));   // (a row of document ids starts anywhere)

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWaves = 4, kThreads = 64 * kWaves, kTile = 32;
constexpr int kSeqWords = 700;   // of a launch's table, with the other arguments under 4 KB
constexpr int kSeqEntry = 8;     // words of a sequence of its own: k, v, stride of a head (bytes), length, unused

struct SeqTable { uint32_t w[kSeqWords]; };
// The table of a launch where its arguments lie (its kernel's one argument is a RowsCall): a word at a computed place is a scalar
// load.  Asked of the argument itself, the compiler copied all of it to every lane's scratch first.
typedef const __attribute__((address_space(4))) uint32_t *TableWords;

struct RowsDev {
    const char *q;
    char *out;
    int B, Hq, Hkv, Sq, G, D;
    // shared prefix
    const char *pk, *pv;
    int64_t p_stride_h, p_stride_t;   // bytes
    int P, p_splits, p_row_tiles, p_tiles;   // p_tiles, own_tiles: key tiles of a range
    // own keys: regular (one base, strides) or a table entry per sequence
    const char *k, *v;
    int64_t stride_b, stride_h, stride_t;
    int regular;                // 0: table of entries, 1: table of lengths, 2: every sequence has Sk keys
    int Sk, own_splits, own_row_tiles, own_tiles, seq0, n_seq;
    float scale, cap;
    int causal;
    const float *slopes;        // [Hq]
    const int *docs;            // [B, Sk]
    const int *prefix_lens;     // [B]
    // partials [splits][B * Hq * Sq][D], then [splits][2][B * Hq * Sq]
    float *part_o, *part_ml;
    int64_t part_rows;
    int splits;                 // p_splits + own_splits; 1: no partials, rows go to `out`
};

struct RowsCall { RowsDev p; SeqTable tab; };
__device__ __forceinline__ TableWords table_words(size_t at = offsetof(RowsCall, tab)) {
    return reinterpret_cast<TableWords>(reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr()) + at);
}

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(_Float16 x) { return (float)x; }

struct OwnKeys { const char *k, *v; int len; };

__device__ __forceinline__ OwnKeys own_keys(const RowsDev &p, int b, int kvh) {
    OwnKeys o;
    const TableWords words = table_words();
    if (p.regular) {
        o.k = p.k + (int64_t)b * p.stride_b + (int64_t)kvh * p.stride_h;
        o.v = p.v + (int64_t)b * p.stride_b + (int64_t)kvh * p.stride_h;
        o.len = p.regular == 2 ? p.Sk : (int)words[b - p.seq0];
    } else {
        const TableWords e = words + (b - p.seq0) * kSeqEntry;
        const int64_t sh = (int64_t)((uint64_t)e[4] | ((uint64_t)e[5] << 32));
        o.k = reinterpret_cast<const char *>((uint64_t)e[0] | ((uint64_t)e[1] << 32)) + kvh * sh;
        o.v = reinterpret_cast<const char *>((uint64_t)e[2] | ((uint64_t)e[3] << 32)) + kvh * sh;
        o.len = (int)e[6];
    }
    return o;
}

// tanh for the f32 rows: the library's, accurate to an ulp or two near zero.  For f16 rows 1 - 2 / (e^2x + 1), whose absolute
// error of 1e-7 times the cap is far below what the rounding of the weights to f16 leaves.
template <typename T>
__device__ __forceinline__ float cap_tanh(float x) {
    if constexpr (std::is_same<T, float>::value) return tanhf(x);
    return 1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * (2.0f * kLog2e)) + 1.0f);
}

// ---- any head size, any alignment: a workgroup per query row -------------------------------------------------------

constexpr int kAnyThreads = 256, kAnyMaxD = 2048;

template <typename T>
__global__ __launch_bounds__(kAnyThreads) void sdpa_rows_any_kernel(RowsCall call) {
    const RowsDev &p = call.p;
    __shared__ float lds_q[kAnyMaxD], lds_o[kAnyMaxD], lds_p[kAnyThreads], lds_red[2 * kWaves];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, D = p.D;
    const int qh = blockIdx.x % p.Hq, i = blockIdx.x / p.Hq, b = p.seq0 + blockIdx.y, kvh = qh / p.G;
    const OwnKeys own = own_keys(p, b, kvh);
    const int64_t row = ((int64_t)b * p.Hq + qh) * p.Sq + i;
    const T *q = reinterpret_cast<const T *>(p.q) + row * D;
    for (int d = tid; d < D; d += kAnyThreads) lds_q[d] = widen(q[d]);
    const int at = i + own.len - p.Sq;
    int lim = p.causal ? at : own.len - 1;
    if (p.prefix_lens) lim = max(lim, p.prefix_lens[b] - 1);
    lim = min(lim, own.len - 1);
    const float slope = p.slopes ? p.slopes[qh] : 0.0f;
    const int *docs = p.docs ? p.docs + (int64_t)b * p.Sk : nullptr;
    const int my_doc = docs && at >= 0 ? docs[at] : -1;
    float m_run = -INFINITY, l_run = 0.0f;
    for (int d = tid; d < D; d += kAnyThreads) lds_o[d] = 0.0f;   // (a thread's own features)
    __syncthreads();
#pragma unroll 1
    for (int src = 0; src < 2; src++) {
        const int n = src ? lim + 1 : p.P;
        const char *kb = src ? own.k : p.pk + (int64_t)kvh * p.p_stride_h, *vb = src ? own.v : p.pv + (int64_t)kvh * p.p_stride_h;
        const int64_t st = src ? p.stride_t : p.p_stride_t;
#pragma unroll 1
        for (int j0 = 0; j0 < n; j0 += kAnyThreads) {
            const int j = j0 + tid;
            const bool sees = j < n && (!src || !docs || (docs[j] == my_doc && my_doc >= 0));
            float s = -INFINITY;
            if (sees) {
                const T *k = reinterpret_cast<const T *>(kb + (int64_t)j * st);
                float dot = 0.0f;
#pragma unroll 1
                for (int d = 0; d < D; d++) dot = __builtin_fmaf(lds_q[d], widen(k[d]), dot);
                s = dot * p.scale;
                if (p.cap > 0.0f) s = p.cap * cap_tanh<T>(s / p.cap);
                if (src && p.slopes) s -= slope * (float)abs(at - j);
                s *= kLog2e;
            }
            float m = s;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
            if (lane == 0) lds_red[w] = m;
            __syncthreads();
            m = fmaxf(fmaxf(lds_red[0], lds_red[1]), fmaxf(lds_red[2], lds_red[3]));
            const float m_new = fmaxf(m_run, m), ref = m_new == -INFINITY ? 0.0f : m_new;
            const float keep = __builtin_amdgcn_exp2f(m_run - ref);
            const float e = sees ? __builtin_amdgcn_exp2f(s - ref) : 0.0f;
            float l = e;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d, 64);
            if (lane == 0) lds_red[kWaves + w] = l;
            lds_p[tid] = sees ? e : -1.0f;   // (what is hidden is not read: it may hold anything)
            __syncthreads();
            l_run = l_run * keep + (lds_red[kWaves] + lds_red[kWaves + 1] + lds_red[kWaves + 2] + lds_red[kWaves + 3]);
            m_run = m_new;
            const int cnt = min(kAnyThreads, n - j0);
#pragma unroll 1
            for (int d = tid; d < D; d += kAnyThreads) {
                float acc = lds_o[d] * keep;
#pragma unroll 1
                for (int jj = 0; jj < cnt; jj++)
                    if (lds_p[jj] >= 0.0f) acc = __builtin_fmaf(lds_p[jj], widen(reinterpret_cast<const T *>(vb + (int64_t)(j0 + jj) * st)[d]), acc);
                lds_o[d] = acc;
            }
            __syncthreads();
        }
    }
    T *out = reinterpret_cast<T *>(p.out) + row * D;
    for (int d = tid; d < D; d += kAnyThreads) out[d] = (T)(l_run > 0.0f ? lds_o[d] / l_run : 0.0f);
}

// ---- new rows into the caches of their sequences ---------------------------------------------------------------------

// k_new, v_new dense [B, Hkv, n, D]; entry b's planes take them from its length on.  A 4-byte word per thread.
__global__ __launch_bounds__(256) void append_rows_kernel(SeqTable, const uint32_t *__restrict__ k_new, const uint32_t *__restrict__ v_new, int seq0, int Hkv,
                                                          int words_per_head, int64_t row_bytes) {
    const int kvh = blockIdx.y, b = seq0 + blockIdx.z;
    const TableWords e = table_words(0) + blockIdx.z * kSeqEntry;
    const int64_t sh = (int64_t)((uint64_t)e[4] | ((uint64_t)e[5] << 32)), at = kvh * sh + (int64_t)(int)e[6] * row_bytes;
    uint32_t *k = reinterpret_cast<uint32_t *>(reinterpret_cast<char *>((uint64_t)e[0] | ((uint64_t)e[1] << 32)) + at);
    uint32_t *v = reinterpret_cast<uint32_t *>(reinterpret_cast<char *>((uint64_t)e[2] | ((uint64_t)e[3] << 32)) + at);
    const int64_t from = ((int64_t)b * Hkv + kvh) * words_per_head;
    for (int i = blockIdx.x * 256 + threadIdx.x; i < words_per_head; i += gridDim.x * 256) {
        k[i] = k_new[from + i];
        v[i] = v_new[from + i];
    }
}

int check_launch(const char *what) {
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail("%s launch failed: %s", what, hipGetErrorString(e));
}

// Entries of sequences [first, first + n) of a call.
void fill_table(const SdpaRowsArgs &a, int64_t first, int64_t n, SeqTable &tab) {
    if (a.lens) {
        for (int64_t i = 0; i < n; i++) tab.w[i] = (uint32_t)a.lens[first + i];
    } else if (a.seqs) {
        for (int64_t i = 0; i < n; i++) {
            const SdpaRowsSeq &s = a.seqs[first + i];
            const uint64_t f[3] = {(uint64_t)(uintptr_t)s.k, (uint64_t)(uintptr_t)s.v, (uint64_t)(s.stride_h * (int64_t)elem_bytes(a.dtype))};
            uint32_t *e = tab.w + i * kSeqEntry;
            for (int x = 0; x < 3; x++) e[2 * x] = (uint32_t)f[x], e[2 * x + 1] = (uint32_t)(f[x] >> 32);
            e[6] = (uint32_t)s.len, e[7] = 0;
        }
    }
}
int64_t table_holds(const SdpaRowsArgs &a) { return a.lens ? kSeqWords : a.seqs ? kSeqWords / kSeqEntry : a.B; }

void fill_rows(const SdpaRowsArgs &a, RowsDev &p) {
    const int64_t es = (int64_t)elem_bytes(a.dtype);
    memset(&p, 0, sizeof(p));
    p.q = (const char *)a.q, p.out = (char *)a.out;
    p.B = (int)a.B, p.Hq = (int)a.Hq, p.Hkv = (int)a.Hkv, p.Sq = (int)a.Sq, p.G = (int)(a.Hq / a.Hkv), p.D = (int)a.D;
    p.pk = (const char *)a.pk, p.pv = (const char *)a.pv, p.P = (int)a.P;
    p.p_stride_h = a.p_stride_h * es, p.p_stride_t = a.p_stride_t * es;
    p.k = (const char *)a.k, p.v = (const char *)a.v;
    p.stride_b = a.stride_b * es, p.stride_h = a.stride_h * es, p.stride_t = a.stride_t * es;
    p.regular = a.lens ? 1 : a.seqs ? 0 : 2;
    p.Sk = (int)a.Sk, p.scale = a.scale, p.cap = a.softcap, p.causal = a.causal;
    p.slopes = a.slopes, p.docs = a.documents, p.prefix_lens = a.prefix_lens;
    p.part_rows = a.B * a.Hq * a.Sq;
}

}  // namespace

// Partial rows for as many ranges as the launch below makes of a call: some hundred workgroups' tiles, two ranges at least.
size_t sdpa_shared_workspace_bytes(int64_t B, int64_t Hq, int64_t Sq, int64_t D) {
    const int64_t rows = B * Hq * Sq, most = rows > 0 ? (1 << 16) / rows : 2;
    const int64_t splits = most < 2 ? 2 : most > 64 ? 64 : most;
    return kWsCounterBytes + kWsPlanBytes + (size_t)rows * splits * (size_t)(D + 2) * sizeof(float) + 256;
}

int launch_append_rows(const SdpaRowsArgs &a, const void *k_new, const void *v_new, hipStream_t s) {
    const int64_t row_bytes = a.D * (int64_t)elem_bytes(a.dtype), words = a.Sq * row_bytes / 4;
    TROCM_REQUIRE(words < (1 << 30), "append: too many new tokens");
    if (words == 0) return 0;
    const int64_t step = table_holds(a);
    for (int64_t b = 0; b < a.B; b += step) {
        const int64_t n = a.B - b < step ? a.B - b : step;
        SeqTable tab;
        fill_table(a, b, n, tab);
        const int64_t blocks = (words + 255) / 256;
        hipLaunchKernelGGL(append_rows_kernel, dim3((unsigned)(blocks < 64 ? blocks : 64), (unsigned)a.Hkv, (unsigned)n), dim3(256), 0, s, tab,
                           (const uint32_t *)k_new, (const uint32_t *)v_new, (int)b, (int)a.Hkv, (int)words, row_bytes);
        if (check_launch("append_rows")) return 1;
    }
    return 0;
}

int launch_sdpa_rows(const SdpaRowsArgs &a, hipStream_t s) {
    if (a.B == 0 || a.Hq == 0 || a.Sq == 0 || a.D == 0) return 0;
    RowsCall call;
    RowsDev &p = call.p;
    fill_rows(a, p);
    TROCM_REQUIRE(a.D <= kAnyMaxD, "attention: head_dim %lld is above %d", (long long)a.D, kAnyMaxD);
    TROCM_REQUIRE(a.Hq * a.Sq < (1ll << 31), "attention: too many query rows per sequence");
    const int64_t holds = table_holds(a), step = holds < 65535 ? holds : 65535;
    for (int64_t b = 0; b < a.B; b += step) {
        const int64_t n = a.B - b < step ? a.B - b : step;
        fill_table(a, b, n, call.tab);
        p.seq0 = (int)b;
        const dim3 grid((unsigned)(a.Hq * a.Sq), (unsigned)n);
        if (a.dtype == TROCM_F16) hipLaunchKernelGGL((sdpa_rows_any_kernel<_Float16>), grid, dim3(kAnyThreads), 0, s, call);
        else hipLaunchKernelGGL((sdpa_rows_any_kernel<float>), grid, dim3(kAnyThreads), 0, s, call);
        if (check_launch("sdpa_rows")) return 1;
    }
    return 0;
}

}  // namespace trocm
