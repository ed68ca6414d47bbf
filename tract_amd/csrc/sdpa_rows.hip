// Attention of a few or many query rows over streamed keys: over a prefix that a batch shares, kept once, followed by
// the sequences' own keys; and over keys whose scores are capped, biased by distance or cut into documents.  f16 and f32.
//
// All query rows that read the same keys are rows of one matrix product.  Row r of a kv head is (b, i, g) =
// (r / (Sq G), r / G % Sq, r % G): sequence, query, head of the group.  Over a sequence's own keys a tile takes rows of one
// sequence; over the shared prefix it takes rows of any, so that the prefix is read once for as many sequences as a tile
// has rows.  The formulation is the transposed one of the other MFMA kernels, S^T = K Q^T and O^T = V^T P^T: every softmax
// scalar of a row sits in one lane.
//
// Work item = (kv head, tile of 16 or 32 rows, part of the keys); a workgroup of 4 waves takes one.  The waves take the part's
// tiles of 32 keys in turn, each with private tiles in LDS and the next one in flight in registers: no barrier in the loop.  A long prefix
// under many rows of f16 takes tiles of 128 rows, whose four waves share each tile of 64 keys.  Waves are joined through LDS, parts
// through the workspace (partial rows of f32: unnormalised O, maximum, sum), by the last workgroup to arrive or a launch after it.
//
// What bounds it, and what it takes (f16, 8 kv heads of 128 features unless said otherwise): HBM where rows are few, 8 x 8193 keys
// under 4 rows 45.6 us (5.9 TB/s; a copy's rate is 5.2), 16 x 6000 65 us (6.0 TB/s); HBM and the f32 parts behind a prefix, 64 sequences of 64 to 512
// keys behind 8192 under 4 rows each 32 us for 118 MB and 28 MB of parts written and read, 200 of up to 300 behind 1500 of 64 features
// under 8 rows each 24 us; the chain of a launch where it is short, 4 x 40 keys behind 777 8.5 us.  f32: 16 sequences of up to 600 keys behind
// 4096, 32 kv heads of 64 features, 31.5 us for 134 MB; f32 chunks are bound by the f32 matrix instructions of one wave per SIMD.
#include <hip/hip_fp16.h>
#include <limits.h>
#include <stddef.h>
#include <string.h>
#include <type_traits>
#include "common.h"
#include "fast_div.h"

namespace trocm {
namespace {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float16_t __attribute__((ext_vector_type(16)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));

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
    int P, p_items, p_splits, p_row_tiles;   // p_items: of this launch
    // own keys: regular (one base, strides) or a table entry per sequence
    const char *k, *v;
    int64_t stride_b, stride_h, stride_t;
    int regular;                // 0: table of entries, 1: table of lengths, 2: every sequence has Sk keys
    int Sk, own_splits, own_row_tiles, own_tiles, seq0, items;   // items: of this launch
    float scale, cap;
    int causal;
    const float *slopes;        // [Hq]
    const int *docs;            // [B, Sk]
    const int *prefix_lens;     // [B]
    // partials [splits][B * Hq * Sq][D], then [splits][2][B * Hq * Sq]
    float *part_o, *part_ml;
    int64_t part_rows;
    int *counters;              // != NULL: the last workgroup of a unit joins its parts; else a launch after this one
    int splits;                 // p_splits + own_splits; 1: no partials, rows go to `out`
    FastDiv by_g, by_sq, by_p_row_tiles, by_own_splits, by_own_row_tiles, by_own_tiles;   // own_tiles: key tiles of a part, about
};

struct RowsCall { RowsDev p; SeqTable tab; };
__device__ __forceinline__ TableWords table_words(size_t at = offsetof(RowsCall, tab)) {
    return reinterpret_cast<TableWords>(reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr()) + at);
}

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(_Float16 x) { return (float)x; }

// 16 bytes of device memory.  Pointers that come out of a table are generic ones to the compiler, whose loads go by the LDS's
// counter too: every wait for LDS would wait for the tile in flight.  ONCE: past the caches.
template <bool ONCE = false>
__device__ __forceinline__ u32x4 load16(const char *base, uint32_t off) {
    const auto *at = (const __attribute__((address_space(1))) u32x4 *)(base + off);
    return ONCE ? __builtin_nontemporal_load(at) : *at;
}

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

// tanh for f32 rows and for large caps: the library's, accurate to an ulp or two near zero.  For f16 rows under a cap of up to
// kFastTanhCap 1 - 2 / (e^2x + 1).
__device__ __forceinline__ float fast_tanh(float x) {
    return 1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * (2.0f * kLog2e)) + 1.0f);
}

// a - b of scores as they are rounded: a product fused into it would differ from `b`, which is one of them, by up to half its last place.
__device__ __forceinline__ float less(float a, float b) {
#pragma clang fp contract(off)
    return a - b;
}

// ---- any head size, any alignment: a workgroup per query row -------------------------------------------------------

constexpr int kAnyThreads = 256, kAnyMaxD = kRowsMaxD;

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
    if (p.prefix_lens) lim = max(lim, max(p.prefix_lens[b], 0) - 1);
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
                if (p.cap > 0.0f) s = p.cap * tanhf(s / p.cap);
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
            lds_p[tid] = sees ? e : -1.0f;   // (what is hidden is not read: it may hold anything; a weight of NaN is not hidden)
            __syncthreads();
            l_run = l_run * keep + (lds_red[kWaves] + lds_red[kWaves + 1] + lds_red[kWaves + 2] + lds_red[kWaves + 3]);
            m_run = m_new;
            const int cnt = min(kAnyThreads, n - j0);
#pragma unroll 1
            for (int d = tid; d < D; d += kAnyThreads) {
                float acc = lds_o[d] * keep;
#pragma unroll 1
                for (int jj = 0; jj < cnt; jj++)
                    if (!(lds_p[jj] < 0.0f)) acc = __builtin_fmaf(lds_p[jj], widen(reinterpret_cast<const T *>(vb + (int64_t)(j0 + jj) * st)[d]), acc);
                lds_o[d] = acc;
            }
            __syncthreads();
        }
    }
    T *out = reinterpret_cast<T *>(p.out) + row * D;
    for (int d = tid; d < D; d += kAnyThreads) out[d] = (T)(l_run == 0.0f ? 0.0f : lds_o[d] / l_run);
}

// ---- new rows into the caches of their sequences ---------------------------------------------------------------------

// k_new, v_new dense [B, Hkv, n, D]; entry b's planes take them from its length on.  A word per thread: 4 bytes where rows and addresses
// are whole ones, else 2.
template <typename W>
__global__ __launch_bounds__(256) void append_rows_kernel(SeqTable, const W *__restrict__ k_new, const W *__restrict__ v_new, int seq0, int Hkv,
                                                          int words_per_head, int64_t row_bytes) {
    const int kvh = blockIdx.y, b = seq0 + blockIdx.z;
    const TableWords e = table_words(0) + blockIdx.z * kSeqEntry;
    const int64_t sh = (int64_t)((uint64_t)e[4] | ((uint64_t)e[5] << 32)), at = kvh * sh + (int64_t)(int)e[6] * row_bytes;
    W *k = reinterpret_cast<W *>(reinterpret_cast<char *>((uint64_t)e[0] | ((uint64_t)e[1] << 32)) + at);
    W *v = reinterpret_cast<W *>(reinterpret_cast<char *>((uint64_t)e[2] | ((uint64_t)e[3] << 32)) + at);
    const int64_t from = ((int64_t)b * Hkv + kvh) * words_per_head;
    for (int i = blockIdx.x * 256 + threadIdx.x; i < words_per_head; i += gridDim.x * 256) {
        k[i] = k_new[from + i];
        v[i] = v_new[from + i];
    }
}

// ---- head sizes 64 and 128 on the matrix cores ---------------------------------------------------------------------

// Transposing 64-bit LDS load of 16-bit elements: in each block of 16 lanes, lane i receives
// element i%4 of the four 8-byte rows addressed by lanes i/4, i/4+4, i/4+8, i/4+12.
__device__ __forceinline__ half4_t lds_read_tr16(const _Float16 *lds_ptr) {
    typedef __attribute__((address_space(3))) short4_t *lds_v4_ptr;
    short4_t r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4_ptr)(uintptr_t)(uint32_t)(uintptr_t)lds_ptr);
    return __builtin_bit_cast(half4_t, r);
}

// Orders a wave's LDS accesses across its lanes (no instruction: the LDS serves a wave in order).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr int kListMax = 4096;   // key tiles of a range that documents are looked up for

// Partial results for whichever workgroup joins them: written through to where every compute unit sees them once they complete.
__device__ __forceinline__ void put(float *at, float x) { __hip_atomic_store(at, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float get(const float *at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
typedef float float2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void put2(float *at, float2_t x) { __hip_atomic_store(reinterpret_cast<uint64_t *>(at), __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float2_t get2(const float *at) { return __builtin_bit_cast(float2_t, __hip_atomic_load(reinterpret_cast<const uint64_t *>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)); }

// What a workgroup has to do: rows [row0, row_end) of a kv head over its share of the first `tiles` key tiles of one set of keys.  `parts`
// workgroups share them; part `part` takes groups of `kWaves` tiles (a tall tile: tiles) in turn, so that the parts stream through
// neighbouring memory together.
struct RowsWork {
    const char *k, *v;
    int64_t st;              // bytes between tokens
    int kvh, b;              // b: whose own keys (-1: the prefix)
    int row0, row_end, n_keys, tiles, part, parts, split;   // split: where its partial rows go
};

// Where row r of a kv head lies among the q and output rows.
struct RowPlace { int64_t at; int i, qh; };   // i: its place in the sequence's queries
__device__ __forceinline__ RowPlace q_row(const RowsDev &p, int kvh, int r) {
    const int bi = p.by_g.by(r), qh = kvh * p.G + r - bi * p.G, b = p.by_sq.by(bi), i = bi - b * p.Sq;
    return {((int64_t)b * p.Hq + qh) * p.Sq + i, i, qh};
}

// Places of the first t_end key tiles that hold a token of a document in [dmin, dmax]; bit 15: all of the tile's tokens are of
// document `one`, that of every row but padding (-1: they differ).  All threads; returns how many.  A wave looks at two
// tiles at a time, a token per lane.
__device__ __forceinline__ int list_document_tiles(const int *docs, int n_keys, int t_end, int dmin, int dmax, int one, uint16_t *list, int *counts) {
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    constexpr int PW = 32;   // tiles that a wave looks at before the waves compare
    const int dlow = max(dmin, 0);
    int n = 0;
    for (int t0 = 0; t0 < t_end; t0 += kWaves * PW) {
        const int first = t0 + w * PW;
        const uint32_t there = first >= t_end ? 0 : first + PW <= t_end ? ~0u : (1u << (t_end - first)) - 1;
        uint32_t active = 0, whole = 0;
#pragma unroll 1
        for (int x0 = 0; x0 < PW; x0 += 16) {   // (eight loads in flight; more of them, or their masks at once, spill scalar registers)
            int ids[8];
#pragma unroll
            for (int x = 0; x < 8; x++) ids[x] = docs[min((first + x0 + 2 * x) * kTile + lane, n_keys - 1)];
            uint32_t a16 = 0, w16 = 0;
#pragma unroll
            for (int x = 0; x < 8; x++) {
                const uint64_t in = __builtin_amdgcn_ballot_w64(ids[x] >= dlow && ids[x] <= dmax), other = __builtin_amdgcn_ballot_w64(ids[x] != one);
                a16 |= ((uint32_t)in != 0 ? 1u << 2 * x : 0) | ((uint32_t)(in >> 32) != 0 ? 2u << 2 * x : 0);
                w16 |= ((uint32_t)other == 0 ? 1u << 2 * x : 0) | ((uint32_t)(other >> 32) == 0 ? 2u << 2 * x : 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            active |= a16 << x0, whole |= w16 << x0;
        }
        if (one < 0) whole = 0;
        active &= there;
        if (lane == 0) counts[w] = __popc(active);
        __syncthreads();
        int at = n;
        for (int x = 0; x < kWaves; x++) {
            if (x < w) at += counts[x];
            n += counts[x];
        }
        if (lane < PW && ((active >> lane) & 1)) list[at + __popc(active & ((1u << lane) - 1))] = (uint16_t)((first + lane) | ((whole >> lane) & 1 ? 0x8000 : 0));
        __syncthreads();
    }
    return n;
}

// A tile of 16 or 32 rows, R of them; the four waves take the range's key tiles in turn.
//   R == 16: 16x16 MFMAs; R == 32: 32x32.  V goes through a wave-private LDS tile, and so does K but for 16 rows of f32, where it goes
//   straight from memory into fragments (four lanes read 64 consecutive bytes of a key's row; the tiles of two workgroups fit a compute
//   unit's LDS then).  K through LDS | straight: f16, 8 x 8193 keys 52.8 | 60.4 us; f32, 4 x 5000 keys 54.0 | 47.4 us.
template <typename T, int D, int R, bool SCORED, bool ONCE>
__device__ __forceinline__ void rows_body(const RowsDev &p, const RowsWork &wk, unsigned char *lds, uint16_t *s_list, int *s_counts) {
    constexpr bool H16 = sizeof(T) == 2;
    constexpr int DB = D / R, NG = 64 / R;        // feature blocks of the output; lane groups (4 or 2), whose lanes hold a row each
    constexpr int NS = kTile / NG;                // scores of a lane
    constexpr int KROW = H16 ? D + 8 : D + 4;     // elements per K row in LDS: 128-bit reads of 16 rows hit 64 distinct banks
    constexpr int VROW = H16 ? D + 16 : R == 16 ? D + 4 : D + 8;   // (rows of a read in different banks)
    constexpr bool KL = R == 32 || H16;
    constexpr int PRIV = kTile * (VROW + (KL ? KROW : 0)) * (int)sizeof(T);   // a wave's tile
    constexpr int CROW = D + 4;                   // floats per row where waves are joined
    constexpr int LPRW = D * (int)sizeof(T) / 16, RPI = 64 / LPRW, NI = kTile / RPI;   // lanes per key row, rows per load, loads per tile and tensor
    constexpr int KS = D * (int)sizeof(T) / (16 * NG);   // 16-byte pieces of a lane's share of a row
    static_assert(kWaves * R * CROW * 4 + kWaves * 2 * R * 4 <= kWaves * PRIV, "waves are joined where the tiles were");
    typedef typename std::conditional<R == 16, float4_t, float16_t>::type Acc;
    constexpr int NA = R == 16 ? 4 : 16;

    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, grp = lane / R, lr = lane % R;
    const bool own = wk.b >= 0;
    const int n_keys = wk.n_keys;
    // this lane's row
    const RowPlace place = q_row(p, wk.kvh, min(wk.row0 + lr, wk.row_end - 1));
    const int64_t out_row = place.at;
    const int at = place.i + n_keys - p.Sq;
    int lim = n_keys - 1, doc = 0;
    if (own && p.causal) lim = min(lim, SCORED && p.prefix_lens ? max(at, max(p.prefix_lens[wk.b], 0) - 1) : at);   // (of any value: a negative one is no prefix)
    float slope = 0.0f;
    const int *docs = nullptr;
    int n_tiles = wk.part < wk.parts ? wk.tiles : 0;   // of all parts; with documents those that are listed
    bool listed = false;
    if constexpr (SCORED) {
        if (p.slopes) slope = p.slopes[place.qh] * kLog2e;
        if (p.docs) {
            docs = p.docs + (int64_t)wk.b * p.Sk;
            doc = docs[at];
            if (doc < 0) lim = -1;   // padding sees nothing
            if (n_tiles > 0 && n_tiles <= kListMax) {
                int dmin = doc >= 0 ? doc : INT_MAX, dmax = doc;
#pragma unroll
                for (int d = 1; d < R; d <<= 1) dmin = min(dmin, __shfl_xor(dmin, d, 64)), dmax = max(dmax, __shfl_xor(dmax, d, 64));
                n_tiles = list_document_tiles(docs, n_keys, n_tiles, dmin, dmax, dmin == dmax ? dmin : -1, s_list, s_counts);
                listed = true;
            }
        }
    }
    float *part_ml = p.part_ml + (int64_t)wk.split * 2 * p.part_rows;
    const int first = wk.part * kWaves, step = wk.parts * kWaves;
    if (n_tiles <= first && p.splits > 1) {   // nothing to add: a maximum of -inf and a sum of 0 say so
        if (w == 0 && grp < 2 && wk.row0 + lr < wk.row_end) put(part_ml + out_row + (grp ? p.part_rows : 0), grp ? 0.0f : -INFINITY);
        return;
    }

    float m_run = -INFINITY, l_run = 0.0f;
    Acc o[DB];
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int r = 0; r < NA; r++) o[db][r] = 0.0f;

    T *lds_v = reinterpret_cast<T *>(lds + w * PRIV), *lds_k = lds_v + kTile * VROW;   // (lds_k: KL)
    const int kr = lane / LPRW, ch = lane % LPRW;
    constexpr int NK = !KL ? 2 * KS : NI;
    u32x4 kpre[NK], vpre[NI];
    int id_pre = 0;   // lane%32's token's document
    auto tile_at = [&](int n) -> int {
        if (SCORED && listed) return __builtin_amdgcn_readfirstlane(s_list[n] & 0x7fff);
        return n;
    };
    // (rows past the last key repeat it; rows of at most 2^25 bytes)
    auto prefetch_k = [&](int n) __attribute__((always_inline)) {
        const int k_lo = tile_at(n) * kTile, most = n_keys - 1 - k_lo;
        const char *tk = wk.k + (int64_t)k_lo * wk.st;
        if constexpr (!KL) {
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                const uint32_t off = (uint32_t)min(16 * kb + lr, most) * (uint32_t)wk.st + grp * 16;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) kpre[kb * KS + ks] = load16(tk, off + ks * 64);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NI; j++) kpre[j] = load16<ONCE>(tk, (uint32_t)min(j * RPI + kr, most) * (uint32_t)wk.st + ch * 16);
        }
        if (SCORED && docs) id_pre = docs[k_lo + min(lane & 31, most)];
    };
    auto prefetch_v = [&](int n) __attribute__((always_inline)) {
        const int k_lo = tile_at(n) * kTile, most = n_keys - 1 - k_lo;
        const char *tv = wk.v + (int64_t)k_lo * wk.st;
#pragma unroll
        for (int j = 0; j < NI; j++) vpre[j] = load16<ONCE>(tv, (uint32_t)min(j * RPI + kr, most) * (uint32_t)wk.st + ch * 16);
    };
    const float to_log2 = p.scale * kLog2e, cap_log2 = p.cap * kLog2e, to_cap = p.cap > 0.0f ? within_f32(p.scale / p.cap) : 0.0f;
    // key of score x of this lane, from the tile's first: groups of four consecutive ones
    auto key_of = [](int x) { return R == 16 ? 16 * (x >> 2) + (x & 3) : 8 * (x >> 2) + (x & 3); };   // + 4 grp

    if (first + w < n_tiles) prefetch_k(first + w), prefetch_v(first + w);
    u32x4 qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) qf[ks] = load16(p.q + out_row * (D * (int)sizeof(T)), ks * 16 * NG + grp * 16);
    for (int n = first + w; n < n_tiles; n += step) {
        const int k_lo = tile_at(n) * kTile;
        const bool by_id = SCORED && docs && !(listed && __builtin_amdgcn_readfirstlane(s_list[n] & 0x8000));
        const int id_tile = id_pre;
        const uint32_t padding = SCORED && by_id ? (uint32_t)__builtin_amdgcn_ballot_w64(id_tile < 0) : 0;   // a bit per key of the tile

        // ---- S^T = K Q^T --------------------------------------------------------------------------------------
        float s[NS];
        if constexpr (R == 16 && KL) {
#pragma unroll
            for (int j = 0; j < NI; j++) *reinterpret_cast<u32x4 *>(lds_k + (j * RPI + kr) * KROW + ch * (16 / (int)sizeof(T))) = kpre[j];
            if (n + step < n_tiles) prefetch_k(n + step);
            wave_sync();
            float4_t acc[2];
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int r = 0; r < 4; r++) acc[kb][r] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int kb = 0; kb < 2; kb++) {
                    const u32x4 kf = *reinterpret_cast<const u32x4 *>(lds_k + (16 * kb + lr) * KROW + (ks * 64 + grp * 16) / (int)sizeof(T));
                    if constexpr (H16) {
                        acc[kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, kf), __builtin_bit_cast(half8_t, qf[ks]), acc[kb], 0, 0, 0);
                    } else {
                        const float4_t a = __builtin_bit_cast(float4_t, kf), c = __builtin_bit_cast(float4_t, qf[ks]);
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[kb] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], c[e], acc[kb], 0, 0, 0);
                    }
                }
#pragma unroll
            for (int x = 0; x < NS; x++) s[x] = acc[x >> 2][x & 3];
        } else if constexpr (!KL) {
            float4_t acc[2];
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int r = 0; r < 4; r++) acc[kb][r] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int kb = 0; kb < 2; kb++) {   // (f32; one feature of each group's four at a time)
                    const float4_t a = __builtin_bit_cast(float4_t, kpre[kb * KS + ks]), c = __builtin_bit_cast(float4_t, qf[ks]);
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[kb] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], c[e], acc[kb], 0, 0, 0);
                }
#pragma unroll
            for (int x = 0; x < NS; x++) s[x] = acc[x >> 2][x & 3];
            if (n + step < n_tiles) prefetch_k(n + step);
        } else {
#pragma unroll
            for (int j = 0; j < NI; j++) *reinterpret_cast<u32x4 *>(lds_k + (j * RPI + kr) * KROW + ch * (16 / (int)sizeof(T))) = kpre[j];
            if (n + step < n_tiles) prefetch_k(n + step);
            wave_sync();
            float16_t acc;
#pragma unroll
            for (int r = 0; r < 16; r++) acc[r] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const u32x4 kf = *reinterpret_cast<const u32x4 *>(lds_k + lr * KROW + (ks * 32 + grp * 16) / (int)sizeof(T));
                if constexpr (H16) {
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, kf), __builtin_bit_cast(half8_t, qf[ks]), acc, 0, 0, 0);
                } else {
                    const float4_t a = __builtin_bit_cast(float4_t, kf), c = __builtin_bit_cast(float4_t, qf[ks]);
#pragma unroll
                    for (int e = 0; e < 4; e++) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], c[e], acc, 0, 0, 0);
                }
            }
#pragma unroll
            for (int x = 0; x < NS; x++) s[x] = acc[x];
        }
#pragma unroll
        for (int j = 0; j < NI; j++) {
            if (by_id && ((padding >> (j * RPI)) >> kr & 1)) vpre[j] = u32x4{0, 0, 0, 0};   // padding may hold anything
            *reinterpret_cast<u32x4 *>(lds_v + (j * RPI + kr) * VROW + ch * (16 / (int)sizeof(T))) = vpre[j];
        }
        if (n + step < n_tiles) prefetch_v(n + step);

        // ---- softmax of this lane's row over its keys k_lo + 4 grp + key_of(x) -----------------------------------
        if constexpr (SCORED) __builtin_amdgcn_sched_barrier(0);   // (V's fragments asked for during the scores' arithmetic spill registers)
        if constexpr (SCORED) {
            if (H16 && p.cap > 0.0f && p.cap <= kFastTanhCap) {
#pragma unroll
                for (int x = 0; x < NS; x++) s[x] = cap_log2 * fast_tanh(s[x] * to_cap);
            } else if (p.cap > 0.0f) {
#pragma unroll
                for (int x = 0; x < NS; x++) s[x] = cap_log2 * tanhf(s[x] * to_cap);
            } else {
#pragma unroll
                for (int x = 0; x < NS; x++) s[x] *= to_log2;
            }
            if (p.slopes) {
                const float d0 = (float)(at - k_lo - 4 * grp);
#pragma unroll
                for (int x = 0; x < NS; x++) s[x] = __builtin_fmaf(-slope, fabsf(d0 - (float)key_of(x)), s[x]);
            }
            if (by_id) {
#pragma unroll
                for (int x = 0; x < NS; x++) {
                    int id = __builtin_amdgcn_readlane(id_tile, key_of(x));
#pragma unroll
                    for (int y = 1; y < NG; y++) {
                        const int other = __builtin_amdgcn_readlane(id_tile, key_of(x) + 4 * y);
                        id = grp == y ? other : id;
                    }
                    s[x] = id == doc ? s[x] : -INFINITY;
                }
            }
        } else {
#pragma unroll
            for (int x = 0; x < NS; x++) s[x] *= to_log2;
        }
        const int last = lim - k_lo - 4 * grp;
        if (__builtin_amdgcn_ballot_w64(last < 28) != 0) {
#pragma unroll
            for (int x = 0; x < NS; x++) s[x] = key_of(x) <= last ? s[x] : -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int x = 1; x < NS; x++) top = fmaxf(top, s[x]);
#pragma unroll
        for (int d = R; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
        // f16: the reference moves only when the maximum exceeds it by more than 8 (weights reach 2^8 at most, far inside f16)
        // (the difference: m_run + 8 is m_run + 16 or m_run where a step of 32 bits is 16)
        const bool moved = less(top, m_run) > (H16 ? 8.0f : 0.0f);
        const float m_new = moved ? top : m_run, ref = m_new == -INFINITY ? 0.0f : m_new;
        const float keep = moved ? __builtin_amdgcn_exp2f(m_run - ref) : 1.0f;
        m_run = m_new;
        half8_t pf[NS / 8];
        float sum = 0.0f;
#pragma unroll
        for (int x = 0; x < NS; x++) {
            float e = __builtin_amdgcn_exp2f(less(s[x], ref));
            // The product with V takes f16 operands: weights are rounded, half a step each, and the row's sum takes the same ones, so that a row of
            // equal values stays that value.  (Their remainders would be a second product; outputs are off by 2.2e-4 to 2.7e-4 against 64 bits,
            // of which the result's own rounding is 2.1e-4.)
            if constexpr (H16) {
                pf[x >> 3][x & 7] = (_Float16)e;
                e = (float)pf[x >> 3][x & 7];
            }
            s[x] = e;
            sum += e;
        }
        l_run = l_run * keep + sum;
        if (__builtin_amdgcn_ballot_w64(moved) != 0) {
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int r = 0; r < NA; r++) o[db][r] *= keep;
        }
        if constexpr (SCORED) __builtin_amdgcn_sched_barrier(0);

        // ---- O^T += V^T P^T --------------------------------------------------------------------------------
        wave_sync();
        if constexpr (H16) {
            // this lane as a source of the transposing loads: key (lane%16)/4 of a group of four, features 4 (lane%4) of a block of 16
            const _Float16 *vsrc = reinterpret_cast<const _Float16 *>(lds_v) + (4 * grp + ((lane & 15) >> 2)) * VROW + (R == 32 ? 16 * ((lane >> 4) & 1) : 0) + 4 * (lane & 3);
#pragma unroll
            for (int st = 0; st < NS / 8; st++)
#pragma unroll
                for (int db = 0; db < DB; db++) {
                    // keys 4 grp + 0..3 of the two groups that the lane's weights st are of
                    const half4_t lo = lds_read_tr16(vsrc + key_of(8 * st) * VROW + R * db), hi = lds_read_tr16(vsrc + key_of(8 * st + 4) * VROW + R * db);
                    const half8_t vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                    if constexpr (R == 16) o[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[st], o[db], 0, 0, 0);
                    else o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[st], o[db], 0, 0, 0);
                }
        } else {
#pragma unroll
            for (int x = 0; x < NS; x++)
#pragma unroll
                for (int db = 0; db < DB; db++) {
                    const float a = lds_v[(key_of(x) + 4 * grp) * VROW + R * db + lr];
                    if constexpr (R == 16) o[db] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, s[x], o[db], 0, 0, 0);
                    else o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, s[x], o[db], 0, 0, 0);
                }
        }
        wave_sync();   // (the next tile goes where this one was)
    }

    // ---- the four waves' results joined ------------------------------------------------------------------------
    float *comb = reinterpret_cast<float *>(lds), *comb_ml = comb + kWaves * R * CROW;
#pragma unroll
    for (int d = R; d < 64; d <<= 1) l_run += __shfl_xor(l_run, d, 64);
    __syncthreads();   // the tiles are done with
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int x = 0; x < NA / 4; x++)
            *reinterpret_cast<float4_t *>(comb + (w * R + lr) * CROW + R * db + (R == 32 ? 8 : 16) * x + 4 * grp) = float4_t{o[db][4 * x], o[db][4 * x + 1], o[db][4 * x + 2], o[db][4 * x + 3]};
    if (grp < 2) comb_ml[(w * 2 + grp) * R + lr] = grp ? l_run : m_run;
    __syncthreads();
    constexpr int TPR = kThreads / R, PER = D / TPR;   // threads per row, features per thread
    const int row = tid / TPR, r = wk.row0 + row;
    if (r >= wk.row_end) return;
    float mm = -INFINITY, l = 0.0f, f[kWaves];
#pragma unroll
    for (int x = 0; x < kWaves; x++) mm = fmaxf(mm, comb_ml[x * 2 * R + row]);
    const float ref = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
    for (int x = 0; x < kWaves; x++) {
        f[x] = __builtin_amdgcn_exp2f(comb_ml[x * 2 * R + row] - ref);
        l += f[x] * comb_ml[(x * 2 + 1) * R + row];
    }
    const int64_t orow = q_row(p, wk.kvh, r).at;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < PER; e += 2) {
        const int d = (tid % TPR) * 2 + e * TPR;   // (8 bytes per thread, threads of a row side by side: a store covers whole lines)
        float2_t acc = {0.0f, 0.0f};
#pragma unroll
        for (int x = 0; x < kWaves; x++) {
            const float2_t v = *reinterpret_cast<const float2_t *>(comb + (x * R + row) * CROW + d);
#pragma unroll
            for (int y = 0; y < 2; y++) acc[y] = __builtin_fmaf(f[x], v[y], acc[y]);
        }
        if (p.splits == 1) {
            struct alignas(2 * sizeof(T)) Two { T e[2]; } two;
            two.e[0] = (T)(acc[0] * inv), two.e[1] = (T)(acc[1] * inv);
            *reinterpret_cast<Two *>(reinterpret_cast<T *>(p.out) + orow * D + d) = two;
        } else {
            put2(p.part_o + ((int64_t)wk.split * p.part_rows + orow) * D + d, acc);
        }
    }
    if (p.splits > 1 && tid % TPR == 0) {
        put(part_ml + orow, mm);
        put(part_ml + orow + p.part_rows, l);
    }
}

// A tile of 128 f16 rows over a prefix: a tile of 64 keys is staged once for the four waves, 32 rows each (as sdpa_scored.hip has
// it).  Tiles count 64 keys.  Always a part: `splits` > 1.
constexpr int kTallTile = 64;
template <int D>
__device__ __forceinline__ void tall_body(const RowsDev &p, const RowsWork &wk, unsigned char *lds) {
    constexpr int KS = D / 16, DB = D / 32, KROW = D + 8, VROW = D + 16;
    constexpr int PPR = D / 8, RPI = kThreads / PPR, NL = kTallTile / RPI;   // 16-byte pieces per row, rows per load of the workgroup, loads per tile and tensor
    constexpr int K_TILE = kTallTile * KROW, V_TILE = kTallTile * VROW;
    _Float16 *lds_k = reinterpret_cast<_Float16 *>(lds), *lds_v = lds_k + 2 * K_TILE;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hb = lane >> 5, l32 = lane & 31;
    const int my_row = wk.row0 + 32 * w + l32, n_tiles = (wk.tiles - wk.part + wk.parts - 1) / wk.parts;
    const bool wave_has_rows = wk.row0 + 32 * w < wk.row_end;
    const int64_t out_row = q_row(p, wk.kvh, min(my_row, wk.row_end - 1)).at;
    const int key0 = tid / PPR, ch = tid % PPR;
    const uint32_t lane_off = (uint32_t)key0 * (uint32_t)wk.st + ch * 16;
    u32x4 kpre[NL], vpre[NL];
    auto prefetch = [&](int n) __attribute__((always_inline)) {
        const int k_lo = (wk.part + n * wk.parts) * kTallTile, most = wk.n_keys - 1 - k_lo;
        const char *tk = wk.k + (int64_t)k_lo * wk.st, *tv = wk.v + (int64_t)k_lo * wk.st;
        if (most >= kTallTile - 1) {   // wave-uniform addresses and one offset per lane
            uint32_t o = lane_off;
            asm volatile("" : "+v"(o));   // (stays a 32-bit offset up to the loads)
#pragma unroll
            for (int j = 0; j < NL; j++) {
                kpre[j] = load16(tk + (int64_t)(j * RPI) * wk.st, o);
                vpre[j] = load16(tv + (int64_t)(j * RPI) * wk.st, o);
            }
        } else {   // rows past the last key repeat it
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const uint32_t o = (uint32_t)min(key0 + j * RPI, most) * (uint32_t)wk.st + ch * 16;
                kpre[j] = load16(tk, o);
                vpre[j] = load16(tv, o);
            }
        }
    };
    auto stage = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NL; j++) {
            *reinterpret_cast<u32x4 *>(lds_k + buf * K_TILE + (key0 + j * RPI) * KROW + ch * 8) = kpre[j];
            *reinterpret_cast<u32x4 *>(lds_v + buf * V_TILE + (key0 + j * RPI) * VROW + ch * 8) = vpre[j];
        }
    };
    float m_run = -INFINITY, s_ref = 0.0f, l_run = 0.0f;   // (a reference as sdpa_scored.hip has it: NaN from 2^20 on)
    float16_t o[DB];
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int x = 0; x < 16; x++) o[db][x] = 0.0f;
    const float to_log2 = p.scale * kLog2e;
    u32x4 qf[KS];
    prefetch(0);
#pragma unroll
    for (int ks = 0; ks < KS; ks++) qf[ks] = load16(p.q + out_row * (2 * D), 32 * ks + 16 * hb);
#pragma unroll
    for (int ks = 0; ks < KS; ks++) asm volatile("" : "+v"(qf[ks]));   // settled here, not by a wait in the loop that would take the prefetch in too
    stage(0);
    if (n_tiles > 1) prefetch(1);
    for (int n = 0; n < n_tiles; n++) {
        const int buf = n & 1;
        __syncthreads();   // tile n is in LDS; every wave is done with the buffers about to be overwritten
        if (wave_has_rows) {
            float16_t s[2];
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int x = 0; x < 16; x++) s[kb][x] = 0.0f;
            const _Float16 *ksrc = lds_k + buf * K_TILE + l32 * KROW + 8 * hb;
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int kb = 0; kb < 2; kb++)
                    s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const half8_t *>(ksrc + 32 * kb * KROW + 16 * ks), __builtin_bit_cast(half8_t, qf[ks]), s[kb], 0, 0, 0);
            // this lane's keys: 4 hb + c, c = 32 kb + 8 (x / 4) + x % 4
            const int last = wk.n_keys - 1 - (wk.part + n * wk.parts) * kTallTile - 4 * hb;
            if (last < 60) {
#pragma unroll
                for (int kb = 0; kb < 2; kb++)
#pragma unroll
                    for (int x = 0; x < 16; x++) s[kb][x] = 32 * kb + 8 * (x >> 2) + (x & 3) <= last ? s[kb][x] : -INFINITY;
            }
            // Weights against the reference that the row has.  Only in the first tile, and where a lane's come to 2^15 or more (f16 ends at 2^16), a
            // look at the maximum: the reference moves where that is more than 8 above it.
            half8_t pf[4];
            float sum;
            auto weights = [&](float from) __attribute__((always_inline)) {
                const half2_t ones = {(_Float16)1.0f, (_Float16)1.0f};
                sum = 0.0f;
#pragma unroll
                for (int st = 0; st < 4; st++) {
#pragma unroll
                    for (int x = 0; x < 8; x++) pf[st][x] = (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[st >> 1][8 * (st & 1) + x], to_log2, from));
#pragma unroll
                    for (int x = 0; x < 4; x++) sum = __builtin_amdgcn_fdot2(half2_t{pf[st][2 * x], pf[st][2 * x + 1]}, ones, sum, false);   // the same rounded weights (see rows_body)
                }
            };
            bool look = n == 0;
            if (!look) {
                weights(-m_run);
                look = __builtin_amdgcn_ballot_w64(!(sum < 32768.0f)) != 0;
            }
            if (look) {
                float top = s[0][0];
#pragma unroll
                for (int kb = 0; kb < 2; kb++)
#pragma unroll
                    for (int x = 0; x < 16; x++) top = fmaxf(top, s[kb][x]);
                const float s_top = fmaxf(top, __shfl_xor(top, 32, 64));
                top = s_top * to_log2;   // (scale > 0: the maximum commutes with it)
                const bool far = m_run != m_run, moved = top > m_run + 8.0f || (far && s_top > s_ref);
                const float keep = moved ? __builtin_amdgcn_exp2f(far ? (s_ref - s_top) * to_log2 : m_run - top) : 1.0f;
                if (moved) s_ref = s_top, m_run = fabsf(top) < 0x1p20f ? top : __builtin_nanf("");
                l_run *= keep;
#pragma unroll
                for (int db = 0; db < DB; db++)
#pragma unroll
                    for (int x = 0; x < 16; x++) o[db][x] *= keep;
                float from = -m_run;
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(m_run != m_run) != 0, 0)) {
                    const float less = m_run != m_run ? s_ref : 0.0f;   // (rows of ordinary scores stay as they are)
#pragma unroll
                    for (int kb = 0; kb < 2; kb++)
#pragma unroll
                        for (int x = 0; x < 16; x++) s[kb][x] -= less;
                    if (m_run != m_run) from = 0.0f;
                }
                weights(from);
            }
            l_run += sum;
            const _Float16 *vsrc = lds_v + buf * V_TILE + (4 * hb + ((lane & 15) >> 2)) * VROW + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
            for (int st = 0; st < 4; st++)
#pragma unroll
                for (int db = 0; db < DB; db++) {
                    const half4_t lo = lds_read_tr16(vsrc + 16 * st * VROW + 32 * db), hi = lds_read_tr16(vsrc + (16 * st + 8) * VROW + 32 * db);
                    o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), pf[st], o[db], 0, 0, 0);
                }
        }
        if (n + 1 < n_tiles) {   // the next tile to LDS after this one's arithmetic
            stage(buf ^ 1);
            if (n + 2 < n_tiles) prefetch(n + 2);
        }
    }
    l_run += __shfl_xor(l_run, 32, 64);
    if (m_run != m_run) m_run = s_ref * to_log2;
    if (my_row < wk.row_end) p.part_ml[((int64_t)wk.split * 2 + hb) * p.part_rows + out_row] = hb ? l_run : m_run;
    // rows to their places in whole lines, through a corner of LDS of the wave's own
    constexpr int CROW = D + 4, LPR = D / 4, RPS = 64 / LPR;
    static_assert(kWaves * 32 * CROW * 4 <= 2 * (K_TILE + V_TILE) * 2, "the output goes through the tiles' LDS");
    float *tr = reinterpret_cast<float *>(lds) + w * 32 * CROW;
    __syncthreads();
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int x = 0; x < 4; x++) *reinterpret_cast<float4_t *>(tr + l32 * CROW + 32 * db + 8 * x + 4 * hb) = float4_t{o[db][4 * x], o[db][4 * x + 1], o[db][4 * x + 2], o[db][4 * x + 3]};
    wave_sync();
    float *po = p.part_o + (int64_t)wk.split * p.part_rows * D;
#pragma unroll 4
    for (int j = 0; j < 32 / RPS; j++) {
        const int row = j * RPS + lane / LPR, r = wk.row0 + 32 * w + row;
        if (r < wk.row_end) *reinterpret_cast<float4_t *>(po + q_row(p, wk.kvh, r).at * D + lane % LPR * 4) = *reinterpret_cast<const float4_t *>(tr + row * CROW + lane % LPR * 4);
    }
}

// Whether a part has keys for a row: one without has a maximum of -inf and a sum of 0 (and rows of zeros, or none at all).  Scores that are all
// NaN raise no maximum either, but their sum is NaN, which has to come out.
__device__ __forceinline__ bool part_has(float m, float l) { return m != -INFINITY || l != 0.0f; }

// A row's parts -> its output, by D / 4 lanes of a wave.  Everything that some 8 ranges have is asked for at once: one latency for up to
// 8 of them.  (At most 64.)
template <typename T, int D>
__device__ __forceinline__ void join_row(const float *part_o, const float *part_ml, T *out, int64_t row, int64_t rows, int splits) {
    constexpr int LPR = D / 4, MOST = 64 / LPR, BATCH = 8;
    const int lr = threadIdx.x % LPR;
    const float *po = part_o + row * D + 2 * lr;   // this lane's features: two, and two half a row on
    float f[MOST], ls[MOST], l = 0.0f, mm = -INFINITY;
#pragma unroll
    for (int x = 0; x < MOST; x++) {
        const int s = min(x * LPR + lr, splits - 1);
        f[x] = get(part_ml + (int64_t)s * 2 * rows + row);
        ls[x] = get(part_ml + ((int64_t)s * 2 + 1) * rows + row);
    }
    float2_t v[BATCH][2];
    auto ask = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
        for (int y = 0; y < BATCH; y++) {
            const float *at = po + (int64_t)min(s0 + y, splits - 1) * rows * D;
            v[y][0] = get2(at), v[y][1] = get2(at + D / 2);
        }
    };
    ask(0);
#pragma unroll
    for (int x = 0; x < MOST; x++) {
        if (x * LPR + lr >= splits) f[x] = -INFINITY, ls[x] = 0.0f;
        mm = fmaxf(mm, f[x]);
    }
#pragma unroll
    for (int w = 1; w < LPR; w <<= 1) mm = fmaxf(mm, __shfl_xor(mm, w, 64));
    const float ref = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
    for (int x = 0; x < MOST; x++) {
        const bool has = part_has(f[x], ls[x]);
        f[x] = has ? __builtin_amdgcn_exp2f(f[x] - ref) : 0.0f;
        l += has ? f[x] * ls[x] : 0.0f;
    }
#pragma unroll
    for (int w = 1; w < LPR; w <<= 1) l += __shfl_xor(l, w, 64);
    float2_t acc[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
    for (int s0 = 0; s0 < splits; s0 += BATCH) {
#pragma unroll
        for (int y = 0; y < BATCH; y++) {
            float g = 0.0f;
#pragma unroll
            for (int x = 0; x < MOST; x++) {
                const float h = __shfl(f[x], (s0 + y) % LPR, LPR);
                g = (s0 + y) / LPR == x ? h : g;
            }
            if (s0 + y >= splits) g = 0.0f;
#pragma unroll
            for (int z = 0; z < 2; z++)
#pragma unroll
                for (int e = 0; e < 2; e++) acc[z][e] = g != 0.0f ? __builtin_fmaf(g, v[y][z][e], acc[z][e]) : acc[z][e];
        }
        if (s0 + BATCH < splits) ask(s0 + BATCH);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;   // (a sum of NaN comes out)
#pragma unroll
    for (int z = 0; z < 2; z++) {
        struct alignas(2 * sizeof(T)) Two { T e[2]; } pair;
        pair.e[0] = (T)(acc[z][0] * inv), pair.e[1] = (T)(acc[z][1] * inv);
        *reinterpret_cast<Two *>(out + row * D + z * (D / 2) + 2 * lr) = pair;
    }
}

// The last workgroup to bring a part of a unit's rows joins them.  A unit is a tile of one sequence's rows (own keys) or, where no
// sequence has keys of its own, a tile of rows of the prefix; a tile over the prefix holds rows of up to 16 units and brings a
// part to each.  Counters are zero between launches.
template <typename T, int D, int PRE, int OWN>
__device__ __forceinline__ void arrive(const RowsDev &p, const RowsWork &wk, uint32_t *s_done) {
    const int tid = threadIdx.x, seq_rows = p.Sq * p.G, n_units = p.own_row_tiles ? p.B * p.own_row_tiles : p.p_row_tiles;
    auto unit_of = [&](int r) {
        if (!p.own_row_tiles) return r / (PRE ? PRE : 1);
        const int b = p.by_sq.by(p.by_g.by(r));
        return b * p.own_row_tiles + (r - b * seq_rows) / OWN;
    };
    auto rows_of = [&](int u, int &r0, int &r1) {
        if (!p.own_row_tiles) {
            r0 = u * (PRE ? PRE : 1), r1 = min(r0 + (PRE ? PRE : 1), p.B * seq_rows);
        } else {
            const int b = p.by_own_row_tiles.by(u);
            r0 = b * seq_rows + (u - b * p.own_row_tiles) * OWN, r1 = min(r0 + OWN, (b + 1) * seq_rows);
        }
    };
    const int first = unit_of(wk.row0), n = unit_of(wk.row_end - 1) - first + 1;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this thread's parts have completed
    __syncthreads();                                     // ... and so have the whole workgroup's
    if (tid < 64) {
        bool last = false;
        if (tid < n) {
            int r0, r1;
            rows_of(first + tid, r0, r1);
            int parts = p.p_splits;
            if (p.own_row_tiles) parts = p.own_splits + (PRE ? parts * ((r1 - 1) / (PRE ? PRE : 1) - r0 / (PRE ? PRE : 1) + 1) : 0);
            int *counter = p.counters + (int64_t)wk.kvh * n_units + first + tid;
            last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
            if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        const uint64_t done = __builtin_amdgcn_ballot_w64(last);
        if (tid == 0) *s_done = (uint32_t)done;   // (n <= 16)
    }
    __syncthreads();
    const uint32_t done = *s_done;
    if (done == 0) return;
    int begin, end, unused;
    rows_of(first, begin, unused), rows_of(first + n - 1, unused, end);
    constexpr int LPR = D / 4;
    for (int r = begin + tid / LPR; r < end; r += kThreads / LPR)   // (whole groups of LPR lanes stay or leave)
        if ((done >> (unit_of(r) - first)) & 1)
            join_row<T, D>(p.part_o, p.part_ml, reinterpret_cast<T *>(p.out), q_row(p, wk.kvh, r).at, p.part_rows, p.splits);
}

constexpr int rows_lds(int es, int D, int R) {   // rows_body's LDS
    return kWaves * kTile * ((es == 2 ? D + 16 : R == 16 ? D + 4 : D + 8) + (R == 32 || es == 2 ? (es == 2 ? D + 8 : D + 4) : 0)) * es;
}
constexpr int tall_lds(int D) { return 2 * kTallTile * (2 * D + 24) * 2; }
constexpr int most_of(int a, int b) { return a > b ? a : b; }

// PRE: rows of a tile over the prefix, 128 the tall body (0: there is none); OWN: over own keys.
template <typename T, int D, int PRE, int OWN, bool SCORED, bool ONCE>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 && D == 128 && (PRE == 32 || OWN == 32) ? 1 : 2) void sdpa_rows_kernel(RowsCall call) {
    const RowsDev &p = call.p;
    constexpr int ES = sizeof(T);
    __shared__ __attribute__((aligned(16))) unsigned char lds[most_of(rows_lds(ES, D, OWN), PRE == 128 ? tall_lds(D) : PRE ? rows_lds(ES, D, PRE) : 0)];
    __shared__ uint16_t s_list[SCORED ? kListMax : 1];
    __shared__ int s_counts[kWaves];
    __shared__ uint32_t s_done;
    int item = blockIdx.y + blockIdx.z * gridDim.y;   // (z: a grid's y has 65535 places)
    if (item >= p.items) return;
    bool there = false;   // the work is done
    RowsWork wk;
    wk.kvh = blockIdx.x;   // (consecutive workgroups go to the 8 XCDs in turn: a kv head's keys meet in few L2 caches)
    if (PRE && item < p.p_items) {
        constexpr int ROWS = PRE ? PRE : 1, TILE = PRE == 128 ? kTallTile : kTile;
        wk.b = -1;
        wk.split = p.by_p_row_tiles.by(item);
        wk.row0 = (item - wk.split * p.p_row_tiles) * ROWS, wk.row_end = min(wk.row0 + ROWS, p.B * p.Sq * p.G);
        wk.k = p.pk + (int64_t)wk.kvh * p.p_stride_h, wk.v = p.pv + (int64_t)wk.kvh * p.p_stride_h, wk.st = p.p_stride_t;
        wk.n_keys = p.P;
        wk.tiles = (p.P + TILE - 1) / TILE, wk.part = wk.split, wk.parts = p.p_splits;
        if constexpr (PRE == 128) {
            tall_body<D>(p, wk, lds);
            return;
        } else if constexpr (PRE != 0 && PRE != OWN) {
            rows_body<T, D, PRE, false, false>(p, wk, lds, nullptr, nullptr);
            there = true;
        }
    } else {
        if (PRE) item -= p.p_items;
        const int at = p.by_own_splits.by(item), split = item - at * p.own_splits, b = p.by_own_row_tiles.by(at);
        const int rt = p.own_row_tiles - 1 - (at - b * p.own_row_tiles);   // (the longest first)
        wk.b = p.seq0 + b;
        const OwnKeys own = own_keys(p, wk.b, wk.kvh);
        wk.k = own.k, wk.v = own.v, wk.st = p.stride_t, wk.n_keys = own.len;
        wk.row0 = wk.b * p.Sq * p.G + rt * OWN, wk.row_end = min(wk.row0 + OWN, (wk.b + 1) * p.Sq * p.G);
        int n_vis = own.len;
        if (p.causal) {
            n_vis = p.by_g.by(wk.row_end - 1) - wk.b * p.Sq + own.len - p.Sq + 1;
            if (SCORED && p.prefix_lens) n_vis = max(n_vis, p.prefix_lens[wk.b]);
            n_vis = max(0, min(n_vis, own.len));
        }
        wk.tiles = (n_vis + kTile - 1) / kTile, wk.part = split, wk.parts = min(p.own_splits, max(1, p.by_own_tiles.by(wk.tiles + p.own_tiles - 1)));
        wk.split = p.p_splits + split;
    }
    if (!there) rows_body<T, D, OWN, SCORED, ONCE>(p, wk, lds, s_list, s_counts);
    if constexpr (PRE <= 16 && OWN == 16)   // (parts of more rows are joined by a launch)
        if (p.counters) arrive<T, D, PRE, OWN>(p, wk, &s_done);
}

// The same in a launch of its own: after tall tiles, whose last workgroup would have 128 rows to join.  NG groups of D / 4 lanes take a row's
// parts in turn, so that all of 8 NG are asked for at once; one group where there are no more than 8.  (f16: 2048 rows of 17 parts,
// D = 128, the call in one group each 40.6 us, in two 39.7; 12800 rows of 4 parts, D = 64, 25.2 us, in four groups 27.1.)
template <typename T, int D, int NG>
__global__ __launch_bounds__(256) void sdpa_rows_merge_kernel(const float *__restrict__ part_o, const float *__restrict__ part_ml, T *__restrict__ out, int64_t rows, int splits) {
    constexpr int LPR = D / 4, LANES = LPR * NG, BATCH = 8;
    const int lane = threadIdx.x % LANES, grp = lane / LPR, lr = lane % LPR;
    const int64_t row = min((int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES, rows - 1);   // (rows past the last write it again, the same)
    const int mine = min(lane, splits - 1);   // (no more parts than lanes: 64, or 8)
    float f = part_ml[(int64_t)mine * 2 * rows + row];
    float ls = part_ml[((int64_t)mine * 2 + 1) * rows + row];
    const float *po = part_o + row * D + 4 * lr;
    float4_t v[BATCH];
    auto ask = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
        for (int y = 0; y < BATCH; y++) v[y] = *reinterpret_cast<const float4_t *>(po + (int64_t)min(s0 + y * NG + grp, splits - 1) * rows * D);
    };
    ask(0);
    if (lane >= splits) f = -INFINITY, ls = 0.0f;
    float mm = f;
#pragma unroll
    for (int w = 1; w < LANES; w <<= 1) mm = fmaxf(mm, __shfl_xor(mm, w, 64));
    const bool has = part_has(f, ls);
    f = has ? __builtin_amdgcn_exp2f(f - (mm == -INFINITY ? 0.0f : mm)) : 0.0f;
    float l = has ? f * ls : 0.0f;
#pragma unroll
    for (int w = 1; w < LANES; w <<= 1) l += __shfl_xor(l, w, 64);
    float4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < splits; s0 += BATCH * NG) {
#pragma unroll
        for (int y = 0; y < BATCH; y++) {
            const float h = __shfl(f, (s0 + y * NG + grp) % LANES, LANES), g = s0 + y * NG + grp < splits ? h : 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] = g != 0.0f ? __builtin_fmaf(g, v[y][e], acc[e]) : acc[e];
        }
        if (s0 + BATCH * NG < splits) ask(s0 + BATCH * NG);
    }
#pragma unroll
    for (int w = LPR; w < LANES; w <<= 1)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[e] += __shfl_xor(acc[e], w, 64);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;   // (a sum of NaN comes out)
    if (grp == 0) {
        struct alignas(4 * sizeof(T)) Four { T e[4]; } four;
#pragma unroll
        for (int e = 0; e < 4; e++) four.e[e] = (T)(acc[e] * inv);
        *reinterpret_cast<Four *>(out + row * D + 4 * lr) = four;
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
    const int64_t row_bytes = a.D * (int64_t)elem_bytes(a.dtype);
    const bool whole = row_bytes % 4 == 0 && (uintptr_t)k_new % 4 == 0 && (uintptr_t)v_new % 4 == 0;   // (f16 rows of an odd size are not)
    const int64_t words = a.Sq * row_bytes / (whole ? 4 : 2);
    TROCM_REQUIRE(words < (1 << 30), "append: too many new tokens");
    if (words == 0) return 0;
    const int64_t step = table_holds(a);
    for (int64_t b = 0; b < a.B; b += step) {
        const int64_t n = a.B - b < step ? a.B - b : step;
        SeqTable tab;
        fill_table(a, b, n, tab);
        const int64_t blocks = (words + 255) / 256;
        const dim3 grid((unsigned)(blocks < 64 ? blocks : 64), (unsigned)a.Hkv, (unsigned)n);
        if (whole) hipLaunchKernelGGL((append_rows_kernel<uint32_t>), grid, dim3(256), 0, s, tab, (const uint32_t *)k_new, (const uint32_t *)v_new, (int)b, (int)a.Hkv, (int)words, row_bytes);
        else hipLaunchKernelGGL((append_rows_kernel<uint16_t>), grid, dim3(256), 0, s, tab, (const uint16_t *)k_new, (const uint16_t *)v_new, (int)b, (int)a.Hkv, (int)words, row_bytes);
        if (check_launch("append_rows")) return 1;
    }
    return 0;
}

namespace {

template <typename T, int D, int PRE, int OWN, bool SCORED, bool ONCE>
int launch_tiles(const SdpaRowsArgs &a, RowsCall &call, hipStream_t s) {
    RowsDev &p = call.p;
    const int64_t prefix_items = (int64_t)p.p_splits * p.p_row_tiles, per_seq = (int64_t)p.own_row_tiles * p.own_splits, most = 1 << 30, in_y = 65535;
    int64_t holds = table_holds(a);   // sequences of a launch
    if (per_seq && holds > (most - prefix_items) / per_seq) holds = (most - prefix_items) / per_seq;
    TROCM_REQUIRE(holds > 0 && prefix_items <= most, "attention: too many workgroups");
    TROCM_REQUIRE(!p.counters || (PRE <= 16 && OWN == 16), "attention: parts that nothing joins");
    for (int64_t b = 0; b < a.B; b += holds) {   // the prefix, for all rows, with the first sequences' own keys
        const int64_t n = a.B - b < holds ? a.B - b : holds;
        fill_table(a, b, n, call.tab);
        p.seq0 = (int)b;
        p.p_items = b == 0 ? (int)prefix_items : 0;
        p.items = (int)(p.p_items + n * per_seq);
        if (p.items == 0) continue;
        hipLaunchKernelGGL((sdpa_rows_kernel<T, D, PRE, OWN, SCORED, ONCE>), dim3((unsigned)a.Hkv, (unsigned)(p.items < in_y ? p.items : in_y), (unsigned)((p.items + in_y - 1) / in_y)), dim3(kThreads), 0, s, call);
        if (check_launch("sdpa_rows")) return 1;
    }
    if (p.splits > 1 && !p.counters) {
        if (p.splits <= 8) hipLaunchKernelGGL((sdpa_rows_merge_kernel<T, D, 1>), dim3((unsigned)((p.part_rows * (D / 4) + 255) / 256)), dim3(256), 0, s, p.part_o, p.part_ml, (T *)p.out, p.part_rows, p.splits);
        else hipLaunchKernelGGL((sdpa_rows_merge_kernel<T, D, 256 / D>), dim3((unsigned)((p.part_rows + 3) / 4)), dim3(256), 0, s, p.part_o, p.part_ml, (T *)p.out, p.part_rows, p.splits);
        if (check_launch("sdpa_rows_merge")) return 1;
    }
    return 0;
}

// ONCE where it pays, for tiles of 16 rows: keys that one workgroup reads, and that are more than the 256 MB behind the L2 caches keep from call
// to call.  (Through the caches | past them, us: 8 x 8193 keys of 8 x 128 features 50.3 | 45.6, 16 x 6000 73.5 | 65.1, 64 x 8192 + 512 35.7 | 32.1;
// but 64 x 512 17.3 | 18.2, one sequence of 8193 14.4 | 15.2.  f32, where it is the values alone, since a key's row is read in pieces of 64
// bytes: 16 x 4096 + 600 35.5 | 31.5, 4 x 5000 capped 38.0 | 35.5; with the keys as well 37.2.)
template <typename T, int D, int PRE, bool SCORED>
int launch_tiles_16(const SdpaRowsArgs &a, RowsCall &call, bool once, hipStream_t s) {
    if (once) return launch_tiles<T, D, PRE, 16, SCORED, true>(a, call, s);
    return launch_tiles<T, D, PRE, 16, SCORED, false>(a, call, s);
}

template <typename T, int D>
int launch_tiles_of(const SdpaRowsArgs &a, RowsCall &call, int pre, int own, bool is_scored, bool once, hipStream_t s) {
    if constexpr (sizeof(T) == 2 || D == 128)
        if (own == 32 && is_scored) return launch_tiles<T, D, 0, 32, true, false>(a, call, s);
    if (is_scored) return launch_tiles_16<T, D, 0, true>(a, call, once, s);
    if constexpr (sizeof(T) == 2)
        if (pre == 128) return own == 32 ? launch_tiles<T, D, 128, 32, false, false>(a, call, s) : launch_tiles_16<T, D, 128, false>(a, call, once, s);
    if constexpr (sizeof(T) == 2 || D == 128)
        if (own == 32) return launch_tiles<T, D, 32, 32, false, false>(a, call, s);
    if constexpr (sizeof(T) == 2 && D == 128)
        if (pre == 32) return launch_tiles_16<T, D, 32, false>(a, call, once, s);
    return launch_tiles_16<T, D, 16, false>(a, call, once, s);
}

// Sequences of one length: how many of its `all` key tiles a part of each unit of rows takes.  A workgroup's round of a tile per wave takes
// `full` us where `target` workgroups share the memory's rate, and no less than `least` where fewer do; no more of them than that, or
// another turn of all (f16, us, by parts: 4 x 8193 keys x 8 kv heads 1: 109, 2: 61, 4: 37.1, 6: 29.1, 8: 29.5, 16: 30.6; one sequence
// 8: 18.0, 16: 13.7, 32: 14.7; eight 2: 64.0, 3: 50.3, 4: 51.1, 5: 59.2, 8: 52.3).
int64_t tiles_of_a_part(int64_t units, int64_t all, int64_t es, int64_t D) {
    const double kb = (double)(kTile * D * es * 2) / 1024, cus = num_compute_units();
    const double target = kb < 16 ? 2 * cus : cus, least = es == 4 ? 4.7 * (D == 128 ? 1.0 : 0.55) : 1.85, full = kb < 16 ? 3.05 : 3.05 * kb / 16;
    int64_t best_n = 1;
    double best = 1e30;
    for (int64_t n = 1; n <= 64 && n <= (all + kWaves - 1) / kWaves; n++) {
        const double wgs = (double)(units * n), turns = (double)(int64_t)((wgs + target - 1) / target), share = full * (wgs < target ? wgs / target : 1.0);
        const double rounds = (double)((all + kWaves * n - 1) / (kWaves * n));
        const double t = turns * (2.5 + rounds * (share > least ? share : least)) + (n > 1 ? 1.0 + 0.25 * (double)n : 0.0);
        if (t < best) best = t, best_n = n;
    }
    return (all + best_n - 1) / best_n;
}

// What a call is expected to take (us) with `pn` parts of the prefix and `on` of the own keys.  A workgroup takes `start` and a round, a
// tile for each of its waves, `p_round` or `o_round`.  The call takes the longest workgroup and some more where not all run at once; or
// what memory needs for the keys and parts, and the last one's tail; or the workgroups' rounds over all that run at once; and the join.  The
// constants were fitted to 767 measured choices of 46 calls (f16 and f32, 64 and 128 features, 1 to 200 sequences, prefixes of 0 to
// 30000 keys), of which it picked one within 2 % of the best on average and 15 % at worst.
struct RowsCost {
    int64_t kv_heads, units, p_row_tiles, p_all, own_all;   // units: rows' tiles of all sequences, over own keys
    int pre, own;
    double o_round, p_round, slots, bytes_us, part_mb;
    bool merged;   // parts are joined by a launch of their own
    double rounds(int64_t tiles, int64_t parts) const { return (double)(((uint32_t)(tiles + parts - 1) / (uint32_t)parts + kWaves - 1) / kWaves); }
    double us(int64_t pn, int64_t on, double own_wgs, double own_rounds) const {
        const double start = 2.1, parts = (double)(pn + on), wgs_p = (double)(kv_heads * p_row_tiles * pn), all_own = (double)(kv_heads * units * on);
        const double p_chain = pn ? start + (pre == 128 ? (double)((p_all + pn - 1) / pn) : rounds(p_all, pn)) * p_round : 0.0;
        const double o_chain = on ? start + rounds(own_all, on) * o_round : 0.0, longest = p_chain > o_chain ? p_chain : o_chain;
        const double run = longest + (own_wgs + wgs_p > slots ? 0.7 * o_chain : 0.0);
        const double memory = start + bytes_us + 0.43 * parts * part_mb + 0.24 * longest;
        const double busy = (own_rounds * o_round + all_own * 2.2 * start + wgs_p * p_chain) / slots + 0.26 * longest;
        const double most = run > memory ? (run > busy ? run : busy) : (memory > busy ? memory : busy);
        return most + (parts <= 1 ? 0.0 : merged ? 2.0 + parts * (0.07 + 0.64 * part_mb) : 1.0 + parts * (0.27 + 3.1 * part_mb));
    }
};

// On the matrix cores: 0 done, 1 failed, 2 not covered.
int launch_sdpa_rows_tiles(const SdpaRowsArgs &a, hipStream_t s) {
    const int64_t es = (int64_t)elem_bytes(a.dtype);
    if (a.D != 64 && a.D != 128) return 2;
    const int64_t G = a.Hq / a.Hkv, rows = a.B * a.Sq * G, rows_all = rows * a.Hkv;
    if (rows >= (1ll << 30)) return 2;
    auto aligned = [&](const void *x) { return (uintptr_t)x % 16 == 0; };
    auto strides = [&](int64_t x) { return x * es % 16 == 0; };
    int64_t longest = a.lens || a.seqs ? 0 : a.Sk, own_tiles_all = 0;
    const int64_t seq_rows = a.Sq * G;
    bool ok = aligned(a.q) && aligned(a.out) && a.stride_t * es <= (1 << 25) && a.p_stride_t * es <= (1 << 25) && strides(a.stride_t);
    for (int64_t b = 0; b < a.B && (a.lens || a.seqs); b++) {
        const int64_t n = a.lens ? a.lens[b] : a.seqs[b].len;
        longest = n > longest ? n : longest;
        own_tiles_all += (n + kTile - 1) / kTile;
        if (a.seqs && n) ok = ok && aligned(a.seqs[b].k) && aligned(a.seqs[b].v) && strides(a.seqs[b].stride_h);
    }
    if (!(a.lens || a.seqs)) own_tiles_all = a.B * ((a.Sk + kTile - 1) / kTile);
    if (a.P) ok = ok && aligned(a.pk) && aligned(a.pv) && strides(a.p_stride_h) && strides(a.p_stride_t);
    if (longest && !a.seqs) ok = ok && aligned(a.k) && aligned(a.v) && strides(a.stride_b) && strides(a.stride_h);
    if (!ok || (a.P == 0 && longest == 0)) return 2;

    const bool is_scored = a.softcap > 0.0f || a.slopes || a.documents || a.prefix_lens;
    // Rows of a tile over own keys, where a sequence has more than 16 (tiles of 16 | 32, us).  f16: 6 queries of 4 heads a kv head behind 5000 keys
    // 27.7 | 22.9, 40 behind 8000 36.5 | 27.0, 300 of 64 features 10.0 | 8.5.  f32 of 128 features: 333 behind 1000 in documents 51.4 | 48.6,
    // without 108 | 118, 500 45.7 | 41.1, 10 behind 8000 41.6 | 35.2; of 64: 900 27.9 | 35.5, 10 behind 8000 23.9 | 28.0.
    const int own = seq_rows <= 16 || (es == 4 && a.D == 64) ? 16 : 32;
    const int64_t room = a.workspace && aligned(a.workspace) && a.workspace_bytes > kWsCounterBytes + kWsPlanBytes + 256
                             ? (int64_t)(a.workspace_bytes - kWsCounterBytes - kWsPlanBytes - 256) / ((a.D + 2) * (int64_t)sizeof(float)) / rows_all : 0;
    // Rows of a tile over the prefix.  f16: 128 from so many rows times keys on; under that 32 at 128 features, 16 at 64.  (16 | 32 | 128 rows,
    // us, 128 features: 64 rows over 8192 keys 18.8 | 16.1 | 17.9, 256 over 2500 18.8 | 15.0 | 17.5, 256 over 8192 39 | 28.5 | 24.7, 1024 over 700 37 |
    // 25.1 | 25.7, 1024 over 8192 113 | 82 | 60; 64 features: 40 over 700 7.3 | 9.8 | 10.1, 80 over 4000 10.5 | 14.1 | 11.6, 320 over 700 10.4 | 10.9 |
    // 10.9, 160 over 4000 13.8 | 15.9 | 12.4, 1600 over 1500 33 | 30 | 24.)  The tall body stores parts only and takes the largest product for the largest score.
    const bool tall = es == 2 && rows > 32 && a.P > kTallTile && room >= 2 && a.scale > 0.0f && rows * a.P > (a.D == 128 ? 1150000 : 450000);
    const int pre = a.P == 0 || es == 4 ? own : tall ? 128 : rows > 16 && (a.D == 128 || own == 32) ? 32 : own;
    RowsCall call;
    RowsDev &p = call.p;
    fill_rows(a, p);
    const int64_t p_tile = pre == 128 ? kTallTile : kTile, p_all = (a.P + p_tile - 1) / p_tile, own_all = (longest + kTile - 1) / kTile;
    p.p_row_tiles = a.P ? (int)((rows + pre - 1) / pre) : 0;
    p.own_row_tiles = longest ? (int)((seq_rows + own - 1) / own) : 0;
    // Into how many parts the keys go (at most as many as there is room for).
    const bool f32 = es == 4, uniform = !a.lens && !a.seqs;
    const double wide = a.D == 128 ? 1.0 : 0.5, cus = num_compute_units();
    auto round_of = [&](int rows_) { return f32 ? (rows_ == 32 ? 4.6 * wide : 4.4 * (0.43 + 0.57 * wide)) : (rows_ == 32 ? 2.0 : 1.26) * (0.35 + 0.65 * wide); };
    RowsCost cost;
    cost.kv_heads = a.Hkv, cost.units = a.B * p.own_row_tiles, cost.p_row_tiles = p.p_row_tiles, cost.p_all = p_all, cost.own_all = own_all;
    cost.pre = pre, cost.own = own, cost.o_round = round_of(own), cost.p_round = pre == 128 ? 2.26 * (0.35 + 0.65 * wide) : round_of(pre);
    cost.slots = cus * (a.D == 64 ? 3 : f32 && (own == 32 || pre == 32) ? 1 : 2);
    cost.bytes_us = (double)((own_tiles_all + p_all * (p_tile / kTile)) * kTile * a.Hkv) * (double)(a.D * es * 2) / 5e6;
    cost.part_mb = (double)rows_all * (double)(a.D + 2) * 4e-6;
    // Joined by the last to arrive where that is at most 16 rows: 4 x 777 + 40 keys 9.5 -> 8.5 us; but 16 x 2000 + 600 keys in tiles of 32 rows
    // over the prefix 13.5 -> 19.3 us, 10 x 4000 + 50 of 64 features 10.4 -> 14.
    const int64_t joined = a.P ? (rows < pre ? rows : pre) : own, units = a.Hkv * (p.own_row_tiles ? a.B * p.own_row_tiles : p.p_row_tiles);
    cost.merged = joined > 16 || units > (int64_t)(kWsCounterBytes / sizeof(int));
    const int64_t p_most = a.P ? (pre == 128 ? p_all : (p_all + kWaves - 1) / kWaves) : 0, o_most = longest ? (own_all + kWaves - 1) / kWaves : 0;
    static const int kParts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
    const int64_t p_least = pre == 128 && o_most == 0 ? 2 : 1, parts_most = room < 64 ? room : 64;
    const bool fixed = uniform && longest && (a.documents || p.own_row_tiles == 1);
    int64_t fixed_n = 1;   // (documents: how much of its keys a row's document has is not known here)
    if (fixed && p.own_row_tiles == 1) {
        const int64_t per = tiles_of_a_part(a.Hkv * a.B, own_all, es, a.D);
        fixed_n = (own_all + per - 1) / per;
        if (fixed_n > parts_most) fixed_n = parts_most > 1 ? parts_most : 1;
    }
    double best = 1e30;
    for (int x = 0; x < (int)(sizeof(kParts) / sizeof(int)); x++) {
        if (x && (fixed || kParts[x - 1] >= o_most)) break;
        const int64_t on = fixed ? fixed_n : kParts[x] < o_most ? kParts[x] : o_most;
        // tiles of a part; workgroups with something to do, and their rounds
        const int64_t op = on ? (own_all + on - 1) / on : 1;
        double own_wgs = 0.0, own_rounds = 0.0;
        auto add = [&](int64_t tiles, double times) {
            if (tiles == 0) return;
            const uint32_t n = (uint32_t)(tiles + op - 1) / (uint32_t)op, parts = n < on ? n : (uint32_t)on;
            own_wgs += times * parts, own_rounds += times * parts * cost.rounds(tiles, parts);
        };
        if (uniform && on) {
            const int64_t hidden = a.causal && !a.prefix_lens ? (a.Sq - 1) / 2 / kTile : 0;   // of a tile of rows, on average
            add(own_all > hidden ? own_all - hidden : 1, (double)cost.units);
        } else if (on) {
            for (int64_t b = 0; b < a.B; b++) add(((a.lens ? a.lens[b] : a.seqs[b].len) + kTile - 1) / kTile, (double)p.own_row_tiles);
        }
        own_wgs *= a.Hkv, own_rounds *= a.Hkv;
        for (int y = 0; y < (int)(sizeof(kParts) / sizeof(int)); y++) {
            if (y && kParts[y - 1] >= p_most) break;
            const int64_t pn = kParts[y] < p_most ? kParts[y] : p_most;
            if ((p_most && pn < p_least) || (pn + on > 1 && pn + on > parts_most)) continue;
            const double t = cost.us(pn, on, own_wgs, own_rounds);
            if (t < best) best = t, p.p_splits = (int)pn, p.own_splits = (int)on, p.own_tiles = (int)op;
        }
        if (own_wgs > 4 * cost.slots) break;   // (more of them would not run sooner)
    }
    if (best == 1e30) return 2;   // (no room to join prefix and own keys in)
    p.splits = p.p_splits + p.own_splits;
    const bool once = p.own_row_tiles <= 1 && cost.bytes_us > 20.0;   // (100 MB)
    p.by_g = fast_div(G), p.by_sq = fast_div(a.Sq), p.by_p_row_tiles = fast_div(p.p_row_tiles);
    p.by_own_splits = fast_div(p.own_splits), p.by_own_row_tiles = fast_div(p.own_row_tiles), p.by_own_tiles = fast_div(p.own_tiles);
    p.part_o = (float *)((char *)a.workspace + kWsCounterBytes + kWsPlanBytes);
    p.part_ml = p.part_o + (int64_t)p.splits * p.part_rows * a.D;
    if (p.splits == 1) p.part_o = p.part_ml = nullptr;
    if (p.splits > 1 && !cost.merged) p.counters = (int *)a.workspace;
    if (a.dtype == TROCM_F16) return a.D == 64 ? launch_tiles_of<_Float16, 64>(a, call, pre, own, is_scored, once, s) : launch_tiles_of<_Float16, 128>(a, call, pre, own, is_scored, once, s);
    return a.D == 64 ? launch_tiles_of<float, 64>(a, call, pre, own, is_scored, once, s) : launch_tiles_of<float, 128>(a, call, pre, own, is_scored, once, s);
}

}  // namespace

int launch_sdpa_rows(const SdpaRowsArgs &a, hipStream_t s) {
    if (a.B == 0 || a.Hq == 0 || a.Sq == 0 || a.D == 0) return 0;
    const int rc = launch_sdpa_rows_tiles(a, s);
    if (rc != 2) return rc;
    RowsCall call;
    RowsDev &p = call.p;
    fill_rows(a, p);
    TROCM_REQUIRE(a.D <= kAnyMaxD, "attention: head_dim %lld is above %d", (long long)a.D, kAnyMaxD);
    TROCM_REQUIRE(a.Hq * a.Sq < (1ll << 24), "attention: too many query rows per sequence");   // (a launch has fewer than 2^32 threads)
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
