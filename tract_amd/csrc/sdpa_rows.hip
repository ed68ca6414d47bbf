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
    int P, p_items, p_splits, p_row_tiles, p_tiles;   // p_items: of this launch; p_tiles, own_tiles: key tiles of a range
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

// tanh for f32 rows and for large caps: the library's, accurate to an ulp or two near zero.  For f16 rows under a cap of up to
// kFastTanhCap 1 - 2 / (e^2x + 1).
__device__ __forceinline__ float fast_tanh(float x) {
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

// Places of the key tiles [t_begin, t_end) that hold a token of a document in [dmin, dmax]; bit 15: all of the tile's tokens are of
// document `one`, that of every row but padding (-1: they differ).  All threads; returns how many.
__device__ __forceinline__ int list_document_tiles(const int *docs, int n_keys, int t_begin, int t_end, int dmin, int dmax, int one, uint16_t *list, int *counts) {
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    int n = 0;
    for (int t0 = t_begin; t0 < t_end; t0 += kThreads) {
        const int t = t0 + tid;
        int lo = INT_MAX, hi = -1, neg = 0;
        if (t < t_end) {
            const int first = t * kTile, last = min(first + kTile, n_keys);
            for (int j = first; j < last; j++) {
                const int id = docs[j];
                if (id >= 0) lo = min(lo, id), hi = max(hi, id);
                else neg = 1;
            }
        }
        const bool active = hi >= dmin && lo <= dmax;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(active);
        if (lane == 0) counts[w] = __popcll(mask);
        __syncthreads();
        int at = n;
        for (int x = 0; x < kWaves; x++) {
            if (x < w) at += counts[x];
            n += counts[x];
        }
        if (active) list[at + __popcll(mask & ((1ull << lane) - 1))] = (uint16_t)((t - t_begin) | (lo == hi && lo == one && !neg ? 0x8000 : 0));
        __syncthreads();
    }
    return n;
}

template <typename T, int D, int RB, bool SCORED>
__global__ __launch_bounds__(kThreads, RB == 1 && sizeof(T) == 2 ? 2 : 1) void sdpa_rows_kernel(RowsCall call) {
    const RowsDev &p = call.p;
    constexpr bool H16 = sizeof(T) == 2;
    constexpr int MR = 32 * RB, DB = D / 32;
    constexpr int KROW = H16 ? D + 8 : D + 4;     // elements per K row in LDS: 128-bit reads of 16 rows hit 64 distinct banks
    constexpr int VROW = H16 ? D + 16 : D + 8;    // f16: the 4 rows of a transposing read sit 8 banks apart; f32: rows 4 apart 32 banks apart
    constexpr int PRIV = kTile * (KROW + VROW) * (int)sizeof(T);   // a wave's tile
    constexpr int CROW = D + 4;                   // floats per row where waves are joined
    constexpr int LPRW = D * (int)sizeof(T) / 16, RPI = 64 / LPRW, NI = kTile / RPI;   // lanes per key row, rows per load, loads per tile and tensor
    constexpr int KS = H16 ? D / 16 : D / 8;      // 16-byte pieces of a lane's share of a row
    static_assert(kWaves * 32 * CROW * 4 + kWaves * 64 * 4 <= kWaves * PRIV, "waves are joined where the tiles were");
    __shared__ __attribute__((aligned(16))) unsigned char lds[kWaves * PRIV];
    __shared__ uint16_t s_list[SCORED ? kListMax : 1];
    __shared__ int s_counts[kWaves];

    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, hb = lane >> 5, l32 = lane & 31;
    int item = blockIdx.x;
    const int kvh = item % p.Hkv;   // (consecutive workgroups go to the 8 XCDs in turn: a kv head's keys meet in few L2 caches)
    item /= p.Hkv;
    const bool pre = item < p.p_items;
    int row0, row_end, split, n_keys, n_vis, t_begin, b = 0;
    const char *kb, *vb;
    int64_t st;
    if (pre) {
        row0 = item % p.p_row_tiles * MR, row_end = min(row0 + MR, p.B * p.Sq * p.G);
        split = item / p.p_row_tiles;
        kb = p.pk + (int64_t)kvh * p.p_stride_h, vb = p.pv + (int64_t)kvh * p.p_stride_h, st = p.p_stride_t;
        n_keys = n_vis = p.P;
        t_begin = split * p.p_tiles;
    } else {
        item -= p.p_items;
        split = item % p.own_splits, item /= p.own_splits;
        const int rt = p.own_row_tiles - 1 - item % p.own_row_tiles;   // (the longest first)
        b = p.seq0 + item / p.own_row_tiles;
        const OwnKeys own = own_keys(p, b, kvh);
        kb = own.k, vb = own.v, st = p.stride_t, n_keys = own.len;
        row0 = b * p.Sq * p.G + rt * MR, row_end = min(row0 + MR, (b + 1) * p.Sq * p.G);
        n_vis = n_keys;
        if (p.causal) {
            n_vis = (row_end - 1) / p.G - b * p.Sq + n_keys - p.Sq + 1;
            if (SCORED && p.prefix_lens) n_vis = max(n_vis, p.prefix_lens[b]);
            n_vis = max(0, min(n_vis, n_keys));
        }
        t_begin = split * p.own_tiles;
        split += p.p_splits;
    }
    const int t_end = min((n_vis + kTile - 1) / kTile, t_begin + (pre ? p.p_tiles : p.own_tiles));
    const int n_rb = (row_end - row0 + 31) / 32;

    // this lane's rows: one of each block of 32
    int lim[RB], at[RB], doc[RB];
    float slope[RB];
    int64_t out_row[RB];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        const int r = min(row0 + 32 * rb + l32, row_end - 1), bi = r / p.G, g = r - bi * p.G, rb_b = bi / p.Sq, i = bi - rb_b * p.Sq;
        out_row[rb] = ((int64_t)rb_b * p.Hq + kvh * p.G + g) * p.Sq + i;
        at[rb] = i + n_keys - p.Sq;
        lim[rb] = n_keys - 1;
        if (!pre && p.causal) lim[rb] = min(lim[rb], SCORED && p.prefix_lens ? max(at[rb], p.prefix_lens[b] - 1) : at[rb]);
        if constexpr (SCORED) {
            slope[rb] = p.slopes ? p.slopes[kvh * p.G + g] * kLog2e : 0.0f;
            doc[rb] = p.docs ? p.docs[(int64_t)b * p.Sk + at[rb]] : 0;
            if (doc[rb] < 0) lim[rb] = -1;   // padding sees nothing
        }
    }
    const int *docs = SCORED && p.docs ? p.docs + (int64_t)b * p.Sk : nullptr;
    int n_tiles = max(0, t_end - t_begin);
    bool listed = false;
    if constexpr (SCORED) {
        if (docs && n_tiles > 0 && n_tiles <= kListMax) {
            int dmin = INT_MAX, dmax = -1;
#pragma unroll
            for (int rb = 0; rb < RB; rb++)
                if (doc[rb] >= 0) dmin = min(dmin, doc[rb]), dmax = max(dmax, doc[rb]);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) dmin = min(dmin, __shfl_xor(dmin, d, 64)), dmax = max(dmax, __shfl_xor(dmax, d, 64));
            n_tiles = list_document_tiles(docs, n_keys, t_begin, t_end, dmin, dmax, dmin == dmax ? dmin : -1, s_list, s_counts);
            listed = true;
        }
    }
    auto part_m = [&](int64_t row) { return p.part_ml + (int64_t)split * 2 * p.part_rows + row; };
    if (n_tiles == 0 && p.splits > 1) {   // nothing to add: a maximum of -inf says so
        if (w == 0 && hb == 0)
#pragma unroll
            for (int rb = 0; rb < RB; rb++)
                if (row0 + 32 * rb + l32 < row_end) *part_m(out_row[rb]) = -INFINITY;
        return;
    }

    u32x4 qf[RB][KS];
#pragma unroll
    for (int rb = 0; rb < RB; rb++)
#pragma unroll
        for (int ks = 0; ks < KS; ks++) qf[rb][ks] = *reinterpret_cast<const u32x4 *>(p.q + out_row[rb] * (D * (int)sizeof(T)) + ks * 32 + hb * 16);

    float m_run[RB], l_run[RB];
    float16_t o[RB][DB];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        m_run[rb] = -INFINITY, l_run[rb] = 0.0f;
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[rb][db][r] = 0.0f;
    }

    T *lds_k = reinterpret_cast<T *>(lds + w * PRIV), *lds_v = lds_k + kTile * KROW;
    const int kr = lane / LPRW, ch = lane % LPRW;
    u32x4 kpre[NI], vpre[NI];
    int id_pre = 0;   // lane%32's token's document
    auto tile_at = [&](int n) -> int {
        if (SCORED && listed) return t_begin + __builtin_amdgcn_readfirstlane(s_list[n] & 0x7fff);
        return t_begin + n;
    };
    auto prefetch = [&](int n) {
        const int k_lo = tile_at(n) * kTile, most = n_keys - 1 - k_lo;   // (rows past the last key repeat it)
        const char *tk = kb + (int64_t)k_lo * st, *tv = vb + (int64_t)k_lo * st;
#pragma unroll
        for (int j = 0; j < NI; j++) {
            const uint32_t off = (uint32_t)min(j * RPI + kr, most) * (uint32_t)st + ch * 16;
            kpre[j] = *reinterpret_cast<const u32x4 *>(tk + off);
            vpre[j] = *reinterpret_cast<const u32x4 *>(tv + off);
        }
        if (SCORED && docs) id_pre = docs[k_lo + min(l32, most)];
    };
    const float to_log2 = p.scale * kLog2e, cap_log2 = p.cap * kLog2e, to_cap = p.cap > 0.0f ? p.scale / p.cap : 0.0f;

    if (w < n_tiles) prefetch(w);
    for (int n = w; n < n_tiles; n += kWaves) {
        const int k_lo = tile_at(n) * kTile;
        const bool by_id = SCORED && docs && !(listed && __builtin_amdgcn_readfirstlane(s_list[n] & 0x8000));
        const int id_tile = id_pre;
        const uint32_t padding = SCORED && by_id ? (uint32_t)__builtin_amdgcn_ballot_w64(id_tile < 0) : 0;   // a bit per key of the tile
#pragma unroll
        for (int j = 0; j < NI; j++) {
            *reinterpret_cast<u32x4 *>(lds_k + (j * RPI + kr) * KROW + ch * (16 / (int)sizeof(T))) = kpre[j];
            if (by_id && ((padding >> (j * RPI)) >> kr & 1)) vpre[j] = u32x4{0, 0, 0, 0};   // padding may hold anything
            *reinterpret_cast<u32x4 *>(lds_v + (j * RPI + kr) * VROW + ch * (16 / (int)sizeof(T))) = vpre[j];
        }
        if (n + kWaves < n_tiles) prefetch(n + kWaves);
        wave_sync();

        // ---- S^T = K Q^T: 32 keys x 32 rows each --------------------------------------------------------
        float16_t s[RB];
#pragma unroll
        for (int rb = 0; rb < RB; rb++)
#pragma unroll
            for (int r = 0; r < 16; r++) s[rb][r] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const u32x4 kf = *reinterpret_cast<const u32x4 *>(lds_k + l32 * KROW + (ks * 32 + hb * 16) / (int)sizeof(T));
#pragma unroll
            for (int rb = 0; rb < RB; rb++) {
                if constexpr (H16) {
                    s[rb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, kf), __builtin_bit_cast(half8_t, qf[rb][ks]), s[rb], 0, 0, 0);
                } else {   // (one feature of each half's four at a time)
                    const float4_t a = __builtin_bit_cast(float4_t, kf), c = __builtin_bit_cast(float4_t, qf[rb][ks]);
#pragma unroll
                    for (int e = 0; e < 4; e++) s[rb] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], c[e], s[rb], 0, 0, 0);
                }
            }
        }

        // ---- softmax of row lane%32 over this lane's 16 keys k_lo + 8 (r / 4) + 4 hb + r % 4 -------------
        half8_t pf[RB][2];
        if constexpr (SCORED) __builtin_amdgcn_sched_barrier(0);   // (V's fragments asked for during the scores' arithmetic spill registers)
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            if (rb > 0 && rb >= n_rb) break;
            if constexpr (SCORED) {
                if (H16 && p.cap > 0.0f && p.cap <= kFastTanhCap) {
#pragma unroll
                    for (int r = 0; r < 16; r++) s[rb][r] = cap_log2 * fast_tanh(s[rb][r] * to_cap);
                } else if (p.cap > 0.0f) {
#pragma unroll
                    for (int r = 0; r < 16; r++) s[rb][r] = cap_log2 * tanhf(s[rb][r] * to_cap);
                } else {
#pragma unroll
                    for (int r = 0; r < 16; r++) s[rb][r] *= to_log2;
                }
                if (p.slopes) {
                    const float d0 = (float)(at[rb] - k_lo - 4 * hb);
#pragma unroll
                    for (int r = 0; r < 16; r++) s[rb][r] = __builtin_fmaf(-slope[rb], fabsf(d0 - (float)(8 * (r >> 2) + (r & 3))), s[rb][r]);
                }
                if (by_id) {
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int c = 8 * (r >> 2) + (r & 3), even = __builtin_amdgcn_readlane(id_tile, c), odd = __builtin_amdgcn_readlane(id_tile, c + 4), id = hb ? odd : even;
                        s[rb][r] = id == doc[rb] ? s[rb][r] : -INFINITY;
                    }
                }
            } else {
#pragma unroll
                for (int r = 0; r < 16; r++) s[rb][r] *= to_log2;
            }
            const int last = lim[rb] - k_lo - 4 * hb;
            if (__builtin_amdgcn_ballot_w64(last < 28) != 0) {
#pragma unroll
                for (int r = 0; r < 16; r++) s[rb][r] = 8 * (r >> 2) + (r & 3) <= last ? s[rb][r] : -INFINITY;
            }
            float top = s[rb][0];
#pragma unroll
            for (int r = 1; r < 16; r++) top = fmaxf(top, s[rb][r]);
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            // f16: the reference moves only when the maximum exceeds it by more than 8 (weights reach 2^8 at most, far inside f16)
            const bool moved = top > m_run[rb] + (H16 ? 8.0f : 0.0f);
            const float m_new = moved ? top : m_run[rb], ref = m_new == -INFINITY ? 0.0f : m_new;
            const float keep = moved ? __builtin_amdgcn_exp2f(m_run[rb] - ref) : 1.0f;
            m_run[rb] = m_new;
            float sum = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                float e = __builtin_amdgcn_exp2f(s[rb][r] - ref);
                if constexpr (H16) {   // the product with V takes f16 weights, and the row's sum the same ones
                    pf[rb][r >> 3][r & 7] = (_Float16)e;
                    e = (float)pf[rb][r >> 3][r & 7];
                }
                s[rb][r] = e;
                sum += e;
            }
            l_run[rb] = l_run[rb] * keep + sum;
            if (__builtin_amdgcn_ballot_w64(moved) != 0) {
#pragma unroll
                for (int db = 0; db < DB; db++)
#pragma unroll
                    for (int r = 0; r < 16; r++) o[rb][db][r] *= keep;
            }
        }

        if constexpr (SCORED) __builtin_amdgcn_sched_barrier(0);
        // ---- O^T += V^T P^T --------------------------------------------------------------------------------
        if constexpr (H16) {
            // this lane as a source of the transposing loads: key (lane%16)/4 of a group of four, features 16 (lane/16 % 2) + 4 (lane%4)
            const _Float16 *vsrc = reinterpret_cast<const _Float16 *>(lds_v) + (4 * hb + ((lane & 15) >> 2)) * VROW + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
            for (int st2 = 0; st2 < 2; st2++)
#pragma unroll
                for (int db = 0; db < DB; db++) {
                    const half4_t lo = lds_read_tr16(vsrc + (16 * st2) * VROW + 32 * db);       // keys 16 st2 + 4 hb + 0..3
                    const half4_t hi = lds_read_tr16(vsrc + (16 * st2 + 8) * VROW + 32 * db);   // ... + 8
                    const half8_t vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                    for (int rb = 0; rb < RB; rb++)
                        if (rb == 0 || rb < n_rb) o[rb][db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[rb][st2], o[rb][db], 0, 0, 0);
                }
        } else {
#pragma unroll
            for (int r = 0; r < 16; r++)
#pragma unroll
                for (int db = 0; db < DB; db++) {
                    const float a = lds_v[(8 * (r >> 2) + 4 * hb + (r & 3)) * VROW + 32 * db + l32];
#pragma unroll
                    for (int rb = 0; rb < RB; rb++)
                        if (rb == 0 || rb < n_rb) o[rb][db] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, s[rb][r], o[rb][db], 0, 0, 0);
                }
        }
        wave_sync();   // (the next tile goes where this one was)
    }

    // ---- the four waves' results joined, a block of 32 rows at a time ------------------------------------------
    float *comb = reinterpret_cast<float *>(lds), *comb_ml = comb + kWaves * 32 * CROW;
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
        if (rb >= n_rb) break;
        l_run[rb] += __shfl_xor(l_run[rb], 32, 64);
        __syncthreads();   // tiles, or the block before, are done with
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int x = 0; x < 4; x++)
                *reinterpret_cast<float4_t *>(comb + (w * 32 + l32) * CROW + 32 * db + 8 * x + 4 * hb) =
                    float4_t{o[rb][db][4 * x], o[rb][db][4 * x + 1], o[rb][db][4 * x + 2], o[rb][db][4 * x + 3]};
        comb_ml[w * 64 + lane] = hb ? l_run[rb] : m_run[rb];
        __syncthreads();
        constexpr int TPR = kThreads / 32, PER = D / TPR;   // threads per row, features per thread
        const int row = tid / TPR, r = row0 + 32 * rb + row;
        if (r < row_end) {
            float mm = -INFINITY, l = 0.0f, f[kWaves];
#pragma unroll
            for (int x = 0; x < kWaves; x++) mm = fmaxf(mm, comb_ml[x * 64 + row]);
            const float ref = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
            for (int x = 0; x < kWaves; x++) {
                f[x] = __builtin_amdgcn_exp2f(comb_ml[x * 64 + row] - ref);
                l += f[x] * comb_ml[x * 64 + 32 + row];
            }
            const int bi = r / p.G, g = r - bi * p.G, rb_b = bi / p.Sq, i = bi - rb_b * p.Sq;
            const int64_t orow = ((int64_t)rb_b * p.Hq + kvh * p.G + g) * p.Sq + i;
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
            for (int e = 0; e < PER; e += 4) {
                const int d = (tid % TPR) * 4 + e * TPR;   // (16 bytes per thread, threads of a row side by side)
                float4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < kWaves; x++) {
                    const float4_t v = *reinterpret_cast<const float4_t *>(comb + (x * 32 + row) * CROW + d);
#pragma unroll
                    for (int y = 0; y < 4; y++) acc[y] = __builtin_fmaf(f[x], v[y], acc[y]);
                }
                if (p.splits == 1) {
                    T *out = reinterpret_cast<T *>(p.out) + orow * D + d;
                    struct alignas(4 * sizeof(T)) Four { T e[4]; } four;
#pragma unroll
                    for (int y = 0; y < 4; y++) four.e[y] = (T)(acc[y] * inv);
                    *reinterpret_cast<Four *>(out) = four;
                } else {
                    *reinterpret_cast<float4_t *>(p.part_o + ((int64_t)split * p.part_rows + orow) * D + d) = acc;
                }
            }
            if (p.splits > 1 && tid % TPR == 0) {
                *part_m(orow) = mm;
                *(part_m(orow) + p.part_rows) = l;
            }
        }
    }
}

// The ranges' partial rows -> output rows: D / 4 lanes per row.
template <typename T, int D>
__global__ __launch_bounds__(256) void sdpa_rows_merge_kernel(const float *__restrict__ part_o, const float *__restrict__ part_ml, T *__restrict__ out, int64_t rows, int splits) {
    constexpr int LPR = D / 4;
    const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
    const int d = threadIdx.x % LPR * 4;
    if (row >= rows) return;
    float mm = -INFINITY;
    for (int s = 0; s < splits; s++) mm = fmaxf(mm, part_ml[(int64_t)s * 2 * rows + row]);
    float l = 0.0f;
    float4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < splits; s++) {
        const float m = part_ml[(int64_t)s * 2 * rows + row];
        if (m == -INFINITY) continue;   // (a range without keys for the row has stored nothing else)
        const float f = __builtin_amdgcn_exp2f(m - mm);
        const float4_t v = *reinterpret_cast<const float4_t *>(part_o + ((int64_t)s * rows + row) * D + d);
        l += f * part_ml[((int64_t)s * 2 + 1) * rows + row];
#pragma unroll
        for (int y = 0; y < 4; y++) acc[y] = __builtin_fmaf(f, v[y], acc[y]);
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    struct alignas(4 * sizeof(T)) Four { T e[4]; } four;
#pragma unroll
    for (int y = 0; y < 4; y++) four.e[y] = (T)(acc[y] * inv);
    *reinterpret_cast<Four *>(out + row * D + d) = four;
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

namespace {

template <typename T, int D, int RB, bool SCORED>
int launch_tiles(const SdpaRowsArgs &a, RowsCall &call, hipStream_t s) {
    RowsDev &p = call.p;
    const int64_t holds = table_holds(a);
    for (int64_t b = 0; b < a.B; b += holds) {   // the prefix, for all rows, with the first sequences' own keys
        const int64_t n = a.B - b < holds ? a.B - b : holds;
        fill_table(a, b, n, call.tab);
        p.seq0 = (int)b;
        p.p_items = b == 0 ? p.p_splits * p.p_row_tiles : 0;
        const int64_t grid = a.Hkv * (p.p_items + n * p.own_row_tiles * p.own_splits);
        if (grid == 0) continue;
        TROCM_REQUIRE(grid < (1ll << 31), "attention: too many workgroups");
        hipLaunchKernelGGL((sdpa_rows_kernel<T, D, RB, SCORED>), dim3((unsigned)grid), dim3(kThreads), 0, s, call);
        if (check_launch("sdpa_rows")) return 1;
    }
    if (p.splits > 1) {
        constexpr int ROWS = 256 / (D / 4);
        hipLaunchKernelGGL((sdpa_rows_merge_kernel<T, D>), dim3((unsigned)((p.part_rows + ROWS - 1) / ROWS)), dim3(256), 0, s, p.part_o, p.part_ml, (T *)p.out, p.part_rows, p.splits);
        if (check_launch("sdpa_rows_merge")) return 1;
    }
    return 0;
}

template <typename T, int D>
int launch_tiles_of(const SdpaRowsArgs &a, RowsCall &call, int rb, bool is_scored, hipStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (rb == 2) return launch_tiles<T, D, 2, false>(a, call, s);
    return is_scored ? launch_tiles<T, D, 1, true>(a, call, s) : launch_tiles<T, D, 1, false>(a, call, s);
}

// On the matrix cores: 0 done, 1 failed, 2 not covered.
int launch_sdpa_rows_tiles(const SdpaRowsArgs &a, hipStream_t s) {
    const int64_t es = (int64_t)elem_bytes(a.dtype);
    if (a.D != 64 && a.D != 128) return 2;
    const int64_t G = a.Hq / a.Hkv, rows = a.B * a.Sq * G;
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
    const int rb = es == 2 && !is_scored && (a.P ? rows : seq_rows) > 32 ? 2 : 1, MR = 32 * rb;
    RowsCall call;
    RowsDev &p = call.p;
    fill_rows(a, p);
    const int64_t p_all = (a.P + kTile - 1) / kTile, own_all = (longest + kTile - 1) / kTile;
    p.p_row_tiles = a.P ? (int)((rows + MR - 1) / MR) : 0;
    p.own_row_tiles = longest ? (int)((seq_rows + MR - 1) / MR) : 0;
    // Ranges: as much work for each workgroup as makes `target` of them in all, a multiple of a tile per wave.
    const int64_t target = (int64_t)num_compute_units() * (rb == 1 && es == 2 ? 2 : 1);
    const int64_t work = a.Hkv * (p.p_row_tiles * p_all + p.own_row_tiles * own_tiles_all);
    int64_t per = ((work + target - 1) / target + kWaves - 1) / kWaves * kWaves;
    const int64_t room = a.workspace && aligned(a.workspace) && a.workspace_bytes > kWsCounterBytes + kWsPlanBytes + 256
                             ? (int64_t)(a.workspace_bytes - kWsCounterBytes - kWsPlanBytes - 256) / ((a.D + 2) * (int64_t)sizeof(float)) / p.part_rows : 0;
    for (;; per *= 2) {
        p.p_tiles = p.own_tiles = (int)per;
        p.p_splits = (int)((p_all + per - 1) / per), p.own_splits = (int)((own_all + per - 1) / per);
        p.splits = p.p_splits + p.own_splits;
        if (p.splits == 1 || (p.splits <= room && p.splits <= 64)) break;
        if (p.p_splits <= 1 && p.own_splits <= 1) return 2;   // (no room to join prefix and own keys in)
    }
    p.part_o = (float *)((char *)a.workspace + kWsCounterBytes + kWsPlanBytes);
    p.part_ml = p.part_o + (int64_t)p.splits * p.part_rows * a.D;
    if (p.splits == 1) p.part_o = p.part_ml = nullptr;
    if (a.dtype == TROCM_F16) return a.D == 64 ? launch_tiles_of<_Float16, 64>(a, call, rb, is_scored, s) : launch_tiles_of<_Float16, 128>(a, call, rb, is_scored, s);
    return a.D == 64 ? launch_tiles_of<float, 64>(a, call, rb, is_scored, s) : launch_tiles_of<float, 128>(a, call, rb, is_scored, s);
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
