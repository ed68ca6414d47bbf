// Attention over pages of keys and values: o = softmax(scale q k^T) v for one or a few new tokens of every sequence, whose keys lie in
// pages anywhere, found through a table, and whose lengths are read from device memory.  f16 and f32.
//
// The query rows of a kv head (heads of the group, queries) are rows of matrix tiles, S^T = K Q^T and O^T = V^T P^T, so that every softmax
// scalar of a row sits in one lane.  A tile is 32 keys: two halves of 16 that lie in a page each (pages are multiples of 16 tokens).  One
// pass over the keys, with the running maximum m and sum l of every row: o <- o 2^(m - m') + 2^(s - m') v, f32.
//
// The host does not know the lengths, so the work is shared out on the device: all units (sequence, kv head, up to four tiles of 16 rows) one
// behind the other are a line of steps of 128 keys, a tile for each of a workgroup's waves, and every workgroup takes a stretch of the line,
// all of the same length.  A unit inside of a stretch goes straight to the output; one that a stretch's end cuts goes to the workspace in
// parts (unnormalised O, maximum, sum, f32), which the last workgroup to arrive joins, always in the same order.  Two workgroups a compute
// unit, whose rows of the next tile are on their way while one is worked on (1, 3, 4 and 8 were slower).  A line counted in tiles, whose
// stretches began anywhere, left waves of a step without a tile and put short sequences behind one another (64 sequences of up to 8192 keys
// 195 us for 190.5, one token behind 777 10.4 for 7.7, 9 sequences of up to 120 in f32 23.9 for 10.2).
//
// What bounds it: the pages' bytes where there are many (64 sequences of 64 to 8192 keys of 8 x 128, f16, 1.18 GB: 190.5 us, 6.2 TB/s; 3
// queries behind 90000 and 100001 keys 137 us, 5.8 TB/s; 16 sequences of up to 3000 keys of 32 x 64, f32, 82 us, 5.2 TB/s), matrix
// instructions busy for 4 to 34 % of the SIMDs' cycles; the chain lengths - table - keys - join where there are few (7.7 us).
#include <hip/hip_fp16.h>
#include <math.h>
#include <algorithm>
#include "common.h"
#include "fast_div.h"

namespace trocm {
namespace {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWaves = 4, kThreads = 64 * kWaves, kTile = 32, kRows = 16;
constexpr int kStep = kTile * kWaves;   // keys of a step: a tile for each wave

struct PagedDev {
    const char *q, *k, *v;
    char *out;
    const int *table, *lens;
    int64_t table_width, stride_page, stride_h, stride_t;   // strides: bytes
    int B, Hq, Hkv, Sq, G, D, n_pages, most;                // most: tokens that a row of the table has pages for
    float scale;
    int causal;
    FastDiv by_page;
    // tiles of 16 rows
    int *counters;
    float *parts;
    FastDiv by_g, by_workgroups;
    float part_cost;            // kPartCost, of the rows, for the average of the sequences
    FastDiv row_units[3];       // by the units of a kv head's rows, where they take one, two and four tiles
};

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(_Float16 x) { return (float)x; }

// ---- any head size, page size and alignment: a workgroup per query row ----------------------------------------------------

constexpr int64_t kMostBlocks = 1 << 22;   // (a launch counts threads in 32 bits)
constexpr int kAnyThreads = 256, kAnyWaves = kAnyThreads / 64;

template <typename T>
__global__ __launch_bounds__(kAnyThreads) void sdpa_paged_any_kernel(PagedDev p) {
    __shared__ float lds_q[kRowsMaxD], lds_o[kRowsMaxD], lds_p[kAnyThreads], lds_red[2 * kAnyWaves];
    __shared__ int64_t lds_at[kAnyThreads];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, D = p.D;
    const int64_t per = (int64_t)p.Hq * p.Sq;   // rows of a sequence, queries in turn
    for (int64_t x = blockIdx.x; x < per * p.B; x += gridDim.x) {
        const int b = (int)(x / per), rest = (int)(x - b * per), qh = rest % p.Hq, i = rest / p.Hq, kvh = qh / p.G;
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
                    float dot[4] = {0.0f, 0.0f, 0.0f, 0.0f};   // (sums of a quarter of the terms: nearer, and not one behind the other)
                    int d = 0;
#pragma unroll 1
                    for (; d + 4 <= D; d += 4)
#pragma unroll
                        for (int e = 0; e < 4; e++) dot[e] = __builtin_fmaf(lds_q[d + e], widen(k[d + e]), dot[e]);
                    for (; d < D; d++) dot[0] = __builtin_fmaf(lds_q[d], widen(k[d]), dot[0]);
                    s = ((dot[0] + dot[1]) + (dot[2] + dot[3])) * (p.scale * kLog2e);
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

// ---- head sizes 64 and 128, pages of multiples of 16 tokens: matrix tiles ---------------------------------------------------

// 16 bytes of device memory; ONCE: past the caches.
template <bool ONCE>
__device__ __forceinline__ u32x4 load16(const char *base, uint32_t off) {
    const auto *at = (const __attribute__((address_space(1))) u32x4 *)(base + off);
    return ONCE ? __builtin_nontemporal_load(at) : *at;
}

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

// Partial results for whichever workgroup joins them: written through to where every compute unit sees them once they complete.
__device__ __forceinline__ void put(float *at, float x) { __hip_atomic_store(at, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float get(const float *at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void put2(float *at, float2_t x) { __hip_atomic_store(reinterpret_cast<uint64_t *>(at), __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float2_t get2(const float *at) { return __builtin_bit_cast(float2_t, __hip_atomic_load(reinterpret_cast<const uint64_t *>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)); }

// a - b of scores as they are rounded: a product fused into it would differ from `b`, which is one of them, by up to half its last place.
__device__ __forceinline__ float less(float a, float b) {
#pragma clang fp contract(off)
    return a - b;
}

// A kernel's one argument where it lies, as loads from here on: kept from the beginning, what only some places look at would leave the loop too
// few scalar registers.
typedef const __attribute__((address_space(4))) PagedDev &Arguments;
__device__ __forceinline__ Arguments arguments_again() {
    auto at = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
    asm volatile("" : "+s"(at));
    return *reinterpret_cast<const __attribute__((address_space(4))) PagedDev *>(at);
}
__device__ __forceinline__ int divided(const __attribute__((address_space(4))) FastDiv &by, int n) { return FastDiv{by.d, by.mul, by.shift}.by(n); }

// Where row r of a kv head lies among the q and output rows, and which query it is.
struct RowPlace { int64_t at; int i; };
__device__ __forceinline__ RowPlace q_row(Arguments p, int b, int kvh, int r) {
    const int i = divided(p.by_g, r);
    return {((int64_t)b * p.Hq + kvh * p.G + r - i * p.G) * p.Sq + i, i};
}

constexpr int kLinePart(int D) { return kRows * D + 2 * kRows; }   // floats of a part: rows of O, their maxima, their sums

constexpr int in_lds(int es, int D) { return es == 4 && D == 128 ? kRows * D * es : 0; }   // bytes of queries
constexpr int line_lds(int es, int D) { return kWaves * kTile * (es == 2 ? 2 * D + 24 : D + 4) * es + in_lds(es, D); }

// Steps [first, end) of a unit; `part`: where its partial rows go, a row tile's behind the other's (NULL: it is the whole unit, rows go to the
// output).
struct Stretch {
    int b, kvh, row0, rows, len, first, end;
    float *part;
};

// A wave-uniform value out of LDS.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The sum of the values of features d and d + 1 that are not finite, over the keys of a stretch that row r sees and not all rows do.
template <typename T, int D>
__device__ __forceinline__ float2_t not_finite(const Stretch &u, int r, int d) {
    Arguments p = arguments_again();
    const int seen = u.len - p.Sq + q_row(p, u.b, u.kvh, r).i, end = min(min(u.end * kStep, u.len) - 1, seen);
    float2_t sum = {0.0f, 0.0f};
    for (int key = max(u.len - p.Sq + 1, u.first * kStep); key <= end; key++) {
        const int pi = divided(p.by_page, key), id = p.table[u.b * p.table_width + pi];
        if ((unsigned)id >= (unsigned)p.n_pages) continue;
        const T *v = reinterpret_cast<const T *>(p.v + id * p.stride_page + u.kvh * p.stride_h + (key - pi * (int)p.by_page.d) * p.stride_t) + d;
#pragma unroll
        for (int y = 0; y < 2; y++) sum[y] += fabsf(widen(v[y])) < INFINITY ? 0.0f : widen(v[y]);
    }
    return sum;
}

// SOLO: a unit of this wave alone, in tiles one after the other.
template <typename T, int D, int RT, bool ONCE, bool SOLO>
__device__ __forceinline__ void stretch_body(const Stretch &u, int &s_poison, unsigned char *lds) {
    constexpr bool H16 = sizeof(T) == 2;
    constexpr int DB = D / 16;                    // feature blocks of the output
    constexpr int KROW = D + 8, VROW = H16 ? D + 16 : D + 4;   // elements per row in LDS: rows of a read in different banks
    constexpr int PRIV = kTile * (VROW + (H16 ? KROW : 0)) * (int)sizeof(T);   // a wave's tile
    constexpr int CROW = D + 4;                   // floats per row where waves are joined
    constexpr int LPRW = D * (int)sizeof(T) / 16, RPI = 64 / LPRW, NI = kTile / RPI;   // lanes per key row, rows per load, loads per tile and tensor
    constexpr int KS = D * (int)sizeof(T) / 64;   // 16-byte pieces of a lane's share of a row
    constexpr int NK = H16 ? NI : 2 * KS;
    constexpr float kMost = H16 ? 15.0f : 0.0f;   // weights are 2^kMost at most
    static_assert(kWaves * kRows * CROW * 4 + kWaves * 2 * kRows * 4 <= kWaves * PRIV, "waves are joined where the tiles were");

    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, grp = lane / 16, lr = lane % 16;
    Arguments p = arguments_again();
    int64_t q_at[RT];
    int lim[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
        const RowPlace place = q_row(p, u.b, u.kvh, u.row0 + min(16 * t + lr, u.rows - 1));
        q_at[t] = place.at, lim[t] = p.causal ? min(u.len - 1, u.len - p.Sq + place.i) : u.len - 1;
    }
    const int last_key = u.len - 1;
    // From here on keys that not all rows see.  A weight of zero does not take an infinity or a NaN out of a product: values from here on that are
    // not finite are zeros in the tiles, and are added where waves are joined, to the rows that see them.
    const int some_see = p.causal ? max(u.len - p.Sq + 1, 0) : u.len;
    const char *kb = p.k + u.kvh * p.stride_h, *vb = p.v + u.kvh * p.stride_h;
    const uint32_t st = (uint32_t)p.stride_t;     // (below 2^27: checked by the host)
    const float to_log2 = p.scale * kLog2e;
    auto tile_at = [&](int i) { return SOLO ? i : (u.first + i) * kWaves + w; };   // this wave takes a tile of every step
    const int n_mine = SOLO ? last_key / kTile + 1 : min(u.end - u.first, (last_key / kTile - u.first * kWaves - w + kWaves) / kWaves);

    // Where the halves of 32 of this wave's tiles lie: lane 2 i + h has tile i's half h, as bytes from the pool's beginning (-1: a hole, or
    // behind the last key).
    auto ask_pages = [&](int i0) __attribute__((always_inline)) {
        Arguments p = arguments_again();
        const int key = tile_at(i0 + (lane >> 1)) * kTile + 16 * (lane & 1);
        return key <= last_key && i0 + (lane >> 1) < n_mine ? p.table[u.b * p.table_width + divided(p.by_page, key)] : -1;
    };
    auto bytes_at = [&](int id, int i0) __attribute__((always_inline)) {
        Arguments p = arguments_again();
        const int key = tile_at(i0 + (lane >> 1)) * kTile + 16 * (lane & 1);
        const int in_page = key - divided(p.by_page, key) * (int)p.by_page.d;
        return (unsigned)id < (unsigned)p.n_pages ? id * p.stride_page + (int64_t)in_page * p.stride_t : (int64_t)-1;
    };
    int64_t at = -1;
    int ids_next = -1;

    float m_run[RT], l_run[RT];
    float4_t o[RT][DB];
#pragma unroll
    for (int t = 0; t < RT; t++) {
        m_run[t] = -INFINITY, l_run[t] = 0.0f;
#pragma unroll
        for (int db = 0; db < DB; db++) o[t][db] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }

    T *lds_v = reinterpret_cast<T *>(lds + w * PRIV), *lds_k = lds_v + kTile * VROW;   // (lds_k: f16)
    const int kr = lane / LPRW, ch = lane % LPRW;
    u32x4 kpre[NK], vpre[NI];
    struct Halves { int64_t at[2]; };   // (of the tile whose rows are in flight)
    int there = 0, there_next = 0;      // bits: which halves are
    auto halves_of = [&](int i) __attribute__((always_inline)) {
        Halves r;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int from = 2 * (i & 31) + h;
            r.at[h] = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint64_t)at, from) | ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)((uint64_t)at >> 32), from) << 32));
        }
        return r;
    };
    // (halves that are not there read the other one's rows, or the pool's first: they weigh nothing; rows behind the last key repeat it)
    auto row_base = [&](const Halves &x, int h) __attribute__((always_inline)) { return x.at[h] >= 0 ? x.at[h] : x.at[1 - h] >= 0 ? x.at[1 - h] : 0; };
    auto rows_of = [&](int i, const Halves &x, int h) __attribute__((always_inline)) {   // the last row of a half that may be read
        const int most = last_key - tile_at(i) * kTile;
        if (x.at[0] < 0 && x.at[1] < 0) return 0;
        return min(most - 16 * (x.at[h] >= 0 ? h : 1 - h), 15);
    };
    auto prefetch_k = [&](int i, const Halves &x) __attribute__((always_inline)) {
        if constexpr (H16) {
#pragma unroll
            for (int j = 0; j < NI; j++) {
                const int h = j * RPI / 16;
                kpre[j] = load16<ONCE>(kb + row_base(x, h), (uint32_t)min(j * RPI % 16 + kr, rows_of(i, x, h)) * st + ch * 16);
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const char *base = kb + row_base(x, h);
                const uint32_t off = (uint32_t)min(lr, rows_of(i, x, h)) * st + grp * 16;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) kpre[h * KS + ks] = load16<false>(base, off + ks * 64);   // (64 bytes of a row at a time: the caches join them)
            }
        }
    };
    auto prefetch_v = [&](int i, const Halves &x) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NI; j++) {
            const int h = j * RPI / 16;
            vpre[j] = load16<ONCE>(vb + row_base(x, h), (uint32_t)min(j * RPI % 16 + kr, rows_of(i, x, h)) * st + ch * 16);
        }
    };
    // key of score x of this lane, from the tile's first: two groups of four consecutive ones
    auto key_of = [](int x) { return 16 * (x >> 2) + (x & 3); };   // + 4 grp

    if (n_mine > 0) {
        const int ids = ask_pages(0);
        ids_next = ask_pages(32);
        at = bytes_at(ids, 0);
        const Halves first = halves_of(0);
        there = (first.at[0] >= 0) + 2 * (first.at[1] >= 0);
        prefetch_k(0, first), prefetch_v(0, first);
    }
    // queries: in registers, or, where those are all taken, in LDS
    constexpr bool QL = in_lds(sizeof(T), D) > 0 && !SOLO, QT = in_lds(sizeof(T), D) > 0 && SOLO;   // QT: a few at a time, with every tile again
    static_assert(!QL || RT == 1, "one row tile's");
    u32x4 qf[RT][QL || QT ? 1 : KS], *lds_q = reinterpret_cast<u32x4 *>(lds + kWaves * PRIV);
    if constexpr (QL) {
        for (int ks = w; ks < KS; ks += kWaves) lds_q[ks * 64 + lane] = load16<false>(p.q + q_at[0] * (D * (int)sizeof(T)), ks * 64 + grp * 16);
        __syncthreads();
    } else if constexpr (!QT) {
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++) qf[t][ks] = load16<false>(p.q + q_at[t] * (D * (int)sizeof(T)), ks * 64 + grp * 16);
    }
    bool poisoned = false;   // SOLO
    for (int i = 0; i < n_mine; i++) {
        const int k_lo = tile_at(i) * kTile;
        const bool more = i + 1 < n_mine;
        Halves next = {-1, -1};
        if (more) {
            if (((i + 1) & 31) == 0) at = bytes_at(ids_next, i + 1), ids_next = ask_pages(i + 33);
            next = halves_of(i + 1);
            there_next = (next.at[0] >= 0) + 2 * (next.at[1] >= 0);
        }
        const bool odd = there != 3 || k_lo + kTile > u.len;   // a hole, or the last key inside

        // ---- S^T = K Q^T --------------------------------------------------------------------------------------
        float4_t acc[RT][2];
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
            for (int h = 0; h < 2; h++) acc[t][h] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (H16) {
#pragma unroll
            for (int j = 0; j < NI; j++) *reinterpret_cast<u32x4 *>(lds_k + (j * RPI + kr) * KROW + ch * 8) = kpre[j];
            if (more) prefetch_k(i + 1, next);
            wave_sync();
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const half8_t kf = __builtin_bit_cast(half8_t, *reinterpret_cast<const u32x4 *>(lds_k + (16 * h + lr) * KROW + ks * 32 + grp * 8));
#pragma unroll
                    for (int t = 0; t < RT; t++) acc[t][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, __builtin_bit_cast(half8_t, qf[t][ks]), acc[t][h], 0, 0, 0);
                }
        } else {
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    const float4_t c = __builtin_bit_cast(float4_t, QT ? load16<false>(p.q + q_at[t] * (D * (int)sizeof(T)), ks * 64 + grp * 16) : QL ? lds_q[ks * 64 + lane] : qf[t][QL ? 0 : ks]);
#pragma unroll
                    for (int h = 0; h < 2; h++) {   // (one feature of each group's four at a time)
                        const float4_t a = __builtin_bit_cast(float4_t, kpre[h * KS + ks]);
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[t][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], c[e], acc[t][h], 0, 0, 0);
                    }
                }
            if (more) prefetch_k(i + 1, next);
        }
        int kr = lane / LPRW;
        asm("" : "+v"(kr));   // (or what is made of it waits in registers, which four row tiles do not have)
        if (odd) {   // rows that are not the sequence's may hold anything
#pragma unroll
            for (int j = 0; j < NI; j++) {
                const int r = j * RPI + kr;
                if (!((there >> (j * RPI / 16)) & 1) || k_lo + r > last_key) vpre[j] = u32x4{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int j = 0; j < NI; j++) *reinterpret_cast<u32x4 *>(lds_v + (j * RPI + kr) * VROW + ch * (16 / (int)sizeof(T))) = vpre[j];
        if (more) prefetch_v(i + 1, next);
        // ---- softmax of this lane's rows over their keys k_lo + 4 grp + key_of(x) --------------------------------
        half8_t pf[RT];        // weights: f16
        float e[RT][8];        // ... and f32
#pragma unroll
        for (int t = 0; t < RT; t++) {
            float s[8];
#pragma unroll
            for (int x = 0; x < 8; x++) s[x] = acc[t][x >> 2][x & 3] * to_log2;
            const int last = lim[t] - k_lo - 4 * grp;
            if (odd || __builtin_amdgcn_ballot_w64(last < 28) != 0) {
#pragma unroll
                for (int x = 0; x < 8; x++) s[x] = key_of(x) <= last && ((there >> (x >> 2)) & 1) ? s[x] : -INFINITY;
            }
            float top = s[0];
#pragma unroll
            for (int x = 1; x < 8; x++) top = fmaxf(top, s[x]);
#pragma unroll
            for (int d = 16; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
            // f16: weights are f16 numbers of 2^15 at most, which keep all their bits down to 2^-14 and are gone below 2^-25, so the reference is 14
            // below the maximum where it moves, and moves when the maximum is more than 15 above: 2^-28 of the largest weight is whole, 2^-39 is
            // something.  (Beside one key with nearly all of the weight, and a value of next to nothing, those are the result.)  Maxima beyond
            // 2^25, from which 14 may round to 16, are references themselves.
            const bool moved = less(top, m_run[t]) > kMost;
            if (__builtin_amdgcn_ballot_w64(moved) != 0) {
                float m_new = H16 ? less(top, kMost - 1.0f) : top;
                if (H16) m_new = less(top, m_new) > kMost ? top : m_new;
                const float keep = moved ? __builtin_amdgcn_exp2f(m_run[t] - m_new) : 1.0f;
                m_run[t] = moved ? m_new : m_run[t];
                l_run[t] *= keep;
#pragma unroll
                for (int db = 0; db < DB; db++) o[t][db] *= keep;
            }
            const float ref = m_run[t] == -INFINITY ? 0.0f : m_run[t];
            float sum = 0.0f;
#pragma unroll
            for (int x = 0; x < 8; x++) {
                e[t][x] = __builtin_amdgcn_exp2f(less(s[x], ref));
                // The product with V takes f16 operands: weights are rounded, half a step each, and the row's sum takes the same ones, so that
                // a row of equal values stays that value.
                if constexpr (H16) {
                    pf[t][x] = (_Float16)e[t][x];
                    e[t][x] = (float)pf[t][x];
                }
                sum += e[t][x];
            }
            l_run[t] += sum;
        }

        if (k_lo + kTile > some_see && some_see <= last_key) {
            wave_sync();
            uint32_t found = 0;
            for (int r = max(some_see - k_lo, 0) + kr; r <= min(last_key - k_lo, kTile - 1); r += RPI) {
                u32x4 &piece = *reinterpret_cast<u32x4 *>(lds_v + r * VROW + ch * (16 / (int)sizeof(T))), x = piece;
#pragma unroll
                for (int y = 0; y < 4; y++) {   // a one for every exponent of all ones: in bits 0 and 16, or 0
                    const uint32_t ones = H16 ? ((x[y] & 0x7fff7fffu) + 0x04000400u) >> 15 & 0x00010001u : ((x[y] & 0x7fffffffu) + 0x00800000u) >> 31;
                    x[y] &= H16 ? ~(ones * 0xffffu) : ones - 1, found |= ones;
                }
                piece = x;
            }
            if constexpr (SOLO) poisoned |= __builtin_amdgcn_ballot_w64(found != 0) != 0;
            else if (found) s_poison = 1;
        }

        // ---- O^T += V^T P^T --------------------------------------------------------------------------------
        wave_sync();
        if constexpr (H16) {
            // this lane as a source of the transposing loads: key (lane%16)/4 of a group of four, features 4 (lane%4) of a block of 16
            const _Float16 *vsrc = reinterpret_cast<const _Float16 *>(lds_v) + (4 * grp + ((lane & 15) >> 2)) * VROW + 4 * (lane & 3);
#pragma unroll
            for (int db = 0; db < DB; db++) {
                const half4_t lo = lds_read_tr16(vsrc + 16 * db), hi = lds_read_tr16(vsrc + 16 * VROW + 16 * db);
#pragma unroll
                for (int t = 0; t < RT; t++) o[t][db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), pf[t], o[t][db], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int x = 0; x < 8; x++)
#pragma unroll
                for (int db = 0; db < DB; db++) {
                    const float v = lds_v[(key_of(x) + 4 * grp) * VROW + 16 * db + lr];
#pragma unroll
                    for (int t = 0; t < RT; t++) o[t][db] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, e[t][x], o[t][db], 0, 0, 0);
                }
        }
        wave_sync();   // (the next tile goes where this one was)
        there = there_next;
    }

    if constexpr (SOLO) {
        static_assert(RT == 1, "one row tile");
        float l = l_run[0];
#pragma unroll
        for (int d = 16; d < 64; d <<= 1) l += __shfl_xor(l, d, 64);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (lr < u.rows) {
            Arguments p = arguments_again();
            T *out = reinterpret_cast<T *>(p.out) + q_row(p, u.b, u.kvh, u.row0 + lr).at * D + 4 * grp;
#pragma unroll
            for (int db = 0; db < DB; db++) {
                struct alignas(4 * sizeof(T)) Four { T e[4]; } four;
#pragma unroll
                for (int y = 0; y < 4; y++) four.e[y] = (T)(o[0][db][y] * inv);
                *reinterpret_cast<Four *>(out + 16 * db) = four;
            }
            if (poisoned)
#pragma unroll 1
                for (int x = 0; x < 2 * DB; x++) {
                    T *at = out + 16 * (x >> 1) + 2 * (x & 1);
                    const float2_t add = not_finite<T, D>(u, u.row0 + lr, 16 * (x >> 1) + 4 * grp + 2 * (x & 1));
#pragma unroll
                    for (int y = 0; y < 2; y++) at[y] = (T)(widen(at[y]) + add[y]);
                }
        }
        return;
    }
    // ---- the four waves' results joined ------------------------------------------------------------------------
    float *comb = reinterpret_cast<float *>(lds), *comb_ml = comb + kWaves * kRows * CROW;
    constexpr int TPR = kThreads / kRows, PER = D / TPR;   // threads per row, features per thread
    const int row = tid / TPR;
    int poison = 0;
#pragma unroll
    for (int t = 0; t < RT; t++) {
#pragma unroll
        for (int d = 16; d < 64; d <<= 1) l_run[t] += __shfl_xor(l_run[t], d, 64);
        __syncthreads();   // the tiles, or the last rows, are done with
        if (t == 0) poison = s_poison;
#pragma unroll
        for (int db = 0; db < DB; db++) *reinterpret_cast<float4_t *>(comb + (w * kRows + lr) * CROW + 16 * db + 4 * grp) = o[t][db];
        if (grp < 2) comb_ml[(w * 2 + grp) * kRows + lr] = grp ? l_run[t] : m_run[t];
        __syncthreads();
        if (t == 0 && tid == 0) s_poison = 0;   // (everybody has seen it)
        if (16 * t + row < u.rows) {
            float mm = -INFINITY, l = 0.0f, f[kWaves];
#pragma unroll
            for (int x = 0; x < kWaves; x++) mm = fmaxf(mm, comb_ml[x * 2 * kRows + row]);
            const float ref = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
            for (int x = 0; x < kWaves; x++) {
                f[x] = __builtin_amdgcn_exp2f(comb_ml[x * 2 * kRows + row] - ref);
                l += f[x] * comb_ml[(x * 2 + 1) * kRows + row];
            }
            Arguments p = arguments_again();
            float *part = u.part + t * kLinePart(D);
            const int64_t orow = q_row(p, u.b, u.kvh, u.row0 + 16 * t + row).at;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int e = 0; e < PER; e += 2) {
                const int d = (tid % TPR) * 2 + e * TPR;   // (8 bytes per thread, threads of a row side by side: a store covers whole lines)
                float2_t sum = {0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < kWaves; x++) {
                    const float2_t v = *reinterpret_cast<const float2_t *>(comb + (x * kRows + row) * CROW + d);
#pragma unroll
                    for (int y = 0; y < 2; y++) sum[y] = __builtin_fmaf(f[x], v[y], sum[y]);
                }
                if (!u.part) {
                    struct alignas(2 * sizeof(T)) Two { T e[2]; } two;
                    two.e[0] = (T)(sum[0] * inv), two.e[1] = (T)(sum[1] * inv);
                    *reinterpret_cast<Two *>(reinterpret_cast<T *>(p.out) + orow * D + d) = two;
                } else {
                    put2(part + row * D + d, sum);
                }
            }
            if (u.part && tid % TPR == 0) put(part + kRows * D + row, mm), put(part + kRows * D + kRows + row, l);
        }
    }
    if (uniform(poison)) {   // (every thread to what it has written)
        int tid = threadIdx.x;
        asm("" : "+v"(tid));   // (or what is made of it waits in registers all the time)
        const int row = tid / TPR;
#pragma unroll 1
        for (int x = 0; x < RT * PER / 2; x++) {
            const int r = 16 * (x / (PER / 2)) + row, d = (tid % TPR) * 2 + x % (PER / 2) * 2 * TPR;
            if (r >= u.rows) continue;
            const float2_t add = not_finite<T, D>(u, u.row0 + r, d);
            if (u.part) {
                float *at = u.part + r / 16 * kLinePart(D) + (r & 15) * D + d;
                put2(at, get2(at) + add);
            } else {
                Arguments p = arguments_again();
                T *at = reinterpret_cast<T *>(p.out) + q_row(p, u.b, u.kvh, u.row0 + r).at * D + d;
#pragma unroll
                for (int y = 0; y < 2; y++) at[y] = (T)(widen(at[y]) + add[y]);
            }
        }
    }
    __syncthreads();   // (the next stretch's tiles go where these rows were)
}

// The parts of a unit -> its output.  Part x of [0, n) is at part_of(x).  Sixteen lanes take a row; where there are few rows, several groups
// of lanes share a row's parts and are joined through LDS.
template <typename T, int D, typename PartOf>
__device__ __forceinline__ void join_unit(const Stretch &u, int tile, int n, PartOf part_of, unsigned char *lds) {
    constexpr int PER = D / 16, BATCH = 4, CROW = D + 4;
    const int tid = threadIdx.x, t = tid % 16, who = tid / 16;
    const int rows = min(u.rows - 16 * tile, kRows);   // of this row tile
    int live = 1;
    while (live < rows) live *= 2;
    const int row = who & (live - 1), group = who / live, groups = 16 / live, at_row = min(row, rows - 1);
    float m_run = -INFINITY, l_run = 0.0f;
    float2_t acc[PER / 2];
#pragma unroll
    for (int e = 0; e < PER / 2; e++) acc[e] = float2_t{0.0f, 0.0f};
    for (int x0 = group; x0 < n; x0 += groups * BATCH) {
        float m[BATCH], l[BATCH];
        float2_t v[BATCH][PER / 2];
#pragma unroll
        for (int y = 0; y < BATCH; y++) {
            const float *part = part_of(min(x0 + y * groups, n - 1));
            m[y] = get(part + kRows * D + at_row), l[y] = get(part + kRows * D + kRows + at_row);
#pragma unroll
            for (int e = 0; e < PER / 2; e++) v[y][e] = get2(part + at_row * D + 2 * t + 32 * e);
        }
#pragma unroll
        for (int y = 0; y < BATCH; y++) {
            // (without keys: a maximum of -inf and a sum of 0; scores that are all NaN raise no maximum either, but their sum is NaN)
            const bool has = x0 + y * groups < n && (m[y] != -INFINITY || l[y] != 0.0f);
            const float mm = has ? fmaxf(m_run, m[y]) : m_run, ref = mm == -INFINITY ? 0.0f : mm;
            const float keep = __builtin_amdgcn_exp2f(m_run - ref), f = has ? __builtin_amdgcn_exp2f(m[y] - ref) : 0.0f;
            const float was = m_run == -INFINITY && l_run == 0.0f ? 0.0f : keep;
            l_run = l_run * was + (has ? f * l[y] : 0.0f);
#pragma unroll
            for (int e = 0; e < PER / 2; e++)
#pragma unroll
                for (int z = 0; z < 2; z++) acc[e][z] = acc[e][z] * was + (has ? f * v[y][e][z] : 0.0f);
            m_run = mm;
        }
    }
    float *comb = reinterpret_cast<float *>(lds), *comb_ml = comb + 16 * CROW;
#pragma unroll
    for (int e = 0; e < PER / 2; e++) *reinterpret_cast<float2_t *>(comb + who * CROW + 2 * t + 32 * e) = acc[e];
    if (t == 0) comb_ml[2 * who] = m_run, comb_ml[2 * who + 1] = l_run;
    __syncthreads();
    if (who < rows) {   // (who == row of group 0)
        float mm = -INFINITY, l = 0.0f;
        for (int g = 0; g < groups; g++) mm = fmaxf(mm, comb_ml[2 * (g * live + who)]);
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float2_t sum[PER / 2];
#pragma unroll
        for (int e = 0; e < PER / 2; e++) sum[e] = float2_t{0.0f, 0.0f};
        for (int g = 0; g < groups; g++) {
            const int from = g * live + who;
            const float m = comb_ml[2 * from], lg = comb_ml[2 * from + 1];
            const bool has = m != -INFINITY || lg != 0.0f;
            const float f = has ? __builtin_amdgcn_exp2f(m - ref) : 0.0f;
            l += has ? f * lg : 0.0f;
#pragma unroll
            for (int e = 0; e < PER / 2; e++) {
                const float2_t v = *reinterpret_cast<const float2_t *>(comb + from * CROW + 2 * t + 32 * e);
#pragma unroll
                for (int z = 0; z < 2; z++) sum[e][z] = has ? __builtin_fmaf(f, v[z], sum[e][z]) : sum[e][z];
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        Arguments p = arguments_again();
        T *out = reinterpret_cast<T *>(p.out) + q_row(p, u.b, u.kvh, u.row0 + 16 * tile + who).at * D;
#pragma unroll
        for (int e = 0; e < PER / 2; e++) {
            struct alignas(2 * sizeof(T)) Two { T e[2]; } two;
            two.e[0] = (T)(sum[e][0] * inv), two.e[1] = (T)(sum[e][1] * inv);
            *reinterpret_cast<Two *>(out + 2 * t + 32 * e) = two;
        }
    }
    __syncthreads();
}

// Whether a sequence begins with its neighbour's page, as beams of a request do.  Pages that one workgroup reads go past the caches (64 sequences
// of 64 to 8192 keys 195 us, through them 217; 8 x 1000 13.0 | 13.5), those that several do through them (32 requests of 8 beams over 700 common
// keys 64 us, past them 86; 8 of 8 over 4000 67 | 76).
__device__ __forceinline__ bool shares_pages(Arguments p, int b) {
    if (p.table_width == 0) return false;
    const int mine = p.table[b * p.table_width], left = p.table[max(b - 1, 0) * p.table_width], right = p.table[min(b + 1, p.B - 1) * p.table_width];
    return (b > 0 && left == mine) || (b + 1 < p.B && right == mine);
}

// Sums of a wave's lanes up to each one: along the rows of 16 lanes, then over the rows.
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int wave_sums(int x) {
    constexpr int kUp = 0x110, kRow15 = 0x142, kRow31 = 0x143;
    x += moved<kUp + 1, 0xf>(x), x += moved<kUp + 2, 0xf>(x), x += moved<kUp + 4, 0xf>(x), x += moved<kUp + 8, 0xf>(x);
    x += moved<kRow15, 0xa>(x), x += moved<kRow31, 0xc>(x);
    return x;
}

// Where a workgroup stands on the line: what is looked at between stretches alone is in LDS, since the loop needs the scalar registers.
struct Line { int per, at, end, b, unit, len, steps, first, once, last, poison; };

// A workgroup's stretch, unit by unit; units of a step a wave each, side by side (200 sequences of 30 keys of 32 heads, f16, 24.7 us, one after the
// other 50.3; of 64 38.9 | 55.3, of 100 61.1 | 67.2; of 30 to 60, f32, 84.6 | 122).
template <typename T, int D, int RT, bool MAY_ONCE>
__device__ __forceinline__ void walk_line(Line &s_line, unsigned char *lds) {
    const int tid = threadIdx.x;
    for (;;) {
        Stretch u;
        {
            Arguments p = arguments_again();
            const int unit = uniform(s_line.unit), steps = uniform(s_line.steps);
            u.b = uniform(s_line.b), u.len = uniform(s_line.len), u.first = uniform(s_line.first);
            const auto &row_units = p.row_units[RT >> 1];
            u.kvh = divided(row_units, unit);
            u.row0 = (unit - u.kvh * (int)row_units.d) * RT * kRows, u.rows = min(RT * kRows, p.Sq * p.G - u.row0);
            u.end = min(steps, u.first + uniform(s_line.end) - uniform(s_line.at));
            u.part = u.first == 0 && u.end == steps ? nullptr : p.parts + (2 * (int64_t)blockIdx.x + (u.first == 0)) * (RT * kLinePart(D));
        }
        int done = 1;   // units, where they are short
        if constexpr (RT == 1) {
            Arguments p = arguments_again();
            if (u.len <= kStep) done = min(min(kWaves, p.Hkv * (int)p.row_units[0].d - uniform(s_line.unit)), uniform(s_line.end) - uniform(s_line.at));
        }
        if (RT == 1 && done > 1) {
            if constexpr (RT == 1) {
                const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
                if (w < done) {
                    Arguments p = arguments_again();
                    const int unit = uniform(s_line.unit) + w;
                    u.kvh = divided(p.row_units[0], unit);
                    u.row0 = (unit - u.kvh * (int)p.row_units[0].d) * kRows, u.rows = min(kRows, p.Sq * p.G - u.row0);
                    if (MAY_ONCE && uniform(s_line.once)) stretch_body<T, D, 1, MAY_ONCE, true>(u, s_line.poison, lds);
                    else stretch_body<T, D, 1, false, true>(u, s_line.poison, lds);
                }
            }
        } else if (MAY_ONCE && uniform(s_line.once)) stretch_body<T, D, RT, MAY_ONCE, false>(u, s_line.poison, lds);
        else stretch_body<T, D, RT, false, false>(u, s_line.poison, lds);
        if (u.part) {
            Arguments p = arguments_again();
            const unsigned per = uniform(s_line.per), unit_at = uniform(s_line.at) - u.first;
            const int first = (int)(unit_at / per), n = (int)((unit_at + uniform(s_line.steps) - 1) / per) - first + 1;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this thread's parts have completed
            __syncthreads();                                     // ... and so have the whole workgroup's
            if (tid == 0) {
                int *counter = p.counters + first;   // (a workgroup cuts one unit at most at its end)
                s_line.last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
                if (s_line.last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            float *parts = p.parts;
            if (s_line.last)
                for (int y = 0; y < RT && 16 * y < u.rows; y++)
                    join_unit<T, D>(u, y, n, [&](int x) { return parts + ((2 * (int64_t)(first + x) + (x == 0)) * RT + y) * kLinePart(D); }, lds);
        }
        const int steps_done = done > 1 ? done : u.end - u.first;
        if (uniform(s_line.at) + steps_done >= uniform(s_line.end)) return;
        __syncthreads();   // (everybody has read where the line stands)
        if (tid == 0) {
            Arguments p = arguments_again();
            s_line.at += steps_done, s_line.unit += done, s_line.first = 0;
            if (s_line.unit == p.Hkv * (int)p.row_units[RT >> 1].d) {
                const int len = min(max(p.lens[u.b + 1], 0), p.most);
                s_line.once = p.row_units[RT >> 1].d == 1 && !shares_pages(p, u.b + 1);
                s_line.unit = 0, s_line.b = u.b + 1, s_line.len = len, s_line.steps = max((len + kStep - 1) / kStep, 1);
            }
        }
        __syncthreads();
    }
}

// A unit of s steps in stretches of n is joined out of s / n parts by one workgroup: n + (s / n) c is least at n = sqrt(s c), and c, what a part
// costs there against a step, goes with its rows (s: of the sequences on average).  Without, with 0.01, 0.02 and 0.04 a row, us: 100000 keys of one kv head
// with 8 rows 57.7, 34.0, 36.7, 41.9; 2 x 27741 of two with 7 22.8, 20.9, 19.8, 19.8; 5264 of eight with 8, f32, 25.9, 25.8, 22.2, 25.1; 4000 of two with 12
// 16.2, 16.4, 14.5, 17.3.
constexpr float kPartCost = 0.02f;

// RT: row tiles of a unit, which share the keys that it reads.  Where that leaves no more than a step or two per workgroup and tile, units take
// half as many, and again: what a workgroup does for one tile after the other is then what takes the time.  In us, more tiles and half as many: 2
// sequences of up to 300 keys, 7 heads' 5 queries 12.9 (four), 9.8, 7.8; 4 of 3000 to 6000, 8 heads' 6 queries 35.3 (four), 26.3; 20 of up to 900, 8
// heads' 4 queries 20.0 (two), 16.2; beyond the rule 40 of 500 to 900, 4 heads' 5 queries of 128 37.0 (two), 45.2.  Where sequences are of two steps
// on average, or fewer, one tile: a unit of a step is then a wave's (150 of up to 60, 8 heads' 4 queries 17.9 with two tiles, 12.4; 200 of 60 to 200, 4
// heads' 5 queries of 128 46.5, 43.5).
template <typename T, int D, int RT>
__global__ __launch_bounds__(kThreads, 2) void sdpa_paged_kernel(PagedDev) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[line_lds(sizeof(T), D)];
    __shared__ int s_sums[kWaves], s_totals[kWaves];
    __shared__ Line s_line;
    int rt = RT;
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    {
        Arguments p = arguments_again();
        auto len_of = [&](int b) { return min(max(p.lens[b], 0), p.most); };
        auto steps_of = [&](int len) { return max((len + kStep - 1) / kStep, 1); };   // (one for nothing: its rows are zeros)

        // the line's length (below 2^28 of units of RT tiles: checked by the host; below 2^30 of any), and this workgroup's stretch
        int len = tid < p.B ? len_of(tid) : 0, mine = tid < p.B ? steps_of(len) : 0, all = mine;
        bool shares = tid < p.B && shares_pages(p, tid);
        for (int b = tid + kThreads; b < p.B; b += kThreads) all += steps_of(len_of(b));
        int up = wave_sums(mine);
        const int sum = p.B > kThreads ? wave_sums(all) : up;
        if (lane == 63) s_sums[w] = up, s_totals[w] = sum;
        __syncthreads();
        const int all_steps = s_totals[0] + s_totals[1] + s_totals[2] + s_totals[3];   // of one unit of every sequence
        auto units_of = [&](int rt) { return p.Hkv * (int)p.row_units[rt >> 1].d; };   // of a sequence
        while (rt > 1 && (all_steps * units_of(rt) <= rt * (int)gridDim.x || all_steps <= 2 * p.B)) rt >>= 1;
        const int units = units_of(rt), total = all_steps * units;
        const int per = max(divided(p.by_workgroups, total + (int)gridDim.x - 1), max((int)__builtin_amdgcn_sqrtf((float)all_steps * p.part_cost), 1));
        const int begin = blockIdx.x * per, end = min(begin + per, total);
        if (begin >= end) return;
        // the sequence where it begins
        for (int b0 = 0, carry = 0;;) {
            int before = carry;
            for (int x = 0; x < w; x++) before += s_sums[x];
            const int from = (before + up - mine) * units;
            if (b0 + tid < p.B && from <= begin && begin < from + mine * units) {
                s_line.b = b0 + tid, s_line.len = len, s_line.steps = mine;
                s_line.unit = (unsigned)(begin - from) / (unsigned)mine, s_line.first = (unsigned)(begin - from) % (unsigned)mine;
                s_line.once = units == p.Hkv && !shares;
            }
            carry += s_sums[0] + s_sums[1] + s_sums[2] + s_sums[3];
            b0 += kThreads;
            if (b0 >= p.B || carry * units > begin) break;
            len = b0 + tid < p.B ? len_of(b0 + tid) : 0, mine = b0 + tid < p.B ? steps_of(len) : 0;
            shares = b0 + tid < p.B && shares_pages(p, b0 + tid);
            up = wave_sums(mine);
            __syncthreads();
            if (lane == 63) s_sums[w] = up;
            __syncthreads();
        }
        if (tid == 0) s_line.per = per, s_line.at = begin, s_line.end = end, s_line.poison = 0;
        __syncthreads();
    }
    if (rt == RT) return walk_line<T, D, RT, true>(s_line, lds);
    if constexpr (RT > 2)
        if (rt == 2) return walk_line<T, D, 2, false>(s_line, lds);
    if constexpr (RT > 1) walk_line<T, D, 1, false>(s_line, lds);
}

template <typename T, int D, int RT>
int launch_line(const PagedDev &p, int workgroups, hipStream_t s) {
    sdpa_paged_kernel<T, D, RT><<<dim3((unsigned)workgroups), kThreads, 0, s>>>(p);
    TROCM_HIP(hipGetLastError());
    return 0;
}

int line_workgroups() { return 2 * num_compute_units(); }

}  // namespace

// Row tiles of a unit, at most: as many as a lane's registers hold (f32 of head size 128 has no place for two rows' queries in LDS either).  91
// sequences of 2880 to 5761 keys: 8 heads' 5 queries of head size 64 in four tiles 175 us, in two 300; 4 heads' 5 of 128 in two 275, in one 561.
static int row_tiles_of_unit(int64_t rows, int64_t es, int64_t D) {
    if (rows <= kRows || in_lds((int)es, (int)D)) return 1;
    return rows > 2 * kRows && es == 2 && D == 64 ? 4 : 2;
}

static size_t bytes_for(int64_t row_tiles, int64_t D) { return kWsCounterBytes + (size_t)(2 * line_workgroups() * row_tiles * kLinePart((int)D)) * 4; }

size_t sdpa_paged_workspace_bytes(int64_t, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D) {
    return D == 64 || D == 128 ? bytes_for(row_tiles_of_unit(Hq / Hkv * Sq, 2, D), D) : kWsCounterBytes;
}

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
    const uint64_t bits = (uint64_t)(uintptr_t)a.q | (uint64_t)(uintptr_t)a.out | (uint64_t)(uintptr_t)a.k | (uint64_t)(uintptr_t)a.v | (uint64_t)p.stride_page | (uint64_t)p.stride_h | (uint64_t)p.stride_t;
    if ((a.D == 64 || a.D == 128) && a.page_size % 16 == 0 && bits % 16 == 0 && a.n_pages > 0 && p.stride_t < (1 << 27) && a.workspace &&
        a.workspace_bytes >= bytes_for(1, a.D)) {
        const int64_t rows = a.Hq / a.Hkv * a.Sq;
        int rt = row_tiles_of_unit(rows, es, a.D);
        while (rt > 1 && a.workspace_bytes < bytes_for(rt, a.D)) rt /= 2;
        for (int i = 0; i < 3; i++) p.row_units[i] = fast_div((rows + (kRows << i) - 1) / (kRows << i));
        p.by_g = fast_div(p.G), p.by_workgroups = fast_div(line_workgroups());
        p.counters = (int *)a.workspace, p.parts = (float *)((char *)a.workspace + kWsCounterBytes);
        // a line's tiles are counted in 31 bits: as many sequences in a launch as cannot be more
        const int64_t most_steps = std::max<int64_t>((p.most + kStep - 1) / kStep, 1) * a.Hkv * p.row_units[rt >> 1].d, seqs = (1 << 28) / most_steps;
        if (seqs > 0) {
            for (int64_t b0 = 0; b0 < a.B; b0 += seqs) {
                PagedDev part = p;
                part.B = (int)std::min(seqs, a.B - b0), part.part_cost = kPartCost * (float)std::min<int64_t>(rows, kRows) / (float)part.B;
                part.q += b0 * a.Hq * a.Sq * a.D * es, part.out += b0 * a.Hq * a.Sq * a.D * es;
                part.table += b0 * a.table_width, part.lens += b0;
                const int n = line_workgroups();
                int rc;
                if (a.dtype == TROCM_F16) {
                    if (rt == 4) rc = launch_line<_Float16, 64, 4>(part, n, s);
                    else if (rt == 1) rc = a.D == 64 ? launch_line<_Float16, 64, 1>(part, n, s) : launch_line<_Float16, 128, 1>(part, n, s);
                    else rc = a.D == 64 ? launch_line<_Float16, 64, 2>(part, n, s) : launch_line<_Float16, 128, 2>(part, n, s);
                } else if (a.D == 64) {
                    rc = rt == 1 ? launch_line<float, 64, 1>(part, n, s) : launch_line<float, 64, 2>(part, n, s);
                } else {
                    rc = launch_line<float, 128, 1>(part, n, s);
                }
                if (rc) return rc;
            }
            return 0;
        }
    }
    TROCM_REQUIRE(a.D <= kRowsMaxD, "sdpa_paged: head_dim %lld is more than %d", (long long)a.D, kRowsMaxD);
    const dim3 grid((unsigned)std::min<int64_t>(a.B * a.Hq * a.Sq, kMostBlocks));
    if (a.dtype == TROCM_F16) sdpa_paged_any_kernel<_Float16><<<grid, kAnyThreads, 0, s>>>(p);
    else sdpa_paged_any_kernel<float><<<grid, kAnyThreads, 0, s>>>(p);
    TROCM_HIP(hipGetLastError());
    return 0;
}

}  // namespace trocm
