// The best continuations of a request's beams: of all values c = score + x - log sum exp(x) over beams and vocabulary the `keep` largest,
// ties to the lowest (beam, token).
//
// Within a beam the order of c is the order of the logits, which is exact; only between beams does c itself count.  So the vocabulary is
// read once: a workgroup streams a part of a row through registers, makes its maximum and sum (f32 for eight values, then f64) and keeps its
// `keep` largest logits; the last workgroup of a request to arrive puts the parts together in f64.  Where values of two beams are nearer than
// those sums can be told apart, the beams' sums are made again, exactly, against the beams' own largest values: rows that are others shifted, or in
// another order, tie exactly.  They are made exactly, too, where 64 bits hold one value for several logits (logits next to nothing, scores of 1e9 and
// more), which are then looked for in the rows themselves.
//
// The largest of a wave's values: the K-th largest of its lanes' maxima is found, nearly, by bisection over the upper bits of an order-preserving
// integer (ballots and counts); at least K values reach it, and few more than that, which are listed in LDS and ranked by counting.
//
// What bounds it: one request (4 beams of 32000, f32) is a chain of stages, 10.2 us; 32 requests of 8 beams of 128256 in f16 take 30.9 us.  By the
// device's clock its 768 workgroups, which all begin within 0.5 us, end their streams after 9.3 to 19.7 us (half of them after 15.2; alone, without
// others' ends beside them, the streams take 13.4, 4.9 TB/s; the vector ALUs are busy for half of the time, exponentials for most of that); what one
// does behind its stream takes 4.0, its count 0.7, a request's join 5.5, and behind the last streams there is nothing left to overlap those with.
//
// What an exact sum takes: 58 us a beam of 128256, one after the other: a request of 8 beams that are copies of one another 470 us for 16 (f16 and f32),
// 32 of them 850 and 1080 for 31 and 33; of 32000 in f32 four copies 77 for 10.  Masks of -inf are no slower (39 us where 20 tokens of
// 128256 are allowed); a finite mask, of which a workgroup sees nothing else, is found out to be one value in another turn over its part (417 us in f16,
// 617 in f32; one request 57).
#include <hip/hip_fp16.h>
#include <math.h>
#include <algorithm>
#include "common.h"
#include "fast_div.h"

namespace trocm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kPiece = 8;                     // consecutive values of a lane
constexpr int kWaveList = 512;                // values that a wave lists
constexpr uint32_t kLowest = 0x007fffffu;     // key_of(-inf); 0 is below all values: nothing there

struct alignas(8) Candidate { float x; int token; };     // token < 0: none

struct SelectDev {
    const char *logits;
    int64_t row_bytes;
    int vocab, parts, turns, keep, beams, eos, row0;   // row0: of this launch's first row, for parents
    int *counters;              // of a request: how many of its parts are there
    float *part_max;
    double *part_sum;
    Candidate *part_best;       // [row][part][keep], best first
    const float *scores;
    const int *ended;
    float *scores_out;
    int *parents, *tokens, *ended_out;
    FastDiv by_parts, by_row_candidates, by_keep, by_beams;
};

// Integers in the order of the numbers; both zeros are one number and NaN counts as -inf.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    const uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return x != x ? kLowest : k;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __builtin_bit_cast(float, k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }

__device__ __forceinline__ int lanes_below(uint64_t mask) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0)); }

// A t that at least `count` of the wave's keys (one per lane) reach, and few more: the largest one of 20 bits and zeros; 0 if there are fewer
// keys.  Two bits a step.
__device__ __forceinline__ uint32_t bound_of_lanes(uint32_t key, int count) {
    auto reach = [&](uint32_t t) __attribute__((always_inline)) { return __popcll(__builtin_amdgcn_ballot_w64(key >= t)) >= count; };
    uint32_t t = 0;
#pragma unroll 1
    for (int at = 30; at >= 12; at -= 2) {
        const bool one = reach(t | 1u << at), two = reach(t | 2u << at), three = reach(t | 3u << at);
        t |= three ? 3u << at : two ? 2u << at : one ? 1u << at : 0u;
    }
    return t;
}

// A wave's largest value and its sum, everywhere: along the rows of 16 lanes, then over the rows; the last lane has it.
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int none, int x) { return __builtin_amdgcn_update_dpp(none, x, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ float larger(float x) {
    return fmaxf(x, __builtin_bit_cast(float, moved<CTRL, ROWS>(__builtin_bit_cast(int, -INFINITY), __builtin_bit_cast(int, x))));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double plus(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = (uint32_t)moved<CTRL, ROWS>(0, (int)(uint32_t)b), hi = (uint32_t)moved<CTRL, ROWS>(0, (int)(uint32_t)(b >> 32));
    return x + __builtin_bit_cast(double, (uint64_t)lo | (uint64_t)hi << 32);
}
constexpr int kShift = 0x110, kRow15 = 0x142, kRow31 = 0x143;   // lanes up within a row by n; lane 15 of a row to the next row; lane 31 to the upper half
__device__ __forceinline__ float wave_most(float x) {
    x = fmaxf(x, -INFINITY);
    x = larger<kShift + 1, 0xf>(x), x = larger<kShift + 2, 0xf>(x), x = larger<kShift + 4, 0xf>(x), x = larger<kShift + 8, 0xf>(x);
    x = larger<kRow15, 0xa>(x), x = larger<kRow31, 0xc>(x);
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
__device__ __forceinline__ double wave_sum(double x) {
    x = plus<kShift + 1, 0xf>(x), x = plus<kShift + 2, 0xf>(x), x = plus<kShift + 4, 0xf>(x), x = plus<kShift + 8, 0xf>(x);
    x = plus<kRow15, 0xa>(x), x = plus<kRow31, 0xc>(x);
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, 63) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), 63) << 32);
}

// The same among a row's 16 lanes, everywhere in the row: rotations by 8, 4, 2, 1.
constexpr int kRotate = 0x120;
__device__ __forceinline__ float row_most(float x) {
    x = larger<kRotate + 8, 0xf>(x), x = larger<kRotate + 4, 0xf>(x), x = larger<kRotate + 2, 0xf>(x);
    return larger<kRotate + 1, 0xf>(x);
}
__device__ __forceinline__ double row_sum(double x) {
    x = plus<kRotate + 8, 0xf>(x), x = plus<kRotate + 4, 0xf>(x), x = plus<kRotate + 2, 0xf>(x);
    return plus<kRotate + 1, 0xf>(x);
}

// What a workgroup leaves for the one that puts a request together: written through to where every compute unit sees it once it completes.
template <typename X>
__device__ __forceinline__ void put(X *at, X x) {
    static_assert(sizeof(X) == 8 || sizeof(X) == 4, "one store");
    if constexpr (sizeof(X) == 8) __hip_atomic_store(reinterpret_cast<uint64_t *>(at), __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else __hip_atomic_store(reinterpret_cast<uint32_t *>(at), __builtin_bit_cast(uint32_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename X>
__device__ __forceinline__ X get(const X *at) {
    if constexpr (sizeof(X) == 8) return __builtin_bit_cast(X, __hip_atomic_load(reinterpret_cast<const uint64_t *>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    else return __builtin_bit_cast(X, __hip_atomic_load(reinterpret_cast<const uint32_t *>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

template <typename T> using Eight = T __attribute__((ext_vector_type(kPiece)));

struct ScanLds {
    int list[kWaves][kWaveList];      // tokens
    uint64_t all[kWaves * kWaveList];   // values' keys above what their tokens lack of 2^32: the order of the choice
    double sum[kWaves];
    float max[kWaves];
    uint32_t bound[kWaves];
    int total;
};

// A part of a row: `turns` tiles of kThreads * kPiece * C values, the next one in flight while one is looked at.
template <typename T, int C>
__device__ __forceinline__ void scan_part(const SelectDev &p, int row, int part, ScanLds &lds) {
    constexpr int kTile = kThreads * kPiece * C, kStep = kThreads * kPiece;
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const T *from = reinterpret_cast<const T *>(p.logits + row * p.row_bytes);
    const int begin = part * p.turns * kTile, turns = min(p.turns, (p.vocab - begin + kTile - 1) / kTile), mine = begin + tid * kPiece;
    // (rows begin where they begin: pieces are loaded from any element on; what is behind the row's end is -inf)
    auto piece_at = [&](int i) __attribute__((always_inline)) {
        Eight<T> v;
        if (i <= p.vocab - kPiece) {
            __builtin_memcpy(&v, from + i, sizeof(v));
        } else {
#pragma unroll
            for (int e = 0; e < kPiece; e++) v[e] = i + e < p.vocab ? from[i + e] : (T)-INFINITY;
        }
        return v;
    };
    Eight<T> x[C], coming[C];
    auto load = [&](int turn) __attribute__((always_inline)) {
        const int i = mine + turn * kTile;
        if (begin + turn * kTile <= p.vocab - kTile) {
#pragma unroll
            for (int c = 0; c < C; c++) __builtin_memcpy(&coming[c], from + i + c * kStep, sizeof(coming[c]));
        } else {
#pragma unroll
            for (int c = 0; c < C; c++) coming[c] = piece_at(i + c * kStep);
        }
    };
    int *list = lds.list[w];
    int n = 0;
    uint32_t bound_key = 0;
    float least = -INFINITY, m = -INFINITY, top = -INFINITY;
    double all = 0.0;
    // Weights against a reference c, a = log2 e as f32 has it (what a is off by counts for x - m alone: join_request's err has it).  f16: 2^(x a - c)
    // in one step, c = m a rounded, and what that is off by, 2^-8 at most, is put right with the whole sum.  f32: 2^((x - c) a), c = m itself:
    // beyond 2^24, where masks are, m a would be off by 1 and more, and from 1e10 on by more than f32 has exponents.
    constexpr bool kProduct = sizeof(T) == 2;
    float c_m = 0.0f;
    auto reference = [&] { return kProduct ? m * kLog2e : m; };
    auto weight = [&](T v) __attribute__((always_inline)) { return __builtin_amdgcn_exp2f(kProduct ? __builtin_fmaf((float)v, kLog2e, -c_m) : ((float)v - c_m) * kLog2e); };
    auto step = [&](double to) { return exp(kProduct ? to * 0.6931471805599453 : to); };   // of references
    load(0);
#pragma unroll 1
    for (int turn = 0; turn < turns; turn++) {
#pragma unroll
        for (int c = 0; c < C; c++) x[c] = coming[c];
        if (turn + 1 < turns) load(turn + 1);
        T most[C], top_t = (T)-INFINITY;   // of a piece; NaN only where all are
#pragma unroll
        for (int c = 0; c < C; c++) {
            auto v4 = __builtin_elementwise_max(__builtin_shufflevector(x[c], x[c], 0, 1, 2, 3), __builtin_shufflevector(x[c], x[c], 4, 5, 6, 7));
            auto v2 = __builtin_elementwise_max(__builtin_shufflevector(v4, v4, 0, 1), __builtin_shufflevector(v4, v4, 2, 3));
            most[c] = __builtin_elementwise_max(v2[0], v2[1]);
            top_t = __builtin_elementwise_max(top_t, most[c]);
        }
        const float now = (float)top_t;
        top = fmaxf(top, now);
        // Maximum and sum: f32 for the values of a piece, f64 from there on.  m is the largest value of the first tile, or of a later one that has
        // one more than 2 above.
        if (__builtin_amdgcn_ballot_w64(now - m > 2.0f)) {
            const float was = m, c_was = c_m;
            m = wave_most(top);
            c_m = reference();
            all = was == -INFINITY ? 0.0 : all * step((double)c_was - (double)c_m);
        }
#pragma unroll
        for (int c = 0; c < C; c++) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < kPiece; e++) sum += weight(x[c][e]);
            all += (double)sum;
        }
        if (__builtin_amdgcn_ballot_w64(all != all) && m < INFINITY) {   // a NaN counts as -inf: the sum so far again
            all = 0.0;
#pragma unroll 1
            for (int i = mine; i < min(mine + (turn + 1) * kTile, p.vocab); i += kStep) {
                const Eight<T> v = piece_at(i);
#pragma unroll
                for (int e = 0; e < kPiece; e++) {
                    const float t = weight(v[e]);
                    all += t == t ? (double)t : 0.0;
                }
            }
        }
        // The values that could be among the best: of the first tile at least `keep` reach its bound (all but -inf is listed where fewer
        // lanes have a value); from then on they do of all.
        if (turn == 0) bound_key = max(bound_of_lanes(key_of(top), p.keep), kLowest), least = value_of(bound_key);
        if (__builtin_amdgcn_ballot_w64(now >= least && now > -INFINITY)) {
            uint32_t hits = 0;   // bit 8 c + e
#pragma unroll
            for (int c = 0; c < C; c++)
                if (__builtin_amdgcn_ballot_w64((float)most[c] >= least)) {
                    asm("" : "+v"(x[c]));   // (halves that are kept as 32 bits from the sum to here would take twice the registers)
#pragma unroll
                    for (int e = 0; e < kPiece; e++) hits |= (float)x[c][e] >= least && (float)x[c][e] > -INFINITY ? 1u << (c * kPiece + e) : 0u;
                }
            while (const uint64_t in = __builtin_amdgcn_ballot_w64(hits != 0)) {
                const int b = __ffs(hits) - 1, at = n + lanes_below(in);
                if (hits && at < kWaveList) list[at] = mine + turn * kTile + (b / kPiece) * kStep + b % kPiece;
                hits &= hits - 1;
                n += __popcll(in);
            }
        }
    }
    // (the first values of the list are asked for ahead of what does not need them)
    constexpr int kAhead = 2;
    int token[kAhead];
    float value[kAhead];
#pragma unroll
    for (int y = 0; y < kAhead; y++) {
        token[y] = lane + 64 * y < min(n, kWaveList) ? list[lane + 64 * y] : -1;
        value[y] = token[y] >= 0 ? (float)from[token[y]] : -INFINITY;
    }
    const uint32_t wave_bound = max(bound_of_lanes(key_of(top), p.keep), bound_key);
    if (lane == 0) lds.bound[w] = wave_bound;
    if (tid == 0) lds.total = 0;
    if (kProduct && m < INFINITY) all = m == -INFINITY ? 0.0 : all * step((double)c_m - (double)m * (double)kLog2e);   // against m (exact but for f64)
    all = wave_sum(all);
    if (lane == 0) lds.max[w] = m, lds.sum[w] = all;
    __syncthreads();
    bound_key = max(max(lds.bound[0], lds.bound[1]), max(lds.bound[2], lds.bound[3]));   // (at least `keep` values reach the largest of the waves')
    least = value_of(bound_key);

    // Where the list does not hold what reaches the wave's own bound, equal values above all, or the workgroup's bound is -inf: what is above the
    // bound, and of what equals it only so many as could be among the best, in their order: tiles, pieces, lanes, values of a piece.
    if (n > kWaveList || least == -INFINITY) {
        const int end = min(begin + turns * kTile, p.vocab);
        auto count = [&](float reach) {
            int k = 0;
#pragma unroll 1
            for (int i = mine; i - lane * kPiece < end; i += kStep) {
                const Eight<T> v = piece_at(i);
#pragma unroll
                for (int e = 0; e < kPiece; e++) k += __popcll(__builtin_amdgcn_ballot_w64((float)v[e] >= reach));
            }
            return k;
        };
        bool above = __builtin_amdgcn_ballot_w64(top > least) != 0;
        if (above && count(value_of(bound_key + 1)) > kWaveList - kBeamMaxKeep) {   // the bound of all values, above which there are fewer than `keep`
            bound_key = 0;
#pragma unroll 1
            for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
                if ((bound_key | bit) <= kLowest || ((bound_key | bit) <= 0xff800000u && count(value_of(bound_key | bit)) >= p.keep)) bound_key |= bit;
            bound_key = max(bound_key, kLowest);
        }
        const float bound = value_of(bound_key);
        n = 0;
        int equal = 0;
#pragma unroll 1
        for (int i = mine; i - lane * kPiece < end && (above || equal < p.keep); i += kStep) {
            const Eight<T> v = piece_at(i);
            uint32_t hits = 0, ties = 0;
#pragma unroll
            for (int e = 0; e < kPiece; e++) {
                const float f = (float)v[e] == (float)v[e] ? (float)v[e] : -INFINITY;
                hits |= (f > bound ? 1u : 0u) << e, ties |= (f == bound && i + e < p.vocab ? 1u : 0u) << e;
            }
            while (const uint64_t in = __builtin_amdgcn_ballot_w64(hits != 0)) {
                if (hits) list[n + lanes_below(in)] = i + __ffs(hits) - 1;
                hits &= hits - 1;
                n += __popcll(in);
            }
            if (equal >= p.keep) continue;
            int before = equal, here = 0;
#pragma unroll
            for (int bit = 0; bit < 4; bit++) {
                const uint64_t lanes = __builtin_amdgcn_ballot_w64((__popc(ties) >> bit) & 1);
                before += lanes_below(lanes) << bit, here += __popcll(lanes) << bit;
            }
            for (int at = n + before - equal; ties && before < p.keep; ties &= ties - 1, at++, before++) list[at] = i + __ffs(ties) - 1;
            n += min(here, p.keep - equal), equal = min(equal + here, p.keep);
        }
        least = -INFINITY;   // (all of the list)
#pragma unroll
        for (int y = 0; y < kAhead; y++) {
            token[y] = lane + 64 * y < n ? list[lane + 64 * y] : -1;
            value[y] = token[y] >= 0 ? (float)from[token[y]] : -INFINITY;
        }
    }

    // the workgroup's: every listed value counts those before it
    auto add = [&](int t, float v) __attribute__((always_inline)) {
        const bool in = t >= 0 && !(v < least);   // (NaN: -inf, where that is looked for)
        const uint64_t lanes = __builtin_amdgcn_ballot_w64(in);
        if (!lanes) return;
        int at = 0;
        if (lane == 0) at = atomicAdd(&lds.total, __popcll(lanes));
        at = __builtin_amdgcn_readfirstlane(at) + lanes_below(lanes);
        if (in) lds.all[at] = (uint64_t)key_of(v) << 32 | (uint32_t)~t;
    };
#pragma unroll
    for (int y = 0; y < kAhead; y++) add(token[y], value[y]);
    for (int j0 = 64 * kAhead; j0 < n; j0 += 64) {
        const int t = j0 + lane < n ? list[j0 + lane] : -1;
        add(t, t >= 0 ? (float)from[t] : -INFINITY);
    }
    __syncthreads();
    const int total = lds.total;
    const int64_t at_part = (int64_t)row * p.parts + part;
    Candidate *best = p.part_best + at_part * p.keep;
    for (int j = tid; j < total; j += kThreads) {
        const uint64_t c = lds.all[j];
        int rank = 0;
#pragma unroll 8
        for (int z = 0; z < total; z++) rank += lds.all[z] > c ? 1 : 0;
        if (rank < p.keep) put(best + rank, Candidate{value_of((uint32_t)(c >> 32)), (int)~(uint32_t)c});
    }
    for (int j = total + tid; j < p.keep; j += kThreads) put(best + j, Candidate{-INFINITY, -1});
    if (w == 0) {   // (a lane per wave's sum)
        const float mine_m = lds.max[lane & 3], mm = fmaxf(fmaxf(lds.max[0], lds.max[1]), fmaxf(lds.max[2], lds.max[3]));
        double l = mine_m == -INFINITY ? 0.0 : lds.sum[lane & 3] * exp((double)mine_m - (double)mm);
        l += __shfl_xor(l, 1, 64);
        l += __shfl_xor(l, 2, 64);
        if (lane == 0) put(p.part_max + at_part, mm), put(p.part_sum + at_part, l);
    }
}

// ---- parts and beams put together: the last workgroup of a request ----------------------------------------------------------

constexpr int kJoinList = 1024, kJoinParts = 1024;   // parts of a request: checked by the host
struct alignas(16) Choice { double c; int place, beam; };   // place: beam * vocab + token (below 2^31, checked by the host); < 0: none

__device__ __forceinline__ bool before(double c, int place, double d, int other) { return c > d || (c == d && place < other); }

// 2^t for t <= 0 times 2^shift, in f64: the exponential's series for the fraction, of at most a half (the term behind the last is 1e-19).  Zero
// from 2^-2000 on, -inf among them (of which the fraction would be no number).
__device__ __forceinline__ double exp2_scaled(double t, int shift) {
    t = fmax(t, -2000.0);
    const double n = __builtin_rint(t), r = (t - n) * 0.6931471805599453;
    double y = 1.0 / 87178291200.0;
    constexpr double kInverse[14] = {1.0 / 6227020800.0, 1.0 / 479001600.0, 1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0, 1.0 / 120.0, 1.0 / 24.0, 1.0 / 6.0, 0.5, 1.0, 1.0};
#pragma unroll
    for (int i = 0; i < 14; i++) y = __builtin_fma(y, r, kInverse[i]);
    return __builtin_ldexp(y, (int)n + shift);
}

// log sum exp(x - m) of a row whose largest value is m, the same for the same differences in any order: terms of 64 bits, rounded to whole multiples of
// 2^-61 of the largest and added as integers of 128: off by 2^-51 and 2^-62 a term.  All threads; only where two beams are nearer than their 32-bit sums tell apart.
template <typename T>
__device__ __forceinline__ double exact_log_sum(const T *x, int vocab, float m, uint64_t *lds_sums) {
    constexpr int kShift = 61;
    const int tid = threadIdx.x;
    uint64_t sum = 0, high = 0;
    auto plus = [&](uint64_t low, uint64_t upper) { sum += low, high += upper + (sum < low ? 1 : 0); };
    auto add = [&](float v) { plus(v == v ? (uint64_t)(exp2_scaled(((double)v - (double)m) * 1.4426950408889634, kShift) + 0.5) : 0, 0); };
    constexpr int kStep = kThreads * kPiece;
    const int whole = vocab / kPiece * kPiece;
    Eight<T> coming;
    if (tid * kPiece < whole) __builtin_memcpy(&coming, x + tid * kPiece, sizeof(coming));
#pragma unroll 1
    for (int i = tid * kPiece; i < whole; i += kStep) {
        const Eight<T> now = coming;
        if (i + kStep < whole) __builtin_memcpy(&coming, x + i + kStep, sizeof(coming));
#pragma unroll
        for (int e = 0; e < kPiece; e++) add((float)now[e]);
    }
    if (whole + tid < vocab) add((float)x[whole + tid]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t low = (uint64_t)__shfl_xor((unsigned long long)sum, d, 64), upper = (uint64_t)__shfl_xor((unsigned long long)high, d, 64);
        plus(low, upper);
    }
    __syncthreads();
    if ((tid & 63) == 0) lds_sums[2 * (tid >> 6)] = sum, lds_sums[2 * (tid >> 6) + 1] = high;
    __syncthreads();
    sum = high = 0;
    for (int y = 0; y < kWaves; y++) plus(lds_sums[2 * y], lds_sums[2 * y + 1]);
    return log(ldexp((double)high, 64 - kShift) + ldexp((double)sum, -kShift));
}

struct JoinLds {
    double c[kJoinList];
    int2 at[kJoinList];   // place, beam
    double log_sum[kBeamMaxBeams], score[kBeamMaxBeams], err[kBeamMaxBeams], best_c[kWaves];
    uint64_t sums[2 * kWaves];
    float max[kBeamMaxBeams], ref[kBeamMaxBeams];   // the largest value; what the sum is against
    int kind[kBeamMaxBeams], ended[kBeamMaxBeams];   // kind 0: goes on, 1: stays at the token of the ended, 2: has no candidates but of -inf
    int part[kJoinParts], parts;
    int again[kBeamMaxBeams], any, count, best_place[kWaves], best_beam[kWaves];
    uint32_t bound[kWaves];
    double cut;   // the last value chosen
    int above;    // how many are larger, where they were chosen one after the other
};

// A kernel's one argument where it lies, as loads from here on: kept from the beginning, what only the end looks at would leave too few scalar
// registers for what is between.
template <typename Args>
__device__ __forceinline__ const __attribute__((address_space(4))) Args &arguments_again() {
    auto at = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
    asm volatile("" : "+s"(at));
    return *reinterpret_cast<const __attribute__((address_space(4))) Args *>(at);
}

__device__ __forceinline__ void put_chosen(const __attribute__((address_space(4))) SelectDev &p, int request, const JoinLds &lds, int rank, double c, int place, int beam) {
    const int token = place - beam * p.vocab;
    const int64_t at = (int64_t)request * p.keep + rank;
    p.scores_out[at] = (float)c;
    p.parents[at] = p.row0 + request * p.beams + beam;
    p.tokens[at] = token;
    if (p.ended_out) p.ended_out[at] = token == p.eos || lds.ended[beam];
}

// Whether 64 bits may hold one c for logits of a beam that differ: the logit below x is x 2^-25 or more away (f16's 2^-24 at least), and the three
// roundings of c are 2^-50 of the sizes that it is made of, so only logits that are next to nothing beside those can do that.
template <typename T>
__device__ __forceinline__ bool one_for_several(const JoinLds &lds, int beam, double c) {
    const double score = lds.score[beam], ref = lds.ref[beam], log_sum = lds.log_sum[beam], x = ((c - score) + log_sum) + ref;
    const bool next_to_nothing = !(fabs(x) > 0x1p-24 * (fabs(score) + fabs(x) + fabs(ref) + fabs(log_sum)));
    return next_to_nothing & (lds.kind[beam] == 0) & (c > -INFINITY) & (sizeof(T) == 4 || fabs(score) >= 0x1p23);   // (no branches: all loads at once)
}

// Values that equal the last one chosen go by their places, and of those a part holds the ones of its largest logits alone: where one value may stand
// for several logits, all of them have to be looked at, with exact sums.  A wave's lanes.
template <typename T>
__device__ __forceinline__ bool more_may_equal(const __attribute__((address_space(4))) SelectDev &p, const JoinLds &lds) {
    const int lane = threadIdx.x & 63;
    return __builtin_amdgcn_ballot_w64(one_for_several<T>(lds, lane, lds.cut) & (lane < p.beams)) != 0;
}

// A wave looks for all that equal the last one chosen, in the order of their places, for the ranks behind those of larger values.
template <typename T>
__device__ __forceinline__ void choose_equal(const __attribute__((address_space(4))) SelectDev &p, int request, const JoinLds &lds) {
    constexpr int kLook = 8;
    const int lane = threadIdx.x & 63;
    const double cut = lds.cut;
    int rank = 0;
    if (lds.count > kJoinList) rank = lds.above;
    else
        for (int o = 0; o < lds.count; o++) rank += lds.c[o] > cut ? 1 : 0;
    for (int beam = 0; beam < p.beams && rank < p.keep; beam++) {
        const int kind = lds.kind[beam];
        const double score = lds.score[beam], ref = lds.ref[beam], log_sum = lds.log_sum[beam];
        if (kind == 1 && score == cut) {
            if (lane == 0) put_chosen(p, request, lds, rank, cut, beam * p.vocab + p.eos, beam);
            rank++;
        }
        if (kind != 0) continue;
        const T *row = reinterpret_cast<const T *>(p.logits + ((int64_t)request * p.beams + beam) * p.row_bytes);
        for (int i0 = lane; i0 - lane < p.vocab && rank < p.keep; i0 += kLook * 64) {
            uint32_t is = 0;
#pragma unroll
            for (int e = 0; e < kLook; e++) {
                const int i = i0 + e * 64;
                is |= i < p.vocab && score + (((double)(float)row[min(i, p.vocab - 1)] - ref) - log_sum) == cut ? 1u << e : 0u;
            }
#pragma unroll 1
            for (int e = 0; __builtin_amdgcn_ballot_w64(is >> e) != 0; e++) {
                const uint64_t lanes = __builtin_amdgcn_ballot_w64((is >> e) & 1);
                const int at = rank + lanes_below(lanes);
                if (((is >> e) & 1) && at < p.keep) put_chosen(p, request, lds, at, cut, beam * p.vocab + i0 + e * 64, beam);
                rank += __popcll(lanes);
            }
        }
    }
}

// What is chosen, best first.  EXACT: behind a join, with exact sums for all beams.
template <typename T, bool EXACT>
__device__ __forceinline__ void join_request(const __attribute__((address_space(4))) SelectDev &p, int request, JoinLds &lds) {
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const int per_row = p.parts * p.keep, n = p.beams * per_row;
    const Candidate *all = p.part_best + (int64_t)request * n;
    // What a thread asks for ahead of all, and keeps: candidates, or, where those are more, the best one of every part; of those parts that reach
    // the bound the others are looked at later (8 beams of 128256, f16, in 63 parts each of which 16 are kept: 21.5 us, 48.5 with all 8064 looked
    // at twice).
    constexpr int kHeld = 2;
    const bool few = n <= kHeld * kThreads;
    // (the argument is read again wherever it is looked at: kept, it takes scalar registers that are not there)
    auto beam_of = [](const __attribute__((address_space(4))) SelectDev &p, int j) { return FastDiv{p.by_row_candidates.d, p.by_row_candidates.mul, p.by_row_candidates.shift}.by(j); };
    Candidate first_of[kHeld];
    int held_beam[kHeld], held_k[kHeld];   // beam < 0: none
#pragma unroll
    for (int y = 0; y < kHeld; y++) {
        const int i = tid + y * kThreads, j = i * (few ? 1 : p.keep);
        first_of[y] = j < n ? get(all + j) : Candidate{-INFINITY, -1};
        held_beam[y] = j < n ? beam_of(p, j) : -1, held_k[y] = j - held_beam[y] * per_row;
    }
    constexpr int kLanes = 16;   // of a beam
    for (int beam = EXACT ? p.beams : tid / kLanes; beam < p.beams; beam += kThreads / kLanes) {
        const int64_t row = (int64_t)request * p.beams + beam;
        const float *pm = p.part_max + row * p.parts;
        const double *ps = p.part_sum + row * p.parts;
        const Candidate *first = all + beam * per_row;     // of every part its best
        const float score = p.scores[row];
        const bool ended = p.ended && p.ended[row] != 0;
        // (the largest reference, the largest value, how far one is above its part's reference; sums against the largest so far)
        float m = -INFINITY, top = -INFINITY, over = 0.0f;
        double l = 0.0;
        for (int i = tid % kLanes; i < p.parts; i += kLanes) {
            const float ref = get(pm + i), most = get(first + i * (int64_t)p.keep).x;
            const double sum = get(ps + i);
            top = fmaxf(top, most), over = fmaxf(over, most - ref);   // (NaN where both are infinite: no number)
            if (l == 0.0) {
                l = ref == -INFINITY ? 0.0 : sum, m = ref;
            } else if (ref != -INFINITY) {
                const double step = exp(-fabs((double)ref - (double)m));
                l = ref > m ? l * step + sum : l + sum * step;
                m = fmaxf(m, ref);
            }
        }
        const float mine = m;
        m = row_most(m), top = row_most(top), over = row_most(over);
        l = row_sum(mine == -INFINITY ? 0.0 : l * exp((double)mine - (double)m));
        if (tid % kLanes == 0) {
            const bool dead = !(fabsf(score) < INFINITY);
            const double log_l = log(l);
            lds.score[beam] = dead ? -INFINITY : (double)score;
            lds.log_sum[beam] = log_l, lds.ref[beam] = m;
            lds.max[beam] = top;
            lds.ended[beam] = ended;
            lds.kind[beam] = dead ? 2 : ended ? 1 : !(fabsf(m) < INFINITY) ? 2 : 0;
            // What the sum may be off by, relatively, is what its logarithm is: exponents x - ref by a half step of f32, f32's by one more for the
            // product, and a quarter for log2 e, weighted by the weights at most ln vocab - ln l of them (their entropy is ref - x + ln l on
            // average) and twice what lies above the reference, which is at most `over` and what a wave's may be below its part's, 2; the
            // exponential's two, a piece's seven additions; f64 from there on.  (ln vocab is at most 0.6932 times the bits of it.)  The
            // reference's own weight is 1, so the sum is no less, and no c is NaN: ranks by comparison are a permutation.  c's own three roundings,
            // which a sum that is off may turn the other way, are of 2^-50 of the score and of c at most (c's where it is looked at).
            lds.err[beam] = lds.kind[beam] == 0 ? ((sizeof(T) == 2 ? 1.5 : 2.5) * (fmax(0.6932 * (32 - __clz(p.vocab)) - log_l, 0.0) + 2.0 * over + 4.0) + 10.0) * 0x1p-24 + 0x1p-50 * fabs((double)score) : 0.0;
            lds.again[beam] = 0;
        }
    }
    if (tid == 0) lds.any = 0;
    __syncthreads();

    auto choice = [&](int beam, int k, const Candidate &c) {   // k: which one of the beam
        Choice r = {-INFINITY, -1, beam};
        if (lds.kind[beam] == 0) {
            if (c.token >= 0) r.c = lds.score[beam] + (((double)c.x - (double)lds.ref[beam]) - lds.log_sum[beam]), r.place = beam * p.vocab + c.token;
        } else if (k < p.keep) {   // the token that an ended beam stays at, and then, as in a beam without values, tokens in their order
            const bool stays = lds.kind[beam] == 1 && k == 0;
            const int token = lds.kind[beam] == 1 ? (stays ? p.eos : k - 1 < p.eos ? k - 1 : k) : k;
            if (stays) r.c = lds.score[beam];
            if (token < p.vocab) r.place = beam * p.vocab + token;
        }
        return r;
    };
    auto candidate = [&](int j) {
        const auto &p = arguments_again<SelectDev>();
        const int beam = beam_of(p, j);
        return choice(beam, j - beam * (p.parts * p.keep), get(p.part_best + (int64_t)request * (p.beams * p.parts * p.keep) + j));
    };
    auto chosen = [&](int rank, double c, int place, int beam) { put_chosen(arguments_again<SelectDev>(), request, lds, rank, c, place, beam); };
    auto make_exact = [&](int which) {   // the sums of the beams that are marked so
        for (int beam = 0; beam < p.beams; beam++)
            if (lds.again[beam] == which && lds.kind[beam] == 0) {
                const auto &p = arguments_again<SelectDev>();
                const double log_sum = exact_log_sum(reinterpret_cast<const T *>(p.logits + ((int64_t)request * p.beams + beam) * p.row_bytes), p.vocab, lds.max[beam], lds.sums);
                if (tid == 0) lds.log_sum[beam] = log_sum, lds.ref[beam] = lds.max[beam], lds.again[beam] = 1;
            }
        __syncthreads();
    };
    if constexpr (EXACT) make_exact(0);
    double err = 0.0;
    for (int beam = 0; beam < p.beams; beam++) err = fmax(err, lds.err[beam]);
    for (int again = EXACT;; again++) {
        // at least `keep` of a wave's candidates reach its bound (of f32, whose order is that of f64 but for ties), so the largest bound will
        // do; all that could be among the best are listed
        int tid = threadIdx.x;
        asm("" : "+v"(tid));   // (comparisons again: kept, they take scalar registers)
        const int lane = tid & 63;
        Choice held[kHeld];
        uint32_t top = 0;
#pragma unroll
        for (int y = 0; y < kHeld; y++) {
            int beam = held_beam[y], k = held_k[y];
            asm("" : "+v"(beam), "+v"(k));   // (likewise)
            held[y] = beam >= 0 ? choice(beam, k, first_of[y]) : Choice{-INFINITY, -1, 0};
            if (held[y].place >= 0) top = max(top, key_of((float)held[y].c));
        }
        const int bests = few ? 0 : p.beams * p.parts;
        for (int i = tid + kHeld * kThreads; i < bests; i += kThreads) {
            const Choice r = candidate(i * p.keep);
            if (r.place >= 0) top = max(top, key_of((float)r.c));
        }
        const uint32_t wave_bound = bound_of_lanes(top, p.keep);
        __syncthreads();   // (what the last turn has listed is done with)
        if (lane == 0) lds.bound[w] = wave_bound;
        if (tid == 0) lds.count = lds.parts = 0;
        __syncthreads();
        auto bound_of_waves = [&] { return value_of(max(max(max(lds.bound[0], lds.bound[1]), max(lds.bound[2], lds.bound[3])), kLowest)); };
        auto from_of = [&](float b) { return (double)b - 0x1p-23 * fabs((double)b) - 0x1p-149 - 2.0 * err; };   // (-inf stays that)
        float bound = bound_of_waves();
        double from = from_of(bound);
        auto reaches = [&](const Choice &r) { return r.place >= 0 && (r.c >= from || bound == -INFINITY); };
        auto add = [&](const Choice &r) __attribute__((always_inline)) {
            const bool in = reaches(r);
            const uint64_t lanes = __builtin_amdgcn_ballot_w64(in);
            if (lanes) {
                int at = 0;
                if (lane == 0) at = atomicAdd(&lds.count, __popcll(lanes));
                at = __builtin_amdgcn_readfirstlane(at) + lanes_below(lanes);
                if (in && at < kJoinList) lds.c[at] = r.c, lds.at[at] = make_int2(r.place, r.beam);
            }
        };
        if (few) {
#pragma unroll
            for (int y = 0; y < kHeld; y++) add(held[y]);
        } else {
#pragma unroll
            for (int y = 0; y < kHeld; y++)
                if (reaches(held[y])) lds.part[atomicAdd(&lds.parts, 1)] = tid + y * kThreads;
            for (int i = tid + kHeld * kThreads; i < bests; i += kThreads)
                if (reaches(candidate(i * p.keep))) lds.part[atomicAdd(&lds.parts, 1)] = i;
            __syncthreads();
            constexpr int kDeep = 4;
            const auto &p = arguments_again<SelectDev>();
            const FastDiv by_keep = {p.by_keep.d, p.by_keep.mul, p.by_keep.shift};
            const int there = lds.parts * p.keep;
            for (int x0 = 0; x0 < there; x0 += kDeep * kThreads) {
                int j[kDeep];
                Candidate c[kDeep];
#pragma unroll
                for (int y = 0; y < kDeep; y++) {
                    const int x = x0 + y * kThreads + tid, i = by_keep.by(min(x, there - 1));
                    j[y] = x < there ? lds.part[i] * p.keep + x - i * p.keep : -1;
                    c[y] = get(p.part_best + (int64_t)request * (p.beams * p.parts * p.keep) + max(j[y], 0));
                }
                // (best ones alone make a low bound where one beam has most of what is chosen: again, of these)
                Choice r[kDeep];
                uint32_t top = 0;
#pragma unroll
                for (int y = 0; y < kDeep; y++) {
                    const int beam = beam_of(p, max(j[y], 0));
                    r[y] = j[y] >= 0 ? choice(beam, j[y] - beam * (p.parts * p.keep), c[y]) : Choice{-INFINITY, -1, 0};
                    if (r[y].place >= 0) top = max(top, key_of((float)r[y].c));
                }
                const uint32_t wave_bound = bound_of_lanes(top, p.keep);
                if (lane == 0) lds.bound[w] = wave_bound;
                __syncthreads();
                bound = fmaxf(bound, bound_of_waves()), from = from_of(bound);
#pragma unroll
                for (int y = 0; y < kDeep; y++) add(r[y]);
                __syncthreads();
            }
        }
        __syncthreads();
        const int listed = min(lds.count, kJoinList);
        const bool whole = lds.count <= kJoinList;
        // Every listed value counts those before it; a value that is nearer to another beam's than sums of 32-bit terms tell apart asks for
        // both beams' sums to be made again.  Equal values are common (f16: steps of 2^-7 at 10): up to two near ones are looked at without
        // another pass over the list (32 x 8 beams of 128256 32.8 us with one, 30.6 without).
        constexpr int kMine = kJoinList / kThreads;
        int rank[kMine];
#pragma unroll
        for (int y = 0; y < kMine; y++) {
            const int j = tid + y * kThreads;
            rank[y] = p.keep;
            if (!whole || j >= listed) continue;
            const double c = lds.c[j], own = c > -INFINITY ? 0x1p-50 * fabs(c) : 0.0;
            int r = 0, near = 0, one = j, two = j;   // near: others; the last two of them
#pragma unroll 4
            for (int o = 0; o < listed; o++) {
                const double d = lds.c[o];
                const bool is_near = !(fabs(d - c) > 2.0 * err + own) && o != j;   // (two of -inf are)
                r += d > c ? 1 : 0;
                near += is_near ? 1 : 0;
                two = is_near ? one : two, one = is_near ? o : one;
            }
            if (near > 0 && r < p.keep) {
                const int2 mine = lds.at[j];
                auto look = [&](int o) {
                    const int2 other = lds.at[o];
                    const double d = lds.c[o], off = lds.err[mine.y] + lds.err[other.y];
                    r += d == c && other.x < mine.x ? 1 : 0;
                    if (again == 0 && off > 0.0 && fabs(d - c) <= off + own && (other.y != mine.y || (o != j && one_for_several<T>(lds, mine.y, c)))) lds.again[mine.y] = lds.again[other.y] = 1, lds.any = 1;
                };
                if (near <= 2) {   // (itself in place of one that is not there)
                    look(one), look(two);
                } else {
                    for (int o = 0; o < listed; o++) look(o);
                }
            }
            rank[y] = r;
        }
        if (!whole) {
            if (tid < p.beams) lds.again[tid] = 1;
            if (tid == 0) lds.any = 1;
        }
#pragma unroll
        for (int y = 0; y < kMine; y++)
            if (rank[y] == p.keep - 1) lds.cut = lds.c[tid + y * kThreads];
        __syncthreads();
        if (!EXACT && again == 0 && lds.any) {
            make_exact(1);
            continue;
        }
        if (!whole) break;
#pragma unroll
        for (int y = 0; y < kMine; y++)
            if (rank[y] < p.keep) {
                const int2 at = lds.at[tid + y * kThreads];
                chosen(rank[y], lds.c[tid + y * kThreads], at.x, at.y);
            }
        return;
    }
    // more than the list holds (equal values above all): one after the other
    const auto &q = arguments_again<SelectDev>();
    const int all_there = q.beams * q.parts * q.keep;
    double last_c = INFINITY;
    int last_place = -1;
    for (int rank = 0; rank < q.keep; rank++) {
        Choice best = {-INFINITY, -1, 0};
        for (int j = tid; j < all_there; j += kThreads) {
            const Choice r = candidate(j);
            if (r.place >= 0 && before(last_c, last_place, r.c, r.place) && (best.place < 0 || before(r.c, r.place, best.c, best.place))) best = r;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double c = __shfl_xor(best.c, d, 64);
            const int place = __shfl_xor(best.place, d, 64), beam = __shfl_xor(best.beam, d, 64);
            if (place >= 0 && (best.place < 0 || before(c, place, best.c, best.place))) best = {c, place, beam};
        }
        if (lane == 0) lds.best_c[w] = best.c, lds.best_place[w] = best.place, lds.best_beam[w] = best.beam;
        __syncthreads();
        best = {-INFINITY, -1, 0};
        for (int y = 0; y < kWaves; y++)
            if (lds.best_place[y] >= 0 && (best.place < 0 || before(lds.best_c[y], lds.best_place[y], best.c, best.place))) best = {lds.best_c[y], lds.best_place[y], lds.best_beam[y]};
        if (tid == 0 && best.place >= 0) chosen(rank, best.c, best.place, best.beam);
        if (tid == 0 && best.c < last_c) lds.above = rank;
        last_c = best.c, last_place = best.place;
        if (tid == 0) lds.cut = last_c;
        __syncthreads();
    }
}

template <typename T, int C>
__global__ __launch_bounds__(kThreads, 4) void beam_select_kernel(SelectDev p) {
    __shared__ union Lds { ScanLds scan; JoinLds join; __device__ Lds() {} } lds;
    __shared__ int s_last;
    const int row = p.by_parts.by(blockIdx.x), part = blockIdx.x - row * p.parts, request = p.by_beams.by(row);
    scan_part<T, C>(p, row, part, lds.scan);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // what this thread leaves has completed
    __syncthreads();                                     // ... and what the whole workgroup does
    if (threadIdx.x == 0) {
        s_last = __hip_atomic_fetch_add(p.counters + request, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == p.parts * p.beams - 1;
        if (s_last) __hip_atomic_store(p.counters + request, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!s_last) return;
    join_request<T, false>(arguments_again<SelectDev>(), request, lds.join);
    if (!more_may_equal<T>(arguments_again<SelectDev>(), lds.join)) return;
    const int beam = threadIdx.x & 63;
    const bool inexact = __builtin_amdgcn_ballot_w64(beam < arguments_again<SelectDev>().beams && lds.join.kind[beam] == 0 && !lds.join.again[beam]) != 0;
    __syncthreads();   // (all have been put where they go)
    if (inexact) {
        join_request<T, true>(arguments_again<SelectDev>(), request, lds.join);
        if (!more_may_equal<T>(arguments_again<SelectDev>(), lds.join)) return;
        __syncthreads();
    }
    const auto &q = arguments_again<SelectDev>();
    if (threadIdx.x < 64) choose_equal<T>(q, FastDiv{q.by_beams.d, q.by_beams.mul, q.by_beams.shift}.by(FastDiv{q.by_parts.d, q.by_parts.mul, q.by_parts.shift}.by(blockIdx.x)), lds.join);
}

// How rows are cut into parts: tiles of 4 pieces of 8 values a thread, or of 1 where there are fewer than an eighth as many tiles as compute
// units (us of 1 and 4 pieces: 1 x 4 rows of 32000 in 16 tiles 10.2, 10.9; 8 x 3 of 5000 in 24 10.2, 11.4; 3 x 4 of 32000 in 48 13.0, 11.5; 1 x 8 of
// 128256 in 128, 16 kept, 22.3, 18.0); and as many tiles one after the other as leave each compute unit kPerUnit workgroups.  (Three for each
// run at once with what they hold, so nothing waits for a second round; us with 2, 3 and 4: 32 x 8 rows of 128256, f16 32.5, 30.7, 34.2 and f32
// 33.9, 34.9, 37.5; 64 x 4 of 32000, f16 16.2, 16.2, 18.1.  Parts of the same length end their streams at the same time: 34.2 for 33.0.)
constexpr int kPerUnit = 3;
struct Cut { int pieces; int64_t parts, turns; };
Cut cut_of(int64_t batch, int64_t beams, int64_t vocab) {
    const int64_t rows = batch * beams;
    Cut c;
    auto tiles = [&](int pieces) { return (vocab + kThreads * kPiece * pieces - 1) / (kThreads * kPiece * pieces); };
    c.pieces = 8 * rows * tiles(4) >= num_compute_units() ? 4 : 1;
    const int64_t all = tiles(c.pieces);
    c.parts = std::min(all, std::max<int64_t>(1, ((int64_t)kPerUnit * num_compute_units() + rows - 1) / rows));
    c.parts = std::min(c.parts, kJoinParts / beams);
    c.turns = (all + c.parts - 1) / c.parts;
    c.parts = (all + c.turns - 1) / c.turns;
    return c;
}

constexpr int64_t kCounters = kWsCounterBytes / 4;   // requests of a launch, at most
size_t bytes_for(int64_t rows, int64_t parts, int64_t keep) { return kWsCounterBytes + (size_t)(rows * parts) * (sizeof(double) + sizeof(float) + sizeof(Candidate) * (size_t)keep); }

}  // namespace

size_t beam_select_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int64_t keep) {
    return bytes_for(batch * beams, cut_of(batch, beams, vocab).parts, keep);
}

int launch_beam_select(const BeamSelectArgs &a, hipStream_t s) {
    if (a.batch == 0) return 0;
    const int64_t rows = a.batch * a.beams, es = (int64_t)elem_bytes(a.dtype);
    const Cut cut = cut_of(a.batch, a.beams, a.vocab);
    TROCM_REQUIRE(a.workspace && a.workspace_bytes >= bytes_for(rows, cut.parts, a.keep), "beam_select: the workspace must hold %zu bytes", bytes_for(rows, cut.parts, a.keep));
    TROCM_REQUIRE(kCounters * a.beams * cut.parts < (1ll << 31) && a.beams * cut.parts * a.keep < (1ll << 31), "beam_select: tensor too large");
    for (int64_t first = 0; first < a.batch; first += kCounters) {
        const int64_t batch = std::min(a.batch - first, kCounters), row0 = first * a.beams;
        SelectDev p;
        p.logits = (const char *)a.logits + row0 * a.row_stride * es, p.row_bytes = a.row_stride * es;
        p.vocab = (int)a.vocab, p.parts = (int)cut.parts, p.turns = (int)cut.turns, p.keep = (int)a.keep, p.beams = (int)a.beams, p.eos = a.eos;
        p.counters = (int *)a.workspace;
        p.part_sum = (double *)((char *)a.workspace + kWsCounterBytes);
        p.part_best = (Candidate *)(p.part_sum + rows * cut.parts);
        p.part_max = (float *)(p.part_best + rows * cut.parts * a.keep);
        p.scores = a.scores + row0, p.ended = a.ended ? a.ended + row0 : nullptr;
        p.scores_out = a.scores_out + first * a.keep, p.parents = a.parents + first * a.keep, p.tokens = a.tokens + first * a.keep;
        p.ended_out = a.ended_out ? a.ended_out + first * a.keep : nullptr;
        p.row0 = (int)row0;
        p.by_parts = fast_div(cut.parts), p.by_row_candidates = fast_div(cut.parts * a.keep), p.by_keep = fast_div(a.keep), p.by_beams = fast_div(a.beams);
        const dim3 grid((unsigned)(batch * a.beams * cut.parts));
        if (a.dtype == TROCM_F16) {
            if (cut.pieces == 4) beam_select_kernel<_Float16, 4><<<grid, kThreads, 0, s>>>(p);
            else beam_select_kernel<_Float16, 1><<<grid, kThreads, 0, s>>>(p);
        } else {
            if (cut.pieces == 4) beam_select_kernel<float, 4><<<grid, kThreads, 0, s>>>(p);
            else beam_select_kernel<float, 1><<<grid, kThreads, 0, s>>>(p);
        }
        TROCM_HIP(hipGetLastError());
    }
    return 0;
}

}  // namespace trocm
