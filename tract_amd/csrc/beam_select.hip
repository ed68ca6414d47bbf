// The best continuations of a request's beams: of all values c = score + x - log sum exp(x) over beams and vocabulary the `keep` largest,
// ties to the lowest (beam, token).
//
// Within a beam the order of c is the order of the logits, which is exact; only between beams does c itself count.  So the vocabulary is
// read once: a workgroup holds a part of a row in registers, makes its maximum and sum (f32 for eight values, then f64) and keeps its `keep`
// largest logits; a second launch puts the parts together in f64, one workgroup per request.  Where values of two beams are nearer than those
// sums can be told apart, the beams' sums are made again, exactly.
//
// The largest of a wave's values: the K-th largest of the 64 lanes' maxima is found by bisection over the bits of an order-preserving
// integer (a ballot and a count per bit); at least K values are not below it, and few more than that, which are compacted into LDS and
// ranked by counting.  Where more values than the list holds pass, the bisection is over all values instead of the lanes' maxima.
#include <hip/hip_fp16.h>
#include <math.h>
#include <algorithm>
#include <type_traits>
#include "common.h"
#include "fast_div.h"

namespace trocm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kPiece = 8;                     // consecutive values of a lane
constexpr int kWaveList = 512;                // values that a wave lists
constexpr uint32_t kLowest = 0x007fffffu;     // key_of(-inf); 0 is below all values: nothing there

struct Candidate { float x; int token; };     // token < 0: none

struct SelectDev {
    const char *logits;
    int64_t row_bytes;
    int vocab, parts, keep, beams, eos;
    float *part_max;
    double *part_sum;
    Candidate *part_best;       // [row][part][keep], best first
    const float *scores;
    const int *ended;
    float *scores_out;
    int *parents, *tokens, *ended_out;
    FastDiv by_parts, by_row_candidates;
};

// Integers in the order of the numbers; both zeros are one number and NaN counts as -inf.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    const uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return x != x ? kLowest : k;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __builtin_bit_cast(float, k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }

__device__ __forceinline__ int lanes_below(uint64_t mask) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0)); }

// The largest t that at least `count` of the wave's keys (one per lane) reach; 0 if there are fewer.
__device__ __forceinline__ uint32_t bound_of_lanes(uint32_t key, int count) {
    uint32_t t = 0;
#pragma unroll 1
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
        if (__popcll(__builtin_amdgcn_ballot_w64(key >= (t | bit))) >= count) t |= bit;
    return t;
}

template <typename T> using Eight = T __attribute__((ext_vector_type(kPiece)));

// A part of a row: kThreads * kPiece * C values, all of them asked for before the first is looked at.
template <typename T, int C>
__global__ __launch_bounds__(kThreads) void beam_scan_kernel(SelectDev p) {
    constexpr int kPart = kThreads * kPiece * C, kStep = kThreads * kPiece, kAtOnce = C < 4 ? C : 4;
    __shared__ int s_list[kWaves * kWaveList];        // tokens
    __shared__ Candidate s_all[kWaves * kWaveList];
    __shared__ int s_total;
    __shared__ uint32_t s_bound[kWaves];
    __shared__ float s_max[kWaves];
    __shared__ double s_sum[kWaves];
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const int row = p.by_parts.by(blockIdx.x), part = blockIdx.x - row * p.parts;
    const T *from = reinterpret_cast<const T *>(p.logits + row * p.row_bytes);
    const int i0 = part * kPart + tid * kPiece;
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
    Eight<T> x[C];
    if (part * kPart <= p.vocab - kPart) {
#pragma unroll
        for (int c = 0; c < C; c++) __builtin_memcpy(&x[c], from + i0 + c * kStep, sizeof(x[c]));
    } else {
#pragma unroll
        for (int c = 0; c < C; c++) x[c] = piece_at(i0 + c * kStep);
    }
    // (Each look at the values begins with what was loaded: kept in 32 bits from one look to the next, halves would take twice the registers.)
    auto again = [&](int c) __attribute__((always_inline)) { asm("" : "+v"(x[c])); };
    T most[C];   // of a piece; NaN only where all are
    T top_t = (T)-INFINITY;
#pragma unroll
    for (int c = 0; c < C; c++) {
        auto v4 = __builtin_elementwise_max(__builtin_shufflevector(x[c], x[c], 0, 1, 2, 3), __builtin_shufflevector(x[c], x[c], 4, 5, 6, 7));
        auto v2 = __builtin_elementwise_max(__builtin_shufflevector(v4, v4, 0, 1), __builtin_shufflevector(v4, v4, 2, 3));
        most[c] = __builtin_elementwise_max(v2[0], v2[1]);
        top_t = __builtin_elementwise_max(top_t, most[c]);
    }
    const float top = (float)top_t;

    // at least `keep` values of a wave reach its bound, so the largest bound will do for the workgroup
    const uint32_t wave_bound = max(bound_of_lanes(key_of(top), p.keep), kLowest);
    float m = top;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    if (lane == 0) s_bound[w] = wave_bound;
    if (tid == 0) s_total = 0;

    // Maximum and sum: f32 for the values of a piece, f64 from there on.  A weight is 2^(x a - c) in one step, a = log2 e as f32 has it, c = m a
    // rounded; what c is off by is put right at the end, what a is off by counts for x - m alone (beam_join_kernel's s_err has both).
    const float c_m = m == -INFINITY ? 0.0f : m * kLog2e;
    double all = 0.0;
#pragma unroll
    for (int c = 0; c < C; c++) {
        again(c);
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < kPiece; e++) sum += __builtin_amdgcn_exp2f(__builtin_fmaf((float)x[c][e], kLog2e, -c_m));
        all += (double)sum;
    }
    if (__builtin_amdgcn_ballot_w64(all != all)) {   // a NaN counts as -inf
        all = 0.0;
#pragma unroll 1
        for (int i = i0; i < min(part * kPart + kPart, p.vocab); i += kStep) {
            const Eight<T> v = piece_at(i);
#pragma unroll
            for (int e = 0; e < kPiece; e++) {
                const float t = __builtin_amdgcn_exp2f(__builtin_fmaf((float)v[e], kLog2e, -c_m));
                all += t == t ? (double)t : 0.0;
            }
        }
    }
    if (m != -INFINITY) all += all * (((double)c_m - (double)m * (double)kLog2e) * 0.6931471805599453);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) all += __shfl_xor(all, d, 64);
    if (lane == 0) s_max[w] = m, s_sum[w] = all;
    __syncthreads();

    // the values that reach the bound
    const float least = value_of(max(max(s_bound[0], s_bound[1]), max(s_bound[2], s_bound[3])));
    int *list = s_list + w * kWaveList;
    int n = 0;
    auto list_four = [&](auto first) __attribute__((always_inline)) {   // pieces first .. of kAtOnce
        constexpr int c0 = decltype(first)::value;
        uint32_t hits = 0;   // bit 8 c + e
#pragma unroll
        for (int c = 0; c < kAtOnce; c++) {
            if (__builtin_amdgcn_ballot_w64((float)most[c0 + c] >= least)) {
                again(c0 + c);
#pragma unroll
                for (int e = 0; e < kPiece; e++) hits |= x[c0 + c][e] >= (T)least ? 1u << (c * kPiece + e) : 0u;
            }
        }
        while (const uint64_t in = __builtin_amdgcn_ballot_w64(hits != 0)) {
            const int b = __ffs(hits) - 1, at = n + lanes_below(in);
            if (hits && at < kWaveList) list[at] = i0 + (c0 + b / kPiece) * kStep + b % kPiece;
            hits &= hits - 1;
            n += __popcll(in);
        }
    };
    if (__builtin_amdgcn_ballot_w64(!(top < least))) {   // (a lane of NaN too: they tie at -inf)
        list_four(std::integral_constant<int, 0>{});
        if constexpr (C > 4) list_four(std::integral_constant<int, 4>{});
        if constexpr (C > 8) list_four(std::integral_constant<int, 8>{}), list_four(std::integral_constant<int, 12>{});
    }
    // -inf is the bound of waves that have little else, and what lies behind the row's end has it too; and where more values reach the
    // bound than the list holds, equal ones above all, only so many of them are wanted as could be among the best: both in the values' order,
    // pieces, lanes, values of a piece.
    if (n > kWaveList || (least == -INFINITY && __builtin_amdgcn_ballot_w64(!(top < least)))) {
        uint32_t bound_key = key_of(least);
        int above = 0;
        auto count = [&](float reach) __attribute__((always_inline)) {
            int k = 0;
#pragma unroll
            for (int c = 0; c < C; c++) {
                again(c);
#pragma unroll
                for (int e = 0; e < kPiece; e++) k += __popcll(__builtin_amdgcn_ballot_w64((float)x[c][e] >= reach));
            }
            return k;
        };
        if (__builtin_amdgcn_ballot_w64(top > least)) above = count(value_of(bound_key + 1));
        if (above > kWaveList - kBeamMaxKeep) {   // the bound of all values, above which there are fewer than `keep`
            bound_key = 0;
#pragma unroll 1
            for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
                if ((bound_key | bit) <= kLowest || ((bound_key | bit) <= 0xff800000u && count(value_of(bound_key | bit)) >= p.keep)) bound_key |= bit;
            bound_key = max(bound_key, kLowest);
            above = kWaveList;
        }
        const float bound = value_of(bound_key);
        n = 0;
        int equal = 0;
#pragma unroll 1
        for (int c = 0; c < C && (above > 0 || equal < p.keep); c++) {
            const int i = i0 + c * kStep;
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
            const int mine = __popc(ties);
            int before = equal, here = 0;
#pragma unroll
            for (int bit = 0; bit < 4; bit++) {
                const uint64_t lanes = __builtin_amdgcn_ballot_w64((mine >> bit) & 1);
                before += lanes_below(lanes) << bit, here += __popcll(lanes) << bit;
            }
            for (int at = n + before - equal; ties && before < p.keep; ties &= ties - 1, at++, before++) list[at] = i + __ffs(ties) - 1;
            n += min(here, p.keep - equal), equal = min(equal + here, p.keep);
        }
    }

    // the workgroup's: every listed value counts those before it
    for (int j0 = 0; j0 < n; j0 += 64) {
        Candidate c = {-INFINITY, -1};
        if (j0 + lane < n) {
            c.token = list[j0 + lane];
            const float v = (float)from[c.token];
            c.x = v == v ? v : -INFINITY;
        }
        const uint64_t lanes = __builtin_amdgcn_ballot_w64(c.token >= 0);
        int at = 0;
        if (lane == 0) at = atomicAdd(&s_total, __popcll(lanes));
        at = __builtin_amdgcn_readfirstlane(at) + lanes_below(lanes);
        if (c.token >= 0) s_all[at] = c;
    }
    __syncthreads();
    const int total = s_total;
    Candidate *best = p.part_best + (int64_t)blockIdx.x * p.keep;
    for (int j = tid; j < total; j += kThreads) {
        const Candidate c = s_all[j];
        int rank = 0;
#pragma unroll 4
        for (int z = 0; z < total; z++) {
            const Candidate d = s_all[z];
            rank += d.x > c.x || (d.x == c.x && d.token < c.token);
        }
        if (rank < p.keep) best[rank] = c;
    }
    for (int j = total + tid; j < p.keep; j += kThreads) best[j] = Candidate{-INFINITY, -1};
    if (tid == 0) {
        float mm = s_max[0];
        for (int y = 1; y < kWaves; y++) mm = fmaxf(mm, s_max[y]);
        double l = 0.0;
        for (int y = 0; y < kWaves; y++) l += s_max[y] == -INFINITY ? 0.0 : s_sum[y] * exp((double)s_max[y] - (double)mm);
        p.part_max[blockIdx.x] = mm, p.part_sum[blockIdx.x] = l;
    }
}

// ---- parts and beams put together: a workgroup per request ------------------------------------------------------------------

constexpr int kJoinList = 1024;
struct Choice { double c; int place, beam; };   // place: beam * vocab + token (below 2^31, checked by the host); < 0: none

__device__ __forceinline__ bool before(double c, int place, double d, int other) { return c > d || (c == d && place < other); }

// log sum exp of a row whose largest value is m, the same for the same values in any order: terms of 64 bits, rounded to whole multiples of
// 2^-shift of the largest and added as integers.  All threads; only where two beams are nearer than their 32-bit sums tell apart (about
// one launch in twenty of 32 requests of 8 beams over 128256 tokens).
template <typename T>
__device__ __forceinline__ double exact_lse(const T *x, int vocab, float m, uint64_t *lds_sums) {
    const int shift = 61 - (32 - __clz(vocab)), tid = threadIdx.x;
    uint64_t sum = 0;
#pragma unroll 8
    for (int i = tid; i < vocab; i += kThreads) {
        const float v = (float)x[i];
        sum += v == v ? (uint64_t)(ldexp(exp((double)v - (double)m), shift) + 0.5) : 0;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += (uint64_t)__shfl_xor((unsigned long long)sum, d, 64);
    __syncthreads();
    if ((tid & 63) == 0) lds_sums[tid >> 6] = sum;
    __syncthreads();
    sum = 0;
    for (int y = 0; y < kWaves; y++) sum += lds_sums[y];
    return (double)m + log(ldexp((double)sum, -shift));
}

template <typename T>
__global__ __launch_bounds__(kThreads) void beam_join_kernel(SelectDev p) {
    __shared__ double s_lse[kBeamMaxBeams], s_score[kBeamMaxBeams], s_err[kBeamMaxBeams];
    __shared__ float s_max[kBeamMaxBeams];
    __shared__ int s_kind[kBeamMaxBeams], s_ended[kBeamMaxBeams];   // kind 0: goes on, 1: stays at the token of the ended, 2: has no candidates but of -inf
    __shared__ int s_again[kBeamMaxBeams], s_any;
    __shared__ Choice s_list[kJoinList];
    __shared__ double s_best_c[kWaves];
    __shared__ int s_count, s_best_place[kWaves], s_best_beam[kWaves];
    __shared__ uint64_t s_sums[kWaves];
    __shared__ uint32_t s_bound[kWaves];
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, request = blockIdx.x;
    constexpr int kLanes = 16;   // of a beam
    for (int beam = tid / kLanes; beam < p.beams; beam += kThreads / kLanes) {
        const int64_t row = (int64_t)request * p.beams + beam;
        const float *pm = p.part_max + row * p.parts;
        const double *ps = p.part_sum + row * p.parts;
        float m = -INFINITY;
        for (int i = tid % kLanes; i < p.parts; i += kLanes) m = fmaxf(m, pm[i]);
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
        double l = 0.0;
        for (int i = tid % kLanes; i < p.parts; i += kLanes) l += pm[i] == -INFINITY ? 0.0 : ps[i] * exp((double)pm[i] - (double)m);
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) l += __shfl_xor(l, d, 64);
        if (tid % kLanes == 0) {
            const float score = p.scores[row];
            const bool dead = !(fabsf(score) < INFINITY);
            s_score[beam] = dead ? -INFINITY : (double)score;
            s_lse[beam] = (double)m + log(l);
            s_max[beam] = m;
            s_ended[beam] = p.ended && p.ended[row] != 0;
            s_kind[beam] = dead ? 2 : s_ended[beam] ? 1 : !(fabsf(m) < INFINITY) ? 2 : 0;
            // What the sum may be off by, relatively, is what its logarithm is: exponents d by a half step of f32 and a quarter for log2 e, weighted
            // by the weights at most ln(vocab / l) of them (their entropy is d + ln l on average); another for the part's maximum, to which d
            // counts from there; the exponential's two, a piece's seven additions; f64 from there on.
            s_err[beam] = s_kind[beam] == 0 ? (1.5 * fmax(log((double)p.vocab / l), 0.0) + 10.0) * 0x1p-24 : 0.0;
            s_again[beam] = 0;
        }
    }
    if (tid == 0) s_any = 0;
    __syncthreads();

    const int per_row = p.parts * p.keep, n = p.beams * per_row;
    const Candidate *all = p.part_best + (int64_t)request * n;
    auto candidate = [&](int j) {
        const int beam = p.by_row_candidates.by(j), k = j - beam * per_row;
        Choice r = {-INFINITY, -1, beam};
        if (s_kind[beam] == 0) {
            const Candidate c = all[j];
            if (c.token >= 0) r.c = s_score[beam] + ((double)c.x - s_lse[beam]), r.place = beam * p.vocab + c.token;
        } else if (k < p.keep) {   // the token that an ended beam stays at, and then, as in a beam without values, tokens in their order
            const bool stays = s_kind[beam] == 1 && k == 0;
            const int token = s_kind[beam] == 1 ? (stays ? p.eos : k - 1 < p.eos ? k - 1 : k) : k;
            if (stays) r.c = s_score[beam];
            if (token < p.vocab) r.place = beam * p.vocab + token;
        }
        return r;
    };
    auto put = [&](int rank, double c, int place, int beam) {
        const int token = place - beam * p.vocab;
        const int64_t at = (int64_t)request * p.keep + rank;
        p.scores_out[at] = (float)c;
        p.parents[at] = request * p.beams + beam;
        p.tokens[at] = token;
        if (p.ended_out) p.ended_out[at] = token == p.eos || s_ended[beam];
    };
    double err = 0.0;
    for (int beam = 0; beam < p.beams; beam++) err = fmax(err, s_err[beam]);
    for (int again = 0;; again++) {
        // at least `keep` of a wave's candidates reach its bound (of f32, whose order is that of f64 but for ties); all that could be among the
        // best are listed
        uint32_t top = 0;
        for (int j = tid; j < n; j += kThreads) {
            const Choice r = candidate(j);
            if (r.place >= 0) top = max(top, key_of((float)r.c));
        }
        const uint32_t wave_bound = bound_of_lanes(top, p.keep);
        __syncthreads();   // (what the last turn has listed is done with)
        if (lane == 0) s_bound[w] = wave_bound;
        if (tid == 0) s_count = 0;
        __syncthreads();
        const float bound = value_of(max(max(max(s_bound[0], s_bound[1]), max(s_bound[2], s_bound[3])), kLowest));
        const double from = (double)bound - 0x1p-23 * fabs((double)bound) - 0x1p-149 - 2.0 * err;   // (-inf stays that)
        for (int j0 = 0; j0 < n; j0 += kThreads) {
            const int j = j0 + tid;
            Choice r = {-INFINITY, -1, 0};
            if (j < n) r = candidate(j);
            const bool in = r.place >= 0 && (r.c >= from || bound == -INFINITY);
            const uint64_t lanes = __builtin_amdgcn_ballot_w64(in);
            if (lanes) {
                int at = 0;
                if (lane == 0) at = atomicAdd(&s_count, __popcll(lanes));
                at = __builtin_amdgcn_readfirstlane(at) + lanes_below(lanes);
                if (in && at < kJoinList) s_list[at] = r;
            }
        }
        __syncthreads();
        const int listed = min(s_count, kJoinList);
        const bool whole = s_count <= kJoinList;
        // Every listed value counts those before it; a value that is nearer to another beam's than sums of 32-bit terms tell apart asks for
        // both beams' sums to be made again.
        constexpr int kMine = kJoinList / kThreads;
        int rank[kMine];
#pragma unroll
        for (int y = 0; y < kMine; y++) {
            const int j = tid + y * kThreads;
            rank[y] = p.keep;
            if (!whole || j >= listed) continue;
            const Choice c = s_list[j];
            int r = 0, near = 0;
#pragma unroll 4
            for (int o = 0; o < listed; o++) {
                const Choice d = s_list[o];
                r += before(d.c, d.place, c.c, c.place);
                near |= d.beam != c.beam && fabs(d.c - c.c) <= 2.0 * err ? 1 : 0;
            }
            rank[y] = r;
            if (again == 0 && near && r < p.keep) {
                for (int o = 0; o < listed; o++) {
                    const Choice d = s_list[o];
                    const double off = s_err[c.beam] + s_err[d.beam];
                    if (d.beam != c.beam && off > 0.0 && fabs(d.c - c.c) <= off) s_again[c.beam] = s_again[d.beam] = 1, s_any = 1;
                }
            }
        }
        if (again == 0) {
            if (!whole) {
                for (int beam = tid; beam < p.beams; beam += kThreads) s_again[beam] = 1;
                if (tid == 0) s_any = 1;
            }
            __syncthreads();
            if (s_any) {
                for (int beam = 0; beam < p.beams; beam++)
                    if (s_again[beam] && s_kind[beam] == 0) {
                        const double lse = exact_lse(reinterpret_cast<const T *>(p.logits + ((int64_t)request * p.beams + beam) * p.row_bytes), p.vocab, s_max[beam], s_sums);
                        if (tid == 0) s_lse[beam] = lse;
                    }
                __syncthreads();
                continue;
            }
        }
        if (whole) {
#pragma unroll
            for (int y = 0; y < kMine; y++)
                if (rank[y] < p.keep) {
                    const Choice c = s_list[tid + y * kThreads];
                    put(rank[y], c.c, c.place, c.beam);
                }
            return;
        }
        break;
    }
    // more than the list holds (equal values above all): one after the other
    double last_c = INFINITY;
    int last_place = -1;
    for (int rank = 0; rank < p.keep; rank++) {
        Choice best = {-INFINITY, -1, 0};
        for (int j = tid; j < n; j += kThreads) {
            const Choice r = candidate(j);
            if (r.place >= 0 && before(last_c, last_place, r.c, r.place) && (best.place < 0 || before(r.c, r.place, best.c, best.place))) best = r;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double c = __shfl_xor(best.c, d, 64);
            const int place = __shfl_xor(best.place, d, 64), beam = __shfl_xor(best.beam, d, 64);
            if (place >= 0 && (best.place < 0 || before(c, place, best.c, best.place))) best = {c, place, beam};
        }
        if (lane == 0) s_best_c[w] = best.c, s_best_place[w] = best.place, s_best_beam[w] = best.beam;
        __syncthreads();
        best = {-INFINITY, -1, 0};
        for (int y = 0; y < kWaves; y++)
            if (s_best_place[y] >= 0 && (best.place < 0 || before(s_best_c[y], s_best_place[y], best.c, best.place))) best = {s_best_c[y], s_best_place[y], s_best_beam[y]};
        if (tid == 0 && best.place >= 0) put(rank, best.c, best.place, best.beam);
        last_c = best.c, last_place = best.place;
        __syncthreads();
    }
}

// Pieces of 8 values that a thread takes: few where rows are few, so that there are workgroups for the compute units; of at most 256 bytes,
// what its registers hold.
int pieces_of(int64_t rows, int64_t vocab, int dtype) {
    for (int c = dtype == TROCM_F16 ? 16 : 8; c > 1; c /= 4)
        if (rows * ((vocab + kThreads * kPiece * c - 1) / (kThreads * kPiece * c)) >= 2 * num_compute_units()) return c;
    return dtype == TROCM_F16 ? 1 : 2;
}

size_t bytes_for(int64_t rows, int64_t parts, int64_t keep) { return (size_t)(rows * parts) * (sizeof(double) + sizeof(float) + sizeof(Candidate) * (size_t)keep) + 64; }

}  // namespace

size_t beam_select_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int64_t keep) {   // (of either type)
    const int64_t rows = batch * beams;
    size_t most = 0;
    for (int dtype : {TROCM_F16, TROCM_F32}) {
        const int64_t part = (int64_t)kThreads * kPiece * pieces_of(rows, vocab, dtype);
        most = std::max(most, bytes_for(rows, (vocab + part - 1) / part, keep));
    }
    return most;
}

int launch_beam_select(const BeamSelectArgs &a, hipStream_t s) {
    if (a.batch == 0) return 0;
    const int pieces = pieces_of(a.batch * a.beams, a.vocab, a.dtype);
    const int64_t rows = a.batch * a.beams, part = (int64_t)kThreads * kPiece * pieces, parts = (a.vocab + part - 1) / part;
    TROCM_REQUIRE(a.workspace && a.workspace_bytes >= bytes_for(rows, parts, a.keep), "beam_select: the workspace must hold %zu bytes", bytes_for(rows, parts, a.keep));
    TROCM_REQUIRE(rows * parts < (1ll << 31) && a.beams * parts * a.keep < (1ll << 31), "beam_select: tensor too large");
    SelectDev p;
    p.logits = (const char *)a.logits, p.row_bytes = a.row_stride * (int64_t)elem_bytes(a.dtype);
    p.vocab = (int)a.vocab, p.parts = (int)parts, p.keep = (int)a.keep, p.beams = (int)a.beams, p.eos = a.eos;
    p.part_sum = (double *)(((uintptr_t)a.workspace + 15) & ~(uintptr_t)15);
    p.part_best = (Candidate *)(p.part_sum + rows * parts);
    p.part_max = (float *)(p.part_best + rows * parts * a.keep);
    p.scores = a.scores, p.ended = a.ended, p.scores_out = a.scores_out, p.parents = a.parents, p.tokens = a.tokens, p.ended_out = a.ended_out;
    p.by_parts = fast_div(parts), p.by_row_candidates = fast_div(parts * a.keep);
    const dim3 grid((unsigned)(rows * parts));
    if (a.dtype == TROCM_F16) {
        if (pieces == 16) beam_scan_kernel<_Float16, 16><<<grid, kThreads, 0, s>>>(p);
        else if (pieces == 4) beam_scan_kernel<_Float16, 4><<<grid, kThreads, 0, s>>>(p);
        else beam_scan_kernel<_Float16, 1><<<grid, kThreads, 0, s>>>(p);
    } else {
        if (pieces == 8) beam_scan_kernel<float, 8><<<grid, kThreads, 0, s>>>(p);
        else beam_scan_kernel<float, 2><<<grid, kThreads, 0, s>>>(p);
    }
    TROCM_HIP(hipGetLastError());
    if (a.dtype == TROCM_F16) beam_join_kernel<_Float16><<<dim3((unsigned)a.batch), kThreads, 0, s>>>(p);
    else beam_join_kernel<float><<<dim3((unsigned)a.batch), kThreads, 0, s>>>(p);
    TROCM_HIP(hipGetLastError());
    return 0;
}

}  // namespace trocm
