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
#include "common.h"
#include "fast_div.h"

namespace trocm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kPiece = 8;                     // consecutive values of a lane
constexpr int kWaveList = 256;                // values above the bound that a wave lists; ties up to `keep` come on top
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

template <typename T> struct alignas(sizeof(T)) Piece { T x[kPiece]; };   // (rows begin where they begin: whole pieces are loaded from any element)

// A part of a row: kThreads * kPiece * C values.
template <typename T, int C>
__global__ __launch_bounds__(kThreads) void beam_scan_kernel(SelectDev p) {
    constexpr int E = C * kPiece, kPart = kThreads * E;
    __shared__ Candidate s_list[kWaves * (kWaveList + kBeamMaxKeep)];
    __shared__ int s_count[kWaves];
    __shared__ float s_max[kWaves];
    __shared__ double s_sum[kWaves];
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const int row = p.by_parts.by(blockIdx.x), part = blockIdx.x - row * p.parts;
    const T *x = reinterpret_cast<const T *>(p.logits + row * p.row_bytes);
    const int i0 = part * kPart + tid * kPiece;
    uint32_t key[E];
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int i = i0 + c * kThreads * kPiece;
        if (i + kPiece <= p.vocab) {
            Piece<T> piece;
            __builtin_memcpy(&piece, x + i, sizeof(piece));
#pragma unroll
            for (int e = 0; e < kPiece; e++) key[c * kPiece + e] = key_of((float)piece.x[e]);
        } else {
#pragma unroll
            for (int e = 0; e < kPiece; e++) key[c * kPiece + e] = i + e < p.vocab ? key_of((float)x[i + e]) : 0;
        }
    }
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < E; e++) top = max(top, key[e]);

    // maximum and sum; a wave without values has the sum 0 at -inf
    uint32_t wave_top = top;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) wave_top = max(wave_top, (uint32_t)__shfl_xor((int)wave_top, d, 64));
    const float m = value_of(max(wave_top, kLowest)), ref = m == -INFINITY ? 0.0f : m;
    // (f32 for the values of a piece, f64 from there on: beam_join_kernel's s_err says what that may be off by)
    double all = 0.0;
#pragma unroll
    for (int c = 0; c < C; c++) {
        float sum = 0.0f;
#pragma unroll
        for (int e = c * kPiece; e < (c + 1) * kPiece; e++) sum += key[e] ? __builtin_amdgcn_exp2f((value_of(key[e]) - ref) * kLog2e) : 0.0f;
        all += (double)sum;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) all += __shfl_xor(all, d, 64);
    if (lane == 0) s_max[w] = m, s_sum[w] = all;

    // the wave's largest values
    Candidate *list = s_list + w * (kWaveList + kBeamMaxKeep);
    uint32_t bound = bound_of_lanes(top, p.keep);
    int above = 0;
#pragma unroll
    for (int e = 0; e < E; e++) above += __popcll(__builtin_amdgcn_ballot_w64(key[e] > bound));
    if (above > kWaveList) {
        bound = 0;
#pragma unroll 1
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
            int n = 0;
#pragma unroll
            for (int e = 0; e < E; e++) n += __popcll(__builtin_amdgcn_ballot_w64(key[e] >= (bound | bit)));
            if (n >= p.keep) bound |= bit;
        }
    }
    int n = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const uint64_t in = __builtin_amdgcn_ballot_w64(key[e] > bound);
        if (in) {
            if (key[e] > bound) list[n + lanes_below(in)] = Candidate{value_of(key[e]), i0 + (e / kPiece) * kThreads * kPiece + e % kPiece};
            n += __popcll(in);
        }
    }
    // and those that equal the bound, in their order: pieces, lanes, values of a piece
    if (bound) {
        const int most = max(n, p.keep);
#pragma unroll
        for (int c = 0; c < C; c++) {
            uint32_t ties = 0;
#pragma unroll
            for (int e = 0; e < kPiece; e++) ties |= (key[c * kPiece + e] == bound ? 1u : 0u) << e;
            if (n < most && __builtin_amdgcn_ballot_w64(ties != 0)) {
                const int mine = __popc(ties);
                int at = n, here = 0;
#pragma unroll
                for (int bit = 0; bit < 4; bit++) {
                    const uint64_t lanes = __builtin_amdgcn_ballot_w64((mine >> bit) & 1);
                    at += lanes_below(lanes) << bit, here += __popcll(lanes) << bit;
                }
                for (uint32_t left = ties; left && at < most; left &= left - 1, at++)
                    list[at] = Candidate{value_of(bound), i0 + c * kThreads * kPiece + __ffs(left) - 1};
                n = min(n + here, most);
            }
        }
    }
    if (lane == 0) s_count[w] = n;
    __syncthreads();

    // the workgroup's: every listed value counts those before it
    int counts[kWaves], total = 0;
#pragma unroll
    for (int y = 0; y < kWaves; y++) counts[y] = s_count[y], total += counts[y];
    Candidate *best = p.part_best + (int64_t)blockIdx.x * p.keep;
    for (int j = tid; j < total; j += kThreads) {
        int from = j, y = 0;
        while (from >= counts[y]) from -= counts[y++];
        const Candidate c = s_list[y * (kWaveList + kBeamMaxKeep) + from];
        int rank = 0;
        for (int o = 0; o < kWaves; o++)
            for (int z = 0; z < counts[o]; z++) {
                const Candidate d = s_list[o * (kWaveList + kBeamMaxKeep) + z];
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
    auto add = [&](float v) { sum += v == v ? (uint64_t)(ldexp(exp((double)v - (double)m), shift) + 0.5) : 0; };
    constexpr int kDeep = 4, kStep = kDeep * kThreads * kPiece;
    for (int i0 = 0; i0 < vocab; i0 += min(kStep, vocab - i0)) {
        Piece<T> piece[kDeep];
#pragma unroll
        for (int y = 0; y < kDeep; y++) {
            const int i = i0 + (y * kThreads + tid) * kPiece;
            if (i <= vocab - kPiece) __builtin_memcpy(&piece[y], x + i, sizeof(piece[y]));
        }
#pragma unroll
        for (int y = 0; y < kDeep; y++) {
            const int i = i0 + (y * kThreads + tid) * kPiece;
            if (i <= vocab - kPiece) {
#pragma unroll 1
                for (int e = 0; e < kPiece; e++) add((float)piece[y].x[e]);
            } else {
                for (int e = i; e < vocab; e++) add((float)x[e]);
            }
        }
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
    __shared__ double s_c[kJoinList], s_best_c[kWaves];
    __shared__ int s_place[kJoinList], s_count, s_best_place[kWaves], s_best_beam[kWaves];
    __shared__ uint64_t s_sums[kWaves];
    __shared__ uint8_t s_beam[kJoinList];
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, request = blockIdx.x;
    for (int beam = w; beam < p.beams; beam += kWaves) {
        const int64_t row = (int64_t)request * p.beams + beam;
        const float *pm = p.part_max + row * p.parts;
        const double *ps = p.part_sum + row * p.parts;
        float m = -INFINITY;
        for (int i = lane; i < p.parts; i += 64) m = fmaxf(m, pm[i]);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
        double l = 0.0;
        for (int i = lane; i < p.parts; i += 64) l += pm[i] == -INFINITY ? 0.0 : ps[i] * exp((double)pm[i] - (double)m);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d, 64);
        if (lane == 0) {
            const float score = p.scores[row];
            const bool dead = !(fabsf(score) < INFINITY);
            s_score[beam] = dead ? -INFINITY : (double)score;
            s_lse[beam] = (double)m + log(l);
            s_max[beam] = m;
            s_ended[beam] = p.ended && p.ended[row] != 0;
            s_kind[beam] = dead ? 2 : s_ended[beam] ? 1 : !(fabsf(m) < INFINITY) ? 2 : 0;
            // What the sum may be off by, relatively, is what its logarithm is: exponents d by two half steps of f32, weighted by the weights at
            // most ln(vocab / l) of them (their entropy is d + ln l on average), the exponential's two, a piece's seven additions; f64 from there on.
            s_err[beam] = s_kind[beam] == 0 ? (2.0 * fmax(log((double)p.vocab / l), 0.0) + 10.0) * 0x1p-24 : 0.0;
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
        const float bound = value_of(max(bound_of_lanes(top, p.keep), kLowest));
        const double from = (double)bound - 0x1p-23 * fabs((double)bound) - 0x1p-149 - 2.0 * err;   // (-inf stays that)
        if (tid == 0) s_count = 0;
        __syncthreads();
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
                if (in && at < kJoinList) s_c[at] = r.c, s_place[at] = r.place, s_beam[at] = (uint8_t)r.beam;
            }
        }
        __syncthreads();
        const int listed = min(s_count, kJoinList);
        const bool whole = s_count <= kJoinList;
        if (again == 0) {   // beams whose values are too near for sums of 32-bit terms
            if (!whole) {
                for (int beam = tid; beam < p.beams; beam += kThreads) s_again[beam] = s_kind[beam] == 0;
                if (tid == 0) s_any = 1;
            }
            for (int j = tid; whole && j < listed; j += kThreads) {
                const double c = s_c[j];
                const int place = s_place[j], beam = s_beam[j];
                int rank = 0, near = 0;
                for (int o = 0; o < listed; o++) {
                    rank += before(s_c[o], s_place[o], c, place);
                    near |= s_beam[o] != beam && fabs(s_c[o] - c) <= s_err[beam] + s_err[s_beam[o]] ? 1 : 0;
                }
                if (near && rank < p.keep) {
                    for (int o = 0; o < listed; o++) {
                        const int other = s_beam[o];
                        if (other != beam && s_err[beam] + s_err[other] > 0.0 && fabs(s_c[o] - c) <= s_err[beam] + s_err[other]) s_again[beam] = s_again[other] = 1, s_any = 1;
                    }
                }
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
            for (int j = tid; j < listed; j += kThreads) {
                const double c = s_c[j];
                const int place = s_place[j];
                int rank = 0;
                for (int o = 0; o < listed; o++) rank += before(s_c[o], s_place[o], c, place);
                if (rank < p.keep) put(rank, c, place, s_beam[j]);
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

// Values of a row that a workgroup takes.
int64_t part_of(int64_t rows, int64_t vocab) { return rows * ((vocab + 8191) / 8192) >= 256 ? 8192 : 2048; }

size_t bytes_for(int64_t rows, int64_t parts, int64_t keep) { return (size_t)(rows * parts) * (sizeof(double) + sizeof(float) + sizeof(Candidate) * (size_t)keep) + 64; }

}  // namespace

size_t beam_select_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int64_t keep) {
    const int64_t rows = batch * beams, part = part_of(rows, vocab);
    return bytes_for(rows, (vocab + part - 1) / part, keep);
}

int launch_beam_select(const BeamSelectArgs &a, hipStream_t s) {
    if (a.batch == 0) return 0;
    const int64_t rows = a.batch * a.beams, part = part_of(rows, a.vocab), parts = (a.vocab + part - 1) / part;
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
        if (part == 8192) beam_scan_kernel<_Float16, 4><<<grid, kThreads, 0, s>>>(p);
        else beam_scan_kernel<_Float16, 1><<<grid, kThreads, 0, s>>>(p);
    } else {
        if (part == 8192) beam_scan_kernel<float, 4><<<grid, kThreads, 0, s>>>(p);
        else beam_scan_kernel<float, 1><<<grid, kThreads, 0, s>>>(p);
    }
    TROCM_HIP(hipGetLastError());
    if (a.dtype == TROCM_F16) beam_join_kernel<_Float16><<<dim3((unsigned)a.batch), kThreads, 0, s>>>(p);
    else beam_join_kernel<float><<<dim3((unsigned)a.batch), kThreads, 0, s>>>(p);
    TROCM_HIP(hipGetLastError());
    return 0;
}

}  // namespace trocm
