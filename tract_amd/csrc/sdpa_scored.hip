// Prompts whose scores are capped, biased by distance, or cut into documents: f16, head sizes 64 and 128.
//
//   s = scale q.k;   s = cap tanh(s / cap);   s -= slope |i - j|;   softmax over the visible j;   out = P V
//
// The rows of a kv head are (query, head of the group), heads fastest, so that a workgroup of 4 waves x 32 rows covers few
// queries and its causal frontier is short.  S^T = K Q^T and O^T = V^T P^T on 32x32x16 MFMAs: every softmax scalar of a row
// sits in one lane.  A tile of 64 keys is staged into LDS once for the four waves, double buffered, its loads issued two
// tiles ahead: one barrier per tile.  Two groups of four waves may take a workgroup's tiles in turn (NK == 2) and join their rows
// at the end.  Two workgroups (head size 64: three) share a compute unit without knowing of each
// other, so that one's softmax runs beside the other's MFMAs.
//
// What bounds it: the sum of a SIMD's vector and matrix streams, which take turns.  4096 queries of 32 heads over 8, 128 features, capped: 187 to 194 us
// from card to card (709 to 735 TFLOP/s of visible products; a large product alone reaches 1176), vector instructions 53 % of the cycles and matrix
// instructions 34 %.  Per
// 64 scores the cap takes two of the three exponentials and reciprocals (8 cycles each) and two of the four other instructions (4).
// 64 heads of 64 features 221 us.  Two batches of 4096 in 9 documents, 14 heads over 2, 64 features, with slopes: 50 us; there the compute
// units have unlike shares (on average 27 tiles, 49 at most); in 40 documents, where a workgroup's start and end are most of it, 23 us.
//
// Weights are rounded to f16, half a step each, since the product with V takes f16 operands: what is left of them would be a second product, and
// the matrix stream is a third of the time.  The row's sum takes the rounded weights, so that a row of equal values stays that value.  Against 64
// bits outputs are off by 2.3e-4 (2-norm, relative), of which the rounding of the result is 2.1e-4.  All else is f32.
#include <hip/hip_fp16.h>
#include <limits.h>
#include <string.h>
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
constexpr int kWaves = 4, kTile = 64, kRows = 32 * kWaves;   // waves with rows of their own, of each of NK groups
constexpr float kNone = -1.7e38f;   // the reference of a row that has seen nothing: finite, so that a hidden score stays at minus infinity against it
constexpr int kListMax = 4096;   // key tiles that documents are looked up for

struct ScoredDev {
    const char *q;
    _Float16 *out;
    const char *k, *v;
    int64_t stride_b, stride_h, stride_t;   // bytes
    int B, Hq, Hkv, Sq, G, Sk, row_tiles;
    FastDiv by_g;
    float scale, cap;
    int causal;
    const float *slopes;
    const int *docs, *prefix_lens;
};

__device__ __forceinline__ half4_t lds_read_tr16(const _Float16 *lds_ptr) {   // (see sdpa_rows.hip)
    typedef __attribute__((address_space(3))) short4_t *lds_v4_ptr;
    short4_t r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4_ptr)(uintptr_t)(uint32_t)(uintptr_t)lds_ptr);
    return __builtin_bit_cast(half4_t, r);
}

template <int D, int NK, bool CAP, bool SLOPES, bool DOCS>
__global__ __launch_bounds__(256 * NK, D == 128 || NK == 2 ? 2 : 3) void sdpa_scored_kernel(ScoredDev p) {
    constexpr int KS = D / 16, DB = D / 32;
    constexpr int KROW = D + 8, VROW = D + 16;        // halves per row in LDS (bank spread of the two kinds of reads)
    constexpr int kThreads = 64 * kWaves;             // of a group
    constexpr int PPR = D / 8, RPI = kThreads / PPR, NL = kTile / RPI;   // 16-byte pieces per row, rows per load of a group, loads per tile and tensor
    constexpr int K_TILE = kTile * KROW, V_TILE = kTile * VROW, OROW = D + 8, JROW = D + 4;
    static_assert(kWaves * 32 * OROW <= 2 * V_TILE, "the output goes through the V buffers");
    __shared__ __attribute__((aligned(16))) _Float16 lds_all[NK][2 * K_TILE + 2 * V_TILE];
    __shared__ uint16_t s_list[DOCS ? kListMax : 1];
    __shared__ int s_counts[NK * kWaves], s_range[2][kWaves];
    __shared__ __attribute__((aligned(16))) int s_ids_all[NK][2][DOCS ? kTile : 4];   // documents of the staged tiles' tokens

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wave / kWaves, w = wave % kWaves;   // group, wave of it
    const int tid = threadIdx.x % kThreads, lane = tid & 63, hb = lane >> 5, l32 = lane & 31;
    const int kvh = blockIdx.x;   // (consecutive workgroups go to the 8 XCDs in turn: a kv head's keys meet in few L2 caches)
    const int b = blockIdx.y, rt = p.row_tiles - 1 - (int)blockIdx.z;   // (the longest first)
    _Float16 (*lds_k)[K_TILE] = reinterpret_cast<_Float16 (*)[K_TILE]>(&lds_all[kg][0]), (*lds_v)[V_TILE] = reinterpret_cast<_Float16 (*)[V_TILE]>(&lds_all[kg][2 * K_TILE]);
    int (*s_ids)[DOCS ? kTile : 4] = s_ids_all[kg];
    const int seq_rows = p.Sq * p.G, row0 = rt * kRows, off = p.Sk - p.Sq;

    const int r = min(row0 + 32 * w + l32, seq_rows - 1), i = p.by_g.by(r), g = r - i * p.G;
    const int64_t out_row = ((int64_t)b * p.Hq + kvh * p.G + g) * p.Sq + i;
    const int at = i + off;
    int lim = p.Sk - 1, n_vis = p.Sk;
    const int pre = p.prefix_lens ? max(p.prefix_lens[b], 0) : 0;   // (of any value: a negative one is no prefix)
    if (p.causal) {
        lim = min(lim, max(at, pre - 1));
        n_vis = max(0, min(p.Sk, max(p.by_g.by(min(row0 + kRows, seq_rows) - 1) + off + 1, pre)));
    }
    const int wave_lim = __builtin_amdgcn_readfirstlane(p.causal ? max(p.by_g.by(min(row0 + 32 * w + 32, seq_rows) - 1) + off, pre - 1) : p.Sk - 1);
    const bool wave_has_rows = row0 + 32 * w < seq_rows;
    const int t_end = (n_vis + kTile - 1) / kTile;
    int n_tiles = t_end;

    const char *kb = p.k + (int64_t)b * p.stride_b + (int64_t)kvh * p.stride_h, *vb = p.v + (int64_t)b * p.stride_b + (int64_t)kvh * p.stride_h;
    const int key0 = tid / PPR, ch = tid % PPR;
    const uint32_t lane_off = (uint32_t)key0 * (uint32_t)p.stride_t + ch * 16;
    const int *docs = DOCS ? p.docs + (int64_t)b * p.Sk : nullptr;
    u32x4 kpre[NL], vpre[NL];
    int id_pre = 0;   // documents: of this tile's token `lane`
    auto prefetch = [&](int k_lo) {
        const int most = p.Sk - 1 - k_lo;
        const char *tk = kb + (int64_t)k_lo * p.stride_t, *tv = vb + (int64_t)k_lo * p.stride_t;
        if (most >= kTile - 1) {   // wave-uniform addresses and one offset per lane
            uint32_t o = lane_off;
            asm volatile("" : "+v"(o));   // (stays a 32-bit offset up to the loads)
#pragma unroll
            for (int j = 0; j < NL; j++) {
                kpre[j] = *reinterpret_cast<const u32x4 *>(tk + (int64_t)(j * RPI) * p.stride_t + o);
                vpre[j] = *reinterpret_cast<const u32x4 *>(tv + (int64_t)(j * RPI) * p.stride_t + o);
            }
        } else {   // rows past the last key repeat it
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const uint32_t o = (uint32_t)min(key0 + j * RPI, most) * (uint32_t)p.stride_t + ch * 16;   // (rows of at most 2^25 bytes)
                kpre[j] = *reinterpret_cast<const u32x4 *>(tk + o);
                vpre[j] = *reinterpret_cast<const u32x4 *>(tv + o);
            }
        }
        if (DOCS) id_pre = docs[k_lo + min(lane, most)];
    };
    // The last tile first, that of the rows' own tokens: it is asked for before anything is known of the documents.
    // (So are the queries and the first ids: one latency for all.)
    const int guess = t_end - 1 - kg;
    constexpr int PW = 16;   // tiles whose ids a wave looks at before the waves compare: four at a time, four tokens per lane
    struct alignas(4) Ids { int e[4]; } ids[DOCS ? PW / 4 : 1];
    auto ask_ids = [&](int first) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < PW / 4; x++)   // (past the last token: the last four again, which may only make a tile look at more)
            ids[x] = *reinterpret_cast<const Ids *>(docs + min((first + 4 * x) * kTile + 4 * lane, p.Sk - 4));
    };
    const int doc = DOCS ? docs[at] : 0;
    if constexpr (DOCS) ask_ids(wave * PW);
    if (guess >= 0) prefetch(guess * kTile);
    half8_t qf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ks++) qf[ks] = *reinterpret_cast<const half8_t *>(p.q + out_row * (2 * D) + 32 * ks + 16 * hb);

    // A score in the log2 domain is base + to_log2 s, of s the product with the key or, capped, 1 / (e^2x + 1) with x = scale q.k / cap:
    // cap log2e tanh(x) = A - 2 A / (e^2x + 1).  The largest score is the smallest s there.  Only weights take the whole sum.
    const float base = CAP ? p.cap * kLog2e : 0.0f, to_log2 = CAP ? -2.0f * base : p.scale * kLog2e, cap_k = CAP ? within_f32(p.scale / p.cap * (2.0f * kLog2e)) : 0.0f;
    const float hidden = CAP ? INFINITY : -INFINITY, slope = SLOPES ? -kLog2e / to_log2 * p.slopes[kvh * p.G + g] : 0.0f;
    if (DOCS && doc < 0) lim = -1;   // padding sees nothing
    bool listed = false;
    if constexpr (DOCS) {
        // The tiles with a token of the documents of these rows (a smallest and a largest id: ids in any order are fine), and of them
        // those whose tokens are all of the rows' one document, which need no look at the ids.
        if (n_tiles <= kListMax) {
            int dmin = doc >= 0 ? doc : INT_MAX, dmax = doc;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) dmin = min(dmin, __shfl_xor(dmin, d, 64)), dmax = max(dmax, __shfl_xor(dmax, d, 64));
            if (kg == 0 && lane == 0) s_range[0][w] = dmin, s_range[1][w] = dmax;
            __syncthreads();
            dmin = INT_MAX, dmax = -1;
#pragma unroll
            for (int x = 0; x < kWaves; x++) dmin = min(dmin, s_range[0][x]), dmax = max(dmax, s_range[1][x]);
            const int one_doc = dmin == dmax ? dmin : INT_MIN, dlow = max(dmin, 0);   // (no tile is whole of what is no document)
            int n = 0;
            for (int t0 = 0; t0 < t_end; t0 += NK * kWaves * PW) {
                const int first = t0 + wave * PW;
                const uint32_t there = first >= t_end ? 0 : (1u << min(PW, t_end - first)) - 1;
                uint32_t active = 0, whole = 0;
                if (t0) ask_ids(first);
#pragma unroll
                for (int x = 0; x < PW / 4; x++) {
                    bool in = false, other = false;
#pragma unroll
                    for (int y = 0; y < 4; y++) in = in || (ids[x].e[y] >= dlow && ids[x].e[y] <= dmax), other = other || ids[x].e[y] != one_doc;
                    const uint64_t a = __builtin_amdgcn_ballot_w64(in), o = __builtin_amdgcn_ballot_w64(other);
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        active |= ((a >> 16 * y) & 0xffff) != 0 ? 1u << (4 * x + y) : 0;
                        whole |= ((o >> 16 * y) & 0xffff) == 0 ? 1u << (4 * x + y) : 0;
                    }
                }
                active &= there;
                if (lane == 0) s_counts[wave] = __popc(active);
                __syncthreads();
                int place = n;
                for (int x = 0; x < NK * kWaves; x++) {
                    if (x < wave) place += s_counts[x];
                    n += s_counts[x];
                }
                if (lane < PW && ((active >> lane) & 1)) s_list[place + __popc(active & ((1u << lane) - 1))] = (uint16_t)((first + lane) | (one_doc >= 0 && ((whole >> lane) & 1) ? 0x8000 : 0));
                __syncthreads();
            }
            n_tiles = n;
            listed = true;
        }
    }
    auto entry = [&](int n) -> int { return DOCS && listed ? __builtin_amdgcn_readfirstlane(s_list[n_tiles - 1 - n]) : n_tiles - 1 - n; };
    auto tile_lo = [&](int e) -> int { return (DOCS && listed ? e & 0x7fff : e) * kTile; };

    auto stage = [&](int buf) {
        if (DOCS) {
            if (tid < kTile) s_ids[buf][tid] = id_pre;
            const uint64_t padding = __builtin_amdgcn_ballot_w64(id_pre < 0);
            if (padding != 0) {   // values of padding may hold anything
#pragma unroll
                for (int j = 0; j < NL; j++)
                    if ((padding >> (key0 + j * RPI)) & 1) vpre[j] = u32x4{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int j = 0; j < NL; j++) {
            *reinterpret_cast<u32x4 *>(&lds_k[buf][(key0 + j * RPI) * KROW + ch * 8]) = kpre[j];
            *reinterpret_cast<u32x4 *>(&lds_v[buf][(key0 + j * RPI) * VROW + ch * 8]) = vpre[j];
        }
    };

    // A row's reference: s_ref among the scores, m_run in the log2 domain.  What the rounding of m_run left out is a factor that all weights
    // taken from it share, unless it is an exponent that f16 does not have: from 2^20 on m_run is NaN up to the end, so that every tile of
    // the row gets a look, which takes weights from s_ref and moves it to whatever is larger.
    float m_run = kNone, s_ref = 0.0f, l_run = 0.0f;
    float16_t o[DB];
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int x = 0; x < 16; x++) o[db][x] = 0.0f;
    if (DOCS && kg < n_tiles && tile_lo(entry(kg)) != guess * kTile) prefetch(tile_lo(entry(kg)));   // (padding, or a prefix)
#pragma unroll
    for (int ks = 0; ks < KS; ks++) asm volatile("" : "+v"(qf[ks]));   // settled here, not by a wait in the loop that would take the prefetch in too
    if (kg < n_tiles) {
        stage(0);
        if (kg + NK < n_tiles) prefetch(tile_lo(entry(kg + NK)));
    }
    for (int n = kg, it = 0; n - kg < n_tiles; n += NK, it++) {   // (as many rounds for every group)
        __syncthreads();   // tile n is in LDS; every wave is done with the buffers about to be overwritten
        const int buf = it & 1, e = NK == 1 || n < n_tiles ? entry(n) : 0, k_lo = tile_lo(e);
        if (wave_has_rows && (NK == 1 || n < n_tiles) && k_lo <= wave_lim) {
            float16_t s[2];
#pragma unroll
            for (int kb2 = 0; kb2 < 2; kb2++)
#pragma unroll
                for (int x = 0; x < 16; x++) s[kb2][x] = 0.0f;
            const _Float16 *ksrc = &lds_k[buf][l32 * KROW + 8 * hb];
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int kb2 = 0; kb2 < 2; kb2++)
                    s[kb2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const half8_t *>(ksrc + 32 * kb2 * KROW + 16 * ks), qf[ks], s[kb2], 0, 0, 0);

            // this lane's keys: k_lo + 4 hb + c, c = 32 kb2 + 8 (x / 4) + x % 4
            float d0 = (float)(at - k_lo - 4 * hb);
            // (asked for once the products are there: all 32 distances computed beside the MFMAs spill registers; of the group of four
            // at hand, so that what is subtracted are inline constants)
            if constexpr (SLOPES) asm volatile("" : "+v"(d0), "+v"(s[1]));
            if constexpr (CAP) {
#pragma unroll
                for (int kb2 = 0; kb2 < 2; kb2++)
#pragma unroll
                    for (int x = 0; x < 16; x++) s[kb2][x] = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[kb2][x] * cap_k) + 1.0f);
            }
            if constexpr (DOCS) {
                if (!(listed && (e & 0x8000))) {
#pragma unroll
                    for (int kb2 = 0; kb2 < 2; kb2++)
#pragma unroll
                        for (int x = 0; x < 16; x += 4) {
                            const int4 four = *reinterpret_cast<const int4 *>(&s_ids[buf][32 * kb2 + 2 * x + 4 * hb]);
                            s[kb2][x] = four.x == doc ? s[kb2][x] : hidden;
                            s[kb2][x + 1] = four.y == doc ? s[kb2][x + 1] : hidden;
                            s[kb2][x + 2] = four.z == doc ? s[kb2][x + 2] : hidden;
                            s[kb2][x + 3] = four.w == doc ? s[kb2][x + 3] : hidden;
                        }
                }
            }
            if constexpr (SLOPES) {
#pragma unroll
                for (int kb2 = 0; kb2 < 2; kb2++)
#pragma unroll
                    for (int x = 0; x < 16; x++) {
                        const float d = (x & 3) == 0 ? d0 : (x & 3) == 1 ? d0 - 1.0f : (x & 3) == 2 ? d0 - 2.0f : (d0 - 2.0f) - 1.0f;
                        s[kb2][x] = __builtin_fmaf(slope, fabsf(d), s[kb2][x]);
                        if ((x & 3) == 3) d0 -= 8.0f;
                    }
            }
            const int last = lim - k_lo - 4 * hb;
            if (__builtin_amdgcn_ballot_w64(last < 60) != 0) {
#pragma unroll
                for (int kb2 = 0; kb2 < 2; kb2++)
#pragma unroll
                    for (int x = 0; x < 16; x++) s[kb2][x] = 32 * kb2 + 8 * (x >> 2) + (x & 3) <= last ? s[kb2][x] : hidden;
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
                    for (int x = 0; x < 4; x++) sum = __builtin_amdgcn_fdot2(half2_t{pf[st][2 * x], pf[st][2 * x + 1]}, ones, sum, false);   // the same rounded weights
                }
            };
            bool look = !DOCS && n == kg;   // (documents: weights against no reference come to infinity; asked for by place, the first tile spills scalar registers)
            if (!look) {
                weights(base - m_run);
                look = __builtin_amdgcn_ballot_w64(!(sum < 32768.0f)) != 0;
            }
            if (look) {
                float top = s[0][0];
#pragma unroll
                for (int kb2 = 0; kb2 < 2; kb2++)
#pragma unroll
                    for (int x = 0; x < 16; x++) top = CAP ? fminf(top, s[kb2][x]) : fmaxf(top, s[kb2][x]);
                const float other = __shfl_xor(top, 32, 64), s_top = CAP ? fminf(top, other) : fmaxf(top, other);
                top = __builtin_fmaf(s_top, to_log2, base);
                const bool far = m_run != m_run, moved = top > m_run + 8.0f || (far && (CAP ? s_top < s_ref : s_top > s_ref));
                const float keep = moved ? __builtin_amdgcn_exp2f(far ? (s_ref - s_top) * to_log2 : m_run - top) : 1.0f;
                if (moved) s_ref = s_top, m_run = fabsf(top) < 0x1p20f ? top : __builtin_nanf("");
                l_run *= keep;
#pragma unroll
                for (int db = 0; db < DB; db++)
#pragma unroll
                    for (int x = 0; x < 16; x++) o[db][x] *= keep;
                float from = base - m_run;
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(m_run != m_run) != 0, 0)) {
                    const float less = m_run != m_run ? s_ref : 0.0f;   // (rows of ordinary scores stay as they are)
#pragma unroll
                    for (int kb2 = 0; kb2 < 2; kb2++)
#pragma unroll
                        for (int x = 0; x < 16; x++) s[kb2][x] -= less;
                    if (m_run != m_run) from = 0.0f;
                }
                weights(from);
            }
            l_run += sum;
            const _Float16 *vsrc = &lds_v[buf][(4 * hb + ((lane & 15) >> 2)) * VROW + 16 * ((lane >> 4) & 1) + 4 * (lane & 3)];
#pragma unroll
            for (int st = 0; st < 4; st++)
#pragma unroll
                for (int db = 0; db < DB; db++) {
                    const half4_t lo = lds_read_tr16(vsrc + 16 * st * VROW + 32 * db), hi = lds_read_tr16(vsrc + (16 * st + 8) * VROW + 32 * db);
                    o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), pf[st], o[db], 0, 0, 0);
                }
        }
        if (n + NK < n_tiles) {   // the next tile to LDS after this one's arithmetic, which covers its loads' latency
            stage(buf ^ 1);
            if (n + 2 * NK < n_tiles) prefetch(tile_lo(entry(n + 2 * NK)));
        }
    }
    l_run += __shfl_xor(l_run, 32, 64);
    if (NK == 2 && m_run != m_run) m_run = __builtin_fmaf(s_ref, to_log2, base);

    if constexpr (NK == 2) {   // the second group's rows join the first's, through the tiles' LDS
        float *comb = reinterpret_cast<float *>(&lds_all[0][0]) + w * 32 * JROW, *comb_ml = reinterpret_cast<float *>(&lds_all[0][0]) + kWaves * 32 * JROW + w * 64;
        static_assert(kWaves * (32 * JROW + 64) * 4 <= (int)sizeof(lds_all), "rows are joined where the tiles were");
        __syncthreads();
        if (kg == 1) {
#pragma unroll
            for (int db = 0; db < DB; db++)
#pragma unroll
                for (int x = 0; x < 4; x++)
                    *reinterpret_cast<float4_t *>(comb + l32 * JROW + 32 * db + 8 * x + 4 * hb) = float4_t{o[db][4 * x], o[db][4 * x + 1], o[db][4 * x + 2], o[db][4 * x + 3]};
            comb_ml[lane] = hb ? l_run : m_run;
        }
        __syncthreads();
        if (kg == 1) return;
        const float m2 = comb_ml[l32], l2 = comb_ml[32 + l32], mm = fmaxf(m_run, m2);
        const float f1 = __builtin_amdgcn_exp2f(m_run - mm), f2 = __builtin_amdgcn_exp2f(m2 - mm);
        l_run = l_run * f1 + l2 * f2;
#pragma unroll
        for (int db = 0; db < DB; db++)
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const float4_t v = *reinterpret_cast<const float4_t *>(comb + l32 * JROW + 32 * db + 8 * x + 4 * hb);
#pragma unroll
                for (int y = 0; y < 4; y++) o[db][4 * x + y] = o[db][4 * x + y] * f1 + v[y] * f2;
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");   // (a wave's corner is its own)
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    } else {
        __syncthreads();
    }
    // rows to their places in whole lines, through a corner of LDS of the wave's own
    if (!wave_has_rows) return;
    const float inv = l_run > 0.0f ? 1.0f / l_run : 0.0f;
    _Float16 *tr = NK == 2 ? reinterpret_cast<_Float16 *>(reinterpret_cast<float *>(&lds_all[0][0]) + w * 32 * JROW) : &lds_v[0][0] + w * 32 * OROW;
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
        for (int x = 0; x < 4; x++) {
            half4_t h4;
#pragma unroll
            for (int y = 0; y < 4; y++) h4[y] = (_Float16)(o[db][4 * x + y] * inv);
            *reinterpret_cast<half4_t *>(tr + l32 * OROW + 32 * db + 8 * x + 4 * hb) = h4;
        }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    constexpr int LPR = D / 8, RPS = 64 / LPR;
#pragma unroll
    for (int j = 0; j < 32 / RPS; j++) {
        const int row = j * RPS + lane / LPR, rr = row0 + 32 * w + row, ii = p.by_g.by(rr), gg = rr - ii * p.G;
        if (rr < seq_rows)
            *reinterpret_cast<u32x4 *>(p.out + (((int64_t)b * p.Hq + kvh * p.G + gg) * p.Sq + ii) * D + lane % LPR * 8) = *reinterpret_cast<const u32x4 *>(tr + row * OROW + lane % LPR * 8);
    }
}

template <int D, int NK>
void launch_of(const ScoredDev &p, hipStream_t s) {
    const bool cap = p.cap > 0.0f, slopes = p.slopes != nullptr, docs = p.docs != nullptr;
    const dim3 g((unsigned)p.Hkv, (unsigned)p.B, (unsigned)p.row_tiles), t(64 * kWaves * NK);
    if (docs) {
        if (cap && slopes) hipLaunchKernelGGL((sdpa_scored_kernel<D, NK, true, true, true>), g, t, 0, s, p);
        else if (cap) hipLaunchKernelGGL((sdpa_scored_kernel<D, NK, true, false, true>), g, t, 0, s, p);
        else if (slopes) hipLaunchKernelGGL((sdpa_scored_kernel<D, NK, false, true, true>), g, t, 0, s, p);
        else hipLaunchKernelGGL((sdpa_scored_kernel<D, NK, false, false, true>), g, t, 0, s, p);
    } else {
        if (cap && slopes) hipLaunchKernelGGL((sdpa_scored_kernel<D, NK, true, true, false>), g, t, 0, s, p);
        else if (cap) hipLaunchKernelGGL((sdpa_scored_kernel<D, NK, true, false, false>), g, t, 0, s, p);
        else if (slopes) hipLaunchKernelGGL((sdpa_scored_kernel<D, NK, false, true, false>), g, t, 0, s, p);
        else hipLaunchKernelGGL((sdpa_scored_kernel<D, NK, false, false, false>), g, t, 0, s, p);
    }
}

}  // namespace

// 0 done, 1 failed, 2 not covered (the kernels of sdpa_rows.hip take it).
int launch_sdpa_scored_prompt(const SdpaRowsArgs &a, hipStream_t s) {
    if (a.dtype != TROCM_F16 || (a.D != 64 && a.D != 128) || a.P || a.lens || a.seqs || a.Sk == 0 || a.softcap > kFastTanhCap) return 2;
    if (a.softcap > 0.0f ? a.softcap < 1e-6f : !(a.scale > 1e-6f)) return 2;   // (slopes are divided by it, and the largest product stands for the largest score)
    const double per = a.softcap > 0.0f ? 2.0 * a.softcap : a.scale;   // (slopes of up to 1e30 times a distance, so divided, and as they are, stay inside f32)
    if (a.slopes && (double)(a.Sk + a.Sq) > 1e8 * (per < 1.0 ? per : 1.0)) return 2;
    auto aligned = [](const void *x) { return (uintptr_t)x % 16 == 0; };
    const int64_t G = a.Hq / a.Hkv, rows = a.Sq * G;
    if (!aligned(a.q) || !aligned(a.out) || !aligned(a.k) || !aligned(a.v) || a.stride_b % 8 || a.stride_h % 8 || a.stride_t % 8 || a.stride_t * 2 > (1 << 25)) return 2;
    if (rows >= (1 << 30)) return 2;
    const int64_t row_tiles = (rows + kRows - 1) / kRows, grid = a.B * a.Hkv * row_tiles;
    if (rows <= 32 || a.B > 65535 || row_tiles > 65535 || (a.documents && a.Sk < 4)) return 2;   // (four documents' ids in a load)
    // Up to two workgroups per compute unit (one, where documents leave them unlike work) take their tiles in two groups of waves.
    // Fewer tiles still go faster as tiles of 32 rows whose four waves share the keys (sdpa_rows.hip), which take about 1.5 times as long
    // per product but are four times as many.  What either takes, in us: a start, then the longest workgroup's tiles of 64 keys, or all
    // tiles over the chip.  (Capped, 32 heads over 8, D = 128, one group | two | there: 300 queries 12.9 | 12.8 | 10.1; 500 18.4 | 16.9 |
    // 12.5; 1000 32.7 | 28.0 | 31.4; 2048 65.3 | 58.2 | 86.1; 4096 194 | 200 | 295; 500 behind 3000 97.5 | 75.6 | 61.6.  D = 64, 64 heads:
    // 300 10.2 | 9.6 | 8.4; 1000 26.9 | 25.2 | 30.6; 4096 234 | 288 | 355.)
    const int nk = grid <= (int64_t)num_compute_units() * (a.documents ? 1 : 2) ? 2 : 1;
    const double cus = num_compute_units(), wide = a.D == 128 ? 1.0 : 0.62, last = (double)((a.Sk + kTile - 1) / kTile);
    const double first = a.causal && !a.prefix_lens ? (double)((a.Sk - a.Sq > 0 ? a.Sk - a.Sq : 0) / kTile + 1) : last;
    const double all = (double)grid * (first + last) / 2 / cus, longest = nk == 2 ? (double)(int64_t)((last + 1) / 2) * 2.75 : last * 1.8;
    const double tall = 4.0 + (longest > all * 1.44 ? longest : all * 1.44) * wide, each = all * 2.25 + (last - first) * 0.5;
    const double flat = 4.0 + (last > each ? last : each) * wide;
    if (flat < tall) return 2;
    ScoredDev p;
    memset(&p, 0, sizeof(p));
    p.q = (const char *)a.q, p.out = (_Float16 *)a.out, p.k = (const char *)a.k, p.v = (const char *)a.v;
    p.stride_b = a.stride_b * 2, p.stride_h = a.stride_h * 2, p.stride_t = a.stride_t * 2;
    p.B = (int)a.B, p.Hq = (int)a.Hq, p.Hkv = (int)a.Hkv, p.Sq = (int)a.Sq, p.G = (int)G, p.Sk = (int)a.Sk, p.row_tiles = (int)row_tiles, p.by_g = fast_div(G);
    p.scale = a.scale, p.cap = a.softcap, p.causal = a.causal;
    p.slopes = a.slopes, p.docs = a.documents, p.prefix_lens = a.prefix_lens;
    if (a.D == 64) nk == 2 ? launch_of<64, 2>(p, s) : launch_of<64, 1>(p, s);
    else nk == 2 ? launch_of<128, 2>(p, s) : launch_of<128, 1>(p, s);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail("sdpa_scored launch failed: %s", hipGetErrorString(e));
    return 0;
}

}  // namespace trocm
