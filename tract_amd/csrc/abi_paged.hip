// Entry points over pages of keys and values, and beam search's choice: checks of arguments, in the manner of abi.hip.
#include <math.h>
#include <string.h>
#include <algorithm>
#include <initializer_list>
#include <numeric>
#include "common.h"

using namespace trocm;

namespace {

constexpr int64_t kMostTokens = 1ll << 30, kMostPage = 1ll << 20, kMostReclaimed = 1ll << 24;

// (far more than there is memory, and sums of a few such products stay inside of 64 bits)
constexpr double kReach = 281474976710656.0;
bool within_reach(int64_t rows, int64_t stride) { return (double)rows * (double)stride < kReach; }

struct Range { const void *at; size_t bytes; const char *name; };

int apart(const char *what, std::initializer_list<Range> outs, std::initializer_list<Range> ins) {
    for (const Range *o = outs.begin(); o != outs.end(); o++) {
        if (!o->at || !o->bytes) continue;
        for (const Range &i : ins)
            TROCM_REQUIRE(!i.at || !i.bytes || !ranges_meet(o->at, o->bytes, i.at, i.bytes), "%s: %s overlaps %s", what, o->name, i.name);
        for (const Range *p = outs.begin(); p != o; p++)
            TROCM_REQUIRE(!p->at || !p->bytes || !ranges_meet(o->at, o->bytes, p->at, p->bytes), "%s: %s overlaps %s", what, o->name, p->name);
    }
    return 0;
}

int aligned(const char *what, std::initializer_list<Range> all, size_t to) {
    for (const Range &r : all) TROCM_REQUIRE((uintptr_t)r.at % to == 0, "%s: %s is not aligned to its elements", what, r.name);
    return 0;
}

int pages_check(const char *what, int64_t n_pages, int64_t page_size) {
    TROCM_REQUIRE(n_pages >= 0, "%s: negative dimension", what);
    TROCM_REQUIRE(page_size >= 1 && page_size <= kMostPage, "%s: page_size must be 1 to %lld (got %lld)", what, (long long)kMostPage, (long long)page_size);
    TROCM_REQUIRE(n_pages <= kMostTokens / page_size, "%s: the pages hold more than 2^30 tokens", what);
    return 0;
}

int table_check(const char *what, int64_t n_seq, int64_t table_width, int64_t page_size, int64_t most_seqs) {
    TROCM_REQUIRE(n_seq >= 0 && table_width >= 0, "%s: negative dimension", what);
    TROCM_REQUIRE(n_seq <= most_seqs, "%s: %lld sequences are more than %lld", what, (long long)n_seq, (long long)most_seqs);
    TROCM_REQUIRE(table_width <= kMostTokens / page_size, "%s: a row of the table is of more than 2^30 tokens", what);
    return 0;
}

// Strides of the pools, checked; dense ones where none are given.
int page_strides_check(const char *what, int dtype, int64_t n_pages, int64_t kv_heads, int64_t head_dim, int64_t page_size, const int64_t *given, int64_t *st) {
    TROCM_REQUIRE(dtype == TROCM_F32 || dtype == TROCM_F16, "%s: dtype must be F32 or F16", what);
    TROCM_REQUIRE(kv_heads >= 0 && head_dim >= 0, "%s: negative dimension", what);
    TROCM_REQUIRE(head_dim < (1 << 24) && kv_heads <= 65535 && head_dim * page_size <= (1 << 29) && head_dim * kv_heads < (1 << 29), "%s: tensor too large", what);
    st[0] = kv_heads * page_size * head_dim, st[1] = page_size * head_dim, st[2] = head_dim;
    if (!given) return 0;
    for (int i = 0; i < 3; i++) {
        TROCM_REQUIRE(given[i] >= 0, "%s: negative page strides", what);
        TROCM_REQUIRE(given[i] < (1ll << 40), "%s: page strides too large", what);
        st[i] = given[i];
    }
    TROCM_REQUIRE(within_reach(n_pages, st[0]) && (double)kv_heads * st[1] + (double)page_size * st[2] < kReach, "%s: page strides too large", what);
    return 0;
}

size_t pool_bytes(int64_t n_pages, int64_t kv_heads, int64_t page_size, int64_t head_dim, const int64_t *st, int dtype) {
    if (!n_pages || !kv_heads || !head_dim) return 0;
    return (size_t)((n_pages - 1) * st[0] + (kv_heads - 1) * st[1] + (page_size - 1) * st[2] + head_dim) * elem_bytes(dtype);
}

// Whether two pools of these sizes and strides, `by` bytes apart, lie in one another's gaps (K and V halves of one tensor): with the largest strides
// outside, whose combinations are multiples of g bytes, and the others inside, which reach over e, what is at least e past a multiple of g and ends
// before the next one meets nothing.
bool interleaved(uint64_t by, int64_t n_pages, int64_t kv_heads, int64_t page_size, int64_t head_dim, const int64_t *st, int dtype) {
    struct Axis { int64_t n, stride; } axes[3] = {{n_pages, st[0]}, {kv_heads, st[1]}, {page_size, st[2]}};
    std::sort(axes, axes + 3, [](const Axis &a, const Axis &b) { return a.stride > b.stride; });
    uint64_t g = 0;
    for (int outer = 1; outer <= 3; outer++) {
        if (axes[outer - 1].n > 1) g = std::gcd(g, (uint64_t)axes[outer - 1].stride * elem_bytes(dtype));
        uint64_t e = (uint64_t)head_dim;
        for (int i = outer; i < 3; i++) e += (uint64_t)(axes[i].n - 1) * (uint64_t)axes[i].stride;
        e *= elem_bytes(dtype);
        if (g && by % g >= e && by % g + e <= g) return true;
    }
    return false;
}

}  // namespace

extern "C" {

int trocm_paged_plan(const int32_t *lens, const int32_t *n_new, int64_t n_seq, int64_t page_size, int32_t *table, int64_t table_width,
                     const int32_t *free_pages, const int32_t *free_count, int64_t n_pages, int32_t *refs, int64_t n_tokens, int32_t *lens_out,
                     int32_t *starts, int32_t *slots, int32_t *positions, int32_t *free_count_out, int32_t *refused, void *stream) {
    if (pages_check("paged_plan", n_pages, page_size) || table_check("paged_plan", n_seq, table_width, page_size, kPagedMaxSeqs)) return 1;
    TROCM_REQUIRE(n_tokens >= 0, "paged_plan: negative dimension");
    TROCM_REQUIRE(n_tokens <= kMostTokens, "paged_plan: %lld tokens are more than 2^30", (long long)n_tokens);
    if (n_seq) {
        TROCM_NOT_NULL(lens);
        TROCM_NOT_NULL(n_new);
        TROCM_NOT_NULL(lens_out);
        if (table_width) TROCM_NOT_NULL(table);
    }
    if (n_pages) TROCM_NOT_NULL(free_pages);
    TROCM_NOT_NULL(free_count);
    TROCM_NOT_NULL(free_count_out);
    TROCM_NOT_NULL(refused);
    if (n_tokens) TROCM_NOT_NULL(slots);
    const size_t n = (size_t)n_seq * 4, t = (size_t)n_tokens * 4, f = (size_t)n_pages * 4;
    const std::initializer_list<Range> outs = {{table, (size_t)n_seq * (size_t)table_width * 4, "table"}, {refs, f, "refs"}, {lens_out, n, "lens_out"}, {starts, n + 4, "starts"},
                                               {slots, t, "slots"}, {positions, t, "positions"}, {free_count_out, 4, "free_count_out"}, {refused, 4, "refused"}},
                                       ins = {{lens, n, "lens"}, {n_new, n, "n_new"}, {free_pages, f, "free_pages"}, {free_count, 4, "free_count"}};
    if (apart("paged_plan", outs, ins) || aligned("paged_plan", outs, 4) || aligned("paged_plan", ins, 4)) return 1;
    hipStream_t s;
    if (resolve_stream(stream, &s)) return 1;
    PagedPlanArgs a;
    a.lens = lens, a.n_new = n_new, a.free_pages = free_pages, a.free_count = free_count;
    a.table = table, a.refs = refs, a.lens_out = lens_out, a.starts = starts, a.slots = slots, a.positions = positions;
    a.free_count_out = free_count_out, a.refused = refused;
    a.n_seq = n_seq, a.page_size = page_size, a.table_width = table_width, a.n_pages = n_pages, a.n_tokens = n_tokens;
    return launch_paged_plan(a, s);
}

int trocm_paged_append(const void *k_new, const void *v_new, int dtype, int64_t n_tokens, int64_t kv_heads, int64_t head_dim,
                       const int64_t *k_strides, const int64_t *v_strides, const int32_t *slots, void *k_pages, void *v_pages,
                       int64_t n_pages, int64_t page_size, const int64_t *page_strides, void *stream) {
    PagedAppendArgs a;
    if (pages_check("paged_append", n_pages, page_size)) return 1;
    if (page_strides_check("paged_append", dtype, n_pages, kv_heads, head_dim, page_size, page_strides, a.page_strides)) return 1;
    TROCM_REQUIRE(n_tokens >= 0, "paged_append: negative dimension");
    TROCM_REQUIRE(n_tokens <= kMostTokens, "paged_append: tensor too large");
    if (n_tokens == 0 || kv_heads == 0 || head_dim == 0 || n_pages == 0) return 0;
    TROCM_NOT_NULL(k_new);
    TROCM_NOT_NULL(v_new);
    TROCM_NOT_NULL(slots);
    TROCM_NOT_NULL(k_pages);
    TROCM_NOT_NULL(v_pages);
    size_t rows[2];
    for (int y = 0; y < 2; y++) {
        const int64_t *given = y ? v_strides : k_strides;
        a.src_strides[y][0] = kv_heads * head_dim, a.src_strides[y][1] = head_dim;
        for (int i = 0; given && i < 2; i++) {
            TROCM_REQUIRE(given[i] >= 0, "paged_append: negative strides");
            TROCM_REQUIRE(given[i] < (1ll << 30), "paged_append: strides too large");
            a.src_strides[y][i] = given[i];
        }
        rows[y] = (size_t)((n_tokens - 1) * a.src_strides[y][0] + (kv_heads - 1) * a.src_strides[y][1] + head_dim) * elem_bytes(dtype);
    }
    const size_t pool = pool_bytes(n_pages, kv_heads, page_size, head_dim, a.page_strides, dtype), t = (size_t)n_tokens * 4;
    const std::initializer_list<Range> ins = {{k_new, rows[0], "k_new"}, {v_new, rows[1], "v_new"}, {slots, t, "slots"}};
    if (apart("paged_append", {{k_pages, pool, "k_pages"}}, ins) || apart("paged_append", {{v_pages, pool, "v_pages"}}, ins)) return 1;
    const uintptr_t at[2] = {(uintptr_t)k_pages, (uintptr_t)v_pages};
    TROCM_REQUIRE(!ranges_meet(k_pages, pool, v_pages, pool) || interleaved(std::max(at[0], at[1]) - std::min(at[0], at[1]), n_pages, kv_heads, page_size, head_dim, a.page_strides, dtype),
                  "paged_append: v_pages overlaps k_pages");
    if (aligned("paged_append", {{k_new, 0, "k_new"}, {v_new, 0, "v_new"}, {k_pages, 0, "k_pages"}, {v_pages, 0, "v_pages"}}, elem_bytes(dtype))) return 1;
    if (aligned("paged_append", {{slots, t, "slots"}}, 4)) return 1;
    hipStream_t s;
    if (resolve_stream(stream, &s)) return 1;
    a.src[0] = k_new, a.src[1] = v_new, a.dst[0] = k_pages, a.dst[1] = v_pages, a.dtype = dtype;
    a.n_tokens = n_tokens, a.kv_heads = kv_heads, a.D = head_dim, a.n_pages = n_pages, a.page_size = page_size, a.slots = slots;
    return launch_paged_append(a, s);
}

int trocm_sdpa_paged_workspace_bytes(int64_t n_seq, int64_t q_heads, int64_t kv_heads, int64_t q_len, int64_t head_dim, size_t *bytes) {
    TROCM_NOT_NULL(bytes);
    TROCM_REQUIRE(n_seq >= 0 && q_heads >= 0 && kv_heads >= 1 && q_len >= 0 && head_dim >= 0, "sdpa_paged: negative dimension");
    TROCM_REQUIRE(q_heads % kv_heads == 0, "Q heads (%lld) must be a multiple of K/V heads (%lld)", (long long)q_heads, (long long)kv_heads);
    *bytes = sdpa_paged_workspace_bytes(n_seq, q_heads, kv_heads, q_len, head_dim);
    return 0;
}

int trocm_sdpa_paged(const void *q, int dtype, int64_t n_seq, int64_t q_heads, int64_t kv_heads, int64_t q_len, int64_t head_dim,
                     const void *k_pages, const void *v_pages, int64_t n_pages, int64_t page_size, const int64_t *page_strides,
                     const int32_t *table, int64_t table_width, const int32_t *lens, void *out, float scale, int causal, void *workspace,
                     size_t workspace_bytes, void *stream) {
    int64_t st[3];
    if (pages_check("sdpa_paged", n_pages, page_size) || table_check("sdpa_paged", n_seq, table_width, page_size, (1 << 24) - 1)) return 1;
    TROCM_REQUIRE(q_heads >= 0 && kv_heads >= 1 && q_len >= 0, "sdpa_paged: negative dimension");
    if (page_strides_check("sdpa_paged", dtype, n_pages, kv_heads, head_dim, page_size, page_strides, st)) return 1;
    TROCM_REQUIRE(q_heads % kv_heads == 0, "Q heads (%lld) must be a multiple of K/V heads (%lld)", (long long)q_heads, (long long)kv_heads);
    TROCM_REQUIRE(q_heads < (1 << 24) && q_len < (1 << 24) && q_heads * q_len < (1ll << 30) && n_seq * q_heads * q_len < (1ll << 31), "sdpa_paged: tensor too large");
    if (n_seq == 0 || q_heads == 0 || q_len == 0 || head_dim == 0) return 0;
    TROCM_NOT_NULL(q);
    TROCM_NOT_NULL(out);
    TROCM_NOT_NULL(lens);
    if (n_pages) {
        TROCM_NOT_NULL(k_pages);
        TROCM_NOT_NULL(v_pages);
    }
    if (table_width) TROCM_NOT_NULL(table);
    const size_t q_bytes = (size_t)(n_seq * q_heads * q_len * head_dim) * elem_bytes(dtype), pool = pool_bytes(n_pages, kv_heads, page_size, head_dim, st, dtype);
    if (apart("sdpa_paged", {{out, q_bytes, "out"}, {workspace, workspace_bytes, "workspace"}}, {{q, q_bytes, "q"}, {k_pages, pool, "k_pages"}, {v_pages, pool, "v_pages"},
                                                     {table, (size_t)n_seq * (size_t)table_width * 4, "table"}, {lens, (size_t)n_seq * 4, "lens"}})) return 1;
    if (aligned("sdpa_paged", {{q, 0, "q"}, {out, 0, "out"}, {k_pages, 0, "k_pages"}, {v_pages, 0, "v_pages"}}, elem_bytes(dtype))) return 1;
    if (aligned("sdpa_paged", {{table, 0, "table"}, {lens, 0, "lens"}}, 4)) return 1;
    TROCM_REQUIRE((uintptr_t)workspace % 16 == 0, "sdpa_paged: workspace must be 16-byte aligned");
    hipStream_t s;
    if (resolve_stream(stream, &s)) return 1;
    SdpaPagedArgs a;
    a.q = q, a.out = out, a.dtype = dtype, a.B = n_seq, a.Hq = q_heads, a.Hkv = kv_heads, a.Sq = q_len, a.D = head_dim;
    a.k = k_pages, a.v = v_pages, a.n_pages = n_pages, a.page_size = page_size, a.stride_page = st[0], a.stride_h = st[1], a.stride_t = st[2];
    a.table = table, a.table_width = table_width, a.lens = lens;
    a.scale = isnan(scale) ? 1.0f / sqrtf((float)head_dim) : scale, a.causal = causal != 0;
    a.workspace = workspace, a.workspace_bytes = workspace_bytes;
    return launch_sdpa_paged(a, s);
}

int trocm_paged_reorder(const int32_t *parents, int64_t n_seq, int64_t page_size, const int32_t *table, int64_t table_width, const int32_t *lens,
                        const int32_t *refs, const int32_t *free_pages, const int32_t *free_count, int64_t n_pages, int32_t *table_out,
                        int32_t *lens_out, int32_t *refs_out, int32_t *free_pages_out, int32_t *free_count_out, int32_t *copies,
                        int32_t *missing, void *stream) {
    if (pages_check("paged_reorder", n_pages, page_size) || table_check("paged_reorder", n_seq, table_width, page_size, kPagedMaxSeqs)) return 1;
    TROCM_REQUIRE(n_pages <= kMostReclaimed, "paged_reorder: %lld pages are more than 2^24", (long long)n_pages);   // (every 16384 of them count all others')
    if (n_seq) {
        TROCM_NOT_NULL(parents);
        TROCM_NOT_NULL(lens);
        TROCM_NOT_NULL(lens_out);
        TROCM_NOT_NULL(copies);
        if (table_width) TROCM_NOT_NULL(table);
        if (table_width) TROCM_NOT_NULL(table_out);
    }
    if (n_pages) {
        TROCM_NOT_NULL(refs);
        TROCM_NOT_NULL(free_pages);
        TROCM_NOT_NULL(refs_out);
        TROCM_NOT_NULL(free_pages_out);
    }
    TROCM_NOT_NULL(free_count);
    TROCM_NOT_NULL(free_count_out);
    TROCM_NOT_NULL(missing);
    const size_t n = (size_t)n_seq * 4, f = (size_t)n_pages * 4, rows = n * (size_t)table_width;
    const std::initializer_list<Range> outs = {{table_out, rows, "table_out"}, {lens_out, n, "lens_out"}, {refs_out, f, "refs_out"}, {free_pages_out, f, "free_pages_out"},
                                               {free_count_out, 4, "free_count_out"}, {copies, 3 * n, "copies"}, {missing, 4, "missing"}},
                                       ins = {{parents, n, "parents"}, {table, rows, "table"}, {lens, n, "lens"}, {refs, f, "refs"}, {free_pages, f, "free_pages"}, {free_count, 4, "free_count"}};
    if (apart("paged_reorder", outs, ins) || aligned("paged_reorder", outs, 4) || aligned("paged_reorder", ins, 4)) return 1;
    hipStream_t s;
    if (resolve_stream(stream, &s)) return 1;
    PagedReorderArgs a;
    a.parents = parents, a.table = table, a.lens = lens, a.refs = refs, a.free_pages = free_pages, a.free_count = free_count;
    a.table_out = table_out, a.lens_out = lens_out, a.refs_out = refs_out, a.free_pages_out = free_pages_out, a.free_count_out = free_count_out;
    a.copies = copies, a.missing = missing;
    a.n_seq = n_seq, a.page_size = page_size, a.table_width = table_width, a.n_pages = n_pages;
    return launch_paged_reorder(a, s);
}

int trocm_paged_copy(const int32_t *copies, int64_t n_copies, void *const *pools, int64_t n_pools, int dtype, int64_t kv_heads, int64_t head_dim,
                     int64_t n_pages, int64_t page_size, const int64_t *page_strides, void *stream) {
    PagedCopyArgs a;
    if (pages_check("paged_copy", n_pages, page_size)) return 1;
    if (page_strides_check("paged_copy", dtype, n_pages, kv_heads, head_dim, page_size, page_strides, a.page_strides)) return 1;
    TROCM_REQUIRE(n_copies >= 0 && n_pools >= 0, "paged_copy: negative dimension");
    TROCM_REQUIRE(n_copies <= (1 << 22), "paged_copy: %lld entries are more than 2^22", (long long)n_copies);
    if (n_copies == 0 || n_pools == 0 || n_pages == 0) return 0;
    TROCM_NOT_NULL(copies);
    TROCM_NOT_NULL(pools);
    const size_t bytes = pool_bytes(n_pages, kv_heads, page_size, head_dim, a.page_strides, dtype);
    for (int64_t i = 0; i < n_pools; i++) {
        TROCM_REQUIRE(pools[i] != nullptr, "paged_copy: pool %lld is null", (long long)i);
        if (aligned("paged_copy", {{pools[i], 0, "a pool"}}, elem_bytes(dtype)) || apart("paged_copy", {{pools[i], bytes, "a pool"}}, {{copies, (size_t)n_copies * 12, "copies"}})) return 1;
    }
    if (aligned("paged_copy", {{copies, 0, "copies"}}, 4)) return 1;
    hipStream_t s;
    if (resolve_stream(stream, &s)) return 1;
    a.copies = copies, a.pools = pools, a.dtype = dtype, a.n_copies = n_copies, a.n_pools = n_pools, a.kv_heads = kv_heads, a.D = head_dim;
    a.n_pages = n_pages, a.page_size = page_size;
    return launch_paged_copy(a, s);
}

static int beam_check(int64_t batch, int64_t beams, int64_t vocab, int64_t keep) {
    TROCM_REQUIRE(batch >= 0, "beam_select: negative dimension");
    TROCM_REQUIRE(beams >= 1 && beams <= kBeamMaxBeams, "beam_select: beams must be 1 to %d (got %lld)", kBeamMaxBeams, (long long)beams);
    TROCM_REQUIRE(keep >= 1 && keep <= kBeamMaxKeep, "beam_select: keep must be 1 to %d (got %lld)", kBeamMaxKeep, (long long)keep);
    TROCM_REQUIRE(vocab >= 1 && vocab <= kMostTokens && beams * vocab < (1ll << 31), "beam_select: vocab must be 1 to 2^30, beams * vocab below 2^31");
    TROCM_REQUIRE(keep <= beams * vocab, "beam_select: %lld of %lld continuations asked for", (long long)keep, (long long)(beams * vocab));
    TROCM_REQUIRE(batch < (1 << 24) && batch * beams < (1 << 24), "beam_select: tensor too large");
    return 0;
}

int trocm_beam_select_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int64_t keep, size_t *bytes) {
    TROCM_NOT_NULL(bytes);
    if (beam_check(batch, beams, vocab, keep)) return 1;
    *bytes = beam_select_workspace_bytes(batch, beams, vocab, keep);
    return 0;
}

int trocm_beam_select(const void *logits, int dtype, int64_t batch, int64_t beams, int64_t vocab, int64_t row_stride, const float *scores,
                      const int32_t *ended, int32_t eos, int64_t keep, float *scores_out, int32_t *parents, int32_t *tokens, int32_t *ended_out,
                      void *workspace, size_t workspace_bytes, void *stream) {
    TROCM_REQUIRE(dtype == TROCM_F32 || dtype == TROCM_F16, "beam_select: dtype must be F32 or F16");
    if (beam_check(batch, beams, vocab, keep)) return 1;
    if (row_stride == 0) row_stride = vocab;
    TROCM_REQUIRE(row_stride >= vocab && within_reach(std::max<int64_t>(batch * beams, 1), row_stride), "beam_select: row_stride %lld does not hold a row of %lld", (long long)row_stride, (long long)vocab);
    TROCM_REQUIRE(eos >= -1 && eos < vocab, "beam_select: eos must be -1 or a token (got %d)", eos);
    TROCM_REQUIRE(!ended || eos >= 0, "beam_select: beams that have ended need eos");
    if (batch == 0) return 0;
    TROCM_NOT_NULL(logits);
    TROCM_NOT_NULL(scores);
    TROCM_NOT_NULL(scores_out);
    TROCM_NOT_NULL(parents);
    TROCM_NOT_NULL(tokens);
    TROCM_NOT_NULL(workspace);
    const size_t es = elem_bytes(dtype), out = (size_t)(batch * keep) * 4, in = (size_t)(batch * beams) * 4;
    if (apart("beam_select", {{scores_out, out, "scores_out"}, {parents, out, "parents"}, {tokens, out, "tokens"}, {ended_out, out, "ended_out"}, {workspace, workspace_bytes, "workspace"}},
              {{logits, (size_t)((batch * beams - 1) * row_stride + vocab) * es, "logits"}, {scores, in, "scores"}, {ended, in, "ended"}})) return 1;
    if (aligned("beam_select", {{logits, 0, "logits"}}, es)) return 1;
    if (aligned("beam_select", {{scores, 0, "scores"}, {ended, 0, "ended"}, {scores_out, 0, "scores_out"}, {parents, 0, "parents"}, {tokens, 0, "tokens"}, {ended_out, 0, "ended_out"}}, 4)) return 1;
    TROCM_REQUIRE((uintptr_t)workspace % 16 == 0, "beam_select: workspace must be 16-byte aligned");
    hipStream_t s;
    if (resolve_stream(stream, &s)) return 1;
    BeamSelectArgs a;
    a.logits = logits, a.dtype = dtype, a.batch = batch, a.beams = beams, a.vocab = vocab, a.row_stride = row_stride, a.keep = keep;
    a.scores = scores, a.ended = ended, a.eos = eos, a.scores_out = scores_out, a.parents = parents, a.tokens = tokens, a.ended_out = ended_out;
    a.workspace = workspace, a.workspace_bytes = workspace_bytes;
    return launch_beam_select(a, s);
}

}  // extern "C"
