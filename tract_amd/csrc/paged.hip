// Pages of keys and values that many sequences share: the tables of a step, built on the device from the sequences' lengths; the append
// of new rows through them; sequences that go on from other sequences, and the copies of the pages that those cannot share.
//
// All state (lengths, tables, counts of holders, the stack of free pages) is read and written by kernels alone, so a step can be
// recorded once and replayed.  Every id that comes from device memory is checked before it becomes an address.
#include <algorithm>
#include "common.h"
#include "fast_div.h"

namespace trocm {
namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kSumTop = 1 << 30;   // where sums of lengths stay (adding never wraps)

__device__ __forceinline__ int add_up_to_top(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)kSumTop); }   // (both of 0 ..= kSumTop)

// Exclusive prefix sums of a value per thread over the workgroup; `total` is the sum.  All threads.
__device__ __forceinline__ int block_scan(int x, int *lds_waves, int &total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, waves = blockDim.x >> 6;
    int up = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(up, d, 64);
        if (lane >= d) up = add_up_to_top(up, y);
    }
    __syncthreads();   // (lds_waves may still be read from the scan before)
    if (lane == 63) lds_waves[w] = up;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int i = 0; i < waves; i++) {
        if (i == w) before = total;
        total = add_up_to_top(total, lds_waves[i]);
    }
    const int left = __shfl_up(up, 1, 64);
    return add_up_to_top(before, lane ? left : 0);
}

// The first place of a sorted a[0, n) that is larger than x; n if none is.
__device__ __forceinline__ int first_above(const int *a, int n, int x) {
    int lo = 0;
    for (int len = n; len > 0;) {
        const int half = len >> 1;
        if (a[lo + half] <= x) lo += half + 1, len -= half + 1;
        else len = half;
    }
    return lo;
}

struct PlanDev {
    const int *lens, *n_new, *free_pages, *free_count;
    int *table, *refs, *lens_out, *starts, *slots, *positions, *free_count_out, *refused;
    int64_t table_width;
    int n_seq, n_pages, n_tokens, most;   // most: tokens that a table's row has pages for
    FastDiv by_page;
};

// Pages of the step and where its tokens go.  Every workgroup makes the prefix sums over the sequences itself (at most four a thread)
// and takes its share of the tokens and pages, so that no workgroup waits for another.
__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PlanDev p) {
    __shared__ int s_ends[kPagedMaxSeqs], s_offs[kPagedMaxSeqs + 1], s_waves[kPlanWaves];
    const int tid = threadIdx.x, page = (int)p.by_page.d;
    const int per = (p.n_seq + blockDim.x - 1) / blockDim.x, i0 = min(tid * per, p.n_seq), i1 = min(i0 + per, p.n_seq);
    const int count = min(max(p.free_count[0], 0), p.n_pages);
    auto pages_of = [&](int tokens) { return p.by_page.by(tokens + page - 1); };
    // (tokens + page - 1 stays below 2^31: `most` is at most 2^30 and a page at most 2^20 tokens)
    auto fits = [&](int len, int add, int end) { return len >= 0 && add >= 0 && len <= p.most && add <= p.most - len && end <= p.n_tokens; };

    int sum = 0, total;
    for (int i = i0; i < i1; i++) sum = add_up_to_top(sum, min(max(p.n_new[i], 0), kSumTop));
    int at = block_scan(sum, s_waves, total);
    int needs = 0;
    const int start = at;
    for (int i = i0; i < i1; i++) {
        const int len = p.lens[i], add = p.n_new[i];
        if (blockIdx.x == 0 && p.starts) p.starts[i] = at;
        at = add_up_to_top(at, min(max(add, 0), kSumTop));
        s_ends[i] = at;
        if (fits(len, add, at)) needs = add_up_to_top(needs, pages_of(len + add) - pages_of(len));
    }
    if (blockIdx.x == 0 && p.starts && tid == 0) p.starts[p.n_seq] = total;
    int all_needs;
    int off = block_scan(needs, s_waves, all_needs);
    at = start;
    int refused = 0, taken = 0;
    for (int i = i0; i < i1; i++) {
        const int len = p.lens[i], add = p.n_new[i];
        at = add_up_to_top(at, min(max(add, 0), kSumTop));
        const bool fit = fits(len, add, at);
        const int need = fit ? pages_of(len + add) - pages_of(len) : 0;
        s_offs[i] = off;
        off = add_up_to_top(off, need);
        const bool in = fit && (need == 0 || off <= count);
        refused += !in;
        if (in) taken += need;
        if (blockIdx.x == 0) p.lens_out[i] = in ? len + add : len;
    }
    if (tid == 0) s_offs[p.n_seq] = all_needs;
    int all_taken, all_refused;
    block_scan(taken, s_waves, all_taken);
    block_scan(refused, s_waves, all_refused);   // (and what the threads wrote to LDS can be read)
    if (blockIdx.x == 0 && tid == 0) p.free_count_out[0] = count - all_taken, p.refused[0] = all_refused;

    // the pages taken, in the sequences' order, from the end of the stack
    for (int o = blockIdx.x * blockDim.x + tid; o < all_taken; o += gridDim.x * blockDim.x) {
        const int i = first_above(s_offs, p.n_seq + 1, o) - 1, id = p.free_pages[count - 1 - o];
        p.table[i * p.table_width + pages_of(p.lens[i]) + o - s_offs[i]] = id;
        if (p.refs && (unsigned)id < (unsigned)p.n_pages) p.refs[id] = 1;
    }
    // where the tokens go
    for (int t = blockIdx.x * blockDim.x + tid; t < p.n_tokens; t += gridDim.x * blockDim.x) {
        const int i = first_above(s_ends, p.n_seq, t);
        int slot = -1, pos = -1;
        if (i < p.n_seq) {
            const int len = p.lens[i], add = p.n_new[i], need = s_offs[i + 1] - s_offs[i];
            if (fits(len, add, s_ends[i]) && (need == 0 || s_offs[i + 1] <= count)) {
                pos = len + t - (s_ends[i] - add);
                const int pi = p.by_page.by(pos), have = pages_of(len);
                const int id = pi < have ? p.table[i * p.table_width + pi] : p.free_pages[count - 1 - (s_offs[i] + pi - have)];
                if ((unsigned)id < (unsigned)p.n_pages) slot = id * page + (pos - pi * page);
            }
        }
        p.slots[t] = slot;
        if (p.positions) p.positions[t] = pos;
    }
}

// ---- rows through a slot map -----------------------------------------------------------------------------------------

struct AppendDev {
    const char *src[2];
    char *dst[2];
    int64_t src_token[2], src_head[2], dst_page, dst_head, dst_token;   // bytes
    const int *slots;
    int n_tokens, n_slots, words_per_token, tokens_per_block;
    FastDiv by_words_per_token, by_words_per_row, by_page;
};

// A word of a K row and the same of the V row per thread and turn; W is the widest word that divides rows and addresses.  Workgroups
// take several tokens where those are short.
template <typename W>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendDev p) {
    const int t0 = blockIdx.x * p.tokens_per_block, words = min(p.tokens_per_block, p.n_tokens - t0) * p.words_per_token;
#pragma unroll 4
    for (int x = threadIdx.x; x < words; x += 256) {
        const int t = p.by_words_per_token.by(x), in_token = x - t * p.words_per_token;
        const int h = p.by_words_per_row.by(in_token), c = in_token - h * (int)p.by_words_per_row.d;
        const int slot = p.slots[t0 + t];
        if ((unsigned)slot >= (unsigned)p.n_slots) continue;
        const int pg = p.by_page.by(slot), r = slot - pg * (int)p.by_page.d;
        const int64_t to = pg * p.dst_page + h * p.dst_head + r * p.dst_token + (int64_t)c * (int64_t)sizeof(W);
#pragma unroll
        for (int y = 0; y < 2; y++)
            *reinterpret_cast<W *>(p.dst[y] + to) = *reinterpret_cast<const W *>(p.src[y] + (t0 + t) * p.src_token[y] + h * p.src_head[y] + (int64_t)c * (int64_t)sizeof(W));
    }
}

// ---- sequences that go on from others ----------------------------------------------------------------------------------

struct ReorderDev {
    const int *parents, *table, *lens, *refs, *free_pages, *free_count;
    int *table_out, *lens_out, *refs_out, *free_pages_out, *free_count_out, *copies, *missing;
    int64_t table_width;
    int n_seq, n_pages, most;
    FastDiv by_page;
};

// What sequence s holds: full pages and the tokens of the partial one (0: none).  Lengths outside of the table hold nothing.
__device__ __forceinline__ int2 held_pages(const ReorderDev &p, int s) {
    const int len = p.lens[s];
    if (len < 0 || len > p.most) return make_int2(0, 0);
    const int full = p.by_page.by(len);
    return make_int2(full, len - full * (int)p.by_page.d);
}

// First launch.  Workgroup 0: who needs a copy of the partial page and which free page takes it; the others: counts of holders as they were.
__global__ __launch_bounds__(kPlanThreads) void paged_reorder_begin_kernel(ReorderDev p) {
    const int tid = threadIdx.x;
    if (blockIdx.x > 0) {
        const int x = (blockIdx.x - 1) * kPlanThreads + tid;
        if (x < p.n_pages) p.refs_out[x] = p.refs[x];
        return;
    }
    __shared__ int s_first[kPagedMaxSeqs], s_waves[kPlanWaves];
    for (int s = tid; s < p.n_seq; s += kPlanThreads) s_first[s] = p.n_seq;
    __syncthreads();
    for (int j = tid; j < p.n_seq; j += kPlanThreads) {
        const int from = p.parents[j];
        if ((unsigned)from < (unsigned)p.n_seq) atomicMin(&s_first[from], j);
    }
    __syncthreads();
    const int per = (p.n_seq + kPlanThreads - 1) / kPlanThreads, j0 = min(tid * per, p.n_seq), j1 = min(j0 + per, p.n_seq);
    const int count = min(max(p.free_count[0], 0), p.n_pages);
    // (partial page, its tokens) where sequence j needs a copy of it, else (-1, 0)
    auto copied = [&](int j) {
        const int from = p.parents[j];
        if ((unsigned)from >= (unsigned)p.n_seq) return make_int2(-1, 0);
        const int2 held = held_pages(p, from);
        if (held.y == 0) return make_int2(-1, 0);
        const int id = p.table[from * p.table_width + held.x];
        if ((unsigned)id >= (unsigned)p.n_pages || (s_first[from] == j && p.refs[id] == 1)) return make_int2(-1, 0);
        return make_int2(id, held.y);
    };
    int mine = 0, total;
    for (int j = j0; j < j1; j++) mine += copied(j).x >= 0;
    int at = block_scan(mine, s_waves, total);
    const bool enough = total <= count;
    for (int j = j0; j < j1; j++) {
        const int2 c = copied(j);
        int *out = p.copies + 3 * j;
        const bool go = enough && c.x >= 0;
        out[0] = go ? c.x : -1, out[1] = go ? p.free_pages[count - 1 - at] : -1, out[2] = go ? c.y : 0;
        at += c.x >= 0;
        const int from = p.parents[j];
        p.lens_out[j] = !enough ? p.lens[j] : (unsigned)from < (unsigned)p.n_seq ? p.lens[from] : 0;
    }
    if (tid == 0) p.missing[0] = enough ? 0 : total - count;
}

// Second launch, a workgroup per sequence: its new row of the table, and what its old row's pages lose or gain: a holder for every child
// but one.
__global__ __launch_bounds__(256) void paged_reorder_tables_kernel(ReorderDev p) {
    __shared__ int s_children[4];
    const int j = blockIdx.x, tid = threadIdx.x, width = (int)p.table_width;
    const int *old_row = p.table + j * p.table_width;
    int *row = p.table_out + j * p.table_width;
    if (p.missing[0] > 0) {   // nothing changes
        for (int x = tid; x < width; x += 256) row[x] = old_row[x];
        return;
    }
    const int from = p.parents[j];
    const bool there = (unsigned)from < (unsigned)p.n_seq;
    const int src = there ? from : j;
    int2 held = held_pages(p, src);
    if (!there) held = make_int2(0, 0);
    const int dst_page = p.copies[3 * j + 1], pages = held.x + (held.y > 0);
    const int *from_row = p.table + src * p.table_width;
    for (int x = tid; x < width; x += 256) row[x] = x >= pages ? -1 : x == held.x && dst_page >= 0 ? dst_page : from_row[x];
    if (tid == 0 && (unsigned)dst_page < (unsigned)p.n_pages) atomicAdd(&p.refs_out[dst_page], 1);

    int children = 0;
    for (int x = tid; x < p.n_seq; x += 256) children += p.parents[x] == j;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) children += __shfl_xor(children, d, 64);
    if ((tid & 63) == 0) s_children[tid >> 6] = children;
    __syncthreads();
    children = s_children[0] + s_children[1] + s_children[2] + s_children[3];
    const int2 mine = held_pages(p, j);
    if (children != 1) {
        for (int x = tid; x < mine.x; x += 256) {
            const int id = old_row[x];
            if ((unsigned)id < (unsigned)p.n_pages) atomicAdd(&p.refs_out[id], children - 1);
        }
    }
    if (tid == 0 && mine.y > 0) {   // the partial page stays with the first child, if nobody else holds it
        const int id = old_row[mine.x];
        if ((unsigned)id < (unsigned)p.n_pages && !(children > 0 && p.refs[id] == 1)) atomicAdd(&p.refs_out[id], -1);
    }
}

// Third launch: pages that nobody holds any more go onto the stack, in ascending order behind what is left of it.  A workgroup takes
// kReclaim pages and counts the freed ones of all others itself, so that none waits for another.
constexpr int kReclaim = 16 * kPlanThreads;
__global__ __launch_bounds__(kPlanThreads) void paged_reclaim_kernel(ReorderDev p) {
    __shared__ int s_waves[kPlanWaves];
    const int tid = threadIdx.x;
    int taken = 0, n;
    for (int j = tid; j < p.n_seq; j += kPlanThreads) taken += p.copies[3 * j] >= 0;
    block_scan(taken, s_waves, n);
    const int left = min(max(p.free_count[0], 0), p.n_pages) - n;
    auto freed = [&](int x) { return x < p.n_pages && p.refs_out[x] <= 0 && p.refs[x] > 0; };
    int before = 0, all = 0, mine = 0;
    const int my0 = blockIdx.x * kReclaim + tid * 16;
    for (int x0 = 0; x0 < p.n_pages; x0 += kReclaim) {
        int here = 0;
        for (int x = 0; x < 16; x++) here += freed(x0 + tid * 16 + x);
        if (x0 < (int)blockIdx.x * kReclaim) before += here;
        if (x0 == (int)blockIdx.x * kReclaim) mine = here;
        all += here;
    }
    int sum_before, sum_all, unused;
    block_scan(before, s_waves, sum_before);
    block_scan(all, s_waves, sum_all);
    int at = left + sum_before + block_scan(mine, s_waves, unused);
    for (int x = my0; x < my0 + 16; x++)
        if (freed(x) && at < p.n_pages) p.free_pages_out[at++] = x;   // (more free pages than there are pages: counts that were not kept)
    for (int x = blockIdx.x * kReclaim + tid; x < min(p.n_pages, ((int)blockIdx.x + 1) * kReclaim); x += kPlanThreads) {
        if (x < left) p.free_pages_out[x] = p.free_pages[x];
        else if (x >= left + sum_all) p.free_pages_out[x] = -1;
    }
    if (blockIdx.x == 0 && tid == 0) p.free_count_out[0] = min(left + sum_all, p.n_pages);
}

// ---- copies of pages ------------------------------------------------------------------------------------------------------

struct CopyDev {
    char *pools[kPagedMaxPools];
    const int *copies;
    int64_t page_stride, head_stride, token_stride;   // bytes
    int n_pages, page, heads, words_per_row;
    FastDiv by_words_per_row;
};

// A workgroup per copy, pool and head group.
template <typename W>
__global__ __launch_bounds__(256) void paged_copy_kernel(CopyDev p) {
    const int *c = p.copies + 3 * (int64_t)blockIdx.x;
    const int from = c[0], to = c[1], tokens = min(c[2], p.page);
    if ((unsigned)from >= (unsigned)p.n_pages || (unsigned)to >= (unsigned)p.n_pages || from == to || tokens <= 0) return;
    // (the pointer where the arguments lie: asked of the argument itself, the compiler copies all of them into every lane's scratch)
    typedef const __attribute__((address_space(4))) uint64_t *Words;
    char *pool = reinterpret_cast<char *>(reinterpret_cast<Words>(reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr()))[blockIdx.y]);
    const char *src = pool + from * p.page_stride;
    char *dst = pool + to * p.page_stride;
    const int words_per_head = tokens * p.words_per_row;
    for (int h = blockIdx.z; h < p.heads; h += gridDim.z)
        for (int x = threadIdx.x; x < words_per_head; x += 256) {
            const int r = p.by_words_per_row.by(x), w = x - r * p.words_per_row;
            const int64_t at = h * p.head_stride + r * p.token_stride + (int64_t)w * (int64_t)sizeof(W);
            *reinterpret_cast<W *>(dst + at) = *reinterpret_cast<const W *>(src + at);
        }
}

}  // namespace

int launch_paged_plan(const PagedPlanArgs &a, hipStream_t s) {
    PlanDev p;
    p.lens = a.lens, p.n_new = a.n_new, p.free_pages = a.free_pages, p.free_count = a.free_count;
    p.table = a.table, p.refs = a.refs, p.lens_out = a.lens_out, p.starts = a.starts, p.slots = a.slots, p.positions = a.positions;
    p.free_count_out = a.free_count_out, p.refused = a.refused;
    p.table_width = a.table_width, p.n_seq = (int)a.n_seq, p.n_pages = (int)a.n_pages, p.n_tokens = (int)a.n_tokens;
    p.most = (int)std::min<int64_t>(a.table_width * a.page_size, kSumTop);
    p.by_page = fast_div(a.page_size);
    const int64_t blocks = std::min<int64_t>(std::max<int64_t>((a.n_tokens + kPlanThreads - 1) / kPlanThreads, 1), 256);
    paged_plan_kernel<<<dim3((unsigned)blocks), kPlanThreads, 0, s>>>(p);
    TROCM_HIP(hipGetLastError());
    return 0;
}

// Bytes of the widest word (16, 4 or 2) that divides all of `bits`: addresses, strides and row lengths or'ed together.
static int word_of(uint64_t bits) { return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2; }

int launch_paged_append(const PagedAppendArgs &a, hipStream_t s) {
    if (a.n_tokens == 0 || a.kv_heads == 0 || a.D == 0) return 0;
    const int64_t es = (int64_t)elem_bytes(a.dtype);
    AppendDev p;
    uint64_t bits = (uint64_t)(a.D * es);
    for (int y = 0; y < 2; y++) {
        p.src[y] = (const char *)a.src[y], p.dst[y] = (char *)a.dst[y];
        p.src_token[y] = a.src_strides[y][0] * es, p.src_head[y] = a.src_strides[y][1] * es;
        bits |= (uint64_t)p.src_token[y] | (uint64_t)p.src_head[y] | (uint64_t)(uintptr_t)p.src[y] | (uint64_t)(uintptr_t)p.dst[y];
    }
    p.dst_page = a.page_strides[0] * es, p.dst_head = a.page_strides[1] * es, p.dst_token = a.page_strides[2] * es;
    bits |= (uint64_t)p.dst_page | (uint64_t)p.dst_head | (uint64_t)p.dst_token;
    const int word = word_of(bits);
    p.slots = a.slots, p.n_tokens = (int)a.n_tokens, p.n_slots = (int)(a.n_pages * a.page_size);
    p.words_per_token = (int)(a.kv_heads * a.D * es / word);
    p.tokens_per_block = std::max(1, 1024 / p.words_per_token);
    p.by_words_per_token = fast_div(p.words_per_token), p.by_words_per_row = fast_div(a.D * es / word), p.by_page = fast_div(a.page_size);
    const dim3 grid((unsigned)((a.n_tokens + p.tokens_per_block - 1) / p.tokens_per_block));
    if (word == 16) paged_append_kernel<uint4><<<grid, 256, 0, s>>>(p);
    else if (word == 4) paged_append_kernel<uint32_t><<<grid, 256, 0, s>>>(p);
    else paged_append_kernel<uint16_t><<<grid, 256, 0, s>>>(p);
    TROCM_HIP(hipGetLastError());
    return 0;
}

int launch_paged_reorder(const PagedReorderArgs &a, hipStream_t s) {
    ReorderDev p;
    p.parents = a.parents, p.table = a.table, p.lens = a.lens, p.refs = a.refs, p.free_pages = a.free_pages, p.free_count = a.free_count;
    p.table_out = a.table_out, p.lens_out = a.lens_out, p.refs_out = a.refs_out, p.free_pages_out = a.free_pages_out;
    p.free_count_out = a.free_count_out, p.copies = a.copies, p.missing = a.missing;
    p.table_width = a.table_width, p.n_seq = (int)a.n_seq, p.n_pages = (int)a.n_pages;
    p.most = (int)std::min<int64_t>(a.table_width * a.page_size, kSumTop);
    p.by_page = fast_div(a.page_size);
    paged_reorder_begin_kernel<<<dim3((unsigned)(1 + (a.n_pages + kPlanThreads - 1) / kPlanThreads)), kPlanThreads, 0, s>>>(p);
    TROCM_HIP(hipGetLastError());
    if (a.n_seq) paged_reorder_tables_kernel<<<dim3((unsigned)a.n_seq), 256, 0, s>>>(p);
    TROCM_HIP(hipGetLastError());
    paged_reclaim_kernel<<<dim3((unsigned)std::max<int64_t>((a.n_pages + kReclaim - 1) / kReclaim, 1)), kPlanThreads, 0, s>>>(p);
    TROCM_HIP(hipGetLastError());
    return 0;
}

int launch_paged_copy(const PagedCopyArgs &a, hipStream_t s) {
    if (a.n_copies == 0 || a.n_pools == 0 || a.kv_heads == 0 || a.D == 0 || a.n_pages == 0) return 0;
    const int64_t es = (int64_t)elem_bytes(a.dtype);
    for (int64_t first = 0; first < a.n_pools; first += kPagedMaxPools) {
        CopyDev p;
        const int n = (int)std::min<int64_t>(a.n_pools - first, kPagedMaxPools);
        uint64_t bits = (uint64_t)(a.D * es);
        for (int i = 0; i < kPagedMaxPools; i++) {
            p.pools[i] = i < n ? (char *)a.pools[first + i] : nullptr;
            bits |= (uint64_t)(uintptr_t)p.pools[i];
        }
        p.copies = a.copies;
        p.page_stride = a.page_strides[0] * es, p.head_stride = a.page_strides[1] * es, p.token_stride = a.page_strides[2] * es;
        bits |= (uint64_t)p.page_stride | (uint64_t)p.head_stride | (uint64_t)p.token_stride;
        const int word = word_of(bits);
        p.n_pages = (int)a.n_pages, p.page = (int)a.page_size, p.heads = (int)a.kv_heads, p.words_per_row = (int)(a.D * es / word);
        p.by_words_per_row = fast_div(p.words_per_row);
        const dim3 grid((unsigned)a.n_copies, (unsigned)n, (unsigned)std::min<int64_t>(a.kv_heads, 64));
        if (word == 16) paged_copy_kernel<uint4><<<grid, 256, 0, s>>>(p);
        else if (word == 4) paged_copy_kernel<uint32_t><<<grid, 256, 0, s>>>(p);
        else paged_copy_kernel<uint16_t><<<grid, 256, 0, s>>>(p);
        TROCM_HIP(hipGetLastError());
    }
    return 0;
}

}  // namespace trocm
