// Pages of keys and values that many sequences share: the tables of a step, built on the device from the sequences' lengths; the append
// of new rows through them; sequences that go on from other sequences, and the copies of the pages that those cannot share.
//
// All state (lengths, tables, counts of holders, the stack of free pages) is read and written by kernels alone, so a step can be
// recorded once and replayed.  Every id that comes from device memory is checked before it becomes an address.
//
// Tables are kilobytes: what bounds plan and reorder is the chain of dependent accesses and barriers (a plan of 256 sequences 5.1 us, 4.4 of
// them the kernel's; 4 beams reordered 11 us in two launches with the copy, 256 beams in eight layers 25 in four).  Prefix sums go along the
// lanes (shuffles through LDS: 6.9 us for the plan, then 5.5).  The append and the copies are bound by their bytes.
#include <algorithm>
#include "common.h"
#include "fast_div.h"

namespace trocm {
namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kSumTop = 1 << 30;   // where sums of lengths stay (adding never wraps)

__device__ __forceinline__ int add_up_to_top(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)kSumTop); }   // (both of 0 ..= kSumTop)

// Lane l's value to lane l + n of a row of 16, lane 15's of a row to the next row, lane 31's to the upper half; 0 where none comes.
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
constexpr int kUp = 0x110, kRow15 = 0x142, kRow31 = 0x143;
__device__ __forceinline__ int row_sums(int x) {   // of a row's lanes up to this one
    x = add_up_to_top(x, moved<kUp + 1, 0xf>(x)), x = add_up_to_top(x, moved<kUp + 2, 0xf>(x));
    x = add_up_to_top(x, moved<kUp + 4, 0xf>(x)), x = add_up_to_top(x, moved<kUp + 8, 0xf>(x));
    return x;
}
__device__ __forceinline__ int wave_sums(int x) {   // of a wave's
    x = row_sums(x);
    x = add_up_to_top(x, moved<kRow15, 0xa>(x));
    return add_up_to_top(x, moved<kRow31, 0xc>(x));
}
__device__ __forceinline__ int wave_most(int x) {   // of values that are not negative
    x = max(x, moved<kUp + 1, 0xf>(x)), x = max(x, moved<kUp + 2, 0xf>(x)), x = max(x, moved<kUp + 4, 0xf>(x)), x = max(x, moved<kUp + 8, 0xf>(x));
    x = max(x, moved<kRow15, 0xa>(x)), x = max(x, moved<kRow31, 0xc>(x));
    return __builtin_amdgcn_readlane(x, 63);
}

// Exclusive prefix sums of a value per thread over the workgroup; `total` is the sum.  All threads; lds_waves[16] may be used again after the
// next barrier.
__device__ __forceinline__ int block_scan(int x, int *lds_waves, int &total) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int up = wave_sums(x);
    if (lane == 63) lds_waves[w] = up;
    __syncthreads();
    const int sums = row_sums(lane < waves ? lds_waves[lane] : 0);   // (at most 16 waves)
    total = __builtin_amdgcn_readlane(sums, 15);
    const int before = w ? __builtin_amdgcn_readlane(sums, w - 1) : 0;
    const int left = __shfl_up(up, 1, 64);   // (not up - x: sums stop at the top)
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
    __shared__ int s_ends[kPagedMaxSeqs], s_offs[kPagedMaxSeqs + 1], s_lens[kPagedMaxSeqs];   // s_lens: -1 of a sequence that is refused
    __shared__ int s_waves[2][kPlanWaves], s_taken, s_refused;
    constexpr int kMine = kPagedMaxSeqs / kPlanThreads;
    const int tid = threadIdx.x, lane = tid & 63, page = (int)p.by_page.d;
    const int per = (p.n_seq + kPlanThreads - 1) / kPlanThreads, i0 = min(tid * per, p.n_seq), mine = min(per, p.n_seq - i0);
    const int count = min(max(p.free_count[0], 0), p.n_pages);
    auto pages_of = [&](int tokens) { return p.by_page.by(tokens + page - 1); };   // (below 2^31: `most` is at most 2^30 and a page at most 2^20 tokens)
    int len[kMine], add[kMine], need[kMine];
#pragma unroll
    for (int y = 0; y < kMine; y++) len[y] = y < mine ? p.lens[i0 + y] : 0, add[y] = y < mine ? p.n_new[i0 + y] : 0;
    if (tid == 0) s_taken = 0, s_refused = 0;

    int sum = 0, total, all_needs;
#pragma unroll
    for (int y = 0; y < kMine; y++) sum = add_up_to_top(sum, min(max(add[y], 0), kSumTop));
    int at = block_scan(sum, s_waves[0], total);
    int needs = 0;
    uint32_t fits = 0;
#pragma unroll
    for (int y = 0; y < kMine; y++) {
        if (y < mine && blockIdx.x == 0 && p.starts) p.starts[i0 + y] = at;
        const int rows = p.n_tokens - at;   // that are left (not by where it ends: sums stop at 2^30, which may be n_tokens)
        at = add_up_to_top(at, min(max(add[y], 0), kSumTop));
        if (y < mine) s_ends[i0 + y] = at;
        const bool fit = y < mine && len[y] >= 0 && add[y] >= 0 && len[y] <= p.most && add[y] <= p.most - len[y] && add[y] <= rows;
        fits |= (fit ? 1u : 0u) << y;
        need[y] = fit ? pages_of(len[y] + add[y]) - pages_of(len[y]) : 0;
        needs = add_up_to_top(needs, need[y]);
    }
    if (blockIdx.x == 0 && p.starts && tid == 0) p.starts[p.n_seq] = total;
    int off = block_scan(needs, s_waves[1], all_needs);
    int refused = 0, taken = 0;   // (what is taken ends where the last sequence that gets pages ends)
#pragma unroll
    for (int y = 0; y < kMine; y++) {
        if (y >= mine) continue;
        s_offs[i0 + y] = off;
        off = add_up_to_top(off, need[y]);
        const bool in = ((fits >> y) & 1) && (need[y] == 0 || off <= count);
        refused += !in;
        if (in && need[y]) taken = off;
        s_lens[i0 + y] = in ? len[y] : -1;
        if (blockIdx.x == 0) p.lens_out[i0 + y] = in ? len[y] + add[y] : len[y];
    }
    if (tid == 0) s_offs[p.n_seq] = all_needs;
    taken = wave_most(taken), refused = __builtin_amdgcn_readlane(wave_sums(refused), 63);
    if (lane == 0 && taken) atomicMax(&s_taken, taken);
    if (lane == 0 && refused) atomicAdd(&s_refused, refused);
    __syncthreads();
    const int all_taken = s_taken;
    if (blockIdx.x == 0 && tid == 0) p.free_count_out[0] = count - all_taken, p.refused[0] = s_refused;

    // the pages taken, in the sequences' order, from the end of the stack
    for (int o = blockIdx.x * kPlanThreads + tid; o < all_taken; o += gridDim.x * kPlanThreads) {
        const int id = p.free_pages[count - 1 - o], i = first_above(s_offs, p.n_seq + 1, o) - 1;
        p.table[i * p.table_width + pages_of(s_lens[i]) + o - s_offs[i]] = id;
        if (p.refs && (unsigned)id < (unsigned)p.n_pages) p.refs[id] = 1;
    }
    // where the tokens go
    for (int t = blockIdx.x * kPlanThreads + tid; t < p.n_tokens; t += gridDim.x * kPlanThreads) {
        const int i = first_above(s_ends, p.n_seq, t), held = i < p.n_seq ? s_lens[i] : -1;
        int slot = -1, pos = -1;
        if (held >= 0) {
            pos = held + t - (i ? s_ends[i - 1] : 0);
            const int pi = p.by_page.by(pos), have = pages_of(held);
            const int id = pi < have ? p.table[i * p.table_width + pi] : p.free_pages[count - 1 - (s_offs[i] + pi - have)];
            if ((unsigned)id < (unsigned)p.n_pages) slot = id * page + (pos - pi * page);
        }
        p.slots[t] = slot;
        if (p.positions) p.positions[t] = pos;
    }
}

typedef uint32_t Quad __attribute__((ext_vector_type(4)));

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
// take several tokens where those are short, and a thread's words of kTurns turns are all on their way before the first is stored.  Nothing
// is computed: the bytes of the rows, read and written, bound it.  Stores go past the caches: a row is read again by the attention at the
// earliest, mostly on another chip's L2.  16001 tokens of 8 heads of 128, f16, 131 MB: 21.9 us, 6.0 TB/s (through the caches 29.5, loads past
// them too 25.1); with the attention that reads all of them behind it, 16 x 1000 tokens 38.7 for 40.8, 32 x 256 24.3 for 24.1, 64 x 64 16.6
// for 17.2.
constexpr int kTurns = 4;
template <typename W>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendDev p) {
    const int t0 = blockIdx.x * p.tokens_per_block, words = min(p.tokens_per_block, p.n_tokens - t0) * p.words_per_token;
#pragma unroll 1
    for (int x0 = threadIdx.x; x0 < words; x0 += 256 * kTurns) {
        W word[kTurns][2];
        int64_t to[kTurns];   // < 0: nowhere
#pragma unroll
        for (int u = 0; u < kTurns; u++) {
            const int x = min(x0 + u * 256, words - 1);
            const int t = p.by_words_per_token.by(x), in_token = x - t * p.words_per_token;
            const int h = p.by_words_per_row.by(in_token), c = in_token - h * (int)p.by_words_per_row.d;
#pragma unroll
            for (int y = 0; y < 2; y++) word[u][y] = *reinterpret_cast<const W *>(p.src[y] + (t0 + t) * p.src_token[y] + h * p.src_head[y] + (int64_t)c * (int64_t)sizeof(W));
            const int slot = p.slots[t0 + t];
            const bool goes = x0 + u * 256 < words && (unsigned)slot < (unsigned)p.n_slots;
            const int pg = p.by_page.by(goes ? slot : 0), r = (goes ? slot : 0) - pg * (int)p.by_page.d;
            to[u] = goes ? pg * p.dst_page + h * p.dst_head + r * p.dst_token + (int64_t)c * (int64_t)sizeof(W) : -1;
        }
#pragma unroll
        for (int u = 0; u < kTurns; u++)
            if (to[u] >= 0) {
#pragma unroll
                for (int y = 0; y < 2; y++) __builtin_nontemporal_store(word[u][y], reinterpret_cast<W *>(p.dst[y] + to[u]));
            }
    }
}

// ---- sequences that go on from others ----------------------------------------------------------------------------------

struct ReorderDev {
    const int *parents, *table, *lens, *refs, *free_pages, *free_count;
    int *table_out, *lens_out, *refs_out, *free_pages_out, *free_count_out, *copies, *missing;
    int64_t table_width;
    int n_seq, n_pages, most;
    FastDiv by_page, by_width;
};

// What a sequence of so many tokens holds: full pages and the tokens of the partial one (0: none).  Lengths outside of the table hold nothing.
__device__ __forceinline__ int2 held_by(const ReorderDev &p, int len) {
    if (len < 0 || len > p.most) return make_int2(0, 0);
    const int full = p.by_page.by(len);
    return make_int2(full, len - full * (int)p.by_page.d);
}
__device__ __forceinline__ int2 held_pages(const ReorderDev &p, int s) { return held_by(p, p.lens[s]); }

// Who needs a copy of the partial page, and which free page takes it.  All threads of a workgroup of kPlanThreads, which take sequences j0 .. of
// `mine`; s_first[n_seq] is left with the destination of every sequence's copy (-1: none).
constexpr int kMine = kPagedMaxSeqs / kPlanThreads;
struct Begun { int copies, total; bool enough; };   // of this thread, of all
__device__ __forceinline__ Begun begin_reorder(const ReorderDev &p, int j0, int mine, int count, int *s_first, int *s_lens, int *s_waves) {
    int from[kMine], partial[kMine];
    int2 held[kMine];
#pragma unroll
    for (int y = 0; y < kMine; y++) {
        from[y] = y < mine ? p.parents[j0 + y] : -1;
        if (y < mine) s_first[j0 + y] = p.n_seq, s_lens[j0 + y] = p.lens[j0 + y];
    }
    __syncthreads();
#pragma unroll
    for (int y = 0; y < kMine; y++) {
        if ((unsigned)from[y] >= (unsigned)p.n_seq) from[y] = -1;
        if (from[y] >= 0) atomicMin(&s_first[from[y]], j0 + y);
        held[y] = from[y] >= 0 ? held_by(p, s_lens[from[y]]) : make_int2(0, 0);
        partial[y] = held[y].y ? p.table[from[y] * p.table_width + held[y].x] : -1;
    }
    __syncthreads();
    Begun r = {0, 0, false};
    uint32_t copied = 0;   // (bits: with -1 put into partial[y] where there is none, this compiler left the first one as it was)
#pragma unroll
    for (int y = 0; y < kMine; y++) {
        bool need = (unsigned)partial[y] < (unsigned)p.n_pages;
        if (need) need = !(s_first[from[y]] == j0 + y && p.refs[partial[y]] == 1);
        copied |= (need ? 1u : 0u) << y;
    }
    r.copies = __popc(copied);
    int at = block_scan(r.copies, s_waves, r.total);
    r.enough = r.total <= count;
    if (threadIdx.x == 0) p.missing[0] = r.enough ? 0 : r.total - count;
#pragma unroll
    for (int y = 0; y < kMine; y++) {
        if (y >= mine) continue;
        int *out = p.copies + 3 * (j0 + y);
        const bool need = (copied >> y) & 1, go = r.enough && need;
        const int dst = go ? p.free_pages[count - 1 - at] : -1;
        at += need;
        out[0] = go ? partial[y] : -1, out[1] = dst, out[2] = go ? held[y].y : 0;
        p.lens_out[j0 + y] = !r.enough ? s_lens[j0 + y] : from[y] >= 0 ? s_lens[from[y]] : 0;
        s_first[j0 + y] = dst;   // (the firsts have been looked at)
    }
    return r;
}

// First launch.  Workgroup 0: the copies; the others: counts of holders as they were.
__global__ __launch_bounds__(kPlanThreads) void paged_reorder_begin_kernel(ReorderDev p) {
    const int tid = threadIdx.x;
    if (blockIdx.x > 0) {
        const int x = (blockIdx.x - 1) * kPlanThreads + tid;
        if (x < p.n_pages) p.refs_out[x] = p.refs[x];
        return;
    }
    __shared__ int s_first[kPagedMaxSeqs], s_lens[kPagedMaxSeqs], s_waves[kPlanWaves];
    const int per = (p.n_seq + kPlanThreads - 1) / kPlanThreads, j0 = min(tid * per, p.n_seq);
    begin_reorder(p, j0, min(per, p.n_seq - j0), min(max(p.free_count[0], 0), p.n_pages), s_first, s_lens, s_waves);
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
struct Reclaim { int left, freed; };   // free pages that are left, and how many come back

// Sixteen consecutive numbers of [0, n) from x0 on, `none` behind the end: whole loads and stores where they are whole, and all of them at once.
struct Sixteen { int v[16]; };
__device__ __forceinline__ Sixteen load_sixteen(const int *from, int x0, int n, int none) {
    Sixteen r;
    if (x0 <= n - 16) {
        __builtin_memcpy(&r, from + x0, sizeof(r));
    } else {
#pragma unroll
        for (int x = 0; x < 16; x++) r.v[x] = x0 + x < n ? from[x0 + x] : none;
    }
    return r;
}
__device__ __forceinline__ void store_sixteen(int *to, int x0, int n, const Sixteen &r) {
    if (x0 <= n - 16) {
        __builtin_memcpy(to + x0, &r, sizeof(r));
    } else {
#pragma unroll
        for (int x = 0; x < 16; x++)
            if (x0 + x < n) to[x0 + x] = r.v[x];
    }
}

// was, now: holders of this thread's pages, block * kReclaim + tid * 16 .., free: that part of the stack; `taken`: this thread's share of the
// copies.  now_of(x0): holders of 16 other pages.  All threads.
template <typename NowOf>
__device__ __forceinline__ Reclaim reclaim_pages(const ReorderDev &p, int block, int count, int taken, const Sixteen &was, const Sixteen &now, Sixteen free, NowOf now_of,
                                                 int *lds_waves, int *lds_sums) {
    const int tid = threadIdx.x, my0 = block * kReclaim + tid * 16;
    auto freed_of = [&](const Sixteen &w, const Sixteen &n) {   // a bit for each page that somebody held and nobody does any more
        uint32_t bits = 0;
#pragma unroll
        for (int x = 0; x < 16; x++) bits |= (n.v[x] <= 0 && w.v[x] > 0 ? 1u : 0u) << x;
        return bits;
    };
    const uint32_t mine = freed_of(was, now);
    int before = 0, others = 0;
    if (p.n_pages > kReclaim) {
        if (tid < 2) lds_sums[tid] = 0;
        __syncthreads();
        for (int b = 0; b * kReclaim < p.n_pages; b++) {
            if (b == block) continue;
            const int x0 = b * kReclaim + tid * 16, n = __popc(freed_of(load_sixteen(p.refs, x0, p.n_pages, 0), now_of(x0)));
            others += n;
            if (b < block) before += n;
        }
        before = __builtin_amdgcn_readlane(wave_sums(before), 63), others = __builtin_amdgcn_readlane(wave_sums(others), 63);
        if ((tid & 63) == 0) atomicAdd(&lds_sums[0], before), atomicAdd(&lds_sums[1], others);
    }
    // (both sums of a scan in one word: 16 pages a thread, and at most four sequences)
    int total;
    const int scan = block_scan(__popc(mine) | taken << 16, lds_waves, total);
    if (p.n_pages > kReclaim) before = lds_sums[0], others = lds_sums[1];
    const int left = count - (total >> 16), freed = others + (total & 0xffff);
    int at = left + before + (scan & 0xffff);
    for (uint32_t bits = mine; bits; bits &= bits - 1, at++)   // (more free pages than there are pages: counts that were not kept)
        if (at < p.n_pages) p.free_pages_out[at] = my0 + __ffs(bits) - 1;
    bool whole = true;
#pragma unroll
    for (int x = 0; x < 16; x++) {
        if (my0 + x >= left + freed) free.v[x] = -1;
        else if (my0 + x >= left) whole = false;
    }
    if (whole) {
        store_sixteen(p.free_pages_out, my0, p.n_pages, free);
    } else {
#pragma unroll
        for (int x = 0; x < 16; x++)
            if (my0 + x < p.n_pages && (my0 + x < left || my0 + x >= left + freed)) p.free_pages_out[my0 + x] = free.v[x];
    }
    return {left, freed};
}

__global__ __launch_bounds__(kPlanThreads) void paged_reclaim_kernel(ReorderDev p) {
    __shared__ int s_waves[kPlanWaves], s_sums[2];
    const int x0 = blockIdx.x * kReclaim + threadIdx.x * 16, count = min(max(p.free_count[0], 0), p.n_pages);
    const Sixteen was = load_sixteen(p.refs, x0, p.n_pages, 0), now = load_sixteen(p.refs_out, x0, p.n_pages, 0), free = load_sixteen(p.free_pages, x0, p.n_pages, -1);
    int taken = 0;
#pragma unroll
    for (int y = 0; y < kPagedMaxSeqs / kPlanThreads; y++) {
        const int j = threadIdx.x + y * kPlanThreads;
        taken += j < p.n_seq && p.copies[3 * j] >= 0;
    }
    const Reclaim r = reclaim_pages(p, blockIdx.x, count, taken, was, now, free, [&](int x) { return load_sixteen(p.refs_out, x, p.n_pages, 0); }, s_waves, s_sums);
    if (blockIdx.x == 0 && threadIdx.x == 0) p.free_count_out[0] = min(r.left + r.freed, p.n_pages);
}

// All of it by one workgroup, with the counts of holders in LDS, where pages and tables are few: three launches and their memory accesses
// cost more than the one compute unit takes (one | three launches, with the copies that follow, by entries: 8 a sequence 1536 11.4 | 17.7 us, 6144
// 16.7 | 17.6, 12288 23.5 | 20.0; 46 a sequence 2944 12.1 | 17.7, 5888 14.8 | 17.7, 11776 20.3 | 17.8; 256 a sequence 1536 11.0 | 17.7, 6144 15.3 | 17.8,
// 12288 20.2 | 17.9).
constexpr int kSmallPages = kReclaim, kSmallEntries = 6144;
// The argument where it lies, as loads from here on: kept from the beginning, it would not leave enough scalar registers.
__device__ __forceinline__ ReorderDev arguments_again() {
    auto at = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
    asm volatile("" : "+s"(at));
    struct Words { uint64_t w[sizeof(ReorderDev) / 8]; } r;
#pragma unroll
    for (size_t i = 0; i < sizeof(ReorderDev) / 8; i++) r.w[i] = reinterpret_cast<const __attribute__((address_space(4))) uint64_t *>(at)[i];
    return __builtin_bit_cast(ReorderDev, r);
}
__global__ __launch_bounds__(kPlanThreads) void paged_reorder_kernel(ReorderDev) {
    ReorderDev p = arguments_again();
    __shared__ int s_refs[kSmallPages + kSmallPages / 16], s_first[kPagedMaxSeqs], s_children[kPagedMaxSeqs], s_lens[kPagedMaxSeqs], s_from[kPagedMaxSeqs], s_waves[2][kPlanWaves];
    auto page_at = [](int x) { return x + (x >> 4); };   // (threads that take 16 pages each are in different banks)
    const int tid = threadIdx.x, width = (int)p.table_width, per = (p.n_seq + kPlanThreads - 1) / kPlanThreads, j0 = min(tid * per, p.n_seq), mine = min(per, p.n_seq - j0);
    const Sixteen was = load_sixteen(p.refs, tid * 16, p.n_pages, 0), free = load_sixteen(p.free_pages, tid * 16, p.n_pages, -1);
    const int count = min(max(p.free_count[0], 0), p.n_pages);
#pragma unroll
    for (int y = 0; y < kMine; y++)
        if (y < mine) {
            const int from = p.parents[j0 + y];
            s_from[j0 + y] = (unsigned)from < (unsigned)p.n_seq ? from : -1, s_children[j0 + y] = 0;
        }
#pragma unroll
    for (int x = 0; x < 16; x++)
        if (tid * 16 + x < p.n_pages) s_refs[page_at(tid * 16 + x)] = was.v[x];
    const Begun begun = begin_reorder(p, j0, mine, count, s_first, s_lens, s_waves[0]);
    const bool enough = begun.enough;
#pragma unroll
    for (int y = 0; y < kMine; y++)
        if (y < mine && s_from[j0 + y] >= 0) atomicAdd(&s_children[s_from[j0 + y]], 1);
    __syncthreads();
    p = arguments_again();
    // the tables, a thread per entry, several entries' loads at once; what old rows' pages lose or gain
    const FastDiv by_width = p.by_width;
    constexpr int kDeep = 4;
    for (int x0 = tid; x0 < p.n_seq * width; x0 += kDeep * kPlanThreads) {
        int mine_id[kDeep], new_id[kDeep];
#pragma unroll
        for (int y = 0; y < kDeep; y++) {
            const int x = min(x0 + y * kPlanThreads, p.n_seq * width - 1), j = by_width.by(x), src = s_from[j];
            mine_id[y] = p.table[x];
            new_id[y] = src >= 0 ? p.table[src * p.table_width + x - j * width] : -1;
        }
#pragma unroll
        for (int y = 0; y < kDeep; y++) {
            const int x = x0 + y * kPlanThreads;
            if (x >= p.n_seq * width) continue;
            const int j = by_width.by(x), pi = x - j * width, src = s_from[j], dst = s_first[j], children = s_children[j], old = mine_id[y];
            if (!enough) {
                p.table_out[x] = old;
                continue;
            }
            int2 h = src >= 0 ? held_by(p, s_lens[src]) : make_int2(0, 0);
            int id = pi < h.x + (h.y > 0) ? new_id[y] : -1;
            if (h.y && pi == h.x && dst >= 0) {
                id = dst;
                if (dst < p.n_pages) atomicAdd(&s_refs[page_at(dst)], 1);
            }
            p.table_out[x] = id;
            h = held_by(p, s_lens[j]);
            if (pi < h.x + (h.y > 0) && (unsigned)old < (unsigned)p.n_pages) {
                // (the partial page stays with the first child, if nobody else holds it)
                const int change = pi < h.x ? children - 1 : children > 0 && p.refs[old] == 1 ? 0 : -1;
                if (change) atomicAdd(&s_refs[page_at(old)], change);
            }
        }
    }
    __syncthreads();
    p = arguments_again();
    Sixteen now;
#pragma unroll
    for (int x = 0; x < 16; x++) now.v[x] = tid * 16 + x < p.n_pages ? s_refs[page_at(tid * 16 + x)] : 0;
    store_sixteen(p.refs_out, tid * 16, p.n_pages, now);
    const Reclaim r = reclaim_pages(p, 0, count, enough ? begun.copies : 0, was, now, free, [&](int) { return now; }, s_waves[1], nullptr);
    if (tid == 0) p.free_count_out[0] = min(r.left + r.freed, p.n_pages);
}

// ---- copies of pages ------------------------------------------------------------------------------------------------------

struct CopyDev {
    char *pools[kPagedMaxPools];
    const int *copies;
    int64_t page_stride, head_stride, token_stride;   // bytes
    int n_pages, page, heads, words_per_row;
    FastDiv by_words_per_row;
};

// A workgroup per copy and pool: threads side by side along a head's rows, which lie side by side where tokens do, and heads in turn.  256
// entries of which some 90 copy half a page, in 16 pools of 8 heads of 128, f16, 43 MB: 12.6 us, most of it the rows' way there and back (loads
// past the caches 5 us more: a page is copied for several others).
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
    const int words = tokens * p.words_per_row;   // of a head
    int wide = 256;                               // threads of a head
    while (wide > 16 && wide / 2 >= words) wide /= 2;
    const int h0 = threadIdx.x / wide, step = 256 / wide;
    for (int x = threadIdx.x % wide; x < words; x += wide) {
        const int r = p.by_words_per_row.by(x);
        const int64_t at = r * p.token_stride + (int64_t)(x - r * p.words_per_row) * (int64_t)sizeof(W);
        for (int h = h0; h < p.heads; h += kTurns * step) {   // (all on their way before the first is stored)
            W word[kTurns];
#pragma unroll
            for (int u = 0; u < kTurns; u++) word[u] = *reinterpret_cast<const W *>(src + at + min(h + u * step, p.heads - 1) * p.head_stride);
#pragma unroll
            for (int u = 0; u < kTurns; u++)
                if (h + u * step < p.heads) *reinterpret_cast<W *>(dst + at + (h + u * step) * p.head_stride) = word[u];
        }
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
    p.slots = a.slots, p.n_slots = (int)(a.n_pages * a.page_size);
    p.words_per_token = (int)(a.kv_heads * a.D * es / word);
    p.tokens_per_block = std::max(1, 256 * kTurns / p.words_per_token);
    p.by_words_per_token = fast_div(p.words_per_token), p.by_words_per_row = fast_div(a.D * es / word), p.by_page = fast_div(a.page_size);
    // (a launch counts threads in 32 bits)
    const int64_t turn = std::min<int64_t>((int64_t)p.tokens_per_block << 22, 1 << 30);
    for (int64_t first = 0; first < a.n_tokens; first += turn) {
        p.n_tokens = (int)std::min(turn, a.n_tokens - first);
        const dim3 grid((unsigned)((p.n_tokens + p.tokens_per_block - 1) / p.tokens_per_block));
        if (word == 16) paged_append_kernel<Quad><<<grid, 256, 0, s>>>(p);
        else if (word == 4) paged_append_kernel<uint32_t><<<grid, 256, 0, s>>>(p);
        else paged_append_kernel<uint16_t><<<grid, 256, 0, s>>>(p);
        TROCM_HIP(hipGetLastError());
        p.slots += turn;
        for (int y = 0; y < 2; y++) p.src[y] += turn * p.src_token[y];
    }
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
    p.by_width = fast_div(a.table_width);
    if (a.n_pages <= kSmallPages && a.n_seq * a.table_width <= kSmallEntries) {
        paged_reorder_kernel<<<dim3(1), kPlanThreads, 0, s>>>(p);
        TROCM_HIP(hipGetLastError());
        return 0;
    }
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
        const dim3 grid((unsigned)a.n_copies, (unsigned)n);
        if (word == 16) paged_copy_kernel<Quad><<<grid, 256, 0, s>>>(p);
        else if (word == 4) paged_copy_kernel<uint32_t><<<grid, 256, 0, s>>>(p);
        else paged_copy_kernel<uint16_t><<<grid, 256, 0, s>>>(p);
        TROCM_HIP(hipGetLastError());
    }
    return 0;
}

}  // namespace trocm
