// Pages of the int8 KV cache (gfx950): forking and freeing sequences, room for new tokens
// with copy on write, compacting the pool, copying pages, and keeping the accepted ones of
// a sequence's drafted tokens.
//
// A block table [batch, max_blocks] names the 16-token page of every block (-1: none), and
// page_refs [pages] counts the table entries that name each page (0: the page is free). One
// table usually serves every layer, so the bookkeeping runs once and leaves lists of
// (source, destination) pages, which copy_pages carries out on each layer's pool.
//
// Every result is the same from run to run: free pages are handed out lowest first, in the
// order of the sequences and their blocks; atomics only count references. The bookkeeping is
// bound by latency (a few KB of integers), the copies by memory.
#include <algorithm>

#include "reef_common.hpp"

namespace reef {
namespace {

__device__ __forceinline__ bool page_ok(int page, int num_pages) {
    return page >= 0 && page < num_pages;
}

// One table entry fewer names the page. False where none was counted (a table and counts
// that do not belong together); the count stays.
__device__ __forceinline__ bool drop_ref(int32_t *refs, int page) {
    if (atomicSub(refs + page, 1) > 0) return true;
    atomicAdd(refs + page, 1);
    return false;
}

// ---- free, fork ------------------------------------------------------------------------

struct TableArgs {
    int32_t *table;
    int64_t max_blocks;
    int32_t *lens;
    int32_t batch;
    int32_t *refs;
    int32_t num_pages;
    uint32_t *status;
};

__global__ void free_sequences(TableArgs a, const int32_t *sequences) {
    const int b = sequences[blockIdx.y];
    if (b < 0) return;  // padding
    if (b >= a.batch) {
        if (blockIdx.x == 0 && threadIdx.x == 0) flag_status(a.status, REEF_STATUS_BIT_BAD_LENGTH);
        return;
    }
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i == 0) a.lens[b] = 0;
    if (i >= a.max_blocks) return;
    // (exchanged, so that a sequence listed twice gives its pages back once)
    const int page = atomicExch(a.table + b * a.max_blocks + i, -1);
    if (page < 0) return;
    if (page >= a.num_pages || !drop_ref(a.refs, page))
        flag_status(a.status, REEF_STATUS_BIT_BAD_PAGE);
}

__global__ void fork_sequences(TableArgs a, const int32_t *parents, const int32_t *children) {
    const int p = parents[blockIdx.y], c = children[blockIdx.y];
    if (p < 0 || c < 0 || p == c) return;  // padding, or nothing to do
    const bool first = blockIdx.x == 0 && threadIdx.x == 0;
    if (p >= a.batch || c >= a.batch) {
        if (first) flag_status(a.status, REEF_STATUS_BIT_BAD_LENGTH);
        return;
    }
    const int len = a.lens[p];
    if (len < 0 || len > a.max_blocks * kPage) {
        if (first) flag_status(a.status, REEF_STATUS_BIT_BAD_LENGTH);
        return;
    }
    if (first) a.lens[c] = len;
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= a.max_blocks) return;
    // Blocks that hold tokens are shared; room that the parent has beyond them is not.
    int page = i * kPage < len ? a.table[p * a.max_blocks + i] : -1;
    if (page >= a.num_pages) {
        flag_status(a.status, REEF_STATUS_BIT_BAD_PAGE);
        page = -1;
    }
    if (page >= 0) atomicAdd(a.refs + page, 1);
    const int old = atomicExch(a.table + c * a.max_blocks + i, page < 0 ? -1 : page);
    if (old < 0) return;
    if (old >= a.num_pages || !drop_ref(a.refs, old))
        flag_status(a.status, REEF_STATUS_BIT_BAD_PAGE);
}

// ---- reserve ---------------------------------------------------------------------------

constexpr int kScanThreads = 1024, kScanWaves = kScanThreads / kWave;

// Exclusive prefix of `x` over the workgroup's threads, and its total. sWave: kScanWaves.
__device__ __forceinline__ int block_scan(int x, int &total, int *sWave) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    int s = x;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int y = __shfl_up(s, o);
        if (lane >= o) s += y;
    }
    if (lane == kWave - 1) sWave[wave] = s;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kScanWaves; ++w) {
        if (w < wave) before += sWave[w];
        total += sWave[w];
    }
    __syncthreads();
    return before + s - x;
}

struct ReserveArgs {
    TableArgs t;  // (lens is only read)
    int32_t new_tokens, nb;  // blocks that new_tokens can touch
    int64_t items;           // batch * nb
    int32_t *copy_src, *copy_dst;  // [batch]
    int32_t *free_pages, *old_pages;  // workspace, `items` each
};

// What block i of the touched ones of sequence b needs: a page (due), instead of `old` where
// that is shared; copy where it holds tokens.
struct Need {
    bool due, copy;
    int old;
    int64_t entry;
    uint32_t flags;
};

// AGAIN: the counts as this launch's own drops left them.
template <bool AGAIN = false>
__device__ __forceinline__ Need need_of(const ReserveArgs &a, int64_t item) {
    Need n = {false, false, -1, 0, 0};
    const int b = (int)(item / a.nb), i = (int)(item % a.nb);
    const int len = a.t.lens[b];
    if (len < 0 || (int64_t)len + a.new_tokens > a.t.max_blocks * kPage) {
        if (i == 0) n.flags = len < 0 ? REEF_STATUS_BIT_BAD_LENGTH : REEF_STATUS_BIT_CAPACITY;
        return n;
    }
    const int64_t block = len / kPage + i;
    if (block * kPage >= (int64_t)len + a.new_tokens) return n;
    n.entry = b * a.t.max_blocks + block;
    const int page = a.t.table[n.entry];
    const bool holds = block * kPage < len;
    if (page < 0) {
        n.due = true;
        if (holds) n.flags = REEF_STATUS_BIT_BAD_PAGE;  // tokens without a page
    } else if (page >= a.t.num_pages) {
        n.flags = REEF_STATUS_BIT_BAD_PAGE;
    } else if ((AGAIN ? __hip_atomic_load(a.t.refs + page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                      : a.t.refs[page]) > 1) {
        n.due = true;
        n.old = page;
        n.copy = holds;
    }
    return n;
}

// One workgroup: the needs are counted, that many free pages listed lowest first, and
// handed out in order. The references that are given up are dropped last, so that what a
// block needs never depends on the order of the others (two sharers both copy, and the
// page that neither keeps becomes free).
__global__ __launch_bounds__(kScanThreads) void reserve_pages(ReserveArgs a) {
    __shared__ int sWave[kScanWaves];
    const int tid = threadIdx.x;
    for (int b = tid; b < a.t.batch; b += kScanThreads) {
        a.copy_src[b] = -1;
        a.copy_dst[b] = -1;
    }
    int count = 0, wanted = 0;
    uint32_t flags = 0;
    for (int64_t i = tid; i < a.items; i += kScanThreads) {
        const Need n = need_of(a, i);
        count += n.due;
        flags |= n.flags;
    }
    block_scan(count, wanted, sWave);
    if (flags) flag_status(a.t.status, flags);
    if (wanted == 0) return;
    int found = 0;
    for (int64_t base = 0; base < a.t.num_pages && found < wanted; base += 4 * kScanThreads) {
        const int64_t p = base + 4 * tid;
        bool is_free[4];
        int refs[4], mine = 0, all;
#pragma unroll
        for (int j = 0; j < 4; ++j) refs[j] = a.t.refs[min(p + j, (int64_t)a.t.num_pages - 1)];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            is_free[j] = p + j < a.t.num_pages && refs[j] == 0;
            mine += is_free[j];
        }
        int rank = found + block_scan(mine, all, sWave);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (is_free[j]) {
                if (rank < wanted) a.free_pages[rank] = (int)(p + j);
                ++rank;
            }
        found += all;
    }
    found = min(found, wanted);
    __syncthreads();
    int given = 0;
    for (int64_t base = 0; base < a.items; base += kScanThreads) {
        const int64_t i = base + tid;
        Need n = {false, false, -1, 0, 0};
        if (i < a.items) n = need_of(a, i);
        int all;
        const int rank = given + block_scan(n.due, all, sWave);
        given += all;
        if (!n.due) continue;
        if (rank >= found) continue;  // no page left: the block stays as it is
        const int page = a.free_pages[rank];
        a.t.table[n.entry] = page;
        a.t.refs[page] = 1;
        a.old_pages[rank] = n.old;
        if (n.copy) {
            const int b = (int)(i / a.nb);
            a.copy_src[b] = n.old;
            a.copy_dst[b] = page;
        }
    }
    __syncthreads();
    for (int r = tid; r < found; r += kScanThreads)
        if (a.old_pages[r] >= 0) drop_ref(a.t.refs, a.old_pages[r]);
    if (found == wanted) return;
    // Pages ran out. A block that got none may still have what it needs: the last sharer of a page
    // that the others have left.
    __syncthreads();
    bool lacking = false;
    for (int64_t i = tid; i < a.items; i += kScanThreads) lacking |= need_of<true>(a, i).due;
    if (lacking) flag_status(a.t.status, REEF_STATUS_BIT_CAPACITY);
}

// ---- compact ---------------------------------------------------------------------------
//
// With L live pages, the live ones at or past L move into the free places before L: the k-th
// live page from the pool's end into the k-th free place from its front, so the ranks come
// from one prefix count of the live pages.

// (8192 pages: 4 a thread are 2.3 us faster than 16, 1 a thread 0.5 more, but then a pool of a
// million has each of its 4096 workgroups add up as many counts)
constexpr int kCompactThreads = 256, kCompactEach = 4;
constexpr int kCompactChunk = kCompactThreads * kCompactEach;

struct CompactArgs {
    TableArgs t;  // (no lens)
    int32_t *src, *dst;  // [num_pages / 2]
    int32_t *num_live;   // may be null
    int32_t *rank;       // workspace: [num_pages], a moving page's place in src
    int32_t *counts;     // workspace: live pages of each chunk, then the number of moves
    int32_t chunks;
};

__global__ __launch_bounds__(kCompactThreads) void count_live(CompactArgs a) {
    __shared__ int sSum;
    if (threadIdx.x == 0) sSum = 0;
    __syncthreads();
    // (loads without a branch between them: one round trip, not four)
    int refs[kCompactEach], n = 0;
#pragma unroll
    for (int j = 0; j < kCompactEach; ++j) {
        const int64_t p = (int64_t)blockIdx.x * kCompactChunk + j * kCompactThreads + threadIdx.x;
        refs[j] = a.t.refs[min(p, (int64_t)a.t.num_pages - 1)];
        if (p >= a.t.num_pages) refs[j] = 0;
    }
#pragma unroll
    for (int j = 0; j < kCompactEach; ++j) n += refs[j] > 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
    if ((threadIdx.x & 63) == 0) atomicAdd(&sSum, n);
    __syncthreads();
    if (threadIdx.x == 0) a.counts[blockIdx.x] = sSum;
}

__global__ __launch_bounds__(kCompactThreads) void list_moves(CompactArgs a) {
    constexpr int W = kCompactThreads / kWave;
    constexpr int kCounts = kCompactEach * W;
    static_assert(kCounts <= kWave, "one count per lane");
    __shared__ int sBefore[W], sTotal[W], sLive[kWave];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // Page j of this thread is tid + 256 j of the chunk: in order, (j, wave, lane).
    const int64_t base = (int64_t)blockIdx.x * kCompactChunk + tid;
    int refs[kCompactEach];
#pragma unroll
    for (int j = 0; j < kCompactEach; ++j)
        refs[j] = a.t.refs[min(base + j * kCompactThreads, (int64_t)a.t.num_pages - 1)];
    int before = 0, total = 0;
    for (int c = tid; c < a.chunks; c += kCompactThreads) {
        const int n = a.counts[c];
        total += n;
        before += c < (int)blockIdx.x ? n : 0;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        before += __shfl_xor(before, o);
        total += __shfl_xor(total, o);
    }
    uint64_t live[kCompactEach];
#pragma unroll
    for (int j = 0; j < kCompactEach; ++j) {
        live[j] = __ballot(base + j * kCompactThreads < a.t.num_pages && refs[j] > 0);
        if (lane == j) sLive[W * j + wave] = __popcll(live[j]);
    }
    if (lane == 0) {
        sBefore[wave] = before;
        sTotal[wave] = total;
    }
    __syncthreads();
    before = total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        before += sBefore[w];
        total += sTotal[w];
    }
    const int own = lane < kCounts ? sLive[lane] : 0;
    int s = own;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int y = __shfl_up(s, o);
        if (lane >= o) s += y;
    }
    s += before - own;  // live pages before the 64 of (j, wave) = (lane / W, lane % W)
#pragma unroll
    for (int j = 0; j < kCompactEach; ++j) {
        const int64_t p = base + j * kCompactThreads;
        const int n = __shfl(s, W * j + wave) + (int)__popcll(live[j] & ((1ull << lane) - 1));
        if (p >= a.t.num_pages) continue;
        const bool is_live = live[j] >> lane & 1u;
        if (p == total) a.counts[a.chunks] = total - n;  // moves: the live pages from here on
        int rank = -1;
        if (is_live && p >= total) {
            rank = total - 1 - n;
            a.src[rank] = (int)p;
        } else if (!is_live && p < total) {
            a.dst[p - n] = (int)p;
        }
        a.rank[p] = rank;
    }
    if (blockIdx.x == 0 && tid == 0) {
        if (total == a.t.num_pages) a.counts[a.chunks] = 0;
        if (a.num_live) *a.num_live = total;
    }
}

__global__ __launch_bounds__(256) void apply_moves(CompactArgs a) {
    const int moves = a.counts[a.chunks];
    const int64_t step = (int64_t)gridDim.x * blockDim.x;
    const int64_t first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t entries = a.t.batch * a.t.max_blocks;
    for (int64_t e = first; e < entries; e += step) {
        const int page = a.t.table[e];
        if (page < 0) continue;
        if (page >= a.t.num_pages) {
            flag_status(a.t.status, REEF_STATUS_BIT_BAD_PAGE);
            continue;
        }
        const int r = a.rank[page];
        if (r >= 0) a.t.table[e] = a.dst[r];
    }
    for (int64_t k = first; k < a.t.num_pages / 2; k += step) {
        if (k < moves) {
            a.t.refs[a.dst[k]] = a.t.refs[a.src[k]];
            a.t.refs[a.src[k]] = 0;
        } else {
            a.src[k] = -1;
            a.dst[k] = -1;
        }
    }
}

// ---- copy ------------------------------------------------------------------------------

struct CopyArgs {
    const int32_t *src, *dst;
    int64_t pairs;
    int8_t *pages[2];
    float *scales[2];
    int32_t page_words, scale_words;  // 16-byte words of a page and of its scales
    int32_t num_pages;
    uint32_t *status;
};

constexpr int kCopyThreads = 256;

// One workgroup per pair and pool (keys, values).
__global__ __launch_bounds__(kCopyThreads) void copy_pages(CopyArgs a) {
    const int64_t pair = linear_block();
    if (pair >= a.pairs) return;
    const int s = a.src[pair], d = a.dst[pair];
    if (s < 0 || d < 0 || s == d) return;
    const int tid = threadIdx.x;
    if (s >= a.num_pages || d >= a.num_pages) {
        if (tid == 0) flag_status(a.status, REEF_STATUS_BIT_BAD_PAGE);
        return;
    }
    i32x4 *page = reinterpret_cast<i32x4 *>(a.pages[blockIdx.y]);
    i32x4 *scale = reinterpret_cast<i32x4 *>(a.scales[blockIdx.y]);
    const i32x4 *from = page + (int64_t)s * a.page_words;
    i32x4 *to = page + (int64_t)d * a.page_words;
    constexpr int kAhead = 4;
    for (int w = tid; w < a.page_words; w += kAhead * kCopyThreads) {
        i32x4 v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (w + j * kCopyThreads < a.page_words) v[j] = from[w + j * kCopyThreads];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (w + j * kCopyThreads < a.page_words) to[w + j * kCopyThreads] = v[j];
    }
    for (int w = tid; w < a.scale_words; w += kCopyThreads)
        scale[(int64_t)d * a.scale_words + w] = scale[(int64_t)s * a.scale_words + w];
}

// ---- keep ------------------------------------------------------------------------------

constexpr int kKeepThreads = 256;

struct KeepArgs {
    const int32_t *kept, *kept_lens, *lens;
    int32_t *new_lens;
    int8_t *k, *v;
    float *ks, *vs;
    const int32_t *table;  // paged only
    int32_t kv_heads, drafts, max_context, max_blocks, num_pages;
    uint32_t *status;
};

// One workgroup per (sequence, kv head). A kept row may be the place of another: every row
// is read into LDS before one is written.
template <int D, bool PAGED>
__global__ __launch_bounds__(kKeepThreads) void keep_rows(KeepArgs a) {
    __shared__ __attribute__((aligned(16))) int8_t sK[kMaxDrafts * D];
    __shared__ int8_t sV[kMaxDrafts * D];
    __shared__ float sScale[2][kMaxDrafts];
    __shared__ int64_t sFrom[kMaxDrafts], sTo[kMaxDrafts];  // 16 x (page, kv head) + slot
    const int tid = threadIdx.x, lane = tid & 63;
    const int b = blockIdx.y, kvh = blockIdx.x;
    const int len = a.lens[b], n = a.kept_lens[b], first = len - a.drafts;
    const bool one = kvh == 0 && tid == 0;
    if (len < a.drafts || len > a.max_context || n < 0 || n > a.drafts) {
        if (one) flag_status(a.status, REEF_STATUS_BIT_BAD_LENGTH);
        if (one && a.new_lens) a.new_lens[b] = len;
        return;
    }
    // Row i (this lane's, in every wave) and the one that takes its place.
    const int row = lane < n ? a.kept[(int64_t)b * a.drafts + lane] : a.drafts;
    const int before = __shfl_up(row, 1);
    const bool bad = lane < n && (row < 0 || row >= a.drafts || (lane > 0 && row <= before));
    // (ascending rows from 0 on: row >= lane, so the first `same` rows stay where they are)
    int64_t from = 0, to = 0;
    bool bad_page = false;
    if (!bad && lane < n) {
        const int pf = first + row, pt = first + lane;
        if (PAGED) {
            const int32_t *t = a.table + (int64_t)b * a.max_blocks;
            const int f = t[pf / kPage], o = t[pt / kPage];
            bad_page = !page_ok(f, a.num_pages) || !page_ok(o, a.num_pages);
            from = ((int64_t)f * a.kv_heads + kvh) * kPage + pf % kPage;
            to = ((int64_t)o * a.kv_heads + kvh) * kPage + pt % kPage;
        } else {
            const int64_t base = ((int64_t)b * a.kv_heads + kvh) * a.max_context;
            from = base + pf;
            to = base + pt;
        }
    }
    const bool any_bad = __any(bad), any_bad_page = __any(bad_page);
    if (any_bad || any_bad_page) {
        if (one)
            flag_status(a.status, any_bad ? REEF_STATUS_BIT_BAD_LENGTH : REEF_STATUS_BIT_BAD_PAGE);
        if (one && a.new_lens) a.new_lens[b] = len;
        return;
    }
    if (one && a.new_lens) a.new_lens[b] = first + n;
    const int same = __popcll(__ballot(lane < n && row == lane));
    if (same == n) return;
    if (tid < kMaxDrafts) {
        sFrom[tid] = from;
        sTo[tid] = to;
    }
    __syncthreads();
    constexpr int KC = D / 16;  // 16-byte chunks of a key row
    auto value = [&](int64_t at, int ch) {  // channel ch of token `at` in the transposed pages
        return a.v + (at / kPage) * (kPage * D) + ch * kPage + at % kPage;
    };
    for (int o = same * KC + tid; o < n * KC; o += kKeepThreads)
        *reinterpret_cast<i32x4 *>(sK + 16 * o) =
            *reinterpret_cast<const i32x4 *>(a.k + sFrom[o / KC] * D + 16 * (o % KC));
    for (int o = same * D + tid; o < n * D; o += kKeepThreads) sV[o] = *value(sFrom[o / D], o % D);
    if (tid >= same && tid < n) {
        sScale[0][tid] = a.ks[from];
        sScale[1][tid] = a.vs[from];
    }
    __syncthreads();
    for (int o = same * KC + tid; o < n * KC; o += kKeepThreads)
        *reinterpret_cast<i32x4 *>(a.k + sTo[o / KC] * D + 16 * (o % KC)) =
            *reinterpret_cast<const i32x4 *>(sK + 16 * o);
    for (int o = same * D + tid; o < n * D; o += kKeepThreads) *value(sTo[o / D], o % D) = sV[o];
    if (tid >= same && tid < n) {
        a.ks[to] = sScale[0][tid];
        a.vs[to] = sScale[1][tid];
    }
}

// ---- host ------------------------------------------------------------------------------

reef_status table_args(TableArgs &a, int32_t *block_table, int64_t max_blocks, int32_t *lens,
                       int64_t batch, int32_t *refs, int64_t num_pages, uint32_t *status) {
    if (!block_table || !refs || max_blocks <= 0 || batch <= 0 || num_pages <= 0)
        return REEF_INVALID_ARGUMENT;
    if (batch > 65535 || num_pages >= (int64_t(1) << 31) || max_blocks >= (int64_t(1) << 26))
        return REEF_UNSUPPORTED;
    a = {block_table, max_blocks, lens, (int32_t)batch, refs, (int32_t)num_pages, status};
    return REEF_OK;
}

int64_t touched_blocks(int64_t new_tokens) { return (new_tokens + kPage - 2) / kPage + 1; }

reef_status keep(const reef_kv_append_params *p, const int32_t *kept, const int32_t *kept_lens,
                 const int32_t *lens, const int32_t *table, int64_t max_blocks, int64_t num_pages,
                 int8_t *k, int8_t *v, float *ks, float *vs, int32_t *new_lens, uint32_t *status,
                 hipStream_t stream) {
    if (!p || !kept || !kept_lens || !lens || !k || !v || !ks || !vs || !aligned(k, 16))
        return REEF_INVALID_ARGUMENT;
    if (p->batch <= 0 || p->kv_heads <= 0 || p->head_dim <= 0 || p->new_tokens <= 0 ||
        p->max_context <= 0 || p->max_context % kPage != 0)
        return REEF_INVALID_ARGUMENT;
    if (p->new_tokens > p->max_context) return REEF_CAPACITY;
    if (p->new_tokens > kMaxDrafts || (p->head_dim != 64 && p->head_dim != 128) ||
        p->max_context >= (int64_t(1) << 30) || p->batch > 65535 || p->kv_heads > 65535)
        return REEF_UNSUPPORTED;
    // every workgroup of a sequence reads its length, its kept rows and their number
    auto overlaps = [&](const int32_t *x, int64_t n) {
        const uintptr_t x0 = reinterpret_cast<uintptr_t>(x), n0 = reinterpret_cast<uintptr_t>(new_lens);
        return new_lens && x0 < n0 + 4 * (uintptr_t)p->batch && n0 < x0 + 4 * (uintptr_t)n;
    };
    if (overlaps(lens, p->batch) || overlaps(kept_lens, p->batch) ||
        overlaps(kept, p->batch * p->new_tokens))
        return REEF_INVALID_ARGUMENT;
    KeepArgs a = {kept, kept_lens, lens, new_lens, k, v, ks, vs, table, (int32_t)p->kv_heads,
                  (int32_t)p->new_tokens, (int32_t)p->max_context, (int32_t)max_blocks,
                  (int32_t)num_pages, status};
    const dim3 grid((unsigned)p->kv_heads, (unsigned)p->batch), block(kKeepThreads);
    if (table && p->head_dim == 128)
        hipLaunchKernelGGL((keep_rows<128, true>), grid, block, 0, stream, a);
    else if (table)
        hipLaunchKernelGGL((keep_rows<64, true>), grid, block, 0, stream, a);
    else if (p->head_dim == 128)
        hipLaunchKernelGGL((keep_rows<128, false>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((keep_rows<64, false>), grid, block, 0, stream, a);
    return launch_status();
}

}  // namespace
}  // namespace reef

using namespace reef;

extern "C" reef_status reef_kv_free(const int32_t *sequences, int64_t n, int32_t *block_table,
                                    int64_t max_blocks_per_seq, int32_t *context_lens,
                                    int64_t batch, int32_t *page_refs, int64_t num_pages,
                                    uint32_t *status_word, hipStream_t stream) {
    TableArgs a;
    const reef_status s = table_args(a, block_table, max_blocks_per_seq, context_lens, batch,
                                     page_refs, num_pages, status_word);
    if (s != REEF_OK) return s;
    if (!sequences || !context_lens || n <= 0) return REEF_INVALID_ARGUMENT;
    if (n > 65535) return REEF_UNSUPPORTED;
    hipLaunchKernelGGL(free_sequences, dim3((unsigned)ceil_div(max_blocks_per_seq, 256), (unsigned)n),
                       dim3(256), 0, stream, a, sequences);
    return launch_status();
}

extern "C" reef_status reef_kv_fork(const int32_t *parents, const int32_t *children, int64_t n,
                                    int32_t *block_table, int64_t max_blocks_per_seq,
                                    int32_t *context_lens, int64_t batch, int32_t *page_refs,
                                    int64_t num_pages, uint32_t *status_word, hipStream_t stream) {
    TableArgs a;
    const reef_status s = table_args(a, block_table, max_blocks_per_seq, context_lens, batch,
                                     page_refs, num_pages, status_word);
    if (s != REEF_OK) return s;
    if (!parents || !children || !context_lens || n <= 0) return REEF_INVALID_ARGUMENT;
    if (n > 65535) return REEF_UNSUPPORTED;
    hipLaunchKernelGGL(fork_sequences, dim3((unsigned)ceil_div(max_blocks_per_seq, 256), (unsigned)n),
                       dim3(256), 0, stream, a, parents, children);
    return launch_status();
}

extern "C" size_t reef_kv_reserve_workspace_bytes(int64_t batch, int64_t new_tokens) {
    if (batch <= 0 || new_tokens <= 0) return 0;
    return (size_t)(8 * batch * touched_blocks(new_tokens));
}

extern "C" reef_status reef_kv_reserve(int32_t *block_table, int64_t max_blocks_per_seq,
                                       const int32_t *context_lens, int64_t batch,
                                       int64_t new_tokens, int32_t *page_refs, int64_t num_pages,
                                       int32_t *copy_src, int32_t *copy_dst, void *workspace,
                                       size_t workspace_bytes, uint32_t *status_word,
                                       hipStream_t stream) {
    ReserveArgs a;
    const reef_status s =
        table_args(a.t, block_table, max_blocks_per_seq, const_cast<int32_t *>(context_lens), batch,
                   page_refs, num_pages, status_word);
    if (s != REEF_OK) return s;
    if (!context_lens || !copy_src || !copy_dst || new_tokens <= 0 || !workspace ||
        !aligned(workspace, 4))
        return REEF_INVALID_ARGUMENT;
    if (new_tokens > max_blocks_per_seq * kPage) return REEF_CAPACITY;
    a.nb = (int32_t)touched_blocks(new_tokens);
    a.items = batch * a.nb;
    if (new_tokens >= (int64_t(1) << 30) || a.items >= (int64_t(1) << 31)) return REEF_UNSUPPORTED;
    if (workspace_bytes < reef_kv_reserve_workspace_bytes(batch, new_tokens))
        return REEF_INVALID_ARGUMENT;
    a.new_tokens = (int32_t)new_tokens;
    a.copy_src = copy_src;
    a.copy_dst = copy_dst;
    a.free_pages = static_cast<int32_t *>(workspace);
    a.old_pages = a.free_pages + a.items;
    hipLaunchKernelGGL(reserve_pages, dim3(1), dim3(kScanThreads), 0, stream, a);
    return launch_status();
}

extern "C" size_t reef_kv_compact_workspace_bytes(int64_t num_pages) {
    if (num_pages <= 0) return 0;
    return (size_t)(4 * (num_pages + ceil_div(num_pages, kCompactChunk) + 1));
}

extern "C" reef_status reef_kv_compact(int32_t *block_table, int64_t max_blocks_per_seq,
                                       int64_t batch, int32_t *page_refs, int64_t num_pages,
                                       int32_t *copy_src, int32_t *copy_dst, int32_t *num_live,
                                       void *workspace, size_t workspace_bytes,
                                       uint32_t *status_word, hipStream_t stream) {
    CompactArgs a;
    const reef_status s = table_args(a.t, block_table, max_blocks_per_seq, nullptr, batch,
                                     page_refs, num_pages, status_word);
    if (s != REEF_OK) return s;
    if (!copy_src || !copy_dst || !workspace || !aligned(workspace, 4) ||
        workspace_bytes < reef_kv_compact_workspace_bytes(num_pages))
        return REEF_INVALID_ARGUMENT;
    a.src = copy_src;
    a.dst = copy_dst;
    a.num_live = num_live;
    a.rank = static_cast<int32_t *>(workspace);
    a.counts = a.rank + num_pages;
    a.chunks = (int32_t)ceil_div(num_pages, kCompactChunk);
    hipLaunchKernelGGL(count_live, dim3((unsigned)a.chunks), dim3(kCompactThreads), 0, stream, a);
    hipLaunchKernelGGL(list_moves, dim3((unsigned)a.chunks), dim3(kCompactThreads), 0, stream, a);
    const int64_t work = std::max(batch * max_blocks_per_seq, num_pages / 2);
    hipLaunchKernelGGL(apply_moves, dim3((unsigned)std::min<int64_t>(ceil_div(work, 256), 4096)),
                       dim3(256), 0, stream, a);
    return launch_status();
}

namespace {

// Pools of `row_bytes` bytes a key row: 16 of them a head's page, and as many value bytes.
reef_status copy(const int32_t *src, const int32_t *dst, int64_t n, int64_t kv_heads,
                 int64_t head_dim, int64_t row_bytes, void *k_pages, void *v_pages,
                 float *k_scale_pages, float *v_scale_pages, int64_t num_pages,
                 uint32_t *status_word, hipStream_t stream) {
    if (!src || !dst || n <= 0 || kv_heads <= 0 || head_dim <= 0 || num_pages <= 0 || !k_pages ||
        !v_pages || !k_scale_pages || !v_scale_pages || !aligned(k_pages, 16) ||
        !aligned(v_pages, 16) || !aligned(k_scale_pages, 16) || !aligned(v_scale_pages, 16))
        return REEF_INVALID_ARGUMENT;
    if ((head_dim != 64 && head_dim != 128) || kv_heads > 65535 || n >= (int64_t(1) << 31) ||
        num_pages >= (int64_t(1) << 31))
        return REEF_UNSUPPORTED;
    CopyArgs a;
    a.src = src;
    a.dst = dst;
    a.pairs = n;
    a.pages[0] = static_cast<int8_t *>(k_pages);
    a.pages[1] = static_cast<int8_t *>(v_pages);
    a.scales[0] = k_scale_pages;
    a.scales[1] = v_scale_pages;
    a.page_words = (int32_t)(kv_heads * row_bytes);  // 16 rows of row_bytes a head
    a.scale_words = (int32_t)(kv_heads * 4);        // 16 floats a head
    a.num_pages = (int32_t)num_pages;
    a.status = status_word;
    hipLaunchKernelGGL(copy_pages, linear_grid(n, 2), dim3(kCopyThreads), 0, stream, a);
    return launch_status();
}

}  // namespace

extern "C" reef_status reef_kv_copy_pages(const int32_t *src, const int32_t *dst, int64_t n,
                                          int64_t kv_heads, int64_t head_dim, int8_t *k_pages,
                                          int8_t *v_pages, float *k_scale_pages,
                                          float *v_scale_pages, int64_t num_pages,
                                          uint32_t *status_word, hipStream_t stream) {
    return copy(src, dst, n, kv_heads, head_dim, head_dim, k_pages, v_pages, k_scale_pages,
                v_scale_pages, num_pages, status_word, stream);
}

extern "C" reef_status reef_kv_copy_pages_int4(const int32_t *src, const int32_t *dst, int64_t n,
                                               int64_t kv_heads, int64_t head_dim,
                                               uint8_t *k_pages, uint8_t *v_pages,
                                               float *k_scale_pages, float *v_scale_pages,
                                               int64_t num_pages, uint32_t *status_word,
                                               hipStream_t stream) {
    return copy(src, dst, n, kv_heads, head_dim, head_dim / 2, k_pages, v_pages, k_scale_pages,
                v_scale_pages, num_pages, status_word, stream);
}

extern "C" reef_status reef_kv_keep_int8(const reef_kv_append_params *p, const int32_t *kept,
                                         const int32_t *kept_lens, const int32_t *context_lens,
                                         int8_t *k_cache, int8_t *v_cache, float *k_scales,
                                         float *v_scales, int32_t *new_lens, uint32_t *status_word,
                                         hipStream_t stream) {
    return keep(p, kept, kept_lens, context_lens, nullptr, 0, 0, k_cache, v_cache, k_scales,
                v_scales, new_lens, status_word, stream);
}

extern "C" reef_status reef_kv_keep_int8_paged(
    const reef_kv_append_params *p, const int32_t *kept, const int32_t *kept_lens,
    const int32_t *context_lens, const int32_t *block_table, int64_t max_blocks_per_seq,
    int64_t num_pages, int8_t *k_pages, int8_t *v_pages, float *k_scale_pages,
    float *v_scale_pages, int32_t *new_lens, uint32_t *status_word, hipStream_t stream) {
    if (!p || !block_table || max_blocks_per_seq <= 0 || num_pages <= 0 ||
        max_blocks_per_seq * kPage < p->max_context || num_pages >= (int64_t(1) << 31) ||
        max_blocks_per_seq >= (int64_t(1) << 26))
        return REEF_INVALID_ARGUMENT;
    return keep(p, kept, kept_lens, context_lens, block_table, max_blocks_per_seq, num_pages,
                k_pages, v_pages, k_scale_pages, v_scale_pages, new_lens, status_word, stream);
}
