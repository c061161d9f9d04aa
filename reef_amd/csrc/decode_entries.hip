// Decode attention over a cache held in 4 bits, and over the pages of either cache that a list
// names (gfx950). decode.hip's step with two things changed:
//
// A block of 64 keys is four pages named by entries: the sequence's pages one after the other, or
// its list's.
//
// Such a block's bytes take less time than decode.hip's arithmetic on the 16 instruction columns,
// of which G = q_heads / kv_heads are live. Here the scores of a page's 16 keys move into the dead
// columns, HEADS keys to a column (HEADS: 4, 8 or 16, at least G), so that every lane has live ones
// and a lane's share is HEADS scores instead of 16. A column's weights are zero for the other
// columns' keys, each column keeps a softmax of its own, and the columns of a head are merged when
// a run of keys ends.
//
// A short chunk of a prompt over the 4-bit cache runs here too (its rows and the group's heads are
// the columns, 16 or fewer to an item, with an end of their own each): a launch without the copy of
// the cache that prefill_cache.hip makes for a long one.
#include "decode_block.hpp"

namespace reef {
namespace {

constexpr int kEntryThreads = 64 * kDecodeWaves;
// Blocks a part of an item has at least where workgroups take a part each: two a wave. (With 4 the
// merges of more parts outweigh them, with 16 the waves wait: 12.5, 12.4, 14.9 us for 8 heads of
// 256 listed pages.)
constexpr int kLeastBlocks = 8;

// The block of four pages named by entries (numbers of the sequence's pages, -1: none) that lanes
// l % 4 hold, with their page numbers from the block table.
// (Of a chunk's sequence a page that is not there reads as zero codes, elsewhere it takes no part.)
template <int D, int BITS, int HEADS, bool PAGED, bool NT, bool CHUNK>
__device__ __forceinline__ void load_entries(const DecodeArgs &a, int b, int kvh, int n_pages,
                                             int entries, int pages, int col, int grp,
                                             DecodeBlock<D, BITS, HEADS> &x, bool &bad_page) {
    const int ke = __shfl(entries, col >> 2), ge = __shfl(entries, grp);
    // (none is a page past the sequence to page_ref: dead)
    const PageRef kp = page_ref<D, BITS, PAGED>(a, b, kvh, ke < 0 ? n_pages : ke, n_pages,
                                                PAGED ? __shfl(pages, col >> 2) : 0);
    const PageRef gp = page_ref<D, BITS, PAGED>(a, b, kvh, ge < 0 ? n_pages : ge, n_pages,
                                                PAGED ? __shfl(pages, grp) : 0);
    x.pos = max(ge, 0) * kPage;
    load_pages<D, BITS, HEADS, NT>(kp, gp, col, grp, x, bad_page);
    if constexpr (CHUNK && PAGED) x.ok = gp.ok;
}

// What an item reads: a sequence's pages, a list's, or a sequence's for a chunk's rows.
enum Form { kAll, kListed, kChunk };

struct EntryArgs : DecodeArgs {
    // kChunk: an item is (sequence, kv head, tile) of HEADS columns of q_len rows x group heads
    int64_t q_sb, q_sh, q_st, o_sb, o_sh, o_st;
    int32_t tiles, q_len, query_start;
    // dealing out: whether by blocks, whether of few items, the blocks a part has at least where
    // there is room, the workgroups that run at once
    int32_t planned, few, least, round;
};

// The chunk's row that column c of a tile is of (past the last: the last).
template <int HEADS>
__device__ __forceinline__ int chunk_row(const EntryArgs &a, int tile, int c) {
    return min((tile * HEADS + c) / a.group, a.q_len - 1);
}

template <int HEADS, Form FORM>
__device__ __forceinline__ ItemKeys entry_keys(const EntryArgs &a, int item) {
    if constexpr (FORM != kChunk) {
        return item_keys<FORM == kListed>(a, item);
    } else {
        const int tile = item % a.tiles;
        const int first = a.query_start + chunk_row<HEADS>(a, tile, 0);
        ItemKeys r;
        r.bad = false;
        r.count = 0;
        r.len = a.query_start + chunk_row<HEADS>(a, tile, HEADS - 1) + 1;
        r.lo = a.window > 0 ? max(0, first + 1 - a.window) : 0;
        r.first_block = r.lo / kBlockKeys;
        r.blocks = (r.len + kBlockKeys - 1) / kBlockKeys - r.first_block;
        return r;
    }
}

// Keys [k_begin, k_end) of (sequence b, kv head kvh) in steps of k_step: the sequence's, or (listed)
// the places of its list, 16 to an entry, `count` entries in all; this lane's column sees those in
// [lo, len). The next block's loads, the
// page numbers of the one after and the entries of the one after that are issued before the current
// block is computed, and all of them always, of the last block again where there is none: under a
// branch the compiler would wait for all loads in flight at the next use of any. (Two blocks in
// flight instead of one gain nothing.)
template <int D, int BITS, int HEADS, bool PAGED, Form FORM>
__device__ __forceinline__ void run_entries(const EntryArgs &a, int item, int b, int kvh, int lo,
                                            int len, int count, int k_begin, int k_end, int k_step,
                                            int n_pages, const Query<D> &q, int lane,
                                            DecodeRun<D> &st, bool &bad_page) {
    if (k_begin >= k_end) return;
    const int col = lane & 15, grp = lane >> 4;
    const int last = (k_end - k_begin - 1) / k_step;
    auto entry = [&](int i) {
        const int at = (k_begin + min(i, last) * k_step) / kPage + (lane & 3);
        if constexpr (FORM == kListed) {
            const int e = a.sel_pages[(int64_t)item * a.max_sel + min(at, count - 1)];
            bad_page |= at < count && e >= n_pages;
            return at < count && e < n_pages ? max(e, -1) : -1;
        } else {
            return at < n_pages ? at : -1;
        }
    };
    auto page = [&](int e) {
        return PAGED ? a.block_table[(int64_t)b * a.max_blocks + max(e, 0)] : 0;
    };
    DecodeBlock<D, BITS, HEADS> cur, next;
    auto load = [&](int e, int p) {
        // (Whole sequences stream past the caches: non-temporal loads take 54.5 us instead of 60 for
        // 64 x 8 heads of 4096 tokens in pages, 50 instead of 58 in one piece, and no longer where
        // sequences share their pages. Listed pages do not (22.3
        // us, non-temporal 24.6), nor a chunk's, which several tiles read.)
        load_entries<D, BITS, HEADS, PAGED, FORM == kAll, FORM == kChunk>(a, b, kvh, n_pages, e, p, col,
                                                                          grp, next, bad_page);
    };
    auto math = [&](int i) {
        if constexpr (FORM == kChunk && PAGED) {
            if (__any(!cur.ok)) {  // (zero codes: scores and values of zero, which take part)
#pragma unroll
                for (int j = 0; j < DecodeBlock<D, BITS, HEADS>::S; ++j) {
                    cur.ks[j] = cur.ok ? cur.ks[j] : 0.0f;
                    cur.vs[j] = cur.ok ? cur.vs[j] : 0.0f;
                }
                cur.live |= !cur.ok;
            }
        }
        block_math<D, BITS, HEADS, FORM != kAll>(cur, k_begin + i * k_step, lo,
                                                 FORM == kAll ? k_end : len, q, lane, st);
    };
    const int e0 = entry(0);
    int e1 = entry(1), e2 = entry(2);  // of the next block and the one after
    const int p0 = page(e0);
    int p1 = page(e1);
    load(e0, p0);
    for (int i = 0; i < last; ++i) {
        const int p2 = page(e2), e3 = entry(i + 3);
        cur = next;
        load(e1, p1);
        math(i);
        e1 = e2;
        p1 = p2;
        e2 = e3;
    }
    cur = next;
    math(last);
}

// The columns of a head as one: every lane of the row that holds the head has the result.
template <int ROTATE>
__device__ __forceinline__ float row_rotated(float x) {
    return __int_as_float(
        __builtin_amdgcn_mov_dpp(__float_as_int(x), 0x120 + ROTATE, 0xf, 0xf, true));
}
template <int ROTATE>
__device__ __forceinline__ float row_sum(float x) { return x + row_rotated<ROTATE>(x); }

template <int D, int HEADS>
__device__ __forceinline__ void merge_columns(float &m, float &l, f32x4 (&o)[D / 16]) {
    if constexpr (HEADS < 16) {
        float mt = fmaxf(m, row_rotated<8>(m));
        if constexpr (HEADS == 4) mt = fmaxf(mt, row_rotated<4>(mt));
        const float e = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mt);
        m = mt;
        auto sum = [&](float x) {
            x = row_sum<8>(x * e);
            if constexpr (HEADS == 4) x = row_sum<4>(x);
            return x;
        };
        l = sum(l);
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][i] = sum(o[d][i]);
    }
}

// Results of the kernels over entries lie by rows: slot s of D HEADS / 4 holds four channels,
// 4 (s % (D / 4)) .., of head s / (D / 4), with the head's (max, sum) beside. A workgroup's waves
// leave theirs in LDS, all threads merge a slot each, and a part in the workspace is the slots in
// order: whole lines, of the live heads alone.
template <int D, int HEADS>
struct RowSlots {
    static constexpr int N = D * HEADS / 4;
    static constexpr int THREADS = kEntryThreads;
    static constexpr int PER = N > THREADS ? N / THREADS : 1;     // slots a thread
    static constexpr int GROUPS = N < THREADS ? THREADS / N : 1;  // parts that threads take at once
    static_assert((2 * N + HEADS) <= DecodeSlot<D>::ELEMS, "a part's place in the workspace");
};

struct RowRun {
    float m, l;
    f32x4 o;
};
__device__ __forceinline__ void merge_rows(RowRun &r, float m, float l, f32x4 o) {
    const float mn = fmaxf(r.m, m);
    const float er = r.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(r.m - mn);
    const float ep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    r.l = __builtin_fmaf(ep, l, r.l * er);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.o[i] = __builtin_fmaf(ep, o[i], r.o[i] * er);
    r.m = mn;
}

// The first `n` runs of slot s in LDS, in order.
template <int D, int HEADS>
__device__ __forceinline__ RowRun merge_slot(const f32x4 *sRow, const float2 *sML, int s, int n) {
    constexpr int N = RowSlots<D, HEADS>::N;
    const int h = s / (D / 4);
    RowRun r = {sML[h].x, sML[h].y, sRow[s]};
    for (int w = 1; w < n; ++w) {
        const float2 ml = sML[w * 16 + h];
        merge_rows(r, ml.x, ml.y, sRow[w * N + s]);
    }
    return r;
}

// --- dealing out -----------------------------------------------------------------------------

// A workgroup-wide sum of x (every thread gets it; sWave holds a word a wave).
__device__ __forceinline__ int workgroup_sum(int x, int32_t *sWave) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sWave[threadIdx.x >> 6] = x;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int w = 0; w < kDecodeWaves; ++w) s += sWave[w];
    return __builtin_amdgcn_readfirstlane(s);
}

// A sum over the lanes of a wave, in a scalar register.
__device__ __forceinline__ int wave_sum(int x) {
    return __builtin_amdgcn_readfirstlane(
        (int)wave_reduce((uint32_t)x, [](uint32_t y, uint32_t z) { return y + z; }));
}

// A share of `total` blocks (below 2^31) among n, rounded up: their sum with n may pass 31 bits (300
// lists that name a few pages 28 million times each).
__host__ __device__ constexpr int share_of(int total, int n) {
    return (int)(((uint32_t)total + (uint32_t)n - 1) / (uint32_t)n);
}
static_assert(share_of(INT32_MAX, 512) == 1 << 22 && share_of(INT32_MAX, 1 << 20) == 1 << 11 &&
              share_of(1, 512) == 1 && share_of(1025, 512) == 3, "rounded up, without overflow");

// A workgroup's part: item, number of it, the item's parts and the first one's slot.
struct Part {
    int item, part, parts, slot;
};

// The plan of few items (below; kWaveItems at most, as they are where no splits are asked for): each
// wave makes it by itself, K items a lane in registers, without a barrier. Workgroup g's part, or
// none (item < 0). (In LDS over the workgroup it took 1 us longer: 12.3 us instead of 11.1 for 8 heads
// of 256 listed pages, 27.7 instead of 26.7 for 128 sequences of 512 .. 8192 tokens.)
constexpr int kWaveItems = 4 * kWave;

template <int HEADS, Form FORM, int K>
__device__ __forceinline__ Part wave_plan(const EntryArgs &a, int g, int lane) {
    int n[K], mine = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int i = k * kWave + lane;
        n[k] = entry_keys<HEADS, FORM>(a, min(i, a.items - 1)).blocks;
        if (i >= a.items) n[k] = 0;
        mine += n[k];
    }
    const int total = wave_sum(mine);
    const int spare = a.round - a.items / 2;  // (parts are rounded up by half of one)
    int p[K], c = max(a.least, share_of(total, spare));
    for (;; c += max(1, c >> 4)) {
        mine = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            p[k] = (int)((uint32_t)(n[k] + c - 1) / (uint32_t)c);
            mine += p[k];
        }
        if (wave_sum(mine) <= a.round) break;
    }
    Part r = {-1, 0, 1, 0};
    int before = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int upto = before + wave_scan(p[k]), first = upto - p[k];
        const uint64_t mask = __builtin_amdgcn_ballot_w64(g >= first && g < upto);
        if (mask) {
            const int at = __builtin_ctzll(mask);
            r.item = k * kWave + at;
            r.slot = __builtin_amdgcn_readlane(first, at);
            r.part = g - r.slot;
            r.parts = __builtin_amdgcn_readlane(p[k], at);
        }
        before = __builtin_amdgcn_readlane(upto, kWave - 1);
    }
    return r;
}

// The launch's work is the items' (sequence, kv head) 64-key blocks, at least one an item. A
// workgroup takes one part of an item. With at most kPlanItems items every workgroup counts the
// blocks (from the lengths; in LDS where items are many) and finds its own; parts are of at most c
// blocks, an item's equal to a block:
//   few items (half the workgroups that run at once at most): c is the least, within a sixteenth,
//             that needs no more parts than those. (Equal runs of blocks over the items' borders
//             cost two starts and two merges each: 31 us instead of 27 for 128 sequences of 512 ..
//             8192 tokens.)
//   more:     c is a workgroup's share of all blocks: an item no longer than that is one part, and
//             a workgroup takes several parts in turn. (Equal runs of blocks: 94 us instead of 48
//             for 128 x 16 heads of 16 .. 1024 tokens.)
// With more items, or none of more than kLeastBlocks blocks, a part is an item. The 4 waves take a
// part's blocks in turn, keep a flash-decoding state each and merge in LDS; an item in one part is
// stored, the parts of others go to the workspace, and the part that arrives last merges them all.
// (Registers: lists of the int8 cache at head_dim 128 take all 256, and for 8 or 16 heads spill 20 to
// 64 bytes a lane outside the loop over blocks, at a part's start and its merge: 22.0 us with 8 heads
// to a kv head, 21.0 with 4, for 16 x 8 kv heads of 128 pages.)
template <int D, int BITS, int HEADS, bool PAGED, Form FORM>
__global__ __launch_bounds__(kEntryThreads, kWgPerCu) void decode_entries(EntryArgs a, float *out) {
    using Slots = RowSlots<D, HEADS>;
    constexpr int DB = D / 16;  // 16-wide output blocks
    constexpr int N = Slots::N, QD = D / 4;
    __shared__ int32_t sPlan[kPlanItems + 1];  // blocks of the items, then prefixes
    __shared__ int32_t sWave[kDecodeWaves];
    __shared__ f32x4 sRow[kDecodeWaves * N];
    __shared__ float2 sML[kDecodeWaves * 16];
    __shared__ int32_t sItem, sPart, sParts, sSlot;
    __shared__ uint32_t sLast;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int g = blockIdx.x;

    Part part_of = {g, 0, 1, 0};
    const bool by_wave = a.few && a.items <= kWaveItems;
    if (a.planned && by_wave) {
        part_of = a.items <= kWave ? wave_plan<HEADS, FORM, 1>(a, g, lane)
                                   : wave_plan<HEADS, FORM, 4>(a, g, lane);
        if (part_of.item < 0) return;
    }
    const int per = (a.items + kEntryThreads - 1) / kEntryThreads;  // items of a thread's plan
    const int from = min(tid * per, a.items), to = min(from + per, a.items);
    int units = a.planned && by_wave ? g + 1 : a.items;  // parts
    if (a.planned && !by_wave) {
        int mine = 0;
        for (int i = from; i < to; ++i) {
            const int n = entry_keys<HEADS, FORM>(a, i).blocks;
            sPlan[i] = n;
            mine += n;
        }
        const int total = workgroup_sum(mine, sWave);
        int c = max(a.least, share_of(total, a.round));
        auto parts_of = [&](int i) { return (int)((uint32_t)(sPlan[i] + c - 1) / (uint32_t)c); };
        if (a.few) {
            const int spare = a.round - a.items / 2;  // (parts are rounded up by half of one)
            for (c = max(a.least, share_of(total, spare));; c += max(1, c >> 4)) {
                mine = 0;
                for (int i = from; i < to; ++i) mine += parts_of(i);
                if (workgroup_sum(mine, sWave) <= a.round) break;
            }
        }
        // Prefixes of the parts, which are the workgroups, and of those of items with several,
        // which are the slots: in the upper half of a word (few items: the slots are the parts).
        auto words = [&](int n) { return a.few || n == 1 ? n : n | n << 16; };
        int own = 0;
        for (int i = from; i < to; ++i) own += words(parts_of(i));
        int x = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 63) sWave[wave] = x;
        __syncthreads();
        int before = x - own, all = 0;
        for (int w = 0; w < kDecodeWaves; ++w) {
            before += w < wave ? sWave[w] : 0;
            all += sWave[w];
        }
        for (int i = from; i < to; ++i) {
            const int n = words(parts_of(i));
            sPlan[i] = before;
            before += n;
        }
        if (tid == 0) sPlan[a.items] = all;
        units = __builtin_amdgcn_readfirstlane(a.few ? all : all & 0xffff);
        __syncthreads();
    }

    for (int unit = g; unit < units; unit += a.wgs) {
        // The item, this part of it, the item's parts and the first one's slot.
        int item = a.planned && by_wave ? part_of.item : unit, part = part_of.part, parts = part_of.parts;
        int slot = part_of.slot;
        if (a.planned && !by_wave) {
            for (int i = from; i < to; ++i) {
                const int here = sPlan[i], next = sPlan[i + 1];
                const int first = a.few ? here : here & 0xffff, end = a.few ? next : next & 0xffff;
                if (unit >= first && unit < end) {
                    sItem = i;
                    sPart = unit - first;
                    sParts = end - first;
                    sSlot = a.few ? here : here >> 16;
                }
            }
            __syncthreads();
            // Values read from LDS arrive in vector registers; all of these are uniform, and
            // moving them to scalar registers keeps the loop control and the addresses scalar.
            item = __builtin_amdgcn_readfirstlane(sItem);
            part = __builtin_amdgcn_readfirstlane(sPart);
            parts = __builtin_amdgcn_readfirstlane(sParts);
            slot = __builtin_amdgcn_readfirstlane(sSlot);
        }
        ItemKeys ik = entry_keys<HEADS, FORM>(a, item);
        ik.len = __builtin_amdgcn_readfirstlane(ik.len);
        ik.lo = __builtin_amdgcn_readfirstlane(ik.lo);
        ik.first_block = __builtin_amdgcn_readfirstlane(ik.first_block);
        ik.blocks = __builtin_amdgcn_readfirstlane(ik.blocks);
        if constexpr (FORM == kListed) ik.count = __builtin_amdgcn_readfirstlane(ik.count);
        const int tile = FORM == kChunk ? item % a.tiles : 0;
        const int pair = FORM == kChunk ? item / a.tiles : item;
        const int b = pair / a.kv_heads, kvh = pair % a.kv_heads;
        // columns of the item, HEADS at most
        const int cols = FORM == kChunk ? min(HEADS, a.q_len * a.group - tile * HEADS) : a.group;
        // The part's blocks of the item: the first `more` parts have one more than the others.
        const int least = (uint32_t)ik.blocks / (uint32_t)parts, more = ik.blocks - least * parts;
        const int s_blk = part * least + min(part, more);
        const int e_blk = s_blk + least + (part < more ? 1 : 0);
        if (ik.bad && s_blk == 0 && tid == 0) flag_status(a.status, REEF_STATUS_BIT_BAD_LENGTH);

        const int k_begin = (ik.first_block + s_blk + wave) * kBlockKeys;
        const int k_end = min(FORM == kListed ? ik.count * kPage : ik.len,
                              (ik.first_block + e_blk) * kBlockKeys);
        const int n_pages = (ik.len + kPage - 1) / kPage;
        // the column whose operand this lane holds, and the one whose scores
        const int scored = col % HEADS;
        int lo = ik.lo, len = ik.len;
        Query<D> q;
        if constexpr (FORM == kChunk) {
            const int t = chunk_row<HEADS>(a, tile, scored);
            len = a.query_start + t + 1;
            lo = a.window > 0 ? max(0, len - a.window) : 0;
            const auto head = [&](int c) { return kvh * a.group + (tile * HEADS + c) % a.group; };
            const bool live = col < cols, scores = scored < cols;
            const int8_t *qrow = a.q + b * a.q_sb + (live ? head(col) : 0) * a.q_sh +
                                 (live ? chunk_row<HEADS>(a, tile, col) : 0) * a.q_st;
            float scale = 0.0f;
            if (scores) {
                const int h = head(scored);
                scale = a.q_gran == REEF_SCALE_PER_TENSOR ? a.qs[0]
                        : a.q_gran == REEF_SCALE_PER_HEAD ? a.qs[h]
                                                          : a.qs[((int64_t)b * a.q_heads + h) * a.q_len + t];
            }
            q = query_of<D, BITS>(qrow, live, scale * a.score_scale, grp);
        } else {
            const int head = kvh * a.group + col;
            q = load_query<D, BITS>(a, b, head, col < cols, kvh * a.group + scored, scored < cols, grp);
        }
        DecodeRun<D> st;
        reset_run<D>(st);
        bool bad_page = false;
        run_entries<D, BITS, HEADS, PAGED, FORM>(a, item, b, kvh, lo, len, ik.count, k_begin, k_end,
                                                 kDecodeWaves * kBlockKeys, n_pages, q, lane, st,
                                                 bad_page);
        if (bad_page) flag_status(a.status, REEF_STATUS_BIT_BAD_PAGE);
        // Row sums: this lane holds its column's partial over the keys of its lane group.
        float l = st.l_run;
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        float m = st.m_run;
        f32x4 o[DB];
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] = st.acc[d] * (st.s_run * (1.0f / 256.0f));
        merge_columns<D, HEADS>(m, l, o);
        if (col < HEADS) {
#pragma unroll
            for (int d = 0; d < DB; ++d) sRow[wave * N + col * QD + 4 * d + grp] = o[d];
            if (grp == 0) sML[wave * 16 + col] = float2{m, l};
        }
        __syncthreads();

        // A sequence with no keys ends with a sum of 0 and stores zeros.
        auto store = [&](int s, const RowRun &r) {
            if (s / QD >= cols) return;
            const float inv = r.l > 0.0f ? 1.0f / r.l : 0.0f;
            if constexpr (FORM == kChunk) {
                const int c = tile * HEADS + s / QD;
                float *orow = out + b * a.o_sb + (int64_t)(kvh * a.group + c % a.group) * a.o_sh +
                              (int64_t)(c / a.group) * a.o_st;
                *reinterpret_cast<f32x4 *>(orow + 4 * (s % QD)) = r.o * inv;
            } else {
                float *orow = out + ((int64_t)b * a.q_heads + kvh * a.group) * D;
                *reinterpret_cast<f32x4 *>(orow + 4 * s) = r.o * inv;
            }
        };
        if (parts == 1) {  // (uniform)
#pragma unroll
            for (int k = 0; k < Slots::PER; ++k) {
                const int s = tid + k * kEntryThreads;
                if (s < N) store(s, merge_slot<D, HEADS>(sRow, sML, s, kDecodeWaves));
            }
        } else {
            // (written and counted in as in decode.hip)
            auto part_at = [&](int i) {
                return reinterpret_cast<uint64_t *>(a.slots) +
                       (int64_t)(slot + i) * DecodeSlot<D>::ELEMS;
            };
            auto pack = [](float x0, float x1) {
                return (uint64_t)__float_as_uint(x0) | ((uint64_t)__float_as_uint(x1) << 32);
            };
            uint64_t *so = part_at(part);
#pragma unroll
            for (int k = 0; k < Slots::PER; ++k) {
                const int s = tid + k * kEntryThreads;
                if (s < N && s / QD < cols) {
                    const RowRun r = merge_slot<D, HEADS>(sRow, sML, s, kDecodeWaves);
                    part_store(so + s, pack(r.o[0], r.o[1]));
                    part_store(so + N + s, pack(r.o[2], r.o[3]));
                    if (s % QD == 0) part_store(so + 2 * N + s / QD, pack(r.m, r.l));
                }
            }
            part_stores_done();
            __syncthreads();
            if (tid == 0) sLast = part_count(a.counters + item) == (uint32_t)(parts - 1) ? 1u : 0u;
            __syncthreads();  // publishes sLast
            if (__builtin_amdgcn_readfirstlane(sLast)) {
                // Every thread merges its slots of the parts in order (of every GROUPS-th, and the
                // groups then in LDS): the same result whichever part arrived last. It reads
                // several parts before it uses the first: a round trip for them all, not one each.
                constexpr int AHEAD = 16 / Slots::PER;
                const int gi = tid / N;  // (PER > 1: 0)
                auto lo32 = [](uint64_t v) { return __uint_as_float((uint32_t)v); };
                auto hi32 = [](uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); };
                RowRun run[Slots::PER];
                part_claimed();
#pragma unroll
                for (int k = 0; k < Slots::PER; ++k) {
                    const int s = (tid + k * kEntryThreads) % N;
                    run[k] = {-INFINITY, 0.0f, f32x4{}};
                    if (s / QD >= cols) continue;
                    for (int i0 = gi; i0 < parts; i0 += Slots::GROUPS * AHEAD) {
                        uint64_t w[AHEAD][3];
#pragma unroll
                        for (int i = 0; i < AHEAD; ++i) {
                            const uint64_t *sl = part_at(min(i0 + i * Slots::GROUPS, parts - 1));
                            w[i][0] = part_load(sl + s);
                            w[i][1] = part_load(sl + N + s);
                            w[i][2] = part_load(sl + 2 * N + s / QD);
                        }
#pragma unroll
                        for (int i = 0; i < AHEAD; ++i)
                            if (i0 + i * Slots::GROUPS < parts)
                                merge_rows(run[k], lo32(w[i][2]), hi32(w[i][2]),
                                           f32x4{lo32(w[i][0]), hi32(w[i][0]), lo32(w[i][1]),
                                                 hi32(w[i][1])});
                    }
                }
                if (tid == 0) part_reset(a.counters + item);
                if constexpr (Slots::GROUPS == 1) {
#pragma unroll
                    for (int k = 0; k < Slots::PER; ++k) store(tid + k * kEntryThreads, run[k]);
                } else {
                    const int s = tid % N;
                    sRow[gi * N + s] = run[0].o;
                    if (s % QD == 0) sML[gi * 16 + s / QD] = float2{run[0].m, run[0].l};
                    __syncthreads();
                    if (tid < N) store(s, merge_slot<D, HEADS>(sRow, sML, s, Slots::GROUPS));
                }
            }
        }
        __syncthreads();  // frees what this part had in LDS
    }
}

// Launches `a`, whose items have `blocks` 64-key blocks at most (lists that name pages of the cache
// twice may have more); flat: the blocks of all fit 31 bits; num_splits as for decode.
template <int BITS, bool PAGED, Form FORM>
reef_status launch_entries(EntryArgs &a, int64_t head_dim, int64_t columns, int64_t blocks, bool flat,
                           int64_t num_splits, float *out, char *counters, char *slots,
                           hipStream_t stream) {
    const int64_t items = a.items;
    // Two workgroups a compute unit, one where items are few: an item's parts are half as many then
    // and the bytes take no longer (1 x 8 x 131071 tokens: 36 us against 43, 64 parts an item).
    const int64_t cus = compute_units();
    const int64_t round = num_splits > 0 ? ceil_div(items * num_splits, kDecodeWaves)
                                         : (2 * items <= cus ? 1 : kWgPerCu) * cus;
    const int64_t least = num_splits > 0 ? 1 : kLeastBlocks;
    a.few = (num_splits > 0 ? items : 2 * items) <= round;
    // (the plan has words for kPlanItems items and counts blocks in 31 bits; asked for fewer waves
    // than items: items)
    a.planned = flat && items <= kPlanItems && items * blocks < (int64_t(1) << 31) && blocks > least &&
                (a.few || num_splits == 0);
    a.least = (int32_t)least;
    // (of few items as many workgroups as parts: the search keeps to them; of more, slots for 2 round
    // parts are more than the items of several parts have)
    const int64_t wgs = !a.planned ? std::min(items, num_splits > 0 ? items : round)
                        : a.few    ? std::min(round, items * ceil_div(blocks, least)) : round;
    a.wgs = (int32_t)std::max<int64_t>(1, std::min<int64_t>(wgs, 1 << 20));
    a.round = a.wgs;
    a.counters = reinterpret_cast<uint32_t *>(counters);
    a.slots = reinterpret_cast<float *>(slots);
    const auto run = [&](auto *kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)a.wgs), dim3(kEntryThreads), 0, stream, a, out);
    };
    if (head_dim == 128)
        run(columns <= 4   ? decode_entries<128, BITS, 4, PAGED, FORM>
            : columns <= 8 ? decode_entries<128, BITS, 8, PAGED, FORM>
                           : decode_entries<128, BITS, 16, PAGED, FORM>);
    else
        run(columns <= 4   ? decode_entries<64, BITS, 4, PAGED, FORM>
            : columns <= 8 ? decode_entries<64, BITS, 8, PAGED, FORM>
                           : decode_entries<64, BITS, 16, PAGED, FORM>);
    return launch_status();
}

// A decode step's.
template <int BITS, bool PAGED, bool SEL>
reef_status launch_decode(const reef_decode_params *p, EntryArgs &a, float *out, void *workspace,
                          hipStream_t stream) {
    set_decode_args(p, a);
    // The tokens that a sequence may read. A list longer than the cache (pages listed twice)
    // gets no more workgroups than the workspace has slots for.
    const int64_t tokens = SEL ? (int64_t)a.max_sel * kPage : p->max_context;
    char *base = static_cast<char *>(workspace);
    return launch_entries<BITS, PAGED, SEL ? kListed : kAll>(
        a, p->head_dim, a.group, ceil_div(std::min(tokens, p->max_context), kBlockKeys),
        decode_flat(p, p->max_context) && decode_flat(p, tokens), p->num_splits, out, base,
        base + kDecodeCounterBytes, stream);
}

// A paged launch's table, or (block_table NULL) a contiguous cache.
bool use_table(const reef_decode_params *p, const int32_t *block_table,
               int64_t max_blocks_per_seq, int64_t num_pages, EntryArgs &a) {
    if (!a.context_lens || num_pages <= 0 || num_pages >= (int64_t(1) << 31) ||
        max_blocks_per_seq * kPage < p->max_context || max_blocks_per_seq >= (int64_t(1) << 30))
        return false;
    a.block_table = block_table;
    a.max_blocks = (int32_t)max_blocks_per_seq;
    a.num_pages = (int32_t)num_pages;
    return true;
}

// Decode over a cache of BITS, paged where there is a block table, over a list's pages where
// there is a list.
template <int BITS>
reef_status decode_any(const reef_decode_params *p, const int8_t *q, const float *q_scales,
                       const void *k, const void *v, const float *k_scales,
                       const float *v_scales, const int32_t *block_table,
                       int64_t max_blocks_per_seq, int64_t num_pages,
                       const int32_t *context_lens, const reef_page_selection *selection,
                       float *out, void *workspace, size_t workspace_bytes,
                       uint32_t *status_word, hipStream_t stream) {
    const reef_status st = decode_validate(p, q, q_scales, out, workspace, workspace_bytes);
    if (st != REEF_OK) return st;
    if (!k || !v || !k_scales || !v_scales || !aligned(k, 16) || !aligned(v, 16) ||
        !aligned(k_scales, 16) || !aligned(v_scales, 16) || !aligned(out, 16))
        return REEF_INVALID_ARGUMENT;
    EntryArgs a = {};
    a.q = q;
    a.qs = q_scales;
    a.k = static_cast<const int8_t *>(k);
    a.v = static_cast<const int8_t *>(v);
    a.ks = k_scales;
    a.vs = v_scales;
    a.context_lens = context_lens;
    a.status = status_word;
    if (block_table && !use_table(p, block_table, max_blocks_per_seq, num_pages, a))
        return REEF_INVALID_ARGUMENT;
    if (selection) {
        if (!selection->pages || !selection->counts || !context_lens || selection->max_pages <= 0 ||
            !aligned(selection->pages, 4) || !aligned(selection->counts, 4))
            return REEF_INVALID_ARGUMENT;
        if (selection->max_pages >= (int64_t(1) << 26)) return REEF_UNSUPPORTED;
        a.sel_pages = selection->pages;
        a.sel_counts = selection->counts;
        a.max_sel = (int32_t)selection->max_pages;
        return block_table ? launch_decode<BITS, true, true>(p, a, out, workspace, stream)
                           : launch_decode<BITS, false, true>(p, a, out, workspace, stream);
    }
    if constexpr (BITS == 8) return REEF_INVALID_ARGUMENT;  // decode.hip's
    else
        return block_table ? launch_decode<BITS, true, false>(p, a, out, workspace, stream)
                           : launch_decode<BITS, false, false>(p, a, out, workspace, stream);
}

}  // namespace

// A 64-key block of 16 columns costs about 1.4 ns of the whole GPU's time here, one of a 128-row
// tile 9 ns there, behind a copy of the cache and a schedule's start of 25 us. So a chunk runs here
// if it has few blocks (us a call, here against there: 2 x 12 heads of 64, 77 rows over 1021 keys 12
// against 29; 32 heads, 8 of keys, of 128, 64 rows over 4096 23 against 45; 12 heads of 64, 1024 rows
// over 1024 23 against 31) or if its tiles of 128 rows stay part empty (8 x 16 heads of 64, 16 rows
// over 6000 24 against 138; 2 x 32 heads, 4 of keys, of 128, 100 rows over 8000 95 against 98). With
// full tiles and many blocks it does not (32 heads of 128, 1024 rows over 1024: 66 against 44; 2 x 32,
// 512 over 2048 102 against 91); of few full tiles over many keys that gives some away (32 heads, 8 of
// keys, of 128, 128 rows over 8192: 51 against 67, 512 over 4608 99 against 103).
bool chunk_entries_fit(const reef_attention_params *p) {
    constexpr int64_t kRows = 128;
    const int64_t few = p->head_dim == 64 ? 32768 : 16384;
    const int64_t group = p->q_heads / p->kv_heads;
    if (p->q_len > (1 << 20) || p->q_len * group > (1 << 20)) return false;
    const int64_t items = p->batch * p->kv_heads * ceil_div(p->q_len * group, 16);
    const int64_t tiles = p->batch * p->q_heads * ceil_div(p->q_len, kRows);
    const int64_t end = p->query_start + p->q_len;
    const int64_t blocks = ceil_div(p->window > 0 ? std::min(end, std::min(end, p->window) + p->q_len) : end,
                                    kBlockKeys);
    return items <= kPlanItems && (items * blocks <= few || 2 * items <= 13 * tiles);
}

reef_status launch_chunk_int4(const reef_attention_params *p, const int8_t *q, const int64_t (&qst)[3],
                              const float *q_scales, const uint8_t *k_cache, const uint8_t *v_cache,
                              const float *k_scales, const float *v_scales, int64_t max_context,
                              const int32_t *block_table, int64_t max_blocks_per_seq,
                              int64_t num_pages, float *out, const int64_t (&ost)[3], char *counters,
                              char *slots, uint32_t *status_word, hipStream_t stream) {
    EntryArgs a = {};
    a.q = q;
    a.qs = q_scales;
    a.k = reinterpret_cast<const int8_t *>(k_cache);
    a.v = reinterpret_cast<const int8_t *>(v_cache);
    a.ks = k_scales;
    a.vs = v_scales;
    a.status = status_word;
    a.block_table = block_table;
    a.max_blocks = (int32_t)(block_table ? max_blocks_per_seq : 0);
    a.num_pages = (int32_t)(block_table ? num_pages : 0);
    a.batch = (int32_t)p->batch;
    a.q_heads = (int32_t)p->q_heads;
    a.kv_heads = (int32_t)p->kv_heads;
    a.group = (int32_t)(p->q_heads / p->kv_heads);
    a.max_context = (int32_t)(block_table ? 0 : max_context);
    a.window = (int32_t)std::min<int64_t>(p->window, INT32_MAX);
    a.q_gran = p->q_granularity;
    a.score_scale = p->softmax_scale * kLog2e;
    a.q_sb = qst[0], a.q_sh = qst[1], a.q_st = qst[2];
    a.o_sb = ost[0], a.o_sh = ost[1], a.o_st = ost[2];
    a.q_len = (int32_t)p->q_len;
    a.query_start = (int32_t)p->query_start;
    const int64_t columns = p->q_len * a.group, width = columns <= 4 ? 4 : columns <= 8 ? 8 : 16;
    a.tiles = (int32_t)ceil_div(columns, width);
    a.items = (int32_t)(p->batch * p->kv_heads * a.tiles);
    const int64_t blocks = ceil_div(p->query_start + p->q_len, kBlockKeys);
    return block_table ? launch_entries<4, true, kChunk>(a, p->head_dim, columns, blocks, true, 0, out,
                                                         counters, slots, stream)
                       : launch_entries<4, false, kChunk>(a, p->head_dim, columns, blocks, true, 0,
                                                          out, counters, slots, stream);
}

}  // namespace reef

using namespace reef;

extern "C" reef_status reef_attention_decode_int8_selected(
    const reef_decode_params *p, const int8_t *q, const float *q_scales, const int8_t *k_cache,
    const int8_t *v_cache, const float *k_scales, const float *v_scales,
    const int32_t *block_table, int64_t max_blocks_per_seq, int64_t num_pages,
    const int32_t *context_lens, const reef_page_selection *selection, float *out,
    void *workspace, size_t workspace_bytes, uint32_t *status_word, hipStream_t stream) {
    if (!selection) return REEF_INVALID_ARGUMENT;
    return decode_any<8>(p, q, q_scales, k_cache, v_cache, k_scales, v_scales, block_table,
                         max_blocks_per_seq, num_pages, context_lens, selection, out, workspace,
                         workspace_bytes, status_word, stream);
}

extern "C" reef_status reef_attention_decode_int4(
    const reef_decode_params *p, const int8_t *q, const float *q_scales, const uint8_t *k_cache,
    const uint8_t *v_cache, const float *k_scales, const float *v_scales,
    const int32_t *block_table, int64_t max_blocks_per_seq, int64_t num_pages,
    const int32_t *context_lens, const reef_page_selection *selection, float *out,
    void *workspace, size_t workspace_bytes, uint32_t *status_word, hipStream_t stream) {
    return decode_any<4>(p, q, q_scales, k_cache, v_cache, k_scales, v_scales, block_table,
                         max_blocks_per_seq, num_pages, context_lens, selection, out, workspace,
                         workspace_bytes, status_word, stream);
}
