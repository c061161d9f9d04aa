// Pages that a query selects (gfx950): bounds of every page's keys, a query's scores against
// them, and the best `budget` pages of each (sequence, kv head), for the decode step over a list
// of pages (decode_entries.hip).
//
// A page's bounds are the largest and the least key of each channel, hi and lo, as int8 codes of
// one scale S a page, rounded outwards. For any key x of the page and a query q,
//   q . x = sum_d q_d x_d <= S * sum_d (max(q_d, 0) hi_d + min(q_d, 0) lo_d),
// up to fp32's rounding: S and the quotients are rounded before the codes are, and a code past 127
// is cut to it. With codes of q the sum is a product of [max(q, 0), min(q, 0)] and [hi, lo], 2 D
// long: int8 matrix instructions, exact. A page costs 2 D + 4 bytes to score, 1/16 of its int8 keys
// and values.
#include <algorithm>

#include "kv_int4.hpp"
#include "reef_common.hpp"

namespace reef {
namespace {

// --- bounds --------------------------------------------------------------------------------

constexpr int kBoundWaves = 4;  // waves of a workgroup
// Pages a wave takes in turn, the next one's rows loading while one is reduced, where a launch has
// pages for more than kBoundFill waves of them; one otherwise (a decode step's).
constexpr int kBoundPages = 4;
constexpr int64_t kBoundFill = 8192;

struct BoundArgs {
    const uint8_t *k;
    const float *ks;
    const int32_t *start;
    const int32_t *lens;   // may be null
    const int32_t *table;  // paged only
    int8_t *bounds;
    float *scales;
    int32_t kv_heads, new_tokens, max_context, max_blocks, num_pages;
    int32_t turns;  // pages a wave
    uint32_t *status;
};

// A wave takes a page at a time. A lane reads 4 bytes (BITS 8: four channels; 4: four of either half of
// the row) of every R-th token's row, so that a load covers 256 bytes in order, and keeps their
// extremes. Lanes that hold the same channels then meet: over 32 lanes one side keeps the
// largest, the other the least; in 4 bits over 16 lanes either keeps one half of the row; what
// copies are left combine. Each lane ends with four codes of one bound.
template <int D, int BITS>
__global__ __launch_bounds__(kBoundWaves * kWave) void page_bounds(BoundArgs a) {
    constexpr int RB = D * BITS / 8;      // bytes of a row
    constexpr int LPR = RB / 4;           // lanes a row
    constexpr int R = kWave / LPR;        // rows of a load
    constexpr int C = BITS == 8 ? 4 : 8;  // channels of a lane
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b = blockIdx.z, kvh = blockIdx.y;
    const int start = a.start[b];
    if (start < 0 || start > a.max_context - a.new_tokens) {
        if (blockIdx.x == 0 && kvh == 0 && threadIdx.x == 0)
            flag_status(a.status, start < 0 ? REEF_STATUS_BIT_BAD_LENGTH : REEF_STATUS_BIT_CAPACITY);
        return;
    }
    int end = start + a.new_tokens;
    if (a.lens) {
        const int len = a.lens[b];
        if (len < 0 || len > a.max_context) {
            if (blockIdx.x == 0 && kvh == 0 && threadIdx.x == 0)
                flag_status(a.status, REEF_STATUS_BIT_BAD_LENGTH);
            return;
        }
        end = min(end, len);
        if (end <= start) return;
    }
    const int stop = (end + kPage - 1) / kPage;
    int page_idx = start / kPage + (int)blockIdx.x * kBoundWaves * a.turns + wave;
    const int last = min(stop, start / kPage + ((int)blockIdx.x + 1) * kBoundWaves * a.turns) - 1;
    if (page_idx > last) return;
    const int j = lane % LPR, g = lane / LPR;
    struct Rows {
        uint32_t w[kPage / R];
        float s[kPage / R];
        int64_t slot;  // index of this (page, kv head); -1: no such page
    };
    auto load = [&](int idx) {
        Rows r;
        if (a.table) {
            const int page = a.table[(int64_t)b * a.max_blocks + idx];
            r.slot = page < 0 || page >= a.num_pages ? -1 : (int64_t)page * a.kv_heads + kvh;
        } else {
            r.slot = ((int64_t)b * a.kv_heads + kvh) * (a.max_context / kPage) + idx;
        }
        const int64_t at = max(r.slot, (int64_t)0);
        const uint8_t *rows = a.k + at * (kPage * RB) + g * RB + 4 * j;
        const float *ks = a.ks + at * kPage + g;
#pragma unroll
        for (int i = 0; i < kPage / R; ++i) {
            r.w[i] = *reinterpret_cast<const uint32_t *>(rows + i * R * RB);
            r.s[i] = ks[i * R];
        }
        return r;
    };
    Rows next = load(page_idx);
    for (; page_idx <= last; page_idx += kBoundWaves) {
        const Rows rows = next;
        next = load(min(page_idx + kBoundWaves, last));
        const int64_t slot = rows.slot;
        if (slot < 0) {
            if (lane == 0) flag_status(a.status, REEF_STATUS_BIT_BAD_PAGE);
            continue;
        }
        const int live = min(kPage, end - page_idx * kPage);
        float hi[C], lo[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            hi[c] = -INFINITY;
            lo[c] = INFINITY;
        }
        auto key = [&](int i, int c) {
            const int code = BITS == 8 ? (int)(int8_t)(rows.w[i] >> (8 * c))
                                       : (int)((rows.w[i] >> (8 * (c % 4) + 4 * (c / 4))) & 0xf) - kInt4Zero;
            return (float)code * rows.s[i];
        };
        if (live == kPage) {
#pragma unroll
            for (int i = 0; i < kPage / R; i += 2) {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const float x = key(i, c), y = key(i + 1, c);
                    hi[c] = i ? fmaxf(fmaxf(hi[c], x), y) : fmaxf(x, y);
                    lo[c] = i ? fminf(fminf(lo[c], x), y) : fminf(x, y);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPage / R; ++i) {
                const bool in = i * R + g < live;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const float x = key(i, c);
                    hi[c] = in ? fmaxf(hi[c], x) : hi[c];
                    lo[c] = in ? fminf(lo[c], x) : lo[c];
                }
            }
        }
        // Lanes 0-31 go on with the largest, the others with the least, negated: maxima either way.
        // A swap of halves leaves a lane its own and its partner's of what it goes on with.
        auto meet = [](auto r) { return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])); };
        const bool least = lane >= 32;
        float m[C];
#pragma unroll
        for (int c = 0; c < C; ++c)
            m[c] = meet(__builtin_amdgcn_permlane32_swap(__float_as_uint(hi[c]), __float_as_uint(-lo[c]),
                                                         false, false));
        float n[4];
        const bool upper = BITS == 4 && (lane & 16);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            if constexpr (BITS == 4)
                n[c] = meet(__builtin_amdgcn_permlane16_swap(
                    __float_as_uint(m[c]), __float_as_uint(m[C - 4 + c]), false, false));
            else
                n[c] = D == 64 ? xor16_max(m[c]) : m[c];
            if constexpr (BITS == 4 && D == 64)
                n[c] = fmaxf(n[c], __int_as_float(__builtin_amdgcn_mov_dpp(
                                       __float_as_int(n[c]), 0x128, 0xf, 0xf, true)));  // row_ror 8
        }
        constexpr int kSplit = BITS == 4 ? 16 : 32;  // lanes of one bound (and half)
        // (the largest magnitude: not below zero, so the order of the words is the values')
        const float lane_top = fmaxf(fmaxf(fmaxf(n[0], n[1]), fmaxf(n[2], n[3])), 0.0f);
        const float top = __uint_as_float(
            wave_reduce(__float_as_uint(lane_top), [](uint32_t x, uint32_t y) { return max(x, y); }));
        const float scale = int8_scale(top);
        uint32_t packed = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            // ceil(hi / S), or -floor(lo / S) = ceil(-lo / S), rounded outwards
            const float code = fminf(__builtin_ceilf(n[c] / scale), 127.0f);
            packed |= ((uint32_t)(int)(least ? -code : code) & 0xffu) << (8 * c);
        }
        if (lane % kSplit < LPR)
            *reinterpret_cast<uint32_t *>(a.bounds + slot * 2 * D + (least ? D : 0) +
                                          (upper ? D / 2 : 0) + 4 * j) = packed;
        if (lane == 0) a.scales[slot] = scale;
    }
}

template <int BITS>
reef_status launch_bounds(const reef_kv_append_params *p, const int32_t *start, const int32_t *lens,
                          const void *k, const float *ks, const int32_t *block_table,
                          int64_t max_blocks_per_seq, int64_t num_pages, int8_t *bounds,
                          float *bound_scales, uint32_t *status_word, hipStream_t stream) {
    if (!p || !start || !k || !ks || !bounds || !bound_scales || p->batch <= 0 ||
        p->kv_heads <= 0 || p->head_dim <= 0 || p->new_tokens <= 0 || p->max_context <= 0 ||
        p->max_context % kPage != 0)
        return REEF_INVALID_ARGUMENT;
    if (p->new_tokens > p->max_context) return REEF_CAPACITY;
    const int64_t pages = ceil_div(p->new_tokens, kPage) + 1;  // that T tokens may fall in
    const int64_t turns = pages * p->batch * p->kv_heads > kBoundFill * kBoundPages ? kBoundPages : 1;
    const int64_t groups = ceil_div(pages, kBoundWaves * turns);
    if ((p->head_dim != 64 && p->head_dim != 128) || p->max_context >= (int64_t(1) << 30) ||
        p->batch > 65535 || p->kv_heads > 65535 || groups > kGridMost256)
        return REEF_UNSUPPORTED;
    if (!aligned(k, 16) || !aligned(ks, 4) || !aligned(bounds, 16) || !aligned(bound_scales, 4))
        return REEF_INVALID_ARGUMENT;
    if (block_table && (max_blocks_per_seq <= 0 || num_pages <= 0 ||
                        max_blocks_per_seq * kPage < p->max_context ||
                        num_pages >= (int64_t(1) << 31) ||
                        max_blocks_per_seq >= (int64_t(1) << 26)))
        return REEF_INVALID_ARGUMENT;
    BoundArgs a;
    a.k = static_cast<const uint8_t *>(k);
    a.ks = ks;
    a.start = start;
    a.lens = lens;
    a.table = block_table;
    a.bounds = bounds;
    a.scales = bound_scales;
    a.kv_heads = (int32_t)p->kv_heads;
    a.new_tokens = (int32_t)p->new_tokens;
    a.max_context = (int32_t)p->max_context;
    a.max_blocks = (int32_t)(block_table ? max_blocks_per_seq : 0);
    a.num_pages = (int32_t)(block_table ? num_pages : 0);
    a.turns = (int32_t)turns;
    a.status = status_word;
    const dim3 grid((unsigned)groups, (unsigned)p->kv_heads, (unsigned)p->batch);
    if (p->head_dim == 128)
        hipLaunchKernelGGL((page_bounds<128, BITS>), grid, dim3(kBoundWaves * kWave), 0, stream, a);
    else
        hipLaunchKernelGGL((page_bounds<64, BITS>), grid, dim3(kBoundWaves * kWave), 0, stream, a);
    return launch_status();
}

// --- selection -------------------------------------------------------------------------------

constexpr int kPickThreads = 1024; // of a selecting workgroup
constexpr int kPickWaves = kPickThreads / kWave;
// A page's place in the order, larger is better: scores as unsigned words in their order, and
// beyond them the pages that are always taken and those that cannot be.
constexpr uint32_t kAlways = 0xffffffffu, kNever = 0;

struct SelectArgs {
    const int8_t *q;
    const float *qs;
    const int8_t *bounds;
    const float *scales;
    const int32_t *table;  // paged only
    const int32_t *lens;
    uint32_t *keys;  // [items, max_pages]
    int32_t *pages, *counts;
    uint32_t *status;
    int32_t q_heads, kv_heads, group, items;
    int32_t max_context, max_pages;  // max_pages = max_context / 16
    int32_t max_blocks, num_pages;
    int32_t budget, sinks, recent, q_gran;
};

__device__ __forceinline__ uint32_t score_key(float score) {
    const uint32_t u = __float_as_uint(score + 0.0f);  // (-0 is 0)
    const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
    return k < 1 ? 1 : k;
}

// Bytes of a word above and below zero.
__device__ __forceinline__ void split_signs(uint32_t w, uint32_t &above, uint32_t &below) {
    const uint32_t negative = ((w >> 7) & 0x01010101u) * 0xffu;
    above = w & ~negative;
    below = w & negative;
}

__device__ __forceinline__ int item_pages(const SelectArgs &a, int b) {
    const int len = a.lens[b];
    return len < 1 || len > a.max_context ? 0 : (len + kPage - 1) / kPage;
}

// Keys of 64 pages a wave: four 16-page x 16-head products. The bounds' rows are the columns of
// the product (lane % 16), so the group's heads lie in a lane's four registers and over lane
// groups, and lane group t ends with tile t's pages: one key a lane, in page order.
// A wave a workgroup: workgroups go around the XCDs in turn, and with 256 pages each the last pages of
// a cache, which few sequences have, fell to the same ones (selection for 16 x 8 heads of 1024 .. 2048
// pages: 18.6 us instead of 20.0).
template <int D>
__global__ __launch_bounds__(kWave) void score_pages(SelectArgs a) {
    constexpr int S = 2 * D / 64;  // slices of a row of bounds
    const int lane = threadIdx.x, col = lane & 15, grp = lane >> 4;
    const int item = blockIdx.y, b = item / a.kv_heads, kvh = item - b * a.kv_heads;
    const int first = (int)blockIdx.x * kWave;
    const int page_idx = first + lane;
    // (read beside the length, not after it; past the sequence's pages it is not used)
    int page = a.table ? a.table[(int64_t)b * a.max_blocks + min(page_idx, a.max_pages - 1)] : page_idx;
    const int n = item_pages(a, b);
    if (first >= n) return;
    const bool here = page_idx < n;
    const bool ok = !here || !a.table || (page >= 0 && page < a.num_pages);
    if (!here || !ok) page = 0;
    // row of bounds of page 0, between pages
    const int64_t base = a.table ? kvh : (int64_t)item * a.max_pages, step = a.table ? a.kv_heads : 1;
    if (!ok) flag_status(a.status, REEF_STATUS_BIT_BAD_PAGE);
    uint32_t key = kAlways;
    if (n > a.budget) {
        i32x4 x[4][S];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int8_t *row = a.bounds + (base + __shfl(page, 16 * t + col) * step) * (2 * D);
#pragma unroll
            for (int s = 0; s < S; ++s)
                x[t][s] = *reinterpret_cast<const i32x4 *>(row + 64 * s + 16 * grp);
        }
        const float scale = a.scales[base + page * step];
        // The heads' operands: lane % 16 is the head, its slices [above, below].
        i32x4 q[S];
        const bool head_ok = col < a.group;
        const int8_t *qrow = a.q + ((int64_t)b * a.q_heads + kvh * a.group + (head_ok ? col : 0)) * D;
#pragma unroll
        for (int s = 0; s < S / 2; ++s) {
            const i32x4 w = *reinterpret_cast<const i32x4 *>(qrow + 64 * s + 16 * grp);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t above, below;
                split_signs(head_ok ? (uint32_t)w[i] : 0u, above, below);
                q[s][i] = (int)above;
                q[S / 2 + s][i] = (int)below;
            }
        }
        float qs[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int head = kvh * a.group + min(4 * grp + i, a.group - 1);  // (dead ones repeat one)
            qs[i] = a.q_gran == REEF_SCALE_PER_TENSOR ? a.qs[0]
                    : a.q_gran == REEF_SCALE_PER_HEAD ? a.qs[head]
                                                      : a.qs[(int64_t)b * a.q_heads + head];
        }
        float best = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            i32x4 sum = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < S; ++s) sum = mfma_16x16x64_i8(q[s], x[t][s], sum);
            const float ps = __shfl(scale, 16 * t + col);
            float most = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * grp + i < a.group) most = fmaxf(most, (float)sum[i] * (qs[i] * ps));
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            if (grp == t) best = most;
        }
        const bool always = page_idx < a.sinks || page_idx >= n - a.recent;
        key = always ? kAlways : score_key(best);
    }
    if (!ok) key = kNever;
    if (here) a.keys[(int64_t)item * a.max_pages + page_idx] = key;
}

constexpr int kDigit = 8, kBins = 1 << kDigit;
constexpr int kDigits = (32 + kDigit - 1) / kDigit;

struct PickShared {
    int bins[kDigits][kBins];  // keys of each value of a digit
    uint32_t all, any;         // bits of all scores, of any
    int always;                // pages that are taken whatever the scores
    uint32_t least;            // the last key so far, and the keys beyond its digit's value
    int above, done;
    int2 counts[kPickWaves];
};

// Wave 0, after a count of a digit (`shift` bits below it): the largest value that `rem` keys of
// the range reach, or exactly so many. Lane l holds the values 4 l .. 4 l + 3 from the top.
__device__ __forceinline__ void pick_digit(PickShared &sh, const int *bins, uint32_t least, int shift,
                                           int above, int rem, int lane) {
    int c[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c[i] = bins[kBins - 1 - (4 * lane + i)];
        sum += c[i];
    }
    const int upto = wave_scan(sum);  // of this lane's values and those above
    const uint64_t enough = __builtin_amdgcn_ballot_w64(upto >= rem);
    if (enough == 0) {  // fewer than that in all: every one of them
        if (lane == 0) {
            sh.least = least;
            sh.done = 1;
        }
        return;
    }
    if (lane != __builtin_ctzll(enough)) return;
    int run = upto - sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (run + c[i] >= rem) {
            sh.least = least | (uint32_t)(kBins - 1 - (4 * lane + i)) << shift;
            sh.above = above + run;
            sh.done = run + c[i] == rem ? 1 : 0;
            break;
        }
        run += c[i];
    }
}

// Keys of the pages that a thread holds: page first + 64 r + lane for r < R. In registers where a
// cache has up to 1024 R pages (read beside the sequence's length), read again at each use where
// it has more.
template <int R>
struct HeldKeys {
    uint32_t key[R];
    __device__ __forceinline__ HeldKeys(const SelectArgs &a, const uint32_t *keys, int wave, int lane,
                                        int b, int &n) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            key[r] = keys[min((wave * R + r) * kWave + lane, a.max_pages - 1)];
        n = item_pages(a, b);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if ((wave * R + r) * kWave + lane >= n) key[r] = kNever;
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll
        for (int r = 0; r < R; ++r) f(r, key[r]);
    }
};
template <>
struct HeldKeys<0> {
    const uint32_t *keys;
    int first, n, lane, rounds;
    __device__ __forceinline__ HeldKeys(const SelectArgs &a, const uint32_t *k, int wave, int l, int b,
                                        int &count)
        : keys(k), lane(l) {
        count = n = item_pages(a, b);
        rounds = (n + kPickThreads - 1) / kPickThreads;
        first = wave * rounds * kWave;
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        for (int r = 0; r < rounds; ++r) {
            const int i = first + 64 * r + lane;
            f(r, i < n ? keys[i] : kNever);
        }
    }
};

// One workgroup an item: the budget-th largest of its n keys, then the pages above it and the first
// of those at it, in page order. Wave w holds a run of pages, 64 at a time. The last key taken is found digit by
// digit from the highest bit in which scores differ (they share sign and most of the exponent): the
// keys of the range so far are counted by the digit's value in LDS, and the first value that enough
// of them reach is the next range, until exactly enough do. Two digits mostly: 8.1 us of a launch of
// 8 items of 8192 pages (bit by bit 12, with a pass over the keys in memory a bit 63), 5.2 of one of
// 128 items of up to 2048.
template <int R>
__global__ __launch_bounds__(kPickThreads) void pick_pages(SelectArgs a) {
    __shared__ PickShared sh;
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int item = blockIdx.x, b = item / a.kv_heads;
    int n;
    const HeldKeys<R> held(a, a.keys + (int64_t)item * a.max_pages, wave, lane, b, n);
    for (int i = tid; i < kDigits * kBins; i += kPickThreads) sh.bins[0][i] = 0;
    if (tid == 0) {
        sh.all = ~0u;
        sh.any = 0;
        sh.always = 0;
        if (n == 0 && item == b * a.kv_heads) flag_status(a.status, REEF_STATUS_BIT_BAD_LENGTH);
    }
    __syncthreads();
    const int rounds = R ? R : (n + kPickThreads - 1) / kPickThreads;
    const int first = wave * rounds * kWave;
    uint32_t t = kNever;
    if (n > a.budget) {
        uint32_t all = ~0u, any = 0;
        int always = 0;
        held.each([&](int, uint32_t key) {
            if (key != kNever && key != kAlways) {
                all &= key;
                any |= key;
            }
            always += __popcll(__builtin_amdgcn_ballot_w64(key == kAlways));
        });
        all = wave_reduce(all, [](uint32_t x, uint32_t y) { return x & y; });
        any = wave_reduce(any, [](uint32_t x, uint32_t y) { return x | y; });
        if (lane == 0) {
            atomicAnd(&sh.all, all);
            atomicOr(&sh.any, any);
            if (always) atomicAdd(&sh.always, always);
        }
        __syncthreads();
        all = __builtin_amdgcn_readfirstlane(sh.all);
        any = __builtin_amdgcn_readfirstlane(sh.any);
        int above = __builtin_amdgcn_readfirstlane(sh.always);
        const uint32_t differ = all ^ any;
        int left = differ ? 32 - __builtin_clz(differ) : 0;  // bits below those that all share
        t = left == 32 ? 0 : all & ~0u << left;
        if (above >= a.budget) {  // sinks and recent pages are the budget: no score matters
            t = kAlways;
            left = 0;
        }
#pragma unroll
        for (int digit = 0; digit < kDigits; ++digit) {
            if (left == 0) break;
            const int shift = max(left - kDigit, 0);
            held.each([&](int, uint32_t key) {
                // (a digit of fewer bits at the end: values below kBins all the same)
                if (key != kNever && key != kAlways && (left == 32 || (key ^ t) >> left == 0))
                    atomicAdd(&sh.bins[digit][(key - t) >> shift], 1);
            });
            __syncthreads();
            if (wave == 0) pick_digit(sh, sh.bins[digit], t, shift, above, a.budget - above, lane);
            __syncthreads();
            t = (uint32_t)__builtin_amdgcn_readfirstlane((int)sh.least);
            above = __builtin_amdgcn_readfirstlane(sh.above);
            if (__builtin_amdgcn_readfirstlane(sh.done)) break;
            left = shift;
        }
    }
    // the pages above the last key, and those at it (a page that cannot be taken never is)
    int above = 0, at = 0;
    held.each([&](int, uint32_t key) {
        above += __popcll(__builtin_amdgcn_ballot_w64(key > t));
        at += __popcll(__builtin_amdgcn_ballot_w64(key == t && key != kNever));
    });
    if (lane == 0) sh.counts[wave] = make_int2(above, at);
    __syncthreads();
    int before0 = 0, before1 = 0, total0 = 0, total1 = 0;
#pragma unroll
    for (int w = 0; w < kPickWaves; ++w) {
        const int2 x = sh.counts[w];
        before0 += w < wave ? x.x : 0;
        before1 += w < wave ? x.y : 0;
        total0 += x.x;
        total1 += x.y;
    }
    const int need = min(a.budget - total0, total1);  // of those at it
    int out = before0 + min(before1, need), ties = before1;
    int32_t *list = a.pages + (int64_t)item * a.budget;
    const uint64_t below = (uint64_t(1) << lane) - 1;
    held.each([&](int r, uint32_t key) {
        const uint64_t eq = __builtin_amdgcn_ballot_w64(key == t && key != kNever);
        const bool take = key > t || ((eq >> lane & 1) && ties + __popcll(eq & below) < need);
        const uint64_t taken = __builtin_amdgcn_ballot_w64(take);
        if (take) list[out + __popcll(taken & below)] = first + r * kWave + lane;
        out += __popcll(taken);
        ties += __popcll(eq);
    });
    const int count = total0 + need;
    for (int i = count + threadIdx.x; i < a.budget; i += kPickThreads) list[i] = -1;
    if (threadIdx.x == 0) a.counts[item] = count;
}

bool select_sizes(const reef_decode_params *p) {
    return p && p->batch > 0 && p->q_heads > 0 && p->kv_heads > 0 && p->max_context > 0 &&
           p->max_context % kPage == 0 && p->q_heads % p->kv_heads == 0;
}

}  // namespace
}  // namespace reef

using namespace reef;

extern "C" reef_status reef_kv_page_bounds_int8(const reef_kv_append_params *p,
                                                const int32_t *start_positions,
                                                const int8_t *k_cache, const float *k_scales,
                                                const int32_t *block_table,
                                                int64_t max_blocks_per_seq, int64_t num_pages,
                                                int8_t *bounds, float *bound_scales,
                                                uint32_t *status_word, hipStream_t stream) {
    return launch_bounds<8>(p, start_positions, nullptr, k_cache, k_scales, block_table,
                            max_blocks_per_seq, num_pages, bounds, bound_scales, status_word, stream);
}

extern "C" reef_status reef_kv_page_bounds_int4(const reef_kv_append_params *p,
                                                const int32_t *start_positions,
                                                const uint8_t *k_cache, const float *k_scales,
                                                const int32_t *block_table,
                                                int64_t max_blocks_per_seq, int64_t num_pages,
                                                int8_t *bounds, float *bound_scales,
                                                uint32_t *status_word, hipStream_t stream) {
    return launch_bounds<4>(p, start_positions, nullptr, k_cache, k_scales, block_table,
                            max_blocks_per_seq, num_pages, bounds, bound_scales, status_word, stream);
}

extern "C" reef_status reef_kv_page_bounds_int8_ragged(
    const reef_kv_append_params *p, const int32_t *start_positions, const int32_t *context_lens,
    const int8_t *k_cache, const float *k_scales, const int32_t *block_table,
    int64_t max_blocks_per_seq, int64_t num_pages, int8_t *bounds, float *bound_scales,
    uint32_t *status_word, hipStream_t stream) {
    if (!context_lens) return REEF_INVALID_ARGUMENT;
    return launch_bounds<8>(p, start_positions, context_lens, k_cache, k_scales, block_table,
                            max_blocks_per_seq, num_pages, bounds, bound_scales, status_word, stream);
}

extern "C" reef_status reef_kv_page_bounds_int4_ragged(
    const reef_kv_append_params *p, const int32_t *start_positions, const int32_t *context_lens,
    const uint8_t *k_cache, const float *k_scales, const int32_t *block_table,
    int64_t max_blocks_per_seq, int64_t num_pages, int8_t *bounds, float *bound_scales,
    uint32_t *status_word, hipStream_t stream) {
    if (!context_lens) return REEF_INVALID_ARGUMENT;
    return launch_bounds<4>(p, start_positions, context_lens, k_cache, k_scales, block_table,
                            max_blocks_per_seq, num_pages, bounds, bound_scales, status_word, stream);
}

extern "C" size_t reef_kv_select_pages_workspace_bytes(const reef_decode_params *p) {
    if (!select_sizes(p) || p->batch * p->kv_heads > 65535 || p->max_context >= (int64_t(1) << 30))
        return 0;
    return (size_t)(p->batch * p->kv_heads * (p->max_context / kPage) * 4);
}

extern "C" reef_status reef_kv_select_pages(
    const reef_decode_params *p, const int8_t *q, const float *q_scales, const int8_t *bounds,
    const float *bound_scales, const int32_t *block_table, int64_t max_blocks_per_seq,
    int64_t num_pages, const int32_t *context_lens, int64_t budget, int64_t sinks, int64_t recent,
    int32_t *pages, int32_t *counts, void *workspace, size_t workspace_bytes,
    uint32_t *status_word, hipStream_t stream) {
    if (!select_sizes(p) || !q || !q_scales || !bounds || !bound_scales || !context_lens ||
        !pages || !counts ||
        (p->q_granularity != REEF_SCALE_PER_TENSOR && p->q_granularity != REEF_SCALE_PER_HEAD &&
         p->q_granularity != REEF_SCALE_PER_TOKEN))
        return REEF_INVALID_ARGUMENT;
    if (sinks < 0 || recent < 1 || budget < 1 || sinks > budget || recent > budget - sinks)
        return REEF_INVALID_ARGUMENT;
    if ((p->head_dim != 64 && p->head_dim != 128) || p->q_heads / p->kv_heads > 16 ||
        p->batch > 65535 || p->kv_heads > 65535 || p->batch * p->kv_heads > 65535 ||
        p->max_context >= (int64_t(1) << 30) || budget >= (int64_t(1) << 26))
        return REEF_UNSUPPORTED;
    if (!aligned(q, 16) || !aligned(q_scales, 4) || !aligned(bounds, 16) ||
        !aligned(bound_scales, 4) || !aligned(context_lens, 4) || !aligned(pages, 4) ||
        !aligned(counts, 4))
        return REEF_INVALID_ARGUMENT;
    if (block_table && (num_pages <= 0 || num_pages >= (int64_t(1) << 31) ||
                        max_blocks_per_seq <= 0 || max_blocks_per_seq * kPage < p->max_context ||
                        max_blocks_per_seq >= (int64_t(1) << 30)))
        return REEF_INVALID_ARGUMENT;
    if (!workspace || !aligned(workspace, 16) ||
        workspace_bytes < reef_kv_select_pages_workspace_bytes(p))
        return REEF_INVALID_ARGUMENT;
    SelectArgs a;
    a.q = q;
    a.qs = q_scales;
    a.bounds = bounds;
    a.scales = bound_scales;
    a.table = block_table;
    a.lens = context_lens;
    a.keys = static_cast<uint32_t *>(workspace);
    a.pages = pages;
    a.counts = counts;
    a.status = status_word;
    a.q_heads = (int32_t)p->q_heads;
    a.kv_heads = (int32_t)p->kv_heads;
    a.group = (int32_t)(p->q_heads / p->kv_heads);
    a.items = (int32_t)(p->batch * p->kv_heads);
    a.max_context = (int32_t)p->max_context;
    a.max_pages = (int32_t)(p->max_context / kPage);
    a.max_blocks = (int32_t)(block_table ? max_blocks_per_seq : 0);
    a.num_pages = (int32_t)(block_table ? num_pages : 0);
    a.budget = (int32_t)budget;
    a.sinks = (int32_t)sinks;
    a.recent = (int32_t)recent;
    a.q_gran = p->q_granularity;
    const dim3 grid((unsigned)ceil_div(a.max_pages, kWave), (unsigned)a.items);
    if (p->head_dim == 128)
        hipLaunchKernelGGL(score_pages<128>, grid, dim3(kWave), 0, stream, a);
    else
        hipLaunchKernelGGL(score_pages<64>, grid, dim3(kWave), 0, stream, a);
    if (hipGetLastError() != hipSuccess) return REEF_HIP_ERROR;
    const auto pick = [&](auto *kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)a.items), dim3(kPickThreads), 0, stream, a);
    };
    pick(a.max_pages <= 2 * kPickThreads   ? pick_pages<2>
         : a.max_pages <= 8 * kPickThreads ? pick_pages<8>
                                           : pick_pages<0>);
    return launch_status();
}
