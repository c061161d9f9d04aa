// Attention of a tree of drafted tokens over an int8 KV cache for gfx950 (speculative
// decoding): T query tokens per sequence, whose keys and values the cache already holds in
// its last T places. Row i sees every token before them and, of the drafted ones, those whose
// bit its mask sets (its ancestors and itself).
//
//   s_j = float(int32 q_i . k_j) * (s_q * s_k[j]) * softmax_scale
//   out_i = sum_j softmax(s)_j * float(v_j) * s_v[j]
//
// The products are those of the decode kernel (decode.hip): 64-key blocks straight from
// memory into operand registers, S^T = K . q^T on v_mfma_i32_16x16x64_i8, out^T = V^T . P^T on
// v_mfma_f32_16x16x32_f16 with P split into fp16 hi + lo. The instruction's 16 columns hold
// (token, query head) pairs of one KV head, column t * group + g, so T tokens of a group of G
// heads are T G columns in tiles of 16. A wave keeps NC tiles: what it reads and converts of a
// block serves them all.
#include <algorithm>
#include <cmath>

#include "decode_common.hpp"

namespace reef {
namespace {

constexpr int kWaves = 4;      // waves of a workgroup, one per SIMD
constexpr int kWgPerCu = 2;    // workgroups of a compute unit
constexpr int kMinBlocks = 2;  // blocks of a wave in a run, at least, while items are whole
constexpr int kPlan = 2048;    // sequences of a launch (more are launched in slices)
constexpr int kMaxGroup = 1024;  // query heads of a kv head
constexpr int kCounters = 2048;

struct TreeArgs {
    const int8_t *q;
    const float *qs;
    const int8_t *k, *v;  // contiguous cache or page pool
    const float *ks, *vs;
    const int32_t *block_table;   // paged only
    const int32_t *context_lens;  // may be null
    const uint64_t *mask;         // [batch, drafts]; null: row i sees drafted tokens 0 .. i
    float *out;
    uint32_t *counters;  // one per workgroup; zero between launches
    uint64_t *slots;
    uint32_t *status;
    int64_t q_sb, q_sh, q_st, o_sb, o_sh, o_st;
    int32_t batch, q_heads, kv_heads, group, drafts;
    uint32_t group_inverse;  // floor(2^32 / group) + 1: i / group for i * group < 2^32
    int32_t max_context, window;
    int32_t chunks;  // column ranges of 16 NC columns; an item is (sequence, kv head, range)
    int32_t extra;   // units that an item counts beside its blocks
    int32_t max_blocks, num_pages;  // paged only
    int32_t q_gran;
    float score_scale;  // softmax_scale * log2(e)
};

// A sequence's keys: its length (0 if out of range), the tokens before the drafts, the first
// key any row sees, and its 64-key blocks from the one with that key on. A sequence with no
// keys counts one block, so that some workgroup stores its zeros.
struct SeqKeys {
    int len, prefix, lo, first_block, blocks;
    // (an int: the padding behind a bool became an array in LDS when segments were copied, at
    // places worked out from the dispatch packet, and reading that packet, which lies in host
    // memory, held up every launch by 4 us and more)
    int bad;
};

__device__ __forceinline__ SeqKeys seq_keys(const TreeArgs &a, int b) {
    SeqKeys r;
    int len = a.context_lens ? a.context_lens[b] : a.max_context;
    r.bad = len < a.drafts || len > a.max_context;
    if (r.bad) len = 0;
    r.len = len;
    r.prefix = max(0, len - a.drafts);
    r.lo = a.window > 0 ? max(0, r.prefix + 1 - a.window) : 0;  // (the shallowest row's)
    r.first_block = r.lo / kBlockKeys;
    r.blocks = len > 0 ? (len + kBlockKeys - 1) / kBlockKeys - r.first_block : 1;
    return r;
}

// sOff[i] = units of an item of each of sequences 0 .. i - 1, added, for i <= batch (a
// workgroup-wide scan).
__device__ void plan_blocks(const TreeArgs &a, int32_t *sOff, int32_t *sWave) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid == 0) sOff[0] = 0;
    int32_t run = 0;
    for (int base = 0; base < a.batch; base += 64 * kWaves) {
        const int i = base + tid;
        int32_t x = i < a.batch ? seq_keys(a, i).blocks + a.extra : 0;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int32_t y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        if (lane == 63) sWave[wave] = x;
        __syncthreads();
        int32_t before = run;
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) before += sWave[w];
            run += sWave[w];
        }
        if (i < a.batch) sOff[i + 1] = before + x;
        __syncthreads();
    }
}

// Where a 64-key block lies, in units of one kv head's 16-token page: the page of this lane's
// K row, and that of its lane group.
struct BlockAt {
    uint32_t k_slot, g_slot;
    bool live;  // the lane group's page holds keys of this sequence
};

template <bool PAGED>
__device__ __forceinline__ BlockAt block_at(const TreeArgs &a, int b, int kvh, int kb,
                                            const SeqKeys &sk, int pages, int col, int grp,
                                            bool &bad_page) {
    BlockAt r;
    const int kp = kb / kPage + (col >> 2), gp = kb / kPage + grp;
    // Pages past the sequence's last, or wholly before the first key that any row sees (they
    // may have been given back), are not read: their lanes read a safe page.
    const int n_pages = (sk.len + kPage - 1) / kPage, first = sk.lo / kPage;
    const bool k_in = kp >= first && kp < n_pages, g_in = gp >= first && gp < n_pages;
    if (PAGED) {
        const int ke = __shfl(pages, col >> 2), ge = __shfl(pages, grp);
        const bool k_ok = k_in && ke >= 0 && ke < a.num_pages;
        const bool g_ok = g_in && ge >= 0 && ge < a.num_pages;
        bad_page |= g_in && !g_ok;
        r.live = g_ok;
        r.k_slot = (uint32_t)((k_ok ? ke : 0) * a.kv_heads + kvh);
        r.g_slot = (uint32_t)((g_ok ? ge : 0) * a.kv_heads + kvh);
    } else {
        const uint32_t seq = (uint32_t)((b * a.kv_heads + kvh) * (a.max_context / kPage));
        r.live = g_in;
        r.k_slot = seq + (k_in ? kp : 0);
        r.g_slot = seq + (g_in ? gp : 0);
    }
    return r;
}

// Table entries of the block at key kb: lane l holds that of page l % 4.
template <bool PAGED>
__device__ __forceinline__ int block_pages(const TreeArgs &a, int b, int kb, const SeqKeys &sk,
                                           int lane) {
    const int p = kb / kPage + (lane & 3);
    if (!PAGED || p >= (sk.len + kPage - 1) / kPage || p < sk.lo / kPage) return 0;
    return a.block_table[(int64_t)b * a.max_blocks + p];
}

// Largest x over the 16 lanes of a row, in every lane of it.
template <int CTRL>
__device__ __forceinline__ float dpp_fmax(float x) {
    return fmaxf(x, __int_as_float(
                        __builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xF, 0xF, false)));
}
__device__ __forceinline__ float row_fmax(float x) {
    x = dpp_fmax<0xB1>(x);   // quad_perm [1, 0, 3, 2]
    x = dpp_fmax<0x4E>(x);   // quad_perm [2, 3, 0, 1]
    x = dpp_fmax<0x141>(x);  // row_half_mirror
    return dpp_fmax<0x140>(x);  // row_mirror
}
// max / sum of x over lanes l and l ^ 16 (v_permlane16_swap: no trip through LDS).
__device__ __forceinline__ float xor16_max(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor16_sum(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_or(uint32_t x) {
    return x | (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t row_or(uint32_t x) {
    x = dpp_or<0xB1>(x);
    x = dpp_or<0x4E>(x);
    x = dpp_or<0x141>(x);
    return dpp_or<0x140>(x);
}

// Bits lo .. hi - 1 of 16, for any lo and hi.
__device__ __forceinline__ uint32_t bits16(int lo, int hi) {
    lo = min(max(lo, 0), 16);
    hi = min(max(hi, 0), 16);
    return (0xffffu >> (16 - hi)) & ~((1u << lo) - 1u);
}

// A column of one tile: a row of the tree for one query head, or nothing.
struct Column {
    bool live;  // a column of this launch
    int head, token;
};

__device__ __forceinline__ Column column_of(const TreeArgs &a, int kvh, int index) {
    const bool live = index < a.drafts * a.group;
    const int i = live ? index : 0;
    const int token = a.group == 1 ? i : (int)__umulhi((uint32_t)i, a.group_inverse);
    return {live, kvh * a.group + i - token * a.group, token};
}

// Values accumulate in units of 2^-8 of a power of two (kLeastScale at least), so that the unit's
// inverse is exact and one subtraction.

// The power of two at or above x > 0 (2^127 for all above it).
__device__ __forceinline__ float power_above(float x) {
    return fminf(__uint_as_float((__float_as_uint(x) + 0x7fffffu) & 0x7f800000u), 0x1p127f);
}
__device__ __forceinline__ float inverse_unit(float power) {  // 2^8 / power
    return __uint_as_float((262u << 23) - __float_as_uint(power));
}

// Largest |x| of a row's 16 lanes among those that bit r of `bits` names for lane r.
template <int R = 0>
__device__ __forceinline__ float row_top(float x, uint32_t bits, float top = 0.0f) {
    if constexpr (R % 4 == 0) asm("" : "+v"(x), "+v"(top), "+v"(bits));
    const float v = __int_as_float(
        __builtin_amdgcn_mov_dpp(__float_as_int(x), 0x150 + R, 0xf, 0xf, true));
    top = bits >> R & 1u ? fmaxf(top, __builtin_fabsf(v)) : top;
    if constexpr (R < 15) return row_top<R + 1>(x, bits, top);
    return top;
}

// What the column's row sees: the first token before the drafts, and the drafted ones.
struct Sight {
    int lo;
    uint64_t drafts;
};

// The drafted tokens that a row sees, of its mask word (without masks: the chain).
__device__ __forceinline__ uint64_t seen_drafts(const TreeArgs &a, int token, uint64_t word) {
    const uint64_t all = a.drafts == 64 ? ~0ull : (1ull << a.drafts) - 1;
    return a.mask ? word & all : (2ull << token) - 1;
}

__device__ __forceinline__ Sight sight_of(const TreeArgs &a, int b, const SeqKeys &sk, uint64_t m) {
    Sight r = {0, m};
    if (a.window > 0) {
        // Row i sits at prefix + |mask_i| - 1 (its ancestors before it); a drafted token as
        // far back as the window is hidden.
        const int depth = (int)__popcll(m) - 1;
        r.lo = max(0, sk.prefix + depth + 1 - a.window);
        if (a.window < a.drafts) {
            for (int j = 0; j < a.drafts; ++j) {
                const uint64_t word = a.mask ? a.mask[(int64_t)b * a.drafts + j] : 0;
                const int dj = (int)__popcll(seen_drafts(a, j, word)) - 1;
                if (dj <= depth - a.window) r.drafts &= ~(1ull << j);
            }
        }
    }
    if (m == 0 || sk.len == 0) r = {INT32_MAX, 0};  // padding, or no keys
    return r;
}

// One part of one tile in the workspace: the output in [d][half][lane] order, then (max, sum).
template <int D>
struct TreeSlot {
    static constexpr int O = 2 * (D / 16);
    static constexpr int ELEMS = (O + 1) * kWave;
};

__device__ __forceinline__ uint64_t pack(float x, float y) {
    return (uint64_t)__float_as_uint(x) | ((uint64_t)__float_as_uint(y) << 32);
}
__device__ __forceinline__ float lo32(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi32(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }

// A workgroup's part of one item (sequence, kv head, column range): its blocks [s_blk, e_blk).
struct Segment {
    SeqKeys sk;
    int b, kvh, chunk, s_blk, e_blk;
    int first_u;  // the item's first block in the launch's numbering
    int units;    // of the run, the item's extra ones included
};

// An offset added where it is used: as part of a base address that outlives the key loop it took
// registers that then spilled, and the reload held up every segment's first block (16 x U[512,
// 8192] keys, 16 drafted: 57 us against 59).
__device__ __forceinline__ int held(int offset) {
    asm volatile("" : "+v"(offset));
    return offset;
}

// Waits for this wave's LDS accesses, then for the workgroup; loads in flight stay so
// (__syncthreads() would wait for them).
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The kernel's argument, read again: each phase of a segment loads what it needs (from the
// scalar cache) instead of holding every pointer and stride through the key loop, which
// spilled a hundred scalar registers into vector lanes.
__device__ __forceinline__ TreeArgs reread_args() {
    auto p = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const TreeArgs *)p;
}

// The launch's work is the 64-key blocks of all items, dealt out to the workgroups in equal
// runs. An item counts some units before its blocks, for the time that its rows, its merge
// and its stores take: workgroups with many short items get fewer blocks. Within a run each
// item's part is one segment: the workgroup's four waves take the segment's blocks in turn,
// keep a running softmax each and merge in LDS. An item inside one run is stored directly; the
// parts of an item cut by a run's end go to the workspace, and the one that counts in last
// merges them in order (reef_common.hpp, cross-workgroup parts).
//
// Bound by memory with few columns (64 x 4096 keys x 8 heads of 128, 3 drafted, 12 columns:
// 558 MB in 90 us, 6.2 TB/s), by the softmax's vector work and the items' fixed costs with many
// (32 sequences of one head, 64 drafted, 512 columns: 71 M scores in 74 to 88 us by the lengths).
template <int D, bool PAGED, int NC>
__global__ __launch_bounds__(64 * kWaves, kWgPerCu) void tree_kernel(TreeArgs arg) {
    constexpr int DB = D / 16, KS = D / 64;
    // One tile of columns has one reader of the cache: kept out of the caches (64 x 4096 keys, 3
    // drafted: 90 us against 98).
    constexpr bool NT = !PAGED && NC == 1;
    __shared__ int32_t sOff[kPlan + 1];
    __shared__ int32_t sWave[kWaves];
    __shared__ f32x4 sO[kWaves][DB][kWave];
    __shared__ float2 sML[kWaves][kWave];
    __shared__ i32x4 sQ[kWaves][NC * KS][kWave];  // query operands, each wave its own
    __shared__ Sight sSight[kWaves][NC][16];
    __shared__ uint32_t sLast;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;

    const bool same = arg.context_lens == nullptr;
    const int nb = same ? seq_keys(arg, 0).blocks + arg.extra : 0;
    if (!same) plan_blocks(arg, sOff, sWave);
    auto units_before = [&](int b) -> int {  // of an item of each sequence before b
        return same ? b * nb : __builtin_amdgcn_readfirstlane(sOff[b]);
    };
    const int per_seq = arg.kv_heads * arg.chunks;  // items of a sequence
    const int T = units_before(arg.batch) * per_seq;  // (fits: checked for full caches)
    // No more workgroups than there are items, or parts with kMinBlocks for every wave: more
    // parts are a longer merge, fewer a longer run (with at least 1, 2 and 3 blocks a wave:
    // 1 x 8192 keys, 8/1 heads of 128, 16 drafted 23.4, 21.7, 22.4 us; 1 x 8192, 8/8 heads, 1
    // drafted 22.2, 19.2, 19.4; 3 x 1000-3000, 8/1 heads, 64 drafted 22.5, 20.8, 22.9).
    const int items = arg.batch * per_seq;
    const int G = min((int)gridDim.x, max(items, (T - items * arg.extra + kMinBlocks * kWaves - 1) /
                                                     (kMinBlocks * kWaves)));
    // Workgroup w's run: T / G units, one more for each of the first T % G.
    const int quota = T / G, longer = T - quota * G;
    auto run_start = [&](int w) { return w * quota + min(w, longer); };
    auto run_of = [&](int u) {
        const int mid = longer * (quota + 1);
        return u < mid ? u / (quota + 1) : longer + (u - mid) / quota;
    };
    // With several tiles the workgroups of one XCD hold consecutive runs: the column ranges of
    // one (sequence, kv head) meet in its L2 (32 sequences of one head, 64 drafted 90 us against
    // 99). With one tile nothing is shared, and plain order is faster (64 x 4096 x 8 heads of
    // 128, 3 drafted: 90 us against 100).
    int g = blockIdx.x;
    if (NC == 1) {
        if (g >= G) return;
    } else {
        const int x = blockIdx.x % kXcds, place = blockIdx.x / kXcds;
        const int per = G / kXcds, rem = G % kXcds;
        if (place >= per + (x < rem ? 1 : 0)) return;
        g = x * per + min(x, rem) + place;
    }
    const int u0 = run_start(g), u1 = run_start(g + 1);

    auto segment_at = [&](const TreeArgs &a, int u, int b) {
        Segment s;
        s.b = b;
        s.sk = seq_keys(a, b);
        s.sk.len = __builtin_amdgcn_readfirstlane(s.sk.len);
        s.sk.prefix = __builtin_amdgcn_readfirstlane(s.sk.prefix);
        s.sk.lo = __builtin_amdgcn_readfirstlane(s.sk.lo);
        s.sk.first_block = __builtin_amdgcn_readfirstlane(s.sk.first_block);
        s.sk.blocks = __builtin_amdgcn_readfirstlane(s.sk.blocks);
        const int in_seq = u - units_before(b) * per_seq;
        const int per_item = s.sk.blocks + a.extra, hc = in_seq / per_item;
        const int at = in_seq - hc * per_item, end = min(per_item, at + (u1 - u));
        s.s_blk = max(0, at - a.extra);
        s.e_blk = max(0, end - a.extra);  // (none where the run ends before the item's blocks)
        s.units = end - at;
        s.kvh = hc / a.chunks;
        s.chunk = hc - s.kvh * a.chunks;
        s.first_u = u - at + a.extra;
        return s;
    };
    auto first_key = [&](const Segment &s) {
        return (s.sk.first_block + s.s_blk + wave) * kBlockKeys;
    };
    auto end_key = [&](const Segment &s) {
        return min(s.sk.len, (s.sk.first_block + s.e_blk) * kBlockKeys);
    };
    auto first_tile = [&](const Segment &s) { return s.chunk * NC; };
    auto column = [&](const TreeArgs &a, const Segment &s, int t) {
        return column_of(a, s.kvh, 16 * (first_tile(s) + t) + col);
    };
    constexpr int k_step = kWaves * kBlockKeys;

    // A block's operands, and what a segment's rows need, in registers.
    i32x4 kop[4][KS], vop[DB];
    float ks = 0.0f, vs = 0.0f, cs[NC];
    uint32_t shown = 0;  // bit t: this lane's row of tile t sees something
    BlockAt at;
    bool bad_page = false;
    int pg_next;
    auto load_k = [&](const TreeArgs &a) {
        const int in_page = held((col & 3) * D + 16 * grp);
        const int8_t *p = a.k + (int64_t)at.k_slot * (kPage * D) + in_page;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int s = 0; s < KS; ++s)
                kop[t][s] = load_stream<NT>(reinterpret_cast<const i32x4 *>(p + 4 * t * D + 64 * s));
        ks = a.ks[(int64_t)at.g_slot * kPage + col];
    };
    auto load_v = [&](const TreeArgs &a) {
        const int8_t *p = a.v + (int64_t)at.g_slot * (kPage * D) + col * kPage;
#pragma unroll
        for (int d = 0; d < DB; ++d)
            vop[d] = load_stream<NT>(reinterpret_cast<const i32x4 *>(p + 16 * d * kPage));
        vs = a.vs[(int64_t)at.g_slot * kPage + col];
    };
    // Whether this wave has anything to do in a segment.
    auto busy = [&](const Segment &s) { return first_key(s) < end_key(s); };
    // A segment's rows on their way to LDS (each wave its own places). All their loads leave
    // together, from addresses without a branch: one round trip. (Kept in registers across the
    // segment before, they were spilled as they came, one round trip after another: 16 x U[512,
    // 8192] keys, 16 drafted 76 us, 71 this way.)
    struct Rows {
        i32x4 q[NC][KS];
        float c[NC];
        uint64_t m[NC];
    };
    auto load_rows = [&](const TreeArgs &a, const Segment &s) {
        Rows r;
        const uint64_t *masks = a.mask ? a.mask : reinterpret_cast<const uint64_t *>(a.q);
#pragma unroll
        for (int t = 0; t < NC; ++t) {
            const Column cn = column(a, s, t);
            r.m[t] = masks[a.mask ? (int64_t)s.b * a.drafts + cn.token : 0];
            const int64_t row = ((int64_t)s.b * a.q_heads + cn.head) * a.drafts + cn.token;
            r.c[t] = a.qs[a.q_gran == REEF_SCALE_PER_TOKEN ? row
                          : a.q_gran == REEF_SCALE_PER_HEAD ? cn.head
                                                            : 0];
            const int8_t *qrow = a.q + s.b * a.q_sb + cn.head * a.q_sh + cn.token * a.q_st;
#pragma unroll
            for (int e = 0; e < KS; ++e)
                r.q[t][e] = *reinterpret_cast<const i32x4 *>(qrow + 64 * e + 16 * grp);
        }
        return r;
    };
    auto put_rows = [&](const TreeArgs &a, const Segment &s, const Rows &r) {
        shown = 0;
#pragma unroll
        for (int t = 0; t < NC; ++t) {
            const Column cn = column(a, s, t);
            const uint64_t m = cn.live ? seen_drafts(a, cn.token, r.m[t]) : 0;
            // (a factor of 0 would make a hidden key's -inf a NaN: scores of 0 times 1 instead)
            const float c = r.c[t] * a.score_scale;
            const bool scaled = cn.live && c != 0.0f;
#pragma unroll
            for (int e = 0; e < KS; ++e)
                sQ[wave][t * KS + e][lane] = scaled ? r.q[t][e] : i32x4{0, 0, 0, 0};
            cs[t] = scaled ? c : 1.0f;
            shown |= (m != 0 ? 1u : 0u) << t;
            const Sight sight = sight_of(a, s.b, s.sk, m);
            if (grp == 0) sSight[wave][t][col] = sight;
        }
    };
    // The loads of a segment's first block (pages: its table entries).
    auto issue = [&](const TreeArgs &a, const Segment &s, int pages) {
        at = block_at<PAGED>(a, s.b, s.kvh, first_key(s), s.sk, pages, col, grp, bad_page);
        load_k(a);
        load_v(a);
    };

    // The run's first sequence: the last one that begins at or before u0, among 64 evenly
    // spaced ones, then among the kPlan / 64 of its stretch.
    int b = 0;
    if (same) {
        b = u0 / (nb * per_seq);
    } else {
        constexpr int kStretch = kPlan / 64;
        static_assert(kStretch <= 64, "two steps of a wave");
        const int far = lane * kStretch;
        b = kStretch * (__popcll(__ballot(far < arg.batch && sOff[far] * per_seq <= u0)) - 1);
        const int near = b + lane;
        b += __popcll(__ballot(lane < kStretch && near < arg.batch && sOff[near] * per_seq <= u0)) - 1;
        b = __builtin_amdgcn_readfirstlane(b);
    }
    Segment seg = segment_at(arg, u0, b);
    if (seg.e_blk <= seg.s_blk) return;  // (uniform)
    pg_next = block_pages<PAGED>(arg, b, first_key(seg) + k_step, seg.sk, lane);
    {
        const int pages = block_pages<PAGED>(arg, b, first_key(seg), seg.sk, lane);
        if (busy(seg)) {
            const Rows rows = load_rows(arg, seg);
            issue(arg, seg, pages);
            put_rows(arg, seg, rows);
        }
    }
    for (int u = u0;;) {
        TreeArgs a = reread_args();
        if (seg.sk.bad && seg.s_blk == 0 && seg.kvh == 0 && seg.chunk == 0 && threadIdx.x == 0)
            flag_status(a.status, REEF_STATUS_BIT_BAD_LENGTH);
        const bool mine = busy(seg);  // wave-uniform
        // The next segment, and the table entries of its first two blocks.
        u += seg.units;
        bool more_segs = u < u1;
        Segment nxt = seg;
        int pg_first = 0, pg_second = 0;
        if (more_segs) {
            const bool same_seq = u < units_before(seg.b + 1) * per_seq;
            nxt = segment_at(a, u, same_seq ? seg.b : seg.b + 1);
            more_segs = nxt.e_blk > nxt.s_blk;
            pg_first = block_pages<PAGED>(a, nxt.b, first_key(nxt), nxt.sk, lane);
            pg_second = block_pages<PAGED>(a, nxt.b, first_key(nxt) + k_step, nxt.sk, lane);
        }

        float m_run[NC], l_run[NC], s_run[NC], s_least = kLeastScale;
        f32x4 acc[NC][DB];
#pragma unroll
        for (int t = 0; t < NC; ++t) {
            m_run[t] = -INFINITY;
            l_run[t] = 0.0f;
            s_run[t] = kLeastScale;
#pragma unroll
            for (int d = 0; d < DB; ++d) acc[t][d] = f32x4{};
        }
        const int k_end = end_key(seg);
        // Keys that every row sees: [full_lo, prefix).
        const int full_lo = a.window > 0 ? max(0, seg.sk.prefix + a.drafts - a.window) : 0;
        if (mine) {
            for (int kb = first_key(seg); kb < k_end; kb += k_step) {
                const bool more = kb + k_step < k_end;
                const bool live = at.live;
                const float ks_now = ks;
                const int pg_after = block_pages<PAGED>(a, seg.b, kb + 2 * k_step, seg.sk, lane);
                // Scores of every tile, times the key's scale.
                float xs[NC][16];
                {
                    float ksc[16];
                    row_lanes(ks, ksc);
#pragma unroll
                    for (int t = 0; t < NC; ++t) {
                        i32x4 qop[KS];
#pragma unroll
                        for (int e = 0; e < KS; ++e) qop[e] = sQ[wave][t * KS + e][lane];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            i32x4 s = {0, 0, 0, 0};
#pragma unroll
                            for (int e = 0; e < KS; ++e) s = mfma_16x16x64_i8(kop[j][e], qop[e], s);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                xs[t][4 * j + i] = (float)s[i] * ksc[4 * j + i];
                        }
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                // The key registers are free: the next block's keys fly from here on (after a
                // segment's last block the next segment's first), its values as the products
                // below free theirs. With nothing to follow, this block's are read again.
                if (more || more_segs) {
                    at = block_at<PAGED>(a, more ? seg.b : nxt.b, more ? seg.kvh : nxt.kvh,
                                         more ? kb + k_step : first_key(nxt), more ? seg.sk : nxt.sk,
                                         more ? pg_next : pg_first, col, grp, bad_page);
                }
                load_k(a);
                const int8_t *v_next =
                    a.v + (int64_t)at.g_slot * (kPage * D) + held(col * kPage);
                __builtin_amdgcn_sched_barrier(0);
                pg_next = pg_after;
                // Blocks that every row sees whole skip the masks. In the others a hidden key's
                // score is -inf, and the value scale of a key that no row of the wave sees
                // is 0 (the cache there may hold anything). A token whose key or value scale is
                // not finite makes the rows that see it NaN through their scores (an infinite key
                // scale alone would be a weight of 0 where the product is negative), and no
                // others: its value scale is 0 too.
                const int kk = kb + 16 * grp;
                float vsc = vs;
                uint32_t seen = ~0u;  // 16 bits a tile: which of its 16 keys this lane's row sees
                static_assert(NC <= 2, "tiles in one word");
                const bool whole =
                    kb >= full_lo && kb + kBlockKeys <= seg.sk.prefix && __all(live);
                if (!whole) {
                    uint32_t any = seen = 0;
                    const bool finite =
                        __builtin_fabsf(vsc) < INFINITY && __builtin_fabsf(ks_now) < INFINITY;
                    const uint32_t nan = row_or(finite ? 0u : 1u << col);
#pragma unroll
                    for (int t = 0; t < NC; ++t) {
                        const Sight sight = sSight[wave][t][col];
                        uint32_t vis = bits16(sight.lo - kk, seg.sk.prefix - kk);
                        const int j = kk - seg.sk.prefix;  // drafted token of the group's first key
                        vis |= (j >= 0 ? (j < 64 ? (uint32_t)(sight.drafts >> j) : 0u)
                                       : (j > -16 ? (uint32_t)(sight.drafts << -j) : 0u)) & 0xffffu;
                        if (!live) vis = 0;
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (!(vis >> r & 1u)) xs[t][r] = -INFINITY;
                        if (vis & nan) {
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                if (vis & nan & 1u << r) xs[t][r] = __builtin_nanf("");
                        }
                        any |= vis;
                        seen |= vis << (16 * t);
                    }
                    any = row_or(any);
                    if (!finite || !(any >> col & 1u)) vsc = 0.0f;
                }
                float mt[NC];  // over this lane's keys
                bool grow = __builtin_fabsf(vsc) > s_least * 2.0f;
#pragma unroll
                for (int t = 0; t < NC; ++t) {
                    float m = fmaxf(fmaxf(xs[t][0], xs[t][1]), xs[t][2]);
#pragma unroll
                    for (int r = 3; r < 15; r += 2) m = fmaxf(fmaxf(m, xs[t][r]), xs[t][r + 1]);
                    m = fmaxf(m, xs[t][15]);
                    mt[t] = m * cs[t];
                    grow |= mt[t] > m_run[t] + 6.0f;
                }
                // Lazy rescale: a row's maximum moves only when it grows by more than 2^6, and
                // the unit of its accumulator (s_run / 2^8, s_run a power of two at or above the
                // largest value scale that the row has seen) only when a value scale passes s_run
                // 2-fold, so a weight p * v_scale * 2^8 / s_run stays below 2^15 in fp16, and is
                // off by at most half a subnormal step, 2^-33 of s_run (hi and lo keep 11 bits
                // each). Each row by what it sees itself: a drafted token of large values does not
                // push the weights of the rows that do not see it into the subnormals. Whether any
                // row may have to move is asked of each lane's keys and of s_least, the least
                // s_run; the rows' own maxima are taken only then.
                if (__any(grow)) {
                    float least = INFINITY;
#pragma unroll
                    for (int t = 0; t < NC; ++t) {
                        const float ct = whole ? row_fmax(__builtin_fabsf(vsc))
                                               : row_top(vsc, seen >> (16 * t));
                        const float s_new = power_above(fmaxf(s_run[t], xor32_max(xor16_max(ct))));
                        const float units = s_run[t] / s_new;
                        s_run[t] = s_new;
                        least = fminf(least, s_new);
                        const float m_new = fmaxf(m_run[t], xor32_max(xor16_max(mt[t])));
                        const float alpha =
                            m_run[t] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[t] - m_new);
                        m_run[t] = m_new;
                        l_run[t] *= alpha;
                        const float alpha_o = alpha * units;
#pragma unroll
                        for (int d = 0; d < DB; ++d) acc[t][d] *= alpha_o;
                    }
                    s_least = __int_as_float(
                        __builtin_amdgcn_readfirstlane(__float_as_int(-row_fmax(-least))));
                }
                // P operands: lane group g's keys 16 g + 8 h + e for the two halves h.
                f16x8 hi[NC][2], lo[NC][2];
                {
                    float vv[16];
                    row_lanes(vsc, vv);
#pragma unroll
                    for (int t = 0; t < NC; ++t) {
                        const float m_use = m_run[t] == -INFINITY ? 0.0f : m_run[t];
                        const float inv_s = inverse_unit(s_run[t]);
                        float sum[2] = {0.0f, 0.0f};
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float w[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const float p = __builtin_amdgcn_exp2f(
                                    __builtin_fmaf(xs[t][8 * h + e], cs[t], -m_use));
                                sum[e & 1] += p;
                                // (p first: what the row does not see has p = 0)
                                w[e] = p * inv_s * vv[8 * h + e];
                            }
                            split_weights(w, hi[t][h], lo[t][h]);
                        }
                        l_run[t] += sum[0] + sum[1];
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                if (NC > 1) __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int d = 0; d < DB; d += 2) {
                    f16x8 v[2][2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        int8x16_to_f16(vop[d + i], v[i][0], v[i][1]);
                        vop[d + i] = load_stream<NT>(
                            reinterpret_cast<const i32x4 *>(v_next + 16 * (d + i) * kPage));
                    }
                    // Products of one accumulator are NC * 2 apart.
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int t = 0; t < NC; ++t)
                                acc[t][d + i] = mfma_16x16x32_f16(v[i][h], hi[t][h], acc[t][d + i]);
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int t = 0; t < NC; ++t)
                                acc[t][d + i] = mfma_16x16x32_f16(v[i][h], lo[t][h], acc[t][d + i]);
                    }
                }
                if (NC > 1) __builtin_amdgcn_s_setprio(0);
                vs = a.vs[(int64_t)at.g_slot * kPage + col];
            }
        }
        a = reread_args();
        if (bad_page) flag_status(a.status, REEF_STATUS_BIT_BAD_PAGE);
        bad_page = false;
        // The next segment's first block flies while this one is merged (a wave that had none of
        // this segment asks for it now).
        if (more_segs) {
            if (!mine && busy(nxt)) issue(a, nxt, pg_first);
            pg_next = pg_second;
        }
        a = reread_args();

        // The workgroups that hold a part of this item: gf .. gl, each with at least one block.
        const int gf = run_of(seg.first_u);
        const int parts = run_of(seg.first_u + seg.sk.blocks - 1) - gf + 1;
        constexpr int64_t slot_elems = NC * TreeSlot<D>::ELEMS;
        // A workgroup has two slots: for an item that begins in its run, and one that began
        // before.
        uint64_t *own = a.slots + (2 * (int64_t)g + (g == gf ? 1 : 0)) * slot_elems;
        auto tile_slot = [&](uint64_t *s, int t) { return s + t * TreeSlot<D>::ELEMS; };
        auto store_out = [&](const Column &cn, int d, f32x4 o, float l) {
            if (!cn.live) return;
            float *row = a.out + seg.b * a.o_sb + cn.head * a.o_sh + cn.token * a.o_st;
            f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
            if (l != 0.0f) y = o * (1.0f / l);  // (NaN where the row's sum is)
            *reinterpret_cast<f32x4 *>(row + 16 * d + 4 * grp) = y;
        };
        // The waves merge tile by tile through LDS, each the channel blocks d = wave, wave + 4,
        // ... A row that sees nothing has the sum 0.
#pragma unroll
        for (int t = 0; t < NC; ++t) {
            const Column cn = column(a, seg, t);
            float l = xor32_sum(xor16_sum(l_run[t]));
            if (!(shown >> t & 1u)) {
                l = 0.0f;
                m_run[t] = -INFINITY;
            }
#pragma unroll
            for (int d = 0; d < DB; ++d)
                sO[wave][d][lane] = acc[t][d] * (s_run[t] * (1.0f / 256.0f));
            sML[wave][lane] = float2{m_run[t], l};
            lds_barrier();
            float2 ml[kWaves];
            float m = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                ml[w] = sML[w][lane];
                m = fmaxf(m, ml[w].x);
            }
            l = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                ml[w].x = ml[w].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[w].x - m);
                l = __builtin_fmaf(ml[w].x, ml[w].y, l);
            }
#pragma unroll
            for (int n = 0; n < DB / kWaves; ++n) {
                const int d = wave + n * kWaves;
                f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    const f32x4 p = sO[w][d][lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(ml[w].x, p[e], o[e]);
                }
                if (parts == 1) {
                    store_out(cn, d, o, l);
                } else if (cn.live) {
                    uint64_t *s = tile_slot(own, t);
                    part_store(s + (2 * d) * kWave + lane, pack(o[0], o[1]));
                    part_store(s + (2 * d + 1) * kWave + lane, pack(o[2], o[3]));
                }
            }
            if (parts > 1 && wave == 0 && cn.live)
                part_store(tile_slot(own, t) + TreeSlot<D>::O * kWave + lane, pack(m, l));
            lds_barrier();  // frees sO / sML
        }
        if (parts > 1) {
            part_stores_done();
            __syncthreads();
            if (threadIdx.x == 0)
                sLast = part_count(a.counters + gf) == (uint32_t)(parts - 1) ? 1u : 0u;
            __syncthreads();
            if (__builtin_amdgcn_readfirstlane(sLast)) {
                part_claimed();
                if (threadIdx.x == 0) part_reset(a.counters + gf);
                // A chain of round trips beneath the caches: kAhead parts' loads in flight at a
                // time, all of a wave's channel blocks of a tile.
                constexpr int kAhead = 4, ND = DB / kWaves;
#pragma unroll
                for (int t = 0; t < NC; ++t) {
                    const Column cn = column(a, seg, t);
                    if (!cn.live) continue;
                    float m = -INFINITY, l = 0.0f;
                    f32x4 o[ND];
#pragma unroll
                    for (int n = 0; n < ND; ++n) o[n] = f32x4{};
                    for (int p0 = 0; p0 < parts; p0 += kAhead) {
                        uint64_t ml[kAhead], v[kAhead][ND][2];
#pragma unroll
                        for (int i = 0; i < kAhead; ++i) {
                            const int p = min(p0 + i, parts - 1);
                            const uint64_t *s = tile_slot(
                                a.slots + (2 * (int64_t)(gf + p) + (p == 0 ? 1 : 0)) * slot_elems, t) + lane;
                            ml[i] = part_load(s + TreeSlot<D>::O * kWave);
#pragma unroll
                            for (int n = 0; n < ND; ++n)
#pragma unroll
                                for (int h = 0; h < 2; ++h)
                                    v[i][n][h] = part_load(s + (2 * (wave + n * kWaves) + h) * kWave);
                        }
#pragma unroll
                        for (int i = 0; i < kAhead; ++i) {
                            if (p0 + i >= parts) break;
                            const float mp = lo32(ml[i]), mn = fmaxf(m, mp);
                            const float er = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
                            const float ep = mp == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mp - mn);
                            l = __builtin_fmaf(ep, hi32(ml[i]), l * er);
#pragma unroll
                            for (int n = 0; n < ND; ++n)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    o[n][2 * h] = __builtin_fmaf(ep, lo32(v[i][n][h]), o[n][2 * h] * er);
                                    o[n][2 * h + 1] =
                                        __builtin_fmaf(ep, hi32(v[i][n][h]), o[n][2 * h + 1] * er);
                                }
                            m = mn;
                        }
                    }
#pragma unroll
                    for (int n = 0; n < ND; ++n) store_out(cn, wave + n * kWaves, o[n], l);
                }
            }
            __syncthreads();  // sLast is read before the next segment writes it
        }
        if (!more_segs) break;
        seg = nxt;
        if (busy(seg)) {
            a = reread_args();
            put_rows(a, seg, load_rows(a, seg));
        }
    }
}

// ---- host ------------------------------------------------------------------------------

// How a launch of `batch` sequences is laid out: tiles per wave, the column ranges, the
// workgroups, and the units that an item counts beside its blocks.
struct TreeShape {
    int64_t nc, chunks, wgs, extra;
};

TreeShape tree_shape(const reef_tree_params *p, int64_t batch) {
    TreeShape s;
    const int64_t cus = compute_units();
    const int64_t tiles = ceil_div(p->draft_len * (p->q_heads / p->kv_heads), 16);
    s.nc = tiles > 1 ? 2 : 1;
    // More columns become further items that read the same keys, from L2 mostly: split over
    // the waves of a workgroup instead, the keys were cut into more parts (an earlier form: 32 x
    // 8/1 heads, 64 drafted, 512 columns 102 us in ranges of 32, 103 of 64, 109 of 128; 1 x 8192
    // keys, 128 columns 27 in ranges of 32, 35 of 64).
    s.chunks = ceil_div(tiles, s.nc);
    // (with 2, 3 and 5 a wave for two tiles: 16 x U[512, 8192] keys, 8/32 heads, 16 drafted
    // 62.7, 63.6, 65 us, 3 x 1000-3000 keys, 64 drafted 20.3, 19.6, 20.9; with 1 and 2 for
    // one tile: 1 x 8192 keys, 8/8 heads, 1 drafted 20.3, 19.2)
    s.extra = (s.nc == 2 ? 3 : 2) * kWaves;
    const int64_t units =
        batch * p->kv_heads * s.chunks * ceil_div(p->max_context, kBlockKeys);
    s.wgs = std::max<int64_t>(1, std::min(std::min(kWgPerCu * cus, units), (int64_t)kCounters));
    return s;
}

constexpr int64_t kCounterBytes = kCounters * 4;

int64_t tree_workspace(const reef_tree_params *p) {
    const int64_t elems = p->head_dim == 128 ? TreeSlot<128>::ELEMS : TreeSlot<64>::ELEMS;
    // the slices of a large batch: full ones and the last
    int64_t most = 0;
    for (const int64_t batch : {std::min<int64_t>(p->batch, kPlan), p->batch % kPlan}) {
        if (batch == 0) continue;
        const TreeShape s = tree_shape(p, batch);
        most = std::max(most, s.wgs * 2 * s.nc * elems * 8);
    }
    return kCounterBytes + most;
}

bool params_ok(const reef_tree_params *p) {
    return p && p->batch > 0 && p->q_heads > 0 && p->kv_heads > 0 && p->head_dim > 0 &&
           p->draft_len > 0 && p->max_context > 0 && p->q_heads % p->kv_heads == 0;
}

bool params_supported(const reef_tree_params *p) {
    return (p->head_dim == 64 || p->head_dim == 128) && p->draft_len <= kMaxDrafts &&
           p->q_heads <= 65535 && p->q_heads / p->kv_heads <= kMaxGroup && p->batch <= 65535 &&
           p->max_context < (int64_t(1) << 30);
}

bool strides_ok(const reef_strides *s, int64_t unit) {
    return !s || (s->batch >= 0 && s->head >= 0 && s->token >= 0 && s->batch % unit == 0 &&
                  s->head % unit == 0 && s->token % unit == 0);
}

reef_status validate(const reef_tree_params *p, const int8_t *q, const reef_strides *q_strides,
                     const float *q_scales, const int8_t *k, const int8_t *v, const float *ks,
                     const float *vs, const uint64_t *mask, const float *out,
                     const reef_strides *out_strides, const void *workspace,
                     size_t workspace_bytes) {
    if (!params_ok(p) || !q || !q_scales || !k || !v || !ks || !vs || !out ||
        p->max_context % kPage != 0 || p->window < 0 || !std::isfinite(p->softmax_scale) ||
        !(p->softmax_scale > 0.0f) || p->flags != 0 ||
        (p->q_granularity != REEF_SCALE_PER_TENSOR && p->q_granularity != REEF_SCALE_PER_HEAD &&
         p->q_granularity != REEF_SCALE_PER_TOKEN))
        return REEF_INVALID_ARGUMENT;
    if (!params_supported(p)) return REEF_UNSUPPORTED;
    if (p->draft_len > p->max_context) return REEF_CAPACITY;
    if (!aligned(q, 16) || !strides_ok(q_strides, 16) || !aligned(out, 16) ||
        !strides_ok(out_strides, 4) || !aligned(k, 16) || !aligned(v, 16) || !aligned(ks, 4) ||
        !aligned(vs, 4) || !aligned(mask, 8))
        return REEF_INVALID_ARGUMENT;
    if (!workspace || !aligned(workspace, 16) ||
        workspace_bytes < (size_t)tree_workspace(p))
        return REEF_INVALID_ARGUMENT;
    // pages of one kv head are numbered in 31 bits (of 2 KB each, keys and values)
    if (p->batch * p->kv_heads * (p->max_context / kPage) >= (int64_t(1) << 31))
        return REEF_UNSUPPORTED;
    const TreeShape s = tree_shape(p, std::min<int64_t>(p->batch, kPlan));
    if (std::min<int64_t>(p->batch, kPlan) * p->kv_heads * s.chunks *
            (ceil_div(p->max_context, kBlockKeys) + s.extra) >= (int64_t(1) << 31))
        return REEF_UNSUPPORTED;
    return REEF_OK;
}

template <bool PAGED>
reef_status launch_tree(const reef_tree_params *p, TreeArgs &a, const reef_strides *qs,
                        const reef_strides *os, void *workspace, hipStream_t stream) {
    const int64_t D = p->head_dim, T = p->draft_len, Hq = p->q_heads;
    a.q_sb = qs ? qs->batch : Hq * T * D;
    a.q_sh = qs ? qs->head : T * D;
    a.q_st = qs ? qs->token : D;
    a.o_sb = os ? os->batch : Hq * T * D;
    a.o_sh = os ? os->head : T * D;
    a.o_st = os ? os->token : D;
    a.q_heads = (int32_t)Hq;
    a.kv_heads = (int32_t)p->kv_heads;
    a.group = (int32_t)(Hq / p->kv_heads);
    a.group_inverse = (uint32_t)((uint64_t(1) << 32) / (uint64_t)a.group + 1);
    a.drafts = (int32_t)T;
    a.max_context = (int32_t)p->max_context;
    a.window = (int32_t)std::min<int64_t>(p->window, int64_t(1) << 30);
    a.q_gran = p->q_granularity;
    a.score_scale = p->softmax_scale * kLog2e;
    a.counters = static_cast<uint32_t *>(workspace);
    a.slots = reinterpret_cast<uint64_t *>(static_cast<char *>(workspace) + kCounterBytes);
    for (int64_t b0 = 0; b0 < p->batch; b0 += kPlan) {  // (the slices follow one another)
        const int64_t batch = std::min<int64_t>(kPlan, p->batch - b0);
        const TreeShape s = tree_shape(p, batch);
        TreeArgs c = a;
        c.batch = (int32_t)batch;
        c.chunks = (int32_t)s.chunks;
        c.extra = (int32_t)s.extra;
        c.q += b0 * a.q_sb;
        c.out += b0 * a.o_sb;
        if (a.q_gran == REEF_SCALE_PER_TOKEN) c.qs += b0 * Hq * T;
        if (a.mask) c.mask += b0 * T;
        if (a.context_lens) c.context_lens += b0;
        if (PAGED) {
            c.block_table += b0 * a.max_blocks;
        } else {
            const int64_t tokens = b0 * p->kv_heads * p->max_context;
            c.k += tokens * D;
            c.v += tokens * D;
            c.ks += tokens;
            c.vs += tokens;
        }
        const dim3 grid((unsigned)s.wgs), block(64 * kWaves);
        if (D == 128 && s.nc == 1)
            hipLaunchKernelGGL((tree_kernel<128, PAGED, 1>), grid, block, 0, stream, c);
        else if (D == 128)
            hipLaunchKernelGGL((tree_kernel<128, PAGED, 2>), grid, block, 0, stream, c);
        else if (s.nc == 1)
            hipLaunchKernelGGL((tree_kernel<64, PAGED, 1>), grid, block, 0, stream, c);
        else
            hipLaunchKernelGGL((tree_kernel<64, PAGED, 2>), grid, block, 0, stream, c);
        if (hipGetLastError() != hipSuccess) return REEF_HIP_ERROR;
    }
    return REEF_OK;
}

}  // namespace
}  // namespace reef

using namespace reef;

extern "C" size_t reef_attention_decode_tree_workspace_bytes(const reef_tree_params *p) {
    if (!params_ok(p) || !params_supported(p)) return 0;
    return (size_t)tree_workspace(p);
}

extern "C" reef_status reef_attention_decode_tree_int8(
    const reef_tree_params *p, const int8_t *q, const reef_strides *q_strides,
    const float *q_scales, const int8_t *k_cache, const int8_t *v_cache, const float *k_scales,
    const float *v_scales, const int32_t *context_lens, const uint64_t *tree_mask, float *out,
    const reef_strides *out_strides, void *workspace, size_t workspace_bytes,
    uint32_t *status_word, hipStream_t stream) {
    const reef_status s = validate(p, q, q_strides, q_scales, k_cache, v_cache, k_scales, v_scales,
                                   tree_mask, out, out_strides, workspace, workspace_bytes);
    if (s != REEF_OK) return s;
    TreeArgs a = {};
    a.q = q;
    a.qs = q_scales;
    a.k = k_cache;
    a.v = v_cache;
    a.ks = k_scales;
    a.vs = v_scales;
    a.context_lens = context_lens;
    a.mask = tree_mask;
    a.out = out;
    a.status = status_word;
    return launch_tree<false>(p, a, q_strides, out_strides, workspace, stream);
}

extern "C" reef_status reef_attention_decode_tree_int8_paged(
    const reef_tree_params *p, const int8_t *q, const reef_strides *q_strides,
    const float *q_scales, const int8_t *k_pages, const int8_t *v_pages,
    const float *k_scale_pages, const float *v_scale_pages, const int32_t *block_table,
    int64_t max_blocks_per_seq, int64_t num_pages, const int32_t *context_lens,
    const uint64_t *tree_mask, float *out, const reef_strides *out_strides, void *workspace,
    size_t workspace_bytes, uint32_t *status_word, hipStream_t stream) {
    const reef_status s =
        validate(p, q, q_strides, q_scales, k_pages, v_pages, k_scale_pages, v_scale_pages,
                 tree_mask, out, out_strides, workspace, workspace_bytes);
    if (s != REEF_OK) return s;
    if (!block_table || !context_lens || num_pages <= 0 || num_pages >= (int64_t(1) << 31) ||
        max_blocks_per_seq * kPage < p->max_context || max_blocks_per_seq >= (int64_t(1) << 30))
        return REEF_INVALID_ARGUMENT;
    if (num_pages * p->kv_heads >= (int64_t(1) << 31)) return REEF_UNSUPPORTED;
    TreeArgs a = {};
    a.q = q;
    a.qs = q_scales;
    a.k = k_pages;
    a.v = v_pages;
    a.ks = k_scale_pages;
    a.vs = v_scale_pages;
    a.block_table = block_table;
    a.max_blocks = (int32_t)max_blocks_per_seq;
    a.num_pages = (int32_t)num_pages;
    a.context_lens = context_lens;
    a.mask = tree_mask;
    a.out = out;
    a.status = status_word;
    return launch_tree<true>(p, a, q_strides, out_strides, workspace, stream);
}
