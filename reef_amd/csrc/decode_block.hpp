// What the decode kernels share (gfx950): one 64-key block of a cache in 8 or 4 bits in registers,
// its scores, softmax and products. decode.hip reads int8 sequences front to back with it,
// decode_entries.hip 4-bit caches and the pages that a list names.
#pragma once

#include <algorithm>
#include <cmath>

#include "decode_common.hpp"
#include "kv_int4.hpp"

namespace reef {

constexpr int kDecodeWaves = 4;          // waves per workgroup
constexpr int kPlanItems = 2048;         // items whose block offsets a workgroup plans in LDS
constexpr int kWgPerCu = 2;              // resident workgroups per compute unit (at most)

struct DecodeArgs {
    const int8_t *q;
    const float *qs;
    const int8_t *k;        // contiguous cache or page pool
    const int8_t *v;
    const float *ks, *vs;
    const int32_t *block_table;  // paged only
    const int32_t *context_lens; // may be null
    uint32_t *counters;     // one per (sequence, kv head); zero between launches
    float *slots;           // DecodeSlot each: two a workgroup (decode.hip: the first and the last of
                            // its run), or one a part, in the plan's order (decode_entries.hip)
    uint32_t *status;
    int32_t batch, q_heads, kv_heads, group;
    int32_t max_context, window;
    int32_t items;  // batch * kv_heads: one (sequence, kv head) each
    int32_t wgs;    // workgroups of the launch
    int32_t flat;   // 1: the launch's keys are dealt out by 64-key blocks, 0: by items
    int32_t max_blocks, num_pages;               // paged only
    const int32_t *sel_pages;   // SEL only: [items, max_sel] page numbers of the sequence
    const int32_t *sel_counts;  // [items]
    int32_t max_sel;
    int32_t q_gran;
    float score_scale;  // softmax_scale * log2(e)
};

// Page number of page_idx of sequence b from the block table (paged only), read
// ahead of the page's data: pages at or past n_pages (the sequence's
// ceil(len / 16)) are not looked up.
template <bool PAGED>
__device__ __forceinline__ int table_page(const DecodeArgs &a, int b, int page_idx, int n_pages) {
    if (!PAGED || page_idx >= n_pages) return 0;
    return a.block_table[(int64_t)b * a.max_blocks + page_idx];
}

// Addresses of one 16-token page of (sequence b, kv head kvh), `page` its number
// from table_page. Pages at or past n_pages point at a safe page and are dead. A
// page number outside [0, num_pages) is an error.
struct PageRef {
    const int8_t *k;   // [16, D]
    const int8_t *vt;  // [D, 16]
    const float *ks, *vs;  // [16]
    bool live;  // holds keys of this sequence
    bool ok;    // false: the block table held an out-of-range page number
};

template <int D, int BITS, bool PAGED>
__device__ __forceinline__ PageRef page_ref(const DecodeArgs &a, int b, int kvh, int page_idx,
                                            int n_pages, int page) {
    PageRef r;
    const bool in_seq = page_idx < n_pages;
    if (PAGED) {
        const bool valid = page >= 0 && page < a.num_pages;
        r.ok = valid || !in_seq;
        r.live = in_seq && valid;
        if (!valid) page = 0;
        const int64_t slot = (int64_t)page * a.kv_heads + kvh;
        r.k = a.k + slot * (kPage * D * BITS / 8);
        r.vt = a.v + slot * (kPage * D * BITS / 8);
        r.ks = a.ks + slot * kPage;
        r.vs = a.vs + slot * kPage;
    } else {
        r.ok = true;
        r.live = in_seq;
        const int64_t seq = (int64_t)b * a.kv_heads + kvh;
        const int64_t tok = seq * a.max_context + (int64_t)(in_seq ? page_idx : 0) * kPage;
        r.k = a.k + tok * (D * BITS / 8);
        r.vt = a.v + tok * (D * BITS / 8);  // pages of [D, 16] are contiguous in the same order
        r.ks = a.ks + tok;
        r.vs = a.vs + tok;
    }
    return r;
}

// One 64-key block in registers: the operands of both matrix products and the scales of the
// lane's keys. (With 16 heads a column, per lane, those of key 16 grp + col: the 16 lanes of a
// group hold the 16 scales of its page, handed around within the row.)
template <int D, int BITS>
struct BlockRows {
    i32x4 k[4][D / 64];
    i32x4 v[D / 16];
};

// In 4 bits a lane's 16 (head_dim 64: 8) bytes of a key row hold the low nibbles' channels and,
// D/2 further, the high ones', and a channel's 16 tokens take 8 bytes.
template <int D>
struct BlockRows<D, 4> {
    typedef int32_t Row __attribute__((ext_vector_type(D / 32)));
    Row k[4];
    i32x2 v[D / 16];
};

template <int D, int BITS, int HEADS>
struct DecodeBlock : BlockRows<D, BITS> {
    static constexpr int S = HEADS == 16 ? 1 : HEADS;  // scales a lane loads
    float ks[S], vs[S];
    bool live;
    int pos;  // entries: position of the first token of this lane group's page
    bool ok;  // a chunk's entries: whether that page is there
};

// A wave's running state over its keys: max (log2 units), row sum, the value
// normalizer s_run and the accumulator in units of s_run.
template <int D>
struct DecodeRun {
    float m_run, l_run, s_run, inv_s;
    f32x4 acc[D / 16];
};

// 8-byte elements of one workgroup's part in the workspace: the output in
// [element][lane] order, then (max, sum).
template <int D>
struct DecodeSlot {
    static constexpr int O = 2 * (D / 16);
    static constexpr int ELEMS = (O + 1) * kWave;
};

template <int D>
__device__ __forceinline__ void reset_run(DecodeRun<D> &r) {
    r.m_run = -INFINITY;
    r.l_run = 0.0f;
    r.s_run = 0.0f;
    r.inv_s = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) r.acc[d] = f32x4{};
}

// Issues the loads of a block: the page of K rows (kp) and of scales, P and V (gp) of this lane.
template <int D, int BITS, int HEADS, bool NT>
__device__ __forceinline__ void load_pages(const PageRef &kp, const PageRef &gp, int col, int grp,
                                           DecodeBlock<D, BITS, HEADS> &x, bool &bad_page) {
    bad_page |= !gp.ok;
    x.live = gp.live;
    if constexpr (BITS == 8) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int s = 0; s < D / 64; ++s)
                x.k[t][s] = load_stream<NT>(reinterpret_cast<const i32x4 *>(
                    kp.k + (4 * t + (col & 3)) * D + 64 * s + 16 * grp));
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
            x.v[d] = load_stream<NT>(reinterpret_cast<const i32x4 *>(gp.vt + (16 * d + col) * kPage));
    } else {
        using Row = typename BlockRows<D, BITS>::Row;
#pragma unroll
        for (int t = 0; t < 4; ++t)
            x.k[t] = load_stream<NT>(reinterpret_cast<const Row *>(
                kp.k + (4 * t + (col & 3)) * (D / 2) + D / 8 * grp));
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
            x.v[d] = load_stream<NT>(
                reinterpret_cast<const i32x2 *>(gp.vt + (16 * d + col) * (kPage / 2)));
    }
    if constexpr (HEADS == 16) {
        x.ks[0] = gp.ks[col];
        x.vs[0] = gp.vs[col];
    } else {
        const int key = col / HEADS * HEADS;  // of the page: this column's first
#pragma unroll
        for (int i = 0; i < HEADS; i += 4) {
            const f32x4 ks = *reinterpret_cast<const f32x4 *>(gp.ks + key + i);
            const f32x4 vs = *reinterpret_cast<const f32x4 *>(gp.vs + key + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x.ks[i + j] = ks[j];
                x.vs[i + j] = vs[j];
            }
        }
    }
}

// A lane's query operand. In 4 bits at head_dim 64 its channels are those of the nibbles that
// a lane group loads; `zero` is what the 8 added to every key code adds to a score, negated: the
// start of the accumulators.
template <int D>
struct Query {
    i32x4 op[D / 64];
    float c;   // the head's score factor in units of log 2
    int zero;  // BITS 4
};

// Scores of 16 keys as int32, exactly.
template <int D>
__device__ __forceinline__ i32x4 tile_scores(const BlockRows<D, 8> &x, int t, const Query<D> &q) {
    i32x4 s = {0, 0, 0, 0};
#pragma unroll
    for (int ks = 0; ks < D / 64; ++ks) s = mfma_16x16x64_i8(x.k[t][ks], q.op[ks], s);
    return s;
}
template <int D>
__device__ __forceinline__ i32x4 tile_scores(const BlockRows<D, 4> &x, int t, const Query<D> &q) {
    i32x4 lo, hi, s = {q.zero, q.zero, q.zero, q.zero};
    if constexpr (D == 128) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lo[i] = (int)low_nibbles((uint32_t)x.k[t][i]);
            hi[i] = (int)high_nibbles((uint32_t)x.k[t][i]);
        }
        s = mfma_16x16x64_i8(lo, q.op[0], s);
        return mfma_16x16x64_i8(hi, q.op[1], s);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            lo[i] = (int)low_nibbles((uint32_t)x.k[t][i]);
            lo[2 + i] = (int)high_nibbles((uint32_t)x.k[t][i]);
        }
        return mfma_16x16x64_i8(lo, q.op[0], s);
    }
}

// One channel's 16 values as the operands of two products, exactly.
__device__ __forceinline__ void value_operands(i32x4 w, f16x8 &lo, f16x8 &hi) {
    int8x16_to_f16(w, lo, hi);
}
__device__ __forceinline__ void value_operands(i32x2 w, f16x8 &lo, f16x8 &hi) {
    lo = int4x8_to_f16((uint32_t)w[0]);
    hi = int4x8_to_f16((uint32_t)w[1]);
}

// The scores of a page's 16 keys, HEADS to a column: column HEADS j + h takes head h's of keys
// HEADS j .. HEADS j + HEADS - 1 (of tile HEADS j / 4 on), one masked row shift each.
template <int SHIFT, int BANKS>
__device__ __forceinline__ int from_column(int own, int x) {
    return __builtin_amdgcn_update_dpp(own, x, 0x110 + SHIFT, 0xf, BANKS, false);
}
__device__ __forceinline__ void spread(const i32x4 (&s)[4], int (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        x[i] = from_column<12, 8>(from_column<8, 4>(from_column<4, 2>(s[0][i], s[1][i]), s[2][i]),
                                  s[3][i]);
}
__device__ __forceinline__ void spread(const i32x4 (&s)[4], int (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = from_column<8, 12>(s[i / 4][i % 4], s[2 + i / 4][i % 4]);
}

// Scores, online softmax and P.V of one block for keys [lo, k_end).
template <int D, int BITS, int HEADS, bool SEL>
__device__ __forceinline__ void block_math(const DecodeBlock<D, BITS, HEADS> &cur, int kb, int lo,
                                           int k_end, const Query<D> &q, int lane,
                                           DecodeRun<D> &st) {
    constexpr int DB = D / 16;
    const int grp = lane >> 4, col = lane & 15;
    const auto &vop = cur.v;
    const float c = q.c;
    float ksc[HEADS], vsc[HEADS];
    if constexpr (HEADS == 16) {
        row_lanes(cur.ks[0], ksc);
        row_lanes(cur.vs[0], vsc);
    } else {
#pragma unroll
        for (int r = 0; r < HEADS; ++r) {
            ksc[r] = cur.ks[r];
            vsc[r] = cur.vs[r];
        }
    }
    const bool live_g = cur.live;

    float x[HEADS];
    if constexpr (HEADS == 16) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const i32x4 s = tile_scores<D>(cur, t, q);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[4 * t + i] = (float)s[i] * (c * ksc[4 * t + i]);
        }
    } else {
        i32x4 s[4];
        int sx[HEADS];
#pragma unroll
        for (int t = 0; t < 4; ++t) s[t] = tile_scores<D>(cur, t, q);
        spread(s, sx);
#pragma unroll
        for (int r = 0; r < HEADS; ++r) x[r] = (float)sx[r] * (c * ksc[r]);
    }
    // Blocks wholly inside [lo, k_end) on live pages skip the masks. In the
    // others, keys outside or on a dead page take no part: score -inf and
    // value scale 0 (the cache past a sequence's end may hold anything).
    const int pos = SEL ? cur.pos : kb + 16 * grp;  // of this lane group's page
    const bool full = SEL ? __all(live_g && pos >= lo && pos + kPage <= k_end)
                          : kb >= lo && kb + kBlockKeys <= k_end && __all(live_g);
    float vv[HEADS];
    if (full) {
#pragma unroll
        for (int r = 0; r < HEADS; ++r) vv[r] = vsc[r];
    } else {
        const int first = HEADS == 16 ? pos : pos + col / HEADS * HEADS;  // of this column
#pragma unroll
        for (int r = 0; r < HEADS; ++r) {
            const int key = first + r;
            const bool vis = key >= lo && key < k_end && live_g;
            if (!vis) x[r] = -INFINITY;
            vv[r] = vis ? vsc[r] : 0.0f;
        }
    }
    float mt = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    float vmax = fmaxf(fmaxf(vv[0], vv[1]), fmaxf(vv[2], vv[3]));
#pragma unroll
    for (int r = 4; r < HEADS; r += 2) {
        mt = fmaxf(mt, fmaxf(x[r], x[r + 1]));
        vmax = fmaxf(vmax, fmaxf(vv[r], vv[r + 1]));
    }
    if constexpr (HEADS == 16) {
        mt = fmaxf(mt, __shfl_xor(mt, 16));
        mt = fmaxf(mt, __shfl_xor(mt, 32));
        vmax = fmaxf(vmax, __shfl_xor(vmax, 16));
        vmax = fmaxf(vmax, __shfl_xor(vmax, 32));
    } else {
        mt = xor32_max(xor16_max(mt));
        vmax = xor32_max(xor16_max(vmax));
    }

    // Lazy rescale: the running max moves only when a head's block max exceeds
    // it by more than 2^6, and the value normalizer s_run (values accumulate in
    // units of s_run / 2^8, s_run the largest value scale so far) only when a value
    // scale exceeds it 2-fold, so the weight p * v_scale * 2^8 / s_run stays below
    // 2^15 in fp16, and above its subnormals (hi and lo keep 11 bits each) wherever
    // its share of the row sum (of p itself) exceeds 2^-21.
    if (__any(mt > st.m_run + 6.0f || vmax > st.s_run * 2.0f)) {
        const float m_new = fmaxf(st.m_run, mt);
        const float s_new = fmaxf(fmaxf(st.s_run, vmax), kLeastScale);
        const float alpha = st.m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st.m_run - m_new);
        const float alpha_o = alpha * (st.s_run / s_new);
        st.inv_s = 256.0f / s_new;
        st.m_run = m_new;
        st.s_run = s_new;
        st.l_run *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d) st.acc[d] *= alpha_o;
    }
    const float m_use = st.m_run == -INFINITY ? 0.0f : st.m_run;

    // P operand: lane group g's keys 16g + 8h + e for the two halves h, each weight
    // p * v_scale / s_run split into an fp16 part and the fp16 of its remainder
    // (22 significant bits together: one fp16 alone moves an output by up to
    // 2^-12 of the values' magnitude, about 1e-3 for |v| ~ 4). The products run
    // on both; the row sum stays the fp32 sum of p.
    f16x8 pop[2], plo[2];
    float lp[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    auto weight = [&](int r) {
        const float p = __builtin_amdgcn_exp2f(x[r] - m_use);
        lp[r & 3] += p;
        return p * (vv[r] * st.inv_s);
    };
    if constexpr (HEADS == 16) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = weight(8 * h + e);
            split_weights(w, pop[h], plo[h]);
        }
    } else {
        // this column's keys alone, in their places of the 16
        typedef _Float16 Part __attribute__((ext_vector_type(HEADS)));
        typedef int32_t Words __attribute__((ext_vector_type(HEADS / 2)));
        float w[HEADS];
#pragma unroll
        for (int r = 0; r < HEADS; ++r) w[r] = weight(r);
        Part hi, lo_part;
        split_weights(w, hi, lo_part);
        const Words wh = __builtin_bit_cast(Words, hi), wl = __builtin_bit_cast(Words, lo_part);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            i32x4 oh, ol;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool mine = col / HEADS == (8 * h + 2 * i) / HEADS;
                oh[i] = mine ? wh[i % (HEADS / 2)] : 0;
                ol[i] = mine ? wl[i % (HEADS / 2)] : 0;
            }
            pop[h] = __builtin_bit_cast(f16x8, oh);
            plo[h] = __builtin_bit_cast(f16x8, ol);
        }
    }
    st.l_run += (lp[0] + lp[1]) + (lp[2] + lp[3]);
    // out^T = V^T . P^T: the output column is the head (lane % 16), the lane
    // that owns the head's running max, so the rescale above is per lane.
#pragma unroll
    for (int d = 0; d < DB; ++d) {
        f16x8 v0, v1;
        value_operands(vop[d], v0, v1);
        st.acc[d] = mfma_16x16x32_f16(v0, pop[0], st.acc[d]);
        st.acc[d] = mfma_16x16x32_f16(v0, plo[0], st.acc[d]);
        st.acc[d] = mfma_16x16x32_f16(v1, pop[1], st.acc[d]);
        st.acc[d] = mfma_16x16x32_f16(v1, plo[1], st.acc[d]);
    }
}

// The q^T operand of a query row (zeros for a dead column), with the score factor c.
template <int D, int BITS>
__device__ __forceinline__ Query<D> query_of(const int8_t *qrow, bool live, float c, int grp) {
    Query<D> q;
    q.zero = 0;
    if constexpr (BITS == 4 && D == 64) {
        const i32x2 lo = *reinterpret_cast<const i32x2 *>(qrow + 8 * grp);
        const i32x2 hi = *reinterpret_cast<const i32x2 *>(qrow + 32 + 8 * grp);
        q.op[0] = live ? i32x4{lo[0], lo[1], hi[0], hi[1]} : i32x4{0, 0, 0, 0};
    } else {
#pragma unroll
        for (int s = 0; s < D / 64; ++s)
            q.op[s] = live ? *reinterpret_cast<const i32x4 *>(qrow + 64 * s + 16 * grp)
                           : i32x4{0, 0, 0, 0};
    }
    if constexpr (BITS == 4) {
        int sum = 0;
#pragma unroll
        for (int s = 0; s < D / 64; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_sdot4(q.op[s][i], 0x01010101, sum, false);
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        q.zero = -kInt4Zero * sum;
    }
    q.c = c;
    return q;
}

// The q^T operand of query head `head` of sequence b (zeros for dead heads) and the log2-domain
// score factor of head `scored` (the one whose scores the lane holds; zero for a dead one).
template <int D, int BITS>
__device__ __forceinline__ Query<D> load_query(const DecodeArgs &a, int b, int head, bool head_ok,
                                               int scored, bool scored_ok, int grp) {
    const int8_t *qrow = a.q + ((int64_t)b * a.q_heads + (head_ok ? head : 0)) * D;
    float cq = 0.0f;
    if (scored_ok) {
        cq = a.q_gran == REEF_SCALE_PER_TENSOR ? a.qs[0]
             : a.q_gran == REEF_SCALE_PER_HEAD ? a.qs[scored]
                                                : a.qs[(int64_t)b * a.q_heads + scored];
    }
    return query_of<D, BITS>(qrow, head_ok, cq * a.score_scale, grp);
}

// Keys of one item (sequence b = item / kv_heads): its length (0 if the length is
// out of range), the first visible key, and its 64-key blocks from the block that
// holds that key. An item with no keys still counts one block, so that some
// workgroup stores its (zero) output.
struct ItemKeys {
    int len, lo, first_block, blocks;
    int count;  // SEL: entries of its list, whose blocks are the item's
    bool bad;
};

template <bool SEL>
__device__ __forceinline__ ItemKeys item_keys(const DecodeArgs &a, int item) {
    ItemKeys r;
    const int b = item / a.kv_heads;
    int len = a.context_lens ? a.context_lens[b] : a.max_context;
    r.bad = len < 1 || len > a.max_context;
    r.count = 0;
    if constexpr (SEL) {
        r.count = a.sel_counts[item];
        r.bad |= r.count < 0 || r.count > a.max_sel;
        if (r.bad) r.count = 0;
    }
    if (r.bad) len = 0;
    r.len = len;
    r.lo = a.window > 0 ? max(0, len - a.window) : 0;
    if constexpr (SEL) {
        constexpr int kEntries = kBlockKeys / kPage;
        r.first_block = 0;
        r.blocks = max(1, (r.count + kEntries - 1) / kEntries);
        return r;
    }
    r.first_block = r.lo / kBlockKeys;
    r.blocks = len > 0 ? (len + kBlockKeys - 1) / kBlockKeys - r.first_block : 1;
    return r;
}

// --- host: checks and sizes of a decode call (decode.hip) -----------------------------------

reef_status decode_validate(const reef_decode_params *p, const int8_t *q, const float *q_scales,
                            float *out, void *workspace, size_t workspace_bytes);

// Whether the launch deals out 64-key blocks of sequences of `tokens` tokens at most (the items'
// prefix fits the LDS plan and the block count of the largest possible launch fits 31 bits).
bool decode_flat(const reef_decode_params *p, int64_t tokens);

// The workspace's counters, one per (sequence, kv head), ahead of the part slots.
constexpr int64_t kDecodeCounterBytes = kPlanItems * 4;

// A chunk's attention over the 4-bit cache in decode_entries.hip: whether it is small enough to be
// the faster way, and the launch (arguments as prefill_cache.hip has checked them; counters zero
// and left so, slots for two parts a workgroup, two workgroups a compute unit).
bool chunk_entries_fit(const reef_attention_params *p);
reef_status launch_chunk_int4(const reef_attention_params *p, const int8_t *q, const int64_t (&qst)[3],
                              const float *q_scales, const uint8_t *k_cache, const uint8_t *v_cache,
                              const float *k_scales, const float *v_scales, int64_t max_context,
                              const int32_t *block_table, int64_t max_blocks_per_seq,
                              int64_t num_pages, float *out, const int64_t (&ost)[3], char *counters,
                              char *slots, uint32_t *status_word, hipStream_t stream);

inline void set_decode_args(const reef_decode_params *p, DecodeArgs &a) {
    a.batch = (int32_t)p->batch;
    a.q_heads = (int32_t)p->q_heads;
    a.kv_heads = (int32_t)p->kv_heads;
    a.group = (int32_t)(p->q_heads / p->kv_heads);
    a.max_context = (int32_t)p->max_context;
    a.window = (int32_t)std::min<int64_t>(p->window, INT32_MAX);
    a.q_gran = p->q_granularity;
    a.score_scale = p->softmax_scale * kLog2e;
    a.items = (int32_t)(p->batch * p->kv_heads);
}

}  // namespace reef
