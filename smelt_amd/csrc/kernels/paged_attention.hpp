// Attention of new token rows over a paged key / value cache, with a prefix that the whole batch shares.
//
//   y(row) = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c (q.k_j - m)),  c = |scale| * log2(e),  m the running maximum of q.k (q negated for
//   a negative scale)
//
// over the keys j the row sees (causal, within the window).  Scores, maxima, sums and the output accumulators are 32-bit; p is
// rounded to the 16-bit type for the second product (relative error half a step of that type, averaged over the keys), its sum is not.
// The maximum only moves when a score passes it by more than 8 / c (p then stays below 2^8, far inside fp16), so most key tiles
// rescale nothing.
//
// Rows are (token, head of the group) pairs of one kv head, 32 to a tile, and both products are formed transposed, so that a lane
// owns one row throughout (v_mfma_f32_32x32x16, lane l: row l % 32):
//   S^T [32 keys x 32 rows] = K Q^T       a lane ends up with 16 of the 32 scores of its row, lane ^ 32 with the others
//   O^T [dim x 32 rows]    += V^T P^T     the lane's own 16 probabilities are its operand as they stand: the order of the keys of
//                                         a contraction is free, so V rows are taken in the order the first product left them
// Maximum, sum and rescaling are per lane; nothing crosses lanes but one exchange of the maximum.  K is stored in operand order
// ([dim / 8][key][8] within a page and head: a load covers 512 contiguous bytes per half wave); V rows are read as they are stored.
//
// A workgroup's way to its first key is a chain of dependent loads and of instructions fetched for the first time; the code in
// front of the key loops is kept rolled for that reason (unrolled, it cost about 8 us a launch).
#pragma once
#include "common.hpp"
#include "serving_args.hpp"

namespace smelt {

using smelt_serving::AttentionArgs;
using smelt_serving::AttentionEntry;

typedef __bf16 attn_bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 attn_bf16x2_t __attribute__((ext_vector_type(2)));
typedef float attn_float2_t __attribute__((ext_vector_type(2)));

template <class ActT>
__device__ __forceinline__ float16_t attn_mfma(uint4_t a, uint4_t b, float16_t c) {
    if constexpr (ActT::kIsF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(attn_bf16x8_t, a), __builtin_bit_cast(attn_bf16x8_t, b), c, 0, 0, 0);
}

// two values to the 16-bit type, round to nearest even, lo in the low half
template <class ActT>
__device__ __forceinline__ uint32_t attn_pack2(float lo, float hi) {
    if constexpr (ActT::kIsF16) {
        const half2_t h = {(_Float16)lo, (_Float16)hi};
        return __builtin_bit_cast(uint32_t, h);
    } else {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((attn_float2_t{lo, hi}), attn_bf16x2_t));
    }
}

// maximum and sum of a lane's value and lane ^ 32's
__device__ __forceinline__ float attn_halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float attn_halves_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}
__device__ __forceinline__ float attn_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
using smelt_serving::AttentionSpan;
using smelt_serving::AttentionSplit;
using smelt_serving::AttentionTiles;

// Lengths and page tables are read through the scalar cache where they are the same for the whole wave (nobody writes them while a
// launch runs): a vector load's wait would be one for the key and value loads in flight before it.
typedef const __attribute__((address_space(4))) int32_t* scalar_table;
__device__ __forceinline__ scalar_table as_scalar(const int32_t* p) { return (scalar_table)(uintptr_t)p; }
struct AttnScalarLoad { __device__ __forceinline__ int32_t operator()(const int32_t* p, uint32_t i) const { return as_scalar(p)[__builtin_amdgcn_readfirstlane(i)]; } };
__device__ __forceinline__ AttentionEntry attn_entry(const AttentionArgs& a, uint32_t index) { return smelt_serving::attention_entry(a, index, AttnScalarLoad()); }

// What a workgroup looks for: its first unit (or its segment), the first unit of the workgroup after it, or the entry of a token.
enum AttnWanted { kFirstUnit, kCut, kToken };
struct AttnWork {
    AttentionSplit split;    // of the whole launch
    uint32_t entry;          // where the wanted unit, segment or row lies (~0: nowhere)
    uint32_t base;           // units (segments where each workgroup takes one) before that entry
    uint32_t at;             // the wanted unit (segment)
};

// Each wave looks for itself (no barrier), an entry a lane: once through the entries for their total, then for the wanted one.
template <AttnWanted WANTED>
__device__ __forceinline__ AttnWork find_work(const AttentionArgs& a, uint32_t want) {
    const uint32_t entries = smelt_serving::attention_entries(a), lane = threadIdx.x % kWave;
    AttnWork w;
    w.entry = ~0u;
    w.base = w.at = 0;
    uint32_t mine[2] = {0, 0}, before[2] = {0, 0}, all[2] = {0, 0};      // units and segments: the lane's entry, the entries before it in the round, the round's
    bool here = false;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        uint32_t run[2] = {0, 0};
#pragma unroll 1
        for (uint32_t base = 0; base < entries; base += kWave) {
            const uint32_t index = base + lane;
            if (pass == 0 || entries > (uint32_t)kWave) {
                mine[0] = mine[1] = 0;
                here = false;
                if (index < entries) {
                    const AttentionEntry e = smelt_serving::attention_entry(a, index);
                    mine[0] = smelt_serving::attention_units(a, e);
                    mine[1] = smelt_serving::attention_segments(a, e);
                    here = want >= e.first_token && want - e.first_token < e.tokens;
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t sum = mine[k];
#pragma unroll
                    for (uint32_t d = 1; d < (uint32_t)kWave; d <<= 1) {
                        const uint32_t up = __shfl_up(sum, d);
                        if (lane >= d) sum += up;
                    }
                    before[k] = sum - mine[k];
                    all[k] = __builtin_amdgcn_readlane(sum, kWave - 1);
                }
            }
            if (pass == 1) {
                const int k = w.split.whole ? 1 : 0;
                const uint32_t first = run[k] + before[k];
                const bool ok = WANTED == kToken ? here : w.at >= first && w.at - first < mine[k];
                const unsigned long long who = __ballot(ok);
                if (who) {
                    const int from = __builtin_ctzll(who);
                    w.entry = __builtin_amdgcn_readfirstlane(base + from);
                    w.base = __builtin_amdgcn_readlane(first, from);
                    return w;
                }
            }
            run[0] += all[0];
            run[1] += all[1];
        }
        if (pass == 1) break;
        w.split = smelt_serving::attention_split(a, run[0], run[1]);
        if (WANTED != kToken) {
            const uint32_t group = want + (WANTED == kCut ? 1u : 0u);
            if (group >= w.split.groups || (WANTED == kCut && w.split.whole)) return w;
            w.at = w.split.whole ? group : smelt_serving::attention_start(w.split, group);
        }
    }
    return w;
}

// A segment and the part of its key tiles that a workgroup takes.
struct AttnSegment {
    uint32_t kv_head, row_tile;
    AttentionTiles tiles;        // the segment's
    uint32_t first, last;        // the workgroup's part of them
    bool whole;
    uint32_t begin;              // the segment's first unit
};
// the segment that holds unit `unit` of entry e, whose units start at `base`; false (and g.begin behind them) when the entry has fewer
__device__ __forceinline__ bool attn_segment(const AttentionArgs& a, const AttentionEntry& e, uint32_t base, uint32_t unit, uint32_t unit_end, AttnSegment& g) {
    uint32_t rel = unit - base;
    g.begin = base;
#pragma unroll 1
    for (g.row_tile = 0; g.row_tile < e.row_tiles; ++g.row_tile) {
        g.tiles = smelt_serving::attention_tiles(a, e, g.row_tile);
        const uint32_t tiles = g.tiles.hi - g.tiles.lo, size = tiles * a.kv_heads;
        if (rel >= size) { rel -= size; g.begin += size; continue; }
        g.kv_head = rel / tiles;
        const uint32_t done = rel - g.kv_head * tiles;
        g.begin += g.kv_head * tiles;
        g.first = g.tiles.lo + done;
        g.last = tiles - done < unit_end - unit ? g.tiles.hi : g.first + (unit_end - unit);
        g.whole = done == 0 && g.last == g.tiles.hi;
        return true;
    }
    return false;
}
// segment `index` of entry e (whole), the longest first: rows at the end of a sequence see the most keys
__device__ __forceinline__ void attn_whole_segment(const AttentionArgs& a, const AttentionEntry& e, uint32_t index, AttnSegment& g) {
    g.row_tile = e.row_tiles - 1 - index / a.kv_heads;
    g.kv_head = index % a.kv_heads;
    g.tiles = smelt_serving::attention_tiles(a, e, g.row_tile);
    g.first = g.tiles.lo;
    g.last = g.tiles.hi;
    g.whole = true;
    g.begin = 0;
}

// the sequence of a token row: offsets is ascending, tokens before offsets[sequences] belong to one
__device__ __forceinline__ uint32_t sequence_of(const AttentionArgs& a, uint32_t token) {
    uint32_t lo = 0, hi = a.sequences;   // offsets[lo] <= token < offsets[hi]
#pragma unroll 1
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (smelt_serving::clamp_count(a.offsets[mid], a.tokens) <= token) lo = mid;
        else hi = mid;
    }
    return lo;
}

// What a lane knows of its row.
struct AttnRow {
    bool live;
    uint32_t token, head;     // head: within the kv head's group
    int32_t position;         // among prefix and own keys
};

__device__ __forceinline__ AttnRow attn_row(const AttentionArgs& a, const AttentionEntry& e, uint32_t row) {
    AttnRow r;
    r.live = row < e.tokens * a.group;
    const uint32_t i = r.live ? row / a.group : 0u;
    r.head = r.live ? row - i * a.group : 0u;
    r.token = e.first_token + i;
    uint32_t first = e.first_token, count = e.tokens, own = e.own;
    if (e.sequence < 0) {
        const uint32_t s = sequence_of(a, r.token);
        first = smelt_serving::clamp_count(a.offsets[s], a.tokens);
        count = smelt_serving::clamp_count(a.offsets[s + 1], a.tokens) - first;
        own = smelt_serving::clamp_count(a.kv_lens[s], a.pages_per_sequence << a.page_shift);
    }
    r.position = (int32_t)(e.prefix + own + (r.token - first)) - (int32_t)count;
    return r;
}

// Keys of one run that a row sees: lo <= key < hi.
struct AttnBounds { int32_t lo, hi; };
__device__ __forceinline__ AttnBounds attn_bounds(const AttentionArgs& a, const AttnRow& r, int32_t run_base, int32_t run_len) {
    AttnBounds b{0, run_len};
    if (!r.live) return b;
    const int32_t p = r.position - run_base;
    b.hi = p + 1 < run_len ? p + 1 : run_len;
    if (a.window != 0 && p >= (int32_t)a.window) b.lo = p - (int32_t)a.window + 1;
    return b;
}

// Keys of one run that some row of a wave sees, and that all of its rows see.
struct AttnRun { int32_t len, lo, hi, all_lo, all_hi; };
__device__ __forceinline__ AttnRun attn_run(const AttentionArgs& a, const AttentionEntry& e, int run, uint32_t row0, const AttnRow& row) {
    AttnRun u;
    u.len = (int32_t)(run ? e.own : e.front);
    u.lo = u.all_lo = 0;
    u.hi = u.all_hi = u.len;
    const int32_t base = run ? (int32_t)e.prefix : 0;
    if (e.sequence < 0) {        // rows of many sequences: they mostly see all of it
        const AttnBounds b = attn_bounds(a, row, 0, u.len);
        if (__any(b.lo != 0 || b.hi != u.len)) u.all_hi = 0;
    } else if (row0 < e.tokens * a.group) {
        const AttentionSpan s = smelt_serving::attention_span(a, e, row0, 32);
        const int32_t hi = s.hi - base, all_hi = s.all_hi - base;
        u.lo = s.lo - base > 0 ? s.lo - base : 0;
        u.all_lo = s.all_lo - base > 0 ? s.all_lo - base : 0;
        u.hi = hi < u.len ? hi : u.len;
        u.all_hi = all_hi < u.len ? all_hi : u.len;
    } else {
        u.hi = 0;                // no rows here
    }
    return u;
}
__device__ __forceinline__ bool attn_seen(const AttnRun& u, int32_t key0) { return key0 < u.hi && key0 + (int32_t)smelt_serving::kKeyTile > u.lo; }
__device__ __forceinline__ bool attn_masked(const AttnRun& u, int32_t key0) { return key0 + (int32_t)smelt_serving::kKeyTile > u.all_hi || key0 < u.all_lo; }

// One wave's state: 32 rows.
template <int D>
struct AttnAcc {
    float16_t o[D / 32];     // o[j][i]: value (D / 32) * (8 (i / 4) + 4 (lane / 32) + i % 4) + j of the lane's row
    float m, l;              // running maximum of q.k and this half's sum
};

template <class ActT, int D>
__device__ __forceinline__ void attn_load_q(const AttentionArgs& a, const AttnRow& r, uint32_t kv_head, uint4_t* qf) {
    const int half = (threadIdx.x & 63) >> 5;
    const uint16_t* q = a.q + (size_t)r.token * a.q_stride + (size_t)(kv_head * a.group + r.head) * D + 8 * half;
    if ((reinterpret_cast<uintptr_t>(a.q) & 15u) == 0 && (a.q_stride & 7u) == 0) {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) qf[t] = r.live ? *reinterpret_cast<const uint4_t*>(q + 16 * t) ^ a.flip_q : uint4_t{0, 0, 0, 0};
    } else {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = r.live ? (uint32_t)q[16 * t + 2 * k] | ((uint32_t)q[16 * t + 2 * k + 1] << 16) : 0u;
            qf[t] = uint4_t{w[0], w[1], w[2], w[3]} ^ a.flip_q;
        }
    }
}

// Address of one key tile: the page (two for pages of 16) and whether it is one of the pool's.
template <bool SMALL>
struct AttnTile {
    size_t base[SMALL ? 2 : 1];      // element offset of the page's head
    uint32_t known;                  // bits 0 and 1: the pages of the tile's halves are the pool's
    uint32_t off;                    // first key within the page
};

template <bool SMALL, int D>
__device__ __forceinline__ AttnTile<SMALL> attn_tile(const AttentionArgs& a, const int32_t* table, uint32_t kv_head, uint32_t run_len, uint32_t tile) {
    AttnTile<SMALL> t;
    const uint32_t key = tile * smelt_serving::kKeyTile;
    const uint32_t last_page = run_len ? (run_len - 1) >> a.page_shift : 0u;
    t.known = 0;
    t.off = SMALL ? 0u : key & ((1u << a.page_shift) - 1u);
#pragma unroll
    for (int k = 0; k < (SMALL ? 2 : 1); ++k) {
        uint32_t index = (key >> a.page_shift) + k;
        if (index > last_page) index = last_page;      // behind the run: masked by its length
        const uint32_t page = (uint32_t)as_scalar(table)[__builtin_amdgcn_readfirstlane(index)];
        const bool known = page < a.pages;
        t.known |= known ? (SMALL ? 1u << k : 3u) : 0u;
        t.base[k] = (((size_t)(known ? page : 0u) * a.kv_heads + kv_head) * D) << a.page_shift;
    }
    return t;
}

template <int D, bool SMALL>
__device__ __forceinline__ void attn_load_k(const AttentionArgs& a, const AttnTile<SMALL>& t, uint4_t* kf) {
    const uint32_t lane = threadIdx.x & 63, half = lane >> 5, key = lane & 31;
    const uint16_t* base;
    uint32_t at;
    if (SMALL) { base = a.k_cache + (key < 16 ? t.base[0] : t.base[SMALL ? 1 : 0]); at = key & 15; }
    else { base = a.k_cache + t.base[0]; at = t.off + key; }
    const uint32_t lane_off = ((half << a.page_shift) + at) * 8;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) kf[s] = *reinterpret_cast<const uint4_t*>(base + lane_off + ((uint32_t)(2 * s) << a.page_shift) * 8);
}

// D / 32 neighbouring values of 16 keys: vf[u][r] is key 16 u + 8 (r / 4) + 4 half + r % 4 of the tile
template <int D>
struct AttnV { uint32_t w[2][8][D / 64]; };

template <int D, bool SMALL>
__device__ __forceinline__ void attn_load_v(const AttentionArgs& a, const AttnTile<SMALL>& t, AttnV<D>& vf) {
    const uint32_t lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const uint32_t key = 8 * (r / 4) + 4 * half + (r % 4) + (SMALL ? 0u : 16 * u + t.off);
            const uint32_t* src = reinterpret_cast<const uint32_t*>(a.v_cache + t.base[SMALL ? u : 0] + key * D) + col * (D / 64);
            if constexpr (D == 256) { const uint4_t v = *reinterpret_cast<const uint4_t*>(src); vf.w[u][r][0] = v.x; vf.w[u][r][1] = v.y; vf.w[u][r][2] = v.z; vf.w[u][r][3] = v.w; }
            else if constexpr (D == 128) { const uint2_t v = *reinterpret_cast<const uint2_t*>(src); vf.w[u][r][0] = v.x; vf.w[u][r][1] = v.y; }
            else vf.w[u][r][0] = *src;
        }
}

// one key tile: scores, running maximum and sum, second product
template <class ActT, int D, bool SMALL>
__device__ __forceinline__ void attn_scores(const AttentionArgs& a, const uint4_t* qf, const uint4_t* kf, float16_t& s) {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) s = attn_mfma<ActT>(kf[t], qf[t], s);
}

// scores of NS key tiles to probabilities: the running maximum and sum move on; s becomes p
struct AttnScale { float c, slack; };     // c, and what a score may pass the maximum by: 8 / c
__device__ __forceinline__ AttnScale attn_scale(const AttentionArgs& a) {
    return AttnScale{a.scale_log2, __builtin_fminf(8.0f / a.scale_log2, 1.0e38f)};
}

// hides the keys of a tile that the row does not see, `known`: bit 0 and 1 for the pages of its two halves
__device__ __forceinline__ void attn_hide(float16_t& s, int32_t key0, const AttnBounds& b, uint32_t known) {
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int32_t key = key0 + 8 * (i / 4) + 4 * half + i % 4;
        const bool ok = key >= b.lo && key < b.hi && ((known >> (i / 8)) & 1u);
        s[i] = ok ? s[i] : -__builtin_inff();
    }
}

template <int D, int NS>
__device__ __forceinline__ void attn_softmax(const AttnScale& c, AttnAcc<D>& acc, float16_t* s) {
    float top = s[0][0];
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int i = 0; i < 16; i += 2) top = __builtin_fmaxf(__builtin_fmaxf(top, s[n][i]), s[n][i + 1]);
    top = attn_halves_max(top);
    if (__any(top > acc.m + c.slack)) {      // also the first finite score: the maximum starts at -inf
        const float m = __builtin_fmaxf(acc.m, top);
        const float f = m == -__builtin_inff() ? 1.0f : attn_exp2((acc.m - m) * c.c);
        acc.l *= f;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc.o[j][i] *= f;
        acc.m = m;
    }
    const float shift = acc.m == -__builtin_inff() ? 0.0f : -acc.m * c.c;
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) { s[n][i] = attn_exp2(__builtin_fmaf(s[n][i], c.c, shift)); sum[i & 1] += s[n][i]; }
    acc.l += sum[0] + sum[1];
}

// the second product's operand of 16 keys
template <class ActT>
__device__ __forceinline__ uint4_t attn_pack(const float16_t& p, int u) {
    return uint4_t{attn_pack2<ActT>(p[8 * u], p[8 * u + 1]), attn_pack2<ActT>(p[8 * u + 2], p[8 * u + 3]), attn_pack2<ActT>(p[8 * u + 4], p[8 * u + 5]),
                   attn_pack2<ActT>(p[8 * u + 6], p[8 * u + 7])};
}

template <class ActT, int D>
__device__ __forceinline__ void attn_values(AttnAcc<D>& acc, const float16_t& p, const AttnV<D>& vf) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const uint4_t pf = attn_pack<ActT>(p, u);
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
            uint4_t v;
            v.x = __builtin_amdgcn_perm(vf.w[u][1][j / 2], vf.w[u][0][j / 2], sel);
            v.y = __builtin_amdgcn_perm(vf.w[u][3][j / 2], vf.w[u][2][j / 2], sel);
            v.z = __builtin_amdgcn_perm(vf.w[u][5][j / 2], vf.w[u][4][j / 2], sel);
            v.w = __builtin_amdgcn_perm(vf.w[u][7][j / 2], vf.w[u][6][j / 2], sel);
            acc.o[j] = attn_mfma<ActT>(v, pf, acc.o[j]);
        }
    }
}

// Values of keys behind the run's end (or on a page that is none of the pool's) are whatever memory holds: zero them, since a zero
// probability does not silence an infinity or a NaN.
template <int D, bool SMALL>
__device__ __forceinline__ void attn_clear_v(AttnV<D>& vf, const AttnTile<SMALL>& t, int32_t key0, int32_t run_len) {
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const bool ok = key0 + 16 * u + 8 * (r / 4) + 4 * half + r % 4 < run_len && ((t.known >> u) & 1u);
#pragma unroll
            for (int k = 0; k < D / 64; ++k) vf.w[u][r][k] = ok ? vf.w[u][r][k] : 0u;
        }
}

// Where the finished rows of a segment go that are not the whole answer (kOwnKeys, kPrefix).
__device__ __forceinline__ float* attn_whole_row(const AttentionArgs& a, uint32_t token, uint32_t head, uint32_t dim) {
    return a.rows + ((size_t)token * a.heads + head) * (dim + 4);
}

template <int D>
__device__ __forceinline__ void attn_clear(AttnAcc<D>& acc) {
    acc.m = -__builtin_inff();
    acc.l = 0.0f;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc.o[j][i] = 0.0f;
}

// LDS of the streaming kernel: partial outputs of the four waves, their maxima and sums
template <int D>
struct AttnShared {
    float o[4][32][D + 4];      // (four floats of padding: a half wave's 16-byte stores cover all banks)
    float m[4][32], l[4][32];
};

// Few rows a sequence (decoding, drafted tokens): bound by the cache's bytes.  A workgroup takes a run of units and works
// through the segments it crosses, its four waves on every fourth key tile, straight from the cache: a lane takes dim / 32 neighbouring
// values of 16 keys of V, and pairs of keys are put side by side with one v_perm per operand dword.  At a segment's end the
// waves' results meet in LDS.  A segment that lies whole in one workgroup is finished there; the parts of the others go to the workspace
// (two slots a workgroup are enough: only its first and last segment can be shared) and are joined by the second launch, in a
// fixed order.
template <class ActT, int D, bool SMALL>
__device__ __forceinline__ void attn_stream(const AttentionArgs& a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    AttnShared<D>& sh = *reinterpret_cast<AttnShared<D>*>(smem);
    constexpr uint32_t R = 32;
    const AttnWork work = find_work<kFirstUnit>(a, blockIdx.x);
    if (work.entry == ~0u) return;
    uint32_t unit = work.at, index = work.entry, base = work.base;
    const uint32_t unit_end = smelt_serving::attention_start(work.split, blockIdx.x + 1);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const AttnScale scale = attn_scale(a);
#pragma unroll 1
    while (unit < unit_end) {
        const AttentionEntry e = attn_entry(a, index);
        AttnSegment g;
        if (!attn_segment(a, e, base, unit, unit_end, g)) { base = g.begin; ++index; continue; }
        const uint32_t row0 = g.row_tile * R;
        const AttnRow row = attn_row(a, e, row0 + (lane & 31));
        AttnAcc<D> acc;
        attn_clear<D>(acc);
        uint4_t qf[D / 16];
        attn_load_q<ActT, D>(a, row, g.kv_head, qf);
#pragma unroll 1
        for (int run = 0; run < 2; ++run) {
            const AttnRun u = attn_run(a, e, run, row0, row);
            const int32_t tile0 = run ? (int32_t)e.front_tiles : 0, tiles = (u.len + 31) / 32;
            const AttnBounds b = attn_bounds(a, row, run ? (int32_t)e.prefix : 0, u.len);
            const int32_t* table = run ? a.page_table + (size_t)e.sequence * a.pages_per_sequence : a.prefix_table;
            int32_t t1 = (int32_t)g.last - tile0, tile = (int32_t)g.first - tile0;
            t1 = t1 > tiles ? tiles : t1;
            // (the segment's tiles are those that one of its rows sees: none in between is to be skipped)
            tile = (tile < 0 ? 0 : tile) + (int32_t)wave;
            if (tile >= t1) continue;
            // K of the next tile is under way while this one's probabilities and V are worked on, V while the scores are
            AttnTile<SMALL> at = attn_tile<SMALL, D>(a, table, g.kv_head, (uint32_t)u.len, (uint32_t)tile);
            uint4_t kf[D / 16];
            attn_load_k<D, SMALL>(a, at, kf);
#pragma unroll 1
            for (; tile < t1; tile += 4) {
                const int32_t key0 = tile * (int32_t)smelt_serving::kKeyTile;
                AttnV<D> vf;
                float16_t s;
                attn_load_v<D, SMALL>(a, at, vf);
                const AttnTile<SMALL> next = attn_tile<SMALL, D>(a, table, g.kv_head, (uint32_t)u.len, (uint32_t)(tile + 4 < t1 ? tile + 4 : tile));
                attn_scores<ActT, D, SMALL>(a, qf, kf, s);
                __builtin_amdgcn_sched_barrier(0);
                attn_load_k<D, SMALL>(a, next, kf);      // (once more the last tile's, from cache, at the end)
                __builtin_amdgcn_sched_barrier(0);
                const bool bad = at.known != 3u;
                if (bad || attn_masked(u, key0)) attn_hide(s, key0, b, at.known);
                attn_softmax<D, 1>(scale, acc, &s);
                if (bad || key0 + (int32_t)smelt_serving::kKeyTile > u.len) attn_clear_v<D, SMALL>(vf, at, key0, u.len);
                attn_values<ActT, D>(acc, s, vf);
                at = next;
            }
        }
        // the waves meet
        const float l = attn_halves_sum(acc.l);
        const uint32_t half = lane >> 5;
        if (lane < 32) { sh.m[wave][lane] = acc.m; sh.l[wave][lane] = l; }
        if (row.live) {
            constexpr int E = D / 32;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float* dst = &sh.o[wave][lane & 31][E * (8 * (i / 4) + 4 * half + i % 4)];
                if constexpr (E >= 4) {
#pragma unroll
                    for (int j = 0; j < E; j += 4) *reinterpret_cast<float4_t*>(dst + j) = float4_t{acc.o[j][i], acc.o[j + 1][i], acc.o[j + 2][i], acc.o[j + 3][i]};
                } else {
#pragma unroll
                    for (int j = 0; j < E; ++j) dst[j] = acc.o[j][i];
                }
            }
        }
        __syncthreads();
        const uint32_t rows_live = e.tokens * a.group - row0 < R ? e.tokens * a.group - row0 : R;
        float* piece = a.pieces + ((size_t)blockIdx.x * 2 + (g.first == g.tiles.lo ? 1 : 0)) * smelt_serving::piece_floats(R, D);
#pragma unroll 1
        for (uint32_t item = threadIdx.x; item < rows_live * (D / 4); item += blockDim.x) {
            const uint32_t r = item / (D / 4), d = (item % (D / 4)) * 4;
            float m = sh.m[0][r];
#pragma unroll
            for (int w = 1; w < 4; ++w) m = __builtin_fmaxf(m, sh.m[w][r]);
            float4_t y = {0, 0, 0, 0};
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = m == -__builtin_inff() ? 1.0f : attn_exp2((sh.m[w][r] - m) * scale.c);
                y += f * *reinterpret_cast<const float4_t*>(&sh.o[w][r][d]);
                sum += f * sh.l[w][r];
            }
            const uint32_t i = (row0 + r) / a.group, token = e.first_token + i, head = g.kv_head * a.group + (row0 + r) - i * a.group;
            if (!g.whole) {
                *reinterpret_cast<float4_t*>(piece + 2 * R + r * D + d) = y;
                if (d == 0) { piece[r] = m; piece[R + r] = sum; }
            } else if (a.part != smelt_serving::kWholeSequences) {
                float* dst = attn_whole_row(a, token, head, D);
                *reinterpret_cast<float4_t*>(dst + d) = y;
                if (d == 0) { dst[D] = m; dst[D + 1] = sum; }
            } else {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                *reinterpret_cast<uint2_t*>(a.out + ((size_t)token * a.heads + head) * D + d) = uint2_t{attn_pack2<ActT>(y.x * inv, y.y * inv), attn_pack2<ActT>(y.z * inv, y.w * inv)};
            }
        }
        __syncthreads();
        unit += g.last - g.first;
    }
}

// Many rows (prompts, the prefix against a batch): bound by the matrix cores.  A workgroup's WAVES waves hold 32 rows each and walk
// the key tiles together: a stage of NS tiles is read once from the cache into registers while the stage before it is
// worked on, and put down in LDS (two stages, one barrier a stage), from where every wave takes it: K in operand order, V through the
// transposing LDS read (16 lanes take 4 keys x 16 values and get one value of 4 keys each), its 16-byte pieces placed so that the
// four keys of such a read lie on different banks.  Heads of up to 128 run two waves a SIMD, one's softmax under the other's
// products; heads of 256 need the whole register file for one.
typedef short attn_short4_t __attribute__((ext_vector_type(4)));
template <int D, int NS>
struct AttnTilesShared { uint16_t k[2][NS][32 * D], v[2][NS][32 * D]; };

// where 16-byte piece c of V row r lies in its row: bits 2 and 3 of the piece turned by the row
template <int D>
__device__ __forceinline__ uint32_t attn_v_turn(uint32_t row) { return D == 64 ? (row >> 1) & 1u : row & 3u; }

template <class ActT, int D, int WAVES, int NS, bool SMALL>
__device__ __forceinline__ void attn_tiles(const AttentionArgs& a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    AttnTilesShared<D, NS>& sh = *reinterpret_cast<AttnTilesShared<D, NS>*>(smem);
    constexpr uint32_t R = 32 * WAVES, T = 64 * WAVES;
    constexpr int P = 8 * D / T;                         // 16-byte pieces of a key tile (K, then V) that a thread stages
    const AttnWork work = find_work<kFirstUnit>(a, blockIdx.x);
    if (work.entry == ~0u) return;
    uint32_t unit = work.at, index = work.entry, base = work.base;
    const uint32_t unit_end = work.split.whole ? unit + 1 : smelt_serving::attention_start(work.split, blockIdx.x + 1);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave, half = lane >> 5;
    const AttnScale scale = attn_scale(a);
    // the lane's share of a transposing read: key row and 8-byte piece; the pieces of 32 values further on are turned by the row
    const uint32_t v_row = 4 * half + (lane & 15) / 4, v_turn = attn_v_turn<D>(v_row);
    const uint32_t v_lane = v_row * 2 * D + ((lane & 31) / 16) * 32 + (lane & 3) * 8;
#pragma unroll 1
    while (unit < unit_end) {
        const AttentionEntry e = attn_entry(a, index);
        AttnSegment g;
        if (work.split.whole) attn_whole_segment(a, e, unit - base, g);
        else if (!attn_segment(a, e, base, unit, unit_end, g)) { base = g.begin; ++index; continue; }
        const uint32_t row0 = g.row_tile * R + wave * 32;
        const AttnRow row = attn_row(a, e, row0 + (lane & 31));
        AttnAcc<D> acc;
        attn_clear<D>(acc);
        uint4_t qf[D / 16];
        attn_load_q<ActT, D>(a, row, g.kv_head, qf);
        const AttnRun front = attn_run(a, e, 0, row0, row), own = attn_run(a, e, 1, row0, row);
        const AttnBounds front_b = attn_bounds(a, row, 0, front.len), own_b = attn_bounds(a, row, (int32_t)e.prefix, own.len);
        const int32_t* own_table = a.page_table + (size_t)(e.sequence < 0 ? 0 : e.sequence) * a.pages_per_sequence;

        uint4_t stage[NS][P];
        uint32_t known_next = 0;                          // two bits a tile: its pages are the pool's
        auto fetch = [&](uint32_t first) {
            known_next = 0;
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                const uint32_t ct = first + n;
                const bool some = ct < g.last && ct < e.tiles, run = ct >= e.front_tiles;
                if (!some) {
#pragma unroll
                    for (int p = 0; p < P; ++p) stage[n][p] = uint4_t{0, 0, 0, 0};
                    continue;
                }
                const uint32_t tile = ct - (run ? e.front_tiles : 0u), len = run ? e.own : e.front;
                const AttnTile<SMALL> at = attn_tile<SMALL, D>(a, run ? own_table : a.prefix_table, g.kv_head, len, tile);
                known_next |= at.known << (2 * n);
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const uint32_t piece = p * T + threadIdx.x;
                    if (piece < 4 * D) {                                                                    // K: [dim / 8][key][8]
                        const uint32_t chunk = piece / 32, key = piece % 32;
                        const size_t kb = SMALL && key >= 16 ? at.base[SMALL ? 1 : 0] : at.base[0];
                        stage[n][p] = *reinterpret_cast<const uint4_t*>(a.k_cache + kb + (((chunk << a.page_shift) + (SMALL ? key & 15 : at.off + key)) << 3));
                    } else {                                                                                // V: [key][dim]
                        const uint32_t key = (piece - 4 * D) / (D / 8), col = (piece - 4 * D) % (D / 8);
                        const size_t vb = SMALL && key >= 16 ? at.base[SMALL ? 1 : 0] : at.base[0];
                        const uint4_t v = *reinterpret_cast<const uint4_t*>(a.v_cache + vb + (SMALL ? key & 15 : at.off + key) * D + col * 8);
                        // (values behind the run's end or outside the pool are whatever memory holds)
                        const bool ok = tile * 32 + key < len && ((at.known >> (key / 16)) & 1u);
                        stage[n][p] = ok ? v : uint4_t{0, 0, 0, 0};
                    }
                }
            }
        };
        auto put = [&](int buffer) {
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const uint32_t piece = p * T + threadIdx.x;
                    if (piece < 4 * D) reinterpret_cast<uint4_t*>(sh.k[buffer][n])[piece] = stage[n][p];
                    else {
                        const uint32_t key = (piece - 4 * D) / (D / 8), col = (piece - 4 * D) % (D / 8);
                        reinterpret_cast<uint4_t*>(sh.v[buffer][n])[key * (D / 8) + (col ^ (4 * attn_v_turn<D>(key)))] = stage[n][p];
                    }
                }
        };
        fetch(g.first);
        put(0);
        uint32_t known = known_next;
        __syncthreads();
        int buffer = 0;
#pragma unroll 1
        for (uint32_t first = g.first; first < g.last; first += NS, buffer ^= 1) {
            const bool more = first + NS < g.last;
            if (more) fetch(first + NS);
            // what the wave's rows see of the stage
            bool seen = false, edge[NS];
            int32_t key0[NS];
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                const uint32_t ct = first + n;
                const bool some = ct < g.last && ct < e.tiles, run = ct >= e.front_tiles;
                const AttnRun& u = run ? own : front;
                key0[n] = (int32_t)(ct - (run ? e.front_tiles : 0u)) * (int32_t)smelt_serving::kKeyTile;
                seen = seen || (some && attn_seen(u, key0[n]));
                edge[n] = !some || ((known >> (2 * n)) & 3u) != 3u || attn_masked(u, key0[n]);
            }
            if (seen) {
                float16_t s[NS];
#pragma unroll
                for (int n = 0; n < NS; ++n) {
                    const uint4_t* kl = reinterpret_cast<const uint4_t*>(sh.k[buffer][n]) + lane;
                    s[n] = attn_mfma<ActT>(kl[0], qf[0], float16_t{});
#pragma unroll
                    for (int d = 1; d < D / 16; ++d) s[n] = attn_mfma<ActT>(kl[d * 64], qf[d], s[n]);
                }
#pragma unroll
                for (int n = 0; n < NS; ++n)
                    if (edge[n]) attn_hide(s[n], key0[n], first + n >= e.front_tiles ? own_b : front_b, first + n < g.last && first + n < e.tiles ? known >> (2 * n) : 0u);
                attn_softmax<D, NS>(scale, acc, s);
#pragma unroll
                for (int n = 0; n < NS; ++n) {
                    const char* vl = reinterpret_cast<const char*>(sh.v[buffer][n]) + v_lane;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint4_t pf = attn_pack<ActT>(s[n], u);
#pragma unroll
                        for (int j = 0; j < D / 32; ++j) {
                            const char* at = vl + 16 * u * 2 * D + ((j & ~3) | ((j & 3) ^ v_turn)) * 64;
                            typedef __attribute__((address_space(3))) attn_short4_t* lds_ptr;
                            const uint2_t lo = __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)at));
                            const uint2_t hi = __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at + 8 * 2 * D)));
                            acc.o[j] = attn_mfma<ActT>(uint4_t{lo.x, lo.y, hi.x, hi.y}, pf, acc.o[j]);
                        }
                    }
                }
            }
            if (more) put(buffer ^ 1);
            known = known_next;
            __syncthreads();
        }
        // a lane holds its row's values 32 j + 8 (i / 4) + 4 half + i % 4
        float* piece = a.pieces + ((size_t)blockIdx.x * 2 + (g.first == g.tiles.lo ? 1 : 0)) * smelt_serving::piece_floats(R, D);
        const float l = attn_halves_sum(acc.l);
        if (row.live) {
            const uint32_t r = wave * 32 + (lane & 31), head = g.kv_head * a.group + row.head;
            if (g.whole && a.part == smelt_serving::kWholeSequences) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                uint16_t* out = a.out + ((size_t)row.token * a.heads + head) * D + 4 * half;
#pragma unroll
                for (int j = 0; j < D / 32; ++j)
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        *reinterpret_cast<uint2_t*>(out + 32 * j + 2 * i) = uint2_t{attn_pack2<ActT>(acc.o[j][i] * inv, acc.o[j][i + 1] * inv),
                                                                                   attn_pack2<ActT>(acc.o[j][i + 2] * inv, acc.o[j][i + 3] * inv)};
            } else {
                float* dst = g.whole ? attn_whole_row(a, row.token, head, D) : piece + 2 * R + r * D;
                if (half == 0) {
                    if (g.whole) { dst[D] = acc.m; dst[D + 1] = l; }
                    else { piece[r] = acc.m; piece[R + r] = l; }
                }
#pragma unroll
                for (int j = 0; j < D / 32; ++j)
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        *reinterpret_cast<float4_t*>(dst + 4 * half + 32 * j + 2 * i) = float4_t{acc.o[j][i], acc.o[j][i + 1], acc.o[j][i + 2], acc.o[j][i + 3]};
            }
        }
        unit += work.split.whole ? 1 : g.last - g.first;
    }
}

// Joins what the first launches left.
struct AttnJoin { float m, l; float4_t y; };
__device__ __forceinline__ void attn_join(AttnJoin& j, float m, float l, float4_t y, float c) {
    const float top = __builtin_fmaxf(j.m, m);
    const float f = top == -__builtin_inff() ? 1.0f : attn_exp2((j.m - top) * c), g = top == -__builtin_inff() ? 1.0f : attn_exp2((m - top) * c);
    j.y = f * j.y + g * y;
    j.l = f * j.l + g * l;
    j.m = top;
}
// row r of the segment's parts that workgroups w0 .. w1 left
template <int D>
__device__ __forceinline__ void attn_join_pieces(AttnJoin& j, const AttentionArgs& a, const AttentionSplit& split, uint32_t begin, uint32_t w0, uint32_t w1, uint32_t r, uint32_t d, float c) {
    constexpr uint32_t U = 8;      // parts whose loads are under way together
    for (uint32_t base = w0; base <= w1; base += U) {
        float m[U], l[U];
        float4_t y[U];
#pragma unroll
        for (uint32_t k = 0; k < U; ++k) {
            const uint32_t w = base + k <= w1 ? base + k : w1;
            const uint32_t slot = smelt_serving::attention_start(split, w) <= begin ? 1u : 0u;
            const float* piece = a.pieces + ((size_t)w * 2 + slot) * smelt_serving::piece_floats(a.row_tile, D);
            m[k] = piece[r];
            l[k] = piece[a.row_tile + r];
            y[k] = *reinterpret_cast<const float4_t*>(piece + 2 * a.row_tile + r * D + d);
        }
#pragma unroll
        for (uint32_t k = 0; k < U; ++k)
            if (base + k <= w1) attn_join(j, m[k], l[k], y[k], c);
    }
}
template <class ActT>
__device__ __forceinline__ void attn_finish(const AttnJoin& j, uint16_t* out) {
    const float inv = j.l == 0.0f ? 0.0f : 1.0f / j.l;
    uint2_t w;
    w.x = attn_pack2<ActT>(j.y.x * inv, j.y.y * inv);
    w.y = attn_pack2<ActT>(j.y.z * inv, j.y.w * inv);
    *reinterpret_cast<uint2_t*>(out) = w;
}

// kWholeSequences.  Grid: cuts between workgroups x slices of a segment's rows.  The first cut inside a segment stands for it.
template <class ActT, int D>
__device__ __forceinline__ void attn_combine(const AttentionArgs& a) {
    const AttnWork work = find_work<kCut>(a, blockIdx.x);
    if (work.entry == ~0u) return;
    const AttentionEntry e = attn_entry(a, work.entry);
    AttnSegment g;
    if (!attn_segment(a, e, work.base, work.at, ~0u, g)) return;
    const uint32_t end = g.begin + (g.tiles.hi - g.tiles.lo);
    if (g.begin == work.at || smelt_serving::attention_start(work.split, blockIdx.x) > g.begin) return;     // not inside a segment, or not the first
    const uint32_t w1 = smelt_serving::attention_owner(work.split, end - 1);
    const uint32_t row0 = g.row_tile * a.row_tile, left = e.tokens * a.group - row0, rows = left < a.row_tile ? left : a.row_tile;
#pragma unroll 1
    for (uint32_t item = blockIdx.y * blockDim.x + threadIdx.x; item < rows * (D / 4); item += gridDim.y * blockDim.x) {
        const uint32_t r = item / (D / 4), d = (item % (D / 4)) * 4;
        AttnJoin j{-__builtin_inff(), 0.0f, {0, 0, 0, 0}};
        attn_join_pieces<D>(j, a, work.split, g.begin, blockIdx.x, w1, r, d, a.scale_log2);
        const uint32_t i = (row0 + r) / a.group, token = e.first_token + i, head = g.kv_head * a.group + (row0 + r) - i * a.group;
        attn_finish<ActT>(j, a.out + ((size_t)token * a.heads + head) * D + d);
    }
}

// kPrefix and kOwnKeys.  Grid: tokens x kv heads: a row's two halves, each in parts or whole.
template <class ActT, int D>
__device__ __forceinline__ void attn_combine_shared(const smelt_serving::AttentionJoinArgs& both) {
    const uint32_t token = blockIdx.x, kv_head = blockIdx.y;
    AttnWork work[2];
    work[1] = find_work<kToken>(both.own, token);
    if (work[1].entry == ~0u) return;       // a row behind the last sequence
    work[0] = find_work<kToken>(both.front, token);
    const uint32_t group = both.own.group;
#pragma unroll 1
    for (uint32_t item = threadIdx.x; item < group * (D / 4); item += blockDim.x) {
        const uint32_t g = item / (D / 4), d = (item % (D / 4)) * 4, head = kv_head * group + g;
        AttnJoin j{-__builtin_inff(), 0.0f, {0, 0, 0, 0}};
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
            const AttentionArgs& x = k ? both.own : both.front;
            const AttnWork w = k ? work[1] : work[0];
            if (w.entry == ~0u) continue;       // no prefix
            const AttentionEntry e = attn_entry(x, w.entry);
            const uint32_t flat = (token - e.first_token) * group + g, row_tile = flat / x.row_tile, r = flat % x.row_tile;
            uint32_t begin = w.base;
            AttentionTiles s = smelt_serving::attention_tiles(x, e, 0);
#pragma unroll 1
            for (uint32_t t = 1; t <= row_tile; ++t) { begin += (s.hi - s.lo) * x.kv_heads; s = smelt_serving::attention_tiles(x, e, t); }
            begin += (s.hi - s.lo) * kv_head;
            uint32_t w0 = 0, w1 = 0;
            if (!w.split.whole) { w0 = smelt_serving::attention_owner(w.split, begin); w1 = smelt_serving::attention_owner(w.split, begin + (s.hi - s.lo) - 1); }
            if (w0 == w1) {
                const float* row = attn_whole_row(x, token, head, D);
                attn_join(j, row[D], row[D + 1], *reinterpret_cast<const float4_t*>(row + d), x.scale_log2);
            } else {
                attn_join_pieces<D>(j, x, w.split, begin, w0, w1, r, d, x.scale_log2);
            }
        }
        attn_finish<ActT>(j, both.own.out + ((size_t)token * both.own.heads + head) * D + d);
    }
}

}  // namespace smelt

// (one wave a SIMD where accumulators, q and the tiles in flight take the whole register file)
#define SMELT_ATTENTION_KERNELS(T, ACT, D, STREAM_WAVES, WAVES, NS, TILE_WAVES)                                                                                                   \
    extern "C" __global__ __launch_bounds__(256, STREAM_WAVES) void smelt_attention_stream_d##D##_##T(smelt_serving::AttentionArgs a) { smelt::attn_stream<ACT, D, false>(a); }          \
    extern "C" __global__ __launch_bounds__(256, STREAM_WAVES) void smelt_attention_stream_d##D##_p16_##T(smelt_serving::AttentionArgs a) { smelt::attn_stream<ACT, D, true>(a); }       \
    extern "C" __global__ __launch_bounds__(64 * WAVES, TILE_WAVES) void smelt_attention_tiles_d##D##_##T(smelt_serving::AttentionArgs a) { smelt::attn_tiles<ACT, D, WAVES, NS, false>(a); }   \
    extern "C" __global__ __launch_bounds__(64 * WAVES, TILE_WAVES) void smelt_attention_tiles_d##D##_p16_##T(smelt_serving::AttentionArgs a) { smelt::attn_tiles<ACT, D, WAVES, NS, true>(a); } \
    extern "C" __global__ __launch_bounds__(256) void smelt_attention_join_d##D##_##T(smelt_serving::AttentionArgs a) { smelt::attn_combine<ACT, D>(a); }                              \
    extern "C" __global__ __launch_bounds__(256) void smelt_attention_join_shared_d##D##_##T(smelt_serving::AttentionJoinArgs a) { smelt::attn_combine_shared<ACT, D>(a); }
