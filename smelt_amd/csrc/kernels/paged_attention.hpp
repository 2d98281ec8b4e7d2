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

// Where a workgroup begins.
struct AttnWork {
    AttentionSplit split;    // of the whole launch
    uint32_t entry;          // where its first unit (its segment) lies, ~0: nowhere
    uint32_t base;           // units (segments where each workgroup takes one) before that entry
    uint32_t at;             // the unit (segment)
    uint32_t parts;          // kPrefix: of each segment
    smelt_serving::AttentionJob job;
};

// Each wave looks for itself (no barrier), an entry a lane: once through the entries for their total, then for the wanted one.
__device__ __forceinline__ AttnWork find_work(const AttentionArgs& a, uint32_t group) {
    const uint32_t entries = smelt_serving::attention_entries(a), lane = threadIdx.x % kWave;
    AttnWork w;
    w.entry = ~0u;
    w.base = w.at = w.parts = 0;
    w.split = AttentionSplit{0, 0, 0, 0, false};
    w.job = smelt_serving::AttentionJob{0, 0, 0, false};
    if (a.part == smelt_serving::kPrefix) {
        const AttentionEntry e = attn_entry(a, 0);
        w.parts = smelt_serving::attention_parts(a, e);
        w.job = smelt_serving::attention_job(a, e, w.parts, group);
        if (w.job.some) w.entry = 0;
        return w;
    }
    uint32_t mine[2] = {0, 0}, before[2] = {0, 0}, all[2] = {0, 0};      // units and segments: the lane's entry, the entries before it in the round, the round's
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        uint32_t run[2] = {0, 0};
#pragma unroll 1
        for (uint32_t base = 0; base < entries; base += kWave) {
            const uint32_t index = base + lane;
            if (pass == 0 || entries > (uint32_t)kWave) {
                mine[0] = mine[1] = 0;
                if (index < entries) {
                    const AttentionEntry e = smelt_serving::attention_entry(a, index);
                    mine[0] = smelt_serving::attention_units(a, e);
                    mine[1] = smelt_serving::attention_segments(a, e);
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
                const unsigned long long who = __ballot(w.at >= first && w.at - first < mine[k]);
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
        if (group >= w.split.groups) return w;
        w.at = w.split.whole ? group : smelt_serving::attention_start(w.split, group);
    }
    return w;
}

// A segment and the part of its key tiles that a workgroup takes.
struct AttnSegment {
    uint32_t kv_head, row_tile;
    AttentionTiles tiles;        // the segment's
    uint32_t first, last;        // the workgroup's part of them (none when its run ends within the segment's lead)
    bool whole;
    uint32_t begin;              // the unit of the segment's first key tile
    uint32_t units;              // of the workgroup's run that lie in the segment
    uint32_t slot;               // of the part
};
// the segment that holds unit `unit` of entry e, whose units start at `base`; false (and g.begin behind them) when the entry has fewer
__device__ __forceinline__ bool attn_segment(const AttentionArgs& a, const AttentionEntry& e, uint32_t base, uint32_t unit, uint32_t unit_end, AttnSegment& g) {
    uint32_t rel = unit - base;
    g.begin = base;
#pragma unroll 1
    for (g.row_tile = 0; g.row_tile < e.row_tiles; ++g.row_tile) {
        g.tiles = smelt_serving::attention_tiles(a, e, g.row_tile);
        const uint32_t each = g.tiles.hi - g.tiles.lo + a.lead, size = each * a.kv_heads;
        if (rel >= size) { rel -= size; g.begin += size; continue; }
        g.kv_head = rel / each;
        const uint32_t done = rel - g.kv_head * each, left = each - done;
        g.begin += g.kv_head * each + a.lead;
        g.units = left < unit_end - unit ? left : unit_end - unit;
        g.first = g.tiles.lo + (done > a.lead ? done - a.lead : 0u);
        g.last = g.tiles.lo + (done + g.units > a.lead ? done + g.units - a.lead : 0u);
        g.whole = g.first == g.tiles.lo && g.last == g.tiles.hi;
        g.slot = 2 * blockIdx.x + (g.first == g.tiles.lo ? 1u : 0u);
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
    g.begin = g.slot = 0;
    g.units = 1;
}
// the prefix's
__device__ __forceinline__ void attn_part(const AttentionArgs& a, const AttentionEntry& e, const AttnWork& work, AttnSegment& g) {
    const smelt_serving::AttentionJob& j = work.job;
    const uint32_t parts = work.parts;
    g.row_tile = j.row_tile;
    g.kv_head = j.kv_head;
    g.tiles = AttentionTiles{0, e.front_tiles};
    const uint32_t each = e.front_tiles / parts, longer = e.front_tiles - each * parts;
    g.first = j.part * each + (j.part < longer ? j.part : longer);
    g.last = g.first + each + (j.part < longer ? 1u : 0u);
    g.whole = parts == 1;
    g.begin = 0;
    g.units = 1;
    g.slot = (j.row_tile * a.kv_heads + j.kv_head) * parts + j.part;
}

// where the part of a segment goes that is not the whole of it
__device__ __forceinline__ float* attn_piece(const AttentionArgs& a, const AttnSegment& g, uint32_t dim) {
    return a.pieces + (size_t)g.slot * smelt_serving::piece_floats(a.row_tile, dim);
}
// the last workgroup that has a part of a segment
__device__ __forceinline__ uint32_t attn_last(const AttentionSplit& split, const AttnSegment& g) {
    return smelt_serving::attention_owner(split, g.begin + (g.tiles.hi - g.tiles.lo) - 1);
}
// kWholeSequences: the workgroup's note for the join (every workgroup leaves one: none at its start, overwritten by the same thread)
__device__ __forceinline__ void attn_note_cut(const AttentionArgs& a, const smelt_serving::AttentionCut& cut) {
    if (a.part == smelt_serving::kWholeSequences && blockIdx.x < a.workgroups && threadIdx.x == 0) a.cuts[blockIdx.x] = cut;
}
__device__ __forceinline__ smelt_serving::AttentionCut attn_cut(const AttentionArgs& a, const AttentionEntry& e, const AttentionSplit& split, const AttnSegment& g) {
    const uint32_t row0 = g.row_tile * a.row_tile, left = e.tokens * a.group - row0;
    return {attn_last(split, g), g.kv_head, e.first_token, row0, left < a.row_tile ? left : a.row_tile, {0, 0, 0}};
}
// kOwnKeys, kPrefix: ends a row (r within its tile) of a segment that begins here
__device__ __forceinline__ void attn_end_row(float* end, const AttentionArgs& a, const AttnWork& work, const AttnSegment& g, uint32_t r, float max, float sum) {
    const uint32_t parts = g.whole ? 1u : (work.parts ? work.parts : attn_last(work.split, g) - blockIdx.x + 1u);
    *reinterpret_cast<smelt_serving::AttentionRowEnd*>(end) = smelt_serving::AttentionRowEnd{max, sum, g.slot, parts << 8 | r};
}

// The sequence of a lane's token row: offsets is ascending, tokens before offsets[sequences] belong to one.  The wave takes 64 of the
// offsets at once (the steps of a search in memory are a load's latency each, six or more of them).
__device__ __forceinline__ uint32_t sequence_of(const AttentionArgs& a, uint32_t token) {
    const uint32_t step = (a.sequences + kWave - 1) / kWave, mine = (threadIdx.x % kWave) * step;
    const uint32_t sample = mine < a.sequences ? smelt_serving::clamp_count(a.offsets[mine], a.tokens) : ~0u;
    uint32_t lo = 0;
#pragma unroll
    for (uint32_t bit = kWave / 2; bit; bit /= 2) lo = (uint32_t)__shfl((int)sample, (int)(lo + bit)) <= token ? lo + bit : lo;
    lo *= step;
    uint32_t hi = lo + step < a.sequences ? lo + step : a.sequences;   // offsets[lo] <= token < offsets[hi]
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

// Keys of one run that some of `count` rows from row0 on sees, and that all of them see (b: the lane's own).
struct AttnRun { int32_t lo, hi, all_lo, all_hi; };
__device__ __forceinline__ AttnRun attn_run(const AttentionArgs& a, const AttentionEntry& e, int run, uint32_t row0, uint32_t count, const AttnBounds* b, int bounds) {
    const int32_t len = (int32_t)(run ? e.own : e.front), base = run ? (int32_t)e.prefix : 0;
    AttnRun u{0, len, 0, len};
    if (e.sequence < 0) {        // rows of many sequences: they mostly see all of it
        bool all = true;
        for (int t = 0; t < bounds; ++t) all = all && b[t].lo == 0 && b[t].hi == len;
        if (!__all(all)) u.all_hi = 0;
    } else if (row0 < e.tokens * a.group) {
        const AttentionSpan s = smelt_serving::attention_span(a, e, row0, count);
        const int32_t hi = s.hi - base, all_hi = s.all_hi - base;
        u.lo = s.lo - base > 0 ? s.lo - base : 0;
        u.all_lo = s.all_lo - base > 0 ? s.all_lo - base : 0;
        u.hi = hi < len ? hi : len;
        u.all_hi = all_hi < len ? all_hi : len;
    } else {
        u.hi = 0;                // no rows here
    }
    return u;
}
__device__ __forceinline__ bool attn_masked(const AttnRun& u, int32_t key0) { return key0 + (int32_t)smelt_serving::kKeyTile > u.all_hi || key0 < u.all_lo; }

// One wave's state: 32 rows.
template <int D>
struct AttnAcc {
    float16_t o[D / 32];     // o[j][i]: value (D / 32) * (8 (i / 4) + 4 (lane / 32) + i % 4) + j of the lane's row
    float m, l;              // running maximum of q.k and this half's sum
};

// N pieces of eight values of a q row, `step` apart; rows that are none (they point at a row that is one) are zero
template <int N>
__device__ __forceinline__ void attn_load_q(const AttentionArgs& a, const AttnRow& r, const uint16_t* q, uint32_t step, uint4_t* qf) {
    if ((reinterpret_cast<uintptr_t>(a.q) & 15u) == 0 && (a.q_stride & 7u) == 0) {
#pragma unroll
        for (int k = 0; k < N; ++k) qf[k] = *reinterpret_cast<const uint4_t*>(q + k * step);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (uint32_t)q[k * step + 2 * i] | ((uint32_t)q[k * step + 2 * i + 1] << 16);
            qf[k] = uint4_t{w[0], w[1], w[2], w[3]};
        }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) qf[k] = r.live ? qf[k] ^ a.flip_q : uint4_t{0, 0, 0, 0};
}

// Address of one key tile, in halves of 16 keys (a page holds one at least): where each lies and whether its page is one of the pool's.
struct AttnTile {
    size_t page[2];                  // element offset of the page's head
    uint32_t off[2];                 // first key within the page
    uint32_t known;                  // bits 0 and 1
};
template <int D>
__device__ __forceinline__ AttnTile attn_tile(const AttentionArgs& a, const int32_t* table, uint32_t kv_head, uint32_t run_len, uint32_t tile) {
    AttnTile t;
    const uint32_t last_page = run_len ? (run_len - 1) >> a.page_shift : 0u;
    t.known = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint32_t key = tile * smelt_serving::kKeyTile + 16 * k;
        uint32_t index = key >> a.page_shift;
        if (index > last_page) index = last_page;      // behind the run: masked by its length
        const uint32_t page = (uint32_t)as_scalar(table)[__builtin_amdgcn_readfirstlane(index)];
        const bool known = page < a.pages;
        t.known |= known ? 1u << k : 0u;
        t.page[k] = (((size_t)(known ? page : 0u) * a.kv_heads + kv_head) * D) << a.page_shift;
        t.off[k] = key & ((1u << a.page_shift) - 1u);
    }
    return t;
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

// The outputs stay in the matrix instructions' own registers on both ways around the rare rescaling (the compiler would copy all of them
// to vector registers in front of it and back, for every tile).
template <int D>
__device__ __forceinline__ void attn_keep(AttnAcc<D>& acc) {
    if constexpr (D < 256) return;       // (two waves a SIMD: they have no others)
#pragma unroll
    for (int j = 0; j < D / 32; ++j) asm volatile("" : "+a"(acc.o[j]));
}

template <int D, int NS>
__device__ __forceinline__ void attn_softmax(const AttnScale& c, AttnAcc<D>& acc, float16_t* s) {
    float top = s[0][0];
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int i = 0; i < 16; i += 2) top = __builtin_fmaxf(__builtin_fmaxf(top, s[n][i]), s[n][i + 1]);
    top = attn_halves_max(top);
    attn_keep(acc);
    if (__any(top > acc.m + c.slack)) {      // also the first finite score: the maximum starts at -inf
        const float m = __builtin_fmaxf(acc.m, top);
        const float f = m == -__builtin_inff() ? 1.0f : attn_exp2((acc.m - m) * c.c);
        acc.l *= f;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc.o[j][i] *= f;
        acc.m = m;
        attn_keep(acc);
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

// Values are multiplied with a zero probability where one of a tile's rows does not see a key and another does, and a zero does not silence
// an infinity or a NaN.  Rows that came out as NaN are therefore formed once more at a segment's end, over the keys they see (maxima and
// sums are right: hidden scores are taken out before those).  That is rare and stands outside of the key loops: a search for such values
// within them cost a fifth of their time.  Two kinds of rows are left as they are, since NaN is their answer.  A row whose sum is a NaN has
// seen a score that is one (a NaN in q or in a key, or an infinite score).  And where every value that is not finite is a NaN that all of the
// tile's rows see, it is theirs.  One sequence with a NaN among many: 64 that decode 84 us for a score, as without, and 120 for a value
// (formed again 13000); four with 50000 to 65536 keys 182 and 390 (71000); two prompt chunks 150 and 385 (82000), and 14600 for a value
// in the last key, which the tile's rows before it do not see; drafted tokens 65 and 86, and 390 for one in the last key (11000).

// The keys of run 0 (prefix) or 1 (own) that a workgroup's part of a segment has, and their pages.
struct AttnKeys { uint32_t first, last, len; const int32_t* table; };
__device__ __forceinline__ AttnKeys attn_keys(const AttentionArgs& a, const AttentionEntry& e, const AttnSegment& g, int run) {
    const uint32_t len = run ? e.own : e.front, tile0 = run ? e.front_tiles : 0u;
    const uint32_t first = (g.first > tile0 ? g.first - tile0 : 0u) * smelt_serving::kKeyTile, last = (g.last > tile0 ? g.last - tile0 : 0u) * smelt_serving::kKeyTile;
    return AttnKeys{first, last < len ? last : len, len, run ? a.page_table + (size_t)e.sequence * a.pages_per_sequence : a.prefix_table};
}

// the lane, for code that seldom runs: nothing of it is worked out ahead and held in registers through the key loops
__device__ __forceinline__ uint32_t attn_cold_lane() {
    uint32_t lane = threadIdx.x % kWave;
    asm volatile("" : "+v"(lane));
    return lane;
}

// Whether rows that came out as NaN are to be formed again: among the part's values one is not finite that a row of the tile does not see, or
// one is an infinity (which a probability that rounds to zero makes a NaN).  seen(run) tells what all of the rows see.  By a wave, 16 bytes a
// lane and eight loads under way.
template <class ActT, int D, class Seen>
__device__ __forceinline__ bool attn_again(const AttentionArgs& a, const AttentionEntry& e, const AttnSegment& g, Seen seen) {
    constexpr uint32_t U = 8, kKeys = 512 / D, kInfinity = ActT::kIsF16 ? 0x7C00u : 0x7F80u;
    const uint32_t lane = attn_cold_lane();
    bool found = false;
#pragma unroll 1
    for (int run = 0; run < 2; ++run) {
        const AttnKeys part = attn_keys(a, e, g, run);
        const AttnRun u = seen(run);
#pragma unroll 1
        for (uint32_t base = part.first; base < part.last; base += kKeys * U) {
            uint32_t page[U];
            uint4_t v[U];
#pragma unroll
            for (uint32_t k = 0; k < U; ++k) {
                const uint32_t key = base + k * kKeys + lane / (D / 8);
                page[k] = (uint32_t)part.table[(key < part.last ? key : part.last - 1) >> a.page_shift];
            }
#pragma unroll
            for (uint32_t k = 0; k < U; ++k) {
                const uint32_t key = base + k * kKeys + lane / (D / 8), off = (key < part.last ? key : part.last - 1) & ((1u << a.page_shift) - 1u);
                const size_t at = (((size_t)(page[k] < a.pages ? page[k] : 0u) * a.kv_heads + g.kv_head) * D) << a.page_shift;
                v[k] = *reinterpret_cast<const uint4_t*>(a.v_cache + at + off * D + (lane % (D / 8)) * 8);
            }
#pragma unroll
            for (uint32_t k = 0; k < U; ++k) {
                const int32_t key = (int32_t)(base + k * kKeys + lane / (D / 8));
                const bool hidden = key < u.all_lo || key >= u.all_hi;
                bool odd = false;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t size = (v[k][i / 2] >> (16 * (i & 1))) & 0x7FFFu;
                    odd = odd || size == kInfinity || (hidden && size > kInfinity);
                }
                found = found || (odd && key < (int32_t)part.last && page[k] < a.pages);
            }
        }
    }
    return __any(found);
}

// Forms row r of the tile (a token's head, at its position, of the given maximum and sum) over the part's keys that it sees and puts it where
// the segment's rows go, by a wave: a key a lane for the scores, D / 64 values a lane for the output.
template <class ActT, int D>
__device__ __forceinline__ void attn_form_row(const AttentionArgs& a, const AttentionEntry& e, const AttnSegment& g, uint32_t r, uint32_t token, uint32_t head, int32_t position,
                                              float m, float sum, float c) {
    constexpr uint32_t E = D / 64, U = 8;
    const uint32_t lane = attn_cold_lane(), mask = (1u << a.page_shift) - 1u;
    const float shift = m == -__builtin_inff() ? 0.0f : -m * c;
    const uint16_t* row = a.q + (size_t)token * a.q_stride + (size_t)head * D + lane * E;
    int q[E];
    float y[E];
#pragma unroll
    for (uint32_t n = 0; n < E; ++n) { q[n] = __builtin_bit_cast(int, ActT::widen((uint16_t)(row[n] ^ (uint16_t)a.flip_q))); y[n] = 0.0f; }
#pragma unroll 1
    for (int run = 0; run < 2; ++run) {
        const AttnKeys part = attn_keys(a, e, g, run);
        const AttnBounds b = attn_bounds(a, AttnRow{true, token, 0, position}, run ? (int32_t)e.prefix : 0, (int32_t)part.len);
        const uint32_t first = __builtin_amdgcn_readfirstlane((int32_t)part.first > b.lo ? part.first : (uint32_t)b.lo);
        const int32_t last = __builtin_amdgcn_readfirstlane((int32_t)part.last < b.hi ? (int32_t)part.last : b.hi);
#pragma unroll 1
        for (uint32_t base = first; (int32_t)base < last; base += kWave) {
            const uint32_t key = (int32_t)(base + lane) < last ? base + lane : (uint32_t)last - 1, page = (uint32_t)part.table[key >> a.page_shift], off = key & mask;
            const bool seen = (int32_t)(base + lane) < last && page < a.pages;
            const size_t at = (((size_t)(page < a.pages ? page : 0u) * a.kv_heads + g.kv_head) * D) << a.page_shift, value = at + off * D;
            const uint16_t* k = a.k_cache + at + off * 8;
            float dot = 0.0f;
#pragma unroll 8
            for (uint32_t d = 0; d < D / 8; ++d) {
                const uint4_t x = *reinterpret_cast<const uint4_t*>(k + (d << (a.page_shift + 3)));
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i)
                    dot = __builtin_fmaf(__builtin_bit_cast(float, __builtin_amdgcn_readlane(q[i % E], d * (8 / E) + i / E)), ActT::widen((uint16_t)(x[i / 2] >> (16 * (i & 1)))), dot);
            }
            const int p = __builtin_bit_cast(int, attn_exp2(__builtin_fmaf(dot, c, shift)));
            const unsigned long long who = __ballot(seen);
#pragma unroll 1
            for (uint32_t n = 0; n < (uint32_t)kWave && (int32_t)(base + n) < last; n += U) {
                struct alignas(2 * E) Values { uint16_t x[E]; } v[U];
#pragma unroll
                for (uint32_t k2 = 0; k2 < U; ++k2) {
                    const uint64_t from = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(value >> 32), n + k2) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)value, n + k2);
                    v[k2] = *reinterpret_cast<const Values*>(a.v_cache + from + lane * E);
                }
#pragma unroll
                for (uint32_t k2 = 0; k2 < U; ++k2) {
                    const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(p, n + k2));
#pragma unroll
                    for (uint32_t i = 0; i < E; ++i) y[i] = (who >> (n + k2)) & 1u ? __builtin_fmaf(w, ActT::widen(v[k2].x[i]), y[i]) : y[i];
                }
            }
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const bool answer = g.whole && a.part == smelt_serving::kWholeSequences;
    float* dst = (g.whole ? attn_whole_row(a, token, head, D) : attn_piece(a, g, D) + 2 * a.row_tile + r * D) + lane * E;
#pragma unroll
    for (uint32_t n = 0; n < E; ++n) {
        if (answer) a.out[((size_t)token * a.heads + head) * D + lane * E + n] = ActT::narrow(y[n] * inv);
        else dst[n] = y[n];
    }
}
// maximum and sum over a lane's row of the streaming kernel: lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float attn_quarters_max(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return attn_halves_max(__builtin_fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])));
}
__device__ __forceinline__ float attn_quarters_sum(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return attn_halves_sum(__builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]));
}

template <class ActT>
__device__ __forceinline__ float4_t attn_mfma16(uint4_t a, uint4_t b, float4_t c) {
    if constexpr (ActT::kIsF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(attn_bf16x8_t, a), __builtin_bit_cast(attn_bf16x8_t, b), c, 0, 0, 0);
}

// LDS of the streaming kernel: partial outputs of the four waves, their maxima and sums
template <int D, int RT>
struct AttnShared {
    float o[4][16 * RT][D + 4];      // (four floats of padding: neighbouring rows' 16-byte stores lie on different banks)
    float m[4][16 * RT], l[4][16 * RT];
    int32_t position[16 * RT];
};

// Few rows a sequence (decoding, drafted tokens): bound by the cache's bytes.  Four sequences of 50000 to 65536 keys, heads of 256: 183 us
// with the join's 8 (947 MB, 5.2 TB/s, a copy reaches 5.1); the own keys of 64 sequences of 17 to 1024: 32 us in a run of launches
// (136 MB, 4.3 TB/s), 39 by themselves; one token behind 1000 keys: 9 us, of which 4 pass before its first key.  A workgroup takes a run of units and works
// through the segments it crosses, its four waves on every fourth key tile, straight from the cache.  Here the products are
// v_mfma_f32_16x16x32 (lane l: row l % 16, quarter l / 16), one or two tiles of 16 rows against each key tile: with one, heads of
// 256 leave room for two workgroups a compute unit, whose starts and ends hide behind each other.  V: a lane takes 8 neighbouring
// values (4 for heads of 64) of the 8 keys whose probabilities it holds, and pairs of keys are put side by side with one
// v_perm per operand dword.  At a segment's end the waves' results meet in LDS.  A segment that lies whole in one workgroup is
// finished there; the parts of the others go to the workspace (two slots a workgroup are enough: only its first and last segment can be
// shared) and are joined by the second launch, in a fixed order.
template <class ActT, int D, int RT>
__device__ __forceinline__ void attn_stream(const AttentionArgs& a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    AttnShared<D, RT>& sh = *reinterpret_cast<AttnShared<D, RT>*>(smem);
    constexpr uint32_t R = 16 * RT;
    constexpr int KS = D / 32, VE = D == 64 ? 4 : 8, VC = D == 256 ? 2 : 1, MT = D / 16;   // k steps of a score; values a lane takes of a V row, in VC pieces; tiles of 16 values
    const AttnWork work = find_work(a, blockIdx.x);
    attn_note_cut(a, {});
    if (work.entry == ~0u) return;
    uint32_t unit = work.at, index = work.entry, base = work.base;
    const uint32_t unit_end = work.parts ? unit + 1 : smelt_serving::attention_start(work.split, blockIdx.x + 1);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave, quarter = lane >> 4, col = lane & 15;
    const AttnScale scale = attn_scale(a);
#pragma unroll 1
    while (unit < unit_end) {
        const AttentionEntry e = attn_entry(a, index);
        AttnSegment g;
        if (work.parts) attn_part(a, e, work, g);
        else if (!attn_segment(a, e, base, unit, unit_end, g)) { base = g.begin; ++index; continue; }
        unit += g.units;
        if (g.first >= g.last) continue;                 // (only some of its lead)
        const uint32_t row0 = g.row_tile * R;
        AttnRow row[RT];
        float4_t o[RT][MT];
        float m[RT], l[RT];
        uint4_t qf[RT][KS];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            row[t] = attn_row(a, e, row0 + 16 * t + col);
            m[t] = -__builtin_inff();
            l[t] = 0.0f;
#pragma unroll
            for (int j = 0; j < MT; ++j) o[t][j] = float4_t{0, 0, 0, 0};
            const uint16_t* q = a.q + (size_t)row[t].token * a.q_stride + (size_t)(g.kv_head * a.group + row[t].head) * D + 8 * quarter;
            attn_load_q<KS>(a, row[t], q, 32, qf[t]);
        }
#pragma unroll 1
        for (int run = 0; run < 2; ++run) {
            const int32_t len = (int32_t)(run ? e.own : e.front), run_base = run ? (int32_t)e.prefix : 0;
            const int32_t tile0 = run ? (int32_t)e.front_tiles : 0, tiles = (len + 31) / 32;
            int32_t t1 = (int32_t)g.last - tile0, tile = (int32_t)g.first - tile0;
            t1 = t1 > tiles ? tiles : t1;
            // (the segment's tiles are those that one of its rows sees: none in between is to be skipped)
            tile = (tile < 0 ? 0 : tile) + (int32_t)wave;
            if (tile >= t1) continue;
            const int32_t* table = run ? a.page_table + (size_t)e.sequence * a.pages_per_sequence : a.prefix_table;
            AttnBounds b[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t) b[t] = attn_bounds(a, row[t], run_base, len);
            const AttnRun u = attn_run(a, e, run, row0, R, b, RT);
            AttnTile at = attn_tile<D>(a, table, g.kv_head, (uint32_t)len, (uint32_t)tile);
            uint4_t kf[2][KS];
            auto load_k = [&](const AttnTile& x) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint16_t* k = a.k_cache + x.page[h] + (((quarter << a.page_shift) + x.off[h] + col) << 3);
#pragma unroll
                    for (int s = 0; s < KS; ++s) kf[h][s] = *reinterpret_cast<const uint4_t*>(k + ((uint32_t)(4 * s) << (a.page_shift + 3)));
                }
            };
            load_k(at);
#pragma unroll 1
            for (; tile < t1; tile += 4) {
                // K of the next tile is under way while this one's probabilities and V are worked on, V while the scores are
                const int32_t key0 = tile * (int32_t)smelt_serving::kKeyTile;
                uint32_t vf[8][VC][VE / 2];
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const uint16_t* v = a.v_cache + at.page[r / 4] + (at.off[r / 4] + 4 * quarter + r % 4) * D + col * VE;
#pragma unroll
                    for (int c = 0; c < VC; ++c) {
                        if constexpr (VE == 8) { const uint4_t x = *reinterpret_cast<const uint4_t*>(v + 128 * c); vf[r][c][0] = x.x; vf[r][c][1] = x.y; vf[r][c][2] = x.z; vf[r][c][3] = x.w; }
                        else { const uint2_t x = *reinterpret_cast<const uint2_t*>(v); vf[r][c][0] = x.x; vf[r][c][1] = x.y; }
                    }
                }
                const AttnTile next = attn_tile<D>(a, table, g.kv_head, (uint32_t)len, (uint32_t)(tile + 4 < t1 ? tile + 4 : tile));
                float4_t s[RT][2];
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        s[t][h] = attn_mfma16<ActT>(kf[h][0], qf[t][0], float4_t{0, 0, 0, 0});
#pragma unroll
                        for (int k = 1; k < KS; ++k) s[t][h] = attn_mfma16<ActT>(kf[h][k], qf[t][k], s[t][h]);
                    }
                __builtin_amdgcn_sched_barrier(0);
                load_k(next);                            // (once more the last tile's, from cache, at the end)
                __builtin_amdgcn_sched_barrier(0);
                // Values of keys behind the run's end, or on a page that is none of the pool's, are whatever memory holds: zero them, since
                // a zero probability does not silence an infinity or a NaN.
                if (at.known != 3u || key0 + (int32_t)smelt_serving::kKeyTile > len) {
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const bool ok = key0 + 16 * (r / 4) + 4 * (int32_t)quarter + r % 4 < len && ((at.known >> (r / 4)) & 1u);
#pragma unroll
                        for (int c = 0; c < VC; ++c)
#pragma unroll
                            for (int k = 0; k < VE / 2; ++k) vf[r][c][k] = ok ? vf[r][c][k] : 0u;
                    }
                }
                const bool edge = at.known != 3u || attn_masked(u, key0);
                uint4_t pf[RT];
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    if (edge) {
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int32_t key = key0 + 16 * h + 4 * (int32_t)quarter + i;
                                const bool ok = key >= b[t].lo && key < b[t].hi && ((at.known >> h) & 1u);
                                s[t][h][i] = ok ? s[t][h][i] : -__builtin_inff();
                            }
                    }
                    float top = __builtin_fmaxf(s[t][0][0], s[t][1][0]);
#pragma unroll
                    for (int i = 1; i < 4; ++i) top = __builtin_fmaxf(__builtin_fmaxf(top, s[t][0][i]), s[t][1][i]);
                    top = attn_quarters_max(top);
                    if (__any(top > m[t] + scale.slack)) {      // also the first finite score: the maximum starts at -inf
                        const float to = __builtin_fmaxf(m[t], top);
                        const float f = to == -__builtin_inff() ? 1.0f : attn_exp2((m[t] - to) * scale.c);
                        l[t] *= f;
#pragma unroll
                        for (int j = 0; j < MT; ++j) o[t][j] *= f;
                        m[t] = to;
                    }
                    const float shift = m[t] == -__builtin_inff() ? 0.0f : -m[t] * scale.c;
                    float p[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) p[i] = attn_exp2(__builtin_fmaf(s[t][i / 4][i % 4], scale.c, shift));
                    l[t] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                    pf[t] = uint4_t{attn_pack2<ActT>(p[0], p[1]), attn_pack2<ActT>(p[2], p[3]), attn_pack2<ActT>(p[4], p[5]), attn_pack2<ActT>(p[6], p[7])};
                }
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    const int c = j / VE, x = (j % VE) / 2;
                    const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
                    uint4_t v;
                    v.x = __builtin_amdgcn_perm(vf[1][c][x], vf[0][c][x], sel);
                    v.y = __builtin_amdgcn_perm(vf[3][c][x], vf[2][c][x], sel);
                    v.z = __builtin_amdgcn_perm(vf[5][c][x], vf[4][c][x], sel);
                    v.w = __builtin_amdgcn_perm(vf[7][c][x], vf[6][c][x], sel);
#pragma unroll
                    for (int t = 0; t < RT; ++t) o[t][j] = attn_mfma16<ActT>(v, pf[t], o[t][j]);
                }
                at = next;
            }
        }
        // the waves meet: o[t][j][i] is value VE (4 quarter + i) + j % VE + 128 (j / VE) of the lane's row
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const float sum = attn_quarters_sum(l[t]);
            if (lane < 16) { sh.m[wave][16 * t + lane] = m[t]; sh.l[wave][16 * t + lane] = sum; sh.position[16 * t + lane] = row[t].position; }
            if (row[t].live) {
#pragma unroll
                for (int c = 0; c < VC; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float* dst = &sh.o[wave][16 * t + col][VE * (4 * quarter + i) + 128 * c];
#pragma unroll
                        for (int j = 0; j < VE; j += 4)
                            *reinterpret_cast<float4_t*>(dst + j) = float4_t{o[t][c * VE + j][i], o[t][c * VE + j + 1][i], o[t][c * VE + j + 2][i], o[t][c * VE + j + 3][i]};
                    }
            }
        }
        __syncthreads();
        const uint32_t rows_live = e.tokens * a.group - row0 < R ? e.tokens * a.group - row0 : R;
        const bool begins = g.first == g.tiles.lo;
        if (begins && !g.whole) attn_note_cut(a, attn_cut(a, e, work.split, g));
        float* piece = attn_piece(a, g, D);
        uint32_t nans = 0;                               // rows that came out as NaN for no NaN score (a row's values lie in one wave)
#pragma unroll 1
        for (uint32_t item = threadIdx.x; item < rows_live * (D / 4); item += blockDim.x) {
            const uint32_t r = item / (D / 4), d = (item % (D / 4)) * 4;
            float top = sh.m[0][r];
#pragma unroll
            for (int w = 1; w < 4; ++w) top = __builtin_fmaxf(top, sh.m[w][r]);
            float4_t y = {0, 0, 0, 0};
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = top == -__builtin_inff() ? 1.0f : attn_exp2((sh.m[w][r] - top) * scale.c);
                y += f * *reinterpret_cast<const float4_t*>(&sh.o[w][r][d]);
                sum += f * sh.l[w][r];
            }
            const uint32_t i = (row0 + r) / a.group, token = e.first_token + i, head = g.kv_head * a.group + (row0 + r) - i * a.group;
            if (sum == sum && (y.x != y.x || y.y != y.y || y.z != y.z || y.w != y.w)) nans |= 1u << r;
            float* dst = attn_whole_row(a, token, head, D);
            if (a.part != smelt_serving::kWholeSequences && begins && d == 0) attn_end_row(dst + D, a, work, g, r, top, sum);
            if (!g.whole) {
                *reinterpret_cast<float4_t*>(piece + 2 * R + r * D + d) = y;
                if (d == 0) *reinterpret_cast<float2*>(piece + 2 * r) = float2{top, sum};
            } else if (a.part != smelt_serving::kWholeSequences) {
                *reinterpret_cast<float4_t*>(dst + d) = y;
            } else {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                *reinterpret_cast<uint2_t*>(a.out + ((size_t)token * a.heads + head) * D + d) = uint2_t{attn_pack2<ActT>(y.x * inv, y.y * inv), attn_pack2<ActT>(y.z * inv, y.w * inv)};
            }
        }
        if (__builtin_expect(__any(nans != 0), 0) && attn_again<ActT, D>(a, e, g, [&](int run) {
                AttnBounds b[RT];
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    b[t] = attn_bounds(a, AttnRow{16 * t + col < rows_live, 0, 0, sh.position[16 * t + col]}, run ? (int32_t)e.prefix : 0, (int32_t)(run ? e.own : e.front));
                return attn_run(a, e, run, row0, R, b, RT);
            })) {
#pragma unroll 1
            while (const unsigned long long who = __ballot(nans != 0)) {
                const uint32_t r = __builtin_ctz(__builtin_amdgcn_readlane(nans, __builtin_ctzll(who))), i = (row0 + r) / a.group;
                nans &= ~(1u << r);
                float top = sh.m[0][r], sum = 0.0f;
#pragma unroll
                for (int w = 1; w < 4; ++w) top = __builtin_fmaxf(top, sh.m[w][r]);
#pragma unroll
                for (int w = 0; w < 4; ++w) sum += (top == -__builtin_inff() ? 1.0f : attn_exp2((sh.m[w][r] - top) * scale.c)) * sh.l[w][r];
                attn_form_row<ActT, D>(a, e, g, r, e.first_token + i, g.kv_head * a.group + (row0 + r) - i * a.group, sh.position[r], top, sum, scale.c);
            }
        }
        __syncthreads();
    }
}

// Many rows (prompts, the prefix against a batch): bound by the matrix cores and by what their waves issue besides.  A workgroup's WAVES
// waves hold 32 rows each and walk the key tiles of a run together, in stages of NS tiles that are loaded from the cache straight to
// LDS (no registers in between) while the kAttnBuffers - 1 stages before are waited for and worked on, one barrier a stage.  Every load of a
// wave lies within one half tile and so within one page: a scalar base (page ids are fetched a stage ahead) and offsets of the
// lanes that never change.  Every wave takes its operands from LDS: K in operand order, V through the transposing LDS read (16 lanes take
// 4 keys x 16 values and get one value of 4 keys each), the 16-byte pieces of V rows placed so that the four keys of such a read lie
// on different banks.
//
// Two prompt chunks of 900 and 1024 tokens behind up to 4000 keys, 32 heads of 128: 138 us with the join's 5, 750 TFLOP/s (a large library
// product reaches 1190); 160 us by itself.  The matrix cores are busy for 31 % of the launch: its 248 segments have 105 key tiles on
// average and 127 at most, and what is not in the stages is their start and end.  A stage takes about 4450 cycles a SIMD: its two waves' matrix instructions fill 2100 of them and their vector instructions (24 cycles a score and
// lane) 1500; the barrier keeps both in the same phase for the rest.  Heads of 256 have one wave a SIMD, 1.5 us a tile against 0.5 of matrix
// instructions: a wave issues one instruction every four cycles, so every scalar one counts.  With the turns written out as the matrix
// instructions' shadows (scores of the next tile beside this one's probabilities; four waves of 64 rows for heads of 128) they took 34
// us against 34.5 here for a prefix of 8192 against 384 rows, and the prompt chunks 185 us against 138.
typedef short attn_short4_t __attribute__((ext_vector_type(4)));
constexpr int kAttnBuffers = 4;

// 16-byte piece c of V row r lies at piece c ^ (4 * turn): the rows of a read on different banks
template <int D>
__device__ __forceinline__ uint32_t attn_v_turn(uint32_t row) { return D == 64 ? (row >> 1) & 1u : row & 3u; }

// 16 bytes a lane from base + offset to LDS at `lds` + 16 * lane; counts as a vector load, in order.  (Five wait states: the compiler
// does not see that a vector load reads the base, which a vector instruction may have written just before.)
__device__ __forceinline__ void attn_load_lds(uint64_t base, uint32_t offset, uint32_t lds) {
    base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(base >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)base);
    lds = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds) : "memory", "m0");
}
// waits until at most N of the wave's vector loads are under way
template <int N>
__device__ __forceinline__ void attn_wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory"); }

template <class ActT, int D, int WAVES, int NS>
__device__ __forceinline__ void attn_tiles(const AttentionArgs& a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    constexpr uint32_t R = 32 * WAVES, kHalf = 16 * D * 2, kTile = 4 * kHalf, kStage = NS * kTile;      // bytes: K halves, V halves
    constexpr int P = D / (8 * WAVES), kPerHalf = D / 32;       // loads of a wave a tile; wave loads a half
    constexpr bool kOneHalf = WAVES >= 2 * kPerHalf;            // a wave's loads are all of one half's keys or values
    constexpr uint32_t kRowShift = D == 256 ? 9 : (D == 128 ? 8 : 7);   // bytes of a V row
    constexpr uint32_t kAllThere = (1u << 2 * NS) - 1;
    const AttnWork work = find_work(a, blockIdx.x);
    attn_note_cut(a, {});
    if (work.entry == ~0u) return;
    uint32_t unit = work.at, index = work.entry, base = work.base;
    const uint32_t unit_end = work.parts || work.split.whole ? unit + 1 : smelt_serving::attention_start(work.split, blockIdx.x + 1);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave, half = lane >> 5;
    const uint32_t my_half = (wave / kPerHalf) & 1u;
    const bool my_value = wave / (2 * kPerHalf) != 0;
    const AttnScale scale = attn_scale(a);
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem);
    // the lane's place in each of the wave's loads: piece `at` of a half, K [dim / 8][key][8] or V [key][dim]
    uint32_t offset[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const uint32_t q = p * WAVES + wave, at = (q % kPerHalf) * 64 + lane;
        const uint32_t key = at / (D / 8), col = (at % (D / 8)) ^ (4 * attn_v_turn<D>(key));
        offset[p] = q < 2 * kPerHalf ? ((at / 16 << a.page_shift) + at % 16) * 16 : (key * D + col * 8) * 2;
    }
    // ... and of a transposing read: key row and 8-byte piece; the pieces of 32 values further on are turned by the row
    const uint32_t v_row = 4 * half + (lane & 15) / 4, v_turn = attn_v_turn<D>(v_row);
    const uint32_t v_lane = v_row * 2 * D + ((lane & 31) / 16) * 32 + (lane & 3) * 8;
    const uint32_t k_lane = ((lane & 31) / 16) * kHalf + half * 256 + (lane & 15) * 16;
#pragma unroll 1
    while (unit < unit_end) {
        const AttentionEntry e = attn_entry(a, index);
        AttnSegment g;
        if (work.parts) attn_part(a, e, work, g);
        else if (work.split.whole) attn_whole_segment(a, e, unit - base, g);
        else if (!attn_segment(a, e, base, unit, unit_end, g)) { base = g.begin; ++index; continue; }
        unit += g.units;
        if (g.first >= g.last) continue;                 // (only some of its lead)
        const uint32_t row0 = g.row_tile * R + wave * 32;
        const AttnRow row = attn_row(a, e, row0 + (lane & 31));
        AttnAcc<D> acc;
        attn_clear<D>(acc);
        uint4_t qf[D / 16];
        attn_load_q<D / 16>(a, row, a.q + (size_t)row.token * a.q_stride + (size_t)(g.kv_head * a.group + row.head) * D + 8 * half, 16, qf);
        const uint32_t page_bytes = (a.kv_heads * D * 2) << a.page_shift, head_bytes = __builtin_amdgcn_readfirstlane((g.kv_head * D * 2) << a.page_shift);
        const uint64_t k_base = (uint64_t)(uintptr_t)a.k_cache + head_bytes, v_base = (uint64_t)(uintptr_t)a.v_cache + head_bytes;
#pragma unroll 1
        for (int run = 0; run < 2; ++run) {
            const uint32_t len = run ? e.own : e.front, tile0 = run ? e.front_tiles : 0u, tiles = (len + 31) / 32;
            const uint32_t first = g.first > tile0 ? g.first - tile0 : 0u;
            uint32_t last = g.last > tile0 ? g.last - tile0 : 0u;
            last = last < tiles ? last : tiles;
            if (first >= last) continue;
            const scalar_table table = as_scalar(run ? a.page_table + (size_t)e.sequence * a.pages_per_sequence : a.prefix_table);
            const uint32_t last_page = (len - 1) >> a.page_shift, page_mask = (1u << a.page_shift) - 1u;
            const AttnBounds b = attn_bounds(a, row, run ? (int32_t)e.prefix : 0, (int32_t)len);
            const AttnRun u = attn_run(a, e, run, row0, 32, &b, 1);
            const uint32_t stages = (last - first + NS - 1) / NS;

            // stages whose every key all of the wave's rows see (so the run does not end inside one either)
            const uint32_t seen_lo = u.all_lo > 0 ? ((uint32_t)u.all_lo + 31) / 32 : 0u, seen_hi = u.all_hi > 0 ? (uint32_t)u.all_hi / 32 : 0u;
            const uint32_t plain_lo = __builtin_amdgcn_readfirstlane(seen_lo > first ? (seen_lo - first + NS - 1) / NS : 0u);
            const uint32_t plain_hi = __builtin_amdgcn_readfirstlane(seen_hi > first ? (seen_hi - first) / NS : 0u);
            const uint32_t plain_n = plain_hi > plain_lo ? plain_hi - plain_lo : 0u;

            // pages of a stage's half tiles; past the run's part its last tile once more, so that every stage is the same number of loads
            struct Pages { uint32_t id[NS][2]; };
            auto pages_of = [&](uint32_t stage) {
                Pages p;
#pragma unroll
                for (int n = 0; n < NS; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t tile = first + stage * NS + n;
                        tile = tile < last ? tile : last - 1;
                        uint32_t i = (tile * 32 + 16 * h) >> a.page_shift;
                        i = i < last_page ? i : last_page;      // behind the run: masked by its length
                        p.id[n][h] = (uint32_t)table[__builtin_amdgcn_readfirstlane(i)];
                    }
                return p;
            };
            uint32_t there = 0;                           // 2 NS bits a stage, the last fetched lowest: the half tiles that are there, on pages of the pool's
            auto fetch = [&](uint32_t stage, const Pages& pages) {
                const uint32_t to = lds0 + (stage % kAttnBuffers) * kStage;
                there <<= 2 * NS;
#pragma unroll
                for (int n = 0; n < NS; ++n) {
                    uint32_t tile = first + stage * NS + n;
                    const bool some = tile < last;
                    tile = some ? tile : last - 1;
                    uint64_t at[2];
                    uint32_t off[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const bool known = pages.id[n][h] < a.pages;
                        there |= known && some ? 1u << (2 * n + h) : 0u;
                        at[h] = (uint64_t)(known ? pages.id[n][h] : 0u) * page_bytes;
                        off[h] = (tile * 32 + 16 * h) & page_mask;
                    }
                    if constexpr (kOneHalf) {
                        at[0] = my_half ? at[1] : at[0];
                        off[0] = my_half ? off[1] : off[0];
                    }
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        const int h = kOneHalf ? 0 : (p * WAVES / kPerHalf) & 1;
                        const bool value = P == 1 ? my_value : p >= P / 2;
                        attn_load_lds((value ? v_base : k_base) + at[h] + (off[h] << (value ? kRowShift : 4u)), offset[p], to + n * kTile + (p * WAVES + wave) * 1024);
                    }
                }
            };
#pragma unroll 1
            for (uint32_t s = 0; s < kAttnBuffers - 1; ++s) {
                if (s < stages) fetch(s, pages_of(s));
                else there <<= 2 * NS;
            }
            Pages pages = pages_of(kAttnBuffers - 1);
            // (the compiler counts its own loads alone: from here on only stages are under way)
            if (run == 0 || e.front_tiles == 0) attn_wait_loads<0>();

#pragma unroll 1
            for (uint32_t stage = 0; stage < stages; ++stage) {
                const uint32_t buffer = stage % kAttnBuffers;
                // this stage is complete when only the later ones' loads are left
                if (stage + kAttnBuffers - 1 <= stages) attn_wait_loads<(kAttnBuffers - 2) * P * NS>();
                else attn_wait_loads<0>();
                __syncthreads();
                const uint32_t known = (there >> (2 * NS * (kAttnBuffers - 2))) & kAllThere;
                const bool plain = stage - plain_lo < plain_n && known == kAllThere;
                const unsigned char* st = smem + buffer * kStage;
                if (known != kAllThere || (first + (stage + 1) * NS) * smelt_serving::kKeyTile > len) {
                    // Values of keys behind the run's end, or on a page that is none of the pool's, are whatever memory holds: zero them,
                    // since a zero probability does not silence an infinity or a NaN.
#pragma unroll 1
                    for (int n = 0; n < NS; ++n) {
                        const uint32_t key0 = (first + stage * NS + n) * smelt_serving::kKeyTile;
                        uint4_t* v = reinterpret_cast<uint4_t*>(smem + buffer * kStage + n * kTile + 2 * kHalf);
                        for (uint32_t p = threadIdx.x; p < 4 * D; p += 64 * WAVES) {
                            const uint32_t key = p / (D / 8);
                            if (key0 + key >= len || !((known >> (2 * n + key / 16)) & 1u)) v[p] = uint4_t{0, 0, 0, 0};
                        }
                    }
                    __syncthreads();
                }
                // operands are read well before the products that take them: K of a tile while the one before is multiplied, V before the softmax
                float16_t s[NS];
                uint4_t kf[2][D / 16];
                auto load_k = [&](int n) {
                    const uint4_t* kl = reinterpret_cast<const uint4_t*>(st + n * kTile + k_lane);
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) kf[n & 1][d] = kl[d * 32];
                };
                load_k(0);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 0; n < NS; ++n) {
                    if (n + 1 < NS) { load_k(n + 1); __builtin_amdgcn_sched_barrier(0); }
                    s[n] = attn_mfma<ActT>(kf[n & 1][0], qf[0], float16_t{});
#pragma unroll
                    for (int d = 1; d < D / 16; ++d) s[n] = attn_mfma<ActT>(kf[n & 1][d], qf[d], s[n]);
                }
                if (stage + kAttnBuffers - 1 < stages) {
                    fetch(stage + kAttnBuffers - 1, pages);
                    pages = pages_of(stage + kAttnBuffers);
                } else {
                    there <<= 2 * NS;
                }
                uint4_t vf[NS][2][D / 32];
#pragma unroll
                for (int n = 0; n < NS; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < D / 32; ++j) {
                            const unsigned char* at = st + n * kTile + 2 * kHalf + v_lane + h * kHalf + ((j & ~3) | ((j & 3) ^ v_turn)) * 64;
                            typedef __attribute__((address_space(3))) attn_short4_t* lds_ptr;
                            const uint2_t lo = __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)at));
                            const uint2_t hi = __builtin_bit_cast(uint2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at + 8 * 2 * D)));
                            vf[n][h][j] = uint4_t{lo.x, lo.y, hi.x, hi.y};
                        }
                __builtin_amdgcn_sched_barrier(0);
                if (!plain) {
#pragma unroll
                    for (int n = 0; n < NS; ++n) attn_hide(s[n], (int32_t)((first + stage * NS + n) * smelt_serving::kKeyTile), b, known >> (2 * n));
                }
                attn_softmax<D, NS>(scale, acc, s);
#pragma unroll
                for (int n = 0; n < NS; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint4_t pf = attn_pack<ActT>(s[n], h);
#pragma unroll
                        for (int j = 0; j < D / 32; ++j) acc.o[j] = attn_mfma<ActT>(vf[n][h][j], pf, acc.o[j]);
                    }
            }
            __syncthreads();                              // (the next loads overwrite the stages)
        }
        // a lane holds its row's values 32 j + 8 (i / 4) + 4 half + i % 4
        const bool begins = g.first == g.tiles.lo;
        if (begins && !g.whole) attn_note_cut(a, attn_cut(a, e, work.split, g));
        float* piece = attn_piece(a, g, D);
        const float l = attn_halves_sum(acc.l);
        bool nan = false;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) nan = nan || acc.o[j][i] != acc.o[j][i];
        const unsigned long long nans = __ballot(nan && l == l && row.live);
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
                float* whole = attn_whole_row(a, row.token, head, D);
                float* dst = g.whole ? whole : piece + 2 * R + r * D;
                if (half == 0) {
                    if (a.part != smelt_serving::kWholeSequences && begins) attn_end_row(whole + D, a, work, g, r, acc.m, l);
                    if (!g.whole) *reinterpret_cast<float2*>(piece + 2 * r) = float2{acc.m, l};
                }
#pragma unroll
                for (int j = 0; j < D / 32; ++j)
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        *reinterpret_cast<float4_t*>(dst + 4 * half + 32 * j + 2 * i) = float4_t{acc.o[j][i], acc.o[j][i + 1], acc.o[j][i + 2], acc.o[j][i + 3]};
            }
        }
        // (the other waves' rows see other keys, so each wave looks and forms for itself)
        if (__builtin_expect(nans != 0, 0)) {
            const bool again = attn_again<ActT, D>(a, e, g, [&](int run) {
                const AttnBounds b = attn_bounds(a, row, run ? (int32_t)e.prefix : 0, (int32_t)(run ? e.own : e.front));
                return attn_run(a, e, run, row0, 32, &b, 1);
            });
#pragma unroll 1
            for (uint32_t set = again ? (uint32_t)nans | (uint32_t)(nans >> 32) : 0u; set; set &= set - 1) {
                const int from = __builtin_ctz(set);
                attn_form_row<ActT, D>(a, e, g, wave * 32 + from, __builtin_amdgcn_readlane(row.token, from), g.kv_head * a.group + __builtin_amdgcn_readlane(row.head, from),
                                       __builtin_amdgcn_readlane(row.position, from), __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, acc.m), from)),
                                       __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, l), from)), scale.c);
            }
        }
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
// row r of `parts` parts of a segment, the first in slot `first`
template <int D>
__device__ __forceinline__ void attn_join_pieces(AttnJoin& j, const AttentionArgs& a, uint32_t first, uint32_t parts, uint32_t r, uint32_t d, float c) {
    constexpr uint32_t U = 12;     // parts whose loads are under way together
#pragma unroll 1
    for (uint32_t base = 0; base < parts; base += U) {
        float2 ml[U];
        float4_t y[U];
#pragma unroll
        for (uint32_t k = 0; k < U; ++k) {
            const uint32_t w = base + k < parts ? base + k : parts - 1;
            uint32_t slot = a.part == smelt_serving::kPrefix ? first + w : (w ? 2 * (first / 2 + w) : first);
            slot = slot < a.slots ? slot : a.slots - 1;
            const float* piece = a.pieces + (size_t)slot * smelt_serving::piece_floats(a.row_tile, D);
            ml[k] = *reinterpret_cast<const float2*>(piece + 2 * r);
            y[k] = *reinterpret_cast<const float4_t*>(piece + 2 * a.row_tile + r * D + d);
        }
#pragma unroll
        for (uint32_t k = 0; k < U; ++k)
            if (base + k < parts) attn_join(j, ml[k].x, ml[k].y, y[k], c);
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

// kWholeSequences.  Grid: workgroups of the first launch x slices of a segment's rows.
template <class ActT, int D>
__device__ __forceinline__ void attn_combine(const AttentionArgs& a) {
    typedef const __attribute__((address_space(4))) smelt_serving::AttentionCut* scalar_cut;
    const scalar_cut c = (scalar_cut)(uintptr_t)(a.cuts + blockIdx.x);
    const uint32_t last = c->last, kv_head = c->kv_head, first_token = c->first_token, row0 = c->row0, rows = c->rows;
    if (last == 0) return;
#pragma unroll 1
    for (uint32_t item = blockIdx.y * blockDim.x + threadIdx.x; item < rows * (D / 4); item += gridDim.y * blockDim.x) {
        const uint32_t r = item / (D / 4), d = (item % (D / 4)) * 4;
        AttnJoin j{-__builtin_inff(), 0.0f, {0, 0, 0, 0}};
        attn_join_pieces<D>(j, a, 2 * blockIdx.x + 1, last - blockIdx.x + 1, r, d, a.scale_log2);
        const uint32_t i = (row0 + r) / a.group, token = first_token + i, head = kv_head * a.group + (row0 + r) - i * a.group;
        attn_finish<ActT>(j, a.out + ((size_t)token * a.heads + head) * D + d);
    }
}

// kPrefix and kOwnKeys.  Grid: tokens x kv heads: a row's two halves, each in parts or whole.
template <class ActT, int D>
__device__ __forceinline__ void attn_combine_shared(const smelt_serving::AttentionJoinArgs& both) {
    const AttentionArgs& own = both.own;
    const uint32_t token = blockIdx.x, kv_head = blockIdx.y;
    if (token >= smelt_serving::clamp_count(as_scalar(own.offsets)[own.sequences], own.tokens)) return;     // a row behind the last sequence
    const bool prefix = as_scalar(own.prefix_len)[0] > 0;
#pragma unroll 1
    for (uint32_t item = threadIdx.x; item < own.group * (D / 4); item += blockDim.x) {
        const uint32_t head = kv_head * own.group + item / (D / 4), d = (item % (D / 4)) * 4;
        const float* front_row = attn_whole_row(both.front, token, head, D);
        const float* own_row = attn_whole_row(own, token, head, D);
        const smelt_serving::AttentionRowEnd front_end = *reinterpret_cast<const smelt_serving::AttentionRowEnd*>(front_row + D);
        const smelt_serving::AttentionRowEnd own_end = *reinterpret_cast<const smelt_serving::AttentionRowEnd*>(own_row + D);
        const float4_t front_y = *reinterpret_cast<const float4_t*>(front_row + d), own_y = *reinterpret_cast<const float4_t*>(own_row + d);
        AttnJoin j{-__builtin_inff(), 0.0f, {0, 0, 0, 0}};
        auto join = [&](const AttentionArgs& x, const smelt_serving::AttentionRowEnd& end, float4_t y) {
            // (offsets that do not ascend leave rows without a segment: whatever is there stays within the slots)
            uint32_t parts = end.parts_row >> 8, r = end.parts_row & 255u;
            parts = parts < x.slots ? parts : x.slots;
            r = r < x.row_tile ? r : x.row_tile - 1;
            if (parts <= 1) attn_join(j, end.max, end.sum, y, x.scale_log2);
            else attn_join_pieces<D>(j, x, end.piece < x.slots ? end.piece : 0u, parts, r, d, x.scale_log2);
        };
        if (prefix) join(both.front, front_end, front_y);
        join(own, own_end, own_y);
        attn_finish<ActT>(j, own.out + ((size_t)token * own.heads + head) * D + d);
    }
}

}  // namespace smelt

// (one wave a SIMD where accumulators, q and the tiles in flight take the whole register file)
#define SMELT_ATTENTION_KERNELS(T, ACT, D, STREAM16, STREAM32, WAVES, NS, TILE_WAVES)                                                                                           \
    extern "C" __global__ __launch_bounds__(256, STREAM16) void smelt_attention_stream16_d##D##_##T(smelt_serving::AttentionArgs a) { smelt::attn_stream<ACT, D, 1>(a); }             \
    extern "C" __global__ __launch_bounds__(256, STREAM32) void smelt_attention_stream32_d##D##_##T(smelt_serving::AttentionArgs a) { smelt::attn_stream<ACT, D, 2>(a); }             \
    extern "C" __global__ __launch_bounds__(64 * WAVES, TILE_WAVES) void smelt_attention_tiles_d##D##_##T(smelt_serving::AttentionArgs a) { smelt::attn_tiles<ACT, D, WAVES, NS>(a); } \
    extern "C" __global__ __launch_bounds__(256) void smelt_attention_join_d##D##_##T(smelt_serving::AttentionArgs a) { smelt::attn_combine<ACT, D>(a); }                            \
    extern "C" __global__ __launch_bounds__(1024) void smelt_attention_join_shared_d##D##_##T(smelt_serving::AttentionJoinArgs a) { smelt::attn_combine_shared<ACT, D>(a); }
