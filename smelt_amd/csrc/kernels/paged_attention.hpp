// Attention of new token rows over a paged key / value cache, with a prefix that the whole batch shares.
//
//   y(row) = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q.k_j - m),  c = scale * log2(e),  m the running maximum
//
// over the keys j the row sees (causal, within the window).  Scores, maxima, sums and the output accumulators are 32-bit; p is
// rounded to the 16-bit type for the second product (relative error half a step of that type, averaged over the keys), its sum is not.
// The maximum only moves when a score passes it by more than 2^8 (p then stays below 256, far inside fp16), so most key tiles
// rescale nothing.
//
// Rows are (token, head of the group) pairs of one kv head, 32 to a tile, and both products are formed transposed, so that a lane
// owns one row throughout (v_mfma_f32_32x32x16, lane l: row l % 32):
//   S^T [32 keys x 32 rows] = K Q^T       a lane ends up with 16 of the 32 scores of its row, lane ^ 32 with the others
//   O^T [dim x 32 rows]    += V^T P^T     the lane's own 16 probabilities are its operand as they stand: the order of the keys of
//                                         a contraction is free, so V rows are taken in the order the first product left them
// Maximum, sum and rescaling are per lane; nothing crosses lanes but one exchange of the maximum.  K is stored in operand order
// ([dim / 8][key][8] within a page and head: a load covers 512 contiguous bytes per half wave); V rows are read as they are stored (a
// lane takes dim / 32 neighbouring values of 16 keys) and pairs of keys are put side by side with one v_perm per operand dword.
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

__device__ __forceinline__ float attn_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float attn_other_half(float v) { return __shfl_xor(v, 32); }

// sum of one value per thread over the workgroup's threads before this one and over all of them
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* wave_sums, uint64_t* total) {
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
    uint64_t run = v;
#pragma unroll
    for (uint32_t d = 1; d < (uint32_t)kWave; d <<= 1) {
        const uint64_t up = __shfl_up(run, d);
        if (lane >= d) run += up;
    }
    __syncthreads();
    if (lane == kWave - 1) wave_sums[wave] = run;
    __syncthreads();
    uint64_t before = 0, all = 0;
    for (uint32_t w = 0; w < waves; ++w) {
        if (w < wave) before += wave_sums[w];
        all += wave_sums[w];
    }
    *total = all;
    return before + run - v;
}

struct AttnWork {
    uint64_t units;          // of the whole launch
    uint32_t entry;          // where the wanted unit (or row) lies
    uint64_t entry_base;     // units before that entry
};

// Walks the entries in chunks of one per thread.  FIND_ROW: looks for the entry of token `want`, else for the entry of
// workgroup `want`'s first unit (entry = ~0 when the workgroup has none).
template <bool FIND_ROW>
__device__ __forceinline__ AttnWork find_work(const AttentionArgs& a, uint32_t want, uint64_t* scratch) {
    const uint32_t entries = a.sequences + a.cascade;
    uint32_t* found_entry = reinterpret_cast<uint32_t*>(scratch + 8);
    AttnWork w;
    w.units = 0;
    uint64_t kept_before = 0, kept_units = 0;
    if (threadIdx.x == 0) *found_entry = ~0u;
    for (uint32_t base = 0; base < entries; base += blockDim.x) {
        const uint32_t index = base + threadIdx.x;
        AttentionEntry e;
        uint64_t mine = 0, all;
        if (index < entries) { e = smelt_serving::attention_entry(a, index); mine = smelt_serving::attention_units(a, e); }
        const uint64_t before = w.units + block_scan(mine, scratch, &all);
        if (FIND_ROW && index < entries && e.sequence >= 0 && want >= e.first_token && want - e.first_token < e.tokens) {
            *found_entry = index;
            scratch[9] = before;
        }
        kept_before = before; kept_units = mine;
        w.units += all;
    }
    if (!FIND_ROW) {
        const uint32_t groups = smelt_serving::attention_groups(a, w.units);
        if (want < groups) {
            const uint64_t u = smelt_serving::attention_start(w.units, groups, want);
            if (entries <= blockDim.x) {
                if (u >= kept_before && u - kept_before < kept_units) { *found_entry = threadIdx.x; scratch[9] = kept_before; }
            } else {
                uint64_t run = 0;
                for (uint32_t base = 0; base < entries; base += blockDim.x) {
                    const uint32_t index = base + threadIdx.x;
                    uint64_t mine = 0, all;
                    if (index < entries) mine = smelt_serving::attention_units(a, smelt_serving::attention_entry(a, index));
                    const uint64_t before = run + block_scan(mine, scratch, &all);
                    if (u >= before && u - before < mine) { *found_entry = index; scratch[9] = before; }
                    run += all;
                }
            }
        }
    }
    __syncthreads();
    w.entry = *found_entry;
    w.entry_base = scratch[9];
    __syncthreads();
    return w;
}

// the sequence of a token row: offsets is ascending, tokens before offsets[sequences] belong to one
__device__ __forceinline__ uint32_t sequence_of(const AttentionArgs& a, uint32_t token) {
    uint32_t lo = 0, hi = a.sequences;   // offsets[lo] <= token < offsets[hi]
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
    uint32_t s, first, count, own;
    if (e.sequence >= 0) { s = (uint32_t)e.sequence; first = e.first_token; count = e.tokens; own = e.own; }
    else {
        s = sequence_of(a, r.token);
        first = smelt_serving::clamp_count(a.offsets[s], a.tokens);
        count = smelt_serving::clamp_count(a.offsets[s + 1], a.tokens) - first;
        own = smelt_serving::clamp_count(a.kv_lens[s], a.pages_per_sequence << a.page_shift);
    }
    const uint32_t front = a.prefix_len ? smelt_serving::clamp_count(a.prefix_len[0], a.prefix_pages << a.page_shift) : 0u;
    r.position = (int32_t)(front + own + (r.token - first)) - (int32_t)count;
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
    if (a.window > 0x7FFFFFFFu) b.lo = 0;
    return b;
}

template <int CTRL_MAX>
__device__ __forceinline__ int32_t wave_reduce_int(int32_t v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const int32_t o = __shfl_xor(v, off);
        v = CTRL_MAX ? (o > v ? o : v) : (o < v ? o : v);
    }
    return v;
}

// One wave's state: 32 rows.
template <int D>
struct AttnAcc {
    float16_t o[D / 32];     // o[j][i]: value (D / 32) * (8 (i / 4) + 4 (lane / 32) + i % 4) + j of the lane's row
    float m, l;              // running maximum (log2 domain) and this half's sum
};

template <class ActT, int D>
__device__ __forceinline__ void attn_load_q(const AttentionArgs& a, const AttnRow& r, uint32_t kv_head, uint4_t* qf) {
    const int half = (threadIdx.x & 63) >> 5;
    const uint16_t* q = a.q + (size_t)r.token * a.q_stride + (size_t)(kv_head * a.group + r.head) * D + 8 * half;
    if ((reinterpret_cast<uintptr_t>(a.q) & 15u) == 0 && (a.q_stride & 7u) == 0) {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) qf[t] = r.live ? *reinterpret_cast<const uint4_t*>(q + 16 * t) : uint4_t{0, 0, 0, 0};
    } else {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = r.live ? (uint32_t)q[16 * t + 2 * k] | ((uint32_t)q[16 * t + 2 * k + 1] << 16) : 0u;
            qf[t] = uint4_t{w[0], w[1], w[2], w[3]};
        }
    }
}

// Address of one key tile: the page (two for pages of 16) and whether it is one of the pool's.
template <bool SMALL>
struct AttnTile {
    size_t base[SMALL ? 2 : 1];      // element offset of the page's head
    bool valid[SMALL ? 2 : 1];
    uint32_t off;                    // first key within the page
};

template <bool SMALL, int D>
__device__ __forceinline__ AttnTile<SMALL> attn_tile(const AttentionArgs& a, const int32_t* table, uint32_t kv_head, uint32_t run_len, uint32_t tile) {
    AttnTile<SMALL> t;
    const uint32_t key = tile * smelt_serving::kKeyTile;
    const uint32_t last_page = run_len ? (run_len - 1) >> a.page_shift : 0u;
    t.off = SMALL ? 0u : key & ((1u << a.page_shift) - 1u);
#pragma unroll
    for (int k = 0; k < (SMALL ? 2 : 1); ++k) {
        uint32_t index = (key >> a.page_shift) + k;
        if (index > last_page) index = last_page;      // behind the run: masked by its length
        const uint32_t page = __builtin_amdgcn_readfirstlane(table[index]);
        t.valid[k] = page < a.pages;
        t.base[k] = (((size_t)(t.valid[k] ? page : 0u) * a.kv_heads + kv_head) * D) << a.page_shift;
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

template <class ActT, int D, bool SMALL>
__device__ __forceinline__ void attn_softmax(const AttentionArgs& a, AttnAcc<D>& acc, float16_t& s, const AttnTile<SMALL>& t, int32_t key0, const AttnBounds& b, bool masked) {
    const int half = (threadIdx.x & 63) >> 5;
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] *= a.scale_log2;
    if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int32_t key = key0 + 8 * (i / 4) + 4 * half + i % 4;
            const bool ok = key >= b.lo && key < b.hi && t.valid[SMALL ? i / 8 : 0];
            s[i] = ok ? s[i] : -__builtin_inff();
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, s[i]);
    top = __builtin_fmaxf(top, attn_other_half(top));
    if (__any(top > acc.m + 8.0f)) {      // also the first finite score: the maximum starts at -inf
        const float m = __builtin_fmaxf(acc.m, top);
        const float f = m == -__builtin_inff() ? 1.0f : attn_exp2(acc.m - m);
        acc.l *= f;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc.o[j][i] *= f;
        acc.m = m;
    }
    const float m = acc.m == -__builtin_inff() ? 0.0f : acc.m;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) { s[i] = attn_exp2(s[i] - m); sum += s[i]; }
    acc.l += sum;
}

template <class ActT, int D>
__device__ __forceinline__ void attn_values(AttnAcc<D>& acc, const float16_t& p, const AttnV<D>& vf) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        uint4_t pf;
        pf.x = attn_pack2<ActT>(p[8 * u], p[8 * u + 1]);
        pf.y = attn_pack2<ActT>(p[8 * u + 2], p[8 * u + 3]);
        pf.z = attn_pack2<ActT>(p[8 * u + 4], p[8 * u + 5]);
        pf.w = attn_pack2<ActT>(p[8 * u + 6], p[8 * u + 7]);
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
            const bool ok = key0 + 16 * u + 8 * (r / 4) + 4 * half + r % 4 < run_len && t.valid[SMALL ? u : 0];
#pragma unroll
            for (int k = 0; k < D / 64; ++k) vf.w[u][r][k] = ok ? vf.w[u][r][k] : 0u;
        }
}

// cascade: where a row of a segment that one workgroup finished waits for its other part (which 0: prefix, 1: own keys)
__device__ __forceinline__ float* attn_whole_row(const AttentionArgs& a, uint32_t which, uint32_t token, uint32_t head, uint32_t dim) {
    return a.rows + (((size_t)which * a.tokens + token) * a.heads + head) * (dim + 4);
}

// LDS of the streaming kernel: partial outputs of the four waves, their maxima and sums, the partition's scratch
template <int D>
struct AttnShared {
    float o[4][32][D + 4];      // (four floats of padding: a half wave's 16-byte stores cover all banks)
    float m[4][32], l[4][32];
    uint64_t scratch[16];
};

// Few rows a sequence (decoding, drafted tokens): bound by the cache's bytes.  A workgroup takes a run of units and works
// through the segments it crosses, its four waves on every fourth key tile; at a segment's end the waves' results meet in LDS.
// A segment that lies whole in one workgroup is finished there; the parts of the others go to the workspace (two slots a workgroup
// are enough: only its first and last segment can be shared) and are joined by the second launch, in a fixed order.
template <class ActT, int D, bool SMALL>
__device__ __forceinline__ void attn_stream(const AttentionArgs& a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    AttnShared<D>& sh = *reinterpret_cast<AttnShared<D>*>(smem);
    const AttnWork work = find_work<false>(a, blockIdx.x, sh.scratch);
    if (work.entry == ~0u) return;
    const uint32_t groups = smelt_serving::attention_groups(a, work.units);
    uint64_t unit = smelt_serving::attention_start(work.units, groups, blockIdx.x);
    const uint64_t unit_end = smelt_serving::attention_start(work.units, groups, blockIdx.x + 1);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const uint32_t page = 1u << a.page_shift;
    uint32_t index = work.entry;
    uint64_t base = work.entry_base;
    while (unit < unit_end) {
        const AttentionEntry e = smelt_serving::attention_entry(a, index);
        const uint64_t size = smelt_serving::attention_units(a, e);
        if (unit - base >= size) { base += size; ++index; continue; }
        const uint64_t rel = unit - base;
        const uint32_t segment = (uint32_t)(rel / e.key_tiles), first = (uint32_t)(rel - (uint64_t)segment * e.key_tiles);
        const uint32_t kv_head = segment / e.row_tiles, row_tile = segment - kv_head * e.row_tiles;
        const uint32_t last = (uint64_t)(e.key_tiles - first) < unit_end - unit ? e.key_tiles : first + (uint32_t)(unit_end - unit);

        const AttnRow row = attn_row(a, e, row_tile * smelt_serving::kRowTile + (lane & 31));
        AttnAcc<D> acc;
        acc.m = -__builtin_inff(); acc.l = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc.o[j][i] = 0.0f;
        uint4_t qf[D / 16];
        attn_load_q<ActT, D>(a, row, kv_head, qf);
        const uint32_t front = a.prefix_len ? smelt_serving::clamp_count(a.prefix_len[0], a.prefix_pages * page) : 0u;
        for (int run = 0; run < 2; ++run) {
            const uint32_t run_len = run ? e.own : e.front;
            const uint32_t tile0 = run ? e.front_tiles : 0u, tiles = (run_len + smelt_serving::kKeyTile - 1) / smelt_serving::kKeyTile;
            if (tiles == 0) continue;
            const int32_t* table = run ? a.page_table + (size_t)e.sequence * a.pages_per_sequence : a.prefix_table;
            const AttnBounds b = attn_bounds(a, row, run ? (int32_t)front : 0, (int32_t)run_len);
            // what no row of the tile sees is not read; what all of them see needs no mask
            const int32_t most = wave_reduce_int<1>(row.live ? b.hi : 0), least = wave_reduce_int<0>(row.live ? b.lo : (int32_t)run_len);
            const int32_t all_hi = wave_reduce_int<0>(b.hi), all_lo = wave_reduce_int<1>(b.lo);
            int32_t t0 = (int32_t)first - (int32_t)tile0, t1 = (int32_t)last - (int32_t)tile0;
            t0 = t0 < 0 ? 0 : t0;
            t1 = t1 > (int32_t)tiles ? (int32_t)tiles : t1;
            if (t0 < least / (int32_t)smelt_serving::kKeyTile) t0 = least / (int32_t)smelt_serving::kKeyTile;
            const int32_t seen = most <= 0 ? 0 : (most + (int32_t)smelt_serving::kKeyTile - 1) / (int32_t)smelt_serving::kKeyTile;
            if (t1 > seen) t1 = seen;
            for (int32_t tile = t0 + (int32_t)wave; tile < t1; tile += 4) {
                const int32_t key0 = tile * (int32_t)smelt_serving::kKeyTile;
                const AttnTile<SMALL> at = attn_tile<SMALL, D>(a, table, kv_head, run_len, (uint32_t)tile);
                uint4_t kf[D / 16];
                AttnV<D> vf;
                float16_t s;
                attn_load_k<D, SMALL>(a, at, kf);
                attn_load_v<D, SMALL>(a, at, vf);
                attn_scores<ActT, D, SMALL>(a, qf, kf, s);
                const bool bad = !at.valid[0] || !at.valid[SMALL ? 1 : 0];
                const bool masked = bad || key0 + (int32_t)smelt_serving::kKeyTile > all_hi || key0 < all_lo;
                attn_softmax<ActT, D, SMALL>(a, acc, s, at, key0, b, masked);
                if (bad || key0 + (int32_t)smelt_serving::kKeyTile > (int32_t)run_len) attn_clear_v<D, SMALL>(vf, at, key0, (int32_t)run_len);
                attn_values<ActT, D>(acc, s, vf);
            }
        }
        // the waves meet
        const float l = acc.l + attn_other_half(acc.l);
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
        const bool whole = first == 0 && last == e.key_tiles;
        const uint32_t rows_live = e.tokens * a.group - row_tile * smelt_serving::kRowTile < smelt_serving::kRowTile ? e.tokens * a.group - row_tile * smelt_serving::kRowTile : smelt_serving::kRowTile;
        float* piece = a.pieces + ((size_t)blockIdx.x * 2 + (first == 0 ? 1 : 0)) * smelt_serving::piece_floats(D);
        for (uint32_t item = threadIdx.x; item < rows_live * (D / 4); item += blockDim.x) {
            const uint32_t r = item / (D / 4), d = (item % (D / 4)) * 4;
            float m = sh.m[0][r];
#pragma unroll
            for (int w = 1; w < 4; ++w) m = __builtin_fmaxf(m, sh.m[w][r]);
            float4_t y = {0, 0, 0, 0};
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = m == -__builtin_inff() ? 1.0f : attn_exp2(sh.m[w][r] - m);
                y += f * *reinterpret_cast<const float4_t*>(&sh.o[w][r][d]);
                sum += f * sh.l[w][r];
            }
            const uint32_t flat = row_tile * smelt_serving::kRowTile + r;
            const uint32_t token = e.first_token + flat / a.group, head = kv_head * a.group + flat % a.group;
            if (!whole) {
                *reinterpret_cast<float4_t*>(piece + 2 * smelt_serving::kRowTile + r * D + d) = y;
                if (d == 0) { piece[r] = m; piece[smelt_serving::kRowTile + r] = sum; }
            } else if (a.cascade) {
                float* dst = attn_whole_row(a, e.sequence < 0 ? 0u : 1u, token, head, D);
                *reinterpret_cast<float4_t*>(dst + d) = y;
                if (d == 0) { dst[D] = m; dst[D + 1] = sum; }
            } else {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                uint2_t w;
                w.x = attn_pack2<ActT>(y.x * inv, y.y * inv);
                w.y = attn_pack2<ActT>(y.z * inv, y.w * inv);
                *reinterpret_cast<uint2_t*>(a.out + ((size_t)token * a.heads + head) * D + d) = w;
            }
        }
        __syncthreads();
        unit += last - first;
    }
}

// Joins what the first launch left of one token's rows of one kv head: the parts of its own segment and, in a cascade, of the
// prefix's.  Nothing to do where one workgroup finished the segment.
struct AttnJoin { float m, l; float4_t y; };
__device__ __forceinline__ void attn_join(AttnJoin& j, float m, float l, float4_t y) {
    const float top = __builtin_fmaxf(j.m, m);
    const float f = top == -__builtin_inff() ? 1.0f : attn_exp2(j.m - top), g = top == -__builtin_inff() ? 1.0f : attn_exp2(m - top);
    j.y = f * j.y + g * y;
    j.l = f * j.l + g * l;
    j.m = top;
}

template <class ActT, int D>
__device__ __forceinline__ void attn_combine(const AttentionArgs& a) {
    __shared__ uint64_t scratch[16];
    const uint32_t token = blockIdx.x, kv_head = blockIdx.y;
    const AttnWork work = find_work<true>(a, token, scratch);
    if (work.entry == ~0u) return;       // a row behind the last sequence
    const uint32_t groups = smelt_serving::attention_groups(a, work.units);
    const AttentionEntry own = smelt_serving::attention_entry(a, work.entry);
    const AttentionEntry front = smelt_serving::attention_entry(a, 0);
    const bool cascade = a.cascade && front.key_tiles > 0;
    for (uint32_t item = threadIdx.x; item < a.group * (D / 4); item += blockDim.x) {
        const uint32_t g = item / (D / 4), d = (item % (D / 4)) * 4, head = kv_head * a.group + g;
        AttnJoin j{-__builtin_inff(), 0.0f, {0, 0, 0, 0}};
        bool done = false;
        for (uint32_t part = cascade ? 0u : 1u; part < 2; ++part) {
            const AttentionEntry& e = part ? own : front;
            const uint32_t flat = (token - e.first_token) * a.group + g, row_tile = flat / smelt_serving::kRowTile, r = flat % smelt_serving::kRowTile;
            const uint64_t begin = (part ? work.entry_base : 0) + ((uint64_t)kv_head * e.row_tiles + row_tile) * e.key_tiles, end = begin + e.key_tiles;
            const uint32_t w0 = smelt_serving::attention_owner(work.units, groups, begin), w1 = smelt_serving::attention_owner(work.units, groups, end - 1);
            if (w0 == w1) {
                if (!a.cascade) { done = true; break; }
                const float* row = attn_whole_row(a, part, token, head, D);
                attn_join(j, row[D], row[D + 1], *reinterpret_cast<const float4_t*>(row + d));
                continue;
            }
            for (uint32_t w = w0; w <= w1; ++w) {
                const uint32_t slot = smelt_serving::attention_start(work.units, groups, w) <= begin ? 1u : 0u;
                const float* piece = a.pieces + ((size_t)w * 2 + slot) * smelt_serving::piece_floats(D);
                attn_join(j, piece[r], piece[smelt_serving::kRowTile + r], *reinterpret_cast<const float4_t*>(piece + 2 * smelt_serving::kRowTile + r * D + d));
            }
        }
        if (done) continue;
        const float inv = j.l == 0.0f ? 0.0f : 1.0f / j.l;
        uint2_t w;
        w.x = attn_pack2<ActT>(j.y.x * inv, j.y.y * inv);
        w.y = attn_pack2<ActT>(j.y.z * inv, j.y.w * inv);
        *reinterpret_cast<uint2_t*>(a.out + ((size_t)token * a.heads + head) * D + d) = w;
    }
}

}  // namespace smelt

// (one workgroup a compute unit for heads of 256: accumulators, q and the tiles in flight take the whole register file)
#define SMELT_ATTENTION_KERNELS(T, ACT, D, WAVES)                                                                                                                  \
    extern "C" __global__ __launch_bounds__(256, WAVES) void smelt_attention_stream_d##D##_##T(smelt_serving::AttentionArgs a) { smelt::attn_stream<ACT, D, false>(a); } \
    extern "C" __global__ __launch_bounds__(256, WAVES) void smelt_attention_stream_d##D##_p16_##T(smelt_serving::AttentionArgs a) { smelt::attn_stream<ACT, D, true>(a); } \
    extern "C" __global__ __launch_bounds__(256) void smelt_attention_join_d##D##_##T(smelt_serving::AttentionArgs a) { smelt::attn_combine<ACT, D>(a); }
