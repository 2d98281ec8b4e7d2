// Argument blocks of the serving kernels (rotary positions, paged cache, attention over it, draft verification), shared by
// the host side that fills them and the kernels that take them by value, and the index arithmetic both sides use.
#pragma once
#include <stdint.h>

#ifdef __HIP__
#define SMELT_HD __host__ __device__ __forceinline__
#else
#define SMELT_HD inline
#endif

namespace smelt_serving {

// ---- rotary positions ----------------------------------------------------------------------------------------------
constexpr uint32_t kRopeThreads = 256;
constexpr uint32_t kRopeMaxPerToken = 65535;   // work units of one token: the kernels' reciprocal division is exact below this

// One set of rows that a rotary launch walks: `heads` heads of `dim` values a token.
struct RopeRows {
    const uint16_t* src = nullptr;
    uint16_t* dst = nullptr;         // rows (q, x), or the cache (k, v)
    uint32_t heads = 0, src_stride = 0, dst_stride = 0;   // strides in elements
    uint32_t units = 0;              // work units of a token: heads * units per head
};

// x / q rows in `q`; k and v (with the cache) only in append launches.
struct RopeArgs {
    RopeRows q, k, v;
    const int32_t* positions = nullptr;
    const double* table = nullptr;     // radians a position, one per rotated pair
    const int32_t* slots = nullptr;    // append: page * page_size + offset, negative = nowhere
    uint32_t tokens = 0, dim = 0, rot = 0, interleaved = 0;
    float amplitude = 1.0f;
    uint32_t tokens_per_group = 1;     // tokens of one workgroup, a power of two up to 4
    uint32_t per_token = 0, q_units_inv = 0, v_units_inv = 0;   // units of one token; ceil(2^32 / units) of its q and v
    uint32_t per_head = 0, per_head_inv = 0;     // units of one rotated head and ceil(2^32 / units)
    uint32_t per_copy = 0, per_copy_inv = 0;     // units of one head that is only copied (v)
    uint32_t page_shift = 0, pages = 0;
};

// ---- attention over the paged cache ----------------------------------------------------------------------------------
// Sequence s has the token rows offsets[s] .. offsets[s + 1] and kv_lens[s] keys of its own, its new tokens' included, on the
// pages of its row of the page table; keys 0 .. prefix_len of every sequence are the shared prefix.  A launch covers a list of
// work entries: the sequences with their prefix and own keys, the sequences with their own keys only, or the prefix against all rows at
// once.  An entry is cut into segments: a tile of `row_tile` rows (token, head of the group) of one kv head, against the key
// tiles that any of its rows sees.  The workgroups take equal runs of the resulting units: `lead` units for beginning a segment,
// then one for each of its key tiles; row tiles ascending, within them the kv heads, within them the units.  Where there are enough
// segments for that, each workgroup takes one.  The prefix's segments are all alike and are cut into equal parts instead, a workgroup
// each.
constexpr uint32_t kKeyTile = 32;
enum AttentionPart : uint32_t { kWholeSequences = 0, kOwnKeys = 1, kPrefix = 2 };

// A segment whose parts several workgroups left, noted under the number of the first of them, whose part begins it.
struct AttentionCut {
    uint32_t last;                 // the last of the workgroups, 0: the workgroup begins no such segment
    uint32_t kv_head, first_token, row0, rows;   // rows row0 .. row0 + rows of the entry that has its tokens from first_token on
    uint32_t unused[3];
};

// Ends a row of AttentionArgs::rows: of a segment that one workgroup finished, or where the parts of it are.
struct alignas(16) AttentionRowEnd {
    float max, sum;
    uint32_t piece;                // the first part's slot
    uint32_t parts_row;            // parts << 8 | row within the tile
};

struct AttentionArgs {
    const uint16_t* q = nullptr;
    const uint16_t* k_cache = nullptr;
    const uint16_t* v_cache = nullptr;
    const int32_t* page_table = nullptr;
    const int32_t* kv_lens = nullptr;
    const int32_t* offsets = nullptr;
    const int32_t* prefix_table = nullptr;
    const int32_t* prefix_len = nullptr;
    uint16_t* out = nullptr;
    float* pieces = nullptr;       // slots of [row_tile] (max, sum), [row_tile][dim]
    float* rows = nullptr;         // not kWholeSequences: [dim] and an AttentionRowEnd a (token, head)
    AttentionCut* cuts = nullptr;  // kWholeSequences: one a workgroup
    uint32_t tokens = 0, sequences = 0, heads = 0, kv_heads = 0, group = 0;
    uint32_t pages = 0, page_shift = 0, pages_per_sequence = 0, prefix_pages = 0;
    uint32_t window = 0, q_stride = 0, workgroups = 0, part = 0;
    uint32_t row_tile = 0;
    uint32_t slots = 0;
    uint32_t rounds = 1;           // kPrefix: workgroups times rounds that a launch has at most
    uint32_t lead = 0;             // what beginning a segment costs, in key tiles
    uint32_t least_units = 1;      // a workgroup takes at least this many units (kPrefix: key tiles)
    uint32_t whole_from = ~0u;     // segments from which on each workgroup takes one
    float scale_log2 = 0;          // |scale| * log2(e)
    uint32_t flip_q = 0;           // 0x80008000 for a negative scale
};

struct AttentionJoinArgs { AttentionArgs own, front; };

SMELT_HD uint32_t piece_floats(uint32_t row_tile, uint32_t dim) { return row_tile * (dim + 2); }
SMELT_HD uint32_t clamp_count(int32_t v, uint32_t most) { return v < 0 ? 0u : ((uint32_t)v > most ? most : (uint32_t)v); }
SMELT_HD uint32_t attention_entries(const AttentionArgs& a) { return a.part == kPrefix ? 1u : a.sequences; }

// One work entry: its rows and its two runs of keys.
struct AttentionEntry {
    uint32_t first_token = 0, tokens = 0;
    uint32_t row_tiles = 0;
    uint32_t prefix = 0;                // prefix length, covered by this entry or not
    uint32_t front = 0, own = 0;        // keys of the prefix run and of the sequence's own run
    uint32_t front_tiles = 0, tiles = 0;
    int32_t sequence = -1;              // -1: the prefix against all rows
};

struct AttentionPlainLoad { SMELT_HD int32_t operator()(const int32_t* p, uint32_t i) const { return p[i]; } };
template <class Load = AttentionPlainLoad>
SMELT_HD AttentionEntry attention_entry(const AttentionArgs& a, uint32_t index, Load load = Load()) {
    AttentionEntry e;
    const uint32_t page = 1u << a.page_shift;
    e.prefix = a.prefix_len ? clamp_count(load(a.prefix_len, 0), a.prefix_pages * page) : 0u;
    if (a.part == kPrefix) {
        e.tokens = e.prefix ? clamp_count(load(a.offsets, a.sequences), a.tokens) : 0u;
        e.front = e.prefix;
    } else {
        const uint32_t lo = clamp_count(load(a.offsets, index), a.tokens), hi = clamp_count(load(a.offsets, index + 1), a.tokens);
        e.sequence = (int32_t)index;
        e.first_token = lo;
        e.tokens = hi > lo ? hi - lo : 0u;
        e.own = clamp_count(load(a.kv_lens, index), a.pages_per_sequence * page);
        if (a.part == kWholeSequences) e.front = e.prefix;
    }
    e.front_tiles = (e.front + kKeyTile - 1) / kKeyTile;
    e.tiles = e.front_tiles + (e.own + kKeyTile - 1) / kKeyTile;
    e.row_tiles = (e.tokens * a.group + a.row_tile - 1) / a.row_tile;
    return e;
}

// Keys, counted from the prefix's first, that the rows first .. first + count of a sequence's entry see: some row those of [lo, hi), every
// row those of [all_lo, all_hi).  (Positions stay below 2^31.)
struct AttentionSpan { int32_t lo, hi, all_lo, all_hi; };
SMELT_HD AttentionSpan attention_span(const AttentionArgs& a, const AttentionEntry& e, uint32_t first, uint32_t count) {
    const int32_t zero = (int32_t)(e.prefix + e.own) - (int32_t)e.tokens;       // position of the entry's first row
    const uint32_t last = (first + count - 1) / a.group;
    const int32_t p0 = zero + (int32_t)(first / a.group), p1 = zero + (int32_t)(last < e.tokens ? last : e.tokens - 1);
    AttentionSpan s{0, p1 + 1, 0, p0 + 1};
    // (a window that a position is within hides nothing of it; the differences stay at 0 and above)
    if (a.window && p0 >= (int32_t)a.window) s.lo = p0 - (int32_t)a.window + 1;
    if (a.window && p1 >= (int32_t)a.window) s.all_lo = p1 - (int32_t)a.window + 1;
    return s;
}

// Key tiles lo .. hi of a row tile: those that a row of it sees, one at least (rows that see nothing are still written).
struct AttentionTiles { uint32_t lo, hi; };
SMELT_HD uint32_t attention_tile_of(const AttentionEntry& e, uint32_t key, uint32_t round) {   // round 0: the tile that holds a key, kKeyTile - 1: the tiles before one
    const bool front = key < e.prefix + (round ? 1u : 0u);
    return front ? (e.front ? (key + round) / kKeyTile : 0u) : e.front_tiles + (key - e.prefix + round) / kKeyTile;
}
SMELT_HD AttentionTiles attention_tiles(const AttentionArgs& a, const AttentionEntry& e, uint32_t row_tile) {
    AttentionTiles t{0, e.tiles};
    if (e.sequence >= 0) {
        const AttentionSpan s = attention_span(a, e, row_tile * a.row_tile, a.row_tile);
        t.hi = s.hi <= 0 ? 0u : attention_tile_of(e, (uint32_t)s.hi < e.prefix + e.own ? (uint32_t)s.hi : e.prefix + e.own, kKeyTile - 1);
        if (s.lo > 0) t.lo = attention_tile_of(e, (uint32_t)s.lo, 0);
    }
    if (t.lo >= t.hi) { t.lo = t.lo < e.tiles ? t.lo : 0; t.hi = t.lo + 1; }
    return t;
}

// (the host refuses shapes whose units could pass 2^31)
SMELT_HD uint32_t attention_units(const AttentionArgs& a, const AttentionEntry& e) {
    uint32_t n = 0;
#pragma unroll 1
    for (uint32_t r = 0; r < e.row_tiles; ++r) { const AttentionTiles t = attention_tiles(a, e, r); n += t.hi - t.lo + a.lead; }
    return n * a.kv_heads;
}
SMELT_HD uint32_t attention_segments(const AttentionArgs& a, const AttentionEntry& e) { return a.kv_heads * e.row_tiles; }

// How the units fall to the launch's workgroups: runs of `each`, the first `longer` of them one longer; or a segment each.
struct AttentionSplit { uint32_t units, groups, each, longer; bool whole; };
SMELT_HD AttentionSplit attention_split(const AttentionArgs& a, uint32_t units, uint32_t segments) {
    AttentionSplit s{units, 0, 0, 0, segments >= a.whole_from};
    const uint32_t most = units / a.least_units + (units % a.least_units != 0);
    s.groups = s.whole ? segments : (most < a.workgroups ? most : a.workgroups);
    if (s.groups) { s.each = units / s.groups; s.longer = units - s.each * s.groups; }
    return s;
}
// first unit of workgroup w
SMELT_HD uint32_t attention_start(const AttentionSplit& s, uint32_t w) { return w * s.each + (w < s.longer ? w : s.longer); }
// the workgroup whose run holds unit u
SMELT_HD uint32_t attention_owner(const AttentionSplit& s, uint32_t u) {
    const uint32_t border = s.longer * (s.each + 1);
    return u < border ? u / (s.each + 1) : s.longer + (u - border) / s.each;
}

// The parts that the prefix's segments are cut into (0: no rows): one, two ... workgroups for every place the machine has, whichever
// ends first, `lead` being what a part costs besides its key tiles.
SMELT_HD uint32_t attention_parts(const AttentionArgs& a, const AttentionEntry& e) {
    const uint32_t segments = attention_segments(a, e), tiles = e.front_tiles;
    if (segments == 0) return 0;
    uint32_t most = a.slots / segments, best = 1, cost = ~0u;
    const uint32_t long_enough = tiles / a.least_units;
    most = most < long_enough ? most : long_enough;
    for (uint32_t r = 1; r <= a.rounds; ++r) {
        uint32_t parts = r * a.workgroups / segments;
        parts = parts < most ? parts : most;
        parts = parts ? parts : 1u;
        const uint32_t took = (segments * parts + a.workgroups - 1) / a.workgroups * ((tiles + parts - 1) / parts + a.lead);
        if (took < cost) { cost = took; best = parts; }
    }
    return best;
}
// What workgroup w of a prefix launch takes.  The row tiles that read the same keys are neighbours, and neighbours are the workgroups that
// share a second-level cache (every eighth).
struct AttentionJob { uint32_t row_tile, kv_head, part; bool some; };
SMELT_HD AttentionJob attention_job(const AttentionArgs& a, const AttentionEntry& e, uint32_t parts, uint32_t w) {
    const uint32_t jobs = attention_segments(a, e) * parts, each = (jobs + 7) / 8, job = (w % 8) * each + w / 8;
    AttentionJob j{0, 0, 0, w / 8 < each && job < jobs};
    if (j.some) {
        j.row_tile = job % e.row_tiles;
        const uint32_t rest = job / e.row_tiles;
        j.kv_head = rest / parts;
        j.part = rest - j.kv_head * parts;
    }
    return j;
}

// ---- verification of drafted tokens ----------------------------------------------------------------------------------
// A row's logits are cut into `runs` runs of `span` (a multiple of kVerifyStep), each the work of one wave; the launches leave a
// record per run.
constexpr uint32_t kVerifyStep = 512;      // logits that a wave loads 16 bytes at a time
constexpr uint32_t kVerifyMaxSpan = 4096;  // four logits a thread of the last launch

struct VerifyStat {
    float top;          // largest logit of the run, -inf when there is none
    float sum;          // sum of exp((logit - top) / temperature)
};

// what the second launch leaves of a sequence
struct VerifyChoice {
    uint32_t taken;     // accepted drafts
    uint32_t where;     // greedy: the token to draw (~0: none)
    float top, draft_top;   // largest logits of the chosen row
};

struct VerifyArgs {
    const uint16_t* target = nullptr;
    const uint16_t* draft = nullptr;         // null: the drafts are given, with certainty
    const int32_t* draft_tokens = nullptr;
    const int32_t* offsets = nullptr;
    const float* u_accept = nullptr;
    const float* u_sample = nullptr;
    const float* temperature = nullptr;
    int32_t* tokens = nullptr;
    int32_t* counts = nullptr;
    VerifyStat* stats = nullptr;             // [2][rows][runs]: target, draft
    uint32_t* where = nullptr;               // [rows][runs]: lowest index of the target run's largest logit (greedy rows)
    double* sums = nullptr;                  // [sequences][3][runs]: target, draft, leftover of the chosen row
    VerifyChoice* choice = nullptr;          // [sequences]
    uint32_t rows = 0, sequences = 0, vocab = 0, stride = 0;
    uint32_t runs = 0, span = 0, vector = 0;
};

SMELT_HD uint32_t reciprocal(uint32_t d) { return d <= 1 ? 0u : (uint32_t)((0x100000000ull + d - 1) / d); }

}  // namespace smelt_serving
