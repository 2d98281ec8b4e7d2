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
    uint32_t tokens_per_group = 1;     // tokens of one workgroup
    uint32_t per_token = 0, per_token_inv = 0;   // units of one token and ceil(2^32 / units)
    uint32_t per_head = 0, per_head_inv = 0;     // units of one rotated head
    uint32_t per_copy = 0, per_copy_inv = 0;     // units of one head that is only copied (v)
    uint32_t page_shift = 0, pages = 0;
};

// ---- attention over the paged cache ----------------------------------------------------------------------------------
// Sequence s has the token rows offsets[s] .. offsets[s + 1] and kv_lens[s] keys of its own, its new tokens' included, on the
// pages of its row of the page table; keys 0 .. prefix_len of every sequence are the shared prefix.  A launch covers a list
// of work entries: with `cascade` entry 0 is the prefix against all rows at once and entry s + 1 the sequence's own keys; without it
// entry s is the sequence's prefix keys and own keys.  An entry is cut into (kv head, tile of kRowTile rows) segments of `key_tiles`
// tiles of kKeyTile keys, in that order, and the workgroups take equal runs of the resulting units.
constexpr uint32_t kRowTile = 32;
constexpr uint32_t kKeyTile = 32;
constexpr uint32_t kTilesPerGroup = 4;      // a workgroup takes at least this many key tiles: one for each of its waves

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
    float* pieces = nullptr;       // two slots a workgroup: [kRowTile] max, [kRowTile] sum, [kRowTile][dim]
    float* rows = nullptr;         // cascade: whole segments, a row of (dim + 4) a (token, head): [dim], max, sum
    uint32_t tokens = 0, sequences = 0, heads = 0, kv_heads = 0, group = 0;
    uint32_t pages = 0, page_shift = 0, pages_per_sequence = 0, prefix_pages = 0;
    uint32_t window = 0, q_stride = 0, workgroups = 0, cascade = 0;
    float scale_log2 = 0;          // scale * log2(e)
};

SMELT_HD uint32_t piece_floats(uint32_t dim) { return kRowTile * (dim + 2); }
SMELT_HD uint32_t clamp_count(int32_t v, uint32_t most) { return v < 0 ? 0u : ((uint32_t)v > most ? most : (uint32_t)v); }

// One work entry: rows first_row .. first_row + rows of the launch's tokens (times `group` heads), its two runs of keys.
struct AttentionEntry {
    uint32_t first_token = 0, tokens = 0;
    uint32_t row_tiles = 0;
    uint32_t front = 0, own = 0;        // keys of the prefix run and of the sequence's own run
    uint32_t front_tiles = 0, key_tiles = 0;
    int32_t sequence = -1;              // -1: the prefix against all rows
};

SMELT_HD AttentionEntry attention_entry(const AttentionArgs& a, uint32_t index) {
    AttentionEntry e;
    const uint32_t page = 1u << a.page_shift;
    const uint32_t front = a.prefix_len ? clamp_count(a.prefix_len[0], a.prefix_pages * page) : 0u;
    if (a.cascade && index == 0) {
        e.tokens = clamp_count(a.offsets[a.sequences], a.tokens);
        e.front = front;
        e.front_tiles = e.key_tiles = (front + kKeyTile - 1) / kKeyTile;
    } else {
        const uint32_t s = index - a.cascade;
        const uint32_t lo = clamp_count(a.offsets[s], a.tokens), hi = clamp_count(a.offsets[s + 1], a.tokens);
        e.sequence = (int32_t)s;
        e.first_token = lo;
        e.tokens = hi > lo ? hi - lo : 0u;
        e.own = clamp_count(a.kv_lens[s], a.pages_per_sequence * page);
        if (!a.cascade) e.front = front;
        e.front_tiles = (e.front + kKeyTile - 1) / kKeyTile;
        e.key_tiles = e.front_tiles + (e.own + kKeyTile - 1) / kKeyTile;
        if (e.key_tiles == 0) e.key_tiles = 1;   // rows that see nothing are still written
    }
    e.row_tiles = (e.tokens * a.group + kRowTile - 1) / kRowTile;
    return e;
}

SMELT_HD uint64_t attention_units(const AttentionArgs& a, const AttentionEntry& e) { return (uint64_t)a.kv_heads * e.row_tiles * e.key_tiles; }
SMELT_HD uint32_t attention_groups(const AttentionArgs& a, uint64_t units) {
    const uint64_t most = (units + kTilesPerGroup - 1) / kTilesPerGroup;
    return most < a.workgroups ? (uint32_t)most : a.workgroups;
}
// first unit of workgroup w of `groups`
SMELT_HD uint64_t attention_start(uint64_t units, uint32_t groups, uint32_t w) { return units * w / groups; }
// the workgroup whose run holds unit u
SMELT_HD uint32_t attention_owner(uint64_t units, uint32_t groups, uint64_t u) {
    uint32_t w = (uint32_t)(u * groups / units);
    while (w + 1 < groups && attention_start(units, groups, w + 1) <= u) ++w;
    while (w > 0 && attention_start(units, groups, w) > u) --w;
    return w;
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
