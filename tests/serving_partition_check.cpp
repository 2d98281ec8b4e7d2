// Host build of the attention's work partition, for the CPU tests.
#include <vector>

#include "../smelt_amd/csrc/kernels/serving_args.hpp"

using namespace smelt_serving;

extern "C" {

// entry: {first_token, tokens, row_tiles, front, own, front_tiles, tiles, sequence}; tiles: {lo, hi} of each row tile of each entry, in
// order; returns the entry count
int check_entries(const int32_t* offsets, const int32_t* lens, int sequences, int tokens, int group, int kv_heads, int page_shift,
                  int pages_per_sequence, const int32_t* prefix_len, int prefix_pages, int part, int row_tile, int window, int64_t* out,
                  int64_t* tiles, uint64_t* units) {
    AttentionArgs a;
    a.offsets = offsets; a.kv_lens = lens; a.sequences = sequences; a.tokens = tokens; a.group = group; a.kv_heads = kv_heads;
    a.page_shift = page_shift; a.pages_per_sequence = pages_per_sequence; a.prefix_len = prefix_len; a.prefix_pages = prefix_pages;
    a.part = part; a.row_tile = row_tile; a.window = window;
    uint64_t total = 0;
    const int n = (int)attention_entries(a);
    for (int i = 0; i < n; ++i) {
        const AttentionEntry e = attention_entry(a, i);
        const int64_t f[8] = {e.first_token, e.tokens, e.row_tiles, e.front, e.own, e.front_tiles, e.tiles, e.sequence};
        for (int k = 0; k < 8; ++k) out[8 * i + k] = f[k];
        for (uint32_t r = 0; r < e.row_tiles; ++r) {
            const AttentionTiles t = attention_tiles(a, e, r);
            *tiles++ = t.lo;
            *tiles++ = t.hi;
        }
        total += attention_units(a, e);
    }
    *units = total;
    return n;
}

// every unit has one owner, owners are in order, and the owner's run holds the unit; 0 or the first bad unit + 1
uint64_t check_owners(uint32_t units, uint32_t workgroups, uint32_t least) {
    AttentionArgs a;
    a.workgroups = workgroups;
    a.least_units = least;
    const AttentionSplit s = attention_split(a, units, 1);
    if (s.groups == 0 || s.groups > workgroups || s.whole) return 1;
    if (attention_start(s, 0) != 0 || attention_start(s, s.groups) != units) return 1;
    for (uint32_t u = 0; u < units; ++u) {
        const uint32_t w = attention_owner(s, u);
        if (w >= s.groups || attention_start(s, w) > u || attention_start(s, w + 1) <= u) return (uint64_t)u + 1;
    }
    return 0;
}

// a prefix launch: parts of each segment, and what each of `grid` workgroups takes, {row_tile, kv_head, part} a workgroup that has some
// (in order); returns how many have
int check_jobs(const int32_t* offsets, int tokens, int sequences, int group, int kv_heads, int prefix, int row_tile, uint32_t workgroups, uint32_t rounds,
               uint32_t slots, uint32_t least, uint32_t lead, uint32_t grid, uint32_t* parts, int32_t* jobs) {
    AttentionArgs a;
    const int32_t lens = 0;
    a.offsets = offsets; a.kv_lens = &lens; a.sequences = sequences; a.tokens = tokens; a.group = group; a.kv_heads = kv_heads;
    a.page_shift = 4; a.pages_per_sequence = 1; a.prefix_len = &prefix; a.prefix_pages = (prefix + 15) / 16; a.part = kPrefix;
    a.row_tile = row_tile; a.workgroups = workgroups; a.rounds = rounds; a.slots = slots; a.least_units = least; a.lead = lead;
    const AttentionEntry e = attention_entry(a, 0);
    *parts = attention_parts(a, e);
    int n = 0;
    for (uint32_t w = 0; w < grid; ++w) {
        const AttentionJob j = attention_job(a, e, *parts, w);
        if (!j.some) continue;
        jobs[3 * n] = j.row_tile; jobs[3 * n + 1] = j.kv_head; jobs[3 * n + 2] = j.part;
        ++n;
    }
    return n;
}

uint32_t check_reciprocal(uint32_t d, uint32_t most) {
    const uint64_t inv = reciprocal(d);
    for (uint32_t n = 0; n <= most; ++n) {
        const uint32_t q = d <= 1 ? n : (uint32_t)((n * inv) >> 32);
        if (q != n / d) return n + 1;
    }
    return 0;
}
}
