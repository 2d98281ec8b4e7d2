// Host build of the attention's work partition, for the CPU tests.
#include <vector>

#include "../smelt_amd/csrc/kernels/serving_args.hpp"

using namespace smelt_serving;

extern "C" {

// entry: {first_token, tokens, row_tiles, front, own, front_tiles, key_tiles, sequence}; returns the entry count
int check_entries(const int32_t* offsets, const int32_t* lens, int sequences, int tokens, int group, int kv_heads, int page_shift,
                  int pages_per_sequence, const int32_t* prefix_len, int prefix_pages, int cascade, int64_t* out, uint64_t* units) {
    AttentionArgs a;
    a.offsets = offsets; a.kv_lens = lens; a.sequences = sequences; a.tokens = tokens; a.group = group; a.kv_heads = kv_heads;
    a.page_shift = page_shift; a.pages_per_sequence = pages_per_sequence; a.prefix_len = prefix_len; a.prefix_pages = prefix_pages; a.cascade = cascade;
    uint64_t total = 0;
    for (int i = 0; i < sequences + cascade; ++i) {
        const AttentionEntry e = attention_entry(a, i);
        const int64_t f[8] = {e.first_token, e.tokens, e.row_tiles, e.front, e.own, e.front_tiles, e.key_tiles, e.sequence};
        for (int k = 0; k < 8; ++k) out[8 * i + k] = f[k];
        total += attention_units(a, e);
    }
    *units = total;
    return sequences + cascade;
}

// every unit has one owner, owners are in order, and the owner's run holds the unit; 0 or the first bad unit + 1
uint64_t check_owners(uint64_t units, uint32_t workgroups) {
    AttentionArgs a;
    a.workgroups = workgroups;
    const uint32_t groups = attention_groups(a, units);
    if (groups == 0 || groups > workgroups) return 1;
    if (attention_start(units, groups, 0) != 0 || attention_start(units, groups, groups) != units) return 1;
    for (uint64_t u = 0; u < units; ++u) {
        const uint32_t w = attention_owner(units, groups, u);
        if (w >= groups || attention_start(units, groups, w) > u || attention_start(units, groups, w + 1) <= u) return u + 1;
    }
    return 0;
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
