// Serving operators on the host: pipeline names, argument checks, launch plans.  No device is touched here.
#include "serving.hpp"

#include <algorithm>
#include <cmath>
#include <cstring>

#include "../../include/smelt_hip.h"

namespace smelt_host {

using namespace smelt_serving;

namespace {

// What beginning a segment of rows and keys costs, in key tiles (own keys of 64 sequences 38.8 / 37.5 / 37.6 us, one token 12.9 / 13.1 /
// 14.0 us with 2 / 4 / 8) ...
constexpr uint32_t kSegmentLead = 4;
// ... and a workgroup's part of the prefix, whose 13 to 15 us besides the tiles' 1.5 weigh where a second round is looked at.
constexpr uint32_t kPartLead = 8;

// "_d256" at `at`: the number behind the letters, and the position behind it
bool number_after(const std::string& s, const char* letters, size_t* at, uint32_t* out) {
    const size_t n = strlen(letters);
    if (s.compare(*at, n, letters) != 0) return false;
    size_t p = *at + n, q = p;
    while (q < s.size() && s[q] >= '0' && s[q] <= '9') ++q;
    if (q == p || q - p > 6) return false;
    *out = (uint32_t)std::stoul(s.substr(p, q - p));
    *at = q;
    return true;
}

bool take(const std::string& s, const char* word, size_t* at) {
    const size_t n = strlen(word);
    if (s.compare(*at, n, word) != 0) return false;
    *at += n;
    return true;
}

bool page_ok(uint32_t p) { return p == 16 || p == 32 || p == 64 || p == 128 || p == 256; }
uint32_t log2_of(uint32_t v) { uint32_t n = 0; while ((1u << n) < v) ++n; return n; }

}  // namespace

ResolveStatus resolve_serving(const std::string& entry, const char* act, ResolvedPipeline* out, std::string* why) {
    auto malformed = [&](const std::string& m) { *why = m + " in '" + entry + "'"; return kResolveMalformed; };
    const std::string t = std::string("_") + act;
    size_t at = 0;
    const bool append = take(entry, "paged_kv_append", &at);
    if (append || (take(entry, "rope", &at) && at < entry.size() && (entry[at] == '_'))) {
        const bool with_q = append && take(entry, "_q", &at);
        const bool interleaved = take(entry, "_interleaved", &at);
        if (!interleaved && !take(entry, "_half", &at)) return kResolveUnknown;
        uint32_t dim = 0, rot = 0, kv_heads = 0, page = 0;
        if (!number_after(entry, "_d", &at, &dim) || !number_after(entry, "_r", &at, &rot)) return kResolveUnknown;
        if (append && (!number_after(entry, "_kv", &at, &kv_heads) || !number_after(entry, "_p", &at, &page))) return kResolveUnknown;
        if (at != entry.size()) return kResolveUnknown;
        if (dim == 0 || dim > 1024) return malformed("head dimension must be 1 to 1024");
        if (rot > dim || rot % 2 != 0 || (!append && rot == 0)) return malformed("rotated dimensions must be even and at most the head's");
        out->kinds = append ? (with_q ? "PPPPPPPPPUUUUFUUUUUUUU" : "PPPPPPPUUUUFUUUUU") : "PPPPUUUUFUUU";
        out->appended = {dim, rot, interleaved ? 1u : 0u};
        if (append) {
            if (dim != 64 && dim != 128 && dim != 256) return malformed("cached heads hold 64, 128 or 256 values");
            if (kv_heads == 0 || kv_heads > 1024) return malformed("kv heads must be 1 to 1024");
            if (!page_ok(page)) return malformed("pages hold 16, 32, 64, 128 or 256 tokens");
            out->appended.push_back(kv_heads);
            out->appended.push_back(page);
        }
        out->family = append ? (with_q ? kFamPagedAppendQ : kFamPagedAppend) : kFamRope;
        const char* stem = append ? "smelt_paged_append_" : "smelt_rope_";
        out->serving_symbols = {std::string(stem) + "vec" + t, std::string(stem) + "any" + t};
        out->symbol = out->serving_symbols[0];
        return kResolveOk;
    }
    at = 0;
    if (take(entry, "paged_attention", &at)) {
        const bool shared = take(entry, "_shared", &at);
        uint32_t dim = 0, heads = 0, kv_heads = 0, page = 0;
        if (!number_after(entry, "_d", &at, &dim) || !number_after(entry, "_h", &at, &heads) || !number_after(entry, "_kv", &at, &kv_heads) ||
            !number_after(entry, "_p", &at, &page) || at != entry.size())
            return kResolveUnknown;
        if (dim != 64 && dim != 128 && dim != 256) return malformed("cached heads hold 64, 128 or 256 values");
        if (kv_heads == 0 || heads == 0 || heads > 1024 || heads % kv_heads != 0) return malformed("heads must be a multiple of kv heads, at most 1024");
        if (!page_ok(page)) return malformed("pages hold 16, 32, 64, 128 or 256 tokens");
        out->family = shared ? kFamPagedAttentionShared : kFamPagedAttention;
        out->kinds = shared ? "PPPPPPPPPUUUUUFUUUUUU" : "PPPPPPPUUUUFUUUUUU";
        out->appended = {dim, heads, kv_heads, page};
        const std::string tail = "_d" + std::to_string(dim) + t;
        for (const char* k : {"stream16", "stream32", "tiles", "join", "join_shared"}) out->serving_symbols.push_back(std::string("smelt_attention_") + k + tail);
        out->symbol = out->serving_symbols[0];
        return kResolveOk;
    }
    if (entry == "verify_drafts" || entry == "verify_drafts_given") {
        const bool given = entry != "verify_drafts";
        out->family = given ? kFamVerifyDraftsGiven : kFamVerifyDrafts;
        out->kinds = given ? "PPPPPPPPUUUU" : "PPPPPPPPPUUUU";
        for (const char* k : {"stats", "choose", "leftover", "draw"}) out->serving_symbols.push_back(std::string("smelt_verify_") + k + t);
        out->symbol = out->serving_symbols[0];
        return kResolveOk;
    }
    *why = "no HIP kernel named '" + entry + "'";
    return kResolveUnknown;
}

namespace {

struct Planner {
    const ResolvedPipeline& r;
    const uint32_t* value;
    const ServingDevice& dev;
    ServingPlan* plan;
    std::string* why;
    bool too_wide = false;      // a launch of more threads than one can have

    int fail(int code, const std::string& m) { *why = m; return code; }
    int bad(const std::string& m) { return fail(SMELT_HIP_ERR_UNSUPPORTED_GEOMETRY, m); }
    uint32_t U(size_t i) const { return value[i]; }
    float F(size_t i) const { float f; memcpy(&f, &value[i], 4); return f; }
    template <class T> T* P(int i) const { return static_cast<T*>(plan->operand[i].ptr); }
    void need(int i, size_t bytes, size_t align = 2, bool written = false) {
        ServingOperand& o = plan->operand[i];
        o.need = bytes; o.align = align; o.written = written;
        o.row = o.stride = 0;
    }
    // `tokens` rows of `count` 16-bit values at `stride`
    void need_rows(int i, uint32_t tokens, uint32_t count, uint32_t stride, bool written = false) {
        need(i, row_bytes(tokens, count, stride), 2, written);
        plan->operand[i].row = (size_t)count * 2;
        plan->operand[i].stride = (size_t)stride * 2;
    }
    template <class A> ServingStep& step(int kernel, const A& args, uint32_t gx, uint32_t gy, uint32_t gz, uint32_t threads, size_t lds) {
        static_assert(sizeof(A) <= kServingArgBytes, "argument block");
        too_wide = too_wide || (uint64_t)gx * threads > 0xFFFFFFFFull;
        ServingStep& s = plan->step[plan->steps++];
        s.kernel = kernel;
        s.grid[0] = gx; s.grid[1] = gy; s.grid[2] = gz;
        s.threads = threads;
        s.lds = lds;
        s.arg_bytes = sizeof(A);
        memcpy(s.args, &args, sizeof(A));
        return s;
    }
    // bytes of `tokens` rows of `count` 16-bit values at `stride`
    static size_t row_bytes(uint32_t tokens, uint32_t count, uint32_t stride) { return tokens ? ((size_t)(tokens - 1) * stride + count) * 2 : 0; }
    // Whether two operands share a byte.  Rows at one stride (q, k and v within the rows of a fused projection) are compared row by row: row
    // j of y lies distance + (j - i) * stride behind row i of x, and the least j - i is looked for that is not wholly before it.
    static bool meet(const ServingOperand& x, const ServingOperand& y) {
        const char *a = static_cast<const char*>(x.ptr), *b = static_cast<const char*>(y.ptr);
        if (!(a < b + y.need && b < a + x.need)) return false;
        if (x.stride == 0 || x.stride != y.stride) return true;
        typedef __int128 wide;
        const wide stride = x.stride, distance = (wide)(intptr_t)b - (wide)(intptr_t)a, from = -(wide)y.row - distance;
        const wide rows_x = (x.need - x.row) / x.stride, rows_y = (y.need - y.row) / y.stride;      // less one each
        wide k = (from >= 0 ? from / stride : -((-from + stride - 1) / stride)) + 1;
        k = k > -rows_x ? k : -rows_x;
        return k <= rows_y && distance + k * stride < (wide)x.row;
    }
    // operand `w` is written: it must not overlap any other one, but for `same`, which may be the very same rows
    int apart(int w, int same = -1, bool same_rows = false) {
        const ServingOperand& o = plan->operand[w];
        for (int i = 0; i < plan->operands; ++i) {
            const ServingOperand& x = plan->operand[i];
            if (i == w || x.need == 0 || o.need == 0) continue;
            if (i == same && same_rows && x.ptr == o.ptr) continue;
            if (meet(o, x))
                return fail(SMELT_HIP_ERR_INVALID_ARGUMENT, "output argument " + std::to_string(w) + " overlaps argument " + std::to_string(i));
        }
        return 0;
    }

    int rope();
    int attention();
    int verify();
};

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int Planner::rope() {
    const bool append = r.family != kFamRope, with_q = r.family == kFamPagedAppendQ;
    // first value argument, and the shape behind the record's own values
    const size_t o = r.family == kFamRope ? 4 : (with_q ? 9 : 7);
    const size_t shape = o + (r.family == kFamRope ? 5 : (with_q ? 8 : 5));
    RopeArgs a;
    a.tokens = U(o);
    a.dim = U(shape); a.rot = U(shape + 1); a.interleaved = U(shape + 2);
    if (a.tokens == 0) return 0;
    const uint32_t half = a.rot / 2;
    uint32_t q_heads = 0, kv_heads = 0, page = 0;
    a.positions = P<int32_t>(2);
    if (!append) {
        q_heads = U(o + 1);
        a.amplitude = F(o + 4);
        a.q.src = P<uint16_t>(0); a.q.dst = P<uint16_t>(1);
        a.q.src_stride = U(o + 2); a.q.dst_stride = U(o + 3);
        a.table = P<double>(3);
        need_rows(0, a.tokens, q_heads * a.dim, a.q.src_stride);
        need_rows(1, a.tokens, q_heads * a.dim, a.q.dst_stride, true);
        need(2, (size_t)a.tokens * 4, 4);
        need(3, (size_t)half * 8, 8);
    } else {
        kv_heads = U(shape + 3); page = U(shape + 4);
        a.k.src_stride = U(o + 1); a.v.src_stride = U(o + 2);
        a.pages = U(o + 3);
        a.amplitude = F(o + 4);
        a.page_shift = log2_of(page);
        a.k.src = P<uint16_t>(0); a.v.src = P<uint16_t>(1);
        a.slots = P<int32_t>(3);
        a.table = P<double>(4);
        a.k.dst = P<uint16_t>(5); a.v.dst = P<uint16_t>(6);
        a.k.heads = a.v.heads = kv_heads;
        if (a.pages == 0 || (uint64_t)a.pages * page > 0x7FFFFFFFull) return bad("the pool must hold 1 to 2^31 - 1 tokens");
        const size_t cache = (size_t)a.pages * page * kv_heads * a.dim * 2;
        need_rows(0, a.tokens, kv_heads * a.dim, a.k.src_stride);
        need_rows(1, a.tokens, kv_heads * a.dim, a.v.src_stride);
        need(2, half ? (size_t)a.tokens * 4 : 0, 4);
        need(3, (size_t)a.tokens * 4, 4);
        need(4, (size_t)half * 8, 8);
        need(5, cache, 16, true);
        need(6, cache, 16, true);
        if (with_q) {
            q_heads = U(o + 5);
            a.q.src = P<uint16_t>(7); a.q.dst = P<uint16_t>(8);
            a.q.src_stride = U(o + 6); a.q.dst_stride = U(o + 7);
            need_rows(7, a.tokens, q_heads * a.dim, a.q.src_stride);
            need_rows(8, a.tokens, q_heads * a.dim, a.q.dst_stride, true);
        }
        if (a.k.src_stride < kv_heads * a.dim || a.v.src_stride < kv_heads * a.dim) return bad("a row stride is shorter than its heads");
    }
    if (!append || with_q) {
        if (q_heads == 0 || q_heads > 1024) return bad("heads must be 1 to 1024");
        if (a.q.src_stride < q_heads * a.dim || a.q.dst_stride < q_heads * a.dim) return bad("a row stride is shorter than its heads");
        const int src = append ? 7 : 0, dst = append ? 8 : 1;
        if (int e = apart(dst, src, a.q.src_stride == a.q.dst_stride)) return e;
    }
    if (append) {
        if (int e = apart(5)) return e;
        if (int e = apart(6)) return e;
    }
    a.q.heads = q_heads;
    // 16-byte pieces where every row, piece and pair of pieces is one; single values otherwise
    bool vec = a.dim % 8 == 0 && a.rot % (a.interleaved ? 8 : 16) == 0;
    auto pieces = [&](const RopeRows& x, bool rows) { return !x.heads || (aligned16(x.src) && x.src_stride % 8 == 0 && (!rows || (aligned16(x.dst) && x.dst_stride % 8 == 0))); };
    vec = vec && pieces(a.q, true) && pieces(a.k, false) && pieces(a.v, false);
    a.per_copy = vec ? a.dim / 8 : a.dim;
    a.per_head = vec ? a.rot / (a.interleaved ? 8 : 16) + (a.dim - a.rot) / 8 : half + (a.dim - a.rot);
    a.q.units = q_heads * a.per_head;
    a.k.units = kv_heads * a.per_head;
    a.v.units = kv_heads * a.per_copy;
    a.per_token = a.q.units + a.k.units + a.v.units;
    if (a.per_token > kRopeMaxPerToken) return bad("one token has more than " + std::to_string(kRopeMaxPerToken) + " pieces to move");
    a.per_head_inv = reciprocal(a.per_head);
    a.q_units_inv = reciprocal(a.q.units);
    a.v_units_inv = reciprocal(a.v.units);
    a.per_copy_inv = reciprocal(a.per_copy);
    // Append: a workgroup takes up to four tokens when there are enough for two workgroups a compute unit all the same, so that what
    // neighbouring tokens put into a key page (16 bytes each) makes 64 contiguous bytes (8000 tokens of 8 heads of 128: 26.2 / 18.3 /
    // 19.9 us at 1 / 4 / 8 tokens).  Rows: two, so that few heads keep the threads busy (8192 tokens of 32 heads of 128: 27.5 / 27.7 / 29.0
    // us at 1 / 2 / 4).  n * d of the reciprocal division stays below 2^32 (65535 pieces a token, 65536 units a workgroup).
    uint32_t group = 1;
    const uint32_t most = append ? 4 : 2, least = (append ? 2 : 4) * dev.compute_units;
    while (group < most && a.tokens / (group * 2) >= least && (uint64_t)group * 2 * a.per_token <= 65536) group *= 2;
    a.tokens_per_group = group;
    step(vec ? 0 : 1, a, (a.tokens + group - 1) / group, 1, 1, kRopeThreads, (size_t)group * half * 8 + 64);
    return 0;
}

int Planner::attention() {
    const bool shared = r.family == kFamPagedAttentionShared;
    const size_t o = shared ? 9 : 7, shape = o + (shared ? 8 : 7);
    size_t v = o;
    AttentionArgs a;
    a.tokens = U(v++); a.sequences = U(v++); a.pages = U(v++); a.pages_per_sequence = U(v++);
    if (shared) a.prefix_pages = U(v++);
    const float scale = F(v++);
    a.window = U(v++); a.q_stride = U(v++);
    const uint32_t dim = U(shape), page = U(shape + 3);
    a.heads = U(shape + 1); a.kv_heads = U(shape + 2);
    a.group = a.heads / a.kv_heads;
    a.page_shift = log2_of(page);
    if (a.tokens == 0 || a.sequences == 0) return 0;
    if (a.pages == 0 || (uint64_t)a.pages * page > 0x7FFFFFFFull) return bad("the pool must hold 1 to 2^31 - 1 tokens");
    if (a.pages_per_sequence == 0) return bad("a sequence needs a page table of one page at least");
    if (((uint64_t)a.pages_per_sequence + a.prefix_pages) * page + a.tokens > 0x7FFFFFFFull) return bad("positions pass 2^31 - 1");
    if ((uint64_t)a.tokens * a.heads > 0x7FFFFFFFull) return bad("more than 2^31 - 1 rows");
    if (a.q_stride < a.heads * dim) return bad("q's row stride is shorter than its heads");
    if (!std::isfinite(scale)) return bad("the scale must be finite");
    if (a.window > 0x7FFFFFFFu) return bad("the window passes 2^31 - 1");
    // (a scale of zero weighs every key alike; the smallest normal number does the same and keeps a hidden key's -inf one)
    a.scale_log2 = std::fmax(std::fabs(scale) * 1.4426950408889634f, 1.2e-38f);
    a.flip_q = scale < 0.0f ? 0x80008000u : 0u;
    const size_t cache = (size_t)a.pages * page * a.kv_heads * dim * 2;
    need_rows(0, a.tokens, a.heads * dim, a.q_stride);
    need(1, cache, 16);
    need(2, cache, 16);
    need(3, (size_t)a.sequences * a.pages_per_sequence * 4, 4);
    need(4, (size_t)a.sequences * 4, 4);
    need(5, ((size_t)a.sequences + 1) * 4, 4);
    need(6, (size_t)a.tokens * a.heads * dim * 2, 8, true);
    if (shared) {
        need(7, (size_t)a.prefix_pages * 4, 4);
        need(8, 4, 4);
    }
    if (int e = apart(6)) return e;
    a.q = P<uint16_t>(0); a.k_cache = P<uint16_t>(1); a.v_cache = P<uint16_t>(2);
    a.page_table = P<int32_t>(3); a.kv_lens = P<int32_t>(4); a.offsets = P<int32_t>(5);
    a.out = P<uint16_t>(6);
    if (shared && a.prefix_pages) { a.prefix_table = P<int32_t>(7); a.prefix_len = P<int32_t>(8); }

    // The streaming kernel takes the sequences while they have few rows each (one tile of 16 or 32 rows on average), the prefix then
    // being read once against all rows; the tile kernel takes longer runs of rows, whose tiles read prefix and own keys alike.
    // 64 sequences of 6 rows, heads of 256, a prefix of 8192: 86 us, with tiles of 32 rows 93, with the tile kernel for prefix and own keys
    // 191.  24 sequences of 18 rows on average, heads of 128, a prefix of 2500: 67 us, with two tiles of 16 rows a sequence 69, with the
    // tile kernel 60 (24 short sequences fill the machine once, and one launch is less than three).  The host knows the mean of the rows and not
    // the lengths, so the rule does not see that case, nor a batch that mixes single tokens with a long prompt.
    const uint64_t rows = (uint64_t)a.tokens * a.group;
    const bool stream = rows <= (uint64_t)32 * a.sequences;
    const uint32_t tile_rows = dim == 256 ? 128 : 256;
    auto row_tile = [&](uint64_t of, uint64_t over) { return of <= 16 * over ? 16u : (of <= 32 * over ? 32u : tile_rows); };
    // The parts of cut segments live in the context's workspace, a workgroup leaving two at most (of its first and its last segment),
    // or one of the prefix's.
    const size_t row_region = (size_t)a.tokens * a.heads * (dim + 4) * 4;
    auto piece_bytes = [&](uint32_t r) { return (size_t)piece_floats(r, dim) * 4; };
    auto segments = [&](const AttentionArgs& x) { return ((rows + x.row_tile - 1) / x.row_tile + (x.part == kPrefix ? 0 : x.sequences)) * x.kv_heads; };   // there can be
    auto lay_out = [&](AttentionArgs& x, uint32_t r, size_t room) {
        x.row_tile = r;
        // workgroups that the register file holds
        const uint32_t per_cu = r == 16 ? (dim == 256 ? 2 : (dim == 128 ? 3 : 4)) : (r == 32 && dim != 256 ? 2 : 1);
        const size_t most = (size_t)dev.compute_units * per_cu;
        x.slots = (uint32_t)std::min<size_t>(2 * most, room / piece_bytes(r));
        if (x.part == kPrefix) {
            x.workgroups = (uint32_t)most;
            x.lead = kPartLead;
            x.least_units = 8;                // (24 sequences, a prefix of 2500: 68 / 67 / 72 us with parts of 3 / 8 / 16 key tiles at least)
            x.rounds = segments(x) > most / 4 ? 2 : 1;
        } else {
            x.workgroups = (uint32_t)std::min<size_t>(most, x.slots / 2);
            x.lead = kSegmentLead;
            x.least_units = x.lead + (r <= 32 ? 4 : 8);   // a key tile for each of four waves; stages to keep under way
        }
        // a segment each from three quarters of the workgroups on: no parts to write and join (two prompt chunks of 900 and 1024 tokens behind
        // up to 4000 keys, 248 segments: 138 us, in equal runs 150).  Not measured above the number of compute units, where the last
        // round may be mostly empty.
        x.whole_from = r <= 32 ? ~0u : std::max(1u, dev.compute_units * 3 / 4);
    };
    char* ws = static_cast<char*>(dev.workspace);
    auto main_step = [&](const AttentionArgs& x) {
        const uint32_t r = x.row_tile;
        // (as many as there can be segments, where each may take one)
        uint64_t grid = x.part == kPrefix ? (std::max<uint64_t>(segments(x), x.workgroups * x.rounds) + 7) / 8 * 8 : (r <= 32 ? x.workgroups : std::max<uint64_t>(segments(x), x.workgroups));
        grid = std::min<uint64_t>(grid, 0xFFFFFFFFull);       // (refused for its threads)
        if (r <= 32) step(r == 16 ? 0 : 1, x, (uint32_t)grid, 1, 1, 256, (size_t)4 * r * (dim + 4) * 4 + 9 * r * 4);
        else step(2, x, (uint32_t)grid, 1, 1, dim == 256 ? 256 : 512, (size_t)4 * (dim == 256 ? 1 : 2) * 2 * 32 * dim * 2);
    };
    // units are counted in 32 bits
    const uint64_t key_tiles = ((uint64_t)a.pages_per_sequence + a.prefix_pages) * page / kKeyTile + 2;
    const uint64_t row_tiles = rows / 16 + a.sequences + 1;
    if (row_tiles * a.kv_heads > 0x7FFFFFFFull / (key_tiles + kSegmentLead)) return bad("rows times keys pass 2^31 key tiles");
    const uint32_t own_rows = row_tile(rows, a.sequences), front_rows = row_tile(rows, 1);
    if (stream && shared && a.prefix_pages && 2 * row_region <= dev.workspace_bytes) {
        AttentionJoinArgs both;
        both.front = a; both.own = a;
        both.front.part = kPrefix; both.own.part = kOwnKeys;
        both.front.rows = reinterpret_cast<float*>(ws);
        both.own.rows = reinterpret_cast<float*>(ws + row_region);
        const size_t room = dev.workspace_bytes - 2 * row_region;
        lay_out(both.own, own_rows, room / 2);
        const size_t own_bytes = both.own.slots * piece_bytes(own_rows);
        lay_out(both.front, front_rows, room - own_bytes);
        if (both.own.workgroups) {
            both.own.pieces = reinterpret_cast<float*>(ws + 2 * row_region);
            both.front.pieces = reinterpret_cast<float*>(ws + 2 * row_region + own_bytes);
            main_step(both.front);
            main_step(both.own);
            step(4, both, a.tokens, a.kv_heads, 1, std::min(1024u, (a.group * dim / 4 + 63) / 64 * 64), 0);
            return 0;
        }
    }
    a.part = kWholeSequences;
    const size_t note_bytes = (size_t)dev.compute_units * 4 * sizeof(AttentionCut);       // (four workgroups a compute unit at most)
    if (dev.workspace_bytes < note_bytes) return bad("the workspace holds no part of a segment");
    a.cuts = reinterpret_cast<AttentionCut*>(ws);
    a.pieces = reinterpret_cast<float*>(ws + note_bytes);
    lay_out(a, own_rows, dev.workspace_bytes - note_bytes);
    if (a.workgroups == 0) return bad("the workspace holds no part of a segment");
    main_step(a);
    if (a.workgroups > 1) step(3, a, a.workgroups - 1, stream ? 2 : 8, 1, 256, 0);
    return 0;
}

int Planner::verify() {
    const bool given = r.family == kFamVerifyDraftsGiven;
    const int n = given ? 1 : 2;       // logits arguments
    const size_t o = n + 7;
    VerifyArgs a;
    a.rows = U(o); a.sequences = U(o + 1); a.vocab = U(o + 2); a.stride = U(o + 3);
    if (a.sequences == 0 || a.rows == 0) return 0;
    if (a.vocab == 0 || a.vocab > 0x7FFFFFF0u) return bad("the vocabulary must hold 1 to 2^31 - 17 tokens");
    if (a.stride < a.vocab) return bad("the row stride is shorter than the vocabulary");
    if (a.rows > 65535 || a.sequences > 65535) return bad("at most 65535 rows and sequences");
    need_rows(0, a.rows, a.vocab, a.stride);
    if (!given) need_rows(1, a.rows, a.vocab, a.stride);
    need(n, (size_t)a.rows * 4, 4);
    need(n + 1, ((size_t)a.sequences + 1) * 4, 4);
    need(n + 2, (size_t)a.rows * 4, 4);
    need(n + 3, (size_t)a.sequences * 4, 4);
    need(n + 4, (size_t)a.sequences * 4, 4);
    need(n + 5, (size_t)a.rows * 4, 4, true);
    need(n + 6, (size_t)a.sequences * 4, 4, true);
    if (int e = apart(n + 5)) return e;
    if (int e = apart(n + 6)) return e;
    a.target = P<uint16_t>(0);
    if (!given) a.draft = P<uint16_t>(1);
    a.draft_tokens = P<int32_t>(n); a.offsets = P<int32_t>(n + 1);
    a.u_accept = P<float>(n + 2); a.u_sample = P<float>(n + 3); a.temperature = P<float>(n + 4);
    a.tokens = P<int32_t>(n + 5); a.counts = P<int32_t>(n + 6);
    a.vector = a.stride % 8 == 0 && aligned16(a.target) && (given || aligned16(a.draft)) ? 1u : 0u;
    // runs of 512 logits up to 4096, as long as there are eight waves a compute unit (five rows of 151936: 26 us with runs of 512, 29
    // with runs of 4096)
    a.span = kVerifyMaxSpan;
    while (a.span > kVerifyStep && (uint64_t)a.rows * n * ((a.vocab + a.span - 1) / a.span) < 8ull * dev.compute_units) a.span /= 2;
    a.runs = (a.vocab + a.span - 1) / a.span;
    const size_t stats = (size_t)2 * a.rows * a.runs * sizeof(VerifyStat), sums = (size_t)a.sequences * 3 * a.runs * 8;
    const size_t where = (size_t)a.rows * a.runs * 4, all = stats + sums + (size_t)a.sequences * sizeof(VerifyChoice) + where;
    if (all > dev.workspace_bytes)
        return bad("the runs' records (" + std::to_string(all) + " bytes) exceed the workspace (" + std::to_string(dev.workspace_bytes) + " bytes)");
    char* ws = static_cast<char*>(dev.workspace);
    a.stats = reinterpret_cast<VerifyStat*>(ws);
    a.sums = reinterpret_cast<double*>(ws + stats);
    a.choice = reinterpret_cast<VerifyChoice*>(ws + stats + sums);
    a.where = reinterpret_cast<uint32_t*>(ws + stats + sums + (size_t)a.sequences * sizeof(VerifyChoice));
    const uint32_t groups = (a.runs + 3) / 4;
    step(0, a, groups, a.rows, (uint32_t)n, 256, 0);
    step(1, a, groups, a.sequences, 1, 256, 0);
    if (!given) step(2, a, groups, a.sequences, 1, 256, 0);
    step(3, a, a.sequences, 1, 1, 1024, 0);
    return 0;
}

}  // namespace

int plan_serving(const ResolvedPipeline& r, const uint32_t* value, const ServingDevice& dev, ServingPlan* plan, std::string* why) {
    plan->operands = 0;
    while (plan->operands < (int)r.kinds.size() && r.kinds[(size_t)plan->operands] == 'P') ++plan->operands;
    plan->steps = 0;
    Planner p{r, value, dev, plan, why};
    int e;
    switch (r.family) {
        case kFamRope:
        case kFamPagedAppend:
        case kFamPagedAppendQ: e = p.rope(); break;
        case kFamPagedAttention:
        case kFamPagedAttentionShared: e = p.attention(); break;
        case kFamVerifyDrafts:
        case kFamVerifyDraftsGiven: e = p.verify(); break;
        default: return p.bad("not a serving operator");
    }
    return e == 0 && p.too_wide ? p.bad("one launch of more than 2^32 - 1 threads") : e;
}

}  // namespace smelt_host
