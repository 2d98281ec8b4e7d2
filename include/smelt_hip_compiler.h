/*
 * smelt_hip_compiler.h — build-time half of the HIP backend: the pieces of SmeltCompiler that
 * decide which kernel a weight gets, where its bytes live in weights.bin, and which dispatch
 * records drive it.  Pure host code (no GPU needed); exported from the same libsmelt_hip.so.
 *
 * Each group cites the reference code it mirrors (paths relative to the Smelt repository).
 */
#ifndef SMELT_HIP_COMPILER_H
#define SMELT_HIP_COMPILER_H

#include <stddef.h>
#include <stdint.h>

#include "smelt_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- SmeltDType: Sources/SmeltSchema/SmeltManifest.swift:1613-1645 ------------------------ */
enum {
    SMELT_DTYPE_FP16 = 0,
    SMELT_DTYPE_FP32 = 1,
    SMELT_DTYPE_BF16 = 2,
    SMELT_DTYPE_INT32 = 3,
    SMELT_DTYPE_U4_LUT = 4,
    SMELT_DTYPE_AFFINE_U4 = 5,
    SMELT_DTYPE_BINARY1 = 6,
    SMELT_DTYPE_TERNARY2 = 7,
    SMELT_DTYPE_TURBO_QUANT_H = 8,
    SMELT_DTYPE_RAW = 9,
    SMELT_DTYPE_TRIT5 = 10, /* not in the reference: five base-3 digits per byte */
    SMELT_DTYPE_COUNT
};
/* manifest spelling ("affine_u4", "binary1", ...); NULL for an unknown value */
const char *smelt_dtype_name(int dtype);
int smelt_dtype_from_name(const char *name); /* -1 if unknown */

/* ---- MatvecKernelTable: Sources/SmeltCompiler/MatvecKernelTable.swift:51-284 --------------- */
enum { SMELT_ACT_FP16 = 0, SMELT_ACT_BF16 = 1, SMELT_ACT_FP32 = 2 };
enum { SMELT_SHAPE_GEMV = 0, SMELT_SHAPE_GEMM = 1, SMELT_SHAPE_GEMM_TN = 2 };
enum { SMELT_FUSION_NONE = 0, SMELT_FUSION_DUAL_MATVEC = 1, SMELT_FUSION_GATE_UP_SWIGLU = 2, SMELT_FUSION_GATE_UP_GEGLU = 3 };
enum { SMELT_OUT_FP16 = 0, SMELT_OUT_BF16 = 1, SMELT_OUT_FP32 = 2 };
enum { SMELT_SLOT_FIXED = 0, SMELT_SLOT_VARIABLE = 1 };

typedef struct SmeltMatvecCell {
    int activation, weight /* SMELT_DTYPE_* */, shape, fusion, output, slot;
} SmeltMatvecCell;

/* Family: dense families are SMELT_FAMILY_DENSE + weight dtype */
enum {
    SMELT_FAMILY_DENSE = 0,
    SMELT_FAMILY_AFFINE_U4 = 100,
    SMELT_FAMILY_BINARY1 = 101,
    SMELT_FAMILY_TERNARY2 = 102,
    SMELT_FAMILY_LUT_U4 = 103,
    SMELT_FAMILY_TQH = 104,
    SMELT_FAMILY_TRIT5 = 105,
};
enum {
    SMELT_SELECT_OK = 0,
    SMELT_SELECT_MISSING = -20,        /* meaningful cell, no kernel registered in this backend */
    SMELT_SELECT_NOT_MEANINGFUL = -21, /* no consumer needs this combination */
};
/* select(): total over the cell space, never defaults (MatvecKernelTable.swift:258-270).
 * `hip_backend` != 0 additionally reports SMELT_SELECT_MISSING for families this backend has no
 * kernel for (dense, u4_lut, tqh), so an emitter fails loudly instead of falling back. */
int smelt_kernel_table_select(const SmeltMatvecCell *cell, int hip_backend, int *out_family);
/* meaningfulCells (:155-237): returns the count, writes up to `cap` cells */
int smelt_kernel_table_meaningful_cells(SmeltMatvecCell *out, int cap);

/* ---- weights.bin layout: Sources/SmeltCompiler/SmeltWeightPacker.swift:740-872 -------------- */
typedef struct SmeltWeightEntryC {
    uint64_t offset, size_bytes; /* packed codes (or dense elements) */
    int32_t rows, cols;
    int32_t dtype, group_size;
    int32_t packed_row_stride, padded_cols;
    uint64_t scales_offset, scales_size_bytes;
    uint64_t biases_offset, biases_size_bytes;
} SmeltWeightEntryC;

/* makeAffineEntry (:788-826): [packed][scales][biases], each region 128-byte aligned */
int smelt_layout_make_affine_entry(int rows, int cols, int group_size, uint64_t *offset_io,
                                   SmeltWeightEntryC *out);
/* makeSignedEntry (:831-862): [codes][scales], 128-byte aligned, cols padded to whole groups.
 * dtype is binary1, ternary2, or trit5 (16-byte-aligned rows of ceil(cols/5) bytes). */
int smelt_layout_make_signed_entry(int rows, int cols, int dtype, int group_size,
                                   uint64_t *offset_io, SmeltWeightEntryC *out);
/* Projection bank (SmeltWeightLayoutPlanner.swift:404-572): 2-4 same-input members are re-offset
 * so their packed rows form one contiguous slab, followed by one 128-byte-aligned scale slab
 * (and, for affine, one bias slab).  Byte counts are unchanged and every member keeps its own
 * entry; a bank kernel then walks the members as one virtual row space. */
int smelt_layout_make_affine_bank(const int *member_rows, int members, int cols, int group_size,
                                  uint64_t *offset_io, SmeltWeightEntryC *out_members);
/* The same bank for signed members (binary1, ternary2, trit5): one contiguous code slab, then one
 * 128-byte-aligned scale slab. */
int smelt_layout_make_signed_bank(const int *member_rows, int members, int cols, int dtype, int group_size,
                                  uint64_t *offset_io, SmeltWeightEntryC *out_members);
/* dense fp16/bf16/fp32/int32 entry, 16-byte aligned (:700-737) */
int smelt_layout_make_dense_entry(int rows, int cols, int dtype, uint64_t *offset_io,
                                  SmeltWeightEntryC *out);

/* ---- shape routing: SmeltKernelShapeRegistry.swift + SmeltFusionPlanner.swift:71-152 --------- */
typedef struct SmeltRoute {
    char pipeline[128]; /* manifest pipeline entry */
    int32_t specialized; /* 1 fixed-shape name, 0 generic "name:cols:group" entry */
    int32_t rows_per_group; /* output rows one workgroup walks per step */
    int32_t batch_tile;     /* tokens per grid.y step (1 for batch-1 kernels) */
    int32_t threads;        /* workgroup size */
    int32_t grid_w;         /* workgroups along rows */
} SmeltRoute;

/* decodeAffineMatvec (SmeltFusionPlanner.swift:71-82), fused variants (:100-152) */
int smelt_route_decode_affine(int rows, int cols, int group, int fusion, int compute_units,
                              SmeltRoute *out);
/* prefillAffineFull / prefillAffineBatched (:96-152): max_batch chooses matvec vs MFMA tiles */
int smelt_route_prefill_affine(int rows, int cols, int group, int fusion, int max_batch,
                               int compute_units, SmeltRoute *out);

/* ---- record emitters: SmeltCodeEmitter.swift:1092-1263, 2380-2576; PrefillEmitter.swift:1123-1417 */
typedef struct smelt_emitter smelt_emitter;

typedef struct SmeltBinding {
    int32_t slot; /* >= 0, or SMELT_SLOT_CUR / SMELT_SLOT_ALT */
    uint64_t offset;
    uint8_t offset_kind;
} SmeltBinding;

int smelt_emitter_create(int act_dtype /* SMELT_HIP_ACT_* */, int compute_units, smelt_emitter **out);
void smelt_emitter_destroy(smelt_emitter *e);
const char *smelt_emitter_last_error(const smelt_emitter *e);

/* emitAffineMatvec / emitSignedMatvec through the dtype gateway (emitMatvecImpl, :3997-4082).
 * batch_size > 1 or dynamic != 0 lowers to the batched / qmm families with seqLen-driven grids. */
int smelt_emit_matvec(smelt_emitter *e, int weights_slot, const SmeltWeightEntryC *w,
                      SmeltBinding input, SmeltBinding output, int batch_size, int dynamic);
/* fused_*_matvec_add: output = round(matvec) + residual */
int smelt_emit_matvec_add(smelt_emitter *e, int weights_slot, const SmeltWeightEntryC *w,
                          SmeltBinding input, SmeltBinding output, SmeltBinding residual);
/* fused gate+up+SwiGLU (emitFusedAffineGateUpSwiglu :2380-2425; signed :1926-2030) */
int smelt_emit_gate_up_swiglu(smelt_emitter *e, int weights_slot, const SmeltWeightEntryC *gate,
                              const SmeltWeightEntryC *up, SmeltBinding input, SmeltBinding output,
                              int batch_size, int dynamic);
/* rms_norm_scale_only (norms.metal:944-1008): writes one fp32 scale per row; the first dispatch of the
 * scale-only + norm-scale pair (emitNormScaleAffineMatvecIfPossible, SmeltCodeEmitter.swift:2680-2754). */
int smelt_emit_rms_norm_scale_only(smelt_emitter *e, SmeltBinding input, SmeltBinding scale_output,
                                   int dim, float eps, int batch_size);
/* norm_scale_affine_matvec (lut_matvec.metal:1294-1469; fixed shapes :2743-3170): the kernel reads a
 * precomputed RMS scale and multiplies x_norm = half((x * scale) * (1 + norm_weight)); the normalised
 * row is also stored to norm_output.  affine_u4 weights, one token. */
int smelt_emit_norm_scale_matvec(smelt_emitter *e, int weights_slot, const SmeltWeightEntryC *w,
                                 SmeltBinding norm_scale, SmeltBinding input, SmeltBinding norm_weight,
                                 SmeltBinding norm_output, SmeltBinding output);
/* norm_scale_affine_gate_up_swiglu / _geglu (lut_matvec.metal:1471-1700): same prologue in front of
 * the fused gate+up projection; geglu != 0 selects the GeGLU product (:2235-2243). */
int smelt_emit_norm_scale_gate_up(smelt_emitter *e, int weights_slot, const SmeltWeightEntryC *gate,
                                  const SmeltWeightEntryC *up, int geglu, SmeltBinding norm_scale,
                                  SmeltBinding input, SmeltBinding norm_weight, SmeltBinding output);
/* AtomicNormFusionPass (SmeltDispatchOptimizer.swift:918-1046; kernels fused_norm_matvec.metal:19-297):
 * rms_norm_1pw and its affine consumer in one dispatch.  up == NULL: matvec, the normalised row is also
 * stored (norm_output required).  up != NULL: gate+up+SwiGLU, norm_output ignored.  scratch holds two
 * 32-bit words {scale, ready flag}. */
int smelt_emit_fused_norm_matvec(smelt_emitter *e, int weights_slot, const SmeltWeightEntryC *w,
                                 const SmeltWeightEntryC *up, SmeltBinding input, SmeltBinding norm_weight,
                                 const SmeltBinding *norm_output, SmeltBinding output, SmeltBinding scratch,
                                 float eps);
/* fused_dual_affine_matvec: two weights, one input, two outputs */
int smelt_emit_dual_matvec(smelt_emitter *e, int weights_slot, const SmeltWeightEntryC *w1,
                           const SmeltWeightEntryC *w2, SmeltBinding input, SmeltBinding output1,
                           SmeltBinding output2);
/* Common-input projection bank (emitSignedPackedProjectionBankIfPossible,
 * SmeltCodeEmitter.swift:1264-1340): one dispatch for 2-4 members whose slabs are contiguous.
 * Returns 1 (nothing emitted) when the members do not form a bank, so callers keep
 * independent matvecs. */
int smelt_emit_bank_matvec(smelt_emitter *e, int weights_slot, const SmeltWeightEntryC *members,
                           int count, SmeltBinding input, const SmeltBinding *outputs);
/* lm_head: affine_matvec_argmax + lm_head_argmax_reduce (TopLevelEmitter.swift:907) */
int smelt_emit_lm_head_argmax(smelt_emitter *e, int weights_slot, const SmeltWeightEntryC *w,
                              SmeltBinding input, SmeltBinding partial_keys, SmeltBinding token_out,
                              int batch_size, float logit_cap);
/* emitRMSNorm1PW (SmeltCodeEmitter.swift:2837-2872) and its batched / residual forms: one
 * threadgroup per token.  eps == 1e-6 selects the fixed-dimension pipeline
 * "rms_norm_1pw_d{dim}[_add][_batched]" (no constants); any other eps the generic
 * "rms_norm_1pw[_batched]" with dim and eps as constants 3 and 4 (no residual form exists for it).
 * `weight` is [dim] 16-bit values (a delta from 1); residual may be NULL. */
int smelt_emit_rms_norm_1pw(smelt_emitter *e, SmeltBinding input, SmeltBinding weight,
                            SmeltBinding output, const SmeltBinding *residual, int dim, float eps,
                            int batch_size);
/* emitElementwiseAdd (SmeltCodeEmitter.swift:2944-2966) / elementwise_mul: dispatchThreads over count */
int smelt_emit_elementwise(smelt_emitter *e, int multiply, SmeltBinding a, SmeltBinding b,
                           SmeltBinding output, int count);
/* staged swiglu_fused over `count` gate / up values (DenseTrunkEmitter.swift:209) */
int smelt_emit_swiglu_fused(smelt_emitter *e, SmeltBinding gate, SmeltBinding up,
                            SmeltBinding output, int count);
/* Signed activation views (emitSignedActivationBitplanes / emitSignedBitplane*IfPossible,
 * SmeltCodeEmitter.swift; kernels signed_quant.metal:746-2260).  A view is `planes` bit planes
 * (2..6) of [cols / 128] groups plus one 16-bit scale per group, built once per projection-bank
 * input and consumed by every binary1 / ternary2 member of the bank.
 *   smelt_emit_activation_view     signed_activation_bitplanes_i{N}_g128[_batched]
 *   smelt_emit_view_matvec         signed_{binary,ternary}_bitplane_i{N}_matvec[_add]_g128_rows8
 *   smelt_emit_view_gate_up_swiglu signed_{binary,ternary}_bitplane_i{N}_gate_up_swiglu_g128_rows8 */
int smelt_emit_activation_view(smelt_emitter *e, int planes, SmeltBinding input,
                               SmeltBinding view_planes, SmeltBinding view_scales, int cols,
                               int batch_size);
int smelt_emit_view_matvec(smelt_emitter *e, int weights_slot, const SmeltWeightEntryC *w, int planes,
                           SmeltBinding view_planes, SmeltBinding view_scales, SmeltBinding output,
                           const SmeltBinding *residual, int batch_size);
int smelt_emit_view_gate_up_swiglu(smelt_emitter *e, int weights_slot, const SmeltWeightEntryC *gate,
                                   const SmeltWeightEntryC *up, int planes, SmeltBinding view_planes,
                                   SmeltBinding view_scales, SmeltBinding output, int batch_size);
/* ---- serving operators: what runs between the q|k|v bank and the o projection, and behind the lm_head --------------------
 * (No counterpart in the reference's names: its attention, rope and sampling shaders are not mirrored here.)
 * Every value of a record but the first (`tokens` / `rows`, which resolves to seqLen when dynamic != 0) is fixed when it is
 * emitted; lengths, positions and page tables are data in bound slots, so a captured graph follows them.  The record's grid is
 * nominal.  The emitter runs the launch's own checks of shapes, strides and overlaps within a slot (with the workspace of a context)
 * and refuses what they refuse.  What only the memory tells is left to the launch: whether a slot is large enough, whether an operand
 * lies where its type needs it (keys, values: 16 bytes, attention's output and the frequency table: 8, 32-bit data: 4, other rows: 2), and
 * whether two slots name the same bytes.
 *
 * Rotary positions.  A head's first rotary_dim values are rotated by position * table[i], pair i being (i, i + rotary_dim / 2), or
 * (2 i, 2 i + 1) when interleaved; the rest is copied.  cos and sin are multiplied by `amplitude`.  The table is
 * rotary_dim / 2 doubles (radians a position); positions are int32, one a token. */
typedef struct SmeltRope {
    int32_t head_dim;   /* 1 .. 1024 (64, 128 or 256 where the rows go to a cache) */
    int32_t rotary_dim; /* even, at most head_dim */
    int32_t interleaved;
    float amplitude;
} SmeltRope;

/* Frequencies for contexts longer than the `positions` the model was trained on, by `factor`:
 *   PLAIN   base^(-2 i / rotary_dim)
 *   LINEAR  all divided by factor
 *   BASE    the base multiplied by factor^(rotary_dim / (rotary_dim - 2)): the slowest pair divided, the fastest kept
 *   BANDS   pairs of fewer than `low` turns over `positions` divided, of more than `high` kept, linear in the turns between
 *   PARTS   as BANDS, but linear in the pair's index between those two (rounded outwards), amplitude 0.1 ln(factor) + 1 */
enum { SMELT_ROPE_PLAIN = 0, SMELT_ROPE_LINEAR = 1, SMELT_ROPE_BASE = 2, SMELT_ROPE_BANDS = 3, SMELT_ROPE_PARTS = 4 };
typedef struct SmeltRopeScaling {
    int32_t kind;
    double base, factor, positions, low, high;
} SmeltRopeScaling;
/* writes rotary_dim / 2 doubles and (when not NULL) the amplitude; SMELT_HIP_ERR_INVALID_ARGUMENT for values without a meaning */
int smelt_rope_table(const SmeltRopeScaling *scaling, int rotary_dim, double *out_table, float *out_amplitude);

/* "rope_{half,interleaved}_d{D}_r{R}": `tokens` rows of `heads` heads, strides in elements (>= heads * head_dim).  Output may be the
 * input itself (same slot, offset and stride), or lie beside it within the same rows; other overlaps are refused.  (Rows at equal strides
 * overlap where they share a byte, rows at different ones where what they span does.) */
int smelt_emit_rope(smelt_emitter *e, const SmeltRope *rope, SmeltBinding input, SmeltBinding output,
                    SmeltBinding positions, SmeltBinding table, int heads, int input_stride,
                    int output_stride, int tokens, int dynamic);

/* A paged cache: pages of page_size (16, 32, 64, 128, 256) tokens, keys and values apart, 16-bit.
 *   keys    [pages][kv_heads][head_dim / 8][page_size][8]   (what the matrix cores take, a page and head contiguous)
 *   values  [pages][kv_heads][page_size][head_dim] */
typedef struct SmeltPagedCache {
    SmeltBinding k, v;
    int32_t head_dim /* 64, 128, 256 */, kv_heads, page_size, pages;
} SmeltPagedCache;

/* "paged_kv_append[_q]_{half,interleaved}_d{D}_r{R}_kv{H}_p{P}": token rows k (rotated) and v put to place slots[token] = page *
 * page_size + offset; a negative slot, or one behind the pool, puts the token nowhere.  Tokens that name the same place leave one of
 * them, element by element unspecified which.  With q and q_out (both or neither) the q rows are rotated in the same launch,
 * also those of tokens without a place; q_out may be q itself, also within rows [q | k | v] that one projection wrote.  rotary_dim 0
 * rotates nothing. */
int smelt_emit_paged_kv_append(smelt_emitter *e, const SmeltRope *rope, const SmeltPagedCache *cache,
                               SmeltBinding k, SmeltBinding v, SmeltBinding positions,
                               SmeltBinding slots, SmeltBinding table, const SmeltBinding *q,
                               const SmeltBinding *q_out, int q_heads, int k_stride, int v_stride,
                               int q_stride, int q_out_stride, int tokens, int dynamic);

/* "paged_attention[_shared]_d{D}_h{H}_kv{H}_p{P}": sequence s has the rows offsets[s] .. offsets[s + 1] (int32[sequences + 1],
 * ascending from 0) of q and output ([tokens][heads * head_dim]; rows from offsets[sequences] on are left as they were) and
 * kv_lens[s] keys of its own, its new tokens' included, on the pages of page_table[s][pages_per_sequence].  prefix_table (at most
 * prefix_pages pages) and prefix_len (one int32) name a prefix that stands before every sequence's own keys; it is read once for
 * all of them when they have few rows each.  The last row of a sequence is the newest key's; a row sees the keys up to its
 * own and, with window > 0, only the last `window` of them.  A row that sees nothing is zero.  Infinities and NaN among keys and values
 * that a row does not see leave it as it is (rows of such a tile are formed a second time, slowly).  Lengths are cut to what the tables
 * hold; keys on a page outside the pool are not seen.  Offsets that do not ascend leave rows unspecified, and nothing else touched. */
int smelt_emit_paged_attention(smelt_emitter *e, const SmeltPagedCache *cache, SmeltBinding q,
                               SmeltBinding page_table, SmeltBinding kv_lens, SmeltBinding offsets,
                               SmeltBinding output, const SmeltBinding *prefix_table,
                               const SmeltBinding *prefix_len, int prefix_pages, int heads,
                               int q_stride, int pages_per_sequence, float scale, int window,
                               int sequences, int tokens, int dynamic);

/* "verify_drafts" / "verify_drafts_given" (draft NULL): drafted tokens against the target's probabilities.  Sequence s has the logits
 * rows offsets[s] .. offsets[s + 1] of target (16-bit, `vocab` logits at `stride` elements): row i is what follows the i-th
 * drafted token's prefix, so its last row has no draft.  With p = softmax(target / temperature[s]) and q = softmax(draft /
 * temperature[s]) (draft NULL: q is 1 on the drafted token): draft x of row i is taken while u_accept[row] * q(x) < p(x).  The
 * first one refused is replaced by a token drawn from max(p - q, 0); if all are taken one more is drawn from the last row's
 * p.  Drawing takes the lowest token whose running sum of weights passes u_sample[s] * their total (max(p - q, 0) all zero: p's).
 * temperature <= 0 (or not a number): a draft is taken while it is the row's largest logit (lowest token of equal ones), and
 * that token is drawn.  A draft outside the vocabulary is refused; a NaN logit counts as -inf, +inf as the largest finite number; a row
 * without any weight draws -1.  tokens[row]: the taken drafts, the drawn token, then -1; counts[s]: taken drafts.  Rows from
 * offsets[sequences] on are left as they were; a sequence without rows counts 0 (but a record of no rows at all launches nothing).  Whether a
 * draft is taken is decided from 32-bit sums, which can turn it where u_accept lies within a few 1e-7 of p / q; what is drawn, from 64-bit ones.
 * At most 65535 rows and sequences. */
int smelt_emit_verify_drafts(smelt_emitter *e, SmeltBinding target, const SmeltBinding *draft,
                             SmeltBinding draft_tokens, SmeltBinding offsets, SmeltBinding u_accept,
                             SmeltBinding u_sample, SmeltBinding temperature, SmeltBinding tokens,
                             SmeltBinding counts, int rows, int sequences, int vocab, int stride);
/* swap cur/alt (SmeltDispatchRecord.swap) */
int smelt_emit_swap(smelt_emitter *e);

size_t smelt_emitter_record_count(const smelt_emitter *e);
const SmeltDispatchRecord *smelt_emitter_records(const smelt_emitter *e); /* dispatches.bin bytes */
size_t smelt_emitter_pipeline_count(const smelt_emitter *e);
const char *smelt_emitter_pipeline_name(const smelt_emitter *e, size_t index);
/* bytes a partial-key buffer must hold for the argmax records emitted so far */
size_t smelt_emitter_argmax_partial_bytes(const smelt_emitter *e);

/* Resolve a pipeline entry without a device: writes the kernel symbol and argument kinds.
 * Returns 0, SMELT_HIP_ERR_UNKNOWN_PIPELINE or SMELT_HIP_ERR_INVALID_PACKAGE. */
int smelt_hip_resolve_pipeline_name(const char *entry, int default_act, char *symbol,
                                    size_t symbol_cap, char *kinds, size_t kinds_cap);

/* Launch plans of the kernels a record is re-routed to, without a device (no counterpart in the
 * reference: one kernel per pipeline name there; for tests and for integrators who want to know
 * what a record will run).  Each writes its answer as unsigned 32-bit fields and returns 1 when
 * the shape takes the kernel, 0 when it keeps the kernel its pipeline names, negative on error.
 *
 * smelt_hip_plan_qmm: an affine qmm record (groups of 64, 128 or 32 columns; plain, +add: nmat 1;
 * gate+up: nmat 2) of `batch` tokens.  (The plans of the other re-routed forms are not exposed here: the per-token
 * small-batch names of small matrices, which take the single-token kernel with a grid row per token, the norm-scale
 * qmm names, which run as normalised rows plus this plan, the ternary qmm and the binary / ternary records over
 * several tokens.)  out[0] = 1 streaming kernel, 2 token-tile kernel; out[1] row tiles per wave;
 * out[2] waves along K (streaming: waves of the workgroup); out[3] = 1 when the two matrices go to
 * separate waves; out[4] workgroups that share a tile along K; out[5..7] grid; out[8] threads;
 * out[9] LDS bytes; out[10] workspace bytes of the K split (low 32 bits).
 *
 * smelt_hip_plan_matvec: a single-token matvec of code layout 0 affine u4, 1 binary1, 2 ternary2,
 * 3 trit5.  out[0] 128-byte segments per wave; out[1] waves per workgroup; out[2] workgroups;
 * out[3] threads; out[4] LDS bytes. */
int smelt_hip_plan_qmm(uint32_t rows, uint32_t cols, uint32_t group, uint32_t nmat, uint32_t batch,
                       uint32_t compute_units, size_t lds_limit, size_t workspace_bytes,
                       uint32_t out[11]);
int smelt_hip_plan_matvec(int code_layout, uint32_t rows, uint32_t cols, uint32_t group,
                          uint32_t nmat, size_t lds_limit, int force, uint32_t out[5]);

#ifdef __cplusplus
}
#endif
#endif /* SMELT_HIP_COMPILER_H */
