/*
 * roost_amd.h -- the per-op entry points of the MI355X (gfx950) Roost kernel library, exported by name.
 *
 * A Roost loader reaches these through the registration table that roost_register() fills (RoostOpEntry.run / plan /
 * workspace); they are also exported under the names below so a C, ctypes or P/Invoke caller can bind them directly.
 * Each one replaces the reference entry point named beside it, with the same arguments, statuses and ownership rules
 * (caller-owned workspaces, no allocation, no host synchronisation, typed refusals before any launch).
 */
#ifndef ROOST_AMD_H_
#define ROOST_AMD_H_

#include "roost_kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Library identity: the file is libroost_kernels_gfx950.so, roost_register() reports library_name
 * "roost-kernels-gfx950", and every entry's constraints.sm_min is ROOST_AMD_ARCH_ID. */
#define ROOST_AMD_ARCH_ID 950u

/* PagedAttention, variant "paged-attention-gfx950" (DETERMINISTIC | BATCH_INVARIANT | NEEDS_PLAN).
 * Replaces roost_paged_attention_workspace / _plan / _run of the reference
 * (kernels/src/paged_attention.cu:183-198, :200-250, :252-349; declared in kernels/src/roost_internal.h:45-47). */
ROOST_API RoostStatus roost_paged_attention_workspace(RoostContext* ctx, const void* params, RoostWorkspaceSizes* sizes);
ROOST_API RoostStatus roost_paged_attention_plan(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                                 void* stream);
ROOST_API RoostStatus roost_paged_attention_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                                void* stream);

/* PagedAttention with Qwen3.5's attention output gate (SigmoidMul, out = out * sigmoid(gate)) folded into the kernels
 * that write the output. No counterpart in the reference, whose Qwen3.5 worker runs roost_paged_attention_run and then
 * roost_sigmoid_mul_run on its output (Qwen35EagerModel.cs:94-97 lists both kernels; semantics CpuOps.Gating.cs:84-96).
 * This call computes the same output bit for bit and writes it once: each output element, rounded to the output type,
 * is multiplied by sigmoid(gate) with the SigmoidMul op's own arithmetic where the decode, tile and merge kernels store
 * it. `params` is a planned RoostPagedAttentionParams (plan() and the workspace as for roost_paged_attention_run);
 * `gate_params` a RoostSigmoidMulParams whose input and output are both the attention output (the gate applies in
 * place), rows = tokens, dim = q_heads * head_dim, and whose gate (same dtype as the output, 8-byte aligned) does not
 * overlap the output. The lse output, when requested, is that of the ungated attention. */
ROOST_API RoostStatus roost_amd_paged_attention_gated_run(RoostContext* ctx, const void* params, const void* gate_params,
                                                          const RoostWorkspace* ws, void* stream);

/* CacheWrite, variant "cache-write-gfx950" (GRAPH_CAPTURABLE | DETERMINISTIC | BATCH_INVARIANT), no workspace.
 * Replaces roost_cache_write_run (kernels/src/m0_ops.cu:388-429; declared in kernels/src/roost_internal.h:42). */
ROOST_API RoostStatus roost_cache_write_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                            void* stream);

/* GatedDeltaRule chunked prefill, variant "gated-delta-rule-chunk-gfx950"
 * (DETERMINISTIC | BATCH_INVARIANT | NEEDS_PLAN). Replaces roost_gdn_chunk_workspace / _plan / _run
 * (kernels/src/ops/gated_delta_rule.cu:380-576; declared in kernels/src/roost_internal.h:81-83). */
ROOST_API RoostStatus roost_gdn_chunk_workspace(RoostContext* ctx, const void* params, RoostWorkspaceSizes* sizes);
ROOST_API RoostStatus roost_gdn_chunk_plan(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                           void* stream);
ROOST_API RoostStatus roost_gdn_chunk_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws, void* stream);

/* GatedDeltaRule recurrent (decode and short continuations), variant "gated-delta-rule-recurrent-aot" -- the id the
 * worker names (reference src/Starlings.Roost.Worker/Eager/CudaOps.cs:28) -- flagged
 * GRAPH_CAPTURABLE | DETERMINISTIC | BATCH_INVARIANT, no plan. Replaces roost_gdn_recurrent_workspace / _run
 * (kernels/src/ops/gated_delta_rule.cu:580-649; declared in kernels/src/roost_internal.h:84-85). */
ROOST_API RoostStatus roost_gdn_recurrent_workspace(RoostContext* ctx, const void* params, RoostWorkspaceSizes* sizes);
ROOST_API RoostStatus roost_gdn_recurrent_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                              void* stream);

/* GatedDeltaRule recurrent variant without a workspace argument. This entry point has no counterpart in the reference:
 * it is for callers that cannot allocate device memory (code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc). It computes exactly what roost_gdn_recurrent_run computes, with the routing scratch (chunk
 * tables and per-(chunk, head) records of the sequences of 16+ tokens) in a static 24 MiB device array per GPU instead
 * of ws->device. A call whose routing could need more than the array (the workspace query of the recurrent variant
 * reports above 24 MiB: room for 76 chunks of 64 tokens x 16 heads, e.g. one 4,700-token sequence, or a worker step of
 * 1,072 tokens over 50 sequences) is refused with ROOST_STATUS_INVALID_ARGUMENT before any launch. The context's device must be
 * current. Calls that overlap on one GPU race on its array. It calls no hipMalloc/hipFree. */
ROOST_API RoostStatus roost_amd_gdn_recurrent_run_noalloc(RoostContext* ctx, const void* params, void* stream);

/* GatedDeltaRuleGates folded into the recurrent GatedDeltaRule variant. No counterpart in the reference, whose Qwen3.5
 * layer runs roost_gated_delta_rule_gates_run (g, beta from a, b, a_log, dt_bias) and then the recurrent variant on
 * them (CpuOps.Gating.cs:21-58, CpuOps.Hybrid.cs:30-157). This call computes the same outputs and states bit for bit
 * without writing or reading g and beta: each kernel that reads a token's gates computes them from the gates' inputs
 * with the gates op's own arithmetic (beta rounded to bf16, as that op's bf16 output holds it). `params` is a
 * RoostGatedDeltaRuleParams whose g and beta spans are not read; `gates` a RoostGatedDeltaRuleGatesParams (tokens and
 * v_heads equal to the GDN call's; a and b bf16 or f32 row-strided views, a_log and dt_bias bf16 or f32) whose g and
 * beta spans are not read. Workspace as roost_gdn_recurrent_workspace sizes it. */
ROOST_API RoostStatus roost_amd_gdn_recurrent_gated_run(RoostContext* ctx, const void* params, const void* gates,
                                                         const RoostWorkspace* ws, void* stream);

/* One decode step of a Gated DeltaNet layer in one call: CausalConv1d, GatedDeltaRuleGates, the recurrent GatedDeltaRule
 * and GatedRmsNorm. No counterpart in the reference, whose Qwen3.5 worker runs the four ops one after another
 * (Qwen35EagerModel.cs:89-92 lists them; semantics CpuOps.Hybrid.cs:30-157, 160-263 and CpuOps.Gating.cs:21-83). The
 * norm's output, the GDN output, the recurrent states and the convolution states equal the four calls' bit for bit
 * (sequences that share a state slot run in batch order, as the recurrent variant runs them); the convolution's output
 * is not written (its span is only checked). `conv_params` is a RoostCausalConv1dParams
 * over bf16 activations with at most 4 taps and the GDN call's batch, tokens and cu_seqlens; `gdn_params` a
 * RoostGatedDeltaRuleParams whose q, k and v are column views of the convolution's output (row stride = channels) and
 * whose cu_seqlens_host is given: every sequence must be shorter than 16 tokens (longer ones run on the chunk kernels in
 * the recurrent variant), else UNSUPPORTED; `gates_params` a RoostGatedDeltaRuleGatesParams as for
 * roost_amd_gdn_recurrent_gated_run, or NULL to read g and beta from the GDN params; `norm_params` a
 * RoostGatedRmsNormParams of bf16 rows = tokens x v_heads, dim = 128, whose input is the GDN output, with input, gate and
 * output 16-byte aligned, and whose output overlaps none of the layer's other inputs or states. No workspace. */
ROOST_API RoostStatus roost_amd_gdn_decode_layer_run(RoostContext* ctx, const void* conv_params,
                                                      const void* gates_params, const void* gdn_params,
                                                      const void* norm_params, void* stream);

/* One Gated DeltaNet layer of any step (decode, prefill or mixed) over the recurrent variant in one call: CausalConv1d,
 * GatedDeltaRuleGates, GatedDeltaRule and GatedRmsNorm. No counterpart in the reference (the same four calls, one after
 * another; the worker names the recurrent variant for every length, CudaOps.cs:28). A step whose sequences are all
 * shorter than 16 tokens (known from tokens < 16 or from cu_seqlens_host) with the norm in its single-pass bf16 form
 * runs as roost_amd_gdn_decode_layer_run does; any other step runs the convolution, the recurrent variant with g and
 * beta computed from the gates' inputs (its sequences of 16+ tokens on the chunk kernels) and the norm. The norm's
 * output, the recurrent states and the convolution states equal the four calls' bit for bit (the convolution's output
 * is written on the second path only). Params as for roost_amd_gdn_decode_layer_run, without its
 * length limit; `ws` is the recurrent variant's workspace (roost_gdn_recurrent_workspace of `gdn_params`; NULL is
 * enough when it reports zero bytes). */
ROOST_API RoostStatus roost_amd_gdn_layer_run(RoostContext* ctx, const void* conv_params, const void* gates_params,
                                              const void* gdn_params, const void* norm_params, const RoostWorkspace* ws,
                                              void* stream);

/* One prefill pass of a Gated DeltaNet layer over the chunk variant in one call: CausalConv1d, GatedDeltaRuleGates, the
 * chunked GatedDeltaRule and GatedRmsNorm. No counterpart in the reference (the same four calls as above, one after
 * another). The chunk kernels compute g and beta from the gates' inputs where they read them (the gates op's
 * arithmetic), so g and beta never reach memory. The convolution's output, the GDN output, the norm's output, the
 * recurrent states and the convolution states equal the four calls' bit for bit. Params as for
 * roost_amd_gdn_decode_layer_run, except that the sequences may have any lengths (cu_seqlens_host may be NULL at run)
 * and the norm may take any form roost_gated_rms_norm_run takes. `ws` is the chunk variant's workspace, sized by
 * roost_gdn_chunk_workspace and planned by roost_amd_gdn_chunk_layer_plan for the same gates and GDN params (else
 * NOT_PLANNED). */
ROOST_API RoostStatus roost_amd_gdn_chunk_layer_run(RoostContext* ctx, const void* conv_params,
                                                     const void* gates_params, const void* gdn_params,
                                                     const void* norm_params, const RoostWorkspace* ws, void* stream);
/* plan() of roost_amd_gdn_chunk_layer_run: roost_gdn_chunk_plan of `gdn_params` (host chunk tables from cu_seqlens_host,
 * copied to ws on the stream), except that with `gates_params` given the GDN params' g and beta are not read. */
ROOST_API RoostStatus roost_amd_gdn_chunk_layer_plan(RoostContext* ctx, const void* gates_params, const void* gdn_params,
                                                      const RoostWorkspace* ws, void* stream);

/* The Gated DeltaNet layer's neighbour ops, each flagged GRAPH_CAPTURABLE | DETERMINISTIC | BATCH_INVARIANT, no plan
 * and no workspace:
 * GatedDeltaRuleGates, variant "gated-delta-rule-gates-gfx950" -- replaces roost_gated_delta_rule_gates_run
 *   (kernels/src/ops/gating.cu:110-177);
 * GatedRmsNorm, variant "gated-rms-norm-gfx950" -- replaces roost_gated_rms_norm_run (gating.cu:179-229);
 * SigmoidMul, variant "sigmoid-mul-gfx950" -- replaces roost_sigmoid_mul_run (gating.cu:231-269);
 * CausalConv1d, variant "causal-conv1d-gfx950" -- replaces roost_causal_conv1d_run
 *   (kernels/src/ops/causal_conv1d.cu:122-175);
 * RecurrentStateCopy / RecurrentStateSnapshot, variants "recurrent-state-copy-gfx950" / "recurrent-state-snapshot-gfx950"
 *   -- replace roost_recurrent_state_copy_run / _snapshot_run (kernels/src/ops/recurrent_state.cu:58-108).
 * All are registered by kernels/src/ops/hybrid_entries.cu:75-148 in the reference. */
ROOST_API RoostStatus roost_gated_delta_rule_gates_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                                       void* stream);
ROOST_API RoostStatus roost_gated_rms_norm_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                               void* stream);
ROOST_API RoostStatus roost_sigmoid_mul_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                            void* stream);
ROOST_API RoostStatus roost_causal_conv1d_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                              void* stream);
ROOST_API RoostStatus roost_recurrent_state_copy_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                                     void* stream);
ROOST_API RoostStatus roost_recurrent_state_snapshot_run(RoostContext* ctx, const void* params,
                                                         const RoostWorkspace* ws, void* stream);

/* The attention layer's input ops, each flagged GRAPH_CAPTURABLE | DETERMINISTIC | BATCH_INVARIANT, no plan and no
 * workspace:
 * QkNorm, variant "qk-norm-gfx950" -- replaces the reference's QkNormRun (kernels/src/m0_ops.cu:89-130, registered as
 *   "qk-norm-flashinfer" at kernels/src/m0_registry.cu:77);
 * Rope, variant "rope-gfx950" -- replaces RopeRun (kernels/src/m0_ops.cu:210-255, "rope-roost" at m0_registry.cu:79). */
ROOST_API RoostStatus roost_qk_norm_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws, void* stream);
ROOST_API RoostStatus roost_rope_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws, void* stream);

/* QkvQkNormRopeCacheWrite (ROOST_OP_QKV_QK_NORM_ROPE_CACHE_WRITE, 67), variant "qkv-qk-norm-rope-cache-write-gfx950".
 * The reference's C header names only the op id: the op exists in its CPU reference (src/Starlings.Roost.Ops/
 * CpuOps.Fused.cs:37-95) with the argument struct QkvQkNormRopeCacheWriteArgs (src/Starlings.Roost.Ops/OpArgs.cs:
 * 629-683), and no CUDA library implements it. This record carries those arguments field for field in the ABI's
 * style; the activation type is qkv's dtype and the cache type k_cache's. Each [q | k | v] row of qkv is split: q
 * heads are RmsNormed with q_weight, rotated (full rotary width, default frequencies, NeoX halves) and written to q;
 * k heads are RmsNormed with k_weight, rotated and written into k_cache at slot_mapping[t] (NHD pools, unit scale);
 * v heads are copied into v_cache there. A negative or out-of-pool slot writes no cache row; qkv is left as it was. */
typedef struct RoostQkvQkNormRopeCacheWriteParams {
  uint32_t struct_size;
  uint32_t abi_minor;
  RoostDeviceSpan qkv;          /* [tokens, (q_heads + 2 * kv_heads) * head_dim] */
  RoostDeviceSpan q;            /* [tokens, q_heads, head_dim] output */
  RoostDeviceSpan q_weight;     /* [head_dim] */
  RoostDeviceSpan k_weight;     /* [head_dim] */
  RoostDeviceSpan positions;    /* [tokens] int32 */
  RoostDeviceSpan k_cache;      /* [pages, page_size, kv_heads, head_dim] */
  RoostDeviceSpan v_cache;      /* same */
  RoostDeviceSpan slot_mapping; /* [tokens] int64 */
  uint32_t tokens;
  uint32_t q_heads;
  uint32_t kv_heads;
  uint32_t head_dim;
  uint32_t page_size;
  float eps;
  float theta;
  uint32_t reserved0;
} RoostQkvQkNormRopeCacheWriteParams;

ROOST_API RoostStatus roost_qkv_qk_norm_rope_cache_write_run(RoostContext* ctx, const void* params,
                                                             const RoostWorkspace* ws, void* stream);

/* The fused ops between a layer's residual stream and its projections: ROOST_OP_ADD_RMS_NORM (64),
 * ROOST_OP_ADD_RMS_NORM_QUANT (65), ROOST_OP_SILU_MUL_QUANT (66) and ROOST_OP_GEMM_LORA_EPILOGUE (68), of which the
 * reference's C header names the ids only. They are reached by name, outside the registration table, whose variants a
 * Roost loader checks against its manifest. Every call may be captured into a HIP graph, is deterministic, allocates
 * nothing and does not synchronise; the context's device must be current. Row strides are elements between rows, 0 for
 * contiguous rows; rows need only their element type's alignment unless stated. */

/* AddRmsNorm. Per row, in f32: s = input + residual; residual_out = s; output = s / sqrt(mean(s^2) + eps) * weight.
 * The norm takes the f32 sum, not the rounded residual_out; each output is rounded once. Without a residual (NULL
 * address) s = input; without a residual_out the sum is not stored. output and residual_out may each be exactly the
 * input or the residual (same address, stride and type); any other overlap is refused. A row's result does not depend on
 * the other rows of the call. dim <= 32768; rows up to 4,194,303 of any width. */
typedef struct RoostAmdAddRmsNormParams {
  uint32_t struct_size;
  uint32_t abi_minor;
  RoostDeviceSpan input;        /* [rows, dim] bf16 or f32 */
  RoostDeviceSpan residual;     /* [rows, dim] bf16 or f32, or NULL */
  RoostDeviceSpan weight;       /* [dim] bf16 or f32 */
  RoostDeviceSpan residual_out; /* [rows, dim] the residual's type (the input's without one), or NULL */
  RoostDeviceSpan output;       /* [rows, dim] the input's type */
  uint32_t rows;
  uint32_t dim;
  uint32_t input_stride;
  uint32_t residual_stride;
  uint32_t residual_out_stride;
  uint32_t output_stride;
  float eps;
  uint32_t reserved0;
} RoostAmdAddRmsNormParams;

ROOST_API RoostStatus roost_amd_add_rms_norm_run(RoostContext* ctx, const void* params, void* stream);

/* AddRmsNormQuant. AddRmsNorm with its output y in 8 bits (OCP e4m3) and a scale for each cell: a whole row
 * (group_size 0) or group_size consecutive columns of it (a power of two from 16 to 512; the last cell of a row may be
 * shorter). scale = max(max|y| / 448, 2^-126) over the cell's f32 values, code = the f32 quotient y / scale rounded to
 * nearest, ties to even, so code * scale stands for y and a cell of zeros has zero codes. A cell that holds a NaN has a NaN
 * scale and NaN codes; one that holds an infinity has an infinite scale, zero codes for its finite values and NaN codes for
 * the others. */
typedef struct RoostAmdAddRmsNormQuantParams {
  uint32_t struct_size;
  uint32_t abi_minor;
  RoostDeviceSpan input;        /* [rows, dim] bf16 or f32 */
  RoostDeviceSpan residual;     /* [rows, dim] bf16 or f32, or NULL */
  RoostDeviceSpan weight;       /* [dim] bf16 or f32 */
  RoostDeviceSpan residual_out; /* [rows, dim] the residual's type (the input's without one), or NULL */
  RoostDeviceSpan output;       /* [rows, dim] f8e4m3 */
  RoostDeviceSpan scales;       /* [rows, cells of a row] f32, contiguous */
  uint32_t rows;
  uint32_t dim;
  uint32_t input_stride;
  uint32_t residual_stride;
  uint32_t residual_out_stride;
  uint32_t output_stride;
  float eps;
  uint32_t group_size;
} RoostAmdAddRmsNormQuantParams;

ROOST_API RoostStatus roost_amd_add_rms_norm_quant_run(RoostContext* ctx, const void* params, void* stream);

/* SiluMulQuant. y = gate * sigmoid(gate) * up in f32, then 8 bits and scales as AddRmsNormQuant's. gate and up may be the
 * halves of one fused projection (row strides); the outputs overlap nothing. dim <= 32768;
 * rows up to 4,194,303 of any width. */
typedef struct RoostAmdSiluMulQuantParams {
  uint32_t struct_size;
  uint32_t abi_minor;
  RoostDeviceSpan gate;   /* [rows, dim] bf16 or f32 */
  RoostDeviceSpan up;     /* [rows, dim] the gate's type */
  RoostDeviceSpan output; /* [rows, dim] f8e4m3 */
  RoostDeviceSpan scales; /* [rows, cells of a row] f32, contiguous */
  uint32_t rows;
  uint32_t dim;
  uint32_t gate_stride;
  uint32_t up_stride;
  uint32_t output_stride;
  uint32_t group_size;
} RoostAmdSiluMulQuantParams;

ROOST_API RoostStatus roost_amd_silu_mul_quant_run(RoostContext* ctx, const void* params, void* stream);

/* GemmLora: a projection shared by every sequence, with each sequence's own low-rank adapter on top. For row t of sequence
 * b (cu_seqlens[b] <= t < cu_seqlens[b + 1]) with adapter a = lora_slots[b] (a C2 step plan's lora_slot):
 *   output_t = weight x_t + lora_scale[a] * B_a[:, :rank] (A_a[:rank] x_t) + addend_t,  rank = ranks[a] (max_rank if NULL).
 * A slot below 0 or at or past `adapters` means no adapter; ranks are clamped to [0, max_rank], and what a pool holds past
 * an adapter's rank is not read into a result. Rows of no sequence (behind cu_seqlens[batch], in a padded batch) are left
 * as they were. One adapter's values never reach another sequence's rows, NaN and infinity included.
 *   - x bf16: weight bf16, adapters bf16, output bf16 or f32. x f32: all f32. x f8e4m3 (as AddRmsNormQuant leaves rows with
 *     group_size 0): weight f8e4m3, a scale for each row of x and of weight, adapters bf16, output bf16 or f32.
 *   - weight NULL: the adapters alone, on top of the addend (a product that ran elsewhere) or alone.
 *   - lora_a NULL: no adapters (adapters = max_rank = 0; lora_slots, lora_b, lora_scale and ranks unused).
 *   - addend: bf16 or f32, may be exactly the output (same address, stride and type); any other overlap of the output is
 *     refused.
 * Sums are f32. Beside bf16 adapters the low-rank rows lora_scale[a] A_a x_t may be rounded to bf16 once under a bf16 output
 * (off by at most 2^-8 of each); under an f32 output they keep 24 bits. f8e4m3 products under a bf16 output are those of the
 * e4m3 matrix instructions, which cut the products of eight neighbouring elements at 2^-13 of the power of two of the largest
 * of the eight; under an f32 output the codes are multiplied as bf16, exactly.
 * x, weight, lora_a and lora_b are 16-byte aligned; in_dim and x_stride are multiples of 16 bytes and, like out_dim, at most
 * 2^20 elements; tokens are below 2^20; max_rank is a multiple of 8 up to 128. cu_seqlens[0] = 0 and cu_seqlens does not go
 * backwards (device data, not checked; a table that breaks this leaves the rows in question unwritten or undefined, and reads
 * and writes nothing outside the spans). The results of a row may differ in rounding with the number of tokens of the call. */
typedef struct RoostAmdGemmLoraParams {
  uint32_t struct_size;
  uint32_t abi_minor;
  RoostDeviceSpan x;          /* [tokens, in_dim] */
  RoostDeviceSpan x_scale;    /* [tokens] f32 with f8e4m3 rows, else NULL */
  RoostDeviceSpan weight;     /* [out_dim, in_dim] or NULL */
  RoostDeviceSpan w_scale;    /* [out_dim] f32 with f8e4m3 weights, else NULL */
  RoostDeviceSpan lora_a;     /* [adapters, max_rank, in_dim] or NULL */
  RoostDeviceSpan lora_b;     /* [adapters, out_dim, max_rank] */
  RoostDeviceSpan lora_scale; /* [adapters] f32, or NULL for 1 */
  RoostDeviceSpan ranks;      /* [adapters] i32, or NULL */
  RoostDeviceSpan lora_slots; /* [batch] i32 */
  RoostDeviceSpan cu_seqlens; /* [batch + 1] i32 */
  RoostDeviceSpan addend;     /* [tokens, out_dim] or NULL */
  RoostDeviceSpan output;     /* [tokens, out_dim] */
  uint32_t tokens;
  uint32_t batch;
  uint32_t in_dim;
  uint32_t out_dim;
  uint32_t adapters;
  uint32_t max_rank;
  uint32_t x_stride;
  uint32_t addend_stride;
  uint32_t output_stride;
  uint32_t reserved0;
} RoostAmdGemmLoraParams;

/* Device scratch of a call (sizes->device_bytes; the low-rank rows). Its contents are undefined before and after. */
ROOST_API RoostStatus roost_amd_gemm_lora_workspace(RoostContext* ctx, const void* params, RoostWorkspaceSizes* sizes);
ROOST_API RoostStatus roost_amd_gemm_lora_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                              void* stream);

/* ---- A KV cache held in 4 bits ----------------------------------------------------------------------------------------
 * One layer's K and V in e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, two a byte, the lower dim in the low
 * half) with one power-of-two scale for each 32 consecutive dims of a row: 4.25 bits a value. A scale byte b stands for
 * 2^(b - 127), 7 <= b <= 252; 255 marks a block that held a NaN or an infinity, which reads as NaN. Calls of this section and
 * of the next are reached by name, outside the registration table. Every run call may be captured into a HIP graph, allocates
 * nothing, does not synchronise and is deterministic; the context's device must be current.
 *
 * Codes lie as [pages, kv_heads, page_size, head_dim / 2], scales as [pages, kv_heads, head_dim / 32, page_size] bytes: one
 * head's part of a page is contiguous, and so are its tokens' scales of one block. head_dim is 64, 128 or 256, page_size a
 * power of two from 16 to 1024, every address 16-byte aligned. `length` of k and v counts values (two a byte), of the scales
 * bytes; a span may hold more than whole pages, and the pool has the pages that all four hold. */
typedef struct RoostAmdCacheF4 {
  RoostDeviceSpan k;        /* f4e2m1 [pages, kv_heads, page_size, head_dim] */
  RoostDeviceSpan k_scales; /* u8 [pages, kv_heads, head_dim / 32, page_size] */
  RoostDeviceSpan v;
  RoostDeviceSpan v_scales;
  uint32_t kv_heads;
  uint32_t head_dim;
  uint32_t page_size;
  uint32_t reserved0;
} RoostAmdCacheF4;

/* CacheWriteF4: token t's K and V rows into slot slot_mapping[t] = page * page_size + offset; a slot below 0 or past the pool
 * skips the token. Per block of 32 dims with largest magnitude a: scale = the smallest power of two with a <= 7 scale, held to
 * 2^-120 .. 2^125 (a block of zeros has 2^-120); code = x / scale rounded to nearest, ties to the even code, at most 6. So a
 * value is off by at most one scale, half the grid's last step (two scales where a is above 7 * 2^125). Slots of one call
 * differ; a slot named twice holds parts of both tokens' rows.
 * CacheReadF4: the same record the other way, every value exactly (bf16 or f32); rows of a skipped token are left as they were.
 * k and v are [tokens, kv_heads, head_dim], heads contiguous, tokens k_stride / v_stride elements apart (0 for contiguous
 * rows): column views of one projection. They are 16-byte aligned and their strides multiples of 16 bytes; tokens are below
 * 2^24. CacheReadF4's k and v overlap nothing. */
typedef struct RoostAmdCacheF4Params {
  uint32_t struct_size;
  uint32_t abi_minor;
  RoostDeviceSpan k; /* bf16, f16 (write only) or f32 */
  RoostDeviceSpan v; /* k's type */
  RoostAmdCacheF4 cache;
  RoostDeviceSpan slot_mapping; /* [tokens] i64 */
  uint32_t tokens;
  uint32_t k_stride;
  uint32_t v_stride;
  uint32_t reserved0;
} RoostAmdCacheF4Params;

ROOST_API RoostStatus roost_amd_cache_write_f4_run(RoostContext* ctx, const void* params, void* stream);
ROOST_API RoostStatus roost_amd_cache_read_f4_run(RoostContext* ctx, const void* params, void* stream);

/* PagedAttentionF4: attention of a step's queries over such a cache, decode rows, prompt chunks and both in one call. Sequence
 * b's queries are rows cu_seqlens[b] .. cu_seqlens[b + 1] of q and stand at its last positions: with n of them and `len` keys,
 * query i is at position len - n + i and sees the keys up to it, from position - window_left on where window_left >= 0; all keys,
 * wherever it stands, unless causal (a window needs causal). Per query head h with KV head h / (q_heads / kv_heads):
 *   s_j = sm_scale q . k_j, with logits_soft_cap > 0 then cap tanh(s_j / cap); p = softmax(s); out = sum_j p_j v_j;
 *   lse = log2 sum_j exp(s_j).
 * A query that sees no key has zero output and an lse of minus infinity. Rows of no sequence (behind cu_seqlens[batch], in a
 * padded batch) are left as they were. Keys that a query does not see never reach it, NaN blocks included.
 * Tables, all device data, so that one captured call serves steps of other lengths, in either of two forms:
 *   - block_tables [table_rows, max_blocks] and kv_lens [table_rows], as the page calls below keep them; sequence b's row is
 *     sequences[b], or b where sequences is NULL;
 *   - kv_indptr [batch + 1], block_tables [.] and kv_lens [batch] as the plan region's kv_indptr, kv_indices and
 *     kv_last_page_len; max_blocks, table_rows and sequences are 0.
 * A page id outside the pool holds no keys; a row outside the tables has none; lengths are cut to the row's pages. Causal
 * queries in front of the first key (n > len) see none; cu_seqlens[0] = 0 and cu_seqlens does not go backwards (else the rows in
 * question are undefined or unwritten, and nothing outside the spans is read or written).
 * max_q_len and max_kv_len are the largest n and len that the caller expects (0: unknown). They choose how the work is cut and
 * bound nothing: longer sequences are computed too, only less evenly spread. Without max_q_len a step of decode rows also launches
 * what prompt chunks need. In a batch of more than 704 sequences each one's keys stay with one workgroup a KV head.
 * Unlike RoostPagedAttentionParams, a window_left of 0 (each query sees itself) is taken, and of the negative ones -1 alone; a
 * negative cap and a window without causal are refused.
 * Scores and sums are f32; each probability is rounded to bf16 once, in front of its product with v. The sums before their
 * division stay in f32 where |v| < 2^120 / len. q is 16-byte aligned, its token stride a multiple of 8; q_heads is a multiple of
 * kv_heads, at most 32 to each; tokens are below 2^24. */
typedef struct RoostAmdPagedAttentionF4Params {
  uint32_t struct_size;
  uint32_t abi_minor;
  RoostDeviceSpan q;      /* bf16 [tokens, q_heads, head_dim], tokens q_stride apart (0: contiguous) */
  RoostDeviceSpan output; /* bf16 [tokens, q_heads, head_dim] */
  RoostDeviceSpan lse;    /* f32 [tokens, q_heads], or NULL */
  RoostAmdCacheF4 cache;
  RoostDeviceSpan cu_seqlens;   /* [batch + 1] i32 */
  RoostDeviceSpan block_tables; /* i32 */
  RoostDeviceSpan kv_lens;      /* i32 */
  RoostDeviceSpan kv_indptr;    /* [batch + 1] i32, or NULL */
  RoostDeviceSpan sequences;    /* [batch] i32, or NULL */
  uint32_t batch;
  uint32_t tokens;
  uint32_t q_heads;
  uint32_t q_stride;
  uint32_t table_rows;
  uint32_t max_blocks;
  uint32_t max_q_len;
  uint32_t max_kv_len;
  float sm_scale;        /* at most 2^126; 0 = 1/sqrt(head_dim) */
  float logits_soft_cap; /* 0 = off */
  int32_t window_left;   /* -1 = no sliding window */
  uint32_t causal;
} RoostAmdPagedAttentionF4Params;

/* Device scratch of a call (partial results of sequences whose keys are split). Undefined before and after; a function of the
 * record's numbers, not of its device data. */
ROOST_API RoostStatus roost_amd_paged_attention_f4_workspace(RoostContext* ctx, const void* params,
                                                             RoostWorkspaceSizes* sizes);
ROOST_API RoostStatus roost_amd_paged_attention_f4_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                                       void* stream);

/* ---- Pages of a cache ---------------------------------------------------------------------------------------------------
 * Pools of any element type whose page p is page_bytes bytes at address + layer * layer_bytes + p * page_bytes, in each of
 * `layers` layers. Addresses are 16-byte aligned, page_bytes and layer_bytes multiples of 16; pools do not overlap. */
typedef struct RoostAmdPagePool {
  void* address;
  uint64_t page_bytes;
  uint64_t layer_bytes;
  uint32_t layers;
  uint32_t reserved0;
} RoostAmdPagePool;

#define ROOST_AMD_MAX_PAGE_POOLS 16u

/* CacheCopy: page pairs[i][0] to page pairs[i][1] in every layer of every pool, with the result of one pair after the other
 * (RecurrentStateCopy's order). A pair that names a page outside the pools is skipped. Pairs that share no page with another
 * as a destination run side by side; the others one after the other. count is at most 65,536. */
typedef struct RoostAmdCacheCopyParams {
  uint32_t struct_size;
  uint32_t abi_minor;
  const RoostAmdPagePool* pools; /* host memory, read during the call */
  uint32_t pool_count;
  uint32_t pages;
  RoostDeviceSpan pairs; /* [count, 2] i32 */
  uint32_t count;
  uint32_t reserved0;
} RoostAmdCacheCopyParams;

/* Device scratch of a call of more than 1,024 pairs; zero bytes for others, which take a NULL workspace. */
ROOST_API RoostStatus roost_amd_cache_copy_workspace(RoostContext* ctx, const void* params, RoostWorkspaceSizes* sizes);
ROOST_API RoostStatus roost_amd_cache_copy_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws, void* stream);

/* Which pages the sequences hold, on the device: sequence s has lengths[s] tokens in the first ceil(lengths[s] / page_size)
 * pages of its row of block_tables; refs[p] is how many rows hold page p, 0 for a free page. Whole pages may be shared; a last,
 * partly filled page is its sequence's own, so that it can be written. The calls below keep to that, and read the state from
 * before the call throughout: a request does not see what another of the same call did. Free pages are given in the order of
 * the requests, lowest page first. Page ids outside the pool are left alone wherever a row holds them. */
typedef struct RoostAmdCachePagesParams {
  uint32_t struct_size;
  uint32_t abi_minor;
  const RoostAmdPagePool* pools; /* host memory, read during the call; fork and compact */
  uint32_t pool_count;
  uint32_t count;               /* requests, at most 1,024 */
  RoostDeviceSpan block_tables; /* [sequences, max_blocks] i32 */
  RoostDeviceSpan lengths;      /* [sequences] i32 */
  RoostDeviceSpan refs;         /* [pages] i32 */
  RoostDeviceSpan requests;     /* i32: fork [count, 2] (parent, child), grow and free [count] */
  RoostDeviceSpan cu_seqlens;   /* grow: [count + 1] i32 */
  RoostDeviceSpan slot_mapping; /* grow: [tokens] i64 */
  RoostDeviceSpan status;       /* i32: fork and grow [count], or NULL; compact [1], or NULL */
  uint32_t sequences;
  uint32_t max_blocks;
  uint32_t pages;               /* at most 4,194,304 */
  uint32_t page_size;           /* a power of two */
} RoostAmdCachePagesParams;

/* Device scratch of fork, grow and compact: one size for all three, from `pages` alone. Undefined before and after. */
ROOST_API RoostStatus roost_amd_cache_pages_workspace(RoostContext* ctx, const void* params, RoostWorkspaceSizes* sizes);

/* CacheFork: the child gets its parent's length and pages: whole ones shared (refs + 1), a last partly filled one copied, in
 * every layer of every pool, into a free page (refs 1). status 1. Status 0, nothing done: the parent is empty, the child is
 * not, either is no sequence, an earlier request names the same child, or no free page is left for it. */
ROOST_API RoostStatus roost_amd_cache_fork_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws, void* stream);

/* CacheGrow: sequence requests[i] gets room for cu_seqlens[i + 1] - cu_seqlens[i] more tokens: free pages (refs 1) at the end of
 * its row, its new length, and slot_mapping[cu_seqlens[i] ..] = its new tokens' slots, as CacheWrite and CacheWriteF4 take
 * them. status 1. Status 0 and slots of -1, nothing else done: no such sequence, one that an earlier request names, more tokens
 * than its row holds, or fewer free pages left than this request and the earlier ones need. Entries of slot_mapping behind the
 * last request's are left as they were; cu_seqlens[0] = 0 and cu_seqlens does not go backwards. */
ROOST_API RoostStatus roost_amd_cache_grow_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws, void* stream);

/* CacheFree: sequence requests[i] ends: refs - 1 for each of its pages, their entries of its row -1, its length 0. Empty
 * sequences, and numbers of no sequence, are skipped; naming one twice frees it once. */
ROOST_API RoostStatus roost_amd_cache_free_run(RoostContext* ctx, const void* params, void* stream);

/* CacheCompact: with `live` pages in use (refs above 0), the i-th used page from page `live` on moves to the i-th free page
 * below it, in every layer of every pool, with its refs; the sequences' rows follow. Then pages 0 .. live - 1 are in use and
 * the others free. status[0] = live. What the others hold stays. */
ROOST_API RoostStatus roost_amd_cache_compact_run(RoostContext* ctx, const void* params, const RoostWorkspace* ws,
                                                  void* stream);

/* The plan region: the batch tables and slot mapping of one worker step, from its sequences. Replaces the worker's
 * PlanRegionWriter.Fill (reference src/Starlings.Roost.Worker/Eager/PlanRegionWriter.cs:19-64), which the reference runs
 * in C# on a host mirror of the region before one host-to-device copy. For sequence b (in order):
 *   q_indptr[b] = cu_seqlens[b] = token_start[b]; kv_indptr[b] = blocks listed before b;
 *   kv_indices[kv_indptr[b] + i] = its block i; kv_last_page_len[b] = kv_length[b] - (its blocks - 1) * block_size;
 *   state_slots[b] = recurrent_slot[b];
 *   for t < token_count[b], at index = token_start[b] + t and position = position_offset[b] + t:
 *     positions[index] = position; slot_mapping[index] = block[position / block_size] * block_size + position % block_size;
 * and the [batch] entries of q_indptr and cu_seqlens are the last sequence's token_start + token_count, of kv_indptr
 * the number of blocks. The region's token ids and sampling rows (embedding and sampler inputs) are not written here.
 * state_slots / recurrent_slot and positions may be NULL (not written). Entries no sequence writes are left alone. */
typedef struct RoostAmdPlanRegion {
  uint32_t batch;                 /* sequences */
  uint32_t tokens;                /* entries of positions and slot_mapping */
  uint32_t block_size;            /* tokens per KV page, > 0 */
  uint32_t reserved0;             /* 0 */
  const int32_t* token_start;     /* [batch] */
  const int32_t* token_count;     /* [batch] */
  const int32_t* position_offset; /* [batch]: position of the sequence's first token of this step */
  const int32_t* kv_length;       /* [batch]: keys after this step */
  const int32_t* block_indptr;    /* [batch + 1], from 0: sequence b's blocks are blocks[block_indptr[b] ..) */
  const int32_t* blocks;          /* [block_indptr[batch]] */
  const int32_t* recurrent_slot;  /* [batch] or NULL */
  int32_t* q_indptr;              /* [batch + 1] */
  int32_t* cu_seqlens;            /* [batch + 1] */
  int32_t* kv_indptr;             /* [batch + 1] */
  int32_t* kv_indices;            /* [block_indptr[batch]] */
  int32_t* kv_last_page_len;      /* [batch] */
  int32_t* state_slots;           /* [batch] or NULL */
  int32_t* positions;             /* [tokens] or NULL */
  int64_t* slot_mapping;          /* [tokens] */
} RoostAmdPlanRegion;

/* Host memory: fills the tables on the calling thread. A sequence whose tokens fall outside [0, tokens), whose
 * positions reach past its blocks, or whose block_indptr goes backwards is refused with ROOST_STATUS_INVALID_ARGUMENT
 * (the reference's Fill throws on the same plans) and nothing is written. */
ROOST_API RoostStatus roost_amd_plan_region_fill(const RoostAmdPlanRegion* region);

/* Device memory: one launch on `stream` writes the same tables on the GPU from the device copies of the sequences'
 * fields, so a step's per-token work never crosses PCIe. The device arrays are not validated on the host: a token
 * index outside [0, tokens) is skipped and a position past its sequence's blocks gets slot -1 (CacheWrite skips it). */
ROOST_API RoostStatus roost_amd_plan_region_run(RoostContext* ctx, const RoostAmdPlanRegion* region, void* stream);

/* The same tables read straight from a C2 step plan: the shared buffer the engine writes (RoostStepPlanHeader and its
 * tables, reference kernels/include/roost_worker_shm.h:57-141), in place of the worker's StepPlanReader.Read +
 * PlanRegionWriter.Fill (src/Starlings.Roost.Worker/Eager/StepPlanReader.cs:195-345, PlanRegionWriter.cs:19-64).
 * Sequence b's KV blocks are the first ceil((position_offset + token_count) / block_size) ids of its group_blocks entry
 * b * group_count + attention_group; its keys after the step are position_offset + token_count. Besides the tables of
 * roost_amd_plan_region_fill it writes ids[index] = token_ids[index] and, for each sequence with the sample flag
 * (0x2) in plan order, rows[r] = its last token index. The plan is checked as the reader checks the fields used here
 * (magic, table bounds and counts, contiguous non-empty token ranges, consecutive positions, group_blocks_start ==
 * b * group_count, enough blocks listed); a plan that fails, or outputs shorter than it needs, is refused with
 * ROOST_STATUS_INVALID_ARGUMENT and nothing is written. Host memory only. */
typedef struct RoostAmdStepTables {
  uint32_t attention_group;  /* the state group whose block lists hold the attention KV blocks */
  uint32_t block_size;       /* tokens per KV page, > 0 */
  uint32_t max_batch;        /* sequences the per-sequence outputs hold (indptr arrays hold max_batch + 1) */
  uint32_t max_tokens;       /* entries of ids, positions and slot_mapping */
  uint32_t max_blocks;       /* entries of kv_indices */
  uint32_t batch;            /* out: sequences */
  uint32_t tokens;           /* out: tokens */
  uint32_t blocks;           /* out: kv_indices entries written */
  uint32_t rows_written;     /* out: sampling rows written */
  uint32_t attention_blocks; /* blocks in the attention KV pool, > 0: block ids outside [0, attention_blocks) are refused */
  int32_t* q_indptr;         /* [batch + 1] */
  int32_t* cu_seqlens;       /* [batch + 1] */
  int32_t* kv_indptr;        /* [batch + 1] */
  int32_t* kv_indices;       /* [blocks] */
  int32_t* kv_last_page_len; /* [batch] */
  int32_t* state_slots;      /* [batch] or NULL */
  int32_t* ids;              /* [tokens] or NULL */
  int32_t* positions;        /* [tokens] or NULL */
  int64_t* slot_mapping;     /* [tokens] */
  int32_t* rows;             /* [max_batch] or NULL */
} RoostAmdStepTables;

ROOST_API RoostStatus roost_amd_plan_region_from_step(const void* plan, uint64_t plan_bytes, RoostAmdStepTables* tables);

#ifdef __cplusplus
}
#endif

#endif /* ROOST_AMD_H_ */
