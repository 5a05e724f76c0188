/*
 * libnxrt_ep_rocm.so — MI355X (gfx950) execution provider for com.microsoft::MatMulNBits, bits=4.
 *
 * Three groups of C entry points:
 *   1. the nxrt plugin exports (nxrt_abi.h) and the nxmem allocator exports (nxmem_abi.h);
 *   2. a C mirror of the reference's ExecutionProvider / KernelFactory / Kernel traits for this one
 *      operator, because NxrtKernelVtable.execute (vtable.rs:108-122) carries raw pointers only —
 *      no shapes, dtypes or attributes — and the reference's own nxrt wrapper still leaves
 *      get_capability / compile / get_allocator unwired (vtable.rs:355-398);
 *   3. entry points for the pieces the parity contract names one by one (dequantized weights,
 *      activation codes, int32 block accumulators) and for timing on the provider's stream.
 *
 * Every pointer named "device" is device memory obtained from nxrt_rocm_ep_allocate (or any HIP
 * allocation on the provider's GPU). Nothing here takes or returns a torch / C++ type. All calls on
 * one provider are issued on that provider's single HIP stream, in call order; host-visible results
 * require nxrt_rocm_ep_sync or a copy_to_host (which synchronises).
 */
#ifndef NXRT_EP_ROCM_H
#define NXRT_EP_ROCM_H

#include "nxmem_abi.h"
#include "nxrt_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct NxrtRocmEp NxrtRocmEp;                     /* one provider = one GPU + one stream */
typedef struct NxrtRocmMatMulNBits NxrtRocmMatMulNBits;   /* one kernel = one MatMulNBits node */

/* ---- ExecutionProvider (crates/onnx-runtime-ep-api/src/provider.rs:708-1600) ------------------ */

/* initialize(&EpConfig) — provider.rs:93 (string map). keys/values: n_config NUL-terminated pairs.
 * Known keys: "acc4_rounding" = "mlas" (ties to even, default) | "native" (ties away) | "auto" (native below
 *             "acc4_native_below" rows, else mlas: the CPU provider's route, matmul_nbits.rs:640-660);
 *             "prepack" = "1" (default: constant weights are copied once into the decode kernels' streaming order) | "0";
 *             "dense_gemm_min_rows" = rows from which a 16-bit call expands the weights to a dense [N, K] matrix and runs
 *             the library GEMM (hipBLASLt) instead of this provider's own tiled kernel: opt-in, default "0" = never (256 once
 *             "dense_weights" = "resident" is chosen; the CUDA provider's dequantize + cuBLASLt route,
 *             onnx-runtime-ep-cuda/src/kernels/matmul_nbits.rs:6176-6222);
 *             "dense_gemm_max_mb" = largest dense copy of one weight (default 1024, as matmul_nbits.rs:6212);
 *             "dense_weights" = "transient" (default: one buffer per provider, refilled by every such call) |
 *             "resident" (a constant weight keeps its dense copy: 2 bytes per weight of HBM for a call that is the
 *             GEMM alone);
 *             "rmsnorm_in_kernel_max_cols" = widest launch (columns; both projections of a gate/up node together) whose
 *             decode kernel applies an RMS-normalization prologue itself at up to four rows; wider nodes and "0" normalize
 *             in a launch of their own (default 8192: every workgroup repeats the row's normalization, which pays only
 *             while there are few of them);
 *             "decode_waves", "decode_col_groups", "prefill_tile" = launch overrides (tests, tuning).
 * The same settings are read from NXRT_ROCM_RMSNORM_IN_KERNEL_MAX_COLS, NXRT_ROCM_ACC4_ROUNDING, NXRT_SQNBIT_DECODE_MIN, NXRT_ROCM_PREPACK,
 * NXRT_ROCM_DENSE_GEMM_MIN_ROWS, NXRT_ROCM_DENSE_GEMM_MAX_MB, NXRT_ROCM_DENSE_WEIGHTS, NXRT_ROCM_DECODE_WAVES,
 * NXRT_ROCM_DECODE_COL_GROUPS, NXRT_ROCM_PREFILL_TILE when the map does not give them. */
NxrtStatus nxrt_rocm_ep_create(uint32_t device_ordinal, const char* const* config_keys,
                               const char* const* config_values, uint32_t n_config, NxrtRocmEp** out_ep);
/* shutdown + drop. Frees the stream and every buffer the provider still owns. Kernels and allocator vtables made from the
 * provider each hold a reference to it: the host may release them and the provider in any order, and the provider's
 * resources go with the last of them. */
void nxrt_rocm_ep_release(NxrtRocmEp* ep);
/* name() / device_type() / device_id() / memory_vendor_id() — provider.rs:708-731. */
const char* nxrt_rocm_ep_name(const NxrtRocmEp* ep);                   /* "RocmExecutionProvider" */
uint32_t nxrt_rocm_ep_device_type(const NxrtRocmEp* ep);               /* NXRT_DEVICE_ROCM */
uint32_t nxrt_rocm_ep_device_id(const NxrtRocmEp* ep);
uint32_t nxrt_rocm_ep_memory_vendor_id(const NxrtRocmEp* ep);          /* 0x1002 */
/* Architecture string ("gfx950..."), compute units, bytes of device memory. */
NxrtStatus nxrt_rocm_ep_device_info(const NxrtRocmEp* ep, char* arch, size_t arch_len, uint32_t* compute_units, uint64_t* total_memory);
/* allocate(size, align) / deallocate — provider.rs (DeviceBuffer); align <= 256 is always met. */
NxrtStatus nxrt_rocm_ep_allocate(NxrtRocmEp* ep, size_t size, size_t align, void** out_device);
NxrtStatus nxrt_rocm_ep_deallocate(NxrtRocmEp* ep, void* device);
/* copy_from_host / copy_to_host (provider.rs:1434,1502), copy (device to device), sync. */
NxrtStatus nxrt_rocm_ep_copy_from_host(NxrtRocmEp* ep, void* dst_device, const void* src_host, size_t bytes);
NxrtStatus nxrt_rocm_ep_copy_to_host(NxrtRocmEp* ep, void* dst_host, const void* src_device, size_t bytes);
NxrtStatus nxrt_rocm_ep_copy(NxrtRocmEp* ep, void* dst_device, const void* src_device, size_t bytes);
NxrtStatus nxrt_rocm_ep_sync(NxrtRocmEp* ep);
/* A benchmark's yardstick, not part of the reference's interface: enqueues a kernel that reads `bytes` of device memory (16-byte
 * loads, four in flight per lane, one workgroup per 16 KiB) and keeps nothing. Its time is the least any kernel can spend
 * pulling that many bytes from HBM; bench.py --read-floor reports it beside the decode kernels' times. */
NxrtStatus nxrt_rocm_ep_read_probe(NxrtRocmEp* ep, const void* src_device, size_t bytes);
/* Diagnostic for benchmarks (no counterpart in the reference): bytes per clock one CU's LDS moves with `waves` waves (1..16)
 * of a workgroup repeating 16-byte accesses. mode 0: reads; 1: writes; 2: global memory straight into LDS; 3: half the waves
 * read while the others write. Synchronous; allocates and frees its own small buffers. */
NxrtStatus nxrt_rocm_ep_lds_probe(NxrtRocmEp* ep, uint32_t mode, uint32_t waves, uint32_t iters, double* bytes_per_clock);
/* The nxrt EP vtable whose ctx is this provider (what NxrtEpFactoryVtable.create_ep hands out);
 * the inverse recovers the provider from a vtable obtained through the plugin exports. */
NxrtRocmEp* nxrt_rocm_ep_from_vtable(const NxrtEpVtable* vtable);

/* ---- KernelFactory + Kernel (registry.rs:39-45, kernel.rs:548-706) ----------------------------- */

/* Node attributes of MatMulNBits. `present` has bit i set when attribute i was on the node:
 * 0=K 1=N 2=bits 3=block_size 4=accuracy_level 5=weight_prepacked
 * (onnx-runtime-ep-cpu/src/kernels/matmul_nbits.rs:1410-1481; bits 2, 4 (default) or 8 as there - 4 is the tuned path, and the
 * only one with accuracy_level = 4; weight_prepacked must be 0), and 6=folded_bias: the marker an optimizer pass sets
 * when it folds a standalone Add into the bias input (the CUDA provider's `_cuda_matmul_nbits_folded_bias`,
 * onnx-runtime-ep-cuda/src/optimizer.rs:35, kernels/matmul_nbits.rs:1189-1212). With folded_bias = 1 and a 16-bit
 * output the result is round(round(acc) + bias), bit for bit what the two nodes gave; otherwise round(acc + bias).
 * 7=gate_up_swiglu, 8=decomposed_silu: the CUDA provider's fused gate/up node (`_cuda_gate_up_swiglu`, `_cuda_decomposed_silu`,
 * onnx-runtime-ep-cuda/src/optimizer.rs:14, 36-46; kernels/matmul_nbits.rs:9017-9130). With gate_up_swiglu = 1 the inputs are
 * [x, W_gate, scales_gate, W_up, scales_up, (gamma: must be absent), (zp_gate, zp_up: both or neither)], x and Y Float16 or
 * BFloat16, and Y = round16(silu(round16(x W_gate^T)) * round16(x W_up^T)) - bit for bit what the two projections followed by
 * the 16-bit silu-and-multiply give (kernels/matmul_nbits.rs:4207-4233, 4375-4386). workspace_requirement then sizes the
 * two 16-bit [M, N] intermediates.
 * 9=rmsnorm_prologue, 10=rmsnorm_epsilon (default 1e-5): the CUDA provider's `_cuda_matmul_nbits_rmsnorm_prologue` / `_epsilon`
 * (optimizer.rs:48-60). The activations (Float16 or BFloat16, K % 128 == 0) are RMS-normalized before the product,
 * x' = round16((x / sqrt(mean(x^2) + epsilon)) * gamma), with gamma [K] (Float32 or the activations' dtype) at input 6, or
 * input 5 of the fused gate/up node - the arithmetic and summation order of kernels/matmul_nbits.rs:4125-4205.
 * struct_size tells which fields the caller's struct has: fields past its end are read as 0. */
typedef struct NxrtRocmMatMulNBitsAttrs {
  uint32_t struct_size;
  uint32_t present;
  int64_t K, N, bits, block_size, accuracy_level, weight_prepacked;
  int64_t folded_bias;
  int64_t gate_up_swiglu, decomposed_silu;
  int64_t rmsnorm_prologue;
  double rmsnorm_epsilon;
} NxrtRocmMatMulNBitsAttrs;

/* C layout of TensorView / TensorMut (crates/onnx-runtime-ep-api/src/tensor.rs:132-143, 241).
 * data == NULL marks an absent optional input (tensor.rs:173-192). strides are in elements;
 * NULL means contiguous row-major. */
typedef struct NxrtRocmTensorView {
  void* data;
  uint32_t dtype;        /* NXRT_DT_* */
  uint32_t ndim;
  const uint64_t* shape;
  const int64_t* strides;
  uint64_t byte_offset;
  uint32_t device_type;  /* NXRT_DEVICE_* */
  uint32_t device_index;
} NxrtRocmTensorView;

/* kernel.rs:508-524 */
typedef struct NxrtRocmWorkspaceRequirement {
  uint64_t bytes;
  uint64_t alignment;
} NxrtRocmWorkspaceRequirement;

/* supports_op(node, opset, shapes, dtypes, layouts) -> KernelMatch (kernel.rs:118-130).
 * Returns 1 when the provider takes the node; otherwise 0 with an actionable reason. */
int nxrt_rocm_ep_supports_matmul_nbits(const NxrtRocmEp* ep, const NxrtRocmMatMulNBitsAttrs* attrs,
                                       const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason, size_t reason_len);

/* get_kernel -> KernelFactory::create (matmul_nbits.rs:1410-1481): attribute checks, same messages. */
NxrtStatus nxrt_rocm_matmul_nbits_create(NxrtRocmEp* ep, const NxrtRocmMatMulNBitsAttrs* attrs,
                                         const NxrtTensorDesc* input_shapes, uint32_t n_inputs,
                                         NxrtRocmMatMulNBits** out_kernel);
/* Kernel::set_constant_inputs (kernel.rs:548-, matmul_nbits.rs:1483-1488). */
void nxrt_rocm_matmul_nbits_set_constant_inputs(NxrtRocmMatMulNBits* kernel, const uint8_t* is_constant, uint32_t n);
/* Kernel::workspace_requirement: scratch for these input shapes (accuracy_level 4 activation codes). */
NxrtStatus nxrt_rocm_matmul_nbits_workspace_requirement(const NxrtRocmMatMulNBits* kernel, const NxrtTensorDesc* inputs,
                                                        uint32_t n_inputs, NxrtRocmWorkspaceRequirement* out);
/* Kernel::execute / execute_with_workspace (matmul_nbits.rs:1490-1600, 2320-2330).
 * inputs: A, B, scales, [zero_points], [g_idx], [bias]; outputs: Y. workspace may be NULL: the
 * kernel then keeps its own scratch, grown on demand (an allocation inside the call). B is [N, kb, block_size * bits / 8],
 * zero_points [N, ceil(kb * bits / 8)]; g_idx (Int32 [K] or [kb * block_size], accuracy_level 0 only) is range-checked on first
 * use (matmul_nbits.rs:3515-3521). bias has N elements in any shape ([N], [1, N], [1, 1, N]: broadcast over the rows), or
 * rows * N elements: a per-token residual folded into the bias slot, row stride N
 * (onnx-runtime-ep-cuda/src/kernels/matmul_nbits.rs:7728-7735, 7891-7897). A required tensor with a NULL data pointer is
 * refused with a status, never launched. Fused nodes (gate_up_swiglu, rmsnorm_prologue) take their own input lists, see the attributes. */
NxrtStatus nxrt_rocm_matmul_nbits_execute(NxrtRocmMatMulNBits* kernel, const NxrtRocmTensorView* inputs, uint32_t n_inputs,
                                          NxrtRocmTensorView* outputs, uint32_t n_outputs,
                                          void* workspace_device, uint64_t workspace_bytes);
/* execute for callers that cannot allocate: code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc. It has no counterpart in the reference. Same inputs, outputs, validation and results as
 * nxrt_rocm_matmul_nbits_execute on a plain MatMulNBits node (fused gate/up and RMS-normalization nodes are refused), but the
 * call allocates and frees nothing and calls no library routine that might: whatever scratch its kernels need (activation
 * codes and scales of accuracy_level 4; partial sums of a tall call that cuts K into slices) lives in a static device array
 * of NXRT_ROCM_STATIC_SCRATCH_BYTES that is part of the library's code object - one copy per GPU, held until the process
 * ends, its address resolved once when the provider is created. Consequences:
 *   - a call whose scratch does not fit is refused with INVALID_ARGUMENT and the sizes (accuracy_level 4 needs about
 *     rows * K * (1 + 12 / block_size) bytes: at K = 8192, block 64, up to ~860 rows); optional scratch (K slices) shrinks to fit;
 *   - nothing is set up on the fly: constant weights that have no repacked copy yet are streamed in the caller's layout, the
 *     library GEMM route is not taken, a g_idx tensor must have been range-checked by an earlier execute;
 *   - every call on one GPU shares that GPU's array, which keeps the last call's contents (the kernels overwrite all they
 *     read). Calls through one provider are ordered by its stream. Calls through different providers on the same GPU are
 *     chained on the GPU: each call records an event behind its launches, and a call on another stream waits for it
 *     (hipStreamWaitEvent) before its own - they run one after the other, in the order in which the host made them. The
 *     exception is a call made while its provider has a graph capture open: it neither waits nor records (an event from
 *     outside a capture cannot be waited for inside one), so graphs recorded through several providers of one GPU must not
 *     be replayed at the same time; the host orders them. */
#define NXRT_ROCM_STATIC_SCRATCH_BYTES (8u << 20)
NxrtStatus nxrt_rocm_matmul_nbits_execute_static(NxrtRocmMatMulNBits* kernel, const NxrtRocmTensorView* inputs, uint32_t n_inputs,
                                                 NxrtRocmTensorView* outputs, uint32_t n_outputs);
/* Kernel::estimated_flops (matmul_nbits.rs:2338): 2*M*N*K, 0 when M is not known from the shapes. */
uint64_t nxrt_rocm_matmul_nbits_estimated_flops(const NxrtRocmMatMulNBits* kernel);
/* record_kernel_variant (kernel.rs:361): which kernel served the last execute. */
const char* nxrt_rocm_matmul_nbits_last_variant(const NxrtRocmMatMulNBits* kernel);
/* record_kernel_metrics (onnx-runtime-ep-api/src/kernel.rs:243-267, called at matmul_nbits.rs:1588-1597): what the last plain
 * execute moved and computed by the reference's count - bytes = the bytes of every present input tensor + the output's;
 * flops = 2*M*N*K, + M*N with a bias. Zero before the first call. */
void nxrt_rocm_matmul_nbits_last_metrics(const NxrtRocmMatMulNBits* kernel, uint64_t* flops, uint64_t* bytes);
void nxrt_rocm_matmul_nbits_release(NxrtRocmMatMulNBits* kernel);
/* The same kernel behind the nxrt kernel vtable (raw pointers only: the shapes are those given at
 * create time, M taken from input_shapes[0]). The host calls release(ctx) once. */
NxrtStatus nxrt_rocm_matmul_nbits_as_vtable(NxrtRocmMatMulNBits* kernel, NxrtKernelVtable** out_vtable);

/* ---- pieces of the operator the parity contract checks one by one ------------------------------ */

/* w[n,k] = (q - zp) * scale as f32 [N, K] (matmul_nbits.rs:1360-1363, 3502-3661; the CUDA sibling's
 * matmul_nbits_dequant_f32, ep-cuda matmul_nbits.rs:414-455). scales dtype: f32 / f16 / bf16. */
NxrtStatus nxrt_rocm_matmul_nbits_dequantize(NxrtRocmEp* ep, const void* b_device, const void* scales_device, uint32_t scale_dtype,
                                             const void* zero_points_device, uint64_t n, uint64_t k, uint32_t block_size,
                                             float* out_nk_device);
/* The same at bits = 2, 4 or 8 (NBitsLayout, matmul_nbits.rs:1276-1321): b is [N, kb, block_size * bits / 8], zero points
 * [N, ceil(kb * bits / 8)], default zero point 1 << (bits - 1). */
NxrtStatus nxrt_rocm_matmul_nbits_dequantize_bits(NxrtRocmEp* ep, const void* b_device, const void* scales_device, uint32_t scale_dtype,
                                                  const void* zero_points_device, uint64_t n, uint64_t k, uint32_t block_size, uint32_t bits,
                                                  float* out_nk_device);
/* accuracy_level=4 activation quantizer (simd_quant.rs:131-143 / sqnbitgemm_kernel_avx512.cpp:349-426).
 * rounding: 0 = ties to even (MLAS), 1 = ties away from zero (native). qa: int8 [M, kb*bs];
 * qscale: f32 [M, kb]. */
NxrtStatus nxrt_rocm_matmul_nbits_quantize_a(NxrtRocmEp* ep, const void* a_device, uint32_t a_dtype, uint64_t m, uint64_t k,
                                             uint32_t block_size, uint32_t rounding, int8_t* qa_device, float* qscale_device);
/* acc[m,n,b] = sum_{k in block b} qa[m,k] * (q[n,k] - zp[n,b]), int32 [M, N, kb]
 * (matmul_nbits.rs:3360-3412 + 9159-9177; qnbitgemm.cpp:727-893). */
NxrtStatus nxrt_rocm_matmul_nbits_block_acc(NxrtRocmEp* ep, const int8_t* qa_device, const void* b_device,
                                            const void* zero_points_device, uint64_t m, uint64_t n, uint64_t k,
                                            uint32_t block_size, int32_t* acc_device);

/* The same integers as the production kernels hold them: with a probe buffer set (int32 [M, N, kb] device memory, NULL
 * clears it), every later accuracy_level=4 execute of this kernel that runs on the int8 matrix cores also stores each
 * block accumulator at the moment it is scaled into the f32 result (matmul_nbits.rs:9159-9177: `acc` of `int8_row`).
 * The launch is the same kernel with the store compiled in; a call the dot-product catch-all would serve is refused. */
NxrtStatus nxrt_rocm_matmul_nbits_set_block_acc_probe(NxrtRocmMatMulNBits* kernel, int32_t* acc_device, uint64_t capacity_elements);
/* Device buffers the kernel object has replaced (outgrown scratch, a repacked or dense copy of weights that changed) and
 * keeps until it is released, because a HIP graph recorded earlier may still replay through them. */
uint64_t nxrt_rocm_matmul_nbits_retired_buffers(const NxrtRocmMatMulNBits* kernel);

/* ---- operators beside MatMulNBits: what stands between the quantized products of a decoder layer ---- */

/* One node of one of the operators below. The contract is that of a MatMulNBits kernel: tensors contiguous and on the provider's GPU, an absent optional
 * tensor has data = NULL, calls run on the provider's stream in call order, one call at a time per node. No node copies or remembers its weights. Outputs may not
 * overlap inputs unless said so. A node keeps a reference on its provider. Calls may be recorded into a graph; a call that needs scratch takes the caller's workspace
 * or the node's own, which an eager call of that height has to have made before (nothing is allocated while a capture is open). Outgrown scratch of the node's own is
 * freed while the provider has opened no capture yet; from then on, since a graph may name it, it stays until the node is released. */
typedef struct NxrtRocmNode NxrtRocmNode;

/* com.microsoft::QMoE with activation_type "swiglu" (or "silu" with fc3; the struct has no activation_type: a host keeps nodes with another one, or with none, whose
 * default is "relu", to itself): a mixture-of-experts layer over 4-bit weights, from router logits to the weighted sum.
 *   inputs: 0 input [.., H] Float16 / BFloat16; 1 router_probs [.., E] logits of any float type; 2 fc1_experts_weights [E, F, kb, block_size / 2] (or
 *           [E, F, kb * block_size / 2]) Uint8, 3 fc1_scales [E, F, kb], 4 fc1_experts_bias [E, F] or absent; 5, 6, 7 the same of fc2 ([E, H, ..] over I);
 *           8, 9, 10 of fc3 or absent; 11, 12, 13 zero points [E, F, ceil(kb / 2)] of fc1, fc2, fc3 or absent (8; fc1's come with fc3's).
 *           Packing is MatMulNBits's; scales of the input's type or Float32, all alike, as are the biases.
 *   output: [.., H] of the input's type.
 *   swiglu_fusion 1: F = 2 I, gate and up rows alternate; 2: I gate rows, then I up rows; 0: F = I, gate in fc1 and up in fc3.
 * For token t: p = softmax(logits); S = the k experts of the largest logits, the lowest index first among equal ones, without those whose p is 0; w = p, or p over
 * its sum on S with normalize_routing_weights. h = g sigmoid(activation_alpha g) (u + activation_beta), g <= swiglu_limit, |u| <= swiglu_limit (g, u: the
 * products with bias); y = sum over S of w (fc2 h + bias), summed in f32 and rounded once. With more than four tokens h is rounded to the input's type in between, and
 * y's error is then about 1.4 times its own rounding's; with up to four tokens (and up to 256 experts, 128 choices in all and rows * ceil(H / 2048) <= 12) h keeps
 * twice that type's bits, so that a token alone and the same token in a larger call may differ in their last bits. With Float16 an h beyond 65504 is an infinity
 * in either. A row whose logits are all -inf (padding) gives zeros and reads no expert; a NaN or +inf among a row's logits gives NaN. An infinity or NaN in a row
 * of `input` gives no finite value in that row, unless swiglu_limit takes each infinity back that comes of it.
 * Weights are exact (q - zp) * scale. block_size: a power of two >= 32. E <= 1024, k <= 64. Weights start at multiples of 16 bytes. */
typedef struct NxrtRocmQMoEAttrs {
  uint32_t struct_size;
  uint32_t present;      /* bit i: 0 k (default 1), 1 block_size (required), 2 expert_weight_bits (4), 3 normalize_routing_weights (0), 4 swiglu_fusion (0),
                            5 activation_alpha (1), 6 activation_beta (0), 7 swiglu_limit (none) */
  int64_t k, block_size, expert_weight_bits, normalize_routing_weights, swiglu_fusion;
  double activation_alpha, activation_beta, swiglu_limit;
} NxrtRocmQMoEAttrs;
int nxrt_rocm_ep_supports_qmoe(const NxrtRocmEp* ep, const NxrtRocmQMoEAttrs* attrs, const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason, size_t reason_len);
NxrtStatus nxrt_rocm_qmoe_create(NxrtRocmEp* ep, const NxrtRocmQMoEAttrs* attrs, NxrtRocmNode** out_node);

/* MatMulInt8: Y = (codes of A) B^T with a scale per token and per output channel.
 *   inputs: 0 A [.., K] Float32 / Float16 / BFloat16, or its Int8 codes; 1 B [N, K] Int8; 2 b_scale [N] of a float type; 3 a_scale [rows] Float32: with codes, and
 *           only then; 4 bias, absent, [N], or of Y's shape (a residual), of a float type.
 *   output: Y [.., N] of a float type.
 * Codes of a row: scale = max|a| / 127, code = a / scale to the nearest, ties to even; a row of zeros has scale 0. A row that holds an infinity or a NaN gives NaN.
 * Integer sums are exact. K < 131072. B starts at a multiple of 16 bytes where K is one of 16, else anywhere. */
typedef struct NxrtRocmMatMulInt8Attrs {
  uint32_t struct_size;
  uint32_t present;      /* bit i: 0 K, 1 N: both required */
  int64_t K, N;
} NxrtRocmMatMulInt8Attrs;
int nxrt_rocm_ep_supports_matmul_int8(const NxrtRocmEp* ep, const NxrtRocmMatMulInt8Attrs* attrs, const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason, size_t reason_len);
NxrtStatus nxrt_rocm_matmul_int8_create(NxrtRocmEp* ep, const NxrtRocmMatMulInt8Attrs* attrs, NxrtRocmNode** out_node);

/* GatedResidualNorm: the norm behind a block, its gate, the scaled residual stream, and the norm before the next block.
 *   inputs: 0 residual [.., H] Float32 / Float16 / BFloat16; 1 block [.., H] of the same type, or absent; 2 post_gamma [H] or absent (then no norm behind the
 *           block); 3 gate [H], or [G, H] with G dividing the rows (row r has gate r / (rows / G)), or absent; 4 pre_gamma [H] or absent (1); 5 pre_beta [H] or
 *           absent; 6 post_beta [H] or absent. Weights of the residual's type or Float32.
 *   outputs: 0 Z [.., H] of the residual's type or absent; 1 N [.., H] of that type, or Int8, or absent; 2 n_scale [rows] Float32: with Int8 N.
 *   p = post_gamma ? unit(block) * post_gamma + post_beta : block;  Z = residual_scale * residual + block_scale * gate * p;  N = unit(Z) * pre_gamma + pre_beta
 *   unit(x) = x / sqrt(mean(x^2) + epsilon), with layer_norm (x - mean) / sqrt(mean((x - mean)^2) + epsilon)
 * All in f32 (N from Z before its rounding), each output rounded once; Int8 N are codes as MatMulInt8 makes them. Z and a float N may be written over residual or
 * block. H <= 32768. */
typedef struct NxrtRocmGatedResidualNormAttrs {
  uint32_t struct_size;
  uint32_t present;      /* bit i: 0 epsilon (default 1e-5), 1 residual_scale (1), 2 block_scale (1), 3 layer_norm (0) */
  double epsilon, residual_scale, block_scale;
  int64_t layer_norm;
} NxrtRocmGatedResidualNormAttrs;
int nxrt_rocm_ep_supports_gated_residual_norm(const NxrtRocmEp* ep, const NxrtRocmGatedResidualNormAttrs* attrs, const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason,
                                              size_t reason_len);
NxrtStatus nxrt_rocm_gated_residual_norm_create(NxrtRocmEp* ep, const NxrtRocmGatedResidualNormAttrs* attrs, NxrtRocmNode** out_node);

/* ---- a paged 8-bit cache of keys and values, from the qkv product to the o product ----
 *
 * One layer's cache: k_cache [P, KV, B, D] and v_cache [P, KV, D, B] of Int8 or Float8E4M3FN codes (both alike), k_scale and v_scale [P, KV] Float32, not negative. A page
 * holds B tokens (16, 32, 64 or 128) of each of KV heads of D elements; the value of a code is code * scale of its page and head. Of the values a page holds
 * the tokens of one element side by side.
 * A call's new tokens are rows, T in all, those of a sequence behind one another: cumulative_lengths [N + 1] Int32, the first 0, sequence b has rows
 * cumulative_lengths[b] up to cumulative_lengths[b + 1]; rows behind the last sequence belong to none (without sequences, N = 0, all of them, and a call does nothing). past_lengths [N] Int32: tokens of a sequence in front of them.
 * block_table [N, W] Int32: token t of sequence b is slot t % B of page block_table[b, t / B].
 * What these tensors hold is read on the GPU and not reported: lengths are taken into 0 .. T, past lengths into 0 .. W B, and a page outside 0 .. P - 1 holds no tokens.
 * D: 64, 80, 96, 128 or 256 for CacheAttention, a multiple of 16 up to 256 for CacheAppend. W B < 2^30, N KV < 2^20; T < 2^26 for CacheAppend, T num_heads < 2^29 for
 * CacheAttention. */

/* com.microsoft::RotaryEmbedding: pairs of a head's elements turned by their row's position.
 *   inputs: 0 input [.., C] Float32 / Float16 / BFloat16, the heads of a row side by side; or, with rank 4, [N, H, S, D]; 1 position_ids Int64 / Int32, one for each row (of
 *           rank 4: [N, S]), or one element, the position of the first row of each sequence (the last dimension but one counts its rows); 2 cos_cache, 3 sin_cache [M, R / 2]
 *           of any float type, or both absent.
 *   output: of the input's shape and type; it may be written over the input.
 * D = head_size. The first num_heads heads of a row turn (0: all of C, which D then divides), what lies behind them passes through: packed queries, keys and values. R =
 * rotary_embedding_dim (0: D), even, up to 512: elements of a head that turn; pairs (i, i + R / 2), or (2 i, 2 i + 1) with interleaved.
 *   a' = a c - b s, b' = b c + a s; c, s = row position of the caches (a position that they do not have gives NaN), or magnitude * cos, sin(position * f_i) in 64 bits:
 *   f_i = rope_theta^(-2 i / R); scaling 1 (linear): f_i / factor; 2 (llama3): f_i / factor below low_freq_factor turns within original_max_position, f_i above
 *   high_freq_factor, in between a blend by turns; 3 (yarn): f_i / factor below beta_slow turns, f_i above beta_fast, in between a blend by pairs; magnitude =
 *   attention_factor, by default 1, with yarn and a factor above 1  0.1 ln(factor) + 1. Positions are exact up to 2^53. In f32, rounded once. */
typedef struct NxrtRocmRotaryEmbeddingAttrs {
  uint32_t struct_size;
  uint32_t present;      /* bit i: 0 head_size (required), 1 num_heads (0), 2 rotary_embedding_dim (0), 3 interleaved (0), 4 scaling (0), 5 original_max_position (8192),
                            6 rope_theta (10000), 7 factor (1), 8 low_freq_factor (1), 9 high_freq_factor (4), 10 beta_fast (32), 11 beta_slow (1), 12 attention_factor */
  int64_t head_size, num_heads, rotary_embedding_dim, interleaved, scaling, original_max_position;
  double rope_theta, factor, low_freq_factor, high_freq_factor, beta_fast, beta_slow, attention_factor;
} NxrtRocmRotaryEmbeddingAttrs;
int nxrt_rocm_ep_supports_rotary_embedding(const NxrtRocmEp* ep, const NxrtRocmRotaryEmbeddingAttrs* attrs, const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason,
                                           size_t reason_len);
NxrtStatus nxrt_rocm_rotary_embedding_create(NxrtRocmEp* ep, const NxrtRocmRotaryEmbeddingAttrs* attrs, NxrtRocmNode** out_node);

/* CacheAppend: new tokens' keys and values into their pages.
 *   inputs: 0 key [T, KV D] of a float type, 1 value of the same shape and type; or 0 packed rows [T, (num_heads + 2 KV) D], queries, keys, values, and 1 absent;
 *           2 k_cache, 3 v_cache, 4 k_scale, 5 v_scale, 6 cumulative_lengths, 7 past_lengths, 8 block_table.
 *   outputs: 0 k_cache, 1 v_cache, 2 k_scale, 3 v_scale: the inputs' own tensors, changed where they are.
 * A page whose first token is new gets scale = max|x| / top over its new tokens (top: 127, or 448), code = x / scale to the nearest, ties to even, at most top; a scale of 0 gives
 * codes 0. A page that has tokens gets scale' = max(scale, max|x| / top), and where that is larger, its codes become code * (scale / scale') to the nearest: each such
 * step adds up to half a step of rounding to the tokens before. An infinity or a NaN makes the scale NaN and the new codes 0 (and those before), until the page begins
 * again. Slots that no token has are left as they are. Two sequences may share pages, but a page that a call writes stands in one place of one table row only. */
typedef struct NxrtRocmCacheAppendAttrs {
  uint32_t struct_size;
  uint32_t present;      /* bit i: 0 num_heads (0; read for packed rows), 1 kv_num_heads (required), 2 head_size (required) */
  int64_t num_heads, kv_num_heads, head_size;
} NxrtRocmCacheAppendAttrs;
int nxrt_rocm_ep_supports_cache_append(const NxrtRocmEp* ep, const NxrtRocmCacheAppendAttrs* attrs, const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason, size_t reason_len);
NxrtStatus nxrt_rocm_cache_append_create(NxrtRocmEp* ep, const NxrtRocmCacheAppendAttrs* attrs, NxrtRocmNode** out_node);

/* CacheAttention: attention of the new tokens over their sequences' pages, which hold them already (CacheAppend goes before).
 *   inputs: 0 query [T, num_heads D] Float16 / BFloat16, or packed rows [T, (num_heads + 2 KV) D], whose first columns are read; 1 k_cache, 2 v_cache, 3 k_scale, 4 v_scale,
 *           5 cumulative_lengths, 6 past_lengths, 7 block_table.
 *   output: [T, num_heads D] of the query's type; rows of no sequence are left as they are.
 * Head h reads key head h / (num_heads / KV). New token i of sequence b sees slots t <= past_lengths[b] + i, with local_window_size the last so many of them (itself is one):
 *   y = softmax(z) v,  z = scale (q . k), with softcap  softcap tanh(z / softcap);  scale 0 (the default): 1 / sqrt(D).
 * A row that sees no slot is zero. Products, softmax and sums in f32 over f16 operands: codes exact, queries to 2^-22 of their row's largest, weights times
 * their page's scale rounded to 11 bits, or to 2^-36 of the largest such product that the row sees. A page of scale NaN gives NaN to the rows that see it, and to no other;
 * a NaN code of Float8E4M3FN (CacheAppend makes none) may reach rows that do not see its slot. */
typedef struct NxrtRocmCacheAttentionAttrs {
  uint32_t struct_size;
  uint32_t present;      /* bit i: 0 num_heads, 1 kv_num_heads, 2 head_size (all required), 3 local_window_size (-1: none), 4 scale (0), 5 softcap (0: none) */
  int64_t num_heads, kv_num_heads, head_size, local_window_size;
  double scale, softcap;
} NxrtRocmCacheAttentionAttrs;
int nxrt_rocm_ep_supports_cache_attention(const NxrtRocmEp* ep, const NxrtRocmCacheAttentionAttrs* attrs, const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason,
                                          size_t reason_len);
NxrtStatus nxrt_rocm_cache_attention_create(NxrtRocmEp* ep, const NxrtRocmCacheAttentionAttrs* attrs, NxrtRocmNode** out_node);

/* CachePages: the block table of the next step and the pages that move for it; or, with compact, a pool whose pages in use are its first ones.
 *   inputs: 0 block_table [S, W] Int32, 1 lengths [S] Int32: tokens cached of each sequence; 2 parents [S] Int32 or absent (each its own): the sequence that slot i goes on from,
 *           -1: none, the slot is free; 3 new_tokens [S] Int32 or absent (0): tokens that slot i is going to get; 4 .. 13 pools [L, P, ..] of any type: what moves with a page,
 *           L layers of P pages each.
 *   outputs: 0 next table [S, W] Int32, entries without a page -1; 1 next lengths [S] Int32: past_lengths of the next step; 2 moves [S, 2] ([P / 2, 2] with compact, in rising
 *           order) Int32: from, to, or -1; 3 counts [2] Int32: pages in use, pages that were missing; 4 .. the pools, the inputs' own tensors.
 * Slot i has the pages of its parent that are whole. A begun one stays with the lowest slot that continues it, if no slot has it as a whole page; the others get a copy in a
 * fresh page. Fresh pages, copies first and then those that new_tokens need, are the lowest that no slot has, dealt out slot by slot. Where they run out, entries are -1 and
 * count as missing (as do entries outside 0 .. P - 1), and no page that the inputs' table has is written, so that it still stands: a copy into one is not made, its entry and move are -1.
 * No count is kept beside the table: a page is free if no slot has it.
 * With compact (parents and new_tokens absent) the k-th page in use beyond the first n goes to the k-th free one among them, n the pages in use.
 * Without slots (S = 0) counts are 0 and moves -1, and the other tensors may be absent. S <= 1024, P <= 2^18, W page_size < 2^30, S W < 2^31. */
typedef struct NxrtRocmCachePagesAttrs {
  uint32_t struct_size;
  uint32_t present;      /* bit i: 0 page_size (required; 1..=2^20), 1 compact (0) */
  int64_t page_size, compact;
} NxrtRocmCachePagesAttrs;
int nxrt_rocm_ep_supports_cache_pages(const NxrtRocmEp* ep, const NxrtRocmCachePagesAttrs* attrs, const NxrtTensorDesc* inputs, uint32_t n_inputs, char* reason, size_t reason_len);
NxrtStatus nxrt_rocm_cache_pages_create(NxrtRocmEp* ep, const NxrtRocmCachePagesAttrs* attrs, NxrtRocmNode** out_node);

/* As the functions of the same names for MatMulNBits; but which inputs are constant makes no difference to a node, which reads its weights as they are in each call. */
void nxrt_rocm_node_set_constant_inputs(NxrtRocmNode* node, const uint8_t* is_constant, uint32_t n);
NxrtStatus nxrt_rocm_node_workspace_requirement(const NxrtRocmNode* node, const NxrtTensorDesc* inputs, uint32_t n_inputs, NxrtRocmWorkspaceRequirement* out);
NxrtStatus nxrt_rocm_node_execute(NxrtRocmNode* node, const NxrtRocmTensorView* inputs, uint32_t n_inputs, NxrtRocmTensorView* outputs, uint32_t n_outputs,
                                  void* workspace_device, uint64_t workspace_bytes);
const char* nxrt_rocm_node_last_variant(const NxrtRocmNode* node);
uint64_t nxrt_rocm_node_retired_buffers(const NxrtRocmNode* node);
void nxrt_rocm_node_release(NxrtRocmNode* node);

/* ---- timing on the provider's stream (HIP events) ---------------------------------------------- */

typedef struct NxrtRocmEvent NxrtRocmEvent;
NxrtStatus nxrt_rocm_ep_event_create(NxrtRocmEp* ep, NxrtRocmEvent** out_event);
NxrtStatus nxrt_rocm_ep_event_record(NxrtRocmEp* ep, NxrtRocmEvent* event);
NxrtStatus nxrt_rocm_ep_event_elapsed_ms(NxrtRocmEp* ep, NxrtRocmEvent* start, NxrtRocmEvent* stop, float* out_ms);
void nxrt_rocm_ep_event_destroy(NxrtRocmEp* ep, NxrtRocmEvent* event);

/* ---- graph capture (Kernel::capture_support in kernel.rs; the CUDA sibling's capture-safe decode path,
 * ep-cuda matmul_nbits.rs:11136-11162) ---------------------------------------------------------
 * Between begin and end, execute calls on this provider are recorded instead of run. Only calls that
 * allocate nothing may be recorded: accuracy_level 0 always, accuracy_level 4 with a caller workspace.
 * A recorded graph does on the same device pointers what the calls would have done, bit for bit, though not launch for launch: calls
 * made in a row that read the same activations and do not depend on each other may share a launch (*out_num_nodes is smaller
 * then), and a launch may read weights of the recorded call behind it into the caches ahead of time. */
typedef struct NxrtRocmGraph NxrtRocmGraph;
NxrtStatus nxrt_rocm_ep_capture_begin(NxrtRocmEp* ep);
NxrtStatus nxrt_rocm_ep_capture_end(NxrtRocmEp* ep, NxrtRocmGraph** out_graph, uint64_t* out_num_nodes);
NxrtStatus nxrt_rocm_ep_graph_replay(NxrtRocmEp* ep, NxrtRocmGraph* graph);
void nxrt_rocm_ep_graph_release(NxrtRocmEp* ep, NxrtRocmGraph* graph);

/* Counters a harness reads to prove the provider, not a fallback, did the work
 * (the role of nxrt_ep_compiled_node_count in ep-cuda-plugin/src/lib.rs:345-372). */
/* Counts the steps of calls that were run or recorded: one for a product, with all that it takes (quantized rows, expanded weights,
 * blocks of rows, slices of K), one for each normalization, gather of act-order rows and SwiGLU epilogue beside it, and one for a call of a node. A recorded
 * call counts the same whether it is a launch of its own or shares one; replays do not count. */
uint64_t nxrt_rocm_ep_kernel_launch_count(const NxrtRocmEp* ep);
uint64_t nxrt_rocm_live_provider_count(void);
/* Device allocations (hipMalloc calls) the library has made in this process so far. */
uint64_t nxrt_rocm_device_allocation_count(void);

#ifdef __cplusplus
}
#endif
#endif /* NXRT_EP_ROCM_H */
