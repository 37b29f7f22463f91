/*
 * nnc_hip.h - lifecycle, memory and measurement entry points of
 * libnnc_hip.so, the gfx950 (MI355X) implementation of the nnc operator ABI
 * declared in nnc_ops.h.
 *
 * The reference has no device: generated tensors.c points every Tensor into a
 * static host pool (codegen/x86_emitters/tensors.py:589-600, 826-868) and
 * constants_loader.c fread()s weights into static arrays
 * (x86_emitters/constants_loader.py:196-291). The HIP target keeps the memory
 * plan (cost_aware offsets) but places it in ONE hipMalloc'd HBM arena:
 *
 *     nnc_hip_init(0);
 *     nnc_hip_arena_reserve(NNC_MEMORY_SIZE);   // one allocation
 *     nnc_hip_bind(&tensor_x, OFFSET_x);        // per tensor, at load time
 *     nnc_hip_upload(&tensor_w, host_bytes);    // constants, inputs
 *     nnc_run();                                // enqueues nnc_* kernels
 *     nnc_hip_download(&tensor_output, host);   // waits, copies back
 *
 * Threads: the O0-O2 generated code is serial (c_emitter.py:832-847); the
 * reference's O3 runtime calls ops from four pthreads
 * (codegen/x86_emitters/model_source.py:609-674). Every nnc_* entry point is
 * reentrant: each calling host thread gets its own pair of library streams
 * with its own stream-K scratch on its first call (released for reuse when
 * the thread exits), and its calls run in order on its own streams. Work is
 * not ordered across threads: a thread that hands a tensor to another calls
 * nnc_hip_sync() first. The arena, the spill pool, nnc_hip_init and
 * nnc_hip_shutdown are process-wide: reserve and shut down while no other
 * thread is calling. Return codes: 0 = success, otherwise an NNC_HIP_E*
 * value, also kept (process-wide) for nnc_hip_last_error().
 */
#ifndef NNC_HIP_H
#define NNC_HIP_H

#include <stddef.h>
#include <stdint.h>
#include "nnc_types.h"

#ifdef __cplusplus
extern "C" {
#endif

enum {
    NNC_HIP_OK = 0,
    NNC_HIP_EINVAL = 1,   /* bad argument (NULL tensor, bad rank, shape) */
    NNC_HIP_ENOMEM = 2,   /* device allocation failed / arena too small  */
    NNC_HIP_EDEVICE = 3,  /* a HIP runtime call failed                   */
    NNC_HIP_EUNSUPP = 4,  /* argument combination not implemented        */
    NNC_HIP_ESTATE = 5    /* called before nnc_hip_init                  */
};

/* Select the device and create the calling thread's library streams
 * (default priority) and workspace. Idempotent for the same device; another
 * thread's first call (this or any nnc_* call) sets up that thread. */
int nnc_hip_init(int device);
/* Wait for the device, free the arena, every thread's streams and scratch. */
void nnc_hip_shutdown(void);

/* ---- the HBM arena ----------------------------------------------------- */
/* Reserve the arena with one hipMalloc (256-byte aligned base). Calling it
 * again with a larger size replaces the arena (previous bindings dangle). */
int nnc_hip_arena_reserve(size_t bytes);
void* nnc_hip_arena_base(void);
size_t nnc_hip_arena_size(void);
/* t->data = arena + offset; fails if [offset, offset + t->nbytes) is outside
 * the arena or offset is not 16-byte aligned. */
int nnc_hip_bind(Tensor* t, size_t offset);

/* ---- the spill pool (a fast-memory budget below the plan's peak) ------- */
/* Replaces the reference's `_nnc_slow_pool` and the memcpy calls of its
 * spill/reload code (codegen/x86_emitters/model_source.py:259-290,
 * 1535-1659): the HBM arena is the fast pool, pinned host memory the slow
 * one. nnc_hip_spill_reserve allocates it with one hipHostMalloc (again with
 * a larger size: replaced, previous bindings dangle; refused during graph
 * capture); nnc_hip_bind_spill sets t->data = pool + offset like
 * nnc_hip_bind. */
int nnc_hip_spill_reserve(size_t bytes);
void* nnc_hip_spill_base(void);
int nnc_hip_bind_spill(Tensor* t, size_t offset);
/* Copy src's t->nbytes bytes to dst (same nbytes) asynchronously on the
 * selected library stream: a spill (arena -> pool) or a reload (pool ->
 * arena); under graph capture a memcpy node. Errors as for nnc_* calls. */
void nnc_hip_transfer(Tensor* src, Tensor* dst);

/* ---- explicit allocations (tests and callers without an arena) --------- */
void* nnc_hip_malloc(size_t bytes);
void nnc_hip_free(void* ptr);
/* pinned host memory (hipHostMalloc): a spill pool of one's own */
void* nnc_hip_host_malloc(size_t bytes);
void nnc_hip_host_free(void* ptr);

/* ---- host <-> device (synchronous with respect to the calling thread's
 * library streams) ---------------------------------------------------------- */
int nnc_hip_upload(Tensor* t, const void* host_src);    /* t->nbytes bytes */
int nnc_hip_download(const Tensor* t, void* host_dst);  /* t->nbytes bytes */
int nnc_hip_memcpy_h2d(void* dst, const void* src, size_t bytes);
int nnc_hip_memcpy_d2h(void* dst, const void* src, size_t bytes);

/* ---- synchronisation and errors ---------------------------------------- */
int nnc_hip_sync(void);             /* waits for the calling thread's streams */
void* nnc_hip_stream(void);         /* the calling thread's stream 0, for callers
                                       that order their own work after ours */
int nnc_hip_last_error(void);       /* last non-zero code since reset */
const char* nnc_hip_last_error_message(void);
void nnc_hip_clear_error(void);

/* ---- a second stream for independent branches ---------------------------
 * Per calling thread: its calls go to its stream 0 unless it selects its
 * stream 1. The compiler's O3
 * schedule (mi355x target) runs a branch that only depends on the fork
 * point - a residual block's 1x1 downsample convolution - on stream 1 while
 * the main branch continues on stream 0:
 *   nnc_hip_stream_fork();       stream 1 waits for stream 0's work so far
 *   nnc_hip_stream_select(1); ...branch calls...; nnc_hip_stream_select(0);
 *   ...main calls...
 *   nnc_hip_stream_join();       stream 0 waits for stream 1's work so far
 * Both streams have default priority and their own scratch (stream-K
 * partials, counters), so concurrent calls never share it; nnc_hip_sync and
 * the host copies wait for both. A graph capture starts and ends on stream
 * 0 and records forked branches as parallel graph branches. No counterpart
 * in the reference, whose O3 executor runs its resource queues on host
 * threads (codegen/x86_emitters/model_source.py:502-735). */
int nnc_hip_stream_fork(void);
int nnc_hip_stream_select(int slot);
int nnc_hip_stream_join(void);

/* ---- per-kernel timing --------------------------------------------------
 * While enabled, every kernel launch is bracketed by hipEvents recorded on
 * the stream it runs on; durations accumulate per kernel name in one
 * process-wide table. Reading the table waits for the recorded events. Used
 * by bench.py for the roofline figures. */
void nnc_hip_profile_enable(int on);
void nnc_hip_profile_reset(void);
int nnc_hip_profile_count(void);
/* Entry i: copies the kernel name (NUL-terminated, truncated to cap), the
 * number of launches and the summed milliseconds. Returns 0 on success. */
int nnc_hip_profile_entry(int i, char* name, int cap, int64_t* launches,
                          double* total_ms);
/* Entry i: algorithmic work summed over its launches - flops for the matrix
 * kernels, bytes every launch must move through HBM at least once for the
 * bandwidth-bound kernels (0 where not applicable). */
int nnc_hip_profile_work(int i, double* flops, double* bytes);

/* ---- launch capture ------------------------------------------------------
 * Record every kernel the calling thread's following nnc_* calls enqueue
 * into a hipGraph (one per thread) and replay it with one launch on that
 * thread's stream 0. Between begin and end nothing of it executes. The graph
 * keeps the device pointers of the captured calls. */
int nnc_hip_graph_begin(void);
int nnc_hip_graph_end(void);
int nnc_hip_graph_launch(void);
void nnc_hip_graph_destroy(void);

/* ---- per-tensor debug dump ------------------------------------------------
 * Replaces the dump code the reference emits into nnc_run() in debug mode
 * (src/nnc_py/codegen/x86_emitters/model_source.py:136-184, 297-428): waits
 * for the library stream, copies the tensor to the host and writes it in the
 * reference's text format,
 *   DEBUG_TENSOR_START <name> <node_idx>
 *   SHAPE <ndim>
 *   DIM <i> <extent>                      (one line per dimension)
 *   DATA_START
 *   <value printed with %f>               (one line per element)
 *   DATA_END
 *   DEBUG_TENSOR_END <name>               (then an empty line)
 * to `file` (a FILE*; NULL: stdout), so the reference's parser
 * (src/nnc_py/tools/debug_compare.py:17-106) reads it unchanged. Float32
 * elements print as themselves, bool/uint8/int8 and int32/int64 as their
 * value converted to float. Not while a graph is being captured
 * (NNC_HIP_ESTATE). */
int nnc_hip_debug_dump(const Tensor* t, const char* name, int node_idx, void* file);

/* ---- fused operators of the mi355x target --------------------------------
 * No counterpart in the reference ABI (runtime/include/nnc_ops.h); emitted by
 * the mi355x compiler target at O3.
 *
 * nnc_hip_conv_add_relu: a residual block's Conv -> Add -> Relu in one
 * kernel: out = relu(conv(in, w) + bias + res), equal to nnc_conv followed by
 * nnc_add_relu(conv_out, res, out) (same rounding sequence). `res` has the
 * output's shape and may be the same buffer as `out`; `b` may be NULL. */
void nnc_hip_conv_add_relu(Tensor* in, Tensor* w, Tensor* b, Tensor* res, Tensor* out, int kh, int kw,
                           int sh, int sw, int ph, int pw);

/* nnc_hip_conv_packed: convolution with the weights packed tap-major,
 * [Co][kh][kw][Ci] (the compiler transposes the constant), which lets the
 * kernel stream weights and input straight into LDS. out = act(conv(in, w) +
 * bias (+ res)); act 0 none, 1 relu, 2 sigmoid. `b` and `res` may be NULL;
 * `res` has the output's shape and may be the same buffer as `out`. Needs
 * Ci % 32 == 0, a 1x1 or 3x3 kernel and 16-byte aligned weights
 * (NNC_HIP_EUNSUPP otherwise). */
void nnc_hip_conv_packed(Tensor* in, Tensor* w, Tensor* b, Tensor* res, Tensor* out, int kh, int kw, int sh,
                         int sw, int ph, int pw, int act);

/* nnc_hip_conv_proj: a residual block's last convolution with its 1x1
 * projection shortcut folded into the same contraction:
 *   out = act(conv(in, W3) + conv1x1(x, Wp, stride psh x psw) + b)
 * with w packed [Co][kh*kw*Ci + Cx]: each row is W3 tap-major
 * ([kh][kw][Ci]) followed by the Cx projection weights, and b the sum of the
 * two biases. Equal to nnc_conv + nnc_conv1x1 + nnc_add_relu (act 1) up to
 * fp32 accumulation order. Needs a 3x3 kernel, Ci and Cx multiples of 32,
 * every (oh * psh, ow * psw) inside x, 16-byte aligned weights
 * (NNC_HIP_EUNSUPP / NNC_HIP_EINVAL otherwise). */
void nnc_hip_conv_proj(Tensor* in, Tensor* w, Tensor* b, Tensor* x, Tensor* out, int kh, int kw, int sh, int sw,
                       int ph, int pw, int psh, int psw, int act);

/* nnc_hip_conv_maxpool: ResNet's stem - convolution on packed [Co][Kp]
 * rows (3 channels, 7x7), bias, relu - streamed into the 3x3 / stride 2 /
 * pad 1 max pool that follows it:
 *   out = maxpool(relu(conv(in, w) + b)), out [N][Co][Ho/2][Wo/2]
 * with Ho, Wo the convolution's output size from in, the kernel, stride and
 * pads. The convolution output never reaches HBM: each workgroup pools the
 * rows it computes. Same convolution (within the conv bar of the reference's
 * double sums) and the same max (bit for bit on that convolution) as
 * nnc_hip_conv_packed + nnc_maxpool2d. Needs Co <= 64, Ho and Wo even,
 * Wo <= 128 (NNC_HIP_EUNSUPP otherwise). Emitted by the mi355x target's O3
 * tile-streaming pass. No counterpart in the reference ABI. */
void nnc_hip_conv_maxpool(Tensor* in, Tensor* w, Tensor* b, Tensor* out, int kh, int kw, int sh, int sw, int ph,
                          int pw);

/* nnc_hip_gap_gemm_nt: GlobalAveragePool -> Flatten -> Gemm(transB = 1) in
 * one kernel, the pooled [N, C] tensor never leaving the workgroup:
 *   out[n][o] = alpha * sum_c mean_hw(in[n][c]) * w[o][c] + beta * c
 * with in [N][C][H][W], w [O][C], c [O] or [N][O] or NULL, out [N][O]. The
 * means are nnc_avgpool2d's over the whole plane, bit for bit; the dot
 * products are nnc_gemm_nt's exact float products summed in double in
 * another fixed order (per-lane sums and a shuffle tree instead of one
 * chain: the float result differs only where the double sums straddle a
 * float rounding boundary). Needs C % 4 == 0, C <= 1024, C * (H*W + 2)
 * floats <= 128 KB, at most 65535 images and 16-byte aligned in and w
 * (NNC_HIP_EUNSUPP otherwise). Emitted by the mi355x target's O3 tile-streaming pass. No
 * counterpart in the reference ABI. */
void nnc_hip_gap_gemm_nt(Tensor* in, Tensor* w, Tensor* c, Tensor* out, float alpha, float beta);

/* nnc_hip_fused_eltwise: a chain of element-wise ops evaluated in registers
 * in one pass over HBM, no intermediate tensor written. ins: n_in (1..4)
 * tensors of numel(out) elements each (no broadcast). prog: n_steps (1..8)
 * steps of three ints {op, x, y} computing acc = op(x, y), an operand being
 * -1 (acc, the previous step's value; not in step 0) or an input index; y is
 * ignored by the unary ops. consts: two floats per step, Clip's lo and hi
 * (may be NULL without Clip steps). out = acc after the last step; out may be
 * one of the inputs. Ops (NNC_EW_*): ADD 0, SUB 1, MUL 2, DIV 3, ADD_RELU 4
 * (s > 0 ? s : 0, as nnc_add_relu), ADD_SIGMOID 5, RELU 6 (as nnc_relu),
 * SIGMOID 7, TANH 8, CLIP 9. Every step is the corresponding nnc_* op's
 * arithmetic, so the result equals the ops run one call after another
 * through temporaries (bit for bit on this library). NNC_HIP_EINVAL for a
 * malformed program or a short input. Emitted by the mi355x target's O3
 * pass for element-wise nodes each feeding only the next. No counterpart in
 * the reference ABI (which runs each op as its own call, runtime/x86/
 * ops.c:82-258, 2253-2262, 3233-3346). */
enum { NNC_EW_ADD = 0, NNC_EW_SUB, NNC_EW_MUL, NNC_EW_DIV, NNC_EW_ADD_RELU, NNC_EW_ADD_SIGMOID, NNC_EW_RELU,
       NNC_EW_SIGMOID, NNC_EW_TANH, NNC_EW_CLIP, NNC_EW_OPS };
void nnc_hip_fused_eltwise(Tensor** ins, int n_in, const int* prog, int n_steps, const float* consts, Tensor* out);

/* nnc_hip_ew_chain_specialized: 1 if nnc_hip_fused_eltwise runs this chain
 * (n_in inputs, prog of n_steps steps as that call takes them) on a kernel
 * compiled for it - its steps as compile-time code, for the chains the
 * mi355x O3 compiler emits and a few common short ones - and 0 if it runs on
 * the general kernel that reads the steps at run time (same results). A
 * table lookup on the host: no GPU, no device call. No counterpart in the
 * reference ABI. */
int nnc_hip_ew_chain_specialized(int n_in, const int* prog, int n_steps);

/* nnc_hip_add_layernorm: out = layernorm(a + b) over dims [axis:] with
 * scale and bias indexed by the axis dimension - a transformer's residual
 * add and the normalisation after it in one pass, the sum never written.
 * a and b have the same element count (no broadcast). The same bits as
 * nnc_add(a, b, t) then nnc_layernorm(t, scale, bias, out, axis, eps) on this
 * library (the sum is that of nnc_add, the normalisation that of
 * nnc_layernorm). Emitted by the mi355x target's O3 pass for an Add whose
 * only reader is a LayerNormalization. No counterpart in the reference ABI
 * (runtime/x86/ops.c:82-119 then 2095-2171). */
void nnc_hip_add_layernorm(Tensor* a, Tensor* b, Tensor* scale, Tensor* bias, Tensor* out, int axis, float eps);

/* nnc_hip_scaled_softmax: out = softmax(in / div[0]) over axis - attention's
 * score scaling and the softmax after it in one pass, the quotient never
 * written. div has one element; out is the size of in. The same bits as
 * nnc_div(in, div, t) then nnc_softmax(t, out, axis) on this library.
 * Emitted by the mi355x target's O3 pass for a Div by a one-element tensor
 * whose only reader is a Softmax. No counterpart in the reference ABI
 * (runtime/x86/ops.c:82-224 then 260-310). */
void nnc_hip_scaled_softmax(Tensor* in, Tensor* div, Tensor* out, int axis);

/* nnc_hip_transpose_slice: out = transpose(view, perm), where view is the
 * block of columns [col0, col0 + width) of in (in read as rows of its last
 * extent W), taken row-major and shaped as out and perm imply (view.shape
 * [perm[d]] = out.shape[d]) - a Split piece along the last axis, reshaped
 * and transposed, read straight from the unsplit tensor. 4-byte elements.
 * The same bits as nnc_split, then nnc_transpose of the reshaped piece.
 * Emitted by the mi355x target's O3 pass for attention's head split. No
 * counterpart in the reference ABI (runtime/x86/ops.c:2183-2251 nnc_split,
 * then 1531-1581 nnc_transpose). */
void nnc_hip_transpose_slice(Tensor* in, Tensor* out, int64_t* perm, int ndim, int col0, int width);

/* nnc_hip_attention: a transformer layer's attention block in one kernel.
 * qkv holds batch * seq rows of ld = qkv.shape[-1] floats (the fused QKV
 * projection's output); head h of Q is columns q_col + h * head_dim ..
 * + head_dim of a batch's seq rows, K and V likewise from k_col and v_col.
 * For every batch b and head h: out[b * seq + i][h * head_dim + d] =
 * sum_j P[i][j] V[j][d], P = softmax over j of (Q K^T)[i][j] / div[0] - the
 * context in the merged-head layout the output projection reads, out of
 * batch * seq rows of heads * head_dim floats. Float32; div one element;
 * head_dim 32 or 64; seq a multiple of 32 up to 128; qkv rows, ld and the
 * three column offsets 16-byte aligned (NNC_HIP_EUNSUPP otherwise). fp32
 * MFMA products and the hardware exponential: within 1e-4 abs / 1e-3 rel of
 * the calls it replaces. Emitted by the mi355x target's O3 pass for the
 * head split (nnc_hip_transpose_slice of the QKV projection), Q K^T, the
 * scaled softmax, the product with V and the head merge. No counterpart in
 * the reference ABI (runtime/x86/ops.c:2183-2251 nnc_split, 1531-1581
 * nnc_transpose, 1607-1730 nnc_matmul, 82-224 nnc_div, 260-310 nnc_softmax;
 * tests/__snapshots__/test_snapshots_simple_transformer.ambr:114-216). */
void nnc_hip_attention(Tensor* qkv, Tensor* div, Tensor* out, int batch, int seq, int heads, int head_dim, int q_col,
                       int k_col, int v_col);

/* nnc_hip_conv_packed_noalloc: nnc_hip_conv_packed for callers that cannot
 * allocate device memory (code under graph capture, tight serving loops,
 * harnesses that forbid hipMalloc). No counterpart in the reference ABI.
 * Same arguments, kernels and results (to the bit) as nnc_hip_conv_packed,
 * but it allocates nothing: its stream-K partial tiles and tile counters
 * live in a static device array of 64 MiB + 16384 counters that each GPU
 * holds until the process ends; a shape needing more fails with
 * NNC_HIP_EUNSUPP before any launch. Calls on one GPU share that array, so
 * they are ordered on the device: each call's stream first waits for the
 * previous call's work (an event recorded after every call, whatever thread
 * or stream made it); inside a graph capture the captured calls are ordered
 * by the graph, and a replay is not ordered against calls made outside it.
 * The calling thread must have its library state already (nnc_hip_init on that thread, or any
 * earlier nnc_* call there): NNC_HIP_ESTATE otherwise. */
void nnc_hip_conv_packed_noalloc(Tensor* in, Tensor* w, Tensor* b, Tensor* res, Tensor* out, int kh, int kw,
                                 int sh, int sw, int ph, int pw, int act);

/* ---- 8-bit serving operators ----------------------------------------------
 * What a decoder layer does with 8-bit activations, weights and cache. No
 * counterpart in the reference ABI. Activations are float32 or float16, all
 * tensors of a call that hold activations of one type; 8-bit values are int8
 * whole numbers -127 .. 127 with float32 scales, value = whole number * scale.
 * Sums, statistics and scales are float32 or wider; attention's weights are
 * rounded before they meet the values, to float16 for float16 outputs and to 22
 * bits for float32 ones, whose queries have 22 bits of the row's largest.
 * Rows, heads, dims and batches are any size (0: nothing happens) where no
 * limit is named.
 *
 * To 8 bits: u = the largest absolute value / 127, rounded once; each whole
 * number is the nearest to x / u, ties to even. Largest value below 2^-100:
 * zeros, scale 0. A NaN or an infinity among the values: scale NaN, whole
 * numbers 0, so all of them read back as NaN.
 *
 * nnc_hip_rms_norm: s = in (+ res), rounded to the activations' type;
 * y = s * w / sqrt(mean(s^2) + eps) over the last extent. `res` may be NULL;
 * `sum`, if not NULL, receives s (it may be the same buffer as `res` or
 * `in`); `out` of in's type may be the same as `in` if `sum` is not. weight:
 * one row. out of in's type: y, scale NULL. out int8: the product s * w,
 * rounded to float32, is quantised row by row and `scale` (one for each row) is
 * its step u times 1 / sqrt(...), so the whole numbers do not depend on the
 * order of the sum of squares. That is float32's; values may be of any finite
 * size.
 *
 * nnc_hip_quantize_rows / nnc_hip_dequantize_rows: rows (of the last extent)
 * to 8 bits with a scale each, and back: activations between an attention or
 * an element-wise op and the next product, weights [N][K] once.
 *
 * nnc_hip_matmul_i8: out[m][n] = (sum_k a[m][k] w[n][k]) * (a_scale[m] *
 * w_scale[n]) + bias[n]: a [M][K] int8 (leading extents count as rows), w
 * [N][K] int8, bias float32 or NULL. The sum is exact; K up to 131071. */
void nnc_hip_rms_norm(Tensor* in, Tensor* res, Tensor* weight, Tensor* sum, Tensor* out, Tensor* scale, float eps);
void nnc_hip_quantize_rows(Tensor* in, Tensor* out, Tensor* scale);
void nnc_hip_dequantize_rows(Tensor* in, Tensor* scale, Tensor* out);
void nnc_hip_matmul_i8(Tensor* a, Tensor* a_scale, Tensor* w, Tensor* w_scale, Tensor* bias, Tensor* out);

/* A paged cache: k_cache int8 [pages][kv_heads][page][dim], v_cache int8
 * [pages][kv_heads][dim][page], k_scale and v_scale float32 [pages][kv_heads];
 * page a multiple of 16 up to 256, dim 32, 64, 128 or 256, kv_heads up to
 * 32767, 16-byte aligned. table int32 [batch][width]: position t of sequence b
 * is in page table[b][t / page]. starts int32 [batch + 1], lengths int32 [batch]:
 * sequence b's rows of the activations are starts[b] .. starts[b + 1] (never
 * decreasing), and they are its last positions, lengths[b] being its length
 * with them. table, starts and lengths are device memory, read when the call
 * runs; starts and lengths outside what there is are clamped, a page number
 * outside [0, pages) is a page that cannot be read or written. Rows of no
 * sequence (padding behind the last) are neither read nor written.
 *
 * nnc_hip_kv_write: row r's keys are k's columns k_col .. k_col + kv_heads *
 * dim, its values v's from v_col (k and v may be one tensor: the rows of a
 * fused projection). A page that keeps positions from before the call gets
 * the larger of its old scale and the new rows'; if that is larger than the
 * old one, the kept whole numbers become the nearest to their value under it.
 * A page that the new rows begin in gets theirs. Positions behind the length
 * stay as they were. Scales are 0, 2^-107 or more (values of 2^-100), or NaN.
 * No page may belong to two sequences that write to it in one call, nor be in
 * its table twice; pages of a common prefix that no row touches may be shared.
 *
 * nnc_hip_kv_read: the opposite: rows starts[b] .. starts[b + 1] of k and v
 * receive sequence b's last positions.
 *
 * nnc_hip_kv_attention: for every row and head, out = softmax over the
 * sequence's positions j of scale * q . k_j, times v_j; row i of n at
 * position p = length - n + i sees j <= p, and with window > 0 j > p -
 * window. q's columns from q_col: heads * dim, heads a multiple of kv_heads,
 * head h reading cached head h / (heads / kv_heads). out [rows][heads * dim],
 * 16-byte aligned. A row that sees nothing (no length, more rows than
 * positions, only pages that cannot be read) gets zeros; what is in the cache
 * at positions that a row does not see does not reach its result. The pages'
 * scales may be any that kv_write makes, in any mix: a key has its weight in
 * the divisor whatever the size of its page's values. max_length: the longest
 * sequence if the caller knows it, 0 otherwise (then the table's width); like
 * the batch it decides how the work is divided, and so the order of the sums,
 * but not which positions are seen. */
void nnc_hip_kv_write(Tensor* k, Tensor* v, Tensor* k_cache, Tensor* v_cache, Tensor* k_scale, Tensor* v_scale,
                      Tensor* table, Tensor* starts, Tensor* lengths, int k_col, int v_col);
void nnc_hip_kv_read(Tensor* k_cache, Tensor* v_cache, Tensor* k_scale, Tensor* v_scale, Tensor* table, Tensor* starts,
                     Tensor* lengths, Tensor* k, Tensor* v, int k_col, int v_col);
void nnc_hip_kv_attention(Tensor* q, Tensor* k_cache, Tensor* v_cache, Tensor* k_scale, Tensor* v_scale, Tensor* table,
                          Tensor* starts, Tensor* lengths, Tensor* out, int q_col, int heads, float scale, int window,
                          int max_length);

/* ---- positions, drafted tokens, answers -------------------------------------
 * The rest of a decoder's serving path, float32 or float16 activations as
 * above. No counterpart in the reference ABI.
 *
 * nnc_hip_rope: norms of query and key heads and their rotation by position, in
 * one pass. in [rows][ld], its columns from col being `heads` heads of `dim`
 * values; out likewise from out_col, of in's type: the same columns of the
 * same buffer, or columns that do not overlap in's (NNC_HIP_EINVAL). For each
 * head y = x * w / sqrt(mean(x^2) + eps) over its dim values if `weight` (in's
 * type, [dim] or [heads][dim]) is not NULL, else y = x. Then, if `angles` is
 * not NULL, its first rot dims are rotated: angles float32 [places][rot] holds
 * rot / 2 cosines and then as many sines for each place, rot even, 2 to dim;
 * positions int32 [rows] names each row's place (device memory, clamped to
 * those that there are). Pair i is dims i and i + rot / 2, or 2 i and 2 i + 1
 * if `interleaved`: (y_a, y_b) becomes (y_a cos - y_b sin, y_b cos + y_a sin).
 * Computed in float64, rounded to float32 and then to in's type. Queries and
 * keys that lie side by side are one call: heads = both, weight a row each.
 *
 * nnc_hip_rope_kv_write: nnc_hip_rope of a call's queries and keys, the keys
 * and the values going into the paged cache as by nnc_hip_kv_write; the
 * results are those of the three calls, bit for bit on rows and weights of the
 * same alignment (the order of a sum of squares goes by it). q's columns from q_col:
 * heads * dim, to q_out ([rows][heads * dim]), or in place if that is NULL; no
 * queries if q is NULL. q, k and v may be one tensor, but rotated queries must
 * not lie over keys or values (NNC_HIP_EINVAL). q_weight [dim] or
 * [heads][dim], k_weight [dim] or [kv_heads][dim], either may be NULL. angles
 * as above, NULL: none; positions NULL: each row's place is its position in
 * its sequence (drafts that share one have to name it). Rows of no sequence
 * are neither read nor written. May use the stream's scratch.
 *
 * nnc_hip_kv_tree_attention: nnc_hip_kv_attention for drafted tokens: the
 * sequence's rows do not see each other in order but by masks. tree int32
 * [rows][words] (device memory): row i sees row m of its sequence if bit m %
 * 32 of word m / 32 of its mask is set (itself by its own bit; rows that the
 * words do not reach are not seen). Every row sees the positions before the
 * sequence's first row; with window > 0 those of them that are later than p -
 * window, p = the first row's position + the row's set bits - 1, which is its
 * position if its mask names the drafts that lead to it and itself. Drafts that
 * a mask names are seen whatever the window; a mask of the last `window` drafts
 * that lead to a row gives it what nnc_hip_kv_attention gives to a run of tokens,
 * and no context where they are that many. Everything else as for
 * nnc_hip_kv_attention; window and rows, too, decide how the work is divided.
 *
 * nnc_hip_token_logprobs: of rows of logits [rows][vocab], p = softmax(scale *
 * logits): logprob float32 [rows] = log p[tokens[row]] (tokens int32 [rows]);
 * entropy float32 [rows] = -sum p log p; top_index int32 and top_logprob
 * float32 [rows][n]: the n likeliest tokens (n from 1 to 64), the earlier of
 * equal ones first, and their log p. Any of the three may be NULL (tokens with
 * logprob). Logits of -infinity have probability 0; a row whose largest is not
 * finite (a NaN or +infinity in it, or nothing but -infinity) has NaN for
 * results and -1 for tokens. A token outside [0, vocab): NaN. Where there are
 * fewer than n tokens: -1, -infinity. Terms are float32's; up to 16 of them are
 * summed in float32, these sums in float64, and the largest is counted: a log
 * probability is off by less than 2^-21 + 2^-22 D before it is rounded to float32,
 * or 2^-18 + 2^-22 D where several workgroups have a row (of up to ten million
 * logits), D being the mean, by p, of scale times the distance to the largest. */
void nnc_hip_rope(Tensor* in, Tensor* weight, Tensor* angles, Tensor* positions, Tensor* out, int col, int out_col,
                  int heads, int dim, int interleaved, float eps);
void nnc_hip_rope_kv_write(Tensor* q, Tensor* k, Tensor* v, Tensor* q_weight, Tensor* k_weight, Tensor* angles,
                           Tensor* positions, Tensor* q_out, Tensor* k_cache, Tensor* v_cache, Tensor* k_scale,
                           Tensor* v_scale, Tensor* table, Tensor* starts, Tensor* lengths, int q_col, int heads,
                           int k_col, int v_col, int interleaved, float eps);
void nnc_hip_kv_tree_attention(Tensor* q, Tensor* k_cache, Tensor* v_cache, Tensor* k_scale, Tensor* v_scale,
                               Tensor* table, Tensor* starts, Tensor* lengths, Tensor* tree, Tensor* out, int q_col,
                               int heads, float scale, int window, int max_length);
void nnc_hip_token_logprobs(Tensor* logits, Tensor* tokens, Tensor* logprob, Tensor* entropy, Tensor* top_index,
                            Tensor* top_logprob, float scale);

#ifdef __cplusplus
}
#endif

#endif /* NNC_HIP_H */
