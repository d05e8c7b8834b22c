/*
 * paraconv2d.h -- C ABI of the B200 (sm_100a) ParaConv2d paraboloid convolution.
 *
 * libpc2d_sm100.so exports these entry points.  The signatures use only plain
 * C types: device pointers, sizes, a CUDA stream passed as void*.  They do not
 * use torch types.  The torch op library libptparaconv2d.so (schema
 * ptparaconv2d::forward / ptparaconv2d::backward, identical to the reference)
 * is a thin client of this ABI.
 *
 * Semantics follow the reference op GeoND-tech/ParaConv2d:
 *   input   [n][channels][height][width], already padded by the caller
 *   pars    [h0 (m) | h (m*d) | p (m*d) | p0 (m)], d = channels*k0*k1,
 *           h and p row-major [m][channels][k0][k1]   (paraconv2d.cc:23-37)
 *   output, hsum  [n][m][out_height][out_width]
 *   out_height = (height - dl0*(k0-1) - 1)/s0 + 1     (paraconv2d.cc:268-269)
 *   hsum   = h0[j] + sum_k h[j,k] * win[k]
 *   output = f * (hsum^2 - sum_k (win[k] - p[j,k])^2 - p0[j]^2)
 * The window is flipped: tap (ix2, iy2) reads input row
 * oy*s0 + (k0-1-ix2)*dl0 and column ox*s1 + (k1-1-iy2)*dl1 (paraconv2d.cc:89-92).
 * The backward pass returns inputgrad [n][channels][height][width] (scaled by
 * 2, with no output factor, paraconv2d.cc:166-183) and parsgrad, packed like
 * pars (scaled by 2f, paraconv2d.cc:226-237).  When skip_input_grad is
 * nonzero, inputgrad is written as all zeros (paraconv2d.cc:147,153).
 *
 * Conventions of every compute entry point:
 *   - all tensor pointers are device pointers to contiguous arrays of the
 *     given dtype; inputs are read only; outputs are fully overwritten;
 *   - work is enqueued on `stream` (a cudaStream_t; NULL = legacy default);
 *     nothing synchronises the host, and nothing allocates device memory:
 *     scratch comes from the caller's `workspace` of at least the size
 *     reported by the matching *_workspace_size query (256-byte aligned);
 *   - the return value is a pc2d_status; on failure pc2d_last_error()
 *     gives a message (thread local).  Odd kernel sizes only: even sizes make
 *     the reference read outside the window and are rejected.
 *   - kernels that wait on on-chip barriers give up after a bounded time;
 *     they then record PC2D_ERR_TIMEOUT in a device-side status word that
 *     pc2d_device_status() reads (it synchronises the device), and in a
 *     mirror of it in pinned host memory.  Every later compute call in that
 *     CUDA context reads the mirror on entry (no synchronisation) and returns
 *     PC2D_ERR_TIMEOUT until pc2d_clear_device_status() is called.  The
 *     first compute call in a context allocates the mirror (cudaHostAlloc),
 *     so make it before any stream capture; pc2d_forward_noalloc never does.
 */
#ifndef PARACONV2D_B200_H_
#define PARACONV2D_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PC2D_ABI_VERSION 1

typedef enum {
  PC2D_OK = 0,
  PC2D_ERR_INVALID_ARGUMENT = 1, /* bad shape, dtype, null pointer, pars length ... */
  PC2D_ERR_UNSUPPORTED = 2,      /* valid for the reference but not supported here */
  PC2D_ERR_WORKSPACE = 3,        /* workspace missing, too small or misaligned */
  PC2D_ERR_CUDA = 4,             /* a CUDA runtime call or launch failed */
  PC2D_ERR_TIMEOUT = 5           /* a device-side barrier wait gave up */
} pc2d_status;

/* F16 and BF16 are element types of the sequence operators (dropout, causal
 * convolution, state space scan) only. */
typedef enum { PC2D_DTYPE_F32 = 0, PC2D_DTYPE_F64 = 1, PC2D_DTYPE_F16 = 2, PC2D_DTYPE_BF16 = 3 } pc2d_dtype;

/* Kernel families.  AUTO picks the tcgen05 tensor-core kernels (3xTF32 split
 * precision) for fp32 shapes they support and the CUDA-core kernels
 * otherwise; SIMT forces the CUDA-core kernels (fp32 or fp64 FMA). */
typedef enum { PC2D_ALGO_AUTO = 0, PC2D_ALGO_SIMT = 1, PC2D_ALGO_TC = 2 } pc2d_algo;

/* Library ABI version (PC2D_ABI_VERSION). */
int pc2d_abi_version(void);

/* Output extent along one axis (reference paraconv2d.cc:268-269); <= 0 means empty/invalid. */
int pc2d_out_size(int in, int kernel, int stride, int dilation);

/* Number of output channels implied by the flat parameter count
 * (reference paraconv2d.cc:266: m = npars / (2*(d+1))); -1 when npars is not
 * a positive multiple of 2*(d+1). */
int64_t pc2d_infer_m(int64_t npars, int channels, int k0, int k1);

/* Process-wide kernel family selection (default PC2D_ALGO_AUTO).  Returns the previous value. */
int pc2d_set_algo(int algo);
int pc2d_get_algo(void);

/* Scratch bytes pc2d_forward needs for this problem (0 is possible). */
size_t pc2d_forward_workspace_size(int dtype, int n, int channels, int height, int width, int m,
                                   int k0, int k1, int s0, int s1, int dl0, int dl1);

/* Forward pass.  Replaces the reference's paraconv2d_forward_cuda_main<T>
 * (paraconv2d.cu:81-123) and the kernels it launches
 * (paraconv2dkernels.cu:27-141); `factor` is the op's `doublefactor`
 * argument (paraconv2d.cc:292). */
int pc2d_forward(int dtype, const void *input, const void *pars, double factor,
                 int k0, int k1, int s0, int s1, int dl0, int dl1,
                 int n, int channels, int height, int width, int m,
                 void *output, void *hsum, void *workspace, size_t workspace_bytes, void *stream);

/* Forward pass that allocates nothing and takes no workspace.  It has no
 * counterpart in the reference.  It is meant for callers that may not
 * allocate device memory while the op runs, such as plugin interfaces that
 * pass an operator only its input and output buffers, or real-time code with
 * a fixed memory budget: cudaMalloc can synchronise the device or fail, and
 * those hosts forbid it.  The scratch lives in a static 8 MiB device array
 * that every GPU loading the library keeps until exit.  Problems needing more
 * scratch than that fail with PC2D_ERR_WORKSPACE.  The first call in each
 * CUDA context (with a device's primary context current: the first call on
 * that device) resolves the array's address with cudaGetSymbolAddress, so
 * make that first call before any stream capture.  All calls share the
 * array: calls that overlap on the GPU race and must be serialised by the
 * caller.  Arguments, results and the other errors are those of pc2d_forward. */
int pc2d_forward_noalloc(int dtype, const void *input, const void *pars, double factor,
                         int k0, int k1, int s0, int s1, int dl0, int dl1,
                         int n, int channels, int height, int width, int m,
                         void *output, void *hsum, void *stream);

/* Scratch bytes pc2d_backward needs for this problem. */
size_t pc2d_backward_workspace_size(int dtype, int n, int channels, int height, int width, int m,
                                    int k0, int k1, int s0, int s1, int dl0, int dl1,
                                    int skip_input_grad);

/* Backward pass.  Replaces the reference's paraconv2d_backward_cuda_main<T>
 * (paraconv2d.cu:131-223) and the kernels it launches
 * (paraconv2dgradkernels.cu:27-249). */
int pc2d_backward(int dtype, const void *grad, const void *input, const void *pars, const void *hsum,
                  double factor, int k0, int k1, int s0, int s1, int dl0, int dl1,
                  int n, int channels, int height, int width, int m, int skip_input_grad,
                  void *inputgrad, void *parsgrad, void *workspace, size_t workspace_bytes, void *stream);

/* The two steps of the reference module's forward before the op
 * (ptparaconv2d.py:216-217: `x = input_factor * input`, then a constant-zero
 * F.pad) as one pass: output[n][c][y][x] = scale * input[n][c][y - pad_top]
 * [x - pad_left] inside, 0 in the padding; output is
 * [n][channels][height+pad_top+pad_bottom][width+pad_left+pad_right].  fp32 or
 * fp64; pads must be >= 0 (F.pad's negative pads crop; use torch for those). */
int pc2d_pad_scale(int dtype, const void *input, int n, int channels, int height, int width,
                   int pad_top, int pad_bottom, int pad_left, int pad_right, double scale,
                   void *output, void *stream);

/* Backward pass of the reference module around the op
 * (ptparaconv2d.py:52-58 and the backward of its pad and input factor,
 * :216-217): as pc2d_backward on the padded input, but the input gradient is
 * written only for the unpadded input, rows pad_top .. height-pad_bottom-1
 * and columns pad_left .. width-pad_right-1, into an
 * [n][channels][height-pad_top-pad_bottom][width-pad_left-pad_right] array,
 * multiplied by dx_scale (the module's input_factor * grad_factor).  This
 * replaces the module's slice of the padded gradient and its two scalings
 * (three passes over the input gradient) with the kernels' own stores.  With
 * skip_input_grad nonzero, inputgrad is zero-filled, or left alone when it is
 * NULL (a caller that does not need it).  Workspace: as pc2d_backward. */
int pc2d_backward_interior(int dtype, const void *grad, const void *input, const void *pars, const void *hsum,
                           double factor, int k0, int k1, int s0, int s1, int dl0, int dl1,
                           int n, int channels, int height, int width, int m, int skip_input_grad,
                           int pad_top, int pad_bottom, int pad_left, int pad_right, double dx_scale,
                           void *inputgrad, void *parsgrad, void *workspace, size_t workspace_bytes,
                           void *stream);

/* ---------------------------------------------------------------------------
 * Data-parallel training: the backward pass with the parameter gradient
 * summed over the ranks (one process per GPU, up to 8 GPUs of one node with
 * peer access), over NVLink peer memory instead of a separate all-reduce.
 * The reference has no multi-GPU path; this replaces the all-reduce (SUM) of
 * pars.grad after the backward in a data-parallel loop.
 *
 * Setup, once per process group (allocates: do it before any stream capture):
 *   pc2d_comm_create   -> this rank's exchange buffer (cudaMalloc) and an IPC
 *                         handle of pc2d_comm_handle_bytes() bytes;
 *   (the caller gathers every rank's handle, in rank order, by any channel,
 *    e.g. torch.distributed.all_gather_object)
 *   pc2d_comm_connect  -> maps every peer's buffer;
 *   pc2d_comm_destroy  -> unmaps and frees (after every rank's last call has
 *                         completed: a barrier first).
 * pc2d_backward_sum: as pc2d_backward (fp32), with parsgrad receiving the sum
 * of all ranks' parameter gradients, the same bits on every rank (fixed rank
 * order).  Every rank must make the same sequence of pc2d_backward_sum calls
 * on its communicator (like a collective); the calls of one communicator go
 * on one stream.  A rank that waits longer than 2 s for its peers records
 * PC2D_ERR_TIMEOUT in the device status (see above) and returns its own
 * gradient.
 * pc2d_comm_allreduce: dst = the sum over the ranks of every rank's src
 * (count fp32 values, count <= max_params; dst may be src), the same bits on
 * every rank, through the same exchange buffer: e.g. one bucket of several
 * layers' parameter gradients after an autograd backward.  It shares the
 * call sequence of pc2d_backward_sum (every rank the same calls, in the same
 * order, on one stream) and its timeout behaviour (dst = own src). */
typedef struct pc2d_comm pc2d_comm;
size_t pc2d_comm_handle_bytes(void);
int pc2d_comm_create(int rank, int world, size_t max_params, pc2d_comm **comm, void *handle_out);
int pc2d_comm_connect(pc2d_comm *comm, const void *handles);
int pc2d_comm_destroy(pc2d_comm *comm);
int pc2d_backward_sum(pc2d_comm *comm, int dtype, const void *grad, const void *input, const void *pars,
                      const void *hsum, double factor, int k0, int k1, int s0, int s1, int dl0, int dl1,
                      int n, int channels, int height, int width, int m, int skip_input_grad,
                      void *inputgrad, void *parsgrad, void *workspace, size_t workspace_bytes, void *stream);
int pc2d_comm_allreduce(pc2d_comm *comm, const void *src, void *dst, size_t count, void *stream);

/* ---------------------------------------------------------------------------
 * Optimizer step on one layer's flat parameter vector [h0 | h | p | p0]
 * (m output channels, window of d = C*k0*k1 elements), using the multipliers
 * the module attaches to `pars` (reference ptparaconv2d.py:194-198):
 *   d_i   = grad_i + (weight_decay * wd_factor) * w_i
 *   buf_i = momentum * buf_i + d_i     (buf_i = d_i when first_step != 0;
 *                                       momentum_buf unused when momentum == 0)
 *   w_i  -= (lr * factor_i) * buf_i,   factor = h_lr_factor on [h0 | h] (the
 *                                       first m*(1+d) values), p_lr_factor on [p | p0]
 * i.e. torch.optim.SGD (no dampening, no Nesterov) with the learning rate and
 * weight decay scaled per parameter group, in one pass over HBM.  dtype F32 or
 * F64; pars, grad and momentum_buf hold 2*m*(1+d) values each. */
int pc2d_param_step(int dtype, void *pars, const void *grad, void *momentum_buf, int m, int d, double lr,
                    double h_lr_factor, double p_lr_factor, double weight_decay, double wd_factor,
                    double momentum, int first_step, void *stream);

/* ---------------------------------------------------------------------------
 * Sequence operators, beside the convolution and over the maps it writes: an
 * [N][C][H][W] map is [batch][channels][length] with length = H*W.  They have
 * no counterpart in the reference.  All arrays are contiguous; activations,
 * states, checkpoints and their gradients are 16-byte aligned, all others
 * aligned to their elements (what is off the boundary that a call needs is
 * refused); no output may overlap an input.  float32, float16 and bfloat16 (dropout float64 too); sums
 * and states are held in 32 bits and rounded once to the outputs' type.  The
 * results do not depend on the order in which blocks run.  With `lengths`
 * (int32 on the device, one per batch row, taken as 0 .. length), the
 * positions of a row behind its length are not read: outputs and gradients
 * there are 0 and the states are those after the row's last token.
 *
 * Dropout.  Element i is kept when its 16 random bits are at least
 * thr = round(65536 p), and multiplied by 65536/(65536 - thr); it is 0
 * otherwise, whatever it held.  output = residual + that (residual may be
 * NULL).  The bits are half i % 8 (low half of word 0 first) of the four words
 * that Philox4x32-10 gives for the counter (i/8, key[1]) under the key key[0]
 * (64-bit values, low words first); `key` is int64[2] on the device, so that
 * a captured call can be replayed with other numbers.  The same call on the
 * output's gradient, without residual, is the backward pass: no mask is kept.
 * pc2d_dropout_next_key copies {state[0], state[1]} to key and adds 1 to
 * state[1] atomically: every call of it, a replayed one too, gives another
 * key. */
int pc2d_dropout(int dtype, const void *input, const void *residual, const int64_t *key, double p, int64_t n,
                 void *output, void *stream);
int pc2d_dropout_next_key(int64_t *state, int64_t *key, void *stream);

/* Causal convolution along the length, one filter of `taps` (1 to 8) per
 * channel.  With line = [initial_state (taps-1 values; NULL: zeros) | the
 * row's tokens]: pre_t = bias[c] + sum_k weight[c][k] line[t+k]; output = pre,
 * or pre * sigmoid(pre) with silu; final_state = the last taps-1 values of
 * line.  weight [channels][taps], bias [channels] (NULL: none): of the
 * inputs' type or float32 (wdtype).  States: [batch][channels][taps-1] of the
 * inputs' type.  final_state, grad_final, weightgrad, biasgrad and
 * initialgrad may be NULL.  pc2d_causal_conv_step takes one token per row
 * and moves its state on in place: `state` [places][channels][taps-1], row b
 * uses place slots[b] (int32; NULL: b).  slots[b] = -1 marks a row without
 * request: its output is 0 and no state changes.  A place outside the array,
 * or one that an earlier row of the call has too, makes the row's output NaN
 * and changes no state. */
int pc2d_causal_conv_forward(int dtype, int wdtype, const void *input, const void *weight, const void *bias,
                             const void *initial_state, const int *lengths, int batch, int channels, int length,
                             int taps, int silu, void *output, void *final_state, void *stream);
size_t pc2d_causal_conv_backward_workspace_size(int batch, int channels, int length, int taps);
int pc2d_causal_conv_backward(int dtype, int wdtype, const void *grad, const void *grad_final, const void *input,
                              const void *weight, const void *bias, const void *initial_state, const int *lengths,
                              int batch, int channels, int length, int taps, int silu, void *inputgrad,
                              void *weightgrad, void *biasgrad, void *initialgrad, void *workspace,
                              size_t workspace_bytes, void *stream);
int pc2d_causal_conv_step(int dtype, int wdtype, const void *input, void *state, const void *weight, const void *bias,
                          const int *slots, int batch, int places, int channels, int taps, int silu, void *output,
                          void *stream);

/* State space scan.  Per channel c, with `states` (1 to 128) states n and the
 * inputs B, C [batch][groups][states][length] of the channel's group (equal
 * groups of channels/groups channels):
 *   d_t = delta_t + delta_bias[c]        (softplus of it with delta_softplus)
 *   h_t[n] = exp(d_t A[c][n]) h_{t-1}[n] + d_t u_t B_t[n]
 *   output_t = (sum_n C_t[n] h_t[n] + skip[c] u_t) * (z_t sigmoid(z_t) with z)
 * from h = initial_state (NULL: 0); final_state = h after the last token.  Up to
 * 2^24 rows (batch * channels; of the step too) and 2^30 tokens.
 * u, delta, z and output [batch][channels][length]; A [channels][states],
 * skip and delta_bias [channels] (NULL: 0), states [batch][channels][states]:
 * float32.  `checkpoints` (NULL: none) receives the states that the backward
 * pass starts its tiles from, pc2d_ssm_scan_checkpoint_size() bytes.  The
 * backward pass gives the gradients of all inputs (skipgrad, biasgrad,
 * initialgrad and grad_final may be NULL; zgrad goes with z).  Its workspace is
 * about states^2 / 64 bytes per channel and token (blocks have fewer channels
 * the more states these have, and each has shares of Bgrad and Cgrad of its own).
 * pc2d_ssm_scan_step takes one token per row (u, delta, z [batch][channels],
 * B, C [batch][groups][states]) and moves its state [places][channels][states]
 * on in place; slots as for pc2d_causal_conv_step. */
size_t pc2d_ssm_scan_checkpoint_size(int batch, int channels, int length, int states);
size_t pc2d_ssm_scan_forward_workspace_size(int batch, int channels, int length, int states, int groups);
int pc2d_ssm_scan_forward(int dtype, const void *u, const void *delta, const float *A, const void *B, const void *C,
                          const float *skip, const void *z, const float *delta_bias, const float *initial_state,
                          const int *lengths, int delta_softplus, int batch, int channels, int length, int states,
                          int groups, void *output, float *final_state, float *checkpoints, void *workspace,
                          size_t workspace_bytes, void *stream);
size_t pc2d_ssm_scan_backward_workspace_size(int batch, int channels, int length, int states, int groups);
int pc2d_ssm_scan_backward(int dtype, const void *grad, const float *grad_final, const void *u, const void *delta,
                           const float *A, const void *B, const void *C, const float *skip, const void *z,
                           const float *delta_bias, const int *lengths, const float *checkpoints, int delta_softplus,
                           int batch, int channels, int length, int states, int groups, void *ugrad, void *deltagrad,
                           float *Agrad, void *Bgrad, void *Cgrad, float *skipgrad, void *zgrad, float *biasgrad,
                           float *initialgrad, void *workspace, size_t workspace_bytes, void *stream);
int pc2d_ssm_scan_step(int dtype, const void *u, const void *delta, float *state, const float *A, const void *B,
                       const void *C, const float *skip, const void *z, const float *delta_bias, const int *slots,
                       int delta_softplus, int batch, int places, int channels, int states, int groups, void *output,
                       void *stream);

/* ---------------------------------------------------------------------------
 * Group norm over [batch][channels][length] maps, or with channels_last over
 * [batch][length][channels], with an optional SiLU:
 *   xhat = (x - mean) / sqrt(variance + eps), over the channels/groups channels
 *   of a group and all tokens of a batch row (population variance);
 *   pre = xhat weight[c] + bias[c];  output = pre, or pre sigmoid(pre) with silu.
 * float32, float16 and bfloat16; weight and bias [channels] (NULL: 1 and 0) of
 * the input's type or float32 (wdtype).  lengths as for the sequence operators
 * (NULL: all tokens).  stats [batch][groups][2] (NULL: not kept) receives the
 * mean and 1/sqrt(variance + eps), which the backward pass takes; weightgrad
 * and biasgrad may be NULL.  Arrays need their elements' alignment (16 bytes
 * are faster); no output may overlap an input.  Up to 8192 channels a group,
 * 2^24 batch * groups and 2^30 positions. */
size_t pc2d_group_norm_workspace_size(int dtype, int channels_last, int batch, int channels, int length, int groups,
                                      int backward);
int pc2d_group_norm_forward(int dtype, int wdtype, int channels_last, const void *input, const void *weight,
                            const void *bias, const int *lengths, int batch, int channels, int length, int groups,
                            double eps, int silu, void *output, float *stats, void *workspace, size_t workspace_bytes,
                            void *stream);
int pc2d_group_norm_backward(int dtype, int wdtype, int channels_last, const void *grad, const void *input,
                             const void *weight, const void *bias, const int *lengths, const float *stats, int batch,
                             int channels, int length, int groups, int silu, void *inputgrad, void *weightgrad,
                             void *biasgrad, void *workspace, size_t workspace_bytes, void *stream);

/* ---------------------------------------------------------------------------
 * Linear attention with a decay for each head.  Per batch row and head:
 *   S_t = exp(g_t) S_(t-1) + k_t v_t^T  (dk x dv);  output_t = scale S_t^T q_t
 * q, k [batch][groups][dk][length], each group for heads/groups neighbouring
 * heads; v and output [batch][heads][dv][length]; log_decay g (float32, at
 * most 0 in use; -inf forgets) [heads], or with decay_per_token
 * [batch][heads][length].  States [batch][heads][dk][dv] are float32;
 * initial_state (NULL: 0), lengths and final_state (NULL: not wanted) as for
 * the sequence operators.  1 to 128 for dk and dv, up to 2^30 tokens and 2^20
 * rows times heads.  `states` (NULL: none), ..._states_size() bytes, receives
 * what the backward pass starts its chunks from: 4 dk dv bytes for every 64
 * tokens of a head (every 32 in float32 and float16).  The backward pass gives all gradients
 * (grad_final and initialgrad may be NULL), decaygrad in the decays' shape.
 * Arrays need their elements' alignment (16 bytes and lengths that are
 * multiples of 8 are faster), `states` 16 bytes.  pc2d_linear_attention_step takes one token per
 * row (q, k [batch][groups][dk], v [batch][heads][dv], log_decay [heads] or
 * with decay_per_row [batch][heads]) and moves its state [places][heads][dk]
 * [dv] (16-byte aligned) on in place; slots as for pc2d_causal_conv_step. */
size_t pc2d_linear_attention_states_size(int dtype, int batch, int heads, int length, int dk, int dv);
size_t pc2d_linear_attention_workspace_size(int dtype, int batch, int heads, int groups, int length, int dk, int dv,
                                            int backward);
int pc2d_linear_attention_forward(int dtype, const void *q, const void *k, const void *v, const float *log_decay,
                                  int decay_per_token, const float *initial_state, const int *lengths, int batch,
                                  int heads, int groups, int length, int dk, int dv, double scale, void *output,
                                  float *final_state, float *states, void *workspace, size_t workspace_bytes,
                                  void *stream);
int pc2d_linear_attention_backward(int dtype, const void *grad, const float *grad_final, const void *q, const void *k,
                                   const void *v, const float *log_decay, int decay_per_token, const float *states,
                                   const int *lengths, int batch, int heads, int groups, int length, int dk, int dv,
                                   double scale, void *qgrad, void *kgrad, void *vgrad, float *decaygrad,
                                   float *initialgrad, void *workspace, size_t workspace_bytes, void *stream);
int pc2d_linear_attention_step(int dtype, const void *q, const void *k, const void *v, const float *log_decay,
                               int decay_per_row, float *state, const int *slots, int batch, int places, int heads,
                               int groups, int dk, int dv, double scale, void *output, void *stream);

/* ---------------------------------------------------------------------------
 * AdamW over many tensors of one or several types, with the moments in 32 or
 * in 8 bits (state_bits).  At step t = ++*step (int64 on the device), for each
 * element w of tensor i with gradient g = grad * *grad_scale (NULL: 1):
 *   m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
 *   w = (1 - lr rate weight_decay decay) w - lr rate m / (1 - beta1^t) / (sqrt(v / (1 - beta2^t)) + eps)
 * in 32 bits; rate is rate_first for the first `split` elements and rate_rest
 * behind them.  *lr_device (NULL: lr) lets a captured call follow a schedule.
 * dtype F32, F16 or BF16; gradients of the same type or F32.  With `master`
 * (16-bit parameters only) w is held there in float32, and the parameter is
 * its rounding.  Written arrays may not overlap any other.
 * 32 bits: exp_avg (m) and exp_avg_sq (v) are float32 [n].  8 bits: they are
 * codes [n], and scales [ceil(n/256)][2] holds the exponent byte E of each
 * moment for every 256 elements; zeros are zero moments.  A code's size c (m:
 * the low 7 bits, the sign above them) stands for c/8 s below 8 and for
 * 2^((c >> 3) - 1) (1 + (c & 7)/8) s from there on, s = 2^(E - 127); E = 255
 * (a value of the block was not finite): NaN.  E brings the block's largest
 * value, rounded up to a code, into the topmost binade, and values are rounded up with the
 * probability of what is cut off: size/step + (r + 1/2)/256, rounded down,
 * where r is byte j of the first (m) or of the last (v) two words that
 * Philox4x32-10 gives for the counter (element/8, i, t low, t high) under the
 * key `seed`, j = element % 8 (pc2d_adamw_step_numbered takes numbers[i], from 0
 * to 2^31 - 1, in the place of i: a tensor's random numbers then do not depend on its
 * place in the list; numbers is read before the call returns); a v that is not zero gets code 1 at least.  Per call: two launches, and more beyond 320 tensors
 * or for more types.  workspace: pc2d_adamw_workspace_size() bytes.
 * pc2d_adamw_state_values writes the values of 8-bit moments (exp_avg,
 * exp_avg_sq, scales and n of each tensor) as F32 or BF16, both exact. */
typedef struct {
  int dtype, grad_dtype;
  void *param;
  const void *grad;
  void *exp_avg, *exp_avg_sq;
  float *master;         /* NULL: none */
  unsigned char *scales; /* 8 bits only */
  int64_t n, split;
  double rate_first, rate_rest, decay;
} pc2d_adamw_tensor;
size_t pc2d_adamw_workspace_size(void);
int pc2d_adamw_step(int state_bits, const pc2d_adamw_tensor *tensors, int count, int64_t *step, const float *lr_device,
                    double lr, double beta1, double beta2, double eps, double weight_decay, const float *grad_scale,
                    int64_t seed, void *workspace, size_t workspace_bytes, void *stream);
int pc2d_adamw_step_numbered(int state_bits, const pc2d_adamw_tensor *tensors, int count, const int64_t *numbers,
                             int64_t *step, const float *lr_device, double lr, double beta1, double beta2, double eps,
                             double weight_decay, const float *grad_scale, int64_t seed, void *workspace,
                             size_t workspace_bytes, void *stream);
int pc2d_adamw_state_values(int dtype, const pc2d_adamw_tensor *tensors, int count, void *const *exp_avgs,
                            void *const *exp_avg_sqs, void *stream);

/* Human-readable name of a pc2d_status. */
const char *pc2d_status_string(int status);

/* Message of the last failing call on this host thread ("" if none). */
const char *pc2d_last_error(void);

/* Synchronises the current device and returns PC2D_OK, or the first
 * device-side error (PC2D_ERR_TIMEOUT) recorded since the last call to
 * pc2d_clear_device_status(); also reports pending CUDA errors as PC2D_ERR_CUDA. */
int pc2d_device_status(void);
int pc2d_clear_device_status(void);

/* Kernel timing (profiling aid, off by default).  While enabled, every main
 * kernel the library launches is bracketed by two CUDA events recorded on its
 * stream; pc2d_timing_read synchronises those events and returns, for the
 * kernel family `kernel` ("forward", "dgrad", "wgrad", "simt_forward",
 * "simt_dgrad", "simt_wgrad"), the summed duration in milliseconds and the
 * launch count since the last reset.  Returns PC2D_OK, or
 * PC2D_ERR_INVALID_ARGUMENT for an unknown name. */
int pc2d_timing_enable(int on);
int pc2d_timing_reset(void);
int pc2d_timing_read(const char *kernel, double *total_ms, int *launches);

/* Test hook: a kernel that waits on an mbarrier that nothing completes, with
 * a wait limit of `timeout_us` microseconds; it must return by itself and
 * record PC2D_ERR_TIMEOUT.  Used to check the bounded-wait path without
 * faulting or hanging the GPU. */
int pc2d_selftest_bounded_wait(unsigned int timeout_us, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* PARACONV2D_B200_H_ */
