// Launch wrappers of the token operators (layer norm, rotary positions,
// attention) and of the AdamW step. Pointers are device pointers; every
// wrapper queues its kernels on `st` of the current device and returns the
// launches' cudaError_t. Storage types are gpu::F32 and gpu::BF16.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace illumina {
namespace gpu {

// ---- layer norm (norm.cu) ---------------------------------------------------

cudaError_t layer_norm(int T, const void *x, long long x_stride, long long rows, int c, const float *w, const float *b,
                       float eps, void *y, long long y_stride, float *mean, float *rstd, cudaStream_t st);
// Row blocks whose partial weight gradients layer_norm_backward keeps in its
// workspace ([blocks][2][c] floats).
int layer_norm_blocks(long long rows, int c);
cudaError_t layer_norm_backward(int T, const void *dy, long long dy_stride, const void *x, long long x_stride,
                                long long rows, int c, const float *w, const float *mean, const float *rstd, void *dx,
                                long long dx_stride, float *dw, float *db, float *ws, cudaStream_t st);

// ---- rotary positions (rotary.cu) -------------------------------------------

struct RotaryTensor {
  const void *x = nullptr;
  void *y = nullptr;
  int heads = 0;
  long long xs[3] = {0, 0, 0}, ys[3] = {0, 0, 0};  // batch, token, head
};
struct RotaryParams {
  RotaryTensor t[2];  // t[1].heads may be 0
  long long batch = 0, tokens = 0;
  int head_dim = 0, pairs = 0, axes = 0;
  int interleaved = 0, inverse = 0;
  const void *pos = nullptr;
  int pos_float = 0;
  long long ps[3] = {0, 0, 0};  // axis, batch, token
  const double *turns = nullptr;  // [pairs] turns (frequency / 2 pi) per unit of position
  const int *axis = nullptr;      // [pairs]
};
cudaError_t rotary(int T, const RotaryParams &p, cudaStream_t st);

// ---- attention (attention.cu, attention_tc.cu) --------------------------------

struct AttnTensor {
  const void *p = nullptr;
  long long s[3] = {0, 0, 0};  // batch, token, head
};
struct AttnParams {
  int batch = 0, heads = 0, kv_heads = 0, head_dim = 0;
  int q_tokens = 0, k_tokens = 0;
  AttnTensor q, k, v, out;
  const int *q_lens = nullptr, *k_lens = nullptr;  // [batch] or null
  int causal_block = 0;
  float scale = 1.0f;
  float *lse = nullptr;  // [batch][heads][q_tokens]
  // backward
  AttnTensor dout, dq, dk, dv;
  // workspace: forward: partial outputs and sums of the splits; backward: row
  // sums of dout * out
  float *ws = nullptr;
  int *err = nullptr;  // host-mapped word: a tensor-core kernel gave up a bounded wait
  long long wait = 0;  // cycles such a wait may take; 0: the default
};
// Bytes of workspace of the forward / backward.
size_t attention_workspace(int T, const AttnParams &p, bool backward);
cudaError_t attention(int T, const AttnParams &p, cudaStream_t st);
cudaError_t attention_backward(int T, const AttnParams &p, cudaStream_t st);
// The tensor-core kernels (bf16): whether they take these tensors (head sizes
// that are multiples of 8, 16-byte aligned rows, a positive scale), the shares
// the forward splits the keys into, and the kernels without the joining or the
// row sums that surround them.
bool attention_tc_takes(const AttnParams &p, bool backward);
int attention_tc_splits(const AttnParams &p);
cudaError_t attention_tc(const AttnParams &p, bool backward, cudaStream_t st);

// ---- AdamW (adamw.cu) -----------------------------------------------------------

constexpr int kAdamwBlock = 256;   // elements that share the scales of 8-bit moments
constexpr int kAdamwChunk = 8;     // blocks one CTA updates
constexpr int kAdamwGrads = 440;   // gradient pointers one launch carries
// Up to kAdamwChunk blocks of one tensor.
struct AdamwChunk {
  float *param;           // its first element
  long long state_block;  // of the flat moments
  int tensor, block;      // first block within the tensor
  int elems, decay;
};
struct AdamwState {
  void *m, *v;             // f32 or int8 / uint8, [blocks * kAdamwBlock]
  float *m_scale, *v_scale;  // [blocks], 8 bits only
};
// Device words of an optimiser: the steps taken, and the CTAs of the running
// step that have read them.
struct AdamwClock {
  long long step;
  unsigned int done;
  unsigned int pad;
};
struct AdamwHyper {
  float lr, beta1, one_minus_beta1, beta2, one_minus_beta2, eps, weight_decay;
  double log_beta1, log_beta2;
};
struct AdamwGrads {
  const void *p[kAdamwGrads];
};
// One launch over `chunks` of tensors [first_tensor, ...), whose gradients are
// grads.p[tensor - first_tensor]. `last`: the launch ends the step and advances
// the clock.
cudaError_t adamw_step(int bits, int grad_type, const AdamwChunk *chunks, long long n_chunks, int first_tensor,
                       const AdamwGrads &grads, const AdamwState &state, const AdamwHyper &h, const float *lr_device,
                       AdamwClock *clock, bool last, cudaStream_t st);
// The f32 values of 8-bit moments.
cudaError_t adamw_moments(const AdamwState &state, long long blocks, float *m, float *v, cudaStream_t st);

}  // namespace gpu
}  // namespace illumina
