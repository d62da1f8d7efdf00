// C entry points of the token operators and of the AdamW step: argument
// checks, and the optimiser's tensor table.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <utility>
#include <vector>

#include "api.h"
#include "host.h"
#include "illumina.h"
#include "kernels.h"
#include "token_ops.h"

using namespace illumina;

namespace {

constexpr long long kMostRows = 1ll << 31;   // a launch's grid
constexpr long long kMostBlocks = 1ll << 30;

void require_precision(int precision, const char *op) {
  require(precision == ILLUMINA_PRECISION_F32 || precision == ILLUMINA_PRECISION_BF16,
          std::string(op) + ": unknown precision");
}
bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
// Vectors of 32-bit values (weights, statistics, lengths); any may be null.
template <typename... P>
bool words(const P *...p) {
  return (aligned(p, 4) && ...);
}
size_t size_of(int precision) { return precision == ILLUMINA_PRECISION_F32 ? 4 : 2; }

void check_norm(int precision, long long rows, int c, const char *op) {
  require_precision(precision, op);
  require(rows >= 0 && rows < kMostRows, std::string(op) + ": rows outside [0, 2^31)");
  require(c > 0 && c < (1 << 28), std::string(op) + ": width outside [1, 2^28)");
}

gpu::RotaryTensor rotary_tensor(const illumina_rotary_tensor &t, int precision, bool some) {
  require(t.heads >= 0, "rotary: negative head count");
  require(!some || t.heads == 0 || (t.x && t.y), "rotary: null pointer");
  require(aligned(t.x, size_of(precision)) && aligned(t.y, size_of(precision)), "rotary: misaligned tensor");
  gpu::RotaryTensor r;
  r.x = t.x, r.y = t.y, r.heads = t.heads;
  for (int i = 0; i < 3; i++) r.xs[i] = t.x_stride[i], r.ys[i] = t.y_stride[i];
  return r;
}

gpu::AttnTensor attn_tensor(const illumina_attention_tensor &t, int precision, bool some) {
  require(!some || t.data, "attention: null pointer");
  require(aligned(t.data, size_of(precision)), "attention: misaligned tensor");
  gpu::AttnTensor r;
  r.p = t.data;
  for (int i = 0; i < 3; i++) r.s[i] = t.stride[i];
  return r;
}

// Sizes alone (a workspace query), or with pointers.
gpu::AttnParams attn_params(const illumina_attention_args *a, bool backward, bool pointers) {
  require(a != nullptr, "attention: null arguments");
  require_precision(a->precision, "attention");
  require(a->batch >= 0 && a->heads >= 0 && a->q_tokens >= 0 && a->k_tokens >= 0, "attention: negative size");
  require(a->kv_heads > 0 ? a->heads % a->kv_heads == 0 : a->heads == 0,
          "attention: heads must be a multiple of kv_heads");
  require(a->head_dim >= 1 && a->head_dim <= 128, "attention: head_dim outside [1, 128]");
  require(a->q_tokens <= (1 << 28) && a->k_tokens <= (1 << 28), "attention: more than 2^28 tokens");
  require(a->causal_block >= 0, "attention: negative causal_block");
  const double rows = (double)a->batch * a->heads * ((double)a->q_tokens + 32) / 32;
  const double keys = (double)a->batch * a->kv_heads * ((double)a->k_tokens + 32) / 32;
  require(rows < 16e6 && keys < 1e9, "attention: too many rows for one call");
  require(words(a->q_lens, a->k_lens, a->lse), "attention: misaligned lengths or lse");
  gpu::AttnParams p;
  p.batch = a->batch, p.heads = a->heads, p.kv_heads = a->kv_heads, p.head_dim = a->head_dim;
  p.q_tokens = a->q_tokens, p.k_tokens = a->k_tokens, p.causal_block = a->causal_block, p.scale = a->scale;
  p.q_lens = a->q_lens, p.k_lens = a->k_lens, p.lse = a->lse, p.ws = (float *)a->workspace;
  const bool q = pointers && (long long)a->batch * a->heads * a->q_tokens > 0;
  const bool k = pointers && (long long)a->batch * a->kv_heads * a->k_tokens > 0;
  p.q = attn_tensor(a->q, a->precision, q), p.k = attn_tensor(a->k, a->precision, k);
  p.v = attn_tensor(a->v, a->precision, k), p.out = attn_tensor(a->out, a->precision, q);
  if (pointers) require(!q || a->lse, "attention: null lse");
  if (backward) {
    p.dout = attn_tensor(a->dout, a->precision, q), p.dq = attn_tensor(a->dq, a->precision, q);
    p.dk = attn_tensor(a->dk, a->precision, k), p.dv = attn_tensor(a->dv, a->precision, k);
  }
  if (pointers) {
    const size_t need = gpu::attention_workspace(a->precision, p, backward);
    require(need == 0 || (a->workspace && aligned(a->workspace, 16)), "attention: workspace missing or misaligned");
    require(a->workspace_bytes >= need, "attention: workspace holds " + std::to_string(a->workspace_bytes) +
                                            " bytes, " + std::to_string(need) + " are needed");
  }
  return p;
}

// Allows a scope calls that a capture, on whichever thread, would otherwise be
// ended by: allocating and freeing memory that the capture does not know.
struct Uncaptured {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  const bool set = cudaThreadExchangeStreamCaptureMode(&mode) == cudaSuccess;
  ~Uncaptured() {
    if (set) cudaThreadExchangeStreamCaptureMode(&mode);
  }
};

// The words that attention kernels set when they give up a bounded wait, one a
// device: host memory that every device can write, allocated on first use (a
// call that is being captured included).
constexpr int kMostDevices = 64;
int *attention_words() {
  static int *const words = [] {
    const Uncaptured scope;
    void *p = nullptr;
    cuda_check(cudaHostAlloc(&p, kMostDevices * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped),
               "attention: cudaHostAlloc");
    std::memset(p, 0, kMostDevices * sizeof(int));
    return (int *)p;
  }();
  return words;
}
// The current device's word; whoever finds it set clears it and reports it.
int *attention_error() {
  int device = 0;
  cuda_check(cudaGetDevice(&device), "attention: cudaGetDevice");
  require(device < kMostDevices, "attention: more devices than expected");
  int *word = attention_words() + device;
  if (__atomic_exchange_n(word, 0, __ATOMIC_ACQ_REL))
    throw Error(ILLUMINA_TIMEOUT, "attention: a kernel of an earlier call on this device gave up a bounded wait");
  return word;
}
thread_local long long g_attention_wait = 0;

}  // namespace

struct illumina_adamw {
  int device = 0, tensors = 0, bits = 32, grad_precision = 0;
  long long blocks = 0;
  std::vector<long long> counts;
  // launches: chunks [chunk0, chunk1) of tensors from `first` on
  struct Group {
    int first, end;
    long long chunk0, chunk1;
  };
  std::vector<Group> groups;
  void *memory = nullptr;  // clock, chunk table
  gpu::AdamwClock *clock = nullptr;
  gpu::AdamwChunk *chunks = nullptr;
  gpu::AdamwState state{};
  ~illumina_adamw() {  // at any time, if an interpreter collects it
    const Uncaptured scope;
    if (memory) cudaFree(memory);
  }
};

namespace {

// Makes the optimiser's device current for a scope.
struct OnDevice {
  int before = -1;
  explicit OnDevice(int device) {
    cuda_check(cudaGetDevice(&before), "cudaGetDevice");
    if (before == device) before = -1;
    else cuda_check(cudaSetDevice(device), "cudaSetDevice");
  }
  ~OnDevice() {
    if (before >= 0) cudaSetDevice(before);
  }
};

long long blocks_of(long long count) { return (count + gpu::kAdamwBlock - 1) / gpu::kAdamwBlock; }

}  // namespace

extern "C" {

illumina_status illumina_op_layer_norm(int precision, const void *x, long long x_stride, long long rows, int c,
                                       const float *w, const float *b, float eps, void *y, long long y_stride,
                                       float *mean, float *rstd, void *stream) {
  ILL_TRY
  check_norm(precision, rows, c, "layer_norm");
  require(rows == 0 || (x && y), "layer_norm: null pointer");
  require(aligned(x, size_of(precision)) && aligned(y, size_of(precision)), "layer_norm: misaligned tensor");
  require(words(w, b, mean, rstd), "layer_norm: misaligned weights or statistics");
  require(eps >= 0, "layer_norm: eps must not be negative");
  cuda_check(gpu::layer_norm(precision, x, x_stride, rows, c, w, b, eps, y, y_stride, mean, rstd, (cudaStream_t)stream),
             "layer_norm");
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_op_layer_norm_workspace(long long rows, int c, size_t *bytes) {
  ILL_TRY
  require(bytes != nullptr, "layer_norm: null pointer");
  check_norm(ILLUMINA_PRECISION_F32, rows, c, "layer_norm");
  *bytes = (size_t)gpu::layer_norm_blocks(rows, c) * 2 * c * sizeof(float);
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_op_layer_norm_backward(int precision, const void *dy, long long dy_stride, const void *x,
                                                long long x_stride, long long rows, int c, const float *w,
                                                const float *mean, const float *rstd, void *dx, long long dx_stride,
                                                float *dw, float *db, void *workspace, size_t workspace_bytes,
                                                void *stream) {
  ILL_TRY
  check_norm(precision, rows, c, "layer_norm_backward");
  require(rows == 0 || (dy && x && mean && rstd), "layer_norm_backward: null pointer");
  const size_t e = size_of(precision);
  require(aligned(x, e) && aligned(dy, e) && aligned(dx, e), "layer_norm_backward: misaligned tensor");
  require(words(w, mean, rstd, dw, db), "layer_norm_backward: misaligned weights or statistics");
  if (dw || db) {
    const size_t need = (size_t)gpu::layer_norm_blocks(rows, c) * 2 * c * sizeof(float);
    require(need == 0 || (workspace && aligned(workspace, 16)), "layer_norm_backward: workspace missing or misaligned");
    require(workspace_bytes >= need, "layer_norm_backward: workspace holds " + std::to_string(workspace_bytes) +
                                         " bytes, " + std::to_string(need) + " are needed");
  }
  cuda_check(gpu::layer_norm_backward(precision, dy, dy_stride, x, x_stride, rows, c, w, mean, rstd, dx, dx_stride, dw,
                                      db, (float *)workspace, (cudaStream_t)stream),
             "layer_norm_backward");
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_op_rotary(const illumina_rotary_args *a, void *stream) {
  ILL_TRY
  require(a != nullptr, "rotary: null arguments");
  require_precision(a->precision, "rotary");
  require(a->batch >= 0 && a->tokens >= 0, "rotary: negative size");
  require(a->batch == 0 || a->tokens < kMostBlocks / a->batch, "rotary: more than 2^30 tokens");
  require(a->head_dim >= 1 && a->head_dim <= 1024, "rotary: head_dim outside [1, 1024]");
  require(a->pairs >= 1 && a->pairs <= a->head_dim / 2, "rotary: pairs outside [1, head_dim / 2]");
  require(a->axes >= 1, "rotary: axes must be positive");
  const bool some = a->batch * a->tokens > 0 && (a->first.heads > 0 || a->second.heads > 0);
  gpu::RotaryParams p;
  p.t[0] = rotary_tensor(a->first, a->precision, some);
  p.t[1] = rotary_tensor(a->second, a->precision, some);
  require((long long)a->first.heads + a->second.heads <= 65536, "rotary: more than 65536 heads");
  require(!some || (a->positions && a->turns && a->axis), "rotary: null pointer");
  require(aligned(a->positions, 4) && aligned(a->turns, 8) && words(a->axis), "rotary: misaligned positions or plan");
  p.batch = a->batch, p.tokens = a->tokens, p.head_dim = a->head_dim, p.pairs = a->pairs, p.axes = a->axes;
  p.interleaved = a->interleaved, p.inverse = a->inverse, p.pos = a->positions, p.pos_float = a->positions_float;
  p.turns = a->turns, p.axis = a->axis;
  for (int i = 0; i < 3; i++) p.ps[i] = a->position_stride[i];
  cuda_check(gpu::rotary(a->precision, p, (cudaStream_t)stream), "rotary");
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_op_attention_workspace(const illumina_attention_args *a, int backward, size_t *bytes) {
  ILL_TRY
  require(bytes != nullptr, "attention: null pointer");
  *bytes = gpu::attention_workspace(a ? a->precision : 0, attn_params(a, backward != 0, false), backward != 0);
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_op_attention(const illumina_attention_args *a, void *stream) {
  ILL_TRY
  gpu::AttnParams p = attn_params(a, false, true);
  p.err = attention_error(), p.wait = g_attention_wait;
  cuda_check(gpu::attention(a->precision, p, (cudaStream_t)stream), "attention");
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_op_attention_backward(const illumina_attention_args *a, void *stream) {
  ILL_TRY
  gpu::AttnParams p = attn_params(a, true, true);
  p.err = attention_error(), p.wait = g_attention_wait;
  cuda_check(gpu::attention_backward(a->precision, p, (cudaStream_t)stream), "attention_backward");
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_op_attention_status(void) {
  ILL_TRY
  attention_error();
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_op_attention_set_wait_limit(long long cycles) {
  ILL_TRY
  require(cycles >= 0, "attention: negative wait limit");
  g_attention_wait = cycles;
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_adamw_blocks(const long long *counts, int tensors, long long *blocks) {
  ILL_TRY
  require(blocks && tensors >= 0 && (counts || tensors == 0), "adamw: bad arguments");
  long long n = 0;
  for (int i = 0; i < tensors; i++) {
    require(counts[i] >= 0 && counts[i] < (1ll << 40), "adamw: tensor size outside [0, 2^40)");
    n += blocks_of(counts[i]);
    require(n <= kMostBlocks, "adamw: more than 2^30 blocks");
  }
  *blocks = n;
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_adamw_create(const illumina_adamw_options *o, illumina_adamw **out) {
  ILL_TRY
  require(o && out, "adamw: null argument");
  require(o->tensors > 0 && o->params && o->counts, "adamw: no tensors");
  require(o->moment_bits == 32 || o->moment_bits == 8, "adamw: moment_bits must be 32 or 8");
  require_precision(o->grad_precision, "adamw");
  long long blocks = 0;
  const illumina_status st = illumina_adamw_blocks(o->counts, o->tensors, &blocks);
  if (st != ILLUMINA_OK) return st;
  require(blocks > 0, "adamw: every tensor is empty");
  require(o->m && o->v && aligned(o->m, 16) && aligned(o->v, 16), "adamw: moments missing or misaligned");
  require(o->moment_bits == 32 || (o->m_scale && o->v_scale), "adamw: 8-bit moments need scales");
  require(words(o->m_scale, o->v_scale), "adamw: misaligned scales");
  std::unique_ptr<illumina_adamw> opt(new illumina_adamw);
  opt->device = o->device, opt->tensors = o->tensors, opt->bits = o->moment_bits;
  opt->grad_precision = o->grad_precision, opt->blocks = blocks;
  opt->counts.assign(o->counts, o->counts + o->tensors);
  std::vector<gpu::AdamwChunk> chunks;
  long long first = 0;
  for (int i = 0; i < o->tensors; i++) {
    const long long n = blocks_of(o->counts[i]);
    require(n == 0 || (o->params[i] && aligned(o->params[i], 4)), "adamw: parameter pointer missing or misaligned");
    if (opt->groups.empty() || i - opt->groups.back().first >= gpu::kAdamwGrads)
      opt->groups.push_back({i, i, (long long)chunks.size(), (long long)chunks.size()});
    const int decay = o->decay ? o->decay[i] != 0 : 1;
    constexpr long long most = gpu::kAdamwChunk * gpu::kAdamwBlock;
    for (long long b = 0; b < n; b += gpu::kAdamwChunk) {
      const long long at = b * gpu::kAdamwBlock, left = o->counts[i] - at;
      chunks.push_back({o->params[i] + at, first + b, i, (int)b, (int)(left < most ? left : most), decay});
    }
    first += n;
    opt->groups.back().end = i + 1;
    opt->groups.back().chunk1 = (long long)chunks.size();
  }
  std::vector<std::pair<uintptr_t, uintptr_t>> places;
  for (int i = 0; i < o->tensors; i++)
    if (o->counts[i] > 0) {
      const uintptr_t p = reinterpret_cast<uintptr_t>(o->params[i]);
      places.emplace_back(p, p + (uintptr_t)o->counts[i] * sizeof(float));
    }
  std::sort(places.begin(), places.end());
  for (size_t i = 1; i < places.size(); i++)
    require(places[i - 1].second <= places[i].first, "adamw: parameters overlap, or one is listed twice");
  OnDevice on(o->device);
  const size_t a = 256, cb = chunks.size() * sizeof(chunks[0]);
  cuda_check(cudaMalloc(&opt->memory, a + cb), "adamw: cudaMalloc");
  char *base = (char *)opt->memory;
  opt->clock = (gpu::AdamwClock *)base;
  opt->chunks = (gpu::AdamwChunk *)(base + a);
  cuda_check(cudaMemset(base, 0, a), "adamw: clear");
  cuda_check(cudaMemcpy(opt->chunks, chunks.data(), cb, cudaMemcpyHostToDevice), "adamw: upload");
  cuda_check(cudaStreamSynchronize(nullptr), "adamw: upload");  // steps may run on streams that do not wait for this one
  opt->state.m = o->m, opt->state.v = o->v, opt->state.m_scale = o->m_scale, opt->state.v_scale = o->v_scale;
  *out = opt.release();
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_adamw_destroy(illumina_adamw *opt) {
  ILL_TRY
  if (!opt) return ILLUMINA_OK;
  OnDevice on(opt->device);
  delete opt;  // cudaFree waits for the device's queued steps
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_adamw_step(illumina_adamw *opt, const void *const *grads, const illumina_adamw_hyper *h,
                                    void *stream) {
  ILL_TRY
  require(opt && grads && h, "adamw: null argument");
  require(h->beta1 >= 0 && h->beta1 < 1 && h->beta2 >= 0 && h->beta2 < 1, "adamw: betas outside [0, 1)");
  require(h->eps == 0 || h->eps >= FLT_MIN, "adamw: eps must be 0 or a normal float");
  require(std::isfinite(h->lr) && std::isfinite(h->weight_decay), "adamw: bad hyperparameter");
  require(words(h->lr_device), "adamw: misaligned lr");
  const size_t e = size_of(opt->grad_precision);
  for (int i = 0; i < opt->tensors; i++)
    require(opt->counts[i] == 0 || (grads[i] && aligned(grads[i], e)),
            "adamw: gradient " + std::to_string(i) + " missing or misaligned");
  gpu::AdamwHyper d;
  d.lr = (float)h->lr, d.beta1 = (float)h->beta1, d.one_minus_beta1 = (float)(1.0 - h->beta1);
  d.beta2 = (float)h->beta2, d.one_minus_beta2 = (float)(1.0 - h->beta2), d.eps = (float)h->eps;
  d.weight_decay = (float)h->weight_decay, d.log_beta1 = std::log(h->beta1), d.log_beta2 = std::log(h->beta2);
  OnDevice on(opt->device);
  size_t last = opt->groups.size();
  while (last > 0 && opt->groups[last - 1].chunk1 == opt->groups[last - 1].chunk0) last--;
  for (size_t g = 0; g < last; g++) {
    const auto &group = opt->groups[g];
    if (group.chunk1 == group.chunk0) continue;
    gpu::AdamwGrads gr{};
    for (int i = group.first; i < group.end; i++) gr.p[i - group.first] = grads[i];
    cuda_check(gpu::adamw_step(opt->bits, opt->grad_precision, opt->chunks + group.chunk0,
                               group.chunk1 - group.chunk0, group.first, gr, opt->state, d, h->lr_device, opt->clock,
                               g == last - 1, (cudaStream_t)stream),
               "adamw_step");
  }
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_adamw_get_steps(illumina_adamw *opt, long long *steps, void *stream) {
  ILL_TRY
  require(opt && steps, "adamw: null argument");
  OnDevice on(opt->device);
  cuda_check(cudaMemcpyAsync(steps, &opt->clock->step, sizeof(*steps), cudaMemcpyDeviceToHost, (cudaStream_t)stream),
             "adamw_get_steps");
  cuda_check(cudaStreamSynchronize((cudaStream_t)stream), "adamw_get_steps");
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_adamw_set_steps(illumina_adamw *opt, long long steps, void *stream) {
  ILL_TRY
  require(opt && steps >= 0, "adamw: bad arguments");
  OnDevice on(opt->device);
  cuda_check(cudaMemcpyAsync(&opt->clock->step, &steps, sizeof(steps), cudaMemcpyHostToDevice, (cudaStream_t)stream),
             "adamw_set_steps");
  cuda_check(cudaStreamSynchronize((cudaStream_t)stream), "adamw_set_steps");  // `steps` is on this frame
  return ILLUMINA_OK;
  ILL_CATCH
}

illumina_status illumina_adamw_moments(illumina_adamw *opt, float *m, float *v, void *stream) {
  ILL_TRY
  require(opt && m && v && aligned(m, 16) && aligned(v, 16), "adamw: moments missing or misaligned");
  require(opt->bits == 8, "adamw: the moments are in 32 bits already");
  OnDevice on(opt->device);
  cuda_check(gpu::adamw_moments(opt->state, opt->blocks, m, v, (cudaStream_t)stream), "adamw_moments");
  return ILLUMINA_OK;
  ILL_CATCH
}

}  // extern "C"
