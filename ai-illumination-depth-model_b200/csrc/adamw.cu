// AdamW over many tensors in one launch, with moments in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// Bound by HBM: p, g, m and v are read once, p, m and v written once. A CTA
// takes a chunk of 8 blocks of 256 elements of one tensor, a warp one block:
// lane l holds elements 4l..4l+3 and 128+4l..128+4l+3, so that every access
// of aligned tensors is a whole vector. The moments of all tensors lie in flat
// arrays in which every tensor begins at a block.
//
// 8-bit moments: a block keeps m as code * scale, code in -127..127, and the
// root of v as code * scale, code in 0..255 (the root halves the range of
// exponents that the codes have to span). A moment moves by as little as a
// thousandth a step, much less than a code, so rounding to the nearest code
// would hold it in place; the code is floor(x + u) with a threshold u that
// steps evenly through [0, 1) from step to step (multiples of the golden
// ratio, offset by the element's place), which is right on average and needs
// no random state. Every operation on the way to a code is rounded on its
// own (no contraction), so that a code does not depend on the compiler. A
// root that is not zero never becomes code 0: the next step would divide by
// almost nothing.
//
// The step count lives on the device, so that a captured step can be
// replayed: every CTA reads it, the last one to finish advances it.
#include "token_common.cuh"
#include "token_ops.h"

namespace illumina {
namespace gpu {
namespace {

using namespace tok;

constexpr int kThreads = 32 * kAdamwChunk;

// The larger of two values, NaN if either is: a gradient that is not finite
// shows in its block's scale instead of being skipped by the maximum.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

template <typename G>
__device__ __forceinline__ void load_grad(const G *g, bool vec, int n, float (&o)[4]) {
  if (vec) {
    Pack<G, 4>::load(g, o);
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = j < n ? to_f32(g[j]) : 0.0f;
  }
}

// floor(x * inv + u) within [lo, hi]; codes are whole numbers in floats.
__device__ __forceinline__ float code_of(float x, float inv, float u, float lo, float hi) {
  return fminf(fmaxf(floorf(__fadd_rn(__fmul_rn(x, inv), u)), lo), hi);
}

template <int BITS, typename G>
__global__ void __launch_bounds__(kThreads) k_adamw(const AdamwTensor *__restrict__ tensors,
                                                    const AdamwChunk *__restrict__ chunks, int first_tensor,
                                                    const __grid_constant__ AdamwGrads grads, const AdamwState state,
                                                    const AdamwHyper h, const float *lr_device, AdamwClock *clock,
                                                    int last) {
  __shared__ float s_c1, s_c2;
  __shared__ long long s_t;
  const AdamwChunk chunk = chunks[blockIdx.x];
  const AdamwTensor &t = tensors[chunk.tensor];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long blk = chunk.block + warp;
  const long long at = blk * kAdamwBlock;
  const long long left = t.count - at;
  float p[2][4], g[2][4], m[2][4], v[2][4];
  float *pp = t.param + at;
  const G *gp = (const G *)grads.p[chunk.tensor - first_tensor] + at;
  const bool pvec = (reinterpret_cast<uintptr_t>(pp) & 15) == 0, gvec = (reinterpret_cast<uintptr_t>(gp) % (4 * sizeof(G))) == 0;
  const long long sb = t.first_block + blk;  // block of the flat moments
  if (left > 0) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int e = 128 * k + 4 * lane;
      const int n = (int)min(max(left - e, 0ll), 4ll);
      load_grad<G>(gp + e, gvec && n == 4, n, g[k]);
      load_grad<float>(pp + e, pvec && n == 4, n, p[k]);
      const long long i = sb * kAdamwBlock + e;
      if constexpr (BITS == 32) {
        Pack<float, 4>::load((const float *)state.m + i, m[k]);
        Pack<float, 4>::load((const float *)state.v + i, v[k]);
      } else {
        const float ms = state.m_scale[sb], vs = state.v_scale[sb];
        const char4 mc = *reinterpret_cast<const char4 *>((const int8_t *)state.m + i);
        const uchar4 vc = *reinterpret_cast<const uchar4 *>((const uint8_t *)state.v + i);
        m[k][0] = __fmul_rn(mc.x, ms), m[k][1] = __fmul_rn(mc.y, ms);
        m[k][2] = __fmul_rn(mc.z, ms), m[k][3] = __fmul_rn(mc.w, ms);
        v[k][0] = __fmul_rn(vc.x, vs), v[k][1] = __fmul_rn(vc.y, vs);
        v[k][2] = __fmul_rn(vc.z, vs), v[k][3] = __fmul_rn(vc.w, vs);
#pragma unroll
        for (int j = 0; j < 4; j++) v[k][j] = __fmul_rn(v[k][j], v[k][j]);
      }
    }
  }
  if (threadIdx.x == 0) {
    const long long step = *(volatile long long *)&clock->step + 1;
    const double c1 = -expm1((double)step * h.log_beta1), c2 = -expm1((double)step * h.log_beta2);
    s_t = step;
    s_c1 = (float)((lr_device ? (double)*lr_device : (double)h.lr) / c1);
    s_c2 = (float)(1.0 / sqrt(c2));
    if (last) {
      // the clock moves on once every CTA of this launch has read it
      __threadfence();
      if (atomicAdd(&clock->done, 1u) == gridDim.x - 1) {
        clock->done = 0;
        clock->step = step;
      }
    }
  }
  __syncthreads();
  if (left <= 0) return;
  const float lr = lr_device ? *lr_device : h.lr;
  const float keep = t.decay ? 1.0f - lr * h.weight_decay : 1.0f;
  const float c1 = s_c1, c2 = s_c2;
  float mtop = 0, rtop = 0;
#pragma unroll
  for (int k = 0; k < 2; k++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float gg = g[k][j];
      m[k][j] = __fadd_rn(__fmul_rn(m[k][j], h.beta1), __fmul_rn(gg, h.one_minus_beta1));
      v[k][j] = __fadd_rn(__fmul_rn(v[k][j], h.beta2), __fmul_rn(__fmul_rn(gg, gg), h.one_minus_beta2));
      const float root = __fsqrt_rn(v[k][j]);
      p[k][j] = p[k][j] * keep - c1 * m[k][j] / (root * c2 + h.eps);
      if constexpr (BITS == 8) {
        v[k][j] = root;
        mtop = max_nan(mtop, fabsf(m[k][j]));
        rtop = max_nan(rtop, root);
      }
    }
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const int e = 128 * k + 4 * lane;
    const int n = (int)min(max(left - e, 0ll), 4ll);
    if (pvec && n == 4) {
      Pack<float, 4>::store(pp + e, p[k]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (j < n) pp[e + j] = p[k][j];
    }
  }
  if constexpr (BITS == 32) {
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const long long i = sb * kAdamwBlock + 128 * k + 4 * lane;
      Pack<float, 4>::store((float *)state.m + i, m[k]);
      Pack<float, 4>::store((float *)state.v + i, v[k]);
    }
  } else {
    constexpr float kTiny = 7.888609e-31f;  // 2^-100: below it the reciprocal of a scale would overflow
    mtop = warp_max(mtop);
    rtop = warp_max(rtop);
    const float ms = mtop < kTiny ? 0.0f : __fmul_rn(mtop, (float)(1.0 / 127.0));
    const float rs = rtop < kTiny ? 0.0f : __fmul_rn(rtop, (float)(1.0 / 255.0));
    const float mi = ms == 0.0f ? 0.0f : __frcp_rn(ms), ri = rs == 0.0f ? 0.0f : __frcp_rn(rs);
    if (lane == 0) state.m_scale[sb] = ms, state.v_scale[sb] = rs;
    const uint32_t sweep = (uint32_t)s_t * 0x9E3779B9u;
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const long long i = sb * kAdamwBlock + 128 * k + 4 * lane;
      int mc[4], vc[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float u = (float)(((uint32_t)(i + j) * 0x85EBCA6Bu + sweep) >> 8) * 0x1p-24f;
        mc[j] = (int)code_of(m[k][j], mi, u, -127.0f, 127.0f);
        const float root = v[k][j];
        vc[j] = (int)code_of(root, ri, u, root > 0.0f && rs > 0.0f ? 1.0f : 0.0f, 255.0f);
      }
      *reinterpret_cast<char4 *>((int8_t *)state.m + i) =
          make_char4((signed char)mc[0], (signed char)mc[1], (signed char)mc[2], (signed char)mc[3]);
      *reinterpret_cast<uchar4 *>((uint8_t *)state.v + i) = make_uchar4(vc[0], vc[1], vc[2], vc[3]);
    }
  }
}

__global__ void __launch_bounds__(256) k_adamw_moments(const AdamwState state, long long n4, float *__restrict__ m,
                                                       float *__restrict__ v) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n4; i += (long long)gridDim.x * 256) {
    const long long b = i / (kAdamwBlock / 4);
    const float ms = state.m_scale[b], vs = state.v_scale[b];
    const char4 mc = reinterpret_cast<const char4 *>(state.m)[i];
    const uchar4 vc = reinterpret_cast<const uchar4 *>(state.v)[i];
    const float r0 = vc.x * vs, r1 = vc.y * vs, r2 = vc.z * vs, r3 = vc.w * vs;
    reinterpret_cast<float4 *>(m)[i] = make_float4(mc.x * ms, mc.y * ms, mc.z * ms, mc.w * ms);
    reinterpret_cast<float4 *>(v)[i] = make_float4(r0 * r0, r1 * r1, r2 * r2, r3 * r3);
  }
}

}  // namespace

cudaError_t adamw_step(int bits, int grad_type, const AdamwTensor *tensors, const AdamwChunk *chunks, long long n,
                       int first_tensor, const AdamwGrads &grads, const AdamwState &state, const AdamwHyper &h,
                       const float *lr_device, AdamwClock *clock, bool last, cudaStream_t st) {
  const unsigned grid = (unsigned)n;
  if (bits == 32 && grad_type == 0)
    k_adamw<32, float><<<grid, kThreads, 0, st>>>(tensors, chunks, first_tensor, grads, state, h, lr_device, clock, last);
  else if (bits == 32)
    k_adamw<32, bf16><<<grid, kThreads, 0, st>>>(tensors, chunks, first_tensor, grads, state, h, lr_device, clock, last);
  else if (grad_type == 0)
    k_adamw<8, float><<<grid, kThreads, 0, st>>>(tensors, chunks, first_tensor, grads, state, h, lr_device, clock, last);
  else
    k_adamw<8, bf16><<<grid, kThreads, 0, st>>>(tensors, chunks, first_tensor, grads, state, h, lr_device, clock, last);
  return cudaGetLastError();
}

cudaError_t adamw_moments(const AdamwState &state, long long blocks, float *m, float *v, cudaStream_t st) {
  const long long n4 = blocks * (kAdamwBlock / 4);
  if (n4 == 0) return cudaSuccess;
  const long long want = (n4 + 255) / 256;
  k_adamw_moments<<<(unsigned)(want < 148 * 16 ? want : 148 * 16), 256, 0, st>>>(state, n4, m, v);
  return cudaGetLastError();
}

}  // namespace gpu
}  // namespace illumina
