// AdamW over many tensors in one launch, with moments in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// Bound by HBM: p, g, m and v are read once, p, m and v written once. A CTA
// takes chunks of 8 blocks of 256 elements of one tensor, a warp one block:
// lane l holds elements 4l..4l+3 and 128+4l..128+4l+3, so that every access
// of aligned tensors is a whole vector. The grid fills the GPU once and walks
// the chunks, the next one's loads in flight while one is computed: a CTA a
// chunk spent most of its life on the step's bias corrections (in 64 bits). The moments of all tensors lie in flat
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
#include <cstring>
#include <type_traits>

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

// What a lane holds of a block as it lies in memory: elements 128 k + 4 l + j.
template <int BITS, typename G>
struct Held {
  typedef typename RawPack<G, 4>::type RawG;
  typedef typename std::conditional<BITS == 32, float4, uint32_t>::type RawM;
  float4 p[2];
  RawG g[2];
  RawM m[2], v[2];
  float ms, vs;
};

template <typename T>
__device__ __forceinline__ typename RawPack<T, 4>::type load_raw(const T *p, int n) {
  typedef typename RawPack<T, 4>::type Raw;
  if (n == 4 && reinterpret_cast<uintptr_t>(p) % sizeof(Raw) == 0) return *reinterpret_cast<const Raw *>(p);
  T e[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if (j < n) e[j] = p[j];
    else from_f32(e[j], 0.0f);
  }
  Raw raw;
  memcpy(&raw, e, sizeof(raw));
  return raw;
}

// Byte j of w as a float, without the conversion unit (which the square roots
// and reciprocals need): 2^23 + byte, minus 2^23 (and the bias of signed codes).
__device__ __forceinline__ float byte_value(uint32_t w, int j, float bias) {
  return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7650 + j)) - bias;
}
// floor(x * inv + u) within [lo, hi], as 1.5 * 2^23 + the code: a sum rounded
// down to a whole number.
__device__ __forceinline__ uint32_t code_of(float x, float inv, float u, float lo, float hi) {
  constexpr float kMagic = 12582912.0f;
  const float s = __fadd_rd(__fadd_rn(__fmul_rn(x, inv), u), kMagic);
  return __float_as_uint(fminf(fmaxf(s, kMagic + lo), kMagic + hi));
}
// The low bytes of four codes.
__device__ __forceinline__ uint32_t pack_codes(const uint32_t (&c)[4]) {
  return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}

template <int BITS, typename G>
__global__ void __launch_bounds__(kThreads) k_adamw(const AdamwChunk *__restrict__ chunks, int n_chunks, int first_tensor,
                                                    const __grid_constant__ AdamwGrads grads, const AdamwState state,
                                                    const AdamwHyper h, const float *lr_device, AdamwClock *clock,
                                                    int last) {
  __shared__ float s_c1, s_c2;
  __shared__ uint32_t s_t;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  AdamwChunk chunk;
  Held<BITS, G> held;
  auto fetch = [&](int c) {
    if (c >= n_chunks) return;
    chunk = chunks[c];
    const int left = chunk.elems - warp * kAdamwBlock;
    if (left <= 0) return;
    const G *gp = (const G *)grads.p[chunk.tensor - first_tensor] + ((long long)chunk.block + warp) * kAdamwBlock;
    const float *pp = chunk.param + warp * kAdamwBlock;
    const long long sb = chunk.state_block + warp;
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int e = 128 * k + 4 * lane, n = min(max(left - e, 0), 4);
      held.p[k] = load_raw<float>(pp + e, n);
      held.g[k] = load_raw<G>(gp + e, n);
      const long long i = (sb * kAdamwBlock + e) / 4;
      held.m[k] = ((const typename Held<BITS, G>::RawM *)state.m)[i];
      held.v[k] = ((const typename Held<BITS, G>::RawM *)state.v)[i];
    }
    if constexpr (BITS == 8) held.ms = state.m_scale[sb], held.vs = state.v_scale[sb];
  };
  fetch(blockIdx.x);
  if (threadIdx.x == 0) {
    const long long step = *(volatile long long *)&clock->step + 1;
    const double c1 = -expm1((double)step * h.log_beta1), c2 = -expm1((double)step * h.log_beta2);
    s_t = (uint32_t)step;
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
  const float lr = lr_device ? *lr_device : h.lr;
  const float c1 = s_c1, c2 = s_c2, decayed = 1.0f - lr * h.weight_decay;
  const uint32_t sweep = s_t * 0x9E3779B9u;
  for (int c = blockIdx.x; c < n_chunks; c += gridDim.x) {
    const AdamwChunk now = chunk;
    const int left = now.elems - warp * kAdamwBlock;
    float p[2][4], g[2][4], m[2][4], v[2][4];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      RawPack<float, 4>::unpack(held.p[k], p[k]);
      RawPack<G, 4>::unpack(held.g[k], g[k]);
      if constexpr (BITS == 32) {
        RawPack<float, 4>::unpack(held.m[k], m[k]);
        RawPack<float, 4>::unpack(held.v[k], v[k]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          // signed codes with their sign bit flipped are 128 too large
          m[k][j] = __fmul_rn(byte_value(held.m[k] ^ 0x80808080u, j, 8388736.0f), held.ms);
          const float root = __fmul_rn(byte_value(held.v[k], j, 8388608.0f), held.vs);
          v[k][j] = __fmul_rn(root, root);
        }
      }
    }
    fetch(c + gridDim.x);  // the next chunk's loads run under this one's arithmetic
    if (left <= 0) continue;
    float *pp = now.param + warp * kAdamwBlock;
    const long long sb = now.state_block + warp;
    const bool pvec = (reinterpret_cast<uintptr_t>(pp) & 15) == 0;
    const float keep = now.decay ? decayed : 1.0f;
    float mtop = 0, rtop = 0;
#pragma unroll
    for (int k = 0; k < 2; k++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float gg = g[k][j];
        m[k][j] = __fadd_rn(__fmul_rn(m[k][j], h.beta1), __fmul_rn(gg, h.one_minus_beta1));
        v[k][j] = __fadd_rn(__fmul_rn(v[k][j], h.beta2), __fmul_rn(__fmul_rn(gg, gg), h.one_minus_beta2));
        const float root = __fsqrt_rn(v[k][j]);
        // within 2 steps of the quotient: steps of the update, not of the parameter
        p[k][j] = fmaf(p[k][j], keep, -__fdividef(c1 * m[k][j], fmaf(root, c2, h.eps)));
        if constexpr (BITS == 8) {
          v[k][j] = root;
          mtop = max_nan(mtop, fabsf(m[k][j]));
          rtop = max_nan(rtop, root);
        }
      }
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int e = 128 * k + 4 * lane, n = min(max(left - e, 0), 4);
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
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const long long i = sb * kAdamwBlock + 128 * k + 4 * lane;
        uint32_t mc[4], vc[4];
        uint32_t place = (uint32_t)i * 0x85EBCA6Bu + sweep;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float u = (float)(place >> 8) * 0x1p-24f;
          place += 0x85EBCA6Bu;
          mc[j] = code_of(m[k][j], mi, u, -127.0f, 127.0f);
          const float root = v[k][j];
          vc[j] = code_of(root, ri, u, root > 0.0f && rs > 0.0f ? 1.0f : 0.0f, 255.0f);
        }
        ((uint32_t *)state.m)[i / 4] = pack_codes(mc);
        ((uint32_t *)state.v)[i / 4] = pack_codes(vc);
      }
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

cudaError_t adamw_step(int bits, int grad_type, const AdamwChunk *chunks, long long n, int first_tensor,
                       const AdamwGrads &grads, const AdamwState &state, const AdamwHyper &h, const float *lr_device,
                       AdamwClock *clock, bool last, cudaStream_t st) {
  const int nc = (int)n;
  const long long resident = (bits == 32 ? 2 : 3) * 148;  // by registers
  const unsigned grid = (unsigned)(n < resident ? n : resident);
  if (bits == 32 && grad_type == 0)
    k_adamw<32, float><<<grid, kThreads, 0, st>>>(chunks, nc, first_tensor, grads, state, h, lr_device, clock, last);
  else if (bits == 32)
    k_adamw<32, bf16><<<grid, kThreads, 0, st>>>(chunks, nc, first_tensor, grads, state, h, lr_device, clock, last);
  else if (grad_type == 0)
    k_adamw<8, float><<<grid, kThreads, 0, st>>>(chunks, nc, first_tensor, grads, state, h, lr_device, clock, last);
  else
    k_adamw<8, bf16><<<grid, kThreads, 0, st>>>(chunks, nc, first_tensor, grads, state, h, lr_device, clock, last);
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
