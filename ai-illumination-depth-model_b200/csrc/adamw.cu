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
// almost nothing. It stays at code 1 then, above its own value, while the
// largest of its block is 255 times as large: its element's steps are too
// small on average, by as much as the root is too large.
//
// Measured: 112 tensors of 1.4 M elements, 32-bit moments: 10 us on the GPU,
// 12 us a call (the pointers are checked and sent each time); 8-bit moments,
// bf16 gradients: 213 us for 81.9 M elements (5.4 TB/s, 14 bytes an element),
// bound by instruction issue: 64 instructions an element, where one value an
// instruction took 82 and 255 us. The moments as floats: 135 us (6.1 TB/s).
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
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// a / b for b = 0 or normal, within 2 steps.
__device__ __forceinline__ float quotient(float a, float b) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(b));
  return a * r;
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
__device__ __forceinline__ typename RawPack<T, 4>::type load_raw(const T *p, int n, bool whole) {
  typedef typename RawPack<T, 4>::type Raw;
  if (whole) return *reinterpret_cast<const Raw *>(p);
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

template <typename T>
__device__ __forceinline__ void unpack_pairs(typename RawPack<T, 4>::type raw, float2 *to) {
  float e[4];
  RawPack<T, 4>::unpack(raw, e);
  to[0] = make_float2(e[0], e[1]), to[1] = make_float2(e[2], e[3]);
}

// A sum of products that must not be merged with them: the compiler merges
// packed products and sums, rounding modes or not, but not across widths.
__device__ __forceinline__ float2 add_apart(float2 a, float2 b) {
  return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y));
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// Bytes j and j + 1 of w as floats, without the conversion unit (which the square roots
// and reciprocals need): 2^23 + byte, minus 2^23 (and the bias of signed codes).
__device__ __forceinline__ float2 byte_values(uint32_t w, int j, float bias) {
  return __fadd2_rn(make_float2(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7650 + j)),
                                __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7651 + j))),
                    both(-bias));
}
// floor(x * inv + u), as 1.5 * 2^23 + the code: a sum rounded down to a whole
// number. The caller limits it.
constexpr float kMagic = 12582912.0f;
__device__ __forceinline__ float2 codes_of(float2 x, float2 inv, float2 u) {
  return __fadd2_rd(add_apart(__fmul2_rn(x, inv), u), both(kMagic));
}
__device__ __forceinline__ uint32_t limited(float s, float lo, float hi) {
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
    const bool pw = left >= kAdamwBlock && reinterpret_cast<uintptr_t>(pp) % sizeof(float4) == 0;
    const bool gw = left >= kAdamwBlock && reinterpret_cast<uintptr_t>(gp) % sizeof(held.g[0]) == 0;
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int e = 128 * k + 4 * lane, n = min(max(left - e, 0), 4);
      held.p[k] = load_raw<float>(pp + e, n, pw);
      held.g[k] = load_raw<G>(gp + e, n, gw);
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
    // elements 128 k + 4 l + 2 q and the next: two operations an instruction
    float2 p[4], g[4], m[4], v[4];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      unpack_pairs<float>(held.p[k], p + 2 * k);
      unpack_pairs<G>(held.g[k], g + 2 * k);
      if constexpr (BITS == 32) {
        unpack_pairs<float>(held.m[k], m + 2 * k);
        unpack_pairs<float>(held.v[k], v + 2 * k);
      } else {
#pragma unroll
        for (int q = 0; q < 2; q++) {
          // signed codes with their sign bit flipped are 128 too large
          m[2 * k + q] = __fmul2_rn(byte_values(held.m[k] ^ 0x80808080u, 2 * q, 8388736.0f), both(held.ms));
          const float2 root = __fmul2_rn(byte_values(held.v[k], 2 * q, 8388608.0f), both(held.vs));
          v[2 * k + q] = __fmul2_rn(root, root);
        }
      }
    }
    fetch(c + gridDim.x);  // the next chunk's loads run under this one's arithmetic
    if (left <= 0) continue;
    float *pp = now.param + warp * kAdamwBlock;
    const long long sb = now.state_block + warp;
    const bool whole = left >= kAdamwBlock && (reinterpret_cast<uintptr_t>(pp) & 15) == 0;
    const float keep = now.decay ? decayed : 1.0f;
    float mtop = 0, rtop = 0;
#pragma unroll
    for (int q = 0; q < 4; q++) {
      m[q] = add_apart(__fmul2_rn(m[q], both(h.beta1)), __fmul2_rn(g[q], both(h.one_minus_beta1)));
      v[q] = add_apart(__fmul2_rn(v[q], both(h.beta2)), __fmul2_rn(__fmul2_rn(g[q], g[q]), both(h.one_minus_beta2)));
      const float2 root = make_float2(__fsqrt_rn(v[q].x), __fsqrt_rn(v[q].y));
      // within 2 steps of the quotient: steps of the update, not of the parameter
      const float2 up = __fmul2_rn(m[q], both(-c1)), down = __ffma2_rn(root, both(c2), both(h.eps));
      p[q] = __ffma2_rn(p[q], both(keep), make_float2(quotient(up.x, down.x), quotient(up.y, down.y)));
      if constexpr (BITS == 8) {
        v[q] = root;
        mtop = max_nan(max_nan(mtop, fabsf(m[q].x)), fabsf(m[q].y));
        rtop = max_nan(max_nan(rtop, root.x), root.y);
      }
    }
#pragma unroll
    for (int k = 0; k < 2; k++) {
      const int e = 128 * k + 4 * lane, n = min(max(left - e, 0), 4);
      const float o[4] = {p[2 * k].x, p[2 * k].y, p[2 * k + 1].x, p[2 * k + 1].y};
      if (whole) {
        Pack<float, 4>::store(pp + e, o);
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (j < n) pp[e + j] = o[j];
      }
    }
    if constexpr (BITS == 32) {
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const long long i = sb * kAdamwBlock + 128 * k + 4 * lane;
        *reinterpret_cast<float4 *>((float *)state.m + i) = make_float4(m[2 * k].x, m[2 * k].y, m[2 * k + 1].x, m[2 * k + 1].y);
        *reinterpret_cast<float4 *>((float *)state.v + i) = make_float4(v[2 * k].x, v[2 * k].y, v[2 * k + 1].x, v[2 * k + 1].y);
      }
    } else {
      constexpr float kTiny = 7.888609e-31f;  // 2^-100: below it the reciprocal of a scale would overflow
      mtop = warp_max(mtop);
      rtop = warp_max(rtop);
      const float ms = mtop < kTiny ? 0.0f : __fmul_rn(mtop, (float)(1.0 / 127.0));
      const float rs = rtop < kTiny ? 0.0f : __fmul_rn(rtop, (float)(1.0 / 255.0));
      const float mi = ms == 0.0f ? 0.0f : __frcp_rn(ms), ri = rs == 0.0f ? 0.0f : __frcp_rn(rs);
      const float least = rs > 0.0f ? 1.0f : 0.0f;
      if (lane == 0) state.m_scale[sb] = ms, state.v_scale[sb] = rs;
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const long long i = sb * kAdamwBlock + 128 * k + 4 * lane;
        uint32_t mc[4], vc[4];
        uint32_t place = (uint32_t)i * 0x85EBCA6Bu + sweep;
#pragma unroll
        for (int q = 0; q < 2; q++) {
          const float2 u = __fmul2_rn(make_float2((float)(place >> 8), (float)((place + 0x85EBCA6Bu) >> 8)), both(0x1p-24f));
          place += 2 * 0x85EBCA6Bu;
          const float2 root = v[2 * k + q];
          const float2 cm = codes_of(m[2 * k + q], both(mi), u), cv = codes_of(root, both(ri), u);
          mc[2 * q] = limited(cm.x, -127.0f, 127.0f), mc[2 * q + 1] = limited(cm.y, -127.0f, 127.0f);
          vc[2 * q] = limited(cv.x, root.x > 0.0f ? least : 0.0f, 255.0f);
          vc[2 * q + 1] = limited(cv.y, root.y > 0.0f ? least : 0.0f, 255.0f);
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
