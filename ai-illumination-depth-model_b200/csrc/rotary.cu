// Rotary positions with several axes: pair j of a head, which belongs to axis
// a(j), is rotated by position[a(j)] * frequency[j].
//
//   (u, v) -> (u cos - v sin, u sin + v cos)
//
// Bound by HBM: queries and keys are read and written once. A CTA takes a few
// tokens and computes each (token, pair) angle once for all heads. Angles are
// kept as turns in 64 bits: turns = position * (frequency / 2 pi), of which
// the whole part is dropped before sincospi in 32 bits, so that a position of
// a million costs no more phase error than one of ten.
//
// Measured: 2 clips of 32 frames of 196 tokens, 12 + 4 heads of 64, three axes,
// bf16: 13 us (3.9 TB/s), a third of it launch and ramp; one frame 5 us on
// the GPU, 10 us a call.
#include "token_common.cuh"
#include "token_ops.h"

namespace illumina {
namespace gpu {
namespace {

using namespace tok;

constexpr int kThreads = 256;
constexpr int kTrig = 1024;  // (token, pair) angles a CTA holds

// VW: elements a thread moves at once; halves: pairs are (j, j + pairs), so a
// thread reads VW of each half, else neighbours (2j, 2j + 1).
template <typename T, int VW, bool HALVES>
__global__ void __launch_bounds__(kThreads) k_rotary(const RotaryParams p, int tb) {
  __shared__ __align__(16) float cs[kTrig], sn[kTrig];
  const long long total = p.batch * p.tokens, first = (long long)blockIdx.x * tb;
  const int nt = (int)min((long long)tb, total - first);
  const long long b0 = first / p.tokens, n0 = first - b0 * p.tokens;
  // batch and token of the CTA's token t; the division is for the few CTAs that pass the end of a sequence
  auto token = [&](int t, long long &b, long long &n) {
    b = b0, n = n0 + t;
    if (n >= p.tokens) {
      const long long more = n / p.tokens;
      b += more, n -= more * p.tokens;
    }
  };
  for (int i = threadIdx.x; i < nt * p.pairs; i += kThreads) {
    const int t = i / p.pairs, j = i - t * p.pairs;
    long long b, n;
    token(t, b, n);
    const int a = min(max(p.axis[j], 0), p.axes - 1);
    const long long at = a * p.ps[0] + b * p.ps[1] + n * p.ps[2];
    const double pos = p.pos_float ? (double)((const float *)p.pos)[at] : (double)((const int *)p.pos)[at];
    double u = pos * p.turns[j];
    u -= rint(u);
    float s, c;
    sincospif(2.0f * (float)u, &s, &c);
    cs[i] = c;
    sn[i] = p.inverse ? -s : s;
  }
  __syncthreads();
  constexpr int kPart = VW == 1 ? 1 : 4;  // pairs are a multiple of VW then
  struct alignas(4 * kPart) Part {
    float v[kPart];
  };
  const int turned = HALVES ? p.pairs / VW : (VW == 1 ? p.pairs : 2 * p.pairs / VW);
  const int rest = (p.head_dim - 2 * p.pairs) / VW;
  const int per_head = turned + rest, heads = p.t[0].heads + p.t[1].heads, per_token = per_head * heads;
  for (int i = threadIdx.x; i < nt * per_token; i += kThreads) {
    const int t = i / per_token, r = i - t * per_token;
    int h = r / per_head;
    const int e = r - h * per_head;
    const bool second = h >= p.t[0].heads;
    const RotaryTensor &q = p.t[second];
    if (second) h -= p.t[0].heads;
    long long b, n;
    token(t, b, n);
    const T *x = (const T *)q.x + b * q.xs[0] + n * q.xs[1] + h * q.xs[2];
    T *y = (T *)q.y + b * q.ys[0] + n * q.ys[1] + h * q.ys[2];
    const float *ct = cs + t * p.pairs, *st = sn + t * p.pairs;
    if (e >= turned) {
      const int d = 2 * p.pairs + (e - turned) * VW;
      float v[VW];
      Pack<T, VW>::load(x + d, v);
      Pack<T, VW>::store(y + d, v);
    } else if constexpr (HALVES) {
      const int j = e * VW;
      float u[VW], v[VW];
      Pack<T, VW>::load(x + j, u);
      Pack<T, VW>::load(x + p.pairs + j, v);
      float cj[VW], sj[VW];
#pragma unroll
      for (int k = 0; k < VW; k += kPart) {
        const Part c = *reinterpret_cast<const Part *>(ct + j + k), s = *reinterpret_cast<const Part *>(st + j + k);
#pragma unroll
        for (int l = 0; l < kPart; l++) cj[k + l] = c.v[l], sj[k + l] = s.v[l];
      }
#pragma unroll
      for (int k = 0; k < VW; k++) {
        const float c = cj[k], s = sj[k], a = u[k];
        u[k] = a * c - v[k] * s;
        v[k] = a * s + v[k] * c;
      }
      Pack<T, VW>::store(y + j, u);
      Pack<T, VW>::store(y + p.pairs + j, v);
    } else if constexpr (VW == 1) {
      float u[1], v[1];
      Pack<T, 1>::load(x + 2 * e, u);
      Pack<T, 1>::load(x + 2 * e + 1, v);
      const float c = ct[e], s = st[e], a = u[0];
      u[0] = a * c - v[0] * s;
      v[0] = a * s + v[0] * c;
      Pack<T, 1>::store(y + 2 * e, u);
      Pack<T, 1>::store(y + 2 * e + 1, v);
    } else {
      float u[VW];
      Pack<T, VW>::load(x + e * VW, u);
#pragma unroll
      for (int k = 0; k < VW / 2; k++) {
        const float c = ct[e * (VW / 2) + k], s = st[e * (VW / 2) + k], a = u[2 * k];
        u[2 * k] = a * c - u[2 * k + 1] * s;
        u[2 * k + 1] = a * s + u[2 * k + 1] * c;
      }
      Pack<T, VW>::store(y + e * VW, u);
    }
  }
}

template <typename T>
void launch(const RotaryParams &p, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  bool vec = p.head_dim % V == 0 && (p.interleaved ? 2 * p.pairs : p.pairs) % V == 0;
  for (const RotaryTensor &t : p.t) {
    if (!t.heads) continue;
    vec = vec && aligned16(t.x) && aligned16(t.y);
    for (int i = 0; i < 3; i++) vec = vec && t.xs[i] % V == 0 && t.ys[i] % V == 0;
  }
  const long long total = p.batch * p.tokens;
  int tb = kTrig / p.pairs < 8 ? kTrig / p.pairs : 8;  // 2 x 6272 tokens, 16 heads of 64: 13.2 us, with 16 tokens 15.0, with 4 16.3
  while (tb > 1 && (total + tb - 1) / tb < 2 * 148) tb = (tb + 1) / 2;
  const unsigned grid = (unsigned)((total + tb - 1) / tb);
  if (vec && p.interleaved) k_rotary<T, V, false><<<grid, kThreads, 0, st>>>(p, tb);
  else if (vec) k_rotary<T, V, true><<<grid, kThreads, 0, st>>>(p, tb);
  else if (p.interleaved) k_rotary<T, 1, false><<<grid, kThreads, 0, st>>>(p, tb);
  else k_rotary<T, 1, true><<<grid, kThreads, 0, st>>>(p, tb);
}

}  // namespace

cudaError_t rotary(int T, const RotaryParams &p, cudaStream_t st) {
  if (p.batch * p.tokens == 0 || p.t[0].heads + p.t[1].heads == 0) return cudaSuccess;
  if (T == 0) launch<float>(p, st);
  else launch<bf16>(p, st);
  return cudaGetLastError();
}

}  // namespace gpu
}  // namespace illumina
