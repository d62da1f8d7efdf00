// Layer norm over the last dimension, forward and backward.
//
//   y  = (x - mean) * rstd * w + b,  rstd = 1 / sqrt(var + eps)
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat)),  g = w * dy
//   dw = sum over rows of dy * xhat,  db = sum over rows of dy
//
// Bound by HBM: the forward reads x and writes y, the backward reads x and dy
// and writes dx. The forward keeps a row's elements in registers between the
// statistics (two passes over the registers: the mean, then the squared
// distances from it) and the output. One warp takes a row of up to 1024
// elements (no block barrier), a CTA of 256 threads one of up to 4096, and
// rows beyond that are re-read. In the backward a thread owns the same columns
// in every row it sees, so dw and db accumulate in registers; one partial row
// per CTA goes to the workspace and a second launch adds the partials in a
// fixed order, so that results do not depend on scheduling.
//
// Measured at 50176 rows of 704, bf16: forward 31 us (4.5 TB/s), backward with
// its second launch 44 us (4.9 TB/s, 67 us with the rows in registers); at
// 25088 rows of 1024, f32, backward 57 us (5.4 TB/s). A single frame of 196
// rows is a launch: 4 us on the GPU, 10 us a call.
#include <algorithm>

#include "token_common.cuh"
#include "token_ops.h"

namespace illumina {
namespace gpu {
namespace {

using namespace tok;

constexpr int kThreads = 256, kSms = 148;

// VW values of w or b; vectors when they are aligned like the columns (the
// caller checked).
template <int VW>
__device__ __forceinline__ void load_params(const float *p, float (&o)[VW]) {
  if constexpr (VW % 4 == 0) {
#pragma unroll
    for (int j = 0; j < VW; j += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4 *>(p + j));
      o[j] = v.x, o[j + 1] = v.y, o[j + 2] = v.z, o[j + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < VW; j++) o[j] = __ldg(p + j);
  }
}

template <int LANES>
__device__ __forceinline__ float row_sum(float v, float *red) {
  v = warp_sum(v);
  if constexpr (LANES > 32) {
    const int w = threadIdx.x >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[w] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < LANES / 32; i++) v += red[i];
  }
  return v;
}

// A thread group of LANES threads takes ROWS rows at once: their loads are in
// flight together, and w and b (from the L1) are read once for all of them.
template <typename T, int VW, int VPT, int LANES, int ROWS>
__global__ void __launch_bounds__(kThreads) k_norm(const T *__restrict__ x, long long xs, long long rows, int c,
                                                   const float *__restrict__ w, const float *__restrict__ b, float eps,
                                                   T *__restrict__ y, long long ys, float *mean, float *rstd) {
  __shared__ float red[kThreads / 32];
  const int lane = threadIdx.x % LANES;
  const long long row = ((long long)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES) * ROWS;
  if (row >= rows) return;  // uniform over the threads of a group
  float v[ROWS][VPT][VW];
#pragma unroll
  for (int k = 0; k < ROWS; k++)
#pragma unroll
    for (int i = 0; i < VPT; i++) {
      const int col = (i * LANES + lane) * VW;
      if (col < c && row + k < rows) {
        Pack<T, VW>::load(x + (row + k) * xs + col, v[k][i]);
      } else {
#pragma unroll
        for (int j = 0; j < VW; j++) v[k][i][j] = 0;
      }
    }
  const float inv = 1.0f / c;
  float r[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; k++) {
    float s = 0;
#pragma unroll
    for (int i = 0; i < VPT; i++)
#pragma unroll
      for (int j = 0; j < VW; j++) s += v[k][i][j];
    const float mu = row_sum<LANES>(s, red) * inv;
    float q = 0;
#pragma unroll
    for (int i = 0; i < VPT; i++) {
      const bool in = (i * LANES + lane) * VW < c;
#pragma unroll
      for (int j = 0; j < VW; j++) {
        v[k][i][j] -= mu;
        if (in) q += v[k][i][j] * v[k][i][j];
      }
    }
    r[k] = 1.0f / sqrtf(row_sum<LANES>(q, red) * inv + eps);
    if (lane == 0 && row + k < rows) {
      if (mean) mean[row + k] = mu;
      if (rstd) rstd[row + k] = r[k];
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    const int col = (i * LANES + lane) * VW;
    if (col >= c) break;
    float wv[VW], bv[VW];
#pragma unroll
    for (int j = 0; j < VW; j++) wv[j] = 1, bv[j] = 0;
    if (w) load_params<VW>(w + col, wv);
    if (b) load_params<VW>(b + col, bv);
#pragma unroll
    for (int k = 0; k < ROWS; k++) {
      if (row + k >= rows) break;
      float o[VW];
#pragma unroll
      for (int j = 0; j < VW; j++) o[j] = fmaf(v[k][i][j] * r[k], wv[j], bv[j]);
      Pack<T, VW>::store(y + (row + k) * ys + col, o);
    }
  }
}

// Rows longer than the registers hold: three readings of x.
template <typename T>
__global__ void __launch_bounds__(kThreads) k_norm_long(const T *__restrict__ x, long long xs, int c,
                                                        const float *__restrict__ w, const float *__restrict__ b,
                                                        float eps, T *__restrict__ y, long long ys, float *mean,
                                                        float *rstd) {
  __shared__ float red[kThreads / 32];
  const long long row = blockIdx.x;
  const T *xr = x + row * xs;
  float s = 0;
  for (int i = threadIdx.x; i < c; i += kThreads) s += to_f32(xr[i]);
  const float mu = row_sum<kThreads>(s, red) / c;
  float q = 0;
  for (int i = threadIdx.x; i < c; i += kThreads) {
    const float d = to_f32(xr[i]) - mu;
    q += d * d;
  }
  const float r = 1.0f / sqrtf(row_sum<kThreads>(q, red) / c + eps);
  if (threadIdx.x == 0) {
    if (mean) mean[row] = mu;
    if (rstd) rstd[row] = r;
  }
  for (int i = threadIdx.x; i < c; i += kThreads) {
    float o = (to_f32(xr[i]) - mu) * r;
    if (w) o *= w[i];
    if (b) o += b[i];
    from_f32(y[row * ys + i], o);
  }
}

// part: [gridDim.x][2][c], or null when neither dw nor db is wanted. PRE: the
// next row's loads are issued before this row's sums, where the registers
// allow it.
template <typename T, int VW, int VPT, int LANES, bool PRE>
__global__ void __launch_bounds__(kThreads) k_norm_bwd(const T *__restrict__ dy, long long dys,
                                                       const T *__restrict__ x, long long xs, long long rows, int c,
                                                       const float *__restrict__ w, const float *__restrict__ mean,
                                                       const float *__restrict__ rstd, T *__restrict__ dx,
                                                       long long dxs, float *__restrict__ part) {
  extern __shared__ float sums[];  // [rows per CTA][c] when a warp takes a row
  __shared__ float red[kThreads / 32];
  cudaTriggerProgrammaticLaunchCompletion();  // the sum over the partial rows
  constexpr int kRows = kThreads / LANES;
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  typedef typename RawPack<T, VW>::type Raw;
  float aw[VPT][VW], ab[VPT][VW];
#pragma unroll
  for (int i = 0; i < VPT; i++)
#pragma unroll
    for (int j = 0; j < VW; j++) aw[i][j] = ab[i][j] = 0;
  Raw rx[VPT], rg[VPT];
  float mu = 0, r = 0;
  const float inv = 1.0f / c;
  const long long step = (long long)gridDim.x * kRows;
  auto fetch = [&](long long row) {
    if (row >= rows) return;
    mu = __ldg(mean + row), r = __ldg(rstd + row);
#pragma unroll
    for (int i = 0; i < VPT; i++) {
      const int col = (i * LANES + lane) * VW;
      if (col < c) {
        rx[i] = *reinterpret_cast<const Raw *>(x + row * xs + col);
        rg[i] = *reinterpret_cast<const Raw *>(dy + row * dys + col);
      }
    }
  };
  const long long row0 = (long long)blockIdx.x * kRows + group;
  if (PRE) fetch(row0);
  for (long long row = row0; row < rows; row += step) {
    if (!PRE) fetch(row);
    float h[VPT][VW], g[VPT][VW];
    float s0 = 0, s1 = 0;
    const float rs = r;
#pragma unroll
    for (int i = 0; i < VPT; i++) {
      const int col = (i * LANES + lane) * VW;
      if (col >= c) break;
      RawPack<T, VW>::unpack(rx[i], h[i]);
      RawPack<T, VW>::unpack(rg[i], g[i]);
      float wv[VW];
#pragma unroll
      for (int j = 0; j < VW; j++) wv[j] = 1;
      if (w) load_params<VW>(w + col, wv);
#pragma unroll
      for (int j = 0; j < VW; j++) {
        h[i][j] = (h[i][j] - mu) * rs;
        aw[i][j] = fmaf(g[i][j], h[i][j], aw[i][j]);
        ab[i][j] += g[i][j];
        g[i][j] *= wv[j];
        s0 += g[i][j];
        s1 = fmaf(g[i][j], h[i][j], s1);
      }
    }
    if (PRE) fetch(row + step);
    s0 = row_sum<LANES>(s0, red) * inv;
    s1 = row_sum<LANES>(s1, red) * inv;
    if (dx) {
      T *dr = dx + row * dxs;
#pragma unroll
      for (int i = 0; i < VPT; i++) {
        const int col = (i * LANES + lane) * VW;
        if (col >= c) break;
        float o[VW];
#pragma unroll
        for (int j = 0; j < VW; j++) o[j] = rs * (g[i][j] - s0 - h[i][j] * s1);
        Pack<T, VW>::store(dr + col, o);
      }
    }
  }
  if (!part) return;
  float *out = part + (size_t)blockIdx.x * 2 * c;
  if constexpr (LANES == kThreads) {
#pragma unroll
    for (int i = 0; i < VPT; i++) {
      const int col = (i * LANES + lane) * VW;
      if (col >= c) break;
#pragma unroll
      for (int j = 0; j < VW; j++) out[col + j] = aw[i][j], out[c + col + j] = ab[i][j];
    }
  } else {
    for (int which = 0; which < 2; which++) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VPT; i++) {
        const int col = (i * LANES + lane) * VW;
        if (col >= c) break;
#pragma unroll
        for (int j = 0; j < VW; j++) sums[group * c + col + j] = which ? ab[i][j] : aw[i][j];
      }
      __syncthreads();
      for (int i = threadIdx.x; i < c; i += kThreads) {
        float t = 0;
#pragma unroll
        for (int k = 0; k < kRows; k++) t += sums[k * c + i];
        out[which * c + i] = t;
      }
    }
  }
}

__device__ __forceinline__ void copy_async(uint4 *to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// 16 bytes of a row as pairs.
__device__ __forceinline__ void unpack16(uint4 u, float2 (&o)[2], float) {
  o[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
  o[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
}
__device__ __forceinline__ void unpack16(uint4 u, float2 (&o)[4], bf16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int k = 0; k < 4; k++) o[k] = make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
}

// The ring of a thread group that has VPT chunks of 16 bytes of a row a
// thread: CTAs an SM, bytes of a stage, stages (by the shared memory that the
// CTAs and w leave, at most 8 small ones or 4 large ones). 704 columns of bf16
// have registers for three CTAs, but two with a stage more are faster (44 us
// at 50176 rows, against 62).
template <typename T, int VPT, int LANES>
struct BwdRing {
  static constexpr int kVec = 16 / sizeof(T), kElems = VPT * kVec;
  static constexpr int kCtas = kElems <= 8 ? 4 : kElems <= 24 || sizeof(T) == 2 ? 2 : 1;
  static constexpr int kStage = kThreads * VPT * 16 * 2, kWeights = LANES * kElems * 4;
  static constexpr int kFit = ((228 << 10) / kCtas - 1024 - (LANES == 32 ? 0 : 32) - kWeights) / kStage;
  static constexpr int kMost = kStage <= 8 << 10 ? 8 : 4, kDepth = kFit < kMost ? kFit : kMost;
};

// The same for rows of whole, aligned 16-byte chunks. x and dy come through a
// ring of rows in shared memory, where a thread copies the chunks that it uses
// (so that only it waits for them), and are read twice there, for the sums and
// for dx: with nothing but the sums of the columns in registers, up to three
// times the warps fit, and more rows are under way. w is in shared memory too:
// the ring leaves the L1 too small to keep it. Copies of 8 bytes, which pass
// through the L1, were no faster than the loads above.
template <typename T, int VPT, int LANES>
__global__ void __launch_bounds__(kThreads, BwdRing<T, VPT, LANES>::kCtas)
    k_norm_bwd_ring(const T *__restrict__ dy, long long dys, const T *__restrict__ x, long long xs, long long rows, int c,
                    const float *__restrict__ w, const float *__restrict__ mean, const float *__restrict__ rstd,
                    T *__restrict__ dx, long long dxs, float *__restrict__ part) {
  typedef BwdRing<T, VPT, LANES> Ring;
  constexpr int V = Ring::kVec, kRows = kThreads / LANES, kDepth = Ring::kDepth;
  extern __shared__ uint4 smem[];  // the ring and w; after the rows [rows per CTA][c] sums when a warp takes a row
  float *red = nullptr;
  if constexpr (LANES > 32) {
    __shared__ float s_red[kThreads / 32];
    red = s_red;
  }
  cudaTriggerProgrammaticLaunchCompletion();  // the sum over the partial rows
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  uint4 *ring = smem + threadIdx.x;  // [stage][x, dy][VPT][thread]
  float *weights = reinterpret_cast<float *>(smem + kDepth * (Ring::kStage / 16));  // [V / 4][chunk][4]
  float2 aw[VPT][V / 2], ab[VPT][V / 2];
#pragma unroll
  for (int i = 0; i < VPT; i++)
#pragma unroll
    for (int k = 0; k < V / 2; k++) aw[i][k] = ab[i][k] = make_float2(0, 0);
  const float inv = 1.0f / c;
  const long long step = (long long)gridDim.x * kRows, row0 = (long long)blockIdx.x * kRows + group;
  auto fetch = [&](long long row, int stage) {
    if (row < rows) {
      uint4 *to = ring + stage * 2 * VPT * kThreads;
#pragma unroll
      for (int i = 0; i < VPT; i++) {
        const int col = (i * LANES + lane) * V;
        if (col < c) {
          copy_async(to + i * kThreads, x + row * xs + col);
          copy_async(to + (VPT + i) * kThreads, dy + row * dys + col);
        }
      }
    }
    copies_commit();
  };
  float mu = 0, r = 0;
  auto moments = [&](long long row) {
    if (row < rows) mu = __ldg(mean + row), r = __ldg(rstd + row);
  };
  moments(row0);
  for (int i = 0; i < kDepth; i++) fetch(row0 + i * step, i);
  for (int i = threadIdx.x; i < c; i += kThreads)
    weights[((i % V) / 4 * LANES * VPT + i / V) * 4 + i % 4] = w ? w[i] : 1.0f;
  __syncthreads();
  int stage = 0;
  for (long long row = row0; row < rows; row += step) {
    const uint4 *from = ring + stage * 2 * VPT * kThreads;
    const float2 rs = make_float2(r, r), away = make_float2(-mu, -mu);
    // xhat, dy and w of chunk i
    auto take = [&](int i, float2 (&h)[V / 2], float2 (&g)[V / 2], float2 (&wv)[V / 2]) {
      unpack16(from[i * kThreads], h, T());
      unpack16(from[(VPT + i) * kThreads], g, T());
#pragma unroll
      for (int k = 0; k < V / 2; k++) h[k] = __fmul2_rn(__fadd2_rn(h[k], away), rs);
#pragma unroll
      for (int k = 0; k < V / 4; k++) {
        const float4 v = *reinterpret_cast<const float4 *>(weights + (k * LANES * VPT + i * LANES + lane) * 4);
        wv[2 * k] = make_float2(v.x, v.y), wv[2 * k + 1] = make_float2(v.z, v.w);
      }
    };
    moments(row + step);
    copies_wait<kDepth - 1>();
    float2 s0 = make_float2(0, 0), s1 = s0;
#pragma unroll
    for (int i = 0; i < VPT; i++) {
      if ((i * LANES + lane) * V >= c) break;
      float2 h[V / 2], g[V / 2], wv[V / 2];
      take(i, h, g, wv);
#pragma unroll
      for (int k = 0; k < V / 2; k++) {
        aw[i][k] = __ffma2_rn(g[k], h[k], aw[i][k]);
        ab[i][k] = __fadd2_rn(ab[i][k], g[k]);
        g[k] = __fmul2_rn(g[k], wv[k]);
        s0 = __fadd2_rn(s0, g[k]);
        s1 = __ffma2_rn(g[k], h[k], s1);
      }
    }
    const float m0 = row_sum<LANES>(s0.x + s0.y, red) * inv, m1 = row_sum<LANES>(s1.x + s1.y, red) * inv;
    if (dx) {
      const float2 n0 = make_float2(-m0, -m0), n1 = make_float2(-m1, -m1);
      T *dr = dx + row * dxs;
#pragma unroll
      for (int i = 0; i < VPT; i++) {
        const int col = (i * LANES + lane) * V;
        if (col >= c) break;
        float2 h[V / 2], g[V / 2], wv[V / 2];
        take(i, h, g, wv);
        float o[V];
#pragma unroll
        for (int k = 0; k < V / 2; k++) {
          const float2 v = __fmul2_rn(rs, __ffma2_rn(h[k], n1, __ffma2_rn(g[k], wv[k], n0)));
          o[2 * k] = v.x, o[2 * k + 1] = v.y;
        }
        Pack<T, V>::store(dr + col, o);
      }
    }
    fetch(row + kDepth * step, stage);
    stage = stage + 1 == kDepth ? 0 : stage + 1;
  }
  if (!part) return;
  float *out = part + (size_t)blockIdx.x * 2 * c, *sums = reinterpret_cast<float *>(smem);
  for (int which = 0; which < 2; which++) {
    float *to = LANES == kThreads ? out + which * c : sums + group * c;
    if (LANES < kThreads) __syncthreads();  // the ring, or the sums of dw, have been read
#pragma unroll
    for (int i = 0; i < VPT; i++) {
      const int col = (i * LANES + lane) * V;
      if (col >= c) break;
      const float2 *a = which ? ab[i] : aw[i];
#pragma unroll
      for (int k = 0; k < V / 2; k += 2)
        *reinterpret_cast<float4 *>(to + col + 2 * k) = make_float4(a[k].x, a[k].y, a[k + 1].x, a[k + 1].y);
    }
    if constexpr (LANES < kThreads) {
      __syncthreads();
      for (int i = threadIdx.x; i < c; i += kThreads) {
        float t = 0;
#pragma unroll
        for (int k = 0; k < kRows; k++) t += sums[k * c + i];
        out[which * c + i] = t;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_norm_bwd_long(const T *__restrict__ dy, long long dys,
                                                            const T *__restrict__ x, long long xs, long long rows,
                                                            int c, const float *__restrict__ w,
                                                            const float *__restrict__ mean,
                                                            const float *__restrict__ rstd, T *__restrict__ dx,
                                                            long long dxs, float *__restrict__ part) {
  __shared__ float red[kThreads / 32];
  cudaTriggerProgrammaticLaunchCompletion();  // the sum over the partial rows
  float *out = part ? part + (size_t)blockIdx.x * 2 * c : nullptr;
  if (out)
    for (int i = threadIdx.x; i < 2 * c; i += kThreads) out[i] = 0;  // each thread adds to its own columns only
  __syncthreads();
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + row * xs, *gr = dy + row * dys;
    const float mu = mean[row], r = rstd[row];
    float s0 = 0, s1 = 0;
    for (int i = threadIdx.x; i < c; i += kThreads) {
      const float h = (to_f32(xr[i]) - mu) * r, d = to_f32(gr[i]);
      if (out) out[i] += d * h, out[c + i] += d;
      const float g = w ? d * w[i] : d;
      s0 += g;
      s1 += g * h;
    }
    s0 = row_sum<kThreads>(s0, red) / c;
    s1 = row_sum<kThreads>(s1, red) / c;
    if (dx)
      for (int i = threadIdx.x; i < c; i += kThreads) {
        const float h = (to_f32(xr[i]) - mu) * r, d = to_f32(gr[i]);
        const float g = w ? d * w[i] : d;
        from_f32(dx[row * dxs + i], r * (g - s0 - h * s1));
      }
  }
}

// Column sums of part ([n][2c]) in a fixed order: a CTA takes 8 columns, its 32
// groups of 8 threads every 32nd row, then the groups' sums are added. The rows
// are still being written when the kernel starts: not read-only memory, and
// read past the L1.
__global__ void __launch_bounds__(256) k_norm_reduce(const float *part, int n, int c, float *dw, float *db) {
  __shared__ float s[8][33];
  const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
  const int col = blockIdx.x * 8 + tx;
  float t = 0;
  cudaGridDependencySynchronize();
  if (col < 2 * c) {
#pragma unroll 4
    for (int i = ty; i < n; i += 32) t += __ldcg(part + (size_t)i * 2 * c + col);
  }
  s[tx][ty] = t;
  __syncthreads();
  const int o = blockIdx.x * 8 + (threadIdx.x >> 5);
  t = warp_sum(s[threadIdx.x >> 5][threadIdx.x & 31]);
  if ((threadIdx.x & 31) == 0 && o < 2 * c) {
    if (o < c) {
      if (dw) dw[o] = t;
    } else if (db) {
      db[o - c] = t;
    }
  }
}

struct NormArgs {
  const void *x, *dy;
  long long xs, dys, rows;
  int c;
  const float *w, *b;
  float eps;
  void *y;
  long long ys;
  float *mean, *rstd;
  float *part;
  int blocks;
  cudaStream_t st;
};

template <typename T, int VW, int VPT, int LANES>
void launch(NormArgs &a, bool bwd) {
  constexpr int kRows = kThreads / LANES;
  const T *x = (const T *)a.x;
  if (!bwd) {
    // two rows a warp once there are enough rows to fill the GPU with half the
    // warps, and registers for both
    constexpr int kTwo = LANES == 32 && VW * VPT <= 24 ? 2 : 1;
    if (kTwo == 2 && a.rows >= 148 * 64 * 2)
      k_norm<T, VW, VPT, LANES, kTwo><<<(unsigned)((a.rows + 2 * kRows - 1) / (2 * kRows)), kThreads, 0, a.st>>>(
          x, a.xs, a.rows, a.c, a.w, a.b, a.eps, (T *)a.y, a.ys, a.mean, a.rstd);
    else
      k_norm<T, VW, VPT, LANES, 1><<<(unsigned)((a.rows + kRows - 1) / kRows), kThreads, 0, a.st>>>(
          x, a.xs, a.rows, a.c, a.w, a.b, a.eps, (T *)a.y, a.ys, a.mean, a.rstd);
  } else if constexpr (VW == 8) {  // never: such rows go through the ring
  } else if constexpr (VW == 1 || sizeof(T) == 2 || VPT == 1) {  // longer aligned rows of floats go through the ring
    constexpr bool kPre = VW * VPT * sizeof(T) <= 64;
    const size_t sm = LANES == kThreads || !a.part ? 0 : (size_t)kRows * a.c * sizeof(float);
    a.blocks = std::min(a.blocks, kSms * (VPT <= 8 ? 4 : VPT <= 16 ? 2 : 1));
    k_norm_bwd<T, VW, VPT, LANES, kPre><<<a.blocks, kThreads, sm, a.st>>>(
        (const T *)a.dy, a.dys, x, a.xs, a.rows, a.c, a.w, a.mean, a.rstd, (T *)a.y, a.ys, a.part);
  }
}

template <typename T, int VPT, int LANES>
void launch_ring(NormArgs &a) {
  typedef BwdRing<T, VPT, LANES> Ring;
  constexpr size_t ring = (size_t)Ring::kDepth * Ring::kStage + Ring::kWeights,
                   out = LANES == 32 ? kThreads * Ring::kElems * sizeof(float) : 0, sm = ring > out ? ring : out;
  if (allow_smem<k_norm_bwd_ring<T, VPT, LANES>>(sm) != cudaSuccess) return;  // the error stays for the caller
  a.blocks = std::min(a.blocks, kSms * Ring::kCtas);
  k_norm_bwd_ring<T, VPT, LANES><<<a.blocks, kThreads, sm, a.st>>>((const T *)a.dy, a.dys, (const T *)a.x, a.xs, a.rows, a.c,
                                                                 a.w, a.mean, a.rstd, (T *)a.y, a.ys, a.part);
}
template <typename T>
void pick_ring(NormArgs &a) {
  constexpr int u = sizeof(T) / 2;  // chunks of 8 columns
  if (a.c <= 256) launch_ring<T, u, 32>(a);
  else if (a.c <= 384 && u == 2) launch_ring<T, 3, 32>(a);
  else if (a.c <= 512) launch_ring<T, 2 * u, 32>(a);
  else if (a.c <= 768) launch_ring<T, 3 * u, 32>(a);
  else if (a.c <= 1024) launch_ring<T, 4 * u, 32>(a);
  else if (a.c <= 2048) launch_ring<T, u, 256>(a);
  else launch_ring<T, 2 * u, 256>(a);
}

// Smallest register tile that holds a row of c columns.
template <typename T, int VW>
bool pick(NormArgs &a, bool bwd) {
  constexpr int u = 4 / VW;  // a thread holds at least 4 columns
  const int quads = (a.c + 3) / 4;  // groups of 4 columns
  if (quads <= 32) launch<T, VW, u, 32>(a, bwd);
  else if (quads <= 64) launch<T, VW, 2 * u, 32>(a, bwd);
  else if (quads <= 96) launch<T, VW, 3 * u, 32>(a, bwd);
  else if (quads <= 128) launch<T, VW, 4 * u, 32>(a, bwd);
  else if (quads <= 192) launch<T, VW, 6 * u, 32>(a, bwd);
  else if (quads <= 256) launch<T, VW, 8 * u, 32>(a, bwd);
  else if (quads <= 512) launch<T, VW, 2 * u, 256>(a, bwd);
  else if (quads <= 1024) launch<T, VW, 4 * u, 256>(a, bwd);
  else return false;
  return true;
}

// The forward of bf16 rows in 16-byte chunks, where a warp takes two rows
// (704 columns 31 us at 50176 rows, 36 in 8-byte chunks; one row of 1024 a
// warp 25 us at 25088 rows, 24.6 in 8-byte chunks).
void pick8(NormArgs &a) {
  if (a.c <= 256) launch<bf16, 8, 1, 32>(a, false);
  else if (a.c <= 512) launch<bf16, 8, 2, 32>(a, false);
  else launch<bf16, 8, 3, 32>(a, false);
}

template <typename T>
void dispatch(NormArgs &a, bool bwd) {
  // four columns at a time: 8 or 16 bytes of T, 16 bytes of w and b
  auto fits = [](const void *p, long long stride) {
    return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0 && stride % 4 == 0;
  };
  const bool vec = a.c % 4 == 0 && fits(a.x, a.xs) && fits(a.y, a.ys) && (!bwd || fits(a.dy, a.dys)) && aligned16(a.w) &&
                   aligned16(a.b);
  auto chunks = [](const void *p, long long stride) { return aligned16(p) && stride * sizeof(T) % 16 == 0; };
  // half the ring's threads would idle up to 128 columns of bf16 (17 us at 50176 rows, 22 through the ring)
  if (bwd && a.c > 128 && a.c <= 4096 && a.c * sizeof(T) % 16 == 0 && chunks(a.x, a.xs) && chunks(a.y, a.ys) && chunks(a.dy, a.dys))
    return pick_ring<T>(a);
  if constexpr (sizeof(T) == 2)
    if (!bwd && a.c > 128 && a.c <= 768 && a.c % 8 == 0 && chunks(a.x, a.xs) && chunks(a.y, a.ys) && aligned16(a.w) &&
        aligned16(a.b))
      return pick8(a);
  if (vec ? pick<T, 4>(a, bwd) : pick<T, 1>(a, bwd)) return;
  if (!bwd)
    k_norm_long<T><<<(unsigned)a.rows, kThreads, 0, a.st>>>((const T *)a.x, a.xs, a.c, a.w, a.b, a.eps, (T *)a.y, a.ys,
                                                            a.mean, a.rstd);
  else
    k_norm_bwd_long<T><<<a.blocks, kThreads, 0, a.st>>>((const T *)a.dy, a.dys, (const T *)a.x, a.xs, a.rows, a.c, a.w,
                                                        a.mean, a.rstd, (T *)a.y, a.ys, a.part);
}

}  // namespace

cudaError_t layer_norm(int T, const void *x, long long xs, long long rows, int c, const float *w, const float *b,
                       float eps, void *y, long long ys, float *mean, float *rstd, cudaStream_t st) {
  if (rows == 0) return cudaSuccess;
  NormArgs a{};
  a.x = x, a.xs = xs, a.rows = rows, a.c = c, a.w = w, a.b = b, a.eps = eps, a.y = y, a.ys = ys, a.mean = mean;
  a.rstd = rstd, a.st = st;
  if (T == 0) dispatch<float>(a, false);
  else dispatch<bf16>(a, false);
  return cudaGetLastError();
}

int layer_norm_blocks(long long rows, int c) {
  // Every CTA leaves one partial row: at most as many as are resident at once,
  // which the launch lowers to what its kernel's registers allow.
  const long long per = c <= 1024 ? kThreads / 32 : 1;
  const long long want = (rows + per - 1) / per, most = kSms * (c <= 256 ? 4 : 2);
  return (int)(want < most ? want : most);
}

cudaError_t layer_norm_backward(int T, const void *dy, long long dys, const void *x, long long xs, long long rows,
                                int c, const float *w, const float *mean, const float *rstd, void *dx, long long dxs,
                                float *dw, float *db, float *ws, cudaStream_t st) {
  NormArgs a{};
  a.dy = dy, a.dys = dys, a.x = x, a.xs = xs, a.rows = rows, a.c = c, a.w = w, a.mean = const_cast<float *>(mean);
  a.rstd = const_cast<float *>(rstd), a.y = dx, a.ys = dxs, a.st = st;
  a.part = dw || db ? ws : nullptr;
  a.blocks = layer_norm_blocks(rows, c);
  if (rows > 0) {
    if (T == 0) dispatch<float>(a, true);
    else dispatch<bf16>(a, true);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !(dw || db)) return e;
  return launch_next(k_norm_reduce, (2 * c + 7) / 8, 256, 0, st, ws, a.blocks, c, dw, db);
}

}  // namespace gpu
}  // namespace illumina
