// Attention and its backward pass on the CUDA cores: the path of 32-bit
// storage, and of bf16 tensors whose addresses or head sizes the tensor-core
// kernels (attention_tc.cu) do not take.
//
//   S = scale Q K', masked; P = softmax(S); O = P V; lse = log sum exp S
//   dV = P' dO; dP = dO V'; dS = P (dP - rowsum(dO O)); dQ = scale dS K; dK = scale dS' Q
//
// All three kernels have one shape: a tile of kFix rows stays in shared memory
// (queries; in the key pass keys), tiles of STR rows of the other side stream
// past it, products run as outer products from transposed tiles ([d][row]),
// 4 x STR/16 results a thread. The probabilities are never stored: the backward
// recomputes them from lse. It has two passes, one over key tiles for every
// query tile (dQ) and one over query tiles for every key tile (dK, dV, summed
// over the query heads that share a key head), so no result needs an atomic
// and the order of every sum is fixed. Where there are too few of them for
// every SM, the streamed tiles are shared out and the shares joined in order.
// Bound by the FP32 pipe and shared memory when there are tiles for every SM
// (3 heads of 104, batch of 4, 160 queries over 2134 keys, f32, forward: 121 us,
// 14 TFLOP/s), by latencies with one warp a scheduler when there are not: 2 x 4 heads of 32,
// 197 tokens, f32: forward 16 us, backward 35 us.
#include "attention.cuh"
#include "kernels.h"
#include <algorithm>
#include "token_common.cuh"

namespace illumina {
namespace gpu {
namespace {

using namespace tok;

constexpr int kThreads = 128;
constexpr int kFix = 32;
constexpr int kFixLd = kFix + 4;

// Rows [row0, row0 + ROWS) of one head, on their way into shared memory as
// floats, [d][row]; rows from `end` on and columns from head_dim on are zeros.
// All of a thread's loads are in flight together, and those of a streamed tile
// run while the one before it is computed: with one warp a scheduler, nothing
// else would hide them.
template <typename T, int ROWS, int DP>
struct Tile {
  static constexpr int kCount = ROWS * (DP / 4) / kThreads;
  float v[kCount][4];
  __device__ __forceinline__ void fetch(const AttnTensor &t, long long base, int row0, int end, int d, bool vec) {
    const T *p = (const T *)t.p + base;
#pragma unroll
    for (int k = 0; k < kCount; k++) {
      const int i = k * kThreads + threadIdx.x, r = row0 + i % ROWS, c = i / ROWS * 4;
#pragma unroll
      for (int j = 0; j < 4; j++) v[k][j] = 0;
      if (r < end) {
        const T *q = p + (long long)r * t.s[1] + c;
        if (vec && c + 4 <= d) {
          Pack<T, 4>::load(q, v[k]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (c + j < d) v[k][j] = to_f32(q[j]);
        }
      }
    }
  }
  __device__ __forceinline__ void put(float *dst) const {
#pragma unroll
    for (int k = 0; k < kCount; k++) {
      const int i = k * kThreads + threadIdx.x, r = i % ROWS, c = i / ROWS * 4;
#pragma unroll
      for (int j = 0; j < 4; j++) dst[(c + j) * (ROWS + 4) + r] = v[k][j];
    }
  }
};

// acc[i][j] += sum over d of a[d][4 ty + i] * b[d][n tx + j].
template <int STR, int DP>
__device__ __forceinline__ void outer(float (&acc)[4][STR / 16], const float *a, const float *b, int ty, int tx) {
  constexpr int N = STR / 16;
#pragma unroll 4
  for (int d = 0; d < DP; d++) {
    const float4 x = *reinterpret_cast<const float4 *>(a + d * kFixLd + 4 * ty);
    float y[N];
    if constexpr (N == 4) {
      const float4 w = *reinterpret_cast<const float4 *>(b + d * (STR + 4) + 4 * tx);
      y[0] = w.x, y[1] = w.y, y[2] = w.z, y[3] = w.w;
    } else {
      const float2 w = *reinterpret_cast<const float2 *>(b + d * (STR + 4) + 2 * tx);
      y[0] = w.x, y[1] = w.y;
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
      acc[0][j] += x.x * y[j];
      acc[1][j] += x.y * y[j];
      acc[2][j] += x.z * y[j];
      acc[3][j] += x.w * y[j];
    }
  }
}

// acc[i][c] += sum over n of p[n][4 ty + i] * b[tx + 16 c][n].
template <int STR, int DP>
__device__ __forceinline__ void inner(float (&acc)[4][DP / 16], const float *p, const float *b, int ty, int tx) {
  for (int n = 0; n < STR; n += 4) {
    float4 x[4];
#pragma unroll
    for (int k = 0; k < 4; k++) x[k] = *reinterpret_cast<const float4 *>(p + (n + k) * kFixLd + 4 * ty);
#pragma unroll
    for (int c = 0; c < DP / 16; c++) {
      const float4 y = *reinterpret_cast<const float4 *>(b + (tx + 16 * c) * (STR + 4) + n);
      acc[0][c] += x[0].x * y.x + x[1].x * y.y + x[2].x * y.z + x[3].x * y.w;
      acc[1][c] += x[0].y * y.x + x[1].y * y.y + x[2].y * y.z + x[3].y * y.w;
      acc[2][c] += x[0].z * y.x + x[1].z * y.y + x[2].z * y.z + x[3].z * y.w;
      acc[3][c] += x[0].w * y.x + x[1].w * y.y + x[2].w * y.z + x[3].w * y.w;
    }
  }
}

__device__ __forceinline__ float half_warp_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// The workspace of the backward begins with delta, rounded up to 16 bytes.
__host__ __device__ __forceinline__ long long delta_floats(const AttnParams &p) {
  return ((long long)p.batch * p.heads * p.q_tokens + 3) / 4 * 4;
}

// The sum a row's probabilities divide by, in the exponent; a row whose logits
// are all -inf (lse -inf) has probabilities of zero.
__device__ __forceinline__ float row_lse(float v) { return v == -INFINITY ? INFINITY : v; }

struct Vecs {
  bool q, k, v, dout;
};

// Writes rows of a fixed tile: out[row][tx + 16 c] = acc * factor[i].
template <typename T, int DP>
__device__ __forceinline__ void store_rows(const AttnTensor &t, long long base, int row0, int end, int d, int ty, int tx,
                                           const float (&acc)[4][DP / 16], const float (&f)[4]) {
  T *p = (T *)t.p + base;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = row0 + 4 * ty + i;
    if (r >= end) continue;
#pragma unroll
    for (int c = 0; c < DP / 16; c++)
      if (tx + 16 * c < d) from_f32(p[(long long)r * t.s[1] + tx + 16 * c], acc[i][c] * f[i]);
  }
}

// One CTA: kFix queries of one head, key tiles [split * per, ...) of `splits`
// shares. With splits > 1 the share's output and lse go to the workspace.
template <typename T, int DP, int STR>
__global__ void __launch_bounds__(kThreads) k_attn(const AttnParams p, int q_tiles, int splits, Vecs vec) {
  extern __shared__ __align__(16) float sm[];
  float *sq = sm, *sk = sq + DP * kFixLd, *sp = sk + DP * (STR + 4);
  cudaTriggerProgrammaticLaunchCompletion();  // the join of shares
  constexpr int N = STR / 16;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  long long id = blockIdx.x;
  const int split = (int)(id % splits);
  id /= splits;
  const int qt = q_tiles - 1 - (int)(id % q_tiles);  // long rows first
  id /= q_tiles;
  const int h = (int)(id % p.heads), n = (int)(id / p.heads);
  const AttnMask mask(p, n);
  const int row0 = qt * kFix, hk = h / (p.heads / p.kv_heads);
  int end[4], most = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) end[i] = mask.key_end(row0 + 4 * ty + i);
  most = mask.key_end(min(row0 + kFix, mask.q_len) - 1);
  if (row0 >= mask.q_len) most = 0;
  const int tiles = (most + STR - 1) / STR, per = (tiles + splits - 1) / splits;
  const int t0 = split * per, t1 = min(tiles, t0 + per);
  Tile<T, STR, DP> next;
  auto fetch_k = [&](int t) { next.fetch(p.k, n * p.k.s[0] + hk * p.k.s[2], t * STR, mask.k_len, p.head_dim, vec.k); };
  {
    Tile<T, kFix, DP> q;
    q.fetch(p.q, n * p.q.s[0] + h * p.q.s[2], row0, mask.q_len, p.head_dim, vec.q);
    if (t0 < t1) fetch_k(t0);
    q.put(sq);
  }
  float acc[4][DP / 16], top[4], sum[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    top[i] = -INFINITY, sum[i] = 0;
#pragma unroll
    for (int c = 0; c < DP / 16; c++) acc[i][c] = 0;
  }
  for (int t = t0; t < t1; t++) {
    __syncthreads();
    next.put(sk);
    __syncthreads();
    next.fetch(p.v, n * p.v.s[0] + hk * p.v.s[2], t * STR, mask.k_len, p.head_dim, vec.v);
    float s[4][N];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < N; j++) s[i][j] = 0;
    outer<STR, DP>(s, sq, sk, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float m = top[i];
#pragma unroll
      for (int j = 0; j < N; j++) {
        s[i][j] = t * STR + N * tx + j < end[i] ? s[i][j] * p.scale : -INFINITY;
        m = fmaxf(m, s[i][j]);
      }
      m = half_warp_max(m);
      const float base = m == -INFINITY ? 0.0f : m;  // a row that has seen no key yet
      const float f = expf(top[i] - base);
      top[i] = m;
      float add = 0;
#pragma unroll
      for (int j = 0; j < N; j++) {
        s[i][j] = expf(s[i][j] - base);
        add += s[i][j];
      }
      sum[i] = sum[i] * f + half_warp_sum(add);
#pragma unroll
      for (int c = 0; c < DP / 16; c++) acc[i][c] *= f;
    }
#pragma unroll
    for (int j = 0; j < N; j++)
      *reinterpret_cast<float4 *>(sp + (N * tx + j) * kFixLd + 4 * ty) =
          make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
    __syncthreads();
    next.put(sk);
    __syncthreads();
    if (t + 1 < t1) fetch_k(t + 1);
    inner<STR, DP>(acc, sp, sk, ty, tx);
  }
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    f[i] = sum[i] > 0 ? 1.0f / sum[i] : (sum[i] == 0 ? 0.0f : NAN);
    sum[i] = sum[i] == 0 ? -INFINITY : top[i] + logf(sum[i]);
  }
  const long long row = ((long long)n * p.heads + h) * p.q_tokens + row0;
  if (splits == 1) {
    store_rows<T, DP>(p.out, n * p.out.s[0] + h * p.out.s[2], row0, p.q_tokens, p.head_dim, ty, tx, acc, f);
    if (tx == 0)
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (row0 + 4 * ty + i < p.q_tokens) p.lse[row + 4 * ty + i] = sum[i];
    return;
  }
  const long long rows = (long long)p.batch * p.heads * p.q_tokens;
  AttnTensor part;
  part.p = p.ws + split * rows * p.head_dim;
  part.s[1] = p.head_dim;
  store_rows<float, DP>(part, (row - row0) * p.head_dim, row0, p.q_tokens, p.head_dim, ty, tx, acc, f);
  if (tx == 0)
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (row0 + 4 * ty + i < p.q_tokens) p.ws[splits * rows * p.head_dim + split * rows + row + 4 * ty + i] = sum[i];
}

// Joins the shares of a split forward: a warp takes one row.
//   lse = log sum_s exp(lse_s),  out = sum_s exp(lse_s - lse) out_s
constexpr int kMostSplits = 2 * 148;
template <typename T>
__global__ void __launch_bounds__(256) k_attn_join(const AttnParams p, int splits) {
  __shared__ float weights[8][kMostSplits];
  const long long rows = (long long)p.batch * p.heads * p.q_tokens;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);  // warp 0 of every CTA has one
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  float *w = weights[threadIdx.x >> 5];
  cudaGridDependencySynchronize();
  const float *sums = p.ws + splits * rows * p.head_dim + row;
  float top = -INFINITY;
  bool nan = false;
  for (int s = lane; s < splits; s += 32) {
    const float v = sums[s * rows];
    w[s] = v;
    top = fmaxf(top, v);
    nan = nan || v != v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (__any_sync(0xffffffffu, nan)) top = NAN;
  const float base = top == -INFINITY ? 0.0f : top;
  float total = 0;
  for (int s = lane; s < splits; s += 32) {
    w[s] = expf(w[s] - base);
    total += w[s];
  }
  total = warp_sum(total);
  __syncwarp();
  const float inv = total == 0 ? 0.0f : 1.0f / total;
  const long long i = row % p.q_tokens, bh = row / p.q_tokens;
  T *out = (T *)p.out.p + bh / p.heads * p.out.s[0] + i * p.out.s[1] + bh % p.heads * p.out.s[2];
  const float *part = p.ws + row * p.head_dim;
  const long long step = rows * p.head_dim;
  if (p.head_dim % 4 == 0) {
    // half a warp takes the even shares, half the odd ones, 16 bytes a lane
    for (int d = 0; d < p.head_dim; d += 64) {
      const int at = d + 4 * (lane & 15);
      float o[4] = {0, 0, 0, 0};
#pragma unroll 8
      for (int s = lane >> 4; s < splits; s += 2)  // a share without keys (weight 0) has no output
        if (w[s] != 0 && at < p.head_dim) {
          const float4 v = __ldcg(reinterpret_cast<const float4 *>(part + s * step + at));
          o[0] = fmaf(w[s], v.x, o[0]), o[1] = fmaf(w[s], v.y, o[1]);
          o[2] = fmaf(w[s], v.z, o[2]), o[3] = fmaf(w[s], v.w, o[3]);
        }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        o[k] = (o[k] + __shfl_xor_sync(0xffffffffu, o[k], 16)) * inv;
        if (lane < 16 && at < p.head_dim) from_f32(out[at + k], o[k]);
      }
    }
  } else {
    for (int d = lane; d < p.head_dim; d += 32) {
      float o = 0;
      for (int s = 0; s < splits; s++)
        if (w[s] != 0) o = fmaf(w[s], __ldcg(part + s * step + d), o);
      from_f32(out[d], o * inv);
    }
  }
  if (lane == 0) p.lse[row] = total == 0 ? -INFINITY : top + logf(total);
}

// dQ, and delta[row] = sum over d of dout * out on the way: one CTA takes kFix
// queries of one head past the keys they see.
template <typename T, int DP, int STR>
__global__ void __launch_bounds__(kThreads, 3) k_attn_dq(const AttnParams p, int q_tiles, Vecs vec) {
  extern __shared__ __align__(16) float sm[];
  float *sq = sm, *sg = sq + DP * kFixLd, *sk = sg + DP * kFixLd, *sv = sk + DP * (STR + 4),
        *sp = sv + DP * (STR + 4);
  constexpr int N = STR / 16;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  long long id = blockIdx.x;
  const int qt = q_tiles - 1 - (int)(id % q_tiles);
  id /= q_tiles;
  const int h = (int)(id % p.heads), n = (int)(id / p.heads);
  const AttnMask mask(p, n);
  const int row0 = qt * kFix, hk = h / (p.heads / p.kv_heads);
  const int most = row0 < mask.q_len ? mask.key_end(min(row0 + kFix, mask.q_len) - 1) : 0;
  Tile<T, STR, DP> k_next, v_next;
  auto fetch = [&](int k0) {
    k_next.fetch(p.k, n * p.k.s[0] + hk * p.k.s[2], k0, mask.k_len, p.head_dim, vec.k);
    v_next.fetch(p.v, n * p.v.s[0] + hk * p.v.s[2], k0, mask.k_len, p.head_dim, vec.v);
  };
  {
    Tile<T, kFix, DP> q, g;
    q.fetch(p.q, n * p.q.s[0] + h * p.q.s[2], row0, mask.q_len, p.head_dim, vec.q);
    g.fetch(p.dout, n * p.dout.s[0] + h * p.dout.s[2], row0, mask.q_len, p.head_dim, vec.dout);
    q.put(sq), g.put(sg);
  }
  if (most > 0) fetch(0);
  __syncthreads();
  float acc[4][DP / 16], lse[4], delta[4], f[4];
  int end[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = row0 + 4 * ty + i;
    const long long row = ((long long)n * p.heads + h) * p.q_tokens + r;
    end[i] = mask.key_end(r);
    lse[i] = end[i] ? row_lse(p.lse[row]) : 0.0f;
    float part = 0;
    if (r < mask.q_len) {
      const T *out = (const T *)p.out.p + n * p.out.s[0] + (long long)r * p.out.s[1] + h * p.out.s[2];
#pragma unroll
      for (int c = 0; c < DP / 16; c++)
        if (tx + 16 * c < p.head_dim) part += sg[(tx + 16 * c) * kFixLd + 4 * ty + i] * to_f32(out[tx + 16 * c]);
    }
    delta[i] = half_warp_sum(part);
    if (tx == 0 && r < mask.q_len) p.ws[row] = delta[i];
    f[i] = p.scale;
#pragma unroll
    for (int c = 0; c < DP / 16; c++) acc[i][c] = 0;
  }
  for (int k0 = 0; k0 < most; k0 += STR) {
    __syncthreads();
    k_next.put(sk), v_next.put(sv);
    __syncthreads();
    if (k0 + STR < most) fetch(k0 + STR);
    float s[4][N], g[4][N];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < N; j++) s[i][j] = g[i][j] = 0;
    outer<STR, DP>(s, sq, sk, ty, tx);
    outer<STR, DP>(g, sg, sv, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < N; j++)
        s[i][j] = k0 + N * tx + j < end[i] ? expf(s[i][j] * p.scale - lse[i]) * (g[i][j] - delta[i]) : 0.0f;
#pragma unroll
    for (int j = 0; j < N; j++)
      *reinterpret_cast<float4 *>(sp + (N * tx + j) * kFixLd + 4 * ty) =
          make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
    __syncthreads();
    inner<STR, DP>(acc, sp, sk, ty, tx);
  }
  store_rows<T, DP>(p.dq, n * p.dq.s[0] + h * p.dq.s[2], row0, p.q_tokens, p.head_dim, ty, tx, acc, f);
}

// dK, dV: one CTA takes kFix keys of one key head past the queries that see
// them, of every query head that shares it, or one of `splits` shares of these
// tiles, whose sums go to the workspace, [share][dK, dV][batch, key head, key].
template <typename T, int DP, int STR>
__global__ void __launch_bounds__(kThreads) k_attn_dkv(const AttnParams p, int k_tiles, int splits, Vecs vec) {
  extern __shared__ __align__(16) float sm[];
  float *sk = sm, *sv = sk + DP * kFixLd, *sq = sv + DP * kFixLd, *sg = sq + DP * (STR + 4),
        *sp = sg + DP * (STR + 4), *ss = sp + STR * kFixLd;
  constexpr int N = STR / 16;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  long long id = blockIdx.x;
  const int split = (int)(id % splits);
  id /= splits;
  const int kt = (int)(id % k_tiles);
  id /= k_tiles;
  const int hk = (int)(id % p.kv_heads), n = (int)(id / p.kv_heads), group = p.heads / p.kv_heads;
  const AttnMask mask(p, n);
  const int key0 = kt * kFix;
  {
    Tile<T, kFix, DP> k, v;
    k.fetch(p.k, n * p.k.s[0] + hk * p.k.s[2], key0, mask.k_len, p.head_dim, vec.k);
    v.fetch(p.v, n * p.v.s[0] + hk * p.v.s[2], key0, mask.k_len, p.head_dim, vec.v);
    k.put(sk), v.put(sv);
  }
  cudaGridDependencySynchronize();  // delta comes from the kernel of dQ
  float dk[4][DP / 16], dv[4][DP / 16];
  int begin[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int key = key0 + 4 * ty + i;
    begin[i] = key < mask.k_len ? mask.row_begin(key) : mask.q_len;
#pragma unroll
    for (int c = 0; c < DP / 16; c++) dk[i][c] = dv[i][c] = 0;
  }
  const int first = key0 < mask.k_len ? mask.row_begin(key0) / STR * STR : mask.q_len;
  Tile<T, STR, DP> q_next, g_next;
  float lse_next[N], delta_next[N];
  auto fetch = [&](int h, int q0) {
    q_next.fetch(p.q, n * p.q.s[0] + h * p.q.s[2], q0, mask.q_len, p.head_dim, vec.q);
    g_next.fetch(p.dout, n * p.dout.s[0] + h * p.dout.s[2], q0, mask.q_len, p.head_dim, vec.dout);
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int r = q0 + N * tx + j;
      const long long row = ((long long)n * p.heads + h) * p.q_tokens + r;
      lse_next[j] = r < mask.q_len ? row_lse(p.lse[row]) : 0.0f;
      delta_next[j] = r < mask.q_len ? p.ws[row] : 0.0f;
    }
  };
  const int tiles = max(0, mask.q_len - first + STR - 1) / STR, all = tiles * group;  // of one query head, of the group
  const int per = (all + splits - 1) / splits, it0 = min(all, split * per), it1 = min(all, it0 + per);
  int h = hk * group, q0 = first;
  if (it0 < it1) h += it0 / tiles, q0 += it0 % tiles * STR, fetch(h, q0);
  for (int it = it0; it < it1; it++) {
    __syncthreads();
    q_next.put(sq), g_next.put(sg);
    float lse[N], delta[N];
#pragma unroll
    for (int j = 0; j < N; j++) lse[j] = lse_next[j], delta[j] = delta_next[j];
    __syncthreads();
    const int now = q0;
    q0 += STR;
    if (q0 >= mask.q_len) h++, q0 = first;
    if (it + 1 < it1) fetch(h, q0);
    float s[4][N], g[4][N];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < N; j++) s[i][j] = g[i][j] = 0;
    outer<STR, DP>(s, sk, sq, ty, tx);
    outer<STR, DP>(g, sv, sg, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j < N; j++) {
        const int r = now + N * tx + j;
        const float pr = r >= begin[i] && r < mask.q_len ? expf(s[i][j] * p.scale - lse[j]) : 0.0f;
        s[i][j] = pr;
        g[i][j] = r >= begin[i] && r < mask.q_len ? pr * (g[i][j] - delta[j]) : 0.0f;
      }
#pragma unroll
    for (int j = 0; j < N; j++) {
      *reinterpret_cast<float4 *>(sp + (N * tx + j) * kFixLd + 4 * ty) =
          make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
      *reinterpret_cast<float4 *>(ss + (N * tx + j) * kFixLd + 4 * ty) =
          make_float4(g[0][j], g[1][j], g[2][j], g[3][j]);
    }
    __syncthreads();
    inner<STR, DP>(dv, sp, sg, ty, tx);
    inner<STR, DP>(dk, ss, sq, ty, tx);
  }
  const float one[4] = {1, 1, 1, 1}, sc[4] = {p.scale, p.scale, p.scale, p.scale};
  if (splits > 1) {
    const long long rows = (long long)p.batch * p.kv_heads * p.k_tokens;
    AttnTensor part;
    part.p = p.ws + delta_floats(p) + split * 2 * rows * p.head_dim;
    part.s[1] = p.head_dim;
    const long long base = ((long long)n * p.kv_heads + hk) * p.k_tokens * p.head_dim;
    store_rows<float, DP>(part, base, key0, p.k_tokens, p.head_dim, ty, tx, dk, one);
    store_rows<float, DP>(part, base + rows * p.head_dim, key0, p.k_tokens, p.head_dim, ty, tx, dv, one);
    return;
  }
  store_rows<T, DP>(p.dk, n * p.dk.s[0] + hk * p.dk.s[2], key0, p.k_tokens, p.head_dim, ty, tx, dk, sc);
  store_rows<T, DP>(p.dv, n * p.dv.s[0] + hk * p.dv.s[2], key0, p.k_tokens, p.head_dim, ty, tx, dv, one);
}

// Adds the shares of dK and dV in their order; a thread takes one element.
template <typename T>
__global__ void __launch_bounds__(256) k_attn_dkv_join(const AttnParams p, int splits) {
  cudaGridDependencySynchronize();
  const long long size = (long long)p.batch * p.kv_heads * p.k_tokens * p.head_dim;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= 2 * size) return;
  const float *part = p.ws + delta_floats(p) + i;
  float s = 0;
#pragma unroll 4
  for (int k = 0; k < splits; k++) s += __ldcg(part + k * 2 * size);
  const bool v = i >= size;
  const long long e = v ? i - size : i, row = e / p.head_dim, bh = row / p.k_tokens;
  const AttnTensor &t = v ? p.dv : p.dk;
  from_f32(((T *)t.p)[bh / p.kv_heads * t.s[0] + row % p.k_tokens * t.s[1] + bh % p.kv_heads * t.s[2] + e % p.head_dim],
           v ? s : s * p.scale);
}

// A tensor whose rows can be read four elements at a time.
template <typename T>
bool vec_rows(const AttnTensor &t) {
  return reinterpret_cast<uintptr_t>(t.p) % (4 * sizeof(T)) == 0 && t.s[0] % 4 == 0 && t.s[1] % 4 == 0 && t.s[2] % 4 == 0;
}

int ceil_div(long long a, int b) { return (int)((a + b - 1) / b); }

// `want` shares of `tiles`, without those that would be left empty.
int even_shares(int tiles, int want) { return ceil_div(tiles, ceil_div(tiles, want)); }

// Shares of the keys in the forward: as many as give every SM two CTAs, while a
// share keeps at least four key tiles (joining costs another launch).
template <int STR>
int simt_splits(const AttnParams &p) {
  const long long ctas = (long long)p.batch * p.heads * ceil_div(p.q_tokens, kFix);
  const int tiles = ceil_div(p.k_tokens, STR);
  if (ctas == 0 || ctas >= 148 || tiles < 8) return 1;
  return even_shares(tiles, (int)std::min<long long>(kMostSplits / ctas, tiles / 4));
}

// Shares of the query tiles that the keys of one CTA of dK and dV see: the same
// rule, with two tiles a share. 24 heads of 104 on 6, 324 tokens, f32: 139 us and
// 9 to join, against 345 whole; 4 on 1, 1400 tokens: 377 and 11, against 1386.
template <int STR>
int dkv_splits(const AttnParams &p) {
  const long long ctas = (long long)p.batch * p.kv_heads * ceil_div(p.k_tokens, kFix);
  if (ctas == 0 || ctas >= 148) return 1;
  const int tiles = ceil_div(p.q_tokens, STR) * (p.heads / p.kv_heads);
  const long long want = std::min<long long>(kMostSplits / ctas, tiles / 2);
  return want <= 1 ? 1 : even_shares(tiles, (int)want);
}

template <typename T, int DP, int STR>
cudaError_t run_simt(const AttnParams &p, bool bwd, cudaStream_t st) {
  const Vecs vec{vec_rows<T>(p.q), vec_rows<T>(p.k), vec_rows<T>(p.v), bwd && vec_rows<T>(p.dout)};
  const int q_tiles = ceil_div(p.q_tokens, kFix), k_tiles = ceil_div(p.k_tokens, kFix);
  const long long rows = (long long)p.batch * p.heads * p.q_tokens;
  constexpr size_t fix = sizeof(float) * DP * kFixLd, str = sizeof(float) * DP * (STR + 4),
                   prob = sizeof(float) * STR * kFixLd;
  cudaError_t e;
  if (!bwd) {
    const int splits = simt_splits<STR>(p);
    const size_t sm = fix + str + prob;
    if ((e = allow_smem<k_attn<T, DP, STR>>(sm)) != cudaSuccess) return e;
    const long long grid = (long long)p.batch * p.heads * q_tiles * splits;
    if (grid > 0) k_attn<T, DP, STR><<<(unsigned)grid, kThreads, sm, st>>>(p, q_tiles, splits, vec);
    if ((e = cudaGetLastError()) != cudaSuccess || splits == 1) return e;
    return launch_next(k_attn_join<T>, (rows + 7) / 8, 256, 0, st, p, splits);
  }
  if (rows > 0) {
    const size_t sm = 2 * fix + 2 * str + prob;
    if ((e = allow_smem<k_attn_dq<T, DP, STR>>(sm)) != cudaSuccess) return e;
    k_attn_dq<T, DP, STR><<<(unsigned)((long long)p.batch * p.heads * q_tiles), kThreads, sm, st>>>(p, q_tiles, vec);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
  }
  const int splits = dkv_splits<STR>(p);
  const long long grid = (long long)p.batch * p.kv_heads * k_tiles * splits;
  if (grid > 0) {
    const size_t sm = 2 * fix + 2 * str + 2 * prob;
    if ((e = allow_smem<k_attn_dkv<T, DP, STR>>(sm)) != cudaSuccess) return e;
    e = launch_next(k_attn_dkv<T, DP, STR>, grid, kThreads, sm, st, p, k_tiles, splits, vec);
    const long long elems = 2ll * p.batch * p.kv_heads * p.k_tokens * p.head_dim;
    if (e != cudaSuccess || splits == 1) return e;
    return launch_next(k_attn_dkv_join<T>, (elems + 255) / 256, 256, 0, st, p, splits);
  }
  return cudaSuccess;
}

template <typename T>
cudaError_t run_simt(const AttnParams &p, bool bwd, cudaStream_t st) {
  if (p.head_dim <= 32) return run_simt<T, 32, 64>(p, bwd, st);
  if (p.head_dim <= 64) return run_simt<T, 64, 64>(p, bwd, st);
  return run_simt<T, 128, 32>(p, bwd, st);
}

}  // namespace

// By sizes alone, so that it does not depend on which path the tensors'
// addresses and strides allow.
size_t attention_workspace(int T, const AttnParams &p, bool backward) {
  const size_t rows = (size_t)p.batch * p.heads * p.q_tokens;
  if (backward) {
    const size_t splits = p.head_dim <= 64 ? dkv_splits<64>(p) : dkv_splits<32>(p);
    const size_t parts = splits == 1 ? 0 : splits * 2 * p.batch * p.kv_heads * p.k_tokens * p.head_dim;
    return (delta_floats(p) + parts) * sizeof(float);
  }
  int splits = p.head_dim <= 64 ? simt_splits<64>(p) : simt_splits<32>(p);
  if (T == BF16) splits = std::max(splits, attention_tc_splits(p));
  return splits == 1 ? 0 : splits * rows * (p.head_dim + 1) * sizeof(float);
}

cudaError_t attention(int T, const AttnParams &p, cudaStream_t st) {
  if (T == F32) return run_simt<float>(p, false, st);
  if (!attention_tc_takes(p, false)) return run_simt<bf16>(p, false, st);
  const cudaError_t e = attention_tc(p, false, st);
  const int splits = attention_tc_splits(p);
  if (e != cudaSuccess || splits == 1) return e;
  const long long rows = (long long)p.batch * p.heads * p.q_tokens;
  return launch_next(k_attn_join<bf16>, (rows + 7) / 8, 256, 0, st, p, splits);
}

cudaError_t attention_backward(int T, const AttnParams &p, cudaStream_t st) {
  if (T == F32) return run_simt<float>(p, true, st);
  return attention_tc_takes(p, true) ? attention_tc(p, true, st) : run_simt<bf16>(p, true, st);
}

}  // namespace gpu
}  // namespace illumina
