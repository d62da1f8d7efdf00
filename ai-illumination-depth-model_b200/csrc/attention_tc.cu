// Attention and its backward pass on the tensor cores, for bf16 storage.
//
//   S = scale Q K', masked; P = softmax(S); O = P V; lse = log sum exp S
//   dV = P' dO; dP = dO V'; dS = P (dP - rowsum(dO O)); dQ = scale dS K; dK = scale dS' Q
//
// Every product is a tcgen05.mma of 128 rows with its accumulator in TMEM.
// Operand tiles come by TMA into 128-byte swizzled images (128 rows x 64
// columns; two for head sizes over 64, the columns past head_dim filled with
// zeros by the copy) and serve both as K-major and, transposed by the matrix
// descriptor, as MN-major operands. Probabilities and their gradients go from
// registers to TMEM as bf16 and are the A operand of the following product
// from there, so that they never pass through shared memory.
//
// A query tile holds the G query heads that share a key head for 128 / G
// consecutive tokens (row r: token r / G, head r % G): key and value tiles are
// read once for all of them, and a single token's heads fill one tile.
//
// Warps: two or four warpgroups compute (one TMEM lane, that is one row, a
// thread, so a row's maximum and sum need no shuffles), one thread issues the
// copies, and one for each of the two pipelines (query tiles, or halves of the
// streamed tile) its products: a product's issue takes as long as the tensor
// cores take for it, and while one thread waits for its warpgroups the other's
// products run. All waits are on mbarriers and bounded.
//
// Rows of padding inside the last tile may hold NaN: where such rows are a
// contraction index (V; K in dQ; Q and dO in dK, dV), 0 * NaN would spoil the
// sum, so another warp clears them in shared memory first.
//
// Roundings to bf16: the operands P (against the running maximum, so at most
// 2^8) and dS, which a 16-bit product needs, and the results. The row sums are
// taken over P before it is rounded, delta over the rounded O that the forward
// stored. Together they put dQ and dK at 2.5e-3 of their norm, where the
// rounding of the result alone gives 1.7e-3. Everything else is 32 bits.
//
// Bound, with the tensor cores and the exponential unit each about half busy,
// by the chain S -> exponentials -> P -> product of every tile, whose waits and
// instruction issue two pipelines only partly cover. Measured (bf16; arithmetic
// of the visible pairs, 4 T^2 D forward, 10 backward, against 1617 TFLOP/s of a
// plain product):
//   12 heads of 64, 6272 tokens, frame-causal: forward 116 us (0.54 PFLOP/s),
//     dQ 122, dK and dV 156 us (0.56 together)
//   16 heads of 128 on 4, batch of 4 padded to 2500, causal: 92, 137, 167 us
//   6 heads of 64, batch of 8, 784 tokens: 35, 39, 46 us
//   one frame of 196 tokens over 12544 keys, 12 heads on 4: 26 us + 7 to join
//     11 shares
// The forward spills a little (36 bytes stored and 172 loaded a thread at head
// size 64, 76 and 176 at 128).
#include "attention.cuh"
#include "kernels.h"
#include "tc_common.cuh"
#include "token_common.cuh"

#include <cudaTypedefs.h>

#include <algorithm>

namespace illumina {
namespace gpu {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

namespace {

using namespace tcx;
using tok::allow_smem;
using tok::bf16;

// Compute warpgroups, then one of single warps: copies, the products of one
// pipeline, those of the other, clearing of padding (and row sums).
constexpr int kFwdGroups = 2, kBwdGroups = 4;
constexpr int threads_of(int groups) { return 128 * (groups + 1); }
struct Roles {
  int copy, product, second, clear;
  __host__ __device__ constexpr explicit Roles(int groups)
      : copy(4 * groups), product(4 * groups + 1), second(4 * groups + 2), clear(4 * groups + 3) {}
};
constexpr uint32_t kImage = 128 * 128;  // 128 rows x 64 bf16 columns
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct TcArgs {
  int group, tpt;        // query heads a key head has; tokens of a query tile
  int q_tiles, k_tiles;  // per (batch, key head)
  int splits;
  int n16;               // head_dim rounded up to the MMA's 16 columns
  long long wait;        // cycles a wait may take
  int qh, qb, kh, kb, vh, vb, gh, gb;  // 0: that dimension of the tensor is broadcast (stride 0)
};

__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(a));
}
__device__ __forceinline__ void tmem_ld16(uint32_t a, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(a));
}
__device__ __forceinline__ void tmem_st16(uint32_t a, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t *r) {
  tmem_st16(a, r);
  tmem_st16(a + 16, r + 16);
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Operand descriptors of an image, as the low word (address and stride of the
// next 64 columns' image; steps within a tile are added to it) and the high
// word, which all share (8-row groups 1024 bytes apart, version 1, 128-byte
// swizzle). K-major: K is the 64 columns. MN-major: the columns are the N
// index, 8-row groups are steps of K.
constexpr uint32_t kDescHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t addr) { return ((addr >> 4) & 0x3FFF) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t addr) { return ((addr >> 4) & 0x3FFF) | ((kImage >> 4) << 16); }
constexpr uint32_t kBMnMajor = 1u << 16;

// Products are issued by one thread, chosen by elect.sync: behind its answer
// the compiler keeps descriptors in uniform registers. An issue then takes 31
// cycles (64-column accumulator, operand in TMEM: the tensor core's own rate),
// 47 (64 columns from shared memory, whose bandwidth bounds it) or 63 (128
// columns); behind a comparison of the thread index 44, 48 and 63, and with
// the instruction predicated in converged code 67 to 72.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}
// ACC: 1 adds to the accumulator, 0 overwrites it, -1 as `acc` says.
template <int ACC>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc = 0) {
  if constexpr (ACC >= 0)
    asm volatile(
        "{\n .reg .b64 da, db;\n mov.b64 da, {%1, %4};\n mov.b64 db, {%2, %4};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, %5;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "n"(kDescHigh), "n"(ACC)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 da, db;\n mov.b64 da, {%1, %4};\n mov.b64 db, {%2, %4};\n setp.ne.b32 p, %5, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "n"(kDescHigh), "r"(acc)
        : "memory");
}
template <int ACC>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc = 0) {
  if constexpr (ACC >= 0)
    asm volatile(
        "{\n .reg .b64 db;\n mov.b64 db, {%2, %4};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, %5;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "n"(kDescHigh), "n"(ACC)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 db;\n mov.b64 db, {%2, %4};\n setp.ne.b32 p, %5, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "n"(kDescHigh), "r"(acc)
        : "memory");
}
// d[128][n] = a(image rows)[128][nk * 16] * b(image rows)[n][nk * 16]', with
// a and b K-major descriptors of the tiles.
template <int DP>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t b, int nk, uint32_t idesc) {
  mma_ss<0>(d, a, b, idesc);
#pragma unroll
  for (int k = 1; k < DP / 16; k++) {
    constexpr uint32_t image = kImage >> 4;
    const uint32_t o = (k >> 2) * image + (k & 3) * 2;
    if (k < nk) mma_ss<1>(d, a + o, b + o, idesc);
  }
}
// d[128][n] (+)= a(TMEM, bf16 pairs)[128][K] * b(image)[K][n], with b an
// MN-major descriptor; every 32 of K lie GAP columns apart.
template <int K, uint32_t GAP = 16>
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool first) {
  mma_ts<-1>(d, a, b, idesc, !first);
#pragma unroll
  for (int k = 1; k < K / 16; k++) mma_ts<1>(d, a + (k >> 1) * GAP + (k & 1) * 8, b + k * 128, idesc);
}
constexpr uint32_t kHalfRows = 64 * 128 >> 4;  // descriptor step from row 0 to row 64 of an image

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&b);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Without a suspend time the wait is the barrier's own: it returns as soon as
// the phase completes. (With one, a failed test is followed by a sleep.)
__device__ __forceinline__ bool try_wait(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// A wait that ends when another role of the CTA has given up, too.
struct Waiter {
  volatile int *fail;  // in shared memory; the cycles a wait may take follow it
  static __device__ __forceinline__ void init(volatile int *fail, long long limit) {
    *fail = 0;
    *reinterpret_cast<volatile long long *>(fail + 1) = limit;
  }
  __device__ __forceinline__ bool operator()(uint64_t *bar, uint32_t parity) const {
    if (try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (!try_wait(bar, parity)) {
      if (*fail || clock64() - t0 > *reinterpret_cast<volatile long long *>(fail + 1)) {
        *fail = 1;
        return false;
      }
    }
    return true;
  }
  // The same for the computing warps, whose every tile has several waits on its
  // critical path: a thread that gives up goes on without waiting any more (its
  // results are lost, its loops end), so that no warp has to agree on going on.
  __device__ __forceinline__ void pass(uint64_t *bar, uint32_t parity) const {
    if (!try_wait(bar, parity)) (*this)(bar, parity);
    __syncwarp();
  }
  // The same for a whole warp: all of its threads go on, or none.
  __device__ __forceinline__ bool warp(uint64_t *bar, uint32_t parity) const {
    return __all_sync(0xffffffffu, (*this)(bar, parity));
  }
};

// Loads `boxes` 64-column images of a tile.
__device__ __forceinline__ void load_images(uint32_t dst, const CUtensorMap *map, int boxes, int head, int token, int b,
                                            uint64_t *bar) {
  for (int i = 0; i < boxes; i++) tma_load_4d(dst + i * kImage, map, i * 64, head, token, b, bar);
}

// Clears rows [from, 128) of a tile's images; one warp.
__device__ __forceinline__ void clear_rows(uint8_t *tile, int boxes, int from) {
  const int lane = threadIdx.x & 31;
  for (int i = 0; i < boxes; i++)
    for (int o = from * 128 + lane * 16; o < (int)kImage; o += 512)
      *reinterpret_cast<uint4 *>(tile + i * kImage + o) = make_uint4(0, 0, 0, 0);
  fence_async_smem();
  __syncwarp();
}

// The two warps that share an SM quarter begin their exponentials in turns (g:
// warpgroup, others: iterations of the other warpgroup): in step they would
// share its exponential unit, and leave it idle together during everything
// else. The turn passes after a quarter of them: one warp alone leaves the
// unit half idle (an exponential instruction every 8.7 cycles, against 4 with
// four warps).
__device__ __forceinline__ void my_turn(const Waiter &wait, uint64_t *turn, int g, int it, int others) {
  if (g == 0 ? it > 0 && it <= others : it < others)
    wait.pass(turn + 4 * g + (threadIdx.x >> 5 & 3), (g == 0 ? it - 1 : it) & 1);
}
__device__ __forceinline__ void pass_turn(uint64_t *turn, int g) {
  if ((threadIdx.x & 31) == 0) mbar_arrive(turn + 4 * (g ^ 1) + (threadIdx.x >> 5 & 3));
}

// Writes n (a multiple of 8, at most 32) values as bf16, times f.
__device__ __forceinline__ void store_bf16(bf16 *dst, const uint32_t *r, int n, float f) {
#pragma unroll
  for (int c = 0; c < 32; c += 8)
    if (c < n) {
      uint4 u;
      u.x = pack2(__uint_as_float(r[c]) * f, __uint_as_float(r[c + 1]) * f);
      u.y = pack2(__uint_as_float(r[c + 2]) * f, __uint_as_float(r[c + 3]) * f);
      u.z = pack2(__uint_as_float(r[c + 4]) * f, __uint_as_float(r[c + 5]) * f);
      u.w = pack2(__uint_as_float(r[c + 6]) * f, __uint_as_float(r[c + 7]) * f);
      *reinterpret_cast<uint4 *>(dst + c) = u;
    }
}
__device__ __forceinline__ void store_zeros(bf16 *dst, int n) {
  for (int c = 0; c < n; c += 8) *reinterpret_cast<uint4 *>(dst + c) = make_uint4(0, 0, 0, 0);
}

// The end of every kernel: copies and products of a CTA that gave up are
// drained, then TMEM is freed.
__device__ __forceinline__ void leave(uint32_t tmem, const Roles &roles, int warp, volatile int *fail, uint64_t *drain,
                                      int *err) {
  __syncwarp();
  if (warp == roles.product || warp == roles.second) {
    if (elect_one()) {  // the thread that issued the products
      mma_commit(drain);
      mbar_wait(drain, 0);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *fail) report_gave_up(err);
  if (warp == roles.product) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

__device__ __forceinline__ uint8_t *align1024(uint8_t *p) {
  return p + ((1024u - (smem_u32(p) & 1023u)) & 1023u);
}

// ---------------------------------------------------------------------------
// Forward: two query tiles past one stream of key and value tiles. The two
// warpgroups alternate on the tensor cores: while one turns its S into P, the
// other's products run. The output accumulator is rescaled only when a row's
// maximum has grown by more than 2^8 since the exponent's base was chosen
// (the probabilities stay exact in relation to the sum).
// ---------------------------------------------------------------------------

template <int DP>
struct FwdSmem {
  static constexpr int kBoxes = DP / 64, kStages = DP == 64 ? 3 : 2;
  static constexpr uint32_t kTile = kBoxes * kImage;
  static constexpr size_t kBytes = 1024 + (2 + 2 * kStages) * kTile + 512;
};

template <int DP>
__global__ void __launch_bounds__(threads_of(kFwdGroups), 1)
    k_attn_tc(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
              const __grid_constant__ CUtensorMap mv, const AttnParams p, const TcArgs a) {
  using L = FwdSmem<DP>;
  // TMEM: S 2 x 128 columns, O 2 x DP. Where 128 columns are left, P has a
  // place of its own and the next S is computed while this one becomes P;
  // else P replaces S.
  constexpr bool kApart = DP == 64;
  extern __shared__ uint8_t raw[];
  uint8_t *base = align1024(raw);
  uint8_t *sq = base, *sk = sq + 2 * L::kTile, *sv = sk + L::kStages * L::kTile;
  uint64_t *bars = reinterpret_cast<uint64_t *>(sv + L::kStages * L::kTile);
  uint64_t *q_full = bars, *s_full = bars + 2, *p_full = bars + 4, *o_full = bars + 6, *drain = bars + 8,
           *ask = bars + 9, *clean = bars + 10, *s_free = bars + 11, *turn = bars + 13, *k_full = bars + 21, *k_empty = k_full + L::kStages, *v_full = k_empty + L::kStages,
           *v_empty = v_full + L::kStages;
  uint32_t *tmem_ptr = reinterpret_cast<uint32_t *>(bars + 21 + 4 * L::kStages);
  volatile int *fail = reinterpret_cast<volatile int *>(tmem_ptr + 1);
  constexpr Roles roles(kFwdGroups);
  const int warp = threadIdx.x >> 5;

  long long id = blockIdx.x;
  const int pairs = (a.q_tiles + 1) / 2;
  const int split = (int)(id % a.splits);
  id /= a.splits;
  const int hk = (int)(id % p.kv_heads);
  id /= p.kv_heads;
  const int n = (int)(id % p.batch);
  const int pair = pairs - 1 - (int)(id / p.batch);  // the longest causal rows of all heads first
  const AttnMask mask(p, n);
  // key tiles [t0, t1[i]) of query tile i
  int t0, t1[2], most = 0;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int first = (2 * pair + i) * a.tpt;
    const int end = 2 * pair + i < a.q_tiles && first < mask.q_len
                        ? mask.key_end(min(first + a.tpt, mask.q_len) - 1)
                        : 0;
    t1[i] = (end + 127) / 128;
    most = max(most, t1[i]);
  }
  const int per = (most + a.splits - 1) / a.splits;
  t0 = split * per;
#pragma unroll
  for (int i = 0; i < 2; i++) t1[i] = min(t1[i], t0 + per);
  most = max(t1[0], t1[1]);
  const int clear_at = mask.k_len % 128 ? mask.k_len / 128 : INT_MAX;  // the value tile that holds padding

  cudaTriggerProgrammaticLaunchCompletion();  // the join of shares
  if (threadIdx.x == 0) {
    Waiter::init(fail, a.wait);
    for (int i = 0; i < 2; i++) mbar_init(q_full + i, 1), mbar_init(s_full + i, 1), mbar_init(p_full + i, 4), mbar_init(o_full + i, 1), mbar_init(s_free + i, 4);
    mbar_init(drain, 2);
    mbar_init(ask, 2);
    mbar_init(clean, 1);
    for (int i = 0; i < 8; i++) mbar_init(turn + i, 1);
    for (int i = 0; i < L::kStages; i++)
      mbar_init(k_full + i, 1), mbar_init(k_empty + i, 2), mbar_init(v_full + i, 1), mbar_init(v_empty + i, 2);
    fence_barrier_init();
  }
  if (warp == roles.product) tmem_alloc(tmem_ptr, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  const Waiter wait{fail};

  if (warp >= roles.copy) {
    reg_dealloc<88>();
    if (warp == roles.copy && (threadIdx.x & 31) == 0 && t0 < most) {
      int queries = 0;
      for (int i = 0; i < 2; i++)
        if (t0 < t1[i]) {
          mbar_expect_tx(q_full + i, L::kBoxes * a.group * a.tpt * 128);
          load_images(smem_u32(sq + i * L::kTile), &mq, L::kBoxes, a.qh * hk * a.group, (2 * pair + i) * a.tpt, a.qb * n,
                      q_full + i);
          queries |= 1 << i;
        }
      int issued_k = 0, issued_v = 0;
      for (int j = t0; j < most; j++) {
        const int s = (j - t0) % L::kStages, use = (j - t0) / L::kStages;
        if (use > 0 && !wait(k_empty + s, (use - 1) & 1)) break;
        mbar_expect_tx(k_full + s, L::kTile);
        load_images(smem_u32(sk + s * L::kTile), &mk, L::kBoxes, a.kh * hk, j * 128, a.kb * n, k_full + s);
        issued_k++;
        if (use > 0 && !wait(v_empty + s, (use - 1) & 1)) break;
        mbar_expect_tx(v_full + s, L::kTile);
        load_images(smem_u32(sv + s * L::kTile), &mv, L::kBoxes, a.vh * hk, j * 128, a.vb * n, v_full + s);
        issued_v++;
      }
      // every copy has landed before the CTA leaves
      for (int i = 0; i < 2; i++)
        if (queries >> i & 1) mbar_wait(q_full + i, 0);
      for (int i = max(0, issued_k - L::kStages); i < issued_k; i++) mbar_wait(k_full + i % L::kStages, (i / L::kStages) & 1);
      for (int i = max(0, issued_v - L::kStages); i < issued_v; i++) mbar_wait(v_full + i % L::kStages, (i / L::kStages) & 1);
    } else if (warp == roles.clear && clear_at < most && clear_at >= t0) {
      const int it = clear_at - t0, s = it % L::kStages;
      if (wait.warp(ask, 0) && wait.warp(v_full + s, (it / L::kStages) & 1)) {
        clear_rows(sv + s * L::kTile, L::kBoxes, mask.k_len - clear_at * 128);
        if ((threadIdx.x & 31) == 0) mbar_arrive(clean);
      }
    } else if ((warp == roles.product || warp == roles.second) && t0 < most && elect_one()) {
      const int i = warp == roles.second;  // this thread's query tile
      const int end = i ? t1[1] : t1[0];
      const uint32_t dq = desc_k(smem_u32(sq)), dk = desc_k(smem_u32(sk)), dv = desc_mn(smem_u32(sv));
      constexpr uint32_t kStep = L::kTile >> 4;  // descriptors of the next tile
      const uint32_t id_s = instr_desc(1, 128), id_o = instr_desc(1, a.n16) | kBMnMajor;
      const int nk = a.n16 / 16;
      bool ok = wait(k_full, 0);
      if (ok && t0 < end) ok = wait(q_full + i, 0);
      if (ok) {
        if (t0 < end) {
          mma_rows<DP>(tmem + i * 128, dq + i * kStep, dk, nk, id_s);
          mma_commit(s_full + i);
        }
        mma_commit(k_empty);
      }
      int s = 0, use = 0;  // stage of tile j, parity of its use
      // past this query tile's own keys the stages are only passed on
      for (int j = t0; j < most && ok; j++) {
        const int s1 = s + 1 == L::kStages ? 0 : s + 1, use1 = s1 ? use : use ^ 1, parity = (j - t0) & 1;
        const bool more = j + 1 < most;
        if (more) {
          ok = wait(k_full + s1, use1);
          if (!ok) break;
          if (kApart) {
            if (j + 1 < end) {
              ok = wait(s_free + i, parity);
              if (!ok) break;
              tc_fence_after();
              mma_rows<DP>(tmem + i * 128, dq + i * kStep, dk + s1 * kStep, nk, id_s);
              mma_commit(s_full + i);
            }
            mma_commit(k_empty + s1);
          }
        }
        ok = wait(v_full + s, use);
        if (!ok) break;
        if (j == clear_at) {  // asks for the clearing of padding, waits for it
          mbar_arrive(ask);
          ok = wait(clean, 0);
          if (!ok) break;
        }
        if (j < end) {
          ok = wait(p_full + i, parity);
          if (!ok) break;
          tc_fence_after();
          mma_tmem<128>(tmem + 256 + i * DP, kApart ? tmem + 384 + i * 64 : tmem + i * 128, dv + s * kStep, id_o, j == t0);
          mma_commit(o_full + i);
          if (!kApart && j + 1 < end) {
            mma_rows<DP>(tmem + i * 128, dq + i * kStep, dk + s1 * kStep, nk, id_s);
            mma_commit(s_full + i);
          }
        }
        mma_commit(v_empty + s);
        if (!kApart && more) mma_commit(k_empty + s1);
        s = s1, use = use1;
      }
    }
    __syncwarp();
  } else {
    reg_alloc<208>();
    const int i = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lane_base = (uint32_t)(warp & 3) << 21;  // 32 TMEM lanes a warp
    const uint32_t ts = tmem + lane_base + i * 128, to = tmem + lane_base + 256 + i * DP;
    const uint32_t tp = kApart ? tmem + lane_base + 384 + i * 64 : ts;
    const int tile = 2 * pair + i;
    const int token = tile * a.tpt + row / a.group, h = hk * a.group + row % a.group;
    const bool mine = tile < a.q_tiles && row < a.group * a.tpt && token < p.q_tokens;
    const int end = mine ? mask.key_end(token) : 0;
    const float sl2 = p.scale * kLog2e;
    float top = -INFINITY, sum = 0;  // the exponent's base (scaled logits, base 2)
    for (int j = t0; j < t1[i]; j++) {
      const int it = j - t0;
      wait.pass(s_full + i, it & 1);
      tc_fence_after();
      uint32_t r[128];
#pragma unroll
      for (int c = 0; c < 4; c++) tmem_ld32(ts + 32 * c, r + 32 * c);
      tmem_wait_ld();
      if constexpr (kApart) {
        tc_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(s_free + i);
      }
      const int left = end - j * 128;
      if (__any_sync(0xffffffffu, left < 128)) {
#pragma unroll
        for (int c = 0; c < 128; c++)
          if (c >= left) r[c] = 0xff800000u;
      }
      float m4[4];
#pragma unroll
      for (int c = 0; c < 4; c++) m4[c] = __uint_as_float(r[c]);
#pragma unroll
      for (int c = 4; c < 124; c += 8)
#pragma unroll
        for (int k = 0; k < 4; k++) m4[k] = max3(m4[k], __uint_as_float(r[c + k]), __uint_as_float(r[c + 4 + k]));
#pragma unroll
      for (int c = 0; c < 4; c++) m4[c] = fmaxf(m4[c], __uint_as_float(r[124 + c]));
      const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * sl2;
      bool grow = false;
      float f = 1.0f;
      if (top == -INFINITY) {
        top = m;  // nothing summed yet
      } else if (m > top + 8.0f) {
        f = ex2(top - m);
        top = m;
        sum *= f;
        grow = true;
      }
      grow = __any_sync(0xffffffffu, grow);
      if (it > 0 && (kApart || grow)) {  // the previous product: it reads P's place, or is about to be rescaled
        wait.pass(o_full + i, (it - 1) & 1);
        tc_fence_after();
      }
      if (grow) {
#pragma unroll
        for (int c = 0; c < DP; c += 32) {
          uint32_t o[32];
          tmem_ld32(to + c, o);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
          tmem_st32(to + c, o);
        }
      }
      const float shift = top == -INFINITY ? 0.0f : -top;
      if constexpr (kApart) my_turn(wait, turn, i, it, t1[i ^ 1] - t0);
      const float2 scale2 = make_float2(sl2, sl2), shift2 = make_float2(shift, shift);
      float2 s2[2] = {make_float2(0, 0), make_float2(0, 0)};
#pragma unroll
      for (int c = 0; c < 128; c += 32) {
        uint32_t q[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          float2 x = __ffma2_rn(make_float2(__uint_as_float(r[c + k]), __uint_as_float(r[c + k + 1])), scale2, shift2);
          x = make_float2(ex2(x.x), ex2(x.y));
          s2[k / 2 & 1] = __fadd2_rn(s2[k / 2 & 1], x);
          q[k / 2] = pack2(x.x, x.y);
        }
        tmem_st16(tp + c / 2, q);
        if (kApart && c == 0) pass_turn(turn, i);
      }
      sum += (s2[0].x + s2[0].y) + (s2[1].x + s2[1].y);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(p_full + i);
    }
    // output
    const long long rows = (long long)p.batch * p.heads * p.q_tokens;
    const long long at = ((long long)n * p.heads + h) * p.q_tokens + token;
    const float f = sum > 0 ? 1.0f / sum : (sum == 0 ? 0.0f : NAN);
    const float lse = sum == 0 ? -INFINITY : (top + log2f(sum)) * kLn2;
    const bool some = t0 < t1[i];
    if (some) wait.pass(o_full + i, (t1[i] - 1 - t0) & 1);
    tc_fence_after();
    const bool have = some && end > 0;
    if (a.splits == 1) {
      bf16 *dst = (bf16 *)p.out.p + n * p.out.s[0] + token * p.out.s[1] + h * p.out.s[2];
      if (some) {
#pragma unroll
        for (int c = 0; c < DP; c += 32) {
          uint32_t o[32];
          tmem_ld32(to + c, o);
          tmem_wait_ld();
          if (mine && have) store_bf16(dst + c, o, p.head_dim - c, f);
        }
      }
      if (mine && !have) store_zeros(dst, p.head_dim);
      if (mine) p.lse[at] = lse;
    } else if (mine || some) {
      float *dst = p.ws + (split * rows + at) * p.head_dim;
      if (some) {
#pragma unroll
        for (int c = 0; c < DP; c += 32) {
          uint32_t o[32];
          tmem_ld32(to + c, o);
          tmem_wait_ld();
          if (mine && have)
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              if (c + k < p.head_dim)
                *reinterpret_cast<float4 *>(dst + c + k) =
                    make_float4(__uint_as_float(o[k]) * f, __uint_as_float(o[k + 1]) * f, __uint_as_float(o[k + 2]) * f,
                                __uint_as_float(o[k + 3]) * f);
        }
      }
      // a share without keys has lse -inf: its output is not read
      if (mine) p.ws[a.splits * rows * p.head_dim + split * rows + at] = lse;
    }
  }
  leave(tmem, roles, warp, fail, drain, p.err);
}

// ---------------------------------------------------------------------------
// Backward, dK and dV: one key tile (its rows are the TMEM lanes) past the
// query tiles that see it. Per query tile: S' = K Q', dP' = V dO', and from
// TMEM dV += P' dO, dK += dS' Q. A warpgroup takes 32 query columns: the
// arithmetic is bound by its latencies, which four warps an SM quarter cover
// for one another. P' and dS' replace S' and dP' in TMEM. The columns go to the
// products in halves, two pipelines of their own:
//   P(j): dV, S'(j+1)   dS'(j): dK, dP'(j+1)
// Up to head size 64 each has its thread and its own accumulators, which are
// added at the end; beyond, TMEM holds one pair, and one thread serves both
// halves in turn. The order of the sums is fixed in both.
// ---------------------------------------------------------------------------

template <int DP>
struct BwdSmem {
  static constexpr int kBoxes = DP / 64, kStages = DP == 64 ? 3 : 2;
  static constexpr uint32_t kTile = kBoxes * kImage;
  static constexpr uint32_t kRowSums = (2 * 256 + 4) * 4;  // shifts and deltas of two query tiles, two flags
  static constexpr size_t kBytes = 1024 + (2 + 2 * kStages) * kTile + kRowSums + 512;
};

template <int DP>
__global__ void __launch_bounds__(threads_of(kBwdGroups), 1)
    k_attn_dkv_tc(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                  const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mg, const AttnParams p,
                  const TcArgs a) {
  using L = BwdSmem<DP>;
  constexpr bool kTwin = DP == 64;
  extern __shared__ uint8_t raw[];
  uint8_t *base = align1024(raw);
  uint8_t *sk = base, *sv = sk + L::kTile, *sq = sv + L::kTile, *sg = sq + L::kStages * L::kTile;
  float *row_sums = reinterpret_cast<float *>(sg + L::kStages * L::kTile);
  uint64_t *bars = reinterpret_cast<uint64_t *>(sg + L::kStages * L::kTile + L::kRowSums);
  uint64_t *kv_full = bars, *s_full = bars + 1, *g_full = bars + 3, *p_full = bars + 5, *d_full = bars + 7,
           *done = bars + 9, *drain = bars + 10, *clean = bars + 11, *full = bars + 12, *empty = full + L::kStages;
  uint32_t *tmem_ptr = reinterpret_cast<uint32_t *>(bars + 12 + 2 * L::kStages);
  volatile int *fail = reinterpret_cast<volatile int *>(tmem_ptr + 1);
  constexpr Roles roles(kBwdGroups);
  const int warp = threadIdx.x >> 5;

  long long id = blockIdx.x;
  const int hk = (int)(id % p.kv_heads);
  id /= p.kv_heads;
  const int n = (int)(id % p.batch), kt = (int)(id / p.batch);  // the keys that most queries see first
  const AttnMask mask(p, n);
  const int key0 = kt * 128;
  const int t0 = key0 < mask.k_len ? mask.row_begin(key0) / a.tpt : 0;
  const int t1 = key0 < mask.k_len ? (mask.q_len + a.tpt - 1) / a.tpt : 0;
  const bool some = t0 < t1;
  const int clear_at = mask.q_len % a.tpt ? mask.q_len / a.tpt : INT_MAX;  // the query tile that holds padding

  if (threadIdx.x == 0) {
    Waiter::init(fail, a.wait);
    mbar_init(kv_full, 1), mbar_init(done, kTwin ? 2 : 1), mbar_init(drain, 2), mbar_init(clean, 1);
    for (int i = 0; i < 2; i++)
      mbar_init(s_full + i, 2), mbar_init(g_full + i, 1), mbar_init(p_full + i, 8), mbar_init(d_full + i, 8);
    for (int i = 0; i < L::kStages; i++) mbar_init(full + i, 1), mbar_init(empty + i, kTwin ? 2 : 1);
    fence_barrier_init();
  }
  // rows of the query images past group * tpt are never written by the copies
  if (a.group * a.tpt < 128)
    for (int t = warp; t < 2 * L::kStages; t += threads_of(kBwdGroups) / 32) clear_rows(sq + t * L::kTile, L::kBoxes, a.group * a.tpt);
  if (warp == roles.product) tmem_alloc(tmem_ptr, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // delta comes from the kernel of dQ, which may still be at work; all threads
  // stop here, so that no bounded wait runs against its time
  cudaGridDependencySynchronize();
  const uint32_t tmem = *tmem_ptr;
  // S', dP' (P' and dS' in the first half of every warpgroup's 32 columns), the
  // accumulators of the first pipeline, and t_next further those of the second
  const uint32_t t_s = tmem, t_g = tmem + 128, t_dv = tmem + 256, t_dk = tmem + (kTwin ? 384 : 256 + DP);
  constexpr uint32_t t_next = kTwin ? 64 : 0;
  const Waiter wait{fail};

  if (warp == roles.copy && (threadIdx.x & 31) == 0 && some) {
    mbar_expect_tx(kv_full, 2 * L::kTile);
    load_images(smem_u32(sk), &mk, L::kBoxes, a.kh * hk, key0, a.kb * n, kv_full);
    load_images(smem_u32(sv), &mv, L::kBoxes, a.vh * hk, key0, a.vb * n, kv_full);
    int issued = 0;
    for (int j = t0; j < t1; j++) {
      const int s = (j - t0) % L::kStages, use = (j - t0) / L::kStages;
      if (use > 0 && !wait(empty + s, (use - 1) & 1)) break;
      mbar_expect_tx(full + s, 2 * L::kBoxes * a.group * a.tpt * 128);
      load_images(smem_u32(sq + s * L::kTile), &mq, L::kBoxes, a.qh * hk * a.group, j * a.tpt, a.qb * n, full + s);
      load_images(smem_u32(sg + s * L::kTile), &mg, L::kBoxes, a.gh * hk * a.group, j * a.tpt, a.gb * n, full + s);
      issued++;
    }
    mbar_wait(kv_full, 0);
    for (int i = max(0, issued - L::kStages); i < issued; i++) mbar_wait(full + i % L::kStages, (i / L::kStages) & 1);
  } else if (warp == roles.clear && some) {
    // lse and delta of every query tile's rows, half a tile ahead of their use:
    // shift (base 2; -inf where a row has no probabilities) and -delta
    const int lane = threadIdx.x & 31;
    int column[4];  // token within a query tile
    const float *lse_of[4], *delta_of[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int r = k * 32 + lane;
      column[k] = r < a.group * a.tpt ? r / a.group : INT_MAX / 2;
      const long long at = ((long long)n * p.heads + hk * a.group + r % a.group) * p.q_tokens;
      lse_of[k] = p.lse + at, delta_of[k] = p.ws + at;
    }
    for (int j = t0; j < t1; j++) {
      const int it = j - t0;
      float l[4], d[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int token = j * a.tpt + column[k];
        l[k] = -INFINITY, d[k] = 0;
        if (token < mask.q_len) l[k] = lse_of[k][token], d[k] = delta_of[k][token];
      }
      // with the probabilities of tile j - 1 the warpgroups are done with
      // tile j - 2 (a wait for that tile itself could miss its phase)
      if (it >= 1 && !(wait.warp(p_full, (it - 1) & 1) && wait.warp(p_full + 1, (it - 1) & 1))) break;
      if (j == clear_at) {
        const int s = it % L::kStages, from = (mask.q_len - j * a.tpt) * a.group;
        if (!wait.warp(full + s, (it / L::kStages) & 1)) break;
        clear_rows(sq + s * L::kTile, L::kBoxes, from);
        clear_rows(sg + s * L::kTile, L::kBoxes, from);
        if (lane == 0) mbar_arrive(clean);
      }
      float *to = row_sums + (it & 1) * 256;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        to[k * 32 + lane] = l[k] == -INFINITY ? -INFINITY : -l[k] * kLog2e;
        to[128 + k * 32 + lane] = -d[k];
      }
      __syncwarp();
      if (lane < 2) mbar_arrive(s_full + lane);
    }
  } else if ((warp == roles.product || (kTwin && warp == roles.second)) && some && elect_one()) {
    const int first = warp == roles.second, last = kTwin ? first : 1;  // this thread's halves
    const uint32_t dk = desc_k(smem_u32(sk)), dv = desc_k(smem_u32(sv)), dq = desc_k(smem_u32(sq)),
                   dg = desc_k(smem_u32(sg)), dq_mn = desc_mn(smem_u32(sq)), dg_mn = desc_mn(smem_u32(sg));
    constexpr uint32_t kStep = L::kTile >> 4;
    const uint32_t id_s = instr_desc(1, 64), id_o = instr_desc(1, a.n16) | kBMnMajor;
    const int nk = a.n16 / 16;
    bool ok = wait(kv_full, 0) && wait(full, 0) && (t0 != clear_at || wait(clean, 0));
#pragma unroll 1
    for (int w = first; w <= last && ok; w++) {
      mma_rows<DP>(t_s + w * 64, dk, dq + w * kHalfRows, nk, id_s);
      mma_commit(s_full + w);
      mma_rows<DP>(t_g + w * 64, dv, dg + w * kHalfRows, nk, id_s);
      mma_commit(g_full + w);
    }
    int s = 0, use = 0;
    for (int j = t0; j < t1 && ok; j++) {
      const int s1 = s + 1 == L::kStages ? 0 : s + 1, use1 = s1 ? use : use ^ 1, parity = (j - t0) & 1;
      const bool more = j + 1 < t1;
#pragma unroll 1
      for (int w = first; w <= last; w++) {
        ok = wait(p_full + w, parity);
        if (!ok) break;
        tc_fence_after();
        mma_tmem<64, 32>(t_dv + w * t_next, t_s + w * 64, dg_mn + s * kStep + w * kHalfRows, id_o,
                         j == t0 && (kTwin || w == 0));
        if (more) {
          if (w == first) ok = wait(full + s1, use1) && (j + 1 != clear_at || wait(clean, 0));
          if (!ok) break;
          mma_rows<DP>(t_s + w * 64, dk, dq + s1 * kStep + w * kHalfRows, nk, id_s);
          mma_commit(s_full + w);
        }
        ok = wait(d_full + w, parity);
        if (!ok) break;
        tc_fence_after();
        mma_tmem<64, 32>(t_dk + w * t_next, t_g + w * 64, dq_mn + s * kStep + w * kHalfRows, id_o,
                         j == t0 && (kTwin || w == 0));
        if (w == last) mma_commit(empty + s);
        if (more) {
          mma_rows<DP>(t_g + w * 64, dv, dg + s1 * kStep + w * kHalfRows, nk, id_s);
          mma_commit(g_full + w);
        }
      }
      s = s1, use = use1;
    }
    if (ok) mma_commit(done);
  } else if (warp < roles.copy) {
    const int wg = warp >> 2, half = wg >> 1, row = threadIdx.x & 127, lane = threadIdx.x & 31;
    const uint32_t lane_base = (uint32_t)(warp & 3) << 21;
    const uint32_t ts = t_s + lane_base + wg * 32, tg = t_g + lane_base + wg * 32;
    const int key = key0 + row;
    const int begin = key < mask.k_len ? mask.row_begin(key) : INT_MAX / 2;
    const float sl2 = p.scale * kLog2e;
    const float2 scale2 = make_float2(sl2, sl2);
    for (int j = t0; j < t1; j++) {
      const int it = j - t0;
      const float *mine_shift = row_sums + (it & 1) * 256 + wg * 32, *mine_delta = mine_shift + 128;
      // columns below `skip` are queries that do not see this key
      const int skip = min(max(min(max(begin - j * a.tpt, 0), 128) * a.group - wg * 32, 0), 32);
      const bool masked = __any_sync(0xffffffffu, skip > 0);
      wait.pass(s_full + half, it & 1);
      tc_fence_after();
      uint32_t r[32];
      tmem_ld32(ts, r);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        const float4 l = *reinterpret_cast<const float4 *>(mine_shift + c);
        const float2 x = __ffma2_rn(make_float2(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), scale2, make_float2(l.x, l.y));
        const float2 y = __ffma2_rn(make_float2(__uint_as_float(r[c + 2]), __uint_as_float(r[c + 3])), scale2, make_float2(l.z, l.w));
        r[c] = __float_as_uint(ex2(x.x)), r[c + 1] = __float_as_uint(ex2(x.y));
        r[c + 2] = __float_as_uint(ex2(y.x)), r[c + 3] = __float_as_uint(ex2(y.y));
      }
      if (masked) {
#pragma unroll
        for (int c = 0; c < 32; c++)
          if (c < skip) r[c] = 0;
      }
      uint32_t q[16];
#pragma unroll
      for (int c = 0; c < 16; c++) q[c] = pack2(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1]));
      tmem_st16(ts, q);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + half);
      wait.pass(g_full + half, it & 1);
      tc_fence_after();
      uint32_t g[32];
      tmem_ld32(tg, g);
      tmem_wait_ld();
      if (masked) {
#pragma unroll
        for (int c = 0; c < 32; c++)
          if (c < skip) g[c] = 0;
      }
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        const float4 d = *reinterpret_cast<const float4 *>(mine_delta + c);
        const float2 x = __fmul2_rn(make_float2(__uint_as_float(r[c]), __uint_as_float(r[c + 1])),
                                    __fadd2_rn(make_float2(__uint_as_float(g[c]), __uint_as_float(g[c + 1])), make_float2(d.x, d.y)));
        const float2 y = __fmul2_rn(make_float2(__uint_as_float(r[c + 2]), __uint_as_float(r[c + 3])),
                                    __fadd2_rn(make_float2(__uint_as_float(g[c + 2]), __uint_as_float(g[c + 3])), make_float2(d.z, d.w)));
        q[c / 2] = pack2(x.x, x.y);
        q[c / 2 + 1] = pack2(y.x, y.y);
      }
      tmem_st16(tg, q);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(d_full + half);
    }
    if (some) wait.pass(done, 0);
    tc_fence_after();
    const bool inside = key < p.k_tokens, have = some && key < mask.k_len;
    // warpgroups 0 and 1 write dV, 2 and 3 dK, half of the columns each
    constexpr int kCols = DP / 2;
    const AttnTensor &t = half ? p.dk : p.dv;
    const int first = (wg & 1) * kCols;
    bf16 *dst = (bf16 *)t.p + n * t.s[0] + (long long)key * t.s[1] + hk * t.s[2] + first;
    if (some) {
#pragma unroll
      for (int c = 0; c < kCols; c += 32) {
        uint32_t o[32];
        tmem_ld32((half ? t_dk : t_dv) + lane_base + first + c, o);
        tmem_wait_ld();
        if constexpr (kTwin) {
          uint32_t o2[32];
          tmem_ld32((half ? t_dk : t_dv) + t_next + lane_base + first + c, o2);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) + __uint_as_float(o2[k]));
        }
        if (inside && have) store_bf16(dst + c, o, p.head_dim - first - c, half ? p.scale : 1.0f);
      }
    }
    if (inside && !have) store_zeros(dst, min(kCols, p.head_dim - first));
  }
  leave(tmem, roles, warp, fail, drain, p.err);
}

// ---------------------------------------------------------------------------
// Backward, dQ: one query tile past the key tiles it sees. S = Q K' and
// dP = dO V' are recomputed, dQ += dS K from TMEM, where dS replaces dP. The
// warpgroups take 32 key columns each; the halves of the columns are two
// pipelines, with a product thread and an accumulator each:
//   S free: S(j+1)   dS(j): dQ, dP(j+1)
// A thread's lse and delta stay in registers. This pass runs first and leaves
// the row sums delta in the workspace for the other.
// ---------------------------------------------------------------------------

template <int DP>
__global__ void __launch_bounds__(threads_of(kBwdGroups), 1)
    k_attn_dq_tc(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                 const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mg, const AttnParams p,
                 const TcArgs a) {
  using L = BwdSmem<DP>;
  extern __shared__ uint8_t raw[];
  uint8_t *base = align1024(raw);
  uint8_t *sq = base, *sg = sq + L::kTile, *sk = sg + L::kTile, *sv = sk + L::kStages * L::kTile;
  float *row_sums = reinterpret_cast<float *>(sv + L::kStages * L::kTile);
  uint64_t *bars = reinterpret_cast<uint64_t *>(sv + L::kStages * L::kTile + L::kRowSums);
  uint64_t *q_full = bars, *s_full = bars + 1, *g_full = bars + 3, *s_free = bars + 5, *d_full = bars + 7,
           *done = bars + 9, *drain = bars + 10, *ask = bars + 11, *clean = bars + 12, *full = bars + 13, *empty = full + L::kStages;
  uint32_t *tmem_ptr = reinterpret_cast<uint32_t *>(bars + 13 + 2 * L::kStages);
  volatile int *fail = reinterpret_cast<volatile int *>(tmem_ptr + 1);
  constexpr Roles roles(kBwdGroups);
  const int warp = threadIdx.x >> 5;

  long long id = blockIdx.x;
  const int hk = (int)(id % p.kv_heads);
  id /= p.kv_heads;
  const int n = (int)(id % p.batch);
  const int qt = a.q_tiles - 1 - (int)(id / p.batch);  // the longest causal rows first
  const AttnMask mask(p, n);
  const int first = qt * a.tpt;
  const int t1 = first < mask.q_len ? (mask.key_end(min(first + a.tpt, mask.q_len) - 1) + 127) / 128 : 0;
  const int clear_at = mask.k_len % 128 ? mask.k_len / 128 : INT_MAX;  // the key tile that holds padding

  cudaTriggerProgrammaticLaunchCompletion();  // dK and dV
  if (threadIdx.x == 0) {
    Waiter::init(fail, a.wait);
    mbar_init(q_full, 1), mbar_init(done, 2), mbar_init(drain, 2), mbar_init(ask, 2), mbar_init(clean, 1);
    for (int i = 0; i < 2; i++)
      mbar_init(s_full + i, 1), mbar_init(g_full + i, 1), mbar_init(s_free + i, 8), mbar_init(d_full + i, 8);
    for (int i = 0; i < L::kStages; i++) mbar_init(full + i, 1), mbar_init(empty + i, 2);
    fence_barrier_init();
  }
  if (warp == roles.product) tmem_alloc(tmem_ptr, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  const uint32_t t_s = tmem, t_g = tmem + 128, t_dq = tmem + 256;
  const Waiter wait{fail};

  if (warp == roles.copy && (threadIdx.x & 31) == 0 && t1 > 0) {
    mbar_expect_tx(q_full, 2 * L::kBoxes * a.group * a.tpt * 128);
    load_images(smem_u32(sq), &mq, L::kBoxes, a.qh * hk * a.group, first, a.qb * n, q_full);
    load_images(smem_u32(sg), &mg, L::kBoxes, a.gh * hk * a.group, first, a.gb * n, q_full);
    int issued = 0;
    for (int j = 0; j < t1; j++) {
      const int s = j % L::kStages, use = j / L::kStages;
      if (use > 0 && !wait(empty + s, (use - 1) & 1)) break;
      mbar_expect_tx(full + s, 2 * L::kTile);
      load_images(smem_u32(sk + s * L::kTile), &mk, L::kBoxes, a.kh * hk, j * 128, a.kb * n, full + s);
      load_images(smem_u32(sv + s * L::kTile), &mv, L::kBoxes, a.vh * hk, j * 128, a.vb * n, full + s);
      issued++;
    }
    mbar_wait(q_full, 0);
    for (int i = max(0, issued - L::kStages); i < issued; i++) mbar_wait(full + i % L::kStages, (i / L::kStages) & 1);
  } else if (warp == roles.clear && clear_at < t1) {
    const int s = clear_at % L::kStages;
    if (wait.warp(ask, 0) && wait.warp(full + s, (clear_at / L::kStages) & 1)) {
      clear_rows(sk + s * L::kTile, L::kBoxes, mask.k_len - clear_at * 128);
      if ((threadIdx.x & 31) == 0) mbar_arrive(clean);
    }
  } else if ((warp == roles.product || warp == roles.second) && t1 > 0 && elect_one()) {
    const int w = warp == roles.second;  // this thread's half
    const uint32_t dq = desc_k(smem_u32(sq)), dg = desc_k(smem_u32(sg)), dk = desc_k(smem_u32(sk)) + w * kHalfRows,
                   dv = desc_k(smem_u32(sv)) + w * kHalfRows, dk_mn = desc_mn(smem_u32(sk)) + w * kHalfRows;
    constexpr uint32_t kStep = L::kTile >> 4;
    const uint32_t id_s = instr_desc(1, 64), id_o = instr_desc(1, a.n16) | kBMnMajor;
    const int nk = a.n16 / 16;
    const uint32_t ts = t_s + w * 64, tg = t_g + w * 64, tq = t_dq + w * DP;
    // key tile j is there, its padding cleared
    auto ready = [&](int j, int s, int use) {
      if (!wait(full + s, use)) return false;
      if (j != clear_at) return true;
      mbar_arrive(ask);
      return wait(clean, 0);
    };
    bool ok = wait(q_full, 0) && ready(0, 0, 0);
    if (ok) {
      mma_rows<DP>(ts, dq, dk, nk, id_s);
      mma_commit(s_full + w);
      mma_rows<DP>(tg, dg, dv, nk, id_s);
      mma_commit(g_full + w);
    }
    int s = 0, use = 0;
    for (int j = 0; j < t1 && ok; j++) {
      const int s1 = s + 1 == L::kStages ? 0 : s + 1, use1 = s1 ? use : use ^ 1, parity = j & 1;
      const bool more = j + 1 < t1;
      if (more) {
        ok = ready(j + 1, s1, use1) && wait(s_free + w, parity);
        if (!ok) break;
        tc_fence_after();
        mma_rows<DP>(ts, dq, dk + s1 * kStep, nk, id_s);
        mma_commit(s_full + w);
      }
      ok = wait(d_full + w, parity);
      if (!ok) break;
      tc_fence_after();
      mma_tmem<64, 32>(tq, tg, dk_mn + s * kStep, id_o, j == 0);
      mma_commit(empty + s);
      if (more) {
        mma_rows<DP>(tg, dg, dv + s1 * kStep, nk, id_s);
        mma_commit(g_full + w);
      }
      s = s1, use = use1;
    }
    if (ok) mma_commit(done);
  } else if (warp < roles.copy) {
    const int wg = warp >> 2, half = wg >> 1, row = threadIdx.x & 127, lane = threadIdx.x & 31;
    const uint32_t lane_base = (uint32_t)(warp & 3) << 21;
    const uint32_t ts = t_s + lane_base + wg * 32, tg = t_g + lane_base + wg * 32;
    const int token = first + row / a.group, h = hk * a.group + row % a.group;
    const bool mine = row < a.group * a.tpt && token < p.q_tokens;
    const int end = mine ? mask.key_end(token) : 0;
    const long long at = ((long long)n * p.heads + h) * p.q_tokens + token;
    const float v = end ? p.lse[at] : -INFINITY;
    const float shift = v == -INFINITY ? -INFINITY : -v * kLog2e;
    // delta = rowsum(dO O): a warpgroup adds every fourth 8 columns
    float part = 0;
    if (end > 0) {
      const bf16 *x = (const bf16 *)p.dout.p + n * p.dout.s[0] + token * p.dout.s[1] + h * p.dout.s[2];
      const bf16 *y = (const bf16 *)p.out.p + n * p.out.s[0] + token * p.out.s[1] + h * p.out.s[2];
#pragma unroll
      for (int c = 0; c < DP; c += 32)
        if (c + wg * 8 < p.head_dim) {
          float u[8], w[8];
          tok::Pack<bf16, 8>::load(x + c + wg * 8, u);
          tok::Pack<bf16, 8>::load(y + c + wg * 8, w);
#pragma unroll
          for (int k = 0; k < 8; k++) part = fmaf(u[k], w[k], part);
        }
    }
    row_sums[wg * 128 + row] = part;
    bar_named(1, 512);
    const float delta = (row_sums[row] + row_sums[128 + row]) + (row_sums[256 + row] + row_sums[384 + row]);
    if (wg == 0 && mine) p.ws[at] = delta;  // for the key pass
    const float sl2 = p.scale * kLog2e;
    const float2 scale2 = make_float2(sl2, sl2), shift2 = make_float2(shift, shift), delta2 = make_float2(-delta, -delta);
    for (int j = 0; j < t1; j++) {
      const int left = end - j * 128 - wg * 32;
      const bool masked = __any_sync(0xffffffffu, left < 32);
      wait.pass(s_full + half, j & 1);
      tc_fence_after();
      uint32_t r[32];
      tmem_ld32(ts, r);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free + half);
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        const float2 x = __ffma2_rn(make_float2(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), scale2, shift2);
        r[c] = __float_as_uint(ex2(x.x)), r[c + 1] = __float_as_uint(ex2(x.y));
      }
      wait.pass(g_full + half, j & 1);
      tc_fence_after();
      uint32_t g[32], q[16];
      tmem_ld32(tg, g);
      tmem_wait_ld();
      if (masked) {
#pragma unroll
        for (int c = 0; c < 32; c++)
          if (c >= left) r[c] = 0, g[c] = 0;
      }
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        float2 x = __fmul2_rn(make_float2(__uint_as_float(r[c]), __uint_as_float(r[c + 1])),
                              __fadd2_rn(make_float2(__uint_as_float(g[c]), __uint_as_float(g[c + 1])), delta2));
        q[c / 2] = pack2(x.x, x.y);
      }
      tmem_st16(tg, q);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(d_full + half);
    }
    if (t1 > 0) wait.pass(done, 0);
    tc_fence_after();
    const bool have = t1 > 0 && end > 0;
    bf16 *dst = (bf16 *)p.dq.p + n * p.dq.s[0] + token * p.dq.s[1] + h * p.dq.s[2];
    // a warpgroup writes a quarter of the columns
    constexpr int kCols = DP / 4;
    const int c0 = wg * kCols;
    if (t1 > 0) {
      uint32_t o[32], o2[32];  // of both pipelines
      if constexpr (kCols == 32) {
        tmem_ld32(t_dq + lane_base + c0, o);
        tmem_ld32(t_dq + DP + lane_base + c0, o2);
      } else {
        tmem_ld16(t_dq + lane_base + c0, o);
        tmem_ld16(t_dq + DP + lane_base + c0, o2);
      }
      tmem_wait_ld();
#pragma unroll
      for (int k = 0; k < kCols; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) + __uint_as_float(o2[k]));
      if (mine && have) store_bf16(dst + c0, o, min(kCols, p.head_dim - c0), p.scale);
    }
    if (mine && !have && wg == 0) store_zeros(dst, p.head_dim);
  }
  leave(tmem, roles, warp, fail, drain, p.err);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

bool tma_tensor(const AttnTensor &t, int tokens, int heads, int batch) {
  if (reinterpret_cast<uintptr_t>(t.p) & 15) return false;
  const int extent[3] = {batch, tokens, heads};
  for (int i = 0; i < 3; i++) {
    if (extent[i] == 1) continue;
    if (t.s[i] % 8 || t.s[i] < 0 || t.s[i] >= (1ll << 38) || (t.s[i] == 0 && i == 1)) return false;
  }
  return true;
}
bool wide_rows(const AttnTensor &t) {
  return (reinterpret_cast<uintptr_t>(t.p) & 15) == 0 && t.s[0] % 8 == 0 && t.s[1] % 8 == 0 && t.s[2] % 8 == 0;
}

// [batch][tokens][heads][d] as a 4-D map (d, head, token, batch) with boxes of
// 64 columns x `heads_box` heads x `rows_box` tokens. A broadcast dimension has
// extent 1.
bool encode(CUtensorMap *m, const AttnTensor &t, int d, int heads, int tokens, int batch, int heads_box, int rows_box,
            bool &has_heads, bool &has_batch) {
  has_heads = t.s[2] != 0 || heads == 1;
  has_batch = t.s[0] != 0 || batch == 1;
  if (!has_heads && heads_box > 1) return false;
  cuuint64_t dim[4] = {(cuuint64_t)d, (cuuint64_t)(has_heads ? heads : 1), (cuuint64_t)tokens, (cuuint64_t)(has_batch ? batch : 1)};
  // strides of dimensions of extent 1 are never used: any valid one will do
  cuuint64_t stride[3] = {(cuuint64_t)t.s[2] * 2, (cuuint64_t)t.s[1] * 2, (cuuint64_t)t.s[0] * 2};
  for (int i = 0; i < 3; i++)
    if (dim[i + 1] == 1) stride[i] = (cuuint64_t)((d * 2 + 15) / 16 * 16);
  cuuint32_t box[4] = {64, (cuuint32_t)heads_box, (cuuint32_t)rows_box, 1}, step[4] = {1, 1, 1, 1};
  auto fn = tensor_map_encoder();
  return fn && fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(t.p), dim, stride, box, step,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

TcArgs shape_of(const AttnParams &p) {
  TcArgs a{};
  a.group = p.heads / p.kv_heads;
  a.tpt = 128 / a.group;
  a.q_tiles = (p.q_tokens + a.tpt - 1) / a.tpt;
  a.k_tiles = (p.k_tokens + 127) / 128;
  a.n16 = (p.head_dim + 15) / 16 * 16;
  a.splits = 1;
  a.wait = p.wait > 0 ? p.wait : kWaitCycles;
  return a;
}

// Shares of the keys in the forward: enough for a CTA on every SM, while a
// share keeps at least two key tiles, and none is empty.
int tc_splits(const AttnParams &p, const TcArgs &a) {
  const long long ctas = (long long)p.batch * p.kv_heads * ((a.q_tiles + 1) / 2);
  const int sms = 148, most = a.k_tiles / 2;
  if (ctas == 0 || ctas * 2 > sms || most < 2) return 1;
  const int want = std::min((int)(sms / ctas), most), per = (a.k_tiles + want - 1) / want;
  return (a.k_tiles + per - 1) / per;
}

template <int DP>
cudaError_t forward_tc(const AttnParams &p, const TcArgs &a, const CUtensorMap &mq, const CUtensorMap &mk,
                       const CUtensorMap &mv, cudaStream_t st) {
  constexpr size_t sm = FwdSmem<DP>::kBytes;
  const cudaError_t e = allow_smem<k_attn_tc<DP>>(sm);
  if (e != cudaSuccess) return e;
  const long long grid = (long long)p.batch * p.kv_heads * ((a.q_tiles + 1) / 2) * a.splits;
  k_attn_tc<DP><<<(unsigned)grid, threads_of(kFwdGroups), sm, st>>>(mq, mk, mv, p, a);
  return cudaGetLastError();
}

template <int DP>
cudaError_t backward_tc(const AttnParams &p, const TcArgs &a, const CUtensorMap &mq, const CUtensorMap &mk,
                        const CUtensorMap &mv, const CUtensorMap &mg, cudaStream_t st) {
  constexpr size_t sm = BwdSmem<DP>::kBytes;
  cudaError_t e = allow_smem<k_attn_dq_tc<DP>>(sm);
  if (e == cudaSuccess) e = allow_smem<k_attn_dkv_tc<DP>>(sm);
  if (e != cudaSuccess) return e;
  const long long heads = (long long)p.batch * p.kv_heads;
  k_attn_dq_tc<DP><<<(unsigned)(heads * a.q_tiles), threads_of(kBwdGroups), sm, st>>>(mq, mk, mv, mg, p, a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return tok::launch_next(k_attn_dkv_tc<DP>, heads * a.k_tiles, threads_of(kBwdGroups), sm, st, mq, mk, mv, mg, p, a);
}

}  // namespace

bool attention_tc_takes(const AttnParams &p, bool backward) {
  if (p.head_dim % 8 || !(p.scale > 0) || p.scale > 1e30f) return false;
  if (!p.batch || !p.heads || !p.q_tokens || !p.k_tokens || p.heads / p.kv_heads > 128) return false;
  const bool grouped = p.heads > p.kv_heads;
  if (!tma_tensor(p.q, p.q_tokens, p.heads, p.batch) || !tma_tensor(p.k, p.k_tokens, p.kv_heads, p.batch) ||
      !tma_tensor(p.v, p.k_tokens, p.kv_heads, p.batch) || (grouped && p.q.s[2] == 0))
    return false;
  if (!backward) return wide_rows(p.out);
  return tma_tensor(p.dout, p.q_tokens, p.heads, p.batch) && wide_rows(p.out) && !(grouped && p.dout.s[2] == 0) && wide_rows(p.dq) &&
         wide_rows(p.dk) && wide_rows(p.dv);
}

int attention_tc_splits(const AttnParams &p) {
  if (!p.batch || !p.heads || !p.q_tokens || !p.k_tokens || p.heads / p.kv_heads > 128) return 1;
  return tc_splits(p, shape_of(p));
}

cudaError_t attention_tc(const AttnParams &p, bool backward, cudaStream_t st) {
  TcArgs a = shape_of(p);
  CUtensorMap mq, mk, mv, mg;
  bool h, b;
  if (!encode(&mq, p.q, p.head_dim, p.heads, p.q_tokens, p.batch, a.group, a.tpt, h, b)) return cudaErrorInvalidValue;
  a.qh = h, a.qb = b;
  if (!encode(&mk, p.k, p.head_dim, p.kv_heads, p.k_tokens, p.batch, 1, 128, h, b)) return cudaErrorInvalidValue;
  a.kh = h, a.kb = b;
  if (!encode(&mv, p.v, p.head_dim, p.kv_heads, p.k_tokens, p.batch, 1, 128, h, b)) return cudaErrorInvalidValue;
  a.vh = h, a.vb = b;
  if (!backward) {
    a.splits = tc_splits(p, a);
    return p.head_dim <= 64 ? forward_tc<64>(p, a, mq, mk, mv, st) : forward_tc<128>(p, a, mq, mk, mv, st);
  }
  if (!encode(&mg, p.dout, p.head_dim, p.heads, p.q_tokens, p.batch, a.group, a.tpt, h, b)) return cudaErrorInvalidValue;
  a.gh = h, a.gb = b;
  return p.head_dim <= 64 ? backward_tc<64>(p, a, mq, mk, mv, mg, st) : backward_tc<128>(p, a, mq, mk, mv, mg, st);
}

}  // namespace gpu
}  // namespace illumina
