// Linear layer: out = residual + act(x_scale * w_scale * (x weights^T) + bias), binary16 or e4m3 operands, 32 bit sums.
//
// Three kernels, four variants:
//   linear_rows   (ROWS)       up to 16 rows: the call is the time to stream the weights.  Warp MMAs with the weights as
//                              the 16 row operand, straight from global memory into registers.  One row, 4096 to 4096:
//                              7.2 us, 4.7 TB/s of weights.
//   linear_split  (SPLIT)      few rows: tcgen05 with 128 output channels as the MMA's rows and the tokens as its columns;
//                              c_in split over a cluster, partial sums joined through distributed shared memory.
//                              100 rows, 2048 to 8192 with gelu: 14.4 us (2.5 TB/s; weights at memory speed for 6 of
//                              them, the rest is set-up and the join).
//   linear_tile   (TILE, ANY)  persistent tcgen05 tiles of 128 rows per block, or of 256 rows over a pair of blocks
//                              (cta_group::2); ANY fills the same shared memory tiles with plain loads.  8192 x 4096 x
//                              16384 binary16 with gelu: 750 to 890 us by clock (1.24 to 1.47 PFLOP/s), tensor pipe
//                              88 % busy, bound by the power limit; 2088960 rows of 96 to 64: 105 us, 6.35 TB/s;
//                              522240 rows of 9 to 32 (GROUPED): 21 us.
#include "internal.h"
#include "tc_ptx.h"
#include <cuda.h>
#include <cuda_fp8.h>
#include <atomic>
#include <math.h>
#include <mutex>
#include <new>
#include <string.h>

namespace dnxcu {
namespace {

struct LinArgs {
  alignas(64) CUtensorMap tm_x, tm_w, tm_out, tm_res;
  const uint8_t *x, *w;
  const float *x_scale, *w_scale;
  const __half *bias, *res;
  __half *out;
  long long xs, ws, rs, os;  // row strides: x and w in bytes, residual and out in elements
  int M, N, K;
  int act;
  float alpha;
  int BN;        // tile: output channels per tile; split: rows (tokens) per tile
  int mt, nt;    // tiles along rows and output channels
  int kb;        // 128 byte wide steps along c_in
  int stages;
  int per_stage; // tile: 128 byte steps per stage (1 or 2)
  int split;     // split: blocks per cluster
  int overlay;   // split: the received partial sums lie over the operand stages
  int teams;     // tile: epilogue teams
  int bufs;      // tile: accumulators
  int w_res;     // tile: the weights of the (one) column of tiles stay in shared memory
  int gr, n1, k1;  // tile: rows taken together as one (see GROUPED), and the channels of a single one; gr = 1: none
  int group;     // tile: tiles along the rows that are walked together
  int out_tma, res_tma;
  int out_pack, res_pack;  // tile: packed rows of at most 64 channels: 32 of them are one piece of memory on a 16 byte boundary
  int *status;
  unsigned long long wait_limit;
};

// ---- epilogue arithmetic ----------------------------------------------------
template <int ACT>
__device__ __forceinline__ float act_one(float v, float alpha) {
  if (ACT == DNXCU_ACT_RELU) return v < 0.0f ? 0.0f : v;  // (a NaN stays one)
  if (ACT == DNXCU_ACT_LEAKY) return v > 0.0f ? v : alpha * v;
  if (ACT == DNXCU_ACT_GELU) return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
  if (ACT == DNXCU_ACT_GELU_TANH) {
    // (1 + tanh u) / 2 = 1 / (1 + exp(-2u))
    const float u2 = v * (1.5957691216057308f + 0.071354816272600243f * v * v);
    return __fdividef(v, 1.0f + __expf(-u2));
  }
  if (ACT == DNXCU_ACT_SILU) return __fdividef(v, 1.0f + __expf(-v));
  return v;
}
template <int ACT, int N>
__device__ __forceinline__ void act_all(float (&v)[N], float alpha) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = act_one<ACT>(v[i], alpha);
}
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act, float alpha) {
  switch (act) {
    case DNXCU_ACT_RELU: act_all<DNXCU_ACT_RELU>(v, alpha); break;
    case DNXCU_ACT_LEAKY: act_all<DNXCU_ACT_LEAKY>(v, alpha); break;
    case DNXCU_ACT_GELU: act_all<DNXCU_ACT_GELU>(v, alpha); break;
    case DNXCU_ACT_GELU_TANH: act_all<DNXCU_ACT_GELU_TANH>(v, alpha); break;
    case DNXCU_ACT_SILU: act_all<DNXCU_ACT_SILU>(v, alpha); break;
    default: break;
  }
}

// ---- PTX that only these kernels use ----------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t mapped) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(mapped) : "memory");
}
// (x coordinates are multiples of 128 bytes throughout)
template <int CG>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const void *tmap, int c0, int c1, uint32_t bar) {
  if (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(dst),
        "l"(tmap), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(tmap), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_store_2d(const void *tmap, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(tmap), "r"(c0), "r"(c1),
               "r"(src)
               : "memory");
}
__device__ __forceinline__ void bulk_group_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_group_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_group_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Operand tiles: rows of 128 bytes (64 binary16 or 128 e4m3 channels) with the 128 byte swizzle, K major.  Descriptor:
// start address, 1024 bytes between groups of 8 rows, layout code 2.  A K step is 32 bytes for either type.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t operand_desc(uint32_t addr) { return (addr >> 4) | (1u << 16); }
// The MMA warp walks its loops as one warp, so that descriptors live in uniform registers; the lane with `leader` set
// alone issues.  Descriptors are a constant high word and a low word.
template <int CG, bool F8>
__device__ __forceinline__ void mma_step(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate,
                                         uint32_t leader) {
#define DNXCU_MMA(group, kind)                                                             \
  asm volatile(                                                                            \
      "{\n\t"                                                                              \
      ".reg .pred p, e;\n\t"                                                               \
      ".reg .b64 da, db;\n\t"                                                              \
      "mov.b64 da, {%1, %4};\n\t"                                                          \
      "mov.b64 db, {%2, %4};\n\t"                                                          \
      "setp.ne.b32 p, %5, 0;\n\t"                                                          \
      "setp.ne.b32 e, %6, 0;\n\t"                                                          \
      "@e tcgen05.mma.cta_group::" group ".kind::" kind " [%0], da, db, %3, p;\n\t"        \
      "}" ::"r"(d),                                                                        \
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(kDescHi), "r"(accumulate), "r"(leader)         \
      : "memory")
  if (CG == 2 && F8) DNXCU_MMA("2", "f8f6f4");
  else if (CG == 2) DNXCU_MMA("2", "f16");
  else if (F8) DNXCU_MMA("1", "f8f6f4");
  else DNXCU_MMA("1", "f16");
#undef DNXCU_MMA
}
// The `n` (1 to 4) steps of one stage, straight line code for each n: an MMA in a loop costs its thread about 200 cycles
// of issue, one in straight line code about 60 (522240 rows, 32 to 32 channels: 22.0 us with a loop, 20.6 without).
template <int CG, bool F8, int N>
__device__ __forceinline__ void mma_steps_n(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate, uint32_t leader) {
  mma_step<CG, F8>(d, a, b, idesc, accumulate, leader);
#pragma unroll
  for (int k = 1; k < N; ++k) mma_step<CG, F8>(d, a + 2 * k, b + 2 * k, idesc, 1u, leader);
}
template <int CG, bool F8>
__device__ __forceinline__ void mma_steps(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate, int n,
                                          uint32_t leader) {
  if (n == 4) mma_steps_n<CG, F8, 4>(d, a, b, idesc, accumulate, leader);
  else if (n == 2) mma_steps_n<CG, F8, 2>(d, a, b, idesc, accumulate, leader);
  else if (n == 1) mma_steps_n<CG, F8, 1>(d, a, b, idesc, accumulate, leader);
  else mma_steps_n<CG, F8, 3>(d, a, b, idesc, accumulate, leader);
}
// Arrives on `bar` (of both blocks of a pair) when the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t bar, uint32_t leader) {
  if (CG == 2)
    asm volatile(
        "{\n\t"
        ".reg .pred e;\n\t"
        "setp.ne.b32 e, %2, 0;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t"
        "}" ::"r"(bar),
        "h"((uint16_t)3), "r"(leader)
        : "memory");
  else
    asm volatile(
        "{\n\t"
        ".reg .pred e;\n\t"
        "setp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
        "}" ::"r"(bar),
        "r"(leader)
        : "memory");
}
// Bounded wait of a whole warp: the same answer in every lane.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, int *status, int code) {
  if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity) != 0)) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, code));
}
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t cols) {
  if (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
  if (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Instruction descriptor: 32 bit accumulators, both operands binary16 (0) or e4m3 (0 of the 8 bit kinds), K major.
__device__ __forceinline__ uint32_t mma_idesc(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// The MMA steps (32 bytes of channels each) of 128 byte step `kb`: 4 but for the last, whose rest the copies zero filled.
template <bool F8>
__device__ __forceinline__ int k_steps(const LinArgs &g, int kb) {
  const int bytes = (F8 ? g.K : 2 * g.K) - kb * 128;
  return bytes >= 128 ? 4 : (bytes + 31) / 32;
}

constexpr int MAX_STAGES = 12;
constexpr int MAX_BUFS = 4;  // accumulators in tensor memory
constexpr int HDR_FULL = 0, HDR_EMPTY = 8 * MAX_STAGES, HDR_TFULL = 16 * MAX_STAGES, HDR_TEMPTY = HDR_TFULL + 8 * MAX_BUFS,
              HDR_RES = HDR_TEMPTY + 8 * MAX_BUFS, HDR_WRES = HDR_RES + 64, HDR_TMEM = HDR_WRES + 8, HDR_ABORT = HDR_TMEM + 4;
static_assert((HDR_ABORT + 4) % 8 == 0 && HDR_ABORT + 12 <= 1024, "header layout");
constexpr int HEADER = 1024;
constexpr uint32_t kSmemLimit = 232448;

__device__ __forceinline__ uint32_t aligned_base(const void *dyn) { return (smem_u32(dyn) + 1023u) & ~1023u; }

// ---- TILE and ANY -----------------------------------------------------------
// Warps: 0 fetches operand tiles, 1 issues MMAs, 2 owns the tensor memory, 4-7 and 8-11 are two epilogue teams that take
// turns (or one that takes all); 2 or 4 accumulators rotate, so tiles are multiplied while the teams finish the ones
// before.  (Four teams, 96 registers each: 522240 rows, 32 to 32 channels 20.0 us, with two 19.1.)  ANY: seven warps (0, 2, 3, 12-15) fetch with plain loads instead, each a whole stage, so that as many
// stages are on their way at any time.  Where all of c_out is one column of tiles and the weights are small (a pointwise layer over pixels), they are
// fetched once per block and only rows of x stream.
constexpr int TILE_THREADS = 384, ANY_THREADS = 512;
constexpr int COLBUF = 512;              // per epilogue warp: bias and weight scale of 64 channels
constexpr int TILE_FIXED = HEADER + 8 * COLBUF;
constexpr int STAGING = 4096;            // per epilogue warp: 32 rows x 64 channels of binary16

struct TilePos {
  int m, n;
};
// Tiles in groups of `group` along the rows, so that the tiles in flight share operands in L2.
__device__ __forceinline__ TilePos tile_pos(const LinArgs &g, int t) {
  if (g.nt == 1) return {t, 0};
  const int per = g.group * g.nt, grp = t / per, r = t - grp * per;
  const int m0 = grp * g.group, gm = min(g.group, g.mt - m0);
  const int n = r / gm;
  return {m0 + r - n * gm, n};
}

// 16 bytes of an operand row at any alignment, zero beyond the row's end.  The aligned 16 byte words around the piece are
// read (between rows there are bytes of the same buffer) and shifted together; where such a word would reach outside the
// operand (`begin`, `end`: only at its two ends), single elements are read instead.
struct PieceReq {
  uint4 a, b;
  const uint8_t *p;
  int left;  // bytes of the row from the piece on
  bool slow;
};
__device__ __forceinline__ void request_piece(PieceReq &q, const uint8_t *p, int left, bool edge, const uint8_t *begin,
                                              const uint8_t *end) {
  q.left = left;
  q.p = p;
  q.a = q.b = make_uint4(0, 0, 0, 0);
  q.slow = false;
  if (left <= 0) return;
  const int sh = (int)((uintptr_t)p & 15), need = sh + min(left, 16);
  const uint8_t *w = p - sh;
  if (edge) q.slow = w < begin || w + (need > 16 ? 32 : 16) > end;
  if (q.slow) return;
  q.a = __ldg(reinterpret_cast<const uint4 *>(w));
  if (need > 16) q.b = __ldg(reinterpret_cast<const uint4 *>(w + 16));
}
template <bool F8>
__device__ __forceinline__ uint4 finish_piece(const PieceReq &q) {
  uint32_t w[8] = {q.a.x, q.a.y, q.a.z, q.a.w, q.b.x, q.b.y, q.b.z, q.b.w};
  if (q.slow) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = 0;
#pragma unroll
      for (int e = 0; e < (F8 ? 4 : 2); ++e) {
        const int at = i * 4 + e * (F8 ? 1 : 2);
        if (at < q.left)
          w[i] |= (F8 ? (uint32_t)__ldg(q.p + at) : (uint32_t)__ldg(reinterpret_cast<const uint16_t *>(q.p + at))) << (at % 4 * 8);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  const int sh = (int)((uintptr_t)q.p & 15);
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = sh & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = sh & 4 ? w[i + 1] : w[i];
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = __funnelshift_r(w[i], w[i + 1], (sh & 3) * 8);
  if (q.left < 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int keep = q.left - i * 4;  // bytes of this word that lie inside the row
      if (keep < 4) o[i] = keep <= 0 ? 0u : o[i] & (0xffffffffu >> (32 - 8 * keep));
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
// One warp fills `rows` rows (from row `row0` of an operand of `n` rows) of a swizzled tile: the first 2^LP 16 byte pieces
// of 128 byte step `kb` of each; of `step` warps that share the tile it is number `first`.
template <bool F8, int LP>
__device__ __forceinline__ void fill_pieces(uint32_t dst, const uint8_t *op, long long stride, long long row0, int n, int rows,
                                            int kb, int kbytes, int lane, int first, int step) {
  const uint8_t *end = op + (long long)(n - 1) * stride + kbytes, *at0 = op + row0 * stride + kb * 128;
  const bool edge = row0 == 0 || row0 + rows >= n;
  const int left_rows = (int)min((long long)rows, n - row0), items = rows << LP, left0 = kbytes - kb * 128;
  constexpr int B = 8;
  for (int i0 = first * 32 + lane; i0 < items; i0 += 32 * step * B) {
    PieceReq q[B];
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const int i = i0 + 32 * step * u, r = i >> LP, j = i & ((1 << LP) - 1);
      request_piece(q[u], at0 + r * stride + j * 16, r < left_rows ? left0 - j * 16 : 0, edge, op, end);
    }
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const int i = i0 + 32 * step * u, r = i >> LP, j = i & ((1 << LP) - 1);
      const uint4 v = finish_piece<F8>(q[u]);
      if (i < items) sts128(dst + (uint32_t)r * 128u + (uint32_t)((j ^ (r & 7)) << 4), v);
    }
  }
}
template <bool F8>
__device__ __forceinline__ void fill_tile(uint32_t dst, const uint8_t *op, long long stride, long long row0, int n, int rows,
                                          int ks, int kb, int kbytes, int lane, int first, int step) {
  if (ks > 2) fill_pieces<F8, 3>(dst, op, stride, row0, n, rows, kb, kbytes, lane, first, step);
  else if (ks == 2) fill_pieces<F8, 2>(dst, op, stride, row0, n, rows, kb, kbytes, lane, first, step);
  else fill_pieces<F8, 1>(dst, op, stride, row0, n, rows, kb, kbytes, lane, first, step);
}
// ANY: the warps that fetch, numbered.
constexpr int FETCHERS = 7;
__device__ __forceinline__ int fetcher(int warp) { return warp == 0 ? 0 : warp == 2 ? 1 : warp == 3 ? 2 : warp >= 12 ? warp - 9 : -1; }

// GROUPED: thin layers over packed rows (pixels).  `gr` rows side by side are one row of gr * c_in channels, whose product
// with the block diagonal of gr copies of the weights is the gr output rows side by side.  The zeros cost multiplications
// that nothing waits for; in return tiles are wide (a tile of 32 channels takes the epilogue nearly as long as one of 128),
// and rows off 16 byte boundaries become rows on them.  The block diagonal is put together in shared memory, once per block.
template <bool F8>
__device__ __forceinline__ void fill_grouped(uint32_t wres, uint32_t step_bytes, const LinArgs &g) {
  constexpr int E = F8 ? 16 : 8;  // channels per 16 byte piece
  const int per_row = g.kb * 8;
  for (int i = threadIdx.x; i < g.BN * per_row; i += (int)blockDim.x) {
    const int n = i / per_row, j = i - n * per_row, blk = n / g.n1, k0 = j * E - blk * g.k1;
    uint32_t v[4] = {0u, 0u, 0u, 0u};
    if (n < g.N && k0 + E > 0 && k0 < g.k1) {
      const uint8_t *w = g.w + (long long)(n - blk * g.n1) * g.ws;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (k0 + e >= 0 && k0 + e < g.k1) {
          if (F8) v[e >> 2] |= (uint32_t)__ldg(w + k0 + e) << (8 * (e & 3));
          else v[e >> 1] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t *>(w) + k0 + e) << (16 * (e & 1));
        }
    }
    sts128(wres + (uint32_t)(j >> 3) * step_bytes + (uint32_t)n * 128u + (uint32_t)(((j & 7) ^ (n & 7)) << 4),
           make_uint4(v[0], v[1], v[2], v[3]));
  }
}

// A warp's 32 staged rows (swizzled, 128 bytes apart) of `n` <= 64 channels from or to 32 packed rows, by 16 byte accesses.
__device__ __forceinline__ __half *staged_at(uint8_t *stg, int r, int j) {
  return reinterpret_cast<__half *>(stg + r * 128 + ((((j >> 3) ^ (r & 7)) << 4) | ((j & 7) << 1)));
}
template <bool OUT>
__device__ __forceinline__ void copy_packed(uint8_t *stg, __half *rows, int n, int lane) {
  union {
    uint4 v;
    __half h[8];
  } a;
  for (int i = lane; i < 4 * n; i += 32) {
    int r = 8 * i / n, j = 8 * i - r * n;
    if (!OUT) a.v = reinterpret_cast<const uint4 *>(rows)[i];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (OUT) a.h[e] = *staged_at(stg, r, j);
      else *staged_at(stg, r, j) = a.h[e];
      if (++j == n) {
        j = 0;
        ++r;
      }
    }
    if (OUT) reinterpret_cast<uint4 *>(rows)[i] = a.v;
  }
}

// A NaN or an infinity in one row of a group reaches the others through the zeros of the block diagonal.  Sums that are not
// finite are therefore taken again, each from its own row alone: channels [c, c + n) of grouped row `row`, over the staged
// results.  (Rare, and slow: one thread, one channel after the other.)
template <bool F8>
__device__ __forceinline__ void redo_row(const LinArgs &g, uint8_t *stg_p, int lane, long long row, int c, int n) {
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    const int blk = (c + j) / g.n1, ch = c + j - blk * g.n1;
    const uint8_t *x = g.x + row * g.xs + (long long)blk * g.k1 * (F8 ? 1 : 2), *w = g.w + (long long)ch * g.ws;
    float acc = 0.0f;
#pragma unroll 1
    for (int k = 0; k < g.k1; ++k) {
      if (F8) acc = fmaf(__half2float(__half(__nv_cvt_fp8_to_halfraw(x[k], __NV_E4M3))), __half2float(__half(__nv_cvt_fp8_to_halfraw(w[k], __NV_E4M3))), acc);
      else acc = fmaf(__half2float(reinterpret_cast<const __half *>(x)[k]), __half2float(reinterpret_cast<const __half *>(w)[k]), acc);
    }
    float v[1] = {fmaf(acc, g.w_scale ? __ldg(g.w_scale + ch) : 1.0f, g.bias ? __half2float(__ldg(g.bias + ch)) : 0.0f)};
    activate(v, g.act, g.alpha);
    if (g.res) v[0] += __half2float(g.res[row * g.rs + c + j]);
    *staged_at(stg_p, lane, j) = __float2half_rn(v[0]);
  }
}

// NARROW: rows of out or of the residual may be ones that no tensor map takes; a kernel of its own, because the code for
// them costs the others registers (frame 96 -> 64: 106 us without it, up to 129 with).
template <int CG, bool F8, bool ANY, bool NARROW, bool GROUPED>
__global__ void __launch_bounds__(ANY ? ANY_THREADS : TILE_THREADS, 1) linear_tile(const __grid_constant__ LinArgs g) {
  extern __shared__ uint8_t dyn[];
  const uint32_t base = aligned_base(dyn);
  uint8_t *hdr = dyn + (base - smem_u32(dyn));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(hdr + HDR_ABORT);
  const uint32_t b_rows = (uint32_t)g.BN / CG, b_bytes = b_rows * 128u;
  const uint32_t step_bytes = 16384u + (g.w_res ? 0u : b_bytes), stage_bytes = step_bytes * (uint32_t)g.per_stage;
  const uint32_t wres0 = base + TILE_FIXED, stage0 = wres0 + (g.w_res ? (uint32_t)g.kb * b_bytes : 0u);
  const uint32_t staging0 = stage0 + stage_bytes * (uint32_t)g.stages;
  const int ntiles = g.mt * g.nt, step = (int)gridDim.x / CG, first = (int)blockIdx.x / CG;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    *reinterpret_cast<volatile unsigned long long *>(abort_flag + 1) = g.wait_limit;
    for (int i = 0; i < MAX_STAGES; ++i) {
      mbar_init(base + HDR_FULL + 8 * i, 1);
      mbar_init(base + HDR_EMPTY + 8 * i, 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(base + HDR_RES + 8 * i, 1);
    mbar_init(base + HDR_WRES, ANY ? FETCHERS : 1);
    for (int i = 0; i < MAX_BUFS; ++i) {
      mbar_init(base + HDR_TFULL + 8 * i, 1);
      mbar_init(base + HDR_TEMPTY + 8 * i, 4 * CG);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (!ANY) {
      tma_prefetch_map(&g.tm_x);
      tma_prefetch_map(&g.tm_w);
    }
    if (g.out_tma) tma_prefetch_map(&g.tm_out);
    if (g.res_tma) tma_prefetch_map(&g.tm_res);
  }
  if (CG == 2) cluster_sync();  // both blocks run before either touches the pair's tensor memory or barriers
  if (warp == 2) tmem_alloc<CG>(base + HDR_TMEM, 512);
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(hdr + HDR_TMEM);
  pdl_release();  // (after the allocation: blocks that wait for this kernel may hold tensor memory)
  pdl_wait();
  if (GROUPED) {
    fill_grouped<F8>(wres0, b_bytes, g);
    fence_proxy_async();
    __syncthreads();
  }

  if (!ANY && warp == 0) {
    // ---- operand tiles by TMA; the pair's bytes are counted on the first block's barrier ----
    if (lane == 0) {
      if (g.w_res && !GROUPED) {
        mbar_expect_tx(base + HDR_WRES, (uint32_t)g.kb * b_bytes);
        for (int kb = 0; kb < g.kb; ++kb)
          tma_load_2d<1>(wres0 + (uint32_t)kb * b_bytes, &g.tm_w, kb * (F8 ? 128 : 64), 0, base + HDR_WRES);
      }
      int s = 0;
      uint32_t ph = 1;
      bool ok = true;
      for (int t = first; ok && t < ntiles; t += step) {
        const TilePos p = tile_pos(g, t);
        const int row_a = p.m * (128 * CG) + (int)rank * 128, row_b = p.n * g.BN + (int)(rank * b_rows);
        for (int kb = 0; kb < g.kb;) {
          ok = mbar_wait(base + HDR_EMPTY + 8 * s, ph, abort_flag, g.status, 12);
          if (!ok) break;
          const uint32_t full = base + HDR_FULL + 8 * s;
          const int end = min(kb + g.per_stage, g.kb);
          if (rank == 0) mbar_expect_tx(full, step_bytes * (uint32_t)(end - kb) * CG);
          const uint32_t bar = CG == 2 ? map_rank(full, 0) : full;
          uint32_t a = stage0 + stage_bytes * (uint32_t)s;
          for (; kb < end; ++kb, a += step_bytes) {
            tma_load_2d<CG>(a, &g.tm_x, kb * (F8 ? 128 : 64), row_a, bar);
            if (!g.w_res) tma_load_2d<CG>(a + 16384u, &g.tm_w, kb * (F8 ? 128 : 64), row_b, bar);
          }
          if (++s == g.stages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
    }
  } else if (ANY && fetcher(warp) >= 0) {
    // ---- operand tiles by plain loads, swizzled as the copy engine would ----
    const int pw = fetcher(warp);
    const int kbytes = F8 ? g.K : 2 * g.K;
    if (g.w_res) {
      for (int kb = 0; kb < g.kb; ++kb)
        fill_tile<F8>(wres0 + (uint32_t)kb * b_bytes, g.w, g.ws, 0, g.N, g.BN, k_steps<F8>(g, kb), kb, kbytes, lane, pw, FETCHERS);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(base + HDR_WRES);
    }
    // At most as many warps take turns as there are stages: a warp that takes block j has then waited for block
    // j - 2 * stages to be consumed, so the stage's barrier is at most one phase behind and its parity says enough.
    const int turns = min(FETCHERS, g.stages);
    int s = 0, turn = 0;
    uint32_t ph = 1;
    bool ok = pw < turns;
    for (int t = first; ok && t < ntiles; t += step) {
      const TilePos p = tile_pos(g, t);
      for (int kb0 = 0; kb0 < g.kb; kb0 += g.per_stage) {
        if (turn == pw) {
          ok = mbar_wait(base + HDR_EMPTY + 8 * s, ph, abort_flag, g.status, 12);
          ok = __all_sync(0xffffffffu, ok);  // (the warp leaves the loop as one)
          if (!ok) break;
          uint32_t a = stage0 + stage_bytes * (uint32_t)s;
          for (int kb = kb0; kb < min(kb0 + g.per_stage, g.kb); ++kb, a += step_bytes) {
            const int ks = k_steps<F8>(g, kb);
            fill_tile<F8>(a, g.x, g.xs, (long long)p.m * 128, g.M, 128, ks, kb, kbytes, lane, 0, 1);
            if (!g.w_res) fill_tile<F8>(a + 16384u, g.w, g.ws, (long long)p.n * g.BN, g.N, g.BN, ks, kb, kbytes, lane, 0, 1);
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(base + HDR_FULL + 8 * s);
        }
        turn = turn + 1 == turns ? 0 : turn + 1;
        if (++s == g.stages) {
          s = 0;
          ph ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    // ---- MMA issue: one warp of the (first) block ----
    if (rank == 0) {
      const uint32_t leader = lane == 0, idesc = mma_idesc(128 * CG, g.BN);
      const int last = k_steps<F8>(g, g.kb - 1);
      const uint32_t a0 = operand_desc(stage0), a_stage = stage_bytes >> 4, a_step = step_bytes >> 4;
      const uint32_t w0 = operand_desc(wres0), w_step = b_bytes >> 4;
      int s = 0, buf = 0;
      uint32_t ph = 0, bph = 1, a_s = a0;
      bool ok = !g.w_res || GROUPED || warp_wait(base + HDR_WRES, 0, abort_flag, g.status, 11);
      for (int t = first; ok && t < ntiles; t += step) {
        const uint32_t d = tmem + (uint32_t)(buf * g.BN);
        ok = warp_wait(base + HDR_TEMPTY + 8 * buf, bph, abort_flag, g.status, 14);
        if (!ok) break;
        tc_fence_after();
        uint32_t w = w0;
        for (int kb = 0; kb < g.kb;) {
          ok = warp_wait(base + HDR_FULL + 8 * s, ph, abort_flag, g.status, 11);
          if (!ok) break;
          tc_fence_after();
          uint32_t a = a_s;
          mma_steps<CG, F8>(d, a, g.w_res ? w : a + (16384u >> 4), idesc, kb != 0, kb + 1 < g.kb ? 4 : last, leader);
          w += w_step;
          ++kb;
          if (g.per_stage == 2 && kb < g.kb) {
            a += a_step;
            mma_steps<CG, F8>(d, a, g.w_res ? w : a + (16384u >> 4), idesc, 1u, kb + 1 < g.kb ? 4 : last, leader);
            w += w_step;
            ++kb;
          }
          // (the tile's last stage is handed back by the epilogue, which learns of it by the tile's own commit; ANY needs
          // the stages back in order)
          if (ANY || kb < g.kb) mma_commit<CG>(base + HDR_EMPTY + 8 * s, leader);
          a_s += a_stage;
          if (++s == g.stages) {
            s = 0;
            a_s = a0;
            ph ^= 1;
          }
        }
        if (!ok) break;
        mma_commit<CG>(base + HDR_TFULL + 8 * buf, leader);
        if (++buf == g.bufs) {
          buf = 0;
          bph ^= 1;
        }
      }
    }
  } else if (warp >= 4 && warp < 4 + 4 * g.teams) {
    // ---- epilogue: 32 rows x 64 channels at a time through a swizzled staging tile ----
    const int ew = warp - 4, team = ew >> 2, q = warp & 3;
    const uint32_t stg = staging0 + (uint32_t)ew * STAGING;
    uint8_t *stg_p = hdr + (stg - base);
    float *col_b = reinterpret_cast<float *>(hdr + HEADER + ew * COLBUF), *col_s = col_b + 64;
    const uint32_t rbar = base + HDR_RES + 8 * ew;
    const uint32_t my = stg + (uint32_t)lane * 128u;
    const auto staged = [&](int r, int j) {  // channel j of row r in the staging tile
      return staged_at(stg_p, r, j);
    };
    uint32_t rph = 0, bph = 0;
    bool ok = true;
    const int tile_stages = (g.kb + g.per_stage - 1) / g.per_stage % g.stages;
    int turn = 0, buf = 0, s = 0;  // s: the stage after the tile's last one
    bool fresh = true;  // the team's first tile
    for (int t = first; ok && t < ntiles; t += step) {
      s += tile_stages;
      if (s >= g.stages) s -= g.stages;
      const int my_buf = buf;
      const uint32_t my_ph = bph;
      if (++buf == g.bufs) {
        buf = 0;
        bph ^= 1;
      }
      const bool ours = turn == team;
      if (++turn == g.teams) turn = 0;
      if (!ours) continue;
      const TilePos p = tile_pos(g, t);
      const int n0 = p.n * g.BN, nc = min(g.BN, g.N - n0);
      const long long row0 = (long long)p.m * (128 * CG) + (long long)rank * 128 + q * 32, row = row0 + lane;
      const bool live = row0 < g.M;
      const float xs = (g.x_scale && row < g.M) ? __ldg(g.x_scale + row) : 1.0f;
      // What 64 channels need besides the sums: bias, scales and the residual, which goes into the staging tile.
      const auto prepare = [&](int c) {
        if (lane == 0) bulk_group_wait_read();  // the staging tile's last store has read it
        if (g.nt > 1 || g.BN > 64 || fresh)  // (else they are there from the team's first tile)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int j = lane + 32 * h, n = n0 + c + j, n1 = GROUPED ? n % g.n1 : n;
          col_b[j] = (g.bias && n < g.N) ? __half2float(__ldg(g.bias + n1)) : 0.0f;
          col_s[j] = (g.w_scale && n < g.N) ? __ldg(g.w_scale + n1) : 1.0f;
        }
        __syncwarp();
        if (g.res_tma) {
          if (lane == 0) {
            mbar_expect_tx(rbar, STAGING);
            tma_load_2d<1>(stg, &g.tm_res, n0 + c, (int)row0, rbar);
          }
        } else if (NARROW && g.res_pack && row0 + 32 <= g.M) {
          copy_packed<false>(stg_p, const_cast<__half *>(g.res) + row0 * g.N, g.N, lane);
          __syncwarp();
        } else if (NARROW && g.res) {
          // (rows that no tensor map takes: 2 byte loads, 32 of them on their way)
#pragma unroll
          for (int r0 = 0; r0 < 32; r0 += 16) {
            __half v[16][2];
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const bool in = row0 + r0 + r < g.M && c + lane + 32 * h < nc;
                v[r][h] = in ? g.res[(row0 + r0 + r) * g.rs + n0 + c + lane + 32 * h] : __half();
              }
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
              for (int h = 0; h < 2; ++h) *staged(r0 + r, lane + 32 * h) = v[r][h];
          }
          __syncwarp();
        }
      };
      if (live) prepare(0);  // (under the tile's products)
      fresh = false;
      ok = mbar_wait(base + HDR_TFULL + 8 * my_buf, my_ph, abort_flag, g.status, 13);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      if (!ANY && q == 0 && lane == 0) mbar_arrive(base + HDR_EMPTY + 8 * (s == 0 ? g.stages - 1 : s - 1));
      const uint32_t acc = tmem + (uint32_t)(my_buf * g.BN) + ((uint32_t)(q * 32) << 16);
      for (int c = 0; live && c < nc; c += 64) {
        if (c > 0) prepare(c);
        if (g.res_tma) {
          ok = mbar_wait(rbar, rph, abort_flag, g.status, 15);
          rph ^= 1;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        float zero = 0.0f;  // (GROUPED: stays zero while every sum is finite)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (c + 32 * h >= nc) break;  // (uniform)
          uint32_t raw[32];
          tc_ld32(acc + (uint32_t)(c + 32 * h), raw);
          tc_wait_ld();
          if (GROUPED) {
#pragma unroll
            for (int i = 0; i < 32; ++i) zero = fmaf(__uint_as_float(raw[i]), 0.0f, zero);
          }
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 sc = *reinterpret_cast<const float4 *>(col_s + 32 * h + i);
            const float4 bi = *reinterpret_cast<const float4 *>(col_b + 32 * h + i);
            v[i] = fmaf(__uint_as_float(raw[i]) * xs, sc.x, bi.x);
            v[i + 1] = fmaf(__uint_as_float(raw[i + 1]) * xs, sc.y, bi.y);
            v[i + 2] = fmaf(__uint_as_float(raw[i + 2]) * xs, sc.z, bi.z);
            v[i + 3] = fmaf(__uint_as_float(raw[i + 3]) * xs, sc.w, bi.w);
          }
          activate(v, g.act, g.alpha);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t at = my + (uint32_t)(((4 * h + j) ^ (lane & 7)) << 4);
            if (g.res) {
              const uint4 r = lds128(at);
              const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&rw[e]));
                v[8 * j + 2 * e] += f.x;
                v[8 * j + 2 * e + 1] += f.y;
              }
            }
            sts128(at, make_uint4(pack_h2(v[8 * j], v[8 * j + 1]), pack_h2(v[8 * j + 2], v[8 * j + 3]),
                                  pack_h2(v[8 * j + 4], v[8 * j + 5]), pack_h2(v[8 * j + 6], v[8 * j + 7])));
          }
        }
        if (GROUPED && !(zero == 0.0f) && row < g.M) redo_row<F8>(g, stg_p, lane, row, c, min(64, nc - c));
        // (a store through the tensor map writes whole 16 byte pieces: not for a row that ends inside one)
        if (!NARROW || (g.out_tma && (c + 64 <= nc || (g.N & 7) == 0))) {
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&g.tm_out, stg, n0 + c, (int)row0);
            bulk_group_commit();
          }
        } else if (g.out_pack && row0 + 32 <= g.M) {
          __syncwarp();
          copy_packed<true>(stg_p, g.out + row0 * g.N, g.N, lane);
          fence_proxy_async();
        } else {
          __syncwarp();
#pragma unroll 8
          for (int r = 0; r < 32; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (row0 + r < g.M && c + lane + 32 * h < nc)
                g.out[(row0 + r) * g.os + n0 + c + lane + 32 * h] = *staged(r, lane + 32 * h);
          fence_proxy_async();  // (the next residual box comes through the copy engine)
        }
        __syncwarp();
      }
      // the accumulator goes back to the issuing thread
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        const uint32_t te = base + HDR_TEMPTY + 8 * my_buf;
        if (CG == 2) mbar_arrive_cluster(map_rank(te, 0));
        else mbar_arrive(te);
      }
    }
    if (lane == 0) bulk_group_wait();
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  abort_drain(abort_flag);
  if (CG == 2) cluster_sync();
  if (warp == 2) tmem_free<CG>(tmem, 512);
}

// ---- SPLIT ------------------------------------------------------------------
// One tile of 128 output channels x BN rows per cluster; block r of the cluster takes the r-th part of c_in.  The
// accumulator's lanes are output channels, its columns rows of x.  Rows are dealt out over the cluster for the epilogue:
// every block sends each row's partial sums to the block that finishes it (distributed shared memory, [source][row][128
// channels]), and that block adds them in rank order, so the bits do not depend on timing.  Sending instead of fetching
// leaves one cluster barrier on the path and none at the end (the receiving block's own memory is all that is read).
constexpr int SPLIT_THREADS = 256;
constexpr int SPLIT_FIXED = HEADER + 1024;  // header, x scales of the block's rows

template <bool F8>
__global__ void __launch_bounds__(SPLIT_THREADS) linear_split(const __grid_constant__ LinArgs g) {
  extern __shared__ uint8_t dyn[];
  const uint32_t base = aligned_base(dyn);
  uint8_t *hdr = dyn + (base - smem_u32(dyn));
  float *s_xs = reinterpret_cast<float *>(hdr + HEADER);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(hdr + HDR_ABORT);
  const int S = g.split, rank = (int)blockIdx.x % S, ft = (int)blockIdx.x / S;
  const int n0 = ft * 128, m0 = (int)blockIdx.y * g.BN;
  const int kb0 = (int)((long long)g.kb * rank / S), kb1 = (int)((long long)g.kb * (rank + 1) / S);
  const uint32_t stage_bytes = 16384u + (uint32_t)g.BN * 128u, stage0 = base + SPLIT_FIXED;
  const uint32_t recv = stage0 + (g.overlay ? 0u : stage_bytes * (uint32_t)g.stages);
  const uint32_t cols = g.BN <= 32 ? 32u : g.BN <= 64 ? 64u : g.BN <= 128 ? 128u : 256u;
  const int rows = min(g.BN, g.M - m0), per = (rows + S - 1) / S;  // this tile's rows; rows a block finishes
  const int mine = max(0, min(per, rows - rank * per));

  // The steps are walked from a start that differs from tile to tile: blocks that stream rows of the same pitch in step
  // would all ask for the same columns, the same few memory channels, at once.
  const int nkb = kb1 - kb0, rot = (ft * 5) % nkb;
  const auto step_of = [&](int i) { return kb0 + (i + rot < nkb ? i + rot : i + rot - nkb); };
  const auto fetch = [&](int i, int s) {
    const uint32_t full = base + HDR_FULL + 8 * s, a = stage0 + stage_bytes * (uint32_t)s;
    const int x = step_of(i) * (F8 ? 128 : 64);
    mbar_expect_tx(full, stage_bytes);
    tma_load_2d<1>(a, &g.tm_w, x, n0, full);
    tma_load_2d<1>(a + 16384u, &g.tm_x, x, m0, full);
  };
  const int early = min(2, nkb);
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    *reinterpret_cast<volatile unsigned long long *>(abort_flag + 1) = g.wait_limit;
    for (int i = 0; i < MAX_STAGES; ++i) {
      mbar_init(base + HDR_FULL + 8 * i, 1);
      mbar_init(base + HDR_EMPTY + 8 * i, 1);
    }
    mbar_init(base + HDR_TFULL, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tma_prefetch_map(&g.tm_w);
    tma_prefetch_map(&g.tm_x);
    pdl_wait();
    // the first copies need nothing but the barriers: they are on their way while the rest is set up
    for (int i = 0; i < early; ++i) fetch(i, i);
  }
  if (warp == 2) tmem_alloc<1>(base + HDR_TMEM, cols);
  pdl_wait();
  if (warp == 3)
    for (int i = lane; i < mine; i += 32) s_xs[i] = g.x_scale ? __ldg(g.x_scale + m0 + rank * per + i) : 1.0f;
  // the four channels this thread will finish, in every row it finishes
  const int f = lane * 4, n = n0 + f;
  float bias[4], wsc[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    bias[e] = g.bias && n + e < g.N ? __half2float(__ldg(g.bias + n + e)) : 0.0f;
    wsc[e] = g.w_scale && n + e < g.N ? __ldg(g.w_scale + n + e) : 1.0f;
  }
  tc_fence_before();
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (waited for before the first remote store)
  tc_fence_after();
  // Only now, with its tensor memory in hand, does a block let the next kernel start: blocks of that one wait for this one
  // while they hold theirs.
  pdl_release();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(hdr + HDR_TMEM);

  if (warp == 0) {
    if (lane == 0) {
      int s = early % g.stages;
      uint32_t ph = early < g.stages ? 1 : 0;
      for (int i = early; i < nkb; ++i) {
        if (!mbar_wait(base + HDR_EMPTY + 8 * s, ph, abort_flag, g.status, 12)) break;
        fetch(i, s);
        if (++s == g.stages) {
          s = 0;
          ph ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    const uint32_t leader = lane == 0, idesc = mma_idesc(128, g.BN);
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int i = 0; i < nkb; ++i) {
      ok = warp_wait(base + HDR_FULL + 8 * s, ph, abort_flag, g.status, 11);
      if (!ok) break;
      tc_fence_after();
      const uint32_t a = operand_desc(stage0 + stage_bytes * (uint32_t)s);
      mma_steps<1, F8>(tmem, a, a + (16384u >> 4), idesc, i > 0, k_steps<F8>(g, step_of(i)), leader);
      mma_commit<1>(base + HDR_EMPTY + 8 * s, leader);
      if (++s == g.stages) {
        s = 0;
        ph ^= 1;
      }
    }
    if (ok) mma_commit<1>(base + HDR_TFULL, leader);
  }
  __syncwarp();
  bool ok = mbar_wait(base + HDR_TFULL, 0, abort_flag, g.status, 13);
  ok = __all_sync(0xffffffffu, ok);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (g.overlay) cluster_sync();  // the received rows lie over the stages: every block is done with its own
  if (ok) {
    tc_fence_after();
    const int q = warp & 3;
    for (int c = (warp >> 2) * 16; c < rows; c += 32) {
      uint32_t raw[16];
      tc_ld16(tmem + (uint32_t)c + ((uint32_t)(q * 32) << 16), raw);
      tc_wait_ld();
      int to = c / per, r = c - to * per;
      const uint32_t mine0 = recv + (uint32_t)(rank * per * 128 + q * 32 + lane) * 4u;
      uint32_t dst = map_rank(mine0, (uint32_t)to) + (uint32_t)r * 512u;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (c + i < rows) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(dst), "r"(raw[i]) : "memory");
        dst += 512u;
        if (++r == per && c + i + 1 < rows) {
          r = 0;
          dst = map_rank(mine0, (uint32_t)++to);
        }
      }
    }
  }
  tc_fence_before();
  cluster_sync();  // (every block of the cluster comes here, aborted or not)
  tc_fence_after();
  abort_drain(abort_flag);
  if (warp == 2) tmem_free<1>(tmem, cols);
  const bool whole = n + 4 <= g.N && !(g.os & 3) && !((uintptr_t)g.out & 7);  // four channels by one store
  constexpr int R = 4, WARPS = SPLIT_THREADS / 32;  // rows a warp finishes at once
  for (int r0 = warp; r0 < mine && n < g.N; r0 += R * WARPS) {
    float v[4 * R], res[4 * R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const int r = r0 + u * WARPS;
      const __half *rp = g.res + (long long)(m0 + rank * per + r) * g.rs + n;
#pragma unroll
      for (int e = 0; e < 4; ++e) res[4 * u + e] = g.res && r < mine && n + e < g.N ? __half2float(rp[e]) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 4 * R; ++i) v[i] = 0.0f;
    for (int b = 0; b < S; ++b)
#pragma unroll
      for (int u = 0; u < R; ++u) {
        const int r = min(r0 + u * WARPS, mine - 1);
        const uint4 p = lds128(recv + (uint32_t)((b * per + r) * 128 + f) * 4u);
        v[4 * u] += __uint_as_float(p.x);
        v[4 * u + 1] += __uint_as_float(p.y);
        v[4 * u + 2] += __uint_as_float(p.z);
        v[4 * u + 3] += __uint_as_float(p.w);
      }
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const float xs = s_xs[min(r0 + u * WARPS, mine - 1)];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * u + e] = fmaf(v[4 * u + e] * xs, wsc[e], bias[e]);
    }
    activate(v, g.act, g.alpha);
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const int r = r0 + u * WARPS;
      if (r >= mine) break;
      if (g.res) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * u + e] += res[4 * u + e];
      }
      __half *o = g.out + (long long)(m0 + rank * per + r) * g.os + n;
      if (whole) {
        *reinterpret_cast<uint2 *>(o) = make_uint2(pack_h2(v[4 * u], v[4 * u + 1]), pack_h2(v[4 * u + 2], v[4 * u + 3]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < g.N) o[e] = __float2half_rn(v[4 * u + e]);
      }
    }
  }
}

// ---- ROWS -------------------------------------------------------------------
// 16 output channels per block, c_in split over its 8 warps.  mma m16n8k16 with 16 weight rows as operand A and 8 rows of
// x as operand B.  The order of the channels inside a sum is free, so every lane loads 16 consecutive bytes of a row and
// both operands use the same permutation of the channels.  e4m3 becomes binary16 on the way (exactly).
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ld_stream(const uint8_t *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t e4m3_to_h2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)two));
  return r;
}

constexpr int ROWS_THREADS = 256;
// A lane's share of one 64 channel chunk of a row: binary16: bytes 16 t and 64 + 16 t of its 128; e4m3: bytes 16 t of 64.
template <bool F8>
struct Piece {
  uint4 v[F8 ? 1 : 2];
};
// The two registers (4 channels) that the piece gives to MMA step `s` of 4.
template <bool F8>
__device__ __forceinline__ void step_regs(const Piece<F8> &p, int s, uint32_t &r0, uint32_t &r1) {
  if (F8) {
    const uint32_t w = s == 0 ? p.v[0].x : s == 1 ? p.v[0].y : s == 2 ? p.v[0].z : p.v[0].w;
    r0 = e4m3_to_h2(w & 0xffffu);
    r1 = e4m3_to_h2(w >> 16);
  } else {
    const uint4 &v = p.v[(s >> 1) % (F8 ? 1 : 2)];
    r0 = s & 1 ? v.z : v.x;
    r1 = s & 1 ? v.w : v.y;
  }
}
// MT groups of 16 output channels, NT groups of 8 rows of x; w[i] and x[i] are the rows of the lane's group in them.
template <bool F8, int NT, int MT>
struct RowsChunk {
  Piece<F8> w[2 * MT], x[NT];
};
template <bool F8, int NT, int MT>
struct RowsPtr {
  const uint8_t *w[2 * MT], *x[NT];
  bool have[NT];
};
// TAIL: the row may end inside the chunk, at a 16 byte boundary.
template <bool F8, int NT, int MT, bool TAIL>
__device__ __forceinline__ void rows_load(RowsChunk<F8, NT, MT> &r, const RowsPtr<F8, NT, MT> &p, int chunk, int t, int kbytes) {
#pragma unroll
  for (int i = 0; i < (F8 ? 1 : 2); ++i) {
    const int at = chunk * (F8 ? 64 : 128) + i * 64 + t * 16;
    const bool in = !TAIL || at < kbytes;
#pragma unroll
    for (int m = 0; m < 2 * MT; ++m) {
      r.w[m].v[i] = make_uint4(0, 0, 0, 0);
      if (in) r.w[m].v[i] = ld_stream(p.w[m] + at);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      r.x[n].v[i] = make_uint4(0, 0, 0, 0);
      if (in && p.have[n]) r.x[n].v[i] = __ldg(reinterpret_cast<const uint4 *>(p.x[n] + at));
    }
  }
}
template <bool F8, int NT, int MT>
__device__ __forceinline__ void rows_mma(const RowsChunk<F8, NT, MT> &r, float (&acc)[MT][NT][4]) {
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      uint32_t a0, a1, a2, a3;
      step_regs<F8>(r.w[2 * m], s, a0, a2);
      step_regs<F8>(r.w[2 * m + 1], s, a1, a3);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint32_t b0, b1;
        step_regs<F8>(r.x[n], s, b0, b1);
        mma_16816(acc[m][n], a0, a1, a2, a3, b0, b1);
      }
    }
}

// U chunks of 64 channels are on their way per warp at any time.
template <bool F8, int NT, int MT, int U, bool ANY>
__global__ void __launch_bounds__(ROWS_THREADS, 2) linear_rows(const __grid_constant__ LinArgs g) {
  __shared__ float part[8][16 * MT][8 * NT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t = lane & 3;
  const int f0 = (int)blockIdx.x * 16 * MT;
  const int kbytes = F8 ? g.K : 2 * g.K;
  const int chunks = (g.K + 63) / 64, whole = g.K / 64;
  RowsPtr<F8, NT, MT> p;
#pragma unroll
  for (int m = 0; m < 2 * MT; ++m) p.w[m] = g.w + (long long)min(f0 + 8 * m + gr, g.N - 1) * g.ws;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    p.have[n] = n * 8 + gr < g.M;
    p.x[n] = g.x + (p.have[n] ? (long long)(n * 8 + gr) * g.xs : 0);
  }
  float acc[MT][NT][4] = {};
  int c = warp;
  pdl_release();
  pdl_wait();
  if (!ANY) {
    for (; c + 8 * (U - 1) < whole; c += 8 * U) {
      RowsChunk<F8, NT, MT> r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) rows_load<F8, NT, MT, false>(r[u], p, c + 8 * u, t, kbytes);
#pragma unroll
      for (int u = 0; u < U; ++u) rows_mma<F8, NT, MT>(r[u], acc);
    }
    for (; c < chunks; c += 8) {
      RowsChunk<F8, NT, MT> r;
      rows_load<F8, NT, MT, true>(r, p, c, t, kbytes);
      rows_mma<F8, NT, MT>(r, acc);
    }
  } else {
    const uint8_t *wend = g.w + (long long)(g.N - 1) * g.ws + kbytes, *xend = g.x + (long long)(g.M - 1) * g.xs + kbytes;
    for (; c < chunks; c += 8) {
      constexpr int H = F8 ? 1 : 2;
      PieceReq qw[2 * MT][H], qx[NT][H];
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const int at = c * (F8 ? 64 : 128) + i * 64 + t * 16;
#pragma unroll
        for (int m = 0; m < 2 * MT; ++m) request_piece(qw[m][i], p.w[m] + at, kbytes - at, true, g.w, wend);
#pragma unroll
        for (int n = 0; n < NT; ++n) request_piece(qx[n][i], p.x[n] + at, p.have[n] ? kbytes - at : 0, true, g.x, xend);
      }
      RowsChunk<F8, NT, MT> r;
#pragma unroll
      for (int i = 0; i < H; ++i) {
#pragma unroll
        for (int m = 0; m < 2 * MT; ++m) r.w[m].v[i] = finish_piece<F8>(qw[m][i]);
#pragma unroll
        for (int n = 0; n < NT; ++n) r.x[n].v[i] = finish_piece<F8>(qx[n][i]);
      }
      rows_mma<F8, NT, MT>(r, acc);
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      part[warp][16 * m + gr][n * 8 + 2 * t] = acc[m][n][0];
      part[warp][16 * m + gr][n * 8 + 2 * t + 1] = acc[m][n][1];
      part[warp][16 * m + gr + 8][n * 8 + 2 * t] = acc[m][n][2];
      part[warp][16 * m + gr + 8][n * 8 + 2 * t + 1] = acc[m][n][3];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * MT * 8 * NT; i += ROWS_THREADS) {
    const int f = i % (16 * MT), m = i / (16 * MT), n = f0 + f;
    if (m >= g.M || n >= g.N) continue;
    float v[1] = {0.0f};
#pragma unroll
    for (int w = 0; w < 8; ++w) v[0] += part[w][f][m];
    v[0] = fmaf(v[0] * (g.x_scale ? __ldg(g.x_scale + m) : 1.0f), g.w_scale ? __ldg(g.w_scale + n) : 1.0f,
                g.bias ? __half2float(__ldg(g.bias + n)) : 0.0f);
    activate(v, g.act, g.alpha);
    if (g.res) v[0] += __half2float(g.res[m * g.rs + n]);
    g.out[m * g.os + n] = __float2half_rn(v[0]);
  }
}

// ---- operands that no copy engine takes, laid out anew -----------------------
// Rows of any alignment to rows on 16 byte boundaries (what lies behind a row's end in its last piece is zero).  x and the
// weights in one launch: groups of rows [0, groups[0]) are the first operand's.
struct RelayArgs {
  const uint8_t *src[2];
  uint8_t *dst[2];
  long long stride[2], pitch;  // bytes per source row, per laid out row
  int rows[2], groups[2];
  int kbytes, per_row;         // 16 byte pieces per row
  int per_group;               // rows per group: about 1024 pieces
  uint32_t magic;              // 2^32 / per_row, rounded up (0 for 1): quotients of up to 2047 pieces are exact
};
template <bool F8>
__global__ void __launch_bounds__(256) linear_relay(const RelayArgs g) {
  constexpr int B = 4;
  for (int grp = (int)blockIdx.x; grp < g.groups[0] + g.groups[1]; grp += (int)gridDim.x) {
    const int o = grp >= g.groups[0], r0 = (o ? grp - g.groups[0] : grp) * g.per_group;
    const int rows = min(g.per_group, g.rows[o] - r0), pieces = rows * g.per_row;
    const uint8_t *src = g.src[o] + (long long)r0 * g.stride[o];
    const uint8_t *end = g.src[o] + (long long)(g.rows[o] - 1) * g.stride[o] + g.kbytes;
    uint8_t *dst = g.dst[o] + (long long)r0 * g.pitch;
    const bool edge = r0 == 0 || r0 + rows == g.rows[o];
    for (int i0 = threadIdx.x; i0 < pieces; i0 += 256 * B) {
      PieceReq q[B];
      long long to[B];
#pragma unroll
      for (int u = 0; u < B; ++u) {
        const int i = i0 + 256 * u, r = rows == 1 ? 0 : g.magic ? (int)__umulhi((uint32_t)i, g.magic) : i, at = (i - r * g.per_row) * 16;
        to[u] = (long long)r * g.pitch + at;
        request_piece(q[u], src + (long long)r * g.stride[o] + at, i < pieces ? g.kbytes - at : 0, edge, g.src[o], end);
      }
#pragma unroll
      for (int u = 0; u < B; ++u) {
        const uint4 v = finish_piece<F8>(q[u]);
        if (i0 + 256 * u < pieces) *reinterpret_cast<uint4 *>(dst + to[u]) = v;
      }
    }
  }
}

// ---- host side --------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
  static std::once_flag once;
  static EncodeTiledFn fn = nullptr;
  std::call_once(once, [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (EncodeTiledFn)p;
  });
  return fn;
}
// rows x cols matrix; box of 128 bytes x box_rows with the 128 byte swizzle; what lies outside reads as zero and is
// dropped when written.
int matrix_map(CUtensorMap *tm, const void *ptr, bool bytes, long long rows, long long cols, long long stride_bytes,
               int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return DNXCU_E_CUDA;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride_bytes};
  const cuuint32_t box[2] = {bytes ? 128u : 64u, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  CUresult r = CUDA_SUCCESS;
  for (int attempt = 0; attempt < 2; ++attempt) {
    r = fn(tm, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(ptr), dims,
           strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if ((r != CUDA_ERROR_INVALID_CONTEXT && r != CUDA_ERROR_NOT_INITIALIZED) || cudaFree(nullptr) != cudaSuccess) break;
  }
  return r == CUDA_SUCCESS ? DNXCU_OK : DNXCU_E_CUDA;
}
// What a copy through a tensor map asks of a matrix: base and rows on 16 byte boundaries (a single row has no pitch that
// matters, but the map wants one).
bool mappable(const void *p, long long stride_bytes) { return !((uintptr_t)p & 15) && !(stride_bytes & 15); }

struct Rec {  // a checked record: packed strides filled in
  dnxcu_linear d;
  bool f8;
  int es;
};

int check(const dnxcu_linear *d, Rec *r) {
  if (!d || !d->x || !d->weights || !d->out || d->rows <= 0 || d->c_in <= 0 || d->c_out <= 0) return DNXCU_E_BAD_ARG;
  if (d->dtype != DNXCU_DT_F16 && d->dtype != DNXCU_DT_E4M3) return DNXCU_E_BAD_ARG;
  if (d->activation < DNXCU_ACT_NONE || d->activation > DNXCU_ACT_SILU) return DNXCU_E_BAD_ARG;
  if (d->variant < DNXCU_LINEAR_AUTO || d->variant > DNXCU_LINEAR_ANY) return DNXCU_E_BAD_ARG;
  const long long kStride = 1ll << 35;
  if (d->rows > 0x7fffffffll || d->c_in > (1 << 24) || d->c_out > (1 << 24)) return DNXCU_E_LIMIT;
  r->d = *d;
  dnxcu_linear &c = r->d;
  r->f8 = d->dtype == DNXCU_DT_E4M3;
  r->es = r->f8 ? 1 : 2;
  if (!c.x_stride) c.x_stride = c.c_in;
  if (!c.w_stride) c.w_stride = c.c_in;
  if (!c.residual_stride) c.residual_stride = c.c_out;
  if (!c.out_stride) c.out_stride = c.c_out;
  if (c.x_stride < c.c_in || c.w_stride < c.c_in || c.residual_stride < c.c_out || c.out_stride < c.c_out) return DNXCU_E_BAD_ARG;
  if (c.x_stride >= kStride || c.w_stride >= kStride || c.residual_stride >= kStride || c.out_stride >= kStride)
    return DNXCU_E_LIMIT;
  uintptr_t halves = (uintptr_t)c.bias | (uintptr_t)c.residual | (uintptr_t)c.out;
  if (!r->f8) halves |= (uintptr_t)c.x | (uintptr_t)c.weights;
  if ((halves & 1) || (((uintptr_t)c.x_scale | (uintptr_t)c.w_scale | (uintptr_t)c.device_status) & 3)) return DNXCU_E_MISALIGNED;
  const RowSpan out{c.out, c.rows, c.c_out, c.out_stride, 2}, res{c.residual, c.rows, c.c_out, c.residual_stride, 2};
  const bool in_place = c.residual == c.out && c.residual_stride == c.out_stride;
  if (!in_place && rows_overlap(out, res)) return DNXCU_E_BAD_ARG;
  if (rows_overlap(out, {c.x, c.rows, c.c_in, c.x_stride, r->es}) || rows_overlap(out, {c.weights, c.c_out, c.c_in, c.w_stride, r->es}) ||
      rows_overlap(out, {c.bias, 1, c.c_out, c.c_out, 2}) || rows_overlap(out, {c.x_scale, 1, c.rows, c.rows, 4}) ||
      rows_overlap(out, {c.w_scale, 1, c.c_out, c.c_out, 4}) || rows_overlap(out, {c.device_status, 1, 1, 1, 4}))
    return DNXCU_E_BAD_ARG;
  return DNXCU_OK;
}

bool fits_tc(const Rec &r) {
  return mappable(r.d.x, r.d.x_stride * r.es) && mappable(r.d.weights, r.d.w_stride * r.es);
}
bool fits_rows(const Rec &r) { return r.d.rows <= 16 && fits_tc(r) && !((long long)r.d.c_in * r.es & 15); }
bool fits_split(const Rec &r) { return fits_tc(r) && (r.d.rows + 15) / 16 <= 65535; }

int round_up(int v, int m) { return (v + m - 1) / m * m; }

// Time models in microseconds on an otherwise idle B200, fitted to sweeps over 17 .. 8192 rows, 128 .. 16384 channels; they
// only rank the choices.  `kb`: 128 byte steps of c_in.
struct TileShape {
  int bn, cg;  // output channels per tile; blocks that share it (128 rows each)
  double us;
};
// A wave of tiles costs its steps, issue bound at 0.31 us up to 128 channels and growing with the operand bytes above, and
// the epilogue that is not hidden; 512 x 4096 x 4096: 64 channels 45.4 us (two waves), 128 27.3, 256 33.5; 2048 x 2048 x 2048:
// 128 29.4 (two waves), 256 20.8; 1024 x 4096 x 4096: 128 48.8, 256 35.2, pairs of 256 32.0.
TileShape pick_tile(long long rows, int n, int kb, int sms, bool any) {
  TileShape best{0, 1, 0.0};
  const auto consider = [&](int bn, int cg) {
    const long long tiles = (rows + 128 * cg - 1) / (128 * cg) * ((n + bn - 1) / bn), waves = (tiles * cg + sms - 1) / sms;
    const double step = bn <= 128 ? 0.31 : cg == 2 ? 0.37 : 0.31 + (bn - 128) * 0.0006;
    const double us = 5.0 + (double)waves * (kb * step + bn * 0.008);
    if (!best.bn || us < best.us) best = {bn, cg, us};
  };
  const int most = any ? 128 : 256;
  if (n <= most) consider(round_up(n, 16), 1);
  for (int bn = 64; bn <= most && bn < n; bn += 64) consider(bn, 1);
  if (!any && n > 192) consider(256, 2);
  return best;
}
// c_in over blocks up to the number of SMs, by powers of two (16 x 4096 x 4096: 10.6 us with 4 parts, 128 blocks; 12.1 with
// 5, 13.5 with 8); twice that where every part is still 64 steps or more (64 x 8192 x 8192: 28.7 against 30.6 us).
struct SplitShape {
  int bn, split;
  double us;
};
SplitShape pick_split(long long rows, int n, int kb, int sms) {
  SplitShape p{rows >= 256 ? 256 : round_up((int)rows, 16), 1, 0.0};
  const long long tiles = (rows + p.bn - 1) / p.bn * ((n + 127) / 128);
  while (p.split < 8 && tiles * p.split * 2 <= sms && p.split * 2 <= kb) p.split *= 2;
  if (p.split < 8 && kb / p.split >= 64) p.split *= 2;
  const double waves = (double)((tiles * p.split + sms - 1) / sms);
  // (set-up and join are paid by every wave, but for two small blocks that share an SM; 2032 x 112 x 11072: five waves, 63 us)
  const double fixed = (waves <= 2.0 && p.bn <= 64 ? 1.0 : waves) * (4.0 + 0.03 * p.bn);
  p.us = fixed + waves * ((kb + p.split - 1) / p.split) * (0.34 + (p.bn > 128 ? (p.bn - 128) * 0.0012 : 0.0));
  return p;
}
int aligned_variant(long long rows, int n, int kb, int sms) {
  return rows <= 2048 && pick_split(rows, n, kb, sms).us < pick_tile(rows, n, kb, sms, false).us ? DNXCU_LINEAR_SPLIT : DNXCU_LINEAR_TILE;
}
int k_blocks(const Rec &r) { return (int)(((long long)r.d.c_in * r.es + 127) / 128); }

// How many rows to take together as one (GROUPED), 1 for none: packed rows on a 16 byte boundary without scales of their
// own, at most 256 channels out per group, the block diagonal of the weights within 96 KB, tiles for every SM.
// 522240 rows 9 to 32 (leaky): 33 us through scratch, 20.8 grouped; 2088960 rows 3 to 16 91 and 27.8, 16 to 16 66 and 28.7.
// Layers whose rows are on 16 byte boundaries as they are gain only where they are narrow: 32 to 32 20.5 and 18.8 (with
// gelu and residual 43.7 and 46.9), 64 to 64 24.8 and 29.5.
int group_rows(const Rec &r, int sms) {
  const dnxcu_linear &d = r.d;
  if (d.variant != DNXCU_LINEAR_AUTO || d.rows <= 16 || d.x_scale || d.x_stride != d.c_in || d.out_stride != d.c_out ||
      (d.residual && d.residual_stride != d.c_out))
    return 1;
  if (((uintptr_t)d.x | (uintptr_t)d.out | (uintptr_t)d.residual) & 15) return 1;
  if (fits_tc(r) && !(d.c_out & 7) && d.c_out > 24) return 1;
  for (int g = 8; g > 1; g /= 2) {
    const long long k = (long long)g * d.c_in * r.es, n = (long long)g * d.c_out;
    if ((k & 15) || (n & 7) || n > 256) continue;
    if ((k + 127) / 128 * ((n + 15) / 16 * 16) * 128 > 98304) continue;
    if (d.rows / g >= 128ll * sms) return g;
  }
  return 1;
}

// The variant that runs the record.
int pick(const Rec &r, int sms) {
  switch (r.d.variant) {
    case DNXCU_LINEAR_ROWS: return fits_rows(r) ? (int)DNXCU_LINEAR_ROWS : (int)DNXCU_E_UNSUPPORTED;
    case DNXCU_LINEAR_SPLIT: return fits_split(r) ? (int)DNXCU_LINEAR_SPLIT : (int)DNXCU_E_UNSUPPORTED;
    case DNXCU_LINEAR_TILE: return fits_tc(r) ? (int)DNXCU_LINEAR_TILE : (int)DNXCU_E_UNSUPPORTED;
    case DNXCU_LINEAR_ANY: return DNXCU_LINEAR_ANY;
    default: break;
  }
  if (group_rows(r, sms) > 1) return DNXCU_LINEAR_TILE;
  if (!fits_tc(r)) return DNXCU_LINEAR_ANY;
  if (fits_rows(r)) return DNXCU_LINEAR_ROWS;
  return aligned_variant(r.d.rows, r.d.c_out, k_blocks(r), sms);
}

}  // namespace
}  // namespace dnxcu

using namespace dnxcu;

struct dnxcu_linear_plan {
  LinArgs a;
  LinArgs tail;               // the last rows of a grouped layer, fewer than a group (tail_kernel: whether there are any)
  const void *tail_kernel = nullptr;
  dim3 tail_grid;
  RelayArgs relay;            // operands laid out anew in front of the kernel (scratch: where)
  void *scratch = nullptr;
  unsigned relay_grid = 0;
  const void *kernel = nullptr;
  dim3 grid, block;
  uint32_t smem = 0, cluster = 1;
  int device = 0, variant = 0;
  bool f8 = false;
};

namespace dnxcu {
namespace {

constexpr int kMaxDevices = 64;
constexpr int kSmCount = 148;  // of a B200, for the calls that touch no device

int sm_count(int dev) {
  static std::atomic<int> cache[kMaxDevices];
  int n = dev < kMaxDevices ? cache[dev].load(std::memory_order_relaxed) : 0;
  if (n <= 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    if (dev < kMaxDevices) cache[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

#define TILE_KERNEL(cg, f8, any, narrow) (const void *)linear_tile<cg, f8, any, narrow, false>
#define GROUPED_KERNEL(f8) (const void *)linear_tile<1, f8, false, false, true>
// Shared memory opt-in of every kernel, once per device.
int init_device(int dev) {
  static std::atomic<int> done[kMaxDevices];
  if (dev < kMaxDevices && done[dev].load(std::memory_order_acquire)) return DNXCU_OK;
  const void *k[] = {TILE_KERNEL(1, false, false, false), TILE_KERNEL(1, true, false, false), TILE_KERNEL(2, false, false, false),
                     TILE_KERNEL(2, true, false, false),  TILE_KERNEL(1, false, false, true), TILE_KERNEL(1, true, false, true),
                     TILE_KERNEL(2, false, false, true),  TILE_KERNEL(2, true, false, true),  TILE_KERNEL(1, false, true, true),
                     TILE_KERNEL(1, true, true, true),    GROUPED_KERNEL(false),              GROUPED_KERNEL(true),
                     (const void *)linear_split<false>,   (const void *)linear_split<true>};
  for (const void *f : k) DNXCU_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimit));
  if (dev < kMaxDevices) done[dev].store(1, std::memory_order_release);
  return DNXCU_OK;
}

void plan_tile(const Rec &r, int sms, bool any, dnxcu_linear_plan *p) {
  LinArgs &a = p->a;
  const TileShape shape = a.gr > 1 ? TileShape{round_up(a.N, 16), 1, 0.0} : pick_tile(a.M, a.N, a.kb, sms, any);
  const int bn = shape.bn, cg = shape.cg;
  // The weights pass through L2 once per group of rows, so a group is as many rows as keep 36 MB of x (of 126 MB of L2)
  // in flight, 4 to 32 tiles.  Under the power limit 8192 x 4096 x 16384 binary16 takes 867, 848, 940 us with groups of 8,
  // 16 (the rule's), 32 tiles, 8192 x 8192 x 8192 879 (the rule's), 895, 965.
  const long long tile_bytes = 128ll * cg * a.K * r.es;
  a.group = (int)(36000000ll / tile_bytes);
  a.group = a.group < 4 ? 4 : a.group > 32 ? 32 : a.group;
  a.BN = bn;
  a.mt = (int)((a.M + 128ll * cg - 1) / (128 * cg));
  a.nt = (a.N + bn - 1) / bn;
  a.bufs = bn <= 128 ? 4 : 2;
  // two epilogue teams where a tile's products are soon done; one, and more stages, where they take long
  // or where the rows of out or of the residual take 2 byte accesses (8192 x 1024 x 1023 with residual: 76 us with one).
  const bool narrow = !mappable(r.d.out, a.os * 2) || (r.d.residual && !mappable(r.d.residual, a.rs * 2));
  a.teams = a.kb >= 16 && !any && !(narrow && a.kb < 32 && (long long)a.mt * a.nt > sms / cg) ? 1 : 2;
  const uint32_t wbytes = (uint32_t)(bn / cg) * 128u;
  a.w_res = a.gr > 1 || (cg == 1 && a.nt == 1 && a.mt > sms && (long long)a.kb * wbytes <= 65536);
  const uint32_t fixed = 1024u + TILE_FIXED + 4u * (uint32_t)a.teams * STAGING + (a.w_res ? (uint32_t)a.kb * wbytes : 0u);
  // Two steps per stage where three such stages fit: half the waits and commits of the issuing warp, which is what bounds
  // tiles of up to 128 channels.
  uint32_t stage = 16384u + (a.w_res ? 0u : wbytes);
  a.per_stage = a.kb > 1 && (kSmemLimit - fixed) / (2 * stage) >= 3 ? 2 : 1;
  stage *= (uint32_t)a.per_stage;
  a.stages = (int)((kSmemLimit - fixed) / stage);
  if (a.stages > MAX_STAGES) a.stages = MAX_STAGES;
  p->smem = fixed + stage * (uint32_t)a.stages;
  const long long tiles = (long long)a.mt * a.nt;
  const int clusters = (int)(tiles < sms / cg ? tiles : sms / cg);
  p->grid = dim3((unsigned)(clusters * cg));
  p->block = dim3(any ? ANY_THREADS : TILE_THREADS);
  p->cluster = (uint32_t)cg;
  const bool tail = narrow || (a.N & 7);  // (a row that ends inside 16 bytes: see the store)
  if (a.gr > 1) p->kernel = r.f8 ? GROUPED_KERNEL(true) : GROUPED_KERNEL(false);
  else if (any) p->kernel = r.f8 ? TILE_KERNEL(1, true, true, true) : TILE_KERNEL(1, false, true, true);
  else if (cg == 2 && tail) p->kernel = r.f8 ? TILE_KERNEL(2, true, false, true) : TILE_KERNEL(2, false, false, true);
  else if (cg == 2) p->kernel = r.f8 ? TILE_KERNEL(2, true, false, false) : TILE_KERNEL(2, false, false, false);
  else if (tail) p->kernel = r.f8 ? TILE_KERNEL(1, true, false, true) : TILE_KERNEL(1, false, false, true);
  else p->kernel = r.f8 ? TILE_KERNEL(1, true, false, false) : TILE_KERNEL(1, false, false, false);
}

void plan_split(const Rec &r, int sms, dnxcu_linear_plan *p) {
  LinArgs &a = p->a;
  const SplitShape shape = pick_split(a.M, a.N, a.kb, sms);
  a.BN = shape.bn;
  a.split = shape.split;
  a.mt = (a.M + a.BN - 1) / a.BN;
  a.nt = (a.N + 127) / 128;
  const long long tiles = (long long)a.mt * a.nt;
  const uint32_t stage = 16384u + (uint32_t)a.BN * 128u, fixed = 1024u + SPLIT_FIXED;
  const int most = a.BN < a.M ? a.BN : a.M, per = (most + a.split - 1) / a.split;
  const uint32_t recv = (uint32_t)(a.split * per) * 512u;
  // two blocks per SM where there are more blocks than SMs and shared memory leaves both some stages; six stages are
  // as fast as twelve
  uint32_t room = kSmemLimit - fixed;
  if (tiles * a.split > sms && kSmemLimit / 2 - fixed - 1024u >= recv + 3 * stage) room = kSmemLimit / 2 - fixed - 1024u;
  a.overlay = recv + 3 * stage > room;
  int st = (int)((room - (a.overlay ? 0u : recv)) / stage);
  const int steps = (a.kb + a.split - 1) / a.split;
  st = st > 6 ? 6 : st;
  a.stages = st > steps ? (steps > 2 ? steps : 2) : st;
  const uint32_t body = stage * (uint32_t)a.stages;
  p->smem = fixed + (a.overlay ? (body > recv ? body : recv) : body + recv);
  p->grid = dim3((unsigned)(a.nt * a.split), (unsigned)a.mt);
  p->block = dim3(SPLIT_THREADS);
  p->cluster = (uint32_t)a.split;
  p->kernel = r.f8 ? (const void *)linear_split<true> : (const void *)linear_split<false>;
}

// Kernel, geometry and tensor maps of a checked record whose operands start at `x` and `w`, their rows `a.xs` and `a.ws`
// bytes apart (the caller's, or the plan's aligned copies), for variant `v`.
int plan_kernel(const Rec &r, int v, const void *x, const void *w, int sms, dnxcu_linear_plan *p) {
  const dnxcu_linear &d = r.d;
  LinArgs &a = p->a;
  a.x = (const uint8_t *)x;
  a.w = (const uint8_t *)w;
  if (v == DNXCU_LINEAR_ROWS || (v == DNXCU_LINEAR_ANY && a.M <= 16)) {
    p->block = dim3(ROWS_THREADS);
    const bool two = a.M > 8;
    if (v == DNXCU_LINEAR_ANY) {
      if (r.f8) p->kernel = two ? (const void *)linear_rows<true, 2, 1, 1, true> : (const void *)linear_rows<true, 1, 1, 1, true>;
      else p->kernel = two ? (const void *)linear_rows<false, 2, 1, 1, true> : (const void *)linear_rows<false, 1, 1, 1, true>;
    } else if (r.f8) {
      // (16 x 4096 x 12288: 15.1 us with four chunks on their way, 13.3 with two and more blocks per SM; x 4096: 6.3 and 6.6)
      const void *k2 = (a.N + 15) / 16 > 2 * sms ? (const void *)linear_rows<true, 2, 1, 2, false> : (const void *)linear_rows<true, 2, 1, 4, false>;
      p->kernel = two ? k2 : (const void *)linear_rows<true, 1, 1, 4, false>;
    } else {
      p->kernel = two ? (const void *)linear_rows<false, 2, 1, 2, false> : (const void *)linear_rows<false, 1, 1, 4, false>;
    }
    p->grid = dim3((unsigned)((a.N + 15) / 16));
    return DNXCU_OK;
  }
  int st = init_device(p->device);
  if (st) return st;
  if (v == DNXCU_LINEAR_SPLIT) {
    plan_split(r, sms, p);
    st = matrix_map(&a.tm_w, w, r.f8, a.N, a.K, a.ws, 128);
    return st ? st : matrix_map(&a.tm_x, x, r.f8, a.M, a.K, a.xs, a.BN);
  }
  plan_tile(r, sms, v == DNXCU_LINEAR_ANY, p);
  if (v == DNXCU_LINEAR_TILE) {
    st = matrix_map(&a.tm_x, x, r.f8, a.M, a.K, a.xs, 128);
    if (!st && a.gr == 1) st = matrix_map(&a.tm_w, w, r.f8, a.N, a.K, a.ws, a.BN / (int)p->cluster);
    if (st) return st;
  }
  a.out_tma = mappable(d.out, a.os * 2);
  a.res_tma = d.residual && mappable(d.residual, a.rs * 2);
  a.out_pack = a.N <= 64 && a.os == a.N && !((uintptr_t)d.out & 15);
  a.res_pack = d.residual && a.N <= 64 && a.rs == a.N && !((uintptr_t)d.residual & 15);
  if (a.out_tma && (st = matrix_map(&a.tm_out, d.out, false, a.M, a.N, a.os * 2, 32))) return st;
  if (a.res_tma && (st = matrix_map(&a.tm_res, d.residual, false, a.M, a.N, a.rs * 2, 32))) return st;
  return DNXCU_OK;
}

// Device memory outside of any stream's order; a capture that this thread has under way is not disturbed.
bool scratch_alloc(void **p, size_t bytes) {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  cudaThreadExchangeStreamCaptureMode(&mode);
  const bool ok = cudaMalloc(p, bytes) == cudaSuccess;
  cudaThreadExchangeStreamCaptureMode(&mode);
  if (!ok) {
    cudaGetLastError();
    *p = nullptr;
  }
  return ok;
}

// `keep`: the plan outlives this call and may hold scratch memory.
int make_plan(const Rec &r, dnxcu_linear_plan *p, bool keep) {
  const dnxcu_linear &d = r.d;
  DNXCU_CUDA(cudaGetDevice(&p->device));
  const int sms = sm_count(p->device);
  const int v = pick(r, sms);
  if (v < 0) return v;
  for (const void *q : {d.x, d.weights, (const void *)d.x_scale, (const void *)d.w_scale, d.bias, d.residual, (const void *)d.out,
                        (const void *)d.device_status})
    if (!on_current_device(q)) return DNXCU_E_BAD_ARG;
  p->f8 = r.f8;
  LinArgs &a = p->a;
  memset(&a, 0, sizeof(a));
  a.x_scale = d.x_scale;
  a.w_scale = d.w_scale;
  a.bias = (const __half *)d.bias;
  a.res = (const __half *)d.residual;
  a.out = (__half *)d.out;
  a.xs = d.x_stride * r.es;
  a.ws = d.w_stride * r.es;
  a.rs = d.residual_stride;
  a.os = d.out_stride;
  a.M = (int)d.rows;
  a.N = d.c_out;
  a.K = d.c_in;
  a.act = d.activation;
  a.alpha = d.leaky_alpha;
  a.kb = k_blocks(r);
  a.status = d.device_status;
  a.wait_limit = wait_limit_cycles();
  if (a.wait_limit < 2000000ull) a.wait_limit |= 1ull << 63;  // below about a millisecond: strict (see mbar_wait)
  a.gr = 1;
  if (const int gr = v == DNXCU_LINEAR_TILE ? group_rows(r, sms) : 1; gr > 1) {
    const int left = a.M % gr;
    if (left) {
      p->tail = a;
      LinArgs &t = p->tail;
      t.M = left;
      const long long r0 = a.M - left;
      t.x = (const uint8_t *)d.x + r0 * a.xs;
      t.w = (const uint8_t *)d.weights;
      t.out += r0 * a.os;
      if (t.res) t.res += r0 * a.rs;
      p->tail_kernel = r.f8 ? (const void *)linear_rows<true, 1, 1, 1, true> : (const void *)linear_rows<false, 1, 1, 1, true>;
      p->tail_grid = dim3((unsigned)((a.N + 15) / 16));
    }
    a.gr = gr;
    a.n1 = a.N;
    a.k1 = a.K;
    a.M /= gr;
    a.N *= gr;
    a.K *= gr;
    a.xs *= gr;
    a.rs *= gr;
    a.os *= gr;
    a.kb = (a.K * r.es + 127) / 128;
  }
  // Unaligned operands of a kept plan: laid out anew in scratch memory by one kernel, then the aligned variants.
  if (v == DNXCU_LINEAR_ANY && d.variant == DNXCU_LINEAR_AUTO && keep && a.M > 16) {
    RelayArgs &y = p->relay;
    memset(&y, 0, sizeof(y));
    const bool rx = !mappable(d.x, a.xs), rw = !mappable(d.weights, a.ws);
    const long long pitch = ((long long)a.K * r.es + 15) / 16 * 16;
    y.kbytes = a.K * r.es;
    y.per_row = (int)(pitch / 16);
    y.per_group = y.per_row < 1024 ? 1024 / y.per_row : 1;
    y.magic = y.per_row == 1 ? 0u : 0xffffffffu / (uint32_t)y.per_row + 1;
    y.src[0] = (const uint8_t *)d.x;
    y.src[1] = (const uint8_t *)d.weights;
    y.stride[0] = a.xs;
    y.stride[1] = a.ws;
    y.rows[0] = a.M;
    y.rows[1] = a.N;
    y.pitch = pitch;
    if (rx) y.groups[0] = (a.M + y.per_group - 1) / y.per_group;
    if (rw) y.groups[1] = (a.N + y.per_group - 1) / y.per_group;
    const size_t xb = rx ? (size_t)a.M * (size_t)pitch : 0, wb = rw ? (size_t)a.N * (size_t)pitch : 0;
    if (scratch_alloc(&p->scratch, xb + wb)) {
      y.dst[0] = (uint8_t *)p->scratch;
      y.dst[1] = (uint8_t *)p->scratch + xb;
      const int groups = y.groups[0] + y.groups[1];
      p->relay_grid = (unsigned)(groups < 16 * sms ? groups : 16 * sms);
      if (rx) a.xs = pitch;
      if (rw) a.ws = pitch;
      p->variant = v;
      return plan_kernel(r, aligned_variant(a.M, a.N, a.kb, sms), rx ? y.dst[0] : d.x, rw ? y.dst[1] : d.weights, sms, p);
    }
    // (no room: the kernel that fetches by plain loads needs none)
  }
  p->variant = v;
  return plan_kernel(r, v, d.x, d.weights, sms, p);
}

int launch(const dnxcu_linear_plan &p, cudaStream_t s) {
  if (p.relay_grid) {
    void *args[] = {const_cast<RelayArgs *>(&p.relay)};
    DNXCU_CUDA(cudaLaunchKernel(p.f8 ? (const void *)linear_relay<true> : (const void *)linear_relay<false>, dim3(p.relay_grid), dim3(256),
                                args, 0, s));
  }
  void *args[] = {const_cast<LinArgs *>(&p.a)};
  DNXCU_CUDA(launch_dependent(p.kernel, p.grid, p.block, p.smem, p.cluster, s, args));
  if (p.tail_kernel) {
    void *targs[] = {const_cast<LinArgs *>(&p.tail)};
    DNXCU_CUDA(launch_dependent(p.tail_kernel, p.tail_grid, dim3(ROWS_THREADS), 0, 1, s, targs));
  }
  return DNXCU_OK;
}

}  // namespace
}  // namespace dnxcu

extern "C" {

int dnxcu_linear_validate(const dnxcu_linear *d) {
  Rec r;
  const int st = check(d, &r);
  if (st) return st;
  const int v = pick(r, kSmCount);
  return v < 0 ? v : DNXCU_OK;
}

int dnxcu_linear_pick(const dnxcu_linear *d) {
  Rec r;
  const int st = check(d, &r);
  return st ? st : pick(r, kSmCount);
}

int dnxcu_linear_launch(const dnxcu_linear *d, void *stream) {
  Rec r;
  int st = check(d, &r);
  if (st) return st;
  dnxcu_linear_plan p;
  st = make_plan(r, &p, false);
  return st ? st : launch(p, (cudaStream_t)stream);
}

int dnxcu_linear_plan_create(const dnxcu_linear *d, dnxcu_linear_plan **out) {
  if (!out) return DNXCU_E_BAD_ARG;
  Rec r;
  int st = check(d, &r);
  if (st) return st;
  dnxcu_linear_plan *p = new (std::nothrow) dnxcu_linear_plan();
  if (!p) return DNXCU_E_NO_MEMORY;
  st = make_plan(r, p, true);
  if (st) {
    dnxcu_linear_plan_destroy(p);
    return st;
  }
  *out = p;
  return DNXCU_OK;
}

int dnxcu_linear_plan_launch(const dnxcu_linear_plan *p, void *stream) {
  if (!p) return DNXCU_E_BAD_ARG;
  int dev = 0;
  DNXCU_CUDA(cudaGetDevice(&dev));
  if (dev != p->device) return DNXCU_E_STATE;
  return launch(*p, (cudaStream_t)stream);
}

void dnxcu_linear_plan_destroy(dnxcu_linear_plan *p) {
  if (!p) return;
  if (p->scratch) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev != p->device) cudaSetDevice(p->device);
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (cudaFree(p->scratch) != cudaSuccess) cudaGetLastError();  // (waits for launches that still use it)
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (dev != p->device) cudaSetDevice(dev);
  }
  delete p;
}

}  // extern "C"
