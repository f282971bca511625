// Linear layer: out = residual + act(x_scale * w_scale * (x weights^T) + bias), binary16 or e4m3 operands, 32 bit sums.
//
// Three kernels, four variants:
//   linear_rows   (ROWS)       a handful of rows: the call is the time to stream the weights.  Legacy warp MMA with the
//                              weights as the 16 row operand, straight from global memory into registers.
//   linear_split  (SPLIT)      few rows: tcgen05 with 128 output channels as the MMA's rows and the tokens as its columns;
//                              c_in split over a cluster, partial sums joined through distributed shared memory.
//   linear_tile   (TILE, ANY)  persistent tcgen05 tiles of 128 rows per block, or of 256 rows over a pair of blocks
//                              (cta_group::2); ANY fills the same shared memory tiles with plain loads.
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
  int split;     // split: blocks per cluster
  int out_tma, res_tma;
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

template <int CG, bool F8>
__device__ __forceinline__ void mma_step(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
#define DNXCU_MMA(group, kind)                                                             \
  asm volatile(                                                                            \
      "{\n\t"                                                                              \
      ".reg .pred p;\n\t"                                                                  \
      "setp.ne.b32 p, %4, 0;\n\t"                                                          \
      "tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, p;\n\t"           \
      "}" ::"r"(d),                                                                        \
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)                                          \
      : "memory")
  if (CG == 2 && F8) DNXCU_MMA("2", "f8f6f4");
  else if (CG == 2) DNXCU_MMA("2", "f16");
  else if (F8) DNXCU_MMA("1", "f8f6f4");
  else DNXCU_MMA("1", "f16");
#undef DNXCU_MMA
}
// Arrives on `bar` (of both blocks of a pair) when the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
  else
    tc_commit(bar);
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

// Operand tiles: rows of 128 bytes (64 binary16 or 128 e4m3 channels) with the 128 byte swizzle, K major.  Descriptor:
// start address, 1024 bytes between groups of 8 rows, layout code 2.  A K step is 32 bytes for either type.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  return ((uint64_t)kDescHi << 32) | (uint64_t)((addr >> 4) | (1u << 16));
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

constexpr int MAX_STAGES = 8;
constexpr int HDR_FULL = 0, HDR_EMPTY = 8 * MAX_STAGES, HDR_TFULL = 16 * MAX_STAGES, HDR_TEMPTY = HDR_TFULL + 16,
              HDR_RES = HDR_TEMPTY + 16, HDR_TMEM = HDR_RES + 64, HDR_ABORT = HDR_TMEM + 4;
static_assert((HDR_ABORT + 4) % 8 == 0 && HDR_ABORT + 12 <= 1024, "header layout");
constexpr int HEADER = 1024;
constexpr uint32_t kSmemLimit = 232448;

__device__ __forceinline__ uint32_t aligned_base(const void *dyn) { return (smem_u32(dyn) + 1023u) & ~1023u; }

// ---- TILE and ANY -----------------------------------------------------------
// 12 warps: 0 fetches operand tiles, 1 issues MMAs, 2 owns the tensor memory, 4-7 and 8-11 are two epilogue teams that
// take alternate tiles; each team has one of the two accumulators, so one tile is multiplied while the teams finish the
// ones before.  ANY: warps 8-11 fetch instead, one team takes both accumulators.
constexpr int TILE_THREADS = 384;
constexpr int COLBUF = 512;              // per epilogue warp: bias and weight scale of 64 channels
constexpr int TILE_FIXED = HEADER + 8 * COLBUF;
constexpr int STAGING = 4096;            // per epilogue warp: 32 rows x 64 channels of binary16

struct TilePos {
  int m, n;
};
// Tiles in groups of `G` along the rows, so that the tiles in flight share operands in L2.
__device__ __forceinline__ TilePos tile_pos(const LinArgs &g, int t, int G) {
  if (g.nt == 1) return {t, 0};
  const int per = G * g.nt, grp = t / per, r = t - grp * per;
  const int m0 = grp * G, gm = min(G, g.mt - m0);
  const int n = r / gm;
  return {m0 + r - n * gm, n};
}

// 8 elements (16 bytes) or 16 e4m3 of one operand row from channel byte `kbyte` on, zero beyond the row: plain loads.
template <bool F8>
__device__ __forceinline__ uint4 fetch_piece(const uint8_t *row, int kbyte, int kbytes) {
  const int left = kbytes - kbyte;
  if (left <= 0) return make_uint4(0, 0, 0, 0);
  const uint8_t *p = row + kbyte;
  if (left >= 16 && ((uintptr_t)p & 15) == 0) return __ldg(reinterpret_cast<const uint4 *>(p));
  uint32_t w[4];
  if (F8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i * 4 + e < left) w[i] |= (uint32_t)__ldg(p + i * 4 + e) << (8 * e);
    }
  } else {
    const uint16_t *q = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (i * 4 + e * 2 < left) w[i] |= (uint32_t)__ldg(q + i * 2 + e) << (16 * e);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int CG, bool F8, bool ANY>
__global__ void __launch_bounds__(TILE_THREADS, 1) linear_tile(const __grid_constant__ LinArgs g) {
  extern __shared__ uint8_t dyn[];
  const uint32_t base = aligned_base(dyn);
  uint8_t *hdr = dyn + (base - smem_u32(dyn));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(hdr + HDR_ABORT);
  const uint32_t b_rows = (uint32_t)g.BN / CG;
  const uint32_t stage_bytes = 16384u + b_rows * 128u;
  const uint32_t stage0 = base + TILE_FIXED, staging0 = stage0 + stage_bytes * (uint32_t)g.stages;
  const int ntiles = g.mt * g.nt, step = (int)gridDim.x / CG, first = (int)blockIdx.x / CG;
  constexpr int GROUP = CG == 2 ? 8 : 16;
  constexpr int TEAMS = ANY ? 1 : 2;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    *reinterpret_cast<volatile unsigned long long *>(abort_flag + 1) = g.wait_limit;
    for (int i = 0; i < MAX_STAGES; ++i) {
      mbar_init(base + HDR_FULL + 8 * i, ANY ? 4 : 1);
      mbar_init(base + HDR_EMPTY + 8 * i, 1);
      mbar_init(base + HDR_RES + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
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

  if (!ANY && warp == 0) {
    // ---- operand tiles by TMA; the pair's bytes are counted on the first block's barrier ----
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 1;
      bool ok = true;
      for (int t = first; ok && t < ntiles; t += step) {
        const TilePos p = tile_pos(g, t, GROUP);
        const int row_a = p.m * (128 * CG) + (int)rank * 128, row_b = p.n * g.BN + (int)(rank * b_rows);
        for (int kb = 0; kb < g.kb; ++kb) {
          ok = mbar_wait(base + HDR_EMPTY + 8 * s, ph, abort_flag, g.status, 12);
          if (!ok) break;
          const uint32_t full = base + HDR_FULL + 8 * s;
          if (rank == 0) mbar_expect_tx(full, stage_bytes * CG);
          const uint32_t bar = CG == 2 ? map_rank(full, 0) : full;
          const uint32_t a = stage0 + stage_bytes * (uint32_t)s;
          tma_load_2d<CG>(a, &g.tm_x, kb * (F8 ? 128 : 64), row_a, bar);
          tma_load_2d<CG>(a + 16384u, &g.tm_w, kb * (F8 ? 128 : 64), row_b, bar);
          if (++s == g.stages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
    }
  } else if (ANY && warp >= 8) {
    // ---- operand tiles by plain loads, swizzled as the copy engine would ----
    const int tid = threadIdx.x - 256;
    const int kbytes = F8 ? g.K : 2 * g.K;
    int s = 0;
    uint32_t ph = 1;
    bool ok = true;
    for (int t = first; ok && t < ntiles; t += step) {
      const TilePos p = tile_pos(g, t, GROUP);
      for (int kb = 0; kb < g.kb; ++kb) {
        ok = mbar_wait(base + HDR_EMPTY + 8 * s, ph, abort_flag, g.status, 12);
        ok = __all_sync(0xffffffffu, ok);  // (the warp leaves the loop as one)
        if (!ok) break;
        const uint32_t a = stage0 + stage_bytes * (uint32_t)s;
        const int pieces = 2 * k_steps<F8>(g, kb);  // 16 byte pieces of a row that the MMAs will read
        const int items = (128 + g.BN) * pieces;
#pragma unroll 4
        for (int i = tid; i < items; i += 128) {
          const int r = i / pieces, j = i - r * pieces;
          const bool is_w = r >= 128;
          const int rr = is_w ? r - 128 : r;
          const long long row = is_w ? (long long)p.n * g.BN + rr : (long long)p.m * 128 + rr;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (row < (is_w ? g.N : g.M))
            v = fetch_piece<F8>(is_w ? g.w + row * g.ws : g.x + row * g.xs, kb * 128 + j * 16, kbytes);
          sts128(a + (is_w ? 16384u : 0u) + (uint32_t)rr * 128u + (uint32_t)((j ^ (rr & 7)) << 4), v);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(base + HDR_FULL + 8 * s);
        if (++s == g.stages) {
          s = 0;
          ph ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    // ---- MMA issue: one thread of the (first) block ----
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = mma_idesc(128 * CG, g.BN);
      int s = 0, it = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = first; ok && t < ntiles; t += step, ++it) {
        const int buf = it & 1;
        const uint32_t d = tmem + (uint32_t)(buf * g.BN);
        ok = mbar_wait(base + HDR_TEMPTY + 8 * buf, (uint32_t)((it >> 1) & 1) ^ 1u, abort_flag, g.status, 14);
        if (!ok) break;
        tc_fence_after();
        for (int kb = 0; kb < g.kb; ++kb) {
          ok = mbar_wait(base + HDR_FULL + 8 * s, ph, abort_flag, g.status, 11);
          if (!ok) break;
          tc_fence_after();
          const uint64_t a = operand_desc(stage0 + stage_bytes * (uint32_t)s), b = a + (16384u >> 4);
          const int ks = k_steps<F8>(g, kb);
          if (ks == 4) {
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_step<CG, F8>(d, a + 2 * k, b + 2 * k, idesc, (kb | k) != 0);
          } else {
            for (int k = 0; k < ks; ++k) mma_step<CG, F8>(d, a + 2 * k, b + 2 * k, idesc, (kb | k) != 0);
          }
          mma_commit<CG>(base + HDR_EMPTY + 8 * s);
          if (++s == g.stages) {
            s = 0;
            ph ^= 1;
          }
        }
        if (!ok) break;
        mma_commit<CG>(base + HDR_TFULL + 8 * buf);
      }
    }
  } else if (warp >= 4 && warp < 4 + 4 * TEAMS) {
    // ---- epilogue: 32 rows x 64 channels at a time through a swizzled staging tile ----
    const int ew = warp - 4, team = ew >> 2, q = warp & 3;
    const uint32_t stg = staging0 + (uint32_t)ew * STAGING;
    uint8_t *stg_p = hdr + (stg - base);
    float *col_b = reinterpret_cast<float *>(hdr + HEADER + ew * COLBUF), *col_s = col_b + 64;
    const uint32_t rbar = base + HDR_RES + 8 * ew;
    const uint32_t my = stg + (uint32_t)lane * 128u;
    uint32_t rph = 0;
    bool ok = true;
    int it = 0;
    for (int t = first; ok && t < ntiles; t += step, ++it) {
      if (TEAMS == 2 && (it & 1) != team) continue;
      const int buf = it & 1;
      const TilePos p = tile_pos(g, t, GROUP);
      const int n0 = p.n * g.BN, nc = min(g.BN, g.N - n0);
      const long long row0 = (long long)p.m * (128 * CG) + (long long)rank * 128 + q * 32, row = row0 + lane;
      const bool live = row0 < g.M;
      const float xs = (g.x_scale && row < g.M) ? __ldg(g.x_scale + row) : 1.0f;
      const auto fetch_res = [&](int c) {  // (lane 0) the residual's box into the staging tile
        mbar_expect_tx(rbar, STAGING);
        tma_load_2d<1>(stg, &g.tm_res, n0 + c, (int)row0, rbar);
      };
      if (live && g.res_tma && lane == 0) {
        bulk_group_wait_read();
        fetch_res(0);
      }
      ok = mbar_wait(base + HDR_TFULL + 8 * buf, (uint32_t)(it >> 1) & 1u, abort_flag, g.status, 13);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + (uint32_t)(buf * g.BN) + ((uint32_t)(q * 32) << 16);
      for (int c = 0; live && c < nc; c += 64) {
        for (int j = lane; j < 64; j += 32) {
          const int n = n0 + c + j;
          col_b[j] = (g.bias && n < g.N) ? __half2float(__ldg(g.bias + n)) : 0.0f;
          col_s[j] = (g.w_scale && n < g.N) ? __ldg(g.w_scale + n) : 1.0f;
        }
        if (lane == 0 && (!g.res_tma || c > 0)) {
          bulk_group_wait_read();  // the staging tile's last store has read it
          if (g.res_tma) fetch_res(c);
        }
        __syncwarp();
        if (g.res_tma) {
          ok = mbar_wait(rbar, rph, abort_flag, g.status, 15);
          rph ^= 1;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        } else if (g.res) {
          for (int r = 0; r < 32 && row0 + r < g.M; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int j = lane + 32 * h;
              if (c + j < nc)
                *reinterpret_cast<__half *>(stg_p + r * 128 + ((((j >> 3) ^ (r & 7)) << 4) | ((j & 7) << 1))) =
                    g.res[(row0 + r) * g.rs + n0 + c + j];
            }
          __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (c + 32 * h >= nc) break;  // (uniform)
          uint32_t raw[32];
          tc_ld32(acc + (uint32_t)(c + 32 * h), raw);
          tc_wait_ld();
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
        // (a store through the tensor map writes whole 16 byte pieces: not for a row that ends inside one)
        if (g.out_tma && (c + 64 <= nc || (g.N & 7) == 0)) {
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&g.tm_out, stg, n0 + c, (int)row0);
            bulk_group_commit();
          }
        } else {
          __syncwarp();
          for (int r = 0; r < 32 && row0 + r < g.M; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int j = lane + 32 * h;
              if (c + j < nc)
                g.out[(row0 + r) * g.os + n0 + c + j] =
                    *reinterpret_cast<const __half *>(stg_p + r * 128 + ((((j >> 3) ^ (r & 7)) << 4) | ((j & 7) << 1)));
            }
          fence_proxy_async();  // (the next residual box comes through the copy engine)
        }
        __syncwarp();
      }
      // the accumulator goes back to the issuing thread
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        const uint32_t te = base + HDR_TEMPTY + 8 * buf;
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
// accumulator's lanes are output channels, its columns rows of x.  Partial sums go to the block's own shared memory (over
// the operand stages, all read by then) as [row][128 channels]; each block then adds up its share of the items over the
// cluster in rank order and writes them.
constexpr int SPLIT_THREADS = 256;

template <bool F8>
__global__ void __launch_bounds__(SPLIT_THREADS) linear_split(const __grid_constant__ LinArgs g) {
  extern __shared__ uint8_t dyn[];
  const uint32_t base = aligned_base(dyn);
  uint8_t *hdr = dyn + (base - smem_u32(dyn));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(hdr + HDR_ABORT);
  const int S = g.split, rank = (int)blockIdx.x % S, ft = (int)blockIdx.x / S;
  const int n0 = ft * 128, m0 = (int)blockIdx.y * g.BN;
  const int kb0 = (int)((long long)g.kb * rank / S), kb1 = (int)((long long)g.kb * (rank + 1) / S);
  const uint32_t stage_bytes = 16384u + (uint32_t)g.BN * 128u, stage0 = base + HEADER;
  const uint32_t cols = g.BN <= 32 ? 32u : g.BN <= 64 ? 64u : g.BN <= 128 ? 128u : 256u;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    *reinterpret_cast<volatile unsigned long long *>(abort_flag + 1) = g.wait_limit;
    for (int i = 0; i < MAX_STAGES; ++i) {
      mbar_init(base + HDR_FULL + 8 * i, 1);
      mbar_init(base + HDR_EMPTY + 8 * i, 1);
    }
    mbar_init(base + HDR_TFULL, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) tmem_alloc<1>(base + HDR_TMEM, cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(hdr + HDR_TMEM);

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 1;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(base + HDR_EMPTY + 8 * s, ph, abort_flag, g.status, 12)) break;
        const uint32_t full = base + HDR_FULL + 8 * s, a = stage0 + stage_bytes * (uint32_t)s;
        mbar_expect_tx(full, stage_bytes);
        tma_load_2d<1>(a, &g.tm_w, kb * (F8 ? 128 : 64), n0, full);
        tma_load_2d<1>(a + 16384u, &g.tm_x, kb * (F8 ? 128 : 64), m0, full);
        if (++s == g.stages) {
          s = 0;
          ph ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = mma_idesc(128, g.BN);
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = mbar_wait(base + HDR_FULL + 8 * s, ph, abort_flag, g.status, 11);
        if (!ok) break;
        tc_fence_after();
        const uint64_t a = operand_desc(stage0 + stage_bytes * (uint32_t)s), b = a + (16384u >> 4);
        const int ks = k_steps<F8>(g, kb);
        for (int k = 0; k < ks; ++k) mma_step<1, F8>(tmem, a + 2 * k, b + 2 * k, idesc, kb > kb0 || k > 0);
        mma_commit<1>(base + HDR_EMPTY + 8 * s);
        if (++s == g.stages) {
          s = 0;
          ph ^= 1;
        }
      }
      if (ok) mma_commit<1>(base + HDR_TFULL);
    }
  }
  __syncwarp();
  bool ok = mbar_wait(base + HDR_TFULL, 0, abort_flag, g.status, 13);
  ok = __all_sync(0xffffffffu, ok);
  if (ok) {
    tc_fence_after();
    const int q = warp & 3;
    for (int c = (warp >> 2) * 16; c < g.BN; c += 32) {
      uint32_t raw[16];
      tc_ld16(tmem + (uint32_t)c + ((uint32_t)(q * 32) << 16), raw);
      tc_wait_ld();
      const uint32_t dst = stage0 + (uint32_t)(c * 128 + q * 32 + lane) * 4u;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst + (uint32_t)i * 512u), "r"(raw[i]) : "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  abort_drain(abort_flag);
  cluster_sync();  // (every block of the cluster comes here, aborted or not)
  if (warp == 2) tmem_free<1>(tmem, cols);
  const int rows = min(g.BN, g.M - m0);
  // 32 items of 4 channels per row: a warp writes 128 consecutive channels
  for (int i = rank * SPLIT_THREADS + (int)threadIdx.x; i < rows * 32; i += S * SPLIT_THREADS) {
    const int r = i >> 5, f = (i & 31) * 4, n = n0 + f;
    if (n >= g.N) continue;
    const uint32_t at = stage0 + (uint32_t)(r * 128 + f) * 4u;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int b = 0; b < S; ++b) {
      float4 p;
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(p.x), "=f"(p.y), "=f"(p.z), "=f"(p.w)
                   : "r"(map_rank(at, (uint32_t)b)));
      v[0] += p.x;
      v[1] += p.y;
      v[2] += p.z;
      v[3] += p.w;
    }
    const long long m = m0 + r;
    const float xs = g.x_scale ? __ldg(g.x_scale + m) : 1.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[e] = n + e < g.N ? fmaf(v[e] * xs, g.w_scale ? __ldg(g.w_scale + n + e) : 1.0f,
                                g.bias ? __half2float(__ldg(g.bias + n + e)) : 0.0f)
                         : 0.0f;
    activate(v, g.act, g.alpha);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < g.N) {
        const float r0 = g.res ? __half2float(g.res[m * g.rs + n + e]) : 0.0f;
        g.out[m * g.os + n + e] = __float2half_rn(g.res ? v[e] + r0 : v[e]);
      }
  }
  cluster_sync();  // no block leaves while another reads its partial sums
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
template <bool F8>
__device__ __forceinline__ void load_piece(Piece<F8> &p, const uint8_t *row, int chunk, int t, int kbytes, bool stream) {
#pragma unroll
  for (int i = 0; i < (F8 ? 1 : 2); ++i) {
    const int at = chunk * (F8 ? 64 : 128) + i * 64 + t * 16;
    p.v[i] = at < kbytes ? (stream ? ld_stream(row + at) : __ldg(reinterpret_cast<const uint4 *>(row + at))) : make_uint4(0, 0, 0, 0);
  }
}
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

template <bool F8, int NT>
__global__ void __launch_bounds__(ROWS_THREADS) linear_rows(const __grid_constant__ LinArgs g) {
  constexpr int U = NT == 1 ? 4 : 2;  // chunks in flight
  __shared__ float part[8][16][8 * NT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t = lane & 3;
  const int f0 = (int)blockIdx.x * 16;
  const int kbytes = F8 ? g.K : 2 * g.K;
  const int chunks = (g.K + 63) / 64;
  const uint8_t *w0 = g.w + (long long)min(f0 + gr, g.N - 1) * g.ws, *w1 = g.w + (long long)min(f0 + gr + 8, g.N - 1) * g.ws;
  const uint8_t *xr[NT];
  bool have[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    have[n] = n * 8 + gr < g.M;
    xr[n] = g.x + (have[n] ? (long long)(n * 8 + gr) * g.xs : 0);
  }
  float acc[NT][4] = {};
  for (int c0 = warp; c0 < chunks; c0 += 8 * U) {
    Piece<F8> a[U], b[U], x[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + 8 * u;  // (beyond the last chunk: zeros)
      load_piece<F8>(a[u], w0, c, t, kbytes, true);
      load_piece<F8>(b[u], w1, c, t, kbytes, true);
#pragma unroll
      for (int n = 0; n < NT; ++n) load_piece<F8>(x[u][n], xr[n], c, t, have[n] ? kbytes : 0, false);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        uint32_t a0, a1, a2, a3;
        step_regs<F8>(a[u], s, a0, a2);
        step_regs<F8>(b[u], s, a1, a3);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t b0, b1;
          step_regs<F8>(x[u][n], s, b0, b1);
          mma_16816(acc[n], a0, a1, a2, a3, b0, b1);
        }
      }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    part[warp][gr][n * 8 + 2 * t] = acc[n][0];
    part[warp][gr][n * 8 + 2 * t + 1] = acc[n][1];
    part[warp][gr + 8][n * 8 + 2 * t] = acc[n][2];
    part[warp][gr + 8][n * 8 + 2 * t + 1] = acc[n][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * 8 * NT; i += ROWS_THREADS) {
    const int f = i & 15, m = i >> 4, n = f0 + f;
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

// The variant that runs the record.
int pick(const Rec &r) {
  switch (r.d.variant) {
    case DNXCU_LINEAR_ROWS: return fits_rows(r) ? (int)DNXCU_LINEAR_ROWS : (int)DNXCU_E_UNSUPPORTED;
    case DNXCU_LINEAR_SPLIT: return fits_split(r) ? (int)DNXCU_LINEAR_SPLIT : (int)DNXCU_E_UNSUPPORTED;
    case DNXCU_LINEAR_TILE: return fits_tc(r) ? (int)DNXCU_LINEAR_TILE : (int)DNXCU_E_UNSUPPORTED;
    case DNXCU_LINEAR_ANY: return DNXCU_LINEAR_ANY;
    default: break;
  }
  if (!fits_tc(r)) return DNXCU_LINEAR_ANY;
  if (r.d.rows <= 8 && fits_rows(r)) return DNXCU_LINEAR_ROWS;
  return r.d.rows <= 256 ? DNXCU_LINEAR_SPLIT : DNXCU_LINEAR_TILE;
}

}  // namespace
}  // namespace dnxcu

using namespace dnxcu;

struct dnxcu_linear_plan {
  LinArgs a;
  const void *kernel = nullptr;
  dim3 grid, block;
  uint32_t smem = 0, cluster = 1;
  int device = 0, variant = 0;
};

namespace dnxcu {
namespace {

constexpr int kMaxDevices = 64;

int sm_count(int dev) {
  static std::atomic<int> cache[kMaxDevices];
  int n = dev < kMaxDevices ? cache[dev].load(std::memory_order_relaxed) : 0;
  if (n <= 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    if (dev < kMaxDevices) cache[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Shared memory opt-in of every kernel, once per device.
int init_device(int dev) {
  static std::atomic<int> done[kMaxDevices];
  if (dev < kMaxDevices && done[dev].load(std::memory_order_acquire)) return DNXCU_OK;
  const void *k[] = {(const void *)linear_tile<1, false, false>, (const void *)linear_tile<1, true, false>,
                     (const void *)linear_tile<2, false, false>, (const void *)linear_tile<2, true, false>,
                     (const void *)linear_tile<1, false, true>,  (const void *)linear_tile<1, true, true>,
                     (const void *)linear_split<false>,          (const void *)linear_split<true>};
  for (const void *f : k) DNXCU_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemLimit));
  if (dev < kMaxDevices) done[dev].store(1, std::memory_order_release);
  return DNXCU_OK;
}

int round_up(int v, int m) { return (v + m - 1) / m * m; }

void plan_tile(const Rec &r, int sms, bool any, dnxcu_linear_plan *p) {
  LinArgs &a = p->a;
  // a pair of blocks (256 rows) where there are enough rows and channels to fill the machine with such tiles
  const long long m128 = (a.M + 127) / 128;
  int bn = a.N <= 256 ? round_up(a.N, 16) : 256;
  const bool pair = !any && bn == 256 && (m128 + 1) / 2 * ((a.N + 255) / 256) * 2 >= sms;
  if (!pair) {
    if (any) bn = bn > 128 ? 128 : bn;
    while (bn > 64 && m128 * ((a.N + bn - 1) / bn) < sms) bn = bn > 128 ? 128 : 64;
    if (a.N > bn && bn % 64) bn = round_up(bn, 64);
  }
  const int cg = pair ? 2 : 1;
  a.BN = bn;
  a.mt = (int)((a.M + 128ll * cg - 1) / (128 * cg));
  a.nt = (a.N + bn - 1) / bn;
  const uint32_t stage = 16384u + (uint32_t)(bn / cg) * 128u;
  const uint32_t fixed = 1024u + TILE_FIXED + 8u * STAGING;
  a.stages = (int)((kSmemLimit - fixed) / stage);
  if (a.stages > MAX_STAGES) a.stages = MAX_STAGES;
  p->smem = fixed + stage * (uint32_t)a.stages;
  const long long tiles = (long long)a.mt * a.nt;
  const int clusters = (int)(tiles < sms / cg ? tiles : sms / cg);
  p->grid = dim3((unsigned)(clusters * cg));
  p->block = dim3(TILE_THREADS);
  p->cluster = (uint32_t)cg;
  if (any) p->kernel = r.f8 ? (const void *)linear_tile<1, true, true> : (const void *)linear_tile<1, false, true>;
  else if (pair) p->kernel = r.f8 ? (const void *)linear_tile<2, true, false> : (const void *)linear_tile<2, false, false>;
  else p->kernel = r.f8 ? (const void *)linear_tile<1, true, false> : (const void *)linear_tile<1, false, false>;
}

void plan_split(const Rec &r, int sms, dnxcu_linear_plan *p) {
  LinArgs &a = p->a;
  a.BN = a.M >= 256 ? 256 : round_up(a.M, 16);
  a.mt = (a.M + a.BN - 1) / a.BN;
  a.nt = (a.N + 127) / 128;
  const long long tiles = (long long)a.mt * a.nt;
  int s = 1;
  while (s < 8 && s < a.kb && tiles * s < sms) ++s;
  if (s > a.kb) s = a.kb;
  a.split = s;
  const uint32_t stage = 16384u + (uint32_t)a.BN * 128u, part = (uint32_t)a.BN * 512u;
  int st = (int)((kSmemLimit / 2 - 2048u) / stage);  // two blocks per SM where that leaves enough stages
  if (st < 3) st = (int)((kSmemLimit - 2048u) / stage);
  a.stages = st > MAX_STAGES ? MAX_STAGES : st;
  const uint32_t body = stage * (uint32_t)a.stages;
  p->smem = 2048u + (body > part ? body : part);
  p->grid = dim3((unsigned)(a.nt * s), (unsigned)a.mt);
  p->block = dim3(SPLIT_THREADS);
  p->cluster = (uint32_t)s;
  p->kernel = r.f8 ? (const void *)linear_split<true> : (const void *)linear_split<false>;
}

int make_plan(const Rec &r, dnxcu_linear_plan *p) {
  const dnxcu_linear &d = r.d;
  const int v = pick(r);
  if (v < 0) return v;
  p->variant = v;
  DNXCU_CUDA(cudaGetDevice(&p->device));
  for (const void *q : {d.x, d.weights, (const void *)d.x_scale, (const void *)d.w_scale, d.bias, d.residual, (const void *)d.out,
                        (const void *)d.device_status})
    if (!on_current_device(q)) return DNXCU_E_BAD_ARG;
  const int sms = sm_count(p->device);
  LinArgs &a = p->a;
  memset(&a, 0, sizeof(a));
  a.x = (const uint8_t *)d.x;
  a.w = (const uint8_t *)d.weights;
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
  a.kb = (d.c_in * r.es + 127) / 128;
  a.status = d.device_status;
  a.wait_limit = wait_limit_cycles();
  if (a.wait_limit < 2000000ull) a.wait_limit |= 1ull << 63;  // below about a millisecond: strict (see mbar_wait)
  if (v == DNXCU_LINEAR_ROWS) {
    p->grid = dim3((unsigned)((a.N + 15) / 16));
    p->block = dim3(ROWS_THREADS);
    if (r.f8) p->kernel = a.M <= 8 ? (const void *)linear_rows<true, 1> : (const void *)linear_rows<true, 2>;
    else p->kernel = a.M <= 8 ? (const void *)linear_rows<false, 1> : (const void *)linear_rows<false, 2>;
    return DNXCU_OK;
  }
  int st = init_device(p->device);
  if (st) return st;
  if (v == DNXCU_LINEAR_SPLIT) {
    plan_split(r, sms, p);
    st = matrix_map(&a.tm_w, d.weights, r.f8, a.N, a.K, a.ws, 128);
    return st ? st : matrix_map(&a.tm_x, d.x, r.f8, a.M, a.K, a.xs, a.BN);
  }
  plan_tile(r, sms, v == DNXCU_LINEAR_ANY, p);
  if (v == DNXCU_LINEAR_TILE) {
    st = matrix_map(&a.tm_x, d.x, r.f8, a.M, a.K, a.xs, 128);
    if (!st) st = matrix_map(&a.tm_w, d.weights, r.f8, a.N, a.K, a.ws, a.BN / (int)p->cluster);
    if (st) return st;
  }
  a.out_tma = mappable(d.out, a.os * 2);
  a.res_tma = d.residual && mappable(d.residual, a.rs * 2);
  if (a.out_tma && (st = matrix_map(&a.tm_out, d.out, false, a.M, a.N, a.os * 2, 32))) return st;
  if (a.res_tma && (st = matrix_map(&a.tm_res, d.residual, false, a.M, a.N, a.rs * 2, 32))) return st;
  return DNXCU_OK;
}

int launch(const dnxcu_linear_plan &p, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = p.grid;
  cfg.blockDim = p.block;
  cfg.dynamicSmemBytes = p.smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = p.cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.cluster > 1 ? 1 : 0;
  void *args[] = {const_cast<LinArgs *>(&p.a)};
  DNXCU_CUDA(cudaLaunchKernelExC(&cfg, p.kernel, args));
  return DNXCU_OK;
}

}  // namespace
}  // namespace dnxcu

extern "C" {

int dnxcu_linear_validate(const dnxcu_linear *d) {
  Rec r;
  const int st = check(d, &r);
  if (st) return st;
  const int v = pick(r);
  return v < 0 ? v : DNXCU_OK;
}

int dnxcu_linear_pick(const dnxcu_linear *d) {
  Rec r;
  const int st = check(d, &r);
  return st ? st : pick(r);
}

int dnxcu_linear_launch(const dnxcu_linear *d, void *stream) {
  Rec r;
  int st = check(d, &r);
  if (st) return st;
  dnxcu_linear_plan p;
  st = make_plan(r, &p);
  return st ? st : launch(p, (cudaStream_t)stream);
}

int dnxcu_linear_plan_create(const dnxcu_linear *d, dnxcu_linear_plan **out) {
  if (!out) return DNXCU_E_BAD_ARG;
  Rec r;
  int st = check(d, &r);
  if (st) return st;
  dnxcu_linear_plan *p = new (std::nothrow) dnxcu_linear_plan();
  if (!p) return DNXCU_E_NO_MEMORY;
  st = make_plan(r, p);
  if (st) {
    delete p;
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

void dnxcu_linear_plan_destroy(dnxcu_linear_plan *p) { delete p; }

}  // extern "C"
