// Root-mean-square norm over the channels of each row, with the residual's addition in front and, on request, an
// 8 bit output with one scale per row.
//
//   h = x + residual,  y = weight * h / sqrt(mean(h^2) + eps)
//   8 bits:  scale = max|y| / 448,  q = y / scale
//
// One pass over the data: a row's elements stay in registers between the statistics and the output.  The row's
// largest |y| needs no second reduction: 1 / rms is a positive constant of the row, so max|y| = max|weight * h| / rms
// is taken beside the sum of squares, and q = (weight * h) * (448 / max|weight * h|) does not need rms at all.
// The maximum carries a NaN along, so a row that is not finite shows in it; across threads it is taken on the bit patterns,
// whose unsigned order is the values' order with NaN above infinity: one integer `redux` does a warp's.
// With an 8 bit output weight * h takes h's place in the registers as soon as the sum is stored: one product and one fetch of
// the weights per element instead of two, which is power, and that is clock (1000 W are reached by this kernel too).
//
// Bound by bytes: 16384 rows of 4096 with residual to e4m3 72.5 us (6.5 TB/s), 2088960 rows of 32 43.8 us (6.1 TB/s).  Six
// forms, by the row's length and by what the alignment allows (V elements per access, 16 bytes
// where every pointer and stride is a multiple of that):
//   warp form  rows of at most 512 channels: a power of two of lanes per row, several rows per warp; every thread
//              has 32 elements in flight whatever the row's length (U rows of E elements, U * E = 32);
//   block form rows up to 32 elements x 1024 threads: a block per row;
//   shifted form  rows off 16 byte boundaries, but all tensors of the call alike: 16 byte accesses inside the row, single
//              elements at its two ends;
//   packed form   short packed rows of an odd number of channels: groups of rows as one piece of memory;
//   loop form  anything longer (or long and unaligned): a block per row that reads it twice, the second time from L2.
#include "internal.h"
#include <math.h>

namespace dnxcu {
namespace {

struct NormArgs {
  const __half *x, *residual, *weight;
  __half *sum;
  void *out;
  float *scale;
  long long rows, xs, rs, ss, os;  // strides in elements
  int C;
  float eps, inv_c;
};

template <int V> struct Vec;
template <> struct Vec<8> { typedef uint4 H; typedef uint2 Q; };
template <> struct Vec<4> { typedef uint2 H; typedef uint32_t Q; };
template <> struct Vec<2> { typedef uint32_t H; typedef uint16_t Q; };
template <> struct Vec<1> { typedef uint16_t H; typedef uint8_t Q; };

template <int V>
union Halves {
  typename Vec<V>::H v;
  __half h[V];
};

// max(a, |b|), NaN when either is: the largest value of a row also tells whether all of it is finite.
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

// Loads of data that an output of the same call may alias are plain loads (never the read-only path); every thread
// reads an element before it writes it, and no thread reads another's.
// Raw first, all of a thread's loads before the first conversion: that is what keeps them in flight together.
template <int V, bool RES>
struct Raw {
  typename Vec<V>::H x, r;
};
template <int V, bool RES>
__device__ __forceinline__ void load_raw(const NormArgs &g, long long row, int c, bool in, Raw<V, RES> &a) {
  a.x = typename Vec<V>::H();
  if (RES) a.r = typename Vec<V>::H();
  if (in) {
    a.x = *reinterpret_cast<const typename Vec<V>::H *>(g.x + row * g.xs + c);
    if (RES) a.r = *reinterpret_cast<const typename Vec<V>::H *>(g.residual + row * g.rs + c);
  }
}
template <int V, bool RES>
__device__ __forceinline__ void sum_raw(const Raw<V, RES> &a, float (&h)[V]) {
  Halves<V> t;
  t.v = a.x;
#pragma unroll
  for (int e = 0; e < V; ++e) h[e] = __half2float(t.h[e]);
  if (RES) {
    t.v = a.r;
#pragma unroll
    for (int e = 0; e < V; ++e) h[e] += __half2float(t.h[e]);
  }
}
template <int V>
__device__ __forceinline__ void load_weight(const NormArgs &g, int c, float (&w)[V]) {
  if (g.weight) {
    Halves<V> a;
    a.v = __ldg(reinterpret_cast<const typename Vec<V>::H *>(g.weight + c));
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = __half2float(a.h[e]);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = 1.0f;
  }
}
// Two values to binary16 or e4m3 at once.  The packed conversions run on the wide pipes; single ones go through the
// transcendental unit, a fraction as wide.
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint16_t pack_e4m3(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
template <int V>
__device__ __forceinline__ void store_halves(__half *p, const float (&y)[V]) {
  union {
    typename Vec<V>::H v;
    uint32_t w[(V + 1) / 2];
  } a;
  if constexpr (V == 1) {
    *reinterpret_cast<uint16_t *>(p) = (uint16_t)pack_f16(y[0], 0.0f);
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) a.w[e / 2] = pack_f16(y[e], y[e + 1]);
    *reinterpret_cast<typename Vec<V>::H *>(p) = a.v;
  }
}
template <int V>
__device__ __forceinline__ void store_sum(const NormArgs &g, long long row, int c, const float (&h)[V]) {
  store_halves<V>(g.sum + row * g.ss + c, h);
}
// y = weight * h * f, rounded once to the output type.  8 bits: `h` is weight * h already and f = 448 / max|weight * h|; a
// product that the last bit of f puts above 448 saturates to it.
template <int V, bool Q>
__device__ __forceinline__ void store_out(const NormArgs &g, long long row, int c, const float (&h)[V], const float (&w)[V],
                                          float f) {
  float y[V];
#pragma unroll
  for (int e = 0; e < V; ++e) y[e] = Q ? h[e] * f : h[e] * f * w[e];
  if constexpr (!Q) {
    store_halves<V>((__half *)g.out + row * g.os + c, y);
  } else if constexpr (V == 1) {
    ((uint8_t *)g.out)[row * g.os + c] = (uint8_t)pack_e4m3(y[0], 0.0f);
  } else {
    union {
      typename Vec<V>::Q v;
      uint16_t w[V / 2];
    } q;
#pragma unroll
    for (int e = 0; e < V; e += 2) q.w[e / 2] = pack_e4m3(y[e], y[e + 1]);
    *reinterpret_cast<typename Vec<V>::Q *>((uint8_t *)g.out + row * g.os + c) = q.v;
  }
}
// The row's factor from its statistics; `top` = bits of max|weight * h|.
template <bool Q>
__device__ __forceinline__ float row_factor(const NormArgs &g, float ss, uint32_t top, float *scale) {
  const float rstd = 1.0f / sqrtf(ss * g.inv_c + g.eps);
  if (!Q) return rstd;
  if (top >= 0x7f800000u) {  // a value that is not finite: the whole row is NaN
    *scale = __uint_as_float(0x7fffffffu);
    return *scale;
  }
  if (top == 0) {
    *scale = 1.0f;
    return 0.0f;
  }
  *scale = __uint_as_float(top) * rstd * (1.0f / 448.0f);
  return 448.0f / __uint_as_float(top);
}

// ---- warp form --------------------------------------------------------------
// 2^LT lanes per row; a thread holds vectors t, t + 2^LT, ... of U rows.
template <int V, int E, bool Q, bool RES>
__global__ void __launch_bounds__(256) rmsnorm_warp(NormArgs g, int lt) {
  constexpr int N = E / V, U = 32 / E;
  const int tpr = 1 << lt, t = threadIdx.x & (tpr - 1);
  const int per_block = (int)blockDim.x >> lt;
  const long long rows_per_block = (long long)per_block * U;
  const int nv = g.C / V;
  for (long long r0 = (long long)blockIdx.x * rows_per_block; r0 < g.rows; r0 += (long long)gridDim.x * rows_per_block) {
    Raw<V, RES> raw[U][N];
    long long row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      row[u] = r0 + (long long)u * per_block + (threadIdx.x >> lt);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int vi = t + (i << lt);
        load_raw<V, RES>(g, row[u], vi * V, row[u] < g.rows && vi < nv, raw[u][i]);
      }
    }
    float w[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int vi = t + (i << lt);
      if (vi < nv) load_weight<V>(g, vi * V, w[i]);
      else
#pragma unroll
        for (int e = 0; e < V; ++e) w[i][e] = 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float h[N][V], ss = 0.0f, most = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int vi = t + (i << lt);
        sum_raw<V, RES>(raw[u][i], h[i]);
        if (g.sum && row[u] < g.rows && vi < nv) store_sum<V>(g, row[u], vi * V, h[i]);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          ss = fmaf(h[i][e], h[i][e], ss);
          if (Q) {
            h[i][e] *= w[i][e];
            most = max_abs(most, h[i][e]);
          }
        }
      }
      uint32_t top = __float_as_uint(most);
      for (int o = tpr >> 1; o > 0; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (Q) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      }
      if (row[u] >= g.rows) continue;  // (no shuffle follows for this row)
      float scale = 0.0f;
      const float f = row_factor<Q>(g, ss, top, &scale);
      if (Q && t == 0) g.scale[row[u]] = scale;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int vi = t + (i << lt);
        if (vi < nv) store_out<V, Q>(g, row[u], vi * V, h[i], w[i], f);
      }
    }
  }
}

// Sum and maximum over the block; every thread gets both.  `turn` alternates between two halves of the buffer so that
// one barrier per row is enough.
__device__ __forceinline__ void block_reduce(float &ss, uint32_t &top, int turn) {
  __shared__ float s_sum[2][32];
  __shared__ uint32_t s_top[2][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = (int)blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) {
    s_sum[turn][warp] = ss;
    s_top[turn][warp] = top;
  }
  __syncthreads();
  ss = lane < nw ? s_sum[turn][lane] : 0.0f;
  top = lane < nw ? s_top[turn][lane] : 0u;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  top = __reduce_max_sync(0xffffffffu, top);
}

// ---- block form -------------------------------------------------------------
template <int V, int E, bool Q, bool RES>
__global__ void __launch_bounds__(1024) rmsnorm_block(NormArgs g) {
  constexpr int N = E / V;
  const int nv = g.C / V, t = threadIdx.x, nt = blockDim.x;
  int turn = 0;
  for (long long row = blockIdx.x; row < g.rows; row += gridDim.x, turn ^= 1) {
    Raw<V, RES> raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) load_raw<V, RES>(g, row, (t + i * nt) * V, t + i * nt < nv, raw[i]);
    float h[N][V], ss = 0.0f, most = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int vi = t + i * nt;
      sum_raw<V, RES>(raw[i], h[i]);
      if (g.sum && vi < nv) store_sum<V>(g, row, vi * V, h[i]);
#pragma unroll
      for (int e = 0; e < V; ++e) ss = fmaf(h[i][e], h[i][e], ss);
      if (Q && vi < nv) {
        float w[V];
        load_weight<V>(g, vi * V, w);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          h[i][e] *= w[e];
          most = max_abs(most, h[i][e]);
        }
      }
    }
    uint32_t top = __float_as_uint(most);
    block_reduce(ss, top, turn);
    float scale = 0.0f;
    const float f = row_factor<Q>(g, ss, top, &scale);
    if (Q && t == 0) g.scale[row] = scale;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int vi = t + i * nt;
      if (vi < nv) {
        float w[V];
        if (!Q) load_weight<V>(g, vi * V, w);  // (from L1: every row uses the same ones)
        store_out<V, Q>(g, row, vi * V, h[i], w, f);
      }
    }
  }
}

// ---- shifted form -----------------------------------------------------------
// Rows that start anywhere but all tensors of the call at the same place of a 16 byte word (packed rows of an odd number of
// channels): the row is walked in the words of memory, whose first and last one are partly the neighbours'.  Those two go
// element by element, everything between by 16 byte accesses; the weights, whose words lie otherwise, are two words shifted
// together.  LANES threads per row: a warp (several rows per block) or the block.
__device__ __forceinline__ uint4 shift_words(uint4 a, uint4 b, int from) {  // 8 elements from element `from` of a, b
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = from & 4 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = from & 2 ? w[i + 1] : w[i];
  const int bits = (from & 1) * 16;
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits),
                    __funnelshift_r(w[3], w[4], bits));
}
// One word of a row from element c on (c may be negative); `all`: it lies inside the row.
__device__ __forceinline__ uint4 load_word(const __half *row, int c, int C, bool all) {
  if (all) return *reinterpret_cast<const uint4 *>(row + c);
  union {
    uint4 v;
    uint16_t h[8];
  } a;
  a.v = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (c + e >= 0 && c + e < C) a.h[e] = *reinterpret_cast<const uint16_t *>(row + c + e);
  return a.v;
}
template <class T>
__device__ __forceinline__ void store_edge(T *row, int c, int C, const T (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (c + e >= 0 && c + e < C) row[c + e] = v[e];
}
template <int E, bool Q, bool RES, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) rmsnorm_shift(NormArgs g, int w_aligned) {
  constexpr int N = E / 8;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x, nt = WARP ? 32 : blockDim.x;
  const long long row0 = WARP ? blockIdx.x * 8ll + (threadIdx.x >> 5) : blockIdx.x, step = WARP ? gridDim.x * 8ll : gridDim.x;
  int turn = 0;
  for (long long row = row0; row < g.rows; row += step, turn ^= 1) {
    const __half *x = g.x + row * g.xs, *r = RES ? g.residual + row * g.rs : nullptr;
    const int lead = (int)(((uintptr_t)x >> 1) & 7), words = (lead + g.C + 7) >> 3;
    uint4 vx[N], vr[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = t + i * nt, c = 8 * k - lead;
      const bool all = c >= 0 && c + 8 <= g.C;
      vx[i] = vr[i] = make_uint4(0, 0, 0, 0);
      if (k < words) {
        vx[i] = load_word(x, c, g.C, all);
        if (RES) vr[i] = load_word(r, c, g.C, all);
      }
    }
    const auto weight = [&](int k, int c, float (&w)[8]) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (!g.weight) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = 1.0f;
        return;
      }
      if (w_aligned && c >= 0 && 8 * k + 8 <= g.C) {
        const uint4 *wp = reinterpret_cast<const uint4 *>(g.weight) + k;
        v = lead ? shift_words(__ldg(wp - 1), __ldg(wp), 8 - lead) : __ldg(wp);
      } else {
        v = load_word(g.weight, c, g.C, false);
      }
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[e]));
        w[2 * e] = f.x;
        w[2 * e + 1] = f.y;
      }
    };
    float h[N][8], ss = 0.0f, most = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      Raw<8, RES> raw;
      raw.x = vx[i];
      if (RES) raw.r = vr[i];
      sum_raw<8, RES>(raw, h[i]);
      const int k = t + i * nt, c = 8 * k - lead;
      if (g.sum && k < words) {
        if (c >= 0 && c + 8 <= g.C) {
          store_sum<8>(g, row, c, h[i]);
        } else {
          __half v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = __float2half_rn(h[i][e]);
          store_edge(g.sum + row * g.ss, c, g.C, v);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(h[i][e], h[i][e], ss);
      if (Q && k < words) {
        float w[8];
        weight(k, c, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // (an element of the word that is not the row's is 0 and has weight 0, or 1 without weights)
          h[i][e] *= w[e];
          most = max_abs(most, h[i][e]);
        }
      }
    }
    uint32_t top = __float_as_uint(most);
    if (WARP) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (Q) top = __reduce_max_sync(0xffffffffu, top);
    } else {
      block_reduce(ss, top, turn);
    }
    float scale = 0.0f;
    const float f = row_factor<Q>(g, ss, top, &scale);
    if (Q && t == 0) g.scale[row] = scale;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int k = t + i * nt, c = 8 * k - lead;
      if (k >= words) continue;
      const bool all = c >= 0 && c + 8 <= g.C;
      float w[8];
      if (!Q) weight(k, c, w);
      if (all) {
        store_out<8, Q>(g, row, c, h[i], w, f);
      } else if (Q) {
        uint8_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (uint8_t)pack_e4m3(h[i][e] * f, 0.0f);
        store_edge((uint8_t *)g.out + row * g.os, c, g.C, v);
      } else {
        __half v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __float2half_rn(h[i][e] * f * w[e]);
        store_edge((__half *)g.out + row * g.os, c, g.C, v);
      }
    }
  }
}

// ---- packed form ------------------------------------------------------------
// Short packed rows of a number of channels that no wide access divides: a block takes a group of rows (a multiple of 16,
// so that the group starts on a 16 byte boundary in every tensor) as one piece of memory, by 16 byte accesses whatever the
// rows.  A thread keeps its vectors in registers and shows them to the others in shared memory, where `lanes` threads per
// row add it up; then every thread finishes its own vectors with the factors of the rows they touch.
constexpr int kPackElems = 4096;
template <bool Q, bool RES>
__global__ void __launch_bounds__(256) rmsnorm_packed(NormArgs g, int group, int log_lanes) {
  constexpr int NV = kPackElems / 8 / 256;
  __shared__ __align__(16) float s_h[kPackElems];
  __shared__ float s_w[256], s_f[kPackElems / 2];
  const int C = g.C, t = threadIdx.x;
  for (int i = t; i < C; i += 256) s_w[i] = g.weight ? __half2float(__ldg(g.weight + i)) : 1.0f;
  for (long long r0 = (long long)blockIdx.x * group; r0 < g.rows; r0 += (long long)gridDim.x * group) {
    const int rows = (int)(g.rows - r0 < group ? g.rows - r0 : group), n = rows * C;
    const __half *x = g.x + r0 * C, *r = RES ? g.residual + r0 * C : nullptr;
    uint4 vx[NV], vr[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int e0 = (t + 256 * k) * 8;
      vx[k] = vr[k] = make_uint4(0, 0, 0, 0);
      if (e0 < n) {
        vx[k] = load_word(x, e0, n, e0 + 8 <= n);
        if (RES) vr[k] = load_word(r, e0, n, e0 + 8 <= n);
      }
    }
    float h[NV][8];
    __syncthreads();  // (the group before is done with the shared arrays)
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int e0 = (t + 256 * k) * 8;
      Raw<8, RES> raw;
      raw.x = vx[k];
      if (RES) raw.r = vr[k];
      sum_raw<8, RES>(raw, h[k]);
      *reinterpret_cast<float4 *>(s_h + e0) = make_float4(h[k][0], h[k][1], h[k][2], h[k][3]);
      *reinterpret_cast<float4 *>(s_h + e0 + 4) = make_float4(h[k][4], h[k][5], h[k][6], h[k][7]);
    }
    __syncthreads();
    const int lanes = 1 << log_lanes, l = t & (lanes - 1);
    for (int q = t >> log_lanes; q < ((rows + (256 >> log_lanes) - 1) & ~((256 >> log_lanes) - 1)); q += 256 >> log_lanes) {
      float ss = 0.0f, most = 0.0f;
      if (q < rows)
        for (int j = l; j < C; j += lanes) {
          const float v = s_h[q * C + j];
          ss = fmaf(v, v, ss);
          if (Q) most = max_abs(most, v * s_w[j]);
        }
      uint32_t top = __float_as_uint(most);
      for (int o = lanes >> 1; o > 0; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (Q) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      }
      if (q < rows && l == 0) {
        float scale = 0.0f;
        s_f[q] = row_factor<Q>(g, ss, top, &scale);
        if (Q) g.scale[r0 + q] = scale;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int e0 = (t + 256 * k) * 8;
      if (e0 >= n) continue;
      int row = e0 / C, c = e0 - row * C;
      float f[8], w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] = s_f[min(row, rows - 1)];
        w[e] = s_w[c];
        if (++c == C) {
          c = 0;
          ++row;
        }
      }
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = Q ? h[k][e] * w[e] * f[e] : h[k][e] * f[e] * w[e];
      if (e0 + 8 <= n) {
        if (g.sum) store_halves<8>(g.sum + r0 * C + e0, h[k]);
        if (Q) {
          union {
            uint2 v;
            uint16_t p[4];
          } o;
#pragma unroll
          for (int e = 0; e < 8; e += 2) o.p[e / 2] = pack_e4m3(y[e], y[e + 1]);
          *reinterpret_cast<uint2 *>((uint8_t *)g.out + r0 * C + e0) = o.v;
        } else {
          store_halves<8>((__half *)g.out + r0 * C + e0, y);
        }
      } else {
        for (int e = 0; e0 + e < n; ++e) {
          if (g.sum) g.sum[r0 * C + e0 + e] = __float2half_rn(s_h[e0 + e]);
          const int rr = (e0 + e) / C;
          const float v = s_h[e0 + e], ww = s_w[e0 + e - rr * C], ff = s_f[rr];
          if (Q) ((uint8_t *)g.out)[r0 * C + e0 + e] = (uint8_t)pack_e4m3(v * ww * ff, 0.0f);
          else ((__half *)g.out)[r0 * C + e0 + e] = __float2half_rn(v * ff * ww);
        }
      }
    }
  }
}

// ---- loop form --------------------------------------------------------------
template <int V, bool Q, bool RES>
__global__ void __launch_bounds__(1024) rmsnorm_loop(NormArgs g) {
  const int nv = g.C / V, t = threadIdx.x, nt = blockDim.x;
  int turn = 0;
  for (long long row = blockIdx.x; row < g.rows; row += gridDim.x, turn ^= 1) {
    double sum = 0.0;  // (a thread may add thousands of terms one after the other)
    float most = 0.0f;
#pragma unroll 4
    for (int vi = t; vi < nv; vi += nt) {
      float h[V], w[V];
      Raw<V, RES> raw;
      load_raw<V, RES>(g, row, vi * V, true, raw);
      sum_raw<V, RES>(raw, h);
      if (Q) load_weight<V>(g, vi * V, w);
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        ss = fmaf(h[e], h[e], ss);
        if (Q) most = max_abs(most, h[e] * w[e]);
      }
      sum += ss;
    }
    float ss = (float)sum;
    uint32_t top = __float_as_uint(most);
    block_reduce(ss, top, turn);
    float scale = 0.0f;
    const float f = row_factor<Q>(g, ss, top, &scale);
    if (Q && t == 0) g.scale[row] = scale;
#pragma unroll 4
    for (int vi = t; vi < nv; vi += nt) {
      float h[V], w[V];
      Raw<V, RES> raw;
      load_raw<V, RES>(g, row, vi * V, true, raw);
      sum_raw<V, RES>(raw, h);
      load_weight<V>(g, vi * V, w);
      if (g.sum) store_sum<V>(g, row, vi * V, h);
      if (Q) {
#pragma unroll
        for (int e = 0; e < V; ++e) h[e] *= w[e];
      }
      store_out<V, Q>(g, row, vi * V, h, w, f);
    }
  }
}

constexpr unsigned kMaxGrid = 0x7fffffffu;
// Channels from which the shifted form beats accesses of one element: 65536 rows of 255: 41.8 against 39.9 us, of 257 with
// residual to e4m3 71 against 154, 16384 of 999 21.7 against 117, of 5001 79 against 174.
constexpr int kShiftFrom = 256;

template <int V, bool Q, bool RES>
cudaError_t launch_v(const NormArgs &g, cudaStream_t s) {
  const int nv = g.C / V;
  const auto enqueue = [&](const void *kernel, unsigned grid, int threads, int lt = 0) {
    void *args[] = {const_cast<NormArgs *>(&g), &lt};  // (only the warp form takes the second)
    return cudaLaunchKernel(kernel, dim3(grid), dim3((unsigned)threads), args, 0, s);
  };
  if (g.C <= 512) {
    // the fewest lanes (a power of two) that hold the row in 8 or 16 elements per thread, most rows per warp first (with 32,
    // up to 1024 channels, the registers leave too few warps: 50000 rows of 1024 52.8 us, 34.6 in the block form)
    const int e = g.C <= 256 ? 8 : 16;
    int lt = 0;
    while ((e / V) << lt < nv) ++lt;
    const long long per_block = (256 >> lt) * (32 / e);
    const long long blocks = (g.rows + per_block - 1) / per_block;
    const unsigned grid = (unsigned)(blocks < kMaxGrid ? blocks : kMaxGrid);
    return enqueue(e == 8 ? (const void *)rmsnorm_warp<V, 8, Q, RES> : (const void *)rmsnorm_warp<V, 16, Q, RES>, grid, 256, lt);
  }
  const unsigned grid = (unsigned)(g.rows < kMaxGrid ? g.rows : kMaxGrid);
  const auto threads = [&](int e) {
    const int n = e / V, t = (nv + n - 1) / n;
    return (t + 31) / 32 * 32;
  };
  // few rows: as many threads per row as there are, for latency; many rows: 32 elements in flight per thread
  if (g.rows <= 148 && threads(8) <= 1024) return enqueue((const void *)rmsnorm_block<V, 8, Q, RES>, grid, threads(8));
  if (g.rows <= 148 && threads(16) <= 1024) return enqueue((const void *)rmsnorm_block<V, 16, Q, RES>, grid, threads(16));
  if (threads(32) <= 1024) return enqueue((const void *)rmsnorm_block<V, 32, Q, RES>, grid, threads(32));
  return enqueue((const void *)rmsnorm_loop<V, Q, RES>, grid, 1024);
}

// Whether all rows of the call start at the same place of a 16 byte word (of an 8 byte word for an 8 bit output).
bool same_lead(const NormArgs &g, bool q) {
  const auto lead = [](const void *p, int es) { return (int)((uintptr_t)p / es) & 7; };
  const int a = lead(g.x, 2), s = (int)(g.xs & 7);
  if (g.residual && (lead(g.residual, 2) != a || (int)(g.rs & 7) != s)) return false;
  if (g.sum && (lead(g.sum, 2) != a || (int)(g.ss & 7) != s)) return false;
  return lead(g.out, q ? 1 : 2) == a && (int)(g.os & 7) == s;
}
template <bool Q, bool RES>
cudaError_t launch_shift(const NormArgs &g, cudaStream_t s) {
  int aligned = ((uintptr_t)g.weight & 15) == 0;
  void *args[] = {const_cast<NormArgs *>(&g), &aligned};
  const int words = (g.C + 14) / 8;  // of the widest row
  const auto blocks = [](long long n) { return dim3((unsigned)(n < kMaxGrid ? n : kMaxGrid)); };
  if (words <= 64) {
    const void *k = words <= 32 ? (const void *)rmsnorm_shift<8, Q, RES, true> : (const void *)rmsnorm_shift<16, Q, RES, true>;
    return cudaLaunchKernel(k, blocks((g.rows + 7) / 8), dim3(256), args, 0, s);
  }
  const bool few = g.rows <= 148;
  const int n = few && words <= 1024 ? 1 : few && words <= 2048 ? 2 : 4, threads = ((words + n - 1) / n + 31) / 32 * 32;
  const void *k = n == 1   ? (const void *)rmsnorm_shift<8, Q, RES, false>
                  : n == 2 ? (const void *)rmsnorm_shift<16, Q, RES, false>
                           : (const void *)rmsnorm_shift<32, Q, RES, false>;
  return cudaLaunchKernel(k, blocks(g.rows), dim3((unsigned)threads), args, 0, s);
}

// Packed rows of every tensor, all starting on a 16 byte boundary (8 for an 8 bit output).
bool packed(const NormArgs &g, bool q) {
  const uintptr_t at = (uintptr_t)g.x | (uintptr_t)g.residual | (uintptr_t)g.sum | (uintptr_t)g.out << (q ? 1 : 0);
  return !(at & 15) && g.xs == g.C && g.os == g.C && (!g.residual || g.rs == g.C) && (!g.sum || g.ss == g.C);
}
template <bool Q, bool RES>
cudaError_t launch_packed(const NormArgs &g, cudaStream_t s) {
  int group = kPackElems / g.C / 16 * 16, log_lanes = 0;
  if (group > kPackElems / 2) group = kPackElems / 2;
  while (log_lanes < 5 && (group << (log_lanes + 1)) <= 256) ++log_lanes;
  void *args[] = {const_cast<NormArgs *>(&g), &group, &log_lanes};
  const long long n = (g.rows + group - 1) / group;
  return cudaLaunchKernel((const void *)rmsnorm_packed<Q, RES>, dim3((unsigned)(n < kMaxGrid ? n : kMaxGrid)), dim3(256), args, 0, s);
}

template <int V>
cudaError_t launch_q(const NormArgs &g, bool q, cudaStream_t s) {
  if (q && g.residual) return launch_v<V, true, true>(g, s);
  if (q) return launch_v<V, true, false>(g, s);
  if (g.residual) return launch_v<V, false, true>(g, s);
  return launch_v<V, false, false>(g, s);
}

// The record with packed strides filled in, or why it cannot run.
int check(const dnxcu_rmsnorm *d, NormArgs *g) {
  if (!d || !d->x || !d->out || d->rows <= 0 || d->channels <= 0 || d->reserved) return DNXCU_E_BAD_ARG;
  if (d->out_dtype != DNXCU_DT_F16 && d->out_dtype != DNXCU_DT_E4M3) return DNXCU_E_BAD_ARG;
  const bool q = d->out_dtype == DNXCU_DT_E4M3;
  if (q != (d->out_scale != nullptr)) return DNXCU_E_BAD_ARG;
  if (!(d->eps > 0.0f) || !isfinite(d->eps)) return DNXCU_E_BAD_ARG;
  const long long C = d->channels, kStride = 1ll << 35;
  if (d->rows > 0x7fffffffll || C > (1 << 24)) return DNXCU_E_LIMIT;
  const long long xs = d->x_stride ? d->x_stride : C, rs = d->residual_stride ? d->residual_stride : C;
  const long long ss = d->sum_stride ? d->sum_stride : C, os = d->out_stride ? d->out_stride : C;
  if (xs < C || rs < C || ss < C || os < C) return DNXCU_E_BAD_ARG;
  if (xs >= kStride || rs >= kStride || ss >= kStride || os >= kStride) return DNXCU_E_LIMIT;
  const uintptr_t halves = (uintptr_t)d->x | (uintptr_t)d->residual | (uintptr_t)d->weight | (uintptr_t)d->sum_out |
                           (q ? 0 : (uintptr_t)d->out);
  if ((halves & 1) || ((uintptr_t)d->out_scale & 3)) return DNXCU_E_MISALIGNED;
  const RowSpan x{d->x, d->rows, C, xs, 2}, res{d->residual, d->rows, C, rs, 2}, w{d->weight, 1, C, C, 2};
  const RowSpan sum{d->sum_out, d->rows, C, ss, 2}, out{d->out, d->rows, C, os, q ? 1 : 2};
  const RowSpan sc{d->out_scale, 1, d->rows, d->rows, 4};
  const auto same = [](const RowSpan &a, const RowSpan &b) { return a.p == b.p && a.stride == b.stride && a.es == b.es; };
  const auto clash = [&](const RowSpan &o, const RowSpan &in) { return !same(o, in) && rows_overlap(o, in); };
  if (clash(sum, x) || clash(sum, res) || clash(out, x) || clash(out, res)) return DNXCU_E_BAD_ARG;
  if (rows_overlap(sum, w) || rows_overlap(out, w) || rows_overlap(sum, out)) return DNXCU_E_BAD_ARG;
  if (rows_overlap(sc, x) || rows_overlap(sc, res) || rows_overlap(sc, w) || rows_overlap(sc, sum) || rows_overlap(sc, out))
    return DNXCU_E_BAD_ARG;
  g->x = (const __half *)d->x;
  g->residual = (const __half *)d->residual;
  g->weight = (const __half *)d->weight;
  g->sum = (__half *)d->sum_out;
  g->out = d->out;
  g->scale = d->out_scale;
  g->rows = d->rows;
  g->C = d->channels;
  g->xs = xs;
  g->rs = rs;
  g->ss = ss;
  g->os = os;
  g->eps = d->eps;
  g->inv_c = (float)(1.0 / (double)C);
  return DNXCU_OK;
}

}  // namespace

bool rows_overlap(const RowSpan &a, const RowSpan &b) {
  if (!a.p || !b.p) return false;
  const long long sa = a.stride * a.es, sb = b.stride * b.es, la = a.len * a.es, lb = b.len * b.es;
  const uintptr_t a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p;
  const uintptr_t a1 = a0 + (uintptr_t)((a.rows - 1) * sa + la), b1 = b0 + (uintptr_t)((b.rows - 1) * sb + lb);
  if (a1 <= b0 || b1 <= a0) return false;
  if (sa != sb || a.rows < 2 || b.rows < 2) return true;  // (two interleaved spans of different pitch: taken as overlapping)
  // same pitch: windows of the same wider rows; b's start within a's row, wrapped into one pitch
  const long long d = b0 >= a0 ? (long long)((b0 - a0) % (uintptr_t)sa) : (sa - (long long)((a0 - b0) % (uintptr_t)sa)) % sa;
  return d < la || d + lb > sa;
}

bool on_current_device(const void *p) {
  if (!p) return true;
  cudaPointerAttributes at;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaPointerGetAttributes(&at, p) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  if (at.type == cudaMemoryTypeDevice) return at.device == dev;
  return at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeHost && at.devicePointer == p);
}

}  // namespace dnxcu

using namespace dnxcu;

extern "C" {

int dnxcu_rmsnorm_validate(const dnxcu_rmsnorm *d) {
  NormArgs g;
  return check(d, &g);
}

int dnxcu_rmsnorm_launch(const dnxcu_rmsnorm *d, void *stream) {
  NormArgs g;
  const int st = check(d, &g);
  if (st) return st;
  if (!on_current_device(g.x) || !on_current_device(g.residual) || !on_current_device(g.weight) ||
      !on_current_device(g.sum) || !on_current_device(g.out) || !on_current_device(g.scale))
    return DNXCU_E_BAD_ARG;
  const bool q = d->out_dtype == DNXCU_DT_E4M3;
  // elements per access: what every pointer, stride and the row length are multiples of
  const auto fits = [&](int v) {
    const uintptr_t hb = (uintptr_t)v * 2 - 1, ob = (uintptr_t)v * (q ? 1 : 2) - 1;
    if (g.C % v || ((uintptr_t)g.x & hb) || g.xs % v || ((uintptr_t)g.weight & hb)) return false;
    if (g.residual && (((uintptr_t)g.residual & hb) || g.rs % v)) return false;
    if (g.sum && (((uintptr_t)g.sum & hb) || g.ss % v)) return false;
    return !((uintptr_t)g.out & ob) && g.os % v == 0;
  };
  cudaStream_t s = (cudaStream_t)stream;
  // (up to 1024 channels narrower accesses beat it where they are wider than one element: 50000 rows of 516: 49 against 38
  // us, of 1022 80 against 61; 16384 of 4098: 74 against 91, of 4100 with residual to e4m3 101 against 134)
  if (!fits(g.C <= 1024 ? 2 : 8) && g.C >= kShiftFrom && g.C <= 32768 - 14 && same_lead(g, q)) {
    const auto run = q ? (g.residual ? launch_shift<true, true> : launch_shift<true, false>)
                       : (g.residual ? launch_shift<false, true> : launch_shift<false, false>);
    DNXCU_CUDA(run(g, s));
    return DNXCU_OK;
  }
  // (an odd number of channels, or two tensors by 4 byte accesses: 2088960 rows of 9: 63.7 -> 28.3 us, 534016 of 29 with
  // residual to e4m3 96 -> 32, 522240 of 10 with residual 18.4 -> 12.3; without a residual 4 byte accesses are as fast)
  if ((!fits(2) || (g.residual && !fits(4))) && g.C < kShiftFrom && packed(g, q)) {
    const auto run = q ? (g.residual ? launch_packed<true, true> : launch_packed<true, false>)
                       : (g.residual ? launch_packed<false, true> : launch_packed<false, false>);
    DNXCU_CUDA(run(g, s));
    return DNXCU_OK;
  }
  DNXCU_CUDA(fits(8) ? launch_q<8>(g, q, s) : fits(4) ? launch_q<4>(g, q, s) : fits(2) ? launch_q<2>(g, q, s) : launch_q<1>(g, q, s));
  return DNXCU_OK;
}

}  // extern "C"
