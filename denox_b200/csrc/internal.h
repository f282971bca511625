// Internal declarations shared by the translation units of libdnxcu.
#pragma once
#include <cuda_runtime.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <stddef.h>
#include "dnxcu.h"

namespace dnxcu {

// Records a failing CUDA call for dnxcu_last_cuda_error and maps it to a status.
int cuda_fail(cudaError_t e);
#define DNXCU_CUDA(call)                                   \
  do {                                                     \
    cudaError_t _e = (call);                               \
    if (_e != cudaSuccess) return ::dnxcu::cuda_fail(_e);  \
  } while (0)

inline uint32_t cdiv(uint32_t a, uint32_t b) { return (a + b - 1) / b; }

enum VariantKind {
  VK_CONV_DIRECT = 0,  // CUDA core implicit GEMM, fp32 accumulate
  VK_CONV_TC,          // tcgen05 / TMEM implicit GEMM, fp32 accumulate
  VK_POOL,
  VK_UPSAMPLE,
  VK_CONCAT,
  VK_RELU,
  VK_PADC,
  VK_PAD_EDGE,
  VK_SLICE,
};

struct Variant {
  dnxcu_variant_desc desc;
  VariantKind kind;
  // tuning parameters (meaning depends on kind)
  int p0, p1, p2, p3;
  int p4 = 0;
  int p5 = 0;
};

const Variant *get_variant(int id);
int variant_count();

// ---- per family entry points (each validates what only it knows) ----------
int conv_direct_validate(const Variant &v, const dnxcu_dispatch &d);
int conv_direct_launch(const Variant &v, const dnxcu_dispatch &d, cudaStream_t s);
void conv_direct_grid(const Variant &v, const dnxcu_dispatch &d, uint32_t g[3]);
size_t conv_direct_weight_bytes(const Variant &v, int k, int ca, int cb);
void conv_direct_prepare(const Variant &v, const uint16_t *kcrs, int k, int ca, int cb, uint16_t *out);

int conv_tc_validate(const Variant &v, const dnxcu_dispatch &d);
int conv_tc_launch(const Variant &v, const dnxcu_dispatch &d, cudaStream_t s);
// A tensor core conv dispatch planned once (launch parameters + encoded tensor maps), launched many times.
struct ConvTcPlan;
int conv_tc_plan(const Variant &v, const dnxcu_dispatch &d, ConvTcPlan **out);
int conv_tc_launch_plan(const ConvTcPlan &p, cudaStream_t s);
void conv_tc_plan_free(ConvTcPlan *p);
// Sets the per-kernel attributes of every tensor core kernel on the current device (idempotent).
int conv_tc_init_device();
void conv_tc_grid(const Variant &v, const dnxcu_dispatch &d, uint32_t g[3]);
size_t conv_tc_weight_bytes(const Variant &v, int k, int ca, int cb);
void conv_tc_prepare(const Variant &v, const uint16_t *kcrs, int k, int ca, int cb, uint16_t *out);

int mem_launch(const Variant &v, const dnxcu_dispatch &d, cudaStream_t s);
void mem_grid(const Variant &v, const dnxcu_dispatch &d, uint32_t g[3]);

// Limit of every bounded device-side wait in clock64 ticks (dnxcu_set_wait_limit_us).
unsigned long long wait_limit_cycles();

// ---- token and pixel operators ---------------------------------------------
// A matrix of `rows` rows of `len` elements of `es` bytes, `stride` elements apart, for the argument checks.
struct RowSpan {
  const void *p;
  long long rows, len, stride;
  int es;
};
// Whether two row spans share a byte (exactly equal spans do; windows side by side in the same wider rows do not).
bool rows_overlap(const RowSpan &a, const RowSpan &b);
// Whether kernels on the current device may use the pointer: memory of this device, managed or registered host memory.
bool on_current_device(const void *p);

// Programmatic dependent launch.  A kernel launched with launch_dependent() may start while the kernels before it on the
// stream are still finishing: its set-up (barriers, tensor memory, descriptor fetches) hides behind them.  It calls
// pdl_wait() before its first access to memory that any of them may read or write, which returns when they are done and
// their writes are visible.  pdl_release() lets the kernel behind it start in the same way.
#ifdef __CUDACC__
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
#endif
inline cudaError_t launch_dependent(const void *kernel, dim3 grid, dim3 block, size_t smem, unsigned cluster, cudaStream_t s,
                                    void **args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelExC(&cfg, kernel, args);
}

// SHA-256 (hex) of a byte string; used for variant identities and database keys.
void sha256_hex(const void *data, size_t n, char out_hex[65]);

}  // namespace dnxcu
