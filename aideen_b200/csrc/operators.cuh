// Shared parts of the operators on caller-owned device tensors: host-side
// checks and messages, element types, vector access.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/aideen_b200.h"

namespace aideen {

// Message of the calling thread's last refused or failed operator call (a
// string literal or CUDA's own text: nothing is allocated).
void op_set_error(const char *why);
inline int op_invalid(const char *why) {
  op_set_error(why);
  return AIDEEN_E_INVALID;
}
inline int op_cuda(cudaError_t e) {
  if (e == cudaSuccess) return AIDEEN_OK;
  (void)cudaGetLastError();  // reported here: no later check of the caller's trips over it
  op_set_error(cudaGetErrorString(e));
  return AIDEEN_E_CUDA;
}
// SMs of the current device.
int op_sm_count();
// Reads and clears the current device's word that a bounded wait of the linear
// cross entropy sets when it runs out (host-synchronous).
cudaError_t linear_ce_timeout(unsigned int *out);

inline size_t op_elem(uint32_t dtype) { return dtype == AIDEEN_F32 ? 4 : 2; }
inline bool op_aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline size_t op_round(size_t n, size_t a) { return (n + a - 1) / a * a; }

// Hands out 256-byte aligned parts of a workspace; with base = nullptr it
// only adds up their sizes.
struct OpCarve {
  unsigned char *base;
  size_t used = 0;
  explicit OpCarve(void *p) : base(static_cast<unsigned char *>(p)) {}
  template <typename T>
  T *take(size_t n) {
    T *p = base ? reinterpret_cast<T *>(base + used) : nullptr;
    used += op_round(n * sizeof(T), 256);
    return p;
  }
};

// Launches of one call follow each other as programmatic dependents: a kernel may
// be placed, and set up what it needs, while the one before it in the stream drains.
// So every kernel of an operator calls op_begin() in all threads before it touches
// global memory, which waits until everything before it is complete and visible.
// With cluster > 0 the grid is launched in clusters of that many CTAs.
template <typename... P, typename... A>
cudaError_t op_launch_cluster(void (*kernel)(P...), unsigned cluster, dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                              A... args) {
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}
template <typename... P, typename... A>
cudaError_t op_launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... args) {
  return op_launch_cluster(kernel, 0, grid, block, smem, st, args...);
}
__device__ __forceinline__ void op_begin() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

#define OP_CHECK(cond, why)                        \
  do {                                             \
    if (!(cond)) return aideen::op_invalid(why);   \
  } while (0)

// ---- element types ---------------------------------------------------------
template <typename T>
__device__ __forceinline__ float op_load(T v);
template <>
__device__ __forceinline__ float op_load<float>(float v) { return v; }
template <>
__device__ __forceinline__ float op_load<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float op_load<__half>(__half v) { return __half2float(v); }

// One rounding to the stored type (round to nearest even).
template <typename T>
__device__ __forceinline__ T op_store(float v);
template <>
__device__ __forceinline__ float op_store<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 op_store<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half op_store<__half>(float v) { return __float2half_rn(v); }

// VEC consecutive elements, moved with one access of VEC * sizeof(T) bytes.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) OpVec {
  T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ void op_load_vec(const T *p, float (&out)[VEC]) {
  const OpVec<T, VEC> x = *reinterpret_cast<const OpVec<T, VEC> *>(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) out[i] = op_load<T>(x.v[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void op_store_vec(T *p, const float (&in)[VEC]) {
  OpVec<T, VEC> x;
#pragma unroll
  for (int i = 0; i < VEC; ++i) x.v[i] = op_store<T>(in[i]);
  *reinterpret_cast<OpVec<T, VEC> *>(p) = x;
}

// The same, as a load that stays where it is written: a run of them is in flight
// together, instead of each being moved down to its use.
template <typename T, int VEC>
__device__ __forceinline__ void op_load_ahead(const T *p, OpVec<T, VEC> &out) {
  if constexpr (sizeof(T) * VEC == 16) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    out = reinterpret_cast<const OpVec<T, VEC> &>(v);
  } else if constexpr (sizeof(T) * VEC == 4) {
    uint32_t v;
    asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    out = reinterpret_cast<const OpVec<T, VEC> &>(v);
  } else {
    static_assert(sizeof(T) * VEC == 2, "2, 4 or 16 bytes");
    uint16_t v;
    asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p) : "memory");
    out = reinterpret_cast<const OpVec<T, VEC> &>(v);
  }
}

// Whether rows of this base and stride can be moved 16 bytes at a time.
inline bool op_vec16(const void *p, int64_t ld, size_t elem) {
  return op_aligned(p, 16) && ((size_t)ld * elem) % 16 == 0;
}

}  // namespace aideen
