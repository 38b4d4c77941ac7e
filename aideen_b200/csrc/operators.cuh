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

// ---- rows that do not start on 16 bytes ------------------------------------------
// Such a row is still moved 16 bytes at a time: lane by lane the same columns as in an
// aligned row, each lane's 16 bytes cut out of the two aligned blocks that they lie in.

// Bytes [shift, shift + 16) of the 32 in a, b; shift is even and below 16.
__device__ __forceinline__ uint4 op_cut(const uint4 &a, const uint4 &b, uint32_t shift) {
  uint32_t w0 = a.x, w1 = a.y, w2 = a.z, w3 = a.w, w4 = b.x, w5 = b.y;
  if (shift & 8) {
    w0 = a.z; w1 = a.w; w2 = b.x; w3 = b.y; w4 = b.z; w5 = b.w;
  }
  if (shift & 4) {
    w0 = w1; w1 = w2; w2 = w3; w3 = w4; w4 = w5;
  }
  const uint32_t bits = (shift & 3) * 8;
  return make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits), __funnelshift_r(w2, w3, bits),
                    __funnelshift_r(w3, w4, bits));
}
// Where a tensor lies: blocks that reach out of it are not read whole.
struct OpExtent {
  const unsigned char *lo, *hi;
  __device__ __forceinline__ OpExtent(const void *p, long rows, long ld, long dim, int elem)
      : lo(static_cast<const unsigned char *>(p)), hi(lo + ((rows - 1) * ld + dim) * elem) {}
};
// 16 bytes from p on in two steps, so that the loads of several can be in flight
// together; elements from `valid` on become 0 (the tensor has them only below that).
template <typename T>
struct OpAny {
  static constexpr int V = 16 / sizeof(T);
  uint4 a, b;
  __device__ __forceinline__ void load(const T *p, int valid, const OpExtent &e) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p), blk = at & ~(uintptr_t)15;
    const uint32_t shift = (uint32_t)(at & 15);
    a = b = make_uint4(0, 0, 0, 0);
    if (blk >= reinterpret_cast<uintptr_t>(e.lo) && blk + (shift ? 32 : 16) <= reinterpret_cast<uintptr_t>(e.hi)) {
      asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w) : "l"(blk) : "memory");
      if (shift)
        asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "l"(blk + 16) : "memory");
    } else {  // at the tensor's ends: one by one, put where take() finds them
      OpVec<T, V> one[2] = {};
      const int first = (int)(shift / sizeof(T));
#pragma unroll
      for (int i = 0; i < 2 * V; ++i)
        if (i >= first && i - first < valid && i - first < V) one[i / V].v[i % V] = p[i - first];
      a = reinterpret_cast<const uint4 &>(one[0]);
      b = reinterpret_cast<const uint4 &>(one[1]);
    }
  }
  __device__ __forceinline__ OpVec<T, V> take(const T *p, int valid) const {
    const uint4 w = op_cut(a, b, (uint32_t)(reinterpret_cast<uintptr_t>(p) & 15));
    OpVec<T, V> v = reinterpret_cast<const OpVec<T, V> &>(w);
    if (valid < V) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i >= valid) v.v[i] = op_store<T>(0.f);
    }
    return v;
  }
};
// Stores N accesses of a warp that lie next to each other: p is the place of the lane's
// first column, lane 0 of access j follows lane 31 of access j - 1, and the first
// `valid` elements from p on belong to the row.  A lane stores the aligned block that its
// first element lies in, with the last elements of the one before; where a neighbour
// is missing (the warp's ends, the row's end), one by one.  All lanes call it.
template <typename T, int N>
__device__ __forceinline__ void op_store_any(T *p, const OpVec<T, 16 / sizeof(T)> (&v)[N], int valid) {
  constexpr int V = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  const uint32_t shift = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 15);
  const int head = V - (int)(shift / sizeof(T));  // elements in the first block
  uint4 last = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < N; ++j, p += 32 * V, valid -= 32 * V) {
    const uint4 w = reinterpret_cast<const uint4 &>(v[j]);
    const uint4 give = lane == 31 ? last : w;
    const int from = (lane + 31) & 31;
    const uint4 before = make_uint4(__shfl_sync(0xffffffffu, give.x, from), __shfl_sync(0xffffffffu, give.y, from),
                                    __shfl_sync(0xffffffffu, give.z, from), __shfl_sync(0xffffffffu, give.w, from));
    last = w;
    const bool whole = valid >= head && (lane > 0 || j > 0 || shift == 0);
    const bool next = valid - V >= head && (lane < 31 || j + 1 < N);
    if (whole) *reinterpret_cast<uint4 *>(reinterpret_cast<uintptr_t>(p) - shift) = shift ? op_cut(before, w, 16 - shift) : w;
    if (!whole && valid > 0) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i < min(valid, head)) p[i] = v[j].v[i];
    }
    if (!next && valid > head) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i >= head && i < valid) p[i] = v[j].v[i];
    }
  }
}

// Whether rows of this base and stride can be moved 16 bytes at a time.
inline bool op_vec16(const void *p, int64_t ld, size_t elem) {
  return op_aligned(p, 16) && ((size_t)ld * elem) % 16 == 0;
}

}  // namespace aideen
