// Layer normalisation and its gradient on caller-owned tensors.
//
//   y = (x - m) r w + b,  m = mean(x),  r = 1 / sqrt(mean((x - m)^2) + eps)
//   g = dy w,  xh = (x - m) r
//   dx = r (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// Bound: HBM (forward reads x and writes y, the gradient reads x and dy and
// writes dx).  A row stays in the registers of the warps that own it, at most
// 16 elements per lane, so it is read once: the variance is the mean of the
// squared differences from the finished mean, not E[x^2] - m^2.  Rows of up to
// 8192 elements take 1 to 16 warps; longer ones are walked in memory.
#include "common.cuh"
#include "operators.cuh"

namespace aideen {
namespace {

constexpr int kLnThreads = 256;       // threads of a CTA (512 when a row needs 16 warps)
constexpr int kLnLane = 16;           // most elements of a row per lane
constexpr int kLnMaxWarps = 16;       // most warps per row
constexpr int kLnMaxDim = kLnLane * 32 * kLnMaxWarps;

struct LnArgs {
  const void *x, *dy, *w, *b;
  void *y, *dx;
  float *mean, *rstd;
  float *part;  // gradient: [CTAs][2][dim] sums of dy xh and dy
  long rows, x_ld, y_ld, dx_ld;
  int dim, wpr;  // wpr: warps per row
  float eps;
};

// Sum of K values over the wpr warps that share a row.  Each group of warps
// has its own slots of `red` and its own named barrier; `parity` alternates the
// slots, so a second sum needs no barrier before it writes.
template <int K>
__device__ __forceinline__ void row_sum(float (&v)[K], int wpr, int group, float *red, int &parity) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  if (wpr == 1) return;
  const int warp = threadIdx.x >> 5;
  float *slot = red + parity * (K * 16);
  parity ^= 1;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) slot[warp * K + k] = v[k];
  }
  asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * wpr) : "memory");
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = 0.f;
  for (int i = 0; i < wpr; ++i) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += slot[(group * wpr + i) * K + k];
  }
}

// One row per group of wpr warps.  NV accesses of VEC elements per lane.
template <typename T, int VEC, int NV>
__global__ void layer_norm_kernel(const LnArgs a) {
  __shared__ float red[2 * 16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = warp / a.wpr, groups = (int)(blockDim.x >> 5) / a.wpr;
  const int at = (warp % a.wpr) * 32 + lane, step = 32 * a.wpr * VEC;
  const long row = (long)blockIdx.x * groups + group;
  if (group >= groups || row >= a.rows) return;  // whole groups leave together
  const T *x = static_cast<const T *>(a.x) + row * a.x_ld;
  float v[NV][VEC];
  float s[1] = {0.f};
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = at * VEC + j * step;
    if (c < a.dim) {
      op_load_vec<T, VEC>(x + c, v[j]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) s[0] += v[j][i];
  }
  int parity = 0;
  row_sum<1>(s, a.wpr, group, red, parity);
  const float m = s[0] / (float)a.dim;
  s[0] = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (at * VEC + j * step < a.dim) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float c = v[j][i] - m;
        s[0] += c * c;
      }
    }
  }
  row_sum<1>(s, a.wpr, group, red, parity);
  const float r = 1.f / sqrtf(s[0] / (float)a.dim + a.eps);
  if (at == 0) {
    if (a.mean) a.mean[row] = m;
    if (a.rstd) a.rstd[row] = r;
  }
  T *y = static_cast<T *>(a.y) + row * a.y_ld;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = at * VEC + j * step;
    if (c >= a.dim) continue;
    float w[VEC], b[VEC];
    if (a.w) op_load_vec<T, VEC>(static_cast<const T *>(a.w) + c, w);
    if (a.b) op_load_vec<T, VEC>(static_cast<const T *>(a.b) + c, b);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float o = (v[j][i] - m) * r;
      if (a.w) o *= w[i];
      if (a.b) o += b[i];
      v[j][i] = o;
    }
    op_store_vec<T, VEC>(y + c, v[j]);
  }
}

// Rows longer than the registers hold: one CTA per row walks it three times.
template <typename T>
__global__ void layer_norm_long_kernel(const LnArgs a) {
  __shared__ float red[2 * 8 * 32];
  BlockReducer br(red);
  const long row = blockIdx.x;
  const T *x = static_cast<const T *>(a.x) + row * a.x_ld;
  float s[1] = {0.f};
  for (int c = threadIdx.x; c < a.dim; c += blockDim.x) s[0] += op_load<T>(x[c]);
  br.sum<1>(s);
  const float m = s[0] / (float)a.dim;
  s[0] = 0.f;
  for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
    const float d = op_load<T>(x[c]) - m;
    s[0] += d * d;
  }
  br.sum<1>(s);
  const float r = 1.f / sqrtf(s[0] / (float)a.dim + a.eps);
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[row] = m;
    if (a.rstd) a.rstd[row] = r;
  }
  const T *w = static_cast<const T *>(a.w), *b = static_cast<const T *>(a.b);
  T *y = static_cast<T *>(a.y) + row * a.y_ld;
  for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
    float o = (op_load<T>(x[c]) - m) * r;
    if (w) o *= op_load<T>(w[c]);
    if (b) o += op_load<T>(b[c]);
    y[c] = op_store<T>(o);
  }
}

// Gradient: each group of warps takes rows group, group + all groups, ... and
// keeps its columns' sums of dy xh and dy in registers; the CTA's groups are
// added through shared memory in group order into one row of `part`.
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(512) layer_norm_grad_kernel(const LnArgs a) {
  extern __shared__ float sh[];  // [2][dim] when several groups share a CTA
  __shared__ float red[2 * 2 * 16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = warp / a.wpr, groups = (int)(blockDim.x >> 5) / a.wpr;
  const int at = (warp % a.wpr) * 32 + lane, step = 32 * a.wpr * VEC;
  float aw[NV][VEC], ab[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VEC; ++i) aw[j][i] = ab[j][i] = 0.f;
  int parity = 0;
  const float inv = 1.f / (float)a.dim;
  for (long row = (long)blockIdx.x * groups + group; row < a.rows; row += (long)gridDim.x * groups) {
    const T *x = static_cast<const T *>(a.x) + row * a.x_ld;
    const T *dy = static_cast<const T *>(a.dy) + row * a.y_ld;
    const float m = a.mean[row], r = a.rstd[row];
    float xh[NV][VEC], g[NV][VEC];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = at * VEC + j * step;
      if (c < a.dim) {
        op_load_vec<T, VEC>(x + c, xh[j]);
        op_load_vec<T, VEC>(dy + c, g[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = at * VEC + j * step;
      if (c < a.dim) {
        float w[VEC];
        if (a.w) op_load_vec<T, VEC>(static_cast<const T *>(a.w) + c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          xh[j][i] = (xh[j][i] - m) * r;
          aw[j][i] += g[j][i] * xh[j][i];
          ab[j][i] += g[j][i];
          if (a.w) g[j][i] *= w[i];
          s[0] += g[j][i];
          s[1] += g[j][i] * xh[j][i];
        }
      }
    }
    if (!a.dx) continue;
    row_sum<2>(s, a.wpr, group, red, parity);
    const float c1 = s[0] * inv, c2 = s[1] * inv;
    T *dx = static_cast<T *>(a.dx) + row * a.dx_ld;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = at * VEC + j * step;
      if (c >= a.dim) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) g[j][i] = r * (g[j][i] - c1 - xh[j][i] * c2);
      op_store_vec<T, VEC>(dx + c, g[j]);
    }
  }
  if (!a.part) return;
  float *out = a.part + (size_t)blockIdx.x * 2 * a.dim;
  for (int k = 0; k < groups; ++k) {
    if (group == k) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = at * VEC + j * step;
        if (c >= a.dim) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float pw = aw[j][i], pb = ab[j][i];
          if (k > 0) {
            pw += sh[c + i];
            pb += sh[a.dim + c + i];
          }
          if (k + 1 < groups) {
            sh[c + i] = pw;
            sh[a.dim + c + i] = pb;
          } else {
            out[c + i] = pw;
            out[a.dim + c + i] = pb;
          }
        }
      }
    }
    if (k + 1 < groups) __syncthreads();
  }
}

// Long rows: dx by one CTA per row, then the column sums of a slice of rows.
template <typename T>
__global__ void layer_norm_grad_long_kernel(const LnArgs a) {
  __shared__ float red[2 * 8 * 32];
  BlockReducer br(red);
  const long row = blockIdx.x;
  const T *x = static_cast<const T *>(a.x) + row * a.x_ld;
  const T *dy = static_cast<const T *>(a.dy) + row * a.y_ld;
  const T *w = static_cast<const T *>(a.w);
  const float m = a.mean[row], r = a.rstd[row];
  float s[2] = {0.f, 0.f};
  for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
    const float g = op_load<T>(dy[c]) * (w ? op_load<T>(w[c]) : 1.f);
    s[0] += g;
    s[1] += g * ((op_load<T>(x[c]) - m) * r);
  }
  br.sum<2>(s);
  const float c1 = s[0] / (float)a.dim, c2 = s[1] / (float)a.dim;
  T *dx = static_cast<T *>(a.dx) + row * a.dx_ld;
  for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
    const float g = op_load<T>(dy[c]) * (w ? op_load<T>(w[c]) : 1.f);
    const float xh = (op_load<T>(x[c]) - m) * r;
    dx[c] = op_store<T>(r * (g - c1 - xh * c2));
  }
}
template <typename T>
__global__ void layer_norm_columns_kernel(const LnArgs a) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= a.dim) return;
  const T *x = static_cast<const T *>(a.x), *dy = static_cast<const T *>(a.dy);
  float sw = 0.f, sb = 0.f;
  for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float g = op_load<T>(dy[row * a.y_ld + c]);
    sw += g * ((op_load<T>(x[row * a.x_ld + c]) - a.mean[row]) * a.rstd[row]);
    sb += g;
  }
  a.part[((size_t)blockIdx.y * 2) * a.dim + c] = sw;
  a.part[((size_t)blockIdx.y * 2 + 1) * a.dim + c] = sb;
}

// dweight and dbias: the rows of `part` added in a fixed order, 32 columns and
// 8 strided partial sums per CTA (blockIdx.y: 0 = dweight, 1 = dbias).
template <typename T>
__global__ void layer_norm_finish_kernel(const float *part, int n, int dim, T *dw, T *db) {
  __shared__ float sh[8][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  T *out = blockIdx.y ? db : dw;
  if (!out) return;
  float s = 0.f;
  if (c < dim) {
#pragma unroll 4
    for (int i = ty; i < n; i += 8) s += part[((size_t)i * 2 + blockIdx.y) * dim + c];
  }
  sh[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < dim) {
    float t = sh[0][tx];
#pragma unroll
    for (int k = 1; k < 8; ++k) t += sh[k][tx];
    out[c] = op_store<T>(t);
  }
}

// The fewest warps that hold a row at kLnLane elements per lane.
int warps_per_row(int dim) {
  int w = 1;
  while (w * 32 * kLnLane < dim) w *= 2;
  return w;
}

int grad_ctas(const aideen_layer_norm_args *a) {
  if (a->dim > (uint32_t)kLnMaxDim) return a->rows < 64 ? (int)a->rows : 64;
  const int wpr = warps_per_row((int)a->dim);
  const int groups = (wpr == 16 ? 16 : kLnThreads / 32) / wpr;
  const long need = ((long)a->rows + groups - 1) / groups;
  const long most = 2L * op_sm_count();
  return (int)(need < most ? need : most);
}

template <typename T, int VEC, int NV>
cudaError_t forward_run(const LnArgs &a, cudaStream_t st) {
  const int threads = a.wpr == 16 ? 512 : kLnThreads, groups = threads / 32 / a.wpr;
  layer_norm_kernel<T, VEC, NV><<<(unsigned)((a.rows + groups - 1) / groups), threads, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename T, int VEC, int NV>
cudaError_t grad_run(const LnArgs &a, int ctas, cudaStream_t st) {
  const int threads = a.wpr == 16 ? 512 : kLnThreads, groups = threads / 32 / a.wpr;
  const size_t smem = groups > 1 && a.part ? (size_t)2 * a.dim * sizeof(float) : 0;
  layer_norm_grad_kernel<T, VEC, NV><<<ctas, threads, smem, st>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t forward_typed(const LnArgs &a, bool vec, cudaStream_t st) {
  if (a.dim > kLnMaxDim) {
    layer_norm_long_kernel<T><<<(unsigned)a.rows, 1024, 0, st>>>(a);
    return cudaGetLastError();
  }
  constexpr int V = 16 / sizeof(T);
  // fewer accesses per lane where the row is short: no idle register tiles
  const int lane = (a.dim + 32 * a.wpr - 1) / (32 * a.wpr);
  if (!vec) return lane <= 4 ? forward_run<T, 1, 4>(a, st) : forward_run<T, 1, kLnLane>(a, st);
  if (lane <= V) return forward_run<T, V, 1>(a, st);
  return forward_run<T, V, kLnLane / V>(a, st);
}

template <typename T>
cudaError_t grad_typed(LnArgs a, bool vec, int ctas, T *dw, T *db, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  if (a.dim > kLnMaxDim) {
    if (a.dx) {
      layer_norm_grad_long_kernel<T><<<(unsigned)a.rows, 1024, 0, st>>>(a);
      e = cudaGetLastError();
    }
    if (e == cudaSuccess && a.part) {
      layer_norm_columns_kernel<T><<<dim3((a.dim + 255) / 256, ctas), 256, 0, st>>>(a);
      e = cudaGetLastError();
    }
  } else {
    constexpr int V = 16 / sizeof(T);
    const int lane = (a.dim + 32 * a.wpr - 1) / (32 * a.wpr);
    if (!vec) e = lane <= 4 ? grad_run<T, 1, 4>(a, ctas, st) : grad_run<T, 1, kLnLane>(a, ctas, st);
    else if (lane <= V) e = grad_run<T, V, 1>(a, ctas, st);
    else e = grad_run<T, V, kLnLane / V>(a, ctas, st);
  }
  if (e != cudaSuccess || !a.part) return e;
  layer_norm_finish_kernel<T><<<dim3((a.dim + 31) / 32, 2), 256, 0, st>>>(a.part, ctas, a.dim, dw, db);
  return cudaGetLastError();
}

int check_args(const aideen_layer_norm_args *a) {
  OP_CHECK(a, "layer_norm: null args");
  OP_CHECK(a->dtype <= AIDEEN_F16, "layer_norm: unknown dtype");
  OP_CHECK(a->dim >= 1 && a->dim <= (1u << 24), "layer_norm: dim must be in [1, 2^24]");
  OP_CHECK(a->rows <= (1u << 30), "layer_norm: more than 2^30 rows");
  OP_CHECK(a->eps >= 0.f, "layer_norm: eps must be >= 0");
  OP_CHECK(a->x_ld >= (int64_t)a->dim && a->y_ld >= (int64_t)a->dim, "layer_norm: row stride below dim");
  return AIDEEN_OK;
}

}  // namespace
}  // namespace aideen

using namespace aideen;

extern "C" int aideen_layer_norm(const aideen_layer_norm_args *args, const void *x, const void *weight,
                                 const void *bias, void *y, float *mean, float *rstd, void *stream) {
  const int rc = check_args(args);
  if (rc != AIDEEN_OK) return rc;
  if (args->rows == 0) return AIDEEN_OK;
  OP_CHECK(x && y, "layer_norm: null x or y");
  const size_t el = op_elem(args->dtype);
  OP_CHECK(op_aligned(x, el) && op_aligned(y, el) && op_aligned(weight, el) && op_aligned(bias, el) &&
               op_aligned(mean, 4) && op_aligned(rstd, 4),
           "layer_norm: a pointer is not aligned to its type");
  LnArgs a{};
  a.x = x; a.w = weight; a.b = bias; a.y = y; a.mean = mean; a.rstd = rstd;
  a.rows = args->rows; a.dim = (int)args->dim; a.eps = args->eps;
  a.x_ld = args->x_ld; a.y_ld = args->y_ld;
  a.wpr = warps_per_row(a.dim);
  const bool vec = ((size_t)a.dim * el) % 16 == 0 && op_vec16(x, a.x_ld, el) && op_vec16(y, a.y_ld, el) &&
                   op_aligned(weight, 16) && op_aligned(bias, 16);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->dtype == AIDEEN_F32) return op_cuda(forward_typed<float>(a, vec, st));
  if (args->dtype == AIDEEN_BF16) return op_cuda(forward_typed<__nv_bfloat16>(a, vec, st));
  return op_cuda(forward_typed<__half>(a, vec, st));
}

extern "C" int aideen_layer_norm_grad_workspace(const aideen_layer_norm_args *args, size_t *bytes) {
  const int rc = check_args(args);
  if (rc != AIDEEN_OK) return rc;
  OP_CHECK(bytes, "layer_norm: null bytes");
  *bytes = op_round((size_t)grad_ctas(args) * 2 * args->dim * sizeof(float), 256);
  return AIDEEN_OK;
}

extern "C" int aideen_layer_norm_grad(const aideen_layer_norm_args *args, const void *dy, const void *x,
                                      const void *weight, const float *mean, const float *rstd, void *dx,
                                      void *dweight, void *dbias, void *workspace, size_t workspace_bytes,
                                      void *stream) {
  size_t need = 0;
  const int rc = aideen_layer_norm_grad_workspace(args, &need);
  if (rc != AIDEEN_OK) return rc;
  OP_CHECK(!dx || args->dx_ld >= (int64_t)args->dim, "layer_norm_grad: row stride below dim");
  const size_t el = op_elem(args->dtype);
  OP_CHECK(op_aligned(x, el) && op_aligned(dy, el) && op_aligned(weight, el) && op_aligned(dx, el) &&
               op_aligned(dweight, el) && op_aligned(dbias, el) && op_aligned(mean, 4) && op_aligned(rstd, 4),
           "layer_norm_grad: a pointer is not aligned to its type");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->rows == 0) {  // sums over no rows
    cudaError_t e = cudaSuccess;
    if (dweight) e = cudaMemsetAsync(dweight, 0, args->dim * el, st);
    if (dbias && e == cudaSuccess) e = cudaMemsetAsync(dbias, 0, args->dim * el, st);
    return op_cuda(e);
  }
  OP_CHECK(dx || dweight || dbias, "layer_norm_grad: no output wanted");
  OP_CHECK(dy && x && mean && rstd, "layer_norm_grad: null dy, x, mean or rstd");
  const bool sums = dweight || dbias;
  OP_CHECK(!sums || (workspace && op_aligned(workspace, 256) && workspace_bytes >= need),
           "layer_norm_grad: workspace missing, misaligned or too small");
  LnArgs a{};
  a.x = x; a.dy = dy; a.w = weight; a.dx = dx;
  a.mean = const_cast<float *>(mean); a.rstd = const_cast<float *>(rstd);
  a.part = sums ? static_cast<float *>(workspace) : nullptr;
  a.rows = args->rows; a.dim = (int)args->dim; a.eps = args->eps;
  a.x_ld = args->x_ld; a.y_ld = args->y_ld; a.dx_ld = args->dx_ld;
  a.wpr = warps_per_row(a.dim);
  const bool vec = ((size_t)a.dim * el) % 16 == 0 && op_vec16(x, a.x_ld, el) && op_vec16(dy, a.y_ld, el) &&
                   (!dx || op_vec16(dx, a.dx_ld, el)) && op_aligned(weight, 16);
  const int ctas = grad_ctas(args);
  if (args->dtype == AIDEEN_F32)
    return op_cuda(grad_typed<float>(a, vec, ctas, static_cast<float *>(dweight), static_cast<float *>(dbias), st));
  if (args->dtype == AIDEEN_BF16)
    return op_cuda(grad_typed<__nv_bfloat16>(a, vec, ctas, static_cast<__nv_bfloat16 *>(dweight),
                                             static_cast<__nv_bfloat16 *>(dbias), st));
  return op_cuda(grad_typed<__half>(a, vec, ctas, static_cast<__half *>(dweight), static_cast<__half *>(dbias), st));
}
