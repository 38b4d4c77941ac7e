// Layer normalisation and its gradient on caller-owned tensors.
//
//   y = (x - m) r w + b,  m = mean(x),  r = 1 / sqrt(mean((x - m)^2) + eps)
//   g = dy w,  xh = (x - m) r
//   dx = r (g - mean(g) - xh mean(g xh)),  dw = sum_rows dy xh,  db = sum_rows dy
//
// Bound: HBM (forward reads x and writes y, the gradient reads x and dy and
// writes dx).  A row stays in the registers of the warps that own it, 64 bytes per
// lane at most, so it is read once: the variance is the mean of the squared
// differences from the finished mean, not E[x^2] - m^2.  A row takes 1 to 16 warps (8 in the
// gradient, whose column sums need the registers); longer ones are walked in memory.
// 32768 x 1024 bf16 forward: 26 us, 5.1 TB/s (a device copy of the same bytes: 22-24 us).
// 32749 x 1000 f16 gradient with dw and db: 48 us, 4.1 TB/s, where an elementwise sum of
// the same bytes takes 30 us.  Neither issue (42%) nor DRAM (43%) is busy: a row's loads, its
// reduction and its stores follow each other, and the column sums take the registers that
// more rows in flight would need (one row at a time with three CTAs per SM: 55 us).  2048 x
// 512 f32 gradient: 7 us.
// Rows that do not start on 16 bytes cost 1.5 to 2.2 times as much, 3 to 4.4 times what their
// bytes need (32768 x 1001 bf16: 58 us and 104 us; element by element 78 and 190): the
// instructions that cut 16 bytes out of two blocks bound them.
// Rows longer than the registers hold are walked element by element, one CTA per row: 1000 x
// 20000 f32 from a cold cache 92 us and 137 us (bytes: 24 and 37 us).
#include <type_traits>

#include "common.cuh"
#include "operators.cuh"

namespace aideen {
namespace {

// Most warps that share a row in registers; longer rows are walked in memory.
constexpr int kLnMaxWarps = 16, kLnMaxGradWarps = 8;

// The gradient's CTAs by the accesses per lane of a row (the rows at work and the
// column sums stay in registers).
template <int NV>
struct LnShape {
  static constexpr int threads = NV == 1 ? 512 : 256;
  static constexpr int per_sm = NV == 4 ? 1 : 2;
  static constexpr int rows = NV == 4 ? 1 : 2;  // that a group of warps works on at a time
};

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

// One access of a lane: 16 bytes, worked on as pairs (two float32 lanes per instruction).
template <typename T>
struct LnAccess {
  static constexpr int V = 16 / sizeof(T), P = V / 2;
  OpVec<T, V> v;
  __device__ __forceinline__ void load(const T *p) { v = *reinterpret_cast<const OpVec<T, V> *>(p); }
  __device__ __forceinline__ void load_ahead(const T *p) { op_load_ahead<T, V>(p, v); }
  // From a vector of `dim` elements; ANY: wherever it starts, and 0 behind its end.
  template <bool ANY>
  __device__ __forceinline__ void load_of(const T *base, int c, int dim) {
    if (!ANY || (c + V <= dim && (reinterpret_cast<uintptr_t>(base) & 15) == 0)) {
      load(base + c);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v.v[i] = c + i < dim ? base[c + i] : op_store<T>(0.f);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < V; ++i) v.v[i] = op_store<T>(0.f);
  }
  __device__ __forceinline__ float2 get(int i) const {
    if constexpr (sizeof(T) == 4) {
      return make_float2(v.v[2 * i], v.v[2 * i + 1]);
    } else {
      const uint32_t u = reinterpret_cast<const uint32_t *>(&v)[i];
      if constexpr (std::is_same<T, __half>::value) return __half22float2(reinterpret_cast<const __half2 &>(u));
      else return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    }
  }
  __device__ __forceinline__ void set(int i, float2 f) {
    if constexpr (sizeof(T) == 4) {
      v.v[2 * i] = f.x;
      v.v[2 * i + 1] = f.y;
    } else if constexpr (std::is_same<T, __half>::value) {
      reinterpret_cast<__half2 *>(&v)[i] = __float22half2_rn(f);
    } else {
      reinterpret_cast<__nv_bfloat162 *>(&v)[i] = __float22bfloat162_rn(f);
    }
  }
  __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<OpVec<T, V> *>(p) = v; }
};
__device__ __forceinline__ float2 pair(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }

// The part of a row that a lane holds: N accesses, `step` elements apart (zeros behind
// the row).  ANY: rows that start anywhere.
template <typename T, int N, bool ANY>
struct LnRow {
  LnAccess<T> v[N];
  // No branches, or each load would wait for the one before: behind the row its start
  // is read, and cleared.
  __device__ __forceinline__ void load(const T *row, int c0, int step, int dim, const OpExtent &e, bool there = true) {
    if constexpr (ANY) {
      OpAny<T> x[N];
#pragma unroll
      for (int j = 0; j < N; ++j) x[j].load(row + c0 + j * step, dim - (c0 + j * step), e);
#pragma unroll
      for (int j = 0; j < N; ++j) v[j].v = x[j].take(row + c0 + j * step, there ? dim - (c0 + j * step) : 0);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j].load_ahead(row + (c0 + j * step < dim ? c0 + j * step : 0));
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (c0 + j * step >= dim || !there) v[j].clear();
    }
  }
};

// R rows per group of wpr warps: short rows come several at a time, so that a warp has
// as many loads in flight as with a long one.
template <typename T, int N, int R, bool AFFINE, bool ANY>
__global__ void __launch_bounds__(512, ANY ? 1 : 2) layer_norm_kernel(const LnArgs a) {
  constexpr int V = LnAccess<T>::V, P = LnAccess<T>::P;
  __shared__ float red[2 * R * 16];
  op_begin();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = warp / a.wpr, groups = (int)(blockDim.x >> 5) / a.wpr;
  // rows that start anywhere: a warp's columns lie next to each other, for its stores
  const int c0 = ((warp % a.wpr) * (ANY ? N : 1) * 32 + lane) * V, step = 32 * (ANY ? 1 : a.wpr) * V;
  const long row0 = ((long)blockIdx.x * groups + group) * R;
  if (row0 >= a.rows) return;  // whole groups leave together
  const float inv = 1.f / (float)a.dim;
  float2 d[R][N][P];
  float s[R], m[R], r[R];
  {
    LnRow<T, N, ANY> v[R];
    const OpExtent ex(a.x, a.rows, a.x_ld, a.dim, sizeof(T));
#pragma unroll
    for (int q = 0; q < R; ++q)  // behind the last row, the last again, not stored
      v[q].load(static_cast<const T *>(a.x) + min(row0 + q, a.rows - 1) * a.x_ld, c0, step, a.dim, ex);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      float2 t = pair(0.f);
#pragma unroll
      for (int j = 0; j < N; ++j)
#pragma unroll
        for (int i = 0; i < P; ++i) t = add2(t, d[q][j][i] = v[q].v[j].get(i));
      s[q] = t.x + t.y;
    }
  }
  int parity = 0;
  row_sum<R>(s, a.wpr, group, red, parity);
#pragma unroll
  for (int q = 0; q < R; ++q) {
    m[q] = s[q] * inv;
    float2 t = pair(0.f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int valid = a.dim - (c0 + j * step);
      if (valid > 0) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          d[q][j][i] = add2(d[q][j][i], pair(-m[q]));
          if (ANY && valid < V) {  // behind the row
            if (2 * i + 1 >= valid) d[q][j][i].y = 0.f;
            if (2 * i >= valid) d[q][j][i].x = 0.f;
          }
          t = fma2(d[q][j][i], d[q][j][i], t);
        }
      }
    }
    s[q] = t.x + t.y;
  }
  row_sum<R>(s, a.wpr, group, red, parity);
#pragma unroll
  for (int q = 0; q < R; ++q) {
    r[q] = 1.f / sqrtf(s[q] * inv + a.eps);
    if (c0 == 0 && row0 + q < a.rows) {
      if (a.mean) a.mean[row0 + q] = m[q];
      if (a.rstd) a.rstd[row0 + q] = r[q];
    }
  }
  const T *w = static_cast<const T *>(a.w), *b = static_cast<const T *>(a.b);
  T *y = static_cast<T *>(a.y) + row0 * a.y_ld;
  OpVec<T, V> out[R][N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = c0 + j * step;
    if (c >= a.dim) continue;
    LnAccess<T> k, z, o;
    if (AFFINE || a.w) k.template load_of<ANY>(w, c, a.dim);
    if (AFFINE || a.b) z.template load_of<ANY>(b, c, a.dim);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      if (row0 + q >= a.rows) break;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        float2 f = mul2(d[q][j][i], pair(r[q]));
        if constexpr (AFFINE) {
          f = fma2(f, k.get(i), z.get(i));
        } else {
          if (a.w) f = mul2(f, k.get(i));
          if (a.b) f = add2(f, z.get(i));
        }
        o.set(i, f);
      }
      if constexpr (ANY) out[q][j] = o.v;
      else o.store(y + q * a.y_ld + c);
    }
  }
  if constexpr (ANY) {
#pragma unroll
    for (int q = 0; q < R; ++q)
      if (row0 + q < a.rows) op_store_any<T, N>(y + q * a.y_ld + c0, out[q], a.dim - c0);
  }
}

// Rows longer than the registers hold: one CTA per row walks it three times.
template <typename T>
__global__ void layer_norm_long_kernel(const LnArgs a) {
  __shared__ float red[2 * 8 * 32];
  op_begin();
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

// Gradient: each group of warps takes every so many rows and
// keeps its columns' sums of dy xh and dy in registers; the CTA's groups are
// added through shared memory in group order into one row of `part`.
template <typename T, int N, bool WEIGHT, bool ANY>
__global__ void __launch_bounds__(LnShape<N>::threads, LnShape<N>::per_sm) layer_norm_grad_kernel(const LnArgs a) {
  constexpr int V = LnAccess<T>::V, P = LnAccess<T>::P, R = ANY ? 1 : LnShape<N>::rows;
  extern __shared__ __align__(16) float sh[];  // [groups][2][dim] when several share a CTA: 32 KB at most
  __shared__ float red[2 * 2 * R * 16];
  op_begin();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = warp / a.wpr, groups = (int)(blockDim.x >> 5) / a.wpr;
  const int c0 = ((warp % a.wpr) * (ANY ? N : 1) * 32 + lane) * V, step = 32 * (ANY ? 1 : a.wpr) * V;
  const T *x = static_cast<const T *>(a.x), *dy = static_cast<const T *>(a.dy), *w = static_cast<const T *>(a.w);
  const OpExtent ex(x, a.rows, a.x_ld, a.dim, sizeof(T)), edy(dy, a.rows, a.y_ld, a.dim, sizeof(T));
  float2 aw[N][P], ab[N][P];
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < P; ++i) aw[j][i] = ab[j][i] = pair(0.f);
  int parity = 0;
  const float inv = 1.f / (float)a.dim;
  // R rows at a time: their loads are in flight together and share one reduction
  for (long row0 = ((long)blockIdx.x * groups + group) * R; row0 < a.rows; row0 += (long)gridDim.x * groups * R) {
    LnRow<T, N, ANY> xv[R], gv[R];
    float m[R], r[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const bool there = row0 + q < a.rows;  // rows behind the last are zeros and add nothing
      const long row = there ? row0 + q : a.rows - 1;
      xv[q].load(x + row * a.x_ld, c0, step, a.dim, ex, there);
      gv[q].load(dy + row * a.y_ld, c0, step, a.dim, edy, there);
      m[q] = a.mean[row];
      r[q] = a.rstd[row];
    }
    // dy is 0 behind a row, so nothing is added there
    float2 s0[R], s1[R];
#pragma unroll
    for (int q = 0; q < R; ++q) s0[q] = s1[q] = pair(0.f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (c0 + j * step >= a.dim) continue;
      LnAccess<T> k;
      if (WEIGHT) k.template load_of<ANY>(w, c0 + j * step, a.dim);
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 wk = WEIGHT ? k.get(i) : pair(1.f);
#pragma unroll
        for (int q = 0; q < R; ++q) {
          const float2 xh = mul2(add2(xv[q].v[j].get(i), pair(-m[q])), pair(r[q])), d = gv[q].v[j].get(i);
          aw[j][i] = fma2(d, xh, aw[j][i]);
          ab[j][i] = add2(ab[j][i], d);
          const float2 g = WEIGHT ? mul2(d, wk) : d;
          s0[q] = add2(s0[q], g);
          s1[q] = fma2(g, xh, s1[q]);
        }
      }
    }
    if (!a.dx) continue;
    float s[2 * R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      s[2 * q] = s0[q].x + s0[q].y;
      s[2 * q + 1] = s1[q].x + s1[q].y;
    }
    row_sum<2 * R>(s, a.wpr, group, red, parity);
    OpVec<T, V> out[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = c0 + j * step;
      if (c >= a.dim) continue;
      LnAccess<T> k;
      if (WEIGHT) k.template load_of<ANY>(w, c, a.dim);
#pragma unroll
      for (int q = 0; q < R; ++q) {
        if (row0 + q >= a.rows) break;
        const float2 c1 = pair(-s[2 * q] * inv), c2 = pair(-s[2 * q + 1] * inv);
        LnAccess<T> o;
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const float2 xh = mul2(add2(xv[q].v[j].get(i), pair(-m[q])), pair(r[q]));
          const float2 g = WEIGHT ? fma2(gv[q].v[j].get(i), k.get(i), c1) : add2(gv[q].v[j].get(i), c1);
          o.set(i, mul2(fma2(xh, c2, g), pair(r[q])));
        }
        if constexpr (ANY) out[j] = o.v;
        else o.store(static_cast<T *>(a.dx) + (row0 + q) * a.dx_ld + c);
      }
    }
    if constexpr (ANY) op_store_any<T, N>(static_cast<T *>(a.dx) + row0 * a.dx_ld + c0, out, a.dim - c0);
  }
  if (!a.part) return;
  // every group's sums side by side in shared memory, then added in group order
  float *out = a.part + (size_t)blockIdx.x * 2 * a.dim, *mine = groups > 1 ? sh + (size_t)group * 2 * a.dim : out;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = c0 + j * step;
    if (c >= a.dim) continue;
    if constexpr (ANY) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (c + i >= a.dim) break;
        mine[c + i] = i & 1 ? aw[j][i / 2].y : aw[j][i / 2].x;
        mine[a.dim + c + i] = i & 1 ? ab[j][i / 2].y : ab[j][i / 2].x;
      }
    } else {
#pragma unroll
      for (int i = 0; i < P; i += 2) {
        *reinterpret_cast<float4 *>(mine + c + 2 * i) = make_float4(aw[j][i].x, aw[j][i].y, aw[j][i + 1].x, aw[j][i + 1].y);
        *reinterpret_cast<float4 *>(mine + a.dim + c + 2 * i) = make_float4(ab[j][i].x, ab[j][i].y, ab[j][i + 1].x, ab[j][i + 1].y);
      }
    }
  }
  if (groups == 1) return;
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * a.dim; c += blockDim.x) {
    float t = sh[c];
    for (int k = 1; k < groups; ++k) t += sh[(size_t)k * 2 * a.dim + c];
    out[c] = t;
  }
}

// Long rows: dx by one CTA per row, then the column sums of a slice of rows.
template <typename T>
__global__ void layer_norm_grad_long_kernel(const LnArgs a) {
  __shared__ float red[2 * 8 * 32];
  op_begin();
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
  op_begin();
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
// 32 strided partial sums per CTA (blockIdx.y: 0 = dweight, 1 = dbias).
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_finish_kernel(const float *part, int n, int dim, T *dw, T *db) {
  __shared__ float sh[32][33];
  op_begin();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  T *out = blockIdx.y ? db : dw;
  if (!out) return;
  float s = 0.f;
  if (c < dim) {
#pragma unroll 8
    for (int i = ty; i < n; i += 32) s += part[((size_t)i * 2 + blockIdx.y) * dim + c];
  }
  sh[ty][tx] = s;
  __syncthreads();
  const float t = warp_sum(sh[tx][ty]);  // warp ty: column ty's 32 partial sums
  if (tx == 0 && blockIdx.x * 32 + ty < dim) out[blockIdx.x * 32 + ty] = op_store<T>(t);
}

// How a row is spread.  Forward: as few accesses per lane (1, 2 or 4) as hold it in one
// warp, then as many warps as it takes (a barrier costs more than it gives: 32768 x 1024
// bf16 26 us with one warp, 38 us with two).  Gradient: up to 2 warps before a lane takes
// two, 8 before it takes four, so that the column sums leave room for many rows in
// flight (16384 x 1024 f32 41 us with two accesses and four warps, 53 us the other way).
struct Spread {
  int nv, wpr, threads, groups, per_sm, rows;
};
Spread spread(int dim, int elem, bool grad) {
  Spread s{};
  const int one = 16 / elem;  // elements of an access
  s.nv = 1;
  if (grad) {
    if (32 * 2 * one < dim) s.nv = 32 * 2 * one * kLnMaxGradWarps < dim ? 4 : 2;
  } else {
    while (s.nv < 4 && 32 * one * s.nv < dim) s.nv *= 2;
  }
  s.wpr = 1;
  while (32 * one * s.nv * s.wpr < dim) s.wpr *= 2;
  s.threads = grad && s.nv == 1 ? LnShape<1>::threads : 256;
  if (s.threads < 32 * s.wpr) s.threads = 32 * s.wpr;
  s.groups = s.threads / 32 / s.wpr;
  s.rows = s.nv == 4 ? LnShape<4>::rows : s.nv == 2 ? LnShape<2>::rows : LnShape<1>::rows;
  s.per_sm = s.nv == 4 ? LnShape<4>::per_sm : s.nv == 2 ? LnShape<2>::per_sm : LnShape<1>::per_sm;
  return s;
}

// CTAs of the gradient, each leaving one partial row of sums.
int grad_ctas(const aideen_layer_norm_args *a, const Spread &s) {
  if (s.wpr > kLnMaxGradWarps) return a->rows < 64 ? (int)a->rows : 64;
  const long need = ((long)a->rows + s.groups - 1) / s.groups;  // one row per group while there are few
  const long most = (long)s.per_sm * op_sm_count();
  return (int)(need < most ? need : most);
}

template <typename T, int N, bool ANY>
cudaError_t forward_run(const LnArgs &a, const Spread &s, cudaStream_t st) {
  auto run = [&](auto one, auto affine, int rows) {
    const long per = (long)s.groups * rows;
    return op_launch(a.w && a.b ? affine : one, (unsigned)((a.rows + per - 1) / per), s.threads, 0, st, a);
  };
  // several rows per warp once that leaves every SM some warps of them
  constexpr int R = 4 / N;
  if (R > 1 && s.wpr == 1 && a.rows >= (long)op_sm_count() * 16 * R)
    return run(layer_norm_kernel<T, N, R, false, ANY>, layer_norm_kernel<T, N, R, true, ANY>, R);
  return run(layer_norm_kernel<T, N, 1, false, ANY>, layer_norm_kernel<T, N, 1, true, ANY>, 1);
}
template <typename T, bool ANY>
cudaError_t forward_any(const LnArgs &a, const Spread &s, cudaStream_t st) {
  return s.nv == 1 ? forward_run<T, 1, ANY>(a, s, st) : s.nv == 2 ? forward_run<T, 2, ANY>(a, s, st) : forward_run<T, 4, ANY>(a, s, st);
}
template <typename T>
cudaError_t forward_typed(const LnArgs &a, const Spread &s, bool vec, cudaStream_t st) {
  if (s.wpr > kLnMaxWarps) return op_launch(layer_norm_long_kernel<T>, (unsigned)a.rows, 1024, 0, st, a);
  return vec ? forward_any<T, false>(a, s, st) : forward_any<T, true>(a, s, st);
}

template <typename T, int N, bool ANY>
cudaError_t grad_run(const LnArgs &a, const Spread &s, int ctas, cudaStream_t st) {
  const size_t smem = s.groups > 1 && a.part ? (size_t)s.groups * 2 * a.dim * sizeof(float) : 0;
  return op_launch(a.w ? layer_norm_grad_kernel<T, N, true, ANY> : layer_norm_grad_kernel<T, N, false, ANY>, ctas, s.threads, smem, st, a);
}
template <typename T, bool ANY>
cudaError_t grad_any(const LnArgs &a, const Spread &s, int ctas, cudaStream_t st) {
  return s.nv == 1 ? grad_run<T, 1, ANY>(a, s, ctas, st) : s.nv == 2 ? grad_run<T, 2, ANY>(a, s, ctas, st) : grad_run<T, 4, ANY>(a, s, ctas, st);
}
template <typename T>
cudaError_t grad_typed(const LnArgs &a, const Spread &s, bool vec, int ctas, T *dw, T *db, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  if (s.wpr > kLnMaxGradWarps) {
    if (a.dx) e = op_launch(layer_norm_grad_long_kernel<T>, (unsigned)a.rows, 1024, 0, st, a);
    if (e == cudaSuccess && a.part)
      e = op_launch(layer_norm_columns_kernel<T>, dim3((a.dim + 255) / 256, ctas), 256, 0, st, a);
  } else {
    e = vec ? grad_any<T, false>(a, s, ctas, st) : grad_any<T, true>(a, s, ctas, st);
  }
  if (e != cudaSuccess || !a.part) return e;
  return op_launch(layer_norm_finish_kernel<T>, dim3((a.dim + 31) / 32, 2), 1024, 0, st, a.part, ctas, a.dim, dw, db);
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
  const bool vec = ((size_t)a.dim * el) % 16 == 0 && op_vec16(x, a.x_ld, el) && op_vec16(y, a.y_ld, el) &&
                   op_aligned(weight, 16) && op_aligned(bias, 16);
  const Spread s = spread(a.dim, (int)el, false);
  a.wpr = s.wpr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->dtype == AIDEEN_F32) return op_cuda(forward_typed<float>(a, s, vec, st));
  if (args->dtype == AIDEEN_BF16) return op_cuda(forward_typed<__nv_bfloat16>(a, s, vec, st));
  return op_cuda(forward_typed<__half>(a, s, vec, st));
}

extern "C" int aideen_layer_norm_grad_workspace(const aideen_layer_norm_args *args, size_t *bytes) {
  const int rc = check_args(args);
  if (rc != AIDEEN_OK) return rc;
  OP_CHECK(bytes, "layer_norm: null bytes");
  const Spread s = spread((int)args->dim, (int)op_elem(args->dtype), true);
  *bytes = op_round((size_t)grad_ctas(args, s) * 2 * args->dim * sizeof(float), 256);
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
  const bool vec = ((size_t)a.dim * el) % 16 == 0 && op_vec16(x, a.x_ld, el) && op_vec16(dy, a.y_ld, el) &&
                   (!dx || op_vec16(dx, a.dx_ld, el)) && op_aligned(weight, 16);
  const Spread s = spread(a.dim, (int)el, true);
  a.wpr = s.wpr;
  const int ctas = grad_ctas(args, s);
  if (args->dtype == AIDEEN_F32)
    return op_cuda(grad_typed<float>(a, s, vec, ctas, static_cast<float *>(dweight), static_cast<float *>(dbias), st));
  if (args->dtype == AIDEEN_BF16)
    return op_cuda(grad_typed<__nv_bfloat16>(a, s, vec, ctas, static_cast<__nv_bfloat16 *>(dweight),
                                             static_cast<__nv_bfloat16 *>(dbias), st));
  return op_cuda(grad_typed<__half>(a, s, vec, ctas, static_cast<__half *>(dweight), static_cast<__half *>(dbias), st));
}
