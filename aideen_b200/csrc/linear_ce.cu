// Softmax cross entropy of a linear head over the vocabulary, without keeping
// the logits, and its gradient, on caller-owned tensors.
//
//   z = x W^T + b,  lse[n] = log sum_v exp z[n][v],  loss[n] = lse[n] - z[n][t[n]]
//   G = softmax(z) - onehot(t)  (0 where the row is not counted)
//   dx = c G W,  dW = c G^T x,  db = c sum_n G,   c = dloss / counted rows
//
// CUDA-core form: 64 x 64 tiles of z through shared memory.  The loss keeps a
// running maximum and sum per row and vocabulary slice; the gradient forms G for
// a piece of the vocabulary at a time and multiplies it.
#include "common.cuh"
#include "operators.cuh"

namespace aideen {
namespace {

__device__ unsigned int g_ce_timeout;

constexpr int kTile = 64, kStep = 16;
constexpr int kPiece = 4096;  // vocabulary columns of G held at a time
constexpr int kSlices = 64;   // vocabulary slices of the loss

struct CeArgs {
  const void *x, *w, *b;
  const int32_t *tg;
  const float *lse;
  long x_ld, w_ld;
  int rows, dim, vocab;
};

__device__ __forceinline__ bool counted(int32_t t, int vocab) { return t >= 0 && t < vocab; }

// acc[i][j] = sum_k A(m0 + 4 ty + i, k) B(n0 + 4 tx + j, k); fa / fb give 0 outside.
template <typename FA, typename FB>
__device__ __forceinline__ void tile_product(FA fa, FB fb, int K, float (&acc)[4][4], float (*sa)[kTile + 1],
                                             float (*sb)[kTile + 1]) {
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  for (int k0 = 0; k0 < K; k0 += kStep) {
    for (int i = threadIdx.x; i < kTile * kStep; i += 256) {
      sa[i % kStep][i / kStep] = k0 + i % kStep < K ? fa(i / kStep, k0 + i % kStep) : 0.f;
      sb[i % kStep][i / kStep] = k0 + i % kStep < K ? fb(i / kStep, k0 + i % kStep) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][4 * ty + i], sb[k][4 * tx + j], acc[i][j]);
    __syncthreads();
  }
}

template <typename T>
__device__ __forceinline__ void logits_tile(const CeArgs &a, int m0, int n0, float (&acc)[4][4],
                                            float (*sa)[kTile + 1], float (*sb)[kTile + 1]) {
  const T *x = static_cast<const T *>(a.x), *w = static_cast<const T *>(a.w), *b = static_cast<const T *>(a.b);
  tile_product(
      [&](int m, int k) { return m0 + m < a.rows ? op_load<T>(x[(long)(m0 + m) * a.x_ld + k]) : 0.f; },
      [&](int n, int k) { return n0 + n < a.vocab ? op_load<T>(w[(long)(n0 + n) * a.w_ld + k]) : 0.f; }, a.dim, acc,
      sa, sb);
  const int tx = threadIdx.x & 15;
  if (b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float bv = n0 + 4 * tx + j < a.vocab ? op_load<T>(b[n0 + 4 * tx + j]) : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i][j] += bv;
    }
  }
}

__device__ __forceinline__ void merge(float &m, float &s, float m2, float s2) {
  const float mm = fmaxf(m, m2);
  if (mm == -INFINITY) { s += s2; return; }
  s = s * expf(m - mm) + s2 * expf(m2 - mm);
  m = mm;
}

template <typename T>
__global__ void __launch_bounds__(256) ce_stats_kernel(const CeArgs a, float2 *part, float *picked) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  __shared__ float2 st[kTile][16];
  const int m0 = blockIdx.x * kTile, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float m[4], s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) { m[i] = -INFINITY; s[i] = 0.f; }
  for (int n0 = blockIdx.y * kTile; n0 < a.vocab; n0 += kTile * gridDim.y) {
    float acc[4][4];
    logits_tile<T>(a, m0, n0, acc, sa, sb);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = m0 + 4 * ty + i;
      const int t = row < a.rows ? a.tg[row] : -1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = n0 + 4 * tx + j;
        if (col >= a.vocab) continue;
        merge(m[i], s[i], acc[i][j], isinf(acc[i][j]) && acc[i][j] < 0 ? 0.f : 1.f);
        if (col == t) picked[row] = acc[i][j];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) st[4 * ty + i][tx] = make_float2(m[i], s[i]);
  __syncthreads();
  if (threadIdx.x < kTile && m0 + threadIdx.x < a.rows) {
    float mm = -INFINITY, ss = 0.f;
    for (int k = 0; k < 16; ++k) merge(mm, ss, st[threadIdx.x][k].x, st[threadIdx.x][k].y);
    part[(size_t)blockIdx.y * a.rows + m0 + threadIdx.x] = make_float2(mm, ss);
  }
}

__global__ void ce_rows_kernel(const CeArgs a, const float2 *part, int slices, const float *picked, float *row_loss,
                               float *lse) {
  const int n = blockIdx.x * blockDim.x + threadIdx.x;
  if (n >= a.rows) return;
  float l = 0.f, z = 0.f;
  if (counted(a.tg[n], a.vocab)) {
    float m = -INFINITY, s = 0.f;
    for (int k = 0; k < slices; ++k) merge(m, s, part[(size_t)k * a.rows + n].x, part[(size_t)k * a.rows + n].y);
    l = m + logf(s);
    z = picked[n];
  }
  row_loss[n] = l - z;
  if (lse) lse[n] = l;
}

// loss = sum of the rows (fixed order), and the number of counted rows.
__global__ void __launch_bounds__(1024) ce_loss_kernel(const CeArgs a, const float *row_loss, int mean, float *loss,
                                                       float *count) {
  __shared__ float red[2 * 8 * 32];
  BlockReducer br(red);
  float v[2] = {0.f, 0.f};
  for (int n = threadIdx.x; n < a.rows; n += 1024) {
    if (row_loss) v[0] += row_loss[n];
    v[1] += counted(a.tg[n], a.vocab) ? 1.f : 0.f;
  }
  br.sum<2>(v);
  if (threadIdx.x == 0) {
    if (loss) *loss = mean ? v[0] / fmaxf(v[1], 1.f) : v[0];
    if (count) *count = v[1];
  }
}

template <typename T>
__global__ void __launch_bounds__(256) ce_piece_kernel(const CeArgs a, int v0, float *G) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  const int m0 = blockIdx.x * kTile, n0 = v0 + blockIdx.y * kTile, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4];
  logits_tile<T>(a, m0, n0, acc, sa, sb);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = m0 + 4 * ty + i;
    if (row >= a.rows) continue;
    const int t = a.tg[row];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = n0 + 4 * tx + j;
      float g = 0.f;
      if (counted(t, a.vocab) && col < a.vocab) g = expf(acc[i][j] - a.lse[row]) - (col == t ? 1.f : 0.f);
      if (col - v0 < kPiece) G[(size_t)row * kPiece + col - v0] = g;
    }
  }
}

// dx += G W over this piece.
template <typename T>
__global__ void __launch_bounds__(256) ce_dx_kernel(const CeArgs a, int v0, const float *G, float *dx, int first) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  const int m0 = blockIdx.x * kTile, n0 = blockIdx.y * kTile, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const T *w = static_cast<const T *>(a.w);
  const int K = min(kPiece, a.vocab - v0);
  float acc[4][4];
  tile_product([&](int m, int k) { return m0 + m < a.rows ? G[(size_t)(m0 + m) * kPiece + k] : 0.f; },
               [&](int n, int k) { return n0 + n < a.dim ? op_load<T>(w[(long)(v0 + k) * a.w_ld + n0 + n]) : 0.f; },
               K, acc, sa, sb);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = m0 + 4 * ty + i, col = n0 + 4 * tx + j;
      if (row >= a.rows || col >= a.dim) continue;
      float *p = dx + (size_t)row * a.dim + col;
      *p = first ? acc[i][j] : *p + acc[i][j];
    }
}

__device__ __forceinline__ float ce_scale(const float *dloss, const float *count, int mean) {
  return (dloss ? *dloss : 1.f) / (mean ? fmaxf(*count, 1.f) : 1.f);
}

template <typename T>
__global__ void ce_dx_store_kernel(const CeArgs a, const float *acc, const float *dloss, const float *count, int mean,
                                   T *dx, long ld) {
  const float c = ce_scale(dloss, count, mean);
  for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < (size_t)a.rows * a.dim;
       i += (size_t)gridDim.x * blockDim.x)
    dx[(long)(i / a.dim) * ld + i % a.dim] = counted(a.tg[i / a.dim], a.vocab) ? op_store<T>(c * acc[i]) : op_store<T>(0.f);
}

// dW and db of this piece.
template <typename T>
__global__ void __launch_bounds__(256) ce_dw_kernel(const CeArgs a, int v0, const float *G, const float *dloss,
                                                    const float *count, int mean, T *dw, long ld) {
  __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
  const int m0 = blockIdx.x * kTile, n0 = blockIdx.y * kTile, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const T *x = static_cast<const T *>(a.x);
  const int V = min(kPiece, a.vocab - v0);
  float acc[4][4];
  tile_product([&](int m, int k) { return m0 + m < V ? G[(size_t)k * kPiece + m0 + m] : 0.f; },
               [&](int n, int k) {
                 return n0 + n < a.dim && counted(a.tg[k], a.vocab) ? op_load<T>(x[(long)k * a.x_ld + n0 + n]) : 0.f;
               },
               a.rows, acc, sa, sb);
  const float c = ce_scale(dloss, count, mean);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = m0 + 4 * ty + i, col = n0 + 4 * tx + j;
      if (row < V && col < a.dim) dw[(long)(v0 + row) * ld + col] = op_store<T>(c * acc[i][j]);
    }
}
template <typename T>
__global__ void ce_db_kernel(const CeArgs a, int v0, const float *G, const float *dloss, const float *count, int mean,
                             T *db) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= min(kPiece, a.vocab - v0)) return;
  float s = 0.f;
  for (int n = 0; n < a.rows; ++n) s += G[(size_t)n * kPiece + c];
  db[v0 + c] = op_store<T>(ce_scale(dloss, count, mean) * s);
}

int check_args(const aideen_linear_ce_args *a) {
  OP_CHECK(a, "linear_ce: null args");
  OP_CHECK(a->dtype <= AIDEEN_F16, "linear_ce: unknown dtype");
  OP_CHECK(a->reduction <= AIDEEN_CE_SUM, "linear_ce: unknown reduction");
  OP_CHECK(a->dim >= 1 && a->dim <= (1u << 20), "linear_ce: dim must be in [1, 2^20]");
  OP_CHECK(a->vocab >= 1 && a->vocab <= (1u << 24), "linear_ce: vocab must be in [1, 2^24]");
  OP_CHECK(a->rows <= (1u << 24), "linear_ce: more than 2^24 rows");
  OP_CHECK(a->x_ld >= (int64_t)a->dim && a->w_ld >= (int64_t)a->dim, "linear_ce: row stride below dim");
  return AIDEEN_OK;
}

struct Plan {
  float2 *part;
  float *picked, *row_loss, *count, *G, *dx;
  size_t loss_bytes, grad_bytes;
};
Plan make_plan(const aideen_linear_ce_args *a, void *ws) {
  Plan p{};
  OpCarve c(ws);
  p.part = c.take<float2>((size_t)a->rows * kSlices);
  p.picked = c.take<float>(a->rows);
  p.row_loss = c.take<float>(a->rows);
  p.loss_bytes = c.used;
  OpCarve g(ws);
  p.count = g.take<float>(1);
  p.G = g.take<float>((size_t)a->rows * kPiece);
  p.dx = g.take<float>((size_t)a->rows * a->dim);
  p.grad_bytes = g.used;
  return p;
}

CeArgs ce_args(const aideen_linear_ce_args *g, const void *x, const void *w, const void *b, const int32_t *tg) {
  CeArgs a{};
  a.x = x; a.w = w; a.b = b; a.tg = tg; a.x_ld = g->x_ld; a.w_ld = g->w_ld;
  a.rows = (int)g->rows; a.dim = (int)g->dim; a.vocab = (int)g->vocab;
  return a;
}

template <typename T>
cudaError_t loss_run(const CeArgs &a, const Plan &p, int mean, float *loss, float *row_loss, float *lse, cudaStream_t st) {
  float *rl = row_loss ? row_loss : p.row_loss;
  const int tiles = (a.vocab + kTile - 1) / kTile, slices = tiles < kSlices ? tiles : kSlices;
  ce_stats_kernel<T><<<dim3((a.rows + kTile - 1) / kTile, slices), 256, 0, st>>>(a, p.part, p.picked);
  ce_rows_kernel<<<(a.rows + 255) / 256, 256, 0, st>>>(a, p.part, slices, p.picked, rl, lse);
  if (loss) ce_loss_kernel<<<1, 1024, 0, st>>>(a, rl, mean, loss, nullptr);
  return cudaGetLastError();
}

template <typename T>
cudaError_t grad_run(const CeArgs &a, const Plan &p, int mean, const float *dloss, T *dx, long dx_ld, T *dw, long dw_ld,
                     T *db, cudaStream_t st) {
  ce_loss_kernel<<<1, 1024, 0, st>>>(a, nullptr, mean, nullptr, p.count);
  const int mt = (a.rows + kTile - 1) / kTile, dt = (a.dim + kTile - 1) / kTile;
  for (int v0 = 0; v0 < a.vocab; v0 += kPiece) {
    const int V = a.vocab - v0 < kPiece ? a.vocab - v0 : kPiece, vt = (V + kTile - 1) / kTile;
    ce_piece_kernel<T><<<dim3(mt, vt), 256, 0, st>>>(a, v0, p.G);
    if (dx) ce_dx_kernel<T><<<dim3(mt, dt), 256, 0, st>>>(a, v0, p.G, p.dx, v0 == 0);
    if (dw) ce_dw_kernel<T><<<dim3(vt, dt), 256, 0, st>>>(a, v0, p.G, dloss, p.count, mean, dw, dw_ld);
    if (db) ce_db_kernel<T><<<(V + 255) / 256, 256, 0, st>>>(a, v0, p.G, dloss, p.count, mean, db);
  }
  if (dx) ce_dx_store_kernel<T><<<op_sm_count() * 4, 256, 0, st>>>(a, p.dx, dloss, p.count, mean, dx, dx_ld);
  return cudaGetLastError();
}

}  // namespace

cudaError_t linear_ce_timeout(unsigned int *out) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_ce_timeout, sizeof(*out));
  const unsigned int zero = 0;
  if (e == cudaSuccess && *out) e = cudaMemcpyToSymbol(g_ce_timeout, &zero, sizeof(zero));
  return e;
}

}  // namespace aideen

using namespace aideen;

extern "C" int aideen_linear_ce_workspace(const aideen_linear_ce_args *args, size_t *loss_bytes, size_t *grad_bytes) {
  const int rc = check_args(args);
  if (rc != AIDEEN_OK) return rc;
  const Plan p = make_plan(args, nullptr);
  if (loss_bytes) *loss_bytes = p.loss_bytes;
  if (grad_bytes) *grad_bytes = p.grad_bytes;
  return AIDEEN_OK;
}

extern "C" int aideen_linear_ce(const aideen_linear_ce_args *args, const void *x, const void *w, const void *bias,
                                const int32_t *targets, float *loss, float *row_loss, float *lse, void *workspace,
                                size_t workspace_bytes, void *stream) {
  const int rc = check_args(args);
  if (rc != AIDEEN_OK) return rc;
  const size_t el = op_elem(args->dtype);
  OP_CHECK(op_aligned(x, el) && op_aligned(w, el) && op_aligned(bias, el) && op_aligned(targets, 4) &&
               op_aligned(loss, 4) && op_aligned(row_loss, 4) && op_aligned(lse, 4),
           "linear_ce: a pointer is not aligned to its type");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->rows == 0) return loss ? op_cuda(cudaMemsetAsync(loss, 0, sizeof(float), st)) : AIDEEN_OK;
  OP_CHECK(loss || row_loss || lse, "linear_ce: no output wanted");
  OP_CHECK(x && w && targets, "linear_ce: null x, w or targets");
  const Plan p = make_plan(args, workspace);
  OP_CHECK(workspace && op_aligned(workspace, 256) && workspace_bytes >= p.loss_bytes,
           "linear_ce: workspace missing, misaligned or too small");
  const CeArgs a = ce_args(args, x, w, bias, targets);
  const int mean = args->reduction == AIDEEN_CE_MEAN;
  if (args->dtype == AIDEEN_F32) return op_cuda(loss_run<float>(a, p, mean, loss, row_loss, lse, st));
  if (args->dtype == AIDEEN_BF16) return op_cuda(loss_run<__nv_bfloat16>(a, p, mean, loss, row_loss, lse, st));
  return op_cuda(loss_run<__half>(a, p, mean, loss, row_loss, lse, st));
}

extern "C" int aideen_linear_ce_grad(const aideen_linear_ce_args *args, const void *x, const void *w, const void *bias,
                                     const int32_t *targets, const float *lse, const float *dloss, void *dx, void *dw,
                                     void *dbias, void *workspace, size_t workspace_bytes, void *stream) {
  const int rc = check_args(args);
  if (rc != AIDEEN_OK) return rc;
  OP_CHECK((!dx || args->dx_ld >= (int64_t)args->dim) && (!dw || args->dw_ld >= (int64_t)args->dim),
           "linear_ce_grad: row stride below dim");
  const size_t el = op_elem(args->dtype);
  OP_CHECK(op_aligned(x, el) && op_aligned(w, el) && op_aligned(bias, el) && op_aligned(dx, el) &&
               op_aligned(dw, el) && op_aligned(dbias, el) && op_aligned(targets, 4) && op_aligned(lse, 4) &&
               op_aligned(dloss, 4),
           "linear_ce_grad: a pointer is not aligned to its type");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->rows == 0) {  // sums over no rows
    cudaError_t e = cudaSuccess;
    if (dw) e = cudaMemset2DAsync(dw, (size_t)args->dw_ld * el, 0, args->dim * el, args->vocab, st);
    if (dbias && e == cudaSuccess) e = cudaMemsetAsync(dbias, 0, args->vocab * el, st);
    return op_cuda(e);
  }
  OP_CHECK(dx || dw || dbias, "linear_ce_grad: no output wanted");
  OP_CHECK(x && w && targets && lse, "linear_ce_grad: null x, w, targets or lse");
  const Plan p = make_plan(args, workspace);
  OP_CHECK(workspace && op_aligned(workspace, 256) && workspace_bytes >= p.grad_bytes,
           "linear_ce_grad: workspace missing, misaligned or too small");
  CeArgs a = ce_args(args, x, w, bias, targets);
  a.lse = lse;
  const int mean = args->reduction == AIDEEN_CE_MEAN;
  if (args->dtype == AIDEEN_F32)
    return op_cuda(grad_run<float>(a, p, mean, dloss, static_cast<float *>(dx), args->dx_ld, static_cast<float *>(dw),
                                   args->dw_ld, static_cast<float *>(dbias), st));
  if (args->dtype == AIDEEN_BF16)
    return op_cuda(grad_run<__nv_bfloat16>(a, p, mean, dloss, static_cast<__nv_bfloat16 *>(dx), args->dx_ld,
                                           static_cast<__nv_bfloat16 *>(dw), args->dw_ld,
                                           static_cast<__nv_bfloat16 *>(dbias), st));
  return op_cuda(grad_run<__half>(a, p, mean, dloss, static_cast<__half *>(dx), args->dx_ld, static_cast<__half *>(dw),
                                  args->dw_ld, static_cast<__half *>(dbias), st));
}
