// Embedding lookup with scaling and its gradient on caller-owned tensors.
//
//   out[n] = s E[id[n]]            dE[v] (+)= s sum_{n: id[n] = v} dout[n]
//
// Lookup: one warp per token, 16 bytes per lane and access; bound by HBM (by
// the launch for a few tokens).
//
// Gradient, bound by HBM (dout read once, the table's gradient written once):
//   1. one cluster of 8 CTAs sorts (id, position) stably, by least-significant
//      digits of at most 8 bits; every warp ranks its own run of keys with
//      match.any, the CTAs exchange their digit counts through distributed
//      shared memory, and a hardware cluster barrier separates the steps.  The
//      sort is latency, not bandwidth, so the other CTAs of the same launch
//      clear the table's gradient meanwhile.
//   2. the sorted positions are cut into equal tiles, one warp each (per 32
//      accesses of a row), whatever the ids are: a frequent id spreads over
//      many tiles.  A run of one id inside a tile is summed and stored; a run
//      that crosses tiles leaves float32 partial rows.
//   3. the partial rows of each crossing run are added in tile order.
// Nothing is added with atomics: the same call gives the same bits.
#include <cooperative_groups.h>

#include "common.cuh"
#include "operators.cuh"

namespace cg = cooperative_groups;

namespace aideen {
namespace {

constexpr int kSortCtas = 8, kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kDigits = 256;

template <typename T, int VEC>
__global__ void embed_kernel(const int32_t *__restrict__ ids, const T *__restrict__ table, T *__restrict__ out,
                             long n, int dim, int vocab, float scale, long table_ld, long rows_ld) {
  op_begin();
  const int lane = threadIdx.x & 31;
  const long row = (long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (row >= n) return;
  const int id = ids[row];
  T *o = out + row * rows_ld;
  if (id < 0 || id >= vocab) {
    const float zero[VEC] = {};
    for (int c = lane * VEC; c < dim; c += 32 * VEC) op_store_vec<T, VEC>(o + c, zero);
    return;
  }
  const T *e = table + (long)id * table_ld;
  constexpr int U = 4;  // accesses in flight per lane
  for (int c0 = lane * VEC; c0 < dim; c0 += 32 * VEC * U) {
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * 32 * VEC < dim) op_load_vec<T, VEC>(e + c0 + u * 32 * VEC, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c0 + u * 32 * VEC >= dim) break;
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[u][i] *= scale;
      op_store_vec<T, VEC>(o + c0 + u * 32 * VEC, v[u]);
    }
  }
}

struct SortArgs {
  const int32_t *ids;
  unsigned long long *a, *b;  // sorted (key << 32 | position) ends in `a`
  uint32_t n, vocab;
  int passes, digit_bits;
  // table gradient to clear, or null: rows of row_bytes at a stride of ld_bytes
  unsigned char *clear;
  size_t row_bytes, ld_bytes;
  int clear16;  // rows can be cleared 16 bytes at a time
};

// Keys are the ids, every id outside [0, vocab) as vocab (sorted last).
__device__ __forceinline__ uint32_t sort_key(int32_t id, uint32_t vocab) {
  return id >= 0 && (uint32_t)id < vocab ? (uint32_t)id : vocab;
}

__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortThreads)
    embed_sort_kernel(const SortArgs s) {
  op_begin();
  if (blockIdx.x >= kSortCtas) {  // the clusters past the first clear the gradient
    const size_t t = (size_t)(blockIdx.x - kSortCtas) * kSortThreads + threadIdx.x;
    const size_t step = (size_t)(gridDim.x - kSortCtas) * kSortThreads;
    if (s.clear16 && s.row_bytes == s.ld_bytes) {
      const size_t total = s.row_bytes / 16 * s.vocab;
      for (size_t i = t; i < total; i += step) reinterpret_cast<uint4 *>(s.clear)[i] = make_uint4(0, 0, 0, 0);
    } else if (s.clear16) {
      const size_t per = s.row_bytes / 16, total = per * s.vocab;
      for (size_t i = t; i < total; i += step)
        *reinterpret_cast<uint4 *>(s.clear + i / per * s.ld_bytes + i % per * 16) = make_uint4(0, 0, 0, 0);
    } else {
      const size_t per = s.row_bytes / 2, total = per * s.vocab;
      for (size_t i = t; i < total; i += step)
        *reinterpret_cast<uint16_t *>(s.clear + i / per * s.ld_bytes + i % per * 2) = 0;
    }
    return;
  }
  __shared__ uint32_t hist[kSortWarps][kDigits];
  __shared__ uint32_t total[kDigits];  // this CTA's keys per digit, read by its peers
  __shared__ uint32_t wsum[8];
  cg::cluster_group cluster = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cluster.block_rank();
  // every warp of the cluster owns one contiguous run of positions
  const uint32_t run = (s.n + kSortCtas * kSortWarps - 1) / (kSortCtas * kSortWarps);
  const uint32_t w = (uint32_t)(rank * kSortWarps + warp);
  const uint32_t lo = (unsigned long long)w * run < s.n ? w * run : s.n;
  const uint32_t hi = s.n - lo < run ? s.n : lo + run;
  const uint32_t mask = (1u << s.digit_bits) - 1u;
  const uint32_t below = (1u << lane) - 1u;
  for (int p = 0; p < s.passes; ++p) {
    const int shift = p * s.digit_bits;
    // the last pass writes into `a`
    unsigned long long *dst = ((s.passes - 1 - p) & 1) ? s.b : s.a;
    const unsigned long long *src = ((s.passes - 1 - p) & 1) ? s.a : s.b;
    auto load = [&](uint32_t i) -> unsigned long long {
      if (p == 0) return (unsigned long long)sort_key(s.ids[i], s.vocab) << 32 | i;
      return __ldcg(src + i);  // written by another CTA of the cluster
    };
    for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) (&hist[0][0])[i] = 0;
    __syncthreads();
    for (uint32_t i0 = lo; i0 < hi; i0 += 32) {
      const bool in = i0 + lane < hi;
      const uint32_t live = __ballot_sync(0xffffffffu, in);
      if (in) {
        const uint32_t d = ((uint32_t)(load(i0 + lane) >> 32) >> shift) & mask;
        const uint32_t same = __match_any_sync(live, d);
        if ((same & below) == 0) hist[warp][d] += __popc(same);
      }
      __syncwarp();
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {  // counts of the warps before, per digit
      uint32_t sum = 0;
      for (int k = 0; k < kSortWarps; ++k) {
        const uint32_t c = hist[k][threadIdx.x];
        hist[k][threadIdx.x] = sum;
        sum += c;
      }
      total[threadIdx.x] = sum;
    }
    cluster.sync();
    uint32_t before = 0, all = 0, x = 0;
    if (threadIdx.x < kDigits) {
      for (int c = 0; c < kSortCtas; ++c) {
        const uint32_t v = *cluster.map_shared_rank(&total[threadIdx.x], c);
        if (c < rank) before += v;
        all += v;
      }
      x = all;  // inclusive scan over the digits
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) wsum[warp] = x;
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      uint32_t base = x - all + before;
      for (int k = 0; k < warp; ++k) base += wsum[k];
      for (int k = 0; k < kSortWarps; ++k) hist[k][threadIdx.x] += base;
    }
    __syncthreads();
    for (uint32_t i0 = lo; i0 < hi; i0 += 32) {
      const bool in = i0 + lane < hi;
      const uint32_t live = __ballot_sync(0xffffffffu, in);
      uint32_t d = 0, same = 0;
      if (in) {
        const unsigned long long kv = load(i0 + lane);
        d = ((uint32_t)(kv >> 32) >> shift) & mask;
        same = __match_any_sync(live, d);
        dst[hist[warp][d] + __popc(same & below)] = kv;
      }
      __syncwarp();
      if (in && (same & below) == 0) hist[warp][d] += __popc(same);
      __syncwarp();
    }
    cluster.sync();  // the pass's writes and reads of `total` are done everywhere
  }
}

struct SumArgs {
  const unsigned long long *sorted;
  const void *dout;
  void *grad;
  float *part;  // [tiles][2][dim]: the run that enters the tile, the run that leaves it
  uint32_t n, vocab;
  int dim, tile, accumulate;
  float scale;
  long table_ld, rows_ld;
};

template <typename T, int VEC>
__device__ __forceinline__ void embed_finish(const SumArgs &a, uint32_t key, int c, float (&acc)[VEC]) {
  T *g = static_cast<T *>(a.grad) + (long)key * a.table_ld + c;
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] *= a.scale;
  if (a.accumulate) {
    float old[VEC];
    op_load_vec<T, VEC>(g, old);
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] += old[i];
  }
  op_store_vec<T, VEC>(g, acc);
}

// One warp sums tile blockIdx.x * warps + warp over the columns of one lane's
// access (blockIdx.y picks 32 of them).  Keys are uniform over the warp.
template <typename T, int VEC>
__global__ void embed_sum_kernel(const SumArgs a) {
  op_begin();
  const int lane = threadIdx.x & 31;
  const uint32_t tile = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const unsigned long long begin = (unsigned long long)tile * a.tile;
  if (begin >= a.n) return;
  const uint32_t lo = (uint32_t)begin, hi = a.n - lo < (uint32_t)a.tile ? a.n : lo + a.tile;
  const int c = (blockIdx.y * 32 + lane) * VEC;
  const bool live = c < a.dim;
  const T *dout = static_cast<const T *>(a.dout) + c;
  uint32_t key = (uint32_t)(a.sorted[lo] >> 32);
  bool entered = lo > 0 && (uint32_t)(a.sorted[lo - 1] >> 32) == key;
  float acc[VEC] = {};
  constexpr int U = 8;  // rows in flight
  for (uint32_t i0 = lo; i0 < hi; i0 += U) {
    unsigned long long kv[U];
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) kv[u] = i0 + u < hi ? a.sorted[i0 + u] : ~0ull;
    if (live) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if ((uint32_t)(kv[u] >> 32) < a.vocab) op_load_vec<T, VEC>(dout + (long)(uint32_t)kv[u] * a.rows_ld, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u >= hi) break;
      const uint32_t k = (uint32_t)(kv[u] >> 32);
      if (k != key) {  // the run before this position is complete
        if (live && key < a.vocab) {
          if (entered) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) a.part[(size_t)tile * 2 * a.dim + c + i] = acc[i];
          } else {
            embed_finish<T, VEC>(a, key, c, acc);
          }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
        key = k;
        entered = false;
      }
      if (live && k < a.vocab) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += v[u][i];
      }
    }
  }
  if (!live || key >= a.vocab) return;
  const bool leaves = hi < a.n && (uint32_t)(a.sorted[hi] >> 32) == key;
  if (entered || leaves) {
    float *p = a.part + ((size_t)tile * 2 + (entered ? 0 : 1)) * a.dim + c;
#pragma unroll
    for (int i = 0; i < VEC; ++i) p[i] = acc[i];
  } else {
    embed_finish<T, VEC>(a, key, c, acc);
  }
}

// One CTA per tile whose last run begins in it and leaves it: adds the run's
// partial rows.  Warp w takes the parts w, w + 8, ...; the warps are then added
// in order.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_join_kernel(const SumArgs a) {
  __shared__ float sh[8][32 * VEC];
  op_begin();
  const uint32_t tile = blockIdx.x;
  const uint32_t lo = tile * (uint32_t)a.tile;
  const unsigned long long end = (unsigned long long)lo + a.tile;
  if (end >= a.n) return;
  const uint32_t hi = (uint32_t)end;
  const uint32_t key = (uint32_t)(a.sorted[hi - 1] >> 32);
  if (key >= a.vocab || (uint32_t)(a.sorted[hi] >> 32) != key) return;          // nothing leaves
  if ((uint32_t)(a.sorted[lo] >> 32) == key && lo > 0 && (uint32_t)(a.sorted[lo - 1] >> 32) == key) return;  // begun earlier
  // first position behind the run
  uint32_t l = hi, r = a.n;
  while (l < r) {
    const uint32_t m = l + (r - l) / 2;
    if ((uint32_t)(a.sorted[m] >> 32) > key) r = m;
    else l = m + 1;
  }
  const uint32_t last = (l - 1) / a.tile;  // the tile in which the run ends
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = (blockIdx.y * 32 + lane) * VEC;
  float acc[VEC] = {};
  if (c < a.dim) {
#pragma unroll 4
    for (uint32_t t = tile + warp; t <= last; t += 8) {
      const float *p = a.part + ((size_t)t * 2 + (t == tile ? 1 : 0)) * a.dim + c;
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += p[i];
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) sh[warp][lane * VEC + i] = acc[i];
  __syncthreads();
  if (warp != 0 || c >= a.dim) return;
  for (int k = 1; k < 8; ++k) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] += sh[k][lane * VEC + i];
  }
  embed_finish<T, VEC>(a, key, c, acc);
}

// Sorted positions per warp: enough warps to fill the GPU while there are few
// tokens, few partial rows once there are many.
int tile_of(uint32_t n) { return n <= 16384 ? 8 : 32; }

struct GradPlan {
  unsigned long long *a, *b;
  float *part;
  size_t bytes;
  uint32_t tiles;
};
GradPlan grad_plan(const aideen_embed_args *args, void *ws) {
  GradPlan p{};
  OpCarve c(ws);
  const uint32_t n = args->n_tokens;
  p.tiles = (uint32_t)(((unsigned long long)n + tile_of(n) - 1) / tile_of(n));
  p.a = c.take<unsigned long long>(n);
  p.b = c.take<unsigned long long>(n);
  p.part = c.take<float>((size_t)p.tiles * 2 * args->dim);
  p.bytes = c.used;
  return p;
}

template <typename T, int VEC>
cudaError_t embed_run(const aideen_embed_args *a, const int32_t *ids, const void *table, void *out, cudaStream_t st) {
  const int warps = a->n_tokens < 8 ? (int)a->n_tokens : 8;
  return op_launch(embed_kernel<T, VEC>, (unsigned)(((long)a->n_tokens + warps - 1) / warps), warps * 32, 0, st, ids,
                   static_cast<const T *>(table), static_cast<T *>(out), a->n_tokens, a->dim, a->vocab, a->scale,
                   a->table_ld, a->rows_ld);
}

template <typename T, int VEC>
cudaError_t sum_run(const SumArgs &s, uint32_t tiles, cudaStream_t st) {
  const unsigned slabs = (unsigned)((s.dim + 32 * VEC - 1) / (32 * VEC));
  cudaError_t e = op_launch(embed_sum_kernel<T, VEC>, dim3((tiles + 7) / 8, slabs), 256, 0, st, s);
  if (e != cudaSuccess || tiles < 2) return e;
  return op_launch(embed_join_kernel<T, VEC>, dim3(tiles - 1, slabs), 256, 0, st, s);
}

int check_args(const aideen_embed_args *a) {
  OP_CHECK(a, "embed: null args");
  OP_CHECK(a->dtype <= AIDEEN_F16, "embed: unknown dtype");
  OP_CHECK(a->dim >= 1 && a->dim <= (1u << 20), "embed: dim must be in [1, 2^20]");
  OP_CHECK(a->vocab >= 1 && a->vocab <= (1u << 30), "embed: vocab must be in [1, 2^30]");
  OP_CHECK(a->n_tokens <= (1u << 30), "embed: more than 2^30 tokens");
  OP_CHECK(a->accumulate <= 1, "embed: accumulate must be 0 or 1");
  OP_CHECK(a->table_ld >= (int64_t)a->dim && a->rows_ld >= (int64_t)a->dim, "embed: row stride below dim");
  return AIDEEN_OK;
}

}  // namespace
}  // namespace aideen

using namespace aideen;

extern "C" int aideen_embed(const aideen_embed_args *args, const int32_t *ids, const void *table, void *out,
                            void *stream) {
  const int rc = check_args(args);
  if (rc != AIDEEN_OK) return rc;
  if (args->n_tokens == 0) return AIDEEN_OK;
  OP_CHECK(ids && table && out, "embed: null ids, table or out");
  const size_t el = op_elem(args->dtype);
  OP_CHECK(op_aligned(ids, 4) && op_aligned(table, el) && op_aligned(out, el),
           "embed: a pointer is not aligned to its type");
  const bool vec = (args->dim * el) % 16 == 0 && op_vec16(table, args->table_ld, el) && op_vec16(out, args->rows_ld, el);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->dtype == AIDEEN_F32)
    return op_cuda(vec ? embed_run<float, 4>(args, ids, table, out, st) : embed_run<float, 1>(args, ids, table, out, st));
  if (args->dtype == AIDEEN_BF16)
    return op_cuda(vec ? embed_run<__nv_bfloat16, 8>(args, ids, table, out, st)
                       : embed_run<__nv_bfloat16, 1>(args, ids, table, out, st));
  return op_cuda(vec ? embed_run<__half, 8>(args, ids, table, out, st) : embed_run<__half, 1>(args, ids, table, out, st));
}

extern "C" int aideen_embed_grad_workspace(const aideen_embed_args *args, size_t *bytes) {
  const int rc = check_args(args);
  if (rc != AIDEEN_OK) return rc;
  OP_CHECK(bytes, "embed_grad: null bytes");
  *bytes = grad_plan(args, nullptr).bytes;
  return AIDEEN_OK;
}

extern "C" int aideen_embed_grad(const aideen_embed_args *args, const int32_t *ids, const void *dout,
                                 void *table_grad, void *workspace, size_t workspace_bytes, void *stream) {
  const int rc = check_args(args);
  if (rc != AIDEEN_OK) return rc;
  OP_CHECK(table_grad, "embed_grad: null table_grad");
  OP_CHECK(args->n_tokens == 0 || (ids && dout), "embed_grad: null ids or dout");
  const size_t el = op_elem(args->dtype);
  OP_CHECK(op_aligned(ids, 4) && op_aligned(dout, el) && op_aligned(table_grad, el),
           "embed_grad: a pointer is not aligned to its type");
  OP_CHECK(args->n_tokens == 0 ||
               (workspace && op_aligned(workspace, 256) && workspace_bytes >= grad_plan(args, nullptr).bytes),
           "embed_grad: workspace missing, misaligned or too small");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (args->n_tokens == 0 && args->accumulate) return AIDEEN_OK;
  const GradPlan p = grad_plan(args, workspace);
  SortArgs s{};
  s.ids = ids; s.a = p.a; s.b = p.b; s.n = args->n_tokens; s.vocab = args->vocab;
  int bits = 1;
  while (args->vocab >> bits) ++bits;  // keys run up to vocab itself
  s.passes = args->n_tokens ? (bits + 7) / 8 : 0;
  s.digit_bits = s.passes ? (bits + s.passes - 1) / s.passes : 1;
  unsigned grid = kSortCtas;
  if (!args->accumulate) {
    s.clear = static_cast<unsigned char *>(table_grad);
    s.row_bytes = args->dim * el; s.ld_bytes = (size_t)args->table_ld * el;
    s.clear16 = s.row_bytes % 16 == 0 && op_vec16(table_grad, args->table_ld, el);
    // one CTA of 1024 threads per remaining SM, in whole clusters, at most one pass over the table
    const size_t ctas = (s.row_bytes / (s.clear16 ? 16 : 2) * s.vocab + kSortThreads - 1) / kSortThreads;
    const size_t most = (size_t)(op_sm_count() - kSortCtas) / kSortCtas * kSortCtas;
    const size_t want = op_round(ctas, kSortCtas);
    grid += (unsigned)(want < most || most == 0 ? want : most);
  }
  const cudaError_t e = op_launch(embed_sort_kernel, grid, kSortThreads, 0, st, s);
  if (e != cudaSuccess || args->n_tokens == 0) return op_cuda(e);
  SumArgs m{};
  m.sorted = p.a; m.dout = dout; m.grad = table_grad; m.part = p.part;
  m.n = args->n_tokens; m.vocab = args->vocab; m.dim = (int)args->dim; m.tile = tile_of(args->n_tokens);
  m.accumulate = (int)args->accumulate; m.scale = args->scale;
  m.table_ld = args->table_ld; m.rows_ld = args->rows_ld;
  const bool vec = (args->dim * el) % 16 == 0 && op_vec16(dout, args->rows_ld, el) && op_vec16(table_grad, args->table_ld, el);
  if (args->dtype == AIDEEN_F32) return op_cuda(vec ? sum_run<float, 4>(m, p.tiles, st) : sum_run<float, 1>(m, p.tiles, st));
  if (args->dtype == AIDEEN_BF16)
    return op_cuda(vec ? sum_run<__nv_bfloat16, 8>(m, p.tiles, st) : sum_run<__nv_bfloat16, 1>(m, p.tiles, st));
  return op_cuda(vec ? sum_run<__half, 8>(m, p.tiles, st) : sum_run<__half, 1>(m, p.tiles, st));
}
