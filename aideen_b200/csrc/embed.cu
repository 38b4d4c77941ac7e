// Embedding lookup with scaling and its gradient on caller-owned tensors.
//
//   out[n] = s E[id[n]]            dE[v] (+)= s sum_{n: id[n] = v} dout[n]
//
// Lookup: one warp per token, 16 bytes per lane and access; bound by HBM (by
// the launch for a few tokens): 32768 Zipf tokens of 50257 x 1024 bf16 take 19.3 us, the 67 MB
// that are written and the 9900 or so rows that occur, 20 MB, at 4.5 TB/s from and to HBM (the
// other 47 MB of reads come from L2); one token 2.8 us.  Rows that do not start on 16 bytes move
// element by element: 32768 x 1001 from a cold cache 33 us, where 1024 wide ones take 22.5.
//
// Gradient, bound by HBM (dout read once, the table's gradient written once):
//   1. one cluster of 1, 8 or 16 CTAs sorts (id, position) stably, by least-significant
//      digits of at most 8 bits; every warp ranks its own run of keys (lanes of
//      one digit meet in a word of shared memory), the CTAs exchange their digit
//      counts through distributed shared memory, and a hardware cluster barrier
//      separates the steps.  The sort is latency, not bandwidth, so the other CTAs
//      of the same launch clear the table's gradient meanwhile (2048 tokens and
//      103 MB to clear: 18 us, 5.7 TB/s; the sort of 65521 tokens alone about 20 us).
//   2. the sorted positions are cut into tiles of 8 or 32, one warp each (per 32
//      accesses of a row), whatever the ids are: a frequent id spreads over
//      many tiles.  A run of one id inside a tile is summed and stored; a run
//      that crosses tiles leaves float32 partial rows.
//   3. the partial rows of each crossing run are added in a fixed order.
// 2048 Zipf tokens of 50257 x 512 f32 take 27 us, 65521 of bf16 47 us.
// Nothing is added with atomics: the same call gives the same bits.
#include <cooperative_groups.h>

#include "common.cuh"
#include "operators.cuh"

namespace cg = cooperative_groups;

namespace aideen {
namespace {

constexpr int kMaxSortCtas = 16, kSortThreads = 1024, kSortWarps = kSortThreads / 32;
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
  uint32_t ctas;  // that sort: one cluster
  // table gradient to clear, or null: rows of row_bytes at a stride of ld_bytes
  unsigned char *clear;
  size_t row_bytes, ld_bytes;
  int flat, clear16;  // contiguous rows from 16 bytes on; rows can be cleared 16 bytes at a time
};

// Keys are the ids, every id outside [0, vocab) as vocab (sorted last).
__device__ __forceinline__ uint32_t sort_key(int32_t id, uint32_t vocab) {
  return id >= 0 && (uint32_t)id < vocab ? (uint32_t)id : vocab;
}

// Clears the rows: whole 32 KB blocks of zeros go out of shared memory by bulk copy
// where the rows are contiguous, else plain stores.
__device__ __forceinline__ void clear_rows(const SortArgs &s, uint32_t *zeros, size_t cta, size_t ctas) {
  constexpr size_t kBlock = sizeof(uint32_t) * kSortWarps * kDigits;  // 32 KB
  const size_t t = cta * kSortThreads + threadIdx.x, step = ctas * kSortThreads;
  if (s.flat) {
    for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) zeros[i] = 0;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    const size_t all = s.row_bytes * s.vocab, total = all & ~(size_t)15;
    if (cta == 0 && threadIdx.x < (all - total) / 2) reinterpret_cast<uint16_t *>(s.clear + total)[threadIdx.x] = 0;
    if (threadIdx.x == 0) {
      for (size_t at = cta * kBlock; at < total; at += ctas * kBlock) {
        const uint32_t n = (uint32_t)(total - at < kBlock ? total - at : kBlock);
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(s.clear + at),
                     "r"(static_cast<uint32_t>(__cvta_generic_to_shared(zeros))), "r"(n)
                     : "memory");
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
  } else if (s.clear16) {
    const size_t per = s.row_bytes / 16, total = per * s.vocab;
    for (size_t i = t; i < total; i += step)
      *reinterpret_cast<uint4 *>(s.clear + i / per * s.ld_bytes + i % per * 16) = make_uint4(0, 0, 0, 0);
  } else {
    const size_t per = s.row_bytes / 2, total = per * s.vocab;
    for (size_t i = t; i < total; i += step)
      *reinterpret_cast<uint16_t *>(s.clear + i / per * s.ld_bytes + i % per * 2) = 0;
  }
}

__global__ void __launch_bounds__(kSortThreads) embed_sort_kernel(const SortArgs s) {
  extern __shared__ __align__(16) uint32_t sort_smem[];
  uint32_t(*hist)[kDigits] = reinterpret_cast<uint32_t(*)[kDigits]>(sort_smem);               // keys per warp and digit
  uint32_t(*lanes)[kDigits] = reinterpret_cast<uint32_t(*)[kDigits]>(sort_smem + kSortWarps * kDigits);  // lanes per digit
  __shared__ uint32_t total[kDigits];  // this CTA's keys per digit, read by its peers
  __shared__ uint32_t wsum[8];
  op_begin();
  if (blockIdx.x >= s.ctas) {  // the clusters past the first clear the gradient
    clear_rows(s, sort_smem, blockIdx.x - s.ctas, gridDim.x - s.ctas);
    return;
  }
  cg::cluster_group cluster = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)blockIdx.x;
  auto sync_all = [&]() {
    if (s.ctas == 1) __syncthreads();
    else cluster.sync();
  };
  // every warp of the sorting CTAs owns one contiguous run of positions
  const uint32_t run = (s.n + s.ctas * kSortWarps - 1) / (s.ctas * kSortWarps);
  const uint32_t w = (uint32_t)(rank * kSortWarps + warp);
  const uint32_t lo = (unsigned long long)w * run < s.n ? w * run : s.n;
  const uint32_t hi = s.n - lo < run ? s.n : lo + run;
  const uint32_t mask = (1u << s.digit_bits) - 1u;
  const uint32_t below = (1u << lane) - 1u;
  constexpr int U = 4;  // keys per lane at a time
  for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) (&lanes[0][0])[i] = 0;
  for (int p = 0; p < s.passes; ++p) {
    const int shift = p * s.digit_bits;
    // the last pass writes into `a`
    unsigned long long *dst = ((s.passes - 1 - p) & 1) ? s.b : s.a;
    const unsigned long long *src = ((s.passes - 1 - p) & 1) ? s.a : s.b;
    unsigned long long kv[U];
    uint32_t at[U];  // place among the warp's keys of the same digit
    // Loads up to 32 U keys and counts them: lanes of a digit meet in its word of
    // `lanes`, the first of them adds their number to the digit's count.
    auto walk = [&](uint32_t i0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t i = i0 + u * 32 + lane;
        kv[u] = 0;
        if (i < hi) {
          if (p == 0) kv[u] = (unsigned long long)sort_key(s.ids[i], s.vocab) << 32 | i;
          else kv[u] = __ldcg(src + i);  // written by another CTA of the cluster
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i0 + u * 32 >= hi) break;
        const bool in = i0 + u * 32 + lane < hi;
        const uint32_t d = ((uint32_t)(kv[u] >> 32) >> shift) & mask;
        if (in) atomicOr(&lanes[warp][d], 1u << lane);
        __syncwarp();
        const uint32_t same = in ? lanes[warp][d] : 0;
        const uint32_t old = in ? hist[warp][d] : 0;
        at[u] = old + __popc(same & below);
        __syncwarp();
        if (in && (same & below) == 0) {
          hist[warp][d] = old + __popc(same);
          lanes[warp][d] = 0;
        }
        __syncwarp();
      }
    };
    for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) (&hist[0][0])[i] = 0;
    __syncthreads();
    for (uint32_t i0 = lo; i0 < hi; i0 += 32 * U) walk(i0);
    __syncthreads();
    if (threadIdx.x < kDigits) {  // counts of the warps before, per digit
      uint32_t sum = 0, count[kSortWarps];
#pragma unroll
      for (int k = 0; k < kSortWarps; ++k) count[k] = hist[k][threadIdx.x];
#pragma unroll
      for (int k = 0; k < kSortWarps; ++k) {
        hist[k][threadIdx.x] = sum;
        sum += count[k];
      }
      total[threadIdx.x] = sum;
    }
    sync_all();
    uint32_t before = 0, all = 0, x = 0;
    if (threadIdx.x < kDigits) {
      if (s.ctas == 1) {
        all = total[threadIdx.x];
      } else {
        uint32_t v[kMaxSortCtas];
#pragma unroll
        for (int c = 0; c < kMaxSortCtas; ++c) v[c] = c < (int)s.ctas ? *cluster.map_shared_rank(&total[threadIdx.x], c) : 0;
#pragma unroll
        for (int c = 0; c < kMaxSortCtas; ++c) {
          if (c < rank) before += v[c];
          all += v[c];
        }
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
      uint32_t base = x - all + before, count[kSortWarps];
      for (int k = 0; k < warp; ++k) base += wsum[k];
#pragma unroll
      for (int k = 0; k < kSortWarps; ++k) count[k] = hist[k][threadIdx.x];
#pragma unroll
      for (int k = 0; k < kSortWarps; ++k) hist[k][threadIdx.x] = count[k] + base;
    }
    __syncthreads();
    if (hi - lo <= 32 * U) {  // the keys and their places are still here
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (lo + u * 32 + lane < hi) dst[hist[warp][((uint32_t)(kv[u] >> 32) >> shift) & mask] + at[u]] = kv[u];
    } else {  // count again, from the bases on
      for (uint32_t i0 = lo; i0 < hi; i0 += 32 * U) {
        walk(i0);
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (i0 + u * 32 + lane < hi) dst[at[u]] = kv[u];
      }
    }
    sync_all();  // the pass's writes and reads of `total` are done everywhere
  }
}

constexpr int kBatch = 8;       // rows of a warp in flight
constexpr int kJoinWarps = 16;  // tiles that a joining CTA looks at

// Sorted positions per warp: one batch while that gives the GPU too few warps, else
// four, for a quarter of the partial rows (the gradient of 65521 x 512 bf16 takes 52 us
// with two batches, 48 us with four; with 3 CTAs on an SM instead of 4, which leaves a
// second wave of a few CTAs, 74 us).
int tile_of(uint32_t n) { return n <= 16384 ? kBatch : 4 * kBatch; }

struct SumArgs {
  const unsigned long long *sorted;
  const void *dout;
  void *grad;
  float *part;  // [tiles][2][dim]: the run that enters the tile, the run that leaves it
  uint32_t n, vocab;
  int dim, tile, slabs, accumulate;  // slabs: of 32 accesses per row
  float scale;
  long table_ld, rows_ld;
};

template <int VEC>
__device__ __forceinline__ void part_store(float *p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    *p = v[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  }
}

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

// One warp sums a tile over the columns of one access per lane.  The warps of a row's
// slabs are neighbours, so that its bytes are asked for together.  Keys are uniform over
// the warp.
template <typename T, int VEC>
__global__ void __launch_bounds__(256, 4) embed_sum_kernel(const SumArgs a) {
  op_begin();
  const int lane = threadIdx.x & 31;
  const unsigned long long gw = (unsigned long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const uint32_t tile = (uint32_t)(gw / a.slabs);
  const unsigned long long begin = (unsigned long long)tile * a.tile;
  if (begin >= a.n) return;
  const uint32_t lo = (uint32_t)begin;
  const int n = a.n - lo < (uint32_t)a.tile ? (int)(a.n - lo) : a.tile;
  const int c = ((int)(gw % a.slabs) * 32 + lane) * VEC;
  const bool live = c < a.dim;
  // loads without branches (behind the row and outside the table some valid row's start is
  // read and not used), or each would wait for the one before
  const T *dout = static_cast<const T *>(a.dout) + (live ? c : 0);
  const unsigned long long mine = lane < n ? a.sorted[lo + lane] : ~0ull;
  const unsigned long long outer = lane == 0 ? (lo > 0 ? a.sorted[lo - 1] : ~0ull) : lane == 1 && lo + n < a.n ? a.sorted[lo + n] : ~0ull;
  const uint32_t key = (uint32_t)(mine >> 32);
  uint32_t before = __shfl_up_sync(0xffffffffu, key, 1);
  const uint32_t prev = (uint32_t)(__shfl_sync(0xffffffffu, outer, 0) >> 32), next = (uint32_t)(__shfl_sync(0xffffffffu, outer, 1) >> 32);
  if (lane == 0) before = prev;
  const uint32_t starts = __ballot_sync(0xffffffffu, lane < n && key != before);  // positions that begin a run
  float acc[VEC] = {};
  bool entered = !(starts & 1u);  // the run at work began in an earlier tile
  uint32_t at = __shfl_sync(0xffffffffu, key, 0);
  // Stores the finished run: `leaves` where it goes on in the next tile.
  auto finish = [&](bool leaves) {
    if (live && at < a.vocab) {
      if (entered || leaves) part_store<VEC>(a.part + ((size_t)tile * 2 + (entered ? 0 : 1)) * a.dim + c, acc);
      else embed_finish<T, VEC>(a, at, c, acc);
    }
  };
  for (int b0 = 0; b0 < n; b0 += kBatch) {
    OpVec<T, VEC> v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const uint32_t pos = (uint32_t)__shfl_sync(0xffffffffu, mine, min(b0 + u, n - 1));
      op_load_ahead<T, VEC>(dout + (long)pos * a.rows_ld, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (b0 + u >= n) break;
      if (b0 + u > 0 && (starts >> (b0 + u) & 1u)) {
        finish(false);
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
        entered = false;
        at = __shfl_sync(0xffffffffu, key, b0 + u);
      }
      if (at < a.vocab) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += op_load<T>(v[u].v[i]);
      }
    }
  }
  finish(next == at);
}

// Adds the partial rows of the runs that cross tiles, in a fixed order.  Each warp looks
// at one tile: does its last run begin in it and leave it, and how many more tiles does
// it enter?  Up to kShort of them the warp adds alone; longer runs take the whole CTA
// (warp w adds the parts w, w + 16, ..., then the warps are added in order).
template <typename T, int VEC>
__global__ void __launch_bounds__(32 * kJoinWarps) embed_join_kernel(const SumArgs a) {
  constexpr uint32_t kShort = 7;
  __shared__ float sh[kJoinWarps][32 * VEC];
  __shared__ uint32_t more_of[kJoinWarps], key_of[kJoinWarps];
  op_begin();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t tile = blockIdx.x * kJoinWarps + warp;
  const unsigned long long end = ((unsigned long long)tile + 1) * a.tile;
  uint32_t more = 0, key = ~0u;
  if (end < a.n) {
    const uint32_t hi = (uint32_t)end, lo = hi - a.tile;
    key = (uint32_t)(a.sorted[hi - 1] >> 32);
    const uint32_t next = (uint32_t)(a.sorted[hi] >> 32), first = (uint32_t)(a.sorted[lo] >> 32);
    const uint32_t prev = lo > 0 ? (uint32_t)(a.sorted[lo - 1] >> 32) : ~0u;
    if (key < a.vocab && next == key && !(first == key && prev == key)) {
      for (more = 1;; more += 32) {  // lane i: does the run leave tile + more + i too?
        const unsigned long long at = ((unsigned long long)tile + more + lane + 1) * a.tile;
        const bool on = at < a.n && (uint32_t)(a.sorted[at] >> 32) == key;
        const uint32_t off = __ballot_sync(0xffffffffu, !on);
        if (off) {
          more += __ffs(off) - 1;
          break;
        }
      }
    }
  }
  if (lane == 0) {
    more_of[warp] = more;
    key_of[warp] = key;
  }
  const int c = (blockIdx.y * 32 + lane) * VEC;
  auto add = [&](uint32_t t0, uint32_t from, uint32_t by, uint32_t count, float (&acc)[VEC]) {
    if (c >= a.dim) return;
#pragma unroll 8
    for (uint32_t t = from; t <= count; t += by) {
      const float *p = a.part + ((size_t)(t0 + t) * 2 + (t == 0 ? 1 : 0)) * a.dim + c;
      float v[VEC];
      if constexpr (VEC == 1) {
        v[0] = *p;
      } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
          const float4 x = *reinterpret_cast<const float4 *>(p + i);
          v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
        }
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] += v[i];
    }
  };
  if (more > 0 && more <= kShort) {
    float acc[VEC] = {};
    add(tile, 0, 1, more, acc);
    if (c < a.dim) embed_finish<T, VEC>(a, key, c, acc);
  }
  const uint32_t any = __syncthreads_or(more > kShort);
  if (!any) return;
  for (int k = 0; k < kJoinWarps; ++k) {
    if (more_of[k] <= kShort) continue;
    float acc[VEC] = {};
    add(blockIdx.x * kJoinWarps + k, warp, kJoinWarps, more_of[k], acc);
#pragma unroll
    for (int i = 0; i < VEC; ++i) sh[warp][lane * VEC + i] = acc[i];
    __syncthreads();
    if (warp == 0 && c < a.dim) {
      for (int q = 1; q < kJoinWarps; ++q) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] += sh[q][lane * VEC + i];
      }
      embed_finish<T, VEC>(a, key_of[k], c, acc);
    }
    __syncthreads();
  }
}

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
  p.tiles = (n + tile_of(n) - 1) / tile_of(n);
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
cudaError_t sum_run(SumArgs s, uint32_t tiles, cudaStream_t st) {
  s.slabs = (s.dim + 32 * VEC - 1) / (32 * VEC);
  const unsigned long long warps = (unsigned long long)tiles * s.slabs;
  cudaError_t e = op_launch(embed_sum_kernel<T, VEC>, (unsigned)((warps + 7) / 8), 256, 0, st, s);
  if (e != cudaSuccess || tiles < 2) return e;
  return op_launch(embed_join_kernel<T, VEC>, dim3((tiles + kJoinWarps - 1) / kJoinWarps, s.slabs), 32 * kJoinWarps, 0, st, s);
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
  // up to 4 keys per lane of one CTA the cluster's barriers cost more than they save
  s.ctas = args->n_tokens <= 4 * kSortThreads ? 1 : args->n_tokens <= 32 * kSortThreads ? 8 : kMaxSortCtas;
  s.digit_bits = s.passes ? (bits + s.passes - 1) / s.passes : 1;
  unsigned grid = s.ctas;
  if (!args->accumulate) {
    s.clear = static_cast<unsigned char *>(table_grad);
    s.row_bytes = args->dim * el; s.ld_bytes = (size_t)args->table_ld * el;
    s.flat = s.row_bytes == s.ld_bytes && op_aligned(table_grad, 16);
    s.clear16 = s.flat || (s.row_bytes % 16 == 0 && op_vec16(table_grad, args->table_ld, el));
    // several CTAs per SM, so that uneven placement of the clusters evens out
    const size_t stores = s.flat ? s.row_bytes * s.vocab / 16 + 1 : s.row_bytes / (s.clear16 ? 16 : 2) * s.vocab;
    const size_t ctas = (stores + kSortThreads - 1) / kSortThreads;
    const size_t most = op_round(4 * (size_t)op_sm_count(), s.ctas), want = op_round(ctas, s.ctas);
    grid += (unsigned)(want < most ? want : most);
  }
  const int smem = 2 * kSortWarps * kDigits * (int)sizeof(uint32_t);
  cudaError_t e = cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess && s.ctas > 8)  // past the portable size
    e = cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) e = op_launch_cluster(embed_sort_kernel, s.ctas, grid, kSortThreads, smem, st, s);
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
