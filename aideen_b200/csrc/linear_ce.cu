// Softmax cross entropy of a linear head over the vocabulary, without keeping
// the logits, and its gradient, on caller-owned tensors.
//
//   z = x W^T + b,  lse[n] = log sum_v exp z[n][v],  loss[n] = lse[n] - z[n][t[n]]
//   G = softmax(z) - onehot(t)  (0 where the row is not counted)
//   dx = c G W,  dW = c G^T x,  db = c sum_n G,   c = dloss / counted rows
//
// Steps:
//   stage   counted rows of x are gathered to the front (a padded row costs no
//           product and its contents reach nothing) as 16-bit operands; float32
//           becomes two float16 pieces (see below).
//   stats   z tile by tile on the tensor cores; the epilogue keeps a running
//           maximum and sum per row and stores nothing else.
//   rows    joins the partial statistics, forms z[n][t[n]] as a plain dot product.
//   pieces  (gradient) for each piece of the vocabulary: z again, G into a
//           16-bit buffer of one piece, then one launch for both products with G.
//
// Tensor-core kernel (ce_mma_kernel): a persistent grid of CTA pairs, each on
// 256 x 256 tiles (tcgen05.mma cta_group::2: every CTA holds 128 rows of the
// accumulator and loads half of either operand).  Per CTA: warp 0 streams 64-deep
// slices by TMA into a ring that takes what the shared memory has left (up to eight
// stages of 32 KB, or of 16 KB where the row tile of x stays in shared memory and
// only W streams), warp 1 of the leading CTA issues the MMAs into one of two
// 256-column accumulators in tensor memory, and warps 2..9 drain the other one.
// A pair tile is the largest that leaves two accumulators: an operand byte from L2
// carries 256 products, so that L2 does not bound it.
//
// float32: each of x, W and G = softmax - onehot is scaled by powers of two that bring
// its largest magnitude (G: 1) to 2^14..2^15 and written as high + low float16 pieces;
// high x high + high x low + low x high leave out 2^-22 of a product, three passes where
// bfloat16 pieces would take six (training shard 50257 x 512, 2048 rows, loss and gradient:
// 2.23 ms with those, 1.45 ms this way).  For the logits every row of x and of W has its own
// scale, so that a row of W that dwarfs the others costs them nothing: with one scale, a
// masked row 10^8 times the others put lse off by 1e-3.  The products with G add up over
// rows, so there x and W have one scale each, in a second layout of the gradient, where what
// lies below 2^-40 of the largest magnitude is rounded off.
//
// 16 bits: G is rounded to the type before the two products, as the tensor cores take it.  The
// gradients of the large bf16 batch below are then 1.68e-3 from 64 bits in the 2-norm, where
// rounding the results alone gives 1.66e-3 (f16, 1021 x 4999 x 250: 2.2e-4 and 2.1e-4); a second
// piece of G would take the products, 525 us of that batch's 1370, twice.  db needs no product and
// adds up the float32 values.
//
// Bound: the tensor cores (2 N V d for the loss, 6 N V d for the gradient, z being
// formed twice), and behind them the power limit: 8192 rows, nine in ten counted, 50257 x 512
// bf16, loss and gradient take 1.37 ms, 1.10 PFLOP/s, at clocks that the limit holds at 1.3-1.5 GHz.
//
// Every wait is bounded; a wait that runs out sets an error word, issues nothing
// further, lets its copies land, frees the tensor memory and returns.
#include <cuda.h>

#include <type_traits>

#include "common.cuh"
#include "operators.cuh"
#include "tc_common.cuh"

namespace aideen {
namespace {

__device__ unsigned int g_ce_timeout;

constexpr int kTileM = 256, kTileN = 256, kBlockK = 64;
constexpr int kHalfBytes = 128 * kBlockK * 2;  // one CTA's half of an operand slice: 16 KB
constexpr int kMaxStages = 8, kMaxHeld = 8;    // ring depth; slices of x that stay in shared memory
constexpr int kEpiWarps = 8, kThreads = 64 + 32 * kEpiWarps;
constexpr int kBoxBytes = 4096;  // 32 rows of 128 bytes
constexpr uint32_t kWaitLimit = 1u << 24;
constexpr float kLog2e = 1.4426950408889634f;
// float16 keeps softmax - onehot times 2^12: probabilities down to 2^-26 stay
// normal numbers, and the largest magnitude is 2^12
constexpr float kHalfScale = 4096.f;
// and float32's two pieces of it times 2^14
constexpr float kPieceScale = 16384.f;
// Shared memory of a CTA: held slices of x, the ring, the epilogue's boxes, the
// bias of two tiles, barriers, and in float32 the exponents of W's factors.
constexpr int kSmemLimit = 232448, kSmemBarriers = 512;
constexpr int smem_fixed(int mode, size_t elem) {
  return 2 * kTileN * 4 + kSmemBarriers + (elem == 4 && mode != 2 ? 2 * kTileN : 0);
}

enum { kStats = 0, kPiece = 1, kProducts = 2 };

struct MmaArgs {
  const int *count;   // counted rows
  int vocab, dim;
  int planes;         // 16-bit pieces per operand element: 1, or 2 for float32
  // float32: what x and W were divided by: counted rows' and vocabulary rows' own factors
  // (kStats, kPiece), [2] for the products
  const float *xinv, *winv, *unscale;
  uint32_t idesc;     // operand types of the instruction descriptor
  int stages;         // ring depth
  // kStats, kPiece: vocabulary tiles [0, tiles_n) from column v0 on
  int v0, tiles_n;
  const void *bias;
  float2 *stats;      // kStats: [slot][2][256] (maximum, sum of e^(z - maximum))
  const float *lse;   // kPiece: compacted rows' lse
  const int32_t *tgt; // and their targets
  float *db_part;     // [8 tiles_m][tiles_n * 256] column sums of 32 rows each, or null
  float g_scale;
  // kProducts
  int bn;             // columns of an output tile: 128 or 256
  int tiles_d;        // of dim
  int piece_k;        // 64-deep slices of the piece
  int full_k;         // and of the first piece (the last may be shorter)
  int want_dw;
  int slabs;          // slabs of dx (0: dx not wanted)
  uint8_t *cover;     // [row tiles][tiles_d] slabs that hold something
  int first;          // first piece: dx slabs are written, not added to
  int dw_vec;         // dW: elements per access (see row_width); 16 bytes: stored by TMA
  void *dw, *db;
  long dw_ld;
  const float *dloss;
  int mean;
};

__device__ __forceinline__ float grad_scale(const float *dloss, const int *count, int mean) {
  return (dloss ? *dloss : 1.f) / (mean ? fmaxf((float)*count, 1.f) : 1.f);
}

// ---- pair-of-CTAs primitives ------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of the leading CTA's copy of a shared-memory object.
__device__ __forceinline__ uint32_t leader_addr(const void *p) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
  return a;
}
// True in one lane of a converged warp, the same one at every call.  With it, not
// with lane == 0, the compiler knows that a single thread follows, and issues MMAs
// and copies straight from uniform registers (at 8192 x 50257 x 512 the loss kernel
// without its loads went from 1410 to 1680 TFLOP/s).
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ bool wait_bounded(uint64_t *bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  for (uint32_t i = 0; i < kWaitLimit; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}
// Load into this CTA's shared memory; the bytes are counted on `bar` of the
// leading CTA.
__device__ __forceinline__ void pair_load(void *dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void pair_mma(uint32_t tmem, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
      "l"(da), "l"(db), "r"(idesc), "r"(accumulate));
}
// Arrives on `bar` of both CTAs once every MMA issued so far is done.
__device__ __forceinline__ void pair_commit(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void remote_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
      "%28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const float (&v)[32]) {
  uint32_t r[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(v[i]);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
      "%11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, "
      "%28, %29, %30, %31, %32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// e^(a - b).  The difference comes before the change of base: a logit that float32 holds need
// not fit it in base 2, and the largest terms get small exponents, rounded finely.
__device__ __forceinline__ float exp_diff(float a, float b) { return exp2_fast((a - b) * kLog2e); }
// The same for two at a time (two float32 lanes per instruction), b given as (-b, -b).
__device__ __forceinline__ float2 exp_diff(float2 a, float2 minus_b) {
  const float2 e = __fmul2_rn(__fadd2_rn(a, minus_b), make_float2(kLog2e, kLog2e));
  return make_float2(exp2_fast(e.x), exp2_fast(e.y));
}

// A power of two f in two halves, f.x about its square root and f.x f.y = f (also where f is
// Inf).  Applied before and after another factor they leave float32's range only where the
// result does: what one multiplication by both would round to a subnormal number, or
// overflow, may be in range.
__device__ __forceinline__ float2 halves(float f) {
  const int e = (((int)(__float_as_uint(f) >> 23) & 255) - 127) >> 1;
  return make_float2(__uint_as_float((uint32_t)(127 + e) << 23), f * __uint_as_float((uint32_t)(127 - e) << 23));
}

// Products of pieces in the order they are added: low x high, high x low, high x high.
__device__ __forceinline__ void product_pair(int planes, int j, int &pa, int &pb) {
  pa = planes == 2 && j == 0;
  pb = planes == 2 && j == 1;
}

// One output tile of a launch.
struct Unit {
  int m, n;      // tile coordinates (rows of 256, columns of kTileN or bn)
  int kb0, nkb;  // 64-deep slices
  int dw;        // kProducts: 1 = dW tile, 0 = dx tile
  int z;         // dx: slab
  bool first, last;  // chunks of the tile's depth
};

// How a piece's two products are dealt out over the pairs.  dW tiles go out whole
// (tiles of the piece x tiles_d, each as deep as the rows): pairs below n_a
// take w + 1 of them, the others w.  dx fills up what is missing to an equal
// load: its slices, ordered by (tile, depth), are cut into one run per pair, a
// slices for a pair below n_a and b for the others.  A tile that several pairs
// work on takes one float32 slab from each, added in order at the end; a run is
// never shorter than a tile's depth / (slabs - 1), so `slabs` are enough.
struct Deal {
  int w, n_a, depth;
  long a, b, total, load;
  __host__ __device__ Deal(long n_dw, long k_rows, long dx_tiles, int depth_, int slabs, int pairs) {
    depth = depth_;
    w = (int)(n_dw / pairs);
    n_a = (int)(n_dw % pairs);
    total = dx_tiles * depth;
    const long least = slabs > 1 ? (depth + slabs - 2) / (slabs - 1) : depth;
    load = (n_dw * k_rows + total + pairs - 1) / pairs;
    a = n_a ? load - (w + 1) * k_rows : 0;
    b = load - w * k_rows;
    if (a < least) {
      a = 0;
      b = (total + pairs - n_a - 1) / (pairs - n_a);
    }
    if (b < least) b = least;
    if (b < 1) b = 1;
    const long la = n_a ? (w + 1) * k_rows + a : 0, lb = w * k_rows + (total ? b : 0);
    load = la > lb ? la : lb;
  }
  __host__ __device__ long begin(int pair) const {
    const long at = pair < n_a ? pair * a : n_a * a + (pair - n_a) * b;
    return at < total ? at : total;
  }
  __device__ int owner(long slice) const {
    return slice < n_a * a ? (int)(slice / a) : n_a + (int)((slice - n_a * a) / b);
  }
  // slabs that a tile takes
  __device__ int cover(long tile) const { return owner((tile + 1) * depth - 1) - owner(tile * depth) + 1; }
};

// Rows that are worked on: whole tiles, and one tile of zeros (it writes dW)
// where no row is counted.
__device__ __forceinline__ int row_tiles(int count) { return max(1, (count + kTileM - 1) / kTileM); }
__device__ __forceinline__ Deal deal_of(int count, int tiles_v, int tiles_d, int depth, int want_dw, int slabs, int pairs) {
  return Deal(want_dw ? (long)tiles_v * tiles_d : 0, max(1, (count + kBlockK - 1) / kBlockK),
              slabs ? (long)row_tiles(count) * tiles_d : 0, depth, slabs, pairs);
}

// float32's products with G take a tile's depth in chunks of this many slices, each
// added to what the ones before stored: the tensor cores cut where they add, by up to a
// unit of the sum at each 16 deep, always towards zero.  Over the 16384 rows of a dW that
// grew to 1.9e-5 of it; in chunks it stays at 1e-6 for any number of rows, at 8% of the
// gradient's time.  z is cut the same way over its depth, by 4e-7 of it at 512 and eight times
// that at 4096, so deeper logits of float32 are added in chunks too (DEEP below).
constexpr int kChunk = 8;

// Units of one pair.  kStats and kPiece: a contiguous share of the (row tile,
// vocabulary tile) order, so that a pair stays on one row tile.  kProducts: its
// dW tiles, then its run of dx.
template <int MODE, bool CHUNKS>
struct Units {
  const MmaArgs &a;
  Deal deal;
  Unit tile;
  int depth = 0;     // slices of `tile` given out
  int pair, k_dim, k_rows;
  long next, end;    // tiles (kStats, kPiece) or dW tiles
  long dx, dx_end;   // slices of dx
  __device__ __forceinline__ Units(const MmaArgs &args, int count)
      : a(args),
        deal(deal_of(count, args.piece_k * kBlockK / kTileM, args.tiles_d, args.piece_k, args.want_dw, args.slabs,
                     (int)(gridDim.x >> 1))) {
    const long pairs = gridDim.x >> 1;
    pair = (int)(blockIdx.x >> 1);
    k_dim = (a.dim + kBlockK - 1) / kBlockK;
    k_rows = max(1, (count + kBlockK - 1) / kBlockK);
    if (MODE == kProducts) {
      next = (long)pair * deal.w + min(pair, deal.n_a);
      end = next + deal.w + (pair < deal.n_a ? 1 : 0);
      dx = deal.begin(pair);
      dx_end = deal.begin(pair + 1);
    } else {
      const long total = (long)row_tiles(count) * a.tiles_n;
      next = pair * total / pairs;
      end = (pair + 1) * total / pairs;
      dx = dx_end = 0;
    }
    tile.nkb = 0;
  }
  __device__ __forceinline__ bool get(Unit &u) {
    if (!CHUNKS) {
      u.first = u.last = true;
      return get_tile(u);
    }
    if (depth >= tile.nkb) {
      if (!get_tile(tile)) return false;
      depth = 0;
    }
    u = tile;
    u.kb0 += depth;
    u.nkb = min(kChunk, tile.nkb - depth);
    u.first = depth == 0;
    depth += u.nkb;
    u.last = depth >= tile.nkb;
    return true;
  }
  __device__ __forceinline__ bool get_tile(Unit &u) {
    if (next < end) {
      const int per = MODE == kProducts ? a.tiles_d : a.tiles_n;
      u.m = (int)(next / per);
      u.n = (int)(next % per);
      u.kb0 = 0;
      u.nkb = MODE == kProducts ? k_rows : k_dim;
      u.dw = MODE == kProducts;
      u.z = 0;
      ++next;
      return true;
    }
    if (MODE != kProducts || dx >= dx_end) return false;
    const long tile = dx / deal.depth;
    u.m = (int)(tile / a.tiles_d);
    u.n = (int)(tile % a.tiles_d);
    u.kb0 = (int)(dx % deal.depth);
    u.nkb = (int)min((long)(deal.depth - u.kb0), dx_end - dx);
    u.dw = 0;
    u.z = pair - deal.owner(tile * deal.depth);
    dx += u.nkb;
    return true;
  }
};

// Writes 32 columns of a lane's row (two calls fill a box of 64 16-bit columns).
template <typename T>
__device__ __forceinline__ void box_put16(unsigned char *box, int lane, int half, const float (&v)[32]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    OpVec<T, 8> x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x.v[i] = op_store<T>(v[8 * k + i]);
    *reinterpret_cast<OpVec<T, 8> *>(box + lane * 128 + (((half * 4 + k) ^ (lane & 7)) * 16)) = x;
  }
}
__device__ __forceinline__ void box_put32(unsigned char *box, int lane, const float (&v)[32]) {
#pragma unroll
  for (int k = 0; k < 8; ++k)
    *reinterpret_cast<float4 *>(box + lane * 128 + ((k ^ (lane & 7)) * 16)) =
        make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
}

// Sums of 32 columns over the warp's 32 rows; lane l gets column l.  Halves of the columns
// change hands while a lane has several.
__device__ __forceinline__ float column_sums(const float (&v)[32], int lane) {
  float t[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float send = lane & 16 ? v[i] : v[i + 16], keep = lane & 16 ? v[i + 16] : v[i];
    t[i] = keep + __shfl_xor_sync(0xffffffffu, send, 16);
  }
#pragma unroll
  for (int n = 8; n > 0; n >>= 1) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float send = lane & n ? t[i] : t[i + n], keep = lane & n ? t[i + n] : t[i];
      t[i] = keep + __shfl_xor_sync(0xffffffffu, send, n);
    }
  }
  return t[0];
}

// One warp's N staging boxes, used in turn: take() gives one whose last store has
// been read, send() hands it to TMA.
template <int N>
struct Boxes {
  unsigned char *base;
  int n = 0;
  __device__ __forceinline__ unsigned char *take() {
    unsigned char *b = base + (N == 2 ? (n & 1) * kBoxBytes : 0);
    if (elect_one()) bulk_wait_read<N == 2 ? 1 : 0>();
    __syncwarp();
    return b;
  }
  __device__ __forceinline__ void send(const CUtensorMap *map, const unsigned char *box, int x, int y, int z,
                                       bool add) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (elect_one()) {
      if (add) tma_reduce_add_3d(map, box, x, y, z);
      else tma_store_3d(map, box, x, y, z);
      bulk_commit();
    }
    ++n;
  }
};

struct Maps {
  CUtensorMap a, b;    // kStats, kPiece: x and W by rows.  kProducts, dx: G by rows, W by columns
  CUtensorMap a2, b2;  // kProducts, dW: G by columns, x by columns
  CUtensorMap c, c2;   // stores: kPiece: G.  kProducts: dx slabs, dW
};

// db of a piece, by the epilogue warps while they have nothing to drain yet: the
// sums of 32 rows each are added in order, 64 columns and 4 strided partial sums per
// CTA and turn.
template <typename T>
__device__ __forceinline__ void db_columns(const MmaArgs &a, int count, int etid, float *sh) {
  const int groups = row_tiles(count) * 8, cols = a.tiles_n * kTileN;
  const float scale = grad_scale(a.dloss, a.count, a.mean) / a.g_scale;
  for (int c0 = blockIdx.x * 64; c0 < cols; c0 += gridDim.x * 64) {
    const float *part = a.db_part + c0 + (etid & 63);
    float s = 0.f;
#pragma unroll 8
    for (int g = etid >> 6; g < groups; g += 4) s += part[(size_t)g * cols];
    sh[etid] = s;
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
    const int v = a.v0 + c0 + etid;
    if (etid < 64 && v < a.vocab)
      static_cast<T *>(a.db)[v] = op_store<T>(scale * (((sh[etid] + sh[etid + 64]) + sh[etid + 128]) + sh[etid + 192]));
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
  }
}

// 8192 x 50257 x 512 bf16, a tenth of the rows not counted, one launch at a time: kStats
// 235 us (1.62 PFLOP/s), the five kPiece launches 318 us (1.19; G goes out to L2 and HBM
// meanwhile), the five kProducts 529 us (1.43; G comes back for either product).  2048
// rows in float32, three products each: 211 us (1.50), 257 us and 542 us.
//
// HELD (kStats, kPiece with one piece per element and dim <= 512): the row tile of x stays in
// shared memory while the pair walks along the vocabulary, and the ring carries W only.
//
// DEEP (kStats, kPiece in float32 with dim > 512): the chunks of a tile's depth are added in
// float32.  The first stays in its accumulator, the later ones pass one by one through the
// other, and the epilogue adds each to the first in tensor memory; the next tile starts in
// the one that is free first.  It costs 1% of loss and gradients at 2048 x 50257 x 1024 (2.6 ms).
template <int MODE, typename T, bool HELD, bool DEEP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    ce_mma_kernel(const __grid_constant__ Maps maps, const MmaArgs a) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char *sm = smem_raw;
  if (smem_u32(sm) & 1023) {  // the swizzled tiles need it; the same in every CTA
    if (threadIdx.x == 0) atomicCAS(&g_ce_timeout, 0u, 1u);
    return;
  }
  constexpr int kStageBytes = HELD ? kHalfBytes : 2 * kHalfBytes;
  constexpr int kBoxesPerWarp = MODE == kStats ? 0 : HELD ? 1 : 2;
  const int stages = a.stages, held = HELD ? (a.dim + kBlockK - 1) / kBlockK : 0;
  unsigned char *ring = sm + held * kHalfBytes;
  unsigned char *boxes = ring + stages * kStageBytes;
  float *sbias = reinterpret_cast<float *>(boxes + kEpiWarps * kBoxesPerWarp * kBoxBytes);  // [2][kTileN]
  uint64_t *full = reinterpret_cast<uint64_t *>(sbias + 2 * kTileN);
  uint64_t *empty = full + kMaxStages;
  uint64_t *hfull = empty + kMaxStages;   // held slices loaded
  uint64_t *hempty = hfull + kMaxHeld;    // and no longer read
  uint64_t *tfull = hempty + kMaxHeld;
  uint64_t *tempty = tfull + 2;
  uint64_t *done = tempty + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 1);
  uint32_t *err = tmem_slot + 1;
  uint8_t *sfac = reinterpret_cast<uint8_t *>(full) + kSmemBarriers;  // float32: [2][kTileN]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();

  if (tid == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kMaxHeld; ++s) {
      mbar_init(&hfull[s], 1);
      mbar_init(&hempty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 2 * kEpiWarps);
    }
    mbar_init(done, 1);
    *err = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(2u * kTileN));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_barrier();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  op_begin();
  const int count = *a.count;
  const int products = a.planes == 1 ? 1 : 3;
  const int bn = MODE == kProducts ? a.bn : kTileN;  // columns of a tile; either CTA loads half
  constexpr bool kChunks = MODE == kProducts && sizeof(T) == 4;
  Units<MODE, kChunks || DEEP> units(a, count);
  Unit u{};
  // The accumulator that a unit goes to, and how often that was used before: in turn, or as
  // DEEP has it.
  int unit_no = 0, side = 1, used0 = 0, used1 = 0;
  auto place = [&](int &acc, int &use) {
    if constexpr (DEEP) {
      if (u.first) side ^= 1;
      acc = u.first ? side : side ^ 1;
      use = acc ? used1++ : used0++;
    } else {
      acc = unit_no & 1;
      use = unit_no >> 1;
    }
    ++unit_no;
  };

  if (warp == 0) {
    if (elect_one()) {  // ---------------- loads
      uint32_t it = 0, s = 0, turn = 0;  // slices so far, ring place, turn of the ring
      int gen = -1, last_m = -1;         // row tiles held so far
      bool ok = true;
      const uint32_t bytes = 2u * ((HELD ? 0 : kHalfBytes) + bn / 2 * kBlockK * 2);  // of both CTAs
      while (ok && units.get(u)) {
        const int m0 = u.m * kTileM + (int)rank * 128, n0 = u.n * bn + (int)rank * (bn / 2);
        const bool fresh = HELD && u.m != last_m;
        if (fresh) ++gen;
        last_m = u.m;
        for (int j = 0; j < products && ok; ++j) {
          int pa, pb;
          product_pair(a.planes, j, pa, pb);
          for (int kb = 0; kb < u.nkb; ++kb, ++it) {
            const int k0 = (u.kb0 + kb) * kBlockK;
            if (fresh) {
              if (gen > 0 && !wait_bounded(&hempty[kb], (gen - 1) & 1)) { ok = false; break; }
              if (rank == 0) mbar_expect_tx(&hfull[kb], 2 * kHalfBytes);
              pair_load(sm + kb * kHalfBytes, &maps.a, leader_addr(&hfull[kb]), k0, m0, 0);
            }
            if (turn > 0 && !wait_bounded(&empty[s], (turn - 1) & 1)) { ok = false; break; }
            unsigned char *sa = ring + s * kStageBytes, *sb = HELD ? sa : sa + kHalfBytes;
            const uint32_t bar = leader_addr(&full[s]);
            if (rank == 0) mbar_expect_tx(&full[s], bytes);
            if (MODE != kProducts) {
              if (!HELD) pair_load(sa, &maps.a, bar, k0, m0, pa);
              pair_load(sb, &maps.b, bar, k0, a.v0 + n0, pb);
            } else if (u.dw) {
              for (int c = 0; c < 2; ++c) pair_load(sa + c * 8192, &maps.a2, bar, m0 + 64 * c, k0, pa);
              for (int c = 0; c < bn / 128; ++c) pair_load(sb + c * 8192, &maps.b2, bar, n0 + 64 * c, k0, pb);
            } else {
              pair_load(sa, &maps.a, bar, k0, m0, pa);
              for (int c = 0; c < bn / 128; ++c) pair_load(sb + c * 8192, &maps.b, bar, n0 + 64 * c, a.v0 + k0, pb);
            }
            if (++s == (uint32_t)stages) { s = 0; ++turn; }
          }
        }
      }
      if (!ok) atomicExch(err, 1u);
      // every place's last use is over (its arrival has landed here) before this CTA may leave
      const uint32_t used = it < (uint32_t)stages ? it : (uint32_t)stages;
      for (uint32_t i = 0; i < used; ++i) {
        const uint32_t t = i < s ? turn : turn - 1;  // the turn of place i's last load
        if (ok && !wait_bounded(&empty[i], t & 1)) { ok = false; atomicExch(err, 1u); }
        if (!ok && rank == 0) wait_bounded(&full[i], t & 1);  // let a copy in flight land
      }
      for (int kb = 0; kb < held && gen >= 0; ++kb) {
        if (ok && !wait_bounded(&hempty[kb], gen & 1)) { ok = false; atomicExch(err, 1u); }
        if (!ok && rank == 0) wait_bounded(&hfull[kb], gen & 1);
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {  // ---------------- MMAs
      uint32_t s = 0, turn = 0;
      int gen = -1, last_m = -1;
      bool ok = true;
      while (ok && units.get(u)) {
        int acc, use;
        place(acc, use);
        const bool fresh = HELD && u.m != last_m;
        const bool leaving = HELD && (u.n == a.tiles_n - 1 || units.next >= units.end);  // last tile of these rows
        if (fresh) ++gen;
        last_m = u.m;
        if (use > 0 && !wait_bounded(&tempty[acc], (use - 1) & 1)) { ok = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        // rows by 64: 128-byte rows, 8-row groups 1024 apart; columns by 64: blocks of 64
        // columns 8192 apart, 8-row groups 1024 apart
        const bool acol = MODE == kProducts && u.dw, bcol = MODE == kProducts;
        const uint32_t idesc = a.idesc | (acol ? 1u << 15 : 0u) | (bcol ? 1u << 16 : 0u) | (uint32_t)(bn >> 3) << 17 |
                               (uint32_t)(kTileM >> 4) << 24;
        const uint32_t lbo_a = acol ? 8192u : 16u, lbo_b = bcol ? 8192u : 16u;
        const uint32_t ka = acol ? 2048u : 32u, kb_ = bcol ? 2048u : 32u;  // 16 deep
        const uint32_t d = tmem + (uint32_t)acc * kTileN;
        const uint64_t desc_a = sdesc(sm, lbo_a, 1024u, 2u);
        const uint64_t desc_b = sdesc(sm + (HELD ? 0 : kHalfBytes), lbo_b, 1024u, 2u);
        const int ring_at = held * kHalfBytes;
        const int total = products * u.nkb;
        for (int k = 0; k < total; ++k) {
          if (fresh && !wait_bounded(&hfull[k], gen & 1)) { ok = false; break; }
          if (!wait_bounded(&full[s], turn & 1)) { ok = false; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t da = desc_a + ((HELD ? k * kHalfBytes : ring_at + (int)s * kStageBytes) >> 4);
          const uint64_t db = desc_b + ((ring_at + (int)s * kStageBytes) >> 4);
#pragma unroll
          for (int q = 0; q < kBlockK / 16; ++q) pair_mma(d, da + q * (ka >> 4), db + q * (kb_ >> 4), idesc, k > 0 || q > 0);
          pair_commit(&empty[s]);
          if (leaving) pair_commit(&hempty[k]);
          if (++s == (uint32_t)stages) { s = 0; ++turn; }
        }
        if (!ok) break;
        pair_commit(&tfull[acc]);
      }
      if (!ok) atomicExch(err, 1u);
      pair_commit(done);
      wait_bounded(done, 0);  // every MMA of the pair is over
    }
  } else {  // ---------------- epilogue: lanes are accumulator rows
    const int q = warp & 3, half = (warp - 2) >> 2;  // tensor-memory lane quarter, half of the columns
    const uint32_t lane_addr = tmem + ((uint32_t)(q * 32) << 16);
    Boxes<kBoxesPerWarp> box{boxes + (warp - 2) * kBoxesPerWarp * kBoxBytes};
    const int etid = tid - 64;
    int last_m = -1;
    float run_m = -INFINITY, run_s = 0.f;  // kStats: this row's statistics over the pair's tiles
    float lse = 0.f;
    int32_t tgt = -1;
    const float scale = MODE == kProducts ? grad_scale(a.dloss, a.count, a.mean) / a.g_scale : 0.f;
    // float32: x's factor, of the products or of this lane's row
    float2 fx = MODE == kProducts && sizeof(T) == 4 ? halves(a.unscale[0]) : make_float2(1.f, 1.f);
    const Deal full_deal = deal_of(count, a.full_k * kBlockK / kTileM, a.tiles_d, a.full_k, a.want_dw, a.slabs,
                                   (int)(gridDim.x >> 1));
    if (MODE == kProducts && a.slabs) {  // the last piece may be shorter than the others, and deal dx differently
      const long tiles = (long)row_tiles(count) * a.tiles_d;
      for (long t = (long)blockIdx.x * 32 * kEpiWarps + etid; t < tiles; t += (long)gridDim.x * 32 * kEpiWarps)
        a.cover[t] = (uint8_t)max(full_deal.cover(t), units.deal.cover(t));
    }
    if (MODE == kProducts && a.db_part) db_columns<T>(a, count, etid, sbias);
    auto flush = [&]() {
      if (last_m < 0) return;
      const size_t slot = (size_t)(blockIdx.x >> 1) + last_m;
      a.stats[(slot * 2 + half) * kTileM + rank * 128 + q * 32 + lane] = make_float2(run_m, run_s);
    };
    bool dead = false;  // a wait ran out: keep the barriers below in step, touch nothing
    while (units.get(u)) {
      const int turn = unit_no & 1;  // of the buffers of a tile's bias
      int acc, use;
      place(acc, use);
      const float *sb = sbias + turn * kTileN;
      uint32_t some_out = 0;
      if (MODE != kProducts) {
        // this tile's bias (-Inf behind the vocabulary); the buffer's last reader passed
        // the barrier of the tile before
        const int v = a.v0 + u.n * kTileN + etid;
        float b = -INFINITY;
        if (v < a.vocab) b = a.bias ? op_load<T>(static_cast<const T *>(a.bias)[v]) : 0.f;
        sbias[turn * kTileN + etid] = b;
        if (sizeof(T) == 4) sfac[turn * kTileN + etid] = v < a.vocab ? (uint8_t)(__float_as_uint(a.winv[v]) >> 23) : 127;
        // (and whether a bias of -Inf or the vocabulary's end takes some columns out)
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t"
            "setp.ne.u32 q, %1, 0;\n\t"
            "bar.red.or.pred p, 1, %2, q;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(some_out)
            : "r"((uint32_t)(b == -INFINITY)), "n"(32 * kEpiWarps)
            : "memory");
        if (u.m != last_m) {
          const int row = u.m * kTileM + (int)rank * 128 + q * 32 + lane;
          if (sizeof(T) == 4) fx = halves(row < count ? a.xinv[row] : 1.f);
          if (MODE == kStats) {
            flush();
            run_m = -INFINITY;
            run_s = 0.f;
          } else {
            lse = row < count ? a.lse[row] : 0.f;
            tgt = row < count ? a.tgt[row] : -1;
          }
          last_m = u.m;
        }
      }
      if (!dead && (!wait_bounded(&tfull[acc], use & 1) || *(volatile uint32_t *)err)) {
        atomicExch(err, 1u);
        dead = true;
      }
      if (__any_sync(0xffffffffu, dead)) {
        dead = true;
        continue;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int hcols = bn / 2;  // this warp's columns
      auto release = [&](int which) {  // the accumulator has been read: hand it back
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (elect_one()) remote_arrive(leader_addr(&tempty[which]));
      };
      if constexpr (DEEP) {
        if (u.first) continue;  // stays
        const uint32_t from = lane_addr + (uint32_t)(acc * kTileN + half * hcols);
        const uint32_t to = lane_addr + (uint32_t)((acc ^ 1) * kTileN + half * hcols);
#pragma unroll 1
        for (int c = 0; c < kTileN / 2; c += 32) {
          float v[32], w[32];
          tmem_load32(from + c, v);
          if (c + 32 == kTileN / 2) release(acc);
          tmem_load32(to + c, w);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] += w[i];
          tmem_store32(to + c, v);
        }
        if (!u.last) continue;
        acc ^= 1;
      }
      const uint32_t t0 = lane_addr + (uint32_t)(acc * kTileN + half * hcols);
      const int row0 = u.m * kTileM + (int)rank * 128 + q * 32;
      // 32 of this warp's columns; `last`: the accumulator is not read again
      auto fetch = [&](int c, float (&v)[32], bool last) {
        tmem_load32(t0 + c, v);
        if (last) release(acc);
      };
      // Which of 32 columns are taken out, whatever their logits are: an overflow to +Inf would
      // make them NaN.
      auto masked = [&](int c) { return __ballot_sync(0xffffffffu, sb[half * hcols + c + lane] == -INFINITY); };
      // float32: z of columns c.. c + 3 (of this warp's, c a multiple of 4) from their accumulators
      auto unscale4 = [&](float *v, int c) {
        const uint32_t e = reinterpret_cast<const uint32_t *>(sfac + turn * kTileN + half * hcols)[c >> 2];
        const float2 f[2] = {make_float2(__uint_as_float(e << 23 & 0x7f800000u), __uint_as_float(e << 15 & 0x7f800000u)),
                             make_float2(__uint_as_float(e << 7 & 0x7f800000u), __uint_as_float(e >> 1 & 0x7f800000u))};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float2 z = __fmul2_rn(make_float2(v[2 * i], v[2 * i + 1]), make_float2(fx.x, fx.x));
          z = __fmul2_rn(__fmul2_rn(z, f[i]), make_float2(fx.y, fx.y));
          v[2 * i] = z.x;
          v[2 * i + 1] = z.y;
        }
      };
      if (MODE == kStats) {
        auto walk = [&](auto some) {  // some: columns may be taken out
#pragma unroll 1
          for (int c = 0; c < kTileN / 2; c += 32) {
            float v[32];
            fetch(c, v, c + 32 == kTileN / 2);
            float2 z[16];
            const float4 *b4 = reinterpret_cast<const float4 *>(sb + half * hcols + c);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float4 b = b4[k];
              if constexpr (sizeof(T) == 4) unscale4(v + 4 * k, c + 4 * k);
              z[2 * k] = __fadd2_rn(make_float2(v[4 * k], v[4 * k + 1]), make_float2(b.x, b.y));
              z[2 * k + 1] = __fadd2_rn(make_float2(v[4 * k + 2], v[4 * k + 3]), make_float2(b.z, b.w));
            }
            if constexpr (decltype(some)::value) {
              const uint32_t out = masked(c);
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                if (out >> (2 * k) & 1) z[k].x = -INFINITY;
                if (out >> (2 * k + 1) & 1) z[k].y = -INFINITY;
              }
            }
            float top = run_m;
#pragma unroll
            for (int k = 0; k < 16; ++k) top = fmaxf(fmaxf(top, z[k].x), z[k].y);
            const float ref = top == -INFINITY ? 0.f : top;  // nothing but -Inf so far
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 16; ++k) sum = __fadd2_rn(sum, exp_diff(z[k], make_float2(-ref, -ref)));
            run_s = run_s * exp_diff(run_m, ref) + (sum.x + sum.y);
            run_m = top;
          }
        };
        // (a test for them in every step costs 3% at 8192 x 50257 x 128 bf16)
        if (some_out) walk(std::true_type{});
        else walk(std::false_type{});
      } else if (MODE == kPiece) {
        const int n0 = u.n * kTileN + half * hcols;
        const float2 nlse = make_float2(-lse, -lse);
#pragma unroll 1
        for (int c = 0; c < kTileN / 2; c += 64) {
          float v[2][32];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            fetch(c + 32 * h, v[h], c + 64 == kTileN / 2 && h == 1);
            const float4 *b4 = reinterpret_cast<const float4 *>(sb + half * hcols + c + 32 * h);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float4 b = b4[k];
              if constexpr (sizeof(T) == 4) unscale4(v[h] + 4 * k, c + 32 * h + 4 * k);
              const float2 p = exp_diff(__fadd2_rn(make_float2(v[h][4 * k], v[h][4 * k + 1]), make_float2(b.x, b.y)), nlse);
              const float2 q = exp_diff(__fadd2_rn(make_float2(v[h][4 * k + 2], v[h][4 * k + 3]), make_float2(b.z, b.w)), nlse);
              v[h][4 * k] = p.x; v[h][4 * k + 1] = p.y;
              v[h][4 * k + 2] = q.x; v[h][4 * k + 3] = q.y;
            }
          }
          if (some_out || row0 + 32 > count) {  // and rows behind the last, whatever an infinite W made of them
            const float p = exp_diff(-INFINITY, lse);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t out = masked(c + 32 * h);
#pragma unroll
              for (int k = 0; k < 32; ++k) {
                if (out >> k & 1) v[h][k] = p;
                if (row0 + lane >= count) v[h][k] = 0.f;
              }
            }
          }
          const int at = tgt - (a.v0 + n0 + c);  // the target's column among these 64
          if (__any_sync(0xffffffffu, at >= 0 && at < 64)) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (32 * h + k == at) v[h][k] -= 1.f;
          }
          if (a.g_scale != 1.f) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int k = 0; k < 32; k += 2) {
                const float2 g = __fmul2_rn(make_float2(v[h][k], v[h][k + 1]), make_float2(a.g_scale, a.g_scale));
                v[h][k] = g.x; v[h][k + 1] = g.y;
              }
          }
          if (a.db_part) {  // before any rounding
            float *sums = a.db_part + (size_t)(row0 >> 5) * a.tiles_n * kTileN + n0 + c + lane;
            sums[0] = column_sums(v[0], lane);
            sums[32] = column_sums(v[1], lane);
          }
          if constexpr (sizeof(T) == 2) {
            unsigned char *bx = box.take();
            box_put16<T>(bx, lane, 0, v[0]);
            box_put16<T>(bx, lane, 1, v[1]);
            box.send(&maps.c, bx, n0 + c, row0, 0, false);
          } else {
            for (int p = 0; p < 2; ++p) {
              unsigned char *bx = box.take();
              box_put16<__half>(bx, lane, 0, v[0]);
              box_put16<__half>(bx, lane, 1, v[1]);
              box.send(&maps.c, bx, n0 + c, row0, p, false);
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int k = 0; k < 32; ++k) v[h][k] -= __half2float(__float2half_rn(v[h][k]));
            }
          }
        }
      } else {
        const int n0 = u.n * bn + half * hcols;
        // dx: into a slab that an earlier piece wrote already?
        const bool add = !u.first || (!u.dw && !a.first && u.z < full_deal.cover((long)u.m * a.tiles_d + u.n));
        if (kChunks && !u.first) {  // the chunks before have to be there
          if (elect_one()) bulk_wait<0>();
          __syncwarp();
        }
        const int vrow = a.v0 + row0;
        // through a box, so that a warp writes along rows where TMA cannot
        auto write_rows = [&](const unsigned char *bx, int col, int width) {
          __syncwarp();
          T *o = static_cast<T *>(a.dw) + (long)vrow * a.dw_ld + col;
          const int rows = min(32, a.vocab - vrow), cols = min(width, a.dim - col);
          if constexpr (sizeof(T) == 2) {
            if (a.dw_vec == 2) {
              if (2 * lane < cols) {
#pragma unroll 8
                for (int r = 0; r < rows; ++r)
                  *reinterpret_cast<uint32_t *>(o + (long)r * a.dw_ld + 2 * lane) =
                      *reinterpret_cast<const uint32_t *>(bx + r * 128 + ((4 * lane) ^ ((r & 7) * 16)));
              }
              __syncwarp();
              return;
            }
          }
#pragma unroll 4
          for (int r = 0; r < rows; ++r)
            for (int c = lane; c < cols; c += 32) {
              T v = *reinterpret_cast<const T *>(bx + r * 128 + ((c * (int)sizeof(T)) ^ ((r & 7) * 16)));
              if constexpr (kChunks) v += u.first ? 0.f : o[(long)r * a.dw_ld + c];
              o[(long)r * a.dw_ld + c] = v;
            }
          __syncwarp();
        };
#pragma unroll 1
        for (int c = 0; c < hcols; c += 64) {
          float v[2][32];
          fetch(c, v[0], false);
          fetch(c + 32, v[1], c + 64 == hcols);
          const int col = n0 + c;
          if (u.dw) {
            if (col >= a.dim || vrow >= a.vocab) continue;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int k = 0; k < 32; ++k) {
                if constexpr (sizeof(T) == 4) v[h][k] = v[h][k] * fx.x * scale * fx.y;
                else v[h][k] *= scale;
              }
            if constexpr (sizeof(T) == 2) {
              unsigned char *bx = box.take();
              box_put16<T>(bx, lane, 0, v[0]);
              box_put16<T>(bx, lane, 1, v[1]);
              if (a.dw_vec == 8) box.send(&maps.c2, bx, col, vrow, 0, false);
              else write_rows(bx, col, 64);
            } else {
              for (int h = 0; h < 2; ++h) {
                if (col + 32 * h >= a.dim) continue;
                unsigned char *bx = box.take();
                box_put32(bx, lane, h ? v[1] : v[0]);
                if (a.dw_vec == 4) box.send(&maps.c2, bx, col + 32 * h, vrow, 0, add);
                else write_rows(bx, col + 32 * h, 32);
              }
            }
          } else {
            for (int h = 0; h < 2; ++h) {
              if (col + 32 * h >= a.dim) continue;
              unsigned char *bx = box.take();
              box_put32(bx, lane, h ? v[1] : v[0]);
              box.send(&maps.c, bx, col + 32 * h, row0, u.z, add);
            }
          }
        }
      }
    }
    if (MODE == kStats) flush();
    if (elect_one()) bulk_wait<0>();  // stores complete before the shared memory goes away
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (tid == 0 && *(volatile uint32_t *)err) atomicCAS(&g_ce_timeout, 0u, 1u);
  __syncwarp();
  cluster_barrier();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2u * kTileN));
  cluster_barrier();
}

// ---- staging ----------------------------------------------------------------
__device__ __forceinline__ bool counted(int32_t t, int vocab) { return t >= 0 && t < vocab; }

// Writes v as a 16-bit operand: itself, or the high and low float16 pieces of v * scale.
template <typename T>
__device__ __forceinline__ void put_pieces(uint16_t *dst, size_t plane, float v, float scale) {
  if constexpr (sizeof(T) == 2) {
    reinterpret_cast<T *>(dst)[0] = op_store<T>(v);
  } else {
    v *= scale;
    const __half h = __float2half_rn(v);
    reinterpret_cast<__half *>(dst)[0] = h;
    reinterpret_cast<__half *>(dst)[plane] = __float2half_rn(v - __half2float(h));
  }
}
// One row of 16-bit operands from `src` (null: zeros, one at a time), by one warp; VEC
// elements per access where the addresses allow.
template <typename T, int VEC>
__device__ __forceinline__ void put_row(uint16_t *dst, size_t plane, const T *src, int dim, int lane, float scale) {
#pragma unroll 4
  for (int c = lane * VEC; c < dim; c += 32 * VEC) {
    if constexpr (VEC == 1) {
      put_pieces<T>(dst + c, plane, src ? op_load<T>(src[c]) : 0.f, scale);
    } else if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<OpVec<T, VEC> *>(dst + c) = *reinterpret_cast<const OpVec<T, VEC> *>(src + c);
    } else {
      const float4 v = *reinterpret_cast<const float4 *>(src + c);
      const float x[4] = {v.x * scale, v.y * scale, v.z * scale, v.w * scale};
      OpVec<__half, 4> h, l;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        h.v[i] = __float2half_rn(x[i]);
        l.v[i] = __float2half_rn(x[i] - __half2float(h.v[i]));
      }
      *reinterpret_cast<OpVec<__half, 4> *>(dst + c) = h;
      *reinterpret_cast<OpVec<__half, 4> *>(dst + plane + c) = l;
    }
  }
}
template <typename T>
__device__ __forceinline__ void put_row(uint16_t *dst, size_t plane, const T *src, int dim, int lane, float scale, int vec) {
  if (vec == 1) {
    put_row<T, 1>(dst, plane, src, dim, lane, scale);
    return;
  }
  if constexpr (sizeof(T) == 2) {
    if (vec == 2) {
      put_row<T, 2>(dst, plane, src, dim, lane, scale);
      return;
    }
  }
  put_row<T, 16 / sizeof(T)>(dst, plane, src, dim, lane, scale);
}

// The power of two that brings a largest magnitude to 2^14..2^15 (as far as float32
// goes), and its inverse.
__device__ __forceinline__ void range_scale(uint32_t top, float &scale, float &inverse) {
  int k = 14 - ((int)(top >> 23) - 127);
  k = top == 0 ? 0 : min(k, 126);
  scale = __uint_as_float((uint32_t)(k + 127) << 23);
  inverse = __uint_as_float((uint32_t)(127 - k) << 23);
}

// A float32 row with infinities, for the logits: they become +-2^14 and everything finite 0,
// and the row's factor is infinite, so that z is infinite (or NaN, where the other side is 0).
__device__ __forceinline__ void put_infinite_row(uint16_t *dst, size_t plane, const float *src, int dim, int lane) {
  for (int c = lane; c < dim; c += 32) {
    const float v = src[c];
    put_pieces<float>(dst + c, plane, fabsf(v) == INFINITY ? copysignf(16384.f, v) : 0.f, 1.f);
  }
}

struct StageArgs {
  const void *x, *w, *bias;
  long x_ld, w_ld, rows;
  const int32_t *tg;
  int vocab, dim, pitch, per_cta, x_ctas;  // per_cta: rows per CTA, a multiple of 8
  int x_vec, w_vec;                        // elements per access (see row_width)
  size_t xplane, wplane;
  uint16_t *xc, *wc;                       // wc null: W is read where it is
  float *xinv, *winv;                      // float32: what the rows were divided by
  uint32_t *range;                         // float32, gradient: largest magnitudes of x and W, [2], 0 before
  uint16_t *xt, *wt;                       // and the layouts for the products with G, or null
  float *unscale;                          // and what those were divided by
  int32_t *slot;
  int *count;
  unsigned int *ticket;
  const float *lse;  // gradient only
  float *lse_c;
  int32_t *tgt;
};

// Largest finite magnitude of a float32 row, as bits (which order like the magnitudes), by one
// warp; `infinite`: it holds an infinity.
__device__ __forceinline__ uint32_t row_top(const float *p, int dim, int lane, bool vec, bool &infinite) {
  uint32_t top = 0, any = 0;
  auto take = [&](float f) {
    const uint32_t u = __float_as_uint(f) & 0x7fffffffu;
    any = max(any, u);
    if (u < 0x7f800000u) top = max(top, u);
  };
  if (vec) {
#pragma unroll 4
    for (int c = lane * 4; c < dim; c += 128) {
      const float4 f = *reinterpret_cast<const float4 *>(p + c);
      take(f.x); take(f.y); take(f.z); take(f.w);
    }
  } else {
#pragma unroll 4
    for (int c = lane; c < dim; c += 32) take(p[c]);
  }
  infinite = __reduce_max_sync(0xffffffffu, any) == 0x7f800000u;
  return __reduce_max_sync(0xffffffffu, top);
}
// Lays a float32 row out for the logits, scaled by its own largest magnitude (its second
// pass finds the row in L1), and returns that magnitude.
__device__ __forceinline__ uint32_t stage_row(uint16_t *dst, size_t plane, const float *src, int dim, int lane, int vec, float *inverse) {
  bool infinite;
  const uint32_t top = row_top(src, dim, lane, vec == 4, infinite);
  float scale, inv;
  range_scale(top, scale, inv);
  if (infinite) put_infinite_row(dst, plane, src, dim, lane);
  else put_row<float>(dst, plane, src, dim, lane, scale, vec);
  if (lane == 0) *inverse = infinite ? INFINITY : inv;
  return top;
}

// The first CTAs find the counted rows' places (each counts the targets itself: they are
// few bytes, and a scan would be one launch more), gather x there, with lse also lse and
// targets, and zero the rows behind the last up to a whole tile (one at least).  The
// others lay W out, one warp per row (16-bit rows that TMA reads in place need no copy of W,
// and 8192 rows of x take 9 us; 50257 x 512 float32: 32 us, 206 MB in and out at 6.5 TB/s).  The
// largest magnitudes are left for ce_second_kernel: of x, and of W but for rows that a bias of
// -Inf masks and that are nobody's target, since G is 0 there.
template <typename T>
__global__ void __launch_bounds__(256) ce_stage_kernel(const StageArgs a) {
  __shared__ int sh[2][8];
  __shared__ uint32_t tops[2][8];
  op_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t top[2] = {0, 0};
  auto leave_tops = [&]() {
    if (sizeof(T) == 2 || !a.range) return;
    if (lane < 2) tops[lane][warp] = lane ? top[1] : top[0];
    __syncthreads();
    if (threadIdx.x < 2) {
      uint32_t t = 0;
      for (int k = 0; k < 8; ++k) t = max(t, tops[threadIdx.x][k]);
      if (t > *const_cast<volatile uint32_t *>(a.range + threadIdx.x)) atomicMax(a.range + threadIdx.x, t);
    }
  };
  if (blockIdx.x >= a.x_ctas) {
    const long v = (long)(blockIdx.x - a.x_ctas) * 8 + warp;
    if (v < a.vocab) {
      const T *w = static_cast<const T *>(a.w) + v * a.w_ld;
      uint16_t *wc = a.wc + (size_t)v * a.pitch;
      if constexpr (sizeof(T) == 4) {
        const uint32_t t = stage_row(wc, a.wplane, w, a.dim, lane, a.w_vec, a.winv + v);
        if (!a.bias || static_cast<const float *>(a.bias)[v] != -INFINITY) top[1] = t;
      } else {
        put_row<T>(wc, a.wplane, w, a.dim, lane, 1.f, a.w_vec);
      }
    }
    leave_tops();
    return;
  }
  const long r0 = (long)blockIdx.x * a.per_cta;
  int before = 0, total = 0;
#pragma unroll 8
  for (long n = threadIdx.x; n < a.rows; n += 256) {
    const int c = counted(a.tg[n], a.vocab);
    total += c;
    if (n < r0) before += c;
  }
  before = __reduce_add_sync(0xffffffffu, before);
  total = __reduce_add_sync(0xffffffffu, total);
  if (lane == 0) {
    sh[0][warp] = before;
    sh[1][warp] = total;
  }
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    before += sh[0][w];
    total += sh[1][w];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *a.count = total;
    *a.ticket = 0;
  }
  const T *x = static_cast<const T *>(a.x);
  for (long g0 = r0; g0 < a.rows && g0 < r0 + a.per_cta; g0 += 8) {  // 8 rows at a time, one per warp
    const int32_t t = lane < 8 && g0 + lane < a.rows ? a.tg[g0 + lane] : -1;
    const bool in = counted(t, a.vocab);
    const uint32_t mask = __ballot_sync(0xffffffffu, in);
    const int at = before + __popc(mask & ((1u << lane) - 1u));
    if (warp == 0 && lane < 8 && g0 + lane < a.rows) {
      a.slot[g0 + lane] = in ? at : -1;
      if (in && a.lse) {
        a.lse_c[at] = a.lse[g0 + lane];
        a.tgt[at] = t;
      }
    }
    const int to = __shfl_sync(0xffffffffu, at, warp);
    if (mask >> warp & 1) {
      const T *src = x + (g0 + warp) * a.x_ld;
      uint16_t *xc = a.xc + (size_t)to * a.pitch;
      if constexpr (sizeof(T) == 4) {
        top[0] = max(top[0], stage_row(xc, a.xplane, src, a.dim, lane, a.x_vec, a.xinv + to));
        const int32_t target = a.tg[g0 + warp];
        if (a.bias && static_cast<const float *>(a.bias)[target] == -INFINITY) {
          bool infinite;
          top[1] = max(top[1], row_top(static_cast<const float *>(a.w) + target * a.w_ld, a.dim, lane, a.w_vec == 4, infinite));
        }
      } else {
        put_row<T>(xc, a.xplane, src, a.dim, lane, 1.f, a.x_vec);
      }
    }
    before += __popc(mask);
  }
  const long end = (long)row_tiles(total) * kTileM;
  for (long j = total + (long)blockIdx.x * 8 + warp; j < end; j += (long)a.x_ctas * 8)
    put_row<T, 1>(a.xc + (size_t)j * a.pitch, a.xplane, static_cast<const T *>(nullptr), a.dim, lane, 1.f);
  leave_tops();
}

// float32, gradient: x and W once more, each divided by one number, for the products with G;
// one warp per row (50257 x 512: as long as the first layout).
__global__ void __launch_bounds__(256) ce_second_kernel(const StageArgs a) {
  op_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float xscale, wscale, ix, iw;
  range_scale(a.range[0], xscale, ix);
  range_scale(a.range[1], wscale, iw);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.unscale[0] = ix;
    a.unscale[1] = iw;
  }
  if (blockIdx.x < a.x_ctas) {
    const long first = (long)blockIdx.x * 8 + warp, step = (long)a.x_ctas * 8;
    for (long n = first; n < a.rows; n += step) {
      const int at = a.slot[n];
      if (at >= 0)
        put_row<float>(a.xt + (size_t)at * a.pitch, a.xplane, static_cast<const float *>(a.x) + n * a.x_ld, a.dim, lane, xscale, a.x_vec);
    }
    const int total = *a.count;
    const long end = (long)row_tiles(total) * kTileM;
    for (long j = total + first; j < end; j += step)
      put_row<float, 1>(a.xt + (size_t)j * a.pitch, a.xplane, nullptr, a.dim, lane, 1.f);
    return;
  }
  const long v = (long)(blockIdx.x - a.x_ctas) * 8 + warp;
  if (v >= a.vocab) return;
  const float inv = a.winv[v];
  // a row above the range is masked and nobody's target
  put_row<float>(a.wt + (size_t)v * a.pitch, a.wplane, static_cast<const float *>(a.w) + v * a.w_ld, a.dim, lane,
                 inv > iw && inv != INFINITY ? 0.f : wscale, a.w_vec);
}

// A bias of -Inf takes an entry out whatever its product is.
__device__ __forceinline__ float add_bias(float z, float b) { return b == -INFINITY ? b : z + b; }

// ---- joins -------------------------------------------------------------------
__device__ __forceinline__ void merge2(float &m, float &s, float m2, float s2) {
  const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.f : top;
  s = s * exp2f((m - ref) * kLog2e) + s2 * exp2f((m2 - ref) * kLog2e);
  m = top;
}

struct RowsArgs {
  const void *x, *w, *bias;
  long x_ld, w_ld, rows;
  const int32_t *tg, *slot;
  const int *count;
  int dim, tiles_n, pairs, mean;
  const float2 *stats;
  float *row_loss, *lse, *loss;
  unsigned int *ticket;
};

// One warp per row: joins the pairs' partial statistics of its tile and forms its
// target's logit (8192 rows of 512: 14 us).  The CTA that finishes last adds the rows' losses in a fixed order.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) ce_rows_kernel(const RowsArgs a) {
  __shared__ float red[2 * 8 * 32];
  __shared__ bool last;
  op_begin();
  const int lane = threadIdx.x & 31;
  const long n = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const T *w = static_cast<const T *>(a.w), *bias = static_cast<const T *>(a.bias);
  const int count = *a.count;
  const int at = n < a.rows ? a.slot[n] : -1;
  if (at >= 0) {
    const long t = a.tg[n];
    const T *xr = static_cast<const T *>(a.x) + n * a.x_ld, *wr = w + t * a.w_ld;
    float dot = 0.f;
    for (int c = lane * VEC; c < a.dim; c += 32 * VEC) {
      float p[VEC], q[VEC];
      op_load_vec<T, VEC>(xr + c, p);
      op_load_vec<T, VEC>(wr + c, q);
#pragma unroll
      for (int i = 0; i < VEC; ++i) dot = fmaf(p[i], q[i], dot);
    }
    // pairs that worked on this row tile (see Units): pair of tile i = ((i + 1) pairs - 1) / total
    const long m = at / kTileM, total = (long)row_tiles(count) * a.tiles_n;
    const long p0 = ((m * a.tiles_n + 1) * a.pairs - 1) / total, p1 = ((m + 1) * a.tiles_n * a.pairs - 1) / total;
    float top = -INFINITY, sum = 0.f;
    for (long i = lane; i < 2 * (p1 - p0 + 1); i += 32) {
      const long p = p0 + i / 2;
      // fewer tiles than pairs: some had none
      if (total < a.pairs && p * total / a.pairs == (p + 1) * total / a.pairs) continue;
      const float2 v = a.stats[((size_t)(p + m) * 2 + i % 2) * kTileM + at % kTileM];
      merge2(top, sum, v.x, v.y);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      dot += __shfl_xor_sync(0xffffffffu, dot, o);
      const float m2 = __shfl_xor_sync(0xffffffffu, top, o), s2 = __shfl_xor_sync(0xffffffffu, sum, o);
      merge2(top, sum, m2, s2);
    }
    if (lane == 0) {
      const float l = logf(sum);
      if (a.lse) a.lse[n] = top + l;
      a.row_loss[n] = top - add_bias(dot, bias ? op_load<T>(bias[t]) : 0.f) + l;
    }
  } else if (n < a.rows && lane == 0) {
    a.row_loss[n] = 0.f;
    if (a.lse) a.lse[n] = 0.f;
  }
  if (!a.loss) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  BlockReducer br(red);
  float v[1] = {0.f};
#pragma unroll 8
  for (long i = threadIdx.x; i < a.rows; i += 256) v[0] += __ldcg(a.row_loss + i);
  br.sum<1>(v);
  if (threadIdx.x == 0) *a.loss = a.mean ? v[0] / fmaxf((float)count, 1.f) : v[0];
}

// ---- few rows ----------------------------------------------------------------
// Up to 8 rows (a token scored as it is generated) leave the tensor cores idle and
// make W's one pass through the SMs everything: plain float32 dot products from
// registers, without staging, 4 rows of W per warp at a time.  One token against
// 50257 x 512 bf16 takes 18.4 us this way and 30.7 us through the tiles (HBM: 7.9 us).
constexpr int kFewRows = 8, kFewThreads = 512;
constexpr size_t kFewSmem = 64 << 10;  // x as float32

struct FewArgs {
  const void *x, *w, *bias;
  long x_ld, w_ld;
  const int32_t *tg;
  int rows, dim, vocab, mean, ctas;
  float2 *part;   // [CTAs][R] (maximum, sum of e^(z - maximum))
  float *picked;  // [R] target logits
  float *row_loss, *lse, *loss;
};

template <typename T, int VEC, int R>
__global__ void __launch_bounds__(kFewThreads, R <= 2 ? 2 : 1) ce_few_kernel(const FewArgs a) {
  extern __shared__ __align__(16) float xs[];  // [R][dim rounded up to VEC]
  __shared__ float2 sh[kFewThreads / 32][R];
  constexpr int Q = 4, N = Q * R;               // rows of W at a time, sums per warp
  constexpr int kLog = R == 1 ? 2 : R == 2 ? 3 : R == 4 ? 4 : 5;  // log2(N)
  op_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kFewThreads / 32;
  const int pitch = (a.dim + VEC - 1) / VEC * VEC;
  const T *x = static_cast<const T *>(a.x), *w = static_cast<const T *>(a.w), *bias = static_cast<const T *>(a.bias);
  for (int i = threadIdx.x; i < R * pitch; i += kFewThreads) {
    const int r = i / pitch, c = i % pitch;
    xs[i] = r < a.rows && c < a.dim ? op_load<T>(x[r * a.x_ld + c]) : 0.f;
  }
  __syncthreads();
  // after the reduction every lane holds the sum of W row `q` and x row `r`
  const int idx = lane >> (5 - kLog), q = idx / R, r = idx % R;
  const int32_t tgt = r < a.rows ? a.tg[r] : -1;
  float top = -INFINITY, sum = 0.f;
  const long groups = ((long)a.vocab + Q - 1) / Q;
  for (long g = (long)blockIdx.x * warps + warp; g < groups; g += (long)gridDim.x * warps) {
    const long v0 = g * Q;
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
#pragma unroll 2
    for (int c = lane * VEC; c < a.dim; c += 32 * VEC) {
      OpVec<T, VEC> wv[Q];
#pragma unroll
      for (int i = 0; i < Q; ++i)  // behind the last row: the last row again, not used
        wv[i] = *reinterpret_cast<const OpVec<T, VEC> *>(w + min(v0 + i, (long)a.vocab - 1) * a.w_ld + c);
#pragma unroll
      for (int j = 0; j < R; ++j) {
        float xv[VEC];
        if constexpr (VEC == 1) {
          xv[0] = xs[j * pitch + c];
        } else {
#pragma unroll
          for (int e = 0; e < VEC; e += 4) {
            const float4 f = *reinterpret_cast<const float4 *>(xs + j * pitch + c + e);
            xv[e] = f.x; xv[e + 1] = f.y; xv[e + 2] = f.z; xv[e + 3] = f.w;
          }
        }
#pragma unroll
        for (int i = 0; i < Q; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[i * R + j] = fmaf(op_load<T>(wv[i].v[e]), xv[e], acc[i * R + j]);
      }
    }
    // sums over the lanes: halves of the values change hands while there are several
#pragma unroll
    for (int step = 0; step < 5; ++step) {
      const int off = 16 >> step, n = N >> step;
      if (n > 1) {
        const bool upper = lane & off;
#pragma unroll
        for (int i = 0; i < n / 2; ++i) {
          const float send = upper ? acc[i] : acc[i + n / 2], keep = upper ? acc[i + n / 2] : acc[i];
          acc[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
        }
      } else {
        acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], off);
      }
    }
    const long v = v0 + q;
    if (v < a.vocab) {
      const float z = add_bias(acc[0], bias ? op_load<T>(bias[v]) : 0.f);
      if (v == tgt) a.picked[r] = z;
      const float now = fmaxf(top, z), ref = now == -INFINITY ? 0.f : now;
      sum = sum * exp_diff(top, ref) + exp_diff(z, ref);
      top = now;
    }
  }
  // lanes of one group are copies; join over q, then over the warps
#pragma unroll
  for (int off = R << (5 - kLog); off < 32; off <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, top, off), s2 = __shfl_xor_sync(0xffffffffu, sum, off);
    merge2(top, sum, m2, s2);
  }
  if (q == 0 && (lane & ((1 << (5 - kLog)) - 1)) == 0) sh[warp][r] = make_float2(top, sum);
  __syncthreads();
  if (warp < R) {
    const float2 f = lane < warps ? sh[lane][warp] : make_float2(-INFINITY, 0.f);
    top = f.x;
    sum = f.y;
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, top, off), s2 = __shfl_xor_sync(0xffffffffu, sum, off);
      merge2(top, sum, m2, s2);
    }
    if (lane == 0) a.part[(size_t)blockIdx.x * R + warp] = make_float2(top, sum);
  }
}

// Warp r joins the CTAs' statistics of row r; then the loss, in row order.
__global__ void __launch_bounds__(32 * kFewRows) ce_few_join_kernel(const FewArgs a, int R) {
  __shared__ float rl[kFewRows];
  op_begin();
  const int lane = threadIdx.x & 31, r = threadIdx.x >> 5;
  const bool in = r < a.rows && counted(a.tg[r], a.vocab);
  float top = -INFINITY, sum = 0.f, l = 0.f, loss = 0.f;
  if (in) {
    for (int i = lane; i < a.ctas; i += 32) {
      const float2 f = a.part[(size_t)i * R + r];
      merge2(top, sum, f.x, f.y);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, top, off), s2 = __shfl_xor_sync(0xffffffffu, sum, off);
      merge2(top, sum, m2, s2);
    }
    l = logf(sum);
    loss = top - a.picked[r] + l;
    l += top;
  }
  if (lane == 0) {
    rl[r] = loss;
    if (r < a.rows) {
      if (a.lse) a.lse[r] = l;
      if (a.row_loss) a.row_loss[r] = loss;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && a.loss) {
    float s = 0.f, n = 0.f;
    for (int i = 0; i < a.rows; ++i) {
      s += rl[i];
      n += counted(a.tg[i], a.vocab) ? 1.f : 0.f;
    }
    *a.loss = a.mean ? s / fmaxf(n, 1.f) : s;
  }
}

// dx: the slabs added in order, scaled, back to the rows' places.  A CTA takes
// `per_cta` rows, 8 / per_cta warps each; BATCH slabs are in flight at a time (behind the
// last, the last again, not added).  8192 x 512 bf16: 17 us.
template <typename T, int BATCH>
__global__ void __launch_bounds__(256) ce_dx_kernel(const float *slab, size_t slab_stride, int pitch, const MmaArgs a,
                                                    const int32_t *slot, long rows, int per_cta, int vec, T *dx,
                                                    long dx_ld) {
  op_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per_row = 8 / per_cta;
  const long n = (long)blockIdx.x * per_cta + warp / per_row;
  if (n >= rows) return;
  const int at = slot[n];
  const float c = grad_scale(a.dloss, a.count, a.mean) / a.g_scale;
  const float2 fw = sizeof(T) == 4 ? halves(a.unscale[1]) : make_float2(1.f, 1.f);
  for (int i = ((warp % per_row) * 32 + lane) * 4; i < a.dim; i += per_row * 128) {
    float s[4] = {};
    if (at >= 0) {
      const int slabs = a.cover[(size_t)(at / kTileM) * a.tiles_d + i / a.bn];
      const float *p = slab + (size_t)at * pitch + i;  // whole groups of 4: the pitch has room for them
      for (int k0 = 0; k0 < slabs; k0 += BATCH) {
        float v[BATCH][4];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) op_load_vec<float, 4>(p + min(k0 + k, slabs - 1) * slab_stride, v[k]);
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          if (k0 + k >= slabs) break;
#pragma unroll
          for (int e = 0; e < 4; ++e) s[e] += v[k][e];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = at >= 0 ? s[e] * fw.x * c * fw.y : 0.f;  // 0 whatever dloss is
    T *o = dx + n * dx_ld + i;
    if (vec == 4) {
      op_store_vec<T, 4>(o, s);
    } else if (vec == 2) {
      const float lo[2] = {s[0], s[1]}, hi[2] = {s[2], s[3]};
      op_store_vec<T, 2>(o, lo);
      if (i + 2 < a.dim) op_store_vec<T, 2>(o + 2, hi);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < a.dim) o[e] = op_store<T>(s[e]);
    }
  }
}

// ---- host --------------------------------------------------------------------
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

// The loss of up to kFewRows rows whose x fits ce_few_kernel's shared memory.
bool few_rows(const aideen_linear_ce_args *a) {
  return a->rows <= kFewRows && (size_t)a->dim * kFewRows * sizeof(float) <= kFewSmem;
}
// Its grid: CTAs, and the power of two of rows that each takes.
int few_width(uint32_t rows) { return rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 4 ? 4 : 8; }
int few_ctas(uint32_t rows, int sms) { return (few_width(rows) <= 2 ? 2 : 1) * sms; }

// Everything a call lays out.  The row count on the device is only known there,
// so sizes follow from all rows.
struct Plan {
  int planes, pairs, tiles_m, tiles_n, pitch;
  long mpad;
  bool w_direct;       // TMA reads the caller's W
  size_t xplane, wplane;
  // loss
  int32_t *slot;
  int *count;
  unsigned int *ticket;
  float *unscale, *xinv, *winv;
  uint32_t *range;
  uint16_t *xc, *wc, *xt, *wt;
  float2 *stats;
  float *row_loss;
  // gradient
  float *lse_c, *slab, *db_part;
  uint8_t *cover;
  int32_t *tgt;
  uint16_t *G;
  int piece;           // columns of a piece, a multiple of 256
  int slabs, bn, tiles_d;
  long cost;
  long dpitch;
  size_t loss_bytes, grad_bytes;
};

// Vocabulary tiles of a piece.  G of a piece stays within 160 MB, but for the
// columns that dW needs to keep half of the pairs busy (a tile goes to one pair
// whole).  Among those sizes the one is taken whose launches cost least: the
// busiest pair's slices, and about 16 slices' time for each launch.  About 40 sizes are
// looked at, so that the search stays near 1 us of the caller's time.
// The products' tiles are bn columns wide: 256, or 128 where twice the tiles even out
// the load by more than they cost (a slice of 128 columns takes 0.8 of the time of one
// of 256, being nearer to what L2 can feed: 2048 x 50257 x 512 float32 1.07 ms at 256
// and 1.34 ms at 128, but 1021 x 4999 x 250 float16 45 us and 39 us).
void choose_piece(const aideen_linear_ce_args *a, Plan &p, int bn) {
  p.bn = bn;
  p.tiles_d = (int)((a->dim + bn - 1) / bn);
  const int dx_tiles = p.tiles_m ? p.tiles_m * p.tiles_d : 1;
  p.slabs = (p.pairs + dx_tiles - 1) / dx_tiles + 2;  // a run is about depth * dx_tiles / pairs long
  p.piece = kTileN;
  p.cost = 0;
  if (!p.tiles_m) return;  // no rows
  const long bytes = p.mpad * kTileN * 2 * p.planes;
  const long half = (p.pairs / 2 + p.tiles_d - 1) / p.tiles_d;
  long most = (160L << 20) / bytes;
  if (most < half) most = half;
  if (most >= p.tiles_n) most = p.tiles_n;
  const long products = p.planes == 1 ? 1 : 3, k_dim = (a->dim + kBlockK - 1) / kBlockK;
  const long k_rows = ((long)a->rows + kBlockK - 1) / kBlockK;
  auto cost = [&](long tiles) {
    const Deal d(tiles * p.tiles_d, k_rows, (long)p.tiles_m * p.tiles_d, (int)tiles * (kTileN / kBlockK), p.slabs, p.pairs);
    return (5 * ((tiles * p.tiles_m + p.pairs - 1) / p.pairs * k_dim) + (bn == 256 ? 5 : 4) * d.load) * products + 160;
  };
  long best = most, best_cost = -1;
  for (long tiles = most; tiles >= 1 && tiles * 3 >= most; tiles -= 1 + most / 64) {
    const long n = p.tiles_n / tiles, rest = p.tiles_n % tiles;
    const long c = n * cost(tiles) + (rest ? cost(rest) : 0);
    if (best_cost < 0 || c < best_cost) {
      best = tiles;
      best_cost = c;
    }
  }
  p.piece = (int)best * kTileN;
  p.cost = best_cost;
}

Plan make_plan(const aideen_linear_ce_args *a, void *ws, bool grad) {
  Plan p{};
  p.planes = a->dtype == AIDEEN_F32 ? 2 : 1;
  p.pairs = op_sm_count() / 2;
  p.tiles_m = (int)((a->rows + kTileM - 1) / kTileM);
  p.tiles_n = (int)((a->vocab + kTileN - 1) / kTileN);
  p.pitch = (int)op_round(a->dim, 8);
  p.mpad = (long)p.tiles_m * kTileM;
  p.w_direct = p.planes == 1 && a->w_ld % 8 == 0;
  p.xplane = (size_t)p.mpad * p.pitch;
  p.wplane = (size_t)a->vocab * p.pitch;
  OpCarve c(ws);
  if (!grad && few_rows(a)) {  // W is read where it is: the CTAs' statistics and the targets' logits
    const size_t n = few_width(a->rows);
    p.stats = c.take<float2>(few_ctas(a->rows, 2 * p.pairs) * n);
    p.row_loss = c.take<float>(n);
    p.loss_bytes = c.used;
    return p;
  }
  p.slot = c.take<int32_t>(a->rows);
  p.count = c.take<int>(1);
  p.ticket = c.take<unsigned int>(1);
  if (p.planes == 2) {
    p.xinv = c.take<float>(a->rows);
    p.winv = c.take<float>(a->vocab);
  }
  p.xc = c.take<uint16_t>(p.xplane * p.planes);
  p.wc = c.take<uint16_t>(p.w_direct ? 0 : p.wplane * p.planes);
  OpCarve g = c;
  p.stats = c.take<float2>((size_t)(p.pairs + p.tiles_m) * 2 * kTileM);
  p.row_loss = c.take<float>(a->rows);
  p.loss_bytes = c.used;
  if (!grad) return p;
  Plan q = p;
  choose_piece(a, p, 256);
  choose_piece(a, q, 128);
  if (q.cost < p.cost) {
    p.bn = q.bn; p.tiles_d = q.tiles_d; p.slabs = q.slabs; p.piece = q.piece;
  }
  p.dpitch = (long)op_round(a->dim, 4);
  p.xt = p.xc;
  p.wt = p.wc;
  if (p.planes == 2) {
    p.unscale = g.take<float>(2);
    p.range = g.take<uint32_t>(2);
    p.xt = g.take<uint16_t>(p.xplane * p.planes);
    p.wt = g.take<uint16_t>(p.wplane * p.planes);
  }
  p.lse_c = g.take<float>(a->rows);
  p.tgt = g.take<int32_t>(a->rows);
  p.G = g.take<uint16_t>((size_t)p.mpad * p.piece * p.planes);
  p.slab = g.take<float>((size_t)p.slabs * p.mpad * p.dpitch);
  p.db_part = g.take<float>((size_t)p.tiles_m * 8 * p.piece);
  p.cover = g.take<uint8_t>((size_t)(p.tiles_m ? p.tiles_m : 1) * p.tiles_d);
  p.grad_bytes = g.used;
  return p;
}

// Tensor map of a matrix (or its planes); strides in bytes.
bool make_map(CUtensorMap *m, CUtensorMapDataType type, const void *base, size_t e0, size_t e1, size_t e2, size_t s1,
              size_t s2, uint32_t b0, uint32_t b1) {
  EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {e0, e1, e2};
  const cuuint64_t strides[2] = {s1, s2};
  const cuuint32_t box[3] = {b0, b1, 1};
  const cuuint32_t step[3] = {1, 1, 1};
  return fn(m, type, 3, const_cast<void *>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}
constexpr auto kU16 = CU_TENSOR_MAP_DATA_TYPE_UINT16;
constexpr auto kF32 = CU_TENSOR_MAP_DATA_TYPE_FLOAT32;

// x and W as operands (one of their layouts), in boxes of 64 columns by `rows` rows.
bool map_x(CUtensorMap *m, const Plan &p, const uint16_t *x, int dim, uint32_t rows) {
  return make_map(m, kU16, x, dim, p.mpad, p.planes, (size_t)p.pitch * 2, p.xplane * 2, 64, rows);
}
bool map_w(CUtensorMap *m, const Plan &p, const uint16_t *laid_out, const aideen_linear_ce_args *g, const void *w, uint32_t rows) {
  if (p.w_direct)
    return make_map(m, kU16, w, g->dim, g->vocab, 1, (size_t)g->w_ld * 2, (size_t)g->w_ld * 2, 64, rows);
  return make_map(m, kU16, laid_out, g->dim, g->vocab, p.planes, (size_t)p.pitch * 2, p.wplane * 2, 64, rows);
}

// Elements that rows of this base and stride can be moved by: 16 bytes, a pair of 16-bit
// elements, or one.
int row_width(uint32_t dim, const void *p, int64_t ld, size_t el) {
  if (dim % (16 / el) == 0 && op_vec16(p, ld, el)) return (int)(16 / el);
  return el == 2 && dim % 2 == 0 && ld % 2 == 0 && op_aligned(p, 4) ? 2 : 1;
}

template <int MODE, typename T, bool HELD, bool DEEP>
cudaError_t launch_as(const Plan &p, const Maps &maps, MmaArgs a, cudaStream_t st) {
  const int held = HELD ? (a.dim + kBlockK - 1) / kBlockK : 0;
  const int boxes = kEpiWarps * (MODE == kStats ? 0 : HELD ? 1 : 2) * kBoxBytes;
  const int stage = HELD ? kHalfBytes : 2 * kHalfBytes;
  constexpr int fixed = smem_fixed(MODE, sizeof(T));
  a.stages = (kSmemLimit - fixed - boxes - held * kHalfBytes) / stage;
  if (a.stages > kMaxStages) a.stages = kMaxStages;
  const int smem = held * kHalfBytes + a.stages * stage + boxes + fixed;
  auto kernel = ce_mma_kernel<MODE, T, HELD, DEEP>;
  // the attribute belongs to the kernel, not to the call: always the same value, or a call
  // of another thread could lower it between here and the launch
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
  if (e != cudaSuccess) return e;
  return op_launch(kernel, 2 * p.pairs, kThreads, smem, st, maps, a);
}
template <int MODE, typename T>
cudaError_t launch_mma(const Plan &p, const Maps &maps, const MmaArgs &a, cudaStream_t st) {
  if constexpr (MODE != kProducts && sizeof(T) == 2) {
    if (a.dim <= kMaxHeld * kBlockK) return launch_as<MODE, T, true, false>(p, maps, a, st);
  }
  if constexpr (MODE != kProducts && sizeof(T) == 4) {
    if (a.dim > kChunk * kBlockK) return launch_as<MODE, T, false, true>(p, maps, a, st);
  }
  return launch_as<MODE, T, false, false>(p, maps, a, st);
}

template <typename T>
cudaError_t stage_run(const aideen_linear_ce_args *g, const Plan &p, const T *x, const T *w, const T *bias,
                      const int32_t *tg, const float *lse, bool want_dx, bool want_dw, cudaStream_t st) {
  StageArgs s{};
  s.x = x; s.w = w; s.x_ld = g->x_ld; s.w_ld = g->w_ld; s.rows = g->rows; s.tg = tg; s.vocab = (int)g->vocab;
  s.dim = (int)g->dim; s.pitch = p.pitch; s.xplane = p.xplane; s.wplane = p.wplane; s.xc = p.xc; s.wc = p.wc;
  s.slot = p.slot; s.count = p.count; s.ticket = p.ticket; s.lse = lse; s.lse_c = p.lse_c; s.tgt = p.tgt;
  s.bias = bias; s.xinv = p.xinv; s.winv = p.winv;
  s.x_vec = row_width(g->dim, x, g->x_ld, sizeof(T));
  s.w_vec = row_width(g->dim, w, g->w_ld, sizeof(T));
  const long most = 4L * 2 * p.pairs;  // CTAs
  s.per_cta = (int)(8 * ((g->rows + 8 * most - 1) / (8 * most)));
  s.x_ctas = (int)((g->rows + s.per_cta - 1) / s.per_cta);
  const unsigned w_ctas = p.w_direct ? 0 : (g->vocab + 7) / 8;
  cudaError_t e = cudaSuccess;
  if (sizeof(T) == 4 && (want_dx || want_dw)) {
    s.range = p.range; s.unscale = p.unscale; s.xt = p.xt; s.wt = p.wt;
    e = cudaMemsetAsync(p.range, 0, 2 * sizeof(uint32_t), st);
  }
  if (e == cudaSuccess) e = op_launch(ce_stage_kernel<T>, s.x_ctas + w_ctas, 256, 0, st, s);
  if (e != cudaSuccess || !s.range) return e;
  if (!want_dw) s.x_ctas = 0;
  return op_launch(ce_second_kernel, s.x_ctas + (want_dx ? w_ctas : 0), 256, 0, st, s);
}

template <typename T>
MmaArgs mma_args(const aideen_linear_ce_args *g, const Plan &p, const T *bias) {
  MmaArgs a{};
  a.count = p.count;
  a.vocab = (int)g->vocab; a.dim = (int)g->dim; a.planes = p.planes;
  const uint32_t type = g->dtype == AIDEEN_BF16 ? 1u : 0u;  // bf16 or f16 operands, f32 accumulator
  a.idesc = (1u << 4) | (type << 7) | (type << 10);
  a.bias = bias;
  a.g_scale = g->dtype == AIDEEN_F16 ? kHalfScale : g->dtype == AIDEEN_F32 ? kPieceScale : 1.f;
  a.xinv = p.xinv; a.winv = p.winv; a.unscale = p.unscale;
  a.mean = g->reduction == AIDEEN_CE_MEAN;
  return a;
}

template <typename T, int VEC>
cudaError_t few_run(FewArgs a, size_t smem, int sms, cudaStream_t st) {
  const int R = few_width(a.rows);
  auto kernel = R == 1 ? ce_few_kernel<T, VEC, 1> : R == 2 ? ce_few_kernel<T, VEC, 2> : R == 4 ? ce_few_kernel<T, VEC, 4> : ce_few_kernel<T, VEC, 8>;
  a.ctas = few_ctas(a.rows, sms);
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kFewSmem);  // as in launch_as
  if (e == cudaSuccess) e = op_launch(kernel, a.ctas, kFewThreads, smem * R, st, a);
  if (e == cudaSuccess) e = op_launch(ce_few_join_kernel, 1, 32 * kFewRows, 0, st, a, R);
  return e;
}

template <typename T>
cudaError_t loss_run(const aideen_linear_ce_args *g, const Plan &p, const T *x, const T *w, const T *bias,
                     const int32_t *tg, float *loss, float *row_loss, float *lse, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = g->dim % V == 0 && op_vec16(x, g->x_ld, sizeof(T)) && op_vec16(w, g->w_ld, sizeof(T));
  if (few_rows(g)) {
    FewArgs f{};
    f.x = x; f.w = w; f.bias = bias; f.x_ld = g->x_ld; f.w_ld = g->w_ld; f.tg = tg; f.rows = (int)g->rows;
    f.dim = (int)g->dim; f.vocab = (int)g->vocab; f.mean = g->reduction == AIDEEN_CE_MEAN;
    f.part = p.stats; f.picked = p.row_loss; f.row_loss = row_loss; f.lse = lse; f.loss = loss;
    const size_t smem = op_round(g->dim, V) * sizeof(float);
    return vec ? few_run<T, V>(f, smem, 2 * p.pairs, st) : few_run<T, 1>(f, smem, 2 * p.pairs, st);
  }
  cudaError_t e = stage_run<T>(g, p, x, w, bias, tg, nullptr, false, false, st);
  if (e != cudaSuccess) return e;
  Maps maps{};
  if (!map_x(&maps.a, p, p.xc, (int)g->dim, 128) || !map_w(&maps.b, p, p.wc, g, w, 128)) return cudaErrorInvalidValue;
  MmaArgs a = mma_args<T>(g, p, bias);
  a.tiles_n = p.tiles_n;
  a.stats = p.stats;
  e = launch_mma<kStats, T>(p, maps, a, st);
  if (e != cudaSuccess) return e;
  RowsArgs r{};
  r.x = x; r.w = w; r.bias = bias; r.x_ld = g->x_ld; r.w_ld = g->w_ld; r.rows = g->rows; r.tg = tg; r.slot = p.slot;
  r.count = p.count; r.dim = (int)g->dim; r.tiles_n = p.tiles_n; r.pairs = p.pairs; r.mean = a.mean; r.stats = p.stats;
  r.row_loss = row_loss ? row_loss : p.row_loss; r.lse = lse; r.loss = loss; r.ticket = p.ticket;
  const int wx = row_width(g->dim, x, g->x_ld, sizeof(T)), ww = row_width(g->dim, w, g->w_ld, sizeof(T));
  const int width = wx < ww ? wx : ww;
  auto rows = width == 1 ? ce_rows_kernel<T, 1> : ce_rows_kernel<T, V>;
  if constexpr (sizeof(T) == 2) {
    if (width == 2) rows = ce_rows_kernel<T, 2>;
  }
  return op_launch(rows, (g->rows + 7) / 8, 256, 0, st, r);
}

template <typename T>
cudaError_t grad_run(const aideen_linear_ce_args *g, const Plan &p, const T *x, const T *w, const T *bias,
                     const int32_t *tg, const float *lse, const float *dloss, T *dx, T *dw, T *db, cudaStream_t st) {
  cudaError_t e = stage_run<T>(g, p, x, w, bias, tg, lse, dx, dw, st);
  if (e != cudaSuccess) return e;
  const int dim = (int)g->dim;
  const size_t gplane = (size_t)p.mpad * p.piece;
  Maps lm{}, pm{};
  bool ok = map_x(&lm.a, p, p.xc, dim, 128) && map_w(&lm.b, p, p.wc, g, w, 128) &&
            make_map(&lm.c, kU16, p.G, p.piece, p.mpad, p.planes, (size_t)p.piece * 2, gplane * 2, 64, 32);
  ok = ok && make_map(&pm.a, kU16, p.G, p.piece, p.mpad, p.planes, (size_t)p.piece * 2, gplane * 2, 64, 128) &&
       map_w(&pm.b, p, p.wt, g, w, 64) &&
       make_map(&pm.a2, kU16, p.G, p.piece, p.mpad, p.planes, (size_t)p.piece * 2, gplane * 2, 64, 64) &&
       map_x(&pm.b2, p, p.xt, dim, 64) &&
       make_map(&pm.c, kF32, p.slab, dim, p.mpad, p.slabs, p.dpitch * 4, p.mpad * p.dpitch * 4, 32, 32);
  const size_t el = sizeof(T);
  const int dw_vec = !dw ? 1 : op_vec16(dw, g->dw_ld, el) ? (int)(16 / el) : row_width(g->dim, dw, g->dw_ld, el);
  if (dw_vec > 2)
    ok = ok && make_map(&pm.c2, el == 4 ? kF32 : kU16, dw, dim, g->vocab, 1, g->dw_ld * el, g->dw_ld * el,
                        128 / el, 32);
  if (!ok) return cudaErrorInvalidValue;
  MmaArgs a = mma_args<T>(g, p, bias);
  a.lse = p.lse_c; a.tgt = p.tgt; a.db_part = db ? p.db_part : nullptr;
  a.bn = p.bn; a.tiles_d = p.tiles_d; a.slabs = dx ? p.slabs : 0; a.cover = p.cover; a.want_dw = dw != nullptr;
  a.full_k = p.piece / kBlockK;
  a.dw = dw; a.db = db; a.dw_ld = g->dw_ld; a.dw_vec = dw_vec; a.dloss = dloss;
  for (int v0 = 0; v0 < (int)g->vocab; v0 += p.piece) {
    const int left = (int)g->vocab - v0, cols = left < p.piece ? (left + kTileN - 1) / kTileN * kTileN : p.piece;
    a.v0 = v0;
    a.tiles_n = cols / kTileN;
    e = launch_mma<kPiece, T>(p, lm, a, st);
    if (e != cudaSuccess) return e;
    a.piece_k = cols / kBlockK;
    a.first = v0 == 0;
    e = launch_mma<kProducts, T>(p, pm, a, st);
    if (e != cudaSuccess) return e;
  }
  if (!dx) return cudaSuccess;
  auto fits = [&](int n) { return dim % n == 0 && g->dx_ld % n == 0 && op_aligned(dx, n * el); };
  const int vec = fits(4) ? 4 : fits(2) ? 2 : 1;
  const int per_cta = g->rows >= 4096 ? 8 : 2;  // with few rows there are many slabs: more warps on each
  return op_launch(p.slabs <= 4 ? ce_dx_kernel<T, 4> : ce_dx_kernel<T, 8>, (g->rows + per_cta - 1) / per_cta, 256, 0, st,
                   p.slab, (size_t)p.mpad * p.dpitch, p.dpitch, a, p.slot, g->rows, per_cta, vec, dx, g->dx_ld);
}

template <typename T>
cudaError_t loss_typed(const aideen_linear_ce_args *g, const Plan &p, const void *x, const void *w, const void *bias,
                       const int32_t *tg, float *loss, float *row_loss, float *lse, cudaStream_t st) {
  return loss_run<T>(g, p, static_cast<const T *>(x), static_cast<const T *>(w), static_cast<const T *>(bias), tg, loss,
                     row_loss, lse, st);
}
template <typename T>
cudaError_t grad_typed(const aideen_linear_ce_args *g, const Plan &p, const void *x, const void *w, const void *bias,
                       const int32_t *tg, const float *lse, const float *dloss, void *dx, void *dw, void *db,
                       cudaStream_t st) {
  return grad_run<T>(g, p, static_cast<const T *>(x), static_cast<const T *>(w), static_cast<const T *>(bias), tg, lse,
                     dloss, static_cast<T *>(dx), static_cast<T *>(dw), static_cast<T *>(db), st);
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
  if (loss_bytes) *loss_bytes = make_plan(args, nullptr, false).loss_bytes;
  if (grad_bytes) *grad_bytes = make_plan(args, nullptr, true).grad_bytes;
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
  const Plan p = make_plan(args, workspace, false);
  OP_CHECK(!p.w_direct || op_aligned(w, 16), "linear_ce: w must be 16-byte aligned at this type and row stride");
  OP_CHECK(workspace && op_aligned(workspace, 256) && workspace_bytes >= p.loss_bytes,
           "linear_ce: workspace missing, misaligned or too small");
  if (args->dtype == AIDEEN_F32) return op_cuda(loss_typed<float>(args, p, x, w, bias, targets, loss, row_loss, lse, st));
  if (args->dtype == AIDEEN_BF16)
    return op_cuda(loss_typed<__nv_bfloat16>(args, p, x, w, bias, targets, loss, row_loss, lse, st));
  return op_cuda(loss_typed<__half>(args, p, x, w, bias, targets, loss, row_loss, lse, st));
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
  const Plan p = make_plan(args, workspace, true);
  OP_CHECK(!p.w_direct || op_aligned(w, 16), "linear_ce_grad: w must be 16-byte aligned at this type and row stride");
  OP_CHECK(workspace && op_aligned(workspace, 256) && workspace_bytes >= p.grad_bytes,
           "linear_ce_grad: workspace missing, misaligned or too small");
  if (args->dtype == AIDEEN_F32)
    return op_cuda(grad_typed<float>(args, p, x, w, bias, targets, lse, dloss, dx, dw, dbias, st));
  if (args->dtype == AIDEEN_BF16)
    return op_cuda(grad_typed<__nv_bfloat16>(args, p, x, w, bias, targets, lse, dloss, dx, dw, dbias, st));
  return op_cuda(grad_typed<__half>(args, p, x, w, bias, targets, lse, dloss, dx, dw, dbias, st));
}
