// bsattn_bwd.cu — block-sparse attention backward for sm_100a.
//
// With P = exp(scale * Q K^T - lse) over the kept 128x128 blocks (0 elsewhere),
// delta_i = sum_d dO_id O_id - dlse_i and dP = dO V^T, the gradients are
//   dV = P^T dO,   dS = P o (dP - delta),   dQ = scale dS K,   dK = scale dS^T Q.
// The probabilities are recomputed from Q, K and the row statistics of the
// forward pass; nothing of size Sq x Sk is stored.
//
// Two kinds of tiles run through one persistent kernel:
//   kind 0  one key block, over the query blocks that keep it (a mask column):
//           dK and dV stay in TMEM.   X = K Q^T (= S^T),  Y = V dO^T (= dP^T),
//           dV += P^T dO,  dK += dS^T Q          (4 products per kept block)
//   kind 1  one query block, over its kept key blocks (a mask row): dQ stays in
//           TMEM.   X = Q K^T,  Y = dO V^T,  dQ += dS K            (3 products)
// Both have the same shape: two resident 128x128 tiles A1, A2, two streamed
// tiles B1, B2 per block, X = A1 B1^T, Y = A2 B2^T, acc1 += P B2 (kind 0),
// acc2 += dS B1. The transposed S of kind 0 makes P^T and dS^T the TMEM A
// operands of their products, so neither ever passes through shared memory.
// Recomputing S and dP for dQ costs 7 products per kept block where 5 would
// do, and buys gradients that are each summed by one CTA in list order: no
// atomics, the same bits on every run, and no fp32 dQ buffer in HBM (64 KB of
// reductions per kept block).

#include <math.h>

#include "sa_common.cuh"

namespace sa {
namespace attn_bwd {

constexpr int kT = 128;            // rows of every tile; head dim
// Ring slots. B1 of a block is held from X to the block's last product, B2 not
// as long; 64 KB of resident tiles leave room for five.
constexpr int kB1 = 3, kB2 = 2;
constexpr int kGroups = 4;         // warpgroups of arithmetic
constexpr int kCols = kT / kGroups;  // columns of X and Y each of them owns
constexpr int kWorkers = kGroups * 128;
constexpr int kThreads = 128 + kWorkers;  // 4 role warps, then the workers
constexpr int kTileBytes = kT * kT * 2;
constexpr int kBoxBytes = kTileBytes / 2;      // one 64-column box
constexpr int kStatBytes = 2 * kT * 4;         // -lse (log2 units) and -delta of 128 rows
constexpr int kMaxBlocks = 1024;               // per mask row or column (S <= 131072)
constexpr int kLeastPiece = 8;                 // blocks
constexpr int kJoin = 8;                       // pieces added up at a time
constexpr int kFewTiles = 4;                   // per SM
constexpr int kListReaders = 2 + kWorkers;
constexpr uint32_t kColX = 0, kColY = 128, kColAcc1 = 256, kColAcc2 = 384;

struct Mask {
  const uint8_t* mask;
  int64_t s0, s1, s2, s3;
  const int32_t* head_mask_type;
  int heads;
  // The mask column (kind 0) or row (kind 1) blk of a head; true when the head
  // is dense, with nothing to read.
  __device__ __forceinline__ bool line(int kind, int b, int h, int blk, const uint8_t*& m,
                                       int64_t& step) const {
    int mh = h;
    if (head_mask_type != nullptr) {
      const int ty = head_mask_type[h];
      // an entry past the mask's heads has no slice to read: dense, and reported
      // by the row statistics
      if (ty <= 0 || ty > heads) return true;
      mh = ty - 1;
    }
    m = mask + b * s0 + mh * s1 + blk * (kind ? s2 : s3);
    step = kind ? s3 : s2;
    return false;
  }
};

struct Params {
  int B, H, Sq, Sk, nq, nk;
  Mask mask;
  float scale, scale_log2;
  const float* nstat;   // [B*H][nq*128][.]: first all -lse*log2(e), then all -delta
  int64_t stat_plane;   // elements of one plane
  __nv_bfloat16 *dq, *dk, *dv;
  int64_t dqs0, dqs1, dqs2, dks0, dks1, dks2, dvs0, dvs1, dvs2;
  int* next_item;
  int32_t* status;
  // Work items: where tiles may be cut, one of `count` kept blocks is cut into
  // max(1, count / least) pieces, least from the total count. Pieces 1, 2, ...
  // of the cut tiles are dealt out to the CTAs first, then every tile's piece 0
  // is taken from a counter, kind 0 before kind 1.
  int tiles[2];
  const int* counts[2];  // kept blocks of every tile; NULL where none is cut
  const int* eights;     // the same of every eight tiles: sum * 2048 + largest; by kind
  // Pieces are numbered over all cut tiles of a kind. A piece has at least
  // 1 / SMs of the kind's blocks, so there are max_extra <= SMs of the pieces
  // 1, 2, ...; with f of them before the tile's, its piece i > 0 is kept in slot
  // f + i - 1, its piece 0 in slot max_extra + f.
  int max_extra;
  float* part[2];  // [slot] fp32 sums of a piece
  int* joined[2];  // [slot][worker warp] arrivals of pieces or of groups of them
};

// A work item as the list warp publishes it: a tile, or a piece of one.
struct __align__(16) Item {
  int n;        // kept blocks; -1: no more items
  int kind, blk, h, b;
  int pieces, piece, first;  // first: slot of piece 1
  // The tile of acc 0 (dV) and 1 (dK or dQ): first row, row pitch, and the rows
  // that exist. Looked up ahead of the epilogue, where first reads of these
  // parameters took 2 us of a launch.
  __nv_bfloat16* out[2];
  int64_t pitch[2];
  int rows;
};

struct __align__(16) SmemCtl {
  // [block parity] -lse and -delta of the rows of a query block: of each block
  // of kind 0, of a kind-1 tile with its first block
  float stats[2][2 * kT];
  uint64_t b1_full[kB1], b2_full[kB2];
  uint64_t st_full[2];             // [block parity] statistics loaded, or none to load
  uint64_t a_full[2], a_empty[2];  // [0] A1, [1] A2
  uint64_t list_full[2], list_empty[2];
  uint64_t x_full[2];    // [block parity] X computed (commit)
  // kind 0: [c] half c of each warpgroup's P columns written over X; kind 1: X
  // copied out. kWorkers arrivals
  uint64_t x_done[2];
  uint64_t y_full[2];    // [block parity] Y computed (commit)
  uint64_t ds_full[2];   // [block parity] dS written over Y, kWorkers arrivals
  uint64_t acc_full;     // a tile's sums are complete (commit)
  uint64_t acc_free;     // a tile's sums have been read, kWorkers arrivals
  uint64_t claim;        // the producer has issued an item's last loads
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
  Item item[2];          // [slot]
  uint32_t kept[2][kMaxBlocks / 32];  // [slot] bit c of word i: block 32 i + c is kept
};

// The tiles need 1024-byte alignment (128-byte swizzle); dynamic shared memory
// starts on it (checked by the kernel), so no slack is reserved.
constexpr size_t kSmemBytes = (2 + kB1 + kB2) * kTileBytes + sizeof(SmemCtl);
static_assert(kSmemBytes <= 227 * 1024, "shared memory of one CTA");

// Row statistics: one 16-lane group per query row sums dO . O in fp32. Rows
// past Sq and rows without a finite log-sum-exp (no kept key) get -inf, which
// makes every P of theirs 0. Bound by reading dO and O once.
constexpr int kPrepRows = 4;  // rows of a 16-lane group, loaded together
__global__ void __launch_bounds__(256)
    row_stats_kernel(const __nv_bfloat16* dout, const __nv_bfloat16* out, int64_t ds0, int64_t ds1,
                     int64_t ds2, int64_t os0, int64_t os1, int64_t os2, const float* lse,
                     const float* dlse, int H, int Sq, int rows_pad, float* nstat, int64_t plane,
                     int* next_item, int* joined, int n_joined, int* counts0, int* counts1,
                     int* eights, const Mask mask, int B, int nk, int32_t* status) {
  release_next_kernel();  // it waits for this one's completion all the same
  // The call before may still be ending: calls in a row then take 48.0 -> 45.6 us
  // (4 heads of 4096) and 14.3 -> 12.4 us (2 heads of 300). The main kernel lets
  // nothing start early: waiting blocks in its tail cost 1 to 3%.
  wait_prior_kernel();
  const int nq = rows_pad / kT;
  const int block = blockIdx.y * gridDim.x + blockIdx.x, blocks = gridDim.x * gridDim.y;
  if (block == 0 && threadIdx.x == 0) *next_item = 0;
  if (block == 0 && mask.head_mask_type != nullptr)
    for (int i = threadIdx.x; i < H; i += 256)
      if (mask.head_mask_type[i] > mask.heads) report_status(status, SA_DEV_BAD_INDEX);
  for (int i = block * 256 + threadIdx.x; i < n_joined; i += blocks * 256) joined[i] = 0;
  // kept blocks of every tile of the kinds that may be cut, a warp per tile, and
  // of eight tiles together, as one number: sum * 2048 + largest
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ int of_warp[8];
  for (int kind = 0; kind < 2; ++kind) {
    int* counts = kind ? counts1 : counts0;
    if (counts == nullptr) continue;
    const int per_head = kind ? nq : nk, n = kind ? nk : nq, tiles = B * H * per_head;
    for (int e = block; e * 8 < tiles; e += blocks) {
      const int t = e * 8 + warp, bh = t / per_head;
      const uint8_t* m;
      int64_t step;
      int c = 0;
      if (t < tiles) {
        c = n;
        if (!mask.line(kind, bh / H, bh % H, t - bh * per_head, m, step)) {
          c = 0;
#pragma unroll 8
          for (int i = lane; i < n; i += 32) c += m[i * step] != 0;
          c = __reduce_add_sync(0xffffffffu, c);
        }
        if (lane == 0) counts[t] = c;
      }
      if (lane == 0) of_warp[warp] = c;
      __syncthreads();
      if (threadIdx.x == 0) {
        int sum = 0, most = 0;
        for (int w = 0; w < 8; ++w) {
          sum += of_warp[w];
          most = max(most, of_warp[w]);
        }
        eights[e] = sum * 2048 + most;
      }
      __syncthreads();
    }
    eights += (tiles + 7) / 8;
  }
  const int bh = blockIdx.x;
  const int h = bh % H, b = bh / H;
  const int g = threadIdx.x >> 4, l = threadIdx.x & 15;
  const int r0 = blockIdx.y * (16 * kPrepRows) + g;
  uint4 x[kPrepRows], y[kPrepRows];
  float row_lse[kPrepRows], row_dlse[kPrepRows];
#pragma unroll
  for (int i = 0; i < kPrepRows; ++i) {
    const int r = r0 + 16 * i;
    x[i] = y[i] = make_uint4(0, 0, 0, 0);
    row_lse[i] = -INFINITY;
    row_dlse[i] = 0.f;
    if (r < Sq) {
      if (l == 0) {
        row_lse[i] = lse[(int64_t)bh * Sq + r];
        if (dlse != nullptr) row_dlse[i] = dlse[(int64_t)bh * Sq + r];
      }
      x[i] = reinterpret_cast<const uint4*>(dout + b * ds0 + h * ds1 + (int64_t)r * ds2)[l];
      y[i] = __ldcs(reinterpret_cast<const uint4*>(out + b * os0 + h * os1 + (int64_t)r * os2) + l);
    }
  }
#pragma unroll
  for (int i = 0; i < kPrepRows; ++i) {
    const int r = r0 + 16 * i;
    const uint32_t* a = reinterpret_cast<const uint32_t*>(&x[i]);
    const uint32_t* c = reinterpret_cast<const uint32_t*>(&y[i]);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s = fmaf(__uint_as_float(a[e] << 16), __uint_as_float(c[e] << 16), s);
      s = fmaf(__uint_as_float(a[e] & 0xffff0000u), __uint_as_float(c[e] & 0xffff0000u), s);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (l == 0 && r < rows_pad) {
      float nl = -INFINITY, nd = 0.f;
      if (row_lse[i] != -INFINITY) {
        nl = -row_lse[i] * 1.4426950408889634f;
        nd = row_dlse[i] - s;
      }
      const int64_t o0 = (int64_t)bh * rows_pad + r;
      nstat[o0] = nl;
      nstat[plane + o0] = nd;
    }
  }
}

// This thread's part of a 128x128 fp32 accumulator: kCols columns of its row.
__device__ __forceinline__ void load_acc(uint32_t taddr, uint32_t (&o)[kCols]) {
  tmem_ld32(taddr, o);
  tmem_wait_ld();
  reg_fence32(o);
}

// Writes a warp's 32 rows x kCols columns (a row per lane, fp32 times mul) as
// bf16. dst: this warp's first row and column; rows are `pitch` elements
// apart, `rows` of them exist. Groups of four lanes first exchange 16-byte
// pieces, so that each store covers 64 contiguous bytes of 8 rows: with a row
// per lane, 16 bytes of 32 rows each, the stores of a tile took 2 to 4 us.
static_assert(kCols == 32, "four 16-byte pieces of a row per lane");
__device__ __forceinline__ void store_rows(const uint32_t (&o)[kCols], float mul,
                                           __nv_bfloat16* dst, int64_t pitch, int rows,
                                           int lane) {
  uint32_t w[4][4];  // [piece][word]
#pragma unroll
  for (int v = 0; v < 4; ++v)
#pragma unroll
    for (int u = 0; u < 4; ++u)
      w[v][u] = pack_bf16x2(__uint_as_float(o[8 * v + 2 * u]) * mul,
                            __uint_as_float(o[8 * v + 2 * u + 1]) * mul);
  // 4x4 transpose over lanes 4a..4a+3: afterwards w[i] is piece (lane & 3) of
  // row 4a + i
#pragma unroll
  for (int step = 1; step < 4; step <<= 1) {
    const bool hi = (lane & step) != 0;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      if (v & step) continue;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t give = hi ? w[v][u] : w[v + step][u];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, give, step);
        if (hi) w[v][u] = got; else w[v + step][u] = got;
      }
    }
  }
  __nv_bfloat16* d = dst + (int64_t)(lane & ~3) * pitch + (lane & 3) * 8;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if ((lane & ~3) + i < rows)
      *reinterpret_cast<uint4*>(d + i * pitch) = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
}

__device__ __forceinline__ void zero_rows(__nv_bfloat16* dst, int64_t pitch, int rows, int lane) {
  __nv_bfloat16* d = dst + (int64_t)(lane & ~3) * pitch + (lane & 3) * 8;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if ((lane & ~3) + i < rows) *reinterpret_cast<uint4*>(d + i * pitch) = make_uint4(0, 0, 0, 0);
}

// A piece's sums in fp32, 16-byte units by lane: each warp reads back only
// what the same warp of another CTA stored.
__device__ __forceinline__ void keep_part(const uint32_t (&o)[kCols], float* dst, int lane) {
#pragma unroll
  for (int v = 0; v < kCols / 4; ++v)
    __stcg(reinterpret_cast<uint4*>(dst) + v * 32 + lane,
           make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]));
}

__device__ __forceinline__ void add_part(uint32_t (&o)[kCols], const float* src, int lane) {
#pragma unroll
  for (int v = 0; v < kCols / 4; ++v) {
    const uint4 x = __ldcg(reinterpret_cast<const uint4*>(src) + v * 32 + lane);
    const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int u = 0; u < 4; ++u)
      o[4 * v + u] = __float_as_uint(__uint_as_float(o[4 * v + u]) + __uint_as_float(y[u]));
  }
}

__device__ __forceinline__ const uint32_t (&first16(const uint32_t (&r)[32]))[16] {
  return reinterpret_cast<const uint32_t(&)[16]>(r);
}

// x = hi + lo in bf16 each, two values: 16 significant bits instead of 8.
__device__ __forceinline__ void split_bf16x2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  hi = pack_bf16x2(x0, x1);
  lo = pack_bf16x2(x0 - __uint_as_float(hi << 16), x1 - __uint_as_float(hi & 0xffff0000u));
}

// P and dS enter their products as bf16, which with fp32 sums leaves an error
// like that of the bf16 results (1.4 times it together). Over a few tokens
// single roundings show, up to twice that, so FINE keeps P and dS as two bf16
// halves, each a product of its own in the columns that X and Y leave free.
// The launch takes it where the blocks do not fill the GPU once and the extra
// products hide behind latencies (300 tokens, 2 heads, in a captured graph: 11.9
// us become 13.4).
// MODE: what may happen to the tiles. Compiled apart, as code that a launch does
// not need costs it time: 2 us of 300 tokens, 2 heads (cold caches: 19.3 and 17.4
// us), 0.6% of long ones.
enum Mode {
  kPlain,  // nothing
  kFew,    // few tiles, none cut
  kCut     // tiles may be cut into pieces, and may be few
};
template <bool FINE, Mode MODE>
__global__ void __launch_bounds__(kThreads, 1)
    bsattn_bwd_kernel(const __grid_constant__ CUtensorMap tm_q,
                      const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ CUtensorMap tm_do, const Params p) {
  constexpr bool CUT = MODE == kCut;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* a_tile = smem;                       // A1, A2
  uint8_t* b1_ring = smem + 2 * kTileBytes;
  uint8_t* b2_ring = b1_ring + kB1 * kTileBytes;
  SmemCtl* ctl = reinterpret_cast<SmemCtl*>(b2_ring + kB2 * kTileBytes);

  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);  // warp-uniform
  const int lane = threadIdx.x & 31;
  if ((smem_u32(smem) & 1023u) != 0u) {
    if (threadIdx.x == 0) report_timeout(p.status);
    return;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < kB1; ++i) mbar_init(&ctl->b1_full[i], 1);
    for (int i = 0; i < kB2; ++i) mbar_init(&ctl->b2_full[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->st_full[i], 1);
      mbar_init(&ctl->a_full[i], 1);
      mbar_init(&ctl->a_empty[i], 1);
      mbar_init(&ctl->list_full[i], 1);
      mbar_init(&ctl->list_empty[i], kListReaders);
      mbar_init(&ctl->x_full[i], 1);
      mbar_init(&ctl->y_full[i], 1);
      mbar_init(&ctl->ds_full[i], kWorkers);
    }
    mbar_init(&ctl->x_done[0], kWorkers);
    mbar_init(&ctl->x_done[1], kWorkers);
    mbar_init(&ctl->acc_full, 1);
    mbar_init(&ctl->acc_free, kWorkers);
    mbar_init(&ctl->claim, 1);
    mbar_init(&ctl->drain, 1);
    ctl->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tm_q);
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
    prefetch_tensormap(&tm_do);
  }
  if (warp == 2) {
    tmem_alloc(&ctl->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  wait_prior_kernel();  // the row statistics, the item counter and the counts

  const uint32_t tmem = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);
  volatile int* abort_flag = &ctl->abort_flag;

  if (warp == 2) {
    // ---------------- work items and their kept blocks, two ahead ----------------
    int least = 0x7fffffff, extra[2] = {0, 0}, before_lane[2] = {0, 0}, span[2] = {1, 1};
    const auto extras_of = [&](int count) { return max(1, count / least) - 1; };
    if (CUT) {
      // pieces of about half an SM's share of the blocks of both kinds, 8 at least
      const int n0 = p.counts[0] != nullptr ? (p.tiles[0] + 7) / 8 : 0;
      const int n = n0 + (p.counts[1] != nullptr ? (p.tiles[1] + 7) / 8 : 0);
      int most[2] = {0, 0}, total = 0;
#pragma unroll 6
      for (int i = lane * 4; i < n; i += 128) {
        const int4 x = *reinterpret_cast<const int4*>(p.eights + i);
        const int y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = i + e < n ? y[e] : 0;
          total += c >> 11;
          if (i + e < n0) most[0] = max(most[0], c & 2047);
          else most[1] = max(most[1], c & 2047);
        }
      }
      total = __reduce_add_sync(0xffffffffu, total);
      if (n0 > 0 && n > n0) total >>= 1;  // of one kind: both have the same
      most[0] = __reduce_max_sync(0xffffffffu, most[0]);
      most[1] = __reduce_max_sync(0xffffffffu, most[1]);
      least = max(kLeastPiece, (total + (int)gridDim.x - 1) / (int)gridDim.x);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (most[q] < 2 * least) continue;
        span[q] = (p.tiles[q] + 31) >> 5;  // consecutive tiles of a lane
        int own = 0;
        for (int i = lane * span[q]; i < min(p.tiles[q], (lane + 1) * span[q]); ++i)
          own += extras_of(p.counts[q][i]);
        int sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += x;
        }
        extra[q] = __shfl_sync(0xffffffffu, sum, 31);
        before_lane[q] = sum - own;
      }
    }
    // With many tiles the next item is claimed as soon as a slot is free, which
    // hides the way from the counter to its first tiles best. With few, that
    // gives every CTA its second tile at the start; so it is claimed once the
    // loads of the one before are issued, and where tiles are counted the long
    // ones are taken first. Up to four per SM: 2 heads of 8192 tokens 60.6 -> 53.4
    // us, 24 of 1024 33.9 -> 29.2, 6 of 5000 80.0 -> 71.0, 4 of 9000 116 -> 111.5;
    // beyond: 4680 x 500 tokens 94 -> 97, 30 heads of 4096 206.7 -> 213.8.
    const int all = p.tiles[0] + p.tiles[1];
    const bool few = MODE == kFew || (CUT && all <= kFewTiles * (int)gridDim.x);
    const bool by_length = CUT && few && p.counts[0] != nullptr && p.counts[1] != nullptr;
    // With two tiles per SM and few pieces, the SMs that add a tile's pieces up are
    // the last to finish their first item, so they claim the next one, if any is
    // left, only then: 4 heads of 4096 44.0 -> 38.2 us, 3 of 4096 39.1 -> 33.7, 5 of
    // 3700 52.2 -> 48.0, one of 18000 67.2 -> 62.5; one of 8192 42.1 -> 42.9. Where
    // most items are pieces all would wait (+3%).
    const bool piece_alone = CUT && all <= 2 * (int)gridDim.x &&
                             2 * (extra[0] + extra[1]) <= (int)gridDim.x;
    bool was_piece = false;
    int dealt = blockIdx.x;  // this CTA's next extra piece
    for (int k = 0;; ++k) {
      const int slot = k & 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&ctl->list_empty[slot], ((uint32_t)(k >> 1) & 1u) ^ 1u,
                                             p.status, abort_flag)))
        break;
      if (few && k > 0 &&
          !__all_sync(0xffffffffu, mbar_wait(&ctl->claim, (uint32_t)(k - 1) & 1u, p.status,
                                             abort_flag)))
        break;
      if (piece_alone && was_piece) {
        // one lane's reading for all: other CTAs count on meanwhile
        int claimed = 0;
        if (lane == 0) claimed = *reinterpret_cast<volatile int*>(p.next_item);
        claimed = __shfl_sync(0xffffffffu, claimed, 0);
        if (claimed < (by_length ? 2 * all : all) &&
            !__all_sync(0xffffffffu,
                        mbar_wait(&ctl->list_empty[slot ^ 1], (uint32_t)((k - 1) >> 1) & 1u,
                                  p.status, abort_flag)))
          break;
      }
      Item w;
      w.n = -1;
      uint32_t word = 0;  // lane i: blocks 32 i .. 32 i + 31
      w.kind = -1;
      int tile = 0;
      w.piece = w.first = 0;
      if (CUT && dealt < extra[0] + extra[1]) {
        // which tile the dealt-out piece belongs to: first the lane, then the
        // tile among that lane's
        w.kind = dealt >= extra[0] ? 1 : 0;
        const int r = dealt - (w.kind ? extra[0] : 0);
        const int before = w.kind ? before_lane[1] : before_lane[0];
        const int* counts = w.kind ? p.counts[1] : p.counts[0];
        const int owner = 31 - __clz(__ballot_sync(0xffffffffu, before <= r));
        int first = __shfl_sync(0xffffffffu, before, owner);
        for (int t = owner * (w.kind ? span[1] : span[0]);; t += 32) {
          const int more = t + lane < p.tiles[w.kind] ? extras_of(counts[t + lane]) : 0;
          int sum = more;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
          }
          const uint32_t past = __ballot_sync(0xffffffffu, r < first + sum);
          if (past != 0u) {
            const int i = __ffs(past) - 1;
            tile = t + i;
            first += __shfl_sync(0xffffffffu, sum - more, i);
            break;
          }
          first += __shfl_sync(0xffffffffu, sum, 31);
        }
        w.piece = 1 + r - first;
        w.first = first;
        dealt += gridDim.x;
      } else {
        for (;;) {
          int it = 0;
          if (lane == 0) it = atomicAdd(p.next_item, 1);
          it = __shfl_sync(0xffffffffu, it, 0);
          if (it >= (by_length ? 2 * all : all)) break;
          const bool second = by_length && it >= all;
          if (second) it -= all;
          const int kind = it >= p.tiles[0] ? 1 : 0;
          tile = it - (kind ? p.tiles[0] : 0);
          const bool maybe_cut = (kind ? extra[1] : extra[0]) > 0;
          if (CUT && (by_length || maybe_cut)) {
            const int* counts = kind ? p.counts[1] : p.counts[0];
            const int count = counts[tile];
            if (by_length && (count >= least) == second) continue;
            if (maybe_cut && count >= 2 * least) {
              const int width = kind ? span[1] : span[0], owner = tile / width;
              int sum = 0;
              for (int i = owner * width + lane; i < tile; i += 32) sum += extras_of(counts[i]);
              w.first = __shfl_sync(0xffffffffu, kind ? before_lane[1] : before_lane[0], owner) +
                        __reduce_add_sync(0xffffffffu, sum);
            }
          }
          w.kind = kind;
          break;
        }
      }
      if (w.kind >= 0) {
        const int kind = w.kind;
        const int per_head = kind ? p.nq : p.nk;
        const int bh = tile / per_head;
        w.blk = tile - bh * per_head;
        w.b = bh / p.H;
        w.h = bh - w.b * p.H;
        const uint8_t* m = nullptr;
        int64_t step = 0;
        const bool dense = p.mask.line(kind, w.b, w.h, w.blk, m, step);
        const int n = kind ? p.nk : p.nq;
        // all mask bytes are loaded before any is used; bit i of `bits` is block
        // 32 i + lane
        const int nw = (n + 31) >> 5;
        uint32_t bits = 0;
#pragma unroll 8
        for (int i = 0; i < nw; ++i) {
          const int c = i * 32 + lane;
          const bool keep = c < n && (dense || m[c * step] != 0);
          bits |= (uint32_t)keep << i;
        }
        int count = 0;
        int before = 0;  // kept blocks in the words of lower lanes
        for (int i = 0; i < nw; ++i) {
          const uint32_t bal = __ballot_sync(0xffffffffu, (bits >> i) & 1u);
          if (lane == i) {
            word = bal;
            before = count;
          }
          count += __popc(bal);
        }
        w.pieces = 1;
        if (CUT && (kind ? extra[1] : extra[0]) > 0) w.pieces += extras_of(count);
        if (CUT && w.pieces > 1) {
          // this piece: the kept blocks number lo .. hi-1 of the tile
          const int lo = (int)((int64_t)w.piece * count / w.pieces);
          const int hi = (int)((int64_t)(w.piece + 1) * count / w.pieces);
          uint32_t rest = word;
          word = 0;
          for (int r = before; rest != 0u && r < hi; ++r) {
            const uint32_t low = rest & (0u - rest);
            rest ^= low;
            if (r >= lo) word |= low;
          }
          count = hi - lo;
        }
        was_piece = w.pieces > 1;
        w.n = count;
        const int64_t row = (int64_t)w.blk * kT;
        w.rows = (kind ? p.Sq : p.Sk) - (int)row;
        w.pitch[0] = p.dvs2;
        w.pitch[1] = kind ? p.dqs2 : p.dks2;
        w.out[0] = p.dv + w.b * p.dvs0 + w.h * p.dvs1 + row * p.dvs2;
        w.out[1] = (kind ? p.dq + w.b * p.dqs0 + w.h * p.dqs1
                         : p.dk + w.b * p.dks0 + w.h * p.dks1) +
                   row * w.pitch[1];
      }
      ctl->kept[slot][lane] = word;
      __syncwarp();
      if (lane == 0) {
        ctl->item[slot] = w;
        mbar_arrive(&ctl->list_full[slot]);
      }
      __syncwarp();
      if (w.n < 0) break;
    }
  } else if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      int J = 0, e = 0;        // blocks and tiles loaded
      int sent[4] = {0, 0, 0, 0};  // loads issued: A1, A2, B1, B2
      int kinds = 0;               // bit i: kind of the block i + 1 before this one
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok) ok = mbar_wait(bar, parity, p.status, abort_flag);
        return ok;
      };
      auto wait_x = [&](int i) { return wait(&ctl->x_full[i & 1], (uint32_t)(i >> 1) & 1u); };
      auto wait_y = [&](int i) { return wait(&ctl->y_full[i & 1], (uint32_t)(i >> 1) & 1u); };
      auto load = [&](const CUtensorMap* map, uint64_t* bar, uint8_t* dst, int blk,
                      const Item& tl) {
        mbar_arrive_expect_tx(bar, kTileBytes);
        tma_load_4d(map, bar, dst, 0, blk * kT, tl.h, tl.b);
        tma_load_4d(map, bar, dst + kBoxBytes, 64, blk * kT, tl.h, tl.b);
      };
      for (int k = 0; ok; ++k) {
        const int slot = k & 1;
        if (!wait(&ctl->list_full[slot], (uint32_t)(k >> 1) & 1u)) break;
        const Item tl = ctl->item[slot];
        const int n = tl.n;
        if (n < 0) break;
        const CUtensorMap* ma[2] = {tl.kind ? &tm_q : &tm_k, tl.kind ? &tm_do : &tm_v};
        const CUtensorMap* mb[2] = {tl.kind ? &tm_k : &tm_q, tl.kind ? &tm_v : &tm_do};
        const float* stat = p.nstat + (int64_t)(tl.b * p.H + tl.h) * p.nq * kT;
        int word = 0;
        uint32_t bits = ctl->kept[slot][0];
        for (int j = 0; j < n; ++j, ++J) {
          while (bits == 0u) bits = ctl->kept[slot][++word];  // n bits are set in all
          const int blk = word * 32 + __ffs(bits) - 1;
          bits &= bits - 1u;
          // the resident tiles are free once the previous tile's last X / Y is complete
          if (j == 0) {
            if (!wait(&ctl->a_empty[0], ((uint32_t)e & 1u) ^ 1u)) break;
            load(ma[0], &ctl->a_full[0], a_tile, tl.blk, tl);
            ++sent[0];
          }
          const int s1 = J % kB1, s2 = J % kB2;
          // A slot is free once the last product that reads it is complete. The
          // products complete in order, so a later X or Y tells: Y of J-2 follows
          // dK of J-3, X of J-1 follows dQ of J-3 and dV of J-2.
          if (J >= kB1 && !((kinds >> 2) & 1 ? wait_x(J - 1) : wait_y(J - 2))) break;
          load(mb[0], &ctl->b1_full[s1], b1_ring + s1 * kTileBytes, blk, tl);
          ++sent[2];
          if (j == 0) {
            if (!wait(&ctl->a_empty[1], ((uint32_t)e & 1u) ^ 1u)) break;
            load(ma[1], &ctl->a_full[1], a_tile + kTileBytes, tl.blk, tl);
            ++sent[1];
          }
          if (J >= kB2 && !((kinds >> 1) & 1 ? wait_y(J - 2) : wait_x(J - 1))) break;
          load(mb[1], &ctl->b2_full[s2], b2_ring + s2 * kTileBytes, blk, tl);
          ++sent[3];
          // the statistics of two blocks ago have been read once their dS is written
          if (J >= 2 && !wait(&ctl->ds_full[J & 1], (uint32_t)((J - 2) >> 1) & 1u)) break;
          if (tl.kind == 0 || j == 0) {
            const float* src = stat + (int64_t)(tl.kind ? tl.blk : blk) * kT;
            mbar_arrive_expect_tx(&ctl->st_full[J & 1], kStatBytes);
            bulk_load(ctl->stats[J & 1], src, kT * 4, &ctl->st_full[J & 1]);
            bulk_load(ctl->stats[J & 1] + kT, src + p.stat_plane, kT * 4, &ctl->st_full[J & 1]);
          } else {
            mbar_arrive(&ctl->st_full[J & 1]);
          }
          kinds = kinds << 1 | tl.kind;
        }
        if (!ok) break;
        if (n > 0) ++e;
        if (MODE != kPlain) mbar_arrive(&ctl->claim);
        mbar_arrive(&ctl->list_empty[slot]);
      }
      // no copy of this CTA may be in flight when it exits
      for (int w = 0; w < 2; ++w)
        if (sent[w] > 0) mbar_wait_drain(&ctl->a_full[w], (uint32_t)(sent[w] - 1) & 1u);
      for (int i = max(0, sent[2] - kB1); i < sent[2]; ++i)
        mbar_wait_drain(&ctl->b1_full[i % kB1], (uint32_t)(i / kB1) & 1u);
      for (int i = max(0, sent[3] - kB2); i < sent[3]; ++i)
        mbar_wait_drain(&ctl->b2_full[i % kB2], (uint32_t)(i / kB2) & 1u);
      for (int i = max(0, J - 2); i < J; ++i)
        mbar_wait_drain(&ctl->st_full[i & 1], (uint32_t)(i >> 1) & 1u);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    // The elected-thread region in warp-uniform control flow and descriptors
    // that are built once and moved by constants keep the issue short. Beside
    // two arithmetic warps that fill the scheduler, 8 MMAs of 128x128x16 (512
    // clocks of tensor core) took 791 clocks to issue this way and 1715 from a
    // `lane == 0` branch (519 and 513 alone; in isolation, all SMs).
    if (elect_one_sync()) {
      constexpr uint32_t idesc_kk = make_idesc_bf16(kT, kT, 0, 0);  // B rows are N, K-major
      constexpr uint32_t idesc_mn = make_idesc_bf16(kT, kT, 0, 1);  // B rows are K, N-major
      const uint64_t a_desc = make_sdesc_sw128(smem_u32(a_tile), 16, 1024);
      const uint64_t b1_kk = make_sdesc_sw128(smem_u32(b1_ring), 16, 1024);
      const uint64_t b2_kk = make_sdesc_sw128(smem_u32(b2_ring), 16, 1024);
      const uint64_t b1_mn = make_sdesc_sw128(smem_u32(b1_ring), kBoxBytes, 1024);
      const uint64_t b2_mn = make_sdesc_sw128(smem_u32(b2_ring), kBoxBytes, 1024);
      constexpr uint64_t kTileDesc = kTileBytes >> 4;
      int J = 0;   // blocks of earlier tiles
      int e = 0;   // earlier tiles with blocks
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok) ok = mbar_wait(bar, parity, p.status, abort_flag);
        return ok;
      };
      // D = A B^T with both tiles K-major in shared memory
      auto mma_x = [&](uint64_t a, uint64_t b, uint32_t d_col) {
        const uint32_t d = tmem + d_col;
#pragma unroll
        for (int kk = 0; kk < kT / 16; ++kk) {
          const uint64_t off = ((kk >> 2) * kBoxBytes + (kk & 3) * 32) >> 4;
          mma_ss(d, a + off, b + off, idesc_kk, kk > 0 ? 1u : 0u);
        }
      };
      // acc (+)= A . B, A = bf16 pairs in TMEM: the kCols columns of each
      // warpgroup lie packed in the first half of the columns it read. Half c:
      // the c-th half of every warpgroup's columns.
      auto mma_acc_half = [&](int c, uint32_t a_col, uint64_t b, uint32_t d_col, bool first) {
        constexpr int per = kCols / 16;  // 16-column steps of a warpgroup
        const uint32_t d = tmem + d_col, a = tmem + a_col;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int kk = (u / (per / 2)) * per + c * (per / 2) + u % (per / 2);
          mma_ts(d, a + (kk / per) * kCols + (kk % per) * 8, b + ((kk * 2048) >> 4), idesc_mn,
                 u > 0 || !first ? 1u : 0u);
          if (FINE)
            mma_ts(d, a + (kk / per) * kCols + kCols / 2 + (kk % per) * 8, b + ((kk * 2048) >> 4),
                   idesc_mn, 1u);
        }
      };
      for (int k = 0; ok; ++k) {
        const int slot = k & 1;
        if (!wait(&ctl->list_full[slot], (uint32_t)(k >> 1) & 1u)) break;
        const int n = ctl->item[slot].n, kind = ctl->item[slot].kind;
        if (n < 0) break;
        if (n > 0) {
          // kind 1 has no acc1: its columns are the second Y buffer
          auto y_col = [&](int j) { return (kind && (j & 1)) ? kColAcc1 : kColY; };
          bool acc_ready = e == 0;
          auto wait_acc = [&]() {
            if (!acc_ready) acc_ready = wait(&ctl->acc_free, (uint32_t)(e - 1) & 1u);
            return ok;
          };
          auto issue_x = [&](int j) {
            const int i = J + j;
            if (j == 0 && !wait(&ctl->a_full[0], (uint32_t)e & 1u)) return;
            if (!wait(&ctl->b1_full[i % kB1], (uint32_t)(i / kB1) & 1u)) return;
            tc_fence_after();
            mma_x(a_desc, b1_kk + (uint64_t)(i % kB1) * kTileDesc, kColX);
            mma_commit(&ctl->x_full[i & 1]);
            if (j == n - 1) mma_commit(&ctl->a_empty[0]);
          };
          auto issue_y = [&](int j) {
            const int i = J + j;
            if (j == 0 && !wait(&ctl->a_full[1], (uint32_t)e & 1u)) return;
            if (kind && j == 1 && !wait_acc()) return;
            if (!wait(&ctl->b2_full[i % kB2], (uint32_t)(i / kB2) & 1u)) return;
            tc_fence_after();
            mma_x(a_desc + kTileDesc, b2_kk + (uint64_t)(i % kB2) * kTileDesc, y_col(j));
            mma_commit(&ctl->y_full[i & 1]);
            if (j == n - 1) mma_commit(&ctl->a_empty[1]);
          };
          issue_x(0);
          issue_y(0);
          for (int j = 0; j < n && ok; ++j) {
            const int i = J + j;
            if (!kind) {
              // each half of P is used as soon as it is there
              const uint64_t b = b2_mn + (uint64_t)(i % kB2) * kTileDesc;
              if (!wait_acc() || !wait(&ctl->x_done[0], (uint32_t)i & 1u)) break;
              tc_fence_after();
              mma_acc_half(0, kColX, b, kColAcc1, j == 0);
              if (!wait(&ctl->x_done[1], (uint32_t)i & 1u)) break;
              tc_fence_after();
              mma_acc_half(1, kColX, b, kColAcc1, false);
            } else {
              if (!wait(&ctl->x_done[1], (uint32_t)i & 1u)) break;
              tc_fence_after();
            }
            if (j + 1 < n) {
              issue_x(j + 1);
              if (kind) issue_y(j + 1);
            }
            if (!wait(&ctl->ds_full[i & 1], (uint32_t)(i >> 1) & 1u)) break;
            if (!wait_acc()) break;
            tc_fence_after();
            const uint64_t b = b1_mn + (uint64_t)(i % kB1) * kTileDesc;
            mma_acc_half(0, y_col(j), b, kColAcc2, j == 0);
            mma_acc_half(1, y_col(j), b, kColAcc2, false);
            if (j + 1 < n && !kind) issue_y(j + 1);
          }
          if (!ok) break;
          mma_commit(&ctl->acc_full);
          J += n;
          ++e;
        }
        mbar_arrive(&ctl->list_empty[slot]);
      }
      mma_commit(&ctl->drain);
      mbar_wait_drain(&ctl->drain, 0);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ---------------- probabilities, dS and the outputs ----------------
    // Warpgroup g owns columns kCols g, ... of X and Y; a thread one row (TMEM
    // lane) of them. P is kept in fp32 registers from X to dS. Four warps per
    // scheduler hide each other's TMEM and barrier latencies.
    const int g = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_self = tmem + lane_off + g * kCols;
    const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
    bool ok = true;
    int J = 0, e = 0;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      // warp-uniform: the TMEM accesses that follow are warp-collective
      ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status, abort_flag));
      return ok;
    };
    for (int k = 0; ok; ++k) {
      const int slot = k & 1;
      if (!wait(&ctl->list_full[slot], (uint32_t)(k >> 1) & 1u)) break;
      const int n = ctl->item[slot].n, kind = ctl->item[slot].kind;
      if (n < 0) break;
      // this warp's part of an output
      const auto output = [&](int acc, auto&& write) {
        const Item& t = ctl->item[slot];
        const int r = (warp & 3) * 32;
        write(t.out[acc] + r * t.pitch[acc] + g * kCols, t.pitch[acc], t.rows - r);
      };
      const auto store = [&](int acc, const uint32_t(&o)[kCols]) {
        output(acc, [&](__nv_bfloat16* to, int64_t pitch, int rows) {
          store_rows(o, acc ? p.scale : 1.0f, to, pitch, rows, lane);
        });
      };
      if (n == 0) {
        for (int acc = kind; acc < 2; ++acc)
          output(acc, [&](__nv_bfloat16* to, int64_t pitch, int rows) {
            zero_rows(to, pitch, rows, lane);
          });
        mbar_arrive(&ctl->list_empty[slot]);
        continue;
      }
      // the last key block of a ragged length, if it is kept
      const bool ragged = kind && (p.Sk % kT) != 0 &&
                          ((ctl->kept[slot][(p.nk - 1) >> 5] >> ((p.nk - 1) & 31)) & 1u);
      uint64_t row_nl2 = 0ull, row_nd2 = 0ull;  // kind 1: this row's statistics
      for (int j = 0; j < n; ++j) {
        const uint32_t jp = (uint32_t)(J + j);
        uint64_t pr[kCols / 2];  // the probabilities, in pairs
        if (!wait(&ctl->st_full[jp & 1u], (jp >> 1) & 1u)) break;
        if (!kind) {
          const float* st = ctl->stats[jp & 1u];
          if (!wait(&ctl->x_full[jp & 1u], (jp >> 1) & 1u)) break;
          tc_fence_after();
          const ulonglong2* nl = reinterpret_cast<const ulonglong2*>(st + g * kCols);
          uint32_t later[16];  // FINE writes over all columns: read them first
          if (FINE) tmem_ld16(t_self + kColX + 16, later);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t r[16], pk[8], pl[8];
            if (FINE && c == 1) {
#pragma unroll
              for (int u = 0; u < 16; ++u) r[u] = later[u];
            } else {
              tmem_ld16(t_self + kColX + c * 16, r);
              tmem_wait_ld();
              reg_fence16(r);
              if (FINE) reg_fence16(later);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const ulonglong2 s2 = nl[c * 4 + (u >> 1)];
              const uint64_t x2 = f2_fma(
                  f2_pack(__uint_as_float(r[2 * u]), __uint_as_float(r[2 * u + 1])), scale2,
                  u & 1 ? s2.y : s2.x);
              float x0, x1;
              f2_unpack(x2, x0, x1);
              x0 = ex2_approx(x0);
              x1 = ex2_approx(x1);
              pr[c * 8 + u] = f2_pack(x0, x1);
              if (FINE) split_bf16x2(x0, x1, pk[u], pl[u]);
              else pk[u] = pack_bf16x2(x0, x1);
            }
            tmem_st8(t_self + kColX + c * 8, pk);
            if (FINE) tmem_st8(t_self + kColX + kCols / 2 + c * 8, pl);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&ctl->x_done[c]);
          }
          if (!wait(&ctl->y_full[jp & 1u], (jp >> 1) & 1u)) break;
          tc_fence_after();
          const ulonglong2* nd = reinterpret_cast<const ulonglong2*>(st + kT + g * kCols);
          uint32_t r[32], pk[16];
          tmem_ld32(t_self + kColY, r);
          tmem_wait_ld();
          reg_fence32(r);
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            const ulonglong2 s2 = nd[u >> 1];
            const uint64_t d2 = f2_mul(
                pr[u], f2_add(f2_pack(__uint_as_float(r[2 * u]), __uint_as_float(r[2 * u + 1])),
                              u & 1 ? s2.y : s2.x));
            float d0, d1;
            f2_unpack(d2, d0, d1);
            if (FINE) split_bf16x2(d0, d1, pk[u], r[u]);
            else pk[u] = pack_bf16x2(d0, d1);
          }
          tmem_st16(t_self + kColY, pk);
          if (FINE) tmem_st16(t_self + kColY + kCols / 2, first16(r));
        } else {
          if (j == 0) {
            const float nl = ctl->stats[jp & 1u][row], nd = ctl->stats[jp & 1u][kT + row];
            row_nl2 = f2_pack(nl, nl);
            row_nd2 = f2_pack(nd, nd);
          }
          if (!wait(&ctl->x_full[jp & 1u], (jp >> 1) & 1u)) break;
          tc_fence_after();
          uint32_t r[32], pk[16];
          tmem_ld32(t_self + kColX, r);
          tmem_wait_ld();
          reg_fence32(r);
          tc_fence_before();
          mbar_arrive(&ctl->x_done[0]);  // unused here, kept in step with kind 0
          mbar_arrive(&ctl->x_done[1]);
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            const uint64_t x2 =
                f2_fma(f2_pack(__uint_as_float(r[2 * u]), __uint_as_float(r[2 * u + 1])), scale2,
                       row_nl2);
            float x0, x1;
            f2_unpack(x2, x0, x1);
            pr[u] = f2_pack(ex2_approx(x0), ex2_approx(x1));
          }
          // keys past Sk: their K rows are 0, but exp(-lse) may overflow
          if (ragged && j == n - 1) {
            const int valid = p.Sk - (p.nk - 1) * kT - g * kCols;
#pragma unroll
            for (int u = 0; u < 16; ++u) {
              float x0, x1;
              f2_unpack(pr[u], x0, x1);
              pr[u] = f2_pack(2 * u < valid ? x0 : 0.f, 2 * u + 1 < valid ? x1 : 0.f);
            }
          }
          if (!wait(&ctl->y_full[jp & 1u], (jp >> 1) & 1u)) break;
          tc_fence_after();
          const uint32_t y = t_self + ((j & 1) ? kColAcc1 : kColY);
          tmem_ld32(y, r);
          tmem_wait_ld();
          reg_fence32(r);
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            const uint64_t d2 = f2_mul(
                pr[u], f2_add(f2_pack(__uint_as_float(r[2 * u]), __uint_as_float(r[2 * u + 1])),
                              row_nd2));
            float d0, d1;
            f2_unpack(d2, d0, d1);
            if (FINE) split_bf16x2(d0, d1, pk[u], r[u]);
            else pk[u] = pack_bf16x2(d0, d1);
          }
          tmem_st16(y, pk);
          if (FINE) tmem_st16(y + kCols / 2, first16(r));
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&ctl->ds_full[jp & 1u]);
      }
      if (!ok) break;
      if (!wait(&ctl->acc_full, (uint32_t)e & 1u)) break;
      tc_fence_after();
      uint32_t o[kCols];
      const Item& tl = ctl->item[slot];
      if (!CUT || tl.pieces == 1) {
        if (!kind) {
          load_acc(t_self + kColAcc1, o);
          store(0, o);
        }
        load_acc(t_self + kColAcc2, o);
        tc_fence_before();
        mbar_arrive(&ctl->acc_free);
        store(1, o);
      } else {
        // Every warp stores its part of the piece's sums. The warp that stores
        // the last of a group of kJoin pieces adds them up in piece order; the
        // warp that finishes the last group adds the groups' sums in order. So
        // the result does not depend on who comes last, and no warp reads more
        // than a few pieces after the other (128 pieces of one tile, added by
        // one warp per part, took 200 us).
        const int64_t size = (kind ? 1 : 2) * kT * kT;
        float* parts = p.part[kind] + (warp - 4) * 32 * kCols;
        const auto slot_of = [&](int i) {
          return i > 0 ? tl.first + i - 1 : p.max_extra + tl.first;
        };
#pragma unroll 1
        for (int acc = kind; acc < 2; ++acc) {
          load_acc(t_self + (acc ? kColAcc2 : kColAcc1), o);
          keep_part(o, parts + slot_of(tl.piece) * size + (acc - kind) * kT * kT, lane);
        }
        tc_fence_before();
        mbar_arrive(&ctl->acc_free);
        int* joined = p.joined[kind] + (warp - 4);
        const int group = tl.piece / kJoin * kJoin;  // its first piece
        int from = group, step = 1, n_parts = min(kJoin, tl.pieces - group);
        // arrivals: of a group at its first piece's slot, of the groups at
        // piece 1's, which begins no group
        int at = slot_of(group);
#pragma unroll 1
        for (bool last = tl.pieces <= kJoin;; last = true) {
          __threadfence();
          __syncwarp();
          int done = 0;
          if (lane == 0) done = atomicAdd(joined + at * (kWorkers / 32), 1) + 1;
          done = __shfl_sync(0xffffffffu, done, 0);
          if (done != n_parts) break;
          __threadfence();
#pragma unroll 1
          for (int acc = kind; acc < 2; ++acc) {
            float* of_acc = parts + (acc - kind) * kT * kT;
#pragma unroll
            for (int v = 0; v < kCols; ++v) o[v] = 0u;
            for (int i = 0; i < n_parts; ++i)
              add_part(o, of_acc + slot_of(from + i * step) * size, lane);
            if (last) store(acc, o);
            else keep_part(o, of_acc + slot_of(group) * size, lane);
          }
          if (last) break;
          from = 0;
          step = kJoin;
          n_parts = (tl.pieces + kJoin - 1) / kJoin;
          at = slot_of(1);
        }
      }
      J += n;
      ++e;
      mbar_arrive(&ctl->list_empty[slot]);
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, 512);
}

}  // namespace attn_bwd
}  // namespace sa

namespace {

// Which kinds of tiles may be cut, and where everything lies in the workspace.
// Few tiles do not fill the GPU, and among more of them a long one (a key block
// that every query keeps) holds one SM after the others are done: one head of
// 65536 tokens, a twentieth of its blocks kept, takes 800 us without cutting
// and 304 with it. With 16 tiles per SM and a sixteenth of the blocks kept a full
// line is within an SM's share, and the counting is saved.
struct Layout {
  int tiles[2], max_extra, n_joined, n_eights;
  bool cut[2];
  size_t counts[2], eights, joined[2], stats, part[2], bytes;
};

Layout layout_of(int B, int H, int Sq, int Sk, int sms) {
  using namespace sa::attn_bwd;
  Layout l;
  const int64_t bh = (int64_t)B * H;
  const int n[2] = {(Sk + kT - 1) / kT, (Sq + kT - 1) / kT};  // tiles of a head; the other's blocks
  size_t at = 256;
  auto take = [&](bool needed, size_t bytes) {
    const size_t o = at;
    if (needed) at += (bytes + 255) / 256 * 256;
    return o;
  };
  const int64_t pieces = (int64_t)n[0] * n[1] * bh / kLeastPiece;
  l.max_extra = pieces < sms ? (int)pieces : sms;
  l.n_joined = l.n_eights = 0;
  for (int k = 0; k < 2; ++k) {
    l.tiles[k] = (int)(n[k] * bh);
    l.cut[k] = n[k] * bh < 16 * sms && n[1 - k] >= 2 * kLeastPiece;
    l.joined[k] = 256 + l.n_joined * sizeof(int);
    if (l.cut[k]) l.n_joined += 2 * l.max_extra * (kWorkers / 32);
  }
  take(true, l.n_joined * sizeof(int));
  for (int k = 0; k < 2; ++k) l.counts[k] = take(l.cut[k], l.tiles[k] * sizeof(int));
  for (int k = 0; k < 2; ++k) l.n_eights += l.cut[k] ? (l.tiles[k] + 7) / 8 : 0;
  l.eights = take(true, l.n_eights * sizeof(int));
  l.stats = take(true, 2 * sizeof(float) * bh * n[1] * kT);
  for (int k = 0; k < 2; ++k)
    l.part[k] = take(l.cut[k], (size_t)2 * l.max_extra * (2 - k) * kT * kT * 4);
  l.bytes = at;
  return l;
}

}  // namespace

extern "C" size_t sa_bsattn_bwd_workspace_size(int B, int H, int Sq, int Sk) {
  using namespace sa::attn_bwd;
  if (B < 1 || H < 1 || Sq < 1 || Sk < 1 || Sq > kMaxBlocks * kT || Sk > kMaxBlocks * kT ||
      (int64_t)B * H > 65535)
    return 0;
  return layout_of(B, H, Sq, Sk, sa::sm_count_current_device()).bytes;
}

extern "C" int sa_bsattn_bwd(const void* dout, const void* q, const void* k, const void* v,
                             const void* out, const int64_t do_strides[4],
                             const int64_t q_strides[4], const int64_t k_strides[4],
                             const int64_t v_strides[4], const int64_t o_strides[4],
                             const float* lse, const float* dlse, int B, int H, int Sq, int Sk,
                             int D, const uint8_t* block_mask, const int64_t m_strides[4], int Hm,
                             const int32_t* head_mask_type, float softmax_scale, void* dq,
                             void* dk, void* dv, const int64_t dq_strides[4],
                             const int64_t dk_strides[4], const int64_t dv_strides[4],
                             void* workspace, size_t ws_bytes, int32_t* status,
                             cudaStream_t stream) {
  using namespace sa::attn_bwd;
  const char* fn = "sa_bsattn_bwd";
  SA_CHECK_ARG(dout && q && k && v && out && lse && block_mask && dq && dk && dv,
               "%s: null tensor pointer", fn);
  SA_CHECK_ARG(do_strides && q_strides && k_strides && v_strides && o_strides && m_strides &&
                   dq_strides && dk_strides && dv_strides,
               "%s: null stride array", fn);
  SA_CHECK_ARG(D == kT, "%s: head dim must be 128, got %d", fn, D);
  SA_CHECK_ARG(B >= 1 && H >= 1 && Sq >= 1 && Sk >= 1,
               "%s: B, H, Sq, Sk must be >= 1 (got %d, %d, %d, %d)", fn, B, H, Sq, Sk);
  SA_CHECK_ARG(Sq <= kMaxBlocks * kT && Sk <= kMaxBlocks * kT,
               "%s: Sq, Sk must be at most %d (got %d, %d)", fn, kMaxBlocks * kT, Sq, Sk);
  const int nq = (Sq + kT - 1) / kT, nk = (Sk + kT - 1) / kT;
  SA_CHECK_ARG((int64_t)B * H <= 65535 && (int64_t)(nq + nk) * H * B <= 0x40000000,
               "%s: too many heads or tiles (B %d, H %d)", fn, B, H);
  const int64_t* all[] = {do_strides, q_strides,  k_strides,  v_strides,
                          o_strides,  dq_strides, dk_strides, dv_strides};
  for (const int64_t* st : all)
    SA_CHECK_ARG(sa::strides16_ok(st),
                 "%s: tensors need stride(dim)=1 and other strides multiple of 8 elements "
                 "(16 bytes)", fn);
  SA_CHECK_ARG(((uintptr_t)dout | (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out |
                (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) % 16 == 0,
               "%s: tensor base pointers must be 16-byte aligned", fn);
  SA_CHECK_ARG(Hm >= 1 && (head_mask_type != nullptr || Hm == H),
               "%s: mask has %d heads but H=%d and no head_mask_type", fn, Hm, H);
  const int sms = sa::sm_count_current_device();
  const Layout l = layout_of(B, H, Sq, Sk, sms);
  SA_CHECK_ARG(workspace != nullptr && ws_bytes >= l.bytes && (uintptr_t)workspace % 256 == 0,
               "%s: workspace of %zu bytes, 256-byte aligned, needed (got %zu)", fn, l.bytes,
               ws_bytes);
  CUtensorMap tq, tk, tv, td;
  int rc;
  if ((rc = sa::tile_map_bhsd(&tq, q, q_strides, B, H, Sq, D)) != SA_OK) return rc;
  if ((rc = sa::tile_map_bhsd(&tk, k, k_strides, B, H, Sk, D)) != SA_OK) return rc;
  if ((rc = sa::tile_map_bhsd(&tv, v, v_strides, B, H, Sk, D)) != SA_OK) return rc;
  if ((rc = sa::tile_map_bhsd(&td, dout, do_strides, B, H, Sq, D)) != SA_OK) return rc;

  Params p;
  p.B = B; p.H = H; p.Sq = Sq; p.Sk = Sk; p.nq = nq; p.nk = nk;
  p.mask = sa::attn_bwd::Mask{block_mask, m_strides[0], m_strides[1], m_strides[2], m_strides[3],
                              head_mask_type, Hm};
  p.scale = softmax_scale > 0.f ? softmax_scale : 1.0f / sqrtf((float)D);
  p.scale_log2 = p.scale * 1.4426950408889634f;
  char* ws = static_cast<char*>(workspace);
  float* nstat = reinterpret_cast<float*>(ws + l.stats);
  p.nstat = nstat;
  p.stat_plane = (int64_t)B * H * nq * kT;
  p.dq = static_cast<__nv_bfloat16*>(dq);
  p.dk = static_cast<__nv_bfloat16*>(dk);
  p.dv = static_cast<__nv_bfloat16*>(dv);
  p.dqs0 = dq_strides[0]; p.dqs1 = dq_strides[1]; p.dqs2 = dq_strides[2];
  p.dks0 = dk_strides[0]; p.dks1 = dk_strides[1]; p.dks2 = dk_strides[2];
  p.dvs0 = dv_strides[0]; p.dvs1 = dv_strides[1]; p.dvs2 = dv_strides[2];
  p.next_item = static_cast<int*>(workspace);
  p.status = status;
  int* counts[2];
  for (int k = 0; k < 2; ++k) {
    p.tiles[k] = l.tiles[k];
    p.counts[k] = counts[k] = l.cut[k] ? reinterpret_cast<int*>(ws + l.counts[k]) : nullptr;
    p.joined[k] = reinterpret_cast<int*>(ws + l.joined[k]);
    p.part[k] = reinterpret_cast<float*>(ws + l.part[k]);
  }
  const bool cut = l.cut[0] || l.cut[1];
  int* eights = reinterpret_cast<int*>(ws + l.eights);
  p.eights = eights;
  p.max_extra = l.max_extra;

  const bool fine = (int64_t)nq * nk * B * H <= sms;
  const int64_t tiles = (int64_t)p.tiles[0] + p.tiles[1];
  const bool few = tiles > sms && tiles <= kFewTiles * sms;
  const auto kernel = fine ? cut ? bsattn_bwd_kernel<true, kCut> : bsattn_bwd_kernel<true, kPlain>
                      : cut ? bsattn_bwd_kernel<false, kCut>
                      : few ? bsattn_bwd_kernel<false, kFew> : bsattn_bwd_kernel<false, kPlain>;
  if ((rc = sa::func_attr_once((const void*)kernel,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes)) !=
      SA_OK)
    return rc;
  // heads run fastest: with the heads of a token side by side in memory, blocks
  // that run together then read it in order; at least a block for eight counted tiles
  const int64_t chunks = (nq * kT + 16 * kPrepRows - 1) / (16 * kPrepRows);
  const int64_t counting = (l.n_eights + (int64_t)B * H - 1) / ((int64_t)B * H);
  const dim3 pg((unsigned)(B * H), (unsigned)(chunks > counting ? chunks : counting));
  SA_CUDA_TRY(sa::launch_after(
      row_stats_kernel, pg, dim3(256), 0, stream, static_cast<const __nv_bfloat16*>(dout),
      static_cast<const __nv_bfloat16*>(out),
      do_strides[0], do_strides[1], do_strides[2], o_strides[0], o_strides[1], o_strides[2], lse,
      dlse, H, Sq, nq * kT, nstat, p.stat_plane, p.next_item, p.joined[0], l.n_joined,
      counts[0], counts[1], eights, p.mask, B, nk, status));
  // one CTA per SM; fewer only where there are fewer tiles and none may be cut
  SA_CUDA_TRY(sa::launch_after(kernel, dim3((unsigned)(cut || tiles > sms ? sms : tiles)),
                               dim3(kThreads), kSmemBytes, stream, tq, tk, tv, td, p));
  return SA_OK;
}
