// Linear layer and softmax cross entropy in pieces of the vocabulary, and the gradients.
//
//   z = h W^T,  lse_i = log sum_v exp z_iv,  loss_i = lse_i - z_i,y_i
//   dz_iv = c_i (exp(z_iv - lse_i) - [v = y_i]),  dh = dz W,  dW = dz^T h
//
// Four products on the tensor cores, one persistent kernel for all (product_kernel):
//   stats     tiles of z, reduced in registers to a maximum, a sum and the target's logit
//   dz        a piece of z again, turned into dz and written in 16 bits
//   products  dh += dz W and dW = dz^T h of that piece, in one launch: their tiles fill the
//             SMs' last round together
// The piece of dz is the only thing of the size tokens x vocabulary that ever exists, and it
// is bounded: kPieceBytes, or kLeastColumns of every token where those are more.  Making z twice
// costs a quarter of the whole step's products.
//
// Only tokens with a target take part: pack_rows_kernel moves their rows to the front (in order)
// and the others behind them as zeros, so an ignored token costs nothing and whatever its
// row holds reaches no gradient.  It also gives every row the alignment that TMA needs.
//
// Bits.  bfloat16: the sums of a product stay in the tensor cores over all of K, in 32 bits, but
// their adder truncates: each 16 of K drop up to 2^-23 of the sum so far, and logits come out a little
// small (the losses of 4096 x 32768 x 1024 and 8192 x 131072 x 2048 are off by 3.3e-7 and 5.6e-7 of
// themselves, by 2e-8 and less with products in float32).  The operands' own rounding is 2^-9.
// dz is rounded to bfloat16 for its two products, whose operands have one type: the rounding
// differs from element to element and the sums average it, so gradients move by 3 to 6.4e-4, and
// their error against 64 bits stays what their own rounding to bfloat16 makes it (1.67e-3, against
// 1.66e-3 with dz in 32 bits).  More bits would be a second part of dz, and twice the products.
//
// float32: a value is the exact sum of three bfloat16 parts, and the six products of parts
// that matter (the rest is below 2^-22 of |a||b|) go into one accumulator.
#include <algorithm>

#include "ops_common.cuh"
#include "ops_umma.cuh"

namespace purin {
namespace ops {
namespace {

using namespace umma;

constexpr int kRows = 128;      // rows of a CTA's tile
constexpr int kDepth = 64;      // K per stage: one 128-byte row
constexpr int kGroupRows = 4096;      // rows whose tiles run together (their share of h stays in L2)
// Piece of dz: smaller ones fit L2 better but make dh's sums be read and written more often
// (backward of 8192 x 131072 x 2048: 64 MB 11.0 ms, 128 MB 10.4, 256 MB 10.2, 512 MB 10.15).
constexpr size_t kPieceBytes = size_t(256) << 20;
constexpr int64_t kLeastColumns = 1024;  // of a piece, more bytes or not: 131072 tokens and up in bfloat16
constexpr size_t kStatsBytes = size_t(256) << 20;
constexpr float kLog2E = 1.4426950408889634f;

enum Mode { kStats, kDz, kProducts };

struct Targets {
  const void* p;
  bool is_64bit;
  int64_t vocab, ignore;
  __device__ __forceinline__ int32_t operator[](int64_t i) const {  // -1: no target
    const int64_t y = is_64bit ? static_cast<const int64_t*>(p)[i]
                               : int64_t(static_cast<const int32_t*>(p)[i]);
    return y >= 0 && y < vocab && y != ignore ? int32_t(y) : -1;
  }
};

// What the epilogue knows of a packed row.
struct Row {
  float top, inverse;  // the row's softmax is exp2(z log2 e - top) * inverse
  float scale;         // cotangent of the row's loss, 1 if all rows have the same one
  int32_t target;
};

struct Product {
  // stats, dz: [0] hidden, [1] weight.  products: [0], [1] dz and weight for dh, [2], [3] dz
  // and hidden for dW.
  CUtensorMap map[4];
  int32_t tokens, dim;
  int32_t begin, length;  // the vocabulary's piece
  int32_t tiles_at_once;  // stats: column tiles reduced to one partial result
  int32_t pitch;          // of a row of dz
  int32_t splits, split_blocks;  // dh: parts of the piece's K that are summed apart, K blocks of each
  int32_t want_hidden, want_weight, first;
  int32_t sum_pitch;
  int32_t columns;        // products: columns of a tile, a multiple of 64
  int32_t weight_sectors; // rows of grad_weight start at multiples of 32 bytes
  const int32_t* valid;   // rows with a target (null: all `tokens` rows take part, as given)
  const Row* row;
  Targets targets;        // of rows that are not packed
  float2* stats;          // (maximum, sum) [group of column tiles][half][token]
  float* at_target;
  __nv_bfloat16* dz;      // [part][token][pitch]
  float* sum;             // dh [split][token][sum_pitch]
  void* grad_weight;
  // The cotangent that all rows share (null: none): it multiplies the gradients in 32 bits,
  // since in dz its rounding to 16 bits would be the same relative error everywhere.
  const float* cotangent;
  const float* divisor;
  int32_t* error;
};

__device__ __forceinline__ float shared_scale(const float* cotangent, const float* divisor) {
  return cotangent ? *cotangent / (divisor ? *divisor : 1.f) : 1.f;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Item {
  int m0, n0, tiles;  // first row and column; column tiles in a row
  int k0, k1;         // K blocks
  int split, group;
  bool weight;        // products: dW instead of dh
};

template <int kGroup, Mode kMode, int kColumns>
struct Schedule {
  const Product& p;
  int valid, row_tiles, column_tiles, column_groups, dim_tiles, hidden_items, k_blocks;
  __device__ explicit Schedule(const Product& product) : p(product) {
    constexpr int kTileRows = kRows * kGroup;
    valid = p.valid ? *p.valid : p.tokens;
    row_tiles = (valid + kTileRows - 1) / kTileRows;
    dim_tiles = kMode == kProducts ? (p.dim + p.columns - 1) / p.columns : 0;
    column_tiles = (p.length + kColumns - 1) / kColumns;
    column_groups = kMode == kStats ? (column_tiles + p.tiles_at_once - 1) / p.tiles_at_once : column_tiles;
    k_blocks = ((kMode == kProducts ? p.length : p.dim) + kDepth - 1) / kDepth;
    hidden_items = kMode == kProducts && p.want_hidden ? row_tiles * dim_tiles * p.splits : 0;
  }
  // Item of step t of a worker (a CTA or pair), -1 behind its last one.  Items of one kind go
  // round the workers.  The products' two kinds differ in length by K: the longer ones go
  // round first, then the workers that got one less make up for it with shorter ones, then
  // the rest goes round.  (8192 x 131072 x 2048: 14.0 of 13.8 rounds, without it 15.)
  __device__ __forceinline__ int64_t nth(int64_t worker, int64_t workers, int64_t t) const {
    if (kMode != kProducts) {
      const int64_t i = worker + t * workers;
      return i < int64_t(row_tiles) * column_groups ? i : -1;
    }
    const int64_t weight_items =
        p.want_weight ? int64_t((p.length + kRows * kGroup - 1) / (kRows * kGroup)) * dim_tiles : 0;
    const int64_t hidden_k = p.split_blocks, weight_k = (valid + kDepth - 1) / kDepth;
    const bool hidden_first = hidden_k >= weight_k;
    const int64_t longer = hidden_first ? hidden_items : weight_items;
    const int64_t shorter = hidden_first ? weight_items : hidden_items;
    const int64_t long_start = hidden_first ? 0 : hidden_items, short_start = hidden_first ? hidden_items : 0;
    const int64_t each = longer / workers, extra = longer - each * workers;
    const int64_t mine = each + (worker < extra);
    if (t < mine) return long_start + worker + t * workers;
    t -= mine;
    const int64_t low = hidden_first ? weight_k : hidden_k, high = hidden_first ? hidden_k : weight_k;
    const int64_t ratio = extra && low ? (high + low / 2) / low : 0;
    int64_t j;
    if (worker >= extra && t < ratio) {
      j = worker - extra + t * (workers - extra);
    } else {
      if (worker >= extra) t -= ratio;
      j = (workers - extra) * ratio + worker + t * workers;
    }
    return j < shorter ? short_start + j : -1;
  }
  __device__ __forceinline__ Item item(int64_t i) const {
    constexpr int kTileRows = kRows * kGroup;
    Item it;
    it.tiles = 1;
    it.split = it.group = 0;
    it.weight = false;
    if (kMode != kProducts) {
      // Rows fastest within a group of rows, so that a weight tile is read by its rows' CTAs
      // at about the same time.
      constexpr int kGroupTiles = kGroupRows / kTileRows;
      const int64_t per_group = int64_t(kGroupTiles) * column_groups;
      const int g = int(i / per_group);
      const int64_t in = i - g * per_group;
      const int tiles = min(kGroupTiles, row_tiles - g * kGroupTiles);
      it.m0 = (g * kGroupTiles + int(in % tiles)) * kTileRows;
      it.group = int(in / tiles);
      const int first = kMode == kStats ? it.group * p.tiles_at_once : it.group;
      it.n0 = first * kColumns;
      if (kMode == kStats) it.tiles = min(p.tiles_at_once, column_tiles - first);
      it.k0 = 0;
      it.k1 = k_blocks;
    } else if (i < hidden_items) {
      const int d = int(i % dim_tiles), rest = int(i / dim_tiles);
      it.m0 = rest % row_tiles * kTileRows;
      it.n0 = d * p.columns;
      it.split = rest / row_tiles;
      it.k0 = min(it.split * p.split_blocks, k_blocks);
      it.k1 = min(it.k0 + p.split_blocks, k_blocks);
    } else {
      const int64_t j = i - hidden_items;
      it.weight = true;
      it.m0 = int(j / dim_tiles) * kTileRows;
      it.n0 = int(j % dim_tiles) * p.columns;
      it.k0 = 0;
      it.k1 = (valid + kDepth - 1) / kDepth;
    }
    return it;
  }
};

// Parts of product q of a K block: 02, 20, 11, 01, 10, 00, small ones first: the adder of the
// tensor cores truncates, by less while the sum is small.
__host__ __device__ constexpr int part_a(int q) { return (0x010120 >> (4 * q)) & 15; }
__host__ __device__ constexpr int part_b(int q) { return (0x001102 >> (4 * q)) & 15; }

__device__ __forceinline__ void split_parts(float x, __nv_bfloat16 (&part)[3]) {
  part[0] = __float2bfloat16_rz(x);  // towards zero: a large finite value stays finite
  const float first = __bfloat162float(part[0]);
  const float rest = isfinite(first) ? x - first : 0.f;
  part[1] = __float2bfloat16_rn(rest);
  part[2] = __float2bfloat16_rn(rest - __bfloat162float(part[1]));
}

// 32 bytes of a row: 8 values of 32 bits, or 16 rounded to bfloat16.
__device__ __forceinline__ void store_row(float* to, const float* v) {
  uint32_t r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = __float_as_uint(v[j]);
  store32(to, r);
}
__device__ __forceinline__ void store_row(__nv_bfloat16* to, const float* v) {
  uint32_t r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const __nv_bfloat162 q = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
    r[j] = reinterpret_cast<const uint32_t&>(q);
  }
  store32(to, r);
}

// float32 sums leave the tensor cores after every K block and are added up in registers,
// rounded to nearest: the tensor cores' adder truncates, which over a long K shows in 32
// bits.  A thread holds half a row of the tile.  (4096 x 16384 x 1024: 2.16 ms forward and
// backward, 2.6 with tiles of 128 columns, whose operands the products read twice as often.)
template <typename T, int kGroup>
struct Shape {
  // float32 on a single CTA: half the columns, so that two stages fit.
  static constexpr int kColumns = sizeof(T) == 4 && kGroup == 1 ? 128 : 256;
  static constexpr bool kAddUp = sizeof(T) == 4;
  static constexpr int kParts = sizeof(T) == 2 ? 1 : 3, kProductsOfParts = kParts == 1 ? 1 : 6;
  static constexpr int kABytes = kRows * kDepth * 2;
  static constexpr int kBBytes = kColumns / kGroup * kDepth * 2;
  // A stage holds a K block; of float32 its three parts, loaded once for six products, each
  // with barriers of its own: the last part is free again after two of the products.
  static constexpr int kPartBytes = kABytes + kBBytes;
  static constexpr int kStageBytes = kParts * kPartBytes;
  static constexpr int kStages = 196608 / kStageBytes;
  // TMA warp, MMA warp and the epilogue's: one for each quarter of the rows (a warp reads only
  // its quarter of tensor memory), or two with half of the columns each, where a thread holds
  // its sums.
  static constexpr int kHalves = kAddUp && kColumns == 256 ? 2 : 1;
  static constexpr int kEpilogueWarps = 4 * kHalves, kThreads = 64 + 32 * kEpilogueWarps;
  static constexpr int kSharedBytes = kStages * kStageBytes + 1024;
};

// T: element type of hidden, weight and their gradients.
template <typename T, int kGroup, Mode kMode>
__global__ void __launch_bounds__(Shape<T, kGroup>::kThreads, 1)
product_kernel(const __grid_constant__ Product p) {
  using S = Shape<T, kGroup>;
  constexpr int kStages = S::kStages, kColumns = S::kColumns, kHalves = S::kHalves;
  extern __shared__ uint8_t raw[];
  constexpr int kRing = kStages * S::kParts;
  __shared__ uint64_t full[kRing], empty[kRing], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_place;
  __shared__ float turned[kMode == kProducts ? S::kEpilogueWarps : 1][32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Without pack_rows_kernel nobody else has cleared the flag (it is raised only after a wait of
  // kWaitNs) and the ticket behind it.
  if (kMode == kStats && !p.row && blockIdx.x == 0 && threadIdx.x == 0) p.error[0] = p.error[1] = 0;
  const uint32_t rank = kGroup == 2 ? cta_rank() : 0;
  const uint32_t stages = (shared_address(raw) + 1023) & ~1023u;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kRing; ++s) {
      barrier_init(shared_address(&full[s]), 1);
      barrier_init(shared_address(&empty[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      barrier_init(shared_address(&acc_full[s]), 1);
      barrier_init(shared_address(&acc_empty[s]), S::kEpilogueWarps * kGroup);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    for (int i = 0; i < (kMode == kProducts ? 4 : 2); ++i) prefetch_map(&p.map[i]);
  }
  if (warp == 1) tmem_alloc<kGroup>(shared_address(&tmem_place), 512);
  fence_before();
  __syncthreads();
  if constexpr (kGroup == 2) cluster_sync();
  fence_after();
  const uint32_t tmem = tmem_place;
  wait_for_previous();
  let_next_start();

  const Schedule<kGroup, kMode, kColumns> schedule(p);
  const int columns = kMode == kProducts ? p.columns : kColumns;
  const int64_t worker = blockIdx.x / kGroup, workers = gridDim.x / kGroup;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int64_t issued = 0;
      for (int64_t t = 0, i; ok && (i = schedule.nth(worker, workers, t)) >= 0; ++t) {
        const Item it = schedule.item(i);
        const CUtensorMap* map_a = &p.map[it.weight ? 2 : 0];
        const CUtensorMap* map_b = &p.map[it.weight ? 3 : 1];
        const int a_row = it.m0 + int(rank) * kRows;
        for (int tile = 0; ok && tile < it.tiles; ++tile) {
          const int b_row = it.n0 + tile * kColumns + int(rank) * (columns / kGroup);
          for (int k = it.k0; k < it.k1; ++k) {
            const int x = k * kDepth, y = it.weight ? x : p.begin + x;
#pragma unroll
            for (int j = 0; j < S::kParts; ++j) {
              const int z = (S::kParts - j) % S::kParts;  // 0, 2, 1: as the products take them
              const int slot = stage * S::kParts + z;
              if (!(ok = barrier_wait(shared_address(&empty[slot]), phase ^ 1))) break;
              const uint32_t own = shared_address(&full[slot]);
              const uint32_t bar = kGroup == 2 ? in_cta(own, 0) : own;
              if (rank == 0) barrier_expect(own, S::kPartBytes * kGroup);
              const uint32_t a = stages + slot * S::kPartBytes, b = a + S::kABytes;
              if (kMode != kProducts) {
                tma_load<kGroup>(a, map_a, bar, x, a_row, z);
                tma_load<kGroup>(b, map_b, bar, x, p.begin + b_row, z);
              } else {
                if (it.weight) {
                  for (int m = 0; m < kRows / 64; ++m)
                    tma_load<kGroup>(a + m * 8192, map_a, bar, a_row + m * 64, x, z);
                } else {
                  tma_load<kGroup>(a, map_a, bar, x, a_row, z);
                }
                for (int n = 0; n < kColumns / kGroup / 64; ++n)
                  tma_load<kGroup>(b + n * 8192, map_b, bar, b_row + n * 64, y, z);
              }
            }
            if (!ok) break;
            ++issued;
            if (++stage == kStages) { stage = 0; phase ^= 1; }
          }
        }
      }
      if (!ok) {
        // Give up only once the copies in flight have landed: those counted at this CTA's
        // barriers are waited for (with the same limit), the others given time.
        const int64_t from = issued > kStages ? issued - kStages : 0;
        for (int64_t n = from; kGroup == 1 && n < issued; ++n)
          for (int z = 0; z < S::kParts; ++z)
            barrier_wait(shared_address(&full[n % kStages * S::kParts + z]), uint32_t(n / kStages) & 1);
        for (const unsigned long long start = now_ns(); now_ns() - start < 20000000ull;) __nanosleep(1000);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      for (int64_t t = 0, i; ok && (i = schedule.nth(worker, workers, t)) >= 0; ++t) {
        const Item it = schedule.item(i);
        if (it.k0 >= it.k1) continue;
        const bool a_mn = kMode == kProducts && it.weight, b_mn = kMode == kProducts;
        const uint32_t idesc = instruction(kRows * kGroup, columns, a_mn, b_mn);
        const uint64_t a_step = (a_mn ? kMnStepMajor : kKStepMajor) >> 4;
        const uint64_t b_step = (b_mn ? kMnStepMajor : kKStepMajor) >> 4;
        // Sums of a tile that go to the epilogue apart: one, or one per K block.
        const int sums = it.tiles * (S::kAddUp ? it.k1 - it.k0 : 1);
        const int per_sum = S::kAddUp ? 1 : it.k1 - it.k0;
        for (int n = 0; ok && n < sums; ++n) {
          if (!(ok = barrier_wait(shared_address(&acc_empty[acc]), acc_phase ^ 1))) break;
          fence_after();
          const uint32_t to = tmem + acc * kColumns;
          bool add = false;
          for (int b = 0; b < per_sum; ++b) {
            const uint32_t first = stages + stage * S::kStageBytes;
            const uint64_t da = descriptor(first, a_mn), db = descriptor(first + S::kABytes, b_mn);
            auto wait_part = [&](int z) {
              ok = ok && barrier_wait(shared_address(&full[stage * S::kParts + z]), phase);
              fence_after();
            };
            auto free_part = [&](int z) { commit<kGroup>(shared_address(&empty[stage * S::kParts + z])); };
            wait_part(0);
            if (S::kParts == 3) wait_part(2);
#pragma unroll
            for (int q = 0; q < S::kProductsOfParts; ++q) {
              if (S::kParts == 3 && q == 2) wait_part(1);
              if (!ok) break;
              const int za = S::kParts == 1 ? 0 : part_a(q), zb = S::kParts == 1 ? 0 : part_b(q);
#pragma unroll
              for (int k = 0; k < kDepth / 16; ++k) {
                mma<kGroup>(to, da + (za * S::kPartBytes >> 4) + k * a_step,
                            db + (zb * S::kPartBytes >> 4) + k * b_step, idesc, add);
                add = true;
              }
              if (S::kParts == 3 && q == 1) free_part(2);
              if (S::kParts == 3 && q == 4) free_part(1);
            }
            if (!ok) break;
            free_part(0);
            if (++stage == kStages) { stage = 0; phase ^= 1; }
          }
          commit<kGroup>(shared_address(&acc_full[acc]));
          if (++acc == 2) { acc = 0; acc_phase ^= 1; }
        }
      }
    }
  } else {
    const float scale = kMode == kProducts ? shared_scale(p.cotangent, p.divisor) : 1.f;
    const int quarter = warp & 3;  // the lanes of tensor memory that this warp may read
    const int half = (warp - 2) >> 2;
    constexpr int kMine = kColumns / kHalves;
    const int mine = columns / kHalves;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int64_t t = 0, i; ok && (i = schedule.nth(worker, workers, t)) >= 0; ++t) {
      const Item it = schedule.item(i);
      const int r = it.m0 + int(rank) * kRows + quarter * 32 + lane;
      const bool empty_item = it.k0 >= it.k1;
      if (empty_item && !it.weight) continue;  // a split without K in a later, shorter piece
      Row row = {0.f, 0.f, 0.f, -1};
      float top = -INFINITY, sum = 0.f;  // running, in units of log 2
      if (kMode != kProducts && r < schedule.valid) {
        if (p.row) row = p.row[r];
        else row.target = p.targets[r];
      }
      const float factor = row.inverse * row.scale;
      for (int tile = 0; tile < it.tiles; ++tile) {
        const int n0 = it.n0 + tile * kColumns;
        constexpr int kHeld = S::kAddUp ? kMine / 32 : 1;
        float held[kHeld][32];
        if constexpr (S::kAddUp) {
#pragma unroll
          for (int h = 0; h < kHeld; ++h)
#pragma unroll
            for (int j = 0; j < 32; ++j) held[h][j] = 0.f;
        }
        // The last sum of a tile (the only one unless kAddUp) is waited for here and freed below.
        const int sums = empty_item ? 0 : S::kAddUp ? it.k1 - it.k0 : 1;
        for (int n = 0; n < sums; ++n) {
          ok = __all_sync(0xffffffffu, barrier_wait(shared_address(&acc_full[acc]), acc_phase));
          if (!ok) break;
          fence_after();
          if constexpr (S::kAddUp) {
            const uint32_t from = tmem + acc * kColumns + half * mine + (uint32_t(quarter) << 21);
#pragma unroll
            for (int h = 0; h < kHeld; ++h) {
              if (h * 32 >= mine) continue;
              float v[32];
              tmem_load32(from + h * 32, v);
#pragma unroll
              for (int j = 0; j < 32; ++j) held[h][j] += v[j];
            }
            fence_before();
            __syncwarp();
            if (lane == 0) barrier_arrive_cluster(in_cta(shared_address(&acc_empty[acc]), 0));
            if (++acc == 2) { acc = 0; acc_phase ^= 1; }
          }
        }
        if (!ok) break;
        const uint32_t from = tmem + acc * kColumns + half * mine + (uint32_t(quarter) << 21);
#pragma unroll kHeld
        for (int c = 0; c < kMine; c += 32) {
          if (c >= mine) continue;
          float v[32];
          if constexpr (S::kAddUp) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = held[c / 32 % kHeld][j];
          } else if (empty_item) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0.f;
          } else {
            __syncwarp();
            tmem_load32(from + c, v);
          }
          const int col = n0 + half * mine + c;  // within the piece (stats, dz), of dim (products)
          if constexpr (kMode == kStats) {
            const int left = p.length - col;
            if (left < 32) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = j < left ? v[j] : -INFINITY;
            }
            const int at = row.target - p.begin - col;
            if (__any_sync(0xffffffffu, unsigned(at) < 32u)) {
              float z = 0.f;
#pragma unroll
              for (int j = 0; j < 32; ++j) z = j == at ? v[j] : z;
              if (unsigned(at) < 32u) p.at_target[r] = z;
            }
            float high = v[0];
#pragma unroll
            for (int j = 1; j < 31; j += 2) high = max3(high, v[j], v[j + 1]);
            high = fmaxf(top, fmaxf(high, v[31]) * kLog2E);
            if (left > 0 && high > -INFINITY) {  // -inf: every logit so far is
              const Pair scale2(kLog2E, kLog2E), high2(-high, -high);
              Pair part[2];
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                float a, b;
                fma2(Pair(v[j], v[j + 1]), scale2, high2).get(a, b);
                const Pair e(exp2_fast(a), exp2_fast(b));
                part[(j >> 1) & 1] = j < 4 ? e : add2(part[(j >> 1) & 1], e);
              }
              float a, b;
              add2(part[0], part[1]).get(a, b);
              sum = sum * exp2_fast(top - high) + (a + b);
              top = high;
            } else if (left > 0) {
#pragma unroll
              for (int j = 0; j < 32; ++j) sum += isnan(v[j]) ? v[j] : 0.f;
            }
          } else if constexpr (kMode == kDz) {
            if (r < p.tokens) {
              const Pair scale2(kLog2E, kLog2E), top2(-row.top, -row.top), factor2(factor, factor);
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                float a, b;
                fma2(Pair(v[j], v[j + 1]), scale2, top2).get(a, b);
                mul2(Pair(exp2_fast(a), exp2_fast(b)), factor2).get(v[j], v[j + 1]);
              }
              const int at = row.target - p.begin - col;
              if (unsigned(at) < 32u) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] -= j == at ? row.scale : 0.f;
              }
              if (r >= schedule.valid) {  // rows that only fill the last tile
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = 0.f;
              }
              const size_t place = size_t(r) * p.pitch + col;
              if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int j = 0; j < 32; j += 16) store_row(p.dz + place + j, v + j);
              } else {
                const size_t plane = size_t(p.tokens) * p.pitch;
#pragma unroll
                for (int j = 0; j < 32; j += 16) {
                  __nv_bfloat162 q[3][8];
#pragma unroll
                  for (int k = 0; k < 16; ++k) {
                    __nv_bfloat16 part[3];
                    split_parts(v[j + k], part);
#pragma unroll
                    for (int i = 0; i < 3; ++i) (k & 1 ? q[i][k / 2].y : q[i][k / 2].x) = part[i];
                  }
#pragma unroll
                  for (int i = 0; i < 3; ++i)
                    store32(p.dz + i * plane + place + j, reinterpret_cast<const uint32_t(&)[8]>(q[i]));
                }
              }
            }
          } else if (!it.weight) {
            if (r < schedule.valid && col < p.dim) {  // sum_pitch is a multiple of 32
              float* to = p.sum + (size_t(it.split) * p.tokens + r) * p.sum_pitch + col;
              uint32_t old[4][8];
              if (!p.first) {
#pragma unroll
                for (int j = 0; j < 4; ++j) load32(to + 8 * j, old[j]);
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] += __uint_as_float(old[j / 8][j % 8]);
              }
#pragma unroll
              for (int j = 0; j < 32; j += 8) store_row(to + j, v + j);
            }
          } else if (col < p.dim) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= scale;
            T* rows = static_cast<T*>(p.grad_weight) + size_t(p.begin) * p.dim;
            if (p.weight_sectors && col + 32 <= p.dim) {
              if (r < p.length) {
#pragma unroll
                for (int j = 0; j < 32; j += 32 / sizeof(T)) store_row(rows + size_t(r) * p.dim + col + j, v + j);
              }
            } else {
              // Rows that are not aligned, or end here: turned round in shared memory, so that
              // the lanes write one row's adjacent elements (backward of 1000 x 20000 x 515 bf16: 134
              // us, each lane writing its own row 270).
              float(*mine_turned)[33] = turned[warp - 2];
              __syncwarp();
#pragma unroll
              for (int j = 0; j < 32; ++j) mine_turned[lane][j] = v[j];
              __syncwarp();
              const int first = r - lane;
              if (col + lane < p.dim)
                for (int i = 0; i < 32 && first + i < p.length; ++i)
                  rows[size_t(first + i) * p.dim + col + lane] = narrow<T>(mine_turned[i][lane]);
            }
          }
        }
        if (!S::kAddUp && !empty_item) {
          fence_before();
          __syncwarp();
          if (lane == 0) barrier_arrive_cluster(in_cta(shared_address(&acc_empty[acc]), 0));
          if (++acc == 2) { acc = 0; acc_phase ^= 1; }
        }
      }
      if constexpr (kMode == kStats)
        if (ok && r < schedule.valid) p.stats[size_t(it.group * kHalves + half) * p.tokens + r] = make_float2(top, sum);
    }
  }
  if (!ok) atomicExch(p.error, 1);
  __syncwarp();
  fence_before();
  __syncthreads();
  if constexpr (kGroup == 2) cluster_sync();
  fence_after();
  if (warp == 1) tmem_free<kGroup>(tmem, 512);
}

// ---- rows ---------------------------------------------------------------------------

constexpr int kPackThreads = 256;

// Eight values of a row, zeros from `dim` on, as one or three bfloat16 packs.
template <typename T>
__device__ __forceinline__ void pack8(const T* from, int64_t at, int64_t dim, bool aligned,
                                      __nv_bfloat16* to, size_t plane) {
  T x[8];
  if (aligned && at + 8 <= dim) {
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 8; j += W) {
      const Pack<T, W> q = *reinterpret_cast<const Pack<T, W>*>(from + at + j);
#pragma unroll
      for (int k = 0; k < W; ++k) x[j + k] = q.v[k];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = at + j < dim ? from[at + j] : narrow<T>(0.f);
  }
  if constexpr (sizeof(T) == 2) {
    Pack<__nv_bfloat16, 8> q;
#pragma unroll
    for (int j = 0; j < 8; ++j) q.v[j] = x[j];
    *reinterpret_cast<Pack<__nv_bfloat16, 8>*>(to + at) = q;
  } else {
    Pack<__nv_bfloat16, 8> q[3];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      __nv_bfloat16 part[3];
      split_parts(x[j], part);
      q[0].v[j] = part[0];
      q[1].v[j] = part[1];
      q[2].v[j] = part[2];
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<Pack<__nv_bfloat16, 8>*>(to + k * plane + at) = q[k];
  }
}

struct PackRows {
  const void* hidden;
  int64_t stride, tokens, dim, pitch;
  int32_t per_block;
  bool aligned;
  const float2* softmax;   // backward
  const float* grad_loss;  // backward, one per token or null
  int64_t grad_stride;
  const float* divisor;
  __nv_bfloat16* out;      // [part][token][pitch]
  Row* row;
  int32_t* token;          // of each packed row
  int32_t* valid;
  int32_t* error;
  int32_t* ticket;
};

// Block b places tokens [b per_block, (b + 1) per_block).  Every block counts the targets of
// all tokens itself: 8 bytes a token and block, from L2.  At 8192 tokens the 1024 blocks read 64 KB
// each and pack 32 KB of dim 2048; beyond 16384 tokens there are 2048 blocks, however many tokens.
template <typename T>
__global__ void __launch_bounds__(kPackThreads) pack_rows_kernel(PackRows a, Targets y) {
  constexpr int kWarps = kPackThreads / 32;
  __shared__ int32_t sums[2][kWarps];
  __shared__ int32_t place[32];
  wait_for_previous();
  let_next_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t begin = int64_t(blockIdx.x) * a.per_block;
  int32_t before = 0, all = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < a.tokens; i += kPackThreads) {
    const int has = y[i] >= 0;
    all += has;
    before += has && i < begin;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, d);
    all += __shfl_xor_sync(0xffffffffu, all, d);
  }
  if (lane == 0) { sums[0][warp] = before; sums[1][warp] = all; }
  __syncthreads();
  before = all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) { before += sums[0][w]; all += sums[1][w]; }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *a.valid = all;
    *a.error = 0;
    *a.ticket = 0;
  }
  const size_t plane = size_t(a.tokens) * a.pitch;
  const int64_t end = min(begin + a.per_block, a.tokens);
  for (int64_t t0 = begin; t0 < end; t0 += 32) {
    __syncthreads();
    if (warp == 0) {
      const int64_t t = t0 + lane;
      const int32_t target = t < end ? y[t] : -1;
      const unsigned real = __ballot_sync(0xffffffffu, target >= 0);
      const int rank = __popc(real & ((1u << lane) - 1));
      // Tokens without a target follow all others, in order.
      const int32_t to = target >= 0 ? before + rank : int32_t(all + (t0 - before) + lane - rank);
      place[lane] = target >= 0 ? to : ~to;
      if (t < end) {
        Row row = {0.f, 0.f, 1.f, target};
        if (a.softmax && target >= 0) {
          const float2 of = a.softmax[t];
          row.top = of.x;
          row.inverse = 1.f / of.y;
          if (a.grad_loss) row.scale = a.grad_loss[t * a.grad_stride] / (a.divisor ? *a.divisor : 1.f);
        }
        a.row[to] = row;
        a.token[to] = int32_t(t);
      }
      before += __popc(real);
    }
    __syncthreads();
    const int64_t rows = min(int64_t(32), end - t0);
    for (int j = warp; j < rows; j += kWarps) {
      const int32_t to = place[j] >= 0 ? place[j] : ~place[j];
      const int64_t dim = place[j] >= 0 ? a.dim : 0;
      const T* from = static_cast<const T*>(a.hidden) + (t0 + j) * a.stride;
#pragma unroll 4
      for (int64_t at = lane * 8; at < a.pitch; at += 32 * 8)
        pack8(from, at, dim, a.aligned, a.out + size_t(to) * a.pitch, plane);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kPackThreads)
pack_weight_kernel(const T* weight, int64_t stride, int64_t rows, int64_t dim, int64_t pitch,
                   bool aligned, __nv_bfloat16* out) {
  // It shares nothing with pack_rows_kernel before it, and waits only so that what follows
  // finds both done.
  let_next_start();
  const int64_t packs = pitch / 8, total = rows * packs;
  for (int64_t i = int64_t(blockIdx.x) * kPackThreads + threadIdx.x; i < total;
       i += int64_t(gridDim.x) * kPackThreads) {
    const int64_t r = i / packs;
    pack8(weight + r * stride, (i - r * packs) * 8, dim, aligned, out + r * pitch, size_t(rows) * pitch);
  }
  wait_for_previous();
}

// ---- joins --------------------------------------------------------------------------

// Running (maximum, sum) in units of log 2; an empty one is (-inf, 0).
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  s = (m == top ? s : s * exp2_fast(m - top)) + (m2 == top ? s2 : s2 * exp2_fast(m2 - top));
  m = top;
}

constexpr int kJoinGroups = 8;  // threads per row

struct Totals {
  float* sum;  // each may be null
  float* mean;
  float* count;
  int32_t* ticket;
};

// Joins each row's partial results to its loss; the last block to finish adds the losses up, in
// their order.
__global__ void __launch_bounds__(32 * kJoinGroups)
loss_kernel(const float2* stats, const float* at_target, int groups, const int32_t* tokens_of,
            const int32_t* valid, Targets targets, int64_t tokens, const int32_t* error, float2* softmax,
            float* loss, Totals totals) {
  __shared__ float2 part[kJoinGroups][32];
  __shared__ double sums[kJoinGroups];
  __shared__ int32_t counts[kJoinGroups];
  __shared__ bool last;
  wait_for_previous();
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t r = int64_t(blockIdx.x) * 32 + lane;
  // Rows are packed tokens, or (tokens_of null) the tokens themselves.
  const bool real = r < tokens && (tokens_of ? r < *valid : targets[r] >= 0);
  float m = -INFINITY, s = 0.f;
  if (real)
#pragma unroll 4
    for (int k = g; k < groups; k += kJoinGroups) {
      const float2 v = stats[size_t(k) * tokens + r];
      join(m, s, v.x, v.y);
    }
  part[g][lane] = make_float2(m, s);
  __syncthreads();
  if (g == 0 && r < tokens) {
    for (int k = 1; k < kJoinGroups; ++k) join(m, s, part[k][lane].x, part[k][lane].y);
    const int64_t token = tokens_of ? tokens_of[r] : r;
    softmax[token] = make_float2(real ? m : 0.f, real ? s : 1.f);
    // The difference first: it is small where the loss is.
    const float value = real ? (fmaf(-at_target[r], kLog2E, m) + log2f(s)) * 0.69314718055994531f : 0.f;
    loss[token] = *error ? NAN : value;
  }
  if (!totals.sum && !totals.mean && !totals.count) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(totals.ticket, 1) == int32_t(gridDim.x) - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double sum = 0.0;
  int32_t n = 0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < tokens; i += 32 * kJoinGroups) {
    sum += __ldcg(loss + i);
    n += targets[i] >= 0;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, d);
    n += __shfl_xor_sync(0xffffffffu, n, d);
  }
  if (lane == 0) {
    sums[g] = sum;
    counts[g] = n;
  }
  __syncthreads();
  if (threadIdx.x) return;
  for (int k = 1; k < kJoinGroups; ++k) {
    sum += sums[k];
    n += counts[k];
  }
  if (totals.sum) *totals.sum = float(sum);
  if (totals.mean) *totals.mean = n ? float(sum / n) : 0.f;
  if (totals.count) *totals.count = float(n > 1 ? n : 1);
}

__global__ void no_tokens_kernel(Totals totals) {
  if (totals.sum) *totals.sum = 0.f;
  if (totals.mean) *totals.mean = 0.f;
  if (totals.count) *totals.count = 1.f;
}

// dh from its splits' sums, zeros for tokens without a target; NaN everywhere if a product
// gave up waiting.
template <typename T>
__global__ void __launch_bounds__(kPackThreads)
gradients_kernel(const float* sums, int splits, int64_t sum_pitch, const int32_t* tokens_of,
                 const int32_t* valid, int64_t tokens, int64_t dim, int64_t vocab,
                 const float* cotangent, const float* divisor, const int32_t* error, bool aligned,
                 T* grad_hidden, T* grad_weight) {
  wait_for_previous();
  const bool failed = *error != 0;
  const int64_t real = *valid;
  const float scale = failed ? NAN : shared_scale(cotangent, divisor);
  if (grad_hidden) {
    // Items are four columns of a row; sum_pitch is a multiple of 32.
    const int64_t packs = (dim + 3) / 4, total = tokens * packs, step = int64_t(gridDim.x) * kPackThreads;
    for (int64_t i = int64_t(blockIdx.x) * kPackThreads + threadIdx.x; i < total; i += step) {
      const int64_t r = total <= INT32_MAX ? uint32_t(i) / uint32_t(packs) : i / packs;
      const int64_t c = (i - r * packs) * 4;
      float4 v = failed ? make_float4(NAN, NAN, NAN, NAN) : make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < real) {
#pragma unroll 4
        for (int s = 0; s < splits; ++s) {
          const float4 w = *reinterpret_cast<const float4*>(sums + (s * tokens + r) * sum_pitch + c);
          v.x += w.x;
          v.y += w.y;
          v.z += w.z;
          v.w += w.w;
        }
        v = make_float4(scale * v.x, scale * v.y, scale * v.z, scale * v.w);
      }
      T* to = grad_hidden + tokens_of[r] * dim + c;
      Pack<T, 4> q = {{narrow<T>(v.x), narrow<T>(v.y), narrow<T>(v.z), narrow<T>(v.w)}};
      if (aligned) {
        *reinterpret_cast<Pack<T, 4>*>(to) = q;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < dim) to[j] = q.v[j];
      }
    }
  }
  if (grad_weight && failed)
    for (int64_t i = int64_t(blockIdx.x) * kPackThreads + threadIdx.x; i < vocab * dim;
         i += int64_t(gridDim.x) * kPackThreads)
      grad_weight[i] = narrow<T>(NAN);
}

// CTAs of a product: a pair loads each operand tile of B once for 256 rows, which pays in the
// backward (8192 x 131072 x 2048 bf16: 10.2 ms against 11.5 with single CTAs; 4096 x 32768 x
// 1024: 583 us against 656) and in float32 (1021 x 10007 x 515: forward 106 us against 120).  The
// bf16 forward does better on single CTAs (2048 x 50000 x 4096: 683 us against 725; 4096 x 32768
// x 1024: 213 against 217).  Up to 128 rows a pair's second CTA would have none.
int pair_size(const PurinLossArgs* a, bool backward) {
  return a->tokens > kRows && (backward || a->dtype == PURIN_OPS_FLOAT32) ? 2 : 1;
}

// ---- plan ---------------------------------------------------------------------------

struct Plan {
  int parts;
  int64_t pitch;           // of packed rows
  bool weight_packed;
  bool direct;             // forward: hidden is read in place
  int64_t tiles_at_once, groups;   // forward; groups of column tiles, and their halves
  int64_t piece, splits, split_blocks, sum_pitch;  // backward
  size_t hidden, weight, row, token, scalars, stats, at_target, dz, sum, total;
};

Plan plan_of(const PurinLossArgs* a, bool backward, int sms) {
  Plan p;
  const size_t n = size_t(a->tokens);
  p.parts = a->dtype == PURIN_OPS_FLOAT32 ? 3 : 1;
  p.pitch = ceil_div(a->dim, 8) * 8;
  // TMA reads the weight in place if its rows are 16-byte aligned.
  p.weight_packed = p.parts == 3 || !a->weight || reinterpret_cast<uintptr_t>(a->weight) % 16 ||
                    a->weight_stride % 8 || a->weight_stride < a->dim;
  // One tile of rows costs the same whether tokens without a target are in it: in a forward
  // that TMA can read in place they stay, which saves the launch that packs (5 us).
  p.direct = !backward && !p.weight_packed && a->tokens <= kRows && a->hidden &&
             reinterpret_cast<uintptr_t>(a->hidden) % 16 == 0 && a->hidden_stride % 8 == 0 &&
             a->hidden_stride >= a->dim;
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t here = at; at += align256(bytes); return here; };
  p.hidden = take(p.direct ? 0 : p.parts * n * p.pitch * 2);
  p.weight = take(p.weight_packed ? size_t(p.parts) * a->vocab * p.pitch * 2 : 0);
  p.row = take(n * sizeof(Row));
  p.token = take(n * 4);
  p.scalars = take(12);  // valid rows, error, ticket
  p.stats = p.at_target = p.dz = p.sum = 0;
  const int64_t kColumns = p.parts == 3 && pair_size(a, backward) == 1 ? Shape<float, 1>::kColumns : Shape<float, 2>::kColumns;
  const int64_t columns = ceil_div(a->vocab, kColumns);
  const int halves = p.parts == 3 && pair_size(a, backward) == 2 ? Shape<float, 2>::kHalves : 1;
  p.tiles_at_once = p.groups = p.piece = p.splits = p.split_blocks = p.sum_pitch = 0;
  if (!backward) {
    const int64_t most = std::max<int64_t>(1, int64_t(kStatsBytes / (8 * halves) / std::max<size_t>(n, 1)));
    p.tiles_at_once = ceil_div(columns, most);
    p.groups = ceil_div(columns, p.tiles_at_once);
    p.stats = take(size_t(p.groups) * halves * n * 8);
    p.at_target = take(n * 4);
  } else {
    // As many columns of dz as kPieceBytes hold, at least kLeastColumns, in pieces of about one size.
    int64_t most = int64_t(kPieceBytes / (2 * p.parts) / std::max<size_t>(n, 1)) / kColumns;
    most = std::min(std::max<int64_t>(most, kLeastColumns / kColumns), columns);
    p.piece = ceil_div(columns, ceil_div(columns, most)) * kColumns;
    p.dz = take(p.parts * n * p.piece * 2);
    p.sum_pitch = ceil_div(a->dim, 32) * 32;
    // Few tiles of dh: K is split until the SMs have one each, eight K blocks at least.
    const int64_t tiles = std::max<int64_t>(1, ceil_div(a->tokens, kRows) * ceil_div(a->dim, kColumns));
    const int64_t blocks = ceil_div(std::min(p.piece, a->vocab), kDepth);
    p.split_blocks = ceil_div(blocks, std::max<int64_t>(1, std::min(sms / tiles, blocks / 8)));
    p.splits = ceil_div(blocks, p.split_blocks);  // none is empty in the first piece
    p.sum = take(size_t(p.splits) * n * p.sum_pitch * 4);
  }
  p.total = at;
  return p;
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
  static const EncodeTiled found = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult result;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &result) != cudaSuccess ||
        result != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return found;
}

// Boxes of 64 x box_rows elements of a [parts][rows][columns] array, swizzled by 128 bytes.
int32_t make_map(CUtensorMap* map, const void* base, int64_t columns, int64_t rows, int64_t parts,
                 int64_t pitch, int64_t plane, int box_rows) {
  const EncodeTiled encode = encoder();
  if (!encode) return set_error(PURIN_ERR_CUDA, "loss: the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t size[3] = {cuuint64_t(columns), cuuint64_t(rows), cuuint64_t(parts)};
  const cuuint64_t stride[2] = {cuuint64_t(pitch) * 2, cuuint64_t(plane) * 2};
  const cuuint32_t box[3] = {64, cuuint32_t(box_rows), 1}, step[3] = {1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), size, stride,
                            box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? PURIN_OK : set_error(PURIN_ERR_CUDA, "loss: cuTensorMapEncodeTiled failed");
}

// CTA pairs that fit the device at once (a part of it with an odd number of SMs leaves one over).
template <int kGroup>
int groups_that_fit(void (*kernel)(Product), const cudaLaunchConfig_t& config, int device, int sms,
                    std::atomic<int> (&known)[64]) {
  const bool keeps = device >= 0 && device < 64;
  int n = keeps ? known[device].load(std::memory_order_relaxed) : 0;
  if (n > 0) return n;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &config) != cudaSuccess || n <= 0) {
    cudaGetLastError();  // not another call's error
    return sms / kGroup;
  }
  if (keeps) known[device].store(n, std::memory_order_relaxed);
  return n;
}

template <typename T, int kGroup, Mode kMode>
int32_t launch_product(const Product& p, int64_t most_items, int device, int sms, cudaStream_t stream) {
  using S = Shape<T, kGroup>;
  auto kernel = product_kernel<T, kGroup, kMode>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSharedBytes))
    return cuda_status(e);
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(unsigned(sms / kGroup * kGroup));
  config.blockDim = dim3(S::kThreads);
  config.dynamicSmemBytes = S::kSharedBytes;
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim = {kGroup, 1, 1};
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // as launch_after
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = p.row ? 2 : 1;  // without pack_rows_kernel it is the call's first
  if constexpr (kGroup > 1) {
    static std::atomic<int> known[64];  // of each device
    sms = std::min(sms, groups_that_fit<kGroup>(kernel, config, device, sms, known) * kGroup);
  }
  config.gridDim = dim3(unsigned(std::min<int64_t>(most_items, sms / kGroup) * kGroup));
  return cuda_status(cudaLaunchKernelEx(&config, kernel, p));
}

int32_t check_sizes(const PurinLossArgs* a) {
  if (!a) return invalid("loss: null arguments");
  if (a->dtype != PURIN_OPS_BFLOAT16 && a->dtype != PURIN_OPS_FLOAT32)
    return set_error(PURIN_ERR_UNSUPPORTED, "loss: element type must be bfloat16 or float32");
  if (a->tokens < 0 || a->vocab < 1 || a->dim < 1) return invalid("loss: invalid sizes");
  if (a->tokens > INT32_MAX / 2 || a->vocab > INT32_MAX / 2 || a->dim > INT32_MAX / 2)
    return set_error(PURIN_ERR_UNSUPPORTED, "loss: sizes must be below 2^30");
  if (a->hidden_stride < 0 || a->weight_stride < 0) return invalid("loss: negative stride");
  return PURIN_OK;
}

int32_t check(const PurinLossArgs* a) {
  if (int32_t bad = check_sizes(a)) return bad;
  if (a->tokens && (!a->hidden || !a->targets || !a->softmax)) return invalid("loss: null hidden, targets or softmax");
  if (!a->weight) return invalid("loss: null weight");
  return PURIN_OK;
}

template <typename F>
int32_t with_loss_dtype(int32_t dtype, F&& f) {
  return dtype == PURIN_OPS_FLOAT32 ? f(float()) : f(__nv_bfloat16());
}

Targets targets_of(const PurinLossArgs* a) { return {a->targets, a->targets_64bit != 0, a->vocab, a->ignore}; }

// Packed hidden rows (and the weight, where TMA cannot read it in place), the rows' data.
template <typename T>
int32_t pack(const PurinLossArgs* a, const Plan& p, char* ws, bool backward, int sms, cudaStream_t s,
             Product* product) {
  PackRows r;
  r.hidden = a->hidden;
  r.stride = a->hidden_stride;
  r.tokens = a->tokens;
  r.dim = a->dim;
  r.pitch = p.pitch;
  // A row per warp; more only where the blocks would count the targets too often.
  r.per_block = int32_t(std::max<int64_t>(8, ceil_div(a->tokens, 2048)));
  r.aligned = reinterpret_cast<uintptr_t>(a->hidden) % 16 == 0 && a->hidden_stride * sizeof(T) % 16 == 0;
  r.softmax = backward ? reinterpret_cast<const float2*>(a->softmax) : nullptr;
  r.grad_loss = a->grad_stride ? a->grad_loss : nullptr;
  r.grad_stride = a->grad_stride;
  r.divisor = a->divisor;
  r.out = reinterpret_cast<__nv_bfloat16*>(ws + p.hidden);
  r.row = reinterpret_cast<Row*>(ws + p.row);
  r.token = reinterpret_cast<int32_t*>(ws + p.token);
  r.valid = reinterpret_cast<int32_t*>(ws + p.scalars);
  r.error = r.valid + 1;
  r.ticket = r.valid + 2;
  const Targets y = targets_of(a);
  pack_rows_kernel<T><<<unsigned(ceil_div(a->tokens, r.per_block)), kPackThreads, 0, s>>>(r, y);
  if (p.weight_packed) {
    const int64_t blocks = ceil_div(a->vocab * (p.pitch / 8), kPackThreads);
    if (cudaError_t e = launch_after(
            pack_weight_kernel<T>, dim3(unsigned(std::min<int64_t>(blocks, int64_t(sms) * 16))), dim3(kPackThreads),
            0, s, static_cast<const T*>(a->weight), a->weight_stride, a->vocab, a->dim, p.pitch,
            reinterpret_cast<uintptr_t>(a->weight) % 16 == 0 && a->weight_stride * sizeof(T) % 16 == 0,
            reinterpret_cast<__nv_bfloat16*>(ws + p.weight)))
      return cuda_status(e);
  }
  product->tokens = int32_t(a->tokens);
  product->dim = int32_t(a->dim);
  product->valid = r.valid;
  product->error = r.error;
  product->row = r.row;
  product->cotangent = backward && !a->grad_stride ? a->grad_loss : nullptr;
  product->divisor = a->divisor;
  return launched();
}

struct Weight {
  const void* base;
  int64_t columns, pitch, plane;
};
Weight weight_of(const PurinLossArgs* a, const Plan& p, char* ws) {
  if (!p.weight_packed) return {a->weight, a->dim, a->weight_stride, a->vocab * a->weight_stride};
  return {ws + p.weight, p.pitch, p.pitch, a->vocab * p.pitch};
}

template <typename T, int kGroup>
int32_t forward(const PurinLossArgs* a, const Plan& p, char* ws, int sms, cudaStream_t s) {
  constexpr int kColumns = Shape<T, kGroup>::kColumns;
  Product q = {};
  const Weight w = weight_of(a, p, ws);
  if (p.direct) {
    q.tokens = int32_t(a->tokens);
    q.dim = int32_t(a->dim);
    q.targets = targets_of(a);
    q.error = reinterpret_cast<int32_t*>(ws + p.scalars) + 1;
    if (int32_t bad = make_map(&q.map[0], a->hidden, a->dim, a->tokens, 1, a->hidden_stride,
                               a->tokens * a->hidden_stride, kRows)) return bad;
  } else {
    if (int32_t bad = pack<T>(a, p, ws, false, sms, s, &q)) return bad;
    if (int32_t bad = make_map(&q.map[0], ws + p.hidden, p.pitch, a->tokens, p.parts, p.pitch,
                               a->tokens * p.pitch, kRows)) return bad;
  }
  if (int32_t bad = make_map(&q.map[1], w.base, w.columns, a->vocab, p.parts, w.pitch, w.plane,
                             kColumns / kGroup)) return bad;
  q.begin = 0;
  q.length = int32_t(a->vocab);
  q.tiles_at_once = int32_t(p.tiles_at_once);
  q.stats = reinterpret_cast<float2*>(ws + p.stats);
  q.at_target = reinterpret_cast<float*>(ws + p.at_target);
  const int64_t items = ceil_div(a->tokens, kRows * kGroup) * p.groups;
  if (int32_t bad = launch_product<T, kGroup, kStats>(q, items, a->device, sms, s)) return bad;
  return cuda_status(launch_after(
      loss_kernel, dim3(unsigned(ceil_div(a->tokens, 32))), dim3(32 * kJoinGroups), 0, s, q.stats, q.at_target,
      int(p.groups) * Shape<T, kGroup>::kHalves,
      p.direct ? nullptr : reinterpret_cast<const int32_t*>(ws + p.token), q.valid, targets_of(a), a->tokens,
      q.error, reinterpret_cast<float2*>(a->softmax), a->loss, Totals{a->sum, a->mean, a->count, q.error + 1}));
}

template <typename T, int kGroup>
int32_t backward(const PurinLossArgs* a, const Plan& p, char* ws, int sms, cudaStream_t s) {
  constexpr int kColumns = Shape<T, kGroup>::kColumns;
  Product q = {};
  if (int32_t bad = pack<T>(a, p, ws, true, sms, s, &q)) return bad;
  const Weight w = weight_of(a, p, ws);
  const void* hidden = ws + p.hidden;
  const void* dz = ws + p.dz;
  Product z = q;
  if (int32_t bad = make_map(&z.map[0], hidden, p.pitch, a->tokens, p.parts, p.pitch, a->tokens * p.pitch,
                             kRows)) return bad;
  if (int32_t bad = make_map(&z.map[1], w.base, w.columns, a->vocab, p.parts, w.pitch, w.plane,
                             kColumns / kGroup)) return bad;
  z.dz = static_cast<__nv_bfloat16*>(const_cast<void*>(dz));
  z.pitch = int32_t(p.piece);
  if (int32_t bad = make_map(&q.map[1], w.base, w.columns, a->vocab, p.parts, w.pitch, w.plane, 64)) return bad;
  if (int32_t bad = make_map(&q.map[3], hidden, p.pitch, a->tokens, p.parts, p.pitch, a->tokens * p.pitch,
                             64)) return bad;
  q.splits = int32_t(p.splits);
  q.split_blocks = int32_t(p.split_blocks);
  // As few tiles across dim as fit, no wider than they need to be: of 515 columns three of 192
  // (backward of 3000 x 20000 x 300 bf16, two of 192: 273 us against 308 with two of 256).
  const int64_t dim_tiles = ceil_div(a->dim, kColumns);
  q.weight_sectors = a->dim * sizeof(T) % 32 == 0 && reinterpret_cast<uintptr_t>(a->grad_weight) % 32 == 0;
  q.columns = int32_t(ceil_div(ceil_div(a->dim, dim_tiles), 64) * 64);
  q.sum = reinterpret_cast<float*>(ws + p.sum);
  q.sum_pitch = int32_t(p.sum_pitch);
  q.grad_weight = a->grad_weight;
  q.want_hidden = a->grad_hidden != nullptr;
  q.want_weight = a->grad_weight != nullptr;
  int64_t mapped = 0;  // length that the maps of dz were made for
  for (int64_t begin = 0; begin < a->vocab; begin += p.piece) {
    const int64_t length = std::min(p.piece, a->vocab - begin);
    z.begin = q.begin = int32_t(begin);
    z.length = q.length = int32_t(length);
    q.first = begin == 0;
    if (length != mapped) {  // K ends with the piece: columns behind it read as zeros
      if (int32_t bad = make_map(&q.map[0], dz, length, a->tokens, p.parts, p.piece, a->tokens * p.piece,
                                 kRows)) return bad;
      if (int32_t bad = make_map(&q.map[2], dz, length, a->tokens, p.parts, p.piece, a->tokens * p.piece,
                                 64)) return bad;
      mapped = length;
    }
    const int64_t row_tiles = ceil_div(a->tokens, kRows * kGroup);
    if (int32_t bad = launch_product<T, kGroup, kDz>(z, row_tiles * ceil_div(length, kColumns), a->device, sms, s)) return bad;
    const int64_t items = (q.want_hidden ? row_tiles * dim_tiles * p.splits : 0) +
                          (q.want_weight ? ceil_div(length, kRows * kGroup) * dim_tiles : 0);
    if (int32_t bad = launch_product<T, kGroup, kProducts>(q, items, a->device, sms, s)) return bad;
  }
  const int64_t blocks = std::min<int64_t>(ceil_div(a->tokens * ceil_div(a->dim, 4), kPackThreads), int64_t(sms) * 16);
  const bool aligned = a->dim % 4 == 0 && reinterpret_cast<uintptr_t>(a->grad_hidden) % (4 * sizeof(T)) == 0;
  return cuda_status(launch_after(
      gradients_kernel<T>, dim3(unsigned(blocks)), dim3(kPackThreads), 0, s, q.sum, int(p.splits), p.sum_pitch,
      reinterpret_cast<const int32_t*>(ws + p.token), q.valid, a->tokens, a->dim, a->vocab, q.cotangent, q.divisor,
      q.error, aligned,
      static_cast<T*>(a->grad_hidden), static_cast<T*>(a->grad_weight)));
}

}  // namespace
}  // namespace ops
}  // namespace purin

using namespace purin::ops;
using purin::set_error;

extern "C" int32_t purin_loss_workspace_size(const PurinLossArgs* a, int32_t backward, size_t* bytes) {
  return guarded([&]() -> int32_t {
    if (int32_t bad = check_sizes(a)) return bad;
    if (!bytes) return invalid("loss: null arguments");
    *bytes = plan_of(a, backward != 0, sm_count(a->device)).total;
    return PURIN_OK;
  });
}

extern "C" int32_t purin_loss_forward(const PurinLossArgs* a, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  return guarded([&]() -> int32_t {
    if (int32_t bad = check(a)) return bad;
    if (a->tokens && !a->loss) return invalid("loss: null loss");
    const int sms = sm_count(a->device);
    const Plan p = plan_of(a, false, sms);
    if (!workspace || workspace_bytes < p.total)
      return set_error(PURIN_ERR_WORKSPACE, "loss: workspace too small");
    OnDevice on(a->device);
    if (on.error != cudaSuccess) return cuda_status(on.error);
    auto s = static_cast<cudaStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    if (a->tokens == 0) {
      no_tokens_kernel<<<1, 1, 0, s>>>(Totals{a->sum, a->mean, a->count, nullptr});
      return launched();
    }
    return with_loss_dtype(a->dtype, [&](auto t) {
      using T = decltype(t);
      if constexpr (sizeof(T) == 4)
        if (pair_size(a, false) == 2) return forward<T, 2>(a, p, ws, sms, s);
      return forward<T, 1>(a, p, ws, sms, s);
    });
  });
}

extern "C" int32_t purin_loss_backward(const PurinLossArgs* a, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  return guarded([&]() -> int32_t {
    if (int32_t bad = check(a)) return bad;
    if (a->tokens && !a->grad_loss) return invalid("loss: null grad_loss");
    const int sms = sm_count(a->device);
    const Plan p = plan_of(a, true, sms);
    if (!workspace || workspace_bytes < p.total)
      return set_error(PURIN_ERR_WORKSPACE, "loss: workspace too small");
    OnDevice on(a->device);
    if (on.error != cudaSuccess) return cuda_status(on.error);
    auto s = static_cast<cudaStream_t>(stream);
    char* ws = static_cast<char*>(workspace);
    if (!a->grad_hidden && !a->grad_weight) return PURIN_OK;
    if (a->tokens == 0) {
      if (!a->grad_weight) return PURIN_OK;
      return cuda_status(cudaMemsetAsync(a->grad_weight, 0, size_t(a->vocab) * a->dim * dtype_bytes(a->dtype), s));
    }
    return with_loss_dtype(a->dtype, [&](auto t) {
      using T = decltype(t);
      return pair_size(a, true) == 2 ? backward<T, 2>(a, p, ws, sms, s) : backward<T, 1>(a, p, ws, sms, s);
    });
  });
}
