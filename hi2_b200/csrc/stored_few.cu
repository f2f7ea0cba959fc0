// The product of packed rows with tiles of up to 8 activation rows: single tokens, small batches, experts with a few
// tokens each.
//
// A block takes 128 sorted rows and a slice of the columns; the slices of a row tile are a cluster and join
// their sums through distributed shared memory in rank order.  Warps 0..3 and 4..7 take the tile's four groups
// of 32 rows, each half of the warps one half of the columns.  Every warp streams its own part of the packed
// data through a ring of bulk copies, so the loads of a whole block are in flight before anything is
// computed, and no barrier between warps is needed while it lasts.
//
// The slice is taken in blocks of 1024 columns.  First the warps form the activations' fp16 parts of the block
// in shared memory (divided, rotated, relative to a power of two per row and half of the BLOCK, so nothing
// waits for a whole row's largest value); then every warp decodes chunk after chunk straight into the A fragments of
// warp-level products m16n8k16: lane 4 g + t holds 16 columns of rows g, g + 8, g + 16 and g + 24, and the column order
// inside a chunk is the same permutation for both operands, so a lane's 16 columns are contiguous in memory.
//
// What bounds it: decoding and products share the fp16 pipe (183 clocks for 2048 INT2 weights, stored.cuh).  28672 x 8192
// INT2 weights with one row take 40 us where streaming them alone takes 16 and the products without decoding 22; the
// packed bytes ask for 12.  In the smallest calls it is latency: 4096 x 4096 with one row takes 7.2 us.  Measured and
// dropped: three stages per ring with one block per SM; the next chunk's words read ahead of the products.
#include <type_traits>

#include "stored_async.cuh"

namespace hi2 {
namespace stored {
namespace {

constexpr int WARPS = 8, THREADS = 256;
constexpr int BLOCK_CHUNKS = 16, BLOCK_COLUMNS = BLOCK_CHUNKS * CHUNK;
constexpr int HALF_CHUNKS = BLOCK_CHUNKS / 2;
constexpr int RING_STAGES = 2, RING_BYTES = 3 * 1024;  // a stage: four chunks of INT2, two of INT4, one of INT8
constexpr int X_PITCH = BLOCK_COLUMNS + 8;         // halves; the extra 16 bytes keep 128-bit reads of eight rows apart
constexpr int SUM_PITCH = TILE_ROWS + 4;
constexpr int MAX_SPLIT = 8;
template <int PARTS>
constexpr int PLACES = PARTS == 1 ? 16 : 8;        // of a row's 1024 columns in shared memory; at least FEW_WIDTH

struct Shared {
  uint8_t ring[WARPS][RING_STAGES][RING_BYTES];
  float sums[2][FEW_WIDTH][SUM_PITCH];  // of the two halves
  float scale[2][16];                   // of each half and place
  uint32_t out_row[TILE_ROWS];
  unsigned long long full[WARPS][RING_STAGES];
  volatile uint32_t abort;
};
template <int PARTS>
constexpr size_t smem_bytes() {
  return sizeof(Shared) + (size_t)PARTS * PLACES<PARTS> * X_PITCH * sizeof(__half) + 16;
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The lane's 16 columns of its four rows in the chunk at `slab`.
struct LaneRows {
  float lo_min[4], lo_scale[4];
  __half2 step_scale[2];
};
template <int NBITS, bool SMALL>
__device__ __forceinline__ void decode_rows(const uint8_t* slab, int first_word, int pair_unit, const LaneRows& rows, uint32_t (&w)[4][8]) {
  const uint2 pairs = *reinterpret_cast<const uint2*>(slab + 256 * NBITS + 8 * pair_unit);
  Ladder l[4];
  {
    const float min01[2] = {rows.lo_min[0], rows.lo_min[1]}, scale01[2] = {rows.lo_scale[0], rows.lo_scale[1]};
    const float min23[2] = {rows.lo_min[2], rows.lo_min[3]}, scale23[2] = {rows.lo_scale[2], rows.lo_scale[3]};
    ladders<NBITS, SMALL>(pairs.x, min01, scale01, rows.step_scale[0], l[0], l[1]);
    ladders<NBITS, SMALL>(pairs.y, min23, scale23, rows.step_scale[1], l[2], l[3]);
  }
#pragma unroll
  for (int h = 0; h < NBITS / 2; ++h) {
    const uint4 v = *reinterpret_cast<const uint4*>(slab + 512 * h + 4 * first_word);
    const uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int r = 0; r < 4; ++r) decode_word<NBITS, SMALL>(q[r], l[r], w[r] + 16 / NBITS * h);
  }
}

// Where a warp is in its ring.
struct Ring {
  uint8_t* data;
  unsigned long long* full;
  int slab, stage;  // bytes of a chunk; stage
  uint32_t phase;
};

// `count` chunks against the activations at x, whose powers of two are s0 and s1 for the lane's two rows of the result.  One
// part: added to acc as they are.  Two: added with their powers of two.  False when a wait ran out.
template <int PARTS, int NBITS, bool SMALL, typename REFILL>
__device__ __forceinline__ bool multiply(Ring& ring, const __half* x, int count, int first_word, int pair_unit, const LaneRows& rows,
                                         float s0, float s1, float (&acc)[2][4], volatile uint32_t* abort, int32_t* status, const REFILL& refill) {
  constexpr int PER_COPY = 8 / NBITS;
  while (count > 0) {
    if (!__all_sync(0xffffffffu, bar_wait(ring.full + ring.stage, ring.phase, abort, status))) return false;
    const int here = min(PER_COPY, count);
    const uint8_t* slab = ring.data + ring.stage * RING_BYTES;
#pragma unroll 1  // (unrolled, the loops of the code widths push one another out of the instruction cache)
    for (int i = 0; i < here; ++i, x += CHUNK, slab += ring.slab) {
      uint32_t w[4][8];
      decode_rows<NBITS, SMALL>(slab, first_word, pair_unit, rows, w);
      // With two parts a chunk's sum is formed by itself, small parts first, and added in fp32: the tensor cores' accumulator
      // drops what does not fit it at every step, which over 512 columns would cost 1e-6 of a result, always towards zero.
      float sum[2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int q = 0; q < 4; ++q) sum[m][q] = PARTS == 1 ? acc[m][q] : 0.0f;
#pragma unroll
      for (int part = PARTS - 1; part >= 0; --part) {
        const __half* from = x + part * PLACES<PARTS> * X_PITCH;
        const uint4 x0 = *reinterpret_cast<const uint4*>(from), x1 = *reinterpret_cast<const uint4*>(from + 8);
        const uint32_t k[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          mma(sum[0], w[0][2 * s], w[1][2 * s], w[0][2 * s + 1], w[1][2 * s + 1], k[2 * s], k[2 * s + 1]);
          mma(sum[1], w[2][2 * s], w[3][2 * s], w[2][2 * s + 1], w[3][2 * s + 1], k[2 * s], k[2 * s + 1]);
        }
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[m][q] = PARTS == 1 ? sum[m][q] : acc[m][q] + sum[m][q] * (q & 1 ? s1 : s0);
    }
    count -= here;
    __syncwarp();  // every lane has read the stage
    refill(ring.stage);
    if (++ring.stage == RING_STAGES) ring.stage = 0, ring.phase ^= 1;
  }
  return true;
}

template <int PARTS>
__global__ void __launch_bounds__(THREADS, 2)
few_kernel(const Product p, const int split, const int runs) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared& sm = *reinterpret_cast<Shared*>(raw);
  __half* const xs = reinterpret_cast<__half*>((reinterpret_cast<uintptr_t>(raw) + sizeof(Shared) + 15) & ~(uintptr_t)15);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row_tiles = (int)(p.w.groups_per_expert / 4);
  const int rank = (int)(blockIdx.x % split);
  const uint32_t which = blockIdx.x / split;
  // runs of row tiles as equal as they can be, the longer ones first
  const int run = (int)(which % runs), longer = row_tiles % runs;
  int row_tile = run * (row_tiles / runs) + min(run, longer);
  const int last_tile = row_tile + row_tiles / runs - (run < longer ? 0 : 1);
  int32_t* const status = p.w.status;
  TokenTile tile;
  if (p.tiles.index != nullptr && !p.settled) chain_wait();  // which expert comes from an earlier kernel
  if (!p.tiles.get(which / runs, tile)) return;  // the same for all blocks of a cluster
  const int tokens = tile.end - tile.begin;

  // ---- this warp's stream of packed data
  const int half = warp >> 2, quarter = warp & 3;
  const int all = (int)(p.w.k / CHUNK);
  const int c0 = (int)((int64_t)all * rank / split), n = (int)((int64_t)all * (rank + 1) / split) - c0;
  const int blocks = (n + BLOCK_CHUNKS - 1) / BLOCK_CHUNKS;
  const int last_chunks = n - (blocks - 1) * BLOCK_CHUNKS;                      // of the last block
  const int last_half0 = (last_chunks + 1) / 2;
  const int last_mine = half == 0 ? last_half0 : last_chunks - last_half0;
  const int mine = (blocks - 1) * HALF_CHUNKS + last_mine;
  const int64_t first_group = (int64_t)tile.expert * p.w.groups_per_expert + quarter;
  GroupForm form = load_group(p.w.groups, first_group + row_tile * 4);
  RowConsts consts[4];
  auto load_rows = [&](int tile_of_rows) {
#pragma unroll
    for (int r = 0; r < 4; ++r) consts[r] = load_row(p.w.rows, (first_group + tile_of_rows * 4) * GROUP_ROWS + 8 * r + g);
  };
  load_rows(row_tile);
  // What the activations need is asked for ahead of the packed data: behind it, it waited 3 us for its turn at the memory.
  {
    const int64_t first = (int64_t)tile.expert * p.w.k + (int64_t)c0 * CHUNK, columns = (int64_t)n * CHUNK;
    if (p.w.inv_scale != nullptr)
      for (int64_t i = 32 * threadIdx.x; i < columns; i += 32 * THREADS) prefetch_l2(p.w.inv_scale + first + i);
    for (int64_t i = 2048 * threadIdx.x; i < columns; i += 2048 * THREADS) prefetch_l2(p.w.had + (first + i) / 16);
  }
  Ring ring{&sm.ring[warp][0][0], &sm.full[warp][0], 0, 0, 0};
  const uint8_t* data;
  int copy_shift, copies, next_copy;
  auto issue = [&](int copy, int stage) {  // by one lane
    const int j = copy << copy_shift, b = j / HALF_CHUNKS, count = min(1 << copy_shift, mine - j);
    const int chunk = c0 + b * BLOCK_CHUNKS + (half == 0 ? 0 : b == blocks - 1 ? last_half0 : HALF_CHUNKS) + j % HALF_CHUNKS;
    bar_expect(&sm.full[warp][stage], (uint32_t)(count * ring.slab));
    bulk_load(sm.ring[warp][stage], data + (int64_t)chunk * ring.slab, (uint32_t)(count * ring.slab), &sm.full[warp][stage]);
  };
  auto begin_stream = [&]() {  // of the tile of packed rows that `form` belongs to
    ring.slab = form.slab_bytes(), copy_shift = 3 - form.width();                 // 4, 2, 1 chunks
    data = static_cast<const uint8_t*>(p.w.data) + (int64_t)form.base * 16;
    copies = form.width() == 0 ? 0 : (mine + (1 << copy_shift) - 1) >> copy_shift;
    next_copy = RING_STAGES;
    if (lane == 0)
      for (int c = 0; c < RING_STAGES && c < copies; ++c) issue(c, (ring.stage + c) % RING_STAGES);
    __syncwarp();
  };
  auto refill = [&](int stage) {
    if (lane == 0 && next_copy < copies) issue(next_copy, stage);
    ++next_copy;
    __syncwarp();
  };
  if (lane == 0) {
    for (int s = 0; s < RING_STAGES; ++s) bar_init(&sm.full[warp][s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncwarp();
  begin_stream();
  if (threadIdx.x == 0) sm.abort = 0;
  const int first_word = code_word(g, t);

  chain_wait();  // the activations
  chain_next();  // (after the wait: the next product may go by the index or the tile list at once)
  bool ok = true, prepared = false;
  for (;; ++row_tile) {
    LaneRows rows;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const RowConsts c = consts[r];
      rows.lo_min[r] = c.lo_min(), rows.lo_scale[r] = c.lo_scale();
      const __half s = __ushort_as_half((uint16_t)c.step_scale);
      if (r & 1) rows.step_scale[r / 2] = __halves2half2(__low2half(rows.step_scale[r / 2]), s);
      else rows.step_scale[r / 2] = __half2half2(s);
      if (half == 0 && t == 0) sm.out_row[quarter * 32 + 8 * r + g] = c.out_row;
    }
    const int pair_unit = (4 >> form.shift()) * g + (t >> form.shift());
    const bool more = row_tile < last_tile;
    GroupForm next_form{0, 0};
    if (more) next_form = load_group(p.w.groups, first_group + (row_tile + 1) * 4);
    float total[2][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) total[m][i] = 0.0f;
    // Shared memory holds 8 or 16 rows of a block; fewer rows leave room for several blocks, which are prepared together,
    // and once for a run of tiles.
    const int together = PLACES<PARTS> / tokens;
    for (int b0 = 0; b0 < blocks; b0 += together) {
      const int here = min(together, blocks - b0);
      // ---- the activations, a warp per block, row and half: up to 32 pieces of 16 columns, one per lane
      if (!prepared) {
        __syncthreads();  // nobody reads the blocks before any more (and the barriers' words are set)
        for (int u = warp; u < 2 * tokens * here; u += WARPS) {
          const int second = u & 1, place = u >> 1, b = b0 + place / tokens, r = place % tokens;
          const int chunks = b == blocks - 1 ? last_chunks : BLOCK_CHUNKS, half0 = b == blocks - 1 ? last_half0 : HALF_CHUNKS;
          const int piece = (second ? 4 * half0 : 0) + lane;
          const bool in = piece < 4 * (second ? chunks : half0);
          int64_t from = tile.begin + r;
          if (p.tiles.index != nullptr && p.from.kind != FROM_GATED) from = (uint32_t)p.tiles.pair(from) / (uint32_t)p.from.top_k;
          float v[16];
          float top = 0.0f;
          if (in) {
            stored_basis(p.from, p.w, from, tile.expert, (int64_t)(c0 + b * BLOCK_CHUNKS) * 4 + piece, v);
            top = largest(v);
          }
#pragma unroll
          for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          const PowerOfTwo power = power_for(top);
          if (lane == 0) sm.scale[second][place] = power.back;
          if (in) {
            uint4 hi[2], lo[2];
            split16<PARTS>(v, power.to, hi, lo);
            uint4* dst = reinterpret_cast<uint4*>(xs + place * X_PITCH + piece * 16);
            dst[0] = hi[0], dst[1] = hi[1];
            if (PARTS == 2) {
              dst = reinterpret_cast<uint4*>(xs + (PLACES<PARTS> + place) * X_PITCH + piece * 16);
              dst[0] = lo[0], dst[1] = lo[1];
            }
          }
        }
        __syncthreads();
      }
      for (int sub = 0; sub < here; ++sub) {
        const int chunks = b0 + sub == blocks - 1 ? last_chunks : BLOCK_CHUNKS, half0 = b0 + sub == blocks - 1 ? last_half0 : HALF_CHUNKS;
        // ---- this warp's chunks of a block; lanes without a row of their own read the last one's
        const float s0 = sm.scale[half][sub * tokens + min(2 * t, tokens - 1)], s1 = sm.scale[half][sub * tokens + min(2 * t + 1, tokens - 1)];
        float block_sum[2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) block_sum[m][i] = 0.0f;
        float (&acc)[2][4] = PARTS == 1 ? block_sum : total;
        const int first = half == 0 ? 0 : half0, count = half == 0 ? half0 : chunks - half0;
        if (ok) {  // one loop per code width
          const __half* x = xs + (sub * tokens + min(g, tokens - 1)) * X_PITCH + first * CHUNK + 16 * t;
          const auto run = [&](auto nbits, auto small) {
            return multiply<PARTS, decltype(nbits)::value, decltype(small)::value>(ring, x, count, first_word, pair_unit, rows, s0, s1, acc,
                                                                                   &sm.abort, status, refill);
          };
          typedef std::integral_constant<int, 2> Int2;
          typedef std::integral_constant<int, 4> Int4;
          typedef std::integral_constant<int, 8> Int8;
          if (form.width() == 1) ok = form.small_steps() ? run(Int2(), std::true_type()) : run(Int2(), std::false_type());
          else if (form.width() == 2) ok = form.small_steps() ? run(Int4(), std::true_type()) : run(Int4(), std::false_type());
          else if (form.width() == 3) ok = form.small_steps() ? run(Int8(), std::true_type()) : run(Int8(), std::false_type());
        }
#pragma unroll
        for (int m = 0; m < 2 && PARTS == 1; ++m) {
          total[m][0] += acc[m][0] * s0, total[m][1] += acc[m][1] * s1;
          total[m][2] += acc[m][2] * s0, total[m][3] += acc[m][3] * s1;
        }
      }
    }
    prepared = true;  // all of them: a run of several tiles is only made where they fit
    if (more && ok) {  // the next tile's data sets out while this one's sums are joined
      form = next_form;
      begin_stream();
      load_rows(row_tile + 1);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) sm.sums[half][2 * t + (i & 1)][quarter * 32 + 16 * m + 8 * (i >> 1) + g] = total[m][i];
    __syncthreads();
    if (split > 1) cluster_sync();
    const uint32_t here = s32(&sm.sums[0][0][0]);
    for (int i = rank * THREADS + threadIdx.x; i < tokens * TILE_ROWS; i += split * THREADS) {
      const int token = i / TILE_ROWS, row = i % TILE_ROWS;
      const uint32_t off = (uint32_t)(token * SUM_PITCH + row) * 4, other = FEW_WIDTH * SUM_PITCH * 4;
      float v[2 * MAX_SPLIT];
      if (split > 1) {
#pragma unroll
        for (int q = 0; q < MAX_SPLIT; ++q)
          if (q < split) {
            const uint32_t there = in_rank(here, q) + off;
            v[2 * q] = load_cluster(there), v[2 * q + 1] = load_cluster(there + other);
          }
      } else {
        v[0] = sm.sums[0][token][row], v[1] = sm.sums[1][token][row];
      }
      float sum = 0.0f;
#pragma unroll
      for (int q = 0; q < MAX_SPLIT; ++q)
        if (q < split) sum += v[2 * q] + v[2 * q + 1];
      const int64_t at = tile.begin + token;
      if (p.out.pair_weight != nullptr) sum *= p.out.pair_weight[p.tiles.pair(at)];
      const uint32_t col = sm.out_row[row];
      if (col != NO_ROW) p.out.put(at, col, sum);
    }
    if (split > 1) cluster_sync();  // nobody reads this block's sums any more
    else __syncthreads();
    if (!more) break;
  }
  if (__syncthreads_or(!ok)) let_copies_land();
}

template <int PARTS>
int launch(const Product& p, const FewPlan& plan, cudaStream_t stream, const char* what) {
  const size_t smem = smem_bytes<PARTS>();
  if (!reserve_smem<few_kernel<PARTS>>())
    return fail(HI2_ERR_LAUNCH, "stored product: cannot reserve shared memory");
  const int64_t blocks = (int64_t)plan.runs * p.max_tiles * plan.split;
  if (blocks >= (int64_t)1 << 31) return fail(HI2_ERR_ARG, "stored product: too many tiles");
  cudaLaunchConfig_t config = {};
  config.gridDim = (unsigned)blocks, config.blockDim = THREADS, config.dynamicSmemBytes = smem, config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  attribute[1].id = cudaLaunchAttributeClusterDimension;
  attribute[1].val.clusterDim.x = plan.split, attribute[1].val.clusterDim.y = 1, attribute[1].val.clusterDim.z = 1;
  config.attrs = attribute, config.numAttrs = 2;
  cudaLaunchKernelEx(&config, few_kernel<PARTS>, p, plan.split, plan.runs);
  return check_launch(what);
}

}  // namespace

// Slices of the columns and runs of row tiles: what leaves the fullest SM the least work, with what a tile costs besides its
// chunks (start of its stream, the join) counted as eight of them, three more through a cluster, and what a block costs
// (start, activations) as twelve.  The two blocks of an SM share its pipes: a run that is longer than the mean may have a
// shorter one beside it.  Measured, us: 28672 x 8192, one row, whole columns in 224 blocks 39.9, two slices in 148 runs 40.8, in
// 112 runs 41.0; 64 tokens of 64 experts of 2048 x 1024 with both products in runs of six tiles 131, of three 143, of one 172.
FewPlan few_plan(int64_t k, int64_t row_tiles, int64_t tiles, int64_t width, int parts) {
  const int64_t chunks = k / CHUNK, room = 2 * 148;
  const int places = parts == 1 ? PLACES<1> : PLACES<2>;
  FewPlan plan{1, 1, 1e300};
  for (int s = 1; s <= MAX_SPLIT && (s == 1 || chunks >= 4 * s); ++s) {
    const int64_t slice = ceil_div(chunks, (int64_t)s);
    const bool fits = width * ceil_div(slice, (int64_t)BLOCK_CHUNKS) <= places;  // activations stay for a run of tiles
    for (int r = 1; r == 1 || (fits && r <= 16 && r <= row_tiles); ++r) {
      int64_t runs = ceil_div(row_tiles, (int64_t)r);
      const int64_t waves = ceil_div(runs * tiles * s, room), most = waves * room / (tiles * s);
      if (runs < most) runs = most < row_tiles ? most : row_tiles;
      const double run = 0.75 * (double)ceil_div(row_tiles, runs) + 0.25 * (double)row_tiles / (double)runs;
      const double cost = (double)waves * (run * (double)(slice + (s == 1 ? 8 : 11)) + 12);
      if (cost < plan.cost) plan = FewPlan{s, (int)runs, cost};
    }
  }
  return plan;
}

// Of a stack: about as many as there will be, with half of every expert's last one empty.
int64_t few_tiles(int64_t experts, int64_t rows) { return rows / FEW_WIDTH + experts / 2 + 1; }

int product_few(const Product& p, cudaStream_t stream, const char* what) {
  const int64_t width = p.tiles.width < p.tiles.rows ? p.tiles.width : p.tiles.rows;
  const int64_t tiles = p.tiles.count != nullptr ? few_tiles(p.w.experts, p.tiles.rows) : p.max_tiles;
  const FewPlan plan = few_plan(p.w.k, p.w.groups_per_expert / 4, tiles, width, p.parts);
  return p.parts == 1 ? launch<1>(p, plan, stream, what) : launch<2>(p, plan, stream, what);
}

}  // namespace stored
}  // namespace hi2
