// The product of packed rows with many activation rows (prompts, large batches), on CTA pairs.
//
//     D[r, t] = sum_k V[r, k] xs[t, k]        256 sorted rows x up to 192 activation rows per pair
//
// The packed rows are the A operand, kept in tensor memory: a lane decodes the 64 weights of ITS row in a
// chunk of 64 columns (stored.cuh) and writes them as 32 fp16 pairs into its tensor-memory lane (tcgen05.st),
// so decoded weights never pass through shared memory.  The activations are the B operand, K-major boxes of 64
// columns that TMA brings into 128-byte-swizzled shared memory; each block of a pair loads half of a
// tile's activation rows and both halves serve both blocks (cta_group::2), which halves what a block
// asks of the L2: with one block per tile that is 64 bytes per clock at the full rate of the tensor pipe, as much as
// an SM can take.  One thread of the leading block issues the products, M = 256: its block's 128 rows accumulate in its
// tensor memory, the other 128 in its peer's.
//
// Blocks stay for many tiles.  Warps 0..7 decode (warp w: rows 32 (w mod 4) .. of the block's tile, one half of the
// columns), every warp with its own ring of bulk copies that runs on into the next tile; warp 8 loads activations, warp 9
// issues; warps 10..13 take finished tiles out of one of two accumulators (of the tile's width, up to 192 columns) while the
// next tile is computed in the other; behind them are two to four slots of 2 x 32 columns for decoded chunks.  A step is one
// chunk of each half of the columns, in a fixed order: equal inputs give equal bits.
//
// What bounds it: 2048 rows of bf16 x 11008 x 4096 take 212 us, of which the product kernel has 197 with the tensor pipe
// 42 % and issue 44 % busy, and no memory above a quarter.  With two slots the decoding of a step and its products do not
// fully overlap: without the decoding 176 us, without the epilogue 185, without both 145.  With short sums the epilogue
// shows: 32768 pairs of experts of 2048 x 1024 take 850 us, without it 667; its stores of 32 rows of a format touch 11.5
// sectors each, and an SM passes about one per clock.  Measured and dropped: sixteen decoding warps (the same); the
// outputs turned to column order in shared memory first (213 -> 209 us and 850 -> 910: the extra exchange costs four
// warps more than the sectors); eight epilogue warps (96 registers, which spill).
//
// Every mbarrier wait is bounded by a clock limit and raises *status.
#include <cuda.h>

#include <type_traits>

#include "stored_async.cuh"

namespace hi2 {
namespace stored {
namespace {

constexpr int DECODE_WARPS = 8, X_WARP = 8, MMA_WARP = 9, FIRST_EPILOGUE = 10, EPILOGUE_WARPS = 4;
constexpr int THREADS = 32 * (FIRST_EPILOGUE + EPILOGUE_WARPS);
constexpr int MAX_WIDTH = 192, MAX_EXACT_WIDTH = 128;
// Columns of a product for that many activation rows: with A in tensor memory a pair of blocks takes 32, 64, .. of them.
__host__ __device__ constexpr int product_columns(int rows) { return (rows + 31) & ~31; }
static_assert(MAX_WIDTH % 32 == 0 && MAX_EXACT_WIDTH % 32 == 0, "tiles are whole steps of a product's columns");
constexpr int EXACT_STEPS = 1;  // of a sum that the tensor cores form for an fp32 result
constexpr int MAX_SLOTS = 4, A_COLUMNS = CHUNK / 2, SLOT_COLUMNS = 2 * A_COLUMNS;
constexpr int RING_STAGES = 2, RING_BYTES = 3 * 1024;  // a stage: four chunks of INT2, two of INT4, one of INT8
constexpr int MAX_X_STAGES = 6;

struct Control {
  unsigned long long x_full[MAX_X_STAGES], x_empty[MAX_X_STAGES];
  unsigned long long a_full[MAX_SLOTS], a_empty[MAX_SLOTS];
  unsigned long long d_full[2], d_empty[2];
  unsigned long long ring_full[DECODE_WARPS][RING_STAGES];
  alignas(16) float scale[EPILOGUE_WARPS][MAX_WIDTH];
  uint32_t tmem_base;
  volatile uint32_t abort;
};

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// What these arrivals order is tensor memory, which the fences before and after them do.  A release at cluster
// scope would wait for everything else the thread has in flight: from a step to its products 1200 clocks, so 190.
__device__ __forceinline__ void bar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// One box into this block's shared memory; the bytes are counted by the leader's barrier.
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar_cluster_addr, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(s32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster_addr), "r"(x), "r"(y)
      : "memory");
}
// K-major 128-byte-swizzled operand: rows of 128 B, 8-row groups 1024 B apart.
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t saddr) {
  uint64_t d = (uint64_t)((saddr & 0x3ffffu) >> 4);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// kind::f16, A (fp16) from tensor memory, B (fp16) K-major from shared memory, D fp32.
__device__ __forceinline__ void mma_pair(uint32_t d_tmem, uint32_t a_tmem, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
}
// One lane of a converged warp.  (The compiler keeps a branch on this uniform, with descriptors in uniform registers;
// behind `lane == 0` every operand of every product is moved there first.)
__device__ __forceinline__ bool elected() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
// Arrives on the barrier at this offset in BOTH blocks once the products issued so far have finished.
__device__ __forceinline__ void commit_both(unsigned long long* b) {
  const unsigned short mask = 3;
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(s32(b)), "h"(mask)
      : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
      "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const float (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]),
      "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
      : "memory");
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// The lane's row (8 r + g of its group) in a chunk: what it reads, and its 64 weights as 32 pairs of neighbouring
// columns.  The next chunk's words are asked for before the present one's weights are handed on.
struct LaneRow {
  float lo_min[2], lo_scale[2];  // twice the same: two pieces are decoded together
  __half2 step_scale;
};
template <int NBITS>
struct RawRow {
  uint32_t words[2 * NBITS], pairs[2];
  __device__ __forceinline__ void load(const uint8_t* slab, int g, int r, int shift) {
    const uint16_t* from = reinterpret_cast<const uint16_t*>(slab + 256 * NBITS) + 4 * ((4 >> shift) * g) + r;
#pragma unroll
    for (int t = 0; t < 4; t += 2)
      pairs[t / 2] = (uint32_t)from[4 * (t >> shift)] | (uint32_t)from[4 * ((t + 1) >> shift)] << 16;
    const uint32_t* at = reinterpret_cast<const uint32_t*>(slab) + r;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int h = 0; h < NBITS / 2; ++h) words[NBITS / 2 * t + h] = at[128 * h + code_word(g, t)];
  }
  template <bool SMALL>
  __device__ __forceinline__ void expand(const LaneRow& row, uint32_t (&w)[32]) const {
#pragma unroll
    for (int t = 0; t < 4; t += 2) {
      Ladder l[2];
      ladders<NBITS, SMALL>(pairs[t / 2], row.lo_min, row.lo_scale, row.step_scale, l[0], l[1]);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int h = 0; h < NBITS / 2; ++h) decode_word<NBITS, SMALL>(words[NBITS / 2 * (t + u) + h], l[u], w + 8 * (t + u) + 16 / NBITS * h);
    }
  }
};

// One warp's packed data of one item.
struct Stream {
  const uint8_t* src;
  int slab, per_copy, chunks, copies;
};

// A decoding warp's place in its ring and among the slots of decoded chunks.
struct Decoder {
  Control* ctl;
  int32_t* status;
  const uint8_t* ring;
  unsigned long long* ring_full;
  uint32_t tmem;                // of this warp in the first slot
  uint32_t a_full;              // the leading block's first barrier
  int g, r, lane, slots;
  int stage, slot;
  uint32_t phase, slot_phase;
  __device__ __forceinline__ bool wait_ring() { return __all_sync(0xffffffffu, bar_wait(ring_full + stage, phase, &ctl->abort, status)); }
  // The weights (STORE: there are some) into the next slot, and word of it to the leading block.
  __device__ __forceinline__ bool hand_on(const uint32_t (&w)[32], bool store) {
    if (!__all_sync(0xffffffffu, bar_wait(&ctl->a_empty[slot], slot_phase, &ctl->abort, status))) return false;
    fence_after();
    if (store) tmem_store32(tmem + slot * SLOT_COLUMNS, w);
    fence_before();
    __syncwarp();
    if (lane == 0) bar_arrive_cluster(a_full + 8 * slot);
    if (++slot == slots) slot = 0, slot_phase ^= 1;
    return true;
  }
};
// The `count` steps of an item; the last of them lacks this warp's chunk where s.chunks is smaller.  False when a wait ran out.
template <int NBITS, bool SMALL, typename PRODUCE>
__device__ __forceinline__ bool steps(Decoder& d, const Stream& s, int shift, const LaneRow& row, int count, const PRODUCE& produce) {
  constexpr int PER_COPY = 8 / NBITS;
  uint32_t w[32];
  RawRow<NBITS> raw;
  int in_copy = 0;
  if (s.chunks > 0) {
    if (!d.wait_ring()) return false;
    raw.load(d.ring + d.stage * RING_BYTES, d.g, d.r, shift);
  }
  for (int i = 0; i < s.chunks; ++i) {
    raw.template expand<SMALL>(row, w);
    if (++in_copy == PER_COPY || i == s.chunks - 1) {
      in_copy = 0;
      __syncwarp();  // every lane has read the stage
      if (d.lane == 0) produce();
      __syncwarp();
      if (++d.stage == RING_STAGES) d.stage = 0, d.phase ^= 1;
      if (i < s.chunks - 1 && !d.wait_ring()) return false;
    }
    if (i < s.chunks - 1) raw.load(d.ring + d.stage * RING_BYTES + in_copy * s.slab, d.g, d.r, shift);
    if (!d.hand_on(w, true)) return false;
  }
  for (int i = s.chunks; i < count; ++i)
    if (!d.hand_on(w, false)) return false;
  return true;
}
// Rows of padding only: zeros.
__device__ __forceinline__ bool empty_steps(Decoder& d, int chunks, int count) {
  uint32_t w[32];
#pragma unroll
  for (int q = 0; q < 32; ++q) w[q] = 0;
  for (int i = 0; i < count; ++i)
    if (!d.hand_on(w, i < chunks)) return false;
  return true;
}

struct Shape {
  int width;       // activation rows of a tile, a multiple of 32
  int x_stages;
  int slots;       // of decoded chunks
  int splits;      // slices of the columns
  int row_pairs;   // pairs of tiles of packed rows
  int chunks, half0;  // of the columns; of their first half (a step takes a chunk of each)
};

// What one item of work is: a tile of activation rows, two tiles of packed rows, a slice of the columns.
struct Item {
  TokenTile tile;
  int row_tile;    // of this block; may lie behind the last one
  int slice, first, count;  // its first step, and its steps
};
__device__ __forceinline__ bool get_item(const Product& p, const Shape& shape, int64_t item, uint32_t rank, Item& out) {
  const int64_t rest = item / shape.row_pairs;
  out.slice = (int)(rest % shape.splits);
  if (!p.tiles.get(rest / shape.splits, out.tile)) return false;
  out.row_tile = (int)(item % shape.row_pairs) * 2 + (int)rank;
  out.first = shape.half0 * out.slice / shape.splits;
  out.count = shape.half0 * (out.slice + 1) / shape.splits - out.first;
  return true;
}
// Chunks of the second half in an item: the last step of an odd number of chunks lacks one.
__device__ __forceinline__ int second_chunks(const Shape& shape, const Item& item) {
  return min(item.count, shape.chunks - shape.half0 - item.first);
}

__device__ __forceinline__ GroupForm group_form(const Product& p, const Item& item, int quarter) {
  if (item.row_tile >= (int)(p.w.groups_per_expert / 4)) return GroupForm{0, 0};
  return load_group(p.w.groups, (int64_t)item.tile.expert * p.w.groups_per_expert + item.row_tile * 4 + quarter);
}
__device__ __forceinline__ Stream stream_of(const Product& p, const Shape& shape, const Item& item, GroupForm form, int half) {
  Stream s;
  s.slab = form.slab_bytes(), s.per_copy = 8 >> form.width();
  s.chunks = half == 0 ? item.count : second_chunks(shape, item);
  s.copies = s.slab == 0 ? 0 : (s.chunks + s.per_copy - 1) / s.per_copy;
  s.src = static_cast<const uint8_t*>(p.w.data) + (int64_t)form.base * 16 + (int64_t)(item.first + (half == 0 ? 0 : shape.half0)) * s.slab;
  return s;
}

// f of 16 values, its code four times over instead of sixteen.
template <typename F>
__device__ __forceinline__ void each(float (&v)[16], const F& f) {
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    float a = f(v[0]), b = f(v[1]), c = f(v[2]), d = f(v[3]);
#pragma unroll
    for (int t = 0; t < 12; ++t) v[t] = v[t + 4];  // registers move, no index varies
    v[12] = a, v[13] = b, v[14] = c, v[15] = d;
  }
}
// Column `col` of 16 activation rows from `row` on, of which `count` exist.
template <typename T>
__device__ __forceinline__ void read_rows(const void* p, int64_t ld, int64_t row, uint32_t col, int count, float (&v)[16]) {
  const T* from = static_cast<const T*>(p) + row * ld + col;
#pragma unroll
  for (int t = 0; t < 16; ++t, from += ld) v[t] = t < count ? to_float(*from) : 0.0f;
}
template <typename T>
__device__ __forceinline__ void write_rows(void* p, int64_t ld, int64_t row, uint32_t col, int count, const float (&v)[16]) {
  T* to = static_cast<T*>(p) + row * ld + col;
#pragma unroll
  for (int t = 0; t < 16; ++t, to += ld)
    if (t < count) *to = from_float<T>(v[t]);
}
// What follows the product for them.  (One activation's code at a time, none of it repeated for types or rows: the
// decoding warps' loops share the instruction cache with this.)
__device__ __forceinline__ void put_rows(const Epilogue& out, float (&v)[16], int64_t row, uint32_t col, int count, float bias) {
  float res[16];
  if (out.residual != nullptr) {
    if (out.dtype == HI2_BF16) read_rows<__nv_bfloat16>(out.residual, out.ld_residual, row, col, count, res);
    else if (out.dtype == HI2_F16) read_rows<__half>(out.residual, out.ld_residual, row, col, count, res);
    else read_rows<float>(out.residual, out.ld_residual, row, col, count, res);
  }
  if (out.bias != nullptr) {
#pragma unroll
    for (int t = 0; t < 16; ++t) v[t] += bias;
  }
  switch (out.act) {
    case HI2_ACT_RELU:
#pragma unroll
      for (int t = 0; t < 16; ++t) v[t] = activate(v[t], HI2_ACT_RELU);
      break;
    case HI2_ACT_SILU:
#pragma unroll
      for (int t = 0; t < 16; ++t) v[t] = activate(v[t], HI2_ACT_SILU);
      break;
    case HI2_ACT_GELU: each(v, [](float x) { return activate(x, HI2_ACT_GELU); }); break;
    case HI2_ACT_GELU_TANH: each(v, [](float x) { return activate(x, HI2_ACT_GELU_TANH); }); break;
    default: break;
  }
  if (out.residual != nullptr) {
#pragma unroll
    for (int t = 0; t < 16; ++t) v[t] += res[t];
  }
  if (out.dtype == HI2_BF16) write_rows<__nv_bfloat16>(out.out, out.ld_out, row, col, count, v);
  else if (out.dtype == HI2_F16) write_rows<__half>(out.out, out.ld_out, row, col, count, v);
  else write_rows<float>(out.out, out.ld_out, row, col, count, v);
}

// EXACT: fp32 results.  The tensor cores' accumulator drops what does not fit it at every step, always towards zero,
// which over 2048 columns costs 2e-6 of a result.  So a sum there covers one step of 128 columns, small parts first, and the
// epilogue's warps add the sums up in fp32, in tensor memory of their own.  Measured (2048 rows x 11008 x 4096; error of
// 512 tokens through experts of 1024 x 512, where a plain fp32 product has 9.3e-7): one step 428 us, 5.4e-7; two 345 us,
// 1.3e-6; four 325 us, 3.0e-6; slices of the columns joined through memory 1361 us.
template <bool EXACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
wide_kernel(const __grid_constant__ CUtensorMap map, const Product p, const Shape shape) {
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int box_bytes = shape.width / 2 * CHUNK * 2;    // one chunk of one part: this block's half of the rows
  const int stage_bytes = 2 * p.parts * box_bytes;
  uint8_t* rings = smem + (size_t)shape.x_stages * stage_bytes;
  Control* ctl = reinterpret_cast<Control*>(rings + DECODE_WARPS * RING_STAGES * RING_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  int32_t* const status = p.w.status;

  if (threadIdx.x == 0) {
    for (int s = 0; s < shape.x_stages; ++s) bar_init(&ctl->x_full[s], 1), bar_init(&ctl->x_empty[s], 1);
    for (int s = 0; s < MAX_SLOTS; ++s) bar_init(&ctl->a_full[s], 2 * DECODE_WARPS), bar_init(&ctl->a_empty[s], 1);
    for (int b = 0; b < 2; ++b) bar_init(&ctl->d_full[b], 1), bar_init(&ctl->d_empty[b], 2 * EPILOGUE_WARPS);
    for (int w = 0; w < DECODE_WARPS; ++w)
      for (int s = 0; s < RING_STAGES; ++s) bar_init(&ctl->ring_full[w][s], 1);
    ctl->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&ctl->tmem_base)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  cluster_sync();  // the peer's barriers exist before anything signals them
  fence_after();
  const uint32_t tmem = ctl->tmem_base;
  const uint32_t d_columns = (uint32_t)shape.width;
  const uint32_t s_tmem = tmem + 2 * d_columns;  // behind the two accumulators: sums of several, for fp32 results
  const uint32_t a_tmem = s_tmem + (EXACT ? d_columns : 0);
  const int64_t first_item = blockIdx.x >> 1, stride = gridDim.x >> 1;
  // Only the warps that touch what the preparation of the activations writes, or the outputs, wait for it.  The tile list
  // was complete before that one began.
  bool ok = true;
  Item item;

  if (warp < DECODE_WARPS) {
    // ------------------------------------------------------------ decode
    const int quarter = warp & 3, half = warp >> 2, g = lane & 7, r = lane >> 3;
    uint8_t* ring = rings + warp * RING_STAGES * RING_BYTES;
    // the ring is filled ahead of the item being decoded, by one lane with a cursor of its own
    int64_t ahead_item = first_item;
    int ahead_copy = 0, ahead_stage = 0;
    Stream ahead{nullptr, 0, 1, 0, 0};
    bool more = get_item(p, shape, ahead_item, rank, item);
    if (more) ahead = stream_of(p, shape, item, group_form(p, item, quarter), half);
    auto produce = [&]() {
      while (more && ahead_copy == ahead.copies) {
        ahead_item += stride, ahead_copy = 0;
        Item next;
        more = get_item(p, shape, ahead_item, rank, next);
        if (more) ahead = stream_of(p, shape, next, group_form(p, next, quarter), half);
      }
      if (!more) return;
      const int from = ahead_copy * ahead.per_copy, bytes = min(ahead.per_copy, ahead.chunks - from) * ahead.slab;
      bar_expect(&ctl->ring_full[warp][ahead_stage], (uint32_t)bytes);
      bulk_load(ring + ahead_stage * RING_BYTES, ahead.src + (int64_t)from * ahead.slab, (uint32_t)bytes, &ctl->ring_full[warp][ahead_stage]);
      ahead_stage = ahead_stage + 1 == RING_STAGES ? 0 : ahead_stage + 1;
      ++ahead_copy;
    };
    if (lane == 0)
      for (int s = 0; s < RING_STAGES; ++s) produce();
    Decoder out{ctl, status, ring, ctl->ring_full[warp], a_tmem + half * A_COLUMNS + ((uint32_t)(quarter * 32) << 16),
                in_rank(s32(&ctl->a_full[0]), 0), g, r, lane, shape.slots, 0, 0, 0, 1};
    for (int64_t at = first_item; ok && get_item(p, shape, at, rank, item); at += stride) {
      const GroupForm form = group_form(p, item, quarter);
      const Stream s = stream_of(p, shape, item, form, half);
      LaneRow row{};
      if (s.slab != 0) {
        const RowConsts c = load_row(p.w.rows, ((int64_t)item.tile.expert * p.w.groups_per_expert + item.row_tile * 4 + quarter) * GROUP_ROWS + lane);
        row.lo_min[0] = row.lo_min[1] = c.lo_min(), row.lo_scale[0] = row.lo_scale[1] = c.lo_scale();
        row.step_scale = __half2half2(__ushort_as_half((uint16_t)c.step_scale));
      }
      const auto run = [&](auto nbits, auto small) {
        return steps<decltype(nbits)::value, decltype(small)::value>(out, s, form.shift(), row, item.count, produce);
      };
      typedef std::integral_constant<int, 2> Int2;
      typedef std::integral_constant<int, 4> Int4;
      typedef std::integral_constant<int, 8> Int8;
      if (form.width() == 1) ok = form.small_steps() ? run(Int2(), std::true_type()) : run(Int2(), std::false_type());
      else if (form.width() == 2) ok = form.small_steps() ? run(Int4(), std::true_type()) : run(Int4(), std::false_type());
      else if (form.width() == 3) ok = form.small_steps() ? run(Int8(), std::true_type()) : run(Int8(), std::false_type());
      else ok = empty_steps(out, s.chunks, item.count);
    }
  } else if (warp == X_WARP) {
    // ------------------------------------------------------------ activations
    chain_wait();
    int stage = 0;
    uint32_t phase = 1;
    for (int64_t at = first_item; ok && get_item(p, shape, at, rank, item); at += stride) {
      const int cols = product_columns(item.tile.end - item.tile.begin);
      const int y = item.tile.begin + (int)rank * (cols / 2);
      const int second = second_chunks(shape, item);
      for (int i = 0; i < item.count; ++i) {
        ok = __all_sync(0xffffffffu, bar_wait(&ctl->x_empty[stage], phase, &ctl->abort, status));
        if (!ok) break;
        if (lane == 0) {
          const bool two = i < second;
          const int chunk = item.first + i;
          if (rank == 0) bar_expect(&ctl->x_full[stage], (uint32_t)((two ? 2 : 1) * p.parts * box_bytes * 2));  // both blocks' bytes
          const uint32_t full = in_rank(s32(&ctl->x_full[stage]), 0);
          uint8_t* dst = smem + (size_t)stage * stage_bytes;
          for (int part = 0; part < p.parts; ++part) {
            tma_load_pair(dst + part * box_bytes, &map, full, chunk * CHUNK, (int)(part * p.tiles.rows) + y);
            if (two) tma_load_pair(dst + (p.parts + part) * box_bytes, &map, full, (shape.half0 + chunk) * CHUNK, (int)(part * p.tiles.rows) + y);
          }
        }
        __syncwarp();
        if (++stage == shape.x_stages) stage = 0, phase ^= 1;
      }
    }
  } else if (warp == MMA_WARP && rank == 0) {
    // ------------------------------------------------------------ products (leading block only)
    const uint32_t d_first = __shfl_sync(0xffffffffu, tmem, 0), a_first = __shfl_sync(0xffffffffu, a_tmem, 0);
    const uint64_t b_first = desc_kmajor(s32(smem));
    const uint32_t box = (uint32_t)box_bytes >> 4;
    int stage = 0, slot = 0, buf = 0;
    uint32_t phase = 0, slot_phase = 0, d_phase = 1;
    for (int64_t at = first_item; ok && get_item(p, shape, at, rank, item); at += stride) {
      const int cols = product_columns(item.tile.end - item.tile.begin);
      // fp16 operands (format 0 at bits 7 and 10), fp32 accumulator (1 << 4), N >> 3 at bit 17, M >> 4 at bit 24
      const uint32_t idesc = (1u << 4) | ((uint32_t)(cols >> 3) << 17) | ((uint32_t)(2 * TILE_ROWS >> 4) << 24);
      const int second = second_chunks(shape, item);
      int in_sum = 0;
      for (int i = 0; i < item.count; ++i) {
        if (in_sum == 0) {
          ok = __all_sync(0xffffffffu, bar_wait(&ctl->d_empty[buf], d_phase, &ctl->abort, status));
          if (!ok) break;
        }
        const bool last = (EXACT && in_sum + 1 == EXACT_STEPS) || i == item.count - 1;
        const uint32_t d = d_first + buf * d_columns;
        const uint32_t a = a_first + slot * SLOT_COLUMNS;
        const uint64_t b = b_first + (uint32_t)(stage * stage_bytes >> 4);
        ok = bar_wait(&ctl->x_full[stage], phase, &ctl->abort, status);
        ok = ok && bar_wait(&ctl->a_full[slot], slot_phase, &ctl->abort, status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after();
        if (elected()) {
          uint32_t accumulate = in_sum > 0 ? 1u : 0u;
          for (int part = p.parts - 1; part >= 0; --part) {  // small parts first
#pragma unroll
            for (int kk = 0; kk < CHUNK / 16; ++kk) mma_pair(d, a + kk * 8, b + part * box + kk * 2, idesc, kk > 0 ? 1u : accumulate);
            accumulate = 1;
            if (i < second) {
#pragma unroll
              for (int kk = 0; kk < CHUNK / 16; ++kk) mma_pair(d, a + A_COLUMNS + kk * 8, b + (p.parts + part) * box + kk * 2, idesc, 1u);
            }
          }
          commit_both(&ctl->a_empty[slot]);
          commit_both(&ctl->x_empty[stage]);
          if (last) commit_both(&ctl->d_full[buf]);
        }
        __syncwarp();
        if (++stage == shape.x_stages) stage = 0, phase ^= 1;
        if (++slot == shape.slots) slot = 0, slot_phase ^= 1;
        ++in_sum;
        if (last) {
          in_sum = 0;
          if (++buf == 2) buf = 0, d_phase ^= 1;
        }
      }
    }
  } else if (warp >= FIRST_EPILOGUE) {
    // ------------------------------------------------------------ epilogue
    chain_wait();
    // a warp may only touch the 32 tensor-memory lanes of its index modulo 4
    const int quarter = warp & 3;
    int buf = 0;
    uint32_t phase = 0;
    for (int64_t at = first_item; ok && get_item(p, shape, at, rank, item); at += stride) {
      uint32_t col = NO_ROW;
      if (item.row_tile < (int)(p.w.groups_per_expert / 4))
        col = load_row(p.w.rows, ((int64_t)item.tile.expert * p.w.groups_per_expert + item.row_tile * 4 + quarter) * GROUP_ROWS + lane).out_row;
      const float bias = p.out.bias != nullptr && col != NO_ROW ? load_as_float(p.out.bias, p.out.dtype, col) : 0.0f;
      const int tokens = item.tile.end - item.tile.begin;
      float* scale = ctl->scale[warp - FIRST_EPILOGUE];  // of the activation rows; read while the tile is computed
      __syncwarp();
      for (int t = lane; t < tokens; t += 32) {
        scale[t] = p.row_scale[item.tile.begin + t];
        if (p.out.pair_weight != nullptr) scale[t] *= p.out.pair_weight[p.tiles.pair(item.tile.begin + t)];
      }
      __syncwarp();
      Epilogue out = p.out;
      if (shape.splits > 1) out.out = static_cast<float*>(out.out) + (int64_t)item.slice * p.tiles.rows * out.ld_out;
      const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
      const int sums = !EXACT ? 1 : (item.count + EXACT_STEPS - 1) / EXACT_STEPS;
      for (int i = 0; i < sums - 1; ++i) {  // sums that do not end the item are added up behind the accumulators
        ok = __all_sync(0xffffffffu, bar_wait(&ctl->d_full[buf], phase, &ctl->abort, status));
        if (!ok) break;
        fence_after();
#pragma unroll 1
        for (int t0 = 0; t0 < tokens; t0 += 16) {
          float v[16], sum[16];
          tmem_load16(tmem + buf * d_columns + lanes + t0, v);
          if (i > 0) {
            tmem_load16(s_tmem + lanes + t0, sum);
#pragma unroll
            for (int t = 0; t < 16; ++t) v[t] += sum[t];
          }
          tmem_store16(s_tmem + lanes + t0, v);
        }
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive_cluster(in_rank(s32(&ctl->d_empty[buf]), 0));
        if (++buf == 2) buf = 0, phase ^= 1;
      }
      if (!ok) break;
      ok = __all_sync(0xffffffffu, bar_wait(&ctl->d_full[buf], phase, &ctl->abort, status));
      if (!ok) break;
      fence_after();
      const uint32_t taddr = tmem + buf * d_columns + lanes;
#pragma unroll 1
      for (int t0 = 0; t0 < tokens; t0 += 16) {
        float v[16];
        tmem_load16(taddr + t0, v);
        if (EXACT && sums > 1) {
          float sum[16];
          tmem_load16(s_tmem + lanes + t0, sum);
#pragma unroll
          for (int t = 0; t < 16; ++t) v[t] += sum[t];
        }
#pragma unroll
        for (int t = 0; t < 16; t += 4) {
          const float4 f = *reinterpret_cast<const float4*>(scale + t0 + t);
          v[t] *= f.x, v[t + 1] *= f.y, v[t + 2] *= f.z, v[t + 3] *= f.w;
        }
        if (col != NO_ROW) put_rows(out, v, item.tile.begin + t0, col, min(16, tokens - t0), bias);
        __syncwarp();  // the next read of tensor memory is the whole warp's
      }
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive_cluster(in_rank(s32(&ctl->d_empty[buf]), 0));
      if (++buf == 2) buf = 0, phase ^= 1;
    }
  }
  __syncwarp();

  fence_before();
  if (__syncthreads_or(ctl->abort != 0)) let_copies_land();
  cluster_sync();  // neither block leaves while its peer may still signal it or read its operands
  if (warp == MMA_WARP) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// The slices' sums in order, and what follows the product.
__global__ void __launch_bounds__(256)
join_kernel(const float* __restrict__ partial, int splits, int64_t rows, int64_t n, const Epilogue out) {
  chain_wait();
  const int64_t values = rows * n;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < values; i += (int64_t)gridDim.x * blockDim.x) {
    float sum = 0.0f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) sum += partial[s * values + i];
    out.put(i / n, (uint32_t)(i % n), sum);
  }
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                             const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static EncodeFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<EncodeFn>(ptr);
  }();
  return fn;
}

}  // namespace

// Slices of the columns, for tiles that are fewer than the SM pairs: the number that leaves the busiest pair the fewest
// steps, with start and end of an item counted as six of them; each at least four steps.  Of a stack always one.
int wide_splits(int64_t k, int64_t rows_of_tensor, int64_t max_tiles, bool stack) {
  const int64_t items = (ceil_div(rows_of_tensor, (int64_t)TILE_ROWS) + 1) / 2 * max_tiles, count = (k / CHUNK + 1) / 2;
  int best = 1;
  int64_t least = INT64_MAX;
  for (int s = 1; s <= 16 && (s == 1 || (!stack && count >= 4 * s)); ++s) {
    const int64_t cost = ceil_div(items * s, (int64_t)74) * (ceil_div(count, (int64_t)s) + 6);
    if (cost < least) least = cost, best = s;
  }
  return best;
}

int wide_width(int64_t rows, bool exact) {
  const int64_t tiles = ceil_div(rows, (int64_t)(exact ? MAX_EXACT_WIDTH : MAX_WIDTH));
  return product_columns((int)ceil_div(rows, tiles));
}

int product_wide(const Product& p, cudaStream_t stream, const char* what) {
  EncodeFn enc = encoder();
  if (enc == nullptr) return fail(HI2_ERR_DRIVER, "stored product: cuTensorMapEncodeTiled unavailable");
  Shape s;
  s.width = p.tiles.width;
  const int stage_bytes = 2 * p.parts * (s.width / 2) * CHUNK * 2;
  s.x_stages = 144 * 1024 / stage_bytes;  // at least three
  if (s.x_stages > MAX_X_STAGES) s.x_stages = MAX_X_STAGES;
  s.slots = (512 - (p.exact ? 3 : 2) * s.width) / SLOT_COLUMNS;  // at least two
  if (s.slots > MAX_SLOTS) s.slots = MAX_SLOTS;
  s.chunks = (int)(p.w.k / CHUNK), s.half0 = (s.chunks + 1) / 2;
  s.row_pairs = (int)((p.w.groups_per_expert / 4 + 1) / 2);
  s.splits = wide_splits(p.w.k, p.w.rows_per_expert, p.max_tiles, p.tiles.index != nullptr);
  size_t smem = (size_t)s.x_stages * stage_bytes + DECODE_WARPS * RING_STAGES * RING_BYTES + sizeof(Control) + 1024;
  // A block takes all of an SM's tensor memory: two must never be resident on one SM.
  if (smem < 120 * 1024) smem = 120 * 1024;
  Product q = p;
  if (s.splits > 1) {  // plain sums of the slices; joined below
    q.out = Epilogue{};
    q.out.out = p.partial, q.out.ld_out = p.w.rows_per_expert, q.out.dtype = HI2_F32;
  }

  CUtensorMap map;
  const cuuint64_t dims[2] = {(cuuint64_t)p.w.k, (cuuint64_t)(p.tiles.rows * p.parts)};
  const cuuint64_t strides[1] = {(cuuint64_t)p.w.k * 2};
  const cuuint32_t box[2] = {CHUNK, (cuuint32_t)(s.width / 2)};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, p.xs, dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
    return HI2_ERR_DRIVER;
  }
  if (!(p.exact ? reserve_smem<wide_kernel<true>>() : reserve_smem<wide_kernel<false>>()))
    return fail(HI2_ERR_LAUNCH, "stored product: cannot reserve shared memory");
  constexpr int sms = 148;
  const int64_t items = (int64_t)s.row_pairs * s.splits * p.max_tiles;
  cudaLaunchConfig_t config = {};
  config.gridDim = (unsigned)(2 * (items < sms / 2 ? items : sms / 2));
  config.blockDim = THREADS, config.dynamicSmemBytes = smem, config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute, config.numAttrs = 1;
  cudaLaunchKernelEx(&config, p.exact ? wide_kernel<true> : wide_kernel<false>, map, q, s);
  const int rc = check_launch(what);
  if (rc != HI2_OK || s.splits == 1) return rc;
  const int64_t values = p.tiles.rows * p.w.rows_per_expert;
  const int64_t blocks = ceil_div(values, (int64_t)256);
  launch_link(join_kernel, dim3((unsigned)(blocks < 148 * 8 ? blocks : 148 * 8)), dim3(256), 0, stream, p.partial, s.splits, p.tiles.rows,
              p.w.rows_per_expert, p.out);
  return check_launch(what);
}

}  // namespace stored
}  // namespace hi2
