// The product of packed rows with prepared activations on the tensor cores.
//
//     D[r, t] = sum_k V[r, k] xs[t, k]        128 sorted rows x up to 256 activation rows per block
//
// The packed rows are the A operand, kept in tensor memory: a lane decodes the 64 weights of ITS row in a
// chunk of 64 columns (stored.cuh) and writes them as 32 fp16 pairs into its tensor-memory lane
// (tcgen05.st), so decoded weights never pass through shared memory.  The activations are the B operand,
// K-major boxes of 64 columns that TMA brings into 128-byte-swizzled shared memory.  Per chunk four
// tcgen05.mma (128 x width x 16) accumulate in fp32; with two activation parts eight, into one accumulator.
//
// Block: warps 0..7 decode (warp w: rows 32 (w mod 4) .., one half of the block's chunks each), every warp
// with its own ring of bulk copies, so packed bytes stream without any barrier between warps; warp 8
// loads activations, warp 9 issues the products and takes the chunks alternately from the two halves (a fixed
// order: equal inputs give equal bits).  With few tiles the chunks are split over a cluster: each block adds
// its share, gives its tensor memory back, and the partial sums are joined through distributed shared
// memory in rank order.  No block waits for a peer while it holds tensor memory.
//
// Every mbarrier wait is bounded by a clock limit and raises *status.
#include <cuda.h>

#include "stored.cuh"

namespace hi2 {
namespace stored {
namespace {

constexpr int DECODE_WARPS = 8, X_WARP = 8, MMA_WARP = 9;
constexpr int THREADS = 320;
constexpr int MAX_WIDTH = 256;      // activation rows of a tile
constexpr int A_SLOTS = 4;          // decoded chunks in tensor memory: two per half
constexpr int A_COLUMNS = CHUNK / 2;
constexpr int RING_STAGES = 3;
constexpr int RING_BYTES = 2560;    // per stage: four chunks of the smallest format, at least one of any
constexpr int MAX_X_STAGES = 8;
constexpr int MAX_SPLIT = 8;
constexpr long long WAIT_CYCLES = 2000000000LL;  // about one second

struct Control {
  unsigned long long x_full[MAX_X_STAGES], x_empty[MAX_X_STAGES];
  unsigned long long a_full[A_SLOTS], a_empty[A_SLOTS];
  unsigned long long ring_full[DECODE_WARPS][RING_STAGES];
  unsigned long long done;
  uint32_t out_row[TILE_ROWS];
  uint32_t tmem_base;
  volatile uint32_t abort;
};

__device__ __forceinline__ uint32_t s32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(unsigned long long* b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s32(b)), "r"(n));
}
__device__ __forceinline__ void bar_expect(unsigned long long* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(s32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(unsigned long long* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s32(b)) : "memory");
}
__device__ __forceinline__ bool bar_try(unsigned long long* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(s32(b)), "r"(parity) : "memory");
  return ok != 0;
}
// False when the limit ran out or another role of this block gave up.
__device__ __forceinline__ bool bar_wait(unsigned long long* b, uint32_t parity, Control* ctl, int32_t* status) {
  if (bar_try(b, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    if (bar_try(b, parity)) return true;
    if (ctl->abort) return false;
    if (clock64() - t0 > WAIT_CYCLES) {
      ctl->abort = 1;
      atomicExch(status, HI2_ERR_TIMEOUT);
      return false;
    }
  }
}
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, unsigned long long* bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(s32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(s32(bar)), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, unsigned long long* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(s32(dst)), "l"(src), "r"(bytes), "r"(s32(bar)) : "memory");
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
__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint32_t a_tmem, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(db), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void commit_to(unsigned long long* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(s32(b)) : "memory");
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
__device__ __forceinline__ uint32_t in_rank(uint32_t local, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}
__device__ __forceinline__ float load_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct Shape {
  int width;       // activation rows of a tile, a multiple of 16
  int x_stages;
  int split;       // blocks of a cluster
  int columns;     // tensor memory
};

__global__ void __launch_bounds__(THREADS, 2)
product_kernel(const __grid_constant__ CUtensorMap map, const Product p, const Shape shape) {
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  const int x_bytes = shape.width * CHUNK * 2;          // one part of a stage
  uint8_t* rings = smem + (size_t)shape.x_stages * p.parts * x_bytes;
  Control* ctl = reinterpret_cast<Control*>(rings + DECODE_WARPS * RING_STAGES * RING_BYTES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)(blockIdx.x % shape.split);
  const int row_tiles = (int)(p.w.groups_per_expert / 4);
  const int row_tile = (int)(blockIdx.x / shape.split) % row_tiles;
  if (p.tiles.count != nullptr) chain_wait();  // the tile list comes from an earlier kernel of the chain
  TokenTile tile;
  if (!p.tiles.get(blockIdx.x / shape.split / row_tiles, tile)) return;  // the same for all blocks of a cluster
  int32_t* const status = p.w.status;

  if (threadIdx.x == 0) {
    for (int s = 0; s < shape.x_stages; ++s) bar_init(&ctl->x_full[s], 1), bar_init(&ctl->x_empty[s], 1);
    for (int s = 0; s < A_SLOTS; ++s) bar_init(&ctl->a_full[s], 4), bar_init(&ctl->a_empty[s], 1);
    for (int w = 0; w < DECODE_WARPS; ++w)
      for (int s = 0; s < RING_STAGES; ++s) bar_init(&ctl->ring_full[w][s], 1);
    bar_init(&ctl->done, 1);
    ctl->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&ctl->tmem_base)),
                 "r"(shape.columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = ctl->tmem_base;
  const uint32_t a_tmem = tmem + (uint32_t)((shape.width + 31) & ~31);

  // this block's chunks, the first half of them (rounded up) for warps 0..3
  const int all = (int)(p.w.k / CHUNK);
  const int c0 = (int)((int64_t)all * rank / shape.split), n = (int)((int64_t)all * (rank + 1) / shape.split) - c0;
  const int n_half0 = (n + 1) / 2;

  if (warp < DECODE_WARPS) {
    // ------------------------------------------------------------ decode
    const int quarter = warp & 3, half = warp >> 2;
    const int64_t group = (int64_t)tile.expert * p.w.groups_per_expert + row_tile * 4 + quarter;
    const RowForm row = load_row(p.w.rows, group * GROUP_ROWS + lane);
    if (half == 0) ctl->out_row[quarter * 32 + lane] = row.out_row;
    const float lo_min = __half2float(__ushort_as_half((uint16_t)row.lo_consts));
    const float lo_scale = __half2float(__ushort_as_half((uint16_t)(row.lo_consts >> 16)));
    const float step_scale = __half2float(__ushort_as_half((uint16_t)row.step_scale));
    const uint32_t slab = p.w.groups[2 * group + 1] * 16;  // bytes of a chunk; 0: padding only
    const int mine = half == 0 ? n_half0 : n - n_half0;
    const uint8_t* src = static_cast<const uint8_t*>(p.w.data) + (int64_t)p.w.groups[2 * group] * 16 +
                         (int64_t)(c0 + (half == 0 ? 0 : n_half0)) * slab;
    uint8_t* ring = rings + warp * RING_STAGES * RING_BYTES;
    const int per_copy = slab == 0 ? n + 1 : RING_BYTES / (int)slab;
    const int copies = slab == 0 ? 0 : (mine + per_copy - 1) / per_copy;
    auto issue = [&](int copy) {  // by one lane
      const int first = copy * per_copy, count = min(per_copy, mine - first), stage = copy % RING_STAGES;
      bar_expect(&ctl->ring_full[warp][stage], (uint32_t)count * slab);
      bulk_load(ring + stage * RING_BYTES, src + (int64_t)first * slab, (uint32_t)count * slab, &ctl->ring_full[warp][stage]);
    };
    if (lane == 0)
      for (int c = 0; c < RING_STAGES && c < copies; ++c) issue(c);
    int copy = 0, at = 0;
    for (int i = 0; i < mine; ++i) {
      const int stage = copy % RING_STAGES;
      if (slab != 0 && at == 0) {  // a warp gives up as a whole: what follows is executed by all of its lanes
        const bool here = bar_wait(&ctl->ring_full[warp][stage], (copy / RING_STAGES) & 1, ctl, status);
        if (!__all_sync(0xffffffffu, here)) break;
      }
      uint32_t v[CHUNK / 2];
      decode_chunk(ring + stage * RING_BYTES + at * slab, row, lo_min, lo_scale, step_scale, v);
      if (++at == per_copy) {
        at = 0;
        __syncwarp();  // every lane has read the stage
        if (lane == 0 && copy + RING_STAGES < copies) issue(copy + RING_STAGES);
        ++copy;
      }
      const int slot = 2 * half + (i & 1);
      const bool ok = bar_wait(&ctl->a_empty[slot], ((i >> 1) & 1) ^ 1, ctl, status);
      if (!__all_sync(0xffffffffu, ok)) break;
      fence_after();
      tmem_store32(a_tmem + slot * A_COLUMNS + ((uint32_t)(quarter * 32) << 16), v);
      fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(&ctl->a_full[slot]);
    }
  } else if (warp == X_WARP && lane == 0) {
    // ------------------------------------------------------------ activations
    chain_wait();
    for (int i = 0; i < n; ++i) {
      const int stage = i % shape.x_stages;
      if (!bar_wait(&ctl->x_empty[stage], ((i / shape.x_stages) & 1) ^ 1, ctl, status)) break;
      bar_expect(&ctl->x_full[stage], (uint32_t)(p.parts * x_bytes));
      const int chunk = c0 + (i >> 1) + ((i & 1) ? n_half0 : 0);
      uint8_t* dst = smem + (size_t)stage * p.parts * x_bytes;
      tma_load(dst, &map, &ctl->x_full[stage], chunk * CHUNK, tile.begin);
      if (p.parts == 2) tma_load(dst + x_bytes, &map, &ctl->x_full[stage], chunk * CHUNK, (int)p.x_rows + tile.begin);
    }
  } else if (warp == MMA_WARP && lane == 0) {
    // ------------------------------------------------------------ products
    // fp16 operands (format 0 at bits 7 and 10), fp32 accumulator (1 << 4), N >> 3 at bit 17, M >> 4 at bit 24
    const uint32_t idesc = (1u << 4) | ((uint32_t)(shape.width >> 3) << 17) | ((uint32_t)(TILE_ROWS >> 4) << 24);
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int stage = i % shape.x_stages, slot = 2 * (i & 1) + ((i >> 1) & 1);
      if (!(ok = bar_wait(&ctl->x_full[stage], (i / shape.x_stages) & 1, ctl, status))) break;
      if (!(ok = bar_wait(&ctl->a_full[slot], (i >> 2) & 1, ctl, status))) break;
      fence_after();
      const uint32_t sb = s32(smem + (size_t)stage * p.parts * x_bytes);
      for (int part = 0; part < p.parts; ++part)
#pragma unroll
        for (int kk = 0; kk < CHUNK / 16; ++kk)
          mma_f16(tmem, a_tmem + slot * A_COLUMNS + kk * 8, desc_kmajor(sb + part * x_bytes + kk * 32), idesc,
                  i > 0 || part > 0 || kk > 0 ? 1u : 0u);
      commit_to(&ctl->a_empty[slot]);
      commit_to(&ctl->x_empty[stage]);
    }
    if (ok) commit_to(&ctl->done);
  }
  __syncwarp();

  // ---------------------------------------------------------------- epilogue
  const int tokens = tile.end - tile.begin;
  if (warp < DECODE_WARPS) {
    const bool ok = bar_wait(&ctl->done, 0, ctl, status);
    if (__all_sync(0xffffffffu, ok)) {
      chain_wait();  // the row scales, and whatever the outputs overwrite
      fence_after();
      const int quarter = warp & 3, half = warp >> 2, r = quarter * 32 + lane;
      const uint32_t col = ctl->out_row[r];
      for (int t0 = half * 16; t0 < tokens; t0 += 32) {
        float v[16];
        tmem_load16(tmem + ((uint32_t)(quarter * 32) << 16) + t0, v);
        if (shape.split > 1) {
          float* partial = reinterpret_cast<float*>(smem);
#pragma unroll
          for (int t = 0; t < 16; ++t)
            if (t0 + t < tokens) partial[(t0 + t) * TILE_ROWS + r] = v[t];
        } else if (col != NO_ROW) {
#pragma unroll
          for (int t = 0; t < 16; ++t)
            if (t0 + t < tokens) {
              const int64_t at = tile.begin + t0 + t;
              p.out.put(at, col, p.out.scale_of(at), v[t]);
            }
        }
      }
      fence_before();
    }
  }
  const bool gave_up = __syncthreads_or(ctl->abort != 0);
  if (gave_up) {  // copies already issued still land in this block's shared memory: give them time
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) {
    }
  }
  if (warp == MMA_WARP) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(shape.columns) : "memory");
  }
  if (shape.split > 1) {
    cluster_sync();  // the partial sums of all blocks are there
    chain_wait();
    const uint32_t mine = s32(smem);
    for (int i = rank * THREADS + threadIdx.x; i < tokens * TILE_ROWS; i += shape.split * THREADS) {
      float sum = 0.0f;
      for (int q = 0; q < shape.split; ++q) sum += load_cluster(in_rank(mine, q) + i * 4);
      const uint32_t col = ctl->out_row[i % TILE_ROWS];
      const int64_t at = tile.begin + i / TILE_ROWS;
      if (col != NO_ROW) p.out.put(at, col, p.out.scale_of(at), sum);
    }
    cluster_sync();  // nobody reads this block's sums any more
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

int tile_width(int64_t tokens) {
  const int64_t tiles = ceil_div(tokens, (int64_t)MAX_WIDTH);
  return (int)(ceil_div(ceil_div(tokens, tiles), (int64_t)16) * 16);
}

int product(const Product& p, cudaStream_t stream, const char* what) {
  EncodeFn enc = encoder();
  if (enc == nullptr) return fail(HI2_ERR_DRIVER, "stored product: cuTensorMapEncodeTiled unavailable");
  Shape s;
  s.width = p.tiles.width;
  const int x_bytes = s.width * CHUNK * 2 * p.parts;
  s.x_stages = (s.width <= 128 ? 48 : 96) * 1024 / x_bytes;
  if (s.x_stages < 2) s.x_stages = 2;
  if (s.x_stages > MAX_X_STAGES) s.x_stages = MAX_X_STAGES;
  s.columns = ((s.width + 31) & ~31) + A_SLOTS * A_COLUMNS <= 256 ? 256 : 512;
  // few tiles: the chunks are split over a cluster until the blocks fill the SMs twice (once for wide tiles)
  const int64_t tiles = p.w.groups_per_expert / 4 * p.max_tiles, chunks = p.w.k / CHUNK;
  const int64_t room = s.columns == 256 ? 2 * 148 : 148;
  s.split = 1;
  while (s.split < MAX_SPLIT && tiles * s.split * 2 <= room && chunks >= s.split * 2 * 4) s.split *= 2;
  // At most two blocks of 256 columns, or one of 512, fit an SM's shared memory: then the tensor memory of
  // the blocks that can be resident together never runs out, and no allocation waits.
  const size_t least = s.columns == 256 ? 78 * 1024 : 160 * 1024;
  const size_t body = (size_t)s.x_stages * x_bytes + (size_t)DECODE_WARPS * RING_STAGES * RING_BYTES;
  if ((size_t)s.width * TILE_ROWS * sizeof(float) > body) s.split = 1;  // the partial sums take the place of the stages
  size_t smem = body + sizeof(Control) + 1024;
  if (smem < least) smem = least;

  CUtensorMap map;
  const cuuint64_t dims[2] = {(cuuint64_t)p.w.k, (cuuint64_t)(p.x_rows * p.parts)};
  const cuuint64_t strides[1] = {(cuuint64_t)p.w.k * 2};
  const cuuint32_t box[2] = {CHUNK, (cuuint32_t)s.width};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<__half*>(p.xs), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
    return HI2_ERR_DRIVER;
  }
  if (cudaFuncSetAttribute(product_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return fail(HI2_ERR_LAUNCH, "stored product: cannot reserve shared memory");
  cudaLaunchConfig_t config = {};
  if (tiles * s.split >= (int64_t)1 << 31) return fail(HI2_ERR_ARG, "stored product: too many tiles");
  config.gridDim = (unsigned)(tiles * s.split);
  config.blockDim = THREADS, config.dynamicSmemBytes = smem, config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  attribute[1].id = cudaLaunchAttributeClusterDimension;
  attribute[1].val.clusterDim.x = s.split, attribute[1].val.clusterDim.y = 1, attribute[1].val.clusterDim.z = 1;
  config.attrs = attribute, config.numAttrs = 2;
  cudaLaunchKernelEx(&config, product_kernel, map, p, s);
  return check_launch(what);
}

}  // namespace stored
}  // namespace hi2
