// Products of activations with packed weights (hi2/format.py:242-249 reference_linear) and the routed
// experts of a mixture layer over stacks of them: layout of the rows, preparation of the activations,
// dispatch of (token, slot) pairs to experts, and the entry points.
//
// A product is y = act(x' V^T + bias) + residual with V the format's fp16 weights, exactly as stored, and x' the
// activations in the stored basis: divided by the smoothing vector and rotated by the order-16 Hadamard matrix
// in the flagged groups.  x' is formed in fp32 and rounded to fp16 once, relative to a power of two that
// takes the largest value of the row (in the kernel for few rows: of each half of a block of 1024 columns) to
// [2^14, 2^15): 11 bits for every value within 2^-29 of that.  bf16 calls take that one part; fp16 and fp32 calls
// take a second part, fp16(x' - first), and twice the products.
#include <initializer_list>

#include "stored.cuh"

namespace hi2 {
namespace stored {
namespace {

// ---- layout -----------------------------------------------------------------------------------------
// One thread moves one row's 64 columns: codes into their words, parameter pairs behind them.  Its own format follows
// from the length of its code words and pairs; the group's form may be wider, with shorter blocks.
__global__ void __launch_bounds__(256)
lay_out_kernel(const hi2_stored_weight w, const int32_t* __restrict__ src_row, const int32_t* __restrict__ codes,
               const int32_t* __restrict__ code_off, const uint8_t* __restrict__ blk_params,
               const int32_t* __restrict__ param_off, uint8_t* __restrict__ data, int64_t n_rows) {
  const int64_t chunks = w.k / CHUNK;
  const int64_t total = n_rows * chunks;
  for (int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; id < total; id += (int64_t)gridDim.x * blockDim.x) {
    const int64_t chunk = id / n_rows, i = id % n_rows;  // neighbouring threads: rows of one slab
    const int32_t src = src_row[i];
    const GroupForm form = load_group(w.groups, i / GROUP_ROWS);
    if (src < 0 || form.width() == 0) continue;
    const int g = (int)(i & 7), r = (int)(i >> 3 & 3);
    uint8_t* slab = data + (int64_t)form.base * 16 + chunk * form.slab_bytes();
    const int nbits = 1 << form.width(), per_word = 32 / nbits, per_piece = nbits / 2;
    const int own_words = (int)((code_off[src + 1] - code_off[src]) / chunks);  // of a chunk: two per bit of a code
    const int own_bits = own_words / 2, own_pairs = (int)((param_off[src + 1] - param_off[src]) / chunks);
    const uint32_t mask = (1u << own_bits) - 1u;
    const int32_t* words = codes + code_off[src] + chunk * own_words;
    for (int q = 0; q < 2 * nbits; ++q) {
      uint32_t fields = 0;
      for (int f = 0; f < per_word; ++f) {
        const int bit = (q * per_word + f) * own_bits;
        fields |= ((uint32_t)words[bit >> 5] >> (bit & 31) & mask) << ((f >> 1) * nbits + (f & 1) * 16);
      }
      reinterpret_cast<uint32_t*>(slab)[128 * (q % per_piece) + code_word(g, q / per_piece) + r] = fields;
    }
    const int pairs = 4 >> form.shift();
    const uint8_t* from = blk_params + 2 * ((int64_t)param_off[src] + chunk * own_pairs);
    uint8_t* to = slab + form.code_bytes();
    for (int t = 0; t < pairs; ++t) {
      const int unit = 4 * (pairs * g + t) + r, own = t * own_pairs / pairs;
      to[2 * unit] = from[2 * own], to[2 * unit + 1] = from[2 * own + 1];
    }
  }
}

// ---- activations of wide products ---------------------------------------------------------------------
// A team of warps per activation row: largest value, then the fp16 parts relative to its power of two.  A
// lane keeps HOLD pieces of 16 columns in registers; HOLD = 0 forms them twice.
template <int THREADS, int WARPS, int HOLD, int PARTS>
__global__ void __launch_bounds__(THREADS)
prepare_kernel(const Product p, const int32_t* __restrict__ used) {
  chain_wait();
  chain_next();  // the product sets up and decodes its first chunks meanwhile; never before the wait: it goes by the tile list at once
  constexpr int TEAM = WARPS * 32;
  const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
  const int64_t row = (int64_t)blockIdx.x * (THREADS / TEAM) + team;
  if (row >= (used == nullptr ? p.tiles.rows : (int64_t)*used)) return;  // a team of several warps is the whole block
  int64_t from = row;
  int expert = 0;
  if (p.tiles.index != nullptr) {
    const int pair = (int)p.tiles.pair(row);
    expert = (int)p.tiles.index[pair];
    if (p.from.kind != FROM_GATED) from = (uint32_t)pair / (uint32_t)p.from.top_k;
  }
  const int groups = (int)(p.w.k / 16);
  constexpr int KEEP = HOLD == 0 ? 1 : HOLD;
  float v[KEEP][16];
  float top = 0.0f;
  if (HOLD > 0) {
#pragma unroll
    for (int h = 0; h < KEEP; ++h)
      if (lane + h * TEAM < groups) {
        stored_basis(p.from, p.w, from, expert, lane + h * TEAM, v[h]);
        top = fmaxf(top, largest(v[h]));
      }
  } else {
    for (int g = lane; g < groups; g += TEAM) {
      stored_basis(p.from, p.w, from, expert, g, v[0]);
      top = fmaxf(top, largest(v[0]));
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (WARPS > 1) {
    __shared__ float warp_top[WARPS];
    if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WARPS; ++i) top = fmaxf(top, warp_top[i]);
  }
  // (the power of a row that a (token, slot) pair's weight follows is multiplied by it: room for 16 bits below)
  const PowerOfTwo power = power_for(top, p.out.pair_weight != nullptr ? -110 : -126);
  if (lane == 0) p.row_scale[row] = power.back;
  auto store = [&](int g, const float (&x)[16]) {
    uint4 hi[2], lo[2];
    split16<PARTS>(x, power.to, hi, lo);
    uint4* dst = reinterpret_cast<uint4*>(p.xs + row * p.w.k + (int64_t)g * 16);
    dst[0] = hi[0], dst[1] = hi[1];
    if (PARTS == 2) {
      dst = reinterpret_cast<uint4*>(p.xs + (p.tiles.rows + row) * p.w.k + (int64_t)g * 16);
      dst[0] = lo[0], dst[1] = lo[1];
    }
  };
  if (HOLD > 0) {
#pragma unroll
    for (int h = 0; h < KEEP; ++h)
      if (lane + h * TEAM < groups) store(lane + h * TEAM, v[h]);
  } else {
    for (int g = lane; g < groups; g += TEAM) {
      stored_basis(p.from, p.w, from, expert, g, v[0]);
      store(g, v[0]);
    }
  }
}

template <int THREADS, int WARPS, int HOLD>
void launch_prepare(const Product& p, const int32_t* used, cudaStream_t stream) {
  const unsigned grid = (unsigned)ceil_div(p.tiles.rows, (int64_t)(THREADS / 32 / WARPS));
  launch_link(p.parts == 1 ? prepare_kernel<THREADS, WARPS, HOLD, 1> : prepare_kernel<THREADS, WARPS, HOLD, 2>, dim3(grid),
              dim3(THREADS), 0, stream, p, used);
}
// Two warps per row where the rows fill the machine (32768 rows of 2048 columns: 65 us, one warp with four pieces per lane
// 80); else a block per row, one piece per thread as far as that goes (32 rows of 11008 columns: 14 us with 128
// threads, which form everything twice).
int prepare(const Product& p, const int32_t* used, cudaStream_t stream) {
  const int64_t pieces = p.w.k / 16;
  if (pieces <= 128 && p.tiles.rows >= 148 * 16) launch_prepare<64, 2, 2>(p, used, stream);
  else if (pieces <= 128) launch_prepare<128, 4, 1>(p, used, stream);
  else if (pieces <= 512) launch_prepare<512, 16, 1>(p, used, stream);
  else if (pieces <= 1024) launch_prepare<512, 16, 2>(p, used, stream);
  else launch_prepare<512, 16, 0>(p, used, stream);
  return check_launch("stored: activations");
}

// ---- dispatch -----------------------------------------------------------------------------------------
// Counting sort of the (token, slot) pairs by expert: one block counts and makes the list of token tiles, then many place
// the pairs.  Pairs of one expert come in no particular order: a row's result does not depend on its place, so the outputs
// are the same every time.  The products read the index and the tile list before they
// wait for the kernel ahead of them: both kernels here must have ended before that one releases its dependents, as it does after a
// wait of its own.  (One block for both, keeping the order by matching the lanes of a warp, took 36 us for 32768
// pairs, without the order 26 us: its scattered stores all go through one SM.)
constexpr int SORT_THREADS = 1024, SORT_BATCH = 8;
constexpr int MAX_EXPERTS = 1024;

__device__ __forceinline__ int expert_of(const int64_t* index, int64_t pair, int64_t pairs, int experts) {
  const int64_t e = pair < pairs ? index[pair] : -1;
  return e >= 0 && e < experts ? (int)e : -1;
}

__global__ void __launch_bounds__(SORT_THREADS)
count_kernel(const int64_t* __restrict__ index, int64_t pairs, int experts, int tile_width, int32_t* __restrict__ next_row,
             int32_t* __restrict__ used, int32_t* __restrict__ tile_count, TokenTile* __restrict__ tiles) {
  __shared__ int32_t counts[MAX_EXPERTS];
  __shared__ int32_t warp_sums[2][SORT_THREADS / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  counts[threadIdx.x] = 0;
  __syncthreads();
  for (int64_t i = threadIdx.x; i < pairs; i += SORT_THREADS * SORT_BATCH) {
    int e[SORT_BATCH];  // several at a time: a load takes most of a microsecond
#pragma unroll
    for (int b = 0; b < SORT_BATCH; ++b) e[b] = expert_of(index, i + SORT_THREADS * b, pairs, experts);
#pragma unroll
    for (int b = 0; b < SORT_BATCH; ++b)
      if (e[b] >= 0) atomicAdd(counts + e[b], 1);
  }
  __syncthreads();
  // thread e: the expert's total, its first row and its first tile (exclusive sums over the experts)
  const int e = threadIdx.x;
  const int32_t total = counts[e];
  const int32_t own_tiles = (total + tile_width - 1) / tile_width;
  int32_t rows_to = total, tiles_to = own_tiles;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int32_t a = __shfl_up_sync(0xffffffffu, rows_to, d), b = __shfl_up_sync(0xffffffffu, tiles_to, d);
    if (lane >= d) rows_to += a, tiles_to += b;
  }
  if (lane == 31) warp_sums[0][warp] = rows_to, warp_sums[1][warp] = tiles_to;
  __syncthreads();
  for (int v = 0; v < warp; ++v) rows_to += warp_sums[0][v], tiles_to += warp_sums[1][v];
  if (threadIdx.x == SORT_THREADS - 1) *used = rows_to, *tile_count = tiles_to;
  const int32_t begin = rows_to - total;
  if (e < experts) next_row[e] = begin;
  for (int t = 0; t < own_tiles; ++t) {
    const int b = begin + t * tile_width;
    tiles[tiles_to - own_tiles + t] = TokenTile{e, b, b + tile_width < rows_to ? b + tile_width : rows_to};
  }
}

// A block reserves rows for its pairs of every expert at once, and hands them out.
constexpr int PLACE_PAIRS = 2048;
__global__ void __launch_bounds__(SORT_THREADS)
place_kernel(const int64_t* __restrict__ index, int64_t pairs, int experts, int32_t* __restrict__ next_row, int32_t* __restrict__ pair_of,
             int32_t* __restrict__ row_of) {
  __shared__ int32_t next[MAX_EXPERTS];
  constexpr int EACH = PLACE_PAIRS / SORT_THREADS;
  const int64_t first = (int64_t)blockIdx.x * PLACE_PAIRS + threadIdx.x;
  next[threadIdx.x] = 0;
  __syncthreads();
  chain_wait();
  int e[EACH], place[EACH];
#pragma unroll
  for (int b = 0; b < EACH; ++b) e[b] = expert_of(index, first + SORT_THREADS * b, pairs, experts);
#pragma unroll
  for (int b = 0; b < EACH; ++b) place[b] = e[b] >= 0 ? atomicAdd(next + e[b], 1) : 0;
  __syncthreads();
  if (next[threadIdx.x] > 0) next[threadIdx.x] = atomicAdd(next_row + threadIdx.x, next[threadIdx.x]);
  __syncthreads();
#pragma unroll
  for (int b = 0; b < EACH; ++b) {
    const int64_t at = first + SORT_THREADS * b;
    if (at >= pairs) continue;
    const int32_t row = e[b] >= 0 ? next[e[b]] + place[b] : -1;
    if (row >= 0) pair_of[row] = (int32_t)at;
    row_of[at] = row;
  }
}

// out[t] = sum of the token's weighted rows in slot order (a fixed order: the same bits every time).
__global__ void __launch_bounds__(256)
combine_kernel(const float* __restrict__ y, const int32_t* __restrict__ row_of, const int64_t* __restrict__ index,
               int experts, int64_t tokens, int top_k, int64_t hidden, void* __restrict__ out, int dtype, int64_t ld_out) {
  chain_wait();
  const int64_t quads = hidden / 4, total = tokens * quads;
  for (int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; id < total; id += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = id / quads, c = id % quads * 4;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int j = 0; j < top_k; ++j) {
      const int64_t pair = t * top_k + j;
      int64_t row = pair;
      if (row_of != nullptr) row = row_of[pair];
      else if (index[pair] < 0 || index[pair] >= experts) row = -1;
      if (row < 0) continue;
      const float4 v = *reinterpret_cast<const float4*>(y + (int64_t)row * hidden + c);
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    const int64_t at = t * ld_out + c;
    store_float(out, dtype, at, sum.x), store_float(out, dtype, at + 1, sum.y);
    store_float(out, dtype, at + 2, sum.z), store_float(out, dtype, at + 3, sum.w);
  }
}

inline size_t pad256(size_t n) { return (n + 255) & ~(size_t)255; }

// Carves the caller's workspace.
struct Carver {
  uint8_t* at;
  size_t used = 0;
  template <typename T>
  T* take(size_t n) {
    T* p = at == nullptr ? nullptr : reinterpret_cast<T*>(at + used);
    used += pad256(n * sizeof(T));
    return p;
  }
};

// One part for bf16 calls: what 11 bits leave out lies below the rounding of a bf16 result.  Measured, one part / two: errors of
// 512 tokens through experts of 1024 x 512 against 64 bits 1.69e-3 / 1.65e-3 (1.65e-3 is the rounding of the exact result);
// 2048 tokens x 11008 x 4096 212 / 271 us, 4096 tokens through 64 experts of 2048 x 1024 870 / 1105, 64 tokens 130 / 179, one token
// x 28672 x 8192 40 / 52.  fp16 results (11 bits themselves) would show it, fp32 results all the more.
inline int parts_of(int dtype) { return dtype == HI2_BF16 ? 1 : 2; }
// Which kernel takes a product: the one for few rows up to 16 of them, and as long as its tiles of eight are little work (it
// is one launch where the other takes three).  Measured, few / wide, us (and cost): 256 tokens x 512 x 512 8.7 / 15.4
// (27), 77 x 1001 x 1088 in fp32 11.8 / 16.9 (29), 64 x 2048 x 2048 12.8 / 17.4 (39), 24 x 4096 x 4096 19.5 / 19.0 (45),
// 64 x 4096 x 4096 34 / 22 (84); 111 pairs of 5 experts of 192 x 320 in fp32 25.1 / 32.8 (25).
constexpr double FEW_COST = 40;
inline bool few(const hi2_stored_weight& w, int64_t tokens, int parts) {
  return tokens <= 2 * FEW_WIDTH || few_plan(w.k, w.groups_per_expert / 4, ceil_div(tokens, (int64_t)FEW_WIDTH), FEW_WIDTH, parts).cost <= FEW_COST;
}
inline int64_t rows_per_expert(int64_t experts, int64_t pairs) {  // with half as many again as on average
  const int64_t busy = ceil_div(3 * pairs, 2 * experts);
  return busy < pairs ? busy : pairs;
}
inline bool few_experts(const hi2_stored_weight& gate_up, int64_t pairs, int parts) {  // both products, or neither
  if (rows_per_expert(gate_up.experts, pairs) <= 2 * FEW_WIDTH) return true;
  const int64_t tiles = few_tiles(gate_up.experts, pairs), hidden = gate_up.k, inner = gate_up.rows_per_expert / 2;
  return few_plan(hidden, ceil_div(2 * inner, (int64_t)TILE_ROWS), tiles, FEW_WIDTH, parts).cost <= FEW_COST &&
         few_plan(inner, ceil_div(hidden, (int64_t)TILE_ROWS), tiles, FEW_WIDTH, parts).cost <= FEW_COST;
}
inline bool apart(int64_t pairs) { return pairs <= FEW_WIDTH; }  // every pair a tile of its own

inline int64_t size_of(int dtype) { return dtype == HI2_F32 ? 4 : 2; }
inline bool rows_aligned(const void* p, int64_t ld, int dtype) { return aligned16(p) && ld * size_of(dtype) % 16 == 0; }
inline int kind_of(int dtype) { return dtype == HI2_BF16 ? FROM_BF16 : dtype == HI2_F16 ? FROM_F16 : FROM_F32; }

struct LinearSpace {
  __half* xs = nullptr;
  float *scale = nullptr, *partial = nullptr;
  int width = FEW_WIDTH;
  int64_t max_tiles;
  bool small;
  size_t bytes;
  LinearSpace(void* ws, const hi2_stored_weight& w, int dtype, int64_t tokens) : small(few(w, tokens, parts_of(dtype))) {
    Carver c{static_cast<uint8_t*>(ws)};
    if (!small) {
      xs = c.take<__half>((size_t)tokens * w.k * parts_of(dtype));
      scale = c.take<float>(tokens);
      width = wide_width(tokens, dtype == HI2_F32);
    }
    max_tiles = ceil_div(tokens, (int64_t)width);
    if (!small) {
      const int splits = wide_splits(w.k, w.rows_per_expert, max_tiles, false);
      if (splits > 1) partial = c.take<float>((size_t)splits * tokens * w.rows_per_expert);
    }
    bytes = c.used;
  }
};

struct ExpertSpace {
  __half* xs = nullptr;  // of the gate/up product, then of the down product
  float *scale = nullptr, *z, *y;
  int32_t *pair_of = nullptr, *row_of = nullptr, *next_row = nullptr, *used = nullptr, *tile_count = nullptr;
  TokenTile* tiles = nullptr;
  bool small;
  size_t bytes;
  ExpertSpace(void* ws, const hi2_stored_weight& gate_up, int dtype, int64_t tokens, int top_k)
      : small(few_experts(gate_up, tokens * top_k, parts_of(dtype))) {
    const size_t pairs = (size_t)tokens * top_k, hidden = gate_up.k, inner = gate_up.rows_per_expert / 2;
    Carver c{static_cast<uint8_t*>(ws)};
    z = c.take<float>(pairs * inner * 2);
    y = c.take<float>(pairs * hidden);
    if (!apart(pairs)) {
      used = c.take<int32_t>(64);
      tile_count = used == nullptr ? nullptr : used + 32;
      pair_of = c.take<int32_t>(pairs);
      row_of = c.take<int32_t>(pairs);
      next_row = c.take<int32_t>(gate_up.experts);
      tiles = c.take<TokenTile>(pairs / 8 + gate_up.experts + 1);
    }
    if (!small) {
      xs = c.take<__half>(pairs * (hidden > inner ? hidden : inner) * parts_of(dtype));
      scale = c.take<float>(pairs);
    }
    bytes = c.used;
  }
};

bool complete(const hi2_stored_weight* w) {
  return w != nullptr && w->data != nullptr && w->groups != nullptr && w->rows != nullptr && w->had != nullptr &&
         w->status != nullptr && w->experts > 0 && w->rows_per_expert > 0 && w->k > 0 && w->k % CHUNK == 0 &&
         w->groups_per_expert % 4 == 0 && w->groups_per_expert * GROUP_ROWS >= w->rows_per_expert;
}
bool known_dtype(int dtype) { return dtype == HI2_F32 || dtype == HI2_F16 || dtype == HI2_BF16; }

}  // namespace
}  // namespace stored
}  // namespace hi2

using namespace hi2;
using namespace hi2::stored;

extern "C" int hi2_lay_out_rows(const hi2_stored_weight* w, const int32_t* src_row, const int32_t* codes,
                                const int32_t* code_off, const uint8_t* blk_params, const int32_t* param_off, void* data,
                                void* stream) {
  HI2_REQUIRE(complete(w), "lay_out_rows: incomplete weight");
  HI2_REQUIRE(src_row && codes && code_off && blk_params && param_off && data, "lay_out_rows: null pointer");
  const int64_t n_rows = w->experts * w->groups_per_expert * GROUP_ROWS;
  int64_t blocks = ceil_div(n_rows * (w->k / CHUNK), (int64_t)256);
  if (blocks > 148 * 64) blocks = 148 * 64;
  lay_out_kernel<<<(unsigned)blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      *w, src_row, codes, code_off, blk_params, param_off, static_cast<uint8_t*>(data), n_rows);
  return check_launch("lay_out_rows");
}

extern "C" size_t hi2_stored_linear_workspace_bytes(const hi2_stored_weight* w, int dtype, int64_t tokens) {
  if (!complete(w) || !known_dtype(dtype) || tokens <= 0) return 0;
  return LinearSpace(nullptr, *w, dtype, tokens).bytes;
}

extern "C" int hi2_stored_linear(const hi2_stored_weight* w, const void* x, int dtype, int64_t tokens, int64_t ldx,
                                 const void* bias, int act, const void* residual, int64_t ld_residual, void* out,
                                 int64_t ld_out, void* workspace, size_t workspace_bytes, void* stream) {
  HI2_REQUIRE(complete(w), "stored_linear: incomplete weight");
  HI2_REQUIRE(w->experts == 1, "stored_linear: a stack of experts has no single product");
  HI2_REQUIRE(known_dtype(dtype), "stored_linear: activations must be fp32, fp16 or bf16");
  HI2_REQUIRE(act >= HI2_ACT_NONE && act <= HI2_ACT_GELU_TANH, "stored_linear: unknown activation");
  HI2_REQUIRE(tokens >= 0 && tokens < (int64_t)1 << 30, "stored_linear: too many tokens");
  if (tokens == 0) return HI2_OK;
  HI2_REQUIRE(x && out, "stored_linear: null pointer");
  const LinearSpace space(workspace, *w, dtype, tokens);
  if (space.bytes > 0 && (workspace == nullptr || workspace_bytes < space.bytes || !aligned16(workspace)))
    return fail(HI2_ERR_WORKSPACE, "stored_linear: workspace too small");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Product p{*w, Source{x, ldx, kind_of(dtype), HI2_ACT_NONE, rows_aligned(x, ldx, dtype), 1},
                  Tiles{nullptr, nullptr, nullptr, nullptr, tokens, 1, space.width}, space.max_tiles, parts_of(dtype),
                  Epilogue{nullptr, bias, residual, out, ld_residual, ld_out, act, dtype}, dtype == HI2_F32, false, space.xs, space.scale,
                  space.partial};
  if (space.small) return product_few(p, s, "stored_linear");
  const int rc = prepare(p, nullptr, s);
  return rc != HI2_OK ? rc : product_wide(p, s, "stored_linear");
}

extern "C" size_t hi2_stored_experts_workspace_bytes(const hi2_stored_weight* gate_up, int dtype, int64_t tokens, int top_k) {
  if (!complete(gate_up) || !known_dtype(dtype) || tokens <= 0 || top_k <= 0) return 0;
  return ExpertSpace(nullptr, *gate_up, dtype, tokens, top_k).bytes;
}

extern "C" int hi2_stored_experts(const hi2_stored_weight* gate_up, const hi2_stored_weight* down, const void* x, int dtype,
                                  int64_t tokens, int64_t ldx, const int64_t* index, const float* weight, int top_k, int act,
                                  void* out, int64_t ld_out, void* workspace, size_t workspace_bytes, void* stream) {
  HI2_REQUIRE(complete(gate_up) && complete(down), "stored_experts: incomplete weight");
  HI2_REQUIRE(gate_up->experts == down->experts && gate_up->k == down->rows_per_expert &&
                  gate_up->rows_per_expert == 2 * down->k,
              "stored_experts: the gate/up and down stacks do not fit each other");
  HI2_REQUIRE(gate_up->experts <= MAX_EXPERTS, "stored_experts: more than 1024 experts");
  HI2_REQUIRE(known_dtype(dtype), "stored_experts: activations must be fp32, fp16 or bf16");
  HI2_REQUIRE(act >= HI2_ACT_NONE && act <= HI2_ACT_GELU_TANH, "stored_experts: unknown activation");
  HI2_REQUIRE(tokens >= 0 && top_k >= 1 && tokens < (int64_t)1 << 30 &&
                  tokens * top_k < (int64_t)1 << 30, "stored_experts: too many (token, slot) pairs");
  if (tokens == 0) return HI2_OK;
  HI2_REQUIRE(x && index && weight && out, "stored_experts: null pointer");
  const ExpertSpace space(workspace, *gate_up, dtype, tokens, top_k);
  if (workspace == nullptr || workspace_bytes < space.bytes || !aligned16(workspace))
    return fail(HI2_ERR_WORKSPACE, "stored_experts: workspace too small");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t pairs = tokens * top_k, hidden = gate_up->k, inner = down->k;
  const int experts = (int)gate_up->experts, parts = parts_of(dtype);
  Tiles tiles{index, nullptr, nullptr, nullptr, pairs, experts, 1};
  int64_t max_tiles = pairs;
  int rc;
  if (!apart(pairs)) {
    const int64_t busy = rows_per_expert(experts, pairs);
    tiles = Tiles{index, space.pair_of, space.tile_count, space.tiles, pairs, experts, space.small ? FEW_WIDTH : wide_width(busy, dtype == HI2_F32)};
    max_tiles = pairs / tiles.width + experts + 1;
    count_kernel<<<1, SORT_THREADS, 0, s>>>(index, pairs, experts, tiles.width, space.next_row, space.used, space.tile_count, space.tiles);
    if ((rc = check_launch("stored_experts: dispatch")) != HI2_OK) return rc;
    launch_link(place_kernel, dim3((unsigned)ceil_div(pairs, (int64_t)PLACE_PAIRS)), dim3(SORT_THREADS), 0, s, index, pairs, experts,
                space.next_row, space.pair_of, space.row_of);
    if ((rc = check_launch("stored_experts: dispatch")) != HI2_OK) return rc;
  }
  const Product up{*gate_up, Source{x, ldx, kind_of(dtype), HI2_ACT_NONE, rows_aligned(x, ldx, dtype), top_k}, tiles, max_tiles, parts,
                   Epilogue{nullptr, nullptr, nullptr, space.z, 0, 2 * inner, HI2_ACT_NONE, HI2_F32}, dtype == HI2_F32, false, space.xs,
                   space.scale, nullptr};
  const Product dn{*down, Source{space.z, 2 * inner, FROM_GATED, act, true, top_k}, tiles, max_tiles, parts,
                   Epilogue{weight, nullptr, nullptr, space.y, 0, hidden, HI2_ACT_NONE, HI2_F32}, dtype == HI2_F32, true, space.xs,
                   space.scale, nullptr};
  for (const Product* p : {&up, &dn}) {
    if (space.small) {
      rc = product_few(*p, s, "stored_experts");
    } else {
      rc = prepare(*p, space.used, s);
      if (rc == HI2_OK) rc = product_wide(*p, s, "stored_experts");
    }
    if (rc != HI2_OK) return rc;
  }
  int64_t blocks = ceil_div(tokens * (hidden / 4), (int64_t)256);
  if (blocks > 148 * 16) blocks = 148 * 16;
  launch_link(combine_kernel, dim3((unsigned)blocks), dim3(256), 0, s, space.y, space.row_of, index, experts, tokens, top_k, hidden,
              out, dtype, ld_out);
  return check_launch("stored_experts: combine");
}
