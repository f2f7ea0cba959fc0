// Products of activations with packed weights (hi2/format.py:242-249 reference_linear) and the routed
// experts of a mixture layer over stacks of them: layout of the rows, preparation of the activations,
// dispatch of (token, slot) pairs to experts, and the entry points.
//
// A product is y = act(x' V^T + bias) + residual with V the format's fp16 weights, exactly as stored, and x' the
// activations in the stored basis: divided by the smoothing vector and rotated by the order-16 Hadamard matrix
// in the flagged groups.  x' is formed in fp32 and rounded to fp16 once, relative to a power of two that
// takes the row's largest value to [2^14, 2^15): 11 bits for every value within 2^-29 of that.  bf16 calls
// (8 bits) take that one part; fp16 and fp32 calls take a second part, fp16(x' - first), and twice the products.
#include "stored.cuh"

namespace hi2 {
namespace stored {
namespace {

// ---- layout -----------------------------------------------------------------------------------------
// One thread moves one row's 64 columns: codes into their pieces, parameter pairs behind them.
__global__ void __launch_bounds__(256)
lay_out_kernel(const hi2_stored_weight w, const int32_t* __restrict__ src_row, const int32_t* __restrict__ codes,
               const int32_t* __restrict__ code_off, const uint8_t* __restrict__ blk_params,
               const int32_t* __restrict__ param_off, uint8_t* __restrict__ data, int64_t n_rows) {
  const int64_t chunks = w.k / CHUNK;
  const int64_t total = n_rows * chunks;
  for (int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; id < total; id += (int64_t)gridDim.x * blockDim.x) {
    const int64_t chunk = id / n_rows, i = id % n_rows;  // neighbouring threads: rows of one slab
    const int32_t src = src_row[i];
    const RowForm row = load_row(w.rows, i);
    if (src < 0 || row.width() == 0) continue;
    const int64_t g = i / GROUP_ROWS;
    uint8_t* slab = data + ((int64_t)w.groups[2 * g] + chunk * w.groups[2 * g + 1]) * 16;
    const int nbits = 1 << row.width();
    const uint32_t mask = (1u << nbits) - 1u;
    const int32_t* words = codes + code_off[src] + chunk * 2 * nbits;
    const int per_word = 32 / nbits;
    for (int q = 0; q < 2 * nbits; ++q) {  // word q of the chunk stays word q: only its fields move
      const uint32_t v = (uint32_t)words[q];
      uint32_t r = 0;
      for (int f = 0; f < per_word; ++f) r |= (v >> (f * nbits) & mask) << ((f >> 1) * nbits + (f & 1) * 16);
      uint32_t* piece = reinterpret_cast<uint32_t*>(slab) + 4 * (row.piece() + (q >> 2) * row.piece_stride());
      piece[q & 3] = r;
    }
    const int pairs = 4 >> row.block_shift();
    const uint8_t* from = blk_params + 2 * (param_off[src] + chunk * pairs);
    for (int b = 0; b < 2 * pairs; ++b) slab[row.params() + b] = from[b];
  }
}

// ---- activations ------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float as_float(T v);
template <>
__device__ __forceinline__ float as_float(float v) { return v; }
template <>
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ void load16(const T* p, bool vector, float (&v)[16]) {
  if (vector) {
    constexpr int PER = 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < 16 / PER; ++i) {
      const uint4 raw = *(reinterpret_cast<const uint4*>(p) + i);
      const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < PER; ++j) v[PER * i + j] = as_float(t[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = as_float(p[i]);
  }
}

struct Source {
  const void* x;         // [tokens, ldx], or the fp32 [rows, 2 k] result of the gate and up rows
  int64_t ldx;
  int act;               // of the gate rows
  bool vector;           // rows start on 16-byte boundaries
  const int32_t* pair_of;  // stack: row -> (token, slot) pair, else null
  const int64_t* index;  // stack: pair -> expert
  const int32_t* used;   // stack: number of rows in use
  int top_k;
};

// 16 columns of a row in the stored basis.  GATED: the row is act(gate) * up.
template <typename T, bool GATED>
__device__ __forceinline__ void stored_basis(const Source& s, const hi2_stored_weight& w, int64_t row, int64_t expert,
                                             int64_t g, float (&v)[16]) {
  if (GATED) {
    const float* z = static_cast<const float*>(s.x) + row * s.ldx + g * 16;
    float u[16];
    load16(z, true, v);
    load16(z + w.k, true, u);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = activate(v[i], s.act) * u[i];
  } else {
    load16(static_cast<const T*>(s.x) + row * s.ldx + g * 16, s.vector, v);
  }
  if (w.inv_scale != nullptr) {
    float c[16];
    load16(w.inv_scale + expert * w.k + g * 16, true, c);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] *= c[i];
  }
  if (w.had[expert * (w.k / 16) + g] != 0) {
#pragma unroll
    for (int span = 1; span < 16; span *= 2)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if ((i & span) == 0) {
          const float a = v[i], b = v[i + span];
          v[i] = a + b, v[i + span] = a - b;
        }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] *= 0.25f;
  }
}

constexpr int PREP_THREADS = 128;

// One block per activation row: largest value, then the fp16 parts relative to its power of two.
template <typename T, bool GATED>
__global__ void __launch_bounds__(PREP_THREADS)
prepare_kernel(const Source s, const hi2_stored_weight w, int64_t rows, int parts, __half* __restrict__ xs,
               float* __restrict__ row_scale) {
  const int64_t row = blockIdx.x;
  int64_t from = row, expert = 0;
  if (s.pair_of != nullptr) {
    if (row >= *s.used) return;
    const int32_t pair = s.pair_of[row];
    expert = s.index[pair];
    if (!GATED) from = pair / s.top_k;
  }
  const int64_t groups = w.k / 16;
  float top = 0.0f;
  for (int64_t g = threadIdx.x; g < groups; g += PREP_THREADS) {
    float v[16];
    stored_basis<T, GATED>(s, w, from, expert, g, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(v[i]));
  }
  __shared__ float warp_top[PREP_THREADS / 32];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PREP_THREADS / 32; ++i) top = fmaxf(top, warp_top[i]);
  const int biased = (int)(__float_as_uint(top) >> 23);
  int e = biased - 127 - 14;  // a row without values, or with an infinity: left as it is
  if (top == 0.0f || biased == 255) e = 0;
  if (e < -110) e = -110;     // 2^-e has to be an fp32 number
  const float to = __uint_as_float((uint32_t)(127 - e) << 23);
  if (threadIdx.x == 0) row_scale[row] = __uint_as_float((uint32_t)(127 + e) << 23);
  for (int64_t g = threadIdx.x; g < groups; g += PREP_THREADS) {
    float v[16];
    stored_basis<T, GATED>(s, w, from, expert, g, v);
    uint32_t hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = v[2 * i] * to, b = v[2 * i + 1] * to;
      const __half2 h = __floats2half2_rn(a, b);
      hi[i] = bits(h);
      lo[i] = bits(__floats2half2_rn(a - __low2float(h), b - __high2float(h)));
    }
    uint4* dst = reinterpret_cast<uint4*>(xs + row * w.k + g * 16);
    dst[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]), dst[1] = make_uint4(hi[4], hi[5], hi[6], hi[7]);
    if (parts == 2) {
      dst = reinterpret_cast<uint4*>(xs + (rows + row) * w.k + g * 16);
      dst[0] = make_uint4(lo[0], lo[1], lo[2], lo[3]), dst[1] = make_uint4(lo[4], lo[5], lo[6], lo[7]);
    }
  }
}

// ---- dispatch -----------------------------------------------------------------------------------------
// Stable counting sort of the (token, slot) pairs by expert in one block: every warp counts its stretch of
// the pairs (lanes that name the same expert find each other by a match), the counts are summed over
// the warps and experts, and every warp places its stretch.  Also the list of token tiles.
constexpr int SORT_WARPS = 32;
constexpr int MAX_EXPERTS = 1024;

__global__ void __launch_bounds__(SORT_WARPS * 32)
dispatch_kernel(const int64_t* __restrict__ index, int64_t pairs, int experts, int tile_width, int32_t* __restrict__ pair_of,
                int32_t* __restrict__ row_of, int32_t* __restrict__ used, int32_t* __restrict__ tile_count,
                TokenTile* __restrict__ tiles) {
  extern __shared__ int32_t counts[];  // [warps][experts]
  __shared__ int32_t warp_sums[2][SORT_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < SORT_WARPS * experts; i += blockDim.x) counts[i] = 0;
  __syncthreads();
  int32_t* mine = counts + warp * experts;
  const int64_t per = ceil_div(ceil_div(pairs, (int64_t)SORT_WARPS), (int64_t)32) * 32;
  const int64_t first = warp * per, last = first + per < pairs ? first + per : pairs;
  for (int64_t i = first; i < last; i += 32) {
    const int64_t e64 = i + lane < last ? index[i + lane] : -1;
    const int e = e64 >= 0 && e64 < experts ? (int)e64 : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  // thread e: the expert's total, its first row and its first tile (exclusive sums over the experts)
  const int e = threadIdx.x;
  int32_t total = 0;
  if (e < experts)
    for (int v = 0; v < SORT_WARPS; ++v) {
      const int32_t c = counts[v * experts + e];
      counts[v * experts + e] = total;
      total += c;
    }
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
  if (threadIdx.x == blockDim.x - 1) *used = rows_to, *tile_count = tiles_to;
  if (e < experts) {
    const int32_t begin = rows_to - total;
    for (int v = 0; v < SORT_WARPS; ++v) counts[v * experts + e] += begin;
    for (int t = 0; t < own_tiles; ++t) {
      const int b = begin + t * tile_width;
      tiles[tiles_to - own_tiles + t] = TokenTile{e, b, b + tile_width < rows_to ? b + tile_width : rows_to};
    }
  }
  __syncthreads();
  for (int64_t i = first; i < last; i += 32) {
    const bool in = i + lane < last;
    const int64_t e64 = in ? index[i + lane] : -1;
    const int x = e64 >= 0 && e64 < experts ? (int)e64 : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, x);
    if (x >= 0) {
      const int32_t row = mine[x] + __popc(same & ((1u << lane) - 1u));
      pair_of[row] = (int32_t)(i + lane);
      row_of[i + lane] = row;
    } else if (in) {
      row_of[i + lane] = -1;
    }
    __syncwarp();
    if (x >= 0 && lane == __ffs(same) - 1) mine[x] += __popc(same);
    __syncwarp();
  }
}

// out[t] = sum of the token's weighted rows in slot order (a fixed order: the same bits every time).
__global__ void __launch_bounds__(256)
combine_kernel(const float* __restrict__ y, const int32_t* __restrict__ row_of, int64_t tokens, int top_k, int64_t hidden,
               void* __restrict__ out, int dtype, int64_t ld_out) {
  const int64_t quads = hidden / 4, total = tokens * quads;
  for (int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; id < total; id += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = id / quads, c = id % quads * 4;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int j = 0; j < top_k; ++j) {
      const int32_t row = row_of[t * top_k + j];
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

inline int parts_of(int dtype) { return dtype == HI2_BF16 ? 1 : 2; }
inline int64_t size_of(int dtype) { return dtype == HI2_F32 ? 4 : 2; }
inline bool rows_aligned(const void* p, int64_t ld, int dtype) { return aligned16(p) && ld * size_of(dtype) % 16 == 0; }

struct LinearSpace {
  __half* xs;
  float* scale;
  size_t bytes;
  LinearSpace(void* ws, const hi2_stored_weight& w, int dtype, int64_t tokens) {
    Carver c{static_cast<uint8_t*>(ws)};
    xs = c.take<__half>((size_t)tokens * w.k * parts_of(dtype));
    scale = c.take<float>(tokens);
    bytes = c.used;
  }
};

struct ExpertSpace {
  __half *xs, *hs;
  float *x_scale, *h_scale, *z, *y;
  int32_t *pair_of, *row_of, *used, *tile_count;
  TokenTile* tiles;
  size_t bytes;
  ExpertSpace(void* ws, const hi2_stored_weight& gate_up, int dtype, int64_t tokens, int top_k) {
    const size_t pairs = (size_t)tokens * top_k, hidden = gate_up.k, inner = gate_up.rows_per_expert / 2;
    Carver c{static_cast<uint8_t*>(ws)};
    used = c.take<int32_t>(64);
    tile_count = used == nullptr ? nullptr : used + 32;
    pair_of = c.take<int32_t>(pairs);
    row_of = c.take<int32_t>(pairs);
    tiles = c.take<TokenTile>(pairs / 16 + gate_up.experts + 1);
    x_scale = c.take<float>(pairs);
    h_scale = c.take<float>(pairs);
    xs = c.take<__half>(pairs * hidden * parts_of(dtype));
    z = c.take<float>(pairs * inner * 2);
    hs = c.take<__half>(pairs * inner * parts_of(dtype));
    y = c.take<float>(pairs * hidden);
    bytes = c.used;
  }
};

template <bool GATED>
int prepare(const Source& s, const hi2_stored_weight& w, int dtype, int64_t rows, int parts, __half* xs, float* scale,
            cudaStream_t stream) {
  const unsigned grid = (unsigned)rows;
  if (dtype == HI2_BF16) prepare_kernel<__nv_bfloat16, GATED><<<grid, PREP_THREADS, 0, stream>>>(s, w, rows, parts, xs, scale);
  else if (dtype == HI2_F16) prepare_kernel<__half, GATED><<<grid, PREP_THREADS, 0, stream>>>(s, w, rows, parts, xs, scale);
  else prepare_kernel<float, GATED><<<grid, PREP_THREADS, 0, stream>>>(s, w, rows, parts, xs, scale);
  return check_launch("stored: activations");
}

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
  if (workspace == nullptr || workspace_bytes < space.bytes || !aligned16(workspace))
    return fail(HI2_ERR_WORKSPACE, "stored_linear: workspace too small");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Source src{x, ldx, HI2_ACT_NONE, rows_aligned(x, ldx, dtype), nullptr, nullptr, nullptr, 1};
  int rc = prepare<false>(src, *w, dtype, tokens, parts_of(dtype), space.xs, space.scale, s);
  if (rc != HI2_OK) return rc;
  const int width = tile_width(tokens);
  const Product p{*w, space.xs, tokens, parts_of(dtype), Tiles{nullptr, nullptr, tokens, width}, ceil_div(tokens, (int64_t)width),
                  Epilogue{space.scale, nullptr, nullptr, bias, residual, out, ld_residual, ld_out, act, dtype}};
  return product(p, s, "stored_linear");
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
  // tiles wide enough for an expert with half as many tokens again as the average one
  const int64_t busy = ceil_div(3 * pairs, (int64_t)(2 * experts));
  const int width = tile_width(busy < pairs ? busy : pairs);
  const size_t smem = (size_t)SORT_WARPS * experts * sizeof(int32_t);
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(dispatch_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return fail(HI2_ERR_LAUNCH, "stored_experts: cannot reserve shared memory");
  dispatch_kernel<<<1, SORT_WARPS * 32, smem, s>>>(index, pairs, experts, width, space.pair_of, space.row_of, space.used,
                                                  space.tile_count, space.tiles);
  int rc = check_launch("stored_experts: dispatch");
  if (rc != HI2_OK) return rc;
  Source src{x, ldx, HI2_ACT_NONE, rows_aligned(x, ldx, dtype), space.pair_of, index, space.used, top_k};
  rc = prepare<false>(src, *gate_up, dtype, pairs, parts, space.xs, space.x_scale, s);
  if (rc != HI2_OK) return rc;
  const int64_t max_tiles = pairs / width + experts + 1;
  const Tiles tiles{space.tile_count, space.tiles, pairs, width};
  Product p{*gate_up, space.xs, pairs, parts, tiles, max_tiles,
            Epilogue{space.x_scale, space.pair_of, nullptr, nullptr, nullptr, space.z, 0, 2 * inner, HI2_ACT_NONE, HI2_F32}};
  rc = product(p, s, "stored_experts");
  if (rc != HI2_OK) return rc;
  src = Source{space.z, 2 * inner, act, true, space.pair_of, index, space.used, top_k};
  rc = prepare<true>(src, *down, dtype, pairs, parts, space.hs, space.h_scale, s);
  if (rc != HI2_OK) return rc;
  p = Product{*down, space.hs, pairs, parts, tiles, max_tiles,
              Epilogue{space.h_scale, space.pair_of, weight, nullptr, nullptr, space.y, 0, hidden, HI2_ACT_NONE, HI2_F32}};
  rc = product(p, s, "stored_experts");
  if (rc != HI2_OK) return rc;
  int64_t blocks = ceil_div(tokens * (hidden / 4), (int64_t)256);
  if (blocks > 148 * 16) blocks = 148 * 16;
  combine_kernel<<<(unsigned)blocks, 256, 0, s>>>(space.y, space.row_of, tokens, top_k, hidden, out, dtype, ld_out);
  return check_launch("stored_experts: combine");
}
