// Packed weights laid out for products, and how a lane decodes them.
//
// The rows of a tensor (of each expert of a stack) are sorted by row format and dealt out to groups of 32,
// one row per lane.  A group's data is cut into chunks of 64 columns; a chunk holds the codes of
// its 32 rows as 16-byte pieces and behind them their (lo, step) byte pairs, so a warp reads a
// chunk (or a run of chunks) as one contiguous range.  Rows of one format that follow each other in a
// group are a run: piece p of the run's row i lies at piece (first of the run) + p * (rows of the run) + i,
// which keeps the 128-bit shared-memory reads of a warp free of bank conflicts at every code width.
// Inside a 32-bit word the codes of even columns fill the low half from its low bits, those of odd
// columns the high half, so that one mask extracts the codes of two neighbouring columns as an fp16 pair.
#pragma once

#include "common.cuh"

namespace hi2 {
namespace stored {

constexpr int CHUNK = 64;        // columns of a chunk
constexpr int GROUP_ROWS = 32;   // rows of a group: one per lane
constexpr int TILE_ROWS = 128;   // rows of a tile: four groups

// One 16-byte word per sorted row.
struct RowForm {
  uint32_t form;       // bits 0-7 first code piece, 8-19 parameter bytes / 2, 20-21 width, 22-23 block, 24-29 piece stride
  uint32_t out_row;    // row of the tensor (of the expert), or NO_ROW for padding
  uint32_t lo_consts;  // fp16 lo_min | fp16 lo_scale << 16
  uint32_t step_scale; // fp16
  __host__ __device__ int piece() const { return form & 255; }
  __host__ __device__ int params() const { return (form >> 8 & 4095) * 2; }
  __host__ __device__ int width() const { return form >> 20 & 3; }        // 0 padding, else log2 of the bits
  __host__ __device__ int block_shift() const { return form >> 22 & 3; }  // block = 16 << shift
  __host__ __device__ int piece_stride() const { return form >> 24 & 63; }
};
constexpr uint32_t NO_ROW = 0xffffffffu;

__device__ __forceinline__ RowForm load_row(const uint32_t* rows, int64_t i) {
  const uint4 v = __ldg(reinterpret_cast<const uint4*>(rows) + i);
  return RowForm{v.x, v.y, v.z, v.w};
}

__device__ __forceinline__ uint32_t bits(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 half2_of(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }
__device__ __forceinline__ uint32_t dup(uint32_t h) { return __byte_perm(h, h, 0x1010); }

// The pair's ladder as (lo, lo), (step, step): lo = fp16(fma_f32(u, lo_scale, lo_min)), step = fp16(u * step_scale),
// as the format defines them.
struct Ladder {
  __half2 lo, step;
};
__device__ __forceinline__ Ladder ladder(uint32_t pair, float lo_min, float lo_scale, float step_scale) {
  // 2^23 + u has u in its low bits: the bytes become floats without a conversion instruction
  const float u = __uint_as_float(__byte_perm(pair, 0x4b000000u, 0x7440)) - 8388608.0f;
  const float v = __uint_as_float(__byte_perm(pair, 0x4b000000u, 0x7441)) - 8388608.0f;
  const __half2 both = __floats2half2_rn(fmaf(u, lo_scale, lo_min), v * step_scale);
  return Ladder{__low2half2(both), __high2half2(both)};
}

// Two codes at bit `at` of both halves of w -> fp16(lo + code * step).  1024 + code * 2^at is an fp16
// number with the code in its mantissa; one fused multiply-add takes it to the code (exact), a second
// forms the weight with the format's single rounding.
template <int AT, int NBITS>
__device__ __forceinline__ uint32_t weight_pair(uint32_t w, const Ladder& l) {
  constexpr uint32_t mask = ((1u << NBITS) - 1u) << AT;
  const __half2 raw = half2_of((w & (mask | mask << 16)) | 0x64006400u);
  const __half2 scale = __float2half2_rn(1.0f / (float)(1 << AT)), bias = __float2half2_rn(-1024.0f / (float)(1 << AT));
  const __half2 code = AT == 0 ? __hadd2(raw, bias) : __hfma2(raw, scale, bias);
  return bits(__hfma2(code, l.step, l.lo));
}
__device__ __forceinline__ void decode_int2(uint32_t w, const Ladder& l, uint32_t* out) {  // 16 columns
  out[0] = weight_pair<0, 2>(w, l), out[1] = weight_pair<2, 2>(w, l), out[2] = weight_pair<4, 2>(w, l);
  out[3] = weight_pair<6, 2>(w, l), out[4] = weight_pair<8, 2>(w, l);
  w >>= 10;
  out[5] = weight_pair<0, 2>(w, l), out[6] = weight_pair<2, 2>(w, l), out[7] = weight_pair<4, 2>(w, l);
}
__device__ __forceinline__ void decode_int4(uint32_t w, const Ladder& l, uint32_t* out) {  // 8 columns
  out[0] = weight_pair<0, 4>(w, l), out[1] = weight_pair<4, 4>(w, l);
  w >>= 8;
  out[2] = weight_pair<0, 4>(w, l), out[3] = weight_pair<4, 4>(w, l);
}
__device__ __forceinline__ void decode_int8(uint32_t w, const Ladder& l, uint32_t* out) {  // 4 columns
  out[0] = weight_pair<0, 8>(w, l), out[1] = weight_pair<0, 8>(w >> 8, l);
}

// The 64 weights of the lane's row in the chunk at `slab`, two columns per word.  Padding gives zeros.
__device__ __forceinline__ void decode_chunk(const uint8_t* slab, const RowForm& row, float lo_min, float lo_scale,
                                             float step_scale, uint32_t (&out)[CHUNK / 2]) {
  const uint4* piece = reinterpret_cast<const uint4*>(slab) + row.piece();
  const uint16_t* pairs = reinterpret_cast<const uint16_t*>(slab + row.params());
  const int width = row.width();
  if (width == 0) {
#pragma unroll
    for (int i = 0; i < CHUNK / 2; ++i) out[i] = 0;
    return;
  }
  Ladder l[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) l[g] = ladder(pairs[g >> row.block_shift()], lo_min, lo_scale, step_scale);
  if (width == 1) {
    const uint4 v = piece[0];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int g = 0; g < 4; ++g) decode_int2(w[g], l[g], out + 8 * g);
  } else if (width == 2) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const uint4 v = piece[p * row.piece_stride()];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) decode_int4(w[q], l[2 * p + q / 2], out + 16 * p + 4 * q);
    }
  } else {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint4 v = piece[p * row.piece_stride()];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) decode_int8(w[q], l[p], out + 8 * p + 2 * q);
    }
  }
}

// ---- what follows a product ---------------------------------------------------------------------------
__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case HI2_ACT_RELU: return v < 0.0f ? 0.0f : v;  // a NaN stays one
    case HI2_ACT_SILU: return v / (1.0f + expf(-v));
    // the forms without cancellation: 1 + erf(x) = erfc(-x), (1 + tanh(x)) / 2 = 1 / (1 + exp(-2 x))
    case HI2_ACT_GELU: return 0.5f * v * erfcf(-0.70710678118654752f * v);
    case HI2_ACT_GELU_TANH: return v / (1.0f + expf(-1.5957691216057308f * (v + 0.044715f * v * v * v)));
    default: return v;
  }
}
__device__ __forceinline__ float load_as_float(const void* p, int dtype, int64_t i) {
  if (dtype == HI2_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if (dtype == HI2_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_float(void* p, int dtype, int64_t i, float v) {
  if (dtype == HI2_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else if (dtype == HI2_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<float*>(p)[i] = v;
}

// Where a product's values go.  A row of the activations is a token (one tensor) or a (token, slot) pair in
// expert order (a stack).
struct Epilogue {
  const float* row_scale;  // per activation row: the power of two that its fp16 parts were divided by
  const int32_t* pair_of;  // stack: row -> pair, else null
  const float* pair_weight;  // per pair, or null
  const void* bias;        // per output column, or null
  const void* residual;    // or null
  void* out;
  int64_t ld_residual, ld_out;
  int act, dtype;          // of bias, residual and out
  __device__ __forceinline__ void put(int64_t row, uint32_t col, float scale, float acc) const {
    float v = acc * scale;
    if (bias != nullptr) v += load_as_float(bias, dtype, col);
    v = activate(v, act);
    if (residual != nullptr) v += load_as_float(residual, dtype, row * ld_residual + col);
    store_float(out, dtype, row * ld_out + col, v);
  }
  __device__ __forceinline__ float scale_of(int64_t row) const {
    const float s = row_scale[row];
    return pair_weight == nullptr ? s : s * pair_weight[pair_of[row]];
  }
};

// The tile list of a stack, made on the device by the dispatch: activation rows [begin, end) of one expert.
struct TokenTile {
  int expert, begin, end;
};
struct Tiles {
  const int32_t* count;      // null: one tensor, tile t covers rows t * width ..
  const TokenTile* tiles;
  int64_t rows;              // of the activations
  int width;
  __device__ __forceinline__ bool get(int64_t t, TokenTile& out) const {
    if (count == nullptr) {
      const int64_t b = t * width;
      out = TokenTile{0, (int)b, (int)(b + width < rows ? b + width : rows)};
      return b < rows;
    }
    if (t >= *count) return false;
    out = tiles[t];
    return true;
  }
};

// The product of laid-out rows with prepared activations (xs: fp16 [parts, rows, k]; parts is 2 where
// the second half holds what the first one's rounding lost).
struct Product {
  hi2_stored_weight w;
  const __half* xs;
  int64_t x_rows;
  int parts;
  Tiles tiles;
  int64_t max_tiles;
  Epilogue out;
};
int tile_width(int64_t rows);  // of a tile, for that many activation rows of one tensor
int product(const Product& p, cudaStream_t stream, const char* what);

}  // namespace stored
}  // namespace hi2
