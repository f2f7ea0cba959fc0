// Packed weights laid out for products, and how they are decoded.
//
// The rows of a tensor (of each expert of a stack) are sorted by row format and cut into groups of 32 rows.  All rows of
// a group are kept in ONE form: where formats meet, rows with narrower codes or longer blocks take the others' width
// and block (the same codes in wider fields, their parameters repeated), so that only the last group of an expert has
// padding rows.  (Padding every format's last group instead took 17 tiles for 2048 rows of four formats.)  A group's data is cut into
// chunks of 64 columns; a chunk (a slab) holds the codes of its 32 rows and behind them their (lo, step) byte
// pairs, so a warp reads a run of chunks as one contiguous range.  Row 8 r + g of a group (g < 8, r < 4) has in
// a chunk nbits / 2 words of codes for each of its four 16-column pieces t; word h of piece t lies at word
// 128 h + 32 t + 4 ((g + 2 t) mod 8) + r.  One 128-bit read then gives lane 4 g + t the same word of four rows, which is
// what the fragments of a warp-level matrix product ask for, and one 32-bit read a word of all 32 rows; both
// without a bank conflict.  The pairs: pair (g, t, r) at 16-bit unit 4 ((4 >> shift) g + (t >> shift)) + r with
// blocks of 16 << shift columns.
// Inside a word the codes of even columns fill the low half from its low bits, those of odd columns the
// high half, so that one mask extracts the codes of two neighbouring columns as an fp16 pair.
#pragma once

#include "common.cuh"

namespace hi2 {
namespace stored {

constexpr int CHUNK = 64;        // columns of a chunk
constexpr int GROUP_ROWS = 32;
constexpr int TILE_ROWS = 128;   // rows of a tile: four groups
constexpr int MAX_SLAB = 2304;   // bytes of a chunk of a group: INT8 in blocks of 16

struct GroupForm {
  uint32_t base;   // first 16-byte unit of the data
  uint32_t form;   // log2 of the code width (0: padding only, no data) | log2(block / 16) << 2 | SMALL steps << 4
  __host__ __device__ int width() const { return form & 3; }
  __host__ __device__ int shift() const { return form >> 2 & 3; }
  __host__ __device__ bool small_steps() const { return (form >> 4 & 1) != 0; }
  __host__ __device__ int code_bytes() const { return 256 << width(); }  // of a chunk
  __host__ __device__ int slab_bytes() const { return width() == 0 ? 0 : code_bytes() + (256 >> shift()); }
};
__device__ __forceinline__ GroupForm load_group(const uint32_t* groups, int64_t g) {
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(groups) + g);
  return GroupForm{v.x, v.y};
}

// One 16-byte word per sorted row.
constexpr uint32_t NO_ROW = 0xffffffffu;
struct RowConsts {
  uint32_t out_row;    // row of the tensor (of the expert), or NO_ROW for padding
  uint32_t lo_consts;  // fp16 lo_min | fp16 lo_scale << 16
  uint32_t step_scale; // fp16
  __device__ __forceinline__ float lo_min() const { return __half2float(__ushort_as_half((uint16_t)lo_consts)); }
  __device__ __forceinline__ float lo_scale() const { return __half2float(__ushort_as_half((uint16_t)(lo_consts >> 16))); }
};
__device__ __forceinline__ RowConsts load_row(const uint32_t* rows, int64_t i) {
  const uint4 v = __ldg(reinterpret_cast<const uint4*>(rows) + i);
  return RowConsts{v.x, v.y, v.z};
}

// First word of (g, t) in a chunk's codes.
__host__ __device__ __forceinline__ int code_word(int g, int t) { return 32 * t + 4 * ((g + 2 * t) & 7); }

__device__ __forceinline__ uint32_t bits(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 half2_of(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// A ladder as (lo, lo), and (step, step) times the powers of two that the decoder below asks for.  The format
// defines lo = fp16(fma_f32(u, lo_scale, lo_min)) and step = fp16(u * step_scale).
struct Ladder {
  __half2 lo, step[2];
};
// Two codes of neighbouring columns at bit `AT` of both halves of w -> fp16(lo + code * step).
//
// SMALL steps (of all rows of the group: at most 65504 / 2^18 with 2-bit codes, 2^20 with 4-bit, 2^22 with 8-bit ones):
// the field by itself is the fp16 subnormal code * 2^(AT - 24), and one fused multiply-add with step * 2^(24 - AT), an
// fp16 number for fields at bits 6 and 8 (2-bit codes), 4 (4-bit), 2 (8-bit), forms the weight with the format's single
// rounding.
// Any step: 1024 + code * 2^AT is an fp16 number with the code in its mantissa; a fused multiply-add takes
// it to the code (exact), a second one forms the weight.  fp16 arithmetic issues every other clock and shares its pipe
// with the warp-level products: 2048 INT2 weights and their products, out of registers, take a scheduler 183 clocks with small
// steps and 216 without; 2048 INT4 weights with small steps 190, INT8 201.
template <int AT, int NBITS, bool SMALL>
__device__ __forceinline__ uint32_t weight_pair(uint32_t w, __half2 lo, __half2 step) {
  constexpr uint32_t mask = ((1u << NBITS) - 1u) << AT;
  if (SMALL) return bits(__hfma2(half2_of(w & (mask | mask << 16)), step, lo));
  constexpr uint32_t scale = (uint32_t)(15 - AT) << 10, bias = 0x8000u | (uint32_t)(25 - AT) << 10;  // 2^-AT, -2^(10 - AT)
  uint32_t field;  // (w & mask) | magic in one instruction
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(field) : "r"(w), "r"(mask | mask << 16), "r"(0x64006400u));
  const __half2 code = AT == 0 ? __hadd2(half2_of(field), half2_of(bias | bias << 16))
                               : __hfma2(half2_of(field), half2_of(scale | scale << 16), half2_of(bias | bias << 16));
  return bits(__hfma2(code, step, lo));
}
// Two byte pairs of two rows (row 0 in the low half of `pairs`) -> their ladders.  2^23 + u and 1024 + u have
// u in their low bits, so the bytes become numbers without a conversion; an fp16 product of a byte and
// an fp16 number rounds once, as the fp32 product rounded to fp16 does (that one is exact).
template <int NBITS, bool SMALL>
__device__ __forceinline__ void ladders(uint32_t pairs, const float (&lo_min)[2], const float (&lo_scale)[2], __half2 step_scale,
                                        Ladder& a, Ladder& b) {
  const float u = __uint_as_float(__byte_perm(pairs, 0x4b000000u, 0x7440)) - 8388608.0f;
  const float v = __uint_as_float(__byte_perm(pairs, 0x4b000000u, 0x7442)) - 8388608.0f;
  const __half2 lo = __floats2half2_rn(fmaf(u, lo_scale[0], lo_min[0]), fmaf(v, lo_scale[1], lo_min[1]));
  const __half2 steps = __hadd2(half2_of(__byte_perm(pairs, 0x64646464u, 0x4341)), half2_of(0xe400e400u));
  __half2 step[2];
  step[0] = __hmul2(steps, step_scale);
  if (SMALL) {  // 2^10, then 2^6 and 2^8, 2^10 or 2^12 (2^16 is no fp16 number)
    const __half2 up = __hmul2(step[0], half2_of(0x64006400u));
    step[0] = __hmul2(up, half2_of(NBITS == 2 ? 0x54005400u : NBITS == 4 ? 0x64006400u : 0x6c006c00u));
    if (NBITS == 2) step[1] = __hmul2(up, half2_of(0x5c005c00u));
  }
  a.lo = __low2half2(lo), b.lo = __high2half2(lo);
#pragma unroll
  for (int i = 0; i < (SMALL && NBITS == 2 ? 2 : 1); ++i) a.step[i] = __low2half2(step[i]), b.step[i] = __high2half2(step[i]);
}

// Word h of a 16-column piece -> its pairs of neighbouring columns.
template <int NBITS, bool SMALL>
__device__ __forceinline__ void decode_word(uint32_t w, const Ladder& l, uint32_t* out) {
  const __half2 lo = l.lo, st = l.step[0];
  if (NBITS == 2 && SMALL) {
    const uint32_t up = w << 4, down = w >> 4;
    out[0] = weight_pair<8, 2, true>(w << 8, lo, st), out[1] = weight_pair<6, 2, true>(up, lo, l.step[1]);
    out[2] = weight_pair<8, 2, true>(up, lo, st), out[3] = weight_pair<6, 2, true>(w, lo, l.step[1]);
    out[4] = weight_pair<8, 2, true>(w, lo, st), out[5] = weight_pair<6, 2, true>(down, lo, l.step[1]);
    out[6] = weight_pair<8, 2, true>(down, lo, st), out[7] = weight_pair<8, 2, true>(w >> 6, lo, st);
  } else if (NBITS == 2) {
    out[0] = weight_pair<0, 2, false>(w, lo, st), out[1] = weight_pair<2, 2, false>(w, lo, st), out[2] = weight_pair<4, 2, false>(w, lo, st);
    out[3] = weight_pair<6, 2, false>(w, lo, st), out[4] = weight_pair<8, 2, false>(w, lo, st);
    w >>= 10;
    out[5] = weight_pair<0, 2, false>(w, lo, st), out[6] = weight_pair<2, 2, false>(w, lo, st), out[7] = weight_pair<4, 2, false>(w, lo, st);
  } else if (NBITS == 4 && SMALL) {
    out[0] = weight_pair<4, 4, true>(w << 4, lo, st), out[1] = weight_pair<4, 4, true>(w, lo, st);
    out[2] = weight_pair<4, 4, true>(w >> 4, lo, st), out[3] = weight_pair<4, 4, true>(w >> 8, lo, st);
  } else if (NBITS == 4) {
    out[0] = weight_pair<0, 4, false>(w, lo, st), out[1] = weight_pair<4, 4, false>(w, lo, st);
    w >>= 8;
    out[2] = weight_pair<0, 4, false>(w, lo, st), out[3] = weight_pair<4, 4, false>(w, lo, st);
  } else if (SMALL) {
    out[0] = weight_pair<2, 8, true>(w << 2, lo, st), out[1] = weight_pair<2, 8, true>(w >> 6, lo, st);
  } else {
    out[0] = weight_pair<0, 8, false>(w, lo, st), out[1] = weight_pair<0, 8, false>(w >> 8, lo, st);
  }
}

// ---- what follows a product ---------------------------------------------------------------------------
__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case HI2_ACT_RELU: return v < 0.0f ? 0.0f : v;  // a NaN stays one
    case HI2_ACT_SILU: return __fdividef(v, 1.0f + expf(-v));  // (a divisor beyond 2^126 gives 0, as it should)
    // the forms without cancellation: 1 + erf(x) = erfc(-x), (1 + tanh(x)) / 2 = 1 / (1 + exp(-2 x))
    case HI2_ACT_GELU: return 0.5f * v * erfcf(-0.70710678118654752f * v);
    case HI2_ACT_GELU_TANH: return __fdividef(v, 1.0f + expf(-1.5957691216057308f * (v + 0.044715f * v * v * v)));
    default: return v;
  }
}
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
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

// Where the activation rows of a product come from.  A row is a token (one tensor) or a (token, slot) pair of a
// stack, which names its expert.
enum SourceKind { FROM_F32 = 0, FROM_F16 = 1, FROM_BF16 = 2, FROM_GATED = 3 };
struct Source {
  const void* x;         // [tokens, ldx]; FROM_GATED: fp32 [pairs, 2 k], the results of the gate and up rows
  int64_t ldx;
  int kind;
  int act;               // FROM_GATED: of the gate rows
  bool vector;           // rows start on 16-byte boundaries
  int top_k;             // stack: pairs per token
};

// 16 values of row p.
template <typename T>
__device__ __forceinline__ void load16(const T* p, bool vector, float (&v)[16]) {
  if (vector) {
    constexpr int PER = 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < 16 / PER; ++i) {
      const uint4 raw = *(reinterpret_cast<const uint4*>(p) + i);
      const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int j = 0; j < PER; ++j) v[PER * i + j] = to_float(t[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = to_float(p[i]);
  }
}

// Columns 16 g .. 16 g + 15 of a row in the stored basis: divided by the smoothing vector, rotated where flagged.
__device__ __forceinline__ void stored_basis(const Source& s, const hi2_stored_weight& w, int64_t row, int64_t expert,
                                             int64_t g, float (&v)[16]) {
  const bool rotate = w.had[expert * (w.k / 16) + g] != 0;
  if (s.kind == FROM_GATED) {
    const float* z = static_cast<const float*>(s.x) + row * s.ldx + g * 16;
    float u[16];
    load16(z, true, v);
    load16(z + w.k, true, u);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = activate(v[i], s.act) * u[i];
  } else if (s.kind == FROM_BF16) {
    load16(static_cast<const __nv_bfloat16*>(s.x) + row * s.ldx + g * 16, s.vector, v);
  } else if (s.kind == FROM_F16) {
    load16(static_cast<const __half*>(s.x) + row * s.ldx + g * 16, s.vector, v);
  } else {
    load16(static_cast<const float*>(s.x) + row * s.ldx + g * 16, s.vector, v);
  }
  if (w.inv_scale != nullptr) {
    float c[16];
    load16(w.inv_scale + expert * w.k + g * 16, true, c);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] *= c[i];
  }
  if (rotate) {
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

__device__ __forceinline__ float largest(const float (&v)[16]) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(v[i]));
  return top;
}
// The power of two that takes `top` to [2^14, 2^15); values without a size, or with an infinity, stay as they are.  It stops
// at 2^`lowest`, so that both directions are normal fp32 numbers.
struct PowerOfTwo {
  float to, back;
};
__device__ __forceinline__ PowerOfTwo power_for(float top, int lowest = -126) {
  const int biased = (int)(__float_as_uint(top) >> 23);
  int e = biased - 127 - 14;
  if (top == 0.0f || biased == 255) e = 0;
  if (e < lowest) e = lowest;
  return PowerOfTwo{__uint_as_float((uint32_t)(127 - e) << 23), __uint_as_float((uint32_t)(127 + e) << 23)};
}
// The fp16 parts of 16 values times `to`, as two 16-byte words each.
template <int PARTS>
__device__ __forceinline__ void split16(const float (&v)[16], float to, uint4 (&hi)[2], uint4 (&lo)[2]) {
  uint32_t h[8], l[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = v[2 * i] * to, b = v[2 * i + 1] * to;
    const __half2 both = __floats2half2_rn(a, b);
    h[i] = bits(both);
    l[i] = PARTS == 1 ? 0u : bits(__floats2half2_rn(a - __low2float(both), b - __high2float(both)));
  }
  hi[0] = make_uint4(h[0], h[1], h[2], h[3]), hi[1] = make_uint4(h[4], h[5], h[6], h[7]);
  lo[0] = make_uint4(l[0], l[1], l[2], l[3]), lo[1] = make_uint4(l[4], l[5], l[6], l[7]);
}

// Where a product's values go.
struct Epilogue {
  const float* pair_weight;  // stack: per pair, or null
  const void* bias;        // per output column, or null
  const void* residual;    // or null
  void* out;
  int64_t ld_residual, ld_out;
  int act, dtype;          // of bias, residual and out
  __device__ __forceinline__ void put(int64_t row, uint32_t col, float v) const {
    if (bias != nullptr) v += load_as_float(bias, dtype, col);
    v = activate(v, act);
    if (residual != nullptr) v += load_as_float(residual, dtype, row * ld_residual + col);
    store_float(out, dtype, row * ld_out + col, v);
  }
};

// Tiles of activation rows.  One tensor: tile t covers rows t * width ..  A stack: either a list made on
// the device (rows are pairs in expert order; row -> pair by pair_of), or, for a few pairs, every pair a
// tile of its own, rows in the pairs' order.
struct TokenTile {
  int expert, begin, end;
};
struct Tiles {
  const int64_t* index;      // stack: pair -> expert, else null
  const int32_t* pair_of;    // stack with a list: row -> pair
  const int32_t* count;      // stack with a list: number of tiles
  const TokenTile* list;
  int64_t rows;              // of the activations
  int experts, width;
  __device__ __forceinline__ bool get(int64_t t, TokenTile& out) const {
    if (count != nullptr) {
      if (t >= *count) return false;
      out = list[t];
      return true;
    }
    const int64_t b = t * width;
    if (b >= rows) return false;
    int64_t e = 0;
    if (index != nullptr) {
      e = index[b];
      if (e < 0 || e >= experts) return false;
    }
    out = TokenTile{(int)e, (int)b, (int)(b + width < rows ? b + width : rows)};
    return true;
  }
  __device__ __forceinline__ int64_t pair(int64_t row) const { return pair_of == nullptr ? row : pair_of[row]; }
};

// The product of laid-out rows with activations.
struct Product {
  hi2_stored_weight w;
  Source from;
  Tiles tiles;
  int64_t max_tiles;
  int parts;               // fp16 parts of an activation: 2 where the second holds what the first one's rounding lost
  Epilogue out;
  bool exact;              // fp32 results
  bool settled;            // index and tile list were complete before the kernel ahead of this one set out
  // wide products only: the prepared activations fp16 [parts, rows, k], the powers of two they were divided by, and the
  // sums of the slices fp32 [wide_splits, rows, rows of the tensor] where there are several
  __half* xs;
  float* row_scale;
  float* partial;
};

// Products with up to 8 activation rows per tile, which prepare their activations themselves.
constexpr int FEW_WIDTH = 8;
struct FewPlan {
  int split, runs;  // slices of the columns (a cluster); runs of row tiles, a block each
  double cost;      // of the fullest SM, in chunks
};
FewPlan few_plan(int64_t k, int64_t row_tiles, int64_t tiles, int64_t width, int parts);
int64_t few_tiles(int64_t experts, int64_t rows);
int product_few(const Product& p, cudaStream_t stream, const char* what);
// Wide tiles, from prepared activations.
int wide_width(int64_t rows, bool exact);
int wide_splits(int64_t k, int64_t rows_of_tensor, int64_t max_tiles, bool stack);
int product_wide(const Product& p, cudaStream_t stream, const char* what);

}  // namespace stored
}  // namespace hi2
