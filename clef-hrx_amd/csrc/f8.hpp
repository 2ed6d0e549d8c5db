// Block-scaled FP8 (e4m3): layouts, launchers and the device helpers that its
// kernels share. Values are e4m3 codes with one scale for each block of 128
// along k: y[m][n] = sum_b sa[m][b] sw[n / 128][b] sum_{k in block b} qa[m][k] qw[n][k].
//
// Activation ("prepared"): codes row-major [rows][pitch], pitch the width
// rounded up to 128 (the rest zeros), then its scales in two forms: as e8m0
// bytes [rows][kb rounded up to 16] (bits 23..30 of the f32), 16 blocks of k of
// a row in one 16-byte load, which the tiled products keep in LDS, and as f32
// [kb][rows], the rows of a fragment side by side, which the split-k products
// load as they go (with the bytes instead, 64 x 64 tiles took a quarter longer
// at 4096 x 4096 x 12288).
//
// Weight: blocks of 128 rows x 128 k (16 KiB), block (r / 128, k / 128) of one
// matrix at ((r / 128) * kb + k / 128) * 16384; rows and columns past the end
// are zeros. Inside a block the order is that of the matrix operand
// (v_mfma_*_16x16x128): fragment f of 16 rows at 2048 f, its halves h at 1024 h,
// lane l's 16 bytes at 16 l, holding row 16 f + l % 16, k = 64 h + 16 (l / 16)
// .. + 15. So a wave loads a half fragment as one contiguous KiB, into
// registers or LDS alike, and LDS reads of it are conflict-free as they lie.
// Scales f32 [matrices][ceil(rows / 128)][kb].
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "common.hpp"
#include "gemm_dma.hpp"
#include "launch.hpp"

namespace clef {

constexpr int f8_blocks(int64_t width) { return (int)((width + 127) / 128); }
constexpr int64_t f8_pitch(int64_t width) { return (width + 127) / 128 * 128; }
constexpr int64_t f8_scale_pitch(int64_t width) { return (f8_blocks(width) + 15) / 16 * 16; }
constexpr int64_t f8_prepared_bytes(int64_t rows, int64_t width) {
  return rows * (f8_pitch(width) + f8_scale_pitch(width) + 4 * f8_blocks(width));
}
constexpr int64_t f8_weight_bytes(int64_t matrices, int64_t rows, int64_t cols) {
  return matrices * f8_blocks(rows) * f8_blocks(cols) * 16384;
}

// A ragged list of rows per expert: slots[offsets[e] .. offsets[e + 1]) are
// expert e's (slots NULL: the places themselves). Slot s reads activation row
// s / div and writes output row s.
struct F8Lists {
  const int32_t* offsets;
  const int32_t* slots;
  int experts;
  int total;  // slots (and output rows)
  int div;
};

// One product. Without lists: rows m of `a` against one matrix. gate/up: w the
// gate, w2 the up matrices, n the width of h.
struct F8Args {
  const uint8_t* a;
  const uint8_t* ae;  // its scales: e8m0 [rows][kb rounded up to 16]
  const float* as;    // and f32 [kb][rows]
  int64_t rows;     // rows of a
  const uint8_t* w;
  const float* ws;
  const uint8_t* w2;
  const float* ws2;
  int n, kb;  // output columns, blocks of 128 along k
  bool pow2;  // every scale of w is a power of two
  const uint16_t* residual;
  uint16_t* out;
  F8Lists lists;
  // x in bf16 where the kernel quantizes its rows itself
  const uint16_t* x;
  int64_t x_stride;
  int k;
};

// The kernels of the products: tiles of rows x weight rows, the first five of the
// split-k kernel, the others of the tiled one (k128x128k: two blocks of k at a time).
enum class F8Kernel { k16x32, k32x32, k16x64, k32x64, k64x64, k128x128, k128x128k, k256x256 };
// The rule that picks one: a projection of m rows, products over lists of total
// slots (total, experts >= 1).
F8Kernel f8_kernel(int64_t m, int n, int kb, bool gate_up, bool pow2);
F8Kernel f8_kernel_lists(int64_t total, int64_t experts, int n, bool gate_up);

hipError_t launch_f8_prepare(const uint16_t* x, int64_t rows, int width, int64_t x_stride, uint8_t* codes,
                             uint8_t* exponents, float* scales, hipStream_t stream);
hipError_t launch_f8_pack(const uint16_t* w, int64_t matrices, int n, int k, uint8_t* codes, float* scales,
                          hipStream_t stream);
hipError_t launch_f8_retile(const uint8_t* w, int64_t matrices, int n, int k, uint8_t* codes, hipStream_t stream);
hipError_t launch_f8_gemm(const F8Args& x, bool gate_up, hipStream_t stream);
// Whether x [m][k] and the product against n columns run as one launch that
// quantizes the rows itself (F8Args::x).
bool f8_project_fusable(int64_t m, int n, int k);
hipError_t launch_f8_experts(const F8Args& x, bool gate_up, hipStream_t stream);
size_t group_slots_workspace_bytes(int64_t slots, int experts);
hipError_t launch_group_slots(const float* routes, int64_t tokens, int topk, int experts, int32_t* offsets,
                              int32_t* slots, void* workspace, hipStream_t stream);

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef int v8i_t __attribute__((ext_vector_type(8)));

// D = W A^T of a 16 x 16 tile over 128 k, added to c. Lane l holds weight row
// l % 16 in w and activation row l % 16 in a, the 32 values of its k-group
// l / 16 (any order of k that both share); D's lane l holds activation row
// l % 16 and weight rows 4 (l / 16) .. + 3. cbsz = blgp = 0: e4m3 both. The
// scales are e8m0 exponents, in byte 3 of sw (of w's rows) and byte `byte`
// (known when compiled) of sa (of a's rows; lane l's row l % 16).
__device__ __forceinline__ v4f mfma_f8_scaled(v8i_t w, v8i_t a, v4f c, int sw, uint32_t sa, int byte) {
  switch (byte) {
    case 0: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 0, 0, 3, sw, 0, (int)sa);
    case 1: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 0, 0, 3, sw, 1, (int)sa);
    case 2: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 0, 0, 3, sw, 2, (int)sa);
    default: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 0, 0, 3, sw, 3, (int)sa);
  }
}

// Any f32 scale as 2^e for the MFMA (e8m0 in byte 3) and a factor of magnitude
// 1 .. 2 for the fma behind it: with both powers of two in the MFMA a block's
// partial sum leaves f32's range only where the product itself does. Scales
// below 2^-126 take 2^-127, the least there is, and a smaller factor (zero
// itself: no partial sum becomes infinite in front of it), infinities and NaN
// 2^127 and themselves.
struct F8Split {
  int exponent;
  float factor;
};
__device__ __forceinline__ F8Split f8_split_scale(float s) {
  const uint32_t field = as_uint(s) >> 23 & 0xFFu;
  const int e = field < 254u ? (int)field : 254;
  return {e << 24, __builtin_ldexpf(s, 127 - e)};
}

__device__ __forceinline__ v8i_t join_halves(v4i lo, v4i hi) {
  return v8i_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// silu(g) u of two f32 sums. The hardware's exp2 and reciprocal (each within
// 1 ulp): both are far below the bf16 rounding that follows, and their limits
// give silu's (exp2 of -inf is 0, 1 / inf is 0).
__device__ __forceinline__ float f8_swiglu(float g, float u) {
  const float e = __builtin_amdgcn_exp2f(g * -1.44269504088896341f);
  return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}

// Exponent field of a block's scale: the least power of two at or above
// amax / 448, from the bf16 bits of amax: amax = 1.m 2^E is at most 448 2^(E -
// 8) = 1.75 2^E while m <= 0x60. At least 2^-126, so the scale and its
// reciprocal (field 254 - s) are normal.
__device__ __forceinline__ uint32_t f8_scale_field(uint32_t amax_bits) {
  const int f = (int)(amax_bits >> 7) - 8 + ((amax_bits & 0x7Fu) > 0x60u ? 1 : 0);
  return (uint32_t)(f > 1 ? f : 1);
}

// Eight e4m3 codes of bf16 values over `scale` (a power of two: exact), each
// rounded to nearest even once. |value| <= 448 scale by the choice of the scale;
// infinities and NaN become NaN (0x7F; e4m3 has no infinity).
__device__ __forceinline__ uint2 f8_codes8(uint4 v, float scale) {
  using s2 = __attribute__((ext_vector_type(2))) short;
  using b2 = __attribute__((ext_vector_type(2))) __bf16;
  auto two = [&](uint32_t lo, uint32_t hi) {
    s2 w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(s2{0, 0}, __builtin_bit_cast(b2, lo), scale, false);
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(b2, hi), scale, true));
  };
  return uint2{two(v.x, v.y), two(v.z, v.w)};
}

// The largest magnitude of eight bf16 values as bf16 bits, infinities and NaN
// above 0x7F7F (two 16-bit maxima per instruction); FINITE: those as zero.
template <bool FINITE>
__device__ __forceinline__ uint32_t f8_amax8(uint4 v) {
  using u2 = __attribute__((ext_vector_type(2))) unsigned short;
  auto mag = [](uint32_t p) {
    u2 m = __builtin_bit_cast(u2, p & 0x7FFF7FFFu);
    if (FINITE) m = u2{m[0] < 0x7F80 ? m[0] : (unsigned short)0, m[1] < 0x7F80 ? m[1] : (unsigned short)0};
    return m;
  };
  const u2 m = __builtin_elementwise_max(__builtin_elementwise_max(mag(v.x), mag(v.y)),
                                         __builtin_elementwise_max(mag(v.z), mag(v.w)));
  return m[0] > m[1] ? m[0] : m[1];
}

// The largest finite magnitude of the values that 16 lanes hold, 8 each, as bf16
// bits (non-finite ones stay NaN in the codes). Every lane of the wave is here.
__device__ __forceinline__ uint32_t f8_block_amax(uint4 v) {
  uint32_t m = group_max16(f8_amax8<false>(v));
  if (__builtin_expect(__any(m >= 0x7F80u), 0)) m = group_max16(f8_amax8<true>(v));
  return m;
}

// Inclusive sum over the wave's lanes (DPP: shifts within the rows of 16, then
// the rows' last lanes handed on).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, true);
  return v;
}

// The experts' lists cut into tiles of BM slots, experts ascending. find(tile)
// gives a tile's expert, first place and slots; `total` is the number of
// tiles. Offsets outside 0 .. total or descending are clamped, so every place is a
// slot. Each wave looks by itself, 64 experts at a time; the first 128 stay in
// registers between the count and the search.
template <int BM>
struct F8Tiles {
  const F8Lists& l;
  int lo[2], hi[2], incl[2], total;

  __device__ __forceinline__ explicit F8Tiles(const F8Lists& lists) : l(lists), total(0) {
    load(0, lo[0], hi[0]);
    load(64, lo[1], hi[1]);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      incl[c] = wave_scan((hi[c] - lo[c] + BM - 1) / BM) + total;
      total = __builtin_amdgcn_readlane(incl[c], 63);
    }
    for (int c = 128; c < l.experts; c += 64) {
      int x, y;
      load(c, x, y);
      total += __builtin_amdgcn_readlane(wave_scan((y - x + BM - 1) / BM), 63);
    }
  }

  __device__ __forceinline__ void load(int c, int& x, int& y) const {
    const int e = c + (int)(threadIdx.x & 63);
    x = y = 0;
    if (e < l.experts) {
      x = l.offsets[e];
      y = l.offsets[e + 1];
    }
    x = x < 0 ? 0 : x > l.total ? l.total : x;
    y = y < x ? x : y > l.total ? l.total : y;
  }

  __device__ __forceinline__ bool at(int c, int tile, int x, int y, int upto, int& expert, int& first,
                                     int& count) const {
    const unsigned long long mask = __ballot(upto > tile);
    if (mask == 0ull) return false;
    const int lane = __builtin_ctzll(mask);
    const int begin = __builtin_amdgcn_readlane(x, lane), end = __builtin_amdgcn_readlane(y, lane);
    const int before = __builtin_amdgcn_readlane(upto, lane) - (end - begin + BM - 1) / BM;
    expert = c + lane;
    first = begin + (tile - before) * BM;
    count = end - first < BM ? end - first : BM;
    return true;
  }

  // tile < total
  __device__ __forceinline__ void find(int tile, int& expert, int& first, int& count) const {
    if (at(0, tile, lo[0], hi[0], incl[0], expert, first, count)) return;
    if (at(64, tile, lo[1], hi[1], incl[1], expert, first, count)) return;
    int before = __builtin_amdgcn_readlane(incl[1], 63);
    for (int c = 128; c < l.experts; c += 64) {
      int x, y;
      load(c, x, y);
      const int upto = wave_scan((y - x + BM - 1) / BM) + before;
      if (at(c, tile, x, y, upto, expert, first, count)) return;
      before = __builtin_amdgcn_readlane(upto, 63);
    }
  }
};

// The most tiles of bm slots that lists over `total` slots can have.
inline int64_t f8_most_tiles(int64_t total, int experts, int bm) {
  return total / bm + (total < experts ? total : experts);
}

}  // namespace

}  // namespace clef
