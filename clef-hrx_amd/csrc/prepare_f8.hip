// Block-scaled FP8 operands: the quantizer of activation rows and the two
// ways to a tiled weight (bf16 rows quantized, e4m3 rows of a checkpoint
// rearranged). Layouts in f8.hpp.
#include "f8.hpp"

namespace clef {

namespace {

// A dispatch counts the work-items of each dimension in 32 bits: workgroups of
// rows beyond this many go along z.
constexpr int64_t kPartWorkgroups = (int64_t)1 << 22;

// x bf16 [rows][width] (row pitch x_stride) -> codes [rows][pitch], scales as
// e8m0 [rows][kp] and f32 [kb][rows]. 16 lanes hold a block of 128 columns, 8
// values each: one 16-byte load, the maximum over the 16 lanes by DPP, one 8-byte
// store of codes (a whole line per block). A workgroup covers 2^RLOG rows x CPW *
// STEPS blocks, so that the f32 scales of neighbouring rows go out together, with
// STEPS loads in flight per lane. Bound by HBM: 2 bytes read and 1 written per
// value, 4.6 to 5.2 TB/s at 4096 x 12288 (33 us in a graph of inputs and outputs
// that pass the last-level cache, 29 called one by one).
template <int RLOG, int STEPS>
__global__ __launch_bounds__(256) void f8_prepare_kernel(const uint16_t* __restrict__ x, int64_t rows, int width,
                                                         int64_t x_stride, int kb, int kp,
                                                         uint8_t* __restrict__ codes,
                                                         uint8_t* __restrict__ exponents,
                                                         float* __restrict__ scales) {
  constexpr int R = 1 << RLOG, CPW = 16 / R;
  const int group = threadIdx.x >> 4, l = threadIdx.x & 15;
  const int64_t row = ((int64_t)blockIdx.z * kPartWorkgroups + blockIdx.x) * R + (group & (R - 1));
  const int b0 = blockIdx.y * (CPW * STEPS) + (group >> RLOG);
  const bool row_here = row < rows;
  const uint16_t* xr = x + row * x_stride;
  uint4 v[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int col = (b0 + s * CPW) * 128 + 8 * l;  // width % 8 == 0: the 8 columns are all inside or all past the end
    v[s] = uint4{0, 0, 0, 0};
    if (row_here && col < width) v[s] = *reinterpret_cast<const uint4*>(xr + col);
  }
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int b = b0 + s * CPW;
    const uint32_t m = f8_block_amax(v[s]);
    if (!row_here || b >= kp) continue;
    if (b >= kb) {  // the row's bytes behind its exponents: zeros
      if (l == 0) exponents[row * kp + b] = 0;
      continue;
    }
    const uint32_t field = f8_scale_field(m);
    const float scale = as_float(field << 23);
    *reinterpret_cast<uint2*>(codes + row * ((int64_t)kb * 128) + b * 128 + 8 * l) = f8_codes8(v[s], scale);
    if (l == 0) {
      exponents[row * kp + b] = (uint8_t)field;
      scales[(int64_t)b * rows + row] = scale;
    }
  }
}

// Byte of (row, k) of a 128 x 128 block in the operand order (f8.hpp).
__device__ __forceinline__ int f8_block_byte(int row, int k) {
  const int chunk = k >> 4;
  return (row >> 4) * 2048 + (chunk >> 2) * 1024 + ((chunk & 3) * 16 + (row & 15)) * 16 + (k & 15);
}

// One workgroup per 128 x 128 block of a bf16 weight: thread t takes 8 chunks
// of 8 columns (rows t / 16 + 16 i, columns 8 (t % 16) ..), the block's maximum
// meets in LDS, and the codes go out in the operand order. Weights are packed
// once, at load. Bound by HBM, 2 bytes read and 1 written per value: 128 x 2048 x
// 768 112 us (5.4 TB/s), 12288 x 4096 33 us (4.6), 1352 x 4160 6.5 us.
__global__ __launch_bounds__(256) void f8_pack_kernel(const uint16_t* __restrict__ w, int n, int k, int nb, int kb,
                                                      uint8_t* __restrict__ codes, float* __restrict__ scales) {
  __shared__ uint32_t wave_max[4];
  const int64_t block = blockIdx.x;
  const int kt = (int)(block % kb);
  const int64_t panel = block / kb;
  const int rb = (int)(panel % nb);
  const int64_t e = panel / nb;
  const int l = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int col = kt * 128 + 8 * l;
  uint4 v[8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = rb * 128 + r0 + 16 * i;
    v[i] = uint4{0, 0, 0, 0};
    if (row < n && col < k) v[i] = *reinterpret_cast<const uint4*>(w + (e * n + row) * (int64_t)k + col);
    const uint32_t o = f8_amax8<true>(v[i]);
    m = m > o ? m : o;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)m, off);
    m = m > o ? m : o;
  }
  if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) m = m > wave_max[i] ? m : wave_max[i];
  const uint32_t field = f8_scale_field(m);
  const float scale = as_float(field << 23);
  uint8_t* out = codes + block * 16384;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    *reinterpret_cast<uint2*>(out + f8_block_byte(r0 + 16 * i, 8 * l)) = f8_codes8(v[i], scale);
  }
  if (threadIdx.x == 0) scales[block] = scale;
}

// e4m3 rows [matrices][n][k] -> blocks in the operand order; one workgroup per
// block, 8 bytes per thread and row (k % 8 == 0). Bound by HBM, a byte read and a
// byte written per value: 128 x 2048 x 768 79 us (5.1 TB/s), 12288 x 4096 25 us
// (4.1), 1352 x 4160 6.0 us.
__global__ __launch_bounds__(256) void f8_retile_kernel(const uint8_t* __restrict__ w, int n, int k, int nb, int kb,
                                                        uint8_t* __restrict__ codes) {
  const int64_t block = blockIdx.x;
  const int kt = (int)(block % kb);
  const int64_t panel = block / kb;
  const int rb = (int)(panel % nb);
  const int64_t e = panel / nb;
  const int l = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int col = kt * 128 + 8 * l;
  uint8_t* out = codes + block * 16384;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = rb * 128 + r0 + 16 * i;
    uint2 q{0, 0};
    if (row < n && col < k) q = *reinterpret_cast<const uint2*>(w + (e * n + row) * (int64_t)k + col);
    *reinterpret_cast<uint2*>(out + f8_block_byte(r0 + 16 * i, 8 * l)) = q;
  }
}

}  // namespace

hipError_t launch_f8_prepare(const uint16_t* x, int64_t rows, int width, int64_t x_stride, uint8_t* codes,
                             uint8_t* exponents, float* scales, hipStream_t stream) {
  const int kb = f8_blocks(width), kp = (int)f8_scale_pitch(width);
  auto run = [&](auto rlog, auto steps) {
    constexpr int R = 1 << decltype(rlog)::value, per = 16 / R * decltype(steps)::value;
    const int64_t down = (rows + R - 1) / R, parts = (down + kPartWorkgroups - 1) / kPartWorkgroups;
    const dim3 grid((unsigned)(parts > 1 ? kPartWorkgroups : down), (unsigned)((kp + per - 1) / per), (unsigned)parts);
    f8_prepare_kernel<decltype(rlog)::value, decltype(steps)::value>
        <<<grid, 256, 0, stream>>>(x, rows, width, x_stride, kb, kp, codes, exponents, scales);
  };
  using std::integral_constant;
  // Rows and outputs from memory: four loads ahead from 16M values up (4096 x 4096
  // 13.2 us against 13.5 with two, 32768 x 768 17.2 against 19.4), two below (37 x
  // 4160 2.3 against 2.8, 620 x 17408 10.1 with both). Four rows per workgroup
  // (32768 x 768 with 1, 2 or 8: 28.0, 19.3, 18.6), one where there are fewer.
  if (rows >= 3 && rows * width >= (1 << 24))
    run(integral_constant<int, 2>{}, integral_constant<int, 4>{});
  else if (rows >= 3)
    run(integral_constant<int, 2>{}, integral_constant<int, 2>{});
  else
    run(integral_constant<int, 0>{}, integral_constant<int, 2>{});
  return hipGetLastError();
}

hipError_t launch_f8_pack(const uint16_t* w, int64_t matrices, int n, int k, uint8_t* codes, float* scales,
                          hipStream_t stream) {
  const int nb = f8_blocks(n), kb = f8_blocks(k);
  f8_pack_kernel<<<(unsigned)(matrices * nb * kb), 256, 0, stream>>>(w, n, k, nb, kb, codes, scales);
  return hipGetLastError();
}

hipError_t launch_f8_retile(const uint8_t* w, int64_t matrices, int n, int k, uint8_t* codes, hipStream_t stream) {
  const int nb = f8_blocks(n), kb = f8_blocks(k);
  f8_retile_kernel<<<(unsigned)(matrices * nb * kb), 256, 0, stream>>>(w, n, k, nb, kb, codes);
  return hipGetLastError();
}

}  // namespace clef
