// bf16 products with bias, activation and residual in the epilogue (linear.hpp).
#include "linear.hpp"

namespace clef {

namespace {

// Eight values of a row from column k on, zeros past column K: rows start at any
// even byte, so the load is an unaligned one.
__device__ __forceinline__ u4 load8_any(const uint16_t* row, int k, int K) {
  u4 v = {0, 0, 0, 0};
  if (k + 8 <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else {
#pragma unroll
    for (int t = 0; t < 8; ++t)
      if (k + t < K) v[t / 2] |= (uint32_t)row[k + t] << (16 * (t % 2));
  }
  return v;
}

// Every shape, stride and alignment: 64 rows x 64 weight rows (gate/up: 32 gate
// and 32 up) per workgroup of four waves, 64 k at a time through registers into one
// LDS stage (16-byte chunk c of row r at c ^ ((r >> 1) & 7)), the next 64 k on
// their way meanwhile.
template <bool GU>
__global__ __launch_bounds__(256) void linear_any_kernel(const LinearArgs p) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ __align__(16) char lds[2 * 64 * 128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, g = lane >> 4;
  const int wm = wave >> 1, wn = wave & 1;
  constexpr int COLS = GU ? 32 : 64;
  const int64_t m0 = (int64_t)blockIdx.y * 64;
  const int n0 = blockIdx.x * COLS;
  // this thread's chunks: chunk threadIdx.x % 8 of rows threadIdx.x / 8 and + 32
  const int chunk = threadIdx.x & 7;
  const uint16_t *xr[2], *wr[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = (threadIdx.x >> 3) + 32 * i;
    xr[i] = m0 + r < p.m ? p.x + (m0 + r) * p.x_stride : nullptr;
    const int col = n0 + (GU ? r % 32 : r);
    wr[i] = col < p.n ? (GU && i ? p.w2 : p.w) + col * p.w_stride : nullptr;
  }
  u4 xv[2], wv[2];
  auto load = [&](int k0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      xv[i] = xr[i] ? load8_any(xr[i], k0 + 8 * chunk, p.k) : u4{0, 0, 0, 0};
      wv[i] = wr[i] ? load8_any(wr[i], k0 + 8 * chunk, p.k) : u4{0, 0, 0, 0};
    }
  };
  v4f acc[2][2] = {};
  load(0);
  for (int k0 = 0; k0 < p.k; k0 += 64) {
    if (k0) __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (threadIdx.x >> 3) + 32 * i, at = r * 128 + ((chunk ^ ((r >> 1) & 7)) << 4);
      *reinterpret_cast<u4*>(lds + at) = xv[i];
      *reinterpret_cast<u4*>(lds + 8192 + at) = wv[i];
    }
    __syncthreads();
    if (k0 + 64 < p.k) load(k0 + 64);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u4 a[2], b[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int off = ((4 * s + g) ^ (lr >> 1)) << 4;
        a[i] = *reinterpret_cast<const u4*>(lds + (32 * wm + 16 * i + lr) * 128 + off);
        // gate/up: this wave's 16 gate rows, then its 16 up rows
        b[i] = *reinterpret_cast<const u4*>(lds + 8192 + ((GU ? 32 * i + 16 * wn : 32 * wn + 16 * i) + lr) * 128 + off);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma_bf16(b[j], a[i], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t row = m0 + 32 * wm + 16 * i + lr;
    if (row >= p.m) continue;
    if constexpr (GU) {
      linear_store4<true>(p, row, n0 + 16 * wn + 4 * g, acc[i][0], acc[i][1]);
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        linear_store4<false>(p, row, n0 + 32 * wn + 16 * j + 4 * g, acc[i][j], v4f{0, 0, 0, 0});
    }
  }
#endif
}

template <bool GU>
hipError_t launch_any(const LinearArgs& p, hipStream_t stream) {
  constexpr int COLS = GU ? 32 : 64;
  const dim3 grid((unsigned)((p.n + COLS - 1) / COLS), (unsigned)((p.m + 63) / 64));
  linear_any_kernel<GU><<<grid, 256, 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_linear(const LinearArgs& p, bool gate_up, hipStream_t stream) {
  return gate_up ? launch_any<true>(p, stream) : launch_any<false>(p, stream);
}

}  // namespace clef
