// Block-scaled FP8 products for gfx950 (layouts and the formula in f8.hpp).
//
// A block's codes are multiplied by v_mfma_scale_f32_16x16x128_f8f6f4 (one
// instruction covers a block's 128 k, accumulating in f32), and the partial
// sum enters the f32 accumulator by one fma with sa[m] sw: a scale pair is
// rounded once, a block's sum once more in the fma. Output values are rounded
// to bf16 once, behind the residual or SwiGLU. Inside the instruction the
// products of eight neighbouring k are cut to 2^-13 of the largest of them (a
// property of the FP8 matrix unit, measured with single products beside a pair
// that cancels); the eights and everything behind them add in f32. Against 64
// bits the sums are off by about 1e-5 of their size, bf16 by 1.7e-3.
#include "f8.hpp"

namespace clef {

namespace {

// Few rows: each workgroup owns 16 MT rows x 16 NT weight rows (gate/up: NT / 2
// fragments of gate rows and the same of up), its eight waves split the
// blocks of k (wave w: blocks w, w + 8, ..). Operands go straight into
// registers: a weight fragment is two contiguous KiB in the operand order and is
// used by this workgroup's rows only, so LDS would add a trip and nothing
// else. D blocks are in flight per wave. The waves' sums meet in LDS and are
// added in wave order (the result does not depend on timing).
template <int MT, int NT, int D, bool LISTS, bool GU, bool RESID>
__global__ __launch_bounds__(512) void f8_stream_kernel(const F8Args p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int NW = 8, BM = 16 * MT, COLS = 16 * NT / (GU ? 2 : 1), NG = GU ? NT / 2 : NT;
  static_assert(!GU || NT % 2 == 0, "gate and up fragments");
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, g = lane >> 4;
  const int kb = p.kb, pitch = kb * 128;
  int expert = 0, first = 0, here = 0;
  int64_t m0 = 0;
  if constexpr (LISTS) {
    if (!f8_find_tile<BM>(p.lists, blockIdx.y, expert, first, here)) return;
  } else {
    m0 = (int64_t)blockIdx.y * BM;
    here = p.rows - m0 < BM ? (int)(p.rows - m0) : BM;
  }
  const int n0 = blockIdx.x * COLS;

  // activation rows of this lane: byte and scale offsets (rows past the end
  // read the tile's last row; their sums are not stored)
  int a_voff[MT], s_voff[MT];
  __amdgpu_buffer_rsrc_t a_rsrc, a_none, s_rsrc, s_none;
  {
    const uint8_t* base = p.a + (LISTS ? 0 : m0 * pitch);
    const uint32_t bytes = (uint32_t)(LISTS ? p.rows * pitch : (int64_t)here * pitch);
    a_rsrc = make_rsrc(base, bytes);
    a_none = make_rsrc(base, 0);
    s_rsrc = make_rsrc(p.as, (uint32_t)(p.rows * kb * 4));
    s_none = make_rsrc(p.as, 0);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    int r = 16 * i + lr;
    r = r < here ? r : here - 1;
    int64_t row = m0 + r;
    if constexpr (LISTS) {
      const int place = first + r;
      const int slot = p.lists.slots ? p.lists.slots[place] : place;
      // a slot outside the table reads nothing (it is not stored either)
      row = slot >= 0 && slot < p.lists.total ? slot / p.lists.div : 0;
      row = row < p.rows ? row : 0;
      a_voff[i] = (int)((uint32_t)row * (uint32_t)pitch) + 16 * g;
    } else {
      a_voff[i] = r * pitch + 16 * g;
    }
    s_voff[i] = (int)(row * 4);
  }
  const int nb = f8_blocks(p.n);
  const int64_t panel = ((int64_t)expert * nb + n0 / 128) * kb;
  const uint32_t panel_bytes = (uint32_t)kb * 16384u;
  const int w_voff = (n0 & 127) * 128 + lane * 16;
  const uint8_t* wp[2] = {p.w + panel * 16384, GU ? p.w2 + panel * 16384 : nullptr};
  const float* wsp[2] = {p.ws + panel, GU ? p.ws2 + panel : nullptr};
  constexpr int MATS = GU ? 2 : 1;

  struct Block {
    v4i w[NT][2], a[MT][2];
    float sa[MT], sw[MATS];
  } buf[D];
  auto load = [&](Block& b, int kt) {
    // blocks past the end: empty resources, zeros without a request
    const bool in = kt < kb;
    const int k = in ? kt : 0;
    const __amdgpu_buffer_rsrc_t ar = in ? a_rsrc : a_none, sr = in ? s_rsrc : s_none;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int mat = j / NG;
      const __amdgpu_buffer_rsrc_t wr = make_rsrc(wp[mat], in ? panel_bytes : 0u);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        b.w[j][h] = __builtin_amdgcn_raw_buffer_load_b128(wr, w_voff + (j % NG) * 2048 + h * 1024, k * 16384, 0);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) b.a[i][h] = __builtin_amdgcn_raw_buffer_load_b128(ar, a_voff[i] + 64 * h, k * 128, 0);
      b.sa[i] = as_float(__builtin_amdgcn_raw_buffer_load_b32(sr, s_voff[i], (int)(k * p.rows * 4), 0));
    }
#pragma unroll
    for (int m = 0; m < MATS; ++m) b.sw[m] = in ? wsp[m][k] : 0.0f;
  };
  v4f acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0, 0, 0, 0};
#pragma unroll
  for (int d = 0; d < D; ++d) load(buf[d], wave + NW * d);
  for (int k0 = wave; k0 < kb; k0 += NW * D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const Block& b = buf[d];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const v8i_t av = join_halves(b.a[i][0], b.a[i][1]);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const v4f part = mfma_f8(join_halves(b.w[j][0], b.w[j][1]), av, v4f{0, 0, 0, 0});
          const float s = b.sa[i] * b.sw[j / NG];
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[i][j][t] = __builtin_fmaf(part[t], s, acc[i][j][t]);
        }
      }
      load(buf[d], k0 + NW * (D + d));
    }
  }
  // the waves' sums: fragment (i, j) of wave w at ((w MT + i) NT + j) KiB
  v4f* sums = reinterpret_cast<v4f*>(lds);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) sums[((wave * MT + i) * NT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int u = threadIdx.x; u < MT * NG * 64; u += NW * 64) {
    const int l = u & 63, j = (u >> 6) % NG, i = (u >> 6) / NG;
    const int r = 16 * i + (l & 15), col = n0 + 16 * j + 4 * (l >> 4);
    if (r >= here || col >= p.n) continue;
    v4f y = v4f{0, 0, 0, 0}, y2 = v4f{0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      y += sums[((w * MT + i) * NT + j) * 64 + l];
      if constexpr (GU) y2 += sums[((w * MT + i) * NT + NG + j) * 64 + l];
    }
    int64_t row = m0 + r;
    if constexpr (LISTS) {
      const int place = first + r;
      const int slot = p.lists.slots ? p.lists.slots[place] : place;
      if (slot < 0 || slot >= p.lists.total) continue;
      row = slot;
    }
    if constexpr (GU) {
#pragma unroll
      for (int t = 0; t < 4; ++t) y[t] = f8_swiglu(y[t], y2[t]);
    }
    if constexpr (RESID) {
      const uint2 rv = *reinterpret_cast<const uint2*>(p.residual + row * p.n + col);
      y[0] += bf16_lo(rv.x);
      y[1] += bf16_hi(rv.x);
      y[2] += bf16_lo(rv.y);
      y[3] += bf16_hi(rv.y);
    }
    uint2 o;
    o.x = pack_bf16x2(y[0], y[1]);
    o.y = pack_bf16x2(y[2], y[3]);
    *reinterpret_cast<uint2*>(p.out + row * p.n + col) = o;
  }
#endif
}

template <int MT, int NT, int D, bool LISTS, bool GU, bool RESID>
hipError_t launch_stream(const F8Args& x, hipStream_t stream) {
  constexpr int BM = 16 * MT, COLS = 16 * NT / (GU ? 2 : 1), lds = 8 * MT * NT * 1024;
  static_assert(128 % COLS == 0, "a tile's columns lie in one weight block");
  static LaunchCache cache;
  auto* kernel = &f8_stream_kernel<MT, NT, D, LISTS, GU, RESID>;
  if (lds > 64 * 1024)
    if (hipError_t e = ensure_dynamic_lds(cache, reinterpret_cast<const void*>(kernel), lds)) return e;
  const int64_t tiles_m = LISTS ? f8_most_tiles(x.lists.total, x.lists.experts, BM) : (x.rows + BM - 1) / BM;
  if (tiles_m > 65535) return hipErrorInvalidValue;
  const dim3 grid((unsigned)((x.n + COLS - 1) / COLS), (unsigned)tiles_m);
  kernel<<<grid, 512, lds, stream>>>(x);
  return hipGetLastError();
}

template <bool LISTS, bool GU, bool RESID>
hipError_t launch_rows(const F8Args& x, hipStream_t stream) {
  return launch_stream<4, 4, 1, LISTS, GU, RESID>(x, stream);
}

}  // namespace

hipError_t launch_f8_gemm(const F8Args& x, bool gate_up, hipStream_t stream) {
  if (gate_up) return launch_rows<false, true, false>(x, stream);
  return x.residual ? launch_rows<false, false, true>(x, stream) : launch_rows<false, false, false>(x, stream);
}

bool f8_project_fusable(int64_t, int, int) { return false; }

hipError_t launch_f8_experts(const F8Args& x, bool gate_up, hipStream_t stream) {
  return gate_up ? launch_rows<true, true, false>(x, stream) : launch_rows<true, false, false>(x, stream);
}

}  // namespace clef
