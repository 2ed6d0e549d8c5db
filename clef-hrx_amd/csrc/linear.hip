// bf16 products with bias, activation and residual in the epilogue (linear.hpp).
//
// Few rows are bound by the weight's bytes (and by the rows', which every tile of
// columns reads again), many by the matrix unit, whose rate the board's power holds
// at about 1.5 PFLOP/s. Times below are in us, operands from memory (in turn past the
// last-level cache, in a graph); what is compared ran in turn on one card.
#include "linear.hpp"

namespace clef {

namespace {

// Eight values of a row that starts at any even byte.
__device__ __forceinline__ u4 any_load(const uint16_t* from) {
  u4 v;
  __builtin_memcpy(&v, from, 16);
  return v;
}

// From column k on, a multiple of 8: zeros past column K. The dwords that hold them,
// those past the row's last value read there (so that no branch makes the loads wait
// for each other), shifted into place.
__device__ __forceinline__ u4 any_load_tail(const uint16_t* row, int k, int K) {
  const char* const down = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(row) & ~(uintptr_t)3);
  const int odd = (int)(reinterpret_cast<uintptr_t>(row) & 2) / 2;
  const int last = (2 * (K - 1 + odd)) & ~3;  // of the dword that holds value K - 1
  uint32_t d[5];
#pragma unroll
  for (int j = 0; j < 5; ++j) {
    const int at = 2 * k + 4 * j;
    d[j] = *reinterpret_cast<const uint32_t*>(down + (at < last ? at : last));
  }
#pragma unroll
  for (int j = 0; j < 5; ++j) {
    const int left = K - k + odd - 2 * j;  // halves of this dword that are values
    d[j] = left >= 2 ? d[j] : left == 1 ? d[j] & 0xFFFFu : 0u;
  }
  u4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = __builtin_amdgcn_alignbit(d[j + 1], d[j], 16 * odd);
  return v;
}

// Many rows of any alignment: 32 TM rows x 32 WN weight rows (gate/up: half of them
// gate and half up) per workgroup of 2 x WN waves, 64 k at a time through registers
// into one LDS stage (16-byte chunk c of row r at c ^ ((r >> 1) & 7)), the next 64 k
// on their way meanwhile. Bound by the loads, which take twice the time of aligned
// ones: 4096 x 4097 x 4097 on 64 x 64 434 us, on 128 x 128 290 (0.47 PFLOP/s), on 256 x
// 256, of which a CU holds one, 410; 512 x 4097 x 2049, 68 tiles of 128 x 128, 62 and 88.
template <int TM, int WN, bool GU>
__global__ __launch_bounds__(128 * WN) void linear_any_kernel(const LinearArgs p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int BM = 32 * TM, BN = 32 * WN, HALF = 16 * WN;  // HALF: rows of a load of all threads
  static_assert(BM == BN, "two loads of either operand per thread");
  __shared__ __align__(16) char lds[(BM + BN) * 128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, g = lane >> 4;
  const int wm = wave / WN, wn = wave % WN;
  constexpr int COLS = GU ? HALF : BN;
  const int64_t m0 = (int64_t)blockIdx.y * BM;
  const int n0 = blockIdx.x * COLS;
  // this thread's chunks: chunk threadIdx.x % 8 of rows threadIdx.x / 8 and + HALF
  const int chunk = threadIdx.x & 7;
  const uint16_t *xr[2], *wr[2];  // rows past the end repeat the last
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = (threadIdx.x >> 3) + HALF * i;
    xr[i] = p.x + (m0 + r < p.m ? m0 + r : p.m - 1) * p.x_stride;
    const int col = n0 + (GU ? r % HALF : r);
    wr[i] = (GU && i ? p.w2 : p.w) + (col < p.n ? col : p.n - 1) * p.w_stride;
  }
  u4 xv[2], wv[2];
  auto load = [&](int k0) {
    const int k = k0 + 8 * chunk;
    if (k0 + 64 <= p.k) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        xv[i] = any_load(xr[i] + k);
        wv[i] = any_load(wr[i] + k);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        xv[i] = any_load_tail(xr[i], k, p.k);
        wv[i] = any_load_tail(wr[i], k, p.k);
      }
    }
  };
  v4f acc[TM][2] = {};
  load(0);
  for (int k0 = 0; k0 < p.k; k0 += 64) {
    if (k0) __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (threadIdx.x >> 3) + HALF * i, at = r * 128 + ((chunk ^ ((r >> 1) & 7)) << 4);
      *reinterpret_cast<u4*>(lds + at) = xv[i];
      *reinterpret_cast<u4*>(lds + BM * 128 + at) = wv[i];
    }
    __syncthreads();
    if (k0 + 64 < p.k) load(k0 + 64);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u4 a[TM], b[2];
      const int off = ((4 * s + g) ^ (lr >> 1)) << 4;
#pragma unroll
      for (int i = 0; i < TM; ++i) a[i] = *reinterpret_cast<const u4*>(lds + (16 * (TM * wm + i) + lr) * 128 + off);
#pragma unroll
      for (int j = 0; j < 2; ++j)  // gate/up: this wave's 16 gate rows, then its 16 up rows
        b[j] = *reinterpret_cast<const u4*>(lds + (BM + (GU ? HALF * j + 16 * wn : 32 * wn + 16 * j) + lr) * 128 + off);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma_bf16(b[j], a[i], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t row = m0 + 16 * (TM * wm + i) + lr;
    if (row >= p.m) continue;
    if constexpr (GU) {
      linear_epilogue4<true>(p, row, n0 + 16 * wn + 4 * g, acc[i][0], acc[i][1]);
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        linear_epilogue4<false>(p, row, n0 + 32 * wn + 16 * j + 4 * g, acc[i][j], v4f{0, 0, 0, 0});
    }
  }
#endif
}

// Tile of linear_tile_kernel: KG groups of WAVES_M x WAVES_N waves of WM rows x WN
// weight rows, group g multiplying step g of each KG steps of 64 k; two LDS stages
// of KG steps each. A row is 128 bytes of a step, its 16-byte chunk c at c ^ ((r >>
// 1) & 7) (no bank conflicts in reads of 16 rows). v_mfma_f32_32x32x16_bf16 on the
// same tiles: 4096 x 4096 x 12288 344 against 315 (8192 x 8192 x 8192 844, 775).
template <int WM_, int WN_, int WAVES_M_, int WAVES_N_, int GROUPS_ = 1, int KG_ = 1>
struct LinearTile {
  static constexpr int GROUPS = GROUPS_;  // workgroups per CU
  static constexpr int WM = WM_, WN = WN_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_;
  static constexpr int KG = KG_, NWB = WAVES_M * WAVES_N, NW = NWB * KG, THREADS = 64 * NW;
  static constexpr int BM = WM * WAVES_M, BN = WN * WAVES_N;
  static constexpr int TM = WM / 16, TN = WN / 16;  // fragments per wave
  static constexpr int A_BLOCK = BM * 128, B_BLOCK = BN * 128;
  static constexpr int A_BYTES = KG * A_BLOCK, B_BYTES = KG * B_BLOCK, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int A_SLOTS = A_BYTES / 1024 / NW, B_SLOTS = B_BYTES / 1024 / NW;
  // a wave's DMA instructions per stage: first (X) the weight rows and the rows of
  // its first TM / 2 activation fragments, then (Y) the other rows
  static constexpr int Y = A_SLOTS / 2, X = B_SLOTS + A_SLOTS - Y, DMA = X + Y;
  static constexpr int LDS = 2 * STAGE_BYTES;
  static_assert(NW == 8 && LDS <= 160 * 1024, "eight waves");
  static_assert(A_BYTES % (2048 * NW) == 0 && B_BYTES % (2048 * NW) == 0, "whole instructions per wave");
  static_assert(TM % 2 == 0 && TN % 2 == 0 && TM % KG == 0 && KG <= 2, "step");
  static_assert(NW * (TM - TM / KG) * TN * 1024 <= LDS, "the groups' sums meet in the stages");
  static_assert(X <= TM * TN && Y <= 2 * TN, "one DMA instruction per MFMA behind each barrier");
};

// The epilogue of a wave's EM x TN fragments of 16 x 16 sums (gate/up: the first half of
// each row of them the gate's, the other the up's): rows w0 .. of the tile's `here`
// from m0, columns from c0. A lane has four columns of row l % 16 of each fragment.
// Rows that went through LDS to be stored took 4096 x 4096 x 12288 317 us, not 309,
// and 4096 x 512 x 4096 29, not 22.5.
template <int EM, int TN, bool GU, bool RESID>
__device__ __forceinline__ void linear_store_tile(const LinearArgs& p, const v4f (&sum)[EM][TN], int part, int64_t m0,
                                                  int here, int w0, int c0) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int NC = GU ? TN / 2 : TN;
  const int lr = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
  if (p.parts > 1) {
    constexpr int MATS = GU ? 2 : 1;
#pragma unroll
    for (int i = 0; i < EM; ++i) {
      const int r = w0 + 16 * i + lr;
      if (r >= here) continue;
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int col = c0 + 16 * (j % NC) + 4 * g;
        if (col < p.n) *reinterpret_cast<v4f*>(linear_partial4(p, part, j / NC, MATS, m0 + r, col)) = sum[i][j];
      }
    }
    return;
  }
  v4f bias[NC], bias2[GU ? NC : 1];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    bias[j] = linear_bias4(p.bias, p.bias_f32, c0 + 16 * j + 4 * g, p.n);
    if constexpr (GU) bias2[j] = linear_bias4(p.bias2, p.bias_f32, c0 + 16 * j + 4 * g, p.n);
  }
  // Two fragments side by side (or, of one column of them, one below the other) trade
  // halves, so that a lane has eight columns of a row, 16 bytes: lanes of even
  // groups of 16 the first's columns 4 g .., those of odd groups the second's 4 (g -
  // 1) ..
  constexpr bool SIDE = NC > 1;
  auto trade = [](uint2 (&v)[2]) {
    auto swap = [](uint32_t& x, uint32_t& y) {
      const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
      x = r[0], y = r[1];
    };
    swap(v[0].x, v[1].x);
    swap(v[0].y, v[1].y);
  };
  // row and first column of this lane's eight of the pair (i, j)
  auto row_of = [&](int i) { return w0 + 16 * i + (SIDE || !(g & 1) ? 0 : 16) + lr; };
  auto col_of = [&](int j) { return c0 + 16 * j + (SIDE && (g & 1) ? 16 : 0) + 8 * (g >> 1); };
  constexpr int IS = SIDE ? 1 : 2, JS = SIDE ? 2 : 1;
#pragma unroll
  for (int i = 0; i < EM; i += IS)
#pragma unroll
    for (int j = 0; j < NC; j += JS) {
      const int row = row_of(i), col = col_of(j);
      const bool inside = row < here && col < p.n;
      uint2 res[2] = {{0, 0}, {0, 0}};
      if constexpr (RESID) {
        if (inside) linear_load8(p.residual + (m0 + row) * p.residual_stride + col, p.n - col, res);
        trade(res);
      }
      uint2 out[2];
      v4f y[2], y2[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int ii = i + (SIDE ? 0 : h), jj = j + (SIDE ? h : 0);
        y[h] = sum[ii][jj] + bias[jj];
        if constexpr (GU) y2[h] = sum[ii][jj + NC] + bias2[jj];
      }
      linear_act(y, p.act);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (GU) y[h] *= y2[h];
        if constexpr (RESID) y[h] += v4f{bf16_lo(res[h].x), bf16_hi(res[h].x), bf16_lo(res[h].y), bf16_hi(res[h].y)};
        out[h] = uint2{pack_bf16x2(y[h][0], y[h][1]), pack_bf16x2(y[h][2], y[h][3])};
      }
      if (p.out_f32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = w0 + 16 * (i + (SIDE ? 0 : h)) + lr, c = c0 + 16 * (j + (SIDE ? h : 0)) + 4 * g;
          if (r < here && c < p.n) linear_store4(p, m0 + r, c, y[h]);
        }
        continue;
      }
      trade(out);
      if (inside) linear_store8(static_cast<uint16_t*>(p.out) + (m0 + row) * p.out_stride + col, p.n - col, out);
    }
#endif
}

// Many rows: tiles of BM rows x BN weight rows through two LDS stages filled by
// DMA, as the FP8 products' (gemm_f8.hip): a stage is filled in two parts, X and Y.
// Behind a barrier in the middle of a step X has been read by every wave and is
// loaded for two steps on, behind one before the step's last row of MFMAs the same
// goes for Y; each barrier also waits for the part that the MFMAs behind it read.
// So every load has a step and a half to land.
//
// 256 x 256 tiles: 4096 x 4096 x 12288 303 to 313 by card, 1.32 to 1.36 PFLOP/s (the
// library's product 279 to 330), 8192 x 8192 x 8192 743 to 761 (690 to 715). MFMA busy
// two thirds of the cycles at 1.9 to 2.0 GHz; with operands of zeros the same code
// takes 257, so a fifth of the time is the clock that the power leaves. Without the
// epilogue 278. Four waves of 128 x 128, which read a third less LDS, run the main loop
// in the same time and a longer epilogue (322 against 309).
template <class T, bool GU, bool RESID>
__global__ __launch_bounds__(T::THREADS, 2 * T::GROUPS) void linear_tile_kernel(const LinearArgs p, int tiles_m,
                                                                                int tiles_n) {
#if defined(__HIP_DEVICE_COMPILE__)
  extern __shared__ __align__(16) char lds[];
  constexpr int TM = T::TM, TN = T::TN, COLS = GU ? T::BN / 2 : T::BN;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, g = lane >> 4;
  const int kg = T::KG == 1 ? 0 : wave / T::NWB, wb = wave % T::NWB;  // group, wave in it
  const int wm = wb / T::WAVES_N, wn = wb % T::WAVES_N;
  int tm, tn;
  // (an XCD takes tiles of one part: 620 x 17408 x 5120 in 4 parts 113, so 111)
  const int tiles = tiles_m * tiles_n, place = place_of_block(blockIdx.x, gridDim.x);
  const int part = p.parts == 1 ? 0 : place / tiles;
  tile_of_place(place - part * tiles, tiles_m, tiles_n, tm, tn);
  const int64_t m0 = (int64_t)tm * T::BM;
  const int n0 = tn * COLS;
  const int here = p.m - m0 < T::BM ? (int)(p.m - m0) : T::BM, cols = p.n - n0 < COLS ? p.n - n0 : COLS;
  // blocks of 64 k: this part's
  const int all = (p.k + 63) / 64, first = (int)((int64_t)all * part / p.parts);
  const int blocks = (int)((int64_t)all * (part + 1) / p.parts) - first, steps = (blocks + T::KG - 1) / T::KG;

  // This wave's DMA: an instruction moves 8 rows of a step, the first half of a
  // wave's A instructions rows of the first TM / 2 fragments of either row of
  // waves. Rows past the end repeat the last.
  auto a_piece = [&](int s) {  // 8 rows of the block
    constexpr int H = T::A_SLOTS / 2;
    constexpr int PER = T::WM / 16;
    const int hi = s >= H, q = wb * H + s % H;
    return q / PER * (2 * PER) + hi * PER + q % PER;
  };
  auto chunk_of = [&](int r) { return (lane & 7) ^ ((r >> 1) & 7); };
  int a_voff[T::A_SLOTS], b_voff[T::B_SLOTS];
#pragma unroll
  for (int s = 0; s < T::A_SLOTS; ++s) {
    const int r = 8 * a_piece(s) + (lane >> 3), from = r < here ? r : here - 1;
    a_voff[s] = (int)(from * p.x_stride) * 2 + (chunk_of(r) << 4);
  }
#pragma unroll
  for (int s = 0; s < T::B_SLOTS; ++s) {
    const int r = 8 * (wb * T::B_SLOTS + s) + (lane >> 3);
    const int col = GU ? r % COLS : r, from = col < cols ? col : cols - 1;
    b_voff[s] = (int)(from * p.w_stride) * 2 + (chunk_of(r) << 4);
  }
  // gate/up: the first half of a group's waves load the gate's rows
  const bool up = GU && wb >= T::NWB / 2;
  const __amdgpu_buffer_rsrc_t a_rsrc =
      make_rsrc(p.x + m0 * p.x_stride, (uint32_t)(((here - 1) * p.x_stride + p.k) * 2));
  const __amdgpu_buffer_rsrc_t b_rsrc =
      make_rsrc((up ? p.w2 : p.w) + n0 * p.w_stride, (uint32_t)(((cols - 1) * p.w_stride + p.k) * 2));
  const __amdgpu_buffer_rsrc_t none = make_rsrc(p.x, 0);
  // Where k ends inside a step, this lane's chunk of it: past the end (an offset that
  // reads zeros) or not. A lane has two chunks, of odd and even pieces.
  int past[2];
#pragma unroll
  for (int o = 0; o < 2; ++o)
    past[o] = p.k % 64 != 0 && 8 * ((lane & 7) ^ (4 * o + (lane >> 4))) >= p.k % 64 ? (int)0x80000000u : 0;
  // DMA instruction x of step kt into `stage`, X first (steps past the end: zeros
  // that nothing counts, so that every step issues and waits alike)
  auto issue = [&](char* stage, int kt, int x) {
    const int block = T::KG * kt + kg;
    const bool in = block < blocks, last = first + block == all - 1;
    const int k = in ? (first + block) * 128 : 0;
    if (x < T::B_SLOTS) {
      const int piece = wb * T::B_SLOTS + x;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(in ? b_rsrc : none,
                                               (lds_ptr_t)(stage + T::A_BYTES + kg * T::B_BLOCK + piece * 1024), 16,
                                               b_voff[x] | (last ? past[piece & 1] : 0), k, 0, 0);
    } else {
      const int piece = a_piece(x - T::B_SLOTS);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(in ? a_rsrc : none, (lds_ptr_t)(stage + kg * T::A_BLOCK + piece * 1024),
                                               16, a_voff[x - T::B_SLOTS] | (last ? past[piece & 1] : 0), k, 0, 0);
    }
  };

  // a fragment's two halves (32 k each) in a stage
  const int swz = (g ^ (lr >> 1)) << 4;
  const int a_at = kg * T::A_BLOCK + (wm * T::WM + lr) * 128;
  const int b_at = T::A_BYTES + kg * T::B_BLOCK + ((GU ? wn * (T::WN / 2) : wn * T::WN) + lr) * 128;

  v4f acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = v4f{0, 0, 0, 0};
  auto body = [&](auto fragments, char* __restrict__ r0, char* __restrict__ r1) {
    constexpr int LIVE = decltype(fragments)::value;
    u4 av[2][2], bv[TN][2];
    auto read_a = [&](const char* stage, int i, u4 (&v)[2]) {
      v[0] = *reinterpret_cast<const u4*>(stage + a_at + i * 2048 + swz);
      v[1] = *reinterpret_cast<const u4*>(stage + a_at + i * 2048 + (swz ^ 64));
    };
    auto read_b = [&](const char* stage, int j, u4 (&v)[2]) {
      const char* at = stage + b_at + (GU && j >= TN / 2 ? T::B_BLOCK / 2 + (j - TN / 2) * 2048 : j * 2048);
      v[0] = *reinterpret_cast<const u4*>(at + swz);
      v[1] = *reinterpret_cast<const u4*>(at + (swz ^ 64));
    };
    // at most one stage's DMA behind what is waited for
    auto landed = [&]() {
      wait_vmcnt<T::DMA>();
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    auto step = [&](char* cur, const char* next, int kt) {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if (i == TM / 2 - 1) landed();  // this stage's Y; its X has been read
        if (i == TM - 1) landed();      // the next stage's X; this stage has been read
        if (i + 1 < LIVE) read_a(cur, i + 1, av[(i + 1) & 1]);
        if (LIVE && i + 1 == TM) read_a(next, 0, av[0]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < TN; ++j) {
#pragma unroll
          for (int h = 0; i < LIVE && h < 2; ++h) {
            acc[i][j] = mfma_bf16(bv[j][h], av[i & 1][h], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
          }
          if (LIVE && i == TM - 1) read_b(next, j, bv[j]);
          // X behind the first barrier, Y behind the second
          constexpr int SPAN = TM / 2 * TN;
          const int u = (i - (TM / 2 - 1)) * TN + j;
          if (u >= 0 && u < SPAN) {
#pragma unroll
            for (int x = u * T::X / SPAN; x < (u + 1) * T::X / SPAN; ++x) issue(cur, kt + 2, x);
          } else if (i == TM - 1) {
#pragma unroll
            for (int x = j * T::Y / TN; x < (j + 1) * T::Y / TN; ++x) issue(cur, kt + 2, T::X + x);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
#pragma unroll
    for (int x = 0; x < T::DMA; ++x) issue(r0, 0, x);
#pragma unroll
    for (int x = 0; x < T::DMA; ++x) issue(r1, 1, x);
    wait_vmcnt<T::DMA>();
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (LIVE > 0) {
      read_a(r0, 0, av[0]);
#pragma unroll
      for (int j = 0; j < TN; ++j) read_b(r0, j, bv[j]);
    }
    for (int kt = 0; kt < steps; kt += 2) {
      step(r0, r1, kt);
      if (kt + 1 < steps) step(r1, r0, kt + 1);
    }
  };
  // A wave with rows or columns past the end multiplies half of its fragments or none,
  // and shares the loads and barriers of the others (620 x 17408 x 5120 in 4 parts 125,
  // so 117; 300 x 5120 x 17408 on 128 x 128 tiles 89, 86).
  const int rows_left = here - wm * T::WM, cols_left = cols - wn * (GU ? T::WN / 2 : T::WN);
  if (rows_left <= 0 || cols_left <= 0)
    body(std::integral_constant<int, 0>{}, lds, lds + T::STAGE_BYTES);
  else if (rows_left <= T::WM / 2)
    body(std::integral_constant<int, TM / 2>{}, lds, lds + T::STAGE_BYTES);
  else
    body(std::integral_constant<int, TM>{}, lds, lds + T::STAGE_BYTES);

  constexpr int EM = TM / T::KG;  // rows of fragments that this wave stores, from fragment kg EM
  constexpr int NC = GU ? TN / 2 : TN;
  const int w0 = wm * T::WM + kg * EM * 16, c0 = n0 + wn * (16 * NC);
  // no DMA is on its way into LDS that another workgroup may have next
  wait_vmcnt<0>();
  v4f sum[EM][TN];
  if constexpr (T::KG == 1) {
#pragma unroll
    for (int i = 0; i < EM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) sum[i][j] = acc[i][j];
  } else {
    // two groups: each gives the other its part of the rows that the other stores
    __syncthreads();
    v4f* const mine = reinterpret_cast<v4f*>(lds) + wave * (EM * TN * 64) + lane;
    const v4f* const theirs = reinterpret_cast<v4f*>(lds) + (wave ^ T::NWB) * (EM * TN * 64) + lane;
#pragma unroll
    for (int i = 0; i < EM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
#pragma unroll
        for (int t = 0; t < 4; ++t) sum[i][j][t] = kg ? acc[i][j][t] : acc[EM + i][j][t];
        mine[(i * TN + j) * 64] = sum[i][j];
#pragma unroll
        for (int t = 0; t < 4; ++t) sum[i][j][t] = kg ? acc[EM + i][j][t] : acc[i][j][t];
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) sum[i][j] += theirs[(i * TN + j) * 64];
    __syncthreads();
  }
  linear_store_tile<EM, TN, GU, RESID>(p, sum, part, m0, here, w0, c0);
#endif
}

// The parts' sums, in their order, and the epilogue: four columns of a row per thread.
// Bound by the sums' bytes: 620 x 5120 in four parts 51 MB, 13 us.
template <bool GU>
__global__ __launch_bounds__(256) void linear_join_kernel(const LinearArgs p) {
  const int quads = (p.n + 3) / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / quads;
  if (row >= p.m) return;
  const int col = (int)(i - row * quads) * 4;
  constexpr int MATS = GU ? 2 : 1;
  v4f y = {0, 0, 0, 0}, y2 = {0, 0, 0, 0};
#pragma unroll 4
  for (int s = 0; s < p.parts; ++s) {
    y += *reinterpret_cast<const v4f*>(linear_partial4(p, s, 0, MATS, row, col));
    if constexpr (GU) y2 += *reinterpret_cast<const v4f*>(linear_partial4(p, s, 1, MATS, row, col));
  }
  linear_epilogue4<GU>(p, row, col, y, y2);
}

template <bool GU>
hipError_t launch_join(const LinearArgs& p, hipStream_t stream) {
  const int64_t quads = p.m * ((p.n + 3) / 4);
  linear_join_kernel<GU><<<(unsigned)((quads + 255) / 256), 256, 0, stream>>>(p);
  return hipGetLastError();
}

using Tile256 = LinearTile<128, 64, 2, 4>;        // 256 x 256
using Tile128 = LinearTile<64, 32, 2, 4, 2>;      // 128 x 128, two workgroups per CU
using Tile128K = LinearTile<64, 64, 2, 2, 1, 2>;  // 128 x 128, two steps of k at a time
using Tile128x256 = LinearTile<64, 64, 2, 4>;

template <class T, bool GU, bool RESID>
hipError_t launch_tile(const LinearArgs& p, hipStream_t stream) {
  static LaunchCache cache;
  auto* kernel = &linear_tile_kernel<T, GU, RESID>;
  if (hipError_t e = ensure_dynamic_lds(cache, reinterpret_cast<const void*>(kernel), T::LDS)) return e;
  constexpr int COLS = GU ? T::BN / 2 : T::BN;
  const int64_t tiles_m = (p.m + T::BM - 1) / T::BM, tiles_n = (p.n + COLS - 1) / COLS;
  if (tiles_m * tiles_n * p.parts > kMaxTiles) return hipErrorInvalidValue;
  kernel<<<(unsigned)(tiles_m * tiles_n * p.parts), T::THREADS, T::LDS, stream>>>(p, (int)tiles_m, (int)tiles_n);
  return hipGetLastError();
}

// Few rows: a workgroup owns R MT rows x R NT weight rows (gate/up: NT / 2 fragments
// of gate rows and the same of up), its eight waves split k in steps (wave w: steps w,
// w + 8, ..), D steps of each on their way in registers. Eight lanes load 128 bytes of
// a row in a row; through LDS of its own, with no barrier, a wave turns them into
// fragments, whose lanes hold 16 bytes of a row each. (Loads in the fragments' order,
// whose neighbouring lanes lie in different rows, go through the address unit lane
// by lane, 33 bytes per ns and CU: 37 x 4160 x 1352 10.3, so 8.2; 64 x 4096 x 12288
// 40.7, 28.2; 100 x 2048 x 768 7.6, 4.5.) The waves' sums meet in LDS and are added in
// wave order (the result does not depend on timing).
//
// R, the weight rows per fragment: 16, or 8 for up to 16 rows of x. A fragment of 8
// rows holds two pieces of k of each: of the 16 x 16 sums the two blocks on the
// diagonal count, one per piece. So twice as many tiles share the bytes. One row, R = 8
// and 16: 2048 x 128 2.9, 3.5; 4096 x 12288 18.3 (5.5 TB/s), 18.5; 17408 x 5120 32.2, 40.3.
// Two steps on their way gain where a step is one fragment (4096 x 12288 21.1, 19.1)
// and nothing in larger ones.
//
// together: an XCD's workgroups take tiles whose weight rows are the same one after
// another, as far as the weights are more than the output (37 x 4160 x 1352 8.2, 7.1;
// 49 x 8752 x 10278 on 16 x 16 tiles 140, 96; but 200 x 512 x 8192 13.5, 15.0).
//
// ONCE: weight rows that one workgroup alone reads are loaded past the caches' usual
// order (1 x 17408 x 5120 36.0, 32.2; 16 x 5120 x 17408 43.7, 39.5; 64 x 4096 x 12288 28.2, 26.7;
// but rows that other workgroups read too, 64 x 4096 x 12288 on 16 x 16 tiles, 49, 53).
//
// ANY: rows that start at any even byte. 16-byte loads there take twice the time of
// aligned ones (64 x 4097 x 1025 12.6, 64 x 4096 x 1024 7).
template <bool ANY, int R, int MT, int NT, int D, bool GU, bool ONCE>
__global__ __launch_bounds__(512) void linear_stream_kernel(const LinearArgs p, bool together) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int NW = 8, Q = 16 / R, NG = GU ? NT / 2 : NT, BM = R * MT, COLS = R * NG;
  constexpr int SK = 64 * Q;  // k per step
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, g = lane >> 4;
  int tm = blockIdx.y, tn = blockIdx.x;
  if (together) tile_of_block(blockIdx.y * gridDim.x + blockIdx.x, gridDim.x * gridDim.y, gridDim.y, gridDim.x, tm, tn);
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = tn * COLS;
  const int here = p.m - m0 < BM ? (int)(p.m - m0) : BM, cols = p.n - n0 < COLS ? p.n - n0 : COLS;
  const int steps = (p.k + SK - 1) / SK;
  // Load h of a fragment: eight rows of 128 bytes, row lane / 8 (R = 16: + 8 h), the
  // lane's 16 bytes at k = k_lane (R = 8: + 64 h) of a step.
  constexpr int HR = R / 8;  // rows of a fragment per lane
  const int k_lane = 8 * (lane & 7);
  auto row_of = [&](int fragment, int h, int rows) {  // rows past the end repeat the last
    const int r = R * fragment + 8 * h + (lane >> 3);
    return r < rows ? r : rows - 1;
  };
  const __amdgpu_buffer_rsrc_t a_rsrc =
      make_rsrc(p.x + m0 * p.x_stride, (uint32_t)(((here - 1) * p.x_stride + p.k) * 2));
  const uint32_t w_bytes = (uint32_t)(((cols - 1) * p.w_stride + p.k) * 2);
  const __amdgpu_buffer_rsrc_t w_rsrc = make_rsrc(p.w + n0 * p.w_stride, w_bytes);
  const __amdgpu_buffer_rsrc_t w2_rsrc = make_rsrc(GU ? p.w2 + n0 * p.w_stride : p.w, GU ? w_bytes : 0);
  int a_voff[MT][HR], w_voff[NG][HR];
  const uint16_t *a_row[ANY ? MT : 1][HR], *w_row[ANY ? NT : 1][HR];
#pragma unroll
  for (int h = 0; h < HR; ++h) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int64_t r = row_of(i, h, here);
      if constexpr (ANY) a_row[i][h] = p.x + (m0 + r) * p.x_stride;
      else a_voff[i][h] = (int)(r * p.x_stride + k_lane) * 2;
    }
#pragma unroll
    for (int j = 0; j < (ANY ? NT : NG); ++j) {
      const int64_t r = row_of(j % NG, h, cols);
      if constexpr (ANY) w_row[j][h] = (GU && j >= NG ? p.w2 : p.w) + (n0 + r) * p.w_stride;
      else w_voff[j][h] = (int)(r * p.w_stride + k_lane) * 2;
    }
  }
  struct Step {
    u4 w[NT][2], a[MT][2];
  } ring[D];
  auto load = [&](Step& b, int s) {
    if (s >= steps) return;
    if constexpr (ANY) {
      auto all = [&](auto load8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = SK * s + 64 * (R == 8 ? h : 0) + k_lane;
#pragma unroll
          for (int j = 0; j < NT; ++j) b.w[j][h] = load8(w_row[j][h % HR], k);
#pragma unroll
          for (int i = 0; i < MT; ++i) b.a[i][h] = load8(a_row[i][h % HR], k);
        }
      };
      if (SK * (s + 1) <= p.k)
        all([](const uint16_t* row, int k) { return any_load(row + k); });
      else
        all([&](const uint16_t* row, int k) { return any_load_tail(row, k, p.k); });
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        constexpr int PIECE = R == 8 ? 128 : 0;  // bytes of a row between the loads
        // chunks past the end of k: an offset that reads zeros
        const int past = SK * s + PIECE / 2 * h + k_lane >= p.k ? (int)0x80000000u : 0;
        auto load8 = [&](__amdgpu_buffer_rsrc_t rsrc, int voff, auto policy) {
          return __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (voff + PIECE * h) | past, s * (2 * SK),
                                                                              decltype(policy)::value));
        };
        const std::integral_constant<int, 0> usual{};
        const std::integral_constant<int, ONCE ? 2 : 0> weights{};  // (2: non-temporal)
#pragma unroll
        for (int j = 0; j < NT; ++j) b.w[j][h] = load8(GU && j >= NG ? w2_rsrc : w_rsrc, w_voff[j % NG][h % HR], weights);
#pragma unroll
        for (int i = 0; i < MT; ++i) b.a[i][h] = load8(a_rsrc, a_voff[i][h % HR], usual);
      }
    }
  };
  // This wave's fragments in LDS, 2 KiB each: 16 rows (R = 8: row r's piece q is row 8 q
  // + r) of 64 k, 16-byte chunk c of row r at c ^ ((r >> 1) & 7).
  char* const stage = lds + wave * ((MT + NT) * 2048);
  const int put_at = (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 4)) << 4);
  const int get_at = lr * 128 + ((g ^ (lr >> 1)) << 4);
  auto put = [&](int fragment, int h, u4 v) {
    *reinterpret_cast<u4*>(stage + fragment * 2048 + h * 1024 + (put_at ^ (h * 64))) = v;
  };
  auto get = [&](int fragment, int h) {
    return *reinterpret_cast<const u4*>(stage + fragment * 2048 + (get_at ^ (h * 64)));
  };
  v4f acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0, 0, 0, 0};
#pragma unroll
  for (int d = 0; d < D; ++d) load(ring[d], wave + NW * d);
  for (int s = wave; s < steps; s += NW * D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (s + NW * d >= steps) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int j = 0; j < NT; ++j) put(j, h, ring[d].w[j][h]);
#pragma unroll
        for (int i = 0; i < MT; ++i) put(NT + i, h, ring[d].a[i][h]);
      }
      __builtin_amdgcn_sched_barrier(0);
      load(ring[d], s + NW * (d + D));
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u4 w[NT], a[MT];
#pragma unroll
        for (int j = 0; j < NT; ++j) w[j] = get(j, h);
#pragma unroll
        for (int i = 0; i < MT; ++i) a[i] = get(NT + i, h);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j] = mfma_bf16(w[j], a[i], acc[i][j]);
      }
    }
  }
  // the waves' sums: fragment (i, j) of wave w at ((w MT + i) NT + j) KiB, behind the
  // stages (0.1 us less) or, to leave room for other workgroups, over them
  constexpr bool BEHIND = MT * NT == 1;
  if constexpr (!BEHIND) __syncthreads();
  v4f* sums = reinterpret_cast<v4f*>(lds + (BEHIND ? NW * (MT + NT) * 2048 : 0));
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) sums[((wave * MT + i) * NT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  // R rows x R / 4 quads of columns of a fragment
  constexpr int ITEMS = R * R / 4;
  for (int u = threadIdx.x; u < MT * NG * ITEMS; u += NW * 64) {
    const int fr = u % R, quad = u / R % (R / 4), j = u / ITEMS % NG, i = u / (ITEMS * NG);
    const int r = R * i + fr, col = n0 + R * j + 4 * quad;
    if (r >= here || col >= p.n) continue;
    v4f y = {0, 0, 0, 0}, y2 = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int at = (w * MT + i) * NT * 64 + R * q + fr + 16 * (R / 4 * q + quad);
        y += sums[at + j * 64];
        if constexpr (GU) y2 += sums[at + (NG + j) * 64];
      }
    linear_epilogue4<GU>(p, m0 + r, col, y, y2);
  }
#endif
}

template <bool ANY, int R, int MT, int NT, int D, bool GU, bool ONCE>
hipError_t launch_stream_kernel(const LinearArgs& p, hipStream_t stream) {
  constexpr int COLS = R * NT / (GU ? 2 : 1);
  constexpr int sums = 8 * MT * NT * 1024, stages = 8 * (MT + NT) * 2048;
  constexpr int lds = MT * NT == 1 ? sums + stages : sums > stages ? sums : stages;
  static LaunchCache cache;
  auto* kernel = &linear_stream_kernel<ANY, R, MT, NT, D, GU, ONCE>;
  if (lds > 64 * 1024)
    if (hipError_t e = ensure_dynamic_lds(cache, reinterpret_cast<const void*>(kernel), lds)) return e;
  const int64_t tiles_m = (p.m + R * MT - 1) / (R * MT);
  if (tiles_m > 65535) return hipErrorInvalidValue;
  kernel<<<dim3((unsigned)((p.n + COLS - 1) / COLS), (unsigned)tiles_m), 512, lds, stream>>>(
      p, tiles_m > 1 && p.k >= 4 * p.m);
  return hipGetLastError();
}

// ONCE from 16 MiB of weights on: fewer may still be in the last-level cache from the
// call before, where it gains nothing (8 x 4096 x 12288 from there 19.0, 20.4) and where
// others' data are kept from being pushed out. Loads of any alignment gain nothing by
// it, and the rule takes 32 x 16 tiles for fewer weights only.
template <bool ANY, int R, int MT, int NT, int D, bool GU>
hipError_t launch_stream(const LinearArgs& p, hipStream_t stream) {
  constexpr bool MAY = !ANY && !(MT == 2 && NT == 1);
  if (MAY && p.m <= R * MT && (int64_t)p.n * p.k * (GU ? 4 : 2) >= 16 << 20)
    return launch_stream_kernel<ANY, R, MT, NT, D, GU, MAY>(p, stream);
  return launch_stream_kernel<ANY, R, MT, NT, D, GU, false>(p, stream);
}

// Whether both operands' rows start on multiples of 16 bytes, k is whole chunks of
// those and 256 rows lie within 2 GiB (the fast kernels' loads).
bool rows_of_16(const LinearArgs& p) {
  auto at16 = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  constexpr int64_t most = (int64_t)1 << 21;
  return at16(p.x) && at16(p.w) && at16(p.w2) && p.k % 8 == 0 && p.x_stride % 8 == 0 && p.w_stride % 8 == 0 &&
         p.x_stride <= most && p.w_stride <= most;
}

template <int TM, int WN, bool GU>
hipError_t launch_any(const LinearArgs& p, hipStream_t stream) {
  constexpr int BM = 32 * TM, COLS = GU ? 16 * WN : 32 * WN;
  const dim3 grid((unsigned)((p.n + COLS - 1) / COLS), (unsigned)((p.m + BM - 1) / BM));
  linear_any_kernel<TM, WN, GU><<<grid, 128 * WN, 0, stream>>>(p);
  return hipGetLastError();
}

constexpr int64_t kCus = 256;

enum class LinearKernel {
  any, any128, s8x8, s8x16, s16x16, s16x32, s32x16, s32x32, s64x32, s64x64, t128x128, t128x128k, t256x256, t128x256
};

struct LinearPlan {
  LinearKernel kernel;
  int parts;
};

// The kernel for a product of m rows against n weight rows (gate/up: both), and the
// parts that k is split into: of the kernels' times as modelled here, in us, the least.
// The model's rates are measured ones, fitted to 8 to 12 kernels' times at 310 random
// shapes:
//  * few rows: a CU takes 80 bytes per ns of weights and rows (64 x 64: 60; all
//    together 15 TB/s; rows of any alignment 51 and 10), 2 us to sum and store 64 x 64, a part of a round's
//    start that another workgroup does not hide;
//  * tiles: a start and an end, and a step of 64 k each (two workgroups of 128 x 128
//    per CU: 1.0 for both); split, another launch that reads what they wrote;
//  * either no faster than memory (tiles: by the CUs that have one).
// What it decides, in both forms: 37 x 4160 x 1352 on 16 x 16 tiles 7.2, 32 x 16 8.9, 128
// x 128 in parts 12.2; 24 x 4096 x 4096 12.5 on 16 x 16, 10.3 on 16 x 32; 64 x 4096 x
// 12288 on 64 x 64 28.6, on 32 x 32 31.6, on 128 x 128 33.7; 64 x 17408 x 5120 on 64 x
// 32 67, on 128 x 128 in parts 43.8; 200 x 17408 x 5120 on 64 x 64 128, on 128 x 256 in
// parts 64; 512 x 4096 x 4096 on 64 x 64 39.3, on 128 x 128 in parts 31.4; 620 x 17408 x
// 5120 on 128 x 128 159, on 256 x 256 in 4 parts 111; 512 x 2049 x 4096, of any alignment,
// on 64 x 32 52, on 64 x 64 through LDS shared by the waves 33.5. Over 220 other
// random shapes its choice takes 2.5 % longer than the best of eight to twelve kernels.
LinearPlan linear_plan(int64_t m, int64_t rows_of_w, int k, bool gate_up, bool aligned) {
  auto tiles = [&](int bm, int bn) { return (m + bm - 1) / bm * ((rows_of_w + bn - 1) / bn); };
  auto rounds = [](int64_t workgroups, int64_t at_once) { return (float)((workgroups + at_once - 1) / at_once); };
  const float bytes = ((float)(rows_of_w + m) * k + (float)m * rows_of_w) * 2;
  LinearPlan best{LinearKernel::any, 1};
  float least = __builtin_huge_valf();
  auto consider = [&](LinearKernel kernel, int parts, float t) {
    if (t >= least) return;
    least = t;
    best = {kernel, parts};
  };
  // (at_once: workgroups that a CU holds)
  auto stream = [&](LinearKernel kernel, int bm, int bn, int at_once) {
    const int64_t of = tiles(bm, bn);
    const float r = rounds(of, kCus), cus = of < kCus ? of : kCus, all = (aligned ? 15e6f : 10e6f) / cus;
    const float most = !aligned ? 51e3f : bm * bn == 4096 ? 60e3f : 80e3f, rate = most < all ? most : all;
    const float t = r * ((bm + bn) * k * 2 / rate + bm * bn * (aligned ? 2.1f : 3.9f) / 4096) +
                    (r - 1) * (aligned ? 0.7f : 3.2f) / at_once + (bm == 8 ? 0.4f : 0);
    const float least_t = bytes / (bm == 8 && m > 8 ? 3.4e6f : 3.9e6f);
    consider(kernel, 1, (aligned ? 2.1f : 2.8f) + k * 1.2e-4f + (t > least_t ? t : least_t));
  };
  // (of kernels that memory holds alike the first: gate/up 3 x 472 x 2 12506 on 16 x 32
  // tiles 7.9, on 8 x 16 12.1; projections 1 x 5512 x 7229 on 8 x 8 17.5, on 16 x 16 19.5)
  if (m <= 16 && !gate_up) {
    stream(LinearKernel::s8x8, 8, 8, 4);
    stream(LinearKernel::s8x16, 8, 16, 3);
  }
  if (m <= 4096) {  // (a launch has 65535 tiles of rows)
    if (!gate_up) stream(LinearKernel::s16x16, 16, 16, 4);
    stream(LinearKernel::s16x32, 16, 32, 3);
    if (m <= 16 && gate_up) stream(LinearKernel::s8x16, 8, 16, 3);
    if (!gate_up) stream(LinearKernel::s32x16, 32, 16, 3);
    stream(LinearKernel::s32x32, 32, 32, 2);
    stream(LinearKernel::s64x32, 64, 32, 1);
    // (64 x 64 of any alignment does not fit the registers)
    if (aligned) stream(LinearKernel::s64x64, 64, 64, 1);
  }
  const int steps = (k + 63) / 64;
  if (!aligned) {
    const float r = rounds(tiles(64, 64), kCus), r128 = rounds(tiles(128, 128), kCus);
    consider(LinearKernel::any, 1, 3 + 1.2f * r + steps * (0.42f * r > 0.9f ? 0.42f * r : 0.9f));
    consider(LinearKernel::any128, 1, 3 + 2.5f * r128 + steps * (0.9f * r128 > 1.3f ? 0.9f * r128 : 1.3f));
    return best;
  }
  if (m <= 8) return best;  // (no scratch)
  auto from_memory = [&](int64_t workgroups) { return bytes / 4.9e6f * rounds(workgroups, kCus) * kCus / workgroups; };
  auto tile = [&](LinearKernel kernel, int bm, int bn, float start, float step, float pair) {
    const int64_t of = tiles(bm, bn);
    for (int parts : {1, 2, 3, 4, 6, 8}) {
      const bool two = pair > 0 && of * parts > kCus;
      const float r = rounds(of * parts, two ? 2 * kCus : kCus);
      if (parts > 1 && (r > 1 || steps < 8 * parts)) break;
      const float t = r * (start + (steps + parts - 1) / parts * (two ? pair : step));
      const float least_t = from_memory(of * parts) + start;
      consider(kernel, parts,
               (t > least_t ? t : least_t) + (parts > 1 ? 3 + (float)(parts * m * rows_of_w) * 8 / 5e6f : 0));
    }
  };
  tile(LinearKernel::t128x128, 128, 128, 4.5f, 0.57f, 1.0f);
  tile(LinearKernel::t128x128k, 128, 128, 5.5f, 0.53f, 0);
  tile(LinearKernel::t128x256, 128, 256, 6, 0.86f, 0);
  tile(LinearKernel::t256x256, 256, 256, 10, 1.40f, 0);
  return best;
}

template <class T, bool GU>
hipError_t launch_parts(const LinearArgs& p, hipStream_t stream) {
  if (p.parts == 1 && p.residual) return launch_tile<T, GU, !GU>(p, stream);
  if (hipError_t e = launch_tile<T, GU, false>(p, stream)) return e;
  return p.parts > 1 ? launch_join<GU>(p, stream) : hipSuccess;
}

template <bool GU>
hipError_t launch_rows(LinearArgs& p, void* workspace, hipStream_t stream) {
  const bool aligned = rows_of_16(p);
  const LinearPlan plan = linear_plan(p.m, (int64_t)p.n * (GU ? 2 : 1), p.k, GU, aligned);
  p.parts = plan.parts;
  p.partial = static_cast<float*>(workspace);
  auto few = [&](auto any) {
    constexpr bool ANY = decltype(any)::value;
    switch (plan.kernel) {
      case LinearKernel::s8x8: if constexpr (!GU) return launch_stream<ANY, 8, 1, 1, 2, GU>(p, stream);
      case LinearKernel::s8x16: return launch_stream<ANY, 8, 1, 2, 1, GU>(p, stream);
      case LinearKernel::s16x16: if constexpr (!GU) return launch_stream<ANY, 16, 1, 1, 2, GU>(p, stream);
      case LinearKernel::s16x32: return launch_stream<ANY, 16, 1, 2, 1, GU>(p, stream);
      case LinearKernel::s32x16: if constexpr (!GU) return launch_stream<ANY, 16, 2, 1, 1, GU>(p, stream);
      case LinearKernel::s32x32: return launch_stream<ANY, 16, 2, 2, 1, GU>(p, stream);
      case LinearKernel::s64x64: if constexpr (!ANY) return launch_stream<ANY, 16, 4, 4, 1, GU>(p, stream);
      default: return launch_stream<ANY, 16, 4, 2, 1, GU>(p, stream);
    }
  };
  switch (plan.kernel) {
    case LinearKernel::t128x128: return launch_parts<Tile128, GU>(p, stream);
    case LinearKernel::t128x128k: return launch_parts<Tile128K, GU>(p, stream);
    case LinearKernel::t256x256: return launch_parts<Tile256, GU>(p, stream);
    case LinearKernel::t128x256: return launch_parts<Tile128x256, GU>(p, stream);
    case LinearKernel::any: return launch_any<2, 2, GU>(p, stream);
    case LinearKernel::any128: return launch_any<4, 4, GU>(p, stream);
    default: return aligned ? few(std::false_type{}) : few(std::true_type{});
  }
}

}  // namespace

size_t linear_workspace_bytes(const LinearArgs& p, bool gate_up) {
  return rows_of_16(p) ? linear_workspace_bytes(p.m, p.n, p.k, gate_up) : 0;
}

size_t linear_workspace_bytes(int64_t m, int n, int k, bool gate_up) {
  if (k % 8 != 0) return 0;  // (only products of rows on 16 bytes are split)
  const int64_t matrices = gate_up ? 2 : 1;
  const LinearPlan plan = linear_plan(m, n * matrices, k, gate_up, true);
  return plan.parts > 1 ? (size_t)(plan.parts * matrices * m * ((n + 3) & ~3)) * 4 : 0;
}

const char* linear_kernel_name(int64_t m, int n, int k, bool gate_up, bool aligned) {
  static const char* const names[] = {"any",   "any128", "8x8",   "8x16",    "16x16",      "16x32",   "32x16",
                                      "32x32", "64x32",  "64x64", "128x128", "128x128x2", "256x256", "128x256"};
  return names[(int)linear_plan(m, (int64_t)n * (gate_up ? 2 : 1), k, gate_up, aligned).kernel];
}

hipError_t launch_linear(LinearArgs p, bool gate_up, void* workspace, hipStream_t stream) {
  return gate_up ? launch_rows<true>(p, workspace, stream) : launch_rows<false>(p, workspace, stream);
}

}  // namespace clef
