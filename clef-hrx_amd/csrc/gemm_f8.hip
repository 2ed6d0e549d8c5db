// Block-scaled FP8 products for gfx950 (layouts and the formula in f8.hpp).
//
// A block's codes are multiplied by v_mfma_scale_f32_16x16x128_f8f6f4 (one
// instruction covers a block's 128 k, accumulating in f32) with the powers of
// two of both scales in it (f8_split_scale), and the partial sum enters the f32
// accumulator by one fma with the factor that is left of sw, which rounds it once
// more. The tiled kernel lets the instruction add to the accumulator itself where
// every factor is one. Output values are rounded to bf16 once, behind the residual
// or SwiGLU. Inside the instruction the products of eight neighbouring k are cut
// to 2^-13 of the largest of them (a property of the FP8 matrix unit, measured
// with single products beside a pair that cancels); the eights and everything
// behind them add in f32. Against 64 bits the sums are off by about 1e-5 of their
// size, bf16 by 1.7e-3.
//
// Times below are in us. "From memory" means operands in turn that pass the
// last-level cache together (256 MB), as in a model whose layers follow each
// other; where two variants are compared, both ran in turn on one card. Cards
// differ by some percent.
#include "f8.hpp"

namespace clef {

namespace {

// The most values of a tile's rows that a split-k workgroup quantizes itself: ten
// passes of its threads, 0.3 us each (instructions, and loads of rows that every
// workgroup reads), against the quantizer's launch. From memory, m x k x n with
// one launch and with two: 64 x 1024 x 2048, four passes, 4.4 and 5.6; 64 x 1536 x
// 2048, six, 5.5 and 6.0; 8 x 4096 x 2048, eight, 8.9 and 8.5; 16 x 2560 x 2048,
// ten, 8.2 and 7.6, and 8 x 5120 x 8192 13.1 and 12.1. From eight passes up the
// device gains nothing more, but two launches take the host 3.5 us longer (8.6
// against 5.0 through the binding), which is what such calls wait for.
constexpr int kQxValues = 10 * 512 * 8;

// Few rows: each workgroup owns 16 MT rows x 16 NT weight rows (gate/up: NT / 2
// fragments of gate rows and the same of up), its eight waves split the
// blocks of k (wave w: blocks w, w + 8, ..). Operands go straight into
// registers: a weight fragment is two contiguous KiB in the operand order and is
// used by this workgroup's rows only, so LDS would add a trip and nothing
// else. The waves' sums meet in LDS and are added in wave order (the result does
// not depend on timing).
//
// A wave has one block of k on its way: a second or third costs registers, and
// with them workgroups per CU, and gained nothing anywhere (16 x 32 tiles, 1, 2
// and 3 blocks, three weights in turn, mostly from the last-level cache: 37 x 4160 x
// 1352 5.4, 5.8, 5.7; 3 x 15208 x 1960 9.4, 9.5, 10.1; 16 x 64, 60 tokens of 60
// experts top-1 gate/up 408 x 2 2968 46, 55, 67). Waves without a block issue
// nothing: loads through empty resources took as long as others (1 x 448 x 2 1336
// with two blocks 3.1, 2.6 without them).
//
// QX: the rows come in bf16 (p.x) and every workgroup quantizes its tile's into
// LDS first, by the quantizer's rule, while its first weights are on their way.
template <int MT, int NT, bool QX, bool LISTS, bool GU, bool RESID>
__global__ __launch_bounds__(512) void f8_stream_kernel(const F8Args p) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int NW = 8, BM = 16 * MT, COLS = 16 * NT / (GU ? 2 : 1), NG = GU ? NT / 2 : NT;
  static_assert(!GU || NT % 2 == 0, "gate and up fragments");
  static_assert(!QX || (!LISTS && !GU), "rows quantized here");
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, g = lane >> 4;
  const int kb = p.kb, pitch = kb * 128;
  int expert = 0, first = 0, here = 0;
  int64_t m0 = 0;
  if constexpr (LISTS) {
    const F8Tiles<BM> tiles(p.lists);
    if ((int)blockIdx.y >= tiles.total) return;
    tiles.find(blockIdx.y, expert, first, here);
  } else {
    m0 = (int64_t)blockIdx.y * BM;
    here = p.rows - m0 < BM ? (int)(p.rows - m0) : BM;
  }
  const int n0 = blockIdx.x * COLS;

  // activation rows of this lane: byte and scale offsets (rows past the end
  // read the tile's last row; their sums are not stored)
  int a_voff[MT], s_voff[MT];
  __amdgpu_buffer_rsrc_t a_rsrc, s_rsrc;
  {
    const uint8_t* base = p.a + (LISTS ? 0 : m0 * pitch);
    const uint32_t bytes = (uint32_t)(LISTS ? p.rows * pitch : (int64_t)here * pitch);
    a_rsrc = make_rsrc(base, bytes);
    s_rsrc = make_rsrc(p.as, (uint32_t)(p.rows * kb * 4));
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    int r = 16 * i + lr;
    r = r < here ? r : here - 1;
    int64_t row = r;
    if constexpr (LISTS) {
      const int place = first + r;
      const int slot = p.lists.slots ? p.lists.slots[place] : place;
      // a slot outside the table reads nothing (it is not stored either)
      row = slot >= 0 && slot < p.lists.total ? slot / p.lists.div : 0;
      row = row < p.rows ? row : 0;
    }
    a_voff[i] = (int)((uint32_t)row * (uint32_t)pitch) + 16 * g;
    s_voff[i] = (int)((m0 + row) * 4);
  }
  const int nb = f8_blocks(p.n);
  const int64_t panel = ((int64_t)expert * nb + n0 / 128) * kb;
  const uint32_t panel_bytes = (uint32_t)kb * 16384u;
  const int w_voff = (n0 & 127) * 128 + lane * 16;
  const uint8_t* wp[2] = {p.w + panel * 16384, GU ? p.w2 + panel * 16384 : nullptr};
  const float* wsp[2] = {p.ws + panel, GU ? p.ws2 + panel : nullptr};
  constexpr int MATS = GU ? 2 : 1;

  // QX, behind the waves' sums: codes (rows 16 bytes apart beyond the pitch, so
  // that a fragment's 16 rows lie in different banks) and scales [rows][kb]
  const int q_pitch = pitch + 16, q_blocks = here * kb;
  char* const q_codes = lds + NW * MT * NT * 1024;
  float* const q_scales = reinterpret_cast<float*>(q_codes + (int)(p.rows < BM ? p.rows : BM) * q_pitch);
  // 16 lanes take a block, the workgroup 32 blocks in a pass; where the lanes'
  // block of the pass to be loaded, and of the one to be stored, lies
  struct Place {
    int row, block;
  };
  constexpr int QA = 4;  // passes loaded ahead
  uint4 xv[QA];
  const int q_col = (threadIdx.x & 15) * 8, q_rows = 32 / kb, q_rest = 32 - q_rows * kb;
  Place q_in{(int)(threadIdx.x >> 4) / kb, (int)(threadIdx.x >> 4) % kb}, q_out = q_in;
  auto q_next = [&](Place& at) {
    at.block += q_rest;
    at.row += q_rows + (at.block >= kb);
    at.block -= at.block >= kb ? kb : 0;
  };
  auto q_load = [&](int b0) {
#pragma unroll
    for (int s = 0; s < QA; ++s) {
      if (b0 + s * 32 >= q_blocks) break;
      const int col = q_in.block * 128 + q_col;
      xv[s] = uint4{0, 0, 0, 0};
      if (q_in.row < here && col < p.k) xv[s] = *reinterpret_cast<const uint4*>(p.x + (m0 + q_in.row) * p.x_stride + col);
      q_next(q_in);
    }
  };
  auto q_store = [&](int b0) {
#pragma unroll
    for (int s = 0; s < QA; ++s) {
      if (b0 + s * 32 >= q_blocks) break;
      const float scale = as_float(f8_scale_field(f8_block_amax(xv[s])) << 23);
      if (q_out.row < here) {
        *reinterpret_cast<uint2*>(q_codes + q_out.row * q_pitch + q_out.block * 128 + q_col) = f8_codes8(xv[s], scale);
        if (q_col == 0) q_scales[q_out.row * kb + q_out.block] = scale;
      }
      q_next(q_out);
    }
  };
  if constexpr (QX) q_load(0);

  struct Block {
    v4i w[NT][2], a[MT][2];
    float sa[MT], sw[MATS];
  } b;
  auto load = [&](int kt) {
    if (kt >= kb) return;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int mat = j / NG;
      const __amdgpu_buffer_rsrc_t wr = make_rsrc(wp[mat], panel_bytes);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        b.w[j][h] = __builtin_amdgcn_raw_buffer_load_b128(wr, w_voff + (j % NG) * 2048 + h * 1024, kt * 16384, 0);
    }
#pragma unroll
    for (int i = 0; i < (QX ? 0 : MT); ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) b.a[i][h] = __builtin_amdgcn_raw_buffer_load_b128(a_rsrc, a_voff[i] + 64 * h, kt * 128, 0);
      b.sa[i] = as_float(__builtin_amdgcn_raw_buffer_load_b32(s_rsrc, s_voff[i], (int)(kt * p.rows * 4), 0));
    }
#pragma unroll
    for (int m = 0; m < MATS; ++m)
      b.sw[m] = as_float(__builtin_amdgcn_raw_buffer_load_b32(make_rsrc(wsp[m], (uint32_t)kb * 4u), 0, kt * 4, 0));
  };
  v4f acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0, 0, 0, 0};
  load(wave);
  if constexpr (QX) {
    __builtin_amdgcn_sched_barrier(0);
    q_store(0);
    for (int b0 = QA * 32; b0 < q_blocks; b0 += QA * 32) {
      q_load(b0);
      q_store(b0);
    }
    __syncthreads();
  }
  for (int k = wave; k < kb; k += NW) {
    if constexpr (QX) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int r = 16 * i + lr, row = r < here ? r : here - 1;
        const char* at = q_codes + row * q_pitch + k * 128 + 16 * g;
        b.a[i][0] = *reinterpret_cast<const v4i*>(at);
        b.a[i][1] = *reinterpret_cast<const v4i*>(at + 64);
        b.sa[i] = q_scales[row * kb + k];
      }
    }
    F8Split sw[MATS];
#pragma unroll
    for (int m = 0; m < MATS; ++m) sw[m] = f8_split_scale(b.sw[m]);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const v8i_t av = join_halves(b.a[i][0], b.a[i][1]);
      const uint32_t sa = as_uint(b.sa[i]) << 1;  // the exponent in the top byte
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const F8Split& s = sw[j / NG];
        const v4f part = mfma_f8_scaled(join_halves(b.w[j][0], b.w[j][1]), av, v4f{0, 0, 0, 0}, s.exponent, sa, 3);
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[i][j][t] = __builtin_fmaf(part[t], s.factor, acc[i][j][t]);
      }
    }
    // the order as written: loads drawn up to here would need registers of
    // their own for another block
    __builtin_amdgcn_sched_barrier(0);
    load(k + NW);
    __builtin_amdgcn_sched_barrier(0);
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

template <int MT, int NT, bool QX, bool LISTS, bool GU, bool RESID>
hipError_t launch_stream(const F8Args& x, hipStream_t stream) {
  constexpr int BM = 16 * MT, COLS = 16 * NT / (GU ? 2 : 1), sums = 8 * MT * NT * 1024;
  static_assert(128 % COLS == 0, "a tile's columns lie in one weight block");
  // the most that kQxValues of codes, their padding and scales take
  constexpr int most = sums + (QX ? kQxValues + 16 * BM + kQxValues / 32 : 0);
  static_assert(most <= 160 * 1024, "LDS of a workgroup");
  static LaunchCache cache;
  auto* kernel = &f8_stream_kernel<MT, NT, QX, LISTS, GU, RESID>;
  if (most > 64 * 1024)
    if (hipError_t e = ensure_dynamic_lds(cache, reinterpret_cast<const void*>(kernel), most)) return e;
  const int lds = sums + (QX ? (int)(x.rows < BM ? x.rows : BM) * (x.kb * 132 + 16) : 0);
  if (lds > most) return hipErrorInvalidValue;
  const int64_t tiles_m = LISTS ? f8_most_tiles(x.lists.total, x.lists.experts, BM) : (x.rows + BM - 1) / BM;
  if (tiles_m > 65535) return hipErrorInvalidValue;
  const dim3 grid((unsigned)((x.n + COLS - 1) / COLS), (unsigned)tiles_m);
  kernel<<<grid, 512, lds, stream>>>(x);
  return hipGetLastError();
}

// Tile shape of f8_tile_kernel: KG groups of WAVES_M x WAVES_N waves of WM rows x
// WN weight rows, group g multiplying block g of each step's KG blocks of k; two
// LDS stages of one step each, for each block A rows (128 bytes each, 16-byte
// chunk c of row r at c ^ ((r >> 1) & 7)) and B fragments in the operand order.
// Behind the stages the rows' e8m0 scales of 16 blocks of k, as loaded (16 bytes
// per row) and, twice, turned into the order of use (per block of k a lane's TM
// rows side by side), the scales of the tile's one or two weight panels (256
// each, as they are or as pairs of the MFMA's exponent and the fma's factor)
// and, with lists, the tile's output rows.
template <int WM_, int WN_, int WAVES_M_, int WAVES_N_, int GROUPS_ = 1, int KG_ = 1>
struct F8Tile {
  static constexpr int GROUPS = GROUPS_;  // workgroups per CU
  static constexpr int WM = WM_, WN = WN_, WAVES_M = WAVES_M_, WAVES_N = WAVES_N_;
  static constexpr int NST = 2;  // LDS stages
  static constexpr int KG = KG_, NWB = WAVES_M * WAVES_N, NW = NWB * KG, THREADS = 64 * NW;
  static constexpr int BM = WM * WAVES_M, BN = WN * WAVES_N;
  static constexpr int TM = WM / 16, TN = WN / 16;  // fragments per wave
  static constexpr int A_BLOCK = BM * 128, B_BLOCK = BN * 128;
  static constexpr int A_BYTES = KG * A_BLOCK, B_BYTES = KG * B_BLOCK, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int A_SLOTS = A_BYTES / 1024 / NW, B_SLOTS = B_BYTES / 1024 / NW;
  // a wave's DMA instructions per stage: first (X) the weight fragments and the
  // rows of its first TM / 2 activation fragments, then (Y) the other rows
  static constexpr int Y = A_SLOTS / 2, X = B_SLOTS + A_SLOTS - Y, DMA = X + Y;
  static constexpr int SA_BYTES = BM * 16, SA = NST * STAGE_BYTES, ST = SA + SA_BYTES, SW = ST + 2 * SA_BYTES;
  static constexpr int ROWS = SW + 2 * 2048;
  static constexpr int LDS = ROWS + BM * 4;
  static constexpr int EPI = 16 * WN * 2;            // epilogue staging per wave
  static_assert(NW == 8 && (BN == 256 || BN == 128) && BM / 64 <= NW, "eight waves, one or two weight panels");
  static_assert(A_BYTES % (2048 * NW) == 0 && B_BYTES % (2048 * NW) == 0 && LDS <= 160 * 1024, "whole instructions per wave");
  static_assert(TM * TN % 4 == 0 && TM % 4 == 0 && TN % 2 == 0 && TM % KG == 0, "step");
  static_assert(NW * (TM - TM / KG) * TN * 1024 <= NST * STAGE_BYTES, "the groups' sums meet in the stages");
  static_assert(X <= TM / 2 * TN && Y <= TN, "one DMA instruction per MFMA behind each barrier");
};

// Many rows: tiles of BM rows x BN weight rows through a ring of LDS stages
// filled by DMA.
//
// A wave's step (one block of k) is TM rows of fragments times TN weight
// fragments. It holds the weight fragments of the step and reads an activation
// fragment one row of MFMAs ahead of its use. The rows' scales,
// powers of two, go into the MFMA. So do the weight's where they are (HW), and
// the MFMA adds to the accumulator itself. Of other weight scales the power of
// two goes there too (f8_split_scale), and the factor that is left is applied by four
// fmas to a partial sum two MFMAs after the MFMA that made it (half the MFMAs'
// issue time, run under them; with the rows' scales in those fmas 1711 x 5120 x 2
// 17408 took 295 us, not 288, and with all of the weight's 273, not 275, but
// partial sums of rows of 1e35 and more overflowed).
//
// A stage of LDS is filled in two parts: X (weights, the first half of each
// wave's activation rows) and Y (the other half). Behind a barrier in the
// middle of a step X has been read by every wave and is loaded for two steps
// on, behind one before the step's last row of MFMAs the same goes for Y; each
// barrier also waits for the part that the MFMAs behind it read. So every load
// has a step and a half to land, where loading a stage as a whole behind one
// barrier left one, with one DMA instruction per MFMA or less (all of them at
// once: 4 % slower). On 128 x 128 tiles four stages gain no more than two blocks
// of k at a time do (620 x 17408 x 5120 75 and 74 us).
//
// The tile: `here` rows from m0 (lists: the expert's, from place first) and COLS
// columns from n0.
template <class T, bool HW, bool LISTS, bool GU, bool RESID>
__device__ __forceinline__ void f8_tile(const F8Args& p, char* lds, int expert, int first, int here, int64_t m0, int n0) {
  constexpr int TM = T::TM, TN = T::TN;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, g = lane >> 4;
  const int kg = T::KG == 1 ? 0 : wave / T::NWB, wb = wave % T::NWB;  // group, wave in it
  const int wm = wb / T::WAVES_N, wn = wb % T::WAVES_N;
  const int kb = p.kb, pitch = kb * 128, kp = (kb + 15) / 16 * 16;
  const int steps = (kb + T::KG - 1) / T::KG;
  int* out_rows = reinterpret_cast<int*>(lds + T::ROWS);

  // B: this wave's weight fragments, consecutive ones of one panel (gate/up: the
  // first half of the waves the gate's, the second the up's); a panel past the
  // last column is empty
  constexpr int FRAGS = T::B_SLOTS / 2;
  const int nb = f8_blocks(p.n);
  const bool up = GU && wb >= T::NWB / 2;
  const int frag = n0 / 16 + (up ? wb - T::NWB / 2 : wb) * FRAGS, panel = frag / 8;
  const int64_t first_block = (int64_t)expert * nb * kb;
  const __amdgpu_buffer_rsrc_t b_rsrc = make_rsrc((up ? p.w2 : p.w) + (first_block + (int64_t)panel * kb) * 16384,
                                                  panel < nb ? (uint32_t)kb * 16384u : 0u);
  const int b_voff = frag % 8 * 2048 + lane * 16;
  const __amdgpu_buffer_rsrc_t none = make_rsrc(p.a, 0);
  auto issue_b = [&](char* stage, int kt, int x) {
    const int block = T::KG * kt + kg;
    const bool in = block < kb;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(in ? b_rsrc : none,
                                             (lds_ptr_t)(stage + T::A_BYTES + (T::B_SLOTS * wave + x) * 1024), 16, b_voff,
                                             (in ? block : 0) * 16384 + x * 1024, 0, 0);
  };
  // the first weights, before the rows are known (lists: two loads later)
#pragma unroll
  for (int x = 0; x < T::B_SLOTS; ++x) issue_b(lds, 0, x);
#pragma unroll
  for (int x = 0; x < T::B_SLOTS; ++x) issue_b(lds + T::STAGE_BYTES, 1, x);

  // this wave's DMA, of its group's blocks: A instruction s moves 8 rows, the
  // first half of a wave's instructions rows of the first TM / 2 fragments of
  // either row of waves
  int a_voff[T::A_SLOTS];
  auto a_piece = [&](int s) {  // KiB of the block
    constexpr int H = T::A_SLOTS / 2;
    constexpr int PER = T::WM / 16;  // KiB of half of a row of waves' rows
    const int hi = s >= H, q = wb * H + s % H;
    return q / PER * (2 * PER) + hi * PER + q % PER;
  };
  auto source_row = [&](int r) -> int64_t {  // row of a (dense: from m0); rows past the end repeat the last
    r = r < here ? r : here - 1;
    if constexpr (!LISTS) return r;
    const int slot = p.lists.slots ? p.lists.slots[first + r] : first + r;
    const int64_t row = slot >= 0 && slot < p.lists.total ? slot / p.lists.div : 0;
    return row < p.rows ? row : 0;
  };
#pragma unroll
  for (int s = 0; s < T::A_SLOTS; ++s) {
    const int r = 8 * a_piece(s) + (lane >> 3);
    a_voff[s] = (int)((uint32_t)source_row(r) * (uint32_t)pitch) + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
  }
  const __amdgpu_buffer_rsrc_t a_rsrc =
      make_rsrc(p.a + (LISTS ? 0 : m0 * pitch), (uint32_t)(LISTS ? p.rows * pitch : (int64_t)here * pitch));
  // scales: of the rows, 16 blocks of k at a time by the first BM / 64 waves
  const __amdgpu_buffer_rsrc_t s_rsrc =
      make_rsrc(p.ae + m0 * kp, (uint32_t)(LISTS ? p.rows * kp : (int64_t)here * kp));
  const int s_voff = (int)((uint32_t)source_row(64 * wave + lane) * (uint32_t)kp);
  auto issue_scales = [&](int chunk) {
    if (wave < T::BM / 64)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(s_rsrc, (lds_ptr_t)(lds + T::SA + wave * 1024), 16, s_voff, chunk * 16, 0,
                                               0);
  };
  // into the order of use, each row by the lane that loaded it: row wm WM + 16 i
  // + l of block kt at kt BM + wm WM + l TM + i
  auto turn_scales = [&](int chunk) {
    if (wave < T::BM / 64) {
      const int r = 64 * wave + lane;
      const v4u v = *reinterpret_cast<const v4u*>(lds + T::SA + r * 16);
      char* to = lds + T::ST + (chunk & 1) * T::SA_BYTES + r / T::WM * T::WM + r % 16 * TM + r % T::WM / 16;
#pragma unroll
      for (int k = 0; k < 16; ++k) to[k * T::BM] = (char)(v[k / 4] >> (8 * (k % 4)));
    }
  };
  issue_scales(0);
  // and of the panels (gate/up: gate, up), a thread each
  float panel_scale = 0.0f;
  {
    const int q = threadIdx.x >> 8, k = threadIdx.x & 255;
    const int of = n0 / 128 + (GU ? 0 : q);
    if (k < kb && of < nb) panel_scale = (GU && q ? p.ws2 : p.ws)[first_block + (int64_t)of * kb + k];
  }
  if constexpr (LISTS) {
    for (int r = threadIdx.x; r < T::BM; r += T::THREADS) {
      int slot = -1;
      if (r < here) {
        slot = p.lists.slots ? p.lists.slots[first + r] : first + r;
        slot = slot < p.lists.total ? slot : -1;
      }
      out_rows[r] = slot;
    }
  }
  // DMA instruction x of step kt into `stage`, X first (stages past the end:
  // zeros that nothing reads, so that every step issues and waits alike)
  auto issue = [&](char* stage, int kt, int x) {
    const int block = T::KG * kt + kg;
    const bool in = block < kb;
    const int k = in ? block : 0;
    if (x < T::B_SLOTS)
      issue_b(stage, kt, x);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(in ? a_rsrc : none,
                                               (lds_ptr_t)(stage + kg * T::A_BLOCK + a_piece(x - T::B_SLOTS) * 1024), 16,
                                               a_voff[x - T::B_SLOTS], k * 128, 0, 0);
  };

  // a fragment's two halves in a stage
  const int a_at0 = kg * T::A_BLOCK + (wm * T::WM + lr) * 128 + ((g ^ (lr >> 1)) << 4), a_at1 = a_at0 ^ 64;
  const int b_at = T::A_BYTES + kg * T::B_BLOCK + (GU ? wn * (TN / 2) : wn * TN) * 2048 + lane * 16;
  const char* const sa_at = lds + T::ST + wm * T::WM + lr * TM;
  using Panel = std::conditional_t<HW, float, v2f>;
  const Panel* const sw_at = reinterpret_cast<const Panel*>(lds + T::SW) + (GU ? 0 : wn * T::WN / 128) * 256;

  v4f acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = v4f{0, 0, 0, 0};
  auto body = [&](char* __restrict__ r0, char* __restrict__ r1) {
    constexpr int MATS = GU ? 2 : 1;
    v8i_t av[2], bv[TN];
    v4f part[4];               // !HW: partial sums on their way
    float sv[MATS], last[MATS];  // !HW: the panels' factors in this step and in the one before
    uint32_t sa[TM / 4], sa_next[TM / 4];  // the rows' exponents, four in each
    int sw_bits[MATS];         // the panels' exponents, in the top byte
    auto read_a = [&](const char* stage, int i) {
      const v4i lo = *reinterpret_cast<const v4i*>(stage + a_at0 + i * 2048);
      const v4i hi = *reinterpret_cast<const v4i*>(stage + a_at1 + i * 2048);
      return join_halves(lo, hi);
    };
    auto read_b = [&](const char* stage, int j) {
      const char* at = stage + b_at + (GU && j >= TN / 2 ? T::B_BLOCK / 2 + (j - TN / 2) * 2048 : j * 2048);
      return join_halves(*reinterpret_cast<const v4i*>(at), *reinterpret_cast<const v4i*>(at + 1024));
    };
    Panel sw[MATS];
    // of step kt (the step before still takes sa)
    auto read_scales = [&](int kt) {
      // (the block past an odd number of them: its products are zeros, and so is
      // its entry here, which lies below 256)
      const int block = T::KG * kt + kg;
#pragma unroll
      for (int t = 0; t < MATS; ++t) sw[t] = sw_at[t * 256 + (block & 255)];
      const char* at = sa_at + (block >> 4 & 1) * T::SA_BYTES + (block & 15) * T::BM;
      typedef uint32_t pack __attribute__((ext_vector_type(TM / 4)));
      const pack v = *reinterpret_cast<const pack*>(at);
#pragma unroll
      for (int i = 0; i < TM / 4; ++i) sa_next[i] = v[i];
    };
    auto take_scales = [&]() {
#pragma unroll
      for (int i = 0; i < TM / 4; ++i) sa[i] = sa_next[i];
#pragma unroll
      for (int t = 0; t < MATS; ++t) {
        if constexpr (HW) {
          sw_bits[t] = (int)(as_uint(sw[t]) << 1);
        } else {
          sw_bits[t] = (int)as_uint(sw[t][0]);
          last[t] = sv[t];
          sv[t] = sw[t][1];
        }
      }
    };
    auto add = [&](v4f& c, const v4f& v, float s) {
#pragma unroll
      for (int t = 0; t < 4; ++t) c[t] = __builtin_fmaf(v[t], s, c[t]);
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
        if (i == TM - 1) {
          landed();  // the next stage's X; this stage has been read
          read_scales(kt + 1);
        }
        av[(i + 1) & 1] = i + 1 < TM ? read_a(cur, i + 1) : read_a(next, 0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int bits = sw_bits[GU && j >= TN / 2 ? 1 : 0];
          if constexpr (HW) {
            acc[i][j] = mfma_f8_scaled(bv[j], av[i & 1], acc[i][j], bits, sa[i / 4], i % 4);
            __builtin_amdgcn_sched_barrier(0);
          } else {
            part[(i * TN + j) % 4] = mfma_f8_scaled(bv[j], av[i & 1], v4f{0, 0, 0, 0}, bits, sa[i / 4], i % 4);
            __builtin_amdgcn_sched_barrier(0);
            // the MFMA two before
            const int before = i * TN + j - 2, ii = (before + TM * TN) / TN % TM, jj = (before + TN) % TN;
            const int mat = GU && jj >= TN / 2 ? 1 : 0;
            add(acc[ii][jj], part[(before + 4) % 4], before >= 0 ? sv[mat] : last[mat]);
          }
          if (i == TM - 1) bv[j] = read_b(next, j);
          // X behind the first barrier, Y behind the second
          constexpr int SPAN = TM / 2 * TN;
          const int u = (i - (TM / 2 - 1)) * TN + j;
          if (u >= 0 && u < SPAN) {
#pragma unroll
            for (int x = u * T::X / SPAN; x < (u + 1) * T::X / SPAN; ++x) issue(cur, kt + T::NST, x);
          } else if (i == TM - 1 && j < T::Y) {
            issue(cur, kt + T::NST, T::X + j);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      take_scales();
    };
    // the weights of both stages are on their way; then the first scales (turned
    // and split once they have landed) and the rows
#pragma unroll
    for (int x = T::B_SLOTS; x < T::DMA; ++x) issue(r0, 0, x);
#pragma unroll
    for (int x = T::B_SLOTS; x < T::DMA; ++x) issue(r1, 1, x);
    wait_vmcnt<2 * T::A_SLOTS>();
    if constexpr (HW) {
      reinterpret_cast<float*>(lds + T::SW)[threadIdx.x] = panel_scale;
    } else {
      const F8Split split = f8_split_scale(panel_scale);
      reinterpret_cast<v2f*>(lds + T::SW)[threadIdx.x] = v2f{as_float((uint32_t)split.exponent), split.factor};
    }
    turn_scales(0);
    wait_vmcnt<T::A_SLOTS>();
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    read_scales(0);
    av[0] = read_a(r0, 0);
#pragma unroll
    for (int j = 0; j < TN; ++j) bv[j] = read_b(r0, j);
    if constexpr (!HW) {
#pragma unroll
      for (int t = 0; t < 4; ++t) part[t] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < MATS; ++t) sv[t] = 0.0f;
    }
    take_scales();
    // The scales of the next 16 blocks of k are loaded in the first half of these
    // and turned before the second (a branch inside a step instead made the
    // compiler spill).
    constexpr int HALF_STEPS = 8 / T::KG;
    for (int k0 = 0; k0 < steps; k0 += HALF_STEPS) {
      const bool second = k0 & HALF_STEPS;
      const int next = (k0 / (2 * HALF_STEPS) + 1) * 2 * HALF_STEPS;  // first step of the next 16 blocks
      if (next < steps) {
        if (second) {
          wait_vmcnt<T::NST * T::DMA>();
          turn_scales(next / (2 * HALF_STEPS));
        } else {
          issue_scales(next / (2 * HALF_STEPS));
        }
      }
      const int k1 = k0 + HALF_STEPS < steps ? k0 + HALF_STEPS : steps;
      for (int kt = k0; kt < k1; kt += T::NST) {
        step(r0, r1, kt);
        if (kt + 1 < steps) step(r1, r0, kt + 1);
      }
    }
    if constexpr (!HW) {
      // the last two partial sums
      add(acc[TM - 1][TN - 2], part[2], last[GU && TN > 2 ? 1 : 0]);
      add(acc[TM - 1][TN - 1], part[3], last[GU ? 1 : 0]);
    }
  };
  body(lds, lds + T::STAGE_BYTES);

  // epilogue: 16 rows at a time through the wave's own LDS (16-byte chunk c of
  // row r at c ^ (r & 7)), stored as 16-byte pieces of whole row segments; the
  // residual's loads all go out first
  constexpr int EM = TM / T::KG;  // rows of fragments that this wave stores, from fragment kg EM
  const int w0 = wm * T::WM + kg * EM * 16;
  uint2 res[RESID ? EM : 1][RESID ? TN : 1];
  if constexpr (RESID) {
#pragma unroll
    for (int i = 0; i < EM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int r = w0 + 16 * i + lr, col = n0 + wn * T::WN + 16 * j + 4 * g;
        res[i][j] = uint2{0, 0};
        if (r < here && col < p.n) res[i][j] = *reinterpret_cast<const uint2*>(p.residual + (m0 + r) * p.n + col);
      }
  }
  wait_vmcnt<0>();
  __syncthreads();
  v4f sum[EM][TN];
  if constexpr (T::KG == 1) {
#pragma unroll
    for (int i = 0; i < EM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) sum[i][j] = acc[i][j];
  } else {
    // two groups: each gives the other its part of the rows that the other stores
    static_assert(T::KG <= 2, "a pair of groups");
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
  constexpr int WC = GU ? T::WN / 2 : T::WN, ROW = WC * 2, CH = WC / 8;  // columns, bytes, chunks of a row
  constexpr int PER = 64 / CH;                                           // rows per store
  char* own = lds + wave * T::EPI;
  const int c0 = n0 + wn * WC;
#pragma unroll
  for (int i = 0; i < EM; ++i) {
    const int r0 = w0 + 16 * i;
#pragma unroll
    for (int j = 0; j < (GU ? TN / 2 : TN); ++j) {
      v4f y = sum[i][j];
      if constexpr (GU) {
#pragma unroll
        for (int t = 0; t < 4; ++t) y[t] = f8_swiglu(y[t], sum[i][j + TN / 2][t]);
      }
      if constexpr (RESID) {
        y[0] += bf16_lo(res[i][j].x);
        y[1] += bf16_hi(res[i][j].x);
        y[2] += bf16_lo(res[i][j].y);
        y[3] += bf16_hi(res[i][j].y);
      }
      const int chunk = 2 * j + (g >> 1);
      *reinterpret_cast<uint2*>(own + lr * ROW + ((chunk ^ (lr & (CH - 1))) << 4) + 8 * (g & 1)) =
          uint2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
    }
#pragma unroll
    for (int q = 0; q < (16 + PER - 1) / PER; ++q) {
      const int r = q * PER + lane / CH, chunk = lane % CH, col = c0 + 8 * chunk;
      if (PER > 16 && r >= 16) continue;
      const uint4 v = *reinterpret_cast<const uint4*>(own + r * ROW + ((chunk ^ (r & (CH - 1))) << 4));
      if (r0 + r >= here || col >= p.n) continue;
      int64_t row = m0 + r0 + r;
      if constexpr (LISTS) {
        row = out_rows[r0 + r];
        if (row < 0) continue;
      }
      *reinterpret_cast<uint4*>(p.out + row * p.n + col) = v;
    }
    asm volatile("" ::: "memory");
  }
}

// A tile of at most HALF::BM rows (an expert's last, mostly) runs in the shape
// HALF, of as many columns: experts' gate/up of 4096 tokens, 256 rows per expert
// and half of them a few more, 169 -> 155 us, with power-of-two scales 152 -> 144.
template <class T, class HALF, bool HW, bool LISTS, bool GU, bool RESID>
__global__ __launch_bounds__(T::THREADS, 2 * T::GROUPS) void f8_tile_kernel(const F8Args p, int tiles_m, int tiles_n) {
#if defined(__HIP_DEVICE_COMPILE__)
  extern __shared__ __align__(16) char lds[];
  static_assert(HALF::BN == T::BN && HALF::THREADS == T::THREADS && HALF::LDS <= T::LDS, "one launch");
  constexpr int COLS = GU ? T::BN / 2 : T::BN;
  int tm, tn, expert = 0, first = 0, here;
  int64_t m0 = 0;
  if constexpr (LISTS) {
    // consecutive blocks of an XCD take the columns of one tile of rows, then the
    // expert's next rows: both operands stay in its L2. The grid has blocks for
    // the most tiles that such lists can have; those there are shared evenly.
    const F8Tiles<T::BM> tiles(p.lists);
    // (lists that overlap can make more than the grid has blocks for)
    const int blocks = (tiles.total < tiles_m ? tiles.total : tiles_m) * tiles_n, per = blocks / 8, b = blockIdx.x;
    if (b >= blocks) return;
    const int r = b < 8 * per ? (b % 8) * per + b / 8 : b;
    tm = r / tiles_n;
    tn = r - tm * tiles_n;
    tiles.find(tm, expert, first, here);
  } else {
    tile_of_block(blockIdx.x, tiles_m * tiles_n, tiles_m, tiles_n, tm, tn);
    m0 = (int64_t)tm * T::BM;
    here = p.rows - m0 < T::BM ? (int)(p.rows - m0) : T::BM;
  }
  if (HALF::BM < T::BM && here <= HALF::BM)
    f8_tile<HALF, HW, LISTS, GU, RESID>(p, lds, expert, first, here, m0, tn * COLS);
  else
    f8_tile<T, HW, LISTS, GU, RESID>(p, lds, expert, first, here, m0, tn * COLS);
#endif
}

using F8Tile256 = F8Tile<128, 64, 2, 4>;           // 256 x 256
using F8Tile256H = F8Tile<64, 64, 2, 4>;           // 128 x 256
using F8Tile128 = F8Tile<64, 32, 2, 4, 2>;         // 128 x 128, two workgroups per CU
using F8Tile128K = F8Tile<64, 64, 2, 2, 1, 2>;     // 128 x 128, two blocks of k at a time

template <class T, class HALF, bool HW, bool LISTS, bool GU, bool RESID>
hipError_t launch_tile(const F8Args& x, hipStream_t stream) {
  static LaunchCache cache;
  auto* kernel = &f8_tile_kernel<T, HALF, HW, LISTS, GU, RESID>;
  if (hipError_t e = ensure_dynamic_lds(cache, reinterpret_cast<const void*>(kernel), T::LDS)) return e;
  constexpr int COLS = GU ? T::BN / 2 : T::BN;
  const int64_t tiles_m = LISTS ? f8_most_tiles(x.lists.total, x.lists.experts, T::BM) : (x.rows + T::BM - 1) / T::BM;
  const int tiles_n = (x.n + COLS - 1) / COLS;
  if (tiles_m * tiles_n > kMaxTiles) return hipErrorInvalidValue;
  kernel<<<(unsigned)(tiles_m * tiles_n), T::THREADS, T::LDS, stream>>>(x, (int)tiles_m, tiles_n);
  return hipGetLastError();
}

constexpr int64_t kCus = 256;

// Tiles of the split-k kernel for m rows against n weight rows (gate/up: both);
// k256x256 where they are more than the CUs whatever the shape.
F8Kernel stream_kernel(int64_t m, int64_t n) {
  auto tiles = [&](int bm, int bn) { return (m + bm - 1) / bm * ((n + bn - 1) / bn); };
  if (tiles(16, 32) <= kCus || (m <= 16 && tiles(16, 64) > kCus)) return F8Kernel::k16x32;
  if (m <= 32 && tiles(32, 32) <= kCus) return F8Kernel::k32x32;
  if (tiles(16, 64) <= kCus) return F8Kernel::k16x64;
  if (tiles(32, 64) <= kCus) return F8Kernel::k32x64;
  return tiles(64, 64) <= kCus ? F8Kernel::k64x64 : F8Kernel::k256x256;
}

}  // namespace

// From the smallest tiles up (all of it measured from memory, f32 scales): 16 x 32,
// 16 x 64, 32 x 64 and 64 x 64 of the split-k kernel while they are at most one per
// CU (m x k x n: 133 x 5784 x 288 6.4 on 16 x 32 tiles, 7.9, 10.8, 16.6 on the larger
// ones; 170 x 3600 x 3808 25.3, 15.1, 16.1 and 13.4), and 32 x 32 where one tile
// has all rows and reads the weights once (20 x 14512 x 6848 22.6 against 29.7 on
// 16 x 64, 29 x 1072 x 7976 5.1 against 5.7); beyond, 128 x 128 tiles, two
// workgroups per CU (256 x 4096 x 12288: 24.6 against 40.7 on 64 x 64), and 256 x
// 256 tiles from three times their rounds over the CUs up, a 256 x 256 round
// taking about three of 128 x 128 (1024 x 4096 x 12288, 1 and 3 rounds: 53
// against 61; 1536, 2 and 5: 98 against 92; 4096, 3 and 12: 178 against 225).
// One tile of 16 rows against more columns than 256 tiles cover stays on 16 x
// 32 (16 x 5120 x 2 17408: 36 against 45.5 on 128 x 128). Where k is long and the
// 128 x 128 tiles cover a third of the CUs this is not the best: 200 x 17408 x 5120
// takes 71 on them and 66 on 64 x 64.
F8Kernel f8_kernel(int64_t m, int n, int kb, bool gate_up, bool pow2) {
  const int64_t rows_of_w = (int64_t)n * (gate_up ? 2 : 1);
  const F8Kernel few = stream_kernel(m, rows_of_w);
  if (few != F8Kernel::k256x256) return few;
  auto rounds = [&](int bm, int bn) { return ((m + bm - 1) / bm * ((rows_of_w + bn - 1) / bn) + kCus - 1) / kCus; };
  const int64_t small = rounds(128, 128);
  if (small >= 3 * rounds(256, 256)) return F8Kernel::k256x256;
  // One tile per CU: two blocks of k at a time on two groups of waves, which read
  // less LDS per MFMA and have more loads on their way, against a longer start and
  // the groups' sums (from memory, f32 scales, 128 x 128 tiles and these: 620 x
  // 17408 x 5120 82.7 and 76.2, 512 x 4096 x 4096 21.0 and 20.6, 768 x 512 x 4096, 4
  // blocks of k, 7.1 and 8.2; powers of two: 620 x 17408 x 5120 78.8 and 73.8, 300 x
  // 8192 x 8192 38.6 and 35.1, 300 x 5120 x 2 5120 27.7 and 26.1, 256 x 4096 x
  // 12288 24.2 and 24.3, 640 x 2048 x 2048 12.2 and 13.0).
  return small <= 1 && kb >= (pow2 ? 40 : 16) ? F8Kernel::k128x128k : F8Kernel::k128x128;
}

// Experts with few rows, whose weights are read once whatever the tile. As
// many tiles as CUs: 16 x 32, then 16 x 64 (from memory: 8 slots of 128 experts,
// gate/up 2048 x 2 768, 8.3 on 16 x 64, 8.9 on 16 x 32 and 14.3 on 128 x 128; 57 of 8,
// 2928 x 464, 6.8 on 16 x 32, 8.0, 17.3). More: 16 x 64 below sixteen rows per expert
// (gate/up, 540 slots of 128 568 x 2 1440 54.6 against 66.2 on 128 x 128, 793 of
// 60 3112 x 2 712 57.8 against 64.8; 1063 of 64 584 x 2 256, 16.6 rows each, 9.8
// against 9.4). The experts named: about total E / (total + E). Then as without
// lists, as if evenly filled (a little more, for those above the mean).
F8Kernel f8_kernel_lists(int64_t total, int64_t experts, int n, bool gate_up) {
  const int64_t rows_of_w = (int64_t)n * (gate_up ? 2 : 1), least = total < experts ? total : experts;
  const int64_t rows = total * 21 / 20 / least;
  const int64_t named = total * experts / (total + experts) > 1 ? total * experts / (total + experts) : 1;
  const int64_t down = named * ((rows + 15) / 16);
  if (f8_most_tiles(total, (int)experts, 16) <= 65535) {
    if (down * ((rows_of_w + 31) / 32) <= kCus) return F8Kernel::k16x32;
    if (down * ((rows_of_w + 63) / 64) <= kCus || total < 16 * experts) return F8Kernel::k16x64;
  }
  auto rounds = [&](int b) { return (least * ((rows + b - 1) / b) * ((rows_of_w + b - 1) / b) + kCus - 1) / kCus; };
  return rounds(128) >= 3 * rounds(256) ? F8Kernel::k256x256 : F8Kernel::k128x128;
}

namespace {

template <bool LISTS, bool GU, bool RESID>
hipError_t launch_rows(const F8Args& x, hipStream_t stream) {
  const F8Kernel kernel = LISTS ? f8_kernel_lists(x.lists.total, x.lists.experts, x.n, GU)
                                : f8_kernel(x.rows, x.n, x.kb, GU, x.pow2);
  if constexpr (!LISTS && !GU)
    if (x.x != nullptr) switch (kernel) {  // f8_project_fusable
        case F8Kernel::k16x32: return launch_stream<1, 2, true, false, false, RESID>(x, stream);
        case F8Kernel::k32x32: return launch_stream<2, 2, true, false, false, RESID>(x, stream);
        case F8Kernel::k16x64: return launch_stream<1, 4, true, false, false, RESID>(x, stream);
        case F8Kernel::k32x64: return launch_stream<2, 4, true, false, false, RESID>(x, stream);
        default: return hipErrorInvalidValue;
      }
  if constexpr (!LISTS) switch (kernel) {
      case F8Kernel::k32x32: return launch_stream<2, 2, false, false, GU, RESID>(x, stream);
      case F8Kernel::k32x64: return launch_stream<2, 4, false, false, GU, RESID>(x, stream);
      case F8Kernel::k64x64: return launch_stream<4, 4, false, false, GU, RESID>(x, stream);
      case F8Kernel::k128x128k:
        return x.pow2 ? launch_tile<F8Tile128K, F8Tile128K, true, false, GU, RESID>(x, stream)
                      : launch_tile<F8Tile128K, F8Tile128K, false, false, GU, RESID>(x, stream);
      default: break;
    }
  switch (kernel) {
    case F8Kernel::k16x32: return launch_stream<1, 2, false, LISTS, GU, RESID>(x, stream);
    case F8Kernel::k16x64: return launch_stream<1, 4, false, LISTS, GU, RESID>(x, stream);
    case F8Kernel::k128x128:
      return x.pow2 ? launch_tile<F8Tile128, F8Tile128, true, LISTS, GU, RESID>(x, stream)
                    : launch_tile<F8Tile128, F8Tile128, false, LISTS, GU, RESID>(x, stream);
    case F8Kernel::k256x256:
      return x.pow2 ? launch_tile<F8Tile256, F8Tile256H, true, LISTS, GU, RESID>(x, stream)
                    : launch_tile<F8Tile256, F8Tile256H, false, LISTS, GU, RESID>(x, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_f8_gemm(const F8Args& x, bool gate_up, hipStream_t stream) {
  if (gate_up) return launch_rows<false, true, false>(x, stream);
  return x.residual ? launch_rows<false, false, true>(x, stream) : launch_rows<false, false, false>(x, stream);
}

bool f8_project_fusable(int64_t m, int n, int k) {
  const F8Kernel kernel = stream_kernel(m, n);
  const int rows = kernel == F8Kernel::k16x32 || kernel == F8Kernel::k16x64   ? 16
                   : kernel == F8Kernel::k32x32 || kernel == F8Kernel::k32x64 ? 32
                                                                              : 0;
  return rows > 0 && (m < rows ? m : rows) * f8_pitch(k) <= kQxValues;
}

hipError_t launch_f8_experts(const F8Args& x, bool gate_up, hipStream_t stream) {
  return gate_up ? launch_rows<true, true, false>(x, stream) : launch_rows<true, false, false>(x, stream);
}

}  // namespace clef
