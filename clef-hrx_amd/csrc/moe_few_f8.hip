// A whole MoE layer for up to 16 tokens on block-scaled FP8 experts, in two
// launches: route + gate/up + SwiGLU, and down + combine + residual.
//   out[t] = sum_{e in S(t)} p_e Down_e (silu(Gate_e x_t) * Up_e x_t) + residual[t]
// S(t) the topk largest logits (ties: the lower id), p the softmax over them.
//
// What bounds it is the weights of the experts that a token names, each read once:
// 16 rows fill one matrix instruction, so the rows of a fragment are the tokens
// themselves, whether they name the expert or not, and there are no lists of rows.
// The rows stay bf16 (quantizing them would save no byte that counts): a weight's
// e4m3 codes become bf16 on their way to the matrix unit, exact with the scale's
// power of two, whose remaining factor enters the f32 sums behind each block of 128 k.
// The router's probability goes into h, in f32, so that the down products of all
// experts add up in one accumulator. h stays f32: it is held as the three bf16 that
// add up to it, whose products the matrix unit sums one by one, and the output is
// rounded once. (Two bf16 keep 16 bits of h: the layer of one token takes 15.8 us with
// them, 16.3 with three, that of sixteen 76.5 and 81.4.)
//
// Hidden 2048, width 768, 128 experts, top-8, weights from memory, in a graph: one
// token 16.4 us (10 and 6; 38 MB), sixteen 82 (48 and 28; 83 experts, 390 MB, 4.8
// TB/s). What it took: loads without branches between them (a branch makes the
// compiler wait for each, 5 us of the first launch at one token); one workgroup per
// CU over units with the next one's weights on their way (sixteen tokens' first
// launch 57 -> 47); the parts' sums by device-scope atomics instead of fences that
// write back whole caches (the second launch 143 -> 66, with h in two bf16).
#include "f8.hpp"
#include "linear.hpp"
#include "moe_few_f8.hpp"
#include "route.hpp"

namespace clef {

namespace {

constexpr int kTokens = kMoeFewTokens, kMaxExperts = kMoeFewExperts;
constexpr int kHParts = 3;  // bf16 that a value of h is held as

// What the second launch takes from the first: the experts named, ascending, and for
// each the rows of h of its tokens (-1: the token names others).
struct FewTable {
  int count;
  int expert[kMaxExperts];
  alignas(8) int16_t slot[kMaxExperts][kTokens];
};

// Routing of all tokens, in LDS of each workgroup of 512 threads, by expert.
struct FewRoutes {
  float p[kTokens][kMaxExperts];  // the probability
  uint8_t rank[kTokens][kMaxExperts];
  uint32_t tokens[kMaxExperts];   // the tokens that name it
};

// The experts named, one bit each, in scalar registers of every wave.
struct FewNamed {
  unsigned long long low, high;
  __device__ __forceinline__ int count() const { return __popcll(low) + __popcll(high); }
  // the i-th, i < count()
  __device__ __forceinline__ int expert(int i) const {
    const int lows = __popcll(low);
    unsigned long long mask = i < lows ? low : high;
    for (int n = i < lows ? i : i - lows; n > 0; --n) mask &= mask - 1;
    return (i < lows ? 0 : 64) + __builtin_ctzll(mask);
  }
};

// Workgroup barrier behind this wave's LDS accesses alone: global loads stay on
// their way (__syncthreads would wait for them).
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// f32 as integers of the same order, and back. Zeros are one number (v + 0); logits
// that take no part are the least of all.
constexpr int kNoLogit = (int)0x80000000u;
__device__ __forceinline__ int few_key(float v) {
  const int bits = (int)as_uint(v + 0.0f), key = bits ^ (bits >> 31 & 0x7FFFFFFF);
  return v > -__builtin_huge_valf() ? key : kNoLogit;  // (NaN too)
}
__device__ __forceinline__ float few_value(int key) { return as_float((uint32_t)(key ^ (key >> 31 & 0x7FFFFFFF))); }

__device__ __forceinline__ int few_row_max(int v) {
  auto larger = [](int x, int y) { return x > y ? x : y; };
  v = larger(v, route_impl::dpp_row<0xB1>(v));
  v = larger(v, route_impl::dpp_row<0x4E>(v));
  v = larger(v, route_impl::dpp_row<0x124>(v));
  return larger(v, route_impl::dpp_row<0x128>(v));
}
__device__ __forceinline__ float few_row_sum(float v) {
  auto turned = [](float x, auto ctrl) {
    return as_float((uint32_t)route_impl::dpp_row<decltype(ctrl)::value>((int)as_uint(x)));
  };
  v += turned(v, std::integral_constant<int, 0xB1>{});
  v += turned(v, std::integral_constant<int, 0x4E>{});
  v += turned(v, std::integral_constant<int, 0x124>{});
  return v + turned(v, std::integral_constant<int, 0x128>{});
}

// A wave takes a token (and the eighth behind it), its lanes two experts each,
// through topk rounds of "the largest logit left, the lowest id that has it", the
// maximum and the id as scalars; lane k % 64 keeps rank k. Logits of -inf and NaN take
// no part, nor does a probability that is zero: a token may name fewer than topk
// experts, or none.
__device__ __forceinline__ FewNamed few_route(const MoeFewArgs& a, FewRoutes& r) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), experts = a.experts;
  constexpr int PER = kTokens / 8;
  uint32_t bits[PER][2];  // past the last expert or token: of another, not used
  const int logits = a.tokens * experts;
  if (a.logits_f32) {
    const __amdgpu_buffer_rsrc_t lr = make_rsrc(a.logits, (uint32_t)logits * 4);
#pragma unroll
    for (int n = 0; n < PER; ++n)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        bits[n][s] = __builtin_amdgcn_raw_buffer_load_b32(lr, ((wave + 8 * n) * experts + 64 * s + lane) * 4, 0, 0);
  } else {
    const __amdgpu_buffer_rsrc_t lr = make_rsrc(a.logits, (uint32_t)logits * 2);
#pragma unroll
    for (int n = 0; n < PER; ++n)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        bits[n][s] =
            (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(lr, ((wave + 8 * n) * experts + 64 * s + lane) * 2, 0, 0) << 16;
  }
  if (threadIdx.x < kMaxExperts) r.tokens[threadIdx.x] = 0;
  lds_barrier();
  for (int n = 0; n < PER; ++n) {
    const int t = wave + 8 * n;
    if (t >= a.tokens) break;
    int key[2], mine[2] = {kNoLogit, kNoLogit}, id[2] = {0, 0}, first = kNoLogit;
#pragma unroll
    for (int s = 0; s < 2; ++s) key[s] = 64 * s + lane < experts ? few_key(as_float(bits[n][s])) : kNoLogit;
    for (int k = 0; k < a.topk; ++k) {
      const int row = few_row_max(key[0] > key[1] ? key[0] : key[1]);
      int best = __builtin_amdgcn_readlane(row, 0);
#pragma unroll
      for (int l = 16; l < 64; l += 16) {
        const int other = __builtin_amdgcn_readlane(row, l);
        best = other > best ? other : best;
      }
      if (best == kNoLogit) break;
      const unsigned long long low = __ballot(key[0] == best), high = __ballot(key[1] == best);
      const int e = low != 0 ? __builtin_ctzll(low) : 64 + __builtin_ctzll(high);
      first = k == 0 ? best : first;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (64 * s + lane == k) {
          mine[s] = best;
          id[s] = e;
        }
        key[s] = 64 * s + lane == e ? kNoLogit : key[s];
      }
    }
    const float best = few_value(first);
    float p[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      // (equal ones first: infinities have no difference)
      const float v = few_value(mine[s]);
      p[s] = mine[s] == kNoLogit ? 0.0f : v == best ? 1.0f : __builtin_amdgcn_exp2f((v - best) * 1.44269504088896341f);
    }
    const int rows = (int)as_uint(few_row_sum(p[0] + p[1]));
    float sum = 0.0f;
#pragma unroll
    for (int l = 0; l < 64; l += 16) sum += as_float((uint32_t)__builtin_amdgcn_readlane(rows, l));
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const float q = p[s] / sum;
      if (q > 0.0f) {
        r.p[t][id[s]] = q;
        r.rank[t][id[s]] = (uint8_t)(64 * s + lane);
        atomicOr(&r.tokens[id[s]], 1u << t);
      }
    }
  }
  __syncthreads();
  return {__ballot(r.tokens[lane] != 0), __ballot(r.tokens[64 + lane] != 0)};
}

// A block's scale as 2^e, which the codes are converted with, and the factor that is
// left for the f32 sum. |e| <= 110: every code, 2^-9 .. 448, times 2^e is a normal
// bf16, so the conversion is exact; scales beyond keep the rest in the factor.
struct FewScale {
  float pow2, factor;
};
__device__ __forceinline__ FewScale few_scale(float s) {
  const int field = (int)(as_uint(s) >> 23 & 0xFFu), e = field < 17 ? 17 : field > 237 ? 237 : field;
  return {as_float((uint32_t)e << 23), __builtin_ldexpf(s, 127 - e)};
}

// 16 codes of a weight row to bf16 times 2^e.
__device__ __forceinline__ void few_bf16(v4i codes, float pow2, u4 (&out)[2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bf16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[i], pow2, false);
    const bf16x2_t hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[i], pow2, true);
    out[i / 2][2 * (i % 2)] = __builtin_bit_cast(uint32_t, lo);
    out[i / 2][2 * (i % 2) + 1] = __builtin_bit_cast(uint32_t, hi);
  }
}

// Operands of a fragment of R weight rows. R = 16: a block's half h as it lies
// (f8.hpp), lane l row l % 16, k = 64 h + 16 (l / 16) ..; R = 8, for up to 8 tokens:
// both halves in one load, lane l row l % 8 of half l / 8 % 2. The tokens' rows lie
// the same way, so that of R = 8's sums the two blocks on the diagonal count, one per
// half. Twice as many tiles cover the output that way.
template <int R>
struct FewLane {
  static constexpr int HALVES = R == 16 ? 2 : 1;  // loads per fragment and block
  int row, k;                                     // row of the fragment (and of x), first k in a block
  __device__ __forceinline__ FewLane() {
    const int lane = threadIdx.x & 63, lr = lane & 15;
    row = lr % R;
    k = 64 * (lr / R) + 16 * (lane >> 4);
  }
  // bytes into a block of this lane's 16 codes: rows from `first` (a multiple of R)
  __device__ __forceinline__ int at(int first) const {
    return (first >> 4) * 2048 + (first & 15) * 16 + (k >> 6) * 1024 + (k >> 4 & 3) * 256 + row * 16;
  }
};

// 16 codes, which no other workgroup reads. ONCE: past the caches' usual order.
template <bool ONCE>
__device__ __forceinline__ v4i few_weights(const uint8_t* at) {
  if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const v4i*>(at));
  return *reinterpret_cast<const v4i*>(at);
}

// Route, gate/up and SwiGLU. W waves split the blocks of k of 16 columns of h of one
// expert named, wave w of them the blocks w, w + W, .., whose part of x stays in
// registers (NB blocks; 0: any number, loaded each time); a unit is the 8 / W times 16
// columns of the workgroup's waves. The next unit's weights are on their way while a
// unit's sums meet in LDS, where one of the W waves in turn adds them in wave order.
template <int W, int NB, bool ONCE>
__global__ __launch_bounds__(512) void few_gate_up_kernel(const MoeFewArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ FewRoutes routes;
  __shared__ v4f sums[2][8][2][64];
  constexpr int COLS = 16 * (8 / W), R = 16, H = FewLane<R>::HALVES, XB = NB ? NB : 1;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const FewLane<R> me;
  const int kw = wave % W, column = 16 * (wave / W);  // wave of the W, first column in the unit
  const int kb = f8_blocks(a.hidden), tiles = (a.inter + COLS - 1) / COLS, panels = f8_blocks(a.inter);
  const int token = me.row < a.tokens ? me.row : a.tokens - 1;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, (uint32_t)(((a.tokens - 1) * a.x_stride + a.hidden) * 2));
  u4 xv[XB][2 * H];
  auto load_x = [&](int b, u4 (&v)[2 * H]) {
#pragma unroll
    for (int s = 0; s < 2 * H; ++s) {
      const int k = 128 * b + me.k + 64 * (s / 2) + 8 * (s % 2);
      v[s] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(
                                        xr, k < a.hidden ? (int)(token * a.x_stride + k) * 2 : (int)0x80000000u, 0, 0));
    }
  };
  if constexpr (NB > 0) {
#pragma unroll
    for (int i = 0; i < NB; ++i) load_x(kw + W * i, xv[i]);
  }
  const FewNamed named = few_route(a, routes);
  const int count = named.count(), units = count * tiles;
  FewTable& table = *static_cast<FewTable*>(a.table);
  if (blockIdx.x == 0) {
    if (tid == 0) table.count = count;
    for (int i = tid; i < count * kTokens; i += 512) {
      const int t = i % kTokens, e = named.expert(i / kTokens);
      if (t == 0) table.expert[i / kTokens] = e;
      table.slot[i / kTokens][t] = routes.tokens[e] >> t & 1 ? (int16_t)(t * a.topk + routes.rank[t][e]) : (int16_t)-1;
    }
    for (int i = tid; i < a.down_tiles; i += 512) a.arrived[i] = 0;
  }
  struct Unit {
    int e, n0;
    v4i w[XB][2][H];
    float scale[XB][2];
  };
  auto load_block = [&](Unit& q, int i, int b) {
    const int64_t block = ((int64_t)q.e * panels + q.n0 / 128) * kb + b;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const uint8_t* at = (m ? a.up : a.gate) + block * 16384 + me.at(q.n0 & 127);
#pragma unroll
      for (int h = 0; h < H; ++h) q.w[i][m][h] = few_weights<ONCE>(at + 1024 * h);
      q.scale[i][m] = (m ? a.up_scales : a.gate_scales)[block];
    }
  };
  // (without branches, which would make the loads wait for each other: past the
  // last unit or block the last one again, which nothing adds)
  auto load_unit = [&](Unit& q, int u) {
    u = u < units ? u : units - 1;
    q.e = __builtin_amdgcn_readfirstlane(named.expert(u / tiles));
    q.n0 = u % tiles * COLS + column;
#pragma unroll
    for (int i = 0; i < NB; ++i) load_block(q, i, kw + W * i < kb ? kw + W * i : kb - 1);
  };
  v4f acc[2];
  auto add_block = [&](const Unit& q, int i, const u4 (&x)[2 * H]) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const FewScale scale = few_scale(q.scale[i][m]);
      v4f part = {0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < H; ++h) {
        u4 wv[2];
        few_bf16(q.w[i][m][h], scale.pow2, wv);
#pragma unroll
        for (int s = 0; s < 2; ++s) part = mfma_bf16(wv[s], x[2 * h + s], part);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[m][t] = __builtin_fmaf(part[t], scale.factor, acc[m][t]);
    }
  };
  if ((int)blockIdx.x >= units) return;
  Unit q;
  load_unit(q, blockIdx.x);
  int turn = 0;
  for (int u = blockIdx.x; u < units; u += gridDim.x, ++turn) {
    acc[0] = acc[1] = v4f{0, 0, 0, 0};
    const int e = q.e, n0 = q.n0;
    if constexpr (NB > 0) {
#pragma unroll
      for (int i = 0; i < NB; ++i)
        if (kw + W * i < kb) add_block(q, i, xv[i]);
    } else {
      for (int b = kw; b < kb; b += W) {
        load_x(b, xv[0]);
        load_block(q, 0, b);
        add_block(q, 0, xv[0]);
      }
    }
    load_unit(q, u + gridDim.x);
#pragma unroll
    for (int m = 0; m < 2; ++m) sums[turn & 1][wave][m][lane] = acc[m];
    lds_barrier();
    if (kw != turn % W) continue;
    const int t = lane & 15, col = n0 + 4 * (lane >> 4);
    if (t >= a.tokens || !(routes.tokens[e] >> t & 1) || col >= a.inter) continue;
    v4f gate = {0, 0, 0, 0}, up = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      gate += sums[turn & 1][wave - kw + w][0][lane];
      up += sums[turn & 1][wave - kw + w][1][lane];
    }
    const float p = routes.p[t][e];
    uint16_t* at = a.h + (int64_t)(t * a.topk + routes.rank[t][e]) * a.inter + col;
    const int64_t plane = (int64_t)a.tokens * a.topk * a.inter;
    float y[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) y[s] = gate[s] * sigmoid_f32(gate[s]) * up[s] * p;
    // The upper half of what is left, three times: each takes 8 of the 24 bits, and
    // what it leaves is exact.
#pragma unroll
    for (int part = 0; part < kHParts; ++part) {
      uint32_t top[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        top[s] = as_uint(y[s]) & 0xFFFF0000u;
        // (nothing is left of an infinity)
        y[s] = __builtin_isinf(y[s]) ? 0.0f : y[s] - as_float(top[s]);
      }
      *reinterpret_cast<uint2*>(at + part * plane) = uint2{top[1] | top[0] >> 16, top[3] | top[2] >> 16};
    }
  }
#endif
}

// Down, combine and residual: R NT columns of the output. The pairs (expert named,
// block of k) of part blockIdx.y of gridDim.y are split among the eight waves, D on
// their way; their sums meet in LDS. With several parts the last workgroup of a
// tile to arrive adds the parts' sums, in their order.
template <int R, int NT, int D, bool ONCE>
__global__ __launch_bounds__(512) void few_down_kernel(const MoeFewArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ v4f sums[8][NT][64];
  __shared__ int last;
  constexpr int H = FewLane<R>::HALVES, COLS = R * NT;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const FewLane<R> me;
  __shared__ int experts[kMaxExperts];
  __shared__ __align__(8) int16_t slots[kMaxExperts][kTokens];
  const FewTable& table = *static_cast<const FewTable*>(a.table);
  {  // all of the table with one round trip (entries past the last are not used)
    const int e = table.expert[tid % kMaxExperts];
    const uint2 v = reinterpret_cast<const uint2*>(table.slot)[tid];
    if (tid < kMaxExperts) experts[tid] = e;
    reinterpret_cast<uint2*>(slots)[tid] = v;
    static_assert(sizeof(slots) == 512 * 8, "eight bytes per thread");
  }
  const int kb = f8_blocks(a.inter), panels = f8_blocks(a.hidden), n0 = blockIdx.x * COLS;
  const int parts = gridDim.y, part = blockIdx.y, all = table.count * kb;
  const int q0 = all * part / parts, q1 = all * (part + 1) / parts;  // all <= 128 * 256
  const int64_t plane = (int64_t)a.tokens * a.topk * a.inter;
  const __amdgpu_buffer_rsrc_t hr[kHParts] = {make_rsrc(a.h, (uint32_t)(plane * 2)),
                                              make_rsrc(a.h + plane, (uint32_t)(plane * 2)),
                                              make_rsrc(a.h + 2 * plane, (uint32_t)(plane * 2))};
  __syncthreads();
  struct Pair {
    int slot;
    float scale;
    v4i w[NT][H];
    u4 h[kHParts][2 * H];
  } ring[D];
  // Pairs of this wave in turn: expert i of those named, block b. (Loads without
  // branches, which would make them wait for each other: past the last pair the
  // last one read again, which nothing adds.)
  int q = q0 + wave, i = q / kb, b = q - i * kb;
  const int i_step = 8 / kb, b_step = 8 - i_step * kb;
  auto load = [&](Pair& p) {
    const int e = __builtin_amdgcn_readfirstlane(experts[i]);
    const int64_t block = ((int64_t)e * panels + n0 / 128) * kb + b;
    p.slot = slots[i][me.row];
    p.scale = a.down_scales[block];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int h = 0; h < H; ++h)
        p.w[j][h] = few_weights<ONCE>(a.down + block * 16384 + me.at((n0 & 127) + R * j) + 1024 * h);
#pragma unroll
    for (int s = 0; s < 2 * H; ++s) {
      const int k = 128 * b + me.k + 64 * (s / 2) + 8 * (s % 2);
      // tokens that name others: an offset that reads zeros
      const int at = (p.slot * a.inter + k) * 2 | ((p.slot | (a.inter - 1 - k)) & (int)0x80000000u);
#pragma unroll
      for (int part = 0; part < kHParts; ++part)
        p.h[part][s] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(hr[part], at, 0, 0));
    }
    if (q + 8 < q1) {
      q += 8;
      i += i_step;
      b += b_step;
      i += b >= kb;
      b -= b >= kb ? kb : 0;
    }
  };
  // R tokens x R / 4 quads of columns of each fragment, a thread each
  constexpr int ITEMS = R * R / 4;
  const int t = tid % R, quad = tid / R % (R / 4), j = tid / ITEMS, col = n0 + R * j + 4 * quad;
  const bool mine = j < NT && t < a.tokens && col < a.hidden;
  uint2 residual = {0, 0};
  if (a.residual && mine) residual = *reinterpret_cast<const uint2*>(a.residual + (int64_t)t * a.hidden + col);
  v4f acc[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n] = v4f{0, 0, 0, 0};
  if (q < q1) {
#pragma unroll
    for (int d = 0; d < D; ++d) load(ring[d]);
  }
  for (int at = q0 + wave; at < q1; at += 8 * D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (at + 8 * d >= q1) break;
      Pair& p = ring[d];
      const FewScale scale = few_scale(p.scale);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        v4f by[kHParts] = {};  // (one sum would make each MFMA wait for the one before)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          u4 wv[2];
          few_bf16(p.w[n][h], scale.pow2, wv);
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int part = 0; part < kHParts; ++part) by[part] = mfma_bf16(wv[s], p.h[part][2 * h + s], by[part]);
        }
        const v4f sum = by[0] + (by[1] + by[2]);
        // (a token's sum takes nothing of an expert it does not name, NaN weights neither)
        if (p.slot >= 0) {
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[n][t] = __builtin_fmaf(sum[t], scale.factor, acc[n][t]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      load(p);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) sums[wave][n][lane] = acc[n];
  __syncthreads();
  v4f y = {0, 0, 0, 0};
  if (mine) {
#pragma unroll
    for (int w = 0; w < 8; ++w)
#pragma unroll
      for (int s = 0; s < 16 / R; ++s) y += sums[w][j][R * s + t + 16 * (R / 4 * s + quad)];
  }
  if (parts > 1) {
    // The sums go through memory as atomics of device scope, which no cache holds
    // back: a workgroup's are there once its stores have ended (fences of that scope,
    // which write back and drop whole caches, took half of this kernel's time).
    float* const at = static_cast<float*>(a.partial) + ((int64_t)blockIdx.x * parts * (NT * ITEMS) + tid) * 4;
    if (mine) {
#pragma unroll
      for (int s = 0; s < 4; ++s)
        __hip_atomic_store(at + part * (NT * ITEMS * 4) + s, y[s], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // (with the clobber, so that no store is moved behind the wait: neither the waiting
    // builtin nor a barrier of workgroup scope forbids that)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0)
      last = __hip_atomic_fetch_add(&a.arrived[blockIdx.x], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
    __syncthreads();
    if (!last || !mine) return;
    y = v4f{0, 0, 0, 0};
    for (int o = 0; o < parts; ++o) {
#pragma unroll
      for (int s = 0; s < 4; ++s)
        y[s] += __hip_atomic_load(at + o * (NT * ITEMS * 4) + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  if (!mine) return;
  y += v4f{bf16_lo(residual.x), bf16_hi(residual.x), bf16_lo(residual.y), bf16_hi(residual.y)};
  *reinterpret_cast<uint2*>(a.out + (int64_t)t * a.hidden + col) = uint2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
#endif
}

constexpr int kCus = 256, kMostTiles = 32768 / 8, kMostParts = 16;
constexpr size_t kTableBytes = (sizeof(FewTable) + 255) / 256 * 256, kArrivedBytes = kMostTiles * 4;

// The tiles of the output and their parts, as many as fill the CUs (a workgroup each:
// 16 x 2048 x 768, 64 tiles, 83 us in 4 parts, 85 in 8, 101 in 2) but of 70 KB of
// weights at least, for joining them takes 2 us (two tokens of 4 of 64 experts, 512 x
// 512, 32 KB per tile: 10.5 whole, 12.2 in 4 parts; nine of 4 of 128, 256 x 2048, 2 MB
// per tile: 92 whole, 38 in 4 parts, 28 in 16). Up to 16 routes: 8 columns, whose
// workgroups hold all of h's few rows on their way (one token of 8 experts 16.7, on 32
// columns 18.1; two 25.3 both; three 32.3 and 31.8).
//
// once, how weights are loaded, from 64 MB of them on (four tokens 38.2, so 37.5;
// sixteen 87, 82); fewer may still be in the last-level cache from the call before (one
// token 16.6 and 17.4 from memory).
struct FewDown {
  bool small, once;
  int tiles, parts;
};
FewDown few_down(int tokens, int topk, int experts, int hidden, int inter) {
  const bool small = tokens <= 8 && tokens * topk <= 16;
  const int columns = small ? 8 : 32, tiles = (hidden + columns - 1) / columns;
  float others = 1.0f;  // that no token names an expert, evenly chosen
  for (int t = 0; t < tokens; ++t) others *= 1.0f - (float)topk / experts;
  const float named = (1.0f - others) * experts;
  int parts = (int)(named * inter * columns / 70e3f);
  parts = parts < kMostParts ? parts : kMostParts;
  parts = parts < kCus / tiles ? parts : kCus / tiles;
  return {small, named * 3 * hidden * inter >= 64e6f, tiles, parts < 1 ? 1 : parts};
}
// f32 of each part: 16 (or 8) tokens of the tile's columns
size_t few_partial_bytes(const FewDown& d) { return (size_t)d.tiles * d.parts * (d.small ? 8 * 8 : 16 * 32) * 4; }

}  // namespace

size_t moe_few_workspace_bytes(int tokens, int topk, int experts, int hidden, int inter) {
  return kTableBytes + kArrivedBytes + few_partial_bytes(few_down(tokens, topk, experts, hidden, inter)) + (size_t)tokens * topk * inter * 2 * kHParts;
}

namespace {

template <bool ONCE>
hipError_t launch_few(const MoeFewArgs& a, const FewDown& down, hipStream_t stream) {
  const int slots = a.tokens * a.topk, most = slots < a.experts ? slots : a.experts, kb = f8_blocks(a.hidden);
  auto gate_up = [&](auto kernel, int columns) {
    const int units = most * ((a.inter + columns - 1) / columns);
    kernel<<<units < kCus ? units : kCus, 512, 0, stream>>>(a);
  };
  if (kb <= 2)
    gate_up(few_gate_up_kernel<2, 1, ONCE>, 64);
  else if (kb <= 4)
    gate_up(few_gate_up_kernel<4, 1, ONCE>, 32);
  else if (kb <= 8)
    gate_up(few_gate_up_kernel<8, 1, ONCE>, 16);
  else if (kb <= 16)
    gate_up(few_gate_up_kernel<8, 2, ONCE>, 16);
  else if (kb <= 32)
    gate_up(few_gate_up_kernel<8, 4, ONCE>, 16);
  else
    gate_up(few_gate_up_kernel<8, 0, ONCE>, 16);
  if (hipError_t e = hipGetLastError()) return e;
  const dim3 grid(down.tiles, down.parts);
  if (down.small)
    few_down_kernel<8, 1, 2, ONCE><<<grid, 512, 0, stream>>>(a);
  else
    few_down_kernel<16, 2, 1, ONCE><<<grid, 512, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_moe_few(MoeFewArgs a, void* workspace, hipStream_t stream) {
  const FewDown down = few_down(a.tokens, a.topk, a.experts, a.hidden, a.inter);
  char* at = static_cast<char*>(workspace);
  a.table = at;
  a.arrived = reinterpret_cast<int*>(at += kTableBytes);
  a.partial = at += kArrivedBytes;
  a.h = reinterpret_cast<uint16_t*>(at + few_partial_bytes(down));
  a.down_tiles = down.tiles;
  return down.once ? launch_few<true>(a, down, stream) : launch_few<false>(a, down, stream);
}

}  // namespace clef
