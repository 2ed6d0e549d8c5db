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
// power of two, whose remaining factor enters the f32 sums behind each block of 128 k. The router's probability goes into h (in f32, in front of
// its rounding), so that the down products of all experts add up in one
// accumulator. h is held as two bf16 that together keep 16 bits of it: the second
// product costs nothing beside the weights' bytes, and the output is rounded once.
#include "f8.hpp"
#include "linear.hpp"
#include "moe_few_f8.hpp"
#include "route.hpp"

namespace clef {

namespace {

constexpr int kTokens = kMoeFewTokens, kMaxExperts = kMoeFewExperts;

// What the second launch takes from the first: the experts named, ascending, and for
// each the rows of h of its tokens (-1: the token names others).
struct FewTable {
  int count;
  int expert[kMaxExperts];
  int16_t slot[kMaxExperts][kTokens];
};

// Routing of all tokens by one workgroup of 512 threads, in LDS.
struct FewRoutes {
  float v[kTokens][kMaxExperts];         // the logits; -inf: takes no part
  float p[kTokens][kMaxExperts];         // by rank
  uint8_t rank[kTokens][kMaxExperts];    // by expert
  uint32_t tokens[kMaxExperts];          // by expert: the tokens that name it
  unsigned long long named[2];
};

__device__ __forceinline__ float few_logit(const MoeFewArgs& a, int i) {
  const float v = a.logits_f32 ? static_cast<const float*>(a.logits)[i]
                               : bf16_to_f32(static_cast<const uint16_t*>(a.logits)[i]);
  return v != v ? -__builtin_huge_valf() : v;
}

// An expert's rank is the number of logits in front of its own (larger, or equal
// at a lower id). Logits of -inf and NaN take no part, nor does a probability that
// is zero: a token may name fewer than topk experts, or none.
__device__ __forceinline__ void few_route(const MoeFewArgs& a, FewRoutes& r) {
  const int tid = threadIdx.x, experts = a.experts, pairs = a.tokens * experts;
  for (int i = tid; i < pairs; i += 512) r.v[i / experts][i % experts] = few_logit(a, i);
  if (tid < kMaxExperts) r.tokens[tid] = 0;
  __syncthreads();
  // by rank, into p: the logits; ranks of those in front
  for (int i = tid; i < pairs; i += 512) {
    const int t = i / experts, e = i % experts;
    const float v = r.v[t][e];
    int before = 0;
    for (int o = 0; o < experts; ++o) before += r.v[t][o] > v || (r.v[t][o] == v && o < e);
    r.rank[t][e] = (uint8_t)before;
    if (before < a.topk) r.p[t][before] = v;
  }
  __syncthreads();
  float mine[4];  // at most 16 x 128 ranks over 512 threads
  int n = 0;
  for (int i = tid; i < a.tokens * a.topk; i += 512, ++n) {
    const int t = i / a.topk, k = i % a.topk;
    const float best = r.p[t][0];
    float sum = 0.0f;
    for (int o = 0; o < a.topk; ++o) sum += r.p[t][o] == best ? 1.0f : cephes_expf(r.p[t][o] - best);
    const float v = r.p[t][k];
    mine[n & 3] = v == -__builtin_huge_valf() ? 0.0f : (v == best ? 1.0f : cephes_expf(v - best)) / sum;
  }
  __syncthreads();
  n = 0;
  for (int i = tid; i < a.tokens * a.topk; i += 512, ++n) r.p[i / a.topk][i % a.topk] = mine[n & 3];
  __syncthreads();
  for (int i = tid; i < pairs; i += 512) {
    const int t = i / experts, e = i % experts, k = r.rank[t][e];
    if (k < a.topk && r.p[t][k] > 0.0f) atomicOr(&r.tokens[e], 1u << t);
  }
  __syncthreads();
  if (tid < 128) {
    const unsigned long long mask = __ballot(r.tokens[tid] != 0);
    if ((tid & 63) == 0) r.named[tid >> 6] = mask;
  }
  __syncthreads();
}

// The i-th expert named, i < their number.
__device__ __forceinline__ int few_expert(const FewRoutes& r, int i) {
  unsigned long long mask = r.named[0];
  int base = 0;
  const int low = __popcll(mask);
  if (i >= low) {
    i -= low;
    mask = r.named[1];
    base = 64;
  }
  for (; i > 0; --i) mask &= mask - 1;
  return base + __builtin_ctzll(mask);
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

// One unit is the 16 columns `tile` of h of the i-th expert named: eight waves
// split the blocks of k, their sums meet in LDS and are added in wave order.
__global__ __launch_bounds__(512) void few_gate_up_kernel(const MoeFewArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ FewRoutes routes;
  __shared__ v4f sums[8][2][64];
  few_route(a, routes);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, g = lane >> 4;
  const int count = __popcll(routes.named[0]) + __popcll(routes.named[1]);
  FewTable& table = *static_cast<FewTable*>(a.table);
  if (blockIdx.x == 0) {
    if (tid == 0) table.count = count;
    for (int i = tid; i < count * kTokens; i += 512) {
      const int t = i % kTokens, e = few_expert(routes, i / kTokens);
      if (t == 0) table.expert[i / kTokens] = e;
      table.slot[i / kTokens][t] = routes.tokens[e] >> t & 1 ? (int16_t)(t * a.topk + routes.rank[t][e]) : (int16_t)-1;
    }
  }
  const int kb = f8_blocks(a.hidden), tiles = (a.inter + 15) / 16, panels = f8_blocks(a.inter);
  const int row = lr < a.tokens ? lr : a.tokens - 1;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(a.x, (uint32_t)(((a.tokens - 1) * a.x_stride + a.hidden) * 2));
  for (int u = blockIdx.x; u < count * tiles; u += gridDim.x) {
    const int e = __builtin_amdgcn_readfirstlane(few_expert(routes, u / tiles)), n0 = u % tiles * 16;
    const int64_t panel = ((int64_t)e * panels + n0 / 128) * kb;
    v4f acc[2] = {v4f{0, 0, 0, 0}, v4f{0, 0, 0, 0}};
    for (int b = wave; b < kb; b += 8) {
      u4 xv[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int k = 128 * b + 64 * (s / 2) + 16 * g + 8 * (s % 2);
        xv[s] = k < a.hidden ? __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(
                                   xr, (int)(row * a.x_stride + k) * 2, 0, 0))
                             : u4{0, 0, 0, 0};
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const FewScale sw = few_scale((m ? a.up_scales : a.gate_scales)[panel + b]);
        const uint8_t* at = (m ? a.up : a.gate) + (panel + b) * 16384 + (n0 & 127) * 128 + lane * 16;
        v4f part = {0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u4 wv[2];
          few_bf16(*reinterpret_cast<const v4i*>(at + 1024 * h), sw.pow2, wv);
#pragma unroll
          for (int s = 0; s < 2; ++s) part = mfma_bf16(wv[s], xv[2 * h + s], part);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[m][t] = __builtin_fmaf(part[t], sw.factor, acc[m][t]);
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) sums[wave][m][lane] = acc[m];
    __syncthreads();
    if (tid < 64) {
      const int col = n0 + 4 * g;
      if (lr < a.tokens && (routes.tokens[e] >> lr & 1) && col < a.inter) {
        v4f gate = {0, 0, 0, 0}, up = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          gate += sums[w][0][lane];
          up += sums[w][1][lane];
        }
        const int k = routes.rank[lr][e];
        const float p = routes.p[lr][k];
        uint16_t* at = a.h + (int64_t)(lr * a.topk + k) * a.inter + col;
        const int64_t low = (int64_t)a.tokens * a.topk * a.inter;
        uint2 hi, lo;
        float y[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) y[t] = gate[t] * sigmoid_f32(gate[t]) * up[t] * p;
        hi.x = pack_bf16x2(y[0], y[1]);
        hi.y = pack_bf16x2(y[2], y[3]);
        // (nothing is left of what became infinite)
        auto left = [](float v, float r) { return __builtin_isinf(r) ? 0.0f : v - r; };
        lo.x = pack_bf16x2(left(y[0], bf16_lo(hi.x)), left(y[1], bf16_hi(hi.x)));
        lo.y = pack_bf16x2(left(y[2], bf16_lo(hi.y)), left(y[3], bf16_hi(hi.y)));
        *reinterpret_cast<uint2*>(at) = hi;
        *reinterpret_cast<uint2*>(at + low) = lo;
      }
    }
    __syncthreads();
  }
#endif
}

// 16 columns of the output: the waves split the pairs (expert named, block of k).
__global__ __launch_bounds__(512) void few_down_kernel(const MoeFewArgs a) {
#if defined(__HIP_DEVICE_COMPILE__)
  __shared__ v4f sums[8][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, g = lane >> 4;
  const FewTable& table = *static_cast<const FewTable*>(a.table);
  const int kb = f8_blocks(a.inter), panels = f8_blocks(a.hidden), pairs = table.count * kb;
  const int n0 = blockIdx.x * 16;
  const int64_t low = (int64_t)a.tokens * a.topk * a.inter;
  v4f acc = {0, 0, 0, 0};
  for (int q = wave; q < pairs; q += 8) {
    const int i = q / kb, b = q % kb, e = table.expert[i], slot = table.slot[i][lr];
    const int64_t block = ((int64_t)e * panels + n0 / 128) * kb + b;
    const FewScale sw = few_scale(a.down_scales[block]);
    const uint8_t* at = a.down + block * 16384 + (n0 & 127) * 128 + lane * 16;
    v4f part = {0, 0, 0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u4 wv[2];
      few_bf16(*reinterpret_cast<const v4i*>(at + 1024 * h), sw.pow2, wv);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int k = 128 * b + 64 * h + 16 * g + 8 * s;
        u4 hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
        if (slot >= 0 && k < a.inter) {
          const uint16_t* from = a.h + (int64_t)slot * a.inter + k;
          hi = *reinterpret_cast<const u4*>(from);
          lo = *reinterpret_cast<const u4*>(from + low);
        }
        part = mfma_bf16(wv[s], hi, part);
        part = mfma_bf16(wv[s], lo, part);
      }
    }
    // (a token's sum takes nothing of an expert it does not name, NaN weights neither)
    if (slot >= 0) {
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[t] = __builtin_fmaf(part[t], sw.factor, acc[t]);
    }
  }
  sums[wave][lane] = acc;
  __syncthreads();
  const int col = n0 + 4 * g;
  if (tid >= 64 || lr >= a.tokens || col >= a.hidden) return;
  v4f y = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < 8; ++w) y += sums[w][lane];
  if (a.residual) {
    const uint2 r = *reinterpret_cast<const uint2*>(a.residual + (int64_t)lr * a.hidden + col);
    y += v4f{bf16_lo(r.x), bf16_hi(r.x), bf16_lo(r.y), bf16_hi(r.y)};
  }
  *reinterpret_cast<uint2*>(a.out + (int64_t)lr * a.hidden + col) = uint2{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
#endif
}

constexpr size_t kTableBytes = (sizeof(FewTable) + 255) / 256 * 256;

}  // namespace

size_t moe_few_workspace_bytes(int tokens, int topk, int inter) {
  return kTableBytes + (size_t)tokens * topk * inter * 4;
}

hipError_t launch_moe_few(MoeFewArgs a, void* workspace, hipStream_t stream) {
  a.table = workspace;
  a.h = reinterpret_cast<uint16_t*>(static_cast<char*>(workspace) + kTableBytes);
  const int slots = a.tokens * a.topk, most = slots < a.experts ? slots : a.experts;
  const int units = most * ((a.inter + 15) / 16);
  few_gate_up_kernel<<<units < 512 ? units : 512, 512, 0, stream>>>(a);
  if (hipError_t e = hipGetLastError()) return e;
  few_down_kernel<<<(a.hidden + 15) / 16, 512, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace clef
