// A router's choices listed by expert: offsets [experts + 1] and the route
// ordinals t * topk + r, ascending within each expert (a stable counting sort).
//
// Slots are taken in chunks of THREADS * rounds, a workgroup each; its waves
// hold consecutive parts of the chunk and go through them 64 at a time. The
// lanes that name one expert find each other by a ballot per bit of the id, so
// a slot's rank among its wave's equals is the wave's count so far plus the
// equals below its lane; no atomics, the order is the slots' own. One chunk
// runs as one launch. More take two: the chunks' counts, then every
// workgroup sums the counts of the chunks before its own and of the experts
// before each (at most kMaxChunks chunks, so this stays short) and places its
// slots. Slots whose id names no expert are left out; the places behind the
// last list are filled with -1.
#include "f8.hpp"

namespace clef {

namespace {

constexpr int kSlotThreads = 512, kSlotWaves = kSlotThreads / 64, kMaxChunks = 256, kSlotRounds = 4;

int slot_rounds(int64_t slots) {
  const int64_t r = (slots + (int64_t)kMaxChunks * kSlotThreads - 1) / ((int64_t)kMaxChunks * kSlotThreads);
  return r < kSlotRounds ? kSlotRounds : (int)r;
}

__device__ __forceinline__ int slot_expert(const float* __restrict__ routes, int slot, int total, int topk,
                                           int experts) {
  if (slot >= total) return -1;
  const int t = slot / topk;
  const float id = routes[(int64_t)t * 2 * topk + (slot - t * topk)];
  return id > -1.0f && id < (float)experts ? (int)id : -1;
}

// Adds this wave's slots of the chunk to its counts hist[0 .. experts) and
// calls place(slot, expert, rank among the wave's slots of that expert).
template <class F>
__device__ __forceinline__ void slot_ranks(const float* __restrict__ routes, int total, int topk, int experts, int bits,
                                           int rounds, int* hist, F place) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int first = (blockIdx.x * kSlotWaves + wave) * (64 * rounds);
  for (int r = 0; r < rounds; ++r) {
    const int slot = first + 64 * r + lane;
    const int e = slot_expert(routes, slot, total, topk, experts);
    unsigned long long same = __ballot(e >= 0);
    for (int b = 0; b < bits; ++b) {
      const bool bit = (e >> b) & 1;
      const unsigned long long m = __ballot(bit);
      same &= bit ? m : ~m;
    }
    if (e >= 0) {
      const int below = __popcll(same & ((1ull << lane) - 1ull));
      const int before = hist[e];
      place(slot, e, before + below);
      // one wave's LDS operations run in order: every equal has read the
      // count before the lowest of them raises it
      asm volatile("" ::: "memory");
      if (below == 0) hist[e] = before + __popcll(same);
    }
    asm volatile("" ::: "memory");
  }
}

// counts [chunks][experts]
__global__ __launch_bounds__(kSlotThreads) void slot_count_kernel(const float* __restrict__ routes, int total, int topk,
                                                                  int experts, int bits, int rounds,
                                                                  int32_t* __restrict__ counts) {
  extern __shared__ int hist[];  // [kSlotWaves][experts]
  for (int i = threadIdx.x; i < kSlotWaves * experts; i += kSlotThreads) hist[i] = 0;
  __syncthreads();
  slot_ranks(routes, total, topk, experts, bits, rounds, hist + (threadIdx.x >> 6) * experts, [](int, int, int) {});
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += kSlotThreads) {
    int c = 0;
#pragma unroll
    for (int w = 0; w < kSlotWaves; ++w) c += hist[w * experts + e];
    counts[(int64_t)blockIdx.x * experts + e] = c;
  }
}

// Places the chunk's slots. Ranks are kept in LDS words between the two
// passes over the slots (they are found again: the ids are read twice).
__global__ __launch_bounds__(kSlotThreads) void slot_place_kernel(const float* __restrict__ routes, int total, int topk,
                                                                  int experts, int bits, int rounds,
                                                                  const int32_t* __restrict__ counts,
                                                                  int32_t* __restrict__ offsets,
                                                                  int32_t* __restrict__ slots) {
  extern __shared__ int lds[];
  int* hist = lds;                            // [kSlotWaves][experts]: counts, then the place of the wave's next slot
  int* sum = hist + kSlotWaves * experts;     // [experts] all chunks, then the list's begin
  int* mine = sum + experts;                  // [experts] chunks before this one
  int* wave_sum = mine + experts;             // [kSlotWaves]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < kSlotWaves * experts; i += kSlotThreads) hist[i] = 0;
  for (int e = tid; e < experts; e += kSlotThreads) sum[e] = mine[e] = 0;
  __syncthreads();
  slot_ranks(routes, total, topk, experts, bits, rounds, hist + wave * experts, [](int, int, int) {});
  if (counts != nullptr) {
    // parts of the chunks' counts per thread, summed by integer atomics
    const int parts = experts >= kSlotThreads ? 1 : kSlotThreads / experts;
    for (int i = tid; i < parts * experts; i += kSlotThreads) {
      const int e = i % experts, part = i / experts;
      int all = 0, before = 0;
      for (int c = part; c < (int)gridDim.x; c += parts) {
        const int v = counts[(int64_t)c * experts + e];
        all += v;
        before += c < (int)blockIdx.x ? v : 0;
      }
      atomicAdd(&sum[e], all);
      atomicAdd(&mine[e], before);
    }
  }
  __syncthreads();
  if (counts == nullptr)
    for (int e = tid; e < experts; e += kSlotThreads) {
      int c = 0;
#pragma unroll
      for (int w = 0; w < kSlotWaves; ++w) c += hist[w * experts + e];
      sum[e] = c;
    }
  __syncthreads();
  // exclusive scan of sum over the experts, kSlotThreads at a time
  int carry = 0;
  for (int c = 0; c < experts; c += kSlotThreads) {
    const int e = c + tid;
    const int v = e < experts ? sum[e] : 0;
    int incl = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(incl, off, 64);
      if (lane >= off) incl += o;
    }
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    int base = carry, all = 0;
#pragma unroll
    for (int w = 0; w < kSlotWaves; ++w) {
      if (w < wave) base += wave_sum[w];
      all += wave_sum[w];
    }
    if (e < experts) sum[e] = base + incl - v;
    carry += all;
    __syncthreads();
  }
  // places of each wave's first slot per expert
  for (int e = tid; e < experts; e += kSlotThreads) {
    int at = sum[e] + mine[e];
#pragma unroll
    for (int w = 0; w < kSlotWaves; ++w) {
      const int c = hist[w * experts + e];
      hist[w * experts + e] = at;
      at += c;
    }
    if (blockIdx.x == 0) offsets[e] = sum[e];
  }
  if (blockIdx.x == 0 && tid == 0) offsets[experts] = carry;
  __syncthreads();
  slot_ranks(routes, total, topk, experts, bits, rounds, hist + wave * experts,
             [&](int slot, int, int at) { slots[at] = slot; });
  for (int i = carry + (int)blockIdx.x * kSlotThreads + tid; i < total; i += (int)gridDim.x * kSlotThreads) slots[i] = -1;
}

}  // namespace

size_t group_slots_workspace_bytes(int64_t slots, int experts) {
  const int64_t chunk = (int64_t)kSlotThreads * slot_rounds(slots);
  const int64_t chunks = (slots + chunk - 1) / chunk;
  return chunks <= 1 ? 0 : (size_t)(chunks * experts * 4);
}

hipError_t launch_group_slots(const float* routes, int64_t tokens, int topk, int experts, int32_t* offsets,
                              int32_t* slots, void* workspace, hipStream_t stream) {
  const int total = (int)(tokens * topk), rounds = slot_rounds(total);
  const int chunk = kSlotThreads * rounds, chunks = total > 0 ? (total + chunk - 1) / chunk : 1;
  int bits = 0;
  while ((1 << bits) < experts) ++bits;
  int32_t* counts = chunks > 1 ? static_cast<int32_t*>(workspace) : nullptr;
  if (counts != nullptr) {
    slot_count_kernel<<<chunks, kSlotThreads, kSlotWaves * experts * 4, stream>>>(routes, total, topk, experts, bits,
                                                                                 rounds, counts);
    if (hipError_t e = hipGetLastError()) return e;
  }
  const int lds = (kSlotWaves * experts + 2 * experts + kSlotWaves) * 4;
  slot_place_kernel<<<chunks, kSlotThreads, lds, stream>>>(routes, total, topk, experts, bits, rounds, counts, offsets,
                                                           slots);
  return hipGetLastError();
}

}  // namespace clef
