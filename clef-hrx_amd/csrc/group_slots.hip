// A router's choices listed by expert: offsets [experts + 1] and the route
// ordinals t * topk + r, ascending within each expert (a stable counting sort).
//
// Slots are taken in chunks, a workgroup each; its waves hold consecutive
// parts of the chunk and go through them 64 at a time, four loads ahead. The
// lanes that name one expert find each other by a ballot per bit of the id, so
// a slot's rank among its wave's equals is the wave's count so far plus the
// equals below its lane; no global atomics, the order is the slots' own. One
// chunk (2048 slots) runs as one launch. More take two: the chunks' counts,
// then every workgroup sums the counts of all chunks and of those before its
// own (at most kMaxChunks, read as 16-byte pieces that are all in flight
// together) and places its slots. Slots whose id names no expert are left out;
// the places behind the last list are filled with -1.
//
// Bound by latency: 1880 slots take 4.8 us, 7.5 when every 64 ids were loaded and
// ranked in turn, twice. 524288 slots of 128 experts take 4.7 and 9.6 us, 29 with
// the counts read one by one: each of the second launch's 256 workgroups ranks its
// slots again and reads the counts of all chunks (131 KB, 34 MB together, from L2).
#include "f8.hpp"

namespace clef {

namespace {

constexpr int kSlotThreads = 512, kSlotWaves = kSlotThreads / 64, kMaxChunks = 256, kAhead = 4;

// Batches of kAhead rounds of 64 slots per wave.
int slot_batches(int64_t slots) {
  const int64_t most = (int64_t)kMaxChunks * kSlotThreads * kAhead;
  return slots <= most ? 1 : (int)((slots + most - 1) / most);
}

// The experts of slots first + 64 r + lane, r < kAhead (-1 for none).
__device__ __forceinline__ void slot_experts(const float* __restrict__ routes, int first, int total, int topk,
                                             int experts, int (&e)[kAhead]) {
  float id[kAhead];
#pragma unroll
  for (int r = 0; r < kAhead; ++r) {
    const int slot = first + 64 * r + (int)(threadIdx.x & 63);
    const int t = slot / topk;
    id[r] = slot < total ? routes[(int64_t)t * 2 * topk + (slot - t * topk)] : -1.0f;
  }
#pragma unroll
  for (int r = 0; r < kAhead; ++r) e[r] = id[r] > -1.0f && id[r] < (float)experts ? (int)id[r] : -1;
}

// Ranks of these slots among the wave's of the same expert, counted from and
// into hist[0 .. experts).
__device__ __forceinline__ void slot_ranks(const int (&e)[kAhead], int bits, int* hist, int (&rank)[kAhead]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int r = 0; r < kAhead; ++r) {
    unsigned long long same = __ballot(e[r] >= 0);
    for (int b = 0; b < bits; ++b) {
      const bool bit = (e[r] >> b) & 1;
      const unsigned long long m = __ballot(bit);
      same &= bit ? m : ~m;
    }
    rank[r] = 0;
    if (e[r] >= 0) {
      const int below = __popcll(same & ((1ull << lane) - 1ull));
      const int before = hist[e[r]];
      rank[r] = before + below;
      // one wave's LDS operations run in order: every equal has read the
      // count before the lowest of them raises it
      asm volatile("" ::: "memory");
      if (below == 0) hist[e[r]] = before + __popcll(same);
    }
    asm volatile("" ::: "memory");
  }
}

// counts [chunks][pitch]
__global__ __launch_bounds__(kSlotThreads) void slot_count_kernel(const float* __restrict__ routes, int total, int topk,
                                                                  int experts, int pitch, int bits, int batches,
                                                                  int32_t* __restrict__ counts) {
  extern __shared__ int hist[];  // [kSlotWaves][experts]
  const int wave = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < kSlotWaves * experts; i += kSlotThreads) hist[i] = 0;
  __syncthreads();
  const int first = (blockIdx.x * kSlotWaves + wave) * (64 * kAhead * batches);
  for (int b = 0; b < batches; ++b) {
    int e[kAhead], rank[kAhead];
    slot_experts(routes, first + b * 64 * kAhead, total, topk, experts, e);
    slot_ranks(e, bits, hist + wave * experts, rank);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < pitch; e += kSlotThreads) {
    int c = 0;
    if (e < experts) {
#pragma unroll
      for (int w = 0; w < kSlotWaves; ++w) c += hist[w * experts + e];
    }
    counts[(int64_t)blockIdx.x * pitch + e] = c;
  }
}

// Places the chunk's slots. Of a chunk of one batch the experts and ranks stay
// in registers; longer ones are gone through twice.
__global__ __launch_bounds__(kSlotThreads) void slot_place_kernel(const float* __restrict__ routes, int total, int topk,
                                                                  int experts, int pitch, int bits, int batches,
                                                                  const int32_t* __restrict__ counts,
                                                                  int32_t* __restrict__ offsets,
                                                                  int32_t* __restrict__ slots) {
  extern __shared__ int lds[];
  int* hist = lds;                         // [kSlotWaves][experts]: counts, then the place of the wave's first slot
  int* sum = hist + kSlotWaves * experts;  // [pitch] all chunks, then the list's begin
  int* mine = sum + pitch;                 // [pitch] chunks before this one
  int* wave_sum = mine + pitch;            // [kSlotWaves]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int first = (blockIdx.x * kSlotWaves + wave) * (64 * kAhead * batches);
  int e[kAhead], rank[kAhead];
  slot_experts(routes, first, total, topk, experts, e);
  for (int i = tid; i < kSlotWaves * experts; i += kSlotThreads) hist[i] = 0;
  for (int i = tid; i < 2 * pitch; i += kSlotThreads) sum[i] = 0;
  __syncthreads();
  slot_ranks(e, bits, hist + wave * experts, rank);
  for (int b = 1; b < batches; ++b) {
    slot_experts(routes, first + b * 64 * kAhead, total, topk, experts, e);
    slot_ranks(e, bits, hist + wave * experts, rank);
  }
  if (counts != nullptr) {
    // thread: four experts, every parts-th chunk; the parts meet by LDS integer atomics
    const int quads = pitch / 4, parts = kSlotThreads / quads;  // pitch <= 1024: at least 2
    const int q = tid % quads, part = tid / quads, chunks = gridDim.x;
    if (part < parts) {
      int all[4] = {0, 0, 0, 0}, before[4] = {0, 0, 0, 0};
      const int4* at = reinterpret_cast<const int4*>(counts) + q;
#pragma unroll 16
      for (int c = part; c < chunks; c += parts) {
        const int4 v = at[(int64_t)c * quads];
        const int keep = c < (int)blockIdx.x ? -1 : 0;
        all[0] += v.x, all[1] += v.y, all[2] += v.z, all[3] += v.w;
        before[0] += v.x & keep, before[1] += v.y & keep, before[2] += v.z & keep, before[3] += v.w & keep;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        atomicAdd(&sum[4 * q + i], all[i]);
        atomicAdd(&mine[4 * q + i], before[i]);
      }
    }
  }
  __syncthreads();
  // exclusive scan of the experts' totals, kSlotThreads at a time, and the
  // places of each wave's first slots
  int carry = 0;
  for (int c = 0; c < experts; c += kSlotThreads) {
    const int x = c + tid;
    int per[kSlotWaves], v = 0, own = 0;
    if (x < experts) {
#pragma unroll
      for (int w = 0; w < kSlotWaves; ++w) {
        per[w] = hist[w * experts + x];
        own += per[w];
      }
      v = counts != nullptr ? sum[x] : own;
    }
    const int incl = wave_scan(v);
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    int base = carry, all = 0;
#pragma unroll
    for (int w = 0; w < kSlotWaves; ++w) {
      if (w < wave) base += wave_sum[w];
      all += wave_sum[w];
    }
    if (x < experts) {
      const int begin = base + incl - v;
      if (blockIdx.x == 0) offsets[x] = begin;
      int at = begin + mine[x];
#pragma unroll
      for (int w = 0; w < kSlotWaves; ++w) {
        hist[w * experts + x] = at;
        at += per[w];
      }
    }
    carry += all;
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) offsets[experts] = carry;
  if (batches == 1) {
#pragma unroll
    for (int r = 0; r < kAhead; ++r)
      if (e[r] >= 0) slots[hist[wave * experts + e[r]] + rank[r]] = first + 64 * r + lane;
  } else {
    for (int b = 0; b < batches; ++b) {
      const int f = first + b * 64 * kAhead;
      slot_experts(routes, f, total, topk, experts, e);
      slot_ranks(e, bits, hist + wave * experts, rank);
#pragma unroll
      for (int r = 0; r < kAhead; ++r)
        if (e[r] >= 0) slots[rank[r]] = f + 64 * r + lane;
    }
  }
  for (int i = carry + (int)blockIdx.x * kSlotThreads + tid; i < total; i += (int)gridDim.x * kSlotThreads) slots[i] = -1;
}

int slot_pitch(int experts) { return (experts + 3) / 4 * 4; }

}  // namespace

size_t group_slots_workspace_bytes(int64_t slots, int experts) {
  const int64_t chunk = (int64_t)kSlotThreads * kAhead * slot_batches(slots);
  const int64_t chunks = (slots + chunk - 1) / chunk;
  return chunks <= 1 ? 0 : (size_t)(chunks * slot_pitch(experts) * 4);
}

hipError_t launch_group_slots(const float* routes, int64_t tokens, int topk, int experts, int32_t* offsets,
                              int32_t* slots, void* workspace, hipStream_t stream) {
  const int total = (int)(tokens * topk), batches = slot_batches(total), pitch = slot_pitch(experts);
  const int chunk = kSlotThreads * kAhead * batches, chunks = total > 0 ? (total + chunk - 1) / chunk : 1;
  int bits = 0;
  while ((1 << bits) < experts) ++bits;
  int32_t* counts = chunks > 1 ? static_cast<int32_t*>(workspace) : nullptr;
  if (counts != nullptr) {
    slot_count_kernel<<<chunks, kSlotThreads, kSlotWaves * experts * 4, stream>>>(routes, total, topk, experts, pitch,
                                                                                 bits, batches, counts);
    if (hipError_t e = hipGetLastError()) return e;
  }
  const int lds = (kSlotWaves * experts + 2 * pitch + kSlotWaves) * 4;
  slot_place_kernel<<<chunks, kSlotThreads, lds, stream>>>(routes, total, topk, experts, pitch, bits, batches, counts,
                                                           offsets, slots);
  return hipGetLastError();
}

}  // namespace clef
