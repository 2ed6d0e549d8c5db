// A MoE layer of few tokens on block-scaled FP8 experts: arguments and launcher.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace clef {

constexpr int kMoeFewTokens = 16, kMoeFewExperts = 128;

struct MoeFewArgs {
  const uint16_t* x;  // bf16 [tokens][hidden], rows x_stride apart
  int64_t x_stride;
  const void* logits;  // bf16 or f32 [tokens][experts]
  bool logits_f32;
  int tokens, hidden, inter, experts, topk;
  const uint8_t *gate, *up, *down;  // tiled codes (f8.hpp)
  const float *gate_scales, *up_scales, *down_scales;
  const uint16_t* residual;  // bf16 [tokens][hidden] or NULL
  uint16_t* out;
  // in the workspace:
  void* table;
  int down_tiles;  // of the output, with several parts
  int* arrived;    // per tile, the parts done
  void* partial;   // their sums
  uint16_t* h;     // three times bf16 [tokens * topk][inter], their sum is h
};

size_t moe_few_workspace_bytes(int tokens, int topk, int experts, int hidden, int inter);
hipError_t launch_moe_few(MoeFewArgs a, void* workspace, hipStream_t stream);

}  // namespace clef
