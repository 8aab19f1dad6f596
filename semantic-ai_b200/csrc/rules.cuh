// rules.cuh — the rules between logits and token (host/device shared); see svl_logits_rules.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/svl_cuda.h"

namespace svl {

constexpr int kRulesMaxEntries = 65535;  // history or bias entries of a row: 16 bits each

struct RulesParams {
  const void* logits;  // [rows][logits_stride], f32 or bf16
  int64_t logits_stride;
  void* out;           // or null
  int64_t out_stride;
  int32_t* tokens;     // [rows] or null
  int64_t rows;
  int vocab;
  int bf16;
  svl_logits_rules rules;
};
void launch_rules(const RulesParams& p, cudaStream_t s);

}  // namespace svl
