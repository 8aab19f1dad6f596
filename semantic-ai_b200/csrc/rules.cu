// rules.cu — the rules between logits and token: penalties for repeated tokens, biases, grammar
// masks, and the greedy pick.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "entry.h"
#include "rules.cuh"

namespace svl {
namespace {

__device__ __forceinline__ float load_logit(const float* p) { return *p; }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_logit(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// An order-preserving key of a value above -infinity (0: none), then the lowest index: the
// larger key wins.
__device__ __forceinline__ uint64_t pick_key(float v, int i) {
  if (!(v > -INFINITY)) return 0;
  uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);  // -0 and 0 are equal
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)~i;
}
__device__ __forceinline__ uint64_t max_key(uint64_t a, uint64_t b) { return a > b ? a : b; }

constexpr int kThreads = 256;
constexpr int kChunk = 4096;  // tokens whose counts are held at once

// One CTA per row. For a chunk of the vocabulary, `word` holds each token's count in the history
// (low 16 bits) and its first entry in the sparse biases (65,535 minus its index, high 16).
template <class T>
__global__ void __launch_bounds__(kThreads) rules_kernel(const RulesParams p) {
  __shared__ uint32_t word[kChunk];
  __shared__ uint64_t best_sm[kThreads / 32];
  __shared__ int twice;
  const svl_logits_rules& R = p.rules;
  const int t = threadIdx.x;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* in = static_cast<const T*>(p.logits) + r * p.logits_stride;
    T* out = p.out ? static_cast<T*>(p.out) + r * p.out_stride : nullptr;
    const int said = R.d_history ? max(0, min(R.d_lengths[r], R.history_cap)) : 0;
    const int32_t* hist = R.d_history + r * R.history_stride;
    const int32_t* ids = R.d_bias_ids + r * R.bias_stride;
    const float* vals = R.d_bias_values + r * R.bias_stride;
    const int listed = R.d_bias_ids ? R.bias_cap : 0;
    const float rep = R.d_repetition ? R.d_repetition[r] : 1.f;
    const float freq = R.d_frequency ? R.d_frequency[r] : 0.f, pres = R.d_presence ? R.d_presence[r] : 0.f;
    const uint32_t* mask = nullptr;
    if (R.d_masks) {
      const int64_t m = R.d_mask_rows ? R.d_mask_rows[r] : r;
      if (m >= 0 && m < R.n_masks) mask = R.d_masks + m * R.mask_stride;
    }
    uint64_t best = 0;
    for (int v0 = 0; v0 < p.vocab; v0 += kChunk) {
      const int n = min(kChunk, p.vocab - v0);
      __syncthreads();
      for (int i = t; i < n; i += kThreads) word[i] = 0;
      if (t == 0) twice = 0;
      __syncthreads();
      for (int i = t; i < listed; i += kThreads)
        if (ids[i] >= v0 && ids[i] < v0 + n) atomicMax(&word[ids[i] - v0], (uint32_t)(65535 - i) << 16);
      __syncthreads();
      for (int i = t; i < listed; i += kThreads)
        if (ids[i] >= v0 && ids[i] < v0 + n && (word[ids[i] - v0] >> 16) != 65535 - i) twice = 1;
      __syncthreads();
      for (int i = t; i < said; i += kThreads)
        if (hist[i] >= v0 && hist[i] < v0 + n && hist[i] >= R.first_penalised) atomicAdd(&word[hist[i] - v0], 1u);
      __syncthreads();
      for (int i = t; i < n; i += kThreads) {
        const int v = v0 + i;
        float l = load_logit(in + v);
        const uint32_t w = word[i];
        if (w & 65535) {
          l = l > 0.f ? __fdiv_rn(l, rep) : l * rep;
          l = l - (freq * (float)(w & 65535) + pres);
        }
        if (R.d_dense_bias) l = l + R.d_dense_bias[v];
        if (w >> 16) {
          const int first = 65535 - (int)(w >> 16);
          l = l + vals[first];
          if (twice)
            for (int j = first + 1; j < listed; j++)
              if (ids[j] == v) l = l + vals[j];
        }
        if (mask && !((mask[v >> 5] >> (v & 31)) & 1)) l = -INFINITY;
        if (out) store_logit(out + v, l);
        best = max_key(best, pick_key(l, v));
      }
    }
    for (int o = 16; o; o >>= 1) best = max_key(best, __shfl_xor_sync(0xffffffffu, best, o));
    if ((t & 31) == 0) best_sm[t >> 5] = best;
    __syncthreads();
    if (t == 0) {
      for (int w = 1; w < kThreads / 32; w++) best = max_key(best, best_sm[w]);
      const int token = best ? (int)~(uint32_t)best : -1;
      if (p.tokens) p.tokens[r] = token;
      if (R.append && R.d_history && token >= 0 && token >= R.first_penalised) {
        const int len = max(0, R.d_lengths[r]);
        R.d_history[r * R.history_stride + len % R.history_cap] = token;
        // A count that would overflow starts again at the same place of a full ring.
        R.d_lengths[r] = len < INT32_MAX ? len + 1 : R.history_cap + (len % R.history_cap) + 1;
      }
    }
    __syncthreads();
  }
}

}  // namespace

void launch_rules(const RulesParams& p, cudaStream_t s) {
  const int grid = (int)std::min<int64_t>(p.rows, 148 * 64);
  if (p.bf16)
    rules_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(p);
  else
    rules_kernel<float><<<grid, kThreads, 0, s>>>(p);
  check_cuda(cudaGetLastError(), "rules launch");
}

}  // namespace svl

extern "C" SVL_API svl_status svl_logits_rules_device(int32_t device, int64_t rows, int32_t vocab, int32_t dtype,
                                                      const void* d_logits, int64_t logits_stride,
                                                      const svl_logits_rules* rules, void* d_out, int64_t out_stride,
                                                      int32_t* d_tokens, void* cuda_stream) {
  using svl::require;
  return svl::entry([&] {
    require(rows >= 0, "negative row count");
    require(vocab >= 1, "vocab must be positive");
    require(dtype == SVL_DT_F32 || dtype == SVL_DT_BF16, "dtype must be f32 or bf16");
    svl::RulesParams p{};
    if (rules) p.rules = *rules;
    const svl_logits_rules& R = p.rules;
    require(!R.d_history == !R.d_lengths, "d_history and d_lengths go together");
    require(!R.d_history || (R.history_cap >= 1 && R.history_cap <= svl::kRulesMaxEntries),
            "history_cap must be 1..65535");
    require(!R.d_history || R.history_stride >= R.history_cap, "history_stride is below history_cap");
    require(!R.append || R.d_history, "append needs a history");
    require(!R.d_bias_ids == !R.d_bias_values, "d_bias_ids and d_bias_values go together");
    require(!R.d_bias_ids || (R.bias_cap >= 0 && R.bias_cap <= svl::kRulesMaxEntries), "bias_cap must be 0..65535");
    require(!R.d_bias_ids || R.bias_stride >= R.bias_cap, "bias_stride is below bias_cap");
    require(!R.d_masks || (R.n_masks >= 0 && R.mask_stride >= ((int64_t)vocab + 31) / 32),
            "mask_stride is below vocab / 32 words");
    require(!R.d_masks || R.d_mask_rows || R.n_masks >= rows, "fewer masks than rows, and no d_mask_rows");
    if (rows == 0) return;
    require(d_logits && (d_out || d_tokens || R.append), "null argument");
    require(logits_stride >= vocab && (!d_out || out_stride >= vocab), "a row stride is below vocab");
    svl::OnDevice on(device);
    p.rows = rows;
    p.vocab = vocab;
    p.bf16 = dtype == SVL_DT_BF16;
    p.logits = d_logits;
    p.logits_stride = logits_stride;
    p.out = d_out;
    p.out_stride = out_stride;
    p.tokens = d_tokens;
    svl::launch_rules(p, static_cast<cudaStream_t>(cuda_stream));
  });
}
