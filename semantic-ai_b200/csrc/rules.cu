// rules.cu — the rules between logits and token: penalties for repeated tokens, biases, grammar
// masks, and the greedy pick.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "entry.h"
#include "rules.cuh"
#include "sm100.cuh"

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

constexpr int kMaxChunk = 16384;  // tokens whose counts are held at once: 64 KB
constexpr int kAhead = 4;         // 16-byte loads a thread has in flight

// A row is shared by the CTAs of a cluster, each with a contiguous range of the vocabulary. Per
// chunk of the range (one, up to 131,072 tokens in 8 CTAs), `word` holds each token's count in the
// history (low 16 bits) and its first entry in the sparse biases (65,535 minus its index, high
// 16), so lists of any order and any repetition cost one pass of shared-memory atomics, and the
// result does not depend on their timing. The row's first logits are on their way meanwhile.
//
// Positions are counted from the 16-byte boundary at or before the row's start ("lead" elements
// before it), so that every row is read in aligned 16-byte pieces, also where rows of an odd
// vocabulary start anywhere.
template <class T>
__global__ void __launch_bounds__(256, 4) rules_kernel(const RulesParams p, int split, int range, int chunk) {
  constexpr int VE = 16 / sizeof(T);
  extern __shared__ uint32_t word[];
  __shared__ uint64_t best_sm[8], best_of[8];
  __shared__ int twice;
  const svl_logits_rules& R = p.rules;
  const int t = threadIdx.x, threads = blockDim.x;
  const int rank = split > 1 ? (int)cluster_rank() : 0;
  const int64_t r = blockIdx.x / split;
  if (split > 1) cluster_arrive();  // waited for before the ranks' shared memory is written
  pdl_launch();
  pdl_wait();
  const T* in = static_cast<const T*>(p.logits) + r * p.logits_stride;
  T* out = p.out ? static_cast<T*>(p.out) + r * p.out_stride : nullptr;
  const int lead = (int)(reinterpret_cast<uintptr_t>(in) % 16 / sizeof(T));
  const bool wide_out = out && (reinterpret_cast<uintptr_t>(out) - reinterpret_cast<uintptr_t>(in)) % 16 == 0;
  const bool wide_bias = lead == 0 && reinterpret_cast<uintptr_t>(R.d_dense_bias) % 16 == 0;
  const int end = p.vocab + lead;
  const int lo = rank * range, hi = min(lo + range, end);

  // 16 bytes of logits at position u (a multiple of VE), in flight until they are read.
  auto load = [&](int u) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (u >= hi) return v;
    const T* src = in - lead + u;
    if (u >= lead && u + VE <= end) {
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                   : "l"(src)
                   : "memory");
    } else {
      T e[VE];
#pragma unroll
      for (int j = 0; j < VE; j++) e[j] = u + j >= lead && u + j < end ? src[j] : T(0.f);
      v = *reinterpret_cast<uint4*>(e);
    }
    return v;
  };

  const int said = R.d_history ? max(0, min(R.d_lengths[r], R.history_cap)) : 0;
  const int32_t* hist = R.d_history ? R.d_history + r * R.history_stride : nullptr;
  const int listed = R.d_bias_ids ? R.bias_cap : 0;
  const int32_t* ids = listed ? R.d_bias_ids + r * R.bias_stride : nullptr;
  const float* vals = listed ? R.d_bias_values + r * R.bias_stride : nullptr;
  const bool table = said || listed;
  const float rep = R.d_repetition ? R.d_repetition[r] : 1.f;
  const float freq = R.d_frequency ? R.d_frequency[r] : 0.f, pres = R.d_presence ? R.d_presence[r] : 0.f;
  const uint32_t* mask = nullptr;
  if (R.d_masks) {
    const int64_t m = R.d_mask_rows ? R.d_mask_rows[r] : r;
    if (m >= 0 && m < R.n_masks) mask = R.d_masks + m * R.mask_stride;
  }
  uint64_t best = 0;
  for (int c0 = lo; c0 < hi; c0 += chunk) {
    const int c1 = min(c0 + chunk, hi);
    const int step = threads * VE;
    uint4 raw[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++) raw[j] = load(c0 + j * step + t * VE < c1 ? c0 + j * step + t * VE : hi);
    if (table) {
      const int v0 = c0 - lead, v1 = c1 - lead;  // the chunk's tokens (from 0 on)
      const int from = max(v0, 0);
      __syncthreads();
      for (int i = t * 4; i < (c1 - c0 + 31) / 32 * 32; i += threads * 4) *reinterpret_cast<uint4*>(word + i) = make_uint4(0, 0, 0, 0);
      if (t == 0) twice = 0;
      __syncthreads();
      if (listed) {
        for (int i = t; i < listed; i += threads) {
          const int id = ids[i];
          if (id >= from && id < v1) atomicMax(&word[id - v0], (uint32_t)(65535 - i) << 16);
        }
        __syncthreads();
        for (int i = t; i < listed; i += threads) {
          const int id = ids[i];
          if (id >= from && id < v1 && (int)(word[id - v0] >> 16) != 65535 - i) twice = 1;
        }
        __syncthreads();
      }
      for (int i = t; i < said; i += threads) {
        const int id = hist[i];
        if (id >= from && id < v1 && id >= R.first_penalised) atomicAdd(&word[id - v0], 1u);
      }
      __syncthreads();
    }
    for (int u0 = c0 + t * VE; u0 < c1; u0 += kAhead * step) {
      if (u0 >= c0 + kAhead * step) {
#pragma unroll
        for (int j = 0; j < kAhead; j++) raw[j] = load(u0 + j * step < c1 ? u0 + j * step : hi);
      }
#pragma unroll
      for (int j = 0; j < kAhead; j++) {
        const int u = u0 + j * step;
        if (u >= c1) break;
        const int v = u - lead;  // the piece's first token (below 0 before the row)
        T e[VE];
        *reinterpret_cast<uint4*>(e) = raw[j];
        uint32_t allowed = 0xffffffffu;
        if (mask) {
          const int at = max(v, 0) >> 5, sh = max(v, 0) & 31;
          const uint32_t low = mask[at];
          const uint32_t high = sh + VE > 32 && (at + 1) * 32 < p.vocab ? mask[at + 1] : 0u;
          allowed = __funnelshift_r(low, high, sh);
          if (v < 0) allowed <<= -v;
        }
        uint32_t w[VE];
#pragma unroll
        for (int i = 0; i < VE; i++) w[i] = 0;
        if (table) {
#pragma unroll
          for (int i = 0; i < VE; i += 4) *reinterpret_cast<uint4*>(w + i) = *reinterpret_cast<const uint4*>(word + (u - c0) + i);
        }
        float d[VE];
        const bool inside = v >= 0 && v + VE <= p.vocab;
        if (R.d_dense_bias) {
          if (wide_bias && inside) {
#pragma unroll
            for (int i = 0; i < VE; i += 4) *reinterpret_cast<float4*>(d + i) = *reinterpret_cast<const float4*>(R.d_dense_bias + v + i);
          } else {
#pragma unroll
            for (int i = 0; i < VE; i++) d[i] = v + i >= 0 && v + i < p.vocab ? R.d_dense_bias[v + i] : 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < VE; i++) {
          float l = load_logit(e + i);
          if (w[i]) {
            const uint32_t c = w[i] & 65535;
            if (c) {
              l = l > 0.f ? __fdiv_rn(l, rep) : l * rep;
              l = l - (freq * (float)c + pres);
            }
          }
          if (R.d_dense_bias) l = l + d[i];
          if (w[i] >> 16) {
            const int first = 65535 - (int)(w[i] >> 16);
            l = l + vals[first];
            if (twice)
              for (int k = first + 1; k < listed; k++)
                if (ids[k] == v + i) l = l + vals[k];
          }
          if (!((allowed >> i) & 1)) l = -INFINITY;
          store_logit(e + i, l);
          if (inside || (v + i >= 0 && v + i < p.vocab)) best = max_key(best, pick_key(l, v + i));
        }
        if (out) {
          if (wide_out && inside) {
            *reinterpret_cast<uint4*>(out + v) = *reinterpret_cast<uint4*>(e);
          } else {
#pragma unroll
            for (int i = 0; i < VE; i++)
              if (v + i >= 0 && v + i < p.vocab) out[v + i] = e[i];
          }
        }
      }
    }
  }
  for (int o = 16; o; o >>= 1) best = max_key(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((t & 31) == 0) best_sm[t >> 5] = best;
  __syncthreads();
  if (split > 1) cluster_wait();
  if (t == 0) {
    for (int w = 1; w < threads / 32; w++) best = max_key(best, best_sm[w]);
    if (split > 1) dsmem_st64(dsmem_addr(&best_of[rank], 0), best);
  }
  if (split > 1) {
    __syncwarp();
    cluster_sync();  // the ranks' keys are in rank 0, and every rank has read the history
  }
  if (rank == 0 && t == 0) {
    for (int q = 0; q < (split > 1 ? split : 0); q++) best = max_key(best, best_of[q]);
    const int token = best ? (int)~(uint32_t)best : -1;
    if (p.tokens) p.tokens[r] = token;
    if (R.append && token >= 0 && token >= R.first_penalised) {
      const int len = max(0, R.d_lengths[r]);
      R.d_history[r * R.history_stride + len % R.history_cap] = token;
      // A count that would overflow starts again at the same place of a full ring.
      R.d_lengths[r] = len < INT32_MAX ? len + 1 : R.history_cap + (len % R.history_cap) + 1;
    }
  }
}

}  // namespace

// CTAs per row: enough for four per SM, each with 1,024 tokens at least, and the whole range of
// each in one chunk where 8 of them can hold it.
void launch_rules(const RulesParams& p, cudaStream_t s) {
  const int ve = p.bf16 ? 8 : 4;
  const int64_t span = (int64_t)p.vocab + ve - 1;  // with the lead of the worst row
  int split = 1;
  while (split < 8 && (p.rows * split < 4 * 148 || span > (int64_t)split * kMaxChunk) && span >= (int64_t)split * 2 * 1024) split *= 2;
  const int range = (int)((span + split - 1) / split + 31) / 32 * 32;
  const int chunk = std::min(range, kMaxChunk);
  const int threads = std::min(256, std::max(64, (chunk / ve + kAhead - 1) / kAhead + 31) / 32 * 32);
  const size_t smem = p.rules.d_history || p.rules.d_bias_ids ? (size_t)chunk * 4 : 0;
  auto kernel = p.bf16 ? rules_kernel<__nv_bfloat16> : rules_kernel<float>;
  if (smem > 48 * 1024) p.bf16 ? allow_smem<rules_kernel<__nv_bfloat16>>(kMaxChunk * 4) : allow_smem<rules_kernel<float>>(kMaxChunk * 4);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.rows * split));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  check_cuda(cudaLaunchKernelEx(&cfg, kernel, p, split, range, chunk), "rules launch");
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
    require(rows < (1LL << 27) && vocab <= (1 << 30), "too many rows or tokens", SVL_ERR_UNSUPPORTED);
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
