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

constexpr int kMaxThreads = 1024;
constexpr int kMaxChunk = 16384;  // tokens whose counts are held at once: 64 KB
constexpr int kAhead = 4;         // 16-byte loads of logits a thread has in flight
constexpr int kListAhead = 8;     // history entries a thread has in flight
constexpr int kMaxTouched = 4096; // touched tokens of a chunk that are listed (more are searched for)

// Bound by HBM for many tokens, by a chain of a few dependent loads for few. A row is shared by the
// CTAs of a cluster, each with a contiguous range of the vocabulary, taken in chunks (one, up to
// 131,072 tokens in 8 CTAs).
//
// The lists touch few tokens, so they are settled first and the stream over all tokens stays
// short (about ten instructions per token): `word` counts each token in the history (low 16 bits)
// and holds its first entry in the sparse biases (65,535 minus its index, high 16), by atomics whose
// result does not depend on their order. The entry that finds a token's word empty puts the token
// on a list and sets its bit in `touched`; then one thread per listed token computes its value up
// to the grammar and leaves it in `word`. The stream takes touched tokens' values from there. The
// row's first logits and history entries are on their way meanwhile.
//
// Positions are counted from the 16-byte boundary at or before the row's start ("lead" elements
// before it), so that every row is read in aligned 16-byte pieces, also where rows of an odd
// vocabulary start anywhere.
template <class T>
__global__ void __launch_bounds__(kMaxThreads) rules_kernel(const __grid_constant__ RulesParams p, int split, int range,
                                                            int chunk) {
  constexpr int VE = 16 / sizeof(T);
  extern __shared__ uint32_t word[];  // [chunk], then the bits
  __shared__ uint64_t best_sm[kMaxThreads / 32], best_of[8];
  __shared__ int twice, touched_n;
  const svl_logits_rules& R = p.rules;
  const int t = threadIdx.x, threads = blockDim.x;
  const int rank = split > 1 ? (int)cluster_rank() : 0;
  const int64_t r = blockIdx.x / split;
  if (split > 1) cluster_arrive();  // waited for before the ranks' shared memory is written
  pdl_launch();
  pdl_wait();
  uint32_t* touched = word + chunk;  // [chunk / 32], then the list
  uint16_t* list = reinterpret_cast<uint16_t*>(touched + chunk / 32);
  const T* in = static_cast<const T*>(p.logits) + r * p.logits_stride;
  T* out = p.out ? static_cast<T*>(p.out) + r * p.out_stride : nullptr;
  const int lead = (int)(reinterpret_cast<uintptr_t>(in) % 16 / sizeof(T));
  const bool wide_out = out && (reinterpret_cast<uintptr_t>(out) - reinterpret_cast<uintptr_t>(in)) % 16 == 0;
  const float* dense = R.d_dense_bias;
  const bool wide_bias = lead == 0 && reinterpret_cast<uintptr_t>(dense) % 16 == 0;
  const int end = p.vocab + lead;
  const int lo = rank * range, hi = min(lo + range, end);

  // 16 bytes of logits at position u (a multiple of VE), in flight until they are read.
  auto load = [&](int u) {
    uint4 v = make_uint4(0, 0, 0, 0);
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

  const int32_t* hist = R.d_history ? R.d_history + r * R.history_stride : nullptr;
  const int said = R.d_history ? max(0, min(R.d_lengths[r], R.history_cap)) : 0;
  // The first entries, fetched before the length is known to cover them.
  int said_id[kListAhead];
#pragma unroll
  for (int j = 0; j < kListAhead; j++)
    said_id[j] = hist && t + j * threads < R.history_cap ? hist[t + j * threads] : -1;
  const int listed = R.d_bias_ids ? R.bias_cap : 0;
  const int32_t* ids = listed ? R.d_bias_ids + r * R.bias_stride : nullptr;
  const float* vals = listed ? R.d_bias_values + r * R.bias_stride : nullptr;
  const uint32_t* mask = nullptr;
  if (R.d_masks) {
    const int64_t m = R.d_mask_rows ? R.d_mask_rows[r] : r;
    if (m >= 0 && m < R.n_masks) mask = R.d_masks + m * R.mask_stride;
  }
  float bv = -INFINITY;
  int bi = 0;
  for (int c0 = lo; c0 < hi; c0 += chunk) {
    const int c1 = min(c0 + chunk, hi);
    const int step = threads * VE;
    uint4 raw[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const int u = c0 + j * step + t * VE;
      if (u < c1) raw[j] = load(u);
    }
    const bool table = said || listed;
    if (table) {
      const int v0 = c0 - lead;                         // position 0's token, below 0 before the row
      const int from = max(v0, 0), to = c1 - lead;      // the chunk's tokens
      const int floor = max(from, R.first_penalised);   // those that the history counts for
      __syncthreads();
      for (int i = t * 4; i < (c1 - c0 + 31) / 32 * 32; i += threads * 4) *reinterpret_cast<uint4*>(word + i) = make_uint4(0, 0, 0, 0);
      for (int i = t; i < chunk / 32; i += threads) touched[i] = 0;
      if (t == 0) twice = touched_n = 0;
      __syncthreads();
      // Lists a token of the chunk, once per token.
      auto touch = [&](int at) {
        atomicOr(&touched[at >> 5], 1u << (at & 31));
        const int n = atomicAdd(&touched_n, 1);
        if (n < kMaxTouched) list[n] = (uint16_t)at;
      };
      if (listed) {
        for (int i = t; i < listed; i += threads) {
          const int id = ids[i];
          if (id >= from && id < to) atomicMax(&word[id - v0], (uint32_t)(65535 - i) << 16);
        }
        __syncthreads();
        for (int i = t; i < listed; i += threads) {
          const int id = ids[i];
          if (id < from || id >= to) continue;
          if ((int)(word[id - v0] >> 16) == 65535 - i)
            touch(id - v0);
          else
            twice = 1;
        }
      }
      for (int i0 = t; i0 < said; i0 += threads * kListAhead) {
        if (i0 != t) {
#pragma unroll
          for (int j = 0; j < kListAhead; j++) said_id[j] = i0 + j * threads < said ? hist[i0 + j * threads] : -1;
        }
#pragma unroll
        for (int j = 0; j < kListAhead; j++) {
          const int id = said_id[j];
          if (i0 + j * threads < said && id >= floor && id < to && atomicAdd(&word[id - v0], 1u) == 0) touch(id - v0);
        }
      }
      __syncthreads();
      const float rep = R.d_repetition ? R.d_repetition[r] : 1.f;
      const float freq = R.d_frequency ? R.d_frequency[r] : 0.f, pres = R.d_presence ? R.d_presence[r] : 0.f;
      auto settle = [&](int at) {
        const int v = v0 + at;
        const uint32_t w = word[at], c = w & 65535;
        float l = load_logit(in + v);
        if (c) {
          l = l > 0.f ? __fdiv_rn(l, rep) : l * rep;
          l = l - (freq * (float)c + pres);
        }
        if (dense) l = l + dense[v];
        if (w >> 16) {
          const int first = 65535 - (int)(w >> 16);
          l = l + vals[first];
          if (twice)
            for (int k = first + 1; k < listed; k++)
              if (ids[k] == v) l = l + vals[k];
        }
        word[at] = __float_as_uint(l);
      };
      const int n = touched_n;
      if (n <= kMaxTouched) {
        for (int i = t; i < n; i += threads) settle(list[i]);
      } else {
        for (int i = t; i < chunk / 32; i += threads)
          for (uint32_t bits = touched[i]; bits; bits &= bits - 1) settle(i * 32 + __ffs((int)bits) - 1);
      }
      // The next chunk's first entries again, where there is one.
      if (c1 < hi) {
#pragma unroll
        for (int j = 0; j < kListAhead; j++) said_id[j] = t + j * threads < said ? hist[t + j * threads] : -1;
      }
      __syncthreads();
    }
    for (int u0 = c0 + t * VE; u0 < c1; u0 += kAhead * step) {
      if (u0 >= c0 + kAhead * step) {
#pragma unroll
        for (int j = 0; j < kAhead; j++)
          if (u0 + j * step < c1) raw[j] = load(u0 + j * step);
      }
#pragma unroll
      for (int j = 0; j < kAhead; j++) {
        const int u = u0 + j * step;
        if (u >= c1) break;
        const int v = u - lead;  // the piece's first token (below 0 before the row)
        T e[VE];
        *reinterpret_cast<uint4*>(e) = raw[j];
        float l[VE];
#pragma unroll
        for (int i = 0; i < VE; i++) l[i] = load_logit(e + i);
        const bool inside = v >= 0 && v + VE <= p.vocab;
        if (dense) {
          if (wide_bias && inside) {
#pragma unroll
            for (int i = 0; i < VE; i += 4) {
              const float4 d = __ldg(reinterpret_cast<const float4*>(dense + v + i));
              l[i] = l[i] + d.x; l[i + 1] = l[i + 1] + d.y; l[i + 2] = l[i + 2] + d.z; l[i + 3] = l[i + 3] + d.w;
            }
          } else {
#pragma unroll
            for (int i = 0; i < VE; i++) l[i] = l[i] + (v + i >= 0 && v + i < p.vocab ? dense[v + i] : 0.f);
          }
        }
        if (table) {
          const uint32_t bits = touched[(u - c0) >> 5] >> ((u - c0) & 31) & ((1u << VE) - 1);
          if (bits) {
#pragma unroll
            for (int i = 0; i < VE; i++)
              if (bits >> i & 1) l[i] = __uint_as_float(word[u - c0 + i]);
          }
        }
        if (mask) {
          const int at = max(v, 0) >> 5, sh = max(v, 0) & 31;
          const uint32_t low = __ldg(mask + at);
          const uint32_t high = sh + VE > 32 && (at + 1) * 32 < p.vocab ? __ldg(mask + at + 1) : 0u;
          uint32_t allowed = __funnelshift_r(low, high, sh);
          if (v < 0) allowed <<= -v;
#pragma unroll
          for (int i = 0; i < VE; i++)
            if (!(allowed >> i & 1)) l[i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < VE; i++) store_logit(e + i, l[i]);
        if (inside) {
          if (wide_out) {
            *reinterpret_cast<uint4*>(out + v) = *reinterpret_cast<uint4*>(e);
          } else if (out) {
#pragma unroll
            for (int i = 0; i < VE; i++) out[v + i] = e[i];
          }
          float top = l[0];  // fmaxf passes over a NaN
#pragma unroll
          for (int i = 1; i < VE; i++) top = fmaxf(top, l[i]);
          if (top > bv) {
            bv = top;
#pragma unroll
            for (int i = VE - 1; i >= 0; i--)
              if (l[i] == top) bi = v + i;
          }
        } else {
          for (int i = 0; i < VE; i++) {
            if (v + i < 0 || v + i >= p.vocab) continue;
            if (out) out[v + i] = e[i];
            if (l[i] > bv) {
              bv = l[i];
              bi = v + i;
            }
          }
        }
      }
    }
  }
  uint64_t best = pick_key(bv, bi);
  for (int o = 16; o; o >>= 1) best = max_key(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((t & 31) == 0) best_sm[t >> 5] = best;
  __syncthreads();
  if (split > 1) cluster_wait();
  if (t < 32) {
    best = t < threads / 32 ? best_sm[t] : 0;
    for (int o = 16; o; o >>= 1) best = max_key(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (split > 1 && t == 0) dsmem_st64(dsmem_addr(&best_of[rank], 0), best);
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

// CTAs per row: one where it has at most 16,384 tokens to go through (a cluster costs more than its
// share of the work saves), else enough for four per SM and for ranges of one chunk.
void launch_rules(const RulesParams& p, cudaStream_t s) {
  const int ve = p.bf16 ? 8 : 4;
  const int64_t span = (int64_t)p.vocab + ve - 1;  // with the lead of the worst row
  int split = 1;
  if (span > kMaxChunk)
    while (split < 8 && (p.rows * split < 4 * 148 || span > (int64_t)split * kMaxChunk)) split *= 2;
  const int range = (int)((span + split - 1) / split + 31) / 32 * 32;
  const int chunk = std::min(range, kMaxChunk);
  // Two pieces per thread and more threads for a lone row, four and at most 256 threads for many.
  const int most = p.rows * split <= 148 ? kMaxThreads : p.rows * split <= 2 * 148 ? 512 : 256;
  const int threads = std::min(most, std::max(64, ((chunk + 2 * ve - 1) / (2 * ve) + 31) / 32 * 32));
  auto kernel = p.bf16 ? rules_kernel<__nv_bfloat16> : rules_kernel<float>;
  const size_t smem = p.rules.d_history || p.rules.d_bias_ids ? (size_t)chunk * 4 + chunk / 8 + kMaxTouched * 2 : 0;
  if (smem > 46 * 1024) {
    constexpr size_t kMost = kMaxChunk * 4 + kMaxChunk / 8 + kMaxTouched * 2;
    p.bf16 ? allow_smem<rules_kernel<__nv_bfloat16>>(kMost) : allow_smem<rules_kernel<float>>(kMost);
  }
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
  cfg.numAttrs = split > 1 ? 2 : 1;
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
