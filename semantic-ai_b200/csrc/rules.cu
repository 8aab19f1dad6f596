// rules.cu — the rules between logits and token: penalties for repeated tokens, biases, grammar
// masks, and the greedy pick.
#include <algorithm>
#include <atomic>
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

// 16 bytes of logits.
template <class T>
__device__ __forceinline__ void unpack_logits(const uint4& v, float* l) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (sizeof(T) == 4) {
      l[i] = __uint_as_float(w[i]);
    } else {
      l[2 * i] = __uint_as_float(w[i] << 16);
      l[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
template <class T>
__device__ __forceinline__ uint4 pack_logits(const float* l) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (sizeof(T) == 4) {
      w[i] = __float_as_uint(l[i]);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(l[2 * i], l[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 bytes that are read once.
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// An order-preserving key of a value above -infinity (0: none), then the lowest index: the
// larger key wins.
__device__ __forceinline__ uint64_t pick_key(float v, int i) {
  if (!(v > -INFINITY)) return 0;
  uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);  // -0 and 0 are equal
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)~i;
}
__device__ __forceinline__ uint64_t max_key(uint64_t a, uint64_t b) { return a > b ? a : b; }

constexpr int kMaxChunk = 131104;      // tokens of a CTA's chunk at most: 131,072 and the lead
constexpr int kMaxChunkLong = 16416;   // the same with lists of more than kLongLists entries
constexpr int kLongLists = 8192;
constexpr int kDirect = 8192;          // tokens of a chunk that has counts for all of them
constexpr int kAhead = 4;         // 16-byte loads of logits a thread has in flight
constexpr int kSettle = 2;        // touched tokens whose logits a thread has in flight over the stream
constexpr int kSlotBytes = 12;    // a touched token's count, first bias entry and position
constexpr uint32_t kRepeated = 1u << 31;  // in the place of a first entry: the token has several

// Adds the sparse biases of tokens with several entries to their values, in the entries' order, by one warp: 32
// entries at a time, of which those of one token are added lane by lane. Linear in the list, whatever repeats
// (every such token walking the list for itself: one row of 131,072 tokens, 8,192 entries of which one id is there
// twice, 764 us).
__device__ __forceinline__ void add_repeated(const int32_t* ids, const float* vals, int listed, int from, int to, int v0, bool direct,
                                          const uint32_t* first, const uint32_t* touched, const uint32_t* word_slot, uint32_t* value) {
  constexpr uint32_t kAll = 0xffffffffu;
  constexpr int kBatches = 8;  // ids of 256 entries in flight
  const int lane = threadIdx.x;
  for (int k0 = 0; k0 < listed; k0 += kBatches * 32) {
    int id[kBatches];
#pragma unroll
    for (int j = 0; j < kBatches; j++) id[j] = k0 + j * 32 + lane < listed ? ids[k0 + j * 32 + lane] : -1;
#pragma unroll 1
    for (int j = 0; j < kBatches; j++) {
      int at = -1;
      if (id[0] >= from && id[0] < to) {
        const int u = id[0] - v0;
        at = direct ? u : (int)word_slot[u >> 5] + __popc(touched[u >> 5] & ((1u << (u & 31)) - 1));
        if (first[at] != kRepeated) at = -1;
      }
      if (__any_sync(kAll, at >= 0)) {
        const float v = at >= 0 ? vals[k0 + j * 32 + lane] : 0.f;
        const uint32_t same = __match_any_sync(kAll, at);
        float sum = at >= 0 ? __uint_as_float(value[at]) : 0.f;
        uint32_t rest = at >= 0 ? same : 0;
        while (__any_sync(kAll, rest != 0)) {
          const float x = __shfl_sync(kAll, v, rest ? __ffs((int)rest) - 1 : lane);
          if (rest) sum = sum + x;
          rest &= rest - 1;
        }
        if (at >= 0 && __ffs((int)same) - 1 == lane) value[at] = __float_as_uint(sum);
        __syncwarp();
      }
#pragma unroll
      for (int i = 0; i + 1 < kBatches; i++) id[i] = id[i + 1];
    }
  }
}

// Bound by HBM for many tokens, by a chain of a few dependent loads for few. A row is shared by the
// CTAs of a cluster, each with a contiguous range of the vocabulary, taken in chunks (one, up to
// 131,072 tokens in 8 CTAs).
//
// The lists touch few tokens, so these are kept out of the stream over all tokens: each sets a bit in
// `touched`; then every word of bits takes as many slots as it has bits (a token's slot is its word's
// first plus the bits below its own), where the history counts the token and the sparse biases leave
// their first entry, by atomics whose result does not depend on their order. The touched tokens'
// logits are fetched before the stream, which passes over them as it does over tokens that the
// grammar forbids, and written after it. The row's first logits and list entries are on their way
// meanwhile. A chunk of at most 8,192 tokens has a count and an entry for each (`direct`): zeroing them
// takes less than giving slots (256 rows of 4,001 f32 tokens with all rules: 9.0 us, 9.9 with
// slots).
//
// Measured: 1 row of 8,000 f32 tokens with a history of 250, 16 biases and a mask 5.7 us (2.9 without
// rules); 256 rows of 4,001 f32 with all rules 9.0 us; 192 rows of 131,072 bf16 with all rules, a
// history of 2,048 each, 50.4 us (2.1 TB/s), 21 without any rule. More warps per SM would hide
// more of the lists' latency, but below 64 registers, at which the kernels of two and more CTAs per
// SM already spill up to 36 bytes, the spills cost more than they bring.
//
// Positions are counted from the 16-byte boundary at or before the row's start ("lead" elements
// before it), so that every row is read in aligned 16-byte pieces, also where rows of an odd
// vocabulary start anywhere; the elements before the first and after the last whole piece are
// taken one by one. The stream remembers the raw piece of its largest value; which of the piece's
// tokens it was is looked up once, at the end.
template <class T, int Threads, int PerSm>
__global__ void __launch_bounds__(Threads, PerSm) rules_kernel(const __grid_constant__ RulesParams p, int split, int range,
                                                               int chunk, int slots, int direct) {
  constexpr int VE = 16 / sizeof(T);
  constexpr int kListAhead = 2048 / Threads;  // history entries a thread has in flight
  extern __shared__ __align__(16) uint32_t count[];  // [slots]; then a settled value, past the threads' own
  __shared__ uint64_t best_sm[Threads / 32], best_of[8];
  __shared__ float penalty[3];  // repetition, frequency, presence
  __shared__ int twice, touched_n;
  const svl_logits_rules& R = p.rules;
  const int t = threadIdx.x, threads = blockDim.x;
  const int rank = split > 1 ? (int)cluster_rank() : 0;
  const int64_t r = blockIdx.x / split;
  if (split > 1) cluster_arrive();  // waited for before the ranks' shared memory is written
  pdl_launch();
  pdl_wait();
  uint32_t* first = count + slots;  // 65,536 minus the first entry's index, 0: none, or kRepeated
  int* list = reinterpret_cast<int*>(first + slots);
  uint32_t* touched = first + 2 * slots;       // [chunk / 32]
  uint32_t* word_slot = touched + chunk / 32;  // [chunk / 32]
  const T* in = static_cast<const T*>(p.logits) + r * p.logits_stride;
  T* out = p.out ? static_cast<T*>(p.out) + r * p.out_stride : nullptr;
  const int lead = (int)(reinterpret_cast<uintptr_t>(in) % 16 / sizeof(T));
  const bool wide_out = out && (reinterpret_cast<uintptr_t>(out) - reinterpret_cast<uintptr_t>(in)) % 16 == 0;
  const float* dense = R.d_dense_bias;
  const bool wide_bias = lead == 0 && reinterpret_cast<uintptr_t>(dense) % 16 == 0;
  const int end = p.vocab + lead, whole = end / VE * VE;  // whole: the end of the last whole piece
  const int lo = rank * range, hi = min(lo + range, end);

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
  const int bias_id = t < listed ? ids[t] : -1;
  const uint32_t* mask = nullptr;
  if (R.d_masks) {
    const int64_t m = R.d_mask_rows ? R.d_mask_rows[r] : r;
    if (m >= 0 && m < R.n_masks) mask = R.d_masks + m * R.mask_stride;
  }
  if (t < 3) {  // there are barriers before a counted token is settled
    const float* per_row = t == 0 ? R.d_repetition : t == 1 ? R.d_frequency : R.d_presence;
    penalty[t] = per_row ? per_row[r] : t == 0 ? 1.f : 0.f;
  }
  uint64_t best = 0;
  for (int c0 = lo; c0 < hi; c0 += chunk) {
    const int c1 = min(c0 + chunk, hi);
    const int v0 = c0 - lead;  // position 0's token, below 0 before the row
    // The chunk's whole pieces: c0 is a multiple of 32.
    const int w0 = c0 == 0 && lead ? VE : c0, w1 = min(c1, whole);
    const int step = threads * VE;
    uint4 raw[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
      const int u = w0 + j * step + t * VE;
      if (u < w1) raw[j] = load_once(in - lead + u);
    }
    // The elements outside whole pieces, of one thread each.
    int edge = -1;
    if (t < VE && c0 == 0 && t >= lead && t < min(w0, end)) edge = t;
    if (t >= VE && t < 2 * VE && max(whole, w0) + t - VE >= c0 && max(whole, w0) + t - VE < c1) edge = max(whole, w0) + t - VE;
    float edge_l = 0.f, edge_dense = 0.f;
    uint32_t edge_mask = ~0u;
    if (edge >= 0) {
      edge_l = load_logit(in - lead + edge);
      if (dense) edge_dense = dense[edge - lead];
      if (mask) edge_mask = mask[(edge - lead) >> 5];
    }
    const bool table = said || listed;
    int n = 0;  // touched tokens
    float mine[kSettle], mine_dense[kSettle];
    // A touched token's value up to the grammar, of its logit and dense bias; without the sparse biases
    // where it has several.
    auto settled = [&](int i, float l, float d) {
      const int at = direct ? list[i] : i;
      const uint32_t c = count[at], f = first[at];
      if (c) {
        l = l > 0.f ? __fdiv_rn(l, penalty[0]) : l * penalty[0];
        l = l - (penalty[1] * (float)c + penalty[2]);
      }
      if (dense) l = l + d;
      return f && f != kRepeated ? l + vals[65536 - (int)f] : l;
    };
    if (table) {
      const int from = max(v0, 0), to = c1 - lead;      // the chunk's tokens
      const int floor = max(from, R.first_penalised);   // those that the history counts for
      __syncthreads();
      for (int i = t; i < chunk / 32; i += threads) touched[i] = 0;
      if (direct)  // slots is the chunk, a multiple of 32
        for (int i = t * 4; i < 2 * slots; i += threads * 4) *reinterpret_cast<uint4*>(count + i) = make_uint4(0, 0, 0, 0);
      if (t == 0) twice = touched_n = 0;
      __syncthreads();
      auto entries = [&](auto&& biased, auto&& repeated) {
        for (int i = t; i < listed; i += threads) {
          const int id = i == t ? bias_id : ids[i];
          if (id >= from && id < to) biased(i, id - v0);
        }
#pragma unroll
        for (int j = 0; j < kListAhead; j++)
          if (t + j * threads < said && said_id[j] >= floor && said_id[j] < to) repeated(said_id[j] - v0);
        for (int i = t + kListAhead * threads; i < said; i += threads) {
          const int id = hist[i];
          if (id >= floor && id < to) repeated(id - v0);
        }
      };
      // Sets a token's bit; true for the thread that found it unset. Most entries repeat a few tokens,
      // so it looks before the atomic.
      auto touch = [&](int at) {
        const uint32_t bit = 1u << (at & 31);
        if (*reinterpret_cast<volatile uint32_t*>(&touched[at >> 5]) & bit) return false;
        return !(atomicOr(&touched[at >> 5], bit) & bit);
      };
      auto bias = [&](int i, int at) {
        if (!atomicMax(&first[at], 65536u - i)) return;
        atomicMax(&first[at], kRepeated);
        twice = 1;
      };
      if (direct) {
        auto add = [&](int at) {
          if (touch(at)) list[atomicAdd(&touched_n, 1)] = at;
        };
        entries([&](int i, int at) { add(at); bias(i, at); },
                [&](int at) { add(at); atomicAdd(&count[at], 1u); });
        __syncthreads();
      } else {
        entries([&](int, int at) { touch(at); }, [&](int at) { touch(at); });
        __syncthreads();
        for (int w = t; w < chunk / 32; w += threads) {
          uint32_t bits = touched[w];
          if (!bits) continue;
          int i = atomicAdd(&touched_n, __popc(bits));
          word_slot[w] = i;
          for (; bits; bits &= bits - 1, i++) {
            list[i] = w * 32 + __ffs((int)bits) - 1;
            count[i] = first[i] = 0;
          }
        }
        __syncthreads();
        auto slot = [&](int at) { return word_slot[at >> 5] + __popc(touched[at >> 5] & ((1u << (at & 31)) - 1)); };
        entries([&](int i, int at) { bias(i, slot(at)); },
                [&](int at) { atomicAdd(&count[slot(at)], 1u); });
      }
      n = touched_n;
#pragma unroll
      for (int j = 0; j < kSettle; j++) {
        const int i = t + j * threads;
        mine[j] = i < n ? load_logit(in + v0 + list[i]) : 0.f;
        mine_dense[j] = dense && i < n ? dense[v0 + list[i]] : 0.f;
      }
      __syncthreads();
      if (n > kSettle * threads) {
        for (int i = t + kSettle * threads; i < n; i += threads) {
          const int v = v0 + list[i];
          count[direct ? list[i] : i] = __float_as_uint(settled(i, load_logit(in + v), dense ? dense[v] : 0.f));
        }
        __syncthreads();  // the stream may overwrite the logits
      }
    }
    if (edge >= 0) {
      const int v = edge - lead;
      if (dense) edge_l = edge_l + edge_dense;
      if ((n && touched[(edge - c0) >> 5] >> ((edge - c0) & 31) & 1) || !(edge_mask >> (v & 31) & 1)) edge_l = -INFINITY;
      if (out) store_logit(out + v, edge_l);
      best = max_key(best, pick_key(edge_l, v));
    }
    // A piece's values; those of touched and forbidden tokens are -infinity.
    auto values = [&](const uint4& piece, int u, float* l) {
      const int v = u - lead;
      unpack_logits<T>(piece, l);
      if (dense) {
        if (wide_bias) {
#pragma unroll
          for (int i = 0; i < VE; i += 4) {
            const float4 d = __ldg(reinterpret_cast<const float4*>(dense + v + i));
            l[i] = l[i] + d.x; l[i + 1] = l[i + 1] + d.y; l[i + 2] = l[i + 2] + d.z; l[i + 3] = l[i + 3] + d.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < VE; i++) l[i] = l[i] + __ldg(dense + v + i);
        }
      }
      if (mask || n) {
        uint32_t allowed = ~0u;
        if (mask && !lead) {
          allowed = __ldg(reinterpret_cast<const uint8_t*>(mask) + (v >> 3)) >> (v & 4);
        } else if (mask) {
          const int at = v >> 5, sh = v & 31;
          const uint32_t low = __ldg(mask + at);
          const uint32_t high = sh + VE > 32 ? __ldg(mask + at + 1) : 0u;
          allowed = __funnelshift_r(low, high, sh);
        }
        if (n) allowed &= ~(touched[(u - c0) >> 5] >> ((u - c0) & 31));
#pragma unroll
        for (int i = 0; i < VE; i++)
          if (!(allowed >> i & 1)) l[i] = -INFINITY;
      }
    };
    float bv = -INFINITY;
    int bu = -1;
    uint4 piece = make_uint4(0, 0, 0, 0);
    for (int b0 = w0; b0 < w1; b0 += kAhead * step) {
      if (b0 != w0) {
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
          const int u = b0 + j * step + t * VE;
          if (u < w1) raw[j] = load_once(in - lead + u);
        }
      }
#pragma unroll
      for (int j = 0; j < kAhead; j++) {
        const int u = b0 + j * step + t * VE;
        if (u >= w1) continue;
        float l[VE];
        values(raw[j], u, l);
        if (out) {
          const uint4 packed = pack_logits<T>(l);
          if (wide_out) {
            *reinterpret_cast<uint4*>(out - lead + u) = packed;
          } else {
            const T* e = reinterpret_cast<const T*>(&packed);
#pragma unroll
            for (int i = 0; i < VE; i++) out[u - lead + i] = e[i];
          }
        }
        float top = l[0];  // fmaxf passes over a NaN
#pragma unroll
        for (int i = 1; i < VE; i++) top = fmaxf(top, l[i]);
        if (top > bv) {
          bv = top;
          bu = u;
          piece = raw[j];
        }
      }
    }
    if (bu >= 0) {
      float l[VE];
      values(piece, bu, l);
      int i = VE - 1;
#pragma unroll
      for (int j = VE - 2; j >= 0; j--)
        if (l[j] == bv) i = j;
      best = max_key(best, pick_key(bv, bu - lead + i));
    }
    if (n) {
      __syncthreads();  // the stream's stores are made
      auto put = [&](int i, float l) {
        const int v = v0 + list[i];
        if (mask && !(mask[v >> 5] >> (v & 31) & 1)) l = -INFINITY;
        if (out) store_logit(out + v, l);
        best = max_key(best, pick_key(l, v));
      };
      if (twice) {
        // The values of tokens with several entries stand in the place of their counts now.
#pragma unroll
        for (int j = 0; j < kSettle; j++) {
          const int i = t + j * threads, at = i < n ? direct ? list[i] : i : 0;
          if (i < n && first[at] == kRepeated) count[at] = __float_as_uint(settled(i, mine[j], mine_dense[j]));
        }
        __syncthreads();
        if (t < 32) add_repeated(ids, vals, listed, max(v0, 0), c1 - lead, v0, direct, first, touched, word_slot, count);
        __syncthreads();
      }
#pragma unroll
      for (int j = 0; j < kSettle; j++) {
        const int i = t + j * threads;
        if (i >= n) break;
        const int at = direct ? list[i] : i;
        put(i, first[at] == kRepeated ? __uint_as_float(count[at]) : settled(i, mine[j], mine_dense[j]));
      }
      for (int i = t + kSettle * threads; i < n; i += threads) put(i, __uint_as_float(count[direct ? list[i] : i]));
    }
  }
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
    // Arrivals: the rank's key is in rank 0, and it has read the history. Only rank 0 waits.
    cluster_arrive();
    if (rank) return;
    cluster_wait();
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

namespace {
template <auto Kernel>
auto with_smem(size_t bytes) {
  if (bytes > 46 * 1024) allow_smem<Kernel>(220 * 1024);
  return Kernel;
}

// How many clusters of n CTAs run at once, asked once per device: clusters stay inside a group of
// SMs, which leaves some SMs idle for most n.
template <auto Kernel, int Threads, int PerSm>
int64_t clusters_at_once(int n) {
  static std::atomic<int> known[64][9];
  int device = 0;
  check_cuda(cudaGetDevice(&device), "cudaGetDevice");
  std::atomic<int>* slot = device < 64 ? &known[device][n] : nullptr;
  if (slot && slot->load(std::memory_order_relaxed)) return slot->load(std::memory_order_relaxed);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n * PerSm * 148);
  cfg.blockDim = dim3(Threads);
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = n;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int c = 0;
  check_cuda(cudaOccupancyMaxActiveClusters(&c, Kernel, &cfg), "occupancy");
  c = std::max(1, std::min(c, 148 * PerSm / n));
  if (slot) slot->store(c, std::memory_order_relaxed);
  return c;
}

// A CTA's part of a row: its range of the vocabulary, taken in chunks, and the shared memory of their lists.
struct Part {
  int range, chunk, slots;
  bool direct;
  size_t smem;
  Part(int64_t span, int split, int entries) {
    range = (int)((span + split - 1) / split + 31) / 32 * 32;
    chunk = std::min(range, entries > kLongLists ? kMaxChunkLong : kMaxChunk);
    direct = chunk <= kDirect;
    slots = direct ? chunk : std::min(entries, chunk);
    smem = entries ? (size_t)chunk / 4 + (size_t)slots * kSlotBytes : 0;
  }
  // CTAs that an SM's 228 KB hold, each with 1 KB of its own and less than 1 KB of static shared memory.
  int per_sm() const { return (int)(228 * 1024 / (smem + 2048)); }
};

// CTAs per row. One where it has at most 16,384 tokens to go through: a cluster costs more than its
// share of the work saves. Up to 148 rows: the most that still run at once with an SM each (16
// rows of 131,072 bf16 tokens without rules: 6 CTAs 4.2 us, 8 in two waves 7.3; 64 rows: 2 CTAs
// 7.0, 8 CTAs 8.5). Where that is one CTA, two of a half each per SM for rows with lists, if they run
// at once (120 rows of 50,257 f32 tokens, a history of 500: 26 us with one, 21 with two). More
// rows: the number whose waves take the shortest, the lists and the
// joining of a CTA's results counted like 12,000 tokens (192 rows of 131,072 bf16 tokens with all
// rules: 5 CTAs 50.3 us, 2 CTAs 53, 8 CTAs 57, 1 CTA, of 512 threads then, 47; 512 rows of 32,000: 1 CTA 33, 2
// CTAs 41). Long lists leave room for fewer CTAs on an SM than the kernel's registers do, which counts (256 rows
// of 50,257 bf16 tokens with a history of 6,000: 31 us, 56 as if the lists took no memory).
template <class T>
int rules_split(int64_t rows, int64_t span, int entries) {
  if (span <= 16384) return 1;
  int split = 1;
  if (rows <= 148) {
    for (int n = 2; n <= 8; n++)
      if (rows <= clusters_at_once<rules_kernel<T, 512, 1>, 512, 1>(n)) split = n;
    if (split == 1 && entries && Part(span, 2, entries).per_sm() >= 2 && rows <= clusters_at_once<rules_kernel<T, 512, 2>, 512, 2>(2)) split = 2;
    return split;
  }
  int64_t least = INT64_MAX;
  for (int n = 1; n <= 8; n++) {
    const int fit = std::min(4, Part(span, n, entries).per_sm());
    const int64_t at_once = std::max<int64_t>(1, clusters_at_once<rules_kernel<T, 256, 4>, 256, 4>(n) * fit / 4);
    const int64_t t = (rows + at_once - 1) / at_once * (span / n + 12000);
    if (t < least) {
      least = t;
      split = n;
    }
  }
  return split;
}
}  // namespace

void launch_rules(const RulesParams& p, cudaStream_t s) {
  const int ve = p.bf16 ? 8 : 4;
  const int64_t span = (int64_t)p.vocab + ve - 1;  // with the lead of the worst row
  const int entries = (p.rules.d_history ? p.rules.history_cap : 0) + (p.rules.d_bias_ids ? p.rules.bias_cap : 0);
  const int split = p.bf16 ? rules_split<__nv_bfloat16>(p.rows, span, entries) : rules_split<float>(p.rows, span, entries);
  const Part part(span, split, entries);
  // Two pieces per thread; 512 threads where two CTAs per SM take all rows (256 rows of 4,001 f32
  // tokens with all rules: 8.9 us, 12.6 with 256 threads).
  const int64_t ctas = p.rows * split;
  const int most = ctas <= 2 * 148 ? 512 : 256;
  const int threads = std::min(most, std::max(64, ((part.chunk + 2 * ve - 1) / (2 * ve) + 31) / 32 * 32));
  auto launch = [&](auto kernel) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.rows * split));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = part.smem;
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
  check_cuda(cudaLaunchKernelEx(&cfg, kernel, p, split, part.range, part.chunk, part.slots, (int)part.direct), "rules launch");
  };
  auto variant = [&](auto type) {
    using T = decltype(type);
    if (ctas <= 148)
      launch(with_smem<rules_kernel<T, 512, 1>>(part.smem));
    else if (ctas <= 2 * 148)
      launch(with_smem<rules_kernel<T, 512, 2>>(part.smem));
    else
      launch(with_smem<rules_kernel<T, 256, 4>>(part.smem));
  };
  p.bf16 ? variant(__nv_bfloat16()) : variant(float());
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
    svl::require_aligned(dtype == SVL_DT_F32 ? 4 : 2, d_logits, d_out);
    svl::require_aligned(4, d_tokens, R.d_history, R.d_lengths, R.d_repetition, R.d_frequency, R.d_presence,
                         R.d_dense_bias, R.d_bias_ids, R.d_bias_values, R.d_masks, R.d_mask_rows);
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
