// f8_gemm.cu — products of e4m3 rows and e4m3 matrices with f32 scales per block of 128, on the
// 5th-generation tensor cores:
//   out[r][j] = sum_b xs[b][r] * ws[j / 128][b] * (sum_{k in b} xq[r][k] * wq[j][k]) + bias[j].
//
// The scales change every 128 columns, so the tensor cores' own accumulator only ever holds one
// block: each block's 128-wide product (four tcgen05.mma of K = 32) goes into one of several TMEM
// buffers, and warps that do nothing else read it back with tcgen05.ld, scale it and add it to
// running f32 sums in registers, while the next blocks' products run. 128 columns of e4m3 are one
// 128-byte swizzled row, so a block is also one stage of the shared-memory ring.
//
// Roles: one thread loads stages (weight tiles as contiguous 16 KB bulk copies from the packed
// image, rows by TMA), one issues the MMAs, and the epilogue warps keep the sums. Long axes are
// split over a cluster's CTAs when there are too few tiles; the partial sums are pushed to the
// CTA that owns their outputs and added in rank order, so results do not depend on timing.
//
// No load here uses cluster multicast.
#include <algorithm>
#include <type_traits>
#include <cuda_bf16.h>

#include "common.cuh"
#include "entry.h"
#include "f8.cuh"
#include "tcgen05.cuh"

namespace svl {
namespace {

constexpr uint32_t kTile = (uint32_t)kF8TileBytes;  // 16 KB: 128 rows x 128 columns
constexpr int kMaxSplit = 8;

__device__ __forceinline__ void dsmem_st4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d)
               : "memory");
}

struct F8Args {
  F8GemmParams p;
  int kblocks;
  int split;         // CTAs of a cluster, each a contiguous range of blocks
  int ntiles;        // tiles along the matrix rows
  int rtiles;        // tiles along the rows
};

// A block of the MMA issuer's and the loader's loops has to take less than the block's product (512
// clocks for 128 x 256). Their warps run the loops as a whole and elect a lane for the copies and
// products only, so that control flow, waits and addresses stay warp-uniform: a block of four
// products, two commits and two ready waits takes 374 clocks of issue this way and 588 in a
// single-lane branch. Stages are counted, not divided.

// A role's bounded wait; a wait that ran out marks the CTA as failed.
__device__ __forceinline__ bool role_wait(uint32_t bar, uint32_t parity, int* failed) {
  for (uint32_t i = 0; i < kWaitLimit; i++)
    if (mbar_try_wait_at(bar, parity)) return true;
  *failed = 1;
  return false;
}

// The loader's end: its last copies have landed (a CTA must not leave with copies in flight, also
// where another role gave up and stopped reading them).
__device__ __forceinline__ void drain_loads(uint64_t* full, int issued, int stages) {
  for (int i = issued > stages ? issued - stages : 0; i < issued; i++) mbar_wait(&full[i % stages], (i / stages) & 1);
}
// The MMA issuer's end after a wait that ran out: the products it has issued are done.
__device__ __forceinline__ void drain_mma(uint64_t* bar, bool lead) {
  if (lead) umma_commit(bar);
  __syncwarp();
  mbar_wait(bar, 0);
}

// ---- few rows: matrix rows are the MMA's M, up to BN rows its N ------------------------------

// Bound by the weights' bytes: every CTA keeps a ring of about 100 KB of loads in flight, two
// CTAs per SM. A stage of the ring, its TMEM buffer and its scales
// share one index and one phase: `full` (loaded), `done` (multiplied: the stage may be loaded
// again, the buffer read), `read` (the epilogue is through with buffer and scales).
template <int BN>
struct Thin {
  static constexpr int kEpiWarps = 4;
  static constexpr int kThreads = (kEpiWarps + 3) * 32;  // + loader, MMA issuer, scales
  static constexpr uint32_t kXBytes = BN * kF8Block;
  static constexpr uint32_t kStage = kTile + kXBytes;
  static constexpr int kStages = BN == 16 ? 6 : 5;
  static constexpr uint32_t kCols = BN == 16 ? 128 : 256;
  static constexpr size_t kRing = (size_t)kStages * kStage;
  static constexpr size_t kSmem = kRing + kStages * BN * 4 + 1024;
  static_assert(kStages * BN <= (int)kCols, "a TMEM buffer per stage");
  static_assert((size_t)(BN + 4 * kMaxSplit) * kF8Block * 4 <= kRing, "the exchange reuses the ring");
};

template <int BN>
__global__ void __launch_bounds__(Thin<BN>::kThreads, 2)
    f8_thin_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ F8Args a) {
  using C = Thin<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* scale_ring = reinterpret_cast<float*>(smem + C::kRing);
  __shared__ __align__(8) uint64_t full[C::kStages], done[C::kStages], read[C::kStages], scaled[C::kStages], gone;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const F8GemmParams& p = a.p;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int S = a.split;
  const int rank = S > 1 ? (int)cluster_rank() : 0;
  const int tile = blockIdx.x / S;
  const int r0 = blockIdx.y * BN;
  const int b0 = (int)((int64_t)rank * a.kblocks / S), nb = (int)((int64_t)(rank + 1) * a.kblocks / S) - b0;
  const int valid = (int)(p.rows - r0 < BN ? p.rows - r0 : BN);

  if (S > 1) cluster_arrive();  // waited for before the exchange: every CTA of the cluster runs
  const uint8_t* w = p.m.w + ((int64_t)tile * a.kblocks + b0) * kF8TileBytes;
  const int pre = nb < C::kStages ? nb : C::kStages;
  if (tid == C::kEpiWarps * 32) {
    // The weights do not depend on the kernel before, nor on the rest of the setup.
    for (int i = 0; i < C::kStages; i++) mbar_init(&full[i], 1);
    fence_mbar_init();
    for (int i = 0; i < pre; i++) {
      mbar_expect_tx(&full[i], C::kStage);
      bulk_g2s(smem + (size_t)i * C::kStage, w + i * kF8TileBytes, kTile, &full[i]);
    }
  }
  if (tid == 0) {
    for (int i = 0; i < C::kStages; i++) {
      mbar_init(&done[i], 1);
      mbar_init(&read[i], C::kEpiWarps);
      mbar_init(&scaled[i], 1);
    }
    mbar_init(&gone, 1);
    failed = 0;
    fence_mbar_init();
  }
  if (warp == C::kEpiWarps + 1) tmem_alloc(&tmem_slot, C::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  uint64_t acc[BN / 2];
#pragma unroll
  for (int i = 0; i < BN / 2; i++) acc[i] = 0;

  if (warp == C::kEpiWarps) {
    const bool lead = elect_one();
    pdl_wait();
    if (lead)
      for (int i = 0; i < pre; i++)
        tma_load_2d(smem + (size_t)i * C::kStage + kTile, &tm_x, (b0 + i) * kF8Block, r0, &full[i]);
    w += (int64_t)pre * kF8TileBytes;
    int i = pre, st = 0;
    uint32_t parity = 0;
    for (; i < nb; i++) {
      if (!role_wait(smem_addr(&done[st]), parity, &failed)) break;
      if (lead) {
        mbar_expect_tx(&full[st], C::kStage);
        bulk_g2s(smem + (size_t)st * C::kStage, w, kTile, &full[st]);
        tma_load_2d(smem + (size_t)st * C::kStage + kTile, &tm_x, (b0 + i) * kF8Block, r0, &full[st]);
      }
      __syncwarp();
      w += kF8TileBytes;
      if (++st == C::kStages) {
        st = 0;
        parity ^= 1;
      }
    }
    pdl_launch();
    drain_loads(full, i, C::kStages);
  } else if (warp == C::kEpiWarps + 1) {
    constexpr uint32_t idesc = idesc_e4m3(kF8Block, BN);
    const bool lead = elect_one();
    // The rows come after it: the bounded waits below do not count the kernel in front (a step of one STT-1b stream
    // takes 589 us, 584 without).
    pdl_wait();
    const uint32_t full_at = smem_addr(full), read_at = smem_addr(read);
    const uint64_t w_desc = sw128_desc(smem_addr(smem)), x_desc = sw128_desc(smem_addr(smem) + kTile);
    uint32_t parity = 0;
    bool ok = true;
    for (int left = nb; left > 0 && ok; left -= C::kStages, parity ^= 1) {
#pragma unroll
      for (int st = 0; st < C::kStages; st++) {
        if (st >= left || !ok) break;
        ok = role_wait(read_at + 8 * st, parity ^ 1, &failed) && role_wait(full_at + 8 * st, parity, &failed);
        if (!ok) break;
        tc_fence_after();
        if (lead) {
#pragma unroll
          for (int k = 0; k < 4; k++)
            umma_f8(tmem + st * BN, w_desc + (st * C::kStage >> 4) + 2 * k, x_desc + (st * C::kStage >> 4) + 2 * k, idesc, k != 0);
          umma_commit(&done[st]);
        }
        __syncwarp();
      }
    }
    if (!ok) drain_mma(&gone, lead);
  } else if (warp == C::kEpiWarps + 2) {
    // The blocks' scales, row scale times matrix scale; fetched four at a time.
    pdl_wait();
    constexpr int kPer = (BN + 31) / 32;
    const float* ws = p.m.scales + (int64_t)tile * a.kblocks + b0;
    const float* xs = p.scales + (int64_t)b0 * p.scale_stride + r0 + lane;
    float sx[4][kPer], sw[4];
    auto fetch = [&](int j, int i) {
      sw[j] = i < nb ? ws[i] : 0.f;
#pragma unroll
      for (int c = 0; c < kPer; c++) sx[j][c] = i < nb && c * 32 + lane < valid ? xs[(int64_t)i * p.scale_stride + c * 32] : 0.f;
    };
#pragma unroll
    for (int j = 0; j < 4; j++) fetch(j, j);
    bool ok = true;
    int st = 0;
    uint32_t parity = 1;
    for (int i0 = 0; i0 < nb && ok; i0 += 4) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (i0 + j >= nb || !ok) break;
        ok = role_wait(smem_addr(&read[st]), parity, &failed);
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < kPer; c++)
          if (c * 32 + lane < BN) scale_ring[st * BN + c * 32 + lane] = sx[j][c] * sw[j];
        __syncwarp();
        if (lane == 0) mbar_arrive(&scaled[st]);
        if (++st == C::kStages) {
          st = 0;
          parity ^= 1;
        }
      }
      // Not between the arrivals: each would wait for the loads in flight.
#pragma unroll
      for (int j = 0; j < 4; j++) fetch(j, i0 + j + 4);
    }
  } else {
    pdl_wait();
    const uint32_t trow = tmem + ((uint32_t)(warp * 32) << 16);
    int st = 0;
    uint32_t parity = 0;
    for (int i = 0; i < nb; i++) {
      if (!role_wait(smem_addr(&scaled[st]), parity, &failed) || !role_wait(smem_addr(&done[st]), parity, &failed)) break;
      __syncwarp();
      tc_fence_after();
      const ulonglong2* s2 = reinterpret_cast<const ulonglong2*>(scale_ring + st * BN);
      uint64_t t[BN / 2];
      tmem_ld_pairs<BN>(trow + st * BN, t);
#pragma unroll
      for (int j = 0; j < BN / 4; j++) {
        const ulonglong2 s = s2[j];
        fma_pair(acc[2 * j], t[2 * j], s.x);
        fma_pair(acc[2 * j + 1], t[2 * j + 1], s.y);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&read[st]);
      if (++st == C::kStages) {
        st = 0;
        parity ^= 1;
      }
    }
  }
  __syncwarp();

  const int row_l = (warp & 3) * 32 + lane;
  const int n = tile * kF8Block + row_l;
  const float bias = p.m.bias && n < p.m.n ? p.m.bias[n] : 0.f;
  auto put = [&](int64_t at, float y) {  // consecutive lanes, consecutive columns
    if (n >= p.m.n) return;
    if (p.m.bias) y = y + bias;
    if (p.out_bf16)
      static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
    else
      static_cast<float*>(p.out)[at] = y;
  };
  if (S == 1) {
    if (warp < C::kEpiWarps) {
      int64_t at = (int64_t)r0 * p.out_stride + n;
#pragma unroll
      for (int c = 0; c < BN; c++, at += p.out_stride)
        if (c < valid) put(at, c & 1 ? pair_hi(acc[c / 2]) : pair_lo(acc[c / 2]));
    }
  } else {
    // Every CTA of the cluster is done with its ring: it becomes the exchange, [rank][group of
    // kV columns of the owner][matrix row][kV]. Rank o owns the columns [o * cpr, (o + 1) * cpr).
    constexpr int kV = BN <= 16 ? 1 : 4;
    const int cpr = ((valid + S - 1) / S + kV - 1) / kV * kV;
    float* recv = reinterpret_cast<float*>(smem);
    cluster_wait();
    cluster_sync();
    if (warp < C::kEpiWarps) {
      float* mine = recv + ((size_t)rank * cpr * kF8Block + row_l * kV);
      int owner = 0, lc = 0;
      uint32_t to = dsmem_addr(mine, owner);
#pragma unroll
      for (int c = 0; c < BN; c += kV) {
        if (c >= valid) break;
        if constexpr (kV == 1)
          dsmem_st(to + lc * kF8Block * 4, c & 1 ? pair_hi(acc[c / 2]) : pair_lo(acc[c / 2]));
        else
          dsmem_st4(to + lc * kF8Block * 4, pair_lo(acc[c / 2]), pair_hi(acc[c / 2]), pair_lo(acc[c / 2 + 1]), pair_hi(acc[c / 2 + 1]));
        lc += kV;
        if (lc == cpr && c + kV < valid) {
          lc = 0;
          to = dsmem_addr(mine, ++owner);
        }
      }
    }
    cluster_sync();
    if (warp < C::kEpiWarps) {
      const int mine = min(cpr, valid - rank * cpr);
      for (int lc = 0; lc < mine; lc += kV) {
        float y[kV];
#pragma unroll
        for (int e = 0; e < kV; e++) y[e] = 0.f;
#pragma unroll
        for (int q = 0; q < kMaxSplit; q++) {
          if (q >= S) break;
          const float* src = recv + ((size_t)q * cpr + lc) * kF8Block + row_l * kV;
#pragma unroll
          for (int e = 0; e < kV; e++) y[e] += src[e];
        }
        int64_t at = (int64_t)(r0 + rank * cpr + lc) * p.out_stride + n;
#pragma unroll
        for (int e = 0; e < kV; e++, at += p.out_stride)
          if (lc + e < mine) put(at, y[e]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && failed && p.err) atomicExch(p.err, 2);
  if (warp == C::kEpiWarps + 1) tmem_free(tmem, C::kCols);
}

// Stores chunks of 32 bytes per row (8 f32 or 16 bf16 columns) for the 32 rows a warp's lanes hold,
// where a lane cannot store whole sectors itself (rows that start off 32 bytes, a tile's cut last
// columns). Through shared memory (the two 16-byte pieces swapped in every other group of four rows, so that
// neither side has bank conflicts): a lane's own row would make every store touch half a sector
// of 32 lines; this way a store instruction covers whole sectors of 16 rows.
struct RowStore {
  static constexpr uint32_t kPad = 32 * 32;  // bytes of shared memory per warp
  const F8GemmParams& p;
  uint32_t pad;
  int lane;
  int64_t r0;     // the row of lane 0
  bool aligned;   // rows start on 16 bytes
  bool sectors;   // rows start on 32 bytes

  static __device__ __forceinline__ uint32_t place(int row, int j) { return row * 32 + ((j ^ ((row >> 2) & 1)) << 4); }
  // Piece j of this lane's row: 4 f32 or 8 bf16 values.
  __device__ __forceinline__ void piece(int j, uint32_t a, uint32_t b, uint32_t c, uint32_t d) const {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(pad + place(lane, j)), "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
  }
  // The chunk that starts at column n0 (those of its first `width` columns that exist).
  template <class T>
  __device__ __forceinline__ void out(int n0, int width = 32 / sizeof(T)) const {
    constexpr int kPer = 16 / sizeof(T), kCols = 32 / sizeof(T);
    __syncwarp();
    const int cols = min(width, p.m.n - n0);
    T* base = static_cast<T*>(p.out) + r0 * p.out_stride + n0;
    if (aligned && cols == kCols) {
      const int j = lane & 1;
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const int row = i * 16 + (lane >> 1);
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(pad + place(row, j))
                     : "memory");
        if (r0 + row < p.rows) *reinterpret_cast<uint4*>(base + row * p.out_stride + j * kPer) = v;
      }
    } else {
      // One column per lane; four (two) rows per instruction, the shared-memory reads of all first.
      using U = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
      const int c = lane % kCols, row0 = lane / kCols;
      U v[kCols];
#pragma unroll
      for (int i = 0; i < kCols; i++) {
        const uint32_t from = pad + place(row0 + i * (32 / kCols), c / kPer) + c % kPer * sizeof(T);
        if constexpr (sizeof(T) == 4)
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[i]) : "r"(from) : "memory");
        else
          asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v[i]) : "r"(from) : "memory");
      }
      U* to = reinterpret_cast<U*>(base) + row0 * p.out_stride + c;
#pragma unroll
      for (int i = 0; i < kCols; i++, to += 32 / kCols * p.out_stride)
        if (c < cols && r0 + row0 + i * (32 / kCols) < p.rows) *to = v[i];
    }
    __syncwarp();
  }
};

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 32 bytes (a sector), 32-byte aligned.
__device__ __forceinline__ void store_sector(void* to, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// A thread's sums of columns [n0, n0 + N) of its row, plus the bias. Each lane stores the sectors of
// its own row where they are whole (1030 x 11264 x 2048 bf16: 36.4 us; 38.5 with every chunk through
// shared memory), else its warp does together.
template <int N>
__device__ __forceinline__ void store_sums(const RowStore& rs, uint64_t (&acc)[N / 2], int n0, bool bf16) {
  const F8GemmParams& p = rs.p;
  if (p.m.bias) {
#pragma unroll
    for (int c = 0; c < N; c += 2)
      acc[c / 2] = pair_of(pair_lo(acc[c / 2]) + (n0 + c < p.m.n ? p.m.bias[n0 + c] : 0.f),
                           pair_hi(acc[c / 2]) + (n0 + c + 1 < p.m.n ? p.m.bias[n0 + c + 1] : 0.f));
  }
  if (rs.sectors && n0 + N <= p.m.n) {
    const int64_t r = rs.r0 + rs.lane;
    if (r >= p.rows) return;
    if (bf16) {
      __nv_bfloat16* to = static_cast<__nv_bfloat16*>(p.out) + r * p.out_stride + n0;
#pragma unroll
      for (int c = 0; c < N; c += 16) {
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = bf16_pair(pair_lo(acc[c / 2 + e]), pair_hi(acc[c / 2 + e]));
        store_sector(to + c, v);
      }
    } else {
      float* to = static_cast<float*>(p.out) + r * p.out_stride + n0;
#pragma unroll
      for (int c = 0; c < N; c += 8) {
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          v[2 * e] = (uint32_t)acc[c / 2 + e];
          v[2 * e + 1] = (uint32_t)(acc[c / 2 + e] >> 32);
        }
        store_sector(to + c, v);
      }
    }
    return;
  }
  if (bf16) {
#pragma unroll
    for (int c = 0; c < N; c += 16) {
      if (n0 + c >= p.m.n) break;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const uint64_t* v = acc + c / 2 + 4 * j;
        rs.piece(j, bf16_pair(pair_lo(v[0]), pair_hi(v[0])), bf16_pair(pair_lo(v[1]), pair_hi(v[1])),
                 bf16_pair(pair_lo(v[2]), pair_hi(v[2])), bf16_pair(pair_lo(v[3]), pair_hi(v[3])));
      }
      rs.out<__nv_bfloat16>(n0 + c);
    }
  } else {
#pragma unroll
    for (int c = 0; c < N; c += 8) {
      if (n0 + c >= p.m.n) break;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const uint64_t* v = acc + c / 2 + 2 * j;
        rs.piece(j, (uint32_t)v[0], (uint32_t)(v[0] >> 32), (uint32_t)v[1], (uint32_t)(v[1] >> 32));
      }
      rs.out<float>(n0 + c);
    }
  }
}

// ---- many rows: the rows are the MMA's M, C::kTN matrix rows its N --------------------------------

// Bound by the tensor cores and by the operands' way from L2. With the rows as M, a thread of the
// epilogue holds one row, so a block's scale is one number per thread (no shared-memory reads).
// Persistent: a CTA takes every gridDim-th tile, and loads and products of the next tile run
// while one is stored.
struct Wide {
  static constexpr int kTN = 128;
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = (kEpiWarps + 2) * 32;  // + loader, MMA issuer
  static constexpr uint32_t kStage = 2 * kTile;
  static constexpr int kStages = 6;
  static constexpr int kBufs = 4;
  static constexpr size_t kRing = (size_t)kStages * kStage;
  static constexpr size_t kSmem = kRing + kEpiWarps * RowStore::kPad + 1024;
  static constexpr int kCpt = kTN / 2;
  static constexpr int kGroups = kTN / 8;  // groups of 8 columns, the unit of the exchange
  static_assert((size_t)(kGroups + kMaxSplit) * 8 * kF8Block * 4 <= kRing, "the exchange reuses the ring");
};

__global__ void __launch_bounds__(Wide::kThreads, 1) f8_wide_kernel(const __grid_constant__ CUtensorMap tm_x,
                                                                    const __grid_constant__ F8Args a) {
  using C = Wide;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[C::kStages], empty[C::kStages], tfull[C::kBufs], tempty[C::kBufs], gone;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const F8GemmParams& p = a.p;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int S = a.split;
  const int rank = S > 1 ? (int)cluster_rank() : 0;
  const int first = blockIdx.x / S, stride = gridDim.x / S, total = a.ntiles * a.rtiles;
  const int b0 = (int)((int64_t)rank * a.kblocks / S), nb = (int)((int64_t)(rank + 1) * a.kblocks / S) - b0;

  if (tid == 0) {
    for (int i = 0; i < C::kStages; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < C::kBufs; i++) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], C::kEpiWarps);
    }
    mbar_init(&gone, 1);
    failed = 0;
    fence_mbar_init();
  }
  if (warp == C::kEpiWarps + 1) tmem_alloc(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_wait();

  if (warp >= C::kEpiWarps) {
    const bool lead = elect_one();
    if (warp == C::kEpiWarps) {
      int issued = 0, st = 0;
      uint32_t parity = 1;
      bool ok = true;
      for (int tile = first; tile < total && ok; tile += stride) {
        const int nt = tile % a.ntiles, row = tile / a.ntiles * kF8Block;
        const uint8_t* w = p.m.w + ((int64_t)nt * a.kblocks + b0) * kF8TileBytes;
        for (int b = b0; b < b0 + nb; b++, issued++, w += kF8TileBytes) {
          ok = role_wait(smem_addr(&empty[st]), parity, &failed);
          if (!ok) break;
          if (lead) {
            uint64_t* bar = &full[st];
            uint8_t* at = smem + (size_t)st * C::kStage;
            mbar_expect_tx(bar, C::kStage);
            tma_load_2d(at, &tm_x, b * kF8Block, row, bar);
            bulk_g2s(at + kTile, w, kTile, bar);
          }
          __syncwarp();
          if (++st == C::kStages) {
            st = 0;
            parity ^= 1;
          }
        }
      }
      pdl_launch();
      drain_loads(full, issued, C::kStages);
    } else if (warp == C::kEpiWarps + 1) {
      // Tiles make no difference here: every block is a product of its own.
      constexpr uint32_t idesc = idesc_e4m3(kF8Block, C::kTN);
      const uint32_t full_at = smem_addr(full), tempty_at = smem_addr(tempty);
      const uint64_t x_desc = sw128_desc(smem_addr(smem)), w_desc = sw128_desc(smem_addr(smem) + kTile);
      const int blocks = (total - first + stride - 1) / stride * nb;
      int st = 0, buf = 0;
      uint32_t parity = 0, turn = 1;
      bool ok = true, free = true, here = mbar_test_at(full_at, 0);
#pragma unroll 1
      for (int i = 0; i < blocks; i++) {
        ok = (free || role_wait(tempty_at + 8 * buf, turn, &failed)) && (here || role_wait(full_at + 8 * st, parity, &failed));
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * C::kTN;
        const uint64_t at = (uint64_t)(st * (C::kStage >> 4));
        uint64_t *empty_bar = &empty[st], *tfull_bar = &tfull[buf];
        if (++st == C::kStages) {
          st = 0;
          parity ^= 1;
        }
        if (++buf == C::kBufs) {
          buf = 0;
          turn ^= 1;
        }
        // The next block's barriers are looked at while this block's products are issued.
        free = mbar_test_at(tempty_at + 8 * buf, turn);
        here = mbar_test_at(full_at + 8 * st, parity);
        if (lead) {
#pragma unroll
          for (int k = 0; k < 4; k++) umma_f8(d, x_desc + at + 2 * k, w_desc + at + 2 * k, idesc, k != 0);
          umma_commit(empty_bar);
          umma_commit(tfull_bar);
        }
        __syncwarp();
      }
      if (!ok) drain_mma(&gone, lead);
    }
    if (S > 1) {
      __syncwarp();
      cluster_sync();  // the epilogue warps' two barriers count every warp
      cluster_sync();
    }
  } else {
    const int half = warp >> 2, row_l = (warp & 3) * 32 + lane;
    const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16) + half * C::kCpt;
    const bool bf16 = p.out_bf16;
    RowStore rs{p, smem_addr(smem + C::kRing) + warp * RowStore::kPad, lane, 0,
                reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.out_stride % (bf16 ? 8 : 4) == 0,
                reinterpret_cast<uintptr_t>(p.out) % 32 == 0 && p.out_stride % (bf16 ? 16 : 8) == 0};
    auto bias_at = [&](int n) { return p.m.bias && n < p.m.n ? p.m.bias[n] : 0.f; };
    int buf = 0;
    uint32_t parity = 0;
    for (int tile = first; tile < total; tile += stride) {
      const int nt = tile % a.ntiles, rt = tile / a.ntiles;
      const int64_t r = (int64_t)rt * kF8Block + row_l;
      rs.r0 = r - lane;
      const bool live = r < p.rows;
      const float* xs = p.scales + (int64_t)b0 * p.scale_stride + (live ? r : 0);
      const float* ws = p.m.scales + (int64_t)nt * a.kblocks + b0;
      uint64_t acc[C::kCpt / 2];
#pragma unroll
      for (int i = 0; i < C::kCpt / 2; i++) acc[i] = 0;
      // The blocks' scales, four blocks ahead; multiplied where they are used, since a product here
      // would wait for its loads.
      float sx[4], sw[4];
      auto fetch = [&](int j, int b) {
        sx[j] = live && b < nb ? *xs : 0.f;
        sw[j] = live && b < nb ? ws[b] : 0.f;
        xs += p.scale_stride;
      };
#pragma unroll
      for (int j = 0; j < 4; j++) fetch(j, j);
      bool ok = true;
      for (int b1 = 0; b1 < nb && ok; b1 += 4) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (b1 + j >= nb || !ok) break;
          ok = role_wait(smem_addr(&tfull[buf]), parity, &failed);
          if (!ok) break;
          __syncwarp();
          tc_fence_after();
          const float sc = sx[j] * sw[j];
          const uint64_t sc2 = pair_of(sc, sc);
          fetch(j, b1 + j + 4);
#pragma unroll
          for (int c = 0; c < C::kCpt; c += 32) {
            uint64_t t[16];
            tmem_ld_pairs<32>(trow + buf * C::kTN + c, t);
#pragma unroll
            for (int e = 0; e < 16; e++) fma_pair(acc[c / 2 + e], t[e], sc2);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_relaxed(smem_addr(&tempty[buf]));
          if (++buf == C::kBufs) {
            buf = 0;
            parity ^= 1;
          }
        }
      }
      if (S == 1) {
        if (!ok) break;
        store_sums<C::kCpt>(rs, acc, nt * C::kTN + half * C::kCpt, bf16);
      } else {
        // One tile per cluster: its CTAs exchange their sums through the rings they are done
        // with, [rank][group of the owner][two float4][row]. Group g belongs to the rank whose
        // range [rank * groups / S, (rank + 1) * groups / S) holds it.
        cluster_sync();
        constexpr int G = C::kGroups;
        const int most = (G + S - 1) / S;
        float* recv = reinterpret_cast<float*>(smem);
        int owner = half * (G / 2) * S / G;
#pragma unroll
        for (int c = 0; c < C::kCpt; c += 8) {
          const int g = half * (G / 2) + c / 8;
          while (g >= (owner + 1) * G / S) owner++;
          const int lg = g - owner * G / S;
          const uint32_t at = dsmem_addr(recv + (((size_t)rank * most + lg) * 2 * kF8Block + row_l) * 4, owner);
          const uint64_t* v = acc + c / 2;
          dsmem_st4(at, pair_lo(v[0]), pair_hi(v[0]), pair_lo(v[1]), pair_hi(v[1]));
          dsmem_st4(at + kF8Block * 16, pair_lo(v[2]), pair_hi(v[2]), pair_lo(v[3]), pair_hi(v[3]));
        }
        cluster_sync();
        const int g0 = rank * G / S, g1 = (rank + 1) * G / S;
        for (int g = g0 + half; g < g1; g += 2) {
          const int n = nt * C::kTN + g * 8;
          if (n >= p.m.n) break;
          float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 0; q < kMaxSplit; q++) {
            if (q >= S) break;
            const float4* src = reinterpret_cast<const float4*>(recv) + ((size_t)q * most + (g - g0)) * 2 * kF8Block + row_l;
            const float4 u = src[0], v = src[kF8Block];
            y[0] += u.x; y[1] += u.y; y[2] += u.z; y[3] += u.w;
            y[4] += v.x; y[5] += v.y; y[6] += v.z; y[7] += v.w;
          }
          if (p.m.bias) {
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = y[e] + bias_at(n + e);
          }
          if (rs.aligned && n + 8 <= p.m.n) {
            if (r >= p.rows) continue;
            if (bf16) {
              __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + r * p.out_stride + n;
              *reinterpret_cast<uint4*>(o) = make_uint4(bf16_pair(y[0], y[1]), bf16_pair(y[2], y[3]), bf16_pair(y[4], y[5]), bf16_pair(y[6], y[7]));
            } else {
              float* o = static_cast<float*>(p.out) + r * p.out_stride + n;
              reinterpret_cast<float4*>(o)[0] = make_float4(y[0], y[1], y[2], y[3]);
              reinterpret_cast<float4*>(o)[1] = make_float4(y[4], y[5], y[6], y[7]);
            }
          } else if (bf16) {
            rs.piece(0, bf16_pair(y[0], y[1]), bf16_pair(y[2], y[3]), bf16_pair(y[4], y[5]), bf16_pair(y[6], y[7]));
            rs.out<__nv_bfloat16>(n, 8);
          } else {
            rs.piece(0, __float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3]));
            rs.piece(1, __float_as_uint(y[4]), __float_as_uint(y[5]), __float_as_uint(y[6]), __float_as_uint(y[7]));
            rs.out<float>(n);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && failed && p.err) atomicExch(p.err, 2);
  if (warp == C::kEpiWarps + 1) tmem_free(tmem, 512);
}

// ---- very many rows: 128 x 256 tiles ---------------------------------------------------------------

// The same with 256 matrix rows per tile (48 KB of operands per block for the work that takes 64 KB
// as two tiles of 128: with the narrower tiles the operands' way from L2 is the bound). The 20 warps leave a
// thread 96 registers, 64 of which hold its sums; the compiler spills 92 bytes. Scaling and
// adding a block's 128 x 256 products takes the SM's FMA pipes 256 clocks of the 512 that the
// products take, so it is spread over 16 warps, four per scheduler, each with 64 columns of 32
// rows. A warp of its own fetches the rows' scales into shared memory, 8 blocks at a time.
// Persistent: a CTA takes every gridDim-th tile, and loads and products of the next tile start
// while one is stored.
struct Big {
  static constexpr int kTN = 256;
  static constexpr int kEpiWarps = 16;
  static constexpr int kThreads = (kEpiWarps + 4) * 32;  // + loader, MMA issuer, scales, one idle
  static constexpr uint32_t kStage = 3 * kTile;
  static constexpr int kStages = 4;
  static constexpr int kBufs = 2;
  static constexpr int kChunk = 8;  // blocks whose row scales are fetched at once
  static constexpr size_t kRing = (size_t)kStages * kStage;
  static constexpr size_t kSmem = kRing + kEpiWarps * RowStore::kPad + 2 * kChunk * kF8Block * 4 + 1024;
  static constexpr int kCpt = kTN / 4;
};

__global__ void __launch_bounds__(Big::kThreads, 1) f8_big_kernel(const __grid_constant__ CUtensorMap tm_x,
                                                                    const __grid_constant__ F8Args a) {
  using C = Big;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* scale_ring = reinterpret_cast<float*>(smem + C::kRing + C::kEpiWarps * RowStore::kPad);  // [2][chunk][128 rows]
  __shared__ __align__(8) uint64_t full[C::kStages], empty[C::kStages], tfull[C::kBufs], tempty[C::kBufs],
      scaled[2], read[2], gone;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const F8GemmParams& p = a.p;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int first = blockIdx.x, stride = gridDim.x, total = a.ntiles * a.rtiles, nb = a.kblocks;

  if (tid == 0) {
    for (int i = 0; i < C::kStages; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < C::kBufs; i++) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], C::kEpiWarps);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&scaled[i], 1);
      mbar_init(&read[i], C::kEpiWarps);
    }
    mbar_init(&gone, 1);
    failed = 0;
    fence_mbar_init();
  }
  if (warp == C::kEpiWarps + 1) tmem_alloc(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_wait();

  if (warp == C::kEpiWarps) {
    const bool lead = elect_one();
    int issued = 0, st = 0;
    uint32_t parity = 1;
    bool ok = true;
    const int64_t next = (int64_t)nb * kF8TileBytes;  // the same block of the next 128 matrix rows
    for (int tile = first; tile < total && ok; tile += stride) {
      const int wt = tile % a.ntiles * 2, row = tile / a.ntiles * kF8Block;
      const bool both = wt + 1 < p.m.tiles();
      const uint8_t* w = p.m.w + (int64_t)wt * nb * kF8TileBytes;
      for (int b = 0; b < nb; b++, issued++, w += kF8TileBytes) {
        ok = role_wait(smem_addr(&empty[st]), parity, &failed);
        if (!ok) break;
        if (lead) {
          uint64_t* bar = &full[st];
          uint8_t* at = smem + (size_t)st * C::kStage;
          mbar_expect_tx(bar, both ? 3 * kTile : 2 * kTile);
          tma_load_2d(at, &tm_x, b * kF8Block, row, bar);
          bulk_g2s(at + kTile, w, kTile, bar);
          if (both) bulk_g2s(at + 2 * kTile, w + next, kTile, bar);
        }
        __syncwarp();
        if (++st == C::kStages) {
          st = 0;
          parity ^= 1;
        }
      }
    }
    pdl_launch();
    drain_loads(full, issued, C::kStages);
  } else if (warp == C::kEpiWarps + 1) {
    constexpr uint32_t idesc = idesc_e4m3(kF8Block, C::kTN);
    const bool lead = elect_one();
    const uint32_t full_at = smem_addr(full), tempty_at = smem_addr(tempty);
    const uint64_t x_desc = sw128_desc(smem_addr(smem)), w_desc = sw128_desc(smem_addr(smem) + kTile);
    const int blocks = (total - first + stride - 1) / stride * nb;
    int st = 0, buf = 0;
    uint32_t parity = 0, turn = 1;
    bool ok = true;
#pragma unroll 1
    for (int i = 0; i < blocks; i++) {
      ok = role_wait(full_at + 8 * st, parity, &failed) && role_wait(tempty_at + 8 * buf, turn, &failed);
      if (!ok) break;
      tc_fence_after();
      if (lead) {
        const uint64_t at = (uint64_t)(st * (C::kStage >> 4));
#pragma unroll
        for (int k = 0; k < 4; k++) umma_f8(tmem + buf * C::kTN, x_desc + at + 2 * k, w_desc + at + 2 * k, idesc, k != 0);
        umma_commit(&tfull[buf]);
        umma_commit(&empty[st]);
      }
      __syncwarp();
      if (++st == C::kStages) {
        st = 0;
        parity ^= 1;
      }
      buf ^= 1;
      turn ^= buf == 0;
    }
    if (!ok) drain_mma(&gone, lead);
  } else if (warp == C::kEpiWarps + 2) {
    int slot = 0;
    uint32_t parity = 1;
    bool ok = true;
    for (int tile = first; tile < total && ok; tile += stride) {
      const int64_t r0 = (int64_t)(tile / a.ntiles) * kF8Block + lane * 4;
      for (int i0 = 0; i0 < nb; i0 += C::kChunk) {
        float x[C::kChunk][4];
#pragma unroll
        for (int j = 0; j < C::kChunk; j++) {
          const float* xs = p.scales + (int64_t)(i0 + j) * p.scale_stride + r0;
#pragma unroll
          for (int e = 0; e < 4; e++) x[j][e] = i0 + j < nb && r0 + e < p.rows ? xs[e] : 0.f;
        }
        ok = role_wait(smem_addr(&read[slot]), parity, &failed);
        if (!ok) break;
        float4* to = reinterpret_cast<float4*>(scale_ring + slot * C::kChunk * kF8Block) + lane;
#pragma unroll
        for (int j = 0; j < C::kChunk; j++) to[j * 32] = make_float4(x[j][0], x[j][1], x[j][2], x[j][3]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&scaled[slot]);
        slot ^= 1;
        parity ^= slot == 0;
      }
    }
  } else if (warp < C::kEpiWarps) {
    const int cg = warp >> 2, row_l = (warp & 3) * 32 + lane;
    const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16) + cg * C::kCpt;
    int buf = 0, slot = 0;
    uint32_t parity = 0, turn = 0;
    bool ok = true;
    for (int tile = first; tile < total && ok; tile += stride) {
      const int n0 = tile % a.ntiles * C::kTN + cg * C::kCpt;
      const float* ws = p.m.scales + (int64_t)min(n0 / kF8Block, p.m.tiles() - 1) * nb;
      uint64_t acc[C::kCpt / 2];
#pragma unroll
      for (int i = 0; i < C::kCpt / 2; i++) acc[i] = 0;
      float sw = ws[0];
#pragma unroll 1
      for (int i0 = 0; i0 < nb && ok; i0 += C::kChunk) {
        ok = role_wait(smem_addr(&scaled[slot]), turn, &failed);
        if (!ok) break;
        const float* xs = scale_ring + slot * C::kChunk * kF8Block + row_l;
        const int end = min(nb, i0 + C::kChunk);
#pragma unroll 1
        for (int b = i0; b < end; b++, xs += kF8Block) {
          const float sc = *xs * sw;
          const uint64_t sc2 = pair_of(sc, sc);
          sw = ws[min(b + 1, nb - 1)];
          ok = role_wait(smem_addr(&tfull[buf]), parity, &failed);
          if (!ok) break;
          __syncwarp();
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < C::kCpt; c += 16) {
            uint64_t t[8];
            tmem_ld_pairs<16>(trow + buf * C::kTN + c, t);
#pragma unroll
            for (int e = 0; e < 8; e++) fma_pair(acc[c / 2 + e], t[e], sc2);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_relaxed(smem_addr(&tempty[buf]));
          buf ^= 1;
          parity ^= buf == 0;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&read[slot]);
        slot ^= 1;
        turn ^= slot == 0;
      }
      if (!ok) break;
      const bool bf16 = p.out_bf16;
      const RowStore rs{p, smem_addr(smem + C::kRing) + warp * RowStore::kPad, lane,
                        (int64_t)(tile / a.ntiles) * kF8Block + (warp & 3) * 32,
                        reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.out_stride % (bf16 ? 8 : 4) == 0,
                        reinterpret_cast<uintptr_t>(p.out) % 32 == 0 && p.out_stride % (bf16 ? 16 : 8) == 0};
      store_sums<C::kCpt>(rs, acc, n0, bf16);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && failed && p.err) atomicExch(p.err, 2);
  if (warp == C::kEpiWarps + 1) tmem_free(tmem, 512);
}

// ---- host side ----------------------------------------------------------------------------

bool make_rows_map(CUtensorMap* map, const uint8_t* base, int64_t rows, int k, int64_t stride, int box_rows) {
  const EncodeTiled enc = tma_encoder();
  if (!enc) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride};
  const cuuint32_t box[2] = {(cuuint32_t)kF8Block, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <auto kernel>
void launch(dim3 grid, int threads, size_t smem, int split, const CUtensorMap& map, const F8Args& a,
            cudaStream_t s) {
  allow_smem<kernel>(smem);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
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
  check_cuda(cudaLaunchKernelEx(&cfg, kernel, map, a), "product launch");
}

constexpr int kSms = 148;

// The rows' map and the tiles of tn matrix rows x br rows.
CUtensorMap plan(F8Args& a, int tn, int br) {
  CUtensorMap map;
  if (!make_rows_map(&map, a.p.q, a.p.rows, a.p.m.k, a.p.q_stride, br))
    throw Error(SVL_ERR_CUDA, "cannot encode the rows' TMA tensor map");
  a.ntiles = (a.p.m.n + tn - 1) / tn;
  a.rtiles = (int)((a.p.rows + br - 1) / br);
  if ((int64_t)a.ntiles * a.rtiles > INT32_MAX / kMaxSplit) throw Error(SVL_ERR_UNSUPPORTED, "too many output tiles");
  return map;
}

// Tiles of up to 32 rows. Clusters of 4 (2) as long as 200 CTAs are not exceeded and each has two
// blocks: the SMs that a few tiles leave idle then load too (1 x 2048 x 2048: 5.2 us alone, 4.0
// with 2, 3.4 with 4, 3.6 with 8; 1 x 11264 x 2048, 88 tiles: 5.9 alone, 6.2 with 2, 9.6 with 4).
// Clusters of 8 only for very long axes (1 x 2560 x 10240: 8.4 us with 4, 7.2 with 8), other sizes
// never won.
template <int BN>
void launch_thin(F8Args a, cudaStream_t s) {
  const CUtensorMap map = plan(a, kF8Block, BN);
  const int tiles = a.ntiles * a.rtiles;
  a.split = 1;
  while (a.split < 4 && tiles * a.split * 2 <= 200 && a.kblocks >= a.split * 4) a.split *= 2;
  if (a.split == 4 && tiles * 8 <= 200 && a.kblocks >= 80) a.split = 8;
  launch<f8_thin_kernel<BN>>(dim3(a.ntiles * a.split, a.rtiles), Thin<BN>::kThreads, Thin<BN>::kSmem, a.split, map, a, s);
}

// 128 x 128 tiles. The exchange of a split tile costs about as much as 9 blocks, so it is split only
// where it saves more (256 x 2048 x 5632, 32 tiles: 16.5 us alone, 12.5 with 2, 10.4 with 4; 256 x
// 6144 x 2048, 96 tiles: 9.3 alone, 16.9 with 2).
void launch_wide(F8Args a, cudaStream_t s) {
  const CUtensorMap map = plan(a, Wide::kTN, kF8Block);
  const int tiles = a.ntiles * a.rtiles;
  a.split = 1;
  for (int S : {2, 4})
    if (tiles * S <= kSms && a.kblocks * (S - 1) > 9 * S) a.split = S;
  const int grid = a.split > 1 ? tiles * a.split : std::min(tiles, kSms);
  launch<f8_wide_kernel>(dim3(grid), Wide::kThreads, Wide::kSmem, a.split, map, a, s);
}

void launch_big(F8Args a, cudaStream_t s) {
  const CUtensorMap map = plan(a, Big::kTN, kF8Block);
  a.split = 1;
  launch<f8_big_kernel>(dim3(std::min(a.ntiles * a.rtiles, kSms)), Big::kThreads, Big::kSmem, 1, map, a, s);
}

}  // namespace

// Which kernel. Up to 32 rows the matrix rows as M; above too, in tiles of 32 rows, as long as all of
// them run at once and have no more than 2,112 blocks in all, two of which an SM loads about as
// fast as one of a 128 x 128 tile, but whose tiles start, end and share a long axis faster: 147 x
// 225 x 2048 4.4 us against 7.1, 128 x 1024 x 5632 (1,408 blocks) 6.8 against 8.7, 160 x 1024 x 5632
// (1,760) 8.0 against 8.7, 128 x 2048 x 5120 (2,560) 9.0 against 8.5, 128 x 2048 x 5632 (2,816) 9.7
// against 8.9. From 2,048 blocks (8.2 against 7.9 in 128 tiles) to 2,304 (8.6 against 8.2) the two are
// within 5 % of each other, either way (2,112 in 48 tiles: 8.3 against 8.7), and the border lies there.
// Else 128 x 128 tiles or
// 128 x 256: a wave of the larger ones takes 1.55 times as long (1024 x 11264 x 2048: 35 us in 5
// waves, 33 in 3; 512 x 11264 x 2048: 22 us in 3, 23 in 2; 256 x 11264 x 2048: 15.5 us in 2, 13.3 in 1).
void launch_f8_gemm(const F8GemmParams& p, cudaStream_t s) {
  F8Args a{};
  a.p = p;
  a.kblocks = p.m.kblocks();
  const int64_t rt = (p.rows + kF8Block - 1) / kF8Block, thin_tiles = (p.rows + 31) / 32 * p.m.tiles();
  const int64_t wide_waves = (rt * p.m.tiles() + kSms - 1) / kSms, big_waves = (rt * ((p.m.tiles() + 1) / 2) + kSms - 1) / kSms;
  if (p.rows <= 16)
    launch_thin<16>(a, s);
  else if (p.rows <= 32 || (thin_tiles <= 2 * kSms && thin_tiles * a.kblocks <= 2112))
    launch_thin<32>(a, s);
  else if (big_waves * 31 < wide_waves * 20)
    launch_big(a, s);
  else
    launch_wide(a, s);
}

}  // namespace svl
