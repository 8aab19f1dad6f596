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

// The MMA issuer's and the loader's loops are single threads, a block of them has to take less than
// the block's product (512 clocks for 128 x 256), so they keep shared-memory addresses and
// descriptors in registers and count stages instead of dividing.

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
__device__ __forceinline__ void drain_mma(uint64_t* bar) {
  umma_commit(bar);
  mbar_wait(bar, 0);
}

// ---- few rows: matrix rows are the MMA's M, up to BN rows its N ------------------------------

// Bound by the weights' bytes: every CTA keeps a ring of about 100 KB of loads in flight, two
// CTAs per SM (one with 192 KB for 128 rows). A stage of the ring, its TMEM buffer and its scales
// share one index and one phase: `full` (loaded), `done` (multiplied: the stage may be loaded
// again, the buffer read), `read` (the epilogue is through with buffer and scales).
template <int BN>
struct Thin {
  static constexpr int kEpiWarps = BN <= 64 ? 4 : 8;
  static constexpr int kThreads = (kEpiWarps + 3) * 32;  // + loader, MMA issuer, scales
  static constexpr uint32_t kXBytes = BN * kF8Block;
  static constexpr uint32_t kStage = kTile + kXBytes;
  static constexpr int kStages = BN == 16 ? 6 : BN == 32 ? 5 : BN == 64 ? 4 : 4;
  static constexpr uint32_t kCols = BN == 16 ? 128 : BN == 32 ? 256 : BN == 64 ? 256 : 512;
  static constexpr size_t kRing = (size_t)kStages * kStage;
  static constexpr size_t kSmem = kRing + kStages * BN * 4 + 1024;
  static constexpr int kCpt = BN / (kEpiWarps / 4);  // columns (rows of x) per epilogue thread
  static constexpr int kLd = kCpt < 32 ? 16 : 32;    // columns per TMEM load
  static_assert(kStages * BN <= (int)kCols, "a TMEM buffer per stage");
  static_assert((size_t)(BN + 4 * kMaxSplit) * kF8Block * 4 <= kRing, "the exchange reuses the ring");
};

template <int BN>
__global__ void __launch_bounds__(Thin<BN>::kThreads, BN <= 64 ? 2 : 1)
    f8_thin_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ F8Args a) {
  using C = Thin<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* scale_ring = reinterpret_cast<float*>(smem + C::kRing);
  __shared__ __align__(8) uint64_t full[C::kStages], done[C::kStages], read[C::kStages], scaled[C::kStages], gone;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const F8GemmParams& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = a.split;
  const int rank = S > 1 ? (int)cluster_rank() : 0;
  const int tile = blockIdx.x / S;
  const int r0 = blockIdx.y * BN;
  const int b0 = (int)((int64_t)rank * a.kblocks / S), nb = (int)((int64_t)(rank + 1) * a.kblocks / S) - b0;
  const int valid = (int)(p.rows - r0 < BN ? p.rows - r0 : BN);

  if (tid == 0) {
    for (int i = 0; i < C::kStages; i++) {
      mbar_init(&full[i], 1);
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

  uint64_t acc[C::kCpt / 2];
#pragma unroll
  for (int i = 0; i < C::kCpt / 2; i++) acc[i] = 0;

  if (warp == C::kEpiWarps) {
    if (lane == 0) {
      // The weights do not depend on the kernel before: their first stages go out before the wait.
      const uint8_t* w = p.m.w + ((int64_t)tile * a.kblocks + b0) * kF8TileBytes;
      const int pre = nb < C::kStages ? nb : C::kStages;
      for (int i = 0; i < pre; i++) {
        mbar_expect_tx(&full[i], C::kStage);
        bulk_g2s(smem + (size_t)i * C::kStage, w + i * kF8TileBytes, kTile, &full[i]);
      }
      pdl_wait();
      for (int i = 0; i < pre; i++)
        tma_load_2d(smem + (size_t)i * C::kStage + kTile, &tm_x, (b0 + i) * kF8Block, r0, &full[i]);
      w += (int64_t)pre * kF8TileBytes;
      int i = pre, st = 0;
      uint32_t parity = 0;
      for (; i < nb; i++) {
        if (!role_wait(smem_addr(&done[st]), parity, &failed)) break;
        mbar_expect_tx(&full[st], C::kStage);
        bulk_g2s(smem + (size_t)st * C::kStage, w, kTile, &full[st]);
        tma_load_2d(smem + (size_t)st * C::kStage + kTile, &tm_x, (b0 + i) * kF8Block, r0, &full[st]);
        w += kF8TileBytes;
        if (++st == C::kStages) {
          st = 0;
          parity ^= 1;
        }
      }
      pdl_launch();
      drain_loads(full, i, C::kStages);
    }
  } else if (warp == C::kEpiWarps + 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_e4m3(kF8Block, BN);
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
#pragma unroll
          for (int k = 0; k < 4; k++)
            umma_f8(tmem + st * BN, w_desc + (st * C::kStage >> 4) + 2 * k, x_desc + (st * C::kStage >> 4) + 2 * k, idesc, k != 0);
          umma_commit(&done[st]);
        }
      }
      if (!ok) drain_mma(&gone);
    }
  } else if (warp == C::kEpiWarps + 2) {
    // The blocks' scales, row scale times matrix scale; fetched four blocks before they are stored.
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
        fetch(j, i0 + j + 4);
        __syncwarp();
        if (lane == 0) mbar_arrive(&scaled[st]);
        if (++st == C::kStages) {
          st = 0;
          parity ^= 1;
        }
      }
    }
  } else {
    pdl_wait();
    const int c0 = (warp >> 2) * C::kCpt;
    const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0;
    int st = 0;
    uint32_t parity = 0;
    for (int i = 0; i < nb; i++) {
      if (!role_wait(smem_addr(&scaled[st]), parity, &failed) || !role_wait(smem_addr(&done[st]), parity, &failed)) break;
      __syncwarp();
      tc_fence_after();
      const ulonglong2* s2 = reinterpret_cast<const ulonglong2*>(scale_ring + st * BN + c0);
#pragma unroll
      for (int c = 0; c < C::kCpt; c += C::kLd) {
        uint64_t t[C::kLd / 2];
        tmem_ld_pairs<C::kLd>(trow + st * BN + c, t);
#pragma unroll
        for (int j = 0; j < C::kLd / 4; j++) {
          const ulonglong2 s = s2[c / 4 + j];
          fma_pair(acc[c / 2 + 2 * j], t[2 * j], s.x);
          fma_pair(acc[c / 2 + 2 * j + 1], t[2 * j + 1], s.y);
        }
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
      const int c0 = (warp >> 2) * C::kCpt;
      int64_t at = (int64_t)(r0 + c0) * p.out_stride + n;
#pragma unroll
      for (int c = 0; c < C::kCpt; c++, at += p.out_stride)
        if (c0 + c < valid) put(at, c & 1 ? pair_hi(acc[c / 2]) : pair_lo(acc[c / 2]));
    }
  } else {
    // Every CTA of the cluster is done with its ring: it becomes the exchange, [rank][group of
    // kV columns of the owner][matrix row][kV]. Rank o owns the columns [o * cpr, (o + 1) * cpr).
    constexpr int kV = BN <= 16 ? 1 : 4;
    const int cpr = ((valid + S - 1) / S + kV - 1) / kV * kV;
    float* recv = reinterpret_cast<float*>(smem);
    cluster_sync();
    if (warp < C::kEpiWarps) {
      const int c0 = (warp >> 2) * C::kCpt;
      float* mine = recv + ((size_t)rank * cpr * kF8Block + row_l * kV);
      int owner = c0 / cpr, lc = c0 % cpr;
      uint32_t to = c0 < valid ? dsmem_addr(mine, owner) : 0;
#pragma unroll
      for (int c = 0; c < C::kCpt; c += kV) {
        if (c0 + c >= valid) break;
        if constexpr (kV == 1)
          dsmem_st(to + lc * kF8Block * 4, c & 1 ? pair_hi(acc[c / 2]) : pair_lo(acc[c / 2]));
        else
          dsmem_st4(to + lc * kF8Block * 4, pair_lo(acc[c / 2]), pair_hi(acc[c / 2]), pair_lo(acc[c / 2 + 1]), pair_hi(acc[c / 2 + 1]));
        lc += kV;
        if (lc == cpr && c0 + c + kV < valid) {
          lc = 0;
          to = dsmem_addr(mine, ++owner);
        }
      }
    }
    cluster_sync();
    if (warp < C::kEpiWarps) {
      const int mine = min(cpr, valid - rank * cpr);
      for (int lc = (warp >> 2) * kV; lc < mine; lc += C::kEpiWarps / 4 * kV) {
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

// ---- many rows: the rows are the MMA's M, TN matrix rows its N --------------------------------

// Bound by the tensor cores and by the operands' way from L2. With the rows as M, a thread of the
// epilogue holds one row, so a block's scale is one number per thread (no shared-memory reads).
// Persistent: a CTA takes every gridDim-th tile, and loads and products of the next tile run
// while one is stored.
template <int TN>
struct Wide {
  static constexpr int kEpiWarps = 8;
  // Loader and MMA issuer in a third warpgroup, which for TN = 256 gives registers to the other two
  // (128 running sums per thread): 384 x 168 at launch, 2 x 128 x 224 + 128 x 56 afterwards.
  static constexpr bool kShift = TN == 256;
  static constexpr int kThreads = 384;
  static constexpr uint32_t kWBytes = TN * kF8Block;
  static constexpr uint32_t kStage = kTile + kWBytes;
  static constexpr int kStages = (int)(192 * 1024 / kStage);
  static constexpr int kBufs = TN == 256 ? 2 : 3;
  static constexpr size_t kRing = (size_t)kStages * kStage;
  static constexpr uint32_t kPad = 32 * 128;  // bytes per warp: 128 bytes of each of 32 output rows
  static constexpr size_t kSmem = kRing + kEpiWarps * kPad + 1024;
  static constexpr int kCpt = TN / 2;
  static constexpr int kGroups = TN / 8;  // groups of 8 columns, the unit of the exchange
  static_assert(kStages % kBufs == 0, "stages and buffers share one unrolled loop");
  static_assert((size_t)(kGroups + kMaxSplit) * 8 * kF8Block * 4 <= kRing, "the exchange reuses the ring");
};

// Stores chunks of 128 bytes per row (32 f32 or 64 bf16 columns) for the 32 rows a warp's lanes hold.
// Through shared memory (16-byte pieces permuted by row, so neither side has bank conflicts): a
// lane's own row would make every store touch 32 lines; this way one store instruction covers
// whole lines of four rows.
struct RowStore {
  const F8GemmParams& p;
  uint32_t pad;   // this warp's 4 KB of shared memory
  int lane;
  int64_t r0;     // the row of lane 0
  bool aligned;   // rows start on 16 bytes

  // Piece j of this lane's row: 4 f32 or 8 bf16 values of columns n0 + j * 4 (8).
  __device__ __forceinline__ void piece(int j, uint32_t a, uint32_t b, uint32_t c, uint32_t d) const {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(pad + lane * 128 + ((j ^ (lane & 7)) << 4)), "r"(a),
                 "r"(b), "r"(c), "r"(d)
                 : "memory");
  }
  __device__ __forceinline__ uint4 at(int row, int j) const {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(pad + row * 128 + ((j ^ (row & 7)) << 4))
                 : "memory");
    return v;
  }
  // The chunk that starts at column n0, `bytes` (at most 128, for the last columns less) of it.
  template <class T>
  __device__ __forceinline__ void out(int n0) const {
    constexpr int kPer = 16 / sizeof(T);
    __syncwarp();
    const int cols = min(128 / (int)sizeof(T), p.m.n - n0);
    T* base = static_cast<T*>(p.out) + r0 * p.out_stride + n0;
    if (aligned && cols == 128 / (int)sizeof(T)) {
      const int j = lane & 7;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int row = i * 4 + (lane >> 3);
        const uint4 v = at(row, j);
        if (r0 + row < p.rows) *reinterpret_cast<uint4*>(base + row * p.out_stride + j * kPer) = v;
      }
    } else {
      const int rows = (int)min((int64_t)32, p.rows - r0);
      for (int row = 0; row < rows; row++)
        for (int c = lane; c < cols; c += 32) {
          const uint32_t from = pad + row * 128 + (((c / kPer) ^ (row & 7)) << 4) + c % kPer * sizeof(T);
          if constexpr (sizeof(T) == 4) {
            uint32_t v;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(from) : "memory");
            reinterpret_cast<uint32_t*>(base)[row * p.out_stride + c] = v;
          } else {
            uint16_t v;
            asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(from) : "memory");
            reinterpret_cast<uint16_t*>(base)[row * p.out_stride + c] = v;
          }
        }
    }
    __syncwarp();
  }
};

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int TN>
__global__ void __launch_bounds__(Wide<TN>::kThreads, 1) f8_wide_kernel(const __grid_constant__ CUtensorMap tm_x,
                                                                        const __grid_constant__ F8Args a) {
  using C = Wide<TN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[C::kStages], empty[C::kStages], tfull[C::kBufs], tempty[C::kBufs], gone;
  __shared__ uint32_t tmem_slot;
  __shared__ int failed;
  const F8GemmParams& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = a.split;
  const int rank = S > 1 ? (int)cluster_rank() : 0;
  const int first = blockIdx.x / S, stride = gridDim.x / S, total = a.ntiles * a.rtiles;
  const int b0 = (int)((int64_t)rank * a.kblocks / S), nb = (int)((int64_t)(rank + 1) * a.kblocks / S) - b0;
  constexpr int kTiles = TN / kF8Block;  // packed tiles per stage

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
    if (C::kShift) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == C::kEpiWarps && lane == 0) {
      int issued = 0, st = 0;
      uint32_t parity = 1;
      bool ok = true;
      for (int tile = first; tile < total && ok; tile += stride) {
        const int nt = tile % a.ntiles, row = tile / a.ntiles * kF8Block;
        const int have = min(kTiles, p.m.tiles() - nt * kTiles);
        const uint8_t* w = p.m.w + ((int64_t)nt * kTiles * a.kblocks + b0) * kF8TileBytes;
        const int64_t next = (int64_t)a.kblocks * kF8TileBytes;  // the same block of the next 128 matrix rows
        for (int b = b0; b < b0 + nb; b++, issued++, w += kF8TileBytes) {
          ok = role_wait(smem_addr(&empty[st]), parity, &failed);
          if (!ok) break;
          uint64_t* bar = &full[st];
          uint8_t* at = smem + (size_t)st * C::kStage;
          mbar_expect_tx(bar, kTile * (1 + have));
          tma_load_2d(at, &tm_x, b * kF8Block, row, bar);
          bulk_g2s(at + kTile, w, kTile, bar);
          if (kTiles > 1 && have > 1) bulk_g2s(at + 2 * kTile, w + next, kTile, bar);
          if (++st == C::kStages) {
            st = 0;
            parity ^= 1;
          }
        }
      }
      pdl_launch();
      drain_loads(full, issued, C::kStages);
    } else if (warp == C::kEpiWarps + 1 && lane == 0) {
      // Tiles make no difference here: every block is a product of its own.
      constexpr uint32_t idesc = idesc_e4m3(kF8Block, TN);
      constexpr int kTurns = C::kStages / C::kBufs;  // of the buffers per pass over the stages
      const uint32_t full_at = smem_addr(full), tempty_at = smem_addr(tempty);
      const uint64_t x_desc = sw128_desc(smem_addr(smem)), w_desc = sw128_desc(smem_addr(smem) + kTile);
      uint32_t pass = 0;
      bool ok = true;
      for (int left = (total - first + stride - 1) / stride * nb; left > 0 && ok; left -= C::kStages, pass++) {
#pragma unroll
        for (int st = 0; st < C::kStages; st++) {
          if (st >= left || !ok) break;
          constexpr int kB = C::kBufs;
          ok = role_wait(tempty_at + 8 * (st % kB), (pass * kTurns + st / kB + 1) & 1, &failed) &&
               role_wait(full_at + 8 * st, pass & 1, &failed);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < 4; k++)
            umma_f8(tmem + st % kB * TN, x_desc + (st * C::kStage >> 4) + 2 * k, w_desc + (st * C::kStage >> 4) + 2 * k, idesc, k != 0);
          umma_commit(&empty[st]);
          umma_commit(&tfull[st % kB]);
        }
      }
      if (!ok) drain_mma(&gone);
    }
    if (S > 1) {
      __syncwarp();
      cluster_sync();  // the epilogue warps' two barriers count every warp
      cluster_sync();
    }
  } else {
    if (C::kShift) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int half = warp >> 2, row_l = (warp & 3) * 32 + lane;
    const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16) + half * C::kCpt;
    const bool bf16 = p.out_bf16;
    RowStore rs{p, smem_addr(smem + C::kRing) + warp * C::kPad, lane, 0,
                reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.out_stride % (bf16 ? 8 : 4) == 0};
    auto bias_at = [&](int n) { return p.m.bias && n < p.m.n ? p.m.bias[n] : 0.f; };
    int buf = 0;
    uint32_t parity = 0;
    for (int tile = first; tile < total; tile += stride) {
      const int nt = tile % a.ntiles, rt = tile / a.ntiles;
      const int64_t r = (int64_t)rt * kF8Block + row_l;
      rs.r0 = r - lane;
      const int wt = nt * kTiles + (kTiles > 1 ? half : 0);
      const bool live = r < p.rows && wt < p.m.tiles();
      const float* xs = p.scales + (int64_t)b0 * p.scale_stride + (live ? r : 0);
      const float* ws = p.m.scales + (int64_t)(live ? wt : 0) * a.kblocks + b0;
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
          for (int c = 0; c < C::kCpt; c += 16) {
            uint64_t t[8];
            tmem_ld_pairs<16>(trow + buf * TN + c, t);
#pragma unroll
            for (int e = 0; e < 8; e++) fma_pair(acc[c / 2 + e], t[e], sc2);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tempty[buf]);
          if (++buf == C::kBufs) {
            buf = 0;
            parity ^= 1;
          }
        }
      }
      if (S == 1) {
        if (!ok) break;
        const int n0 = nt * TN + half * C::kCpt;
        if (p.m.bias) {
#pragma unroll
          for (int c = 0; c < C::kCpt; c += 2)
            acc[c / 2] = pair_of(pair_lo(acc[c / 2]) + bias_at(n0 + c), pair_hi(acc[c / 2]) + bias_at(n0 + c + 1));
        }
        if (bf16) {
#pragma unroll
          for (int c = 0; c < C::kCpt; c += 64) {
            if (n0 + c >= p.m.n) break;
#pragma unroll
            for (int j = 0; j < 8; j++) {
              const uint64_t* v = acc + c / 2 + 4 * j;
              rs.piece(j, bf16_pair(pair_lo(v[0]), pair_hi(v[0])), bf16_pair(pair_lo(v[1]), pair_hi(v[1])),
                       bf16_pair(pair_lo(v[2]), pair_hi(v[2])), bf16_pair(pair_lo(v[3]), pair_hi(v[3])));
            }
            rs.out<__nv_bfloat16>(n0 + c);
          }
        } else {
#pragma unroll
          for (int c = 0; c < C::kCpt; c += 32) {
            if (n0 + c >= p.m.n) break;
#pragma unroll
            for (int j = 0; j < 8; j++) {
              const uint64_t* v = acc + c / 2 + 2 * j;
              rs.piece(j, (uint32_t)v[0], (uint32_t)(v[0] >> 32), (uint32_t)v[1], (uint32_t)(v[1] >> 32));
            }
            rs.out<float>(n0 + c);
          }
        }
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
          const int n = nt * TN + g * 8;
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
          if (r >= p.rows) continue;
          const bool whole = rs.aligned && n + 8 <= p.m.n;
          if (p.m.bias) {
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = y[e] + bias_at(n + e);
          }
          if (bf16) {
            __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + r * p.out_stride + n;
            if (whole)
              *reinterpret_cast<uint4*>(o) = make_uint4(bf16_pair(y[0], y[1]), bf16_pair(y[2], y[3]), bf16_pair(y[4], y[5]), bf16_pair(y[6], y[7]));
            else
#pragma unroll
              for (int e = 0; e < 8; e++)
                if (n + e < p.m.n) o[e] = __float2bfloat16_rn(y[e]);
          } else {
            float* o = static_cast<float*>(p.out) + r * p.out_stride + n;
            if (whole) {
              reinterpret_cast<float4*>(o)[0] = make_float4(y[0], y[1], y[2], y[3]);
              reinterpret_cast<float4*>(o)[1] = make_float4(y[4], y[5], y[6], y[7]);
            } else
#pragma unroll
              for (int e = 0; e < 8; e++)
                if (n + e < p.m.n) o[e] = y[e];
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

// CTAs per cluster so that `tiles` tiles fill `slots` CTAs, each with at least `least` blocks.
int choose_split(int64_t tiles, int kblocks, int slots, int least) {
  const int64_t s = std::min<int64_t>({slots / std::max<int64_t>(tiles, 1), kMaxSplit, kblocks / least});
  return (int)std::max<int64_t>(s, 1);
}

template <int BN>
void launch_thin(F8Args a, cudaStream_t s) {
  CUtensorMap map;
  if (!make_rows_map(&map, a.p.q, a.p.rows, a.p.m.k, a.p.q_stride, BN))
    throw Error(SVL_ERR_CUDA, "cannot encode the rows' TMA tensor map");
  a.ntiles = a.p.m.tiles();
  a.rtiles = (int)((a.p.rows + BN - 1) / BN);
  a.split = choose_split((int64_t)a.ntiles * a.rtiles, a.kblocks, 2 * 148, 1);
  launch<f8_thin_kernel<BN>>(dim3(a.ntiles * a.split, a.rtiles), Thin<BN>::kThreads, Thin<BN>::kSmem, a.split, map, a, s);
}

template <int TN>
void launch_wide(F8Args a, cudaStream_t s) {
  CUtensorMap map;
  if (!make_rows_map(&map, a.p.q, a.p.rows, a.p.m.k, a.p.q_stride, kF8Block))
    throw Error(SVL_ERR_CUDA, "cannot encode the rows' TMA tensor map");
  a.ntiles = (a.p.m.n + TN - 1) / TN;
  a.rtiles = (int)((a.p.rows + kF8Block - 1) / kF8Block);
  const int64_t tiles = (int64_t)a.ntiles * a.rtiles;
  if (tiles > INT32_MAX) throw Error(SVL_ERR_UNSUPPORTED, "too many output tiles");
  a.split = choose_split(tiles, a.kblocks, 148, 2);
  const int grid = a.split > 1 ? (int)tiles * a.split : (int)std::min<int64_t>(tiles, 148);
  launch<f8_wide_kernel<TN>>(dim3(grid), Wide<TN>::kThreads, Wide<TN>::kSmem, a.split, map, a, s);
}

}  // namespace

void launch_f8_gemm(const F8GemmParams& p, cudaStream_t s) {
  F8Args a{};
  a.p = p;
  a.kblocks = p.m.kblocks();
  if (p.rows <= 16)
    launch_thin<16>(a, s);
  else if (p.rows <= 32)
    launch_thin<32>(a, s);
  else if (p.rows <= 64)
    launch_thin<64>(a, s);
  else if (p.rows <= 128)
    launch_thin<128>(a, s);
  else if ((p.rows + 127) / 128 * ((p.m.n + 255) / 256) < 148)
    launch_wide<128>(a, s);
  else
    launch_wide<256>(a, s);
}

}  // namespace svl
