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

// A role's bounded wait; a wait that ran out marks the CTA as failed.
__device__ __forceinline__ bool role_wait(uint64_t* bar, uint32_t parity, volatile int* failed) {
  if (mbar_wait(bar, parity)) return true;
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
// CTAs per SM.
template <int BN>
struct Thin {
  static constexpr int kEpiWarps = BN <= 64 ? 4 : 8;
  static constexpr int kThreads = (kEpiWarps + 3) * 32;  // + loader, MMA issuer, scales
  static constexpr uint32_t kXBytes = BN * kF8Block;
  static constexpr uint32_t kStage = kTile + kXBytes;
  static constexpr int kStages = (int)(106 * 1024 / kStage);
  static constexpr int kBufs = BN <= 32 ? 4 : 2;
  static constexpr uint32_t kCols = BN * kBufs < 32 ? 32 : BN * kBufs;
  static constexpr int kScaleSlots = 8;
  static constexpr size_t kRing = (size_t)kStages * kStage;
  static constexpr size_t kSmem = kRing + kScaleSlots * BN * 4 + 1024;
  static constexpr int kCpt = BN / (kEpiWarps / 4);  // columns (rows of x) per epilogue thread
  static_assert((size_t)(BN + kMaxSplit) * kF8Block * 4 <= kRing, "the exchange reuses the ring");
};

template <int BN>
__global__ void __launch_bounds__(Thin<BN>::kThreads) f8_thin_kernel(const __grid_constant__ CUtensorMap tm_x,
                                                                     const __grid_constant__ F8Args a) {
  using C = Thin<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* scale_ring = reinterpret_cast<float*>(smem + C::kRing);
  __shared__ __align__(8) uint64_t full[C::kStages], empty[C::kStages], tfull[C::kBufs], tempty[C::kBufs],
      sfull[C::kScaleSlots], sempty[C::kScaleSlots], gone;
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
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < C::kBufs; i++) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], C::kEpiWarps);
    }
    for (int i = 0; i < C::kScaleSlots; i++) {
      mbar_init(&sfull[i], 1);
      mbar_init(&sempty[i], C::kEpiWarps);
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

  float acc[C::kCpt];
#pragma unroll
  for (int i = 0; i < C::kCpt; i++) acc[i] = 0.f;

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
      int i = pre;
      for (; i < nb; i++) {
        const int st = i % C::kStages;
        if (!role_wait(&empty[st], ((i / C::kStages) - 1) & 1, &failed)) break;
        mbar_expect_tx(&full[st], C::kStage);
        bulk_g2s(smem + (size_t)st * C::kStage, w + i * kF8TileBytes, kTile, &full[st]);
        tma_load_2d(smem + (size_t)st * C::kStage + kTile, &tm_x, (b0 + i) * kF8Block, r0, &full[st]);
      }
      pdl_launch();
      drain_loads(full, i, C::kStages);
    }
  } else if (warp == C::kEpiWarps + 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_e4m3(kF8Block, BN);
      for (int i = 0; i < nb; i++) {
        const int st = i % C::kStages, buf = i % C::kBufs;
        if (i >= C::kBufs && !role_wait(&tempty[buf], ((i / C::kBufs) - 1) & 1, &failed)) break;
        if (!role_wait(&full[st], (i / C::kStages) & 1, &failed)) break;
        tc_fence_after();
        const uint32_t wa = smem_addr(smem + (size_t)st * C::kStage), xa = wa + kTile;
#pragma unroll
        for (int k = 0; k < 4; k++)
          umma_f8(tmem + buf * BN, sw128_desc(wa + k * 32), sw128_desc(xa + k * 32), idesc, k != 0);
        umma_commit(&empty[st]);
        umma_commit(&tfull[buf]);
      }
      if (failed) drain_mma(&gone);
    }
  } else if (warp == C::kEpiWarps + 2) {
    // The blocks' scales, row scale times matrix scale, kScaleSlots blocks ahead.
    pdl_wait();
    constexpr int kPer = (BN + 31) / 32;
    const float* ws = p.m.scales + (int64_t)tile * a.kblocks + b0;
    const float* xs = p.scales + (int64_t)b0 * p.scale_stride + r0;
    for (int i0 = 0; i0 < nb; i0 += 4) {
      float v[4][kPer];
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int c = 0; c < kPer; c++) {
          const int col = c * 32 + lane;
          v[j][c] = i0 + j < nb && col < valid ? xs[(int64_t)(i0 + j) * p.scale_stride + col] * ws[i0 + j] : 0.f;
        }
      bool ok = true;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int i = i0 + j;
        if (i >= nb || !ok) break;
        const int slot = i % C::kScaleSlots;
        if (i >= C::kScaleSlots) ok = role_wait(&sempty[slot], ((i / C::kScaleSlots) - 1) & 1, &failed);
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < kPer; c++)
          if (c * 32 + lane < BN) scale_ring[slot * BN + c * 32 + lane] = v[j][c];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sfull[slot]);
      }
      if (!ok) break;
    }
  } else {
    pdl_wait();
    const int c0 = (warp >> 2) * C::kCpt;
    const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0;
    for (int i = 0; i < nb; i++) {
      const int slot = i % C::kScaleSlots, buf = i % C::kBufs;
      if (!role_wait(&sfull[slot], (i / C::kScaleSlots) & 1, &failed)) break;
      if (!role_wait(&tfull[buf], (i / C::kBufs) & 1, &failed)) break;
      __syncwarp();
      tc_fence_after();
      const float4* s4 = reinterpret_cast<const float4*>(scale_ring + slot * BN + c0);
      uint32_t t[16];
#pragma unroll
      for (int c = 0; c < C::kCpt; c += 16) {
        tmem_ld16_async(trow + buf * BN + c, t);
        tmem_wait(t);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float4 s = s4[c / 4 + j];
          acc[c + 4 * j + 0] = fmaf(__uint_as_float(t[4 * j + 0]), s.x, acc[c + 4 * j + 0]);
          acc[c + 4 * j + 1] = fmaf(__uint_as_float(t[4 * j + 1]), s.y, acc[c + 4 * j + 1]);
          acc[c + 4 * j + 2] = fmaf(__uint_as_float(t[4 * j + 2]), s.z, acc[c + 4 * j + 2]);
          acc[c + 4 * j + 3] = fmaf(__uint_as_float(t[4 * j + 3]), s.w, acc[c + 4 * j + 3]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&tempty[buf]);
        mbar_arrive(&sempty[slot]);
      }
    }
  }
  __syncwarp();

  const int row_l = (warp & 3) * 32 + lane;
  const int n = tile * kF8Block + row_l;
  auto put = [&](int c, float y) {  // output (r0 + c, n): consecutive lanes, consecutive columns
    if (n >= p.m.n) return;
    if (p.m.bias) y = y + p.m.bias[n];
    const int64_t at = (int64_t)(r0 + c) * p.out_stride + n;
    if (p.out_bf16)
      static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
    else
      static_cast<float*>(p.out)[at] = y;
  };
  if (S == 1) {
    if (warp < C::kEpiWarps) {
      const int c0 = (warp >> 2) * C::kCpt;
#pragma unroll
      for (int c = 0; c < C::kCpt; c++)
        if (c0 + c < valid) put(c0 + c, acc[c]);
    }
  } else {
    // Every CTA of the cluster is done with its ring: it becomes the exchange [rank][column of the
    // owner][matrix row]. The owner of column c is rank c / cpr.
    const int cpr = (valid + S - 1) / S;
    float* recv = reinterpret_cast<float*>(smem);
    cluster_sync();
    if (warp < C::kEpiWarps) {
      const int c0 = (warp >> 2) * C::kCpt;
#pragma unroll
      for (int c = 0; c < C::kCpt; c++) {
        if (c0 + c >= valid) break;
        const int owner = (c0 + c) / cpr, lc = (c0 + c) % cpr;
        dsmem_st(dsmem_addr(recv + ((size_t)rank * cpr + lc) * kF8Block + row_l, owner), acc[c]);
      }
    }
    cluster_sync();
    if (warp < C::kEpiWarps) {
      const int mine = min(cpr, valid - rank * cpr);
      for (int lc = warp >> 2; lc < mine; lc += C::kEpiWarps / 4) {
        float y = 0.f;
        for (int q = 0; q < S; q++) y += recv[((size_t)q * cpr + lc) * kF8Block + row_l];
        put(rank * cpr + lc, y);
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
template <int TN>
struct Wide {
  static constexpr int kEpiWarps = 8;
  // Loader and MMA issuer in a third warpgroup, which for TN = 256 gives registers to the other two
  // (128 running sums per thread): 384 x 168 at launch, 2 x 128 x 208 + 128 x 72 afterwards.
  static constexpr bool kShift = TN == 256;
  static constexpr int kThreads = 384;
  static constexpr uint32_t kWBytes = TN * kF8Block;
  static constexpr uint32_t kStage = kTile + kWBytes;
  static constexpr int kStages = (int)(192 * 1024 / kStage);
  static constexpr int kBufs = 2;
  static constexpr uint32_t kCols = TN * kBufs;
  static constexpr size_t kRing = (size_t)kStages * kStage;
  static constexpr int kPad = 32 * 9;  // floats per warp: 32 rows x 8 columns, for unaligned outputs
  static constexpr size_t kSmem = kRing + kEpiWarps * kPad * 4 + 1024;
  static constexpr int kCpt = TN / 2;
  static constexpr int kGroups = TN / 8;  // groups of 8 columns, the unit of the exchange
  static_assert((size_t)(kGroups + kMaxSplit) * 8 * kF8Block * 4 <= kRing, "the exchange reuses the ring");
};

template <int TN>
__global__ void __launch_bounds__(Wide<TN>::kThreads, 1) f8_wide_kernel(const __grid_constant__ CUtensorMap tm_x,
                                                                        const __grid_constant__ F8Args a) {
  using C = Wide<TN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* pad = reinterpret_cast<float*>(smem + C::kRing);
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
  if (warp == C::kEpiWarps + 1) tmem_alloc(&tmem_slot, C::kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_wait();

  if (warp >= C::kEpiWarps) {
    if (C::kShift) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == C::kEpiWarps && lane == 0) {
      int it = 0;
      for (int tile = first; tile < total && !failed; tile += stride) {
        const int nt = tile % a.ntiles, rt = tile / a.ntiles;
        const int wt = nt * kTiles, have = min(kTiles, p.m.tiles() - wt);
        for (int b = b0; b < b0 + nb; b++, it++) {
          const int st = it % C::kStages;
          if (it >= C::kStages && !role_wait(&empty[st], ((it / C::kStages) - 1) & 1, &failed)) break;
          mbar_expect_tx(&full[st], kTile * (1 + have));
          uint8_t* at = smem + (size_t)st * C::kStage;
          tma_load_2d(at, &tm_x, b * kF8Block, rt * kF8Block, &full[st]);
          for (int j = 0; j < have; j++)
            bulk_g2s(at + kTile * (1 + j), p.m.w + ((int64_t)(wt + j) * a.kblocks + b) * kF8TileBytes, kTile, &full[st]);
        }
      }
      pdl_launch();
      drain_loads(full, it, C::kStages);
    } else if (warp == C::kEpiWarps + 1 && lane == 0) {
      constexpr uint32_t idesc = idesc_e4m3(kF8Block, TN);
      int it = 0;
      for (int tile = first; tile < total && !failed; tile += stride)
        for (int b = 0; b < nb; b++, it++) {
          const int st = it % C::kStages, buf = it % C::kBufs;
          if (it >= C::kBufs && !role_wait(&tempty[buf], ((it / C::kBufs) - 1) & 1, &failed)) break;
          if (!role_wait(&full[st], (it / C::kStages) & 1, &failed)) break;
          tc_fence_after();
          const uint32_t xa = smem_addr(smem + (size_t)st * C::kStage), wa = xa + kTile;
#pragma unroll
          for (int k = 0; k < 4; k++)
            umma_f8(tmem + buf * TN, sw128_desc(xa + k * 32), sw128_desc(wa + k * 32), idesc, k != 0);
          umma_commit(&empty[st]);
          umma_commit(&tfull[buf]);
        }
      if (failed) drain_mma(&gone);
    }
    if (S > 1) {
      __syncwarp();
      cluster_sync();  // the epilogue warps' two barriers count every warp
      cluster_sync();
    }
  } else {
    if (C::kShift) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int half = warp >> 2, row_l = (warp & 3) * 32 + lane;
    const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16) + half * C::kCpt;
    const bool bf16 = p.out_bf16;
    // 16-byte stores: a row's groups of 8 columns start on 16 bytes.
    const bool aligned = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.out_stride % (bf16 ? 8 : 4) == 0;
    float* my = pad + warp * C::kPad;
    // Columns [n, n + 8) of row r, held by the warp's lanes for 32 consecutive rows.
    auto put8 = [&](int64_t r, int n, float (&y)[8]) {
      if (n >= p.m.n) return;
      if (p.m.bias) {
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = y[j] + (n + j < p.m.n ? p.m.bias[n + j] : 0.f);
      }
      if (aligned && n + 8 <= p.m.n) {
        if (r >= p.rows) return;
        if (bf16) {
          __nv_bfloat162 h[4];
#pragma unroll
          for (int j = 0; j < 4; j++) h[j] = __floats2bfloat162_rn(y[2 * j], y[2 * j + 1]);
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + r * p.out_stride + n) = *reinterpret_cast<uint4*>(h);
        } else {
          float4* o = reinterpret_cast<float4*>(static_cast<float*>(p.out) + r * p.out_stride + n);
          o[0] = make_float4(y[0], y[1], y[2], y[3]);
          o[1] = make_float4(y[4], y[5], y[6], y[7]);
        }
        return;
      }
#pragma unroll
      for (int j = 0; j < 8; j++) my[lane * 9 + j] = y[j];
      __syncwarp();
      const int c = lane & 7;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int rr = j * 4 + (lane >> 3);
        const int64_t at = r - lane + rr;
        if (at < p.rows && n + c < p.m.n) {
          if (bf16)
            static_cast<__nv_bfloat16*>(p.out)[at * p.out_stride + n + c] = __float2bfloat16_rn(my[rr * 9 + c]);
          else
            static_cast<float*>(p.out)[at * p.out_stride + n + c] = my[rr * 9 + c];
        }
      }
      __syncwarp();
    };
    int it = 0;
    for (int tile = first; tile < total; tile += stride) {
      const int nt = tile % a.ntiles, rt = tile / a.ntiles;
      const int64_t r = (int64_t)rt * kF8Block + row_l;
      const int wt = nt * kTiles + (kTiles > 1 ? half : 0);
      const bool live = r < p.rows && wt < p.m.tiles();
      const float* xs = p.scales + (int64_t)b0 * p.scale_stride + (live ? r : 0);
      const float* ws = p.m.scales + (int64_t)(live ? wt : 0) * a.kblocks + b0;
      auto scale_at = [&](int b) { return live && b < nb ? xs[(int64_t)b * p.scale_stride] * ws[b] : 0.f; };
      float acc[C::kCpt];
#pragma unroll
      for (int i = 0; i < C::kCpt; i++) acc[i] = 0.f;
      float s[4];
#pragma unroll
      for (int j = 0; j < 4; j++) s[j] = scale_at(j);
      bool ok = true;
      for (int b1 = 0; b1 < nb && ok; b1 += 4) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (b1 + j >= nb || !ok) break;
          const int buf = it % C::kBufs;
          ok = role_wait(&tfull[buf], (it / C::kBufs) & 1, &failed);
          if (!ok) break;
          __syncwarp();
          tc_fence_after();
          const float sc = s[j];
          s[j] = scale_at(b1 + j + 4);
          uint32_t t[16];
#pragma unroll
          for (int c = 0; c < C::kCpt; c += 16) {
            tmem_ld16_async(trow + buf * TN + c, t);
            tmem_wait(t);
#pragma unroll
            for (int e = 0; e < 16; e++) acc[c + e] = fmaf(__uint_as_float(t[e]), sc, acc[c + e]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tempty[buf]);
          it++;
        }
      }
      if (S == 1) {
        if (ok) {
#pragma unroll
          for (int c = 0; c < C::kCpt; c += 8) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = acc[c + e];
            put8(r, nt * TN + half * C::kCpt + c, y);
          }
        } else {
          break;
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
          dsmem_st4(at, acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
          dsmem_st4(at + kF8Block * 16, acc[c + 4], acc[c + 5], acc[c + 6], acc[c + 7]);
        }
        cluster_sync();
        const int g0 = rank * G / S, g1 = (rank + 1) * G / S;
        for (int g = g0 + half; g < g1; g += 2) {
          float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          for (int q = 0; q < S; q++) {
            const float4* src = reinterpret_cast<const float4*>(recv) + ((size_t)q * most + (g - g0)) * 2 * kF8Block + row_l;
            const float4 u = src[0], v = src[kF8Block];
            y[0] += u.x; y[1] += u.y; y[2] += u.z; y[3] += u.w;
            y[4] += v.x; y[5] += v.y; y[6] += v.z; y[7] += v.w;
          }
          put8(r, nt * TN + g * 8, y);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && failed && p.err) atomicExch(p.err, 2);
  if (warp == C::kEpiWarps + 1) tmem_free(tmem, C::kCols);
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
