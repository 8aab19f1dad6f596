// f8.cuh — e4m3 rows and matrices with f32 scales per block of 128 (host/device shared).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace svl {

constexpr int kF8Block = 128;          // columns (and matrix rows) that share a scale
constexpr int kF8MaxCols = 32768;      // longest row of the norm (it is held on chip)
constexpr float kF8Max = 448.0f;       // largest e4m3 value
constexpr float kF8Tiny = 0x1p-100f;   // least block maximum: keeps 448 / max finite

// Rows to quantise; see svl_add_norm_f8_device. Strides in elements.
struct NormF8Params {
  const void* x;
  int64_t x_stride;
  const void* residual;
  int64_t residual_stride;
  const float* weight;
  const float* bias;
  float eps;
  int norm;   // NormKind
  int bf16;   // x, residual and sum are bf16 (else f32)
  int64_t rows;
  int k;
  void* sum;
  int64_t sum_stride;
  uint8_t* q;
  int64_t q_stride;
  float* scales;
  int64_t scale_stride;
};
void launch_norm_f8(const NormF8Params& p, cudaStream_t s);

// A packed e4m3 matrix. The weights are tiles of 128 rows x 128 columns, 16 KB each, tile
// (t, b) at (t * kblocks + b): row-major 128-byte rows whose 16-byte pieces are permuted
// (piece ^ (row & 7)), the image a 128-byte-swizzled shared-memory operand has, so that a tile
// is one contiguous copy. Rows past n and columns past k are zero.
struct F8Matrix {
  const uint8_t* w = nullptr;
  const float* scales = nullptr;  // [tiles][kblocks]
  const float* bias = nullptr;    // [n] or null
  int n = 0, k = 0;
  __host__ __device__ int tiles() const { return (n + kF8Block - 1) / kF8Block; }
  __host__ __device__ int kblocks() const { return (k + kF8Block - 1) / kF8Block; }
};
constexpr int64_t kF8TileBytes = (int64_t)kF8Block * kF8Block;

// Packs row-major e4m3 rows (stride bytes apart) into a zeroed image.
void launch_f8_pack(const uint8_t* src, int64_t stride, int n, int k, uint8_t* dst, cudaStream_t s);
// Quantises f32 [n][k] into a zeroed image and its scales.
void launch_f8_quantise(const float* src, int n, int k, uint8_t* dst, float* scales, cudaStream_t s);

struct F8GemmParams {
  F8Matrix m;
  const uint8_t* q;
  int64_t q_stride;
  const float* scales;
  int64_t scale_stride;
  int64_t rows;
  void* out;
  int64_t out_stride;
  int out_bf16;
  int* err;  // set to 2 when a bounded wait runs out
};
void launch_f8_gemm(const F8GemmParams& p, cudaStream_t s);

}  // namespace svl
