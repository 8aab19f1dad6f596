// f8.cu — e4m3 rows with a scale per 128 columns: the norm that writes them and the product
// that reads them.
#include <algorithm>
#include <cuda_fp8.h>
#include <memory>
#include <string>

#include "common.cuh"
#include "entry.h"
#include "f8.cuh"
#include "sm100.cuh"

namespace svl {
namespace {

__device__ __forceinline__ uint8_t to_e4m3(float v) {
  return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}
// Maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Eight consecutive values of a row of the stream as f32; `have` of them exist.
template <class T>
__device__ __forceinline__ void load8(const T* p, int have, bool wide, float (&v)[8]) {
  if (wide && have == 8) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      v[0] = bf16_lo(a.x); v[1] = bf16_hi(a.x); v[2] = bf16_lo(a.y); v[3] = bf16_hi(a.y);
      v[4] = bf16_lo(a.z); v[5] = bf16_hi(a.z); v[6] = bf16_lo(a.w); v[7] = bf16_hi(a.w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = j < have ? (float)p[j] : 0.f;
  }
}
template <class T>
__device__ __forceinline__ void store8(T* p, int have, bool wide, const float (&v)[8]) {
  if (wide && have == 8) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      __nv_bfloat162 h[4];
#pragma unroll
      for (int j = 0; j < 4; j++) h[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (j < have) p[j] = sizeof(T) == 4 ? (T)v[j] : (T)__float2bfloat16_rn(v[j]);
  }
}

// The sum of v over a row's threads (a multiple of 32, threadIdx.x of them): warp sums, then the
// warps' sums in order. `red` belongs to the row; its barrier is 1 + threadIdx.y.
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = warp_sum(v);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(1 + threadIdx.y), "r"(blockDim.x) : "memory");
  float s = red[0];
  for (int w = 1; w < warps; w++) s += red[w];
  return s;
}

// A row's threads (threadIdx.x) hold the whole row in registers, I pieces of 8 values each, so x
// and the residual are read once: bound by HBM. 16 consecutive threads hold a block of 128
// columns, whose maximum takes four shuffles. Short rows share a CTA (threadIdx.y).
template <class T, int I>
__global__ void __launch_bounds__(I == 4 ? 1024 : 512) norm_f8_kernel(const NormF8Params p) {
  __shared__ float red_sm[2][32];
  const int64_t r = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  pdl_launch();
  pdl_wait();
  if (r >= p.rows) return;
  // A CTA's rows use disjoint parts of red (blockDim.x / 32 * blockDim.y <= 32 warps).
  float* red = red_sm[0] + threadIdx.y * (blockDim.x >> 5);
  float* red2 = red_sm[1] + threadIdx.y * (blockDim.x >> 5);
  const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
  const T* res = p.residual ? static_cast<const T*>(p.residual) + r * p.residual_stride : nullptr;
  T* sum = p.sum ? static_cast<T*>(p.sum) + r * p.sum_stride : nullptr;
  const bool xw = reinterpret_cast<uintptr_t>(x) % 16 == 0, rw = reinterpret_cast<uintptr_t>(res) % 16 == 0,
             sw = reinterpret_cast<uintptr_t>(sum) % 16 == 0;
  const bool ww = reinterpret_cast<uintptr_t>(p.weight) % 16 == 0, bw = reinterpret_cast<uintptr_t>(p.bias) % 16 == 0;
  float h[I][8];
#pragma unroll
  for (int i = 0; i < I; i++) {
    const int c = (threadIdx.x + i * blockDim.x) * 8;
    load8(x + c, min(8, p.k - c), xw, h[i]);
  }
  if (res) {
#pragma unroll
    for (int i = 0; i < I; i++) {
      const int c = (threadIdx.x + i * blockDim.x) * 8;
      float a[8];
      load8(res + c, min(8, p.k - c), rw, a);
#pragma unroll
      for (int j = 0; j < 8; j++) h[i][j] = sizeof(T) == 4 ? h[i][j] + a[j] : round_bf16(h[i][j] + a[j]);
    }
  }
  if (sum) {
#pragma unroll
    for (int i = 0; i < I; i++) {
      const int c = (threadIdx.x + i * blockDim.x) * 8;
      store8(sum + c, min(8, p.k - c), sw, h[i]);
    }
  }
  if (p.norm != NORM_NONE) {
    float a = 0.f;
    if (p.norm == NORM_LAYER) {
#pragma unroll
      for (int i = 0; i < I; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) a += h[i][j];
      const float mean = row_sum(a, red2) / (float)p.k;
#pragma unroll
      for (int i = 0; i < I; i++) {
        const int c = (threadIdx.x + i * blockDim.x) * 8;
#pragma unroll
        for (int j = 0; j < 8; j++) h[i][j] = c + j < p.k ? h[i][j] - mean : 0.f;
      }
      a = 0.f;
    }
#pragma unroll
    for (int i = 0; i < I; i++)
#pragma unroll
      for (int j = 0; j < 8; j++) a = fmaf(h[i][j], h[i][j], a);
    const float rstd = 1.0f / sqrtf(row_sum(a, red) / (float)p.k + p.eps);
#pragma unroll
    for (int i = 0; i < I; i++) {
      const int c = (threadIdx.x + i * blockDim.x) * 8, have = min(8, p.k - c);
#pragma unroll
      for (int j = 0; j < 8; j++) h[i][j] = h[i][j] * rstd;
      float a8[8];
      if (p.weight) {
        load8(p.weight + c, have, ww, a8);
#pragma unroll
        for (int j = 0; j < 8; j++) h[i][j] = h[i][j] * a8[j];
      }
      if (p.bias && p.norm == NORM_LAYER) {
        load8(p.bias + c, have, bw, a8);
#pragma unroll
        for (int j = 0; j < 8; j++) h[i][j] = h[i][j] + a8[j];
      }
    }
  }
  uint8_t* q = p.q + r * p.q_stride;
#pragma unroll
  for (int i = 0; i < I; i++) {
    const int c = (threadIdx.x + i * blockDim.x) * 8, have = p.k - c;
    float top = kF8Tiny;
#pragma unroll
    for (int j = 0; j < 8; j++) top = max_nan(top, j < have ? fabsf(h[i][j]) : 0.f);
#pragma unroll
    for (int o = 8; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float inv = __fdiv_rn(kF8Max, top);
    if (have >= 8) {
      uint2 v;
      uint16_t* e = reinterpret_cast<uint16_t*>(&v);
#pragma unroll
      for (int j = 0; j < 4; j++)
        e[j] = __nv_cvt_float2_to_fp8x2(make_float2(h[i][2 * j] * inv, h[i][2 * j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
      *reinterpret_cast<uint2*>(q + c) = v;
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (j < have) q[c + j] = to_e4m3(h[i][j] * inv);
    }
    if ((threadIdx.x & 15) == 0 && have > 0)
      p.scales[(int64_t)(c / kF8Block) * p.scale_stride + r] = __fdiv_rn(top, kF8Max);
  }
}

// Byte of (row, col) in the packed image.
__host__ __device__ __forceinline__ int64_t packed_at(int row, int col, int kblocks) {
  const int tr = row % kF8Block, tc = col % kF8Block;
  return ((int64_t)(row / kF8Block) * kblocks + col / kF8Block) * kF8TileBytes + tr * kF8Block +
         (((tc >> 4) ^ (tr & 7)) << 4) + (tc & 15);
}

__global__ void f8_pack_kernel(const uint8_t* src, int64_t stride, int n, int k, int kblocks, uint8_t* dst) {
  const int64_t total = (int64_t)n * k;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int r = (int)(i / k), c = (int)(i % k);
    dst[packed_at(r, c, kblocks)] = src[(int64_t)r * stride + c];
  }
}

// One CTA per 128 x 128 block: its largest magnitude, its scale, its e4m3 values.
__global__ void __launch_bounds__(256) f8_quantise_kernel(const float* src, int n, int k, int half, uint8_t* dst,
                                                          float* scales) {
  __shared__ float red[8];
  const int kb = blockIdx.x, tile = blockIdx.y, kblocks = gridDim.x;
  auto value = [&](int i) -> float {
    const int r = tile * kF8Block + i / kF8Block, c = kb * kF8Block + i % kF8Block;
    if (r >= n || c >= k) return 0.f;
    const int sr = half ? (r & 1) * half + (r >> 1) : r;
    return src[(int64_t)sr * k + c];
  };
  float top = 0.f;
  for (int i = threadIdx.x; i < kF8Block * kF8Block; i += 256) top = max_nan(top, fabsf(value(i)));
  for (int o = 16; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  top = kF8Tiny;
  for (int w = 0; w < 8; w++) top = max_nan(top, red[w]);
  const float inv = kF8Max / top;
  for (int i = threadIdx.x; i < kF8Block * kF8Block; i += 256) {
    const int r = tile * kF8Block + i / kF8Block, c = kb * kF8Block + i % kF8Block;
    if (r < n && c < k) dst[packed_at(r, c, kblocks)] = to_e4m3(value(i) * inv);
  }
  if (threadIdx.x == 0) scales[(int64_t)tile * kblocks + kb] = top / kF8Max;
}

}  // namespace

// Pieces per thread: one up to 4,096 columns (512 threads), then two and four, so that a CTA stays
// small enough for several per SM; rows below 2,048 columns share CTAs of 256 threads.
void launch_norm_f8(const NormF8Params& p, cudaStream_t s) {
  const int pieces = (p.k + 7) / 8;
  const int per = pieces <= 512 ? 1 : pieces <= 1024 ? 2 : 4;
  const int threads = ((pieces + per - 1) / per + 31) / 32 * 32;
  const int share = (int)std::min<int64_t>(std::max(1, 256 / threads), p.rows);
  const int64_t grid = (p.rows + share - 1) / share;
  if (grid > INT32_MAX) throw Error(SVL_ERR_UNSUPPORTED, "too many rows");
  auto kernel = p.bf16 ? (per == 1 ? norm_f8_kernel<__nv_bfloat16, 1> : per == 2 ? norm_f8_kernel<__nv_bfloat16, 2> : norm_f8_kernel<__nv_bfloat16, 4>)
                       : (per == 1 ? norm_f8_kernel<float, 1> : per == 2 ? norm_f8_kernel<float, 2> : norm_f8_kernel<float, 4>);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads, share);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  check_cuda(cudaLaunchKernelEx(&cfg, kernel, p), "norm launch");
}

void launch_f8_pack(const uint8_t* src, int64_t stride, int n, int k, uint8_t* dst, cudaStream_t s) {
  f8_pack_kernel<<<148 * 8, 256, 0, s>>>(src, stride, n, k, (k + kF8Block - 1) / kF8Block, dst);
  check_cuda(cudaGetLastError(), "pack launch");
}

void launch_f8_quantise(const float* src, int n, int k, int interleave_half, uint8_t* dst, float* scales,
                        cudaStream_t s) {
  const dim3 grid((k + kF8Block - 1) / kF8Block, (n + kF8Block - 1) / kF8Block);
  f8_quantise_kernel<<<grid, 256, 0, s>>>(src, n, k, interleave_half, dst, scales);
  check_cuda(cudaGetLastError(), "quantise launch");
}

}  // namespace svl

using svl::entry;
using svl::Error;
using svl::OnDevice;
using svl::require;

struct svl_f8_linear {
  int device = 0;
  svl::DevBuf w, scales, bias, err;
  svl::F8Matrix m;
  // Allocates the zeroed image of an n x k matrix on the current device.
  void alloc(int n, int k, bool with_bias, cudaStream_t st) {
    m.n = n;
    m.k = k;
    w.alloc((size_t)m.tiles() * m.kblocks() * svl::kF8TileBytes);
    scales.alloc((size_t)m.tiles() * m.kblocks() * 4);
    err.alloc(4);
    if (with_bias) bias.alloc((size_t)n * 4);
    svl::check_cuda(cudaMemsetAsync(w.p, 0, w.bytes, st), "memset");
    svl::check_cuda(cudaMemsetAsync(err.p, 0, 4, st), "memset");
    m.w = w.as<uint8_t>();
    m.scales = scales.as<float>();
    m.bias = bias.as<float>();
  }
};

namespace {

// Rows and columns of a matrix whose index arithmetic stays in 32 bits per tile row.
void check_sizes(int32_t n, int32_t k) {
  require(n >= 1 && k >= 1, "n and k must be positive", SVL_ERR_CONFIG);
  require(n <= (1 << 24) && k <= (1 << 20), "n above 2^24 or k above 2^20", SVL_ERR_UNSUPPORTED);
}

void check_device(int32_t device) {
  int count = 0;
  svl::check_cuda(cudaGetDeviceCount(&count), "cudaGetDeviceCount");
  require(device >= 0 && device < count, "no such CUDA device", SVL_ERR_CUDA);
}

}  // namespace

extern "C" {

SVL_API svl_status svl_add_norm_f8_device(int32_t device, int64_t rows, int32_t k, int32_t dtype, const void* d_x,
                                          int64_t x_stride, const void* d_residual, int64_t residual_stride,
                                          int32_t norm_kind, const float* d_weight, const float* d_bias, float eps,
                                          void* d_sum, int64_t sum_stride, uint8_t* d_q, int64_t q_stride,
                                          float* d_scales, int64_t scale_stride, void* cuda_stream) {
  return entry([&] {
    require(rows >= 0, "negative row count");
    require(k >= 1, "k must be positive");
    require(k <= svl::kF8MaxCols, "k above 32768", SVL_ERR_UNSUPPORTED);
    require(dtype == SVL_DT_F32 || dtype == SVL_DT_BF16, "dtype must be f32 or bf16");
    require(norm_kind >= -1 && norm_kind <= SVL_NORM_RMS, "unknown norm kind");
    if (rows == 0) return;
    require(d_x && d_q && d_scales, "null argument");
    require(x_stride >= k && (!d_residual || residual_stride >= k) && (!d_sum || sum_stride >= k),
            "a row stride is below k");
    require(q_stride >= k && q_stride % 16 == 0, "q_stride must be a multiple of 16, at least k");
    require(reinterpret_cast<uintptr_t>(d_q) % 16 == 0, "d_q must be 16-byte aligned");
    require(scale_stride >= rows, "scale_stride is below the row count");
    require(eps >= 0.f, "eps must not be negative");
    OnDevice on(device);
    svl::NormF8Params p{};
    p.x = d_x;
    p.x_stride = x_stride;
    p.residual = d_residual;
    p.residual_stride = residual_stride;
    p.weight = d_weight;
    p.bias = d_bias;
    p.eps = eps;
    p.norm = norm_kind < 0 ? svl::NORM_NONE : norm_kind == SVL_NORM_RMS ? svl::NORM_RMS : svl::NORM_LAYER;
    p.bf16 = dtype == SVL_DT_BF16;
    p.rows = rows;
    p.k = k;
    p.sum = d_sum;
    p.sum_stride = sum_stride;
    p.q = d_q;
    p.q_stride = q_stride;
    p.scales = d_scales;
    p.scale_stride = scale_stride;
    svl::launch_norm_f8(p, static_cast<cudaStream_t>(cuda_stream));
  });
}

SVL_API svl_status svl_f8_linear_create(int32_t n, int32_t k, const svl_tensor_view* tensors, int32_t n_tensors,
                                        int32_t device, svl_f8_linear** out) {
  return entry([&] {
    require(out && (tensors || n_tensors == 0), "null argument");
    *out = nullptr;
    check_sizes(n, k);
    const svl_tensor_view *weight = nullptr, *bias = nullptr;
    for (int i = 0; i < n_tensors; i++) {
      if (!tensors[i].name) continue;
      if (std::string("weight") == tensors[i].name) weight = &tensors[i];
      if (std::string("bias") == tensors[i].name) bias = &tensors[i];
    }
    require(weight && weight->data, "missing tensor weight", SVL_ERR_CONFIG);
    require(weight->numel == (int64_t)n * k, "tensor weight does not have n * k elements", SVL_ERR_CONFIG);
    require(!bias || (bias->data && bias->numel == n), "tensor bias does not have n elements", SVL_ERR_CONFIG);
    check_device(device);
    OnDevice on(device);
    auto L = std::make_unique<svl_f8_linear>();
    L->device = device;
    cudaStream_t st = nullptr;
    L->alloc(n, k, bias != nullptr, st);
    svl::DevBuf staging;
    staging.alloc((size_t)n * k * 4);
    svl::check_cuda(cudaMemcpyAsync(staging.p, weight->data, staging.bytes, cudaMemcpyHostToDevice, st), "upload");
    svl::launch_f8_quantise(staging.as<float>(), n, k, 0, L->w.as<uint8_t>(), L->scales.as<float>(), st);
    if (bias) svl::check_cuda(cudaMemcpyAsync(L->bias.p, bias->data, (size_t)n * 4, cudaMemcpyHostToDevice, st), "upload");
    svl::check_cuda(cudaStreamSynchronize(st), "create");
    *out = L.release();
  });
}

SVL_API svl_status svl_f8_linear_create_device(int32_t n, int32_t k, const uint8_t* d_weight, int64_t weight_stride,
                                               const float* d_scales, const float* d_bias, int32_t device,
                                               void* cuda_stream, svl_f8_linear** out) {
  return entry([&] {
    require(out && d_weight && d_scales, "null argument");
    *out = nullptr;
    check_sizes(n, k);
    require(weight_stride >= k, "weight_stride is below k");
    check_device(device);
    OnDevice on(device);
    auto L = std::make_unique<svl_f8_linear>();
    L->device = device;
    cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    L->alloc(n, k, d_bias != nullptr, st);
    svl::launch_f8_pack(d_weight, weight_stride, n, k, L->w.as<uint8_t>(), st);
    svl::check_cuda(cudaMemcpyAsync(L->scales.p, d_scales, L->scales.bytes, cudaMemcpyDeviceToDevice, st), "copy");
    if (d_bias) svl::check_cuda(cudaMemcpyAsync(L->bias.p, d_bias, (size_t)n * 4, cudaMemcpyDeviceToDevice, st), "copy");
    svl::check_cuda(cudaStreamSynchronize(st), "create");
    *out = L.release();
  });
}

SVL_API void svl_f8_linear_destroy(svl_f8_linear* linear) {
  if (!linear) return;
  entry([&] {
    OnDevice on(linear->device);
    cudaDeviceSynchronize();
    delete linear;
  });
}

SVL_API svl_status svl_f8_linear_device(svl_f8_linear* linear, int64_t rows, const uint8_t* d_q, int64_t q_stride,
                                        const float* d_scales, int64_t scale_stride, int32_t out_dtype, void* d_out,
                                        int64_t out_stride, void* cuda_stream) {
  return entry([&] {
    require(linear, "null argument");
    require(rows >= 0, "negative row count");
    require(rows < (1LL << 31) - 1024, "too many rows", SVL_ERR_UNSUPPORTED);
    require(out_dtype == SVL_DT_F32 || out_dtype == SVL_DT_BF16, "out_dtype must be f32 or bf16");
    if (rows == 0) return;
    require(d_q && d_scales && d_out, "null argument");
    require(q_stride >= linear->m.k && q_stride % 16 == 0, "q_stride must be a multiple of 16, at least k");
    require(reinterpret_cast<uintptr_t>(d_q) % 16 == 0, "d_q must be 16-byte aligned");
    require(scale_stride >= rows, "scale_stride is below the row count");
    require(out_stride >= linear->m.n, "out_stride is below n");
    OnDevice on(linear->device);
    svl::F8GemmParams p{};
    p.m = linear->m;
    p.q = d_q;
    p.q_stride = q_stride;
    p.scales = d_scales;
    p.scale_stride = scale_stride;
    p.rows = rows;
    p.out = d_out;
    p.out_stride = out_stride;
    p.out_bf16 = out_dtype == SVL_DT_BF16;
    p.err = linear->err.as<int>();
    svl::launch_f8_gemm(p, static_cast<cudaStream_t>(cuda_stream));
  });
}

SVL_API svl_status svl_f8_linear_error(svl_f8_linear* linear) {
  return entry([&] {
    require(linear, "null argument");
    OnDevice on(linear->device);
    svl::check_cuda(cudaDeviceSynchronize(), "sync");
    int e = 0;
    svl::check_cuda(cudaMemcpy(&e, linear->err.p, 4, cudaMemcpyDeviceToHost), "d2h");
    if (!e) return;
    svl::check_cuda(cudaMemset(linear->err.p, 0, 4), "memset");
    svl::check_cuda(cudaDeviceSynchronize(), "sync");
    throw Error(SVL_ERR_TIMEOUT, "a bounded device-side wait ran out (code " + std::to_string(e) + ")");
  });
}

}  // extern "C"
