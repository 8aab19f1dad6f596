// f8.cu — e4m3 rows with a scale per 128 columns: the norm that writes them and the product
// that reads them.
#include <algorithm>
#include <cuda_fp8.h>
#include <memory>
#include <string>

#include "common.cuh"
#include "entry.h"
#include "f8.cuh"

namespace svl {
namespace {

__device__ __forceinline__ float load_stream(const float* p) { return *p; }
__device__ __forceinline__ float load_stream(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_stream(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_stream(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ uint8_t to_e4m3(float v) {
  return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}
// Maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr int kNormThreads = 256;

__device__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < kNormThreads / 32; w++) s += red[w];
  return s;
}

// One CTA per row, the row in shared memory.
template <class T>
__global__ void __launch_bounds__(kNormThreads) norm_f8_kernel(const NormF8Params p) {
  extern __shared__ float row[];
  __shared__ float red[kNormThreads / 32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
    const T* res = p.residual ? static_cast<const T*>(p.residual) + r * p.residual_stride : nullptr;
    T* sum = p.sum ? static_cast<T*>(p.sum) + r * p.sum_stride : nullptr;
    float a = 0.f;
    for (int i = t; i < p.k; i += kNormThreads) {
      float h = load_stream(x + i);
      if (res) h = h + load_stream(res + i);
      if (sizeof(T) == 2) h = round_bf16(h);
      if (sum) store_stream(sum + i, h);
      row[i] = h;
      a += p.norm == NORM_LAYER ? h : h * h;
    }
    float mean = 0.f, rstd = 1.f;
    if (p.norm != NORM_NONE) {
      a = block_sum(a, red) / (float)p.k;
      if (p.norm == NORM_LAYER) {
        mean = a;
        float c = 0.f;
        for (int i = t; i < p.k; i += kNormThreads) c += (row[i] - mean) * (row[i] - mean);
        a = block_sum(c, red) / (float)p.k;
      }
      rstd = 1.0f / sqrtf(a + p.eps);
    }
    __syncthreads();
    for (int b = warp; b * kF8Block < p.k; b += kNormThreads / 32) {
      float y[4], top = 0.f;
      for (int j = 0; j < 4; j++) {
        const int i = b * kF8Block + j * 32 + lane;
        y[j] = 0.f;
        if (i < p.k) {
          y[j] = row[i];
          if (p.norm != NORM_NONE) {
            y[j] = (y[j] - mean) * rstd;
            if (p.weight) y[j] = y[j] * p.weight[i];
            if (p.bias && p.norm == NORM_LAYER) y[j] = y[j] + p.bias[i];
          }
        }
        top = max_nan(top, fabsf(y[j]));
      }
      for (int o = 16; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
      top = max_nan(top, kF8Tiny);
      const float inv = kF8Max / top;
      for (int j = 0; j < 4; j++) {
        const int i = b * kF8Block + j * 32 + lane;
        if (i < p.k) p.q[r * p.q_stride + i] = to_e4m3(y[j] * inv);
      }
      if (lane == 0) p.scales[(int64_t)b * p.scale_stride + r] = top / kF8Max;
    }
    __syncthreads();
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

void launch_norm_f8(const NormF8Params& p, cudaStream_t s) {
  const int grid = (int)std::min<int64_t>(p.rows, 148 * 64);
  const size_t smem = (size_t)p.k * 4;
  auto kernel = p.bf16 ? norm_f8_kernel<__nv_bfloat16> : norm_f8_kernel<float>;
  if (smem > 48 * 1024)
    check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "norm");
  kernel<<<grid, kNormThreads, smem, s>>>(p);
  check_cuda(cudaGetLastError(), "norm launch");
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
