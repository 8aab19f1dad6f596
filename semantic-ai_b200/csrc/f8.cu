// f8.cu — e4m3 rows with a scale per 128 columns: the norm that writes them and the product
// that reads them.
#include <algorithm>
#include <memory>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "entry.h"
#include "f8.cuh"
#include "sm100.cuh"
#include "tcgen05.cuh"

namespace svl {
namespace {

// V consecutive values of a row as they lie in memory; `have` of them exist. `wide`: they start on 16
// bytes, `wider`: on 32.
template <class T, int V>
struct Raw {
  uint4 v[V * sizeof(T) / 16];
};
// 32 bytes per lane, 32-byte aligned. Two loads of 16 with 16 between the lanes' would each touch
// twice the lines.
__device__ __forceinline__ void load32(const void* p, uint4& a, uint4& b) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
               : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const uint4& a, const uint4& b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w),
               "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}
template <class T, int V>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p, int have, bool wide, bool wider) {
  constexpr int N = V * sizeof(T) / 16;
  Raw<T, V> r;
  if (N % 2 == 0 && wider && have >= V) {
#pragma unroll
    for (int i = 0; i + 1 < N; i += 2) load32(reinterpret_cast<const uint4*>(p) + i, r.v[i], r.v[i + 1]);
  } else if (wide && have >= V) {
#pragma unroll
    for (int i = 0; i < (int)(V * sizeof(T) / 16); i++) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    T* e = reinterpret_cast<T*>(r.v);
#pragma unroll
    for (int j = 0; j < V; j++) e[j] = j < have ? p[j] : T(0.f);
  }
  return r;
}
template <class T, int V>
__device__ __forceinline__ void store_raw(T* p, const Raw<T, V>& r, int have, bool wide, bool wider) {
  constexpr int N = V * sizeof(T) / 16;
  if (N % 2 == 0 && wider && have >= V) {
#pragma unroll
    for (int i = 0; i + 1 < N; i += 2) store32(reinterpret_cast<uint4*>(p) + i, r.v[i], r.v[i + 1]);
  } else if (wide && have >= V) {
#pragma unroll
    for (int i = 0; i < (int)(V * sizeof(T) / 16); i++) reinterpret_cast<uint4*>(p)[i] = r.v[i];
  } else {
    const T* e = reinterpret_cast<const T*>(r.v);
#pragma unroll
    for (int j = 0; j < V; j++)
      if (j < have) p[j] = e[j];
  }
}
template <class T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& r, float (&v)[V]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(r.v);
#pragma unroll
  for (int j = 0; j < V; j++) v[j] = sizeof(T) == 4 ? __uint_as_float(w[j]) : j & 1 ? bf16_hi(w[j / 2]) : bf16_lo(w[j / 2]);
}
// Rounded to the stream's type.
template <class T, int V>
__device__ __forceinline__ Raw<T, V> pack(const float (&v)[V]) {
  Raw<T, V> r;
  uint32_t* w = reinterpret_cast<uint32_t*>(r.v);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < V; j++) w[j] = __float_as_uint(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[j], v[j + 1]);
      w[j / 2] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return r;
}

// Rows that start anywhere. A thread's V values are read in the aligned 16-byte pieces that hold at
// least one of them (one more than V values take), as they come; `shifted` then cuts the values
// out. (Value by value, every load of a warp would touch a sector per lane: 16,384
// x 2,561 with a residual bf16 took 254 us, 111 this way.)
template <class T, int V>
struct RawOdd {
  uint4 v[V * sizeof(T) / 16 + 1];
};
template <class T, int V>
__device__ __forceinline__ RawOdd<T, V> load_odd(const T* p, int have) {
  constexpr int N = V * sizeof(T) / 16;
  const int off = (int)(reinterpret_cast<uintptr_t>(p) & 15);
  const uint4* base = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) - off);
  RawOdd<T, V> r;
#pragma unroll
  for (int i = 0; i <= N; i++) {
    r.v[i] = make_uint4(0, 0, 0, 0);
    if (have > 0 && i * 16 - off < have * (int)sizeof(T) && (i < N || off)) r.v[i] = base[i];
  }
  return r;
}
// Words [off / 4, off / 4 + M) of w, off bytes in (a multiple of 4 without Halves).
template <bool Halves, int M, int W>
__device__ __forceinline__ void shift_words(const uint32_t (&w)[W], int off, uint32_t (&to)[M]) {
  static_assert(W >= M + 4, "words past the last shifted one");
  uint32_t a[M + 2], b[M + 1];
#pragma unroll
  for (int i = 0; i < M + 2; i++) a[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < M + 1; i++) b[i] = off & 4 ? a[i + 1] : a[i];
#pragma unroll
  for (int i = 0; i < M; i++) to[i] = Halves ? __funnelshift_r(b[i], b[i + 1], (off & 3) * 8) : b[i];
}
template <class T, int V>
__device__ __forceinline__ Raw<T, V> shifted(const RawOdd<T, V>& r, int off, int have) {
  constexpr int M = V * sizeof(T) / 4;
  uint32_t w[M + 4], to[M];
#pragma unroll
  for (int i = 0; i < M / 4 + 1; i++) {
    w[4 * i] = r.v[i].x;
    w[4 * i + 1] = r.v[i].y;
    w[4 * i + 2] = r.v[i].z;
    w[4 * i + 3] = r.v[i].w;
  }
  shift_words<sizeof(T) == 2>(w, off, to);
  if (have < V) {  // what follows the row
#pragma unroll
    for (int j = 0; j < V; j++) {
      if constexpr (sizeof(T) == 4) {
        if (j >= have) to[j] = 0;
      } else {
        if (j >= have) to[j / 2] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
      }
    }
  }
  Raw<T, V> out;
#pragma unroll
  for (int i = 0; i < M / 4; i++) out.v[i] = make_uint4(to[4 * i], to[4 * i + 1], to[4 * i + 2], to[4 * i + 3]);
  return out;
}
// The counterpart for stores, by a whole warp whose lanes hold consecutive values: a lane stores the
// aligned pieces that start in its values, the last of them ending with the next lane's first
// values; what belongs to no whole piece of the warp's is stored value by value.
template <class T, int V>
__device__ __forceinline__ void store_odd(T* p, const Raw<T, V>& r, int have) {
  constexpr int N = V * sizeof(T) / 16, M = 4 * N, es = sizeof(T);
  const int lane = threadIdx.x & 31;
  const int head = (int)(-reinterpret_cast<uintptr_t>(p) & 15);  // bytes before the first aligned piece
  uint32_t w[M + 4], to[M];
#pragma unroll
  for (int i = 0; i < N; i++) {
    w[4 * i] = r.v[i].x;
    w[4 * i + 1] = r.v[i].y;
    w[4 * i + 2] = r.v[i].z;
    w[4 * i + 3] = r.v[i].w;
  }
#pragma unroll
  for (int i = 0; i < 4; i++) w[M + i] = __shfl_down_sync(0xffffffffu, w[i], 1);
  shift_words<sizeof(T) == 2>(w, head, to);
  const T* e = reinterpret_cast<const T*>(r.v);
  int from = 0, rest = V;  // the values that are stored one by one: [0, from) and [rest, V)
  if (lane == 0 || head > have * es) from = head / es;
#pragma unroll
  for (int g = 0; g < N; g++) {
    if (head + 16 * g + 16 <= have * es && (g < N - 1 || lane < 31 || head == 0))
      reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p) + head)[g] = make_uint4(to[4 * g], to[4 * g + 1], to[4 * g + 2], to[4 * g + 3]);
    else
      rest = min(rest, (head + 16 * g) / es);
  }
#pragma unroll
  for (int j = 0; j < V; j++)
    if (j < have && (j < from || j >= rest)) p[j] = e[j];
}

// Values v as their quotients v * 448 / top, rounded once to f32 before they become e4m3 (v * RN(448 / top) is
// rounded twice). A value of few bits, a bf16 one, often lies exactly in the middle of two e4m3 values, and twice
// rounded it falls to either side (333 x 5,637 bf16: 508 of 1.9 M values). p is within 2 ulp of the quotient
// m / b (m = v * 7 / 8, exact for bf16; b = top / 512), and p - (p b - m) / b brings it to within 2^-46, so that a
// quotient of few bits comes out as it is. Neither overflows for finite v: |m| <= |v|, and top is at least 2^-100.
// (Signs are such that -0 stays -0.)
template <int V>
__device__ __forceinline__ void quotients(float (&v)[V], float top) {
  const float q = -512.0f / top, c = top * 0x1p-9f;
  const uint64_t r = pair_of(q, q), b = pair_of(c, c);
#pragma unroll
  for (int j = 0; j < V; j += 2) {
    const uint64_t m = mul_pair(pair_of(v[j], v[j + 1]), pair_of(-0.875f, -0.875f));
    uint64_t p = mul_pair(m, r), e = m;
    fma_pair(e, p, b);
    fma_pair(p, e, r);
    v[j] = pair_lo(p);
    v[j + 1] = pair_hi(p);
  }
}
static_assert(kF8Max == 512.0f * 0.875f, "the quotients' factors");

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

// A row's threads (threadIdx.x) hold the whole row in registers, I pieces of V values each (8 f32
// or 16 bf16: 32 bytes), so x and the residual are read once: bound by HBM. 128 / V consecutive
// threads hold a block of 128 columns. Short rows share a CTA (threadIdx.y). With many rows
// a CTA goes through several of them and has the next one's x and residual on their way while it
// works on one, since sums, scales and stores leave the memory idle otherwise.
//
// Measured with a residual: 16,384 x 2,560 bf16 48 us (6.2 TB/s; 59 with loads of 16 bytes, which made
// L1 the bound), 8,192 x 2,048 f32 35 us (6.2 TB/s); 512 x 1,024 layer norm f32 3.8 us; 1 x 2,048 2.1 us.
// Rows of four pieces have up to 1,024 threads and so 64 registers, of which f32 ones spill 212 bytes and
// bf16 ones 164: 4,096 x 10,240 f32 123 us (4.4 TB/s), 2,048 x 20,000 bf16 91 us (3.1 TB/s).
//
// The compiler's choice of registers is left to it but for bf16 rows of one piece. For odd ones it would
// take too few (16,384 x 727: 47 us, 38.5 with all that one CTA may have; aligned rows: 28); for
// aligned ones too many (3,276 x 5,120: 36.5 us with 103, 23.2 with 64).
template <class T, int I, bool Odd>
constexpr int kLeastCtas = sizeof(T) == 2 && I == 1 ? (Odd ? 1 : 2) : 0;

// Odd: x, the residual or the sum has rows that start off 16 bytes.
template <class T, int V, int I, bool Odd>
__global__ void __launch_bounds__(I == 4 ? 1024 : 512, kLeastCtas<T, I, Odd>) norm_f8_kernel(const __grid_constant__ NormF8Params p) {
  __shared__ float red_sm[2][2][32];
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  int64_t r = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  pdl_launch();
  pdl_wait();
  if (r >= p.rows) return;
  const int width = blockDim.x;
  const bool ww = reinterpret_cast<uintptr_t>(p.weight) % 32 == 0, bw = reinterpret_cast<uintptr_t>(p.bias) % 32 == 0;
  auto on32 = [](const void* base, int64_t stride) { return (reinterpret_cast<uintptr_t>(base) | (uint64_t)stride * sizeof(T)) % 32 == 0; };
  const bool x32 = on32(p.x, p.x_stride), r32 = on32(p.residual, p.residual_stride), s32 = on32(p.sum, p.sum_stride);
  // The longest rows leave few registers for it: 4,096 x 10,241 f32 54 us, 65 with; though with a residual 247, 198 with.
  constexpr bool kShift = Odd && I < 4;
  using Piece = typename std::conditional<kShift, RawOdd<T, V>, Raw<T, V>>::type;
  Piece nx[I], nr[I];
  auto load = [&](const void* base, int64_t at, int have, bool wider) {
    const T* from = static_cast<const T*>(base) + at;
    if constexpr (kShift)
      return load_odd<T, V>(from, have);
    else
      return load_raw<T, V>(from, have, !Odd, !Odd && I < 4 && wider);
  };
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < I; i++) {
      const int c = (threadIdx.x + i * width) * V;
      nx[i] = load(p.x, row * p.x_stride + c, p.k - c, x32);
      if (p.residual) nr[i] = load(p.residual, row * p.residual_stride + c, p.k - c, r32);
    }
  };
  // A loaded piece of row r as values.
  auto values = [&](const Piece& piece, const void* base, int64_t stride, int c) {
    if constexpr (kShift)
      return shifted<T, V>(piece, (int)(reinterpret_cast<uintptr_t>(static_cast<const T*>(base) + r * stride) & 15), p.k - c);
    else
      return piece;
  };
  // Two pieces of f32 leave no registers for a second row and a second CTA, which is worth more
  // (3,276 x 5,120: 53 us with the next row ahead, 40 without); four leave none at all.
  constexpr bool kAhead = I == 1 || (I == 2 && (Odd || sizeof(T) == 2));
  if (kAhead) fetch(r);
  for (int turn = 0; r < p.rows; r += step, turn ^= 1) {
    // A CTA's rows use disjoint parts of red (blockDim.x / 32 * blockDim.y <= 32 warps), and a row
    // and the next one different halves.
    float* red = red_sm[turn][0] + threadIdx.y * (width >> 5);
    float* red2 = red_sm[turn][1] + threadIdx.y * (width >> 5);
    float h[I][V];
    if (!kAhead) fetch(r);
#pragma unroll
    for (int i = 0; i < I; i++) {
      const int c = (threadIdx.x + i * width) * V;
      Raw<T, V> x = values(nx[i], p.x, p.x_stride, c);
      unpack(x, h[i]);
      if (p.residual) {
        float a[V];
        unpack(values(nr[i], p.residual, p.residual_stride, c), a);
#pragma unroll
        for (int j = 0; j < V; j++) h[i][j] = h[i][j] + a[j];
        x = pack<T, V>(h[i]);
        unpack(x, h[i]);
      }
      if (p.sum) {
        T* to = static_cast<T*>(p.sum) + r * p.sum_stride + c;
        if constexpr (kShift)
          store_odd<T, V>(to, x, p.k - c);
        else
          store_raw<T, V>(to, x, p.k - c, !Odd, !Odd && I < 4 && s32);
      }
    }
    if (kAhead && r + step < p.rows) fetch(r + step);
    if (p.norm != NORM_NONE) {
      float a = 0.f;
      if (p.norm == NORM_LAYER) {
#pragma unroll
        for (int i = 0; i < I; i++)
#pragma unroll
          for (int j = 0; j < V; j++) a += h[i][j];
        const float mean = row_sum(a, red2) / (float)p.k;
#pragma unroll
        for (int i = 0; i < I; i++) {
          const int c = (threadIdx.x + i * width) * V;
#pragma unroll
          for (int j = 0; j < V; j++) h[i][j] = c + j < p.k ? h[i][j] - mean : 0.f;
        }
        a = 0.f;
      }
#pragma unroll
      for (int i = 0; i < I; i++)
#pragma unroll
        for (int j = 0; j < V; j++) a = fmaf(h[i][j], h[i][j], a);
      const float rstd = 1.0f / sqrtf(row_sum(a, red) / (float)p.k + p.eps);
#pragma unroll
      for (int i = 0; i < I; i++) {
        const int c = (threadIdx.x + i * width) * V, have = p.k - c;
#pragma unroll
        for (int j = 0; j < V; j++) h[i][j] = h[i][j] * rstd;
        float a8[V];
        if (p.weight) {
          unpack(load_raw<float, V>(p.weight + c, have, false, ww), a8);
#pragma unroll
          for (int j = 0; j < V; j++) h[i][j] = h[i][j] * a8[j];
        }
        if (p.bias && p.norm == NORM_LAYER) {
          unpack(load_raw<float, V>(p.bias + c, have, false, bw), a8);
#pragma unroll
          for (int j = 0; j < V; j++) h[i][j] = h[i][j] + a8[j];
        }
      }
    }
    uint8_t* q = p.q + r * p.q_stride;
#pragma unroll
    for (int i = 0; i < I; i++) {
      const int c = (threadIdx.x + i * width) * V, have = p.k - c;
      // Values past the row's end are zero up to here (0 * rstd * 0 + 0).
      float top = kF8Tiny;
#pragma unroll
      for (int j = 0; j < V; j++) top = max_nan(top, fabsf(h[i][j]));
#pragma unroll
      for (int o = kF8Block / V / 2; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
      // A norm's values have all their bits.
      if (p.norm == NORM_NONE) {
        quotients(h[i], top);
      } else {
        const float inv = __fdiv_rn(kF8Max, top);
#pragma unroll
        for (int j = 0; j < V; j++) h[i][j] = h[i][j] * inv;
      }
      if (have >= V) {
        uint32_t e[V / 4];
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(h[i][j], h[i][j + 1]), __NV_SATFINITE, __NV_E4M3);
          const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(h[i][j + 2], h[i][j + 3]), __NV_SATFINITE, __NV_E4M3);
          e[j / 4] = lo | hi << 16;
        }
        if constexpr (V == 16)
          *reinterpret_cast<uint4*>(q + c) = make_uint4(e[0], e[1], e[2], e[3]);
        else
          *reinterpret_cast<uint2*>(q + c) = make_uint2(e[0], e[1]);
      } else {
#pragma unroll
        for (int j = 0; j < V; j++)
          if (j < have) q[c + j] = to_e4m3(h[i][j]);
      }
      if (threadIdx.x % (kF8Block / V) == 0 && have > 0)
        p.scales[(int64_t)(c / kF8Block) * p.scale_stride + r] = __fdiv_rn(top, kF8Max);
    }
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
__global__ void __launch_bounds__(256) f8_quantise_kernel(const float* src, int n, int k, uint8_t* dst, float* scales) {
  __shared__ float red[8];
  const int tile = blockIdx.x, kb = blockIdx.y, kblocks = gridDim.y;
  auto value = [&](int i) -> float {
    const int r = tile * kF8Block + i / kF8Block, c = kb * kF8Block + i % kF8Block;
    if (r >= n || c >= k) return 0.f;
    return src[(int64_t)r * k + c];
  };
  float top = 0.f;
  for (int i = threadIdx.x; i < kF8Block * kF8Block; i += 256) top = max_nan(top, fabsf(value(i)));
  for (int o = 16; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  top = kF8Tiny;
  for (int w = 0; w < 8; w++) top = max_nan(top, red[w]);
  for (int i = threadIdx.x; i < kF8Block * kF8Block; i += 256) {
    const int r = tile * kF8Block + i / kF8Block, c = kb * kF8Block + i % kF8Block;
    if (r >= n || c >= k) continue;
    float v[2] = {value(i), 0.f};
    quotients(v, top);
    dst[packed_at(r, c, kblocks)] = to_e4m3(v[0]);
  }
  if (threadIdx.x == 0) scales[(int64_t)tile * kblocks + kb] = top / kF8Max;
}

}  // namespace

namespace {

// How a kernel's rows of `warps` warps share an SM best: rows per CTA and CTAs per SM. An SM gives
// registers to four warps at a time, so that rows of five warps alone leave a third of it idle
// (16384 x 2560 bf16: 4 rows of 5 warps at once 8 % slower than 6 in CTAs of three). Asked of the
// runtime once per kernel and width.
struct Shape {
  int share, ctas;
};
template <class T, int V, int I, bool Odd>
Shape shape_of(int warps) {
  static std::atomic<uint32_t> known[33];
  uint32_t v = known[warps].load(std::memory_order_relaxed);
  if (!v) {
    int best = 0;
    for (int share = 1; share <= 8 && share * warps * 32 <= (I == 4 ? 1024 : 512); share++) {
      int ctas = 0;
      check_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, norm_f8_kernel<T, V, I, Odd>, share * warps * 32, 0), "occupancy");
      if (share * ctas > best) {
        best = share * ctas;
        v = (uint32_t)share << 16 | (uint32_t)ctas;
      }
    }
    if (!v) throw Error(SVL_ERR_CUDA, "the norm's kernel does not fit an SM");
    known[warps].store(v, std::memory_order_relaxed);
  }
  return {(int)(v >> 16), (int)(v & 0xffff)};
}

template <class T, int V, int I, bool Odd>
void launch_norm_variant(const NormF8Params& p, cudaStream_t s) {
  const int warps = ((p.k + V * I - 1) / (V * I) + 31) / 32;
  Shape sh = shape_of<T, V, I, Odd>(warps);
  // Few rows go to as many SMs as there are.
  const int64_t spread = std::max<int64_t>(1, p.rows / 148);
  if (sh.share > spread) sh.share = (int)spread;
  const int64_t ctas = (p.rows + sh.share - 1) / sh.share;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>(ctas, 148 * sh.ctas));
  cfg.blockDim = dim3(warps * 32, sh.share);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  check_cuda(cudaLaunchKernelEx(&cfg, norm_f8_kernel<T, V, I, Odd>, p), "norm launch");
}

template <class T, int V, int I>
void launch_norm(const NormF8Params& p, cudaStream_t s) {
  auto odd = [](const void* base, int64_t stride) {
    return base && (reinterpret_cast<uintptr_t>(base) | (uint64_t)stride * sizeof(T)) % 16 != 0;
  };
  if (odd(p.x, p.x_stride) || odd(p.residual, p.residual_stride) || odd(p.sum, p.sum_stride))
    launch_norm_variant<T, V, I, true>(p, s);
  else
    launch_norm_variant<T, V, I, false>(p, s);
}

}  // namespace

// 32 bytes of the stream per thread and piece, 16 of bf16 rows that half a warp would hold (16384 x
// 256: 8 us against 14) and of rows too long for 1,024 threads and two pieces.
void launch_norm_f8(const NormF8Params& p, cudaStream_t s) {
  using B = __nv_bfloat16;
  if (p.bf16) {
    if (p.k <= 256)
      launch_norm<B, 8, 1>(p, s);
    else if (p.k <= 8192)
      launch_norm<B, 16, 1>(p, s);
    else if (p.k <= 16384)
      launch_norm<B, 16, 2>(p, s);
    else
      launch_norm<B, 8, 4>(p, s);
  } else {
    if (p.k <= 4096)
      launch_norm<float, 8, 1>(p, s);
    else if (p.k <= 8192)
      launch_norm<float, 8, 2>(p, s);
    else
      launch_norm<float, 8, 4>(p, s);
  }
}

void launch_f8_pack(const uint8_t* src, int64_t stride, int n, int k, uint8_t* dst, cudaStream_t s) {
  f8_pack_kernel<<<148 * 8, 256, 0, s>>>(src, stride, n, k, (k + kF8Block - 1) / kF8Block, dst);
  check_cuda(cudaGetLastError(), "pack launch");
}

void launch_f8_quantise(const float* src, int n, int k, uint8_t* dst, float* scales, cudaStream_t s) {
  const dim3 grid((n + kF8Block - 1) / kF8Block, (k + kF8Block - 1) / kF8Block);  // up to 2^17 x 2^13
  f8_quantise_kernel<<<grid, 256, 0, s>>>(src, n, k, dst, scales);
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
    svl::require_aligned(dtype == SVL_DT_F32 ? 4 : 2, d_x, d_residual, d_sum);
    svl::require_aligned(4, d_weight, d_bias, d_scales);
    require(!d_weight || norm_kind >= 0, "d_weight without a norm");
    require(!d_bias || norm_kind == SVL_NORM_LAYER, "d_bias needs the layer norm");
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
    svl::launch_f8_quantise(staging.as<float>(), n, k, L->w.as<uint8_t>(), L->scales.as<float>(), st);
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
    svl::require_aligned(4, d_scales, d_bias);
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
    // cudaFree waits for the device. A collector may come here while some thread captures a graph,
    // which a call that may wait would end, but for this mode.
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    delete linear;
    cudaThreadExchangeStreamCaptureMode(&mode);
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
    svl::require_aligned(4, d_scales);
    svl::require_aligned(out_dtype == SVL_DT_F32 ? 4 : 2, d_out);
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
