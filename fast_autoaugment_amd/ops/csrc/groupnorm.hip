// Group normalisation with an activation on channels-last maps, forward and backward.
//
//   xhat = (x - mean_g) * rstd_g,  rstd_g = 1/sqrt(var_g + eps)      (a group: cg channels of one sample)
//   z = xhat * w + b,  y = act(z)
//   dz = dy * act'(z),  dw = sum dz xhat,  db = sum dz,  u = dz * w
//   dx = rstd * (u - mean_g(u) - xhat * mean_g(u xhat))
//
// The work is bound by memory: the floor is x read and y written once forward,
// x and dy read and dx written once backward. xhat and z are made again from x
// in the backward pass, so the forward pass saves one mean and one rstd a group.
//
// Statistics are sums around the mean in fp32, never a difference of squares.
// Sums over pixels are taken channel by channel, in a fixed order: a thread owns
// VEC neighbouring channels, the rows of threads are added through LDS, and
// channels are joined to groups last, so a group may be any number of channels.

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <hip/hip_fp16.h>
#include <numeric>
#include "faa_common.h"

namespace {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SWISH = 2 };

// ------------------------------------------------------------ loads and stores

template <typename T, int VEC> struct Pack;
template <int VEC> struct Pack<float, VEC> {
  typedef __attribute__((ext_vector_type(VEC))) float raw;
  static __device__ __forceinline__ float get(const raw& r, int j) { return r[j]; }
  static __device__ __forceinline__ void set(raw& r, int j, float v) { r[j] = v; }
};
template <> struct Pack<float, 1> {
  typedef float raw;
  static __device__ __forceinline__ float get(const raw& r, int) { return r; }
  static __device__ __forceinline__ void set(raw& r, int, float v) { r = v; }
};
template <typename T> __device__ __forceinline__ float bits_to_float(unsigned short u);
template <> __device__ __forceinline__ float bits_to_float<__hip_bfloat16>(unsigned short u) {
  return __uint_as_float((uint32_t)u << 16);
}
template <> __device__ __forceinline__ float bits_to_float<__half>(unsigned short u) {
  return __half2float(__ushort_as_half(u));
}
template <typename T> __device__ __forceinline__ unsigned short float_to_bits(float v);
template <> __device__ __forceinline__ unsigned short float_to_bits<__hip_bfloat16>(float v) {
  __hip_bfloat16 h = __float2bfloat16(v);
  return *(unsigned short*)&h;
}
template <> __device__ __forceinline__ unsigned short float_to_bits<__half>(float v) {
  return __half_as_ushort(__float2half(v));
}
template <typename T> struct Pack<T, 8> {
  typedef __attribute__((ext_vector_type(8))) unsigned short raw;
  static __device__ __forceinline__ float get(const raw& r, int j) { return bits_to_float<T>(r[j]); }
  static __device__ __forceinline__ void set(raw& r, int j, float v) { r[j] = float_to_bits<T>(v); }
};
template <typename T> struct Pack<T, 1> {
  typedef unsigned short raw;
  static __device__ __forceinline__ float get(const raw& r, int) { return bits_to_float<T>(r); }
  static __device__ __forceinline__ void set(raw& r, int, float v) { r = float_to_bits<T>(v); }
};

// weight or bias of channel c: absent, fp32, or the map's type
template <typename T>
__device__ __forceinline__ float param(const void* p, bool f32, int c, float absent) {
  if (p == nullptr) return absent;
  return f32 ? ((const float*)p)[c] : faa_to_float(((const T*)p)[c]);
}
template <>
__device__ __forceinline__ float param<float>(const void* p, bool, int c, float absent) {
  return p == nullptr ? absent : ((const float*)p)[c];
}
template <>
__device__ __forceinline__ float param<__half>(const void* p, bool f32, int c, float absent) {
  if (p == nullptr) return absent;
  return f32 ? ((const float*)p)[c] : __half2float(((const __half*)p)[c]);
}

__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __expf(-z));
}
__device__ __forceinline__ float act_value(float z, int act) {
  if (act == ACT_RELU) return z < 0.0f ? 0.0f : z;      // a NaN stays one
  if (act == ACT_SWISH) return z * sigmoid(z);
  return z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (act == ACT_SWISH) {
    const float s = sigmoid(z);
    return s * (1.0f + z * (1.0f - s));
  }
  return 1.0f;
}

// ------------------------------------------------------------ sums in a workgroup

// A workgroup's threads lie as rows x cv over a tile of ch = cv*VEC channels.
struct Tile {
  int ch, cv, rows, v, r;
  bool on;
  __device__ __forceinline__ Tile(int ch_, int vec) : ch(ch_), cv(ch_ / vec) {
    rows = (int)blockDim.x / cv;
    r = (int)threadIdx.x / cv;
    v = (int)threadIdx.x - r * cv;
    on = r < rows;
  }
};

// out[k][c] = sum over rows of acc[k][c], for K sums at once. lds: K*blockDim*VEC floats; out: K*ch floats.
template <int VEC, int K>
__device__ __forceinline__ void channel_sums(const Tile& t, const float (&acc)[K][VEC], float* lds,
                                             float* out) {
  const int plane = (int)blockDim.x * VEC;
  __syncthreads();
  if (t.on) {
    #pragma unroll
    for (int k = 0; k < K; ++k)
      #pragma unroll
      for (int j = 0; j < VEC; ++j) lds[k * plane + t.r * t.ch + t.v * VEC + j] = acc[k][j];
  }
  __syncthreads();
  // several threads share a column while there are threads left, and leave their sums in the first rows
  int share = (int)blockDim.x / t.ch;
  share = share < 1 ? 1 : (share > t.rows ? t.rows : share);
  if (share > 1) {
    const int s = (int)threadIdx.x / t.ch, c = (int)threadIdx.x - s * t.ch;
    if (s < share) {
      #pragma unroll
      for (int k = 0; k < K; ++k) {
        float sum = 0.0f;
        for (int r = s; r < t.rows; r += share) sum += lds[k * plane + r * t.ch + c];
        lds[k * plane + s * t.ch + c] = sum;    // row s is this thread's own from here on
      }
    }
    __syncthreads();
  } else {
    share = t.rows;
  }
  for (int i = threadIdx.x; i < K * t.ch; i += blockDim.x) {
    const int k = i / t.ch, c = i - k * t.ch;
    float sum = 0.0f;
    for (int r = 0; r < share; ++r) sum += lds[k * plane + r * t.ch + c];
    out[i] = sum;
  }
  __syncthreads();
}

__device__ __forceinline__ float wave_sum(float v) {
  #pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// Workgroups of one sample run one after another on one XCD, whose L2 then joins their parts of a line.
__device__ __forceinline__ int64_t xcd_order(int64_t wg, int64_t n) {
  const int64_t q = n / 8, rem = n % 8, xcd = wg % 8, i = wg / 8;
  return xcd < rem ? xcd * (q + 1) + i : rem * (q + 1) + (xcd - rem) * q + i;
}

// ------------------------------------------------------------ statistics by chunks of pixels

// Any shape: a workgroup takes a chunk of pixels and a tile of channels, and a channel's mean and
// sum of squares around it go to ws[sample][chunk][{mean, m2}][C].
template <typename T, int VEC, int R>
__global__ __launch_bounds__(256) void gn_chunk_stats_kernel(
    const T* __restrict__ x, float* __restrict__ ws, int S, int C, int tile, int ntile, int nchunk,
    int chunk) {
  extern __shared__ float lds[];
  const int64_t wg = blockIdx.x;
  const int ti = (int)(wg % ntile), ck = (int)(wg / ntile % nchunk);
  const int64_t b = wg / ntile / nchunk;
  const int c0 = ti * tile;
  const Tile t(min(tile, C - c0), VEC);
  const int p0 = ck * chunk, np = min(chunk, S - p0);
  const T* xb = x + (b * S + p0) * C + c0 + t.v * VEC;
  typedef Pack<T, VEC> P;
  typename P::raw raw[R];
  float acc[1][VEC];
  #pragma unroll
  for (int j = 0; j < VEC; ++j) acc[0][j] = 0.0f;
  #pragma unroll
  for (int i = 0; i < R; ++i) {
    const int p = t.r + i * t.rows;
    if (t.on && p < np) {
      raw[i] = *(const typename P::raw*)(xb + (int64_t)p * C);
      #pragma unroll
      for (int j = 0; j < VEC; ++j) acc[0][j] += P::get(raw[i], j);
    }
  }
  float* sums = lds + blockDim.x * VEC;
  channel_sums<VEC, 1>(t, acc, lds, sums);
  float mean[VEC];
  #pragma unroll
  for (int j = 0; j < VEC; ++j) {
    mean[j] = sums[t.v * VEC + j] / np;
    acc[0][j] = 0.0f;
  }
  #pragma unroll
  for (int i = 0; i < R; ++i) {
    const int p = t.r + i * t.rows;
    if (t.on && p < np) {
      #pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = P::get(raw[i], j) - mean[j];
        acc[0][j] += d * d;
      }
    }
  }
  float* out = ws + (b * nchunk + ck) * 2 * C + c0;
  for (int c = threadIdx.x; c < t.ch; c += blockDim.x) out[c] = sums[c] / np;
  channel_sums<VEC, 1>(t, acc, lds, sums);
  for (int c = threadIdx.x; c < t.ch; c += blockDim.x) out[C + c] = sums[c];
}

// one workgroup a group: its mean, and the parts' squares moved to it
__global__ __launch_bounds__(256) void gn_join_stats_kernel(
    const float* __restrict__ ws, float* __restrict__ mean_out, float* __restrict__ rstd_out, int S,
    int C, int cg, int nchunk, int chunk, float eps) {
  __shared__ float lds[4];
  const int G = C / cg;
  const int64_t b = blockIdx.x / G;
  const int g = (int)(blockIdx.x % G);
  const float* p = ws + b * nchunk * 2 * C + g * cg;
  float s = 0.0f;
  for (int i = threadIdx.x; i < cg * nchunk; i += blockDim.x) {
    const int k = i / cg, c = i - k * cg;
    s += p[(int64_t)k * 2 * C + c] * min(chunk, S - k * chunk);
  }
  s = faa_block_reduce_sum(s, lds);
  __shared__ float mean_s;
  const float count = (float)cg * (float)S;
  if (threadIdx.x == 0) mean_s = s / count;
  __syncthreads();
  const float mean = mean_s;
  s = 0.0f;
  for (int i = threadIdx.x; i < cg * nchunk; i += blockDim.x) {
    const int k = i / cg, c = i - k * cg;
    const float d = p[(int64_t)k * 2 * C + c] - mean;
    s += p[(int64_t)k * 2 * C + C + c] + d * d * min(chunk, S - k * chunk);
  }
  s = faa_block_reduce_sum(s, lds);
  if (threadIdx.x == 0) {
    mean_out[blockIdx.x] = mean;
    rstd_out[blockIdx.x] = 1.0f / sqrtf(s / count + eps);
  }
}

// what a thread needs to know of its VEC channels
template <typename T, int VEC>
struct Channels {
  float mean[VEC], rstd[VEC], w[VEC], b[VEC];
  __device__ __forceinline__ void load(const float* mean_p, const float* rstd_p, const void* wp,
                                       const void* bp, bool f32, int c0, int cg) {
    int g = c0 / cg, left = cg - (c0 - g * cg);
    #pragma unroll
    for (int j = 0; j < VEC; ++j) {
      mean[j] = mean_p[g];
      rstd[j] = rstd_p[g];
      w[j] = param<T>(wp, f32, c0 + j, 1.0f);
      b[j] = param<T>(bp, f32, c0 + j, 0.0f);
      if (--left == 0 && j + 1 < VEC) { ++g; left = cg; }
    }
  }
};

template <typename T, int VEC, int R>
__global__ __launch_bounds__(256) void gn_chunk_apply_kernel(
    const T* __restrict__ x, const void* __restrict__ w, const void* __restrict__ bias, bool f32,
    const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ y, int S, int C,
    int cg, int tile, int ntile, int nchunk, int chunk, int act) {
  const int64_t wg = blockIdx.x;
  const int ti = (int)(wg % ntile), ck = (int)(wg / ntile % nchunk);
  const int64_t b = wg / ntile / nchunk;
  const int c0 = ti * tile;
  const Tile t(min(tile, C - c0), VEC);
  if (!t.on) return;
  const int p0 = ck * chunk, np = min(chunk, S - p0), G = C / cg;
  const int64_t at = (b * S + p0) * C + c0 + t.v * VEC;
  typedef Pack<T, VEC> P;
  Channels<T, VEC> ch;
  ch.load(mean + b * G, rstd + b * G, w, bias, f32, c0 + t.v * VEC, cg);
  #pragma unroll
  for (int i = 0; i < R; ++i) {
    const int p = t.r + i * t.rows;
    if (p < np) {
      typename P::raw in = *(const typename P::raw*)(x + at + (int64_t)p * C), out;
      #pragma unroll
      for (int j = 0; j < VEC; ++j)
        P::set(out, j, act_value((P::get(in, j) - ch.mean[j]) * ch.rstd[j] * ch.w[j] + ch.b[j], act));
      *(typename P::raw*)(y + at + (int64_t)p * C) = out;
    }
  }
}

// ws[sample][chunk][{sum dz, sum dz xhat}][C]
template <typename T, int VEC, int R>
__global__ __launch_bounds__(256) void gn_chunk_grads_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const void* __restrict__ w,
    const void* __restrict__ bias, bool f32, const float* __restrict__ mean,
    const float* __restrict__ rstd, float* __restrict__ ws, int S, int C, int cg, int tile, int ntile,
    int nchunk, int chunk, int act) {
  extern __shared__ float lds[];
  const int64_t wg = blockIdx.x;
  const int ti = (int)(wg % ntile), ck = (int)(wg / ntile % nchunk);
  const int64_t b = wg / ntile / nchunk;
  const int c0 = ti * tile;
  const Tile t(min(tile, C - c0), VEC);
  const int p0 = ck * chunk, np = min(chunk, S - p0), G = C / cg;
  const int64_t at = (b * S + p0) * C + c0 + t.v * VEC;
  typedef Pack<T, VEC> P;
  float acc[2][VEC];
  #pragma unroll
  for (int j = 0; j < VEC; ++j) acc[0][j] = acc[1][j] = 0.0f;
  if (t.on) {
    Channels<T, VEC> ch;
    ch.load(mean + b * G, rstd + b * G, w, bias, f32, c0 + t.v * VEC, cg);
    #pragma unroll
    for (int i = 0; i < R; ++i) {
      const int p = t.r + i * t.rows;
      if (p < np) {
        typename P::raw xr = *(const typename P::raw*)(x + at + (int64_t)p * C);
        typename P::raw dr = *(const typename P::raw*)(dy + at + (int64_t)p * C);
        #pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float xh = (P::get(xr, j) - ch.mean[j]) * ch.rstd[j];
          const float dz = P::get(dr, j) * act_slope(xh * ch.w[j] + ch.b[j], act);
          acc[0][j] += dz;
          acc[1][j] += dz * xh;
        }
      }
    }
  }
  float* sums = lds + 2 * blockDim.x * VEC;
  channel_sums<VEC, 2>(t, acc, lds, sums);
  float* out = ws + (b * nchunk + ck) * 2 * C + c0;
  for (int i = threadIdx.x; i < 2 * t.ch; i += blockDim.x) {
    const int k = i / t.ch;
    out[(int64_t)k * C + i - k * t.ch] = sums[i];
  }
}

// means[sample][group] = {mean u, mean u xhat}
template <typename T>
__global__ __launch_bounds__(256) void gn_join_grads_kernel(
    const float* __restrict__ ws, const void* __restrict__ w, bool f32, float* __restrict__ means, int S,
    int C, int cg, int nchunk) {
  __shared__ float lds[4];
  const int G = C / cg;
  const int64_t b = blockIdx.x / G;
  const int g = (int)(blockIdx.x % G);
  const float* p = ws + b * nchunk * 2 * C + g * cg;
  float s1 = 0.0f, s2 = 0.0f;
  for (int i = threadIdx.x; i < cg * nchunk; i += blockDim.x) {
    const int k = i / cg, c = i - k * cg;
    const float wc = param<T>(w, f32, g * cg + c, 1.0f);
    s1 += wc * p[(int64_t)k * 2 * C + c];
    s2 += wc * p[(int64_t)k * 2 * C + C + c];
  }
  s1 = faa_block_reduce_sum(s1, lds);
  __syncthreads();
  s2 = faa_block_reduce_sum(s2, lds);
  if (threadIdx.x == 0) {
    const float count = (float)cg * (float)S;
    means[2 * (int64_t)blockIdx.x] = s1 / count;
    means[2 * (int64_t)blockIdx.x + 1] = s2 / count;
  }
}

template <typename T, int VEC, int R>
__global__ __launch_bounds__(256) void gn_chunk_dx_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const void* __restrict__ w,
    const void* __restrict__ bias, bool f32, const float* __restrict__ mean,
    const float* __restrict__ rstd, const float* __restrict__ means, T* __restrict__ dx, int S, int C,
    int cg, int tile, int ntile, int nchunk, int chunk, int act) {
  const int64_t wg = blockIdx.x;
  const int ti = (int)(wg % ntile), ck = (int)(wg / ntile % nchunk);
  const int64_t b = wg / ntile / nchunk;
  const int c0 = ti * tile;
  const Tile t(min(tile, C - c0), VEC);
  if (!t.on) return;
  const int p0 = ck * chunk, np = min(chunk, S - p0), G = C / cg;
  const int64_t at = (b * S + p0) * C + c0 + t.v * VEC;
  typedef Pack<T, VEC> P;
  Channels<T, VEC> ch;
  ch.load(mean + b * G, rstd + b * G, w, bias, f32, c0 + t.v * VEC, cg);
  float m1[VEC], m2[VEC];
  int g = (c0 + t.v * VEC) / cg, left = cg - (c0 + t.v * VEC - g * cg);
  #pragma unroll
  for (int j = 0; j < VEC; ++j) {
    m1[j] = means[2 * (b * G + g)];
    m2[j] = means[2 * (b * G + g) + 1];
    if (--left == 0 && j + 1 < VEC) { ++g; left = cg; }
  }
  #pragma unroll
  for (int i = 0; i < R; ++i) {
    const int p = t.r + i * t.rows;
    if (p < np) {
      typename P::raw xr = *(const typename P::raw*)(x + at + (int64_t)p * C);
      typename P::raw dr = *(const typename P::raw*)(dy + at + (int64_t)p * C), out;
      #pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float xh = (P::get(xr, j) - ch.mean[j]) * ch.rstd[j];
        const float dz = P::get(dr, j) * act_slope(xh * ch.w[j] + ch.b[j], act);
        P::set(out, j, ch.rstd[j] * (dz * ch.w[j] - m1[j] - xh * m2[j]));
      }
      *(typename P::raw*)(dx + at + (int64_t)p * C) = out;
    }
  }
}

// dw[c], db[c]: the sums over n rows of ws[row][{sum dz, sum dz xhat}][C], 32 columns a workgroup
template <typename W>
__global__ __launch_bounds__(1024) void gn_param_grads_kernel(const float* __restrict__ ws, int64_t n,
                                                              int C, W* __restrict__ dw,
                                                              W* __restrict__ db) {
  __shared__ float lds[32][33];
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + col;       // of the 2C columns
  float s = 0.0f;
  if (i < 2 * (int64_t)C)
    for (int64_t r = row; r < n; r += 32) s += ws[r * 2 * C + i];
  lds[row][col] = s;
  __syncthreads();
  if (row == 0 && i < 2 * (int64_t)C) {
    s = 0.0f;
    #pragma unroll
    for (int r = 0; r < 32; ++r) s += lds[r][col];
    W* out = i < C ? db + i : dw + (i - C);
    if constexpr (sizeof(W) == 4) *(float*)out = s;
    else *(unsigned short*)out = float_to_bits<W>(s);
  }
}

// ------------------------------------------------------------ host

struct Shape {
  int64_t B;
  int S, C, G, cg;
  bool vec;
};

Shape shape_of(const torch::Tensor& x, int64_t groups) {
  TORCH_CHECK(x.is_cuda() && x.is_contiguous() && x.dim() == 3, "group_norm: [N, pixels, C] expected");
  Shape s;
  s.B = x.size(0);
  TORCH_CHECK(x.size(1) * x.size(2) < (int64_t(1) << 31), "group_norm: a sample has 2^31 values or more");
  s.S = (int)x.size(1);
  s.C = (int)x.size(2);
  TORCH_CHECK(groups > 0 && s.C % groups == 0, "group_norm: C is no multiple of the groups");
  s.G = (int)groups;
  s.cg = s.C / s.G;
  return s;
}

bool aligned16(std::initializer_list<const torch::Tensor*> ts) {
  for (auto* t : ts)
    if (reinterpret_cast<uintptr_t>(t->data_ptr()) % 16) return false;
  return true;
}

void check_param(const c10::optional<torch::Tensor>& p, const torch::Tensor& x, int C) {
  if (!p.has_value()) return;
  TORCH_CHECK(p->is_contiguous() && p->dim() == 1 && p->size(0) == C && p->device() == x.device()
              && (p->scalar_type() == x.scalar_type() || p->scalar_type() == torch::kFloat32),
              "group_norm: weight and bias are [C], of the map's type or fp32");
}

// chunks of pixels and tiles of channels for workgroups of 256
struct Chunks { int tile, ntile, nchunk, chunk; int64_t wgs; };
template <int VEC>
Chunks chunks_of(const Shape& s, int R) {
  Chunks c;
  c.tile = std::min(s.C, VEC == 1 ? 64 : 32 * VEC);
  c.ntile = (s.C + c.tile - 1) / c.tile;
  const int rows = 256 / (c.tile / VEC);
  c.chunk = rows * R;
  c.nchunk = (s.S + c.chunk - 1) / c.chunk;
  c.wgs = s.B * c.ntile * c.nchunk;
  TORCH_CHECK(c.wgs < (int64_t(1) << 31) && s.B * s.G < (int64_t(1) << 31), "group_norm: too large");
  return c;
}

template <typename F>
void by_type(torch::ScalarType t, F f) {
  if (t == torch::kFloat32) f(float{});
  else if (t == torch::kBFloat16) f(__hip_bfloat16{});
  else if (t == torch::kFloat16) f(__half{});
  else TORCH_CHECK(false, "group_norm: fp32, bf16 and fp16 are taken");
}

constexpr int kR = 8;

template <typename T, int VEC>
void forward(const Shape& s, const torch::Tensor& x, const void* w, const void* b, bool f32,
             torch::Tensor& y, torch::Tensor& mean, torch::Tensor& rstd, double eps, int act,
             hipStream_t stream) {
  const Chunks c = chunks_of<VEC>(s, kR);
  auto ws = torch::empty({s.B * c.nchunk * 2 * s.C}, mean.options());
  const size_t lds = (256 * VEC + c.tile) * sizeof(float);
  hipLaunchKernelGGL((gn_chunk_stats_kernel<T, VEC, kR>), dim3((unsigned)c.wgs), dim3(256), lds, stream,
                     (const T*)x.data_ptr(), ws.data_ptr<float>(), s.S, s.C, c.tile, c.ntile, c.nchunk,
                     c.chunk);
  hipLaunchKernelGGL(gn_join_stats_kernel, dim3((unsigned)(s.B * s.G)), dim3(256), 0, stream,
                     ws.data_ptr<float>(), mean.data_ptr<float>(), rstd.data_ptr<float>(), s.S, s.C,
                     s.cg, c.nchunk, c.chunk, (float)eps);
  hipLaunchKernelGGL((gn_chunk_apply_kernel<T, VEC, kR>), dim3((unsigned)c.wgs), dim3(256), 0, stream,
                     (const T*)x.data_ptr(), w, b, f32, mean.data_ptr<float>(), rstd.data_ptr<float>(),
                     (T*)y.data_ptr(), s.S, s.C, s.cg, c.tile, c.ntile, c.nchunk, c.chunk, act);
}

// returns the rows of sums that the parameters' gradients are made of
template <typename T, int VEC>
torch::Tensor backward(const Shape& s, const torch::Tensor& dy, const torch::Tensor& x, const void* w,
                       const void* b, bool f32, const torch::Tensor& mean, const torch::Tensor& rstd,
                       torch::Tensor& dx, int act, hipStream_t stream) {
  const Chunks c = chunks_of<VEC>(s, kR);
  auto ws = torch::empty({s.B * c.nchunk, 2 * (int64_t)s.C}, mean.options());
  auto means = torch::empty({s.B * s.G * 2}, mean.options());
  const size_t lds = (2 * 256 * VEC + 2 * c.tile) * sizeof(float);
  hipLaunchKernelGGL((gn_chunk_grads_kernel<T, VEC, kR>), dim3((unsigned)c.wgs), dim3(256), lds, stream,
                     (const T*)dy.data_ptr(), (const T*)x.data_ptr(), w, b, f32,
                     mean.data_ptr<float>(), rstd.data_ptr<float>(), ws.data_ptr<float>(), s.S, s.C,
                     s.cg, c.tile, c.ntile, c.nchunk, c.chunk, act);
  hipLaunchKernelGGL((gn_join_grads_kernel<T>), dim3((unsigned)(s.B * s.G)), dim3(256), 0, stream,
                     ws.data_ptr<float>(), w, f32, means.data_ptr<float>(), s.S, s.C, s.cg, c.nchunk);
  hipLaunchKernelGGL((gn_chunk_dx_kernel<T, VEC, kR>), dim3((unsigned)c.wgs), dim3(256), 0, stream,
                     (const T*)dy.data_ptr(), (const T*)x.data_ptr(), w, b, f32,
                     mean.data_ptr<float>(), rstd.data_ptr<float>(), means.data_ptr<float>(),
                     (T*)dx.data_ptr(), s.S, s.C, s.cg, c.tile, c.ntile, c.nchunk, c.chunk, act);
  return ws;
}

}  // namespace

// x: [N, pixels, C] contiguous. Returns y, mean[N, G], rstd[N, G].
std::vector<torch::Tensor> group_norm_fwd(torch::Tensor x, int64_t groups,
                                          c10::optional<torch::Tensor> weight,
                                          c10::optional<torch::Tensor> bias, double eps, int64_t act) {
  Shape s = shape_of(x, groups);
  check_param(weight, x, s.C);
  check_param(bias, x, s.C);
  TORCH_CHECK(!weight || !bias || weight->scalar_type() == bias->scalar_type(),
              "group_norm: weight and bias are of one type");
  TORCH_CHECK(act >= 0 && act <= 2, "group_norm: activation");
  const c10::OptionalDeviceGuard guard(x.device());
  auto stream = at::hip::getCurrentHIPStream().stream();
  auto y = torch::empty_like(x);
  auto stat = x.options().dtype(torch::kFloat32);
  auto mean = torch::empty({s.B, s.G}, stat), rstd = torch::empty({s.B, s.G}, stat);
  if (x.numel() == 0) return {y, mean, rstd};
  const void* w = weight ? weight->data_ptr() : nullptr;
  const void* b = bias ? bias->data_ptr() : nullptr;
  const auto& any = weight ? weight : bias;
  const bool f32 = any && any->scalar_type() == torch::kFloat32;
  by_type(x.scalar_type(), [&](auto z) {
    using T = decltype(z);
    constexpr int V = 16 / sizeof(T);
    if (s.C % V == 0 && aligned16({&x, &y}))
      forward<T, V>(s, x, w, b, f32, y, mean, rstd, eps, (int)act, stream);
    else
      forward<T, 1>(s, x, w, b, f32, y, mean, rstd, eps, (int)act, stream);
  });
  return {y, mean, rstd};
}

// Returns dx, and dweight and dbias in the parameters' type where param_grads is set.
std::vector<torch::Tensor> group_norm_bwd(torch::Tensor dy, torch::Tensor x, int64_t groups,
                                          c10::optional<torch::Tensor> weight,
                                          c10::optional<torch::Tensor> bias, torch::Tensor mean,
                                          torch::Tensor rstd, int64_t act, bool param_grads) {
  Shape s = shape_of(x, groups);
  check_param(weight, x, s.C);
  check_param(bias, x, s.C);
  TORCH_CHECK(dy.is_contiguous() && dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type()
              && dy.device() == x.device(), "group_norm: dy is like x");
  TORCH_CHECK(mean.numel() == s.B * s.G && rstd.numel() == mean.numel(), "group_norm: statistics");
  const c10::OptionalDeviceGuard guard(x.device());
  auto stream = at::hip::getCurrentHIPStream().stream();
  auto dx = torch::empty_like(x);
  const void* w = weight ? weight->data_ptr() : nullptr;
  const void* b = bias ? bias->data_ptr() : nullptr;
  const auto& any = weight ? weight : bias;
  const bool f32 = any && any->scalar_type() == torch::kFloat32;
  auto popt = any ? any->options() : x.options().dtype(torch::kFloat32);
  if (x.numel() == 0) return {dx, torch::zeros({s.C}, popt), torch::zeros({s.C}, popt)};
  torch::Tensor ws;
  by_type(x.scalar_type(), [&](auto z) {
    using T = decltype(z);
    constexpr int V = 16 / sizeof(T);
    if (s.C % V == 0 && aligned16({&x, &dy, &dx}))
      ws = backward<T, V>(s, dy, x, w, b, f32, mean, rstd, dx, (int)act, stream);
    else
      ws = backward<T, 1>(s, dy, x, w, b, f32, mean, rstd, dx, (int)act, stream);
  });
  if (!param_grads) return {dx};
  auto dw = torch::empty({s.C}, popt), db = torch::empty({s.C}, popt);
  by_type(dw.scalar_type(), [&](auto z) {
    using W = decltype(z);
    hipLaunchKernelGGL((gn_param_grads_kernel<W>), dim3((2 * s.C + 31) / 32), dim3(1024), 0, stream,
                       ws.data_ptr<float>(), ws.size(0), s.C, (W*)dw.data_ptr(), (W*)db.data_ptr());
  });
  return {dx, dw, db};
}
