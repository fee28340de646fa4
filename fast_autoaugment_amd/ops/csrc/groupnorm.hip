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
// Measured (bf16): 100x14x14x672 20 + 29 us, 2.7 TB/s, where a map's groups stay
// in registers; 128x56x56x256 in chunks 52 + 9 + 77 us forward and 92 + 7 + 101
// backward, 3.9 TB/s where it is read alone and 5.3 to 6.1 where the end of what
// the pass before read is still in the last-level cache. The same in slices of
// samples that would stay there whole was slower: 136 + 237 us in two of them.
//
// Statistics are sums around the mean in fp32, never a difference of squares.
// Parts of a group are joined by their means, whose rounding costs the variance the
// digits that a mean far from zero has (rstd up to 1e-4 off at a mean of 1000
// spreads). That is no more than a 16-bit map's own rounding; means of fp32 maps are
// taken of x - base, where base is a value of the group (the middle one of three,
// which no single outlier is). It costs them up to 5 % of the forward pass
// (128x28x28x512 91 us for 87); 16-bit maps it would cost 36 us for 29 at
// 128x56x56x64, where one round of workgroups is bound by instructions.
// Sums over pixels are taken channel by channel, in a fixed order: a thread owns
// VEC neighbouring channels, the rows of threads are added through LDS, and
// channels are joined to groups last, so a group may be any number of channels.

#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <hip/hip_fp16.h>
#include <numeric>
#include <type_traits>
#include "faa_common.h"

namespace {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SWISH = 2 };

// ------------------------------------------------------------ loads and stores

template <typename T, int VEC> struct Pack;
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
template <typename T> struct Pack<T, 4> {
  typedef __attribute__((ext_vector_type(4))) unsigned short raw;
  static __device__ __forceinline__ float get(const raw& r, int j) { return bits_to_float<T>(r[j]); }
  static __device__ __forceinline__ void set(raw& r, int j, float v) { r[j] = float_to_bits<T>(v); }
};
template <> struct Pack<float, 4> {
  typedef __attribute__((ext_vector_type(4))) float raw;
  static __device__ __forceinline__ float get(const raw& r, int j) { return r[j]; }
  static __device__ __forceinline__ void set(raw& r, int j, float v) { r[j] = v; }
};
template <typename T> struct Pack<T, 1> {
  typedef unsigned short raw;
  static __device__ __forceinline__ float get(const raw& r, int) { return bits_to_float<T>(r); }
  static __device__ __forceinline__ void set(raw& r, int, float v) { r = float_to_bits<T>(v); }
};

// VEC values `bytes` behind a base that is the same for a whole wave: one register of address a thread
template <typename T, int VEC>
__device__ __forceinline__ typename Pack<T, VEC>::raw load_at(const T* base, uint32_t bytes) {
  return *(const typename Pack<T, VEC>::raw*)((const char*)base + bytes);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_at(T* base, uint32_t bytes, const typename Pack<T, VEC>::raw& v) {
  *(typename Pack<T, VEC>::raw*)((char*)base + bytes) = v;
}

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

// exp2 without the range handling of expf: what it would give below 2^-126 is nothing next to 1
__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if (ACT == ACT_RELU) return z < 0.0f ? 0.0f : z;      // a NaN stays one
  if (ACT == ACT_SWISH) return z * sigmoid(z);
  return z;
}
// d times the slope at z; where relu holds back, no infinity or NaN of d comes through
template <int ACT>
__device__ __forceinline__ float act_grad(float d, float z) {
  if (ACT == ACT_RELU) return z <= 0.0f ? 0.0f : d;
  if (ACT == ACT_SWISH) {
    const float s = sigmoid(z);
    return d * (s + s * (z - z * s));
  }
  return d;
}
// f(activation as a constant): one branch outside the loops, not one an element
template <typename F>
__device__ __forceinline__ void by_act(int act, F f) {
  if (act == ACT_SWISH) f(std::integral_constant<int, ACT_SWISH>{});
  else if (act == ACT_RELU) f(std::integral_constant<int, ACT_RELU>{});
  else f(std::integral_constant<int, ACT_NONE>{});
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
  int share = min(min((int)blockDim.x / t.ch, t.rows), 8);
  if (share > 1) {
    const int s = (int)threadIdx.x / t.ch, c = (int)threadIdx.x - s * t.ch;
    if (s < share) {
      #pragma unroll
      for (int k = 0; k < K; ++k) {
        float sum = 0.0f;
        #pragma unroll 4
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
    #pragma unroll 4
    for (int r = 0; r < share; ++r) sum += lds[k * plane + r * t.ch + c];
    out[i] = sum;
  }
  __syncthreads();
}

// A channel's mean and sum of squares around it (out[c], out[ch+c]) from those of every thread's own pixels:
// parts are moved to the common mean, so nothing large is subtracted. np: pixels of the tile, row r has
// those r, r+rows, ... lds: 2*blockDim*VEC + 8 floats.
template <int VEC>
__device__ __forceinline__ void channel_moments(const Tile& t, const float (&mean)[VEC],
                                                const float (&m2)[VEC], int np, float* lds, float* out) {
  const int plane = (int)blockDim.x * VEC;
  if (t.on) {
    #pragma unroll
    for (int j = 0; j < VEC; ++j) {
      lds[t.r * t.ch + t.v * VEC + j] = mean[j];
      lds[plane + t.r * t.ch + t.v * VEC + j] = m2[j];
    }
  }
  __syncthreads();
  const int full = np / t.rows, rem = np - full * t.rows, rows = min(t.rows, np);
  const float inv_np = 1.0f / (float)np;
  // rows first, first+by, ... to (mean, m2); their pixels are returned
  auto join = [&](int first, int by, int c, float& mean_o, float& m2_o) {
    float s = 0.0f, n = 0.0f, q = 0.0f;
    #pragma unroll 4
    for (int r = first; r < rows; r += by) {
      const float k = (float)(full + (r < rem));
      s += k * lds[r * t.ch + c];
      n += k;
    }
    const float m = s * __builtin_amdgcn_rcpf(n);
    #pragma unroll 4
    for (int r = first; r < rows; r += by) {
      const float d = lds[r * t.ch + c] - m;
      q += lds[plane + r * t.ch + c] + (float)(full + (r < rem)) * d * d;
    }
    mean_o = m;
    m2_o = q;
    return n;
  };
  const int share = min(min((int)blockDim.x / t.ch, rows), 8);      // threads that share a column
  if (share > 1) {
    float* count = lds + 2 * plane;
    const int s = (int)threadIdx.x / t.ch, c = (int)threadIdx.x - s * t.ch;
    if (s < share) {
      float m, q;
      const float n = join(s, share, c, m, q);
      lds[s * t.ch + c] = m;                  // row s was this thread's own
      lds[plane + s * t.ch + c] = q;
      if (c == 0) count[s] = n;
    }
    __syncthreads();
    if ((int)threadIdx.x < t.ch) {
      float sum = 0.0f, q = 0.0f;
      #pragma unroll 4
      for (int r = 0; r < share; ++r) sum += count[r] * lds[r * t.ch + c];
      const float m = sum * inv_np;
      #pragma unroll 4
      for (int r = 0; r < share; ++r) {
        const float d = lds[r * t.ch + c] - m;
        q += lds[plane + r * t.ch + c] + count[r] * d * d;
      }
      out[c] = m;
      out[t.ch + c] = q;
    }
  } else {
    for (int c = threadIdx.x; c < t.ch; c += blockDim.x) join(0, 1, c, out[c], out[t.ch + c]);
  }
  __syncthreads();
}

template <int VEC>
__device__ __forceinline__ void read_vec(const float* table, int c, float (&out)[VEC]) {
  #pragma unroll
  for (int j = 0; j < VEC; ++j) out[j] = table[c + j];
}

// whether a map's values are taken less a value near their mean
template <typename T> constexpr bool kCentred = sizeof(T) == 4;

// A value of the group of each of VEC channels from c in a sample x, the same for all parts of the group: the middle one
// of its first, a central and its last. Where one of them is no number, so is the group. A wave has one x.
template <typename T, int VEC>
__device__ __forceinline__ void group_base(const T* x, int c, int S, int C, int cg, float (&base)[VEC]) {
  typedef Pack<T, 1> P;
  const T *central = x + (int64_t)(S / 2) * C + cg / 2, *last = x + (int64_t)(S - 1) * C + cg - 1;
  auto of = [&](int first) {
    const uint32_t off = (uint32_t)first * sizeof(T);
    return __builtin_amdgcn_fmed3f(P::get(load_at<T, 1>(x, off), 0), P::get(load_at<T, 1>(central, off), 0),
                                   P::get(load_at<T, 1>(last, off), 0));
  };
  int first = c / cg * cg;
  if (cg >= VEC) {            // one group, or two where a vector is no part of it
    const float one = of(first), two = cg % VEC == 0 ? one : of((c + VEC - 1) / cg * cg);
    #pragma unroll
    for (int j = 0; j < VEC; ++j) base[j] = c + j - first < cg ? one : two;
    return;
  }
  #pragma unroll
  for (int j = 0; j < VEC; ++j) {
    if (c + j - first >= cg) first += cg;
    base[j] = of(first);
  }
}

// mean (less base) and sum of squares around it of a thread's own pixels, channel by channel
template <typename T, int VEC, int R>
__device__ __forceinline__ void own_moments(const Tile& t, const typename Pack<T, VEC>::raw (&raw)[R], int np,
                                            const float (&base)[VEC], float (&mean)[VEC], float (&m2)[VEC]) {
  typedef Pack<T, VEC> P;
  #pragma unroll
  for (int j = 0; j < VEC; ++j) mean[j] = m2[j] = 0.0f;
  float n = 0.0f;
  #pragma unroll
  for (int i = 0; i < R; ++i)
    if (t.on && t.r + i * t.rows < np) {
      n += 1.0f;
      #pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float v = P::get(raw[i], j);
        if constexpr (kCentred<T>) v -= base[j];
        mean[j] += v;
      }
    }
  const float inv = n > 0.0f ? 1.0f / n : 0.0f;
  float around[VEC];        // base is no part of the squares: what rounds here they have squared
  #pragma unroll
  for (int j = 0; j < VEC; ++j) {
    mean[j] *= inv;
    around[j] = mean[j];
    if constexpr (kCentred<T>) around[j] += base[j];
  }
  #pragma unroll
  for (int i = 0; i < R; ++i)
    if (t.on && t.r + i * t.rows < np) {
      #pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = P::get(raw[i], j) - around[j];
        m2[j] += d * d;
      }
    }
}

__device__ __forceinline__ float wave_sum(float v) {
  #pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// Workgroups of one sample run one after another on one XCD, whose L2 then joins their parts of a line.
__device__ __forceinline__ uint32_t xcd_order(uint32_t wg, uint32_t n) {
  const uint32_t q = n / 8, rem = n % 8, xcd = wg % 8, i = wg / 8;
  return xcd < rem ? xcd * (q + 1) + i : rem * (q + 1) + (xcd - rem) * q + i;
}

// ------------------------------------------------------------ statistics by chunks of pixels

// Any shape: a workgroup takes a chunk of pixels and a tile of channels, and a channel's mean (less base) and
// sum of squares around it go to ws[sample][chunk][{mean, m2}][C].
template <typename T, int VEC, int R>
__global__ __launch_bounds__(256) void gn_chunk_stats_kernel(
    const T* __restrict__ x, float* __restrict__ ws, int S, int C, int cg, int tile, int ntile, int nchunk,
    int chunk) {
  extern __shared__ float lds[];
  const uint32_t wg = blockIdx.x, at_tile = wg / (uint32_t)ntile, at_chunk = at_tile / (uint32_t)nchunk;
  const int ti = (int)(wg - at_tile * ntile), ck = (int)(at_tile - at_chunk * nchunk);
  const int64_t b = at_chunk;
  const int c0 = ti * tile;
  const Tile t(min(tile, C - c0), VEC);
  const int p0 = ck * chunk, np = min(chunk, S - p0);
  const T* xb = x + (b * S + p0) * C + c0;
  const uint32_t off = (uint32_t)(t.r * C + t.v * VEC) * sizeof(T), step = (uint32_t)(t.rows * C) * sizeof(T);
  typedef Pack<T, VEC> P;
  typename P::raw raw[R];
  #pragma unroll
  for (int i = 0; i < R; ++i)
    if (t.on && t.r + i * t.rows < np) raw[i] = load_at<T, VEC>(xb, off + i * step);
  float base[VEC], mean[VEC], m2[VEC];
  if constexpr (kCentred<T>) group_base<T, VEC>(x + b * S * C, c0 + t.v * VEC, S, C, cg, base);
  own_moments<T, VEC, R>(t, raw, np, base, mean, m2);
  float* out = lds + 2 * blockDim.x * VEC + 8;
  channel_moments<VEC>(t, mean, m2, np, lds, out);
  float* to = ws + (b * nchunk + ck) * 2 * C + c0;
  for (int c = threadIdx.x; c < t.ch; c += blockDim.x) {
    to[c] = out[c];
    to[C + c] = out[t.ch + c];
  }
}

// Joins: a workgroup has `gt` groups of a sample, so that lines of the chunks' sums are read whole. Threads lie as
// parts x channels; what they leave in LDS is added a channel, then a group (a wave each).
struct Join {
  int64_t b;
  int g0, groups, ch, parts, part, col;
  __device__ __forceinline__ Join(int G, int cg, int gt) {
    const uint32_t tiles = (G + gt - 1) / gt, bi = blockIdx.x / tiles;
    b = bi;
    g0 = (int)(blockIdx.x - bi * tiles) * gt;
    groups = min(gt, G - g0);
    ch = groups * cg;
    parts = max(1, 256 / ch);
    part = (int)threadIdx.x / ch;
    col = (int)threadIdx.x - part * ch;
    if (ch > 256) { part = 0; col = threadIdx.x; }
  }
};

// mean and rstd of every group from the chunks' means and squares, which are moved to the joined means
template <typename T>
__global__ __launch_bounds__(256) void gn_join_stats_kernel(
    const T* __restrict__ x, const float* __restrict__ ws, float* __restrict__ mean_out, float* __restrict__ rstd_out, int S,
    int C, int cg, int gt, int nchunk, int chunk, float eps) {
  extern __shared__ float lds[];                // {mean, m2} x channels, then {n, mean, m2} x threads
  const int G = C / cg;
  const Join j(G, cg, gt);
  const float* p = ws + j.b * nchunk * 2 * C + j.g0 * cg;
  float* share = lds + 2 * j.ch;
  for (int c0 = 0; c0 < j.ch; c0 += 256) {
    const int c = c0 + j.col;
    float s = 0.0f, n = 0.0f, q = 0.0f, m = 0.0f;
    const bool on = j.part < j.parts && c < j.ch;
    if (on) {
      #pragma unroll 4
      for (int k = j.part; k < nchunk; k += j.parts) {
        const float np = (float)min(chunk, S - k * chunk);
        s += p[(int64_t)k * 2 * C + c] * np;
        n += np;
      }
      m = n > 0.0f ? s / n : 0.0f;
      #pragma unroll 4
      for (int k = j.part; k < nchunk; k += j.parts) {
        const float d = p[(int64_t)k * 2 * C + c] - m;
        q += p[(int64_t)k * 2 * C + C + c] + d * d * (float)min(chunk, S - k * chunk);
      }
    }
    __syncthreads();
    share[threadIdx.x] = n;
    share[256 + threadIdx.x] = m;
    share[512 + threadIdx.x] = q;
    __syncthreads();
    if (on && j.part == 0) {
      float sum = 0.0f;
      for (int k = 0; k < j.parts; ++k) sum += share[k * j.ch + j.col] * share[256 + k * j.ch + j.col];
      const float mean = sum / (float)S;
      float m2 = 0.0f;
      for (int k = 0; k < j.parts; ++k) {
        const float d = share[256 + k * j.ch + j.col] - mean;
        m2 += share[512 + k * j.ch + j.col] + share[k * j.ch + j.col] * d * d;
      }
      lds[c] = mean;
      lds[j.ch + c] = m2;
    }
  }
  __syncthreads();
  const int lane = threadIdx.x & 63;
  for (int g = (int)threadIdx.x >> 6; g < j.groups; g += 4) {
    float s = 0.0f, q = 0.0f;
    float base[1] = {0.0f};
    if constexpr (kCentred<T>) group_base<T, 1>(x + j.b * S * C, (j.g0 + g) * cg, S, C, cg, base);
    for (int c = lane; c < cg; c += 64) s += lds[g * cg + c];
    const float mean = wave_sum(s) / (float)cg;
    for (int c = lane; c < cg; c += 64) {
      const float d = lds[g * cg + c] - mean;
      q += lds[j.ch + g * cg + c] + (float)S * d * d;
    }
    const float rstd = 1.0f / sqrtf(wave_sum(q) / ((float)cg * (float)S) + eps);
    if (lane == 0) {
      mean_out[j.b * G + j.g0 + g] = base[0] + mean;
      rstd_out[j.b * G + j.g0 + g] = rstd;
    }
  }
}

// ------------------------------------------------------------ a channel's constants

// z = x a + c with a = rstd w, c = b - mean a;  xhat = x rstd + shift with shift = -mean rstd;
// dx = dz a + x p + q with p = -rstd^2 m2, q = -rstd m1 - shift rstd m2   (m1, m2: means of u, u xhat).
// A mean far from zero costs y the digits that it costs the mean itself. It would cost sum dz xhat = rstd sum dz x +
// shift sum dz more: at a mean of 30 spreads, dw 3e-6 of itself where the formula loses 7e-7. That is far below what
// 16-bit maps hold, whose loops have these two constants a channel; for fp32 maps the backward pass subtracts the mean
// first: with x - mean in the place of x, c is b, shift 0 and q = -rstd m1 (128x28x28x512 160 us for 153).
// A workgroup makes them once for its tile, in LDS; a thread then has those of its VEC channels.
template <typename T, int VEC, int R>
__global__ __launch_bounds__(256) void gn_chunk_apply_kernel(
    const T* __restrict__ x, const void* __restrict__ w, const void* __restrict__ bias, bool f32,
    const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ y, int S, int C,
    int cg, int tile, int ntile, int nchunk, int chunk, int act) {
  extern __shared__ float lds[];                // {a, c} x tile
  // last chunks first: they were read last, and may still be in the cache behind the L2s
  const uint32_t wg = gridDim.x - 1 - blockIdx.x, at_tile = wg / (uint32_t)ntile, at_chunk = at_tile / (uint32_t)nchunk;
  const int ti = (int)(wg - at_tile * ntile), ck = (int)(at_tile - at_chunk * nchunk);
  const int64_t b = at_chunk;
  const int c0 = ti * tile;
  const Tile t(min(tile, C - c0), VEC);
  const int p0 = ck * chunk, np = min(chunk, S - p0), G = C / cg;
  const int64_t at = (b * S + p0) * C + c0;
  const uint32_t off = (uint32_t)(t.r * C + t.v * VEC) * sizeof(T), step = (uint32_t)(t.rows * C) * sizeof(T);
  typedef Pack<T, VEC> P;
  typename P::raw raw[R];
  #pragma unroll
  for (int i = 0; i < R; ++i) {
    const int p = t.r + i * t.rows;
    if (t.on && p < np) raw[i] = load_at<T, VEC>(x + at, off + i * step);
  }
  for (int c = threadIdx.x; c < t.ch; c += blockDim.x) {
    const int64_t g = b * G + (c0 + c) / cg;
    const float a = rstd[g] * param<T>(w, f32, c0 + c, 1.0f);
    lds[c] = a;
    lds[tile + c] = param<T>(bias, f32, c0 + c, 0.0f) - mean[g] * a;
  }
  __syncthreads();
  if (!t.on) return;
  float a[VEC], c[VEC];
  read_vec<VEC>(lds, t.v * VEC, a);
  read_vec<VEC>(lds + tile, t.v * VEC, c);
  by_act(act, [&](auto A) {
    #pragma unroll
    for (int i = 0; i < R; ++i) {
      const int p = t.r + i * t.rows;
      if (p < np) {
        typename P::raw out;
        #pragma unroll
        for (int j = 0; j < VEC; ++j)
          P::set(out, j, act_value<A.value>(P::get(raw[i], j) * a[j] + c[j]));
        store_at<T, VEC>(y + at, off + i * step, out);
      }
    }
  });
}

// the constants of the backward pass's first half: {rstd, shift or mean, a, c} x tile
template <typename T>
__device__ __forceinline__ void backward_table(float* table, int tile, int ch, int c0, int cg,
                                               const float* mean, const float* rstd, const void* w,
                                               const void* bias, bool f32) {
  for (int c = threadIdx.x; c < ch; c += blockDim.x) {
    const int g = (c0 + c) / cg;
    const float r = rstd[g], shift = -mean[g] * r, wc = param<T>(w, f32, c0 + c, 1.0f);
    table[c] = r;
    table[tile + c] = kCentred<T> ? mean[g] : shift;
    table[2 * tile + c] = r * wc;
    table[3 * tile + c] = param<T>(bias, f32, c0 + c, 0.0f) + (kCentred<T> ? 0.0f : shift * wc);
  }
}

// ws[sample][chunk][{sum dz, sum dz xhat}][C]. A chunk is R/H groups of H loads a thread.
template <typename T, int VEC, int R, int H>
__global__ __launch_bounds__(256) void gn_chunk_grads_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const void* __restrict__ w,
    const void* __restrict__ bias, bool f32, const float* __restrict__ mean,
    const float* __restrict__ rstd, float* __restrict__ ws, int S, int C, int cg, int tile, int ntile,
    int nchunk, int chunk, int act) {
  extern __shared__ float lds[];
  const uint32_t wg = blockIdx.x, at_tile = wg / (uint32_t)ntile, at_chunk = at_tile / (uint32_t)nchunk;
  const int ti = (int)(wg - at_tile * ntile), ck = (int)(at_tile - at_chunk * nchunk);
  const int64_t b = at_chunk;
  const int c0 = ti * tile;
  const Tile t(min(tile, C - c0), VEC);
  const int p0 = ck * chunk, np = min(chunk, S - p0), G = C / cg;
  const int64_t at = (b * S + p0) * C + c0;
  const uint32_t off = (uint32_t)(t.r * C + t.v * VEC) * sizeof(T), step = (uint32_t)(t.rows * C) * sizeof(T);
  typedef Pack<T, VEC> P;
  float* table = lds + 2 * blockDim.x * VEC;
  float* sums = table + 4 * tile;
  backward_table<T>(table, tile, t.ch, c0, cg, mean + b * G, rstd + b * G, w, bias, f32);
  __syncthreads();
  float acc[2][VEC];
  #pragma unroll
  for (int j = 0; j < VEC; ++j) acc[0][j] = acc[1][j] = 0.0f;
  if (t.on) {
    float mu[VEC];        // of fp32 maps
    if constexpr (kCentred<T>) read_vec<VEC>(table + tile, t.v * VEC, mu);
    float a[VEC], c[VEC];
    read_vec<VEC>(table + 2 * tile, t.v * VEC, a);
    read_vec<VEC>(table + 3 * tile, t.v * VEC, c);
    by_act(act, [&](auto A) {
      #pragma unroll 1
      for (int o = 0; o < R; o += H) {
        typename P::raw xr[H], dr[H];
        #pragma unroll
        for (int i = 0; i < H; ++i)
          if (t.r + (o + i) * t.rows < np) {
            xr[i] = load_at<T, VEC>(x + at, off + (o + i) * step);
            dr[i] = load_at<T, VEC>(dy + at, off + (o + i) * step);
          }
        #pragma unroll
        for (int i = 0; i < H; ++i)
          if (t.r + (o + i) * t.rows < np) {
            #pragma unroll
            for (int j = 0; j < VEC; ++j) {
              float xv = P::get(xr[i], j);
              if constexpr (kCentred<T>) xv -= mu[j];
              const float dz = act_grad<A.value>(P::get(dr[i], j), xv * a[j] + c[j]);
              acc[0][j] += dz;
              acc[1][j] += dz * xv;
            }
          }
      }
    });
  }
  channel_sums<VEC, 2>(t, acc, lds, sums);
  float* out = ws + (b * nchunk + ck) * 2 * C + c0;
  for (int i = threadIdx.x; i < t.ch; i += blockDim.x) {
    out[i] = sums[i];
    out[C + i] = table[i] * sums[t.ch + i] + (kCentred<T> ? 0.0f : table[tile + i] * sums[i]);
  }
}

// means[sample][group] = {mean u, mean u xhat}, and the chunks' sums joined a channel to
// sample[sample][{sum dz, sum dz xhat}][C], which the parameters' gradients are made of
template <typename T>
__global__ __launch_bounds__(256) void gn_join_grads_kernel(
    const float* __restrict__ ws, const void* __restrict__ w, bool f32, float* __restrict__ means,
    float* __restrict__ sample, int S, int C, int cg, int gt, int nchunk) {
  extern __shared__ float lds[];                // {u, u xhat} x channels, then {dz, dz xhat} x threads
  const int G = C / cg;
  const Join j(G, cg, gt);
  const int at = j.g0 * cg;
  const float* p = ws + j.b * nchunk * 2 * C + at;
  float* share = lds + 2 * j.ch;
  for (int c0 = 0; c0 < j.ch; c0 += 256) {
    const int c = c0 + j.col;
    float a = 0.0f, d = 0.0f;
    const bool on = j.part < j.parts && c < j.ch;
    if (on) {
      #pragma unroll 4
      for (int k = j.part; k < nchunk; k += j.parts) {
        a += p[(int64_t)k * 2 * C + c];
        d += p[(int64_t)k * 2 * C + C + c];
      }
    }
    __syncthreads();
    share[threadIdx.x] = a;
    share[256 + threadIdx.x] = d;
    __syncthreads();
    if (on && j.part == 0) {
      for (int k = 1; k < j.parts; ++k) {
        a += share[k * j.ch + j.col];
        d += share[256 + k * j.ch + j.col];
      }
      sample[j.b * 2 * C + at + c] = a;
      sample[j.b * 2 * C + C + at + c] = d;
      const float wc = param<T>(w, f32, at + c, 1.0f);
      lds[c] = wc * a;
      lds[j.ch + c] = wc * d;
    }
  }
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const float count = (float)cg * (float)S;
  for (int g = (int)threadIdx.x >> 6; g < j.groups; g += 4) {
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = lane; c < cg; c += 64) {
      s1 += lds[g * cg + c];
      s2 += lds[j.ch + g * cg + c];
    }
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    if (lane == 0) {
      means[2 * (j.b * G + j.g0 + g)] = s1 / count;
      means[2 * (j.b * G + j.g0 + g) + 1] = s2 / count;
    }
  }
}

template <typename T, int VEC, int R, int H>
__global__ __launch_bounds__(256) void gn_chunk_dx_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const void* __restrict__ w,
    const void* __restrict__ bias, bool f32, const float* __restrict__ mean,
    const float* __restrict__ rstd, const float* __restrict__ means, T* __restrict__ dx, int S, int C,
    int cg, int tile, int ntile, int nchunk, int chunk, int act) {
  extern __shared__ float lds[];                // {a, c, p, q, mean} x tile
  // last chunks first: they were read last, and may still be in the cache behind the L2s
  const uint32_t wg = gridDim.x - 1 - blockIdx.x, at_tile = wg / (uint32_t)ntile, at_chunk = at_tile / (uint32_t)nchunk;
  const int ti = (int)(wg - at_tile * ntile), ck = (int)(at_tile - at_chunk * nchunk);
  const int64_t b = at_chunk;
  const int c0 = ti * tile;
  const Tile t(min(tile, C - c0), VEC);
  const int p0 = ck * chunk, np = min(chunk, S - p0), G = C / cg;
  const int64_t at = (b * S + p0) * C + c0;
  const uint32_t off = (uint32_t)(t.r * C + t.v * VEC) * sizeof(T), step = (uint32_t)(t.rows * C) * sizeof(T);
  typedef Pack<T, VEC> P;
  for (int c = threadIdx.x; c < t.ch; c += blockDim.x) {
    const int64_t g = b * G + (c0 + c) / cg;
    const float r = rstd[g], shift = -mean[g] * r, wc = param<T>(w, f32, c0 + c, 1.0f);
    const float m1 = means[2 * g], m2 = means[2 * g + 1];
    lds[c] = r * wc;
    lds[tile + c] = param<T>(bias, f32, c0 + c, 0.0f) + (kCentred<T> ? 0.0f : shift * wc);
    lds[2 * tile + c] = -r * r * m2;
    lds[3 * tile + c] = -r * (m1 + (kCentred<T> ? 0.0f : shift * m2));
    if (kCentred<T>) lds[4 * tile + c] = mean[g];
  }
  __syncthreads();
  if (!t.on) return;
  float mu[VEC];        // of fp32 maps
  if constexpr (kCentred<T>) read_vec<VEC>(lds + 4 * tile, t.v * VEC, mu);
  float a[VEC], c[VEC], pp[VEC], q[VEC];
  read_vec<VEC>(lds, t.v * VEC, a);
  read_vec<VEC>(lds + tile, t.v * VEC, c);
  read_vec<VEC>(lds + 2 * tile, t.v * VEC, pp);
  read_vec<VEC>(lds + 3 * tile, t.v * VEC, q);
  by_act(act, [&](auto A) {
    #pragma unroll 1
    for (int o = 0; o < R; o += H) {
      typename P::raw xr[H], dr[H];
      #pragma unroll
      for (int i = 0; i < H; ++i)
        if (t.r + (o + i) * t.rows < np) {
          xr[i] = load_at<T, VEC>(x + at, off + (o + i) * step);
          dr[i] = load_at<T, VEC>(dy + at, off + (o + i) * step);
        }
      #pragma unroll
      for (int i = 0; i < H; ++i)
        if (t.r + (o + i) * t.rows < np) {
          typename P::raw out;
          #pragma unroll
          for (int j = 0; j < VEC; ++j) {
            float xv = P::get(xr[i], j);
            if constexpr (kCentred<T>) xv -= mu[j];
            const float dz = act_grad<A.value>(P::get(dr[i], j), xv * a[j] + c[j]);
            P::set(out, j, dz * a[j] + (xv * pp[j] + q[j]));
          }
          store_at<T, VEC>(dx + at, off + (o + i) * step, out);
        }
    }
  });
}

// ------------------------------------------------------------ a map that stays in registers

// out[g] = sum of a tile's channel sums over each of its groups, a wave a group
__device__ __forceinline__ void group_sums(const float* sums, float* out, int ch, int cg) {
  const int lane = threadIdx.x & 63, waves = (int)blockDim.x >> 6;
  for (int g = (int)threadIdx.x >> 6; g < ch / cg; g += waves) {
    float s = 0.0f;
    for (int c = lane; c < cg; c += 64) s += sums[g * cg + c];
    s = wave_sum(s);
    if (lane == 0) out[g] = s;
  }
  __syncthreads();
}

// A workgroup takes all pixels of `tile` channels (whole groups) of one sample: x is read once.
template <typename T, int VEC, int R>
__global__ __launch_bounds__(1024) void gn_whole_fwd_kernel(
    const T* __restrict__ x, const void* __restrict__ w, const void* __restrict__ bias, bool f32,
    T* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, int S, int C, int cg,
    int tile, int ntile, int act, float eps) {
  extern __shared__ float lds[];
  const uint32_t wg = xcd_order(blockIdx.x, gridDim.x), bi = wg / (uint32_t)ntile;
  const int c0 = (int)(wg - bi * ntile) * tile;
  const int64_t b = bi;
  const Tile t(min(tile, C - c0), VEC);
  const int64_t at = b * S * C + c0;
  const uint32_t off = (uint32_t)(t.r * C + t.v * VEC) * sizeof(T), step = (uint32_t)(t.rows * C) * sizeof(T);
  float* channels = lds + 2 * blockDim.x * VEC + 8; // {mean, m2} x channels
  float* groups = channels + 2 * tile;              // {mean, rstd} x groups
  float* bases = groups + 2 * tile;                 // channels, of fp32 maps
  typedef Pack<T, VEC> P;
  typename P::raw raw[R];
  #pragma unroll
  for (int i = 0; i < R; ++i)
    if (t.on && t.r + i * t.rows < S) raw[i] = load_at<T, VEC>(x + at, off + i * step);
  float base[VEC], m[VEC], m2[VEC];
  if constexpr (kCentred<T>) group_base<T, VEC>(x + b * S * C, c0 + t.v * VEC, S, C, cg, base);
  own_moments<T, VEC, R>(t, raw, S, base, m, m2);
  if constexpr (kCentred<T>)
    if (t.r == 0) {
      #pragma unroll
      for (int j = 0; j < VEC; ++j) bases[t.v * VEC + j] = base[j];
    }
  channel_moments<VEC>(t, m, m2, S, lds, channels);
  const int64_t g0 = b * (C / cg) + c0 / cg;
  const int lane = threadIdx.x & 63;
  for (int g = (int)threadIdx.x >> 6; g < t.ch / cg; g += (int)blockDim.x >> 6) {     // a wave a group
    float s = 0.0f, q = 0.0f;
    for (int c = lane; c < cg; c += 64) s += channels[g * cg + c];
    const float mean = wave_sum(s) / (float)cg;
    for (int c = lane; c < cg; c += 64) {
      const float d = channels[g * cg + c] - mean;
      q += channels[t.ch + g * cg + c] + (float)S * d * d;
    }
    const float rstd = 1.0f / sqrtf(wave_sum(q) / ((float)cg * (float)S) + eps);
    if (lane == 0) {
      groups[2 * g] = mean_out[g0 + g] = kCentred<T> ? bases[g * cg] + mean : mean;
      groups[2 * g + 1] = rstd;
      rstd_out[g0 + g] = rstd;
    }
  }
  __syncthreads();
  // a and c of every channel take the place of the rows
  for (int c = threadIdx.x; c < t.ch; c += blockDim.x) {
    const int g = c / cg;
    const float a = groups[2 * g + 1] * param<T>(w, f32, c0 + c, 1.0f);
    lds[c] = a;
    lds[tile + c] = param<T>(bias, f32, c0 + c, 0.0f) - groups[2 * g] * a;
  }
  __syncthreads();
  if (!t.on) return;
  float a[VEC], c[VEC];
  read_vec<VEC>(lds, t.v * VEC, a);
  read_vec<VEC>(lds + tile, t.v * VEC, c);
  by_act(act, [&](auto A) {
    #pragma unroll
    for (int i = 0; i < R; ++i) {
      const int p = t.r + i * t.rows;
      if (p < S) {
        typename P::raw out;
        #pragma unroll
        for (int j = 0; j < VEC; ++j)
          P::set(out, j, act_value<A.value>(P::get(raw[i], j) * a[j] + c[j]));
        store_at<T, VEC>(y + at, off + i * step, out);
      }
    }
  });
}

// x and dy are read once; sample[b][{sum dz, sum dz xhat}][C] goes to the parameters' gradients
template <typename T, int VEC, int R>
__global__ __launch_bounds__(1024) void gn_whole_bwd_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const void* __restrict__ w,
    const void* __restrict__ bias, bool f32, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, T* __restrict__ dx, float* __restrict__ sample, int S, int C, int cg,
    int tile, int ntile, int act) {
  extern __shared__ float lds[];
  const uint32_t wg = xcd_order(blockIdx.x, gridDim.x), bi = wg / (uint32_t)ntile;
  const int c0 = (int)(wg - bi * ntile) * tile;
  const int64_t b = bi;
  const Tile t(min(tile, C - c0), VEC);
  const int64_t at = b * S * C + c0, g0 = b * (C / cg);
  const uint32_t off = (uint32_t)(t.r * C + t.v * VEC) * sizeof(T), step = (uint32_t)(t.rows * C) * sizeof(T);
  float* table = lds + 2 * blockDim.x * VEC;    // {rstd, shift or mean, a, c} x tile
  float* sums = table + 4 * tile;               // {dz, dz xhat} x channels
  float* groups = sums + 2 * tile;              // {u, u xhat} x groups
  typedef Pack<T, VEC> P;
  typename P::raw xr[R], dr[R];
  #pragma unroll
  for (int i = 0; i < R; ++i) {
    const int p = t.r + i * t.rows;
    if (t.on && p < S) {
      xr[i] = load_at<T, VEC>(x + at, off + i * step);
      dr[i] = load_at<T, VEC>(dy + at, off + i * step);
    }
  }
  backward_table<T>(table, tile, t.ch, c0, cg, mean_in + g0, rstd_in + g0, w, bias, f32);
  __syncthreads();
  float mu[VEC];        // of fp32 maps
  if constexpr (kCentred<T>) read_vec<VEC>(table + tile, t.v * VEC, mu);
  float a[VEC], c[VEC];
  read_vec<VEC>(table + 2 * tile, t.v * VEC, a);
  read_vec<VEC>(table + 3 * tile, t.v * VEC, c);
  float acc[2][VEC];
  #pragma unroll
  for (int j = 0; j < VEC; ++j) acc[0][j] = acc[1][j] = 0.0f;
  by_act(act, [&](auto A) {
    #pragma unroll
    for (int i = 0; i < R; ++i)
      if (t.on && t.r + i * t.rows < S) {
        #pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float xv = P::get(xr[i], j);
          if constexpr (kCentred<T>) xv -= mu[j];
          const float dz = act_grad<A.value>(P::get(dr[i], j), xv * a[j] + c[j]);
          acc[0][j] += dz;
          acc[1][j] += dz * xv;
        }
      }
  });
  channel_sums<VEC, 2>(t, acc, lds, sums);
  for (int i = threadIdx.x; i < t.ch; i += blockDim.x) {
    const float s1 = sums[i], s2 = table[i] * sums[t.ch + i] + (kCentred<T> ? 0.0f : table[tile + i] * s1);
    const float wc = param<T>(w, f32, c0 + i, 1.0f);
    sample[b * 2 * C + c0 + i] = s1;
    sample[(b * 2 + 1) * C + c0 + i] = s2;
    sums[i] = s1 * wc;
    sums[t.ch + i] = s2 * wc;
  }
  __syncthreads();
  group_sums(sums, groups, 2 * t.ch, cg);       // both planes: a tile is whole groups
  const float inv = 1.0f / ((float)cg * (float)S);
  for (int i = threadIdx.x; i < t.ch; i += blockDim.x) {
    const int g = i / cg;
    const float m1 = groups[g] * inv, m2 = groups[t.ch / cg + g] * inv, r = table[i],
                shift = kCentred<T> ? 0.0f : table[tile + i];
    table[i] = -r * r * m2;
    table[tile + i] = -r * (m1 + shift * m2);
  }
  __syncthreads();
  if (!t.on) return;
  float pp[VEC], q[VEC];
  read_vec<VEC>(table, t.v * VEC, pp);
  read_vec<VEC>(table + tile, t.v * VEC, q);
  by_act(act, [&](auto A) {
    #pragma unroll
    for (int i = 0; i < R; ++i) {
      const int p = t.r + i * t.rows;
      if (p < S) {
        typename P::raw out;
        #pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float xv = P::get(xr[i], j);
          if constexpr (kCentred<T>) xv -= mu[j];
          const float dz = act_grad<A.value>(P::get(dr[i], j), xv * a[j] + c[j]);
          P::set(out, j, dz * a[j] + (xv * pp[j] + q[j]));
        }
        store_at<T, VEC>(dx + at, off + i * step, out);
      }
    }
  });
}

// out[y][column] = sum over the rows y*per .. of ws[row][2C], 32 columns a workgroup; where there is one y, the
// columns are db (sum dz) and dw (sum dz xhat)
template <typename W>
__global__ __launch_bounds__(1024) void gn_param_grads_kernel(const float* __restrict__ ws, int64_t n,
                                                              int64_t per, int C, float* __restrict__ out,
                                                              W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float lds[32][33];
  const int col = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + col;       // of the 2C columns
  const int64_t r0 = blockIdx.y * per, r1 = min(r0 + per, n);
  float s = 0.0f;
  if (i < 2 * (int64_t)C)
    #pragma unroll 4
    for (int64_t r = r0 + row; r < r1; r += 32) s += ws[r * 2 * C + i];
  lds[row][col] = s;
  __syncthreads();
  if (row == 0 && i < 2 * (int64_t)C) {
    s = 0.0f;
    #pragma unroll
    for (int r = 0; r < 32; ++r) s += lds[r][col];
    if (out) {
      out[blockIdx.y * 2 * (int64_t)C + i] = s;
      return;
    }
    W* to = i < C ? db + i : dw + (i - C);
    if constexpr (sizeof(W) == 4) *(float*)to = s;
    else *(unsigned short*)to = float_to_bits<W>(s);
  }
}

// ------------------------------------------------------------ host

struct Shape {
  int64_t B;
  int S, C, G, cg;
};

// t with its channels last in memory, whatever its order is: [N, C, ...] over lines of C
torch::Tensor channels_last(const torch::Tensor& t) {
  if (t.dim() == 4) return t.contiguous(at::MemoryFormat::ChannelsLast);
  if (t.dim() == 5) return t.contiguous(at::MemoryFormat::ChannelsLast3d);
  if (t.dim() == 2) return t.contiguous();
  return t.movedim(1, -1).contiguous().movedim(-1, 1);
}

// x: [N, C, ...], channels last
Shape shape_of(const torch::Tensor& x, int64_t groups, const torch::Tensor& w, const torch::Tensor& b,
               int64_t act) {
  TORCH_CHECK(x.is_cuda() && x.dim() >= 2, "group_norm_act: [N, C, ...] on the GPU");
  Shape s;
  s.B = x.size(0);
  const int64_t C = x.size(1), S = x.numel() ? x.numel() / (s.B * C) : 0;
  TORCH_CHECK(S * C < (int64_t(1) << 31), "group_norm_act: a sample has 2^31 values or more");
  TORCH_CHECK(C < (1 << 23), "group_norm_act: 2^23 channels or more");
  // a channel's sums wait in LDS until its group is joined
  TORCH_CHECK(groups <= 0 || C / groups <= 16384, "group_norm_act: a group has more than 16384 channels");
  TORCH_CHECK(groups > 0 && C > 0 && C % groups == 0, "group_norm_act: C is no multiple of the groups");
  s.S = (int)S;
  s.C = (int)C;
  s.G = (int)groups;
  s.cg = s.C / s.G;
  for (const auto* p : {&w, &b})
    TORCH_CHECK(!p->defined() || (p->is_contiguous() && p->dim() == 1 && p->size(0) == C
                && p->device() == x.device()
                && (p->scalar_type() == x.scalar_type() || p->scalar_type() == torch::kFloat32)),
                "group_norm_act: weight and bias are [C], of the map's type or fp32");
  TORCH_CHECK(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(),
              "group_norm_act: weight and bias are of one type");
  TORCH_CHECK(act >= 0 && act <= 2, "group_norm_act: activation");
  return s;
}

const void* data(const torch::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
bool is_f32(const torch::Tensor& w, const torch::Tensor& b) {
  return (w.defined() && w.scalar_type() == torch::kFloat32)
         || (b.defined() && b.scalar_type() == torch::kFloat32);
}

bool aligned16(std::initializer_list<const torch::Tensor*> ts) {
  for (auto* t : ts)
    if (reinterpret_cast<uintptr_t>(t->data_ptr()) % 16) return false;
  return true;
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
  c.nchunk = (int)(((int64_t)s.S + c.chunk - 1) / c.chunk);
  c.wgs = s.B * c.ntile * c.nchunk;
  TORCH_CHECK(c.wgs < (int64_t(1) << 24) && s.B * s.G < (int64_t(1) << 24),
              "group_norm_act: more workgroups than a launch takes");     // 2^32 threads
  return c;
}

template <typename F>
void by_type(torch::ScalarType t, F f) {
  if (t == torch::kFloat32) f(float{});
  else if (t == torch::kBFloat16) f(__hip_bfloat16{});
  else if (t == torch::kFloat16) f(__half{});
  else TORCH_CHECK(false, "group_norm: fp32, bf16 and fp16 are taken");
}

// How a map is cut where its pixels fit the registers of a workgroup.
struct Whole { int tile, ntile, threads, r; };

// Tiles are whole groups and whole vectors. About 2048 vectors of 16 bytes a workgroup are aimed at (256 threads
// with 8 each: several workgroups fit a CU, and some load while others add up): wide tiles where the map is
// small, down to lines of 128, 64 and 32 bytes as long as there are fewer than 1024, 512 and 256 workgroups.
// Over 4096 vectors a CU holds one workgroup or two and waits for each of its phases, and the chunks' second
// read is cheaper, unless all workgroups run at once, when lines of 32 bytes do too. Measured (bf16, forward +
// backward, us, whole/chunks): 128x14x14x1024 26+40/41+64, 128x28x28x512 41+98/62+104, 128x56x56x64 26+53/40+62,
// 128x56x56x256 136+263/125+211.
// Where a CU has two workgroups at most, their own waves have to hide what they wait for: 4 vectors a thread or
// more threads (forward, us, against 8 or 16 vectors in 256): 128x32x32x32 10.9/11.5, 8x32x32x64 9.3/10.2,
// 1x14x14x672 7.7/10.0; fewer than 4 gain nothing, 32x16x16x128 7.1 with 4 and 8.3 with 2.
template <typename T, int VEC, int MOST_R>
bool whole_of(const Shape& s, Whole& out) {
  const int64_t unit = std::lcm((int64_t)s.cg, (int64_t)VEC), line = sizeof(T) * unit;
  if ((int64_t)s.S * s.C * sizeof(T) >= (int64_t(1) << 30) || unit / VEC > 256) return false;   // offsets: 32 bits
  // at most 2048 channels a workgroup: their constants share LDS with the threads' sums (131 KB backward)
  const int64_t units = s.C / unit, sixteen = 16 / sizeof(T), most = std::max<int64_t>(1, 2048 / unit);
  auto vectors = [&](int64_t k) { return k * unit * s.S / sixteen; };
  auto workgroups = [&](int64_t k) { return s.B * ((units + k - 1) / k); };
  auto lines = [&](int64_t bytes) { return std::min(units, std::max<int64_t>(1, bytes / line)); };
  int64_t k = std::min({units, most, std::max(lines(64), 2048 / std::max<int64_t>(1, vectors(1)))});
  for (int bytes : {128, 64, 32})
    while (k > lines(bytes) && workgroups(k) < 8 * bytes) k = std::max(lines(bytes), k / 2);
  if (vectors(k) > 4096) {
    k = lines(32);
    if (vectors(k) > 8192 || workgroups(k) < 256 || workgroups(k) > 768) return false;
  }
  out.tile = (int)(k * unit);
  out.ntile = (int)((units + k - 1) / k);
  if (workgroups(k) >= (int64_t(1) << 22)) return false;
  const int most_r = workgroups(k) <= 512 ? std::min(MOST_R, 4) : MOST_R;
  for (int threads : {256, 512, 1024})
    for (out.r = 1; out.r <= (threads < 1024 ? most_r : MOST_R); out.r *= 2) {
      out.threads = (int)((((int64_t)s.S + out.r - 1) / out.r * (out.tile / VEC) + 63) / 64 * 64);
      if (out.threads <= threads) return true;
    }
  return false;
}

// f(r as a constant), r a power of 2 up to MOST
template <int MOST, typename F>
void by_r(int r, F f) {
  if constexpr (MOST > 1) {
    if (r < MOST) return by_r<MOST / 2>(r, f);
  }
  f(std::integral_constant<int, MOST>{});
}
// f(values a load): 16 bytes, or 8 where 16 do not divide a line of channels, or where whole groups of whole
// 16 bytes are too much for a workgroup and those of 8 are less (EfficientNet's 84 channels a group, 100x14x14x672:
// 20 + 29 us with 8 bytes, 20 + 39 with 16); single values where neither divides it
template <typename T, typename F>
void by_vec(const Shape& s, bool aligned, F f) {
  constexpr int V = 16 / sizeof(T);
  if constexpr (V == 8) {
    const int64_t u8 = std::lcm((int64_t)s.cg, (int64_t)8), u4 = std::lcm((int64_t)s.cg, (int64_t)4);
    if (aligned && s.C % 4 == 0 && (s.C % 8 != 0 || (u4 < u8 && u8 * s.S > 2048 * 8)))
      return f(std::integral_constant<int, 4>{});
  }
  if (aligned && s.C % V == 0) f(std::integral_constant<int, V>{});
  else f(std::integral_constant<int, 1>{});
}

// vectors a thread: as many as registers hold without spilling
template <typename T, int VEC> constexpr int kForwardR = VEC == 1 ? 32 : 16;
template <typename T, int VEC> constexpr int kBackwardR = VEC == 1 ? 32 : (VEC * sizeof(T) == 8 ? 16 : 8);

constexpr int kR = 8;       // vectors a thread in a chunk

// groups that one workgroup joins: lines of 32 channels, 128 bytes
int join_groups(const Shape& s) { return std::min(s.G, std::max(1, 32 / s.cg)); }

template <typename T, int VEC>
void forward_on(const Shape& s, const torch::Tensor& x, const void* w, const void* b, bool f32,
             torch::Tensor& y, torch::Tensor& mean, torch::Tensor& rstd, double eps, int act,
             hipStream_t stream) {
  Whole p;
  if (whole_of<T, VEC, kForwardR<T, VEC>>(s, p)) {
    const size_t lds = (2 * (size_t)p.threads * VEC + 8 + (kCentred<T> ? 5 : 4) * p.tile) * sizeof(float);
    auto go = [&](auto kern) {
      hipLaunchKernelGGL(kern, dim3((unsigned)(s.B * p.ntile)), dim3(p.threads), lds, stream,
                         (const T*)x.data_ptr(), w, b, f32, (T*)y.data_ptr(), mean.data_ptr<float>(),
                         rstd.data_ptr<float>(), s.S, s.C, s.cg, p.tile, p.ntile, act, (float)eps);
    };
    by_r<kForwardR<T, VEC>>(p.r, [&](auto r) { go(gn_whole_fwd_kernel<T, VEC, r.value>); });
    return;
  }
  const Chunks c = chunks_of<VEC>(s, kR);
  auto ws = torch::empty({s.B * c.nchunk * 2 * s.C}, mean.options());
  const size_t lds = (2 * 256 * VEC + 8 + 2 * c.tile) * sizeof(float);
  hipLaunchKernelGGL((gn_chunk_stats_kernel<T, VEC, kR>), dim3((unsigned)c.wgs), dim3(256), lds, stream,
                     (const T*)x.data_ptr(), ws.data_ptr<float>(), s.S, s.C, s.cg, c.tile, c.ntile,
                     c.nchunk, c.chunk);
  const int gt = join_groups(s);
  hipLaunchKernelGGL((gn_join_stats_kernel<T>), dim3((unsigned)(s.B * ((s.G + gt - 1) / gt))), dim3(256),
                     (2 * gt * s.cg + 768) * sizeof(float), stream, (const T*)x.data_ptr(), ws.data_ptr<float>(),
                     mean.data_ptr<float>(), rstd.data_ptr<float>(), s.S, s.C, s.cg, gt, c.nchunk, c.chunk,
                     (float)eps);
  hipLaunchKernelGGL((gn_chunk_apply_kernel<T, VEC, kR>), dim3((unsigned)c.wgs), dim3(256),
                     2 * c.tile * sizeof(float), stream, (const T*)x.data_ptr(), w, b, f32, mean.data_ptr<float>(), rstd.data_ptr<float>(),
                     (T*)y.data_ptr(), s.S, s.C, s.cg, c.tile, c.ntile, c.nchunk, c.chunk, act);
}

// returns the samples' sums, which the parameters' gradients are made of
template <typename T, int VEC>
torch::Tensor backward_on(const Shape& s, const torch::Tensor& dy, const torch::Tensor& x, const void* w,
                       const void* b, bool f32, const torch::Tensor& mean, const torch::Tensor& rstd,
                       torch::Tensor& dx, int act, hipStream_t stream) {
  auto sample = torch::empty({s.B, 2 * (int64_t)s.C}, mean.options());
  Whole p;
  if (whole_of<T, VEC, kBackwardR<T, VEC>>(s, p)) {
    const size_t lds = (2 * (size_t)p.threads * VEC + 8 * p.tile) * sizeof(float);
    auto go = [&](auto kern) {
      hipLaunchKernelGGL(kern, dim3((unsigned)(s.B * p.ntile)), dim3(p.threads), lds, stream,
                         (const T*)dy.data_ptr(), (const T*)x.data_ptr(), w, b, f32,
                         mean.data_ptr<float>(), rstd.data_ptr<float>(), (T*)dx.data_ptr(),
                         sample.data_ptr<float>(), s.S, s.C, s.cg, p.tile, p.ntile, act);
    };
    by_r<kBackwardR<T, VEC>>(p.r, [&](auto r) { go(gn_whole_bwd_kernel<T, VEC, r.value>); });
    return sample;
  }
  const Chunks c = chunks_of<VEC>(s, kR);
  auto ws = torch::empty({s.B * c.nchunk, 2 * (int64_t)s.C}, mean.options());
  auto means = torch::empty({s.B * s.G * 2}, mean.options());
  const size_t lds = (2 * 256 * VEC + 6 * c.tile) * sizeof(float);
  hipLaunchKernelGGL((gn_chunk_grads_kernel<T, VEC, kR, 4>), dim3((unsigned)c.wgs), dim3(256), lds, stream,
                     (const T*)dy.data_ptr(), (const T*)x.data_ptr(), w, b, f32,
                     mean.data_ptr<float>(), rstd.data_ptr<float>(), ws.data_ptr<float>(), s.S, s.C,
                     s.cg, c.tile, c.ntile, c.nchunk, c.chunk, act);
  const int gt = join_groups(s);
  hipLaunchKernelGGL((gn_join_grads_kernel<T>), dim3((unsigned)(s.B * ((s.G + gt - 1) / gt))), dim3(256),
                     (2 * gt * s.cg + 512) * sizeof(float), stream, ws.data_ptr<float>(), w, f32,
                     means.data_ptr<float>(), sample.data_ptr<float>(), s.S, s.C, s.cg, gt, c.nchunk);
  hipLaunchKernelGGL((gn_chunk_dx_kernel<T, VEC, kR, 4>), dim3((unsigned)c.wgs), dim3(256),
                     (kCentred<T> ? 5 : 4) * c.tile * sizeof(float), stream,
                     (const T*)dy.data_ptr(), (const T*)x.data_ptr(), w, b, f32,
                     mean.data_ptr<float>(), rstd.data_ptr<float>(), means.data_ptr<float>(),
                     (T*)dx.data_ptr(), s.S, s.C, s.cg, c.tile, c.ntile, c.nchunk, c.chunk, act);
  return sample;
}

class GroupNormAct : public torch::autograd::Function<GroupNormAct> {
 public:
  // x: [N, C, ...] of any order
  static torch::Tensor forward(torch::autograd::AutogradContext* ctx, torch::Tensor x, int64_t groups,
                               c10::optional<torch::Tensor> weight, c10::optional<torch::Tensor> bias,
                               double eps, int64_t act) {
    const c10::OptionalDeviceGuard guard(x.device());
    auto rows = channels_last(x);
    auto w = weight ? weight->contiguous() : torch::Tensor(), b = bias ? bias->contiguous() : torch::Tensor();
    const Shape s = shape_of(rows, groups, w, b, act);
    auto y = at::empty_strided(rows.sizes(), rows.strides(), rows.options());
    auto stat = x.options().dtype(torch::kFloat32);
    auto mean = torch::empty({s.B, s.G}, stat), rstd = torch::empty({s.B, s.G}, stat);
    if (x.numel() > 0) {
      auto stream = at::hip::getCurrentHIPStream().stream();
      by_type(x.scalar_type(), [&](auto z) {
        using T = decltype(z);
        by_vec<T>(s, aligned16({&rows, &y}), [&](auto v) {
          forward_on<T, v.value>(s, rows, data(w), data(b), is_f32(w, b), y, mean, rstd, eps, (int)act, stream);
        });
      });
    }
    C10_HIP_KERNEL_LAUNCH_CHECK();
    ctx->saved_data["how"] = groups * 4 + act;
    ctx->save_for_backward({rows, w, b, mean, rstd});
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const bool again = at::GradMode::is_enabled();
    auto saved = ctx->get_saved_variables();
    const auto &x = saved[0], &w = saved[1], &b = saved[2], &mean = saved[3], &rstd = saved[4];
    const int64_t how = ctx->saved_data["how"].toInt();
    const int act = (int)(how % 4);
    const c10::OptionalDeviceGuard guard(x.device());
    auto stream = at::hip::getCurrentHIPStream().stream();
    // absent tensors are not counted among the inputs
    const bool nw = w.defined() && ctx->needs_input_grad(1),
               nb = b.defined() && ctx->needs_input_grad(w.defined() ? 2 : 1);
    torch::Tensor dx, dw, db;
    {
      at::NoGradGuard off;
      const Shape s = shape_of(x, how / 4, w, b, act);
      auto dy = channels_last(grads[0]);
      dx = at::empty_strided(x.sizes(), x.strides(), x.options());
      auto popt = (w.defined() ? w : b.defined() ? b : mean).options();
      if (nw || nb) {
        dw = torch::empty({s.C}, popt);
        db = torch::empty({s.C}, popt);
      }
      if (x.numel() == 0) {
        if (nw || nb) {
          dw.zero_();
          db.zero_();
        }
      } else {
        torch::Tensor sums;
        by_type(x.scalar_type(), [&](auto z) {
          using T = decltype(z);
          by_vec<T>(s, aligned16({&x, &dy, &dx}), [&](auto v) {
            sums = backward_on<T, v.value>(s, dy, x, data(w), data(b), is_f32(w, b), mean, rstd, dx, act, stream);
          });
        });
        if (nw || nb)
          by_type(dw.scalar_type(), [&](auto z) {
            using W = decltype(z);
            const unsigned columns = (unsigned)((2 * (int64_t)s.C + 31) / 32);
            int64_t n = sums.size(0);
            if (n > 2048) {       // many small samples: 1024 of them a workgroup first
              const int64_t per = std::max<int64_t>(1024, (n + 32767) / 32768), parts = (n + per - 1) / per;
              auto joined = torch::empty({parts, 2 * (int64_t)s.C}, sums.options());
              hipLaunchKernelGGL((gn_param_grads_kernel<W>), dim3(columns, (unsigned)parts), dim3(1024), 0,
                                 stream, sums.data_ptr<float>(), n, per, s.C, joined.data_ptr<float>(),
                                 (W*)nullptr, (W*)nullptr);
              sums = joined;
              n = parts;
            }
            hipLaunchKernelGGL((gn_param_grads_kernel<W>), dim3(columns), dim3(1024), 0, stream,
                               sums.data_ptr<float>(), n, n, s.C, (float*)nullptr, (W*)dw.data_ptr(),
                               (W*)db.data_ptr());
          });
        C10_HIP_KERNEL_LAUNCH_CHECK();
      }
    }
    torch::autograd::variable_list out{dx, torch::Tensor(), nw ? dw : torch::Tensor(),
                                       nb ? db : torch::Tensor(), torch::Tensor(), torch::Tensor()};
    if (again)      // differentiating these again is an error, not a zero
      for (auto& g : out)
        if (g.defined()) {
          auto err = std::make_shared<torch::autograd::DelayedError>(
              "group_norm_act is differentiable once", 1);
          g = (*err)({g.detach().requires_grad_(true)})[0];
        }
    return out;
  }
};

}  // namespace

torch::Tensor group_norm_act(torch::Tensor x, int64_t groups, c10::optional<torch::Tensor> weight,
                             c10::optional<torch::Tensor> bias, double eps, int64_t act) {
  return GroupNormAct::apply(x, groups, weight, bias, eps, act);
}
