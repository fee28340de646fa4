// Matrix products with bias, residual and activation in their epilogue, and their gradients.
//
//   y  = act(z),  z = x W^T + b + r           x [M,K], W [N,K], b [N], r [M,N]
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum dz,  dr = dz
//
// One kernel computes D[m][n] = sum_k P(m,k) Q(n,k) for 16-bit types, where each
// operand lies either with k contiguous (x and W forward) or with its rows
// contiguous (W for dx; dz and x for dW): no transposed copy is made. A
// workgroup of 4 waves owns a BM x BN tile and steps through k by 64; the next
// step's pieces go from memory to LDS by themselves (buffer loads that write
// LDS, zero outside the operand) while this one's are multiplied. Operands with
// contiguous rows are turned on their way out of LDS (ds_read_b64_tr_b16). The
// roles in the matrix instruction are swapped (its rows are n) and its rows are
// dealt to n so that a lane ends with 8 neighbouring columns of an output row:
// 16-byte loads of the residual and stores of the result.
//
// A long k with few output tiles (dW: k is the batch's pixels) is split over
// workgroups; parts go to a workspace in fp32 and are added in a fixed order by
// a second kernel, which also has the epilogue.
//
// Operands whose lines do not start at 16 bytes are first copied into lines
// that do, which costs less than loads of 2 bytes in the product.
//
// The models' products are bound by memory: 100352x128x512 with residual and
// relu takes 60 us for 231 MB, 3.9 TB/s (a copy reaches 4.9; with two steps of k
// a workgroup's load, product and store hardly overlap). 25088x1024x256 trained
// takes 24 + 28 + 27 us (y, dx, dW) and 15 for dz and its sums. Results that are
// turned in LDS, to leave as lines of 128 bytes, took 98.7 us for 104.6
// (401408x64x256 with residual), but 40.6 for 35.1 (100352x128x512 without).
// Stores past the caches are faster for a product alone (59 us for 63 a call), but
// what reads the result next pays for them: 25088x1024x256 and a product back
// 53 for 47.
// Products of a few hundred rows take 3 to 6 us, which is a launch.
//
// Swish and sigmoid keep their slope in fp32 for the backward pass, and dz enters
// its products as two numbers of 16 bits: the gradients of 128x1152x48 in bf16 are
// then off by the rounding of the results alone (0.0019 of their norm, 0.0024 with a
// sum and a dz of 16 bits). That is 10 bytes more a value of the result to write and
// read, in all passes: 128x1152x48 trained takes 80 us for 78, where a launch counts,
// 25088x1024x256 126 for 92 and 100352x128x512 340 for 213, where memory does.

#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <hip/hip_fp16.h>
#include <type_traits>
#include "faa_common.h"

namespace {

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SWISH = 2, ACT_SIGMOID = 3 };

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

constexpr int BK = 64;

// ------------------------------------------------------------ types

template <typename T> struct Num;
template <> struct Num<float> {
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};
template <> struct Num<__hip_bfloat16> {
  typedef __hip_bfloat16 T;
  static __device__ __forceinline__ float get(const T* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void put(T* p, float v) { *p = __float2bfloat16(v); }
  static __device__ __forceinline__ float of(short u) { return __uint_as_float((uint32_t)(uint16_t)u << 16); }
  static __device__ __forceinline__ short bits(float v) {
    __hip_bfloat16 h = __float2bfloat16(v);
    return *(short*)&h;
  }
  static constexpr float kSecond = 1.0f;      // see Operand::second
  static __device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Num<__half> {
  typedef __half T;
  static __device__ __forceinline__ float get(const T* p) { return __half2float(*p); }
  static __device__ __forceinline__ void put(T* p, float v) { *p = __float2half(v); }
  static __device__ __forceinline__ float of(short u) { return __half2float(__ushort_as_half((unsigned short)u)); }
  static __device__ __forceinline__ short bits(float v) { return (short)__half_as_ushort(__float2half(v)); }
  static constexpr float kSecond = 2048.0f;   // what is left of a value with half a step of error: fp16 has its bits
  static __device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

// 4 neighbours of a row that has `left` of them
template <typename T>
__device__ __forceinline__ f32x4 load4(const T* p, int left, bool vec) {
  f32x4 v = {0, 0, 0, 0};
  if (vec && left >= 4) {
    if constexpr (sizeof(T) == 4) {
      v = *(const f32x4*)p;
    } else {
      s16x4 u = *(const s16x4*)p;
      #pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = Num<T>::of(u[i]);
    }
    return v;
  }
  #pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) v[i] = Num<T>::get(p + i);
  return v;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int left, bool vec, f32x4 v) {
  if (vec && left >= 4) {
    if constexpr (sizeof(T) == 4) {
      *(f32x4*)p = v;
    } else {
      s16x4 u;
      #pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = Num<T>::bits(v[i]);
      *(s16x4*)p = u;
    }
    return;
  }
  #pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) Num<T>::put(p + i, v[i]);
}

// exp2 without the range handling of expf: what it would give below 2^-126 is nothing next to 1
__device__ __forceinline__ float sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if (ACT == ACT_RELU) return z < 0.0f ? 0.0f : z;      // a NaN stays one
  if (ACT == ACT_SWISH) return z * sigmoid(z);
  if (ACT == ACT_SIGMOID) return sigmoid(z);
  return z;
}
// activations whose slope is kept for the backward pass
template <int ACT> constexpr bool kept = ACT == ACT_SWISH || ACT == ACT_SIGMOID;
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  const float s = sigmoid(z);
  return ACT == ACT_SWISH ? s + s * (z - z * s) : s - s * s;
}
// f(activation as a constant): one branch outside the loops, not one an element
template <bool ANY = true, typename F>
__device__ __forceinline__ void by_act(int act, F f) {
  if constexpr (!ANY) return f(std::integral_constant<int, ACT_NONE>{});
  if (act == ACT_SWISH) f(std::integral_constant<int, ACT_SWISH>{});
  else if (act == ACT_RELU) f(std::integral_constant<int, ACT_RELU>{});
  else if (act == ACT_SIGMOID) f(std::integral_constant<int, ACT_SIGMOID>{});
  else f(std::integral_constant<int, ACT_NONE>{});
}

typedef __attribute__((ext_vector_type(8))) float f32x8;

template <typename T>
__device__ __forceinline__ f32x8 widen8(s16x8 u) {
  f32x8 v;
  #pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = Num<T>::of(u[i]);
  return v;
}

// ------------------------------------------------------------ epilogue

template <typename T>
struct Epilogue {
  const T* bias;      // [N] or null
  const T* res;       // [M,N] or null
  T* y;               // [M,N]
  float* slope;       // [M,N] or null: the activation's slope, for the backward pass. It is made of the sum in 32 bits:
                      // a sum held in 16 would be infinite beyond fp16's range, and cost the slope |z| 2^-9 in bf16
  int act;
  bool vec;           // rows of 4 (8 in 16 bits) may be read and written at once

  // 4 columns from n of row m
  template <int ACT>
  __device__ __forceinline__ void four(int64_t m, int n, int N, f32x4 v) const {
    const int left = N - n;
    if (left <= 0) return;
    const int64_t at = m * N + n;
    if (bias) v += load4(bias + n, left, vec);
    if (res) v += load4(res + at, left, vec);
    if constexpr (kept<ACT>)
      if (slope) {
        f32x4 d;
        #pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = act_slope<ACT>(v[i]);
        store4(slope + at, left, vec, d);
      }
    #pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = act_value<ACT>(v[i]);
    store4(y + at, left, vec, v);
  }
  // 8 columns, 16 bytes at once; bias and residual are in v
  template <int ACT>
  __device__ __forceinline__ void eight(int64_t at, f32x8 v) const {
    if constexpr (kept<ACT>)
      if (slope) {
        f32x4 d[2];
        #pragma unroll
        for (int e = 0; e < 8; ++e) d[e >> 2][e & 3] = act_slope<ACT>(v[e]);
        *(f32x4*)(slope + at) = d[0];
        *(f32x4*)(slope + at + 4) = d[1];
      }
    s16x8 out;
    #pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = Num<T>::bits(act_value<ACT>(v[e]));
    *(s16x8*)(y + at) = out;
  }
};

// ------------------------------------------------------------ operands

// P(row, k): row-major with k contiguous, or (ROWS) k-major with rows contiguous. Lines start at 16 bytes.
// An fp32 operand is the sum of two in 16 bits: itself rounded, and `second` bytes further what that left over, times
// kSecond. The product of both terms is exact to 2^-16 (bf16) or 2^-22 (fp16) of every value, at twice the steps.
struct Operand {
  const short* p;
  int rows, kdim;
  int64_t ld;         // a multiple of 8
  int64_t second;
};

// A tile of B rows and 64 k in LDS, pieces of 16 bytes, one after another as lanes load them: which piece of
// the operand a place holds is turned, so that what one instruction reads lies on different banks.
// k contiguous: row r has 8 places; place q holds piece q ^ key(r), and the 8 rows that are read together have
// 8 keys: neighbours (DEALT false), or 0-3 and 8-11 of every 16 (the rows of a dealt fragment).
// rows contiguous: line k has B/8 places. The transposing read of one instruction touches lines {0..3} + 8g
// (g = 0..3): pairs of pieces are moved by the line.
template <int B, bool ROWS, bool DEALT>
struct Lds {
  static constexpr int kPieces = B * BK / 8;
  static __device__ __forceinline__ int key(int row) {
    return DEALT ? (row & 3) | ((row >> 1) & 4) : row & 7;
  }
  static __device__ __forceinline__ int turn(int k) { return ((k & 3) | ((k >> 1) & 4)) & (B / 16 - 1); }
  // what the place c holds
  static __device__ __forceinline__ void held(int c, int& row, int& k) {
    if (ROWS) {
      const int p = c % (B / 8);
      k = c / (B / 8);
      row = (((p >> 1) ^ turn(k)) * 2 + (p & 1)) * 8;
    } else {
      row = c / 8;
      k = ((c % 8) ^ key(row)) * 8;
    }
  }
  // Fragment j of 16 rows of a wave's tile that starts at row0, 32 k from k0: lane i = lane%16 has k
  // (lane/16)*8 .. +7 of row i of the fragment. Fragments are 16 neighbouring rows, or (DEALT) of 32 rows
  // those 8a + 4(j%2) + b for row i = 4a + b: two fragments' results are then 8 neighbours a lane.
  static __device__ __forceinline__ s16x8 fragment(const short* lds, int row0, int j, int k0, int lane) {
    const int i = lane & 15;
    if (!ROWS) {
      const int row = DEALT ? row0 + (j >> 1) * 32 + (i >> 2) * 8 + (j & 1) * 4 + (i & 3) : row0 + j * 16 + i;
      const int q = k0 / 8 + (lane >> 4);
      return *(const s16x8*)(lds + row * BK + ((q ^ key(row)) * 8));
    }
    // lane i of 16 addresses 4 rows (i%4) of line i/4 and is given row i of the 4 lines
    const int k = k0 + (lane >> 4) * 8 + (i >> 2);
    const int row = DEALT ? row0 + (j >> 1) * 32 + (i & 3) * 8 + (j & 1) * 4 : row0 + j * 16 + (i & 3) * 4;
    typedef __attribute__((address_space(3))) s16x4* lds4;
    auto word = [&](int kk) { return lds + kk * B + (((row >> 4) ^ turn(kk)) << 4) + (row & 15); };
    s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)word(k));
    s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)word(k + 4));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// Pieces of a tile on their way to LDS: N a thread
template <int B, bool ROWS, bool DEALT, int THREADS>
struct Loader {
  typedef Lds<B, ROWS, DEALT> L;
  static constexpr int N = L::kPieces / THREADS;
  const char* base;
  int64_t left;         // bytes from base to the operand's end
  uint32_t off[N];      // where a piece starts; out of any range for rows that are not there
  int k[N];
  int kdim;
  int64_t line;         // bytes from one k to the next where rows are contiguous

  __device__ __forceinline__ Loader(const Operand& o, int row0, int tid) {
    const int64_t start = ROWS ? row0 : row0 * o.ld;
    base = (const char*)(o.p + start);
    left = ((int64_t)(ROWS ? o.kdim : o.rows) * o.ld - start) * 2;
    kdim = o.kdim;
    line = o.ld * 2;
    #pragma unroll
    for (int i = 0; i < N; ++i) {
      int row, kk;
      L::held(tid + i * THREADS, row, kk);
      k[i] = kk;
      off[i] = ROWS ? (uint32_t)(kk * o.ld + row) * 2 : (uint32_t)(row * o.ld + kk) * 2;
      if (row0 + row >= o.rows) off[i] = 0xffffffffu;
    }
  }
  // The pieces of k0 .. k0+63 to lds, of the operand or of one `second` bytes further. Reads behind the operand's end give zeros; so do k that are not there, and
  // all of a step that is not wanted: none of these touches memory.
  __device__ __forceinline__ void operator()(int k0, bool wanted, short* lds, int wave, int64_t second = 0) const {
    const int64_t skip = ROWS ? k0 * line : (int64_t)k0 * 2;
    const int64_t rest = wanted ? left - skip : 0;
    const uint32_t bytes = rest > 0xfffffff0ll ? 0xfffffff0u : (uint32_t)rest;
    auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(base + skip + second), 0, bytes, 0x00020000);
    typedef __attribute__((address_space(3))) void* lds_t;
    #pragma unroll
    for (int i = 0; i < N; ++i) {
      uint32_t at = off[i];
      if (!ROWS && k0 + k[i] >= kdim) at = 0xffffffffu;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_t)(lds + (i * THREADS + wave * 64) * 8), 16, at, 0, 0, 0);
    }
  }
};

// Workgroups that share operand rows run one after another on one XCD and find them in its L2.
__device__ __forceinline__ uint32_t xcd_order(uint32_t wg, uint32_t n) {
  const uint32_t q = n / 8, rem = n % 8, xcd = wg % 8, i = wg / 8;
  return xcd < rem ? xcd * (q + 1) + i : rem * (q + 1) + (xcd - rem) * q + i;
}

// ------------------------------------------------------------ the product in 16 bits

// Operands with contiguous rows are those of the gradients, which have no bias, residual or activation.
// TWO: P has two terms. Every step is taken twice, with what is left over (even) and with the rounded values (odd): the
// second finds its piece of Q in the L2. A pass for each took 131 us for 126 at 25088x1024x256 trained.
template <typename T, bool PR, bool QR, int BM, int BN, bool TWO>
__global__ __launch_bounds__(256, 2) void product_kernel(Operand P, Operand Q, Epilogue<T> epi,
                                                      float* __restrict__ part, int tiles_m,
                                                      int tiles_n, int splits) {
  constexpr int FM = BM / 32, FN = BN / 32;         // fragments of a wave: 2 x 2 waves
  typedef Loader<BM, PR, false, 256> LP;
  typedef Loader<BN, QR, true, 256> LQ;
  // two buffers, named apart: what fills one is then known not to touch the other
  __shared__ __align__(16) short p0[BM * BK], p1[BM * BK], q0[BN * BK], q1[BN * BK];
  const uint32_t id = xcd_order(blockIdx.x, gridDim.x), id_m = id / (uint32_t)tiles_n,
                 sp = id_m / (uint32_t)tiles_m;
  const int tn = (int)(id - id_m * tiles_n), tm = (int)(id_m - sp * tiles_m);
  const int m0 = tm * BM, n0 = tn * BN;
  const int steps = (P.kdim + BK - 1) / BK;
  const int s0 = (int)((int64_t)steps * sp / splits) * (TWO ? 2 : 1),
            s1 = (int)((int64_t)steps * (sp + 1) / splits) * (TWO ? 2 : 1);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
  const int M = P.rows, N = Q.rows;
  const LP load_p(P, m0, tid);
  const LQ load_q(Q, n0, tid);

  f32x4 acc[FM][FN], left[TWO ? FM : 1][TWO ? FN : 1];
  #pragma unroll
  for (int i = 0; i < FM; ++i)
    #pragma unroll
    for (int j = 0; j < FN; ++j) {
      acc[i][j] = f32x4{0, 0, 0, 0};
      if constexpr (TWO) left[i][j] = acc[i][j];
    }

  auto fill = [&](int s, short* p, short* q) {
    if constexpr (TWO) {
      load_p(s / 2 * BK, s < s1, p, wave, s % 2 == 0 ? P.second : 0);
      load_q(s / 2 * BK, s < s1, q, wave);
    } else {
      load_p(s * BK, s < s1, p, wave);
      load_q(s * BK, s < s1, q, wave);
    }
  };
  // The older of two steps' pieces have come, here and in the other waves. Loads end in order and every step
  // asks for as many, so a count says so; other loads in flight only make it stricter.
  auto come = [] { asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"(LP::N + LQ::N) : "memory"); };
  // all waves have read their fragments: the buffer may be filled again
  auto read = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  auto add = [&](const short* p, const short* q, auto& acc) {
    #pragma unroll
    for (int k = 0; k < BK; k += 32) {
      s16x8 fp[FM], fq[FN];
      #pragma unroll
      for (int j = 0; j < FN; ++j) fq[j] = LQ::L::fragment(q, wn, j, k, lane);
      #pragma unroll
      for (int i = 0; i < FM; ++i) fp[i] = LP::L::fragment(p, wm, i, k, lane);
      #pragma unroll
      for (int i = 0; i < FM; ++i)
        #pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = Num<T>::mfma(fq[j], fp[i], acc[i][j]);
    }
  };
  auto multiply = [&](const short* p, const short* q) { add(p, q, acc); };
  // the first buffers have even steps; in bf16, where nothing is scaled, both kinds share their sums
  auto multiply_even = [&](const short* p, const short* q) {
    if constexpr (TWO && Num<T>::kSecond != 1.0f) add(p, q, left);
    else add(p, q, acc);
  };
  const int mine = n0 + wn + (lane >> 4) * 8;       // the lane's first column
  // the residual is on its way during the product; where there is none to read at once, zeros are read from nowhere
  typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
  u32x4 res[FM][FN / 2];
  if constexpr (!PR && !QR) {
    const int64_t rest = splits == 1 && epi.vec && epi.res ? ((int64_t)M - m0) * N * 2 : 0;
    auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(epi.res + (int64_t)m0 * N), 0,
                                                  rest > 0xfffffff0ll ? 0xfffffff0u : (uint32_t)rest, 0x00020000);
    #pragma unroll
    for (int i = 0; i < FM; ++i)
      #pragma unroll
      for (int j = 0; j < FN; j += 2) {
        const uint32_t at = (uint32_t)((wm + i * 16 + (lane & 15)) * N + mine + j * 16) * 2;
        res[i][j / 2] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, mine + j * 16 < N ? at : 0xffffffffu, 0, 0);
      }
  }
  fill(s0, p0, q0);
  fill(s0 + 1, p1, q1);
  int s = s0;
  for (; s + 2 < s1; s += 2) {
    come();
    multiply_even(p0, q0);
    read();
    fill(s + 2, p0, q0);
    come();
    multiply(p1, q1);
    read();
    fill(s + 3, p1, q1);
  }
  if (s < s1) {     // one or two steps are left; no others are asked for
    come();
    multiply_even(p0, q0);
  }
  asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  if (s + 1 < s1) multiply(p1, q1);
  if constexpr (TWO && Num<T>::kSecond != 1.0f) {
    #pragma unroll
    for (int i = 0; i < FM; ++i)
      #pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] += left[i][j] * (1.0f / Num<T>::kSecond);
  }

  // lane: output row lane%16 of a fragment; of fragments j, j+1 columns (lane/16)*8 + 0..3 and + 4..7
  auto each = [&](auto f) {
    #pragma unroll
    for (int j = 0; j < FN; j += 2) {
      const int n = mine + j * 16;
      if (n >= N) continue;
      #pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int64_t m = (int64_t)m0 + wm + i * 16 + (lane & 15);
        if (m < M) f(m, n, i, j);
      }
    }
  };
  if (splits > 1) {
    each([&](int64_t m, int n, int i, int j) {
      float* to = part + ((int64_t)sp * M + m) * N + n;
      store4(to, N - n, epi.vec, acc[i][j]);
      store4(to + 4, N - n - 4, epi.vec, acc[i][j + 1]);
    });
  } else if (epi.vec) {
    f32x8 bias[FN / 2];
    #pragma unroll
    for (int j = 0; j < FN; j += 2)
      bias[j / 2] = !PR && !QR && epi.bias && mine + j * 16 < N ? widen8<T>(*(const s16x8*)(epi.bias + mine + j * 16)) : f32x8{};
    by_act<!PR && !QR>(epi.act, [&](auto A) {
      each([&](int64_t m, int n, int i, int j) {
        f32x8 v = __builtin_shufflevector(acc[i][j], acc[i][j + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        if constexpr (!PR && !QR) v += widen8<T>(__builtin_bit_cast(s16x8, res[i][j / 2]));
        epi.template eight<A.value>(m * N + n, v + bias[j / 2]);
      });
    });
  } else {
    by_act<!PR && !QR>(epi.act, [&](auto A) {
      each([&](int64_t m, int n, int i, int j) {
        epi.template four<A.value>(m, n, N, acc[i][j]);
        epi.template four<A.value>(m, n + 4, N, acc[i][j + 1]);
      });
    });
  }
}

// Few outputs: 32 x 32 of them a workgroup, and its 4 waves take every fourth step of k each, with buffers of their
// own and no barrier between them; their sums meet in LDS at the end. One launch where the large tiles would have
// to be split over workgroups and joined.
template <typename T, bool PR, bool QR, bool TWO>
__global__ __launch_bounds__(256) void small_product_kernel(Operand P, Operand Q, Epilogue<T> epi, int tiles_n) {
  constexpr int B = 32;
  typedef Loader<B, PR, false, 64> LP;
  typedef Loader<B, QR, true, 64> LQ;
  __shared__ __align__(16) short p0[4][B * BK], p1[4][B * BK], q0[4][B * BK], q1[4][B * BK];
  const uint32_t tm = blockIdx.x / (uint32_t)tiles_n;
  const int m0 = (int)tm * B, n0 = (int)(blockIdx.x - tm * tiles_n) * B;
  const int steps = (P.kdim + BK - 1) / BK * (TWO ? 2 : 1);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const LP load_p(P, m0, lane);
  const LQ load_q(Q, n0, lane);
  f32x4 acc[2][2];
  #pragma unroll
  for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = f32x4{0, 0, 0, 0};
  auto fill = [&](int s, short* p, short* q) {
    if constexpr (TWO) {      // see product_kernel: waves 0 and 2 have what is left over, 1 and 3 the rounded values
      load_p(s / 2 * BK, s < steps, p, 0, s % 2 == 0 ? P.second : 0);
      load_q(s / 2 * BK, s < steps, q, 0);
    } else {
      load_p(s * BK, s < steps, p, 0);
      load_q(s * BK, s < steps, q, 0);
    }
  };
  // the older of two steps' pieces have come (see product_kernel); fragments are read, and may be overwritten
  auto come = [] { asm volatile("s_waitcnt vmcnt(%0)" ::"i"(LP::N + LQ::N) : "memory"); };
  auto read = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
  auto multiply = [&](const short* p, const short* q) {
    #pragma unroll
    for (int k = 0; k < BK; k += 32) {
      s16x8 fp[2], fq[2];
      #pragma unroll
      for (int i = 0; i < 2; ++i) {
        fp[i] = LP::L::fragment(p, 0, i, k, lane);
        fq[i] = LQ::L::fragment(q, 0, i, k, lane);
      }
      #pragma unroll
      for (int i = 0; i < 2; ++i)
        #pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = Num<T>::mfma(fq[j], fp[i], acc[i][j]);
    }
  };
  fill(wave, p0[wave], q0[wave]);
  fill(wave + 4, p1[wave], q1[wave]);
  for (int s = wave; s < steps; s += 8) {
    come();
    multiply(p0[wave], q0[wave]);
    read();
    fill(s + 8, p0[wave], q0[wave]);
    come();
    multiply(p1[wave], q1[wave]);       // zeros where the step is not there
    read();
    fill(s + 12, p1[wave], q1[wave]);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if constexpr (TWO) {
    const float scale = wave % 2 == 0 ? 1.0f / Num<T>::kSecond : 1.0f;
    #pragma unroll
    for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] *= scale;
  }
  __syncthreads();
  // the waves' sums, 32 lines of 32 and 4 more (a line's start moves by 4 banks)
  constexpr int LD = B + 4;
  __shared__ __align__(16) float sums[4 * B * LD];
  #pragma unroll
  for (int i = 0; i < 2; ++i) {
    float* line = sums + (wave * B + i * 16 + (lane & 15)) * LD + (lane >> 4) * 8;
    *(f32x4*)line = acc[i][0];
    *(f32x4*)(line + 4) = acc[i][1];
  }
  __syncthreads();
  const int row = tid >> 3, col = (tid & 7) * 4, N = Q.rows;
  f32x4 v = {0, 0, 0, 0};
  #pragma unroll
  for (int w = 0; w < 4; ++w) v += *(const f32x4*)(sums + (w * B + row) * LD + col);
  if (m0 + row < P.rows)
    by_act<!PR && !QR>(epi.act, [&](auto A) { epi.template four<A.value>(m0 + row, n0 + col, N, v); });
}

// lines of `from` values into lines of `to`, a multiple of 8, with zeros behind
__global__ __launch_bounds__(256) void widen_lines_kernel(const short* __restrict__ in, short* __restrict__ out,
                                                          int64_t lines, int from, int to) {
  const int pieces = to / 8;
  const int64_t total = lines * pieces;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t l = i / pieces;
    const int c = (int)(i - l * pieces) * 8;
    s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
    #pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < from) v[e] = in[l * from + c + e];
    *(s16x8*)(out + i * 8) = v;
  }
}

// ------------------------------------------------------------ the product in 32 bits

struct OperandF32 {
  const float* p;
  int rows, kdim;
  int64_t ld;
};

// 64 x 64 tiles, 16 k a step; LDS lines hold one k (a lane of the matrix instruction has one k of one row)
template <bool PR, bool QR>
__global__ __launch_bounds__(256) void product_f32_kernel(OperandF32 P, OperandF32 Q,
                                                          Epilogue<float> epi, float* __restrict__ part,
                                                          int tiles_m, int tiles_n, int splits) {
  constexpr int B = 64, K = 16, LD = B + 4;
  __shared__ float lp[2][K][LD], lq[2][K][LD];
  const uint32_t id = xcd_order(blockIdx.x, gridDim.x), id_m = id / (uint32_t)tiles_n,
                 sp = id_m / (uint32_t)tiles_m;
  const int tn = (int)(id - id_m * tiles_n), tm = (int)(id_m - sp * tiles_m);
  const int m0 = tm * B, n0 = tn * B;
  const int steps = (P.kdim + K - 1) / K;
  const int s0 = (int)((int64_t)steps * sp / splits), s1 = (int)((int64_t)steps * (sp + 1) / splits);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  float rp[4], rq[4];
  auto one = [](const OperandF32& o, bool rows, int row, int k) {
    if (row >= o.rows || k >= o.kdim) return 0.0f;
    return rows ? o.p[(int64_t)k * o.ld + row] : o.p[(int64_t)row * o.ld + k];
  };
  auto place = [&](bool rows, int i, int& row, int& k) {
    const int c = tid + i * 256;
    if (rows) { k = c / B; row = c % B; }
    else { row = c / K; k = c % K; }
  };
  auto fetch = [&](int s) {
    int row, k;
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      place(PR, i, row, k);
      rp[i] = one(P, PR, m0 + row, s * K + k);
      place(QR, i, row, k);
      rq[i] = one(Q, QR, n0 + row, s * K + k);
    }
  };
  auto put = [&](int buf) {
    int row, k;
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      place(PR, i, row, k);
      lp[buf][k][row] = rp[i];
      place(QR, i, row, k);
      lq[buf][k][row] = rq[i];
    }
  };
  f32x4 acc[2][2];
  #pragma unroll
  for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = f32x4{0, 0, 0, 0};
  if (s0 < s1) {
    fetch(s0);
    put(0);
    if (s0 + 1 < s1) fetch(s0 + 1);
  }
  __syncthreads();
  for (int s = s0; s < s1; ++s) {
    const int buf = (s - s0) & 1;
    if (s + 1 < s1) {
      put(buf ^ 1);
      if (s + 2 < s1) fetch(s + 2);
    }
    #pragma unroll
    for (int k = 0; k < K; k += 4) {
      float fp[2], fq[2];
      #pragma unroll
      for (int i = 0; i < 2; ++i) {
        fp[i] = lp[buf][k + (lane >> 4)][wm + i * 16 + (lane & 15)];
        fq[i] = lq[buf][k + (lane >> 4)][wn + i * 16 + (lane & 15)];
      }
      #pragma unroll
      for (int i = 0; i < 2; ++i)
        #pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fq[j], fp[i], acc[i][j], 0, 0, 0);
    }
    __syncthreads();
  }
  const int M = P.rows, N = Q.rows;
  by_act(epi.act, [&](auto A) {
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t m = (int64_t)m0 + wm + i * 16 + (lane & 15);
      if (m >= M) continue;
      #pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = n0 + wn + j * 16 + (lane >> 4) * 4;
        if (splits == 1) epi.template four<A.value>(m, n, N, acc[i][j]);
        else if (n < N) store4(part + ((int64_t)sp * M + m) * N + n, N - n, epi.vec, acc[i][j]);
      }
    }
  });
}

// the parts of a split product, added in order, and its epilogue
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ part, Epilogue<T> epi,
                                                   int64_t M, int N, int splits) {
  const int n4 = (N + 3) / 4;
  const int64_t total = M * n4, plane = M * N;
  by_act(epi.act, [&](auto A) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
      const int64_t m = i / n4;
      const int n = (int)(i - m * n4) * 4;
      f32x4 v = {0, 0, 0, 0};
      #pragma unroll 4
      for (int s = 0; s < splits; ++s) v += load4(part + s * plane + m * N + n, N - n, epi.vec);
      epi.template four<A.value>(m, n, N, v);
    }
  });
}

// ------------------------------------------------------------ dz and its column sums

// dz = dy act'(z), unless act is none; sums over a chunk of rows to part[chunk][N], or of all rows to db.
// A thread has VEC columns, a workgroup a tile of columns and a chunk of rows. `of` is what the slope is known from:
// relu's result y, which is above 0 where z is, but for z below half the type's smallest number, or the slope itself.
// Where relu holds back, no infinity or NaN of dy comes through. `left` (or null) is given what dz's rounding left over,
// times kSecond (see Operand): none where dz is infinite.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void slope_kernel(const T* __restrict__ dy, const void* __restrict__ of,
                                                    T* __restrict__ dz, T* __restrict__ left,
                                                    float* __restrict__ part, T* __restrict__ db,
                                                    int64_t M, int N, int tile, int ntile, int chunk,
                                                    int act) {
  __shared__ float lds[256 * VEC];
  const int64_t wg = blockIdx.x;
  const int ti = (int)(wg % ntile);
  const int64_t ck = wg / ntile;
  const int c0 = ti * tile, cols = min(tile, N - c0), cv = cols / VEC, rows = 256 / cv;
  const int r = (int)threadIdx.x / cv, v = (int)threadIdx.x - r * cv;
  const bool on = r < rows;
  const int64_t m0 = ck * chunk, m1 = min(m0 + chunk, M);
  float acc[VEC];
  #pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
  if (on)
    by_act(act, [&](auto A) {
      #pragma unroll 4
      for (int64_t m = m0 + r; m < m1; m += rows) {
        const int64_t at = m * N + c0 + v * VEC;
        constexpr int H = VEC == 1 ? 1 : VEC / 4, E = VEC == 1 ? 1 : 4;
        f32x4 d[H];
        #pragma unroll
        for (int h = 0; h < H; ++h) d[h] = load4(dy + at + 4 * h, E, VEC > 1);
        if constexpr (A.value != ACT_NONE) {
          f32x4 s[H];
          #pragma unroll
          for (int h = 0; h < H; ++h) {
            if constexpr (A.value == ACT_RELU) s[h] = load4((const T*)of + at + 4 * h, E, VEC > 1);
            else s[h] = load4((const float*)of + at + 4 * h, E, VEC > 1);
          }
          #pragma unroll
          for (int h = 0; h < H; ++h) {
            #pragma unroll
            for (int i = 0; i < E; ++i) {
              if constexpr (A.value == ACT_RELU) d[h][i] = s[h][i] <= 0.0f ? 0.0f : d[h][i];
              else d[h][i] *= s[h][i];
            }
            if constexpr (std::is_same<T, __half>::value && A.value != ACT_RELU) {
              // fp16 has an instruction that rounds a product at once: were it taken for one of dz's two uses below,
              // what is left over would be that of another number than the one that is stored
              #pragma unroll
              for (int i = 0; i < E; ++i) {
                float one = d[h][i];
                asm("" : "+v"(one));
                d[h][i] = one;
              }
            }
            store4(dz + at + 4 * h, E, VEC > 1, d[h]);
            if constexpr (sizeof(T) == 2) {
              if constexpr (A.value != ACT_RELU)
                if (left) {
                  f32x4 l;
                  #pragma unroll
                  for (int i = 0; i < E; ++i) {
                    const float held = Num<T>::of(Num<T>::bits(d[h][i]));
                    l[i] = __builtin_isinf(held) ? 0.0f : (d[h][i] - held) * Num<T>::kSecond;
                  }
                  store4(left + at + 4 * h, E, VEC > 1, l);
                }
            }
          }
        }
        #pragma unroll
        for (int h = 0; h < H; ++h)
          #pragma unroll
          for (int i = 0; i < E; ++i) acc[E * h + i] += d[h][i];
      }
    });
  if (!part && !db) return;
  if (on)
    #pragma unroll
    for (int j = 0; j < VEC; ++j) lds[r * cols + v * VEC + j] = acc[j];
  __syncthreads();
  for (int c = threadIdx.x; c < cols; c += 256) {
    float s = 0.0f;
    #pragma unroll 4
    for (int q = 0; q < rows; ++q) s += lds[q * cols + c];
    if (db) Num<T>::put(db + c0 + c, s);
    else part[ck * N + c0 + c] = s;
  }
}

// out[n] = sum over the chunks, 8 columns a workgroup: a few loads a thread
template <typename T>
__global__ __launch_bounds__(1024) void column_join_kernel(const float* __restrict__ part, int64_t chunks,
                                                           int N, T* __restrict__ out) {
  __shared__ float lds[128][9];
  const int col = threadIdx.x & 7, row = threadIdx.x >> 3, n = blockIdx.x * 8 + col;
  float s = 0.0f;
  if (n < N)
    #pragma unroll 4
    for (int64_t r = row; r < chunks; r += 128) s += part[r * N + n];
  lds[row][col] = s;
  __syncthreads();
  #pragma unroll
  for (int w = 64; w >= 8; w >>= 1) {
    if (row < w) lds[row][col] += lds[row + w][col];
    __syncthreads();
  }
  if (row == 0 && n < N) {
    s = 0.0f;
    #pragma unroll
    for (int r = 0; r < 8; ++r) s += lds[r][col];
    Num<T>::put(out + n, s);
  }
}

// ------------------------------------------------------------ host

bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

template <typename F>
void by_type(torch::ScalarType t, F f) {
  if (t == torch::kFloat32) f(float{});
  else if (t == torch::kBFloat16) f(__hip_bfloat16{});
  else if (t == torch::kFloat16) f(__half{});
  else TORCH_CHECK(false, "linear_act: fp32, bf16 and fp16 are taken");
}

// t as an operand; `keep` holds a copy with wider lines where t's do not start at 16 bytes
Operand operand(const torch::Tensor& t, bool rows_contiguous, torch::Tensor& keep, hipStream_t stream) {
  Operand o;
  o.second = 0;
  o.rows = (int)t.size(rows_contiguous ? 1 : 0);
  o.kdim = (int)t.size(rows_contiguous ? 0 : 1);
  o.ld = t.size(1);
  keep = t;
  if (o.ld % 8 != 0 || !aligned(t.data_ptr(), 16)) {
    o.ld = (o.ld + 7) / 8 * 8;
    keep = torch::empty({t.size(0), o.ld}, t.options());
    const int64_t pieces = t.size(0) * o.ld / 8;
    hipLaunchKernelGGL(widen_lines_kernel, dim3((unsigned)std::min<int64_t>((pieces + 255) / 256, 8192)),
                       dim3(256), 0, stream, (const short*)t.data_ptr(), (short*)keep.data_ptr(), t.size(0),
                       (int)t.size(1), (int)o.ld);
  }
  o.p = (const short*)keep.data_ptr();
  return o;
}

// lines of both are equally wide: of one copy or none each, as both start at 16 bytes or neither does
int64_t bytes_between(const Operand& a, const Operand& b) {
  TORCH_CHECK(a.ld == b.ld && a.rows == b.rows && a.kdim == b.kdim, "linear_act: an operand's terms differ in shape");
  return (const char*)b.p - (const char*)a.p;
}

OperandF32 operand_f32(const torch::Tensor& t, bool rows_contiguous) {
  return {t.data_ptr<float>(), (int)t.size(rows_contiguous ? 1 : 0), (int)t.size(rows_contiguous ? 0 : 1),
          t.size(1)};
}

// D[m][n] = sum_k P(m,k) Q(n,k), with the epilogue. TWO: P is p + p_left / kSecond
template <typename T, bool PR, bool QR, bool TWO = false>
void product(const torch::Tensor& p, const torch::Tensor& q, Epilogue<T> epi, hipStream_t stream,
             const torch::Tensor* p_left = nullptr) {
  const int64_t M = p.size(PR ? 1 : 0), N = q.size(QR ? 1 : 0), K = p.size(PR ? 0 : 1);
  constexpr int W = sizeof(T) == 2 ? 8 : 4;
  epi.vec = N % W == 0 && aligned(epi.y, 16) && (!epi.slope || aligned(epi.slope, 16))
            && (!epi.res || aligned(epi.res, 16)) && (!epi.bias || aligned(epi.bias, 16));
  int BM = 64, BN = 64, step = 16;
  if constexpr (sizeof(T) == 2) {
    step = BK;
    // Large tiles read less, small ones fill the card: 128 x 128 or 128 x 64 where there are 384 of them, or where so
    // few (128 x 128) that k is split and a part still has 16 steps. Measured (us, 128x128/128x64/64x64, M x N, K):
    // 25088x256, 1024 (392 tiles of 128x128) 21/24/24; 100352x512, 128 33/35/38; 6272x512, 2048 (196) 24/22/25;
    // 16384x130, 200 (256) 11.0/10.5/9.4; 2048x1000, 1280 (128) 24/12/11; and split, 256x1024, 25088 27/27/35;
    // 2048x512, 6272 27/27/32; 512x128, 100352 46/51/62; but 256x256, 8192 (2 steps) 16/15/11; 256x64, 401408 77/76/69.
    auto tiles = [&](int64_t a, int64_t b) { return ((M + a - 1) / a) * ((N + b - 1) / b); };
    const int64_t large = tiles(128, 128);
    if (M > 64 && N > 64 && (large >= 384 || (large <= 128 && (K + BK - 1) / BK * large >= 16 * 256))) BM = BN = 128;
    else if (M > 64 && tiles(128, 64) >= 384) BM = 128;
  }
  const int64_t tm = (M + BM - 1) / BM, tn = (N + BN - 1) / BN, steps = (K + step - 1) / step;
  // few tiles and a long k: parts for one workgroup a CU, each with 4 steps at least. More parts are more fp32 to
  // write and read again: dW of 25088x1024x256 takes 25 us with 256 workgroups, 27 with 512, 38 with 1024.
  int64_t splits = 1;
  if (tm * tn < 256) splits = std::max<int64_t>(1, std::min<int64_t>(256 / (tm * tn), steps / 4));
  TORCH_CHECK(tm * tn * splits < (int64_t(1) << 24), "linear_act: too many tiles");     // 2^32 threads a launch
  if constexpr (sizeof(T) == 2) {
    // Measured (us, this/large tiles): 128x1152x48 4.5/6.4, 100x1280x1000 4.8/7.5, 512x1280x1000 (512 tiles) 8.7/10.1;
    // but 2048x1280x1000 (2048 tiles) 31/12, k = 6272 for 128x512 17/10, and k = 320 for 512x1280 (640) 7.8/3.9.
    const int64_t sm = (M + 31) / 32, sn = (N + 31) / 32;
    if (tm * tn < 256 && sm * sn <= 512 && steps >= 4 && steps <= 40) {
      torch::Tensor keep_p, keep_q, keep_left;
      Operand P = operand(p, PR, keep_p, stream);
      const Operand Q = operand(q, QR, keep_q, stream);
      if constexpr (TWO) P.second = bytes_between(P, operand(*p_left, PR, keep_left, stream));
      hipLaunchKernelGGL((small_product_kernel<T, PR, QR, TWO>), dim3((unsigned)(sm * sn)), dim3(256), 0, stream, P, Q,
                         epi, (int)sn);
      return;
    }
  }
  torch::Tensor ws;
  float* part = nullptr;
  if (splits > 1) {
    ws = torch::empty({splits * M * N}, p.options().dtype(torch::kFloat32));
    part = ws.data_ptr<float>();
  }
  const dim3 grid((unsigned)(tm * tn * splits)), block(256);
  if constexpr (sizeof(T) == 4) {
    hipLaunchKernelGGL((product_f32_kernel<PR, QR>), grid, block, 0, stream, operand_f32(p, PR),
                       operand_f32(q, QR), epi, part, (int)tm, (int)tn, (int)splits);
  } else {
    torch::Tensor keep_p, keep_q, keep_left;
    Operand P = operand(p, PR, keep_p, stream);
    const Operand Q = operand(q, QR, keep_q, stream);
    if constexpr (TWO) P.second = bytes_between(P, operand(*p_left, PR, keep_left, stream));
    auto go = [&](auto kern) {
      hipLaunchKernelGGL(kern, grid, block, 0, stream, P, Q, epi, part, (int)tm, (int)tn, (int)splits);
    };
    if (BM == 128 && BN == 128) go(product_kernel<T, PR, QR, 128, 128, TWO>);
    else if (BM == 128) go(product_kernel<T, PR, QR, 128, 64, TWO>);
    else go(product_kernel<T, PR, QR, 64, 64, TWO>);
  }
  if (splits > 1) {
    const int64_t work = M * ((N + 3) / 4);
    hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)std::min<int64_t>((work + 255) / 256, 4096)),
                       dim3(256), 0, stream, part, epi, M, (int)N, (int)splits);
  }
}

template <typename T>
void slope(const torch::Tensor& dy, const torch::Tensor* of, torch::Tensor* dz, torch::Tensor* left,
           torch::Tensor* db, int act, hipStream_t stream) {
  const int64_t M = dy.size(0);
  const int N = (int)dy.size(1);
  constexpr int V = 16 / sizeof(T);
  const bool vec = N % V == 0 && aligned(dy.data_ptr(), 16) && (!dz || (aligned(dz->data_ptr(), 16)
                   && aligned(of->data_ptr(), 16))) && (!left || aligned(left->data_ptr(), 16));
  const int vw = vec ? V : 1, tile = std::min(N, (vec ? 32 : 64) * vw), ntile = (N + tile - 1) / tile;
  const int rows = 256 / (tile / vw);
  // 1024 workgroups or more, as long as a thread has 4 rows (25088x256 takes 10 us, with fewer 16); few rows are
  // one chunk, whose sums need no joining
  int64_t chunk = std::max<int64_t>(4, M * ntile / 1024 / rows) * rows;
  if (M <= 16 * rows) chunk = 16 * rows;
  chunk = std::min<int64_t>(chunk, 1 << 24);
  const int64_t chunks = (M + chunk - 1) / chunk;
  TORCH_CHECK(chunks * ntile < (int64_t(1) << 24), "linear_act: too many rows");
  torch::Tensor ws;
  const bool join = db && chunks > 1;
  if (join) ws = torch::empty({chunks * N}, dy.options().dtype(torch::kFloat32));
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((unsigned)(chunks * ntile)), dim3(256), 0, stream,
                       (const T*)dy.data_ptr(), of ? of->data_ptr() : nullptr,
                       dz ? (T*)dz->data_ptr() : nullptr, left ? (T*)left->data_ptr() : nullptr, join ? ws.data_ptr<float>() : nullptr,
                       db && !join ? (T*)db->data_ptr() : nullptr, M, N, tile,
                       ntile, (int)chunk, act);
  };
  if (vec) go(slope_kernel<T, V>);
  else go(slope_kernel<T, 1>);
  if (join)
    hipLaunchKernelGGL((column_join_kernel<T>), dim3((N + 7) / 8), dim3(1024), 0, stream,
                       ws.data_ptr<float>(), chunks, N, (T*)db->data_ptr());
}

void check(const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& b, const torch::Tensor& r,
           int64_t act) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && w.dim() == 2 && x.is_contiguous() && w.is_contiguous(),
              "linear_act: x [M,K] and weight [N,K], contiguous");
  TORCH_CHECK(x.size(1) == w.size(1) && x.size(1) > 0 && w.size(0) > 0, "linear_act: sizes");
  // offsets in a tile of 128 lines, or of 64 lines of 128, are 32 bits
  TORCH_CHECK(x.size(0) < (int64_t(1) << 31) - 256 && x.size(1) <= (1 << 23) && w.size(0) <= (1 << 23),
              "linear_act: 2^31 rows or more, or more than 2^23 columns");
  TORCH_CHECK(w.scalar_type() == x.scalar_type() && w.device() == x.device(), "linear_act: weight");
  TORCH_CHECK(!b.defined() || (b.is_contiguous() && b.dim() == 1 && b.size(0) == w.size(0)
              && b.scalar_type() == x.scalar_type() && b.device() == x.device()), "linear_act: bias");
  TORCH_CHECK(!r.defined() || (r.is_contiguous() && r.dim() == 2 && r.size(0) == x.size(0)
              && r.size(1) == w.size(0) && r.scalar_type() == x.scalar_type()
              && r.device() == x.device()), "linear_act: residual");
  TORCH_CHECK(act >= 0 && act <= 3, "linear_act: activation");
}

class LinearAct : public torch::autograd::Function<LinearAct> {
 public:
  static torch::Tensor forward(torch::autograd::AutogradContext* ctx, torch::Tensor x, torch::Tensor w,
                               c10::optional<torch::Tensor> bias, c10::optional<torch::Tensor> res,
                               int64_t act, bool train) {
    const auto b = bias.value_or(torch::Tensor()), r = res.value_or(torch::Tensor());
    check(x, w, b, r, act);
    const c10::OptionalDeviceGuard guard(x.device());
    auto stream = at::hip::getCurrentHIPStream().stream();
    auto y = torch::empty({x.size(0), w.size(0)}, x.options());
    const bool keep = train && (act == ACT_SWISH || act == ACT_SIGMOID);
    auto slopes = keep ? torch::empty(y.sizes(), y.options().dtype(torch::kFloat32)) : torch::Tensor();
    if (x.size(0) > 0)
      by_type(x.scalar_type(), [&](auto t) {
        using T = decltype(t);
        Epilogue<T> epi{b.defined() ? (const T*)b.data_ptr() : nullptr,
                        r.defined() ? (const T*)r.data_ptr() : nullptr, (T*)y.data_ptr(),
                        keep ? slopes.data_ptr<float>() : nullptr, (int)act, false};
        product<T, false, false>(x, w, epi, stream);
      });
    C10_HIP_KERNEL_LAUNCH_CHECK();
    ctx->saved_data["how"] = act * 4 + b.defined() * 2 + r.defined();
    // relu's slope is known from its result
    ctx->save_for_backward({x, w, keep ? slopes : act == ACT_RELU ? y : torch::Tensor()});
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    auto saved = ctx->get_saved_variables();
    const auto &x = saved[0], &w = saved[1], &of = saved[2];
    const int64_t how = ctx->saved_data["how"].toInt();
    const int act = (int)(how / 4);
    const c10::OptionalDeviceGuard guard(x.device());
    auto stream = at::hip::getCurrentHIPStream().stream();
    // absent tensors are not counted among the inputs
    const bool has_b = how & 2, has_r = how & 1;
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1),
               nb = has_b && ctx->needs_input_grad(2), nr = has_r && ctx->needs_input_grad(has_b ? 3 : 2);
    torch::Tensor dy, dz, left, dx, dw, db;
    const int64_t M = x.size(0), N = w.size(0);
    const bool again = at::GradMode::is_enabled();
    {
      at::NoGradGuard off;
      dy = grads[0].contiguous();
      if (nb) db = torch::empty({N}, x.options());
      if (nx) dx = torch::empty_like(x);
      if (nw) dw = torch::empty_like(w);
      dz = act == ACT_NONE ? dy : torch::empty_like(dy);
      // The slopes of swish and sigmoid make dz a number of 32 bits, which one of 16 cannot hold for the products: a
      // gradient's error in bf16 would be 1.4 times that of its own rounding. Others' dz is dy or 0.
      const bool two = (act == ACT_SWISH || act == ACT_SIGMOID) && dy.element_size() == 2 && (nx || nw);
      if (two) left = torch::empty_like(dy);
      if (M == 0) {
        if (nb) db.zero_();
        if (nw) dw.zero_();
      } else {
        by_type(x.scalar_type(), [&](auto t) {
          using T = decltype(t);
          if (act != ACT_NONE || nb)
            slope<T>(dy, act == ACT_NONE ? nullptr : &of, act == ACT_NONE ? nullptr : &dz, two ? &left : nullptr,
                     nb ? &db : nullptr, act, stream);
          Epilogue<T> epi{nullptr, nullptr, nullptr, nullptr, ACT_NONE, false};
          auto products = [&](auto terms) {
            if (nx) {
              epi.y = (T*)dx.data_ptr();
              product<T, false, true, terms.value>(dz, w, epi, stream, &left);
            }
            if (nw) {
              epi.y = (T*)dw.data_ptr();
              product<T, true, true, terms.value>(dz, x, epi, stream, &left);
            }
          };
          if constexpr (sizeof(T) == 2)
            if (two) return products(std::true_type{});
          products(std::false_type{});
        });
        C10_HIP_KERNEL_LAUNCH_CHECK();
      }
    }
    torch::autograd::variable_list out{dx, dw, db, nr ? dz : torch::Tensor(), torch::Tensor(),
                                       torch::Tensor()};
    if (again)      // differentiating these again is an error, not a zero
      for (auto& g : out)
        if (g.defined()) {
          auto err = std::make_shared<torch::autograd::DelayedError>(
              "linear_act is differentiable once", 1);
          g = (*err)({g.detach().requires_grad_(true)})[0];
        }
    return out;
  }
};

}  // namespace

torch::Tensor linear_act(torch::Tensor x, torch::Tensor weight, c10::optional<torch::Tensor> bias,
                         c10::optional<torch::Tensor> residual, int64_t act) {
  const bool train = at::GradMode::is_enabled()
                     && (x.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad())
                         || (residual && residual->requires_grad()));
  return LinearAct::apply(x, weight, bias, residual, act, train);
}
