// AdamW over every tensor of a model in one launch, moments in 32 or 8 bits.
//
//   g' = g * min(1, clip / (||g|| + 1e-6))            (norm over all tensors)
//   m  = b1 m + (1-b1) g'        v = b2 v + (1-b2) g'^2
//   p  = p (1 - lr wd) - lr (m / (1-b1^t)) / (sqrt(v / (1-b2^t)) + eps)
//
// A table row says where a tensor lies (weights, low-precision copy,
// gradient, place in the moment buffers, length, decay); a second table maps
// each workgroup to 4096 elements of one row, so many small tensors and one
// flat buffer of 36M elements are the same launch. One lane owns 4 neighbours,
// one wave 256: the quantisation block, so a block's largest moment is a
// wave-wide maximum and needs neither LDS nor a barrier.
//
// 8 bits: m and sqrt(v) are held as e4m3 numbers with one fp32 scale
// (largest/448) a block. The root is held rather than v because its range is
// half as wide in the exponent (e4m3 spans 2^18) and the step divides by it.
// Rounding is to nearest: the common decay of a block goes into its fp32
// scale, so a moment that only decays keeps its code. The step itself uses the
// moments before they are rounded. A root that is not zero is held as at least
// the smallest number, since a zero would make the next step m / eps.
//
// The step count, learning rate and clip factor live on the device, so a step
// can be captured and replayed.
//
// Bound by memory. 36.5M bf16 parameters with fp32 weights: with 32-bit moments
// 28 bytes an element in 187 us, 5.5 TB/s; with 8-bit moments 16 bytes in 116 us,
// 5.0 TB/s (a copy reaches 4.9). A clip factor needs all gradients first: 73 MB
// in 26 us. 36 tensors of 16 to 147456 elements take 8 us, and 3 for the scalars.

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <hip/hip_fp16.h>
#include "faa_common.h"

namespace {

constexpr int kChunk = 4096;      // elements a workgroup takes
constexpr int kBlock = 256;       // elements under one scale: one wave's
constexpr int kThreads = 256;
constexpr int kIters = kChunk / (kThreads * 4);
constexpr int kRow = 6;           // int64 fields of a table row
constexpr float kQMax = 448.0f;
constexpr float kQTiny = 7.888609052210118e-31f;   // 2^-100

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(4))) unsigned short u16x4;

struct Row { float* p; void* w; const void* g; int64_t off, n; float wd; int aligned; };

__device__ __forceinline__ Row read_row(const int64_t* __restrict__ rows, int i) {
  const int64_t* r = rows + (int64_t)i * kRow;
  Row o;
  o.p = (float*)r[0];
  o.w = (void*)r[1];
  o.g = (const void*)r[2];
  o.off = r[3];
  o.n = r[4];
  o.wd = __int_as_float((int)(r[5] & 0xffffffff));
  o.aligned = (int)(r[5] >> 32);
  return o;
}

template <typename T> struct Elem;
template <> struct Elem<float> {
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ f32x4 get4(const float* p) { return *(const f32x4*)p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
  static __device__ __forceinline__ void put4(float* p, f32x4 v) { *(f32x4*)p = v; }
};
template <> struct Elem<__hip_bfloat16> {
  typedef __hip_bfloat16 T;
  static __device__ __forceinline__ float get(const T* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ f32x4 get4(const T* p) {
    u16x4 u = *(const u16x4*)p;
    f32x4 v;
    #pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float((uint32_t)u[i] << 16);
    return v;
  }
  static __device__ __forceinline__ void put(T* p, float v) { *p = __float2bfloat16(v); }
  static __device__ __forceinline__ void put4(T* p, f32x4 v) {
    u16x4 u;
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      __hip_bfloat16 h = __float2bfloat16(v[i]);
      u[i] = *(unsigned short*)&h;
    }
    *(u16x4*)p = u;
  }
};
template <> struct Elem<__half> {
  typedef __half T;
  static __device__ __forceinline__ float get(const T* p) { return __half2float(*p); }
  static __device__ __forceinline__ f32x4 get4(const T* p) {
    u16x4 u = *(const u16x4*)p;
    f32x4 v;
    #pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __half2float(__ushort_as_half(u[i]));
    return v;
  }
  static __device__ __forceinline__ void put(T* p, float v) { *p = __float2half(v); }
  static __device__ __forceinline__ void put4(T* p, f32x4 v) {
    u16x4 u;
    #pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __half_as_ushort(__float2half(v[i]));
    *(u16x4*)p = u;
  }
};

// 4 neighbours from element e of a tensor of n; what lies behind it reads as 0
template <typename T>
__device__ __forceinline__ f32x4 load4(const T* p, int64_t e, int64_t n, bool vec) {
  if (vec && e + 4 <= n) return Elem<T>::get4(p + e);
  f32x4 v = {0, 0, 0, 0};
  #pragma unroll
  for (int i = 0; i < 4; ++i)
    if (e + i < n) v[i] = Elem<T>::get(p + e + i);
  return v;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t e, int64_t n, bool vec, f32x4 v) {
  if (vec && e + 4 <= n) { Elem<T>::put4(p + e, v); return; }
  #pragma unroll
  for (int i = 0; i < 4; ++i)
    if (e + i < n) Elem<T>::put(p + e + i, v[i]);
}

__device__ __forceinline__ float wave_max(float v) {
  #pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  return v;
}

__device__ __forceinline__ f32x4 from_e4m3(uint32_t q) {
  f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, false);
  f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)q, true);
  return f32x4{lo[0], lo[1], hi[0], hi[1]};
}
__device__ __forceinline__ uint32_t to_e4m3(f32x4 v) {
  int q = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], q, true);
}

// ------------------------------------------------------------------ norm

__device__ __forceinline__ double wave_sum(double v) {
  #pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// part[block] = sum of squares of the block's chunks, added in a fixed order and in 64 bits: an error of the norm
// would move every gradient the same way, and 8-bit moments over a border.
template <typename T>
__global__ __launch_bounds__(kThreads) void adamw_norm_kernel(
    const int64_t* __restrict__ rows, const int* __restrict__ chunks, int n_chunks,
    double* __restrict__ part) {
  __shared__ double lds[kThreads / FAA_WAVE];
  double acc = 0.0;
  for (int c = blockIdx.x; c < n_chunks; c += gridDim.x) {
    Row r = read_row(rows, chunks[2 * c]);
    if (r.g == nullptr) continue;
    int64_t base = (int64_t)chunks[2 * c + 1] * kChunk + threadIdx.x * 4;
    #pragma unroll
    for (int it = 0; it < kIters; ++it) {
      f32x4 g = load4((const T*)r.g, base + it * kThreads * 4, r.n, r.aligned);
      #pragma unroll
      for (int i = 0; i < 4; ++i) acc += (double)(g[i] * g[i]);
    }
  }
  acc = wave_sum(acc);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x / 64] = acc;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// scal = {clip factor, 1/(1-b1^t), 1/sqrt(1-b2^t)} of the step that begins
__global__ __launch_bounds__(kThreads) void adamw_begin_kernel(
    const double* __restrict__ part, int n_part, int64_t* __restrict__ step,
    float* __restrict__ scal, double b1, double b2, float clip) {
  __shared__ double lds[kThreads / FAA_WAVE];
  double s = 0.0;
  #pragma unroll 4
  for (int i = threadIdx.x; i < n_part; i += kThreads) s += part[i];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x / 64] = s;
  // the powers are taken by other waves meanwhile
  if (threadIdx.x == 64) scal[1] = (float)(1.0 / (1.0 - pow(b1, (double)(step[0] + 1))));
  if (threadIdx.x == 128) scal[2] = (float)(1.0 / sqrt(1.0 - pow(b2, (double)(step[0] + 1))));
  __syncthreads();
  if (threadIdx.x == 0) {
    step[0] += 1;
    float norm = (float)sqrt(lds[0] + lds[1] + lds[2] + lds[3]);
    scal[0] = clip > 0.0f ? fminf(1.0f, clip * (1.0f / (norm + 1e-6f))) : 1.0f;
    if (norm != norm) scal[0] = norm;     // fminf would hide a norm that is no number
  }
}

// ------------------------------------------------------------------ step

struct Moments {
  void* m;        // fp32 or e4m3
  void* r;        // v in fp32, or sqrt(v) in e4m3
  float* ms;      // scales of the 8-bit forms, one a block
  float* rs;
};

template <typename T, int BITS, bool WORK>
__global__ __launch_bounds__(kThreads) void adamw_step_kernel(
    const int64_t* __restrict__ rows, const int* __restrict__ chunks, Moments st,
    const float* __restrict__ scal, const float* __restrict__ lr_p,
    float b1, float c1, float b2, float c2, float eps) {
  // Every operation is rounded by itself and in the CPU path's order, so that moments held in 8 bits are that
  // path's bit for bit: a fused product and sum would leave some of them on the other side of a border.
  #pragma clang fp contract(off)
  const Row r = read_row(rows, chunks[2 * blockIdx.x]);
  if (r.g == nullptr) return;             // no gradient: the tensor is left as it is
  const int64_t base = (int64_t)chunks[2 * blockIdx.x + 1] * kChunk + threadIdx.x * 4;
  const float lr = lr_p[0], coef = scal[0], a1 = scal[1], a2 = scal[2];
  const float keep = 1.0f - lr * r.wd;
  const bool vec = r.aligned;

  f32x4 p[kIters], g[kIters], m[kIters], v[kIters];
  uint32_t qm[kIters], qr[kIters];
  float sm[kIters], sr[kIters];
  #pragma unroll
  for (int it = 0; it < kIters; ++it) {
    const int64_t e = base + it * kThreads * 4;
    p[it] = load4(r.p, e, r.n, vec);
    g[it] = load4((const T*)r.g, e, r.n, vec);
    if constexpr (BITS == 32) {
      m[it] = load4((const float*)st.m + r.off, e, r.n, vec);
      v[it] = load4((const float*)st.r + r.off, e, r.n, vec);
    } else if (e < r.n) {                 // the buffers are whole blocks
      qm[it] = *(const uint32_t*)((const uint8_t*)st.m + r.off + e);
      qr[it] = *(const uint32_t*)((const uint8_t*)st.r + r.off + e);
      sm[it] = st.ms[(r.off + e) / kBlock];
      sr[it] = st.rs[(r.off + e) / kBlock];
    }
  }
  #pragma unroll
  for (int it = 0; it < kIters; ++it) {
    const int64_t e = base + it * kThreads * 4;
    f32x4 mm = {0, 0, 0, 0}, vv = {0, 0, 0, 0}, root;
    if constexpr (BITS == 32) {
      mm = m[it];
      vv = v[it];
    } else if (e < r.n) {
      mm = from_e4m3(qm[it]) * sm[it];
      vv = from_e4m3(qr[it]) * sr[it];
      vv = vv * vv;
    }
    f32x4 pp = p[it];
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float gg = g[it][i] * coef;
      mm[i] = b1 * mm[i] + c1 * gg;
      vv[i] = b2 * vv[i] + (c2 * gg) * gg;
      root[i] = sqrtf(vv[i]);
      pp[i] = pp[i] * keep - lr * (mm[i] * a1 / (root[i] * a2 + eps));
    }
    store4(r.p, e, r.n, vec, pp);
    if constexpr (WORK) store4((T*)r.w, e, r.n, vec, pp);
    if constexpr (BITS == 32) {
      store4((float*)st.m + r.off, e, r.n, vec, mm);
      store4((float*)st.r + r.off, e, r.n, vec, vv);
    } else {
      // lanes behind the tensor's end hold zeros and take part in the maximum
      float tm = fmaxf(fmaxf(fabsf(mm[0]), fabsf(mm[1])), fmaxf(fabsf(mm[2]), fabsf(mm[3])));
      float tr = fmaxf(fmaxf(root[0], root[1]), fmaxf(root[2], root[3]));
      tm = fmaxf(wave_max(tm), kQTiny);
      tr = fmaxf(wave_max(tr), kQTiny);
      if (e < r.n) {
        uint32_t um = to_e4m3(mm * (kQMax * (1.0f / tm)));
        uint32_t ur = to_e4m3(root * (kQMax * (1.0f / tr)));
        #pragma unroll
        for (int i = 0; i < 4; ++i)
          if (root[i] > 0.0f && ((ur >> (8 * i)) & 0xff) == 0) ur |= 1u << (8 * i);
        *(uint32_t*)((uint8_t*)st.m + r.off + e) = um;
        *(uint32_t*)((uint8_t*)st.r + r.off + e) = ur;
        if ((threadIdx.x & 63) == 0) {
          st.ms[(r.off + e) / kBlock] = tm * (1.0f / kQMax);
          st.rs[(r.off + e) / kBlock] = tr * (1.0f / kQMax);
        }
      }
    }
  }
}

template <typename T, bool WORK>
void launch_step(const torch::Tensor& rows, const torch::Tensor& chunks, Moments st, int bits,
                 const float* scal, const float* lr, double b1, double b2, double eps,
                 hipStream_t stream) {
  dim3 grid((unsigned)chunks.size(0)), block(kThreads);
  const float fb1 = (float)b1, c1 = (float)(1.0 - b1), fb2 = (float)b2, c2 = (float)(1.0 - b2);
  if (bits == 32)
    hipLaunchKernelGGL((adamw_step_kernel<T, 32, WORK>), grid, block, 0, stream,
                       rows.data_ptr<int64_t>(), chunks.data_ptr<int>(), st, scal, lr,
                       fb1, c1, fb2, c2, (float)eps);
  else
    hipLaunchKernelGGL((adamw_step_kernel<T, 8, WORK>), grid, block, 0, stream,
                       rows.data_ptr<int64_t>(), chunks.data_ptr<int>(), st, scal, lr,
                       fb1, c1, fb2, c2, (float)eps);
}

}  // namespace

// tables: one [rows, chunks] pair for each gradient type in kinds (0 fp32,
// 1 bf16, 2 fp16); a kind above 0 has fp32 weights beside the low-precision ones.
void adamw_step(std::vector<torch::Tensor> rows, std::vector<torch::Tensor> chunks,
                std::vector<int64_t> kinds, torch::Tensor m, torch::Tensor r,
                torch::Tensor m_scale, torch::Tensor r_scale, torch::Tensor step,
                torch::Tensor scal, torch::Tensor part, torch::Tensor lr, double b1,
                double b2, double eps, double clip) {
  TORCH_CHECK(rows.size() == chunks.size() && rows.size() == kinds.size(), "adamw_step: tables");
  TORCH_CHECK(m.is_cuda() && m.scalar_type() == r.scalar_type() && m.numel() == r.numel(),
              "adamw_step: moments");
  const int bits = m.scalar_type() == torch::kFloat32 ? 32 : 8;
  TORCH_CHECK(bits == 32 || (m.scalar_type() == torch::kFloat8_e4m3fn && m.numel() % kBlock == 0
              && m_scale.numel() == m.numel() / kBlock && r_scale.numel() == m_scale.numel()
              && m_scale.scalar_type() == torch::kFloat32 && r_scale.scalar_type() == torch::kFloat32),
              "adamw_step: moments are fp32, or e4m3 with a scale for every block of 256");
  TORCH_CHECK(step.scalar_type() == torch::kInt64 && scal.numel() >= 3
              && scal.scalar_type() == torch::kFloat32 && lr.scalar_type() == torch::kFloat32
              && part.scalar_type() == torch::kFloat64, "adamw_step: scalars");
  const c10::OptionalDeviceGuard guard(m.device());
  auto stream = at::hip::getCurrentHIPStream().stream();
  const int per = rows.empty() ? 0 : (int)(part.numel() / (int64_t)rows.size());
  int n_part = 0;
  for (size_t i = 0; i < rows.size(); ++i) {
    TORCH_CHECK(rows[i].scalar_type() == torch::kInt64 && rows[i].dim() == 2
                && rows[i].size(1) == kRow && rows[i].device() == m.device()
                && rows[i].is_contiguous(), "adamw_step: rows");
    TORCH_CHECK(chunks[i].scalar_type() == torch::kInt32 && chunks[i].dim() == 2
                && chunks[i].size(1) == 2 && chunks[i].device() == m.device()
                && chunks[i].is_contiguous(), "adamw_step: chunks");
    TORCH_CHECK(kinds[i] >= 0 && kinds[i] <= 2, "adamw_step: kind");
    // the caller may let go of the tables while this stream, which need not be theirs, still reads them
    for (const auto& t : {rows[i], chunks[i]}) t.record_stream(at::hip::getCurrentHIPStreamMasqueradingAsCUDA());
    if (clip <= 0.0 || chunks[i].size(0) == 0) continue;
    const int nc = (int)chunks[i].size(0), grid = std::min(nc, per);
    TORCH_CHECK(grid > 0, "adamw_step: part is too short");
    double* out = part.data_ptr<double>() + n_part;
    auto go = [&](auto kern) {
      hipLaunchKernelGGL(kern, dim3(grid), dim3(kThreads), 0, stream,
                         rows[i].data_ptr<int64_t>(), chunks[i].data_ptr<int>(), nc, out);
    };
    if (kinds[i] == 0) go(adamw_norm_kernel<float>);
    else if (kinds[i] == 1) go(adamw_norm_kernel<__hip_bfloat16>);
    else go(adamw_norm_kernel<__half>);
    n_part += grid;
  }
  hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(kThreads), 0, stream,
                     part.data_ptr<double>(), n_part, step.data_ptr<int64_t>(),
                     scal.data_ptr<float>(), b1, b2, (float)clip);
  Moments st{m.data_ptr(), r.data_ptr(), bits == 8 ? m_scale.data_ptr<float>() : nullptr,
             bits == 8 ? r_scale.data_ptr<float>() : nullptr};
  for (size_t i = 0; i < rows.size(); ++i) {
    if (chunks[i].size(0) == 0) continue;
    const float *s = scal.data_ptr<float>(), *l = lr.data_ptr<float>();
    if (kinds[i] == 0)
      launch_step<float, false>(rows[i], chunks[i], st, bits, s, l, b1, b2, eps, stream);
    else if (kinds[i] == 1)
      launch_step<__hip_bfloat16, true>(rows[i], chunks[i], st, bits, s, l, b1, b2, eps, stream);
    else
      launch_step<__half, true>(rows[i], chunks[i], st, bits, s, l, b1, b2, eps, stream);
  }
  C10_HIP_KERNEL_LAUNCH_CHECK();
}
