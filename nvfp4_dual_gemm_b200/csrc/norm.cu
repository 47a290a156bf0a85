// norm.cu — the norms between two blocks of a transformer, fused with the
// gate and scale of the residual stream and with the quantisation of the next
// product's input:
//
//   u = post ? norm(y) * post_weight + post_bias : y
//   r = x + scale * gate * u        (rounded to the stream's type)
//   z = norm(r) * weight + bias     (16 / 32 bits, or NVFP4 of those)
//
// One pass: a row stays in registers between its one read of x and y and its
// one write of r and z; the row sums go through the warps' shuffles and, for
// rows wider than a warp holds, one word a warp in shared memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "host.h"
#include "nvfp4_dual_gemm.h"
#include "quant.cuh"
#include "sm100_ptx.cuh"

namespace nvfp4dg {
namespace {

constexpr int kAtomBytes = 512;  // scales of 128 rows x 64 elements

struct NormParams {
  nvfp4_block_norm_args a;
  int gate_run;  // rows of one gate row
  int rows_pad;  // rows whose scales are written (NVFP4 output), else rows
};

// Eight consecutive elements as fp32.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    using H2 = typename std::conditional<std::is_same<T, __half>::value,
                                         __half2, __nv_bfloat162>::type;
    v[2 * i] = Half2Ops<H2>::lo(w[i]);
    v[2 * i + 1] = Half2Ops<H2>::hi(w[i]);
  }
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  const float4 b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}

// Rounds eight values to T: `w` gets the bits to store, v the values.
template <typename T>
struct Round8 {
  uint32_t w[4];
  __device__ __forceinline__ void set(float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
        v[2 * i] = Half2Ops<__half2>::lo(w[i]);
        v[2 * i + 1] = Half2Ops<__half2>::hi(w[i]);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
        v[2 * i] = Half2Ops<__nv_bfloat162>::lo(w[i]);
        v[2 * i + 1] = Half2Ops<__nv_bfloat162>::hi(w[i]);
      }
    }
  }
  __device__ __forceinline__ uint32_t word(int i) const { return w[i]; }
  __device__ __forceinline__ void store(T* p) const {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Round8<float> {
  float f[8];
  __device__ __forceinline__ void set(float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = v[i];
  }
  __device__ __forceinline__ uint32_t word(int i) const {
    return __float_as_uint(f[i]);
  }
  __device__ __forceinline__ void store(float* p) const {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};

template <typename T>
__device__ __forceinline__ void load_w8(const void* w, int w_f32, int i,
                                        float (&v)[8]) {
  if (w_f32)
    load8<float>(static_cast<const float*>(w) + i, v);
  else
    load8<T>(static_cast<const T*>(w) + i, v);
}

// Sum over the threads of a row: a warp (WARP_ROW) or the whole CTA.  `slot`
// is a shared buffer of 32 words that the row's previous sum did not use.
template <bool WARP_ROW>
__device__ __forceinline__ float row_sum(float v, float* slot) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if (WARP_ROW) return v;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (lane == 0) slot[warp] = v;
  __syncthreads();
  v = lane < static_cast<int>(blockDim.x) / 32 ? slot[lane] : 0.f;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// v <- norm(v) * w + b over a row of D elements, VPT vectors of eight a
// thread (vector t + i * threads).  The layer norm's variance is summed from
// the centred values, not as a difference of large sums.
template <typename T, int VPT, bool WARP_ROW>
__device__ __forceinline__ void norm_row(float (&v)[VPT][8], int vecs, int t,
                                         int threads, int D, int kind,
                                         float eps, const void* w,
                                         const void* b, int w_f32,
                                         float* slots) {
  if (kind == NVFP4DG_NORM_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (t + i * threads < vecs) {
#pragma unroll
        for (int k = 0; k < 8; ++k) s += v[i][k];
      }
    const float mean = row_sum<WARP_ROW>(s, slots) / D;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) v[i][k] -= mean;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    if (t + i * threads < vecs) {
#pragma unroll
      for (int k = 0; k < 8; ++k) q = fmaf(v[i][k], v[i][k], q);
    }
  const float inv = rsqrtf(row_sum<WARP_ROW>(q, slots + 32) / D + eps);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = t + i * threads;
    if (j < vecs) {
      float f[8];
      if (w != nullptr) {
        load_w8<T>(w, w_f32, 8 * j, f);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = v[i][k] * inv * f[k];
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] *= inv;
      }
      if (b != nullptr) {
        load_w8<T>(b, w_f32, 8 * j, f);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] += f[k];
      }
    }
  }
}

// One half (eight values, rounded to T) of a 16-element block whose other
// half the neighbouring lane holds -> its four bytes of codes and the block's
// scale byte, as the activation quantiser's (quant.cuh).  All lanes of a warp
// call it.
template <typename T>
__device__ __forceinline__ uint32_t quant_half(const float (&v)[8],
                                               const Round8<T>& z,
                                               uint8_t& sb) {
  uint32_t x[8], key = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = __float_as_uint(v[i]);
    key = max(key, x[i] & 0x7FFFFFFFu);
  }
  key = max(key, __shfl_xor_sync(0xffffffffu, key, 1));
  const float amax = __uint_as_float(key);
  sb = __nv_cvt_float_to_fp8(amax / 6.0f, __NV_SATFINITE, __NV_E4M3);
  const float2 r = rcp_pair(sb);
  uint32_t w = sb != 0 ? e2m1_scaled8(x, r.x, r.y) : 0u;
  // a block holding a NaN goes to the compare form, which takes all sixteen
  if (__any_sync(0xffffffffu, key > 0x7F800000u)) {
    const bool hi = threadIdx.x & 1;
    constexpr int kWords = sizeof(T) == 2 ? 4 : 8;
    uint32_t f[2 * kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const uint32_t own = z.word(i);
      const uint32_t other = __shfl_xor_sync(0xffffffffu, own, 1);
      f[i] = hi ? other : own;
      f[kWords + i] = hi ? own : other;
    }
    if (key > 0x7F800000u) {
      uint32_t w0, w1;
      if constexpr (sizeof(T) == 2) {
        using H2 = typename std::conditional<std::is_same<T, __half>::value,
                                             __half2, __nv_bfloat162>::type;
        sb = quant_block16_x2_cmp<H2>(f, w0, w1);
      } else {
        float e[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = __uint_as_float(f[i]);
        sb = quant_block16(e, w0, w1);
      }
      w = hi ? w1 : w0;
    }
  }
  return w;
}

template <typename T, int VPT, bool WARP_ROW, int MAXT>
__global__ void __launch_bounds__(MAXT)
    block_norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ float slots[128];
  const nvfp4_block_norm_args& a = p.a;
  const int t = WARP_ROW ? threadIdx.x % 32 : threadIdx.x;
  const int threads = WARP_ROW ? 32 : blockDim.x;
  const int row = WARP_ROW ? blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32
                           : blockIdx.x;
  griddep_launch_dependents();
  griddep_wait();
  if (row >= p.rows_pad) return;
  const int vecs = a.D / 8;
  const int w_f32 = a.w_dtype == NVFP4DG_DTYPE_F32;
  const bool live = row < a.rows;
  float r[VPT][8];
  if (live) {
    float u[VPT][8];
    const T* x = static_cast<const T*>(a.x) + (size_t)row * a.ldx;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = t + i * threads;
      if (j < vecs) load8<T>(x + 8 * j, r[i]);
    }
    if (a.y != nullptr) {
      const T* y = static_cast<const T*>(a.y) + (size_t)row * a.ldy;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = t + i * threads;
        if (j < vecs) load8<T>(y + 8 * j, u[i]);
      }
      if (a.post)
        norm_row<T, VPT, WARP_ROW>(u, vecs, t, threads, a.D, a.kind, a.eps,
                                   a.post_weight, a.post_bias, w_f32, slots);
      const T* g = a.gate ? static_cast<const T*>(a.gate) +
                                (size_t)(row / p.gate_run) * a.D
                          : nullptr;
      T* R = static_cast<T*>(a.R) + (size_t)row * a.ldr;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = t + i * threads;
        if (j < vecs) {
          if (g != nullptr) {
            float f[8];
            load8<T>(g + 8 * j, f);
#pragma unroll
            for (int k = 0; k < 8; ++k) u[i][k] *= f[k];
          }
#pragma unroll
          for (int k = 0; k < 8; ++k)
            r[i][k] = fmaf(a.scale, u[i][k], r[i][k]);
          Round8<T> o;
          o.set(r[i]);
          o.store(R + 8 * j);
        }
      }
    }
    if (a.Z == nullptr && a.codes == nullptr) return;
    norm_row<T, VPT, WARP_ROW>(r, vecs, t, threads, a.D, a.kind, a.eps,
                               a.weight, a.bias, w_f32, slots + 64);
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = t + i * threads;
    const bool in = live && j < vecs;
    Round8<T> z;
    if (in) {
      z.set(r[i]);
      if (a.Z != nullptr)
        z.store(static_cast<T*>(a.Z) + (size_t)row * a.ldz + 8 * j);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) r[i][k] = 0.f;
      z.set(r[i]);
    }
    if (a.codes == nullptr) continue;
    uint8_t sb;
    const uint32_t w = quant_half<T>(r[i], z, sb);
    if (in)
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.codes) +
                                   (size_t)row * (a.D / 2) + 4 * j) = w;
    // the eight lanes of 64 elements hold four scales, each twice
    const uint32_t s1 = __shfl_down_sync(0xffffffffu, sb, 2);
    const uint32_t s2 = __shfl_down_sync(0xffffffffu, sb, 4);
    const uint32_t s3 = __shfl_down_sync(0xffffffffu, sb, 6);
    if ((j & 7) == 0 && j < vecs)
      *reinterpret_cast<uint32_t*>(
          static_cast<uint8_t*>(a.sf) +
          ((size_t)(row / 128) * (a.D / 64) + j / 8) * kAtomBytes +
          (row % 32) * 16 + ((row % 128) / 32) * 4) =
          static_cast<uint32_t>(sb) | (s1 << 8) | (s2 << 16) | (s3 << 24);
  }
}

template <typename T>
int launch_norm(const NormParams& p, int sms, cudaStream_t stream) {
  const int vecs = p.a.D / 8;
  void (*kernel)(NormParams);
  int threads, grid;
  if (vecs <= 128) {  // a warp holds the row
    threads = p.rows_pad >= 4 * sms ? 256 : 64;
    grid = (p.rows_pad + threads / 32 - 1) / (threads / 32);
    kernel = vecs <= 32   ? block_norm_kernel<T, 1, true, 256>
             : vecs <= 64 ? block_norm_kernel<T, 2, true, 256>
                          : block_norm_kernel<T, 4, true, 256>;
  } else {
    grid = p.rows_pad;
    const int vpt = vecs <= 512 ? 1 : vecs <= 1024 ? 2 : 4;
    threads = ((vecs + vpt - 1) / vpt + 31) / 32 * 32;
    kernel = vpt == 1   ? block_norm_kernel<T, 1, false, 512>
             : vpt == 2 ? block_norm_kernel<T, 2, false, 512>
                        : block_norm_kernel<T, 4, false, 1024>;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = (p.a.flags & NVFP4DG_FLAG_NO_PDL) ? 0 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) return host_cuda_fail(e, "block_norm_kernel launch");
  return NVFP4DG_OK;
}

int check_norm(const nvfp4_block_norm_args* a) {
  if (a == nullptr) return host_fail(NVFP4DG_ERR_INVALID, "args is NULL");
  if (a->rows < 0 || a->rows > (1 << 30) || a->D <= 0 || a->D % 8 != 0 ||
      a->D > 32768)
    return host_fail(NVFP4DG_ERR_INVALID,
                     "rows >= 0, D % 8 == 0 and 8 <= D <= 32768 required");
  if (a->dtype != NVFP4DG_DTYPE_F32 && a->dtype != NVFP4DG_DTYPE_F16 &&
      a->dtype != NVFP4DG_DTYPE_BF16)
    return host_fail(NVFP4DG_ERR_INVALID, "dtype must be F32, F16 or BF16");
  if (a->w_dtype != NVFP4DG_DTYPE_F32 && a->w_dtype != a->dtype)
    return host_fail(NVFP4DG_ERR_INVALID,
                     "weights must be F32 or of the stream's type");
  if (a->kind != NVFP4DG_NORM_RMS && a->kind != NVFP4DG_NORM_LAYER)
    return host_fail(NVFP4DG_ERR_INVALID, "unknown norm");
  if (!(a->eps >= 0.f))
    return host_fail(NVFP4DG_ERR_INVALID, "eps must not be negative");
  if (a->flags & ~NVFP4DG_FLAG_NO_PDL)
    return host_fail(NVFP4DG_ERR_INVALID, "unknown flag bits");
  if (a->rows == 0) return NVFP4DG_OK;
  if (a->x == nullptr) return host_fail(NVFP4DG_ERR_INVALID, "x is NULL");
  if (a->y != nullptr && a->R == nullptr)
    return host_fail(NVFP4DG_ERR_INVALID, "R is required with y");
  if (a->y == nullptr && (a->post || a->gate != nullptr))
    return host_fail(NVFP4DG_ERR_INVALID, "post and gate need y");
  if (a->gate != nullptr &&
      (a->gate_rows < 1 || a->rows % a->gate_rows != 0))
    return host_fail(NVFP4DG_ERR_INVALID,
                     "gate_rows must divide the rows");
  if ((a->codes == nullptr) != (a->sf == nullptr))
    return host_fail(NVFP4DG_ERR_INVALID, "codes and sf come together");
  if (a->codes != nullptr && a->D % 64 != 0)
    return host_fail(NVFP4DG_ERR_INVALID,
                     "NVFP4 output needs D % 64 == 0");
  const long long step = a->dtype == NVFP4DG_DTYPE_F32 ? 4 : 8;
  const void* mats[4] = {a->x, a->y, a->R, a->Z};
  const long long lds[4] = {a->ldx, a->ldy, a->ldr, a->ldz};
  for (int i = 0; i < 4; ++i) {
    if (mats[i] == nullptr) continue;
    if (lds[i] < a->D)
      return host_fail(NVFP4DG_ERR_INVALID,
                       "row pitches must be at least D");
    if (lds[i] % step)
      return host_fail(NVFP4DG_ERR_ALIGN,
                       "row pitches must be multiples of 16 bytes");
  }
  const void* ptrs[11] = {a->x,    a->y, a->weight, a->bias,  a->post_weight,
                          a->post_bias, a->gate, a->R, a->Z, a->codes, a->sf};
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) % 16)
      return host_fail(NVFP4DG_ERR_ALIGN,
                       "every pointer must be 16-byte aligned");
  return NVFP4DG_OK;
}

}  // namespace
}  // namespace nvfp4dg

extern "C" int nvfp4_block_norm_run(const nvfp4_block_norm_args* a,
                                    void* stream) {
  using namespace nvfp4dg;
  host_clear_error();
  int rc = check_norm(a);
  if (rc || a->rows == 0) return rc;
  if (a->y == nullptr && a->Z == nullptr && a->codes == nullptr)
    return NVFP4DG_OK;  // r is x and nothing else is asked for
  HostDevice dev;
  if ((rc = host_device(&dev))) return rc;
  NormParams p;
  p.a = *a;
  p.gate_run = a->gate != nullptr ? a->rows / a->gate_rows : 1;
  p.rows_pad = a->codes != nullptr ? (a->rows + 127) / 128 * 128 : a->rows;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == NVFP4DG_DTYPE_F32) return launch_norm<float>(p, dev.sms, s);
  if (a->dtype == NVFP4DG_DTYPE_F16) return launch_norm<__half>(p, dev.sms, s);
  return launch_norm<__nv_bfloat16>(p, dev.sms, s);
}
