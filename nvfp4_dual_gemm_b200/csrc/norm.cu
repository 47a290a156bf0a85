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
//
// Bound by memory for many wide rows (8192 x 7168 bf16, post and pre RMS norm:
// 75 us replayed from a graph, 6.3 TB/s, 0.96 of the measured copy bandwidth;
// 82 us a call in a long loop), by instructions for
// narrower ones (10800 x 2056: 38 us, 4.7 TB/s; layer norms 52 us), by latency
// for few (1 x 7168: 3.0 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>

#include "host.h"
#include "nvfp4_dual_gemm.h"
#include "quant.cuh"
#include "sm100_ptx.cuh"

namespace nvfp4dg {
namespace {

constexpr int kAtomBytes = 512;  // scales of 128 rows x 64 elements
constexpr int kMaxDepth = 8;     // rows a CTA has in flight

struct NormParams {
  nvfp4_block_norm_args a;
  int gate_run;  // rows of one gate row
  int rows_pad;  // rows whose scales are written (NVFP4 output), else rows
  int depth;     // rows in flight (block_norm_rows_kernel)
  unsigned* err;
};

// The four scales of 64 elements of a row in the blocked layout.
__device__ __forceinline__ uint32_t* scale_word(const nvfp4_block_norm_args& a,
                                                int row, int g) {
  return reinterpret_cast<uint32_t*>(
      static_cast<uint8_t*>(a.sf) +
      ((size_t)(row / 128) * (a.D / 64) + g) * kAtomBytes + (row % 32) * 16 +
      ((row % 128) / 32) * 4);
}

// ---------------------------------------------------------------------------
// Vectors of eight consecutive elements.  The arithmetic runs on pairs of
// fp32 values (fma.rn.f32x2 and its like): at 16 bits an element the kernels
// are bound by instructions before they are by memory.
// ---------------------------------------------------------------------------
template <typename T>
using Pair = typename std::conditional<std::is_same<T, __half>::value,
                                       __half2, __nv_bfloat162>::type;

// As loaded: the bits.
template <typename T>
struct Raw8 {
  uint32_t w[sizeof(T) * 2];
  __device__ __forceinline__ void load(const T* p) {
    const uint4* s = reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
      const uint4 u = s[i];
      w[4 * i] = u.x;
      w[4 * i + 1] = u.y;
      w[4 * i + 2] = u.z;
      w[4 * i + 3] = u.w;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      reinterpret_cast<uint4*>(p)[i] = make_uint4(
          w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
  __device__ __forceinline__ F2 pair(int i) const {  // elements 2i, 2i + 1
    if constexpr (sizeof(T) == 4)
      return {__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1])};
    else
      return {Half2Ops<Pair<T>>::lo(w[i]), Half2Ops<Pair<T>>::hi(w[i])};
  }
  __device__ __forceinline__ void set(int i, F2 v) {  // rounds
    if constexpr (sizeof(T) == 4) {
      w[2 * i] = __float_as_uint(v.x);
      w[2 * i + 1] = __float_as_uint(v.y);
    } else if constexpr (std::is_same<T, __half>::value) {
      const __half2 h = __floats2half2_rn(v.x, v.y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};

struct V8 {
  F2 p[4];
};

// A norm's weight or bias at vector j.
template <typename T>
__device__ __forceinline__ V8 load_param(const void* src, int f32, int j) {
  V8 v;
  if (f32) {
    Raw8<float> r;
    r.load(static_cast<const float*>(src) + 8 * j);
#pragma unroll
    for (int i = 0; i < 4; ++i) v.p[i] = r.pair(i);
  } else {
    Raw8<T> r;
    r.load(static_cast<const T*>(src) + 8 * j);
#pragma unroll
    for (int i = 0; i < 4; ++i) v.p[i] = r.pair(i);
  }
  return v;
}

// One parameter vector of a thread's columns (vector t + i * threads).  HELD
// loads it at the kernel's start, so that its latency hides behind the row's;
// otherwise it is read where it is used (from L1, for a CTA of many rows).
template <typename T, int VPT, bool HELD>
struct Param {
  const void* src;
  int f32;
  V8 v[HELD ? VPT : 1];
  __device__ __forceinline__ void set(const void* s, int is_f32, int vecs,
                                      int t, int threads) {
    src = s;
    f32 = is_f32;
    if (HELD && src != nullptr) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (t + i * threads < vecs)
          v[i] = load_param<T>(src, f32, t + i * threads);
    }
  }
  __device__ __forceinline__ V8 get(int i, int j) const {
    return HELD ? v[i] : load_param<T>(src, f32, j);
  }
};

template <typename T, int VPT, bool HELD, bool HELD_BIAS>
struct Params {
  Param<T, VPT, HELD> weight, post_weight;
  Param<T, VPT, HELD_BIAS> bias, post_bias;
  __device__ __forceinline__ void set(const nvfp4_block_norm_args& a,
                                      int vecs, int t, int threads) {
    const int f32 = a.w_dtype == NVFP4DG_DTYPE_F32;
    post_weight.set(a.post_weight, f32, vecs, t, threads);
    post_bias.set(a.post_bias, f32, vecs, t, threads);
    weight.set(a.weight, f32, vecs, t, threads);
    bias.set(a.bias, f32, vecs, t, threads);
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// A row's vectors of one thread: f(i, j) for vector j = t + i * threads.
template <int VPT, typename F>
__device__ __forceinline__ void each(int vecs, int t, int threads, F f) {
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = t + i * threads;
    if (j < vecs) f(i, j);
  }
}

// Sums over a warp of NR values a lane.  Of two values, each half of the warp
// takes one after the first exchange (five shuffles for both, not ten): lanes
// [0, 16) return the first sum and lanes [16, 32) the second.
template <int NR>
__device__ __forceinline__ float warp_sums(const float (&v)[NR], int lane) {
  if (NR == 1) return warp_sum(v[0]);
  const bool hi = lane >= 16;
  float s = (hi ? v[NR - 1] : v[0]) +
            __shfl_xor_sync(0xffffffffu, hi ? v[0] : v[NR - 1], 16);
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  return s;
}
// Value of row r in the layout warp_sums returns.
template <int NR>
__device__ __forceinline__ float pick(float v, int r) {
  return NR == 1 ? v : __shfl_sync(0xffffffffu, v, 16 * r);
}

// What a thread knows of its rows' sums: the part of the warps' sums it adds
// up after the barrier.  With two rows, each half warp adds one row's.
template <bool WARP_ROW, int NR>
struct Sums {
  int lane, warp, part;      // part: this lane's row
  float per_row, per_warp;   // 1 / values of a row, of this warp
  float n[NR], per[NR];      // values of the warps this lane adds up, and 1 / n
  template <int VPT>
  __device__ __forceinline__ void set(int vecs, int threads, int D) {
    lane = threadIdx.x % 32;
    warp = threadIdx.x / 32;
    part = NR == 1 ? 0 : lane / 16;
    per_row = 1.f / D;
    auto count = [&](int l) {
      int c = 0;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        c += min(32, max(0, min(vecs - i * threads, threads) - 32 * l)) * 8;
      return c;
    };
    const int own = WARP_ROW ? D : count(warp);
    per_warp = own > 0 ? 1.f / own : 0.f;
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      const int c = count(other(k));
      n[k] = c;
      per[k] = c > 0 ? 1.f / c : 0.f;
    }
  }
  // the k-th warp this lane adds up: 32 warps over 32 or 16 lanes
  __device__ __forceinline__ int other(int k) const {
    return NR == 1 ? lane : (lane & 15) + 16 * k;
  }
};

// inv = 1 / sqrt(mean(v^2) + eps) of each of NR rows v, which a layer norm
// centres first; v leaves multiplied by the norm's weight.  A row lies in a
// warp (WARP_ROW) or in the whole CTA, whose warps exchange their sums through
// `slots` (64 floats a row that no thread still reads from, zero behind the
// last warp) and one barrier.  A layer norm's warps each sum the squares about
// their own mean; with n values of sum s and such a square sum q in a warp,
// the row's are sum(q + n (s / n - mean)^2) about the row's mean (Chan, Golub
// and LeVeque, 1979), so nothing is a difference of large sums.
template <bool WARP_ROW, bool LAYER, int NR, int VPT, typename P>
__device__ __forceinline__ void norm_factors(V8 (&v)[NR][VPT], int vecs,
                                             int t, int threads, float eps,
                                             const P& w,
                                             const Sums<WARP_ROW, NR>& u,
                                             float* slots,
                                             float (&inv)[NR]) {
  float s[NR], q[NR], ws = 0.f, wq;
  const bool writes = !WARP_ROW && (u.lane & (NR == 1 ? 31 : 15)) == 0;
  float* mine = slots + 64 * u.part;
  if (LAYER) {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      F2 a = {0.f, 0.f};
      each<VPT>(vecs, t, threads, [&](int i, int) {
#pragma unroll
        for (int k = 0; k < 4; ++k) a = add2(a, v[r][i].p[k]);
      });
      s[r] = a.x + a.y;
    }
    ws = warp_sums<NR>(s, u.lane);
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const float m = LAYER ? -pick<NR>(ws, r) * u.per_warp : 0.f;
    F2 a = {0.f, 0.f};
    each<VPT>(vecs, t, threads, [&](int i, int) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const F2 c = LAYER ? add2(v[r][i].p[k], {m, m}) : v[r][i].p[k];
        a = fma2(c, c, a);
      }
    });
    q[r] = a.x + a.y;
  }
  wq = warp_sums<NR>(q, u.lane);
  if (writes) {
    mine[u.warp] = wq;
    if (LAYER) mine[32 + u.warp] = ws;
  }
  auto weigh = [&] {
    if (w.src != nullptr)
      each<VPT>(vecs, t, threads, [&](int i, int j) {
        const V8 f = w.get(i, j);
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[r][i].p[k] = mul2(v[r][i].p[k], f.p[k]);
      });
  };
  if (!LAYER) weigh();  // under the barrier's wait
  float mean = -ws * u.per_row;
  if (!WARP_ROW) {
    __syncthreads();
    auto across = [&](float x) {  // over the lanes of one row
#pragma unroll
      for (int d = NR == 1 ? 16 : 8; d > 0; d >>= 1)
        x += __shfl_xor_sync(0xffffffffu, x, d);
      return x;
    };
    float sl[NR];
    wq = 0.f;
    if (LAYER) {
      ws = 0.f;
#pragma unroll
      for (int k = 0; k < NR; ++k) ws += sl[k] = mine[32 + u.other(k)];
      mean = -across(ws) * u.per_row;
#pragma unroll
      for (int k = 0; k < NR; ++k) {
        const float d = fmaf(sl[k], u.per[k], mean);
        wq += fmaf(u.n[k] * d, d, mine[u.other(k)]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < NR; ++k) wq += mine[u.other(k)];
    }
    wq = across(wq);
  }
  const float f = rsqrtf(fmaf(wq, u.per_row, eps));
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    inv[r] = pick<NR>(f, r);
    if (LAYER) {
      const float m = pick<NR>(mean, r);
      each<VPT>(vecs, t, threads, [&](int i, int) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          v[r][i].p[k] = add2(v[r][i].p[k], {m, m});
      });
    }
  }
  if (LAYER) weigh();
}

// One half (eight values, rounded to T) of a 16-element block whose other
// half the neighbouring lane holds -> its four bytes of codes and the block's
// scale byte, as the activation quantiser's (quant.cuh).  All lanes of a warp
// call it.
template <typename T>
__device__ __forceinline__ uint32_t quant_half(const Raw8<T>& z, uint8_t& sb) {
  uint32_t x[8], key = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const F2 v = z.pair(i);
    x[2 * i] = __float_as_uint(v.x);
    x[2 * i + 1] = __float_as_uint(v.y);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) key = max(key, x[i] & 0x7FFFFFFFu);
  key = max(key, __shfl_xor_sync(0xffffffffu, key, 1));
  const float amax = __uint_as_float(key);
  sb = __nv_cvt_float_to_fp8(amax / 6.0f, __NV_SATFINITE, __NV_E4M3);
  const float2 r = rcp_pair(sb);
  uint32_t w = sb != 0 ? e2m1_scaled8(x, r.x, r.y) : 0u;
  // a block holding a NaN goes to the compare form, which takes all sixteen
  if (__any_sync(0xffffffffu, key > 0x7F800000u)) {
    const bool hi = threadIdx.x & 1;
    constexpr int kWords = sizeof(T) * 2;
    uint32_t f[2 * kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const uint32_t own = z.w[i];
      const uint32_t other = __shfl_xor_sync(0xffffffffu, own, 1);
      f[i] = hi ? other : own;
      f[kWords + i] = hi ? own : other;
    }
    if (key > 0x7F800000u) {
      uint32_t w0, w1;
      if constexpr (sizeof(T) == 2) {
        sb = quant_block16_x2_cmp<Pair<T>>(f, w0, w1);
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

// NR rows from `row` (the first `live` of them exist): v holds y (x where there
// is no y); x(r, i, j) and gate(r, i, j) give those vectors when they are
// needed; `consumed` runs once every thread of the rows has asked for all.
template <typename T, bool WARP_ROW, bool LAYER, int NR, int VPT, typename P,
          typename X, typename G, typename C>
__device__ __forceinline__ void finish_rows(const nvfp4_block_norm_args& a,
                                            const P& w, int row, int live,
                                            int vecs, int t, int threads,
                                            V8 (&v)[NR][VPT], X x, G gate,
                                            C consumed,
                                            const Sums<WARP_ROW, NR>& sums,
                                            float* slots) {
  float inv[NR];
  if (a.y != nullptr) {
    float s[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) s[r] = a.scale;
    if (a.post) {
      norm_factors<WARP_ROW, LAYER, NR, VPT>(v, vecs, t, threads, a.eps,
                                             w.post_weight, sums, slots, inv);
      if (w.post_bias.src != nullptr)
        each<VPT>(vecs, t, threads, [&](int i, int j) {
          const V8 b = w.post_bias.get(i, j);
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              v[r][i].p[k] = fma2(v[r][i].p[k], {inv[r], inv[r]}, b.p[k]);
        });
      else
#pragma unroll
        for (int r = 0; r < NR; ++r) s[r] *= inv[r];
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      T* R = static_cast<T*>(a.R) + (size_t)(row + r) * a.ldr;
      each<VPT>(vecs, t, threads, [&](int i, int j) {
        if (a.gate != nullptr) {
          const Raw8<T> g = gate(r, i, j);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[r][i].p[k] = mul2(v[r][i].p[k], g.pair(k));
        }
        const Raw8<T> xr = x(r, i, j);
        Raw8<T> o;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          o.set(k, fma2(v[r][i].p[k], {s[r], s[r]}, xr.pair(k)));
          v[r][i].p[k] = o.pair(k);
        }
        if (r < live) o.store(R + 8 * j);
      });
    }
  }
  if (a.Z == nullptr && a.codes == nullptr) {
    if (!WARP_ROW) __syncthreads();
    consumed();
    return;
  }
  norm_factors<WARP_ROW, LAYER, NR, VPT>(v, vecs, t, threads, a.eps, w.weight,
                                         sums, slots + 64 * NR, inv);
  consumed();  // after the barrier of the sums
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int j = t + i * threads;
    const bool in = j < vecs;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      Raw8<T> z;
      if (in) {
        if (w.bias.src != nullptr) {
          const V8 b = w.bias.get(i, j);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            z.set(k, fma2(v[r][i].p[k], {inv[r], inv[r]}, b.p[k]));
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            z.set(k, mul2(v[r][i].p[k], {inv[r], inv[r]}));
        }
        if (a.Z != nullptr && r < live)
          z.store(static_cast<T*>(a.Z) + (size_t)(row + r) * a.ldz + 8 * j);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) z.set(k, {0.f, 0.f});
      }
      if (a.codes == nullptr) continue;
      uint8_t sb;
      const uint32_t c = quant_half<T>(z, sb);
      if (in && r < live)
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.codes) +
                                     (size_t)(row + r) * (a.D / 2) + 4 * j) =
            c;
      // the eight lanes of 64 elements hold four scales, each twice
      const uint32_t s1 = __shfl_down_sync(0xffffffffu, sb, 2);
      const uint32_t s2 = __shfl_down_sync(0xffffffffu, sb, 4);
      const uint32_t s3 = __shfl_down_sync(0xffffffffu, sb, 6);
      if ((j & 7) == 0 && in && r < live)
        *scale_word(a, row + r, j / 8) =
            static_cast<uint32_t>(sb) | (s1 << 8) | (s2 << 16) | (s3 << 24);
    }
  }
}

template <typename T, int VPT>
__device__ __forceinline__ void unpack_row(const Raw8<T> (&r)[VPT],
                                           V8 (&v)[VPT]) {
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) v[i].p[k] = r[i].pair(k);
}

// One row for each warp (WARP_ROW) or CTA: rows of up to 1024 elements, and
// wider ones when there are too few to go round.  Every load is issued before
// the first sum.
template <typename T, int VPT, bool WARP_ROW, bool LAYER, int MAXT>
__global__ void __launch_bounds__(MAXT)
    block_norm_kernel(const __grid_constant__ NormParams p) {
  __shared__ float slots[128];
  const nvfp4_block_norm_args& a = p.a;
  const int t = WARP_ROW ? threadIdx.x % 32 : threadIdx.x;
  const int threads = WARP_ROW ? 32 : blockDim.x;
  const int row = WARP_ROW ? blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32
                           : blockIdx.x;
  griddep_launch_dependents();
  if (!WARP_ROW) {
    for (int i = t; i < 128; i += threads) slots[i] = 0.f;
    __syncthreads();
  }
  griddep_wait();
  const int vecs = a.D / 8;
  if (row >= a.rows) {
    if (row < p.rows_pad)
      for (int g = t; g < vecs / 8; g += threads) *scale_word(a, row, g) = 0u;
    return;
  }
  Sums<WARP_ROW, 1> sums;
  sums.template set<VPT>(vecs, threads, a.D);
  Raw8<T> x[VPT], y[VPT], g[VPT];
  each<VPT>(vecs, t, threads, [&](int i, int j) {
    x[i].load(static_cast<const T*>(a.x) + (size_t)row * a.ldx + 8 * j);
    if (a.y != nullptr)
      y[i].load(static_cast<const T*>(a.y) + (size_t)row * a.ldy + 8 * j);
    if (a.gate != nullptr)
      g[i].load(static_cast<const T*>(a.gate) +
                (size_t)(row / p.gate_run) * a.D + 8 * j);
  });
  Params<T, VPT, VPT == 1, VPT == 1> w;
  w.set(a, vecs, t, threads);
  V8 v[1][VPT];
  if (a.y != nullptr)
    unpack_row<T, VPT>(y, v[0]);
  else
    unpack_row<T, VPT>(x, v[0]);
  finish_rows<T, WARP_ROW, LAYER, 1, VPT>(
      a, w, row, 1, vecs, t, threads, v, [&](int, int i, int) { return x[i]; },
      [&](int, int i, int) { return g[i]; }, [] {}, sums, slots);
}

// Many wide rows: a CTA works through pairs of rows, and bulk copies bring the
// next pairs of x, y (and of a gate that differs from row to row) into shared
// memory while it computes: the copies in flight do not depend on how many
// warps wait in a row's sums.  A thread holds one vector of both rows, so that
// each barrier serves two sums, and the norms' weights stay in its registers.
// (8192 x 7168 bf16: one row a CTA without the ring 130 us, with it 112; fp32
// pairs 98; two rows 85; their sums in one set of shuffles and no divisions
// 75.  With the weights read from L1 for every row, 151.)
constexpr int kPairRows = 2;

template <typename T, bool LAYER, int MAXT, int CTAS>
__global__ void __launch_bounds__(MAXT, CTAS)
    block_norm_rows_kernel(const __grid_constant__ NormParams p) {
  constexpr int NR = kPairRows;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float slots[2][128 * NR];
  __shared__ __align__(8) uint64_t full_bar[kMaxDepth];
  const nvfp4_block_norm_args& a = p.a;
  const int t = threadIdx.x, threads = blockDim.x;
  const int vecs = a.D / 8;
  const uint32_t row_bytes = a.D * sizeof(T);
  const bool gate_rows = a.gate != nullptr && a.gate_rows > 1;
  const uint32_t srcs = 1 + (a.y != nullptr) + gate_rows;
  const uint32_t stage_bytes = NR * srcs * row_bytes;
  if (t == 0) {
    for (int i = 0; i < kMaxDepth; ++i) mbar_init(&full_bar[i], 1);
    fence_mbar_init();
    fence_proxy_async_smem();
    s_wait_failed = 0u;
  }
  for (int i = t; i < 2 * 128 * NR; i += threads) slots[0][i] = 0.f;
  griddep_launch_dependents();
  __syncthreads();
  griddep_wait();
  // a stage: for each row y (where there is one), x and the gate; behind the
  // last row the last row again
  auto fetch = [&](int pair, int stage) {  // thread 0
    uint8_t* dst = ring + stage * stage_bytes;
    uint64_t* bar = &full_bar[stage];
    mbar_arrive_expect_tx(bar, stage_bytes);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int row = min(pair * NR + r, a.rows - 1);
      if (a.y != nullptr) {
        bulk_load(dst, static_cast<const T*>(a.y) + (size_t)row * a.ldy,
                  row_bytes, bar, kPolicyEvictFirst);
        dst += row_bytes;
      }
      bulk_load(dst, static_cast<const T*>(a.x) + (size_t)row * a.ldx,
                row_bytes, bar, kPolicyEvictFirst);
      dst += row_bytes;
      if (gate_rows) {
        bulk_load(dst,
                  static_cast<const T*>(a.gate) +
                      (size_t)(row / p.gate_run) * a.D,
                  row_bytes, bar, kPolicyEvictNormal);
        dst += row_bytes;
      }
    }
  };
  const int stride = gridDim.x;
  const int pairs = (a.rows + NR - 1) / NR;
  int ahead = blockIdx.x;  // thread 0: next pair to fetch
  if (t == 0) {
    for (int i = 0; i < p.depth && ahead < pairs; ++i, ahead += stride)
      fetch(ahead, i);
  }
  Sums<false, NR> sums;
  sums.template set<1>(vecs, threads, a.D);
  Params<T, 1, true, false> w;
  w.set(a, vecs, t, threads);
  int stage = 0, it = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int pair = blockIdx.x; pair < pairs; pair += stride, ++it) {
    // (after a wait that ran out the values are stale, every access is in
    // bounds and the error word reports it; the sums' barriers are still met)
    ok = mbar_wait(&full_bar[stage], phase, p.err, kErrProducer) && ok;
    const T* src = reinterpret_cast<const T*>(ring + stage * stage_bytes);
    const uint32_t x_at = a.y != nullptr ? a.D : 0;
    V8 v[NR][1];
    if (t < vecs) {
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        Raw8<T> u;
        u.load(src + r * srcs * a.D + 8 * t);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[r][0].p[k] = u.pair(k);
      }
    }
    finish_rows<T, false, LAYER, NR, 1>(
        a, w, pair * NR, min(NR, a.rows - pair * NR), vecs, t, threads, v,
        [&](int r, int, int j) {
          Raw8<T> u;
          u.load(src + r * srcs * a.D + x_at + 8 * j);
          return u;
        },
        [&](int r, int, int j) {
          Raw8<T> u;
          u.load(gate_rows ? src + (r + 1) * srcs * a.D - a.D + 8 * j
                           : static_cast<const T*>(a.gate) + 8 * j);
          return u;
        },
        [&] {
          if (t == 0 && ahead < pairs && ok) {
            fence_proxy_async_smem();  // the reads, before the refill
            fetch(ahead, stage);
            ahead += stride;
          }
        },
        sums, slots[it & 1]);
    if (++stage == p.depth) {
      stage = 0;
      phase ^= 1u;
    }
  }
  // after a wait that ran out, copies may be in flight: let them land
  if (t == 0 && !ok) {
    const int n = (ahead - static_cast<int>(blockIdx.x)) / stride;
    for (int i = max(0, n - p.depth); i < n; ++i)
      mbar_wait(&full_bar[i % p.depth], (i / p.depth) & 1, p.err, kErrDrain,
                /*bail_on_err=*/false);
  }
  for (int row = a.rows + blockIdx.x; row < p.rows_pad; row += stride)
    for (int g = t; g < vecs / 8; g += threads) *scale_word(a, row, g) = 0u;
}

// Bytes of a stage of block_norm_rows_kernel, and the most it may use.
int rows_stage(const nvfp4_block_norm_args& a, int elem) {
  const int srcs = 1 + (a.y != nullptr) +
                   (a.gate != nullptr && a.gate_rows > 1);
  return kPairRows * srcs * a.D * elem;
}
constexpr int kRowsSmem = 216 * 1024;

template <typename T, bool LAYER, int MAXT, int CTAS>
int launch_rows(NormParams p, int sms, int dev, int threads,
                cudaLaunchConfig_t& cfg) {
  static std::atomic<unsigned long long> ready{0};
  static std::atomic<int> regs{0};
  auto kernel = block_norm_rows_kernel<T, LAYER, MAXT, CTAS>;
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(ready.load() & bit)) {
    cudaFuncAttributes fa;
    cudaError_t e = cudaFuncGetAttributes(&fa, kernel);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncGetAttributes");
    regs = (fa.numRegs + 7) / 8 * 8;
    e = cudaFuncSetAttribute(
        kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute");
    ready.fetch_or(bit);
  }
  // CTAs an SM holds by its registers (a persistent grid must fit at once)
  // and with two stages or more each
  const int stage = rows_stage(p.a, sizeof(T));
  int ctas =
      std::min(65536 / (regs.load() * threads), kRowsSmem / (2 * stage));
  ctas = std::max(1, std::min(ctas, 8));
  p.depth = std::min(kMaxDepth, (kRowsSmem / ctas - 2048) / stage);
  cfg.gridDim = dim3(std::min((p.a.rows + 1) / 2, sms * ctas), 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(p.depth) * stage;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess)
    return host_cuda_fail(e, "block_norm_rows_kernel launch");
  return NVFP4DG_OK;
}

template <typename T, bool LAYER>
int launch_norm(const NormParams& p, int sms, int dev, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = (p.a.flags & NVFP4DG_FLAG_NO_PDL) ? 0 : 1;
  const int vecs = p.a.D / 8;
  auto cover = [&](int vpt) {  // threads of vpt vectors each
    return ((vecs + vpt - 1) / vpt + 31) / 32 * 32;
  };
  void (*kernel)(NormParams);
  if (vecs <= 128) {  // a warp holds the row
    const int threads = p.rows_pad >= 4 * sms ? 256 : 64;
    cfg.gridDim = dim3((p.rows_pad + threads / 32 - 1) / (threads / 32), 1, 1);
    cfg.blockDim = dim3(threads, 1, 1);
    kernel = vecs <= 32   ? block_norm_kernel<T, 1, true, LAYER, 256>
             : vecs <= 64 ? block_norm_kernel<T, 2, true, LAYER, 256>
                          : block_norm_kernel<T, 4, true, LAYER, 256>;
  } else {
    if (p.a.rows > 2 * sms && vecs <= 1024 &&
        rows_stage(p.a, sizeof(T)) <= kRowsSmem - 2048)
      return vecs <= 512
                 ? launch_rows<T, LAYER, 512, 2>(p, sms, dev, cover(1), cfg)
                 : launch_rows<T, LAYER, 1024, 1>(p, sms, dev, cover(1), cfg);
    const int vpt = vecs <= 1024 ? 1 : vecs <= 2048 ? 2 : 4;
    cfg.gridDim = dim3(p.rows_pad, 1, 1);
    cfg.blockDim = dim3(cover(vpt), 1, 1);
    kernel = vpt == 1   ? block_norm_kernel<T, 1, false, LAYER, 1024>
             : vpt == 2 ? block_norm_kernel<T, 2, false, LAYER, 1024>
                        : block_norm_kernel<T, 4, false, LAYER, 1024>;
  }
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) return host_cuda_fail(e, "block_norm_kernel launch");
  return NVFP4DG_OK;
}

template <typename T>
int launch_norm(const NormParams& p, int sms, int dev, cudaStream_t stream) {
  return p.a.kind == NVFP4DG_NORM_LAYER
             ? launch_norm<T, true>(p, sms, dev, stream)
             : launch_norm<T, false>(p, sms, dev, stream);
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
  // a thread writes the elements of x and y that it has read, and no others:
  // in place is safe, a shift is not
  const long long e = a->dtype == NVFP4DG_DTYPE_F32 ? 4 : 2;
  auto lie = [&](const void* p, long long ldp, const void* q, long long ldq) {
    return host_overlap(p, ldp * e, q, ldq * e, a->rows, a->D * e);
  };
  void* const r = a->y != nullptr ? a->R : nullptr;
  if (lie(r, a->ldr, a->Z, a->ldz) != Overlap::kNone)
    return host_fail(NVFP4DG_ERR_INVALID, "R and Z must not overlap");
  if (lie(r, a->ldr, a->x, a->ldx) == Overlap::kPart ||
      lie(r, a->ldr, a->y, a->ldy) == Overlap::kPart ||
      lie(a->Z, a->ldz, a->x, a->ldx) == Overlap::kPart ||
      lie(a->Z, a->ldz, a->y, a->ldy) == Overlap::kPart)
    return host_fail(NVFP4DG_ERR_INVALID,
                     "R and Z must each be x or y themselves or overlap "
                     "neither");
  // what other rows' CTAs read, and what only they write
  const long long w = (a->w_dtype == NVFP4DG_DTYPE_F32 ? 4ll : 2ll) * a->D;
  struct Bytes {
    const char* name;
    const void* p;
    long long n;
  };
  const Bytes shared[] = {
      {"weight", a->weight, w},
      {"bias", a->bias, w},
      {"post_weight", a->post_weight, w},
      {"post_bias", a->post_bias, w},
      {"gate", a->gate, a->gate != nullptr ? a->gate_rows * (a->D * e) : 0},
  };
  for (const Bytes& in : shared)
    if (host_meets(in.p, in.n, r, a->ldr * e, a->rows, a->D * e) ||
        host_meets(in.p, in.n, a->Z, a->ldz * e, a->rows, a->D * e))
      return host_fail(NVFP4DG_ERR_INVALID,
                       std::string(in.name) + " must not overlap R or Z");
  if (a->codes != nullptr) {
    const Bytes outs[] = {
        {"codes", a->codes, a->rows * (a->D / 2ll)},
        {"sf", a->sf, (a->rows + 127ll) / 128 * (a->D / 64) * kAtomBytes}};
    bool meets = host_meets(outs[0].p, outs[0].n, outs[1].p, outs[1].n, 1,
                            outs[1].n);
    for (const Bytes& out : outs) {
      for (const Bytes& in : shared)
        meets |= host_meets(out.p, out.n, in.p, in.n, 1, in.n);
      for (int i = 0; i < 4; ++i)
        meets |= host_meets(out.p, out.n, i == 2 ? r : mats[i], lds[i] * e,
                            a->rows, a->D * e);
    }
    if (meets)
      return host_fail(NVFP4DG_ERR_INVALID,
                       "codes and sf must not overlap one another or any "
                       "other tensor");
  }
  return NVFP4DG_OK;
}

int run_norm(const nvfp4_block_norm_args* a, void* stream) {
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
  p.depth = 0;
  p.err = dev.err;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->dtype == NVFP4DG_DTYPE_F32)
    return launch_norm<float>(p, dev.sms, dev.id, s);
  if (a->dtype == NVFP4DG_DTYPE_F16)
    return launch_norm<__half>(p, dev.sms, dev.id, s);
  return launch_norm<__nv_bfloat16>(p, dev.sms, dev.id, s);
}

}  // namespace
}  // namespace nvfp4dg

extern "C" int nvfp4_block_norm_run(const nvfp4_block_norm_args* a,
                                    void* stream) {
  return nvfp4dg::host_guarded([&] { return nvfp4dg::run_norm(a, stream); });
}
