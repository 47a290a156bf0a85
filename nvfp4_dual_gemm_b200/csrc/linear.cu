// linear.cu — NVFP4 products with a fused epilogue, and the same products
// grouped by expert:
//
//   C[m, n] = act(alpha * sum_k A[m, k] B[n, k] + bias[n]) * row_scale[m]
//             + residual[m, n]
//
// A (activations, [M, K]) and B (weights, [N, K]) are NVFP4 with blocked
// scales, as for the dual GEMM; C is fp16 or bf16.
//
// Two kernels.  linear_kernel: one CTA a tile of 128 features and 32 or 64
// tokens, the features on the TMEM lanes and the tokens on the accumulator's
// columns (C^T = B A^T): with few tokens, which is where the product is bound
// by reading B once, the column side shrinks while every lane still works, and
// a stage of the operand ring is nearly all weights.  With 128 tokens the two
// change places.  linear_pair_kernel: two SMs a tile of 256 tokens x 256
// features, for many tokens, where the tensor cores' feed is the bound.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <string>
#include <type_traits>

#include "host.h"
#include "nvfp4_dual_gemm.h"
#include "sm100_ptx.cuh"

namespace nvfp4dg {
namespace {

constexpr int kFeat = 128;          // features (rows of B) per tile
constexpr int kRowBytes = 128;      // a stage holds 256 fp4 of K per row
constexpr int kAtomBytes = 512;     // scales of 128 rows x 64 K elements
constexpr int kRunBytes = 4 * kAtomBytes;
constexpr int kThreads = 480;
constexpr int kEpiWarps = 8;        // warps 0-3 and 11-14, see epi_group
constexpr int kProdWWarp = 4;       // copies weights and their scales
constexpr int kProdXWarp = 5;       // copies tokens and their scales
constexpr int kMmaWarp = 6;
constexpr int kSfWarp0 = 7;         // four warps, one per TMEM sub-partition
constexpr int kSfWarps = 4;
constexpr int kEpiWarp1 = 11;
constexpr int kTmemCols = 512;
constexpr int kMaxStages = 8;
constexpr int kMaxGroups = 256;
constexpr int kSmemBudget = 221 * 1024;  // dynamic; static holds the groups

struct LinearParams {
  int M, N, K;       // M: rows of A and C (of all groups)
  int kblocks;       // K blocks of a tile (the kernel's block: 256 or 512)
  int n_tiles;       // ceil(N / 128)
  int m_tiles;       // ceil(M / TN) (one problem)
  int split;         // CTAs of a cluster that share a tile's K range
  int stages;
  const uint8_t* sfa;
  const uint8_t* sfb;
  long long sfb_group;  // bytes from one group's weight scales to the next
  void* C;
  long long ldc;
  const void* bias;
  int bias_f32;
  const void* residual;
  long long ldr;
  const float* row_scale;
  float alpha;
  int act;
  unsigned* err;
  // grouped products: row counts and first rows, from device memory where
  // dev_rows is set (dev_row0 may be null: each group starts at the next
  // multiple of 128), else from the arrays here
  int groups;
  const int* dev_rows;
  const int* dev_row0;
  int rows[kMaxGroups];
  int row0[kMaxGroups];
};

// Grouped products: group g's rows start at row0 of A and C and its tiles are
// [tile0[g], tile0[g + 1]).
struct GroupTable {
  int tile0[kMaxGroups + 1];
  int row0[kMaxGroups];
};

// Rows of group g, whose first row lies in the matrix: its count, cut at the
// last row.  (Read again for each tile, from L1 or the constant cache, to
// leave shared memory to the operands.)
__device__ __forceinline__ int group_rows(const LinearParams& p, int g,
                                          int row0) {
  const int n = p.dev_rows ? p.dev_rows[g] : p.rows[g];
  return min(max(n, 0), p.M - row0);
}

// The last group whose first tile is <= tile (empty groups have none), found
// by a whole warp: each lane looks at groups lane, lane + 32, ..., and the
// groups that start at or below the tile are counted by votes.  (A search by
// the one thread that needs it took ~1500 cycles a tile, as long as a tile of
// short K.)
__device__ __forceinline__ int find_group(const LinearParams& p,
                                          const GroupTable& tab, int tile) {
  const int lane = threadIdx.x % 32;
  int n = 0;
  for (int g = lane; g - lane < p.groups; g += 32)
    n += __popc(__ballot_sync(0xffffffffu,
                              g < p.groups && tab.tile0[g] <= tile));
  return n - 1;
}

struct Tile {
  int g;       // group (batch of B)
  int n0;      // first feature
  int x0;      // first row of A / C
  int rows;    // valid rows from x0 (may exceed the tile)
};

// Built by one warp at the kernel's start.  Counts and first rows may come
// from the device, so nothing about them was checked on the host: a group
// whose first row is no multiple of 128 or lies outside the matrix gets no
// rows, and no group reaches past row M.
__device__ __forceinline__ void build_groups(const LinearParams& p, int tn,
                                             int lane, GroupTable& tab) {
  long long row_end = 0;
  int tile_end = 0;
  for (int base = 0; base < p.groups; base += 32) {
    const int g = base + lane;
    const bool in = g < p.groups;
    int n = 0;
    if (in) n = max(0, p.dev_rows ? p.dev_rows[g] : p.rows[g]);
    // inclusive sums over the warp
    long long pad = (static_cast<long long>(n) + 127) / 128 * 128;
    const long long own = pad;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, pad, d);
      if (lane >= d) pad += o;
    }
    long long r0 = row_end + pad - own;
    row_end += __shfl_sync(0xffffffffu, pad, 31);
    if (in) {
      if (p.dev_rows == nullptr)
        r0 = p.row0[g];
      else if (p.dev_row0 != nullptr)
        r0 = p.dev_row0[g];
    }
    if (r0 < 0 || r0 >= p.M || (r0 & 127)) n = 0;
    n = static_cast<int>(
        min(static_cast<long long>(n), max(p.M - r0, 0ll)));
    int tiles = (n + tn - 1) / tn * p.n_tiles;
    const int mine = tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, tiles, d);
      if (lane >= d) tiles += o;
    }
    if (in) {
      tab.tile0[g] = tile_end + tiles - mine;
      tab.row0[g] = n ? static_cast<int>(r0) : 0;
    }
    tile_end += __shfl_sync(0xffffffffu, tiles, 31);
  }
  if (lane == 0) tab.tile0[p.groups] = tile_end;
}

// Token tiles fastest, so that CTAs of neighbouring tiles read the same
// weights at the same time.  Called by whole warps.
template <int TN>
__device__ __forceinline__ Tile locate(const LinearParams& p,
                                       const GroupTable& tab, int tile) {
  Tile t;
  if (p.groups == 0) {
    const int nt = p.m_tiles == 1 ? tile : tile / p.m_tiles;
    t.g = 0;
    t.n0 = nt * kFeat;
    t.x0 = (tile - nt * p.m_tiles) * TN;
    t.rows = p.M - t.x0;
    return t;
  }
  const int g = find_group(p, tab, tile);
  const int local = tile - tab.tile0[g];
  const int row0 = tab.row0[g];
  const int rows = group_rows(p, g, row0);
  const int mt = (rows + TN - 1) / TN;
  const int nt = mt == 1 ? local : local / mt;
  const int m0 = (local - nt * mt) * TN;
  t.g = g;
  t.n0 = nt * kFeat;
  t.x0 = row0 + m0;
  t.rows = rows - m0;
  return t;
}

// Whether the phase has completed, without waiting.  A wait on a barrier takes
// ~300 cycles even when its phase is already complete, so each role of
// linear_kernel asks for its next stage before it works on the present one and
// waits only when the answer was no (16 x 128 x 14336, one CTA: 26.4 -> 24.7
// us).
__device__ __forceinline__ bool mbar_peek(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// A counter in shared memory that one thread of the CTA raises and another
// waits for (release and acquire, so what the first saw the second sees);
// bounded as mbar_wait is.
__device__ __forceinline__ void flag_set(uint32_t* flag, uint32_t v) {
  asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(
                   smem_u32(flag)),
               "r"(v)
               : "memory");
}
__device__ __forceinline__ bool flag_wait(uint32_t* flag, uint32_t target,
                                          unsigned* err, unsigned code) {
  long long t0 = 0;
  for (uint32_t i = 1;; ++i) {
    uint32_t v;
    asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];"
                 : "=r"(v)
                 : "r"(smem_u32(flag))
                 : "memory");
    if (static_cast<int32_t>(v - target) >= 0) return true;
    if ((i & 4095u) == 0u) {
      const long long now = clock_cycles();
      if (t0 == 0) t0 = now;
      const bool gone = *reinterpret_cast<volatile unsigned*>(err) != 0u;
      if (gone || now - t0 > kWaitLimitCycles) {
        if (!gone) atomicOr(err, code);
        note_wait_failed();
        return false;
      }
    }
  }
}

// Arrives on `bar` of both CTAs of the pair when this thread's 2-SM MMAs are
// done.
__device__ __forceinline__ void tc_commit_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster."
      "multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

// A warpgroup's share of the registers (all four warps together).
template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// 4 consecutive 32-bit TMEM columns of this warp's 32 lanes.
__device__ __forceinline__ void tc_ld_4cols(uint32_t taddr, float (&v)[4]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(taddr)
      : "memory");
}

// The epilogue warps form two groups of four that share a tile's columns: warp
// w of a group owns TMEM lanes 32 (w % 4) .. + 31.  One group of four took
// longer for a tile of short K than the products of the next one.
__device__ __forceinline__ int epi_group(int warp) {
  return warp >= kEpiWarp1 ? 1 : 0;
}
// Barrier of one group, and one that also ANDs a predicate.
__device__ __forceinline__ void epi_bar(int group) {
  asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory");
}
__device__ __forceinline__ bool epi_all(int group, bool pred) {
  uint32_t out;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(out)
      : "r"(static_cast<uint32_t>(pred)), "r"(group + 1)
      : "memory");
  return out != 0;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
  return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// x / (1 + 2^t), given t - kFar: two special-function operations and three
// others.  The denominator is taken 2^-kFar times as large, and its reciprocal
// brought back by an exact factor: a reciprocal below 2^-126 is flushed to
// zero, which would lose results from t = 126 on (silu of x < -87.3) although
// they are normal numbers of bf16 up to t = 132 and of any consequence to it
// up to t = 141, the new limit.  Beyond, and where the denominator is infinite,
// the quotient is a zero.  kFar = 15 keeps t - kFar below 16 where t is small,
// so that its rounding costs at most 2^-21.
// (Packed pairs save two instructions of eleven, but the few-token kernels then
// hold their rows in aligned registers whatever the activation: 1 x 4096 x 4096
// took 5.90 instead of 5.75 us, 64 experts of 2 rows 16.4 instead of 15.8, 16
// of ~94 rows with silu the same 27.4.  The reciprocal by Newton steps on the
// FMA pipe halves the special-function operations and doubles the instructions:
// the last of these cases took 29.7 us without them, 31.9 with.)
constexpr float kFar = 15.f;
__device__ __forceinline__ float quotient(float x, float t) {
  constexpr float kScale = 1.f / 32768.f;  // 2^-kFar
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(kScale + e));
  return x * (r * kScale);
}

// Not inlined: 32 copies of erfc would cost the epilogue its registers.
__device__ __noinline__ float gelu_erf(float x) {
  return 0.5f * x * erfcf(-0.7071067811865476f * x);
}

// act(v), NC values, in fp32.  silu(x) = x / (1 + e^-x);
// 0.5 (1 + tanh u) = 1 / (1 + e^-2u), so the tanh form of gelu is
// x / (1 + e^-2u) with u = sqrt(2/pi) (x + 0.044715 x^3); the erf form is
// 0.5 x erfc(-x / sqrt 2), which keeps its digits for negative x.
template <int NC>
__device__ __forceinline__ void activate(float (&v)[NC], int act) {
  if (act == NVFP4DG_ACT_NONE) return;
  if (act == NVFP4DG_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < NC; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];  // keeps NaN
  } else if (act == NVFP4DG_ACT_SILU) {
    constexpr float k = -1.4426950408889634f;  // -log2(e)
#pragma unroll
    for (int i = 0; i < NC; ++i) v[i] = quotient(v[i], fmaf(k, v[i], -kFar));
  } else if (act == NVFP4DG_ACT_GELU_TANH) {
    constexpr float k = -2.302208198201456f;  // -2 sqrt(2/pi) log2(e)
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const float x = v[i];
      v[i] = quotient(x, fmaf(x, fmaf(0.044715f * k, x * x, k), -kFar));
    }
  } else {
#pragma unroll
    for (int i = 0; i < NC; ++i) v[i] = gelu_erf(v[i]);
  }
}

template <typename T>
__device__ __forceinline__ float load_bias(const LinearParams& p, int g,
                                           int n) {
  if (p.bias == nullptr || n >= p.N) return 0.f;
  const size_t i = (size_t)g * p.N + n;
  return p.bias_f32 ? static_cast<const float*>(p.bias)[i]
                    : to_f32<T>(static_cast<const T*>(p.bias)[i]);
}

// Residual of NC rows of C from row x (valid: `nv` of them), feature n.  Rows
// are addressed by 32-bit offsets from the first one, which is the same for
// the whole warp.
template <typename T, int NC>
__device__ __forceinline__ void load_residual(const LinearParams& p, int x,
                                              int n, int nv, T (&r)[NC]) {
  if (p.residual == nullptr) return;
  const char* src = static_cast<const char*>(p.residual) +
                    (size_t)x * p.ldr * sizeof(T);
  uint32_t off = n * sizeof(T);
  const uint32_t step = p.ldr * sizeof(T);
  if (nv >= NC) {
#pragma unroll
    for (int i = 0; i < NC; ++i, off += step)
      r[i] = *reinterpret_cast<const T*>(src + off);
  } else {
#pragma unroll
    for (int i = 0; i < NC; ++i, off += step)
      if (i < nv) r[i] = *reinterpret_cast<const T*>(src + off);
  }
}

// Row scale of row x + i for lane i (valid: `nv` rows).
__device__ __forceinline__ float load_scale(const LinearParams& p, int x,
                                            int nv, int lane) {
  return p.row_scale != nullptr && lane < nv ? p.row_scale[x + lane] : 0.f;
}

// NP of finish's rows, from its c-th.
template <typename T, int NP, int NC>
__device__ __forceinline__ void finish_part(const LinearParams& p, char* dst,
                                            uint32_t off, uint32_t step,
                                            int c, int nv, float bias,
                                            float scale, const T (&r)[NC],
                                            float (&v)[NC]) {
  float(&w)[NP] = *reinterpret_cast<float(*)[NP]>(v + c);
#pragma unroll
  for (int i = 0; i < NP; ++i) w[i] = fmaf(p.alpha, w[i], bias);
  activate<NP>(w, p.act);
  if (p.row_scale != nullptr) {
#pragma unroll
    for (int i = 0; i < NP; ++i)
      w[i] *= __shfl_sync(0xffffffffu, scale, c + i);
  }
  if (p.residual != nullptr) {
#pragma unroll
    for (int i = 0; i < NP; ++i) w[i] += to_f32<T>(r[c + i]);
  }
  off += c * step;
#pragma unroll
  for (int i = 0; i < NP; ++i, off += step)
    if (c + i < nv) *reinterpret_cast<T*>(dst + off) = from_f32<T>(w[i]);
}

// Epilogue of NC rows (tokens) of one feature: the accumulators v to C.  `cnt`
// rows exist (the same for the whole warp), and `nv` of them are this
// thread's: cnt, or none for a feature beyond N.  Lane i holds row i's scale.
// All rows go at once (32 independent chains hide the latency of a warp that
// has its scheduler almost to itself), or, where rows are missing, eight at a
// time, so that a tile of few tokens does not pay for 32.
template <typename T, int NC>
__device__ __forceinline__ void finish(const LinearParams& p, int x, int n,
                                       int cnt, int nv, float bias,
                                       float scale, const T (&r)[NC],
                                       float (&v)[NC]) {
  char* dst = static_cast<char*>(p.C) + (size_t)x * p.ldc * sizeof(T);
  const uint32_t off = n * sizeof(T), step = p.ldc * sizeof(T);
  if (NC <= 8 || cnt > NC - 8) {
    finish_part<T, NC, NC>(p, dst, off, step, 0, nv, bias, scale, r, v);
  } else {
#pragma unroll
    for (int c = 0; c < NC - 8; c += 8)
      if (c < cnt)
        finish_part<T, NC < 8 ? NC : 8, NC>(p, dst, off, step, c, nv, bias,
                                            scale, r, v);
  }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16),
                     __uint_as_float(u & 0xFFFF0000u));
}

// The same epilogue where a thread is a token row: 32 columns of row x from
// column n.
template <typename T>
__device__ __forceinline__ void load_residual_row(const LinearParams& p,
                                                  int x, int n, bool live,
                                                  uint4 (&r)[4]) {
  if (p.residual == nullptr) return;
  const T* src = static_cast<const T*>(p.residual) + (size_t)x * p.ldr + n;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    r[q] = make_uint4(0u, 0u, 0u, 0u);
    if (live && n + 8 * q < p.N)
      r[q] = *reinterpret_cast<const uint4*>(src + 8 * q);
  }
}

// Elements 2i and 2i + 1.
__device__ __forceinline__ F2 get2(const float (&v)[32], int i) {
  return {v[2 * i], v[2 * i + 1]};
}
__device__ __forceinline__ void set2(float (&v)[32], int i, F2 x) {
  v[2 * i] = x.x;
  v[2 * i + 1] = x.y;
}

// `residual(q)` gives its eight elements from column 8 q, `emit(q, o)` takes
// the outputs there.
template <typename T, typename R, typename E>
__device__ __forceinline__ void finish_row32(const LinearParams& p,
                                             float scale, const float* bias,
                                             float (&v)[32], R residual,
                                             E emit) {
  const F2 alpha = {p.alpha, p.alpha};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 b = reinterpret_cast<const float4*>(bias)[i];
    set2(v, 2 * i, fma2(alpha, get2(v, 2 * i), {b.x, b.y}));
    set2(v, 2 * i + 1, fma2(alpha, get2(v, 2 * i + 1), {b.z, b.w}));
  }
  activate<32>(v, p.act);
  if (p.row_scale != nullptr) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      set2(v, i, mul2(get2(v, i), {scale, scale}));
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (p.residual != nullptr) {
      const uint4 r = residual(q);
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(w[i]);
        set2(v, 4 * q + i, add2(get2(v, 4 * q + i), {f.x, f.y}));
      }
    }
    emit(q, make_uint4(pack2<T>(v[8 * q + 0], v[8 * q + 1]),
                       pack2<T>(v[8 * q + 2], v[8 * q + 3]),
                       pack2<T>(v[8 * q + 4], v[8 * q + 5]),
                       pack2<T>(v[8 * q + 6], v[8 * q + 7])));
  }
}

// Eight outputs of row x from column n.
template <typename T>
__device__ __forceinline__ void store_row8(const LinearParams& p, int x, int n,
                                           const uint4& o) {
  *reinterpret_cast<uint4*>(static_cast<T*>(p.C) + (size_t)x * p.ldc + n) = o;
}

// A stage of linear_kernel's ring holds kSub blocks of 256 along K.  What a
// stage costs beyond its bytes, a wait of ~300 cycles in each role and the MMA
// thread's commit, made a 256-wide block take ~710 cycles whatever the tokens;
// two of them at once take ~535 each (16 x 4096 x 14336: 10.6 -> 10.1 us, by
// then bound by memory).  With 128 tokens a stage is deeper in bytes and one
// block wide.
template <int TN>
struct Cfg {
  // 128 tokens: the tokens take the TMEM lanes and 128 features the columns,
  // the other way round than with fewer.  A thread of the epilogue then holds
  // a row's consecutive columns, which halves its instructions.
  static constexpr bool kRows = TN == 128;
  static constexpr int kSub = TN <= 64 ? 2 : 1;
  static constexpr int kSteps = 4 * kSub;  // MMAs of 64 along K
  static constexpr int kWBox = kFeat * kRowBytes;
  static constexpr int kXBox = TN * kRowBytes;
  static constexpr int kWBytes = kSub * kWBox;
  static constexpr int kXBytes = kSub * kXBox;
  static constexpr int kRun = kSub * kRunBytes;
  static constexpr int kSfCols = 32 * kSub;  // TMEM columns of its scales
  static constexpr int kStageBytes = kWBytes + kXBytes + 2 * kRun;
  // split-K: the partials a CTA receives, fp32
  static constexpr int kRecvBytes = kFeat * TN * 4;
  static constexpr int kSfBase = 2 * TN;  // two accumulators, then scales
  static constexpr int kTmemStages = (kTmemCols - kSfBase) / kSfCols;
  static constexpr int stages(int split) {
    const int room = kSmemBudget - 1024 - (split > 1 ? kRecvBytes : 0);
    const int s = room / kStageBytes;
    const int cap = kTmemStages < kMaxStages ? kTmemStages : kMaxStages;
    return s < cap ? s : cap;
  }
  static constexpr int smem(int split) {
    return stages(split) * kStageBytes + (split > 1 ? kRecvBytes : 0) + 1024;
  }
  static_assert(kStageBytes % 1024 == 0, "stages stay 1024-byte aligned");
};

// Per K block the two producer warps copy [128 x 128 B] boxes of weights, [TN x
// 128 B] boxes of tokens and their scale runs into a ring stage; four scale
// warps move the scales into TMEM; one thread issues a block-scaled MMA
// (M = 128 features, N = TN tokens) for each 64 of K and eight warps finish
// the tile.  Two accumulators, so that a tile's epilogue runs under
// the next tile's products.  K needs only be a multiple of 64: the last
// block's missing 64-wide steps are not issued.
//
// split > 1: the CTAs of a cluster share one tile's K range.  Each sends the
// fp32 partials of the other ranks' token columns into their shared memory
// and finishes its own share, adding the partials in rank order.
//
// Bound by: reading B once (16 x 4096 x 14336, 33 MB: 10.1 us, 3.3 TB/s
// including ~4 us of start, exchange and end that short products consist of;
// 1 x 4096 x 4096: 5.7 us), and for several tiles a CTA by the chain of a K
// block or by the epilogue's instructions, whichever is longer.
template <typename T, int TN>
__global__ void __launch_bounds__(kThreads, 1)
    linear_kernel(const __grid_constant__ CUtensorMap tmW,
                  const __grid_constant__ CUtensorMap tmX,
                  const __grid_constant__ LinearParams p) {
  using Cf = Cfg<TN>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kMaxStages];
  __shared__ __align__(8) uint64_t sfdata_bar[kMaxStages];
  __shared__ __align__(8) uint64_t empty_bar[kMaxStages];
  __shared__ __align__(8) uint64_t acc_full_bar[2];
  __shared__ __align__(8) uint64_t acc_empty_bar[2];
  __shared__ __align__(8) uint64_t drain_bar;
  __shared__ __align__(8) uint64_t recv_bar;
  __shared__ uint32_t tmem_base_sh;
  __shared__ GroupTable tab;
  // kRows: the bias of a tile's features, for each epilogue group, by the
  // accumulator's parity
  __shared__ __align__(16) float
      bias_sh[2][2][Cfg<TN>::kRows ? 128 + 32 : 4];

  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const int S = p.stages;
  const int rank = p.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int kblk64 = p.K / 64;
  // A K block's scale run has the same size for every block: the last
  // block's, when it is short, starts earlier and its first atoms are
  // skipped (`skip` in the scale warps).
  const uint32_t run_bytes =
      static_cast<uint32_t>(min(Cf::kSteps, kblk64)) * kAtomBytes;

  if (warp == 0) {
    uint64_t* bar = nullptr;
    uint32_t count = 1;
    if (lane < 8) {
      bar = full_bar + lane;
      count = kSfWarps;  // the first one's arrival carries the tiles' bytes
    } else if (lane < 16) {
      bar = sfdata_bar + (lane - 8);
    } else if (lane < 24) {
      bar = empty_bar + (lane - 16);
    } else if (lane < 26) {
      bar = acc_full_bar + (lane - 24);
    } else if (lane < 28) {
      bar = acc_empty_bar + (lane - 26);
      count = kEpiWarps;
    } else if (lane == 28) {
      bar = &drain_bar;
    } else if (lane == 29) {
      bar = &recv_bar;
    }
    if (bar != nullptr) {
      mbar_init(bar, count);
      fence_mbar_init();
    }
    if (lane == 30) prefetch_tmap(&tmW);
    if (lane == 31) prefetch_tmap(&tmX);
    if (lane == 0) s_wait_failed = 0u;
    __syncwarp();
    // the first scale fill of every stage; later ones are armed by the scale
    // warps (bytes may land before their arming)
    if (lane < S) mbar_arrive_expect_tx(sfdata_bar + lane, 2 * run_bytes);
    fence_proxy_async_smem();
    __syncwarp();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&tmem_base_sh, kTmemCols);
    tmem_relinquish();
  }
  // the barriers of every CTA of the cluster before any remote use
  if (p.split > 1) cluster_arrive_relaxed();
  griddep_launch_dependents();
  if (p.groups > 0 && warp == 1) {
    if (p.dev_rows != nullptr) griddep_wait();
    build_groups(p, TN, lane, tab);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (p.split > 1) cluster_wait();
  const uint32_t tmem = tmem_base_sh;

  const int total =
      p.groups > 0 ? tab.tile0[p.groups] : p.n_tiles * p.m_tiles;
  const int first = static_cast<int>(blockIdx.x) / p.split;
  const int step = static_cast<int>(gridDim.x) / p.split;
  const int kb0 = static_cast<int>((long long)p.kblocks * rank / p.split);
  const int kb1 =
      static_cast<int>((long long)p.kblocks * (rank + 1) / p.split);

  if (warp == kProdWWarp || warp == kProdXWarp) {
    // ---------------------------------------------------------- producers
    // They only copy; the barriers' expected bytes come with the scale warps'
    // arrivals.
    {
      const bool w_side = warp == kProdWWarp;
      // the 128 lanes' operand comes through the first producer
      const bool weights = w_side != Cf::kRows;
      const CUtensorMap* tm = weights ? &tmW : &tmX;
      const uint64_t pol = weights ? kPolicyEvictNormal : kPolicyEvictLast;
      const uint32_t tile_off = w_side ? 0 : Cf::kWBytes;
      const uint32_t sf_off =
          Cf::kWBytes + Cf::kXBytes + (w_side ? 0 : Cf::kRun);
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      bool ok = true, ready = false;
      griddep_wait();  // global memory only after the previous grid
      for (int tile = first; ok && tile < total; tile += step) {
        const Tile t = locate<TN>(p, tab, tile);  // the whole warp
        const uint8_t* sf =
            weights ? p.sfb + (size_t)t.g * p.sfb_group +
                          (size_t)(t.n0 / 128) * kblk64 * kAtomBytes
                    : p.sfa + (size_t)(t.x0 / 128) * kblk64 * kAtomBytes;
        const int row = weights ? t.n0 : t.x0;
        const int layer = weights ? t.g : 0;
        for (int kb = kb0; lane == 0 && kb < kb1; ++kb) {
          if (issued >= S && !ready &&
              !mbar_wait(&empty_bar[stage], phase ^ 1u, p.err,
                         kErrProducer)) {
            ok = false;
            break;
          }
          const int next = stage + 1 == S ? 0 : stage + 1;
          const uint32_t next_phase = phase ^ (next == 0 ? 1u : 0u);
          ready = mbar_peek(&empty_bar[next], next_phase ^ 1u);
          uint8_t* st = smem + stage * Cf::kStageBytes;
          bulk_load(st + sf_off,
                    sf + (size_t)min(Cf::kSteps * kb,
                                     max(0, kblk64 - Cf::kSteps)) *
                             kAtomBytes,
                    run_bytes, &sfdata_bar[stage], pol);
#pragma unroll
          for (int h = 0; h < Cf::kSub; ++h)  // (zeros beyond K)
            tma_load_3d(st + tile_off + h * (w_side ? Cf::kWBox : Cf::kXBox),
                        tm, &full_bar[stage],
                        (kb * Cf::kSub + h) * kRowBytes, row, layer, pol);
          ++issued;
          stage = next;
          phase = next_phase;
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
      }
      // never leave with copies in flight
      for (int s = 0; s < S; ++s) {  // (lane 0 has issued all)
        if (issued > s) {
          const uint32_t par =
              static_cast<uint32_t>(((issued - 1 - s) / S) & 1);
          mbar_wait(&sfdata_bar[s], par, p.err, kErrDrain, false);
          mbar_wait(&full_bar[s], par, p.err, kErrDrain, false);
        }
      }
    }
    __syncwarp();
  } else if (warp >= kSfWarp0 && warp < kEpiWarp1) {
    // ---------------------------------------------------------- scale warps
    // Lane 32q + i, column c of a K step's four columns holds the scales of
    // rows i + 32c of the 128-row block.  A tile of TN < 128 tokens starts
    // at column (x0 % 128) / 32 of its block.
    const uint32_t q = static_cast<uint32_t>(warp % 4);
    const uint32_t t_lane = tmem + ((32u * q) << 16);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true, ready = false;
    griddep_wait();
    for (int tile = first; ok && tile < total; tile += step) {
      const int part =
          TN == 128 ? 0 : (locate<TN>(p, tab, tile).x0 % 128) / 32;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!__all_sync(0xffffffffu, ready)) {
          const bool got =
              mbar_wait(&sfdata_bar[stage], phase, p.err, kErrMma);
          if (!__all_sync(0xffffffffu, got)) {
            ok = false;
            break;
          }
        }
        const int next = stage + 1 == S ? 0 : stage + 1;
        const uint32_t next_phase = phase ^ (next == 0 ? 1u : 0u);
        ready = mbar_peek(&sfdata_bar[next], next_phase);
        // arm the stage's next fill: it cannot complete before all four
        // scale warps have passed this one
        if (warp == kSfWarp0 && lane == 0)
          mbar_arrive_expect_tx(&sfdata_bar[stage], 2 * run_bytes);
        const int skip =
            Cf::kSteps * kb -
            min(Cf::kSteps * kb, max(0, kblk64 - Cf::kSteps));
        const uint32_t sf_s = smem_u32(smem + stage * Cf::kStageBytes +
                                       Cf::kWBytes + Cf::kXBytes) +
                              16u * lane;
#pragma unroll
        for (int h = 0; h < Cf::kSub; ++h) {
          uint32_t r[32];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            // (past the run for the steps of a short block that are not
            // issued)
            const uint32_t at =
                sf_s + min(4 * h + j + skip, Cf::kSteps - 1) * kAtomBytes;
            const uint4 w = lds128(at);
            const uint4 x = lds128(at + Cf::kRun);
            r[4 * j + 0] = w.x;
            r[4 * j + 1] = w.y;
            r[4 * j + 2] = w.z;
            r[4 * j + 3] = w.w;
            if (TN == 128) {
              r[16 + 4 * j + 0] = x.x;
              r[16 + 4 * j + 1] = x.y;
            } else if (TN == 64) {
              r[16 + 4 * j + 0] = part ? x.z : x.x;
              r[16 + 4 * j + 1] = part ? x.w : x.y;
            } else {
              r[16 + 4 * j + 0] =
                  part < 2 ? (part ? x.y : x.x) : (part == 2 ? x.z : x.w);
              r[16 + 4 * j + 1] = x.y;
            }
            r[16 + 4 * j + 2] = x.z;
            r[16 + 4 * j + 3] = x.w;
          }
          __syncwarp();
          tc_st_32cols(t_lane + Cf::kSfBase + stage * Cf::kSfCols + 32 * h,
                       r);
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (warp == kSfWarp0)
            mbar_arrive_expect_tx(&full_bar[stage],
                                  Cf::kWBytes + Cf::kXBytes);
          else
            mbar_arrive(&full_bar[stage]);
        }
        stage = next;
        phase = next_phase;
      }
    }
  } else if (warp == kMmaWarp) {
    // ---------------------------------------------------------- MMA issuer
    if (lane == 0) {
      constexpr uint32_t kIdesc = idesc_nvf4(kFeat, TN);
      const uint64_t w_desc0 =
          smem_desc(smem_u32(smem), 16, 1024, SmemLayout::kSwizzle128B);
      const uint64_t x_desc0 = smem_desc(smem_u32(smem) + Cf::kWBytes, 16,
                                         1024, SmemLayout::kSwizzle128B);
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;
      bool ok = true, ready = false;
      griddep_wait();  // (the waits' limits count from here)
      for (int tile = first; ok && tile < total; tile += step, ++it) {
        const int a = it & 1;
        if (!mbar_wait(&acc_empty_bar[a], ((it >> 1) & 1) ^ 1u, p.err,
                       kErrMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + a * TN;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!ready &&
              !mbar_wait(&full_bar[stage], phase, p.err, kErrMma)) {
            ok = false;
            break;
          }
          const int next = stage + 1 == S ? 0 : stage + 1;
          const uint32_t next_phase = phase ^ (next == 0 ? 1u : 0u);
          ready = mbar_peek(&full_bar[next], next_phase);
          tc_fence_after();
          const uint32_t soff =
              static_cast<uint32_t>(stage) * (Cf::kStageBytes >> 4);
          const uint32_t sf_t = tmem + Cf::kSfBase + stage * Cf::kSfCols;
          const int steps = min(Cf::kSteps, kblk64 - Cf::kSteps * kb);
#pragma unroll
          for (int j = 0; j < Cf::kSteps; ++j)
            if (j < steps)
              tc_mma_nvf4(
                  d, w_desc0 + soff + (j / 4) * (Cf::kWBox >> 4) + 2u * (j % 4),
                  x_desc0 + soff + (j / 4) * (Cf::kXBox >> 4) + 2u * (j % 4),
                  kIdesc, sf_t + 32 * (j / 4) + 4 * (j % 4),
                  sf_t + 32 * (j / 4) + 16 + 4 * (j % 4),
                  (kb > kb0 || j > 0) ? 1u : 0u);
          tc_commit(&empty_bar[stage]);
          stage = next;
          phase = next_phase;
        }
        if (ok) tc_commit(&acc_full_bar[a]);
      }
      // no MMA may still be running when TMEM is released
      tc_commit(&drain_bar);
      mbar_wait(&drain_bar, 0, p.err, kErrDrain, /*bail_on_err=*/false);
    }
    __syncwarp();
  } else if (Cf::kRows && p.split == 1) {
    // ---------------------------------------------------------- epilogue
    // A thread is a token row; the groups take chunks of 32 features in turn.
    const int q = warp % 4, group = epi_group(warp);
    const int row = 32 * q + lane;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(q * 32) << 16);
    int it = 0;
    griddep_wait();
    for (int tile = first; tile < total; tile += step, ++it) {
      const Tile t = locate<TN>(p, tab, tile);
      const int a = it & 1;
      const int x = t.x0 + row;
      const bool live = row < t.rows;
      const float scale =
          p.row_scale != nullptr && live ? p.row_scale[x] : 0.f;
      bias_sh[group][a][row] = load_bias<T>(p, t.g, t.n0 + row);
      const bool got =
          mbar_wait(&acc_full_bar[a], (it >> 1) & 1, p.err, kErrEpilogue);
      if (!epi_all(group, got)) break;  // (and the bias is visible)
      tc_fence_after();
#pragma unroll 1
      for (int c = group; c < 4; c += 2) {
        const int n = t.n0 + 32 * c;
        if (n >= p.N) break;
        float v[32];
        uint4 r[4];
        load_residual_row<T>(p, x, n, live, r);
        __syncwarp();
        tc_ld_32cols(t_row + a * TN + 32 * c, v);
        tc_wait_ld();
        tie32(v);
        finish_row32<T>(
            p, scale, &bias_sh[group][a][32 * c], v,
            [&](int i) { return r[i]; },
            [&](int i, const uint4& o) {
              if (live && n + 8 * i < p.N) store_row8<T>(p, x, n + 8 * i, o);
            });
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty_bar[a]);
    }
  } else if (p.split == 1) {
    // ---------------------------------------------------------- epilogue
    const int q = warp % 4, group = epi_group(warp);
    const uint32_t t_row = tmem + (static_cast<uint32_t>(q * 32) << 16);
    int it = 0;
    griddep_wait();
    for (int tile = first; tile < total; tile += step, ++it) {
      const Tile t = locate<TN>(p, tab, tile);
      const int a = it & 1;
      const int n = t.n0 + 32 * q + lane;
      const float bias = load_bias<T>(p, t.g, n);
      const int cols = min(t.rows, TN);
      const int rows = n < p.N ? cols : 0;
      // (with the bias, before the wait: their latency passes meanwhile)
      const float scale0 =
          load_scale(p, t.x0 + 32 * group, cols - 32 * group, lane);
      const bool got =
          mbar_wait(&acc_full_bar[a], (it >> 1) & 1, p.err, kErrEpilogue);
      if (!__all_sync(0xffffffffu, got)) break;
      tc_fence_after();
      // the groups take chunks of 32 columns in turn
#pragma unroll 1
      for (int c = group; 32 * c < cols; c += 2) {
        T r[32];
        float v[32];
        load_residual<T, 32>(p, t.x0 + 32 * c, n, rows - 32 * c, r);
        const float scale =
            c == group ? scale0
                       : load_scale(p, t.x0 + 32 * c, cols - 32 * c, lane);
        __syncwarp();
        tc_ld_32cols(t_row + a * TN + 32 * c, v);
        tc_wait_ld();
        tie32(v);
        finish<T, 32>(p, t.x0 + 32 * c, n, cols - 32 * c, rows - 32 * c, bias,
                      scale, r, v);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty_bar[a]);
    }
  } else {
    // ---------------------------------------------------------- split-K
    // Pieces of four token columns; rank d finishes pieces
    // [d * gpr, (d + 1) * gpr).  In the receive buffer, source s, own piece
    // j, row r sit at ((s * gpr + j) * 128 + r) * 16.
    const int q4 = warp % 4, group = epi_group(warp);
    const uint32_t t_row = tmem + (static_cast<uint32_t>(q4 * 32) << 16);
    const int row = 32 * q4 + lane;
    const Tile t = locate<TN>(p, tab, first);
    // columns of the accumulator that are wanted: tokens, or features
    const int nv = Cf::kRows ? min(p.N - t.n0, TN) : min(t.rows, TN);
    const int g4 = (nv + 3) / 4;
    // (kRows: pieces in pairs, 16 bytes of a row)
    const int gpr = Cf::kRows ? (g4 / 2 + p.split - 1) / p.split * 2
                              : (g4 + p.split - 1) / p.split;
    const int g_own = rank * gpr;
    const int n_own = max(0, min(gpr, g4 - g_own));
    const uint32_t recv = smem_u32(smem + S * Cf::kStageBytes);
    if (threadIdx.x == 0 && n_own > 0)
      mbar_arrive_expect_tx(&recv_bar, (p.split - 1) * n_own * 2048);
    griddep_wait();
    const int n = t.n0 + row;
    const float bias = load_bias<T>(p, t.g, n);
    if (Cf::kRows) {
      // (32 more: a chunk of 32 columns may reach past the rank's share)
      bias_sh[group][0][row] = bias;
      if (row < 32) bias_sh[group][0][128 + row] = 0.f;
      epi_bar(group);
    }
    const bool got = mbar_wait(&acc_full_bar[0], 0, p.err, kErrEpilogue);
    if (__all_sync(0xffffffffu, got)) {
      tc_fence_after();
#pragma unroll 1
      for (int c = group; 8 * c < g4; c += 2) {
        float v[32];
        __syncwarp();
        tc_ld_32cols(t_row + 32 * c, v);
        tc_wait_ld();
        tie32(v);
        int d = 8 * c / gpr;       // rank of the piece
        int j = 8 * c - d * gpr;   // its number there
        uint32_t dst = mapa_shared(recv, d);
        uint32_t bar = mapa_shared(smem_u32(&recv_bar), d);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (8 * c + q < g4) {
            if (d != rank) {
              const float f[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2],
                                  v[4 * q + 3]};
              st_async_v4(dst + ((rank * gpr + j) * 128u + row) * 16u, f,
                          bar);
            }
            if (++j == gpr && 8 * c + q + 1 < g4) {
              j = 0;
              ++d;
              dst = mapa_shared(recv, d);
              bar = mapa_shared(smem_u32(&recv_bar), d);
            }
          }
        }
      }
      // this rank's share: 32 columns at a time where it holds more than two
      // pieces (one TMEM round trip and one set of residual loads for eight),
      // else piece by piece; the groups of warps take them in turn.  Partials
      // are added in rank order after the rank's own.
      auto share = [&](auto width) {
        constexpr int kG = decltype(width)::value;
        bool landed = false;
#pragma unroll 1
        for (int o = group * kG; o < n_own; o += 2 * kG) {
          const int col = 4 * (g_own + o);
          const int cnt = min(nv - col, 4 * min(kG, n_own - o));
          [[maybe_unused]] const int rows = n < p.N ? cnt : 0;
          [[maybe_unused]] const int x = t.x0 + row;  // (kRows)
          [[maybe_unused]] const bool live = row < t.rows;
          [[maybe_unused]] T r[Cf::kRows ? 1 : 4 * kG];
          [[maybe_unused]] uint4 rr[4];
          float v[4 * kG], scale;
          if constexpr (Cf::kRows) {
            load_residual_row<T>(p, x, t.n0 + col, live, rr);
            scale = p.row_scale != nullptr && live ? p.row_scale[x] : 0.f;
          } else {
            load_residual<T, 4 * kG>(p, t.x0 + col, n, rows, r);
            scale = load_scale(p, t.x0 + col, cnt, lane);
          }
          __syncwarp();
          if constexpr (kG == 8) {
            tc_ld_32cols(t_row + col, v);
            tc_wait_ld();
            tie32(v);
          } else {
            tc_ld_4cols(t_row + col, v);
            tc_wait_ld();
          }
          if (!landed) {
            const bool in = mbar_wait(&recv_bar, 0, p.err, kErrEpilogue);
            if (!__all_sync(0xffffffffu, in)) break;
            landed = true;
          }
          for (int s = 0; s < p.split; ++s) {
            if (s == rank) continue;
#pragma unroll
            for (int q = 0; q < kG; ++q) {
              if (o + q < n_own) {
                const uint4 u =
                    lds128(recv + ((s * gpr + o + q) * 128u + row) * 16u);
                v[4 * q + 0] += __uint_as_float(u.x);
                v[4 * q + 1] += __uint_as_float(u.y);
                v[4 * q + 2] += __uint_as_float(u.z);
                v[4 * q + 3] += __uint_as_float(u.w);
              }
            }
          }
          if constexpr (Cf::kRows) {
            finish_row32<T>(
                p, scale, &bias_sh[group][0][col], v,
                [&](int i) { return rr[i]; },
                [&](int i, const uint4& out) {
                  if (live && 8 * i < cnt)
                    store_row8<T>(p, x, t.n0 + col + 8 * i, out);
                });
          } else {
            finish<T, 4 * kG>(p, t.x0 + col, n, cnt, rows, bias, scale, r,
                              v);
          }
        }
      };
      if constexpr (Cf::kRows) {
        share(std::integral_constant<int, 8>());
      } else {
        if (n_own > 2)
          share(std::integral_constant<int, 8>());
        else
          share(std::integral_constant<int, 1>());
      }
    }
  }

  // ------------------------------------------------------------ teardown
  tc_fence_before();
  __syncthreads();
  if (p.split > 1) cluster_sync_final();
  if (warp == kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// linear_pair_kernel: many tokens.  A cluster of two CTAs computes 256 tokens
// x 256 features with 2-SM MMAs: CTA r holds token rows [128r, 128r + 128)
// and weight rows [128r, 128r + 128) of the tile, so an SM streams 38 KiB of
// operands per K block for the MMAs of 54 KiB in a tile of its own, and
// receives its 128 token rows of the accumulator.  The even CTA issues; both
// CTAs' tiles land on its `full` barriers.  A thread of the epilogue is a
// token row; outputs leave through shared memory and TMA stores, 64 columns
// at a time.
//
// Up to K of ~2500 bound by a tile's epilogue, 9,000 cycles at K 512 and
// 10,300 at K 2048 by stamps in steady state: ~1,400 from a tile's last store
// until the next accumulator is seen full (the tile's place, its bias, the
// wait), ~450 for the columns to registers, the rest for four chunks of 32
// columns; the products of the next tile start ~1,200 cycles after the
// accumulator was full and are done before its epilogue begins.  A residual,
// read by 16-byte loads of 32 rows a warp, adds ~6,000 to the chunks.  592
// tiles, 8 a pair, take 42.6 us for K of 64, 44.8 for 512, 53.4 for 2048; with
// a residual 71, 72 and 82.
// For longer K bound by a K block's ~740 cycles, where its MMAs take 512, and
// ~2,400 a tile between its last product and the next one's first (118 us for
// K of 7168).  Not by the ring's latency: 72 tiles, one a pair, take 424 ns a
// block with five stages, 445 with four, 550 with three, where latency alone
// would give 530 and 707.  Not by the copies either, if the dual GEMM's pair
// loop is a guide, whose block of the same size takes as long with its tile
// copies left out.  The cause is open.
// In a long loop by power.  (In turns with short pauses: 8192 x 8192 x 28672
// 746 us, 5.2 PFLOP/s; 4096 x 4096 x 14336 with a residual 112 us, 4.3.)
// There is one accumulator: its 256 columns go to registers at once and the
// next tile's products start under the epilogue (126 -> 115 us and 781 -> 768
// us for the two when that was brought in, 122 -> 114 us for 32 experts of
// 16384 rows and K 2048; a tile whose rows are stored one by one is slower, 37
// -> 39 us for 16 experts of ~94 rows, which the schedule gives smaller
// tiles).  That needs 192 registers in the epilogue's threads and hence the
// warpgroups' shares; a spilled register costs more than elsewhere, as shared
// memory leaves next to no L1.  Tried and slower: sixteen epilogue warps with
// half the columns each, outputs stored without boxes, the columns in four
// rounds through 64 registers (122 -> 139 us), and scales copied ahead of
// their stage (two waits in the scale warps: no gain).
// ---------------------------------------------------------------------------
constexpr int kPairThreads = 512;
// Whole warpgroups, whose shares of the launch's registers follow their work:
// epilogue group 0 (warps 0-3), producers, MMA issuer and waiter (4-7), scale
// warps (8-11), epilogue group 1 (12-15).
constexpr int kPairSfWarp0 = 8;
constexpr int kPairEpiWarp1 = 12;
constexpr int kPairRegs = 65536 / kPairThreads;  // a thread's at launch
constexpr int kPairEpiRegs = 192, kPairIssueRegs = 56, kPairSfRegs = 72;
static_assert(2 * kPairEpiRegs + kPairIssueRegs + kPairSfRegs <= 4 * kPairRegs,
              "an increase beyond the launch's registers would never end");
constexpr int kPairStages = 5;
constexpr int kPairTile = 128 * kRowBytes;  // one CTA's token or weight rows
constexpr int kPairStageBytes = 2 * kPairTile + 3 * kRunBytes;
constexpr int kPairSfBase = 256;   // TMEM: accumulator, then the scales
constexpr int kPairSfCols = 48;    // 16 of tokens, 32 of weights per stage
constexpr int kBoxBytes = 128 * 128;  // 128 rows x 64 columns of C
constexpr int kPairSmem = kPairStages * kPairStageBytes + 2 * kBoxBytes + 1024;
constexpr int kBand = 8;  // m tiles of a band, see locate_pair
static_assert(kPairSmem + 4096 <= 227 * 1024, "shared memory");
static_assert(kPairSfBase + kPairStages * kPairSfCols <= kTmemCols, "TMEM");

struct PairTile {
  int g, n0, x0, rows;  // as Tile, x0 the first of 256 token rows
  int sfa_last;         // last row block of the scales that may be read
};

// Tiles of one problem run in bands of eight m tiles, m fastest: the tiles in
// flight then form a block of about 8 x 9 tiles, which reads fewer distinct
// operand rows than whole columns of m tiles do.
__device__ __forceinline__ PairTile locate_pair(const LinearParams& p,
                                                const GroupTable& tab,
                                                int tile) {
  PairTile t;
  if (p.groups == 0) {
    const int per = kBand * p.n_tiles;
    const int band = tile / per;
    const int in = tile - band * per;
    const int width = min(kBand, p.m_tiles - band * kBand);
    const int nt = in / width;
    t.g = 0;
    t.n0 = nt * 256;
    t.x0 = (band * kBand + in - nt * width) * 256;
    t.rows = p.M - t.x0;
    t.sfa_last = (p.M - 1) / 128;
    return t;
  }
  const int g = find_group(p, tab, tile);
  const int local = tile - tab.tile0[g];
  const int row0 = tab.row0[g];
  const int rows = group_rows(p, g, row0);
  const int mt = (rows + 255) / 256;
  const int nt = mt == 1 ? local : local / mt;
  const int m0 = (local - nt * mt) * 256;
  t.g = g;
  t.n0 = nt * 256;
  t.x0 = row0 + m0;
  t.rows = rows - m0;
  t.sfa_last = (row0 + rows - 1) / 128;
  return t;
}

template <typename T>
__global__ void __launch_bounds__(kPairThreads, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap tmW,
                       const __grid_constant__ CUtensorMap tmX,
                       const __grid_constant__ CUtensorMap tmC,
                       const __grid_constant__ LinearParams p) {
  constexpr int S = kPairStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[S];
  __shared__ __align__(8) uint64_t sfdata_bar[S];
  __shared__ __align__(8) uint64_t empty_bar[S];
  __shared__ __align__(8) uint64_t acc_full_bar;
  __shared__ __align__(8) uint64_t acc_empty_bar;
  __shared__ __align__(8) uint64_t drain_bar;
  __shared__ uint32_t tmem_base_sh;
  __shared__ uint32_t landed_sh;  // K blocks ready for the MMA thread
  __shared__ __align__(16) float bias_sh[256];
  __shared__ GroupTable tab;

  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank();  // 0: issues the MMAs
  const bool leader = rank == 0;
  const int kblk64 = p.K / 64;
  // A K block's scale run has the same size for every block: the last
  // block's, when K % 256 != 0, starts earlier and its first atoms are
  // skipped (`skip` in the scale warps).
  const uint32_t run_bytes =
      static_cast<uint32_t>(min(4, kblk64)) * kAtomBytes;

  if (warp == 0) {
    uint64_t* bar = nullptr;
    uint32_t count = 1;
    if (lane < S) {
      bar = full_bar + lane;
      count = 2 * kSfWarps;
    } else if (lane < 2 * S) {
      bar = sfdata_bar + (lane - S);
    } else if (lane < 3 * S) {
      bar = empty_bar + (lane - 2 * S);
    } else if (lane == 3 * S) {
      bar = &acc_full_bar;
    } else if (lane == 3 * S + 1) {
      bar = &acc_empty_bar;
      count = 2 * kEpiWarps;
    } else if (lane == 3 * S + 2) {
      bar = &drain_bar;
    }
    if (bar != nullptr) {
      mbar_init(bar, count);
      fence_mbar_init();
    }
    if (lane == 0) {
      s_wait_failed = 0u;
      landed_sh = 0u;
    }
    if (lane == 29) prefetch_tmap(&tmW);
    if (lane == 30) prefetch_tmap(&tmX);
    if (lane == 31) prefetch_tmap(&tmC);
    __syncwarp();
    if (lane < S) mbar_arrive_expect_tx(sfdata_bar + lane, 3 * run_bytes);
    fence_proxy_async_smem();
    __syncwarp();
  }
  if (warp == kMmaWarp) {
    tmem_alloc_pair(&tmem_base_sh, kTmemCols);
    tmem_relinquish_pair();
  }
  cluster_arrive_relaxed();
  griddep_launch_dependents();
  if (p.groups > 0 && warp == 1) {
    if (p.dev_rows != nullptr) griddep_wait();
    build_groups(p, 256, lane, tab);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  cluster_wait();  // both CTAs' barriers are initialised
  const uint32_t tmem = tmem_base_sh;
  const int total =
      p.groups > 0 ? tab.tile0[p.groups] : p.n_tiles * p.m_tiles;
  const int first = static_cast<int>(blockIdx.x) / 2;
  const int step = static_cast<int>(gridDim.x) / 2;

  if (warp >= kProdWWarp && warp < kPairSfWarp0) {
    reg_dec<kPairIssueRegs>();
    if (warp == kProdWWarp || warp == kProdXWarp) {
      // ---------------------------------------------------------- producers
      // Warp 4: token scales, the first run of weight scales, token rows; warp
      // 5: the second run, weight rows.  They only copy: the expected bytes
      // come with the scale warps' arrivals.
      {
        const bool x_side = warp == kProdWWarp;
        const uint64_t pol = x_side ? kPolicyEvictLast : kPolicyEvictNormal;
        const uint32_t full_c = mapa_shared(smem_u32(&full_bar[0]), 0);
        int stage = 0;
        uint32_t phase = 0;
        long long issued = 0;
        bool ok = true;
        griddep_wait();  // global memory only after the previous grid
        for (int tile = first; ok && tile < total; tile += step) {
          const PairTile t = locate_pair(p, tab, tile);
          const int row = (x_side ? t.x0 : t.n0) + 128 * static_cast<int>(rank);
          // the odd CTA's rows may lie past the problem's last row block, and
          // the second weight run past the last one: they copy the last, whose
          // products are never stored
          const uint8_t* sfa =
              p.sfa + (size_t)min(t.x0 / 128 + static_cast<int>(rank),
                                  t.sfa_last) *
                          kblk64 * kAtomBytes;
          const int nb = t.n0 / 128 + (x_side ? 0 : 1);
          const uint8_t* sfb = p.sfb + (size_t)t.g * p.sfb_group +
                               (size_t)min(nb, (p.N - 1) / 128) * kblk64 *
                                   kAtomBytes;
          for (int kb = 0; lane == 0 && kb < p.kblocks; ++kb) {
            if (issued >= S &&
                !mbar_wait_cluster(&empty_bar[stage], phase ^ 1u, p.err,
                                   kErrProducer)) {
              ok = false;
              break;
            }
            const int next = stage + 1 == S ? 0 : stage + 1;
            const uint32_t next_phase = phase ^ (next == 0 ? 1u : 0u);
            uint8_t* st = smem + stage * kPairStageBytes;
            uint8_t* sf = st + 2 * kPairTile;
            const size_t run =
                (size_t)min(4 * kb, max(0, kblk64 - 4)) * kAtomBytes;
            const uint32_t full_s = full_c + 8u * static_cast<uint32_t>(stage);
            if (x_side) {
              bulk_load(sf, sfa + run, run_bytes, &sfdata_bar[stage], pol);
              bulk_load(sf + kRunBytes, sfb + run, run_bytes,
                        &sfdata_bar[stage], pol);
              tma_load_3d_pair(st, &tmX, full_s, kb * kRowBytes, row, 0, pol);
            } else {
              bulk_load(sf + 2 * kRunBytes, sfb + run, run_bytes,
                        &sfdata_bar[stage], pol);
              tma_load_3d_pair(st + kPairTile, &tmW, full_s, kb * kRowBytes,
                               row, t.g, pol);
            }
            ++issued;
            stage = next;
            phase = next_phase;
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
        }
        const bool ok_all = ok;
        // never leave with copies in flight: scale runs land on this CTA's
        // barriers, both CTAs' tiles on the even one's
        for (int s = 0; s < S; ++s) {
          if (issued > s) {
            const uint32_t par =
                static_cast<uint32_t>(((issued - 1 - s) / S) & 1);
            mbar_wait(&sfdata_bar[s], par, p.err, kErrDrain, false);
            if (x_side && leader)
              mbar_wait_cluster(&full_bar[s], par, p.err, kErrDrain, false);
            // the stage's last commit, which the even CTA sends to both: none
            // may be on its way when a CTA leaves
            if (ok_all)
              mbar_wait_cluster(&empty_bar[s], par, p.err, kErrDrain, false);
          }
        }
      }
      __syncwarp();
    } else if (warp == kMmaWarp) {
      // ---------------------------------------------------------- MMA issuer
      if (lane == 0 && leader) {
        constexpr uint32_t kIdesc = idesc_nvf4(256, 256);
        const uint64_t x_desc0 =
            smem_desc(smem_u32(smem), 16, 1024, SmemLayout::kSwizzle128B);
        const uint64_t w_desc0 = smem_desc(smem_u32(smem) + kPairTile, 16, 1024,
                                           SmemLayout::kSwizzle128B);
        int stage = 0;
        uint32_t acc_phase = 0, block = 0;
        bool ok = true, any = false;
        griddep_wait();  // (the waits' limits count from here)
        for (int tile = first; ok && tile < total; tile += step) {
          if (!mbar_wait_cluster(&acc_empty_bar, acc_phase ^ 1u, p.err,
                                 kErrMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          for (int kb = 0; kb < p.kblocks; ++kb) {
            if (!flag_wait(&landed_sh, ++block, p.err, kErrMma)) {
              ok = false;
              break;
            }
            const int next = stage + 1 == S ? 0 : stage + 1;
            tc_fence_after();
            const uint32_t soff =
                static_cast<uint32_t>(stage) * (kPairStageBytes >> 4);
            const uint32_t sf_t = tmem + kPairSfBase + stage * kPairSfCols;
            const uint32_t acc0 = kb > 0 ? 1u : 0u;
            if (4 * kb + 4 <= kblk64) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                tc_mma_nvf4_pair(tmem, x_desc0 + soff + 2u * j,
                                 w_desc0 + soff + 2u * j, kIdesc, sf_t + 4 * j,
                                 sf_t + 16 + 8 * j, j > 0 ? 1u : acc0);
            } else {
              for (int j = 0; j < kblk64 - 4 * kb; ++j)
                tc_mma_nvf4_pair(tmem, x_desc0 + soff + 2u * j,
                                 w_desc0 + soff + 2u * j, kIdesc, sf_t + 4 * j,
                                 sf_t + 16 + 8 * j, j > 0 ? 1u : acc0);
            }
            tc_commit_both(&empty_bar[stage]);
            any = true;
            stage = next;
          }
          if (!ok) break;
          tc_commit_both(&acc_full_bar);
          acc_phase ^= 1u;
        }
        // the last release of the accumulator (the odd CTA's warps arrive here
        // remotely) is awaited like the others, so that no arrival is in
        // flight when the CTAs leave
        if (ok && any)
          mbar_wait_cluster(&acc_empty_bar, acc_phase ^ 1u, p.err, kErrMma);
        tc_commit_pair(mapa_shared(smem_u32(&drain_bar), 0));
        mbar_wait(&drain_bar, 0, p.err, kErrDrain, /*bail_on_err=*/false);
      }
      __syncwarp();
    } else {
      // ---------------------------------------------------------- waiter
      // Waits for each K block's barrier in the MMA thread's stead and counts
      // the blocks in shared memory, where that thread reads the count in a few
      // cycles: its own wait would keep the tensor cores idle for ~300 cycles a
      // block of 512.
      if (lane == 0 && leader) {
        int stage = 0;
        uint32_t phase = 0, block = 0;
        bool ok = true;
        griddep_wait();
        for (int tile = first; ok && tile < total; tile += step) {
          for (int kb = 0; kb < p.kblocks; ++kb) {
            if (!mbar_wait_cluster(&full_bar[stage], phase, p.err, kErrMma)) {
              ok = false;
              break;
            }
            flag_set(&landed_sh, ++block);
            if (++stage == S) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
      }
      __syncwarp();
    }
  } else if (warp >= kPairSfWarp0 && warp < kPairEpiWarp1) {
    reg_dec<kPairSfRegs>();
    // ---------------------------------------------------------- scale warps
    const uint32_t q = static_cast<uint32_t>(warp % 4);
    const uint32_t t_lane = tmem + ((32u * q) << 16);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    griddep_wait();
    for (int tile = first; ok && tile < total; tile += step) {
      for (int kb = 0; kb < p.kblocks; ++kb) {
        const bool got = mbar_wait(&sfdata_bar[stage], phase, p.err, kErrMma);
        if (!__all_sync(0xffffffffu, got)) {
          ok = false;
          break;
        }
        const int next = stage + 1 == S ? 0 : stage + 1;
        const uint32_t next_phase = phase ^ (next == 0 ? 1u : 0u);
        // arm the stage's next fill: it cannot complete before all four
        // scale warps have passed this one
        if (warp == kPairSfWarp0 && lane == 0)
          mbar_arrive_expect_tx(&sfdata_bar[stage], 3 * run_bytes);
        const int skip = 4 * kb - min(4 * kb, max(0, kblk64 - 4));
        const uint32_t sf_s =
            smem_u32(smem + stage * kPairStageBytes + 2 * kPairTile) +
            16u * lane;
        const uint32_t col = t_lane + kPairSfBase + stage * kPairSfCols;
        uint32_t ra[16], rb[32];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // (past the run for the steps of a short block that are not issued)
          const uint32_t at = sf_s + min(j + skip, 3) * kAtomBytes;
          const uint4 v = lds128(at);
          const uint4 w0 = lds128(at + kRunBytes);
          const uint4 w1 = lds128(at + 2 * kRunBytes);
          ra[4 * j + 0] = v.x;
          ra[4 * j + 1] = v.y;
          ra[4 * j + 2] = v.z;
          ra[4 * j + 3] = v.w;
          rb[8 * j + 0] = w0.x;
          rb[8 * j + 1] = w0.y;
          rb[8 * j + 2] = w0.z;
          rb[8 * j + 3] = w0.w;
          rb[8 * j + 4] = w1.x;
          rb[8 * j + 5] = w1.y;
          rb[8 * j + 6] = w1.z;
          rb[8 * j + 7] = w1.w;
        }
        __syncwarp();
        tc_st_16cols(col, ra);
        tc_st_32cols(col + 16, rb);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          const uint32_t full_s = mapa_shared(smem_u32(&full_bar[stage]), 0);
          if (leader && warp == kPairSfWarp0)
            mbar_arrive_expect_tx_cluster(full_s, 4 * kPairTile);
          else
            mbar_arrive_cluster(full_s);
        }
        stage = next;
        phase = next_phase;
      }
    }
  } else {
    reg_inc<kPairEpiRegs>();
    // ---------------------------------------------------------- epilogue
    // Each group of four warps finishes 128 of the tile's columns, 32 at a
    // time, and stores them 64 at a time through a box of its own.
    const int q4 = warp % 4, group = warp >= kPairEpiWarp1 ? 1 : 0;
    const int row = 32 * q4 + lane;
    const bool stores = row == 0;  // the thread that stores the group's box
    const uint32_t t_row = tmem + (static_cast<uint32_t>(q4 * 32) << 16);
    const uint32_t acc_empty_c = mapa_shared(smem_u32(&acc_empty_bar), 0);
    uint8_t* box = smem + S * kPairStageBytes + group * kBoxBytes;
    float* bias = bias_sh + 128 * group;
    uint32_t acc_phase = 0;
    griddep_wait();
    for (int tile = first; tile < total; tile += step, acc_phase ^= 1u) {
      const PairTile t = locate_pair(p, tab, tile);
      const int rows = t.rows - 128 * static_cast<int>(rank);  // of this CTA
      const int x = t.x0 + 128 * static_cast<int>(rank) + row;
      const bool live = row < rows;
      const float scale =
          p.row_scale != nullptr && live ? p.row_scale[x] : 0.f;
      const int n0 = t.n0 + 128 * group;
      epi_bar(group);  // the previous tile's bias has been read
      bias[row] = load_bias<T>(p, t.g, n0 + row);
      if (p.residual != nullptr && live) {
        // the row's 256 bytes, to L2 while the products run
        const T* r =
            static_cast<const T*>(p.residual) + (size_t)x * p.ldr + n0;
        for (int i = 0; i < 128 && n0 + i < p.N; i += 64) prefetch_l2(r + i);
      }
      const bool got =
          mbar_wait_cluster(&acc_full_bar, acc_phase, p.err, kErrEpilogue);
      // the four warps leave together: they meet at the barriers below
      if (!epi_all(group, got)) break;
      tc_fence_after();
      // the group's 128 columns at once, so that the accumulator is free for
      // the next tile after one round trip
      float v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        tc_ld_32cols(t_row + 128 * group + 32 * c, v[c]);
      tc_wait_ld();
#pragma unroll
      for (int c = 0; c < 4; ++c) tie32(v[c]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc_empty_c);
      // a group's last rows are stored row by row: a box would overwrite the
      // rows behind them
      const bool boxed = p.groups == 0 ? rows > 0 : rows >= 128;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        const int n = n0 + 32 * c, half = c & 1;
        if (n >= p.N) break;
        uint4 res[2];
        if (boxed && half == 0) {
          // the store before has read the box
          if (stores) bulk_wait_group_read0();
          epi_bar(group);
        }
        finish_row32<T>(
            p, scale, bias + 32 * c, v[0], [&](int i) {
              // two at a time: four would not fit the registers
              if ((i & 1) == 0) {
                const T* r = static_cast<const T*>(p.residual) +
                             (size_t)x * p.ldr + n + 8 * i;
                res[0] = res[1] = make_uint4(0u, 0u, 0u, 0u);
                if (live && n + 8 * i < p.N)
                  res[0] = *reinterpret_cast<const uint4*>(r);
                if (live && n + 8 * i + 8 < p.N)
                  res[1] = *reinterpret_cast<const uint4*>(r + 8);
              }
              return res[i & 1];
            },
            [&](int i, const uint4& o) {
              if (boxed)
                sts128(smem_u32(box + row * 128 +
                                (((4 * half + i) ^ (row & 7)) << 4)),
                       o);
              else if (live && n + 8 * i < p.N)
                store_row8<T>(p, x, n + 8 * i, o);
            });
        if (boxed && (half == 1 || n + 32 >= p.N)) {
          fence_proxy_async_smem();
          epi_bar(group);
          if (stores) {
            tma_store_2d(&tmC, box, 2 * (n - 32 * half),
                         t.x0 + 128 * static_cast<int>(rank));
            bulk_commit_group();
          }
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) {  // the next chunk into v[0]
          v[0][i] = v[1][i];
          v[1][i] = v[2][i];
          v[2][i] = v[3][i];
        }
      }
    }
    // the stores must have read their boxes before shared memory goes away
    if (stores) bulk_wait_group_read0();
    __syncwarp();
  }

  // ------------------------------------------------------------ teardown
  tc_fence_before();
  cluster_sync_final();  // no CTA leaves while its peer may still signal it
  if (warp == kMmaWarp) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem, kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct LinearPlan {
  int tn;      // tokens per tile (256: 2-SM pairs)
  int split;   // CTAs that share a tile's K range
  int grid;    // CTAs
  int tiles;
  int kblocks;  // K blocks of a tile
};

// What a launch takes, in microseconds, fitted to B200 timings of 1 to 4000
// tokens (N 512 to 8192, K 512 to 14336, graph-replayed, L2 warm, single
// problems): a start and end, the first wave of tiles, and every further one,
// which is bound by its products or by its epilogue.  `kb`: the 256-wide K
// blocks of a CTA; `tokens`: 0 for groups, whose tiles say it all and which the
// constants were not fitted to.  (500 x 8192 x 512: 8.2 us with 128 tokens,
// 10.2 with pairs; x 7168: 27.0 and 20.1.)
double linear_cost(int tn, double kb, double waves, bool split, int tokens,
                   bool residual) {
  if (tn == 32) {
    const double wave = 0.20 * kb + 0.1;
    return 3.5 + 0.03 * (tokens ? std::min(tokens, 32) : 32) +
           (tokens > 64 ? 0.9 : 0.0) + (split ? 0.25 : 0.0) + wave +
           (waves - 1) * std::max(wave, 1.5);
  }
  if (tn == 64) {
    const double wave = 0.24 * kb + 0.3;
    return 5.0 + (split ? 0.7 : 0.0) + wave +
           (waves - 1) * std::max(wave, 2.6);
  }
  if (tn == 128) {
    const double wave = 0.40 * kb + 0.5;
    return 5.0 + (split ? 0.2 : 0.0) + wave +
           (waves - 1) * (residual ? std::max(wave + 0.9, 4.0)
                                   : std::max(wave, 2.4));
  }
  return (residual ? 10.8 : 8.4) + 0.39 * kb +
         (waves - 1) * (residual ? std::max(0.42 * kb + 2.5, 9.0)
                                 : std::max(0.42 * kb + 1.0, 5.0));
}

// `mts`: token tiles of 32, 64, 128 and 256 tokens (of all groups); `tokens`:
// of all of them; `pairs`: whether pair tiles may be taken.
LinearPlan plan_linear(const long long (&mts)[4], long long tokens, int N,
                       int K, int groups, bool residual, unsigned flags,
                       int sms, bool pairs) {
  const unsigned forced_tile =
      flags & (NVFP4DG_LINEAR_TOKENS32 | NVFP4DG_LINEAR_TOKENS64 |
               NVFP4DG_LINEAR_TOKENS128 | NVFP4DG_LINEAR_PAIR);
  const int forced_split =
      static_cast<int>((flags & NVFP4DG_LINEAR_SPLIT_MASK) >> 8);
  const int kb256 = (K + 255) / 256;
  LinearPlan best{};
  double best_cost = 1e300;
  for (int i = 0; i < 4; ++i) {
    if (forced_tile && !(forced_tile & (1u << i))) continue;
    const int tn = 32 << i;
    const int ctas = tn == 256 ? 2 : 1;
    if (tn == 256 && (sms < 2 || !pairs)) continue;
    LinearPlan pl{};
    pl.tn = tn;
    pl.kblocks = tn <= 64 ? (K + 511) / 512 : kb256;
    const long long n_tiles =
        tn == 256 ? (N + 255) / 256 : (N + kFeat - 1) / kFeat;
    pl.tiles = static_cast<int>(std::min<long long>(mts[i] * n_tiles,
                                                    1 << 30));
    for (int lg = 0; lg < 4; ++lg) {
      const int s = 1 << lg;
      // the CTAs of a cluster share a tile's K range: one problem only, a
      // block for each, and all clusters at once (a cluster lies in one
      // group of SMs, which leaves some of them over)
      const int room = s == 2 ? sms / 2 - 2 : s == 4 ? sms / 4 - 3
                                            : sms / 8 - 4;
      if (s > 1 && (groups > 0 || tn == 256 || s > pl.kblocks)) break;
      if (forced_split && groups == 0 && tn < 256) {
        const bool last = 2 * s > pl.kblocks || lg == 3;
        if (lg + 1 != forced_split && !(last && lg + 1 < forced_split))
          continue;
      } else if (s > 1 && pl.tiles > room) {
        break;
      }
      pl.split = s;
      const long long units = sms / ctas;
      const double waves =
          s > 1 ? 1.0
                : static_cast<double>((pl.tiles + units - 1) / units);
      const double cost =
          linear_cost(tn, static_cast<double>(kb256) / s, waves, s > 1,
                      groups ? 0 : static_cast<int>(tokens),
                      residual);
      if (cost < best_cost) {
        best_cost = cost;
        best = pl;
        best.grid = s > 1 ? pl.tiles * s
                          : ctas * static_cast<int>(
                                       std::min<long long>(pl.tiles, units));
      }
    }
  }
  return best;
}

template <typename T, int TN>
int launch_linear(const LinearParams& kp, const LinearPlan& pl,
                  const CUtensorMap& tw, const CUtensorMap& tx, int dev,
                  unsigned flags, cudaStream_t stream) {
  static std::atomic<unsigned long long> ready{0};
  auto kernel = linear_kernel<T, TN>;
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(ready.load() & bit)) {
    const int most = std::max(Cfg<TN>::smem(1), Cfg<TN>::smem(2));
    cudaError_t e = cudaFuncSetAttribute(
        kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute");
    ready.fetch_or(bit);
  }
  LinearParams p = kp;
  p.stages = Cfg<TN>::stages(pl.split);
  p.m_tiles = (p.M + TN - 1) / TN;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(pl.grid, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg<TN>::smem(pl.split);
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  unsigned na = 0;
  if (!(flags & NVFP4DG_FLAG_NO_PDL)) {
    attrs[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[na].val.programmaticStreamSerializationAllowed = 1;
    ++na;
  }
  if (pl.split > 1) {
    attrs[na].id = cudaLaunchAttributeClusterDimension;
    attrs[na].val.clusterDim.x = pl.split;
    attrs[na].val.clusterDim.y = 1;
    attrs[na].val.clusterDim.z = 1;
    ++na;
  }
  cfg.attrs = attrs;
  cfg.numAttrs = na;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tw, tx, p);
  if (e != cudaSuccess) return host_cuda_fail(e, "linear_kernel launch");
  return NVFP4DG_OK;
}

// Whether linear_pair_kernel can be launched: its warpgroups' shares of the
// registers come out of what the launch allocates, and only a build with
// exactly that many lets every increase end.
template <typename T>
int pair_usable(int dev, bool* usable) {
  static std::atomic<unsigned long long> checked{0}, fits{0};
  auto kernel = linear_pair_kernel<T>;
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(checked.load() & bit)) {
    cudaFuncAttributes fa;
    cudaError_t e = cudaFuncGetAttributes(&fa, kernel);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncGetAttributes");
    if (fa.numRegs == kPairRegs) {
      e = cudaFuncSetAttribute(
          kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem);
      if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute");
      fits.fetch_or(bit);
    }
    checked.fetch_or(bit);
  }
  *usable = (fits.load() & bit) != 0;
  return NVFP4DG_OK;
}

// (pair_usable has been asked)
template <typename T>
int launch_pair(const LinearParams& kp, const LinearPlan& pl,
                const CUtensorMap& tw, const CUtensorMap& tx,
                const CUtensorMap& tc, unsigned flags, cudaStream_t stream) {
  auto kernel = linear_pair_kernel<T>;
  LinearParams p = kp;
  p.m_tiles = (p.M + 255) / 256;
  p.n_tiles = (p.N + 255) / 256;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(pl.grid, 1, 1);
  cfg.blockDim = dim3(kPairThreads, 1, 1);
  cfg.dynamicSmemBytes = kPairSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeClusterDimension;
  attrs[0].val.clusterDim.x = 2;
  attrs[0].val.clusterDim.y = 1;
  attrs[0].val.clusterDim.z = 1;
  attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = (flags & NVFP4DG_FLAG_NO_PDL) ? 1 : 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, tw, tx, tc, p);
  if (e != cudaSuccess) return host_cuda_fail(e, "linear_pair_kernel launch");
  return NVFP4DG_OK;
}

int check_linear_flags(unsigned flags) {
  const unsigned t = flags & (NVFP4DG_LINEAR_TOKENS32 |
                              NVFP4DG_LINEAR_TOKENS64 |
                              NVFP4DG_LINEAR_TOKENS128 | NVFP4DG_LINEAR_PAIR);
  if (t & (t - 1))
    return host_fail(NVFP4DG_ERR_INVALID, "the tile flags are exclusive");
  const unsigned known = NVFP4DG_LINEAR_TOKENS32 | NVFP4DG_LINEAR_TOKENS64 |
                         NVFP4DG_LINEAR_TOKENS128 | NVFP4DG_LINEAR_PAIR |
                         NVFP4DG_LINEAR_SPLIT_MASK |
                         NVFP4DG_LINEAR_TEST_NO_PAIR |
                         NVFP4DG_FLAG_SYNC_CHECK | NVFP4DG_FLAG_NO_PDL;
  if (flags & ~known)
    return host_fail(NVFP4DG_ERR_INVALID, "unknown flag bits");
  if (((flags & NVFP4DG_LINEAR_SPLIT_MASK) >> 8) > 4)
    return host_fail(NVFP4DG_ERR_INVALID, "split must be 1, 2, 4 or 8");
  return NVFP4DG_OK;
}

int check_linear(const nvfp4_linear_args* a, int groups,
                 bool placed_on_device) {
  if (a == nullptr) return host_fail(NVFP4DG_ERR_INVALID, "args is NULL");
  if (a->M < 0 || a->N < 0 || a->K < 0)
    return host_fail(NVFP4DG_ERR_INVALID, "M, N, K must be non-negative");
  if (a->N % 8 != 0)
    return host_fail(NVFP4DG_ERR_INVALID, "N must be a multiple of 8");
  if (a->K == 0 || a->K % 64 != 0)
    return host_fail(NVFP4DG_ERR_INVALID,
                     "K must be a positive multiple of 64");
  if (a->c_dtype != NVFP4DG_DTYPE_F16 && a->c_dtype != NVFP4DG_DTYPE_BF16)
    return host_fail(NVFP4DG_ERR_INVALID, "C must be F16 or BF16");
  if (a->bias != nullptr && a->bias_dtype != NVFP4DG_DTYPE_F32 &&
      a->bias_dtype != a->c_dtype)
    return host_fail(NVFP4DG_ERR_INVALID, "bias must be F32 or of C's type");
  if (a->activation < NVFP4DG_ACT_NONE || a->activation > NVFP4DG_ACT_GELU)
    return host_fail(NVFP4DG_ERR_INVALID, "unknown activation");
  if (const int rc = check_linear_flags(a->flags)) return rc;
  if (a->alpha != a->alpha)
    return host_fail(NVFP4DG_ERR_INVALID, "alpha is NaN");
  if (a->M == 0 || a->N == 0) return NVFP4DG_OK;
  // tile numbers are 32-bit; groups placed by the device may overlap, so each
  // of them counts as all rows
  const long long per = groups && placed_on_device ? groups : 1;
  if (((a->M + 31ll) / 32 * per + groups) * ((a->N + 127ll) / 128) >=
          (1ll << 30) ||
      a->M > (1 << 30) || a->N > (1 << 30) || a->K > (1 << 30))
    return host_fail(NVFP4DG_ERR_INVALID, "too many tiles (M * N too large)");
  if (a->C == nullptr) return host_fail(NVFP4DG_ERR_INVALID, "C is NULL");
  if (a->ldc >= (1 << 23) || (a->residual != nullptr && a->ldr >= (1 << 23)))
    return host_fail(NVFP4DG_ERR_INVALID, "row pitch too large");
  if (a->ldc < a->N || (a->residual != nullptr && a->ldr < a->N))
    return host_fail(NVFP4DG_ERR_INVALID,
                     "the row pitch of C and residual must be at least N");
  const void* ops[4] = {a->A, a->B, a->SFA, a->SFB};
  const char* names[4] = {"A", "B", "SFA", "SFB"};
  for (int i = 0; i < 4; ++i) {
    if (ops[i] == nullptr)
      return host_fail(NVFP4DG_ERR_INVALID,
                       std::string(names[i]) + " is NULL");
    if (reinterpret_cast<uintptr_t>(ops[i]) % 16 != 0)
      return host_fail(NVFP4DG_ERR_ALIGN, std::string(names[i]) +
                                              " is not 16-byte aligned");
  }
  if (reinterpret_cast<uintptr_t>(a->C) % 16 || a->ldc % 8 ||
      reinterpret_cast<uintptr_t>(a->residual) % 16 ||
      (a->residual != nullptr && a->ldr % 8))
    return host_fail(NVFP4DG_ERR_ALIGN,
                     "C, residual and their row pitches must be 16-byte "
                     "aligned");
  const size_t be = a->bias_dtype == NVFP4DG_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a->bias) % be ||
      reinterpret_cast<uintptr_t>(a->row_scale) % 4)
    return host_fail(NVFP4DG_ERR_ALIGN,
                     "bias and row_scale must be aligned to their elements");
  // each output is written by the thread that read its residual, and by no
  // other: in place is safe, a shift is not
  if (host_overlap(a->C, 2 * a->ldc, a->residual, 2 * a->ldr, a->M,
                   2ll * a->N) == Overlap::kPart)
    return host_fail(NVFP4DG_ERR_INVALID,
                     "residual must be C itself or not overlap it");
  return NVFP4DG_OK;
}

// CTAs read the inputs while others write C.
int check_linear_overlap(const nvfp4_linear_args* a, int groups) {
  const long long n = a->N, k = a->K, per = std::max(groups, 1);
  const long long bias = a->bias_dtype == NVFP4DG_DTYPE_F32 ? 4 : 2;
  const struct {
    const char* name;
    const void* p;
    long long bytes;
  } inputs[] = {
      {"A", a->A, a->M * (k / 2)},
      {"B", a->B, per * n * (k / 2)},
      {"SFA", a->SFA, (a->M + 127ll) / 128 * (k / 64) * kAtomBytes},
      {"SFB", a->SFB, per * ((n + 127) / 128) * (k / 64) * kAtomBytes},
      {"bias", a->bias, per * n * bias},
      {"row_scale", a->row_scale, a->M * 4ll},
  };
  for (const auto& in : inputs)
    if (host_meets(in.p, in.bytes, a->C, 2 * a->ldc, a->M, 2 * n))
      return host_fail(NVFP4DG_ERR_INVALID,
                       std::string("C must not overlap ") + in.name);
  return NVFP4DG_OK;
}

int run_linear(const nvfp4_linear_args* a, const int* group_rows,
               const int* group_row0, int groups, bool on_device,
               void* stream_ptr) {
  host_clear_error();
  int rc = check_linear(a, groups, on_device && group_row0 != nullptr);
  if (rc) return rc;
  LinearParams p;
  std::memset(&p, 0, sizeof(p));
  long long mt[4] = {0, 0, 0, 0}, tokens = 0;
  if (groups > 0 && !on_device) {
    long long next = 0;
    for (int g = 0; g < groups; ++g) {
      const long long n = group_rows[g];
      const long long r0 = group_row0 ? group_row0[g] : next;
      if (n < 0 || r0 < 0 || r0 % 128 != 0)
        return host_fail(NVFP4DG_ERR_INVALID,
                         "group " + std::to_string(g) +
                             ": rows must be >= 0 and the first row a "
                             "multiple of 128");
      if (n > 0 && r0 < next)
        return host_fail(NVFP4DG_ERR_INVALID,
                         "group " + std::to_string(g) +
                             " overlaps the previous one (each group's rows "
                             "are rounded up to 128)");
      if (n > 0 && r0 + n > a->M)
        return host_fail(NVFP4DG_ERR_INVALID,
                         "group " + std::to_string(g) +
                             " reaches past the " + std::to_string(a->M) +
                             " rows of A");
      if (n > 0) next = r0 + (n + 127) / 128 * 128;
      p.rows[g] = static_cast<int>(n);
      p.row0[g] = n > 0 ? static_cast<int>(r0) : 0;
      mt[0] += (n + 31) / 32;
      mt[1] += (n + 63) / 64;
      mt[2] += (n + 127) / 128;
      mt[3] += (n + 255) / 256;
    }
    if (mt[0] == 0 || a->N == 0) return NVFP4DG_OK;
    tokens = mt[0] * 32;
  } else {
    if (a->M == 0 || a->N == 0) return NVFP4DG_OK;
    // counts on the device: A's rows spread evenly.  A tight A pads each
    // group to 128 rows, by 127 at most and 64 on average; 96 are taken off,
    // but no more than three quarters.  An A sized for more rows than there
    // are gets the tile of those (32 experts of 4 rows, each in 256 rows of A,
    // 4096 x 2048: 44 us with the pairs this gives, 28 with 32 tokens), which
    // a tile flag prevents.
    long long per = groups ? (a->M + groups - 1) / groups : a->M;
    if (groups) per = std::max(per - 96, (per + 3) / 4);
    tokens = per * std::max(groups, 1);
    const long long g = groups ? groups : 1;
    mt[0] = (per + 31) / 32 * g;
    mt[1] = (per + 63) / 64 * g;
    mt[2] = (per + 127) / 128 * g;
    mt[3] = (per + 255) / 256 * g;
  }
  if ((rc = check_linear_overlap(a, groups))) return rc;
  HostDevice dev;
  if ((rc = host_device(&dev))) return rc;
  const bool bf = a->c_dtype == NVFP4DG_DTYPE_BF16;
  auto plan = [&](bool pairs) {
    return plan_linear(mt, tokens, a->N, a->K, groups, a->residual != nullptr,
                       a->flags, dev.sms, pairs);
  };
  LinearPlan pl = plan(true);
  if (pl.tn == 0)
    return host_fail(NVFP4DG_ERR_INVALID, "pairs need two SMs");
  if (pl.tn == 256) {
    bool usable = false;
    if ((rc = bf ? pair_usable<__nv_bfloat16>(dev.id, &usable)
                 : pair_usable<__half>(dev.id, &usable)))
      return rc;
    if (!usable || (a->flags & NVFP4DG_LINEAR_TEST_NO_PAIR)) pl = plan(false);
    if (pl.tn == 0)
      return host_fail(NVFP4DG_ERR_UNSUPPORTED,
                       "this build's pair kernel cannot be launched");
  }
  // tiles counted by the kernel: a full grid
  if (groups > 0 && on_device)
    pl.grid = pl.tn == 256 ? dev.sms / 2 * 2 : dev.sms;
  p.M = a->M;
  p.N = a->N;
  p.K = a->K;
  p.kblocks = pl.kblocks;
  p.n_tiles = (a->N + kFeat - 1) / kFeat;
  p.split = pl.split;
  p.sfa = static_cast<const uint8_t*>(a->SFA);
  p.sfb = static_cast<const uint8_t*>(a->SFB);
  p.sfb_group = (a->N + 127ll) / 128 * (a->K / 64) * kAtomBytes;
  p.C = a->C;
  p.ldc = a->ldc;
  p.bias = a->bias;
  p.bias_f32 = a->bias_dtype == NVFP4DG_DTYPE_F32;
  p.residual = a->residual;
  p.ldr = a->ldr;
  p.row_scale = a->row_scale;
  p.alpha = a->alpha;
  p.act = a->activation;
  p.err = dev.err;
  p.groups = groups;
  p.dev_rows = on_device ? group_rows : nullptr;
  p.dev_row0 = on_device ? group_row0 : nullptr;
  CUtensorMap tw, tx;
  const long long kb = a->K / 2;
  if ((rc = host_byte_map(a->B, a->N, kb, kb, kFeat, std::max(groups, 1),
                          a->N * kb, &tw)))
    return rc;
  if ((rc = host_byte_map(a->A, a->M, kb, kb, std::min(pl.tn, 128), 1,
                          a->M * kb, &tx)))
    return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
  if (pl.tn == 256) {
    CUtensorMap tc;
    if ((rc = host_byte_map(a->C, a->M, 2ll * a->N, 2 * a->ldc, 128, 0, 0,
                            &tc)))
      return rc;
    rc = bf ? launch_pair<__nv_bfloat16>(p, pl, tw, tx, tc, a->flags, stream)
            : launch_pair<__half>(p, pl, tw, tx, tc, a->flags, stream);
  } else if (pl.tn == 32)
    rc = bf ? launch_linear<__nv_bfloat16, 32>(p, pl, tw, tx, dev.id,
                                               a->flags, stream)
            : launch_linear<__half, 32>(p, pl, tw, tx, dev.id, a->flags,
                                        stream);
  else if (pl.tn == 64)
    rc = bf ? launch_linear<__nv_bfloat16, 64>(p, pl, tw, tx, dev.id,
                                               a->flags, stream)
            : launch_linear<__half, 64>(p, pl, tw, tx, dev.id, a->flags,
                                        stream);
  else
    rc = bf ? launch_linear<__nv_bfloat16, 128>(p, pl, tw, tx, dev.id,
                                                a->flags, stream)
            : launch_linear<__half, 128>(p, pl, tw, tx, dev.id, a->flags,
                                         stream);
  if (rc) return rc;
  return (a->flags & NVFP4DG_FLAG_SYNC_CHECK) ? host_sync_check(stream)
                                              : NVFP4DG_OK;
}

}  // namespace
}  // namespace nvfp4dg

extern "C" {

int nvfp4_linear_run(const nvfp4_linear_args* args, void* stream) {
  return nvfp4dg::host_guarded([&] {
    return nvfp4dg::run_linear(args, nullptr, nullptr, 0, false, stream);
  });
}

int nvfp4_linear_run_grouped(const nvfp4_linear_args* args,
                             const int* group_rows, const int* group_row0,
                             int groups, int on_device, void* stream) {
  return nvfp4dg::host_guarded([&] {
    nvfp4dg::host_clear_error();
    if (groups < 1 || groups > nvfp4dg::kMaxGroups)
      return nvfp4dg::host_fail(
          NVFP4DG_ERR_INVALID,
          "groups must be 1.." + std::to_string(nvfp4dg::kMaxGroups));
    if (group_rows == nullptr)
      return nvfp4dg::host_fail(NVFP4DG_ERR_INVALID,
                                "group_rows is required");
    if (args != nullptr && args->residual != nullptr)
      return nvfp4dg::host_fail(NVFP4DG_ERR_INVALID,
                                "grouped products take no residual");
    return nvfp4dg::run_linear(args, group_rows, group_row0, groups,
                               on_device != 0, stream);
  });
}

int nvfp4_linear_plan(int M, int N, int K, int residual, unsigned flags,
                      int num_sms, int* tokens_out, int* split_out,
                      int* grid_out) {
  return nvfp4dg::host_guarded([&] {
    nvfp4dg::host_clear_error();
    if (M <= 0 || N <= 0 || K <= 0 || N % 8 || K % 64 || num_sms <= 0)
      return nvfp4dg::host_fail(NVFP4DG_ERR_INVALID,
                                "invalid problem for planning");
    if (const int rc = nvfp4dg::check_linear_flags(flags)) return rc;
    const long long mts[4] = {(M + 31ll) / 32, (M + 63ll) / 64,
                              (M + 127ll) / 128, (M + 255ll) / 256};
    const nvfp4dg::LinearPlan pl = nvfp4dg::plan_linear(
        mts, M, N, K, 0, residual != 0, flags, num_sms,
        !(flags & NVFP4DG_LINEAR_TEST_NO_PAIR));
    if (pl.tn == 0)
      return nvfp4dg::host_fail(NVFP4DG_ERR_INVALID, "pairs need two SMs");
    if (tokens_out) *tokens_out = pl.tn;
    if (split_out) *split_out = pl.split;
    if (grid_out) *grid_out = pl.grid;
    return NVFP4DG_OK;
  });
}

}  // extern "C"
