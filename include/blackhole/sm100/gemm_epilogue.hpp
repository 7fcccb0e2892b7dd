#pragma once

// =====================================================================================
// blackhole / sm100 / epilogue of the block-scaled products and its gradient
// -------------------------------------------------------------------------------------
//     z = alpha * A . B^T + bias                       (FP32)
//     u = act(z), or gated: u[:, j] = act(z[:, 2j]) * z[:, 2j + 1]
//     D = bf16(u + beta * residual);   optionally Z = bf16(z), kept for the backward pass
//
// applied to the accumulators between TMEM and the store, in FP32, rounded once.  Gate and up
// features alternate (rows 2j and 2j + 1 of B), so a pair meets in one thread (one-SM and two-SM
// schedules: a thread owns a row's columns) or in two neighbouring lanes (skinny schedule).
//
// Backward, from the stored Z:  dZ = dD * act'(Z), gated dZ[:, 2j] = dD act'(g) u and
// dZ[:, 2j + 1] = dD act(g);  dbias = sum of its rows.  Bound by its bytes.
//
// Measured on B200: 8192^3 NVFP4 without any of it 209 us, SwiGLU 203, bias + GELU + residual 249
// (plain product 203: the epilogue of a tile runs beside the next tile's products, and costs where
// it is longer or competes for issue slots); M = 1, N = 28672, K = 8192 SwiGLU 24.5 us (plain
// 23.4).  Backward, 8192 x 28672 SwiGLU: 1.17 GB in 190-197 us (0.91-0.95 of the measured copy rate).
// =====================================================================================

#include <cmath>
#include <cstdint>

#include <cuda_runtime_api.h>

#include <blackhole/sm100/column_sum.hpp>
#include <blackhole/sm100/f32x2.hpp>
#include <blackhole/sm100/nvfp4_gemm_common.hpp>
#include <blackhole_sm100.h>

namespace blackhole::sm100 {

// (kNoEpilogue: a kernel without one.)
constexpr int kNoEpilogue = -1;
enum Activation : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };

namespace detail {

// Whether two byte ranges meet.
inline bool ranges_overlap(const void* a, int64_t an, const void* b, int64_t bn) {
  if (!a || !b || an <= 0 || bn <= 0) return false;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + static_cast<uintptr_t>(bn) && y < x + static_cast<uintptr_t>(an);
}

}  // namespace detail

// Host-only check of an epilogue for an M x N product (after nvfp4_check_args).
inline cudaError_t epilogue_check_args(int M, int N, const void* D,
                                       const blackhole_sm100_epilogue* e) {
  if (!e) return cudaErrorInvalidValue;
  if (e->activation < kActNone || e->activation > kActSilu) return cudaErrorInvalidValue;
  if (e->gated && N % 16 != 0) return cudaErrorInvalidValue;   // D's rows stay 16-byte aligned
  auto mis = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
  if (mis(e->bias) || mis(e->residual) || mis(e->Z)) return cudaErrorInvalidValue;
  if (e->residual && !std::isfinite(e->beta)) return cudaErrorInvalidValue;
  const int64_t d = int64_t(M) * (e->gated ? N / 2 : N) * 2, z = int64_t(M) * N * 2;
  if (e->residual && e->residual != D && detail::ranges_overlap(e->residual, d, D, d))
    return cudaErrorInvalidValue;
  if (detail::ranges_overlap(e->Z, z, D, d) || detail::ranges_overlap(e->Z, z, e->residual, d))
    return cudaErrorInvalidValue;
  return cudaSuccess;
}

// Warp roles of the tiled schedules with an epilogue: 4 control warps (TMA, MMA, scale-factor
// copies, one idle) and 8 epilogue warps, so that registers can be split by warpgroup: an epilogue
// warp holds a row's 128 accumulators, 64 columns of the residual and the activation's temporaries,
// which at an even split (168 each) spilled 0.4-1.1 KB per thread.  (Sixteen epilogue warps of 64
// columns: 2048 x 8192 x 2048 with GELU, bias, residual and Z 65 -> 55 us, but 8192^3 without any
// of them 212 -> 227 us, through their 64-byte store rows.)
template <class Base>
struct FusedTraits : Base {
  static constexpr bool RegSplit = true;
  static constexpr int NumWarps = 12;
  static constexpr int NumThreads = NumWarps * 32;
  static constexpr int FirstEpiWarp = 4;
  static constexpr int SfWarp = 2;
  static constexpr int ControlRegs = 64;
  static constexpr int EpiRegs = 208;
  static constexpr int MinRegs = (ControlRegs * 128 + EpiRegs * 256 + NumThreads - 1) / NumThreads;   // 160
  static_assert(Base::NumEpiWarps == 8, "two warpgroups of epilogue warps");
};

#if defined(__CUDACC__)

namespace detail {

// ---- activations, on pairs ------------------------------------------------------------------
// exp2 and the reciprocal are the hardware's approximations (relative error about 2^-22.5 and
// 2^-23, against the 2^-9 of the BF16 result).  Every form keeps its relative accuracy in the
// tails, where 1 + tanh or 1 + erf would cancel, and passes NaN on.
__device__ __forceinline__ float2 exp2_2(float2 v) {
  float2 r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(v.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(v.y));
  return r;
}
__device__ __forceinline__ float2 rcp2(float2 v) {
  float2 r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(v.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(v.y));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
constexpr float kLog2e = 1.44269504088896f;
constexpr float kTanhA = 1.59576912160573f;      // 2 sqrt(2 / pi)
constexpr float kTanhB = 0.0713548162726009f;    // 2 sqrt(2 / pi) 0.044715

// 1 / (1 + exp(-w)) for w = k z (1 + ...): sigmoid of the SiLU's or the tanh GELU's argument.
template <int kAct>
__device__ __forceinline__ float2 sigmoid2(float2 z) {
  float2 a;
  if constexpr (kAct == kActSilu) {
    a = mul2(z, both(-kLog2e));
  } else {
    a = mul2(z, fma2(mul2(z, z), both(-kLog2e * kTanhB), both(-kLog2e * kTanhA)));
  }
  return rcp2(add2(exp2_2(a), both(1.f)));
}
// Upper tail of the normal distribution at a = |z| (Q = erfc(a / sqrt 2) / 2) and exp(-a^2 / 2):
// Q = exp(-a^2 / 2) t P(t) with t = 1 / (1 + 0.3 a), the form of Hastings' error function
// approximations; P of degree 7 fitted here to the scaled complementary error function over
// a <= 14 (relative error 1.5e-7; exp underflows beyond).
__device__ __forceinline__ float2 normal_tail2(float2 a, float2& gauss) {
  const float2 t = rcp2(fma2(a, both(0.3f), both(1.f)));
  gauss = exp2_2(mul2(mul2(a, a), both(-0.5f * kLog2e)));
  float2 q = both(0.03567494208754076f);
  q = fma2(q, t, both(-0.15720365847955728f));
  q = fma2(q, t, both(0.20635430300401225f));
  q = fma2(q, t, both(-0.05368421566859173f));
  q = fma2(q, t, both(0.12856185346333843f));
  q = fma2(q, t, both(0.09991344303050201f));
  q = fma2(q, t, both(0.12075396126465843f));
  q = fma2(q, t, both(0.11962929862715543f));
  return mul2(mul2(q, t), gauss);
}

template <int kAct>
__device__ __forceinline__ float2 act_value2(float2 z) {
  if constexpr (kAct == kActRelu) return make_float2(max_nan(z.x, 0.f), max_nan(z.y, 0.f));
  if constexpr (kAct == kActGelu) {
    // z Phi(z) = max(z, 0) - |z| Q(|z|); |z| past 40 has Q = 0
    const float2 a = make_float2(min_nan(fabsf(z.x), 40.f), min_nan(fabsf(z.y), 40.f));
    float2 gauss;
    const float2 q = normal_tail2(a, gauss);
    return fma2(make_float2(-a.x, -a.y), q, make_float2(max_nan(z.x, 0.f), max_nan(z.y, 0.f)));
  }
  if constexpr (kAct == kActGeluTanh || kAct == kActSilu) return mul2(z, sigmoid2<kAct>(z));
  return z;
}

// act(z) and act'(z)
template <int kAct>
__device__ __forceinline__ void act_value_slope2(float2 z, float2& value, float2& slope) {
  if constexpr (kAct == kActRelu) {
    value = act_value2<kActRelu>(z);
    slope = make_float2(z.x > 0.f ? 1.f : z.x <= 0.f ? 0.f : z.x, z.y > 0.f ? 1.f : z.y <= 0.f ? 0.f : z.y);
  } else if constexpr (kAct == kActGelu) {
    const float2 c = make_float2(max_nan(min_nan(z.x, 40.f), -40.f), max_nan(min_nan(z.y, 40.f), -40.f));
    const float2 a = make_float2(fabsf(c.x), fabsf(c.y));
    float2 gauss;
    const float2 q = normal_tail2(a, gauss);
    value = fma2(make_float2(-a.x, -a.y), q, make_float2(max_nan(z.x, 0.f), max_nan(z.y, 0.f)));
    const float2 phi = make_float2(z.x > 0.f ? 1.f - q.x : q.x, z.y > 0.f ? 1.f - q.y : q.y);
    slope = fma2(mul2(c, both(0.398942280401433f)), gauss, phi);
  } else if constexpr (kAct == kActGeluTanh) {
    // past |z| = 30 the sigmoid is 0 or 1 exactly, so its slope is taken at the clamped z, where
    // the cubic does not overflow
    const float2 c = make_float2(max_nan(min_nan(z.x, 30.f), -30.f), max_nan(min_nan(z.y, 30.f), -30.f));
    const float2 s = sigmoid2<kAct>(c);
    value = mul2(z, s);
    const float2 rest = fma2(make_float2(-s.x, -s.y), s, s);                    // s (1 - s)
    slope = fma2(mul2(c, rest), fma2(mul2(c, c), both(3.f * kTanhB), both(kTanhA)), s);
  } else if constexpr (kAct == kActSilu) {
    const float2 s = sigmoid2<kAct>(z);
    value = mul2(z, s);
    slope = mul2(s, fma2(z, add2(both(1.f), make_float2(-s.x, -s.y)), both(1.f)));
  } else {
    value = z;
    slope = both(1.f);
  }
}

// Runs f with the activation as a compile-time constant (the skinny schedule; the tiled schedules
// are built once per activation: choosing among five inside them spilled 0.6 KB per thread).
template <class F>
__device__ __forceinline__ void with_activation(int act, F f) {
  switch (act) {
    case kActRelu: f(std::integral_constant<int, kActRelu>{}); break;
    case kActGelu: f(std::integral_constant<int, kActGelu>{}); break;
    case kActGeluTanh: f(std::integral_constant<int, kActGeluTanh>{}); break;
    case kActSilu: f(std::integral_constant<int, kActSilu>{}); break;
    default: f(std::integral_constant<int, kActNone>{}); break;
  }
}

// ---- forward, on accumulators in registers --------------------------------------------------
struct EpilogueParams {
  CUtensorMap tmap_z;        // Z as D's map (one-SM and two-SM schedules, has_z only)
  const void* bias;
  const uint16_t* residual;  // BF16, rows of n_out
  uint16_t* z;               // BF16, rows of N (skinny schedule)
  float beta;
  int activation, gated, bias_bf16, has_z;
  int n_out;                 // columns of D
  int residual_wide;         // residual rows start on 32-byte boundaries
};

__device__ __forceinline__ float bf16_value(uint16_t bits) {
  return __uint_as_float(static_cast<uint32_t>(bits) << 16);
}
__device__ __forceinline__ float epilogue_bias(const EpilogueParams& e, int n) {
  if (!e.bias) return 0.f;
  return e.bias_bf16 ? bf16_value(__ldg(static_cast<const uint16_t*>(e.bias) + n))
                     : __ldg(static_cast<const float*>(e.bias) + n);
}

__device__ __forceinline__ float2 bits2(const uint32_t* v) {
  return make_float2(__uint_as_float(v[0]), __uint_as_float(v[1]));
}
__device__ __forceinline__ void set_bits2(uint32_t* v, float2 f) {
  v[0] = __float_as_uint(f.x);
  v[1] = __float_as_uint(f.y);
}

// A 16-byte load that stays where it is written: the compiler would otherwise raise a tile's bias
// and residual loads together and spill the accumulators.
__device__ __forceinline__ uint4 load16_here(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

// 32 bytes in one request (32-byte aligned): whole sectors where each lane reads a row of its own.
__device__ __forceinline__ void load32_here(const void* p, uint4& a, uint4& b) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
               : "l"(p)
               : "memory");
}

// z of 32 consecutive columns of a row, in place of the accumulators' bits.
__device__ __forceinline__ void epilogue_z32(uint32_t (&v)[32], float alpha, const EpilogueParams& e,
                                             int col, int N) {
  if (!e.bias) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) set_bits2(v + i, mul2(bits2(v + i), both(alpha)));
    return;
  }
  const int n = N - col;
  if (e.bias_bf16) {
    uint4 q[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      q[g] = make_uint4(0, 0, 0, 0);
      if (8 * g < n) q[g] = load16_here(static_cast<const uint16_t*>(e.bias) + col + 8 * g);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint32_t w[4] = {q[g].x, q[g].y, q[g].z, q[g].w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        set_bits2(v + 8 * g + 2 * i, fma2(bits2(v + 8 * g + 2 * i), both(alpha), unpack2(w[i])));
    }
  } else {
    uint4 q[8];
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      q[g] = make_uint4(0, 0, 0, 0);
      if (4 * g < n) q[g] = load16_here(static_cast<const float*>(e.bias) + col + 4 * g);
    }
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      set_bits2(v + 4 * g, fma2(bits2(v + 4 * g), both(alpha), bits2(&q[g].x)));
      set_bits2(v + 4 * g + 2, fma2(bits2(v + 4 * g + 2), both(alpha), bits2(&q[g].z)));
    }
  }
}

// u of those columns: 32 values, or 16 (in v[0..15]) when gated.
template <int A>
__device__ __forceinline__ void epilogue_act32(uint32_t (&v)[32], const EpilogueParams& e) {
  if (e.gated) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float2 p0 = bits2(v + 2 * i), p1 = bits2(v + 2 * i + 2);      // (gate, up) twice
      set_bits2(v + i, mul2(act_value2<A>(make_float2(p0.x, p1.x)), make_float2(p0.y, p1.y)));
    }
  } else if constexpr (A != kActNone) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) set_bits2(v + i, act_value2<A>(bits2(v + i)));
  }
}

// The residual of up to kCols consecutive columns of D's row (zeros outside D): half of them when
// gated, as D has half the columns of the accumulators.
template <int kCols>
struct ResidualRow {
  uint4 q[kCols / 8];
  __device__ __forceinline__ void fetch(const EpilogueParams& e, int row, int col, int M) {
    if (!e.residual) return;
    const uint16_t* p = e.residual + int64_t(row) * e.n_out + col;
    const int n = row < M ? min(e.n_out - col, e.gated ? kCols / 2 : kCols) : 0;
    if (e.residual_wide) {
#pragma unroll
      for (int c = 0; c < kCols / 8; c += 2) {
        q[c] = q[c + 1] = make_uint4(0, 0, 0, 0);
        if (8 * c < n) load32_here(p + 8 * c, q[c], q[c + 1]);
      }
      return;
    }
#pragma unroll
    for (int c = 0; c < kCols / 8; ++c) {
      q[c] = make_uint4(0, 0, 0, 0);
      if (8 * c < n) q[c] = load16_here(p + 8 * c);
    }
  }
};
// BF16 of 8 FP32 values (their bits), plus beta * residual where q is given.
__device__ __forceinline__ uint4 epilogue_pack8(const uint32_t* v, const EpilogueParams& e, const uint4* q) {
  float2 f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = bits2(v + 2 * i);
  if (q && e.residual) {
    const uint32_t w[4] = {q->x, q->y, q->z, q->w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = fma2(unpack2(w[i]), both(e.beta), f[i]);
  }
  return make_uint4(pack_bf16x2(f[0].x, f[0].y), pack_bf16x2(f[1].x, f[1].y), pack_bf16x2(f[2].x, f[2].y),
                    pack_bf16x2(f[3].x, f[3].y));
}
// Fills the kernels' parameters; box_cols: columns of the schedule's store box (0: no map).
inline cudaError_t make_epilogue(EpilogueParams* p, const blackhole_sm100_epilogue& e, int M, int N,
                                 int box_cols) {
  p->bias = e.bias;
  p->residual = static_cast<const uint16_t*>(e.residual);
  p->z = static_cast<uint16_t*>(e.Z);
  p->beta = e.beta;
  p->activation = e.activation;
  p->gated = e.gated != 0;
  p->bias_bf16 = e.bias_is_bf16 != 0;
  p->has_z = e.Z != nullptr;
  p->n_out = e.gated ? N / 2 : N;
  p->residual_wide = p->n_out % 16 == 0 && (reinterpret_cast<uintptr_t>(e.residual) & 31u) == 0;
  if (e.Z && box_cols > 0) return make_d_tmap(&p->tmap_z, e.Z, M, N, box_cols);
  return cudaSuccess;
}

// ---- backward --------------------------------------------------------------------------------
constexpr int kEpilogueBackCols = 256;      // columns of Z per CTA: 32 lanes x 8
constexpr int kEpilogueBackCluster = 8;     // row chunks a cluster can add up

struct EpilogueBackwardParams {
  const uint16_t *d, *z;
  uint16_t* dz;
  float* dbias;
  float* ws;               // [row chunks][N] partial column sums
  int M, N, gated, chunks, rows_per_chunk;
  int cluster;             // row chunks that are one cluster (1: partial sums through ws)
};

template <int kAct>
__global__ void __launch_bounds__(256) epilogue_backward_kernel(const __grid_constant__ EpilogueBackwardParams p) {
  __shared__ float acc_s[8][kEpilogueBackCols];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kRows = 4;
  const int col = blockIdx.x * kEpilogueBackCols + lane * 8;
  const int row0 = blockIdx.y * p.rows_per_chunk;
  const int row1 = min(p.M, row0 + p.rows_per_chunk);
  ptx::pdl_launch_dependents();
  ptx::pdl_wait_prior_grid();
  float2 acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = both(0.f);
  if (col < p.N) {
    // kRows rows of a warp in flight together: with one the loads' latency set the pace
    for (int row = row0 + warp; row < row1; row += 8 * kRows) {
      uint4 zq[kRows], dq[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const int64_t at = int64_t(row + 8 * u) * p.N + col;
        zq[u] = dq[u] = make_uint4(0, 0, 0, 0);
        if (row + 8 * u < row1) {
          zq[u] = __ldcs(reinterpret_cast<const uint4*>(p.z + at));
          if (p.gated) {
            const uint2 q = __ldcs(reinterpret_cast<const uint2*>(p.d + at / 2));
            dq[u].x = q.x;
            dq[u].y = q.y;
          } else {
            dq[u] = __ldcs(reinterpret_cast<const uint4*>(p.d + at));
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        if (row + 8 * u >= row1) break;
        const float2 z[4] = {unpack2(zq[u].x), unpack2(zq[u].y), unpack2(zq[u].z), unpack2(zq[u].w)};
        const float2 d[4] = {unpack2(dq[u].x), unpack2(dq[u].y), unpack2(dq[u].z), unpack2(dq[u].w)};
        float2 g[4];
        if (p.gated) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float2 value, slope;
            act_value_slope2<kAct>(make_float2(z[2 * i].x, z[2 * i + 1].x), value, slope);
            const float2 dg = mul2(mul2(d[i], make_float2(z[2 * i].y, z[2 * i + 1].y)), slope);
            const float2 du = mul2(d[i], value);
            g[2 * i] = make_float2(dg.x, du.x);
            g[2 * i + 1] = make_float2(dg.y, du.y);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float2 value, slope;
            act_value_slope2<kAct>(z[i], value, slope);
            g[i] = mul2(d[i], slope);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = add2(acc[i], g[i]);
        *reinterpret_cast<uint4*>(p.dz + int64_t(row + 8 * u) * p.N + col) =
            make_uint4(pack_bf16x2(g[0].x, g[0].y), pack_bf16x2(g[1].x, g[1].y), pack_bf16x2(g[2].x, g[2].y),
                       pack_bf16x2(g[3].x, g[3].y));
      }
    }
  }
  if (!p.dbias) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<float2*>(&acc_s[warp][lane * 8 + 2 * i]) = acc[i];
  __syncthreads();
  const int c = blockIdx.x * kEpilogueBackCols + threadIdx.x;
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += acc_s[w][threadIdx.x];
  if (p.cluster == 1) {
    if (c < p.N) (p.chunks == 1 ? p.dbias : p.ws + int64_t(blockIdx.y) * p.N)[c] = s;
    return;
  }
  // the chunks' sums to the cluster's first CTA, which adds them in order
  __shared__ float parts[kEpilogueBackCluster][kEpilogueBackCols];
  const uint32_t rank = ptx::cluster_ctarank();
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(
                   ptx::mapa_shared(ptx::smem_u32(&parts[rank][threadIdx.x]), 0)),
               "f"(s)
               : "memory");
  ptx::cluster_sync();
  if (rank == 0 && c < p.N) {
    float t = parts[0][threadIdx.x];
    for (int k = 1; k < p.chunks; ++k) t += parts[k][threadIdx.x];
    p.dbias[c] = t;
  }
}

static __global__ void __launch_bounds__(1024)
    epilogue_bias_sum_kernel(const __grid_constant__ EpilogueBackwardParams p) {
  __shared__ ColumnSumShared smem;
  ptx::pdl_launch_dependents();
  ptx::pdl_wait_prior_grid();
  column_sum_cta(nullptr, p.ws, p.chunks, p.N, p.dbias, p.N, blockIdx.x, smem);
}

}  // namespace detail

#endif  // __CUDACC__

constexpr int kEpilogueMaxRows = 1 << 30;     // (32-bit row arithmetic)

// Row chunks of the backward kernel, each of whole sets of 8 rows.  Up to kEpilogueClusterRows rows
// they are one cluster of at most 8, which adds the column sums itself: one launch and no
// workspace (333 x 1000: 11.5 -> 7.0 us per call).  Beyond, about eight CTAs per SM (148 SMs) leave partial sums to a
// second kernel.  Fixed by the sizes, so the workspace and the order of the sums are too.
constexpr int kEpilogueClusterRows = 1024;
inline void epilogue_backward_chunks(int M, int N, int* chunks, int* rows_per_chunk) {
  const int64_t cols = (int64_t(N) + 255) / 256;
  int64_t want = M <= kEpilogueClusterRows ? 8 : (148 * 8 + cols - 1) / cols;
  if (want < 1) want = 1;
  int64_t rows = (int64_t(M) + want - 1) / want;
  rows = (rows + 7) / 8 * 8;
  *rows_per_chunk = static_cast<int>(rows);
  *chunks = static_cast<int>((M + rows - 1) / rows);
}

inline int64_t gemm_fused_backward_workspace_bytes(int M, int N) {
  if (M < 1 || M > kEpilogueMaxRows || N < 8 || N % 8 != 0) return -1;
  int chunks, rows;
  epilogue_backward_chunks(M, N, &chunks, &rows);
  return chunks == 1 || M <= kEpilogueClusterRows ? 0 : int64_t(chunks) * N * 4;
}

// Host-only check.
inline cudaError_t gemm_fused_backward_check(int M, int N, const void* dD, const void* Z, const void* dZ,
                                             const float* dbias, int activation, int gated,
                                             const void* workspace, int64_t workspace_bytes) {
  if (M < 1 || M > kEpilogueMaxRows || N < 8 || N % 8 != 0 || (gated && N % 16 != 0))
    return cudaErrorInvalidValue;
  if (activation < kActNone || activation > kActSilu) return cudaErrorInvalidValue;
  if (!dD || !Z || !dZ) return cudaErrorInvalidValue;
  auto mis = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
  if (mis(dD) || mis(Z) || mis(dZ) || mis(dbias) || mis(workspace)) return cudaErrorInvalidValue;
  if (int64_t(M) * N > (int64_t(1) << 46)) return cudaErrorInvalidValue;
  const int64_t z = int64_t(M) * N * 2, d = gated ? z / 2 : z;
  if (dZ != Z && detail::ranges_overlap(dZ, z, Z, z)) return cudaErrorInvalidValue;
  if ((dZ != dD || gated) && detail::ranges_overlap(dZ, z, dD, d)) return cudaErrorInvalidValue;
  const int64_t need = gemm_fused_backward_workspace_bytes(M, N);
  if (dbias && need > 0 && (!workspace || workspace_bytes < need)) return cudaErrorInvalidValue;
  return cudaSuccess;
}

#if defined(__CUDACC__)

inline cudaError_t gemm_fused_backward(int M, int N, const void* dD, const void* Z, void* dZ, float* dbias,
                                       int activation, int gated, void* workspace,
                                       int64_t workspace_bytes, cudaStream_t stream) {
  cudaError_t e = gemm_fused_backward_check(M, N, dD, Z, dZ, dbias, activation, gated, workspace,
                                            workspace_bytes);
  if (e != cudaSuccess) return e;
  detail::EpilogueBackwardParams p;
  p.d = static_cast<const uint16_t*>(dD);
  p.z = static_cast<const uint16_t*>(Z);
  p.dz = static_cast<uint16_t*>(dZ);
  p.dbias = dbias;
  p.ws = static_cast<float*>(workspace);
  p.M = M;
  p.N = N;
  p.gated = gated != 0;
  epilogue_backward_chunks(M, N, &p.chunks, &p.rows_per_chunk);
  p.cluster = dbias && M <= kEpilogueClusterRows ? p.chunks : 1;
  const dim3 grid((N + detail::kEpilogueBackCols - 1) / detail::kEpilogueBackCols, p.chunks);
  void (*kernel)(detail::EpilogueBackwardParams) = nullptr;
  switch (activation) {
    case kActRelu: kernel = detail::epilogue_backward_kernel<kActRelu>; break;
    case kActGelu: kernel = detail::epilogue_backward_kernel<kActGelu>; break;
    case kActGeluTanh: kernel = detail::epilogue_backward_kernel<kActGeluTanh>; break;
    case kActSilu: kernel = detail::epilogue_backward_kernel<kActSilu>; break;
    default: kernel = detail::epilogue_backward_kernel<kActNone>; break;
  }
  e = detail::launch_pdl(kernel, grid, dim3(256), 0, stream, p, static_cast<unsigned>(p.cluster));
  if (e != cudaSuccess) return e;
  if (dbias && p.chunks > 1 && p.cluster == 1) {
    e = detail::launch_pdl(detail::epilogue_bias_sum_kernel, dim3((N + detail::kColumnSumCols - 1) / detail::kColumnSumCols), dim3(1024), 0,
                           stream, p);
    if (e != cudaSuccess) return e;
  }
  return cudaGetLastError();
}

#endif  // __CUDACC__

}  // namespace blackhole::sm100
