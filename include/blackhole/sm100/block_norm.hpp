#pragma once

// =====================================================================================
// blackhole / sm100 / norms before and after a block, fused with its gate and residual scale
// -------------------------------------------------------------------------------------
// Between two block-scaled products of a transformer stands, per row of H features,
//
//     p = o                       or  norm_post(o)       (o: the block's BF16 result)
//     h = x + scale * g * p                              (x: residual stream, g: gate)
//     y = norm(h) * weight + bias                        (the next block's input)
//
// with norm either RMS (v / sqrt(mean(v^2) + eps)) or layer ((v - mean) / sqrt(var + eps)).
// One kernel reads x and o once and writes h and y once; y leaves as BF16, FP32 or quantised as
// the next product's A operand (the recipes of nvfp4_quant.hpp on the FP32 y, no BF16 step in
// between), scale factors in the 128x4 layout.  Everything between the loads and the stores is
// FP32; y uses the FP32 h, not its stored rounding.
//
// Backward (a = dy * weight, n = (h - mean) * rstd from the stored h and statistics):
//     dh' = dh + rstd * (a - [mean(a)] - n * mean(a * n));   dx = dh'
//     dp  = scale * g * dh';   dg = scale * dh' * p, summed over the rows that share a gate row
//     do  = dp, or norm_post's gradient of it (same form)
//     dweight = sum dy * n, dbias = sum dy, and the same two of the post norm
// ([...]: layer norm only).
//
// A row is worked on by one CTA (H <= 8192) or a cluster of two (H <= 16384), 16 columns per
// thread as two 8-column vectors; CTAs are persistent, each over a range of consecutive rows.  Rows
// arrive in shared memory through a ring of bulk copies that runs ahead of the arithmetic, so that
// HBM keeps streaming through the row sums' barriers; the parameter vectors, with gate, scale and
// post weight multiplied into one, stay on the SM from row to row: in registers, or where there
// are biases as each thread's own columns in shared memory.  Measured at 16384 x 8192, BF16 stream,
// RMS norms before and after: to MXFP8 181 us (5.2 TB/s of 0.94 GB), to BF16 189 us (5.7), backward
// 281 us (5.7 of 1.61 GB).
// =====================================================================================

#include <algorithm>
#include <cmath>
#include <cstdint>

#include <cuda_runtime_api.h>

#include <blackhole/common/sf_layout.hpp>
#include <blackhole/sm100/column_sum.hpp>
#include <blackhole/sm100/f32x2.hpp>
#include <blackhole/sm100/gemm_epilogue.hpp>
#include <blackhole/sm100/nvfp4_gemm_common.hpp>
#include <blackhole/sm100/nvfp4_quant.hpp>
#include <blackhole_sm100.h>

namespace blackhole::sm100 {

constexpr int kNormMaxH = 16384;
constexpr int kNormMaxRows = 1 << 30;  // (32-bit row arithmetic)
constexpr int kNormSliceH = 8192;     // columns one CTA works on: 512 threads x 16

enum NormOut : int { kOutBf16 = 0, kOutF32 = 1, kOutNvfp4 = 2, kOutMxfp4 = 3, kOutMxfp8 = 4 };

namespace norm_detail {

struct Geometry {
  int cluster;      // CTAs per row: 1 or 2
  int slice;        // columns of a row per CTA (a multiple of 128 when cluster == 2)
  int threads;      // threads per CTA, 16 columns each
};
inline Geometry geometry(int H) {
  Geometry g;
  g.cluster = H > kNormSliceH ? 2 : 1;
  g.slice = g.cluster == 1 ? H : (((H + 1) / 2 + 127) / 128 * 128);
  g.threads = ((g.slice + 15) / 16 + 31) / 32 * 32;
  return g;
}

// Row ranges: `teams` CTAs (or clusters), each of rows [row_begin(t), row_begin(t + 1)), as many
// as are resident at once (512 threads of 128 registers or 640 of 96 per SM, 148 SMs).  Fixed by the sizes
// alone, so the workspace size and the order of the column sums do not depend on the device.
inline int row_teams(int rows, const Geometry& g, int threads_per_sm) {
  const int per_sm = std::max(1, threads_per_sm / g.threads);
  return std::min(rows, std::max(1, 148 * per_sm / g.cluster));
}
constexpr int kThreadsPerSm = 512;
constexpr int kNarrowThreads = 320, kNarrowThreadsPerSm = 640;
BLACKHOLE_HD inline int64_t row_begin(int64_t team, int64_t rows, int64_t teams) {
  return team * rows / teams;
}
// The team whose range holds `row`.
BLACKHOLE_HD inline int64_t team_of(int64_t row, int64_t rows, int64_t teams) {
  return ((row + 1) * teams - 1) / rows;
}

// Shared memory of a CTA: its share of the SM's, for the ring of row stages (as many as fit, 8 at
// most) and `vectors` FP32 values per column behind it.
constexpr int kSharedBytes = 224 * 1024;
constexpr int kMaxStages = 8;
inline int ring_stages(const Geometry& g, int threads_per_sm, int stage_bytes, int vectors,
                       int rows_per_team) {
  const int per_sm = std::max(1, threads_per_sm / g.threads);
  // (a CTA's static shared memory and its reservation besides, where several share an SM)
  const int share = kSharedBytes / per_sm - (per_sm > 1 ? 1792 : 0) - vectors * 64 * g.threads;
  return std::max(1, std::min({share / stage_bytes, kMaxStages, rows_per_team}));
}

}  // namespace norm_detail

inline int64_t block_norm_backward_workspace_bytes(int rows, int H, int has_gate, int gate_rows) {
  if (rows < 1 || rows > kNormMaxRows || H < 8 || H > kNormMaxH || H % 8 != 0 || gate_rows < 0) return -1;
  const int64_t teams = norm_detail::row_teams(rows, norm_detail::geometry(H), norm_detail::kThreadsPerSm);
  const int64_t vectors = 4 + ((has_gate && gate_rows != 1) ? 2 : 0);
  return teams * vectors * H * 4;
}

inline cudaError_t block_norm_check(const blackhole_sm100_block_norm_args& a) {
  if (a.rows < 1 || a.rows > kNormMaxRows || a.H < 8 || a.H > kNormMaxH || a.H % 8 != 0) return cudaErrorInvalidValue;
  if (a.kind < 0 || a.kind > 1 || a.gate_rows < 0) return cudaErrorInvalidValue;
  if (!(a.eps >= 0.0f) || !std::isfinite(a.eps) || !std::isfinite(a.scale))
    return cudaErrorInvalidValue;
  if (a.out_format < kOutBf16 || a.out_format > kOutMxfp8) return cudaErrorInvalidValue;
  if (!a.x || (!a.out && !a.h)) return cudaErrorInvalidValue;
  // without a block result there is nothing to gate, to norm or to add
  if (!a.o && (a.gate || a.post_norm || a.h)) return cudaErrorInvalidValue;
  if (!a.post_norm && (a.post_weight || a.post_bias)) return cudaErrorInvalidValue;
  if (!a.out && (a.weight || a.bias || a.sf)) return cudaErrorInvalidValue;
  const bool quant = a.out && a.out_format >= kOutNvfp4;
  if (quant != (a.sf != nullptr)) return cudaErrorInvalidValue;
  if (quant && a.H % (a.out_format == kOutNvfp4 ? 16 : 32) != 0) return cudaErrorInvalidValue;
  if (quant && a.out_format == kOutNvfp4 && (!(a.global_scale > 0.0f) || !std::isfinite(a.global_scale)))
    return cudaErrorInvalidValue;
  const void* ptrs[] = {a.x, a.o, a.gate, a.weight, a.bias, a.post_weight, a.post_bias,
                        a.h, a.out, a.sf, a.stats};
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) & 15u) return cudaErrorInvalidValue;
  const int64_t n = int64_t(a.rows) * a.H;
  const int64_t xb = n * (a.x_is_bf16 ? 2 : 4);
  const int64_t yb = a.out_format == kOutBf16 ? n * 2 : a.out_format == kOutF32 ? n * 4
                     : a.out_format == kOutMxfp8 ? n : n / 2;
  if (a.h && a.h != a.x && detail::ranges_overlap(a.h, xb, a.x, xb)) return cudaErrorInvalidValue;
  if (detail::ranges_overlap(a.h, xb, a.o, n * 2) || detail::ranges_overlap(a.h, xb, a.out, yb) ||
      detail::ranges_overlap(a.out, yb, a.x, xb) || detail::ranges_overlap(a.out, yb, a.o, n * 2))
    return cudaErrorInvalidValue;
  return cudaSuccess;
}

inline cudaError_t block_norm_backward_check(const blackhole_sm100_block_norm_backward_args& a) {
  if (a.rows < 1 || a.rows > kNormMaxRows || a.H < 8 || a.H > kNormMaxH || a.H % 8 != 0) return cudaErrorInvalidValue;
  if (a.kind < 0 || a.kind > 1 || a.gate_rows < 0 || !std::isfinite(a.scale))
    return cudaErrorInvalidValue;
  if (!a.h || !a.stats || !a.dx || (!a.dy && !a.dh)) return cudaErrorInvalidValue;
  if (!a.o && (a.gate || a.post_norm || a.d_o || a.dgate)) return cudaErrorInvalidValue;
  if (a.o && !a.d_o) return cudaErrorInvalidValue;
  if (!a.post_norm && (a.post_weight || a.post_bias || a.dpost_weight || a.dpost_bias))
    return cudaErrorInvalidValue;
  if (!a.gate && a.dgate) return cudaErrorInvalidValue;
  const void* ptrs[] = {a.h, a.stats, a.dy, a.dh, a.o, a.gate, a.weight, a.post_weight,
                        a.post_bias, a.dx, a.d_o, a.dweight, a.dbias, a.dpost_weight,
                        a.dpost_bias, a.dgate, a.workspace};
  for (const void* q : ptrs)
    if (reinterpret_cast<uintptr_t>(q) & 15u) return cudaErrorInvalidValue;
  const bool sums = a.dweight || a.dbias || a.dpost_weight || a.dpost_bias ||
                    (a.dgate && a.gate_rows != 1);
  if (sums) {
    const int64_t need = block_norm_backward_workspace_bytes(a.rows, a.H, a.gate != nullptr, a.gate_rows);
    if (!a.workspace || a.workspace_bytes < need) return cudaErrorInvalidValue;
  }
  const int64_t n = int64_t(a.rows) * a.H;
  const int64_t xb = n * (a.x_is_bf16 ? 2 : 4);
  if (a.dx != a.dh && detail::ranges_overlap(a.dx, xb, a.dh, xb)) return cudaErrorInvalidValue;
  if (detail::ranges_overlap(a.dx, xb, a.h, xb) || detail::ranges_overlap(a.dx, xb, a.dy, n * 2) ||
      detail::ranges_overlap(a.dx, xb, a.o, n * 2) || detail::ranges_overlap(a.dx, xb, a.d_o, n * 2) ||
      detail::ranges_overlap(a.d_o, n * 2, a.h, xb) || detail::ranges_overlap(a.d_o, n * 2, a.dh, xb) ||
      detail::ranges_overlap(a.d_o, n * 2, a.dy, n * 2) || detail::ranges_overlap(a.d_o, n * 2, a.o, n * 2))
    return cudaErrorInvalidValue;
  return cudaSuccess;
}

#if defined(__CUDACC__)

namespace norm_detail {

// 8 values of a vector of parameters or gates, BF16 or FP32 (uniform over the launch).
__device__ __forceinline__ void load8_any(const void* p, int64_t at, int is_bf16, float (&v)[8]) {
  if (is_bf16) {
    const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + at);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 a = q[0], b = q[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Pair arithmetic (f32x2.hpp): these kernels were bound by instruction issue before.
using detail::add2;
using detail::both;
using detail::fma2;
using detail::mul2;
using detail::unpack2;

// A thread's 16 columns of a row, as 8 pairs: pairs 0-3 its first 8-column vector, 4-7 its second.
using Row16 = float2[8];

// 8 values at element `at` of a row in shared memory.
template <class T>
__device__ __forceinline__ void shared8(uint32_t row, int at, float2* v) {
  if constexpr (sizeof(T) == 2) {
    const uint4 q = ptx::ld_shared_v4(row + 2 * at);
    v[0] = unpack2(q.x); v[1] = unpack2(q.y); v[2] = unpack2(q.z); v[3] = unpack2(q.w);
  } else {
    const uint4 a = ptx::ld_shared_v4(row + 4 * at), b = ptx::ld_shared_v4(row + 4 * at + 16);
    v[0] = make_float2(__uint_as_float(a.x), __uint_as_float(a.y));
    v[1] = make_float2(__uint_as_float(a.z), __uint_as_float(a.w));
    v[2] = make_float2(__uint_as_float(b.x), __uint_as_float(b.y));
    v[3] = make_float2(__uint_as_float(b.z), __uint_as_float(b.w));
  }
}

// Exchange of one pair of values per warp across a row's CTA or cluster.  Two slot sets in turn: a
// set is written again only after a later barrier that every reader of it has passed.
template <int kCl>
struct RowExchange {
  static constexpr int kWarps = kCl * 16;
  float (*slots)[2][kWarps];      // [2][2][CTA * 16 + warp], zeroed before first use
  const float* counts;            // [CTA * 16 + warp]: columns of the row that the warp holds
  int set = 0;

  __device__ __forceinline__ void put(float a, float b) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if constexpr (kCl == 1) {
      if (lane == 0) {
        slots[set][0][warp] = a;
        slots[set][1][warp] = b;
      }
      __syncthreads();
    } else {
      const uint32_t rank = ptx::cluster_ctarank();
      if (lane < kCl) {
        const float v[2] = {a, b};
#pragma unroll
        for (int k = 0; k < 2; ++k)
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(ptx::mapa_shared(
                           ptx::smem_u32(&slots[set][k][rank * 16 + warp]), uint32_t(lane))),
                       "f"(v[k])
                       : "memory");
      }
      ptx::cluster_sync();
    }
  }
  __device__ __forceinline__ float total(int k) const {
    const float4* q = reinterpret_cast<const float4*>(slots[set][k]);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kWarps / 4; ++i) {
      const float4 t = q[i];
      s = add2(s, add2(make_float2(t.x, t.y), make_float2(t.z, t.w)));
    }
    return s.x + s.y;
  }
  // Sums over the row, the same in every thread, added in a fixed order.  A barrier of the CTA or
  // cluster, unless the CTA is one warp.
  __device__ __forceinline__ float sum(float2 v) {
    const float a = warp_sum(v.x + v.y);
    if (kCl == 1 && blockDim.x == 32) return a;
    put(a, 0.f);
    const float s = total(0);
    set ^= 1;
    return s;
  }
  __device__ __forceinline__ void sum2(float2 va, float2 vb, float& a, float& b) {
    a = warp_sum(va.x + va.y);
    b = warp_sum(vb.x + vb.y);
    if (kCl == 1 && blockDim.x == 32) return;
    put(a, b);
    a = total(0);
    b = total(1);
    set ^= 1;
  }
  // Mean and sum of squares about it of the row's values (0 past its end): each warp's own mean
  // and squares about that first, then merged, so nothing cancels however far the mean is from
  // zero, and one barrier is enough.
  __device__ __forceinline__ void mean_squares(const Row16& v, const bool (&live)[2], float inv_h,
                                               float& mean, float& squares) {
    const int me = (kCl == 1 ? 0 : int(ptx::cluster_ctarank())) * 16 + (threadIdx.x >> 5);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) s = add2(s, v[i]);
    const float n = counts[me];
    float mw, m2;
    if (n == 512.f) {
      // a full warp: every thread's own mean and squares, merged in pairs (equal counts)
      mw = (s.x + s.y) * 0.0625f;
      float2 q2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 d = add2(v[i], both(-mw));
        q2 = fma2(d, d, q2);
      }
      m2 = q2.x + q2.y;
      float half = 8.f;                                 // half the count of either side
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float mo = __shfl_xor_sync(0xFFFFFFFFu, mw, o), qo = __shfl_xor_sync(0xFFFFFFFFu, m2, o);
        const float d = mo - mw;
        m2 = fmaf(d * d, half, m2 + qo);
        mw = 0.5f * (mw + mo);
        half *= 2.f;
      }
    } else {
      mw = n > 0.f ? warp_sum(s.x + s.y) / n : 0.f;
      float2 q2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 d = add2(v[i], both(-mw));
        q2[i / 4] = fma2(d, d, q2[i / 4]);
      }
      m2 = warp_sum((live[0] ? q2[0].x + q2[0].y : 0.f) + (live[1] ? q2[1].x + q2[1].y : 0.f));
    }
    if (kCl == 1 && blockDim.x == 32) {
      mean = mw;
      squares = m2;
      return;
    }
    put(mw, m2);
    // one warp's values per lane, merged by butterflies (the same in every lane; half the
    // shared-memory traffic of every thread reading them all)
    const int at = threadIdx.x & (kWarps - 1);
    const float m = slots[set][0][at], c = counts[at];
    float t = c * m, q = slots[set][1][at];
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
    mean = t * inv_h;
    const float d = m - mean;
    q = fmaf(c * d, d, q);
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) q += __shfl_xor_sync(0xFFFFFFFFu, q, o);
    squares = q;
    set ^= 1;
  }
};

template <class T>
__device__ __forceinline__ void store8(T* p, const float2* v) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(detail::pack_bf16x2(v[0].x, v[0].y), detail::pack_bf16x2(v[1].x, v[1].y),
                   detail::pack_bf16x2(v[2].x, v[2].y), detail::pack_bf16x2(v[3].x, v[3].y));
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
  }
}

// Shared memory of a CTA: the ring's stages first (dynamic), then this.
template <int kCl>
struct __align__(16) RowShared {
  float slots[2][2][kCl * 16];
  float counts[kCl * 16];
  uint64_t bars[kMaxStages];
  int abort_flag;
};

// This thread's columns and the CTA's set-up, the same in both directions.
template <int kCl>
struct RowTeam {
  int rank, team, col[2];
  bool live[2];
  int row0, row1;
  int c0, cols, width;           // the CTA's columns of a row; a stage row's, 16 per thread
  uint32_t ring, bars;
  volatile int* abort_flag;

  __device__ __forceinline__ RowTeam(RowShared<kCl>& sh, uint8_t* ring_ptr, int H, int slice, int rows,
                                     int teams, int stages, uint32_t ring_bytes) {
    rank = kCl == 1 ? 0 : static_cast<int>(ptx::cluster_ctarank());
    team = blockIdx.x / kCl;
    const int T = blockDim.x, tid = threadIdx.x;
    c0 = rank * slice;
    const int c1 = min(H, c0 + slice);
    cols = c1 - c0;
    width = 16 * T;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      col[v] = c0 + (v * T + tid) * 8;
      live[v] = col[v] < c1;
    }
    row0 = static_cast<int>(row_begin(team, rows, teams));
    row1 = static_cast<int>(row_begin(team + 1, rows, teams));
    ring = ptx::smem_u32(ring_ptr);
    bars = ptx::smem_u32(sh.bars);
    abort_flag = &sh.abort_flag;
    for (int i = tid; i < 4 * kCl * 16; i += T) (&sh.slots[0][0][0])[i] = 0.f;
    for (int i = tid; i < kCl * 16; i += T) {       // columns of warp i % 16 of CTA i / 16
      const int b = (i / 16) * slice, e = min(H, b + slice);
      int n = 0;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int from = b + (v * T + (i % 16) * 32) * 8;
        if ((i % 16) * 32 < T) n += max(0, min(e, from + 256) - from);
      }
      sh.counts[i] = static_cast<float>(n);
    }
    // columns past the row's end read as 0: no copy writes there
    if (cols != width)
      for (uint32_t i = 16 * tid; i < ring_bytes; i += 16 * T) ptx::st_shared_v4(ring + i, 0, 0, 0, 0);
    if (tid == 0) {
      for (int s = 0; s < stages; ++s) ptx::mbar_init(bars + 8u * s, 1);
      sh.abort_flag = 0;
      ptx::fence_mbar_init();
      ptx::fence_proxy_async_smem();
    }
    if constexpr (kCl == 1) __syncthreads();
    else ptx::cluster_sync();
  }
  // A stage's rows have arrived (bounded like every wait: a copy that never lands sets the status
  // word, and the kernel runs to its end).
  __device__ __forceinline__ void wait(int stage, uint32_t phase) {
    (void)ptx::wait_bounded(bars + 8u * stage, phase, abort_flag, &detail::g_status, kStatusLoadTimeout);
  }
  // This thread's 16 values of a row in shared memory, 0 past its end.
  template <class T>
  __device__ __forceinline__ void read16(uint32_t row, Row16& v) const {
    shared8<T>(row, threadIdx.x * 8, v);
    shared8<T>(row, (blockDim.x + threadIdx.x) * 8, v + 4);
  }
  template <class T>
  __device__ __forceinline__ void write16(T* row, const Row16& v) const {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (live[k]) store8(row + col[k], v + 4 * k);
  }
  // Every thread of the CTA has read the stage.
  __device__ __forceinline__ void release_barrier() const { __syncthreads(); }
};

// This thread's 16 values of a parameter vector (BF16 or FP32): `none` where it is absent, 0 past
// the row's end.
__device__ __forceinline__ void vector16(const void* p, int64_t at, int is_bf16, const int (&col)[2],
                                         const bool (&live)[2], float none, Row16& out) {
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = live[v] ? none : 0.f;
    if (p && live[v]) load8_any(p, at + col[v], is_bf16, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[4 * v + i] = make_float2(t[2 * i], t[2 * i + 1]);
  }
}

// FP32 vectors in shared memory of which every thread keeps and reads its own 16 values only, as
// four 16-byte quarters a thread stride apart (no bank conflicts).
struct OwnVectors {
  uint8_t* base;
  __device__ __forceinline__ float4* at(int k) const {
    return reinterpret_cast<float4*>(base) + (k * 4) * blockDim.x + threadIdx.x;
  }
  __device__ __forceinline__ void put(int k, const Row16& v) const {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      at(k)[q * blockDim.x] = make_float4(v[2 * q].x, v[2 * q].y, v[2 * q + 1].x, v[2 * q + 1].y);
  }
  __device__ __forceinline__ void get(int k, Row16& v) const {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 t = at(k)[q * blockDim.x];
      v[2 * q] = make_float2(t.x, t.y);
      v[2 * q + 1] = make_float2(t.z, t.w);
    }
  }
};

// What a kernel is built for: RMS norms, RMS norms with a bias (or its gradient) somewhere, layer
// norms.
enum NormMode : int { kRms = 0, kRmsBias = 1, kLayerNorm = 2 };

// E2M1 codes of eight values (round to nearest even, finite values past 6 saturate; NaN as 6, the
// conversion of nvfp4_quant.hpp's e2m1_rne), the first in the lowest nibble.
__device__ __forceinline__ uint32_t e2m1x8(const float2 (&v)[4]) {
  return quant_detail::e2m1x4_cvt(v[0].x, v[0].y, v[1].x, v[1].y) |
         (quant_detail::e2m1x4_cvt(v[2].x, v[2].y, v[3].x, v[3].y) << 16);
}
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
  float d;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

struct NormParams {
  const void *x, *o, *gate, *weight, *bias, *post_weight, *post_bias;
  void *h, *out;
  uint8_t* sf;
  float* stats;
  int rows, H, slice, teams, stages;
  int keep_cw;          // gate, scale and post weight kept as one vector
  int gate_rows, param_bf16, gate_bf16, out_format;
  float scale, eps, global_scale;
};

// Quantisation of a row's 16 columns of this thread, two 8-column vectors; neighbouring lanes hold
// the other columns of a vector's 16- or 32-column block, and the codes of a word's four scale
// factors are on 8 (NVFP4) or 16 (MX) neighbouring lanes.  Every lane of the warp takes part (past
// the row's end all zero).  Recipes and roundings are those of nvfp4_quant.hpp.
__device__ __forceinline__ float max_abs8(const float2* y) {
  float m = max_abs3(max_abs3(max_abs3(y[0].x, y[0].y, y[1].x), y[1].y, y[2].x), y[2].y, y[3].x);
  return max_abs3(m, y[3].y, 0.f);
}

// NVFP4: the scale factor's code; writes the 8 codes.
__device__ __forceinline__ uint32_t quantize8_nvfp4(const float2* y, float m, bool live, float g, float c,
                                                    uint8_t* out, int col) {
  uint32_t q = 0, code = 0;
  if (live && m > 0.f) {
    // as in quantize_kernel: estimates, and exact quotients only next to a rounding threshold
    const float ys = m * c;
    code = quant_detail::ue4m3_cvt(quant_detail::near_ue4m3_threshold(ys) ? (m / 6.0f) / g : ys);
    const float s = quant_detail::ue4m3_value(code);
    if (s != 0.f) {
      const float scale = s * g;
      const float rs = quant_detail::rcp_approx(scale);
      float2 v[4];
      bool near = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = mul2(y[i], both(rs));
        near |= quant_detail::near_e2m1_threshold(v[i].x) || quant_detail::near_e2m1_threshold(v[i].y);
      }
      if (near) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = make_float2(y[i].x / scale, y[i].y / scale);
      }
      q = e2m1x8(v);
    }
  }
  if (live) *reinterpret_cast<uint32_t*>(out + col / 2) = q;
  return code;
}

// MX: the shared exponent comes from the block maximum's exponent bits; writes the 8 codes.
template <int kFmt>
__device__ __forceinline__ uint32_t quantize8_mx(const float2* y, uint32_t ebits, bool live, uint8_t* out,
                                                 int col) {
  // exponent floor(log2 amax) - emax, at least -127 (at most 126 here)
  const int e = max(-127, static_cast<int>(ebits) - (kFmt == kOutMxfp8 ? 135 : 129));
  const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  float2 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = mul2(y[i], both(inv));
  if constexpr (kFmt == kOutMxfp4) {
    const uint32_t q = e2m1x8(v);
    if (live) *reinterpret_cast<uint32_t*>(out + col / 2) = q;
  } else {
    const uint32_t lo = quant_detail::e4m3x2_satfinite(v[0].x, v[0].y) | (quant_detail::e4m3x2_satfinite(v[1].x, v[1].y) << 16);
    const uint32_t hi = quant_detail::e4m3x2_satfinite(v[2].x, v[2].y) | (quant_detail::e4m3x2_satfinite(v[3].x, v[3].y) << 16);
    if (live) *reinterpret_cast<uint2*>(out + col) = make_uint2(lo, hi);
  }
  return live ? static_cast<uint32_t>(e + 127) : 0u;
}

template <int kFmt, class Team>
__device__ __forceinline__ void quantize_row(const Row16& y, const Team& t, float g, float c, void* out,
                                             uint8_t* sf, int64_t r, int H) {
  constexpr int kVec = kFmt == kOutNvfp4 ? 16 : 32, kPer = kVec / 8, kLanes = 4 * kPer;
  const int lane = threadIdx.x & 31, ri = static_cast<int>(r);
  uint8_t* const row = static_cast<uint8_t*>(out) + (kFmt == kOutMxfp8 ? r * H : r * H / 2);
  uint8_t* const sf_row = sf + int64_t(ri >> 7) * ((H / kVec + 3) / 4) * 512 + (ri & 31) * 16 + ((ri >> 5) & 3) * 4;
  uint32_t code[2];
  if constexpr (kFmt == kOutNvfp4) {
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      float m = max_abs8(y + 4 * v);
      m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
      code[v] = quantize8_nvfp4(y + 4 * v, m, t.live[v], g, c, row, t.col[v]);
    }
  } else {
    // both vectors' exponents as two 16-bit halves of one word through the shuffles
    uint32_t e = (__float_as_uint(max_abs8(y)) >> 23) | (__float_as_uint(max_abs8(y + 4)) >> 23 << 16);
    e = __vmaxu2(e, __shfl_xor_sync(0xFFFFFFFFu, e, 1));
    e = __vmaxu2(e, __shfl_xor_sync(0xFFFFFFFFu, e, 2));
    code[0] = quantize8_mx<kFmt>(y, e & 0xFFFFu, t.live[0], row, t.col[0]);
    code[1] = quantize8_mx<kFmt>(y + 4, e >> 16, t.live[1], row, t.col[1]);
  }
  // bytes of four groups, kPer lanes apart, to the first lane of each kLanes: one byte pair per
  // vector after the first exchange, both words after the second
  const uint32_t own = code[0] | (code[1] << 16);
  const uint32_t two = own | (__shfl_xor_sync(0xFFFFFFFFu, own, kPer) << 8);
  const uint32_t four = __shfl_xor_sync(0xFFFFFFFFu, two, 2 * kPer);
  if (lane % kLanes == 0) {
    if (t.live[0])
      *reinterpret_cast<uint32_t*>(sf_row + (t.col[0] / (4 * kVec)) * 512) = (two & 0xFFFFu) | (four << 16);
    if (t.live[1])
      *reinterpret_cast<uint32_t*>(sf_row + (t.col[1] / (4 * kVec)) * 512) = (two >> 16) | (four & 0xFFFF0000u);
  }
}

// Forward.  kPost and p.o select what a row's p is made of; the gate row, the scale and the post
// weight are one vector `cw` (and with the post bias `cb`), made anew only where the gate row
// changes.  RMS norms keep their two vectors in registers.  With biases there are up to four: those
// kernels keep them as FP32 in shared memory, each thread its own columns (no barrier between),
// behind a ring of fewer stages: layer norm of 9472 x 8192, FP32 stream, post norm, 218 us.  (In
// registers they spilled, 270 us; from L1 for every row they did not fit, 259 us, against 241 then.)
//
// kThreads: 512 (128 registers), or for rows of at most 5120 columns 320, built for 96 registers so
// that two CTAs of 320 threads share an SM (layer norm of 9472 x 5120, BF16 stream:
// 95 -> 71 us; one CTA's 10 warps left most issue slots empty).
template <class TX, int kMode, bool kPost, int kCl, int kThreads>
__global__ void __cluster_dims__(kCl, 1, 1) __launch_bounds__(kThreads, kThreads == kNarrowThreads ? 2 : 1)
    block_norm_kernel(const __grid_constant__ NormParams p) {
#if defined(BLACKHOLE_ARCH_SM100)
  constexpr bool kLayer = kMode == kLayerNorm, kBias = kMode != kRms;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ RowShared<kCl> sh;
  ptx::pdl_launch_dependents();
  const uint32_t x_row = uint32_t(blockDim.x) * 16 * sizeof(TX);
  const uint32_t stage_bytes = x_row + (p.o ? uint32_t(blockDim.x) * 32 : 0);
  RowTeam<kCl> t(sh, ring, p.H, p.slice, p.rows, p.teams, p.stages, p.stages * stage_bytes);
  RowExchange<kCl> row{sh.slots, sh.counts};
  const int tid = threadIdx.x, H = p.H;
  const uint32_t x_bytes = uint32_t(t.cols) * sizeof(TX), o_bytes = p.o ? uint32_t(t.cols) * 2 : 0;
  ptx::pdl_wait_prior_grid();

  const uint64_t policy = ptx::l2_policy_evict_first();   // every row is read once
  auto fetch = [&](int r, int stage) {
    const uint32_t bar = t.bars + 8u * stage, dst = t.ring + stage * stage_bytes;
    const int64_t at = int64_t(r) * H + t.c0;
    ptx::mbar_arrive_expect_tx(bar, x_bytes + o_bytes);
    if (o_bytes) ptx::bulk_load(dst + x_row, static_cast<const __nv_bfloat16*>(p.o) + at, o_bytes, bar, policy);
    ptx::bulk_load(dst, static_cast<const TX*>(p.x) + at, x_bytes, bar, policy);
  };
  if (tid == 0)
    for (int i = 0; i < p.stages && t.row0 + i < t.row1; ++i) fetch(t.row0 + i, i);

  Row16 w, cw;
  OwnVectors own{ring + p.stages * stage_bytes};      // (kBias) 0: weight, 1: bias, 2: cw, 3: cb
  vector16(p.weight, 0, p.param_bf16, t.col, t.live, 1.f, w);
  if constexpr (kBias) {
    own.put(0, w);
    vector16(p.bias, 0, p.param_bf16, t.col, t.live, 0.f, w);
    own.put(1, w);
  }
  const float quant_c = __frcp_rn(6.0f) * __frcp_rn(p.global_scale);    // quantize_kernel's estimate
  int gate_row = -1;
  const float inv_h = 1.0f / static_cast<float>(H);
  int stage = 0;
  uint32_t phase = 0;
  for (int r = t.row0; r < t.row1; ++r) {
    const int64_t at = int64_t(r) * H;
    const int g = p.gate_rows ? r / p.gate_rows : 0;
    if (p.o && (!kBias || p.keep_cw) && g != gate_row) {
      gate_row = g;
      vector16(p.gate, int64_t(g) * H, p.gate_bf16, t.col, t.live, 1.f, cw);
#pragma unroll
      for (int i = 0; i < 8; ++i) cw[i] = mul2(cw[i], both(p.scale));
      if constexpr (kPost) {
        Row16 v;
        if constexpr (kBias) {
          vector16(p.post_bias, 0, p.param_bf16, t.col, t.live, 0.f, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = mul2(cw[i], v[i]);
          own.put(3, v);
        }
        vector16(p.post_weight, 0, p.param_bf16, t.col, t.live, 1.f, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) cw[i] = mul2(cw[i], v[i]);
      }
      if (kBias && p.keep_cw) own.put(2, cw);
    }
    const uint32_t xs = t.ring + stage * stage_bytes;
    t.wait(stage, phase);
    Row16 h;
    float mean_post = 0.f, rstd_post = 0.f;
    if (p.o) {
      Row16 o;
      t.template read16<__nv_bfloat16>(xs + x_row, o);
      if constexpr (kPost) {
        float q;
        if constexpr (kLayer) {
          row.mean_squares(o, t.live, inv_h, mean_post, q);
        } else {
          float2 s = make_float2(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < 8; ++i) s = fma2(o[i], o[i], s);
          q = row.sum(s);
        }
        rstd_post = rsqrtf(fmaf(q, inv_h, p.eps));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (kLayer) o[i] = add2(o[i], both(-mean_post));
          o[i] = mul2(o[i], both(rstd_post));
        }
      }
      t.template read16<TX>(xs, h);
      if constexpr (kBias) {
        if (p.keep_cw) {
          own.get(2, cw);
        } else {                         // (no post norm: the gate row itself, from L1)
          vector16(p.gate, int64_t(g) * H, p.gate_bf16, t.col, t.live, 1.f, cw);
#pragma unroll
          for (int i = 0; i < 8; ++i) cw[i] = mul2(cw[i], both(p.scale));
        }
        if constexpr (kPost) {
          own.get(3, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) h[i] = add2(h[i], w[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = fma2(o[i], cw[i], h[i]);
      if (p.h) t.write16(static_cast<TX*>(p.h) + at, h);
    } else {
      t.template read16<TX>(xs, h);
    }
    float mean = 0.f, q = 0.f;
    if (p.out || p.stats) {
      if constexpr (kLayer) {
        row.mean_squares(h, t.live, inv_h, mean, q);
      } else {
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fma2(h[i], h[i], s);
        q = row.sum(s);
      }
      if (blockDim.x == 32) __syncwarp();
    } else {
      t.release_barrier();
    }
    // past that barrier every thread has read the stage
    if (tid == 0 && r + p.stages < t.row1) fetch(r + p.stages, stage);
    const float rstd = rsqrtf(fmaf(q, inv_h, p.eps));
    if (p.stats && t.rank == 0 && tid == 0)
      reinterpret_cast<float4*>(p.stats)[r] = make_float4(mean_post, rstd_post, mean, rstd);
    if (p.out) {
      if constexpr (kBias) own.get(0, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (kLayer) h[i] = add2(h[i], both(-mean));
        h[i] = mul2(mul2(h[i], both(rstd)), w[i]);
      }
      if constexpr (kBias) {
        own.get(1, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = add2(h[i], w[i]);
      }
      switch (p.out_format) {
        case kOutBf16: t.write16(static_cast<__nv_bfloat16*>(p.out) + at, h); break;
        case kOutF32: t.write16(static_cast<float*>(p.out) + at, h); break;
        case kOutNvfp4: quantize_row<kOutNvfp4>(h, t, p.global_scale, quant_c, p.out, p.sf, r, H); break;
        case kOutMxfp4: quantize_row<kOutMxfp4>(h, t, 1.f, 1.f, p.out, p.sf, r, H); break;
        default: quantize_row<kOutMxfp8>(h, t, 1.f, 1.f, p.out, p.sf, r, H); break;
      }
    }
    if (++stage == p.stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  // scale factors of the layout's padding rows
  if (p.out && p.sf && t.rank == 0) {
    const int vs = p.out_format == kOutNvfp4 ? 16 : 32;
    const int words = static_cast<int>(sf_k_atoms_vs(H, vs));
    const int pad = (p.rows + 127) / 128 * 128 - p.rows;
    for (int64_t i = int64_t(t.team) * blockDim.x + tid; i < int64_t(pad) * words;
         i += int64_t(p.teams) * blockDim.x)
      *reinterpret_cast<uint32_t*>(
          p.sf + sf_offset_vs(p.rows + int64_t(i / words), 4 * (i % words), H, vs)) = 0u;
  }
  if constexpr (kCl > 1) ptx::cluster_sync();   // no CTA leaves while its partner writes its slots
#endif
}

struct NormBackwardParams {
  const void *h, *dy, *dh, *o, *gate, *weight, *post_weight, *post_bias;
  const float* stats;
  void *dx, *d_o;
  float *dweight, *dbias, *dpost_weight, *dpost_bias, *dgate;
  float* ws;            // [vector][team][H]: dweight, dbias, dpost_weight, dpost_bias, gate edges
  int rows, H, slice, teams, stages;
  int gate_rows, groups, param_bf16, gate_bf16;
  float scale;
};

// Backward.  With n the post-normed o (o itself without a post norm) and d = dh', a gate row's
// sums A = sum d n and B = sum d give every gradient that the gate takes part in:
//     dgate = scale (post_weight A + post_bias B),  dpost_weight = scale gate A, dpost_bias = scale gate B
// so a thread keeps dweight, A (and where there are biases dbias, B) for its 16 columns, and gate,
// scale and post weight are one vector c.  Over a row sum it keeps n and dh + rstd a, not a itself:
// dh' = (dh + rstd a) - rstd [mean a] - rstd mean(a n) n.  kGate: 0 no gate, 1 one gate row (sums
// closed once, at the end), 2 several (closed at each group's last row).
template <class TX, int kMode, bool kPost, int kGate, int kCl>
__global__ void __cluster_dims__(kCl, 1, 1) __launch_bounds__(512, 1)
    block_norm_backward_kernel(const __grid_constant__ NormBackwardParams p) {
#if defined(BLACKHOLE_ARCH_SM100)
  constexpr bool kLayer = kMode == kLayerNorm, kBias = kMode != kRms;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ RowShared<kCl> sh;
  ptx::pdl_launch_dependents();
  // a stage: h and dh (TX), dy and o (BF16), those that are given
  const uint32_t xs = uint32_t(blockDim.x) * 16 * sizeof(TX), ys = uint32_t(blockDim.x) * 32;
  const uint32_t at_dh = p.dy ? xs : 0, at_dy = at_dh + (p.dh ? xs : 0), at_o = at_dy + (p.dy ? ys : 0);
  const uint32_t stage_bytes = at_o + (p.o ? ys : 0);
  RowTeam<kCl> t(sh, ring, p.H, p.slice, p.rows, p.teams, p.stages, p.stages * stage_bytes);
  RowExchange<kCl> row{sh.slots, sh.counts};
  const int tid = threadIdx.x, H = p.H;
  const uint32_t xb = uint32_t(t.cols) * sizeof(TX), yb = uint32_t(t.cols) * 2;
  const uint32_t row_bytes = (p.dy ? xb + yb : 0) + (p.dh ? xb : 0) + (p.o ? yb : 0);
  ptx::pdl_wait_prior_grid();

  const uint64_t policy = ptx::l2_policy_evict_first();
  auto fetch = [&](int r, int stage) {
    const uint32_t bar = t.bars + 8u * stage, dst = t.ring + stage * stage_bytes;
    const int64_t at = int64_t(r) * H + t.c0;
    ptx::mbar_arrive_expect_tx(bar, row_bytes);
    if (p.dy) {
      ptx::bulk_load(dst, static_cast<const TX*>(p.h) + at, xb, bar, policy);
      ptx::bulk_load(dst + at_dy, static_cast<const __nv_bfloat16*>(p.dy) + at, yb, bar, policy);
    }
    if (p.dh) ptx::bulk_load(dst + at_dh, static_cast<const TX*>(p.dh) + at, xb, bar, policy);
    if (p.o) ptx::bulk_load(dst + at_o, static_cast<const __nv_bfloat16*>(p.o) + at, yb, bar, policy);
  };
  if (tid == 0)
    for (int i = 0; i < p.stages && t.row0 + i < t.row1; ++i) fetch(t.row0 + i, i);

  // where biases' sums leave no registers for the vectors, they are kept in shared memory
  constexpr bool kKeep = !kBias || !kPost;
  OwnVectors own{ring + p.stages * stage_bytes};      // (!kKeep) 0: weight, 1: c
  const float2 zero = make_float2(0.f, 0.f);
  Row16 w, c;
  auto make_c = [&](int g, Row16& out) {
    vector16(kGate ? p.gate : nullptr, int64_t(g) * H, p.gate_bf16, t.col, t.live, 1.f, out);
    Row16 v;
    if (kPost) vector16(p.post_weight, 0, p.param_bf16, t.col, t.live, 1.f, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = mul2(out[i], kPost ? mul2(v[i], both(p.scale)) : both(p.scale));
  };
  vector16(p.weight, 0, p.param_bf16, t.col, t.live, 1.f, w);
  if constexpr (!kKeep) own.put(0, w);
  Row16 dw, db, sa, sb, dwp, dbp;
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[i] = db[i] = sa[i] = sb[i] = dwp[i] = dbp[i] = zero;
  const int64_t vec = int64_t(p.teams) * H;           // floats of one vector's partials
  // dgate of a gate row (or a team's piece of it) from A and B
  auto write_dgate = [&](float* dst) {
    Row16 v, u;
    vector16(kPost ? p.post_weight : nullptr, 0, p.param_bf16, t.col, t.live, 1.f, v);
    if (kPost && kBias) vector16(p.post_bias, 0, p.param_bf16, t.col, t.live, 0.f, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = mul2(v[i], sa[i]);
      if constexpr (kPost && kBias) v[i] = fma2(u[i], sb[i], v[i]);
      v[i] = mul2(v[i], both(p.scale));
    }
    t.write16(dst, v);
  };
  const float inv_h = 1.0f / static_cast<float>(H);
  int gate_row = -1;
  int stage = 0;
  uint32_t phase = 0;
  for (int r = t.row0; r < t.row1; ++r) {
    const int64_t at = int64_t(r) * H;
    const int g = kGate == 2 ? r / p.gate_rows : 0;
    if (p.o && g != gate_row) {
      gate_row = g;
      make_c(g, c);
      if constexpr (!kKeep) own.put(1, c);
    }
    const float4 st = reinterpret_cast<const float4*>(p.stats)[r];
    const uint32_t base = t.ring + stage * stage_bytes;
    t.wait(stage, phase);
    Row16 d;                                          // dh'
    if (p.dh) {
      t.template read16<TX>(base + at_dh, d);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = zero;
    }
    if (p.dy) {
      Row16 n, a;
      t.template read16<TX>(base, n);
      t.template read16<__nv_bfloat16>(base + at_dy, a);
      if constexpr (!kKeep) own.get(0, w);
      float2 s = zero, sm = zero;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (kLayer) n[i] = add2(n[i], both(-st.z));
        n[i] = mul2(n[i], both(st.w));
        dw[i] = fma2(a[i], n[i], dw[i]);
        if constexpr (kBias) db[i] = add2(db[i], a[i]);
        a[i] = mul2(a[i], w[i]);
        s = fma2(a[i], n[i], s);
        if constexpr (kLayer) sm = add2(sm, a[i]);
        d[i] = fma2(a[i], both(st.w), d[i]);
      }
      float along, mean_a = 0.f;
      if constexpr (kLayer) row.sum2(s, sm, along, mean_a);
      else along = row.sum(s);
      const float2 f = both(-st.w * (along * inv_h)), m = both(-st.w * (mean_a * inv_h));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (kLayer) d[i] = add2(d[i], m);
        d[i] = fma2(n[i], f, d[i]);
      }
    }
    t.write16(static_cast<TX*>(p.dx) + at, d);
    Row16 n;
    if (p.o) {
      t.template read16<__nv_bfloat16>(base + at_o, n);
      if constexpr (!kKeep) own.get(1, c);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (kPost && kLayer) n[i] = add2(n[i], both(-st.x));
        if constexpr (kPost) n[i] = mul2(n[i], both(st.y));
        if constexpr (kPost || kGate) sa[i] = fma2(d[i], n[i], sa[i]);
        if constexpr (kPost && kBias) sb[i] = add2(sb[i], d[i]);
        d[i] = mul2(d[i], c[i]);
      }
    }
    if constexpr (kPost) {
      float2 s = zero, sm = zero;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s = fma2(d[i], n[i], s);
        if constexpr (kLayer) sm = add2(sm, d[i]);
      }
      float along, mean_a = 0.f;
      if constexpr (kLayer) row.sum2(s, sm, along, mean_a);
      else along = row.sum(s);
      if (blockDim.x == 32) __syncwarp();
      const float2 f = both(-(along * inv_h)), m = both(-(mean_a * inv_h));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (kLayer) d[i] = add2(d[i], m);
        d[i] = mul2(fma2(n[i], f, d[i]), both(st.y));
      }
    } else {
      t.release_barrier();
    }
    // past that barrier every thread has read the stage
    if (tid == 0 && r + p.stages < t.row1) fetch(r + p.stages, stage);
    if (p.o) t.write16(static_cast<__nv_bfloat16*>(p.d_o) + at, d);

    if constexpr (kGate == 2) {
      const int64_t g0 = int64_t(g) * p.gate_rows, g1 = min(int64_t(p.rows), g0 + p.gate_rows);
      if (r + 1 == t.row1 || r + 1 == g1) {
        // close the group's sums in this team: the whole group's (stored), or an edge piece for
        // the second kernel: slot 0 if the group began in an earlier team, else slot 1
        if (p.dgate)
          write_dgate(g0 >= t.row0 && g1 <= t.row1
                          ? p.dgate + int64_t(g) * H
                          : p.ws + (g0 < t.row0 ? 4 : 5) * vec + int64_t(t.team) * H);
        if constexpr (kPost) {
          Row16 v;
          vector16(p.gate, int64_t(g) * H, p.gate_bf16, t.col, t.live, 1.f, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            v[i] = mul2(v[i], both(p.scale));
            dwp[i] = fma2(v[i], sa[i], dwp[i]);
            if constexpr (kBias) dbp[i] = fma2(v[i], sb[i], dbp[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sa[i] = sb[i] = zero;
      }
    }
    if (++stage == p.stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  float* const mine = p.ws + int64_t(t.team) * H;
  if (p.dweight) t.write16(mine, dw);
  if (kBias && p.dbias) t.write16(mine + vec, db);
  if constexpr (kGate == 1) {          // the only group; a team's piece of it (slot 1 of the first)
    if (p.dgate) write_dgate(p.teams == 1 ? p.dgate : mine + (t.team ? 4 : 5) * vec);
  }
  if constexpr (kPost) {
    if constexpr (kGate != 2) {
      Row16 v;
      vector16(kGate ? p.gate : nullptr, 0, p.gate_bf16, t.col, t.live, 1.f, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = mul2(v[i], both(p.scale));
        dwp[i] = mul2(v[i], sa[i]);
        dbp[i] = mul2(v[i], sb[i]);
      }
    }
    if (p.dpost_weight) t.write16(mine + 2 * vec, dwp);
    if (kBias && p.dpost_bias) t.write16(mine + 3 * vec, dbp);
  }
  if constexpr (kCl > 1) ptx::cluster_sync();
#endif
}

// Adds the teams' partials: y = 0..3 the four parameter vectors, then the gate groups that cross
// from one team into another.  by_group (no more groups than teams): y - 4 is the group; else
// y - 3 is a team, and the group is the one that crosses into it if it is the first it crosses into.
static __global__ void __launch_bounds__(1024)
    block_norm_sums_kernel(const __grid_constant__ NormBackwardParams p) {
  __shared__ detail::ColumnSumShared smem;
  ptx::pdl_launch_dependents();
  ptx::pdl_wait_prior_grid();
  const int64_t vec = int64_t(p.teams) * p.H;
  if (blockIdx.y < 4) {
    float* const outs[4] = {p.dweight, p.dbias, p.dpost_weight, p.dpost_bias};
    float* dst = outs[blockIdx.y];
    if (!dst) return;
    detail::column_sum_cta(nullptr, p.ws + blockIdx.y * vec, p.teams, p.H, dst, p.H, blockIdx.x, smem);
    return;
  }
  const int64_t gr = p.gate_rows ? p.gate_rows : p.rows;
  int64_t g;
  if (p.groups <= p.teams) {
    g = blockIdx.y - 4;
  } else {
    const int64_t into = int64_t(blockIdx.y) - 3, at = row_begin(into, p.rows, p.teams);
    g = at / gr;
    if (g * gr >= at || team_of(g * gr, p.rows, p.teams) != into - 1) return;
  }
  const int64_t first = team_of(g * gr, p.rows, p.teams);
  const int64_t last = team_of(min(int64_t(p.rows), (g + 1) * gr) - 1, p.rows, p.teams);
  if (first == last) return;                          // stored whole by its team
  detail::column_sum_cta(p.ws + 5 * vec + first * p.H, p.ws + 4 * vec + (first + 1) * p.H, last - first,
                         p.H, p.dgate + g * p.H, p.H, blockIdx.x, smem);
}

template <class P>
inline cudaError_t launch_rows(void (*kernel)(P), P& p, const Geometry& g, int threads_per_sm,
                               int stage_bytes, int vectors, cudaStream_t s) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  e = detail::set_smem_once(kernel, kSharedBytes, dev);
  if (e != cudaSuccess) return e;
  p.slice = g.slice;
  p.teams = row_teams(p.rows, g, threads_per_sm);
  p.stages = ring_stages(g, threads_per_sm, stage_bytes, vectors, (p.rows + p.teams - 1) / p.teams);
  return detail::launch_pdl(kernel, dim3(p.teams * g.cluster), dim3(g.threads),
                            static_cast<size_t>(p.stages) * stage_bytes + size_t(vectors) * 64 * g.threads, s, p);
}

template <class TX, int kMode>
inline cudaError_t launch_block_norm(NormParams& p, bool post, cudaStream_t s) {
  const Geometry g = geometry(p.H);
  const int stage_bytes = 16 * g.threads * int(sizeof(TX) + (p.o ? 2 : 0));
  // FP32 vectors kept in shared memory: weight, bias, cw, cb.  Without a post norm cw is only the
  // scaled gate row and may be left to L1.
  int vectors = kMode == kRms ? 0 : !p.o ? 2 : post ? 4 : 3;
  // the narrow build where its smaller share of shared memory still holds two rows
  const int teams = row_teams(p.rows, g, kNarrowThreadsPerSm);
  auto fits = [&](int v) {
    return p.rows <= teams || ring_stages(g, kNarrowThreadsPerSm, stage_bytes, v, 2) == 2;
  };
  bool narrow = g.cluster == 1 && g.threads <= kNarrowThreads;
  if (narrow && !fits(vectors)) {
    narrow = vectors == 3 && fits(2);
    if (narrow) vectors = 2;
  }
  p.keep_cw = kMode != kRms && vectors >= 3;
  auto* kernel = narrow ? (post ? block_norm_kernel<TX, kMode, true, 1, kNarrowThreads> : block_norm_kernel<TX, kMode, false, 1, kNarrowThreads>)
                 : g.cluster == 1 ? (post ? block_norm_kernel<TX, kMode, true, 1, 512> : block_norm_kernel<TX, kMode, false, 1, 512>)
                                  : (post ? block_norm_kernel<TX, kMode, true, 2, 512> : block_norm_kernel<TX, kMode, false, 2, 512>);
  return launch_rows(kernel, p, g, narrow ? kNarrowThreadsPerSm : kThreadsPerSm, stage_bytes, vectors, s);
}

template <class TX, int kMode, bool kPost, int kGate>
inline cudaError_t launch_block_norm_backward(NormBackwardParams& p, cudaStream_t s) {
  const Geometry g = geometry(p.H);
  auto* kernel = g.cluster == 1 ? block_norm_backward_kernel<TX, kMode, kPost, kGate, 1>
                                : block_norm_backward_kernel<TX, kMode, kPost, kGate, 2>;
  const int per = (p.dy ? int(sizeof(TX)) + 2 : 0) + (p.dh ? int(sizeof(TX)) : 0) + (p.o ? 2 : 0);
  return launch_rows(kernel, p, g, kThreadsPerSm, 16 * g.threads * per, kMode != kRms && kPost ? 2 : 0, s);
}
template <class TX, int kMode, bool kPost>
inline cudaError_t launch_block_norm_backward(NormBackwardParams& p, int gate, cudaStream_t s) {
  return gate == 0   ? launch_block_norm_backward<TX, kMode, kPost, 0>(p, s)
         : gate == 1 ? launch_block_norm_backward<TX, kMode, kPost, 1>(p, s)
                     : launch_block_norm_backward<TX, kMode, kPost, 2>(p, s);
}

}  // namespace norm_detail

inline cudaError_t block_norm(const blackhole_sm100_block_norm_args& a, cudaStream_t stream) {
  using namespace norm_detail;
  cudaError_t e = block_norm_check(a);
  if (e != cudaSuccess) return e;
  NormParams p;
  p.x = a.x; p.o = a.o; p.gate = a.gate; p.weight = a.weight; p.bias = a.bias;
  p.post_weight = a.post_weight; p.post_bias = a.post_bias;
  p.h = a.h; p.out = a.out; p.sf = static_cast<uint8_t*>(a.sf); p.stats = a.stats;
  p.rows = a.rows; p.H = a.H;
  p.gate_rows = a.gate ? a.gate_rows : 0;
  p.param_bf16 = a.param_is_bf16; p.gate_bf16 = a.gate_is_bf16; p.out_format = a.out_format;
  p.scale = a.scale; p.eps = a.eps; p.global_scale = a.global_scale;
  const bool post = a.post_norm != 0;
  auto run = [&](auto tx) {
    using T = decltype(tx);
    return a.kind == 1              ? launch_block_norm<T, kLayerNorm>(p, post, stream)
           : a.bias || a.post_bias  ? launch_block_norm<T, kRmsBias>(p, post, stream)
                                    : launch_block_norm<T, kRms>(p, post, stream);
  };
  e = a.x_is_bf16 ? run(__nv_bfloat16{}) : run(float{});
  if (e != cudaSuccess) return e;
  return cudaGetLastError();
}

inline cudaError_t block_norm_backward(const blackhole_sm100_block_norm_backward_args& a,
                                       cudaStream_t stream) {
  using namespace norm_detail;
  cudaError_t e = block_norm_backward_check(a);
  if (e != cudaSuccess) return e;
  NormBackwardParams p;
  p.h = a.h; p.dy = a.dy; p.dh = a.dh; p.o = a.o; p.gate = a.gate; p.weight = a.weight;
  p.post_weight = a.post_weight; p.post_bias = a.post_bias; p.stats = a.stats;
  p.dx = a.dx; p.d_o = a.d_o;
  p.dweight = a.dweight; p.dbias = a.dbias; p.dpost_weight = a.dpost_weight;
  p.dpost_bias = a.dpost_bias; p.dgate = a.dgate;
  p.ws = static_cast<float*>(a.workspace);
  p.rows = a.rows; p.H = a.H;
  p.gate_rows = a.gate ? a.gate_rows : 0;
  p.groups = !a.gate || a.gate_rows == 0 ? 1 : static_cast<int>((int64_t(a.rows) + a.gate_rows - 1) / a.gate_rows);
  p.param_bf16 = a.param_is_bf16; p.gate_bf16 = a.gate_is_bf16;
  p.scale = a.scale;
  // one group closes its sums once, at a team's end
  const int gate = !a.gate ? 0 : p.groups == 1 ? 1 : 2;
  const bool bias = a.dbias || a.dpost_bias || (a.post_bias && a.dgate);
  auto run = [&](auto tx) {
    using T = decltype(tx);
    if (a.kind == 1)
      return a.post_norm ? launch_block_norm_backward<T, kLayerNorm, true>(p, gate, stream)
                         : launch_block_norm_backward<T, kLayerNorm, false>(p, gate, stream);
    if (bias)
      return a.post_norm ? launch_block_norm_backward<T, kRmsBias, true>(p, gate, stream)
                         : launch_block_norm_backward<T, kRmsBias, false>(p, gate, stream);
    return a.post_norm ? launch_block_norm_backward<T, kRms, true>(p, gate, stream)
                       : launch_block_norm_backward<T, kRms, false>(p, gate, stream);
  };
  e = a.x_is_bf16 ? run(__nv_bfloat16{}) : run(float{});
  if (e != cudaSuccess) return e;
  const int edges = a.dgate && a.gate_rows != 1 && p.teams > 1 ? std::min(p.groups, p.teams - 1 + (p.groups <= p.teams)) : 0;
  if (a.dweight || a.dbias || a.dpost_weight || a.dpost_bias || edges) {
    const dim3 grid((a.H + detail::kColumnSumCols - 1) / detail::kColumnSumCols, 4 + edges);
    e = detail::launch_pdl(block_norm_sums_kernel, grid, dim3(1024), 0, stream, p);
    if (e != cudaSuccess) return e;
  }
  return cudaGetLastError();
}

#endif  // __CUDACC__

}  // namespace blackhole::sm100
