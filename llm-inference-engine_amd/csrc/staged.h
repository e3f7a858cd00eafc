// What the staged matrix-core kernels share: waits, buffers, and the epilogue
// of a plain product or of the gated block.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "device_util.h"
#include "ehip.h"

namespace ehip {

typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(4))) int i32x4_t;

// The feed-forward activations (EHIP_ACT_*), fp32. exp by the hardware's base-2
// exponential (one unit in the last place) of x log2 e; 1 / (1 + exp) by its
// reciprocal. An argument of -infinity gives NaN, as x / (1 + exp(-x)) does.
template <int ACT>
__device__ __forceinline__ float Activate(float x) {
  if constexpr (ACT == EHIP_ACT_SILU) {
    return x * __builtin_amdgcn_rcpf(1.f + Exp2(-kLog2e * x));
  } else if constexpr (ACT == EHIP_ACT_GELU) {
    return 0.5f * x * erfcf(-0.70710678118654752f * x);
  } else {
    // 0.5 (1 + tanh u) = 1 / (1 + exp(-2u)), u = sqrt(2 / pi) (x + 0.044715 x^3)
    const float u = x * (1.f + 0.044715f * x * x);
    return x * __builtin_amdgcn_rcpf(1.f + Exp2(-2.f * 0.79788456080286536f * kLog2e * u));
  }
}

// ACT of a plain product; gated ones name their activation, so that a kernel
// holds one activation's code (erfc alone is a hundred instructions a value).
constexpr int kPlain = -1;

// Biases, then the activation and the product, of four columns from `col`: g the
// plain product's or the gate's sums, `up` the other projection's. P has bias[2]
// and n.
template <int ACT, class P>
__device__ __forceinline__ f32x4_t Finish(const P& p, int64_t col, f32x4_t g, f32x4_t up) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = col + i < p.n;
    float v = g[i] + (in && p.bias[0] ? p.bias[0][col + i] : 0.f);
    if constexpr (ACT != kPlain)
      v = Activate<ACT>(v) * (up[i] + (in && p.bias[1] ? p.bias[1][col + i] : 0.f));
    g[i] = v;
  }
  return g;
}

// Four columns of a row of y, as far as they lie in it. P has y, m, n, y_vec.
// STREAM: the least y_vec whose stores go past the caches (0: none's), for the
// results of many rows: 1 where an instruction writes 128 bytes of a row and more,
// 2 where it writes 64, which come together in L2 unless rows are whole lines (MXFP4
// gated 2400 x 896 x 3584 23.7 us streamed and 25.3 cached, 2400 x 300 x 9000, whose
// rows begin inside lines, 56 and 37; bf16, 128 bytes, 81 and 84).
template <int STREAM, class P>
__device__ __forceinline__ void StoreRow4(const P& p, int64_t row, int64_t col, const f32x4_t& v) {
  if (row >= p.m || col >= p.n) return;
  float* y = p.y + row * p.n + col;
  if (STREAM > 0 && p.y_vec >= STREAM) {
    __builtin_nontemporal_store(v, reinterpret_cast<f32x4_t*>(y));
  } else if (p.y_vec) {  // n % 4 == 0
    *reinterpret_cast<f32x4_t*>(y) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < p.n) y[i] = v[i];
  }
}

template <int I>
__device__ __forceinline__ unsigned char* Buffer(unsigned char* b0, unsigned char* b1,
                                                 unsigned char* b2, unsigned char* b3) {
  return I == 0 ? b0 : I == 1 ? b1 : I == 2 ? b2 : b3;
}

// Waits until no more than N vector-memory operations and no LDS one of the
// wavefront are outstanding, then for the other wavefronts.
template <int N>
__device__ __forceinline__ void WaitAndMeet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Keeps the compiler from moving memory operations across.
__device__ __forceinline__ void Fence() { asm volatile("" ::: "memory"); }

// Four columns' sums from `col` on, 2^down times as much, and (COLS) times their
// columns' own powers of two. P has col_scale and col_stride, whole panels and a
// tile's width beyond them.
template <bool COLS, class P>
__device__ __forceinline__ void Rescale(const P& p, int64_t col, int down, f32x4_t* g, f32x4_t* u) {
  i32x4_t dg = {down, down, down, down}, du = dg;
  if constexpr (COLS) {
    dg += *reinterpret_cast<const i32x4_t*>(p.col_scale + col);
    du += *reinterpret_cast<const i32x4_t*>(p.col_scale + p.col_stride + col);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    (*g)[i] = __builtin_amdgcn_ldexpf((*g)[i], dg[i]);
    (*u)[i] = __builtin_amdgcn_ldexpf((*u)[i], du[i]);
  }
}

// A tile's results, acc[XP][WP] of 16 x 16 blocks (lane (n16, q): columns 4q..4q+3
// of row n16; gated: even slots the gate's, odd ones the up projection's), from
// row0 and col0 of y. Through `part` of LDS, the wavefront's own C * 256 * PP
// bytes, so that a store instruction writes whole runs of its columns (256
// bytes a row at WP = 4, gated 128) instead of 64-byte pieces of 16 rows: 16-byte
// chunk c of row r at c ^ r, where the 16 lanes of a pass hit distinct banks.
// SCALED > 0: the sums of panel a's row n16 stand for 2^down[a] times as much, 2:
// the columns' likewise.
template <int XP, int WP, int PP, int ACT, int SCALED, class P>
__device__ __forceinline__ void StoreTile(const P& p, unsigned char* part, int64_t row0,
                                          int64_t col0, const f32x4_t (&acc)[XP][WP],
                                          const int (&down)[XP]) {
  constexpr int PR = ACT != kPlain ? 2 : 1, C = 4 * WP / PR;
  static_assert(XP % PP == 0 && (C & (C - 1)) == 0, "whole passes");
  const int lane = threadIdx.x & 63, n16 = lane & 15, q = lane >> 4;
#pragma unroll
  for (int a0 = 0; a0 < XP; a0 += PP) {
#pragma unroll
    for (int a = 0; a < PP; ++a)
#pragma unroll
      for (int b = 0; b < WP; b += PR) {
        const int c = b / PR * 4 + q;
        f32x4_t g = acc[a0 + a][b], u = acc[a0 + a][b + PR - 1];
        if constexpr (SCALED > 0) Rescale<SCALED == 2>(p, col0 + 4 * c, down[a0 + a], &g, &u);
        *reinterpret_cast<f32x4_t*>(part + ((a * 16 + n16) * C + ((c ^ n16) & (C - 1))) * 16) =
            Finish<ACT>(p, col0 + 4 * c, g, u);
      }
#pragma unroll
    for (int i = 0; i < PP * 16 * C / 64; ++i) {
      const int r = i * (64 / C) + lane / C, c = lane % C;
      const f32x4_t v =
          *reinterpret_cast<const f32x4_t*>(part + (r * C + ((c ^ r) & (C - 1))) * 16);
      StoreRow4<(C >= 8 ? 1 : 2)>(p, row0 + a0 * 16 + r, col0 + 4 * c, v);
    }
  }
}

}  // namespace ehip
