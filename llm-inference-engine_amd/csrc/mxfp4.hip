// Microscaled 4-bit floating point (MXFP4): matrices into panels and back, and
// the products over them (layout and helpers: mxfp4.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "kernels.h"
#include "mxfp4.h"

namespace ehip {
namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((ext_vector_type(4))) int i32x4_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

// ------------------------------------------------------------- quantisation --
//
// One workgroup per (panel, scale group): 16 rows x 512 k, thread (r, i) with
// elements 8i..8i+7 of row r in each of the group's tiles. Four threads hold a
// block: its largest magnitude by two lane exchanges, as integers (the order of
// non-negative floats, infinities and NaN on top).

template <int DT>
__device__ __forceinline__ void Load8(const void* x, int64_t at, float (&v)[8]) {
  if constexpr (DT == EHIP_WEIGHT_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(x) + at);
    const float4 a = p[0], b = p[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + at);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == EHIP_WEIGHT_BF16) {
        v[2 * i] = Bf16Lo(w[i]);
        v[2 * i + 1] = Bf16Hi(w[i]);
      } else {
        v[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i])));
        v[2 * i + 1] =
            static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i] >> 16)));
      }
    }
  }
}

template <int DT>
__device__ __forceinline__ float Load1(const void* x, int64_t at) {
  if constexpr (DT == EHIP_WEIGHT_F32)
    return static_cast<const float*>(x)[at];
  else if constexpr (DT == EHIP_WEIGHT_BF16)
    return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(x)[at]) << 16);
  else
    return static_cast<float>(
        __builtin_bit_cast(_Float16, static_cast<const uint16_t*>(x)[at]));
}

__device__ __forceinline__ uint32_t DppMax4(uint32_t a) {
  a = max(a, static_cast<uint32_t>(
                 __builtin_amdgcn_update_dpp(0, static_cast<int>(a), 0xB1, 0xF, 0xF, false)));
  return max(a, static_cast<uint32_t>(
                    __builtin_amdgcn_update_dpp(0, static_cast<int>(a), 0x4E, 0xF, 0xF, false)));
}

template <int DT>
__global__ __launch_bounds__(256) void MxQuantize(const void* x, int64_t rows, int64_t k,
                                                  int32_t vec, uint32_t* codes,
                                                  uint32_t* scales) {
  const int r = threadIdx.x >> 4, i = threadIdx.x & 15;
  const int64_t tiles = (k + kMxTile - 1) / kMxTile;
  const int64_t groups = (tiles + kMxGroup - 1) / kMxGroup;
  const uint32_t bp = blockIdx.x / static_cast<uint32_t>(groups);
  const int64_t panel = bp, group = blockIdx.x - bp * static_cast<uint32_t>(groups);
  const int64_t row = panel * kMxRows + r;
  float v[kMxGroup][8];
#pragma unroll
  for (int j = 0; j < kMxGroup; ++j) {
    const int64_t k0 = (group * kMxGroup + j) * kMxTile + 8 * i;
    if (vec && row < rows && k0 + 8 <= k) {
      Load8<DT>(x, row * k + k0, v[j]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[j][e] = row < rows && k0 + e < k ? Load1<DT>(x, row * k + k0 + e) : 0.f;
    }
  }
  uint32_t packed = 0;
#pragma unroll
  for (int j = 0; j < kMxGroup; ++j) {
    uint32_t a = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = max(a, __float_as_uint(v[j][e]) & 0x7FFFFFFFu);
    const uint32_t byte = MxScaleByte(DppMax4(a));
    packed |= byte << (8 * j);
    const int64_t tile = group * kMxGroup + j;
    if (tile < tiles)
      codes[((panel * tiles + tile) * 64 + (i >> 2) * 16 + r) * 4 + (i & 3)] =
          MxCodes(v[j], byte);
  }
  if ((i & 3) == 0) scales[(panel * groups + group) * 64 + (i >> 2) * 16 + r] = packed;
}

// Row-major codes [rows, blocks, 16 bytes] and scales [rows, blocks] into
// panels, over the same work split.
__global__ __launch_bounds__(256) void MxPack(const uint8_t* rc, const uint8_t* rs, int64_t rows,
                                              int64_t k, uint32_t* codes, uint32_t* scales) {
  const int r = threadIdx.x >> 4, i = threadIdx.x & 15;
  const int64_t blocks = (k + kMxBlock - 1) / kMxBlock;
  const int64_t tiles = (blocks + 3) / 4;
  const int64_t groups = (tiles + kMxGroup - 1) / kMxGroup;
  const uint32_t bp = blockIdx.x / static_cast<uint32_t>(groups);
  const int64_t panel = bp, group = blockIdx.x - bp * static_cast<uint32_t>(groups);
  const int64_t row = panel * kMxRows + r;
  uint32_t packed = 0;
#pragma unroll
  for (int j = 0; j < kMxGroup; ++j) {
    const int64_t tile = group * kMxGroup + j;
    const int64_t block = 4 * tile + (i >> 2);
    uint32_t c = 0;
    if (row < rows && block < blocks) {
      const uint8_t* src = rc + (row * blocks + block) * 16 + 4 * (i & 3);
      c = src[0] | uint32_t{src[1]} << 8 | uint32_t{src[2]} << 16 | uint32_t{src[3]} << 24;
      // A last block's codes past k take part in no product: zeros here.
      const int64_t left = k - block * kMxBlock - 8 * (i & 3);
      if (left < 8) c = left <= 0 ? 0u : c & ((1u << (4 * left)) - 1u);
      packed |= uint32_t{rs[row * blocks + block]} << (8 * j);
    }
    if (tile < tiles) codes[((panel * tiles + tile) * 64 + (i >> 2) * 16 + r) * 4 + (i & 3)] = c;
  }
  if ((i & 3) == 0) scales[(panel * groups + group) * 64 + (i >> 2) * 16 + r] = packed;
}

// Panels into fp32 rows, over the same work split.
__global__ __launch_bounds__(256) void MxDequantize(const uint32_t* codes, const uint32_t* scales,
                                                    int64_t rows, int64_t k, int32_t vec,
                                                    float* y) {
  const int r = threadIdx.x >> 4, i = threadIdx.x & 15;
  const int64_t tiles = (k + kMxTile - 1) / kMxTile;
  const int64_t groups = (tiles + kMxGroup - 1) / kMxGroup;
  const uint32_t bp = blockIdx.x / static_cast<uint32_t>(groups);
  const int64_t panel = bp, group = blockIdx.x - bp * static_cast<uint32_t>(groups);
  const int64_t row = panel * kMxRows + r;
  if (row >= rows) return;
  const uint32_t packed = scales[(panel * groups + group) * 64 + (i >> 2) * 16 + r];
#pragma unroll
  for (int j = 0; j < kMxGroup; ++j) {
    const int64_t tile = group * kMxGroup + j;
    const int64_t k0 = tile * kMxTile + 8 * i;
    if (k0 >= k) continue;
    const uint32_t c = codes[((panel * tiles + tile) * 64 + (i >> 2) * 16 + r) * 4 + (i & 3)];
    const uint32_t byte = (packed >> (8 * j)) & 255u;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      // E2M1 as fp32: exponent 0 is m / 2, the others 2^(exponent - 1) (1 + m / 2).
      const uint32_t code = (c >> (4 * e)) & 15u, m = code & 7u;
      const float mag = m < 2u ? 0.5f * static_cast<float>(m)
                               : __uint_as_float((126u + (m >> 1)) << 23 | (m & 1u) << 22);
      const float s = code & 8u ? -mag : mag;
      v[e] = byte == 255u ? __builtin_nanf("")
                          : __builtin_amdgcn_ldexpf(s, static_cast<int>(byte) - 127);
    }
    float* out = y + row * k + k0;
    if (vec && k0 + 8 <= k) {
      reinterpret_cast<float4*>(out)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(out)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k0 + e < k) out[e] = v[e];
    }
  }
}

// ------------------------------------------------------------------ products --
//
// y[m, n] = sum_k xq[m, k] wq[n, k]: the scaled matrix-core product of 16 x 16 x
// 128, whose products are exact and whose sums are fp32. The weight is the A
// operand and x the B operand, so that a lane's four results are four
// consecutive columns of one row of y.

template <int J>
__device__ __forceinline__ f32x4_t MxMfma(const i32x4_t& w, uint32_t ws, const i32x4_t& x,
                                          uint32_t xs, const f32x4_t& acc) {
  const i32x8_t a = __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8_t b = __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, J,
                                                          static_cast<int>(ws), J,
                                                          static_cast<int>(xs));
}

// ACT of a plain product; gated ones name their activation, so that a kernel
// holds one activation's code (erfc alone is a hundred instructions a value).
constexpr int kPlain = -1;

// One fragment's results: row n16 of an x panel, columns 4 q .. + 3 of a weight
// panel; `up` the other projection's sums of a gated call.
template <int ACT>
__device__ __forceinline__ void MxStore(const MxGemmParams& p, int64_t row, int64_t col,
                                        f32x4_t g, f32x4_t up) {
  if (row >= p.m || col >= p.n) return;
  float out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = col + i < p.n;
    float v = g[i] + (in && p.bias[0] ? p.bias[0][col + i] : 0.f);
    if constexpr (ACT != kPlain)
      v = Activate<ACT>(v) * (up[i] + (in && p.bias[1] ? p.bias[1][col + i] : 0.f));
    out[i] = v;
  }
  float* y = p.y + row * p.n + col;
  if (p.y_vec && col + 4 <= p.n) {
    *reinterpret_cast<float4*>(y) = make_float4(out[0], out[1], out[2], out[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < p.n) y[i] = out[i];
  }
}

// Few rows: a workgroup per (MP x panels, NP weight panels), its KW wavefronts
// taking the scale groups in turn with their operands straight from memory into
// registers, then one sum over the wavefronts through LDS, in their order.
template <int MP, int NP, int ACT, int KW>
__global__ __launch_bounds__(64 * KW) void MxDirect(MxGemmParams p) {
  constexpr int PR = ACT != kPlain ? 2 : 1;
  __shared__ f32x4_t red[KW][MP * NP * PR][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const uint32_t w_groups = static_cast<uint32_t>((p.w_panels + NP - 1) / NP);
  const uint32_t xb = blockIdx.x / w_groups;
  const int64_t wp0 = int64_t{blockIdx.x - xb * w_groups} * NP, xp0 = int64_t{xb} * MP;
  f32x4_t acc[MP][NP * PR];
#pragma unroll
  for (int a = 0; a < MP; ++a)
#pragma unroll
    for (int b = 0; b < NP * PR; ++b) acc[a][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // Panels past the last read the last one: their results are not stored.
  const i32x4_t* xc[MP];
  const uint32_t* xs[MP];
  const i32x4_t* wc[NP * PR];
  const uint32_t* ws[NP * PR];
#pragma unroll
  for (int a = 0; a < MP; ++a) {
    const int64_t panel = min(xp0 + a, p.x_panels - 1);
    xc[a] = reinterpret_cast<const i32x4_t*>(p.xc) + panel * p.tiles * 64 + lane;
    xs[a] = reinterpret_cast<const uint32_t*>(p.xs) + panel * p.groups * 64 + lane;
  }
#pragma unroll
  for (int b = 0; b < NP * PR; ++b) {
    const int64_t panel = min(wp0 + b / PR, p.w_panels - 1);
    wc[b] = reinterpret_cast<const i32x4_t*>(p.wc[b % PR]) + panel * p.tiles * 64 + lane;
    ws[b] = reinterpret_cast<const uint32_t*>(p.ws[b % PR]) + panel * p.groups * 64 + lane;
  }
  for (int t = wave; t < p.groups; t += KW) {
    uint32_t sx[MP], sw[NP * PR];
#pragma unroll
    for (int a = 0; a < MP; ++a) sx[a] = xs[a][int64_t{t} * 64];
#pragma unroll
    for (int b = 0; b < NP * PR; ++b) sw[b] = ws[b][int64_t{t} * 64];
    auto step = [&](auto j) __attribute__((always_inline)) {
      constexpr int J = decltype(j)::value;
      const int64_t tile = int64_t{t} * kMxGroup + J;
      if (tile >= p.tiles) return;
      i32x4_t x[MP];
#pragma unroll
      for (int a = 0; a < MP; ++a) x[a] = xc[a][tile * 64];
#pragma unroll
      for (int b = 0; b < NP * PR; ++b) {
        const i32x4_t w = wc[b][tile * 64];
#pragma unroll
        for (int a = 0; a < MP; ++a) acc[a][b] = MxMfma<J>(w, sw[b], x[a], sx[a], acc[a][b]);
      }
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    step(std::integral_constant<int, 2>{});
    step(std::integral_constant<int, 3>{});
  }
#pragma unroll
  for (int a = 0; a < MP; ++a)
#pragma unroll
    for (int b = 0; b < NP * PR; ++b) red[wave][a * NP * PR + b][lane] = acc[a][b];
  __syncthreads();
  for (int f = wave; f < MP * NP; f += KW) {
    f32x4_t s[PR];
#pragma unroll
    for (int h = 0; h < PR; ++h) {
      s[h] = red[0][f * PR + h][lane];
      for (int w = 1; w < KW; ++w) s[h] += red[w][f * PR + h][lane];
    }
    const int64_t row = (xp0 + f / NP) * kMxRows + (lane & 15);
    const int64_t panel = wp0 + f % NP;
    if (panel < p.w_panels) MxStore<ACT>(p, row, panel * kMxRows + 4 * (lane >> 4), s[0], s[PR - 1]);
  }
}

// Many rows: a workgroup of WR x WC wavefronts per tile of WR XP x panels by WC WP
// weight panels (gated: their even slots the gate's, the odd ones the up
// projection's). k tiles go from memory straight into LDS (buffer_load ... lds, a
// panel's 1 KiB an instruction, four a wavefront), into four buffers, three
// tiles ahead; an operand is one conflict-free 16-byte read. A wavefront's
// scales, one dword a panel and group, come through registers a group ahead.
template <int WR, int WC, int XP, int WP, int ACT, int OCC>
__global__ __launch_bounds__(64 * WR * WC) __attribute__((amdgpu_waves_per_eu(OCC)))
void MxStaged(MxGemmParams p) {
  constexpr bool GATED = ACT != kPlain;
  constexpr int XT = WR * XP, WT = WC * WP;  // panels of the tile
  static_assert(XT + WT == 4 * WR * WC && XT % 4 == 0, "four panels a wavefront");
  static_assert(!GATED || WP % 2 == 0, "pairs of slots");
  __shared__ __align__(16) unsigned char b0[(XT + WT) * kMxTileBytes];
  __shared__ __align__(16) unsigned char b1[(XT + WT) * kMxTileBytes];
  __shared__ __align__(16) unsigned char b2[(XT + WT) * kMxTileBytes];
  __shared__ __align__(16) unsigned char b3[(XT + WT) * kMxTileBytes];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int wr = wave / WC, wc = wave % WC;

  // Tiles in bands of 4 rows of tiles, columns outer within a band; an XCD (b
  // mod 8) takes consecutive ones, which share their panels in its L2.
  const uint32_t tiles_all = static_cast<uint32_t>(p.row_tiles) * p.col_tiles;
  const uint32_t per = (tiles_all + 7) / 8;
  const uint32_t tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (tile >= tiles_all) return;
  const uint32_t band = tile / (4u * p.col_tiles);
  const uint32_t in_band = tile - band * 4u * p.col_tiles;
  const uint32_t h = min(4u, static_cast<uint32_t>(p.row_tiles) - 4u * band);
  const int ct = __builtin_amdgcn_readfirstlane(in_band / h);
  const int rt = __builtin_amdgcn_readfirstlane(4 * band + in_band % h);
  const int64_t xp0 = int64_t{rt} * XT;
  const int64_t wp0 = int64_t{ct} * (GATED ? WT / 2 : WT);
  const int last_x = static_cast<int>(min(int64_t{XT}, p.x_panels - xp0)) - 1;
  const int last_w = static_cast<int>(min(int64_t{WT}, p.w_panels - wp0)) - 1;

  // The wavefront's four panels of a stage: all of x, or all weight slots.
  // Panels past the last read the last one: their results are not stored.
  const int slot = 4 * wave;
  const bool is_x = slot < XT;
  const int64_t row_bytes = int64_t{p.tiles} * kMxTileBytes;
  const uint8_t* const even = is_x ? p.xc + xp0 * row_bytes : p.wc[0] + wp0 * row_bytes;
  const uint8_t* const odd = is_x || !GATED ? even : p.wc[1] + wp0 * row_bytes;
  const __amdgpu_buffer_rsrc_t re = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(even), 0, 0xFFFFFFFFu, 0x00020000);
  const __amdgpu_buffer_rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(odd), 0, 0xFFFFFFFFu, 0x00020000);
  uint32_t src[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int local = is_x ? min(slot + i, last_x)
                           : min(GATED ? (slot - XT + i) / 2 : slot - XT + i, last_w);
    src[i] = static_cast<uint32_t>(local) * static_cast<uint32_t>(row_bytes);
  }
  auto stage = [&](unsigned char* buf, int t) __attribute__((always_inline)) {
    const uint32_t at = static_cast<uint32_t>(min(t, p.tiles - 1)) * kMxTileBytes;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          i & 1 ? ro : re,
          (__attribute__((address_space(3))) void*)(buf + (slot + i) * kMxTileBytes), 16,
          lane * 16, src[i] + at, 0, 0);
  };

  // Scales of the wavefront's own panels.
  const int64_t row_scales = int64_t{p.groups} * kMxScaleBytes;
  const __amdgpu_buffer_rsrc_t rxs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(p.xs + xp0 * row_scales), 0, 0xFFFFFFFFu, 0x00020000);
  const __amdgpu_buffer_rsrc_t rg = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(p.ws[0] + wp0 * row_scales), 0, 0xFFFFFFFFu, 0x00020000);
  const __amdgpu_buffer_rsrc_t ru =
      GATED ? __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.ws[1] + wp0 * row_scales), 0,
                                                0xFFFFFFFFu, 0x00020000)
            : rg;
  auto load_scales = [&](int g, uint32_t (&sx)[XP], uint32_t (&sw)[WP])
                         __attribute__((always_inline)) {
    const uint32_t at = static_cast<uint32_t>(min(g, p.groups - 1)) * kMxScaleBytes;
    const uint32_t rs = static_cast<uint32_t>(row_scales);
#pragma unroll
    for (int a = 0; a < XP; ++a)
      sx[a] = __builtin_amdgcn_raw_buffer_load_b32(
          rxs, lane * 4, static_cast<uint32_t>(min(wr * XP + a, last_x)) * rs + at, 0);
#pragma unroll
    for (int b = 0; b < WP; ++b) {
      const int local = min(GATED ? (wc * WP + b) / 2 : wc * WP + b, last_w);
      sw[b] = __builtin_amdgcn_raw_buffer_load_b32(GATED && (b & 1) ? ru : rg, lane * 4,
                                                   static_cast<uint32_t>(local) * rs + at, 0);
    }
  };

  f32x4_t acc[XP][WP];
#pragma unroll
  for (int a = 0; a < XP; ++a)
#pragma unroll
    for (int b = 0; b < WP; ++b) acc[a][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  uint32_t sx[XP], sw[WP], nx[XP], nw[WP];

#define EHIP_MX_FENCE() asm volatile("" ::: "memory")
  load_scales(0, sx, sw);
  EHIP_MX_FENCE();
  stage(b0, 0);
  EHIP_MX_FENCE();
  stage(b1, 1);
  EHIP_MX_FENCE();
  stage(b2, 2);
  EHIP_MX_FENCE();
  auto compute = [&](auto j, const unsigned char* buf) __attribute__((always_inline)) {
    constexpr int J = decltype(j)::value;
    i32x4_t w[WP];
#pragma unroll
    for (int b = 0; b < WP; ++b)
      w[b] = *reinterpret_cast<const i32x4_t*>(buf + (XT + wc * WP + b) * kMxTileBytes + lane * 16);
#pragma unroll
    for (int a = 0; a < XP; ++a) {
      const i32x4_t x =
          *reinterpret_cast<const i32x4_t*>(buf + (wr * XP + a) * kMxTileBytes + lane * 16);
#pragma unroll
      for (int b = 0; b < WP; ++b) acc[a][b] = MxMfma<J>(w[b], sw[b], x, sx[a], acc[a][b]);
    }
  };
  // Step t waits for its own tile's loads and meets the other wavefronts', then
  // loads tile t + 3 into the buffer that step t - 1 has read. The loads stay
  // unconditional (past the end: the last tile again), so that the counts
  // hold: behind a tile's loads are two more tiles' (8), and at J = 1 and 2 the
  // next group's XP + WP scales, which are loaded at J = 0.
#define EHIP_MX_STEP(J, BUF, NEXT, PENDING)                                                  \
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(PENDING) : "memory");      \
  if ((J) == 0) {                                                                            \
    load_scales(g + 1, nx, nw);                                                              \
    EHIP_MX_FENCE();                                                                         \
  }                                                                                          \
  stage(NEXT, 4 * g + (J) + 3);                                                              \
  EHIP_MX_FENCE();                                                                           \
  compute(std::integral_constant<int, (J)>{}, BUF);                                          \
  if (4 * g + (J) + 1 >= p.tiles) break
  for (int g = 0;; ++g) {
    EHIP_MX_STEP(0, b0, b3, 8);
    EHIP_MX_STEP(1, b1, b0, 8 + XP + WP);
    EHIP_MX_STEP(2, b2, b1, 8 + XP + WP);
    EHIP_MX_STEP(3, b3, b2, 8);
#pragma unroll
    for (int a = 0; a < XP; ++a) sx[a] = nx[a];
#pragma unroll
    for (int b = 0; b < WP; ++b) sw[b] = nw[b];
  }
  // Loads past the end may still be in flight: they write this workgroup's
  // LDS, so they land before it ends.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#undef EHIP_MX_STEP
#undef EHIP_MX_FENCE

#pragma unroll
  for (int a = 0; a < XP; ++a) {
    const int64_t row = (xp0 + wr * XP + a) * kMxRows + (lane & 15);
#pragma unroll
    for (int b = 0; b < WP; b += GATED ? 2 : 1) {
      const int64_t panel = wp0 + (GATED ? (wc * WP + b) / 2 : wc * WP + b);
      MxStore<ACT>(p, row, panel * kMxRows + 4 * (lane >> 4), acc[a][b],
                     acc[a][GATED ? b + 1 : b]);
    }
  }
}

template <int WR, int WC, int XP, int WP, int ACT, int OCC>
hipError_t LaunchStaged(MxGemmParams p, hipStream_t stream) {
  constexpr int64_t XT = WR * XP, WT = ACT != kPlain ? WC * WP / 2 : WC * WP;
  const int64_t rt = (p.x_panels + XT - 1) / XT, ct = (p.w_panels + WT - 1) / WT;
  if (rt * ct > (int64_t{1} << 30)) return hipErrorInvalidValue;
  p.row_tiles = static_cast<int32_t>(rt);
  p.col_tiles = static_cast<int32_t>(ct);
  const uint32_t grid = static_cast<uint32_t>((rt * ct + 7) / 8 * 8);
  hipLaunchKernelGGL((MxStaged<WR, WC, XP, WP, ACT, OCC>), dim3(grid), dim3(64 * WR * WC), 0,
                     stream, p);
  return hipGetLastError();
}

template <int ACT>
hipError_t LaunchDirect(const MxGemmParams& p, hipStream_t stream) {
  const int64_t n = p.w_panels * ((p.x_panels + 3) / 4);
  if (n > INT32_MAX) return hipErrorInvalidValue;
  const dim3 grid(static_cast<uint32_t>(n));
  if (p.x_panels == 1)
    hipLaunchKernelGGL((MxDirect<1, 1, ACT, 8>), grid, dim3(512), 0, stream, p);
  else
    hipLaunchKernelGGL((MxDirect<4, 1, ACT, 8>), grid, dim3(512), 0, stream, p);
  return hipGetLastError();
}

template <int ACT>
hipError_t LaunchProduct(const MxGemmParams& p, hipStream_t stream) {
  if (p.m > 256) return LaunchStaged<2, 4, 8, 4, ACT, 2>(p, stream);
  if (p.m > 64) return LaunchStaged<2, 2, 4, 4, ACT, 2>(p, stream);
  return LaunchDirect<ACT>(p, stream);
}

// Workgroups of the panel conversions, 0 where a launch cannot hold them.
uint32_t MxConvertGrid(int64_t rows, int64_t k) {
  const int64_t n = MxPanels(rows) * MxGroups(k);
  return n <= INT32_MAX ? static_cast<uint32_t>(n) : 0u;
}

}  // namespace

hipError_t LaunchMxQuantize(const void* x, int dtype, int64_t rows, int64_t k, void* codes,
                            void* scales, hipStream_t stream) {
  const dim3 grid(MxConvertGrid(rows, k)), block(256);
  const int32_t vec = k % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  uint32_t* c = static_cast<uint32_t*>(codes);
  uint32_t* s = static_cast<uint32_t*>(scales);
  if (grid.x == 0) return hipErrorInvalidValue;
  if (dtype == EHIP_WEIGHT_F32)
    hipLaunchKernelGGL(MxQuantize<EHIP_WEIGHT_F32>, grid, block, 0, stream, x, rows, k, vec, c, s);
  else if (dtype == EHIP_WEIGHT_BF16)
    hipLaunchKernelGGL(MxQuantize<EHIP_WEIGHT_BF16>, grid, block, 0, stream, x, rows, k, vec, c, s);
  else
    hipLaunchKernelGGL(MxQuantize<EHIP_WEIGHT_F16>, grid, block, 0, stream, x, rows, k, vec, c, s);
  return hipGetLastError();
}

hipError_t LaunchMxPack(const uint8_t* row_codes, const uint8_t* row_scales, int64_t rows,
                        int64_t k, void* codes, void* scales, hipStream_t stream) {
  const dim3 grid(MxConvertGrid(rows, k));
  if (grid.x == 0) return hipErrorInvalidValue;
  hipLaunchKernelGGL(MxPack, grid, dim3(256), 0, stream, row_codes, row_scales, rows, k,
                     static_cast<uint32_t*>(codes), static_cast<uint32_t*>(scales));
  return hipGetLastError();
}

hipError_t LaunchMxDequantize(const void* codes, const void* scales, int64_t rows, int64_t k,
                              float* y, hipStream_t stream) {
  const dim3 grid(MxConvertGrid(rows, k));
  const int32_t vec = k % 8 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
  if (grid.x == 0) return hipErrorInvalidValue;
  hipLaunchKernelGGL(MxDequantize, grid, dim3(256), 0, stream,
                     static_cast<const uint32_t*>(codes), static_cast<const uint32_t*>(scales),
                     rows, k, vec, y);
  return hipGetLastError();
}

hipError_t LaunchMxGemm(const MxGemmParams& p, bool gated, hipStream_t stream) {
  if (!gated) return LaunchProduct<kPlain>(p, stream);
  switch (p.act) {
    case EHIP_ACT_SILU: return LaunchProduct<EHIP_ACT_SILU>(p, stream);
    case EHIP_ACT_GELU: return LaunchProduct<EHIP_ACT_GELU>(p, stream);
    default: return LaunchProduct<EHIP_ACT_GELU_TANH>(p, stream);
  }
}

}  // namespace ehip
