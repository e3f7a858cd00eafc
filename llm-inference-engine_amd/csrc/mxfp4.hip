// Microscaled 4-bit floating point (MXFP4): matrices into panels and back, and
// the products over them (layout and helpers: mxfp4.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "kernels.h"
#include "mxfp4.h"
#include "staged.h"

namespace ehip {
namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8_t;

// ------------------------------------------------------------- quantisation --
//
// One workgroup per (panel, scale group): 16 rows x 512 k, thread (r, i) with
// elements 8i..8i+7 of row r in each of the group's tiles. Four threads hold a
// block: its largest magnitude by two lane exchanges, as integers (the order of
// non-negative floats, infinities and NaN on top). Bound by bytes: 16384 x 4096 in
// bf16 31 us, 5.4 TB/s; 32 x 4096 2.8 us of latency.

template <int DT>
__device__ __forceinline__ void Load8(const void* x, int64_t at, float (&v)[8]) {
  if constexpr (DT == EHIP_WEIGHT_F32) {
    const f32x4_t* p = reinterpret_cast<const f32x4_t*>(static_cast<const float*>(x) + at);
    const f32x4_t a = p[0], b = p[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
  } else {
    const i32x4_t a = __builtin_nontemporal_load(
        reinterpret_cast<const i32x4_t*>(static_cast<const uint16_t*>(x) + at));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = static_cast<uint32_t>(a[i]);
      if constexpr (DT == EHIP_WEIGHT_BF16) {
        v[2 * i] = Bf16Lo(w);
        v[2 * i + 1] = Bf16Hi(w);
      } else {
        v[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w)));
        v[2 * i + 1] =
            static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w >> 16)));
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

// Panels into fp32 rows. The same work split, but thread (r, i) has elements 4i
// and 64 + 4i of a tile, so that a store instruction writes whole 256-byte runs.
// Bound by bytes, stores mostly: 16384 x 4096 46 us, 6.6 TB/s.
__global__ __launch_bounds__(256) void MxDequantize(const uint16_t* codes, const uint32_t* scales,
                                                    int64_t rows, int64_t k, int32_t vec,
                                                    float* y) {
  const int r = threadIdx.x >> 4, i = threadIdx.x & 15;
  const int64_t tiles = (k + kMxTile - 1) / kMxTile;
  const int64_t groups = (tiles + kMxGroup - 1) / kMxGroup;
  const uint32_t bp = blockIdx.x / static_cast<uint32_t>(groups);
  const int64_t panel = bp, group = blockIdx.x - bp * static_cast<uint32_t>(groups);
  const int64_t row = panel * kMxRows + r;
  if (row >= rows) return;
  // All loads first (past the last tile: the last one's), then the values.
  uint32_t packed[2];
  uint16_t all[kMxGroup][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int lane = (2 * h + (i >> 3)) * 16 + r;
    packed[h] = scales[(panel * groups + group) * 64 + lane];
#pragma unroll
    for (int j = 0; j < kMxGroup; ++j) {
      const int64_t tile = min(group * kMxGroup + j, tiles - 1);
      all[j][h] = codes[((panel * tiles + tile) * 64 + lane) * 8 + (i & 7)];
    }
  }
#pragma unroll
  for (int j = 0; j < kMxGroup; ++j) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t k0 = (group * kMxGroup + j) * kMxTile + 64 * h + 4 * i;
      if (k0 >= k) continue;
      const uint32_t byte = (packed[h] >> (8 * j)) & 255u;
      f32x4_t v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // E2M1 as fp32: exponent 0 is m / 2, the others 2^(exponent - 1) (1 + m / 2).
        const uint32_t code = (uint32_t{all[j][h]} >> (4 * e)) & 15u, m = code & 7u;
        const float mag = m < 2u ? 0.5f * static_cast<float>(m)
                                 : __uint_as_float((126u + (m >> 1)) << 23 | (m & 1u) << 22);
        const float s = code & 8u ? -mag : mag;
        v[e] = byte == 255u ? __builtin_nanf("")
                            : __builtin_amdgcn_ldexpf(s, static_cast<int>(byte) - 127);
      }
      float* out = y + row * k + k0;
      if (vec) {  // k % 4 == 0
        __builtin_nontemporal_store(v, reinterpret_cast<f32x4_t*>(out));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k0 + e < k) out[e] = v[e];
      }
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

// Few rows: a workgroup per (MP x panels, one weight panel a projection), its KW
// wavefronts taking the scale groups in turn with their operands straight from
// memory into registers, a group ahead, then one sum over the wavefronts through
// LDS, in their order. FUSED (MP = 1): x is fp32 rows, which the workgroup
// quantises into LDS while its first weights are on their way. Bound by the
// weights' bytes and the latency of the few rounds that a workgroup has: 48 x 16384
// x 4096 9.7 us (36 MB), gated 1 x 4096 x 16384 13 (71 MB, 5.5 TB/s), 1 x 896 x 896
// 3.4, hardly more than a launch.
template <int MP, int ACT, int KW, bool FUSED>
__global__ __launch_bounds__(64 * KW) void MxDirect(MxGemmParams p) {
  static_assert(!FUSED || MP == 1, "fused quantisation of one panel");
  constexpr int PR = ACT != kPlain ? 2 : 1;
  __shared__ f32x4_t red[KW][MP * PR][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const uint32_t xb = blockIdx.x / static_cast<uint32_t>(p.w_panels);
  const int64_t wp = blockIdx.x - xb * static_cast<uint32_t>(p.w_panels);
  const int64_t xp0 = int64_t{xb} * MP;
  f32x4_t acc[MP][PR];
#pragma unroll
  for (int a = 0; a < MP; ++a)
#pragma unroll
    for (int b = 0; b < PR; ++b) acc[a][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // x panels past the last read the last one: their results are not stored.
  const i32x4_t* xc[MP];
  const uint32_t* xs[MP];
  const i32x4_t* wc[PR];
  const uint32_t* ws[PR];
#pragma unroll
  for (int a = 0; a < MP; ++a) {
    const int64_t panel = min(xp0 + a, p.x_panels - 1);
    xc[a] = reinterpret_cast<const i32x4_t*>(p.xc) + panel * p.tiles * 64 + lane;
    xs[a] = reinterpret_cast<const uint32_t*>(p.xs) + panel * p.groups * 64 + lane;
  }
#pragma unroll
  for (int b = 0; b < PR; ++b) {
    wc[b] = reinterpret_cast<const i32x4_t*>(p.wc[b]) + wp * p.tiles * 64 + lane;
    ws[b] = reinterpret_cast<const uint32_t*>(p.ws[b]) + wp * p.groups * 64 + lane;
  }
  const int row = lane & 15, block = lane >> 4;
  const bool live = row < p.m;
  // FUSED: codes [m][groups][16 blocks][16 bytes], then scales [m][groups][64
  // bytes] in the panels' order within a row (byte j of dword g).
  extern __shared__ __align__(16) uint32_t quant[];
  const int x_dwords = FUSED ? static_cast<int>(p.m) * p.groups * 64 : 0;

  i32x4_t x[kMxGroup][MP], w[kMxGroup][PR];
  uint32_t sx[MP], sw[PR];
  auto load_scales = [&](int t) __attribute__((always_inline)) {
    if constexpr (!FUSED) {
#pragma unroll
      for (int a = 0; a < MP; ++a) sx[a] = xs[a][int64_t{t} * 64];
    }
#pragma unroll
    for (int b = 0; b < PR; ++b) sw[b] = ws[b][int64_t{t} * 64];
  };
  auto load = [&](int t, int j) __attribute__((always_inline)) {
    const int64_t tile = min(t * kMxGroup + j, p.tiles - 1);
    if constexpr (!FUSED) {
#pragma unroll
      for (int a = 0; a < MP; ++a) x[j][a] = xc[a][tile * 64];
    }
#pragma unroll
    for (int b = 0; b < PR; ++b) w[j][b] = wc[b][tile * 64];
  };
  if (wave < p.groups) {
    load_scales(wave);
#pragma unroll
    for (int j = 0; j < kMxGroup; ++j) load(wave, j);
  }
  if constexpr (FUSED) {
    // Four threads a block, eight values each; blocks past k are zeros.
    for (int c = threadIdx.x; c < x_dwords; c += 64 * KW) {
      const int r = c / (p.groups * 64), in_row = c - r * (p.groups * 64);
      const int64_t k0 = int64_t{in_row} * 8;
      const float* src = p.x + r * p.k + k0;
      float v[8];
      if (p.x_vec && k0 + 8 <= p.k) {
        const f32x4_t a = reinterpret_cast<const f32x4_t*>(src)[0];
        const f32x4_t b = reinterpret_cast<const f32x4_t*>(src)[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k0 + e < p.k ? src[e] : 0.f;
      }
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
      const uint32_t byte = MxScaleByte(DppMax4(top));
      quant[c] = MxCodes(v, byte);
      const int blk = in_row / 4;  // in the row: group blk / 16, tile blk / 4 % 4, block blk % 4
      if ((c & 3) == 0)
        reinterpret_cast<uint8_t*>(quant + x_dwords)[((r * p.groups + blk / 16) * 4 + blk % 4) * 4 +
                                                     blk / 4 % 4] = static_cast<uint8_t>(byte);
    }
    __syncthreads();
  }
  for (int t = wave; t < p.groups; t += KW) {
    uint32_t cx[MP], cw[PR];
#pragma unroll
    for (int b = 0; b < PR; ++b) cw[b] = sw[b];
    if constexpr (FUSED) {
#pragma unroll
      for (int j = 0; j < kMxGroup; ++j)
        x[j][0] = live ? *reinterpret_cast<const i32x4_t*>(
                             quant + ((row * p.groups + t) * 16 + 4 * j + block) * 4)
                       : i32x4_t{0, 0, 0, 0};
      cx[0] = live ? quant[x_dwords + (row * p.groups + t) * 4 + block] : 0u;
    } else {
#pragma unroll
      for (int a = 0; a < MP; ++a) cx[a] = sx[a];
    }
    const bool more = t + KW < p.groups;
    if (more) load_scales(t + KW);
    auto step = [&](auto j) __attribute__((always_inline)) {
      constexpr int J = decltype(j)::value;
      if (t * kMxGroup + J < p.tiles) {
#pragma unroll
        for (int b = 0; b < PR; ++b)
#pragma unroll
          for (int a = 0; a < MP; ++a)
            acc[a][b] = MxMfma<J>(w[J][b], cw[b], x[J][a], cx[a], acc[a][b]);
      }
      if (more) load(t + KW, J);
    };
    step(std::integral_constant<int, 0>{});
    step(std::integral_constant<int, 1>{});
    step(std::integral_constant<int, 2>{});
    step(std::integral_constant<int, 3>{});
  }
#pragma unroll
  for (int a = 0; a < MP; ++a)
#pragma unroll
    for (int b = 0; b < PR; ++b) red[wave][a * PR + b][lane] = acc[a][b];
  __syncthreads();
  for (int f = wave; f < MP; f += KW) {
    f32x4_t s[PR];
#pragma unroll
    for (int h = 0; h < PR; ++h) {
      s[h] = red[0][f * PR + h][lane];
#pragma unroll 4
      for (int i = 1; i < KW; ++i) s[h] += red[i][f * PR + h][lane];
    }
    const int64_t col = wp * kMxRows + 4 * block;
    StoreRow4<0>(p, (xp0 + f) * kMxRows + row, col, Finish<ACT>(p, col, s[0], s[PR - 1]));
  }
}

// Many rows: a workgroup of WR x WC wavefronts per tile of WR XP x panels by WC WP
// weight panels (gated: their even slots the gate's, the odd ones the up
// projection's). k tiles go from memory straight into LDS (buffer_load ... lds, a
// panel's 1 KiB an instruction), into four buffers, three tiles ahead; an operand
// is one conflict-free 16-byte read. A wavefront's scales, one dword a panel and
// group, come through registers a group ahead. REG (WR = 1, where no two
// wavefronts share a weight panel): the weights go into registers instead, a tile
// ahead, which takes half of the traffic off LDS.
//
// Bound by the power the card may take, with the loads next: gated 4001 x 4096 x
// 16384 (1.07 TFLOP) takes 303 us at 1.98 GHz with the matrix cores busy 40% of
// them; without any loads it would be 216 us, and a loop of nothing but these
// products reaches 5.8 to 6.7 PFLOP/s on random codes (8.6 on zeros). Steps to it:
// 256 x 256 tiles of eight wavefronts 363, whole-line stores past the caches and
// 128 x 256 tiles, two workgroups a CU, 317, weights in registers 295 to 311.
template <int WR, int WC, int XP, int WP, bool REG, int ACT, int OCC>
__global__ __launch_bounds__(64 * WR * WC) __attribute__((amdgpu_waves_per_eu(OCC)))
void MxStaged(MxGemmParams p) {
  constexpr bool GATED = ACT != kPlain;
  constexpr int XT = WR * XP, WT = WC * WP;  // panels of the tile
  constexpr int LT = XT + (REG ? 0 : WT);  // of them through LDS
  constexpr int ND = LT / (WR * WC);       // panels a wavefront loads into it
  static_assert(ND * WR * WC == LT && WP % 2 == 0, "whole shares, pairs of slots");
  static_assert(!REG || WR == 1, "a wavefront's own weights");
  constexpr int kStage = LT * kMxTileBytes;
  constexpr int C = WP * (GATED ? 2 : 4);  // 16-byte chunks of a wavefront's row of results
  constexpr int kResults = WR * WC * C * 256;
  constexpr int kFirst = kStage > kResults ? kStage : kResults;
  // One array a buffer: the compiler then sees that a tile's loads and the reads
  // of another do not meet, and adds no wait of its own.
  __shared__ __align__(16) unsigned char b0[kFirst];
  __shared__ __align__(16) unsigned char b1[kStage];
  __shared__ __align__(16) unsigned char b2[kStage];
  __shared__ __align__(16) unsigned char b3[kStage];
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
  // Panels are a multiple of the tiles' 1 KiB apart, so with an even count of
  // tiles the reads of one k tile meet in few of the L2's channels (256 bytes
  // each in turn, 16 of them). Workgroups therefore take a group's tiles in
  // different orders, tile j ^ turn at step j, the scales' bytes moved alike.
  const uint32_t turns = p.tiles % 4 == 0 ? 3u : p.tiles % 2 == 0 ? 1u : 0u;
  const int turn = static_cast<int>((blockIdx.x >> 3) & turns);
  const uint32_t bytes = 0x03020100u ^ static_cast<uint32_t>(turn) * 0x01010101u;
  const int last_x = static_cast<int>(min(int64_t{XT}, p.x_panels - xp0)) - 1;
  const int last_w = static_cast<int>(min(int64_t{WT}, p.w_panels - wp0)) - 1;

  // The wavefront's panels of a stage. Panels past the last read the last one:
  // their results are not stored.
  const int64_t row_bytes = int64_t{p.tiles} * kMxTileBytes;
  const uint8_t* src[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    const int slot = ND * wave + i, w = slot - XT;
    src[i] = slot < XT ? p.xc + (xp0 + min(slot, last_x)) * row_bytes
                       : p.wc[GATED ? w & 1 : 0] +
                             (wp0 + min(GATED ? w / 2 : w, last_w)) * row_bytes;
  }
  const uint8_t* wsrc[REG ? WP : 1];
#pragma unroll
  for (int b = 0; b < (REG ? WP : 0); ++b) {
    const int w = wc * WP + b;
    wsrc[b] = p.wc[GATED ? w & 1 : 0] + (wp0 + min(GATED ? w / 2 : w, last_w)) * row_bytes;
  }
  i32x4_t wf[2][WP];
  auto load_w = [&](i32x4_t (&w)[WP], int t) __attribute__((always_inline)) {
    const uint32_t at = static_cast<uint32_t>(min(t ^ turn, p.tiles - 1)) * kMxTileBytes;
#pragma unroll
    for (int b = 0; b < (REG ? WP : 0); ++b)
      w[b] = __builtin_bit_cast(
          i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                       __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(wsrc[b]), 0,
                                                         0xFFFFFFFFu, 0x00020000),
                       lane * 16, at, 0));
  };
  auto stage = [&](unsigned char* buf, int t) __attribute__((always_inline)) {
    const uint32_t at = static_cast<uint32_t>(min(t ^ turn, p.tiles - 1)) * kMxTileBytes;
#pragma unroll
    for (int i = 0; i < ND; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(src[i]), 0, 0xFFFFFFFFu,
                                            0x00020000),
          (__attribute__((address_space(3))) void*)(buf + (ND * wave + i) * kMxTileBytes), 16,
          lane * 16, at, 0, 0);
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

  auto turned = [&](const uint32_t (&ax)[XP], const uint32_t (&aw)[WP])
                    __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < XP; ++a) sx[a] = __builtin_amdgcn_perm(0u, ax[a], bytes);
#pragma unroll
    for (int b = 0; b < WP; ++b) sw[b] = __builtin_amdgcn_perm(0u, aw[b], bytes);
  };
  load_scales(0, nx, nw);
  Fence();
  stage(b0, 0);
  Fence();
  if constexpr (REG) load_w(wf[0], 0);
  Fence();
  stage(b1, 1);
  Fence();
  stage(b2, 2);
  Fence();
  turned(nx, nw);
  auto compute = [&](auto j, const unsigned char* buf, i32x4_t (&w)[WP])
                     __attribute__((always_inline)) {
    constexpr int J = decltype(j)::value;
#pragma unroll
    for (int b = 0; b < (REG ? 0 : WP); ++b)
      w[b] = *reinterpret_cast<const i32x4_t*>(buf + (XT + wc * WP + b) * kMxTileBytes + lane * 16);
    // All operands on their way before the first product (the compiler would keep
    // two): gated 4001 x 4096 x 16384 311 -> 303 us.
    i32x4_t x[XP];
#pragma unroll
    for (int a = 0; a < XP; ++a)
      x[a] = *reinterpret_cast<const i32x4_t*>(buf + (wr * XP + a) * kMxTileBytes + lane * 16);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int a = 0; a < XP; ++a)
#pragma unroll
      for (int b = 0; b < WP; ++b) acc[a][b] = MxMfma<J>(w[b], sw[b], x[a], sx[a], acc[a][b]);
  };
  // Step t waits for its own tile's loads and meets the other wavefronts', then
  // loads tile t + 3 into the buffer that step t - 1 has read. The loads stay
  // unconditional (past the end: the last tile again), so that the counts hold:
  // behind a tile's loads are two more tiles', a set of weights or more, and, at
  // steps 1 and 2 of a group, the next group's scales, which step 0 loads before
  // its tile. True after the last tile.
  int g = 0;
  auto step = [&](auto s) __attribute__((always_inline)) {
    constexpr int J = decltype(s)::value;
    constexpr int kTiles = 2 * ND + (REG ? WP : 0);
    WaitAndMeet<(J == 1 || J == 2) ? kTiles + XP + WP : kTiles>();
    if constexpr (J == 0) {
      load_scales(g + 1, nx, nw);
      Fence();
    }
    stage(Buffer<(J + 3) % 4>(b0, b1, b2, b3), 4 * g + J + 3);
    Fence();  // the counts go by this order
    if constexpr (REG) load_w(wf[(J + 1) % 2], 4 * g + J + 1);
    Fence();
    compute(s, Buffer<J>(b0, b1, b2, b3), wf[REG ? J % 2 : 0]);
    return 4 * g + J + 1 >= p.tiles;
  };
  for (;; ++g) {
    if (step(std::integral_constant<int, 0>{})) break;
    if (step(std::integral_constant<int, 1>{})) break;
    if (step(std::integral_constant<int, 2>{})) break;
    if (step(std::integral_constant<int, 3>{})) break;
    turned(nx, nw);
  }

  // Loads past the end may still be in flight into the buffers: they land first.
  constexpr int kFit = kFirst / kResults, PP = kFit >= 4 ? 4 : kFit >= 2 ? 2 : 1;
  WaitAndMeet<0>();
  const int unscaled[XP] = {};
  StoreTile<XP, WP, PP, ACT, 0>(p, b0 + wave * (PP * C * 256), (xp0 + wr * XP) * kMxRows,
                                    (wp0 + (GATED ? wc * WP / 2 : wc * WP)) * kMxRows, acc,
                                    unscaled);
}

template <int WR, int WC, int XP, int WP, bool REG, int ACT, int OCC>
hipError_t LaunchStaged(MxGemmParams p, hipStream_t stream) {
  constexpr int64_t XT = WR * XP, WT = ACT != kPlain ? WC * WP / 2 : WC * WP;
  const int64_t rt = (p.x_panels + XT - 1) / XT, ct = (p.w_panels + WT - 1) / WT;
  if (rt * ct > (int64_t{1} << 30)) return hipErrorInvalidValue;
  p.row_tiles = static_cast<int32_t>(rt);
  p.col_tiles = static_cast<int32_t>(ct);
  const uint32_t grid = static_cast<uint32_t>((rt * ct + 7) / 8 * 8);
  hipLaunchKernelGGL((MxStaged<WR, WC, XP, WP, REG, ACT, OCC>), dim3(grid), dim3(64 * WR * WC), 0,
                     stream, p);
  return hipGetLastError();
}

template <int MP, int ACT, bool FUSED>
hipError_t LaunchDirect(const MxGemmParams& p, hipStream_t stream) {
  const int64_t n = p.w_panels * ((p.x_panels + MP - 1) / MP);
  if (n > INT32_MAX) return hipErrorInvalidValue;
  const dim3 grid(static_cast<uint32_t>(n));
  const uint32_t lds = FUSED ? static_cast<uint32_t>(p.m * p.groups) * 272u : 0u;
  // A wavefront a scale group, up to 16 (gated, with twice the operands, 8).
  constexpr int kMost = ACT != kPlain ? 8 : 16;
  if (kMost == 16 && p.groups > 8)
    hipLaunchKernelGGL((MxDirect<MP, ACT, kMost, FUSED>), grid, dim3(64 * kMost), lds, stream, p);
  else if (p.groups > 4)
    hipLaunchKernelGGL((MxDirect<MP, ACT, 8, FUSED>), grid, dim3(512), lds, stream, p);
  else if (p.groups > 2)
    hipLaunchKernelGGL((MxDirect<MP, ACT, 4, FUSED>), grid, dim3(256), lds, stream, p);
  else
    hipLaunchKernelGGL((MxDirect<MP, ACT, 2, FUSED>), grid, dim3(128), lds, stream, p);
  return hipGetLastError();
}

// Which kernel, by how many workgroups of each there are (us, this kernel / the
// next one tried, four weight sets in turn):
//   direct, up to 64 rows or 512 workgroups (two a CU): 96 x 4096 x 4096 6.3 / 8.4,
//     128 x 16384 x 4096 20 / 24; past it 200 x 4096 x 4096 10.1 / 8.9.
//   64 x 64 tiles, up to 896 (3.5 a CU): 512 x 4096 x 4096 11.1 / 15.5, gated 500 x
//     896 x 3584 6.9 / 7.8; past it 1024 x 4096 x 4096 20.0 / 17.5.
//   128 x 256 tiles, from 448 of them (1.75 a CU) over 16 k tiles and more: gated
//     4001 x 4096 x 16384 288 / 307, 512 rows 42.3 / 45.3; below, 2382 x 4096 x 4096
//     34.3 / 30.7, and gated 4001 x 896 x 3584 28.1 / 26.2.
//   128 x 128 tiles, three workgroups a CU, between; with the weights in registers,
//     as the 128 x 256 ones: 2382 x 4096 x 4096 31.6, through LDS 34.7, 4096 x
//     4096 x 16384 151 and 156.
template <int ACT>
hipError_t LaunchProduct(const MxGemmParams& p, hipStream_t stream) {
  if (p.x) return LaunchDirect<1, ACT, true>(p, stream);
  const int64_t slots = p.w_panels * (ACT != kPlain ? 2 : 1);
  auto tiles = [&](int64_t x, int64_t w) {
    return (p.x_panels + x - 1) / x * ((slots + w - 1) / w);
  };
  if (p.x_panels <= 4 || (p.x_panels + 3) / 4 * p.w_panels <= 512) {
    switch (p.x_panels) {
      case 1: return LaunchDirect<1, ACT, false>(p, stream);
      case 2: return LaunchDirect<2, ACT, false>(p, stream);
      case 3: return LaunchDirect<3, ACT, false>(p, stream);
      default: return LaunchDirect<4, ACT, false>(p, stream);
    }
  }
  if (tiles(4, 4) <= 896) return LaunchStaged<2, 2, 2, 2, false, ACT, 4>(p, stream);
  if (tiles(8, 16) >= 448 && p.tiles >= 16)
    return LaunchStaged<1, 4, 8, 4, true, ACT, 2>(p, stream);
  return LaunchStaged<1, 4, 8, 2, true, ACT, 3>(p, stream);
}

// Workgroups of the panel conversions, 0 where a launch cannot hold them.
uint32_t MxConvertGrid(int64_t rows, int64_t k) {
  const int64_t n = MxPanels(rows) * MxGroups(k);
  return n <= UINT32_MAX / 256 ? static_cast<uint32_t>(n) : 0u;
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
  const int32_t vec = k % 4 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
  if (grid.x == 0) return hipErrorInvalidValue;
  hipLaunchKernelGGL(MxDequantize, grid, dim3(256), 0, stream,
                     static_cast<const uint16_t*>(codes), static_cast<const uint32_t*>(scales),
                     rows, k, vec, y);
  return hipGetLastError();
}

// Up to 4 rows, as far as LDS holds them twice and more: gated 4096 x 16384 takes 13
// us for one row, 17 for 4, where a launch of its own and the product are 16.5.
bool MxFusesQuantization(int64_t m, int64_t k) { return m <= 4 && m * MxGroups(k) * 272 <= 32768; }

hipError_t LaunchMxGemm(const MxGemmParams& p, bool gated, hipStream_t stream) {
  if (!gated) return LaunchProduct<kPlain>(p, stream);
  switch (p.act) {
    case EHIP_ACT_SILU: return LaunchProduct<EHIP_ACT_SILU>(p, stream);
    case EHIP_ACT_GELU: return LaunchProduct<EHIP_ACT_GELU>(p, stream);
    default: return LaunchProduct<EHIP_ACT_GELU_TANH>(p, stream);
  }
}

}  // namespace ehip
