// The gated feed-forward block over packed weights, both projections, the
// activation and the product in one kernel:
//   y[m, n] = act(x Wg^T + bg) * (x Wu^T + bu),
// x fp32, the weights fp32, bf16 or fp16 in panels [ceil(n/16), k, 16].
//
// GatedStream, for a few rows, reads the panels once and multiplies in fp32 on the
// vector ALUs; GatedDirect, for small calls, in fp32 on the matrix cores.
// GatedStaged, for the others, is on the 16-bit matrix cores: beside bf16 weights
// x is cut into three bf16 planes whose sum is the value to 2^-24. Beside fp16 and
// fp32 weights it is two fp16 planes, the value to 2^-23, after a power of two per
// row that brings the row's largest magnitude to 2^14; fp32 weights are cut alike,
// by rows, and for many rows bf16 ones become one fp16 plane, exact down to 2^-31
// of the row's largest. Products x_i w_j but that of both second planes, smallest
// first, fp32 sums: three matrix-core products a term for bf16 and fp32 weights, two
// for fp16 and for bf16 as fp16. What fp16 planes leave out is below 2^-23 of
// |x||w| a term and 2^-39 of the row's largest |x| times |w|; with fp32 weights
// below 2^-21 at worst, for all of it, in the mean square some 2^-24, where a term
// of fp32 arithmetic loses 2^-25 and the k fp32 sums that follow sqrt(k) 2^-25.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "kernels.h"
#include "staged.h"

namespace ehip {
namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
typedef __attribute__((ext_vector_type(2))) short s16x2_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((ext_vector_type(8))) short s16x8_t;

constexpr int kStreamRows = 8;  // up to these: GatedStream
constexpr int kMostSplits = 8;  // of a tile's steps

constexpr int kRows = 16;   // rows of a panel, of x or a weight
constexpr int kStep = 32;   // k of a step

// A kernel's kind of weight: EHIP_WEIGHT_*, or bf16 taken as fp16.
constexpr int kBf16AsF16 = 3;

template <int WT>
struct Type;
template <>
struct Type<kBf16AsF16> {
  using T = uint16_t;
  static constexpr int XPL = 2, WPL = 1;
  static constexpr bool kHalf = true, kCols = true;
};
template <>
struct Type<EHIP_WEIGHT_F32> {
  using T = float;
  static constexpr int XPL = 2, WPL = 2;  // planes of x and of a weight
  static constexpr bool kHalf = true;     // planes of fp16, x's rows scaled
  static constexpr bool kCols = true;     // and the weights' rows
};
template <>
struct Type<EHIP_WEIGHT_BF16> {
  using T = uint16_t;
  static constexpr int XPL = 3, WPL = 1;
  static constexpr bool kHalf = false, kCols = false;
};
template <>
struct Type<EHIP_WEIGHT_F16> {
  using T = uint16_t;
  static constexpr int XPL = 2, WPL = 1;
  static constexpr bool kHalf = true, kCols = false;
};

// A lane (n16, q) of a matrix-core operand holds eight k of a 32-k step: 4q..4q+3
// and 16+4q..16+4q+3, what two transposed LDS reads of 16-bit panel rows give;
// q, q+4, .. q+28 for fp32 panel rows, whose single reads then meet no bank twice.
template <int WT>
__device__ __forceinline__ int OperandK(int q, int e) {
  return WT == EHIP_WEIGHT_F32 ? q + 4 * e : 4 * q + (e & 3) + 16 * (e >> 2);
}

// v cut into planes: each the nearest 16-bit value of what the earlier ones leave.
template <int WT>
__device__ __forceinline__ void Cut(float v, short (&out)[Type<WT>::XPL]) {
#pragma unroll
  for (int i = 0; i < Type<WT>::XPL; ++i) {
    if constexpr (Type<WT>::kHalf) {
      const _Float16 h = static_cast<_Float16>(v);
      out[i] = __builtin_bit_cast(short, h);
      v -= static_cast<float>(h);
    } else {
      const __bf16 h = static_cast<__bf16>(v);
      out[i] = __builtin_bit_cast(short, h);
      v -= static_cast<float>(h);
    }
  }
}

// The lane exchange CTRL (device_util.h) of an integer.
template <int CTRL>
__device__ __forceinline__ uint32_t Moved(uint32_t v) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, false));
}

// The largest of the wavefront's, as integers: the order of non-negative floats,
// NaN and infinities on top.
__device__ __forceinline__ uint32_t Over16And32(uint32_t v) {
  v = max(v, __float_as_uint(ShflXor(__uint_as_float(v), 16)));
  return max(v, __float_as_uint(ShflXor(__uint_as_float(v), 32)));
}
__device__ __forceinline__ uint32_t Magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
// The power of two that brings this magnitude to [2^14, 2^15); infinities and NaN
// stay.
__device__ __forceinline__ int Exponent(uint32_t top) {
  const int f = static_cast<int>(top >> 23);
  return f == 255 ? 0 : 14 + 127 - f;
}

// Column scales of a weight's panel: a thread takes 16 bytes of every 256th row
// (16-bit weights: 512th).
template <int WT>
__device__ __forceinline__ void ScalePanel(const GatedParams& p, int64_t which, uint32_t* tops) {
  constexpr bool kF32 = WT == EHIP_WEIGHT_F32;
  constexpr int V = kF32 ? 4 : 8, L = kRows / V;  // columns of a thread, threads of a row
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t part = which >= p.w_panels, panel = which - part * p.w_panels;
  const i32x4_t* const from =
      reinterpret_cast<const i32x4_t*>(p.wp[part]) + panel * p.k * L;
  uint32_t top[V] = {};
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < p.k * L; i += 1024) {
    const i32x4_t a = from[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t u = static_cast<uint32_t>(a[e]);
      if constexpr (kF32) {
        top[e] = max(top[e], u & 0x7FFFFFFFu);
      } else {
        top[2 * e] = max(top[2 * e], u << 16 & 0x7FFFFFFFu);
        top[2 * e + 1] = max(top[2 * e + 1], u & 0x7FFF0000u);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if constexpr (L == 2) top[e] = max(top[e], Moved<0x122>(top[e]));
    top[e] = max(top[e], Moved<0x124>(top[e]));
    top[e] = Over16And32(max(top[e], Moved<0x128>(top[e])));
    if (lane < L) tops[wave * kRows + V * lane + e] = top[e];
  }
  __syncthreads();
  if (threadIdx.x < kRows) {
    uint32_t most = 0;
    for (int w = 0; w < 16; ++w) most = max(most, tops[w * kRows + threadIdx.x]);
    p.col_scale[part * p.col_stride + panel * kRows + threadIdx.x] = -Exponent(most);
  }
}

// x [m, k] into operand panels [panels][steps][planes][64 lanes][8]: zero past m
// and k. A workgroup takes `chunk` steps of a panel, a wavefront a step at a time;
// for planes of fp16 every workgroup of a panel first finds its rows' largest
// magnitudes. Beside fp32 weights, and bf16 ones as fp16, further workgroups find
// those of the weights' rows. Bound by bytes, small calls by latency: 2382 x 4096
// 21 us (97 MB, 4.6 TB/s), 48 x 4096 5; with 2 x 16384 x 4096 bf16 weights 68 (365
// MB, 5.4 TB/s), fp32 ones 102.
template <int WT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void CutRows(GatedParams p, int chunk, int cuts) {
  constexpr int PL = Type<WT>::XPL;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  if constexpr (Type<WT>::kCols) {
    static_assert(!Type<WT>::kCols || WAVES == 16, "ScalePanel's");
    __shared__ uint32_t tops[WAVES * kRows];
    if (static_cast<int>(blockIdx.x) >= cuts) return ScalePanel<WT>(p, blockIdx.x - cuts, tops);
  }
  const uint32_t part = blockIdx.x / static_cast<uint32_t>(p.x_panels);
  const int64_t panel = blockIdx.x - part * static_cast<uint32_t>(p.x_panels);
  const int64_t row = panel * kRows + r;
  const float* const src = p.x + (row < p.m ? row : 0) * p.k;
  int up = 0;
  if constexpr (Type<WT>::kHalf) {
    // A wavefront a row.
    static_assert(!Type<WT>::kHalf || WAVES == kRows, "a wavefront a row");
    __shared__ int scale[kRows];
    const int mine = threadIdx.x >> 6;
    const int64_t at = panel * kRows + mine;
    uint32_t top = 0;
    if (at < p.m) {
      const float* const from = p.x + at * p.k;
      if (p.x_vec) {
#pragma unroll 4
        for (int64_t kk = 4 * lane; kk < p.k; kk += 256) {
          const f32x4_t a = *reinterpret_cast<const f32x4_t*>(from + kk);
#pragma unroll
          for (int e = 0; e < 4; ++e) top = max(top, Magnitude(a[e]));
        }
      } else {
#pragma unroll 4
        for (int64_t kk = lane; kk < p.k; kk += 64) top = max(top, Magnitude(from[kk]));
      }
    }
    top = max(top, Moved<0xB1>(top));
    top = max(top, Moved<0x4E>(top));
    top = max(top, Moved<0x141>(top));
    top = Over16And32(max(top, Moved<0x128>(top)));
    if (lane == 0) scale[mine] = Exponent(top);
    __syncthreads();
    up = scale[r];
    if (part == 0 && threadIdx.x < kRows) p.row_scale[row] = -up;
  }
  const int64_t s0 = int64_t{part} * chunk, s1 = min(s0 + chunk, p.steps);
  for (int64_t s = s0 + (threadIdx.x >> 6); s < s1; s += WAVES) {
    float v[8];
    if constexpr (WT == EHIP_WEIGHT_F32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int64_t kk = s * kStep + OperandK<WT>(q, e);
        v[e] = row < p.m && kk < p.k ? src[kk] : 0.f;
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t kk = s * kStep + 16 * h + 4 * q;
        if (p.x_vec && row < p.m && kk + 4 <= p.k) {
          const f32x4_t a = *reinterpret_cast<const f32x4_t*>(src + kk);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * h + e] = a[e];
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * h + e] = row < p.m && kk + e < p.k ? src[kk + e] : 0.f;
        }
      }
    }
    s16x8_t out[PL];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      short parts[PL];
      if constexpr (Type<WT>::kHalf)
        Cut<WT>(__builtin_amdgcn_ldexpf(v[e], up), parts);
      else
        Cut<WT>(v[e], parts);
#pragma unroll
      for (int i = 0; i < PL; ++i) out[i][e] = parts[i];
    }
#pragma unroll
    for (int i = 0; i < PL; ++i)
      reinterpret_cast<s16x8_t*>(p.xp)[((panel * p.steps + s) * PL + i) * 64 + lane] = out[i];
  }
}

// ds_read_b64_tr_b16: lane i of each 16-lane group receives element i % 4 of
// the 8 bytes addressed by lanes 4j + i / 4 of the group, for j = 0..3.
__device__ __forceinline__ s16x4_t TransposedRead(const unsigned char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(p));
}

template <int WT>
__device__ __forceinline__ f32x4_t Mfma(s16x8_t w, s16x8_t x, f32x4_t acc) {
  if constexpr (Type<WT>::kHalf)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, w),
                                                  __builtin_bit_cast(f16x8_t, x), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w),
                                                   __builtin_bit_cast(bf16x8_t, x), acc, 0, 0, 0);
}

// One KiB of every step that a wavefront brings into LDS: from src + t stride
// (zeros past `size` bytes) to `at` of the step's buffer.
struct Unit {
  const unsigned char* src;
  uint32_t size, stride, at;
};
__device__ __forceinline__ void LoadUnit(const Unit& u, unsigned char* buf, uint32_t t, int lane) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<unsigned char*>(u.src), 0, u.size, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      r, (__attribute__((address_space(3))) void*)(buf + u.at), 16, lane * 16 + t * u.stride, 0, 0,
      0);
}

// A workgroup of WR x WC wavefronts per tile of WR XP panels of x by WC WP weight
// slots (slot 2j the gate's panel j, 2j + 1 the up projection's). A step's x
// planes and panel rows go from memory straight into LDS (buffer_load ... lds, 1
// KiB units shared out over the wavefronts), NS - 1 steps
// ahead. The weight is the A operand and x the B operand: a lane's four results
// are four columns of one row of y. Bound by the power the card may take at many
// rows (bf16 as fp16, 2382 x 4096 x 16384, 1.28 PFLOP of products in 1100 us; three
// bf16 planes 1.92 in 1313 at 1.7 GHz, where the matrix cores are busy 72% of the
// cycles), by the panels' way through L2 at some hundred. p.splits > 1: a workgroup
// takes a part of the steps and leaves its sums, fragment by fragment, to
// GatedMerge.
template <int WT, int WR, int WC, int XP, int WP, int NS, int ACT, int OCC>
__global__ __launch_bounds__(64 * WR * WC) __attribute__((amdgpu_waves_per_eu(OCC)))
void GatedStaged(GatedParams p) {
  using T = typename Type<WT>::T;
  constexpr int XPL = Type<WT>::XPL, WPL = Type<WT>::WPL, WU = sizeof(T) / 2;
  constexpr int XT = WR * XP, SL = WC * WP;     // panels of x, weight slots of the tile
  constexpr int kXUnits = XT * XPL, kUnits = kXUnits + SL * WU;
  constexpr int ND = (kUnits + WR * WC - 1) / (WR * WC);  // units a wavefront loads
  constexpr int kStage = kUnits * 1024, C = WP * 2;
  constexpr int kResults = WR * WC * C * 256;
  constexpr int kFirst = kStage > kResults ? kStage : kResults;
  __shared__ __align__(16) unsigned char b0[kFirst];
  __shared__ __align__(16) unsigned char b1[kStage];
  __shared__ __align__(16) unsigned char b2[NS > 2 ? kStage : 16];
  __shared__ __align__(16) unsigned char b3[NS > 3 ? kStage : 16];
  const int lane = threadIdx.x & 63, n16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int wr = wave / WC, wc = wave % WC;

  // Tiles in bands of 4 rows of tiles, columns outer within a band; an XCD (b
  // mod 8) takes consecutive ones, which share their panels in its L2.
  const uint32_t tiles_all = static_cast<uint32_t>(p.row_tiles) * p.col_tiles;
  const uint32_t work = tiles_all * p.splits, per = (work + 7) / 8;
  const uint32_t item = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (item >= work) return;
  const uint32_t split = item / tiles_all, tile = item - split * tiles_all;
  const uint32_t band = tile / (4u * p.col_tiles);
  const uint32_t in_band = tile - band * 4u * p.col_tiles;
  const uint32_t h = min(4u, static_cast<uint32_t>(p.row_tiles) - 4u * band);
  const int ct = __builtin_amdgcn_readfirstlane(in_band / h);
  const int rt = __builtin_amdgcn_readfirstlane(4 * band + in_band % h);
  const int64_t xp0 = int64_t{rt} * XT, wp0 = int64_t{ct} * (SL / 2);
  const int last_x = static_cast<int>(min(int64_t{XT}, p.x_panels - xp0)) - 1;
  const int last_w = static_cast<int>(min(int64_t{SL / 2}, p.w_panels - wp0)) - 1;

  // The wavefront's units. Panels past the last read the last one: their results
  // are not stored. A unit's memory ends with its panel, so that what lies past k
  // and past the last step reads as zeros.
  const int steps = static_cast<int>(p.steps);
  const uint32_t panel_bytes = static_cast<uint32_t>(p.k * kRows * sizeof(T));
  Unit units[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    const int u = min(ND * wave + i, kUnits - 1);
    units[i].at = static_cast<uint32_t>(u) * 1024u;
    uint32_t first, bytes;
    if (u < kXUnits) {
      const int panel = u / XPL;
      first = static_cast<uint32_t>(u % XPL) * 1024u;
      bytes = static_cast<uint32_t>(steps) * (XPL * 1024u);
      units[i].stride = XPL * 1024;
      units[i].src = reinterpret_cast<const unsigned char*>(p.xp) +
                     (xp0 + min(panel, last_x)) * static_cast<int64_t>(bytes) + first;
    } else {
      const int slot = (u - kXUnits) / WU;
      first = static_cast<uint32_t>((u - kXUnits) % WU) * 1024u;
      bytes = panel_bytes;
      units[i].stride = WU * 1024;
      units[i].src = static_cast<const unsigned char*>(p.wp[slot & 1]) +
                     (wp0 + min(slot / 2, last_w)) * static_cast<int64_t>(bytes) + first;
    }
    units[i].size = bytes - min(bytes, first);
    if constexpr (WT == EHIP_WEIGHT_F32) {  // in scalar registers, as the other types' are
      const uint64_t src = reinterpret_cast<uint64_t>(units[i].src);
      const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(src));
      const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(src >> 32));
      units[i].src = reinterpret_cast<const unsigned char*>(uint64_t{hi} << 32 | lo);
      units[i].size = __builtin_amdgcn_readfirstlane(units[i].size);
    }
  }
  // The steps of the workgroup's part, from a place of its own on and round: panels
  // are a power of two apart for usual k, and workgroups at one step of different
  // panels would meet in few of the memory's channels (a split 48 x 4096 x 16384
  // 70 -> 64 us; whole tiles much the same).
  const int s0 = __builtin_amdgcn_readfirstlane(split * p.split_steps);
  const int count = min(p.split_steps, steps - s0);
  const int turn = ct % count;
  auto stage = [&](unsigned char* buf, int t) __attribute__((always_inline)) {
    int at = t + turn;
    at = at >= count ? at - count : at;
    at = s0 + min(at, count - 1);  // past the end: any step, its sums are not taken
#pragma unroll
    for (int i = 0; i < ND; ++i)
      LoadUnit(units[i], buf, static_cast<uint32_t>(at), lane);
  };

  f32x4_t acc[XP][WP];
#pragma unroll
  for (int a = 0; a < XP; ++a)
#pragma unroll
    for (int b = 0; b < WP; ++b) acc[a][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  int up[WP];  // kCols: the powers of two of the lane's columns
  if constexpr (Type<WT>::kCols) {
#pragma unroll
    for (int b = 0; b < WP; ++b)
      up[b] = -p.col_scale[(b & 1) * p.col_stride +
                           (wp0 + min((wc * WP + b) / 2, last_w)) * kRows + n16];
  }

  auto compute = [&](const unsigned char* buf) __attribute__((always_inline)) {
    s16x8_t x[XP][XPL];
#pragma unroll
    for (int a = 0; a < XP; ++a)
#pragma unroll
      for (int i = 0; i < XPL; ++i)
        x[a][i] = *reinterpret_cast<const s16x8_t*>(buf + ((wr * XP + a) * XPL + i) * 1024 +
                                                    lane * 16);
#pragma unroll
    for (int b = 0; b < WP; ++b) {
      const unsigned char* const base = buf + (kXUnits + (wc * WP + b) * WU) * 1024;
      s16x8_t w[WPL];
      if constexpr (WT == EHIP_WEIGHT_F32) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {  // in pairs, as the conversions go
          const float* const at = reinterpret_cast<const float*>(base) + n16;
          const f32x2_t v = {__builtin_amdgcn_ldexpf(at[OperandK<WT>(q, e) * kRows], up[b]),
                             __builtin_amdgcn_ldexpf(at[OperandK<WT>(q, e + 1) * kRows], up[b])};
          const f16x2_t h = __builtin_convertvector(v, f16x2_t);
          const f32x2_t left = {__builtin_fmaf(static_cast<float>(h[0]), -1.f, v[0]),
                                __builtin_fmaf(static_cast<float>(h[1]), -1.f, v[1])};
          const s16x2_t hi = __builtin_bit_cast(s16x2_t, h);
          const s16x2_t lo = __builtin_bit_cast(s16x2_t, __builtin_convertvector(left, f16x2_t));
          w[0][e] = hi[0], w[0][e + 1] = hi[1];
          w[1][e] = lo[0], w[1][e + 1] = lo[1];
        }
      } else {
        const unsigned char* const at = base + ((4 * q + (n16 >> 2)) * kRows + 4 * (n16 & 3)) * 2;
        w[0] = __builtin_shufflevector(TransposedRead(at), TransposedRead(at + 16 * kRows * 2), 0,
                                       1, 2, 3, 4, 5, 6, 7);
        if constexpr (WT == kBf16AsF16) {
          const i32x4_t two = __builtin_bit_cast(i32x4_t, w[0]);
          i32x4_t halves;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t u = static_cast<uint32_t>(two[e]);
            const f32x2_t v = {__builtin_amdgcn_ldexpf(Bf16Lo(u), up[b]),
                               __builtin_amdgcn_ldexpf(Bf16Hi(u), up[b])};
            halves[e] = __builtin_bit_cast(int, __builtin_convertvector(v, f16x2_t));
          }
          w[0] = __builtin_bit_cast(s16x8_t, halves);
        }
      }
      // Products x_i w_j with i + j < planes of x, smallest first.
#pragma unroll
      for (int s = XPL - 1; s >= 0; --s)
#pragma unroll
        for (int j = 0; j < WPL; ++j)
          if (s - j >= 0) {
#pragma unroll
            for (int a = 0; a < XP; ++a) acc[a][b] = Mfma<WT>(w[j], x[a][s - j], acc[a][b]);
          }
    }
  };

  // Step t waits for its own loads and meets the other wavefronts', then
  // loads step t + NS - 1 into the buffer that step t - 1 has read. The loads stay
  // unconditional (past the end: zeros), so that the count holds.
  stage(b0, 0);
  Fence();
  if constexpr (NS > 2) stage(b1, 1);
  Fence();
  if constexpr (NS > 3) stage(b2, 2);
  Fence();
  if constexpr (Type<WT>::kCols) {
#pragma unroll
    for (int b = 0; b < WP; ++b) asm volatile("" : "+v"(up[b]));  // waits here, not in the loop
  }
  int t = 0;
  auto step = [&](auto s) __attribute__((always_inline)) {
    constexpr int S = decltype(s)::value;
    WaitAndMeet<(NS - 2) * ND>();
    stage(Buffer<(S + NS - 1) % NS>(b0, b1, b2, b3), t + NS - 1);
    Fence();
    compute(Buffer<S % NS>(b0, b1, b2, b3));
    return ++t >= count;
  };
  for (;;) {
    if (step(std::integral_constant<int, 0>{})) break;
    if (step(std::integral_constant<int, 1>{})) break;
    if (step(std::integral_constant<int, 2>{})) break;
    if constexpr (NS != 3)
      if (step(std::integral_constant<int, 3>{})) break;
  }
  // Loads past the end may still be in flight into the buffers: they land first.
  constexpr int kFit = kFirst / kResults, PP = kFit >= 4 && XP % 4 == 0   ? 4
                                                   : kFit >= 2 && XP % 2 == 0 ? 2
                                                                              : 1;
  WaitAndMeet<0>();
  if (p.splits > 1) {
    f32x4_t* const to = reinterpret_cast<f32x4_t*>(p.part) +
                        (int64_t{item} * (WR * WC) + wave) * (XP * WP * 64) + lane;
#pragma unroll
    for (int a = 0; a < XP; ++a)
#pragma unroll
      for (int b = 0; b < WP; ++b) to[(a * WP + b) * 64] = acc[a][b];
    return;
  }
  int down[XP];
#pragma unroll
  for (int a = 0; a < XP; ++a)
    down[a] = Type<WT>::kHalf
                  ? p.row_scale[(xp0 + min(wr * XP + a, last_x)) * kRows + n16]
                  : 0;
  StoreTile<XP, WP, PP, ACT, Type<WT>::kCols ? 2 : Type<WT>::kHalf>(
      p, b0 + wave * (PP * C * 256), (xp0 + wr * XP) * kRows, (wp0 + wc * WP / 2) * kRows, acc,
      down);
}

// The split tiles of one row of wavefronts (WR = 1): their sums in split order,
// then what the staged kernel does with whole ones. A workgroup takes a panel of x
// and, in each of a tile's wavefronts' parts, a gate and its up panel: few tiles
// are split many ways, and their sums come from memory side by side (48 x 2048 x
// 2048, 16 tiles in 8 parts, with a workgroup a tile 29.5 us in all).
template <int WT, int WC, int XP, int WP, int ACT>
__global__ __launch_bounds__(64 * WC) void GatedMerge(GatedParams p) {
  const int lane = threadIdx.x & 63, n16 = lane & 15, q = lane >> 4;
  const int wave = static_cast<int>(threadIdx.x >> 6);
  const uint32_t tiles = static_cast<uint32_t>(p.row_tiles) * p.col_tiles;
  const uint32_t tile = blockIdx.x / (XP * (WP / 2)), rest = blockIdx.x - tile * (XP * (WP / 2));
  const uint32_t a = rest / (WP / 2), b = rest - a * (WP / 2);
  // The staged kernel's order of tiles.
  const uint32_t band = tile / (4u * p.col_tiles);
  const uint32_t in_band = tile - band * 4u * p.col_tiles;
  const uint32_t h = min(4u, static_cast<uint32_t>(p.row_tiles) - 4u * band);
  const int64_t row = (int64_t{4 * band + in_band % h} * XP + a) * kRows + n16;
  const int64_t col = (int64_t{in_band / h} * (WC * WP / 2) + wave * WP / 2 + b) * kRows + 4 * q;
  if (row >= p.m) return;
  const int64_t stride = int64_t{tiles} * WC * XP * WP * 64;
  const int64_t block = (int64_t{tile} * WC + wave) * (XP * WP) + a * WP + 2 * b;
  const f32x4_t* const from = reinterpret_cast<const f32x4_t*>(p.part) + block * 64 + lane;
  f32x4_t g[kMostSplits], u[kMostSplits];
#pragma unroll
  for (int i = 0; i < kMostSplits; ++i) {
    const int64_t at = min(i, p.splits - 1) * stride;
    g[i] = from[at];
    u[i] = from[at + 64];
  }
#pragma unroll
  for (int i = 1; i < kMostSplits; ++i)
    if (i < p.splits) {
      g[0] += g[i];
      u[0] += u[i];
    }
  if constexpr (Type<WT>::kHalf) Rescale<Type<WT>::kCols>(p, col, p.row_scale[row], &g[0], &u[0]);
  StoreRow4<0>(p, row, col, Finish<ACT>(p, col, g[0], u[0]));
}

// Few rows (m <= MR): a workgroup per (panel, gate and up), its KW wavefronts
// taking k in turn. A lane reads 16 bytes of a panel row (columns 8h.. of row k;
// 4h.. in fp32) and multiplies them by x's MR values at that k, in fp32, into
// sums of its own. Sums of different values change places between the halves and
// the rows of the wavefront, so that a step adds two of them at once; then a
// row's lanes of a column by rotations; the wavefronts meet in LDS, in order.
// Bound by the panels' bytes: 1 x 4096 x 16384 in bf16 44.7 us, 6.0 TB/s.
template <int WT, int MR, int KW, int U, int ACT>
__global__ __launch_bounds__(64 * KW) void GatedStream(GatedParams p) {
  using T = typename Type<WT>::T;
  constexpr int V = 16 / sizeof(T);        // columns of a lane
  constexpr int L = kRows / V;             // lanes of a panel row
  constexpr int KR = 64 / L;               // k rows of a wavefront's read
  __shared__ float red[KW][2][MR][kRows];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int kr = lane / L, h = lane % L;
  const int64_t panel = blockIdx.x;
  const T* const w0 = static_cast<const T*>(p.wp[0]) + panel * p.k * kRows;
  const T* const w1 = static_cast<const T*>(p.wp[1]) + panel * p.k * kRows;
  float acc[2][MR][V];
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int r = 0; r < MR; ++r)
#pragma unroll
      for (int c = 0; c < V; ++c) acc[g][r][c] = 0.f;
  auto widen = [&](const i32x4_t& a, float (&v)[V]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = static_cast<uint32_t>(a[i]);
      if constexpr (WT == EHIP_WEIGHT_F32) {
        v[i] = __uint_as_float(u);
      } else if constexpr (WT == EHIP_WEIGHT_BF16) {
        v[2 * i] = Bf16Lo(u);
        v[2 * i + 1] = Bf16Hi(u);
      } else {
        v[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(u)));
        v[2 * i + 1] =
            static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(u >> 16)));
      }
    }
  };
  for (int64_t k0 = int64_t{wave} * (KR * U); k0 < p.k; k0 += KW * KR * U) {
    i32x4_t a[U][2];
    float x[U][MR];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t kk = k0 + u * KR + kr;
      const bool in = kk < p.k;
      const int64_t at = (in ? kk : 0) * kRows + h * V;
      a[u][0] = __builtin_nontemporal_load(reinterpret_cast<const i32x4_t*>(w0 + at));
      a[u][1] = __builtin_nontemporal_load(reinterpret_cast<const i32x4_t*>(w1 + at));
      if (!in) a[u][0] = a[u][1] = i32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int r = 0; r < MR; ++r)
        x[u][r] = in && r < p.m ? p.x[r * p.k + kk] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float v[V];
        widen(a[u][g], v);
#pragma unroll
        for (int r = 0; r < MR; ++r)
#pragma unroll
          for (int c = 0; c < V; ++c) acc[g][r][c] = __builtin_fmaf(x[u][r], v[c], acc[g][r][c]);
      }
  }
  // Value v = (g MR + r) V + c. After the two exchanges register j of the lanes in
  // half b5 and odd or even row b4 holds value 4 j + 2 b4 + b5.
  constexpr int N = 2 * MR * V;
  float half[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const int v = 2 * i;
    const auto s = __builtin_amdgcn_permlane32_swap(
        __float_as_uint(acc[v / (MR * V)][v / V % MR][v % V]),
        __float_as_uint(acc[(v + 1) / (MR * V)][(v + 1) / V % MR][(v + 1) % V]), false, false);
    half[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(half[2 * j]),
                                                    __float_as_uint(half[2 * j + 1]), false, false);
    float t = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    t += Dpp<0x128>(t);
    t += Dpp<0x124>(t);
    if constexpr (L == 2) t += Dpp<0x122>(t);
    if ((lane & 15) < L) {
      const int v = 4 * j + 2 * ((lane >> 4) & 1) + (lane >> 5);
      red[wave][v / (MR * V)][v / V % MR][h * V + v % V] = t;
    }
  }
  __syncthreads();
  // Thread (row, column) of the panel's results.
  for (int i = threadIdx.x; i < MR * kRows; i += 64 * KW) {
    const int r = i / kRows, c = i % kRows;
    const int64_t col = panel * kRows + c;
    if (r >= p.m || col >= p.n) continue;
    float g = red[0][0][r][c], u = red[0][1][r][c];
    for (int w = 1; w < KW; ++w) {
      g += red[w][0][r][c];
      u += red[w][1][r][c];
    }
    if (p.bias[0]) g += p.bias[0][col];
    if (p.bias[1]) u += p.bias[1][col];
    p.y[r * p.n + col] = Activate<ACT>(g) * u;
  }
}

// Few rows or small sizes: a workgroup per (XP panels of x, gate and up panel), on
// the fp32 matrix-core product of 16 x 16 x 4, whose operands need no cutting: a
// lane's weights are single words of a panel's rows, and its x four consecutive k
// of one row, in which product i of four takes the i-th. The wavefronts take 16 k in
// turn and meet in LDS, in order. A product costs five times the planes' (16-bit
// weights: eight to sixteen times), but there is one launch, no cutting and no pass
// over the weights. Latency bounds it at few rows (bf16, 9 x 896 x 3584 7 us, 16 x
// 4096 x 4096 18, of which the weights' bytes are 14), its products at more (fp32,
// 40 x 4096 x 4096 39 us, of which the bytes are 28).
template <int WT>
__device__ __forceinline__ float Widen(typename Type<WT>::T v) {
  if constexpr (WT == EHIP_WEIGHT_F32)
    return v;
  else if constexpr (WT == EHIP_WEIGHT_BF16)
    return __uint_as_float(uint32_t{v} << 16);
  else
    return static_cast<float>(__builtin_bit_cast(_Float16, v));
}

template <int WT, int XP, int KW, int ACT>
__global__ __launch_bounds__(64 * KW) void GatedDirect(GatedParams p) {
  using T = typename Type<WT>::T;
  __shared__ f32x4_t red[KW][XP * 2][64];
  const int lane = threadIdx.x & 63, n16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const uint32_t xb = blockIdx.x / static_cast<uint32_t>(p.w_panels);
  const int64_t wp = blockIdx.x - xb * static_cast<uint32_t>(p.w_panels);
  const int64_t row0 = int64_t{xb} * XP * kRows + n16;
  const T* const wg = static_cast<const T*>(p.wp[0]) + wp * p.k * kRows + n16;
  const T* const wu = static_cast<const T*>(p.wp[1]) + wp * p.k * kRows + n16;
  f32x4_t acc[XP][2];
  const float* xr[XP];
#pragma unroll
  for (int a = 0; a < XP; ++a) {
    acc[a][0] = acc[a][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    // Rows past the last read the last one: their results are not stored.
    xr[a] = p.x + min(row0 + a * kRows, p.m - 1) * p.k;
  }
  f32x4_t x[XP];
  // As they are: widened where they are used, not where they are loaded. 16-bit ones
  // one by one (in vectors 16 x 4096 x 4096 24 us, so 19), fp32 ones in vectors (77 x
  // 896 x 3584 15.4, one by one 16.4).
  using Words = std::conditional_t<WT == EHIP_WEIGHT_F32, f32x4_t, T[4]>;
  Words w[2];
  auto load = [&](int64_t k0) __attribute__((always_inline)) {
    const int64_t kk = k0 + 4 * q;
    if (p.x_vec && k0 + 16 <= p.k) {
#pragma unroll
      for (int a = 0; a < XP; ++a) x[a] = *reinterpret_cast<const f32x4_t*>(xr[a] + kk);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[0][i] = wg[(kk + i) * kRows];
        w[1][i] = wu[(kk + i) * kRows];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = kk + i < p.k;
        const int64_t at = in ? kk + i : 0;
#pragma unroll
        for (int a = 0; a < XP; ++a) x[a][i] = in ? xr[a][at] : 0.f;
        w[0][i] = in ? wg[at * kRows] : T{};
        w[1][i] = in ? wu[at * kRows] : T{};
      }
    }
  };
  int64_t k0 = int64_t{wave} * 16;
  if (k0 < p.k) load(k0);
  for (; k0 < p.k; k0 += 16 * KW) {
    f32x4_t cx[XP];
    Words cw[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) cw[0][i] = w[0][i], cw[1][i] = w[1][i];
#pragma unroll
    for (int a = 0; a < XP; ++a) cx[a] = x[a];
    if (k0 + 16 * KW < p.k) load(k0 + 16 * KW);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v[2] = {Widen<WT>(cw[0][i]), Widen<WT>(cw[1][i])};
#pragma unroll
      for (int a = 0; a < XP; ++a)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          acc[a][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[h], cx[a][i], acc[a][h], 0, 0, 0);
    }
  }
#pragma unroll
  for (int a = 0; a < XP; ++a)
#pragma unroll
    for (int h = 0; h < 2; ++h) red[wave][2 * a + h][lane] = acc[a][h];
  __syncthreads();
  for (int a = wave; a < XP; a += KW) {
    f32x4_t s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = red[0][2 * a + h][lane];
      for (int i = 1; i < KW; ++i) s[h] += red[i][2 * a + h][lane];
    }
    const int64_t col = wp * kRows + 4 * q;
    StoreRow4<0>(p, row0 + a * kRows, col, Finish<ACT>(p, col, s[0], s[1]));
  }
}

template <int WT, int XP, int ACT>
hipError_t LaunchDirect(const GatedParams& p, hipStream_t stream) {
  const int64_t n = (p.x_panels + XP - 1) / XP * p.w_panels;
  if (n > UINT32_MAX / 512) return hipErrorInvalidValue;
  // Five panels' sums leave room for four wavefronts: 80 x 4096 x 4096 57 us, 65 with
  // eight; up to four panels eight are faster (128 rows 94 against 99).
  constexpr int kWaves = XP > 4 ? 4 : 8;
  hipLaunchKernelGGL((GatedDirect<WT, XP, kWaves, ACT>), dim3(static_cast<uint32_t>(n)),
                     dim3(64 * kWaves), 0, stream, p);
  return hipGetLastError();
}

template <int WT, int MR, int ACT>
hipError_t LaunchStream(const GatedParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(p.w_panels));
  // Eight rows' sums: four wavefronts where the panels are many (4096 x 16384 60 us,
  // 69 with eight), eight for latency (896 x 3584 7.9 us, 8.6 with four).
  if (MR == 8 && p.w_panels > 512)
    hipLaunchKernelGGL((GatedStream<WT, MR, 4, 4, ACT>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((GatedStream<WT, MR, 8, MR == 1 ? 2 : 4, ACT>), grid, dim3(512), 0, stream,
                       p);
  return hipGetLastError();
}

template <int WT, int WR, int WC, int XP, int WP, int NS, int ACT, int OCC>
hipError_t LaunchTiles(GatedParams p, hipStream_t stream) {
  const int64_t rt = (p.x_panels + WR * XP - 1) / (WR * XP);
  const int64_t ct = (p.w_panels + WC * WP / 2 - 1) / (WC * WP / 2);
  if (rt * ct * p.splits > (int64_t{1} << 30)) return hipErrorInvalidValue;
  p.row_tiles = static_cast<int32_t>(rt);
  p.col_tiles = static_cast<int32_t>(ct);
  const uint32_t grid = static_cast<uint32_t>((rt * ct * p.splits + 7) / 8 * 8);
  hipLaunchKernelGGL((GatedStaged<WT, WR, WC, XP, WP, NS, ACT, OCC>), dim3(grid),
                     dim3(64 * WR * WC), 0, stream, p);
  if constexpr (WR == 1 && WC == 4 && XP <= 4 && WP == 4) {  // the split tiles
    if (p.splits > 1) {
      if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
      hipLaunchKernelGGL((GatedMerge<WT, WC, XP, WP, ACT>),
                         dim3(static_cast<uint32_t>(rt * ct * XP * (WP / 2))), dim3(64 * WC), 0,
                         stream, p);
    }
  }
  return hipGetLastError();
}

template <int WT>
hipError_t LaunchCut(const GatedParams& p, hipStream_t stream) {
  // A step a wavefront; for planes of fp16, whose workgroups read all of their rows
  // first, no more workgroups than CUs.
  constexpr int kWaves = Type<WT>::kHalf ? kRows : 4;
  int64_t chunks = (p.steps + kWaves - 1) / kWaves;
  if (Type<WT>::kHalf) chunks = std::min(chunks, std::max<int64_t>(1, p.cus / p.x_panels));
  const int64_t chunk = (p.steps + chunks - 1) / chunks;
  const int64_t cuts = p.x_panels * ((p.steps + chunk - 1) / chunk);
  const int64_t grid = cuts + (Type<WT>::kCols ? 2 * p.w_panels : 0);
  if (grid > INT32_MAX / (64 * kWaves)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((CutRows<WT, kWaves>), dim3(static_cast<uint32_t>(grid)), dim3(64 * kWaves), 0,
                     stream, p, static_cast<int>(chunk), static_cast<int>(cuts));
  return hipGetLastError();
}

template <int WT, int ACT>
hipError_t Launch(const GatedParams& p, hipStream_t stream) {
  if (p.m <= 1) return LaunchStream<WT, 1, ACT>(p, stream);
  if (p.m <= 2) return LaunchStream<WT, 2, ACT>(p, stream);
  if (p.m <= 4) return LaunchStream<WT, 4, ACT>(p, stream);
  if (p.m <= kStreamRows) return LaunchStream<WT, 8, ACT>(p, stream);
  constexpr bool kF32 = WT == EHIP_WEIGHT_F32, kF16 = WT == EHIP_WEIGHT_F16;
  if (p.tile == GatedTile::kDirect) {
    // As few groups of rows as there can be, alike.
    const int64_t groups = (p.x_panels + 4) / 5;
    switch ((p.x_panels + groups - 1) / groups) {
      case 1: return LaunchDirect<WT, 1, ACT>(p, stream);
      case 2: return LaunchDirect<WT, 2, ACT>(p, stream);
      case 3: return LaunchDirect<WT, 3, ACT>(p, stream);
      case 4: return LaunchDirect<WT, 4, ACT>(p, stream);
      default: return LaunchDirect<WT, 5, ACT>(p, stream);
    }
  }
  if constexpr (WT == EHIP_WEIGHT_BF16) {
    if (p.tile == GatedTile::kAsF16) {
      if (hipError_t e = LaunchCut<kBf16AsF16>(p, stream); e != hipSuccess) return e;
      return LaunchTiles<kBf16AsF16, 1, 4, 8, 4, 2, ACT, 2>(p, stream);
    }
  }
  if (hipError_t e = LaunchCut<WT>(p, stream); e != hipSuccess) return e;
  if constexpr (kF32) {
    switch (p.tile) {
      case GatedTile::k256x128: return LaunchTiles<WT, 2, 4, 8, 4, 2, ACT, 2>(p, stream);
      case GatedTile::k256x64: return LaunchTiles<WT, 2, 4, 8, 2, 2, ACT, 2>(p, stream);
      case GatedTile::k128x64: return LaunchTiles<WT, 2, 2, 4, 4, 2, ACT, 2>(p, stream);
      case GatedTile::k64x32: return LaunchTiles<WT, 2, 2, 2, 2, 3, ACT, 2>(p, stream);
      default: return LaunchTiles<WT, 1, 4, 3, 2, 3, ACT, 2>(p, stream);
    }
  } else {
    switch (p.tile) {
      case GatedTile::k128x128: return LaunchTiles<WT, 1, 4, 8, 4, 2, ACT, 2>(p, stream);
      case GatedTile::k128x64: return LaunchTiles<WT, 2, 2, 4, 4, kF16 ? 3 : 2, ACT, 2>(p, stream);
      case GatedTile::k64x64: return LaunchTiles<WT, 2, 2, 2, 4, 4, ACT, 2>(p, stream);
      case GatedTile::k64x32: return LaunchTiles<WT, 2, 2, 2, 2, 3, ACT, 2>(p, stream);
      case GatedTile::k48x32: return LaunchTiles<WT, 1, 4, 3, 2, 4, ACT, 2>(p, stream);
      default: break;
    }
    switch (std::min<int64_t>(p.x_panels, 4)) {
      case 1: return LaunchTiles<WT, 1, 4, 1, 4, 4, ACT, 1>(p, stream);
      case 2: return LaunchTiles<WT, 1, 4, 2, 4, 4, ACT, 1>(p, stream);
      case 3: return LaunchTiles<WT, 1, 4, 3, 4, 4, ACT, 1>(p, stream);
      default: return LaunchTiles<WT, 1, 4, 4, 4, 4, ACT, 1>(p, stream);
    }
  }
}

template <int WT>
hipError_t LaunchType(const GatedParams& p, hipStream_t stream) {
  switch (p.act) {
    case EHIP_ACT_SILU: return Launch<WT, EHIP_ACT_SILU>(p, stream);
    case EHIP_ACT_GELU: return Launch<WT, EHIP_ACT_GELU>(p, stream);
    default: return Launch<WT, EHIP_ACT_GELU_TANH>(p, stream);
  }
}

// The staged kernel's tile: the one with the least estimated
// time, a CU's share of the workgroups times a step's time, which is much the
// same whether a CU runs them side by side or in turn (us a step, one
// workgroup on a CU and a share of several). What it picks against the others (us;
// tiles in the order below):
//   bf16, 2382 x 4096 x 16384 1313 of (1313, 1387, 1571, 2097, 1795)
//   600 x 4096 x 16384 382 of (391, 382, 416, 539, 471)
//   2382 x 896 x 3584 81 of (94, 81, 81, 88, 83); 64 rows 10.3 of (36, 22, 14, 10.3, 12.4)
//   300 x 4096 x 4096 59 of (138, 82, 72, 71, 59)
//   fp32, 2400 x 4096 x 16384 1695 of (1695, 1863, 1966, 2772, 2746)
//   600 x 4096 x 4096 154 of (270, 154, 174, 177, 182), 1000 x 1111 300 rows 17 of
//   (75, 45, 33, 17, 20), 4096 x 4096 106 of (269, 150, 118, 108, 106)
// and no less than its bytes from L2 take at 9.6 TB/s. Where few rows leave CUs
// idle, 16-bit weights: tiles of up to 64 x 128 whose steps are cut so that most
// CUs have a part, 0.22 us a step and 0.09 for each panel of x, no less than 6.3
// TB/s, and 3 us for the merge. Whole calls, bf16, split and at best whole: 48 x 4096
// x 4096 23 and 35 us, 48 x 4096 x 16384 64 and 69, 17 x 2048 x 8192 21 and 25.
// bf16 weights go as fp16 (their 8 bits fit, after a power of two per row) where
// the third product costs more than a pass over them, 5.6 TB/s, and the
// conversions: 2382 x 4096 x 16384 1100 + 68 of cutting and pass for 1313 + 21, 2382
// x 4096 x 4096 327 + 36 for 379 + 21, 600 x 4096 x 16384 341 + 54 for 416 + 7.
// A call leaves GatedStaged where what comes before it (8 us; fp32 weights 9 and the
// reading of the columns' magnitudes at 5.2 TB/s) and its tiles take longer than
// GatedDirect, 3.2 ns for a k of each panel of x that a CU has in turn. Whole calls,
// direct and staged: fp32, 100 x 4096 x 4096 83 and 95 us, 200 x 896 x 3584 46 and 30;
// bf16, 9 x 896 x 3584 7 and 14, 16 x 4096 x 4096 18 and 24, 40 x 896 x 3584 11 and 14.
void PickTile(int weight_dtype, GatedParams* p) {
  struct Cost {
    GatedTile tile;
    int rows, cols;             // panels of x and of y
    double alone[3], share[3];  // by EHIP_WEIGHT_*; 0: not built
  };
  constexpr Cost kCosts[] = {{GatedTile::k256x128, 16, 8, {2.15}, {2.5}},
                             {GatedTile::k256x64, 16, 4, {1.19}, {1.42}},
                             {GatedTile::k128x128, 8, 8, {0, 1.13, 1.03}, {0, 0.86, 0.76}},
                             {GatedTile::k128x64, 8, 4, {0.91, 0.65, 0.55}, {0.80, 0.52, 0.43}},
                             {GatedTile::k64x64, 4, 4, {0, 0.34, 0.32}, {0, 0.28, 0.26}},
                             {GatedTile::k64x32, 4, 2, {0.50, 0.21, 0.21}, {0.28, 0.20, 0.163}},
                             {GatedTile::k48x32, 3, 2, {0.58, 0.28, 0.145}, {0.215, 0.31, 0.121}}};
  const bool f32 = weight_dtype == EHIP_WEIGHT_F32;
  double least = 0;
  auto tiles = [&](int64_t rows, int64_t cols) {
    return (p->x_panels + rows - 1) / rows * ((p->w_panels + cols - 1) / cols);
  };
  // KiB of a step from L2, over all tiles: the weights once a row of tiles, x once
  // a column; 9.6 TB/s are 9375 KiB a us.
  const int planes = weight_dtype == EHIP_WEIGHT_BF16 ? 3 : 2, unit = f32 ? 2 : 1;
  auto traffic = [&](int64_t rows, int64_t cols) {
    return static_cast<double>(tiles(rows, cols) * (2 * unit * cols + planes * rows) * p->steps);
  };
  for (const Cost& c : kCosts) {
    if (c.share[weight_dtype] == 0) continue;
    const int64_t on_cu = (tiles(c.rows, c.cols) + p->cus - 1) / p->cus;
    const double us = std::max(
        static_cast<double>(on_cu * p->steps) * (on_cu == 1 ? c.alone : c.share)[weight_dtype],
        traffic(c.rows, c.cols) / 9375);
    if (least == 0 || us < least) {
      least = us;
      p->tile = c.tile;
    }
  }
  if (weight_dtype == EHIP_WEIGHT_BF16) {
    const int64_t on_cu = (tiles(8, 8) + p->cus - 1) / p->cus;
    const double pass = static_cast<double>(p->w_panels * kRows * 4) * static_cast<double>(p->k);
    const double us = static_cast<double>(on_cu * p->steps) * (on_cu == 1 ? 1.05 : 0.70);
    if (us + pass / 5.6e6 + 2 < least) {
      p->tile = GatedTile::kAsF16;
      return;
    }
  }
  const int64_t rows = std::min<int64_t>(p->x_panels, 4);
  const int64_t splits = std::min<int64_t>({p->cus / tiles(rows, 8), p->steps / 8, kMostSplits});
  const int64_t part = splits < 2 ? p->steps : (p->steps + splits - 1) / splits;
  const double split_us =
      std::max(static_cast<double>(part) * (0.22 + 0.09 * static_cast<double>(rows)),
               traffic(rows, 8) / 6152) +
      3;
  if (!f32 && splits >= 2 && split_us < least) {
    least = split_us;
    p->tile = GatedTile::kSplit;
    p->split_steps = static_cast<int32_t>(part);
    p->splits = static_cast<int32_t>((p->steps + part - 1) / part);
  }
  const double words = static_cast<double>(p->w_panels * kRows) * static_cast<double>(p->k);
  const int64_t groups = (p->x_panels + 4) / 5, panels = (p->x_panels + groups - 1) / groups;
  const int64_t rounds = (groups * p->w_panels + p->cus - 1) / p->cus;
  const double direct = 3.2e-3 * static_cast<double>(rounds * panels * p->k);
  if (rounds < 32768 && direct < least + (f32 ? 9 + 8 * words / 5.2e6 : 8)) {
    p->tile = GatedTile::kDirect;
    p->splits = 1;
  }
}

}  // namespace

size_t PlanGatedGemm(int64_t m, int64_t k, int64_t n, int weight_dtype, int cus, GatedParams* p) {
  p->m = m;
  p->k = k;
  p->n = n;
  p->cus = cus;
  p->x_panels = (m + kRows - 1) / kRows;
  p->w_panels = (n + kRows - 1) / kRows;
  p->steps = (k + kStep - 1) / kStep;
  p->splits = 1;
  p->split_steps = static_cast<int32_t>(p->steps);
  if (m <= kStreamRows) return 0;
  PickTile(weight_dtype, p);
  if (p->tile == GatedTile::kDirect) return 0;
  const bool as_f16 = p->tile == GatedTile::kAsF16;
  const bool half = weight_dtype != EHIP_WEIGHT_BF16 || as_f16;  // planes of fp16
  const bool cols = weight_dtype == EHIP_WEIGHT_F32 || as_f16;
  auto whole = [](int64_t bytes) { return (static_cast<size_t>(bytes) + 255) & ~size_t{255}; };
  p->scale_at =
      static_cast<size_t>(p->x_panels) * static_cast<size_t>(p->steps) * (half ? 2 : 3) * 1024;
  p->col_at = p->scale_at + whole(half ? p->x_panels * kRows * 4 : 0);
  p->col_stride = (p->w_panels + 8) * kRows;  // a tile's panels beyond the last
  p->part_at = p->col_at + whole(cols ? 2 * p->col_stride * 4 : 0);
  if (p->splits == 1) return p->part_at;
  // A split's sums: a tile's 16 slots by its panels of x, 1 KiB a block.
  const int64_t rows = std::min<int64_t>(p->x_panels, 4);
  const int64_t tiles = (p->x_panels + rows - 1) / rows * ((p->w_panels + 7) / 8);
  return p->part_at + static_cast<size_t>(tiles * p->splits * 16 * rows) * 1024;
}

hipError_t LaunchGatedGemm(const GatedParams& p, int weight_dtype, hipStream_t stream) {
  switch (weight_dtype) {
    case EHIP_WEIGHT_F32: return LaunchType<EHIP_WEIGHT_F32>(p, stream);
    case EHIP_WEIGHT_BF16: return LaunchType<EHIP_WEIGHT_BF16>(p, stream);
    case EHIP_WEIGHT_F16: return LaunchType<EHIP_WEIGHT_F16>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace ehip
