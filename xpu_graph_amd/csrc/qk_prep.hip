// What an attention layer does to its queries and keys before the scores, for gfx950: rotary positions (one axis or
// several, rows of the tables gathered by position) and, in the same pass, the per-head RMS norm.
//
//   n = x rsqrt(mean(x^2) + eps) w                                    (rope_axes: n = x)
//   y[i]       = n[i] c[i]       - n[i + R/2] s[i]                    i < R/2
//   y[i + R/2] = n[i + R/2] c[i + R/2] + n[i] s[i + R/2]
//   y[d]       = n[d]                                                 d >= R
// c, s: row positions[axis(i), b, s] of the tables, with a column per pair ([P, R/2]) or per element ([P, R]).
// A position outside the tables gives NaN in what it rotates (and reads nothing outside them).
//
// Gradients (xg_qk_norm_rope_bwd), rot^T the transposed rotation, xhat = x r, r = rsqrt(mean(x^2) + eps):
//   gn = rot^T(gy),  gw = sum over rows of gn xhat,  gx = r (gn w - xhat mean(gn w xhat))
//
// Memory bound: a row is read once and written once.  A thread owns 8 columns of the rotated lower half and their 8
// partners of the upper half (or two neighbouring vectors of the part that is not rotated), so a row of D elements
// takes D/16 lanes (rounded up to a power of two for the row sums, which stay inside the wavefront), and a thread
// takes kHeads heads of one token, which share the table row.  Queries and keys go out in one launch.  All sums and
// the rotation are fp32; one rounding per output.
// Measured on fresh inputs (bf16, D 128): rope_axes B2 S6144 H32, three axes 39 us, 201 MB, 5.1 TB/s; qk_norm_rope B4 S2048 H32/8
// 32 us, 168 MB, 5.2 TB/s, H32/32 51 us, 268 MB, 5.3 TB/s, its backward with the sum of the weight gradients 78 us, 403 MB, 5.1 TB/s
// (a copy of that size: 6.3).  Loads behind a condition each cost a quarter (47, 45, 72, 93 us), cached loads and results that
// lie head by head where the inputs lie token by token a tenth more.  With three axes and D 96, fp16 B3 S1371 H10/5 takes 10.5 us
// forward, 19 + 4 us backward: a row leaves two of its eight lanes idle, and each axis' position is read before its table row.
// fp32 D 128: rope_axes B1 S4096 H32, three axes 41 us, 134 MB, 3.3 TB/s; qk_norm_rope H32/8 42 us, 168 MB, 4.0 TB/s.
#include "xg_common.hpp"

namespace xg {
namespace {

constexpr int kMaxAxes = 4;
constexpr int kMaxDim = 512;

// n / d for n < 2^31 by a multiplication (d >= 1): m = floor(2^32 (2^s - d) / d) + 1, s = ceil(log2 d).
struct FastDiv {
  uint32_t d = 1, m = 1, s = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    while ((1ull << s) < d) ++s;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t quot(uint32_t n) const {
    const uint32_t t = __umulhi(n, m);
    return (uint32_t)(((uint64_t)t + n) >> s);
  }
};

struct Side {
  const void* x;
  const void* gy;
  void* out;
  const void* w;
  int64_t xs[3], gs[3], os[3];  // element strides of batch, head, sequence
  int H, chunks;                // heads; groups of heads a thread takes
};

struct Prep {
  Side side[2];
  const void* cos;
  const void* sin;
  const void* pos;             // NULL: row s of the tables (row 0 when their stride is 0)
  int64_t ps[3];               // strides of positions: axis, batch, token
  int64_t table_stride, table_rows;
  int half_off;                // columns from a pair's lower to its upper table entry (0: one entry per pair)
  int table_f32, w_f32, pos_64, axes, transpose;
  int D, R, tpr_log2;
  uint32_t units, n_chunks;
  FastDiv by_chunks, by_s;
  float eps, inv_d;
  float* gw_part;              // backward: [blocks][D], query blocks first
  int blocks0;                 // backward: blocks of side 0
  uint16_t axis_bits[kMaxDim / 16];  // two bits per pair, eight pairs per thread
};

template <typename T>
struct Eight {
  typedef T type __attribute__((ext_vector_type(8)));
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&o)[8]) {
  const typename Eight<T>::type v = *reinterpret_cast<const typename Eight<T>::type*>(p);
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = to_f32(v[j]);
}
template <typename T>
__device__ __forceinline__ void load8_as(const void* base, int64_t at, int f32, float (&o)[8]) {
  if constexpr (std::is_same_v<T, float>) {
    load8(reinterpret_cast<const float*>(base) + at, o);
  } else {
    if (f32)
      load8(reinterpret_cast<const float*>(base) + at, o);
    else
      load8(reinterpret_cast<const T*>(base) + at, o);
  }
}

// Sum over the 2^log2 lanes of a row.
__device__ __forceinline__ float row_sum(float v, int log2) {
  auto dpp = [](float x, auto CTRL) {
    constexpr int ctrl = decltype(CTRL)::value;
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl, 0xF, 0xF, true));
  };
  if (log2 > 0) v += dpp(v, std::integral_constant<int, 0xB1>{});
  if (log2 > 1) v += dpp(v, std::integral_constant<int, 0x4E>{});
  if (log2 > 2) v += dpp(v, std::integral_constant<int, 0x141>{});
  if (log2 > 3) v += dpp(v, std::integral_constant<int, 0x140>{});
  if (log2 > 4) v += __shfl_xor(v, 16, kWave);
  return v;
}

// cos and sin of a thread's eight pairs; FULL: tables with a column per element, whose halves may differ.
template <bool FULL>
struct Turn {
  float cl[8], sl[8], ch[FULL ? 8 : 1], sh[FULL ? 8 : 1];
  __device__ __forceinline__ float c_hi(int e) const { return FULL ? ch[e] : cl[e]; }
  __device__ __forceinline__ float s_hi(int e) const { return FULL ? sh[e] : sl[e]; }
};

// The table entries of this thread's eight pairs of token (b, s): one row when they share an axis, else the rows of
// every axis that occurs, picked per pair.
__device__ __forceinline__ int64_t table_row(const Prep& p, int a, int b, int s) {
  if (!p.pos) return s;
  const int64_t at = a * p.ps[0] + b * p.ps[1] + s * p.ps[2];
  return p.pos_64 ? reinterpret_cast<const int64_t*>(p.pos)[at] : (int64_t) reinterpret_cast<const int32_t*>(p.pos)[at];
}
template <typename T, bool FULL>
__device__ __forceinline__ void load_turn(const Prep& p, int j, int b, int s, Turn<FULL>& t) {
  const float nan = __builtin_nanf("");
  const int64_t col = 8 * j;
  if (p.axes == 1) {
    const int64_t row = table_row(p, 0, b, s);
    const bool bad = p.pos && (row < 0 || row >= p.table_rows);
    const int64_t at = (bad ? 0 : row) * p.table_stride + col;
    load8_as<T>(p.cos, at, p.table_f32, t.cl);
    load8_as<T>(p.sin, at, p.table_f32, t.sl);
    if constexpr (FULL) {
      load8_as<T>(p.cos, at + p.half_off, p.table_f32, t.ch);
      load8_as<T>(p.sin, at + p.half_off, p.table_f32, t.sh);
    }
    if (bad) {  // cos alone makes every element it turns NaN
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        t.cl[e] = nan;
        if constexpr (FULL) t.ch[e] = nan;
      }
    }
    return;
  }
  const uint32_t bits = p.axis_bits[j];
  for (int a = 0; a < p.axes; ++a) {
    uint32_t hit = 0;  // pairs of this axis
#pragma unroll
    for (int e = 0; e < 8; ++e) hit |= (uint32_t)(((bits >> (2 * e)) & 3u) == (uint32_t)a) << e;
    if (hit == 0) continue;
    const int64_t row = table_row(p, a, b, s);
    const bool bad = row < 0 || row >= p.table_rows;
    const int64_t at = (bad ? 0 : row) * p.table_stride + col;
    auto pick = [&](const void* table, int64_t from, float (&to)[8]) {
      float x[8];
      load8_as<T>(table, from, p.table_f32, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) to[e] = (hit >> e) & 1u ? (bad ? nan : x[e]) : to[e];
    };
    pick(p.cos, at, t.cl);
    pick(p.sin, at, t.sl);
    if constexpr (FULL) {
      pick(p.cos, at + p.half_off, t.ch);
      pick(p.sin, at + p.half_off, t.sh);
    }
  }
}

// The two vectors of thread j of a row.
__device__ __forceinline__ void columns(const Prep& p, int j, int& lo, int& hi, bool& rotated) {
  const int pairs = p.R >> 4;
  rotated = j < pairs;
  lo = rotated ? 8 * j : p.R + 16 * (j - pairs);
  hi = rotated ? (p.R >> 1) + 8 * j : lo + 8;
}

template <typename T, bool NORM, bool FULL, int kHeads>
__global__ __launch_bounds__(256) void prep_kernel(const Prep p) {
  typedef typename Eight<T>::type V8;
  const int j = threadIdx.x & ((1 << p.tpr_log2) - 1);
  const uint32_t unit = blockIdx.x * (256u >> p.tpr_log2) + (threadIdx.x >> p.tpr_log2);
  if (unit >= p.units) return;  // whole rows leave together: the row sums below stay inside a row's lanes
  const uint32_t token = p.by_chunks.quot(unit);
  const int chunk = (int)(unit - token * p.n_chunks);
  const int b = (int)p.by_s.quot(token);
  const int s = (int)(token - (uint32_t)b * p.by_s.d);
  const bool second = chunk >= p.side[0].chunks;
  const Side& sd = p.side[second];
  const int h0 = (second ? chunk - p.side[0].chunks : chunk) * kHeads;
  const bool live = j < (p.D >> 4);
  int lo_c, hi_c;
  bool rotated;
  columns(p, live ? j : 0, lo_c, hi_c, rotated);

  const T* x = reinterpret_cast<const T*>(sd.x) + b * sd.xs[0] + s * sd.xs[2];
  // loads without a condition, so that all of them are on their way together: a lane or a head too many reads another one's
  V8 lo[kHeads], hi[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const T* row = x + (int64_t)min(h0 + i, sd.H - 1) * sd.xs[1];
    lo[i] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(row + lo_c));
    hi[i] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(row + hi_c));
  }
  Turn<FULL> t{};
  if (live && rotated) {
    load_turn<T, FULL>(p, j, b, s, t);
    if (p.transpose) {  // the transposed rotation is the rotation by the tables (c, -s) with the halves of s swapped
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float l = t.sl[e];
        t.sl[e] = -t.s_hi(e);
        if constexpr (FULL) t.sh[e] = -l;
      }
    }
  }
  float wl[8], wh[8];
  if constexpr (NORM) {
#pragma unroll
    for (int e = 0; e < 8; ++e) wl[e] = wh[e] = 1.f;
    if (live && sd.w) {
      load8_as<T>(sd.w, lo_c, p.w_f32, wl);
      load8_as<T>(sd.w, hi_c, p.w_f32, wh);
    }
  }
  T* out = reinterpret_cast<T*>(sd.out) + b * sd.os[0] + s * sd.os[2];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    float xl[8], xh[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) xl[e] = to_f32(lo[i][e]), xh[e] = to_f32(hi[i][e]);
    if constexpr (NORM) {
      float a = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) a += xl[e] * xl[e] + xh[e] * xh[e];
      if (!live) a = 0.f;
      const float r = rsqrtf(row_sum(a, p.tpr_log2) * p.inv_d + p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xl[e] = xl[e] * r * wl[e];
        xh[e] = xh[e] * r * wh[e];
      }
    }
    V8 ol, oh;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ol[e] = from_f32<T>(rotated ? xl[e] * t.cl[e] - xh[e] * t.sl[e] : xl[e]);
      oh[e] = from_f32<T>(rotated ? xh[e] * t.c_hi(e) + xl[e] * t.s_hi(e) : xh[e]);
    }
    if (live && h0 + i < sd.H) {
      T* row = out + (int64_t)(h0 + i) * sd.os[1];
      __builtin_nontemporal_store(ol, reinterpret_cast<V8*>(row + lo_c));
      __builtin_nontemporal_store(oh, reinterpret_cast<V8*>(row + hi_c));
    }
  }
}

// Backward of norm + rotation.  A block walks the units (token, group of heads) of one side; a lane keeps the same
// columns throughout, so its share of the weight gradient stays in registers and leaves as one row per block.
template <typename T, bool FULL, int kHeads>
__global__ __launch_bounds__(256) void prep_bwd_kernel(const Prep p) {
  typedef typename Eight<T>::type V8;
  __shared__ float red[4096];
  const int j = threadIdx.x & ((1 << p.tpr_log2) - 1);
  const int group = threadIdx.x >> p.tpr_log2;
  const int per_block = 256 >> p.tpr_log2;
  const bool second = (int)blockIdx.x >= p.blocks0;
  const Side& sd = p.side[second];
  const uint32_t first = second ? blockIdx.x - p.blocks0 : blockIdx.x;
  const uint32_t step = (second ? gridDim.x - p.blocks0 : p.blocks0) * per_block;
  const uint32_t tokens = p.units;
  const uint32_t units = tokens * sd.chunks;
  const bool live = j < (p.D >> 4);
  int lo_c, hi_c;
  bool rotated;
  columns(p, live ? j : 0, lo_c, hi_c, rotated);
  float wl[8], wh[8], gwl[8], gwh[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) wl[e] = wh[e] = 1.f, gwl[e] = gwh[e] = 0.f;
  if (live && sd.w) {
    load8_as<T>(sd.w, lo_c, p.w_f32, wl);
    load8_as<T>(sd.w, hi_c, p.w_f32, wh);
  }
  for (uint32_t unit = first * per_block + group; unit < units; unit += step) {
    const uint32_t token = unit / (uint32_t)sd.chunks;
    const int h0 = (int)(unit - token * sd.chunks) * kHeads;
    const int b = (int)p.by_s.quot(token);
    const int s = (int)(token - (uint32_t)b * p.by_s.d);
    const T* x = reinterpret_cast<const T*>(sd.x) + b * sd.xs[0] + s * sd.xs[2];
    const T* g = reinterpret_cast<const T*>(sd.gy) + b * sd.gs[0] + s * sd.gs[2];
    T* out = reinterpret_cast<T*>(sd.out) + b * sd.os[0] + s * sd.os[2];
    V8 xlo[kHeads], xhi[kHeads], glo[kHeads], ghi[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {  // (without a condition, as in the forward)
      const int head = min(h0 + i, sd.H - 1);
      const T* xr = x + (int64_t)head * sd.xs[1];
      const T* gr = g + (int64_t)head * sd.gs[1];
      xlo[i] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(xr + lo_c));
      xhi[i] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(xr + hi_c));
      glo[i] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(gr + lo_c));
      ghi[i] = __builtin_nontemporal_load(reinterpret_cast<const V8*>(gr + hi_c));
    }
    Turn<FULL> t{};
    if (live && rotated) load_turn<T, FULL>(p, j, b, s, t);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      float xl[8], xh[8], gl[8], gh[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xl[e] = to_f32(xlo[i][e]), xh[e] = to_f32(xhi[i][e]);
        const float a = to_f32(glo[i][e]), c = to_f32(ghi[i][e]);
        gl[e] = rotated ? a * t.cl[e] + c * t.s_hi(e) : a;
        gh[e] = rotated ? c * t.c_hi(e) - a * t.sl[e] : c;
      }
      float ss = 0.f, sg = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ss += xl[e] * xl[e] + xh[e] * xh[e];
        sg += gl[e] * wl[e] * xl[e] + gh[e] * wh[e] * xh[e];
      }
      if (!live) ss = sg = 0.f;
      const float r = rsqrtf(row_sum(ss, p.tpr_log2) * p.inv_d + p.eps);
      const float m = row_sum(sg, p.tpr_log2) * p.inv_d * r * r;  // mean(gn w xhat) r
      V8 ol, oh;
      const bool own = live && h0 + i < sd.H;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ol[e] = from_f32<T>(r * (gl[e] * wl[e] - xl[e] * m));
        oh[e] = from_f32<T>(r * (gh[e] * wh[e] - xh[e] * m));
        gwl[e] += own ? gl[e] * xl[e] * r : 0.f;
        gwh[e] += own ? gh[e] * xh[e] * r : 0.f;
      }
      if (own) {
        T* row = out + (int64_t)(h0 + i) * sd.os[1];
        __builtin_nontemporal_store(ol, reinterpret_cast<V8*>(row + lo_c));
        __builtin_nontemporal_store(oh, reinterpret_cast<V8*>(row + hi_c));
      }
    }
  }
  if (p.gw_part == nullptr) return;
  // rows of the block meet in LDS (at most 256 / (D/16) rows of D), then leave as one row
  if (live) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      red[group * p.D + lo_c + e] = gwl[e];
      red[group * p.D + hi_c + e] = gwh[e];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.D; c += 256) {
    float a = 0.f;
    for (int g = 0; g < per_block; ++g) a += red[g * p.D + c];
    p.gw_part[(int64_t)blockIdx.x * p.D + c] = a;
  }
}

// gw[c] = sum over a side's partial rows, in a fixed order: 16 columns x 64 row lanes per block, block (c/16, side).
template <typename WT>
__global__ __launch_bounds__(1024) void gw_sum_kernel(const float* __restrict__ part, int blocks0, int blocks1, int D, WT* __restrict__ gw0,
                                                      WT* __restrict__ gw1) {
  __shared__ float red[64][17];
  const bool second = blockIdx.y != 0;
  WT* gw = second ? gw1 : gw0;
  if (gw == nullptr) return;
  const int c = threadIdx.x & 15, l = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + c;
  const int rows = second ? blocks1 : blocks0;
  const float* src = part + (second ? (int64_t)blocks0 * D : 0) + col;  // (not read where there are no rows)
  float a = 0.f;
#pragma unroll 8
  for (int r = l; r < rows; r += 64) a += src[(int64_t)r * D];
  red[l][c] = a;
  __syncthreads();
  if (l < 4) {  // four lanes of a column add sixteen rows each, then one of them the four
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += red[16 * l + i][c];
    red[16 * l][c] = t;
  }
  __syncthreads();
  if (l == 0) gw[col] = from_f32<WT>((red[0][c] + red[16][c]) + (red[32][c] + red[48][c]));
}

// ------------------------------------------------------------------ host side
int fill_rotary(Prep& p, const xg_rotary* rot, int64_t B, int64_t S, int64_t D, int dtype) {
  if (!rot || !rot->cos_table || !rot->sin_table) return XG_ERR_NULL_PTR;
  if (rot->table_dtype != dtype && rot->table_dtype != XG_F32) return XG_ERR_BAD_DTYPE;
  const int64_t R = rot->rot_dim;
  if (R < 16 || R > D || R % 16 != 0 || (D - R) % 16 != 0) return XG_ERR_BAD_SHAPE;
  if (rot->table_cols != R && rot->table_cols != R / 2) return XG_ERR_BAD_SHAPE;
  if (rot->table_rows <= 0 || rot->table_rows > 0x7fffffff || rot->table_stride < rot->table_cols) return XG_ERR_BAD_SHAPE;
  if (rot->axes < 1 || rot->axes > kMaxAxes) return XG_ERR_BAD_ARG;
  if (!rot->positions && (rot->axes != 1 || (rot->table_rows < S && rot->table_rows != 1))) return XG_ERR_BAD_SHAPE;
  if (rot->axes > 1 && !rot->pair_axis) return XG_ERR_NULL_PTR;
  const int vec = rot->table_dtype == XG_F32 ? 4 : 8;
  if (!aligned_to(rot->cos_table, 16) || !aligned_to(rot->sin_table, 16) || rot->table_stride % vec != 0) return XG_ERR_BAD_ALIGN;
  if (rot->positions && !aligned_to(rot->positions, rot->positions_64bit ? 8 : 4)) return XG_ERR_BAD_ALIGN;
  p.cos = rot->cos_table;
  p.sin = rot->sin_table;
  p.pos = rot->positions;
  for (int i = 0; i < 3; ++i) p.ps[i] = rot->positions ? rot->pos_strides[i] : 0;
  for (int i = 0; i < 3; ++i)
    if (p.ps[i] < 0) return XG_ERR_BAD_SHAPE;
  p.table_rows = rot->table_rows;
  p.table_stride = !rot->positions && rot->table_rows == 1 ? 0 : rot->table_stride;
  p.half_off = rot->table_cols == R ? (int)(R / 2) : 0;
  p.table_f32 = rot->table_dtype == XG_F32;
  p.pos_64 = rot->positions_64bit != 0;
  p.axes = rot->axes;
  p.R = (int)R;
  for (int i = 0; i < kMaxDim / 16; ++i) p.axis_bits[i] = 0;
  if (rot->axes > 1) {
    for (int64_t i = 0; i < R / 2; ++i) {
      if (rot->pair_axis[i] >= rot->axes) return XG_ERR_BAD_ARG;
      p.axis_bits[i / 8] = (uint16_t)(p.axis_bits[i / 8] | (rot->pair_axis[i] << (2 * (i % 8))));
    }
  }
  return XG_OK;
}

bool known_dtype(int dtype) { return dtype == XG_BF16 || dtype == XG_F16 || dtype == XG_F32; }

int fill_strides(int64_t (&to)[3], const int64_t* from, int dtype) {
  if (!from) return XG_ERR_NULL_PTR;
  const int vec = dtype == XG_F32 ? 4 : 8;
  for (int i = 0; i < 3; ++i) {
    if (from[i] < 0) return XG_ERR_BAD_SHAPE;
    if (from[i] % vec) return XG_ERR_BAD_ALIGN;
    to[i] = from[i];
  }
  return XG_OK;
}

int fill_side(Side& sd, const void* x, const void* gy, void* out, const void* w, int64_t H, const int64_t* xs, const int64_t* gs,
              const int64_t* os, int dtype, bool backward) {
  if (H == 0) return XG_OK;
  if (!x || !out || (backward && !gy)) return XG_ERR_NULL_PTR;
  if (!aligned_to(x, 16) || !aligned_to(out, 16) || (gy && !aligned_to(gy, 16)) || (w && !aligned_to(w, 16))) return XG_ERR_BAD_ALIGN;
  if (int st = fill_strides(sd.xs, xs, dtype)) return st;
  if (int st = fill_strides(sd.os, os, dtype)) return st;
  if (backward)
    if (int st = fill_strides(sd.gs, gs, dtype)) return st;
  sd.x = x;
  sd.gy = gy;
  sd.out = out;
  sd.w = w;
  sd.H = (int)H;
  return XG_OK;
}

int fill_common(Prep& p, int64_t B, int64_t S, int64_t D, float eps) {
  p.D = (int)D;
  p.tpr_log2 = 0;
  while ((1 << p.tpr_log2) < D / 16) ++p.tpr_log2;
  p.by_s = FastDiv((uint32_t)S);
  p.eps = eps;
  p.inv_d = 1.0f / (float)D;
  return XG_OK;
}

int check_sizes(int64_t B, int64_t H0, int64_t H1, int64_t S, int64_t D, int dtype) {
  if (!known_dtype(dtype)) return XG_ERR_BAD_DTYPE;
  if (B < 0 || H0 < 0 || H1 < 0 || S < 0 || D <= 0 || D % 16 != 0 || D > kMaxDim) return XG_ERR_BAD_SHAPE;
  if (B > 0x7fffffff || S > 0x7fffffff || H0 > (1 << 20) || H1 > (1 << 20)) return XG_ERR_TOO_LARGE;
  if (B && S && (H0 + H1) && B * S > 0x7fffffffLL / (H0 + H1)) return XG_ERR_TOO_LARGE;
  return XG_OK;
}

template <typename T, bool NORM, bool FULL, int kHeads>
int launch_prep(Prep& p, int64_t tokens, hipStream_t stream) {
  for (Side& sd : p.side) sd.chunks = (sd.H + kHeads - 1) / kHeads;
  p.n_chunks = (uint32_t)(p.side[0].chunks + p.side[1].chunks);
  p.by_chunks = FastDiv(p.n_chunks);
  p.units = (uint32_t)(tokens * p.n_chunks);
  const uint32_t per_block = 256u >> p.tpr_log2, blocks = (p.units + per_block - 1) / per_block;
  if (blocks > 0xffffff) return XG_ERR_TOO_LARGE;  // 2^32 threads
  hipLaunchKernelGGL((prep_kernel<T, NORM, FULL, kHeads>), dim3(blocks), dim3(256), 0, stream, p);
  return status_from_hip(hipGetLastError());
}

template <bool NORM>
int run_prep(Prep& p, int64_t tokens, int dtype, hipStream_t stream) {
  auto go = [&](auto full, auto heads) {
    constexpr bool FULL = decltype(full)::value;
    constexpr int kHeads = decltype(heads)::value;
    if (dtype == XG_BF16) return launch_prep<bf16_t, NORM, FULL, kHeads>(p, tokens, stream);
    if (dtype == XG_F16) return launch_prep<f16_t, NORM, FULL, kHeads>(p, tokens, stream);
    return launch_prep<float, NORM, FULL, kHeads>(p, tokens, stream);
  };
  // Several heads a thread share one read of the tables and keep more bytes on their way; few rows are spread over as many
  // threads as there are.  By the threads that one head each would make, on fresh inputs, us with one / two / four (eight) heads a
  // thread.  bf16 D 128: rope_axes, three axes, H32 131 k (S 512) 5.3 / 5.5 / 6.8 (9.0), 262 k 7.2 / 6.4 / 7.2 (9.1), 524 k 12.5 / 8.8 / 9.1
  // (10.2), 1.05 M 20.2 / 17.6 / 14.0 (14.1), 3.1 M - (39); qk_norm_rope H32/8 328 k (S 1024) 6.7 / 6.9 / 8.0, 655 k 12.3 / 9.6 / 10.2,
  // 1.3 M 20.1 / 18.1 / 16.5, 2.6 M 38.7 / 34.5 / 32.4 (38, registers).  fp16, D 64 and D 96 with three axes: the same within 5 % (D 96 fp16
  // qk_norm_rope 655 k 15.3 / 10.7 / 11.8, 1.3 M 26.6 / 20.7 / 16.2; rope_axes 1.05 M 19.8 / 16.2 / 13.1 (13.8)).  fp32 moves twice the
  // bytes a head and wants two at the most, which the rule does not tell: D 128 qk_norm_rope 328 k 12.3 / 11.3 / 13.7, 655 k 21.2 / 20.0 /
  // 19.0, 1.3 M 38.5 / 37.8 / 41.9, 2.6 M 74 / 73 / 81; rope_axes 524 k 18.8 / 17.7 / 17.7 (23.4), 1.05 M 32.6 / 31.8 / 36.6 (41.1), 2.1 M
  // 60 / 58 / 63 (75); D 96 rope_axes 2.1 M 57 / 52 / 48 (53).
  const int64_t threads = (tokens * (p.side[0].H + p.side[1].H)) << p.tpr_log2;
  auto with = [&](auto heads) { return p.half_off ? go(std::true_type{}, heads) : go(std::false_type{}, heads); };
  constexpr int kMany = NORM ? 4 : 8;
  if (threads >= 4 * 256 * 1024) return with(std::integral_constant<int, kMany>{});
  if (threads >= 256 * 1024) return with(std::integral_constant<int, 2>{});
  return with(std::integral_constant<int, 1>{});
}

constexpr int kBwdHeads = 2;

// Blocks of the two sides of the backward, in proportion to the rows: as many as the chip holds at once (three per compute
// unit by registers; B4 S2048 H32/32 D128 bf16 on one set of inputs: 80.7 us with 768, 84 with 1536, 101 with 1024).
void bwd_blocks(int64_t tokens, int64_t H0, int64_t H1, int64_t D, int& n0, int& n1) {
  int log2 = 0;
  while ((1 << log2) < D / 16) ++log2;
  const int64_t per_block = 256 >> log2;
  auto count = [&](int64_t H) {
    if (H == 0 || tokens == 0) return (int64_t)0;
    const int64_t units = tokens * ((H + kBwdHeads - 1) / kBwdHeads);
    const int64_t most = 768 * H / (H0 + H1);
    const int64_t want = (units + per_block - 1) / per_block;
    return want < (most < 1 ? 1 : most) ? want : (most < 1 ? 1 : most);
  };
  n0 = (int)count(H0);
  n1 = (int)count(H1);
}

// The weight gradients from the blocks' rows (zeros over none).
int sum_weight_grads(const float* part, int n0, int n1, int64_t D, void* gw_q, void* gw_k, int w_dtype, hipStream_t st) {
  const dim3 grid((unsigned)(D / 16), 2);
  auto sum = [&](auto zero) {
    typedef decltype(zero) WT;
    hipLaunchKernelGGL((gw_sum_kernel<WT>), grid, dim3(1024), 0, st, part, n0, n1, (int)D, (WT*)gw_q, (WT*)gw_k);
  };
  if (w_dtype == XG_F32)
    sum(0.f);
  else if (w_dtype == XG_BF16)
    sum((bf16_t)0.f);
  else
    sum((f16_t)0.f);
  return status_from_hip(hipGetLastError());
}

}  // namespace
}  // namespace xg

extern "C" int xg_rope_axes(const void* x, void* out, int64_t B, int64_t H, int64_t S, int64_t D, const int64_t x_strides[3],
                            const int64_t o_strides[3], const xg_rotary* rotary, int transpose, int dtype, xg_stream_t stream) {
  using namespace xg;
  if (int st = check_sizes(B, H, 0, S, D, dtype)) return st;
  Prep p{};
  if (int st = fill_rotary(p, rotary, B, S, D, dtype)) return st;
  if (B == 0 || H == 0 || S == 0) return XG_OK;
  if (int st = fill_side(p.side[0], x, nullptr, out, nullptr, H, x_strides, nullptr, o_strides, dtype, false)) return st;
  if (int st = fill_common(p, B, S, D, 0.f)) return st;
  p.transpose = transpose != 0;
  return run_prep<false>(p, B * S, dtype, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int xg_qk_norm_rope(const void* q, const void* k, const void* q_w, const void* k_w, void* q_out, void* k_out, int64_t B,
                               int64_t H, int64_t Hkv, int64_t S, int64_t D, const int64_t q_strides[3], const int64_t k_strides[3],
                               const int64_t qo_strides[3], const int64_t ko_strides[3], const xg_rotary* rotary, float eps,
                               int dtype, int w_dtype, xg_stream_t stream) {
  using namespace xg;
  if (int st = check_sizes(B, H, Hkv, S, D, dtype)) return st;
  if (w_dtype != dtype && w_dtype != XG_F32) return XG_ERR_BAD_DTYPE;
  Prep p{};
  if (int st = fill_rotary(p, rotary, B, S, D, dtype)) return st;
  if (B == 0 || S == 0 || H + Hkv == 0) return XG_OK;
  if (int st = fill_side(p.side[0], q, nullptr, q_out, q_w, H, q_strides, nullptr, qo_strides, dtype, false)) return st;
  if (int st = fill_side(p.side[1], k, nullptr, k_out, k_w, Hkv, k_strides, nullptr, ko_strides, dtype, false)) return st;
  if (int st = fill_common(p, B, S, D, eps)) return st;
  p.w_f32 = w_dtype == XG_F32;
  return run_prep<true>(p, B * S, dtype, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int64_t xg_qk_norm_rope_bwd_workspace_floats(int64_t B, int64_t H, int64_t Hkv, int64_t S, int64_t D) {
  using namespace xg;
  if (check_sizes(B, H, Hkv, S, D, XG_F32) != XG_OK) return 0;
  int n0, n1;
  bwd_blocks(B * S, H, Hkv, D, n0, n1);
  return (int64_t)(n0 + n1) * D;
}

extern "C" int xg_qk_norm_rope_bwd(const void* q, const void* k, const void* q_w, const void* k_w, const void* gq, const void* gk,
                                   void* dq, void* dk, void* gw_q, void* gw_k, float* workspace, int64_t workspace_floats, int64_t B,
                                   int64_t H, int64_t Hkv, int64_t S, int64_t D, const int64_t q_strides[3], const int64_t k_strides[3],
                                   const int64_t gq_strides[3], const int64_t gk_strides[3], const int64_t dq_strides[3],
                                   const int64_t dk_strides[3], const xg_rotary* rotary, float eps, int dtype, int w_dtype,
                                   xg_stream_t stream) {
  using namespace xg;
  if (int st = check_sizes(B, H, Hkv, S, D, dtype)) return st;
  if (w_dtype != dtype && w_dtype != XG_F32) return XG_ERR_BAD_DTYPE;
  Prep p{};
  if (int st = fill_rotary(p, rotary, B, S, D, dtype)) return st;
  const bool want_gw = gw_q || gw_k;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (B == 0 || S == 0 || H + Hkv == 0) return want_gw ? sum_weight_grads(nullptr, 0, 0, D, gw_q, gw_k, w_dtype, st) : XG_OK;
  if (int st = fill_side(p.side[0], q, gq, dq, q_w, H, q_strides, gq_strides, dq_strides, dtype, true)) return st;
  if (int st = fill_side(p.side[1], k, gk, dk, k_w, Hkv, k_strides, gk_strides, dk_strides, dtype, true)) return st;
  if (int st = fill_common(p, B, S, D, eps)) return st;
  int n0, n1;
  bwd_blocks(B * S, H, Hkv, D, n0, n1);
  if (want_gw) {
    if (!workspace) return XG_ERR_NULL_PTR;
    if (workspace_floats < (int64_t)(n0 + n1) * D) return XG_ERR_BAD_ARG;
    p.gw_part = workspace;
  }
  p.w_f32 = w_dtype == XG_F32;
  for (Side& sd : p.side) sd.chunks = (sd.H + kBwdHeads - 1) / kBwdHeads;
  p.units = (uint32_t)(B * S);  // tokens: the units of a side follow from its heads
  p.blocks0 = n0;
  const dim3 grid(n0 + n1), block(256);
  auto go = [&](auto full) {
    constexpr bool FULL = decltype(full)::value;
    if (dtype == XG_BF16)
      hipLaunchKernelGGL((prep_bwd_kernel<bf16_t, FULL, kBwdHeads>), grid, block, 0, st, p);
    else if (dtype == XG_F16)
      hipLaunchKernelGGL((prep_bwd_kernel<f16_t, FULL, kBwdHeads>), grid, block, 0, st, p);
    else
      hipLaunchKernelGGL((prep_bwd_kernel<float, FULL, kBwdHeads>), grid, block, 0, st, p);
  };
  p.half_off ? go(std::true_type{}) : go(std::false_type{});
  if (hipGetLastError() != hipSuccess) return XG_ERR_LAUNCH;
  return want_gw ? sum_weight_grads(workspace, n0, n1, D, gw_q, gw_k, w_dtype, st) : XG_OK;
}
