// Linear attention with a decay for each head, for gfx950:
//
//   S_t = lam S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   lam = exp(log_decay[h]),   S a [D, D] matrix per head in fp32
//
// Chunked form, 32 tokens at a time; S the state before the chunk, n its tokens, i and j rows in it:
//   P[i][j] = (q_i . k_j) lam^(i-j)   for j <= i, else 0
//   o_i     = scale (sum_j P[i][j] v_j + lam^(i+1) q_i S)
//   S'      = lam^n S + sum_j lam^(n-1-j) k_j v_j^T
//
// Its gradients are the same recurrence with the operands in other roles (F: the forward form, F_rev: the tokens backwards):
//   dq = scale F(do, v, k), state S^T;   dv = F_rev(k, q, do), dk = F_rev(v, do, q), state G = scale sum lam^(t-s) q_t do_t^T
// In F_rev the incoming gradient of the final state enters undecayed, so its state is kept one decay ahead (e = 1 below), and
// what it ends with is the gradient of the initial state.
//
// One kernel serves all of them (Problem says which operand is which).  A workgroup owns one head of one batch entry and a
// segment of its tokens; wave w owns 32 columns of S in its accumulators, where they stay in fp32 from chunk to chunk, and
// computes those columns of O.  The products are transposed (P^T = K Q^T, O^T = S^T Q^T + V^T P^T), so that S and P go from
// accumulator to operand without leaving the lane: the k index of an MFMA may be permuted as long as both operands agree, and
// the order used is the one the accumulators hold.  P is small (32 x 32) and computed by every wave for itself: that costs 8 of
// 34 to 42 MFMAs and saves a round trip through LDS and a barrier.  The rows of S (and the columns of O) are numbered with bits
// 2 and 3 swapped (sigma below), which makes the eight values of a lane in a k-step neighbours in memory: rows of Q and K are
// read, and O written, 16 bytes at a time; the transposing reads of K and V swap two of their pieces instead, at no cost.
// Tiles go from global memory straight to LDS, one chunk ahead.
//
// Roundings to 16 bits: S and P where they are operands of the product that gives O, as the scores of any tiled attention are
// (one rounding each, against the one of O itself).  The state is an fp32 result, and it is carried over the whole sequence, so
// there lam^(n-1-j) v_j is split into three bf16 parts, which hold its 24 bits (two parts, 16 bits, where a segment's running
// state only feeds O).  fp16 tensors have three more bits than bf16 and a range that neither S nor P fits, so their operands are
// split into bf16 parts as well: two each for q, k, v (exact), S and P, and products of the small parts are left out.
//
// A few heads do not fill the chip.  The tokens are then cut into segments: one launch sums up each segment's own state, one
// turns them into the states before each segment (elementwise, in order), and the kernel above runs all segments at once.
//
// The recurrence is causal, and so is the kernel where values are not finite: a chunk whose O shows one is made again token by token.
// Looking for it costs ten instructions a chunk (bf16 D128 H32, in turn: B4 S2048 forward 96.7 -> 99.2 us, backward 163.5 -> 164.3,
// B1 S32768 no change; B8 S4096, whose runs scatter between 220 and 250, at most 4 %, backward 577 -> 581).
//
// What bounds it: memory, and behind it the instructions of a wave (34 to 42 MFMAs of 32 cycles and about 280 others a chunk), of
// which one alone on its SIMD makes a chunk in 1.4 us.  bf16 D 128 H 32: forward B8 S4096 240 us (1.07 GB, 4.5 TB/s), B8 S2048
// 125 us, B4 S2048 99 us, B1 S32768 334 us (eight segments: 1.45 GB by the counters, 4.4 TB/s); backward B8 S4096
// 580 us, B4 S2048 164 us (0.67 GB by the counters: dv and dk share all they can; 384 workgroups on 256 compute units), B1 S32768
// 790 us.  fp16 runs most products two or three times: forward B4 S2048 212 us, backward B1 H64 S4096 379 us against 169.
#include "sdpa_common.hpp"

namespace xg {
namespace linattn {

using sdpa::lds_s16x4;
using sdpa::s16x4;
using sdpa::s16x8;
using sdpa::f32x16;
using sdpa::mma;
using sdpa::swz_v;
using sdpa::Vec8;

constexpr int C = 32;  // tokens per chunk
constexpr float kLog2e = 1.44269504088896340736f;

struct Operand {
  const void* p;
  int64_t s[3];  // element strides of batch, head, token
  int group;     // query heads per head of this tensor
};

struct Problem {
  Operand q, k, v;
  void* out;
  int64_t os[3];
  int out_f32;              // out is fp32 (shares of shared heads), else the tensors' type
  const float* state0;      // [B, H, D, D] or NULL (zeros)
  float* state_out;         // [B, H, D, D] or NULL
  float* seg_states;        // [B H][n_seg][D D] in accumulator order (n_seg > 1)
  int state0_t;             // state0 is read transposed
  int reverse;
  int e;                    // the state is kept e decays ahead
  float s_intra, s_inter, s_state;
};

struct Params {
  Problem pr[3];
  const float* log_decay;
  const void* lengths;      // [B] or NULL
  int len64;
  int B, H, S;
  int n_seg, seg_chunks;
  int group;                // query heads of a key head that are eight blocks apart (see head_of)
};

// Row of an accumulator tile (or lane of an operand) -> row of S, column of V: bits 2 and 3 change places.
__device__ __forceinline__ constexpr int sigma(int x) { return (x & 0x13) | ((x & 4) << 1) | ((x & 8) >> 1); }

// A value in N bf16 parts, largest first.
template <int N>
struct Parts {
  bf16x8 v[N];
};
template <int N>
__device__ __forceinline__ Parts<N> split(const float (&x)[8]) {
  Parts<N> p;
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int k = 0; k < N; ++k) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p.v[k][i] = (bf16_t)r[i];
    if (k + 1 < N) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] -= (float)p.v[k][i];
    }
  }
  return p;
}

// Parts of an element of the tensors: bf16 is one, fp16 is two.
template <typename T>
constexpr int kParts = std::is_same_v<T, f16_t> ? 2 : 1;

template <typename T>
__device__ __forceinline__ Parts<kParts<T>> as_parts(typename Vec8<T>::type x) {
  if constexpr (kParts<T> == 1) {
    return Parts<1>{{x}};
  } else {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)x[i];
    return split<2>(f);
  }
}

// Sum of the products of two split operands; parts i and j meet while i + j < max(NA, NB).
template <int NA, int NB>
__device__ __forceinline__ f32x16 mma_parts(const Parts<NA>& a, const Parts<NB>& b, f32x16 c) {
  constexpr int N = NA > NB ? NA : NB;
#pragma unroll
  for (int i = NA - 1; i >= 0; --i)
#pragma unroll
    for (int j = NB - 1; j >= 0; --j)
      if (i + j < N) c = mma(a.v[i], b.v[j], c);
  return c;
}

// A chunk's rows of one operand in LDS: [32][D], 16-byte pieces swizzled for both kinds of reads.  The addresses of a lane's
// reads are kept in registers; which tile and stage they go to is an immediate offset.
template <typename T, int D>
struct Tile {
  static constexpr int RB = D * 2;
  static constexpr int BYTES = C * RB;
  typedef typename Vec8<T>::type V8;
  typedef __attribute__((address_space(3))) const V8 lds_V8;

  // row lane % 32, columns 16 t + 8 h .. +7
  __device__ static __forceinline__ uint32_t row_address(uint32_t lds, int t, int lane) {
    const int row = lane & 31, h = lane >> 5;
    return lds + row * RB + (((2 * t + h) ^ swz_v<D>(row)) << 4);
  }
  __device__ static __forceinline__ V8 row_frag(uint32_t at) { return *(lds_V8*)at; }
  // column 32 ct + sigma(lane % 32), rows 4 h .. +3 (hi: 8 + 4 h .. +3) of sixteen: a transposing read, in which sixteen lanes address
  // four rows of four 8-byte pieces and lane i of them receives column i; the middle pieces are swapped
  __device__ static __forceinline__ uint32_t col_address(uint32_t lds, int ct, int hi, int lane) {
    const int h = lane >> 5, a16 = lane & 15, b16 = (lane >> 4) & 1;
    const int piece = ((a16 & 1) << 1) | ((a16 >> 1) & 1);
    const int row = 8 * hi + 4 * h + (a16 >> 2), ch = 4 * ct + 2 * b16 + (piece >> 1), sub = (piece & 1) << 3;
    return lds + row * RB + ((ch ^ swz_v<D>(row)) << 4) + sub;
  }
  __device__ static __forceinline__ V8 col_frag(uint32_t lo_at, uint32_t hi_at) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)lo_at);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)hi_at);
    const s16x8 both = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(V8, both);
  }
};

// The addresses of a wave's transposing reads of K (every column) and of V (its own 32).
template <typename T, int D>
struct ColAddresses {
  uint32_t k_lo[D / 32], k_hi[D / 32], v_lo, v_hi;
  __device__ __forceinline__ ColAddresses(uint32_t k_tile, uint32_t v_tile, int w, int lane) {
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      k_lo[dt] = Tile<T, D>::col_address(k_tile, dt, 0, lane);
      k_hi[dt] = Tile<T, D>::col_address(k_tile, dt, 1, lane);
      asm volatile("" : "+v"(k_lo[dt]), "+v"(k_hi[dt]));  // held, not recomputed
    }
    v_lo = Tile<T, D>::col_address(v_tile, w, 0, lane);
    v_hi = Tile<T, D>::col_address(v_tile, w, 1, lane);
    asm volatile("" : "+v"(v_lo), "+v"(v_hi));
  }
};

__device__ __forceinline__ int length_of(const Params& p, int b) {
  if (!p.lengths) return p.S;
  const int64_t n = p.len64 ? reinterpret_cast<const int64_t*>(p.lengths)[b] : (int64_t) reinterpret_cast<const int32_t*>(p.lengths)[b];
  return n < 0 ? 0 : (n > p.S ? p.S : (int)n);
}

// lam^n for whole n >= 0; a decay of minus infinity gives 1, 0, 0, ...
__device__ __forceinline__ float head_log2(const Params& p, int h) {
  const float g = p.log_decay[h] * kLog2e;
  return g < -1e30f ? -1e30f : g;
}
__device__ __forceinline__ float decay(float g2, int n) { return __builtin_amdgcn_exp2f(g2 * (float)n); }

// An LDS address in a scalar register (the compiler would put a known constant, or one that it cannot tell to be uniform, into
// a vector register).
__device__ __forceinline__ uint32_t lds_address(const char* at) {
  uint32_t x = (uint32_t)(uintptr_t)(sdpa::lvoid*)const_cast<char*>(at);
  asm volatile("" : "+v"(x));
  return __builtin_amdgcn_readfirstlane(x);
}

// One operand's chunks on their way from global memory to LDS, in order.
template <typename T, int D>
struct Mover {
  static constexpr int RB = D * 2;
  const char* next;                            // the lowest address of the next whole chunk
  int64_t row_bytes;                           // signed: a reversed operand walks backwards
  int64_t step;                                // from chunk to chunk
  uint32_t off[2];                             // this lane's part of a tile, from its lowest address

  __device__ __forceinline__ void bind(const Operand& o, int b, int head, int len, int reverse, int t0, int tid) {
    row_bytes = (reverse ? -o.s[2] : o.s[2]) * 2;
    step = C * row_bytes;
    const int64_t lowest = reverse ? (int64_t)(len - 1 - t0) - (C - 1) : (int64_t)t0;
    next = reinterpret_cast<const char*>(o.p) + (b * o.s[0] + (head / o.group) * o.s[1] + lowest * o.s[2]) * 2;
    const uint32_t pitch = (uint32_t)(o.s[2] * 2);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int pos = place(tid, i), row = pos / RB, pc = (pos % RB) >> 4;
      off[i] = (uint32_t)(reverse ? C - 1 - row : row) * pitch + (uint32_t)((pc ^ swz_v<D>(row)) << 4);
    }
  }
  // bytes [1024 (2 wave + i) + 16 lane, + 16) of a tile
  __device__ static __forceinline__ int place(int tid, int i) { return (2 * (tid >> 6) + i) * 1024 + (tid & 63) * 16; }

  // 32 whole tokens straight to LDS (waits by vmcnt); `to`: this wave's place in the tile
  __device__ __forceinline__ void load(uint32_t to) {
    const uint64_t base = (uint64_t)(uintptr_t)next;  // the same for every lane
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)base), hi = __builtin_amdgcn_readfirstlane((uint32_t)(base >> 32));
    const void* from = (const void*)(uintptr_t)((uint64_t)hi << 32 | lo);
    load_to_lds16(from, off[0], to);
    load_to_lds16(from, off[1], to + 1024);
    next += step;
  }
  // the last n < 32 tokens, zeros behind them
  __device__ __forceinline__ void load_tail(int n, char* tile, int tid) const {
    const char* first = next + (row_bytes < 0 ? -(C - 1) * row_bytes : 0);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int pos = place(tid, i), row = pos / RB, pc = (pos % RB) >> 4;
      u32x4 x = {0, 0, 0, 0};
      if (row < n) x = *reinterpret_cast<const u32x4*>(first + row * row_bytes + ((pc ^ swz_v<D>(row)) << 4));
      *reinterpret_cast<u32x4*>(tile + pos) = x;
    }
  }
};

// This chunk is whole for every wave, and nobody reads the stage that is filled next any more.  LATER: vector memory operations
// of this wave that were issued after the chunk's loads and may still be in flight (they end in order).
template <int LATER>
__device__ __forceinline__ void chunk_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LATER) : "memory");
}

// S += sum_j x_j k_j on this wave's 32 columns, x[t][jj] the weighed value of the token in slot jj of k-step t.
// Three bf16 parts of x where the state is a result (`whole`), two where it only feeds O.
template <typename T, int D>
__device__ __forceinline__ void add_to_state(f32x16 (&S)[D / 32], const typename Vec8<T>::type (&kc)[2][D / 32], float (&x)[2][8], bool whole) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const Parts<2> xv = split<2>(x[t]);
    Parts<kParts<T>> kf[D / 32];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      kf[dt] = as_parts<T>(kc[t][dt]);
      S[dt] = mma_parts(kf[dt], xv, S[dt]);
    }
    if (whole) {
#pragma unroll
      for (int jj = 0; jj < 8; ++jj) x[t][jj] = (x[t][jj] - (float)xv.v[0][jj]) - (float)xv.v[1][jj];
      const Parts<1> rest = split<1>(x[t]);
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) {
        S[dt] = mma(kf[dt].v[0], rest.v[0], S[dt]);
        if constexpr (kParts<T> == 2) S[dt] = mma(kf[dt].v[1], xv.v[1], S[dt]);
      }
    }
  }
}

// lam^(n-1-j+e) for the tokens j of this lane's slots in a chunk of n.
__device__ __forceinline__ void token_factors(float (&f)[2][8], float g2, int n, int e, float s_state, int h) {
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int jj = 0; jj < 8; ++jj) {
      const int left = n - 1 - (16 * t + 4 * h + (jj & 3) + (jj < 4 ? 0 : 8));
      f[t][jj] = decay(g2, left < 0 ? 0 : left + e) * s_state;
    }
}

// Where register 4 g + r of accumulator tile dt of a lane lies in a state.
__device__ __forceinline__ int state_row(int dt, int g, int h) { return 32 * dt + 16 * (g >> 1) + 8 * h + 4 * (g & 1); }
__device__ __forceinline__ int state_col(int w, int lane) { return 32 * w + sigma(lane & 31); }

// The head (b H + h) of a block.  Neighbours in a token run side by side; the query heads of one key head are eight blocks apart,
// which is one XCD (blocks go to the eight in turn), whose L2 serves their reads of K and V.  (D 128, 8 key heads of 32: forward
// B8 S4096 225 -> 217 us, B1 S32768 286 -> 280, backward B8 S2048 421 -> 412.)
__device__ __forceinline__ int head_of(const Params& p, int i) {
  if (p.group == 1) return i;
  const int span = 8 * p.group, at = i % span;
  return i - at + (at & 7) * p.group + (at >> 3);
}

// Each segment's own state (from zero), in accumulator order; that of the last one is not needed, so segments are whole here.
// Every token is weighed for the end of the segment at once.  Chunks whose weights are all zero in fp32 (lam^n below 2^-150) add
// nothing and are not read.
template <typename T, int D>
__global__ __launch_bounds__(D * 2) __attribute__((amdgpu_waves_per_eu(2, 2))) void segment_states_kernel(const Params p) {
  typedef Tile<T, D> TL;
  constexpr int STAGE = 2 * TL::BYTES;
  __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];  // two stages of K, V
  const Problem& pr = p.pr[2 * blockIdx.y];  // dk's states are dv's transposed
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int heads = p.B * p.H, seg = blockIdx.x / heads, bh = head_of(p, blockIdx.x % heads);
  const int b = bh / p.H, head = bh % p.H;
  const int len = __builtin_amdgcn_readfirstlane(length_of(p, b));
  const int t_beg = seg * p.seg_chunks * C, t_end = t_beg + p.seg_chunks * C;
  if (t_end >= len) return;  // nothing comes after
  const float g2 = head_log2(p, head);
  int t_first = t_beg;
  if (g2 < 0.f) {
    const float live = 150.f / -g2;
    if (live < (float)(t_end - t_beg)) t_first = max(t_beg, t_end - ((int)live / C + 1) * C);
  }
  t_first = __builtin_amdgcn_readfirstlane(t_first);
  int t0 = t_end - C;
  f32x16 S[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) S[dt][i] = 0.f;
  Mover<T, D> km, vm;
  km.bind(pr.k, b, head, len, pr.reverse, t0, tid);
  vm.bind(pr.v, b, head, len, pr.reverse, t0, tid);
  km.step = -km.step;
  vm.step = -vm.step;
  float f[2][8];
  token_factors(f, g2, C, pr.e, pr.s_state, h);
  const uint32_t lds = lds_address(smem);
  const ColAddresses<T, D> at(lds, lds + TL::BYTES, w, lane);
  auto issue = [&](uint32_t stage_at) {
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds + stage_at + 2048 * w);
    km.load(to);
    vm.load(to + TL::BYTES);
  };
  issue(0);
  auto step = [&](auto stage) {
    constexpr int AT = decltype(stage)::value * STAGE;
    chunk_barrier<0>();
    if (t0 > t_first) issue(STAGE - AT);
    const float rest = decay(g2, t_end - t0 - C);
    float x[2][8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const typename TL::V8 vf = TL::col_frag(at.v_lo + AT + 16 * t * TL::RB, at.v_hi + AT + 16 * t * TL::RB);
#pragma unroll
      for (int jj = 0; jj < 8; ++jj) x[t][jj] = (float)vf[jj] * (f[t][jj] * rest);
    }
    typename TL::V8 kc[2][D / 32];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
        kc[t][dt] = TL::col_frag(at.k_lo[dt] + AT + 16 * t * TL::RB, at.k_hi[dt] + AT + 16 * t * TL::RB);
    add_to_state<T, D>(S, kc, x, true);
    t0 -= C;
  };
  while (t0 >= t_first) {
    step(std::integral_constant<int, 0>{});
    if (t0 >= t_first) step(std::integral_constant<int, 1>{});
  }
  float* to = pr.seg_states + ((int64_t)bh * p.n_seg + seg) * (D * D);
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4*>(to + (((w * (D / 32) + dt) * 4 + g) * 64 + lane) * 4) = f32x4{S[dt][4 * g], S[dt][4 * g + 1], S[dt][4 * g + 2], S[dt][4 * g + 3]};
}

// Segment states in order: what segment m added becomes the state before segment m.  One thread per four elements.
template <int D>
__global__ __launch_bounds__(256) void scan_states_kernel(const Params p) {
  const Problem& pr = p.pr[2 * blockIdx.y];
  float* transposed = blockIdx.y == 0 && p.pr[1].out ? p.pr[1].seg_states : nullptr;
  constexpr int PER = D * D / 1024;  // blocks per head
  const int bh = blockIdx.x / PER;
  const int at = (blockIdx.x % PER) * 1024 + threadIdx.x * 4;
  const int b = bh / p.H, head = bh % p.H;
  const int lane = (at >> 2) & 63, g = (at >> 8) & 3, dt = (at >> 10) % (D / 32), w = (at >> 10) / (D / 32);
  const int dk = state_row(dt, g, lane >> 5), dv = state_col(w, lane);
  const int len = length_of(p, b);
  const float g2 = head_log2(p, head);
  f32x4 S = {0.f, 0.f, 0.f, 0.f};
  if (pr.state0) {
    const float* s0 = pr.state0 + (int64_t)bh * (D * D);
#pragma unroll
    for (int r = 0; r < 4; ++r) S[r] = pr.state0_t ? s0[dv * D + dk + r] : s0[(dk + r) * D + dv];
  }
  float* ws = pr.seg_states + (int64_t)bh * p.n_seg * (D * D) + at;
  const int seg_len = p.seg_chunks * C;
  const float lam = decay(g2, seg_len);
  constexpr int BATCH = 8;  // loads in flight (32 segments, B1 S8192 H8 D128: forward 48 -> 42 us; four segments: no change)
  for (int m0 = 0; m0 * seg_len < len; m0 += BATCH) {
    f32x4 own[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if ((m0 + i + 1) * seg_len < len) own[i] = *reinterpret_cast<const f32x4*>(ws + (int64_t)(m0 + i) * (D * D));
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int m = m0 + i;
      if (m * seg_len >= len) break;
      *reinterpret_cast<f32x4*>(ws + (int64_t)m * (D * D)) = S;
      if (transposed) {  // element (dv, dk + r) of that problem's state
        const int slot = ((dk / 32 * (D / 32) + dv / 32) * 4 + 2 * ((dv >> 4) & 1) + ((dv >> 2) & 1)) * 64 + 32 * ((dv >> 3) & 1);
        float* to = transposed + ((int64_t)bh * p.n_seg + m) * (D * D) + (dv & 3);
#pragma unroll
        for (int r = 0; r < 4; ++r) to[(slot + sigma((dk + r) & 31)) * 4] = S[r];
      }
      if ((m + 1) * seg_len < len) S = S * lam + own[i];
    }
  }
  if (len == 0 && pr.state_out) {  // otherwise the last segment ends with it
    float* so = pr.state_out + (int64_t)bh * (D * D);
#pragma unroll
    for (int r = 0; r < 4; ++r) so[(dk + r) * D + dv] = S[r];
  }
}

// Which problem, and which of its n blocks, block i is.  dv and dk of a head read the same rows of q and do in the same order:
// they are started together on one XCD (blocks go to the eight of them in turn), whose L2 then serves one of the two.
__device__ __forceinline__ void block_of(const Params& p, int i, int n, int& problem, int& block) {
  if (!p.pr[1].out || i >= 2 * n) {
    problem = i < n ? 0 : 2;
    block = i < n ? i : i - 2 * n;
    return;
  }
  const int whole = n & ~7, rest = n - whole;
  if (i < 2 * whole) {
    problem = (i >> 3) & 1;
    block = ((i >> 4) << 3) + (i & 7);
  } else {
    problem = i - 2 * whole >= rest;
    block = i - whole - problem * rest;
  }
}

template <typename T, int D>
__global__ __launch_bounds__(D * 2) __attribute__((amdgpu_waves_per_eu(2, 2))) void linear_attn_kernel(const Params p) {
  typedef typename Vec8<T>::type V8;
  typedef Tile<T, D> TL;
  constexpr int OP = kParts<T>;  // parts of S and P as operands of O
  constexpr int STAGE = 3 * TL::BYTES;
  __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];  // two stages of Q, K, V
  const int heads = p.B * p.H;
  int problem, at_block;
  block_of(p, blockIdx.x, heads * p.n_seg, problem, at_block);
  const Problem& pr = p.pr[problem];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int seg = at_block / heads, bh = head_of(p, at_block % heads);
  const int b = bh / p.H, head = bh % p.H;
  const int len = __builtin_amdgcn_readfirstlane(length_of(p, b));
  const int t_beg = seg * p.seg_chunks * C;
  const int s_end = t_beg + p.seg_chunks * C < p.S ? t_beg + p.seg_chunks * C : p.S;
  const int t_end = s_end < len ? s_end : len;
  const float g2 = head_log2(p, head);
  const int64_t out0 = b * pr.os[0] + head * pr.os[1];

  auto clear_rows_behind = [&] {  // zeros
    const int from = t_beg > len ? t_beg : len;
    for (int idx = tid; idx < (s_end - from) * (D / 8); idx += D * 2) {
      const int64_t at = out0 + (int64_t)(from + idx / (D / 8)) * pr.os[2] + (idx % (D / 8)) * 8;
      const u32x4 zero = {0, 0, 0, 0};
      if (pr.out_f32) {
        u32x4* o = reinterpret_cast<u32x4*>(reinterpret_cast<float*>(pr.out) + at);
        o[0] = zero;
        o[1] = zero;
      } else {
        *reinterpret_cast<u32x4*>(reinterpret_cast<T*>(pr.out) + at) = zero;
      }
    }
  };
  if (p.n_seg > 1 && t_beg >= t_end) return clear_rows_behind();

  Mover<T, D> qm, km, vm;
  qm.bind(pr.q, b, head, len, pr.reverse, t_beg, tid);
  km.bind(pr.k, b, head, len, pr.reverse, t_beg, tid);
  vm.bind(pr.v, b, head, len, pr.reverse, t_beg, tid);
  const uint32_t lds = lds_address(smem);
  auto issue = [&](int t0, int stage_at) {
    if (t_end - t0 >= C) {
      const uint32_t to = __builtin_amdgcn_readfirstlane(lds + stage_at + 2048 * w);
      qm.load(to);
      km.load(to + TL::BYTES);
      vm.load(to + 2 * TL::BYTES);
    } else {
      qm.load_tail(t_end - t0, smem + stage_at, tid);
      km.load_tail(t_end - t0, smem + stage_at + TL::BYTES, tid);
      vm.load_tail(t_end - t0, smem + stage_at + 2 * TL::BYTES, tid);
    }
  };

  // the state before the segment
  f32x16 S[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) S[dt][i] = 0.f;
  if (p.n_seg > 1) {
    const float* from = pr.seg_states + ((int64_t)bh * p.n_seg + seg) * (D * D);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(from + (((w * (D / 32) + dt) * 4 + g) * 64 + lane) * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) S[dt][4 * g + r] = x[r];
      }
  } else if (pr.state0) {
    const float* s0 = pr.state0 + (int64_t)bh * (D * D);
    const int dv = state_col(w, lane);
    if (pr.state0_t) {
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(s0 + dv * D + state_row(dt, g, h));
#pragma unroll
          for (int r = 0; r < 4; ++r) S[dt][4 * g + r] = x[r];
        }
    } else {
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) S[dt][i] = s0[(state_row(dt, i >> 2, h) + (i & 3)) * D + dv];
    }
  }
  if (t_beg < t_end) issue(t_beg, 0);
  // the loads of the state end here: left to the first use, the wait for them would stand inside the loop and hold up its prefetch
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) asm volatile("" : "+v"(S[dt]));
  const bool keep_state = pr.state_out && (p.n_seg == 1 || (t_beg < t_end && t_end == len));  // this segment ends with the last token

  if (t_beg < t_end) {
    // what does not change from chunk to chunk: factors, addresses
    float f[2][8];
    token_factors(f, g2, C, pr.e, pr.s_state, h);
    const float row_f = decay(g2, l32 + 1 - pr.e) * pr.s_inter;
    float p_f[16];  // of P^T: lane = query, register 4 g + r = key 8 g + 4 h + r
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int d = l32 - (8 * (i >> 2) + 4 * h + (i & 3));
      p_f[i] = d < 0 ? 0.f : decay(g2, d) * pr.s_intra;
    }
    const float lam_c = decay(g2, C);
    const ColAddresses<T, D> at(lds + TL::BYTES, lds + 2 * TL::BYTES, w, lane);
    uint32_t row_at[D / 16];
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      row_at[t] = TL::row_address(lds, t, lane);
      asm volatile("" : "+v"(row_at[t]));
    }
    // lane: query l32, columns 32 w + 16 t + 8 h .. +7 in registers 8 t .. 8 t + 7
    const int out_size = pr.out_f32 ? 4 : 2;
    const int64_t out_row = (pr.reverse ? -pr.os[2] : pr.os[2]) * out_size;
    char* out = reinterpret_cast<char*>(pr.out) + (out0 + (int64_t)(pr.reverse ? len - 1 - t_beg : t_beg) * pr.os[2] + 32 * w + 8 * h) * out_size + l32 * out_row;

    auto step = [&](auto stage, int t0) {
      constexpr int AT = decltype(stage)::value * STAGE;
      const int n = t_end - t0 < C ? t_end - t0 : C;
      if (t0 == t_beg)
        chunk_barrier<0>();
      else  // two stores or more of the chunk before have been issued since
        chunk_barrier<2>();
      if (t0 + C < t_end) issue(t0 + C, STAGE - AT);

      // P^T = K Q^T and O^T = S^T Q^T from the same rows of Q; each query of O scaled by its decay
      // (rows are read AHEAD k-steps before they are used, where the compiler would wait for each pair: a chunk of one wave a SIMD
      // takes 1.38 us instead of 1.5; fp16's parts leave registers for two)
      constexpr int AHEAD = kParts<T> == 1 ? 4 : 2;
      V8 qr[AHEAD], kr[AHEAD], vf[2], kc[2][D / 32];
#pragma unroll
      for (int t = 0; t < AHEAD; ++t) {
        qr[t] = TL::row_frag(row_at[t] + AT);
        kr[t] = TL::row_frag(row_at[t] + AT + TL::BYTES);
      }
      __builtin_amdgcn_sched_barrier(0);
      f32x16 P, O;
#pragma unroll
      for (int i = 0; i < 16; ++i) P[i] = O[i] = 0.f;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        P = mma(kr[t % AHEAD], qr[t % AHEAD], P);
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = S[t >> 1][8 * (t & 1) + i];
        O = mma_parts(split<OP>(x), as_parts<T>(qr[t % AHEAD]), O);
        __builtin_amdgcn_sched_barrier(0);
        if (t + AHEAD < D / 16) {
          qr[t % AHEAD] = TL::row_frag(row_at[t + AHEAD] + AT);
          kr[t % AHEAD] = TL::row_frag(row_at[t + AHEAD] + AT + TL::BYTES);
        } else if (t + AHEAD < D / 16 + 2) {
          const int i = t + AHEAD - D / 16;
          vf[i] = TL::col_frag(at.v_lo + AT + 16 * i * TL::RB, at.v_hi + AT + 16 * i * TL::RB);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
          kc[t][dt] = TL::col_frag(at.k_lo[dt] + AT + 16 * t * TL::RB, at.k_hi[dt] + AT + 16 * t * TL::RB);
      O *= row_f;

      // O^T += V^T P^T
      const f32x16 before = O;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = P[8 * t + i] * p_f[8 * t + i];
        O = mma_parts(as_parts<T>(vf[t]), split<OP>(x), O);
      }
      float worst = fabsf(O[0]);
#pragma unroll
      for (int i = 1; i < 16; ++i) worst = __builtin_elementwise_maximum(worst, fabsf(O[i]));
      if (__builtin_expect(__any(!(worst < __builtin_inff())), 0)) {
        // The scores of later tokens are zeros, but zero times a value that is not finite is not zero, and a score that is not finite
        // does not become zero: here the tokens come one by one, each kept from the rows before it (9 us a
        // chunk more, 12 in fp16, also in those after it, whose state holds the value)
        O = before;
        asm volatile("" : "+v"(P));  // (weighed again: the loop needs the registers)
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
          asm volatile("" ::: "memory");
          f32x16 with = O;
          const int slot = (j & 15) - 4 * h;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j >> 4 != t) continue;
            float x[8];
            V8 v = TL::col_frag(at.v_lo + AT + 16 * t * TL::RB, at.v_hi + AT + 16 * t * TL::RB);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const bool here = 8 * (i >> 2) + (i & 3) == slot;
              x[i] = here ? P[8 * t + i] * p_f[8 * t + i] : 0.f;
              v[i] = here ? v[i] : (T)0.f;
            }
            with = mma_parts(as_parts<T>(v), split<OP>(x), with);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) O[i] = l32 < j ? O[i] : with[i];
        }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int t = 0; t < 2; ++t) {  // (read again, likewise)
          vf[t] = TL::col_frag(at.v_lo + AT + 16 * t * TL::RB, at.v_hi + AT + 16 * t * TL::RB);
#pragma unroll
          for (int dt = 0; dt < D / 32; ++dt)
            kc[t][dt] = TL::col_frag(at.k_lo[dt] + AT + 16 * t * TL::RB, at.k_hi[dt] + AT + 16 * t * TL::RB);
        }
      }

      if (l32 < n) {
        if (pr.out_f32) {
          float* o = reinterpret_cast<float*>(out);
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(o + 16 * (g >> 1) + 4 * (g & 1)) = f32x4{O[4 * g], O[4 * g + 1], O[4 * g + 2], O[4 * g + 3]};
        } else {
          T* o = reinterpret_cast<T*>(out);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            V8 y;
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = (T)O[8 * t + i];
            *reinterpret_cast<V8*>(o + 16 * t) = y;
          }
        }
      }
      out += C * out_row;

      if (t0 + C < t_end || keep_state) {
        float lam_n = lam_c;
        if (n < C) {
          token_factors(f, g2, n, pr.e, pr.s_state, h);
          lam_n = decay(g2, n);
        }
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) S[dt] *= lam_n;
        float x[2][8];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int jj = 0; jj < 8; ++jj) x[t][jj] = (float)vf[t][jj] * f[t][jj];
        add_to_state<T, D>(S, kc, x, keep_state);
      }
    };
    for (int t0 = t_beg; t0 < t_end; t0 += 2 * C) {
      step(std::integral_constant<int, 0>{}, t0);
      if (t0 + C < t_end) step(std::integral_constant<int, 1>{}, t0 + C);
    }
  }

  clear_rows_behind();
  if (keep_state) {
    float* so = pr.state_out + (int64_t)bh * (D * D);
    const int dv = state_col(w, lane);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) so[(state_row(dt, i >> 2, h) + (i & 3)) * D + dv] = S[dt][i];
  }
}

// Shared heads: the gradient of a key / value head is the sum over its query heads, in their order.  part: [B, H, S, D] fp32.
struct GroupSum {
  const float* part[2];
  void* out[2];
  int64_t os[2][3];
  int64_t n;      // B * Hkv * S * D / 4
  int Hkv, S, D, group;
};
template <typename T>
__global__ __launch_bounds__(256) void group_sum_kernel(const GroupSum p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.n) return;
  const int per_row = p.D / 4;
  const int c = (int)(i % per_row) * 4;
  const int64_t row = i / per_row;
  const int s = (int)(row % p.S);
  const int hk = (int)((row / p.S) % p.Hkv);
  const int64_t b = row / ((int64_t)p.S * p.Hkv);
  const float* src = p.part[blockIdx.y] + (((b * p.Hkv + hk) * p.group) * p.S + s) * (int64_t)p.D + c;
  f32x4 a = {0.f, 0.f, 0.f, 0.f};  // (no query heads at all)
  if (p.group) a = *reinterpret_cast<const f32x4*>(src);
  for (int g = 1; g < p.group; ++g) a += *reinterpret_cast<const f32x4*>(src + (int64_t)g * p.S * p.D);
  typedef T T4 __attribute__((ext_vector_type(4)));
  T4 y;
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = (T)a[r];
  const int64_t* os = p.os[blockIdx.y];
  *reinterpret_cast<T4*>(reinterpret_cast<T*>(p.out[blockIdx.y]) + b * os[0] + hk * os[1] + s * os[2] + c) = y;
}

// One token: the state of a head is read, updated and written in place, and the row q S comes out of the same pass.
// Bound by the state's bytes (two ways): B64 H32 D128 45.4 us, 268 MB, 5.9 TB/s on fresh states; one sequence 3.0 us.  A workgroup
// takes W columns of one head's state, 16 bytes a lane, with streamed loads and stores (cached ones: 54 us).
struct StepParams {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* state;
  const float* log_decay;
  int64_t qs[2], ks[2], vs[2], os[2], ss[2];  // batch, head
  int H, group;
  float scale;
};
template <typename T, int D, int W>
__global__ __launch_bounds__(256) void linear_attn_step_kernel(const StepParams p) {
  constexpr int LANES = W / 4, ROWS = 256 / LANES;  // lanes a row, rows at a time
  __shared__ f32x4 red[4][LANES];
  const int tid = threadIdx.x, l = tid % LANES, c = l * 4, r0 = tid / LANES;
  const int part = blockIdx.x % (D / W), bh = blockIdx.x / (D / W);
  const int64_t b = bh / p.H;
  const int h = bh % p.H, hk = h / p.group;
  const int col = W * part + c;
  float* st = p.state + b * p.ss[0] + h * p.ss[1] + col;
  f32x4 S[D / ROWS];
#pragma unroll
  for (int i = 0; i < D / ROWS; ++i) S[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(st + (int64_t)(r0 + ROWS * i) * D));
  const T* q = reinterpret_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[1];
  const T* k = reinterpret_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[1];
  const T* v = reinterpret_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[1] + col;
  const float lam = expf(p.log_decay[h]);
  f32x4 vv, acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int r = 0; r < 4; ++r) vv[r] = to_f32(v[r]);
  float kr[D / ROWS], qr[D / ROWS];
#pragma unroll
  for (int i = 0; i < D / ROWS; ++i) kr[i] = to_f32(k[r0 + ROWS * i]), qr[i] = to_f32(q[r0 + ROWS * i]);
#pragma unroll
  for (int i = 0; i < D / ROWS; ++i) {
    S[i] = S[i] * lam + kr[i] * vv;
    __builtin_nontemporal_store(S[i], reinterpret_cast<f32x4*>(st + (int64_t)(r0 + ROWS * i) * D));
    acc += qr[i] * S[i];
  }
#pragma unroll
  for (int off = LANES; off < 64; off <<= 1)
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[r] += __shfl_xor(acc[r], off, kWave);
  if ((tid & 63) < LANES) red[tid >> 6][l] = acc;
  __syncthreads();
  if (tid < LANES) {
    f32x4 t = red[0][tid];
#pragma unroll
    for (int i = 1; i < 4; ++i) t += red[i][tid];
    T* o = reinterpret_cast<T*>(p.out) + b * p.os[0] + h * p.os[1] + col;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = from_f32<T>(t[r] * p.scale);
  }
}

// No tokens: the state before them is the state after them (zeros where there is none).
__global__ __launch_bounds__(256) void carry_state_kernel(const f32x4* __restrict__ from, f32x4* __restrict__ to, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) to[i] = from ? from[i] : f32x4{0.f, 0.f, 0.f, 0.f};
}

// ------------------------------------------------------------------ host side
constexpr int64_t kMaxPitch = 1 << 26;  // elements between tokens: 32 rows stay inside 32-bit offsets

int64_t chunks_of(int64_t S) { return (S + C - 1) / C; }

// How many segments the tokens of a head are cut into, four chunks at least each.  Cutting reads K and V twice; not cutting leaves
// the chip idle where there are few heads, each of which takes 1.4 us a chunk.  With fewer than half the heads that fill it with
// one wave a SIMD they are cut to fill it once, or twice where that would be less than four segments.  Measured (us; uncut /
// segments: to fill the chip once, twice).  bf16 D 128 forward: 32 heads S 32768 1362 / 8: 336, 16: 356; 64 heads S 4096 179 / 4: 97,
// 8: 102; 96 heads S 4096 185 / 2: 159, 5: 135; 126 heads S 2048 96 / 2: 92, 4: 94; 128 heads S 2048 99 / 2: 98, 4: 100, S 8192
// 358 / 2: 321, 4: 323; 192 heads S 2048 109 / 2: 132.  Backward (three times the heads) 32 heads S 32768 1242 / 2: 1007, 5: 790, S
// 4096 158 / 2: 145, 5: 114; 42 heads 159 / 2: 151, 4: 139; 43 heads 161 / 3: 150; 48 heads 165 / 3: 160; 56 heads 167 / 3: 181; 64
// heads S 8192 358 / 4: 394.  bf16 D 64 forward: 64 heads S 4096 128 / 8: 57, 16: 63; 128 heads S 2048 68 / 4: 56, 8: 62; 192 heads
// 68 / 2: 83, 5: 75; 252 heads 69 / 2: 90, 4: 92; backward S 2048 64 heads 61 / 2: 76, 5: 61; 80 heads 64 / 2: 83, 4: 77.  So the step at
// half the chip is right for bf16 within 10 % (D 64 between half of it and a third: up to 25 % too early; D 128 with 128 long heads: 11 %
// too early).  fp16's chunk costs two to three times the products for the same bytes, so a cut pays for longer there: D 128 128
// heads S 2048 213 / 4: 161, S 8192 832 / 4: 562, backward 43 heads S 4096 384 / 3: 303; D 64 256 heads 135 / 4: 105, backward 86
// heads S 2048 200 / 3: 118; the rule does not tell the types apart.
void segments(int64_t heads, int64_t n_problems, int64_t S, int64_t D, int& n_seg, int& seg_chunks) {
  const int64_t chunks = chunks_of(S), groups = heads * n_problems, full = 256 * (128 / D);
  int64_t n = groups >= full / 2 ? 1 : (full / groups >= 4 ? full : 2 * full) / groups;
  if (n > chunks / 4) n = chunks / 4;
  if (n < 1) n = 1;
  seg_chunks = (int)((chunks + n - 1) / n);
  n_seg = (int)((chunks + seg_chunks - 1) / seg_chunks);
}

// Floats of the segment states of one problem.
int64_t state_floats(int64_t heads, int64_t n_problems, int64_t S, int64_t D) {
  int n_seg, seg_chunks;
  segments(heads, n_problems, S, D, n_seg, seg_chunks);
  return n_seg > 1 ? heads * n_seg * D * D : 0;
}

int check(int64_t B, int64_t H, int64_t Hkv, int64_t S, int64_t D, float scale, int dtype) {
  if (dtype != XG_BF16 && dtype != XG_F16) return XG_ERR_BAD_DTYPE;
  if (B < 0 || H < 0 || Hkv < 0 || S < 0 || (D != 64 && D != 128)) return XG_ERR_BAD_SHAPE;
  if (B && H && (Hkv == 0 || H % Hkv != 0)) return XG_ERR_BAD_SHAPE;
  if (!(scale == scale) || fabsf(scale) > 3.0e38f) return XG_ERR_BAD_ARG;
  if (S > (1 << 30) || B > (1 << 24) || H > (1 << 24) || B * H > (1 << 20)) return XG_ERR_TOO_LARGE;
  return XG_OK;
}

int fill(int64_t (&to)[3], const int64_t* from) {
  if (!from) return XG_ERR_NULL_PTR;
  for (int i = 0; i < 3; ++i) {
    if (from[i] < 0) return XG_ERR_BAD_SHAPE;
    if (from[i] % 8) return XG_ERR_BAD_ALIGN;
    to[i] = from[i];
  }
  return from[2] < kMaxPitch ? XG_OK : XG_ERR_TOO_LARGE;
}

int fill(Operand& o, const void* p, const int64_t* s, int group) {
  if (!p) return XG_ERR_NULL_PTR;
  if (!aligned_to(p, 16)) return XG_ERR_BAD_ALIGN;
  o.p = p;
  o.group = group;
  return fill(o.s, s);
}

// Whether the states [heads, D, D] at a and b share memory.
bool states_overlap(const float* a, const float* b, int64_t heads, int64_t D) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b), bytes = (uintptr_t)(heads * D * D) * 4;
  return a && b && (x < y ? y - x : x - y) < bytes;
}

// Whether a kernel could reach p: not where there is no device, nor in host memory that HIP does not know.
bool on_gpu(const void* p) {
  hipPointerAttribute_t at;
  const hipError_t e = hipPointerGetAttributes(&at, p);
  if (e == hipSuccess) return at.type != hipMemoryTypeUnregistered;
  (void)hipGetLastError();  // (it would be taken for the next launch's)
  return e != hipErrorNoDevice;
}

// The state results of a call without tokens.  Such a call refuses no pointer, as it reads nothing through q, k and v; so what it
// does read and write is looked at first, and left alone where no kernel could reach it.
int carry_state(const float* from, float* to, int64_t heads, int64_t D, hipStream_t st) {
  if (!to || from == to || heads == 0) return XG_OK;  // (in place)
  if (!aligned_to(to, 16) || (from && !aligned_to(from, 16))) return XG_ERR_BAD_ALIGN;
  if (states_overlap(from, to, heads, D)) return XG_ERR_BAD_ARG;
  if (!on_gpu(to) || (from && !on_gpu(from))) return XG_OK;
  const int64_t n = heads * D * D / 4, blocks = (n + 255) / 256;
  hipLaunchKernelGGL(carry_state_kernel, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, st, reinterpret_cast<const f32x4*>(from),
                     reinterpret_cast<f32x4*>(to), n);
  return status_from_hip(hipGetLastError());
}

template <typename T, int D>
int launch(const Params& p, int n_problems, hipStream_t st) {
  const dim3 grid((unsigned)(p.B * p.H * p.n_seg), (unsigned)n_problems), all(grid.x * grid.y), block(D * 2);
  if (p.n_seg > 1) {
    const unsigned sums = n_problems == 1 ? 1 : 2;
    hipLaunchKernelGGL((segment_states_kernel<T, D>), dim3(grid.x, sums), block, 0, st, p);
    hipLaunchKernelGGL((scan_states_kernel<D>), dim3((unsigned)(p.B * p.H * (D * D / 1024)), sums), dim3(256), 0, st, p);
  }
  hipLaunchKernelGGL((linear_attn_kernel<T, D>), all, block, 0, st, p);
  return status_from_hip(hipGetLastError());
}

int sum_groups(const GroupSum& p, int dtype, hipStream_t st) {
  if (p.n > 0xffffff00LL) return XG_ERR_TOO_LARGE;  // threads of a launch
  const dim3 grid((unsigned)((p.n + 255) / 256), 2);
  if (dtype == XG_BF16)
    hipLaunchKernelGGL((group_sum_kernel<bf16_t>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((group_sum_kernel<f16_t>), grid, dim3(256), 0, st, p);
  return status_from_hip(hipGetLastError());
}

int launch_any(const Params& p, int n_problems, int64_t D, int dtype, hipStream_t st) {
  if (dtype == XG_BF16) return D == 64 ? launch<bf16_t, 64>(p, n_problems, st) : launch<bf16_t, 128>(p, n_problems, st);
  return D == 64 ? launch<f16_t, 64>(p, n_problems, st) : launch<f16_t, 128>(p, n_problems, st);
}

}  // namespace linattn
}  // namespace xg

extern "C" int64_t xg_linear_attn_workspace_floats(int64_t B, int64_t H, int64_t S, int64_t D) {
  using namespace xg::linattn;
  if (check(B, H, H, S, D, 1.f, XG_BF16) != XG_OK || B == 0 || H == 0 || S == 0) return 0;
  return state_floats(B * H, 1, S, D);
}

extern "C" int xg_linear_attn(const void* q, const void* k, const void* v, const float* log_decay, const float* state, const void* lengths,
                              int lengths_64bit, void* out, float* state_out, float* workspace, int64_t workspace_floats, int64_t B, int64_t H,
                              int64_t Hkv, int64_t S, int64_t D, const int64_t q_strides[3], const int64_t k_strides[3],
                              const int64_t v_strides[3], const int64_t o_strides[3], float scale, int dtype, xg_stream_t stream) {
  using namespace xg;
  using namespace xg::linattn;
  if (int rc = check(B, H, Hkv, S, D, scale, dtype)) return rc;
  if (B == 0 || H == 0) return XG_OK;
  if (S == 0) return carry_state(state, state_out, B * H, D, reinterpret_cast<hipStream_t>(stream));
  if (!log_decay || !out) return XG_ERR_NULL_PTR;
  if (!aligned_to(out, 16) || !aligned_to(log_decay, 4) || (state && !aligned_to(state, 16)) || (state_out && !aligned_to(state_out, 16)) ||
      (workspace && !aligned_to(workspace, 16)) || (lengths && !aligned_to(lengths, lengths_64bit ? 8 : 4)))
    return XG_ERR_BAD_ALIGN;
  // in place, each thread writes what it has read; shifted, a head's results would land in another's initial state
  if (state != state_out && states_overlap(state, state_out, B * H, D)) return XG_ERR_BAD_ARG;
  Params p{};
  const int group = (int)(H / Hkv);
  if (int rc = fill(p.pr[0].q, q, q_strides, 1)) return rc;
  if (int rc = fill(p.pr[0].k, k, k_strides, group)) return rc;
  if (int rc = fill(p.pr[0].v, v, v_strides, group)) return rc;
  if (int rc = fill(p.pr[0].os, o_strides)) return rc;
  p.log_decay = log_decay;
  p.lengths = lengths;
  p.len64 = lengths_64bit != 0;
  p.B = (int)B;
  p.H = (int)H;
  p.S = (int)S;
  p.group = B * H % (8 * group) == 0 ? group : 1;
  segments(B * H, 1, S, D, p.n_seg, p.seg_chunks);
  if (p.n_seg > 1) {
    if (!workspace) return XG_ERR_NULL_PTR;
    if (workspace_floats < B * H * p.n_seg * D * D) return XG_ERR_BAD_ARG;
  }
  Problem& pr = p.pr[0];
  pr.out = out;
  pr.state0 = state;
  pr.state_out = state_out;
  pr.seg_states = workspace;
  pr.s_intra = pr.s_inter = scale;
  pr.s_state = 1.f;
  return launch_any(p, 1, D, dtype, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int64_t xg_linear_attn_bwd_workspace_floats(int64_t B, int64_t H, int64_t Hkv, int64_t S, int64_t D) {
  using namespace xg::linattn;
  if (check(B, H, Hkv, S, D, 1.f, XG_BF16) != XG_OK || B == 0 || H == 0 || S == 0) return 0;
  return 3 * state_floats(B * H, 3, S, D) + (H != Hkv ? 2 * B * H * S * D : 0);
}

extern "C" int xg_linear_attn_bwd(const void* q, const void* k, const void* v, const float* log_decay, const float* state, const void* lengths,
                                  int lengths_64bit, const void* d_out, const float* d_state_out, void* dq, void* dk, void* dv, float* d_state,
                                  float* workspace, int64_t workspace_floats, int64_t B, int64_t H, int64_t Hkv, int64_t S, int64_t D,
                                  const int64_t q_strides[3], const int64_t k_strides[3], const int64_t v_strides[3],
                                  const int64_t do_strides[3], const int64_t dq_strides[3], const int64_t dk_strides[3],
                                  const int64_t dv_strides[3], float scale, int dtype, xg_stream_t stream) {
  using namespace xg;
  using namespace xg::linattn;
  if (int rc = check(B, H, Hkv, S, D, scale, dtype)) return rc;
  if (B == 0) return XG_OK;
  if (S == 0) return carry_state(d_state_out, d_state, B * H, D, reinterpret_cast<hipStream_t>(stream));
  GroupSum gs{};
  gs.n = B * Hkv * S * D / 4;
  gs.Hkv = (int)Hkv;
  gs.S = (int)S;
  gs.D = (int)D;
  if (H == 0) {  // sums over no query heads
    if (Hkv == 0) return XG_OK;
    if (Hkv > (1 << 24) || B * Hkv > (1 << 20)) return XG_ERR_TOO_LARGE;  // (as check() for the query heads)
    gs.out[0] = dv;
    gs.out[1] = dk;
    if (!dk || !dv) return XG_ERR_NULL_PTR;
    if (!aligned_to(dk, 16) || !aligned_to(dv, 16)) return XG_ERR_BAD_ALIGN;
    if (int rc = fill(gs.os[0], dv_strides)) return rc;
    if (int rc = fill(gs.os[1], dk_strides)) return rc;
    return sum_groups(gs, dtype, reinterpret_cast<hipStream_t>(stream));
  }
  if (!log_decay || !dq || !dk || !dv) return XG_ERR_NULL_PTR;
  for (const void* t : {(const void*)dq, (const void*)dk, (const void*)dv, (const void*)state, (const void*)d_state_out, (const void*)d_state,
                        (const void*)workspace})
    if (t && !aligned_to(t, 16)) return XG_ERR_BAD_ALIGN;
  if (!aligned_to(log_decay, 4) || (lengths && !aligned_to(lengths, lengths_64bit ? 8 : 4))) return XG_ERR_BAD_ALIGN;
  // dq's workgroups read state and dk's read d_state_out while dv's write d_state
  if (states_overlap(state, d_state, B * H, D) || states_overlap(d_state_out, d_state, B * H, D)) return XG_ERR_BAD_ARG;
  Params p{};
  const int group = (int)(H / Hkv);
  Operand oq, ok, ov, og;
  if (int rc = fill(oq, q, q_strides, 1)) return rc;
  if (int rc = fill(ok, k, k_strides, group)) return rc;
  if (int rc = fill(ov, v, v_strides, group)) return rc;
  if (int rc = fill(og, d_out, do_strides, 1)) return rc;
  p.log_decay = log_decay;
  p.lengths = lengths;
  p.len64 = lengths_64bit != 0;
  p.B = (int)B;
  p.H = (int)H;
  p.S = (int)S;
  p.group = B * H % (8 * group) == 0 ? group : 1;
  segments(B * H, 3, S, D, p.n_seg, p.seg_chunks);
  const int64_t need = xg_linear_attn_bwd_workspace_floats(B, H, Hkv, S, D);
  if (need) {
    if (!workspace) return XG_ERR_NULL_PTR;
    if (workspace_floats < need) return XG_ERR_BAD_ARG;
  }
  const int64_t seg_floats = state_floats(B * H, 3, S, D);
  float* partial = workspace + 3 * seg_floats;
  // dq = scale F(do, v, k), its state the transpose of the forward's
  Problem& a = p.pr[2];
  a.q = og;
  a.k = ov;
  a.v = ok;
  a.out = dq;
  if (int rc = fill(a.os, dq_strides)) return rc;
  a.state0 = state;
  a.state0_t = 1;
  a.s_intra = a.s_inter = scale;
  a.s_state = 1.f;
  // dv = F_rev(k, q, do): its state ends as the gradient of the initial state
  Problem& c = p.pr[0];
  c.q = ok;
  c.k = oq;
  c.v = og;
  c.out = dv;
  if (int rc = fill(c.os, dv_strides)) return rc;
  c.state0 = d_state_out;
  c.state_out = d_state;
  // dk = F_rev(v, do, q): the transposed state
  Problem& d = p.pr[1];
  d.q = ov;
  d.k = og;
  d.v = oq;
  d.out = dk;
  if (int rc = fill(d.os, dk_strides)) return rc;
  d.state0 = d_state_out;
  d.state0_t = 1;
  for (Problem* r : {&c, &d}) {
    r->reverse = r->e = 1;
    r->s_intra = r->s_state = scale;
    r->s_inter = 1.f;
  }
  for (int i = 0; i < 3; ++i) p.pr[i].seg_states = workspace + i * seg_floats;
  if (group > 1) {
    for (int i = 0; i < 2; ++i) {
      Problem& r = p.pr[i];
      gs.part[i] = partial + i * B * H * S * D;
      gs.out[i] = r.out;
      for (int j = 0; j < 3; ++j) gs.os[i][j] = r.os[j];
      r.out = partial + i * B * H * S * D;
      r.os[0] = H * S * D;
      r.os[1] = S * D;
      r.os[2] = D;
      r.out_f32 = 1;
    }
    gs.group = group;
    if (gs.n > 0xffffff00LL) return XG_ERR_TOO_LARGE;  // (before any launch)
  }
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (int rc = launch_any(p, 3, D, dtype, st)) return rc;
  return group > 1 ? sum_groups(gs, dtype, st) : XG_OK;
}

extern "C" int xg_linear_attn_step(const void* q, const void* k, const void* v, const float* log_decay, float* state, void* out, int64_t B,
                                   int64_t H, int64_t Hkv, int64_t D, const int64_t q_strides[2], const int64_t k_strides[2],
                                   const int64_t v_strides[2], const int64_t o_strides[2], const int64_t state_strides[2], float scale,
                                   int dtype, xg_stream_t stream) {
  using namespace xg;
  using namespace xg::linattn;
  if (int rc = check(B, H, Hkv, 1, D, scale, dtype)) return rc;
  if (B == 0 || H == 0) return XG_OK;
  if (!q || !k || !v || !log_decay || !state || !out || !q_strides || !k_strides || !v_strides || !o_strides || !state_strides)
    return XG_ERR_NULL_PTR;
  if (!aligned_to(q, 2) || !aligned_to(k, 2) || !aligned_to(v, 2) || !aligned_to(out, 2) || !aligned_to(state, 16) || !aligned_to(log_decay, 4))
    return XG_ERR_BAD_ALIGN;
  StepParams p;
  for (int i = 0; i < 2; ++i) {
    if (q_strides[i] < 0 || k_strides[i] < 0 || v_strides[i] < 0 || o_strides[i] < 0 || state_strides[i] < 0) return XG_ERR_BAD_SHAPE;
    if (state_strides[i] % 4) return XG_ERR_BAD_ALIGN;
    p.qs[i] = q_strides[i];
    p.ks[i] = k_strides[i];
    p.vs[i] = v_strides[i];
    p.os[i] = o_strides[i];
    p.ss[i] = state_strides[i];
  }
  // states that overlap would be updated by several workgroups at once
  const int64_t inner = D * D, s0 = state_strides[0], s1 = state_strides[1];
  if ((H > 1 && s1 < inner) || (B > 1 && s0 < inner) || (B > 1 && H > 1 && s0 < (H - 1) * s1 + inner && s1 < (B - 1) * s0 + inner))
    return XG_ERR_BAD_SHAPE;
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  p.state = state;
  p.log_decay = log_decay;
  p.H = (int)H;
  p.group = (int)(H / Hkv);
  p.scale = scale;
  // 64 columns a workgroup (B64 H32 D128, replayed from a graph, 47 us; 32: 49, 128: 49; D64 12.9), 32 where those are too few to give every compute unit one
  // (B1 H32 3.5 us with 64, 3.0 with 32; B8 H32 7.5 and 7.9)
  const bool wide = B * H * (D / 64) >= 256;
  const dim3 grid((unsigned)(B * H * (D / (wide ? 64 : 32))));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto go = [&](auto type, auto dim) {
    typedef decltype(type) T;
    constexpr int DIM = decltype(dim)::value;
    if (wide)
      hipLaunchKernelGGL((linear_attn_step_kernel<T, DIM, 64>), grid, dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL((linear_attn_step_kernel<T, DIM, 32>), grid, dim3(256), 0, st, p);
  };
  const std::integral_constant<int, 64> d64;
  const std::integral_constant<int, 128> d128;
  if (dtype == XG_BF16)
    D == 64 ? go(bf16_t{}, d64) : go(bf16_t{}, d128);
  else
    D == 64 ? go(f16_t{}, d64) : go(f16_t{}, d128);
  return status_from_hip(hipGetLastError());
}
