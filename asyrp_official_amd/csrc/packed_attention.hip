// packed_attention.hip -- attention over sequences packed behind each other, forward and backward (f16 / bf16 operands, fp32 sums).
//
//   S = scale * q k^T (causal: keys <= the query), P = softmax(S), o = P v
//   (kept per row for the backward: a reference r of S, in powers of two, and log2 of the sum of 2^(S - r))
//   dv = P^T do,  dS = P * (do v^T - delta) * scale with delta = rowsum(do * o),  dq = dS k,  dk = dS^T q
//
// All three kernels work on v_mfma_f32_32x32x16_{f16,bf16}.  A wave owns 32 queries (forward, dq) or 32 keys (dk/dv) as the COLUMNS of
// its products, so that a column's statistics are one value per lane and a row reduction is a sum over a lane's own 16 registers plus
// one exchange with lane ^ 32.  The result of a product (column = lane & 31, row = 8 (r / 4) + 4 (lane / 32) + r % 4) is used as the second
// operand of the next one without moving a value between lanes: the order in which a product runs over its inner index is free, so
// the first operand is simply read in the order in which the registers hold the second (rows {4h .. 4h+3, 8+4h .. 8+4h+3} of 16, h = lane / 32),
// by the transposing 16-bit LDS read, which hands a lane four rows of one column.
//
// P is rounded to the operands' type before P v and P^T do, dS before dS k and dS^T q (half a step per term, relative to it; f16 under powers of two, so that small ones keep their
// bits; dS as two terms where the mask cuts); every sum, the row maximum, the row sum and delta are fp32.  There is no atomic: dq and dk/dv are two kernels that each form S
// again (7 products instead of 5), and the result does not depend on the order in which workgroups run.
#include "kernels.h"
#include "../../include/asyrp.h"

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

namespace asyrp {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Frag;
template <> struct Frag<_Float16> {
  typedef _Float16 V __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 mma(V a, V b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Frag<__bf16> {
  typedef __bf16 V __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x16 mma(V a, V b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

constexpr int BM = 128;      // rows of a workgroup: four waves of 32
constexpr int BN = 64;       // rows of a tile in LDS
constexpr float LOG2E = 1.4426950408889634f;
template <typename T> constexpr bool is_f16 = std::is_same<T, _Float16>::value;
// What rounding took from an output is kept this many times as large: in f16 it would be nothing under outputs of 2^-14 or so.  It is never over the output's own size.
template <typename T> constexpr float FINER = is_f16<T> ? 2048.f : 1.f;

struct PackedAttnArgs {
  const void *q, *k, *v, *o, *dout;
  void *out, *dq, *dk, *dv;
  void* rest;                // [T][Hq][D]: what rounding took from o, times FINER (delta of the unrounded o halves what dq and dk are off); null: not kept
  // [Hq][T] reference and log2 of the sum.  Apart, since a large score less a reference close to it is exact, and their own sum is not: as one float, P was off by
  // 0.5 % at scores of 1e5 and of any size at 2e7.  (A subtraction an element: 2 % of the backward.)
  float2* sums;
  float* delta;              // [Hq][T]
  const int* cu;
  long long T;
  int nseq, Hq, Hkv, D, causal, fill_tail;
  int parts;                 // workgroups that share the queries of one key tile (dk / dv)
  int splits;                // workgroups that share the keys of one query tile (forward, dq)
  float* partial;            // where there are several, their sums: [parts][T][Hkv][dk, dv][D], [splits][T][Hq][D]
  float2* stats;             // [splits][Hq][T] reference (times scale, base 2) and sum of each part of the forward
  int tiles;                 // row tiles launched per head: T / BM + nseq + 1, at least one more than the sequences have
  float scale;
  long long q_t, q_h, k_t, k_h, v_t, v_h, o_t, o_h, do_t, do_h, dq_t, dq_h, dk_t, dk_h, dv_t, dv_h;
};

// LDS tile [rows][DP]: the 16-byte chunk c of row r lies at chunk c ^ swz(r).  Over 64 banks of 4 bytes both readers are free
// of conflicts: 16 lanes reading one chunk column of 16 rows, and 32 lanes reading four chunks of each of four rows.
template <int DP>
__device__ __forceinline__ int swz(int row) {
  if (DP == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
  if (DP == 64) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  return (row >> 2) & 3;
}
template <int DP>
__device__ __forceinline__ int lds_at(int row, int chunk) { return row * (DP * 2) + ((chunk ^ swz<DP>(row)) << 4); }

// first operand with rows `row0 + lane % 32`, inner index d = 16 * ks + 8 * (lane / 32) + 0..7
template <typename T, int DP>
__device__ __forceinline__ typename Frag<T>::V read_rows(const char* tile, int row0, int ks, int lane) {
  return *reinterpret_cast<const typename Frag<T>::V*>(tile + lds_at<DP>(row0 + (lane & 31), 2 * ks + (lane >> 5)));
}
// first operand with rows d = 32 * dt + lane % 32, inner index = the tile's rows row0 + {4h..4h+3, 8+4h..8+4h+3}
template <typename T, int DP>
__device__ __forceinline__ typename Frag<T>::V read_cols(const char* tile, int row0, int dt, int lane) {
  const int g = lane >> 4, i = lane & 15;
  const int row = row0 + 4 * (g >> 1) + (i >> 2), chunk = 4 * dt + 2 * (g & 1) + ((i & 3) >> 1), b = (i & 1) * 8;
  union { struct { s16x4 lo, hi; } s; typename Frag<T>::V v; } u;
  typedef __attribute__((address_space(3))) s16x4* lp;
  u.s.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(tile + lds_at<DP>(row, chunk) + b));
  u.s.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(tile + lds_at<DP>(row + 8, chunk) + b));
  return u.v;
}

// Stands in a branch that few tiles take: without it the compiler computes the branch's selects for every tile.
__device__ __forceinline__ void stay_a_branch() { asm volatile(""); }

// one row's fragment from global memory: d = 16 * ks + 8 * h + 0..7, zero beyond D or where the row is not there
template <typename T>
__device__ __forceinline__ typename Frag<T>::V load_frag(const T* row, int ks, int h, int D, bool there) {
  union { u32x4 u; typename Frag<T>::V v; } x;
  x.u = u32x4{0, 0, 0, 0};
  const int d = 16 * ks + 8 * h;
  if (there && d < D) x.u = *reinterpret_cast<const u32x4*>(row + d);
  return x.v;
}

// A tile [BN rows][DP] on its way from global memory to LDS, 16 bytes per lane and load, without passing through registers.
// LDS is written in lane order, so the swizzle is in the addresses that the lanes read.  Rows behind the sequence are read from its last
// row, columns behind D from the row's own columns: both are multiplied by probabilities or operands that are zero.
// (Inline assembly, since the compiler waits for all loads in flight before each such load that it can see behind another one;
// nothing is written but LDS, and the wait stands before the barrier that hands the tile over.)
template <typename T, int DP>
struct Tile {
  static constexpr int N = BN * (DP / 8) / 256;
  unsigned off[N];
  int rows;                  // rows that the offsets stand for
  unsigned stride;
  __device__ __forceinline__ void offsets(int have, int D, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = tid + i * 256, row = c / (DP / 8), col = ((c % (DP / 8)) ^ swz<DP>(row)) % (unsigned)(D / 8);
      off[i] = (unsigned)min(row, have - 1) * stride + col * 16;
    }
    rows = have;
  }
  __device__ __forceinline__ void init(long long st, int have, int D, int tid) {
    stride = (unsigned)st * sizeof(T);
    offsets(min(have, BN), D, tid);
  }
  // `have` (at least 1) rows from `base` on; both are the same in all lanes
  __device__ __forceinline__ void load(const T* base, int have, unsigned lds, int D, int tid) {
    have = min(have, BN);
    if (have != rows) offsets(have, D, tid);
    const unsigned w = __builtin_amdgcn_readfirstlane(lds + (tid >> 6) * 1024);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      unsigned keep;
      asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                   : "=&s"(keep)
                   : "v"(off[i]), "s"(base), "s"(w + i * 4096)
                   : "memory");
    }
  }
};
__device__ __forceinline__ unsigned lds_offset(const void* p) { return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p; }
// this wave's tiles have landed, and everybody's have behind the barrier
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }   // one instruction; results under 2^-126 are zero

// Calls step(i, place) for i0 <= i < i1 with place = (i - i0) % N as a constant: which of several LDS tiles a step works on is then part of its instructions, not an
// address to be computed for every read (forward 2 %, dq and dk / dv of 128-wide heads 4 %, at 8192 rows).
template <int N, typename F, int... P>
__device__ __forceinline__ void turns(int i0, int i1, F& step, std::integer_sequence<int, P...>) {
  for (int i = i0; i < i1; i += N) ((i + P < i1 ? step(i + P, std::integral_constant<int, P>()) : void()), ...);
}
template <int N, typename F>
__device__ __forceinline__ void turns(int i0, int i1, F& step) { turns<N>(i0, i1, step, std::make_integer_sequence<int, N>()); }

// a wave's sum, the same in all lanes: within rows of 16 by shifts, then from row to row
__device__ __forceinline__ int wave_sum(int v) {
#define ASYRP_DPP(CTRL, ROWS) v += __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false)
  ASYRP_DPP(0x111, 0xf);
  ASYRP_DPP(0x112, 0xf);
  ASYRP_DPP(0x114, 0xf);
  ASYRP_DPP(0x118, 0xf);
  ASYRP_DPP(0x142, 0xa);
  ASYRP_DPP(0x143, 0xc);
#undef ASYRP_DPP
  return __builtin_amdgcn_readlane(v, 63);
}

// The sequence and the row tile that tile number `t` of the launch stands for.  Up to 64 sequences: tiles are numbered sequence by sequence, and the numbers
// behind the last one share the rows behind the last sequence; every wave finds its own from the 64 lengths, summed over the wave.  More: sequence b's tiles are numbered from
// offset[b] / BM + b on, which leaves room for all of them and is found by looking at 64 offsets at a time (100000 sequences of one row: the forward 50 ms when the lengths in front were summed).
// Offsets are held inside [0, T] and never fall, so that no value of `cu` leads outside the tensors.
struct TileAt { long long start; int len, row0; int idle; int idles; int low, end; };
// lane `src`'s value as one that the compiler knows to be the same in all lanes (all lanes active, src < 64)
__device__ __forceinline__ int uniform(int v, int src) { return __builtin_amdgcn_readlane(v, __builtin_amdgcn_readfirstlane(src)); }
//
// Under the causal mask a tile's work goes with its distance from one end of its sequence, and the workgroups are dealt out in the tiles' order: up to 64
// sequences are therefore numbered heaviest first (`by_weight`: the last row tile of a sequence is the heaviest; `from_end`: the first
// is), which is the t-th largest of all (distance) values, found by bisection over the distance.
enum { IN_ORDER, BY_WEIGHT, BY_WEIGHT_FROM_END };
__device__ __forceinline__ TileAt find_tile(const int* cu, int nseq, long long T, int t, int tiles, int lane, int order) {
  TileAt f{0, 0, 0, 0, 1, 0, 0};
  if (order != IN_ORDER && nseq <= 64) {
    long long s = 0, e = 0;
    if (lane < nseq) { s = cu[lane]; e = cu[lane + 1]; }
    s = s < 0 ? 0 : s > T ? T : s;
    e = e < s ? s : e > T ? T : e;
    const int n = (int)((e - s + BM - 1) / BM);
    const int total = wave_sum(n);
    if (t < total) {
      int lo = 0, hi = (int)(T / BM) + 2;                 // tiles at distance >= lo: more than t; >= hi: at most t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (wave_sum(max(n - mid, 0)) > t) lo = mid; else hi = mid;
      }
      const int rank = t - wave_sum(max(n - lo - 1, 0));  // among the sequences that have a tile at this distance
      const unsigned long long has = __ballot(n > lo);
      const bool mine = n > lo && __popcll(has & ((1ull << lane) - 1)) == rank;
      const int src = __ffsll(__ballot(mine)) - 1;
      f.start = uniform((int)s, src);
      f.len = uniform((int)e, src) - (int)f.start;
      f.row0 = (order == BY_WEIGHT ? lo : uniform(n, src) - 1 - lo) * BM;
      return f;
    }
    f.idle = 1 + (t - total);
    f.idles = tiles - total;
    f.low = uniform((int)s, 0);
    f.end = uniform((int)e, nseq - 1);
    return f;
  }
  if (nseq > 64) {
    const auto first = [&](int b) { const long long s = cu[b]; return (int)((s < 0 ? 0 : s > T ? T : s) / BM) + b; };      // b's first tile
    const int behind = first(nseq);
    if (t >= behind) {
      const long long s = cu[0], e = cu[nseq];
      f.idle = 1 + (t - behind);
      f.idles = tiles - behind;
      f.low = (int)(s < 0 ? 0 : s > T ? T : s);
      f.end = (int)(e < f.low ? f.low : e > T ? T : e);
      return f;
    }
    f.idle = 1;                                           // a number that stands for nothing, unless the search ends at a sequence with so many tiles
    f.end = (int)T;
    int lo = 0, hi = nseq;
    while (hi - lo > 1) {
      const int step = (hi - lo + 63) / 64, b = lo + lane * step;
      const int at_or_before = __popcll(__ballot(b < hi && first(b < hi ? b : lo) <= t));
      if (!at_or_before) return f;
      lo += (at_or_before - 1) * step;
      hi = min(lo + step, hi);
    }
    long long s = cu[lo], e = cu[lo + 1];
    s = s < 0 ? 0 : s > T ? T : s;
    e = e < s ? s : e > T ? T : e;
    const long long row0 = (long long)(t - first(lo)) * BM;
    if (row0 >= 0 && row0 < e - s) {
      f.start = __builtin_amdgcn_readfirstlane((int)s);
      f.len = __builtin_amdgcn_readfirstlane((int)(e - s));
      f.row0 = __builtin_amdgcn_readfirstlane((int)row0);
      f.idle = 0;
    }
    return f;
  }
  long long s = 0, e = 0;
  if (lane < nseq) { s = cu[lane]; e = cu[lane + 1]; }
  s = s < 0 ? 0 : s > T ? T : s;
  e = e < s ? s : e > T ? T : e;                          // T < 2^31
  const int n = (int)((e - s + BM - 1) / BM);
  int sum = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(sum, o);
    if (lane >= o) sum += up;
  }
  const unsigned long long hit = __ballot(n > 0 && t >= sum - n && t < sum);
  if (hit) {
    const int src = __ffsll(hit) - 1;
    f.start = uniform((int)s, src);
    f.len = uniform((int)e, src) - (int)f.start;
    f.row0 = (t - uniform(sum - n, src)) * BM;
  } else {
    const int total = uniform(sum, 63);
    f.idle = 1 + (t - total);
    f.idles = tiles - total;
    f.low = uniform((int)s, 0);
    f.end = uniform((int)e, nseq - 1);
  }
  return f;
}

// zeros in the rows that belong to no sequence (behind the last one, before the first): the idle tiles of each head take them in turn
template <typename T>
__device__ __forceinline__ void zero_tail(T* p, long long st, long long sh, int head, int D, const TileAt& f, long long total, int tid) {
  const int chunks = D / 8;
  const long long rows = f.low + (total - f.end);
  for (long long i = f.idle - 1; i < rows; i += f.idles) {
    const long long row = i < f.low ? i : f.end + (i - f.low);
    for (int c = tid; c < chunks; c += 256) *reinterpret_cast<u32x4*>(p + row * st + head * sh + c * 8) = u32x4{0, 0, 0, 0};
  }
}

__device__ __forceinline__ float both_halves_max(float v) { return fmaxf(v, __shfl_xor(v, 32)); }
__device__ __forceinline__ float both_halves_sum(float v) { return v + __shfl_xor(v, 32); }

// rows d of a transposed result (column = this lane's row of the output tensor) times `m`
template <int DP>
__device__ __forceinline__ void store_cols(float* row, const f32x16 (&acc)[DP / 32], float m, int h, int D) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const int d = 32 * dt + 8 * r4 + 4 * h;
      f32x4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = acc[dt][4 * r4 + j] * m;
      if (d < D) *reinterpret_cast<f32x4*>(row + d) = x;
    }
}
// The same in 16 bits: a row's two lanes hold four values of every eight each; they exchange them, so that each stores 16 bytes.  All lanes of the wave
// come here, `there` says whose row is stored.  `rest`: where given, what the rounding to T took away times FINER, rounded itself.
template <typename T, int DP>
__device__ __forceinline__ void store_cols(T* row, const f32x16 (&acc)[DP / 32], float m, int h, int D, bool there, T* rest = nullptr) {
  typedef T T2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      unsigned w[2][4];                                 // [value, rest][two groups of eight, two words each]
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = acc[dt][8 * i + 2 * j] * m, b = acc[dt][8 * i + 2 * j + 1] * m;
        const T2 v{(T)a, (T)b}, r{(T)((a - (float)v[0]) * FINER<T>), (T)((b - (float)v[1]) * FINER<T>)};
        w[0][j] = __builtin_bit_cast(unsigned, v);
        w[1][j] = __builtin_bit_cast(unsigned, r);
      }
      const int d = 32 * dt + 16 * i + 8 * h;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (k && !rest) break;
        u32x4 x;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const auto both = __builtin_amdgcn_permlane32_swap(w[k][j], w[k][2 + j], false, false);
          x[j] = both[0];
          x[2 + j] = both[1];
        }
        if (there && d < D) *reinterpret_cast<u32x4*>((k ? rest : row) + d) = x;
      }
    }
}

// probabilities (or dS) of 16 rows as the second operand of the next product
template <typename T>
__device__ __forceinline__ typename Frag<T>::V pack8(const f32x16& s, int half) {
  typename Frag<T>::V v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (T)s[8 * half + j];
  return v;
}

// sums += A * dS for 16 rows of a tile.  dS is rounded to the operands' type (f16: under its column's power of two, below), except in the tiles that the mask cuts or the sequence ends in: there it
// goes in as two terms (its rounded value and the rest).  Under the causal mask those tiles hold the rows with few keys, whose dS is largest, and most
// of what dq and dk would be off; all others are many to one of them.
template <typename T, int DP>
__device__ __forceinline__ void add_ds(f32x16 (&acc)[DP / 32], const char* tile, int row0, const f32x16& ds, int half, bool two_terms, int lane) {
  const typename Frag<T>::V hi = pack8<T>(ds, half);
  if (two_terms) {
    typename Frag<T>::V lo;
#pragma unroll
    for (int j = 0; j < 8; ++j) lo[j] = (T)(ds[8 * half + j] - (float)hi[j]);
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = Frag<T>::mma(read_cols<T, DP>(tile, row0, dt, lane), lo, acc[dt]);
  }
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = Frag<T>::mma(read_cols<T, DP>(tile, row0, dt, lane), hi, acc[dt]);
}

// dS on its way into f16 has a power of two for every column (query or key) that keeps what matters of it inside f16's range: gradients of a mean loss over a long
// sequence put dS at 2^-20 and less, where f16 has few bits or none (without it 4 % of dq at do = 1e-4 and 3000 rows), others over 65504.  It is found as
// a softmax finds its reference: the first values of a column that are not zero are taken to 2^8, and where later ones pass 2^14 it falls and the sums with it.  All steps are
// by powers of two, exact.  What is then too small for f16 is 2^-32 of the column's largest.  bf16 has the range of fp32.  (8192 rows, 8 heads, both directions: of 64 447 us without and 454 with it, of 128
// 746 and 755; with a multiplication for every value of dS, instead of in P's exponent or factor, 472 and 771.)
template <typename T> struct Range {
  static constexpr float up = 1.f, shift = 0.f;
  template <int N> __device__ __forceinline__ void fit(f32x16&, f32x16 (&)[N]) {}
  __device__ __forceinline__ float undo() const { return 1.f; }
};
template <> struct Range<_Float16> {
  float up = 1.f, shift = 0.f, limit = 0.f;             // the power of two, its logarithm, what a value may reach under it
  // `ds` comes times `up`
  template <int N> __device__ __forceinline__ void fit(f32x16& ds, f32x16 (&acc)[N]) {
    float t = fabsf(ds[0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) t = fmaxf(t, fabsf(ds[r]));
    if (__any(t > limit)) {
      const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(t), __float_as_uint(t), false, false);
      t = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
      // 2^8 over the power of two in t, no more than 2^30 (dS under 2^-44 reaches no f16 value of dq or dk)
      const int e = t > limit ? min(135 - (int)(__float_as_uint(t) >> 23), 30) : 0;
      const float f = __uint_as_float((unsigned)(127 + e) << 23);
      limit = t > limit ? 16384.f : limit;
      up *= f;
      shift += (float)e;
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] *= f;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= f;
    }
  }
  __device__ __forceinline__ float undo() const { return 1.f / up; }
};

// What a wave of the forward carries from one half tile (32 keys) to the next
template <typename T, int DP>
struct FwdWave {
  typename Frag<T>::V qf[DP / 16];
  f32x16 acc[DP / 32];
  float m, l, mx;            // reference and sum of each column, and the maximum of the next half's scores, in the scores' own units
  float sc;
  static constexpr float LAG = is_f16<T> ? 3.f : 8.f;

  __device__ __forceinline__ void scores(f32x16& s, const char* k, int row0, int lane) const {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) s = Frag<T>::mma(read_rows<T, DP>(k, row0, ks, lane), qf[ks], s);
  }
  // What the exponentials are taken over, in powers of two.  With f16 operands it lies 7 under the reference, so that probabilities of 2^-21 of the largest still have all
  // their bits there (as it is, of 2^-14: where a first key takes nearly everything, outputs were off by 2.6 half steps at 2^-19).
  __device__ __forceinline__ float base() const {
    const float b = m > -INFINITY ? m * sc : 0.f;       // keys of minus infinity so far: their exponentials are zeros
    return is_f16<T> ? b - 7.f : b;
  }
  __device__ __forceinline__ void maximum(const f32x16& s) {
    float a = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) a = fmaxf(a, s[r]);
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(a), false, false);
    mx = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
  }
  // Half a tile: the exponentials and sums of `cur` (values from row `vrow` of `v` on) together with the scores `next` of the half behind it (keys from row
  // `krow` of `k` on), so that one's products run under the other's exponentials.
  __device__ __forceinline__ void half(f32x16& cur, f32x16& next, const char* k, int krow, const char* v, int vrow, int lane) {
    // The reference moves only where a column's maximum has outgrown it by LAG powers of two (and in the first half): most halves leave the sums as they are.  The
    // exponentials stay under 2^8, in f16 under 2^10.  (There has to be room: a base is rounded, and that is worth up to 2^4 at scores of 1e8.)
    if (__any(!((mx - m) * sc <= LAG))) {
      const float mn = fmaxf(m, mx), keep = m > -INFINITY ? exp2_fast((m - mn) * sc) : 0.f;
      m = mn;
      l *= keep;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[dt][r] *= keep;
    }
    const float ms = base();
    scores(next, k, krow, lane);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int r = 8 * b; r < 8 * b + 8; ++r) {
        cur[r] = exp2_fast(__builtin_fmaf(cur[r], sc, -ms));
        l += cur[r];
      }
      const typename Frag<T>::V pf = pack8<T>(cur, b);
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = Frag<T>::mma(read_cols<T, DP>(v, vrow + 16 * b, dt, lane), pf, acc[dt]);
    }
    maximum(next);
  }
};

// Forward.  A workgroup: 128 queries of one head, four waves, over key tiles of 64.  Two workgroups share a CU (230 registers, 80 KB of LDS at DP = 128), so
// that one computes while the other waits at its barrier.  Bound by the matrix pipe and the exponentials together, and by power: one causal prompt of 16384, 8 heads on
// 2, 128 wide, bf16: 0.55 ms = 0.99 PFLOP/s with the matrix pipe 51 % busy at a clock that has fallen to 1.8 GHz (an 8192^3 library product: 1.24).  Tiles through
// registers and without asynchronous loads took 1.46 ms, whole tiles instead of halves the same as this on long prompts and 133 us instead of 117 on
// packed ones (16 heads on 4, 8192 rows in 7 sequences).
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void packed_attn_fwd_kernel(const PackedAttnArgs p) {
  __shared__ __attribute__((aligned(16))) char kt[3][BN * DP * 2], vt[2][BN * DP * 2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int split = blockIdx.x % p.splits, head = blockIdx.x / p.splits % p.Hq, tile = blockIdx.x / p.splits / p.Hq;
  const TileAt f = find_tile(p.cu, p.nseq, p.T, tile, p.tiles, lane, p.causal ? BY_WEIGHT : IN_ORDER);
  if (f.idle) {
    if (p.fill_tail && split == 0) zero_tail((T*)p.out, p.o_t, p.o_h, head, p.D, f, p.T, tid);
    return;
  }
  const int hk = head / (p.Hq / p.Hkv);
  const T* k = (const T*)p.k + f.start * p.k_t + hk * p.k_h;
  const T* v = (const T*)p.v + f.start * p.v_t + hk * p.v_h;
  const int row = f.row0 + wave * 32 + (lane & 31);
  const bool there = row < f.len;
  const T* qrow = (const T*)p.q + (f.start + (there ? row : 0)) * p.q_t + head * p.q_h;
  int kend = p.causal ? min(f.len, f.row0 + BM) : f.len, k0 = 0;
  if (p.splits > 1) {                                   // this part of the key tiles
    const int n = (kend + BN - 1) / BN;
    k0 = n * split / p.splits * BN;
    kend = min(kend, n * (split + 1) / p.splits * BN);
    if (k0 >= kend) {
      if (there && h == 0) p.stats[((long long)split * p.Hq + head) * p.T + f.start + row] = make_float2(-INFINITY, 0.f);
      return;
    }
  }
  // keys that all of this wave's queries see, in whole tiles, and keys that it has to look at
  const bool empty = f.row0 + wave * 32 >= f.len;       // a wave behind the sequence's end only loads
  const int open = empty ? 0 : min(kend, p.causal ? min(f.len, f.row0 + wave * 32 + 1) / BN * BN : f.len / BN * BN);
  const int wend = empty ? 0 : p.causal ? min(f.len, f.row0 + wave * 32 + 32) : f.len;
  Tile<T, DP> ks_, vs_;
  ks_.init(p.k_t, f.len - k0, p.D, tid);
  vs_.init(p.v_t, f.len - k0, p.D, tid);
  ks_.load(k + (long long)k0 * p.k_t, f.len - k0, lds_offset(kt[0]), p.D, tid);
  vs_.load(v + (long long)k0 * p.v_t, f.len - k0, lds_offset(vt[0]), p.D, tid);
  if (k0 + BN < kend) ks_.load(k + (long long)(k0 + BN) * p.k_t, f.len - k0 - BN, lds_offset(kt[1]), p.D, tid);
  FwdWave<T, DP> w;
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) w.qf[ks] = load_frag<T>(qrow, ks, h, p.D, there);
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) w.acc[dt][r] = 0.f;
  w.m = -INFINITY;
  w.l = 0.f;
  w.sc = p.scale * LOG2E;
  f32x16 s0, s1;
  tile_barrier();
  w.scores(s0, kt[0], 0, lane);
  w.maximum(s0);
  // Loads of the tiles behind: the keys run one tile ahead of the values, since a tile's last scores are those of the next one's first half
  auto fetch = [&](char* keys, char* values) {
    if (k0 + 2 * BN < kend) ks_.load(k + (long long)(k0 + 2 * BN) * p.k_t, f.len - k0 - 2 * BN, lds_offset(keys), p.D, tid);
    if (k0 + BN < kend) vs_.load(v + (long long)(k0 + BN) * p.v_t, f.len - k0 - BN, lds_offset(values), p.D, tid);
  };
  const int whole = open > k0 ? (open - k0) / BN : 0;    // tiles without a mask
  auto step = [&](int, auto place) {
    constexpr int a = decltype(place)::value % 3, b = (a + 1) % 3, c = (a + 2) % 3, u = decltype(place)::value & 1;
    fetch(kt[c], vt[u ^ 1]);
    w.half(s0, s1, kt[a], 32, vt[u], 0, lane);
    w.half(s1, s0, kt[b], 0, vt[u], 32, lane);          // (behind the last tile: scores of nothing, which nobody reads)
    k0 += BN;
    tile_barrier();
  };
  turns<6>(0, whole, step);
  // key tiles of this, the next and the next but one; parity of the value tile
  int ka = whole % 3, kb = (whole + 1) % 3, kc = (whole + 2) % 3, vb = whole & 1;
  while (k0 < kend) {                                   // tiles that end or are cut by the mask
    fetch(kt[kc], vt[vb ^ 1]);
    if (k0 < wend) {
      const int last = (p.causal ? min(row, f.len - 1) : f.len - 1) - k0 - 4 * h;    // the last key this column sees
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r >> 2) + (r & 3) > last) s0[r] = -INFINITY;
      w.maximum(s0);
      w.half(s0, s1, kt[ka], 32, vt[vb], 0, lane);
      if (k0 + 32 < wend) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 + 8 * (r >> 2) + (r & 3) > last) s1[r] = -INFINITY;
        w.maximum(s1);
        w.half(s1, s0, kt[kb], 0, vt[vb], 32, lane);
      }
    }
    const int t = ka;
    ka = kb; kb = kc; kc = t;
    vb ^= 1;
    k0 += BN;
    tile_barrier();
  }
  const float l = both_halves_sum(w.l);
  if (p.splits > 1) {
    const long long at = f.start + row;
    if (there) store_cols<DP>(p.partial + ((split * p.T + at) * p.Hq + head) * p.D, w.acc, 1.0f, h, p.D);
    if (there && h == 0) p.stats[((long long)split * p.Hq + head) * p.T + at] = make_float2(w.m > -INFINITY ? w.base() : -INFINITY, l);
    return;
  }
  store_cols<T, DP>((T*)p.out + (f.start + row) * p.o_t + head * p.o_h, w.acc, 1.0f / l, h, p.D, there,
                    p.rest ? (T*)p.rest + ((f.start + row) * p.Hq + head) * p.D : nullptr);
  if (there && p.sums && h == 0) p.sums[(long long)head * p.T + f.start + row] = make_float2(w.base(), log2f(l));
}

// dq, and delta = rowsum(do * o) for the other kernel.  As the forward, with dP beside S; three products a tile and no running maximum.  178 us for the
// packed sequences above: 0.81 PFLOP/s.
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void packed_attn_dq_kernel(const PackedAttnArgs p) {
  __shared__ __attribute__((aligned(16))) char kt[2][BN * DP * 2], vt[2][BN * DP * 2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int split = blockIdx.x % p.splits, head = blockIdx.x / p.splits % p.Hq, tile = blockIdx.x / p.splits / p.Hq;
  const TileAt f = find_tile(p.cu, p.nseq, p.T, tile, p.tiles, lane, p.causal ? BY_WEIGHT : IN_ORDER);
  if (f.idle) {
    if (split == 0) zero_tail((T*)p.dq, p.dq_t, p.dq_h, head, p.D, f, p.T, tid);
    return;
  }
  const int hk = head / (p.Hq / p.Hkv);
  const T* k = (const T*)p.k + f.start * p.k_t + hk * p.k_h;
  const T* v = (const T*)p.v + f.start * p.v_t + hk * p.v_h;
  const int row = f.row0 + wave * 32 + (lane & 31);
  const bool there = row < f.len;
  const long long at = f.start + (there ? row : 0);
  const T* qrow = (const T*)p.q + at * p.q_t + head * p.q_h;
  const T* grow = (const T*)p.dout + at * p.do_t + head * p.do_h;
  const T* orow = (const T*)p.o + at * p.o_t + head * p.o_h;
  const T* rrow = (const T*)p.rest + (at * p.Hq + head) * p.D;
  typename Frag<T>::V qf[DP / 16], gf[DP / 16];
  float delta = 0.f;
  {
    typename Frag<T>::V of[DP / 16], rf[DP / 16];
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      gf[ks] = load_frag<T>(grow, ks, h, p.D, there);
      of[ks] = load_frag<T>(orow, ks, h, p.D, there);
      rf[ks] = load_frag<T>(rrow, ks, h, p.D, there && p.rest);
    }
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) qf[ks] = load_frag<T>(qrow, ks, h, p.D, there);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = __builtin_fmaf((float)gf[ks][j], __builtin_fmaf((float)rf[ks][j], 1.f / FINER<T>, (float)of[ks][j]), delta);
  }
  delta = both_halves_sum(delta);
  const float2 sum = there ? p.sums[(long long)head * p.T + at] : make_float2(0.f, 0.f);
  if (there && h == 0 && split == 0) p.delta[(long long)head * p.T + at] = delta;

  f32x16 acc[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;
  Range<T> range;
  const float sc = p.scale * LOG2E;
  const int all = p.causal ? min(f.len, f.row0 + BM) : f.len, tiles = (all + BN - 1) / BN;
  const int kbeg = tiles * split / p.splits * BN, kend = min(all, tiles * (split + 1) / p.splits * BN);      // this part of the key tiles
  const int wend = f.row0 + wave * 32 >= f.len ? 0 : p.causal ? min(f.len, f.row0 + wave * 32 + 32) : f.len;     // keys this wave has to look at
  Tile<T, DP> ks_, vs_;
  if (kbeg < kend) {
    ks_.init(p.k_t, f.len - kbeg, p.D, tid);
    vs_.init(p.v_t, f.len - kbeg, p.D, tid);
    ks_.load(k + (long long)kbeg * p.k_t, f.len - kbeg, lds_offset(kt[0]), p.D, tid);
    vs_.load(v + (long long)kbeg * p.v_t, f.len - kbeg, lds_offset(vt[0]), p.D, tid);
  }
  auto step = [&](const int i, auto place) {
    constexpr int buf = decltype(place)::value;
    const int k0 = kbeg + i * BN;
    tile_barrier();
    if (k0 + BN < kend) {
      ks_.load(k + (long long)(k0 + BN) * p.k_t, f.len - k0 - BN, lds_offset(kt[buf ^ 1]), p.D, tid);
      vs_.load(v + (long long)(k0 + BN) * p.v_t, f.len - k0 - BN, lds_offset(vt[buf ^ 1]), p.D, tid);
    }
    if (k0 >= wend) return;
    const int last = (there ? (p.causal ? row : f.len - 1) : -1) - k0 - 4 * h;
    const bool edge = k0 + BN > f.len || f.row0 + wave * 32 + 32 > f.len || (p.causal && k0 + BN - 1 > f.row0 + wave * 32);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if (n && k0 + 32 >= wend) break;
      f32x16 s, g;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = g[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        s = Frag<T>::mma(read_rows<T, DP>(kt[buf], 32 * n, ks, lane), qf[ks], s);
        g = Frag<T>::mma(read_rows<T, DP>(vt[buf], 32 * n, ks, lane), gf[ks], g);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = exp2_fast(__builtin_fmaf(s[r], sc, -sum.x) - (sum.y - range.shift)) * (g[r] - delta);
      if (edge) {
        stay_a_branch();
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * n + 8 * (r >> 2) + (r & 3) > last) s[r] = 0.f;
      }
      range.fit(s, acc);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        add_ds<T, DP>(acc, kt[buf], 32 * n + 16 * b, s, b, edge, lane);
      }
    }
  };
  turns<2>(0, (kend - kbeg + BN - 1) / BN, step);
  if (p.splits > 1) {
    if (there) store_cols<DP>(p.partial + ((split * p.T + at) * p.Hq + head) * p.D, acc, p.scale * range.undo(), h, p.D);
    return;
  }
  store_cols<T, DP>((T*)p.dq + at * p.dq_t + head * p.dq_h, acc, p.scale * range.undo(), h, p.D, there);
}

// P on its way into f16 comes 2^14 times as large, which the exponent has for nothing: it keeps all its bits from 2^-28 on (as it is, from 2^-14: dv of keys that many queries see a little was
// off by 280 half steps where P is about 1e-7).  bf16 needs that only where f16 hands it over.
constexpr float LIFT = 14.f, LIFTED = 0x1p14f;

// dk and dv of 128 keys: over the query heads that share them and the query tiles that see them.  A wave's 32 keys and values and both sums stay in its
// registers, which heads of up to 64 columns leave room for two waves a SIMD for.  32 f16 images of 197 rows, 12 heads of 64: 29 us, bound by
// latency (four tiles a workgroup).
template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void packed_attn_dkv_kernel(const PackedAttnArgs p) {
  __shared__ __attribute__((aligned(16))) char qt[2][BN * DP * 2], gt[2][BN * DP * 2];
  __shared__ __attribute__((aligned(16))) float rs[2][BN], ls[2][BN], ds[2][BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int part = blockIdx.x % p.parts, hk = blockIdx.x / p.parts % p.Hkv, tile = blockIdx.x / p.parts / p.Hkv, G = p.Hq / p.Hkv;
  const TileAt f = find_tile(p.cu, p.nseq, p.T, tile, p.tiles, lane, p.causal ? BY_WEIGHT_FROM_END : IN_ORDER);
  if (f.idle) {
    if (part) return;
    zero_tail((T*)p.dk, p.dk_t, p.dk_h, hk, p.D, f, p.T, tid);
    zero_tail((T*)p.dv, p.dv_t, p.dv_h, hk, p.D, f, p.T, tid);
    return;
  }
  const int row = f.row0 + wave * 32 + (lane & 31);     // this lane's key
  const bool there = row < f.len;
  const long long at = f.start + (there ? row : 0);
  const T* krow = (const T*)p.k + at * p.k_t + hk * p.k_h;
  const T* vrow = (const T*)p.v + at * p.v_t + hk * p.v_h;
  typename Frag<T>::V kf[DP / 16], vf[DP / 16];
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    kf[ks] = load_frag<T>(krow, ks, h, p.D, there);
    vf[ks] = load_frag<T>(vrow, ks, h, p.D, there);
  }
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[dt][r] = dv[dt][r] = 0.f;
  Range<T> range;
  const float sc = p.scale * LOG2E;
  const int qbeg = p.causal ? f.row0 : 0;               // a multiple of BN
  const int per = (f.len - qbeg + BN - 1) / BN, total = per * G;
  const int i0 = (int)((long long)total * part / p.parts), i1 = (int)((long long)total * (part + 1) / p.parts);   // this part of the heads' query tiles
  Tile<T, DP> qs, gs;
  qs.init(p.q_t, f.len - qbeg, p.D, tid);
  gs.init(p.do_t, f.len - qbeg, p.D, tid);
  float2 lv_ = make_float2(0.f, 0.f);                   // the next tile's statistics, one row per thread of the first wave
  float dl_ = 0.f;
  int head = hk * G + i0 / per, q0 = qbeg + i0 % per * BN;      // of the tile that is fetched next
  auto fetch = [&](int buf) {
    qs.load((const T*)p.q + (f.start + q0) * p.q_t + head * p.q_h, f.len - q0, lds_offset(qt[buf]), p.D, tid);
    gs.load((const T*)p.dout + (f.start + q0) * p.do_t + head * p.do_h, f.len - q0, lds_offset(gt[buf]), p.D, tid);
    if (tid < BN) {
      const long long a = (long long)head * p.T + f.start + min(q0 + tid, f.len - 1);
      lv_ = p.sums[a];
      dl_ = p.delta[a];
    }
  };
  if (i0 < i1) fetch(0);
  auto step = [&](const int i, auto place) {
    constexpr int buf = decltype(place)::value;
    const int at0 = q0;                                 // first query of this tile
    if (tid < BN) {
      rs[buf][tid] = lv_.x;
      ls[buf][tid] = is_f16<T> ? lv_.y - LIFT : lv_.y;
      ds[buf][tid] = dl_;
    }
    tile_barrier();
    q0 += BN;
    if (q0 >= f.len) {
      q0 = qbeg;
      ++head;
    }
    if (i + 1 < i1) fetch(buf ^ 1);
    // queries that see this lane's key: from `first` on, `seen` of them
    const int first = (p.causal ? row : 0) - at0 - 4 * h, seen = f.len - (p.causal ? row : 0);
    const bool edge = at0 + BN > f.len || (p.causal && at0 < f.row0 + wave * 32 + 31);
    if (f.row0 + wave * 32 >= f.len) return;            // a wave behind the sequence's end only loads
#pragma unroll
    for (int n = 0; n < BN / 32; ++n) {
      // 32 queries behind the end, or all before this wave's keys
      if (edge && (at0 + 32 * n >= f.len || (p.causal && at0 + 32 * n + 32 <= f.row0 + wave * 32))) continue;
      f32x16 s, g;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = g[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        s = Frag<T>::mma(read_rows<T, DP>(qt[buf], 32 * n, ks, lane), kf[ks], s);
        g = Frag<T>::mma(read_rows<T, DP>(gt[buf], 32 * n, ks, lane), vf[ks], g);
      }
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const f32x4 ref = *reinterpret_cast<const f32x4*>(&rs[buf][32 * n + 8 * r4 + 4 * h]), lv = *reinterpret_cast<const f32x4*>(&ls[buf][32 * n + 8 * r4 + 4 * h]);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[4 * r4 + j] = exp2_fast(__builtin_fmaf(s[4 * r4 + j], sc, -ref[j]) - lv[j]);
      }
      if (edge) {
        stay_a_branch();
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if ((unsigned)(32 * n + 8 * (r >> 2) + (r & 3) - first) >= (unsigned)seen) s[r] = 0.f;
      }
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const f32x4 dl = *reinterpret_cast<const f32x4*>(&ds[buf][32 * n + 8 * r4 + 4 * h]);
#pragma unroll
        for (int j = 0; j < 4; ++j) g[4 * r4 + j] = s[4 * r4 + j] * (g[4 * r4 + j] - dl[j]) * range.up;
      }
      range.fit(g, dk);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const typename Frag<T>::V pf = pack8<T>(s, b);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) dv[dt] = Frag<T>::mma(read_cols<T, DP>(gt[buf], 32 * n + 16 * b, dt, lane), pf, dv[dt]);
        add_ds<T, DP>(dk, qt[buf], 32 * n + 16 * b, g, b, edge, lane);
      }
    }
  };
  turns<2>(i0, i1, step);
  const float unit_v = is_f16<T> ? 1.f / LIFTED : 1.f, unit_k = p.scale * unit_v * range.undo();
  if (p.parts > 1) {
    float* to = p.partial + ((part * p.T + at) * p.Hkv + hk) * 2 * p.D;
    if (there) store_cols<DP>(to, dk, unit_k, h, p.D);
    if (there) store_cols<DP>(to + p.D, dv, unit_v, h, p.D);
  } else {
    store_cols<T, DP>((T*)p.dk + at * p.dk_t + hk * p.dk_h, dk, unit_k, h, p.D, there);
    store_cols<T, DP>((T*)p.dv + at * p.dv_t + hk * p.dv_h, dv, unit_v, h, p.D, there);
  }
}

// P in 16 bits on its way from one wave to another, finer than the operands' type, so that dS is nearly rounded once in effect.  It comes 2^14 times as large (LIFT), so that what
// is small has all its bits too: for bf16 operands f16 holds 11 of them from P = 2^-28 on (and under it steps of 2^-38); for f16 ones P, which is never negative, takes five bits of
// exponent and eleven of mantissa: 12 bits from P = 2^-30 on, steps of 2^-41 under it.  (As f16 without the factor, the dk of keys that few queries see lost its bits: 26 half steps
// of bf16 where P is 1e-7.)  bf16's dk is summed under the factor: over 2^113 it becomes infinite.  The clamp is for P that does not belong to its sum: its bits would reach into the neighbour's.
template <typename T> struct Handed;
template <> struct Handed<__bf16> {
  typedef Frag<_Float16>::V V;
  static constexpr float LEFT = LIFTED;                // get() returns this times P (f16 operands: times `up`)
  static __device__ __forceinline__ V pack(const f32x16& s, int half) { return pack8<_Float16>(s, half); }
  static __device__ __forceinline__ float get(const V& v, int j, float) { return (float)v[j]; }
};
template <> struct Handed<_Float16> {
  typedef unsigned V __attribute__((ext_vector_type(4)));
  static constexpr float LEFT = 1.0f;
  static __device__ __forceinline__ unsigned bits(float p) { return __float_as_uint(fminf(p, 0x1.ffep14f) * 0x1p-110f) + 0x800u; }      // exponents 0 .. 31, twelve bits to go
  static __device__ __forceinline__ V pack(const f32x16& s, int half) {
    V v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = bits(s[8 * half + 2 * j]) >> 12 | (bits(s[8 * half + 2 * j + 1]) & ~0xfffu) << 4;
    return v;
  }
  static __device__ __forceinline__ float get(const V& v, int j, float up) {     // up is at most 2^30
    return __uint_as_float(j & 1 ? v[j / 2] >> 4 & ~0xfffu : (v[j / 2] & 0xffffu) << 12) * (0x1p96f * up);
  }
};

// The same for heads wider than 64, where one wave cannot hold both sums, its keys' and values' fragments and the scores in half a SIMD's registers, and a
// wave alone on its SIMD waits out every exponential: eight waves, two on each SIMD, share the four products of 128 keys.  The first of a pair forms S and P
// and sums dv; it hands P over through LDS, and the second forms dP and dS and sums dk one tile behind, so that the only wait is the barrier that there is for the
// tiles.  Three tiles are held.  16 query heads on 4, 128 wide, 8192 rows, causal: 435 us with one wave per SIMD, 310 us with pairs that both form S, 277 us so, and
// 257 us (0.74 PFLOP/s) with constant places of its tiles.
template <typename T, int DP>
__global__ __launch_bounds__(512, 2) void packed_attn_dkv_pair_kernel(const PackedAttnArgs p) {
  __shared__ __attribute__((aligned(16))) char qt[3][BN * DP * 2], gt[3][BN * DP * 2];
  typedef Handed<T> Pass;
  __shared__ typename Pass::V pt[2][4][4][64];          // [tile's parity][pair][half of the tile x half of its rows][lane]
  __shared__ __attribute__((aligned(16))) float rs[3][BN], ls[3][BN], ds[3][BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6) & 3, h = lane >> 5;
  const bool values = __builtin_amdgcn_readfirstlane(tid >> 8);          // this wave forms P and dv, its partner dk
  const int part = blockIdx.x % p.parts, hk = blockIdx.x / p.parts % p.Hkv, tile = blockIdx.x / p.parts / p.Hkv, G = p.Hq / p.Hkv;
  const TileAt f = find_tile(p.cu, p.nseq, p.T, tile, p.tiles, lane, p.causal ? BY_WEIGHT_FROM_END : IN_ORDER);
  if (f.idle) {
    if (part) return;
    if (values) zero_tail((T*)p.dv, p.dv_t, p.dv_h, hk, p.D, f, p.T, tid & 255);
    else zero_tail((T*)p.dk, p.dk_t, p.dk_h, hk, p.D, f, p.T, tid);
    return;
  }
  const int row = f.row0 + wave * 32 + (lane & 31);     // this lane's key
  const bool there = row < f.len;
  const long long at = f.start + (there ? row : 0);
  const T* krow = values ? (const T*)p.k + at * p.k_t + hk * p.k_h : (const T*)p.v + at * p.v_t + hk * p.v_h;
  typename Frag<T>::V kf[DP / 16];                      // the keys for S, or the values for dP
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) kf[ks] = load_frag<T>(krow, ks, h, p.D, there);
  f32x16 acc[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;
  Range<T> range;
  const float sc = p.scale * LOG2E;
  const int qbeg = p.causal ? f.row0 : 0;               // a multiple of BN
  const int per = (f.len - qbeg + BN - 1) / BN, total = per * G;
  const int i0 = (int)((long long)total * part / p.parts), i1 = (int)((long long)total * (part + 1) / p.parts);   // this part of the heads' query tiles
  Tile<T, DP> ts;                                       // four waves load the queries, four the output's gradients
  ts.init(values ? p.do_t : p.q_t, f.len - qbeg, p.D, tid & 255);
  const T* base = values ? (const T*)p.dout + f.start * p.do_t : (const T*)p.q + f.start * p.q_t;
  const long long st = values ? p.do_t : p.q_t, sh = values ? p.do_h : p.q_h;
  float2 lv_ = make_float2(0.f, 0.f);                   // the next tile's statistics, one row per thread of the first wave
  float dl_ = 0.f;
  int head = hk * G + i0 / per, q0 = qbeg + i0 % per * BN;      // of the tile that is fetched next
  auto fetch = [&](int slot) {
    ts.load(base + q0 * st + head * sh, f.len - q0, values ? lds_offset(gt[slot]) : lds_offset(qt[slot]), p.D, tid & 255);
    if (tid < BN) {
      const long long a = (long long)head * p.T + f.start + min(q0 + tid, f.len - 1);
      lv_ = p.sums[a];
      dl_ = p.delta[a];
    }
  };
  if (i0 < i1) fetch(0);
  int here = q0;                                        // first query of this one
  // The barrier of tile i, and behind it the loads of the next one.  (Slots turn by 3, P's by 2.)
  auto begin = [&](int i, auto place) {
    constexpr int cur = decltype(place)::value % 3, next = (cur + 1) % 3;
    if (tid < BN && i < i1) {
      rs[cur][tid] = lv_.x;
      ls[cur][tid] = lv_.y - LIFT;                      // P times 2^14
      ds[cur][tid] = dl_;
    }
    tile_barrier();
    here = q0;
    q0 += BN;
    if (q0 >= f.len) {
      q0 = qbeg;
      ++head;
    }
    if (i + 1 < i1) fetch(next);
  };
  // (each kind of wave has its loop, so that its sums stay where they are; both pass the barriers of i0 .. i1)
  if (i0 < i1 && values) {
    auto step = [&](const int i, auto place) {
      constexpr int cur = decltype(place)::value % 3, turn = decltype(place)::value & 1;
      begin(i, place);
      // queries that see this lane's key: from `first` on, `seen` of them
      const int first = (p.causal ? row : 0) - here - 4 * h, seen = f.len - (p.causal ? row : 0);
      const bool edge = here + BN > f.len || (p.causal && here < f.row0 + wave * 32 + 31);
#pragma unroll
      for (int n = 0; n < BN / 32; ++n) {
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) s = Frag<T>::mma(read_rows<T, DP>(qt[cur], 32 * n, ks, lane), kf[ks], s);
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f32x4 ref = *reinterpret_cast<const f32x4*>(&rs[cur][32 * n + 8 * r4 + 4 * h]), lv = *reinterpret_cast<const f32x4*>(&ls[cur][32 * n + 8 * r4 + 4 * h]);
#pragma unroll
          for (int j = 0; j < 4; ++j) s[4 * r4 + j] = exp2_fast(__builtin_fmaf(s[4 * r4 + j], sc, -ref[j]) - lv[j]);
        }
        if (edge) {
          stay_a_branch();
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if ((unsigned)(32 * n + 8 * (r >> 2) + (r & 3) - first) >= (unsigned)seen) s[r] = 0.f;
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          pt[turn][wave][2 * n + b][lane] = Pass::pack(s, b);
          const typename Frag<T>::V pf = pack8<T>(s, b);
#pragma unroll
          for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = Frag<T>::mma(read_cols<T, DP>(gt[cur], 32 * n + 16 * b, dt, lane), pf, acc[dt]);
        }
      }
    };
    turns<6>(i0, i1, step);
    begin(i1, std::integral_constant<int, 0>());          // (no tile's: its barrier only)
  } else if (i0 < i1) {
    begin(i0, std::integral_constant<int, 0>());
    auto step = [&](const int i, auto place) {
      constexpr int prev = decltype(place)::value % 3, turn = decltype(place)::value & 1;
      const int before = here;
      const bool edge = before + BN > f.len || (p.causal && before < f.row0 + wave * 32 + 31);
      begin(i + 1, std::integral_constant<int, (decltype(place)::value + 1) % 6>());
#pragma unroll
      for (int n = 0; n < BN / 32; ++n) {
        f32x16 g;
#pragma unroll
        for (int r = 0; r < 16; ++r) g[r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) g = Frag<T>::mma(read_rows<T, DP>(gt[prev], 32 * n, ks, lane), kf[ks], g);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const typename Pass::V pr = pt[turn][wave][2 * n + b][lane];
#pragma unroll
          for (int r4 = 2 * b; r4 < 2 * b + 2; ++r4) {
            const f32x4 dl = *reinterpret_cast<const f32x4*>(&ds[prev][32 * n + 8 * r4 + 4 * h]);
#pragma unroll
            for (int j = 0; j < 4; ++j) g[4 * r4 + j] = Pass::get(pr, 4 * (r4 - 2 * b) + j, range.up) * (g[4 * r4 + j] - dl[j]);
          }
        }
        range.fit(g, acc);
#pragma unroll
        for (int b = 0; b < 2; ++b) add_ds<T, DP>(acc, qt[prev], 32 * n + 16 * b, g, b, edge, lane);
      }
    };
    turns<6>(i0, i1, step);
  }
  const float unit = values ? 1.f / LIFTED : p.scale / Pass::LEFT * range.undo();
  if (p.parts > 1) {
    if (there) store_cols<DP>(p.partial + ((part * p.T + at) * p.Hkv + hk) * 2 * p.D + (values ? p.D : 0), acc, unit, h, p.D);
  } else {
    store_cols<T, DP>(values ? (T*)p.dv + at * p.dv_t + hk * p.dv_h : (T*)p.dk + at * p.dk_t + hk * p.dk_h, acc, unit, h, p.D, there);
  }
}

// dk and dv from the parts' sums, in the parts' order; 8 values per thread
template <typename T>
__global__ __launch_bounds__(256) void packed_attn_join_kernel(const PackedAttnArgs p) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 8;
  const long long row = i / (2 * p.D * p.Hkv), begin = p.cu[0] < 0 ? 0 : p.cu[0], end = min(p.T, (long long)p.cu[p.nseq]);
  if (row >= end || row < begin) return;                // rows of no sequence are zero already
  const int c = (int)(i % (2 * p.D)), hk = (int)(i / (2 * p.D) % p.Hkv);
  const float* from = p.partial + i;
  const long long step = p.T * p.Hkv * 2 * p.D;
  float s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] = from[j];
  for (int k = 1; k < p.parts; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] += from[k * step + j];
  typename Frag<T>::V x;
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (T)s[j];
  T* to = c < p.D ? (T*)p.dk + row * p.dk_t + hk * p.dk_h + c : (T*)p.dv + row * p.dv_t + hk * p.dv_h + c - p.D;
  *reinterpret_cast<typename Frag<T>::V*>(to) = x;
}

// dq from the parts' sums, in the parts' order
template <typename T>
__global__ __launch_bounds__(256) void packed_attn_join_dq_kernel(const PackedAttnArgs p) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 8, wide = (long long)p.Hq * p.D;
  const long long row = i / wide, begin = p.cu[0] < 0 ? 0 : p.cu[0], end = min(p.T, (long long)p.cu[p.nseq]);
  if (row >= end || row < begin) return;                // rows of no sequence are zero already
  float s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] = p.partial[i + j];
  for (int k = 1; k < p.splits; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] += p.partial[k * p.T * wide + i + j];
  typename Frag<T>::V x;
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (T)s[j];
  *reinterpret_cast<typename Frag<T>::V*>((T*)p.dq + i) = x;
}
// the forward from its parts: each part's sums are taken to the largest reference
template <typename T>
__global__ __launch_bounds__(256) void packed_attn_join_fwd_kernel(const PackedAttnArgs p) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 8, wide = (long long)p.Hq * p.D;
  const long long row = i / wide, begin = p.cu[0] < 0 ? 0 : p.cu[0], end = min(p.T, (long long)p.cu[p.nseq]);
  if (row >= end || row < begin) return;
  const int head = (int)(i % wide / p.D), d = (int)(i % p.D);
  float m = -INFINITY;
  for (int k = 0; k < p.splits; ++k) m = fmaxf(m, p.stats[((long long)k * p.Hq + head) * p.T + row].x);
  float s[8], l = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] = 0.f;
  for (int k = 0; k < p.splits; ++k) {
    const float2 st = p.stats[((long long)k * p.Hq + head) * p.T + row];
    if (st.y == 0.f) continue;                          // a part that saw no key
    const float w = exp2_fast(st.x - m);
    l = __builtin_fmaf(st.y, w, l);
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = __builtin_fmaf(p.partial[k * p.T * wide + i + j], w, s[j]);
  }
  const float inv = 1.0f / l;
  typename Frag<T>::V x, r;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float o = s[j] * inv;
    x[j] = (T)o;
    r[j] = (T)((o - (float)x[j]) * FINER<T>);
  }
  *reinterpret_cast<typename Frag<T>::V*>((T*)p.out + row * p.o_t + head * p.o_h + d) = x;
  if (p.rest) *reinterpret_cast<typename Frag<T>::V*>((T*)p.rest + i) = r;
  if (p.sums && d == 0) p.sums[(long long)head * p.T + row] = make_float2(m > -INFINITY ? m : 0.f, log2f(l));
}

template <typename T, int DP>
hipError_t launch_forward(const PackedAttnArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((packed_attn_fwd_kernel<T, DP>), dim3((unsigned)a.tiles * a.Hq * a.splits), dim3(256), 0, s, a);
  if (a.splits > 1) hipLaunchKernelGGL((packed_attn_join_fwd_kernel<T>), dim3((unsigned)((a.T * a.Hq * a.D / 8 + 255) / 256)), dim3(256), 0, s, a);
  return hipGetLastError();
}
template <typename T, int DP>
hipError_t launch_backward(const PackedAttnArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((packed_attn_dq_kernel<T, DP>), dim3((unsigned)a.tiles * a.Hq * a.splits), dim3(256), 0, s, a);
  if (a.splits > 1) hipLaunchKernelGGL((packed_attn_join_dq_kernel<T>), dim3((unsigned)((a.T * a.Hq * a.D / 8 + 255) / 256)), dim3(256), 0, s, a);
  const dim3 g((unsigned)a.tiles * a.Hkv * a.parts);
  if constexpr (DP > 64) hipLaunchKernelGGL((packed_attn_dkv_pair_kernel<T, DP>), g, dim3(512), 0, s, a);
  else hipLaunchKernelGGL((packed_attn_dkv_kernel<T, DP>), g, dim3(256), 0, s, a);
  if (a.parts > 1)
    hipLaunchKernelGGL((packed_attn_join_kernel<T>), dim3((unsigned)((a.T * a.Hkv * 2 * a.D / 8 + 255) / 256)), dim3(256), 0, s, a);
  return hipGetLastError();
}
template <typename T>
hipError_t launch(const PackedAttnArgs& a, bool backward, hipStream_t s) {
  // heads are padded with zeros to the next multiple of 32 columns (a whole row tile of the products over d)
  switch ((a.D + 31) / 32) {
    case 1: return backward ? launch_backward<T, 32>(a, s) : launch_forward<T, 32>(a, s);
    case 2: return backward ? launch_backward<T, 64>(a, s) : launch_forward<T, 64>(a, s);
    case 3: return backward ? launch_backward<T, 96>(a, s) : launch_forward<T, 96>(a, s);
    default: return backward ? launch_backward<T, 128>(a, s) : launch_forward<T, 128>(a, s);
  }
}

// Into how many parts a tile's other axis is dealt: the keys of a query tile (forward, dq: `heads` query heads, shared = 1) and the queries of a key tile (dk / dv:
// `heads` key / value heads, each `shared` times the queries).  A launch of few tiles leaves CUs idle and ends with its longest workgroup; the
// parts' fp32 sums cost a write and a read.  Wanted are `want` workgroups and eight tiles a part where all rows are one sequence (their
// lengths are on the device); many short sequences are left whole.  Forward + backward in us, whole and in parts: causal sequences of 1829 / 379 / 312,
// 8 heads on 2 of 64: 285 and 110; one of 6000, one head of 128: 511 and 142 (forward 107 and 41); one of 2000, 4 heads on 1 of 128: 363 and 130; 600 / 500, 4 heads
// of 64: 61 and 52.  (16 heads on 4, 128 wide, 8192 rows: dk and dv in 1 part 1.41 ms, in 2 0.49 ms with their first form; 4 parts are within 1 % of 2.)
int parts_of(long long T, int nseq, int heads, int shared, int want) {
  const long long wgs = std::max<long long>(1, T / BM) * heads;     // full tiles; the ragged ones are light
  int parts = 1;
  while (parts < 8 && wgs * parts < want && T * shared >= 16LL * BN * parts && T / nseq * shared >= 3 * BN) parts *= 2;
  return parts;
}
// More workgroups than CUs; under the causal mask, where the longest workgroup has twice the mean's work, as many as the CUs hold (two each) once the sequences are
// long enough for what the parts cost, and more for the longest.  Forward / both directions in us at 257 and so: one sequence of 16384, 4 heads of 64: 223 / 965 and
// 187 / 775; 5000, 10 heads of 96: 87 / 407 and 87 / 351; 4000, 9 heads of 128: 78 / 336 and 69 / 299; shorter: three of 1024, 16 heads of 64: 25 / 89 and, were
// they dealt out so, 33 / 114.  (The kernel of wide heads' dk and dv fills a CU by itself: 257.)
int wanted(const PackedAttnArgs& a, bool backward) {
  const long long mean = a.T / a.nseq;
  return !a.causal || mean < (backward ? 1280 : 2560) ? 257 : mean < 8192 ? 512 : 513;
}
// floats of workspace: forward {sums, statistics}; backward {delta, sums of dq and then of dk / dv}
long long forward_floats(const PackedAttnArgs& a) { return a.splits > 1 ? a.splits * a.T * a.Hq * (a.D + 2LL) : 0; }
long long delta_floats(const PackedAttnArgs& a) { return (a.T * a.Hq + 3) / 4 * 4; }
long long backward_floats(const PackedAttnArgs& a) {
  return delta_floats(a) + std::max(a.splits > 1 ? a.splits * a.T * a.Hq * a.D : 0LL, a.parts > 1 ? a.parts * a.T * a.Hkv * 2 * a.D : 0LL);
}

int refuse(const char* m) { return set_last_error(ASYRP_EINVAL, m); }

// the checks that both directions share, and how their work is dealt out; 0 or the error
int check(PackedAttnArgs& a, int dtype, const long long* strides, int n, bool backward) {
  if (dtype != ASYRP_F16 && dtype != ASYRP_BF16) return refuse("packed attention takes f16 or bf16 operands");
  if (a.D < 8 || a.D > 128 || a.D % 8) return refuse("packed attention: the head width must be a multiple of 8 from 8 to 128");
  if (a.Hq < 1 || a.Hkv < 1 || a.Hq % a.Hkv) return refuse("packed attention: query heads must be a multiple of key/value heads");
  if (a.nseq < 1 || a.T < 0 || a.T > 0x7fffffffLL) return refuse("packed attention: bad number of sequences or rows");
  if (!(a.scale > 0) || std::isinf(a.scale)) return refuse("packed attention: the scale must be positive and finite");
  for (int i = 0; i < n; ++i)
    if (strides[i] < 0 || strides[i] % 8 || strides[i] > (i % 2 ? 1LL << 40 : 1LL << 23))
      return refuse("packed attention: strides must be multiples of 8 values, not negative, rows at most 2^23 values apart");
  a.tiles = (int)std::min<long long>(a.T / BM + a.nseq + 1, 0x7fffffff);
  a.splits = parts_of(a.T, a.nseq, a.Hq, 1, wanted(a, backward));
  a.parts = parts_of(a.T, a.nseq, a.Hkv, a.Hq / a.Hkv, a.D > 64 ? 257 : wanted(a, backward));
  // a launch has fewer than 2^32 threads: 256 a workgroup of the forward, of dq and of dk / dv of narrow heads, 512 of those of wide ones
  const long long tiles = a.T / BM + a.nseq + 1, most = 0xffffffffLL;
  if (a.Hq > most / 256 / a.splits / tiles)
    return refuse("packed attention: (rows / 128 + sequences) x query heads are too many for one launch (2^24 at most, parts of long sequences counted)");
  if (backward && a.Hkv > most / (a.D > 64 ? 512 : 256) / a.parts / tiles)
    return refuse("packed attention: (rows / 128 + sequences) x key / value heads are too many for one launch (2^24 at most, heads wider than 64 twice and parts of long sequences counted)");
  return 0;
}
bool unaligned(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (!p || ((uintptr_t)p & 15)) return true;
  return false;
}

}  // namespace
}  // namespace asyrp

using namespace asyrp;

extern "C" {

int asyrp_packed_attention_forward(int device, const asyrp_packed_attention* p, const void* q, const void* k, const void* v, const int32_t* cu_seqlens, void* out,
                                   float* sums, void* out_rest, float* workspace, int fill_tail, void* stream) {
  if (!p || !cu_seqlens) return refuse("packed attention: null argument");
  PackedAttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.out = out; a.sums = (float2*)sums; a.cu = cu_seqlens;
  a.T = p->tokens; a.nseq = p->sequences; a.Hq = p->heads; a.Hkv = p->kv_heads; a.D = p->head_dim; a.causal = p->causal != 0; a.scale = p->scale;
  a.q_t = p->q_stride[0]; a.q_h = p->q_stride[1]; a.k_t = p->k_stride[0]; a.k_h = p->k_stride[1]; a.v_t = p->v_stride[0]; a.v_h = p->v_stride[1];
  a.o_t = p->out_stride[0]; a.o_h = p->out_stride[1];
  a.fill_tail = fill_tail; a.rest = out_rest;
  const long long st[] = {a.q_t, a.q_h, a.k_t, a.k_h, a.v_t, a.v_h, a.o_t, a.o_h};
  if (int rc = check(a, p->dtype, st, 8, false)) return rc;
  if (a.T == 0) return 0;
  a.partial = workspace;
  a.stats = reinterpret_cast<float2*>(workspace + (a.splits > 1 ? a.splits * a.T * a.Hq * a.D : 0));
  if (unaligned({q, k, v, out}) || ((uintptr_t)out_rest & 15) || ((uintptr_t)sums & 7) || ((uintptr_t)workspace & 15) || (a.splits > 1 && !workspace)) return refuse("packed attention: tensors must be given and 16-byte aligned");
  DeviceGuard g(device);
  if (g.error != hipSuccess) return set_last_error(ASYRP_EHIP, hipGetErrorString(g.error));
  const hipError_t e = p->dtype == ASYRP_F16 ? launch<_Float16>(a, false, (hipStream_t)stream) : launch<__bf16>(a, false, (hipStream_t)stream);
  return e == hipSuccess ? 0 : set_last_error(ASYRP_EHIP, hipGetErrorString(e));
}

int64_t asyrp_packed_attention_workspace(const asyrp_packed_attention* p, int backward) {
  if (!p) return refuse("packed attention: null argument");
  PackedAttnArgs a{};
  a.T = p->tokens; a.nseq = p->sequences; a.Hq = p->heads; a.Hkv = p->kv_heads; a.D = p->head_dim; a.causal = p->causal != 0; a.scale = p->scale;
  if (int rc = check(a, p->dtype, nullptr, 0, backward != 0)) return rc;
  return backward ? backward_floats(a) : forward_floats(a);
}

int asyrp_packed_attention_backward(int device, const asyrp_packed_attention* p, const void* q, const void* k, const void* v, const int32_t* cu_seqlens,
                                    const void* out, const float* sums, const void* out_rest, const void* d_out, float* workspace, void* dq, void* dk, void* dv, void* stream) {
  if (!p || !cu_seqlens) return refuse("packed attention: null argument");
  PackedAttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.o = out; a.sums = (float2*)sums; a.rest = const_cast<void*>(out_rest); a.dout = d_out; a.delta = workspace; a.dq = dq; a.dk = dk; a.dv = dv; a.cu = cu_seqlens;
  a.T = p->tokens; a.nseq = p->sequences; a.Hq = p->heads; a.Hkv = p->kv_heads; a.D = p->head_dim; a.causal = p->causal != 0; a.scale = p->scale;
  a.q_t = p->q_stride[0]; a.q_h = p->q_stride[1]; a.k_t = p->k_stride[0]; a.k_h = p->k_stride[1]; a.v_t = p->v_stride[0]; a.v_h = p->v_stride[1];
  a.o_t = p->out_stride[0]; a.o_h = p->out_stride[1]; a.do_t = p->dout_stride[0]; a.do_h = p->dout_stride[1];
  a.dq_t = (long long)a.Hq * a.D; a.dk_t = a.dv_t = (long long)a.Hkv * a.D;         // the gradients are contiguous
  a.dq_h = a.dk_h = a.dv_h = a.D;
  const long long st[] = {a.q_t, a.q_h, a.k_t, a.k_h, a.v_t, a.v_h, a.o_t, a.o_h, a.do_t, a.do_h};
  if (int rc = check(a, p->dtype, st, 10, true)) return rc;
  if (a.T == 0) return 0;
  a.partial = workspace + delta_floats(a);
  if (unaligned({q, k, v, out, d_out, dq, dk, dv}) || ((uintptr_t)out_rest & 15) || !sums || ((uintptr_t)sums & 7) || !workspace || ((uintptr_t)workspace & 15)) return refuse("packed attention: tensors must be given and 16-byte aligned");
  DeviceGuard g(device);
  if (g.error != hipSuccess) return set_last_error(ASYRP_EHIP, hipGetErrorString(g.error));
  const hipError_t e = p->dtype == ASYRP_F16 ? launch<_Float16>(a, true, (hipStream_t)stream) : launch<__bf16>(a, true, (hipStream_t)stream);
  return e == hipSuccess ? 0 : set_last_error(ASYRP_EHIP, hipGetErrorString(e));
}

}  // extern "C"
