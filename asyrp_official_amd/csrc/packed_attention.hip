// packed_attention.hip -- attention over sequences packed behind each other, forward and backward (f16 / bf16 operands, fp32 sums).
//
//   S = scale * q k^T (causal: keys <= the query), P = softmax(S), o = P v, lse = log sum exp S
//   dv = P^T do,  dS = P * (do v^T - delta) * scale with delta = rowsum(do * o),  dq = dS k,  dk = dS^T q
//
// All three kernels work on v_mfma_f32_32x32x16_{f16,bf16}.  A wave owns 32 queries (forward, dq) or 32 keys (dk/dv) as the COLUMNS of
// its products, so that a column's statistics are one value per lane and a row reduction is a sum over a lane's own 16 registers plus
// one exchange with lane ^ 32.  The result of a product (column = lane & 31, row = 8 (r / 4) + 4 (lane / 32) + r % 4) is used as the second
// operand of the next one without moving a value between lanes: the order in which a product runs over its inner index is free, so
// the first operand is simply read in the order in which the registers hold the second (rows {4h .. 4h+3, 8+4h .. 8+4h+3} of 16, h = lane / 32),
// by the transposing 16-bit LDS read, which hands a lane four rows of one column.
//
// The probabilities are rounded to the operands' type before P v, P^T do and dS k, dS^T q (half a step per term, relative to it); every
// sum, the row maximum, the row sum and delta are fp32.  There is no atomic: dq and dk/dv are two kernels that each form S
// again (7 products instead of 5), and the result does not depend on the order in which workgroups run.
#include "kernels.h"
#include "../../include/asyrp.h"

#include <algorithm>
#include <cmath>
#include <string>

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
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct PackedAttnArgs {
  const void *q, *k, *v, *o, *dout;
  void *out, *dq, *dk, *dv;
  float* lse;                // [Hq][T]
  float* delta;              // [Hq][T]
  const int* cu;
  long long T;
  int nseq, Hq, Hkv, D, causal, fill_tail;
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

// one row's fragment from global memory: d = 16 * ks + 8 * h + 0..7, zero beyond D or where the row is not there
template <typename T>
__device__ __forceinline__ typename Frag<T>::V load_frag(const T* row, int ks, int h, int D, bool there) {
  union { u32x4 u; typename Frag<T>::V v; } x;
  x.u = u32x4{0, 0, 0, 0};
  const int d = 16 * ks + 8 * h;
  if (there && d < D) x.u = *reinterpret_cast<const u32x4*>(row + d);
  return x.v;
}

template <int DP, int ROWS>
struct Stage {              // a tile on its way from global memory to LDS through registers
  static constexpr int N = ROWS * (DP / 8) / 256;
  u32x4 r[N];
  template <typename T>
  __device__ __forceinline__ void load(const T* base, long long stride, int rows, int D, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = tid + i * 256, row = c / (DP / 8), col = c % (DP / 8);
      r[i] = u32x4{0, 0, 0, 0};
      if (row < rows && col * 8 < D) r[i] = *reinterpret_cast<const u32x4*>(base + row * stride + col * 8);
    }
  }
  __device__ __forceinline__ void store(char* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = tid + i * 256, row = c / (DP / 8), col = c % (DP / 8);
      *reinterpret_cast<u32x4*>(tile + lds_at<DP>(row, col)) = r[i];
    }
  }
};

// The sequence and the row tile that tile number `t` of the launch stands for.  Tiles are numbered sequence by sequence; the numbers
// behind the last one share the rows behind the last sequence.  Every wave finds it by itself: 64 lengths at a time, summed over the wave.
// Offsets are held inside [0, T] and never fall, so that no value of `cu` leads outside the tensors.
struct TileAt { long long start; int len, row0; int idle; int idles; long long end; };
__device__ __forceinline__ TileAt find_tile(const int* cu, int nseq, long long T, int t, int tiles, int lane) {
  TileAt f{0, 0, 0, 0, 1, 0};
  int before = 0;
  bool found = false;
  long long high = 0;
  for (int b0 = 0; b0 < nseq; b0 += 64) {
    const int b = b0 + lane;
    long long s = 0, e = 0;
    if (b < nseq) { s = cu[b]; e = cu[b + 1]; }
    s = s < 0 ? 0 : s > T ? T : s;
    e = e < s ? s : e > T ? T : e;
    const int n = (int)((e - s + BM - 1) / BM);
    int sum = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(sum, o);
      if (lane >= o) sum += up;
    }
    const int first = before + sum - n;
    const unsigned long long hit = __ballot(n > 0 && t >= first && t < first + n);
    if (hit) {
      const int src = __ffsll(hit) - 1;
      f.start = __shfl(s, src);
      f.len = (int)(__shfl(e, src) - f.start);
      f.row0 = (t - __shfl(first, src)) * BM;
      found = true;
      break;
    }
    before += __shfl(sum, 63);
    high = __shfl(e, nseq - 1 - b0 < 63 ? nseq - 1 - b0 : 63);
  }
  if (!found) {
    f.idle = 1 + (t - before);
    f.idles = tiles - before;
    f.end = high;
  }
  return f;
}

// zeros in the rows behind the last sequence: the idle tiles of each head take them in turn
template <typename T>
__device__ __forceinline__ void zero_tail(T* p, long long st, long long sh, int head, int D, const TileAt& f, long long total, int tid) {
  const int chunks = D / 8;
  for (long long row = f.end + (f.idle - 1); row < total; row += f.idles)
    for (int c = tid; c < chunks; c += 256) *reinterpret_cast<u32x4*>(p + row * st + head * sh + c * 8) = u32x4{0, 0, 0, 0};
}

__device__ __forceinline__ float both_halves_max(float v) { return fmaxf(v, __shfl_xor(v, 32)); }
__device__ __forceinline__ float both_halves_sum(float v) { return v + __shfl_xor(v, 32); }

// rows d of a transposed result (column = this lane's row of the output tensor) times `m`, as 8-byte stores
template <typename T, int DP>
__device__ __forceinline__ void store_cols(T* row, const f32x16 (&acc)[DP / 32], float m, int h, int D) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const int d = 32 * dt + 8 * r4 + 4 * h;
      if (d >= D) continue;
      union { T t[4]; u32x2 u; } x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x.t[j] = (T)(acc[dt][4 * r4 + j] * m);
      *reinterpret_cast<u32x2*>(row + d) = x.u;
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

template <typename T, int DP>
__global__ __launch_bounds__(256) void packed_attn_fwd_kernel(const PackedAttnArgs p) {
  __shared__ __attribute__((aligned(16))) char kt[BN * DP * 2], vt[BN * DP * 2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  const int head = blockIdx.x % p.Hq, tile = p.tiles - 1 - blockIdx.x / p.Hq;
  const TileAt f = find_tile(p.cu, p.nseq, p.T, tile, p.tiles, lane);
  if (f.idle) {
    if (p.fill_tail) zero_tail((T*)p.out, p.o_t, p.o_h, head, p.D, f, p.T, tid);
    return;
  }
  const int hk = head / (p.Hq / p.Hkv);
  const T* k = (const T*)p.k + f.start * p.k_t + hk * p.k_h;
  const T* v = (const T*)p.v + f.start * p.v_t + hk * p.v_h;
  const int row = f.row0 + wave * 32 + (lane & 31);
  const bool there = row < f.len;
  const T* qrow = (const T*)p.q + (f.start + (there ? row : 0)) * p.q_t + head * p.q_h;
  typename Frag<T>::V qf[DP / 16];
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) qf[ks] = load_frag<T>(qrow, ks, h, p.D, there);

  f32x16 acc[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;
  float m = -INFINITY, l = 0.f;
  const float sc = p.scale * LOG2E;
  const int kend = p.causal ? min(f.len, f.row0 + BM) : f.len;
  const int wend = p.causal ? min(f.len, f.row0 + wave * 32 + 32) : f.len;     // keys this wave has to look at
  Stage<DP, BN> ks_, vs_;
  ks_.load(k, p.k_t, f.len, p.D, tid);
  vs_.load(v, p.v_t, f.len, p.D, tid);
  for (int k0 = 0; k0 < kend; k0 += BN) {
    __syncthreads();
    ks_.store(kt, tid);
    vs_.store(vt, tid);
    __syncthreads();
    if (k0 + BN < kend) {
      ks_.load(k + (long long)(k0 + BN) * p.k_t, p.k_t, f.len - k0 - BN, p.D, tid);
      vs_.load(v + (long long)(k0 + BN) * p.v_t, p.v_t, f.len - k0 - BN, p.D, tid);
    }
    if (k0 >= wend) continue;
    f32x16 s[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[n][r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) s[n] = Frag<T>::mma(read_rows<T, DP>(kt, 32 * n, ks, lane), qf[ks], s[n]);
    }
    const int last = p.causal ? min(row, f.len - 1) : f.len - 1;    // the last key this column sees
    const bool edge = k0 + BN > f.len || (p.causal && k0 + BN - 1 > f.row0 + wave * 32);
    float mx = -INFINITY;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float x = s[n][r] * sc;
        if (edge && k0 + 32 * n + 8 * (r >> 2) + 4 * h + (r & 3) > last) x = -INFINITY;
        s[n][r] = x;
        mx = fmaxf(mx, x);
      }
    const float mn = fmaxf(m, both_halves_max(mx));
    const float keep = exp2f(m - mn);
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float e = exp2f(s[n][r] - mn);
        s[n][r] = e;
        sum += e;
      }
    l = l * keep + sum;
    m = mn;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[dt][r] *= keep;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const typename Frag<T>::V pf = pack8<T>(s[n], b);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = Frag<T>::mma(read_cols<T, DP>(vt, 32 * n + 16 * b, dt, lane), pf, acc[dt]);
      }
  }
  l = both_halves_sum(l);
  if (there) {
    store_cols<T, DP>((T*)p.out + (f.start + row) * p.o_t + head * p.o_h, acc, 1.0f / l, h, p.D);
    if (p.lse && h == 0) p.lse[(long long)head * p.T + f.start + row] = (m + log2f(l)) * LN2;
  }
}

// dq, and delta = rowsum(do * o) for the other kernel
template <typename T, int DP>
__global__ __launch_bounds__(256) void packed_attn_dq_kernel(const PackedAttnArgs p) {
  __shared__ __attribute__((aligned(16))) char kt[BN * DP * 2], vt[BN * DP * 2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  const int head = blockIdx.x % p.Hq, tile = p.tiles - 1 - blockIdx.x / p.Hq;
  const TileAt f = find_tile(p.cu, p.nseq, p.T, tile, p.tiles, lane);
  if (f.idle) {
    zero_tail((T*)p.dq, p.dq_t, p.dq_h, head, p.D, f, p.T, tid);
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
  typename Frag<T>::V qf[DP / 16], gf[DP / 16];
  float delta = 0.f;
#pragma unroll
  for (int ks = 0; ks < DP / 16; ++ks) {
    qf[ks] = load_frag<T>(qrow, ks, h, p.D, there);
    gf[ks] = load_frag<T>(grow, ks, h, p.D, there);
    const typename Frag<T>::V of = load_frag<T>(orow, ks, h, p.D, there);
#pragma unroll
    for (int j = 0; j < 8; ++j) delta += (float)gf[ks][j] * (float)of[j];
  }
  delta = both_halves_sum(delta);
  const float lse2 = there ? p.lse[(long long)head * p.T + at] * LOG2E : 0.f;
  if (there && h == 0) p.delta[(long long)head * p.T + at] = delta;

  f32x16 acc[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[dt][r] = 0.f;
  const float sc = p.scale * LOG2E;
  const int kend = p.causal ? min(f.len, f.row0 + BM) : f.len;
  const int wend = p.causal ? min(f.len, f.row0 + wave * 32 + 32) : f.len;
  Stage<DP, BN> ks_, vs_;
  ks_.load(k, p.k_t, f.len, p.D, tid);
  vs_.load(v, p.v_t, f.len, p.D, tid);
  for (int k0 = 0; k0 < kend; k0 += BN) {
    __syncthreads();
    ks_.store(kt, tid);
    vs_.store(vt, tid);
    __syncthreads();
    if (k0 + BN < kend) {
      ks_.load(k + (long long)(k0 + BN) * p.k_t, p.k_t, f.len - k0 - BN, p.D, tid);
      vs_.load(v + (long long)(k0 + BN) * p.v_t, p.v_t, f.len - k0 - BN, p.D, tid);
    }
    if (k0 >= wend) continue;
    const int last = there ? (p.causal ? row : f.len - 1) : -1;
    const bool edge = k0 + BN > f.len || f.row0 + wave * 32 + 32 > f.len || (p.causal && k0 + BN - 1 > f.row0 + wave * 32);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      f32x16 s, g;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = g[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        s = Frag<T>::mma(read_rows<T, DP>(kt, 32 * n, ks, lane), qf[ks], s);
        g = Frag<T>::mma(read_rows<T, DP>(vt, 32 * n, ks, lane), gf[ks], g);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float e = exp2f(s[r] * sc - lse2) * (g[r] - delta);
        if (edge && k0 + 32 * n + 8 * (r >> 2) + 4 * h + (r & 3) > last) e = 0.f;
        s[r] = e;
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const typename Frag<T>::V pf = pack8<T>(s, b);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = Frag<T>::mma(read_cols<T, DP>(kt, 32 * n + 16 * b, dt, lane), pf, acc[dt]);
      }
    }
  }
  if (there) store_cols<T, DP>((T*)p.dq + at * p.dq_t + head * p.dq_h, acc, p.scale, h, p.D);
}

// dk and dv of 128 keys: over the query heads that share them and the query tiles that see them
template <typename T, int DP>
__global__ __launch_bounds__(256) void packed_attn_dkv_kernel(const PackedAttnArgs p) {
  __shared__ __attribute__((aligned(16))) char qt[BN * DP * 2], gt[BN * DP * 2];
  __shared__ __attribute__((aligned(16))) float ls[BN], ds[BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
  const int hk = blockIdx.x % p.Hkv, tile = blockIdx.x / p.Hkv, G = p.Hq / p.Hkv;
  const TileAt f = find_tile(p.cu, p.nseq, p.T, tile, p.tiles, lane);
  if (f.idle) {
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
  const float sc = p.scale * LOG2E;
  const int qbeg = p.causal ? f.row0 : 0;               // a multiple of BN
  const int per = (f.len - qbeg + BN - 1) / BN, total = per * G;
  Stage<DP, BN> qs, gs;
  auto fetch = [&](int i) {
    const int head = hk * G + i / per, q0 = qbeg + (i % per) * BN;
    qs.load((const T*)p.q + (f.start + q0) * p.q_t + head * p.q_h, p.q_t, f.len - q0, p.D, tid);
    gs.load((const T*)p.dout + (f.start + q0) * p.do_t + head * p.do_h, p.do_t, f.len - q0, p.D, tid);
  };
  fetch(0);
  for (int i = 0; i < total; ++i) {
    const int head = hk * G + i / per, q0 = qbeg + (i % per) * BN;
    __syncthreads();
    qs.store(qt, tid);
    gs.store(gt, tid);
    if (tid < BN) {
      const bool in = q0 + tid < f.len;
      const long long a = (long long)head * p.T + f.start + q0 + tid;
      ls[tid] = in ? p.lse[a] * LOG2E : 0.f;
      ds[tid] = in ? p.delta[a] : 0.f;
    }
    __syncthreads();
    if (i + 1 < total) fetch(i + 1);
    if (p.causal && q0 + BN <= f.row0 + wave * 32) continue;      // every query lies before this wave's keys
    const bool edge = q0 + BN > f.len || (p.causal && q0 < f.row0 + wave * 32 + 31);
#pragma unroll
    for (int n = 0; n < BN / 32; ++n) {
      f32x16 s, g;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = g[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        s = Frag<T>::mma(read_rows<T, DP>(qt, 32 * n, ks, lane), kf[ks], s);
        g = Frag<T>::mma(read_rows<T, DP>(gt, 32 * n, ks, lane), vf[ks], g);
      }
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const f32x4 lv = *reinterpret_cast<const f32x4*>(&ls[32 * n + 8 * r4 + 4 * h]);
        const f32x4 dl = *reinterpret_cast<const f32x4*>(&ds[32 * n + 8 * r4 + 4 * h]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 4 * r4 + j, q = q0 + 32 * n + 8 * r4 + 4 * h + j;
          float e = exp2f(s[r] * sc - lv[j]);
          if (edge && (q >= f.len || (p.causal && q < row))) e = 0.f;
          s[r] = e;
          g[r] = e * (g[r] - dl[j]);
        }
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const typename Frag<T>::V pf = pack8<T>(s, b), zf = pack8<T>(g, b);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) {
          dv[dt] = Frag<T>::mma(read_cols<T, DP>(gt, 32 * n + 16 * b, dt, lane), pf, dv[dt]);
          dk[dt] = Frag<T>::mma(read_cols<T, DP>(qt, 32 * n + 16 * b, dt, lane), zf, dk[dt]);
        }
      }
    }
  }
  if (there) {
    store_cols<T, DP>((T*)p.dk + at * p.dk_t + hk * p.dk_h, dk, p.scale, h, p.D);
    store_cols<T, DP>((T*)p.dv + at * p.dv_t + hk * p.dv_h, dv, 1.0f, h, p.D);
  }
}

template <typename T, int DP>
hipError_t launch_forward(const PackedAttnArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((packed_attn_fwd_kernel<T, DP>), dim3((unsigned)a.tiles * a.Hq), dim3(256), 0, s, a);
  return hipGetLastError();
}
template <typename T, int DP>
hipError_t launch_backward(const PackedAttnArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((packed_attn_dq_kernel<T, DP>), dim3((unsigned)a.tiles * a.Hq), dim3(256), 0, s, a);
  hipLaunchKernelGGL((packed_attn_dkv_kernel<T, DP>), dim3((unsigned)a.tiles * a.Hkv), dim3(256), 0, s, a);
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

int refuse(const std::string& m) { return set_last_error(ASYRP_EINVAL, m.c_str()); }

// the checks that both directions share; 0 or the error
int check(const PackedAttnArgs& a, int dtype, const long long* strides, int n) {
  if (dtype != ASYRP_F16 && dtype != ASYRP_BF16) return refuse("packed attention takes f16 or bf16 operands");
  if (a.D < 8 || a.D > 128 || a.D % 8) return refuse("packed attention: the head width must be a multiple of 8 from 8 to 128");
  if (a.Hq < 1 || a.Hkv < 1 || a.Hq % a.Hkv) return refuse("packed attention: query heads must be a multiple of key/value heads");
  if (a.nseq < 1 || a.T < 0 || a.T > 0x7fffffffLL) return refuse("packed attention: bad number of sequences or rows");
  if (!(a.scale == a.scale) || std::isinf(a.scale)) return refuse("packed attention: the scale must be finite");
  for (int i = 0; i < n; ++i)
    if (strides[i] < 0 || strides[i] % 8 || strides[i] > (1LL << 40)) return refuse("packed attention: strides must be multiples of 8 values, not negative");
  const long long tiles = a.T / BM + a.nseq + 1;
  if (tiles * a.Hq > 0x7fffffffLL) return refuse("packed attention: too many rows x heads for one launch");
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
                                   float* lse, int fill_tail, void* stream) {
  if (!p || !cu_seqlens) return refuse("packed attention: null argument");
  PackedAttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.out = out; a.lse = lse; a.cu = cu_seqlens;
  a.T = p->tokens; a.nseq = p->sequences; a.Hq = p->heads; a.Hkv = p->kv_heads; a.D = p->head_dim; a.causal = p->causal != 0; a.scale = p->scale;
  a.q_t = p->q_stride[0]; a.q_h = p->q_stride[1]; a.k_t = p->k_stride[0]; a.k_h = p->k_stride[1]; a.v_t = p->v_stride[0]; a.v_h = p->v_stride[1];
  a.o_t = p->out_stride[0]; a.o_h = p->out_stride[1];
  a.fill_tail = fill_tail;
  const long long st[] = {a.q_t, a.q_h, a.k_t, a.k_h, a.v_t, a.v_h, a.o_t, a.o_h};
  if (int rc = check(a, p->dtype, st, 8)) return rc;
  if (a.T == 0) return 0;
  if (unaligned({q, k, v, out})) return refuse("packed attention: tensors must be given and 16-byte aligned");
  a.tiles = (int)(a.T / BM + a.nseq + 1);
  DeviceGuard g(device);
  if (g.error != hipSuccess) return set_last_error(ASYRP_EHIP, hipGetErrorString(g.error));
  const hipError_t e = p->dtype == ASYRP_F16 ? launch<_Float16>(a, false, (hipStream_t)stream) : launch<__bf16>(a, false, (hipStream_t)stream);
  return e == hipSuccess ? 0 : set_last_error(ASYRP_EHIP, hipGetErrorString(e));
}

int asyrp_packed_attention_backward(int device, const asyrp_packed_attention* p, const void* q, const void* k, const void* v, const int32_t* cu_seqlens,
                                    const void* out, const float* lse, const void* d_out, float* delta, void* dq, void* dk, void* dv, void* stream) {
  if (!p || !cu_seqlens) return refuse("packed attention: null argument");
  PackedAttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.o = out; a.lse = const_cast<float*>(lse); a.dout = d_out; a.delta = delta; a.dq = dq; a.dk = dk; a.dv = dv; a.cu = cu_seqlens;
  a.T = p->tokens; a.nseq = p->sequences; a.Hq = p->heads; a.Hkv = p->kv_heads; a.D = p->head_dim; a.causal = p->causal != 0; a.scale = p->scale;
  a.q_t = p->q_stride[0]; a.q_h = p->q_stride[1]; a.k_t = p->k_stride[0]; a.k_h = p->k_stride[1]; a.v_t = p->v_stride[0]; a.v_h = p->v_stride[1];
  a.o_t = p->out_stride[0]; a.o_h = p->out_stride[1]; a.do_t = p->dout_stride[0]; a.do_h = p->dout_stride[1];
  a.dq_t = (long long)a.Hq * a.D; a.dk_t = a.dv_t = (long long)a.Hkv * a.D;         // the gradients are contiguous
  a.dq_h = a.dk_h = a.dv_h = a.D;
  const long long st[] = {a.q_t, a.q_h, a.k_t, a.k_h, a.v_t, a.v_h, a.o_t, a.o_h, a.do_t, a.do_h};
  if (int rc = check(a, p->dtype, st, 10)) return rc;
  if (a.T == 0) return 0;
  if (unaligned({q, k, v, out, d_out, dq, dk, dv}) || !lse || !delta) return refuse("packed attention: tensors must be given and 16-byte aligned");
  a.tiles = (int)(a.T / BM + a.nseq + 1);
  DeviceGuard g(device);
  if (g.error != hipSuccess) return set_last_error(ASYRP_EHIP, hipGetErrorString(g.error));
  const hipError_t e = p->dtype == ASYRP_F16 ? launch<_Float16>(a, true, (hipStream_t)stream) : launch<__bf16>(a, true, (hipStream_t)stream);
  return e == hipSuccess ? 0 : set_last_error(ASYRP_EHIP, hipGetErrorString(e));
}

}  // extern "C"
