// residual_norm.hip -- the seam between two residual blocks in one pass: the norm behind a block, its gate, the residual sum with its scale
// and the norm in front of the next block, forward and backward.
//
//   u = N1(y) (or y),   h = a x + gate * u,   n = N2(h),   N(t) = (t - mean) rstd * w + b  (layer)  or  t rstd * w + b  (rms)
//
// backward, with that = (t - mean) rstd and c = d that = d out * w:   d t = rstd (c - mean(c) - that mean(c that))   (rms: no mean(c)):
//   dh' = dh + N2'(dn),  dx = a dh',  dgate = sum over the gate's rows of dh' u,  dy = N1'(gate dh'),  dw = sum over rows of d out * that
//
// The work is bound by HBM: forward 2 reads and 2 writes of [rows, C], backward 4 reads and 2 writes (x and y are read again
// instead of h: h as stored is rounded to the stream's type, and the statistics and that belong to the unrounded one).  A row lives in
// registers from the first load to the last store.  Statistics, sums and the partial sums of the parameter gradients are fp32;
// mean and variance are taken in two passes over the registers, so no large sum of squares cancels.  Parameter gradients go
// through per-workgroup partial sums and a second kernel that adds them in a fixed order: no atomics.
//
// 65536 x 2048 in bf16, rms on both sides and a gate: forward 204 us (5.2 TB/s of its 1.07 GB), backward 345 us (4.7 TB/s of 1.61 GB) and 9 us for the partial
// sums; a large copy runs at 4.7 TB/s.  What carried it: sums over a wave by DPP instead of LDS exchanges and arithmetic without cases for absent parts
// (backward 462 -> 321 us: it had been bound by its instructions), four values a thread, and the next row's loads ahead of the current row.
#include "kernels.h"
#include "../../include/asyrp.h"

#include <algorithm>
#include <cmath>

namespace asyrp {
namespace {

struct NormArgs {
  const void *x, *y, *dh, *dn;
  void *h, *n, *dx, *dy;
  const float *gate, *w1, *b1, *w2, *b2;
  float *stats;              // [rows][4]: mean and rstd of y, mean and rstd of h (null: not kept)
  float *partial;            // [slots][vectors][C]
  float *dgate;
  float a, eps, inv_c;
  long long rows, per_gate;  // rows of one gate row
  int C, after, before, rms; // which norms there are
  int chunks;                // workgroups per gate row (1 where a workgroup takes whole gate rows)
  long long gates_per_wg, chunk_rows, gates;
  int row_gate;              // every row has its gate (and the walk takes them for one set of rows)
  int want_w1, want_b1, want_w2, want_b2, want_gate;
};
// partial vectors, in this order
enum { V_W2, V_B2, V_W1, V_B1, V_GATE, VECTORS };

// A thread's VPT values of a row: contiguous (VEC: whole groups of the row), or TPR (threads per row) apart, so that neighbouring lanes still read
// neighbouring values of a row of any width and address.
template <typename T, int VPT>
struct Raw {
  typedef T V __attribute__((ext_vector_type(VPT), aligned(sizeof(T) * VPT < 16 ? sizeof(T) * VPT : 16)));
  V v;
};
template <typename T, bool VEC, int TPR, int VPT>
__device__ __forceinline__ void load(const T* row, int t, int C, Raw<T, VPT>& o) {
  if (VEC) {
    if (t * VPT < C) {
      o.v = *reinterpret_cast<const typename Raw<T, VPT>::V*>(row + t * VPT);
    } else {
#pragma unroll
      for (int j = 0; j < VPT; ++j) o.v[j] = (T)0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < VPT; ++j) o.v[j] = j * TPR + t < C ? row[j * TPR + t] : (T)0.f;
  }
}
// The values are there behind this.  It stands before the current row's stores: loads and stores are counted together, and a wait behind
// stores that may or may not have been issued would wait for them too.
template <typename T, int VPT>
__device__ __forceinline__ void landed(Raw<T, VPT>& r) {
  typedef unsigned U __attribute__((ext_vector_type(sizeof(T) * VPT / 4)));
  U u = __builtin_bit_cast(U, r.v);
  asm volatile("" : "+v"(u));
  r.v = __builtin_bit_cast(typename Raw<T, VPT>::V, u);
}
template <typename T, int VPT>
__device__ __forceinline__ void floats(const Raw<T, VPT>& r, float (&o)[VPT]) {
#pragma unroll
  for (int j = 0; j < VPT; ++j) o[j] = (float)r.v[j];
}
template <bool VEC, int TPR, int VPT>
__device__ __forceinline__ void loadf(const float* row, int t, int C, float (&o)[VPT]) {
  Raw<float, VPT> r;
  load<float, VEC, TPR, VPT>(row, t, C, r);
  floats(r, o);
}
template <typename T, bool VEC, int TPR, int VPT>
__device__ __forceinline__ void store(T* row, int t, int C, const float (&o)[VPT]) {
  Raw<T, VPT> x;
#pragma unroll
  for (int j = 0; j < VPT; ++j) x.v[j] = (T)o[j];
  if (VEC) {
    if (t * VPT < C) *reinterpret_cast<typename Raw<T, VPT>::V*>(row + t * VPT) = x.v;
  } else {
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (j * TPR + t < C) row[j * TPR + t] = x.v[j];
  }
}
template <bool VEC, int TPR, int VPT>
__device__ __forceinline__ bool inside(int t, int j, int C) { return VEC ? t * VPT < C : j * TPR + t < C; }

// a wave's sum, in all lanes: within rows of 16 by shifts, then from row to row
__device__ __forceinline__ float wave_sum(float v) {
#define ASYRP_DPP(CTRL, ROWS) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, false))
  ASYRP_DPP(0x111, 0xf);
  ASYRP_DPP(0x112, 0xf);
  ASYRP_DPP(0x114, 0xf);
  ASYRP_DPP(0x118, 0xf);
  ASYRP_DPP(0x142, 0xa);
  ASYRP_DPP(0x143, 0xc);
#undef ASYRP_DPP
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
// sums over the 16 lanes of a row of lanes, in all of them
__device__ __forceinline__ float sum16(float v) {
#define ASYRP_DPP(CTRL) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false))
  ASYRP_DPP(0x121);
  ASYRP_DPP(0x122);
  ASYRP_DPP(0x124);
  ASYRP_DPP(0x128);
#undef ASYRP_DPP
  return v;
}
// sums of K values over the TPR threads of a row.  `buf` holds two sets of one row of K values per wave, used in turn, so that
// one barrier per reduction is enough.
template <int TPR, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* buf, int& turn, int sub, int t) {
  if (TPR == 16 || TPR == 32) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = sum16(v[k]);
      if (TPR == 32) v[k] += __shfl_xor(v[k], 16);
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
  if (TPR > 64) {
    constexpr int W = TPR / 64;
    float* b = buf + (turn * 16 + sub * W) * 2;
    turn ^= 1;
    if ((t & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) b[(t >> 6) * 2 + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (W == 16) {                     // sixteen waves: one read and four steps (4000 x 5041 in fp32, both directions: 450 us, with sixteen reads 596)
        v[k] = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(sum16(b[(t & 15) * 2 + k]))));
      } else {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) s += b[w * 2 + k];
        v[k] = s;
      }
    }
  }
}

// mean and rstd of the values (those behind C are zero and do not count).  The reciprocal root is the hardware's (one unit in the last place), except for
// values near the smallest ones, which eps = 0 alone leaves.
template <bool VEC, int TPR, int VPT>
__device__ __forceinline__ void statistics(const float (&v)[VPT], const NormArgs& p, float* buf, int& turn, int sub, int t, float& mean, float& rstd) {
  mean = 0.f;
  float s[1] = {0.f};
  if (!p.rms) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) s[0] += v[j];
    row_sum<TPR, 1>(s, buf, turn, sub, t);
    mean = s[0] * p.inv_c;
  }
  s[0] = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const float d = inside<VEC, TPR, VPT>(t, j, p.C) ? v[j] - mean : 0.f;
    s[0] = __builtin_fmaf(d, d, s[0]);
  }
  row_sum<TPR, 1>(s, buf, turn, sub, t);
  const float var = __builtin_fmaf(s[0], p.inv_c, p.eps);
  rstd = var > 1e-30f ? __builtin_amdgcn_rsqf(var) : 1.0f / sqrtf(var);
}

// a vector of the columns, or `fill` where there is none (zero behind C)
template <bool VEC, int TPR, int VPT>
__device__ __forceinline__ void columns(const float* row, float fill, int t, int C, float (&o)[VPT]) {
  if (row) {
    loadf<VEC, TPR, VPT>(row, t, C, o);
  } else {
#pragma unroll
    for (int j = 0; j < VPT; ++j) o[j] = inside<VEC, TPR, VPT>(t, j, C) ? fill : 0.f;
  }
}

// Weights, biases and gates that are not given are ones and zeros in registers, so that the arithmetic has no cases; behind C they are zeros, and with them
// whatever a sum over the row would take from there.
//
// Both directions: a workgroup of max(256, TPR) threads, TPR to a row, walks over the rows of one part of a gate row, or of several whole
// gate rows, with the weights (and, backward, the parameter gradients) of its columns in registers.  The next row's loads are issued before
// the current one is worked on, so that the reductions' barriers stand in the shadow of memory.
template <int TPR> constexpr int threads() { return TPR > 256 ? TPR : 256; }

template <typename X, typename Y, bool VEC, int TPR, int VPT>
__global__ __launch_bounds__(threads<TPR>()) void residual_norm_fwd_kernel(const NormArgs p) {
  __shared__ float buf[64];
  constexpr int SUB = threads<TPR>() / TPR;
  const bool row_gate = SUB > 1 && p.row_gate;
  const int sub = threadIdx.x / TPR, t = threadIdx.x % TPR, C = p.C;
  int turn = 0;
  float w1[VPT], w2[VPT], b1[VPT], b2[VPT];
  columns<VEC, TPR, VPT>(p.w1, 1.f, t, C, w1);
  columns<VEC, TPR, VPT>(p.b1, 0.f, t, C, b1);
  columns<VEC, TPR, VPT>(p.w2, 1.f, t, C, w2);
  columns<VEC, TPR, VPT>(p.b2, 0.f, t, C, b2);
  const long long g0 = (long long)(blockIdx.x / p.chunks) * p.gates_per_wg, g1 = min(p.gates, g0 + p.gates_per_wg);
  const int part = blockIdx.x % p.chunks;
  for (long long g = g0; g < g1; ++g) {
    const long long first = g * p.per_gate + part * p.chunk_rows, last = min(p.rows, min((g + 1) * p.per_gate, first + p.chunk_rows));
    float gate[VPT];
    if (!row_gate) columns<VEC, TPR, VPT>(p.gate ? p.gate + g * C : nullptr, 1.f, t, C, gate);
    Raw<X, VPT> xn{};
    Raw<Y, VPT> yn{};
    auto fetch = [&](long long r) {
      const long long row = min(r + sub, last - 1);
      load<Y, VEC, TPR, VPT>((const Y*)p.y + row * C, t, C, yn);
      load<X, VEC, TPR, VPT>((const X*)p.x + row * C, t, C, xn);
    };
    if (first < last) fetch(first);
    for (long long r0 = first; r0 < last; r0 += SUB) {
      const bool there = r0 + sub < last;
      const long long row = there ? r0 + sub : last - 1;
      float x[VPT], y[VPT];
      floats(xn, x);
      floats(yn, y);
      if (r0 + SUB < last) fetch(r0 + SUB);
      if (row_gate) columns<VEC, TPR, VPT>(p.gate + row * C, 1.f, t, C, gate);
      float m1 = 0.f, r1 = 1.f, m2 = 0.f, r2 = 1.f;
      if (p.after) {
        statistics<VEC, TPR, VPT>(y, p, buf, turn, sub, t, m1, r1);
#pragma unroll
        for (int j = 0; j < VPT; ++j) y[j] = __builtin_fmaf((y[j] - m1) * r1, w1[j], b1[j]);
      }
#pragma unroll
      for (int j = 0; j < VPT; ++j) x[j] = __builtin_fmaf(y[j], gate[j], p.a * x[j]);
      if (p.before) {
        statistics<VEC, TPR, VPT>(x, p, buf, turn, sub, t, m2, r2);
#pragma unroll
        for (int j = 0; j < VPT; ++j) y[j] = __builtin_fmaf((x[j] - m2) * r2, w2[j], b2[j]);
      }
      landed(xn);
      landed(yn);
      if (there) store<X, VEC, TPR, VPT>((X*)p.h + row * C, t, C, x);
      if (there && p.before) store<Y, VEC, TPR, VPT>((Y*)p.n + row * C, t, C, y);
      if (p.stats && there && t == 0) reinterpret_cast<float4*>(p.stats)[row] = make_float4(m1, r1, m2, r2);
    }
  }
}

template <typename X, typename Y, bool VEC, int TPR, int VPT>
__global__ __launch_bounds__(threads<TPR>()) void residual_norm_bwd_kernel(const NormArgs p) {
  constexpr int SUB = threads<TPR>() / TPR;
  const bool row_gate = SUB > 1 && p.row_gate;
  __shared__ float buf[64];
  __shared__ float join[SUB > 1 ? SUB * TPR * VPT : 1];
  const int sub = threadIdx.x / TPR, t = threadIdx.x % TPR, C = p.C;
  int turn = 0;
  // eight or sixteen values a thread leave no registers for the weights beside the sums, nor for a row ahead: they are read again for every row, from the caches
  // (8192 x 8192 in bf16, eight values, both directions: 501 us, with spilled registers 805)
  constexpr bool LEAN = VPT > 4;
  float w1[VPT], w2[VPT], b1[VPT];
  if (!LEAN) {
    columns<VEC, TPR, VPT>(p.w1, 1.f, t, C, w1);
    columns<VEC, TPR, VPT>(p.b1, 0.f, t, C, b1);
    columns<VEC, TPR, VPT>(p.w2, 1.f, t, C, w2);
  }
  float sw1[VPT], sb1[VPT], sw2[VPT], sb2[VPT], sg[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) sw1[j] = sb1[j] = sw2[j] = sb2[j] = 0.f;
  const long long g0 = (long long)(blockIdx.x / p.chunks) * p.gates_per_wg, g1 = min(p.gates, g0 + p.gates_per_wg);
  const int part = blockIdx.x % p.chunks;
  float* slot = p.partial + (long long)blockIdx.x * VECTORS * C;

  // adds the row groups' sums of one vector and writes it (join is free again behind it)
  auto put = [&](float (&v)[VPT], float* to) {
    if (SUB > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < VPT; ++j) join[(sub * VPT + j) * TPR + t] = v[j];
      __syncthreads();
      if (sub == 0)
#pragma unroll
        for (int j = 0; j < VPT; ++j)
          for (int s = 1; s < SUB; ++s) v[j] += join[(s * VPT + j) * TPR + t];
    }
    if (sub == 0) store<float, VEC, TPR, VPT>(to, t, C, v);
  };

  for (long long g = g0; g < g1; ++g) {
    const long long first = g * p.per_gate + part * p.chunk_rows, last = min(p.rows, min((g + 1) * p.per_gate, first + p.chunk_rows));
    float gate[VPT];
    if (!LEAN && !row_gate) columns<VEC, TPR, VPT>(p.gate ? p.gate + g * C : nullptr, 1.f, t, C, gate);
#pragma unroll
    for (int j = 0; j < VPT; ++j) sg[j] = 0.f;
    Raw<X, VPT> xn{}, dhn{};
    Raw<Y, VPT> yn{}, dnn{};
    float4 stn;
    auto fetch = [&](long long r) {
      const long long row = min(r + sub, last - 1);
      load<Y, VEC, TPR, VPT>((const Y*)p.y + row * C, t, C, yn);
      load<X, VEC, TPR, VPT>((const X*)p.x + row * C, t, C, xn);
      if (p.dn) load<Y, VEC, TPR, VPT>((const Y*)p.dn + row * C, t, C, dnn);
      if (p.dh) load<X, VEC, TPR, VPT>((const X*)p.dh + row * C, t, C, dhn);
      stn = reinterpret_cast<const float4*>(p.stats)[row];
    };
    if (!LEAN && first < last) fetch(first);
    for (long long r0 = first; r0 < last; r0 += SUB) {
      const bool there = r0 + sub < last;
      const long long row = there ? r0 + sub : last - 1;
      if (LEAN) {
        fetch(r0);
        columns<VEC, TPR, VPT>(p.w1, 1.f, t, C, w1);
        columns<VEC, TPR, VPT>(p.b1, 0.f, t, C, b1);
      }
      float x[VPT], y[VPT], dh[VPT], dn[VPT], u[VPT];
      floats(xn, x);
      floats(yn, y);
      floats(dhn, dh);
      floats(dnn, dn);
      const float4 st = stn;
      if (!LEAN && r0 + SUB < last) fetch(r0 + SUB);
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        y[j] = (y[j] - st.x) * st.y;                          // without the norm behind the block: mean 0, rstd 1
        u[j] = __builtin_fmaf(y[j], w1[j], b1[j]);
      }
      if (LEAN || row_gate) columns<VEC, TPR, VPT>(p.gate ? p.gate + (row_gate ? row : g) * C : nullptr, 1.f, t, C, gate);
      if (LEAN) columns<VEC, TPR, VPT>(p.w2, 1.f, t, C, w2);
      // `keep`: false only for the copies of the last row that fill up a set of rows
      const bool keep = SUB == 1 || there;
      if (p.before && p.dn) {
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
          x[j] = (__builtin_fmaf(u[j], gate[j], p.a * x[j]) - st.z) * st.w;
          if (keep) sw2[j] = __builtin_fmaf(dn[j], x[j], sw2[j]);
        }
        if (p.want_b2 && keep)
#pragma unroll
          for (int j = 0; j < VPT; ++j) sb2[j] += dn[j];
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
          dn[j] *= w2[j];
          s[0] += dn[j];
          s[1] = __builtin_fmaf(dn[j], x[j], s[1]);
        }
        row_sum<TPR, 2>(s, buf, turn, sub, t);
        const float c1 = p.rms ? 0.f : s[0] * p.inv_c, c2 = s[1] * p.inv_c;
#pragma unroll
        for (int j = 0; j < VPT; ++j) dh[j] = __builtin_fmaf(st.w, __builtin_fmaf(-x[j], c2, dn[j] - c1), dh[j]);
      }
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        x[j] = p.a * dh[j];                                   // dx
        u[j] *= dh[j];                                        // of the gate
        if (keep) sg[j] += u[j];
        dh[j] *= gate[j];
      }
      if (p.after) {
        float s[2] = {0.f, 0.f};
        if (keep)
#pragma unroll
          for (int j = 0; j < VPT; ++j) sw1[j] = __builtin_fmaf(dh[j], y[j], sw1[j]);
        if (p.want_b1 && keep)
#pragma unroll
          for (int j = 0; j < VPT; ++j) sb1[j] += dh[j];
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
          dh[j] *= w1[j];
          s[0] += dh[j];
          s[1] = __builtin_fmaf(dh[j], y[j], s[1]);
        }
        row_sum<TPR, 2>(s, buf, turn, sub, t);
        const float c1 = p.rms ? 0.f : s[0] * p.inv_c, c2 = s[1] * p.inv_c;
#pragma unroll
        for (int j = 0; j < VPT; ++j) dh[j] = st.y * __builtin_fmaf(-y[j], c2, dh[j] - c1);
      }
      if (!LEAN) {
        landed(xn);
        landed(yn);
        landed(dhn);
        landed(dnn);
      }
      if (there && row_gate && p.want_gate) store<float, VEC, TPR, VPT>(p.dgate + row * C, t, C, u);
      if (there && p.dx) store<X, VEC, TPR, VPT>((X*)p.dx + row * C, t, C, x);
      if (there && p.dy) store<Y, VEC, TPR, VPT>((Y*)p.dy + row * C, t, C, dh);
    }
    if (p.want_gate && !row_gate) put(sg, p.chunks == 1 ? p.dgate + g * C : slot + V_GATE * C);
  }
  if (p.want_w2) put(sw2, slot + V_W2 * C);
  if (p.want_b2) put(sb2, slot + V_B2 * C);
  if (p.want_w1) put(sw1, slot + V_W1 * C);
  if (p.want_b1) put(sb1, slot + V_B1 * C);
}

// column sums of the partial vectors: 64 columns per workgroup, its sixteen waves take every sixteenth slot
struct NormSumArgs {
  const float* partial;
  float* out[VECTORS];
  int C, slots;              // slots of the weights' gradients
  int chunks;                // slots of one gate row
  long long gates;
};
__global__ __launch_bounds__(1024) void residual_norm_sum_kernel(const NormSumArgs p) {
  __shared__ float part[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  const bool gate = blockIdx.y >= V_GATE;
  const int v = gate ? V_GATE : blockIdx.y;
  const long long g = gate ? blockIdx.y - V_GATE : 0;
  if (!p.out[v]) return;
  const long long s0 = gate ? g * p.chunks : 0, n = gate ? p.chunks : p.slots, step = (long long)VECTORS * p.C;
  const float* from = p.partial + (s0 * VECTORS + v) * p.C + c;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < p.C) {
    long long i = wave;
    for (; i + 240 < n; i += 256) {                     // sixteen loads on their way
      float x[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) x[k] = from[(i + 16 * k) * step];
#pragma unroll
      for (int k = 0; k < 16; ++k) s[k & 3] += x[k];
    }
    for (; i + 48 < n; i += 64)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] += from[(i + 16 * k) * step];
    for (; i < n; i += 16) s[0] += from[i * step];
  }
  part[wave][lane] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (wave == 0 && c < p.C) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += part[k][lane];
    p.out[v][g * p.C + c] = t;
  }
}

// Four values per thread keep the backward's registers (five sums, four weights, two rows) under 128, so that 16 waves share a CU.  Rows of up to 128 share a
// wave (63731 x 33 in fp32, both directions: 35 us, with a wave to each 56).  Rows over 4096 take sixteen values a thread (8192 x 8192 in bf16, both directions:
// 450 us, with eight 501) or, where they are no multiple of sixteen, eight.
constexpr int SHARED_WAVES = 512;        // up to this width a workgroup takes several rows at once
int values_per_thread(int C) { return C <= 4096 ? 4 : C % 16 == 0 ? 16 : 8; }
#define ASYRP_NORM(KERNEL) \
  if (a.C <= 64) hipLaunchKernelGGL((KERNEL<X, Y, VEC, 16, 4>), g, dim3(256), 0, s, a); \
  else if (a.C <= 128) hipLaunchKernelGGL((KERNEL<X, Y, VEC, 32, 4>), g, dim3(256), 0, s, a); \
  else if (a.C <= 256) hipLaunchKernelGGL((KERNEL<X, Y, VEC, 64, 4>), g, dim3(256), 0, s, a); \
  else if (a.C <= SHARED_WAVES) hipLaunchKernelGGL((KERNEL<X, Y, VEC, 128, 4>), g, dim3(256), 0, s, a); \
  else if (a.C <= 1024) hipLaunchKernelGGL((KERNEL<X, Y, VEC, 256, 4>), g, dim3(256), 0, s, a); \
  else if (a.C <= 2048) hipLaunchKernelGGL((KERNEL<X, Y, VEC, 512, 4>), g, dim3(512), 0, s, a); \
  else if (a.C <= 4096) hipLaunchKernelGGL((KERNEL<X, Y, VEC, 1024, 4>), g, dim3(1024), 0, s, a); \
  else if (VEC && values_per_thread(a.C) == 16) hipLaunchKernelGGL((KERNEL<X, Y, true, 512, 16>), g, dim3(512), 0, s, a); \
  else hipLaunchKernelGGL((KERNEL<X, Y, VEC, 1024, 8>), g, dim3(1024), 0, s, a)

template <typename X, typename Y, bool VEC>
hipError_t forward(const NormArgs& a, unsigned wgs, hipStream_t s) {
  const dim3 g(wgs);
  ASYRP_NORM(residual_norm_fwd_kernel);
  return hipGetLastError();
}
template <typename X, typename Y, bool VEC>
hipError_t backward(const NormArgs& a, unsigned wgs, hipStream_t s) {
  const dim3 g(wgs);
  ASYRP_NORM(residual_norm_bwd_kernel);
  return hipGetLastError();
}
#undef ASYRP_NORM
template <typename X, typename Y>
hipError_t launch(const NormArgs& a, bool vec, bool back, unsigned wgs, hipStream_t s) {
  if (back) return vec ? backward<X, Y, true>(a, wgs, s) : backward<X, Y, false>(a, wgs, s);
  return vec ? forward<X, Y, true>(a, wgs, s) : forward<X, Y, false>(a, wgs, s);
}
bool types(int x, int y) { return (x == ASYRP_F32 && (y == ASYRP_F32 || y == ASYRP_F16 || y == ASYRP_BF16)) || (x == y && (x == ASYRP_F16 || x == ASYRP_BF16)); }
hipError_t dispatch(int x, int y, const NormArgs& a, bool vec, bool back, unsigned wgs, hipStream_t s) {
  if (x == ASYRP_F32 && y == ASYRP_F32) return launch<float, float>(a, vec, back, wgs, s);
  if (x == ASYRP_F32 && y == ASYRP_F16) return launch<float, _Float16>(a, vec, back, wgs, s);
  if (x == ASYRP_F32) return launch<float, __bf16>(a, vec, back, wgs, s);
  return x == ASYRP_F16 ? launch<_Float16, _Float16>(a, vec, back, wgs, s) : launch<__bf16, __bf16>(a, vec, back, wgs, s);
}

int refuse(const char* m) { return set_last_error(ASYRP_EINVAL, m); }

int check(const asyrp_residual_norm* p) {
  if (!p) return refuse("residual norm: null argument");
  if (!types(p->stream_dtype, p->branch_dtype)) return refuse("residual norm: types are f32 with any branch, or f16 / bf16 for both");
  if (p->rows < 0 || p->rows > 0x7fffffffLL) return refuse("residual norm: bad number of rows");
  if (p->width < 1 || p->width > 8192) return refuse("residual norm: the width must be 1 .. 8192");
  if (p->kind != ASYRP_NORM_LAYER && p->kind != ASYRP_NORM_RMS) return refuse("residual norm: unknown kind of norm");
  if (p->gates < 0 || (p->gates > 0 && p->rows % p->gates)) return refuse("residual norm: the gate's rows must divide the rows");
  if (!std::isfinite(p->eps) || p->eps < 0 || !std::isfinite(p->residual_scale)) return refuse("residual norm: eps and the residual scale must be finite");
  return 0;
}
// How the rows are dealt out: `want` workgroups where the rows allow, each with a part of one gate row or with several whole ones
void deal(const asyrp_residual_norm* p, NormArgs& a, long long want, unsigned& wgs) {
  a.row_gate = p->gates == p->rows && p->width <= SHARED_WAVES;
  a.gates = p->gates > 0 && !a.row_gate ? p->gates : 1;
  a.per_gate = std::max<long long>(1, a.rows / a.gates);
  want = std::max<long long>(1, want);
  a.chunks = (int)std::max<long long>(1, std::min(want / a.gates, a.per_gate));
  a.chunk_rows = (a.per_gate + a.chunks - 1) / a.chunks;
  a.chunks = (int)((a.per_gate + a.chunk_rows - 1) / a.chunk_rows);
  a.gates_per_wg = a.chunks > 1 ? 1 : (a.gates + want - 1) / want;
  wgs = (unsigned)(((a.gates + a.gates_per_wg - 1) / a.gates_per_wg) * a.chunks);
}
// backward: at least four rows each, so that the partial sums stay a small part of the traffic
long long bwd_want(long long rows) { return std::min<long long>(1024, rows / 4); }
void fill(const asyrp_residual_norm* p, NormArgs& a) {
  a.rows = p->rows;
  a.C = p->width;
  a.rms = p->kind == ASYRP_NORM_RMS;
  a.after = p->after != 0;
  a.before = p->before != 0;
  a.a = p->residual_scale;
  a.eps = p->eps;
  a.inv_c = 1.0f / (float)p->width;
  a.per_gate = p->gates > 0 ? std::max<long long>(1, p->rows / p->gates) : std::max<long long>(1, p->rows);
}
bool aligned(std::initializer_list<const void*> ps) {
  for (const void* q : ps)
    if ((uintptr_t)q & 15) return false;
  return true;
}

}  // namespace
}  // namespace asyrp

using namespace asyrp;

extern "C" {

int asyrp_residual_norm_forward(int device, const asyrp_residual_norm* p, const void* x, const void* y, const float* gate, const float* after_weight,
                                const float* after_bias, const float* before_weight, const float* before_bias, void* h, void* n, float* stats, void* stream) {
  if (int rc = check(p)) return rc;
  if (p->rows == 0) return 0;
  if (!x || !y || !h || (p->before && !n) || (p->gates > 0) != (gate != nullptr)) return refuse("residual norm: null argument");
  NormArgs a{};
  fill(p, a);
  a.x = x; a.y = y; a.gate = gate; a.w1 = after_weight; a.b1 = after_bias; a.w2 = before_weight; a.b2 = before_bias; a.h = h; a.n = n; a.stats = stats;
  if (!aligned({stats})) return refuse("residual norm: the statistics must be 16-byte aligned");
  const bool vec = a.C % values_per_thread(a.C) == 0 && aligned({x, y, gate, after_weight, after_bias, before_weight, before_bias, h, n});
  unsigned wgs = 0;
  deal(p, a, std::min<long long>(4096, a.rows), wgs);
  DeviceGuard g(device);
  if (g.error != hipSuccess) return set_last_error(ASYRP_EHIP, hipGetErrorString(g.error));
  const hipError_t e = dispatch(p->stream_dtype, p->branch_dtype, a, vec, false, wgs, (hipStream_t)stream);
  return e == hipSuccess ? 0 : set_last_error(ASYRP_EHIP, hipGetErrorString(e));
}

int64_t asyrp_residual_norm_workspace(const asyrp_residual_norm* p) {
  if (int rc = check(p)) return rc;
  NormArgs a{};
  fill(p, a);
  unsigned wgs = 0;
  deal(p, a, bwd_want(a.rows), wgs);
  return (int64_t)wgs * VECTORS * a.C;
}

int asyrp_residual_norm_backward(int device, const asyrp_residual_norm* p, const void* x, const void* y, const float* gate, const float* after_weight,
                                 const float* after_bias, const float* before_weight, const float* stats, const void* dh, const void* dn, void* dx, void* dy,
                                 float* dgate, float* d_after_weight, float* d_after_bias, float* d_before_weight, float* d_before_bias, float* workspace,
                                 void* stream) {
  if (int rc = check(p)) return rc;
  float* outs[VECTORS] = {d_before_weight, d_before_bias, d_after_weight, d_after_bias, dgate};
  if (p->rows > 0 && (!x || !y || !stats || !workspace || (!dh && !dn) || (p->gates > 0) != (gate != nullptr) || (dgate && !gate)))
    return refuse("residual norm: null argument");
  if ((dn && !p->before) || ((d_after_weight || d_after_bias) && !p->after) || ((d_before_weight || d_before_bias) && !p->before))
    return refuse("residual norm: a gradient of a norm that is not there");
  if (p->rows == 0) return 0;
  if (!aligned({stats})) return refuse("residual norm: the statistics must be 16-byte aligned");
  NormArgs a{};
  fill(p, a);
  unsigned wgs = 0;
  deal(p, a, bwd_want(a.rows), wgs);
  a.x = x; a.y = y; a.gate = gate; a.w1 = after_weight; a.b1 = after_bias; a.w2 = before_weight; a.stats = const_cast<float*>(stats);
  a.dh = dh; a.dn = dn; a.dx = dx; a.dy = dy; a.partial = workspace; a.dgate = dgate;
  a.want_w2 = d_before_weight != nullptr; a.want_b2 = d_before_bias != nullptr; a.want_w1 = d_after_weight != nullptr; a.want_b1 = d_after_bias != nullptr;
  a.want_gate = dgate != nullptr;
  const bool vec = a.C % values_per_thread(a.C) == 0 && aligned({x, y, gate, after_weight, after_bias, before_weight, dh, dn, dx, dy, dgate, workspace});
  DeviceGuard g(device);
  if (g.error != hipSuccess) return set_last_error(ASYRP_EHIP, hipGetErrorString(g.error));
  hipError_t e = dispatch(p->stream_dtype, p->branch_dtype, a, vec, true, wgs, (hipStream_t)stream);
  if (e == hipSuccess) {
    NormSumArgs sa{};
    sa.partial = workspace;
    for (int i = 0; i < VECTORS; ++i) sa.out[i] = outs[i];
    sa.C = a.C;
    sa.slots = (int)wgs;
    sa.chunks = a.chunks;
    sa.gates = a.gates;
    if (a.chunks == 1 || a.row_gate) sa.out[V_GATE] = nullptr;     // whole gate rows were written by the kernel itself
    bool any = false;
    for (float* o : sa.out) any = any || o;
    if (any) {
      hipLaunchKernelGGL(residual_norm_sum_kernel, dim3((a.C + 63) / 64, V_GATE + (sa.out[V_GATE] ? (unsigned)a.gates : 0)), dim3(1024), 0, (hipStream_t)stream, sa);
      e = hipGetLastError();
    }
  }
  return e == hipSuccess ? 0 : set_last_error(ASYRP_EHIP, hipGetErrorString(e));
}

}  // extern "C"
