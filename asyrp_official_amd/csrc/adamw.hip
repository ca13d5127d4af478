// adamw.hip -- one AdamW step over many tensors at once, with first and second moments in 32 bits or in 8.
//
//   g' = g * min(1, max_norm / (||g|| + 1e-6));  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Everything is fp32 (each constant rounded once from fp64), the norm's sum of squares is fp64.  The work is bound by HBM: 28 bytes
// per fp32 value with 32-bit moments, 16 with 8-bit ones, and a second read of the gradient where they are clipped.  The table of the
// tensors travels in the kernel's arguments (100 tensors per launch), so a step uploads nothing and may be captured into a graph;
// step counts live on the device and are advanced there.
//
// 8-bit moments.  256 consecutive values (one wave's four per lane) share one exponent byte e, a power of two; a value is kept
// relative to it with three bits of mantissa: the first moment as sign, 4 bits of exponent, 3 of mantissa, the second as 5 + 3 without
// a sign.  Rounding is up or down at random in proportion to the distance, so the mean is kept: rounding to nearest would stop a
// second moment from ever falling, since one step changes it by a factor of 0.999 and the codes are 6 to 12 % apart.  The scale is a
// power of two so that it moves a value's place only by whole exponents and values that did not change are not rounded anew when it
// changes.  A second moment of a block that holds anything is never kept as zero (the smallest code is 1): the next first moment is at least
// as coarse, so no quotient of the two can grow beyond its block's.  An exponent byte of 0 is a block of zeros; 255 one that held a value that is
// not finite, and reads as NaN.
//
// 36.6 M fp32 values with 32-bit moments: 170 us (6.0 TB/s of its 1.03 GB).  146 M with 8-bit ones: 435 us (5.4 TB/s of 2.34 GB; 540 us while the codes were
// taken apart in branches and the largest value found through LDS); their moments as fp32 240 us (6.1 TB/s); the norm 4.0 TB/s, what reading alone
// reaches on this card.  The random bits are a hash of the value's place, the step and the caller's seed.
#include "kernels.h"
#include "../../include/asyrp.h"

#include <algorithm>
#include <cmath>

namespace asyrp {
namespace {

constexpr int MAXT = 100;          // tensors per launch: the table stays under the 4 KB of a kernel's arguments
constexpr int CHUNK = 4096;        // values of one workgroup's turn
constexpr int NORM_WGS = ASYRP_ADAMW_PARTIALS;

struct Tensor { void* p; const void* g; long long n, off; };
struct Table {
  Tensor t[MAXT];
  int first[MAXT];                 // number of the tensor's first chunk
  int count, chunks;
};
static_assert(sizeof(Table) < 3700, "the table and the other arguments have to fit a launch");

// per-step scalars on the device
struct Scalars { float step_size, inv_sqrt_bc2, keep, unused; };

struct StepArgs {
  float *m, *v;
  unsigned char *m8, *v8, *me, *ve;
  const Scalars* sc;               // [tensors of the launch]
  const float* clip;               // {factor, skip}, or null
  float b1, nb1, b2, nb2, eps;
  unsigned seed;
  const int* steps;                // this launch's tensors' counts, already advanced
};

__device__ __forceinline__ int tensor_of(const Table& tb, int chunk) {
  int lo = 0, hi = tb.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tb.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <typename T> struct Four { typedef T V __attribute__((ext_vector_type(4))); };

// four values, as one load where all are there and the tensor's address allows it
template <typename T>
__device__ __forceinline__ void load4(const T* p, long long i, long long n, bool whole, float (&o)[4]) {
  if (whole) {
    const typename Four<T>::V v = *reinterpret_cast<const typename Four<T>::V*>(p + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (float)v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = i + j < n ? (float)p[i + j] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, long long i, long long n, bool whole, const float (&o)[4]) {
  if (whole) {
    typename Four<T>::V v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (T)o[j];
    *reinterpret_cast<typename Four<T>::V*>(p + i) = v;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) p[i + j] = (T)o[j];
  }
}

template <typename T>
__global__ __launch_bounds__(256) void grad_sumsq_kernel(const Table tb, double* partial) {
  __shared__ double sm[4];
  double s = 0.0;
  for (int c = blockIdx.x; c < tb.chunks; c += gridDim.x) {
    const int k = tensor_of(tb, c);
    const T* g = (const T*)tb.t[k].g;
    const long long n = tb.t[k].n, base = (long long)(c - tb.first[k]) * CHUNK;
    const bool wide = ((uintptr_t)g & (4 * sizeof(T) - 1)) == 0;
    float v[CHUNK / 1024][4];
#pragma unroll
    for (int it = 0; it < CHUNK / 1024; ++it) load4(g, base + it * 1024 + threadIdx.x * 4, n, wide && base + CHUNK <= n, v[it]);
#pragma unroll
    for (int it = 0; it < CHUNK / 1024; ++it)
#pragma unroll
      for (int j = 0; j < 4; ++j) s += (double)v[it][j] * (double)v[it][j];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) partial[blockIdx.x] = (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

struct CountArgs {
  int* steps;                      // all counts of the caller's group
  int* now;                        // out: the counts of this launch's tensors
  Scalars* sc;                     // out
  float* clip;                     // out: {factor, skip}
  float* norm;                     // out, nullable
  const double* sumsq;             // partial sums of squares, or null: nothing is clipped
  const float* lr_dev;
  double lr, b1, b2, decay, max_norm;
  int index[MAXT], count, n_sumsq;
};
// one workgroup in front of each step: the norm and the factor that clips it, the step counts and what hangs on them
__global__ __launch_bounds__(256) void adamw_count_kernel(const CountArgs a) {
  __shared__ double sm[4];
  bool skip = false;
  if (a.sumsq) {
    double s = 0.0;
    for (int i = threadIdx.x; i < a.n_sumsq; i += 256) s += a.sumsq[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = s;
    __syncthreads();
    const double total = sqrt((sm[0] + sm[1]) + (sm[2] + sm[3])), f = a.max_norm / (total + 1e-6);
    skip = !(total <= 1.7976931348623157e308);                // infinite or NaN
    if (threadIdx.x == 0) {
      if (a.norm) *a.norm = (float)total;
      a.clip[0] = skip ? 0.f : (float)(f < 1.0 ? f : 1.0);
      a.clip[1] = skip ? 1.f : 0.f;
    }
  }
  const int i = threadIdx.x;
  if (i >= a.count) return;
  int t = a.steps[a.index[i]];
  if (!skip) a.steps[a.index[i]] = ++t;
  const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
  a.now[i] = t;
  a.sc[i] = Scalars{(float)(lr / (1.0 - pow(a.b1, (double)t))), (float)(1.0 / sqrt(1.0 - pow(a.b2, (double)t))), (float)(1.0 - lr * a.decay), 0.f};
}

__device__ __forceinline__ unsigned float_bits(float v) { return __float_as_uint(v); }

// exponent byte of a block from its largest magnitude's bits: rounding up may not leave the codes, so the next power of two is taken
// where the largest value is over 1.875 times its own
__device__ __forceinline__ int block_exponent(unsigned top, int lowest) {
  if (top == 0) return 0;
  const int e = (int)((top + 0xFFFFFu) >> 23);
  return e < lowest ? lowest : e > 255 ? 255 : e;
}
// What a block's exponent byte says, worked out once per wave.  A block of zeros (0) holds only codes 0; one that was not finite (255) too, and
// reads as NaN through its unit.
template <int EXP>
struct Block {
  unsigned low;                    // biased exponent of the smallest value with a whole mantissa
  float unit;                      // the step under it
  __device__ __forceinline__ explicit Block(int e) {
    low = (unsigned)max(e, EXP + 2) - (EXP - 2);
    unit = e == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((low - 3) << 23);
  }
  __device__ __forceinline__ float decode(unsigned c) const {
    const float small = (float)c * unit, whole = __uint_as_float((c + ((low - 1) << 3)) << 20);
    return c < 8 ? small : whole;
  }
  // (the product with a power of two is exact: one rounding, as if it stood alone)
  __device__ __forceinline__ unsigned encode(float t, unsigned coin) const {
    const unsigned b = float_bits(t), whole = ((b + coin) >> 20) - ((low - 1) << 3);
    const unsigned small = (unsigned)__builtin_fmaf(t, __uint_as_float((257 - low) << 23), (float)coin * 0x1p-20f);
    return b >= low << 23 ? whole : small;
  }
};
constexpr int M_EXP = 16, V_EXP = 32;
__device__ __forceinline__ float decode_m(unsigned c, const Block<M_EXP>& k) { return __uint_as_float(float_bits(k.decode(c & 127u)) | (c & 128u) << 24); }

// largest value of the wave's lanes, as a scalar: rows of 16 by shifts, then row to row
__device__ __forceinline__ unsigned wave_max(unsigned v) {
#define ASYRP_DPP(CTRL, ROWS) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false))
  ASYRP_DPP(0x111, 0xf);
  ASYRP_DPP(0x112, 0xf);
  ASYRP_DPP(0x114, 0xf);
  ASYRP_DPP(0x118, 0xf);
  ASYRP_DPP(0x142, 0xa);
  ASYRP_DPP(0x143, 0xc);
#undef ASYRP_DPP
  return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}

// One wave's 256 values from `i0` of a tensor on.  WHOLE: all of them are there and may be loaded four at a time.
template <typename T, int BITS, bool WHOLE>
__device__ __forceinline__ void step_block(T* p, const T* g, long long n, long long off, long long i0, int lane, const StepArgs& a, const Scalars& sc, float clip,
                                           unsigned key) {
  const long long i = i0 + lane * 4, si = off + i;
  float pv[4], gv[4], m[4], v[4];
  load4(p, i, n, WHOLE, pv);
  load4(g, i, n, WHOLE, gv);
  if (BITS == 32) {
    const float4 mv = *reinterpret_cast<const float4*>(a.m + si), vv = *reinterpret_cast<const float4*>(a.v + si);
    m[0] = mv.x; m[1] = mv.y; m[2] = mv.z; m[3] = mv.w;
    v[0] = vv.x; v[1] = vv.y; v[2] = vv.z; v[3] = vv.w;
  } else {
    const unsigned mc = *reinterpret_cast<const unsigned*>(a.m8 + si), vc = *reinterpret_cast<const unsigned*>(a.v8 + si);
    const Block<M_EXP> mb(__builtin_amdgcn_readfirstlane(a.me[(off + i0) >> 8]));
    const Block<V_EXP> vb(__builtin_amdgcn_readfirstlane(a.ve[(off + i0) >> 8]));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = decode_m((mc >> (8 * j)) & 255u, mb);
      v[j] = vb.decode((vc >> (8 * j)) & 255u);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float gg = gv[j] * clip;
    m[j] = m[j] * a.b1 + gg * a.nb1;
    v[j] = v[j] * a.b2 + (gg * gg) * a.nb2;
    pv[j] = pv[j] * sc.keep;
    // with 8-bit moments the kernel is as near to its arithmetic as to HBM, and the quotient is taken from the hardware's square root and
    // reciprocal (one unit in the last place each, of a quotient whose moments are 6 to 12 % wide)
    if (BITS == 32) pv[j] = pv[j] - (m[j] / (sqrtf(v[j]) * sc.inv_sqrt_bc2 + a.eps)) * sc.step_size;
    else pv[j] = pv[j] - (m[j] * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[j]) * sc.inv_sqrt_bc2 + a.eps)) * sc.step_size;
  }
  store4(p, i, n, WHOLE, pv);
  if (BITS == 32) {
    *reinterpret_cast<float4*>(a.m + si) = make_float4(m[0], m[1], m[2], m[3]);
    *reinterpret_cast<float4*>(a.v + si) = make_float4(v[0], v[1], v[2], v[3]);
    return;
  }
  unsigned tm = 0, tv = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (!WHOLE && i + j >= n) m[j] = v[j] = 0.f;
    tm = max(tm, float_bits(m[j]) & 0x7fffffffu);
    tv = max(tv, float_bits(v[j]) & 0x7fffffffu);
  }
  const int me = block_exponent(wave_max(tm), M_EXP + 2), ve = block_exponent(wave_max(tv), V_EXP + 2);
  const Block<M_EXP> mb(me);
  const Block<V_EXP> vb(ve);
  const bool some_m = me != 0 && me != 255, some_v = ve != 0 && ve != 255;
  const unsigned at = (unsigned)si, k = key ^ ((unsigned)((off + i0) >> 32) * 0xC2B2AE3Du);
  unsigned mc = 0, vc = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    unsigned x = (at + j) ^ k;                       // `at` is a multiple of four: no carry
    x = (x ^ (x >> 16)) * 0x7FEB352Du;
    x = (x ^ (x >> 15)) * 0x846CA68Bu;
    x ^= x >> 16;
    const unsigned cm = mb.encode(fabsf(m[j]), x & 0xFFFFFu) | (float_bits(m[j]) >> 24 & 128u);
    unsigned cv = max(vb.encode(v[j], (x * 0x9E3779B1u) >> 12), 1u);
    if (!WHOLE && i + j >= n) cv = 0;
    mc |= cm << (8 * j);
    vc |= cv << (8 * j);
  }
  *reinterpret_cast<unsigned*>(a.m8 + si) = some_m ? mc : 0u;
  *reinterpret_cast<unsigned*>(a.v8 + si) = some_v ? vc : 0u;
  if (lane == 0) {
    a.me[(off + i0) >> 8] = (unsigned char)me;
    a.ve[(off + i0) >> 8] = (unsigned char)ve;
  }
}

template <typename T, int BITS>
__global__ __launch_bounds__(256) void adamw_step_kernel(const Table tb, const StepArgs a) {
  if (a.clip && a.clip[1] != 0.f) return;                     // the norm is not finite: nothing changes
  const int chunk = tb.chunks - 1 - blockIdx.x;               // from the end: what the norm's pass read last is still in the caches
  const int k = tensor_of(tb, chunk);
  const float clip = a.clip ? a.clip[0] : 1.f;
  const Scalars sc = a.sc[k];
  T* p = (T*)tb.t[k].p;
  const T* g = (const T*)tb.t[k].g;
  const long long n = tb.t[k].n, off = tb.t[k].off;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long base = (long long)(chunk - tb.first[k]) * CHUNK + wave * 256;
  const bool wide = (((uintptr_t)p | (uintptr_t)g) & (4 * sizeof(T) - 1)) == 0;
  const unsigned key = (a.seed * 0x9E3779B1u) ^ ((unsigned)(BITS == 8 ? a.steps[k] : 0) * 0x85EBCA77u);
  if (wide && base + (CHUNK - 1024) + 256 <= n) {
#pragma unroll
    for (int it = 0; it < CHUNK / 1024; ++it) step_block<T, BITS, true>(p, g, n, off, base + it * 1024, lane, a, sc, clip, key);
  } else {
#pragma unroll 1
    for (long long i0 = base; i0 < base + CHUNK && i0 < n; i0 += 1024) step_block<T, BITS, false>(p, g, n, off, i0, lane, a, sc, clip, key);
  }
}

__global__ __launch_bounds__(256) void adamw_moments_kernel(const unsigned char* m8, const unsigned char* v8, const unsigned char* me, const unsigned char* ve,
                                                            float* m, float* v, long long n) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const unsigned mc = *reinterpret_cast<const unsigned*>(m8 + i), vc = *reinterpret_cast<const unsigned*>(v8 + i);
  const Block<M_EXP> a(me[i >> 8]);
  const Block<V_EXP> b(ve[i >> 8]);
  float4 mo, vo;
  mo.x = decode_m(mc & 255u, a); mo.y = decode_m((mc >> 8) & 255u, a); mo.z = decode_m((mc >> 16) & 255u, a); mo.w = decode_m(mc >> 24, a);
  vo.x = b.decode(vc & 255u); vo.y = b.decode((vc >> 8) & 255u); vo.z = b.decode((vc >> 16) & 255u); vo.w = b.decode(vc >> 24);
  *reinterpret_cast<float4*>(m + i) = mo;
  *reinterpret_cast<float4*>(v + i) = vo;
}

int refuse(const char* m) { return set_last_error(ASYRP_EINVAL, m); }
int failed(hipError_t e) { return e == hipSuccess ? 0 : set_last_error(ASYRP_EHIP, hipGetErrorString(e)); }

int check(const asyrp_adamw_tensor* t, int n, int dtype) {
  if (n < 0 || (n > 0 && !t)) return refuse("AdamW: null argument");
  if (dtype != ASYRP_F32 && dtype != ASYRP_F16 && dtype != ASYRP_BF16) return refuse("AdamW: tensors are f32, f16 or bf16");
  for (int i = 0; i < n; ++i) {
    if (t[i].numel < 0 || t[i].numel > (1LL << 40) || t[i].offset < 0 || t[i].offset % 256) return refuse("AdamW: bad tensor size or state offset");
    if (t[i].numel > 0 && !t[i].grad) return refuse("AdamW: null tensor");
    if (((uintptr_t)t[i].grad | (uintptr_t)t[i].param) & (dtype == ASYRP_F32 ? 3 : 1)) return refuse("AdamW: misaligned tensor");
  }
  return 0;
}
// the next launch's table: tensors from `from` on; returns the number taken
int table(const asyrp_adamw_tensor* t, int n, int from, Table& tb) {
  int i = from;
  long long chunks = 0;
  tb.count = 0;
  for (; i < n && tb.count < MAXT; ++i) {
    const long long c = (t[i].numel + CHUNK - 1) / CHUNK;
    if (chunks + c > 0x7fffffffLL) break;
    tb.t[tb.count] = Tensor{t[i].param, t[i].grad, t[i].numel, t[i].offset};
    tb.first[tb.count] = (int)chunks;
    chunks += c;
    ++tb.count;
  }
  tb.chunks = (int)chunks;
  return i - from;
}

}  // namespace
}  // namespace asyrp

using namespace asyrp;

extern "C" {

int asyrp_grad_sumsq(int device, const asyrp_adamw_tensor* tensors, int n, int dtype, double* partial, void* stream) {
  if (int rc = check(tensors, n, dtype)) return rc;
  if (!partial) return refuse("AdamW: null argument");
  DeviceGuard dg(device);
  if (dg.error != hipSuccess) return failed(dg.error);
  Table tb;
  for (int from = 0; from < n;) {
    const int took = table(tensors, n, from, tb);
    const dim3 g(NORM_WGS), b(256);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == ASYRP_F32) hipLaunchKernelGGL(grad_sumsq_kernel<float>, g, b, 0, s, tb, partial);
    else if (dtype == ASYRP_F16) hipLaunchKernelGGL(grad_sumsq_kernel<_Float16>, g, b, 0, s, tb, partial);
    else hipLaunchKernelGGL(grad_sumsq_kernel<__bf16>, g, b, 0, s, tb, partial);
    if (hipError_t e = hipGetLastError()) return failed(e);
    partial += NORM_WGS;
    from += took;
  }
  return 0;
}

int asyrp_adamw_step(int device, const asyrp_adamw* c, const asyrp_adamw_tensor* tensors, int n, int dtype, void* scratch, void* stream) {
  if (int rc = check(tensors, n, dtype)) return rc;
  if (!c || (n > 0 && (!scratch || !c->steps))) return refuse("AdamW: null argument");
  if (c->state_bits != 32 && c->state_bits != 8) return refuse("AdamW: states are kept in 32 or 8 bits");
  // (tensors without values have a step count and no moments)
  const bool any = std::any_of(tensors, tensors + n, [](const asyrp_adamw_tensor& t) { return t.numel > 0; });
  if (any && (!c->exp_avg || !c->exp_avg_sq || (c->state_bits == 8 && (!c->exp_avg_scale || !c->exp_avg_sq_scale)))) return refuse("AdamW: null state");
  if (((uintptr_t)c->exp_avg | (uintptr_t)c->exp_avg_sq | (uintptr_t)scratch) & 15) return refuse("AdamW: states must be 16-byte aligned");
  if (!(c->beta1 >= 0 && c->beta1 < 1 && c->beta2 >= 0 && c->beta2 < 1) || !(c->eps >= 0) || !std::isfinite(c->eps) || !std::isfinite(c->weight_decay) || !std::isfinite(c->lr))
    return refuse("AdamW: betas must lie in [0, 1), eps, lr and weight decay must be finite");
  for (int i = 0; i < n; ++i)
    if ((tensors[i].numel > 0 && !tensors[i].param) || tensors[i].index < 0 || tensors[i].index > 0x7fffffffLL) return refuse("AdamW: null tensor or bad index");
  if (c->sumsq && (c->sumsq_count < 0 || !(c->max_norm > 0) || !std::isfinite(c->max_norm))) return refuse("AdamW: max_norm must be positive and finite");
  DeviceGuard dg(device);
  if (dg.error != hipSuccess) return failed(dg.error);
  hipStream_t s = (hipStream_t)stream;
  Table tb;
  float* clip = c->sumsq ? (float*)scratch : nullptr;
  Scalars* scalars = (Scalars*)scratch + 1;
  for (int from = 0; from < n;) {
    const int took = table(tensors, n, from, tb);
    CountArgs ca;
    ca.steps = c->steps;
    ca.sc = scalars + from;
    ca.now = reinterpret_cast<int*>(scalars + n) + from;
    ca.clip = clip; ca.norm = c->grad_norm; ca.sumsq = c->sumsq; ca.n_sumsq = c->sumsq_count; ca.max_norm = c->max_norm;
    ca.lr_dev = c->lr_device; ca.lr = c->lr; ca.b1 = c->beta1; ca.b2 = c->beta2; ca.decay = c->weight_decay;
    ca.count = tb.count;
    for (int i = 0; i < tb.count; ++i) ca.index[i] = (int)tensors[from + i].index;
    hipLaunchKernelGGL(adamw_count_kernel, dim3(1), dim3(256), 0, s, ca);
    if (hipError_t e = hipGetLastError()) return failed(e);
    if (tb.chunks > 0) {
      StepArgs a{};
      a.m = (float*)c->exp_avg; a.v = (float*)c->exp_avg_sq; a.m8 = (unsigned char*)c->exp_avg; a.v8 = (unsigned char*)c->exp_avg_sq;
      a.me = c->exp_avg_scale; a.ve = c->exp_avg_sq_scale;
      a.sc = ca.sc; a.steps = ca.now; a.clip = clip; a.seed = c->seed;
      a.b1 = (float)c->beta1; a.nb1 = (float)(1 - c->beta1); a.b2 = (float)c->beta2; a.nb2 = (float)(1 - c->beta2);
      a.eps = (float)c->eps;
      const dim3 g(tb.chunks), b(256);
#define ASYRP_STEP(T) \
  if (c->state_bits == 32) hipLaunchKernelGGL((adamw_step_kernel<T, 32>), g, b, 0, s, tb, a); \
  else hipLaunchKernelGGL((adamw_step_kernel<T, 8>), g, b, 0, s, tb, a)
      if (dtype == ASYRP_F32) { ASYRP_STEP(float); }
      else if (dtype == ASYRP_F16) { ASYRP_STEP(_Float16); }
      else { ASYRP_STEP(__bf16); }
#undef ASYRP_STEP
      if (hipError_t e = hipGetLastError()) return failed(e);
    }
    from += took;
  }
  return 0;
}

int asyrp_adamw_moments(int device, const uint8_t* exp_avg, const uint8_t* exp_avg_sq, const uint8_t* exp_avg_scale, const uint8_t* exp_avg_sq_scale, int64_t n,
                        float* out_avg, float* out_avg_sq, void* stream) {
  if (n < 0 || n % 256 || n / 1024 > 0x7fffffffLL) return refuse("AdamW: the state's length must be a multiple of 256");
  if (n == 0) return 0;
  if (!exp_avg || !exp_avg_sq || !exp_avg_scale || !exp_avg_sq_scale || !out_avg || !out_avg_sq) return refuse("AdamW: null argument");
  if (((uintptr_t)exp_avg | (uintptr_t)exp_avg_sq | (uintptr_t)out_avg | (uintptr_t)out_avg_sq) & 15) return refuse("AdamW: states must be 16-byte aligned");
  DeviceGuard dg(device);
  if (dg.error != hipSuccess) return failed(dg.error);
  hipLaunchKernelGGL(adamw_moments_kernel, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, (hipStream_t)stream, exp_avg, exp_avg_sq, exp_avg_scale,
                     exp_avg_sq_scale, out_avg, out_avg_sq, (long long)n);
  return failed(hipGetLastError());
}

}  // extern "C"
