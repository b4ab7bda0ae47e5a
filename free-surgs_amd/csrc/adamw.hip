// adamw.hip -- AdamW over many tensors at once (moments in 32 or in 8 bits) and the gradients' global norm, for gfx950 (MI355X).
//
//   g' = c g                                          c: the bound on the global norm, or 1
//   m  = b1 m + (1 - b1) g',   v = b2 v + (1 - b2) g'^2
//   w  = w (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// A few dozen operations an element against 16 to 30 bytes: everything here is bound by HBM, so each kernel reads and writes
// every array once, with 16-byte accesses where the type allows, and one launch takes up to 48 tensors.
//
// Which tensor a workgroup belongs to: lane k of every wave compares the workgroup's number with the first workgroup of
// tensor k, and the number of lanes at or past theirs is the answer -- one load and one ballot, no search.
//
// Moments in 8 bits: 128 consecutive elements of a tensor share one power of two for m and one for r = sqrt(v).  The codes are
// OCP e4m3 of m / 2^E and r / 2^E with the smallest E that brings the block's largest finite value to at most 448, stored as
// E + 127 in a byte.  r rather than v, because r needs half the exponent range.  A value between two codes goes up when its
// remainder reaches over the threshold of its element at this step: 20 bits of a Weyl sequence over the elements that each step
// shifts by a hash of its number.  For one element the thresholds of different steps are as good as independent, so a moment
// that moves by less than a code a step still moves in the mean as it should: with b2 = 0.999, r moves by 5e-4 a step and half
// a code is 3e-2 to 6e-2, so that rounding to nearest would hold it for good.  (A quasi-random sequence over the steps too
// lets r fall 7 % too fast: it leaves every code after the mean waiting time exactly, and ln 2 > 1/9 + ... + 1/16.)  r > 0
// keeps at least the smallest code, so that m is never divided by a denominator that the rounding took away.  The step
// itself uses m and r before the rounding.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <cstring>
#include <new>

#include "../../include/fsgs.h"
#include "fsgs_host.h"

using namespace fsgs;

namespace {

constexpr int TENSORS = 48;            // of one launch: the table is a kernel argument, 4 KB at most
constexpr int HYPERS = 8;              // different sets of scalars of one launch
constexpr int THREADS = 256;
constexpr int CHUNK = 4096;            // elements of one workgroup
constexpr int64_t MAX_BLOCKS = 1 << 23;  // workgroups of one launch (256 threads each: 2^31 work items)
constexpr int QBLOCK = FSGS_ADAMW_BLOCK;  // elements that share a power of two
constexpr int NORM_GROUPS = 2048;      // workgroups of one norm launch at most: eight per CU

// what a step's scalars come to; one per tensor where they are formed on the device
struct Hyper {
  float decay;          // 1 - lr wd
  float step_size;      // lr / (1 - b1^t)
  float inv_bc2_sqrt;   // 1 / sqrt(1 - b2^t)
  float eps;
  float b1, omb1, b2, omb2;
  uint32_t shift_m, shift_r;  // the step's part of the rounding thresholds
};
constexpr uint32_t PHASE_M = 0x9E3779B9u, PHASE_R = 0x6A09E667u;  // 2^32 frac(golden ratio), 2^32 frac(sqrt 2)
__host__ __device__ inline uint32_t shift_of(uint32_t x) {  // a hash: multiplication by 2^32 frac(sqrt 3), frac(sqrt 5), made odd
  x ^= x >> 16; x *= 0xBB67AE85u;
  x ^= x >> 15; x *= 0x3C6EF373u;
  return x ^ (x >> 16);
}

__host__ __device__ inline Hyper make_hyper(double lr, double b1, double b2, double eps, double wd, double step) {
  Hyper h;
  h.decay = (float)(1.0 - lr * wd);
  h.step_size = (float)(lr / (1.0 - pow(b1, step)));
  h.inv_bc2_sqrt = (float)(1.0 / sqrt(1.0 - pow(b2, step)));
  h.eps = (float)eps;
  // 1 - beta in double: 1 - 0.999f is off by 4.7e-5 of itself
  h.b1 = (float)b1; h.omb1 = (float)(1.0 - b1); h.b2 = (float)b2; h.omb2 = (float)(1.0 - b2);
  const uint32_t t = (uint32_t)(int64_t)step;
  h.shift_m = shift_of(2 * t); h.shift_r = shift_of(2 * t + 1);
  return h;
}

struct Table {
  void *p[TENSORS];
  const void *g[TENSORS];
  void *m[TENSORS], *v[TENSORS];
  void *w[TENSORS];        // fp32 master weights
  uint8_t *scales[TENSORS];
  int64_t n[TENSORS];
  uint32_t start[TENSORS];  // first workgroup
  uint8_t hyper[TENSORS];
  Hyper h[HYPERS];
  const Hyper *dev_h;       // one per tensor, or NULL: h[hyper[k]]
  const float *coef;        // factor on the gradients, or NULL
  int count;
  float sign;               // -1: ascend
};
static_assert(sizeof(Table) <= 4096, "kernel argument");

__device__ __forceinline__ int owner(const uint32_t *start, int count, uint32_t group) {
  const int lane = threadIdx.x & 63;
  const bool at = lane < count && group >= start[lane < TENSORS ? lane : TENSORS - 1];
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(at)) - 1);
}

// vectors of four that need only their element's alignment: the hardware's wide global accesses ask for no more
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf4u __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 half4u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32u __attribute__((aligned(1)));
typedef uint16_t u16u __attribute__((aligned(1)));
template <typename T> struct Vec4;
template <> struct Vec4<float> { typedef float4u type; };
template <> struct Vec4<__bf16> { typedef bf4u type; };
template <> struct Vec4<_Float16> { typedef half4u type; };

template <typename T> __device__ __forceinline__ void load4(const T *at, float (&x)[4]) {
  const typename Vec4<T>::type a = *(const typename Vec4<T>::type *)at;
#pragma unroll
  for (int j = 0; j < 4; j++) x[j] = (float)a[j];
}
template <typename T> __device__ __forceinline__ void store4(T *at, const float (&x)[4]) {
  typename Vec4<T>::type a;
#pragma unroll
  for (int j = 0; j < 4; j++) a[j] = (T)x[j];  // one rounding to the parameter's type, to nearest even
  *(typename Vec4<T>::type *)at = a;
}
template <typename T> __device__ __forceinline__ void load_some(const T *at, float (&x)[4], int have) {
#pragma unroll
  for (int j = 0; j < 4; j++) x[j] = j < have ? (float)at[j] : 0.0f;
}
template <typename T> __device__ __forceinline__ void store_some(T *at, const float (&x)[4], int have) {
#pragma unroll
  for (int j = 0; j < 4; j++)
    if (j < have) at[j] = (T)x[j];
}

// ---- moments in 32 bits ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void adamw_one(float &w, float g, float &m, float &v, const Hyper &h) {
  m = fmaf(h.b1, m, h.omb1 * g);
  v = fmaf(h.b2, v, h.omb2 * (g * g));
  w = fmaf(w, h.decay, -h.step_size * (m / fmaf(sqrtf(v), h.inv_bc2_sqrt, h.eps)));
}

template <typename T, bool MASTER> __global__ __launch_bounds__(THREADS) void adamw32_kernel(Table t) {
  const int k = owner(t.start, t.count, blockIdx.x);
  const Hyper h = t.dev_h ? t.dev_h[k] : t.h[t.hyper[k]];
  const float scale = t.sign * (t.coef ? *t.coef : 1.0f);
  const int64_t base = (int64_t)(blockIdx.x - t.start[k]) * CHUNK;
  const int64_t left = t.n[k] - base;
  T *p = (T *)t.p[k] + base;
  const T *g = (const T *)t.g[k] + base;
  float *m = (float *)t.m[k] + base, *v = (float *)t.v[k] + base, *w = MASTER ? (float *)t.w[k] + base : nullptr;
  constexpr int U = CHUNK / (THREADS * 4);
  float ww[U][4], gg[U][4], mm[U][4], vv[U][4];
  if (left >= CHUNK) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = (u * THREADS + threadIdx.x) * 4;
      load4(g + i, gg[u]); load4(m + i, mm[u]); load4(v + i, vv[u]);
      if constexpr (MASTER) load4(w + i, ww[u]); else load4(p + i, ww[u]);
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = (u * THREADS + threadIdx.x) * 4, have = (int)left - i;
      load_some(g + i, gg[u], have); load_some(m + i, mm[u], have); load_some(v + i, vv[u], have);
      if constexpr (MASTER) load_some(w + i, ww[u], have); else load_some(p + i, ww[u], have);
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int j = 0; j < 4; j++) adamw_one(ww[u][j], gg[u][j] * scale, mm[u][j], vv[u][j], h);
  if (left >= CHUNK) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = (u * THREADS + threadIdx.x) * 4;
      store4(p + i, ww[u]); store4(m + i, mm[u]); store4(v + i, vv[u]);
      if constexpr (MASTER) store4(w + i, ww[u]);
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = (u * THREADS + threadIdx.x) * 4, have = (int)left - i;
      store_some(p + i, ww[u], have); store_some(m + i, mm[u], have); store_some(v + i, vv[u], have);
      if constexpr (MASTER) store_some(w + i, ww[u], have);
    }
  }
}

// ---- moments in 8 bits ----------------------------------------------------------------------------------------------
// A block of 128 is two halves of 64; 16 lanes hold four elements of each half, so that every access of the 16 lanes is
// contiguous (256 bytes of fp32, 64 of codes) and the block's maximum is four steps within one row of lanes.
__device__ __forceinline__ uint32_t row_max(uint32_t a) {
  a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x128, 0xF, 0xF, false));  // row_ror:8
  a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x124, 0xF, 0xF, false));
  a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x122, 0xF, 0xF, false));
  return max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x121, 0xF, 0xF, false));
}
__device__ __forceinline__ uint32_t finite_bits(float x) {  // |x| as an integer (ordered like |x|), 0 for infinities and NaN
  const uint32_t a = __float_as_uint(x) & 0x7FFFFFFFu;
  return a < 0x7F800000u ? a : 0u;
}
// E + 127 for a block whose largest value has these bits: e - 8, one more where the mantissa is over 1.75 = 448 / 2^8
__device__ __forceinline__ int block_exponent(uint32_t top) { return max(1, (int)((top + 0x1FFFFFu) >> 23) - 8); }

// e4m3 code of |x| 2^-E: `inv` = 2^-E, `u` the threshold in [0, 2^20).  Normal codes: the threshold is added below the three
// mantissa bits that stay.  Below 2^-6 the codes are 2^-9 apart: adding 2^-6 gives a number whose mantissa has that grain.
// Infinities and NaN come out above every code and are held at 127, e4m3's NaN.
__device__ __forceinline__ uint32_t code_of(float x, float inv, uint32_t u) {
  const float y = fabsf(x) * inv;
  const bool low = y < 0x1p-6f;
  const uint32_t bits = __float_as_uint(low ? y + 0x1p-6f : y);
  return min(((bits + u) >> 20) - (low ? 968u : 960u), 127u);
}
// four codes of a moment; thresholds: base + j phase, upper 20 bits
template <bool KEEP>
__device__ __forceinline__ uint32_t codes_of(const float (&x)[4], float inv, uint32_t base, uint32_t phase) {
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    uint32_t c = code_of(x[j], inv, (base + (uint32_t)j * phase) >> 12);
    if constexpr (KEEP) c = max(c, x[j] > 0.0f ? 1u : 0u);
    else c |= (__float_as_uint(x[j]) >> 24) & 0x80u;
    word |= c << (8 * j);
  }
  return word;
}
__device__ __forceinline__ void values_of(uint32_t word, float unit, float (&x)[4]) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, true);
  x[0] = a[0] * unit; x[1] = a[1] * unit; x[2] = b[0] * unit; x[3] = b[1] * unit;
}
__device__ __forceinline__ float power(uint32_t e) { return __uint_as_float(e << 23); }  // 2^(e - 127); 0 for e = 0
__device__ __forceinline__ uint32_t load_codes(const uint8_t *at, int have) {
  if (have >= 4) return *(const u32u *)at;
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 3; j++)
    if (j < have) word |= (uint32_t)at[j] << (8 * j);
  return word;
}
__device__ __forceinline__ void store_codes(uint8_t *at, uint32_t word, int have) {
  if (have >= 4) { *(u32u *)at = word; return; }
#pragma unroll
  for (int j = 0; j < 3; j++)
    if (j < have) at[j] = (uint8_t)(word >> (8 * j));
}

// Each operation is a statement of its own, so that none is contracted: a code then hangs on the same sums and products,
// rounded one by one, that any fp32 program forms (a value next to its threshold is off by a whole code otherwise).
__device__ __forceinline__ void adamw8_one(float &w, float g, float &m, float &r, const Hyper &h) {
  const float m0 = h.b1 * m, m1 = h.omb1 * g;
  m = m0 + m1;
  const float v0 = r * r, g2 = g * g;
  const float v1 = h.b2 * v0, v2 = h.omb2 * g2;
  r = sqrtf(v1 + v2);
  w = fmaf(w, h.decay, -h.step_size * (m / fmaf(r, h.inv_bc2_sqrt, h.eps)));
}

template <typename T, bool MASTER> __global__ __launch_bounds__(THREADS) void adamw8_kernel(Table t) {
  const int k = owner(t.start, t.count, blockIdx.x);
  const Hyper h = t.dev_h ? t.dev_h[k] : t.h[t.hyper[k]];
  const float scale = t.sign * (t.coef ? *t.coef : 1.0f);
  const int64_t base = (int64_t)(blockIdx.x - t.start[k]) * CHUNK;
  const int left = (int)min(t.n[k] - base, (int64_t)CHUNK);
  T *p = (T *)t.p[k] + base;
  const T *g = (const T *)t.g[k] + base;
  uint8_t *m = (uint8_t *)t.m[k] + base, *r = (uint8_t *)t.v[k] + base, *scales = t.scales[k] + 2 * (base / QBLOCK);
  float *w = MASTER ? (float *)t.w[k] + base : nullptr;
  constexpr int U = CHUNK / (THREADS * 8);
  // block of this lane and its first element in it
  const int row = threadIdx.x / 16, at = (threadIdx.x & 15) * 4;
  float ww[U][2][4], gg[U][2][4];
  uint32_t mq[U][2], rq[U][2], sc[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int b = u * (THREADS / 16) + row;
    sc[u] = b * QBLOCK < left ? *(const u16u *)(scales + 2 * b) : 0u;
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const int i = b * QBLOCK + s * 64 + at;
      if (left == CHUNK) {
        load4(g + i, gg[u][s]);
        if constexpr (MASTER) load4(w + i, ww[u][s]); else load4(p + i, ww[u][s]);
        mq[u][s] = *(const u32u *)(m + i);
        rq[u][s] = *(const u32u *)(r + i);
      } else {
        load_some(g + i, gg[u][s], left - i);
        if constexpr (MASTER) load_some(w + i, ww[u][s], left - i); else load_some(p + i, ww[u][s], left - i);
        mq[u][s] = load_codes(m + i, left - i);
        rq[u][s] = load_codes(r + i, left - i);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int b = u * (THREADS / 16) + row;
    float mm[2][4], rr[2][4];
    uint32_t top_m = 0, top_r = 0;
#pragma unroll
    for (int s = 0; s < 2; s++) {
      values_of(mq[u][s], power(sc[u] & 255u), mm[s]);
      values_of(rq[u][s], power(sc[u] >> 8), rr[s]);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        adamw8_one(ww[u][s][j], gg[u][s][j] * scale, mm[s][j], rr[s][j], h);
        top_m = max(top_m, finite_bits(mm[s][j]));
        top_r = max(top_r, finite_bits(rr[s][j]));
      }
    }
    const int em = block_exponent(row_max(top_m)), er = block_exponent(row_max(top_r));
    const float inv_m = power(254 - em), inv_r = power(254 - er);
    if (at == 0 && b * QBLOCK < left) *(u16u *)(scales + 2 * b) = (uint16_t)(em | er << 8);
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const int i = b * QBLOCK + s * 64 + at;
      const uint32_t e = (uint32_t)base + (uint32_t)i;
      const uint32_t cm = codes_of<false>(mm[s], inv_m, e * PHASE_M + h.shift_m, PHASE_M);
      const uint32_t cr = codes_of<true>(rr[s], inv_r, e * PHASE_R + h.shift_r, PHASE_R);
      if (left == CHUNK) {
        store4(p + i, ww[u][s]);
        if constexpr (MASTER) store4(w + i, ww[u][s]);
        *(u32u *)(m + i) = cm;
        *(u32u *)(r + i) = cr;
      } else {
        store_some(p + i, ww[u][s], left - i);
        if constexpr (MASTER) store_some(w + i, ww[u][s], left - i);
        store_codes(m + i, cm, left - i);
        store_codes(r + i, cr, left - i);
      }
    }
  }
}

// ---- 8-bit moments to values and back ---------------------------------------------------------------------------------
struct MomentTable {
  uint8_t *mq[TENSORS], *rq[TENSORS], *scales[TENSORS];
  void *m[TENSORS], *v[TENSORS];
  int64_t n[TENSORS];
  uint32_t start[TENSORS];
  int count;
};
static_assert(sizeof(MomentTable) <= 4096, "kernel argument");

// v = r^2 of a four-bit code has eight significant bits: bf16 holds m and v exactly (within its range)
template <typename T> __global__ __launch_bounds__(THREADS) void moments_read_kernel(MomentTable t) {
  const int k = owner(t.start, t.count, blockIdx.x);
  const int64_t base = (int64_t)(blockIdx.x - t.start[k]) * CHUNK;
  const int left = (int)min(t.n[k] - base, (int64_t)CHUNK);
  const uint8_t *mq = t.mq[k] + base, *rq = t.rq[k] + base, *scales = t.scales[k] + 2 * (base / QBLOCK);
  T *m = (T *)t.m[k] + base, *v = (T *)t.v[k] + base;
  constexpr int U = CHUNK / (THREADS * 4);
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int i = (u * THREADS + threadIdx.x) * 4, have = left - i;
    if (have <= 0) continue;
    const uint32_t sc = *(const u16u *)(scales + 2 * (i / QBLOCK));
    float mm[4], rr[4];
    values_of(load_codes(mq + i, have), power(sc & 255u), mm);
    values_of(load_codes(rq + i, have), power(sc >> 8), rr);
#pragma unroll
    for (int j = 0; j < 4; j++) rr[j] = rr[j] * rr[j];
    if (have >= 4) {
      store4(m + i, mm); store4(v + i, rr);
    } else {
      store_some(m + i, mm, have); store_some(v + i, rr, have);
    }
  }
}

// values to codes, to nearest (the threshold is one half for every element)
__global__ __launch_bounds__(THREADS) void moments_write_kernel(MomentTable t) {
  const int k = owner(t.start, t.count, blockIdx.x);
  const int64_t base = (int64_t)(blockIdx.x - t.start[k]) * CHUNK;
  const int left = (int)min(t.n[k] - base, (int64_t)CHUNK);
  uint8_t *mq = t.mq[k] + base, *rq = t.rq[k] + base, *scales = t.scales[k] + 2 * (base / QBLOCK);
  const float *m = (const float *)t.m[k] + base, *v = (const float *)t.v[k] + base;
  const int row = threadIdx.x / 16, at = (threadIdx.x & 15) * 4;
  constexpr int U = CHUNK / (THREADS * 8);
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int b = u * (THREADS / 16) + row;
    float mm[2][4], rr[2][4];
    uint32_t top_m = 0, top_r = 0;
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const int i = b * QBLOCK + s * 64 + at;
      load_some(m + i, mm[s], left - i); load_some(v + i, rr[s], left - i);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        rr[s][j] = sqrtf(rr[s][j]);
        top_m = max(top_m, finite_bits(mm[s][j]));
        top_r = max(top_r, finite_bits(rr[s][j]));
      }
    }
    const int em = block_exponent(row_max(top_m)), er = block_exponent(row_max(top_r));
    if (at == 0 && b * QBLOCK < left) *(u16u *)(scales + 2 * b) = (uint16_t)(em | er << 8);
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const int i = b * QBLOCK + s * 64 + at;
      store_codes(mq + i, codes_of<false>(mm[s], power(254 - em), 0x80000000u, 0u), left - i);
      store_codes(rq + i, codes_of<true>(rr[s], power(254 - er), 0x80000000u, 0u), left - i);
    }
  }
}

// ---- scalars formed on the device (steps that a graph replays) ----------------------------------------------------------
struct ScalarTable {
  float *step[TENSORS];
  const float *lr_dev[TENSORS];
  double lr[TENSORS], b1[TENSORS], b2[TENSORS], eps[TENSORS], wd[TENSORS];
  Hyper *out;
  int count;
};
static_assert(sizeof(ScalarTable) <= 4096, "kernel argument");

__global__ __launch_bounds__(64) void adamw_scalars_kernel(ScalarTable t) {
  const int k = threadIdx.x;
  if (k >= t.count) return;
  const float step = *t.step[k] + 1.0f;
  *t.step[k] = step;
  t.out[k] = make_hyper(t.lr_dev[k] ? (double)*t.lr_dev[k] : t.lr[k], t.b1[k], t.b2[k], t.eps[k], t.wd[k], (double)step);
}

// ---- global norm --------------------------------------------------------------------------------------------------------
struct GradTable {
  void *g[TENSORS];
  int64_t n[TENSORS];
  uint32_t start[TENSORS + 1];  // first chunk
  uint8_t dtype[TENSORS];
  int count;
};
static_assert(sizeof(GradTable) <= 4096, "kernel argument");

template <typename T> __device__ __forceinline__ double chunk_squares(const T *g, int64_t left) {
  constexpr int U = CHUNK / (THREADS * 4);
  float x[U][4];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int i = (u * THREADS + threadIdx.x) * 4;
    if (left >= CHUNK) load4(g + i, x[u]);
    else load_some(g + i, x[u], (int)left - i);
  }
  double a = 0.0, b = 0.0;
#pragma unroll
  for (int u = 0; u < U; u++) {
    a = fma((double)x[u][0], (double)x[u][0], a); b = fma((double)x[u][1], (double)x[u][1], b);
    a = fma((double)x[u][2], (double)x[u][2], a); b = fma((double)x[u][3], (double)x[u][3], b);
  }
  return a + b;
}

__device__ __forceinline__ double group_sum(double a, double *lds) {  // valid in thread 0
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) a += __shfl_down(a, d, 64);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) lds[wave] = a;
  __syncthreads();
  double s = lds[0];
  for (int k = 1; k < THREADS / 64; k++) s += lds[k];
  return s;
}

// Squares are summed in 64 bits (no overflow, no loss over long sums), each workgroup over its own chunks in a fixed order:
// the same gradients give the same norm to the last bit.
__global__ __launch_bounds__(THREADS) void norm_partial_kernel(GradTable t, double *partial) {
  __shared__ double lds[THREADS / 64];
  double sum = 0.0;
  for (uint32_t c = blockIdx.x; c < t.start[t.count]; c += gridDim.x) {
    const int k = owner(t.start, t.count, c);
    const int64_t base = (int64_t)(c - t.start[k]) * CHUNK, left = t.n[k] - base;
    if (t.dtype[k] == FSGS_DTYPE_F32) sum += chunk_squares((const float *)t.g[k] + base, left);
    else if (t.dtype[k] == FSGS_DTYPE_BF16) sum += chunk_squares((const __bf16 *)t.g[k] + base, left);
    else sum += chunk_squares((const _Float16 *)t.g[k] + base, left);
  }
  const double s = group_sum(sum, lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(THREADS) void norm_finish_kernel(const double *partial, int count, float max_norm, float *out2) {
  __shared__ double lds[THREADS / 64];
  double sum = 0.0;
  for (int i = threadIdx.x; i < count; i += THREADS) sum += partial[i];
  const double s = group_sum(sum, lds);
  if (threadIdx.x == 0) {
    const float norm = (float)sqrt(s), c = max_norm / (norm + 1e-6f);
    out2[0] = norm;
    out2[1] = c > 1.0f ? 1.0f : c;  // NaN stays NaN
  }
}

template <typename T> __device__ __forceinline__ void chunk_scale(T *g, int64_t left, float c) {
  constexpr int U = CHUNK / (THREADS * 4);
  float x[U][4];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int i = (u * THREADS + threadIdx.x) * 4;
    if (left >= CHUNK) load4(g + i, x[u]);
    else load_some(g + i, x[u], (int)left - i);
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int i = (u * THREADS + threadIdx.x) * 4;
#pragma unroll
    for (int j = 0; j < 4; j++) x[u][j] *= c;
    if (left >= CHUNK) store4(g + i, x[u]);
    else store_some(g + i, x[u], (int)left - i);
  }
}

// a factor of exactly 1 leaves every gradient as it is: nothing is read or written then
__global__ __launch_bounds__(THREADS) void grad_scale_kernel(GradTable t, const float *coef) {
  const float c = *coef;
  if (c == 1.0f) return;
  const int k = owner(t.start, t.count, blockIdx.x);
  const int64_t base = (int64_t)(blockIdx.x - t.start[k]) * CHUNK, left = t.n[k] - base;
  if (t.dtype[k] == FSGS_DTYPE_F32) chunk_scale((float *)t.g[k] + base, left, c);
  else if (t.dtype[k] == FSGS_DTYPE_BF16) chunk_scale((__bf16 *)t.g[k] + base, left, c);
  else chunk_scale((_Float16 *)t.g[k] + base, left, c);
}

// ---- host -----------------------------------------------------------------------------------------------------------------
int size_of(int dtype) { return dtype == FSGS_DTYPE_F32 ? 4 : dtype == FSGS_DTYPE_BF16 || dtype == FSGS_DTYPE_F16 ? 2 : 0; }

// Two of the regions that a call writes share memory, or one that it writes shares memory with one that it reads: the
// kernels' workgroups would race.  Regions that are only read may be shared.
struct Regions {
  struct Item { uintptr_t lo, hi; bool write; };
  Item *items = nullptr;
  int count = 0;
  explicit Regions(size_t capacity) : items(new (std::nothrow) Item[capacity ? capacity : 1]) {}
  ~Regions() { delete[] items; }
  void add(const void *p, int64_t bytes, bool write) {
    if (p && bytes > 0) items[count++] = {(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes, write};
  }
  bool clash() {
    std::sort(items, items + count, [](const Item &a, const Item &b) { return a.lo < b.lo; });
    uintptr_t end = 0, end_written = 0;  // of what came before
    for (int i = 0; i < count; i++) {
      if (items[i].lo < (items[i].write ? end : end_written)) return true;
      end = std::max(end, items[i].hi);
      if (items[i].write) end_written = std::max(end_written, items[i].hi);
    }
    return false;
  }
};

int64_t chunks_of(int64_t n) { return (n + CHUNK - 1) / CHUNK; }
int64_t qblocks_of(int64_t n) { return (n + QBLOCK - 1) / QBLOCK; }

template <typename T, bool MASTER> void launch_step(const Table &t, uint32_t groups, int bits, hipStream_t stream) {
  if (bits == 32) hipLaunchKernelGGL((adamw32_kernel<T, MASTER>), dim3(groups), dim3(THREADS), 0, stream, t);
  else hipLaunchKernelGGL((adamw8_kernel<T, MASTER>), dim3(groups), dim3(THREADS), 0, stream, t);
}

}  // namespace

extern "C" {

size_t fsgs_adamw_scratch_bytes(int n_tensors) { return n_tensors > 0 ? (size_t)n_tensors * sizeof(Hyper) : 0; }

int fsgs_adamw_step(int n_tensors, const FsgsAdamWTensor *tensors, int n_hypers, const FsgsAdamWHyper *hypers, int dtype,
                    int state_bits, int maximize, const float *grad_coef, void *scratch, fsgs_stream_t stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  if (n_tensors < 0 || n_hypers < 0 || (n_tensors > 0 && (!tensors || !hypers)) || !size_of(dtype)) return FSGS_ERR_INVALID;
  if (state_bits != 8 && state_bits != 32) return FSGS_ERR_INVALID;
  const int esize = size_of(dtype);
  Regions regions((size_t)n_tensors * 7);
  if (!regions.items) return FSGS_ERR_CAPACITY;
  const bool on_device = n_tensors > 0 && tensors[0].hyper >= 0 && tensors[0].hyper < n_hypers && hypers[tensors[0].hyper].step_dev;
  int master = -1;  // not seen yet
  for (int i = 0; i < n_tensors; i++) {
    const FsgsAdamWTensor &x = tensors[i];
    if (x.n < 0 || x.hyper < 0 || x.hyper >= n_hypers) return FSGS_ERR_INVALID;
    const FsgsAdamWHyper &h = hypers[x.hyper];
    if (!(h.lr >= 0.0) || !(h.beta1 >= 0.0 && h.beta1 < 1.0) || !(h.beta2 >= 0.0 && h.beta2 < 1.0) || !(h.eps >= 0.0) ||
        !(h.weight_decay >= 0.0))
      return FSGS_ERR_INVALID;
    // either every tensor has its step on the device, or none
    if (on_device != (h.step_dev != nullptr) || (!on_device && h.step < 1)) return FSGS_ERR_INVALID;
    if (on_device) regions.add(h.step_dev, 4, true);  // each tensor counts its own steps
    if (x.n == 0) continue;
    if (!x.param || !x.grad || !x.exp_avg || !x.exp_avg_sq || (state_bits == 8 && !x.scales)) return FSGS_ERR_INVALID;
    if (chunks_of(x.n) > MAX_BLOCKS) return FSGS_ERR_INVALID;
    if (master < 0) master = x.master != nullptr;
    if (master != (x.master != nullptr) || (master && dtype == FSGS_DTYPE_F32)) return FSGS_ERR_INVALID;
    regions.add(x.param, x.n * esize, true);
    regions.add(x.grad, x.n * esize, false);
    regions.add(x.exp_avg, x.n * (state_bits / 8), true);
    regions.add(x.exp_avg_sq, x.n * (state_bits / 8), true);
    if (state_bits == 8) regions.add(x.scales, 2 * qblocks_of(x.n), true);
    regions.add(x.master, x.n * 4, true);
  }
  if (on_device && !scratch && n_tensors > 0) return FSGS_ERR_INVALID;
  if (regions.clash()) return FSGS_ERR_INVALID;
  ProfScope ps(PROF_ADAM, stream);
  Hyper *dev_h = on_device ? (Hyper *)scratch : nullptr;
  for (int i = 0; on_device && i < n_tensors; i += TENSORS) {
    ScalarTable s;
    std::memset(&s, 0, sizeof(s));
    s.count = std::min(TENSORS, n_tensors - i);
    s.out = dev_h + i;
    for (int k = 0; k < s.count; k++) {
      const FsgsAdamWHyper &h = hypers[tensors[i + k].hyper];
      s.step[k] = h.step_dev; s.lr_dev[k] = h.lr_dev;
      s.lr[k] = h.lr; s.b1[k] = h.beta1; s.b2[k] = h.beta2; s.eps[k] = h.eps; s.wd[k] = h.weight_decay;
    }
    hipLaunchKernelGGL(adamw_scalars_kernel, dim3(1), dim3(64), 0, stream, s);
    FSGS_HIP(hipGetLastError());
  }
  Table t;
  int i = 0;
  while (i < n_tensors) {
    std::memset(&t, 0, sizeof(t));
    t.coef = grad_coef;
    t.sign = maximize ? -1.0f : 1.0f;
    int64_t groups = 0;
    int used[HYPERS], n_used = 0;
    t.dev_h = dev_h ? dev_h + i : nullptr;
    for (; i < n_tensors && t.count < TENSORS; i++) {
      const FsgsAdamWTensor &x = tensors[i];
      // on the device the scalars' index is the tensor's, so an empty tensor keeps its place (and owns no workgroup)
      if (x.n == 0 && !dev_h) continue;
      if (groups + chunks_of(x.n) > MAX_BLOCKS) break;
      int at = 0;
      if (!dev_h) {
        while (at < n_used && used[at] != x.hyper && std::memcmp(&hypers[used[at]], &hypers[x.hyper], sizeof(FsgsAdamWHyper))) at++;
        if (at == n_used) {
          if (n_used == HYPERS) break;
          const FsgsAdamWHyper &h = hypers[x.hyper];
          used[n_used] = x.hyper;
          t.h[n_used++] = make_hyper(h.lr, h.beta1, h.beta2, h.eps, h.weight_decay, (double)h.step);
        }
      }
      const int k = t.count++;
      t.p[k] = x.param; t.g[k] = x.grad; t.m[k] = x.exp_avg; t.v[k] = x.exp_avg_sq; t.w[k] = x.master;
      t.scales[k] = x.scales; t.n[k] = x.n; t.start[k] = (uint32_t)groups; t.hyper[k] = (uint8_t)at;
      groups += chunks_of(x.n);
    }
    if (groups == 0) continue;
    if (dtype == FSGS_DTYPE_F32) launch_step<float, false>(t, (uint32_t)groups, state_bits, stream);
    else if (dtype == FSGS_DTYPE_BF16 && master > 0) launch_step<__bf16, true>(t, (uint32_t)groups, state_bits, stream);
    else if (dtype == FSGS_DTYPE_BF16) launch_step<__bf16, false>(t, (uint32_t)groups, state_bits, stream);
    else if (master > 0) launch_step<_Float16, true>(t, (uint32_t)groups, state_bits, stream);
    else launch_step<_Float16, false>(t, (uint32_t)groups, state_bits, stream);
    FSGS_HIP(hipGetLastError());
  }
  return FSGS_OK;
}

int fsgs_adamw_moments(int n_tensors, const FsgsAdamWMoments *tensors, int write, int dtype, fsgs_stream_t stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  if (n_tensors < 0 || (n_tensors > 0 && !tensors) || !size_of(dtype) || (write && dtype != FSGS_DTYPE_F32))
    return FSGS_ERR_INVALID;
  Regions regions((size_t)n_tensors * 5);
  if (!regions.items) return FSGS_ERR_CAPACITY;
  for (int i = 0; i < n_tensors; i++) {
    const FsgsAdamWMoments &x = tensors[i];
    if (x.n < 0 || chunks_of(x.n) > MAX_BLOCKS) return FSGS_ERR_INVALID;
    if (x.n == 0) continue;
    if (!x.exp_avg_q || !x.exp_avg_sq_q || !x.scales || !x.exp_avg || !x.exp_avg_sq) return FSGS_ERR_INVALID;
    regions.add(x.exp_avg_q, x.n, write != 0);
    regions.add(x.exp_avg_sq_q, x.n, write != 0);
    regions.add(x.scales, 2 * qblocks_of(x.n), write != 0);
    regions.add(x.exp_avg, x.n * size_of(dtype), write == 0);
    regions.add(x.exp_avg_sq, x.n * size_of(dtype), write == 0);
  }
  if (regions.clash()) return FSGS_ERR_INVALID;
  MomentTable t;
  int i = 0;
  while (i < n_tensors) {
    std::memset(&t, 0, sizeof(t));
    int64_t groups = 0;
    for (; i < n_tensors && t.count < TENSORS; i++) {
      const FsgsAdamWMoments &x = tensors[i];
      if (x.n == 0) continue;
      if (groups + chunks_of(x.n) > MAX_BLOCKS) break;
      const int k = t.count++;
      t.mq[k] = x.exp_avg_q; t.rq[k] = x.exp_avg_sq_q; t.scales[k] = x.scales; t.m[k] = x.exp_avg; t.v[k] = x.exp_avg_sq;
      t.n[k] = x.n; t.start[k] = (uint32_t)groups;
      groups += chunks_of(x.n);
    }
    if (groups == 0) continue;
    const dim3 grid((uint32_t)groups);
    if (write) hipLaunchKernelGGL(moments_write_kernel, grid, dim3(THREADS), 0, stream, t);
    else if (dtype == FSGS_DTYPE_F32) hipLaunchKernelGGL(moments_read_kernel<float>, grid, dim3(THREADS), 0, stream, t);
    else if (dtype == FSGS_DTYPE_BF16) hipLaunchKernelGGL(moments_read_kernel<__bf16>, grid, dim3(THREADS), 0, stream, t);
    else hipLaunchKernelGGL(moments_read_kernel<_Float16>, grid, dim3(THREADS), 0, stream, t);
    FSGS_HIP(hipGetLastError());
  }
  return FSGS_OK;
}

size_t fsgs_grad_norm_scratch_bytes(int n_tensors) {
  // a launch takes 48 tensors, or fewer where they hold over 2^35 elements: no card holds 16 times that
  return n_tensors > 0 ? (size_t)((n_tensors + TENSORS - 1) / TENSORS + 16) * NORM_GROUPS * sizeof(double) : 0;
}

static int check_grads(int n_tensors, const FsgsGradTensor *grads, bool write) {
  if (n_tensors < 0 || (n_tensors > 0 && !grads)) return FSGS_ERR_INVALID;
  Regions regions((size_t)n_tensors);
  if (!regions.items) return FSGS_ERR_CAPACITY;
  for (int i = 0; i < n_tensors; i++) {
    if (grads[i].n < 0 || !size_of(grads[i].dtype) || (grads[i].n > 0 && !grads[i].grad)) return FSGS_ERR_INVALID;
    if (chunks_of(grads[i].n) > MAX_BLOCKS) return FSGS_ERR_INVALID;
    regions.add(grads[i].grad, grads[i].n * size_of(grads[i].dtype), write);
  }
  return regions.clash() ? FSGS_ERR_INVALID : FSGS_OK;
}

// the next up to 48 tensors from `from` on that hold at most MAX_BLOCKS chunks; returns the first that is left
static int fill_grads(GradTable &t, int from, int n_tensors, const FsgsGradTensor *grads) {
  std::memset(&t, 0, sizeof(t));
  int64_t chunks = 0;
  int i = from;
  for (; i < n_tensors && i - from < TENSORS; i++) {
    if (grads[i].n == 0) continue;
    if (chunks + chunks_of(grads[i].n) > MAX_BLOCKS) break;
    const int k = t.count++;
    t.g[k] = grads[i].grad; t.n[k] = grads[i].n; t.dtype[k] = (uint8_t)grads[i].dtype; t.start[k] = (uint32_t)chunks;
    chunks += chunks_of(grads[i].n);
  }
  t.start[t.count] = (uint32_t)chunks;
  return i;
}

int fsgs_grad_norm(int n_tensors, const FsgsGradTensor *grads, float max_norm, void *scratch, size_t scratch_bytes,
                   float *out2, fsgs_stream_t stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  if (int rc = check_grads(n_tensors, grads, false)) return rc;
  if (!out2 || !(max_norm >= 0.0f) || (n_tensors > 0 && !scratch)) return FSGS_ERR_INVALID;
  double *partial = (double *)scratch;
  size_t count = 0;
  GradTable t;
  for (int i = 0; i < n_tensors;) {
    i = fill_grads(t, i, n_tensors, grads);
    if (t.count == 0) continue;
    const uint32_t groups = std::min<uint32_t>(t.start[t.count], NORM_GROUPS);
    if ((count + groups) * sizeof(double) > scratch_bytes) return FSGS_ERR_CAPACITY;
    hipLaunchKernelGGL(norm_partial_kernel, dim3(groups), dim3(THREADS), 0, stream, t, partial + count);
    FSGS_HIP(hipGetLastError());
    count += groups;
  }
  hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(THREADS), 0, stream, partial, (int)count, max_norm, out2);
  FSGS_HIP(hipGetLastError());
  return FSGS_OK;
}

int fsgs_grad_scale(int n_tensors, const FsgsGradTensor *grads, const float *coef, fsgs_stream_t stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  if (int rc = check_grads(n_tensors, grads, true)) return rc;
  if (n_tensors > 0 && !coef) return FSGS_ERR_INVALID;
  GradTable t;
  for (int i = 0; i < n_tensors;) {
    i = fill_grads(t, i, n_tensors, grads);
    if (t.count == 0) continue;
    hipLaunchKernelGGL(grad_scale_kernel, dim3(t.start[t.count]), dim3(THREADS), 0, stream, t, coef);
    FSGS_HIP(hipGetLastError());
  }
  return FSGS_OK;
}

}  // extern "C"
