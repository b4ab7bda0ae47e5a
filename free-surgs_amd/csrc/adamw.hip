// adamw.hip -- AdamW over many tensors at once (moments in 32 or in 8 bits) and the gradients' global norm, for gfx950 (MI355X).
//
//   g' = c g                                          c: the bound on the global norm, or 1
//   m  = b1 m + (1 - b1) g',   v = b2 v + (1 - b2) g'^2
//   w  = w (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// A few dozen operations an element against 16 to 30 bytes: everything here is bound by HBM, so each kernel reads and writes
// every array once, with 16-byte accesses where the type allows, and one launch takes up to 48 tensors (192 gradients).
// The step's loads and stores are non-temporal, what they move is next used a whole step later: 1 M Gaussians (59 M floats)
// 311 -> 280 us (5.9 TB/s) with 32-bit moments, 176 -> 155 us (6.1 TB/s) with 8-bit ones (both sides in one run; 150 to 160
// us over runs and cards); on the loads or on the stores
// alone there is next to nothing to gain (302 and 313 us).  The norm's and the scaling's are not: gradients come from a
// cache as often as not (20 M bf16: 15.6 us against 17.7).
//
// Which tensor a workgroup belongs to: lane k of every wave compares the workgroup's number with the first workgroup of
// tensor k, and the number of lanes at or past theirs is the answer -- one load and one ballot, no search.
//
// Moments in 8 bits: 128 consecutive elements of a tensor share one power of two for m and one for r = sqrt(v).  The codes are
// OCP e4m3 of m / 2^E and r / 2^E with the smallest E that brings the block's largest finite value to at most 448, stored as
// E + 127 in a byte.  r rather than v, because r needs half the exponent range.  A value between two codes goes up when its
// remainder reaches over the threshold of its element at this step: 20 bits of a quasi-random sequence, a Weyl sequence over
// the elements (golden ratio, sqrt 2) that each step moves on by the plastic number's inverse (m) or its square (r).  A moment
// that moves by less than a code a step so still moves: with b2 = 0.999, r moves by 5e-4 a step and half a code is 3e-2 to
// 6e-2, so that rounding to nearest would hold it for good.  How well it follows moments in 32 bits (20 000 elements, b2 =
// 0.999; ratio of r: mean and deviation; of v: mean): Gaussian gradients, steps 1500 to 4000: 1.007, 0.12; 1.03.  Gradients
// in one step of twenty: 0.996, 0.13; 1.01.  1500 steps without any: 0.951, 0.07; 0.91 -- too low, because a code is left
// after the mean waiting time, and 1/9 + ... + 1/16 < ln 2.  Thresholds that are independent from step to step keep r's mean
// there (0.997) but spread three times as far (0.25), and farther than these with gradients too (0.14 and 0.18; v 1.04 and
// 1.06).  r > 0 keeps at least the smallest code, so that m is never divided by a denominator that the rounding took away.
// The step itself uses m and r before the rounding.
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
constexpr int GRADS = 192;             // of one norm or scaling launch
constexpr int HYPERS = 8;              // different sets of scalars of one launch
constexpr int THREADS = 256;
// Elements of one workgroup of a step: two vectors a thread and array.  Four make fewer, larger workgroups (20 k Gaussians,
// 1.2 M floats: 10.1 us against 8.1; 24 bf16 layers of 20 M in 8 bits: 59 us against 54; no difference at 59 M).
constexpr int CHUNK = 2048;
// Bytes of one workgroup's turn in the norm, four 16-byte vectors a thread; the scaling's workgroups take half of one.  Inside a
// clip, two / four / eight vectors: 160 bf16 layers of 64 M: norm 33.6 / 34.2 / 36.3 us; 17.7 M floats 13.6 / 13.0 / 12.6.
// Scaling with one / two / four: 40.8 / 37.2 / 37.6 and 20.7 / 20.9 / 20.3.
constexpr int NORM_BYTES = 16384, SCALE_BYTES = NORM_BYTES / 2;
constexpr int XCDS = 8;  // workgroup b of a launch runs on XCD b % 8, which has an L2 of its own
constexpr int64_t MAX_BLOCKS = (1 << 24) - 1;  // workgroups of one launch (256 threads each: under 2^32 work items)
constexpr int64_t MAX_ELEMENTS = MAX_BLOCKS * CHUNK;  // of one tensor, compared before anything is added to them
constexpr int64_t MAX_TURNS = MAX_BLOCKS / 2 - 8;        // two workgroups of the scaling each, and what fills the last row
constexpr int QBLOCK = FSGS_ADAMW_BLOCK;  // elements that share a power of two
constexpr int NORM_GROUPS = 2048;      // workgroups of one norm launch at most: eight per CU
constexpr int SUMMED = THREADS;        // partial sums that a step or a scaling adds up by itself

// what a step's scalars come to; one per tensor where they are formed on the device
struct Hyper {
  float decay;          // 1 - lr wd
  float step_size;      // lr / (1 - b1^t)
  float inv_bc2_sqrt;   // 1 / sqrt(1 - b2^t)
  float eps;
  float b1, omb1, b2, omb2;
  uint32_t shift_m, shift_r;  // the step's part of the rounding thresholds
};
// 2^32 times the fractions of the golden ratio and of sqrt 2; 2^32 / plastic number (rho^3 = rho + 1), 2^32 / its square
constexpr uint32_t PHASE_M = 0x9E3779B9u, PHASE_R = 0x6A09E667u, TURN_M = 0xC13FA9A9u, TURN_R = 0x91E10DA5u;

__host__ __device__ inline Hyper make_hyper(double lr, double b1, double b2, double eps, double wd, double step) {
  Hyper h;
  h.decay = (float)(1.0 - lr * wd);
  h.step_size = (float)(lr / (1.0 - pow(b1, step)));
  h.inv_bc2_sqrt = (float)(1.0 / sqrt(1.0 - pow(b2, step)));
  h.eps = (float)eps;
  // 1 - beta in double: 1 - 0.999f is off by 4.7e-5 of itself
  h.b1 = (float)b1; h.omb1 = (float)(1.0 - b1); h.b2 = (float)b2; h.omb2 = (float)(1.0 - b2);
  const uint32_t t = (uint32_t)(int64_t)step;
  h.shift_m = t * TURN_M; h.shift_r = t * TURN_R;
  return h;
}

template <int WAVES> __device__ __forceinline__ double group_sum(double a, double *lds) {  // the same in every thread
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) a += __shfl_xor(a, d, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
  __syncthreads();
  double s = lds[0];
#pragma unroll
  for (int k = 1; k < WAVES; k++) s += lds[k];
  return s;
}

// The factor on the gradients: one that another launch has left, or formed here from up to SUMMED partial sums of the squares.
// A launch costs the host 4 us and the GPU 2 to 3; a small step's or scaling's workgroups rather add the sums themselves, one a
// thread, 2 KB from the cache each: clipping 40 tensors of 0.3 M floats 17.6 -> 14.5 us, and at the border (1 M floats, 245
// sums) 12.2 us against 13.9 back to back.  More sums than threads are left to the launch; other borders have not been measured.
struct Bound {
  const double *partial;
  const float *factor;
  float *norm;
  int count;  // of partial; 0: *factor, or 1 where that is NULL
  float max_norm;
};
__device__ __forceinline__ float factor_of(double squares, float max_norm, float *norm) {
  const float x = (float)sqrt(squares), c = max_norm / (x + 1e-6f);
  if (norm) *norm = x;
  return c > 1.0f ? 1.0f : c;  // NaN stays NaN
}
__device__ __forceinline__ float factor_of(const Bound &b) {
  if (b.count == 0) return b.factor ? *b.factor : 1.0f;
  __shared__ double lds[THREADS / 64];
  const double s = group_sum<THREADS / 64>((int)threadIdx.x < b.count ? b.partial[threadIdx.x] : 0.0, lds);
  return factor_of(s, b.max_norm, blockIdx.x == 0 && threadIdx.x == 0 ? b.norm : nullptr);
}

// a tensor's entry is one aligned 64 bytes: arguments are read from the host's memory the first time, line by line
struct Entry {
  void *p;
  const void *g;
  void *m, *v;
  void *w;          // fp32 master weights
  uint8_t *scales;
  int64_t n;
  uint32_t start;   // first workgroup (as in Table::start)
  uint32_t hyper;
};
struct Table {
  uint32_t start[TENSORS];
  int count;
  float sign;               // -1: ascend
  const Hyper *dev_h;       // one per tensor, or NULL: h[hyper]
  Bound bound;
  Hyper h[HYPERS];
  alignas(64) Entry at[TENSORS];
};
static_assert(sizeof(Table) <= 4096 && sizeof(Entry) == 64, "kernel argument");

template <int MAX> __device__ __forceinline__ int owner(const uint32_t *start, int count, uint32_t group) {
  const int lane = threadIdx.x & 63;
  int k = -1;
#pragma unroll
  for (int first = 0; first < MAX; first += 64) {
    if (first > 0 && count <= first) break;
    const int at = first + lane;
    k += __popcll(__ballot(at < count && group >= start[at < MAX ? at : MAX - 1]));
  }
  return __builtin_amdgcn_readfirstlane(k);
}
__device__ __forceinline__ Hyper hyper_of(const Table &t, int k) {
  if (t.dev_h) return t.dev_h[k];
  return t.h[t.at[k].hyper];
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

template <bool STREAM, typename T> __device__ __forceinline__ void load4(const T *at, float (&x)[4]) {
  typename Vec4<T>::type a;
  if constexpr (STREAM) a = __builtin_nontemporal_load((const typename Vec4<T>::type *)at);
  else a = *(const typename Vec4<T>::type *)at;
#pragma unroll
  for (int j = 0; j < 4; j++) x[j] = (float)a[j];
}
template <bool STREAM, typename T> __device__ __forceinline__ void store4(T *at, const float (&x)[4]) {
  typename Vec4<T>::type a;
#pragma unroll
  for (int j = 0; j < 4; j++) a[j] = (T)x[j];  // one rounding to the parameter's type, to nearest even
  if constexpr (STREAM) __builtin_nontemporal_store(a, (typename Vec4<T>::type *)at);
  else *(typename Vec4<T>::type *)at = a;
}
// the first `have` of four elements: a tensor's last workgroup
template <typename T> __device__ __forceinline__ void load_some(const T *at, float (&x)[4], int have) {
  if (have >= 4) return load4<false>(at, x);
#pragma unroll
  for (int j = 0; j < 4; j++) x[j] = j < have ? (float)at[j] : 0.0f;
}
template <typename T> __device__ __forceinline__ void store_some(T *at, const float (&x)[4], int have) {
  if (have >= 4) return store4<false>(at, x);
#pragma unroll
  for (int j = 0; j < 3; j++)
    if (j < have) at[j] = (T)x[j];
}

// ---- moments in 32 bits ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void adamw_one(float &w, float g, float &m, float &v, const Hyper &h) {
  m = fmaf(h.b1, m, h.omb1 * g);
  v = fmaf(h.b2, v, h.omb2 * (g * g));
  w = fmaf(w, h.decay, -h.step_size * (m / fmaf(sqrtf(v), h.inv_bc2_sqrt, h.eps)));
}

// Bound by HBM: 1 M Gaussians (59 M floats) 279 us = 5.9 TB/s, where a 1 GiB copy reaches 5.0 and a 256 MiB one 5.4; the
// counters say 944 MB read and 708 MB written, i.e. every array once.  160 bf16 tensors of 64 M elements with masters: 314 us
// in four launches = 5.7 TB/s.  20 k Gaussians: 8 us, mostly the launch and the first reads of the arguments.  All loads of a
// workgroup are issued before the first is used; workgroups of 128 or 512 threads, one or four vectors a thread and a
// contiguous share of the tensors for each XCD are all within 2 % at 59 M or slower (284 to 303 us).
template <typename T, bool MASTER> __global__ __launch_bounds__(THREADS) void adamw32_kernel(Table t) {
  const int k = owner<TENSORS>(t.start, t.count, blockIdx.x);
  const Entry &e = t.at[k];
  const Hyper h = hyper_of(t, k);
  const int64_t base = (int64_t)(blockIdx.x - e.start) * CHUNK;
  const int64_t left = e.n - base;
  T *p = (T *)e.p + base;
  const T *g = (const T *)e.g + base;
  float *m = (float *)e.m + base, *v = (float *)e.v + base, *w = MASTER ? (float *)e.w + base : nullptr;
  constexpr int U = CHUNK / (THREADS * 4);
  float ww[U][4], gg[U][4], mm[U][4], vv[U][4];
  if (left >= CHUNK) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = (u * THREADS + threadIdx.x) * 4;
      load4<false>(g + i, gg[u]); load4<true>(m + i, mm[u]); load4<true>(v + i, vv[u]);
      if constexpr (MASTER) load4<true>(w + i, ww[u]); else load4<true>(p + i, ww[u]);
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = (u * THREADS + threadIdx.x) * 4, have = (int)left - i;
      load_some(g + i, gg[u], have); load_some(m + i, mm[u], have); load_some(v + i, vv[u], have);
      if constexpr (MASTER) load_some(w + i, ww[u], have); else load_some(p + i, ww[u], have);
    }
  }
  const float scale = t.sign * factor_of(t.bound);  // behind the loads: it may have to wait
#pragma unroll
  for (int u = 0; u < U; u++)
#pragma unroll
    for (int j = 0; j < 4; j++) adamw_one(ww[u][j], gg[u][j] * scale, mm[u][j], vv[u][j], h);
  if (left >= CHUNK) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i = (u * THREADS + threadIdx.x) * 4;
      store4<true>(p + i, ww[u]); store4<true>(m + i, mm[u]); store4<true>(v + i, vv[u]);
      if constexpr (MASTER) store4<true>(w + i, ww[u]);
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

// 16.03 bytes an element in fp32: 1 M Gaussians 157 us = 6.0 TB/s (354 MB written, 590 MB read; 150 to 160 us over runs and
// cards), 24 bf16 tensors of 20 M with masters 54 us.  It runs 88 vector instructions an element, half of what the SIMDs could issue in that time: approximate roots
// and quotients (a fifth fewer) change nothing, so the exact ones stay.  The codes' four-byte accesses are plain: made
// non-temporal they cost 5 % (165 us), the 64 bytes of a half block being too little for a line.
template <typename T, bool MASTER> __global__ __launch_bounds__(THREADS) void adamw8_kernel(Table t) {
  const int k = owner<TENSORS>(t.start, t.count, blockIdx.x);
  const Entry &e = t.at[k];
  const Hyper h = hyper_of(t, k);
  const int64_t base = (int64_t)(blockIdx.x - e.start) * CHUNK;
  const int left = (int)min(e.n - base, (int64_t)CHUNK);
  T *p = (T *)e.p + base;
  const T *g = (const T *)e.g + base;
  uint8_t *m = (uint8_t *)e.m + base, *r = (uint8_t *)e.v + base, *scales = e.scales + 2 * (base / QBLOCK);
  float *w = MASTER ? (float *)e.w + base : nullptr;
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
        load4<false>(g + i, gg[u][s]);
        if constexpr (MASTER) load4<true>(w + i, ww[u][s]); else load4<true>(p + i, ww[u][s]);
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
  const float scale = t.sign * factor_of(t.bound);
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
      const uint32_t place = (uint32_t)base + (uint32_t)i;
      const uint32_t cm = codes_of<false>(mm[s], inv_m, place * PHASE_M + h.shift_m, PHASE_M);
      const uint32_t cr = codes_of<true>(rr[s], inv_r, place * PHASE_R + h.shift_r, PHASE_R);
      if (left == CHUNK) {
        store4<true>(p + i, ww[u][s]);
        if constexpr (MASTER) store4<true>(w + i, ww[u][s]);
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

// 2 bytes in and 4 out for bf16: 1 M Gaussians 57 us = 6.2 TB/s.
// v = r^2 of a four-bit code has eight significant bits: bf16 holds m and v exactly (within its range)
template <typename T> __global__ __launch_bounds__(THREADS) void moments_read_kernel(MomentTable t) {
  const int k = owner<TENSORS>(t.start, t.count, blockIdx.x);
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
      store4<true>(m + i, mm); store4<true>(v + i, rr);
    } else {
      store_some(m + i, mm, have); store_some(v + i, rr, have);
    }
  }
}

// values to codes, to nearest (the threshold is one half for every element)
__global__ __launch_bounds__(THREADS) void moments_write_kernel(MomentTable t) {
  const int k = owner<TENSORS>(t.start, t.count, blockIdx.x);
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
  uint32_t start[GRADS];  // first turn
  uint32_t turns;
  int count;
  struct { void *g; int64_t n_dtype; } at[GRADS];  // n << 2 | dtype
};
static_assert(sizeof(GradTable) <= 4096, "kernel argument");

// two bytes an element: eight of them make 16 bytes
typedef __bf16 bf8u __attribute__((ext_vector_type(8), aligned(2)));
typedef _Float16 half8u __attribute__((ext_vector_type(8), aligned(2)));
typedef float float4r __attribute__((ext_vector_type(4)));
typedef __bf16 bf8r __attribute__((ext_vector_type(8)));
typedef _Float16 half8r __attribute__((ext_vector_type(8)));
template <typename T> struct Vec16;  // in memory, in registers
template <> struct Vec16<float> { typedef float4u mem; typedef float4r reg; };
template <> struct Vec16<__bf16> { typedef bf8u mem; typedef bf8r reg; };
template <> struct Vec16<_Float16> { typedef half8u mem; typedef half8r reg; };

// one turn of a workgroup: F(vector) of up to BYTES of a tensor that has `left` bytes from `g` on, stored again with WRITE
template <typename T, int BYTES, bool WRITE, typename F> __device__ __forceinline__ void turn(T *g, int64_t left, F f) {
  typedef typename Vec16<T>::mem M;
  typedef typename Vec16<T>::reg V;
  constexpr int L = 16 / sizeof(T), U = BYTES / (THREADS * 16);
  V x[U];
  if (left >= BYTES) {
#pragma unroll
    for (int u = 0; u < U; u++) x[u] = *(const M *)(g + (u * THREADS + threadIdx.x) * L);
#pragma unroll
    for (int u = 0; u < U; u++) {
      f(x[u]);
      if constexpr (WRITE) *(M *)(g + (u * THREADS + threadIdx.x) * L) = x[u];
    }
    return;
  }
  const int n = (int)(left / (int)sizeof(T));
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int i = (u * THREADS + threadIdx.x) * L;
    x[u] = V{};
    if (i + L <= n) x[u] = *(const M *)(g + i);
    else
#pragma unroll
      for (int j = 0; j < L; j++)
        if (i + j < n) x[u][j] = g[i + j];
    f(x[u]);
    if constexpr (WRITE) {
      if (i + L <= n) *(M *)(g + i) = x[u];
      else
#pragma unroll
        for (int j = 0; j < L; j++)
          if (i + j < n) g[i + j] = x[u][j];
    }
  }
}
__host__ __device__ inline uint32_t scale_rows(uint32_t turns) { return (turns + XCDS - 1) / XCDS; }

// BYTES from `skip` on of turn `at`
template <int BYTES, bool WRITE, typename F>
__device__ __forceinline__ void turn_of(const GradTable &t, uint32_t at, int skip, F f) {
  const int k = owner<GRADS>(t.start, t.count, at);
  const int64_t nd = t.at[k].n_dtype, n = nd >> 2, done = (int64_t)(at - t.start[k]) * NORM_BYTES + skip;
  char *g = (char *)t.at[k].g + done;
  if ((nd & 3) == FSGS_DTYPE_F32) turn<float, BYTES, WRITE>((float *)g, 4 * n - done, f);
  else if ((nd & 3) == FSGS_DTYPE_BF16) turn<__bf16, BYTES, WRITE>((__bf16 *)g, 2 * n - done, f);
  else turn<_Float16, BYTES, WRITE>((_Float16 *)g, 2 * n - done, f);
}

struct Squares {
  double a = 0.0, b = 0.0;
  template <typename V> __device__ __forceinline__ void operator()(const V &x) {
    constexpr int L = sizeof(V) / sizeof(x[0]);
#pragma unroll
    for (int j = 0; j < L; j += 2) {
      const double p = (double)(float)x[j], q = (double)(float)x[j + 1];
      a = fma(p, p, a);
      b = fma(q, q, b);
    }
  }
};

// Squares are summed in 64 bits (no overflow, no loss over long sums), each workgroup over its own turns in a fixed order:
// the same gradients give the same norm to the last bit.  17.7 M floats 13 us, 64 M bf16 in 160 tensors 34 us behind a scaling
// whose lines are still being written back, and 2 to 5 us for the second launch, which adds up to 2048 partial sums (1024 workgroups are slower at 64 M, 4096 at 17.7 M).
// Held to 64 registers (eight waves a SIMD): the compiler's own choice, 128, takes 10 % longer.
__global__ __launch_bounds__(THREADS, 8) void norm_partial_kernel(GradTable t, double *partial) {
  __shared__ double lds[THREADS / 64];
  Squares sum;
  for (uint32_t at = blockIdx.x; at < t.turns; at += gridDim.x)
    turn_of<NORM_BYTES, false>(t, at, 0, [&](const auto &x) { sum(x); });
  const double s = group_sum<THREADS / 64>(sum.a + sum.b, lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(1024) void norm_finish_kernel(const double *partial, int count, float max_norm, float *norm_out,
                                                              float *factor) {
  __shared__ double lds[16];
  double sum = 0.0;
  for (int i = threadIdx.x; i < count; i += 1024) sum += partial[i];
  const double s = group_sum<16>(sum, lds);
  if (threadIdx.x == 0) {
    *factor = factor_of(s, max_norm, norm_out);
  }
}

// The turns that the norm read last come first, each on the XCD that read it, whose L2 may still hold it: clipping 5.9 M floats
// 20.0 -> 16.5 us, 17.7 M 37.3 -> 35.6 (the scaling 21 us, 6.7 TB/s), 20 M bf16 25.2 -> 23.4, 64 M bf16 77 -> 75 (on another
// card 73 -> 71), 59 M floats as before; in the reverse order on any XCD, or on the same XCD in the norm's order, only the smallest gains.
// Non-temporal loads and stores would make it faster by itself where the gradients outgrow the 256 MB cache (norm and scaling of
// 59 M floats 134 -> 111 us), but the step that follows then reads them from HBM: both together 380 -> 394 us, 111 -> 115 at
// 17.7 M.
// A factor of exactly 1 leaves every gradient as it is: nothing is read or written then.
__global__ __launch_bounds__(THREADS) void grad_scale_kernel(GradTable t, Bound bound) {
  const float c = factor_of(bound);
  if (c == 1.0f) return;
  const uint32_t row = scale_rows(t.turns) - 1 - blockIdx.x / (2 * XCDS), half = blockIdx.x / XCDS % 2;
  const uint32_t at = row * XCDS + blockIdx.x % XCDS;
  if (at >= t.turns) return;
  turn_of<SCALE_BYTES, true>(t, at, half * SCALE_BYTES, [&](auto &x) {
#pragma unroll
    for (int j = 0; j < (int)(sizeof(x) / sizeof(x[0])); j++) x[j] = (decltype(x[j] + x[j]))((float)x[j] * c);
  });
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

int64_t turns_of(const FsgsGradTensor &g) { return (g.n * size_of(g.dtype) + NORM_BYTES - 1) / NORM_BYTES; }

// the next up to 192 gradients (of(i)) from `from` on that make at most MAX_TURNS turns; returns the first that is left
template <typename Of> int fill_grads(GradTable &t, int from, int n_tensors, Of of) {
  std::memset(&t, 0, sizeof(t));
  int64_t turns = 0;
  int i = from;
  for (; i < n_tensors && t.count < GRADS; i++) {
    const FsgsGradTensor g = of(i);
    if (g.n == 0) continue;
    if (turns + turns_of(g) > MAX_TURNS) break;
    const int k = t.count++;
    t.at[k] = {g.grad, g.n << 2 | g.dtype};
    t.start[k] = (uint32_t)turns;
    turns += turns_of(g);
  }
  t.turns = (uint32_t)turns;
  return i;
}

// Partial sums of the squares, and what the next launch makes of them: `own` lets it add up to SUMMED by itself, otherwise, and
// with more or none, norm and factor are formed here.
template <typename Of> int launch_norm(int n_tensors, Of of, float max_norm, void *scratch, size_t scratch_bytes, float *norm,
                                       float *factor, bool own, Bound *bound, hipStream_t stream) {
  double *partial = (double *)scratch;
  size_t count = 0;
  GradTable t;
  for (int i = 0; i < n_tensors;) {
    i = fill_grads(t, i, n_tensors, of);
    if (t.count == 0) continue;
    const uint32_t groups = std::min<uint32_t>(t.turns, NORM_GROUPS);
    if ((count + groups) * sizeof(double) > scratch_bytes) return FSGS_ERR_CAPACITY;
    hipLaunchKernelGGL(norm_partial_kernel, dim3(groups), dim3(THREADS), 0, stream, t, partial + count);
    FSGS_HIP(hipGetLastError());
    count += groups;
  }
  if (own && count > 0 && count <= SUMMED) {
    *bound = {partial, nullptr, norm, (int)count, max_norm};
    return FSGS_OK;
  }
  hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(1024), 0, stream, partial, (int)count, max_norm, norm, factor);
  FSGS_HIP(hipGetLastError());
  *bound = {nullptr, factor, nullptr, 0, max_norm};
  return FSGS_OK;
}

template <typename Of> int launch_scale(int n_tensors, Of of, const Bound &bound, hipStream_t stream) {
  GradTable t;
  for (int i = 0; i < n_tensors;) {
    i = fill_grads(t, i, n_tensors, of);
    if (t.count == 0) continue;
    hipLaunchKernelGGL(grad_scale_kernel, dim3(scale_rows(t.turns) * XCDS * 2), dim3(THREADS), 0, stream, t, bound);
    FSGS_HIP(hipGetLastError());
  }
  return FSGS_OK;
}

template <typename T, bool MASTER> void launch_step(const Table &t, uint32_t groups, int bits, hipStream_t stream) {
  if (bits == 32) hipLaunchKernelGGL((adamw32_kernel<T, MASTER>), dim3(groups), dim3(THREADS), 0, stream, t);
  else hipLaunchKernelGGL((adamw8_kernel<T, MASTER>), dim3(groups), dim3(THREADS), 0, stream, t);
}

}  // namespace

extern "C" {

size_t fsgs_grad_norm_scratch_bytes(int n_tensors) {
  // a launch takes 192 tensors, or fewer where they hold over 2^37 bytes: no card holds that 8 times
  return n_tensors > 0 ? (size_t)((n_tensors + GRADS - 1) / GRADS + 8) * NORM_GROUPS * sizeof(double) : 0;
}

size_t fsgs_adamw_scratch_bytes(int n_tensors) { return n_tensors > 0 ? (size_t)n_tensors * sizeof(Hyper) : 0; }

int fsgs_adamw_step(int n_tensors, const FsgsAdamWTensor *tensors, int n_hypers, const FsgsAdamWHyper *hypers, int dtype,
                    int state_bits, int maximize, const float *grad_factor, float max_norm, float *norm, void *norm_scratch,
                    size_t norm_scratch_bytes, void *scratch, fsgs_stream_t stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  if (n_tensors < 0 || n_hypers < 0 || (n_tensors > 0 && (!tensors || !hypers)) || !size_of(dtype)) return FSGS_ERR_INVALID;
  if (state_bits != 8 && state_bits != 32) return FSGS_ERR_INVALID;
  if (norm && (grad_factor || !(max_norm >= 0.0f) || !norm_scratch || norm_scratch_bytes < 16)) return FSGS_ERR_INVALID;
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
    if (x.n > MAX_ELEMENTS) return FSGS_ERR_INVALID;
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
  Bound bound = {nullptr, grad_factor, nullptr, 0, 0.0f};
  if (norm) {
    const auto of = [&](int i) { return FsgsGradTensor{const_cast<void *>(tensors[i].grad), tensors[i].n, dtype, 0}; };
    if (int rc = launch_norm(n_tensors, of, max_norm, (char *)norm_scratch + 16, norm_scratch_bytes - 16, norm, (float *)norm_scratch,
                             true, &bound, stream))
      return rc;
  }
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
    t.bound = bound;
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
      t.at[k] = {x.param, x.grad, x.exp_avg, x.exp_avg_sq, x.master, x.scales, x.n, (uint32_t)groups, (uint32_t)at};
      t.start[k] = (uint32_t)groups;
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
    if (x.n < 0 || x.n > MAX_ELEMENTS) return FSGS_ERR_INVALID;
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

static int check_grads(int n_tensors, const FsgsGradTensor *grads, bool write) {
  if (n_tensors < 0 || (n_tensors > 0 && !grads)) return FSGS_ERR_INVALID;
  Regions regions((size_t)n_tensors);
  if (!regions.items) return FSGS_ERR_CAPACITY;
  for (int i = 0; i < n_tensors; i++) {
    if (grads[i].n < 0 || !size_of(grads[i].dtype) || (grads[i].n > 0 && !grads[i].grad)) return FSGS_ERR_INVALID;
    if (grads[i].n > INT64_MAX / 16 || turns_of(grads[i]) > MAX_TURNS) return FSGS_ERR_INVALID;
    regions.add(grads[i].grad, grads[i].n * size_of(grads[i].dtype), write);
  }
  return regions.clash() ? FSGS_ERR_INVALID : FSGS_OK;
}

int fsgs_grad_norm(int n_tensors, const FsgsGradTensor *grads, float max_norm, void *scratch, size_t scratch_bytes,
                   float *norm, float *factor, fsgs_stream_t stream) {
  if (int rc = check_grads(n_tensors, grads, false)) return rc;
  if (!norm || !factor || !(max_norm >= 0.0f) || (n_tensors > 0 && !scratch)) return FSGS_ERR_INVALID;
  Bound bound;
  return launch_norm(n_tensors, [&](int i) { return grads[i]; }, max_norm, scratch, scratch_bytes, norm, factor, false, &bound,
                     (hipStream_t)stream);
}

int fsgs_grad_scale(int n_tensors, const FsgsGradTensor *grads, const float *factor, fsgs_stream_t stream) {
  if (int rc = check_grads(n_tensors, grads, true)) return rc;
  if (n_tensors > 0 && !factor) return FSGS_ERR_INVALID;
  return launch_scale(n_tensors, [&](int i) { return grads[i]; }, Bound{nullptr, factor, nullptr, 0, 0.0f}, (hipStream_t)stream);
}

int fsgs_grad_clip(int n_tensors, const FsgsGradTensor *grads, float max_norm, void *scratch, size_t scratch_bytes,
                   float *norm, float *factor, fsgs_stream_t stream) {
  if (int rc = check_grads(n_tensors, grads, true)) return rc;
  if (!norm || !factor || !(max_norm >= 0.0f) || (n_tensors > 0 && !scratch)) return FSGS_ERR_INVALID;
  const auto of = [&](int i) { return grads[i]; };
  Bound bound;
  if (int rc = launch_norm(n_tensors, of, max_norm, scratch, scratch_bytes, norm, factor, true, &bound, (hipStream_t)stream)) return rc;
  return launch_scale(n_tensors, of, bound, (hipStream_t)stream);
}

}  // extern "C"
