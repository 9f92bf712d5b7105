// AdamW over many tensors in one launch, with the moments held in 32 or in 8 bits (gfx950).
//
//   m <- b1 m + (1 - b1) g        v <- b2 v + (1 - b2) g^2
//   p <- p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// HBM-bound: with fp32 parameters and moments 16 bytes are read and 12 written an element (152 M elements in 98 tensors: 801 us =
// 5.3 TB/s; the 14 tensors of a 136-512-512-512-1 tower: 7 us).  The addresses and lengths of up to
// TFR_ADAMW_MAX_TENSORS (TFR_ADAMW8_MAX_TENSORS) tensors travel in the kernel's arguments: no table in device memory that a
// step would have to copy first (the gradients' addresses change from step to step), and a captured launch holds its own.  Tensors that are
// not 16-byte aligned, and the last piece of each, go one element a thread (that tower replayed: 5.1 us a step, 7.8 unaligned).
//
// 8 bits: QBLOCK consecutive elements share two scales.  m is held as a signed code of -127 .. 127, the root of v as an unsigned
// code of 0 .. 255; the root halves the exponent range that 255 steps have to cover.  Codes are the nearest to the updated
// value, but the code of a positive v is at least 1: a denominator is never rounded down to eps, so small second moments slow
// an element down and never blow it up.  Which code a value next to a border gets is decided in fp64 and does not hang on fp32
// rounding.  The parameter's own update uses the moments before they are rounded to codes.  An element whose moments are no longer
// finite keeps the code -128, which stands for NaN, and does not touch its neighbours' scale.
#include "common.h"
#include "elem.h"

using namespace tfr;

namespace {

constexpr int QBLOCK = TFR_ADAMW_QBLOCK;

struct Coef {
  double b1, c1, b2, c2;               // beta and 1 - beta
  float decay, step, root, eps;        // 1 - lr decay, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  const float* now;                    // device (decay, step, root) of a step that is counted on the device, or null
  int stride;                          // 3: the launch's tensors have their own, one after the other; 0: one for all
};

template <int CAP, bool Q>
struct Table {
  Coef coef;
  int count;
  int first[CAP + 1];                  // first workgroup of each tensor
  void* p[CAP];
  const void* g[CAP];
  void* m[CAP];
  void* v[CAP];
  float* ms[Q ? CAP : 1];
  float* vs[Q ? CAP : 1];
  long n[CAP];
};
typedef Table<TFR_ADAMW_MAX_TENSORS, false> Table32;
typedef Table<TFR_ADAMW8_MAX_TENSORS, true> Table8;
static_assert(sizeof(Table32) <= 4096 && sizeof(Table8) <= 4096, "kernel arguments hold 4 KB");

template <typename Tab>
__device__ __forceinline__ int tensor_of(const Tab& t, int block) {
  int lo = 0, hi = t.count;            // t.first[lo] <= block < t.first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.first[mid] <= block) lo = mid; else hi = mid;
  }
  return lo;
}

struct Now { float decay, step, root; };
__device__ __forceinline__ Now now_of(const Coef& c, int tensor) {
  Now w = {c.decay, c.step, c.root};
  if (c.now) {
    const float* n = c.now + c.stride * tensor;
    w = {n[0], n[1], n[2]};
  }
  return w;
}

__device__ __forceinline__ float updated(float p, float m, float v, const Now& w, float eps) {
  return p * w.decay - m * w.step / (sqrtf(v) * w.root + eps);
}

// STREAM: a launch over more than the Infinity Cache (256 MB) goes past the caches (152 M fp32 elements 833 -> 801 us, 246 M bf16 with
// 8-bit moments 536 -> 524; the tower's 14 tensors, 10 MB: 7.1 -> 7.7).
template <typename T, int E, bool STREAM>
__device__ __forceinline__ void get(const T* __restrict__ p, float (&v)[E]) {
  widen<T, E>(STREAM ? load_raw_stream<T, E>(p) : load_raw<T, E>(p), v);
}
template <typename T, int E, bool STREAM>
__device__ __forceinline__ void put(T* __restrict__ p, const float (&v)[E]) {
  if (STREAM) store_pack_stream<T, E>(p, v);
  else store_pack<T, E>(p, v);
}

constexpr int BLOCK32 = 4096;          // elements of a workgroup
constexpr int BLOCK8 = 4096;

template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void adamw_kernel(const Table32 t) {
  const int i = tensor_of(t, blockIdx.x);
  const long n = t.n[i], base = (long)(blockIdx.x - t.first[i]) * BLOCK32;
  T* __restrict__ p = (T*)t.p[i] + base;
  const T* __restrict__ g = (const T*)t.g[i] + base;
  float* __restrict__ m = (float*)t.m[i] + base;
  float* __restrict__ v = (float*)t.v[i] + base;
  const Now w = now_of(t.coef, i);
  const float b1 = (float)t.coef.b1, c1 = (float)t.coef.c1, b2 = (float)t.coef.b2, c2 = (float)t.coef.c2, eps = t.coef.eps;
  const int left = (int)(n - base < BLOCK32 ? n - base : BLOCK32);
  const bool wide = (((uintptr_t)p | (uintptr_t)g) & (4 * sizeof(T) - 1)) == 0 && (((uintptr_t)m | (uintptr_t)v) & 15) == 0;
  if (wide && left == BLOCK32) {
#pragma unroll
    for (int k = 0; k < BLOCK32 / 1024; ++k) {
      const int at = k * 1024 + threadIdx.x * 4;
      float pe[4], ge[4], me[4], ve[4];
      get<T, 4, STREAM>(p + at, pe);
      get<T, 4, STREAM>(g + at, ge);
      get<float, 4, STREAM>(m + at, me);
      get<float, 4, STREAM>(v + at, ve);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        me[e] = b1 * me[e] + c1 * ge[e];
        ve[e] = b2 * ve[e] + c2 * (ge[e] * ge[e]);
        pe[e] = updated(pe[e], me[e], ve[e], w, eps);
      }
      put<float, 4, STREAM>(m + at, me);
      put<float, 4, STREAM>(v + at, ve);
      put<T, 4, STREAM>(p + at, pe);
    }
    return;
  }
  for (int at = threadIdx.x; at < left; at += 256) {
    const float ge = (float)g[at];
    const float me = b1 * m[at] + c1 * ge, ve = b2 * v[at] + c2 * (ge * ge);
    m[at] = me;
    v[at] = ve;
    p[at] = (T)updated((float)p[at], me, ve, w, eps);
  }
}

// The updated moments of one 8-bit element: fp64, in this order, wherever they are needed.
struct Moments {
  double m, v;
};
__device__ __forceinline__ Moments moments(int mc, float vc, float g, double b1_sm, double b2_sv2, double c1, double c2) {
  const double gd = (double)g;
  return {__builtin_fma((double)mc, b1_sm, c1 * gd), __builtin_fma((double)(vc * vc), b2_sv2, c2 * (gd * gd))};
}
__device__ __forceinline__ int signed_code(uint2 w, int e) { return (int)(int8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3))); }
__device__ __forceinline__ float unsigned_code(uint2 w, int e) { return (float)(((e < 4 ? w.x : w.y) >> (8 * (e & 3))) & 255u); }

// Maximum over the 16 lanes of a row (lane / 16), for all of them: rotations of the row.
__device__ __forceinline__ float row_max(float x) {
  x = fmaxf(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xf, 0xf, true)));   // row_ror:8
  x = fmaxf(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x124, 0xf, 0xf, true)));   // row_ror:4
  x = fmaxf(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x122, 0xf, 0xf, true)));   // row_ror:2
  return fmaxf(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x121, 0xf, 0xf, true)));
}

// A thread takes 8 consecutive elements, 16 lanes a scale.  The codes lie in whole blocks (their tensors are padded), the
// parameters and gradients end where they end.
//
// Codes are chosen in fp32 (the value over the scale is off by at most 255 * 5.5 * 2^-24 = 8.4e-5 of a step) and again in fp64 by the
// few threads that hold a value within 1e-4 of a border: the same codes as fp64 throughout, at half the instructions (246 M
// bf16 elements: 787 us with all of it in fp64, bound by instruction issue; 524 us so, 4.7 TB/s, near what a copy reaches).
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void adamw8_kernel(const Table8 t) {
  const int i = tensor_of(t, blockIdx.x);
  const long n = t.n[i], base = (long)(blockIdx.x - t.first[i]) * BLOCK8;
  T* __restrict__ p = (T*)t.p[i];
  const T* __restrict__ g = (const T*)t.g[i];
  int8_t* __restrict__ m = (int8_t*)t.m[i];
  uint8_t* __restrict__ v = (uint8_t*)t.v[i];
  float* __restrict__ ms = t.ms[i];
  float* __restrict__ vs = t.vs[i];
  const Now w = now_of(t.coef, i);
  const double c1 = t.coef.c1, c2 = t.coef.c2;
  const float eps = t.coef.eps;
  const bool tiny_eps = eps < 1e-12f;                          // the fast root takes v below 2^-126 as 0: far below any other eps
  constexpr int W = 16 / sizeof(T);                            // elements of a 16-byte access
  const bool wide = (((uintptr_t)p | (uintptr_t)g) & 15) == 0;
  const long padded = (n + QBLOCK - 1) / QBLOCK * QBLOCK;
#pragma unroll 1
  for (int k = 0; k < BLOCK8 / 2048; ++k) {
    const long at = base + k * 2048 + threadIdx.x * 8;
    if (at >= padded) return;                                   // whole groups of 16 lanes
    float pe[8], ge[8], m32[8], root[8], low[8];
    const bool whole = wide && at + 8 <= n;
    if (whole) {
#pragma unroll
      for (int q = 0; q < 8; q += W) {
        get<T, W, STREAM>(p + at + q, *reinterpret_cast<float(*)[W]>(pe + q));
        get<T, W, STREAM>(g + at + q, *reinterpret_cast<float(*)[W]>(ge + q));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pe[e] = at + e < n ? (float)p[at + e] : 0.f;
        ge[e] = at + e < n ? (float)g[at + e] : 0.f;
      }
    }
    const uint2 mw = *reinterpret_cast<const uint2*>(m + at), vw = *reinterpret_cast<const uint2*>(v + at);
    const double sm = (double)ms[at / QBLOCK], sv = (double)vs[at / QBLOCK];
    const double b1_sm = t.coef.b1 * sm, b2_sv2 = t.coef.b2 * (sv * sv);
    float most_m = 0.f, most_v = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const Moments d = moments(signed_code(mw, e), unsigned_code(vw, e), ge[e], b1_sm, b2_sv2, c1, c2);
      m32[e] = (float)d.m;
      root[e] = (float)d.v;
      low[e] = d.v > 0.0 ? 1.f : 0.f;                           // the least code
    }
    unsigned lost = 0;                                          // bit e: the moments are no longer finite
    const unsigned mx = mw.x ^ 0x80808080u, my = mw.y ^ 0x80808080u;     // a byte of 0 is the code -128
    float all = 0.f;                                            // a gradient that is not finite shows in v
#pragma unroll
    for (int e = 0; e < 8; ++e) all += root[e];
    if ((((mx - 0x01010101u) & ~mx) | ((my - 0x01010101u) & ~my)) & 0x80808080u || !(all < INFINITY)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (signed_code(mw, e) == -128) m32[e] = __builtin_nanf("");
        const bool bad = !(fabsf(m32[e]) < INFINITY) || !(root[e] < INFINITY);
        lost |= bad ? 1u << e : 0u;
        most_m = fmaxf(most_m, bad ? 0.f : fabsf(m32[e]));
        most_v = fmaxf(most_v, bad ? 0.f : root[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        most_m = fmaxf(most_m, fabsf(m32[e]));
        most_v = fmaxf(most_v, root[e]);
      }
    }
    if (tiny_eps) {
#pragma unroll
      for (int e = 0; e < 8; ++e) root[e] = sqrtf(root[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) root[e] = __builtin_amdgcn_sqrtf(root[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      pe[e] = __builtin_fmaf(-m32[e] * w.step, __builtin_amdgcn_rcpf(__builtin_fmaf(root[e], w.root, eps)), pe[e] * w.decay);
    most_m = row_max(most_m);
    most_v = row_max(most_v);
    // in fp64 and rounded once, so that the scale is the same wherever it is computed
    const float new_sm = (float)((double)most_m * (1.0 / 127.0)), new_sv = (float)(sqrt((double)most_v) * (1.0 / 255.0));
    const float over_m = __builtin_amdgcn_rcpf(new_sm), over_v = __builtin_amdgcn_rcpf(new_sv);
    float km[8], kv[8], side = 0.f;                             // farthest from a code
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float ym = m32[e] * over_m, yv = root[e] * over_v;
      km[e] = rintf(ym);
      kv[e] = rintf(yv);
      side = fmaxf(side, fmaxf(fabsf(ym - km[e]), fabsf(yv - kv[e])));
      kv[e] = fmaxf(kv[e], low[e]);
    }
    // near a border, or scales that fp32 does not divide by
    const bool near = !(side < 0.4999f) || most_m < 1e-30f || most_v < 1e-30f;
    if (near) {
      const double wide_m = new_sm > 0.f ? 1.0 / (double)new_sm : 0.0, wide_v = new_sv > 0.f ? 1.0 / (double)new_sv : 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const Moments d = moments(signed_code(mw, e), unsigned_code(vw, e), ge[e], b1_sm, b2_sv2, c1, c2);
        km[e] = (float)fmin(fmax(rint(d.m * wide_m), -127.0), 127.0);
        kv[e] = fmaxf((float)fmin(rint(sqrt(d.v) * wide_v), 255.0), new_sv > 0.f ? low[e] : 0.f);
      }
    }
    uint2 mo = make_uint2(0u, 0u), vo = make_uint2(0u, 0u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // bytes of code + 128: the sign's bit is turned for all at once
      mo.x = __builtin_amdgcn_cvt_pk_u8_f32(km[e] + 128.f, e, mo.x);
      mo.y = __builtin_amdgcn_cvt_pk_u8_f32(km[e + 4] + 128.f, e, mo.y);
      vo.x = __builtin_amdgcn_cvt_pk_u8_f32(kv[e], e, vo.x);
      vo.y = __builtin_amdgcn_cvt_pk_u8_f32(kv[e + 4], e, vo.y);
    }
    mo.x ^= 0x80808080u;
    mo.y ^= 0x80808080u;
    if (lost) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const unsigned byte = lost & (1u << e) ? 255u << (8 * (e & 3)) : 0u, sign = byte & 0x80808080u;
        if (e < 4) {
          mo.x = (mo.x & ~byte) | sign;
          vo.x |= byte;
        } else {
          mo.y = (mo.y & ~byte) | sign;
          vo.y |= byte;
        }
      }
    }
    *reinterpret_cast<uint2*>(m + at) = mo;
    *reinterpret_cast<uint2*>(v + at) = vo;
    if ((threadIdx.x & 15) == 0) {
      ms[at / QBLOCK] = new_sm;
      vs[at / QBLOCK] = new_sv;
    }
    if (whole) {
#pragma unroll
      for (int q = 0; q < 8; q += W) put<T, W, STREAM>(p + at + q, *reinterpret_cast<float(*)[W]>(pe + q));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at + e < n) p[at + e] = (T)pe[e];
    }
  }
}

// The values that codes stand for: 8 a thread.
template <bool SQUARE>
__global__ __launch_bounds__(256) void adamw_dequantize_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales, long n,
                                                               float* __restrict__ out) {
  const long at = ((long)blockIdx.x * 256 + threadIdx.x) * 8;
  if (at >= n) return;
  const uint2 c = *reinterpret_cast<const uint2*>(codes + at);
  const float s = scales[at / QBLOCK];
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const unsigned b = ((e < 4 ? c.x : c.y) >> (8 * (e & 3))) & 255u;
    if (SQUARE) {
      const float r = (float)b * s;
      v[e] = r * r;
    } else {
      v[e] = b == 128u ? __builtin_nanf("") : (float)(int8_t)b * s;
    }
  }
  store_pack<float, 4>(out + at, *reinterpret_cast<float(*)[4]>(v));
  store_pack<float, 4>(out + at + 4, *reinterpret_cast<float(*)[4]>(v + 4));
}

// One more step, counted on the device: coefficients of the launch behind it.
__device__ __forceinline__ void advance(long* __restrict__ count, const float* __restrict__ lr_now, double lr, double b1, double b2, double decay,
                                        float* __restrict__ now) {
  const long t = count[0] + 1;
  count[0] = t;
  if (lr_now) lr = (double)lr_now[0];
  now[0] = (float)(1.0 - lr * decay);
  now[1] = (float)(lr / (1.0 - pow(b1, (double)t)));
  now[2] = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
}
__global__ void adamw_advance_kernel(long* __restrict__ count, const float* __restrict__ lr_now, double lr, double b1, double b2, double decay,
                                     float* __restrict__ now) {
  advance(count, lr_now, lr, b1, b2, decay, now);
}

// The same where every tensor of the launch has a count of its own (a thread each): a parameter that gets its first gradient late is
// corrected by the steps that it took.  `all` (or null) counts the steps of them together.
struct Counts {
  long* at[TFR_ADAMW_MAX_TENSORS];
};
constexpr int COUNT_THREADS = 128;
static_assert(TFR_ADAMW_MAX_TENSORS <= COUNT_THREADS && TFR_ADAMW8_MAX_TENSORS <= TFR_ADAMW_MAX_TENSORS, "a thread a tensor");
__global__ __launch_bounds__(COUNT_THREADS) void adamw_advance_each_kernel(const Counts counts, int n, long* __restrict__ all, const float* __restrict__ lr_now,
                                                                           double lr, double b1, double b2, double decay, float* __restrict__ now) {
  const int i = threadIdx.x;
  if (i == 0 && all) all[0] += 1;
  if (i < n) advance(counts.at[i], lr_now, lr, b1, b2, decay, now + 3 * i);
}

constexpr long kCache = 256l << 20;

template <typename T>
void launch32(const Table32& t, int blocks, hipStream_t st) {
  const auto kernel = (long)blocks * BLOCK32 * (2 * (long)sizeof(T) + 8) > kCache ? adamw_kernel<T, true> : adamw_kernel<T, false>;
  kernel<<<blocks, 256, 0, st>>>(t);
}
template <typename T>
void launch8(const Table8& t, int blocks, hipStream_t st) {
  const auto kernel = (long)blocks * BLOCK8 * (2 * (long)sizeof(T) + 2) > kCache ? adamw8_kernel<T, true> : adamw8_kernel<T, false>;
  kernel<<<blocks, 256, 0, st>>>(t);
}

bool bad_betas(double b1, double b2) { return !(b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0); }

template <typename Tab, int PER>
int fill(Tab& t, int cap, int count, void* const* p, const void* const* g, void* const* m, void* const* v, const int64_t* n, double lr,
         double b1, double b2, double eps, double decay, int64_t step, const float* now, int stride) {
  if (count < 1 || count > cap || !p || !g || !m || !v || !n || bad_betas(b1, b2)) return TFR_EINVAL;
  if (!now && step < 1) return TFR_EINVAL;
  t.coef.b1 = b1;
  t.coef.c1 = 1.0 - b1;
  t.coef.b2 = b2;
  t.coef.c2 = 1.0 - b2;
  t.coef.eps = (float)eps;
  t.coef.now = now;
  t.coef.stride = stride;
  t.coef.decay = (float)(1.0 - lr * decay);
  t.coef.step = now ? 0.f : (float)(lr / (1.0 - __builtin_pow(b1, (double)step)));
  t.coef.root = now ? 0.f : (float)(1.0 / __builtin_sqrt(1.0 - __builtin_pow(b2, (double)step)));
  t.count = count;
  long at = 0;
  for (int i = 0; i < count; ++i) {
    if (n[i] < 0 || (n[i] > 0 && (!p[i] || !g[i] || !m[i] || !v[i]))) return TFR_EINVAL;
    t.first[i] = (int)at;
    t.p[i] = p[i];
    t.g[i] = g[i];
    t.m[i] = m[i];
    t.v[i] = v[i];
    t.n[i] = n[i];
    at += (n[i] + PER - 1) / PER;
    if (at >= (1l << 24)) return TFR_EINVAL;                    // no grid of 2^32 threads
  }
  t.first[count] = (int)at;
  return TFR_OK;
}

template <typename Tab, int PER>
int fill_scales(Tab& t, int cap, int count, void* const* p, const void* const* g, void* const* m, float* const* ms, void* const* v, float* const* vs,
                const int64_t* n, double lr, double b1, double b2, double eps, double decay, int64_t step, const float* now, int stride) {
  if (!ms || !vs) return TFR_EINVAL;
  const int rc = fill<Tab, PER>(t, cap, count, p, g, m, v, n, lr, b1, b2, eps, decay, step, now, stride);
  if (rc != TFR_OK) return rc;
  for (int i = 0; i < count; ++i) {
    t.ms[i] = ms[i];
    t.vs[i] = vs[i];
    if (n[i] > 0 && (!ms[i] || !vs[i] || (((uintptr_t)m[i] | (uintptr_t)v[i]) & 7))) return TFR_EINVAL;
  }
  return TFR_OK;
}

int run(const Table32& t, int dtype, hipStream_t st) {
  const int blocks = t.first[t.count];
  if (blocks == 0) return TFR_OK;
  if (dtype == TFR_DTYPE_F32) launch32<float>(t, blocks, st);
  else if (dtype == TFR_DTYPE_BF16) launch32<__bf16>(t, blocks, st);
  else launch32<_Float16>(t, blocks, st);
  return (int)hipGetLastError();
}
int run(const Table8& t, int dtype, hipStream_t st) {
  const int blocks = t.first[t.count];
  if (blocks == 0) return TFR_OK;
  if (dtype == TFR_DTYPE_F32) launch8<float>(t, blocks, st);
  else if (dtype == TFR_DTYPE_BF16) launch8<__bf16>(t, blocks, st);
  else launch8<_Float16>(t, blocks, st);
  return (int)hipGetLastError();
}

// The counts of a table's tensors are advanced, then the table's launch reads its coefficients.
template <typename Tab>
int run_counted(const Tab& t, int dtype, int64_t* const* steps, int64_t* all, const float* lr_device, double lr, double b1, double b2,
                double decay, float* now, hipStream_t st) {
  Counts counts = {};
  for (int i = 0; i < t.count; ++i) {
    if (!steps[i]) return TFR_EINVAL;
    counts.at[i] = (long*)steps[i];
  }
  adamw_advance_each_kernel<<<1, COUNT_THREADS, 0, st>>>(counts, t.count, (long*)all, lr_device, lr, b1, b2, decay, now);
  const int rc = (int)hipGetLastError();
  return rc != TFR_OK ? rc : run(t, dtype, st);
}

}  // namespace

extern "C" int tfr_adamw(int dtype, int count, void* const* params_host, const void* const* grads_host, void* const* exp_avgs_host,
                         void* const* exp_avg_sqs_host, const int64_t* sizes_host, double lr, double beta1, double beta2, double eps,
                         double weight_decay, int64_t step, const float* now, void* stream) {
  if (!elem_known(dtype)) return TFR_EINVAL;
  Table32 t;
  const int rc = fill<Table32, BLOCK32>(t, TFR_ADAMW_MAX_TENSORS, count, params_host, grads_host, exp_avgs_host, exp_avg_sqs_host, sizes_host,
                                        lr, beta1, beta2, eps, weight_decay, step, now, 0);
  return rc != TFR_OK ? rc : run(t, dtype, (hipStream_t)stream);
}

extern "C" int tfr_adamw8(int dtype, int count, void* const* params_host, const void* const* grads_host, void* const* exp_avgs_host,
                          float* const* exp_avg_scales_host, void* const* exp_avg_sqs_host, float* const* exp_avg_sq_scales_host,
                          const int64_t* sizes_host, double lr, double beta1, double beta2, double eps, double weight_decay, int64_t step,
                          const float* now, void* stream) {
  if (!elem_known(dtype)) return TFR_EINVAL;
  Table8 t;
  const int rc = fill_scales<Table8, BLOCK8>(t, TFR_ADAMW8_MAX_TENSORS, count, params_host, grads_host, exp_avgs_host, exp_avg_scales_host, exp_avg_sqs_host,
                                             exp_avg_sq_scales_host, sizes_host, lr, beta1, beta2, eps, weight_decay, step, now, 0);
  return rc != TFR_OK ? rc : run(t, dtype, (hipStream_t)stream);
}

extern "C" int tfr_adamw_counted(int dtype, int count, void* const* params_host, const void* const* grads_host, void* const* exp_avgs_host,
                                 void* const* exp_avg_sqs_host, const int64_t* sizes_host, int64_t* const* steps_host, int64_t* all,
                                 const float* lr_device, double lr, double beta1, double beta2, double eps, double weight_decay, float* now,
                                 void* stream) {
  if (!elem_known(dtype) || !steps_host || !now) return TFR_EINVAL;
  Table32 t;
  const int rc = fill<Table32, BLOCK32>(t, TFR_ADAMW_MAX_TENSORS, count, params_host, grads_host, exp_avgs_host, exp_avg_sqs_host, sizes_host,
                                        lr, beta1, beta2, eps, weight_decay, 0, now, 3);
  return rc != TFR_OK ? rc : run_counted(t, dtype, steps_host, all, lr_device, lr, beta1, beta2, weight_decay, now, (hipStream_t)stream);
}

extern "C" int tfr_adamw8_counted(int dtype, int count, void* const* params_host, const void* const* grads_host, void* const* exp_avgs_host,
                                  float* const* exp_avg_scales_host, void* const* exp_avg_sqs_host, float* const* exp_avg_sq_scales_host,
                                  const int64_t* sizes_host, int64_t* const* steps_host, int64_t* all, const float* lr_device, double lr,
                                  double beta1, double beta2, double eps, double weight_decay, float* now, void* stream) {
  if (!elem_known(dtype) || !steps_host || !now) return TFR_EINVAL;
  Table8 t;
  const int rc = fill_scales<Table8, BLOCK8>(t, TFR_ADAMW8_MAX_TENSORS, count, params_host, grads_host, exp_avgs_host, exp_avg_scales_host, exp_avg_sqs_host,
                                             exp_avg_sq_scales_host, sizes_host, lr, beta1, beta2, eps, weight_decay, 0, now, 3);
  return rc != TFR_OK ? rc : run_counted(t, dtype, steps_host, all, lr_device, lr, beta1, beta2, weight_decay, now, (hipStream_t)stream);
}

extern "C" int tfr_adamw_advance(int64_t* step, const float* lr_device, double lr, double beta1, double beta2, double weight_decay, float* now,
                                 void* stream) {
  if (!step || !now || bad_betas(beta1, beta2)) return TFR_EINVAL;
  adamw_advance_kernel<<<1, 1, 0, (hipStream_t)stream>>>((long*)step, lr_device, lr, beta1, beta2, weight_decay, now);
  return (int)hipGetLastError();
}

extern "C" int tfr_adamw_dequantize(const void* codes, const float* scales, long n, int square, float* out, void* stream) {
  if (n < 0 || n % QBLOCK || n > (1l << 33)) return TFR_EINVAL;
  if (n == 0) return TFR_OK;
  if (!codes || !scales || !out || ((uintptr_t)codes & 7) || ((uintptr_t)out & 15)) return TFR_EINVAL;
  const unsigned blocks = (unsigned)((n + 2047) / 2048);
  hipStream_t st = (hipStream_t)stream;
  if (square) adamw_dequantize_kernel<true><<<blocks, 256, 0, st>>>((const uint8_t*)codes, scales, n, out);
  else adamw_dequantize_kernel<false><<<blocks, 256, 0, st>>>((const uint8_t*)codes, scales, n, out);
  return (int)hipGetLastError();
}
