// Log probabilities of chosen tokens (or list items) and their gradient (gfx950).
//
//   z = x / T,  logp_n = z_{n, y_n} - log sum_v exp z_nv,  dx_nv = g_n / T (1[v = y_n] - softmax(z_n)_v)
//
// Forward: one pass over the logits with a running maximum and a running sum of exponentials (fp32), the pair
// (max x, sum exp((x - max) / T)) of every row kept for the backward, which is one read and one write of the row:
// p = exp((x - max) / T) / sum.  A row with target < 0 is no target: log probability 0, gradient 0, its logits are not read.
// A target beyond the row: NaN in both.
// Bound by HBM (8192 x 50 021 bf16, a tenth without a target: 123 us forward = 6.0 TB/s, 330 us backward = 4.7 TB/s; a copy
// reaches 4.9).  A row is read by 16-byte accesses between its first and last 16-byte boundary: rows of an odd length start
// anywhere.  Few long rows are split over workgroups and joined by a second launch (2 x 131 072: 5 us), short ones share a
// wavefront (16 384 x 200 fp32: 12 us with the gradient, 17 with a wavefront a row).
#include "common.h"
#include "elem.h"

using namespace tfr;

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int SMALL_VOCAB = 2048;          // up to here a wavefront or a part of it takes a row
constexpr int SPLIT_MIN = 4096;           // elements of a row that a workgroup gets at least when rows are split

struct Rows {                              // logits[b, t, :] at b * stride_b + t * stride_t
  unsigned per;
  long stride_b, stride_t;
  __device__ __forceinline__ long offset(long n) const {       // n < 2^24
    const unsigned b = (unsigned)n / per;
    return b * stride_b + ((unsigned)n - b * per) * stride_t;
  }
};

// Running softmax statistics: m = max x, s = sum exp2((x - m) c).
struct Stat {
  float m, s;
  __device__ __forceinline__ void add(const Stat o, float c) {
    const float m1 = fmaxf(m, o.m), base = m1 == -INFINITY ? 0.f : m1;
    s = s * __builtin_amdgcn_exp2f((m - base) * c) + o.s * __builtin_amdgcn_exp2f((o.m - base) * c);
    m = m1;
  }
  template <int E> __device__ __forceinline__ void take(const float (&v)[E], float c) {
    float m1 = m;
#pragma unroll
    for (int e = 0; e < E; ++e) m1 = fmaxf(m1, v[e]);
    const float base = m1 == -INFINITY ? 0.f : m1;             // a row of -inf so far: exp(-inf) stays 0
    float t = s * __builtin_amdgcn_exp2f((m - base) * c);
#pragma unroll
    for (int e = 0; e < E; ++e) t += __builtin_amdgcn_exp2f((v[e] - base) * c);
    s = t;
    m = m1;
  }
};

// The statistics of LANES neighbouring lanes, for all of them.
template <int LANES = 64>
__device__ __forceinline__ Stat wave_stat(Stat a, float c) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    Stat b;
    b.m = __shfl_xor(a.m, o, 64);
    b.s = __shfl_xor(a.s, o, 64);
    a.add(b, c);
  }
  return a;
}

// Every thread of the workgroup (4 waves) gets the sum.
__device__ __forceinline__ Stat block_stat(Stat a, float c) {
  __shared__ Stat s_part[4];
  a = wave_stat(a, c);
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = a;
  __syncthreads();
  a = s_part[0];
  for (int w = 1; w < 4; ++w) a.add(s_part[w], c);
  return a;
}

// STREAM: logits beyond the Infinity Cache (256 MB) are read, and their gradient written, past the caches (8192 x 50 021 bf16: 175 +
// 311 us through them, 123 + 330 so; 16 384 x 200 fp32, 13 MB: 12.5 us for 13.5).
template <typename T, int E, bool STREAM>
__device__ __forceinline__ void load_row(const T* __restrict__ p, float (&v)[E]) {
  widen<T, E>(STREAM ? load_raw_stream<T, E>(p) : load_raw<T, E>(p), v);
}

// Statistics of x[lo, hi) by THREADS threads: single elements up to the first 16-byte boundary and behind the last.
template <typename T, int THREADS, bool STREAM>
__device__ __forceinline__ Stat row_stat(const T* __restrict__ x, int lo, int hi, int tid, float c) {
  constexpr int E = 16 / sizeof(T);
  Stat a = {-INFINITY, 0.f};
  const int off = (int)(((uintptr_t)(x + lo) & 15) / sizeof(T));
  int head = lo + (off ? E - off : 0);
  if (head > hi) head = hi;
  if (tid < head - lo) {
    float v[1] = {(float)x[lo + tid]};
    a.take<1>(v, c);
  }
  const int packs = (hi - head) / E;
  const T* p = x + head;
  int i = tid;
  for (; i + 3 * THREADS < packs; i += 4 * THREADS) {
    float v[4][E];
#pragma unroll
    for (int k = 0; k < 4; ++k) load_row<T, E, STREAM>(p + (long)(i + k * THREADS) * E, v[k]);
#pragma unroll
    for (int k = 0; k < 4; ++k) a.take<E>(v[k], c);
  }
  for (; i < packs; i += THREADS) {
    float v[E];
    load_row<T, E, STREAM>(p + (long)i * E, v);
    a.take<E>(v, c);
  }
  const int tail = head + packs * E;
  if (tid < hi - tail) {
    float v[1] = {(float)x[tail + tid]};
    a.take<1>(v, c);
  }
  return a;
}

// The chosen token's logit, read while the row is summed; NaN where there is no such token.
template <typename T>
__device__ __forceinline__ float chosen(const T* __restrict__ x, long target, int vocab) {
  return target < vocab ? (float)x[target] : __builtin_nanf("");
}

__device__ __forceinline__ void write_logp(float xy, Stat a, float inv_t, float* logp, float* stats) {
  *logp = (xy - a.m) * inv_t - logf(a.s);
  if (stats) {
    stats[0] = a.m;
    stats[1] = a.s;
  }
}

__device__ __forceinline__ void write_none(float* logp, float* stats) {
  *logp = 0.f;
  if (stats) stats[0] = stats[1] = 0.f;
}

// Short rows: LANES lanes a row.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void logprob_wave_kernel(const T* __restrict__ logits, const Rows rows, const int64_t* __restrict__ target,
                                                           long n, int vocab, float inv_t, float* __restrict__ logp,
                                                           float* __restrict__ stats) {
  const long row = (long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (row >= n) return;
  const int lane = threadIdx.x & (LANES - 1);
  const long y = target[row];
  float* st = stats ? stats + 2 * row : nullptr;
  if (y < 0) {
    if (lane == 0) write_none(logp + row, st);
    return;
  }
  const T* x = logits + rows.offset(row);
  const float c = inv_t * kLog2e;
  const float xy = chosen(x, y, vocab);
  const Stat a = wave_stat<LANES>(row_stat<T, LANES, false>(x, 0, vocab, lane, c), c);
  if (lane == 0) write_logp(xy, a, inv_t, logp + row, st);
}

// One workgroup a row (gridDim.y == 1), or a part of a row whose statistics go to parts[row][blockIdx.y].
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void logprob_block_kernel(const T* __restrict__ logits, const Rows rows, const int64_t* __restrict__ target,
                                                            int vocab, int part, float inv_t, float* __restrict__ logp,
                                                            float* __restrict__ stats, float* __restrict__ parts) {
  const long row = blockIdx.x;
  const long y = target[row];
  float* st = stats ? stats + 2 * row : nullptr;
  if (y < 0) {
    if (blockIdx.y == 0 && threadIdx.x == 0) write_none(logp + row, st);
    return;
  }
  const T* x = logits + rows.offset(row);
  const float c = inv_t * kLog2e;
  const long lo = (long)blockIdx.y * part;
  const int hi = (int)(lo + part < vocab ? lo + part : vocab);
  const float xy = gridDim.y == 1 && threadIdx.x == 0 ? chosen(x, y, vocab) : 0.f;
  const Stat a = block_stat(row_stat<T, 256, STREAM>(x, (int)lo, hi, threadIdx.x, c), c);
  if (threadIdx.x != 0) return;
  if (gridDim.y == 1) {
    write_logp(xy, a, inv_t, logp + row, st);
  } else {
    float* p = parts + 2 * (row * gridDim.y + blockIdx.y);
    p[0] = a.m;
    p[1] = a.s;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void logprob_join_kernel(const T* __restrict__ logits, const Rows rows, const int64_t* __restrict__ target,
                                                           long n, int vocab, int splits, float inv_t, const float* __restrict__ parts,
                                                           float* __restrict__ logp, float* __restrict__ stats) {
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= n) return;
  const int lane = threadIdx.x & 63;
  const long y = target[row];
  if (y < 0) return;                                           // written by the first launch
  const float c = inv_t * kLog2e;
  const float xy = chosen(logits + rows.offset(row), y, vocab);
  Stat a = {-INFINITY, 0.f};
  for (int i = lane; i < splits; i += 64) {
    const Stat b = {parts[2 * (row * splits + i)], parts[2 * (row * splits + i) + 1]};
    a.add(b, c);
  }
  a = wave_stat(a, c);
  if (lane == 0) write_logp(xy, a, inv_t, logp + row, stats ? stats + 2 * row : nullptr);
}

// ------------------------------------------------------------------------------------------------ gradient
// out[lo, hi) of one row by THREADS threads: 16-byte accesses where x and out lie on the same offset from their boundaries, one element
// at a time where they do not (8192 x 50 021 bf16: 364 us for rows that lie so, 566 for the same rows sliced from longer ones).
template <typename T, int THREADS, bool STREAM>
__device__ __forceinline__ void grad_row(const T* __restrict__ x, T* __restrict__ out, int lo, int hi, int tid, long y, float g, float m,
                                         float over_s, float c) {
  constexpr int E = 16 / sizeof(T);
  const int off = (int)(((uintptr_t)(out + lo) & 15) / sizeof(T));
  int head = lo + (off ? E - off : 0);
  if (head > hi) head = hi;
  const int packs = (hi - head) / E, tail = head + packs * E;
  const float scale = -g * over_s;
  auto one = [&](int i) {
    const float p = scale * __builtin_amdgcn_exp2f(((float)x[i] - m) * c);
    out[i] = (T)(i == y ? g + p : p);
  };
  if (tid < head - lo) one(lo + tid);
  if (tid < hi - tail) one(tail + tid);
  if ((((uintptr_t)(x + head) ^ (uintptr_t)(out + head)) & 15) == 0) {
    for (int i = tid; i < packs; i += THREADS) {
      const int at = head + i * E;
      float v[E];
      load_row<T, E, STREAM>(x + at, v);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float p = scale * __builtin_amdgcn_exp2f((v[e] - m) * c);
        v[e] = at + e == y ? g + p : p;
      }
      if (STREAM) store_pack_stream<T, E>(out + at, v);
      else store_pack<T, E>(out + at, v);
    }
  } else {
    for (int i = head + tid; i < tail; i += THREADS) one(i);
  }
}

template <typename T, int THREADS>
__device__ __forceinline__ void fill_row(T* __restrict__ out, int lo, int hi, int tid, float value) {
  constexpr int E = 16 / sizeof(T);
  const int off = (int)(((uintptr_t)(out + lo) & 15) / sizeof(T));
  int head = lo + (off ? E - off : 0);
  if (head > hi) head = hi;
  const int packs = (hi - head) / E, tail = head + packs * E;
  if (tid < head - lo) out[lo + tid] = (T)value;
  if (tid < hi - tail) out[tail + tid] = (T)value;
  float v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = value;
  for (int i = tid; i < packs; i += THREADS) store_pack<T, E>(out + head + (long)i * E, v);
}

template <typename T, int THREADS, bool STREAM>
__device__ __forceinline__ void grad_part(const T* __restrict__ logits, const Rows& rows, const int64_t* __restrict__ target,
                                          const float* __restrict__ stats, const float* __restrict__ upstream, long row, int vocab,
                                          int lo, int hi, int tid, float inv_t, T* __restrict__ out) {
  const long y = target[row];
  T* o = out + row * vocab;
  const float m = stats[2 * row], s = stats[2 * row + 1];
  if (y < 0) {
    fill_row<T, THREADS>(o, lo, hi, tid, 0.f);
  } else if (y >= vocab) {
    fill_row<T, THREADS>(o, lo, hi, tid, __builtin_nanf(""));
  } else {
    grad_row<T, THREADS, STREAM>(logits + rows.offset(row), o, lo, hi, tid, y, upstream[row] * inv_t, m, 1.f / s, inv_t * kLog2e);
  }
}

template <typename T, int LANES>
__global__ __launch_bounds__(256) void logprob_grad_wave_kernel(const T* __restrict__ logits, const Rows rows, const int64_t* __restrict__ target,
                                                                const float* __restrict__ stats, const float* __restrict__ upstream, long n,
                                                                int vocab, float inv_t, T* __restrict__ out) {
  const long row = (long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (row >= n) return;
  grad_part<T, LANES, false>(logits, rows, target, stats, upstream, row, vocab, 0, vocab, threadIdx.x & (LANES - 1), inv_t, out);
}

template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void logprob_grad_block_kernel(const T* __restrict__ logits, const Rows rows, const int64_t* __restrict__ target,
                                                                 const float* __restrict__ stats, const float* __restrict__ upstream,
                                                                 int vocab, int part, float inv_t, T* __restrict__ out) {
  const long lo = (long)blockIdx.y * part;
  const int hi = (int)(lo + part < vocab ? lo + part : vocab);
  grad_part<T, 256, STREAM>(logits, rows, target, stats, upstream, blockIdx.x, vocab, (int)lo, hi, threadIdx.x, inv_t, out);
}

// ------------------------------------------------------------------------------------------------ host
constexpr long kMostRows = (1l << 24) - 1;       // a workgroup a row: no grid gets 2^32 threads
constexpr int kMostVocab = 1 << 28;              // parts of a row are counted in gridDim.y (65 535)

// Workgroups per row of the forward: 1 where the rows alone fill the card twice, else parts of at least SPLIT_MIN elements.
int splits_of(long n, int vocab) {
  if (vocab <= SMALL_VOCAB || n >= 512) return 1;
  long s = (512 + n - 1) / n;
  const long most = vocab / SPLIT_MIN;
  if (s > most) s = most;
  return s < 1 ? 1 : (int)s;
}

bool bad_args(int dtype, long per, long stride_b, long stride_t, long n, int vocab, float temperature) {
  const float inv = 1.f / temperature;
  return !elem_known(dtype) || n < 0 || n > kMostRows || vocab < 1 || vocab > kMostVocab || per < 1 || per > UINT32_MAX || stride_b < 0 || stride_t < 0 ||
         !(temperature > 0.f) || !(inv > 0.f) || inv == INFINITY;
}

template <typename T>
bool beyond_cache(long n, int vocab) { return n * vocab * (long)sizeof(T) > (256l << 20); }

// Lanes of a short row: a few 16-byte accesses each.
template <typename T>
int lanes_of(int vocab) {
  const long bytes = (long)vocab * (long)sizeof(T);
  return bytes <= 256 ? 8 : bytes <= 1024 ? 16 : 64;
}

template <typename T>
int forward(const T* logits, Rows rows, const int64_t* target, long n, int vocab, float inv_t, float* logp, float* stats, float* parts,
            hipStream_t st) {
  if (vocab <= SMALL_VOCAB) {
    const int lanes = lanes_of<T>(vocab);
    const auto kernel = lanes == 8 ? logprob_wave_kernel<T, 8> : lanes == 16 ? logprob_wave_kernel<T, 16> : logprob_wave_kernel<T, 64>;
    kernel<<<(unsigned)((n * lanes + 255) / 256), 256, 0, st>>>(logits, rows, target, n, vocab, inv_t, logp, stats);
    return (int)hipGetLastError();
  }
  const int splits = splits_of(n, vocab);
  const int part = ((vocab + splits - 1) / splits + 7) / 8 * 8;
  const auto kernel = beyond_cache<T>(n, vocab) ? logprob_block_kernel<T, true> : logprob_block_kernel<T, false>;
  kernel<<<dim3((unsigned)n, splits), 256, 0, st>>>(logits, rows, target, vocab, part, inv_t, logp, stats, parts);
  if (splits > 1)
    logprob_join_kernel<T><<<(unsigned)((n + 3) / 4), 256, 0, st>>>(logits, rows, target, n, vocab, splits, inv_t, parts, logp, stats);
  return (int)hipGetLastError();
}

template <typename T>
int backward(const T* logits, Rows rows, const int64_t* target, const float* stats, const float* upstream, long n, int vocab, float inv_t,
             T* out, hipStream_t st) {
  if (vocab <= SMALL_VOCAB) {
    const int lanes = lanes_of<T>(vocab);
    const auto kernel = lanes == 8 ? logprob_grad_wave_kernel<T, 8> : lanes == 16 ? logprob_grad_wave_kernel<T, 16> : logprob_grad_wave_kernel<T, 64>;
    kernel<<<(unsigned)((n * lanes + 255) / 256), 256, 0, st>>>(logits, rows, target, stats, upstream, n, vocab, inv_t, out);
  } else {
    const int part = 256 * 8 * (16 / (int)sizeof(T));
    const auto kernel = beyond_cache<T>(n, vocab) ? logprob_grad_block_kernel<T, true> : logprob_grad_block_kernel<T, false>;
    kernel<<<dim3((unsigned)n, (vocab + part - 1) / part), 256, 0, st>>>(logits, rows, target, stats, upstream, vocab, part, inv_t, out);
  }
  return (int)hipGetLastError();
}

}  // namespace

extern "C" long tfr_token_logprob_workspace_bytes(long n, int vocab) {
  if (n < 0 || n > kMostRows || vocab < 1 || vocab > kMostVocab) return TFR_EINVAL;
  if (n == 0) return 0;
  const int s = splits_of(n, vocab);
  return s > 1 ? 8l * n * s : 0;
}

extern "C" int tfr_token_logprob(const void* logits, int dtype, long per, long stride_b, long stride_t, const int64_t* target, long n,
                                 int vocab, float temperature, float* logp, float* stats, void* workspace, long workspace_bytes,
                                 void* stream) {
  if (bad_args(dtype, per, stride_b, stride_t, n, vocab, temperature)) return TFR_EINVAL;
  if (n == 0) return TFR_OK;
  if (!logits || !target || !logp) return TFR_EINVAL;
  const long need = tfr_token_logprob_workspace_bytes(n, vocab);
  if (need > 0 && (!workspace || workspace_bytes < need)) return TFR_EINVAL;
  const Rows r = {(unsigned)per, stride_b, stride_t};
  hipStream_t st = (hipStream_t)stream;
  const float inv = 1.f / temperature;
  if (dtype == TFR_DTYPE_F32) return forward<float>((const float*)logits, r, target, n, vocab, inv, logp, stats, (float*)workspace, st);
  if (dtype == TFR_DTYPE_BF16) return forward<__bf16>((const __bf16*)logits, r, target, n, vocab, inv, logp, stats, (float*)workspace, st);
  return forward<_Float16>((const _Float16*)logits, r, target, n, vocab, inv, logp, stats, (float*)workspace, st);
}

extern "C" int tfr_token_logprob_grad(const void* logits, int dtype, long per, long stride_b, long stride_t, const int64_t* target,
                                      const float* stats, const float* upstream, long n, int vocab, float temperature, void* dlogits,
                                      void* stream) {
  if (bad_args(dtype, per, stride_b, stride_t, n, vocab, temperature)) return TFR_EINVAL;
  if (n == 0) return TFR_OK;
  if (!logits || !target || !stats || !upstream || !dlogits) return TFR_EINVAL;
  const Rows r = {(unsigned)per, stride_b, stride_t};
  hipStream_t st = (hipStream_t)stream;
  const float inv = 1.f / temperature;
  if (dtype == TFR_DTYPE_F32) return backward<float>((const float*)logits, r, target, stats, upstream, n, vocab, inv, (float*)dlogits, st);
  if (dtype == TFR_DTYPE_BF16) return backward<__bf16>((const __bf16*)logits, r, target, stats, upstream, n, vocab, inv, (__bf16*)dlogits, st);
  return backward<_Float16>((const _Float16*)logits, r, target, stats, upstream, n, vocab, inv, (_Float16*)dlogits, st);
}
