// Embedding lookup with scaling, and its gradient by sorted tokens (gfx950).
//
//   lookup   out[b] = f_b * sum_t W[id_bt]      f_b = scale (no combiner: one token a row; sum) or scale / #{t : id_bt >= 0} (mean)
//   gradient dW[v]  = sum over the occurrences (b, t) of v of f_b * g[b]
//
// An id below 0 is padding: a zero row, no gradient.  An id beyond the table gives a row of NaN and no gradient: nothing
// outside the table is read.
//
// The gradient writes every row of dW exactly once and adds in an order that depends on the ids alone: the occurrences are
// sorted by id (stable radix sort, least significant digit first), a row's occurrences are then a run of the sorted list, and
// the wave that owns the row finds the run by a search.  No atomics on floating point, no separate zero fill.  Runs of common
// tokens are cut: every aligned chunk of CHUNK sorted occurrences that holds one single token is summed by a workgroup of its
// own beforehand, and the row adds those sums and the loose ends (a token that is 6 % of 262 144 costs its row 120 sums
// instead of 16 000 rows).
#include "common.h"
#include "elem.h"

using namespace tfr;

namespace {

constexpr int CHUNK = 128;              // sorted occurrences per chunk sum
constexpr int HEAVY = 64;               // occurrences from which the whole workgroup adds a row
constexpr int SMALL_SORT = 4096;        // lookups that one workgroup sorts in LDS
constexpr int ITEMS = 8;                // sorted items per thread and pass of the large sort

template <typename Id>
__device__ __forceinline__ int id_key(const Id* __restrict__ ids, long i, int rows) {
  const Id v = ids[i];
  return (v < 0 || v >= (Id)rows) ? rows : (int)v;              // everything without a gradient sorts behind the last row
}

// ------------------------------------------------------------------------------------------------ lookup
// A row is handled by a group of `lanes` (a power of two) lanes, E elements a lane and step.
template <typename T, int E, typename Id, int R>
__global__ __launch_bounds__(256) void embedding_lookup_kernel(const T* __restrict__ table, long ld, int rows, int dim,
                                                               const Id* __restrict__ ids, long n, int lanes_log2,
                                                               float scale, T* __restrict__ out) {
  const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1);
  const int groups = 256 >> lanes_log2;
  const long first = (long)blockIdx.x * groups * R + (threadIdx.x >> lanes_log2);
  const int packs = dim / E;
  long id[R];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const long row = first + (long)k * groups;
    id[k] = row < n ? (long)ids[row] : -1;
  }
  for (int c = lane + blockIdx.y * lanes; c < packs; c += lanes * gridDim.y) {
    float v[R][E];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      if (id[k] >= 0 && id[k] < rows) {
        load_pack<T, E>(table + id[k] * ld + (long)c * E, v[k]);
      } else {
        const float fill = id[k] < 0 ? 0.f : __builtin_nanf("");
#pragma unroll
        for (int e = 0; e < E; ++e) v[k][e] = fill;
      }
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const long row = first + (long)k * groups;
      if (row >= n) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) v[k][e] *= scale;
      store_pack<T, E>(out + row * dim + (long)c * E, v[k]);
    }
  }
}

// Pooled: `split` groups share a bag's tokens (1: a group a bag) and are joined through LDS in a fixed order.
template <typename T, int E, typename Id>
__global__ __launch_bounds__(256) void embedding_bag_kernel(const T* __restrict__ table, long ld, int rows, int dim,
                                                            const Id* __restrict__ ids, long bags, int tokens, int lanes_log2,
                                                            int split_log2, bool mean, float scale, T* __restrict__ out) {
  __shared__ float s_acc[256 * E];
  __shared__ int s_count[256];
  const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1);
  const int group = threadIdx.x >> lanes_log2, split = 1 << split_log2;
  const int part = group & (split - 1);
  const long bag = (long)blockIdx.x * (256 >> (lanes_log2 + split_log2)) + (group >> split_log2);
  const int packs = dim / E;
  const Id* my = ids + bag * tokens;
  for (int c0 = blockIdx.y * lanes; c0 < packs; c0 += lanes * gridDim.y) {
    const int c = c0 + lane;
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    int count = 0;
    if (bag < bags) {
      for (int t = part; t < tokens; t += 4 * split) {
        long id[4];
        float v[4][E];
#pragma unroll
        for (int k = 0; k < 4; ++k) id[k] = t + k * split < tokens ? (long)my[t + k * split] : -1;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (id[k] >= 0 && id[k] < rows && c < packs) {
            load_pack<T, E>(table + id[k] * ld + (long)c * E, v[k]);
          } else {
            const float fill = id[k] < 0 ? 0.f : __builtin_nanf("");
#pragma unroll
            for (int e = 0; e < E; ++e) v[k][e] = fill;
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          count += id[k] >= 0 ? 1 : 0;
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += v[k][e];
        }
      }
    }
    if (split > 1) {
      __syncthreads();                                          // the last column step's readers are done
#pragma unroll
      for (int e = 0; e < E; ++e) s_acc[e * 256 + threadIdx.x] = acc[e];
      s_count[threadIdx.x] = count;
      __syncthreads();
      if (part == 0) {
        for (int p = 1; p < split; ++p) {
#pragma unroll
          for (int e = 0; e < E; ++e) acc[e] += s_acc[e * 256 + threadIdx.x + (p << lanes_log2)];
          count += s_count[threadIdx.x + (p << lanes_log2)];
        }
      }
    }
    if (part == 0 && bag < bags && c < packs) {
      const float f = mean ? scale / (float)(count > 0 ? count : 1) : scale;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= f;
      store_pack<T, E>(out + bag * dim + (long)c * E, acc);
    }
  }
}

// Per-bag factor of the mean combiner's gradient: scale / #{t : id >= 0}.
template <typename Id>
__global__ __launch_bounds__(256) void embedding_factor_kernel(const Id* __restrict__ ids, long bags, int tokens, float scale,
                                                               float* __restrict__ factor) {
  const long bag = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (bag >= bags) return;
  int count = 0;
  for (int t = threadIdx.x & 63; t < tokens; t += 64) count += ids[bag * tokens + t] >= 0 ? 1 : 0;
  count = wave_sum_i(count);
  if ((threadIdx.x & 63) == 0) factor[bag] = scale / (float)(count > 0 ? count : 1);
}

// ------------------------------------------------------------------------------------------------ sort
// Lanes of the wave whose digit equals this lane's (`live` lanes only).
__device__ __forceinline__ uint64_t same_digit(int digit, int bits, bool live) {
  uint64_t m = __ballot(live);
  for (int b = 0; b < bits; ++b) {
    const uint64_t one = __ballot((digit >> b) & 1);
    m &= ((digit >> b) & 1) ? one : ~one;
  }
  return m;
}

// Place of this lane's item among the items of the same digit that the wave has seen, in lane order; `counts` (one counter a
// digit, this wave's own) is advanced.
__device__ __forceinline__ int wave_place(int digit, int bits, bool live, int* counts) {
  const int lane = threadIdx.x & 63;
  const uint64_t peers = same_digit(digit, bits, live);
  const int leader = live ? __ffsll((unsigned long long)peers) - 1 : lane;
  int before = 0;
  if (live && lane == leader) before = atomicAdd(&counts[digit], __popcll(peers));
  before = __shfl(before, leader, 64);
  return before + __popcll(peers & ((1ull << lane) - 1ull));
}

// Exclusive prefix sum over `n` (<= 1024) values, one a thread, of a 1024-thread workgroup; `red` holds 16 ints.
__device__ __forceinline__ int block_exclusive_1024(int v, int* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) red[wave] = x;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < wave; ++w) base += red[w];
  return base + x - v;
}

// One workgroup sorts up to SMALL_SORT (id, position) pairs, 8 bits a pass.
template <typename Id>
__global__ __launch_bounds__(1024) void embedding_sort_small_kernel(const Id* __restrict__ ids, int n, int rows, int bits,
                                                                    int* __restrict__ keys_out, int* __restrict__ pos_out) {
  __shared__ uint64_t s_item[SMALL_SORT];
  __shared__ int s_count[16 * 256];
  __shared__ int s_red[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint64_t item[4];
  int place[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = wave * 256 + k * 64 + lane;
    item[k] = i < n ? ((uint64_t)(uint32_t)id_key(ids, i, rows) << 32) | (uint32_t)i : ~0ull;
  }
  for (int shift = 0; shift < bits; shift += 8) {
    for (int i = tid; i < 16 * 256; i += 1024) s_count[i] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k)
      place[k] = wave_place((int)(item[k] >> (32 + shift)) & 255, 8, item[k] != ~0ull, s_count + wave * 256);
    __syncthreads();
    int total = 0;                                              // digit tid: counts of the waves before, and of all
    if (tid < 256) {
      for (int w = 0; w < 16; ++w) {
        const int c = s_count[w * 256 + tid];
        s_count[w * 256 + tid] = total;
        total += c;
      }
    }
    const int base = block_exclusive_1024(tid < 256 ? total : 0, s_red);
    if (tid < 256)
      for (int w = 0; w < 16; ++w) s_count[w * 256 + tid] += base;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (item[k] != ~0ull) s_item[s_count[wave * 256 + ((int)(item[k] >> (32 + shift)) & 255)] + place[k]] = item[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = wave * 256 + k * 64 + lane;
      if (i < n) item[k] = s_item[i];
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int i = wave * 256 + k * 64 + lane;
    if (i < n) {
      keys_out[i] = (int)(item[k] >> 32);
      pos_out[i] = (int)(uint32_t)item[k];
    }
  }
}

// The large sort, one pass = digit counts of every tile, then the scatter; a tile is 1024 * ITEMS consecutive items.
// FIRST: the keys are the ids themselves, and the positions their indexes.
template <typename Id, bool FIRST>
__global__ __launch_bounds__(1024) void embedding_digits_kernel(const Id* __restrict__ ids, const int* __restrict__ keys, int n,
                                                                int rows, int shift, int bits, int* __restrict__ counts) {
  extern __shared__ int s_bins[];
  const int bins = 1 << bits;
  for (int i = threadIdx.x; i < bins; i += 1024) s_bins[i] = 0;
  __syncthreads();
  const long base = (long)blockIdx.x * (1024 * ITEMS);
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const long i = base + k * 1024 + threadIdx.x;
    if (i < n) atomicAdd(&s_bins[((FIRST ? id_key(ids, i, rows) : keys[i]) >> shift) & (bins - 1)], 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < bins; i += 1024) counts[(long)blockIdx.x * bins + i] = s_bins[i];
}

template <typename Id, bool FIRST>
__global__ __launch_bounds__(1024) void embedding_scatter_kernel(const Id* __restrict__ ids, const int* __restrict__ keys,
                                                                 const int* __restrict__ pos, int n, int rows, int shift,
                                                                 int bits, const int* __restrict__ counts, int* __restrict__ keys_out,
                                                                 int* __restrict__ pos_out) {
  extern __shared__ int s_count[];                              // [16][bins], then the 16 ints of the prefix sum
  const int bins = 1 << bits, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int* red = s_count + 16 * bins;
  for (int i = tid; i < 16 * bins; i += 1024) s_count[i] = 0;
  __syncthreads();
  const long base = (long)blockIdx.x * (1024 * ITEMS) + wave * (64 * ITEMS);
  int key[ITEMS], place[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const long i = base + k * 64 + lane;
    key[k] = i < n ? (FIRST ? id_key(ids, i, rows) : keys[i]) : -1;
  }
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) place[k] = wave_place((key[k] >> shift) & (bins - 1), bits, key[k] >= 0, s_count + wave * bins);
  __syncthreads();
  int before = 0, total = 0;
  if (tid < bins) {
    for (int t = 0; t < (int)gridDim.x; ++t) {
      const int c = counts[(long)t * bins + tid];
      before += t < (int)blockIdx.x ? c : 0;
      total += c;
    }
  }
  before += block_exclusive_1024(total, red);
  if (tid < bins) {
    for (int w = 0; w < 16; ++w) {
      const int c = s_count[w * bins + tid];
      s_count[w * bins + tid] = before;
      before += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    if (key[k] < 0) continue;
    const int to = s_count[wave * bins + ((key[k] >> shift) & (bins - 1))] + place[k];
    keys_out[to] = key[k];
    pos_out[to] = FIRST ? (int)(base + k * 64 + lane) : pos[base + k * 64 + lane];
  }
}

// ------------------------------------------------------------------------------------------------ gradient
struct GradArgs {
  const int* keys;                      // [n] sorted ids
  const int* pos;                       // [n] the lookup that each came from
  const float* factor;                  // [bags] or null: scale for all
  float* chunks;                        // [n / CHUNK][dim] sums of the chunks that hold one token
  int n, rows, dim, tokens, lanes_log2, wave_rows;
  float scale;
};

// Adds f_b * g[b] of the sorted occurrences first, first + step, ... < end to acc.
template <typename T, int E>
__device__ __forceinline__ void add_rows(const GradArgs& a, const T* __restrict__ grad, int first, int end, int step, int c, float (&acc)[E]) {
  for (int i = first; i < end; i += 4 * step) {
    int b[4];
    float v[4][E], f[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int at = i + k * step;
      b[k] = at < end ? a.pos[at] : -1;
      if (a.tokens > 1 && b[k] >= 0) b[k] = (int)((unsigned)b[k] / (unsigned)a.tokens);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (b[k] >= 0) {
        load_pack<T, E>(grad + (long)b[k] * a.dim + (long)c * E, v[k]);
        f[k] = a.factor ? a.factor[b[k]] : 1.f;
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[k][e] = 0.f;
        f[k] = 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = b[k] >= 0 ? __builtin_fmaf(f[k], v[k][e], acc[e]) : acc[e];
  }
}

// Joins the groups' sums through LDS in group order; the result is group 0's.
template <int E>
__device__ __forceinline__ void join_groups(float* s_acc, int lanes_log2, float (&acc)[E]) {
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) s_acc[e * 256 + threadIdx.x] = acc[e];
  __syncthreads();
  if ((threadIdx.x >> lanes_log2) == 0) {
    for (int p = 1; p < (256 >> lanes_log2); ++p)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += s_acc[e * 256 + threadIdx.x + (p << lanes_log2)];
  }
}

template <typename T, int E>
__global__ __launch_bounds__(256) void embedding_chunk_kernel(const GradArgs a, const T* __restrict__ grad) {
  __shared__ float s_acc[256 * E];
  const int first = blockIdx.x * CHUNK;
  const int key = a.keys[first];
  if (key >= a.rows || a.keys[first + CHUNK - 1] != key) return;         // the same for the whole workgroup
  const int lane = threadIdx.x & ((1 << a.lanes_log2) - 1), group = threadIdx.x >> a.lanes_log2;
  const int packs = a.dim / E;
  for (int c0 = 0; c0 < packs; c0 += 1 << a.lanes_log2) {
    const int c = c0 + lane;
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    if (c < packs) add_rows<T, E>(a, grad, first + group, first + CHUNK, 256 >> a.lanes_log2, c, acc);
    join_groups<E>(s_acc, a.lanes_log2, acc);
    if (group == 0 && c < packs) store_pack<float, E>(a.chunks + (long)blockIdx.x * a.dim + (long)c * E, acc);
  }
}

// First index of the sorted keys that is not below `row`: 64 probes a step, the whole wave together.
__device__ __forceinline__ int wave_lower_bound(const int* __restrict__ keys, int n, int row) {
  const int lane = threadIdx.x & 63;
  int lo = 0, len = n;                                          // the answer is in [lo, lo + len]
  while (len > 0) {
    const int step = (len + 63) / 64;
    const int at = lo + lane * step + step - 1;                 // the last key of this lane's part
    const bool below = lane * step < len && keys[at < lo + len ? at : lo + len - 1] < row;
    const int whole = __popcll(__ballot(below));                // parts that lie below as a whole
    const int next = lo + whole * step;
    if (next >= lo + len) return lo + len;
    const int left = lo + len - next;
    lo = next;
    len = step == 1 ? 0 : (left < step ? left : step) - 1;      // the part's last key is not below
  }
  return lo;
}

template <typename T, int E>
__global__ __launch_bounds__(256) void embedding_rows_kernel(const GradArgs a, const T* __restrict__ grad, T* __restrict__ out) {
  __shared__ float s_acc[256 * E];
  __shared__ int s_bound[4][65];
  __shared__ int s_heavy[4 * 64], s_heavies;
  const int wave = threadIdx.x >> 6, wlane = threadIdx.x & 63;
  const int lanes = 1 << a.lanes_log2, lane = threadIdx.x & (lanes - 1);
  const int packs = a.dim / E;
  const long r0 = ((long)blockIdx.x * 4 + wave) * a.wave_rows;
  if (threadIdx.x == 0) s_heavies = 0;
  __syncthreads();
  if (r0 < a.rows) {
    const int many = (int)(a.rows - r0 < a.wave_rows ? a.rows - r0 : a.wave_rows);
    const int lo = wave_lower_bound(a.keys, a.n, (int)r0);
    const int hi = wave_lower_bound(a.keys + lo, a.n - lo, (int)r0 + many) + lo;
    int b0 = lo, b1 = hi;                                       // first key of row r0 + wlane
    while (b0 < b1) {
      const int mid = (b0 + b1) >> 1;
      if (a.keys[mid] < (int)r0 + wlane) b0 = mid + 1; else b1 = mid;
    }
    s_bound[wave][wlane] = wlane < many ? b0 : hi;
    if (wlane == 0) s_bound[wave][64] = hi;
  }
  __syncthreads();
  if (r0 < a.rows) {
    const int many = (int)(a.rows - r0 < a.wave_rows ? a.rows - r0 : a.wave_rows);
    for (int r = wlane >> a.lanes_log2; r < many; r += 64 >> a.lanes_log2) {
      const int s = s_bound[wave][r], e = s_bound[wave][r + 1];
      if (e - s > HEAVY) {
        if (lane == 0) s_heavy[atomicAdd(&s_heavies, 1)] = wave * 64 + r;
        continue;
      }
      T* row = out + (r0 + r) * a.dim;
      for (int c = lane; c < packs; c += lanes) {
        float acc[E];
#pragma unroll
        for (int k = 0; k < E; ++k) acc[k] = 0.f;
        add_rows<T, E>(a, grad, s, e, 1, c, acc);
        if (!a.factor) {
#pragma unroll
          for (int k = 0; k < E; ++k) acc[k] *= a.scale;
        }
        store_pack<T, E>(row + (long)c * E, acc);
      }
    }
  }
  __syncthreads();
  const int group = threadIdx.x >> a.lanes_log2, groups = 256 >> a.lanes_log2;
  for (int h = 0; h < s_heavies; ++h) {                         // the list's order does not touch a row's own sum
    const int w = s_heavy[h] >> 6, r = s_heavy[h] & 63;
    const int s = s_bound[w][r], e = s_bound[w][r + 1];
    const int whole0 = (s + CHUNK - 1) / CHUNK, whole1 = e / CHUNK;      // the chunks that lie inside
    T* row = out + (((long)blockIdx.x * 4 + w) * a.wave_rows + r) * a.dim;
    for (int c0 = 0; c0 < packs; c0 += lanes) {
      const int c = c0 + lane;
      float acc[E];
#pragma unroll
      for (int k = 0; k < E; ++k) acc[k] = 0.f;
      if (c < packs) {
        if (whole1 > whole0) {
          add_rows<T, E>(a, grad, s + group, whole0 * CHUNK, groups, c, acc);
          for (int q = whole0 + group; q < whole1; q += groups) {
            float v[E];
            load_pack<float, E>(a.chunks + (long)q * a.dim + (long)c * E, v);
#pragma unroll
            for (int k = 0; k < E; ++k) acc[k] += v[k];
          }
          add_rows<T, E>(a, grad, whole1 * CHUNK + group, e, groups, c, acc);
        } else {
          add_rows<T, E>(a, grad, s + group, e, groups, c, acc);
        }
      }
      join_groups<E>(s_acc, a.lanes_log2, acc);
      if (group == 0 && c < packs) {
        if (!a.factor) {
#pragma unroll
          for (int k = 0; k < E; ++k) acc[k] *= a.scale;
        }
        store_pack<T, E>(row + (long)c * E, acc);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ host
int log2_ceil(long n) {
  int k = 0;
  while ((1l << k) < n) ++k;
  return k;
}

// Widest access, in elements, that the row length, the leading dimensions and the addresses allow: 16 bytes, 4 bytes or one element.
int pack_elems(int dtype, int dim, long ld, const void* p, const void* q) {
  const int b = elem_bytes(dtype);
  for (int w : {16, 4}) {
    const int e = w / b;
    if (e > 1 && dim % e == 0 && ld % e == 0 && ((uintptr_t)p % w) == 0 && ((uintptr_t)q % w) == 0) return e;
  }
  return 1;
}

struct Sizes {
  long keys, pos, keys2, pos2, counts, factor, chunks, total;   // byte offsets
  int tiles, bits, passes;
};

Sizes sizes_of(long n, long bags, long rows, int dim, bool mean) {
  Sizes s;
  s.bits = log2_ceil(rows + 1);
  if (s.bits < 1) s.bits = 1;
  s.passes = (s.bits + 9) / 10;
  s.tiles = (int)((n + 1024 * ITEMS - 1) / (1024 * ITEMS));
  const int digit = (s.bits + s.passes - 1) / s.passes;
  long at = 0;
  auto take = [&at](long bytes) { const long p = at; at += (bytes + 255) / 256 * 256; return p; };
  s.keys = take(4 * n);
  s.pos = take(4 * n);
  const bool large = n > SMALL_SORT;
  s.keys2 = take(large ? 4 * n : 0);
  s.pos2 = take(large ? 4 * n : 0);
  s.counts = take(large ? 4l * s.tiles << digit : 0);
  s.factor = take(mean ? 4 * bags : 0);
  s.chunks = take(4 * (n / CHUNK) * (long)dim);
  s.total = at;
  return s;
}

template <typename T, int E, typename Id>
int launch_lookup(const T* table, long ld, int rows, int dim, const Id* ids, long bags, int tokens, int combiner, float scale, T* out,
                  hipStream_t stream) {
  const int packs = dim / E;
  const int lg = log2_ceil(packs < 64 ? packs : 64);
  const int groups = 256 >> lg;
  if (combiner == TFR_COMBINER_NONE) {
    // Few lookups: a row's columns are spread over workgroups too; many: four rows of a group are in flight together.
    if (bags >= 4l * groups * 1024) {
      embedding_lookup_kernel<T, E, Id, 4><<<dim3((unsigned)((bags + 4 * groups - 1) / (4 * groups))), 256, 0, stream>>>(
          table, ld, rows, dim, ids, bags, lg, scale, out);
    } else {
      int y = (packs + (1 << lg) - 1) >> lg;
      if (y > 16) y = 16;
      embedding_lookup_kernel<T, E, Id, 1><<<dim3((unsigned)((bags + groups - 1) / groups), y), 256, 0, stream>>>(
          table, ld, rows, dim, ids, bags, lg, scale, out);
    }
  } else {
    int split = 0;                       // few bags: share a bag's tokens among groups, at least eight tokens each
    while ((2 << split) <= groups && (bags << split) * (packs >> lg > 0 ? packs >> lg : 1) < 8192 && (tokens >> (split + 1)) >= 8) ++split;
    int y = (packs + (1 << lg) - 1) >> lg;
    if (y > 16) y = 16;
    const long per = 256 >> (lg + split);
    embedding_bag_kernel<T, E, Id><<<dim3((unsigned)((bags + per - 1) / per), y), 256, 0, stream>>>(
        table, ld, rows, dim, ids, bags, tokens, lg, split, combiner == TFR_COMBINER_MEAN, scale, out);
  }
  return (int)hipGetLastError();
}

template <typename T, int E>
int launch_lookup_ids(const void* table, long ld, int rows, int dim, const void* ids, int id_type, long bags, int tokens, int combiner,
                      float scale, void* out, hipStream_t stream) {
  if (id_type == TFR_IDS_I32)
    return launch_lookup<T, E, int32_t>((const T*)table, ld, rows, dim, (const int32_t*)ids, bags, tokens, combiner, scale, (T*)out, stream);
  return launch_lookup<T, E, int64_t>((const T*)table, ld, rows, dim, (const int64_t*)ids, bags, tokens, combiner, scale, (T*)out, stream);
}

template <typename Id>
int launch_sort(const Id* ids, long n, int rows, const Sizes& s, char* ws, int** keys, int** pos, hipStream_t stream) {
  int* k[2] = {(int*)(ws + s.keys), (int*)(ws + s.keys2)};
  int* p[2] = {(int*)(ws + s.pos), (int*)(ws + s.pos2)};
  if (n <= SMALL_SORT) {
    embedding_sort_small_kernel<Id><<<1, 1024, 0, stream>>>(ids, (int)n, rows, s.bits, k[0], p[0]);
    *keys = k[0];
    *pos = p[0];
    return (int)hipGetLastError();
  }
  int* counts = (int*)(ws + s.counts);
  const int digit = (s.bits + s.passes - 1) / s.passes;
  const size_t lds = (16 * (size_t)(1 << digit) + 16) * sizeof(int);
  int from = 0;
  for (int pass = 0; pass < s.passes; ++pass) {
    const int shift = pass * digit, to = from ^ 1;
    if (pass == 0) {
      embedding_digits_kernel<Id, true><<<s.tiles, 1024, sizeof(int) << digit, stream>>>(ids, nullptr, (int)n, rows, shift, digit, counts);
      if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void*)embedding_scatter_kernel<Id, true>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return (int)e;
      }
      embedding_scatter_kernel<Id, true><<<s.tiles, 1024, lds, stream>>>(ids, nullptr, nullptr, (int)n, rows, shift, digit, counts, k[0], p[0]);
      from = 0;
    } else {
      embedding_digits_kernel<Id, false><<<s.tiles, 1024, sizeof(int) << digit, stream>>>(ids, k[from], (int)n, rows, shift, digit, counts);
      if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void*)embedding_scatter_kernel<Id, false>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return (int)e;
      }
      embedding_scatter_kernel<Id, false><<<s.tiles, 1024, lds, stream>>>(ids, k[from], p[from], (int)n, rows, shift, digit, counts, k[to], p[to]);
      from = to;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  *keys = k[from];
  *pos = p[from];
  return TFR_OK;
}

template <typename T, int E>
int launch_grad(GradArgs a, const void* grad, void* out, hipStream_t stream) {
  const int packs = a.dim / E;
  a.lanes_log2 = log2_ceil(packs < 64 ? packs : 64);
  // A wave owns rows of about 8 KB in all: enough to hide its search, and the rows of a wide table still fill the card.
  int wr = 4;
  while (wr < 64 && (long)(2 * wr) * a.dim * (long)sizeof(T) <= 8192) wr *= 2;
  if (wr < (64 >> a.lanes_log2)) wr = 64 >> a.lanes_log2;
  a.wave_rows = wr;
  const int chunks = a.n / CHUNK;
  if (chunks > 0) embedding_chunk_kernel<T, E><<<chunks, 256, 0, stream>>>(a, (const T*)grad);
  embedding_rows_kernel<T, E><<<(unsigned)((a.rows + 4l * wr - 1) / (4l * wr)), 256, 0, stream>>>(a, (const T*)grad, (T*)out);
  return (int)hipGetLastError();
}

constexpr long kMost = 1l << 25;        // rows, bags and lookups: no grid gets 2^32 threads, and indexes stay in 32 bits

int check_args(long rows, int dim, int dtype, int id_type, long bags, int tokens, int combiner) {
  if (!elem_known(dtype) || (id_type != TFR_IDS_I32 && id_type != TFR_IDS_I64)) return TFR_EINVAL;
  if (rows < 0 || rows > kMost || dim < 1 || bags < 0 || tokens < 0) return TFR_EINVAL;
  if (combiner != TFR_COMBINER_NONE && combiner != TFR_COMBINER_SUM && combiner != TFR_COMBINER_MEAN) return TFR_EINVAL;
  if (combiner == TFR_COMBINER_NONE && tokens != 1) return TFR_EINVAL;
  if (bags > kMost || (tokens > 0 && bags > kMost / tokens)) return TFR_EINVAL;
  return TFR_OK;
}

}  // namespace

extern "C" int tfr_embedding_lookup(const void* table, long ld, long rows, int dim, int dtype, const void* ids, int id_type, long bags,
                                    int tokens, int combiner, float scale, void* out, void* stream) {
  const int rc = check_args(rows, dim, dtype, id_type, bags, tokens, combiner);
  if (rc != TFR_OK) return rc;
  if (ld < dim) return TFR_EINVAL;
  if (bags == 0) return TFR_OK;
  if (!out || (rows > 0 && !table) || (tokens > 0 && !ids)) return TFR_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  const int e = pack_elems(dtype, dim, ld, table, out), r = (int)rows;
  if (dtype == TFR_DTYPE_F32)
    return e == 4 ? launch_lookup_ids<float, 4>(table, ld, r, dim, ids, id_type, bags, tokens, combiner, scale, out, st)
                  : launch_lookup_ids<float, 1>(table, ld, r, dim, ids, id_type, bags, tokens, combiner, scale, out, st);
  if (dtype == TFR_DTYPE_BF16)
    return e == 8   ? launch_lookup_ids<__bf16, 8>(table, ld, r, dim, ids, id_type, bags, tokens, combiner, scale, out, st)
           : e == 2 ? launch_lookup_ids<__bf16, 2>(table, ld, r, dim, ids, id_type, bags, tokens, combiner, scale, out, st)
                    : launch_lookup_ids<__bf16, 1>(table, ld, r, dim, ids, id_type, bags, tokens, combiner, scale, out, st);
  return e == 8   ? launch_lookup_ids<_Float16, 8>(table, ld, r, dim, ids, id_type, bags, tokens, combiner, scale, out, st)
         : e == 2 ? launch_lookup_ids<_Float16, 2>(table, ld, r, dim, ids, id_type, bags, tokens, combiner, scale, out, st)
                  : launch_lookup_ids<_Float16, 1>(table, ld, r, dim, ids, id_type, bags, tokens, combiner, scale, out, st);
}

extern "C" long tfr_embedding_grad_workspace_bytes(long rows, int dim, long bags, int tokens, int combiner) {
  if (check_args(rows, dim, TFR_DTYPE_F32, TFR_IDS_I32, bags, tokens, combiner) != TFR_OK) return TFR_EINVAL;
  return sizes_of(bags * tokens, bags, rows, dim, combiner == TFR_COMBINER_MEAN).total;
}

extern "C" int tfr_embedding_grad(const void* grad, int dtype, const void* ids, int id_type, long bags, int tokens, int combiner,
                                  float scale, long rows, int dim, void* grad_table, void* workspace, long workspace_bytes,
                                  void* stream) {
  int rc = check_args(rows, dim, dtype, id_type, bags, tokens, combiner);
  if (rc != TFR_OK) return rc;
  if (rows == 0) return TFR_OK;
  const long n = bags * tokens;
  const bool mean = combiner == TFR_COMBINER_MEAN;
  const Sizes s = sizes_of(n, bags, rows, dim, mean);
  if (!grad_table || (n > 0 && (!grad || !ids))) return TFR_EINVAL;
  if (s.total > 0 && (!workspace || workspace_bytes < s.total || ((uintptr_t)workspace & 15))) return TFR_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  GradArgs a = {};
  a.n = (int)n;
  a.rows = (int)rows;
  a.dim = dim;
  a.tokens = tokens;
  a.scale = scale;
  char* ws = (char*)workspace;
  if (n > 0) {
    if (mean) {
      a.factor = (const float*)(ws + s.factor);
      if (id_type == TFR_IDS_I32)
        embedding_factor_kernel<int32_t><<<(unsigned)((bags + 3) / 4), 256, 0, st>>>((const int32_t*)ids, bags, tokens, scale, (float*)(ws + s.factor));
      else
        embedding_factor_kernel<int64_t><<<(unsigned)((bags + 3) / 4), 256, 0, st>>>((const int64_t*)ids, bags, tokens, scale, (float*)(ws + s.factor));
    }
    int *keys = nullptr, *pos = nullptr;
    rc = id_type == TFR_IDS_I32 ? launch_sort<int32_t>((const int32_t*)ids, n, a.rows, s, ws, &keys, &pos, st)
                                : launch_sort<int64_t>((const int64_t*)ids, n, a.rows, s, ws, &keys, &pos, st);
    if (rc != TFR_OK) return rc;
    a.keys = keys;
    a.pos = pos;
    a.chunks = (float*)(ws + s.chunks);
  }
  const int e = pack_elems(dtype, dim, dim, n > 0 ? grad : grad_table, grad_table);
  if (dtype == TFR_DTYPE_F32) return e == 4 ? launch_grad<float, 4>(a, grad, grad_table, st) : launch_grad<float, 1>(a, grad, grad_table, st);
  if (dtype == TFR_DTYPE_BF16)
    return e == 8   ? launch_grad<__bf16, 8>(a, grad, grad_table, st)
           : e == 2 ? launch_grad<__bf16, 2>(a, grad, grad_table, st)
                    : launch_grad<__bf16, 1>(a, grad, grad_table, st);
  return e == 8   ? launch_grad<_Float16, 8>(a, grad, grad_table, st)
         : e == 2 ? launch_grad<_Float16, 2>(a, grad, grad_table, st)
                  : launch_grad<_Float16, 1>(a, grad, grad_table, st);
}
