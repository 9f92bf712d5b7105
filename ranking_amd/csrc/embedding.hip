// Embedding lookup with scaling, and its gradient by sorted tokens (gfx950).
//
//   lookup   out[b] = f_b * sum_t W[id_bt]      f_b = scale (no combiner: one token a row; sum) or scale / #{t : id_bt >= 0} (mean)
//   gradient dW[v]  = sum over the occurrences (b, t) of v of f_b * g[b]
//
// An id below 0 is padding: a zero row, no gradient.  An id beyond the table gives a row of NaN and no gradient: nothing
// outside the table is read.
//
// The gradient writes every row of dW exactly once and adds in an order that depends on the ids alone: no atomics on floating
// point, no separate zero fill of rows that are written anyway.
//   1. The occurrences are sorted by id (stable radix sort, least significant digit first, at most 10 bits a pass).
//   2. A group of lanes walks a chunk of the sorted list (16 .. 128 occurrences) and adds the rows of each run of equal ids: a run
//      that lies inside its chunk is a finished row of dW; the part of a run that crosses a chunk's border is left as a partial
//      sum.  The work is cut by occurrences and not by rows, so a token that is 6 % of the batch costs what the others cost.
//   3. Runs that cross borders are joined from their partial sums, and rows without an occurrence are filled with zeros.
// Steps 2 and 3 are bound by HBM: 262 144 x 2048 bf16 into 131 072 rows 259 + 74 us (1.07 GB read, 0.54 GB written: 4.8 TB/s),
// 16 384 x 1024 into 65 536 rows 15 + 18 us; the lookups before them 328 and 11 us.
#include "common.h"
#include "elem.h"

using namespace tfr;

namespace {

constexpr int LONG_RUN = 16;            // partial sums from which the whole workgroup joins a run
constexpr int SMALL_SORT = 4096;        // lookups that one workgroup sorts in LDS (9 us; 16 384 of them: 33 us, by the large sort 25)
constexpr int ITEMS = 4;                // items a thread of the large sort holds

template <typename Id>
__device__ __forceinline__ int id_key(const Id* __restrict__ ids, long i, int rows) {
  const Id v = ids[i];
  return (v < 0 || v >= (Id)rows) ? rows : (int)v;              // everything without a gradient sorts behind the last row
}

// ------------------------------------------------------------------------------------------------ lookup
// A group of `lanes` (a power of two) lanes takes one step of a row, E elements a lane; the steps of a row are neighbours, so that a
// workgroup moves whole rows.  One row a group: 8 rows of a group in flight together were slower (262 144 x 2048 bf16: 454 us for
// 378).  STREAM: results beyond the L2 caches go past them (352 us for 378, and the gradient's kernels behind gain 10 us too).
template <typename T, int E, typename Id, bool STREAM>
__global__ __launch_bounds__(256) void embedding_lookup_kernel(const T* __restrict__ table, long ld, int rows, int dim,
                                                               const Id* __restrict__ ids, unsigned jobs, unsigned steps, int lanes_log2,
                                                               float scale, T* __restrict__ out) {
  const unsigned job = blockIdx.x * (256u >> lanes_log2) + (threadIdx.x >> lanes_log2);
  if (job >= jobs) return;
  const unsigned row = job / steps;
  const int c = (int)((job - row * steps) << lanes_log2) + (int)(threadIdx.x & ((1u << lanes_log2) - 1u));
  if (c >= dim / E) return;
  const long id = (long)ids[row];
  float v[E];
  if (id >= 0 && id < rows) {
    load_pack<T, E>(table + id * ld + (long)c * E, v);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] *= scale;
  } else {
    const float fill = id < 0 ? 0.f : __builtin_nanf("");
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = fill;
  }
  if (STREAM) store_pack_stream<T, E>(out + (long)row * dim + (long)c * E, v);
  else store_pack<T, E>(out + (long)row * dim + (long)c * E, v);
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

// ------------------------------------------------------------------------------------------------ sort
// Place of this lane's item among the items of the same digit that the wave has seen, in lane order; `counts` (one counter a
// digit, this wave's own) is advanced.  The lanes of the same digit are found bit by bit; every lane reads its counter and the
// first of the lanes advances it: LDS serves a wave's accesses in order, so neither waits for the other.
__device__ __forceinline__ int wave_place(int digit, int bits, bool live, int* counts) {
  const uint64_t alive = __ballot(live);
  uint32_t lo = (uint32_t)alive, hi = (uint32_t)(alive >> 32);
  for (int b = 0; b < bits; ++b) {
    const uint32_t mine = (uint32_t)((digit << (31 - b)) >> 31);          // all ones where the bit is set
    const uint64_t set = __ballot(mine != 0);
    lo &= ~((uint32_t)set ^ mine);
    hi &= ~((uint32_t)(set >> 32) ^ mine);
  }
  const int below = __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0));
  const int before = counts[digit];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  if (live && below == 0) atomicAdd(&counts[digit], __popc(lo) + __popc(hi));
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  return before + below;
}

// Exclusive prefix sum over one value a thread; `red` holds 16 ints.
__device__ __forceinline__ int block_exclusive(int v, int* red) {
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

// What the first launch of a gradient does beside sorting, on workgroups of its own: every row's first occurrence is set to
// "none", and the mean combiner's factor of every bag, scale / #{t : id >= 0}, is counted.
struct Prepare {
  int* first;
  float* factor;
  long bags;
  int rows, tokens;
  float scale;
};

template <typename Id>
__device__ __forceinline__ void prepare_rows(const Prepare& p, const Id* __restrict__ ids, int block, int blocks) {
  for (long r = (long)block * blockDim.x + threadIdx.x; r < p.rows; r += (long)blocks * blockDim.x) p.first[r] = -1;
  if (!p.factor) return;
  const int waves = blockDim.x >> 6;
  for (long bag = (long)block * waves + (threadIdx.x >> 6); bag < p.bags; bag += (long)blocks * waves) {
    int count = 0;
    for (int t = threadIdx.x & 63; t < p.tokens; t += 64) count += ids[bag * p.tokens + t] >= 0 ? 1 : 0;
    count = wave_sum_i(count);
    if ((threadIdx.x & 63) == 0) p.factor[bag] = p.scale / (float)(count > 0 ? count : 1);
  }
}

// Workgroup 0 sorts up to SMALL_SORT (id, position) pairs, 8 bits a pass; the others prepare the rows.
template <typename Id>
__global__ __launch_bounds__(1024) void embedding_sort_small_kernel(const Id* __restrict__ ids, int n, int rows, int bits, int per_bag, const Prepare prep,
                                                                    int2* __restrict__ out) {
  if (blockIdx.x > 0) {
    prepare_rows(prep, ids, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
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
    const int base = block_exclusive(tid < 256 ? total : 0, s_red);
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
    if (i < n) out[i] = make_int2((int)(item[k] >> 32), (int)((uint32_t)item[k] / (uint32_t)per_bag));
  }
}

// The large sort.  One pass = the digit counts of every tile (a workgroup's `subs` * blockDim.x * ITEMS consecutive items), then
// the scatter, in which a tile adds up the counts of the tiles before it by itself (counts[bin][tile], `pitch` apart) while
// there are few tiles.  The last pass turns positions into bags (per_bag > 1).  FIRST: the keys are the ids themselves, the
// positions their indexes, and the workgroups behind the tiles prepare the rows.
// An id and its position move as one 8-byte item: a tile's items scatter one by one, and it is the number of accesses that counts
// (819 200 lookups: 11 + 9 us the two scatters, 15 + 11 with an array each).
// Bound by latency (a pass is two or three launches of a few dependent round trips): two passes take 24 us at 16 384 lookups, 36 at
// 262 144, 41 at 819 200.
template <typename Id, bool FIRST>
__global__ __launch_bounds__(256) void embedding_digits_kernel(const Id* __restrict__ ids, const int2* __restrict__ items, int n, int rows, int tiles,
                                                                int subs, int shift, int bits, int pitch, const Prepare prep, int* __restrict__ counts) {
  if (FIRST && (int)blockIdx.x >= tiles) {
    prepare_rows(prep, ids, blockIdx.x - tiles, gridDim.x - tiles);
    return;
  }
  extern __shared__ int s_bins[];
  const int bins = 1 << bits;
  for (int i = threadIdx.x; i < bins; i += blockDim.x) s_bins[i] = 0;
  __syncthreads();
  for (int sub = 0; sub < subs; ++sub) {
    const long base = ((long)blockIdx.x * subs + sub) * ((long)blockDim.x * ITEMS);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const long i = base + k * blockDim.x + threadIdx.x;
      if (i < n) atomicAdd(&s_bins[((FIRST ? id_key(ids, i, rows) : items[i].x) >> shift) & (bins - 1)], 1);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < bins; i += blockDim.x) counts[(long)i * pitch + blockIdx.x] = s_bins[i];
}

// Where there are many tiles, between the two: a wave a bin replaces the tiles' counts by the counts before them.
__global__ __launch_bounds__(64) void embedding_scan_kernel(int* __restrict__ counts, int tiles, int pitch, int* __restrict__ totals) {
  const int lane = threadIdx.x;
  int4* c = reinterpret_cast<int4*>(counts + (long)blockIdx.x * pitch);
  int carry = 0;
  for (int t0 = 0; t0 < tiles; t0 += 256) {
    const int t = t0 + 4 * lane;
    int4 v = t < tiles ? c[t / 4] : make_int4(0, 0, 0, 0);
    v.y = t + 1 < tiles ? v.y : 0;
    v.z = t + 2 < tiles ? v.z : 0;
    v.w = t + 3 < tiles ? v.w : 0;
    int x = v.x + v.y + v.z + v.w;
    const int own = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o, 64);
      if (lane >= o) x += y;
    }
    const int at = carry + x - own;
    if (t < tiles) c[t / 4] = make_int4(at, at + v.x, at + v.x + v.y, at + v.x + v.y + v.z);
    carry += __shfl(x, 63, 64);
  }
  if (lane == 0) totals[blockIdx.x] = carry;
}

template <typename Id, bool FIRST>
__global__ __launch_bounds__(256) void embedding_scatter_kernel(const Id* __restrict__ ids, const int2* __restrict__ items, int n,
                                                                 int rows, int subs, int shift, int bits, int pitch, int per_bag,
                                                                 const int* __restrict__ counts, const int* __restrict__ totals,
                                                                 int2* __restrict__ out) {
  extern __shared__ int s_count[];                              // [waves][bins], the 16 ints of the prefix sum, the next place of each bin [bins]
  const int bins = 1 << bits, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
  int* red = s_count + waves * bins;
  int* next = red + 16;
  const int per = bins > (int)blockDim.x ? bins / blockDim.x : 1;        // bins of a thread: 1, 2 or 4, neighbours
  const auto load_items = [&](int sub, int2 (&item)[ITEMS]) {
    const long base = ((long)blockIdx.x * subs + sub) * ((long)blockDim.x * ITEMS) + wave * (64 * ITEMS);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const long i = base + k * 64 + lane;
      item[k] = i >= n ? make_int2(-1, 0) : FIRST ? make_int2(id_key(ids, i, rows), (int)i) : items[i];
    }
  };
  int2 item[ITEMS];
  load_items(0, item);                                            // under way while the counts are added up
  int before[4] = {0, 0, 0, 0}, total[4] = {0, 0, 0, 0};
  if (totals) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j >= per || tid * per >= bins) break;
      before[j] = counts[(long)(tid * per + j) * pitch + blockIdx.x];
      total[j] = totals[tid * per + j];
    }
  } else if (tid * per < bins) {
    const int tiles = gridDim.x, mine = blockIdx.x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j >= per) break;
      const int4* c = reinterpret_cast<const int4*>(counts + (long)(tid * per + j) * pitch);
      for (int t0 = 0; t0 < tiles; t0 += 32) {                  // the counts of a bin lie side by side, padded to whole int4
        int4 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = t0 + 4 * u < tiles ? c[t0 / 4 + u] : make_int4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int t = t0 + 4 * u;
          const int x = t < tiles ? v[u].x : 0, y = t + 1 < tiles ? v[u].y : 0, z = t + 2 < tiles ? v[u].z : 0, w = t + 3 < tiles ? v[u].w : 0;
          before[j] += (t < mine ? x : 0) + (t + 1 < mine ? y : 0) + (t + 2 < mine ? z : 0) + (t + 3 < mine ? w : 0);
          total[j] += x + y + z + w;
        }
      }
    }
  }
  int at = block_exclusive(total[0] + total[1] + total[2] + total[3], red);
  if (tid * per < bins) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j < per) next[tid * per + j] = at + before[j];
      at += total[j];
    }
  }
  for (int sub = 0; sub < subs; ++sub) {
    for (int i = tid; i < waves * bins; i += blockDim.x) s_count[i] = 0;
    __syncthreads();
    int place[ITEMS];
    if (sub > 0) load_items(sub, item);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) place[k] = wave_place((item[k].x >> shift) & (bins - 1), bits, item[k].x >= 0, s_count + wave * bins);
    __syncthreads();
    for (int b = tid; b < bins; b += blockDim.x) {
      int p = next[b];
      for (int w = 0; w < waves; ++w) {
        const int c = s_count[w * bins + b];
        s_count[w * bins + b] = p;
        p += c;
      }
      next[b] = p;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      if (item[k].x < 0) continue;
      const int to = s_count[wave * bins + ((item[k].x >> shift) & (bins - 1))] + place[k];
      out[to] = make_int2(item[k].x, per_bag > 1 ? (int)((unsigned)item[k].y / (unsigned)per_bag) : item[k].y);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ gradient
struct GradArgs {
  const int2* items;                    // [n] sorted ids (rows: no gradient), and the bag that each came from
  const float* factor;                  // [bags] or null: scale for all
  int* first;                           // [rows] where a row's run begins, -1: no occurrence
  int* last;                            // [rows] where it ends (rows with an occurrence)
  void* out;                            // [rows][dim]
  float* parts;                         // [2 * chunks][dim]: of chunk q the run that began before it (2 q) and the one that goes on (2 q + 1)
  int n, rows, dim, chunk_log2, lanes_log2, wave_rows, steps;    // steps: column steps of a group over a row
  float scale;
};

// STREAM: a gradient table beyond the Infinity Cache (256 MB) is written past the caches (131 072 x 2048 bf16: the step's kernels
// 708 -> 657 us in all; 65 536 x 1024, 134 MB: 45 -> 49 us).
template <typename T, int E, bool STREAM>
__device__ __forceinline__ void put_row(T* __restrict__ p, const float (&v)[E]) {
  if (STREAM) store_pack_stream<T, E>(p, v);
  else store_pack<T, E>(p, v);
}

// Step 2: a group of lanes a chunk and column step; the column steps of a chunk are neighbours, so that a workgroup reads whole rows.
// ONCE: every gradient row is read once (no bags), past the caches: 303 -> 262 us for 1 GB of them.  Rows of bags are read again for
// every token (24 -> 36 us past the caches for 25 600 bags of 32).
template <typename T, int E, bool ONCE, bool STREAM>
__global__ __launch_bounds__(256) void embedding_runs_kernel(const GradArgs a, const T* __restrict__ grad) {
  const int lane = threadIdx.x & ((1 << a.lanes_log2) - 1);
  const long block = (long)blockIdx.y * gridDim.x + blockIdx.x;
  const long job = block * (256 >> a.lanes_log2) + (threadIdx.x >> a.lanes_log2);
  const long q = job / a.steps;
  const int column = (int)(job - q * a.steps);
  const long begin = q << a.chunk_log2;
  if (begin >= a.n) return;
  const int lo = (int)begin, hi = a.n - lo < (1 << a.chunk_log2) ? a.n : lo + (1 << a.chunk_log2);
  const int c = (column << a.lanes_log2) + lane;
  const bool on = c < a.dim / E, scribe = lane == 0 && column == 0;
  int row = a.items[lo].x, start = lo;
  bool began_before = lo > 0 && a.items[lo - 1].x == row;
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  // Ends the run of `row` at sorted position `end`; `goes_on`: its next occurrence is the next chunk's first.
  auto finish = [&](int end, bool goes_on) {
    if (row >= a.rows) return;
    if (scribe) {
      if (!began_before) a.first[row] = start;
      if (!goes_on) a.last[row] = end;
    }
    if (!on) return;
    if (began_before || goes_on) {
      store_pack<float, E>(a.parts + (2 * q + (began_before ? 0 : 1)) * a.dim + (long)c * E, acc);
    } else {
      float v[E];
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = a.factor ? acc[e] : acc[e] * a.scale;
      put_row<T, E, STREAM>(static_cast<T*>(a.out) + (long)row * a.dim + (long)c * E, v);
    }
  };
  int2 next[8];
  const auto load_ids = [&](int i) {
#pragma unroll
    for (int k = 0; k < 8; ++k) next[k] = i + k < hi ? a.items[i + k] : make_int2(a.rows, 0);
  };
  load_ids(lo);
  for (int i = lo; i < hi; i += 8) {
    int key[8];
    typename Pack<T, E>::type raw[8];
    float f[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      key[k] = next[k].x;
      if (key[k] < a.rows && on) {
        const T* at = grad + (long)next[k].y * a.dim + (long)c * E;
        raw[k] = ONCE ? load_raw_stream<T, E>(at) : load_raw<T, E>(at);
        f[k] = a.factor ? a.factor[next[k].y] : 1.f;
      }
    }
    if (i + 8 < hi) load_ids(i + 8);                            // under way with the rows
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (i + k >= hi) break;
      if (key[k] != row) {
        finish(i + k, false);
        row = key[k];
        start = i + k;
        began_before = false;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.f;
      }
      if (key[k] < a.rows && on) {
        float v[E];
        widen<T, E>(raw[k], v);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = __builtin_fmaf(f[k], v[e], acc[e]);
      }
    }
  }
  finish(hi, hi < a.n && a.items[hi].x == row);
}

// Adds the partial sums of a run from sorted position s to e: that of its first chunk and those of the chunks behind it, the
// `offset`th and every `step`th from there.
template <int E>
__device__ __forceinline__ void add_parts(const GradArgs& a, int s, int e, int offset, int step, int c, float (&acc)[E]) {
  const long q0 = s >> a.chunk_log2, q1 = (e - 1) >> a.chunk_log2;
  for (long q = q0 + offset; q <= q1; q += 4 * step) {
    float v[4][E];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long p = q + k * step;
      if (p <= q1) {
        load_pack<float, E>(a.parts + (2 * p + (p == q0 ? 1 : 0)) * a.dim + (long)c * E, v[k]);
      } else {
#pragma unroll
        for (int x = 0; x < E; ++x) v[k][x] = 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int x = 0; x < E; ++x) acc[x] += v[k][x];
  }
}

template <typename T, int E>
__device__ __forceinline__ void write_row(const GradArgs& a, int row, int c, float (&acc)[E]) {
  if (!a.factor) {
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= a.scale;
  }
  store_pack<T, E>(static_cast<T*>(a.out) + (long)row * a.dim + (long)c * E, acc);
}

// Step 3: the first `joins` workgroups join the runs that cross the borders of their chunks (a group of lanes a border; long
// runs the whole workgroup, through LDS in a fixed order), the others fill the rows that have no occurrence.
template <typename T, int E, bool STREAM>
__global__ __launch_bounds__(256) void embedding_rows_kernel(const GradArgs a, int joins) {
  __shared__ float s_acc[256 * E];
  __shared__ int s_long[256], s_longs;
  const int lanes = 1 << a.lanes_log2, lane = threadIdx.x & (lanes - 1), group = threadIdx.x >> a.lanes_log2, groups = 256 >> a.lanes_log2;
  const int packs = a.dim / E;
  if ((int)blockIdx.x >= joins) {
    const long r0 = ((long)(blockIdx.x - joins) * 4 + (threadIdx.x >> 6)) * a.wave_rows;
    if (r0 >= a.rows) return;
    const int wlane = threadIdx.x & 63;
    const int many = (int)(a.rows - r0 < a.wave_rows ? a.rows - r0 : a.wave_rows);
    const uint64_t empty = __ballot(wlane < many && (a.first == nullptr || a.first[r0 + wlane] < 0));
    float zero[E];
#pragma unroll
    for (int e = 0; e < E; ++e) zero[e] = 0.f;
    for (int r = wlane >> a.lanes_log2; r < many; r += 64 >> a.lanes_log2) {
      if (!((empty >> r) & 1)) continue;
      T* o = static_cast<T*>(a.out) + (r0 + r) * a.dim;
      for (int c = lane; c < packs; c += lanes) put_row<T, E, STREAM>(o + (long)c * E, zero);
    }
    return;
  }
  if (threadIdx.x == 0) s_longs = 0;
  __syncthreads();
  // the run of the last occurrence of chunk q, if it begins there and goes on
  const long border = (((long)blockIdx.x * groups + group) + 1) << a.chunk_log2;
  if (border < a.n) {
    const int row = a.items[border - 1].x;
    if (row < a.rows && a.items[border].x == row) {
      const int s = a.first[row], e = a.last[row];
      if ((long)s >= border - (1l << a.chunk_log2)) {
        if (((e - 1) >> a.chunk_log2) - (s >> a.chunk_log2) >= LONG_RUN) {
          if (lane == 0) s_long[atomicAdd(&s_longs, 1)] = row;
        } else {
          for (int c = lane; c < packs; c += lanes) {
            float acc[E];
#pragma unroll
            for (int x = 0; x < E; ++x) acc[x] = 0.f;
            add_parts<E>(a, s, e, 0, 1, c, acc);
            write_row<T, E>(a, row, c, acc);
          }
        }
      }
    }
  }
  __syncthreads();
  for (int h = 0; h < s_longs; ++h) {                           // the list's order does not touch a row's own sum
    const int row = s_long[h], s = a.first[row], e = a.last[row];
    for (int c0 = 0; c0 < packs; c0 += lanes) {
      const int c = c0 + lane;
      float acc[E];
#pragma unroll
      for (int x = 0; x < E; ++x) acc[x] = 0.f;
      if (c < packs) add_parts<E>(a, s, e, group, groups, c, acc);
      __syncthreads();
#pragma unroll
      for (int x = 0; x < E; ++x) s_acc[x * 256 + threadIdx.x] = acc[x];
      __syncthreads();
      if (group == 0 && c < packs) {
        for (int p = 1; p < groups; ++p)
#pragma unroll
          for (int x = 0; x < E; ++x) acc[x] += s_acc[x * 256 + threadIdx.x + (p << a.lanes_log2)];
        write_row<T, E>(a, row, c, acc);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ host
constexpr long kMostBlocks = (1l << 24) - 1;                    // workgroups of 256 along an axis: no grid of 2^32 threads

int log2_ceil(long n) {
  int k = 0;
  while ((1l << k) < n) ++k;
  return k;
}

// Widest access, in elements, that the row length, the leading dimensions and the addresses allow: 16 bytes, 4 bytes or one element
// (16 384 bf16 rows of 1024, 1022 and 1023: 10, 20 and 35 us the lookup, 56, 74 and 120 the gradient with its sort).
int pack_elems(int dtype, int dim, long ld, const void* p, const void* q) {
  const int b = elem_bytes(dtype);
  for (int w : {16, 4}) {
    const int e = w / b;
    if (e > 1 && dim % e == 0 && ld % e == 0 && ((uintptr_t)p % w) == 0 && ((uintptr_t)q % w) == 0) return e;
  }
  return 1;
}

struct Sizes {
  long items, items2, counts, factor, first, last, parts, total;   // byte offsets
  int tiles, pitch, subs, digit, passes, bits, chunk_log2;
};

Sizes sizes_of(long n, long bags, long rows, int dim, bool mean) {
  Sizes s;
  s.bits = log2_ceil(rows + 1);
  if (s.bits < 1) s.bits = 1;
  s.passes = (s.bits + 9) / 10;
  s.digit = (s.bits + s.passes - 1) / s.passes;
  // Tiles of 1024, longer ones from 1 M lookups on; up to 32 of them a tile adds up the others' counts (128 bytes a bin, one
  // round of loads), beyond a launch of its own does it for all.
  const long tile = 256 * ITEMS;
  s.subs = (int)((n + 1024 * tile - 1) / (1024 * tile));
  if (s.subs < 1) s.subs = 1;
  s.tiles = (int)((n + s.subs * tile - 1) / (s.subs * tile));
  s.pitch = (s.tiles + 3) / 4 * 4;
  // A chunk is walked by one group of lanes: as long as some thousand waves are left (long chunks leave fewer partial sums), at
  // least 16 occurrences.
  const long lanes = dim >= 256 ? 64 : 1l << log2_ceil((dim + 3) / 4);
  s.chunk_log2 = 4;
  while (s.chunk_log2 < (n <= (1 << 20) ? 6 : 7) && (2l << s.chunk_log2) * 131072 <= n * lanes) ++s.chunk_log2;
  long at = 0;
  auto take = [&at](long bytes) { const long p = at; at += (bytes + 255) / 256 * 256; return p; };
  s.items = take(8 * n);
  const bool large = n > SMALL_SORT;
  s.items2 = take(large ? 8 * n : 0);
  s.counts = take(large ? 4l * (s.pitch + 1) << s.digit : 0);
  s.factor = take(mean ? 4 * bags : 0);
  s.first = take(n > 0 ? 4 * rows : 0);
  s.last = take(n > 0 ? 4 * rows : 0);
  s.parts = take(8 * ((n + (1 << s.chunk_log2) - 1) >> s.chunk_log2) * (long)dim);
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
    const long steps = (packs + (1 << lg) - 1) >> lg;
    const bool stream_out = bags * dim * (long)sizeof(T) > (32l << 20);    // eight L2 caches of 4 MB
    const auto kernel = stream_out ? embedding_lookup_kernel<T, E, Id, true> : embedding_lookup_kernel<T, E, Id, false>;
    const long most = kMostBlocks * groups / steps;            // lookups of a launch: steps < 2^25, so at least one
    for (long b = 0; b < bags; b += most) {
      const long jobs = (bags - b < most ? bags - b : most) * steps;
      kernel<<<(unsigned)((jobs + groups - 1) / groups), 256, 0, stream>>>(table, ld, rows, dim, ids + b, (unsigned)jobs, (unsigned)steps, lg, scale,
                                                                           out + b * dim);
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

template <typename Id, bool FIRST>
int launch_pass(const Id* ids, const int2* items, long n, int rows, const Sizes& s, int shift, int per_bag, const Prepare& prep,
                int extra, int* counts, int2* out, hipStream_t stream) {
  const size_t lds = (5 * (size_t)(1 << s.digit) + 16) * sizeof(int);     // at most 10 bits: 20 KB
  int* totals = s.tiles > 32 ? counts + ((long)s.pitch << s.digit) : nullptr;
  embedding_digits_kernel<Id, FIRST><<<s.tiles + extra, 256, sizeof(int) << s.digit, stream>>>(ids, items, (int)n, rows, s.tiles, s.subs, shift,
                                                                                                     s.digit, s.pitch, prep, counts);
  if (totals) embedding_scan_kernel<<<1 << s.digit, 64, 0, stream>>>(counts, s.tiles, s.pitch, totals);
  embedding_scatter_kernel<Id, FIRST><<<s.tiles, 256, lds, stream>>>(ids, items, (int)n, rows, s.subs, shift, s.digit, s.pitch, per_bag,
                                                                           counts, totals, out);
  return (int)hipGetLastError();
}

template <typename Id>
int launch_sort(const Id* ids, long n, int rows, const Sizes& s, char* ws, const Prepare& prep, int2** sorted, hipStream_t stream) {
  int2* items[2] = {(int2*)(ws + s.items), (int2*)(ws + s.items2)};
  long extra = 1 + prep.rows / 4096;                             // workgroups that prepare the rows
  if (prep.factor && extra < prep.bags / 16) extra = prep.bags / 16;
  if (extra > 2048) extra = 2048;
  if (n <= SMALL_SORT) {
    embedding_sort_small_kernel<Id><<<1 + (unsigned)extra, 1024, 0, stream>>>(ids, (int)n, rows, s.bits, prep.tokens, prep, items[0]);
    *sorted = items[0];
    return (int)hipGetLastError();
  }
  int* counts = (int*)(ws + s.counts);
  int rc = launch_pass<Id, true>(ids, nullptr, n, rows, s, 0, s.passes == 1 ? prep.tokens : 1, prep, (int)extra, counts, items[0], stream);
  int from = 0;
  for (int pass = 1; pass < s.passes && rc == TFR_OK; ++pass, from ^= 1)
    rc = launch_pass<Id, false>(ids, items[from], n, rows, s, pass * s.digit, pass + 1 == s.passes ? prep.tokens : 1, prep, 0, counts, items[from ^ 1],
                                stream);
  *sorted = items[from];
  return rc;
}

template <typename T, int E, bool STREAM>
int launch_rows(GradArgs a, const void* grad, bool once, hipStream_t stream) {
  const int packs = a.dim / E;
  a.lanes_log2 = log2_ceil(packs < 64 ? packs : 64);
  const int groups = 256 >> a.lanes_log2;
  // A wave fills rows of about 8 KB in all.
  int wr = 4;
  while (wr < 64 && (long)(2 * wr) * a.dim * (long)sizeof(T) <= 8192) wr *= 2;
  if (wr < (64 >> a.lanes_log2)) wr = 64 >> a.lanes_log2;
  a.wave_rows = wr;
  const long chunks = ((long)a.n + (1 << a.chunk_log2) - 1) >> a.chunk_log2;
  if (chunks > 0) {
    a.steps = (packs + (1 << a.lanes_log2) - 1) >> a.lanes_log2;
    const long blocks = (chunks * a.steps + groups - 1) / groups;
    const long y = (blocks + kMostBlocks - 1) / kMostBlocks, x = (blocks + y - 1) / y;    // the last ones may find nothing to do
    if (y > 65535) return TFR_EINVAL;                           // its partial sums would be 2^51 bytes
    const dim3 grid((unsigned)x, (unsigned)y);
    if (once) embedding_runs_kernel<T, E, true, STREAM><<<grid, 256, 0, stream>>>(a, (const T*)grad);
    else embedding_runs_kernel<T, E, false, STREAM><<<grid, 256, 0, stream>>>(a, (const T*)grad);
  }
  const unsigned joins = chunks > 1 ? (unsigned)((chunks - 1 + groups - 1) / groups) : 0;
  embedding_rows_kernel<T, E, STREAM><<<joins + (unsigned)((a.rows + 4l * wr - 1) / (4l * wr)), 256, 0, stream>>>(a, (int)joins);
  return (int)hipGetLastError();
}

template <typename T, int E>
int launch_grad(const GradArgs& a, const void* grad, bool once, hipStream_t stream) {
  if ((long)a.rows * a.dim * (long)sizeof(T) > (256l << 20)) return launch_rows<T, E, true>(a, grad, once, stream);
  return launch_rows<T, E, false>(a, grad, once, stream);
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
  a.scale = scale;
  char* ws = (char*)workspace;
  if (n > 0) {
    float* factor = mean ? (float*)(ws + s.factor) : nullptr;
    a.factor = factor;
    a.first = (int*)(ws + s.first);
    a.last = (int*)(ws + s.last);
    const Prepare prep = {a.first, factor, bags, a.rows, tokens, scale};
    int2* items = nullptr;
    rc = id_type == TFR_IDS_I32 ? launch_sort<int32_t>((const int32_t*)ids, n, a.rows, s, ws, prep, &items, st)
                                : launch_sort<int64_t>((const int64_t*)ids, n, a.rows, s, ws, prep, &items, st);
    if (rc != TFR_OK) return rc;
    a.items = items;
    a.parts = (float*)(ws + s.parts);
    a.chunk_log2 = s.chunk_log2;
  }
  a.out = grad_table;
  const int e = pack_elems(dtype, dim, dim, n > 0 ? grad : grad_table, grad_table);
  if (dtype == TFR_DTYPE_F32) return e == 4 ? launch_grad<float, 4>(a, grad, tokens == 1, st) : launch_grad<float, 1>(a, grad, tokens == 1, st);
  if (dtype == TFR_DTYPE_BF16)
    return e == 8   ? launch_grad<__bf16, 8>(a, grad, tokens == 1, st)
           : e == 2 ? launch_grad<__bf16, 2>(a, grad, tokens == 1, st)
                    : launch_grad<__bf16, 1>(a, grad, tokens == 1, st);
  return e == 8   ? launch_grad<_Float16, 8>(a, grad, tokens == 1, st)
         : e == 2 ? launch_grad<_Float16, 2>(a, grad, tokens == 1, st)
                  : launch_grad<_Float16, 1>(a, grad, tokens == 1, st);
}
