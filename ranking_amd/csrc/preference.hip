// Preference loss on paired log ratios, forward and backward (gfx950).
//
// A list holds L answers of up to T tokens with the token log probabilities of the trained model (lp) and, if there is one, of
// the reference model (ref):
//   s_i   = beta sum_{t : m_it} (lp_it - ref_it)         (/ #{t : m_it} where lengths are normalised)
//   loss  = w / P sum_{(i, j) : y_i > y_j >= 0} l(s_i - s_j),   P = number of such pairs (0 pairs: loss 0)
//   l(h)  = (1 - a) softplus(-h) + a softplus(h)   |   max(0, 1 - h)   |   (h - 1/2)^2
//   dloss/dlp_it = m_it f_i sum over the pairs of i of +-l'(h) w / P,   f_i = beta (/ length)
// 9 bytes a token are read (4 + 4 + the mask's 1), those of absent answers are not, and, with the mask once more, 4 written for every
// token: HBM-bound for long answers (512 lists x 6 x 8192 tokens, a sixth of the answers absent: 31 us for the sums = 6.1 TB/s, 19 for the
// gradient = 6.6, 6 for the pairs), launch-bound for a few short ones, and bound by the fp64 exponentials of the pairs and single-token
// reads for very many (282 574 lists x 3 x 13: 105 us with the gradient, 29 by its bytes).
// Sums over tokens are fp64: a margin is the difference of two sums of thousands of tokens.  What stands in masked places or
// in answers with y < 0 is never used (NaN there does no harm).
#include "common.h"
#include "elem.h"

using namespace tfr;

namespace {

constexpr int MAX_ANSWERS = 64;                      // one lane an answer
constexpr int LONG_PART = 8192, SHORT_PART = 2048;   // tokens of an answer that a workgroup sums
constexpr int SMALL_LIST = 8192;                     // tokens of a list that one workgroup takes from its sums to its gradient
constexpr int SHORT_LIST = 1024;                     // and a wavefront or a part of one: 1087 lists of 672 tokens 20 us (39 by workgroups), 2000 of 1800 30 us (20)

struct PrefArgs {
  const float* lp;
  const float* ref;
  const uint8_t* mask;
  const float* labels;
  const float* weights;
  int B, L, T, parts, part, kind;
  bool normalize, wide;                              // wide: addresses allow 16-byte accesses (4 of the mask) at multiples of 4 tokens
  float beta, smoothing, scale;
};

struct Sum {
  double s;
  int n;
};

__device__ __forceinline__ void add_token(Sum& r, float lp, float ref, bool on) {
  r.s += (double)(on ? lp : 0.f) - (double)(on ? ref : 0.f);     // fp64 holds the difference of two fp32 numbers of like size
  r.n += on ? 1 : 0;
}

// STREAM: arrays beyond the L2 caches (32 MB each) go past the caches (100 MB each: sums 48 -> 31 us, gradient 28 -> 19).
template <bool STREAM>
__device__ __forceinline__ void load4(const float* __restrict__ p, float (&v)[4]) {
  widen<float, 4>(STREAM ? load_raw_stream<float, 4>(p) : load_raw<float, 4>(p), v);
}

// Tokens lo .. hi of answer `seq`, by THREADS threads; 4 tokens an access between the first and the last multiple of 4 in memory.
template <int THREADS, bool STREAM>
__device__ __forceinline__ Sum token_sum(const PrefArgs& a, long seq, int lo, int hi, int tid) {
  Sum r = {0.0, 0};
  const long at = seq * a.T + lo, end = seq * a.T + hi;
  const auto one = [&](long t) { add_token(r, a.lp[t], a.ref ? a.ref[t] : 0.f, a.mask ? a.mask[t] != 0 : true); };
  if (!a.wide) {
    for (long t = at + tid; t < end; t += THREADS) one(t);
    return r;
  }
  long head = (at + 3) & ~3l;
  if (head > end) head = end;
  const long tail = head + ((end - head) & ~3l);
  if (tid < head - at) one(at + tid);
  if (tid < end - tail) one(tail + tid);
  for (long t = head + 4 * tid; t < tail; t += 16 * THREADS) {
    float x[4][4], y[4][4];
    uint32_t m[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long u = t + 4l * THREADS * k;
      if (u < tail) {
        load4<STREAM>(a.lp + u, x[k]);
        if (a.ref) load4<STREAM>(a.ref + u, y[k]);
        m[k] = a.mask ? *reinterpret_cast<const uint32_t*>(a.mask + u) : 0x01010101u;
      } else {
        m[k] = 0u;                                              // what is not loaded is not used
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) add_token(r, x[k][e], a.ref ? y[k][e] : 0.f, ((m[k] >> (8 * e)) & 0xffu) != 0);
  }
  return r;
}

// out = m c on tokens lo .. hi of answer `seq`.
template <int THREADS, bool STREAM>
__device__ __forceinline__ void token_fill(const uint8_t* __restrict__ mask, bool wide, long seq, int T, int lo, int hi, int tid, float c,
                                           float* __restrict__ out) {
  const long at = seq * T + lo, end = seq * T + hi;
  const auto one = [&](long t) { out[t] = (mask ? mask[t] != 0 : true) ? c : 0.f; };
  if (!wide) {
    for (long t = at + tid; t < end; t += THREADS) one(t);
    return;
  }
  long head = (at + 3) & ~3l;
  if (head > end) head = end;
  const long tail = head + ((end - head) & ~3l);
  if (tid < head - at) one(at + tid);
  if (tid < end - tail) one(tail + tid);
#pragma unroll 4
  for (long t = head + 4 * tid; t < tail; t += 4 * THREADS) {
    const uint32_t m = mask ? *reinterpret_cast<const uint32_t*>(mask + t) : 0x01010101u;
    const float v[4] = {m & 0xffu ? c : 0.f, m & 0xff00u ? c : 0.f, m & 0xff0000u ? c : 0.f, m & 0xff000000u ? c : 0.f};
    if (STREAM) store_pack_stream<float, 4>(out + t, v);
    else store_pack<float, 4>(out + t, v);
  }
}

__device__ __forceinline__ Sum wave_sum_tokens(Sum v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    v.s += __shfl_xor(v.s, o, 64);
    v.n += __shfl_xor(v.n, o, 64);
  }
  return v;
}

template <bool STREAM>
__global__ __launch_bounds__(256) void preference_sum_kernel(const PrefArgs a, double* __restrict__ part_sum, int* __restrict__ part_n) {
  __shared__ Sum s_part[4];
  const long seq = blockIdx.x;
  const int lo = blockIdx.y * a.part, hi = lo + a.part < a.T ? lo + a.part : a.T;
  Sum v = {0.0, 0};
  if (a.labels[seq] >= 0.f) v = token_sum<256, STREAM>(a, seq, lo, hi, threadIdx.x);
  v = wave_sum_tokens(v);
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 4; ++w) {
      v.s += s_part[w].s;
      v.n += s_part[w].n;
    }
    part_sum[seq * a.parts + blockIdx.y] = v.s;
    part_n[seq * a.parts + blockIdx.y] = v.n;
  }
}

// `lanes` neighbouring lanes (a power of two, at least L), lane i of them = answer i with its grade y (-1 behind the last), its sum and
// number of tokens: the list's loss (all lanes) and this lane's d loss / d sum_t lp_it.
__device__ __forceinline__ void list_pairs(const PrefArgs& a, long b, float y, double sum, int n, int lanes, double* loss_out, double* coef_out) {
  const int base = (threadIdx.x & 63) & ~(lanes - 1);
  const double f = (double)a.beta / (a.normalize ? (double)(n > 0 ? n : 1) : 1.0);
  const double s = f * sum;
  const double w = (a.weights ? (double)a.weights[b] : 1.0) * (double)a.scale;
  double loss = 0.0, slope = 0.0;
  int pairs = 0;
  for (int j = 0; j < a.L; ++j) {
    const double sj = __shfl(s, base + j, 64);
    const float yj = __shfl(y, base + j, 64);
    const bool win = y > yj && yj >= 0.f, lose = yj > y && y >= 0.f;
    if (!win && !lose) continue;
    const double h = win ? s - sj : sj - s;
    double l, d;
    if (a.kind == TFR_PREFERENCE_LOGISTIC) {
      // softplus(+-h) = max(+-h, 0) + log(1 + e) and sigma(h) from one e = exp(-|h|): no overflow at any margin
      const double e = exp(-fabs(h)), q = 1.0 / (1.0 + e);
      l = log1p(e) + (h < 0.0 ? -(1.0 - a.smoothing) * h : a.smoothing > 0.f ? a.smoothing * h : 0.0);   // h may be infinite
      d = (h < 0.0 ? e * q : q) - (1.0 - a.smoothing);
    } else if (a.kind == TFR_PREFERENCE_HINGE) {
      l = h >= 1.0 ? 0.0 : 1.0 - h;                             // a margin that is NaN stays one
      d = h >= 1.0 ? 0.0 : h < 1.0 ? -1.0 : h;
    } else {
      l = (h - 0.5) * (h - 0.5);
      d = 2.0 * h - 1.0;
    }
    if (win) {
      loss += l;
      ++pairs;
    }
    slope += win ? d : -d;
  }
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    loss += __shfl_xor(loss, o, 64);
    pairs += __shfl_xor(pairs, o, 64);
  }
  const double over = pairs > 0 ? w / (double)pairs : 0.0;
  *loss_out = pairs > 0 ? loss * over : 0.0;
  *coef_out = slope != 0.0 ? slope * over * f : 0.0;
}

__global__ __launch_bounds__(64) void preference_pairs_kernel(const PrefArgs a, const double* __restrict__ part_sum, const int* __restrict__ part_n,
                                                              float* __restrict__ loss, float* __restrict__ coef) {
  const int b = blockIdx.x, lane = threadIdx.x;
  double sum = 0.0, l, c;
  int n = 0;
  float y = -1.f;
  if (lane < a.L) {
    const long seq = (long)b * a.L + lane;
    y = a.labels[seq];
    for (int p = 0; p < a.parts; ++p) {
      sum += part_sum[seq * a.parts + p];
      n += part_n[seq * a.parts + p];
    }
  }
  list_pairs(a, b, y, sum, n, 64, &l, &c);
  if (lane == 0) loss[b] = (float)l;
  if (lane < a.L) coef[(long)b * a.L + lane] = (float)c;
}

// The lists' losses (16-byte aligned) added in fp64, in an order that depends on their number alone; 32 values of a thread in flight
// (39 747 lists took 37 us one by one).
template <int THREADS>
__device__ __forceinline__ void total_loss(const float* __restrict__ loss, int B, float* __restrict__ total) {
  __shared__ double s_part[THREADS / 64];
  double t = 0.0;
  const float4* packs = reinterpret_cast<const float4*>(loss);
  for (int p0 = threadIdx.x; p0 < B / 4; p0 += 8 * THREADS) {
    float4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = p0 + k * THREADS < B / 4 ? packs[p0 + k * THREADS] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 8; ++k) t += ((double)v[k].x + (double)v[k].y) + ((double)v[k].z + (double)v[k].w);
  }
  if ((int)threadIdx.x < (B & 3)) t += (double)loss[(B & ~3) + threadIdx.x];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < THREADS / 64; ++w) t += s_part[w];
    total[0] = (float)t;
  }
}

__global__ __launch_bounds__(1024) void preference_total_kernel(const float* __restrict__ loss, int B, float* __restrict__ total) {
  total_loss<1024>(loss, B, total);
}

// dlp[seq, t] = m * coef[seq] * upstream[list]; the last workgroup of the first part adds the lists' losses where a total is wanted.
template <bool STREAM>
__global__ __launch_bounds__(256) void preference_grad_kernel(const float* __restrict__ coef, const float* __restrict__ upstream,
                                                              const uint8_t* __restrict__ mask, int L, int T, int part, bool wide,
                                                              float* __restrict__ out, const float* __restrict__ loss, int B,
                                                              float* __restrict__ total) {
  const long seq = blockIdx.x;
  if (seq == (long)B * L) {
    if (blockIdx.y == 0) total_loss<256>(loss, B, total);
    return;
  }
  const int lo = blockIdx.y * part, hi = lo + part < T ? lo + part : T;
  float c = coef[seq];
  if (upstream) c *= upstream[seq / L];
  token_fill<256, STREAM>(mask, wide, seq, T, lo, hi, threadIdx.x, c, out);
}

// Short lists, `lanes` (a power of two) lanes each, of which an answer has lanes / slots (slots: the power of two that holds the
// answers).  Either the gradient is written (out) or the answers' coefficients (coef).  39 747 lists of 4 answers of 3 tokens: 160 us by
// a workgroup a list, 31 by a wavefront, 6 by 8 lanes.
__global__ __launch_bounds__(256) void preference_wave_kernel(const PrefArgs a, int lanes_log2, int slots_log2, float* __restrict__ loss,
                                                              float* __restrict__ out, float* __restrict__ coef) {
  const int lanes = 1 << lanes_log2, lane = threadIdx.x & 63, base = lane & ~(lanes - 1), li = lane & (lanes - 1);
  const long b = ((long)blockIdx.x * 256 + threadIdx.x) >> lanes_log2;
  const int width_log2 = lanes_log2 - slots_log2, width = 1 << width_log2;
  const int answer = li >> width_log2, first = li & (width - 1);
  const bool list = b < a.B, mine = list && answer < a.L;      // the lanes behind the last list stay: others read them
  const long seq = b * a.L + answer;
  Sum v = {0.0, 0};
  if (mine && a.labels[seq] >= 0.f) {
    for (long t = seq * a.T + first; t < (seq + 1) * a.T; t += width)
      add_token(v, a.lp[t], a.ref ? a.ref[t] : 0.f, a.mask ? a.mask[t] != 0 : true);
  }
  for (int o = width >> 1; o > 0; o >>= 1) {
    v.s += __shfl_xor(v.s, o, 64);
    v.n += __shfl_xor(v.n, o, 64);
  }
  const int from = base + ((li << width_log2) & (lanes - 1));  // lane i of the list takes answer i's sum
  const double sum = __shfl(v.s, from, 64);
  const int n = __shfl(v.n, from, 64);
  double l, c;
  list_pairs(a, list ? b : 0, list && li < a.L ? a.labels[b * a.L + li] : -1.f, sum, n, lanes, &l, &c);
  if (list && li == 0) loss[b] = (float)l;
  if (coef) {
    if (list && li < a.L) coef[b * a.L + li] = (float)c;
    return;
  }
  const float by = __shfl((float)c, base + answer, 64);
  if (mine) {
    for (long t = seq * a.T + first; t < (seq + 1) * a.T; t += width) out[t] = (a.mask ? a.mask[t] != 0 : true) ? by : 0.f;
  }
}

// The gradient of short answers from their coefficients: a thread a token.
__global__ __launch_bounds__(256) void preference_grad_short_kernel(const float* __restrict__ coef, const float* __restrict__ upstream,
                                                                    const uint8_t* __restrict__ mask, unsigned L, unsigned T, unsigned n,
                                                                    float* __restrict__ out) {
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  if (i >= n) return;
  const unsigned seq = i / T;
  float c = coef[seq];
  if (upstream) c *= upstream[seq / L];
  out[i] = (mask ? mask[i] != 0 : true) ? c : 0.f;
}

// A list from its sums to its gradient by one workgroup: an answer a wave and step.
__global__ __launch_bounds__(256) void preference_list_kernel(const PrefArgs a, float* __restrict__ loss, float* __restrict__ out) {
  __shared__ Sum s_sum[MAX_ANSWERS];
  __shared__ float s_coef[MAX_ANSWERS];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = wave; i < a.L; i += 4) {
    const long seq = (long)b * a.L + i;
    Sum v = {0.0, 0};
    if (a.labels[seq] >= 0.f) v = token_sum<64, false>(a, seq, 0, a.T, lane);
    v = wave_sum_tokens(v);
    if (lane == 0) s_sum[i] = v;
  }
  __syncthreads();
  if (wave == 0) {
    const bool here = lane < a.L;
    double l, c;
    list_pairs(a, b, here ? a.labels[(long)b * a.L + lane] : -1.f, here ? s_sum[lane].s : 0.0, here ? s_sum[lane].n : 0, 64, &l, &c);
    if (lane == 0) loss[b] = (float)l;
    if (here) s_coef[lane] = (float)c;
  }
  __syncthreads();
  for (int i = wave; i < a.L; i += 4) token_fill<64, false>(a.mask, a.wide, (long)b * a.L + i, a.T, 0, a.T, lane, s_coef[i], out);
}

constexpr long kMostTokens = 1 << 28;
constexpr long kMostAnswers = (1l << 24) - 2;        // answers of all lists: a workgroup each and one more, no grid gets 2^32 threads

bool bad_sizes(int B, int L, int T) { return B < 0 || L < 1 || L > MAX_ANSWERS || T < 0 || T > kMostTokens || (long)B * L > kMostAnswers; }
// Long parts where there are enough of them to fill the card, short ones else.
bool many_tokens(int B, int L, int T) { return (long)B * L * T >= (1l << 23); }
int part_of(int B, int L, int T) { return many_tokens(B, L, T) ? LONG_PART : SHORT_PART; }
int parts_of(int B, int L, int T) { return T > 0 ? (T + part_of(B, L, T) - 1) / part_of(B, L, T) : 1; }
bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }       // null too

struct Workspace {                                   // losses [B, padded to 4], coefficients [B * L, padded], sums [B * L * parts], numbers
  float* loss;
  float* coef;
  double* sum;
  int* n;
};
long padded(long n) { return (n + 3) & ~3l; }
long workspace_bytes_of(int B, int L, int T) {
  return padded(B) * 4 + padded((long)B * L) * 4 + (long)B * L * parts_of(B, L, T) * 12;
}
Workspace workspace_at(void* p, int B, int L, int T) {
  Workspace w;
  w.loss = (float*)p;
  w.coef = w.loss + padded(B);
  w.sum = (double*)(w.coef + padded((long)B * L));
  w.n = (int*)(w.sum + (long)B * L * parts_of(B, L, T));
  return w;
}

// Short lists (L * T <= SHORT_LIST): a wavefront a list, fewer lanes where there are lists enough to fill the card so.
void launch_short(const PrefArgs& a, float* loss, float* out, float* coef, hipStream_t st) {
  int slots = 0, lanes = 6;
  while ((1 << slots) < a.L) ++slots;
  while (lanes > slots && (4l << lanes) >= (long)a.L * a.T && ((long)a.B << lanes) > 64 * 4096) --lanes;
  preference_wave_kernel<<<(unsigned)((((long)a.B << lanes) + 255) / 256), 256, 0, st>>>(a, lanes, slots, loss, out, coef);
}

void launch_sums(const PrefArgs& a, const Workspace& w, hipStream_t st) {
  const auto kernel = many_tokens(a.B, a.L, a.T) ? preference_sum_kernel<true> : preference_sum_kernel<false>;
  kernel<<<dim3((unsigned)(a.B * a.L), a.parts), 256, 0, st>>>(a, w.sum, w.n);
}

int make_args(PrefArgs* a, const float* log_probs, const float* reference, const uint8_t* mask, const float* labels, const float* list_weights,
              int B, int L, int T, int kind, float beta, float smoothing, int normalize, float scale) {
  if (bad_sizes(B, L, T) || kind < TFR_PREFERENCE_LOGISTIC || kind > TFR_PREFERENCE_SQUARED) return TFR_EINVAL;
  if (!(beta > 0.f) || beta == INFINITY || !(smoothing >= 0.f && smoothing < 0.5f)) return TFR_EINVAL;
  if (B > 0 && (!labels || (T > 0 && !log_probs))) return TFR_EINVAL;
  const bool wide = aligned(log_probs, 16) && aligned(reference, 16) && aligned(mask, 4);
  *a = {log_probs, reference, mask, labels, list_weights, B, L, T, parts_of(B, L, T), part_of(B, L, T), kind, normalize != 0, wide, beta, smoothing, scale};
  return TFR_OK;
}

}  // namespace

extern "C" long tfr_preference_workspace_bytes(int B, int L, int T) {
  if (bad_sizes(B, L, T)) return TFR_EINVAL;
  return workspace_bytes_of(B, L, T);
}

extern "C" int tfr_preference_loss_f32(const float* log_probs, const float* reference, const uint8_t* mask, const float* labels,
                                       const float* list_weights, int B, int L, int T, int kind, float beta, float smoothing,
                                       int normalize, float scale, float* loss, float* coef, void* workspace, long workspace_bytes,
                                       void* stream) {
  PrefArgs a;
  const int rc = make_args(&a, log_probs, reference, mask, labels, list_weights, B, L, T, kind, beta, smoothing, normalize, scale);
  if (rc != TFR_OK) return rc;
  if (B == 0) return TFR_OK;
  if (!loss || !coef || !workspace || workspace_bytes < workspace_bytes_of(B, L, T) || !aligned(workspace, 16)) return TFR_EINVAL;
  const Workspace w = workspace_at(workspace, B, L, T);
  hipStream_t st = (hipStream_t)stream;
  if ((long)L * T <= SHORT_LIST) {
    launch_short(a, loss, nullptr, coef, st);
  } else {
    launch_sums(a, w, st);
    preference_pairs_kernel<<<B, 64, 0, st>>>(a, w.sum, w.n, loss, coef);
  }
  return (int)hipGetLastError();
}

extern "C" int tfr_preference_total_f32(const float* loss, int B, float* total, void* stream) {
  if (B < 0 || B > kMostAnswers || !total || (B > 0 && !loss) || !aligned(loss, 16)) return TFR_EINVAL;
  preference_total_kernel<<<1, 1024, 0, (hipStream_t)stream>>>(loss, B, total);
  return (int)hipGetLastError();
}

extern "C" int tfr_preference_grad_f32(const float* coef, const float* upstream, const uint8_t* mask, int B, int L, int T, float* dlog_probs,
                                       void* stream) {
  if (bad_sizes(B, L, T)) return TFR_EINVAL;
  if (B == 0 || T == 0) return TFR_OK;
  if (!coef || !dlog_probs) return TFR_EINVAL;
  const long n = (long)B * L * T;
  if (T <= 128 && n < (1l << 31)) {                  // a workgroup an answer would leave most of its threads without a token
    preference_grad_short_kernel<<<(unsigned)((n + 255) / 256), 256, 0, (hipStream_t)stream>>>(coef, upstream, mask, L, T, (unsigned)n, dlog_probs);
    return (int)hipGetLastError();
  }
  const auto kernel = many_tokens(B, L, T) ? preference_grad_kernel<true> : preference_grad_kernel<false>;
  kernel<<<dim3((unsigned)(B * L), parts_of(B, L, T)), 256, 0, (hipStream_t)stream>>>(
      coef, upstream, mask, L, T, part_of(B, L, T), aligned(dlog_probs, 16) && aligned(mask, 4), dlog_probs, nullptr, B, nullptr);
  return (int)hipGetLastError();
}

extern "C" int tfr_preference_loss_and_grad_f32(const float* log_probs, const float* reference, const uint8_t* mask, const float* labels,
                                                const float* list_weights, int B, int L, int T, int kind, float beta, float smoothing,
                                                int normalize, float scale, float* total, float* dlog_probs, void* workspace,
                                                long workspace_bytes, void* stream) {
  PrefArgs a;
  const int rc = make_args(&a, log_probs, reference, mask, labels, list_weights, B, L, T, kind, beta, smoothing, normalize, scale);
  if (rc != TFR_OK) return rc;
  if (!total || (B > 0 && T > 0 && !dlog_probs)) return TFR_EINVAL;
  if (B > 0 && (!workspace || workspace_bytes < workspace_bytes_of(B, L, T) || !aligned(workspace, 16))) return TFR_EINVAL;
  const Workspace w = workspace_at(workspace, B, L, T);
  hipStream_t st = (hipStream_t)stream;
  a.wide = a.wide && aligned(dlog_probs, 16);
  if (B == 0 || (long)L * T <= SMALL_LIST) {
    if (B > 0 && (long)L * T <= SHORT_LIST) launch_short(a, w.loss, dlog_probs, nullptr, st);
    else if (B > 0) preference_list_kernel<<<B, 256, 0, st>>>(a, w.loss, dlog_probs);
    preference_total_kernel<<<1, 1024, 0, st>>>(w.loss, B, total);
  } else {
    launch_sums(a, w, st);
    preference_pairs_kernel<<<B, 64, 0, st>>>(a, w.sum, w.n, w.loss, w.coef);
    const auto kernel = many_tokens(B, L, T) ? preference_grad_kernel<true> : preference_grad_kernel<false>;
    kernel<<<dim3((unsigned)(B * L) + 1, a.parts), 256, 0, st>>>(w.coef, nullptr, mask, L, T, a.part, a.wide, dlog_probs, w.loss, B, total);
  }
  return (int)hipGetLastError();
}
