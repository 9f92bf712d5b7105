// Preference loss on paired log ratios, forward and backward (gfx950).
//
// A list holds L answers of up to T tokens with the token log probabilities of the trained model (lp) and, if there is one, of
// the reference model (ref):
//   s_i   = beta sum_{t : m_it} (lp_it - ref_it)         (/ #{t : m_it} where lengths are normalised)
//   loss  = w / P sum_{(i, j) : y_i > y_j >= 0} l(s_i - s_j),   P = number of such pairs (0 pairs: loss 0)
//   l(h)  = (1 - a) softplus(-h) + a softplus(h)   |   max(0, 1 - h)   |   (h - 1/2)^2
//   dloss/dlp_it = m_it f_i sum over the pairs of i of +-l'(h) w / P,   f_i = beta (/ length)
// 9 bytes a token are read (4 + 4 + the mask's 1) and 4 written: HBM-bound for long answers, launch-bound for short ones.
// Sums over tokens are fp64: a margin is the difference of two sums of thousands of tokens.  What stands in masked places or
// in answers with y < 0 is never used (NaN there does no harm).
#include "common.h"
#include "../../include/tfr_hip.h"

using namespace tfr;

namespace {

constexpr int MAX_ANSWERS = 64;                      // one lane an answer
constexpr int PART = 8192;                           // tokens of an answer that a workgroup sums

struct PrefArgs {
  const float* lp;
  const float* ref;
  const uint8_t* mask;
  const float* labels;
  const float* weights;
  int B, L, T, parts, kind;
  bool normalize;
  float beta, smoothing, scale;
};

struct Sum {
  double s;
  int n;
};

__device__ __forceinline__ Sum token_sum(const PrefArgs& a, long seq, int lo, int hi) {
  Sum r = {0.0, 0};
  const float* lp = a.lp + seq * a.T;
  const float* ref = a.ref ? a.ref + seq * a.T : nullptr;
  const uint8_t* m = a.mask ? a.mask + seq * a.T : nullptr;
  for (int t = lo + threadIdx.x; t < hi; t += 256) {
    const bool on = m ? m[t] != 0 : true;
    const double d = (double)lp[t] - (ref ? (double)ref[t] : 0.0);
    r.s += on ? d : 0.0;
    r.n += on ? 1 : 0;
  }
  return r;
}

// Thread 0 gets the workgroup's sum (fixed order).
__device__ __forceinline__ Sum block_sum_tokens(Sum v) {
  __shared__ double s_s[4];
  __shared__ int s_n[4];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    v.s += __shfl_xor(v.s, o, 64);
    v.n += __shfl_xor(v.n, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    s_s[threadIdx.x >> 6] = v.s;
    s_n[threadIdx.x >> 6] = v.n;
  }
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < 4; ++w) {
      v.s += s_s[w];
      v.n += s_n[w];
    }
  return v;
}

__global__ __launch_bounds__(256) void preference_sum_kernel(const PrefArgs a, double* __restrict__ part_sum, int* __restrict__ part_n) {
  const long seq = blockIdx.x;
  const int lo = blockIdx.y * PART, hi = lo + PART < a.T ? lo + PART : a.T;
  Sum v = {0.0, 0};
  if (a.labels[seq] >= 0.f) v = token_sum(a, seq, lo, hi);
  v = block_sum_tokens(v);
  if (threadIdx.x == 0) {
    part_sum[seq * a.parts + blockIdx.y] = v.s;
    part_n[seq * a.parts + blockIdx.y] = v.n;
  }
}

__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

// One wavefront, lane i = answer i: the list's loss (all lanes) and this lane's d loss / d sum_t lp_it.
__device__ __forceinline__ void list_pairs(const PrefArgs& a, int b, const double* __restrict__ part_sum, const int* __restrict__ part_n,
                                           double* loss_out, double* coef_out) {
  const int lane = threadIdx.x & 63;
  double sum = 0.0;
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
  const double f = (double)a.beta / (a.normalize ? (double)(n > 0 ? n : 1) : 1.0);
  const double s = f * sum;
  const double w = (a.weights ? (double)a.weights[b] : 1.0) * (double)a.scale;
  double loss = 0.0, slope = 0.0;
  int pairs = 0;
  for (int j = 0; j < a.L; ++j) {
    const double sj = __shfl(s, j, 64);
    const float yj = __shfl(y, j, 64);
    const bool win = y > yj && yj >= 0.f, lose = yj > y && y >= 0.f;
    if (!win && !lose) continue;
    const double h = win ? s - sj : sj - s;
    double l, d;
    if (a.kind == TFR_PREFERENCE_LOGISTIC) {
      l = (1.0 - a.smoothing) * softplus(-h) + a.smoothing * softplus(h);
      d = 1.0 / (1.0 + exp(-h)) - (1.0 - a.smoothing);
    } else if (a.kind == TFR_PREFERENCE_HINGE) {
      l = fmax(0.0, 1.0 - h);
      d = h < 1.0 ? -1.0 : 0.0;
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
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    loss += __shfl_xor(loss, o, 64);
    pairs += __shfl_xor(pairs, o, 64);
  }
  const double over = pairs > 0 ? w / (double)pairs : 0.0;
  *loss_out = pairs > 0 ? loss * over : 0.0;
  *coef_out = slope != 0.0 ? slope * over * f : 0.0;
}

__global__ __launch_bounds__(64) void preference_pairs_kernel(const PrefArgs a, const double* __restrict__ part_sum, const int* __restrict__ part_n,
                                                              float* __restrict__ loss, float* __restrict__ coef) {
  const int b = blockIdx.x;
  double l, c;
  list_pairs(a, b, part_sum, part_n, &l, &c);
  if (threadIdx.x == 0) loss[b] = (float)l;
  if (threadIdx.x < a.L) coef[(long)b * a.L + threadIdx.x] = (float)c;
}

// dlp[seq, t] = m * coef[seq] * upstream[list]
__global__ __launch_bounds__(256) void preference_grad_kernel(const float* __restrict__ coef, const float* __restrict__ upstream,
                                                              const uint8_t* __restrict__ mask, int L, int T, float* __restrict__ out) {
  const long seq = blockIdx.x;
  const int lo = blockIdx.y * PART, hi = lo + PART < T ? lo + PART : T;
  float c = coef[seq];
  if (upstream) c *= upstream[seq / L];
  const uint8_t* m = mask ? mask + seq * T : nullptr;
  float* o = out + seq * T;
  for (int t = lo + threadIdx.x; t < hi; t += 256) o[t] = (m ? m[t] != 0 : true) ? c : 0.f;
}

constexpr long kMostTokens = 1 << 28;
constexpr long kMostAnswers = (1l << 24) - 1;        // answers of all lists: a workgroup each, no grid gets 2^32 threads

bool bad_sizes(int B, int L, int T) { return B < 0 || L < 1 || L > MAX_ANSWERS || T < 0 || T > kMostTokens || (long)B * L > kMostAnswers; }
int parts_of(int T) { return T > 0 ? (T + PART - 1) / PART : 1; }

}  // namespace

extern "C" long tfr_preference_workspace_bytes(int B, int L, int T) {
  if (bad_sizes(B, L, T)) return TFR_EINVAL;
  return (long)B * L * parts_of(T) * 12;
}

extern "C" int tfr_preference_loss_f32(const float* log_probs, const float* reference, const uint8_t* mask, const float* labels,
                                       const float* list_weights, int B, int L, int T, int kind, float beta, float smoothing,
                                       int normalize, float scale, float* loss, float* coef, void* workspace, long workspace_bytes, void* stream) {
  if (bad_sizes(B, L, T) || kind < TFR_PREFERENCE_LOGISTIC || kind > TFR_PREFERENCE_SQUARED) return TFR_EINVAL;
  if (!(beta > 0.f) || beta == INFINITY || !(smoothing >= 0.f && smoothing < 0.5f)) return TFR_EINVAL;
  if (B == 0) return TFR_OK;
  if (!labels || !loss || !coef || (T > 0 && !log_probs)) return TFR_EINVAL;
  const PrefArgs a = {log_probs, reference, mask, labels, list_weights, B, L, T, parts_of(T), kind, normalize != 0, beta, smoothing, scale};
  if (!workspace || workspace_bytes < (long)B * L * a.parts * 12 || ((uintptr_t)workspace & 7)) return TFR_EINVAL;
  double* part_sum = (double*)workspace;
  int* part_n = (int*)(part_sum + (long)B * L * a.parts);
  hipStream_t st = (hipStream_t)stream;
  preference_sum_kernel<<<dim3((unsigned)(B * L), a.parts), 256, 0, st>>>(a, part_sum, part_n);
  preference_pairs_kernel<<<B, 64, 0, st>>>(a, part_sum, part_n, loss, coef);
  return (int)hipGetLastError();
}

extern "C" int tfr_preference_grad_f32(const float* coef, const float* upstream, const uint8_t* mask, int B, int L, int T, float* dlog_probs,
                                       void* stream) {
  if (bad_sizes(B, L, T)) return TFR_EINVAL;
  if (B == 0 || T == 0) return TFR_OK;
  if (!coef || !dlog_probs) return TFR_EINVAL;
  preference_grad_kernel<<<dim3((unsigned)(B * L), parts_of(T)), 256, 0, (hipStream_t)stream>>>(coef, upstream, mask, L, T, dlog_probs);
  return (int)hipGetLastError();
}
