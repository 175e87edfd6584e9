// Losses on token log-probabilities for gfx950: the preference loss over pairs
// of sequences and the clipped policy loss with a KL term, forward and backward.
//
// Inputs are fp32 [sequences][tokens] with row strides and a byte mask.  Both
// are bandwidth-bound where they are large (9 to 21 bytes and about twenty
// operations a token) and bound by launches where they are small.  Differences
// of log-probabilities are small against their sums over a sequence and cancel
// between a pair's sequences, so all sums are fp64, in a fixed order.
//
// Preference: a group of L lanes owns a pair when the sequences are short or the
// pairs many, and finishes it (margin, loss term, both rows' gradient
// coefficients); few long pairs are cut into chunks of tokens whose sums a second
// kernel joins.  The gradient is one coefficient a row, written by a third.
// Policy: elementwise, four tokens a thread; the mean over a sequence needs its
// token count before the gradient, so a pass over the mask alone makes it.
//
// 4096 x 2048 tokens: preference 16.6 us forward (76 MB, 4.5 TB/s), policy 33.2 us (176 MB
// with per-token advantages and the slopes, 5.3 TB/s), its gradient 10.9 us (67 MB, from the Infinity Cache); 64 x
// 512: 8.8 + 2.7 + 3.1 us.  The kernels of a call take 7 to 50 us; a call with its backward
// 58 to 100, the host's time through autograd's device thread.

#include <cmath>

#include "rv_device.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

__device__ __forceinline__ double group_sum(double v, int lanes) {
  for (int o = lanes >> 1; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ int group_sum(int v, int lanes) {
  for (int o = lanes >> 1; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Sums of N doubles over the workgroup, the waves added in order; the result is
// thread 0's.
template <int N>
__device__ __forceinline__ void block_sum(double (&v)[N]) {
  __shared__ double red[kWaves][N];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = group_sum(v[i], 64);
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) red[wave][i] = v[i];
  __syncthreads();
  if (threadIdx.x == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = red[0][i];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) v[i] += red[w][i];
    }
}

// ---------------------------------------------------------------------------
// Preference loss.
// ---------------------------------------------------------------------------
struct PrefArgs {
  const float* logp; int64_t ld_logp;
  const float* ref; int64_t ld_ref;
  const uint8_t* mask; int64_t ld_mask;  // nullable
  int64_t pairs, tokens;
  double beta, smoothing;
  int average;
  int vec;            // every row starts on a 16-byte (mask: 4-byte) boundary
  float* loss; float* reward; float* coef;
  double* part_loss;  // one per workgroup
  double* part_sum;   // split: [2 pairs][chunks]
  int* part_count;
  int64_t chunks, chunk;
};

// Sum of logp - ref over the counted tokens [begin, end) of a row, and their
// number, by a group of `lanes` lanes (`lane` in it).
__device__ __forceinline__ void row_sum(const PrefArgs& a, int64_t row, int64_t begin, int64_t end,
                                        int lane, int lanes, double& sum, int& count) {
  const float* p = a.logp + row * a.ld_logp;
  const float* q = a.ref + row * a.ld_ref;
  const uint8_t* m = a.mask ? a.mask + row * a.ld_mask : nullptr;
  sum = 0.0;
  count = 0;
  int64_t t = begin + lane * 4;
  if (a.vec) {
#pragma unroll 2
    for (; t + 4 <= end; t += lanes * 4) {
      const float4 x = rv::ld_f4(p + t), y = rv::ld_f4(q + t);
      const uint32_t w = m ? *reinterpret_cast<const uint32_t*>(m + t) : 0x01010101u;
      const float d[4] = {x.x - y.x, x.y - y.y, x.z - y.z, x.w - y.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (w >> (8 * e) & 0xffu) {
          sum += (double)d[e];
          ++count;
        }
    }
    for (int64_t u = t; u < end && u < t + 4; ++u)
      if (!m || m[u]) {
        sum += (double)(p[u] - q[u]);
        ++count;
      }
  } else {
    for (t = begin + lane; t < end; t += lanes)
      if (!m || m[t]) {
        sum += (double)(p[t] - q[t]);
        ++count;
      }
  }
  sum = group_sum(sum, lanes);
  count = group_sum(count, lanes);
}

// A pair's margin, loss term, rewards and gradient coefficients.
__device__ __forceinline__ double finish_pair(const PrefArgs& a, int64_t i, double s0, int n0,
                                              double s1, int n1) {
  const double share0 = a.average ? 1.0 / (n0 > 1 ? n0 : 1) : 1.0;
  const double share1 = a.average ? 1.0 / (n1 > 1 ? n1 : 1) : 1.0;
  const double r0 = a.beta * s0 * share0, r1 = a.beta * s1 * share1;
  const double margin = r0 - r1;
  const double soft = log1p(exp(-fabs(margin)));  // of -log sigmoid(+-margin)
  const double yes = soft + fmax(-margin, 0.0), no = soft + fmax(margin, 0.0);
  const double slope =
      (a.smoothing - 1.0 / (1.0 + exp(margin))) * a.beta / (double)a.pairs;
  a.reward[i] = (float)r0;
  a.reward[a.pairs + i] = (float)r1;
  a.coef[i] = (float)(slope * share0);
  a.coef[a.pairs + i] = (float)(-slope * share1);
  const double loss = (1.0 - a.smoothing) * yes + a.smoothing * no;
  return margin == margin ? loss : margin;  // fmax drops a NaN
}

// The workgroup's loss terms: the loss itself if it is the only one.
__device__ __forceinline__ void end_pairs(const PrefArgs& a, double loss) {
  double v[1] = {loss};
  block_sum(v);
  if (threadIdx.x != 0) return;
  if (gridDim.x == 1) *a.loss = (float)(v[0] / (double)a.pairs);
  else a.part_loss[blockIdx.x] = v[0];
}

// A group of `lanes` lanes per pair.
__global__ __launch_bounds__(kThreads)
void pref_pairs_k(PrefArgs a, int lanes) {
  const int lane = threadIdx.x & (lanes - 1), per = kThreads / lanes;
  double loss = 0.0;
  // every lane of a wave takes the same number of turns: the sums shuffle
  for (int64_t first = (int64_t)blockIdx.x * per; first < a.pairs;
       first += (int64_t)gridDim.x * per) {
    const int64_t i = first + threadIdx.x / lanes;
    const bool live = i < a.pairs;
    double s0, s1;
    int n0, n1;
    row_sum(a, live ? i : 0, 0, live ? a.tokens : 0, lane, lanes, s0, n0);
    row_sum(a, live ? a.pairs + i : 0, 0, live ? a.tokens : 0, lane, lanes, s1, n1);
    if (live && lane == 0) loss += finish_pair(a, i, s0, n0, s1, n1);
  }
  end_pairs(a, loss);
}

// A wave per chunk of a row.
__global__ __launch_bounds__(kThreads)
void pref_chunks_k(PrefArgs a) {
  const int64_t unit = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (unit >= 2 * a.pairs * a.chunks) return;
  const int64_t row = unit / a.chunks, begin = unit % a.chunks * a.chunk;
  const int64_t end = begin + a.chunk < a.tokens ? begin + a.chunk : a.tokens;
  double sum;
  int count;
  row_sum(a, row, begin, end, threadIdx.x & 63, 64, sum, count);
  if ((threadIdx.x & 63) == 0) {
    a.part_sum[unit] = sum;
    a.part_count[unit] = count;
  }
}

// A wave per pair joins its chunks.
__global__ __launch_bounds__(kThreads)
void pref_join_k(PrefArgs a) {
  const int64_t i = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  double loss = 0.0;
  if (i < a.pairs) {
    double s[2] = {0.0, 0.0};
    int n[2] = {0, 0};
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int64_t base = (side * a.pairs + i) * a.chunks;
      for (int64_t c = lane; c < a.chunks; c += 64) {
        s[side] += a.part_sum[base + c];
        n[side] += a.part_count[base + c];
      }
      s[side] = group_sum(s[side], 64);
      n[side] = group_sum(n[side], 64);
    }
    if (lane == 0) loss = finish_pair(a, i, s[0], n[0], s[1], n[1]);
  }
  end_pairs(a, loss);
}

__global__ __launch_bounds__(kThreads)
void pref_total_k(const double* __restrict__ part, int64_t n, int64_t pairs,
                  float* __restrict__ loss) {
  double v[1] = {0.0};
  for (int64_t i = threadIdx.x; i < n; i += kThreads) v[0] += part[i];
  block_sum(v);
  if (threadIdx.x == 0) *loss = (float)(v[0] / (double)pairs);
}

// dlogp = coef[row] * *grad where counted: four consecutive tokens a thread, of
// the contiguous output (they may belong to two rows or more).
// FLAT: the mask is contiguous on a 4-byte boundary, one word a thread (4096 x 2048 tokens
// 15.4 -> 11.6 us; 42 MB, inside the Infinity Cache).
template <bool FLAT>
__global__ __launch_bounds__(kThreads)
void pref_grad_k(const float* __restrict__ coef, const uint8_t* __restrict__ mask,
                 int64_t ld_mask, const float* __restrict__ grad, int64_t n, int64_t tokens,
                 float* __restrict__ out) {
  const float g = *grad;
  const int64_t step = (int64_t)gridDim.x * kThreads * 4;
  for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4; i < n; i += step) {
    int64_t row = n <= UINT32_MAX ? (int64_t)((uint32_t)i / (uint32_t)tokens) : i / tokens;
    int64_t t = i - row * tokens;
    float v[4];
    const bool whole = FLAT && i + 4 <= n;
    const uint32_t m = whole ? *reinterpret_cast<const uint32_t*>(mask + i) : 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = 0.f;
      if (whole ? (m >> (8 * e) & 0xffu) != 0
                : i + e < n && (!mask || mask[row * ld_mask + t]))
        v[e] = coef[row] * g;
      if (++t == tokens) {
        t = 0;
        ++row;
      }
    }
    if (i + 4 <= n) rv::st_f4(out + i, make_float4(v[0], v[1], v[2], v[3]));
    else
      for (int e = 0; i + e < n; ++e) out[i + e] = v[e];
  }
}

// ---------------------------------------------------------------------------
// Policy loss.
// ---------------------------------------------------------------------------
struct PolicyArgs {
  const float* logp; int64_t ld_logp;
  const float* old; int64_t ld_old;
  const float* ref; int64_t ld_ref;      // nullable
  const float* adv; int64_t adv_row, adv_col;
  const uint8_t* mask; int64_t ld_mask;  // nullable
  int64_t seqs, tokens;
  double log_low, log_high;  // log(1 - clip_low), log(1 + clip_high)
  float low, high, kl;       // 1 - clip_low, 1 + clip_high
  const float* weight;       // per sequence; NULL: the mean over all counted tokens
  float* loss;
  float* stats;              // [3]
  float* slope;              // nullable
  double* part;              // [workgroups][4]
};

// Counted tokens of mask[begin, end) by lane `lane` of `lanes`, 16 bytes at a time
// where the address allows it.
__device__ __forceinline__ int count_row(const uint8_t* __restrict__ m, int64_t begin, int64_t end,
                                         int lane, int lanes) {
  int count = 0;
  int64_t t = begin;
  if ((reinterpret_cast<uintptr_t>(m + begin) & 15) == 0) {
    const int64_t vecs = (end - begin) / 16;
#pragma unroll 4
    for (int64_t v = lane; v < vecs; v += lanes) {
      const uint4 w = *reinterpret_cast<const uint4*>(m + begin + v * 16);
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) count += (words[k] >> (8 * e) & 0xffu) != 0;
    }
    t = begin + vecs * 16;
  }
  for (t += lane; t < end; t += lanes) count += m[t] != 0;
  return count;
}

__device__ __forceinline__ float weight_of(int count, int64_t seqs) {
  return (float)(1.0 / ((double)(count > 1 ? count : 1) * (double)seqs));
}

// weight[s] = 1 / (counted tokens * sequences), by a group of `lanes` lanes.
__global__ __launch_bounds__(kThreads)
void policy_weight_k(const uint8_t* __restrict__ mask, int64_t ld, int64_t seqs, int64_t tokens,
                     int lanes, float* __restrict__ weight) {
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t s = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / lanes;
  int count = 0;
  if (s < seqs) {
    if (!mask) count = lane == 0 ? (int)tokens : 0;
    else count = count_row(mask + s * ld, 0, tokens, lane, lanes);
  }
  count = group_sum(count, lanes);
  if (s < seqs && lane == 0) weight[s] = weight_of(count, seqs);
}

// The same for long sequences, in chunks of kCountChunk tokens: a workgroup per chunk,
// then a wave per sequence (8 sequences of 40000 tokens: 199 us with a wave each).
__global__ __launch_bounds__(kThreads)
void policy_count_k(const uint8_t* __restrict__ mask, int64_t ld, int64_t tokens, int64_t chunk,
                    int64_t chunks, int* __restrict__ part) {
  const int64_t s = blockIdx.x / chunks, begin = blockIdx.x % chunks * chunk;
  const int64_t end = begin + chunk < tokens ? begin + chunk : tokens;
  const int count = group_sum(count_row(mask + s * ld, begin, end, threadIdx.x, kThreads), 64);
  __shared__ int red[kWaves];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = count;
  __syncthreads();
  if (threadIdx.x != 0) return;
  int total = red[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) total += red[w];
  part[blockIdx.x] = total;
}
__global__ __launch_bounds__(kThreads)
void policy_join_k(const int* __restrict__ part, int64_t seqs, int64_t chunks,
                   float* __restrict__ weight) {
  const int64_t s = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (s >= seqs) return;
  int count = 0;
  for (int64_t c = threadIdx.x & 63; c < chunks; c += 64) count += part[s * chunks + c];
  count = group_sum(count, 64);
  if ((threadIdx.x & 63) == 0) weight[s] = weight_of(count, seqs);
}

// k = exp(s) - s - 1 and its derivative exp(s) - 1: the differences would leave nothing of
// a small s (k = s^2 / 2), where a model close to its reference spends its time.  Below 1
// the series k = s^2 sum_i s^i / (i + 2)!, to i = 9 (the rest is below 2^-27 of it), and
// k + s; above, k and -s are large where exp(s) - 1 is not.
__device__ __forceinline__ void kl_term(float s, float& k, float& slope) {
  if (fabsf(s) >= 1.f) {
    const float e = expf(s);
    k = e - s - 1.f;
    slope = e - 1.f;
    return;
  }
  constexpr float c[] = {1.f / 39916800, 1.f / 3628800, 1.f / 362880, 1.f / 40320, 1.f / 5040,
                         1.f / 720,      1.f / 120,     1.f / 24,     1.f / 6,     1.f / 2};
  float p = c[0];
#pragma unroll
  for (int i = 1; i < 10; ++i) p = __builtin_fmaf(p, s, c[i]);
  k = s * s * p;
  slope = k + s;
}

// One token: its loss, KL term, whether its ratio is clipped, and d loss / d logp.
// The clip is decided on the logarithms in fp64: a ratio next to a border falls
// on its side of it, and the gradient with it.
__device__ __forceinline__ void policy_token(const PolicyArgs& a, float logp, float old, float ref,
                                             float adv, float& loss, float& k, bool& clipped,
                                             float& slope) {
  const float ratio = expf(logp - old);
  const double delta = (double)logp - (double)old;
  const bool high = adv > 0.f && delta > a.log_high, low = adv < 0.f && delta < a.log_low;
  clipped = high || low;
  loss = -(high ? a.high : low ? a.low : ratio) * adv;
  slope = clipped ? 0.f : -ratio * adv;
  k = 0.f;
  if (a.ref) {
    float away;
    kl_term(ref - logp, k, away);
    if (a.kl != 0.f) {  // 0: the statistic alone, which may be infinite
      loss += a.kl * k;
      slope -= a.kl * away;
    }
  }
}

__device__ __forceinline__ void policy_stats(const PolicyArgs& a, const double (&v)[4]) {
  const double n = v[3] > 1.0 ? v[3] : 1.0;
  *a.loss = (float)(a.weight ? v[0] : v[0] / n);
  a.stats[0] = (float)(v[1] / n);
  a.stats[1] = (float)(v[2] / n);
  a.stats[2] = a.weight ? 1.f : (float)(1.0 / n);
}

// FLAT: every array is contiguous and 16-byte aligned (mask: 4), so four
// consecutive tokens are one vector; otherwise they are loaded one by one.
template <bool FLAT>
__global__ __launch_bounds__(kThreads)
void policy_loss_k(PolicyArgs a) {
  const int64_t n = a.seqs * a.tokens;
  const int64_t step = (int64_t)gridDim.x * kThreads * 4;
  double total[4] = {0.0, 0.0, 0.0, 0.0};
  for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4; i < n; i += step) {
    int64_t row = n <= UINT32_MAX ? (int64_t)((uint32_t)i / (uint32_t)a.tokens) : i / a.tokens;
    int64_t t = i - row * a.tokens;
    float lp[4] = {}, od[4] = {}, rf[4] = {}, ad[4] = {}, w[4], out[4] = {};
    bool on[4] = {};
    if (FLAT && i + 4 <= n) {
      const float4 x = rv::ld_f4(a.logp + i), y = rv::ld_f4(a.old + i);
      const float4 z = a.ref ? rv::ld_f4(a.ref + i) : make_float4(0.f, 0.f, 0.f, 0.f);
      const uint32_t m = a.mask ? *reinterpret_cast<const uint32_t*>(a.mask + i) : 0x01010101u;
      lp[0] = x.x; lp[1] = x.y; lp[2] = x.z; lp[3] = x.w;
      od[0] = y.x; od[1] = y.y; od[2] = y.z; od[3] = y.w;
      rf[0] = z.x; rf[1] = z.y; rf[2] = z.z; rf[3] = z.w;
#pragma unroll
      for (int e = 0; e < 4; ++e) on[e] = (m >> (8 * e) & 0xffu) != 0;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = 1.f;
      if (i + e < n) {
        if (!(FLAT && i + 4 <= n)) {
          on[e] = !a.mask || a.mask[row * a.ld_mask + t];
          lp[e] = a.logp[row * a.ld_logp + t];
          od[e] = a.old[row * a.ld_old + t];
          if (a.ref) rf[e] = a.ref[row * a.ld_ref + t];
        }
        ad[e] = a.adv[row * a.adv_row + t * a.adv_col];
        if (a.weight) w[e] = a.weight[row];
      }
      if (++t == a.tokens) {
        t = 0;
        ++row;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (!on[e]) continue;
      float loss, k;
      bool clipped;
      policy_token(a, lp[e], od[e], rf[e], ad[e], loss, k, clipped, out[e]);
      out[e] *= w[e];
      total[0] += (double)loss * (double)w[e];
      total[1] += (double)k;
      total[2] += clipped ? 1.0 : 0.0;
      total[3] += 1.0;
    }
    if (a.slope) {
      if (i + 4 <= n) rv::st_f4(a.slope + i, make_float4(out[0], out[1], out[2], out[3]));
      else
        for (int e = 0; i + e < n; ++e) a.slope[i + e] = out[e];
    }
  }
  block_sum(total);
  if (threadIdx.x != 0) return;
  if (gridDim.x == 1) policy_stats(a, total);
  else
#pragma unroll
    for (int j = 0; j < 4; ++j) a.part[blockIdx.x * 4 + j] = total[j];
}

__global__ __launch_bounds__(kThreads)
void policy_total_k(PolicyArgs a, int blocks) {
  double total[4] = {0.0, 0.0, 0.0, 0.0};
  for (int b = threadIdx.x; b < blocks; b += kThreads)
#pragma unroll
    for (int j = 0; j < 4; ++j) total[j] += a.part[b * 4 + j];
  block_sum(total);
  if (threadIdx.x == 0) policy_stats(a, total);
}

__global__ __launch_bounds__(kThreads)
void policy_grad_k(const float* __restrict__ slope, const float* __restrict__ factor,
                   const float* __restrict__ grad, int64_t n, float* __restrict__ out) {
  const float g = *factor * *grad;
  const int64_t step = (int64_t)gridDim.x * kThreads * 4;
  for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4; i < n; i += step) {
    if (i + 4 <= n) {
      const float4 v = rv::ld_f4(slope + i);
      rv::st_f4(out + i, make_float4(v.x * g, v.y * g, v.z * g, v.w * g));
    } else {
      for (int64_t j = i; j < n; ++j) out[j] = slope[j] * g;
    }
  }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
constexpr int64_t kChunk = 1024;       // tokens of a row that a wave sums
constexpr int64_t kCountChunk = 8192;  // tokens of a long sequence's mask that a workgroup counts
constexpr int64_t kMaxBlocks = 2048;   // workgroups of a pass that loops over its input

int64_t blocks_of(int64_t threads) {
  const int64_t b = (threads + kThreads - 1) / kThreads;
  return b < 1 ? 1 : b < kMaxBlocks ? b : kMaxBlocks;
}

// Lanes for a row of `tokens`: a power of two, four tokens each.
int lanes_of(int64_t tokens) {
  int lanes = 1;
  while (lanes < 64 && lanes * 4 < tokens) lanes *= 2;
  return lanes;
}

// Few pairs of long sequences: cut into chunks, so that the chip is not left to
// a few waves.
bool pref_split(int64_t pairs, int64_t tokens) { return tokens > 2 * kChunk && pairs < 1024; }

struct PrefPlan {
  int64_t chunks, blocks;  // chunks 0: not split
  int64_t sum_at, count_at, bytes;
};
PrefPlan pref_plan(int64_t pairs, int64_t tokens) {
  PrefPlan p{};
  if (pref_split(pairs, tokens)) {
    p.chunks = (tokens + kChunk - 1) / kChunk;
    p.blocks = (pairs + kWaves - 1) / kWaves;
  } else {
    p.blocks = blocks_of(pairs * lanes_of(tokens));
  }
  p.sum_at = p.blocks * 8;
  p.count_at = p.sum_at + 2 * pairs * p.chunks * 8;
  p.bytes = p.count_at + 2 * pairs * p.chunks * 4;
  return p;
}

// Chunks that a sequence's tokens are counted in; 0: by a group of lanes.
int64_t count_chunks(int64_t tokens) {
  return tokens > kCountChunk ? (tokens + kCountChunk - 1) / kCountChunk : 0;
}

bool aligned(const void* p, int64_t ld, int64_t bytes, int64_t to) {
  return reinterpret_cast<uintptr_t>(p) % to == 0 && ld * bytes % to == 0;
}

// Sizes whose launches hold fewer than 2^32 threads (and token counts in 32 bits).
bool sane(int64_t seqs, int64_t tokens) {
  return tokens <= INT32_MAX && seqs <= ((int64_t)1 << 35) / (tokens > 0 ? tokens : 1);
}

}  // namespace

extern "C" {

int64_t rv_pref_loss_workspace_bytes(int64_t pairs, int64_t tokens) {
  if (pairs <= 0 || tokens < 0) return -(int64_t)RV_ERR_BAD_SIZE;
  if (!sane(2 * pairs, tokens)) return -(int64_t)RV_ERR_UNSUPPORTED;
  return pref_plan(pairs, tokens).bytes;
}

int rv_pref_loss(const float* logp, int64_t ld_logp, const float* ref, int64_t ld_ref,
                 const uint8_t* mask, int64_t ld_mask, int64_t pairs, int64_t tokens, double beta,
                 double smoothing, int average, float* loss, float* reward, float* coef,
                 void* workspace, int64_t workspace_bytes, void* stream) {
  if (pairs <= 0 || tokens < 0 || ld_logp < 0 || ld_ref < 0 || ld_mask < 0) return RV_ERR_BAD_SIZE;
  if ((tokens > 0 && (!logp || !ref)) || !loss || !reward || !coef) return RV_ERR_NULL_POINTER;
  if (!sane(2 * pairs, tokens)) return RV_ERR_UNSUPPORTED;
  const PrefPlan p = pref_plan(pairs, tokens);
  if (!workspace || workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(workspace) % 8)
    return RV_ERR_WORKSPACE;
  char* ws = static_cast<char*>(workspace);
  PrefArgs a{logp, ld_logp, ref, ld_ref, mask, ld_mask, pairs, tokens, beta, smoothing, average,
             aligned(logp, ld_logp, 4, 16) && aligned(ref, ld_ref, 4, 16) &&
                 aligned(mask, ld_mask, 1, 4),
             loss, reward, coef, reinterpret_cast<double*>(ws),
             reinterpret_cast<double*>(ws + p.sum_at), reinterpret_cast<int*>(ws + p.count_at),
             p.chunks, kChunk};
  const hipStream_t s = (hipStream_t)stream;
  const dim3 block(kThreads);
  if (p.chunks) {
    const int64_t units = 2 * pairs * p.chunks;
    hipLaunchKernelGGL(pref_chunks_k, dim3((unsigned)((units + kWaves - 1) / kWaves)), block, 0, s,
                       a);
    hipLaunchKernelGGL(pref_join_k, dim3((unsigned)p.blocks), block, 0, s, a);
  } else {
    hipLaunchKernelGGL(pref_pairs_k, dim3((unsigned)p.blocks), block, 0, s, a, lanes_of(tokens));
  }
  if (p.blocks > 1)
    hipLaunchKernelGGL(pref_total_k, dim3(1), block, 0, s, a.part_loss, p.blocks, pairs, loss);
  return rv_host::check_launch();
}

int rv_pref_grad(const float* coef, const uint8_t* mask, int64_t ld_mask, const float* grad,
                 int64_t seqs, int64_t tokens, float* dlogp, void* stream) {
  if (seqs < 0 || tokens < 0 || ld_mask < 0) return RV_ERR_BAD_SIZE;
  if (seqs == 0 || tokens == 0) return RV_OK;
  if (!coef || !grad || !dlogp) return RV_ERR_NULL_POINTER;
  if (!sane(seqs, tokens) || !rv_host::aligned16(dlogp)) return RV_ERR_UNSUPPORTED;
  const int64_t n = seqs * tokens;
  const dim3 grid((unsigned)blocks_of((n + 3) / 4)), block(kThreads);
  const hipStream_t s = (hipStream_t)stream;
  if (mask && ld_mask == tokens && aligned(mask, 0, 1, 4))
    hipLaunchKernelGGL(pref_grad_k<true>, grid, block, 0, s, coef, mask, ld_mask, grad, n, tokens,
                       dlogp);
  else
    hipLaunchKernelGGL(pref_grad_k<false>, grid, block, 0, s, coef, mask, ld_mask, grad, n, tokens,
                       dlogp);
  return rv_host::check_launch();
}

int64_t rv_policy_loss_workspace_bytes(int64_t seqs, int64_t tokens, int per_sequence) {
  if (seqs < 0 || tokens < 0) return -(int64_t)RV_ERR_BAD_SIZE;
  if (!sane(seqs, tokens)) return -(int64_t)RV_ERR_UNSUPPORTED;
  return blocks_of((seqs * tokens + 3) / 4) * 32 +
         (per_sequence ? seqs * 4 + seqs * count_chunks(tokens) * 4 : 0);
}

int rv_policy_loss(const float* logp, int64_t ld_logp, const float* old_logp, int64_t ld_old,
                   const float* ref, int64_t ld_ref, const float* adv, int64_t adv_row,
                   int64_t adv_col, const uint8_t* mask, int64_t ld_mask, int64_t seqs,
                   int64_t tokens, double clip_low, double clip_high, double kl_coef,
                   int per_sequence, float* loss, float* stats, float* slope, void* workspace,
                   int64_t workspace_bytes, void* stream) {
  if (seqs < 0 || tokens < 0 || ld_logp < 0 || ld_old < 0 || ld_ref < 0 || ld_mask < 0 ||
      adv_row < 0 || adv_col < 0)
    return RV_ERR_BAD_SIZE;
  if (!(clip_low >= 0.0 && clip_low < 1.0) || !(clip_high >= 0.0)) return RV_ERR_BAD_SIZE;
  if (!loss || !stats || (seqs > 0 && tokens > 0 && (!logp || !old_logp || !adv))) return RV_ERR_NULL_POINTER;
  if (!sane(seqs, tokens) || (slope && !rv_host::aligned16(slope))) return RV_ERR_UNSUPPORTED;
  const int64_t blocks = blocks_of((seqs * tokens + 3) / 4);
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 8 ||
      workspace_bytes < rv_policy_loss_workspace_bytes(seqs, tokens, per_sequence))
    return RV_ERR_WORKSPACE;
  PolicyArgs a{logp, ld_logp, old_logp, ld_old, ref, ld_ref, adv, adv_row, adv_col, mask, ld_mask,
               seqs, tokens, std::log1p(-clip_low), std::log1p(clip_high), (float)(1.0 - clip_low),
               (float)(1.0 + clip_high), (float)kl_coef, nullptr, loss, stats, slope,
               static_cast<double*>(workspace)};
  const hipStream_t s = (hipStream_t)stream;
  const dim3 block(kThreads);
  if (per_sequence) {
    float* weight = reinterpret_cast<float*>(a.part + blocks * 4);
    a.weight = weight;
    const int64_t chunks = mask && seqs > 0 ? count_chunks(tokens) : 0;
    const int lanes = lanes_of(tokens / 4);
    const int64_t wgs = chunks ? seqs * chunks : (seqs * lanes + kThreads - 1) / kThreads;
    if (wgs * kThreads >= (int64_t)1 << 32) return RV_ERR_UNSUPPORTED;  // threads a launch holds
    if (chunks) {
      int* part = reinterpret_cast<int*>(weight + seqs);
      hipLaunchKernelGGL(policy_count_k, dim3((unsigned)wgs), block, 0, s, mask, ld_mask, tokens,
                         kCountChunk, chunks, part);
      hipLaunchKernelGGL(policy_join_k, dim3((unsigned)((seqs + kWaves - 1) / kWaves)), block, 0, s,
                         part, seqs, chunks, weight);
    } else if (wgs > 0) {
      hipLaunchKernelGGL(policy_weight_k, dim3((unsigned)wgs), block, 0, s, mask, ld_mask, seqs,
                         tokens, lanes, weight);
    }
  }
  const bool flat = aligned(logp, 0, 4, 16) && aligned(old_logp, 0, 4, 16) &&
                    aligned(ref, 0, 4, 16) && aligned(mask, 0, 1, 4) && ld_logp == tokens &&
                    ld_old == tokens && (!ref || ld_ref == tokens) && (!mask || ld_mask == tokens);
  if (flat) hipLaunchKernelGGL(policy_loss_k<true>, dim3((unsigned)blocks), block, 0, s, a);
  else hipLaunchKernelGGL(policy_loss_k<false>, dim3((unsigned)blocks), block, 0, s, a);
  if (blocks > 1) hipLaunchKernelGGL(policy_total_k, dim3(1), block, 0, s, a, (int)blocks);
  return rv_host::check_launch();
}

int rv_policy_grad(const float* slope, const float* factor, const float* grad, int64_t n,
                   float* dlogp, void* stream) {
  if (n < 0) return RV_ERR_BAD_SIZE;
  if (n == 0) return RV_OK;
  if (!slope || !factor || !grad || !dlogp) return RV_ERR_NULL_POINTER;
  if (!rv_host::aligned16(slope) || !rv_host::aligned16(dlogp)) return RV_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(policy_grad_k, dim3((unsigned)blocks_of((n + 3) / 4)), dim3(kThreads), 0,
                     (hipStream_t)stream, slope, factor, grad, n, dlogp);
  return rv_host::check_launch();
}

}  // extern "C"
