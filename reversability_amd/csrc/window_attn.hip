// Sliding-window causal attention with sinks on the packed projection, forward and
// backward, for gfx950 on MFMA.
//
//   s_ij = q_i . k_j / sqrt(hd)   where j <= i and (i - j < window or j < sinks)
//   p = softmax_j s,  o = p v
//   dv = p^T do,  ds = p (do v^T - rowsum(do o)),  dq = ds k / sqrt(hd),
//   dk = ds^T q / sqrt(hd); dk and dv are summed over the query heads that share a key head
//
// Layouts: qkv 16-bit [B][T][H + 2 KV][HD]: H query heads, KV key heads, KV value
// heads (query head h reads key head h / (H / KV)); out and dout [B][T][H][HD];
// lse and delta fp32 [B*H][T]; dqkv in qkv's layout.
//
// The kernels are the causal ones' (attention.hip: one workgroup of 4 waves = 128
// queries or keys, tiles of 64 streamed through two LDS buffers, online softmax in
// base 2, no atomics) with the tiles that no query of the workgroup sees left out:
// forward and dQ stream the tiles of the sinks and then those of the window; dK/dV
// streams the queries whose window reaches the keys, for the keys of the sinks all
// queries behind them.  Tiles and operands: attn_tile.h.
//
// dK/dV: a key block's work is (heads that share it) x (tiles of queries).  It is cut into
// chunks where a block alone would take much longer than the rest (the sinks' block
// sees the whole sequence) or where there are few blocks; a chunk writes fp32 partials
// and wattn_reduce_k adds them in order.
//
// P and dS are rounded to the type for the products they enter.  Where that shows it is made up
// for by a second product with what the rounding left (REST): for the first 128 queries, which see
// few keys with large weights, and the keys of the first block and of the sinks, whose sums are
// long and of large terms (16384 queries' roundings were half as large as other keys' gradients).
// Of every output the forward also keeps what its rounding left (rest), for D = rowsum(dO O).
// Error of the gradients relative to that of the final rounding alone: without all this 1.5
// to 2.1, with it 1.0 to 1.3, at a few percent of the time.
//
// Measured (us; forward, dQ, dK/dV, sums, each by itself under the profiler, where they run up to 10%
// longer; the whole pass in a row of them; window and sinks behind the comma), with the whole pass's
// rate over the visible pairs' 4 + 10 HD flops:
//   33 x 512, 8 heads of 32, 128 + 4, fp16          23   28        32    5     103   69 TFLOP/s
//   3 x 1999, 20 heads of 64 over 4, 500 + 3, bf16  42   65        65   11     164   288
//   2 x 16384, 10 heads of 128, 2048 + 4, bf16     453   18 + 570  998  14    1840   614
// Short windows are bound by waits: a workgroup has four to eleven tiles, so that its start, the loads
// of its first tiles and its end show; VALU 27-38% busy (an exponential counted as four other
// instructions), matrix cores 4-7% at head size 32 and 14-20% at 64.  Long ones by products and
// softmax that overlap in part: matrix cores 35% and VALU 39% busy in the forward, 42 and 32 in
// dQ, 31 and 22 in dK/dV, whose 128 accumulators and 64 operands leave one wave per SIMD (two spill:
// 1500 us).  The forward at head size 64 spills 11 of its 128 registers to scratch.

#include <algorithm>
#include <cmath>

#include "attn_tile.h"

namespace {

using namespace rv_attn;

struct Geometry {
  int T, H, KV, window, sinks;
};

// Workgroups per CU the register budget is sized for (attention.hip's figures).
template <int HD>
constexpr int kFwdMinBlocks = HD == 128 ? 2 : (HD == 64 ? 4 : 2);
template <int HD>
constexpr int kKvMinBlocks = HD == 128 ? 1 : 2;

// The key tiles that queries [q0, q0 + rows) see: tiles [0, ns) hold sinks, tiles
// [first, end) the window.
struct KeyTiles {
  int ns, first, end;
  __device__ __forceinline__ KeyTiles(const Geometry& g, int q0, int rows) {
    const int last = min(g.T, q0 + rows);
    end = (last + kTile - 1) / kTile;
    ns = min((g.sinks + kTile - 1) / kTile, end);
    first = max(ns, max(0, q0 - g.window + 1) / kTile);
  }
  __device__ __forceinline__ int count() const { return ns + end - first; }
  __device__ __forceinline__ int at(int t) const { return t < ns ? t : first + t - ns; }
};

// Workgroups are dealt to the eight XCDs in turn, each with an L2 of its own: the number that gives
// each XCD a stretch of neighbours, which read the same keys or queries.
__device__ __forceinline__ int near_index() {
  const int n = (int)gridDim.x, x = (int)blockIdx.x % 8, per = n / 8, more = n % 8;
  return x * per + min(x, more) + (int)blockIdx.x / 8;
}

// Whether no / every query of [q0, q0 + 31] sees any / all of the keys [k0, k0 + n).
__device__ __forceinline__ bool none_seen(const Geometry& g, int q0, int k0, int n) {
  return k0 > q0 + kWaveRows - 1 || (k0 + n - 1 <= q0 - g.window && k0 >= g.sinks);
}
__device__ __forceinline__ bool all_seen(const Geometry& g, int q0, int k0, int n) {
  return k0 + n - 1 <= q0 && (k0 > q0 + kWaveRows - 1 - g.window || k0 + n <= g.sinks);
}

// What a lane with one query sees of keys k0 + r, r the lane's row of a tile of keys (no
// branches: two comparisons an element): the window, or the sinks among the keys up to its own.
struct QuerySight {
  int at, sinks;  // query - k0, and sinks up to the query - k0
  unsigned window;
  __device__ __forceinline__ QuerySight(const Geometry& g, int q, int k0)
      : at(q - k0), sinks(min(g.sinks, q + 1) - k0), window((unsigned)g.window) {}
  __device__ __forceinline__ bool operator()(int r) const {
    return ((unsigned)(at - r) < window) | (r < sinks);
  }
};

// Which queries q0 + r a lane with one key is seen by.
struct KeySight {
  int at;  // q0 - key
  unsigned reach;
  __device__ __forceinline__ KeySight(const Geometry& g, int key, int q0)
      : at(q0 - key), reach(key < g.sinks ? 0x80000000u : (unsigned)g.window) {}
  __device__ __forceinline__ bool operator()(int r) const { return (unsigned)(at + r) < reach; }
};

// What the rounding of values 8 h .. 8 h + 7 of an accumulator to `r` left, rounded in its turn.
template <typename E>
__device__ __forceinline__ x8<E> rest8(const f32x16& v, const x8<E>& r, int h) {
  x8<E> left;
#pragma unroll
  for (int i = 0; i < 8; ++i) left[i] = (E)(v[8 * h + i] - (float)r[i]);
  return left;
}

template <int HD>
struct FwdState {
  f32x16 o[HD / 32];
  float m, l;
};

// 32 keys (rows sub * 32 .. of the tile) for one wave's 32 queries.  MASK: some of them are not
// seen by some query; q, k0: the lane's query and the first of the keys.
// REST: what P's roundings left is added by a product of its own.
template <typename E, int HD, bool MASK, bool REST>
__device__ __forceinline__ void fwd_rows(FwdState<HD>& st, const E* Ks, const E* Vs,
                                         const FragOffsets<HD, E>& fo, const x8<E> (&qf)[HD / 16],
                                         const Geometry& g, int sub, int q, int k0, float c,
                                         int lane) {
  constexpr int KK = HD / 16, DT = HD / 32;
  const int hl = lane >> 5;
  prio_mfma();
  x8<E> kf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) kf[kk] = fo.rowf(Ks, sub, kk);
  if constexpr (kReadAhead<HD>) __builtin_amdgcn_sched_barrier(0);
  f32x16 s = mfma(kf[0], qf[0], zero16());
#pragma unroll
  for (int kk = 1; kk < KK; ++kk) s = mfma(kf[kk], qf[kk], s);
  prio_valu();
  float mx = -INFINITY;
  const QuerySight sees(g, q, k0 + hl * 4);
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    if constexpr (MASK) s[j] = sees(acc_row(j)) ? s[j] : -INFINITY;
    mx = fmaxf(mx, s[j]);
  }
  const float mxc = pair_max(mx) * c;
  if (__any(mxc > st.m + kLazy)) {
    // (a row that has seen no key yet keeps m = -inf; its factor is never used)
    const float m_new = fmaxf(st.m, mxc);
    const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(st.m - m_new);
    st.m = m_new;
    st.l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) st.o[dt][e] *= alpha;
  }
  const float neg_m = MASK && st.m == -INFINITY ? 0.f : -st.m;
  x8<E> vf[2][DT];
  if constexpr (kReadAhead<HD>) {
#pragma unroll
    for (int cc = 0; cc < 2; ++cc)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) vf[cc][dt] = fo.trf(Vs, sub, cc, dt);
    __builtin_amdgcn_sched_barrier(0);
  }
  float rowsum = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float p = __builtin_amdgcn_exp2f(fmaf(s[j], c, neg_m));
    rowsum += p;
    s[j] = p;
  }
  st.l += rowsum;
  prio_mfma_tail();
#pragma unroll
  for (int cc = 0; cc < 2; ++cc) {
    const x8<E> pf = pack8<E>(s, cc);
    x8<E> left;
    if constexpr (REST) left = rest8<E>(s, pf, cc);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      if constexpr (!kReadAhead<HD>) vf[cc][dt] = fo.trf(Vs, sub, cc, dt);
      st.o[dt] = mfma(vf[cc][dt], pf, st.o[dt]);
      if constexpr (REST) st.o[dt] = mfma(vf[cc][dt], left, st.o[dt]);
    }
  }
}

template <typename E, int HD, bool REST>
__device__ __forceinline__ void fwd_block(const E* __restrict__ qkv, E* __restrict__ out,
                                          E* __restrict__ rest, float* __restrict__ lse,
                                          const Geometry& g, int bh, int qt, float c,
                                          E (&lds)[2][2][kTile * HD]) {
  constexpr int KK = HD / 16, DT = HD / 32;
  const int b = bh / g.H, h = bh % g.H, kvh = h / (g.H / g.KV);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hl = lane >> 5;
  const int64_t rs = (int64_t)(g.H + 2 * g.KV) * HD;
  const E* base = qkv + (int64_t)b * g.T * rs;
  const E* qb = base + (int64_t)h * HD;
  const E* kb = base + (int64_t)(g.H + kvh) * HD;
  const E* vb = kb + (int64_t)g.KV * HD;
  const int q0 = qt * kBlockRows + wave * kWaveRows;
  const int q = q0 + (lane & 31);
  const FragOffsets<HD, E> fo(lane);

  x8<E> qf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk)
    qf[kk] = q < g.T ? *reinterpret_cast<const x8<E>*>(qb + (int64_t)q * rs + kk * 16 + hl * 8)
                     : x8<E>{};
  FwdState<HD> st;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) st.o[dt] = zero16();
  st.m = -INFINITY;
  st.l = 0.f;

  const KeyTiles tiles(g, qt * kBlockRows, kBlockRows);
  const int n = tiles.count();
  TileCopy<HD> ck(rs), cv(rs);
  ck.load(kb, rs, tiles.at(0) * kTile, g.T);
  cv.load(vb, rs, tiles.at(0) * kTile, g.T);
  ck.store(lds[0][0]);
  cv.store(lds[0][1]);
  __syncthreads();
  // Tile t lives in buffer t % 2; the loop body is written out for both
  // buffers so that each buffer's LDS address is a constant.
#define RV_FWD_STEP(BUF)                                                                     \
  {                                                                                          \
    const int k0 = tiles.at(t) * kTile;                                                      \
    const bool more = t + 1 < n;                                                             \
    if (more) {                                                                              \
      const int next = tiles.at(t + 1) * kTile;                                              \
      ck.load(kb, rs, next, g.T);                                                            \
      cv.load(vb, rs, next, g.T);                                                            \
    }                                                                                        \
    _Pragma("unroll") for (int sub = 0; sub < 2; ++sub) {                                    \
      const int ks = k0 + sub * 32;                                                          \
      if (none_seen(g, q0, ks, 32)) continue;                                                \
      if (all_seen(g, q0, ks, 32))                                                           \
        fwd_rows<E, HD, false, REST>(st, lds[BUF][0], lds[BUF][1], fo, qf, g, sub, q, ks, c, \
                                     lane);                                                  \
      else                                                                                   \
        fwd_rows<E, HD, true, REST>(st, lds[BUF][0], lds[BUF][1], fo, qf, g, sub, q, ks, c,  \
                                    lane);                                                   \
    }                                                                                        \
    if (more) {                                                                              \
      ck.store(lds[1 - (BUF)][0]);                                                           \
      cv.store(lds[1 - (BUF)][1]);                                                           \
    }                                                                                        \
    __syncthreads();                                                                         \
  }
  for (int t = 0; t < n; ++t) {
    RV_FWD_STEP(0)
    if (++t >= n) break;
    RV_FWD_STEP(1)
  }
#undef RV_FWD_STEP
  const float l = pair_sum(st.l);
  if (q < g.T) {
    const float inv = 1.0f / l;
    const int64_t row = (((int64_t)b * g.T + q) * g.H + h) * HD;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int jg = 0; jg < 4; ++jg) {
        const int64_t at = row + dt * 32 + jg * 8 + hl * 4;
        x4<E> v, r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = st.o[dt][4 * jg + e] * inv;
          v[e] = (E)x;
          r[e] = (E)(x - (float)v[e]);
        }
        *reinterpret_cast<x4<E>*>(out + at) = v;
        if (rest) *reinterpret_cast<x4<E>*>(rest + at) = r;
      }
    if (hl == 0) lse[(int64_t)bh * g.T + q] = st.m + __log2f(l);
  }
}

template <typename E, int HD>
__global__ __launch_bounds__(kThreads, kFwdMinBlocks<HD>)
void wattn_fwd_k(const E* __restrict__ qkv, E* __restrict__ out, E* __restrict__ rest,
                 float* __restrict__ lse, Geometry g, int n_qt, float c) {
  __shared__ __attribute__((aligned(16))) E lds[2][2][kTile * HD];
  const int at = near_index(), bh = at / n_qt, qt = at % n_qt;
  if (qt == 0) fwd_block<E, HD, true>(qkv, out, rest, lse, g, bh, qt, c, lds);
  else fwd_block<E, HD, false>(qkv, out, rest, lse, g, bh, qt, c, lds);
}

// ---------------------------------------------------------------------------
// Backward.
// ---------------------------------------------------------------------------
// fp16's dS loses digits below 2^-14 and vanishes below 2^-25, where dK and dQ are sums of thousands
// of such terms: gradients of 2^-10 came out three times as far off as their own rounding, those of
// 2^-12 over 6000 tokens ten times.  Everything behind dO is linear in it, so dS is made of dO times
// a power of two that brings its largest element into [1/4, 1/2) -- a query's own in dQ, that of a
// tile of 64 queries in dK/dV, where the sums are moved from one power to the next -- and the sums
// are divided by it: exact.  Never a smaller power than 1: gradients of 1/4 and more are as they are.
// (|dS| <= max |dO v| / 2: it overflows where values above 2000 agree with dO in sign in
// every column.)  us of dQ and dK/dV in fp16, without and with: 33 x 512, heads of 32, 25.1 -> 27.1
// and 31.3 -> 31.1; 3 x 1999, heads of 64, 64.7 -> 66.6 and 68.3 -> 70.4; 2 x 16384, heads of 128,
// 600 -> 605 and 1058 -> 1120 (a power for each 32 queries 1240: the moves cut the loop's code).
template <typename E>
constexpr bool kScaled = false;
template <>
constexpr bool kScaled<_Float16> = true;

// The power of two for gradients of at most `top`, itself a fp16 number.
__device__ __forceinline__ float grad_scale(float top) {
  const int exponent = (int)(__float_as_uint(top) >> 23 & 255u) - 127;  // top is in [2^e, 2^(e + 1))
  return __uint_as_float((unsigned)(127 + min(max(-2 - exponent, 0), 15)) << 23);
}
// 1 / x of a power of two.
__device__ __forceinline__ float inverse_power(float x) {
  return __uint_as_float((254u << 23) - __float_as_uint(x));
}

// dQ contribution of 32 staged keys to one wave's 32 queries (lanes).  REST: what the roundings of dS
// left is added by a product of its own.
template <typename E, int HD, bool MASK, bool REST>
__device__ __forceinline__ void q_rows(f32x16 (&dq)[HD / 32], const E* Ks, const E* Vs,
                                       const FragOffsets<HD, E>& fo, const x8<E> (&qf)[HD / 16],
                                       const x8<E> (&gf)[HD / 16], const Geometry& g, float Lq,
                                       float Dq, int sub, int q, int k0, float c, int lane) {
  constexpr int KK = HD / 16, DT = HD / 32;
  const int hl = lane >> 5;
  prio_mfma();
  // half of the row operands at a time: all of them do not fit in the registers
  constexpr int KH = KK > 4 ? 4 : KK > 2 ? 2 : KK;
  f32x16 s = zero16(), dp = zero16();
#pragma unroll
  for (int k0h = 0; k0h < KK; k0h += KH) {
    x8<E> kf[KH], vf[KH];
#pragma unroll
    for (int kk = 0; kk < KH; ++kk) {
      kf[kk] = fo.rowf(Ks, sub, k0h + kk);
      vf[kk] = fo.rowf(Vs, sub, k0h + kk);
    }
#pragma unroll
    for (int kk = 0; kk < KH; ++kk) {
      s = mfma(kf[kk], qf[k0h + kk], s);
      dp = mfma(vf[kk], gf[k0h + kk], dp);
    }
  }
  x8<E> kt[2][DT];
  const float neg_l = -Lq;
  prio_valu();
  const QuerySight sees(g, q, k0 + hl * 4);
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float p = __builtin_amdgcn_exp2f(fmaf(s[j], c, neg_l));
    dp[j] = p * (dp[j] - Dq);
    if constexpr (MASK) dp[j] = sees(acc_row(j)) ? dp[j] : 0.f;
  }
#pragma unroll
  for (int cc = 0; cc < 2; ++cc) {
    const x8<E> dsf = pack8<E>(dp, cc);
    x8<E> left;
    if constexpr (REST) left = rest8<E>(dp, dsf, cc);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      kt[cc][dt] = fo.trf(Ks, sub, cc, dt);
      dq[dt] = mfma(kt[cc][dt], dsf, dq[dt]);
      if constexpr (REST) dq[dt] = mfma(kt[cc][dt], left, dq[dt]);
    }
  }
}

// The first blocks of queries and the others in one launch or, where the first ones' products cost the
// others registers, in two: at HD = 128 (559 us against 1170 in one), and at HD = 64 with more blocks than
// the chip runs in a few rounds (forward and backward, ten in a row from the host: 16 x 2048, 16 heads
// 572 us against 603, 2 x 16384, 8 heads 733 against 769; 3 x 1999, 20 heads 182 against 179, 8 x 700,
// 8 heads 113 against 110).
enum Part { kAll, kFirst, kOthers };
constexpr int64_t kOneLaunch = 1024;  // blocks, at HD = 64

template <int HD, Part PART>
constexpr int kQMinBlocks = HD == 64 && PART != kAll ? 3 : 2;

template <typename E, int HD, Part PART>
__global__ __launch_bounds__(kThreads, (kQMinBlocks<HD, PART>))
void wattn_bwd_q_k(const E* __restrict__ qkv, const E* __restrict__ out,
                   const E* __restrict__ rest, const E* __restrict__ dout,
                   const float* __restrict__ lse, float* __restrict__ delta,
                   float* __restrict__ tops, E* __restrict__ dqkv, Geometry g, int n_qt, float c,
                   float scale) {
  constexpr int KK = HD / 16, DT = HD / 32;
  __shared__ __attribute__((aligned(16))) E lds[2][2][kTile * HD];  // [buf][K / V]
  const int per = PART == kFirst ? 1 : PART == kOthers ? n_qt - 1 : n_qt;
  const int number = near_index(), bh = number / per, qt = number % per + (PART == kOthers);
  const bool first = PART == kFirst || (PART == kAll && qt == 0);
  const int b = bh / g.H, h = bh % g.H, kvh = h / (g.H / g.KV);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hl = lane >> 5;
  const int64_t rs = (int64_t)(g.H + 2 * g.KV) * HD, os = (int64_t)g.H * HD;
  const E* base = qkv + (int64_t)b * g.T * rs;
  const E* qb = base + (int64_t)h * HD;
  const E* kb = base + (int64_t)(g.H + kvh) * HD;
  const E* vb = kb + (int64_t)g.KV * HD;
  const E* gb = dout + (int64_t)b * g.T * os + (int64_t)h * HD;
  const int64_t o0 = (int64_t)b * g.T * os + (int64_t)h * HD;
  const int q0 = qt * kBlockRows + wave * kWaveRows;
  const int q = q0 + (lane & 31);
  const bool qok = q < g.T;

  x8<E> qf[KK], gf[KK];
  // delta = sum_d dO O over the query's row (O with what its rounding left): this lane's
  // HD / 2 columns (the fragments' layout), then the other half from lane l ^ 32
  float dsum = 0.f;
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    const int64_t col = kk * 16 + hl * 8;
    qf[kk] = qok ? *reinterpret_cast<const x8<E>*>(qb + (int64_t)q * rs + col) : x8<E>{};
    gf[kk] = qok ? *reinterpret_cast<const x8<E>*>(gb + (int64_t)q * os + col) : x8<E>{};
    const int64_t at = o0 + (int64_t)q * os + col;
    const x8<E> of = qok ? *reinterpret_cast<const x8<E>*>(out + at) : x8<E>{};
    const x8<E> ol = qok && rest ? *reinterpret_cast<const x8<E>*>(rest + at) : x8<E>{};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      dsum = fmaf((float)gf[kk][i], (float)of[i] + (float)ol[i], dsum);
  }
  const float Lq = qok ? lse[(int64_t)bh * g.T + q] : 0.f;
  float Dq = pair_sum(dsum);
  if (qok && hl == 0) delta[(int64_t)bh * g.T + q] = Dq;
  if constexpr (kScaled<E>) {
    float top = 0.f;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf((float)gf[kk][i]));
    top = pair_max(top);
    const float power = grad_scale(top);
    scale *= inverse_power(power);
    Dq *= power;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) gf[kk] *= (E)power;
#pragma unroll
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    if (lane == 0 && qok) tops[(int64_t)bh * ((g.T + 31) / 32) + q0 / 32] = top;
  }
  f32x16 dq[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dq[dt] = zero16();

  const KeyTiles tiles(g, qt * kBlockRows, kBlockRows);
  const int n = tiles.count();
  TileCopy<HD> ck(rs), cv(rs);
  ck.load(kb, rs, tiles.at(0) * kTile, g.T);
  cv.load(vb, rs, tiles.at(0) * kTile, g.T);
  ck.store(lds[0][0]);
  cv.store(lds[0][1]);
  __syncthreads();
  const FragOffsets<HD, E> fo(lane);
#define RV_Q_STEP(BUF)                                                                        \
  {                                                                                           \
    const int k0 = tiles.at(t) * kTile;                                                       \
    const bool more = t + 1 < n;                                                              \
    if (more) {                                                                               \
      const int next = tiles.at(t + 1) * kTile;                                               \
      ck.load(kb, rs, next, g.T);                                                             \
      cv.load(vb, rs, next, g.T);                                                             \
    }                                                                                         \
    _Pragma("unroll") for (int sub = 0; sub < 2; ++sub) {                                     \
      const int ks = k0 + sub * 32;                                                           \
      if (none_seen(g, q0, ks, 32)) continue;                                                 \
      if (first)                                                                               \
        q_rows<E, HD, true, PART != kOthers>(dq, lds[BUF][0], lds[BUF][1], fo, qf, gf, g, Lq,  \
                                             Dq, sub, q, ks, c, lane);                         \
      else if (all_seen(g, q0, ks, 32))                                                        \
        q_rows<E, HD, false, false>(dq, lds[BUF][0], lds[BUF][1], fo, qf, gf, g, Lq, Dq, sub,  \
                                    q, ks, c, lane);                                           \
      else                                                                                     \
        q_rows<E, HD, true, false>(dq, lds[BUF][0], lds[BUF][1], fo, qf, gf, g, Lq, Dq, sub,   \
                                   q, ks, c, lane);                                            \
    }                                                                                         \
    if (more) {                                                                               \
      ck.store(lds[1 - (BUF)][0]);                                                            \
      cv.store(lds[1 - (BUF)][1]);                                                            \
    }                                                                                         \
    __syncthreads();                                                                          \
  }
  for (int t = 0; t < n; ++t) {
    RV_Q_STEP(0)
    if (++t >= n) break;
    RV_Q_STEP(1)
  }
#undef RV_Q_STEP
  if (qok) {
    E* qrow = dqkv + ((int64_t)b * g.T + q) * rs + (int64_t)h * HD;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int jg = 0; jg < 4; ++jg)
        store4<E>(qrow + dt * 32 + jg * 8 + hl * 4, dq[dt][4 * jg] * scale,
                  dq[dt][4 * jg + 1] * scale, dq[dt][4 * jg + 2] * scale,
                  dq[dt][4 * jg + 3] * scale);
  }
}

// dK/dV contribution of 32 staged queries (tile rows sub * 32 ..) to one wave's 32 keys
// (lanes).  Query rows past the sequence hold zeros (Q, dO, lse, delta): their
// P is 1 but dS = 0 and dO = 0, so they add nothing.  REST: what the roundings of P and dS left is
// added by products of its own.  power: what dS is multiplied by (and Ds already is).
template <typename E, int HD, bool MASK, bool REST>
__device__ __forceinline__ void kv_rows(f32x16 (&dk)[HD / 32], f32x16 (&dv)[HD / 32], const E* Qs,
                                        const E* Gs, const float* Ls, const float* Ds,
                                        const FragOffsets<HD, E>& fo, const x8<E> (&kf)[HD / 16],
                                        const x8<E> (&vf)[HD / 16], const Geometry& g, int sub,
                                        int q0, int key, float c, float power, int lane) {
  constexpr int KK = HD / 16, DT = HD / 32;
  const int hl = lane >> 5;
  prio_mfma();
  x8<E> qf[KK], gf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    qf[kk] = fo.rowf(Qs, sub, kk);
    gf[kk] = fo.rowf(Gs, sub, kk);
  }
  if constexpr (kReadAhead<HD>) __builtin_amdgcn_sched_barrier(0);
  f32x16 s = mfma(qf[0], kf[0], zero16());
  f32x16 dp = mfma(gf[0], vf[0], zero16());
#pragma unroll
  for (int kk = 1; kk < KK; ++kk) {
    s = mfma(qf[kk], kf[kk], s);
    dp = mfma(gf[kk], vf[kk], dp);
  }
  x8<E> qt[2][DT], gt[2][DT];
  if constexpr (kReadAhead<HD>) {  // the second half's do not fit in the registers
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      gt[0][dt] = fo.trf(Gs, sub, 0, dt);
      qt[0][dt] = fo.trf(Qs, sub, 0, dt);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  prio_valu();
  const KeySight seen(g, key, q0 + hl * 4);
#pragma unroll
  for (int jg = 0; jg < 4; ++jg) {
    const int r4 = sub * 32 + jg * 8 + hl * 4;
    const float4 L4 = *reinterpret_cast<const float4*>(Ls + r4);
    const float4 D4 = *reinterpret_cast<const float4*>(Ds + r4);
    const float Lr[4] = {L4.x, L4.y, L4.z, L4.w};
    const float Dr[4] = {D4.x, D4.y, D4.z, D4.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = 4 * jg + e;
      const float p = __builtin_amdgcn_exp2f(fmaf(s[j], c, -Lr[e]));
      const float d = p * (kScaled<E> ? fmaf(dp[j], power, -Dr[e]) : dp[j] - Dr[e]);
      const bool on = !MASK || seen(acc_row(j));
      s[j] = on ? p : 0.f;
      dp[j] = on ? d : 0.f;
    }
  }
#pragma unroll
  for (int cc = 0; cc < 2; ++cc) {
    const x8<E> pf = pack8<E>(s, cc), dsf = pack8<E>(dp, cc);
    x8<E> pl, dsl;
    if constexpr (REST) {
      pl = rest8<E>(s, pf, cc);
      dsl = rest8<E>(dp, dsf, cc);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      if (cc == 1 || !kReadAhead<HD>) {
        gt[cc][dt] = fo.trf(Gs, sub, cc, dt);
        qt[cc][dt] = fo.trf(Qs, sub, cc, dt);
      }
      dv[dt] = mfma(gt[cc][dt], pf, dv[dt]);
      dk[dt] = mfma(qt[cc][dt], dsf, dk[dt]);
      if constexpr (REST) {
        dv[dt] = mfma(gt[cc][dt], pl, dv[dt]);
        dk[dt] = mfma(qt[cc][dt], dsl, dk[dt]);
      }
    }
  }
}

// How the dK/dV work of one (sequence, key head) is cut into chunks: key blocks
// [0, sink_blocks), the first and those that hold sinks, take sink_chunks of sink_len steps each, the rest
// near_chunks of near_len.  A step is one tile of queries of one head that shares the keys.
struct KvPlan {
  int blocks, sink_blocks;
  int sink_chunks, sink_len, near_chunks, near_len;
  __host__ __device__ int units() const {
    return sink_blocks * sink_chunks + (blocks - sink_blocks) * near_chunks;
  }
  // Only units of blocks that are cut write partials: the sinks', then the others'.
  __host__ __device__ int cut_sinks() const { return sink_chunks > 1 ? sink_blocks * sink_chunks : 0; }
  __host__ __device__ int cut_units() const {
    return cut_sinks() + (near_chunks > 1 ? (blocks - sink_blocks) * near_chunks : 0);
  }
};

// Tiles of queries that see a key of the block at kbase, the first of them kbase / kTile.
__host__ __device__ inline int query_tiles(const Geometry& g, int kbase) {
  // the last query that sees a key of the block, and one more (in 64 bits: windows are not
  // limited by the sequence)
  int64_t end = (int64_t)kbase + kBlockRows - 1 + g.window;
  if (kbase < g.sinks || end > g.T) end = g.T;
  return (int)((end - kbase + kTile - 1) / kTile);
}

// One unit of the plan, of the sinks' blocks (SINK) or of the others.
template <typename E, int HD, bool SINK>
__device__ __forceinline__ void kv_unit(const E* __restrict__ qkv, const E* __restrict__ dout,
                                        const float* __restrict__ lse,
                                        const float* __restrict__ delta,
                                        const float* __restrict__ tops, E* __restrict__ dqkv,
                                        float* __restrict__ part, const Geometry& g,
                                        const KvPlan& plan, int number, float c, float scale,
                                        E (&lds)[2][2][kTile * HD], float (&rowv)[2][2][kTile]) {
  constexpr int KK = HD / 16, DT = HD / 32;
  const int units = plan.units();
  const int bkv = number / units, unit = number % units;
  const int chunks = SINK ? plan.sink_chunks : plan.near_chunks;
  const int len = SINK ? plan.sink_len : plan.near_len;
  const int at = SINK ? unit : unit - plan.sink_blocks * plan.sink_chunks;
  const int kt = at / chunks + (SINK ? 0 : plan.sink_blocks), chunk = at % chunks;
  const int b = bkv / g.KV, kvh = bkv % g.KV, group = g.H / g.KV;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hl = lane >> 5;
  const int64_t rs = (int64_t)(g.H + 2 * g.KV) * HD, os = (int64_t)g.H * HD;
  const E* base = qkv + (int64_t)b * g.T * rs;
  const E* kb = base + (int64_t)(g.H + kvh) * HD;
  const E* vb = kb + (int64_t)g.KV * HD;
  const int kbase = kt * kBlockRows;
  const int k0w = kbase + wave * kWaveRows;
  const int key = k0w + (lane & 31);

  x8<E> kf[KK], vf[KK];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    const int64_t col = kk * 16 + hl * 8;
    const bool ok = key < g.T;
    kf[kk] = ok ? *reinterpret_cast<const x8<E>*>(kb + (int64_t)key * rs + col) : x8<E>{};
    vf[kk] = ok ? *reinterpret_cast<const x8<E>*>(vb + (int64_t)key * rs + col) : x8<E>{};
  }
  f32x16 dk[DT], dv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    dk[dt] = zero16();
    dv[dt] = zero16();
  }

  // steps [first, last) of this chunk: head by head, the tiles of queries in order
  const int per = query_tiles(g, kbase);
  const int first = chunk * len, last = min(first + len, group * per);
  TileCopy<HD> cq(rs), cg(os);
  float lv = 0.f, dvv = 0.f;
  float top[2] = {0.f, 0.f};  // the largest |dO| of the halves of the tile under way
  float power = 1.f;          // of the staged tile: what dk holds its sums times
  int head = first / per, tile = first % per;
  auto load = [&]() {  // the tile at (head, tile), then on to the next
    const int h = kvh * group + head, q0 = kbase + tile * kTile;
    cq.load(base + (int64_t)h * HD, rs, q0, g.T);
    cg.load(dout + (int64_t)b * g.T * os + (int64_t)h * HD, os, q0, g.T);
    const int64_t row = ((int64_t)b * g.H + h) * g.T;
    lv = load_rowval(lse + row, q0, g.T);
    dvv = load_rowval(delta + row, q0, g.T);
    if constexpr (kScaled<E>) {
      const int groups = (g.T + 31) / 32;
      const float* of_head = tops + ((int64_t)b * g.H + h) * groups;
      top[0] = of_head[q0 / 32];
      top[1] = of_head[min(q0 / 32 + 1, groups - 1)];
    }
    if (++tile == per) tile = 0, ++head;
  };
  auto store_rows = [&](int buf) {
    if constexpr (kScaled<E>) {
      const float next = grad_scale(fmaxf(top[0], top[1]));
      dvv *= next;
      if (__float_as_uint(next) != __float_as_uint(power)) {  // (scalars)
        const float turn = next * inverse_power(power);
        power = next;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) dk[dt] *= turn;
      }
    }
    if (threadIdx.x < kTile) {
      rowv[buf][0][threadIdx.x] = lv;
      rowv[buf][1][threadIdx.x] = dvv;
    }
  };
  const FragOffsets<HD, E> fo(lane);
  int now = first % per;  // the staged tile
  if (first < last) {
    load();
    cq.store(lds[0][0]);
    cg.store(lds[0][1]);
    store_rows(0);
  }
  // vmcnt(0): K and V are there.  The compiler does not know it where no tile was loaded, and would
  // wait for the tile under way in every step.
  __builtin_amdgcn_s_waitcnt(0x0f70);
  __syncthreads();
#define RV_KV_STEP(BUF)                                                                       \
  {                                                                                           \
    const int qt0 = kbase + now * kTile;                                                      \
    if (++now == per) now = 0;                                                                \
    const bool more = t + 1 < last;                                                           \
    if (more) load();                                                                         \
    _Pragma("unroll") for (int sub = 0; sub < 2; ++sub) {                                     \
      const int qs = qt0 + sub * 32;                                                          \
      if (none_seen(g, qs, k0w, kWaveRows)) continue;                                         \
      if constexpr (SINK)                                                                      \
        kv_rows<E, HD, true, true>(dk, dv, lds[BUF][0], lds[BUF][1], rowv[BUF][0],             \
                                   rowv[BUF][1], fo, kf, vf, g, sub, qs, key, c, power, lane); \
      else if (all_seen(g, qs, k0w, kWaveRows))                                                \
        kv_rows<E, HD, false, false>(dk, dv, lds[BUF][0], lds[BUF][1], rowv[BUF][0],           \
                                     rowv[BUF][1], fo, kf, vf, g, sub, qs, key, c, power,      \
                                     lane);                                                    \
      else                                                                                     \
        kv_rows<E, HD, true, false>(dk, dv, lds[BUF][0], lds[BUF][1], rowv[BUF][0],            \
                                    rowv[BUF][1], fo, kf, vf, g, sub, qs, key, c, power,       \
                                    lane);                                                     \
    }                                                                                         \
    if (more) {                                                                               \
      cq.store(lds[1 - (BUF)][0]);                                                            \
      cg.store(lds[1 - (BUF)][1]);                                                            \
      store_rows(1 - (BUF));                                                                  \
    }                                                                                         \
    __syncthreads();                                                                          \
  }
  for (int t = first; t < last; ++t) {
    RV_KV_STEP(0)
    if (++t >= last) break;
    RV_KV_STEP(1)
  }
#undef RV_KV_STEP
  if (key >= g.T) return;
  if constexpr (kScaled<E>) {
    const float back = inverse_power(power);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) dk[dt] *= back;
  }
  if (chunks > 1) {  // [cut unit][K / V][128][HD] fp32
    const int64_t place = (int64_t)bkv * plan.cut_units() + at + (SINK ? 0 : plan.cut_sinks());
    float* row = part + (place * 2 * kBlockRows + key - kbase) * HD;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int jg = 0; jg < 4; ++jg) {
        const int col = dt * 32 + jg * 8 + hl * 4;
        rv::st_f4(row + col, make_float4(dk[dt][4 * jg], dk[dt][4 * jg + 1], dk[dt][4 * jg + 2],
                                         dk[dt][4 * jg + 3]));
        rv::st_f4(row + (int64_t)kBlockRows * HD + col,
                  make_float4(dv[dt][4 * jg], dv[dt][4 * jg + 1], dv[dt][4 * jg + 2],
                              dv[dt][4 * jg + 3]));
      }
    return;
  }
  E* krow = dqkv + ((int64_t)b * g.T + key) * rs + (int64_t)(g.H + kvh) * HD;
  E* vrow = krow + (int64_t)g.KV * HD;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int jg = 0; jg < 4; ++jg) {
      const int col = dt * 32 + jg * 8 + hl * 4;
      store4<E>(krow + col, dk[dt][4 * jg] * scale, dk[dt][4 * jg + 1] * scale,
                dk[dt][4 * jg + 2] * scale, dk[dt][4 * jg + 3] * scale);
      store4<E>(vrow + col, dv[dt][4 * jg], dv[dt][4 * jg + 1], dv[dt][4 * jg + 2],
                dv[dt][4 * jg + 3]);
    }
}

template <typename E, int HD>
__global__ __launch_bounds__(kThreads, kKvMinBlocks<HD>)
void wattn_bwd_kv_k(const E* __restrict__ qkv, const E* __restrict__ dout,
                    const float* __restrict__ lse, const float* __restrict__ delta,
                    const float* __restrict__ tops, E* __restrict__ dqkv,
                    float* __restrict__ part, Geometry g, KvPlan plan, float c, float scale) {
  __shared__ __attribute__((aligned(16))) E lds[2][2][kTile * HD];  // [buf][Q / dO]
  __shared__ __attribute__((aligned(16))) float rowv[2][2][kTile];  // [buf][lse / delta]
  const int number = near_index();
  if (number % plan.units() < plan.sink_blocks * plan.sink_chunks)
    kv_unit<E, HD, true>(qkv, dout, lse, delta, tops, dqkv, part, g, plan, number, c, scale, lds,
                         rowv);
  else
    kv_unit<E, HD, false>(qkv, dout, lse, delta, tops, dqkv, part, g, plan, number, c, scale, lds,
                          rowv);
}

// Sums of the chunks' partials, in order.  One workgroup = 32 rows of one cut key
// block and side (K / V); grid (8 * cut blocks, B * KV), the cut blocks being the sinks', the
// others, or all.
template <typename E, int HD>
__global__ __launch_bounds__(kThreads)
void wattn_reduce_k(const float* __restrict__ part, E* __restrict__ dqkv, Geometry g, KvPlan plan,
                    float scale) {
  const int side = (blockIdx.x >> 2) & 1;
  int kt = blockIdx.x >> 3;
  if (plan.sink_chunks == 1) kt += plan.sink_blocks;  // only the others are cut
  const bool sink = kt < plan.sink_blocks;
  const int chunks = sink ? plan.sink_chunks : plan.near_chunks;
  const int64_t unit = (int64_t)blockIdx.y * plan.cut_units() +
                       (sink ? kt * chunks : plan.cut_sinks() + (kt - plan.sink_blocks) * chunks);
  const int b = (int)blockIdx.y / g.KV, kvh = (int)blockIdx.y % g.KV;
  const float factor = side ? 1.f : scale;
  for (int i = threadIdx.x; i < 32 * HD / 4; i += kThreads) {
    const int r = (blockIdx.x & 3) * 32 + i / (HD / 4), col = (i % (HD / 4)) * 4;
    const int key = kt * kBlockRows + r;
    if (key >= g.T) continue;
    const float* src = part + ((unit * 2 + side) * kBlockRows + r) * HD + col;
    float4 sum = rv::ld_f4(src);
#pragma unroll 8
    for (int j = 1; j < chunks; ++j) {
      const float4 v = rv::ld_f4(src + (int64_t)j * 2 * kBlockRows * HD);
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    E* dst = dqkv + ((int64_t)b * g.T + key) * (g.H + 2 * g.KV) * HD +
             (int64_t)(g.H + (side ? g.KV : 0) + kvh) * HD + col;
    store4<E>(dst, sum.x * factor, sum.y * factor, sum.z * factor, sum.w * factor);
  }
}

// Steps that a chunk has at least, and the most that the sinks' blocks are cut into (their
// partials' memory).
constexpr int kLeastSteps = 4;
constexpr double kSinkStep = 1.6;  // steps of other blocks that one of the sinks' takes as long as
constexpr int kMostUnits = 4096;

// Chunks that the other blocks are cut into: of the plans with 1, 2, 3 .. the one that takes the fewest
// steps in a row, where `slots` chunks run at once (a workgroup's start and end count
// as three steps, the partials by their bytes at 4 TB/s and a launch, a step as 2 us).
// 3 x 1999 tokens, 20 heads of 64 over 4, window 500 (492 chunks): 3 of 17 steps a block in two
// rounds 77 + 11.7 us (sums, then partials), 2 of 25 in one 67 + 10.9.
KvPlan kv_plan(const Geometry& g, int64_t batch, int64_t hd) {
  const int group = g.H / g.KV;
  const int64_t outer = batch * g.KV, slots = 256 * (hd == 32 ? 3 : hd == 64 ? 2 : 1);
  KvPlan best{};
  best.blocks = (g.T + kBlockRows - 1) / kBlockRows;
  best.sink_blocks = std::min(std::max(1, (g.sinks + kBlockRows - 1) / kBlockRows), best.blocks);
  // steps of the first block without sinks (no later one has more), and of the very first
  const int near = best.sink_blocks < best.blocks
                       ? group * query_tiles(g, best.sink_blocks * kBlockRows) : 0;
  const int most = group * query_tiles(g, 0);
  double least = 0;
  // (odd: the sinks' chunks shorter by the time that a step of theirs takes longer)
  for (int i = 2; i < 4 || (i < 130 && i / 2 <= std::max(near, most) / kLeastSteps); ++i) {
    const int chunks = i / 2;
    KvPlan p = best;
    p.near_len = near ? (near + chunks - 1) / chunks : 1;
    p.near_chunks = near ? (near + p.near_len - 1) / p.near_len : 1;
    p.sink_len = p.sink_chunks = 1;
    if (p.sink_blocks) {
      int64_t len = near ? p.near_len : (most + chunks - 1) / chunks;
      if (i & 1) len = (int64_t)(len / kSinkStep);
      len = std::max<int64_t>(len, kLeastSteps);
      len = std::max(len, (outer * p.sink_blocks * most + kMostUnits - 1) / kMostUnits);
      p.sink_len = (int)std::min<int64_t>(len, most);
      p.sink_chunks = (most + p.sink_len - 1) / p.sink_len;
    }
    const int64_t rounds = (outer * p.units() + slots - 1) / slots;
    double steps = (double)rounds * (std::max(near ? (double)p.near_len : 0.0,
                                              p.sink_blocks ? kSinkStep * p.sink_len : 0.0) + 3);
    if (p.near_chunks > 1 || p.sink_chunks > 1) {
      steps += 2 + (double)(outer * p.cut_units()) * 2 * kBlockRows * hd * 4 * 2 / 4e12 / 2e-6;
    }
    if (i == 2 || steps < least) {
      least = steps;
      best.near_len = p.near_len, best.near_chunks = p.near_chunks;
      best.sink_len = p.sink_len, best.sink_chunks = p.sink_chunks;
    }
  }
  return best;
}

// The workspace: delta, one fp32 a query and head, the largest |dO| of every 32 of them, and the
// partials, each from a multiple of four values on.
int64_t delta_values(int64_t batch, int64_t heads, int64_t seq) {
  return (batch * heads * seq + 3) / 4 * 4;
}
int64_t top_values(int64_t batch, int64_t heads, int64_t seq) {
  return (batch * heads * ((seq + 31) / 32) + 3) / 4 * 4;
}

int64_t partial_bytes(const KvPlan& p, int64_t outer, int64_t hd) {
  return outer * p.cut_units() * 2 * kBlockRows * hd * 4;
}

// Sizes the kernels take: a kTile-row tile of qkv spans less than 2 GiB, so a tile's
// buffer resource and byte offsets fit; a launch has fewer than 2^32 threads.
bool sizes_ok(int64_t batch, int64_t seq, int64_t heads, int64_t kv, int64_t hd, int dtype) {
  return (hd == 32 || hd == 64 || hd == 128) && (dtype == RV_F16 || dtype == RV_BF16) &&
         heads % kv == 0 && seq < (1 << 28) && heads < (1 << 16) && batch < (1 << 16) &&
         batch * heads * ((seq + kBlockRows - 1) / kBlockRows) < (1 << 24) &&
         batch * kv < (1 << 16) &&
         (int64_t)kTile * (heads + 2 * kv) * hd * 2 < (int64_t(1) << 31);
}

bool args_ok(int64_t batch, int64_t seq, int64_t heads, int64_t kv, int64_t hd, int64_t window,
             int64_t sinks) {
  return batch > 0 && seq > 0 && heads > 0 && kv > 0 && hd > 0 && window > 0 && sinks >= 0;
}

// Windows and sinks beyond the sequence are the sequence's length.
Geometry geometry(int64_t seq, int64_t heads, int64_t kv, int64_t window, int64_t sinks) {
  return Geometry{(int)seq, (int)heads, (int)kv, (int)std::min(window, seq),
                  (int)std::min(sinks, seq)};
}

template <typename E, int HD>
int launch_fwd(const void* qkv, int64_t batch, const Geometry& g, void* out, void* rest,
               float* lse, hipStream_t s) {
  const int n_qt = (g.T + kBlockRows - 1) / kBlockRows;
  const float c = (float)(1.4426950408889634 / std::sqrt((double)HD));
  const dim3 grid((unsigned)(n_qt * batch * g.H)), block(kThreads);
  const E* x = static_cast<const E*>(qkv);
  E *o = static_cast<E*>(out), *r = static_cast<E*>(rest);
  hipLaunchKernelGGL((wattn_fwd_k<E, HD>), grid, block, 0, s, x, o, r, lse, g, n_qt, c);
  return rv_host::check_launch();
}

template <typename E, int HD>
int launch_bwd(const void* qkv, const void* out, const void* rest, const void* dout,
               const float* lse, int64_t batch, const Geometry& g, void* dqkv, float* ws, hipStream_t s) {
  const int n_qt = (g.T + kBlockRows - 1) / kBlockRows;
  const double scale = 1.0 / std::sqrt((double)HD);
  const float c = (float)(1.4426950408889634 * scale);
  const KvPlan plan = kv_plan(g, batch, HD);
  float* delta = ws;
  float* tops = delta + delta_values(batch, g.H, g.T);
  float* part = tops + top_values(batch, g.H, g.T);
  const E* x = static_cast<const E*>(qkv);
  const E* go = static_cast<const E*>(dout);
  E* dx = static_cast<E*>(dqkv);
  // the dQ kernel writes delta and tops, which the dK/dV kernel reads
  const int64_t bh = batch * g.H;
  auto queries = [&](auto kernel, int blocks) {
    if (blocks)
      hipLaunchKernelGGL(kernel, dim3((unsigned)(blocks * bh)), dim3(kThreads), 0, s, x,
                         static_cast<const E*>(out), static_cast<const E*>(rest), go, lse, delta,
                         tops, dx, g, n_qt, c, (float)scale);
  };
  bool two = HD >= 64;
  if constexpr (HD < 128) {
    two = HD == 64 && n_qt * bh > kOneLaunch;
    if (!two) queries(wattn_bwd_q_k<E, HD, kAll>, n_qt);
  }
  if constexpr (HD >= 64) {
    if (two) {
      queries(wattn_bwd_q_k<E, HD, kFirst>, 1);
      queries(wattn_bwd_q_k<E, HD, kOthers>, n_qt - 1);
    }
  }
  int rc = rv_host::check_launch();
  if (rc != RV_OK) return rc;
  hipLaunchKernelGGL((wattn_bwd_kv_k<E, HD>), dim3((unsigned)(plan.units() * batch * g.KV)),
                     dim3(kThreads), 0, s, x, go, lse, delta, tops, dx, part, g, plan, c,
                     (float)scale);
  rc = rv_host::check_launch();
  if (rc != RV_OK) return rc;
  const int cut = (plan.sink_chunks > 1 ? plan.sink_blocks : 0) +
                  (plan.near_chunks > 1 ? plan.blocks - plan.sink_blocks : 0);
  if (cut) {
    hipLaunchKernelGGL((wattn_reduce_k<E, HD>),
                       dim3((unsigned)(8 * cut), (unsigned)(batch * g.KV)),
                       dim3(kThreads), 0, s, part, dx, g, plan, (float)scale);
    rc = rv_host::check_launch();
  }
  return rc;
}

}  // namespace

extern "C" {

int rv_window_attn_fwd(const void* qkv, int64_t batch, int64_t seq, int64_t heads,
                       int64_t kv_heads, int64_t head_dim, int dtype, int64_t window,
                       int64_t sinks, void* out, void* rest, float* lse, void* stream) {
  if (!qkv || !out || !lse) return RV_ERR_NULL_POINTER;
  if (!args_ok(batch, seq, heads, kv_heads, head_dim, window, sinks)) return RV_ERR_BAD_SIZE;
  if (!sizes_ok(batch, seq, heads, kv_heads, head_dim, dtype)) return RV_ERR_UNSUPPORTED;
  if (!rv_host::aligned16(qkv) || !rv_host::aligned16(out) || !rv_host::aligned16(rest))
    return RV_ERR_UNSUPPORTED;
  const Geometry g = geometry(seq, heads, kv_heads, window, sinks);
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == RV_F16) {
    if (head_dim == 32) return launch_fwd<_Float16, 32>(qkv, batch, g, out, rest, lse, s);
    if (head_dim == 64) return launch_fwd<_Float16, 64>(qkv, batch, g, out, rest, lse, s);
    return launch_fwd<_Float16, 128>(qkv, batch, g, out, rest, lse, s);
  }
  if (head_dim == 32) return launch_fwd<__bf16, 32>(qkv, batch, g, out, rest, lse, s);
  if (head_dim == 64) return launch_fwd<__bf16, 64>(qkv, batch, g, out, rest, lse, s);
  return launch_fwd<__bf16, 128>(qkv, batch, g, out, rest, lse, s);
}

int64_t rv_window_attn_bwd_workspace_bytes(int64_t batch, int64_t seq, int64_t heads,
                                           int64_t kv_heads, int64_t head_dim, int64_t window,
                                           int64_t sinks) {
  if (!args_ok(batch, seq, heads, kv_heads, head_dim, window, sinks)) return -RV_ERR_BAD_SIZE;
  if (!sizes_ok(batch, seq, heads, kv_heads, head_dim, RV_F16)) return -RV_ERR_UNSUPPORTED;
  const KvPlan p = kv_plan(geometry(seq, heads, kv_heads, window, sinks), batch, head_dim);
  return (delta_values(batch, heads, seq) + top_values(batch, heads, seq)) * 4 +
         partial_bytes(p, batch * kv_heads, head_dim);
}

int rv_window_attn_bwd(const void* qkv, const void* out, const void* rest, const void* dout,
                       const float* lse, int64_t batch, int64_t seq, int64_t heads, int64_t kv_heads,
                       int64_t head_dim, int dtype, int64_t window, int64_t sinks, void* dqkv,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  if (!qkv || !out || !dout || !lse || !dqkv) return RV_ERR_NULL_POINTER;
  if (!args_ok(batch, seq, heads, kv_heads, head_dim, window, sinks)) return RV_ERR_BAD_SIZE;
  if (!sizes_ok(batch, seq, heads, kv_heads, head_dim, dtype)) return RV_ERR_UNSUPPORTED;
  if (!rv_host::aligned16(qkv) || !rv_host::aligned16(out) || !rv_host::aligned16(dout) ||
      !rv_host::aligned16(dqkv) || !rv_host::aligned16(rest) || !rv_host::aligned16(workspace))
    return RV_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < rv_window_attn_bwd_workspace_bytes(
                                          batch, seq, heads, kv_heads, head_dim, window, sinks))
    return RV_ERR_WORKSPACE;
  const Geometry g = geometry(seq, heads, kv_heads, window, sinks);
  const hipStream_t s = (hipStream_t)stream;
  float* ws = static_cast<float*>(workspace);
  if (dtype == RV_F16) {
    if (head_dim == 32) return launch_bwd<_Float16, 32>(qkv, out, rest, dout, lse, batch, g, dqkv, ws, s);
    if (head_dim == 64) return launch_bwd<_Float16, 64>(qkv, out, rest, dout, lse, batch, g, dqkv, ws, s);
    return launch_bwd<_Float16, 128>(qkv, out, rest, dout, lse, batch, g, dqkv, ws, s);
  }
  if (head_dim == 32) return launch_bwd<__bf16, 32>(qkv, out, rest, dout, lse, batch, g, dqkv, ws, s);
  if (head_dim == 64) return launch_bwd<__bf16, 64>(qkv, out, rest, dout, lse, batch, g, dqkv, ws, s);
  return launch_bwd<__bf16, 128>(qkv, out, rest, dout, lse, batch, g, dqkv, ws, s);
}

}  // extern "C"
