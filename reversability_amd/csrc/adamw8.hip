// AdamW over many fp32 tensors with its moments in 8 bits, for gfx950.
//
// The update is adamw.hip's (torch.optim.AdamW, driven through GradScaler, the
// step count and the overflow flag on the device); m and v are held between steps
// as e4m3 values with one power-of-two scale per 32 consecutive elements of a
// tensor (the last block of a tensor may be short), the layout of the OCP
// microscaling formats: value = e4m3 * 2^(byte - 127).  A block's byte brings its
// largest magnitude to [2^7, 2^8), below the largest e4m3 value (448).
//
//     m  = b1 m + (1 - b1) g
//     v  = b2 v + (1 - b2) g g
//     p  = p (1 - lr wd) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The parameter takes the fp32 m and v of this step; only what the next step
// starts from is rounded.  v moves by (1 - b2) of itself a step, less than half
// a step of e4m3: to the nearest it would stand still, or climb only, so it is
// rounded up or down at random with the fractions as probabilities, which keeps its
// expectation.  m goes to the nearest value where 1 - b1 is at least 2^-4, the largest
// half step (2^-4 of it: it is replaced within 1 / (1 - b1) steps, and a zero gradient
// takes every value to a smaller one); with a slower b1 it would stand still like v, and is
// rounded at random too (303 us where the nearest takes 293, below).  The random bits are
// MurmurHash3's 32-bit finalizer (A. Appleby) of the element's index plus a key of seed,
// tensor and step: the same call gives the same bits.  A v > 0 stays > 0: a zero v under an m that is not would make the next
// update as large as 1 / eps.
//
// Memory-bound: 16.125 bytes a parameter (p 8, g 4, codes 4, scales 4 / 32; 28 with fp32
// moments) against about 85 VALU instructions.  93.2 M parameters in 6 tensors,
// operands evicted: 291 us, 5.2 TB/s (fp32 moments 498 us); 355 us with one unit of four
// elements a thread and correctly rounded divisions, 312 with one unit, 311 with four
// (the bias corrections, in fp64, and the tensor's search are paid per thread; four
// units leave fewer waves); streaming hints on the parameters 294 -> 291, left out.

#include <cmath>

#include "rv_device.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTensors = 48;
constexpr int kBlock = 32;                        // elements per scale: 8 lanes of 4
constexpr int kUnits = 2;                         // of four elements per thread
constexpr int64_t kChunk = kThreads * 4 * kUnits;  // elements per workgroup
constexpr int kGridRow = 1 << 22;                 // a launch dimension holds < 2^32 threads

struct Table {
  float* p[kMaxTensors];
  const float* g[kMaxTensors];
  uint8_t* m[kMaxTensors];
  uint8_t* ms[kMaxTensors];
  uint8_t* v[kMaxTensors];
  uint8_t* vs[kMaxTensors];
  int64_t n[kMaxTensors];
  uint32_t key[kMaxTensors];
  int chunk_start[kMaxTensors + 1];
  int count;
};

struct Hyper {
  float beta1, beta2, eps, decay, w1, w2;  // decay = 1 - lr wd, w = 1 - beta
  double lr, log2_beta1, log2_beta2;
  const float* step;       // t after this update (already advanced)
  const float* found_inf;  // nullable
  const float* inv_scale;  // nullable
  const float* clip;       // nullable
};

__device__ __forceinline__ uint32_t mix(uint32_t h) {
  h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
  h = (h ^ (h >> 13)) * 0xC2B2AE35u;
  return h ^ (h >> 16);
}

// Largest of the 8 lanes that hold a block.
__device__ __forceinline__ uint32_t block_max(uint32_t x) {
  auto take = [](uint32_t a, int b) { return a > (uint32_t)b ? a : (uint32_t)b; };
  x = take(x, __builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xf, 0xf, false));   // lane ^ 1
  x = take(x, __builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xf, 0xf, false));   // lane ^ 2
  return take(x, __builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, false));  // 7 - lane
}

// A finite value's magnitude as ordered bits; 0 for the others, which have codes of
// their own and leave their block's scale alone.
__device__ __forceinline__ uint32_t magnitude(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// The scale byte of a block whose largest magnitude has these bits.
__device__ __forceinline__ int scale_byte(uint32_t bits) {
  const int e = (int)(bits >> 23) - 7;
  return e > 0 ? e : 0;
}

__device__ __forceinline__ void decode(uint32_t codes, int scale, float (&x)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  x[0] = __builtin_ldexpf(lo[0], scale - 127);
  x[1] = __builtin_ldexpf(lo[1], scale - 127);
  x[2] = __builtin_ldexpf(hi[0], scale - 127);
  x[3] = __builtin_ldexpf(hi[1], scale - 127);
}

// e4m3 codes of x at the scale, to nearest even (NaN and infinities: NaN).
__device__ __forceinline__ uint32_t encode(const float (&x)[4], int scale) {
  float q[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    q[e] = __builtin_ldexpf(x[e], 127 - scale);
    if (fabsf(q[e]) > 448.f) q[e] = NAN;  // an infinity: finite ones are below 2^8
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
  return (uint32_t)w;
}

// e4m3 code of v >= 0 at the scale, up with probability `noise` 2^-20 against the
// fraction that is cut off.
__device__ __forceinline__ uint32_t round_random(float v, int scale, uint32_t noise) {
  const float q = __builtin_ldexpf(v, 127 - scale);
  if (!(q < 512.f)) return 0x7f;  // infinity or NaN
  // 3 of 23 mantissa bits stay; fp32's exponent 120 is e4m3's 0 (values below 2^-6,
  // in steps of 2^-9)
  const uint32_t normal = ((__float_as_uint(q) + noise) >> 20) - 960u;
  const uint32_t tiny = (uint32_t)(q * 512.f + (float)noise * 0x1p-20f);
  return q < 0x1p-6f ? tiny : normal;
}

// e4m3 codes of x at the scale, rounded at random with 16 bits an element; POSITIVE:
// x >= 0, and at least the smallest value for x > 0.
template <bool POSITIVE>
__device__ __forceinline__ uint32_t encode_random(const float (&x)[4], int scale, uint32_t first,
                                                  uint32_t key) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t bits = mix(first + e / 2 + key);  // of two elements
    const uint32_t noise = (e & 1 ? bits >> 16 : bits & 0xffffu) << 4 | 8u;
    uint32_t code = round_random(POSITIVE ? x[e] : fabsf(x[e]), scale, noise);
    if (POSITIVE) code = code == 0 && x[e] > 0.f ? 1u : code;
    else code |= __float_as_uint(x[e]) >> 31 << 7;
    w |= code << (8 * e);
  }
  return w;
}

__device__ __forceinline__ int tensor_of(const int* chunk_start, int count, int block) {
  int t = 0, above = count;
  while (above - t > 1) {
    const int mid = (t + above) >> 1;
    if (chunk_start[mid] <= block) t = mid;
    else above = mid;
  }
  return t;
}

struct Scalars {
  float step_size, inv_bc2, inv, clip;
  uint32_t key, m_key;
};

// Four elements of a thread: where they are and what was loaded.
struct Four {
  float* p;
  uint8_t *m, *v, *ms, *vs;   // codes of the four, scales of their block
  int here;                   // elements inside the tensor
  bool full;                  // all four, on vector boundaries
  float pp[4], gg[4];
  uint32_t mw, vw;
  int mscale, vscale;
};

__device__ __forceinline__ void load(Four& f, const float* g) {
#pragma unroll
  for (int e = 0; e < 4; ++e) f.pp[e] = f.gg[e] = 0.f;
  f.mw = f.vw = 0;
  f.mscale = f.vscale = 0;
  if (f.full) {
    const float4 a = rv::ld_f4(f.p), b = rv::ld_f4(g);
    f.mw = *reinterpret_cast<const uint32_t*>(f.m);
    f.vw = *reinterpret_cast<const uint32_t*>(f.v);
    f.pp[0] = a.x; f.pp[1] = a.y; f.pp[2] = a.z; f.pp[3] = a.w;
    f.gg[0] = b.x; f.gg[1] = b.y; f.gg[2] = b.z; f.gg[3] = b.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < f.here) {
        f.pp[e] = f.p[e];
        f.gg[e] = g[e];
        f.mw |= (uint32_t)f.m[e] << (8 * e);
        f.vw |= (uint32_t)f.v[e] << (8 * e);
      }
  }
  if (f.here > 0) {
    f.mscale = *f.ms;
    f.vscale = *f.vs;
  }
}

// The update and the stores; every lane of a block takes part.  `pair`: the counter
// of the first two elements' random bits.  RANDOM_M: m is rounded at random too.
template <bool RANDOM_M>
__device__ __forceinline__ void update(Four& f, const Hyper& h, const Scalars& s, uint32_t pair) {
  float m[4], v[4];
  decode(f.mw, f.mscale, m);
  decode(f.vw, f.vscale, v);
  uint32_t mtop = 0, vtop = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float u = f.gg[e] * s.inv * s.clip;  // unscale_'s multiply, then clip_grad_norm_'s
    m[e] = m[e] * h.beta1 + u * h.w1;
    v[e] = v[e] * h.beta2 + u * h.w2 * u;
    // v_rcp_f32 (1 ulp) instead of a division: the quotient is off by 2 ulps at most,
    // and is added to p after a multiplication by the learning rate
    const float denom = sqrtf(v[e]) * s.inv_bc2 + h.eps;
    f.pp[e] = f.pp[e] * h.decay - s.step_size * (m[e] * __builtin_amdgcn_rcpf(denom));
    if (e < f.here) {
      const uint32_t a = magnitude(m[e]), b = magnitude(v[e]);
      mtop = a > mtop ? a : mtop;
      vtop = b > vtop ? b : vtop;
    }
  }
  const int ms = scale_byte(block_max(mtop)), vs = scale_byte(block_max(vtop));
  const uint32_t vw = encode_random<true>(v, vs, pair, s.key);
  uint32_t mw;
  if constexpr (RANDOM_M) mw = encode_random<false>(m, ms, pair, s.m_key);
  else mw = encode(m, ms);
  if (f.full) {
    rv::st_f4(f.p, make_float4(f.pp[0], f.pp[1], f.pp[2], f.pp[3]));
    *reinterpret_cast<uint32_t*>(f.m) = mw;
    *reinterpret_cast<uint32_t*>(f.v) = vw;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < f.here) {
        f.p[e] = f.pp[e];
        f.m[e] = (uint8_t)(mw >> (8 * e));
        f.v[e] = (uint8_t)(vw >> (8 * e));
      }
  }
  if ((threadIdx.x & 7) == 0 && f.here > 0) {
    *f.ms = (uint8_t)ms;
    *f.vs = (uint8_t)vs;
  }
}

template <bool RANDOM_M>
__global__ __launch_bounds__(kThreads)
void adamw8_k(Table tab, Hyper h) {
  if (h.found_inf != nullptr && *h.found_inf != 0.0f) return;  // uniform skip
  const int64_t block = (int64_t)blockIdx.y * kGridRow + blockIdx.x;
  if (block >= tab.chunk_start[tab.count]) return;  // past the last row's end
  const int t = tensor_of(tab.chunk_start, tab.count, (int)block);
  const int64_t n = tab.n[t];
  const int64_t first = (block - tab.chunk_start[t]) * kChunk + threadIdx.x * 4;
  const bool vec = ((reinterpret_cast<uintptr_t>(tab.p[t]) | reinterpret_cast<uintptr_t>(tab.g[t])) &
                    15) == 0 &&
                   ((reinterpret_cast<uintptr_t>(tab.m[t]) | reinterpret_cast<uintptr_t>(tab.v[t])) &
                    3) == 0;
  Four f[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int64_t i = first + u * (kThreads * 4), at = i / kBlock;
    f[u].here = i >= n ? 0 : i + 4 <= n ? 4 : (int)(n - i);
    f[u].full = vec && i + 4 <= n;
    f[u].p = tab.p[t] + i;
    f[u].m = tab.m[t] + i;
    f[u].v = tab.v[t] + i;
    f[u].ms = tab.ms[t] + at;
    f[u].vs = tab.vs[t] + at;
    load(f[u], tab.g[t] + i);
  }
  __builtin_amdgcn_sched_barrier(0);
  const double step = (double)*h.step;
  Scalars s;
  s.step_size = (float)(h.lr / (1.0 - exp2(step * h.log2_beta1)));
  s.inv_bc2 = (float)(1.0 / sqrt(1.0 - exp2(step * h.log2_beta2)));
  s.inv = h.inv_scale != nullptr ? *h.inv_scale : 1.0f;
  s.clip = h.clip != nullptr ? *h.clip : 1.0f;
  s.key = mix(tab.key[t] + (uint32_t)*h.step);
  s.m_key = RANDOM_M ? mix(s.key + 0x9E3779B9u) : 0u;
#pragma unroll
  for (int u = 0; u < kUnits; ++u)
    update<RANDOM_M>(f[u], h, s, (uint32_t)((first + u * (kThreads * 4)) >> 1));
}

uint32_t host_mix(uint32_t h) {
  h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
  h = (h ^ (h >> 13)) * 0xC2B2AE35u;
  return h ^ (h >> 16);
}

}  // namespace

extern "C" {

int rv_adamw8_max_tensors(void) { return kMaxTensors; }
int rv_adamw8_block(void) { return kBlock; }

int rv_adamw8_step(int count, float* const* params, const float* const* grads,
                   uint8_t* const* exp_avg, uint8_t* const* exp_avg_scale,
                   uint8_t* const* exp_avg_sq, uint8_t* const* exp_avg_sq_scale,
                   const int64_t* numel, const uint32_t* ordinal, uint32_t seed, double lr,
                   double beta1, double beta2, double eps, double weight_decay, const float* step,
                   const float* found_inf, const float* inv_scale, const float* clip_coef,
                   void* stream) {
  if (count <= 0) return count == 0 ? RV_OK : RV_ERR_BAD_SIZE;
  if (count > kMaxTensors) return RV_ERR_UNSUPPORTED;
  if (!params || !grads || !exp_avg || !exp_avg_scale || !exp_avg_sq || !exp_avg_sq_scale ||
      !numel || !ordinal || !step)
    return RV_ERR_NULL_POINTER;
  Table tab{};
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    if (!params[i] || !grads[i] || !exp_avg[i] || !exp_avg_scale[i] || !exp_avg_sq[i] ||
        !exp_avg_sq_scale[i])
      return RV_ERR_NULL_POINTER;
    if (numel[i] <= 0) return RV_ERR_BAD_SIZE;
    tab.p[i] = params[i];
    tab.g[i] = grads[i];
    tab.m[i] = exp_avg[i];
    tab.ms[i] = exp_avg_scale[i];
    tab.v[i] = exp_avg_sq[i];
    tab.vs[i] = exp_avg_sq_scale[i];
    tab.n[i] = numel[i];
    tab.key[i] = host_mix(seed + 0x9E3779B9u * (ordinal[i] + 1u));
    tab.chunk_start[i] = (int)chunks;
    chunks += (numel[i] + kChunk - 1) / kChunk;
    if (chunks > 0x7fffffff) return RV_ERR_UNSUPPORTED;
  }
  tab.chunk_start[count] = (int)chunks;
  tab.count = count;
  Hyper h{};
  h.beta1 = (float)beta1;
  h.beta2 = (float)beta2;
  h.eps = (float)eps;
  h.decay = (float)(1.0 - lr * weight_decay);
  h.w1 = (float)(1.0 - beta1);
  h.w2 = (float)(1.0 - beta2);
  h.lr = lr;
  h.log2_beta1 = std::log2(beta1);  // beta 0: -inf, and 2^-inf = 0 = beta^t for t >= 1
  h.log2_beta2 = std::log2(beta2);
  h.step = step;
  h.found_inf = found_inf;
  h.inv_scale = inv_scale;
  h.clip = clip_coef;
  const dim3 grid((unsigned)(chunks < kGridRow ? chunks : kGridRow),
                  (unsigned)((chunks + kGridRow - 1) / kGridRow));
  if (1.0 - beta1 < 0x1p-4)
    hipLaunchKernelGGL(adamw8_k<true>, grid, dim3(kThreads), 0, (hipStream_t)stream, tab, h);
  else
    hipLaunchKernelGGL(adamw8_k<false>, grid, dim3(kThreads), 0, (hipStream_t)stream, tab, h);
  return rv_host::check_launch();
}

}  // extern "C"
