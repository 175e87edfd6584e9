// Tiles and operands of the attention kernels on MFMA (gfx950), fp16 or bf16.
//
// MFMA operand layout (32x32x16): mfma(X, Y, acc) takes 8
// halves of row l % 32 of X and of Y at k = (l/32)*8 + 0..7 from lane l, and
// acc value j of lane l is sum_k X[(j/4)*8 + (l/32)*4 + j%4][k] Y[l%32][k].
// A product contracted over keys (or queries) takes its k order from the
// accumulator that produced P or dS: k index (l/32)*8 + i stands for tile row
// sigma = (i/4)*8 + (l/32)*4 + i%4, so a lane passes its own accumulator
// values 0..7 (and 8..15 for the next 16 rows) as the operand unchanged, and
// the other operand is read with ds_read_b64_tr_b16 from those rows.
//
// LDS tiles are [row][HD] 16-bit values with the 16-byte chunk index XOR-swizzled per
// row (swz); for HD = 32, 64, 128 both the row reads (ds_read_b128, lane ->
// row l % 32) and the transposed reads (rows sigma, 16 columns per 16 lanes)
// are free of bank conflicts for 32- and 64-bank LDS models.
#pragma once

#include "rv_device.h"

namespace rv_attn {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
#define RV_LDS __attribute__((address_space(3)))

// Vectors of an element type.
template <typename E>
struct Vec;
template <>
struct Vec<_Float16> {
  static constexpr unsigned kExponent = 0x7c00u;  // its bits
  typedef f16x8 x8;
  typedef f16x4 x4;
};
template <>
struct Vec<__bf16> {
  static constexpr unsigned kExponent = 0x7f80u;
  typedef b16x8 x8;
  typedef b16x4 x4;
};
template <typename E>
using x8 = typename Vec<E>::x8;
template <typename E>
using x4 = typename Vec<E>::x4;

constexpr int kThreads = 256;
constexpr int kWaveRows = 32;    // queries (forward, dQ) or keys (dK/dV) per wave
constexpr int kBlockRows = 128;  // per workgroup
constexpr int kTile = 64;        // rows per streamed LDS tile

template <int HD>
__device__ __forceinline__ int swz(int r, int c) {
  if constexpr (HD == 32) return c ^ (((r >> 2) & 1) | ((((r >> 1) ^ (r >> 3)) & 1) << 1));
  else if constexpr (HD == 64) return c ^ (((r >> 2) ^ ((r & 3) << 1)) & 7);
  else return c ^ ((r & 3) | (((r ^ (r >> 2)) & 1) << 2) | ((((r >> 1) ^ (r >> 3)) & 1) << 3));
}

// Half index of tile element (r, col).
template <int HD>
__device__ __forceinline__ int lds_at(int r, int col) {
  return r * HD + (swz<HD>(r, col >> 3) << 3) + (col & 7);
}

__device__ __forceinline__ f32x16 mfma(f16x8 x, f16x8 y, f32x16 acc) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(b16x8 x, b16x8 y, f32x16 acc) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, acc, 0, 0, 0);
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = 0.f;
  return z;
}

// Values 8 h .. 8 h + 7 of an accumulator as a 16-bit operand.
template <typename E = _Float16>
__device__ __forceinline__ x8<E> pack8(const f32x16& v, int h) {
  x8<E> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (E)v[8 * h + i];
  return r;
}

constexpr int kRsrcWord3 = 0x00020000;  // raw buffer resource, gfx9 data format

// Global -> registers -> LDS copy of a tile of kTile rows x HD halves.  The
// loads go through a buffer resource that starts at the tile's first row and
// ends with row `valid - 1`'s HD halves: rows at or past `valid` read as zero
// (the buffer range check), so no row needs a predicate, and a thread's byte
// offset inside a tile is the same for every tile (row stride `stride`
// halves; launch checks keep kTile rows of it below 2 GiB).
template <int HD>
struct TileCopy {
  static constexpr int kPer = kTile * HD / 8 / kThreads;
  static_assert(kPer >= 1, "tile smaller than one chunk per thread");
  u32x4 v[kPer];
  uint32_t off[kPer];
  __device__ __forceinline__ explicit TileCopy(int64_t stride) {
#pragma unroll
    for (int it = 0; it < kPer; ++it) {
      const int ch = it * kThreads + threadIdx.x;
      const int r = ch / (HD / 8), c = ch % (HD / 8);
      off[it] = (uint32_t)(((int64_t)r * stride + c * 8) * 2);
    }
  }
  template <typename P>
  __device__ __forceinline__ void load(const P* base, int64_t stride, int row0, int valid) {
    static_assert(sizeof(P) == 2, "16-bit elements");
    const int rows = min(valid - row0, kTile);
    const int bytes = rows > 0 ? (int)(((int64_t)(rows - 1) * stride + HD) * 2) : 0;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<P*>(base + (int64_t)row0 * stride), 0, bytes, kRsrcWord3);
#pragma unroll
    for (int it = 0; it < kPer; ++it)
      v[it] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)off[it], 0, 0);
  }
  template <typename E>
  __device__ __forceinline__ void store(E* t) const {
#pragma unroll
    for (int it = 0; it < kPer; ++it) {
      const int ch = it * kThreads + threadIdx.x;
      const int r = ch / (HD / 8), c = ch % (HD / 8);
      *reinterpret_cast<u32x4*>(t + r * HD + (swz<HD>(r, c) << 3)) = v[it];
    }
  }
};

// 64 fp32 per-row values (lse or delta) of a tile into LDS; rows past
// `valid` get 0.
__device__ __forceinline__ float load_rowval(const float* src, int row0, int valid) {
  const int r = row0 + (int)threadIdx.x;
  return (threadIdx.x < kTile && r < valid) ? src[r] : 0.f;
}

// Store 4 consecutive 16-bit values (8 bytes).
template <typename E = _Float16, typename P>
__device__ __forceinline__ void store4(P* dst, float a, float b, float c, float d) {
  static_assert(sizeof(P) == 2, "16-bit elements");
  x4<E> v = {(E)a, (E)b, (E)c, (E)d};
  *reinterpret_cast<x4<E>*>(dst) = v;
}

// Value of lane l ^ 32 combined with the lane's own (v_permlane32_swap: the
// two 32-lane halves exchange; both halves get the same combination, lower
// half's value first).
__device__ __forceinline__ float pair_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Row of tile element j of a 32 x 32 accumulator, relative to the lane's own
// first row (l/32)*4: (j/4)*8 + j%4.
__device__ __forceinline__ constexpr int acc_row(int j) { return (j >> 2) * 8 + (j & 3); }

// A lane's LDS offsets (halves) inside one [64][HD] tile, fixed for the whole
// kernel: row operands of rows 0..31 (rows 32..63 add 32 HD: the swizzle
// depends on the row's low five bits only) and transposed operands of the
// rows sigma of each 16-row group, upper half of each read pair included.
template <int HD, typename E = _Float16>
struct FragOffsets {
  int row[HD / 16];           // frag_row(t, lane % 32, kk, hl)
  int tr[2][HD / 32][2];      // frag_tr(t, cc * 16, dt * 32, lane): [cc][dt][first / second]
  __device__ __forceinline__ explicit FragOffsets(int lane) {
    const int hl = lane >> 5, g = lane >> 4, i = lane & 15;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
      row[kk] = (lane & 31) * HD + (swz<HD>(lane & 31, kk * 2 + hl) << 3);
#pragma unroll
    for (int cc = 0; cc < 2; ++cc)
#pragma unroll
      for (int dt = 0; dt < HD / 32; ++dt) {
        const int r = cc * 16 + (g >> 1) * 4 + (i >> 2);
        const int col = dt * 32 + (g & 1) * 16 + 4 * (i & 3);
        tr[cc][dt][0] = lds_at<HD>(r, col);
        tr[cc][dt][1] = lds_at<HD>(r + 8, col);
      }
  }
  __device__ __forceinline__ x8<E> rowf(const E* t, int sub, int kk) const {
    return *reinterpret_cast<const x8<E>*>(t + sub * 32 * HD + row[kk]);
  }
  __device__ __forceinline__ x8<E> trf(const E* t, int sub, int cc, int dt) const {
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (RV_LDS i16x4*)(t + sub * 32 * HD + tr[cc][dt][0]));
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (RV_LDS i16x4*)(t + sub * 32 * HD + tr[cc][dt][1]));
    const x4<E> a = __builtin_bit_cast(x4<E>, lo), b = __builtin_bit_cast(x4<E>, hi);
    return x8<E>{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
};

// Wave priorities inside one SIMD: a wave issues its score MFMA chains (S,
// and dP in the backward) at priority 2, the forward's P V chain at 1 and its
// softmax arithmetic at 0, so that the instruction arbiter prefers the wave
// with matrix work ready and the other waves' exponentials fill the matrix
// core's gaps (16 x 2048 tokens, 16 heads of 64: causal forward 214-219 -> 208 us,
// backward -1%; results unchanged).
__device__ __forceinline__ void prio_mfma() { __builtin_amdgcn_s_setprio(2); }
__device__ __forceinline__ void prio_mfma_tail() { __builtin_amdgcn_s_setprio(1); }
__device__ __forceinline__ void prio_valu() { __builtin_amdgcn_s_setprio(0); }

// The running max is moved only when a score exceeds it by more than kLazy
// (base-2 units): p = 2^(S c - m) then stays below 2^kLazy (exact in fp16's
// exponent range), and the rescale of o and l is skipped on most tiles.
constexpr float kLazy = 8.0f;

// LDS fragments are read ahead of the work that hides their latency: the row
// fragments of a 32-row half before its score MFMAs, the transposed ones before
// the exponentials (in the dK/dV kernel half of them: the rest would not fit
// beside two workgroups per CU).  The scheduling barriers keep them there; left
// to itself the compiler reads each pair next to its two MFMAs and waits for
// the LDS every time.  Same bits.  us of the causal kernels, before -> after: forward
// 16 x 1024 tokens, 8 heads of 128 86 -> 77, 16 x 2048, 16 heads of 64 208 -> 200, 16 x 700
// 35.6 -> 34.1; backward 224 -> 211, 630 -> 623, 114 -> 107, 2 x 2048, 8 heads of 64 91 -> 83.
// At HD = 32 the dQ kernel passes 128 registers and loses a workgroup per CU (16 x 2048, 16
// heads 403 -> 414), and the forward gains nothing (41.9 -> 43.3, 159 -> 153).
template <int HD>
constexpr bool kReadAhead = HD >= 64;

}  // namespace rv_attn
