// Attention of new tokens over a paged cache of keys and values, for gfx950 on MFMA: one
// token a sequence, a chunk of a prompt, or a tree of drafted tokens.
//
//   s_ij = q_i . k_j / sqrt(hd) where i sees j, p = softmax_j s, o = p v (0 where i sees nothing)
//
// A sequence holds lengths[b] tokens, the last n = starts[b + 1] - starts[b] of them new: token i
// of the new ones is at slot context + i, context = lengths[b] - n.  It sees the slots up to its
// own or, with a tree, all of the context and the new tokens whose bits its mask has; its position
// is then context + (bits of its mask) - 1.  With a window it sees of these the tokens less
// than `window` positions before it and the first `sinks` positions.
//
// Layouts: keys and values 16-bit [pages][KV][page][HD]; q [tokens][H][HD] with a row stride;
// out [tokens][H][HD].  The rows that share a key head are the MFMA's columns: row r of a
// sequence and key head is token r / G, head kvh G + r % G, G = H / KV.
//
// Few rows (at most 32 of a sequence and key head; cached_few_k): one workgroup takes 16 NR rows
// and a stretch of keys; its four waves take the tiles of 32 keys in turn, each with a softmax of
// its own (no barrier in the loop), and are joined at the end.  Per tile a wave
// loads K straight into MFMA operands (16 keys x 32 columns, 64-byte pieces; a page holds 16 keys
// at least, so 16 keys share one table entry) and V through its own LDS tile, from which
// ds_read_b64_tr_b16 gives the transposed operand; both are loaded a tile ahead, the table
// entries of 32 tiles at once and 32 tiles ahead.
//
//   S^T [32 keys][16 rows] = K Q^T (v_mfma 16x16x32: lane l has row l % 16 and keys (l/16)*4 + 0..3 of
//   each 16), O^T [HD][16 rows] += V^T P^T, k index (l/16)*8 + i standing for key
//   (i/4)*16 + (l/16)*4 + i%4, so that a lane's own P are its operand.
//
// Rows of V that no row of the workgroup sees (behind the last token, before the window, of a
// page that does not exist) are taken as zeros and their scores as -inf, whatever the cache holds.
// A token that only some rows see reaches those alone, also where it is not a number (exact_rows).
//
// Measured (the stretches + their joining, each by itself under the profiler): 33 sequences of 100 to
// 65536 tokens, a token each, 8 key heads of 128, 306 + 6 us, 5.6 TB/s of keys and values, past a large
// copy's rate; one sequence of 200 tokens 6 us, the chain of its loads; 8 trees over 4000 tokens 24 + 7 us
// (29 the whole call in a row of them) and four chunks of up to 512 tokens over 12000, 16 heads of 128
// over 2 with a window of 4096, 76 + 18 us (84 the call): there the matrix cores are 4 and 14% busy and
// the VALU 14 and 27, the stretches being short (the rest is their start, a single tile in flight, softmax
// and partials).  Looking for values that are not finite costs 0.4 us of the single sequence's 6, 1.5 of
// the trees' 23 and 2 of the chunks (of 87 at that time).  At HD = 128 registers spill to scratch: 8 of
// cached_few_k's 256 with 17 to 32 rows, 15 of cached_many_k's for a chunk and 30 for a tree (HD = 32 and
// 64: none); exact_rows accounts for one or two of them.
//
// The weights are rounded to the type for the product with V, and nothing is made up for: errors against
// 64 bits are 1.1 to 1.4 times those of the output's own rounding (fp16 2.4e-4 to 2.9e-4, 2.1e-4; bf16
// 2.1e-3 to 2.3e-3, 1.7e-3).

#include <algorithm>
#include <climits>
#include <cmath>

#include "attn_tile.h"

namespace {

using namespace rv_attn;

constexpr int kKeys = 32;  // keys per tile of a wave (few rows)
constexpr int kWaves = 4;

__device__ __forceinline__ f32x4 mfma16(f16x8 x, f16x8 y, f32x4 acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(b16x8 x, b16x8 y, f32x4 acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, acc, 0, 0, 0);
}

struct Cached {
  const void* q;
  const void* keys;
  const void* values;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* starts;
  const int64_t* tree;  // null: a chunk
  void* out;
  float* part;  // [tokens][H][splits][HD] sums, then [tokens][H][splits][2] their m and l
  int64_t q_ld, table_ld, table_pages;
  int tokens, seqs, H, KV, pages, page_shift, max_query;
  int window, sinks;  // window 0: none
  int row_blocks, splits, split_tiles;
  float c;
};

// What a block of rows of a sequence sees: slots [lo, hi) and those below `sinks`, as tiles
// [0, sink_tiles) and [first, first + count - sink_tiles).
struct View {
  int start, n, context;
  int i0, i1;  // its tokens, both included
  int lo, hi;
  int sink_tiles, first, count;

  __device__ __forceinline__ View(const Cached& a, int b, int rb, int rows, int keys) {
    const int group = a.H / a.KV;
    start = min(max(a.starts[b], 0), a.tokens);
    const int end = min(max(a.starts[b + 1], start), a.tokens);
    // The new tokens are where the plan puts them, also where the pages hold only some of them: what is
    // cut to the pages is what can be read.  (A sequence whose pages do not even hold its first new
    // token is cut as a whole: none of its new tokens was stored.)
    const int held = (int)min(a.table_pages << a.page_shift, (int64_t)1 << 30);
    int len = max(a.lengths[b], 0);
    if (len - (end - start) >= held) len = held;
    context = len - (end - start);
    n = min(end - start, a.max_query);
    i0 = rb * rows / group;
    i1 = min(n - 1, (rb * rows + rows - 1) / group);
    hi = min(min(len, held), a.tree ? context + n : context + i1 + 1);
    lo = 0;
    if (a.window) lo = max(0, (a.tree ? context : context + i0 + 1) - a.window);
    count = sink_tiles = first = 0;
    if (i0 < n && hi > 0) {
      const int all = (hi + keys - 1) / keys;
      first = min(lo / keys, all);
      sink_tiles = min((a.sinks + keys - 1) / keys, first);
      count = sink_tiles + all - first;
    }
  }
  __device__ __forceinline__ int tile(int v) const {
    return v < sink_tiles ? v : first + v - sink_tiles;
  }
};

constexpr int kXcds = 8;

// A workgroup's stretch, block of rows, key head and sequence.  Workgroups are dealt to the eight XCDs in
// turn, each with an L2 of its own: the blocks of rows that read the same keys go to one of them
// (four chunks of up to 512 tokens over 12000 96 -> 89 us).  The stretches are numbered slowest: those behind the
// shorter sequences' ends come last, and leave at once.
struct Place {
  int split, rb, kvh, b;
  __device__ __forceinline__ explicit Place(const Cached& a) {
    const int turn = (int)blockIdx.x / kXcds, eight = turn / a.row_blocks;
    // (turned by 5 each time: one sequence's stretches, eight groups apart, meet all XCDs)
    const int group = eight * kXcds + (((int)blockIdx.x + 5 * eight) & (kXcds - 1));
    rb = turn % a.row_blocks;
    kvh = group % a.KV;
    b = group / a.KV % a.seqs;
    split = group / a.KV / a.seqs;  // (>= splits: one of the last few, without work)
  }
};

// Value of the lane's row over the four lanes that hold it (l % 16).
__device__ __forceinline__ float row_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return pair_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float row_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return pair_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// The position of the token at slot `key`: a drafted one's goes by its mask.
__device__ __forceinline__ int position_of(const Cached& a, const View& w, int key) {
  if (key < w.context || key - w.context >= w.n) return key;
  const uint64_t bits = w.n < 64 ? (uint64_t(1) << w.n) - 1 : ~uint64_t(0);
  return w.context + __popcll((uint64_t)a.tree[w.start + key - w.context] & bits) - 1;
}

// Whether a row sees the slot `key` as far as order goes: up to its own (limit), or the context and what
// its mask has.  Without branches: it is asked for every element of a tile at an edge.
__device__ __forceinline__ bool in_order(bool tree, int context, int key, int limit,
                                         uint64_t mask) {
  if (!tree) return key <= limit;
  return (key < context) | ((mask >> ((key - context) & 63) & 1) != 0);
}

// Half index of element (r, col) of a V tile [32][HD]: pairs of 16-byte chunks XOR-swizzled so that
// eight rows' 32 bytes of one column block lie on different banks.
template <int HD>
__device__ __forceinline__ int v_at(int r, int col) {
  const int turn = (r / (128 / HD)) & (HD / 16 - 1);
  return r * HD + ((((col >> 4) ^ turn) << 4) | (col & 15));
}

// The page of the 16 keys from `key` on, -1 where there is none or none of them is needed.
__device__ __forceinline__ int page_of(const Cached& a, const View& w, int b, int key) {
  if (key >= w.hi) return -1;
  const int page = a.table[b * a.table_ld + (key >> a.page_shift)];
  return page >= 0 && page < a.pages ? page : -1;
}

// Values that are not numbers, or infinite, in V of keys that some rows see and others do not: 0 times
// them is NaN, and would reach rows that do not see them.  They are looked for in the tiles at an edge
// alone, where masks are; a workgroup that meets one makes its rows again key by key (exact_rows).
template <typename E>
__device__ __forceinline__ bool finite(const x8<E>& v) {
  constexpr unsigned kExp = Vec<E>::kExponent;
  const u32x4 w = __builtin_bit_cast(u32x4, v);
  bool yes = true;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    yes = yes & ((w[i] & kExp) != kExp) & ((w[i] & (kExp << 16)) != (kExp << 16));
  return yes;
}

// Where K and V of the token at slot `key` lie in the caches, -1 where there is none.
template <int HD>
__device__ __forceinline__ int64_t row_of(const Cached& a, const View& w, int b, int kvh, int key) {
  const int page = page_of(a, w, b, key);
  return page < 0 ? -1
                  : ((((int64_t)page * a.KV + kvh) << a.page_shift) +
                     (key & ((1 << a.page_shift) - 1))) * HD;
}

// The rows of a workgroup over its stretch [v0, v_end) of tiles of `keys` keys, one row a wave at a time:
// lanes are keys for the scores, columns for the sums.  Slow, and seldom called.
template <typename E, int HD>
__device__ __forceinline__ void exact_rows(const Cached& a, const View& w, int b,
                                                     int kvh, int row0, int rows, int split,
                                                     int v0, int v_end, int keys) {
  const int lane = threadIdx.x & 63, group = a.H / a.KV;
  const uint64_t bits = w.n < 64 ? (uint64_t(1) << w.n) - 1 : ~uint64_t(0);
  const int reach = a.window ? a.window : INT_MAX;
  for (int row = row0 + (int)(threadIdx.x >> 6); row < row0 + rows; row += kWaves) {
    const int token = row / group, head = kvh * group + row % group;
    if (token >= w.n) return;
    const uint64_t mask = a.tree ? (uint64_t)a.tree[w.start + token] & bits : 0;
    const int limit = w.context + token;
    const int place = a.tree ? w.context + __popcll(mask) - 1 : limit;
    const E* q = static_cast<const E*>(a.q) + (int64_t)(w.start + token) * a.q_ld + head * HD;
    float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
    for (int v = v0; v < v_end; ++v) {
      const int k0 = w.tile(v) * keys, key = k0 + lane;
      int64_t at = -1;
      if (lane < keys && key < w.hi && in_order(a.tree != nullptr, w.context, key, limit, mask)) {
        const int kp = a.tree && a.window ? position_of(a, w, key) : key;
        if (place - kp < reach || kp < a.sinks) at = row_of<HD>(a, w, b, kvh, key);
      }
      uint64_t seen = __ballot(at >= 0);
      if (!seen) continue;
      float s = 0.f;
      for (int i = 0; i < HD; i += 8) {
        const x8<E> x = *reinterpret_cast<const x8<E>*>(q + i);
        const x8<E> y = *reinterpret_cast<const x8<E>*>(static_cast<const E*>(a.keys) +
                                                        (at < 0 ? 0 : at) + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf((float)x[e], (float)y[e], s);
      }
      s = at < 0 ? -INFINITY : s * a.c;
      float top = s;
#pragma unroll
      for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
      const float m_new = fmaxf(m, top), base = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(m - base);
      const float p = __builtin_amdgcn_exp2f(s - base);
      m = m_new;
      l = l * alpha + rv::wave_sum(p);
      o[0] *= alpha, o[1] *= alpha;
      while (seen) {
        const int k = __builtin_ctzll(seen);
        seen &= seen - 1;
        const float pk = (float)(E)__shfl(p, k);
        const E* vr = static_cast<const E*>(a.values) + __shfl(at, k);
        o[0] += pk * (float)vr[lane % HD];
        if (HD == 128) o[1] += pk * (float)vr[64 + lane];
      }
    }
    const int64_t to = (int64_t)(w.start + token) * a.H + head;
    if (a.splits == 1 || w.count <= a.split_tiles) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      E* dst = static_cast<E*>(a.out) + to * HD;
      if (lane < HD) dst[lane] = (E)(o[0] * inv);
      if (HD == 128) dst[64 + lane] = (E)(o[1] * inv);
    } else {
      float* dst = a.part + (to * a.splits + split) * HD;
      if (lane < HD) dst[lane] = o[0];
      if (HD == 128) dst[64 + lane] = o[1];
      float* stat = a.part + (int64_t)a.tokens * a.H * a.splits * HD + (to * a.splits + split) * 2;
      if (lane == 0) stat[0] = m, stat[1] = l;
    }
  }
}

// K operands and V rows of one tile on their way through registers.
template <typename E, int HD>
struct Tile {
  static constexpr int KK = HD / 32, VC = HD / 16;
  x8<E> k[2][KK];
  x8<E> v[VC];
  bool whole;  // both groups' pages exist and all rows lie in [lo, hi)

  // ids: entry_of's of the block of tiles, this tile the it-th of them.
  __device__ __forceinline__ void load(const Cached& a, const View& w, int kvh, int ids, int it,
                                       int k0, int lane) {
    const E* keys = static_cast<const E*>(a.keys);
    const E* values = static_cast<const E*>(a.values);
    int64_t at[2];
    bool ok[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int key = k0 + 16 * g;
      const int page = __builtin_amdgcn_readlane(ids, 2 * it + g);
      ok[g] = page >= 0;
      at[g] = ((((int64_t)(ok[g] ? page : 0) * a.KV + kvh) << a.page_shift) +
               (key & ((1 << a.page_shift) - 1))) * HD;
    }
    whole = ok[0] && ok[1] && k0 + kKeys <= w.hi && (k0 >= w.lo || k0 + kKeys <= a.sinks);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const E* row = keys + at[g] + (lane & 15) * HD + (lane >> 4) * 8;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) k[g][kk] = *reinterpret_cast<const x8<E>*>(row + kk * 32);
    }
#pragma unroll
    for (int it = 0; it < VC; ++it) {
      const int ch = it * 64 + lane, r = ch / (HD / 8), col = (ch % (HD / 8)) * 8;
      const int g = it / (VC / 2);  // the rows of one load lie in one group
      v[it] = *reinterpret_cast<const x8<E>*>(values + at[g] + (r & 15) * HD + col);
    }
    if (!whole) {
      seen[0] = ok[0], seen[1] = ok[1];
#pragma unroll
      for (int it = 0; it < VC; ++it) {
        const int r = (it * 64 + lane) / (HD / 8), key = k0 + r;
        if (!ok[it / (VC / 2)] || key >= w.hi || (key < w.lo && key >= a.sinks)) v[it] = x8<E>{};
      }
    }
  }
  bool seen[2];
  __device__ __forceinline__ bool odd() const {  // of the wave: some V is not finite
    bool yes = true;
#pragma unroll
    for (int it = 0; it < VC; ++it) yes = yes & finite<E>(v[it]);
    return __any(!yes);
  }
  __device__ __forceinline__ void store_v(E* t, int lane) const {
#pragma unroll
    for (int it = 0; it < VC; ++it) {
      const int ch = it * 64 + lane, r = ch / (HD / 8), col = (ch % (HD / 8)) * 8;
      *reinterpret_cast<x8<E>*>(t + v_at<HD>(r, col)) = v[it];
    }
  }
};

template <typename E, int HD, int NR>
__global__ __launch_bounds__(kThreads, 2)
void cached_few_k(Cached a) {
  constexpr int KK = HD / 32, DT = HD / 16, R = 16 * NR;
  constexpr int kVBytes = kWaves * kKeys * HD * 2, kOBytes = 2 * R * HD * 4;
  __shared__ __attribute__((aligned(16))) char lds[kVBytes > kOBytes ? kVBytes : kOBytes];
  __shared__ float ml[2][kWaves][R];
  __shared__ int odds[kWaves];
  const Place at(a);
  if (at.split >= a.splits) return;
  const int split = at.split, rb = at.rb, kvh = at.kvh, b = at.b;
  const int lane = threadIdx.x & 63, hl = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const View w(a, b, rb, R, kKeys);
  if (w.i0 >= w.n) return;  // no such rows
  // (the last stretch takes what is left of a sequence that is longer than was said)
  const int v_end = split + 1 == a.splits ? w.count : min(w.count, (split + 1) * a.split_tiles);
  if (split && split * a.split_tiles >= w.count) return;  // (the first writes zeros if need be)
  const int group = a.H / a.KV;

  // the lane's rows: token and head, last slot seen (chunk) or mask (tree), position
  x8<E> qf[NR][KK];
  int token[NR], limit[NR], place[NR];
  uint64_t mask[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int row = rb * R + r * 16 + (lane & 15);
    token[r] = row / group;
    const bool ok = token[r] < w.n;
    const int head = kvh * group + row % group;
    limit[r] = ok ? w.context + token[r] : -1;
    place[r] = limit[r];
    mask[r] = 0;
    if (a.tree && ok) {
      const uint64_t bits = w.n < 64 ? (uint64_t(1) << w.n) - 1 : ~uint64_t(0);
      mask[r] = (uint64_t)a.tree[w.start + token[r]] & bits;
      place[r] = w.context + __popcll(mask[r]) - 1;
    }
    const E* src = static_cast<const E*>(a.q) + (int64_t)(w.start + token[r]) * a.q_ld +
                   (int64_t)head * HD + hl * 8;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
      qf[r][kk] = ok ? *reinterpret_cast<const x8<E>*>(src + kk * 32) : x8<E>{};
  }
  f32x4 o[DT][NR];
  float m[NR], l[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt][r] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int reach = a.window ? a.window : INT_MAX;
  // slots below `below` are seen by every row as far as order goes, from `from` on as far as the
  // window goes
  const int below = a.tree ? w.context : w.context + w.i0 + 1;
  const int last = a.tree ? w.context + w.n - 1 : w.context + w.i1;
  const int from = a.window ? last - a.window + 1 : 0;

  auto sees = [&](int key, int r) {
    const int kp = a.tree && a.window ? position_of(a, w, key) : key;
    return (key < w.hi) & in_order(a.tree != nullptr, w.context, key, limit[r], mask[r]) &
           ((place[r] - kp < reach) | (kp < a.sinks));
  };

  E* vt = reinterpret_cast<E*>(lds) + wave * kKeys * HD;
  const int i = lane & 15;
  Tile<E, HD> next;
  int v = split * a.split_tiles + wave;
  // table entries of the wave's next 32 tiles, two a tile, in the lanes
  auto entries = [&](int from_tile) {
    const int x = from_tile + (lane >> 1) * kWaves;
    return x < v_end ? page_of(a, w, b, w.tile(x) * kKeys + 16 * (lane & 1)) : -1;
  };
  int ids = entries(v), ids_next = entries(v + 32 * kWaves), it = 0, odd = 0;
  if (v < v_end) next.load(a, w, kvh, ids, 0, w.tile(v) * kKeys, lane);
  for (; v < v_end; v += kWaves) {
    const int k0 = w.tile(v) * kKeys;
    const Tile<E, HD> now = next;
    const bool plain = now.whole && k0 + kKeys <= below && (k0 >= from || k0 + kKeys <= a.sinks);
    if (!plain && now.odd()) odd = 1;
    if (++it == 32) {
      it = 0;
      ids = ids_next;
      ids_next = entries(v + 33 * kWaves);
    }
    // the wave's last reads of the tile come before these writes, the reads below behind
    // them: one wave's LDS accesses keep their order, the fences keep the compiler's
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    now.store_v(vt, lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (v + kWaves < v_end) next.load(a, w, kvh, ids, it, w.tile(v + kWaves) * kKeys, lane);

    f32x4 s[2][NR];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        s[g][r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) s[g][r] = mfma16(now.k[g][kk], qf[r][kk], s[g][r]);
      }
    if (!plain) {
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = k0 + g * 16 + hl * 4 + j;
          const bool there = now.seen[g] | now.whole;
#pragma unroll
          for (int r = 0; r < NR; ++r)
            s[g][r][j] = there & sees(key, r) ? s[g][r][j] : -INFINITY;
        }
    }
    bool up = false;
    float mx[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const f32x4 x = s[0][r], y = s[1][r];
      mx[r] = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                    fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]))) * a.c;
      up = up || mx[r] > m[r] + kLazy;
    }
    if (__any(up)) {
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float m_new = fmaxf(m[r], row_max(mx[r]));
        const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - m_new);
        m[r] = m_new;
        l[r] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt][r] *= alpha;
      }
    }
    x8<E> pf[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float neg_m = m[r] == -INFINITY ? 0.f : -m[r];
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][r][e & 3], a.c, neg_m));
        sum += p;
        pf[r][e] = (E)p;
      }
      l[r] += sum;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (RV_LDS i16x4*)(vt + v_at<HD>(hl * 4 + (i >> 2), dt * 16 + 4 * (i & 3))));
      const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (RV_LDS i16x4*)(vt + v_at<HD>(16 + hl * 4 + (i >> 2), dt * 16 + 4 * (i & 3))));
      const x4<E> p = __builtin_bit_cast(x4<E>, x), q = __builtin_bit_cast(x4<E>, y);
      const x8<E> vf = {p[0], p[1], p[2], p[3], q[0], q[1], q[2], q[3]};
#pragma unroll
      for (int r = 0; r < NR; ++r) o[dt][r] = mfma16(vf, pf[r], o[dt][r]);
    }
  }

  // the four waves' sums in one: scaled to the common maximum, then added in pairs
  float all_m[NR], all_l[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    l[r] = row_sum(l[r]);
    if (hl == 0) {
      ml[0][wave][r * 16 + i] = m[r];
      ml[1][wave][r * 16 + i] = l[r];
    }
  }
  if (lane == 0) odds[wave] = odd;
  __syncthreads();  // (also: every wave is done with its V tile)
  if (odds[0] | odds[1] | odds[2] | odds[3]) {
    exact_rows<E, HD>(a, w, b, kvh, rb * R, R, split, split * a.split_tiles, v_end, kKeys);
    return;
  }
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    all_m[r] = -INFINITY;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) all_m[r] = fmaxf(all_m[r], ml[0][x][r * 16 + i]);
    const float top = all_m[r] == -INFINITY ? 0.f : all_m[r];
    all_l[r] = 0.f;
#pragma unroll
    for (int x = 0; x < kWaves; ++x)
      all_l[r] += ml[1][x][r * 16 + i] * __builtin_amdgcn_exp2f(ml[0][x][r * 16 + i] - top);
    const float factor = __builtin_amdgcn_exp2f(m[r] - top);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt][r] *= factor;
  }
  f32x4* swap = reinterpret_cast<f32x4*>(lds);
#pragma unroll
  for (int step = 2; step; step >>= 1) {
    if (wave >= step && wave < 2 * step) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < NR; ++r)
          swap[(((wave - step) * DT + dt) * NR + r) * 64 + lane] = o[dt][r];
    }
    __syncthreads();
    if (wave < step) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < NR; ++r) o[dt][r] += swap[((wave * DT + dt) * NR + r) * 64 + lane];
    }
    __syncthreads();
  }
  if (wave) return;
  const bool alone = a.splits == 1 || w.count <= a.split_tiles;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if (token[r] >= w.n) continue;
    const int row = rb * R + r * 16 + i;
    const int64_t at = (int64_t)(w.start + token[r]) * a.H + kvh * group + row % group;
    if (alone) {
      const float inv = all_l[r] == 0.f ? 0.f : 1.f / all_l[r];
      E* dst = static_cast<E*>(a.out) + at * HD + hl * 4;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        store4<E>(dst + dt * 16, o[dt][r][0] * inv, o[dt][r][1] * inv, o[dt][r][2] * inv,
                  o[dt][r][3] * inv);
    } else {
      float* dst = a.part + (at * a.splits + split) * HD + hl * 4;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(dst + dt * 16) = o[dt][r];
      if (hl == 0) {
        float* stat = a.part + (int64_t)a.tokens * a.H * a.splits * HD + (at * a.splits + split) * 2;
        stat[0] = all_m[r];
        stat[1] = all_l[r];
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows.
// ---------------------------------------------------------------------------
// A tile of 64 keys of K and V on its way into LDS.  The rows of one wave's load lie in one group of 16:
// their page's offset is the wave's, the rest of the address the thread's for good.
template <typename E, int HD>
struct PagedCopy {
  static constexpr int kPer = kTile * HD / 8 / kThreads;
  u32x4 k[kPer], v[kPer];

  static __device__ __forceinline__ int row(int i) { return (i * kThreads + threadIdx.x) / (HD / 8); }
  static __device__ __forceinline__ int chunk() { return threadIdx.x % (HD / 8); }

  // ids: the pages of the tile's four groups of 16 keys in lanes 4 * it .. 4 * it + 3.
  __device__ __forceinline__ void load(const E* keys, const E* values, const Cached& a, int kvh,
                                       int ids, int it, int k0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int g = __builtin_amdgcn_readfirstlane(row(i) >> 4);
      const int page = __builtin_amdgcn_readlane(ids, 4 * it + g);
      const int64_t at = ((((int64_t)max(page, 0) * a.KV + kvh) << a.page_shift) +
                          ((k0 + 16 * g) & ((1 << a.page_shift) - 1))) * HD;
      const unsigned own = (row(i) & 15) * HD + chunk() * 8;
      k[i] = *reinterpret_cast<const u32x4*>(keys + at + own);
      v[i] = *reinterpret_cast<const u32x4*>(values + at + own);
    }
  }
  // missing: the groups without a page; rows of V that no row of the workgroup sees become zeros.
  // Returns whether at an edge some V that the thread holds is not finite.
  __device__ __forceinline__ bool store(E* ks, E* vs, const Cached& a, const View& w, int k0,
                                        unsigned missing, bool edge) {
    if (missing || k0 + kTile > w.hi || (k0 < w.lo && k0 + kTile > a.sinks)) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int key = k0 + row(i);
        if ((missing >> (row(i) >> 4) & 1u) || key >= w.hi || (key < w.lo && key >= a.sinks))
          v[i] = u32x4{0, 0, 0, 0};
      }
    }
    bool odd = false;
    if (edge) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) odd = odd | !finite<E>(__builtin_bit_cast(x8<E>, v[i]));
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = row(i), to = r * HD + (swz<HD>(r, chunk()) << 3);
      *reinterpret_cast<u32x4*>(ks + to) = k[i];
      *reinterpret_cast<u32x4*>(vs + to) = v[i];
    }
    return odd;
  }
};

template <int HD>
struct State {
  f32x16 o[HD / 32];
  float m, l;
};

// Halves of V's operands that are read ahead of the exponentials: at HD = 128 both do not fit beside
// two workgroups per CU.
template <int HD>
constexpr int kAhead = HD == 64 ? 2 : 0;

// 32 keys of a staged tile for one wave's 32 rows (lanes); sees(key) where MASK.
template <typename E, int HD, bool MASK, typename Sees>
__device__ __forceinline__ void many_rows(State<HD>& st, const E* Ks, const E* Vs,
                                          const FragOffsets<HD, E>& fo,
                                          const x8<E> (&qf)[HD / 16], int sub, float c,
                                          const Sees& sees) {
  constexpr int KK = HD / 16, DT = HD / 32;
  prio_mfma();
  constexpr int KH = HD == 128 ? KK / 2 : KK;
  f32x16 s = zero16();
#pragma unroll
  for (int k0 = 0; k0 < KK; k0 += KH) {
    x8<E> kf[KH];
#pragma unroll
    for (int kk = 0; kk < KH; ++kk) kf[kk] = fo.rowf(Ks, sub, k0 + kk);
    if constexpr (HD == 64) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kk = 0; kk < KH; ++kk) s = mfma(kf[kk], qf[k0 + kk], s);
  }
  prio_valu();
  float mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    if constexpr (MASK) {
      s[j] = sees(acc_row(j)) ? s[j] : -INFINITY;
    }
    mx = fmaxf(mx, s[j]);
  }
  const float mxc = pair_max(mx) * c;
  if (__any(mxc > st.m + kLazy)) {
    const float m_new = fmaxf(st.m, mxc);
    const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(st.m - m_new);
    st.m = m_new;
    st.l *= alpha;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) st.o[dt][e] *= alpha;
  }
  const float neg_m = st.m == -INFINITY ? 0.f : -st.m;
  x8<E> vf[2][DT];
  if constexpr (kReadAhead<HD>) {
#pragma unroll
    for (int cc = 0; cc < kAhead<HD>; ++cc)
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
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      if (cc >= kAhead<HD>) vf[cc][dt] = fo.trf(Vs, sub, cc, dt);
      st.o[dt] = mfma(vf[cc][dt], pf, st.o[dt]);
    }
  }
}

template <typename E, int HD, bool TREE>
__global__ __launch_bounds__(kThreads, 2)
void cached_many_k(Cached a) {
  constexpr int KK = HD / 16, DT = HD / 32, kBlock = 16;  // kBlock: tiles of one load of entries
  __shared__ __attribute__((aligned(16))) E lds[2][2][kTile * HD];
  __shared__ int odds[kWaves];
  const Place at(a);
  if (at.split >= a.splits) return;
  const View w(a, at.b, at.rb, kBlockRows, kTile);
  if (w.i0 >= w.n) return;
  const int v0 = at.split * a.split_tiles;
  const int v_end = at.split + 1 == a.splits ? w.count : min(w.count, v0 + a.split_tiles);
  if (at.split && v0 >= w.count) return;
  const int lane = threadIdx.x & 63, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = a.H / a.KV;

  // the lane's row; the wave's tokens [t0, t1]
  const int row0 = at.rb * kBlockRows + wave * kWaveRows, row = row0 + (lane & 31);
  const int t0 = row0 / group, t1 = min(w.n - 1, (row0 + kWaveRows - 1) / group);
  const int token = row / group, head = at.kvh * group + row % group;
  const bool ok = token < w.n, busy = t0 < w.n;
  const uint64_t bits = w.n < 64 ? (uint64_t(1) << w.n) - 1 : ~uint64_t(0);
  const int limit = ok ? w.context + token : -1;
  int place = limit;
  uint64_t mask = 0;
  if (TREE && ok) {
    mask = (uint64_t)a.tree[w.start + token] & bits;
    place = w.context + __popcll(mask) - 1;
  }
  x8<E> qf[KK];
  const E* src = static_cast<const E*>(a.q) + (int64_t)(w.start + token) * a.q_ld +
                 (int64_t)head * HD + hl * 8;
#pragma unroll
  for (int kk = 0; kk < KK; ++kk)
    qf[kk] = ok ? *reinterpret_cast<const x8<E>*>(src + kk * 16) : x8<E>{};
  State<HD> st;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) st.o[dt] = zero16();
  st.m = -INFINITY;
  st.l = 0.f;
  // for the wave: slots below `below` are seen by every row as far as order goes, from `from`
  // on as far as the window goes; slots from `end` on, and between the sinks and `begin`, by none
  const int below = TREE ? w.context : w.context + t0 + 1;
  const int from = a.window ? (TREE ? w.context + w.n - 1 : w.context + t1) - a.window + 1 : 0;
  const int end = TREE ? w.hi : min(w.hi, w.context + t1 + 1);
  const int begin = a.window && !TREE ? w.context + t0 - a.window + 1 : w.lo;

  const E* kc = static_cast<const E*>(a.keys);
  const E* vc = static_cast<const E*>(a.values);
  PagedCopy<E, HD> copy;
  auto entries = [&](int tile) {
    const int x = tile + (lane >> 2);
    return x < v_end ? page_of(a, w, at.b, w.tile(x) * kTile + 16 * (lane & 3)) : -1;
  };
  const FragOffsets<HD, E> fo(lane);
  int ids = entries(v0), ids_next = entries(v0 + kBlock), it = 0;
  unsigned missing = 0;  // tiles' groups without a page: of the staged tile, then of the next
  auto load = [&](int k0) {
    missing = (unsigned)(__ballot(ids < 0) >> (4 * it)) & 15u;
    copy.load(kc, vc, a, at.kvh, ids, it, k0);
  };
  // whether some row of the workgroup does not see some key of a tile, though another may
  const int all_below = TREE ? w.context : w.context + w.i0 + 1;
  const int all_from =
      a.window ? (TREE ? w.context + w.n - 1 : w.context + w.i1) - a.window + 1 : 0;
  auto edge = [&](int k0) {
    return k0 + kTile > all_below || (k0 < all_from && k0 + kTile > a.sinks);
  };
  int odd = 0;
  auto store = [&](int buf, int k0) {
    if (__any(copy.store(lds[buf][0], lds[buf][1], a, w, k0, missing, edge(k0)))) odd = 1;
  };
  if (v0 < v_end) {
    load(w.tile(v0) * kTile);
    store(0, w.tile(v0) * kTile);
  }
  unsigned now = missing;
  __syncthreads();
#define RV_MANY_STEP(BUF)                                                                       \
  {                                                                                             \
    const int k0 = w.tile(v) * kTile;                                                           \
    const bool more = v + 1 < v_end;                                                            \
    if (more) {                                                                                 \
      if (++it == kBlock) {                                                                     \
        it = 0;                                                                                 \
        ids = ids_next;                                                                         \
        ids_next = entries(v + 1 + kBlock);                                                     \
      }                                                                                         \
      load(w.tile(v + 1) * kTile);                                                             \
    }                                                                                          \
    _Pragma("unroll") for (int sub = 0; sub < 2; ++sub) {                                       \
      const int ks = k0 + sub * 32;                                                             \
      if (!busy || ks >= end || (ks + 32 <= begin && ks >= a.sinks)) continue;                  \
      if (ks + 32 <= below && (ks >= from || ks + 32 <= a.sinks) && !(now >> (2 * sub) & 3u)) { \
        many_rows<E, HD, false>(st, lds[BUF][0], lds[BUF][1], fo, qf, sub, a.c,                \
                                [](int) { return true; });                                     \
      } else {                                                                                 \
        const unsigned lost = now >> (2 * sub);                                                \
        many_rows<E, HD, true>(st, lds[BUF][0], lds[BUF][1], fo, qf, sub, a.c, [&](int r) {    \
          return ((lost >> (r >> 4) & 1u) == 0) & sees(ks + r + hl * 4);                       \
        });                                                                                    \
      }                                                                                        \
    }                                                                                          \
    now = missing;                                                                              \
    if (more) store(1 - (BUF), w.tile(v + 1) * kTile);                                         \
    __syncthreads();                                                                            \
  }
  const int reach = a.window ? a.window : INT_MAX;
  auto sees = [&](int key) {
    const int kp = TREE && a.window ? position_of(a, w, key) : key;
    return (key < w.hi) & in_order(TREE, w.context, key, limit, mask) &
           ((place - kp < reach) | (kp < a.sinks));
  };
  for (int v = v0; v < v_end; ++v) {
    RV_MANY_STEP(0)
    if (++v >= v_end) break;
    RV_MANY_STEP(1)
  }
#undef RV_MANY_STEP
  if (lane == 0) odds[wave] = odd;
  __syncthreads();
  if (odds[0] | odds[1] | odds[2] | odds[3]) {
    exact_rows<E, HD>(a, w, at.b, at.kvh, at.rb * kBlockRows, kBlockRows, at.split, v0, v_end,
                      kTile);
    return;
  }
  const float l = pair_sum(st.l);
  if (!ok) return;
  const int64_t to = (int64_t)(w.start + token) * a.H + head;
  if (a.splits == 1 || w.count <= a.split_tiles) {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    E* dst = static_cast<E*>(a.out) + to * HD + hl * 4;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int jg = 0; jg < 4; ++jg)
        store4<E>(dst + dt * 32 + jg * 8, st.o[dt][4 * jg] * inv, st.o[dt][4 * jg + 1] * inv,
                  st.o[dt][4 * jg + 2] * inv, st.o[dt][4 * jg + 3] * inv);
    return;
  }
  float* dst = a.part + (to * a.splits + at.split) * HD + hl * 4;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int jg = 0; jg < 4; ++jg)
      rv::st_f4(dst + dt * 32 + jg * 8, make_float4(st.o[dt][4 * jg], st.o[dt][4 * jg + 1],
                                                    st.o[dt][4 * jg + 2], st.o[dt][4 * jg + 3]));
  if (hl == 0) {
    float* stat = a.part + (int64_t)a.tokens * a.H * a.splits * HD + (to * a.splits + at.split) * 2;
    stat[0] = st.m;
    stat[1] = l;
  }
}

// ---------------------------------------------------------------------------
// Joins the stretches of the rows that were cut: WAVES waves a row of HD columns, rows of one
// sequence numbered token by token.  HD / 4 threads take four columns each of a stretch, the
// others the next ones; their sums are added in order.
// ---------------------------------------------------------------------------
template <typename E, int HD, int WAVES>
__global__ __launch_bounds__(kThreads)
void cached_join_k(Cached a, int rows_per_block, int keys) {
  constexpr int kRow = 64 * WAVES, kRows = kThreads / kRow;  // threads of a row, rows
  constexpr int kCols = HD / 4, kSides = kRow / kCols;       // threads of a stretch, stretches at once
  __shared__ __attribute__((aligned(16))) f32x4 sums[kRows][WAVES == 1 ? 1 : kSides][kCols];
  __shared__ float ls[kRows][WAVES == 1 ? 1 : kSides];
  const int64_t per = ((int64_t)a.max_query * a.H + kRows - 1) / kRows;
  const int b = (int)(blockIdx.x / per), own = threadIdx.x / kRow, t = threadIdx.x % kRow;
  const int64_t row = blockIdx.x % per * kRows + own;
  const int token = (int)(row / a.H), head = (int)(row % a.H), group = a.H / a.KV;
  const View w(a, b, (token * group + head % group) / rows_per_block, rows_per_block, keys);
  // (rows of the same wave leave together, and with WAVES > 1 the whole workgroup has one row)
  if (token >= w.n || w.count <= a.split_tiles) return;
  const int used = min((w.count + a.split_tiles - 1) / a.split_tiles, a.splits);
  const int64_t to = (int64_t)(w.start + token) * a.H + head, at = to * a.splits;
  const float* stat = a.part + (int64_t)a.tokens * a.H * a.splits * HD + at * 2;
  const int side = t / kCols, col = t % kCols * 4;
  float top = -INFINITY;
  for (int s = threadIdx.x & 63; s < used; s += 64) top = fmaxf(top, stat[2 * s]);
#pragma unroll
  for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
  if (top == -INFINITY) top = 0.f;
  float l = 0.f;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = side; s0 < used; s0 += 4 * kSides) {  // four loads under way
    f32x4 v[4];
    float m[4], n[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int s = min(s0 + y * kSides, used - 1);
      v[y] = *reinterpret_cast<const f32x4*>(a.part + (at + s) * HD + col);
      m[y] = stat[2 * s], n[y] = stat[2 * s + 1];
    }
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const float f = s0 + y * kSides < used ? __builtin_amdgcn_exp2f(m[y] - top) : 0.f;
      l += n[y] * f;
      sum += v[y] * f;
    }
  }
  if constexpr (WAVES > 1) {
    sums[own][side][t % kCols] = sum;
    if (t % kCols == 0) ls[own][side] = l;
    __syncthreads();
    if (side) return;
#pragma unroll
    for (int x = 1; x < kSides; ++x) {
      sum += sums[own][x][t];
      l += ls[own][x];
    }
  } else {
#pragma unroll
    for (int x = 32; x >= kCols; x >>= 1) {
      l += __shfl_xor(l, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], x);
    }
    if (side) return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  store4<E>(static_cast<E*>(a.out) + to * HD + col, sum[0] * inv, sum[1] * inv, sum[2] * inv,
            sum[3] * inv);
}

// Rows and keys a tile, blocks of rows, stretches of keys.
struct Plan {
  int rows, keys, row_blocks, splits, split_tiles;
};

// Workgroups for the chip's 256 CUs.  Few rows: half as many 318 us, twice as many 319, 1024 318 (33 sequences
// of 100 to 65536 tokens, a token each; one of 65536 48, 51, 49).  Many rows, where sequences of unlike
// lengths share the chip: 512 113 us, 1024 94, 2048 87, 4096 96 (four chunks of up to 512 tokens over
// 12000), 811, 620, 488, 489 (two of 2048 over 30000); one sequence's stretches are alike and gain
// nothing from more (700 tokens over 20000, heads of 32: 58 us with 1024, 64 with 2048).
constexpr int64_t kFewWanted = 1024, kManyWanted = 2048, kAloneWanted = 1024;
// Keys of a stretch at least, twice as many with many rows: 128 19.4 us, 256 15.5, 512 15.5 (a sequence
// of 200 tokens), 29, 30, 41 (8 trees of up to 64 tokens over 4000).
constexpr int kLeastKeys = 256;
// And at most, twice as many with many rows; a longer one keeps a few workgroups busy alone: 512 339 us,
// 1024 318, 2048 313 (the 33 sequences), many rows 2048 499, 4096 488 (the two chunks).
constexpr int kMostKeys = 2048;
constexpr int kMostSplits = 256;

Plan plan_of(int64_t seqs, int64_t heads, int64_t kv, int64_t max_query, int64_t max_length,
             int64_t window, int64_t sinks) {
  Plan p;
  window = std::min<int64_t>(window, 1 << 30), sinks = std::min<int64_t>(sinks, 1 << 30);
  const int64_t rows = max_query * (heads / kv);
  // 32 rows of 8 sequences over 4000 tokens: 10.3 us as few, 15.6 as many; 4 of 64 over 2000 (or one over
  // 65536) 41 and 57
  p.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : kBlockRows;
  const bool many = p.rows == kBlockRows;
  p.keys = many ? kTile : kKeys;
  p.row_blocks = (int)((rows + p.rows - 1) / p.rows);
  int64_t seen = max_length;  // of one block of rows, at most (and the tiles' edges)
  if (window) seen = std::min(seen, window + sinks + std::min<int64_t>(max_query, 128) + 3 * p.keys);
  const int64_t tiles = std::max<int64_t>(1, (seen + p.keys - 1) / p.keys);
  const int64_t blocks = seqs * kv * p.row_blocks;
  const int64_t wanted = !many ? kFewWanted : seqs > 1 ? kManyWanted : kAloneWanted;
  const int64_t least = (many ? 2 : 1) * kLeastKeys / p.keys;
  const int64_t most = (many ? 2 : 1) * kMostKeys / p.keys;
  // (what one sequence alone fills the chip with is enough for the longest: 8 chunks of 65536
  // tokens, 32 heads of 128, want no partials, where 16 stretches have 136 GB of them)
  const int64_t alone = kv * p.row_blocks;
  const int64_t shorter = std::min((tiles + most - 1) / most, (wanted + alone - 1) / alone);
  int64_t splits = std::max((wanted + blocks - 1) / blocks, shorter);
  splits = std::min<int64_t>(splits, (tiles + least - 1) / least);
  splits = std::max<int64_t>(1, std::min<int64_t>(splits, kMostSplits));
  p.split_tiles = (int)((tiles + splits - 1) / splits);
  p.splits = (int)((tiles + p.split_tiles - 1) / p.split_tiles);
  return p;
}

int page_shift_of(int64_t page) {
  if (page < 16 || page > 256 || (page & (page - 1))) return -1;
  return __builtin_ctzll((unsigned long long)page);
}

bool args_ok(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv, int64_t hd,
             int64_t max_query, int64_t max_length, int64_t window, int64_t sinks) {
  return tokens >= 0 && seqs > 0 && heads > 0 && kv > 0 && heads % kv == 0 && hd > 0 &&
         max_query > 0 && max_length > 0 && window >= 0 && sinks >= 0;
}

// Rows that a workgroup joins: a few stretches take a wave a row, many the whole workgroup (33 sequences of
// up to 65536 tokens in 64 stretches 11.5 -> 7.8 us).
int join_rows(const Plan& p) { return p.splits > 16 ? 1 : kWaves; }

int64_t join_blocks(int64_t seqs, int64_t heads, int64_t max_query, const Plan& p) {
  return p.splits == 1 ? 0 : (max_query * heads + join_rows(p) - 1) / join_rows(p) * seqs;
}

// Sizes that the kernels take (and whose products plan_of forms).
bool sizes_ok(int64_t tokens, int64_t seqs, int64_t heads, int64_t hd, int64_t max_query,
              int64_t max_length) {
  return (hd == 32 || hd == 64 || hd == 128) && heads < (1 << 16) && tokens < (1 << 26) &&
         seqs < (1 << 24) && max_query < (1 << 26) && max_length <= (1 << 30) &&
         max_query * heads < (1 << 30);
}

bool overlap(const void* a, uint64_t a_bytes, const void* b, uint64_t b_bytes) {
  const uint64_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y + b_bytes && y < x + a_bytes;
}

// A launch has fewer than 2^32 threads.
bool launch_ok(int64_t seqs, int64_t heads, int64_t kv, int64_t max_query, const Plan& p) {
  return (seqs * kv * p.splits + 7) * p.row_blocks < (1 << 24) &&
         join_blocks(seqs, heads, max_query, p) < (1 << 24);
}

int64_t workspace_bytes(int64_t tokens, int64_t heads, int64_t hd, const Plan& p) {
  return p.splits == 1 ? 0 : tokens * heads * p.splits * (hd + 2) * 4;
}

template <typename E, int HD>
int launch(const Cached& a, const Plan& p, hipStream_t s) {
  const int64_t groups = ((int64_t)a.seqs * a.KV * p.splits + kXcds - 1) / kXcds * kXcds;
  const dim3 grid((unsigned)(groups * p.row_blocks)), block(kThreads);
  if (p.rows == 16)
    hipLaunchKernelGGL((cached_few_k<E, HD, 1>), grid, block, 0, s, a);
  else if (p.rows == 32)
    hipLaunchKernelGGL((cached_few_k<E, HD, 2>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((a.tree ? cached_many_k<E, HD, true> : cached_many_k<E, HD, false>), grid,
                       block, 0, s, a);
  int rc = rv_host::check_launch();
  if (rc != RV_OK || p.splits == 1) return rc;
  const int64_t blocks = join_blocks(a.seqs, a.H, a.max_query, p);
  hipLaunchKernelGGL((join_rows(p) == 1 ? cached_join_k<E, HD, kWaves> : cached_join_k<E, HD, 1>),
                     dim3((unsigned)blocks), block, 0, s, a, p.rows, p.keys);
  return rv_host::check_launch();
}

}  // namespace

extern "C" {

int64_t rv_cached_attn_workspace_bytes(int64_t tokens, int64_t seqs, int64_t heads,
                                       int64_t kv_heads, int64_t head_dim, int64_t max_query,
                                       int64_t max_length, int64_t window, int64_t sinks) {
  if (!args_ok(tokens, seqs, heads, kv_heads, head_dim, max_query, max_length, window, sinks))
    return -RV_ERR_BAD_SIZE;
  if (!sizes_ok(tokens, seqs, heads, head_dim, max_query, max_length)) return -RV_ERR_UNSUPPORTED;
  const Plan p = plan_of(seqs, heads, kv_heads, max_query, max_length, window, sinks);
  if (!launch_ok(seqs, heads, kv_heads, max_query, p)) return -RV_ERR_UNSUPPORTED;
  return workspace_bytes(tokens, heads, head_dim, p);
}

int rv_cached_attn(const void* q, int64_t q_ld, const void* keys, const void* values,
                   const int32_t* page_table, int64_t ld_table, int64_t table_pages,
                   const int32_t* lengths, const int32_t* starts, const int64_t* tree,
                   int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads,
                   int64_t head_dim, int dtype, int64_t pages, int64_t page_size,
                   int64_t max_query, int64_t max_length, int64_t window, int64_t sinks,
                   void* out, void* workspace, int64_t workspace_bytes_given, void* stream) {
  if (!q || !keys || !values || !page_table || !lengths || !starts || !out)
    return RV_ERR_NULL_POINTER;
  if (!args_ok(tokens, seqs, heads, kv_heads, head_dim, max_query, max_length, window, sinks) ||
      pages <= 0 || table_pages <= 0 || ld_table < table_pages || q_ld < heads * head_dim)
    return RV_ERR_BAD_SIZE;
  const int shift = page_shift_of(page_size);
  if (!sizes_ok(tokens, seqs, heads, head_dim, max_query, max_length) ||
      (dtype != RV_F16 && dtype != RV_BF16) || shift < 0 || (tree && max_query > 64) ||
      pages >= (int64_t(1) << 31) || table_pages >= (int64_t(1) << 31) || q_ld % 8 ||
      !rv_host::aligned16(q) || !rv_host::aligned16(keys) || !rv_host::aligned16(values) ||
      !rv_host::aligned16(out) || !rv_host::aligned16(workspace))
    return RV_ERR_UNSUPPORTED;
  const Plan p = plan_of(seqs, heads, kv_heads, max_query, max_length, window, sinks);
  if (!launch_ok(seqs, heads, kv_heads, max_query, p)) return RV_ERR_UNSUPPORTED;
  const int64_t need = workspace_bytes(tokens, heads, head_dim, p);
  if (need && (!workspace || workspace_bytes_given < need)) return RV_ERR_WORKSPACE;
  if (!tokens) return RV_OK;
  // other workgroups still read what one has written over
  const uint64_t row = heads * head_dim * 2, size = tokens * row;
  const uint64_t cache = (uint64_t)pages * kv_heads * page_size * head_dim * 2;
  if (overlap(out, size, q, (tokens - 1) * (uint64_t)q_ld * 2 + row) ||
      overlap(out, size, keys, cache) || overlap(out, size, values, cache))
    return RV_ERR_UNSUPPORTED;
  Cached a{};
  a.q = q, a.keys = keys, a.values = values, a.out = out;
  a.table = page_table, a.lengths = lengths, a.starts = starts, a.tree = tree;
  a.part = static_cast<float*>(workspace);
  a.q_ld = q_ld, a.table_ld = ld_table, a.table_pages = table_pages;
  a.tokens = (int)tokens, a.seqs = (int)seqs, a.H = (int)heads, a.KV = (int)kv_heads;
  a.pages = (int)pages, a.page_shift = shift, a.max_query = (int)max_query;
  // windows and sinks beyond what a cache holds see all of it
  a.window = (int)std::min<int64_t>(window, 1 << 30);
  a.sinks = window ? (int)std::min<int64_t>(sinks, 1 << 30) : 0;
  a.row_blocks = p.row_blocks, a.splits = p.splits, a.split_tiles = p.split_tiles;
  a.c = (float)(1.4426950408889634 / std::sqrt((double)head_dim));
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == RV_F16) {
    if (head_dim == 32) return launch<_Float16, 32>(a, p, s);
    if (head_dim == 64) return launch<_Float16, 64>(a, p, s);
    return launch<_Float16, 128>(a, p, s);
  }
  if (head_dim == 32) return launch<__bf16, 32>(a, p, s);
  if (head_dim == 64) return launch<__bf16, 64>(a, p, s);
  return launch<__bf16, 128>(a, p, s);
}

}  // extern "C"
