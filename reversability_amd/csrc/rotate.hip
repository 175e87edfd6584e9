// Rotation of queries and keys by position, on the packed projection or on the way
// into a paged cache.
//
//   a pair (a, b) of a head's columns at position p, angle = p base^(-2 i / hd):
//   (a cos - b sin, a sin + b cos); the gradient is the rotation by -angle
//
// A head's pairs are its columns (i, i + hd / 2) or, interleaved, (2 i, 2 i + 1).  The angles'
// cosines and sines come from a table, fp32 [positions][hd / 2][2] of values made in 64
// bits: at position 10^5 a product of the position and a 32-bit rate is off by up to 4e-3 rad.
//
// One thread = 8 pairs of one head of one token: two 16-byte loads and stores, 64 bytes of the
// table (which the heads of a token share in L1).  Bound by the memory's bandwidth: 16 x 2048 tokens of
// 28 heads of 64 46 us a pass, 5.1 TB/s; four prompts of 4096 tokens, 48 heads of 128, into the cache
// 57 us, 5.5 TB/s (a large copy here 4.75).

#include "attn_tile.h"

namespace {

using namespace rv_attn;

constexpr int kRotThreads = 256;

template <typename E>
struct Pairs {
  x8<E> v[2];  // halves: columns i.. and i + hd / 2..; interleaved: 16 columns in order

  template <bool INTERLEAVED>
  __device__ __forceinline__ void turn(const float* __restrict__ cs, bool back) {
    float t[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(t + 4 * i) = rv::ld_f4(cs + 4 * i);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float cos = t[2 * i], sin = back ? -t[2 * i + 1] : t[2 * i + 1];
      E& first = INTERLEAVED ? reinterpret_cast<E*>(v)[2 * i] : reinterpret_cast<E*>(v)[i];
      E& second = INTERLEAVED ? reinterpret_cast<E*>(v)[2 * i + 1]
                              : reinterpret_cast<E*>(v)[8 + i];
      const float a = (float)first, b = (float)second;
      first = (E)(a * cos - b * sin);
      second = (E)(a * sin + b * cos);
    }
  }
  __device__ __forceinline__ void bad() {  // a position outside the table
#pragma unroll
    for (int i = 0; i < 16; ++i) reinterpret_cast<E*>(v)[i] = (E)__builtin_nanf("");
  }
};

struct Rotation {
  const float* table;        // null: no rotation
  const int32_t* positions;  // null: the token's index in its sequence
  int64_t table_rows;
  int64_t seq;
};

// Unit u of a head's hd / 16: where its two 16-byte pieces are.
template <bool INTERLEAVED>
__device__ __forceinline__ void pieces(int u, int hd, int& first, int& second) {
  first = INTERLEAVED ? 16 * u : 8 * u;
  second = INTERLEAVED ? 16 * u + 8 : hd / 2 + 8 * u;
}

// dst = src with the heads [0, turned) rotated, the others copied; both [tokens][all][hd].
template <typename E, bool INTERLEAVED>
__global__ __launch_bounds__(kRotThreads)
void rotate_k(const E* __restrict__ src, E* __restrict__ dst, int64_t items, int all, int turned,
              int hd, Rotation r, bool back) {
  const int64_t item = (int64_t)blockIdx.x * kRotThreads + threadIdx.x;
  if (item >= items) return;
  const int units = hd / 16;
  const int64_t token = item / (all * units);
  const int rest = (int)(item - token * (all * units)), head = rest / units, u = rest % units;
  int first, second;
  pieces<INTERLEAVED>(u, hd, first, second);
  const int64_t at = (token * all + head) * hd;
  Pairs<E> p;
  p.v[0] = *reinterpret_cast<const x8<E>*>(src + at + first);
  p.v[1] = *reinterpret_cast<const x8<E>*>(src + at + second);
  if (head < turned) {
    const int64_t pos = r.positions ? r.positions[token] : token % r.seq;
    if (pos < 0 || pos >= r.table_rows) p.bad();
    else p.template turn<INTERLEAVED>(r.table + (pos * (hd / 2) + 8 * u) * 2, back);
  }
  *reinterpret_cast<x8<E>*>(dst + at + first) = p.v[0];
  *reinterpret_cast<x8<E>*>(dst + at + second) = p.v[1];
}

// Heads [skip, heads + 2 kv) of the tokens' packed rows: queries to q (rotated), keys (rotated)
// and values to the cache's slots.
template <typename E, bool INTERLEAVED>
__global__ __launch_bounds__(kRotThreads)
void append_k(const E* __restrict__ qkv, int64_t ld, E* __restrict__ q, E* __restrict__ keys,
              E* __restrict__ values, const int64_t* __restrict__ slots, int64_t items, int heads,
              int kv, int skip, int hd, int page_shift, int64_t slot_count, Rotation r) {
  const int64_t item = (int64_t)blockIdx.x * kRotThreads + threadIdx.x;
  if (item >= items) return;
  const int units = hd / 16, all = heads + 2 * kv - skip;
  const int64_t token = item / (all * units);
  const int rest = (int)(item - token * (all * units)), head = skip + rest / units,
            u = rest % units;
  int first, second;
  pieces<INTERLEAVED>(u, hd, first, second);
  E* dst;
  if (head < heads) {
    dst = q + (token * heads + head) * hd;
  } else {
    const int64_t slot = slots[token];
    if (slot < 0 || slot >= slot_count) return;  // a token that is not kept
    const int64_t page = slot >> page_shift, row = slot & ((1 << page_shift) - 1);
    const bool value = head >= heads + kv;
    const int h = head - heads - (value ? kv : 0);
    dst = (value ? values : keys) + (((page * kv + h) << page_shift) + row) * hd;
  }
  const E* src = qkv + token * ld + (int64_t)head * hd;
  Pairs<E> p;
  p.v[0] = *reinterpret_cast<const x8<E>*>(src + first);
  p.v[1] = *reinterpret_cast<const x8<E>*>(src + second);
  if (r.table && head < heads + kv) {
    const int64_t pos = r.positions[token];
    if (pos < 0 || pos >= r.table_rows) p.bad();
    else p.template turn<INTERLEAVED>(r.table + (pos * (hd / 2) + 8 * u) * 2, false);
  }
  *reinterpret_cast<x8<E>*>(dst + first) = p.v[0];
  *reinterpret_cast<x8<E>*>(dst + second) = p.v[1];
}

// Where the new tokens of a batch of sequences go: token n of sequence b is the
// (n - starts[b])-th of its starts[b + 1] - starts[b] new ones, the last of its lengths[b].
__global__ __launch_bounds__(kRotThreads)
void cache_plan_k(const int32_t* __restrict__ table, int64_t ld_table, int64_t table_pages,
                  const int32_t* __restrict__ lengths, const int32_t* __restrict__ starts,
                  const int64_t* __restrict__ tree, int64_t seqs, int64_t tokens, int page_shift,
                  int64_t* __restrict__ slots, int32_t* __restrict__ positions) {
  const int64_t n = (int64_t)blockIdx.x * kRotThreads + threadIdx.x;
  if (n >= tokens) return;
  int64_t slot = -1, position = 0;
  if (n >= starts[0] && n < starts[seqs]) {
    int64_t low = 0, high = seqs;  // starts[low] <= n < starts[high]
    while (high - low > 1) {
      const int64_t mid = (low + high) >> 1;
      if (starts[mid] <= n) low = mid;
      else high = mid;
    }
    const int64_t count = (int64_t)starts[low + 1] - starts[low];
    const int64_t context = (int64_t)lengths[low] - count;
    const int64_t at = context + n - starts[low];
    position = at;
    if (tree) {  // bits of tokens that the sequence does not have say nothing
      const uint64_t bits = count < 64 ? (uint64_t(1) << count) - 1 : ~uint64_t(0);
      position = context + __popcll((uint64_t)tree[n] & bits) - 1;
    }
    if (position < 0) position = 0;
    const int64_t page = at >> page_shift;
    if (at >= 0 && page < table_pages) {
      const int64_t id = table[low * ld_table + page];
      if (id >= 0) slot = (id << page_shift) + (at & ((1 << page_shift) - 1));
    }
  }
  slots[n] = slot;
  positions[n] = (int32_t)position;
}

bool head_ok(int64_t heads, int64_t kv) {
  return heads > 0 && kv > 0 && heads % kv == 0 && heads < (1 << 16);
}

bool type_ok(int64_t hd, int dtype) {
  return (hd == 32 || hd == 64 || hd == 128) && (dtype == RV_F16 || dtype == RV_BF16);
}

int page_shift_of(int64_t page) {
  if (page < 16 || page > 256 || (page & (page - 1))) return -1;
  return __builtin_ctzll((unsigned long long)page);
}

int64_t blocks_of(int64_t items) { return (items + kRotThreads - 1) / kRotThreads; }

// A launch has fewer than 2^32 threads.
bool fits(int64_t tokens, int64_t heads, int64_t kv, int64_t hd) {
  return tokens < ((int64_t(1) << 32) - kRotThreads) / ((heads + 2 * kv) * (hd / 16));
}

template <typename E>
int launch_rotate(const void* src, void* dst, int64_t tokens, int64_t heads, int64_t kv,
                  int64_t hd, const Rotation& r, bool interleaved, bool back, hipStream_t s) {
  const int all = (int)(heads + 2 * kv), turned = (int)(heads + kv);
  const int64_t items = tokens * all * (hd / 16);
  const dim3 grid((unsigned)blocks_of(items)), block(kRotThreads);
  const E* x = static_cast<const E*>(src);
  E* y = static_cast<E*>(dst);
  if (interleaved)
    hipLaunchKernelGGL((rotate_k<E, true>), grid, block, 0, s, x, y, items, all, turned, (int)hd,
                       r, back);
  else
    hipLaunchKernelGGL((rotate_k<E, false>), grid, block, 0, s, x, y, items, all, turned, (int)hd,
                       r, back);
  return rv_host::check_launch();
}

template <typename E>
int launch_append(const void* qkv, int64_t ld, void* q, void* keys, void* values,
                  const int64_t* slots, int64_t tokens, int64_t heads, int64_t kv, int64_t hd,
                  int page_shift, int64_t pages, const Rotation& r, bool interleaved,
                  hipStream_t s) {
  const int skip = q ? 0 : (int)heads;
  const int64_t items = tokens * (heads + 2 * kv - skip) * (hd / 16);
  const dim3 grid((unsigned)blocks_of(items)), block(kRotThreads);
  const E* x = static_cast<const E*>(qkv);
  E *qo = static_cast<E*>(q), *k = static_cast<E*>(keys), *v = static_cast<E*>(values);
  const int64_t count = pages << page_shift;
  if (interleaved)
    hipLaunchKernelGGL((append_k<E, true>), grid, block, 0, s, x, ld, qo, k, v, slots, items,
                       (int)heads, (int)kv, skip, (int)hd, page_shift, count, r);
  else
    hipLaunchKernelGGL((append_k<E, false>), grid, block, 0, s, x, ld, qo, k, v, slots, items,
                       (int)heads, (int)kv, skip, (int)hd, page_shift, count, r);
  return rv_host::check_launch();
}

}  // namespace

extern "C" {

int rv_rotate_qkv(const void* src, void* dst, int64_t tokens, int64_t seq, int64_t heads,
                  int64_t kv_heads, int64_t head_dim, int dtype, const float* table,
                  int64_t table_rows, const int32_t* positions, int interleaved, int back,
                  void* stream) {
  if (!src || !dst || !table) return RV_ERR_NULL_POINTER;
  if (tokens < 0 || seq <= 0 || table_rows <= 0 || !head_ok(heads, kv_heads))
    return RV_ERR_BAD_SIZE;
  if (!type_ok(head_dim, dtype) || !rv_host::aligned16(src) || !rv_host::aligned16(dst) ||
      !rv_host::aligned16(table) || !fits(tokens, heads, kv_heads, head_dim))
    return RV_ERR_UNSUPPORTED;
  if (!tokens) return RV_OK;
  const Rotation r{table, positions, table_rows, seq};
  const hipStream_t s = (hipStream_t)stream;
  return dtype == RV_F16
             ? launch_rotate<_Float16>(src, dst, tokens, heads, kv_heads, head_dim, r,
                                       interleaved != 0, back != 0, s)
             : launch_rotate<__bf16>(src, dst, tokens, heads, kv_heads, head_dim, r,
                                     interleaved != 0, back != 0, s);
}

int rv_append_kv(const void* qkv, int64_t ld, void* q, void* keys, void* values,
                 const int64_t* slots, int64_t tokens, int64_t heads, int64_t kv_heads,
                 int64_t head_dim, int dtype, int64_t pages, int64_t page_size,
                 const float* table, int64_t table_rows, const int32_t* positions,
                 int interleaved, void* stream) {
  if (!qkv || !keys || !values || !slots) return RV_ERR_NULL_POINTER;
  if (table && (!q || !positions)) return RV_ERR_NULL_POINTER;
  if (tokens < 0 || pages <= 0 || !head_ok(heads, kv_heads) ||
      ld < (heads + 2 * kv_heads) * head_dim || (table && table_rows <= 0))
    return RV_ERR_BAD_SIZE;
  const int shift = page_shift_of(page_size);
  if (!type_ok(head_dim, dtype) || shift < 0 || ld % 8 || !rv_host::aligned16(qkv) ||
      (q && !rv_host::aligned16(q)) || !rv_host::aligned16(keys) || !rv_host::aligned16(values) ||
      (table && !rv_host::aligned16(table)) || pages >= (int64_t(1) << 31) ||
      !fits(tokens, heads, kv_heads, head_dim))
    return RV_ERR_UNSUPPORTED;
  if (!tokens) return RV_OK;
  const Rotation r{table, positions, table_rows, 1};
  const hipStream_t s = (hipStream_t)stream;
  return dtype == RV_F16
             ? launch_append<_Float16>(qkv, ld, q, keys, values, slots, tokens, heads, kv_heads,
                                       head_dim, shift, pages, r, interleaved != 0, s)
             : launch_append<__bf16>(qkv, ld, q, keys, values, slots, tokens, heads, kv_heads,
                                     head_dim, shift, pages, r, interleaved != 0, s);
}

int rv_cache_plan(const int32_t* page_table, int64_t ld_table, int64_t table_pages,
                  const int32_t* lengths, const int32_t* starts, const int64_t* tree,
                  int64_t seqs, int64_t tokens, int64_t page_size, int64_t* slots,
                  int32_t* positions, void* stream) {
  if (!page_table || !lengths || !starts || !slots || !positions) return RV_ERR_NULL_POINTER;
  if (seqs <= 0 || tokens < 0 || table_pages <= 0 || ld_table < table_pages)
    return RV_ERR_BAD_SIZE;
  const int shift = page_shift_of(page_size);
  if (shift < 0 || tokens >= (int64_t(1) << 31) || seqs >= (int64_t(1) << 31))
    return RV_ERR_UNSUPPORTED;
  if (!tokens) return RV_OK;
  hipLaunchKernelGGL(cache_plan_k, dim3((unsigned)blocks_of(tokens)), dim3(kRotThreads), 0,
                     (hipStream_t)stream, page_table, ld_table, table_pages, lengths, starts, tree,
                     seqs, tokens, shift, slots, positions);
  return rv_host::check_launch();
}

}  // extern "C"
