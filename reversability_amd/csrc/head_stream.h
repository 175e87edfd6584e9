// The tied head's logits for narrow models (d <= 256), streamed through the matrix
// cores and reduced or differentiated on the way: no logit reaches memory in the
// forward, only their 16-bit gradients do in the backward.
//
// A wave keeps its 64 rows of x as MFMA fragments in registers for the whole
// kernel; the head passes through LDS once per 256 rows, 64 of its rows (columns of
// the logits) a stage, in two buffers that direct-to-LDS loads fill a stage ahead.
// Per 32 columns a wave issues KS reads of 16 bytes a lane and 2 KS MFMAs (half the
// LDS traffic per MFMA of a tile whose two operands come from LDS), and between the
// MFMAs of one block the exponentials of the block before: a multiply-add, a v_exp
// and an add per value, about 24 VALU cycles beside 32 of the MFMA.
//
// z log2e is taken once per value, z's products in fp32: exp(z - lse) =
// exp2(z log2e - R) with one rounding, R = the running maximum of z log2e rounded
// (forward) or lse log2e (backward).
//
// 16896 x 256 over 50257, fp16 (435 GFLOP): forward 390-440 us, 990-1115 TFLOP/s (the
// 256 x 256 tiles of gemm_kernel with the LogProb epilogue 626), backward 440-510 us with
// its 1.7 GB of stores (846; 485-560 in panels of 64 columns, where a store instruction
// wrote halves of 16 rows' 128 bytes instead of a whole KB; without its stores it would take
// about as long as the forward); width 128 forward 244 us (417), backward 355 us (457 in
// panels of 64 columns, 640 row by row).  Bound by the matrix cores' power: at 1.7 GHz they
// are busy 66% of the forward's time, and a wave waits 0.4 of its own.  A few rows are bound by the first bytes' way from HBM and the join (51
// rows 12 + 4 us; 64 rows to a workgroup, so that no wave idles, 22.0 -> 21.6 us of a
// call: left out).  Wider than 256 the rows' fragments no longer fit beside the
// accumulators of 64 rows, and with 32 rows a wave every MFMA would read 1 KB of LDS, all
// that the LDS delivers.
//
// Registers: all 256 at widths 129 to 256.  Forward and backward keep 3 values in scratch and
// read them after the loop or where a label falls; with remainders (GradLow) it is 17, a
// fragment of x among them, which every block reads again behind a wait for all loads and
// stores: 300 x 256 over 50257 37 us where the forward takes 22 (0.54 of 4 matrix cores busy).
//
// Included by mlp_gemm.hip, whose staging, LDS and epilogue helpers it uses.
#pragma once

// What the kernel leaves behind: log-probabilities' statistics, the logits' gradients in 16
// bits, or those and what the 16 bits left out.
enum class Stream { Logp, Grad, GradLow };

struct StreamArgs {
  const __half* x;        // [m][d]
  const __half* head;     // [n][d]
  int64_t m, n, d;
  int64_t stages, chunk;  // stages of 64 columns in all, and per workgroup
  int64_t tiles_m, tiles; // workgroups: 256 rows x chunk stages, tiles_m fastest
  float2* part;           // forward: [tile column][m]
  __half* out;            // backward: panels [n / 32][panel_rows][32]
  HeadLogp head_logp;
  int64_t panel_rows;     // m, or 2 m with the rows' remainders behind them
};

// One lane's 16-byte chunk address in a stage: column (row of the head) c, 16-byte
// chunk q is at c * 32 KS + ((q ^ (c & 15)) * 16): the columns' reads of one chunk
// fall on different banks.
template <int KS, bool BF, Stream MODE>
__device__ __forceinline__ void head_stream(const StreamArgs& a) {
  constexpr bool GRAD = MODE != Stream::Logp;
  constexpr int kRow = KS * 32;              // bytes of a column in LDS
  constexpr int kStage = 64 * kRow;          // bytes of a stage
  constexpr int kDma = kStage / 1024 / 4;    // loads per wave and stage
  constexpr int kCols = 1024 / kRow;         // columns per load
  constexpr int D = 4;                       // fragment reads in flight
  static_assert(KS >= 8 && KS % D == 0 && kCols >= 1 && 16 % (4 * kCols) == 0, "staging");
  __shared__ __attribute__((aligned(1024))) char lds[2 * kStage];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // workgroups go to the XCDs round robin: each XCD takes a contiguous share of the
  // tiles, whose workgroups read the same columns at a time
  const int64_t share = (a.tiles + 7) >> 3;
  const int64_t tile = (int64_t)(blockIdx.x & 7) * share + (blockIdx.x >> 3);
  if ((int64_t)(blockIdx.x >> 3) >= share || tile >= a.tiles) return;
  const int64_t tm = tile % a.tiles_m, tn = tile / a.tiles_m;
  const int64_t first = tn * a.chunk;
  const int stages = __builtin_amdgcn_readfirstlane(
      (int)(a.stages - first < a.chunk ? a.stages - first : a.chunk));
  const int64_t m0 = tm * 256 + wave * 64;   // the wave's first row
  const bool live = m0 < a.m;                // a wave without rows only loads

  // staging: load `it` of a wave fills columns (it * 4 + wave) * kCols ..; the swizzle
  // repeats every 16 columns, i.e. every kTurn loads
  constexpr int kTurn = 16 / (4 * kCols);
  uint32_t off[kTurn];
#pragma unroll
  for (int t = 0; t < kTurn; ++t) {
    const int c = (t * 4 + wave) * kCols + lane / (kRow / 16);
    const int q = (lane % (kRow / 16)) ^ (c & 15);
    off[t] = q * 8 < a.d ? (uint32_t)((c * a.d + q * 8) * 2) : 0x80000000u;  // past d: zeros
  }
  const int64_t bytes = a.n * a.d * 2, step = 64 * a.d * 2;
  const int64_t base = uniform(reinterpret_cast<int64_t>(a.head));
  const int turn = __builtin_amdgcn_readfirstlane((int)(16 * a.d * 2));
  auto fill = [&](int st) __attribute__((always_inline)) {  // a stage past the end reads nothing (and is not used)
    const int64_t at = (first + st) * step, left = st < stages ? bytes - at : 0;
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
        reinterpret_cast<char*>(base + at), 0,
        left <= 0 ? 0 : left < INT32_MAX ? (int)left : INT32_MAX, kRsrcWord3);
    char* to = lds + (st & 1) * kStage;
#pragma unroll
    for (int it = 0; it < kDma; ++it)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (RV_LDS void*)(to + (it * 4 + wave) * 1024),
                                               16, off[it % kTurn] + (it / kTurn) * turn, 0, 0,
                                               0);
  };
  fill(0);

  // x: fragment (i, ks) holds row i * 32 + lane % 32, k = ks * 16 + (lane / 32) * 8 ..
  f16x8 fx[2][KS];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t row = m0 + i * 32 + (lane & 31);
    const __half* src = a.x + (row < a.m ? row : a.m - 1) * a.d;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int k = ks * 16 + (lane >> 5) * 8;
      fx[i][ks] = k < a.d ? *reinterpret_cast<const f16x8*>(src + k) : f16x8{};
    }
  }

  // per row i of this lane: its label (relative to the columns at hand), and the
  // running reference and sum (forward) or the factors of the gradient (backward)
  const int64_t col0 = first * 64;
  int label[2];
  float top[2], ref[2], sum[2], g[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t row = m0 + i * 32 + (lane & 31);
    const bool in = row < a.m;
    const int64_t y = in ? a.head_logp.labels[row] : a.head_logp.ignore;
    const bool ignored = y == a.head_logp.ignore;
    const bool bad = !ignored && (y < 0 || y >= a.head_logp.vocab);
    // as 32 bits: only a label in the chunk's columns matters
    const int64_t c = y - col0;
    label[i] = !ignored && !bad && c >= 0 && c < (int64_t)stages * 64 ? (int)c : -1;
    if constexpr (GRAD) {
      g[i] = ignored ? 0.f : bad ? NAN
             : a.head_logp.grad[row] * a.head_logp.scale[row * a.head_logp.scale_step];
      const float lse = ignored ? INFINITY : a.head_logp.lse[row];
      ref[i] = lse * kLog2e;  // its rounding is taken back in sum
      sum[i] = ignored ? 0.f
                       : -g[i] * __builtin_amdgcn_exp2f(-__builtin_fmaf(lse, kLog2e, -ref[i]));
    } else {
      g[i] = sum[i] = 0.f;
      top[i] = kLowest;  // finite: differences of it are numbers
      ref[i] = top[i] * kLog2e;
    }
  }
  // backward: the wave's 64 rows of a panel (32 columns: a block); rows past the end are
  // past the resource
  const int rows_here = (int)uniform(a.m - m0 < 64 ? (a.m - m0 < 0 ? 0 : a.m - m0) : 64);
  const int64_t out0 = uniform(reinterpret_cast<int64_t>(a.out) + (first * 2 * a.panel_rows + m0) * 64);
  const uint32_t out_off = (uint32_t)((lane & 15) * 64 + (lane >> 4 & 1) * 32 + (lane >> 5) * 16);

  fill(1);  // both buffers are free at the start

  const uint32_t lds0 = (uint32_t)(size_t)(RV_LDS void*)lds;
  const uint32_t at = (lane & 31) * kRow + (((lane >> 5) ^ (lane & 15)) << 4);
  f32x16 acc[2][2];  // [block of the pair][row block]
  f16x8 fb[D];

  // Row block i of a finished block (its columns start at `col`, counted from col0):
  // what has to be known before its exponentials.
  auto open = [&](f32x16 (&z)[2], int i, int col) __attribute__((always_inline)) {
    if (col0 + col + 32 > a.head_logp.vocab) {  // the last columns
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (col0 + col + (e >> 2) * 8 + (lane >> 5) * 4 + (e & 3) >= a.head_logp.vocab)
          z[i][e] = -INFINITY;
    }
    const int c = label[i] - col;
    const bool mine = c >= 0 && c < 32 && (c & 4) == (lane >> 5) * 4;
    if constexpr (!GRAD) {
#pragma unroll
      for (int e = 0; e < 16; ++e) top[i] = fmaxf(top[i], z[i][e]);
      const float next = top[i] * kLog2e;
      sum[i] *= __builtin_amdgcn_exp2f(ref[i] - next);
      ref[i] = next;
      if (__any(mine)) {
        const int e0 = (c >> 3) * 4 + (c & 3);
        float v = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (e == e0) v = z[i][e];
        if (mine) a.head_logp.label_logit[m0 + i * 32 + (lane & 31)] = v;
      }
    }
  };
  // Value e of row block i.
  auto value = [&](f32x16 (&z)[2], int i, int e) __attribute__((always_inline)) {
    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(z[i][e], kLog2e, -ref[i]));
    // pinned here: the compiler would move the work behind the MFMAs, to its use
    if constexpr (GRAD) {
      float v = p * sum[i];
      asm volatile("" : "+v"(v));
      z[i][e] = v;
    } else {
      sum[i] += p;
      asm volatile("" : "+v"(sum[i]));
    }
  };
  // The 16-bit results of row block i and their stores to the panels at `to`.  A lane
  // holds 4 consecutive columns of each 8; the swap of the halves' odd and even
  // groups leaves it 8 consecutive ones of each 16.
  auto put = [&](const f32x16 (&z)[2], int i, int col, int64_t to) __attribute__((always_inline)) {
    uint32_t w[8];  // pairs of columns; word 2 q + k: columns 8 q + cq + 2 k
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = pack2<BF>(z[i][2 * k], z[i][2 * k + 1]);
    // halves: word 4 h + k holds columns 16 h + 8 (lane / 32) + 2 k of its row
#pragma unroll
    for (int k = 0; k < 8; k += 4)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const auto t = __builtin_amdgcn_permlane32_swap(w[k + u], w[k + 2 + u], false, false);
        w[k + u] = t[0];
        w[k + 2 + u] = t[1];
      }
    // rows: store r covers rows 16 r + lane % 16, columns 16 (lane / 16 % 2) + 8 (lane /
    // 32) ..: 1 KB of a panel
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const auto t = __builtin_amdgcn_permlane16_swap(w[k], w[k + 4], false, false);
      w[k] = t[0];
      w[k + 4] = t[1];
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const u32x4 v = {w[4 * r], w[4 * r + 1], w[4 * r + 2], w[4 * r + 3]};
      // all of the offset in the vector register: with a scalar part the compiler
      // leaves no wait state between a 16-byte store and the next write of its data
      // registers, and lanes 12 .. 15 of each 16 stored what came after.  Streaming.
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(
          reinterpret_cast<char*>(to + (int64_t)(col >> 5) * a.panel_rows * 64), 0, rows_here * 64,
          kRsrcWord3);
      __builtin_amdgcn_raw_buffer_store_b128(
          v, rsrc, (int)(out_off + (uint32_t)((i * 32 + r * 16) * 64)), 0, 2);
    }
  };
  // After its values: the label's part and the results.
  auto close = [&](f32x16 (&z)[2], int i, int col) __attribute__((always_inline)) {
    if constexpr (GRAD) {
      const int c = label[i] - col;
      const bool mine = c >= 0 && c < 32 && (c & 4) == (lane >> 5) * 4;
      if (__any(mine)) {
        const int e0 = mine ? (c >> 3) * 4 + (c & 3) : -1;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (e == e0) z[i][e] += g[i];
      }
      if (col0 + col + 32 > a.head_logp.vocab) {  // pad columns: zero, whatever the row's g
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (col0 + col + (e >> 2) * 8 + (lane >> 5) * 4 + (e & 3) >= a.head_logp.vocab)
            z[i][e] = 0.f;
      }
      put(z, i, col, out0);
      if constexpr (MODE == Stream::GradLow) {
#pragma unroll
        for (int e = 0; e < 16; ++e) z[i][e] -= round16<BF>(z[i][e]);
        put(z, i, col, out0 + a.head_logp.low * 64);
      }
    }
  };
  // Fragment read r (0 .. 2 KS - 1) of a stage at LDS byte `tile`.
  auto read = [&](auto rc, uint32_t tile) __attribute__((always_inline)) {
    constexpr int r = decltype(rc)::value;
    fb[r % D] = b128_read<(r / KS) * 32 * kRow>((tile + at) ^ ((r % KS) * 32));
  };
  // The MFMAs of block J of the stage at `tile`, with the work on the block before
  // (`done`, columns from `col`) between them.  Reads run D ahead, to the stage's end.
  auto block = [&](auto jc, auto wc, uint32_t tile, f32x16 (&z)[2], f32x16 (&done)[2],
                   int col) __attribute__((always_inline)) {
    constexpr int J = decltype(jc)::value;
    constexpr bool work = decltype(wc)::value;
    if constexpr (work) {
      open(done, 0, col);
      open(done, 1, col);
    }
    static_for<KS>([&](auto kc) __attribute__((always_inline)) {
      constexpr int ks = decltype(kc)::value, r = J * KS + ks;
      lds_wait<(2 * KS - 1 - r < D - 1 ? 2 * KS - 1 - r : D - 1)>();
      after_wait(fb[r % D]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const f32x16 zero{};
        const f32x16 c = ks == 0 ? zero : z[i];
        if constexpr (BF)
          z[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fb[r % D]),
                                                         __builtin_bit_cast(bf16x8, fx[i][ks]), c,
                                                         0, 0, 0);
        else
          z[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fb[r % D], fx[i][ks], c, 0, 0, 0);
        if constexpr (work) {
#pragma unroll
          for (int e = 0; e < 32; ++e)  // 32 values over the block's MFMAs
            if (e * KS * 2 / 32 == ks * 2 + i) value(done, e / 16, e % 16);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (r + D < 2 * KS) read(std::integral_constant<int, r + D>{}, tile);
    });
    if constexpr (work) {
      close(done, 0, col);
      close(done, 1, col);
    }
  };
  constexpr std::integral_constant<int, 0> j0{};
  constexpr std::integral_constant<int, 1> j1{};
  constexpr std::integral_constant<bool, true> yes{};
  // Stage st: `begun` once a block is waiting for its exponentials.
  auto stage = [&](int st, auto begun) __attribute__((always_inline)) {
    // this wave's loads of the stage have to have landed.  Newer than them are, in the
    // backward, the stores of two blocks (of one in the second stage), four a block or
    // eight (then the wait is for some of them too), always issued in full
    if constexpr (!decltype(begun)::value) wait_vmcnt<kDma>();  // the next stage's
    else if (GRAD && live && st > 1) wait_vmcnt<8>();
    else if (GRAD && live) wait_vmcnt<4>();
    else wait_vmcnt<0>();
    lds_barrier();  // every wave's loads have landed, and none reads the stage before
    if constexpr (decltype(begun)::value) fill(st + 1);
    if (!live) return;
    const uint32_t tile = lds0 + (st & 1) * kStage;
    static_for<D>([&](auto rc) __attribute__((always_inline)) { read(rc, tile); });
    block(j0, begun, tile, acc[0], acc[1], st * 64 - 32);
    block(j1, yes, tile, acc[1], acc[0], st * 64);
  };
  stage(0, std::integral_constant<bool, false>{});
  for (int st = 1; st < stages; ++st) stage(st, yes);
  wait_vmcnt<0>();  // the stage past the end
  if (!live) return;
  const int col = stages * 64 - 32;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    open(acc[1], i, col);
#pragma unroll
    for (int e = 0; e < 16; ++e) value(acc[1], i, e);
    close(acc[1], i, col);
    if constexpr (!GRAD) {
      // the other half of the row's columns is the partner lane's; the references'
      // rounding is taken back
      const float other = __shfl_xor(top[i], 32, 64), s = __shfl_xor(sum[i], 32, 64);
      const float r = __shfl_xor(ref[i], 32, 64);
      const float both = fmaxf(top[i], other), next = fmaxf(ref[i], r);
      float total = sum[i] * __builtin_amdgcn_exp2f(ref[i] - next) +
                    s * __builtin_amdgcn_exp2f(r - next);
      total *= __builtin_amdgcn_exp2f(-__builtin_fmaf(both, kLog2e, -next));
      const int64_t row = m0 + i * 32 + (lane & 31);
      if (lane < 32 && row < a.m) a.part[tn * a.m + row] = make_float2(both, total);
    }
  }
}

template <int KS, bool BF, Stream MODE>
__global__ __launch_bounds__(256, 2)
void head_stream_k(StreamArgs a) {
  head_stream<KS, BF, MODE>(a);
}
