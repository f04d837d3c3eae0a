// Block-scaled 8-bit matrix products of many rows whose results are rounded to 16 bits (linear, down): the tile kernel.
//
//   y[m, n] = sum over blocks b of 2^e(m, b) s(n, b) sum over k in b of x[m, k] w[n, k]
//
// A workgroup of four wavefronts computes up to 128 rows x 256 weight rows over 128-wide k slabs.  An 8-bit slab row is
// 128 bytes, as a 64-wide slab row of the 16-bit kernels is, so the movement of data is theirs: activation rows go to an
// LDS ring by direct global -> LDS copies with 16-byte chunks swizzled by row; weight fragments come straight from the
// tiled layout into alternating register sets; everything is requested two to six slabs ahead (tl_depth) and vector
// memory is awaited by count.  A slab is one 16x16x128 matrix instruction per 16 x 16 tile where the 16-bit kernels have
// two of half the rate: the same bytes feed twice the arithmetic.
//
// Scales: the activations' E8M0 bytes of the whole tile are laid out in LDS once, the eight bytes that a
// lane's eight row tiles need for a slab side by side, and enter the instruction as its own operand.  The
// weights' fp32 scales multiply the slab's sum on its way into the accumulator, or, where all those of the tile are
// powers of two, enter the instruction as exponents (4096 rows of 2048 by 5632 weight rows: 65 -> 57 us).  A tile
// looks at its scales and chooses by itself: what a row comes out as depends on its own weights' scales alone, as
// they are at the time of the call, and not on the other matrices of the call.  (The branch waits for the scales: 0.7 us
// of such a call.  Behind the first copies instead, registers spill.)
//
// What bounds it: two workgroups share a compute unit, whose matrix pipes are busy for 52 % of the cycles in which it has
// work (linear; down 40 %); the 4.5 us before a tile's first slab and 4 us behind its last are covered by the other
// workgroup only.  4096 rows of 2048 by 5632 weight rows: 51 us, 1.85 PFLOP/s (a library 8-bit product of that size:
// 51 us).  Down of 4096 tokens, 6 of 64 experts of 1408 x 2048, shared 2816: 189 GFLOP in 124 us.  Lower tiles for a
// fuller last round lose: 96 rows 54 us, 64 rows 63.
#include <type_traits>

#include "fp8_tile.h"

namespace sparse {

constexpr int kTlRowBytes = kF8Block;               // LDS row of one k slab
constexpr int kTlSlab = kPfBM * kTlRowBytes;
constexpr int kTlRing = kPfStages * kTlSlab;

// A tile of 32 NMI rows keeps S slabs of weight fragments in registers and S + 1 slabs of rows in LDS.  What a
// low tile saves in accumulators and rows goes into depth: its slab is half the work or less, and four slabs
// ahead its weights are as far away in time.
constexpr int tl_depth(int nmi, bool narrow) { return narrow ? 6 : nmi == 1 ? 4 : nmi == 2 ? 3 : 2; }
// "The copies of the next slab have landed": its copies were followed by their own slab's 2 NG fragment loads and by
// S - 1 slabs of NMI copies and 2 NG loads each.
constexpr int tl_younger(int nmi, bool narrow) {
  const int loads = narrow ? 4 : 8;
  return loads + (tl_depth(nmi, narrow) - 1) * (nmi + loads);
}
// The last slabs, those behind the loop, request nothing (nobody would use it, and the compiler drops a load without a
// user, so that a count could not rely on it).  In number j of them the next slab's copies are followed by its own
// fragment loads and by copies and loads of the S - 2 - j slabs behind it.
constexpr int tl_younger_tail(int nmi, bool narrow, int j) {
  const int loads = narrow ? 4 : 8, behind = tl_depth(nmi, narrow) - 2 - j;
  return loads + behind * (nmi + loads);
}
static_assert(tl_younger(4, false) == 20, "the count of the 16-bit kernels");
static_assert(tl_younger_tail(2, false, -1) == tl_younger(2, false) && tl_younger_tail(1, true, 4) == 4, "one rule for both");
static_assert(tl_younger(2, false) < 64 && tl_younger(1, false) < 64 && tl_younger(1, true) < 64, "six bits");
static_assert((tl_depth(1, false) + 1) * 32 * kTlRowBytes <= kTlRing && (tl_depth(2, false) + 1) * 64 * kTlRowBytes <= kTlRing, "rings fit");
constexpr int kTlNarrowRows = 32;
constexpr int kTlNarrowRing = (tl_depth(1, true) + 1) * kTlNarrowRows * kTlRowBytes;
constexpr int kTlScaleBytes = kPfBM + 2 * sizeof(float);   // per slab: activation bytes, two weight scales
static_assert(kTlSlab == kPfLdsA, "the slab geometry is that of the 16-bit kernels");

// F: the 16-bit format of outputs, route weights and gate logits
// kNarrow: tiles of 32 rows by 128, three workgroups to a compute unit instead of two
template <typename F, bool kNarrow>
__global__ __launch_bounds__(kPfThreads, kNarrow ? 3 : 2) void f8_tile_kernel(const TileArgs a) {
  constexpr int NG = kNarrow ? 2 : 4;                         // 16-row groups of weights per wavefront
  constexpr int kRows = kNarrow ? kTlNarrowRows : kPfBM;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kNarrow ? kTlNarrowRing : kTlRing];
  __shared__ float s_row[kPfBM];          // factor of a row
  extern __shared__ __attribute__((aligned(16))) uint8_t s_scales[];   // [nk][128] bytes, then [nk][2] floats

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int fr = lane & 15, fq = lane >> 4;
  const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) uint8_t*)(&lds[0])));

  // ---- which tile (wavefront-uniform) ------------------------------------------------
  int slot, r0, M, bn;
  if (a.map != nullptr) {
    if (!tl_queued(a, slot, r0, M, bn)) return;
  } else {
    // block b runs on XCD b % 8; an XCD takes a contiguous share of the (column tile, row tile) order
    const int total = a.mt * a.nt, xcd = blockIdx.x % kPfXcds, rank = blockIdx.x / kPfXcds;
    const int first = static_cast<int>(static_cast<int64_t>(total) * xcd / kPfXcds);
    const int end = static_cast<int>(static_cast<int64_t>(total) * (xcd + 1) / kPfXcds);
    if (first + rank >= end) return;
    bn = (first + rank) / a.mt;
    r0 = (first + rank - bn * a.mt) * a.rows;
    M = min(a.rows, a.p.T - r0);
    slot = -1;
  }
  if (M <= 0) return;
  const bool dense = slot < 0;
  const int Kdim = dense ? a.p.Ks : a.p.Kr, N = dense ? a.p.Ns : a.p.Nr;
  const int nk = (Kdim + kF8Block - 1) / kF8Block;
  const uint32_t ld = static_cast<uint32_t>(nk) * kF8Block;
  const int n0 = bn * 64 * NG;   // first output column of this tile

  // ---- operand addresses ------------------------------------------------------------
  // Row r keeps chunk 2q + h at position (q + 4h) ^ f(r), f(r) = ((r >> 1) & 7) ^ ((r & 1) << 2); of eight rows
  // from 8 i on, f depends on i through its low bit only, which flips bit 0 of the chunk.
  const int l3 = lane >> 3;
  const int pos0 = (lane & 7) ^ ((l3 >> 1) ^ ((l3 & 1) << 2));
  const uint32_t chunk0 = ((pos0 & 3) << 1) | (pos0 >> 2);
  // rows are addressed from the tile's first one, so that 32-bit offsets always reach
  const uint8_t* abase = uniform_ptr((dense ? a.p.act_s : a.p.act_r) + static_cast<size_t>(r0) * ld);
  const uint8_t* sbase = (dense ? a.p.act_ss : a.p.act_rs) + static_cast<size_t>(r0) * nk;
  auto source_row = [&](int m) { return static_cast<uint32_t>(min(m, M - 1)); };
  // The wavefront's 64 weight rows are four 16-row groups; a group's slab is 2 KB, its two halves 1 KB each in lane order.
  const uint8_t* wbase[NG];
  const float *ws0, *ws1;      // the scales of the tile's two 128-row blocks
  const uint32_t woff = lane * 16;
  {
    const uint8_t* w0 = a.p.w0;
    const float* s0 = a.p.s0;
    if (!dense) {
      const uint8_t* base = a.p.slab + static_cast<uint64_t>(slot) * a.p.slot_stride;
      w0 = base + a.p.off0;
      s0 = reinterpret_cast<const float*>(base + a.p.soff0);
    }
    const int last16 = ((N + 15) & ~15) - 16;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int n = min(n0 + wave * 16 * NG + g * 16, last16);
      wbase[g] = uniform_ptr(w0 + static_cast<size_t>(n >> 4) * nk * kF8TileBytes);
    }
    const int nblk = (N + kF8Block - 1) / kF8Block, b0 = n0 / kF8Block;
    ws0 = s0 + static_cast<size_t>(b0) * nk;
    ws1 = s0 + static_cast<size_t>(min(b0 + 1, nblk - 1)) * nk;
  }
  typedef const __attribute__((address_space(1))) char* gptr_t;
  auto wload = [&](int g, int slab, int h) __attribute__((always_inline)) {
    gptr_t p = (gptr_t)(reinterpret_cast<uintptr_t>(wbase[g]) + static_cast<size_t>(slab) * kF8TileBytes + h * 1024);
    return *reinterpret_cast<const __attribute__((address_space(1))) i32x4*>(p + woff);
  };

  // ---- scales to LDS, row factors ------------------------------------------------------
  // Bytes are fetched eight at a time before the first is stored: one by one, each would wait a memory latency.
  // Every wavefront looks at all weight scales (and stores a quarter of them); returns whether all are exponents.
  auto fill_scales = [&]() __attribute__((always_inline)) {
    bool odd = false;
    constexpr int kShare = kPfThreads / kRows;    // threads of a row
    const int m = tid / kShare, part = tid % kShare;
    const uint8_t* src = sbase + static_cast<size_t>(source_row(m)) * nk;
    uint8_t* dst = s_scales + (m & 15) * 8 + (m >> 4);
    float* w = reinterpret_cast<float*>(s_scales + nk * kPfBM);
    for (int kb0 = part; kb0 < nk; kb0 += 8 * kShare) {
      uint8_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = src[min(kb0 + kShare * i, nk - 1)];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (kb0 + kShare * i < nk) dst[(kb0 + kShare * i) * kPfBM] = v[i];
    }
    for (int i = lane; i < 2 * nk; i += 64) {
      const float v = ((i & 1) ? ws1 : ws0)[i >> 1];
      if (((i >> 6) & 3) == wave) w[i] = v;
      odd |= !(kNarrow && (i & 1)) && !tl_is_exponent<-126, 127>(v);      // (a narrow tile lies in one 128-row block)
    }
    // factor of each row, the route weight or the sigmoid of the shared expert's gate
    if (tid < kPfBM) {
      float sc = 1.f;
      if (tid < M) {
        const int p = r0 + tid;
        if (!dense) sc = F::from_bits(static_cast<const uint16_t*>(a.p.topv)[a.p.perm[p]]);
        else if (a.p.gate_s != nullptr) sc = sigmoid_f32(F::from_bits(static_cast<const uint16_t*>(a.p.gate_s)[p]));
      }
      s_row[tid] = sc;
    }
    return !__any(odd);
  };

  // Byte offset of the lane's piece of each copy inside k slab 0: a wavefront copies a quarter of the tile's sub-tiles
  // of 32 rows (past the last one the offsets repeat the tile's last row and go unused).
  const int nmi = kNarrow ? 1 : (M + 31) >> 5;
  uint32_t doff[kNarrow ? 1 : 4];
#pragma unroll
  for (int it = 0; it < (kNarrow ? 1 : 4); ++it)
    doff[it] = source_row((wave * nmi + it) * 8 + l3) * ld + ((chunk0 ^ ((wave * nmi + it) & 1)) << 4);
  const bool pow2 = fill_scales() && a.p.pow2 != 0;

  // The tile's rows are processed in sub-tiles of 32; a segment's last tile is specialised on how many of
  // them hold rows.  kPow2: every weight scale of the tile enters the instruction as its exponent.
  auto body = [&](auto nmi_c, auto pow2_c) __attribute__((always_inline)) {
    constexpr int NMI = decltype(nmi_c)::value;
    constexpr bool kPow2 = decltype(pow2_c)::value;
    constexpr int NMT = 2 * NMI;                  // 16-row tiles
    // While slab kt is multiplied, the rows of slab kt+S travel to the LDS buffer slab kt-1 has left and the
    // fragments of slab kt+S to the registers the last row pair has just finished with.  Vector memory retires
    // in order, so what has landed is known by counting.  Slabs past the end refetch the last one; the up to S - 1
    // slabs behind the loop find everything requested.
    constexpr int S = tl_depth(NMI, kNarrow), kSlab = 32 * NMI * kTlRowBytes, kWait = tl_wait(tl_younger(NMI, kNarrow));
    uint32_t off[NMI];
#pragma unroll
    for (int it = 0; it < NMI; ++it) off[it] = doff[it];
    auto stage_slab = [&](int slab, int buf) __attribute__((always_inline)) {
      const uint8_t* sb = abase + static_cast<size_t>(slab) * kF8Block;
#pragma unroll
      for (int it = 0; it < NMI; ++it) {
        const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_base + buf * kSlab + (wave * NMI + it) * 1024);
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off[it]), "s"(sb), "s"(dst)
                     : "memory", "m0");
      }
    };
    i32x4 wfrag[S][2][NG];   // [stage][k half][16-row group]
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int st = 0; st < S; ++st) stage_slab(min(st, nk - 1), st);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int st = 0; st < S; ++st)
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int h = 0; h < 2; ++h) wfrag[st][h][g] = wload(g, min(st, nk - 1), h);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(kWait);
    __syncthreads();

    vf32x4 acc[NMT][NG];
#pragma unroll
    for (int mt = 0; mt < NMT; ++mt)
#pragma unroll
      for (int g = 0; g < NG; ++g) acc[mt][g] = vf32x4{0.f, 0.f, 0.f, 0.f};

    // fragment of lane (r, q), tile mt, half h: row 16*mt + r, position (q + 4h) ^ f(r)
    const int fsw = ((fr >> 1) & 7) ^ ((fr & 1) << 2);
    const int a_row = fr * kTlRowBytes, a_x = (fq ^ fsw) << 4;
    int cur = 0, ahead = S;   // buffer of slab kt, buffer of slab kt+S
    // tail_c: -1 in the loop, else the number of the slab behind it (whose stage has the same number)
    auto slab = [&](auto stage_c, auto tail_c, int kt) {
      constexpr int st = decltype(stage_c)::value, kTail = decltype(tail_c)::value;
      constexpr int NP = NMT / 2;                 // pairs of 16-row tiles
      const int kts = min(kt + S, nk - 1);
      const uint8_t* la = lds + cur * kSlab + a_row;
      const uint2 sb = *reinterpret_cast<const uint2*>(s_scales + kt * kPfBM + fr * 8);
      const float2 sw = *reinterpret_cast<const float2*>(s_scales + nk * kPfBM + kt * 8);
      const float w = kNarrow || wave < 2 ? sw.x : sw.y;
      i32x4 fa[2][2][2];   // [parity][tile of the pair][half]
      if (NP == 1 && kTail < 0) {       // the copies go first, so that every height issues vector memory in the counted order
        stage_slab(kts, ahead);
        __builtin_amdgcn_sched_barrier(0);
      }
      auto rd = [&](int pr, i32x4 (&f)[2][2]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            f[i][h] = *reinterpret_cast<const i32x4*>(la + (2 * pr + i) * 16 * kTlRowBytes + (a_x ^ (h << 6)));
      };
      auto mul = [&](auto mt_c, auto g_c, const i32x4 (&f)[2]) __attribute__((always_inline)) {
        constexpr int mt = decltype(mt_c)::value, g = decltype(g_c)::value;
        const int sbv = static_cast<int>(mt < 4 ? sb.x : sb.y);
        const i32x8 wf = f8_join(wfrag[st][0][g], wfrag[st][1][g]), xf = f8_join(f[0], f[1]);
        if constexpr (kPow2) {
          acc[mt][g] = f8_mfma<0, mt & 3>(wf, xf, acc[mt][g], static_cast<int>(__float_as_uint(w) >> 23), sbv);
        } else {
          const vf32x4 part = f8_mfma<0, mt & 3>(wf, xf, vf32x4{0.f, 0.f, 0.f, 0.f}, kF8One, sbv);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[mt][g][j] = fmaf(part[j], w, acc[mt][g][j]);
        }
      };
      rd(0, fa[0]);
      auto pair = [&](auto pr_c) __attribute__((always_inline)) {
        constexpr int pr = decltype(pr_c)::value;
        if constexpr (pr < NP) {
          if (pr + 1 < NP) rd(pr + 1, fa[(pr + 1) & 1]);
          __builtin_amdgcn_sched_barrier(0);    // the next pair's reads stay ahead of this pair's products
          auto group = [&](auto g_c) __attribute__((always_inline)) {
            constexpr int g = decltype(g_c)::value;
            mul(std::integral_constant<int, 2 * pr>{}, g_c, fa[pr & 1][0]);
            mul(std::integral_constant<int, 2 * pr + 1>{}, g_c, fa[pr & 1][1]);
            if constexpr (pr == NP - 1 && kTail < 0) {       // last user of group g's fragments: request those of slab kt+S
              __builtin_amdgcn_sched_barrier(0);
#pragma unroll
              for (int h = 0; h < 2; ++h) wfrag[st][h][g] = wload(g, kts, h);
              __builtin_amdgcn_sched_barrier(0);
            }
          };
          group(std::integral_constant<int, 0>{});
          group(std::integral_constant<int, 1>{});
          if constexpr (NG > 2) {
            group(std::integral_constant<int, 2>{});
            group(std::integral_constant<int, 3>{});
          }
          __builtin_amdgcn_sched_barrier(0);
          if (NP > 1 && pr == 0 && kTail < 0) {   // the copies of slab kt+S go out once the matrix pipe has work
            stage_slab(kts, ahead);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      };
      pair(std::integral_constant<int, 0>{});
      pair(std::integral_constant<int, 1>{});
      pair(std::integral_constant<int, 2>{});
      pair(std::integral_constant<int, 3>{});
      __builtin_amdgcn_s_waitcnt(kTail < 0 ? kWait : tl_wait(tl_younger_tail(NMI, kNarrow, kTail < 0 ? 0 : kTail)));
      __syncthreads();
      cur = (cur == S) ? 0 : cur + 1;
      ahead = (ahead == S) ? 0 : ahead + 1;
    };
    int kt = 0;
    auto turn = [&](auto st_c) __attribute__((always_inline)) {
      if constexpr (decltype(st_c)::value < S) slab(st_c, std::integral_constant<int, -1>{}, kt + decltype(st_c)::value);
    };
    for (; kt + S <= nk; kt += S) {
      turn(std::integral_constant<int, 0>{});
      turn(std::integral_constant<int, 1>{});
      turn(std::integral_constant<int, 2>{});
      turn(std::integral_constant<int, 3>{});
      turn(std::integral_constant<int, 4>{});
      turn(std::integral_constant<int, 5>{});
    }
    auto tail = [&](auto st_c) __attribute__((always_inline)) {
      if constexpr (decltype(st_c)::value < S - 1)
        if (kt + decltype(st_c)::value < nk) slab(st_c, st_c, kt + decltype(st_c)::value);
    };
    tail(std::integral_constant<int, 0>{});
    tail(std::integral_constant<int, 1>{});
    tail(std::integral_constant<int, 2>{});
    tail(std::integral_constant<int, 3>{});
    tail(std::integral_constant<int, 4>{});
    __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);  // no copy may land in LDS after the epilogue starts to reuse it
    __syncthreads();

    // ---- epilogue ----------------------------------------------------------------
    // The product was formed as W * X^T: a lane holds row m = 16*mt + fr and, per 16-row weight group, four
    // consecutive output columns 4*fq + j.
    // 16-bit rows times their factor, staged per wavefront in two 32-column passes into 16-byte stores
    uint8_t* st = lds + wave * (kRows * 64);
    uint16_t* out = static_cast<uint16_t*>(dense ? a.p.out_s : a.p.out_r);
    // whole 16-byte stores need rows that start on 16-byte boundaries
    const bool whole = N % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
#pragma unroll
    for (int pass = 0; pass < NG / 2; ++pass) {
      if (pass) __syncthreads();  // staging rows are reused
#pragma unroll
      for (int mt = 0; mt < NMT; ++mt) {
        const int m = mt * 16 + fr;
        const float sc = s_row[m];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const vf32x4 v = acc[mt][2 * pass + p];
          uint2 pk;
          pk.x = F::pack2(v[0] * sc, v[1] * sc);
          pk.y = F::pack2(v[2] * sc, v[3] * sc);
          const int chunk = (2 * p + (fq >> 1)) ^ ((m >> 1) & 3);
          *reinterpret_cast<uint2*>(st + m * 64 + chunk * 16 + (fq & 1) * 8) = pk;
        }
      }
      __syncthreads();
      const int ncol0 = n0 + wave * 16 * NG + pass * 32;
#pragma unroll
      for (int it = 0; it < 2 * NMI; ++it) {
        const int m = it * 16 + (lane >> 2), q = lane & 3;
        const uint4 val = *reinterpret_cast<const uint4*>(st + m * 64 + (q ^ ((m >> 1) & 3)) * 16);
        const int n = ncol0 + q * 8;
        if (m >= M || n >= N) continue;
        uint16_t* o = out + static_cast<size_t>(r0 + m) * N + n;
        if (whole) {
          *reinterpret_cast<uint4*>(o) = val;
        } else {
          const uint32_t v[4] = {val.x, val.y, val.z, val.w};
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (n + j < N) o[j] = static_cast<uint16_t>(v[j >> 1] >> (16 * (j & 1)));
        }
      }
    }
  };
  auto bodies = [&](auto pow2_c) __attribute__((always_inline)) {
    if constexpr (kNarrow) body(std::integral_constant<int, 1>{}, pow2_c);
    else switch (nmi) {
      case 1: body(std::integral_constant<int, 1>{}, pow2_c); break;
      case 2: body(std::integral_constant<int, 2>{}, pow2_c); break;
      case 3: body(std::integral_constant<int, 3>{}, pow2_c); break;
      default: body(std::integral_constant<int, 4>{}, pow2_c); break;
    }
  };
  if (pow2) bodies(std::true_type{});
  else bodies(std::false_type{});
}

template <bool kNarrow>
static int launch_tile(const TileArgs& a, int64_t grid, hipStream_t st) {
  SP_REQUIRE(grid < (1ll << 31), "fp8 product: grid too large");
  const int Kmax = a.p.Ks > a.p.Kr ? a.p.Ks : a.p.Kr;
  const unsigned dyn = static_cast<unsigned>(f8_blocks(Kmax)) * kTlScaleBytes;
  if (a.p.dtype == SPARSE_HIP_F16)
    hipLaunchKernelGGL((f8_tile_kernel<Fp16, kNarrow>), dim3(static_cast<unsigned>(grid)), dim3(kPfThreads), dyn, st, a);
  else
    hipLaunchKernelGGL((f8_tile_kernel<Bf16, kNarrow>), dim3(static_cast<unsigned>(grid)), dim3(kPfThreads), dyn, st, a);
  SP_LAUNCH_CHECK("f8_tile_kernel");
  return SPARSE_HIP_OK;
}

int f8_tile_columns(int tile_rows) { return tile_rows <= kTlNarrowRows ? kPfBR / 2 : kPfBR; }

int f8_tile_down(const F8Product& p, const PfQueues& q, int tile_rows, hipStream_t st) {
  TileArgs a = {};
  a.p = p;
  a.map = q.map_dn;
  a.qhdr = q.hdr + 16;
  return tile_rows <= kTlNarrowRows ? launch_tile<true>(a, tl_queue_grid(q.cap_dn), st)
                                    : launch_tile<false>(a, tl_queue_grid(q.cap_dn), st);
}

int f8_tile_linear(const F8Product& p, int tile_rows, hipStream_t st) {
  TileArgs a = {};
  a.p = p;
  a.rows = tile_rows;
  a.mt = (p.T + tile_rows - 1) / tile_rows;
  const int columns = f8_tile_columns(tile_rows);
  a.nt = (p.Ns + columns - 1) / columns;
  const int64_t total = static_cast<int64_t>(a.mt) * a.nt;
  SP_REQUIRE(total < (1ll << 30), "fp8_linear: too many tiles");
  const int64_t grid = (total + kPfXcds - 1) / kPfXcds * kPfXcds;
  return tile_rows <= kTlNarrowRows ? launch_tile<true>(a, grid, st) : launch_tile<false>(a, grid, st);
}

}  // namespace sparse
