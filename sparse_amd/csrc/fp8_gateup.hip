// Gate and up projections of many rows on block-scaled 8-bit weights, and the quantised intermediate: tiles.
//
//   h[m, n] = Q(silu(g[m, n]) u[m, n]),   g, u = sum over blocks b of s(n, b) sum over k in b of x[m, k] w[n, k]
//   x: rows that the quantiser has rounded to 8 bits, its scale included, held in bf16
//
// The products are taken in bf16 and added in fp32, four 16x16x32 matrix instructions per 16 x 16 tile and 128-wide
// slab.  The 8-bit instruction would be half as many cycles, but cuts products off 13 bits below the largest of eight,
// and as h is rounded to 8 bits next, some of it then lands on the other side of a rounding border: rows of the whole FFN
// were 0.0012 off the 64-bit formula instead of 0.0002 (norm of the error over norm; fp16, 301 tokens, 3 of 16 experts of
// 704 x 1024), 0.0025 instead of 0.0017 (bf16, the call below), where calls of fewer tokens, which add in fp32, have
// the smaller figures.
//
// A workgroup of four wavefronts computes up to 128 rows x 128 neurons (128 gate rows and the 128 up rows of the same
// neurons) over 128-wide k slabs.  Rows come from the quantiser as bf16 (times half their scale, 2^-121 to 2^119, which
// bf16 holds exactly), so that they are widened once and not by every wavefront of every tile: a conversion of two values
// takes eight cycles, and the launch below took 345 us.  They go to an LDS ring by direct global -> LDS copies, gathered
// through the permutation, their 16-byte chunks swizzled by row.  Weight fragments come straight from the tiled layout
// into registers and are widened there, half a slab at a time, times their scale where all scales of the tile are powers
// of two; otherwise the fp32 scales multiply each half slab's sum on its way into the accumulator.  A tile looks at its
// scales and chooses by itself: what a row comes out as depends on its own weights' scales alone, as they are at the
// time of the call.
//
// The epilogue is the quantiser: a tile's 128 neurons are one run of the intermediate, its largest magnitude is found
// across the four wavefronts in LDS, and 8-bit rows with their scales leave.
//
// 4096 tokens, 6 of 64 experts of 1408 x 2048, shared 2816, 378 GFLOP: 311 us, 1.2 PFLOP/s (a library
// bf16 product of 8192^3 reaches 1.5).  The matrix pipes are busy for 61 % of the cycles in which compute units have
// work.  Requesting weights two slabs ahead, for which no more than a quarter slab can be held widened, takes 2 % off
// and was left out; reading rows two or three steps ahead takes nothing.
#include <type_traits>

#include "fp8_tile.h"

namespace sparse {

constexpr int kGuRowBytes = 2 * kF8Block;           // LDS row of one k slab
constexpr int kGuRing = 2 * kPfBM * kGuRowBytes;
constexpr int kGuCopyRows = 1024 / kGuRowBytes;     // rows that one copy of a wavefront brings

// A tile of 32 NMI rows keeps S slabs of weight fragments in registers and S + 1 slabs of rows in LDS.
constexpr int gu_depth(int nmi) { return nmi == 1 ? 4 : nmi == 2 ? 3 : 1; }
// "The copies of the next slab have landed": they were followed by their own slab's 8 fragment loads and by 2 NMI copies
// and 8 loads for each slab requested since, S - 1 of them in the loop, S - 2 - j in slab number j behind it, where
// nothing is requested any more.
constexpr int gu_younger(int nmi, int j) { return 8 + (gu_depth(nmi) - 2 - j) * (2 * nmi + 8); }
static_assert(gu_younger(1, -1) < 64 && gu_younger(2, -1) < 64, "six bits");
static_assert((gu_depth(1) + 1) * 32 * kGuRowBytes <= kGuRing && (gu_depth(2) + 1) * 64 * kGuRowBytes <= kGuRing &&
              (gu_depth(3) + 1) * 96 * kGuRowBytes <= kGuRing && (gu_depth(4) + 1) * 128 * kGuRowBytes <= kGuRing, "rings fit");

__global__ __launch_bounds__(kPfThreads, 2) void f8_gateup_kernel(const TileArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kGuRing];
  __shared__ float s_amax[4][kPfBM];
  extern __shared__ __attribute__((aligned(16))) float s_scales[];   // [nk] gate's and up's

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int fr = lane & 15, fq = lane >> 4;
  const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) uint8_t*)(&lds[0])));

  int slot, r0, M, bn;
  if (!tl_queued(a, slot, r0, M, bn)) return;
  const bool dense = slot < 0;
  const int Kdim = dense ? a.p.Ks : a.p.Kr, N = dense ? a.p.Ns : a.p.Nr;
  const int nk = (Kdim + kF8Block - 1) / kF8Block;
  const int n0 = bn * (kPfBR / 2);                    // first neuron of this tile

  // ---- rows -------------------------------------------------------------------------------
  // A slab row is 16 chunks of 16 bytes: lane quarter q multiplies k = 32 q + 8 e + (0 .. 7), e = 0 .. 3, chunk 4 q + e in
  // memory.  In LDS, row r keeps it at position (q + 4 e) ^ (r % 16): the lanes that a wide read serves together are of
  // two quarters, eight rows each, and so lie in different banks (with 4 q + e instead, conflicts take a sixth of the cycles).
  // A lane of copy `it` of wavefront w brings row 4 (w NC + it) + lane / 16, position lane % 16.
  const int nmi = (M + 31) >> 5;
  const uint8_t* rows = dense ? a.p.act_s : a.p.act_r;
  auto source = [&](int m) -> const uint8_t* {        // the lane's chunk of a row in slab 0
    const int mm = min(m, M - 1);                     // (rows past the end repeat the last and are not stored)
    uint32_t t = static_cast<uint32_t>(r0 + mm);
    if (!dense) {
      t = static_cast<uint32_t>(a.p.perm[r0 + mm]);
      if (a.topk_magic != 0) t = __umulhi(t, a.topk_magic);
    }
    const int c = (lane & 15) ^ (m & 15);
    return rows + static_cast<size_t>(t) * nk * kGuRowBytes + (((c & 3) << 2 | c >> 2) << 4);
  };
  const uint8_t* src[8];
#pragma unroll
  for (int it = 0; it < 8; ++it) src[it] = source((wave * 2 * nmi + it) * kGuCopyRows + fq);

  // ---- weights ----------------------------------------------------------------------------
  // The wavefront's 64 weight rows are four 16-row groups: 0, 1 gate rows of 32 neurons, 2, 3 the up rows of the same
  // neurons; a group's slab is 2 KB, its two halves 1 KB each in lane order.
  const uint8_t *w0 = a.p.w0, *w1 = a.p.w1;
  const float *s0 = a.p.s0, *s1 = a.p.s1;
  if (!dense) {
    const uint8_t* base = a.p.slab + static_cast<uint64_t>(slot) * a.p.slot_stride;
    w0 = base + a.p.off0;
    w1 = base + a.p.off1;
    s0 = reinterpret_cast<const float*>(base + a.p.soff0);
    s1 = reinterpret_cast<const float*>(base + a.p.soff1);
  }
  const uint8_t* wbase[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int n = min(n0 + wave * 32 + (g & 1) * 16, ((N + 15) & ~15) - 16);
    wbase[g] = uniform_ptr((g >= 2 ? w1 : w0) + static_cast<size_t>(n >> 4) * nk * kF8TileBytes);
  }
  typedef const __attribute__((address_space(1))) char* gptr_t;
  const uint32_t woff = lane * 16;
  auto wload = [&](int g, int slab, int h) __attribute__((always_inline)) {
    gptr_t p = (gptr_t)(reinterpret_cast<uintptr_t>(wbase[g]) + static_cast<size_t>(slab) * kF8TileBytes + h * 1024);
    return *reinterpret_cast<const __attribute__((address_space(1))) i32x4*>(p + woff);
  };

  // Every wavefront looks at all scales of the tile and stores a quarter of them.
  s0 += static_cast<size_t>(bn) * nk;
  s1 += static_cast<size_t>(bn) * nk;
  bool odd = false;
  for (int i = lane; i < 2 * nk; i += 64) {
    const float v = ((i & 1) ? s1 : s0)[i >> 1];
    if (((i >> 6) & 3) == wave) s_scales[i] = v;
    odd |= !tl_is_exponent<-121, 119>(v);
  }
  const bool pow2 = !__any(odd) && a.p.pow2 != 0;

  // The tile's rows are processed in sub-tiles of 32; a segment's last tile is specialised on how many of them hold rows.
  // kPow2: the scales are folded into the widening of the weights.
  auto body = [&](auto nmi_c, auto pow2_c) __attribute__((always_inline)) {
    constexpr int NMI = decltype(nmi_c)::value, NMT = 2 * NMI, NC = 2 * NMI;   // 16-row tiles, copies of a wavefront
    constexpr bool kPow2 = decltype(pow2_c)::value;
    // While slab kt is multiplied, the rows of slab kt+S travel to the LDS buffer slab kt-1 has left and the
    // fragments of slab kt+S to the registers their widening has freed.  Vector memory retires in order, so what has
    // landed is known by counting.  Slabs past the end refetch the last one; the up to S - 1 slabs behind the loop find
    // everything requested.
    constexpr int S = gu_depth(NMI), kSlab = 32 * NMI * kGuRowBytes;
    const uint8_t* from[NC];
#pragma unroll
    for (int it = 0; it < NC; ++it) from[it] = src[it];
    auto stage_slab = [&](int slab, int buf) __attribute__((always_inline)) {
#pragma unroll
      for (int it = 0; it < NC; ++it) {
        const uint8_t* p = from[it] + static_cast<size_t>(slab) * kGuRowBytes;
        const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_base + buf * kSlab + (wave * NC + it) * 1024);
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(dst) : "memory", "m0");
      }
    };
    i32x4 wfrag[S][2][4];    // [stage][k half][16-row group]
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int st = 0; st < S; ++st) stage_slab(min(st, nk - 1), st);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int st = 0; st < S; ++st)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int g = 0; g < 4; ++g) wfrag[st][h][g] = wload(g, min(st, nk - 1), h);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(tl_wait(gu_younger(NMI, -1)));
    __syncthreads();

    vf32x4 acc[NMT][4];
#pragma unroll
    for (int mt = 0; mt < NMT; ++mt)
#pragma unroll
      for (int g = 0; g < 4; ++g) acc[mt][g] = vf32x4{0.f, 0.f, 0.f, 0.f};

    const int a_row = fr * kGuRowBytes, a_x = (fq ^ fr) << 4;
    int cur = 0, ahead = S;   // buffer of slab kt, buffer of slab kt+S
    // tail_c: -1 in the loop, else the number of the slab behind it (whose stage has the same number)
    auto slab = [&](auto stage_c, auto tail_c, int kt) __attribute__((always_inline)) {
      constexpr int st = decltype(stage_c)::value, kTail = decltype(tail_c)::value;
      const int kts = min(kt + S, nk - 1);
      const uint8_t* la = lds + cur * kSlab + a_row;
      const float2 sw = *reinterpret_cast<const float2*>(s_scales + 2 * kt);
      if (kTail < 0) stage_slab(kts, ahead);
      __builtin_amdgcn_sched_barrier(0);
      // steps of half a slab of one 16-row tile
      bf16x8 x[2][2];
      auto rd = [&](int step, bf16x8 (&f)[2]) __attribute__((always_inline)) {
        const int h = step / NMT, mt = step % NMT;
#pragma unroll
        for (int p = 0; p < 2; ++p)
          f[p] = *reinterpret_cast<const bf16x8*>(la + mt * 16 * kGuRowBytes + (a_x ^ ((h * 2 + p) << 6)));
      };
      rd(0, x[0]);
      bf16x8 w[4][2];
#pragma unroll
      for (int step = 0; step < 2 * NMT; ++step) {
        const int h = step / NMT, mt = step % NMT;
        if (mt == 0) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float sc = kPow2 ? (g < 2 ? sw.x : sw.y) : 1.f;
            w[g][0] = f8_widen8(wfrag[st][h][g][0], wfrag[st][h][g][1], sc);
            w[g][1] = f8_widen8(wfrag[st][h][g][2], wfrag[st][h][g][3], sc);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (kTail < 0) {             // their last user: request those of slab kt+S
#pragma unroll
            for (int g = 0; g < 4; ++g) wfrag[st][h][g] = wload(g, kts, h);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        if (step + 1 < 2 * NMT) rd(step + 1, x[(step + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);    // the next step's reads stay ahead of this step's products
        const bf16x8(&xf)[2] = x[step & 1];
        vf32x4 part[4];
#pragma unroll
        for (int g = 0; g < 4; ++g)
          part[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[g][0], xf[0], kPow2 ? acc[mt][g] : vf32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          part[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[g][1], xf[1], part[g], 0, 0, 0);
          if (kPow2) acc[mt][g] = part[g];
        }
        if (!kPow2) {
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[mt][g][j] = fmaf(part[g][j], g < 2 ? sw.x : sw.y, acc[mt][g][j]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_waitcnt(tl_wait(gu_younger(NMI, kTail)));
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
    }
    auto tail = [&](auto st_c) __attribute__((always_inline)) {
      if constexpr (decltype(st_c)::value < S - 1)
        if (kt + decltype(st_c)::value < nk) slab(st_c, st_c, kt + decltype(st_c)::value);
    };
    tail(std::integral_constant<int, 0>{});
    tail(std::integral_constant<int, 1>{});
    tail(std::integral_constant<int, 2>{});
    __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);  // no copy may land in LDS after the epilogue starts to reuse it
    __syncthreads();

    // ---- epilogue ----------------------------------------------------------------
    // The product was formed as W * X^T: a lane holds row m = 16*mt + fr and, per 16-row weight group, four
    // consecutive neurons 4*fq + j.  SwiGLU (rows came with half their scale), then the row's largest magnitude over
    // the tile's 128 neurons: over a lane's values, its row's four lanes, the four wavefronts.
#pragma unroll
    for (int mt = 0; mt < NMT; ++mt) {
      float m = 0.f;
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float h = silu_f32(2.f * acc[mt][p][j]) * (2.f * acc[mt][2 + p][j]);
          acc[mt][p][j] = n0 + wave * 32 + p * 16 < N ? h : 0.f;   // columns behind the matrix's end (a multiple of 16)
          m = fmaxf(m, f8_magnitude(acc[mt][p][j]));
        }
      m = fmaxf(m, __shfl_xor(m, 16));
      m = fmaxf(m, __shfl_xor(m, 32));
      if (fq == 0) s_amax[wave][mt * 16 + fr] = m;
    }
    __syncthreads();
    uint8_t* st = lds;             // 128 rows x 128 bytes, 16-byte chunks swizzled by row
#pragma unroll
    for (int mt = 0; mt < NMT; ++mt) {
      const int m = mt * 16 + fr;
      const float top = fmaxf(fmaxf(s_amax[0][m], s_amax[1][m]), fmaxf(s_amax[2][m], s_amax[3][m]));
      const float inv = f8_inverse(f8_exponent(top));
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int chunk = (wave * 2 + p) ^ (m & 7);
        *reinterpret_cast<uint32_t*>(st + m * 128 + chunk * 16 + fq * 4) =
            f8_pack4(acc[mt][p][0] * inv, acc[mt][p][1] * inv, acc[mt][p][2] * inv, acc[mt][p][3] * inv);
      }
    }
    __syncthreads();
    const int nb = (N + kF8Block - 1) / kF8Block;
    uint8_t* out = dense ? a.q_s : a.q_r;
    uint8_t* outs = dense ? a.qs_s : a.qs_r;
#pragma unroll
    for (int it = 0; it < NMI; ++it) {
      const int m = it * 32 + (tid >> 3), c = tid & 7;
      const i32x4 v = *reinterpret_cast<const i32x4*>(st + m * 128 + (c ^ (m & 7)) * 16);
      if (m < M) *reinterpret_cast<i32x4*>(out + (static_cast<size_t>(r0 + m) * nb + bn) * kF8Block + c * 16) = v;
    }
    if (tid < M) {
      const float top = fmaxf(fmaxf(s_amax[0][tid], s_amax[1][tid]), fmaxf(s_amax[2][tid], s_amax[3][tid]));
      outs[static_cast<size_t>(r0 + tid) * nb + bn] = static_cast<uint8_t>(f8_exponent(top) + kF8Bias);
    }
  };
  auto bodies = [&](auto pow2_c) __attribute__((always_inline)) {
    switch (nmi) {
      case 1: body(std::integral_constant<int, 1>{}, pow2_c); break;
      case 2: body(std::integral_constant<int, 2>{}, pow2_c); break;
      case 3: body(std::integral_constant<int, 3>{}, pow2_c); break;
      default: body(std::integral_constant<int, 4>{}, pow2_c); break;
    }
  };
  if (pow2) bodies(std::true_type{});
  else bodies(std::false_type{});
}

int f8_tile_gateup(const F8Product& p, const PfQueues& q, void* h, void* hs, void* sh, void* shs, hipStream_t st) {
  TileArgs a = {};
  a.p = p;
  a.map = q.map_gu;
  a.qhdr = q.hdr;
  a.topk_magic = tl_magic(p.topk);
  a.q_r = static_cast<uint8_t*>(h);
  a.qs_r = static_cast<uint8_t*>(hs);
  a.q_s = static_cast<uint8_t*>(sh);
  a.qs_s = static_cast<uint8_t*>(shs);
  const int64_t grid = tl_queue_grid(q.cap_gu);
  SP_REQUIRE(grid < (1ll << 31), "fp8 product: grid too large");
  const unsigned dyn = static_cast<unsigned>(f8_blocks(p.Ks > p.Kr ? p.Ks : p.Kr)) * 2 * sizeof(float);
  hipLaunchKernelGGL(f8_gateup_kernel, dim3(static_cast<unsigned>(grid)), dim3(kPfThreads), dyn, st, a);
  SP_LAUNCH_CHECK("f8_gateup_kernel");
  return SPARSE_HIP_OK;
}

}  // namespace sparse
