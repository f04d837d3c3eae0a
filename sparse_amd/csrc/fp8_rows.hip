// Block-scaled 8-bit matrix products of three to a few dozen rows that are 8-bit already: weights and rows both
// go straight from memory to registers.
//
//   y[m, n] = sum over blocks b of 2^e(m, b) s(n, b) sum over k in b of x[m, k] w[n, k]
//
// What bounds it is the weights' way from HBM.  A workgroup owns 16 output columns of two matrices (gate and up
// of one expert) or of one, and up to 16 NTmax rows of a segment.  Its wavefronts, four or, for a single matrix of
// long rows, eight (kF8LongBlocks), deal the 128-wide k blocks among themselves, one block a register stage, two stages in flight: that leaves registers for four to five
// wavefronts on a SIMD, whose loads together keep HBM busy (two blocks a stage: down of 8 tokens 15.6 us instead
// of 14.4; two column groups a workgroup: 23).  Rows are read from L2 by every workgroup of their segment, in the
// matrix instruction's own layout: no LDS and no barrier before the wavefronts' sums meet.  Quantising the rows
// in here instead of in a launch before (fp8_few.hip does) repeats that work in every workgroup: 24.4 + 14.4 us
// become 30.4 + 33.1.
//
// Gate and up are products of the values widened to bf16, added in fp32, as their result is rounded to 8 bits next
// and the 8-bit instruction's cut-off would move values across rounding borders; the matrix cycles are hidden
// behind the loads.  Down and single products, rounded to 16 bits, take the 8-bit instruction with the rows'
// scales as its operand.
//
// 8 tokens of 4 among 60 experts of 1408 x 2048 and a shared one of 5632: gate/up 170 MB in 24.4 us (7.0 TB/s),
// down 85 MB in 14 us (6.1 TB/s).  From some 64 rows on the tile kernel is faster (fp8.hip has both sides).
#include <type_traits>

#include "fp8.h"

namespace sparse {

// NTmax: 16-row groups at most; a segment takes the form of the groups it has.
// kRwWaves: wavefronts of a workgroup
template <typename F, bool kGateUp, int NTmax, int kRwWaves>
__global__ __launch_bounds__(kRwWaves * 64) void f8_rows_kernel(const F8Product a, int tiles_r, int tiles_s) {
  constexpr int NM = kGateUp ? 2 : 1;
  __shared__ vf32x4 red[kRwWaves][NTmax * NM][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 15, q = lane >> 4;
  F8Where own;
  if (!f8_where(a, blockIdx.x, tiles_r, tiles_s, own)) return;
  const bool dense = own.dense;
  const int nb = own.nb, N = own.N, n0 = own.n0;
  const uint8_t* wp[NM];
  const float* sp[NM];
#pragma unroll
  for (int mi = 0; mi < NM; ++mi) {
    wp[mi] = (mi ? own.w1 : own.w0) + lane * 16;
    sp[mi] = mi ? own.s1 : own.s0;
  }
  const int m0 = blockIdx.y * 16 * NTmax, M = min(own.rows() - m0, 16 * NTmax), r0 = own.first_row() + m0;
  if ((NTmax > 1 || blockIdx.y > 0) && M <= 0) return;
  auto body = [&](auto nt_c) __attribute__((always_inline)) {
  constexpr int NT = decltype(nt_c)::value;
  vf32x4 acc[NM][NT];
#pragma unroll
  for (int mi = 0; mi < NM; ++mi)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[mi][nt] = vf32x4{0.f, 0.f, 0.f, 0.f};

  struct Stage {
    i32x4 w[NM][2], x[NT][2];
    int xs[NT];
    float ws[NM];
  };
  auto load_weights = [&](Stage& st, int i) __attribute__((always_inline)) {   // the wavefront's block number i (past the end: the last)
    const int kb = min(wave + i * kRwWaves, nb - 1);
#pragma unroll
    for (int mi = 0; mi < NM; ++mi) {
      const uint8_t* p = wp[mi] + static_cast<size_t>(kb) * kF8TileBytes;
      st.w[mi][0] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(p));
      st.w[mi][1] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(p + 1024));
    }
  };
  auto load_scales = [&](Stage& st, int i) __attribute__((always_inline)) {
    const int kb = min(wave + i * kRwWaves, nb - 1);
#pragma unroll
    for (int mi = 0; mi < NM; ++mi) st.ws[mi] = sp[mi][kb];
  };
  const uint8_t *xp[NT], *xs[NT];
  auto load_rows = [&](Stage& st, int i) __attribute__((always_inline)) {
    const int kb = min(wave + i * kRwWaves, nb - 1);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint8_t* p = xp[nt] + kb * kF8Block;
      st.x[nt][0] = *reinterpret_cast<const i32x4*>(p);
      st.x[nt][1] = *reinterpret_cast<const i32x4*>(p + 16);
      st.xs[nt] = xs[nt][kb];
    }
  };
  auto load = [&](Stage& st, int i) __attribute__((always_inline)) {
    load_weights(st, i);
    load_rows(st, i);
    load_scales(st, i);
  };
  auto use = [&](const Stage& st) __attribute__((always_inline)) {
    if constexpr (kGateUp) {
      F8Wide x[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) x[nt] = f8_widen(st.x[nt][0], st.x[nt][1]);
#pragma unroll
      for (int mi = 0; mi < NM; ++mi) {
        const F8Wide w = f8_widen(st.w[mi][0], st.w[mi][1]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const vf32x4 part = f8_mfma_wide(w, x[nt]);
          const float scale = __uint_as_float(static_cast<uint32_t>(st.xs[nt]) << 23);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[mi][nt][j] = fmaf(part[j] * scale, st.ws[mi], acc[mi][nt][j]);
        }
      }
    } else {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const vf32x4 part = f8_mfma<0, 0>(f8_join(st.w[0][0], st.w[0][1]), f8_join(st.x[nt][0], st.x[nt][1]),
                                          vf32x4{0.f, 0.f, 0.f, 0.f}, kF8One, st.xs[nt]);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[0][nt][j] = fmaf(part[j], st.ws[0], acc[0][nt][j]);
      }
    }
  };
  const int n = (nb - wave + kRwWaves - 1) / kRwWaves;     // blocks of this wavefront
  // The first weights go out before anything that waits for the segment's rows.
  Stage a0, a1;
  load_weights(a0, 0);
  __builtin_amdgcn_sched_barrier(0);
  if (M <= 0) return;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    size_t row = r0 + min(nt * 16 + r, M - 1);   // rows past the end repeat the last and are not stored
    if (own.perm != nullptr) row = static_cast<uint32_t>(own.perm[row]) / static_cast<uint32_t>(own.topk);
    xp[nt] = own.act + row * nb * kF8Block + q * 32;
    xs[nt] = own.acts + row * nb;
  }
  load_rows(a0, 0);
  load_scales(a0, 0);
  __builtin_amdgcn_sched_barrier(0);
  load(a1, 1);
  __builtin_amdgcn_sched_barrier(0);
  const int my_m = wave * 16 + r;                // wavefront nt stores row group nt
  float factor = 1.f;
  if (!kGateUp && wave < NT && my_m < M) {
    if (!dense) factor = F::from_bits(static_cast<const uint16_t*>(a.topv)[a.perm[r0 + my_m]]);
    else if (a.gate_s != nullptr) factor = F::from_bits(static_cast<const uint16_t*>(a.gate_s)[r0 + my_m]);
  }
  __builtin_amdgcn_sched_barrier(0);
  int c = 0;
  for (; c + 4 <= n; c += 2) {           // (no branch in here: the waits count what is in flight)
    use(a0);
    __builtin_amdgcn_sched_barrier(0);
    load(a0, c + 2);
    __builtin_amdgcn_sched_barrier(0);
    use(a1);
    __builtin_amdgcn_sched_barrier(0);
    load(a1, c + 3);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (c < n) use(a0);                    // up to three blocks are left
  if (c + 2 < n) load(a0, c + 2);
  if (c + 1 < n) use(a1);
  if (c + 2 < n) use(a0);

  // ---- the wavefronts' sums meet in LDS ------------------------------------------------------
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mi = 0; mi < NM; ++mi) red[wave][nt * NM + mi][lane] = acc[mi][nt];
  __syncthreads();
  auto sum = [&](int f) {
    vf32x4 v = red[0][f][lane];
#pragma unroll
    for (int w = 1; w < kRwWaves; ++w) v += red[w][f][lane];
    return v;
  };
  if (wave >= NT || my_m >= M) return;
  const int col = n0 + q * 4;
  const size_t at = static_cast<size_t>(r0 + my_m) * N + col;
  if (kGateUp) {
    const vf32x4 g = sum(wave * NM), u = sum(wave * NM + NM - 1);
    vf32x4 h;
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = silu_f32(g[j]) * u[j];
    *reinterpret_cast<vf32x4*>(static_cast<float*>(dense ? a.out_s : a.out_r) + at) = h;
  } else if (col < N) {
    const float sc = dense && a.gate_s != nullptr ? sigmoid_f32(factor) : factor;
    f8_store4<F>(static_cast<uint16_t*>(dense ? a.out_s : a.out_r) + at, sum(wave), sc, N, col);
  }
  };
  if (NTmax == 1 || M <= 16) body(std::integral_constant<int, 1>{});
  else body(std::integral_constant<int, NTmax>{});
}

template <typename F, bool kGateUp, int NT, int W>
static int launch_rows(const F8Product& p, int tiles_r, int tiles_s, hipStream_t st) {
  const int64_t grid = tiles_s + static_cast<int64_t>(tiles_r) * p.segs.n;
  const int64_t groups = (p.T + 16 * NT - 1) / (16 * NT);
  if (grid == 0) return SPARSE_HIP_OK;
  SP_REQUIRE(grid < (1ll << 31) && groups < 65536, "fp8 product: grid too large");
  hipLaunchKernelGGL((f8_rows_kernel<F, kGateUp, NT, W>), dim3(static_cast<unsigned>(grid), static_cast<unsigned>(groups)),
                     dim3(W * 64), 0, st, p, tiles_r, tiles_s);
  SP_LAUNCH_CHECK("f8_rows_kernel");
  return SPARSE_HIP_OK;
}

template <typename F>
static int rows_as(const F8Product& p, bool gateup, bool routed, bool dense, hipStream_t st) {
  const int groups_r = routed ? (p.Nr + 15) / 16 : 0, groups_s = dense ? (p.Ns + 15) / 16 : 0;
  if (gateup) return p.T <= 16 ? launch_rows<F, true, 1, 4>(p, groups_r, groups_s, st) : launch_rows<F, true, 2, 4>(p, groups_r, groups_s, st);
  if (p.T > 16) return launch_rows<F, false, 2, 4>(p, groups_r, groups_s, st);
  return !routed && f8_blocks(p.Ks) > kF8LongBlocks ? launch_rows<F, false, 1, 8>(p, groups_r, groups_s, st)
                                                    : launch_rows<F, false, 1, 4>(p, groups_r, groups_s, st);
}

int f8_rows(const F8Product& p, bool gateup, bool routed, bool dense, hipStream_t st) {
  return p.dtype == SPARSE_HIP_F16 ? rows_as<Fp16>(p, gateup, routed, dense, st) : rows_as<Bf16>(p, gateup, routed, dense, st);
}

}  // namespace sparse
