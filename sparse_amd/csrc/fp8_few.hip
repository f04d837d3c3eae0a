// Block-scaled 8-bit matrix products of one or two rows: a stream of weights past rows that are quantised into
// LDS on the way.
//
//   y[m, n] = sum over blocks b of 2^e(m, b) s(n, b) sum over k in b of q[m, k] w[n, k],  q, e: the quantiser's
//
// A workgroup owns 16 output columns (weight rows) of two matrices (gate and up of one expert) or of one.  Its
// wavefronts, four or, for a single matrix of long rows, eight (kF8LongBlocks), deal the 128-wide k blocks among
// themselves, a chunk of KW blocks each at a time; each wavefront requests
// its weights of a chunk (2 KB a block, straight from the tiled layout into registers) two chunks ahead, and while
// they travel the workgroup quantises its rows of the chunk: 16 lanes hold a run of 128, find its largest
// magnitude, round to 8 bits and put the rounded values down as bf16, which holds them exactly, with the run's
// scale behind the row.  A launch less than quantising before, and for two rows quickly done.  KW = 2 (gate/up
// and down of one token, KW = 1, 2, 4: 12.2 + 10.4, 11.7 + 8.4, 14.2 + 8.2 us).
//
// The product itself is taken in bf16: an e4m3 value is a bf16 value, 16 conversions of two turn a lane's 32
// weights into four operands.  The 8-bit instruction would be half as many cycles, but what bounds this kernel
// is the weights' way from HBM, and the 8-bit instruction cuts products off 13 bits below the largest of
// eight while bf16 products are added in fp32: an intermediate that is to be rounded to 8 bits then lands on
// the other side of a rounding border a tenth as often.  A block's sum is multiplied by the run's power of two
// and the weights' fp32 scale on its way into the accumulator.
//
// One token of 4 among 60 experts of 1408 x 2048 and a shared one of 5632: gate/up 46 MB in 9 to 11 us, down 23 MB in
// 7.9 to 9.2; a single 5632 x 2048 matrix, 11.5 MB, 5.3 us (from the last-level cache).  At the 7 TB/s of longer
// streams that would be 6.6 and 3.3 us: the rest is the start of a launch (2.5 us until the first weights arrive, by
// time stamps in the kernel) and its end (1.5 us of sums and stores), and in down the shared expert's six chunks.
#include "fp8.h"

namespace sparse {

constexpr int kSrc16 = kF8From16, kSrc32 = kF8From32, kSrc8 = kF8From8;
constexpr int KW = 2;                             // blocks of a chunk per wavefront

// Eight values of a run, one sixteenth of it, on their way to LDS.
__device__ __forceinline__ u32x4 fw_round(const float (&v)[8], float& scale) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, f8_magnitude(v[j]));
  const int s = f8_exponent(f8_row16_max(m));
  const float inv = f8_inverse(s);
  scale = __uint_as_float(static_cast<uint32_t>(s + kF8Bias) << 23);
  return __builtin_bit_cast(u32x4, f8_widen8(f8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                                             f8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv)));
}
// kVec: rows of the 16-bit type start on 16-byte boundaries and hold a multiple of 8 values
template <typename F, int kSrc, bool kVec>
struct Source;
template <typename F, bool kVec>
struct Source<F, kSrc16, kVec> {
  u32x4 v;
  __device__ __forceinline__ void load(const uint8_t* base, const uint8_t*, size_t row, int K, int, int kb, int at) {
    const int k = kb * kF8Block + at;
    const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + row * K + k;
    if (kVec) {
      v = k < K ? *reinterpret_cast<const u32x4*>(p) : u32x4{0, 0, 0, 0};
    } else {
      uint32_t e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = k + j < K ? p[j] : 0u;
      v = u32x4{e[0] | (e[1] << 16), e[2] | (e[3] << 16), e[4] | (e[5] << 16), e[6] | (e[7] << 16)};
    }
  }
  __device__ __forceinline__ u32x4 rounded(float& scale) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = F::from_bits(static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1))));
    return fw_round(f, scale);
  }
};
template <typename F, bool kVec>
struct Source<F, kSrc32, kVec> {
  vf32x4 a, b;
  __device__ __forceinline__ void load(const uint8_t* base, const uint8_t*, size_t row, int K, int, int kb, int at) {
    const int k = kb * kF8Block + at;    // K a multiple of 64
    const float* p = reinterpret_cast<const float*>(base) + row * K + k;
    a = b = vf32x4{0.f, 0.f, 0.f, 0.f};
    if (k < K) {
      a = *reinterpret_cast<const vf32x4*>(p);
      b = *reinterpret_cast<const vf32x4*>(p + 4);
    }
  }
  __device__ __forceinline__ u32x4 rounded(float& scale) const {
    const float f[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return fw_round(f, scale);
  }
};
template <typename F, bool kVec>
struct Source<F, kSrc8, kVec> {
  uint2 v;
  uint8_t e;
  __device__ __forceinline__ void load(const uint8_t* base, const uint8_t* scales, size_t row, int, int nb, int kb, int at) {
    v = *reinterpret_cast<const uint2*>(base + (row * nb + kb) * kF8Block + at);
    e = scales[row * nb + kb];
  }
  __device__ __forceinline__ u32x4 rounded(float& scale) const {
    scale = __uint_as_float(static_cast<uint32_t>(e) << 23);
    return __builtin_bit_cast(u32x4, f8_widen8(v.x, v.y));
  }
};

// kGateUp: two matrices, gate and up, fp32 SwiGLU out.  Otherwise one.  kFwWaves: wavefronts of a workgroup.
template <typename F, bool kGateUp, int kSrc, bool kVec, int kFwWaves>
__global__ __launch_bounds__(kFwWaves * 64) void f8_few_kernel(const F8Product a, int tiles_r, int tiles_s) {
  constexpr int NM = kGateUp ? 2 : 1;
  constexpr int KC = kFwWaves * KW;                 // blocks of a chunk
  constexpr int kFwValues = KC * kF8Block * 2;      // LDS row of a chunk: values, scales
  constexpr int kFwStride = kFwValues + KC * 4;
  static_assert(kFwWaves * 4 == kF8FewRows * KC, "one run of a chunk for each 16 lanes");
  constexpr int kStage = 2 * kF8FewRows * kFwStride, kSums = kFwWaves * NM * 64 * static_cast<int>(sizeof(vf32x4));
  __shared__ __attribute__((aligned(16))) uint8_t lds[kStage > kSums ? kStage : kSums];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 15, q = lane >> 4;
  F8Where own;
  if (!f8_where(a, blockIdx.x, tiles_r, tiles_s, own)) return;
  const bool dense = own.dense;
  const int nb = own.nb, K = own.K, N = own.N, n0 = own.n0;
  const uint8_t* wp[NM];
  const float* sp[NM];
#pragma unroll
  for (int mi = 0; mi < NM; ++mi) {
    wp[mi] = (mi ? own.w1 : own.w0) + lane * 16;
    sp[mi] = mi ? own.s1 : own.s0;
  }

  vf32x4 acc[NM];
#pragma unroll
  for (int mi = 0; mi < NM; ++mi) acc[mi] = vf32x4{0.f, 0.f, 0.f, 0.f};

  // ---- the chunks --------------------------------------------------------------------------
  // Two register stages in turn: while a chunk is multiplied the next one's loads are in flight.  Loads
  // complete in order, so a chunk's rows, which are wanted first, are requested before its weights; only the
  // first chunk's weights go ahead of its rows, whose addresses wait for the permutation.
  const int my_m = threadIdx.x / (16 * KC), my_kb = (threadIdx.x >> 4) % KC, gl = threadIdx.x & 15;
  struct Stage {
    i32x4 w[KW][NM][2];
    float ws[KW][NM];
    Source<F, kSrc, kVec> src;
  };
  auto load_weights = [&](Stage& st, int chunk) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < KW; ++i) {
      const int kb = min(chunk * KC + wave + i * kFwWaves, nb - 1);
#pragma unroll
      for (int mi = 0; mi < NM; ++mi) {
        const uint8_t* p = wp[mi] + static_cast<size_t>(kb) * kF8TileBytes;
        // read once per launch: a non-temporal load leaves the caches to the activations
        st.w[i][mi][0] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(p));
        st.w[i][mi][1] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(p + 1024));
      }
    }
  };
  auto load_scales = [&](Stage& st, int chunk) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < KW; ++i)
#pragma unroll
      for (int mi = 0; mi < NM; ++mi) st.ws[i][mi] = sp[mi][min(chunk * KC + wave + i * kFwWaves, nb - 1)];
  };
  // ---- the first weights go out before anything that waits for the segment's rows ------------
  Stage s0_, s1_;
  load_weights(s0_, 0);
  __builtin_amdgcn_sched_barrier(0);
  const int r0 = own.first_row(), M = min(own.rows(), kF8FewRows);   // (the ids of a token are distinct: a segment has T rows at most)
  if (M <= 0) return;
  // (a second row that is not there repeats the first; of one token every row is its)
  size_t my_row = r0 + min(my_m, M - 1);
  if (own.perm != nullptr) my_row = own.T == 1 ? 0 : static_cast<uint32_t>(own.perm[my_row]) / static_cast<uint32_t>(own.topk);
  auto load_rows = [&](Stage& st, int chunk) __attribute__((always_inline)) {
    st.src.load(own.act, own.acts, my_row, K, nb, min(chunk * KC + my_kb, nb - 1), gl * 8);
  };
  auto use = [&](const Stage& st, int chunk, uint8_t* buf) __attribute__((always_inline)) {
    const int c0 = chunk * KC;
    float scale;
    const u32x4 rounded = st.src.rounded(scale);
    if (my_m < M) {
      uint8_t* row = buf + my_m * kFwStride;
      *reinterpret_cast<u32x4*>(row + my_kb * (kF8Block * 2) + gl * 16) = rounded;
      if (gl == 0) *reinterpret_cast<float*>(row + kFwValues + my_kb * 4) = scale;
    }
    __syncthreads();     // (the other buffer may still be read by a slower wavefront: this one is not)
#pragma unroll
    for (int i = 0; i < KW; ++i) {
      const int kl = wave + i * kFwWaves;
      if (c0 + kl < nb) {
        const uint8_t* row = buf + min(r, M - 1) * kFwStride;    // columns past the rows are not stored
        const uint8_t* values = row + kl * (kF8Block * 2) + q * 64;
        F8Wide x;
#pragma unroll
        for (int j = 0; j < 4; ++j) x.v[j] = *reinterpret_cast<const bf16x8*>(values + j * 16);
        const float xs = *reinterpret_cast<const float*>(row + kFwValues + kl * 4);
#pragma unroll
        for (int mi = 0; mi < NM; ++mi) {
          const vf32x4 part = f8_mfma_wide(f8_widen(st.w[i][mi][0], st.w[i][mi][1]), x);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[mi][j] = fmaf(part[j] * xs, st.ws[i][mi], acc[mi][j]);
        }
      }
    }
  };
  const int chunks = (nb + KC - 1) / KC;
  uint8_t *const buf0 = lds, *const buf1 = lds + kF8FewRows * kFwStride;
  load_rows(s0_, 0);
  load_rows(s1_, 1);
  __builtin_amdgcn_sched_barrier(0);
  load_weights(s1_, 1);
  __builtin_amdgcn_sched_barrier(0);
  load_scales(s0_, 0);
  load_scales(s1_, 1);
  // The factor of the row whose sum this lane stores at the end, asked for once the loads of
  // the first chunks are on their way.
  float factor = 1.f;
  if (!kGateUp && wave == 0 && r < M) {
    if (!dense) factor = F::from_bits(static_cast<const uint16_t*>(a.topv)[a.perm[r0 + r]]);
    else if (a.gate_s != nullptr) factor = F::from_bits(static_cast<const uint16_t*>(a.gate_s)[r0 + r]);
  }
  __builtin_amdgcn_sched_barrier(0);
  int c = 0;
  for (; c + 4 <= chunks; c += 2) {      // (no branch in here: the waits count what is in flight)
    use(s0_, c, buf0);
    __builtin_amdgcn_sched_barrier(0);
    load_rows(s0_, c + 2);
    load_weights(s0_, c + 2);
    load_scales(s0_, c + 2);
    __builtin_amdgcn_sched_barrier(0);
    use(s1_, c + 1, buf1);
    __builtin_amdgcn_sched_barrier(0);
    load_rows(s1_, c + 3);
    load_weights(s1_, c + 3);
    load_scales(s1_, c + 3);
    __builtin_amdgcn_sched_barrier(0);
  }
  use(s0_, c, buf0);                     // one to three chunks are left
  if (c + 2 < chunks) {
    load_rows(s0_, c + 2);
    load_weights(s0_, c + 2);
    load_scales(s0_, c + 2);
  }
  if (c + 1 < chunks) use(s1_, c + 1, buf1);
  if (c + 2 < chunks) use(s0_, c + 2, buf0);

  // ---- the wavefronts' sums meet in LDS ------------------------------------------------------
  __syncthreads();
  vf32x4* red = reinterpret_cast<vf32x4*>(lds);
#pragma unroll
  for (int mi = 0; mi < NM; ++mi) red[(wave * NM + mi) * 64 + lane] = acc[mi];
  __syncthreads();
  auto sum = [&](int mi) {
    vf32x4 v = red[mi * 64 + lane];
#pragma unroll
    for (int w = 1; w < kFwWaves; ++w) v += red[(w * NM + mi) * 64 + lane];
    return v;
  };
  if (wave != 0 || r >= M) return;
  const int n = n0 + q * 4;
  const size_t at = static_cast<size_t>(r0 + r) * N + n;
  if (kGateUp) {
    const vf32x4 g = sum(0), u = sum(NM - 1);
    vf32x4 h;
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = silu_f32(g[j]) * u[j];
    *reinterpret_cast<vf32x4*>(static_cast<float*>(dense ? a.out_s : a.out_r) + at) = h;
  } else if (n < N) {
    const float sc = dense && a.gate_s != nullptr ? sigmoid_f32(factor) : factor;
    f8_store4<F>(static_cast<uint16_t*>(dense ? a.out_s : a.out_r) + at, sum(0), sc, N, n);
  }
}

template <typename F, bool kGateUp, int kSrc, bool kVec, int W = 4>
static int launch_few(const F8Product& p, int tiles_r, int tiles_s, hipStream_t st) {
  const int64_t grid = tiles_s + static_cast<int64_t>(tiles_r) * p.segs.n;
  if (grid == 0) return SPARSE_HIP_OK;
  SP_REQUIRE(grid < (1ll << 31), "fp8 product: grid too large");
  SP_REQUIRE(p.T <= kF8FewRows, "fp8 product: %d rows", p.T);
  hipLaunchKernelGGL((f8_few_kernel<F, kGateUp, kSrc, kVec, W>), dim3(static_cast<unsigned>(grid)), dim3(W * 64), 0, st, p,
                     tiles_r, tiles_s);
  SP_LAUNCH_CHECK("f8_few_kernel");
  return SPARSE_HIP_OK;
}

template <typename F>
static int few_as(const F8Product& p, int source, bool gateup, bool routed, bool dense, hipStream_t st) {
  const int tr = routed ? (p.Nr + 15) / 16 : 0, ts = dense ? (p.Ns + 15) / 16 : 0;
  if (source == kF8From32) return launch_few<F, false, kSrc32, true>(p, tr, ts, st);
  const bool wide = !routed && f8_blocks(p.Ks) > kF8LongBlocks;
  if (source == kF8From8)
    return wide ? launch_few<F, false, kSrc8, true, 8>(p, tr, ts, st) : launch_few<F, false, kSrc8, true>(p, tr, ts, st);
  // 16-byte loads of the rows need aligned rows of a multiple of eight values
  const int K = dense ? p.Ks : p.Kr;
  const bool vec = K % 8 == 0 && ((reinterpret_cast<uintptr_t>(p.act_s) | reinterpret_cast<uintptr_t>(p.act_r)) & 15) == 0;
  if (gateup) return vec ? launch_few<F, true, kSrc16, true>(p, tr, ts, st) : launch_few<F, true, kSrc16, false>(p, tr, ts, st);
  if (wide) return vec ? launch_few<F, false, kSrc16, true, 8>(p, tr, ts, st) : launch_few<F, false, kSrc16, false, 8>(p, tr, ts, st);
  return vec ? launch_few<F, false, kSrc16, true>(p, tr, ts, st) : launch_few<F, false, kSrc16, false>(p, tr, ts, st);
}

int f8_few(const F8Product& p, int source, bool gateup, bool routed, bool dense, hipStream_t st) {
  return p.dtype == SPARSE_HIP_F16 ? few_as<Fp16>(p, source, gateup, routed, dense, st)
                                   : few_as<Bf16>(p, source, gateup, routed, dense, st);
}

}  // namespace sparse
