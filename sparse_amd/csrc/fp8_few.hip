// Block-scaled 8-bit matrix products of few rows: a stream of weights past activations that fit in LDS.
//
// A workgroup owns 16 output columns (weight rows) of two matrices (gate and up of one expert) or 16 or 32 of
// one, and up to 16 NT rows.  Its four wavefronts deal the 128-wide k blocks among themselves; a chunk of 4 KW
// blocks at a time; each wavefront requests its weights of a chunk (2 KB a block, straight from the tiled
// layout into registers) two chunks ahead, and while they travel the workgroup quantises its rows of the chunk into LDS:
// 16 lanes hold a run of 128, find its largest magnitude, round to 8 bits and put the rounded values down as
// bf16, which holds them exactly, with the run's scale behind the row.  Quantising here costs a launch less
// than quantising before, and a row or two of a segment are quickly done.
//
// The product itself is taken in bf16: an e4m3 value is a bf16 value, 16 conversions of two turn a lane's 32
// weights into four operands.  The 8-bit instruction would be half as many cycles, but what bounds this kernel
// is the weights' way from HBM, and the 8-bit instruction cuts products off 13 bits below the largest of
// eight while bf16 products are added in fp32: an intermediate that is to be rounded to 8 bits then lands on
// the other side of a rounding border a tenth as often.
//
// A block's sum is multiplied by the run's power of two and the weights' fp32 scale on its way into the
// accumulator.
#include "fp8.h"

namespace sparse {

constexpr int kFwThreads = 256;
constexpr int kFwWaves = kFwThreads / 64;
constexpr int kFwBatch = 3;       // runs a group of 16 lanes fetches at a time, after the first of a chunk
constexpr int kSrc16 = kF8From16, kSrc32 = kF8From32, kSrc8 = kF8From8;

// LDS row of a chunk: values, scales, and as much more as spreads 16 rows over the banks
__host__ __device__ constexpr int fw_values(int kw) { return kFwWaves * kw * kF8Block * 2; }
__host__ __device__ constexpr int fw_stride(int kw) { return fw_values(kw) + 80; }
static_assert(kFwWaves * 2 * sizeof(float) <= 64, "the scales of a chunk fit behind its values");

// Two e4m3 bytes (the low or the high half of `w`) as bf16, exactly; the wide forms of four and of eight.
template <bool kHigh>
__device__ __forceinline__ uint32_t fw_widen2(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, kHigh));
}
__device__ __forceinline__ bf16x8 fw_widen8(uint32_t lo, uint32_t hi) {
  const u32x4 v = {fw_widen2<false>(lo), fw_widen2<true>(lo), fw_widen2<false>(hi), fw_widen2<true>(hi)};
  return __builtin_bit_cast(bf16x8, v);
}

// Eight values of a run, one sixteenth of it, on their way to LDS.
__device__ __forceinline__ u32x4 fw_round(const float (&v)[8], float& scale) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, f8_magnitude(v[j]));
  const int s = f8_exponent(f8_row16_max(m));
  const float inv = f8_inverse(s);
  scale = __uint_as_float(static_cast<uint32_t>(s + kF8Bias) << 23);
  return __builtin_bit_cast(u32x4, fw_widen8(f8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                                             f8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv)));
}
template <typename F, int kSrc>
struct Source;
template <typename F>
struct Source<F, kSrc16> {
  u32x4 v;
  __device__ __forceinline__ void load(const uint8_t* base, const uint8_t*, size_t row, int K, int, int kb, int at, bool vec) {
    const int k = kb * kF8Block + at;
    const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + row * K + k;
    if (vec) {
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
template <typename F>
struct Source<F, kSrc32> {
  vf32x4 a, b;
  __device__ __forceinline__ void load(const uint8_t* base, const uint8_t*, size_t row, int K, int, int kb, int at, bool) {
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
template <typename F>
struct Source<F, kSrc8> {
  uint2 v;
  uint8_t e;
  __device__ __forceinline__ void load(const uint8_t* base, const uint8_t* scales, size_t row, int, int nb, int kb, int at, bool) {
    v = *reinterpret_cast<const uint2*>(base + (row * nb + kb) * kF8Block + at);
    e = scales[row * nb + kb];
  }
  __device__ __forceinline__ u32x4 rounded(float& scale) const {
    scale = __uint_as_float(static_cast<uint32_t>(e) << 23);
    return __builtin_bit_cast(u32x4, fw_widen8(v.x, v.y));
  }
};

// kGateUp: the two matrices are gate and up, fp32 SwiGLU out.  Otherwise NM 16-row groups of one matrix.
template <typename F, bool kGateUp, int NM, int NT, int KW, int kSrc>
__global__ __launch_bounds__(kFwThreads) void f8_few_kernel(const F8Product a, int tiles_r, int tiles_s, int vec) {
  constexpr int KC = kFwWaves * KW, kStride = fw_stride(KW);
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 15, q = lane >> 4;
  const bool dense = static_cast<int>(blockIdx.x) < tiles_s;

  const uint8_t *w0, *w1;
  const float *s0, *s1;
  int K, N, tile, M, r0 = 0;
  if (dense) {
    tile = blockIdx.x;
    K = a.Ks;
    N = a.Ns;
    M = a.T;
    w0 = a.w0;
    w1 = a.w1;
    s0 = a.s0;
    s1 = a.s1;
  } else {
    const int b = blockIdx.x - tiles_s, si = b / tiles_r;
    tile = b - si * tiles_r;
    int eid, slot_id;
    if (a.segs.eids_dev != nullptr) {
      if (si >= min(a.segs.count_dev[0], a.segs.n)) return;
      eid = a.segs.eids_dev[si];
      slot_id = a.expert_slot[eid];
    } else {
      eid = a.segs.eids[si];
      slot_id = a.segs.slots[si];
    }
    K = a.Kr;
    N = a.Nr;
    r0 = a.seg_offsets[eid];
    M = a.seg_offsets[eid + 1] - r0;
    const uint8_t* slot = a.slab + static_cast<uint64_t>(slot_id) * a.slot_stride;
    w0 = slot + a.off0;
    w1 = slot + a.off1;
    s0 = reinterpret_cast<const float*>(slot + a.soff0);
    s1 = reinterpret_cast<const float*>(slot + a.soff1);
  }
  const int m0 = blockIdx.y * 16 * NT;     // a dense call of more rows takes them in groups
  M = min(M - m0, min(16 * NT, a.T));      // (a segment has at most T rows)
  if (M <= 0) return;
  r0 += m0;
  const int nb = (K + kF8Block - 1) / kF8Block;
  const int n0 = tile * 16 * (kGateUp ? 1 : NM);
  const uint8_t* wp[NM];
  const float* sp[NM];
#pragma unroll
  for (int mi = 0; mi < NM; ++mi) {
    const int last16 = ((N + 15) & ~15) - 16;
    const int n = kGateUp ? n0 : min(n0 + mi * 16, last16);   // behind the last group: computed, not stored
    wp[mi] = (kGateUp && mi ? w1 : w0) + static_cast<size_t>(n >> 4) * nb * kF8TileBytes + lane * 16;
    sp[mi] = (kGateUp && mi ? s1 : s0) + static_cast<size_t>(n / kF8Block) * nb;
  }

  vf32x4 acc[NM][NT];
#pragma unroll
  for (int mi = 0; mi < NM; ++mi)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[mi][nt] = vf32x4{0.f, 0.f, 0.f, 0.f};

  // The factor of the row whose sum this lane stores at the end, asked for now.
  const int my_m = (wave / NM) * 16 + r;   // wavefront f stores fragment f = nt * NM + mi
  float factor = 1.f;
  if (!kGateUp && wave < NT * NM && my_m < M) {
    if (!dense) factor = F::from_bits(static_cast<const uint16_t*>(a.topv)[a.perm[r0 + my_m]]);
    else if (a.gate_s != nullptr) factor = F::from_bits(static_cast<const uint16_t*>(a.gate_s)[r0 + my_m]);
  }

  // ---- the chunks --------------------------------------------------------------------------
  // Two register stages in turn: while a chunk is multiplied the next one's loads are in flight.  Loads
  // complete in order, so a chunk's rows, which are wanted first, are requested before its weights; only the
  // first chunk's weights go ahead of its rows, whose addresses wait for the permutation.
  const int group = threadIdx.x >> 4, gl = threadIdx.x & 15;
  const int runs = M * KC;               // run i of a chunk: row i / KC, block i % KC
  auto request = [&](int i, int c0) {    // runs past the end repeat the last row
    const int m = min(i / KC, M - 1), kb = min(c0 + i % KC, nb - 1);
    size_t row = r0 + m;
    if (!dense && a.gather) row = static_cast<uint32_t>(a.perm[r0 + m]) / static_cast<uint32_t>(a.topk);
    Source<F, kSrc> src;
    src.load(dense ? a.act_s : a.act_r, dense ? a.act_ss : a.act_rs, row, K, nb, kb, gl * 8, vec != 0);
    return src;
  };
  auto lay = [&](const Source<F, kSrc>& src, int i, uint8_t* buf) {
    float scale;
    const u32x4 out = src.rounded(scale);
    if (i >= runs) return;
    uint8_t* row = buf + (i / KC) * kStride;
    *reinterpret_cast<u32x4*>(row + (i % KC) * (kF8Block * 2) + gl * 16) = out;
    if (gl == 0) *reinterpret_cast<float*>(row + fw_values(KW) + (i % KC) * 4) = scale;
  };
  struct Stage {
    i32x4 w[KW][NM][2];
    float ws[KW][NM];
    Source<F, kSrc> src;
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
        st.ws[i][mi] = sp[mi][kb];
      }
    }
  };
  auto load_rows = [&](Stage& st, int chunk) __attribute__((always_inline)) { st.src = request(group, chunk * KC); };
  auto use = [&](const Stage& st, int chunk, uint8_t* buf) __attribute__((always_inline)) {
    const int c0 = chunk * KC;
    lay(st.src, group, buf);
    for (int p = 1; p * 16 < runs; p += kFwBatch) {     // more rows than the stage holds
      Source<F, kSrc> more[kFwBatch];
#pragma unroll
      for (int j = 0; j < kFwBatch; ++j) more[j] = request((p + j) * 16 + group, c0);
#pragma unroll
      for (int j = 0; j < kFwBatch; ++j) lay(more[j], (p + j) * 16 + group, buf);
    }
    __syncthreads();     // (the other buffer may still be read by a slower wavefront: this one is not)
#pragma unroll
    for (int i = 0; i < KW; ++i) {
      const int kl = wave + i * kFwWaves;
      if (c0 + kl < nb) {
        vf32x4 part[NM][NT];
#pragma unroll
        for (int mi = 0; mi < NM; ++mi)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) part[mi][nt] = vf32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {    // 32 k of the block: a lane's bytes 8 j .. 8 j + 7
          bf16x8 b[NT];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            b[nt] = *reinterpret_cast<const bf16x8*>(buf + min(nt * 16 + r, M - 1) * kStride + kl * (kF8Block * 2) + q * 64 + j * 16);
#pragma unroll
          for (int mi = 0; mi < NM; ++mi) {
            const i32x4 half = st.w[i][mi][j >> 1];
            const bf16x8 wa = fw_widen8(half[2 * (j & 1)], half[2 * (j & 1) + 1]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              part[mi][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wa, b[nt], part[mi][nt], 0, 0, 0);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float xs = *reinterpret_cast<const float*>(buf + min(nt * 16 + r, M - 1) * kStride + fw_values(KW) + kl * 4);
#pragma unroll
          for (int mi = 0; mi < NM; ++mi)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[mi][nt][j] = fmaf(part[mi][nt][j] * xs, st.ws[i][mi], acc[mi][nt][j]);
        }
      }
    }
  };
  const int chunks = (nb + KC - 1) / KC;
  const int buf_rows = min(a.T, 16 * NT);
  uint8_t *const buf0 = lds, *const buf1 = lds + buf_rows * kStride;
  Stage s0_, s1_;
  load_weights(s0_, 0);
  __builtin_amdgcn_sched_barrier(0);
  load_rows(s0_, 0);
  load_rows(s1_, 1);
  __builtin_amdgcn_sched_barrier(0);
  load_weights(s1_, 1);
  __builtin_amdgcn_sched_barrier(0);
  int c = 0;
  for (; c + 4 <= chunks; c += 2) {      // (no branch in here: the waits count what is in flight)
    use(s0_, c, buf0);
    __builtin_amdgcn_sched_barrier(0);
    load_rows(s0_, c + 2);
    load_weights(s0_, c + 2);
    __builtin_amdgcn_sched_barrier(0);
    use(s1_, c + 1, buf1);
    __builtin_amdgcn_sched_barrier(0);
    load_rows(s1_, c + 3);
    load_weights(s1_, c + 3);
    __builtin_amdgcn_sched_barrier(0);
  }
  use(s0_, c, buf0);                     // one to three chunks are left
  if (c + 2 < chunks) {
    load_rows(s0_, c + 2);
    load_weights(s0_, c + 2);
  }
  if (c + 1 < chunks) use(s1_, c + 1, buf1);
  if (c + 2 < chunks) use(s0_, c + 2, buf0);

  // ---- the wavefronts' sums meet in LDS ------------------------------------------------------
  __syncthreads();
  vf32x4* red = reinterpret_cast<vf32x4*>(lds);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mi = 0; mi < NM; ++mi) red[(wave * NT * NM + nt * NM + mi) * 64 + lane] = acc[mi][nt];
  __syncthreads();
  auto sum = [&](int f) {
    vf32x4 v = red[f * 64 + lane];
#pragma unroll
    for (int w = 1; w < kFwWaves; ++w) v += red[(w * NT * NM + f) * 64 + lane];
    return v;
  };
  if (kGateUp) {
    for (int nt = wave; nt < NT; nt += kFwWaves) {
      const int m = nt * 16 + r;
      if (m >= M) continue;
      const vf32x4 g = sum(nt * NM), u = sum(nt * NM + 1);
      vf32x4 h;
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = silu_f32(g[j]) * u[j];
      *reinterpret_cast<vf32x4*>(static_cast<float*>(dense ? a.out_s : a.out_r) + static_cast<size_t>(r0 + m) * N + n0 + q * 4) = h;
    }
  } else {
    static_assert(NT * NM <= kFwWaves, "one fragment per wavefront at most");
    const int mi = wave % NM, m = my_m, n = n0 + mi * 16 + q * 4;
    if (wave < NT * NM && m < M && n < N) {
      const vf32x4 v = sum(wave);
      const float sc = dense && a.gate_s != nullptr ? sigmoid_f32(factor) : factor;
      uint16_t* o = static_cast<uint16_t*>(dense ? a.out_s : a.out_r) + static_cast<size_t>(r0 + m) * N + n;
      uint2 pk;
      pk.x = F::pack2(v[0] * sc, v[1] * sc);
      pk.y = F::pack2(v[2] * sc, v[3] * sc);
      if (N % 4 == 0 && (reinterpret_cast<uintptr_t>(o) & 7) == 0) {
        *reinterpret_cast<uint2*>(o) = pk;
      } else {
        const uint32_t e[2] = {pk.x, pk.y};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < N) o[j] = static_cast<uint16_t>(e[j >> 1] >> (16 * (j & 1)));
      }
    }
  }
}

template <typename F, bool kGateUp, int NM, int NT, int KW, int kSrc>
static int launch_few(const F8Product& p, int tiles_r, int tiles_s, int vec, hipStream_t st) {
  const int64_t grid = tiles_s + static_cast<int64_t>(tiles_r) * p.segs.n;
  const int64_t groups = tiles_r == 0 ? (p.T + 16 * NT - 1) / (16 * NT) : 1;
  if (grid == 0) return SPARSE_HIP_OK;
  SP_REQUIRE(grid < (1ll << 31) && groups < 65536, "fp8 product: grid too large");
  const int rows = p.T < 16 * NT ? p.T : 16 * NT;
  const int stage = 2 * rows * fw_stride(KW), red = kFwWaves * NM * NT * 64 * static_cast<int>(sizeof(vf32x4));
  hipLaunchKernelGGL((f8_few_kernel<F, kGateUp, NM, NT, KW, kSrc>), dim3(static_cast<unsigned>(grid), static_cast<unsigned>(groups)),
                     dim3(kFwThreads), static_cast<unsigned>(stage > red ? stage : red), st, p, tiles_r, tiles_s, vec);
  SP_LAUNCH_CHECK("f8_few_kernel");
  return SPARSE_HIP_OK;
}

template <typename F, bool kGateUp, int NM, int kSrc>
static int few_by_rows(const F8Product& p, int tiles_r, int tiles_s, int vec, hipStream_t st) {
  // A chunk is eight blocks, or four for 17 rows and more: two buffers of the rows then take 34 KB of LDS at
  // most for 8 rows and 71 KB for 32.
  if constexpr (kSrc == kSrc32) {
    SP_REQUIRE(p.T <= 16, "fp8 product: %d rows of fp32", p.T);
    return launch_few<F, kGateUp, NM, 1, 2, kSrc>(p, tiles_r, tiles_s, vec, st);
  } else if (p.T <= 16) {
    return launch_few<F, kGateUp, NM, 1, 2, kSrc>(p, tiles_r, tiles_s, vec, st);
  } else {
    return launch_few<F, kGateUp, NM, 2, 1, kSrc>(p, tiles_r, tiles_s, vec, st);
  }
}

template <typename F>
static int few_as(const F8Product& p, int source, bool gateup, bool routed, bool dense, hipStream_t st) {
  const int groups_r = routed ? (p.Nr + 15) / 16 : 0, groups_s = dense ? (p.Ns + 15) / 16 : 0;
  // 16-byte loads of the rows need aligned rows of a multiple of eight values
  const int K = dense ? p.Ks : p.Kr;
  const int vec = K % 8 == 0 && ((reinterpret_cast<uintptr_t>(p.act_s) | reinterpret_cast<uintptr_t>(p.act_r)) & 15) == 0;
  if (gateup) return few_by_rows<F, true, 2, kSrc16>(p, groups_r, groups_s, vec, st);
  // Two 16-row groups per workgroup halve the rows' traffic; one keeps the device full when groups are few.
  const bool two = groups_s + static_cast<int64_t>(groups_r) * (p.segs.n < p.T * p.topk ? p.segs.n : p.T * p.topk) >= 2048;
  const int tr = two ? (groups_r + 1) / 2 : groups_r, ts = two ? (groups_s + 1) / 2 : groups_s;
#define SP_FEW(S) (two ? few_by_rows<F, false, 2, S>(p, tr, ts, vec, st) : few_by_rows<F, false, 1, S>(p, tr, ts, vec, st))
  if (source == kF8From16) return SP_FEW(kSrc16);
  if (source == kF8From32) return SP_FEW(kSrc32);
  return SP_FEW(kSrc8);
#undef SP_FEW
}

int f8_few(const F8Product& p, int source, bool gateup, bool routed, bool dense, hipStream_t st) {
  return p.dtype == SPARSE_HIP_F16 ? few_as<Fp16>(p, source, gateup, routed, dense, st)
                                   : few_as<Bf16>(p, source, gateup, routed, dense, st);
}

}  // namespace sparse
