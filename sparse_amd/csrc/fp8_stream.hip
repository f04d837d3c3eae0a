// Block-scaled 8-bit matrix products by streaming the weights past a few rows: y[t, n] =
// sum over blocks b of 2^s[t,b] * w[n/128, b] * (sum of q[t,k] q[n,k] over the block's 128 k).
//
// A workgroup owns 16 output columns (weight rows) of one matrix, or of the gate and the up matrix of one
// expert, and all rows of the segment, 16 NT at a time.  Its wavefronts take the 128-wide k blocks in turn;
// a block is one 16x16x128 matrix instruction per 16 rows, into which the activation's scale goes as the
// instruction's own operand; the weight's scale, an fp32 number, multiplies the block's sum on its way into
// the accumulator.
#include "fp8.h"

namespace sparse {

constexpr int kStThreads = 256;
constexpr int kStWaves = kStThreads / 64;

// 16 or 32-bit tensors by dtype code
__device__ __forceinline__ float ld_any(const void* p, size_t i, int dtype) {
  if (dtype == SPARSE_HIP_BF16) return Elem<uint16_t>::load(static_cast<const uint16_t*>(p) + i);
  if (dtype == SPARSE_HIP_F16) return Elem<f16_t>::load(static_cast<const f16_t*>(p) + i);
  return static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void st_any(void* p, size_t i, int dtype, float v) {
  if (dtype == SPARSE_HIP_BF16) Elem<uint16_t>::store(static_cast<uint16_t*>(p) + i, v);
  else if (dtype == SPARSE_HIP_F16) Elem<f16_t>::store(static_cast<f16_t*>(p) + i, v);
  else static_cast<float*>(p)[i] = v;
}

template <bool kGateUp, int NT>
__global__ __launch_bounds__(kStThreads) void f8_stream_kernel(const F8Product a, int tiles_r, int tiles_s) {
  constexpr int NM = kGateUp ? 2 : 1;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int r = lane & 15, q = lane >> 4;
  const bool dense = static_cast<int>(blockIdx.x) < tiles_s;

  const uint8_t *w0, *w1 = nullptr;
  const float *s0, *s1 = nullptr;
  int nb, N, tile, M, r0 = 0;
  if (dense) {
    tile = blockIdx.x;
    nb = (a.Ks + kF8Block - 1) / kF8Block;
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
    nb = (a.Kr + kF8Block - 1) / kF8Block;
    N = a.Nr;
    r0 = a.seg_offsets[eid];
    M = a.seg_offsets[eid + 1] - r0;
    const uint8_t* slot = a.slab + static_cast<uint64_t>(slot_id) * a.slot_stride;
    w0 = slot + a.off0;
    w1 = slot + a.off1;
    s0 = reinterpret_cast<const float*>(slot + a.soff0);
    s1 = reinterpret_cast<const float*>(slot + a.soff1);
  }
  const int n0 = tile * 16;
  const size_t panel = static_cast<size_t>(tile) * nb * kF8TileBytes + lane * 16;
  w0 += panel;
  w1 += panel;
  s0 += static_cast<size_t>(n0 / kF8Block) * nb;
  s1 += static_cast<size_t>(n0 / kF8Block) * nb;
  const size_t ld = static_cast<size_t>(nb) * kF8Block;

  __shared__ vf32x4 red[kStWaves][NT * NM][64];
  for (int m0 = blockIdx.y * 16 * NT; m0 < M; m0 += gridDim.y * 16 * NT) {
    const uint8_t *brow[NT], *bscale[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int m = min(m0 + nt * 16 + r, M - 1);     // rows past the end repeat the last and are not stored
      if (dense) {
        brow[nt] = a.act_s + m * ld;
        bscale[nt] = a.act_ss + static_cast<size_t>(m) * nb;
      } else {
        const size_t g = a.gather ? a.perm[r0 + m] / a.topk : r0 + m;
        brow[nt] = a.act_r + g * ld;
        bscale[nt] = a.act_rs + g * nb;
      }
      brow[nt] += q * 32;
    }
    vf32x4 acc[NM][NT];
#pragma unroll
    for (int mi = 0; mi < NM; ++mi)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[mi][nt] = vf32x4{0.f, 0.f, 0.f, 0.f};
    for (int kb = wave; kb < nb; kb += kStWaves) {
      i32x8 w[NM];
      float ws[NM];
#pragma unroll
      for (int mi = 0; mi < NM; ++mi) {
        const uint8_t* p = (mi ? w1 : w0) + static_cast<size_t>(kb) * kF8TileBytes;
        w[mi] = f8_join(*reinterpret_cast<const i32x4*>(p), *reinterpret_cast<const i32x4*>(p + 1024));
        ws[mi] = (mi ? s1 : s0)[kb];
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint8_t* p = brow[nt] + kb * kF8Block;
        const i32x8 b = f8_join(*reinterpret_cast<const i32x4*>(p), *reinterpret_cast<const i32x4*>(p + 16));
        const int bs = bscale[nt][kb];
#pragma unroll
        for (int mi = 0; mi < NM; ++mi) {
          const vf32x4 part = f8_mfma<0, 0>(w[mi], b, vf32x4{0.f, 0.f, 0.f, 0.f}, kF8One, bs);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[mi][nt][j] = fmaf(part[j], ws[mi], acc[mi][nt][j]);
        }
      }
    }
    __syncthreads();     // an earlier chunk's sums have been read
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int mi = 0; mi < NM; ++mi) red[wave][nt * NM + mi][lane] = acc[mi][nt];
    __syncthreads();
    for (int nt = wave; nt < NT; nt += kStWaves) {
      const int m = m0 + nt * 16 + r;
      if (m >= M) continue;
      vf32x4 v = red[0][nt * NM][lane], u = kGateUp ? red[0][nt * NM + NM - 1][lane] : vf32x4{0.f, 0.f, 0.f, 0.f};
      for (int w = 1; w < kStWaves; ++w) {
        v += red[w][nt * NM][lane];
        if (kGateUp) u += red[w][nt * NM + NM - 1][lane];
      }
      void* out = dense ? a.out_s : a.out_r;
      const size_t at = static_cast<size_t>(r0 + m) * N + n0 + q * 4;
      float f = 1.f;
      if (!kGateUp) {
        if (!dense) f = ld_any(a.topv, a.perm[r0 + m], a.dtype);
        else if (a.gate_s != nullptr) f = sigmoid_f32(ld_any(a.gate_s, m, a.dtype));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (n0 + q * 4 + j >= N) break;
        if (kGateUp) static_cast<float*>(out)[at + j] = silu_f32(v[j]) * u[j];
        else st_any(out, at + j, a.dtype, v[j] * f);
      }
    }
  }
}

template <bool kGateUp>
static int launch_stream(const F8Product& p, int tiles_r, int tiles_s, unsigned chunks, hipStream_t st) {
  const int64_t grid = tiles_s + static_cast<int64_t>(tiles_r) * p.segs.n;
  if (grid == 0) return SPARSE_HIP_OK;
  SP_REQUIRE(grid < (1ll << 31), "fp8 product: grid too large");
  if (chunks > 1)
    hipLaunchKernelGGL((f8_stream_kernel<kGateUp, 2>), dim3(static_cast<unsigned>(grid), chunks), dim3(kStThreads), 0, st, p,
                       tiles_r, tiles_s);
  else
    hipLaunchKernelGGL((f8_stream_kernel<kGateUp, 1>), dim3(static_cast<unsigned>(grid)), dim3(kStThreads), 0, st, p,
                       tiles_r, tiles_s);
  SP_LAUNCH_CHECK("f8_stream_kernel");
  return SPARSE_HIP_OK;
}

int f8_stream(const F8Product& p, bool gateup, bool routed, bool dense, hipStream_t st) {
  const int tiles_r = routed ? (p.Nr + 15) / 16 : 0, tiles_s = dense ? (p.Ns + 15) / 16 : 0;
  const unsigned chunks = p.T <= 16 ? 1 : static_cast<unsigned>(p.T + 31) / 32 < 64u ? static_cast<unsigned>(p.T + 31) / 32 : 64u;
  return gateup ? launch_stream<true>(p, tiles_r, tiles_s, chunks, st) : launch_stream<false>(p, tiles_r, tiles_s, chunks, st);
}

}  // namespace sparse
