// Block-scaled 8-bit floating point (OCP e4m3): what the quantiser and the matrix kernels share.
//
// Activations: rows of e4m3 values padded with zeros to a multiple of 128, one power-of-two scale (an
// E8M0 byte, value 2^(byte - 127)) for each run of 128.  Weights: 16-row x 128-column tiles of 2 KB in
// the order of the 16-bit layout taken byte by byte (row r, k: 1 KB half (k/16)%2, then k quarter
// (k/32)%4, row r%16, 16 bytes), one fp32 scale for each 128 x 128 block.
#pragma once

#include "common.h"

namespace sparse {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float vf32x4 __attribute__((ext_vector_type(4)));

constexpr int kF8Block = 128;          // values that share a scale
constexpr int kF8Bias = 127;           // E8M0
constexpr int kF8LowestExp = -120;     // smallest exponent the quantiser chooses
constexpr int kF8One = 0x7f7f7f7f;     // four E8M0 scales of 1
constexpr int kF8TileBytes = 16 * kF8Block;

inline int f8_blocks(int k) { return (k + kF8Block - 1) / kF8Block; }
inline size_t f8_padded(int k) { return static_cast<size_t>(f8_blocks(k)) * kF8Block; }
inline int f8_rows16(int n) { return (n + 15) & ~15; }

// Exponent of the scale of a run whose largest finite magnitude is `amax`: the smallest s >= -120 with
// amax <= 448 * 2^s.  448 = 1.75 * 2^8, so it is read off amax's own exponent and fraction: no logarithm,
// no division, the same bits on every machine.  (A power of two loses nothing against amax / 448: the
// quotient x / 2^s is exact, so a value is rounded once, to e4m3, whose steps are relative.)
__device__ __forceinline__ int f8_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int s = static_cast<int>(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(s, kF8LowestExp);
}
// 2^-s for an exponent in [-120, 120]
__device__ __forceinline__ float f8_inverse(int s) { return __uint_as_float(static_cast<uint32_t>(127 - s) << 23); }
// Largest of magnitudes over the 16 lanes of a DPP row, in every one of them.
__device__ __forceinline__ float f8_row16_max(float v) {
  v = fmaxf(v, dpp_move<0x121, 0xf>(0.f, v));   // row_ror:1, 2, 4, 8
  v = fmaxf(v, dpp_move<0x122, 0xf>(0.f, v));
  v = fmaxf(v, dpp_move<0x124, 0xf>(0.f, v));
  v = fmaxf(v, dpp_move<0x128, 0xf>(0.f, v));
  return v;
}
// ... over the 8 lanes of half a row.
__device__ __forceinline__ float f8_row8_max(float v) {
  v = fmaxf(v, dpp_move<0xb1, 0xf>(0.f, v));    // quad_perm 1,0,3,2
  v = fmaxf(v, dpp_move<0x4e, 0xf>(0.f, v));    // quad_perm 2,3,0,1
  v = fmaxf(v, dpp_move<0x141, 0xf>(0.f, v));   // row_half_mirror
  return v;
}
// The magnitude that counts towards amax: NaN and infinities do not (they become NaN in 8 bits).
__device__ __forceinline__ float f8_magnitude(float v) {
  const float a = fabsf(v);
  return a < INFINITY ? a : 0.f;
}
// Four values (already divided by the scale) as e4m3 bytes, round to nearest even.  Finite ones fit by the
// choice of scale; infinities go in as NaN, which is what e4m3 has for them.
__device__ __forceinline__ float f8_finite(float v) { return fabsf(v) < INFINITY ? v : __uint_as_float(0x7fc00000u); }
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
  int p = __builtin_amdgcn_cvt_pk_fp8_f32(f8_finite(a), f8_finite(b), 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f8_finite(c), f8_finite(d), p, true));
}

__device__ __forceinline__ i32x8 f8_join(i32x4 lo, i32x4 hi) {
  return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}
// c + a b over 128 k; `sa` / `sb` hold E8M0 scales, one byte of which counts (kSa, kSb).  A: lane l holds
// row l % 16, B: column l % 16, 32 bytes each, the same k in both; the scale of a lane's row or column is
// the same in the four lanes that share it, as one scale covers all 128 k.
//
// The instruction adds the products of eight consecutive k with the smaller ones cut off 13 bits below the
// largest (sum of the factors' exponents) and goes on in fp32 from there; the narrower 8-bit instructions do
// the same.  On rows of unit normal values that is an error of some 2^-15 of the result, next to 2^-5 that
// rounding the factors to 8 bits has cost, and at most 2^-10 of a group's largest power of two (eight products, each
// short by less than 2^-13 of it).  It rules out fp32 outputs, which the operators do not offer, and gate and up, whose
// result is rounded to 8 bits next: those are products widened to bf16 in every kernel.
template <int kSa, int kSb>
__device__ __forceinline__ vf32x4 f8_mfma(i32x8 a, i32x8 b, vf32x4 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, kSa, sa, kSb, sb);
}

// Four consecutive columns n .. n + 3 of a row of N, times `sc`, rounded once.
template <typename F>
__device__ __forceinline__ void f8_store4(uint16_t* o, vf32x4 v, float sc, int N, int n) {
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

// Eight e4m3 bytes as bf16, which holds them exactly, also times a power of two from 2^-121 to 2^119 (the smallest
// become subnormal numbers, which conversion and matrix instruction keep).
template <bool kHigh>
__device__ __forceinline__ uint32_t f8_widen2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, kHigh));
}
__device__ __forceinline__ bf16x8 f8_widen8(uint32_t lo, uint32_t hi, float scale = 1.f) {
  const u32x4 v = {f8_widen2<false>(lo, scale), f8_widen2<true>(lo, scale), f8_widen2<false>(hi, scale), f8_widen2<true>(hi, scale)};
  return __builtin_bit_cast(bf16x8, v);
}
// The 32 bytes of one operand of a 128-wide block as the operands of four 32-wide bf16 instructions, and the
// product of two such: products added in fp32 (no scales), where the 8-bit instruction cuts them off.
struct F8Wide {
  bf16x8 v[4];
};
__device__ __forceinline__ F8Wide f8_widen(i32x4 lo, i32x4 hi) {
  F8Wide r;
  r.v[0] = f8_widen8(lo[0], lo[1]);
  r.v[1] = f8_widen8(lo[2], lo[3]);
  r.v[2] = f8_widen8(hi[0], hi[1]);
  r.v[3] = f8_widen8(hi[2], hi[3]);
  return r;
}
__device__ __forceinline__ vf32x4 f8_mfma_wide(const F8Wide& a, const F8Wide& b) {
  vf32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[j], b.v[j], c, 0, 0, 0);
  return c;
}

// How a slot of the expert slab is laid out: gate values [I, Hp] | up [I, Hp] | down [H, Ip], then their
// scales [nI, nH] | [nI, nH] | [nH, nI] in fp32 (Hp, Ip: rounded up to 128; nH, nI: number of blocks).
struct F8Slot {
  uint64_t up, down, sgate, sup, sdown, bytes;
};
inline F8Slot f8_slot(int H, int I) {
  F8Slot s;
  const uint64_t gu = static_cast<uint64_t>(I) * f8_padded(H), dn = static_cast<uint64_t>(H) * f8_padded(I);
  const uint64_t sc = static_cast<uint64_t>(f8_blocks(H)) * f8_blocks(I) * sizeof(float);
  s.up = gu;
  s.down = 2 * gu;
  s.sgate = 2 * gu + dn;
  s.sup = s.sgate + sc;
  s.sdown = s.sup + sc;
  s.bytes = (s.sdown + sc + 255) & ~255ull;
  return s;
}

// ---- launches of the other files ---------------------------------------------------------------
// rows of x (dtype code) -> values [T, Kp], scales [T, blocks]; a second matrix of the same type in the same
// launch if T2 > 0
struct F8Quantize {
  const void* x;
  int64_t T;
  int32_t K;
  void *values, *scales;
};
int f8_quantize(const F8Quantize& a, const F8Quantize& b, int dtype, hipStream_t st);
// one matrix to rows in bf16 that the 8-bit values are times half their scales, for f8_tile_gateup (no scales are
// written), and in the same launch the tile queues of its call
struct PfxMapArgs;
int f8_quantize_and_queue(const F8Quantize& a, int dtype, const PfxMapArgs& queue, hipStream_t st);

// One matrix product of a call, over the routed segments of an expert slab, a dense matrix, or both.
struct F8Product {
  // routed operands
  const uint8_t* slab;
  uint64_t slot_stride, off0, off1, soff0, soff1;   // bytes: matrices (second: up) and their scales in a slot
  const int32_t *expert_slot, *perm, *seg_offsets;
  const void* topv;
  const uint8_t *act_r, *act_rs;                    // rows, scales of 8-bit ones; gathered through perm when gather != 0
  void* out_r;
  int32_t topk, Kr, Nr, gather;
  // dense operands
  const uint8_t *w0, *w1;
  const float *s0, *s1;
  const uint8_t *act_s, *act_ss;
  const void* gate_s;                               // [T] logits of the rows' sigmoid factor, or NULL
  void* out_s;
  int32_t Ks, Ns, T;
  int32_t dtype;                                    // of topv, gate_s and outputs
  int32_t pow2;                                     // tiles may take scales that are powers of two as exponents
  sparse_hip_seglist segs;
};

// Lists that an earlier launch wrote, read with scalar loads.
typedef const __attribute__((address_space(4))) int32_t* f8_list;

// Which 16 output columns of which matrix a workgroup of the streaming kernels owns, and for which rows.
struct F8Where {
  const uint8_t *w0, *w1;      // the tile's panels
  const float *s0, *s1;        // and their scales
  const uint8_t *act, *acts;   // the rows' values and scales
  const int32_t* perm;         // gathered rows: flat row -> token * topk + slot; else NULL
  f8_list range;               // routed: the segment's first row and the one behind its last
  int topk, T, nb, K, N, n0;
  bool dense;
  __device__ __forceinline__ int first_row() const { return dense ? 0 : range[0]; }
  __device__ __forceinline__ int rows() const { return dense ? T : range[1] - range[0]; }
};
// At the start of a kernel every load takes up to a microsecond, and the compiler places each behind the wait for the
// one before.  Passing values through an empty statement has them loaded together and kept: the kernel's arguments,
// then the segment count with the expert, then (where the slots are in a list) the slot.  The segment's rows
// are asked for later: the weights' addresses do not need them.
__device__ __forceinline__ bool f8_where(const F8Product& a, int block, int tiles_r, int tiles_s, F8Where& w) {
  const int32_t *slots = a.expert_slot, *eids = a.segs.eids_dev, *counts = a.segs.count_dev;
  uint64_t stride = a.slot_stride, off0 = a.off0, off1 = a.off1, soff0 = a.soff0, soff1 = a.soff1;
  int n = a.segs.n, gather = a.gather, Kr = a.Kr, Nr = a.Nr;
  w.K = a.Ks;
  w.N = a.Ns;
  w.topk = a.topk;
  w.T = a.T;
  w.range = reinterpret_cast<f8_list>(reinterpret_cast<uintptr_t>(a.seg_offsets));
  asm volatile("" : "+s"(tiles_r), "+s"(tiles_s), "+s"(stride), "+s"(off0), "+s"(off1), "+s"(soff0), "+s"(soff1), "+s"(w.range),
               "+s"(slots), "+s"(eids), "+s"(counts), "+s"(n), "+s"(gather), "+s"(Kr), "+s"(Nr)
               : "s"(a.slab), "s"(a.w0), "s"(a.w1), "s"(a.s0), "s"(a.s1), "s"(a.act_r), "s"(a.act_rs), "s"(a.act_s), "s"(a.act_ss),
                 "s"(a.perm));
  asm volatile("" : "+s"(w.K), "+s"(w.N), "+s"(w.topk), "+s"(w.T));
  w.dense = block < tiles_s;
  int tile = block;
  if (w.dense) {
    w.act = a.act_s;
    w.acts = a.act_ss;
    w.perm = nullptr;
    w.w0 = a.w0;
    w.w1 = a.w1;
    w.s0 = a.s0;
    w.s1 = a.s1;
  } else {
    const int b = block - tiles_s, si = b / tiles_r;
    tile = b - si * tiles_r;
    int eid, slot_id;
    if (eids != nullptr) {
      int count = reinterpret_cast<f8_list>(reinterpret_cast<uintptr_t>(counts))[0];
      eid = reinterpret_cast<f8_list>(reinterpret_cast<uintptr_t>(eids))[si];
      asm volatile("" : "+s"(count), "+s"(eid));
      if (si >= min(count, n)) return false;
      slot_id = slots != nullptr ? reinterpret_cast<f8_list>(reinterpret_cast<uintptr_t>(slots))[eid] : eid;
    } else {
      eid = __builtin_amdgcn_readfirstlane(a.segs.eids[si]);
      slot_id = __builtin_amdgcn_readfirstlane(a.segs.slots[si]);
    }
    w.range += eid;
    w.K = Kr;
    w.N = Nr;
    w.act = a.act_r;
    w.acts = a.act_rs;
    w.perm = gather ? a.perm : nullptr;
    const uint8_t* slot = a.slab + static_cast<uint64_t>(slot_id) * stride;
    w.w0 = slot + off0;
    w.w1 = slot + off1;
    w.s0 = reinterpret_cast<const float*>(slot + soff0);
    w.s1 = reinterpret_cast<const float*>(slot + soff1);
  }
  w.n0 = tile * 16;
  w.nb = (w.K + kF8Block - 1) / kF8Block;
  const size_t panel = static_cast<size_t>(tile) * w.nb * kF8TileBytes, scales = static_cast<size_t>(w.n0 / kF8Block) * w.nb;
  w.w0 += panel;
  w.w1 += panel;
  w.s0 += scales;
  w.s1 += scales;
  return true;
}
// Two rows at most: gate/up (SwiGLU of two products, fp32 out) or a single product, of rows that are
// quantised on the way in (from the 16-bit type, from fp32) or were before.
constexpr int kF8FewRows = 2;
// From this many blocks of 128 on, workgroups of 8 wavefronts instead of 4 stream a single matrix past up to 16 rows:
// its 16-column workgroups do not fill the device, and the depth of a wavefront's share is the call's time.  One row of
// 5632 by 2048 weight rows 7.2 -> 5.7 us, of 4096 by 4096 6.6 -> 5.9; of 2048 by 5632, 16 blocks, 5.5 -> 5.9.
constexpr int kF8LongBlocks = 20;
enum { kF8From16 = 0, kF8From32 = 1, kF8From8 = 2 };
int f8_few(const F8Product& p, int source, bool gateup, bool routed, bool dense, hipStream_t st);

// The same of more rows, 8-bit ones.
int f8_rows(const F8Product& p, bool gateup, bool routed, bool dense, hipStream_t st);

// The same of many rows: 128 x 256 tiles.  gate/up takes rows in bf16 and writes quantised ones; routed and dense tiles
// come from one set of queues.
struct PfQueues;
int f8_tile_gateup(const F8Product& p, const PfQueues& q, void* h, void* hs, void* sh, void* shs, hipStream_t st);
// (tiles of 32 rows are 128 columns wide in down and linear)
int f8_tile_columns(int tile_rows);
int f8_tile_down(const F8Product& p, const PfQueues& q, int tile_rows, hipStream_t st);
int f8_tile_linear(const F8Product& p, int tile_rows, hipStream_t st);

}  // namespace sparse
