// Expert selection with a balance bias: scores (softmax or sigmoid of the logits), the bias added for the
// ranking only, group limit, top-k, weights from the scores without the bias.
//
// One wavefront per token; lane l holds experts l, l + 64, ...  The order is that of the scores in 64 bits: the
// sum of a score and a bias has no order of its own that 32 bits would keep (with 256 experts and 4096 tokens,
// a handful of neighbours in the ranking lie within one fp32 rounding of each other), so in 32 bits the
// selected experts would be a function of how exp was rounded.  Ties go to the lower expert id.
//
// The ranking runs in 32 bits all the same, on values known to 2^-19 + 2^-22 |r|, and every comparison that
// decides something is checked: the gap between two neighbours of the ranking, the last chosen and the first
// not chosen among them, and between any two groups, is larger than both errors, or the token starts over in
// 64 bits (about one token in a hundred of 256 random logits; equal 16-bit logits without a bias always do).
// A group's sum of two is as far off as its two terms together, however small it is itself: where large biases
// of both signs cancel in it, the 32-bit sum may be rounding alone.
// 32-bit maxima cross the lanes in one instruction a step where 64-bit ones take a dozen: one token of 256
// experts in 8 groups 8.7 -> 5.8 us, 4096 tokens 17.1 -> 13.6 us.  What is left is the latency of the K + 1
// maxima, one behind the other, of the groups and of the exponentials in 64 bits: 4 MB of logits are read in a
// microsecond.
#include "common.h"

namespace sparse {

constexpr int kSelWaves = 4;
static_assert(SPARSE_HIP_MAX_EXPERTS <= 256, "four experts per lane at most");
constexpr int kSelMaxGroups = 64;
constexpr int kSelMaxTokens = 1 << 28;       // token numbers of the last workgroup stay within 32 bits

struct SelectArgs {
  const void* logits;
  const float* bias;
  void* topv;
  int64_t* topi;
  int32_t T, E, K, sigmoid, n_group, topk_group, top2, renorm;
  float scale;
};

constexpr int kNobody = 0x7fffffff;

// 64-bit moves across lanes, halves separately (see wave_max).
template <int kCtrl, int kRowMask>
__device__ __forceinline__ double dpp_move(double identity, double v) {
  const uint64_t i = __builtin_bit_cast(uint64_t, identity), b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(static_cast<int>(i), static_cast<int>(b), kCtrl, kRowMask, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(static_cast<int>(i >> 32), static_cast<int>(b >> 32), kCtrl, kRowMask, 0xf, false);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ __forceinline__ double read_lane(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(b), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), lane);
  return __builtin_bit_cast(double, (static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ __forceinline__ float read_lane(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ __forceinline__ double wave_max(double v) {
  constexpr double kLow = -INFINITY;
  v = fmax(v, dpp_move<0x111, 0xf>(kLow, v));
  v = fmax(v, dpp_move<0x112, 0xf>(kLow, v));
  v = fmax(v, dpp_move<0x114, 0xf>(kLow, v));
  v = fmax(v, dpp_move<0x118, 0xf>(kLow, v));
  v = fmax(v, dpp_move<0x142, 0xa>(kLow, v));
  v = fmax(v, dpp_move<0x143, 0xc>(kLow, v));
  return read_lane(v, 63);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Which expert lane k < K has in k-th place, by the values r (expert lane + 64 j).  V = double: the order,
// ties to the lower id.  V = float: the same if it is clear; false if a comparison was too close to call.
template <typename V, int NV>
__device__ __forceinline__ bool select_by(const SelectArgs& a, V (&r)[NV], V* s_rank, int lane, int& sel) {
  constexpr bool kExact = sizeof(V) == 8;
  constexpr V kLow = -INFINITY;
  // twice what a 32-bit value may be off
  const auto size = [](V v) { return v < 0 ? -v : v; };
  const auto slack = [&](V v) { return static_cast<V>(3.814697e-6f) + static_cast<V>(4.76837e-7f) * size(v); };
  bool clear = true;
  int id[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) id[j] = lane + 64 * j < a.E ? lane + 64 * j : kNobody;
  if (a.topk_group < a.n_group) {
    const int gsz = a.E / a.n_group;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (lane + 64 * j < a.E) s_rank[lane + 64 * j] = r[j];
    __builtin_amdgcn_wave_barrier();
    // L lanes share a group: each the best two of every L-th expert, then the L of them
    const int L = 1 << (31 - __clz(64 / a.n_group)), g = lane / L, part = lane & (L - 1);
    V best = kLow, second = kLow;
    if (g < a.n_group) {
      for (int i = part; i < gsz; i += L) {
        const V v = s_rank[g * gsz + i];
        second = v > best ? best : (v > second ? v : second);
        best = v > best ? v : best;
      }
    }
    for (int o = 1; o < L; o <<= 1) {
      const V b2 = __shfl_xor(best, o), s2 = __shfl_xor(second, o);
      second = b2 > best ? (best > s2 ? best : s2) : (second > b2 ? second : b2);
      best = b2 > best ? b2 : best;
    }
    V mag = size(best);                        // of what a group's score is the sum of
    if (a.top2 && gsz > 1) {
      mag += size(second);
      best += second;
    }
    if (!(best == best)) best = kLow;          // an infinite bias beside a score that ranks last
    int before = 0;
    for (int i = 0; i < a.n_group; ++i) {
      const V v = read_lane(best, i * L);
      before += v > best || (kExact && v == best && i < g);
      if (!kExact) clear &= i == g || g >= a.n_group || size(v - best) > slack(mag) + slack(read_lane(mag, i * L));
    }
    const unsigned long long keep = __ballot(g < a.n_group && part == 0 && before < a.topk_group);
    const float per = 1.f / static_cast<float>(gsz);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int eg = static_cast<int>((static_cast<float>(lane + 64 * j) + 0.5f) * per);   // (lane + 64 j) / gsz
      if (!((keep >> ((eg * L) & 63)) & 1ull)) {
        r[j] = kLow;
        id[j] = kNobody;
      }
    }
  }
  // a lane's values in their order, so that only its first one takes part in each round
  auto order = [&](int i, int j) {
    const bool swap = r[i] < r[j] || (kExact && r[i] == r[j] && id[i] > id[j]);
    const V x = swap ? r[j] : r[i], y = swap ? r[i] : r[j];
    const int p = swap ? id[j] : id[i], q = swap ? id[i] : id[j];
    r[i] = x;
    r[j] = y;
    id[i] = p;
    id[j] = q;
  };
  if constexpr (NV == 2) order(0, 1);
  if constexpr (NV == 4) {
    order(0, 1);
    order(2, 3);
    order(0, 2);
    order(1, 3);
    order(1, 2);
  }
  V last = INFINITY;
  for (int k = 0; k <= a.K; ++k) {
    if (kExact && k == a.K) break;
    const V w = wave_max(r[0]);
    if (!kExact) {
      clear &= last - w > slack(size(last) < size(w) ? last : w);   // (before the first and behind the last: infinite)
      if (k == a.K) break;
      last = w;
    }
    const unsigned long long who = __ballot(r[0] == w && id[0] != kNobody);
    int lw = who != 0ull ? __builtin_ctzll(who) : 0;
    if (who == 0ull || (who & (who - 1)) != 0ull) {
      if (!kExact) return false;
      const int first = wave_min_int(r[0] == w ? id[0] : kNobody);
      lw = first & 63;
    }
    const int wi = __builtin_amdgcn_readlane(id[0], lw);
    if (lane == k) sel = wi;
    if (lane == lw) {
#pragma unroll
      for (int j = 0; j + 1 < NV; ++j) {
        r[j] = r[j + 1];
        id[j] = id[j + 1];
      }
      r[NV - 1] = kLow;
      id[NV - 1] = kNobody;
    }
  }
  return __all(clear);
}

// NV: experts per lane
template <typename TL, typename TO, int NV>
__global__ __launch_bounds__(kSelWaves * 64) void gate_select_kernel(const SelectArgs a) {
  __shared__ double s_rank[kSelWaves][64 * NV];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int t = blockIdx.x * kSelWaves + wave;
  if (t >= a.T) return;
  const TL* row = static_cast<const TL*>(a.logits) + static_cast<size_t>(t) * a.E;

  float l[NV], b[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e = lane + 64 * j;
    l[j] = e < a.E ? Elem<TL>::load(row + e) : -INFINITY;
    b[j] = e < a.E && a.bias != nullptr ? a.bias[e] : 0.f;
  }
  // softmax: the largest logit and the sum, in 64 bits.  A row without a finite logit has no largest one to
  // subtract: its scores are 0, not NaN.
  float m = -INFINITY;
  double total = 1.0;
  if (!a.sigmoid) {
#pragma unroll
    for (int j = 0; j < NV; ++j) m = fmaxf(m, l[j]);
    m = wave_max(m);
    total = 0.0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (lane + 64 * j < a.E) total += (m == -INFINITY && l[j] == -INFINITY) ? 0.0 : exp(static_cast<double>(l[j]) - m);
    total = wave_sum_f64(total);
  }
  auto score = [&](float logit) -> double {
    if (a.sigmoid) return 1.0 / (1.0 + exp(-static_cast<double>(logit)));
    if (m == -INFINITY && logit == -INFINITY) return 0.0;
    return exp(static_cast<double>(logit) - m) / total;
  };

  int sel = 0;
  float r[NV];
  bool usual = true;      // neither NaN nor infinity among the values to rank
  const float scale = a.sigmoid ? 1.f : static_cast<float>(1.0 / total);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const float e = __builtin_amdgcn_exp2f((a.sigmoid ? -l[j] : l[j] - m) * 1.44269504f);
    r[j] = (a.sigmoid ? __builtin_amdgcn_rcpf(1.f + e) : e * scale) + b[j];
    if (lane + 64 * j < a.E) usual = usual && fabsf(r[j]) < INFINITY;
    else r[j] = -INFINITY;
  }
  if (!__all(usual) || !select_by<float, NV>(a, r, reinterpret_cast<float*>(s_rank[wave]), lane, sel)) {
    double x[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      x[j] = -INFINITY;
      if (lane + 64 * j < a.E) x[j] = score(l[j]) + static_cast<double>(b[j]);
      if (!(x[j] == x[j])) x[j] = -INFINITY;   // NaN ranks last, so that the ids stay distinct and in range
    }
    select_by<double, NV>(a, x, s_rank[wave], lane, sel);
  }

  double v = 0.0;
  if (lane < a.K) v = score(Elem<TL>::load(row + sel));
  if (a.renorm) {
    double sum = 0.0;
    for (int k = 0; k < a.K; ++k) sum += read_lane(v, k);
    v /= fmax(sum, 1e-20);
  }
  if (lane < a.K) {
    Elem<TO>::store(static_cast<TO*>(a.topv) + static_cast<size_t>(t) * a.K + lane, static_cast<float>(v * a.scale));
    a.topi[static_cast<size_t>(t) * a.K + lane] = sel;
  }
}

template <typename TL, typename TO>
static int launch_select(const SelectArgs& a, hipStream_t st) {
  const dim3 grid((a.T + kSelWaves - 1) / kSelWaves), block(kSelWaves * 64);
  if (a.E <= 64) hipLaunchKernelGGL((gate_select_kernel<TL, TO, 1>), grid, block, 0, st, a);
  else if (a.E <= 128) hipLaunchKernelGGL((gate_select_kernel<TL, TO, 2>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((gate_select_kernel<TL, TO, 4>), grid, block, 0, st, a);
  SP_LAUNCH_CHECK("gate_select_kernel");
  return SPARSE_HIP_OK;
}
template <typename TL>
static int launch_select(const SelectArgs& a, int out_dtype, hipStream_t st) {
  if (out_dtype == SPARSE_HIP_BF16) return launch_select<TL, uint16_t>(a, st);
  if (out_dtype == SPARSE_HIP_F16) return launch_select<TL, f16_t>(a, st);
  return launch_select<TL, float>(a, st);
}

}  // namespace sparse

using namespace sparse;

extern "C" int sparse_hip_gate_select(const void* logits_dev, int logits_dtype, const float* bias_dev, int T, int E,
                                      int K, int score, int n_group, int topk_group, int group_score, int renorm,
                                      float scale, int out_dtype, void* topv_dev, int64_t* topi_dev, void* stream) {
  SP_REQUIRE(valid_dtype(logits_dtype) && valid_dtype(out_dtype), "gate_select: unknown dtype %d / %d", logits_dtype, out_dtype);
  SP_REQUIRE(E >= 1 && E <= SPARSE_HIP_MAX_EXPERTS, "gate_select: E=%d outside [1,%d]", E, SPARSE_HIP_MAX_EXPERTS);
  SP_REQUIRE(K >= 1 && K <= SPARSE_HIP_MAX_TOPK && K <= E, "gate_select: K=%d outside [1,min(%d,E=%d)]", K, SPARSE_HIP_MAX_TOPK, E);
  SP_REQUIRE(score == SPARSE_HIP_SCORE_SOFTMAX || score == SPARSE_HIP_SCORE_SIGMOID, "gate_select: unknown score %d", score);
  SP_REQUIRE(group_score == SPARSE_HIP_GROUP_MAX || group_score == SPARSE_HIP_GROUP_TOP2,
             "gate_select: unknown group score %d", group_score);
  SP_REQUIRE(n_group >= 1 && n_group <= kSelMaxGroups && E % n_group == 0,
             "gate_select: n_group=%d must divide E=%d and be at most %d", n_group, E, kSelMaxGroups);
  SP_REQUIRE(topk_group >= 1 && topk_group <= n_group, "gate_select: topk_group=%d outside [1,%d]", topk_group, n_group);
  SP_REQUIRE(K <= topk_group * (E / n_group), "gate_select: K=%d exceeds the %d experts of %d groups", K,
             topk_group * (E / n_group), topk_group);
  SP_REQUIRE(T >= 0 && T <= kSelMaxTokens, "gate_select: T=%d outside [0,%d]", T, kSelMaxTokens);
  if (T == 0) return SPARSE_HIP_OK;
  SP_REQUIRE(logits_dev && topv_dev && topi_dev, "gate_select: NULL pointer");
  const SelectArgs a = {logits_dev, bias_dev, topv_dev, topi_dev, T, E, K, score == SPARSE_HIP_SCORE_SIGMOID,
                        n_group, topk_group, group_score == SPARSE_HIP_GROUP_TOP2, renorm, scale};
  hipStream_t st = as_stream(stream);
  if (logits_dtype == SPARSE_HIP_BF16) return launch_select<uint16_t>(a, out_dtype, st);
  if (logits_dtype == SPARSE_HIP_F16) return launch_select<f16_t>(a, out_dtype, st);
  return launch_select<float>(a, out_dtype, st);
}
