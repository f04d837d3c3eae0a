// Expert selection with a balance bias: scores (softmax or sigmoid of the logits), the bias added for the
// ranking only, group limit, top-k, weights from the scores without the bias.
//
// One wavefront per token; lane l holds experts l, l + 64, ...  The ranking is done in 64 bits: the sum of
// a score and a bias has no order of its own that 32 bits would keep (with 256 experts and 4096 tokens, a
// handful of neighbours in the ranking lie within one fp32 rounding of each other), so in 32 bits the
// selected experts would be a function of how exp was rounded.  Ties go to the lower expert id.
#include "common.h"

namespace sparse {

constexpr int kSelWaves = 4;
constexpr int kSelNV = SPARSE_HIP_MAX_EXPERTS / 64;
constexpr int kSelMaxGroups = 64;

struct SelectArgs {
  const void* logits;
  const float* bias;
  void* topv;
  int64_t* topi;
  int32_t T, E, K, sigmoid, n_group, topk_group, top2, renorm;
  float scale;
};

__device__ __forceinline__ double wave_max_f64(double v) {
  for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o));
  return v;
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

template <typename TL, typename TO>
__global__ __launch_bounds__(kSelWaves * 64) void gate_select_kernel(const SelectArgs a) {
  __shared__ double s_rank[kSelWaves][SPARSE_HIP_MAX_EXPERTS];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int t = blockIdx.x * kSelWaves + wave;
  if (t >= a.T) return;
  const TL* row = static_cast<const TL*>(a.logits) + static_cast<size_t>(t) * a.E;

  double p[kSelNV], r[kSelNV];   // score, what is ranked
  unsigned alive = 0u;
  double m = -INFINITY;
#pragma unroll
  for (int j = 0; j < kSelNV; ++j) {
    const int e = lane + 64 * j;
    p[j] = -INFINITY;
    if (e < a.E) {
      p[j] = Elem<TL>::load(row + e);
      alive |= 1u << j;
      m = fmax(m, p[j]);
    }
  }
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < kSelNV; ++j)
      if ((alive >> j) & 1u) p[j] = 1.0 / (1.0 + exp(-p[j]));
  } else {
    // a row without a finite logit has no largest one to subtract: its scores are 0, not NaN
    m = wave_max_f64(m);
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < kSelNV; ++j) {
      if ((alive >> j) & 1u) {
        p[j] = (m == -INFINITY && p[j] == -INFINITY) ? 0.0 : exp(p[j] - m);
        s += p[j];
      }
    }
    s = wave_sum_f64(s);
#pragma unroll
    for (int j = 0; j < kSelNV; ++j)
      if ((alive >> j) & 1u) p[j] = s == 0.0 ? 0.0 : p[j] / s;
  }
#pragma unroll
  for (int j = 0; j < kSelNV; ++j) {
    r[j] = -INFINITY;
    if ((alive >> j) & 1u) {
      r[j] = p[j] + (a.bias != nullptr ? static_cast<double>(a.bias[lane + 64 * j]) : 0.0);
      if (!(r[j] == r[j])) r[j] = -INFINITY;   // NaN ranks last, so that the ids stay distinct and in range
    }
  }

  if (a.topk_group < a.n_group) {
    const int gsz = a.E / a.n_group;
#pragma unroll
    for (int j = 0; j < kSelNV; ++j)
      if ((alive >> j) & 1u) s_rank[wave][lane + 64 * j] = r[j];
    __builtin_amdgcn_wave_barrier();
    double best = -INFINITY, second = -INFINITY;
    if (lane < a.n_group) {
      for (int i = 0; i < gsz; ++i) {
        const double v = s_rank[wave][lane * gsz + i];
        second = fmax(second, fmin(best, v));
        best = fmax(best, v);
      }
      if (a.top2 && gsz > 1) best += second;
      if (!(best == best)) best = -INFINITY;   // an infinite bias beside a score that ranks last
    }
    unsigned long long keep = 0ull;
    for (int k = 0; k < a.topk_group; ++k) {
      const bool cand = lane < a.n_group && !((keep >> lane) & 1ull);
      const double w = wave_max_f64(cand ? best : -INFINITY);
      keep |= 1ull << wave_min_int((cand && best == w) ? lane : 0x7fffffff);
    }
#pragma unroll
    for (int j = 0; j < kSelNV; ++j)
      if (((alive >> j) & 1u) && !((keep >> ((lane + 64 * j) / gsz)) & 1ull)) alive &= ~(1u << j);
  }

  double sel_v = 0.0, sum = 0.0;
  int sel_i = 0;
  for (int k = 0; k < a.K; ++k) {
    double bv = -INFINITY, bp = 0.0;
    int bi = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < kSelNV; ++j) {
      if (((alive >> j) & 1u) && (bi == 0x7fffffff || r[j] > bv)) {
        bv = r[j];
        bp = p[j];
        bi = lane + 64 * j;
      }
    }
    const double w = wave_max_f64(bv);
    const int wi = wave_min_int(bv == w ? bi : 0x7fffffff);
    if ((wi & 63) == lane) alive &= ~(1u << (wi >> 6));
    const double wp = __shfl(bp, wi & 63);
    if (lane == k) {
      sel_v = wp;
      sel_i = wi;
    }
    sum += wp;
  }
  if (lane < a.K) {
    if (a.renorm) sel_v /= fmax(sum, 1e-20);
    Elem<TO>::store(static_cast<TO*>(a.topv) + static_cast<size_t>(t) * a.K + lane, static_cast<float>(sel_v * a.scale));
    a.topi[static_cast<size_t>(t) * a.K + lane] = sel_i;
  }
}

template <typename TL, typename TO>
static int launch_select(const SelectArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((gate_select_kernel<TL, TO>), dim3((a.T + kSelWaves - 1) / kSelWaves), dim3(kSelWaves * 64), 0, st, a);
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
  SP_REQUIRE(group_score == SPARSE_HIP_GROUP_MAX || group_score == SPARSE_HIP_GROUP_TOP2, "gate_select: unknown group score %d", group_score);
  SP_REQUIRE(n_group >= 1 && n_group <= kSelMaxGroups && E % n_group == 0, "gate_select: n_group=%d must divide E=%d and be at most %d", n_group, E, kSelMaxGroups);
  SP_REQUIRE(topk_group >= 1 && topk_group <= n_group, "gate_select: topk_group=%d outside [1,%d]", topk_group, n_group);
  SP_REQUIRE(K <= topk_group * (E / n_group), "gate_select: K=%d exceeds the %d experts of %d groups", K, topk_group * (E / n_group), topk_group);
  SP_REQUIRE(T >= 0, "gate_select: T=%d", T);
  if (T == 0) return SPARSE_HIP_OK;
  SP_REQUIRE(logits_dev && topv_dev && topi_dev, "gate_select: NULL pointer");
  const SelectArgs a = {logits_dev, bias_dev, topv_dev, topi_dev, T, E, K, score == SPARSE_HIP_SCORE_SIGMOID,
                        n_group, topk_group, group_score == SPARSE_HIP_GROUP_TOP2, renorm, scale};
  hipStream_t st = as_stream(stream);
  if (logits_dtype == SPARSE_HIP_BF16) return launch_select<uint16_t>(a, out_dtype, st);
  if (logits_dtype == SPARSE_HIP_F16) return launch_select<f16_t>(a, out_dtype, st);
  return launch_select<float>(a, out_dtype, st);
}
