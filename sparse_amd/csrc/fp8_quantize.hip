// Rows to e4m3 with a power-of-two scale for each run of 128 values.
#include "fp8.h"

namespace sparse {

constexpr int kQzThreads = 256;
constexpr int kQzLane = 8;                       // values per lane: 16 lanes make a run
constexpr int kQzRuns = kQzThreads * kQzLane / kF8Block;

// kVec: rows start on 16-byte boundaries and K is a multiple of 8
template <typename T, bool kVec>
__global__ __launch_bounds__(kQzThreads) void f8_quantize_kernel(const T* __restrict__ x, int64_t runs, int K, int nb,
                                                                 uint8_t* __restrict__ values,
                                                                 uint8_t* __restrict__ scales) {
  const int64_t run = static_cast<int64_t>(blockIdx.x) * kQzRuns + (threadIdx.x >> 4);
  if (run >= runs) return;                       // 16 lanes leave together
  const int64_t t = run / nb;
  const int k = static_cast<int>(run - t * nb) * kF8Block + (threadIdx.x & 15) * kQzLane;
  const T* row = x + t * K;
  float v[kQzLane];
  if (kVec) {
    // a multiple of 8: a lane's eight values are all inside the row or all behind it
    typedef T vec __attribute__((ext_vector_type(kQzLane)));
    vec u = {};
    if (k < K) u = *reinterpret_cast<const vec*>(row + k);
#pragma unroll
    for (int j = 0; j < kQzLane; ++j) {
      const T e = u[j];
      v[j] = Elem<T>::load(&e);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kQzLane; ++j) v[j] = k + j < K ? Elem<T>::load(row + k + j) : 0.f;
  }
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < kQzLane; ++j) m = fmaxf(m, f8_magnitude(v[j]));
  m = f8_row16_max(m);
  const int s = f8_exponent(m);
  const float inv = f8_inverse(s);
  uint2 q;
  q.x = f8_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
  q.y = f8_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
  *reinterpret_cast<uint2*>(values + t * nb * kF8Block + k) = q;
  if ((threadIdx.x & 15) == 0) scales[run] = static_cast<uint8_t>(s + kF8Bias);
}

template <typename T>
static int quantize_as(const void* x, int64_t Trows, int K, void* values, void* scales, hipStream_t st) {
  const int nb = f8_blocks(K);
  const int64_t runs = Trows * nb, grid = (runs + kQzRuns - 1) / kQzRuns;
  SP_REQUIRE(grid < (1ll << 31), "fp8_quantize: too many rows");
  const bool vec = K % kQzLane == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  if (vec)
    hipLaunchKernelGGL((f8_quantize_kernel<T, true>), dim3(static_cast<unsigned>(grid)), dim3(kQzThreads), 0, st,
                       static_cast<const T*>(x), runs, K, nb, static_cast<uint8_t*>(values), static_cast<uint8_t*>(scales));
  else
    hipLaunchKernelGGL((f8_quantize_kernel<T, false>), dim3(static_cast<unsigned>(grid)), dim3(kQzThreads), 0, st,
                       static_cast<const T*>(x), runs, K, nb, static_cast<uint8_t*>(values), static_cast<uint8_t*>(scales));
  SP_LAUNCH_CHECK("f8_quantize_kernel");
  return SPARSE_HIP_OK;
}

int f8_quantize(const void* x, int dtype, int64_t Trows, int K, void* values, void* scales, hipStream_t st) {
  if (dtype == SPARSE_HIP_BF16) return quantize_as<uint16_t>(x, Trows, K, values, scales, st);
  if (dtype == SPARSE_HIP_F16) return quantize_as<f16_t>(x, Trows, K, values, scales, st);
  return quantize_as<float>(x, Trows, K, values, scales, st);
}

}  // namespace sparse
