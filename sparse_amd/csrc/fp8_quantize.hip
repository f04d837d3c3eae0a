// Rows to e4m3 with a power-of-two scale for each run of 128 values:
//   s = the smallest exponent >= -120 with max|x| <= 448 * 2^s over the run's finite values,  q = e4m3(x / 2^s)
//
// One pass: eight lanes hold a run, 16 values each (two 16-byte loads, one 16-byte store a lane; with 8 values a
// lane 13.9 us instead of 12.2), the largest magnitude crosses the eight lanes in registers.  Bound by HBM: 4096
// bf16 rows of 5632, 69 MB read and written in 12.2 us, 5.7 TB/s, above the 4.8 that a copy of 2 GiB reaches, as
// the rows were in the last-level cache.  Small calls are the launch: 333 rows of 1000 in 2.9 us.
#include "fp8.h"
#include "prefill_queue.h"

namespace sparse {

constexpr int kQzThreads = 256;
constexpr int kQzLane = 16;                      // values per lane: 8 lanes make a run
constexpr int kQzLanes = kF8Block / kQzLane;     // lanes per run
constexpr int kQzRuns = kQzThreads * kQzLane / kF8Block;

struct QuantizeArgs {
  const void* x[2];
  int64_t runs[2];
  int32_t K[2], nb[2];
  uint8_t *values[2], *scales[2];
  uint32_t first_blocks;     // workgroups of the first matrix
};

// kVec: rows start on 16-byte boundaries and K is a multiple of 8
// kWide: what has been rounded to 8 bits leaves in bf16, times half its scale, and no scales (for kernels that multiply
// in bf16: 2^-121 to 2^119 times an e4m3 value is a bf16 value)
template <typename T, bool kVec, bool kWide>
__device__ __forceinline__ void quantize_block(const QuantizeArgs& a, uint32_t block) {
  const int which = block >= a.first_blocks;
  if (which) block -= a.first_blocks;
  const int64_t run = static_cast<int64_t>(block) * kQzRuns + threadIdx.x / kQzLanes;
  if (run >= a.runs[which]) return;              // a run's lanes leave together
  const int K = a.K[which], nb = a.nb[which];
  // (a row's number fits 32 bits; so does almost every run's, and the short division is several times faster)
  const int64_t t = run < (1ll << 32) ? static_cast<uint32_t>(run) / static_cast<uint32_t>(nb) : run / nb;
  const int k = static_cast<int>(run - t * nb) * kF8Block + (threadIdx.x % kQzLanes) * kQzLane;
  const T* row = static_cast<const T*>(a.x[which]) + t * K;
  float v[kQzLane];
  if (kVec) {
    // a multiple of 8: eight of a lane's values are all inside the row or all behind it
    typedef T vec __attribute__((ext_vector_type(8)));
    vec u[2] = {};
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (k + 8 * c < K) u[c] = *reinterpret_cast<const vec*>(row + k + 8 * c);
#pragma unroll
    for (int j = 0; j < kQzLane; ++j) {
      const T e = u[j >> 3][j & 7];
      v[j] = Elem<T>::load(&e);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kQzLane; ++j) v[j] = k + j < K ? Elem<T>::load(row + k + j) : 0.f;
  }
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < kQzLane; ++j) m = fmaxf(m, f8_magnitude(v[j]));
  m = f8_row8_max(m);
  const int s = f8_exponent(m);
  const float inv = f8_inverse(s);
  uint32_t q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) q[j] = f8_pack4(v[4 * j] * inv, v[4 * j + 1] * inv, v[4 * j + 2] * inv, v[4 * j + 3] * inv);
  const int64_t at = t * nb * kF8Block + k;
  if constexpr (kWide) {
    const float half = __uint_as_float(static_cast<uint32_t>(s - 1 + kF8Bias) << 23);
    uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.values[which]) + at);
#pragma unroll
    for (int j = 0; j < 2; ++j)
      out[j] = __builtin_bit_cast(uint4, f8_widen8(q[2 * j], q[2 * j + 1], half));
    return;
  }
  *reinterpret_cast<uint4*>(a.values[which] + at) = make_uint4(q[0], q[1], q[2], q[3]);
  if (threadIdx.x % kQzLanes == 0) a.scales[which][run] = static_cast<uint8_t>(s + kF8Bias);
}

template <typename T, bool kVec>
__global__ __launch_bounds__(kQzThreads) void f8_quantize_kernel(const QuantizeArgs a) {
  quantize_block<T, kVec, false>(a, blockIdx.x);
}
// The queue build is 20 workgroups that wait for memory most of their 5 to 10 us; beside the quantiser they cost
// nothing.  They go first.
static_assert(kQzThreads == 256, "the queue build counts on 256 threads");
template <typename T, bool kVec>
__global__ __launch_bounds__(kQzThreads) void f8_quantize_queue_kernel(const QuantizeArgs a, const PfxMapArgs queue, uint32_t queue_blocks) {
  if (blockIdx.x < queue_blocks) prefill_queue_block(queue, blockIdx.x);
  else quantize_block<T, kVec, true>(a, blockIdx.x - queue_blocks);
}

template <typename T>
static int quantize_as(const F8Quantize& a, const F8Quantize& b, const PfxMapArgs* queue, hipStream_t st) {
  QuantizeArgs q = {};
  int64_t blocks[2];
  bool vec = true;
  for (int i = 0; i < 2; ++i) {
    const F8Quantize& m = i ? b : a;
    q.x[i] = m.x;
    q.K[i] = m.K;
    q.nb[i] = f8_blocks(m.K);
    q.runs[i] = m.T * q.nb[i];
    q.values[i] = static_cast<uint8_t*>(m.values);
    q.scales[i] = static_cast<uint8_t*>(m.scales);
    blocks[i] = (q.runs[i] + kQzRuns - 1) / kQzRuns;
    vec = vec && m.K % 8 == 0 && (reinterpret_cast<uintptr_t>(m.x) & 15) == 0;
  }
  SP_REQUIRE(blocks[0] + blocks[1] < (1ll << 31) - (1 << 20), "fp8_quantize: too many rows");
  if (blocks[0] + blocks[1] == 0) return SPARSE_HIP_OK;
  q.first_blocks = static_cast<uint32_t>(blocks[0]);
  const uint32_t extra = queue != nullptr ? queue->nt_gu + queue->nt_dn + 2 : 0;
  const dim3 grid(static_cast<unsigned>(blocks[0] + blocks[1] + extra));
  if (queue != nullptr) {
    if (vec) hipLaunchKernelGGL((f8_quantize_queue_kernel<T, true>), grid, dim3(kQzThreads), 0, st, q, *queue, extra);
    else hipLaunchKernelGGL((f8_quantize_queue_kernel<T, false>), grid, dim3(kQzThreads), 0, st, q, *queue, extra);
    SP_LAUNCH_CHECK("f8_quantize_queue_kernel");
    return SPARSE_HIP_OK;
  }
  if (vec) hipLaunchKernelGGL((f8_quantize_kernel<T, true>), grid, dim3(kQzThreads), 0, st, q);
  else hipLaunchKernelGGL((f8_quantize_kernel<T, false>), grid, dim3(kQzThreads), 0, st, q);
  SP_LAUNCH_CHECK("f8_quantize_kernel");
  return SPARSE_HIP_OK;
}

int f8_quantize(const F8Quantize& a, const F8Quantize& b, int dtype, hipStream_t st) {
  if (dtype == SPARSE_HIP_BF16) return quantize_as<uint16_t>(a, b, nullptr, st);
  if (dtype == SPARSE_HIP_F16) return quantize_as<f16_t>(a, b, nullptr, st);
  return quantize_as<float>(a, b, nullptr, st);
}

int f8_quantize_and_queue(const F8Quantize& a, int dtype, const PfxMapArgs& queue, hipStream_t st) {
  if (dtype == SPARSE_HIP_F16) return quantize_as<f16_t>(a, {}, &queue, st);
  return quantize_as<uint16_t>(a, {}, &queue, st);
}

}  // namespace sparse
