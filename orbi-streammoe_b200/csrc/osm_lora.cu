// osm_lora.cu -- a Q4 projection shared by every token beside the low-rank
// adapters of many requests (osm_q4_gemv_lora):
//   y[t] = W x[t] + gain[a] B_a (A_a x[t]),   a = adapter[t], none if negative
// W is MLX-affine Q4 (group 64 along the input, w = scale q + bias), A_a is
// [rank][in], B_a [out][rank] in bf16 or fp16; only the first ranks[a] rows of
// an adapter count.  Rows are fp32, bf16 or fp16; every sum is held in fp32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "osm_common.cuh"
#include "osm_kernels.cuh"

namespace osm {
namespace {

template <int TYPE>
__device__ __forceinline__ float load_val(const void* p, size_t i) {
  if constexpr (TYPE == 0) return static_cast<const float*>(p)[i];
  if constexpr (TYPE == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if constexpr (TYPE == 2) return __half2float(static_cast<const __half*>(p)[i]);
}
template <int TYPE>
__device__ __forceinline__ void store_val(void* p, size_t i, float v) {
  if constexpr (TYPE == 0) static_cast<float*>(p)[i] = v;
  if constexpr (TYPE == 1) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  if constexpr (TYPE == 2) static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// The adapter of token t and its rank; rank 0 where there is none.  An index
// past the table counts as none and sets the status bit.
__device__ __forceinline__ int adapter_of(const LoraArgs& a, long long t, int& rank) {
  rank = 0;
  const int id = a.adapter[t];
  if (id < 0) return -1;
  if (id >= a.count) {
    atomicOr(a.status, kStatusBadAdapter);
    return -1;
  }
  rank = a.ranks ? (int)min(a.ranks[id], (uint32_t)a.rank) : a.rank;
  return id;
}

// v[t][j] = gain A_a[j] . x[t]: one block per token, one warp per row j
template <int XT, int AT>
__global__ void __launch_bounds__(256) lora_shrink_kernel(const LoraArgs a) {
  const long long t = blockIdx.x;
  const int lane = threadIdx.x & 31;
  int rank;
  const int id = adapter_of(a, t, rank);
  if (id < 0) return;
  const float gain = a.gain ? a.gain[id] : 1.0f;
  for (int j = threadIdx.x >> 5; j < rank; j += blockDim.x >> 5) {
    const size_t row = (size_t)id * a.a_stride + (size_t)j * a.K;
    float s = 0.0f;
    for (int i = lane; i < a.K; i += 32)
      s = fmaf(load_val<AT>(a.a, row + i), load_val<XT>(a.x, (size_t)t * a.x_stride + i), s);
    s = warp_sum(s);
    if (lane == 0) a.v[(size_t)t * a.rank + j] = gain * s;
  }
}

// y[t][o]: one warp per output; lane l takes words l, l + 32, ... of the row
template <int XT, int AT>
__global__ void __launch_bounds__(256) lora_project_kernel(const LoraArgs a) {
  const int lane = threadIdx.x & 31;
  const long long o = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (o >= a.N) return;
  for (long long t = blockIdx.y; t < a.tokens; t += gridDim.y) {
    const uint32_t* q = a.packed + (size_t)o * (a.K / 8);
    float s = 0.0f;
    for (int w = lane; w < a.K / 8; w += 32) {
      const size_t g = (size_t)o * (a.K / 64) + w / 8;
      const float sc = bf16_bits_to_f32(a.scales[g]), bi = bf16_bits_to_f32(a.biases[g]);
      const uint32_t word = q[w];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        s = fmaf(fmaf(sc, (float)((word >> (4 * i)) & 15u), bi),
                 load_val<XT>(a.x, (size_t)t * a.x_stride + w * 8 + i), s);
    }
    if (a.adapter) {
      int rank;
      const int id = adapter_of(a, t, rank);
      for (int j = lane; j < rank; j += 32)
        s = fmaf(load_val<AT>(a.b, (size_t)id * a.b_stride + (size_t)o * a.rank + j),
                 a.v[(size_t)t * a.rank + j], s);
    }
    s = warp_sum(s);
    if (lane == 0) store_val<XT>(a.y, (size_t)t * a.y_stride + o, s);
  }
}

template <int XT, int AT>
cudaError_t launch(const LoraArgs& a, cudaStream_t s, uint64_t* launches) {
  if (a.adapter) {
    lora_shrink_kernel<XT, AT><<<(unsigned)a.tokens, 256, 0, s>>>(a);
    if (launches) *launches += 1;
  }
  const dim3 grid((unsigned)((a.N + 7) / 8), (unsigned)(a.tokens < 65535 ? a.tokens : 65535));
  lora_project_kernel<XT, AT><<<grid, 256, 0, s>>>(a);
  if (launches) *launches += 1;
  return cudaGetLastError();
}

}  // namespace

size_t lora_workspace(const LoraArgs& a) {
  return a.adapter ? (size_t)a.tokens * a.rank * sizeof(float) : 0;
}

cudaError_t launch_lora(const LoraArgs& a, cudaStream_t s, uint64_t* launches) {
  if (a.adapter && a.a_type == 2) {
    if (a.x_type == 0) return launch<0, 2>(a, s, launches);
    if (a.x_type == 1) return launch<1, 2>(a, s, launches);
    return launch<2, 2>(a, s, launches);
  }
  if (a.x_type == 0) return launch<0, 1>(a, s, launches);
  if (a.x_type == 1) return launch<1, 1>(a, s, launches);
  return launch<2, 1>(a, s, launches);
}

}  // namespace osm
