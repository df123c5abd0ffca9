// osm_route.cu -- the choice of experts from router logits in the forms the
// softmax top-k router of osm_router.cu does not cover: sigmoid scores, a bias
// that balances the load, groups of experts, masked experts, a scale on the
// weights (osm_route_scores, osm_moe_route_scores).
//
// One warp per token.  For token t with logits l_e:
//   s_e = exp(l_e - max l) / sum exp(l - max l)   or   1 / (1 + exp(-l_e))
//   c_e = s_e + b_e                               (the choice; b: balance bias)
//   value of a group = best c, or the sum of its two best
//   the top_groups groups of largest value stay, then the top_k experts of
//   largest c among them; every tie goes to the lower index
//   w_j = s of pick j; mass = sum w_j; w_j /= mass (renormalize); w_j *= scale
// An expert whose logit is -infinity or its type's lowest finite value is
// masked: it is never available, in a group or as a pick.  Without a bias the
// choice is the logit itself, which orders experts as their scores do and
// does not saturate; a group's sum of two is of scores in every case.
//
// The picks are those of the formula in 64 bits: two choices that 32 bits
// cannot tell apart (a sigmoid near a border, a bias that nearly cancels a
// difference of scores) would otherwise depend on the order of operations.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "osm_common.cuh"
#include "osm_kernels.cuh"

namespace osm {
namespace {

constexpr uint32_t kAll = 0xFFFFFFFFu;
constexpr int kRouteWarps = 4;

template <int TYPE>
__device__ __forceinline__ float load_logit(const void* p, size_t i) {
  if constexpr (TYPE == 0) return static_cast<const float*>(p)[i];
  if constexpr (TYPE == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  if constexpr (TYPE == 2) return __half2float(static_cast<const __half*>(p)[i]);
}
// The lowest finite value of the logits' type: at or below it an expert is masked.
template <int TYPE>
__device__ __forceinline__ float lowest() {
  return TYPE == 0 ? -3.402823466e38f : TYPE == 1 ? -3.389531390e38f : -65504.0f;
}

__device__ __forceinline__ double warp_max_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

template <int TYPE>
__global__ void __launch_bounds__(kRouteWarps * 32) route_scores_kernel(const RouteArgs a) {
  const int lane = threadIdx.x & 31;
  const long long t = (long long)blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
  if (t >= a.tokens) return;
  extern __shared__ double route_smem[];
  double* c = route_smem + (size_t)(threadIdx.x >> 5) * a.E;  // choice of each expert
  const size_t row = (size_t)t * a.row_stride;
  uint32_t* ids = a.ids + (size_t)t * a.k;
  float* w = a.weights + (size_t)t * a.k;

  bool bad = false;
  double m = -INFINITY;
  for (int e = lane; e < a.E; e += 32) {
    const float l = load_logit<TYPE>(a.logits, row + e);
    bad |= isnan(l) || l == INFINITY;
    m = fmax(m, (double)l);
  }
  if (__any_sync(kAll, bad)) {
    for (int j = lane; j < a.k; j += 32) {
      ids[j] = 0;
      w[j] = 0.0f;
    }
    if (lane == 0) {
      if (a.mass) a.mass[t] = 0.0f;
      atomicOr(a.status, kStatusNonFinite);
    }
    return;
  }
  m = warp_max_d(m);
  double sum = 1.0;
  if (!a.sigmoid) {
    double s = 0.0;
    for (int e = lane; e < a.E; e += 32) {
      const float l = load_logit<TYPE>(a.logits, row + e);
      if (l > lowest<TYPE>()) s += exp((double)l - m);
    }
    sum = warp_sum_d(s);
  }
  auto score = [&](float l) -> double {
    if (!(l > lowest<TYPE>())) return 0.0;
    return a.sigmoid ? 1.0 / (1.0 + exp(-(double)l)) : exp((double)l - m) / sum;
  };
  for (int e = lane; e < a.E; e += 32) {
    const float l = load_logit<TYPE>(a.logits, row + e);
    const double x = a.bias ? score(l) + (double)a.bias[e] : (double)l;
    c[e] = l > lowest<TYPE>() && isfinite(x) ? x : -INFINITY;
  }
  __syncwarp();
  if (a.groups > 1) {
    const int size = a.E / a.groups;
    double v = -INFINITY;
    if (lane < a.groups) {
      double second = -INFINITY;
      for (int i = 0; i < size; ++i) {
        const double x = c[lane * size + i];
        if (x > v) {
          second = v;
          v = x;
        } else if (x > second) {
          second = x;
        }
      }
      if (a.pair && v > -INFINITY) {
        if (!a.bias) v = score((float)v);
        if (second > -INFINITY) v += a.bias ? second : score((float)second);
      }
    }
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const double o = __shfl_sync(kAll, v, g);
      rank += o > v || (o == v && g < lane);
    }
    __syncwarp();
    if (lane < a.groups && rank >= a.top_groups)
      for (int i = 0; i < size; ++i) c[lane * size + i] = -INFINITY;
    __syncwarp();
  }
  // k times the best; unavailable experts (all of value -infinity) come last, lowest index first
  double mine = 0.0;
  int my_id = 0;
  for (int j = 0; j < a.k; ++j) {
    double best = 0.0;
    int at = a.E;  // E: nothing left in this lane
    for (int e = lane; e < a.E; e += 32) {
      const double x = c[e];
      if (!isnan(x) && (at == a.E || x > best)) {
        best = x;
        at = e;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ob = __shfl_xor_sync(kAll, best, o);
      const int oa = __shfl_xor_sync(kAll, at, o);
      if (oa < a.E && (at == a.E || ob > best || (ob == best && oa < at))) {
        best = ob;
        at = oa;
      }
    }
    __syncwarp();
    if (lane == 0) c[at] = NAN;  // taken
    __syncwarp();
    if (lane == j) {
      my_id = at;
      mine = best > -INFINITY ? score(load_logit<TYPE>(a.logits, row + at)) : 0.0;
    }
  }
  const double mass = warp_sum_d(mine);
  if (lane == 0 && !(mass > 0.0)) atomicOr(a.status, kStatusBadMass);
  if (a.renorm) mine = mass > 0.0 ? mine / mass : 0.0;
  if (lane < a.k) {
    ids[lane] = (uint32_t)my_id;
    w[lane] = (float)(mine * (double)a.scale);
  }
  if (lane == 0 && a.mass) a.mass[t] = (float)mass;
}

}  // namespace

cudaError_t launch_route_scores(const RouteArgs& a, cudaStream_t s, uint64_t* launches) {
  const dim3 grid((unsigned)((a.tokens + kRouteWarps - 1) / kRouteWarps)), block(kRouteWarps * 32);
  const size_t sm = (size_t)kRouteWarps * a.E * sizeof(double);
  if (a.type == 0) route_scores_kernel<0><<<grid, block, sm, s>>>(a);
  else if (a.type == 1) route_scores_kernel<1><<<grid, block, sm, s>>>(a);
  else route_scores_kernel<2><<<grid, block, sm, s>>>(a);
  if (launches) *launches += 1;
  return cudaGetLastError();
}

}  // namespace osm
