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
// They are found in 32 bits and certified: every choice carries a bound on its
// error, and where two that decide something lie closer than their bounds, the
// few candidates are ranked again in 64 bits (route_scores_64 where a group's
// value is in doubt).  Logits need no certificate.
//
// A lane holds a run of experts of one group in registers, so group values are
// shuffles.  The picks: the k-th largest of the 32 lanes' maxima is no larger
// than the k-th choice, so only what reaches it can matter, usually k to 2 k
// experts; these are ranked against each other, at most two per lane.
//
// Small batches are bound by the launch (one token of 512 to 4096 tokens of 512
// experts: 6 to 6.5 us a call), large ones by instructions: 16384 fp32 tokens of 256
// experts in 8 groups with a bias take 21 to 27 us, about 1000 warp instructions a
// token at 0.75 per clock, where their 18 MB would take 2.7.  The whole in 64
// bits, expert by expert in shared memory with top_k rounds of an argmax, took
// 72 us for these and 31 for the 4096.
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

// the warp's largest value, NaN aside, in one instruction
__device__ __forceinline__ float redux_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
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

// The whole of a token in 64 bits, expert by expert in shared memory: for what
// the 32-bit path leaves open, for rows with fewer experts than picks, and for
// scores below fp32's range.
template <int TYPE>
__device__ __noinline__ void route_scores_64(const RouteArgs& a, long long t, double* c) {
  const int lane = threadIdx.x & 31;
  const size_t row = (size_t)t * a.row_stride;
  double m = -INFINITY;
  for (int e = lane; e < a.E; e += 32) m = fmax(m, (double)load_logit<TYPE>(a.logits, row + e));
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
    a.ids[(size_t)t * a.k + lane] = (uint32_t)my_id;
    a.weights[(size_t)t * a.k + lane] = (float)(mine * (double)a.scale);
  }
  if (lane == 0 && a.mass) a.mass[t] = (float)mass;
}

// 1 / (1 + exp(-l)) from the approximate power of two and reciprocal: within
// (2 + 1.173 |l|) + 1.5 ulp; for choices that carry a bound only.
__device__ __forceinline__ float rough_sigmoid(float l) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(l * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}

constexpr int kCand = 64;   // candidates ranked at once

// NV: experts per lane, at least a.chunk.  Lane l holds experts [base, base +
// count) of group l / a.lanes (lanes behind the last group hold none); runs
// rise with the lane, so a lower lane or place is a lower expert.
template <int TYPE, int NV>
__global__ void __launch_bounds__(kRouteWarps * 32) route_scores_kernel(const __grid_constant__ RouteArgs a) {
  __shared__ int s_id[kRouteWarps][kCand];
  __shared__ alignas(16) float s_key[kRouteWarps][kCand];
  extern __shared__ double route_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = (long long)blockIdx.x * kRouteWarps + warp;
  pdl_wait();
  if (t >= a.tokens) return;
  double* c64 = route_smem + (size_t)warp * a.E;
  const size_t row = (size_t)t * a.row_stride;
  const int size = a.E / a.groups, grp = lane / a.lanes, sub = lane % a.lanes;
  const int base = grp * size + sub * a.chunk;
  const int count = grp < a.groups ? max(0, min(a.chunk, size - sub * a.chunk)) : 0;

  float l[NV];
  if (a.vec) {
    // whole runs of whole 16-byte vectors
    constexpr int PER = TYPE == 0 ? 4 : 8;
#pragma unroll
    for (int i = 0; i < NV; i += PER) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (i < count) v = *reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(a.logits) +
                                                        (row + base + i) * (TYPE == 0 ? 4 : 2));
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < PER && i + e < NV; ++e) {
        if constexpr (TYPE == 0) l[i + e] = __uint_as_float(w[e]);
        if constexpr (TYPE == 1) l[i + e] = __uint_as_float(e & 1 ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16);
        if constexpr (TYPE == 2)
          l[i + e] = __half2float(__ushort_as_half((unsigned short)(w[e >> 1] >> (16 * (e & 1)))));
        if (i + e >= count) l[i + e] = -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) l[i] = i < count ? load_logit<TYPE>(a.logits, row + base + i) : -INFINITY;
  }
  bool bad = false;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    bad |= !(l[i] < INFINITY);
    if (!(l[i] > lowest<TYPE>())) l[i] = -INFINITY;
    m = fmaxf(m, l[i]);
  }
  if (__any_sync(kAll, bad)) {
    if (lane < a.k) {
      a.ids[(size_t)t * a.k + lane] = 0;
      a.weights[(size_t)t * a.k + lane] = 0.0f;
    }
    if (lane == 0) {
      if (a.mass) a.mass[t] = 0.0f;
      atomicOr(a.status, kStatusNonFinite);
    }
    return;
  }
  m = redux_max(m);
  const bool scored = a.bias != nullptr || (a.pair && a.groups > 1);   // group or picks by scores
  float sum = 1.0f, inv = 1.0f;
  if (!a.sigmoid) {
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) sum += expf(l[i] - m);
    sum = warp_sum(sum);
    inv = 1.0f / sum;
  }
  // How far a choice may be off, S being the token's largest score.  Sigmoid:
  // rough_sigmoid's exponential is off by 2 + 1.173 |l| ulp, which counts by
  // exp(-l) / (1 + exp(-l)), its reciprocal by 1 ulp, the sum by half of one;
  // s (2 + 1.173 |l|) is largest at the largest logit m for negative ones, and
  // s |l| / (1 + exp(l)) under 0.28 for positive ones: under
  // S (6.5e-7 + 1.5e-7 max(-m, 0)).  Softmax: the exponential of a rounded
  // difference d (|d| exp(-|d|) is under 0.37), a sum of NV + 5 additions whose
  // terms are off by |d| half-ulps each (their mean |d| is under log E), a
  // reciprocal and a product: under (NV + 40) 6e-8 S.  Adding the bias: under
  // 6e-8 of the choice.
  float key[NV], kmax = -INFINITY, cabs = 0.0f;
  if (!scored) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      key[i] = l[i];
      kmax = fmaxf(kmax, l[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) key[i] = l[i];
    if (a.sigmoid) {
#pragma unroll
      for (int i = 0; i < NV; ++i) key[i] = rough_sigmoid(key[i]);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) key[i] = expf(key[i] - m) * inv;
    }
    if (a.bias) {
      if (a.vec) {
#pragma unroll
        for (int i = 0; i < NV; i += 4) {
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (i < count) v = *reinterpret_cast<const float4*>(a.bias + base + i);
          key[i] += v.x;
          if (i + 1 < NV) key[i + 1] += v.y;
          if (i + 2 < NV) key[i + 2] += v.z;
          if (i + 3 < NV) key[i + 3] += v.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) key[i] += i < count ? a.bias[base + i] : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      // masked, or a bias that is not finite: not available
      const bool there = l[i] > -INFINITY && fabsf(key[i]) < INFINITY;
      cabs = there ? fmaxf(cabs, fabsf(key[i])) : cabs;
      key[i] = there ? key[i] : -INFINITY;
      kmax = fmaxf(kmax, key[i]);
    }
  }
  float bound = 0.0f;
  if (scored) {
    const float rel = a.sigmoid ? 6.5e-7f + 1.5e-7f * fmaxf(-m, 0.0f) : (NV + 40) * 6e-8f;
    const float most = a.sigmoid ? fminf(1.0f, 1.01f * __expf(m)) : inv;
    bound = rel * most + 1.3e-7f * redux_max(cabs) + 1e-37f;
  }
  bool doubt = false;
  if (a.groups > 1) {
    float v1 = kmax, v2 = -INFINITY;
    if (a.pair) {
      bool seen = false;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const bool top = !seen && key[i] == kmax;
        seen |= top;
        if (!top) v2 = fmaxf(v2, key[i]);
      }
    }
    for (int o = 1; o < a.lanes; o <<= 1) {
      const float w1 = __shfl_xor_sync(kAll, v1, o), w2 = __shfl_xor_sync(kAll, v2, o);
      v2 = fmaxf(fminf(v1, w1), fmaxf(v2, w2));
      v1 = fmaxf(v1, w1);
    }
    float value = v1;
    if (a.pair && v2 > -INFINITY) value = v1 + v2;
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const float o = __shfl_sync(kAll, value, g * a.lanes);
      rank += o > value || (o == value && g < grp);
    }
    const bool kept = rank < a.top_groups && count > 0;
    if (scored) {
      // the worst group kept against the best one left
      const float in = redux_max(grp < a.groups && rank < a.top_groups ? -value : -INFINITY);
      const float out = redux_max(grp < a.groups && rank >= a.top_groups ? value : -INFINITY);
      doubt = !(-in - out > 4.0f * bound + 1.3e-7f * fabsf(out)) && out > -INFINITY;
    }
    if (!kept) {
      kmax = -INFINITY;
#pragma unroll
      for (int i = 0; i < NV; ++i) key[i] = -INFINITY;
    }
    // without a bias the picks go by the logits
    if (!a.bias && a.pair && kept) {
      kmax = -INFINITY;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (key[i] > -INFINITY) key[i] = l[i];
        kmax = fmaxf(kmax, key[i]);
      }
    }
  }
  const float slack = a.bias ? bound : 0.0f;   // of a pick's key
  // the k-th largest of the lanes' maxima
  float theta = kmax;
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
    for (int o = n >> 1; o > 0; o >>= 1) {
      const float p = __shfl_xor_sync(kAll, theta, o);
      const bool down = (lane & n) == 0;   // falling runs
      theta = ((lane & o) == 0) == down ? fmaxf(theta, p) : fminf(theta, p);
    }
  theta = __shfl_sync(kAll, theta, a.k - 1) - 2.0f * slack;
  uint64_t mask = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) mask |= (uint64_t)(key[i] >= theta && key[i] > -INFINITY) << i;
  int incl = __popcll(mask);
  const int own = incl;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(kAll, incl, o);
    if (lane >= o) incl += up;
  }
  const int n = __shfl_sync(kAll, incl, 31);
  if (doubt || n > kCand || n < a.k) {
    route_scores_64<TYPE>(a, t, c64);
    return;
  }
  {
    int at = incl - own;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (mask >> i & 1) {
        s_id[warp][at] = base + i;
        s_key[warp][at++] = key[i];
      }
  }
  __syncwarp();
  // Rank of candidate lane (and lane + 32), lower places first among equals;
  // then everything in that order.
  const float k0 = lane < n ? s_key[warp][lane] : -INFINITY, k1 = lane + 32 < n ? s_key[warp][lane + 32] : -INFINITY;
  int r0 = 0, r1 = 0;
  for (int i = 0; i < n; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(&s_key[warp][i]);
    const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e < n) {
        r0 += i + e < lane ? o[e] >= k0 : o[e] > k0;
        if (n > 32) r1 += i + e < lane + 32 ? o[e] >= k1 : o[e] > k1;
      }
  }
  auto place = [&]() {
    const int i0 = lane < n ? s_id[warp][lane] : 0, i1 = lane + 32 < n ? s_id[warp][lane + 32] : 0;
    __syncwarp();
    if (lane < n) s_id[warp][r0] = i0;
    if (lane + 32 < n) s_id[warp][r1] = i1;
  };
  place();
  if (lane < n) s_key[warp][r0] = k0;
  if (lane + 32 < n) s_key[warp][r1] = k1;
  __syncwarp();
  if (slack > 0.0f) {
    const bool close = lane < a.k && lane + 1 < n && !(s_key[warp][lane] - s_key[warp][lane + 1] > 2.0f * slack);
    if (__any_sync(kAll, close)) {
      // two picks closer than their bounds: the candidates again in 64 bits
      double sum64 = 1.0;
      if (!a.sigmoid) {
        double s = 0.0;
        for (int i = 0; i < count; ++i) {
          const float x = load_logit<TYPE>(a.logits, row + base + i);
          if (x > lowest<TYPE>()) s += exp((double)x - (double)m);
        }
        sum64 = warp_sum_d(s);
      }
      auto choice = [&](int at, int& id) -> double {
        if (at >= n) return 0.0;
        id = s_id[warp][at];
        const double x = load_logit<TYPE>(a.logits, row + id);
        return (a.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - (double)m) / sum64) + (double)a.bias[id];
      };
      int i0 = 0, i1 = 0;
      const double c0 = choice(lane, i0), c1 = choice(lane + 32, i1);
      r0 = r1 = 0;
      for (int i = 0; i < n; ++i) {
        const double o = __shfl_sync(kAll, i < 32 ? c0 : c1, i & 31);
        const int oi = s_id[warp][i];
        r0 += o > c0 || (o == c0 && oi < i0);
        r1 += o > c1 || (o == c1 && oi < i1);
      }
      place();
      __syncwarp();
    }
  }
  const int id = lane < a.k ? s_id[warp][lane] : 0;
  const float lg = lane < a.k ? load_logit<TYPE>(a.logits, row + id) : 0.0f;
  float s = 0.0f;
  if (lane < a.k) s = a.sigmoid ? 1.0f / (1.0f + expf(-lg)) : expf(lg - m) / sum;
  const float mass = warp_sum(s);
  // a score that fp32 does not hold (a bias can pick it): of no weight beside a
  // large mass, but a small one brings it back into range
  const bool under = a.renorm && __any_sync(kAll, lane < a.k && s < 1e-36f);
  if (!(mass > 1e-30f) || (under && mass < 0.1f)) {
    route_scores_64<TYPE>(a, t, c64);
    return;
  }
  if (lane < a.k) {
    a.ids[(size_t)t * a.k + lane] = (uint32_t)id;
    a.weights[(size_t)t * a.k + lane] = (a.renorm ? s / mass : s) * a.scale;
  }
  if (lane == 0 && a.mass) a.mass[t] = mass;
}

template <int TYPE>
cudaError_t launch_type(const RouteArgs& a, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((a.tokens + kRouteWarps - 1) / kRouteWarps));
  cfg.blockDim = dim3(kRouteWarps * 32);
  cfg.dynamicSmemBytes = (size_t)kRouteWarps * a.E * sizeof(double);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (a.chunk <= 1) return cudaLaunchKernelEx(&cfg, route_scores_kernel<TYPE, 1>, a);
  if (a.chunk <= 2) return cudaLaunchKernelEx(&cfg, route_scores_kernel<TYPE, 2>, a);
  if (a.chunk <= 4) return cudaLaunchKernelEx(&cfg, route_scores_kernel<TYPE, 4>, a);
  if (a.chunk <= 8) return cudaLaunchKernelEx(&cfg, route_scores_kernel<TYPE, 8>, a);
  if (a.chunk <= 16) return cudaLaunchKernelEx(&cfg, route_scores_kernel<TYPE, 16>, a);
  if (a.chunk <= 32) return cudaLaunchKernelEx(&cfg, route_scores_kernel<TYPE, 32>, a);
  return cudaLaunchKernelEx(&cfg, route_scores_kernel<TYPE, 64>, a);
}

}  // namespace

cudaError_t launch_route_scores(const RouteArgs& args, cudaStream_t s, uint64_t* launches) {
  RouteArgs a = args;
  // lanes of a group: the largest power of two that leaves one for every group
  a.lanes = 32;
  while (a.lanes * a.groups > 32) a.lanes >>= 1;
  const int size = a.E / a.groups, per = a.type == 0 ? 4 : 8;
  const size_t es = a.type == 0 ? 4 : 2;
  a.chunk = (size + a.lanes - 1) / a.lanes;
  a.vec = size == a.chunk * a.lanes && (reinterpret_cast<uintptr_t>(a.bias) & 15) == 0 && a.chunk % per == 0 &&
          ((reinterpret_cast<uintptr_t>(a.logits) | (a.tokens > 1 ? a.row_stride * es : 0)) & 15) == 0;
  if (launches) *launches += 1;
  if (a.type == 0) return launch_type<0>(a, s);
  if (a.type == 1) return launch_type<1>(a, s);
  return launch_type<2>(a, s);
}

}  // namespace osm
