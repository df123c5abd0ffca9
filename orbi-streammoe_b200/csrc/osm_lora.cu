// osm_lora.cu -- a Q4 projection shared by every token beside the low-rank
// adapters of many requests (osm_q4_gemv_lora):
//   y[t] = W x[t] + gain[a] B_a (A_a x[t]),   a = adapter[t], none if negative
// W is MLX-affine Q4 (group 64 along the input, w = scale q + bias), A_a is
// [rank][in], B_a [out][rank] in bf16 or fp16; only the first ranks[a] rows of
// an adapter count.  Rows are fp32, bf16 or fp16.
//
// Up to 4 tokens: lora_decode_kernel (W x on CUDA cores, v[t] = gain A_a x[t]
// in every block, then B_a v).  One token 2048 -> 512 of rank 16: 7.5 us a
// call, of which the launch is the larger part.
//
// Decode batches (up to 256 tokens while the products are fewer than what
// preparing operands costs): lora_v_rows_kernel and, beside it,
// lora_batch_kernel on mma.sync.  32 bf16 tokens 2048 x 2048, 32 adapters of
// rank 16: 10 to 12 us; 256 fp16 tokens 512 -> 2048, 64 adapters of rank up to
// 32: 18.5 us.
//
// More: lora_prep_kernel writes the rows of x as fp16 operands of the tensor
// cores, each row scaled by a power of two so that its largest value lies in
// [2^14, 2^15) (fp32 rows as hi + lo, 22 bits; bf16 and fp16 rows exactly), and
// the sums of their groups of 64 as hi + lo.  lora_gemm_kernel then computes
// D[128 rows of W][N tokens] on tcgen05.  A weight is scale (q - 8) + (bias + 8
// scale): the first term is exact in fp16 (8 + 3 bits), scaled by a power of
// two per row of W; the second, as hi + lo too, multiplies the group sums in
// further steps of the same sum (the two terms nearly cancel where the weights of
// a row are of one sign, so neither may have fewer bits than the sum).  So are
// the adapters: for the distinct adapters of the tile,
// B_a against v with zeros in the tokens of other adapters, in bf16 planes,
// which have the range for any ratio between W, B, x and v.  A tile of many
// requests needs no sorting and no second pass over y.  v is computed by tf32
// matrix products (x as hi + lo for fp32 rows), once for every distinct adapter
// of a tile of tokens, in the prep kernel or, from 4096 tokens on, in
// lora_v_kernel.  4096 bf16 tokens 2048 x 2048, 8 adapters of rank 16: 80 us (62
// without adapters; one after the other with cold caches v takes 17, operands 16,
// products 64); 6001 fp32 tokens, 12 adapters of rank 64: 249 us (53, 28, 188).
//
// What rounds there: fp32 rows hold 22 bits of x (products to about 2^-22) and
// sum 16 products per step; the tensor core's accumulation drops what lies below
// the accumulator's last place, so after every 4 K groups (32 steps) the
// partial sum leaves tensor memory and is added in registers, which keeps the
// loss under 1e-6.  16-bit rows keep one sum in tensor memory (the epilogue has
// no registers for those of 256 tokens), of which a step loses less than 2^-23,
// and hold v in 16 bits: within 2^-17 of the adapters' term, a 32nd of what
// rounding an fp16 y of that size does, where a third plane of v would cost
// every block of adapters another stage.  y is rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "osm_common.cuh"
#include "osm_kernels.cuh"
#include "osm_tcgen05.cuh"

namespace osm {
namespace {

constexpr uint32_t kAllLanes = 0xFFFFFFFFu;

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
// the two values of a 16-bit pair
template <int TYPE>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
  if constexpr (TYPE == 1) {
    a = bf_lo(w);
    b = bf_hi(w);
  } else {
    const float2 f = __half22float2(u2h(w));
    a = f.x;
    b = f.y;
  }
}
// 8 consecutive values; `vec`: the address is 16-byte aligned
template <int TYPE>
__device__ __forceinline__ void load8(const void* p, size_t i, bool vec, float (&v)[8]) {
  if (vec) {
    if constexpr (TYPE == 0) {
      const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
      const float4 a = q[0], b = q[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
      unpack2<TYPE>(a.x, v[0], v[1]);
      unpack2<TYPE>(a.y, v[2], v[3]);
      unpack2<TYPE>(a.z, v[4], v[5]);
      unpack2<TYPE>(a.w, v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = load_val<TYPE>(p, i + e);
  }
}

// Chunks of 64 columns that the groups' sums and the biases take behind K's nk
// groups.  fp32 rows: a column per group, hi and lo in planes of their own.
// 16-bit rows: three columns per group, (c hi, sum hi), (c hi, sum lo), (c lo,
// sum hi), so that one plane holds them.
__host__ __device__ constexpr int bias_chunks(int nk, bool f32) { return ((f32 ? nk : 3 * nk) + 63) / 64; }

// Exponent e of a row whose largest magnitude is m: m 2^-e lies in
// [2^14, 2^15); 0 for a zero row.  Not below -100, so that 2^-e and what it
// multiplies stay in range (rows under 2^-86 then lie lower).
__device__ __forceinline__ int row_exponent(float m) {
  if (!(m > 0.0f)) return 0;
  const int e = (int)(__float_as_uint(m) >> 23) - 127 - 14;
  return max(e, -100);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // |e| <= 126
// The adapter of token t and its rank; -1 and rank 0 where there is none.  An
// index past the table counts as none and sets the status bit.
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

// ---------------------------------------------------------------- v = gain A x

__device__ __forceinline__ void mma_tf32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the same for pairs of 16-bit values, 16 of K
template <int TYPE>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if constexpr (TYPE == 1) {
    mma_bf16_16816(d, a0, a1, a2, a3, b0, b1);
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
// per half, the larger of m and |x| (a NaN in x is passed over, as by fmaxf)
template <int TYPE>
__device__ __forceinline__ uint32_t max16(uint32_t m, uint32_t x) {
  uint32_t r;
  if constexpr (TYPE == 1) asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(x & 0x7FFF7FFFu));
  else asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(x & 0x7FFF7FFFu));
  return r;
}

constexpr int kPrepWarps = 16;
constexpr int kPrepThreads = kPrepWarps * 32;
constexpr int kVCols = 32;   // rows of A per pass of prep_v
constexpr size_t kPrepRed = (size_t)kPrepWarps * 16 * kVCols * 4;   // its partial sums

// 8 consecutive values as loaded: two words of four bytes per value pair for
// fp32, one for 16-bit types
template <int TYPE>
struct Raw8 {
  uint32_t w[TYPE == 0 ? 8 : 4];
};
template <int TYPE>
__device__ __forceinline__ Raw8<TYPE> load_raw8(const void* p, size_t i, bool vec) {
  Raw8<TYPE> r;
  if constexpr (TYPE == 0) {
    float v[8];
    load8<0>(p, i, vec, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) r.w[e] = __float_as_uint(v[e]);
  } else if (vec) {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    r.w[0] = a.x;
    r.w[1] = a.y;
    r.w[2] = a.z;
    r.w[3] = a.w;
  } else {
    const uint16_t* q = static_cast<const uint16_t*>(p) + i;
#pragma unroll
    for (int e = 0; e < 4; ++e) r.w[e] = pack2(q[2 * e], q[2 * e + 1]);
  }
  return r;
}
// values 2 s and 2 s + 1
template <int TYPE>
__device__ __forceinline__ void raw_pair(const Raw8<TYPE>& r, int s, float& a, float& b) {
  if constexpr (TYPE == 0) {
    a = __uint_as_float(r.w[2 * s]);
    b = __uint_as_float(r.w[2 * s + 1]);
  } else {
    unpack2<TYPE>(r.w[s], a, b);
  }
}

// What the blocks for v share: the tile's adapters and, for the matrix kernel,
// the largest magnitude of each row per warp.
struct VShared {
  int id[32], rank[32], list[32], n;
  float max[kPrepWarps][16];
};

// The adapters of TOK tokens from t0 on: each token's, and the first token of
// each distinct one.  All threads.
template <int TOK>
__device__ __forceinline__ void list_adapters(const LoraArgs& a, long long t0, VShared& S) {
  const int tid = threadIdx.x, lane = tid & 31;
  if (tid < TOK) {
    int rank = 0, id = -1;
    if (t0 + tid < a.tokens) id = adapter_of(a, t0 + tid, rank);
    S.id[tid] = id;
    S.rank[tid] = rank;
  }
  __syncthreads();
  if (tid < 32) {
    int base = 0;
    for (int b = 0; b < TOK; b += 32) {
      const int i = b + lane;
      bool first = i < TOK && S.rank[i < TOK ? i : 0] > 0;
      const int mine = i < TOK ? S.id[i] : -1;
#pragma unroll 8
      for (int j = 0; j < b + 32 && j < TOK; ++j) first = first && !(j < i && S.id[j] == mine);
      const uint32_t firsts = __ballot_sync(kAllLanes, first);
      if (first) S.list[base + __popc(firsts & ((1u << lane) - 1u))] = i;
      base += __popc(firsts);
    }
    if (lane == 0) S.n = base;
  }
  __syncthreads();
}

// v of one token and two neighbouring columns, as bf16 planes of v 2^-ex.
__device__ __forceinline__ void store_planes(const LoraArgs& a, long long t, int j, float v0, float v1, int ex) {
  const float sc = pow2(-ex);
  v0 *= sc;
  v1 *= sc;
  uint16_t* at = reinterpret_cast<uint16_t*>(a.v) + (size_t)t * a.v_planes * a.v_stride + j;
  for (int p = 0; p < a.v_planes; ++p) {
    const uint32_t b = pack_bf2(v0, v1);
    *reinterpret_cast<uint32_t*>(at + (size_t)p * a.v_stride) = b;
    v0 -= bf_lo(b);
    v1 -= bf_hi(b);
  }
}

// Below 4096 tokens: tiles of 16, v for the tile's distinct adapters slot, slot
// + v_slots, ...; the 16 warps split K.  v goes out as planes for the matrix
// kernel, [token][plane][v_stride].
template <int XT, int AT>
__device__ __forceinline__ void prep_v(const LoraArgs& a, int block, float* red, VShared& S) {
  constexpr int TOK = 16, KW = kPrepWarps;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // the first adapters of all tiles first: blocks without work lie together
  const int v_tiles = (int)((a.tokens + TOK - 1) / TOK), slot = block / v_tiles;
  const long long t0 = (long long)(block % v_tiles) * TOK;
  list_adapters<TOK>(a, t0, S);
  const int g = lane >> 2, q = lane & 3;
  for (int d = slot; d < S.n; d += a.v_slots) {
    const int id = S.id[S.list[d]], rank = S.rank[S.list[d]];
    const float gain = a.gain ? a.gain[id] : 1.0f;
    const bool in0 = S.id[g] == id, in1 = S.id[g + 8] == id;
    const size_t x0 = (size_t)(t0 + g) * a.x_stride, x1 = (size_t)(t0 + g + 8) * a.x_stride;
    const size_t arow = (size_t)id * a.a_stride;
    for (int j0 = 0; j0 < rank; j0 += kVCols) {
      float acc[kVCols / 8][4] = {};
      float m0 = 0.0f, m1 = 0.0f;
      // K in steps of 32: the thread's 8 values of a row are the k and k + 4
      // positions of four 8-wide matrix steps (the order of K is free as long
      // as both operands use the same one)
#pragma unroll 2
      for (int c = warp; c < a.K / 32; c += KW) {
        const int i = c * 32 + q * 8;
        Raw8<XT> xa{}, xb{};
        Raw8<AT> w[kVCols / 8] = {};
        if (in0) xa = load_raw8<XT>(a.x, x0 + i, a.x_vec);
        if (in1) xb = load_raw8<XT>(a.x, x1 + i, a.x_vec);
#pragma unroll
        for (int n = 0; n < kVCols / 8; ++n) {
          const int j = j0 + n * 8 + g;
          if (j < rank) w[n] = load_raw8<AT>(a.a, arow + (size_t)j * a.K + i, a.a_vec);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          float f[4];
          raw_pair<XT>(xa, s, f[0], f[2]);
          raw_pair<XT>(xb, s, f[1], f[3]);
          m0 = fmaxf(m0, fmaxf(fabsf(f[0]), fabsf(f[2])));
          m1 = fmaxf(m1, fmaxf(fabsf(f[1]), fabsf(f[3])));
          uint32_t h[4], l[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            h[e] = __float_as_uint(f[e]);
            if constexpr (XT == 0) {
              h[e] &= 0xFFFFE000u;
              l[e] = __float_as_uint(f[e] - __uint_as_float(h[e]));
            }
          }
#pragma unroll
          for (int n = 0; n < kVCols / 8; ++n) {
            if (j0 + n * 8 >= rank) continue;
            float b0, b1;
            raw_pair<AT>(w[n], s, b0, b1);
            if constexpr (XT == 0)
              mma_tf32(acc[n], l[0], l[1], l[2], l[3], __float_as_uint(b0), __float_as_uint(b1));
            mma_tf32(acc[n], h[0], h[1], h[2], h[3], __float_as_uint(b0), __float_as_uint(b1));
          }
        }
      }
      m0 = fmaxf(m0, __shfl_xor_sync(kAllLanes, m0, 1));
      m0 = fmaxf(m0, __shfl_xor_sync(kAllLanes, m0, 2));
      m1 = fmaxf(m1, __shfl_xor_sync(kAllLanes, m1, 1));
      m1 = fmaxf(m1, __shfl_xor_sync(kAllLanes, m1, 2));
      if (q == 0) {
        S.max[warp][g] = m0;
        S.max[warp][g + 8] = m1;
      }
#pragma unroll
      for (int n = 0; n < kVCols / 8; ++n) {
        float* at = red + ((size_t)warp * TOK + g) * kVCols + n * 8 + 2 * q;
        *reinterpret_cast<float2*>(at) = make_float2(acc[n][0], acc[n][1]);
        *reinterpret_cast<float2*>(at + 8 * kVCols) = make_float2(acc[n][2], acc[n][3]);
      }
      __syncthreads();
      if (tid < TOK * kVCols / 2) {
        const int r = tid / (kVCols / 2), j = tid % (kVCols / 2) * 2;
        float2 s = make_float2(0.0f, 0.0f);
        float m = 0.0f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const float2 p = *reinterpret_cast<const float2*>(red + ((size_t)w * TOK + r) * kVCols + j);
          s.x += p.x;
          s.y += p.y;
          m = fmaxf(m, S.max[w][r]);
        }
        // whole pieces of 16: zeros behind the adapter's rank
        if (S.id[r] == id && j0 + j < ((rank + 15) & ~15)) {
          s.x = j0 + j < rank ? gain * s.x : 0.0f;
          s.y = j0 + j + 1 < rank ? gain * s.y : 0.0f;
          store_planes(a, t0 + r, j0 + j, s.x, s.y, row_exponent(m));
        }
      }
      __syncthreads();
    }
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ int ld_cluster_i(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Many tokens: tiles of 32, so that a prompt's tokens share the rows of A; K in
// stages of 64 through shared memory (rows of x and A as they are, padded so
// that a warp's 16-byte reads meet all banks), 2 x 2 warps of 16 tokens by 32
// rows of A.  Rows of other adapters are not loaded: they mean nothing in x's
// part and their sums are not stored; neither do rows behind the rank.  A
// cluster of 4 CTAs splits K and adds its sums, in the order of K: with one CTA
// per tile an SM has 4 warps to hide every latency.
template <int XT>
struct VBig {
  static constexpr int TOK = 32, COLS = 64, STAGES = 3, THREADS = 128, KSPLIT = 4;
  static constexpr int XPITCH = XT == 0 ? 272 : 192, APITCH = 192;   // bytes
  static constexpr size_t STAGE = (size_t)TOK * XPITCH + (size_t)COLS * APITCH;
  static constexpr size_t BYTES = STAGES * STAGE;
};
template <int XT, int AT>
__global__ void __launch_bounds__(VBig<XT>::THREADS) lora_v_kernel(const __grid_constant__ LoraArgs a) {
  extern __shared__ uint4 v_smem[];
  __shared__ VShared S;
  unsigned char* const sm = reinterpret_cast<unsigned char*>(v_smem);
  using B = VBig<XT>;
  const int block = (int)blockIdx.x / B::KSPLIT, krank = (int)cluster_rank();
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int v_tiles = (int)((a.tokens + B::TOK - 1) / B::TOK), slot = block / v_tiles;   // as in prep_v
  const long long t0 = (long long)(block % v_tiles) * B::TOK;
  list_adapters<B::TOK>(a, t0, S);
  const int g = lane >> 2, q = lane & 3, wm = warp & 1, wn = warp >> 1;
  const int r0 = wm * 16 + g;
  const int s_lo = a.K / 64 * krank / B::KSPLIT, steps = a.K / 64 * (krank + 1) / B::KSPLIT - s_lo;
  constexpr int XB = XT == 0 ? 4 : 2, XU = XT == 0 ? 16 : 8;   // bytes of a value, 16-byte pieces of a row's stage
  constexpr int NX = B::TOK * XU / B::THREADS, NA = B::COLS * 8 / B::THREADS;   // pieces per thread and stage
  auto copy16 = [&](unsigned char* to, const unsigned char* from, bool vec, int align) {
    if (vec) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(to)), "l"(from) : "memory");
    } else if (align == 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        reinterpret_cast<uint32_t*>(to)[e] = reinterpret_cast<const uint32_t*>(from)[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        reinterpret_cast<uint16_t*>(to)[e] = reinterpret_cast<const uint16_t*>(from)[e];
    }
  };
  for (int d = slot; d < S.n; d += a.v_slots) {
    const int id = S.id[S.list[d]], rank = S.rank[S.list[d]];
    const float gain = a.gain ? a.gain[id] : 1.0f;
    const bool in0 = S.id[r0] == id, in1 = S.id[r0 + 8] == id;
    for (int j0 = 0; j0 < rank; j0 += B::COLS) {
      const bool work = __any_sync(kAllLanes, in0 || in1) && j0 + wn * 32 < rank;
      // this thread's pieces of a stage, null where there is nothing to load
      const unsigned char *px[NX], *pa[NA];
#pragma unroll
      for (int e = 0; e < NX; ++e) {
        const int i = tid + e * B::THREADS, r = i / XU, u = i % XU;
        px[e] = S.id[r] == id
                    ? static_cast<const unsigned char*>(a.x) + ((size_t)(t0 + r) * a.x_stride + s_lo * 64) * XB + u * 16 : nullptr;
      }
#pragma unroll
      for (int e = 0; e < NA; ++e) {
        const int i = tid + e * B::THREADS, r = i >> 3, u = i & 7;
        pa[e] = j0 + r < rank ? static_cast<const unsigned char*>(a.a) +
                                    ((size_t)id * a.a_stride + (size_t)(j0 + r) * a.K + s_lo * 64) * 2 + u * 16 : nullptr;
      }
      auto load = [&](int st) {
        if (st < steps) {
          unsigned char* sx = sm + (size_t)(st % B::STAGES) * B::STAGE;
          unsigned char* sa = sx + (size_t)B::TOK * B::XPITCH;
#pragma unroll
          for (int e = 0; e < NX; ++e) {
            const int i = tid + e * B::THREADS;
            if (px[e]) {
              copy16(sx + (i / XU) * B::XPITCH + (i % XU) * 16, px[e], a.x_vec, XB);
              px[e] += 64 * XB;
            }
          }
#pragma unroll
          for (int e = 0; e < NA; ++e) {
            const int i = tid + e * B::THREADS;
            if (pa[e]) {
              copy16(sa + (i >> 3) * B::APITCH + (i & 7) * 16, pa[e], a.a_vec, 2);
              pa[e] += 128;
            }
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      float acc[4][4] = {};
      float m0 = 0.0f, m1 = 0.0f;
      uint32_t p0 = 0, p1 = 0;               // the same as pairs of 16-bit values
      for (int st = 0; st < B::STAGES - 1; ++st) load(st);
      for (int st = 0; st < steps; ++st) {
        asm volatile("cp.async.wait_group %0;" ::"n"(B::STAGES - 2) : "memory");
        __syncthreads();   // stage st is here, and stage st - 1 has been read by all
        load(st + B::STAGES - 1);
        if (!work) continue;
        const unsigned char* sx = sm + (size_t)(st % B::STAGES) * B::STAGE;
        const unsigned char* sa = sx + (size_t)B::TOK * B::XPITCH;
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {   // 32 of K: this thread's 8 as in prep_v
          const int i = h2 * 32 + q * 8;
          const Raw8<XT> xa = load_raw8<XT>(sx + r0 * B::XPITCH, i, true);
          const Raw8<XT> xb = load_raw8<XT>(sx + (r0 + 8) * B::XPITCH, i, true);
          Raw8<AT> w[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) w[n] = load_raw8<AT>(sa + (wn * 32 + n * 8 + g) * B::APITCH, i, true);
          if constexpr (XT == AT) {
            // one type: its own matrix steps of 16, exact products all the same
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              p0 = max16<XT>(p0, xa.w[e]);
              p1 = max16<XT>(p1, xb.w[e]);
            }
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
              for (int n = 0; n < 4; ++n)
                  mma16<XT>(acc[n], xa.w[2 * s], xb.w[2 * s], xa.w[2 * s + 1], xb.w[2 * s + 1], w[n].w[2 * s],
                            w[n].w[2 * s + 1]);
          } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              float f[4];
              raw_pair<XT>(xa, s, f[0], f[2]);
              raw_pair<XT>(xb, s, f[1], f[3]);
              m0 = fmaxf(m0, fmaxf(fabsf(f[0]), fabsf(f[2])));
              m1 = fmaxf(m1, fmaxf(fabsf(f[1]), fabsf(f[3])));
              uint32_t h[4], l[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                h[e] = __float_as_uint(f[e]);
                if constexpr (XT == 0) {
                  h[e] &= 0xFFFFE000u;
                  l[e] = __float_as_uint(f[e] - __uint_as_float(h[e]));
                }
              }
#pragma unroll
              for (int n = 0; n < 4; ++n) {
                float b0, b1;
                raw_pair<AT>(w[n], s, b0, b1);
                if constexpr (XT == 0)
                  mma_tf32(acc[n], l[0], l[1], l[2], l[3], __float_as_uint(b0), __float_as_uint(b1));
                mma_tf32(acc[n], h[0], h[1], h[2], h[3], __float_as_uint(b0), __float_as_uint(b1));
              }
            }
          }
        }
      }
      if constexpr (XT == AT) {
        float lo, hi;
        unpack2<XT>(p0, lo, hi);
        m0 = fmaxf(lo, hi);
        unpack2<XT>(p1, lo, hi);
        m1 = fmaxf(lo, hi);
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncthreads();   // all stages read: their memory takes the sums
      float* red = reinterpret_cast<float*>(sm);   // [token][COLS], then each token's largest |x|
      m0 = fmaxf(m0, __shfl_xor_sync(kAllLanes, m0, 1));
      m0 = fmaxf(m0, __shfl_xor_sync(kAllLanes, m0, 2));
      m1 = fmaxf(m1, __shfl_xor_sync(kAllLanes, m1, 1));
      m1 = fmaxf(m1, __shfl_xor_sync(kAllLanes, m1, 2));
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        float* at = red + (size_t)r0 * B::COLS + wn * 32 + n * 8 + 2 * q;
        *reinterpret_cast<float2*>(at) = make_float2(acc[n][0], acc[n][1]);
        *reinterpret_cast<float2*>(at + 8 * B::COLS) = make_float2(acc[n][2], acc[n][3]);
      }
      if (wn == 0 && q == 0) {
        red[B::TOK * B::COLS + r0] = m0;
        red[B::TOK * B::COLS + r0 + 8] = m1;
      }
      __syncwarp();
      cluster_sync_all();
      // this CTA's quarter of the tokens, pairs of columns
      constexpr int MINE = B::TOK / B::KSPLIT;
      for (int o = tid; o < MINE * B::COLS / 2; o += B::THREADS) {
        const int r = krank * MINE + o / (B::COLS / 2), c = o % (B::COLS / 2) * 2, j = j0 + c;
        if (S.id[r] != id || j >= ((rank + 15) & ~15)) continue;   // whole pieces of 16: zeros behind the rank
        float v0 = 0.0f, v1 = 0.0f, m = 0.0f;
#pragma unroll
        for (int z = 0; z < B::KSPLIT; ++z) {
          const uint32_t at = map_rank(smem_addr(red), (uint32_t)z);
          v0 += ld_cluster(at + (uint32_t)(r * B::COLS + c) * 4);
          v1 += ld_cluster(at + (uint32_t)(r * B::COLS + c) * 4 + 4);
          m = fmaxf(m, ld_cluster(at + (uint32_t)(B::TOK * B::COLS + r) * 4));
        }
        store_planes(a, t0 + r, j, j < rank ? gain * v0 : 0.0f, j + 1 < rank ? gain * v1 : 0.0f, row_exponent(m));
      }
      __syncwarp();
      cluster_sync_all();   // read by all before the next sums
    }
  }
}

// ---------------------------------------------------------------- x as operands

// fp16 planes of one row, TPR threads per row: a warp where there are rows
// enough to fill the GPU, else a block (one trip to memory for a row of 2048
// values instead of eight).  A thread keeps its first vectors in registers
// between the maximum and the conversion.
template <int XT, int TPR>
__device__ __forceinline__ void prep_row(const LoraArgs& a, long long t) {
  constexpr int PB = XT == 0 ? 2 : 1, KEEP = TPR == 32 ? 4 : 1;
  __shared__ float s_max[kPrepWarps];
  const int lane = threadIdx.x % TPR;
  const bool live = t < a.tokens;
  const size_t row = (size_t)t * a.x_stride;
  const int row_in = (int)(t % a.NT), nk = a.K >> 6, nkp = nk + bias_chunks(nk, XT == 0);
  unsigned char* tile = a.planes + (size_t)(t / a.NT) * nkp * PB * a.NT * 128 + (size_t)row_in * 128;
  float kept[KEEP][8];
  float m = 0.0f;
#pragma unroll
  for (int c = 0; c < KEEP; ++c) {
    const int i = (c * TPR + lane) * 8;
    if (live && i < a.K) {
      load8<XT>(a.x, row + i, a.x_vec, kept[c]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) kept[c][e] = 0.0f;
    }
  }
#pragma unroll
  for (int c = 0; c < KEEP; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(kept[c][e]));
  if (live) {
#pragma unroll 4
    for (int i = (KEEP * TPR + lane) * 8; i < a.K; i += TPR * 8) {
      float v[8];
      load8<XT>(a.x, row + i, a.x_vec, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[e]));
    }
  }
  m = warp_max(m);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPrepWarps; ++w) m = fmaxf(m, s_max[w]);
  }
  const int ex = row_exponent(m);
  if (lane == 0) a.ex[t] = ex;
  const float sc = pow2(-ex);
  auto chunk_at = [&](int k, int unit) {
    return tile + (size_t)k * PB * a.NT * 128 + ((unit ^ (row_in & 7)) << 4);
  };
  // column c of the groups' sums
  auto column_at = [&](int c) { return chunk_at(nk + (c >> 6), (c & 63) >> 3) + (c & 7) * 2; };
  // the 8 values from i on and, by 8 threads together, their group's sum
  auto put = [&](int i, const float (&v)[8]) {
    uint32_t hi[4], lo[4];
    float sum = 0.0f;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const float x0 = v[p] * sc, x1 = v[p + 4] * sc;   // the order of the weights' pairs
      sum += x0 + x1;
      const __half2 h = __floats2half2_rn(x0, x1);
      hi[p] = h2u(h);
      if constexpr (PB == 2) {
        const float2 f = __half22float2(h);
        lo[p] = h2u(__floats2half2_rn(x0 - f.x, x1 - f.y));
      }
    }
    unsigned char* at = chunk_at(i >> 6, (i >> 3) & 7);
    *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if constexpr (PB == 2) *reinterpret_cast<uint4*>(at + (size_t)a.NT * 128) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    // whole groups are in or out, so these 8 lanes are all here
    const uint32_t mask = 0xFFu << (threadIdx.x & 24);
    sum += __shfl_xor_sync(mask, sum, 1);
    sum += __shfl_xor_sync(mask, sum, 2);
    sum += __shfl_xor_sync(mask, sum, 4);
    // the first of them store it, a column (or plane) each
    const int part = threadIdx.x & 7;
    if (part < (PB == 2 ? 2 : 3)) {
      const int grp = i >> 6;
      const float x = sum * (1.0f / 64.0f);  // stays below 2^15; the biases carry the 64
      const __half h = __float2half_rn(x), l = __float2half_rn(x - __half2float(h));
      unsigned char* gat = PB == 2 ? column_at(grp) + (size_t)part * a.NT * 128 : column_at(3 * grp + part);
      *reinterpret_cast<__half*>(gat) = part == 1 ? l : h;
    }
  };
#pragma unroll
  for (int c = 0; c < KEEP; ++c) {
    const int i = (c * TPR + lane) * 8;
    if (i < a.K) put(i, kept[c]);
  }
#pragma unroll 4
  for (int i = (KEEP * TPR + lane) * 8; i < a.K; i += TPR * 8) {
    float v[8] = {};
    if (live) load8<XT>(a.x, row + i, a.x_vec, v);
    put(i, v);
  }
  // zeros behind the last group's sum
  for (int c = (PB == 2 ? nk : 3 * nk) + lane; c < (nkp - nk) * 64; c += TPR) {
    unsigned char* at = column_at(c);
    *reinterpret_cast<__half*>(at) = __float2half_rn(0.0f);
    if constexpr (PB == 2) *reinterpret_cast<__half*>(at + (size_t)a.NT * 128) = __float2half_rn(0.0f);
  }
}

__device__ __forceinline__ uint4 load_meta(const LoraArgs& a, const uint16_t* base, int o, int k8);
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i);

// The exponents of 128 rows of W and their biases as operands.  A weight is
// scale (q - 8) + c with c = bias + 8 scale; the exponent is that of the largest
// of 16 |scale|, which keeps the converters' 24 scale in range, and 64 |c| (the
// groups' sums of x are kept as 1/64, so c carries the 64).  Operands
// [stage][pair of columns][row], fp16 pairs: for fp32 rows of x a column per
// group, hi, and lo in a stage of its own; else the three columns per group of
// bias_chunks.  Four threads per row.
template <bool F32>
__device__ __forceinline__ void prep_weights(const LoraArgs& a, int tile) {
  constexpr int PARTS = kPrepThreads / 128;
  const int row = threadIdx.x / PARTS, part = threadIdx.x % PARTS, o = tile * 128 + row;
  const int nk = a.K >> 6, n8 = (nk + 7) / 8, nbk = bias_chunks(nk, F32);
  auto mid = [](float s, float b) { return 64.0f * fmaf(8.0f, s, b); };
  float m = 0.0f;
  if (o < a.N) {
#pragma unroll 4
    for (int k8 = part; k8 < n8; k8 += PARTS) {
      const uint4 sv = load_meta(a, a.scales, o, k8), bv = load_meta(a, a.biases, o, k8);
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const uint32_t sw = word_of(sv, p), bw = word_of(bv, p);
        m = fmaxf(m, fmaxf(16.0f * fabsf(bf_lo(sw)), fabsf(mid(bf_lo(sw), bf_lo(bw)))));
        m = fmaxf(m, fmaxf(16.0f * fabsf(bf_hi(sw)), fabsf(mid(bf_hi(sw), bf_hi(bw)))));
      }
    }
  }
  m = fmaxf(m, __shfl_xor_sync(kAllLanes, m, 1));
  m = fmaxf(m, __shfl_xor_sync(kAllLanes, m, 2));
  const int ew = row_exponent(m);
  if (part == 0) a.ew[o] = ew;
  const float sc = pow2(-ew);
  uint32_t* out = a.wbias + (size_t)tile * (F32 ? 2 : 1) * nbk * 32 * 128 + row;
#pragma unroll 4
  for (int k8 = part; k8 < (F32 ? nbk * 8 : (nbk * 32 + 11) / 12); k8 += PARTS) {
    uint4 sv = make_uint4(0, 0, 0, 0), bv = sv;
    if (o < a.N && k8 < n8) {
      sv = load_meta(a, a.scales, o, k8);
      bv = load_meta(a, a.biases, o, k8);
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t sw = word_of(sv, p), bw = word_of(bv, p);
      const float f0 = mid(bf_lo(sw), bf_lo(bw)) * sc, f1 = mid(bf_hi(sw), bf_hi(bw)) * sc;
      const __half2 h = __floats2half2_rn(f0, f1);
      const float2 f = __half22float2(h);
      const uint32_t hw = h2u(h), lw = h2u(__floats2half2_rn(f0 - f.x, f1 - f.y));
      if constexpr (F32) {
        const int bi = k8 >> 3, col = (k8 & 7) * 4;
        out[(size_t)((bi * 2) * 32 + col + p) * 128] = hw;
        out[(size_t)((bi * 2 + 1) * 32 + col + p) * 128] = lw;
      } else {
        // two groups, six columns: hi0 hi0 | lo0 hi1 | hi1 lo1
        const uint32_t w[3] = {prmt(hw, hw, 0x1010), prmt(lw, hw, 0x7610), prmt(hw, lw, 0x7632)};
        const int at = k8 * 12 + p * 3;
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (at + e < nbk * 32) out[(size_t)(at + e) * 128] = w[e];
      }
    }
  }
}

// The adapters of one tile of the matrix kernel: pieces of 16 rows of each, in
// the order of their first tokens, {adapter, first row | rows from there << 16};
// and each token's first piece and number of pieces (0: no adapter).
__device__ __forceinline__ void prep_list(const LoraArgs& a, int tile) {
  constexpr int kMost = 256;               // tokens of a tile
  __shared__ alignas(16) int s_id[kMost];
  __shared__ int s_goff[kMost], s_sum[kMost / 32];
  const int n = threadIdx.x, lane = n & 31;
  const long long t = (long long)tile * a.NT + n;
  int rank = 0, id = -1;
  if (n < a.NT && t < a.tokens) id = adapter_of(a, t, rank);
  if (rank == 0) id = -1;
  if (n < kMost) s_id[n] = id;
  __syncthreads();
  int first = n;
  if (id >= 0) {
    const int4* ids4 = reinterpret_cast<const int4*>(s_id);
    for (int j = 0; j * 4 < n; ++j) {
      const int4 v = ids4[j];
      const int f = v.x == id ? 0 : v.y == id ? 1 : v.z == id ? 2 : v.w == id ? 3 : 4;
      if (f < 4) {
        first = min(first, j * 4 + f);
        break;
      }
    }
  }
  const int pieces = id >= 0 ? (rank + 15) >> 4 : 0, mine = first == n ? pieces : 0;
  int incl = mine;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const int up = __shfl_up_sync(kAllLanes, incl, s);
    if (lane >= s) incl += up;
  }
  if (n < kMost && lane == 31) s_sum[n >> 5] = incl;
  __syncthreads();
  int base = 0, all = 0;
  for (int w = 0; w < kMost / 32; ++w) {
    if (w < (n >> 5)) base += s_sum[w];
    all += s_sum[w];
  }
  const int goff = base + incl - mine;
  if (n < kMost) s_goff[n] = goff;
  __syncthreads();
  int2* gran = a.gran + (size_t)tile * a.gran_stride;
  for (int i = 0; i < mine; ++i) gran[goff + i] = make_int2(id, i * 16 | (rank - i * 16) << 16);
  if (n < a.NT && t < (a.tokens + 15) / 16 * 16) a.tok[t] = make_int2(id >= 0 ? s_goff[first] : 0, pieces);
  if (n == 0) a.n_gran[tile] = all;
}

// First the blocks for v, then the tiles' lists, then those for W, then rows of
// x, up to the next multiple of 16 (zero rows behind the last).
template <int XT, int AT>
__global__ void __launch_bounds__(kPrepThreads, 2) lora_prep_kernel(const __grid_constant__ LoraArgs a) {
  extern __shared__ uint4 prep_smem[];     // the partial sums of prep_v
  __shared__ VShared s_v;
  // behind lora_v_kernel this one does not wait for it to begin: that kernel has
  // waited for everything before it, and neither reads what the other writes
  if (!a.after_v) pdl_wait();
  pdl_trigger();
  long long b = blockIdx.x;
  if (b < a.v_blocks) {
    prep_v<XT, AT>(a, (int)b, reinterpret_cast<float*>(prep_smem), s_v);
  } else if ((b -= a.v_blocks) < a.l_blocks) {
    prep_list(a, (int)b);
  } else if ((b -= a.l_blocks) < a.w_blocks) {
    prep_weights<XT == 0>(a, (int)b);
  } else {
    b -= a.w_blocks;
    if (a.row_threads == kPrepThreads) {
      prep_row<XT, kPrepThreads>(a, b);
    } else {
      const long long t = b * kPrepWarps + (threadIdx.x >> 5);
      if (t < (a.tokens + 15) / 16 * 16) prep_row<XT, 32>(a, t);
    }
  }
  if (a.after_v) pdl_wait();               // who waits for this kernel has v too
}

// ---------------------------------------------------------------- few tokens

// Up to 4 tokens (8 took 19.5 us here and 13.5 on mma.sync, 2048 x 2048): the
// projection on CUDA cores in fp32, one warp per ROWS rows
// of W and all tokens, lane l the groups l, l + 32, ... of a row.  Bound by
// latency: a launch reads about 2.4 MB for 2048 x 2048.  v is computed by every
// block for itself while that reads little (v_self), which spares a launch;
// otherwise this kernel starts beside the one that computes v and waits for it
// only before the adapters' term.
// x is kept in shared memory in fp32; 16-byte piece c of group g sits at piece
// c ^ (g & 15), so that the lanes of a warp, which read the same piece of 32
// groups, meet all banks.
constexpr int kDecWarps = 8;
constexpr int kDecTokens = 4;
constexpr int kDecSelf = 256;            // tokens by rank of v in shared memory, most
constexpr size_t kDecSmem = 128 << 10;   // x in shared memory, most

template <int XT, int AT, int TT, int ROWS>
__global__ void __launch_bounds__(kDecWarps * 32) lora_decode_kernel(const __grid_constant__ LoraArgs a) {
  extern __shared__ float4 dec_x[];   // [token][K / 4]
  __shared__ float s_v[kDecSelf];     // [token][rank] where this kernel computes v
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.K >> 6, T = (int)a.tokens;
  const int o0 = ((int)blockIdx.x * kDecWarps + warp) * ROWS;
  // without a kernel for v before it this one may start early itself
  if (!a.adapter || a.v_self) pdl_wait();
  for (int i = tid; i < T * G * 8; i += kDecWarps * 32) {
    const int t = i / (G * 8), p = i - t * (G * 8);   // 8 values from 8 p on
    float v[8];
    load8<XT>(a.x, (size_t)t * a.x_stride + p * 8, a.x_vec, v);
    const int g = p >> 3, c = (p & 7) * 2;
    float4* row = dec_x + ((size_t)t * G + g) * 16;
    row[c ^ (g & 15)] = make_float4(v[0], v[1], v[2], v[3]);
    row[(c + 1) ^ (g & 15)] = make_float4(v[4], v[5], v[6], v[7]);
  }
  float acc[ROWS][TT];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[r][t] = 0.0f;
  uint4 w[ROWS][2];
  float sc[ROWS], bi[ROWS];
  auto load_w = [&](int g) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int o = min(o0 + r, a.N - 1);
      const uint32_t* p = a.packed + (size_t)o * (a.K >> 3) + g * 8;
      if (a.w_vec) {
        w[r][0] = __ldg(reinterpret_cast<const uint4*>(p));
        w[r][1] = __ldg(reinterpret_cast<const uint4*>(p) + 1);
      } else {
        w[r][0] = make_uint4(p[0], p[1], p[2], p[3]);
        w[r][1] = make_uint4(p[4], p[5], p[6], p[7]);
      }
      sc[r] = bf16_bits_to_f32(a.scales[(size_t)o * G + g]);
      bi[r] = bf16_bits_to_f32(a.biases[(size_t)o * G + g]);
    }
  };
  if (o0 < a.N && lane < G) load_w(lane);
  __syncthreads();
  if (a.v_self) {
    for (int p = warp; p < T * a.rank; p += kDecWarps) {
      const int t = p / a.rank, j = p - t * a.rank;
      int rank;
      const int id = adapter_of(a, t, rank);
      if (j >= rank) continue;
      const size_t row = (size_t)id * a.a_stride + (size_t)j * a.K;
      float s = 0.0f;
#pragma unroll 8
      for (int k = lane * 8; k < a.K; k += 256) {
        float v[8];
        load8<AT>(a.a, row + k, a.a_vec, v);
        const int g = k >> 6, c = (k >> 2) & 15;
        const float4* xg = dec_x + ((size_t)t * G + g) * 16;
        const float4 x0 = xg[c ^ (g & 15)], x1 = xg[(c + 1) ^ (g & 15)];
        s = fmaf(v[3], x0.w, fmaf(v[2], x0.z, fmaf(v[1], x0.y, fmaf(v[0], x0.x, s))));
        s = fmaf(v[7], x1.w, fmaf(v[6], x1.z, fmaf(v[5], x1.y, fmaf(v[4], x1.x, s))));
      }
      s = warp_sum(s);
      if (lane == 0) s_v[p] = (a.gain ? a.gain[id] : 1.0f) * s;
    }
    __syncthreads();
  }
  if (o0 >= a.N) return;
  for (int g = lane; g < G; g += 32) {
    if (g >= 32) load_w(g);
    const float4* xg = dec_x + (size_t)g * 16;
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      float wf[ROWS][4];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const uint4 v = w[r][c >> 3];
        const uint32_t word = (c >> 1 & 3) == 0 ? v.x : (c >> 1 & 3) == 1 ? v.y : (c >> 1 & 3) == 2 ? v.z : v.w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // 2^23 + q, exactly q after the subtraction
          const float f = __uint_as_float(((word >> (16 * (c & 1) + 4 * e)) & 15u) | 0x4B000000u) - 8388608.0f;
          wf[r][e] = fmaf(sc[r], f, bi[r]);
        }
      }
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        if (t < T) {
          const float4 x = xg[(size_t)t * G * 16 + (c ^ (g & 15))];
#pragma unroll
          for (int r = 0; r < ROWS; ++r)
            acc[r][t] = fmaf(wf[r][3], x.w, fmaf(wf[r][2], x.z, fmaf(wf[r][1], x.y, fmaf(wf[r][0], x.x, acc[r][t]))));
        }
      }
    }
  }
  if (a.adapter) {
    int id[TT], rank[TT];
    float b[ROWS][TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      id[t] = -1;
      rank[t] = 0;
      if (t < T) id[t] = adapter_of(a, t, rank[t]);
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        b[r][t] = lane < rank[t] && o0 + r < a.N
                      ? load_val<AT>(a.b, (size_t)id[t] * a.b_stride + (size_t)(o0 + r) * a.rank + lane) : 0.0f;
    }
    if (!a.v_self) pdl_wait();  // v is complete from here on
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      for (int j = lane; j < rank[t]; j += 32) {
        const float v = a.v_self ? s_v[t * a.rank + j] : __ldcg(a.v + (size_t)t * a.v_stride + j);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const float bv = j == lane ? b[r][t]
                           : o0 + r < a.N
                               ? load_val<AT>(a.b, (size_t)id[t] * a.b_stride + (size_t)(o0 + r) * a.rank + j) : 0.0f;
          acc[r][t] = fmaf(bv, v, acc[r][t]);
        }
      }
    }
  }
  pdl_trigger();
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int t = 0; t < TT; ++t)
      if (t < T) {
        const float s = warp_sum(acc[r][t]);
        if (lane == (r * TT + t) % 32 && o0 + r < a.N) store_val<XT>(a.y, (size_t)t * a.y_stride + o0 + r, s);
      }
}

// ---------------------------------------------------------------- decode batches

// v = gain A x in fp32 on CUDA cores, one warp per ROWS rows of a token's
// adapter: for decode batches, whose tokens seldom share an adapter.  Bound by
// latency (32 tokens of rank 16 from 2048: 6.5 us with cold caches, mostly
// before the batch kernel needs v).  Tiles of 16 tokens that share the reads of
// their adapters were slower throughout: whole calls of 128 bf16 tokens 4096 ->
// 512 with 4 adapters of rank 128 took 57 us against 36, with 128 adapters 64
// against 51; 128 tokens 2048 -> 512 with 8 of rank 64 took 21 against 20.
constexpr int kRowWarps = 4;
template <int XT, int AT, int ROWS>
__global__ void __launch_bounds__(kRowWarps * 32) lora_v_rows_kernel(const __grid_constant__ LoraArgs a) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int chunks = (a.rank + ROWS - 1) / ROWS;
  const long long w = (long long)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  const long long t = w / chunks;
  const int j0 = (int)(w - t * chunks) * ROWS;
  if (t >= a.tokens) return;
  int rank;
  const int id = adapter_of(a, t, rank);
  if (j0 >= rank) return;
  float acc[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) acc[r] = 0.0f;
  const size_t xr = (size_t)t * a.x_stride, ar = (size_t)id * a.a_stride + (size_t)j0 * a.K;
#pragma unroll 4
  for (int k = lane * 8; k < a.K; k += 256) {
    float x[8];
    load8<XT>(a.x, xr + k, a.x_vec, x);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (j0 + r >= rank) break;
      float b[8];
      load8<AT>(a.a, ar + (size_t)r * a.K + k, a.a_vec, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[r] = fmaf(x[e], b[e], acc[r]);
    }
  }
  const float gain = a.gain ? a.gain[id] : 1.0f;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const float s = warp_sum(acc[r]);
    if (lane == r && j0 + r < rank) a.v[(size_t)t * a.v_stride + j0 + r] = gain * s;
  }
}

// A decode batch: W x on mma.sync, 16 MT rows of W by 8 NT tokens per CTA, the
// groups of K dealt to its 8 warps.  A group's sum of (q - 8) x and its sum of
// x are taken exactly as the operands stand (q - 8 in the rows' 16-bit type;
// fp32 rows as three bf16 planes, which hold all 24 bits) and meet scale and
// c = bias + 8 scale in fp32, so no operand is rounded and nothing has to be
// prepared.  For bf16 the left operands are scaled by 2^-10 and 2^-6, so that no
// sum over a group overflows.  A lane's share of a group is 16 consecutive k of a
// row of W (two Q4 words) and of a token: the order of k within a matrix step is
// free as long as both sides agree, so both come straight from memory, each W
// word as the pairs (q_p, q_p+4).  The warps' sums are added in shared memory in
// their order, then B_a v in fp32; v comes from the kernel before, which this one
// waits for only there.
constexpr int kBatWarps = 8;
constexpr int kBatRank = 128;   // the largest rank of any call: v in shared memory

template <int XT, int MT, int NT>
struct BatSmem {
  static constexpr int PITCH = 16 * MT + 4;
  static constexpr size_t BYTES = (size_t)kBatWarps * 8 * NT * PITCH * 4;
};

template <int XT, int AT, int MT, int NT>
__global__ void __launch_bounds__(kBatWarps * 32, MT == 4 ? 1 : 2)
    lora_batch_kernel(const __grid_constant__ LoraArgs a) {
  constexpr int MR = 16 * MT, TOK = 8 * NT, PL = XT == 0 ? 3 : 1, PITCH = BatSmem<XT, MT, NT>::PITCH;
  constexpr int OT = XT == 2 ? 2 : 1;   // type of the operands
  extern __shared__ float4 bat_smem[];
  float* bat_sum = reinterpret_cast<float*>(bat_smem);                    // [warp][token][PITCH]
  float* bat_v = bat_sum + BatSmem<XT, MT, NT>::BYTES / 4;                // [token][v_stride]
  __shared__ int s_id[TOK], s_rank[TOK];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
  const int G = a.K >> 6, row_tiles = (a.N + MR - 1) / MR;
  const int o0 = (int)(blockIdx.x % row_tiles) * MR;
  const long long t0 = (long long)(blockIdx.x / row_tiles) * TOK;
  // without a kernel for v before it this one may start early itself
  if (!a.adapter) pdl_wait();
  if (tid < TOK) {
    int rank = 0, id = -1;
    if (a.adapter && t0 + tid < a.tokens) id = adapter_of(a, t0 + tid, rank);
    s_id[tid] = id;
    s_rank[tid] = rank;
  }
  float acc[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][n][e] = 0.0f;
  const uint32_t ones = XT == 2 ? 0x3C003C00u : 0x3C803C80u;   // 1, or 2^-6 in bf16

  for (int grp = warp; grp < G; grp += kBatWarps) {
    uint32_t w[MT][2][2];
    uint16_t sc[MT][2], bi[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const size_t o = (size_t)min(o0 + 16 * m + 8 * h + g, a.N - 1);
        const uint32_t* p = a.packed + o * (a.K >> 3) + grp * 8 + 2 * q;
        if (a.w_vec) {
          const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
          w[m][h][0] = v.x;
          w[m][h][1] = v.y;
        } else {
          w[m][h][0] = __ldg(p);
          w[m][h][1] = __ldg(p + 1);
        }
        sc[m][h] = __ldg(a.scales + o * G + grp);
        bi[m][h] = __ldg(a.biases + o * G + grp);
      }
    // right operands: [n][plane][pair of k]
    uint32_t xb[NT][PL][8];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const long long t = min(t0 + 8 * n + g, a.tokens - 1);
      const size_t at = (size_t)t * a.x_stride + (size_t)grp * 64 + 16 * q;
      if constexpr (XT == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float f[8];
          load8<0>(a.x, at + 8 * h, a.x_vec, f);
#pragma unroll
          for (int pl = 0; pl < 3; ++pl) {
#pragma unroll
            for (int p = 0; p < 4; ++p)
              xb[n][pl][4 * h + p] = prmt(__float_as_uint(f[p]), __float_as_uint(f[p + 4]), 0x7632);
            if (pl < 2)
#pragma unroll
              for (int e = 0; e < 8; ++e) f[e] -= __uint_as_float(__float_as_uint(f[e]) & 0xFFFF0000u);
          }
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t r[4];
          const uint16_t* p = static_cast<const uint16_t*>(a.x) + at + 8 * h;
          if (a.x_vec) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = p[2 * e] | (uint32_t)p[2 * e + 1] << 16;
          }
          xb[n][0][4 * h] = prmt(r[0], r[2], 0x5410);
          xb[n][0][4 * h + 1] = prmt(r[0], r[2], 0x7632);
          xb[n][0][4 * h + 2] = prmt(r[1], r[3], 0x5410);
          xb[n][0][4 * h + 3] = prmt(r[1], r[3], 0x7632);
        }
      }
    }
    float gs[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int pl = PL - 1; pl >= 0; --pl)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          mma16<OT>(d, ones, ones, ones, ones, xb[n][pl][2 * j], xb[n][pl][2 * j + 1]);
      gs[n][0] = d[0];
      gs[n][1] = d[1];
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      uint32_t l[2][8];   // left operands: [row half][pair of k]
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t v = w[m][h][e >> 2] >> (4 * (e & 3)) & 0x000F000Fu;
          if constexpr (XT == 2) l[h][e] = h2u(__hsub2(u2h(v | 0x64006400u), u2h(0x64086408u)));   // 1024 + q - 1032
          else l[h][e] = bf2_fma(v | 0x43004300u, 0x3A803A80u, 0xBE08BE08u);   // (128 + q) 2^-10 - 136 2^-10
        }
      const float up = XT == 2 ? 1.0f : 1024.0f, upc = XT == 2 ? 1.0f : 64.0f;
      float s[2], c[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float sf = bf16_bits_to_f32(sc[m][h]);
        s[h] = sf * up;
        c[h] = fmaf(8.0f, sf, bf16_bits_to_f32(bi[m][h])) * upc;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int pl = PL - 1; pl >= 0; --pl)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma16<OT>(d, l[0][2 * j], l[1][2 * j], l[0][2 * j + 1], l[1][2 * j + 1], xb[n][pl][2 * j],
                      xb[n][pl][2 * j + 1]);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[m][n][e] = fmaf(s[e >> 1], d[e], fmaf(c[e >> 1], gs[n][e & 1], acc[m][n][e]));
      }
    }
  }
  float* mine = bat_sum + (size_t)warp * TOK * PITCH;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        mine[(8 * n + 2 * q + (e & 1)) * PITCH + 16 * m + 8 * (e >> 1) + g] = acc[m][n][e];
  if (a.adapter) {
    __syncthreads();   // s_rank
    pdl_wait();        // v is complete from here on
    const int stride = (int)a.v_stride;
    for (int i = tid * 4; i < TOK * stride; i += kBatWarps * 128) {
      const int tk = i / stride, j = i - tk * stride;
      if (j < s_rank[tk])   // what lies behind the rank is not used
        *reinterpret_cast<float4*>(bat_v + i) = __ldcg(reinterpret_cast<const float4*>(a.v + (size_t)(t0 + tk) * stride + j));
    }
  }
  __syncthreads();
  const int used = G < kBatWarps ? G : kBatWarps;
#pragma unroll 2
  for (int i = tid; i < MR * TOK; i += kBatWarps * 32) {
    const int r = i % MR, tk = i / MR, o = o0 + r;
    if (o >= a.N || t0 + tk >= a.tokens) continue;
    float y = 0.0f;
    if (used == kBatWarps) {
#pragma unroll
      for (int k = 0; k < kBatWarps; ++k) y += bat_sum[(k * TOK + tk) * PITCH + r];
    } else {
      for (int k = 0; k < used; ++k) y += bat_sum[(k * TOK + tk) * PITCH + r];
    }
    const int rank = s_rank[tk];
    if (rank) {
      const size_t br = (size_t)s_id[tk] * a.b_stride + (size_t)o * a.rank;
      const float* v = bat_v + tk * (int)a.v_stride;
      float z = 0.0f;
      int j = 0;
#pragma unroll 4
      for (; j + 8 <= rank; j += 8) {
        float b[8];
        load8<AT>(a.b, br + j, a.b_vec, b);
        const float4 v0 = *reinterpret_cast<const float4*>(v + j), v1 = *reinterpret_cast<const float4*>(v + j + 4);
        z = fmaf(b[3], v0.w, fmaf(b[2], v0.z, fmaf(b[1], v0.y, fmaf(b[0], v0.x, z))));
        z = fmaf(b[7], v1.w, fmaf(b[6], v1.z, fmaf(b[5], v1.y, fmaf(b[4], v1.x, z))));
      }
      for (; j < rank; ++j) z = fmaf(load_val<AT>(a.b, br + j), v[j], z);
      y += z;
    }
    store_val<XT>(a.y, (size_t)(t0 + tk) * a.y_stride + o, y);
  }
}

// ---------------------------------------------------------------- gemm

// What the prep kernel wrote is read with __ldcg: this kernel starts beside
// that one, so lines of an earlier call could still be in L1.

constexpr int kLgM = 128;                 // rows of W per tile
constexpr int kLgConv = 8;                // converter warps, two groups of four
constexpr int kLgEpi = 8;                 // epilogue warps, two per quarter of the rows
constexpr int kLgThreads = (2 + kLgConv + kLgEpi) * 32;
constexpr int kLgRO = 4;                  // operand stages (one K group each)
constexpr int kLgRQ = 2;                  // Q4 tiles (32 rows of one K group) in flight per converter warp
constexpr int kLgQPitch = 48;             // bytes per row of a Q4 tile: 16-byte reads of 8 rows meet all banks
constexpr size_t kLgA = 16384;            // W's part of a stage, 128 rows of 64 fp16
constexpr size_t kLgX = 32768;            // x's part: 256 tokens of one plane or 128 of two
constexpr size_t kLgStage = kLgA + kLgX;
constexpr size_t kLgQTile = (size_t)32 * kLgQPitch;

// Both operands are in shared memory, which leaves tensor memory to two buffers
// of 256 tokens' sums, so that a tile's epilogue runs beside the next tile's
// products.  By what a stage moves through shared memory (operands of the matrix
// unit, Q4 tiles, converted weights: 800 clocks for 256 tokens) the products of
// 4096 bf16 tokens 2048 x 2048 need 30 us, by their matrix steps 16; they take 64
// on their own (the unit 32 % active, 0.39 instructions per scheduler and clock, 29
// % of the load/store wavefronts), so what a stage waits for is the way of the
// weights: Q4 tile, conversion, operand.  16384 tokens: 285 us the whole call, 214
// without adapters.
template <bool F32>
struct LgCfg {
  static constexpr int PL = F32 ? 2 : 1;        // planes of x
  static constexpr int NMAX = F32 ? 128 : 256;  // tokens per tile
  static constexpr int GROUP = F32 ? 4 : 1 << 30;  // stages per partial sum
  static constexpr int NV = F32 ? 3 : 2;        // bf16 planes of v
};
// Stages that a block of adapters takes in a tile of `tokens`: the nv planes of
// v in one where they fit beside each other (256 rows), else in two; and for fp16
// adapters (`lo`) one for the low part of B, which meets all planes but the last.
// Both hold for 3 planes of up to 128 tokens and 2 of up to 256.
__host__ __device__ constexpr int lora_passes(int nv, int tokens, bool lo) {
  return (nv * tokens <= 256 ? 1 : 2) + (lo ? 1 : 0);
}
// A converter warp's first block of adapters in a tile, brought ahead: the
// pieces, and the entries of its threads' tokens.
struct alignas(16) LgAhead {
  int2 gran[4], tok[2][32];
};
struct LgShared {
  LgAhead ahead[kLgConv];
  float fx[kLgEpi][128];    // 2^exponent of an epilogue warp's tokens
  int ew[kLgM];             // exponents of the tile's rows of W
  int bad;                  // some B held a non-finite value
  volatile int abort;
  uint32_t tmem;
  uint64_t opfull[kLgRO], opempty[kLgRO], accfull[2], accempty[2];
};
constexpr size_t kLgSmem = kLgRO * kLgStage + kLgConv * kLgRQ * kLgQTile + sizeof(LgShared) + 1024;

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}
// bf16 scales (or biases) of groups 8 k8 .. 8 k8 + 7 of a row, zero behind G
__device__ __forceinline__ uint4 load_meta(const LoraArgs& a, const uint16_t* base, int o, int k8) {
  const int G = a.K >> 6;
  const uint16_t* s = base + (size_t)o * G + 8 * k8;
  if (a.m_vec && 8 * k8 + 8 <= G) return __ldg(reinterpret_cast<const uint4*>(s));
  uint32_t v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 8 * k8 + e < G ? s[e] : 0u;
  return make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
}

// Adds to y[t][o] the terms of B's values that are not finite (their places in
// the matrix product were taken as zero).
template <int XT, int AT>
__device__ __noinline__ void add_bad_terms(const LoraArgs& a, int o, long long t) {
  int rank;
  const int id = adapter_of(a, t, rank);
  float s = 0.0f;
  bool any = false;
  for (int j = 0; j < rank; ++j) {
    const float w = load_val<AT>(a.b, (size_t)id * a.b_stride + (size_t)o * a.rank + j);
    if (!isfinite(w)) {
      float v = 0.0f;
      for (int p = a.v_planes - 1; p >= 0; --p)
        v += bf16_bits_to_f32(__ldcg(reinterpret_cast<const uint16_t*>(a.v) +
                                     ((size_t)t * a.v_planes + p) * a.v_stride + j));
      s += w * (v * pow2(__ldcg(a.ex + t)));   // the planes hold v 2^-ex
      any = true;
    }
  }
  const size_t at = (size_t)t * a.y_stride + o;
  if (any) store_val<XT>(a.y, at, load_val<XT>(a.y, at) + s);
}

// Bounded wait on an mbarrier phase: after about two seconds (4e9 clocks) the
// status bit is set and the CTA-wide abort flag makes all later waits return.
// It counts clocks, not the global timer, whose read takes long enough to show
// on every wait that does not succeed at once.
// NAP: the waiting warp stays off the issue slots between polls (waits that are
// long and not on the way of the matrix steps).
template <bool NAP = false>
__device__ __forceinline__ bool lg_wait(uint64_t* bar, uint32_t parity, volatile int* abort, uint32_t* status) {
  if (mbar_try_sleep(bar, parity)) return true;
  const long long t0 = clock64();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i) {
      if (NAP) __nanosleep(200);
      if (mbar_try_sleep(bar, parity)) return true;
    }
    if (*abort) return false;
    if (clock64() - t0 > 4000000000ll) break;
  }
  *abort = 1;
  atomicOr(status, kStatusCopyTimeout);
  return false;
}
// By a whole warp, with one outcome for all its lanes.
template <bool NAP = false>
__device__ __forceinline__ bool lg_warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, uint32_t* status) {
  return __all_sync(kAllLanes, lg_wait<NAP>(bar, parity, abort, status));
}

// D[tmem] (+)= A[smem desc] * B[smem desc]
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(ad), "l"(bd), "r"(idesc), "r"(acc));
}

// Warp 0 brings x, warp 1 issues the matrix steps, 8 warps convert weights and
// adapters (two groups, every other stage each), 8 warps read the sums (fp32
// rows after every four stages) and write y.
template <int XT, int AT>
__global__ void __launch_bounds__(kLgThreads, 1) lora_gemm_kernel(const __grid_constant__ LoraArgs a) {
  constexpr bool F32 = XT == 0;
  using C = LgCfg<F32>;
  constexpr int PL = C::PL, M = kLgM;
  extern __shared__ unsigned char lg_raw[];
  unsigned char* stages = lg_raw + ((1024u - (smem_addr(lg_raw) & 1023u)) & 1023u);
  unsigned char* qtiles = stages + kLgRO * kLgStage;
  LgShared& S = *reinterpret_cast<LgShared*>(qtiles + kLgConv * kLgRQ * kLgQTile);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = a.split, rank_c = split > 1 ? (int)cluster_rank() : 0;
  const int mt = (a.N + M - 1) / M, nt = (int)((a.tokens + a.NT - 1) / a.NT);
  const int tiles = mt * nt;
  const int first_tile = split > 1 ? (int)blockIdx.x / split : (int)blockIdx.x;
  const int step = split > 1 ? tiles : (int)gridDim.x;  // a cluster has one tile
  // K in stages: nk groups of 64, then the groups' sums against the biases, 64
  // columns a stage (fp32 rows: the biases' hi and lo parts in two stages)
  const int nk = a.K >> 6, nbk = bias_chunks(nk, F32), nkv = nk + (F32 ? 2 : 1) * nbk;
  const int k_lo = nkv * rank_c / split, nkm = nkv * (rank_c + 1) / split - k_lo;
  const int nq = max(0, min(nk - k_lo, nkm));   // of them from Q4 rows
  volatile int* abort = &S.abort;
  if (tid == 0) {
    for (int i = 0; i < kLgRO; ++i) {
      mbar_init(&S.opfull[i], 5);   // the four warps that wrote the stage, and the producer
      mbar_init(&S.opempty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S.accfull[i], 1);
      mbar_init(&S.accempty[i], kLgEpi);
    }
    S.bad = 0;
    S.abort = 0;
    mbar_init_fence();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&S.tmem)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = S.tmem;
  auto tokens_of = [&](int tile) { return (int)min((long long)a.NT, a.tokens - (long long)(tile / mt) * a.NT); };
  // The adapters' stages: blocks of 64 columns, this CTA's share of them, each
  // in the passes of lora_passes: every stage has matrix steps (a partial sum
  // that began with a stage without any would hold what its buffer held before).
  constexpr bool BLO = AT == 2;
  auto v_planes = [&](int npad) { return min(C::NV, 256 / npad); };
  auto pieces_at = [&](int tile) { return a.adapter && tile < tiles ? __ldcg(a.n_gran + tile / mt) : 0; };
  auto stages_of = [&](int npad, int ng) {
    const int nb = (ng + 3) >> 2;
    return nkm + (nb > rank_c ? (nb - rank_c + split - 1) / split * lora_passes(C::NV, npad, BLO) : 0);
  };

  if (warp == 0) {
    // ---------------- producer: x by bulk copies ----------------
    if (lane == 0) {
      pdl_wait();
      uint32_t os = 0;
      bool ok = true;
      int ng = pieces_at(first_tile);
      for (int tile = first_tile; tile < tiles && ok; tile += step) {
        const int npad = (tokens_of(tile) + 15) & ~15;
        const unsigned char* src = a.planes + (size_t)(tile / mt) * (nk + nbk) * PL * a.NT * 128;
        const int total = stages_of(npad, ng);
        ng = pieces_at(tile + step);
        for (int c = 0; c < total; ++c, ++os) {
          const int st = (int)(os % kLgRO);
          if (os >= (uint32_t)kLgRO && !lg_wait(&S.opempty[st], ((os / kLgRO) - 1) & 1, abort, a.status)) {
            ok = false;
            break;
          }
          if (c < nkm) {
            unsigned char* dst = stages + (size_t)st * kLgStage + kLgA;
            const int k = k_lo + c, kp = k < nk ? k : nk + (F32 ? (k - nk) >> 1 : k - nk);
            mbar_arrive_expect(&S.opfull[st], (uint32_t)(PL * npad * 128));
#pragma unroll
            for (int p = 0; p < PL; ++p)
              bulk_load(dst + (size_t)p * C::NMAX * 128, src + ((size_t)kp * PL + p) * a.NT * 128,
                        (uint32_t)(npad * 128), &S.opfull[st]);
          } else {
            mbar_arrive(&S.opfull[st]);
          }
        }
      }
      // no copy may still be landing when the CTA ends
      if (!ok)
        for (uint32_t i = os > (uint32_t)kLgRO ? os - kLgRO : 0; i < os; ++i)
          for (int n = 0; n < 1 << 16 && !mbar_test(&S.opfull[i % kLgRO], (i / kLgRO) & 1); ++n) {
          }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      pdl_wait();   // the lists
      const uint64_t adesc0 = desc_sw128(smem_addr(stages)), bdesc0 = adesc0 + (kLgA >> 4);
      uint32_t os = 0, gq = 0;
      bool ok = true;
      int ng = pieces_at(first_tile);
      for (int tile = first_tile; tile < tiles && ok; tile += step) {
        const int npad = (tokens_of(tile) + 15) & ~15;
        const uint32_t idf = idesc16(kLgM, npad, false), idb = idesc16(kLgM, npad, true);
        const int vpl = v_planes(npad), passes = lora_passes(C::NV, npad, BLO);
        const int total = stages_of(npad, ng);
        ng = pieces_at(tile + step);
        for (int c = 0; c < total; ++c, ++os) {
          bool first = c % C::GROUP == 0;
          if (first && gq >= 2 && !lg_wait(&S.accempty[gq & 1], ((gq >> 1) - 1) & 1, abort, a.status)) {
            ok = false;
            break;
          }
          const uint32_t d = tmem + (gq & 1) * 256;
          const int st = (int)(os % kLgRO);
          if (!lg_wait(&S.opfull[st], (os / kLgRO) & 1, abort, a.status)) {
            ok = false;
            break;
          }
          fence_after();
          const uint64_t so = (uint64_t)st * (kLgStage >> 4);
          auto issue = [&](uint32_t boff, uint32_t id) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              mma_ss(d, adesc0 + so + (uint64_t)(ks * 2), bdesc0 + so + (uint64_t)((boff + ks * 32) >> 4), id,
                     first && ks == 0 ? 0u : 1u);
            first = false;
          };
          if (c < nkm) {
            issue(0, idf);
            // the lo part of x; not for the lo part of the biases
            if (F32 && (k_lo + c < nk || ((k_lo + c - nk) & 1) == 0)) issue((uint32_t)C::NMAX * 128, idf);
          } else {
            const int pass = (c - nkm) % passes;
            const bool lo_part = BLO && pass == passes - 1;
            const int planes = lo_part ? C::NV - 1 : min(vpl, C::NV - pass * vpl);
            for (int p = 0; p < planes; ++p) issue((uint32_t)(p * npad * 128), idb);
          }
          commit(&S.opempty[st]);
          if (c % C::GROUP == C::GROUP - 1 || c == total - 1) {
            commit(&S.accfull[gq & 1]);
            ++gq;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp < 2 + kLgConv) {
    // ---------------- converters: group 0 the even stages of a tile, group 1 the odd ones ----------------
    const int grp = (warp - 2) >> 2;
    const int row = ((warp - 2) & 3) * 32 + lane;   // row of the tile
    unsigned char* ring = qtiles + (size_t)(warp - 2) * kLgRQ * kLgQTile;
    // Q4 tiles of this warp's stages, kLgRQ of them ahead: 16 bytes per lane and
    // copy, two lanes per row
    int f_tile = grp < nq ? first_tile : tiles, f_c = grp;
    uint32_t f_n = 0, used = 0;
    const uint32_t* f_src[2];                // this lane's two pieces, null behind the last row
    auto f_rows = [&]() {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = (f_tile % mt) * M + (row & 96) + (lane >> 1) + 16 * i;
        f_src[i] = f_tile < tiles && r < a.N
                       ? a.packed + (size_t)r * (a.K >> 3) + (size_t)(k_lo + grp) * 8 + (lane & 1) * 4 : nullptr;
      }
    };
    f_rows();
    auto fetch = [&]() {
      if (f_tile < tiles) {
        unsigned char* to = ring + (f_n % kLgRQ) * kLgQTile + (lane >> 1) * kLgQPitch + (lane & 1) * 16;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (f_src[i] == nullptr) continue;
          if (a.w_vec)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(to + i * 16 * kLgQPitch)),
                         "l"(f_src[i]) : "memory");
          else
            *reinterpret_cast<uint4*>(to + i * 16 * kLgQPitch) =
                make_uint4(f_src[i][0], f_src[i][1], f_src[i][2], f_src[i][3]);
          f_src[i] += 16;
        }
        f_c += 2;
        if (f_c >= nq) {
          f_tile += step;
          f_c = grp;
          f_rows();
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      ++f_n;
    };
    for (int i = 0; i < kLgRQ; ++i) fetch();
    pdl_wait();
    uint32_t os = 0;                         // stages before this tile
    bool ok = true;
    int ng_next = pieces_at(first_tile), ew_next = __ldcg(a.ew + (first_tile % mt) * M + row);
    for (int tile = first_tile; tile < tiles && ok; tile += step) {
      const int o = (tile % mt) * M + row;
      const bool live = o < a.N;
      const long long tn = (long long)(tile / mt) * a.NT;
      const float wsc = pow2(-ew_next);
      const int ntok = tokens_of(tile), npad = (ntok + 15) & ~15;
      const int ng = ng_next, total = stages_of(npad, ng);
      ng_next = pieces_at(tile + step);
      if (tile + step < tiles) ew_next = __ldcg(a.ew + ((tile + step) % mt) * M + row);
      uint4 meta = make_uint4(0, 0, 0, 0), meta_n = meta;
      int m8 = -1;
      auto slot_free = [&](uint32_t oc) {
        return oc < (uint32_t)kLgRO || lg_warp_wait(&S.opempty[oc % kLgRO], ((oc / kLgRO) - 1) & 1, abort, a.status);
      };
      auto slot_done = [&](int st) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.opfull[st]);
      };
      // 16 bytes of this row's operand, in the 128-byte swizzle
      auto put = [&](int st, int u, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
        *reinterpret_cast<uint4*>(stages + (size_t)st * kLgStage + row * 128 + ((u ^ (row & 7)) << 4)) =
            make_uint4(x, y, z, w);
      };
      // ---- a stage of weights or biases ----
      auto weights = [&](int c) -> bool {
        const uint32_t oc = os + (uint32_t)c;
        const int st = (int)(oc % kLgRO);
        uint32_t av[32];
        if (c < nq) {
          const int k = k_lo + c;
          if (live && (k >> 3) != m8) {
            meta = m8 >= 0 && (k >> 3) == m8 + 1 ? meta_n : load_meta(a, a.scales, o, k >> 3);
            m8 = k >> 3;
            if ((m8 + 1) * 8 < nk) meta_n = load_meta(a, a.scales, o, m8 + 1);
          }
          asm volatile("cp.async.wait_group %0;" ::"n"(kLgRQ - 1) : "memory");
          __syncwarp();                      // the other lanes' copies too
          const unsigned char* q = ring + (used % kLgRQ) * kLgQTile + lane * kLgQPitch;
          const uint4 w0 = *reinterpret_cast<const uint4*>(q), w1 = *reinterpret_cast<const uint4*>(q + 16);
          ++used;
          __syncwarp();                      // read by all lanes before the tile is filled again
          fetch();
          const uint32_t wv[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
          const uint32_t sw = word_of(meta, (k >> 1) & 3);
          // scale (q - 8), at most 8 + 3 significant bits and so exact in fp16:
          // a nibble in the mantissa of 16.0 is 16 + q, and 24 scale is exact too.
          // The pairs are (q_i, q_i+4) of a word; x is laid out alike.
          const __half2 s2 = __float2half2_rn((k & 1 ? bf_hi(sw) : bf_lo(sw)) * wsc),
                        m24 = __hmul2(s2, __float2half2_rn(-24.0f));
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            const uint32_t v[4] = {wv[w] << 6, wv[w] << 2, wv[w] >> 2, wv[w] >> 6};
#pragma unroll
            for (int p = 0; p < 4; ++p)
              av[4 * w + p] = h2u(__hfma2(u2h((v[p] & 0x03C003C0u) | 0x4C004C00u), s2, m24));
          }
        } else {
          // 64 columns of biases
          const uint32_t* b =
              a.wbias + ((size_t)(o >> 7) * (nkv - nk) + (size_t)(k_lo + c - nk)) * 32 * 128 + (row & 127);
#pragma unroll
          for (int e = 0; e < 32; ++e) av[e] = __ldcg(b + e * 128);
        }
        if (!slot_free(oc)) return false;
#pragma unroll
        for (int u = 0; u < 8; ++u) put(st, u, av[4 * u], av[4 * u + 1], av[4 * u + 2], av[4 * u + 3]);
        slot_done(st);
        return true;
      };
      // ---- a stage of adapters: a block of 64 columns, four pieces of 16 rows ----
      const int vpl = v_planes(npad), passes = lora_passes(C::NV, npad, BLO);
      auto block_of = [&](int c) { return rank_c + (c - nkm) / passes * split; };
      const int c_first = nkm + ((nkm ^ grp) & 1);   // this group's first such stage
      LgAhead& ahead = S.ahead[warp - 2];
      if (c_first < total) {
        // its lists, beside the stages of weights
        const unsigned char* from = nullptr;
        unsigned char* to = nullptr;
        if (lane < 2) {
          from = reinterpret_cast<const unsigned char*>(a.gran + (size_t)(tile / mt) * a.gran_stride + block_of(c_first) * 4) +
                 lane * 16;
          to = reinterpret_cast<unsigned char*>(ahead.gran) + lane * 16;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(to)), "l"(from) : "memory");
        }
        const int n = (row & 96) + (lane >> 4) * 128 + (lane & 15) * 2;   // two tokens a lane
        if (n < npad) {
          from = reinterpret_cast<const unsigned char*>(a.tok + tn + n);
          to = reinterpret_cast<unsigned char*>(&ahead.tok[lane >> 4][(lane & 15) * 2]);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(to)), "l"(from) : "memory");
        }
      }
      auto adapters = [&](int c) -> bool {
        const uint32_t oc = os + (uint32_t)c;
        const int st = (int)(oc % kLgRO);
        const int blk = block_of(c), pass = (c - nkm) % passes;
        const bool lo_part = BLO && pass == passes - 1;
        const int p0 = lo_part ? 0 : pass * vpl;
        const int planes = lo_part ? C::NV - 1 : min(vpl, C::NV - p0);
        const bool here = c == c_first;
        if (here) {
          asm volatile("cp.async.wait_all;" ::: "memory");
          __syncwarp();
        }
        const int2* gran = a.gran + (size_t)(tile / mt) * a.gran_stride + blk * 4;
        int left[4];                         // rows of the adapter from this piece on, 0: no piece
        uint4 raw[4][2];
        int2 tk[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = row + 128 * i;
          tk[i] = n >= npad ? make_int2(0, 0) : here ? ahead.tok[i][lane] : __ldcg(a.tok + tn + n);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int2 gr = blk * 4 + q >= ng ? make_int2(0, 0) : here ? ahead.gran[q] : __ldcg(gran + q);
          raw[q][0] = raw[q][1] = make_uint4(0, 0, 0, 0);
          left[q] = live ? gr.y >> 16 : 0;
          if (left[q] > 0) {
            const int jq = gr.y & 0xFFFF;
            const uint16_t* at =
                static_cast<const uint16_t*>(a.b) + (size_t)gr.x * a.b_stride + (size_t)o * a.rank + jq;
            if (a.b_vec && jq + 16 <= a.rank) {
              raw[q][0] = __ldg(reinterpret_cast<const uint4*>(at));
              raw[q][1] = __ldg(reinterpret_cast<const uint4*>(at) + 1);
            } else {
              uint32_t h[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) h[e] = e < left[q] ? at[e] : 0u;
              raw[q][0] = make_uint4(pack2(h[0], h[1]), pack2(h[2], h[3]), pack2(h[4], h[5]), pack2(h[6], h[7]));
              raw[q][1] = make_uint4(pack2(h[8], h[9]), pack2(h[10], h[11]), pack2(h[12], h[13]), pack2(h[14], h[15]));
            }
          }
        }
        if (!slot_free(oc)) return false;
        // ---- v: each token's planes in its own columns, zeros elsewhere ----
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = row + 128 * i;
          if (n >= npad) continue;
          const int q0 = tk[i].x - blk * 4, q1 = q0 + tk[i].y;   // its pieces in the block's numbers
          const uint16_t* v = reinterpret_cast<const uint16_t*>(a.v) +
                              ((size_t)(tn + n) * C::NV + p0) * a.v_stride - q0 * 16;
          unsigned char* at = stages + (size_t)st * kLgStage + kLgA + (size_t)n * 128;
          for (int p = 0; p < planes; ++p) {
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const bool in = (u >> 1) >= q0 && (u >> 1) < q1;
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                               smem_addr(at + (size_t)p * npad * 128 + ((u ^ (n & 7)) << 4))),
                           "l"(in ? v + (size_t)p * a.v_stride + u * 8 : reinterpret_cast<const uint16_t*>(a.v)),
                           "r"(in ? 16 : 0)
                           : "memory");
            }
          }
        }
        // ---- B ----
        const uint32_t wsc2 = pack_bf2(wsc, wsc);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t w[8] = {raw[q][0].x, raw[q][0].y, raw[q][0].z, raw[q][0].w,
                           raw[q][1].x, raw[q][1].y, raw[q][1].z, raw[q][1].w};
          if (left[q] < 16) {
#pragma unroll
            for (int p = 0; p < 8; ++p)
              w[p] &= (2 * p < left[q] ? 0xFFFFu : 0u) | (2 * p + 1 < left[q] ? 0xFFFF0000u : 0u);
          }
          // a non-finite value must not meet the zeros of other tokens: an
          // exponent of all ones carries into the sign place
          constexpr uint32_t kExp = AT == 2 ? 0x7C007C00u : 0x7F807F80u, kOne = AT == 2 ? 0x04000400u : 0x00800080u;
          uint32_t any = 0;
#pragma unroll
          for (int p = 0; p < 8; ++p) any |= (w[p] & kExp) + kOne;
          if (any & 0x80008000u) {
            S.bad = 1;
#pragma unroll
            for (int p = 0; p < 8; ++p) {
              const uint32_t b = ((w[p] & kExp) + kOne) & 0x80008000u;
              w[p] &= ~((b >> 15) * 0xFFFFu);
            }
          }
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            if constexpr (AT == 2) {
              float w0, w1;
              unpack2<AT>(w[p], w0, w1);
              w0 *= wsc;
              w1 *= wsc;
              w[p] = pack_bf2(w0, w1);
              if (lo_part) w[p] = pack_bf2(w0 - bf_lo(w[p]), w1 - bf_hi(w[p]));
            } else {
              w[p] = bf2_fma(w[p], wsc2, 0x80008000u);   // a power of two: exact
            }
          }
          put(st, 2 * q, w[0], w[1], w[2], w[3]);
          put(st, 2 * q + 1, w[4], w[5], w[6], w[7]);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        slot_done(st);
        return true;
      };
      for (int c = grp; c < total && ok; c += 2) ok = c < nkm ? weights(c) : adapters(c);
      os += (uint32_t)total;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // ---------------- epilogue ----------------
    const int quad = warp & 3;               // the quarter of tensor memory a warp can reach
    const int half = (warp - 2 - kLgConv) >> 2;   // 16-token pieces half, half + 2, ...
    const int row = quad * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    uint32_t gq = 0;
    pdl_wait();
    for (int tile = first_tile; tile < tiles; tile += step) {
      const int o = (tile % mt) * M + row;
      const bool live = o < a.N;
      const long long tn = (long long)(tile / mt) * a.NT;
      const int ntok = tokens_of(tile), npad = (ntok + 15) & ~15;
      const int ew = __ldcg(a.ew + o);
      const int total = stages_of(npad, pieces_at(tile));
      // 2^exponent of this warp's tokens, piece by piece, before there is a sum
      // to wait for
      float* fx = S.fx[warp - 2 - kLgConv];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < C::NMAX / 64; ++i) {
        const int n = (half + 4 * i + (lane >> 4) * 2) * 16 + (lane & 15);
        fx[32 * i + lane] = n < npad ? pow2(__ldcg(a.ex + tn + n)) : 0.0f;
      }
      __syncwarp();
      auto sum_wait = [&]() {
        if (!lg_warp_wait<true>(&S.accfull[gq & 1], (gq >> 1) & 1, abort, a.status)) return false;
        fence_after();
        return true;
      };
      auto sum_done = [&]() {
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.accempty[gq & 1]);
        ++gq;
      };
      // a sum times 2^(ew + ex): within range in this order, as |ew| above 60 is
      // taken in two steps
      const int ewc = max(-60, min(60, ew));
      const float fw = pow2(ewc), fr = pow2(ew - ewc);
      float* part = reinterpret_cast<float*>(stages);   // split: [token][M rows]
      using Y = std::conditional_t<F32, float, uint16_t>;
      auto put16 = [&](int i, const float (&v)[16]) {
        const int n0 = (half + 2 * i) * 16;
        if (split > 1) {
#pragma unroll
          for (int e = 0; e < 16; ++e) part[(n0 + e) * M + row] = v[e];
          return;
        }
        if (!live) return;
        float r[16];
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const float4 f = *reinterpret_cast<const float4*>(fx + 16 * i + 4 * e4);
          r[4 * e4] = v[4 * e4] * fw * f.x;
          r[4 * e4 + 1] = v[4 * e4 + 1] * fw * f.y;
          r[4 * e4 + 2] = v[4 * e4 + 2] * fw * f.z;
          r[4 * e4 + 3] = v[4 * e4 + 3] * fw * f.w;
        }
        if (ew != ewc) {
#pragma unroll
          for (int e = 0; e < 16; ++e) r[e] *= fr;
        }
        Y* at = static_cast<Y*>(a.y) + (size_t)(tn + n0) * a.y_stride + o;
        if (n0 + 16 <= ntok) {
#pragma unroll
          for (int e = 0; e < 16; ++e, at += a.y_stride) store_val<XT>(at, 0, r[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e, at += a.y_stride)
            if (n0 + e < ntok) store_val<XT>(at, 0, r[e]);
        }
      };
      if constexpr (F32) {
        float acc[4][16] = {};
        bool ok = true;
        for (int c = 0; c < total && ok; c += C::GROUP) {
          ok = sum_wait();
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int n0 = (half + 2 * i) * 16;
            if (n0 < npad) {
              uint32_t d[16];
              ld16(tmem + lane_addr + (gq & 1) * 256 + (uint32_t)n0, d);
              wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) acc[i][e] += __uint_as_float(d[e]);
            }
          }
          sum_done();
        }
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((half + 2 * i) * 16 < npad) put16(i, acc[i]);
      } else {
        if (!sum_wait()) break;
#pragma unroll
        for (int i = 0; i < C::NMAX / 32; ++i) {
          const int n0 = (half + 2 * i) * 16;
          if (n0 >= npad) continue;
          uint32_t d[16];
          ld16(tmem + lane_addr + (gq & 1) * 256 + (uint32_t)n0, d);
          wait_ld();
          float v[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = __uint_as_float(d[e]);
          put16(i, v);
        }
        sum_done();
      }
      if (split > 1) {
        if (half == 0) S.ew[row] = ew;
      } else if (live && S.bad && a.adapter) {
        // terms that are not finite, after the fact: they decide their values
        for (int n0 = half * 16; n0 < ntok; n0 += 32)
          for (int n = n0; n < min(n0 + 16, ntok); ++n) add_bad_terms<XT, AT>(a, o, tn + n);
      }
    }
  }
  if (split > 1) {
    // the cluster's partial sums, each CTA a share of the tokens, added in the order of K
    __syncwarp();
    cluster_sync_all();
    const int tile = first_tile, ntok = tokens_of(tile);
    const long long tn = (long long)(tile / mt) * a.NT;
    const int n_lo = ntok * rank_c / split, n_hi = ntok * (rank_c + 1) / split;
    bool bad = false;
    for (int r = 0; r < split; ++r) bad |= ld_cluster_i(map_rank(smem_addr(&S.bad), (uint32_t)r)) != 0;
    for (int i = tid; i < (n_hi - n_lo) * M; i += kLgThreads) {
      const int n = n_lo + i / M, row = i % M, o = (tile % mt) * M + row;
      if (o >= a.N || S.abort) continue;
      const uint32_t at = smem_addr(stages) + (uint32_t)(n * M + row) * 4;
      float p[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) p[r] = r < split ? ld_cluster(map_rank(at, (uint32_t)r)) : 0.0f;
      float v = p[0];
#pragma unroll
      for (int r = 1; r < 8; ++r) v += p[r];
      const int ew = S.ew[row], ewc = max(-60, min(60, ew));
      v = v * pow2(ewc) * pow2(__ldcg(a.ex + tn + n)) * pow2(ew - ewc);
      store_val<XT>(a.y, (size_t)(tn + n) * a.y_stride + o, v);
      if (bad && a.adapter) add_bad_terms<XT, AT>(a, o, tn + n);
    }
    cluster_sync_all();  // no CTA ends while another reads its sums
  }
  fence_before();
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

// ---------------------------------------------------------------- launches

bool decodes(const LoraArgs& a) {
  return a.tokens <= kDecTokens && (size_t)a.tokens * a.K * 4 <= kDecSmem;
}

// Rows of W per warp of the decode kernel: more of them share the reads of x
// from shared memory, fewer leave more warps.
int dec_rows(const LoraArgs& a) { return a.tokens > 2 && a.N >= 1024 ? 2 : 1; }
unsigned dec_blocks(const LoraArgs& a) {
  const int rows = dec_rows(a) * kDecWarps;
  return (unsigned)((a.N + rows - 1) / rows);
}
// Bytes of the adapters that all blocks together may read again for v: about
// what a launch costs.  One fp32 token 2048 -> 512 of rank 16 (4 MB): 9.1 us in
// one launch, 11.4 in two; four tokens 2048 x 2048 (32 MB): 22.8 against 11.8.
constexpr double kSelfBytes = 8e6;
bool v_by_self(const LoraArgs& a) {
  return decodes(a) && a.tokens * a.rank <= kDecSelf &&
         (double)a.tokens * a.rank * a.K * 2 * dec_blocks(a) <= kSelfBytes;
}
// Up to here a decode batch, for which no kernel prepares operands: mma.sync
// products (three per product for fp32 rows) against operands that cost about
// 15 us to prepare.  bf16 2048 x 2048: 128 tokens 21 us against 34, 256 tokens
// 33 against 25; fp16 512 -> 2048, 256 tokens: 18.5 against 37.
constexpr int kBatTokens = 256;
constexpr double kBatWork = 1e9;
bool batches(const LoraArgs& a) {
  return !decodes(a) && a.tokens <= kBatTokens &&
         (double)a.tokens * a.N * a.K * (a.x_type == 0 ? 3 : 1) <= kBatWork;
}
bool v_by_rows(const LoraArgs& a) { return (decodes(a) || batches(a)) && !v_by_self(a); }

// Tokens per tile and CTAs per tile (K and the adapters split over a cluster):
// the smallest of a plain estimate in clocks.  A stage costs its matrix steps
// (N / 2 clocks each, 4 per plane of x), what it moves through shared memory at
// 128 bytes a clock, or the conversion of its weights, whichever is longest; a
// stage of adapters, of which a tile of few tokens may have one for every few
// tokens, about 1500; a tile adds its epilogue, a split the exchange of the sums.
void lg_shape(const LoraArgs& a, int sms, int* NT, int* split) {
  const bool f32 = a.x_type == 0;
  const int nmax = f32 ? 128 : 256, nk = a.K >> 6, pl = f32 ? 2 : 1;
  double best = 1e300;
  *NT = 16;
  *split = 1;
  const long long mt = (a.N + kLgM - 1) / kLgM;
  for (int n = 16; n <= nmax; n += 16) {
    if (n > 16 && n - 16 >= a.tokens) break;
    const long long tiles = mt * ((a.tokens + n - 1) / n);
    double lora = 0.0;
    if (a.adapter) {
      const int passes = lora_passes(f32 ? 3 : 2, n, a.a_type == 2);
      const double many = a.tokens <= 512 ? (a.count < n ? a.count : n) : 2.0;
      lora = passes * (many * ((a.rank + 15) / 16) / 4.0 + 0.5);
    }
    for (int s = 1; s <= 8; s *= 2) {
      if (s > nk || (s > 1 && tiles * s > (s == 8 ? 128 : sms))) break;
      const double waves = (double)((tiles * s + sms - 1) / sms);
      const double smem = (4.0 * pl * (4096.0 + 32.0 * n) + 20480.0 + 128.0 * n * pl) / 128.0;
      const double stage = smem > 400.0 ? smem : 400.0;
      const double t = waves * (((nk + s - 1) / s) * stage + (lora / s) * 1500.0 + 2000.0 + 10.0 * n +
                                (s > 1 ? 1500.0 : 0.0));
      if (t < best) {
        best = t;
        *NT = n;
        *split = s;
      }
    }
  }
}

// `most`: dynamic shared memory of any launch of the kernel.  More than 48 KB
// with the static part (under 8 KB here) is asked for at the first launch on a
// device that needs it, not when a context is made: that loads the kernel, and
// all of this file's take 24 ms.
template <auto KERNEL>
cudaError_t launch_cfg(unsigned grid, unsigned block, size_t smem, size_t most, int cluster, cudaStream_t s,
                       const LoraArgs& a) {
  static std::atomic<uint64_t> asked{0};   // a bit per device
  auto ask = [&]() {
    return cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
  };
  const bool big = smem > (40 << 10);
  if (big) {
    int device = 0;
    if (const cudaError_t e = cudaGetDevice(&device)) return e;
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (!(asked.load(std::memory_order_relaxed) & bit)) {
      if (const cudaError_t e = ask()) return e;
      asked.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  cfg.attrs = attr;
  cudaError_t e = cudaLaunchKernelEx(&cfg, KERNEL, a);
  if (e == cudaErrorInvalidValue && big && ask() == cudaSuccess) {   // a device reset since then has undone it
    cudaGetLastError();
    e = cudaLaunchKernelEx(&cfg, KERNEL, a);
  }
  return e;
}

template <int XT, int AT, int TT>
cudaError_t launch_decode(const LoraArgs& a, cudaStream_t s) {
  const size_t sm = (size_t)a.tokens * a.K * 4;
  if (TT >= 4 && dec_rows(a) == 2)
    return launch_cfg<lora_decode_kernel<XT, AT, TT, 2>>(dec_blocks(a), kDecWarps * 32, sm, kDecSmem, 1, s, a);
  return launch_cfg<lora_decode_kernel<XT, AT, TT, 1>>(dec_blocks(a), kDecWarps * 32, sm, kDecSmem, 1, s, a);
}

// The most rows per CTA that still give every SM one (for 16-bit rows 64 rows
// leave no room for a second CTA on the SM: 23.4 us against 18.5).
template <int XT, int AT>
cudaError_t launch_batch(const LoraArgs& a, int sms, cudaStream_t s) {
  constexpr int NT = XT == 0 ? 2 : 4;
  const unsigned tt = (unsigned)((a.tokens + 8 * NT - 1) / (8 * NT));
  const size_t v = a.adapter ? (size_t)8 * NT * a.v_stride * 4 : 0;
  auto tiles = [&](int mt) { return (unsigned)((a.N + 16 * mt - 1) / (16 * mt)) * tt; };
  auto go = [&](auto mt) {
    constexpr int MT = decltype(mt)::value;
    constexpr size_t bytes = BatSmem<XT, MT, NT>::BYTES;
    return launch_cfg<lora_batch_kernel<XT, AT, MT, NT>>(tiles(MT), kBatWarps * 32, bytes + v,
                                                         bytes + 8 * NT * kBatRank * 4, 1, s, a);
  };
  if constexpr (XT == 0)
    if (tiles(4) >= (unsigned)sms) return go(std::integral_constant<int, 4>{});
  if (tiles(2) >= (unsigned)sms) return go(std::integral_constant<int, 2>{});
  return go(std::integral_constant<int, 1>{});
}

template <int XT, int AT>
cudaError_t launch(const LoraArgs& a, int sms, cudaStream_t s, uint64_t* launches) {
  const bool dec = decodes(a) || batches(a);
  if (a.adapter && v_by_rows(a)) {
    auto blocks = [&](int rows) {
      return (unsigned)((a.tokens * ((a.rank + rows - 1) / rows) + kRowWarps - 1) / kRowWarps);
    };
    const cudaError_t e =
        a.tokens * a.rank <= 1024
            ? launch_cfg<lora_v_rows_kernel<XT, AT, 1>>(blocks(1), kRowWarps * 32, 0, 0, 1, s, a)
            : launch_cfg<lora_v_rows_kernel<XT, AT, 4>>(blocks(4), kRowWarps * 32, 0, 0, 1, s, a);
    if (e != cudaSuccess) return e;
    if (launches) *launches += 1;
  }
  const long long rows = (a.tokens + 15) / 16 * 16;
  const long long row_blocks = dec ? 0 : a.row_threads == 32 ? rows / kPrepWarps : rows;
  const long long prep = a.v_blocks + a.l_blocks + a.w_blocks + row_blocks;
  if (a.after_v) {
    const cudaError_t e = launch_cfg<lora_v_kernel<XT, AT>>((unsigned)a.after_v * VBig<XT>::KSPLIT, VBig<XT>::THREADS,
                                                            VBig<XT>::BYTES, VBig<XT>::BYTES, VBig<XT>::KSPLIT, s, a);
    if (e != cudaSuccess) return e;
    if (launches) *launches += 1;
  }
  if (prep) {
    const cudaError_t e = launch_cfg<lora_prep_kernel<XT, AT>>((unsigned)prep, kPrepThreads, a.v_blocks ? kPrepRed : 0,
                                                               kPrepRed, 1, s, a);
    if (e != cudaSuccess) return e;
    if (launches) *launches += 1;
  }
  if (launches) *launches += 1;
  if (batches(a)) return launch_batch<XT, AT>(a, sms, s);
  if (dec) {
    if (a.tokens == 1) return launch_decode<XT, AT, 1>(a, s);
    if (a.tokens == 2) return launch_decode<XT, AT, 2>(a, s);
    return launch_decode<XT, AT, 4>(a, s);
  }
  const long long tiles = (long long)((a.N + kLgM - 1) / kLgM) * ((a.tokens + a.NT - 1) / a.NT);
  const unsigned grid = (unsigned)(a.split > 1 ? tiles * a.split : tiles < sms ? tiles : sms);
  return launch_cfg<lora_gemm_kernel<XT, AT>>(grid, kLgThreads, kLgSmem, kLgSmem, a.split, s, a);
}

constexpr size_t kWsAlign = 1024;
size_t up(size_t v) { return (v + kWsAlign - 1) / kWsAlign * kWsAlign; }

// Tokens per round of launches, a multiple of 256: as many as 256 MB hold the
// operands, v and lists of, which bounds the workspace beside what W takes (a
// small K with a large rank has more of v than of x).
long long block_tokens(const LoraArgs& a) {
  const bool f32 = a.x_type == 0;
  const int nk = a.K >> 6;
  long long row = (long long)(nk + bias_chunks(nk, f32)) * 128 * (f32 ? 2 : 1) + 4;   // planes, ex
  if (a.adapter) {
    const long long pieces = (a.rank + 15) / 16;
    row += pieces * 16 * 2 * (f32 ? 3 : 2) + pieces * 8 + 8;                           // v, gran, tok
  }
  const long long n = (256ll << 20) / row / 256 * 256;
  return n < 256 ? 256 : n;
}

// The shape of the launches for a.tokens tokens and the workspace they take.
size_t shape(LoraArgs& a, int sms, unsigned char* base) {
  const bool dec = decodes(a) || batches(a);
  size_t off = 0;
  a.w_blocks = 0;
  if (!dec) {
    lg_shape(a, sms, &a.NT, &a.split);
    const long long tiles = (a.tokens + a.NT - 1) / a.NT, nk = a.K >> 6;
    a.planes = base;
    const int nbk = bias_chunks((int)nk, a.x_type == 0);
    off += up((size_t)tiles * a.NT * (nk + nbk) * 128 * (a.x_type == 0 ? 2 : 1));
    a.ex = reinterpret_cast<int*>(base + off);
    off += up((size_t)((a.tokens + 15) / 16 * 16) * 4);
    a.row_threads = a.tokens >= 1024 ? 32 : kPrepThreads;
    a.w_blocks = (a.N + kLgM - 1) / kLgM;
    a.ew = reinterpret_cast<int*>(base + off);
    off += up((size_t)a.w_blocks * kLgM * 4);
    a.wbias = reinterpret_cast<uint32_t*>(base + off);
    off += up((size_t)a.w_blocks * (a.x_type == 0 ? 2 : 1) * nbk * 32 * kLgM * 4);
  }
  a.v_blocks = a.l_blocks = a.after_v = a.v_self = 0;
  a.v_stride = 0;
  a.v_slots = 1;
  if (a.adapter) {
    a.v_stride = ((size_t)a.rank + 15) / 16 * 16;
    a.v_planes = dec ? 0 : a.x_type == 0 ? 3 : 2;
    const long long most = a.tokens < a.count ? a.tokens : a.count;
    // v: tiles of 16 tokens in the prep kernel while a tile's adapters are worth
    // blocks of their own, a kernel of its own where a prompt's tokens share them
    // (2500 bf16 tokens 2048 x 2048, 8 adapters of rank 16: 72 us against 74; 3500,
    // every token another of 64: 245 against 338; 3500 fp32 tokens 2048 -> 768, 8
    // adapters of rank 64: 98 against 96; above, prompts decide: 4096 tokens of 8
    // requests 86 against 80, 6000 fp32 tokens of 12 of rank 64 260 against 243,
    // though 6000 tokens that each take another of 64 would gain, 385 against 548)
    a.v_self = v_by_self(a);
    if (a.v_self || v_by_rows(a)) {
      // no tiles
    } else if (a.tokens < 4096) {
      a.v_slots = (int)(most < 16 ? most : 16);
      a.v_blocks = (int)((a.tokens + 15) / 16 * a.v_slots);
    } else {
      // one cluster per tile for all of its adapters where the tiles fill the
      // GPU (clusters without an adapter cost about as much as their launch)
      const long long vt = (a.tokens + 31) / 32, fill = sms / vt;
      a.v_slots = (int)(fill < 1 ? 1 : fill < most ? fill : most);
      a.after_v = (int)(vt * a.v_slots);
    }
    if (!dec) {
      a.l_blocks = (int)((a.tokens + a.NT - 1) / a.NT);
      a.gran_stride = (size_t)a.NT * ((a.rank + 15) / 16);
      a.gran = reinterpret_cast<int2*>(base + off);
      off += up((size_t)a.l_blocks * a.gran_stride * 8);
      a.tok = reinterpret_cast<int2*>(base + off);
      off += up((size_t)((a.tokens + 15) / 16 * 16) * 8);
      a.n_gran = reinterpret_cast<int*>(base + off);
      off += up((size_t)a.l_blocks * 4);
    }
    a.v = reinterpret_cast<float*>(base + off);
    if (!a.v_self) off += up((size_t)a.tokens * a.v_stride * (dec ? 4 : 2 * a.v_planes));
  }
  return off;
}

}  // namespace

size_t lora_workspace(const LoraArgs& args, int sms) {
  const long long most = block_tokens(args);
  size_t need = 0;
  for (long long n : {args.tokens < most ? args.tokens : most, args.tokens % most}) {
    if (n == 0) continue;
    LoraArgs a = args;
    a.tokens = n;
    const size_t b = shape(a, sms, nullptr);
    need = b > need ? b : need;
  }
  return need;
}

cudaError_t launch_lora(const LoraArgs& args, void* workspace, int sms, cudaStream_t s, uint64_t* launches) {
  const long long most = block_tokens(args);
  const size_t ts = args.x_type == 0 ? 4 : 2;
  auto aligned = [](const void* p, size_t stride_bytes) {
    return ((reinterpret_cast<uintptr_t>(p) | stride_bytes) & 15) == 0;
  };
  for (long long t0 = 0; t0 < args.tokens; t0 += most) {
    LoraArgs a = args;
    a.tokens = args.tokens - t0 < most ? args.tokens - t0 : most;
    a.x = static_cast<const unsigned char*>(args.x) + (size_t)t0 * args.x_stride * ts;
    a.y = static_cast<unsigned char*>(args.y) + (size_t)t0 * args.y_stride * ts;
    if (a.adapter) a.adapter = args.adapter + t0;
    shape(a, sms, static_cast<unsigned char*>(workspace));
    a.x_vec = aligned(a.x, a.tokens > 1 ? a.x_stride * ts : 0);
    a.w_vec = aligned(a.packed, 0);
    a.m_vec = aligned(a.scales, (size_t)(a.K / 64) * 2) && aligned(a.biases, 0);
    a.a_vec = a.adapter && aligned(a.a, a.a_stride * 2);
    a.b_vec = a.adapter && aligned(a.b, a.b_stride * 2 | (size_t)a.rank * 2);
    cudaError_t e;
    if (a.adapter && a.a_type == 2) {
      e = a.x_type == 0   ? launch<0, 2>(a, sms, s, launches)
          : a.x_type == 1 ? launch<1, 2>(a, sms, s, launches)
                          : launch<2, 2>(a, sms, s, launches);
    } else {
      e = a.x_type == 0   ? launch<0, 1>(a, sms, s, launches)
          : a.x_type == 1 ? launch<1, 1>(a, sms, s, launches)
                          : launch<2, 1>(a, sms, s, launches);
    }
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace osm
