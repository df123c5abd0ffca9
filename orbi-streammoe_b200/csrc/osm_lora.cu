// osm_lora.cu -- a Q4 projection shared by every token beside the low-rank
// adapters of many requests (osm_q4_gemv_lora):
//   y[t] = W x[t] + gain[a] B_a (A_a x[t]),   a = adapter[t], none if negative
// W is MLX-affine Q4 (group 64 along the input, w = scale q + bias), A_a is
// [rank][in], B_a [out][rank] in bf16 or fp16; only the first ranks[a] rows of
// an adapter count.  Rows are fp32, bf16 or fp16.
//
// Two kernels, whatever the number of tokens.
//
// lora_prep_kernel, over tiles of 16 tokens: the rows of x as fp16 operands of
// the tensor cores, each row scaled by a power of two so that its largest
// value lies in [2^14, 2^15) (fp32 rows as hi + lo, 22 bits; bf16 and fp16
// rows exactly), and v[t] = gain A_a x[t] by tf32 matrix products (x as hi +
// lo for fp32 rows), once for every distinct adapter of a tile.
//
// lora_gemm_kernel: D[128 rows of W][N tokens] on tcgen05.  Weights go from Q4
// to fp16 (hi + lo for fp32 rows) into tensor memory, scaled by a power of two
// per row of W in the same way; x comes by bulk copies.  The adapters are
// further steps of the same sum: for the distinct adapters of the tile, B_a
// (rows of W) against v with zeros in the tokens of other adapters, in bf16
// planes, which have the range for any ratio between W, B, x and v.  So a tile
// of many requests needs no sorting and no second pass over y.
//
// What rounds: fp32 rows hold 22 bits of x and w (products to about 2^-22) and
// sums of 16 products per step; the tensor core's accumulation drops what lies
// below the accumulator's last place, so after every 4 K groups (16 steps) the
// partial sum leaves tensor memory and is added in registers, which keeps the
// loss under 1e-6.  16-bit rows round each weight once to fp16 (2^-12, below
// the rounding of y), v to 16 bits, and y once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

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

// Exponent e of a row whose largest magnitude is m: m 2^-e lies in
// [2^14, 2^15); 0 for a zero row.  Not below -100, so that 2^-e and what it
// multiplies stay in range (rows under 2^-86 then lie lower).
__device__ __forceinline__ int row_exponent(float m) {
  if (!(m > 0.0f)) return 0;
  const int e = (int)(__float_as_uint(m) >> 23) - 127 - 14;
  return max(e, -100);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // |e| <= 126
// v 2^e for any e a product of two rows' exponents can have
__device__ __forceinline__ float scale_by(float v, int e) {
  const int h = e >> 1;
  return v * pow2(h) * pow2(e - h);
}

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

// ---------------------------------------------------------------- prep

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr int kPrepRows = 16;   // tokens per tile of the prep kernel
constexpr int kPrepWarps = 8;
constexpr int kPrepCols = 32;   // rank columns per pass

// Blocks (tile, 0): operand planes of 16 rows.  Blocks (tile, y > 0): v for the
// tile's distinct adapters y - 1, y - 1 + (gridDim.y - 1), ...
template <int XT, int AT>
__global__ void __launch_bounds__(kPrepWarps * 32) lora_prep_kernel(const LoraArgs a) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long t0 = (long long)blockIdx.x * kPrepRows;
  pdl_wait();
  pdl_trigger();
  constexpr int PB = XT == 0 ? 2 : 1;
  if (blockIdx.y == 0) {
    for (int r = warp; r < kPrepRows; r += kPrepWarps) {
      const long long t = t0 + r;
      const bool live = t < a.tokens;
      const size_t row = (size_t)t * a.x_stride;
      int ex = 0;
      if (live) {
        float m = 0.0f;
        for (int i = lane * 8; i < a.K; i += 256) {
          float v[8];
          load8<XT>(a.x, row + i, a.x_vec, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[e]));
        }
        ex = row_exponent(warp_max(m));
      }
      if (lane == 0) a.ex[t] = ex;
      const float sc = pow2(-ex);
      const int row_in = (int)(t % a.NT);
      unsigned char* tile = a.planes + (size_t)(t / a.NT) * (a.K >> 6) * PB * a.NT * 128 + (size_t)row_in * 128;
      for (int i = lane * 8; i < a.K; i += 256) {
        float v[8] = {};
        if (live) load8<XT>(a.x, row + i, a.x_vec, v);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const float x0 = v[2 * p] * sc, x1 = v[2 * p + 1] * sc;
          const __half2 h = __floats2half2_rn(x0, x1);
          hi[p] = h2u(h);
          if constexpr (PB == 2) {
            const float2 f = __half22float2(h);
            lo[p] = h2u(__floats2half2_rn(x0 - f.x, x1 - f.y));
          }
        }
        unsigned char* at = tile + (size_t)(i >> 6) * PB * a.NT * 128 + ((((i >> 3) & 7) ^ (row_in & 7)) << 4);
        *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if constexpr (PB == 2)
          *reinterpret_cast<uint4*>(at + (size_t)a.NT * 128) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    return;
  }
  __shared__ int s_id[kPrepRows], s_rank[kPrepRows], s_list[kPrepRows], s_n;
  __shared__ float s_red[kPrepWarps][kPrepRows][kPrepCols];
  if (warp == 0) {
    int rank = 0, id = -1;
    if (lane < kPrepRows && t0 + lane < a.tokens) id = adapter_of(a, t0 + lane, rank);
    if (lane < kPrepRows) {
      s_id[lane] = id;
      s_rank[lane] = rank;
    }
    const uint32_t same = __match_any_sync(kAllLanes, id);
    const bool first = lane < kPrepRows && rank > 0 && (int)(__ffs(same) - 1) == lane;
    const uint32_t firsts = __ballot_sync(kAllLanes, first);
    if (first) s_list[__popc(firsts & ((1u << lane) - 1u))] = lane;
    if (lane == 0) s_n = __popc(firsts);
  }
  __syncthreads();
  const int g = lane >> 2, q = lane & 3;
  for (int d = (int)blockIdx.y - 1; d < s_n; d += (int)gridDim.y - 1) {
    const int id = s_id[s_list[d]], rank = s_rank[s_list[d]];
    const bool in0 = s_id[g] == id, in1 = s_id[g + 8] == id;
    const size_t x0 = (size_t)(t0 + g) * a.x_stride, x1 = (size_t)(t0 + g + 8) * a.x_stride;
    const size_t arow = (size_t)id * a.a_stride;
    for (int j0 = 0; j0 < rank; j0 += kPrepCols) {
      float acc[kPrepCols / 8][4] = {};
      // K in steps of 32: the thread's 8 values of a row are the k and k + 4
      // positions of four 8-wide matrix steps (the order of K is free as long
      // as both operands use the same one)
#pragma unroll 2
      for (int c = warp; c < a.K / 32; c += kPrepWarps) {
        const int i = c * 32 + q * 8;
        float xa[8] = {}, xb[8] = {};
        if (in0) load8<XT>(a.x, x0 + i, a.x_vec, xa);
        if (in1) load8<XT>(a.x, x1 + i, a.x_vec, xb);
#pragma unroll
        for (int n = 0; n < kPrepCols / 8; ++n) {
          const int j = j0 + n * 8 + g;
          float w[8] = {};
          if (j0 + n * 8 < rank) {
            if (j < rank) load8<AT>(a.a, arow + (size_t)j * a.K + i, a.a_vec, w);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              const uint32_t b0 = __float_as_uint(w[2 * s]), b1 = __float_as_uint(w[2 * s + 1]);
              uint32_t h[4] = {__float_as_uint(xa[2 * s]), __float_as_uint(xb[2 * s]), __float_as_uint(xa[2 * s + 1]),
                               __float_as_uint(xb[2 * s + 1])};
              if constexpr (XT == 0) {
                uint32_t l[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float f = __uint_as_float(h[e]);
                  h[e] &= 0xFFFFE000u;
                  l[e] = __float_as_uint(f - __uint_as_float(h[e]));
                }
                mma_tf32(acc[n], l, b0, b1);
              }
              mma_tf32(acc[n], h, b0, b1);
            }
          }
        }
      }
#pragma unroll
      for (int n = 0; n < kPrepCols / 8; ++n) {
        s_red[warp][g][n * 8 + 2 * q] = acc[n][0];
        s_red[warp][g][n * 8 + 2 * q + 1] = acc[n][1];
        s_red[warp][g + 8][n * 8 + 2 * q] = acc[n][2];
        s_red[warp][g + 8][n * 8 + 2 * q + 1] = acc[n][3];
      }
      __syncthreads();
      const float gain = a.gain ? a.gain[id] : 1.0f;
      for (int o = tid; o < kPrepRows * kPrepCols; o += kPrepWarps * 32) {
        const int r = o / kPrepCols, j = o % kPrepCols;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kPrepWarps; ++w) s += s_red[w][r][j];
        // whole granules of 16: zeros behind the adapter's rank
        if (s_id[r] == id && j0 + j < ((rank + 15) & ~15))
          a.v[(size_t)(t0 + r) * a.v_stride + j0 + j] = j0 + j < rank ? gain * s : 0.0f;
      }
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------- gemm

constexpr int kLgM = 128;                 // rows of W per tile
constexpr int kLgConv = 8;                // converter warps, two groups of four
constexpr int kLgEpi = 8;                 // epilogue warps, two per quarter of the rows
constexpr int kLgWarps = 2 + kLgConv + kLgEpi;
constexpr int kLgThreads = kLgWarps * 32;
constexpr int kLgMaxN = 256;
constexpr int kLgGran = kLgMaxN * 8;      // 16-wide pieces of adapters: 256 tokens of rank 128

template <bool F32>
struct LgCfg {
  static constexpr int PL = F32 ? 2 : 1;        // operand planes of W and of x
  static constexpr int NMAX = F32 ? 128 : 256;  // tokens per tile
  static constexpr int RO = F32 ? 4 : 5;        // operand stages (one K group each)
  static constexpr int GROUP = F32 ? 4 : 1 << 30;  // stages per partial sum
  static constexpr uint32_t A_COLS = 32 * PL;
  static constexpr uint32_t TMEM_A = 256;       // below: two sums of 128 tokens or one of 256
  static constexpr size_t STAGE = (size_t)NMAX * 128 * PL;
};
// Per-tile lists, two buffers: written by the epilogue warps for all roles.
struct alignas(16) LgList {
  int id[kLgMaxN];          // adapter of each token, -1 none
  uint16_t first[kLgMaxN];  // first token of the tile with the same adapter, 0xFFFF none
  uint16_t rank[kLgMaxN];
  int ex[kLgMaxN];          // exponents of the tokens' rows
  uint16_t gran[kLgGran];   // piece: first token << 4 | index of the 16 rows
  int n_gran;
  int wsum[kLgEpi];
};
struct LgShared {
  LgList list[2];
  int ew[kLgM];             // exponents of the tile's rows of W
  int bad;                  // some B held a non-finite value
  volatile int abort;
  uint32_t tmem;
  uint64_t opfull[8], opempty[8], accfull[2], accempty[2], listfull[2], epi;
};

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

// The exponent of row o of W: of the largest |scale q + bias| its groups allow.
__device__ __forceinline__ int weight_exponent(const LoraArgs& a, int o) {
  if (o >= a.N) return 0;
  const int G = a.K >> 6;
  const uint16_t* s = a.scales + (size_t)o * G;
  const uint16_t* b = a.biases + (size_t)o * G;
  float m = 0.0f;
  for (int g = 0; g < G; ++g) {
    const float sc = bf16_bits_to_f32(s[g]), bi = bf16_bits_to_f32(b[g]);
    m = fmaxf(m, fmaxf(fabsf(bi), fabsf(fmaf(15.0f, sc, bi))));
  }
  return row_exponent(m);
}

// What the rows of B of one adapter that are not finite add to y[o] of token t
// (their places in the matrix product were taken as zero).
template <int AT>
__device__ __noinline__ float bad_terms(const LoraArgs& a, int id, int rank, int o, long long t) {
  float s = 0.0f;
  for (int j = 0; j < rank; ++j) {
    const float w = load_val<AT>(a.b, (size_t)id * a.b_stride + (size_t)o * a.rank + j);
    if (!isfinite(w)) s += w * a.v[(size_t)t * a.v_stride + j];
  }
  return s;
}

template <int XT, int AT>
__global__ void __launch_bounds__(kLgThreads, 1) lora_gemm_kernel(const LoraArgs a) {
  constexpr bool F32 = XT == 0;
  using C = LgCfg<F32>;
  constexpr int PL = C::PL;
  extern __shared__ unsigned char lg_raw[];
  unsigned char* stages = lg_raw + ((1024u - (smem_addr(lg_raw) & 1023u)) & 1023u);
  LgShared& S = *reinterpret_cast<LgShared*>(stages + C::RO * C::STAGE);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = a.split, rank_c = split > 1 ? (int)cluster_rank() : 0;
  const int mt = (a.N + kLgM - 1) / kLgM, nt = (int)((a.tokens + a.NT - 1) / a.NT);
  const int tiles = mt * nt;
  const int first_tile = split > 1 ? (int)blockIdx.x / split : (int)blockIdx.x;
  const int step = split > 1 ? tiles : (int)gridDim.x;  // a cluster has one tile
  const int nk = a.K >> 6;
  const int k_lo = nk * rank_c / split, k_hi = nk * (rank_c + 1) / split, nkm = k_hi - k_lo;
  const int nbuf = a.NT <= 128 ? 2 : 1;
  // passes over the adapters' pieces: fp32 rows (B hi, lo) x (v0, v1), B x v2;
  // 16-bit rows B hi x v0, B hi x v1, and for fp16 adapters B lo x v0
  const int passes = F32 ? 2 : AT == 2 ? 3 : 2;
  volatile int* abort = &S.abort;
  if (tid == 0) {
    for (int i = 0; i < C::RO; ++i) {
      mbar_init(&S.opfull[i], 5);   // the four warps that wrote the stage, and the producer
      mbar_init(&S.opempty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&S.accfull[i], 1);
      mbar_init(&S.accempty[i], kLgEpi);
      mbar_init(&S.listfull[i], kLgEpi);
    }
    mbar_init(&S.epi, kLgEpi);
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
  // stages this CTA adds for the adapters of a tile (its share of the blocks of 64 columns)
  auto lora_stages = [&](int ng) {
    const int nb = (ng + 3) >> 2;
    return nb > rank_c ? (nb - rank_c + split - 1) / split * passes : 0;
  };

  if (warp == 0) {
    // ---------------- producer: x by bulk copies ----------------
    if (lane == 0) {
      pdl_wait();
      uint32_t os = 0;
      int ti = 0;
      bool ok = true;
      for (int tile = first_tile; tile < tiles && ok; tile += step, ++ti) {
        const int npad = (tokens_of(tile) + 15) & ~15;
        const unsigned char* src = a.planes + (size_t)(tile / mt) * nk * PL * a.NT * 128;
        int total = nkm;
        for (int c = 0; c < total; ++c, ++os) {
          if (c == nkm - 1) {
            if (!tc_wait(&S.listfull[ti & 1], (ti >> 1) & 1, abort, a.status)) {
              ok = false;
              break;
            }
            total += lora_stages(S.list[ti & 1].n_gran);
          }
          const int st = (int)(os % C::RO);
          if (os >= (uint32_t)C::RO && !tc_wait(&S.opempty[st], ((os / C::RO) - 1) & 1, abort, a.status)) {
            ok = false;
            break;
          }
          if (c < nkm) {
            unsigned char* dst = stages + (size_t)st * C::STAGE;
            mbar_arrive_expect(&S.opfull[st], (uint32_t)(PL * npad * 128));
#pragma unroll
            for (int p = 0; p < PL; ++p)
              bulk_load(dst + (size_t)p * C::NMAX * 128, src + ((size_t)(k_lo + c) * PL + p) * a.NT * 128,
                        (uint32_t)(npad * 128), &S.opfull[st]);
          } else {
            mbar_arrive(&S.opfull[st]);
          }
        }
      }
      // no copy may still be landing when the CTA ends
      if (!ok)
        for (uint32_t i = os > (uint32_t)C::RO ? os - C::RO : 0; i < os; ++i)
          for (int n = 0; n < 1 << 16 && !mbar_test(&S.opfull[i % C::RO], (i / C::RO) & 1); ++n) {
          }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      const uint64_t bdesc0 = desc_sw128(smem_addr(stages));
      uint32_t os = 0, gq = 0;
      int ti = 0;
      bool ok = true;
      for (int tile = first_tile; tile < tiles && ok; tile += step, ++ti) {
        const int npad = (tokens_of(tile) + 15) & ~15;
        const uint32_t idf = idesc16(kLgM, npad, false), idb = idesc16(kLgM, npad, true);
        int total = nkm;
        uint32_t d = 0;
        for (int c = 0; c < total; ++c, ++os) {
          if (c == nkm - 1) {
            if (!tc_wait(&S.listfull[ti & 1], (ti >> 1) & 1, abort, a.status)) {
              ok = false;
              break;
            }
            total += lora_stages(S.list[ti & 1].n_gran);
          }
          const int b = nbuf == 2 ? (int)(gq & 1) : 0;
          bool first = c % C::GROUP == 0;
          if (first) {
            const uint32_t use = nbuf == 2 ? gq >> 1 : gq;
            if (use > 0 && !tc_wait(&S.accempty[b], (use - 1) & 1, abort, a.status)) {
              ok = false;
              break;
            }
            d = tmem + (uint32_t)(b * 128);
          }
          const int st = (int)(os % C::RO);
          if (!tc_wait(&S.opfull[st], (os / C::RO) & 1, abort, a.status)) {
            ok = false;
            break;
          }
          fence_after();
          const uint32_t ab = tmem + C::TMEM_A + (uint32_t)st * C::A_COLS;
          const uint64_t bd = bdesc0 + (uint64_t)st * (C::STAGE >> 4);
          auto issue = [&](int pa, int pb, uint32_t id) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
              mma_ts(d, ab + (uint32_t)(pa * 32 + ks * 8),
                     bd + (uint64_t)(((size_t)pb * C::NMAX * 128 + ks * 32) >> 4), id, first && ks == 0 ? 0u : 1u);
            }
            first = false;
          };
          if (c < nkm) {
            issue(0, 0, idf);
            if constexpr (F32) {
              issue(0, 1, idf);
              issue(1, 0, idf);
            }
          } else if constexpr (F32) {
            const int pass = (c - nkm) % passes;
            issue(0, 0, idb);
            if (pass == 0) {
              issue(0, 1, idb);
              if (AT == 2) {
                issue(1, 0, idb);
                issue(1, 1, idb);
              }
            }
          } else {
            issue(0, 0, idb);
          }
          commit(&S.opempty[st]);
          if (c % C::GROUP == C::GROUP - 1 || c == total - 1) {
            commit(&S.accfull[b]);
            ++gq;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp < 2 + kLgConv) {
    // ---------------- converters ----------------
    const int grp = (warp - 2) >> 2;         // stages with os % 2 == grp
    const int quad = warp & 3;
    const int row = quad * 32 + lane;        // tensor-memory lane = row of the tile
    const int gt = ((warp - 2) & 3) * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    const int G = nk;
    struct Raw {
      uint4 w0, w1;
      uint32_t s, b;
    };
    auto load_raw = [&](int tile, int c, Raw& r) {
      const int o = (tile % mt) * kLgM + row;
      if (o >= a.N) {
        r.w0 = r.w1 = make_uint4(0, 0, 0, 0);
        r.s = r.b = 0;
        return;
      }
      const int k = k_lo + c;
      const uint32_t* p = a.packed + (size_t)o * (a.K >> 3) + k * 8;
      if (a.w_vec) {
        r.w0 = __ldg(reinterpret_cast<const uint4*>(p));
        r.w1 = __ldg(reinterpret_cast<const uint4*>(p) + 1);
      } else {
        r.w0 = make_uint4(p[0], p[1], p[2], p[3]);
        r.w1 = make_uint4(p[4], p[5], p[6], p[7]);
      }
      r.s = a.scales[(size_t)o * G + k];
      r.b = a.biases[(size_t)o * G + k];
    };
    uint32_t os = 0;
    int ti = 0;
    bool ok = true, waited = false;
    for (int tile = first_tile; tile < tiles && ok; tile += step, ++ti) {
      const int o = (tile % mt) * kLgM + row;
      // this group's stages of the tile: c = c0, c0 + 2, ...
      const int c0 = (int)((os ^ (uint32_t)grp) & 1u);
      Raw cur, nxt;
      if (c0 < nkm) load_raw(tile, c0, cur);
      if (c0 + 2 < nkm) load_raw(tile, c0 + 2, nxt);
      const int ew = weight_exponent(a, o);
      const float wsc = pow2(-ew);
      const LgList& L = S.list[ti & 1];
      int total = nkm, ng = 0;
      bool listed = false;
      const int npad = (tokens_of(tile) + 15) & ~15;
      for (int c = c0; ok; c += 2) {
        if (c >= nkm && !listed) {
          if (!warp_wait(&S.listfull[ti & 1], (ti >> 1) & 1, abort, a.status)) {
            ok = false;
            break;
          }
          ng = L.n_gran;
          total = nkm + lora_stages(ng);
          listed = true;
        }
        if (c >= total) break;
        const uint32_t oc = os + (uint32_t)c;
        const int st = (int)(oc % C::RO);
        if (oc >= (uint32_t)C::RO && !warp_wait(&S.opempty[st], ((oc / C::RO) - 1) & 1, abort, a.status)) {
          ok = false;
          break;
        }
        fence_after();
        const uint32_t ab = tmem + lane_addr + C::TMEM_A + (uint32_t)st * C::A_COLS;
        if (c < nkm) {
          const uint32_t wv[8] = {cur.w0.x, cur.w0.y, cur.w0.z, cur.w0.w, cur.w1.x, cur.w1.y, cur.w1.z, cur.w1.w};
          const float s = bf16_bits_to_f32(cur.s) * wsc, bi = bf16_bits_to_f32(cur.b) * wsc;
          cur = nxt;
          if (c + 4 < nkm) load_raw(tile, c + 4, nxt);
          if constexpr (F32) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint32_t hi[16], lo[16];
#pragma unroll
              for (int w = 0; w < 4; ++w) {
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                  const uint32_t word = wv[half * 4 + w] >> (8 * p);
                  const float f0 = fmaf(s, (float)(word & 15u), bi), f1 = fmaf(s, (float)((word >> 4) & 15u), bi);
                  const __half2 h = __floats2half2_rn(f0, f1);
                  const float2 b2 = __half22float2(h);
                  hi[4 * w + p] = h2u(h);
                  lo[4 * w + p] = h2u(__floats2half2_rn(f0 - b2.x, f1 - b2.y));
                }
              }
              st16(ab + (uint32_t)(half * 16), hi);
              st16(ab + (uint32_t)(32 + half * 16), lo);
            }
          } else {
            const __half2 s2 = __float2half2_rn(s), b2 = __float2half2_rn(bi), k1024 = u2h(0x64006400u);
            uint32_t av[32];
#pragma unroll
            for (int w = 0; w < 8; ++w) {
              const uint32_t l = wv[w] & 0x0F0F0F0Fu, h = (wv[w] >> 4) & 0x0F0F0F0Fu;
#pragma unroll
              for (int p = 0; p < 4; ++p)
                av[4 * w + p] = h2u(__hfma2(__hsub2(u2h(nib_pair(l, h, p) | 0x64006400u), k1024), s2, b2));
            }
            st32(ab, av);
          }
        } else {
          // a block of 64 columns: four pieces of 16 rows of adapters
          if (!waited) {
            pdl_wait();
            waited = true;
          }
          const int lc = c - nkm, blk = rank_c + lc / passes * split, pass = lc % passes;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int gi = blk * 4 + q;
            const int gr = gi < ng ? L.gran[gi] : 0xFFFF;
            uint32_t hi[8] = {}, lo[8] = {};
            if (gr != 0xFFFF && o < a.N) {
              const int id = L.id[gr >> 4], rank = L.rank[gr >> 4], j0 = (gr & 15) * 16;
              const size_t at = (size_t)id * a.b_stride + (size_t)o * a.rank + j0;
              float w[16];
              if (a.b_vec && j0 + 16 <= a.rank) {
                float w0[8], w1[8];
                load8<AT>(a.b, at, true, w0);
                load8<AT>(a.b, at + 8, true, w1);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  w[e] = j0 + e < rank ? w0[e] : 0.0f;
                  w[8 + e] = j0 + 8 + e < rank ? w1[e] : 0.0f;
                }
              } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) w[e] = j0 + e < rank ? load_val<AT>(a.b, at + e) : 0.0f;
              }
              bool bad = false;
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                if (!isfinite(w[e])) {
                  bad = true;
                  w[e] = 0.0f;
                }
                w[e] *= wsc;
              }
              if (bad) S.bad = 1;
#pragma unroll
              for (int p = 0; p < 8; ++p) {
                hi[p] = pack_bf2(w[2 * p], w[2 * p + 1]);
                lo[p] = pack_bf2(w[2 * p] - bf_lo(hi[p]), w[2 * p + 1] - bf_hi(hi[p]));
              }
            }
            __syncwarp();
            if constexpr (F32) {
              st8(ab + (uint32_t)(q * 8), hi);
              st8(ab + (uint32_t)(32 + q * 8), lo);
            } else {
              if (pass == 2) st8(ab + (uint32_t)(q * 8), lo);
              else st8(ab + (uint32_t)(q * 8), hi);
            }
          }
          unsigned char* dst = stages + (size_t)st * C::STAGE;
          for (int n = gt; n < npad; n += 128) {
            const int mine = L.first[n];
            const long long t = (long long)(tile / mt) * a.NT + n;
            const float xsc = mine != 0xFFFF ? pow2(-a.ex[t]) : 0.0f;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int gi = blk * 4 + q;
              const int gr = gi < ng ? L.gran[gi] : 0xFFFF;
              uint32_t p0[8] = {}, p1[8] = {};
              if (gr != 0xFFFF && (gr >> 4) == mine) {
                const float4* v = reinterpret_cast<const float4*>(a.v + (size_t)t * a.v_stride + (gr & 15) * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float4 f4 = v[e];
                  const float f[4] = {f4.x * xsc, f4.y * xsc, f4.z * xsc, f4.w * xsc};
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    const uint32_t v0 = pack_bf2(f[2 * h], f[2 * h + 1]);
                    const float r0 = f[2 * h] - bf_lo(v0), r1 = f[2 * h + 1] - bf_hi(v0);
                    const uint32_t v1 = pack_bf2(r0, r1);
                    if constexpr (F32) {
                      const uint32_t v2 = pack_bf2(r0 - bf_lo(v1), r1 - bf_hi(v1));
                      p0[2 * e + h] = pass == 0 ? v0 : v2;
                      p1[2 * e + h] = v1;
                    } else {
                      p0[2 * e + h] = pass == 1 ? v1 : v0;
                    }
                  }
                }
              }
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                unsigned char* at = dst + (size_t)n * 128 + (((2 * q + u) ^ (n & 7)) << 4);
                *reinterpret_cast<uint4*>(at) = make_uint4(p0[4 * u], p0[4 * u + 1], p0[4 * u + 2], p0[4 * u + 3]);
                if constexpr (F32)
                  *reinterpret_cast<uint4*>(at + (size_t)C::NMAX * 128) =
                      make_uint4(p1[4 * u], p1[4 * u + 1], p1[4 * u + 2], p1[4 * u + 3]);
              }
            }
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.opfull[st]);
      }
      if (!ok) break;
      if (!listed) {
        if (!warp_wait(&S.listfull[ti & 1], (ti >> 1) & 1, abort, a.status)) break;
        total = nkm + lora_stages(L.n_gran);
      }
      os += (uint32_t)total;
    }
  } else {
    // ---------------- epilogue ----------------
    const int quad = warp & 3, half = (warp - 2 - kLgConv) >> 2;
    const int row = quad * 32 + lane;
    const int n_mine = (warp - 2 - kLgConv) * 32 + lane;  // the token this thread lists
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    uint32_t eb = 0, gq = 0;
    // all epilogue warps meet (bounded, unlike a named barrier)
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.epi);
      const bool w = warp_wait(&S.epi, eb & 1, abort, a.status);
      ++eb;
      return w;
    };
    int ti = 0;
    for (int tile = first_tile; tile < tiles; tile += step, ++ti) {
      LgList& L = S.list[ti & 1];
      const long long tb = (long long)(tile / mt) * a.NT;
      const int ntok = tokens_of(tile), npad = (ntok + 15) & ~15;
      const int o = (tile % mt) * kLgM + row;
      // ---- the tile's adapters: first token of each, pieces of 16 rows ----
      int rank = 0, id = -1;
      if (a.adapter && n_mine < ntok) id = adapter_of(a, tb + n_mine, rank);
      L.id[n_mine] = id;
      L.rank[n_mine] = (uint16_t)rank;
      if (!meet()) break;
      int first = n_mine;
      if (id >= 0 && rank > 0) {
        const int4* ids4 = reinterpret_cast<const int4*>(L.id);
        for (int j = 0; j * 4 < n_mine; ++j) {
          const int4 v = ids4[j];
          const int f = v.x == id ? 0 : v.y == id ? 1 : v.z == id ? 2 : v.w == id ? 3 : 4;
          if (f < 4) {
            first = min(first, j * 4 + f);
            break;
          }
        }
      }
      L.first[n_mine] = id >= 0 && rank > 0 ? (uint16_t)first : (uint16_t)0xFFFF;
      const int mine = id >= 0 && rank > 0 && first == n_mine ? (rank + 15) >> 4 : 0;
      int incl = mine;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int up = __shfl_up_sync(kAllLanes, incl, s);
        if (lane >= s) incl += up;
      }
      if (lane == 31) L.wsum[warp - 2 - kLgConv] = incl;
      if (!meet()) break;
      int base = 0, all = 0;
      for (int w = 0; w < kLgEpi; ++w) {
        if (w < warp - 2 - kLgConv) base += L.wsum[w];
        all += L.wsum[w];
      }
      for (int i = 0; i < mine; ++i) L.gran[base + incl - mine + i] = (uint16_t)(n_mine << 4 | i);
      if (n_mine == 0) L.n_gran = all;
      __syncwarp();
      if (lane == 0) mbar_arrive(&S.listfull[ti & 1]);
      if (ti == 0) pdl_wait();  // what the prep kernel wrote; y may still be read before it
      L.ex[n_mine] = n_mine < ntok ? a.ex[tb + n_mine] : 0;
      const int ew = weight_exponent(a, o);
      if (half == 0) S.ew[row] = ew;
      if (!meet()) break;
      const int total = nkm + lora_stages(all);
      const bool live = o < a.N;
      float* part = reinterpret_cast<float*>(stages);  // split: [token][128 rows]
      auto put = [&](int n, float v) {
        v = scale_by(v, ew + L.ex[n]);
        if (S.bad && L.first[n] != 0xFFFF) v += bad_terms<AT>(a, L.id[n], L.rank[n], o, tb + n);
        store_val<XT>(a.y, (size_t)(tb + n) * a.y_stride + o, v);
      };
      if constexpr (F32) {
        float acc[64];
#pragma unroll
        for (int e = 0; e < 64; ++e) acc[e] = 0.0f;
        bool ok = true;
        for (int c = 0; c < total; c += C::GROUP, ++gq) {
          const int b = (int)(gq & 1);
          if (!warp_wait(&S.accfull[b], (gq >> 1) & 1, abort, a.status)) {
            ok = false;
            break;
          }
          fence_after();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c0 = (2 * i + half) * 16;
            if (c0 < npad) {
              uint32_t d[16];
              ld16(tmem + lane_addr + (uint32_t)(b * 128 + c0), d);
              wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) acc[i * 16 + e] += __uint_as_float(d[e]);
            }
          }
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&S.accempty[b]);
        }
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int n = (2 * i + half) * 16 + e;
            if (split > 1) {
              if (n < npad) part[n * kLgM + row] = acc[i * 16 + e];
            } else if (live && n < ntok) {
              put(n, acc[i * 16 + e]);
            }
          }
        }
      } else {
        const int b = nbuf == 2 ? (int)(gq & 1) : 0;
        if (!warp_wait(&S.accfull[b], (nbuf == 2 ? gq >> 1 : gq) & 1, abort, a.status)) break;
        fence_after();
        ++gq;
        for (int c0 = half * 16; c0 < npad; c0 += 32) {
          uint32_t d[16];
          ld16(tmem + lane_addr + (uint32_t)(b * 128 + c0), d);
          wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int n = c0 + e;
            if (split > 1) part[n * kLgM + row] = __uint_as_float(d[e]);
            else if (live && n < ntok) put(n, __uint_as_float(d[e]));
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&S.accempty[b]);
      }
    }
  }
  if (split > 1) {
    // the cluster's partial sums, each CTA a share of the tokens, added in the order of K
    __syncwarp();
    cluster_sync_all();
    const LgList& L = S.list[0];
    const int tile = first_tile, ntok = tokens_of(tile);
    const long long tb = (long long)(tile / mt) * a.NT;
    const int n_lo = ntok * rank_c / split, n_hi = ntok * (rank_c + 1) / split;
    bool bad = false;
    for (int r = 0; r < split; ++r) bad |= ld_cluster_i(map_rank(smem_addr(&S.bad), (uint32_t)r)) != 0;
    for (int i = tid; i < (n_hi - n_lo) * kLgM; i += kLgThreads) {
      const int n = n_lo + i / kLgM, row = i % kLgM, o = (tile % mt) * kLgM + row;
      if (o >= a.N || S.abort) continue;
      const uint32_t at = smem_addr(stages) + (uint32_t)(n * kLgM + row) * 4;
      float v = 0.0f;
      for (int r = 0; r < split; ++r) v += ld_cluster(map_rank(at, (uint32_t)r));
      v = scale_by(v, S.ew[row] + L.ex[n]);
      if (bad && L.first[n] != 0xFFFF) v += bad_terms<AT>(a, L.id[n], L.rank[n], o, tb + n);
      store_val<XT>(a.y, (size_t)(tb + n) * a.y_stride + o, v);
    }
    cluster_sync_all();  // no CTA ends while another reads its sums
  }
  fence_before();
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

template <bool F32>
constexpr size_t lg_smem() {
  return (size_t)LgCfg<F32>::RO * LgCfg<F32>::STAGE + sizeof(LgShared) + 1024;
}

// Tokens per tile and CTAs per tile (K split over a cluster): the smallest of
// a plain estimate in clocks.  A stage costs its matrix steps (N / 2 clocks
// each) or the conversion of its 128 x 64 weights, whichever is longer; a tile
// adds its epilogue, a split the exchange of the sums.
void lg_shape(const LoraArgs& a, int sms, int* NT, int* split) {
  const bool f32 = a.x_type == 0;
  const int nmax = f32 ? 128 : 256, nk = a.K >> 6;
  const long long mt = (a.N + kLgM - 1) / kLgM;
  double best = 1e300;
  *NT = 16;
  *split = 1;
  for (int n = 16; n <= nmax; n += 16) {
    if (n > 16 && n - 16 >= a.tokens) break;
    const long long tiles = mt * ((a.tokens + n - 1) / n);
    for (int s = 1; s <= 8; s *= 2) {
      if (s > nk || (s > 1 && tiles * s > (s == 8 ? 128 : sms))) break;
      const double waves = (double)((tiles * s + sms - 1) / sms);
      const double stage = f32 ? (6.0 * n > 450.0 ? 6.0 * n : 450.0) : (2.0 * n > 220.0 ? 2.0 * n : 220.0);
      const double t = waves * (((nk + s - 1) / s) * stage + 1500.0 + 12.0 * n + (s > 1 ? 1500.0 : 0.0));
      if (t < best) {
        best = t;
        *NT = n;
        *split = s;
      }
    }
  }
}

template <typename K>
cudaError_t launch_cfg(K kernel, dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t s, const LoraArgs& a) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
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
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int XT, int AT>
cudaError_t launch(const LoraArgs& a, int sms, cudaStream_t s, uint64_t* launches) {
  const unsigned tiles16 = (unsigned)((a.tokens + kPrepRows - 1) / kPrepRows);
  // blocks per tile for the adapters: up to the 16 a tile can hold, fewer
  // where the tiles alone fill the GPU
  unsigned ay = 0;
  if (a.adapter) {
    ay = (unsigned)(8 * sms) / tiles16;
    ay = ay < 1 ? 1 : ay > kPrepRows ? kPrepRows : ay;
    if (ay > (unsigned)a.count) ay = (unsigned)a.count;
    if (ay > (unsigned)a.tokens) ay = (unsigned)a.tokens;
  }
  cudaError_t e = launch_cfg(lora_prep_kernel<XT, AT>, dim3(tiles16, 1 + ay), dim3(kPrepWarps * 32), 0, 1, s, a);
  if (e != cudaSuccess) return e;
  const long long tiles = (long long)((a.N + kLgM - 1) / kLgM) * ((a.tokens + a.NT - 1) / a.NT);
  const unsigned grid = (unsigned)(a.split > 1 ? tiles * a.split : tiles < sms ? tiles : sms);
  e = launch_cfg(lora_gemm_kernel<XT, AT>, dim3(grid), dim3(kLgThreads), lg_smem<XT == 0>(), a.split, s, a);
  if (launches) *launches += 2;
  return e;
}

constexpr size_t kWsAlign = 1024;
size_t up(size_t v) { return (v + kWsAlign - 1) / kWsAlign * kWsAlign; }

// Tokens per pair of launches: operand planes of at most 256 MB, which keeps
// the workspace bounded (a multiple of 256 tokens).
long long block_tokens(const LoraArgs& a) {
  const long long row = (long long)a.K * (a.x_type == 0 ? 4 : 2);
  long long n = (256ll << 20) / row / 256 * 256;
  return n < 256 ? 256 : n;
}

size_t carve(LoraArgs& a, unsigned char* base) {
  const long long tiles = (a.tokens + a.NT - 1) / a.NT;
  const size_t planes = up((size_t)tiles * a.NT * a.K * (a.x_type == 0 ? 4 : 2));
  const size_t ex = up((size_t)((a.tokens + 15) / 16 * 16) * 4);
  a.v_stride = a.adapter ? ((size_t)a.rank + 15) / 16 * 16 : 0;
  a.planes = base;
  a.ex = reinterpret_cast<int*>(base + planes);
  a.v = reinterpret_cast<float*>(base + planes + ex);
  return planes + ex + up((size_t)a.tokens * a.v_stride * 4);
}

}  // namespace

cudaError_t init_lora_attributes(int max_smem) {
  if ((int)lg_smem<true>() > max_smem || (int)lg_smem<false>() > max_smem) return cudaErrorInvalidConfiguration;
  cudaError_t e = cudaSuccess;
  auto set = [&](auto kernel, size_t sm) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm);
  };
  set(lora_gemm_kernel<0, 1>, lg_smem<true>());
  set(lora_gemm_kernel<0, 2>, lg_smem<true>());
  set(lora_gemm_kernel<1, 1>, lg_smem<false>());
  set(lora_gemm_kernel<1, 2>, lg_smem<false>());
  set(lora_gemm_kernel<2, 1>, lg_smem<false>());
  set(lora_gemm_kernel<2, 2>, lg_smem<false>());
  return e;
}

size_t lora_workspace(const LoraArgs& args, int sms) {
  LoraArgs a = args;
  const long long all = a.tokens, most = block_tokens(a);
  size_t need = 0;
  for (long long n : {all < most ? all : most, all % most}) {
    if (n == 0) continue;
    a.tokens = n;
    lg_shape(a, sms, &a.NT, &a.split);
    const size_t b = carve(a, nullptr);
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
    lg_shape(a, sms, &a.NT, &a.split);
    carve(a, static_cast<unsigned char*>(workspace));
    a.x_vec = aligned(a.x, a.x_stride * ts);
    a.w_vec = aligned(a.packed, 0);
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
