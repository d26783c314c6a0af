// A whole mixture-of-experts layer for a few tokens (at most 64):
//
//   l = x Wr^T;  S = the k largest of a token's l (ties: lowest index);  p = softmax of l over S
//   out = shared + sum over e in S of  p_e Wout_e ( silu(Wg_e x) * (Wu_e x) )        Win_e = [Wg_e; Wu_e]
//
// With few tokens all time goes into reading the weights of the experts that some token takes, once each:
// 3 F D elements per expert, against N k 6 F D operations. So the weights travel straight from global memory
// into the registers of the warp that multiplies them, with nothing staged and nothing waited for in between,
// and the multiplication has to cost few instructions rather than reach a high rate. It is done on
// mma.sync tiles with the expert's tokens as the 16 rows and 8 weight rows as the columns: a lane then holds
// weights of one row only, and since a product's summands may be taken in any order, the four lanes of a
// weight row take 16 contiguous bytes each and tokens are read in the same order. (The tcgen05 tiles would need
// both operands in shared memory, 128 rows high, for 1 to 16 tokens.)
//
// Three launches, each waiting for its predecessor on the device: routing (one cluster), gate and up products
// with the activation, down product with the sum over a token's experts.
#include <algorithm>

#include "nsb_common.cuh"

namespace nsb {
namespace {

constexpr int kMaxTokens = 64, kMaxExperts = 1024, kMaxTopK = 16, kMaxSlots = kMaxTokens * kMaxTopK;
constexpr int kRouterCtas = 8, kRouterThreads = 1024;
constexpr int kWarps = 4, kThreads = 32 * kWarps;

struct MoeParams {
  const void *x, *shared, *w_router, *w_in, *w_out;
  void* out;
  long long x_stride;
  int N, E, K, D, F, Fp;  // Fp: F rounded up to whole 16-byte pieces
  int tiles;              // of the down product
  int* ids;               // [N, K] experts of a token, best first
  float* probs;           // [N, K]
  float* logits;          // [N, E]
  int* used;              // number of experts in use
  int* entries;           // [min(E, N K)][3] expert, first place in `slots`, number of tokens
  int* slots;             // [N K] token * K + j, by expert
  unsigned int* done;     // [tiles] units of the down product that have finished
  void* act;              // [N K, Fp] hidden values times p: bf16 as two terms, otherwise fp32
  float* part;            // [N K, D] down products
};

template <typename T>
__device__ __forceinline__ Vec<T, 16 / sizeof(T)> zero_chunk() {
  Vec<T, 16 / sizeof(T)> v;
#pragma unroll
  for (int i = 0; i < (int)(16 / sizeof(T)); ++i) v.v[i] = Elem<T>::zero();
  return v;
}
// 16 bytes of a row starting at element k, zeros beyond n. VEC: rows are 16-byte aligned and n is a multiple
// of a chunk. STREAM: read once, so it should not displace the tokens in the first-level cache.
template <typename T, bool VEC, bool STREAM>
__device__ __forceinline__ Vec<T, 16 / sizeof(T)> load_chunk(const T* row, int k, int n) {
  constexpr int C = 16 / sizeof(T);
  Vec<T, C> v = zero_chunk<T>();
  if constexpr (VEC) {
    if (row && k < n) {
      uint4 u;
      if constexpr (STREAM)
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(row + k));
      else
        u = *reinterpret_cast<const uint4*>(row + k);
      *reinterpret_cast<uint4*>(&v) = u;
    }
  } else {
    if (row)
#pragma unroll
      for (int i = 0; i < C; ++i)
        if (k + i < n) v.v[i] = row[k + i];
  }
  return v;
}

__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// v = hi + lo with hi and lo of 11 significant bits: what is left of v is below 2^-22 of it
__device__ __forceinline__ void split_tf32(float v, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(v));
  const float r = v - __uint_as_float(hi);
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(isfinite(r) ? r : 0.0f));
}

// acc += (token rows g and g + 8) x (weight row g) over one chunk per lane, inputs as they are
template <typename T>
__device__ __forceinline__ void mul_chunk(float (&acc)[4], const Vec<T, 8>& lo_row, const Vec<T, 8>& hi_row,
                                          const Vec<T, 8>& w) {
  const uint32_t* a = reinterpret_cast<const uint32_t*>(&lo_row);
  const uint32_t* b = reinterpret_cast<const uint32_t*>(&hi_row);
  const uint32_t* q = reinterpret_cast<const uint32_t*>(&w);
  mma16(acc, a[0], b[0], a[1], b[1], q[0], q[1], T());
  mma16(acc, a[2], b[2], a[3], b[3], q[2], q[3], T());
}
// fp32 operands: three products of 11-bit terms (the fourth, lo x lo, is below 2^-22)
template <int C>
__device__ __forceinline__ void mul_f32(float (&acc)[4], const float* a, const float* b, const float (&w)[C],
                                        bool w_exact) {
#pragma unroll
  for (int i = 0; i < C; i += 2) {
    uint32_t h[6], l[6];
    split_tf32(a[i], h[0], l[0]), split_tf32(b[i], h[1], l[1]);
    split_tf32(a[i + 1], h[2], l[2]), split_tf32(b[i + 1], h[3], l[3]);
    if (w_exact) h[4] = __float_as_uint(w[i]), h[5] = __float_as_uint(w[i + 1]);
    else split_tf32(w[i], h[4], l[4]), split_tf32(w[i + 1], h[5], l[5]);
    mma_tf32(acc, l[0], l[1], l[2], l[3], h[4], h[5]);
    if (!w_exact) mma_tf32(acc, h[0], h[1], h[2], h[3], l[4], l[5]);
    mma_tf32(acc, h[0], h[1], h[2], h[3], h[4], h[5]);
  }
}
__device__ __forceinline__ void mul_chunk(float (&acc)[4], const Vec<float, 4>& lo_row, const Vec<float, 4>& hi_row,
                                          const Vec<float, 4>& w) {
  mul_f32<4>(acc, lo_row.v, hi_row.v, w.v, false);
}

// ------------------------------------------------------------------------------------------ routing

__device__ __forceinline__ unsigned long long order_key(float v, int index) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // (-0 and 0 tie)
  const uint32_t s = (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return ((unsigned long long)s << 32) | (0xffffffffu - (uint32_t)index);
}

// One cluster of 8 CTAs. A warp takes an expert and four tokens at a time; when all logits are there, the
// first CTA picks every token's experts (a warp per token) and lists the tokens of every expert.
template <typename T, bool VEC>
__global__ void __cluster_dims__(kRouterCtas, 1, 1) __launch_bounds__(kRouterThreads) moe_route_kernel(const MoeParams p) {
  constexpr int C = 16 / sizeof(T);
  __shared__ uint16_t s_ids[kMaxSlots];
  __shared__ int s_count[kMaxExperts], s_first[kMaxExperts], s_place[kMaxExperts], s_warp[2][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_dependents_may_launch();
  const T* x = static_cast<const T*>(p.x);
  const T* wr = static_cast<const T*>(p.w_router);
  const int groups = (p.N + 3) / 4;
  for (int i = blockIdx.x * (kRouterThreads / 32) + warp; i < p.E * groups; i += kRouterCtas * (kRouterThreads / 32)) {
    const int e = i % p.E, n0 = i / p.E * 4;
    float acc[4] = {};
    for (int k = lane * C; k < p.D; k += 32 * C) {
      const Vec<T, C> w = load_chunk<T, VEC, false>(wr + (long long)e * p.D, k, p.D);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const Vec<T, C> v = load_chunk<T, VEC, false>(n0 + t < p.N ? x + (n0 + t) * p.x_stride : nullptr, k, p.D);
#pragma unroll
        for (int j = 0; j < C; ++j) acc[t] = fmaf(Elem<T>::to_f32(v.v[j]), Elem<T>::to_f32(w.v[j]), acc[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[t] += __shfl_xor_sync(0xffffffffu, acc[t], o);
      if (lane == 0 && n0 + t < p.N) p.logits[(n0 + t) * p.E + e] = acc[t];
    }
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (blockIdx.x != 0) return;

  for (int n = warp; n < p.N; n += kRouterThreads / 32) {
    uint32_t taken = 0;
    float best = 0.0f, l_j = 0.0f;
    for (int j = 0; j < p.K; ++j) {
      unsigned long long top = 0;
      for (int i = 0; i * 32 + lane < p.E; ++i)
        if (!((taken >> i) & 1u)) {
          const unsigned long long key = order_key(p.logits[n * p.E + i * 32 + lane], i * 32 + lane);
          top = key > top ? key : top;
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long q = __shfl_xor_sync(0xffffffffu, top, o);
        top = q > top ? q : top;
      }
      const int e = (int)(0xffffffffu - (uint32_t)top);
      if ((e & 31) == lane) taken |= 1u << (e >> 5);
      const float l = p.logits[n * p.E + e];
      if (j == 0) best = l;
      if (lane == j) l_j = l;
      if (lane == 0) {
        p.ids[n * p.K + j] = e;
        s_ids[n * p.K + j] = (uint16_t)e;
      }
    }
    const float w = lane < p.K ? expf(l_j - best) : 0.0f;
    float sum = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane < p.K) p.probs[n * p.K + lane] = w / sum;
  }
  __syncthreads();
  // thread e counts expert e's tokens; sums over the threads before it give its place among the experts in
  // use and in the list of slots
  const int e = threadIdx.x, slots = p.N * p.K;
  int count = 0;
  if (e < p.E)
    for (int i = 0; i < slots; ++i) count += s_ids[i] == e;
  int before = count, rank = count > 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, before, o), b = __shfl_up_sync(0xffffffffu, rank, o);
    if (lane >= o) before += a, rank += b;
  }
  if (lane == 31) s_warp[0][warp] = before, s_warp[1][warp] = rank;
  __syncthreads();
  for (int w = 0; w < warp; ++w) before += s_warp[0][w], rank += s_warp[1][w];
  if (threadIdx.x == kRouterThreads - 1) *p.used = rank;
  if (count > 0) {
    int at = before - count;
    p.entries[3 * (rank - 1)] = e;
    p.entries[3 * (rank - 1) + 1] = at;
    p.entries[3 * (rank - 1) + 2] = count;
    for (int i = 0; i < slots; ++i)
      if (s_ids[i] == e) p.slots[at++] = i;
  }
  for (int i = threadIdx.x; i < p.tiles; i += kRouterThreads) p.done[i] = 0u;
}

// ------------------------------------------------------------------------------------------ products

// How the warps of a CTA share out a unit: WK of them take every WK-th block of the summation index, 4 / WK units
// lie side by side. Block: 4 steps of 4 chunks.
constexpr int kSteps = 4;

__device__ __forceinline__ float silu(float v) { return v / (1.0f + expf(-v)); }

template <typename T>
struct ActRow;  // a token's hidden values for one chunk, as the down product wants them
template <>
struct ActRow<__nv_bfloat16> {
  // bf16 weights: the hidden value as the sum of two bf16 numbers, 16 significant bits; rounding it to one would
  // add an error as large as that of the rounded output itself
  Vec<__nv_bfloat16, 8> hi, lo;
};
template <>
struct ActRow<__half> {  // fp16 weights are exact in 11 bits, and the hidden value may lie outside fp16's range
  Vec<float, 8> v;
};
template <>
struct ActRow<float> {
  Vec<float, 4> v;
};
__device__ __forceinline__ void mul_act(float (&acc)[4], const ActRow<__nv_bfloat16>& a, const ActRow<__nv_bfloat16>& b,
                                        const Vec<__nv_bfloat16, 8>& w) {
  mul_chunk<__nv_bfloat16>(acc, a.lo, b.lo, w);
  mul_chunk<__nv_bfloat16>(acc, a.hi, b.hi, w);
}
__device__ __forceinline__ void mul_act(float (&acc)[4], const ActRow<__half>& a, const ActRow<__half>& b,
                                        const Vec<__half, 8>& w) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __half2float(w.v[i]);
  mul_f32<8>(acc, a.v.v, b.v.v, f, true);
}
__device__ __forceinline__ void mul_act(float (&acc)[4], const ActRow<float>& a, const ActRow<float>& b,
                                        const Vec<float, 4>& w) {
  mul_f32<4>(acc, a.v.v, b.v.v, w.v, false);
}
template <typename T>
__device__ __forceinline__ ActRow<T> load_act(const void* act, long long slots, int slot, int Fp, int k) {
  ActRow<T> r;
  if constexpr (sizeof(T) == 2 && Elem<T>::kDtype == NSB_BF16) {
    r.hi = r.lo = zero_chunk<T>();
    if (slot >= 0 && k < Fp) {
      const T* row = static_cast<const T*>(act) + (long long)slot * Fp + k;
      r.hi = *reinterpret_cast<const Vec<T, 8>*>(row);
      r.lo = *reinterpret_cast<const Vec<T, 8>*>(row + slots * Fp);
    }
  } else {
    constexpr int C = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < C; ++i) r.v.v[i] = 0.0f;
    if (slot >= 0 && k < Fp) {
      const float* row = static_cast<const float*>(act) + (long long)slot * Fp + k;
#pragma unroll
      for (int i = 0; i < C; i += 4)
        *reinterpret_cast<Vec<float, 4>*>(&r.v.v[i]) = *reinterpret_cast<const Vec<float, 4>*>(row + i);
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store_act(void* act, long long slots, int slot, int Fp, int f, float v) {
  if constexpr (sizeof(T) == 2 && Elem<T>::kDtype == NSB_BF16) {
    T* at = static_cast<T*>(act) + (long long)slot * Fp + f;
    const T hi = __float2bfloat16_rn(v);
    const float r = v - __bfloat162float(hi);
    at[0] = hi;
    at[slots * Fp] = __float2bfloat16_rn(isfinite(r) ? r : 0.0f);
  } else {
    static_cast<float*>(act)[(long long)slot * Fp + f] = v;
  }
}

// Adds up the WK warps' accumulators of a unit in the order of the warps; the first of them has the sum.
template <int R>
__device__ __forceinline__ void add_up(float (&acc)[R], float* buf, int wk, int WK) {
  if (WK == 1) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i) buf[i * kThreads + threadIdx.x] = acc[i];
  __syncthreads();
  if (wk == 0)
    for (int w = 1; w < WK; ++w)
#pragma unroll
      for (int i = 0; i < R; ++i) acc[i] += buf[i * kThreads + threadIdx.x + 32 * w];
}

// Unit: 8 hidden values of one expert for all its tokens (8 gate rows and 8 up rows of Win).
template <typename T, bool VEC, int MT>
__global__ void __launch_bounds__(kThreads) moe_up_kernel(const MoeParams p, int WK) {
  constexpr int C = 16 / sizeof(T);
  __shared__ float buf[MT * 8 * kThreads];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int wk = warp % WK, per_cta = kWarps / WK;
  grid_dependents_may_launch();
  grid_dependency_wait();
  const int per_expert = (p.F + 7) / 8, ctas = (per_expert + per_cta - 1) / per_cta;
  const int place = blockIdx.x / ctas;
  if (place >= *p.used) return;
  const int e = p.entries[3 * place], first = p.entries[3 * place + 1], n = p.entries[3 * place + 2];
  const int f0 = ((blockIdx.x % ctas) * per_cta + warp / WK) * 8;
  const int mtiles = (n + 15) / 16;
  const T* gate_row = nullptr;
  const T* up_row = nullptr;
  if (f0 + g < p.F) {
    gate_row = static_cast<const T*>(p.w_in) + ((long long)e * 2 * p.F + f0 + g) * p.D;
    up_row = gate_row + (long long)p.F * p.D;
  }
  const T* rows[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = m * 16 + h * 8 + g;
      rows[m][h] = i < n ? static_cast<const T*>(p.x) + (p.slots[first + i] / p.K) * p.x_stride : nullptr;
    }
  float acc[MT * 8];
#pragma unroll
  for (int i = 0; i < MT * 8; ++i) acc[i] = 0.0f;
  auto part = [&](int i) -> float(&)[4] { return *reinterpret_cast<float(*)[4]>(&acc[4 * i]); };
  constexpr int kBlock = kSteps * 4 * C;
  for (int k0 = wk * kBlock; k0 < p.D; k0 += WK * kBlock) {
    Vec<T, C> wg[kSteps], wu[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int k = k0 + (s * 4 + t) * C;
      wg[s] = load_chunk<T, VEC, true>(gate_row, k, p.D);
      wu[s] = load_chunk<T, VEC, true>(up_row, k, p.D);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m >= mtiles) break;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int k = k0 + (s * 4 + t) * C;
        const Vec<T, C> a = load_chunk<T, VEC, false>(rows[m][0], k, p.D);
        const Vec<T, C> b = load_chunk<T, VEC, false>(rows[m][1], k, p.D);
        mul_chunk(part(2 * m), a, b, wg[s]);
        mul_chunk(part(2 * m + 1), a, b, wu[s]);
      }
    }
  }
  add_up<MT * 8>(acc, buf, wk, WK);
  if (wk != 0) return;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = m * 16 + (i >> 1) * 8 + g, f = f0 + 2 * t + (i & 1);
      if (row < n && f < p.Fp) {
        const int slot = p.slots[first + row];
        const float v = f < p.F ? silu(part(2 * m)[i]) * part(2 * m + 1)[i] * p.probs[slot] : 0.0f;
        store_act<T>(p.act, p.N * p.K, slot, p.Fp, f, v);
      }
    }
}

// Unit: 16 outputs of one expert for all its tokens. The last unit of an output tile adds up the token's experts.
template <typename T, bool VEC, int MT>
__global__ void __launch_bounds__(kThreads) moe_down_kernel(const MoeParams p, int WK) {
  constexpr int C = 16 / sizeof(T);
  __shared__ float buf[MT * 8 * kThreads];
  __shared__ bool s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int wk = warp % WK, per_cta = kWarps / WK;
  grid_dependency_wait();
  const int ctas = p.tiles;  // tiles of 16 per_cta outputs
  const int place = blockIdx.x / ctas, tile = blockIdx.x % ctas, used = *p.used;
  if (place >= used) return;
  const int e = p.entries[3 * place], first = p.entries[3 * place + 1], n = p.entries[3 * place + 2];
  const int d0 = (tile * per_cta + warp / WK) * 16;
  const int mtiles = (n + 15) / 16;
  const T* w_row[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    w_row[h] = d0 + 8 * h + g < p.D ? static_cast<const T*>(p.w_out) + ((long long)e * p.D + d0 + 8 * h + g) * p.F : nullptr;
  int rows[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = m * 16 + h * 8 + g;
      rows[m][h] = i < n ? p.slots[first + i] : -1;
    }
  float acc[MT * 8];
#pragma unroll
  for (int i = 0; i < MT * 8; ++i) acc[i] = 0.0f;
  auto part = [&](int i) -> float(&)[4] { return *reinterpret_cast<float(*)[4]>(&acc[4 * i]); };
  constexpr int kBlock = kSteps * 4 * C;
  for (int k0 = wk * kBlock; k0 < p.F; k0 += WK * kBlock) {
    Vec<T, C> w[kSteps][2];
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) w[s][h] = load_chunk<T, VEC, true>(w_row[h], k0 + (s * 4 + t) * C, p.F);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m >= mtiles) break;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int k = k0 + (s * 4 + t) * C;
        const ActRow<T> a = load_act<T>(p.act, p.N * p.K, rows[m][0], p.Fp, k);
        const ActRow<T> b = load_act<T>(p.act, p.N * p.K, rows[m][1], p.Fp, k);
        mul_act(part(2 * m), a, b, w[s][0]);
        mul_act(part(2 * m + 1), a, b, w[s][1]);
      }
    }
  }
  add_up<MT * 8>(acc, buf, wk, WK);
  if (wk == 0) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = m * 16 + ((i >> 1) & 1) * 8 + g, d = d0 + (i >> 2) * 8 + 2 * t + (i & 1);
        if (row < n && d < p.D) p.part[(long long)p.slots[first + row] * p.D + d] = acc[m * 8 + i];
      }
    __threadfence();
  }
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(p.done + tile, 1u) + 1u == (unsigned)used;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  const int width = 16 * per_cta, base = tile * width;
  for (int i = threadIdx.x; i < p.N * width; i += kThreads) {
    const int tok = i / width, d = base + i % width;
    if (d >= p.D) continue;
    float sum = p.shared ? Elem<T>::to_f32(static_cast<const T*>(p.shared)[(long long)tok * p.D + d]) : 0.0f;
    for (int j = 0; j < p.K; ++j) sum += __ldcg(p.part + ((long long)tok * p.K + j) * p.D + d);
    static_cast<T*>(p.out)[(long long)tok * p.D + d] = Elem<T>::from_f32(sum);
  }
}

// ------------------------------------------------------------------------------------------ host

bool ok_dtype(int d) { return d == NSB_F32 || d == NSB_BF16 || d == NSB_F16; }
bool fits(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
long long up16(long long n) { return (n + 15) / 16 * 16; }

struct Layout {  // of the workspace, in bytes
  long long logits, used, entries, slots, done, act, part, bytes;
};
Layout layout(long long N, long long E, long long K, long long D, long long F) {
  const long long S = N * K, Fp = (F + 7) / 8 * 8;
  Layout l;
  l.logits = 0;
  l.used = up16(N * E * 4);
  l.entries = l.used + 16;
  l.slots = l.entries + up16(12 * std::min(E, S));
  l.done = l.slots + up16(4 * S);
  l.act = l.done + up16(4 * ((D + 15) / 16));
  l.part = l.act + 4 * S * Fp;
  l.bytes = l.part + 4 * S * D;
  return l;
}
int check_sizes(int64_t N, int64_t E, int64_t K, int64_t D, int64_t F) {
  if (N < 0 || E < 1 || K < 1 || K > E || D < 0 || F < 0) return NSB_ERR_INVALID_ARG;
  if (N > kMaxTokens || E > kMaxExperts || K > kMaxTopK || D > (1 << 20) || F > (1 << 20)) return NSB_ERR_TOO_LARGE;
  return NSB_OK;
}

// Warps along the summation index: as few as leave two CTAs per SM's worth of units, so that the fewest units
// (one token, two experts) still read from every SM.
int split(long long units, int sms) {
  int wk = 1;
  while (wk < kWarps && units * wk < 8LL * kWarps * sms) wk *= 2;
  return wk;
}

template <typename T, bool VEC, int MT>
int launch_products(MoeParams p, int sms, cudaStream_t st) {
  const long long experts = std::min(p.E, p.N * p.K);
  const int per_up = (p.F + 7) / 8, wk_up = split(experts * per_up, sms);
  const int ctas_up = (per_up + kWarps / wk_up - 1) / (kWarps / wk_up);
  const int per_down = (p.D + 15) / 16, wk_down = split(experts * per_down, sms);
  p.tiles = (per_down + kWarps / wk_down - 1) / (kWarps / wk_down);
  if (experts * std::max(ctas_up, p.tiles) > 0x7fffffffLL) return NSB_ERR_TOO_LARGE;
  moe_route_kernel<T, VEC><<<kRouterCtas, kRouterThreads, 0, st>>>(p);
  NSB_CUDA_TRY(cudaGetLastError(), "launch moe_route_kernel");
  if (p.D == 0) return NSB_OK;
  if (p.F > 0)
    NSB_CUDA_TRY(launch_dependent(moe_up_kernel<T, VEC, MT>, dim3((unsigned)(experts * ctas_up)), dim3(kThreads), 0, st, p, wk_up),
                 "launch moe_up_kernel");
  NSB_CUDA_TRY(launch_dependent(moe_down_kernel<T, VEC, MT>, dim3((unsigned)(experts * p.tiles)), dim3(kThreads), 0, st, p,
                                wk_down), "launch moe_down_kernel");
  return NSB_OK;
}
template <typename T>
int launch_moe(MoeParams p, cudaStream_t st) {
  DeviceInfo dev;
  const int r = get_device_info(&dev);
  if (r != NSB_OK) return r;
  constexpr int C = 16 / sizeof(T);
  bool vec = p.D % C == 0 && p.F % C == 0 && p.x_stride % C == 0;
  for (const void* q : {p.x, p.w_router, p.w_in, p.w_out}) vec = vec && fits(q, 16);
  const int mt = p.N <= 16 ? 1 : p.N <= 32 ? 2 : 4;
#define NSB_GO(V_) \
  (mt == 1 ? launch_products<T, V_, 1>(p, dev.sm_count, st) : mt == 2 ? launch_products<T, V_, 2>(p, dev.sm_count, st) \
                                                                      : launch_products<T, V_, 4>(p, dev.sm_count, st))
  return vec ? NSB_GO(true) : NSB_GO(false);
#undef NSB_GO
}

}  // namespace
}  // namespace nsb

using namespace nsb;

extern "C" int64_t nsb_moe_few_tokens_scratch_bytes(int64_t N, int64_t E, int64_t K, int64_t D, int64_t F) {
  return check_sizes(N, E, K, D, F) == NSB_OK ? layout(N, E, K, D, F).bytes : 0;
}

extern "C" int nsb_moe_few_tokens(const void* x, int64_t x_stride, const void* w_router, const void* w_in, const void* w_out,
                                  const void* shared, void* out, int32_t* ids, float* probs, void* scratch, int64_t N,
                                  int64_t E, int64_t K, int64_t D, int64_t F, int dtype, void* stream) {
  if (!ok_dtype(dtype)) return NSB_ERR_INVALID_ARG;
  const int r = check_sizes(N, E, K, D, F);
  if (r != NSB_OK) return r;
  if (N == 0) return NSB_OK;
  const size_t es = dtype_size(dtype);
  if (!ids || !probs || !scratch || !fits(ids, 4) || !fits(probs, 4) || !fits(scratch, 16)) return NSB_ERR_INVALID_ARG;
  if (D > 0 && (!x || !w_router || !out || (F > 0 && (!w_in || !w_out)))) return NSB_ERR_INVALID_ARG;
  for (const void* q : {x, w_router, w_in, w_out, shared, (const void*)out})
    if (!fits(q, es)) return NSB_ERR_INVALID_ARG;
  MoeParams p = {};
  p.x = x, p.shared = shared, p.w_router = w_router, p.w_in = w_in, p.w_out = w_out, p.out = out;
  p.x_stride = x_stride;
  p.N = (int)N, p.E = (int)E, p.K = (int)K, p.D = (int)D, p.F = (int)F, p.Fp = (int)((F + 7) / 8 * 8);
  const Layout l = layout(N, E, K, D, F);
  char* base = static_cast<char*>(scratch);
  p.ids = ids, p.probs = probs;
  p.logits = reinterpret_cast<float*>(base + l.logits);
  p.used = reinterpret_cast<int*>(base + l.used);
  p.entries = reinterpret_cast<int*>(base + l.entries);
  p.slots = reinterpret_cast<int*>(base + l.slots);
  p.done = reinterpret_cast<unsigned int*>(base + l.done);
  p.act = base + l.act;
  p.part = reinterpret_cast<float*>(base + l.part);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case NSB_F32: return launch_moe<float>(p, st);
    case NSB_BF16: return launch_moe<__nv_bfloat16>(p, st);
    default: return launch_moe<__half>(p, st);
  }
}
