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
  float* lparts;          // [CTAs of the cluster][N, E] partial logits
  int* used;              // number of experts in use
  int* entries;           // [min(E, N K)][3] expert, first place in `slots`, number of tokens
  int* slots;             // [N K] token * K + j, by expert
  unsigned int* done;     // [tiles] units of the down product that have finished
  void* act;              // hidden values times p, [terms][N K, Fp]: bf16 three bf16 terms, fp16 two tf32 ones, fp32 one
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
// of a chunk. STREAM: read once, so it should not displace the tokens in the first-level cache. WHOLE: all of the chunk
// lies before n.
template <typename T, bool VEC, bool STREAM, bool WHOLE>
__device__ __forceinline__ Vec<T, 16 / sizeof(T)> load_chunk(const T* row, int k, int n) {
  constexpr int C = 16 / sizeof(T);
  Vec<T, C> v;
  if constexpr (VEC) {
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (WHOLE || k < n) {
      if constexpr (STREAM)
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(row + k));
      else
        u = *reinterpret_cast<const uint4*>(row + k);
    }
    *reinterpret_cast<uint4*>(&v) = u;
  } else {
    v = zero_chunk<T>();
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (WHOLE || k + i < n) v.v[i] = row[k + i];
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

// acc += (token rows g and g + 8) x (weight row g) over one chunk per lane, inputs as they are (from zero: see add_chunk)
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
__device__ __forceinline__ void mul_chunk(float (&acc)[4], const Vec<float, 4>& lo_row, const Vec<float, 4>& hi_row,
                                          const Vec<float, 4>& w) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    uint32_t h[6], l[6];
    split_tf32(lo_row.v[i], h[0], l[0]), split_tf32(hi_row.v[i], h[1], l[1]);
    split_tf32(lo_row.v[i + 1], h[2], l[2]), split_tf32(hi_row.v[i + 1], h[3], l[3]);
    split_tf32(w.v[i], h[4], l[4]), split_tf32(w.v[i + 1], h[5], l[5]);
    mma_tf32(acc, l[0], l[1], l[2], l[3], h[4], h[5]);
    mma_tf32(acc, h[0], h[1], h[2], h[3], l[4], l[5]);
    mma_tf32(acc, h[0], h[1], h[2], h[3], h[4], h[5]);
  }
}

// The tensor core rounds what it adds to an accumulator toward zero, so one that lived for a whole row would shrink by up to
// a unit in the last place per product: outputs 2.1e-5 off in fp32 for 64 tokens, 4096 x 1792, where the sum to the nearest
// is 2e-7 off. So a chunk's product starts from zero, and chunks are added up in fp32 to the nearest (920 -> 1001 us there; no
// time in bf16).
__device__ __forceinline__ void add_chunk(float (&acc)[4], const float (&part)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] += part[i];
}

// ------------------------------------------------------------------------------------------ routing

__device__ __forceinline__ unsigned long long order_key(float v, int index) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // (-0 and 0 tie)
  const uint32_t s = (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return ((unsigned long long)s << 32) | (0xffffffffu - (uint32_t)index);
}

// How the cluster's warps share out the logits: tiles of 16 tokens x 8 experts; the blocks of the summation index go
// round the CTAs, and within a CTA `split` warps take every split-th of its blocks of a tile.
struct RouteShare {
  int etiles, tiles, split;
  __host__ __device__ RouteShare(int N, int E) {
    etiles = (E + 7) / 8;
    tiles = (N + 15) / 16 * etiles;
    split = 1;
    while (split * 2 * (tiles > 0 ? tiles : 1) <= kRouterThreads / 32) split *= 2;
  }
};
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// One cluster of 8 CTAs: partial logits, their sums, every token's choice (a warp per token), and in the first CTA the
// list of every expert's tokens; a cluster barrier between each. The partial sums are added in a fixed order.
template <typename T, bool VEC>
__global__ void __cluster_dims__(kRouterCtas, 1, 1) __launch_bounds__(kRouterThreads) moe_route_kernel(const MoeParams p) {
  constexpr int C = 16 / sizeof(T);
  __shared__ __align__(16) uint16_t s_ids[kMaxSlots];
  __shared__ int s_warp[2][32];
  __shared__ float s_acc[4][kRouterThreads];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = blockIdx.x;
  const int g = lane >> 2, t = lane & 3;
  grid_dependents_may_launch();
  const RouteShare share(p.N, p.E);
  const T* x = static_cast<const T*>(p.x);
  const T* wr = static_cast<const T*>(p.w_router);
  const int sw = warp % share.split, parts = kRouterCtas * share.split;
  float* part = p.lparts + (long long)rank * p.N * p.E;
  for (int i = warp / share.split; i < share.tiles; i += kRouterThreads / 32 / share.split) {
    const int n0 = i / share.etiles * 16, e0 = i % share.etiles * 8;
    // (rows beyond the last stand for tokens and experts that nobody asks for)
    const T* row_a = x + min(n0 + g, p.N - 1) * p.x_stride;
    const T* row_b = x + min(n0 + g + 8, p.N - 1) * p.x_stride;
    const T* row_w = wr + (long long)min(e0 + g, p.E - 1) * p.D;
    float acc[4] = {};
#pragma unroll 4
    for (int k = (rank * share.split + sw) * 4 * C + t * C; k - t * C < p.D; k += parts * 4 * C) {
      float part_acc[4] = {};
      mul_chunk(part_acc, load_chunk<T, VEC, false, false>(row_a, k, p.D), load_chunk<T, VEC, false, false>(row_b, k, p.D),
                load_chunk<T, VEC, false, false>(row_w, k, p.D));
      add_chunk(acc, part_acc);
    }
    if (share.split > 1) {  // (then every warp has one tile at most)
#pragma unroll
      for (int j = 0; j < 4; ++j) s_acc[j][threadIdx.x] = acc[j];
    }
    if (share.split == 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + g + (j >> 1) * 8, e = e0 + 2 * t + (j & 1);
        if (n < p.N && e < p.E) part[n * p.E + e] = acc[j];
      }
  }
  if (share.split > 1) {
    __syncthreads();
    const int i = warp / share.split, n0 = i / share.etiles * 16, e0 = i % share.etiles * 8;
    if (sw == 0 && i < share.tiles)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + g + (j >> 1) * 8, e = e0 + 2 * t + (j & 1);
        float sum = s_acc[j][threadIdx.x];
        for (int k = 1; k < share.split; ++k) sum += s_acc[j][threadIdx.x + 32 * k];
        if (n < p.N && e < p.E) part[n * p.E + e] = sum;
      }
  }
  cluster_barrier();
  for (int i = rank * kRouterThreads + threadIdx.x; i < p.N * p.E; i += kRouterCtas * kRouterThreads) {
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kRouterCtas; ++j) sum += __ldcg(p.lparts + (long long)j * p.N * p.E + i);
    p.logits[i] = sum;
  }
  cluster_barrier();
  for (int n = rank + kRouterCtas * warp; n < p.N; n += kRouterCtas * (kRouterThreads / 32)) {
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
      if (lane == 0) p.ids[n * p.K + j] = e;
    }
    const float w = lane < p.K ? expf(l_j - best) : 0.0f;
    float sum = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane < p.K) p.probs[n * p.K + lane] = w / sum;
  }
  cluster_barrier();
  if (rank != 0) return;

  // thread e counts expert e's tokens; sums over the threads before it give its place among the experts in
  // use and in the list of slots
  const int e = threadIdx.x, slots = p.N * p.K;
  for (int i = threadIdx.x; i < kMaxSlots; i += kRouterThreads) s_ids[i] = i < slots ? (uint16_t)__ldcg(p.ids + i) : 0xffffu;
  __syncthreads();
  auto visit = [&](auto f) {  // f(slot) for every slot of expert e, in order
    for (int i = 0; i < slots; i += 8) {
      const uint4 q = *reinterpret_cast<const uint4*>(s_ids + i);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if ((w[j] & 0xffffu) == (uint32_t)e) f(i + 2 * j);
        if (w[j] >> 16 == (uint32_t)e) f(i + 2 * j + 1);
      }
    }
  };
  int count = 0;
  if (e < p.E) visit([&](int) { ++count; });
  int before = count, place = count > 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, before, o), b = __shfl_up_sync(0xffffffffu, place, o);
    if (lane >= o) before += a, place += b;
  }
  if (lane == 31) s_warp[0][warp] = before, s_warp[1][warp] = place;
  __syncthreads();
  for (int w = 0; w < warp; ++w) before += s_warp[0][w], place += s_warp[1][w];
  if (threadIdx.x == kRouterThreads - 1) *p.used = place;
  if (count > 0) {
    int at = before - count;
    p.entries[3 * (place - 1)] = e;
    p.entries[3 * (place - 1) + 1] = at;
    p.entries[3 * (place - 1) + 2] = count;
    visit([&](int i) { p.slots[at++] = i; });
  }
  for (int i = threadIdx.x; i < p.tiles; i += kRouterThreads) p.done[i] = 0u;
}

// ------------------------------------------------------------------------------------------ products

// WK warps of a CTA share a unit, each with every WK-th block of the summation index, and 4 / WK units lie side by side.
// Block: some steps of 4 chunks.
// Steps of a block and CTAs per SM (registers): a warp of the up product has 4 x 1 KB of weights and the tokens' chunks for
// them on their way; the down product, whose tokens come as two or three terms, 1 x 1 KB, and more warps. Measured with others, by
// steps and CTAs: the up product, with two terms in both, (4, 3) 156 us for 16 tokens in fp16 and 303 us for 64 in bf16, (2, 5) 167 and
// 314 beside (2, 4) below; the down product (1, 5) 208 (it spills) and 316, (1, 4) 157 and 324, (1, 3) 174 and 352, (2, 3) 208 and 336.
constexpr int kUpSteps = 4, kDownSteps = 1;
template <typename T>
constexpr int kDownCtas = Elem<T>::kDtype == NSB_F16 ? 4 : 5;

__device__ __forceinline__ float silu(float v) { return v / (1.0f + expf(-v)); }

// A token's hidden values for one chunk, as the down product wants them: with fp32's range (in fp16 they may overflow) and its
// digits, because an error of theirs is one of the output before it is rounded. bf16 weights: the sum of three bf16 numbers,
// 3 x 8 bits, which leaves 2^-24. fp16 weights: they are tf32 numbers as they stand, and the hidden value is the
// sum of two of those, which leaves 2^-22. (Two bf16 terms for both, 2^-16, rounded two to three times as many outputs to a
// neighbour of the plain form's value. For 64 tokens x 4 of 32 experts, 4096 x 1792, they took 291 us instead of 316 in bf16 and 322 instead of
// 350 in fp16; for 16 tokens in fp16 157 both.)
template <typename T>
struct ActRow;
template <>
struct ActRow<__nv_bfloat16> {
  Vec<__nv_bfloat16, 8> v[3];
};
template <>
struct ActRow<__half> {
  Vec<float, 4> hi[2], lo[2];
};
template <>
struct ActRow<float> {
  Vec<float, 4> v;
};
__device__ __forceinline__ void mul_act(float (&acc)[4], const ActRow<__nv_bfloat16>& a, const ActRow<__nv_bfloat16>& b,
                                        const Vec<__nv_bfloat16, 8>& w) {
#pragma unroll
  for (int i = 2; i >= 0; --i) mul_chunk<__nv_bfloat16>(acc, a.v[i], b.v[i], w);
}
__device__ __forceinline__ void mul_act(float (&acc)[4], const ActRow<__half>& a, const ActRow<__half>& b,
                                        const Vec<__half, 8>& w) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w.v[i]));
    const uint32_t w0 = __float_as_uint(f.x), w1 = __float_as_uint(f.y);
    const int h = i / 4, j = i % 4;
    mma_tf32(acc, __float_as_uint(a.lo[h].v[j]), __float_as_uint(b.lo[h].v[j]), __float_as_uint(a.lo[h].v[j + 1]),
             __float_as_uint(b.lo[h].v[j + 1]), w0, w1);
    mma_tf32(acc, __float_as_uint(a.hi[h].v[j]), __float_as_uint(b.hi[h].v[j]), __float_as_uint(a.hi[h].v[j + 1]),
             __float_as_uint(b.hi[h].v[j + 1]), w0, w1);
  }
}
__device__ __forceinline__ void mul_act(float (&acc)[4], const ActRow<float>& a, const ActRow<float>& b,
                                        const Vec<float, 4>& w) {
  mul_chunk(acc, a.v, b.v, w);
}
// `terms`: elements between the terms of a value
template <typename T, bool WHOLE>
__device__ __forceinline__ ActRow<T> load_act(const char* row, long long terms, int k, int Fp) {
  ActRow<T> r;
  if constexpr (Elem<T>::kDtype == NSB_BF16) {
    const __nv_bfloat16* at = reinterpret_cast<const __nv_bfloat16*>(row);
#pragma unroll
    for (int i = 0; i < 3; ++i) r.v[i] = load_chunk<__nv_bfloat16, true, false, WHOLE>(at + i * terms, k, Fp);
  } else if constexpr (Elem<T>::kDtype == NSB_F16) {
    const float* at = reinterpret_cast<const float*>(row);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      r.hi[i] = load_chunk<float, true, false, WHOLE>(at, k + 4 * i, Fp);
      r.lo[i] = load_chunk<float, true, false, WHOLE>(at + terms, k + 4 * i, Fp);
    }
  } else {
    r.v = load_chunk<float, true, false, WHOLE>(reinterpret_cast<const float*>(row), k, Fp);
  }
  return r;
}
template <typename T>
constexpr int kActBytes = Elem<T>::kDtype == NSB_BF16 ? 2 : 4;  // of a term
template <typename T>
__device__ __forceinline__ void store_act(void* act, long long slots, int slot, int Fp, int f, float v) {
  const long long at = (long long)slot * Fp + f, terms = slots * Fp;
  if constexpr (Elem<T>::kDtype == NSB_BF16) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const __nv_bfloat16 q = __float2bfloat16_rn(v);
      static_cast<__nv_bfloat16*>(act)[at + i * terms] = q;
      v -= __bfloat162float(q);
      v = isfinite(v) ? v : 0.0f;
    }
  } else if constexpr (Elem<T>::kDtype == NSB_F16) {
    uint32_t hi, lo;
    split_tf32(v, hi, lo);
    static_cast<uint32_t*>(act)[at] = hi;
    static_cast<uint32_t*>(act)[at + terms] = lo;
  } else {
    static_cast<float*>(act)[at] = v;
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

// The products of two tiles of 8 weight rows (lane's rows w0 and w1 of n elements) with up to 16 MT tokens:
// `tokens(whole, m, h, k)` is the lane's chunk at k of its token row h of 16-row tile m, `mul(acc, a, b, w)` the product of
// a chunk. A warp takes every WK-th block of the summation index; only the last, partial one looks where its row
// ends. With one tile of tokens, the usual case, the next block's weights are on their way while this one's are
// multiplied, and the first block's while `prepare` looks up where the tokens lie.
struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };
template <typename T, bool VEC, int MT, int KS, typename Prepare, typename Tokens, typename Mul>
__device__ __forceinline__ void weight_products(float (&acc)[MT * 8], const T* w0, const T* w1, int n, int wk, int WK, int mtiles,
                                                Prepare prepare, Tokens tokens, Mul mul) {
  constexpr int C = 16 / sizeof(T), kBlock = KS * 4 * C;
  const int t = threadIdx.x & 3;
  using Row = decltype(tokens(Yes(), 0, 0, 0));
  struct Block {
    Vec<T, C> w[KS][2];
    Row x[KS][2];
  };
  auto at = [&](int k0, int s) { return k0 + (s * 4 + t) * C; };
  auto load_weights = [&](auto whole, Block& b, int k0) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      b.w[s][0] = load_chunk<T, VEC, true, decltype(whole)::value>(w0, at(k0, s), n);
      b.w[s][1] = load_chunk<T, VEC, true, decltype(whole)::value>(w1, at(k0, s), n);
    }
  };
  auto load_tokens = [&](auto whole, Block& b, int m, int k0) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      b.x[s][0] = tokens(whole, m, 0, at(k0, s));
      b.x[s][1] = tokens(whole, m, 1, at(k0, s));
    }
  };
  auto multiply = [&](Block& b, int m) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float part[2][4] = {};
      mul(part[0], b.x[s][0], b.x[s][1], b.w[s][0]);
      mul(part[1], b.x[s][0], b.x[s][1], b.w[s][1]);
      add_chunk(*reinterpret_cast<float(*)[4]>(&acc[8 * m]), part[0]);
      add_chunk(*reinterpret_cast<float(*)[4]>(&acc[8 * m + 4]), part[1]);
    }
  };
  const int step = WK * kBlock;
  int k0 = wk * kBlock;
  Block a;
  if constexpr (MT == 1) {
    Block b;
    if (k0 + kBlock <= n) load_weights(Yes(), a, k0);
    prepare();
    if (k0 + kBlock <= n) load_tokens(Yes(), a, 0, k0);
    auto next = [&](Block& from, Block& to) {
      if (k0 + step + kBlock <= n) {
        load_weights(Yes(), to, k0 + step);
        load_tokens(Yes(), to, 0, k0 + step);
      }
      multiply(from, 0);
      k0 += step;
    };
    while (k0 + kBlock <= n) {
      next(a, b);
      if (k0 + kBlock > n) break;
      next(b, a);
    }
  } else {
    prepare();
    for (; k0 + kBlock <= n; k0 += step) {
      load_weights(Yes(), a, k0);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m >= mtiles) break;
        load_tokens(Yes(), a, m, k0);
        multiply(a, m);
      }
    }
  }
  if (k0 < n) {
    load_weights(No(), a, k0);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m >= mtiles) break;
      load_tokens(No(), a, m, k0);
      multiply(a, m);
    }
  }
}

// Unit: 8 hidden values of one expert for all its tokens (8 gate rows and 8 up rows of Win).
template <typename T, bool VEC, int MT>
__device__ __forceinline__ void up_unit(const MoeParams& p, int e, int first, int n, int f0, int wk, int WK, float* buf) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // (rows of weights and tokens beyond the last stand for products that are not kept)
  const T* gate_row = static_cast<const T*>(p.w_in) + ((long long)e * 2 * p.F + min(f0 + g, p.F - 1)) * p.D;
  const T* up_row = gate_row + (long long)p.F * p.D;
  const T* rows[MT][2];
  auto prepare = [&] {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        rows[m][h] = static_cast<const T*>(p.x) + (p.slots[first + min(m * 16 + h * 8 + g, n - 1)] / p.K) * p.x_stride;
  };
  float acc[MT * 8];
#pragma unroll
  for (int i = 0; i < MT * 8; ++i) acc[i] = 0.0f;
  weight_products<T, VEC, MT, kUpSteps>(
      acc, gate_row, up_row, p.D, wk, WK, (n + 15) / 16, prepare,
      [&](auto whole, int m, int h, int k) { return load_chunk<T, VEC, false, decltype(whole)::value>(rows[m][h], k, p.D); },
      [](float (&c)[4], const auto& a, const auto& b, const auto& w) { mul_chunk(c, a, b, w); });
  add_up<MT * 8>(acc, buf, wk, WK);
  if (wk != 0) return;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = m * 16 + (i >> 1) * 8 + g, f = f0 + 2 * t + (i & 1);
      if (row < n && f < p.Fp) {
        const int slot = p.slots[first + row];
        const float v = f < p.F ? silu(acc[8 * m + i]) * acc[8 * m + 4 + i] * p.probs[slot] : 0.0f;
        store_act<T>(p.act, p.N * p.K, slot, p.Fp, f, v);
      }
    }
}
template <typename T, bool VEC, int MT>
__global__ void __launch_bounds__(kThreads, 3) moe_up_kernel(const MoeParams p, int WK) {
  __shared__ float buf[MT * 8 * kThreads];
  const int warp = threadIdx.x >> 5, per_cta = kWarps / WK;
  const int per_expert = (p.F + 7) / 8, ctas = (per_expert + per_cta - 1) / per_cta;
  const int place = blockIdx.x / ctas, f0 = ((blockIdx.x % ctas) * per_cta + warp / WK) * 8;
  grid_dependents_may_launch();
  grid_dependency_wait();
  const int used = *p.used, e = p.entries[3 * place], first = p.entries[3 * place + 1], n = p.entries[3 * place + 2];
  if (place >= used) return;  // (there is an entry, of no meaning, for every CTA)
  if constexpr (MT > 1)
    if (n > 16) {
      up_unit<T, VEC, MT>(p, e, first, n, f0, warp % WK, WK, buf);
      return;
    }
  up_unit<T, VEC, 1>(p, e, first, n, f0, warp % WK, WK, buf);
}

// Unit: 16 outputs of one expert for all its tokens. The last unit of an output tile adds up the token's experts.
template <typename T, bool VEC, int MT>
__device__ __forceinline__ void down_unit(const MoeParams& p, int e, int first, int n, int d0, int wk, int WK, float* buf) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const T* w = static_cast<const T*>(p.w_out) + (long long)e * p.D * p.F;
  const char* rows[MT][2];
  const long long terms = (long long)p.N * p.K * p.Fp;
  auto prepare = [&] {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        rows[m][h] = static_cast<const char*>(p.act) +
                     (long long)p.slots[first + min(m * 16 + h * 8 + g, n - 1)] * p.Fp * kActBytes<T>;
  };
  float acc[MT * 8];
#pragma unroll
  for (int i = 0; i < MT * 8; ++i) acc[i] = 0.0f;
  weight_products<T, VEC, MT, kDownSteps>(
      acc, w + (long long)min(d0 + g, p.D - 1) * p.F, w + (long long)min(d0 + 8 + g, p.D - 1) * p.F, p.F, wk, WK, (n + 15) / 16, prepare,
      [&](auto whole, int m, int h, int k) { return load_act<T, decltype(whole)::value>(rows[m][h], terms, k, p.Fp); },
      [](float (&c)[4], const auto& a, const auto& b, const auto& q) { mul_act(c, a, b, q); });
  add_up<MT * 8>(acc, buf, wk, WK);
  if (wk != 0) return;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = m * 16 + ((i >> 1) & 1) * 8 + g, d = d0 + (i >> 2) * 8 + 2 * t + (i & 1);
      if (row < n && d < p.D) p.part[(long long)p.slots[first + row] * p.D + d] = acc[m * 8 + i];
    }
}
template <typename T, bool VEC, int MT>
__global__ void __launch_bounds__(kThreads, kDownCtas<T>) moe_down_kernel(const MoeParams p, int WK) {
  __shared__ float buf[MT * 8 * kThreads];
  __shared__ bool s_last;
  const int warp = threadIdx.x >> 5, per_cta = kWarps / WK;
  const int place = blockIdx.x / p.tiles, tile = blockIdx.x % p.tiles;  // tiles of 16 per_cta outputs
  const int d0 = (tile * per_cta + warp / WK) * 16;
  grid_dependency_wait();
  const int used = *p.used, e = p.entries[3 * place], first = p.entries[3 * place + 1], n = p.entries[3 * place + 2];
  if (place >= used) return;
  bool wide = false;
  if constexpr (MT > 1) wide = n > 16;
  if (wide) down_unit<T, VEC, MT>(p, e, first, n, d0, warp % WK, WK, buf);
  else down_unit<T, VEC, 1>(p, e, first, n, d0, warp % WK, WK, buf);
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(p.done + tile, 1u) + 1u == (unsigned)used;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  const int width = 16 * per_cta, base = tile * width;
  auto add_experts = [&](auto quad) {  // four outputs per thread and turn, or one where rows do not divide by four
    constexpr int Q = decltype(quad)::value ? 4 : 1;
    const int across = width / Q;
#pragma unroll 4
    for (int i = threadIdx.x; i < p.N * across; i += kThreads) {
      const int tok = i / across, d = base + i % across * Q;
      if (d >= p.D) continue;
      const long long at = (long long)tok * p.D + d;
      float sum[Q];
#pragma unroll
      for (int q = 0; q < Q; ++q) sum[q] = p.shared ? Elem<T>::to_f32(static_cast<const T*>(p.shared)[at + q]) : 0.0f;
      const float* part = p.part + (long long)tok * p.K * p.D + d;
#pragma unroll 4
      for (int j = 0; j < p.K; ++j, part += p.D) {
        float v[Q];
        if constexpr (Q == 4) {
          const float4 f = __ldcg(reinterpret_cast<const float4*>(part));
          v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        } else {
          v[0] = __ldcg(part);
        }
#pragma unroll
        for (int q = 0; q < Q; ++q) sum[q] += v[q];
      }
#pragma unroll
      for (int q = 0; q < Q; ++q) static_cast<T*>(p.out)[at + q] = Elem<T>::from_f32(sum[q]);
    }
  };
  if (p.D % 4 == 0) add_experts(Yes()); else add_experts(No());
}

// ------------------------------------------------------------------------------------------ host

bool ok_dtype(int d) { return d == NSB_F32 || d == NSB_BF16 || d == NSB_F16; }
bool fits(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
long long up16(long long n) { return (n + 15) / 16 * 16; }

struct Layout {  // of the workspace, in bytes
  long long logits, lparts, used, entries, slots, done, act, part, bytes;
};
Layout layout(long long N, long long E, long long K, long long D, long long F) {
  const long long S = N * K, Fp = (F + 7) / 8 * 8;
  Layout l;
  l.logits = 0;
  l.lparts = up16(N * E * 4);
  l.used = l.lparts + up16(N * E * 4 * kRouterCtas);
  l.entries = l.used + 16;
  l.slots = l.entries + up16(12 * std::min(E, S));
  l.done = l.slots + up16(4 * S);
  l.act = l.done + up16(4 * ((D + 15) / 16));
  l.part = l.act + 8 * S * Fp;  // (fp16's; the others take less)
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
  p.lparts = reinterpret_cast<float*>(base + l.lparts);
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
