// Gated linear recurrence (the PLIF membrane without its spike, gate from a raw projection):
//
//   f_t = sigmoid(raw_t + bias)      h_t = f_t h_{t-1} + (1 - f_t) x_t      y_t = h_t
//
// and its reverse-time gradient. With K_{t+1} = f_{t+1} G_{t+1} what step t + 1 hands back to step t:
//
//   G_t = dy_t + K_{t+1}     dx_t = (1 - f_t) G_t     draw_t = G_t (h_{t-1} - x_t) f_t (1 - f_t)
//
// Each step is an affine map of the state, h -> P h + H, and such maps compose associatively, so time is
// cut into chunks that are worked on side by side. A CTA takes one chunk of one block of columns: every
// warp holds S steps of 32 V columns in registers, finds their composed map, the CTA's warps exchange
// their maps through shared memory, CTAs exchange theirs through global memory (below), and every warp then
// runs its steps once more from its true starting state. Each input is read once and each output written
// once; the only other traffic is 4-12 bytes per chunk and column.
//
// Hand-over between the chunks of a column block. Chunks come in groups of g: a chunk publishes its map
// (P, H), the last chunk of a group publishes the state after it instead. A chunk's starting state is the
// state after the group before, taken through the maps of the chunks of its own group that precede it, always
// in the same order: results do not depend on timing. A published word is its own flag: the scratch is
// filled with 0xff bytes, which no published value has (see publishable), and 8-byte words are written
// whole. Work is handed out by a ticket counter in order of time, so whatever a CTA waits for belongs to a
// CTA that is running or has finished; every wait is bounded all the same and hands on NaN if it gives up.
#include <algorithm>

#include "nsb_common.cuh"

namespace nsb {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr uint32_t kEmpty = 0xffffffffu;
constexpr uint32_t kErrGated = 0x00400000u;

struct GatedParams {
  const void *raw, *x, *dy;
  const float *bias, *h0, *dh_last;
  const int* cu;                    // packed sequences: their first rows, and the end of the last
  void *y, *d_raw, *d_x;
  float *h_last, *ckpt, *d_h0, *d_bias_part;
  long long raw_st, raw_sb, x_st, x_sb;  // strides in elements between rows and between blocks of Dw columns
  long long T, cols, Dw, D;         // D: period of the bias
  long long nb;                     // column blocks
  int nchunks, g, wt, S_seqs;
  uint32_t* ticket;
  uint2* maps;                      // [nchunks][cols] (P, H)
  uint32_t* states;                 // [nchunks / g][cols]
  uint32_t* err;
  unsigned long long limit_ns;
};

// sigmoid(a) and sigmoid(-a), both to a few units in the last place of fp32 over the whole range: the
// exponential is taken of -|a|, so it neither overflows nor is subtracted from one.
__device__ __forceinline__ void gate(float a, float& f, float& m) {
  const float t = __expf(-fabsf(a));
  const float big = __fdividef(1.0f, 1.0f + t), small = t * big;
  f = a >= 0.0f ? big : small;
  m = a >= 0.0f ? small : big;
}

// The pair in one register: the smaller of f and 1 - f, negative where that is f. The other is one minus it,
// which costs neither any digits.
__device__ __forceinline__ float gate_packed(float a) {
  const float t = __expf(-fabsf(a));
  return copysignf(t * __fdividef(1.0f, 1.0f + t), a);
}
__device__ __forceinline__ void gate_unpack(float g, float& f, float& m) {
  const float small = fabsf(g), big = 1.0f - small;
  const bool shut = __float_as_int(g) < 0;
  f = shut ? small : big;
  m = shut ? big : small;
}

__device__ __forceinline__ uint32_t publishable(float v) {
  const uint32_t b = __float_as_uint(v);
  return b == kEmpty ? 0x7fffffffu : b;
}
__device__ __forceinline__ uint32_t peek32(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 peek64(const uint2* p) {
  unsigned long long v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return make_uint2((uint32_t)v, (uint32_t)(v >> 32));
}
__device__ __forceinline__ void post32(uint32_t* p, uint32_t v) {
  asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
__device__ __forceinline__ void post64(uint2* p, uint32_t a, uint32_t b) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"((unsigned long long)a | ((unsigned long long)b << 32))
               : "memory");
}

// Bounded wait for a published word; NaN if it gives up (and the error word says so).
template <typename Peek, typename Full>
__device__ __forceinline__ auto await_word(Peek peek, Full full, const GatedParams& p) {
  auto v = peek();
  if (full(v)) return v;
  const uint64_t t0 = global_timer_ns();
  uint32_t it = 0;
  while (!full(v = peek())) {
    if ((++it & 0x3F) == 0 && (global_timer_ns() - t0 > p.limit_ns || it > (1u << 28))) {
      if (p.err) atomicOr(reinterpret_cast<unsigned int*>(p.err), kErrGated);
      break;
    }
  }
  return v;
}
__device__ __forceinline__ float await_state(const uint32_t* w, const GatedParams& p) {
  const uint32_t v = await_word([&] { return peek32(w); }, [](uint32_t b) { return b != kEmpty; }, p);
  return __uint_as_float(v == kEmpty ? 0x7fffffffu : v);
}
__device__ __forceinline__ float2 await_map(const uint2* w, const GatedParams& p) {
  uint2 v = await_word([&] { return peek64(w); }, [](uint2 b) { return b.x != kEmpty; }, p);
  if (v.x == kEmpty) v = make_uint2(0x7fffffffu, 0x7fffffffu);
  return make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
}

// What the S rows of a warp are: bit s of `in` - row s belongs to a sequence; `first`, `last` - it is that
// sequence's first or last row. Lane s keeps the number of row s's sequence.
struct Rows {
  uint32_t in, first, last;
  int seq;
};
template <int S, bool PACKED>
__device__ __forceinline__ Rows row_kinds(const GatedParams& p, long long t0, int lane) {
  Rows r;
  const long long t = t0 + lane;
  bool in = lane < S && t < p.T, first = false, last = false;
  r.seq = 0;
  if constexpr (PACKED) {
    if (in) {
      int lo = 0, hi = p.S_seqs;  // sequences that end at or before row t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(p.cu + mid + 1) <= t) lo = mid + 1; else hi = mid;
      }
      in = lo < p.S_seqs && __ldg(p.cu + lo) <= t;
      if (in) {
        r.seq = lo;
        first = __ldg(p.cu + lo) == t;
        last = __ldg(p.cu + lo + 1) == t + 1;
      }
    }
  } else {
    first = in && t == 0;
    last = in && t == p.T - 1;
  }
  r.in = __ballot_sync(0xffffffffu, in);
  r.first = __ballot_sync(0xffffffffu, first);
  r.last = __ballot_sync(0xffffffffu, last);
  return r;
}

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
  return *reinterpret_cast<const Vec<T, V>*>(p);
}

// The map h -> P h + H of one step or of several. Where a sequence begins, the state from before must not come
// in, not even as 0 * NaN: such a map has P = -0 (a product of gates is never negative) and gives H.
template <int V>
struct MapV {
  float P[V], H[V];
};
constexpr float kCut = -0.0f;
__device__ __forceinline__ bool is_cut(float P) { return __float_as_uint(P) == 0x80000000u; }
__device__ __forceinline__ float apply_map(float P, float H, float h) { return is_cut(P) ? H : fmaf(P, h, H); }
// (P, H) followed by (P2, H2)
__device__ __forceinline__ void then_map(float& P, float& H, float P2, float H2) {
  H = apply_map(P2, H2, H);
  P = is_cut(P2) || is_cut(P) ? kCut : P * P2;
}

// The state (or, in reverse, the hand-back) that a chunk starts from. `pos` counts chunks in the order in
// which they are worked on. Every time warp takes the maps of some of the preceding chunks of the group and
// composes them in order; the parts meet in shared memory. Returns the same value in every time warp.
template <int V>
__device__ __forceinline__ void chunk_start(const GatedParams& p, int pos, long long col, bool on, int wt_idx, int wt,
                                            MapV<V>* part, int lane_slot, float (&start)[V]) {
  const int group = pos / p.g, j = pos - group * p.g;
  const int per = (j + wt - 1) / wt;
  MapV<V> m;
#pragma unroll
  for (int v = 0; v < V; ++v) m.P[v] = 1.0f, m.H[v] = 0.0f;
  if (on) {
    const int a = wt_idx * per, b = min(j, a + per);
    const uint2* w = p.maps + (long long)(group * p.g + a) * p.cols + col;
    for (int i = a; i < b; ++i, w += p.cols)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float2 q = await_map(w + v, p);
        then_map(m.P[v], m.H[v], q.x, q.y);
      }
    if (wt_idx == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float s = group ? await_state(p.states + (long long)(group - 1) * p.cols + col + v, p) : 0.0f;
        m.H[v] = apply_map(m.P[v], m.H[v], s);
      }
    }
  }
  part[lane_slot] = m;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) start[v] = 0.0f;
  const int stride = 32;
  for (int i = 0; i < wt; ++i) {
    const MapV<V> q = part[(lane_slot % stride) + i * stride + (lane_slot / (wt * stride)) * (wt * stride)];
#pragma unroll
    for (int v = 0; v < V; ++v) start[v] = i == 0 ? q.H[v] : apply_map(q.P[v], q.H[v], start[v]);
  }
}

template <typename T, int V, int S, bool PACKED, bool CHAIN>
__global__ void __launch_bounds__(kThreads) gated_fwd_kernel(const GatedParams p) {
  __shared__ MapV<V> maps[kThreads], part[CHAIN ? kThreads : 1];
  __shared__ uint32_t s_ticket;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wt = p.wt, wt_idx = warp % wt, wc_idx = warp / wt, wc = kWarps / wt;
  long long work = blockIdx.x;
  if constexpr (CHAIN) {
    if (threadIdx.x == 0) s_ticket = atomicAdd(p.ticket, 1u) + 1u;  // (the counter starts at 0xffffffff)
    __syncthreads();
    work = s_ticket;
  }
  const int chunk = (int)(work / p.nb);
  const long long col = ((work % p.nb) * wc + wc_idx) * (32 * V) + (long long)lane * V;
  const bool on = col < p.cols;
  const long long t0 = ((long long)chunk * wt + wt_idx) * S;
  const T* raw = static_cast<const T*>(p.raw);
  const T* x = static_cast<const T*>(p.x);

  Vec<T, V> vr[S], vx[S];
  if (on) {
    const long long b = col / p.Dw, d = col - b * p.Dw;
    raw += t0 * p.raw_st + b * p.raw_sb + d;
    x += t0 * p.x_st + b * p.x_sb + d;
  }
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (on && t0 + s < p.T) {
      vr[s] = load_vec<T, V>(raw + s * p.raw_st);
      vx[s] = load_vec<T, V>(x + s * p.x_st);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) vr[s].v[v] = vx[s].v[v] = Elem<T>::zero();
    }
  }
  float bias[V];
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = (p.bias && on) ? p.bias[(col + v) % p.D] : 0.0f;
  const Rows rows = row_kinds<S, PACKED>(p, t0, lane);
  auto h0_at = [&](int s, float (&h)[V]) {
    const int q = PACKED ? __shfl_sync(0xffffffffu, rows.seq, s) : 0;
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = (p.h0 && on) ? p.h0[(long long)q * p.cols + col + v] : 0.0f;
  };

  float f[S][V], u[S][V];
  MapV<V> mine;
#pragma unroll
  for (int v = 0; v < V; ++v) mine.P[v] = 1.0f, mine.H[v] = 0.0f;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if ((rows.first >> s) & 1u) {
      h0_at(s, mine.H);
#pragma unroll
      for (int v = 0; v < V; ++v) mine.P[v] = kCut;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float m;
      gate(Elem<T>::to_f32(vr[s].v[v]) + bias[v], f[s][v], m);
      u[s][v] = m * Elem<T>::to_f32(vx[s].v[v]);
      mine.P[v] *= f[s][v];
      mine.H[v] = fmaf(f[s][v], mine.H[v], u[s][v]);
    }
  }
  maps[threadIdx.x] = mine;
  __syncthreads();

  // the warps of this column group: maps[(wc_idx * wt + i) * 32 + lane], i = 0 .. wt - 1 in time order
  const int first_slot = wc_idx * wt * 32 + lane;
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = 0.0f;
  if constexpr (CHAIN) {
    const bool group_end = chunk % p.g == p.g - 1;
    const bool more = chunk + 1 < p.nchunks;
    MapV<V> all;
    if (wt_idx == wt - 1 && more) {
      all = maps[first_slot];
      for (int i = 1; i < wt; ++i) {
        const MapV<V> q = maps[first_slot + i * 32];
#pragma unroll
        for (int v = 0; v < V; ++v) then_map(all.P[v], all.H[v], q.P[v], q.H[v]);
      }
      if (!group_end && on)
#pragma unroll
        for (int v = 0; v < V; ++v)
          post64(p.maps + (long long)chunk * p.cols + col + v, publishable(all.P[v]), publishable(all.H[v]));
    }
    chunk_start<V>(p, chunk, col, on, wt_idx, wt, part, threadIdx.x, h);
    if (wt_idx == wt - 1 && more && group_end && on)
#pragma unroll
      for (int v = 0; v < V; ++v)
        post32(p.states + (long long)(chunk / p.g) * p.cols + col + v, publishable(apply_map(all.P[v], all.H[v], h[v])));
    if (p.ckpt && wt_idx == 0 && on)
#pragma unroll
      for (int v = 0; v < V; ++v) p.ckpt[(long long)chunk * p.cols + col + v] = h[v];
  }
  for (int i = 0; i < wt_idx; ++i) {
    const MapV<V> q = maps[first_slot + i * 32];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = apply_map(q.P[v], q.H[v], h[v]);
  }
  T* y = static_cast<T*>(p.y) + t0 * p.cols + col;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if ((rows.first >> s) & 1u) h0_at(s, h);
    Vec<T, V> o;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      h[v] = fmaf(f[s][v], h[v], u[s][v]);
      o.v[v] = ((rows.in >> s) & 1u) ? Elem<T>::from_f32(h[v]) : Elem<T>::zero();
    }
    if (on && t0 + s < p.T) *reinterpret_cast<Vec<T, V>*>(y + s * p.cols) = o;
    if ((rows.last >> s) & 1u) {
      const int q = PACKED ? __shfl_sync(0xffffffffu, rows.seq, s) : 0;
      if (on)
#pragma unroll
        for (int v = 0; v < V; ++v) p.h_last[(long long)q * p.cols + col + v] = h[v];
    }
  }
  if constexpr (PACKED) {  // an empty sequence ends in the state that it starts from
    if (chunk == 0 && on)
      for (int q = wt_idx; q < p.S_seqs; q += wt)
        if (p.cu[q + 1] <= p.cu[q])
#pragma unroll
          for (int v = 0; v < V; ++v)
            p.h_last[(long long)q * p.cols + col + v] = p.h0 ? p.h0[(long long)q * p.cols + col + v] : 0.0f;
  }
}

// Reverse pass of a chunk. Both directions need only the products of f and a partial sum each, so one exchange
// carries them: (P, H) takes a state forward through a warp's steps (the forward's states are computed again
// from the chunk's saved starting state), (P, K) takes the hand-back through them in reverse.
template <int V>
struct TripleV {
  float P[V], H[V], K[V];
};

template <typename T, int V, int S, bool PACKED, bool CHAIN>
__global__ void __launch_bounds__(kThreads) gated_bwd_kernel(const GatedParams p) {
  __shared__ TripleV<V> trip[kThreads];
  __shared__ MapV<V> part[CHAIN ? kThreads : 1];
  __shared__ uint32_t s_ticket;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wt = p.wt, wt_idx = warp % wt, wc_idx = warp / wt, wc = kWarps / wt;
  long long work = blockIdx.x;
  if constexpr (CHAIN) {
    if (threadIdx.x == 0) s_ticket = atomicAdd(p.ticket, 1u) + 1u;
    __syncthreads();
    work = s_ticket;
  }
  const int pos = (int)(work / p.nb), chunk = p.nchunks - 1 - pos;
  const long long col = ((work % p.nb) * wc + wc_idx) * (32 * V) + (long long)lane * V;
  const bool on = col < p.cols;
  const long long t0 = ((long long)chunk * wt + wt_idx) * S;
  const T* raw = static_cast<const T*>(p.raw);
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);

  Vec<T, V> vr[S], vx[S], vg[S];
  if (on) {
    const long long b = col / p.Dw, d = col - b * p.Dw;
    raw += t0 * p.raw_st + b * p.raw_sb + d;
    x += t0 * p.x_st + b * p.x_sb + d;
    dy += t0 * p.cols + col;
  }
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (on && t0 + s < p.T) {
      vr[s] = load_vec<T, V>(raw + s * p.raw_st);
      vx[s] = load_vec<T, V>(x + s * p.x_st);
      vg[s] = load_vec<T, V>(dy + s * p.cols);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) vr[s].v[v] = vx[s].v[v] = vg[s].v[v] = Elem<T>::zero();
    }
  }
  float bias[V], h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    bias[v] = (p.bias && on) ? p.bias[(col + v) % p.D] : 0.0f;
    h[v] = (CHAIN && on) ? p.ckpt[(long long)chunk * p.cols + col + v] : 0.0f;
  }
  const Rows rows = row_kinds<S, PACKED>(p, t0, lane);
  auto state_at = [&](const float* from, int s, float (&o)[V]) {
    const int q = PACKED ? __shfl_sync(0xffffffffu, rows.seq, s) : 0;
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = (from && on) ? from[(long long)q * p.cols + col + v] : 0.0f;
  };

  float gt[S][V];
  TripleV<V> mine;
#pragma unroll
  for (int v = 0; v < V; ++v) mine.P[v] = 1.0f, mine.H[v] = 0.0f, mine.K[v] = 0.0f;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if ((rows.first >> s) & 1u) state_at(p.h0, s, mine.H);
    // a state does not pass a sequence's border in either direction: one product serves both
    const bool cut = ((rows.first | rows.last | ~rows.in) >> s) & 1u;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float f, m;
      gt[s][v] = gate_packed(Elem<T>::to_f32(vr[s].v[v]) + bias[v]);
      gate_unpack(gt[s][v], f, m);
      mine.H[v] = fmaf(f, mine.H[v], m * Elem<T>::to_f32(vx[s].v[v]));
      mine.P[v] = cut ? kCut : mine.P[v] * f;
    }
  }
#pragma unroll
  for (int s = S - 1; s >= 0; --s) {
    if ((rows.last >> s) & 1u) state_at(p.dh_last, s, mine.K);
    const bool in = (rows.in >> s) & 1u;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float f, m;
      gate_unpack(gt[s][v], f, m);
      mine.K[v] = in ? f * (mine.K[v] + Elem<T>::to_f32(vg[s].v[v])) : 0.0f;
    }
  }
  trip[threadIdx.x] = mine;
  __syncthreads();

  const int first_slot = wc_idx * wt * 32 + lane;
  float K[V];
#pragma unroll
  for (int v = 0; v < V; ++v) K[v] = 0.0f;
  if constexpr (CHAIN) {
    const bool group_end = pos % p.g == p.g - 1;
    const bool more = chunk > 0;
    MapV<V> all;
    if (wt_idx == 0 && more) {
      const TripleV<V> l = trip[first_slot + (wt - 1) * 32];
#pragma unroll
      for (int v = 0; v < V; ++v) all.P[v] = l.P[v], all.H[v] = l.K[v];
      for (int i = wt - 2; i >= 0; --i) {
        const TripleV<V> q = trip[first_slot + i * 32];
#pragma unroll
        for (int v = 0; v < V; ++v) then_map(all.P[v], all.H[v], q.P[v], q.K[v]);
      }
      if (!group_end && on)
#pragma unroll
        for (int v = 0; v < V; ++v)
          post64(p.maps + (long long)pos * p.cols + col + v, publishable(all.P[v]), publishable(all.H[v]));
    }
    chunk_start<V>(p, pos, col, on, wt_idx, wt, part, threadIdx.x, K);
    if (wt_idx == 0 && more && group_end && on)
#pragma unroll
      for (int v = 0; v < V; ++v)
        post32(p.states + (long long)(pos / p.g) * p.cols + col + v, publishable(apply_map(all.P[v], all.H[v], K[v])));
  }
  for (int i = 0; i < wt_idx; ++i) {
    const TripleV<V> q = trip[first_slot + i * 32];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = apply_map(q.P[v], q.H[v], h[v]);
  }
  for (int i = wt - 1; i > wt_idx; --i) {
    const TripleV<V> q = trip[first_slot + i * 32];
#pragma unroll
    for (int v = 0; v < V; ++v) K[v] = apply_map(q.P[v], q.K[v], K[v]);
  }

  float d[S][V];  // h_{t-1} - x_t
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if ((rows.first >> s) & 1u) state_at(p.h0, s, h);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float xv = Elem<T>::to_f32(vx[s].v[v]);
      float f, m;
      gate_unpack(gt[s][v], f, m);
      d[s][v] = h[v] - xv;
      h[v] = fmaf(f, h[v], m * xv);
    }
  }
  float db[V];
#pragma unroll
  for (int v = 0; v < V; ++v) db[v] = 0.0f;
  T* o_raw = static_cast<T*>(p.d_raw) + t0 * p.cols + col;
  T* o_x = static_cast<T*>(p.d_x) + t0 * p.cols + col;
#pragma unroll
  for (int s = S - 1; s >= 0; --s) {
    if ((rows.last >> s) & 1u) state_at(p.dh_last, s, K);
    const bool in = (rows.in >> s) & 1u;
    Vec<T, V> a, c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float G = K[v] + Elem<T>::to_f32(vg[s].v[v]);
      float f, m;
      gate_unpack(gt[s][v], f, m);
      K[v] = f * G;
      const float g_x = in ? m * G : 0.0f, g_a = in ? K[v] * m * d[s][v] : 0.0f;
      db[v] += g_a;
      a.v[v] = Elem<T>::from_f32(g_a);
      c.v[v] = Elem<T>::from_f32(g_x);
    }
    if (on && t0 + s < p.T) {
      if (p.d_raw) *reinterpret_cast<Vec<T, V>*>(o_raw + s * p.cols) = a;
      if (p.d_x) *reinterpret_cast<Vec<T, V>*>(o_x + s * p.cols) = c;
    }
    if (((rows.first >> s) & 1u) && p.d_h0) {
      const int q = PACKED ? __shfl_sync(0xffffffffu, rows.seq, s) : 0;
      if (on)
#pragma unroll
        for (int v = 0; v < V; ++v) p.d_h0[(long long)q * p.cols + col + v] = K[v];
    }
  }
  if (p.d_bias_part) {  // this chunk's sum over time, in the order of the warps
    __syncthreads();
    float* acc = reinterpret_cast<float*>(trip);
#pragma unroll
    for (int v = 0; v < V; ++v) acc[threadIdx.x * V + v] = db[v];
    __syncthreads();
    if (wt_idx == 0 && on)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float sum = 0.0f;
        for (int i = 0; i < wt; ++i) sum += acc[(first_slot + i * 32) * V + v];
        p.d_bias_part[(long long)chunk * p.cols + col + v] = sum;
      }
  }
  if constexpr (PACKED) {
    if (chunk == 0 && on && p.d_h0)
      for (int q = wt_idx; q < p.S_seqs; q += wt)
        if (p.cu[q + 1] <= p.cu[q])
#pragma unroll
          for (int v = 0; v < V; ++v)
            p.d_h0[(long long)q * p.cols + col + v] = p.dh_last ? p.dh_last[(long long)q * p.cols + col + v] : 0.0f;
  }
}

// d_bias[d] = sum over rows of part[row][d], in 64 bits, in a fixed order: thread (i, j) of a CTA takes rows
// i, i + 32, ... of column j, and the 32 sums of a column are added one after the other.
__global__ void __launch_bounds__(1024) gated_bias_kernel(const float* __restrict__ part, float* __restrict__ out,
                                                          long long rows, long long D) {
  __shared__ double acc[32][33];
  grid_dependency_wait();
  const int j = threadIdx.x & 31, i = threadIdx.x >> 5;
  const long long d = (long long)blockIdx.x * 32 + j;
  double sum = 0.0;
  if (d < D) {
#pragma unroll 4
    for (long long r = i; r < rows; r += 32) sum += (double)part[r * D + d];
  }
  acc[i][j] = sum;
  __syncthreads();
  if (i == 0 && d < D) {
    for (int k = 1; k < 32; ++k) sum += acc[k][j];
    out[d] = (float)sum;
  }
}

// One step of every row, the state in place.
template <typename T, int V>
__global__ void __launch_bounds__(256) gated_step_kernel(const T* __restrict__ raw, const T* __restrict__ x,
                                                         const float* __restrict__ bias, float* __restrict__ h,
                                                         T* __restrict__ y, long long B, long long D,
                                                         long long raw_sb, long long x_sb) {
  const long long dv = D / V, n = B * dv;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
    const long long b = i / dv, d = (i - b * dv) * V;
    const Vec<T, V> vr = load_vec<T, V>(raw + b * raw_sb + d), vx = load_vec<T, V>(x + b * x_sb + d);
    Vec<float, V> vh = load_vec<float, V>(h + b * D + d);
    Vec<T, V> o;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float f, m;
      gate(Elem<T>::to_f32(vr.v[v]) + (bias ? bias[d + v] : 0.0f), f, m);
      vh.v[v] = fmaf(f, vh.v[v], m * Elem<T>::to_f32(vx.v[v]));
      o.v[v] = Elem<T>::from_f32(vh.v[v]);
    }
    *reinterpret_cast<Vec<float, V>*>(h + b * D + d) = vh;
    *reinterpret_cast<Vec<T, V>*>(y + b * D + d) = o;
  }
}

// ------------------------------------------------------------------------------------------------ host

constexpr int kSteps = 8;  // steps of a warp's tile

struct GatedPlan {
  int wt, nchunks, g;
  long long nb;
};

// Warps of a CTA along time: as many as the steps need, up to all of them; the rest lie side by side over
// the columns. Chunks hand on states one by one (g = 1) where a row of column blocks fills the GPU, so that
// a chunk's predecessor has finished long before; with fewer blocks, 32 chunks run side by side and pass maps.
GatedPlan plan_gated(long long T, long long cols, int V, int sms) {
  GatedPlan q;
  q.wt = 1;
  while (q.wt < kWarps && (long long)q.wt * kSteps < T) q.wt *= 2;
  const long long rows = (long long)q.wt * kSteps, width = 32LL * V * (kWarps / q.wt);
  q.nchunks = (int)((T + rows - 1) / rows);
  q.nb = (cols + width - 1) / width;
  q.g = q.nb >= 3LL * sms ? 1 : 32;
  return q;
}
int chunk_rows(long long T) {
  const GatedPlan q = plan_gated(T, 1, 1, 148);
  return q.wt * kSteps;
}

bool ok_dtype(int d) { return d == NSB_F32 || d == NSB_BF16 || d == NSB_F16; }
bool fits(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// scratch: [ticket, 3 words of padding][states][maps], filled with 0xff by one memset
long long scratch_words(long long T, long long cols) {
  const long long chunks = (T + chunk_rows(T) - 1) / chunk_rows(T);
  if (chunks <= 1) return 0;
  // whatever g the plan takes: all chunks' maps, or all chunks' states
  return 4 + ((chunks / 32 + 1) * cols + 3) / 4 * 4 + 2 * chunks * cols;
}

template <typename T>
int launch_gated(GatedParams p, bool backward, uint32_t* scratch, cudaStream_t st) {
  DeviceInfo dev;
  int r = get_device_info(&dev);
  if (r != NSB_OK) return r;
  int V = 2;
  auto all_fit = [&](int v) {
    const size_t a = sizeof(T) * v;
    bool ok = p.Dw % v == 0 && p.raw_st % v == 0 && p.raw_sb % v == 0 && p.x_st % v == 0 && p.x_sb % v == 0 &&
              p.cols % v == 0;
    for (const void* q : {p.raw, p.x, p.dy, (const void*)p.y, (const void*)p.d_raw, (const void*)p.d_x})
      ok = ok && fits(q, a);
    return ok;
  };
  while (V > 1 && !all_fit(V)) V /= 2;
  const GatedPlan q = plan_gated(p.T, p.cols, V, dev.sm_count);
  p.nb = q.nb, p.nchunks = q.nchunks, p.g = q.g, p.wt = q.wt;
  const bool chain = q.nchunks > 1, packed = p.cu != nullptr;
  if (chain) {
    if (!scratch || !fits(scratch, 16)) return NSB_ERR_INVALID_ARG;
    const long long nstates = (q.nchunks / q.g + 1) * p.cols;
    const long long nmaps = q.g > 1 ? 2LL * q.nchunks * p.cols : 0;
    p.ticket = scratch;
    p.states = scratch + 4;
    p.maps = reinterpret_cast<uint2*>(scratch + 4 + (nstates + 3) / 4 * 4);
    NSB_CUDA_TRY(cudaMemsetAsync(scratch, 0xff, 4 * (4 + (nstates + 3) / 4 * 4 + nmaps), st), "memset gated scratch");
  }
  const long long grid = q.nb * q.nchunks;
  if (grid > 0x7fffffffLL) return NSB_ERR_TOO_LARGE;
#define NSB_GO(V_, P_, C_)                                                                          \
  (backward ? gated_bwd_kernel<T, V_, kSteps, P_, C_><<<(unsigned)grid, kThreads, 0, st>>>(p)       \
            : gated_fwd_kernel<T, V_, kSteps, P_, C_><<<(unsigned)grid, kThreads, 0, st>>>(p))
#define NSB_GO_V(V_) \
  (packed ? (chain ? NSB_GO(V_, true, true) : NSB_GO(V_, true, false)) \
          : (chain ? NSB_GO(V_, false, true) : NSB_GO(V_, false, false)))
  if (V == 2) NSB_GO_V(2); else NSB_GO_V(1);
#undef NSB_GO_V
#undef NSB_GO
  NSB_CUDA_TRY(cudaGetLastError(), backward ? "launch gated_bwd_kernel" : "launch gated_fwd_kernel");
  return NSB_OK;
}

int check_sizes(int64_t T, int64_t B, int64_t D, int64_t seqs, const int32_t* cu, int dtype) {
  if (T < 0 || B < 0 || D < 0 || seqs < 0 || !ok_dtype(dtype)) return NSB_ERR_INVALID_ARG;
  if (cu ? (B != 1 || !fits(cu, 4)) : seqs != 0) return NSB_ERR_INVALID_ARG;
  if (T > 0x7fffffffLL || seqs > 0x7ffffffeLL) return NSB_ERR_TOO_LARGE;
  return NSB_OK;
}

}  // namespace
}  // namespace nsb

using namespace nsb;

extern "C" int64_t nsb_gated_scratch_words(int64_t T, int64_t cols) {
  return T <= 0 || cols <= 0 ? 0 : scratch_words(T, cols);
}
extern "C" int64_t nsb_gated_chunks(int64_t T) { return T <= 0 ? 0 : (T + chunk_rows(T) - 1) / chunk_rows(T); }

extern "C" int nsb_gated_recurrence_fwd(const void* raw, int64_t raw_stride_t, int64_t raw_stride_b, const void* x,
                                        int64_t x_stride_t, int64_t x_stride_b, const float* bias, const float* h0,
                                        const int32_t* cu_seqlens, int64_t seqs, void* y, float* h_last, float* ckpt,
                                        uint32_t* scratch, int64_t T, int64_t B, int64_t D, int dtype, void* stream) {
  int r = check_sizes(T, B, D, seqs, cu_seqlens, dtype);
  if (r != NSB_OK) return r;
  const int64_t cols = B * D;
  if (cols == 0 || (T == 0 && cu_seqlens && seqs == 0)) return NSB_OK;
  if ((!h_last && !(cu_seqlens && seqs == 0)) || !fits(h_last, 4) || !fits(h0, 4) || !fits(bias, 4) || !fits(ckpt, 4)) return NSB_ERR_INVALID_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {  // every sequence is empty
    const size_t n = (size_t)(cu_seqlens ? seqs : 1) * cols * sizeof(float);
    if (h0) NSB_CUDA_TRY(cudaMemcpyAsync(h_last, h0, n, cudaMemcpyDeviceToDevice, st), "copy h0");
    else NSB_CUDA_TRY(cudaMemsetAsync(h_last, 0, n, st), "memset h_last");
    return NSB_OK;
  }
  const size_t es = dtype_size(dtype);
  if (!raw || !x || !y || !fits(raw, es) || !fits(x, es) || !fits(y, es)) return NSB_ERR_INVALID_ARG;
  if ((r = sticky_device_error()) != NSB_OK) return r;
  GatedParams p = {};
  p.raw = raw, p.x = x, p.bias = bias, p.h0 = h0, p.cu = cu_seqlens, p.S_seqs = (int)seqs;
  p.y = y, p.h_last = h_last, p.ckpt = ckpt;
  p.raw_st = raw_stride_t, p.raw_sb = raw_stride_b, p.x_st = x_stride_t, p.x_sb = x_stride_b;
  p.T = T, p.cols = cols, p.D = D;
  p.Dw = (raw_stride_b == D && x_stride_b == D) || B == 1 ? cols : D;
  if (!(p.err = device_error_word_ptr())) return NSB_ERR_CUDA;
  p.limit_ns = get_wait_limit_ns();
  switch (dtype) {
    case NSB_F32: return launch_gated<float>(p, false, scratch, st);
    case NSB_BF16: return launch_gated<__nv_bfloat16>(p, false, scratch, st);
    default: return launch_gated<__half>(p, false, scratch, st);
  }
}

extern "C" int nsb_gated_recurrence_bwd(const void* raw, int64_t raw_stride_t, int64_t raw_stride_b, const void* x,
                                        int64_t x_stride_t, int64_t x_stride_b, const float* bias, const float* h0,
                                        const int32_t* cu_seqlens, int64_t seqs, const float* ckpt, const void* dy,
                                        const float* dh_last, void* d_raw, void* d_x, float* d_bias, float* d_h0,
                                        float* bias_part, uint32_t* scratch, int64_t T, int64_t B, int64_t D,
                                        int dtype, void* stream) {
  int r = check_sizes(T, B, D, seqs, cu_seqlens, dtype);
  if (r != NSB_OK) return r;
  const int64_t cols = B * D;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (const void* q : {(const void*)bias, (const void*)h0, (const void*)ckpt, (const void*)dh_last,
                        (const void*)d_bias, (const void*)d_h0, (const void*)bias_part})
    if (!fits(q, 4)) return NSB_ERR_INVALID_ARG;
  if (cols == 0 || T == 0) {
    if (d_bias && D > 0) NSB_CUDA_TRY(cudaMemsetAsync(d_bias, 0, (size_t)D * sizeof(float), st), "memset d_bias");
    const size_t n = (size_t)(cu_seqlens ? seqs : 1) * cols * sizeof(float);
    if (d_h0 && n) {
      if (dh_last) NSB_CUDA_TRY(cudaMemcpyAsync(d_h0, dh_last, n, cudaMemcpyDeviceToDevice, st), "copy dh_last");
      else NSB_CUDA_TRY(cudaMemsetAsync(d_h0, 0, n, st), "memset d_h0");
    }
    return NSB_OK;
  }
  const size_t es = dtype_size(dtype);
  if (!raw || !x || !dy) return NSB_ERR_INVALID_ARG;
  for (const void* q : {raw, x, dy, (const void*)d_raw, (const void*)d_x})
    if (!fits(q, es)) return NSB_ERR_INVALID_ARG;
  if ((d_bias && !bias_part) || (nsb_gated_chunks(T) > 1 && !ckpt)) return NSB_ERR_INVALID_ARG;
  if ((r = sticky_device_error()) != NSB_OK) return r;
  GatedParams p = {};
  p.raw = raw, p.x = x, p.dy = dy, p.bias = bias, p.h0 = h0, p.dh_last = dh_last, p.cu = cu_seqlens;
  p.S_seqs = (int)seqs, p.d_raw = d_raw, p.d_x = d_x, p.d_h0 = d_h0;
  p.ckpt = const_cast<float*>(ckpt), p.d_bias_part = d_bias ? bias_part : nullptr;
  p.raw_st = raw_stride_t, p.raw_sb = raw_stride_b, p.x_st = x_stride_t, p.x_sb = x_stride_b;
  p.T = T, p.cols = cols, p.D = D;
  p.Dw = (raw_stride_b == D && x_stride_b == D) || B == 1 ? cols : D;
  if (!(p.err = device_error_word_ptr())) return NSB_ERR_CUDA;
  p.limit_ns = get_wait_limit_ns();
  switch (dtype) {
    case NSB_F32: r = launch_gated<float>(p, true, scratch, st); break;
    case NSB_BF16: r = launch_gated<__nv_bfloat16>(p, true, scratch, st); break;
    default: r = launch_gated<__half>(p, true, scratch, st);
  }
  if (r != NSB_OK || !d_bias) return r;
  NSB_CUDA_TRY(launch_dependent(gated_bias_kernel, dim3((unsigned)((D + 31) / 32)), dim3(1024), 0, st,
                                (const float*)bias_part, d_bias, (long long)(nsb_gated_chunks(T) * B), (long long)D),
               "launch gated_bias_kernel");
  return NSB_OK;
}

extern "C" int nsb_gated_recurrence_step(const void* raw, int64_t raw_stride_b, const void* x, int64_t x_stride_b,
                                         const float* bias, float* h, void* y, int64_t B, int64_t D, int dtype,
                                         void* stream) {
  if (B < 0 || D < 0 || !ok_dtype(dtype)) return NSB_ERR_INVALID_ARG;
  if (B * D == 0) return NSB_OK;
  const size_t es = dtype_size(dtype);
  if (!raw || !x || !h || !y || !fits(raw, es) || !fits(x, es) || !fits(y, es) || !fits(h, 4) || !fits(bias, 4))
    return NSB_ERR_INVALID_ARG;
  DeviceInfo dev;
  const int r = get_device_info(&dev);
  if (r != NSB_OK) return r;
  int V = 4;
  auto ok = [&](int v) {
    return D % v == 0 && raw_stride_b % v == 0 && x_stride_b % v == 0 && fits(raw, es * v) && fits(x, es * v) &&
           fits(y, es * v) && fits(h, 4 * v);
  };
  while (V > 1 && !ok(V)) V /= 2;
  const long long n = B * (D / V);
  const int blocks = (int)std::max<long long>(1, std::min<long long>((n + 255) / 256, (long long)dev.sm_count * 16));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define NSB_GO(T_, V_)                                                                                             \
  gated_step_kernel<T_, V_><<<blocks, 256, 0, st>>>(static_cast<const T_*>(raw), static_cast<const T_*>(x), bias, \
                                                    h, static_cast<T_*>(y), B, D, raw_stride_b, x_stride_b)
#define NSB_GO_T(T_)        \
  if (V == 4) NSB_GO(T_, 4); \
  else if (V == 2) NSB_GO(T_, 2); \
  else NSB_GO(T_, 1)
  switch (dtype) {
    case NSB_F32: NSB_GO_T(float); break;
    case NSB_BF16: NSB_GO_T(__nv_bfloat16); break;
    default: NSB_GO_T(__half); break;
  }
#undef NSB_GO_T
#undef NSB_GO
  NSB_CUDA_TRY(cudaGetLastError(), "launch gated_step_kernel");
  return NSB_OK;
}
