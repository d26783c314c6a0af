// Gated linear recurrence (the PLIF membrane without its spike, gate from a raw projection):
//
//   f_t = sigmoid(raw_t + bias)      h_t = f_t h_{t-1} + (1 - f_t) x_t      y_t = h_t
//
// and its reverse-time gradient. With K_{t+1} = f_{t+1} G_{t+1} what step t + 1 hands back to step t:
//
//   G_t = dy_t + K_{t+1}     dx_t = (1 - f_t) G_t     draw_t = G_t (h_{t-1} - x_t) f_t (1 - f_t)
//
// Each step is an affine map of the state, h -> P h + H, and such maps compose associatively, so time is
// cut into chunks that are worked on side by side. A tile is one chunk (at most 128 steps, 64 in the backward) of one block of columns:
// every warp has S steps of 32 V columns in registers, finds their composed map, the CTA's warps exchange
// their maps through shared memory, CTAs exchange theirs through global memory (below), and every warp then
// runs its steps once more from its true starting state. Each input is read once and each output written
// once; the only other traffic is 4-12 bytes per chunk and column.
//
// Hand-over between the chunks of a column block. Chunks come in groups of g: a chunk publishes its map
// (P, H), the last chunk of a group publishes the state after it instead. A chunk's starting state is the
// state after the group before, taken through the maps of the chunks of its own group that precede it, always
// in the same order: results do not depend on timing. A published word is its own flag: the scratch is
// filled with 0xff bytes, which no published value has (see publishable), and 8-byte words are written
// whole. Tiles are handed out by a ticket counter in order of time and a CTA works on its tickets in order, so
// whatever a tile waits for is being worked on or finished; every wait is bounded all the same and hands on NaN
// if it gives up.
//
// CTAs stay and take tile after tile: the next tile's inputs are copied to shared memory (by the thread that
// will use them, so that nothing needs a barrier) while this one is worked on.
//
// Long forwards with packed sequences or few columns go another way: one launch finds the maps of all chunks, one
// takes the state through them, and one works on the chunks from known states, reading the inputs a second time.
#include <algorithm>
#include <atomic>

#include "nsb_cols.cuh"

namespace nsb {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kFwdSteps = 16, kBwdSteps = 8;  // steps of a warp's tile
constexpr int kCkptRows = 64;                 // rows between the states that the forward saves: a backward chunk
constexpr uint32_t kEmpty = 0xffffffffu;
constexpr uint32_t kErrGated = 0x00400000u;

struct GatedParams {
  const void *raw, *x, *dy;
  const float *bias, *h0, *dh_last;
  const int* cu;                    // packed sequences: their first rows, and the end of the last
  void *y, *d_raw, *d_x;
  float *h_last, *ckpt, *d_h0, *d_bias_part;
  long long raw_st, raw_sb, x_st, x_sb;  // strides in elements between rows and between blocks of Dw columns
  int T, cols, Dw, D;               // D: period of the bias
  int nb, nchunks, g, g_log2, wt, S_seqs;  // nb: column blocks
  uint32_t d_magic;                 // col / D = __umulhi(col, d_magic) >> d_shift, for col below 2^31 and D > 1
  int d_shift;
  uint32_t* ticket;
  uint2* maps;                      // [nchunks][cols] (P, H)
  uint32_t* states;                 // [nchunks / g][cols]
  float* starts;                    // [nchunks][cols]: the states before the chunks, of three launches
  uint32_t* err;
  unsigned long long limit_ns;
};

// f = sigmoid(a + b) and m = sigmoid(-(a + b)) from e = exp(-(a + b)): f = 1 / (1 + e), m = e f, neither of them
// a difference, so both keep their digits however small they are. a + b comes first: of two large numbers that nearly
// cancel, scaled by log2(e) one by one, the roundings would be left. The exponent is capped where f is 2^-126
// (e f must not become inf * 0); min.NaN lets a NaN through.
//
// An error of f counts 1 / (1 - f) times in the states, and the reciprocal's is biased: with gates of 0.998 outputs were up to
// 9 times further from 64 bits than with a rounded quotient. So the quotient takes one Newton step on the residual
// 1 - f - m, in which 1 - f is exact from f = 1/2 up and nothing hangs on the rounding of 1 + e. f is then off by half a unit
// in the last place and by what e and m are off, which counts 1 - f times (8192 x 49152 bf16: forward 557 -> 585 us, backward
// 1128 -> 1146). m keeps the approximation's last place: an error of m counts once.
template <int V>
__device__ __forceinline__ void gate(const Cols<V>& a, const Cols<V>& b, Cols<V>& f, Cols<V>& m) {
  Cols<V> q = mul<V>(add<V>(a, b), all<V>(-kLog2e)), e;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    asm("min.NaN.f32 %0, %1, 0f42FC0000;" : "=f"(q[v]) : "f"(q[v]));  // 126
    e[v] = ex2(q[v]);
  }
  q = add<V>(e, all<V>(1.0f));
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = rcp(q[v]);
  m = mul<V>(e, f);
  q = fma<V>(m, all<V>(-1.0f), fma<V>(f, all<V>(-1.0f), all<V>(1.0f)));
  f = fma<V>(f, q, f);
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
__device__ __forceinline__ unsigned long long peek64(const uint2* p) {
  unsigned long long v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ float published(uint32_t w) { return __uint_as_float(w == kEmpty ? 0x7fffffffu : w); }
__device__ __forceinline__ void post32(uint32_t* p, uint32_t v) {
  asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
__device__ __forceinline__ void post64(uint2* p, uint32_t a, uint32_t b) {
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"((unsigned long long)a | ((unsigned long long)b << 32))
               : "memory");
}

// Bounded wait of a whole warp for published words. `look(missing)` reads a lane's words, all at once, and if they are
// not all there leaves the address of (the low half of) one that is missing. With `watch` one lane watches that word
// alone and the warp looks again when it has come, which leaves the second-level cache to the others; without, every lane
// looks again at once, which saves a round trip where chunk after chunk waits for the one before (fp32 65536 x 768
// forward: 196 us, and 293 us watching; 8192 x 49152 bf16 backward, chunks long done: 1149 us watching, 1220 without). Words
// that never come read as NaN (and the error word says so).
template <typename Look>
__device__ __forceinline__ void await(Look look, bool watch, const GatedParams& p) {
  const uint32_t* missing = nullptr;
  bool there = look(missing);
  uint32_t waiting = __ballot_sync(0xffffffffu, !there);
  if (waiting == 0) return;
  const uint64_t t0 = global_timer_ns();
  uint32_t it = 0;
  do {
    bool gave_up = false;
    if ((threadIdx.x & 31) == __ffs(waiting) - 1) {
      do {
        gave_up = (++it & 0x3F) == 0 && (global_timer_ns() - t0 > p.limit_ns || it > (1u << 28));
      } while (watch && !gave_up && peek32(missing) == kEmpty);
      if (gave_up && p.err) atomicOr(reinterpret_cast<unsigned int*>(p.err), kErrGated);
    }
    if (__any_sync(0xffffffffu, gave_up)) return;
    there = there || look(missing);
  } while ((waiting = __ballot_sync(0xffffffffu, !there)) != 0);
}

// What the S rows of a warp are: bit s of `in` - row s belongs to a sequence; `first`, `last` - it is that
// sequence's first or last row. Lane s keeps the number of row s's sequence.
struct Rows {
  uint32_t in, first, last;
  int seq;
  // nothing but rows in the middle of a sequence
  __device__ __forceinline__ bool plain(int S) const { return in == (1u << S) - 1u && !(first | last); }
};
template <int S, bool PACKED>
__device__ __forceinline__ Rows row_kinds(const GatedParams& p, int t0, int lane) {
  Rows r;
  r.seq = 0;
  if constexpr (PACKED) {
    // 32 guesses at a time: lo = number of sequences that end at or before row t0
    int lo = 0, n = p.S_seqs;  // it lies in lo .. lo + n
    while (n > 0) {
      const int step = (n + 31) / 32, at = lane * step;
      const uint32_t b = __ballot_sync(0xffffffffu, at < n && __ldg(p.cu + lo + at + 1) <= t0);
      const int k = __popc(b);  // guesses 0 .. k - 1 hold, guess k does not
      if (k == 0) break;
      lo += (k - 1) * step + 1;
      n = min(step - 1, n - (k - 1) * step - 1);
    }
    // the ends around there, one per lane; each row counts those it has passed
    const int w = lo + lane <= p.S_seqs ? __ldg(p.cu + lo + lane) : 0x7fffffff;
    bool in = false, first = false, last = false;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int t = t0 + s;
      const uint32_t passed = __ballot_sync(0xffffffffu, lane > 0 && w <= t);
      int q = lo + __popc(passed), begin, end;
      if (passed == 0xfffffffeu) {  // over 30 sequences, nearly all of them empty, end among these rows
        int hi = p.S_seqs;
        while (q < hi) {
          const int mid = (q + hi) >> 1;
          if (__ldg(p.cu + mid + 1) <= t) q = mid + 1; else hi = mid;
        }
        begin = q < p.S_seqs ? __ldg(p.cu + q) : 0;
        end = q < p.S_seqs ? __ldg(p.cu + q + 1) : 0;
      } else {
        begin = __shfl_sync(0xffffffffu, w, q - lo);
        end = __shfl_sync(0xffffffffu, w, q - lo + 1);
      }
      if (lane == s) {
        in = t < p.T && q < p.S_seqs && begin <= t;
        r.seq = in ? q : 0;
        first = in && begin == t;
        last = in && end == t + 1;
      }
    }
    r.in = __ballot_sync(0xffffffffu, in);
    r.first = __ballot_sync(0xffffffffu, first);
    r.last = __ballot_sync(0xffffffffu, last);
  } else {
    const int left = p.T - t0;
    r.in = left >= S ? (1u << S) - 1u : left > 0 ? (1u << left) - 1u : 0u;
    r.first = t0 == 0 ? 1u : 0u;
    r.last = left > 0 && left <= S ? 1u << (left - 1) : 0u;
  }
  return r;
}

// The map h -> P h + H of one step or of several. Where a sequence of a packed batch begins, the state from before
// must not come in, not even as 0 * NaN: such a map has P = -0 (a product of gates is never negative) and gives H.
template <int V>
struct MapV {
  Cols<V> P, H;
};
constexpr float kCut = -0.0f;
__device__ __forceinline__ bool is_cut(float P) { return __float_as_uint(P) == 0x80000000u; }
template <bool PACKED, int V>
__device__ __forceinline__ Cols<V> apply_map(const Cols<V>& P, const Cols<V>& H, const Cols<V>& h) {
  Cols<V> r = fma<V>(P, h, H);
  if constexpr (PACKED)
#pragma unroll
    for (int v = 0; v < V; ++v) r[v] = is_cut(P[v]) ? H[v] : r[v];
  return r;
}
// m, then (P, H)
template <bool PACKED, int V>
__device__ __forceinline__ void then_map(MapV<V>& m, const Cols<V>& P, const Cols<V>& H) {
  m.H = apply_map<PACKED, V>(P, H, m.H);
  Cols<V> r = mul<V>(m.P, P);
  if constexpr (PACKED)
#pragma unroll
    for (int v = 0; v < V; ++v) r[v] = is_cut(m.P[v]) || is_cut(P[v]) ? kCut : r[v];
  m.P = r;
}

// The state (or, in reverse, the hand-back) that a chunk starts from. `pos` counts chunks in the order in
// which they are worked on. The state before the group was looked for when the tile was begun (`early`). With g = 1
// that is all; otherwise every time warp takes the maps of four of the preceding chunks of the group and composes
// them in order, and the parts meet in shared memory. Same value in every time warp.
template <int V>
struct Early {
  uint32_t w[V];
  __device__ __forceinline__ void look(const GatedParams& p, int row, int col, bool on) {
#pragma unroll
    for (int v = 0; v < V; ++v) w[v] = 0;
    if (row >= 0 && on)
#pragma unroll
      for (int v = 0; v < V; ++v) w[v] = peek32(p.states + (long long)row * p.cols + col + v);
  }
};
template <int V>
__device__ __forceinline__ Cols<V> state_before(const GatedParams& p, Early<V>& early, int row, int col, bool on) {
  bool looked = true;  // (when the tile was begun)
  await([&](const uint32_t*& missing) {
    if (!looked) early.look(p, row, col, on);
    looked = false;
    bool r = true;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (early.w[v] == kEmpty) r = false, missing = p.states + (long long)row * p.cols + col + v;
    return r;
  }, p.g == 1, p);
  Cols<V> r;
#pragma unroll
  for (int v = 0; v < V; ++v) r[v] = published(early.w[v]);
  return r;
}
// `part`: shared memory that nobody else uses from here to the caller's next barrier
template <bool PACKED, int V>
__device__ __forceinline__ Cols<V> chunk_start(const GatedParams& p, Early<V>& early, int pos, int col, bool on,
                                               int wt_idx, int wt, MapV<V>* part, int first_slot) {
  const int group = pos >> p.g_log2;
  if (p.g == 1) return state_before<V>(p, early, group - 1, col, on);
  const int j = pos - group * p.g;
  constexpr int kMost = 4;  // 31 maps among 8 warps; with fewer time warps there is one chunk
  MapV<V> m = {all<V>(1.0f), all<V>(0.0f)};
  const int n = min(kMost, j - wt_idx * kMost);
  if (n > 0) {
    const uint2* w = p.maps + (long long)(group * p.g + wt_idx * kMost) * p.cols + col;
    unsigned long long q[kMost][V];
    await([&](const uint32_t*& missing) {
#pragma unroll
      for (int i = 0; i < kMost; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) q[i][v] = on && i < n ? peek64(w + (long long)i * p.cols + v) : 0ull;
      bool r = true;
#pragma unroll
      for (int i = 0; i < kMost; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v)
          if ((uint32_t)q[i][v] == kEmpty) r = false, missing = &w[(long long)i * p.cols + v].x;
      return r;
    }, false, p);
#pragma unroll
    for (int i = 0; i < kMost; ++i)
      if (i < n) {
        Cols<V> P, H;
#pragma unroll
        for (int v = 0; v < V; ++v) P[v] = published((uint32_t)q[i][v]), H[v] = published((uint32_t)(q[i][v] >> 32));
        then_map<PACKED, V>(m, P, H);
      }
  }
  if (wt_idx == 0) m.H = apply_map<PACKED, V>(m.P, m.H, state_before<V>(p, early, group - 1, col, on));
  part[threadIdx.x] = m;
  __syncthreads();
  Cols<V> start = part[first_slot].H;
  for (int i = 1; i < wt; ++i) start = apply_map<PACKED, V>(part[first_slot + i * 32].P, part[first_slot + i * 32].H, start);
  return start;
}

// A thread's inputs in shared memory: slot (stream, step) of B bytes = V elements.
template <typename T, int V, int S>
struct Stage {
  static constexpr int B = sizeof(T) * V;
  static constexpr int kSlot = B < 4 ? 4 : B;  // (a slot also takes an fp32 intermediate)
  static constexpr int kStream = S * kThreads * kSlot;  // bytes of one stream's rows
  char* base;
  __device__ __forceinline__ char* slot(int stream, int s) const {
    return base + ((stream * S + s) * kThreads + threadIdx.x) * kSlot;
  }
  // Rows of one stream, from its element in row t0. Copies of 4 bytes and more run asynchronously; single 16-bit
  // elements go through registers. Rows beyond T read as zeros.
  __device__ __forceinline__ void fill(int stream, const T* at, long long stride, int rows) const {
    if constexpr (B >= 4) {
      const uint32_t to = smem_u32(slot(stream, 0));
      if (rows >= S) {
#pragma unroll
        for (int s = 0; s < S; ++s, at += stride)
          asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to + s * kThreads * kSlot), "l"(at), "n"(B) : "memory");
      } else {
#pragma unroll
        for (int s = 0; s < S; ++s)
          asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to + s * kThreads * kSlot),
                       "l"(s < rows ? at + s * stride : at), "n"(B), "r"(s < rows ? B : 0)
                       : "memory");
      }
    } else {
      T v[S];
#pragma unroll
      for (int s = 0; s < S; ++s) v[s] = s < rows ? at[s * stride] : Elem<T>::zero();
#pragma unroll
      for (int s = 0; s < S; ++s) *reinterpret_cast<T*>(slot(stream, s)) = v[s];
    }
  }
  __device__ __forceinline__ Cols<V> get(int stream, int s) const { return widen<T, V>(*reinterpret_cast<const Vec<T, V>*>(slot(stream, s))); }
  // V fp32 values of a step in its slots of the streams 0 and 1, as many in each as fit
  static constexpr int kFloats = kSlot / 4;
  __device__ __forceinline__ void put_f32(int s, const Cols<V>& c) const {
#pragma unroll
    for (int v = 0; v < V; v += kFloats) {
      Vec<float, kFloats> q;
#pragma unroll
      for (int i = 0; i < kFloats; ++i) q.v[i] = c[v + i];
      *reinterpret_cast<Vec<float, kFloats>*>(slot(v / kFloats, s)) = q;
    }
  }
  __device__ __forceinline__ Cols<V> get_f32(int s) const {
    Cols<V> c;
#pragma unroll
    for (int v = 0; v < V; v += kFloats) {
      const Vec<float, kFloats> q = *reinterpret_cast<const Vec<float, kFloats>*>(slot(v / kFloats, s));
#pragma unroll
      for (int i = 0; i < kFloats; ++i) c[v + i] = q.v[i];
    }
    return c;
  }
};
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait_but_last() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// What a CTA works on: a block of columns in a chunk, the pos-th in the order of work. pos < 0: nothing is left.
struct Tile {
  int pos, block;
};
// A CTA's tiles. CHAIN: tickets, drawn by one thread and passed on at the barrier that every tile has. Where chunks
// pass maps, the next one is drawn when a tile is begun, not earlier: tiles are then begun nearly in the order of
// their numbers, and none that others wait for lies behind another tile in its own CTA (two drawn at the start
// put every second one there, 3.5 times the time). With g = 1 only the block's own previous
// chunk matters, long done, so tickets are drawn, and inputs copied, one tile further ahead. Without CHAIN there is
// one chunk, and every CTA has its share of its blocks.
template <bool CHAIN>
struct Tickets {
  Tile* shared;  // [2]
  uint32_t drawn;
  __device__ __forceinline__ Tile tile(const GatedParams& p) const {
    const int pos = drawn / (uint32_t)p.nb;
    return pos < p.nchunks ? Tile{pos, (int)(drawn - (uint32_t)pos * p.nb)} : Tile{-1, 0};
  }
  __device__ __forceinline__ Tile first(const GatedParams& p) {
    if constexpr (CHAIN) return another(p);
    drawn = blockIdx.x;
    return Tile{0, (int)drawn};
  }
  __device__ __forceinline__ Tile another(const GatedParams& p) {
    if constexpr (!CHAIN) return receive(p, 0);
    draw(p);
    pass_on(p, 1);
    __syncthreads();
    const Tile t = shared[1];
    __syncthreads();
    return t;
  }
  __device__ __forceinline__ void draw(const GatedParams& p) {
    if constexpr (CHAIN)
      if (threadIdx.x == 0) drawn = atomicAdd(p.ticket, 1u) + 1u;  // (the counter starts at 0xffffffff)
  }
  __device__ __forceinline__ void pass_on(const GatedParams& p, int parity) {
    if constexpr (CHAIN)
      if (threadIdx.x == 0) shared[parity] = tile(p);
  }
  __device__ __forceinline__ Tile receive(const GatedParams& p, int parity) {
    if constexpr (CHAIN) return shared[parity];
    drawn += gridDim.x;
    return drawn < (uint32_t)p.nb ? Tile{0, (int)drawn} : Tile{-1, 0};
  }
};

__device__ __forceinline__ long long input_at(const GatedParams& p, int col, long long st, long long sb, int t0) {
  if (p.Dw == p.cols) return t0 * st + col;
  const int b = col / p.Dw;
  return t0 * st + b * sb + (col - b * p.Dw);
}
template <int V>
__device__ __forceinline__ Cols<V> load_bias(const GatedParams& p, int col, bool on) {
  Cols<V> b = all<V>(0.0f);
  if (p.bias && on) {
    int d = p.D == p.cols ? col : p.D == 1 ? 0 : col - p.D * (int)(__umulhi((uint32_t)col, p.d_magic) >> p.d_shift);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      b[v] = __ldg(p.bias + d);
      d = d + 1 == p.D ? 0 : d + 1;
    }
  }
  return b;
}
template <bool PACKED, int V>
__device__ __forceinline__ Cols<V> state_at(const GatedParams& p, const float* from, const Rows& rows, int s, int col, bool on) {
  const int q = PACKED ? __shfl_sync(0xffffffffu, rows.seq, s) : 0;
  Cols<V> o;
#pragma unroll
  for (int v = 0; v < V; ++v) o[v] = (from && on) ? from[(long long)q * p.cols + col + v] : 0.0f;
  return o;
}
template <bool PACKED, int V>
__device__ __forceinline__ void put_state(const GatedParams& p, float* to, const Rows& rows, int s, int col, bool on,
                                          const Cols<V>& o) {
  const int q = PACKED ? __shfl_sync(0xffffffffu, rows.seq, s) : 0;
  if (on && to)
#pragma unroll
    for (int v = 0; v < V; ++v) to[(long long)q * p.cols + col + v] = o[v];
}
// An empty sequence ends in the state that it starts from (and hands back what it is handed).
template <int V>
__device__ __forceinline__ void empty_sequences(const GatedParams& p, const float* from, float* to, int col, int first, int step) {
  if (to)
    for (int q = first; q < p.S_seqs; q += step)
      if (__ldg(p.cu + q + 1) <= __ldg(p.cu + q))
#pragma unroll
        for (int v = 0; v < V; ++v)
          to[(long long)q * p.cols + col + v] = from ? from[(long long)q * p.cols + col + v] : 0.0f;
}
template <int V>
__device__ __forceinline__ void post_map(const GatedParams& p, int pos, int col, const MapV<V>& m) {
#pragma unroll
  for (int v = 0; v < V; ++v)
    post64(p.maps + (long long)pos * p.cols + col + v, publishable(m.P[v]), publishable(m.H[v]));
}
template <int V>
__device__ __forceinline__ void post_state(const GatedParams& p, int pos, int col, const Cols<V>& h) {
#pragma unroll
  for (int v = 0; v < V; ++v) post32(p.states + (long long)(pos >> p.g_log2) * p.cols + col + v, publishable(h[v]));
}
struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

template <typename T, int V, bool PACKED, bool CHAIN>
__global__ void __launch_bounds__(kThreads, 2) gated_fwd_kernel(const GatedParams p) {
  constexpr int S = kFwdSteps;
  extern __shared__ __align__(16) char smem[];
  __shared__ MapV<V> maps[2][kThreads], part[CHAIN ? kThreads : 1];
  __shared__ Tile s_tiles[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wt = p.wt, wt_idx = warp % wt, wc_idx = warp / wt;
  const int first_slot = wc_idx * wt * 32 + lane;  // the warps of this column group: first_slot + 32 i in time order
  const int my_col = wc_idx * (32 * V) + lane * V, width = 32 * V * (kWarps / wt);
  auto stage = [&](int i) { return Stage<T, V, S>{smem + i * (2 * Stage<T, V, S>::kStream)}; };
  auto fill = [&](const Tile t, const Stage<T, V, S> st, Cols<V>& bias) {
    const int col = t.block * width + my_col, t0 = (t.pos * wt + wt_idx) * S;
    const bool on = t.pos >= 0 && col < p.cols;
    if (on) {
      st.fill(0, static_cast<const T*>(p.raw) + input_at(p, col, p.raw_st, p.raw_sb, t0), p.raw_st, p.T - t0);
      st.fill(1, static_cast<const T*>(p.x) + input_at(p, col, p.x_st, p.x_sb, t0), p.x_st, p.T - t0);
    }
    copies_commit();
    bias = load_bias<V>(p, col, on);
  };
  Tickets<CHAIN> tickets{s_tiles};
  Tile tile = tickets.first(p), next = {-1, 0};
  Cols<V> bias, next_bias;
  fill(tile, stage(0), bias);
  const bool ahead = !CHAIN || p.g == 1;
  if (ahead) next = tickets.another(p);

  for (int parity = 0; tile.pos >= 0; parity ^= 1) {
    if (ahead) fill(next, stage(parity ^ 1), next_bias);
    tickets.draw(p);
    const int col = tile.block * width + my_col, t0 = (tile.pos * wt + wt_idx) * S;
    const bool on = col < p.cols;
    Early<V> early;
    if constexpr (CHAIN) early.look(p, (tile.pos >> p.g_log2) - 1, col, on && (p.g == 1 || wt_idx == 0));
    const Rows rows = row_kinds<S, PACKED>(p, t0, lane);
    const bool plain = rows.plain(S);
    const Stage<T, V, S> in = stage(parity);
    if (ahead) copies_wait_but_last(); else copies_wait();

    Cols<V> f[S], u[S];
    MapV<V> mine = {all<V>(1.0f), all<V>(0.0f)};
    auto local = [&](auto special) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if constexpr (decltype(special)::value)
          if ((rows.first >> s) & 1u) mine = {all<V>(kCut), state_at<PACKED, V>(p, p.h0, rows, s, col, on)};
        Cols<V> m;
        gate<V>(in.get(0, s), bias, f[s], m);
        u[s] = mul<V>(m, in.get(1, s));
        mine.P = mul<V>(mine.P, f[s]);
        mine.H = fma<V>(f[s], mine.H, u[s]);
      }
    };
    if (plain) local(No()); else local(Yes());
    maps[parity][threadIdx.x] = mine;
    tickets.pass_on(p, parity);
    __syncthreads();
    const Tile drawn = tickets.receive(p, parity);
    if (!ahead) fill(next = drawn, stage(parity ^ 1), next_bias);

    Cols<V> h = all<V>(0.0f);
    const bool speaker = CHAIN && wt_idx == wt - 1 && on && tile.pos + 1 < p.nchunks;
    const bool group_end = CHAIN && (tile.pos & (p.g - 1)) == p.g - 1;
    if constexpr (CHAIN) {
      if (speaker && !group_end) {
        MapV<V> whole = maps[parity][first_slot];
        for (int i = 1; i < wt; ++i) then_map<PACKED, V>(whole, maps[parity][first_slot + i * 32].P, maps[parity][first_slot + i * 32].H);
        post_map<V>(p, tile.pos, col, whole);
      }
      h = chunk_start<PACKED, V>(p, early, tile.pos, col, on, wt_idx, wt, part, first_slot);
    }
    for (int i = 0; i < wt_idx; ++i) h = apply_map<PACKED, V>(maps[parity][first_slot + i * 32].P, maps[parity][first_slot + i * 32].H, h);
    if (p.ckpt && t0 % kCkptRows == 0 && t0 < p.T && on)
#pragma unroll
      for (int v = 0; v < V; ++v) p.ckpt[(long long)(t0 / kCkptRows) * p.cols + col + v] = h[v];
    if (speaker && group_end) post_state<V>(p, tile.pos, col, apply_map<PACKED, V>(mine.P, mine.H, h));
    T* y = static_cast<T*>(p.y) + (long long)t0 * p.cols + col;
    auto run = [&](auto special) {
#pragma unroll
      for (int s = 0; s < S; ++s, y += p.cols) {
        if constexpr (decltype(special)::value)
          if ((rows.first >> s) & 1u) h = state_at<PACKED, V>(p, p.h0, rows, s, col, on);
        h = fma<V>(f[s], h, u[s]);
        if constexpr (decltype(special)::value) {
          if (on && t0 + s < p.T)
            *reinterpret_cast<Vec<T, V>*>(y) = narrow<T, V>(((rows.in >> s) & 1u) ? h : all<V>(0.0f));
          if ((rows.last >> s) & 1u) put_state<PACKED, V>(p, p.h_last, rows, s, col, on, h);
        } else {
          if (on) *reinterpret_cast<Vec<T, V>*>(y) = narrow<T, V>(h);
        }
      }
    };
    if (plain) run(No()); else run(Yes());
    if constexpr (PACKED)
      if (tile.pos == 0 && on) empty_sequences<V>(p, p.h0, p.h_last, col, wt_idx, p.wt);
    tile = next;
    next = drawn;
    bias = next_bias;
  }
}

// Reverse pass of a chunk. Both directions need only the products of f and a partial sum each, so one exchange
// carries them: (P, H) takes a state forward through a warp's steps (the forward's states are computed again
// from the chunk's saved starting state), (P, K) takes the hand-back through them in reverse. f and 1 - f stay in
// registers, x and dy in shared memory, and h_{t-1} - x_t takes the place of raw and x there. The exchange has one
// buffer and a barrier before it is written again.
template <int V>
struct TripleV {
  Cols<V> P, H, K;
};

template <typename T, int V, bool PACKED, bool CHAIN>
__global__ void __launch_bounds__(kThreads, 3) gated_bwd_kernel(const GatedParams p) {
  constexpr int S = kBwdSteps;
  extern __shared__ __align__(16) char smem[];
  __shared__ TripleV<V> trip[kThreads];
  __shared__ Cols<V> s_db[kThreads];
  __shared__ Tile s_tiles[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int wt = p.wt, wt_idx = warp % wt, wc_idx = warp / wt;
  const int first_slot = wc_idx * wt * 32 + lane;
  const int my_col = wc_idx * (32 * V) + lane * V, width = 32 * V * (kWarps / wt);
  auto stage = [&](int i) { return Stage<T, V, S>{smem + i * (3 * Stage<T, V, S>::kStream)}; };
  auto fill = [&](const Tile t, const Stage<T, V, S> st, Cols<V>& bias, Cols<V>& ckpt) {
    const int chunk = p.nchunks - 1 - t.pos, col = t.block * width + my_col, t0 = (chunk * wt + wt_idx) * S;
    const bool on = t.pos >= 0 && col < p.cols;
    if (on) {
      st.fill(0, static_cast<const T*>(p.raw) + input_at(p, col, p.raw_st, p.raw_sb, t0), p.raw_st, p.T - t0);
      st.fill(1, static_cast<const T*>(p.x) + input_at(p, col, p.x_st, p.x_sb, t0), p.x_st, p.T - t0);
      st.fill(2, static_cast<const T*>(p.dy) + (long long)t0 * p.cols + col, p.cols, p.T - t0);
    }
    copies_commit();
    bias = load_bias<V>(p, col, on);
#pragma unroll
    for (int v = 0; v < V; ++v) ckpt[v] = (on && p.ckpt) ? __ldg(p.ckpt + (long long)chunk * p.cols + col + v) : 0.0f;
  };
  // the sum over a tile's steps of d_raw, added up in the order of the warps one barrier later
  auto bias_sum = [&](const Tile t) {
    const int col = t.block * width + my_col;
    if (p.d_bias_part && wt_idx == 0 && col < p.cols) {
      Cols<V> sum = s_db[first_slot];
      for (int i = 1; i < wt; ++i) sum = add<V>(sum, s_db[first_slot + i * 32]);
#pragma unroll
      for (int v = 0; v < V; ++v) p.d_bias_part[(long long)(p.nchunks - 1 - t.pos) * p.cols + col + v] = sum[v];
    }
  };
  Tickets<CHAIN> tickets{s_tiles};
  Tile tile = tickets.first(p), next = {-1, 0}, before = {-1, 0};
  Cols<V> bias, next_bias, h, next_h;
  fill(tile, stage(0), bias, h);
  const bool ahead = !CHAIN || p.g == 1;
  if (ahead) next = tickets.another(p);

  for (int parity = 0; tile.pos >= 0; parity ^= 1) {
    if (ahead) fill(next, stage(parity ^ 1), next_bias, next_h);
    tickets.draw(p);
    const int chunk = p.nchunks - 1 - tile.pos, col = tile.block * width + my_col, t0 = (chunk * wt + wt_idx) * S;
    const bool on = col < p.cols;
    Early<V> early;
    if constexpr (CHAIN) early.look(p, (tile.pos >> p.g_log2) - 1, col, on && (p.g == 1 || wt_idx == 0));
    const Rows rows = row_kinds<S, PACKED>(p, t0, lane);
    const bool plain = rows.plain(S);
    const Stage<T, V, S> in = stage(parity);
    if (ahead) copies_wait_but_last(); else copies_wait();

    Cols<V> f[S], m[S];
    TripleV<V> mine = {all<V>(1.0f), all<V>(0.0f), all<V>(0.0f)};
    auto local = [&](auto special) {
      constexpr bool kSpecial = decltype(special)::value;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if constexpr (kSpecial)
          if ((rows.first >> s) & 1u) mine.H = state_at<PACKED, V>(p, p.h0, rows, s, col, on);
        gate<V>(in.get(0, s), bias, f[s], m[s]);
        mine.H = fma<V>(f[s], mine.H, mul<V>(m[s], in.get(1, s)));
        mine.P = mul<V>(mine.P, f[s]);
      }
      // A state does not pass a sequence's border in either direction: one product serves both. The cut is made behind the
      // products, which a NaN on either side of the border would undo.
      if constexpr (kSpecial)
        if ((rows.first | rows.last | ~rows.in) & ((1u << S) - 1u)) mine.P = all<V>(kCut);
#pragma unroll
      for (int s = S - 1; s >= 0; --s) {
        if constexpr (kSpecial)
          if ((rows.last >> s) & 1u) mine.K = state_at<PACKED, V>(p, p.dh_last, rows, s, col, on);
        mine.K = mul<V>(f[s], add<V>(mine.K, in.get(2, s)));
        if constexpr (kSpecial)
          if (!((rows.in >> s) & 1u)) mine.K = all<V>(0.0f);
      }
    };
    if (plain) local(No()); else local(Yes());
    tickets.pass_on(p, parity);
    __syncthreads();  // the exchange of the tile before has been read
    trip[threadIdx.x] = mine;
    const Tile drawn = tickets.receive(p, parity);
    if (!ahead) fill(next = drawn, stage(parity ^ 1), next_bias, next_h);
    if (before.pos >= 0) bias_sum(before);
    __syncthreads();

    Cols<V> K = all<V>(0.0f);
    const bool speaker = CHAIN && wt_idx == 0 && on && chunk > 0;
    const bool group_end = CHAIN && (tile.pos & (p.g - 1)) == p.g - 1;
    if constexpr (CHAIN) {
      if (speaker && !group_end) {
        const TripleV<V>& l = trip[first_slot + (wt - 1) * 32];
        MapV<V> whole = {l.P, l.K};
        for (int i = wt - 2; i >= 0; --i) then_map<PACKED, V>(whole, trip[first_slot + i * 32].P, trip[first_slot + i * 32].K);
        post_map<V>(p, tile.pos, col, whole);
      }
    }
    for (int i = 0; i < wt_idx; ++i) h = apply_map<PACKED, V>(trip[first_slot + i * 32].P, trip[first_slot + i * 32].H, h);
    MapV<V> behind = {all<V>(1.0f), all<V>(0.0f)};  // what lies between this warp's steps and the chunk's end
    for (int i = wt - 1; i > wt_idx; --i) then_map<PACKED, V>(behind, trip[first_slot + i * 32].P, trip[first_slot + i * 32].K);
    if constexpr (CHAIN) {
      if (p.g > 1) __syncthreads();  // the parts of the starting state take the place of the exchange
      K = chunk_start<PACKED, V>(p, early, tile.pos, col, on, wt_idx, wt, reinterpret_cast<MapV<V>*>(trip), first_slot);
    }
    K = apply_map<PACKED, V>(behind.P, behind.H, K);
    if (speaker && group_end) post_state<V>(p, tile.pos, col, apply_map<PACKED, V>(mine.P, mine.K, K));

    Cols<V> db = all<V>(0.0f);
    auto run = [&](auto special) {
      constexpr bool kSpecial = decltype(special)::value;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if constexpr (kSpecial)
          if ((rows.first >> s) & 1u) h = state_at<PACKED, V>(p, p.h0, rows, s, col, on);
        const Cols<V> x = in.get(1, s);
        const Cols<V> d = fma<V>(x, all<V>(-1.0f), h);
        in.put_f32(s, d);
        h = fma<V>(f[s], h, mul<V>(m[s], x));
      }
      T* o_raw = static_cast<T*>(p.d_raw) + (long long)(t0 + S - 1) * p.cols + col;
      T* o_x = static_cast<T*>(p.d_x) + (long long)(t0 + S - 1) * p.cols + col;
#pragma unroll
      for (int s = S - 1; s >= 0; --s, o_raw -= p.cols, o_x -= p.cols) {
        if constexpr (kSpecial)
          if ((rows.last >> s) & 1u) K = state_at<PACKED, V>(p, p.dh_last, rows, s, col, on);
        const Cols<V> d = in.get_f32(s);
        const Cols<V> G = add<V>(K, in.get(2, s));
        K = mul<V>(f[s], G);
        Cols<V> g_x = mul<V>(m[s], G), g_a = mul<V>(mul<V>(K, m[s]), d);
        if constexpr (kSpecial)
          if (!((rows.in >> s) & 1u)) g_x = g_a = all<V>(0.0f);
        db = add<V>(db, g_a);
        if (on && (!kSpecial || t0 + s < p.T)) {
          if (p.d_raw) *reinterpret_cast<Vec<T, V>*>(o_raw) = narrow<T, V>(g_a);
          if (p.d_x) *reinterpret_cast<Vec<T, V>*>(o_x) = narrow<T, V>(g_x);
        }
        if constexpr (kSpecial)
          if ((rows.first >> s) & 1u) put_state<PACKED, V>(p, p.d_h0, rows, s, col, on, K);
      }
    };
    if (plain) run(No()); else run(Yes());
    s_db[threadIdx.x] = db;
    if constexpr (PACKED)
      if (chunk == 0 && on) empty_sequences<V>(p, p.dh_last, p.d_h0, col, wt_idx, p.wt);
    before = tile;
    tile = next;
    next = drawn;
    bias = next_bias;
    h = next_h;
  }
  __syncthreads();
  if (before.pos >= 0) bias_sum(before);
}

// ---- long forwards: three launches instead of one
//
// Handing states from chunk to chunk inside a launch costs a round of waiting per round of resident tiles, and with
// packed sequences the search for those of a tile's rows lies on that path. Three launches read the inputs twice
// instead: the chunks' maps, their composition along time, then every chunk from its starting state. A warp has 64 steps
// of 32 V columns to itself, one after the other, so nothing is kept, exchanged or waited for inside a launch. Blocks whose
// rows and columns are all there load without conditions (28 + 33 us where 32 + 38 were, for 32768 x 768 bf16, before the gate's
// Newton step). Now 29 + 8 + 34 us, 3.5 and 4.4 TB/s, at half an instruction per cycle and scheduler and 28 % of the warps' places
// taken (384 CTAs for 444 places): what is loaded is waited for with little else to do.

// row_kinds of a whole chunk at once: the search for the sequences of its rows runs once, a row per lane and turn
struct ChunkRows {
  unsigned long long in, first, last;
  int seq[2];  // lane l: of rows l and l + 32
  template <int S>
  __device__ __forceinline__ Rows block(int i, int lane) const {
    Rows r;
    const uint32_t mask = (1u << S) - 1u;
    r.in = (uint32_t)(in >> (i * S)) & mask;
    r.first = (uint32_t)(first >> (i * S)) & mask;
    r.last = (uint32_t)(last >> (i * S)) & mask;
    r.seq = __shfl_sync(0xffffffffu, i * S < 32 ? seq[0] : seq[1], (i * S + lane) & 31);
    return r;
  }
};
template <bool PACKED>
__device__ __forceinline__ ChunkRows chunk_rows(const GatedParams& p, int t0, int lane) {
  ChunkRows c = {0ull, 0ull, 0ull, {0, 0}};
  if constexpr (PACKED) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = t0 + 32 * h + lane;
      int lo = 0, hi = t < p.T ? p.S_seqs : 0;  // sequences that end at or before row t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(p.cu + mid + 1) <= t) lo = mid + 1; else hi = mid;
      }
      bool in = t < p.T && lo < p.S_seqs, first = false, last = false;
      if (in) {
        const int begin = __ldg(p.cu + lo), end = __ldg(p.cu + lo + 1);
        in = begin <= t;
        first = begin == t;
        last = in && end == t + 1;
      }
      c.seq[h] = in ? lo : 0;
      c.in |= (unsigned long long)__ballot_sync(0xffffffffu, in) << (32 * h);
      c.first |= (unsigned long long)__ballot_sync(0xffffffffu, first) << (32 * h);
      c.last |= (unsigned long long)__ballot_sync(0xffffffffu, last) << (32 * h);
    }
  } else {
    const int left = p.T - t0;
    c.in = left >= 64 ? ~0ull : (1ull << left) - 1ull;
    c.first = t0 == 0 ? 1ull : 0ull;
    c.last = left <= 64 ? 1ull << (left - 1) : 0ull;
  }
  return c;
}
static_assert(kCkptRows == 64, "");

// Rows that a warp requests together: 2 KB of each input, or 16 rows. (A second set of registers to request the next rows
// into spilled and was slower: 44 us instead of 37 for the last launch of 32768 x 768 bf16.)
template <typename T, int V>
constexpr int kRowsInFlight = V * sizeof(T) == 8 ? 8 : 16;

// The map (P, H) of every chunk.
template <typename T, int V, bool PACKED>
__global__ void __launch_bounds__(kThreads, 3) gated_maps_kernel(const GatedParams p) {
  constexpr int S = kRowsInFlight<T, V>;
  const int lane = threadIdx.x & 31;
  const long long id = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  grid_dependents_may_launch();
  const int chunk = (int)(id / p.nb), col = (int)(id - (long long)chunk * p.nb) * (32 * V) + lane * V;
  if (chunk >= p.nchunks) return;
  const bool on = col < p.cols, whole = col - lane * V + 32 * V <= p.cols;  // (cols below 2^31 - 2^8)
  const T* raw = static_cast<const T*>(p.raw) + (on ? input_at(p, col, p.raw_st, p.raw_sb, 0) : 0);
  const T* x = static_cast<const T*>(p.x) + (on ? input_at(p, col, p.x_st, p.x_sb, 0) : 0);
  const Cols<V> bias = load_bias<V>(p, col, on);
  MapV<V> m = {all<V>(1.0f), all<V>(0.0f)};
  const ChunkRows kinds = chunk_rows<PACKED>(p, chunk * kCkptRows, lane);
  for (int i = 0; i < kCkptRows / S; ++i) {
    const int t0 = chunk * kCkptRows + i * S;
    const T* raw_t = raw + t0 * p.raw_st;
    const T* x_t = x + t0 * p.x_st;
    Vec<T, V> vr[S], vx[S];
    if (whole && t0 + S <= p.T) {
#pragma unroll
      for (int s = 0; s < S; ++s, raw_t += p.raw_st, x_t += p.x_st) {
        vr[s] = *reinterpret_cast<const Vec<T, V>*>(raw_t);
        vx[s] = *reinterpret_cast<const Vec<T, V>*>(x_t);
      }
    } else {
#pragma unroll
      for (int s = 0; s < S; ++s, raw_t += p.raw_st, x_t += p.x_st) {
        const bool in = on && t0 + s < p.T;
        vr[s] = load_if<T, V>(in, raw_t);
        vx[s] = load_if<T, V>(in, x_t);
      }
    }
    const Rows rows = kinds.block<S>(i, lane);
    auto steps = [&](auto special) {
      constexpr bool kSpecial = decltype(special)::value;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if constexpr (kSpecial)
          if ((rows.first >> s) & 1u) m = {all<V>(kCut), state_at<PACKED, V>(p, p.h0, rows, s, col, on)};
        Cols<V> f, u;
        gate<V>(widen<T, V>(vr[s]), bias, f, u);
        m.P = mul<V>(m.P, f);
        m.H = fma<V>(f, m.H, mul<V>(u, widen<T, V>(vx[s])));
      }
    };
    if (rows.plain(S)) steps(No()); else steps(Yes());
  }
  if (on)
#pragma unroll
    for (int v = 0; v < V; ++v)
      p.maps[(long long)chunk * p.cols + col + v] = make_uint2(__float_as_uint(m.P[v]), __float_as_uint(m.H[v]));
}

// starts[i] = the state after the maps 0 .. i - 1, from zero. A CTA has 32 columns; warp w composes the w-th part of the chunks,
// takes the parts before its own from shared memory, and goes through its chunks again.
template <bool PACKED>
__global__ void __launch_bounds__(1024) gated_chain_kernel(const GatedParams p) {
  __shared__ MapV<1> parts[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  grid_dependents_may_launch();
  grid_dependency_wait();
  const int per = (p.nchunks + 31) / 32, a = min(w * per, p.nchunks), b = min(a + per, p.nchunks);
  const bool on = col < p.cols;
  const uint2* maps = p.maps + col;
  constexpr int kBatch = 16;  // maps on their way together
  uint2 q[kBatch];
  auto load = [&](int from) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      q[k] = on && from + k < b ? __ldcg(maps + (long long)(from + k) * p.cols) : make_uint2(0x3f800000u, 0u);
  };
  auto map_of = [&](int k) {
    MapV<1> m;
    m.P[0] = __uint_as_float(q[k].x), m.H[0] = __uint_as_float(q[k].y);
    return m;
  };
  MapV<1> m = {all<1>(1.0f), all<1>(0.0f)};
  for (int i = a; i < b; i += kBatch) {
    load(i);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const MapV<1> t = map_of(k);
      then_map<PACKED, 1>(m, t.P, t.H);
    }
  }
  parts[w][lane] = m;
  __syncthreads();
  Cols<1> h = all<1>(0.0f);
#pragma unroll 4
  for (int i = 0; i < w; ++i) h = apply_map<PACKED, 1>(parts[i][lane].P, parts[i][lane].H, h);
  for (int i = a; i < b; i += kBatch) {
    if (per > kBatch) load(i);
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (i + k < b) {
        const MapV<1> t = map_of(k);
        if (on) p.starts[(long long)(i + k) * p.cols + col] = h[0];
        h = apply_map<PACKED, 1>(t.P, t.H, h);
      }
  }
}

// Every chunk from its starting state, the last chunks first: they are the ones the cache still holds.
template <typename T, int V, bool PACKED>
__global__ void __launch_bounds__(kThreads, 3) gated_apply_kernel(const GatedParams p) {
  constexpr int S = kRowsInFlight<T, V>;
  const int lane = threadIdx.x & 31;
  const long long id = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int back = (int)(id / p.nb), chunk = p.nchunks - 1 - back, col = (int)(id - (long long)back * p.nb) * (32 * V) + lane * V;
  if (chunk < 0) return;
  const bool on = col < p.cols, whole = col - lane * V + 32 * V <= p.cols;  // (cols below 2^31 - 2^8)
  const T* raw = static_cast<const T*>(p.raw) + (on ? input_at(p, col, p.raw_st, p.raw_sb, 0) : 0);
  const T* x = static_cast<const T*>(p.x) + (on ? input_at(p, col, p.x_st, p.x_sb, 0) : 0);
  T* y = static_cast<T*>(p.y) + col;
  const Cols<V> bias = load_bias<V>(p, col, on);
  Cols<V> h;
  const ChunkRows kinds = chunk_rows<PACKED>(p, chunk * kCkptRows, lane);
  for (int i = 0; i < kCkptRows / S; ++i) {
    const int t0 = chunk * kCkptRows + i * S;
    const T* raw_t = raw + t0 * p.raw_st;
    const T* x_t = x + t0 * p.x_st;
    T* y_t = y + (long long)t0 * p.cols;
    Vec<T, V> vr[S], vx[S];
    if (whole && t0 + S <= p.T) {
#pragma unroll
      for (int s = 0; s < S; ++s, raw_t += p.raw_st, x_t += p.x_st) {
        vr[s] = *reinterpret_cast<const Vec<T, V>*>(raw_t);
        vx[s] = *reinterpret_cast<const Vec<T, V>*>(x_t);
      }
    } else {
#pragma unroll
      for (int s = 0; s < S; ++s, raw_t += p.raw_st, x_t += p.x_st) {
        const bool in = on && t0 + s < p.T;
        vr[s] = load_if<T, V>(in, raw_t);
        vx[s] = load_if<T, V>(in, x_t);
      }
    }
    const Rows rows = kinds.block<S>(i, lane);
    if (i == 0) {
      grid_dependency_wait();
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = on ? __ldcg(p.starts + (long long)chunk * p.cols + col + v) : 0.0f;
    }
    auto steps = [&](auto special) {
      constexpr bool kSpecial = decltype(special)::value;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if constexpr (kSpecial)
          if ((rows.first >> s) & 1u) h = state_at<PACKED, V>(p, p.h0, rows, s, col, on);
        Cols<V> f, m;
        gate<V>(widen<T, V>(vr[s]), bias, f, m);
        h = fma<V>(f, h, mul<V>(m, widen<T, V>(vx[s])));
        if (on && (!kSpecial || t0 + s < p.T))
          *reinterpret_cast<Vec<T, V>*>(y_t) =
              narrow<T, V>(!kSpecial || ((rows.in >> s) & 1u) ? h : all<V>(0.0f));
        if constexpr (kSpecial)
          if ((rows.last >> s) & 1u) put_state<PACKED, V>(p, p.h_last, rows, s, col, on, h);
        y_t += p.cols;
      }
    };
    if (rows.plain(S)) steps(No()); else steps(Yes());
  }
  if constexpr (PACKED)
    if (chunk == 0 && on) empty_sequences<V>(p, p.h0, p.h_last, col, 0, 1);
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
    const Vec<T, V> vr = *reinterpret_cast<const Vec<T, V>*>(raw + b * raw_sb + d);
    const Vec<T, V> vx = *reinterpret_cast<const Vec<T, V>*>(x + b * x_sb + d);
    Vec<float, V> vh = *reinterpret_cast<const Vec<float, V>*>(h + b * D + d);
    Cols<V> c, f, m, hv;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      c[v] = bias ? bias[d + v] : 0.0f;
      hv[v] = vh.v[v];
    }
    gate<V>(widen<T, V>(vr), c, f, m);
    hv = fma<V>(f, hv, mul<V>(m, widen<T, V>(vx)));
#pragma unroll
    for (int v = 0; v < V; ++v) vh.v[v] = hv[v];
    *reinterpret_cast<Vec<float, V>*>(h + b * D + d) = vh;
    *reinterpret_cast<Vec<T, V>*>(y + b * D + d) = narrow<T, V>(hv);
  }
}

// ------------------------------------------------------------------------------------------------ host

struct GatedPlan {
  int wt, nchunks, g, nb;
};

// Warps of a CTA along time: as many as the steps need, up to all of them; the rest lie side by side over
// the columns. Chunks hand on states one by one (g = 1) where a row of column blocks occupies all CTAs, so that
// a chunk's predecessor has finished long before; with fewer blocks, 32 chunks run side by side and pass maps.
GatedPlan plan_gated(long long T, long long cols, int V, int steps, long long ctas) {
  GatedPlan q;
  q.wt = 1;
  while (q.wt < kWarps && (long long)q.wt * steps < T) q.wt *= 2;
  const long long rows = (long long)q.wt * steps, width = 32LL * V * (kWarps / q.wt);
  q.nchunks = (int)((T + rows - 1) / rows);
  q.nb = (int)((cols + width - 1) / width);
  q.g = q.nb >= ctas ? 1 : 32;
  return q;
}
// chunks of the backward, which are the smaller ones
long long bwd_chunks(long long T) { return (T + kCkptRows - 1) / kCkptRows; }
static_assert(kBwdSteps * kWarps == kCkptRows && kFwdSteps * kWarps >= kCkptRows && kCkptRows % kFwdSteps == 0, "");

bool ok_dtype(int d) { return d == NSB_F32 || d == NSB_BF16 || d == NSB_F16; }
bool fits(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Scratch of a launch that hands over: [ticket, 3 words of padding][states][maps], filled with 0xff by one memset. Of three
// launches: [maps][starting states].
long long scratch_words(long long T, long long cols) {
  const long long chunks = bwd_chunks(T);
  if (chunks <= 1) return 0;
  // whatever the plan takes: all chunks' maps and all states
  return 4 + (3 * chunks * cols + cols + 3) / 4 * 4;
}

template <typename T, int V, bool BACKWARD, bool PACKED, bool CHAIN>
int start_kernel(const GatedParams& p, int ctas, int device, cudaStream_t st) {
  const int smem = 2 * (BACKWARD ? 3 * Stage<T, V, kBwdSteps>::kStream : 2 * Stage<T, V, kFwdSteps>::kStream);
  void (*kern)(const GatedParams);
  if constexpr (BACKWARD) kern = gated_bwd_kernel<T, V, PACKED, CHAIN>;
  else kern = gated_fwd_kernel<T, V, PACKED, CHAIN>;
  static std::atomic<uint64_t> set_on{0};  // devices that know of the kernel's shared memory
  const uint64_t bit = device < 64 ? 1ull << device : 0ull;
  if (!(set_on.load(std::memory_order_relaxed) & bit)) {
    NSB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "shared memory of the gated recurrence");
    set_on.fetch_or(bit, std::memory_order_relaxed);
  }
  const unsigned grid = (unsigned)std::min<long long>((long long)p.nb * p.nchunks, ctas);
  kern<<<grid, kThreads, smem, st>>>(p);
  NSB_CUDA_TRY(cudaGetLastError(), BACKWARD ? "launch gated_bwd_kernel" : "launch gated_fwd_kernel");
  return NSB_OK;
}

// Three launches read the inputs twice and cost some 25 us of their own, but in none does a chunk wait for another. They
// are taken for packed sequences (whose search lies on the path of the hand-over) from 40 MB of inputs, else from 64 MB
// and where there are few columns for the steps. Forward in us, three launches and one, inputs not in any cache:
//   packed, three taken   bf16 13100 x 768 43 and 51, 16384 x 768 51 and 61, 24000 x 768 55 and 78, 32768 x 768 63 and 104,
//     4096 x 6144 64 and 139, 32768 x 6144 352 and 590; fp16 20011 x 1001 71 and 146
//   packed, one taken     bf16 8192 x 768 30 and 37, 12288 x 768 35 and 49: the slower side (with 24 sequences)
//   else, three taken     bf16 24000 x 768 53 and 57, 32768 x 768 61 and 74, 65536 x 768 110 and 137; fp32 32768 x 768 90 and 109,
//     65536 x 768 172 and 204; fp16 20011 x 1001 66 and 102; bf16 32768 x 2048 135 and 155
//   else, one taken       bf16 12288 x 768 33 and 33, 16384 x 768 49 and 43, 8192 x 6144 106 and 102,
//     2048 x 49152 210 and 158, 8192 x 49152 680 and 578, 512 x 393216 498 and 311, fp32 16384 x 6144 313 and 293, fp16 20001 x 8008
//     297 and 297; the slower side by 1 to 5 %: bf16 16384 x 2048 82 and 84, 16384 x 4096 135 and 138, 16384 x 6144 188 and 190,
//     32768 x 6144 346 and 364
// The backward's three launches came out within 8% either way of its one, and were dropped.
bool three_launches(long long T, long long cols, size_t es, bool packed) {
  const double bytes = 2.0 * (double)T * (double)cols * (double)es;
  return packed ? bytes >= 40e6 : bytes >= 64e6 && T / 16 >= cols;
}

template <typename T, int V, bool PACKED>
int launch_maps(GatedParams p, cudaStream_t st) {
  p.nb = (int)((p.cols + 32LL * V - 1) / (32 * V));
  const long long warps = (long long)p.nb * p.nchunks;
  gated_maps_kernel<T, V, PACKED><<<(unsigned)((warps + kWarps - 1) / kWarps), kThreads, 0, st>>>(p);
  NSB_CUDA_TRY(cudaGetLastError(), "launch gated_maps_kernel");
  NSB_CUDA_TRY(launch_dependent(gated_chain_kernel<PACKED>, dim3((unsigned)((p.cols + 31) / 32)), dim3(1024), 0, st, p),
               "launch gated_chain_kernel");
  NSB_CUDA_TRY(launch_dependent(gated_apply_kernel<T, V, PACKED>, dim3((unsigned)((warps + kWarps - 1) / kWarps)), dim3(kThreads), 0, st, p),
               "launch gated_apply_kernel");
  return NSB_OK;
}

void set_bias_division(GatedParams& p) {
  if (p.D <= 1) return;
  int l = 0;  // division by multiplication (Granlund and Montgomery 1994): m = floor(2^(31 + l) / D) + 1, l = ceil(log2 D)
  while ((1LL << l) < p.D) ++l;
  p.d_magic = (uint32_t)((1ull << (31 + l)) / (uint64_t)p.D + 1);
  p.d_shift = l - 1;
}

template <typename T, bool BACKWARD>
int launch_gated(GatedParams p, uint32_t* scratch, cudaStream_t st) {
  DeviceInfo dev;
  int r = get_device_info(&dev);
  if (r != NSB_OK) return r;
  // 4 bytes of a row per lane: with 8 a warp's steps do not fit the registers as well (forward 16 steps x 4 bytes on
  // two CTAs per SM against 8 x 8: 97 and 143 us for 8192 x 6144 columns bf16; backward 8 x 4 on three against 8 x 8
  // on two: 194 and 226 us). One element where rows are not aligned to that or a warp would span all columns twice.
  auto all_fit = [&](int v) {
    const size_t a = sizeof(T) * v;
    bool ok = p.cols % v == 0 && p.raw_st % v == 0 && p.x_st % v == 0;
    if (p.Dw != p.cols) ok = ok && p.Dw % v == 0 && p.raw_sb % v == 0 && p.x_sb % v == 0;
    for (const void* q : {p.raw, p.x, p.dy, (const void*)p.y, (const void*)p.d_raw, (const void*)p.d_x})
      ok = ok && fits(q, a);
    return ok;
  };
  const bool packed = p.cu != nullptr;
  const long long chunks = bwd_chunks(p.T);
  if (!BACKWARD && chunks > 2 && three_launches(p.T, p.cols, sizeof(T), packed)) {
    if (!scratch || !fits(scratch, 16)) return NSB_ERR_INVALID_ARG;
    p.nchunks = (int)chunks;
    set_bias_division(p);
    p.maps = reinterpret_cast<uint2*>(scratch);
    p.starts = p.ckpt ? p.ckpt : reinterpret_cast<float*>(scratch + 2 * chunks * p.cols);
    // 8 bytes of a row per lane, fewer if the chunks then do not give every SM 8 warps
    int V = 8 / (int)sizeof(T);
    while (V > 1 && (!all_fit(V) || p.cols <= 16 * V || (p.cols + 32LL * V - 1) / (32 * V) * chunks < 8LL * dev.sm_count)) V /= 2;
#define NSB_GO_V(V_) (packed ? launch_maps<T, V_, true>(p, st) : launch_maps<T, V_, false>(p, st))
    if constexpr (sizeof(T) == 2)
      if (V == 4) return NSB_GO_V(4);
    return V == 2 ? NSB_GO_V(2) : NSB_GO_V(1);
#undef NSB_GO_V
  }
  int V = 4 / (int)sizeof(T);
  while (V > 1 && (!all_fit(V) || p.cols <= 16 * V)) V /= 2;
  const int ctas = dev.sm_count * (BACKWARD ? 3 : 2);
  const GatedPlan q = plan_gated(p.T, p.cols, V, BACKWARD ? kBwdSteps : kFwdSteps, ctas);
  p.nb = q.nb, p.nchunks = q.nchunks, p.g = q.g, p.wt = q.wt;
  while (1 << p.g_log2 < p.g) ++p.g_log2;
  set_bias_division(p);
  if ((long long)q.nb * q.nchunks > 0x7fffffffLL - 2 * ctas) return NSB_ERR_TOO_LARGE;
  const bool chain = q.nchunks > 1;
  if (chain) {
    if (!scratch || !fits(scratch, 16)) return NSB_ERR_INVALID_ARG;
    const long long nstates = (q.nchunks / q.g + 1LL) * p.cols;
    const long long nmaps = q.g > 1 ? 2LL * q.nchunks * p.cols : 0;
    p.ticket = scratch;
    p.states = scratch + 4;
    p.maps = reinterpret_cast<uint2*>(scratch + 4 + (nstates + 3) / 4 * 4);
    NSB_CUDA_TRY(cudaMemsetAsync(scratch, 0xff, 4 * (4 + (nstates + 3) / 4 * 4 + nmaps), st), "memset gated scratch");
  }
#define NSB_GO_V(V_)                                                                           \
  (packed ? (chain ? start_kernel<T, V_, BACKWARD, true, true>(p, ctas, dev.device, st)        \
                   : start_kernel<T, V_, BACKWARD, true, false>(p, ctas, dev.device, st))      \
          : (chain ? start_kernel<T, V_, BACKWARD, false, true>(p, ctas, dev.device, st)       \
                   : start_kernel<T, V_, BACKWARD, false, false>(p, ctas, dev.device, st)))
  if constexpr (sizeof(T) == 2)
    if (V == 2) return NSB_GO_V(2);
  return NSB_GO_V(1);
#undef NSB_GO_V
}

int check_sizes(int64_t T, int64_t B, int64_t D, int64_t seqs, const int32_t* cu, int dtype) {
  if (T < 0 || B < 0 || D < 0 || seqs < 0 || !ok_dtype(dtype)) return NSB_ERR_INVALID_ARG;
  if (cu ? (B != 1 || !fits(cu, 4)) : seqs != 0) return NSB_ERR_INVALID_ARG;
  if (T > 0x7fffff00LL || seqs > 0x7ffffff0LL || (D > 0 && B > 0x7fffff00LL / D)) return NSB_ERR_TOO_LARGE;
  return NSB_OK;
}

}  // namespace
}  // namespace nsb

using namespace nsb;

extern "C" int64_t nsb_gated_scratch_words(int64_t T, int64_t cols) {
  return T <= 0 || cols <= 0 ? 0 : scratch_words(T, cols);
}
extern "C" int64_t nsb_gated_chunks(int64_t T) { return T <= 0 ? 0 : bwd_chunks(T); }

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
  p.T = (int)T, p.cols = (int)cols, p.D = (int)D;
  p.Dw = (raw_stride_b == D && x_stride_b == D) || B == 1 ? p.cols : p.D;
  if (!(p.err = device_error_word_ptr())) return NSB_ERR_CUDA;
  p.limit_ns = get_wait_limit_ns();
  switch (dtype) {
    case NSB_F32: return launch_gated<float, false>(p, scratch, st);
    case NSB_BF16: return launch_gated<__nv_bfloat16, false>(p, scratch, st);
    default: return launch_gated<__half, false>(p, scratch, st);
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
  p.T = (int)T, p.cols = (int)cols, p.D = (int)D;
  p.Dw = (raw_stride_b == D && x_stride_b == D) || B == 1 ? p.cols : p.D;
  if (!(p.err = device_error_word_ptr())) return NSB_ERR_CUDA;
  p.limit_ns = get_wait_limit_ns();
  switch (dtype) {
    case NSB_F32: r = launch_gated<float, true>(p, scratch, st); break;
    case NSB_BF16: r = launch_gated<__nv_bfloat16, true>(p, scratch, st); break;
    default: r = launch_gated<__half, true>(p, scratch, st);
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
