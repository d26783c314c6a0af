// Group norm with an activation, channels last: x [N, L, C], statistics of a sample and a group of Cg = C / G
// channels over all L positions,
//
//   xh = (x - mean) * rstd     z = w xh + b     y = z sigmoid(z)  or  z
//
// and its gradient, with d = dy act'(z) and g = d w:
//
//   dx = rstd (g - mean(g) - xh mean(g xh))      dw = sum d xh      db = sum d
//
// Two layouts of the work. With one position (L = 1, the heads of a token) a group is Cg contiguous values: a
// thread keeps 16 bytes of a row and the few threads of a group exchange sums, everything in one pass. With
// more positions a sample's group is spread over rows, and its statistics come from several CTAs: a first
// launch leaves (count, mean, sum of squares about it) per group and slab of rows, a second joins them in a
// fixed order and applies them, walking the tensor backwards so that it starts with what the first read last.
//
// Variances are sums of squares about a mean of the same values, never a difference of large sums; partial
// ones are joined by Chan, Golub and LeVeque's formula. All sums are fp32; of dw and db those over a CTA's rows (its
// share of all rows where there is one position, else a slab of a sample), and the CTAs' parts are added in 64 bits.
//
// What this does not suit: a slab's CTA belongs to one sample and 256 channels. Samples of few positions, and groups of over
// 256 channels with one position, leave most of its threads without a row, and the backward writes two floats per sample
// and channel and has them added by C / 16 CTAs. Forward + backward, bf16, beside the same in elementary torch operations: 65536 x 768
// in 2 groups 7.1 ms and 3.5 (3 groups, of 256: 0.23 ms), 16384 x 4096 in 8 groups 6.8 ms and 4.4 (16 groups: 0.25 ms), 65536 x 3 x 48
// in 2 groups 2.3 ms and 0.9, 8192 x 8 x 768 in 12 groups 0.88 ms and 3.8.
#include <algorithm>

#include "nsb_cols.cuh"

namespace nsb {
namespace {

constexpr int kThreads = 256, kChannels = 256;  // most threads; channels of a CTA in the slab layout

struct NormParams {
  const void *x, *dy;
  const float *w, *b;
  void* y;
  float *mean, *rstd, *part, *sums;  // part: per group and slab; sums: per channel and slab (dw, db)
  float *dw, *db;
  long long N, L, parts;             // parts: rows of sums
  int C, G, Cg, act;
  float eps;
  int gpb, pieces, cblks, nslab;  // groups of a channel block, pieces of a group, channel blocks, slabs of rows
  long long slab_rows;
};

// sigmoid(z); where exp(-z) overflows the quotient is 0, as the limit is
template <int V>
__device__ __forceinline__ Cols<V> sigmoid(const Cols<V>& z) {
  Cols<V> q = mul<V>(z, all<V>(-kLog2e));
#pragma unroll
  for (int v = 0; v < V; ++v) q[v] = ex2(q[v]);
  q = add<V>(q, all<V>(1.0f));
#pragma unroll
  for (int v = 0; v < V; ++v) q[v] = rcp(q[v]);
  return q;
}
template <int V>
__device__ __forceinline__ Cols<V> activate(const Cols<V>& z, int act) {
  return act ? mul<V>(z, sigmoid<V>(z)) : z;
}
// d = dy act'(z), with silu' = s (1 + z (1 - s))
template <int V>
__device__ __forceinline__ Cols<V> act_grad(const Cols<V>& z, const Cols<V>& dy, int act) {
  if (!act) return dy;
  const Cols<V> s = sigmoid<V>(z), one = all<V>(1.0f);
  return mul<V>(dy, mul<V>(s, fma<V>(z, fma<V>(s, all<V>(-1.0f), one), one)));
}
template <int V>
__device__ __forceinline__ Cols<V> centred(const Cols<V>& x, float mean) { return add<V>(x, all<V>(-mean)); }
template <int V>
__device__ __forceinline__ float total(const Cols<V>& c) {
  if constexpr (V == 1) {
    return c[0];
  } else {
    Cols<V / 2> lo, hi;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) lo[i] = c[i], hi[i] = c[i + V / 2];
    return total<V / 2>(add<V / 2>(lo, hi));
  }
}
template <int V>
__device__ __forceinline__ Cols<V> load_affine(const float* p, int c, float other) {
  Cols<V> o;
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = p ? __ldg(p + c + i) : other;
  return o;
}
// Sums of U values over the `team` consecutive threads that share a group; every thread gets them. SHUF: a
// power of two of at most 32 threads, which then lie in one warp.
template <int U, bool SHUF>
__device__ __forceinline__ void team_sum(float (&v)[U], int team, float* buf) {
  if constexpr (SHUF) {
    for (int o = team >> 1; o > 0; o >>= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] += __shfl_xor_sync(0xffffffffu, v[u], o);
  } else {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) buf[u * kThreads + threadIdx.x] = v[u];
    __syncthreads();
    const int first = threadIdx.x / team * team, most = blockDim.x - 1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float s = 0.0f;
      for (int i = 0; i < team; ++i) s += buf[u * kThreads + min(first + i, most)];
      v[u] = s;
    }
  }
}

// ---- one position per sample: thread (r, v) of a CTA has vector v of the CTA's channels in rows r, r + rp, ...; the
// rows of its next turn are requested before it works on those of this one

// The rows of a thread: turns of U rows each, row u of a turn if the turn's number is below most[u].
template <int U>
struct Turns {
  int most[U], count;
  long long row, turn, between;
  __device__ __forceinline__ Turns(const NormParams& p, int r, int rp) {
    between = rp;
    turn = (long long)rp * U * gridDim.y;
    const long long base = (long long)blockIdx.y * rp * U;
    row = base + r;
    count = base < p.N ? (int)((p.N - base + turn - 1) / turn) : 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long left = p.N - row - u * between;
      most[u] = r < rp && left > 0 ? (int)((left + turn - 1) / turn) : 0;  // (none beyond the last whole row of vectors)
    }
  }
};

template <typename T, int VE, bool SHUF>
__global__ void __launch_bounds__(kThreads, 3) norm_rows_fwd_kernel(const NormParams p) {
  constexpr int U = 2;
  __shared__ float buf[SHUF ? 1 : U * kThreads];
  const int team = p.Cg / VE, nv = min(p.gpb, p.G - (int)blockIdx.x * p.gpb) * team, rp = blockDim.x / nv;
  const int r = threadIdx.x / nv, v = threadIdx.x % nv;
  const int c = blockIdx.x * p.gpb * p.Cg + v * VE;
  const float inv = 1.0f / (float)p.Cg;
  const Cols<VE> w = load_affine<VE>(p.w, c, 1.0f), b = load_affine<VE>(p.b, c, 0.0f);
  const Turns<U> t(p, r, rp);
  const T* x = static_cast<const T*>(p.x) + t.row * p.C + c;
  T* y = static_cast<T*>(p.y) + t.row * p.C + c;
  const bool speaker = p.mean && v % team == 0;
  long long stat = t.row * p.G + c / p.Cg;
  const long long between = t.between * p.C, ahead = t.turn * p.C;
  Vec<T, VE> next[U];
#pragma unroll
  for (int u = 0; u < U; ++u) next[u] = load_if<T, VE>(t.most[u] > 0, x + u * between);
  for (int i = 0; i < t.count; ++i, y += ahead, stat += t.turn * p.G) {
    Cols<VE> a[U];
    float s[U], q[U];
    x += ahead;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      a[u] = widen<T, VE>(next[u]);
      next[u] = load_if<T, VE>(i + 1 < t.most[u], x + u * between);
      s[u] = total<VE>(a[u]);
    }
    team_sum<U, SHUF>(s, team, buf);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] *= inv;
      a[u] = centred<VE>(a[u], s[u]);
      q[u] = total<VE>(mul<VE>(a[u], a[u]));
    }
    team_sum<U, SHUF>(q, team, buf);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i < t.most[u]) {
        const float rstd = rsqrtf(fmaf(q[u], inv, p.eps));
        if (speaker) {
          p.mean[stat + u * t.between * p.G] = s[u];
          p.rstd[stat + u * t.between * p.G] = rstd;
        }
        a[u] = activate<VE>(fma<VE>(mul<VE>(a[u], all<VE>(rstd)), w, b), p.act);
        *reinterpret_cast<Vec<T, VE>*>(y + u * between) = narrow<T, VE>(a[u]);
      }
  }
}

template <typename T, int VE, bool SHUF>
__global__ void __launch_bounds__(kThreads, 2) norm_rows_bwd_kernel(const NormParams p) {
  constexpr int U = 2;
  __shared__ float buf[2 * U * kThreads];
  const int team = p.Cg / VE, nv = min(p.gpb, p.G - (int)blockIdx.x * p.gpb) * team, rp = blockDim.x / nv;
  const int r = threadIdx.x / nv, v = threadIdx.x % nv;
  const int c = blockIdx.x * p.gpb * p.Cg + v * VE;
  const float inv = 1.0f / (float)p.Cg;
  const Cols<VE> w = load_affine<VE>(p.w, c, 1.0f), b = load_affine<VE>(p.b, c, 0.0f);
  Cols<VE> dw = all<VE>(0.0f), db = all<VE>(0.0f);
  const Turns<U> t(p, r, rp);
  long long at = t.row * p.C + c, stat = t.row * p.G + c / p.Cg;
  const long long between = t.between * p.C, ahead = t.turn * p.C;
  Vec<T, VE> next_x[U], next_g[U];
  float next_mean[U], next_rstd[U];
  auto load = [&](int u, bool on) {
    next_x[u] = load_if<T, VE>(on, static_cast<const T*>(p.x) + at + u * between);
    next_g[u] = load_if<T, VE>(on, static_cast<const T*>(p.dy) + at + u * between);
    next_mean[u] = on ? __ldg(p.mean + stat + u * t.between * p.G) : 0.0f;
    next_rstd[u] = on ? __ldg(p.rstd + stat + u * t.between * p.G) : 0.0f;
  };
#pragma unroll
  for (int u = 0; u < U; ++u) load(u, t.most[u] > 0);
  for (int i = 0; i < t.count; ++i) {
    T* dx = static_cast<T*>(p.y) + at;
    Cols<VE> xh[U], g[U];
    float s[2 * U], rstd[U];
    at += ahead, stat += t.turn * p.G;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      rstd[u] = next_rstd[u];
      xh[u] = mul<VE>(centred<VE>(widen<T, VE>(next_x[u]), next_mean[u]), all<VE>(rstd[u]));
      g[u] = widen<T, VE>(next_g[u]);
      load(u, i + 1 < t.most[u]);
      const Cols<VE> d = act_grad<VE>(fma<VE>(xh[u], w, b), g[u], p.act);  // (0 in rows beyond the last)
      db = add<VE>(db, d);
      dw = fma<VE>(d, xh[u], dw);
      g[u] = mul<VE>(d, w);
      s[2 * u] = total<VE>(g[u]);
      s[2 * u + 1] = total<VE>(mul<VE>(g[u], xh[u]));
    }
    team_sum<2 * U, SHUF>(s, team, buf);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i < t.most[u] && p.y) {
        const Cols<VE> q = fma<VE>(xh[u], all<VE>(-s[2 * u + 1] * inv), centred<VE>(g[u], s[2 * u] * inv));
        *reinterpret_cast<Vec<T, VE>*>(dx + u * between) = narrow<T, VE>(mul<VE>(q, all<VE>(rstd[u])));
      }
  }
  if (!p.sums) return;
  // the CTA's rows r = 0 .. rp - 1 of accumulators, added in that order
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    __syncthreads();
    buf[threadIdx.x] = dw[i];
    buf[kThreads + threadIdx.x] = db[i];
    __syncthreads();
    if (r == 0) {
      float sw = 0.0f, sb = 0.0f;
      for (int k = 0; k < rp; ++k) sw += buf[k * nv + v], sb += buf[kThreads + k * nv + v];
      p.sums[((long long)blockIdx.y * 2) * p.C + c + i] = sw;
      p.sums[((long long)blockIdx.y * 2 + 1) * p.C + c + i] = sb;
    }
  }
}

// ---- several positions per sample: CTA = (slab of rows, channel block, sample)

struct Moments {
  float n, mean, m2;
};
// Both parts' values as one (Chan, Golub and LeVeque 1979). The weight comes first: beside an empty part d is a whole mean,
// whose square may overflow, and counts nothing.
__device__ __forceinline__ Moments join(Moments a, Moments b) {
  const float n = a.n + b.n, d = b.mean - a.mean, f = n > 0.0f ? __fdividef(b.n, n) : 0.0f;
  return {n, fmaf(d, f, a.mean), fmaf(a.n * f * d, d, a.m2 + b.m2)};
}
__device__ __forceinline__ Moments warp_join(Moments m) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    Moments q;
    q.n = __shfl_xor_sync(0xffffffffu, m.n, o);
    q.mean = __shfl_xor_sync(0xffffffffu, m.mean, o);
    q.m2 = __shfl_xor_sync(0xffffffffu, m.m2, o);
    // in lane order whichever side asks, so that all lanes get the same bits
    m = (threadIdx.x & o) ? join(q, m) : join(m, q);
  }
  return m;
}

// What a CTA of the slab layout works on.
template <int VE>
struct Slab {
  long long n, at;  // sample; this thread's first element
  int rows;         // rows of this thread: 0, rp, 2 rp, ... below this
  int c, nv, rp, r, v, groups, g0, team, slab, piece;  // groups g0 .. g0 + groups - 1, or one piece of group g0
  __device__ __forceinline__ Slab(const NormParams& p, int block) {
    slab = block % p.nslab;
    block /= p.nslab;
    const int cb = block % p.cblks;
    n = block / p.cblks;
    int width;
    if (p.pieces == 1) {
      piece = 0;
      g0 = cb * p.gpb;
      groups = min(p.gpb, p.G - g0);
      c = g0 * p.Cg;
      width = groups * p.Cg;
      team = p.Cg / VE;
    } else {
      piece = cb % p.pieces;
      g0 = cb / p.pieces;
      groups = 1;
      c = g0 * p.Cg + piece * kChannels;
      width = min(kChannels, p.Cg - piece * kChannels);
      team = width / VE;
    }
    nv = width / VE;
    rp = kThreads / nv;
    r = threadIdx.x / nv;
    v = threadIdx.x % nv;
    c += v * VE;
    const long long row0 = slab * p.slab_rows;
    rows = r < rp ? (int)(min(p.L - row0, p.slab_rows) - r) : 0;  // (none beyond the last whole row of threads)
    at = (n * p.L + row0 + r) * p.C + c;
  }
  // place of this CTA's partial result of its group i
  __device__ __forceinline__ long long part_at(const NormParams& p, int i) const {
    return ((n * p.G + g0 + i) * p.pieces + piece) * p.nslab + slab;
  }
};

template <typename T, int VE>
__global__ void __launch_bounds__(kThreads, 4) norm_stats_kernel(const NormParams p) {
  constexpr int U = 4;
  __shared__ Moments buf[kThreads];
  grid_dependents_may_launch();
  const Slab<VE> s(p, blockIdx.x);
  const T* x = static_cast<const T*>(p.x) + s.at;
  const long long step = (long long)s.rp * p.C;
  Moments m = {0.0f, 0.0f, 0.0f};
  Vec<T, VE> next[U];
#pragma unroll
  for (int u = 0; u < U; ++u) next[u] = load_if<T, VE>(u * s.rp < s.rows, x + u * step);
  for (int row = 0; row < s.rows;) {
    Vec<T, VE> a[U];
    int k = 0;  // rows of this turn
#pragma unroll
    for (int u = 0; u < U; ++u) {
      a[u] = next[u];
      k += row + u * s.rp < s.rows;
    }
    row += s.rp * U, x += U * step;
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = load_if<T, VE>(row + u * s.rp < s.rows, x + u * step);
    Cols<VE> sum = widen<T, VE>(a[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) sum = add<VE>(sum, widen<T, VE>(a[u]));
    Moments q;
    q.n = (float)(k * VE);
    q.mean = __fdividef(total<VE>(sum), q.n);
    Cols<VE> sq = all<VE>(0.0f);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Cols<VE> d = u < k ? centred<VE>(widen<T, VE>(a[u]), q.mean) : all<VE>(0.0f);
      sq = fma<VE>(d, d, sq);
    }
    q.m2 = total<VE>(sq);
    m = join(m, q);
  }
  buf[threadIdx.x] = m;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < s.groups; i += kThreads / 32) {
    m = {0.0f, 0.0f, 0.0f};
    for (int k = lane; k < s.team * s.rp; k += 32) m = join(m, buf[k / s.team * s.nv + i * s.team + k % s.team]);
    m = warp_join(m);
    if (lane == 0) {
      float* o = p.part + 3 * s.part_at(p, i);
      o[0] = m.n, o[1] = m.mean, o[2] = m.m2;
    }
  }
}

template <typename T, int VE>
__global__ void __launch_bounds__(kThreads, 4) norm_apply_kernel(const NormParams p) {
  constexpr int U = 2;
  __shared__ float s_mean[kChannels], s_rstd[kChannels];
  const Slab<VE> s(p, gridDim.x - 1 - blockIdx.x);
  const Cols<VE> w = load_affine<VE>(p.w, s.c, 1.0f), b = load_affine<VE>(p.b, s.c, 0.0f);
  const int gi = s.v / s.team;
  const T* x = static_cast<const T*>(p.x) + s.at;
  const long long step = (long long)s.rp * p.C;
  Vec<T, VE> next[U];
#pragma unroll
  for (int u = 0; u < U; ++u) next[u] = load_if<T, VE>(u * s.rp < s.rows, x + u * step);
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, parts = p.pieces * p.nslab;
  for (int i = threadIdx.x >> 5; i < s.groups; i += kThreads / 32) {
    const long long at = s.n * p.G + s.g0 + i;
    const float* q = p.part + 3 * at * parts;
    Moments m = {0.0f, 0.0f, 0.0f};
    for (int k = lane; k < parts; k += 32) m = join(m, Moments{q[3 * k], q[3 * k + 1], q[3 * k + 2]});
    m = warp_join(m);
    if (lane == 0) {
      s_mean[i] = m.mean;
      s_rstd[i] = rsqrtf(m.m2 / m.n + p.eps);
      if (p.mean && s.slab == 0) p.mean[at] = s_mean[i], p.rstd[at] = s_rstd[i];  // (pieces write the same)
    }
  }
  __syncthreads();
  const float mean = s_mean[gi], rstd = s_rstd[gi];
  T* y = static_cast<T*>(p.y) + s.at;
  for (int row = 0; row < s.rows; row += s.rp * U, y += U * step) {
    Vec<T, VE> a[U];
    x += U * step;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      a[u] = next[u];
      next[u] = load_if<T, VE>(row + (U + u) * s.rp < s.rows, x + u * step);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * s.rp < s.rows)
        *reinterpret_cast<Vec<T, VE>*>(y + u * step) = narrow<T, VE>(activate<VE>(
            fma<VE>(mul<VE>(centred<VE>(widen<T, VE>(a[u]), mean), all<VE>(rstd)), w, b), p.act));
  }
}

// Per channel and slab the sums of d xh and d (dw, db), and per group and slab those of g and g xh.
template <typename T, int VE>
__global__ void __launch_bounds__(kThreads, 3) norm_bwd_sums_kernel(const NormParams p) {
  __shared__ float buf[2 * kThreads];
  grid_dependents_may_launch();
  const Slab<VE> s(p, blockIdx.x);
  const long long at = s.n * p.G + s.g0 + s.v / s.team;
  const float mean = __ldg(p.mean + at), rstd = __ldg(p.rstd + at);
  const Cols<VE> w = load_affine<VE>(p.w, s.c, 1.0f), b = load_affine<VE>(p.b, s.c, 0.0f);
  Cols<VE> dw = all<VE>(0.0f), db = all<VE>(0.0f);
  const T* x = static_cast<const T*>(p.x) + s.at;
  const T* dy = static_cast<const T*>(p.dy) + s.at;
  const long long step = (long long)s.rp * p.C;
  Vec<T, VE> next_x = load_if<T, VE>(s.rows > 0, x), next_g = load_if<T, VE>(s.rows > 0, dy);
  for (int row = 0; row < s.rows; row += s.rp) {
    const Cols<VE> xh = mul<VE>(centred<VE>(widen<T, VE>(next_x), mean), all<VE>(rstd)), g = widen<T, VE>(next_g);
    x += step, dy += step;
    next_x = load_if<T, VE>(row + s.rp < s.rows, x);
    next_g = load_if<T, VE>(row + s.rp < s.rows, dy);
    const Cols<VE> d = act_grad<VE>(fma<VE>(xh, w, b), g, p.act);
    db = add<VE>(db, d);
    dw = fma<VE>(d, xh, dw);
  }
  float s1 = 0.0f, s2 = 0.0f;
  float* out = p.sums + ((s.n * p.nslab + s.slab) * 2) * p.C + s.c;
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    __syncthreads();
    buf[threadIdx.x] = dw[i];
    buf[kThreads + threadIdx.x] = db[i];
    __syncthreads();
    if (s.r == 0) {
      float sw = 0.0f, sb = 0.0f;
      for (int k = 0; k < s.rp; ++k) sw += buf[k * s.nv + s.v], sb += buf[kThreads + k * s.nv + s.v];
      out[i] = sw;
      out[p.C + i] = sb;
      s1 = fmaf(sb, w[i], s1);
      s2 = fmaf(sw, w[i], s2);
    }
  }
  __syncthreads();
  buf[threadIdx.x] = s1;
  buf[kThreads + threadIdx.x] = s2;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < s.groups; i += kThreads / 32) {
    s1 = s2 = 0.0f;
    for (int k = lane; k < s.team; k += 32) s1 += buf[i * s.team + k], s2 += buf[kThreads + i * s.team + k];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s1 += __shfl_xor_sync(0xffffffffu, s1, o);
      s2 += __shfl_xor_sync(0xffffffffu, s2, o);
    }
    if (lane == 0) {
      float* q = p.part + 2 * s.part_at(p, i);
      q[0] = s1, q[1] = s2;
    }
  }
}

// dw or db from the rows of sums [parts][2][C], in 64 bits and a fixed order: CTA `block` has 32 channels of one of them,
// thread (i, j) rows i, i + 8, ... of channel j.
__device__ __forceinline__ void param_sums(const NormParams& p, int block) {
  __shared__ double acc[kThreads / 32][33];
  const int j = threadIdx.x & 31, i = threadIdx.x >> 5, which = block & 1;
  const int c = (block >> 1) * 32 + j;
  float* out = which ? p.db : p.dw;
  if (!out) return;
  double sum = 0.0;
  if (c < p.C) {
#pragma unroll 8
    for (long long r = i; r < p.parts; r += kThreads / 32) sum += (double)__ldcg(p.sums + (2 * r + which) * p.C + c);
  }
  acc[i][j] = sum;
  __syncthreads();
  if (i == 0 && c < p.C) {
    for (int k = 1; k < kThreads / 32; ++k) sum += acc[k][j];
    out[c] = (float)sum;
  }
}
inline int param_blocks(int C) { return (C + 31) / 32 * 2; }

// dx; the CTAs beyond `slabs` add up the parameters' gradients beside it
template <typename T, int VE>
__global__ void __launch_bounds__(kThreads, 3) norm_bwd_apply_kernel(const NormParams p, int slabs) {
  __shared__ float s_m1[kChannels], s_m2[kChannels];
  if ((int)blockIdx.x >= slabs) {
    grid_dependency_wait();
    param_sums(p, blockIdx.x - slabs);
    return;
  }
  const Slab<VE> s(p, slabs - 1 - blockIdx.x);
  const Cols<VE> w = load_affine<VE>(p.w, s.c, 1.0f), b = load_affine<VE>(p.b, s.c, 0.0f);
  const int gi = s.v / s.team;
  const float mean = __ldg(p.mean + s.n * p.G + s.g0 + gi), rstd = __ldg(p.rstd + s.n * p.G + s.g0 + gi);
  const T* x = static_cast<const T*>(p.x) + s.at;
  const T* dy = static_cast<const T*>(p.dy) + s.at;
  const long long step = (long long)s.rp * p.C;
  Vec<T, VE> next_x = load_if<T, VE>(s.rows > 0, x), next_g = load_if<T, VE>(s.rows > 0, dy);
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, parts = p.pieces * p.nslab;
  const float inv = 1.0f / ((float)p.Cg * (float)p.L);
  for (int i = threadIdx.x >> 5; i < s.groups; i += kThreads / 32) {
    const float* q = p.part + 2 * (s.n * p.G + s.g0 + i) * parts;
    float s1 = 0.0f, s2 = 0.0f;
    for (int k = lane; k < parts; k += 32) s1 += q[2 * k], s2 += q[2 * k + 1];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s1 += __shfl_xor_sync(0xffffffffu, s1, o);
      s2 += __shfl_xor_sync(0xffffffffu, s2, o);
    }
    if (lane == 0) s_m1[i] = s1 * inv, s_m2[i] = s2 * inv;
  }
  __syncthreads();
  const float m1 = s_m1[gi], m2 = s_m2[gi];
  T* dx = static_cast<T*>(p.y) + s.at;
  for (int row = 0; row < s.rows; row += s.rp, dx += step) {
    const Cols<VE> xh = mul<VE>(centred<VE>(widen<T, VE>(next_x), mean), all<VE>(rstd)), g = widen<T, VE>(next_g);
    x += step, dy += step;
    next_x = load_if<T, VE>(row + s.rp < s.rows, x);
    next_g = load_if<T, VE>(row + s.rp < s.rows, dy);
    const Cols<VE> gg = mul<VE>(act_grad<VE>(fma<VE>(xh, w, b), g, p.act), w);
    *reinterpret_cast<Vec<T, VE>*>(dx) = narrow<T, VE>(mul<VE>(fma<VE>(xh, all<VE>(-m2), centred<VE>(gg, m1)), all<VE>(rstd)));
  }
}

// dw and db alone (rows, or no dx wanted)
__global__ void __launch_bounds__(kThreads) norm_param_kernel(const NormParams p) {
  grid_dependency_wait();
  param_sums(p, blockIdx.x);
}

// ------------------------------------------------------------------------------------------ host

bool ok_dtype(int d) { return d == NSB_F32 || d == NSB_BF16 || d == NSB_F16; }
bool fits(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

constexpr int kPlanSms = 148;  // (the buffers' sizes must not depend on the device that asks)

// One position per sample and a group that fits a CTA's threads whatever the vector: a row layout. (Wider groups: see above.)
bool by_rows(long long L, int Cg) { return L == 1 && Cg <= kThreads; }

void plan_slabs(NormParams& p, bool backward) {
  p.gpb = std::min(p.G, std::max(1, kChannels / p.Cg));
  p.pieces = (p.Cg + kChannels - 1) / kChannels;
  p.cblks = p.pieces > 1 ? p.G * p.pieces : (p.G + p.gpb - 1) / p.gpb;
  if (p.pieces == 1) p.gpb = (p.G + p.cblks - 1) / p.cblks;  // blocks of equal width
  // as many CTAs as are resident at once, not one more (608 for 592 places took a second round: 20 us where
  // one takes 13), but no slab under 32 rows: a slab costs two reductions over the CTA
  const long long blocks = p.N * p.cblks, most = (p.L + 31) / 32;
  p.nslab = (int)std::max<long long>(1, std::min<long long>((backward ? 3LL : 4LL) * kPlanSms / blocks, most));
  p.slab_rows = (p.L + p.nslab - 1) / p.nslab;
  p.nslab = (int)((p.L + p.slab_rows - 1) / p.slab_rows);
}
// Row chunks of the row layout's backward, each with a row of parameter sums.
int row_chunks(long long N) { return (int)std::max<long long>(1, std::min<long long>((N + 7) / 8, 4LL * kPlanSms)); }

int check_sizes(int64_t N, int64_t L, int64_t C, int64_t G, int act, int dtype) {
  if (N < 0 || L < 0 || C < 0 || G < 1 || C % G || (act != NSB_ACT_NONE && act != NSB_ACT_SILU) || !ok_dtype(dtype))
    return NSB_ERR_INVALID_ARG;
  if (C > (1 << 24)) return NSB_ERR_TOO_LARGE;
  return NSB_OK;
}
NormParams make(int64_t N, int64_t L, int64_t C, int64_t G, bool backward) {
  NormParams p = {};
  p.N = N, p.L = L, p.C = (int)C, p.G = (int)G, p.Cg = (int)(C / G);
  plan_slabs(p, backward);
  return p;
}

template <typename T, int VE>
int launch_norm(NormParams p, bool backward, cudaStream_t st) {
  const bool params = p.dw || p.db;
  if (by_rows(p.L, p.Cg)) {
    const int team = p.Cg / VE;
    p.gpb = std::min(p.G, kThreads / team);
    const unsigned cb = (unsigned)((p.G + p.gpb - 1) / p.gpb);
    p.gpb = (p.G + (int)cb - 1) / (int)cb;
    const int rp = kThreads / (p.gpb * team);
    const unsigned threads = (unsigned)((rp * p.gpb * team + 31) / 32 * 32);  // whole rows of vectors
    const bool shuf = team <= 32 && (team & (team - 1)) == 0;
    // forward: as many CTAs as 80 registers a thread let be resident
    const int resident = kPlanSms * (65536 / (80 * (int)threads));
    const dim3 grid(cb, backward ? (unsigned)(p.parts = row_chunks(p.N))
                                 : (unsigned)std::max<long long>(1, std::min<long long>((p.N + 2 * rp - 1) / (2 * rp), resident / (int)cb)));
    if (backward && shuf) norm_rows_bwd_kernel<T, VE, true><<<grid, threads, 0, st>>>(p);
    else if (backward) norm_rows_bwd_kernel<T, VE, false><<<grid, threads, 0, st>>>(p);
    else if (shuf) norm_rows_fwd_kernel<T, VE, true><<<grid, threads, 0, st>>>(p);
    else norm_rows_fwd_kernel<T, VE, false><<<grid, threads, 0, st>>>(p);
    NSB_CUDA_TRY(cudaGetLastError(), "launch norm_rows kernel");
  } else {
    const long long slabs = p.N * p.cblks * p.nslab, grid = slabs + (backward && params ? param_blocks(p.C) : 0);
    if (grid > 0x7fffffffLL) return NSB_ERR_TOO_LARGE;
    p.parts = p.N * p.nslab;
    const dim3 g((unsigned)slabs);
    if (!backward) {
      norm_stats_kernel<T, VE><<<g, kThreads, 0, st>>>(p);
      NSB_CUDA_TRY(cudaGetLastError(), "launch norm_stats_kernel");
      NSB_CUDA_TRY(launch_dependent(norm_apply_kernel<T, VE>, g, dim3(kThreads), 0, st, p), "launch norm_apply_kernel");
      return NSB_OK;
    }
    norm_bwd_sums_kernel<T, VE><<<g, kThreads, 0, st>>>(p);
    NSB_CUDA_TRY(cudaGetLastError(), "launch norm_bwd_sums_kernel");
    if (p.y) {
      NSB_CUDA_TRY(launch_dependent(norm_bwd_apply_kernel<T, VE>, dim3((unsigned)grid), dim3(kThreads), 0, st, p, (int)slabs),
                   "launch norm_bwd_apply_kernel");
      return NSB_OK;
    }
  }
  if (backward && params)
    NSB_CUDA_TRY(launch_dependent(norm_param_kernel, dim3((unsigned)param_blocks(p.C)), dim3(kThreads), 0, st, p), "launch norm_param_kernel");
  return NSB_OK;
}
template <typename T>
int go(const NormParams& p, bool backward, cudaStream_t st) {
  DeviceInfo dev;
  const int r = get_device_info(&dev);
  if (r != NSB_OK) return r;
  // A thread's vector lies in one group, and in one piece of 256 channels of a group.
  auto ok = [&](int ve) {
    return p.Cg % ve == 0 && fits(p.x, sizeof(T) * ve) && fits(p.y, sizeof(T) * ve) && fits(p.dy, sizeof(T) * ve);
  };
  if constexpr (sizeof(T) == 2)
    if (ok(8)) return launch_norm<T, 8>(p, backward, st);
  if (ok(4)) return launch_norm<T, 4>(p, backward, st);
  return launch_norm<T, 1>(p, backward, st);
}
int dispatch(const NormParams& p, int dtype, bool backward, cudaStream_t st) {
  switch (dtype) {
    case NSB_F32: return go<float>(p, backward, st);
    case NSB_BF16: return go<__nv_bfloat16>(p, backward, st);
    default: return go<__half>(p, backward, st);
  }
}

}  // namespace
}  // namespace nsb

using namespace nsb;

extern "C" int64_t nsb_group_norm_scratch_floats(int64_t N, int64_t L, int64_t C, int64_t G, int backward) {
  if (check_sizes(N, L, C, G, 0, NSB_F32) != NSB_OK || N * L * C == 0) return 0;
  const NormParams p = make(N, L, C, G, backward != 0);
  if (by_rows(p.L, p.Cg)) return backward ? 2LL * row_chunks(N) * C : 0;
  const long long groups = N * G * p.pieces * p.nslab;
  return backward ? 2 * groups + 2 * N * p.nslab * C : 3 * groups;
}

extern "C" int nsb_group_norm_fwd(const void* x, const float* weight, const float* bias, void* y, float* mean, float* rstd,
                                  float* scratch, int64_t N, int64_t L, int64_t C, int64_t G, float eps, int activation,
                                  int dtype, void* stream) {
  int r = check_sizes(N, L, C, G, activation, dtype);
  if (r != NSB_OK) return r;
  if (N * L * C == 0) return NSB_OK;
  const size_t es = dtype_size(dtype);
  if (!x || !y || !fits(x, es) || !fits(y, es) || !mean != !rstd) return NSB_ERR_INVALID_ARG;
  for (const void* q : {weight, bias, (const float*)mean, (const float*)rstd, (const float*)scratch})
    if (!fits(q, 4)) return NSB_ERR_INVALID_ARG;
  NormParams p = make(N, L, C, G, false);
  if (!by_rows(L, p.Cg) && !scratch) return NSB_ERR_INVALID_ARG;
  p.x = x, p.w = weight, p.b = bias, p.y = y, p.mean = mean, p.rstd = rstd, p.part = scratch, p.eps = eps;
  p.act = activation;
  return dispatch(p, dtype, false, static_cast<cudaStream_t>(stream));
}

extern "C" int nsb_group_norm_bwd(const void* dy, const void* x, const float* weight, const float* bias, const float* mean,
                                  const float* rstd, void* dx, float* dweight, float* dbias, float* scratch, int64_t N,
                                  int64_t L, int64_t C, int64_t G, int activation, int dtype, void* stream) {
  int r = check_sizes(N, L, C, G, activation, dtype);
  if (r != NSB_OK) return r;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (const void* q : {weight, bias, mean, rstd, (const float*)dweight, (const float*)dbias, (const float*)scratch})
    if (!fits(q, 4)) return NSB_ERR_INVALID_ARG;
  if (N * L * C == 0) {
    if (dweight && C) NSB_CUDA_TRY(cudaMemsetAsync(dweight, 0, (size_t)C * 4, st), "memset dweight");
    if (dbias && C) NSB_CUDA_TRY(cudaMemsetAsync(dbias, 0, (size_t)C * 4, st), "memset dbias");
    return NSB_OK;
  }
  const size_t es = dtype_size(dtype);
  if (!dy || !x || !mean || !rstd || !scratch || !fits(x, es) || !fits(dy, es) || !fits(dx, es)) return NSB_ERR_INVALID_ARG;
  if (!dx && !dweight && !dbias) return NSB_OK;
  NormParams p = make(N, L, C, G, true);
  p.x = x, p.dy = dy, p.w = weight, p.b = bias, p.y = dx, p.act = activation;
  p.mean = const_cast<float*>(mean), p.rstd = const_cast<float*>(rstd);
  p.sums = scratch;
  if (!by_rows(L, p.Cg)) p.part = scratch + 2 * N * p.nslab * C;
  else if (!dweight && !dbias) p.sums = nullptr;
  p.dw = dweight, p.db = dbias;
  return dispatch(p, dtype, true, st);
}
