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
// ones are joined by Chan, Golub and LeVeque's formula. All sums are fp32, those over N in 64 bits.
#include <algorithm>

#include "nsb_common.cuh"

namespace nsb {
namespace {

constexpr int kThreads = 256, kChannels = 256;  // channels of a CTA in the slab layout
constexpr int kRowUnroll = 4;                   // rows of a thread that are in flight together

struct NormParams {
  const void *x, *dy;
  const float *w, *b;
  void* y;
  float *mean, *rstd, *part, *sums;  // part: per group and slab; sums: per channel and slab (dw, db)
  long long N, L;
  int C, G, Cg, act;
  float eps;
  int gpb, pieces, cblks, nslab;  // groups of a channel block, pieces of a group, channel blocks, slabs of rows
  long long slab_rows;
};

__device__ __forceinline__ float sigmoid_f(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }
__device__ __forceinline__ float activate(float z, int act) {
  // for z below -88 the exponential overflows and the quotient is 0, as the limit is
  return act ? z * sigmoid_f(z) : z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
  if (!act) return 1.0f;
  const float s = sigmoid_f(z);
  return s * fmaf(z, 1.0f - s, 1.0f);
}

template <typename T, int VE>
__device__ __forceinline__ void load_f32(const T* p, float (&o)[VE]) {
  const Vec<T, VE> v = *reinterpret_cast<const Vec<T, VE>*>(p);
#pragma unroll
  for (int i = 0; i < VE; ++i) o[i] = Elem<T>::to_f32(v.v[i]);
}
template <typename T, int VE>
__device__ __forceinline__ void store_f32(T* p, const float (&o)[VE]) {
  Vec<T, VE> v;
#pragma unroll
  for (int i = 0; i < VE; ++i) v.v[i] = Elem<T>::from_f32(o[i]);
  *reinterpret_cast<Vec<T, VE>*>(p) = v;
}
template <int VE>
__device__ __forceinline__ void load_affine(const float* p, int c, float other, float (&o)[VE]) {
#pragma unroll
  for (int i = 0; i < VE; ++i) o[i] = p ? p[c + i] : other;
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
    const int first = threadIdx.x / team * team;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float s = 0.0f;
      for (int i = 0; i < team; ++i) s += buf[u * kThreads + min(first + i, kThreads - 1)];
      v[u] = s;
    }
  }
}

// ---- one position per sample: thread (r, v) of a CTA has vector v of the CTA's channels in rows r, r + rp, ...

template <typename T, int VE, bool SHUF>
__global__ void __launch_bounds__(kThreads) norm_rows_fwd_kernel(const NormParams p) {
  constexpr int U = kRowUnroll;
  __shared__ float buf[SHUF ? 1 : U * kThreads];
  const int team = p.Cg / VE, nv = min(p.gpb, p.G - (int)blockIdx.x * p.gpb) * team, rp = kThreads / nv;
  const int r = threadIdx.x / nv, v = threadIdx.x % nv;
  const int c = blockIdx.x * p.gpb * p.Cg + v * VE, grp = c / p.Cg;
  const float inv = 1.0f / (float)p.Cg;
  float w[VE], b[VE];
  load_affine<VE>(p.w, c, 1.0f, w);
  load_affine<VE>(p.b, c, 0.0f, b);
  const T* x = static_cast<const T*>(p.x);
  T* y = static_cast<T*>(p.y);
  const long long step = (long long)rp * U * gridDim.y;
  for (long long base = (long long)blockIdx.y * rp * U; base < p.N; base += step) {
    float a[U][VE], s[U], q[U];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long n = base + u * rp + r;
      on[u] = r < rp && n < p.N;
      if (on[u]) load_f32<T, VE>(x + n * p.C + c, a[u]);
      else
#pragma unroll
        for (int i = 0; i < VE; ++i) a[u][i] = 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] = 0.0f;
#pragma unroll
      for (int i = 0; i < VE; ++i) s[u] += a[u][i];
    }
    team_sum<U, SHUF>(s, team, buf);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[u] *= inv;
      q[u] = 0.0f;
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        a[u][i] -= s[u];
        q[u] = fmaf(a[u][i], a[u][i], q[u]);
      }
    }
    team_sum<U, SHUF>(q, team, buf);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!on[u]) continue;
      const long long n = base + u * rp + r;
      const float rstd = rsqrtf(fmaf(q[u], inv, p.eps));
      if (p.mean && v % team == 0) {
        p.mean[n * p.G + grp] = s[u];
        p.rstd[n * p.G + grp] = rstd;
      }
#pragma unroll
      for (int i = 0; i < VE; ++i) a[u][i] = activate(fmaf(a[u][i] * rstd, w[i], b[i]), p.act);
      store_f32<T, VE>(y + n * p.C + c, a[u]);
    }
  }
}

template <typename T, int VE, bool SHUF>
__global__ void __launch_bounds__(kThreads) norm_rows_bwd_kernel(const NormParams p) {
  constexpr int U = 2;
  __shared__ float buf[2 * U * kThreads];
  const int team = p.Cg / VE, nv = min(p.gpb, p.G - (int)blockIdx.x * p.gpb) * team, rp = kThreads / nv;
  const int r = threadIdx.x / nv, v = threadIdx.x % nv;
  const int c = blockIdx.x * p.gpb * p.Cg + v * VE, grp = c / p.Cg;
  const float inv = 1.0f / (float)p.Cg;
  float w[VE], b[VE], dw[VE], db[VE];
  load_affine<VE>(p.w, c, 1.0f, w);
  load_affine<VE>(p.b, c, 0.0f, b);
#pragma unroll
  for (int i = 0; i < VE; ++i) dw[i] = db[i] = 0.0f;
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.dy);
  T* dx = static_cast<T*>(p.y);
  const long long step = (long long)rp * U * gridDim.y;
  for (long long base = (long long)blockIdx.y * rp * U; base < p.N; base += step) {
    float xh[U][VE], g[U][VE], s[2 * U], rstd[U];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long n = base + u * rp + r;
      on[u] = r < rp && n < p.N;
      rstd[u] = 0.0f;
      if (on[u]) {
        load_f32<T, VE>(x + n * p.C + c, xh[u]);
        load_f32<T, VE>(dy + n * p.C + c, g[u]);
        const float mean = p.mean[n * p.G + grp];
        rstd[u] = p.rstd[n * p.G + grp];
#pragma unroll
        for (int i = 0; i < VE; ++i) xh[u][i] = (xh[u][i] - mean) * rstd[u];
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) xh[u][i] = g[u][i] = 0.0f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s[2 * u] = s[2 * u + 1] = 0.0f;
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const float d = g[u][i] * act_slope(fmaf(xh[u][i], w[i], b[i]), p.act);
        db[i] += d;
        dw[i] = fmaf(d, xh[u][i], dw[i]);
        g[u][i] = d * w[i];
        s[2 * u] += g[u][i];
        s[2 * u + 1] = fmaf(g[u][i], xh[u][i], s[2 * u + 1]);
      }
    }
    team_sum<2 * U, SHUF>(s, team, buf);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!on[u] || !dx) continue;
      const float m1 = s[2 * u] * inv, m2 = s[2 * u + 1] * inv;
#pragma unroll
      for (int i = 0; i < VE; ++i) g[u][i] = rstd[u] * (g[u][i] - m1 - xh[u][i] * m2);
      store_f32<T, VE>(dx + (base + u * rp + r) * p.C + c, g[u]);
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
// Both parts' values as one (Chan, Golub and LeVeque 1979)
__device__ __forceinline__ Moments join(Moments a, Moments b) {
  const float n = a.n + b.n, d = b.mean - a.mean, f = n > 0.0f ? b.n / n : 0.0f;
  return {n, fmaf(d, f, a.mean), a.m2 + b.m2 + d * d * a.n * f};
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
  long long n, row0, row1;
  int c, nv, rp, r, v, groups, g0, team;  // groups g0 .. g0 + groups - 1, or one piece of group g0
  __device__ __forceinline__ Slab(const NormParams& p, long long block) {
    const int slab = (int)(block % p.nslab);
    const int cb = (int)(block / p.nslab % p.cblks);
    n = block / p.nslab / p.cblks;
    row0 = slab * p.slab_rows;
    row1 = min(p.L, row0 + p.slab_rows);
    int width;
    if (p.pieces == 1) {
      g0 = cb * p.gpb;
      groups = min(p.gpb, p.G - g0);
      c = g0 * p.Cg;
      width = groups * p.Cg;
      team = p.Cg / VE;
    } else {
      g0 = cb / p.pieces;
      groups = 1;
      const int at = cb % p.pieces * kChannels;
      c = g0 * p.Cg + at;
      width = min(kChannels, p.Cg - at);
      team = width / VE;
    }
    nv = width / VE;
    rp = kThreads / nv;
    r = threadIdx.x / nv;
    v = threadIdx.x % nv;
    c += v * VE;
    if (r >= rp) row1 = row0;  // (threads beyond the last whole row)
  }
  // place of this CTA's partial result of its group i
  __device__ __forceinline__ long long part_at(const NormParams& p, long long block, int i) const {
    const int slab = (int)(block % p.nslab), cb = (int)(block / p.nslab % p.cblks);
    return ((n * p.G + g0 + i) * p.pieces + (p.pieces == 1 ? 0 : cb % p.pieces)) * p.nslab + slab;
  }
};

template <typename T, int VE>
__global__ void __launch_bounds__(kThreads) norm_stats_kernel(const NormParams p) {
  constexpr int U = kRowUnroll;
  __shared__ Moments buf[kThreads];
  grid_dependents_may_launch();
  const Slab<VE> s(p, blockIdx.x);
  const T* x = static_cast<const T*>(p.x) + s.n * p.L * p.C + s.c;
  Moments m = {0.0f, 0.0f, 0.0f};
  for (long long row = s.row0 + s.r; row < s.row1; row += s.rp * U) {
    float a[U][VE];
    Moments q = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * s.rp < s.row1) load_f32<T, VE>(x + (row + u * s.rp) * p.C, a[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * s.rp < s.row1) {
        q.n += VE;
#pragma unroll
        for (int i = 0; i < VE; ++i) q.mean += a[u][i];
      }
    q.mean = __fdividef(q.mean, q.n);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * s.rp < s.row1)
#pragma unroll
        for (int i = 0; i < VE; ++i) q.m2 = fmaf(a[u][i] - q.mean, a[u][i] - q.mean, q.m2);
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
      float* o = p.part + 3 * s.part_at(p, blockIdx.x, i);
      o[0] = m.n, o[1] = m.mean, o[2] = m.m2;
    }
  }
}

template <typename T, int VE>
__global__ void __launch_bounds__(kThreads) norm_apply_kernel(const NormParams p) {
  constexpr int U = kRowUnroll;
  __shared__ float s_mean[kChannels], s_rstd[kChannels];
  grid_dependency_wait();
  const long long block = gridDim.x - 1 - blockIdx.x;
  const Slab<VE> s(p, block);
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
      if (p.mean && block % p.nslab == 0) p.mean[at] = s_mean[i], p.rstd[at] = s_rstd[i];  // (pieces write the same)
    }
  }
  __syncthreads();
  const int gi = s.v / s.team;
  const float mean = s_mean[gi], rstd = s_rstd[gi];
  float w[VE], b[VE];
  load_affine<VE>(p.w, s.c, 1.0f, w);
  load_affine<VE>(p.b, s.c, 0.0f, b);
  const T* x = static_cast<const T*>(p.x) + s.n * p.L * p.C + s.c;
  T* y = static_cast<T*>(p.y) + s.n * p.L * p.C + s.c;
  for (long long row = s.row0 + s.r; row < s.row1; row += s.rp * U) {
    float a[U][VE];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * s.rp < s.row1) load_f32<T, VE>(x + (row + u * s.rp) * p.C, a[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * s.rp < s.row1) {
#pragma unroll
        for (int i = 0; i < VE; ++i) a[u][i] = activate(fmaf((a[u][i] - mean) * rstd, w[i], b[i]), p.act);
        store_f32<T, VE>(y + (row + u * s.rp) * p.C, a[u]);
      }
  }
}

// Per channel and slab the sums of d xh and d (dw, db), and per group and slab those of g and g xh.
template <typename T, int VE>
__global__ void __launch_bounds__(kThreads) norm_bwd_sums_kernel(const NormParams p) {
  constexpr int U = 2;
  __shared__ float buf[2 * kThreads];
  grid_dependents_may_launch();
  const Slab<VE> s(p, blockIdx.x);
  const long long at = s.n * p.G + s.g0 + s.v / s.team;
  const float mean = p.mean[at], rstd = p.rstd[at];
  float w[VE], b[VE], dw[VE], db[VE];
  load_affine<VE>(p.w, s.c, 1.0f, w);
  load_affine<VE>(p.b, s.c, 0.0f, b);
#pragma unroll
  for (int i = 0; i < VE; ++i) dw[i] = db[i] = 0.0f;
  const T* x = static_cast<const T*>(p.x) + s.n * p.L * p.C + s.c;
  const T* dy = static_cast<const T*>(p.dy) + s.n * p.L * p.C + s.c;
  for (long long row = s.row0 + s.r; row < s.row1; row += s.rp * U) {
    float a[U][VE], g[U][VE];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * s.rp < s.row1) {
        load_f32<T, VE>(x + (row + u * s.rp) * p.C, a[u]);
        load_f32<T, VE>(dy + (row + u * s.rp) * p.C, g[u]);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * s.rp < s.row1)
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const float xh = (a[u][i] - mean) * rstd, d = g[u][i] * act_slope(fmaf(xh, w[i], b[i]), p.act);
          db[i] += d;
          dw[i] = fmaf(d, xh, dw[i]);
        }
  }
  float s1 = 0.0f, s2 = 0.0f;
  float* out = p.sums + ((s.n * p.nslab + blockIdx.x % p.nslab) * 2) * p.C + s.c;
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
      float* q = p.part + 2 * s.part_at(p, blockIdx.x, i);
      q[0] = s1, q[1] = s2;
    }
  }
}

template <typename T, int VE>
__global__ void __launch_bounds__(kThreads) norm_bwd_apply_kernel(const NormParams p) {
  constexpr int U = 2;
  __shared__ float s_m1[kChannels], s_m2[kChannels];
  grid_dependents_may_launch();
  grid_dependency_wait();
  const long long block = gridDim.x - 1 - blockIdx.x;
  const Slab<VE> s(p, block);
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
  const int gi = s.v / s.team;
  const long long at = s.n * p.G + s.g0 + gi;
  const float mean = p.mean[at], rstd = p.rstd[at], m1 = s_m1[gi], m2 = s_m2[gi];
  float w[VE], b[VE];
  load_affine<VE>(p.w, s.c, 1.0f, w);
  load_affine<VE>(p.b, s.c, 0.0f, b);
  const T* x = static_cast<const T*>(p.x) + s.n * p.L * p.C + s.c;
  const T* dy = static_cast<const T*>(p.dy) + s.n * p.L * p.C + s.c;
  T* dx = static_cast<T*>(p.y) + s.n * p.L * p.C + s.c;
  for (long long row = s.row0 + s.r; row < s.row1; row += s.rp * U) {
    float a[U][VE], g[U][VE];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * s.rp < s.row1) {
        load_f32<T, VE>(x + (row + u * s.rp) * p.C, a[u]);
        load_f32<T, VE>(dy + (row + u * s.rp) * p.C, g[u]);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (row + u * s.rp < s.row1) {
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const float xh = (a[u][i] - mean) * rstd;
          const float gg = g[u][i] * act_slope(fmaf(xh, w[i], b[i]), p.act) * w[i];
          a[u][i] = rstd * (gg - m1 - xh * m2);
        }
        store_f32<T, VE>(dx + (row + u * s.rp) * p.C, a[u]);
      }
  }
}

// dw and db from the per-slab rows of sums [parts][2][C], in 64 bits and a fixed order.
__global__ void __launch_bounds__(1024) norm_param_kernel(const float* __restrict__ sums, float* __restrict__ dw,
                                                          float* __restrict__ db, long long parts, int C) {
  __shared__ double acc[32][33];
  grid_dependency_wait();
  const int j = threadIdx.x & 31, i = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + j;
  float* out = blockIdx.y ? db : dw;
  if (!out) return;
  double sum = 0.0;
  if (c < C) {
#pragma unroll 4
    for (long long r = i; r < parts; r += 32) sum += (double)sums[(2 * r + blockIdx.y) * C + c];
  }
  acc[i][j] = sum;
  __syncthreads();
  if (i == 0 && c < C) {
    for (int k = 1; k < 32; ++k) sum += acc[k][j];
    out[c] = (float)sum;
  }
}

// ------------------------------------------------------------------------------------------ host

bool ok_dtype(int d) { return d == NSB_F32 || d == NSB_BF16 || d == NSB_F16; }
bool fits(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

constexpr int kPlanSms = 148;  // (the buffers' sizes must not depend on the device that asks)

// One position per sample and a group that fits a CTA's threads whatever the vector: a row layout.
bool by_rows(long long L, int Cg) { return L == 1 && Cg <= kThreads; }

void plan_slabs(NormParams& p) {
  p.gpb = std::min(p.G, std::max(1, kChannels / p.Cg));
  p.pieces = (p.Cg + kChannels - 1) / kChannels;
  p.cblks = p.pieces > 1 ? p.G * p.pieces : (p.G + p.gpb - 1) / p.gpb;
  // four CTAs per SM, but no slab under 32 rows: a slab costs two reductions over the CTA
  const long long blocks = p.N * p.cblks, most = (p.L + 31) / 32;
  p.nslab = (int)std::max<long long>(1, std::min<long long>((4LL * kPlanSms + blocks - 1) / blocks, most));
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
NormParams make(int64_t N, int64_t L, int64_t C, int64_t G) {
  NormParams p = {};
  p.N = N, p.L = L, p.C = (int)C, p.G = (int)G, p.Cg = (int)(C / G);
  plan_slabs(p);
  return p;
}

template <typename T, int VE>
int launch_norm(NormParams p, bool backward, float* dw, float* db, cudaStream_t st) {
  long long parts;
  if (by_rows(p.L, p.Cg)) {
    const int team = p.Cg / VE;
    p.gpb = std::min(p.G, kThreads / team);
    const unsigned cb = (unsigned)((p.G + p.gpb - 1) / p.gpb);
    const bool shuf = team <= 32 && (team & (team - 1)) == 0;
    if (backward) {
      const dim3 grid(cb, (unsigned)(parts = row_chunks(p.N)));
      if (shuf) norm_rows_bwd_kernel<T, VE, true><<<grid, kThreads, 0, st>>>(p);
      else norm_rows_bwd_kernel<T, VE, false><<<grid, kThreads, 0, st>>>(p);
    } else {
      const long long rp = kThreads / (std::min(p.gpb, p.G) * team);
      const dim3 grid(cb, (unsigned)std::min<long long>((p.N + rp * kRowUnroll - 1) / (rp * kRowUnroll), 65535));
      if (shuf) norm_rows_fwd_kernel<T, VE, true><<<grid, kThreads, 0, st>>>(p);
      else norm_rows_fwd_kernel<T, VE, false><<<grid, kThreads, 0, st>>>(p);
    }
    NSB_CUDA_TRY(cudaGetLastError(), "launch norm_rows kernel");
  } else {
    const long long grid = p.N * p.cblks * p.nslab;
    if (grid > 0x7fffffffLL) return NSB_ERR_TOO_LARGE;
    parts = p.N * p.nslab;
    const dim3 g((unsigned)grid);
    if (backward) {
      norm_bwd_sums_kernel<T, VE><<<g, kThreads, 0, st>>>(p);
      NSB_CUDA_TRY(cudaGetLastError(), "launch norm_bwd_sums_kernel");
      if (p.y) NSB_CUDA_TRY(launch_dependent(norm_bwd_apply_kernel<T, VE>, g, dim3(kThreads), 0, st, p), "launch norm_bwd_apply_kernel");
    } else {
      norm_stats_kernel<T, VE><<<g, kThreads, 0, st>>>(p);
      NSB_CUDA_TRY(cudaGetLastError(), "launch norm_stats_kernel");
      NSB_CUDA_TRY(launch_dependent(norm_apply_kernel<T, VE>, g, dim3(kThreads), 0, st, p), "launch norm_apply_kernel");
    }
  }
  if (backward && (dw || db))
    NSB_CUDA_TRY(launch_dependent(norm_param_kernel, dim3((unsigned)((p.C + 31) / 32), 2), dim3(1024), 0, st,
                                  (const float*)p.sums, dw, db, parts, p.C), "launch norm_param_kernel");
  return NSB_OK;
}
template <typename T>
int go(const NormParams& p, bool backward, float* dw, float* db, cudaStream_t st) {
  DeviceInfo dev;
  const int r = get_device_info(&dev);
  if (r != NSB_OK) return r;
  // A thread's vector lies in one group, and in one piece of 256 channels of a group.
  auto ok = [&](int ve) {
    return p.Cg % ve == 0 && fits(p.x, sizeof(T) * ve) && fits(p.y, sizeof(T) * ve) && fits(p.dy, sizeof(T) * ve);
  };
  if constexpr (sizeof(T) == 2)
    if (ok(8)) return launch_norm<T, 8>(p, backward, dw, db, st);
  if (ok(4)) return launch_norm<T, 4>(p, backward, dw, db, st);
  return launch_norm<T, 1>(p, backward, dw, db, st);
}
int dispatch(const NormParams& p, int dtype, bool backward, float* dw, float* db, cudaStream_t st) {
  switch (dtype) {
    case NSB_F32: return go<float>(p, backward, dw, db, st);
    case NSB_BF16: return go<__nv_bfloat16>(p, backward, dw, db, st);
    default: return go<__half>(p, backward, dw, db, st);
  }
}

}  // namespace
}  // namespace nsb

using namespace nsb;

extern "C" int64_t nsb_group_norm_scratch_floats(int64_t N, int64_t L, int64_t C, int64_t G, int backward) {
  if (check_sizes(N, L, C, G, 0, NSB_F32) != NSB_OK || N * L * C == 0) return 0;
  const NormParams p = make(N, L, C, G);
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
  NormParams p = make(N, L, C, G);
  if (!by_rows(L, p.Cg) && !scratch) return NSB_ERR_INVALID_ARG;
  p.x = x, p.w = weight, p.b = bias, p.y = y, p.mean = mean, p.rstd = rstd, p.part = scratch, p.eps = eps;
  p.act = activation;
  return dispatch(p, dtype, false, nullptr, nullptr, static_cast<cudaStream_t>(stream));
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
  NormParams p = make(N, L, C, G);
  p.x = x, p.dy = dy, p.w = weight, p.b = bias, p.y = dx, p.act = activation;
  p.mean = const_cast<float*>(mean), p.rstd = const_cast<float*>(rstd);
  p.sums = scratch;
  if (!by_rows(L, p.Cg)) p.part = scratch + 2 * N * p.nslab * C;
  else if (!dweight && !dbias) p.sums = nullptr;
  return dispatch(p, dtype, true, dweight, dbias, st);
}
