// Group normalisation with an activation, both layouts, forward and backward.
//
//   over the n = C / G * S elements of group g of image b:  mu, var;  rstd = 1 / sqrt(var + eps)
//   xhat = (x - mu) rstd,  z = xhat w_c + b_c,  y = act(z)
//   dz = gy act'(z),  S1 = sum_s dz,  S2 = sum_s dz xhat for every channel of an image,
//   gx = rstd (dz w_c - (sum_c w_c S1 + xhat sum_c w_c S2) / n),  gw_c = sum_b S2,  gb_c = sum_b S1
//
// Bound: HBM.  Tiles of an image leave partial results, which are added up in a fixed order, and the tiles are read a
// second time for the output.
//
// Statistics: a thread's run of at most RUN values is summed as differences from its first value K.  K is one of the run, so
// n (K - mean)^2 <= n M2 and sum d^2 - (sum d)^2 / n loses at most log2(n) + 1 bits, wherever the values lie and whatever else
// the image holds; runs are then merged with their means (M2 = sum M2_i + n_i (mean_i - mean)^2).
#include "mix.cuh"

namespace mc {
namespace norm {
using mix::act_slope;
using mix::act_value;

constexpr int THREADS = 256, RUN = 32;
constexpr int SEGMENT = 4096;  // elements of a plane that a warp takes at a time (NCHW)

template <typename CT> struct Part { CT n, mean, m2; };
template <typename CT> struct Two { CT a, b; };

struct Args {
  const void *x, *w, *b, *gy;
  void *y, *gx, *gw, *gb;
  void* stats;  // mean and rstd of every group of every image
  void* part;   // what a tile leaves
  void* sums;   // backward: S1, S2 of every channel of every image
  void* coef;   // backward: the two sums over a group, divided by n
  long long S, B;
  int C, G, Cg, act;
  double eps;
  // channels-last: tiles of `px` pixels, in columns of at most 256 vectors
  int px, tiles, cols, V, R, lanes;
  // planes: segments of a plane
  int segs;
  long long items;  // partial results in all
};

template <typename T> struct Vec { static constexpr int N = 16 / sizeof(T); };

// N values from p (16-byte aligned if N > 1) as CT
template <int N, typename T, typename CT>
__device__ __forceinline__ void load_vec(const T* p, CT (&v)[N]) {
  if constexpr (N == 1) {
    v[0] = (CT)ldv(p);
  } else {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
    if constexpr (sizeof(T) == 2) {
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    } else {
      const T* f = reinterpret_cast<const T*>(&q);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = f[i];
    }
  }
}
template <int N, typename T, typename CT>
__device__ __forceinline__ void store_vec(T* p, const CT (&v)[N]) {
  if constexpr (N == 1) {
    stv(p, v[0]);
  } else {
    __align__(16) T o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) stv(o + i, v[i]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(o);
  }
}
// the vector at elements [i, i + N) of [lo, hi); elements outside read as zero and are not written
template <int N, typename T, typename CT>
__device__ __forceinline__ void load_in(const T* p, long long i, long long lo, long long hi, CT (&v)[N]) {
  if (i >= lo && i + N <= hi) return load_vec<N>(p + i, v);
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = i + e >= lo && i + e < hi ? (CT)ldv(p + i + e) : CT(0);
}
template <int N, typename T, typename CT>
__device__ __forceinline__ void store_in(T* p, long long i, long long lo, long long hi, const CT (&v)[N]) {
  if (i >= lo && i + N <= hi) return store_vec<N>(p + i, v);
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (i + e >= lo && i + e < hi) stv(p + i + e, v[e]);
}
template <typename CT>
__device__ __forceinline__ CT warp_sum(CT v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// ---- channels-last ------------------------------------------------------------------------------------
// R pixels are V vectors of N elements; vector j of such a row of pixels holds the same channels everywhere.  A thread keeps one
// vector (of a column of 256) and takes every lanes-th row of the tile.
struct Place {
  long long row0, image;  // flat index of the tile's first element and of the image
  long long end;          // flat index behind the tile
  int j, lane, vc;        // vector of the row, which of the rows, vectors of this column
  bool on;
};
template <int N>
__device__ __forceinline__ Place place_of(const Args& a, long long item) {
  Place p;
  const int col = (int)(item % a.cols);
  const long long t = item / a.cols % a.tiles, b = item / a.cols / a.tiles;
  p.image = b * a.S * a.C;
  p.row0 = p.image + t * a.px * a.C;
  const long long left = a.S - t * a.px;
  p.end = p.row0 + (left < a.px ? left : a.px) * a.C;
  p.vc = min(256, a.V - col * 256);
  p.lane = threadIdx.x / p.vc;
  p.j = col * 256 + threadIdx.x % p.vc;
  p.on = p.lane < a.lanes;
  return p;
}

template <typename T, int N>
__global__ void __launch_bounds__(THREADS) rows_stats_kernel(const Args a) {
  typedef typename Traits<T>::CT CT;
  __shared__ Part<CT> sm[N][THREADS];
  const T* x = (const T*)a.x;
  const Place p = place_of<N>(a, blockIdx.x);
  CT k[N], s[N], q[N], n[N];
#pragma unroll
  for (int e = 0; e < N; ++e) k[e] = s[e] = q[e] = n[e] = CT(0);
  if (p.on) {
    const long long step = (long long)a.lanes * a.V * N;
    long long i = p.row0 + ((long long)p.lane * a.V + p.j) * N;
    load_in<N>(x, i, p.row0, p.end, k);
    for (; i < p.end; i += step) {
      CT v[N];
      load_in<N>(x, i, p.row0, p.end, v);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (i + e >= p.end) continue;
        const CT d = v[e] - k[e];
        s[e] += d, q[e] += d * d, n[e] += CT(1);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const CT m = n[e] > CT(0) ? s[e] / n[e] : CT(0);
    sm[e][threadIdx.x] = Part<CT>{n[e], k[e] + m, fmax(q[e] - s[e] * m, CT(0)) + (q[e] - q[e])};  // (NaN and infinities stay)
  }
  __syncthreads();
  // one warp per group: its channels appear R times in a row of pixels
  const int col = (int)(blockIdx.x % a.cols), wl = threadIdx.x % 32;
  const int entries = a.Cg * a.R * a.lanes;
  Part<CT>* out = (Part<CT>*)a.part + blockIdx.x * (long long)a.G;
  for (int g = threadIdx.x / 32; g < a.G; g += THREADS / 32) {
    const auto entry = [&](int i, Part<CT>& v) {
      const int c = g * a.Cg + i % a.Cg, r = i / a.Cg % a.R, l = i / a.Cg / a.R;
      const int f = r * a.C + c, j = f / N - col * 256;
      if (j < 0 || j >= p.vc) return false;
      v = sm[f % N][l * p.vc + j];
      return v.n > CT(0);
    };
    CT cnt = CT(0), sum = CT(0), m2 = CT(0);
    Part<CT> v;
    for (int i = wl; i < entries; i += 32)
      if (entry(i, v)) cnt += v.n, sum += v.n * v.mean;
    cnt = warp_sum(cnt), sum = warp_sum(sum);
    const CT mean = cnt > CT(0) ? sum / cnt : CT(0);
    for (int i = wl; i < entries; i += 32)
      if (entry(i, v)) m2 += v.m2 + v.n * (v.mean - mean) * (v.mean - mean);
    m2 = warp_sum(m2);
    if (wl == 0) out[g] = Part<CT>{cnt, mean, m2};
  }
}

// The coefficients of a thread's channels: z = (x - mean) scale + shift.
template <int N, typename T, typename CT>
struct Coefs {
  CT mean[N], scale[N], shift[N];
  __device__ __forceinline__ void load(const Args& a, long long b, int c, int e) {
    const CT* st = (const CT*)a.stats + 2 * (b * a.G + c / a.Cg);
    const CT w = a.w ? (CT)ldv((const T*)a.w + c) : CT(1);
    mean[e] = st[0], scale[e] = st[1] * w, shift[e] = a.b ? (CT)ldv((const T*)a.b + c) : CT(0);
  }
  __device__ __forceinline__ CT z(CT x, int e) const { return (x - mean[e]) * scale[e] + shift[e]; }
};

template <typename T, int N>
__global__ void __launch_bounds__(THREADS) rows_apply_kernel(const Args a) {
  typedef typename Traits<T>::CT CT;
  const Place p = place_of<N>(a, blockIdx.x);
  if (!p.on) return;
  const long long b = blockIdx.x / a.cols / a.tiles;
  Coefs<N, T, CT> k;
#pragma unroll
  for (int e = 0; e < N; ++e) k.load(a, b, (int)(((long long)p.j * N + e) % a.C), e);
  const long long step = (long long)a.lanes * a.V * N;
  for (long long i = p.row0 + ((long long)p.lane * a.V + p.j) * N; i < p.end; i += step) {
    CT v[N];
    load_in<N>((const T*)a.x, i, p.row0, p.end, v);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = act_value<CT>(a.act, k.z(v[e], e));
    store_in<N>((T*)a.y, i, p.row0, p.end, v);
  }
}

template <typename T, int N>
__global__ void __launch_bounds__(THREADS) rows_sums_kernel(const Args a) {
  typedef typename Traits<T>::CT CT;
  __shared__ Two<CT> sm[N][THREADS];
  const Place p = place_of<N>(a, blockIdx.x);
  const long long b = blockIdx.x / a.cols / a.tiles;
  CT s1[N], s2[N];
#pragma unroll
  for (int e = 0; e < N; ++e) s1[e] = s2[e] = CT(0);
  if (p.on) {
    Coefs<N, T, CT> k;
#pragma unroll
    for (int e = 0; e < N; ++e) k.load(a, b, (int)(((long long)p.j * N + e) % a.C), e);
    const long long step = (long long)a.lanes * a.V * N;
    for (long long i = p.row0 + ((long long)p.lane * a.V + p.j) * N; i < p.end; i += step) {
      CT v[N], g[N];
      load_in<N>((const T*)a.x, i, p.row0, p.end, v);
      load_in<N>((const T*)a.gy, i, p.row0, p.end, g);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (i + e >= p.end) continue;
        const CT dz = g[e] * act_slope<CT>(a.act, k.z(v[e], e));
        s1[e] += dz, s2[e] += dz * (v[e] - k.mean[e]);  // (times rstd below)
      }
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) sm[e][threadIdx.x] = Two<CT>{s1[e], s2[e]};
  __syncthreads();
  const int col = (int)(blockIdx.x % a.cols), entries = a.R * a.lanes;
  // threads that share a channel, as many as the channels leave
  const int sub = a.C >= 128 ? 1 : a.C >= 32 ? 8 : 32;
  Two<CT>* out = (Two<CT>*)a.part + blockIdx.x * (long long)a.C;
  for (int c0 = 0; c0 < a.C; c0 += THREADS / sub) {
    const int c = c0 + threadIdx.x / sub;
    CT u = CT(0), v = CT(0);
    if (c < a.C)
      for (int i = threadIdx.x % sub; i < entries; i += sub) {
        const int r = i % a.R, l = i / a.R, f = r * a.C + c, j = f / N - col * 256;
        if (j >= 0 && j < p.vc) u += sm[f % N][l * p.vc + j].a, v += sm[f % N][l * p.vc + j].b;
      }
    for (int o = sub / 2; o; o >>= 1) u += __shfl_xor_sync(~0u, u, o), v += __shfl_xor_sync(~0u, v, o);
    if (c < a.C && threadIdx.x % sub == 0) out[c] = Two<CT>{u, v * ((const CT*)a.stats)[2 * (b * a.G + c / a.Cg) + 1]};
  }
}

template <typename T, int N>
__global__ void __launch_bounds__(THREADS) rows_grad_kernel(const Args a) {
  typedef typename Traits<T>::CT CT;
  const Place p = place_of<N>(a, blockIdx.x);
  if (!p.on) return;
  const long long b = blockIdx.x / a.cols / a.tiles;
  Coefs<N, T, CT> k;
  CT c0[N], c1[N];  // gx = dz scale - c0 - (x - mean) c1
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int c = (int)(((long long)p.j * N + e) % a.C);
    k.load(a, b, c, e);
    const CT rstd = ((const CT*)a.stats)[2 * (b * a.G + c / a.Cg) + 1];
    const Two<CT> t = ((const Two<CT>*)a.coef)[b * a.G + c / a.Cg];
    c0[e] = rstd * t.a, c1[e] = rstd * rstd * t.b;
  }
  const long long step = (long long)a.lanes * a.V * N;
  for (long long i = p.row0 + ((long long)p.lane * a.V + p.j) * N; i < p.end; i += step) {
    CT v[N], g[N];
    load_in<N>((const T*)a.x, i, p.row0, p.end, v);
    load_in<N>((const T*)a.gy, i, p.row0, p.end, g);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const CT dz = g[e] * act_slope<CT>(a.act, k.z(v[e], e));
      g[e] = dz * k.scale[e] - c0[e] - (v[e] - k.mean[e]) * c1[e];
    }
    store_in<N>((T*)a.gx, i, p.row0, p.end, g);
  }
}

// ---- planes ---------------------------------------------------------------------------------------------
// A warp takes a segment of a plane; vectors start on 16 bytes wherever the plane does (all tensors lie alike).
template <int N>
struct Segment {
  long long lo, hi, i;  // flat: first element, behind the last, this lane's first vector
  long long b;
  int c;
  __device__ Segment(const Args& a, long long item) {
    const long long plane = item / a.segs;
    const int k = (int)(item % a.segs);
    c = (int)(plane % a.C), b = plane / a.C;
    lo = plane * a.S + (long long)k * SEGMENT;
    hi = lo + min((long long)SEGMENT, a.S - (long long)k * SEGMENT);
    i = lo / N * N + threadIdx.x % 32 * N;
  }
};
template <typename T, int N>
__global__ void __launch_bounds__(THREADS) planes_stats_kernel(const Args a) {
  typedef typename Traits<T>::CT CT;
  const long long item = blockIdx.x * (long long)(THREADS / 32) + threadIdx.x / 32;
  if (item >= a.items) return;
  Segment<N> g(a, item);
  CT n = CT(0), s = CT(0), q = CT(0);
  // (the lane's first value; a lane whose first vector starts before the segment takes the segment's first)
  const CT k = g.i < g.hi ? (CT)ldv((const T*)a.x + max(g.i, g.lo)) : CT(0);
  for (long long i = g.i; i < g.hi; i += 32 * N) {
    CT v[N];
    load_in<N>((const T*)a.x, i, g.lo, g.hi, v);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (i + e < g.lo || i + e >= g.hi) continue;
      const CT d = v[e] - k;
      s += d, q += d * d, n += CT(1);
    }
  }
  const CT m = n > CT(0) ? s / n : CT(0);
  CT m2 = fmax(q - s * m, CT(0)) + (q - q);
  const CT mean = k + m, cnt = warp_sum(n), all = warp_sum(n * mean) / cnt;
  m2 = warp_sum(m2 + n * (mean - all) * (mean - all));
  if (threadIdx.x % 32 == 0) ((Part<CT>*)a.part)[item] = Part<CT>{cnt, all, m2};
}
template <typename T, int N>
__global__ void __launch_bounds__(THREADS) planes_apply_kernel(const Args a) {
  typedef typename Traits<T>::CT CT;
  const long long item = blockIdx.x * (long long)(THREADS / 32) + threadIdx.x / 32;
  if (item >= a.items) return;
  Segment<N> g(a, item);
  Coefs<1, T, CT> k;
  k.load(a, g.b, g.c, 0);
  for (long long i = g.i; i < g.hi; i += 32 * N) {
    CT v[N];
    load_in<N>((const T*)a.x, i, g.lo, g.hi, v);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = act_value<CT>(a.act, k.z(v[e], 0));
    store_in<N>((T*)a.y, i, g.lo, g.hi, v);
  }
}
template <typename T, int N>
__global__ void __launch_bounds__(THREADS) planes_sums_kernel(const Args a) {
  typedef typename Traits<T>::CT CT;
  const long long item = blockIdx.x * (long long)(THREADS / 32) + threadIdx.x / 32;
  if (item >= a.items) return;
  Segment<N> g(a, item);
  Coefs<1, T, CT> k;
  k.load(a, g.b, g.c, 0);
  CT s1 = CT(0), s2 = CT(0);
  for (long long i = g.i; i < g.hi; i += 32 * N) {
    CT v[N], d[N];
    load_in<N>((const T*)a.x, i, g.lo, g.hi, v);
    load_in<N>((const T*)a.gy, i, g.lo, g.hi, d);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (i + e < g.lo || i + e >= g.hi) continue;
      const CT dz = d[e] * act_slope<CT>(a.act, k.z(v[e], 0));
      s1 += dz, s2 += dz * (v[e] - k.mean[0]);
    }
  }
  s1 = warp_sum(s1), s2 = warp_sum(s2);
  if (threadIdx.x % 32 == 0)
    ((Two<CT>*)a.part)[item] = Two<CT>{s1, s2 * ((const CT*)a.stats)[2 * (g.b * a.G + g.c / a.Cg) + 1]};
}
template <typename T, int N>
__global__ void __launch_bounds__(THREADS) planes_grad_kernel(const Args a) {
  typedef typename Traits<T>::CT CT;
  const long long item = blockIdx.x * (long long)(THREADS / 32) + threadIdx.x / 32;
  if (item >= a.items) return;
  Segment<N> g(a, item);
  Coefs<1, T, CT> k;
  k.load(a, g.b, g.c, 0);
  const long long group = g.b * a.G + g.c / a.Cg;
  const CT rstd = ((const CT*)a.stats)[2 * group + 1];
  const Two<CT> t = ((const Two<CT>*)a.coef)[group];
  const CT c0 = rstd * t.a, c1 = rstd * rstd * t.b;
  for (long long i = g.i; i < g.hi; i += 32 * N) {
    CT v[N], d[N];
    load_in<N>((const T*)a.x, i, g.lo, g.hi, v);
    load_in<N>((const T*)a.gy, i, g.lo, g.hi, d);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const CT dz = d[e] * act_slope<CT>(a.act, k.z(v[e], 0));
      d[e] = dz * k.scale[0] - c0 - (v[e] - k.mean[0]) * c1;
    }
    store_in<N>((T*)a.gx, i, g.lo, g.hi, d);
  }
}

// ---- between the two passes ---------------------------------------------------------------------------
// Partial results of group (b, g): `count` of them, the i-th at first + i / run * jump + i % run ... of one kind or the other.
struct Parts {
  long long first, count;
  int step;
  __device__ Parts(const Args& a, bool rows, long long b, int g) {
    if (rows) count = (long long)a.tiles * a.cols, first = b * count * a.G + g, step = a.G;
    else count = (long long)a.Cg * a.segs, first = (b * a.C + (long long)g * a.Cg) * a.segs, step = 1;
  }
};
// one warp per group of an image, in double
template <typename CT>
__global__ void __launch_bounds__(THREADS) stats_kernel(const Args a, bool rows) {
  const long long group = blockIdx.x * (long long)(THREADS / 32) + threadIdx.x / 32;
  if (group >= a.B * a.G) return;
  const Parts p(a, rows, group / a.G, (int)(group % a.G));
  const Part<CT>* part = (const Part<CT>*)a.part + p.first;
  const int lane = threadIdx.x % 32;
  double n = 0, sum = 0, m2 = 0;
  for (long long i = lane; i < p.count; i += 32) n += part[i * p.step].n, sum += (double)part[i * p.step].n * part[i * p.step].mean;
  n = warp_sum(n), sum = warp_sum(sum);
  const double mean = sum / n;
  for (long long i = lane; i < p.count; i += 32) {
    const Part<CT> v = part[i * p.step];
    if (v.n > CT(0)) m2 += v.m2 + (double)v.n * (v.mean - mean) * (v.mean - mean);
  }
  m2 = warp_sum(m2);
  if (lane == 0) {
    CT* st = (CT*)a.stats + 2 * group;
    st[0] = (CT)mean, st[1] = (CT)(1.0 / sqrt(m2 / n + a.eps));
  }
}
// S1, S2 of every channel of an image and what a group's gradient subtracts: one block per group of an image
template <typename T>
__global__ void __launch_bounds__(THREADS) coef_kernel(const Args a, bool rows) {
  typedef typename Traits<T>::CT CT;
  __shared__ double sm[2][THREADS / 32];
  const long long b = blockIdx.x / a.G;
  const int g = (int)(blockIdx.x % a.G), warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  double u = 0, v = 0;
  for (int i = warp; i < a.Cg; i += THREADS / 32) {
    const int c = g * a.Cg + i;
    const long long count = rows ? (long long)a.tiles * a.cols : a.segs;
    const Two<CT>* part = (const Two<CT>*)a.part + (rows ? b * count * a.C + c : (b * a.C + c) * count);
    double s1 = 0, s2 = 0;
    for (long long k = lane; k < count; k += 32) s1 += part[rows ? k * a.C : k].a, s2 += part[rows ? k * a.C : k].b;
    s1 = warp_sum(s1), s2 = warp_sum(s2);
    const double w = a.w ? (double)ldv((const T*)a.w + c) : 1.0;
    u += w * s1, v += w * s2;
    if (lane == 0) ((Two<double>*)a.sums)[b * a.C + c] = Two<double>{s1, s2};
  }
  if (lane == 0) sm[0][warp] = u, sm[1][warp] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    u = v = 0;
    for (int i = 0; i < THREADS / 32; ++i) u += sm[0][i], v += sm[1][i];
    const double n = (double)a.Cg * (double)a.S;
    ((Two<CT>*)a.coef)[blockIdx.x] = Two<CT>{(CT)(u / n), (CT)(v / n)};
  }
}
template <typename T>
__global__ void __launch_bounds__(THREADS) params_kernel(const Args a) {
  const int c = blockIdx.x * (THREADS / 32) + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (c >= a.C) return;
  double u = 0, v = 0;
  for (long long b = lane; b < a.B; b += 32) {
    const Two<double> t = ((const Two<double>*)a.sums)[b * a.C + c];
    u += t.a, v += t.b;
  }
  u = warp_sum(u), v = warp_sum(v);
  typedef typename Traits<T>::CT CT;
  if (lane == 0 && a.gb) stv((T*)a.gb + c, (CT)u);
  if (lane == 0 && a.gw) stv((T*)a.gw + c, (CT)v);
}

// ---- host -----------------------------------------------------------------------------------------------
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
static int csize(int dtype) { return dtype == MC_F64 ? 8 : 4; }
static int esize(int dtype) { return dtype == MC_F64 ? 8 : dtype == MC_F32 ? 4 : 2; }
static int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

static int check_desc(const mc_norm_desc* d) {
  if (!d || d->B <= 0 || d->S <= 0 || d->C <= 0 || d->groups <= 0 || d->C % d->groups) return MC_ERR_BAD_ARG;
  if (d->dtype != MC_F32 && d->dtype != MC_F64 && d->dtype != MC_BF16) return MC_ERR_BAD_ARG;
  if (d->layout != MC_NCHW && d->layout != MC_NHWC) return MC_ERR_BAD_ARG;
  if (d->act < MC_ACT_NONE || d->act > MC_ACT_SIGMOID || !(d->eps >= 0)) return MC_ERR_BAD_ARG;
  if (d->S >= (1ll << 31) || d->B >= (1ll << 31) || d->B * d->S > (1ll << 31) - 256 || d->C > (1 << 20)) return MC_ERR_TOO_LARGE;
  return MC_OK;
}

struct Plan {
  Args a{};
  bool rows, vec;
  size_t part_f, part_b, sums, coef;  // bytes
  unsigned blocks;
};
// Blocks of a launch: at most 2^31 - 1.
static int plan(const mc_norm_desc* d, Plan& p) {
  Args& a = p.a;
  a.S = d->S, a.B = d->B, a.C = d->C, a.G = d->groups, a.Cg = d->C / d->groups, a.act = d->act, a.eps = d->eps;
  const int N = 16 / esize(d->dtype), ct = csize(d->dtype);
  p.rows = d->layout == MC_NHWC || d->S == 1;
  long long blocks;
  if (p.rows) {
    p.vec = d->B == 1 || d->S * d->C % N == 0;  // every image starts on 16 bytes
    const int n = p.vec ? N : 1;
    a.R = n / gcd(n, d->C), a.V = (int)((long long)a.R * d->C / n);
    a.cols = (a.V + 255) / 256;
    a.lanes = a.cols > 1 ? 1 : 256 / a.V;
    const long long step = (long long)a.lanes * a.R;
    long long k = (d->B * d->S / step * a.cols) / (148 * 8);
    k = k < 1 ? 1 : k > RUN ? RUN : k;
    a.px = (int)(step * k);
    a.tiles = (int)((d->S + a.px - 1) / a.px);
    a.items = blocks = d->B * a.tiles * a.cols;
    p.part_f = (size_t)blocks * a.G * 3 * ct, p.part_b = (size_t)blocks * a.C * 2 * ct;
  } else {
    p.vec = true;
    a.segs = (int)((d->S + SEGMENT - 1) / SEGMENT);
    a.items = d->B * d->C * a.segs;
    blocks = (a.items + THREADS / 32 - 1) / (THREADS / 32);
    p.part_f = (size_t)a.items * 3 * ct, p.part_b = (size_t)a.items * 2 * ct;
  }
  p.sums = (size_t)d->B * d->C * 16, p.coef = (size_t)d->B * d->groups * 2 * ct;
  if (blocks >= (1ll << 31) || d->B * d->groups >= (1ll << 31)) return MC_ERR_TOO_LARGE;
  p.blocks = (unsigned)blocks;
  return MC_OK;
}
static bool on(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

#define MC_NORM_KERNEL(name)                                                                        \
  template <typename T>                                                                             \
  static void name(const Plan& p, cudaStream_t st) {                                                \
    constexpr int N = Vec<T>::N;                                                                    \
    if (!p.rows) planes_##name##_kernel<T, N><<<p.blocks, THREADS, 0, st>>>(p.a);                   \
    else if (p.vec) rows_##name##_kernel<T, N><<<p.blocks, THREADS, 0, st>>>(p.a);                  \
    else rows_##name##_kernel<T, 1><<<p.blocks, THREADS, 0, st>>>(p.a);                             \
    MC_COUNT(1);                                                                                    \
  }
MC_NORM_KERNEL(stats)
MC_NORM_KERNEL(apply)
MC_NORM_KERNEL(sums)
MC_NORM_KERNEL(grad)
#undef MC_NORM_KERNEL

template <typename T>
static int forward(const Plan& p, cudaStream_t st) {
  typedef typename Traits<T>::CT CT;
  stats<T>(p, st);
  stats_kernel<CT><<<(unsigned)((p.a.B * p.a.G + 7) / 8), THREADS, 0, st>>>(p.a, p.rows), MC_COUNT(1);
  apply<T>(p, st);
  MC_CHECK_LAUNCH();
  return MC_OK;
}
template <typename T>
static int backward(const Plan& p, cudaStream_t st) {
  sums<T>(p, st);
  coef_kernel<T><<<(unsigned)(p.a.B * p.a.G), THREADS, 0, st>>>(p.a, p.rows), MC_COUNT(1);
  if (p.a.gw || p.a.gb) params_kernel<T><<<(p.a.C + 7) / 8, THREADS, 0, st>>>(p.a), MC_COUNT(1);
  if (p.a.gx) grad<T>(p, st);
  MC_CHECK_LAUNCH();
  return MC_OK;
}

}  // namespace norm
}  // namespace mc
using namespace mc;

extern "C" {

size_t mc_group_norm_stats_bytes(const mc_norm_desc* d) {
  return norm::check_desc(d) ? 0 : (size_t)d->B * d->groups * 2 * norm::csize(d->dtype);
}
size_t mc_group_norm_workspace_bytes(const mc_norm_desc* d, int32_t phase) {
  norm::Plan p;
  if (norm::check_desc(d) || norm::plan(d, p)) return 0;
  if (phase != MC_PHASE_BACKWARD) return norm::up256(p.part_f);
  return norm::up256(p.part_b) + norm::up256(p.sums) + norm::up256(p.coef);
}
int mc_group_norm_fwd(const mc_norm_desc* d, const void* x, const void* w, const void* bias, void* y, void* stats, void* ws,
                      size_t ws_bytes, void* stream) {
  if (const int rc = norm::check_desc(d)) return rc;
  if (!x || !y || !stats) return MC_ERR_BAD_ARG;
  const size_t e = norm::esize(d->dtype);
  if (!norm::on(x, 16) || !norm::on(y, 16) || !norm::on(w, e) || !norm::on(bias, e) || !norm::on(stats, 16) || !norm::on(ws, 16))
    return MC_ERR_BAD_ARG;
  norm::Plan p;
  if (const int rc = norm::plan(d, p)) return rc;
  if (!ws || ws_bytes < norm::up256(p.part_f)) return MC_ERR_WORKSPACE;
  p.a.x = x, p.a.w = w, p.a.b = bias, p.a.y = y, p.a.stats = stats, p.a.part = ws;
  if (d->dtype == MC_F32) return norm::forward<float>(p, (cudaStream_t)stream);
  if (d->dtype == MC_F64) return norm::forward<double>(p, (cudaStream_t)stream);
  return norm::forward<bf16>(p, (cudaStream_t)stream);
}
int mc_group_norm_bwd(const mc_norm_desc* d, const void* gy, const void* x, const void* w, const void* bias, const void* stats,
                      void* gx, void* gw, void* gb, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = norm::check_desc(d)) return rc;
  if (!gy || !x || !stats) return MC_ERR_BAD_ARG;
  const size_t e = norm::esize(d->dtype);
  if (!norm::on(x, 16) || !norm::on(gy, 16) || !norm::on(gx, 16) || !norm::on(w, e) || !norm::on(bias, e) || !norm::on(gw, e) ||
      !norm::on(gb, e) || !norm::on(stats, 16) || !norm::on(ws, 16))
    return MC_ERR_BAD_ARG;
  norm::Plan p;
  if (const int rc = norm::plan(d, p)) return rc;
  if (!ws || ws_bytes < mc_group_norm_workspace_bytes(d, MC_PHASE_BACKWARD)) return MC_ERR_WORKSPACE;
  char* at = (char*)ws;
  p.a.x = x, p.a.w = w, p.a.b = bias, p.a.gy = gy, p.a.gx = gx, p.a.gw = gw, p.a.gb = gb, p.a.stats = (void*)stats;
  p.a.part = at, at += norm::up256(p.part_b);
  p.a.sums = at, at += norm::up256(p.sums);
  p.a.coef = at;
  if (d->dtype == MC_F32) return norm::backward<float>(p, (cudaStream_t)stream);
  if (d->dtype == MC_F64) return norm::backward<double>(p, (cudaStream_t)stream);
  return norm::backward<bf16>(p, (cudaStream_t)stream);
}

}  // extern "C"
