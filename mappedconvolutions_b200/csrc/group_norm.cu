// Group normalisation with an activation, both layouts, forward and backward.
//
//   over the n = C / G * S elements of group g of image b:  mu, var;  rstd = 1 / sqrt(var + eps)
//   xhat = (x - mu) rstd,  z = xhat w_c + b_c,  y = act(z)
//   dz = gy act'(z),  S1 = sum_s dz,  S2 = sum_s dz xhat for every channel of an image,
//   gx = rstd (dz w_c - (sum_c w_c S1 + xhat sum_c w_c S2) / n),  gw_c = sum_b S2,  gb_c = sum_b S1
//
// Bound: HBM.  Three launches: every tile's sums, what they add up to for each group (in a fixed order), the output.  The second and
// third start while the one before them runs (the third fetches its first vectors meanwhile) and wait for it before they read what it
// wrote; the third walks the tiles backwards: what the first read last is still in L2.
// Measured instead and taken back: one launch whose blocks draw tiles and read an image a second time while it is in L2, each tile
// waiting for its image's sums.  64 x 10 242 x 256 bf16, forward / backward: 236 / 348 us, with a DRAM traffic that was none the
// smaller - to keep the blocks busy through the waits took more tiles at a time than L2 holds.
//
// Statistics: a thread's run of at most RUN values (planes: 128) is summed as differences from its first value K.  K is one of the
// run, so n (K - mean)^2 <= n M2 and sum d^2 - (sum d)^2 / n loses at most log2(n) + 1 bits, wherever the values lie and whatever else
// the image holds; runs are then merged with their means (M2 = sum M2_i + n_i (mean_i - mean)^2).
#include <type_traits>

#include "act_pairs.cuh"
#include "mix.cuh"

namespace mc {
namespace norm {

constexpr int THREADS = 256, WARPS = THREADS / 32, RUN = 32;
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
  int tiles;  // of an image
  int param_blocks;  // of the third launch
  // channels-last: tiles of `px` pixels, in columns of at most 256 vectors
  int px, cols, V, R, lanes;
  // Elements of a whole column; channels and groups that the part of a column has room for: all there are, or those that a column can
  // hold any of, from its first one on and around the end.  (Room for all in each column: scratch of C^2, 8.6 GB for 4 MB of 2^20 channels.)
  int column, chans, grps;
  bool wide;    // more than a column to a row
  bool joined;  // the channels of a vector are of one group, and w and b start on 16 bytes
  // planes: segments of a plane, and how many a warp takes
  int segs, per;
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
  } else if constexpr (sizeof(T) == 2) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
  } else {
    __align__(16) T o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = v[i];
    __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(o));
  }
}
// A vector as it lies in memory, on its way.
template <typename T, int N> struct Raw {
  uint4 q;
  __device__ __forceinline__ void load(const T* p) { q = __ldg(reinterpret_cast<const uint4*>(p)); }
  template <typename CT>
  __device__ __forceinline__ void unpack(CT (&v)[N]) const {
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
};
template <typename T> struct Raw<T, 1> {
  typename Traits<T>::CT q;
  __device__ __forceinline__ void load(const T* p) { q = ldv(p); }
  template <typename CT>
  __device__ __forceinline__ void unpack(CT (&v)[1]) const { v[0] = q; }
};
// the vector at elements [i, i + N) of [lo, hi); elements outside read as zero and are not written
template <int N, typename T, typename CT>
__device__ __forceinline__ void load_in(const T* p, long long i, long long lo, long long hi, CT (&v)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = i + e >= lo && i + e < hi ? (CT)ldv(p + i + e) : CT(0);
}
template <int N, typename T, typename CT>
__device__ __forceinline__ void store_in(T* p, long long i, long long lo, long long hi, const CT (&v)[N]) {
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

// ---- arithmetic on N values, float32 in pairs --------------------------------------------------------------
#define MC_PAIRS(CT, N) if constexpr (sizeof(CT) == 4 && N % 2 == 0)
#define MC_2(v, i) make_float2((v)[2 * (i)], (v)[2 * (i) + 1])
template <typename CT, int N>
__device__ __forceinline__ void fma_to(CT (&d)[N], const CT (&a)[N], const CT (&b)[N], const CT (&c)[N]) {  // d = a b + c
  MC_PAIRS(CT, N) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 r = mix::fma2(MC_2(a, i), MC_2(b, i), MC_2(c, i));
      d[2 * i] = r.x, d[2 * i + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = fma(a[i], b[i], c[i]);
  }
}
template <typename CT, int N>
__device__ __forceinline__ void add_to(CT (&d)[N], const CT (&a)[N], const CT (&b)[N]) {
  MC_PAIRS(CT, N) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 r = mix::add2(MC_2(a, i), MC_2(b, i));
      d[2 * i] = r.x, d[2 * i + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = a[i] + b[i];
  }
}
template <typename CT, int N>
__device__ __forceinline__ void mul_to(CT (&d)[N], const CT (&a)[N], const CT (&b)[N]) {
  MC_PAIRS(CT, N) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 r = mix::mul2(MC_2(a, i), MC_2(b, i));
      d[2 * i] = r.x, d[2 * i + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = a[i] * b[i];
  }
}

// z <- act(z), or s = act'(z).  ACT < 0: looked up at run time.  bf16 vectors take the short forms (a slope comes with its value there).
template <int ACT> struct Short { typedef mix::ActNone type; };
template <> struct Short<MC_ACT_RELU> { typedef mix::ActRelu type; };
template <> struct Short<MC_ACT_GELU> { typedef mix::ActGelu type; };
template <> struct Short<MC_ACT_GELU_TANH> { typedef mix::ActGeluTanh type; };
template <> struct Short<MC_ACT_SILU> { typedef mix::ActSilu type; };
template <> struct Short<MC_ACT_SIGMOID> { typedef mix::ActSigmoid type; };
template <typename T, int ACT, typename CT, int N>
__device__ __forceinline__ void value_of(int act, CT (&z)[N]) {
  if constexpr (sizeof(T) == 2 && N == 8 && ACT >= 0) {
    float2 p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = MC_2(z, i);
    Short<ACT>::type::value(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) z[2 * i] = p[i].x, z[2 * i + 1] = p[i].y;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = mix::act_value<CT>(ACT >= 0 ? ACT : act, z[i]);
  }
}
template <typename T, int ACT, typename CT, int N>
__device__ __forceinline__ void slope_of(int act, const CT (&z)[N], CT (&s)[N]) {
  if constexpr (sizeof(T) == 2 && N == 8 && ACT >= 0) {
    float2 p[4], q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = MC_2(z, i);
    Short<ACT>::type::both(p, q);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[2 * i] = q[i].x, s[2 * i + 1] = q[i].y;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = mix::act_slope<CT>(ACT >= 0 ? ACT : act, z[i]);
  }
}

// What the kernel before this one wrote can be read behind this; before it, only what was there when that one began.
__device__ __forceinline__ void behind_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;"); }

// ---- one vector at a time -----------------------------------------------------------------------------------
// The coefficients of a vector's channels: z = (x - mean) scale + shift.  (Statistics of this call are read behind L1.)
template <typename T, typename CT, int N>
struct Coefs {
  CT neg_mean[N], scale[N], shift[N];
  __device__ __forceinline__ void load(const Args& a, long long b, int c, int e) {
    const CT* st = (const CT*)a.stats + 2 * (b * a.G + c / a.Cg);
    const CT w = a.w ? (CT)ldv((const T*)a.w + c) : CT(1);
    neg_mean[e] = -__ldcg(st), scale[e] = __ldcg(st + 1) * w, shift[e] = a.b ? (CT)ldv((const T*)a.b + c) : CT(0);
  }
  // N neighbouring channels from c on (wrapping around); J: of one group
  template <bool J>
  __device__ __forceinline__ void load_all(const Args& a, long long b, int c) {
    if constexpr (J) {
      const CT* st = (const CT*)a.stats + 2 * (b * a.G + c / a.Cg);
      const CT mean = __ldcg(st), rstd = __ldcg(st + 1);
      if (a.w) load_vec<N>((const T*)a.w + c, scale);
      if (a.b) load_vec<N>((const T*)a.b + c, shift);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        neg_mean[e] = -mean, scale[e] = a.w ? scale[e] * rstd : rstd;
        if (!a.b) shift[e] = CT(0);
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        load(a, b, c, e);
        if (++c == a.C) c = 0;
      }
    }
  }
};
template <typename CT, int N>
struct Run {  // of differences from the run's first values
  CT k[N], s[N], q[N];
  __device__ __forceinline__ void start(const CT (&v)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) k[e] = -v[e], s[e] = q[e] = CT(0);
  }
  __device__ __forceinline__ void add(const CT (&v)[N]) {
    CT d[N];
    add_to(d, v, k);
    add_to(s, s, d);
    fma_to(q, d, d, q);
  }
  __device__ __forceinline__ void add_one(CT v, int e) {
    const CT d = v + k[e];
    s[e] += d, q[e] = fma(d, d, q[e]);
  }
  __device__ __forceinline__ Part<CT> part(int e, CT n) const {
    const CT m = n > CT(0) ? s[e] / n : CT(0);
    return Part<CT>{n, m - k[e], fmax(q[e] - s[e] * m, CT(0)) + (q[e] - q[e])};  // (NaN and infinities stay)
  }
};
// n values whose differences from `near` add up to c, their squares to m2.  (A mean from a sum of means is off by several roundings of a
// value far from zero; differences from it give the rest.)
template <typename CT>
__device__ __forceinline__ Part<CT> centred(CT n, CT near, CT c, CT m2) {
  const CT m = n > CT(0) ? c / n : CT(0);
  return Part<CT>{n, near + m, fmax(m2 - c * m, CT(0)) + (m2 - m2)};
}
// What a vector adds to S1 and S2 (without rstd), and its gradient.
template <typename T, int ACT, typename CT, int N>
__device__ __forceinline__ void slope_terms(const Args& a, const Coefs<T, CT, N>& k, CT (&x)[N], CT (&g)[N]) {  // x <- x - mean, g <- dz
  CT z[N], s[N];
  add_to(x, x, k.neg_mean);
  if constexpr (ACT != MC_ACT_NONE) {
    fma_to(z, x, k.scale, k.shift);
    slope_of<T, ACT>(a.act, z, s);
    mul_to(g, g, s);
  }
}
template <typename CT, int N>
struct Sums {
  CT s1[N], s2[N];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int e = 0; e < N; ++e) s1[e] = s2[e] = CT(0);
  }
  __device__ __forceinline__ void add(const CT (&d)[N], const CT (&dz)[N]) {
    add_to(s1, s1, dz);
    fma_to(s2, d, dz, s2);
  }
};
template <typename T, typename CT, int N>
struct Grads {  // gx = dz scale + c0 + (x - mean) c1
  CT c0[N], c1[N];
  __device__ __forceinline__ void load(const Args& a, long long b, int c, int e) {
    const long long group = b * a.G + c / a.Cg;
    const CT rstd = __ldcg((const CT*)a.stats + 2 * group + 1);
    const CT* t = (const CT*)a.coef + 2 * group;
    c0[e] = -rstd * __ldcg(t), c1[e] = -rstd * rstd * __ldcg(t + 1);
  }
  template <bool J>
  __device__ __forceinline__ void load_all(const Args& a, long long b, int c) {
    if constexpr (J) {
      load(a, b, c, 0);
#pragma unroll
      for (int e = 1; e < N; ++e) c0[e] = c0[0], c1[e] = c1[0];
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        load(a, b, c, e);
        if (++c == a.C) c = 0;
      }
    }
  }
  __device__ __forceinline__ void value(const Coefs<T, CT, N>& k, const CT (&d)[N], CT (&dz)[N]) const {
    CT r[N];
    fma_to(r, d, c1, c0);
    fma_to(dz, dz, k.scale, r);
  }
};

// ---- a thread's vectors of a tile ----------------------------------------------------------------------------
// `rows` whole vectors, `step` elements apart, from element `at` on, U at a time.  The first ones are fetched before prepare(), which waits
// for what the arithmetic needs.
struct Span {
  long long at, step;
  int rows;
};
template <int U, typename T, int N, typename F, typename G>
__device__ __forceinline__ void walk(const Span& s, const T* x, G prepare, F f) {
  Raw<T, N> v[U];
  const auto fetch = [&](int r, const T* p) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + u < s.rows) v[u].load(p + u * s.step);
  };
  fetch(0, x + s.at);
  prepare();
  long long i = s.at;
#pragma unroll 1
  for (int r = 0; r < s.rows;) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + u < s.rows) {
        typename Traits<T>::CT w[N];
        v[u].unpack(w);
        f(i + u * s.step, w);
      }
    r += U, i += U * s.step;
    fetch(r, x + i);
  }
}
template <int U, typename T, int N, typename F, typename G>
__device__ __forceinline__ void walk_two(const Span& s, const T* x, const T* gy, G prepare, F f) {
  Raw<T, N> v[U], g[U];
  const auto fetch = [&](int r, long long i) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + u < s.rows) v[u].load(x + i + u * s.step), g[u].load(gy + i + u * s.step);
  };
  fetch(0, s.at);
  prepare();
  long long i = s.at;
#pragma unroll 1
  for (int r = 0; r < s.rows;) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (r + u < s.rows) {
        typename Traits<T>::CT w[N], d[N];
        v[u].unpack(w), g[u].unpack(d);
        f(i + u * s.step, w, d);
      }
    r += U, i += U * s.step;
    fetch(r, i);
  }
}
// Vectors on their way, of one tensor and of two.  (2 and 1: 192 and 352 us for 64 x 10 242 x 256 bf16, 181 and 294 with these; of two
// tensors 2: 300 us, and 236 instead of 194 for 32 x 100 x 200 x 128 in groups of four channels.)
constexpr int ONE = 4, BOTH = 4;
template <typename T, int ACT, typename CT, int N>
__device__ __forceinline__ void output(const Args& a, const Coefs<T, CT, N>& k, CT (&v)[N]) {
  add_to(v, v, k.neg_mean);
  fma_to(v, v, k.scale, k.shift);
  value_of<T, ACT>(a.act, v);
}

// ---- channels-last ------------------------------------------------------------------------------------
// R pixels are V vectors of N elements; vector j of such a row of pixels holds the same channels everywhere.  A thread keeps one
// vector (of a column of 256) and takes every lanes-th row of the tile.
template <int N>
struct Place {
  Span span;                // this thread's whole vectors
  long long end, tail;      // flat: behind the tile; the vector of the row that the tile's end cuts, or end
  int col, j, lane, vc;     // column, vector of the row, which of the rows, vectors of the column
  __device__ int channel(const Args& a) const {  // of the vector's first element
    const long long c = (long long)j * N;
    return a.R == 1 ? (int)c : (int)(c % a.C);
  }
  __device__ Place(const Args& a, long long b, int tile) {
    col = a.cols == 1 ? 0 : tile % a.cols;
    const long long t = a.cols == 1 ? tile : tile / a.cols, image = b * a.S * a.C, row0 = image + t * a.px * a.C, left = a.S - t * a.px;
    end = row0 + (left < a.px ? left : a.px) * a.C;
    vc = min(256, a.V - col * 256);
    lane = threadIdx.x / vc;
    j = col * 256 + threadIdx.x % vc;
    const int row = a.V * N, whole = (int)((end - row0) / row);
    span.step = (long long)a.lanes * row;
    span.at = row0 + (long long)lane * row + j * N;
    span.rows = lane < a.lanes && whole > lane ? (whole - lane + a.lanes - 1) / a.lanes : 0;
    tail = end;
    if (a.R > 1 && lane < a.lanes && whole % a.lanes == lane) {
      tail = row0 + (long long)whole * row + j * N;
      if (tail > end) tail = end;
    }
  }
};
// Whose sums come first in the part of a column, and where those of group g stand.
__device__ __forceinline__ int first_channel(const Args& a, int col) { return a.chans < a.C ? (int)((long long)col * a.column % a.C) : 0; }
__device__ __forceinline__ int first_group(const Args& a, int col) { return a.grps < a.G ? (int)((long long)col * a.column % a.C) / a.Cg : 0; }
__device__ __forceinline__ int group_slot(const Args& a, int col, int g) {
  const int s = g - first_group(a, col);
  return s < 0 ? s + a.G : s;
}
template <typename CT, int N> union Shared {
  Part<CT> part[N][THREADS];
  Two<CT> two[N][THREADS];
};

template <typename T, bool J, typename CT, int N>
__device__ __forceinline__ void rows_stats(const Args& a, Shared<CT, N>& sm, long long b, int tile) {
  const T* x = (const T*)a.x;
  const Place<N> p(a, b, tile);
  const int rows = p.span.rows;
  Run<CT, N> run;
  CT first[N];
  if (rows) load_vec<N>(x + p.span.at, first);
  else load_in<N>(x, p.tail, 0, p.end, first);
  walk<ONE, T, N>(p.span, x, [&] { run.start(first); }, [&](long long, CT (&v)[N]) { run.add(v); });
  if (p.tail < p.end) {
    CT v[N];
    load_in<N>(x, p.tail, 0, p.end, v);
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (p.tail + e < p.end) run.add_one(v[e], e);
  }
  if constexpr (J) {
    Part<CT> q[N];
    CT mean = CT(0), m2 = CT(0);
#pragma unroll
    for (int e = 0; e < N; ++e) q[e] = run.part(e, (CT)rows), mean += q[e].mean - q[0].mean;
    mean /= CT(N);  // (from the first channel's mean)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const CT d = q[e].mean - q[0].mean - mean;
      m2 += q[e].m2 + (CT)rows * d * d;
    }
    sm.part[0][threadIdx.x] = Part<CT>{(CT)rows * CT(N), q[0].mean + mean, m2};
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) sm.part[e][threadIdx.x] = run.part(e, (CT)(rows + (p.tail + e < p.end ? 1 : 0)));
  }
  __syncthreads();
  // what the threads of a group's channels left, a few threads to a group
  Part<CT>* out = (Part<CT>*)a.part + (b * a.tiles + tile) * a.grps;
  const auto groups = [&](auto wide) {
    constexpr bool WIDE = decltype(wide)::value;
    const int each = J ? a.Cg / N : a.Cg * a.R, entries = WIDE ? min(each, J ? 256 : a.column) : each * a.lanes;
    const int sub = entries > 16 ? 32 : entries > 8 ? 16 : entries > 4 ? 8 : 4, me = threadIdx.x % sub;
    const int g0 = WIDE ? first_group(a, p.col) : 0;
    for (int s0 = 0; s0 < a.grps; s0 += THREADS / sub) {
      const int slot = s0 + threadIdx.x / sub;
      const bool on = slot < a.grps;
      int g = slot + g0;
      if (WIDE && g >= a.G) g -= a.G;
      // f(part) of every one of this group's in the column, this thread's share of them
      const auto each_entry = [&](auto f) {
        if (!on) return;
        if constexpr (!WIDE) {
          for (int i = me; i < entries; i += sub) {
            const int l = i / each, k = i - l * each;
            int e = 0, j;
            if constexpr (J) {
              j = g * each + k;
            } else {
              const int rr = k / a.Cg, at = rr * a.C + g * a.Cg + k - rr * a.Cg;
              j = at / N, e = at % N;
            }
            const Part<CT> v = sm.part[e][l * p.vc + j];
            if (v.n > CT(0)) f(v);
          }
        } else {  // (one lane: the group's elements in each pixel of the row, as far as the column reaches)
          const int from = p.col * a.column, to = from + p.vc * N;
          for (int r = 0; r < a.R; ++r) {
            const int lo = max(r * a.C + g * a.Cg, from) - from, hi = min(r * a.C + (g + 1) * a.Cg, to) - from;
            for (int i = (J ? lo / N : lo) + me; i < (J ? hi / N : hi); i += sub) {
              const Part<CT> v = J ? sm.part[0][i] : sm.part[i % N][i / N];
              if (v.n > CT(0)) f(v);
            }
          }
        }
      };
      CT cnt = CT(0), sum = CT(0), m2 = CT(0);
      each_entry([&](const Part<CT>& w) { cnt += w.n, sum += w.n * w.mean; });
      for (int o = sub / 2; o; o >>= 1) cnt += __shfl_xor_sync(~0u, cnt, o), sum += __shfl_xor_sync(~0u, sum, o);
      const CT mean = cnt > CT(0) ? sum / cnt : CT(0);
      CT c = CT(0);  // what the roundings of that sum left of the differences
      each_entry([&](const Part<CT>& w) {
        const CT d = w.mean - mean;
        m2 += w.m2 + w.n * d * d, c += w.n * d;
      });
      for (int o = sub / 2; o; o >>= 1) m2 += __shfl_xor_sync(~0u, m2, o), c += __shfl_xor_sync(~0u, c, o);
      if (on && me == 0) out[slot] = centred(cnt, mean, c, m2);
    }
  };
  a.wide ? groups(std::true_type()) : groups(std::false_type());
}

template <typename T, int ACT, bool J, typename CT, int N>
__device__ __forceinline__ void rows_apply(const Args& a, long long b, int tile) {
  const Place<N> p(a, b, tile);
  const T* x = (const T*)a.x;
  T* y = (T*)a.y;
  Coefs<T, CT, N> k;
  walk<ONE, T, N>(
      p.span, x,
      [&] {
        behind_previous_kernel();
        k.template load_all<J>(a, b, p.channel(a));
      },
      [&](long long i, CT (&v)[N]) {
        output<T, ACT>(a, k, v);
        store_vec<N>(y + i, v);
      });
  if (p.tail < p.end) {
    CT v[N];
    load_in<N>(x, p.tail, 0, p.end, v);
    output<T, ACT>(a, k, v);
    store_in<N>(y, p.tail, 0, p.end, v);
  }
}

template <typename T, int ACT, bool J, typename CT, int N>
__device__ __forceinline__ void rows_sums(const Args& a, Shared<CT, N>& sm, long long b, int tile) {
  const T *x = (const T*)a.x, *gy = (const T*)a.gy;
  const Place<N> p(a, b, tile);
  Sums<CT, N> sums;
  Coefs<T, CT, N> k;
  sums.clear();
  walk_two<BOTH, T, N>(
      p.span, x, gy, [&] { k.template load_all<J>(a, b, p.channel(a)); },
      [&](long long, CT (&v)[N], CT (&g)[N]) { slope_terms<T, ACT>(a, k, v, g), sums.add(v, g); });
  if (p.tail < p.end) {
    CT v[N], g[N];
    load_in<N>(x, p.tail, 0, p.end, v), load_in<N>(gy, p.tail, 0, p.end, g);
    slope_terms<T, ACT>(a, k, v, g);
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (p.tail + e < p.end) sums.s1[e] += g[e], sums.s2[e] += v[e] * g[e];
  }
#pragma unroll
  for (int e = 0; e < N; ++e) sm.two[e][threadIdx.x] = Two<CT>{sums.s1[e], sums.s2[e]};
  __syncthreads();
  const bool once = a.C > a.column;  // each channel of a column is in one place of it
  const int entries = once ? 1 : a.R * a.lanes;
  // threads that share a channel, as many as the channels leave
  const int sub = a.C >= 128 ? 1 : a.C >= 32 ? 8 : 32;
  Two<CT>* out = (Two<CT>*)a.part + (b * a.tiles + tile) * a.chans;
  for (int s0 = 0; s0 < a.chans; s0 += THREADS / sub) {
    const int slot = s0 + threadIdx.x / sub;
    int c = slot + first_channel(a, p.col);
    if (c >= a.C) c -= a.C;
    CT u = CT(0), v = CT(0);
    if (slot < a.chans)
      for (int i = threadIdx.x % sub; i < entries; i += sub) {
        const int l = a.R == 1 ? i : i / a.R, r = i - l * a.R, f = once ? slot : r * a.C + c, j = once ? f / N : f / N - p.col * 256;
        if (j >= 0 && j < p.vc) {
          const Two<CT> t = sm.two[f % N][l * p.vc + j];
          u += t.a, v += t.b;
        }
      }
    for (int o = sub / 2; o; o >>= 1) u += __shfl_xor_sync(~0u, u, o), v += __shfl_xor_sync(~0u, v, o);
    if (slot < a.chans && threadIdx.x % sub == 0)
      out[slot] = Two<CT>{u, v * __ldcg((const CT*)a.stats + 2 * (b * a.G + c / a.Cg) + 1)};
  }
}

template <typename T, int ACT, bool J, typename CT, int N>
__device__ __forceinline__ void rows_grad(const Args& a, long long b, int tile) {
  const Place<N> p(a, b, tile);
  const T *x = (const T*)a.x, *gy = (const T*)a.gy;
  T* gx = (T*)a.gx;
  Coefs<T, CT, N> k;
  Grads<T, CT, N> q;
  const auto grad = [&](CT (&v)[N], CT (&g)[N]) { slope_terms<T, ACT>(a, k, v, g), q.value(k, v, g); };
  walk_two<BOTH, T, N>(
      p.span, x, gy,
      [&] {
        behind_previous_kernel();
        k.template load_all<J>(a, b, p.channel(a)), q.template load_all<J>(a, b, p.channel(a));
      },
      [&](long long i, CT (&v)[N], CT (&g)[N]) {
        grad(v, g);
        store_vec<N>(gx + i, g);
      });
  if (p.tail < p.end) {
    CT v[N], g[N];
    load_in<N>(x, p.tail, 0, p.end, v), load_in<N>(gy, p.tail, 0, p.end, g);
    grad(v, g);
    store_in<N>(gx, p.tail, 0, p.end, g);
  }
}

// ---- planes ---------------------------------------------------------------------------------------------
// A warp takes segments of planes; vectors start on 16 bytes wherever the plane does (all tensors lie alike).
template <int N>
struct Segment {
  long long lo, hi;  // flat: first element, behind the last
  long long first, last;  // whole vectors lie between them
  int c;
  Span span;
  __device__ Segment(const Args& a, long long b, int item) {
    const int plane = item / a.segs, k = item - plane * a.segs, lane = threadIdx.x % 32;
    c = plane;
    lo = (b * a.C + plane) * a.S + (long long)k * SEGMENT;
    hi = lo + min((long long)SEGMENT, a.S - (long long)k * SEGMENT);
    first = (lo + N - 1) / N * N, last = hi / N * N;
    const int vectors = last > first ? (int)((last - first) / N) : 0;
    span.at = first + lane * N, span.step = 32 * N, span.rows = vectors > lane ? (vectors - lane + 31) / 32 : 0;
  }
  // f(i): the vector that an end of the segment cuts, in the lane that takes it
  template <typename F>
  __device__ __forceinline__ void edges(F f) const {
    const int lane = threadIdx.x % 32;
    if (lane == 0 && first > lo) f(first - N);
    if (lane == 31 && last < hi && last >= first) f(last);
  }
};
// items of a warp in a tile
template <typename F>
__device__ __forceinline__ void each_item(const Args& a, int tile, F f) {
  const int first = (tile * WARPS + threadIdx.x / 32) * a.per, all = a.C * a.segs;
  for (int k = 0; k < a.per && first + k < all; ++k) f(first + k);
}
template <typename CT, int N>
__device__ __forceinline__ void spread(CT (&v)[N]) {
#pragma unroll
  for (int e = 1; e < N; ++e) v[e] = v[0];
}
template <typename T, typename CT, int N>
__device__ __forceinline__ void planes_stats(const Args& a, long long b, int tile) {
  const T* x = (const T*)a.x;
  each_item(a, tile, [&](int item) {
    const Segment<N> g(a, b, item);
    Run<CT, N> run;
    CT k[N], n = CT(g.span.rows) * CT(N);
    // (a value of the lane's own run: its first vector's first, or where it has only an end of the segment, that end's)
    k[0] = (CT)ldv(x + (threadIdx.x % 32 ? min(g.hi - 1, g.span.at) : g.lo));
    spread(k);
    walk<ONE, T, N>(g.span, x, [&] { run.start(k); }, [&](long long, CT (&v)[N]) { run.add(v); });
    g.edges([&](long long i) {
      CT v[N];
      load_in<N>(x, i, g.lo, g.hi, v);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i + e >= g.lo && i + e < g.hi) run.add_one(v[e], e), n += CT(1);
    });
    CT s = CT(0), q = CT(0);
#pragma unroll
    for (int e = 0; e < N; ++e) s += run.s[e], q += run.q[e];
    const CT m = n > CT(0) ? s / n : CT(0);
    CT m2 = fmax(q - s * m, CT(0)) + (q - q);
    const CT mean = k[0] + m, cnt = warp_sum(n), all = warp_sum(n > CT(0) ? n * mean : CT(0)) / cnt;
    const CT d = mean - all, c = warp_sum(n > CT(0) ? n * d : CT(0));
    m2 = warp_sum(n > CT(0) ? m2 + n * d * d : CT(0));
    if (threadIdx.x % 32 == 0) ((Part<CT>*)a.part)[b * a.C * a.segs + item] = centred(cnt, all, c, m2);
  });
}
template <typename T, int ACT, typename CT, int N>
__device__ __forceinline__ void planes_apply(const Args& a, long long b, int tile) {
  const T* x = (const T*)a.x;
  T* y = (T*)a.y;
  each_item(a, tile, [&](int item) {
    const Segment<N> g(a, b, item);
    Coefs<T, CT, N> k;
    walk<ONE, T, N>(
        g.span, x,
        [&] {
          behind_previous_kernel();
          k.load(a, b, g.c, 0);
          spread(k.neg_mean), spread(k.scale), spread(k.shift);
        },
        [&](long long i, CT (&v)[N]) {
          output<T, ACT>(a, k, v);
          store_vec<N>(y + i, v);
        });
    g.edges([&](long long i) {
      CT v[N];
      load_in<N>(x, i, g.lo, g.hi, v);
      output<T, ACT>(a, k, v);
      store_in<N>(y, i, g.lo, g.hi, v);
    });
  });
}
template <typename T, int ACT, typename CT, int N>
__device__ __forceinline__ void planes_sums(const Args& a, long long b, int tile) {
  const T *x = (const T*)a.x, *gy = (const T*)a.gy;
  each_item(a, tile, [&](int item) {
    const Segment<N> g(a, b, item);
    Coefs<T, CT, N> k;
    Sums<CT, N> sums;
    sums.clear();
    walk_two<BOTH, T, N>(
        g.span, x, gy,
        [&] {
          k.load(a, b, g.c, 0);
          spread(k.neg_mean), spread(k.scale), spread(k.shift);
        },
        [&](long long, CT (&v)[N], CT (&d)[N]) { slope_terms<T, ACT>(a, k, v, d), sums.add(v, d); });
    g.edges([&](long long i) {
      CT v[N], d[N];
      load_in<N>(x, i, g.lo, g.hi, v), load_in<N>(gy, i, g.lo, g.hi, d);
      slope_terms<T, ACT>(a, k, v, d);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i + e >= g.lo && i + e < g.hi) sums.s1[e] += d[e], sums.s2[e] += v[e] * d[e];
    });
    CT s1 = CT(0), s2 = CT(0);
#pragma unroll
    for (int e = 0; e < N; ++e) s1 += sums.s1[e], s2 += sums.s2[e];
    s1 = warp_sum(s1), s2 = warp_sum(s2);
    if (threadIdx.x % 32 == 0)
      ((Two<CT>*)a.part)[b * a.C * a.segs + item] = Two<CT>{s1, s2 * __ldcg((const CT*)a.stats + 2 * (b * a.G + g.c / a.Cg) + 1)};
  });
}
template <typename T, int ACT, typename CT, int N>
__device__ __forceinline__ void planes_grad(const Args& a, long long b, int tile) {
  const T *x = (const T*)a.x, *gy = (const T*)a.gy;
  T* gx = (T*)a.gx;
  each_item(a, tile, [&](int item) {
    const Segment<N> g(a, b, item);
    Coefs<T, CT, N> k;
    Grads<T, CT, N> q;
    walk_two<BOTH, T, N>(
        g.span, x, gy,
        [&] {
          behind_previous_kernel();
          k.load(a, b, g.c, 0), q.load(a, b, g.c, 0);
          spread(k.neg_mean), spread(k.scale), spread(k.shift), spread(q.c0), spread(q.c1);
        },
        [&](long long i, CT (&v)[N], CT (&d)[N]) {
          slope_terms<T, ACT>(a, k, v, d), q.value(k, v, d);
          store_vec<N>(gx + i, d);
        });
    g.edges([&](long long i) {
      CT v[N], d[N];
      load_in<N>(x, i, g.lo, g.hi, v), load_in<N>(gy, i, g.lo, g.hi, d);
      slope_terms<T, ACT>(a, k, v, d), q.value(k, v, d);
      store_in<N>(gx, i, g.lo, g.hi, d);
    });
  });
}

// ---- between the two readings ---------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ Two<T> peek(const Two<T>* p) {  // (behind L1)
  return Two<T>{__ldcg(&p->a), __ldcg(&p->b)};
}
// Statistics of a group by `sub` threads, in double: with d the distance of a part's mean from that of the part of the group's first
// value, M2 = sum m2 + sum n d^2 - (sum n d)^2 / N  (one pass, its loads independent of each other).
template <typename CT>
__global__ void __launch_bounds__(THREADS) stats_kernel(const __grid_constant__ Args a, bool rows, int sub) {
  let_next_kernel_start();
  behind_previous_kernel();
  const long long group = (blockIdx.x * (long long)THREADS + threadIdx.x) / sub;
  const long long b = group / a.G;
  const int g = (int)(group % a.G), me = threadIdx.x % sub;
  double n = 0, s = 0, q = 0, base = 0;
  const auto merge = [&](const Part<CT>* p) {
    const double k = __ldcg(&p->n), m = __ldcg(&p->mean), m2 = __ldcg(&p->m2), d = k > 0 ? m - base : 0.0;
    n += k, s += k * d, q += m2 + k * d * d;
  };
  if (b < a.B && !rows) {
    const Part<CT>* part = (const Part<CT>*)a.part + (b * a.C + (long long)g * a.Cg) * a.segs;
    base = __ldcg(&part->mean);
#pragma unroll 4
    for (int i = me; i < a.Cg * a.segs; i += sub) merge(part + i);
  } else if (b < a.B) {
    const Part<CT>* part = (const Part<CT>*)a.part + b * a.tiles * a.grps;
    const auto at = [&](int col) { return part + (long long)col * a.grps + group_slot(a, col, g); };
    // (the first tile's column that holds the group's first channel; parts of other columns may be empty)
    base = __ldcg(&at(a.wide ? g * a.Cg / a.column : 0)->mean);
    if (a.C <= a.column) {  // every part has room for every group
      const Part<CT>* p = at(0);
#pragma unroll 4
      for (int i = me; i < a.tiles; i += sub) merge(p + (long long)i * a.grps);
    } else {  // the columns that hold any of the group, pixel by pixel of a row
      const long long step = (long long)a.cols * a.grps;
      const int count = a.tiles / a.cols;
      int done = 0;
      for (int r = 0; r < a.R; ++r) {
        const int f = r * a.C + g * a.Cg, lo = max(f / a.column, done), hi = min((f + a.Cg - 1) / a.column + 1, a.cols), wide = hi - lo;
        if (wide <= 0) continue;
        for (long long i = me; i < (long long)wide * count; i += sub) merge(at(lo + (int)(i % wide)) + i / wide * step);
        done = hi;
      }
    }
  }
  for (int o = sub / 2; o; o >>= 1) n += __shfl_xor_sync(~0u, n, o), s += __shfl_xor_sync(~0u, s, o), q += __shfl_xor_sync(~0u, q, o);
  if (b < a.B && threadIdx.x % sub == 0) {
    CT* st = (CT*)a.stats + 2 * group;
    const double var = fmax((q - s / n * s) / n, 0.0) + (q - q);  // (NaN and infinities stay)
    st[0] = (CT)(base + s / n), st[1] = (CT)(1.0 / sqrt(var + a.eps));
  }
}
// S1, S2 of every channel of an image, `sub` threads to a channel, and what a group's gradients subtract: one block per group
template <typename T>
__global__ void __launch_bounds__(THREADS) coef_kernel(const __grid_constant__ Args a, bool rows, int sub) {
  typedef typename Traits<T>::CT CT;
  __shared__ double sm[2][WARPS];
  let_next_kernel_start();
  behind_previous_kernel();
  const long long b = blockIdx.x / a.G;
  const bool once = rows && a.C > a.column;  // a column has room for some channels only; else each part has a place for every one
  const int g = (int)(blockIdx.x % a.G);
  Two<double>* sums = (Two<double>*)a.sums + b * a.C;
  double gu = 0, gv = 0;
  for (int i0 = 0; i0 < a.Cg; i0 += THREADS / sub) {
    const int i = i0 + threadIdx.x / sub, c = g * a.Cg + i;
    double u = 0, v = 0;
    const auto add = [&](const Two<CT>* part, int count, long long step) {
#pragma unroll 8
      for (int k = threadIdx.x % sub; k < count; k += sub) {
        const Two<CT> t = peek(part + k * step);
        u += t.a, v += t.b;
      }
    };
    if (i < a.Cg && !once) {
      const int count = rows ? a.tiles : a.segs;
      add((const Two<CT>*)a.part + (rows ? b * count * a.C + c : (b * a.C + c) * count), count, rows ? a.C : 1);
    } else if (i < a.Cg) {
      for (int r = 0; r < a.R; ++r) {
        const int f = r * a.C + c, col = f / a.column;
        if (col >= a.cols) break;
        add((const Two<CT>*)a.part + (b * a.tiles + col) * a.chans + f - col * a.column, a.tiles / a.cols, (long long)a.cols * a.chans);
      }
    }
    for (int o = sub / 2; o; o >>= 1) u += __shfl_xor_sync(~0u, u, o), v += __shfl_xor_sync(~0u, v, o);
    if (i < a.Cg && threadIdx.x % sub == 0) {
      sums[c] = Two<double>{u, v};
      const double w = a.w ? (double)ldv((const T*)a.w + c) : 1.0;
      gu += w * u, gv += w * v;
    }
  }
  gu = warp_sum(gu), gv = warp_sum(gv);
  if (threadIdx.x % 32 == 0) sm[0][threadIdx.x / 32] = gu, sm[1][threadIdx.x / 32] = gv;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < WARPS; ++i) gu += sm[0][i], gv += sm[1][i];
    const double n = (double)a.Cg * (double)a.S;
    ((Two<CT>*)a.coef)[blockIdx.x] = Two<CT>{(CT)(gu / n), (CT)(gv / n)};
  }
}
// gradients of the parameters from all images' sums: eight threads to a channel
template <typename T>
__device__ __forceinline__ void param_grads(const Args& a, int block) {
  typedef typename Traits<T>::CT CT;
  const int c = block * (THREADS / 8) + threadIdx.x / 8;
  double u = 0, v = 0;
  if (c < a.C) {
#pragma unroll 4
    for (long long b = threadIdx.x % 8; b < a.B; b += 8) {
      const Two<double> t = peek((const Two<double>*)a.sums + b * a.C + c);
      u += t.a, v += t.b;
    }
  }
  for (int o = 4; o; o >>= 1) u += __shfl_xor_sync(~0u, u, o), v += __shfl_xor_sync(~0u, v, o);
  if (c < a.C && threadIdx.x % 8 == 0) {
    if (a.gb) stv((T*)a.gb + c, (CT)u);
    if (a.gw) stv((T*)a.gw + c, (CT)v);
  }
}

// ---- the first and the third launch -----------------------------------------------------------------------------
template <typename T, int N, bool ROWS, bool BWD, int ACT, bool J>
__global__ void __launch_bounds__(THREADS) first_kernel(const __grid_constant__ Args a) {
  typedef typename Traits<T>::CT CT;
  __shared__ Shared<CT, ROWS ? N : 1> sm;
  let_next_kernel_start();
  const long long b = blockIdx.x / a.tiles;
  const int tile = (int)(blockIdx.x % a.tiles);
  if constexpr (BWD) {
    if constexpr (ROWS) rows_sums<T, ACT, J, CT, N>(a, sm, b, tile);
    else planes_sums<T, ACT, CT, N>(a, b, tile);
  } else {
    if constexpr (ROWS) rows_stats<T, J, CT, N>(a, sm, b, tile);
    else planes_stats<T, CT, N>(a, b, tile);
  }
}
template <typename T, int N, bool ROWS, bool BWD, int ACT, bool J>
__global__ void __launch_bounds__(THREADS) second_kernel(const __grid_constant__ Args a) {
  typedef typename Traits<T>::CT CT;
  if (BWD && blockIdx.x < a.param_blocks) {
    behind_previous_kernel();
    param_grads<T>(a, blockIdx.x);
    return;
  }
  const unsigned t = gridDim.x - 1 - blockIdx.x;
  const long long b = t / a.tiles;
  const int tile = (int)(t % a.tiles);
  if constexpr (BWD) {
    if constexpr (ROWS) rows_grad<T, ACT, J, CT, N>(a, b, tile);
    else planes_grad<T, ACT, CT, N>(a, b, tile);
  } else {
    if constexpr (ROWS) rows_apply<T, ACT, J, CT, N>(a, b, tile);
    else planes_apply<T, ACT, CT, N>(a, b, tile);
  }
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
static int plan(const mc_norm_desc* d, Plan& p) {
  Args& a = p.a;
  a.S = d->S, a.B = d->B, a.C = d->C, a.G = d->groups, a.Cg = d->C / d->groups, a.act = d->act, a.eps = d->eps;
  const int N = 16 / esize(d->dtype), ct = csize(d->dtype);
  p.rows = d->layout == MC_NHWC || d->S == 1;
  long long tiles;
  if (p.rows) {
    p.vec = d->B == 1 || d->S * d->C % N == 0;  // every image starts on 16 bytes
    const int n = p.vec ? N : 1;
    a.R = n / gcd(n, d->C), a.V = (int)((long long)a.R * d->C / n);
    a.joined = a.R == 1 && n > 1 && a.Cg % n == 0;
    a.cols = (a.V + 255) / 256, a.column = 256 * n, a.wide = a.V > 256;
    if (a.wide && d->S < a.R) a.cols = (int)((d->S * d->C + a.column - 1) / a.column);  // (of a row that the only image does not fill)
    a.chans = d->C > a.column ? a.column : d->C;
    a.grps = d->C > a.column && a.column / a.Cg + 2 < a.G ? a.column / a.Cg + 2 : a.G;
    a.lanes = a.wide ? 1 : 256 / a.V;
    const long long step = (long long)a.lanes * a.R;
    // A thread's rows: as many as a run holds, fewer where that leaves an SM less than eight blocks.  (At most 16, 8: 64 x 10 242 x 256
    // bf16 forward 196, 230 us instead of 181; backward, with two vectors of either tensor on their way, 309, 350 instead of 300.)
    long long k = d->B * d->S / step * a.cols / (148 * 8);
    k = k < 1 ? 1 : k > RUN ? RUN : k;
    a.px = (int)(step * k);
    tiles = (d->S + a.px - 1) / a.px * a.cols;
    p.part_f = (size_t)(d->B * tiles) * a.grps * 3 * ct, p.part_b = (size_t)(d->B * tiles) * a.chans * 2 * ct;
  } else {
    p.vec = true;
    a.segs = (int)((d->S + SEGMENT - 1) / SEGMENT);
    const long long items = (long long)d->C * a.segs;
    if (items >= (1ll << 30)) return MC_ERR_TOO_LARGE;
    // small planes: several to a warp, about a segment in all, as long as there are blocks enough
    long long per = d->S >= SEGMENT ? 1 : SEGMENT / d->S, most = d->B * items / (148 * 8 * WARPS);
    per = per > most ? most : per;
    a.per = (int)(per < 1 ? 1 : per);
    tiles = (items + WARPS * a.per - 1) / (WARPS * a.per);
    p.part_f = (size_t)(d->B * items) * 3 * ct, p.part_b = (size_t)(d->B * items) * 2 * ct;
  }
  p.sums = (size_t)d->B * d->C * 16, p.coef = (size_t)d->B * d->groups * 2 * ct;
  // (a grid's blocks: tiles and blocks of parameter gradients, groups)
  if (d->B * tiles >= (1ll << 31) - (1 << 20) || d->B * d->groups >= (1ll << 31)) return MC_ERR_TOO_LARGE;
  a.tiles = (int)tiles, p.blocks = (unsigned)(d->B * tiles);
  return MC_OK;
}
static bool on(const void* p, size_t n) { return (uintptr_t)p % n == 0; }
// Threads that share one of the sums of `count` parts, where there are `sums` of them.
static int sharers(long long sums, int count) {
  int sub = 1;
  while (sub < 32 && sub < count && sums * sub < 148 * THREADS) sub *= 2;
  return sub;
}
template <typename... A>
static int launch(void (*kern)(A...), unsigned blocks, bool behind, cudaStream_t st, A... args) {
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = behind ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kern, args...) != cudaSuccess) return MC_ERR_LAUNCH;
  MC_COUNT(1);
  return MC_OK;
}
template <typename T, int N, bool ROWS, bool BWD, int ACT, bool J>
static int three(const Plan& p, cudaStream_t st) {
  typedef typename Traits<T>::CT CT;
  Args a = p.a;
  int rc = launch(first_kernel<T, N, ROWS, BWD, BWD ? ACT : 0, J>, p.blocks, false, st, (Args)a);
  if (rc) return rc;
  const long long groups = a.B * a.G;
  if (BWD) {
    int sub = sharers(a.B * a.C, !ROWS ? a.segs : a.C > a.column ? a.tiles / a.cols : a.tiles);
    while (sub < 32 && sub * a.Cg < THREADS) sub *= 2;  // (a block has one group's channels only)
    rc = launch(coef_kernel<T>, (unsigned)groups, true, st, (Args)a, (bool)ROWS, (int)sub);
    a.param_blocks = a.gw || a.gb ? (a.C + THREADS / 8 - 1) / (THREADS / 8) : 0;
  } else {
    const int sub = sharers(groups, ROWS ? a.tiles : a.Cg * a.segs);
    rc = launch(stats_kernel<CT>, (unsigned)((groups * sub + THREADS - 1) / THREADS), true, st, (Args)a, (bool)ROWS, (int)sub);
  }
  const unsigned blocks = a.param_blocks + (BWD && !a.gx ? 0 : p.blocks);
  if (rc || !blocks) return rc;
  return launch(second_kernel<T, N, ROWS, BWD, ACT, J>, blocks, true, st, (Args)a);
}
// bf16 and float32 vectors have a kernel for each activation
template <typename T, int N, bool ROWS, bool BWD, bool J>
static int by_act(const Plan& p, cudaStream_t st) {
  if constexpr (sizeof(T) == 8 || N == 1) {
    return three<T, N, ROWS, BWD, -1, J>(p, st);
  } else {
    switch (p.a.act) {
      case MC_ACT_RELU: return three<T, N, ROWS, BWD, MC_ACT_RELU, J>(p, st);
      case MC_ACT_GELU: return three<T, N, ROWS, BWD, MC_ACT_GELU, J>(p, st);
      case MC_ACT_GELU_TANH: return three<T, N, ROWS, BWD, MC_ACT_GELU_TANH, J>(p, st);
      case MC_ACT_SILU: return three<T, N, ROWS, BWD, MC_ACT_SILU, J>(p, st);
      case MC_ACT_SIGMOID: return three<T, N, ROWS, BWD, MC_ACT_SIGMOID, J>(p, st);
      default: return three<T, N, ROWS, BWD, MC_ACT_NONE, J>(p, st);
    }
  }
}
template <typename T, bool BWD>
static int run_typed(const Plan& p, cudaStream_t st) {
  constexpr int N = Vec<T>::N;
  if (!p.rows) return by_act<T, N, false, BWD, false>(p, st);
  if (!p.vec) return by_act<T, 1, true, BWD, false>(p, st);
  return p.a.joined ? by_act<T, N, true, BWD, true>(p, st) : by_act<T, N, true, BWD, false>(p, st);
}
template <bool BWD>
static int run(const mc_norm_desc* d, Plan& p, cudaStream_t st) {
  if (!on(p.a.w, 16) || !on(p.a.b, 16)) p.a.joined = false;
  if (d->dtype == MC_F32) return run_typed<float, BWD>(p, st);
  if (d->dtype == MC_F64) return run_typed<double, BWD>(p, st);
  return run_typed<bf16, BWD>(p, st);
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
  if (!ws || ws_bytes < mc_group_norm_workspace_bytes(d, MC_PHASE_FORWARD)) return MC_ERR_WORKSPACE;
  p.a.x = x, p.a.w = w, p.a.b = bias, p.a.y = y, p.a.stats = stats;
  p.a.part = ws;
  return norm::run<false>(d, p, (cudaStream_t)stream);
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
  if (!gx && !gw && !gb) return MC_OK;
  char* at = (char*)ws;
  p.a.x = x, p.a.w = w, p.a.b = bias, p.a.gy = gy, p.a.gx = gx, p.a.gw = gw, p.a.gb = gb, p.a.stats = (void*)stats;
  p.a.part = at, at += norm::up256(p.part_b);
  p.a.sums = at, at += norm::up256(p.sums);
  p.a.coef = at;
  return norm::run<true>(d, p, (cudaStream_t)stream);
}

}  // extern "C"
