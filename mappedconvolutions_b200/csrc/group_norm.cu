// Group normalisation with an activation, both layouts, forward and backward.
//
//   over the n = C / G * S elements of group g of image b:  mu, var;  rstd = 1 / sqrt(var + eps)
//   xhat = (x - mu) rstd,  z = xhat w_c + b_c,  y = act(z)
//   dz = gy act'(z),  S1 = sum_s dz,  S2 = sum_s dz xhat for every channel of an image,
//   gx = rstd (dz w_c - (sum_c w_c S1 + xhat sum_c w_c S2) / n),  gw_c = sum_b S2,  gb_c = sum_b S1
//
// Bound: HBM.  An image's tiles are read twice, first for the sums, then for the output; one launch does both, and the second
// reading of an image follows `lag` images behind its first, so that it comes from L2.  Blocks draw tickets: the tiles in the order in which they
// are to be done.  Whoever finishes the last first reading of an image adds its tiles' results up, in their order, and raises the
// image's flag; a second reading waits for it.  A ticket waits for tickets before it only, and those are held by blocks that run: no
// order of the blocks can leave a wait unanswered.
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

// Device status word: 0, or the code of the first bounded wait that ran out (mc_device_status).
__device__ int g_status = 0;
constexpr int WAIT_CODE = 0x161;
constexpr long long WAIT_LIMIT_CYCLES = 4000000000LL;

template <typename CT> struct Part { CT n, mean, m2; };
template <typename CT> struct Two { CT a, b; };

struct Args {
  const void *x, *w, *b, *gy;
  void *y, *gx, *gw, *gb;
  void* stats;  // mean and rstd of every group of every image
  void* part;   // what a tile leaves
  void* sums;   // backward: S1, S2 of every channel of every image
  void* coef;   // backward: the two sums over a group, divided by n
  unsigned* ticket;
  unsigned *images_done, *arrived, *ready;  // (the latter two: of every image)
  long long S, B;
  int C, G, Cg, act;
  double eps;
  int tiles;  // of an image
  int lag;    // images
  unsigned tickets;
  // channels-last: tiles of `px` pixels, in columns of at most 256 vectors
  int px, cols, V, R, lanes;
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

// ---- one vector at a time -----------------------------------------------------------------------------------
// The coefficients of a vector's channels: z = (x - mean) scale + shift.  (Written by other SMs a moment ago: read behind L1.)
template <typename T, typename CT, int N>
struct Coefs {
  CT neg_mean[N], scale[N], shift[N];
  __device__ __forceinline__ void load(const Args& a, long long b, int c, int e) {
    const CT* st = (const CT*)a.stats + 2 * (b * a.G + c / a.Cg);
    const CT w = a.w ? (CT)ldv((const T*)a.w + c) : CT(1);
    neg_mean[e] = -__ldcg(st), scale[e] = __ldcg(st + 1) * w, shift[e] = a.b ? (CT)ldv((const T*)a.b + c) : CT(0);
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
  __device__ __forceinline__ void value(const Coefs<T, CT, N>& k, const CT (&d)[N], CT (&dz)[N]) const {
    CT r[N];
    fma_to(r, d, c1, c0);
    fma_to(dz, dz, k.scale, r);
  }
};

// ---- channels-last ------------------------------------------------------------------------------------
// R pixels are V vectors of N elements; vector j of such a row of pixels holds the same channels everywhere.  A thread keeps one
// vector (of a column of 256) and takes every lanes-th row of the tile.
template <int N>
struct Place {
  long long at, step, end;  // flat: this thread's first vector, from row to row, behind the tile
  int rows;                 // whole rows of this thread
  long long tail;           // its vector of the row that the tile's end cuts, or end
  int col, j, lane, vc;     // column, vector of the row, which of the rows, vectors of the column
  __device__ Place(const Args& a, long long b, int tile) {
    col = tile % a.cols;
    const long long t = tile / a.cols, image = b * a.S * a.C, row0 = image + t * a.px * a.C, left = a.S - t * a.px;
    end = row0 + (left < a.px ? left : a.px) * a.C;
    vc = min(256, a.V - col * 256);
    lane = threadIdx.x / vc;
    j = col * 256 + threadIdx.x % vc;
    const int row = a.V * N, whole = (int)((end - row0) / row);
    step = (long long)a.lanes * row;
    at = row0 + (long long)lane * row + j * N;
    rows = lane < a.lanes && whole > lane ? (whole - lane + a.lanes - 1) / a.lanes : 0;
    tail = end;
    if (lane < a.lanes && whole % a.lanes == lane) {
      tail = row0 + (long long)whole * row + j * N;
      if (tail > end) tail = end;
    }
  }
};
template <typename CT, int N> union Shared {
  Part<CT> part[N][THREADS];
  Two<CT> two[N][THREADS];
};

template <typename T, typename CT, int N>
__device__ __forceinline__ void rows_stats(const Args& a, Shared<CT, N>& sm, long long b, int tile) {
  constexpr int U = 4;
  const T* x = (const T*)a.x;
  const Place<N> p(a, b, tile);
  Run<CT, N> run;
  CT v[U][N];
  if (p.rows) load_vec<N>(x + p.at, v[0]);
  else load_in<N>(x, p.tail, 0, p.end, v[0]);
  run.start(v[0]);
  int r = 0;
  long long i = p.at;
  for (; r + U <= p.rows; r += U, i += U * p.step) {
#pragma unroll
    for (int u = 0; u < U; ++u) load_vec<N>(x + i + u * p.step, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) run.add(v[u]);
  }
  for (; r < p.rows; ++r, i += p.step) {
    load_vec<N>(x + i, v[0]);
    run.add(v[0]);
  }
  if (p.tail < p.end) {
    load_in<N>(x, p.tail, 0, p.end, v[0]);
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (p.tail + e < p.end) run.add_one(v[0][e], e);
  }
  // one warp per group adds up what its channels left
  const bool joined = a.R == 1 && a.Cg % N == 0;  // a thread's channels are of one group
  if (joined) {
    Part<CT> q[N];
    CT mean = CT(0), m2 = CT(0);
#pragma unroll
    for (int e = 0; e < N; ++e) q[e] = run.part(e, (CT)p.rows), mean += q[e].mean;
    mean /= CT(N);
#pragma unroll
    for (int e = 0; e < N; ++e) m2 += q[e].m2 + (CT)p.rows * (q[e].mean - mean) * (q[e].mean - mean);
    sm.part[0][threadIdx.x] = Part<CT>{(CT)p.rows * CT(N), mean, m2};
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) sm.part[e][threadIdx.x] = run.part(e, (CT)(p.rows + (p.tail + e < p.end ? 1 : 0)));
  }
  __syncthreads();
  const int lane = threadIdx.x % 32, each = joined ? a.Cg / N : a.Cg * a.R, entries = each * a.lanes;
  Part<CT>* out = (Part<CT>*)a.part + (b * a.tiles + tile) * a.G;
  for (int g = threadIdx.x / 32; g < a.G; g += WARPS) {
    const auto entry = [&](int i, Part<CT>& v) {
      const int l = i / each, k = i - l * each;
      int e = 0, j;
      if (joined) {
        j = g * each + k - p.col * 256;
      } else {
        const int rr = k / a.Cg, f = rr * a.C + g * a.Cg + k - rr * a.Cg;
        j = f / N - p.col * 256, e = f % N;
      }
      if (j < 0 || j >= p.vc) return false;
      v = sm.part[e][l * p.vc + j];
      return v.n > CT(0);
    };
    CT cnt = CT(0), sum = CT(0), m2 = CT(0);
    Part<CT> w;
    for (int i = lane; i < entries; i += 32)
      if (entry(i, w)) cnt += w.n, sum += w.n * w.mean;
    cnt = warp_sum(cnt), sum = warp_sum(sum);
    const CT mean = cnt > CT(0) ? sum / cnt : CT(0);
    for (int i = lane; i < entries; i += 32)
      if (entry(i, w)) m2 += w.m2 + w.n * (w.mean - mean) * (w.mean - mean);
    m2 = warp_sum(m2);
    if (lane == 0) out[g] = Part<CT>{cnt, mean, m2};
  }
}

template <typename T, int ACT, typename CT, int N>
__device__ __forceinline__ void rows_apply(const Args& a, long long b, int tile) {
  constexpr int U = N == 8 ? 2 : 4;
  const Place<N> p(a, b, tile);
  if (!p.rows && p.tail >= p.end) return;
  const T* x = (const T*)a.x;
  T* y = (T*)a.y;
  Coefs<T, CT, N> k;
#pragma unroll
  for (int e = 0; e < N; ++e) k.load(a, b, (int)(((long long)p.j * N + e) % a.C), e);
  const auto value = [&](CT (&v)[N]) {
    add_to(v, v, k.neg_mean);
    fma_to(v, v, k.scale, k.shift);
    value_of<T, ACT>(a.act, v);
  };
  CT v[U][N];
  int r = 0;
  long long i = p.at;
  for (; r + U <= p.rows; r += U, i += U * p.step) {
#pragma unroll
    for (int u = 0; u < U; ++u) load_vec<N>(x + i + u * p.step, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) value(v[u]), store_vec<N>(y + i + u * p.step, v[u]);
  }
  for (; r < p.rows; ++r, i += p.step) {
    load_vec<N>(x + i, v[0]);
    value(v[0]);
    store_vec<N>(y + i, v[0]);
  }
  if (p.tail < p.end) {
    load_in<N>(x, p.tail, 0, p.end, v[0]);
    value(v[0]);
    store_in<N>(y, p.tail, 0, p.end, v[0]);
  }
}

template <typename T, int ACT, typename CT, int N>
__device__ __forceinline__ void rows_sums(const Args& a, Shared<CT, N>& sm, long long b, int tile) {
  constexpr int U = 2;
  const T *x = (const T*)a.x, *gy = (const T*)a.gy;
  const Place<N> p(a, b, tile);
  Sums<CT, N> sums;
  sums.clear();
  if (p.rows || p.tail < p.end) {
    Coefs<T, CT, N> k;
#pragma unroll
    for (int e = 0; e < N; ++e) k.load(a, b, (int)(((long long)p.j * N + e) % a.C), e);
    CT v[U][N], g[U][N];
    int r = 0;
    long long i = p.at;
    for (; r + U <= p.rows; r += U, i += U * p.step) {
#pragma unroll
      for (int u = 0; u < U; ++u) load_vec<N>(x + i + u * p.step, v[u]), load_vec<N>(gy + i + u * p.step, g[u]);
#pragma unroll
      for (int u = 0; u < U; ++u) slope_terms<T, ACT>(a, k, v[u], g[u]), sums.add(v[u], g[u]);
    }
    for (; r < p.rows; ++r, i += p.step) {
      load_vec<N>(x + i, v[0]), load_vec<N>(gy + i, g[0]);
      slope_terms<T, ACT>(a, k, v[0], g[0]), sums.add(v[0], g[0]);
    }
    if (p.tail < p.end) {
      load_in<N>(x, p.tail, 0, p.end, v[0]), load_in<N>(gy, p.tail, 0, p.end, g[0]);
      slope_terms<T, ACT>(a, k, v[0], g[0]);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (p.tail + e < p.end) sums.s1[e] += g[0][e], sums.s2[e] += v[0][e] * g[0][e];
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e) sm.two[e][threadIdx.x] = Two<CT>{sums.s1[e], sums.s2[e]};
  __syncthreads();
  const int entries = a.R * a.lanes;
  // threads that share a channel, as many as the channels leave
  const int sub = a.C >= 128 ? 1 : a.C >= 32 ? 8 : 32;
  Two<CT>* out = (Two<CT>*)a.part + (b * a.tiles + tile) * a.C;
  for (int c0 = 0; c0 < a.C; c0 += THREADS / sub) {
    const int c = c0 + threadIdx.x / sub;
    CT u = CT(0), v = CT(0);
    if (c < a.C)
      for (int i = threadIdx.x % sub; i < entries; i += sub) {
        const int l = i / a.R, r = i - l * a.R, f = r * a.C + c, j = f / N - p.col * 256;
        if (j >= 0 && j < p.vc) {
          const Two<CT> t = sm.two[f % N][l * p.vc + j];
          u += t.a, v += t.b;
        }
      }
    for (int o = sub / 2; o; o >>= 1) u += __shfl_xor_sync(~0u, u, o), v += __shfl_xor_sync(~0u, v, o);
    if (c < a.C && threadIdx.x % sub == 0) out[c] = Two<CT>{u, v * __ldcg((const CT*)a.stats + 2 * (b * a.G + c / a.Cg) + 1)};
  }
}

template <typename T, int ACT, typename CT, int N>
__device__ __forceinline__ void rows_grad(const Args& a, long long b, int tile) {
  constexpr int U = 2;
  const Place<N> p(a, b, tile);
  if (!p.rows && p.tail >= p.end) return;
  const T *x = (const T*)a.x, *gy = (const T*)a.gy;
  T* gx = (T*)a.gx;
  Coefs<T, CT, N> k;
  Grads<T, CT, N> q;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int c = (int)(((long long)p.j * N + e) % a.C);
    k.load(a, b, c, e), q.load(a, b, c, e);
  }
  CT v[U][N], g[U][N];
  int r = 0;
  long long i = p.at;
  for (; r + U <= p.rows; r += U, i += U * p.step) {
#pragma unroll
    for (int u = 0; u < U; ++u) load_vec<N>(x + i + u * p.step, v[u]), load_vec<N>(gy + i + u * p.step, g[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) slope_terms<T, ACT>(a, k, v[u], g[u]), q.value(k, v[u], g[u]), store_vec<N>(gx + i + u * p.step, g[u]);
  }
  for (; r < p.rows; ++r, i += p.step) {
    load_vec<N>(x + i, v[0]), load_vec<N>(gy + i, g[0]);
    slope_terms<T, ACT>(a, k, v[0], g[0]), q.value(k, v[0], g[0]);
    store_vec<N>(gx + i, g[0]);
  }
  if (p.tail < p.end) {
    load_in<N>(x, p.tail, 0, p.end, v[0]), load_in<N>(gy, p.tail, 0, p.end, g[0]);
    slope_terms<T, ACT>(a, k, v[0], g[0]), q.value(k, v[0], g[0]);
    store_in<N>(gx, p.tail, 0, p.end, g[0]);
  }
}

// ---- planes ---------------------------------------------------------------------------------------------
// A warp takes segments of planes; vectors start on 16 bytes wherever the plane does (all tensors lie alike).  f(vectors at i ..,
// whole) is called for up to U vectors of this lane at a time, whole ones, or with one that the segment's ends may cut.
template <int N>
struct Segment {
  long long lo, hi;  // flat: first element, behind the last
  int c;
  __device__ Segment(const Args& a, long long b, int item) {
    const int plane = item / a.segs, k = item - plane * a.segs;
    c = plane;
    lo = (b * a.C + plane) * a.S + (long long)k * SEGMENT;
    hi = lo + min((long long)SEGMENT, a.S - (long long)k * SEGMENT);
  }
  template <int U, typename F, typename E>
  __device__ __forceinline__ void walk(F f, E edge) const {
    const int lane = threadIdx.x % 32;
    const long long first = (lo + N - 1) / N * N, last = hi / N * N;  // whole vectors lie between them
    if (lane == 0 && first > lo) edge(first - N);
    if (lane == 31 && last < hi && last >= first) edge(last);
    long long i = first + lane * N;
    for (; i + (U - 1) * 32 * N < last; i += U * 32 * N) f(std::integral_constant<int, U>(), i);
    for (; i < last; i += 32 * N) f(std::integral_constant<int, 1>(), i);
  }
};
// items of a warp in a tile
template <typename F>
__device__ __forceinline__ void each_item(const Args& a, int tile, F f) {
  const int first = (tile * WARPS + threadIdx.x / 32) * a.per, all = a.C * a.segs;
  for (int k = 0; k < a.per && first + k < all; ++k) f(first + k);
}
template <typename T, typename CT, int N>
__device__ __forceinline__ void planes_stats(const Args& a, long long b, int tile) {
  const T* x = (const T*)a.x;
  each_item(a, tile, [&](int item) {
    const Segment<N> g(a, b, item);
    // (a value of the lane's own run: its first vector's first, or where it has only an end of the segment, that end's)
    Run<CT, N> run;
    CT k[N], n = CT(0);
    const int lane = threadIdx.x % 32;
    const CT k0 = (CT)ldv(x + (lane ? min(g.hi - 1, (g.lo + N - 1) / N * N + lane * N) : g.lo));
#pragma unroll
    for (int e = 0; e < N; ++e) k[e] = k0;
    run.start(k);
    g.template walk<4>(
        [&](auto count, long long i) {
          constexpr int U = decltype(count)::value;
          CT v[U][N];
#pragma unroll
          for (int u = 0; u < U; ++u) load_vec<N>(x + i + u * 32 * N, v[u]);
#pragma unroll
          for (int u = 0; u < U; ++u) run.add(v[u]);
          n += CT(U * N);
        },
        [&](long long i) {
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
    const CT mean = k0 + m, cnt = warp_sum(n), all = warp_sum(n > CT(0) ? n * mean : CT(0)) / cnt;
    m2 = warp_sum(n > CT(0) ? m2 + n * (mean - all) * (mean - all) : CT(0));
    if (threadIdx.x % 32 == 0) ((Part<CT>*)a.part)[b * a.C * a.segs + item] = Part<CT>{cnt, all, m2};
  });
}
template <typename CT, int N>
__device__ __forceinline__ void spread(CT (&v)[N]) {
#pragma unroll
  for (int e = 1; e < N; ++e) v[e] = v[0];
}
template <typename T, int ACT, typename CT, int N>
__device__ __forceinline__ void planes_apply(const Args& a, long long b, int tile) {
  const T* x = (const T*)a.x;
  T* y = (T*)a.y;
  each_item(a, tile, [&](int item) {
    const Segment<N> g(a, b, item);
    Coefs<T, CT, N> k;
    k.load(a, b, g.c, 0);
    spread(k.neg_mean), spread(k.scale), spread(k.shift);
    const auto value = [&](CT (&v)[N]) {
      add_to(v, v, k.neg_mean);
      fma_to(v, v, k.scale, k.shift);
      value_of<T, ACT>(a.act, v);
    };
    g.template walk<N == 8 ? 2 : 4>(
        [&](auto count, long long i) {
          constexpr int U = decltype(count)::value;
          CT v[U][N];
#pragma unroll
          for (int u = 0; u < U; ++u) load_vec<N>(x + i + u * 32 * N, v[u]);
#pragma unroll
          for (int u = 0; u < U; ++u) value(v[u]), store_vec<N>(y + i + u * 32 * N, v[u]);
        },
        [&](long long i) {
          CT v[N];
          load_in<N>(x, i, g.lo, g.hi, v);
          value(v);
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
    k.load(a, b, g.c, 0);
    spread(k.neg_mean), spread(k.scale), spread(k.shift);
    Sums<CT, N> sums;
    sums.clear();
    g.template walk<2>(
        [&](auto count, long long i) {
          constexpr int U = decltype(count)::value;
          CT v[U][N], d[U][N];
#pragma unroll
          for (int u = 0; u < U; ++u) load_vec<N>(x + i + u * 32 * N, v[u]), load_vec<N>(gy + i + u * 32 * N, d[u]);
#pragma unroll
          for (int u = 0; u < U; ++u) slope_terms<T, ACT>(a, k, v[u], d[u]), sums.add(v[u], d[u]);
        },
        [&](long long i) {
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
    k.load(a, b, g.c, 0), q.load(a, b, g.c, 0);
    spread(k.neg_mean), spread(k.scale), spread(k.shift), spread(q.c0), spread(q.c1);
    g.template walk<2>(
        [&](auto count, long long i) {
          constexpr int U = decltype(count)::value;
          CT v[U][N], d[U][N];
#pragma unroll
          for (int u = 0; u < U; ++u) load_vec<N>(x + i + u * 32 * N, v[u]), load_vec<N>(gy + i + u * 32 * N, d[u]);
#pragma unroll
          for (int u = 0; u < U; ++u)
            slope_terms<T, ACT>(a, k, v[u], d[u]), q.value(k, v[u], d[u]), store_vec<N>(gx + i + u * 32 * N, d[u]);
        },
        [&](long long i) {
          CT v[N], d[N];
          load_in<N>(x, i, g.lo, g.hi, v), load_in<N>(gy, i, g.lo, g.hi, d);
          slope_terms<T, ACT>(a, k, v, d), q.value(k, v, d);
          store_in<N>(gx, i, g.lo, g.hi, d);
        });
  });
}

// ---- between the two readings of an image, by the whole block -----------------------------------------------
template <typename T>
__device__ __forceinline__ Two<T> peek(const Two<T>* p) {  // (behind L1)
  return Two<T>{__ldcg(&p->a), __ldcg(&p->b)};
}
// statistics of the groups, one warp to a group, in double
template <typename CT>
__device__ void merge_stats(const Args& a, bool rows, long long b) {
  const int lane = threadIdx.x % 32, count = rows ? a.tiles : a.Cg * a.segs, step = rows ? a.G : 1;
  for (int g = threadIdx.x / 32; g < a.G; g += WARPS) {
    const Part<CT>* part = (const Part<CT>*)a.part + (rows ? b * a.tiles * a.G + g : (b * a.C + (long long)g * a.Cg) * a.segs);
    double n = 0, sum = 0, m2 = 0;
    for (int i = lane; i < count; i += 32) {
      const double k = __ldcg(&part[(long long)i * step].n);
      if (k > 0) n += k, sum += k * (double)__ldcg(&part[(long long)i * step].mean);
    }
    n = warp_sum(n), sum = warp_sum(sum);
    const double mean = sum / n;
    for (int i = lane; i < count; i += 32) {
      const Part<CT>* p = part + (long long)i * step;
      const double k = __ldcg(&p->n), d = (double)__ldcg(&p->mean) - mean;
      if (k > 0) m2 += (double)__ldcg(&p->m2) + k * d * d;
    }
    m2 = warp_sum(m2);
    if (lane == 0) {
      CT* st = (CT*)a.stats + 2 * (b * a.G + g);
      st[0] = (CT)mean, st[1] = (CT)(1.0 / sqrt(m2 / n + a.eps));
    }
  }
}
// S1 and S2 of every channel, then what a group's gradients subtract
template <typename T, typename CT>
__device__ void merge_sums(const Args& a, bool rows, long long b) {
  const int lane = threadIdx.x % 32;
  Two<double>* sums = (Two<double>*)a.sums + b * a.C;
  if (rows) {
    // neighbouring threads: neighbouring channels; as many threads to a channel as the channels leave
    const int sub = a.C >= 256 ? 1 : a.C >= 64 ? 4 : a.C >= 16 ? 16 : 32;
    const Two<CT>* part = (const Two<CT>*)a.part + b * a.tiles * a.C;
    for (int c0 = 0; c0 < a.C; c0 += THREADS / sub) {
      const int c = c0 + threadIdx.x / sub;
      double u = 0, v = 0;
      if (c < a.C) {
#pragma unroll 8
        for (int i = threadIdx.x % sub; i < a.tiles; i += sub) {
          const Two<CT> t = peek(part + (long long)i * a.C + c);
          u += t.a, v += t.b;
        }
      }
      for (int o = sub / 2; o; o >>= 1) u += __shfl_xor_sync(~0u, u, o), v += __shfl_xor_sync(~0u, v, o);
      if (c < a.C && threadIdx.x % sub == 0) sums[c] = Two<double>{u, v};
    }
  } else {
    const Two<CT>* part = (const Two<CT>*)a.part + b * a.C * a.segs;
    const int sub = a.segs >= 16 ? 32 : a.segs >= 3 ? 4 : 1;
    for (int c0 = 0; c0 < a.C; c0 += THREADS / sub) {
      const int c = c0 + threadIdx.x / sub;
      double u = 0, v = 0;
      if (c < a.C)
        for (int i = threadIdx.x % sub; i < a.segs; i += sub) {
          const Two<CT> t = peek(part + (long long)c * a.segs + i);
          u += t.a, v += t.b;
        }
      for (int o = sub / 2; o; o >>= 1) u += __shfl_xor_sync(~0u, u, o), v += __shfl_xor_sync(~0u, v, o);
      if (c < a.C && threadIdx.x % sub == 0) sums[c] = Two<double>{u, v};
    }
  }
  __syncthreads();
  for (int g = threadIdx.x / 32; g < a.G; g += WARPS) {
    double u = 0, v = 0;
    for (int i = lane; i < a.Cg; i += 32) {
      const int c = g * a.Cg + i;
      const double w = a.w ? (double)ldv((const T*)a.w + c) : 1.0;
      u += w * sums[c].a, v += w * sums[c].b;
    }
    u = warp_sum(u), v = warp_sum(v);
    const double n = (double)a.Cg * (double)a.S;
    if (lane == 0) ((Two<CT>*)a.coef)[b * a.G + g] = Two<CT>{(CT)(u / n), (CT)(v / n)};
  }
}
// gradients of the parameters from all images' sums
template <typename T, typename CT>
__device__ void merge_params(const Args& a) {
  const int sub = a.B < 8 ? 1 : 8;
  for (int c0 = 0; c0 < a.C; c0 += THREADS / sub) {
    const int c = c0 + threadIdx.x / sub;
    double u = 0, v = 0;
    if (c < a.C) {
#pragma unroll 4
      for (long long b = threadIdx.x % sub; b < a.B; b += sub) {
        const Two<double> t = peek((const Two<double>*)a.sums + b * a.C + c);
        u += t.a, v += t.b;
      }
    }
    for (int o = sub / 2; o; o >>= 1) u += __shfl_xor_sync(~0u, u, o), v += __shfl_xor_sync(~0u, v, o);
    if (c < a.C && threadIdx.x % sub == 0) {
      if (a.gb) stv((T*)a.gb + c, (CT)u);
      if (a.gw) stv((T*)a.gw + c, (CT)v);
    }
  }
}

// One arrival of the block at *p, behind everything that it has written; true in the block whose arrival is the last of `all`.
__device__ __forceinline__ bool last_to_arrive(unsigned* p, unsigned all, int* flag) {
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    const unsigned n = atomicAdd(p, 1u);
    __threadfence();
    *flag = n == all - 1;
  }
  __syncthreads();
  return *flag != 0;
}

// What a ticket stands for: the tile of an image, its first or second reading.
struct Job {
  long long image;
  int tile;
  bool second;
};
__device__ __forceinline__ Job job_of(const Args& a, unsigned t) {
  const unsigned T = a.tiles, ahead = (unsigned)a.lag * T, both = 2u * ((unsigned)a.B - a.lag) * T;
  if (t < ahead) return Job{t / T, (int)(t % T), false};
  t -= ahead;
  if (t < both) {
    const unsigned q = t / 2;
    return t % 2 ? Job{q / T, (int)(q % T), true} : Job{a.lag + q / T, (int)(q % T), false};
  }
  t -= both;
  return Job{(long long)a.B - a.lag + t / T, (int)(t % T), true};
}

template <typename T, int N, bool ROWS, bool BWD, int ACT>
__global__ void __launch_bounds__(THREADS) norm_kernel(const __grid_constant__ Args a) {
  typedef typename Traits<T>::CT CT;
  __shared__ Shared<CT, ROWS ? N : 1> sm;
  __shared__ unsigned ticket_s[2];
  __shared__ int flag_s;
  const bool seconds = !BWD || a.gx != nullptr;
  if (threadIdx.x == 0) ticket_s[0] = atomicAdd(a.ticket, 1u);
  __syncthreads();
  for (int turn = 0;; turn ^= 1) {
    const unsigned t = ticket_s[turn];
    if (t >= a.tickets) break;
    // (the next ticket is drawn while this one is worked on; it still waits for smaller ones only)
    if (threadIdx.x == 0) ticket_s[turn ^ 1] = atomicAdd(a.ticket, 1u);
    const Job job = seconds ? job_of(a, t) : Job{t / (unsigned)a.tiles, (int)(t % (unsigned)a.tiles), false};
    if (!job.second) {
      if constexpr (BWD) {
        if constexpr (ROWS) rows_sums<T, ACT, CT, N>(a, sm, job.image, job.tile);
        else planes_sums<T, ACT, CT, N>(a, job.image, job.tile);
      } else {
        if constexpr (ROWS) rows_stats<T, CT, N>(a, sm, job.image, job.tile);
        else planes_stats<T, CT, N>(a, job.image, job.tile);
      }
      if (last_to_arrive(a.arrived + job.image, a.tiles, &flag_s)) {
        if constexpr (BWD) merge_sums<T, CT>(a, ROWS, job.image);
        else merge_stats<CT>(a, ROWS, job.image);
        __syncthreads();
        if (threadIdx.x == 0) {
          __threadfence();
          asm volatile("st.release.gpu.u32 [%0], %1;" ::"l"(a.ready + job.image), "r"(1u) : "memory");
        }
        if (BWD && (a.gw || a.gb) && last_to_arrive(a.images_done, (unsigned)a.B, &flag_s)) merge_params<T, CT>(a);
      }
    } else {
      if (threadIdx.x == 0) {
        flag_s = 1;
        const long long t0 = clock64();
        for (;;) {
          unsigned up;
          asm volatile("ld.acquire.gpu.u32 %0, [%1];" : "=r"(up) : "l"(a.ready + job.image) : "memory");
          if (up) break;
          if (clock64() - t0 > WAIT_LIMIT_CYCLES) {
            flag_s = 0;
            atomicCAS(&g_status, 0, WAIT_CODE);
            break;
          }
          __nanosleep(64);
        }
      }
      __syncthreads();
      if (!flag_s) return;
      if constexpr (BWD) {
        if constexpr (ROWS) rows_grad<T, ACT, CT, N>(a, job.image, job.tile);
        else planes_grad<T, ACT, CT, N>(a, job.image, job.tile);
      } else {
        if constexpr (ROWS) rows_apply<T, ACT, CT, N>(a, job.image, job.tile);
        else planes_apply<T, ACT, CT, N>(a, job.image, job.tile);
      }
    }
    __syncthreads();
  }
}

int status_read(int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_status, sizeof(int)) != cudaSuccess) return MC_ERR_LAUNCH;
  if (reset && v != 0) {
    const int z = 0;
    cudaMemcpyToSymbol(g_status, &z, sizeof(int));
  }
  return v;
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
  size_t counters, part_f, part_b, sums, coef;  // bytes
};
// Bytes that lie between the first reading of an image and its second.
constexpr long long LAG_BYTES = 24 << 20;
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
    a.cols = (a.V + 255) / 256;
    a.lanes = a.cols > 1 ? 1 : 256 / a.V;
    const long long step = (long long)a.lanes * a.R;
    long long k = d->B * d->S / step * a.cols / (148 * 8);
    k = k < 1 ? 1 : k > RUN ? RUN : k;
    a.px = (int)(step * k);
    tiles = (d->S + a.px - 1) / a.px * a.cols;
    p.part_f = (size_t)(d->B * tiles) * a.G * 3 * ct, p.part_b = (size_t)(d->B * tiles) * a.C * 2 * ct;
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
  p.counters = (2 + 2 * (size_t)d->B) * 4;
  if (2 * d->B * tiles >= (1ll << 31)) return MC_ERR_TOO_LARGE;
  a.tiles = (int)tiles, a.tickets = (unsigned)(2 * d->B * tiles);
  return MC_OK;
}
static void set_lag(Args& a, long long image_bytes) {
  long long lag = (LAG_BYTES + image_bytes - 1) / image_bytes;
  if (lag * a.tiles < 148 * 8) lag = (148 * 8 + a.tiles - 1) / a.tiles;  // (every block has something else to do first)
  a.lag = (int)(lag < a.B ? lag : a.B);
}
static bool on(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

// Blocks that run at one time, per kernel and device.
template <auto kern>
static int blocks_at_once() {
  static std::atomic<int> known[16];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  std::atomic<int>* slot = dev < 16 ? &known[dev] : nullptr;
  int n = slot ? slot->load(std::memory_order_relaxed) : 0;
  if (n) return n;
  int per = 0, sms = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, THREADS, 0) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  n = per * sms;
  if (slot) slot->store(n, std::memory_order_relaxed);
  return n;
}
template <typename T, int N, bool ROWS, bool BWD, int ACT>
static int launch(const Args& a, cudaStream_t st) {
  const int most = blocks_at_once<norm_kernel<T, N, ROWS, BWD, ACT>>();
  if (most <= 0) return MC_ERR_LAUNCH;
  const unsigned blocks = a.tickets < (unsigned)most ? a.tickets : (unsigned)most;
  norm_kernel<T, N, ROWS, BWD, ACT><<<blocks, THREADS, 0, st>>>(a), MC_COUNT(1);
  MC_CHECK_LAUNCH();
  return MC_OK;
}
// bf16 and float32 vectors have a kernel for each activation
template <typename T, int N, bool ROWS, bool BWD>
static int launch_act(const Args& a, cudaStream_t st) {
  if constexpr (sizeof(T) == 8 || N == 1) {
    return launch<T, N, ROWS, BWD, -1>(a, st);
  } else {
    switch (a.act) {
      case MC_ACT_RELU: return launch<T, N, ROWS, BWD, MC_ACT_RELU>(a, st);
      case MC_ACT_GELU: return launch<T, N, ROWS, BWD, MC_ACT_GELU>(a, st);
      case MC_ACT_GELU_TANH: return launch<T, N, ROWS, BWD, MC_ACT_GELU_TANH>(a, st);
      case MC_ACT_SILU: return launch<T, N, ROWS, BWD, MC_ACT_SILU>(a, st);
      case MC_ACT_SIGMOID: return launch<T, N, ROWS, BWD, MC_ACT_SIGMOID>(a, st);
      default: return launch<T, N, ROWS, BWD, MC_ACT_NONE>(a, st);
    }
  }
}
template <typename T, bool BWD>
static int run_typed(const Plan& p, cudaStream_t st) {
  constexpr int N = Vec<T>::N;
  if (!p.rows) return launch_act<T, N, false, BWD>(p.a, st);
  return p.vec ? launch_act<T, N, true, BWD>(p.a, st) : launch_act<T, 1, true, BWD>(p.a, st);
}
template <bool BWD>
static int run(const mc_norm_desc* d, Plan& p, cudaStream_t st) {
  set_lag(p.a, d->S * d->C * esize(d->dtype) * (BWD ? 2 : 1));
  if (BWD && !p.a.gx) p.a.tickets /= 2;  // (no second readings)
  if (cudaMemsetAsync(p.a.ticket, 0, p.counters, st) != cudaSuccess) return MC_ERR_LAUNCH;
  if (d->dtype == MC_F32) return run_typed<float, BWD>(p, st);
  if (d->dtype == MC_F64) return run_typed<double, BWD>(p, st);
  return run_typed<bf16, BWD>(p, st);
}
static char* set_counters(Args& a, void* ws, size_t bytes) {
  a.ticket = (unsigned*)ws, a.images_done = a.ticket + 1, a.arrived = a.ticket + 2, a.ready = a.arrived + a.B;
  return (char*)ws + up256(bytes);
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
  const size_t counters = norm::up256(p.counters);
  if (phase != MC_PHASE_BACKWARD) return counters + norm::up256(p.part_f);
  return counters + norm::up256(p.part_b) + norm::up256(p.sums) + norm::up256(p.coef);
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
  p.a.part = norm::set_counters(p.a, ws, p.counters);
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
  char* at = norm::set_counters(p.a, ws, p.counters);
  p.a.x = x, p.a.w = w, p.a.b = bias, p.a.gy = gy, p.a.gx = gx, p.a.gw = gw, p.a.gb = gb, p.a.stats = (void*)stats;
  p.a.part = at, at += norm::up256(p.part_b);
  p.a.sums = at, at += norm::up256(p.sums);
  p.a.coef = at;
  return norm::run<true>(d, p, (cudaStream_t)stream);
}

}  // extern "C"
