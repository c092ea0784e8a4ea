// AdamW over many tensors at once, moments in 32 bits or in 8 bits with a scale for 256 elements.
//
//   m <- b1 m + (1 - b1) g,   v <- b2 v + (1 - b2) g^2,   p <- p (1 - lr decay) - rate m / (sqrt(v) / root + eps)
//   with rate = lr / (1 - b1^t), root = sqrt(1 - b2^t) of the tensor's own step count t
//
// 8 bits: a block is 256 consecutive elements; with a the largest |m| and s = a / 127^2, m is kept as the integer c nearest to
// sqrt(|m| / s), with m's sign, and stands for c |c| s.  v is kept through its root r: a the largest r, s = a / 255^2, c nearest to
// sqrt(r / s), v stands for (c^2 s)^2.  Squares as codes: neighbours are 1.6 % (m) and 0.8 % (r) apart at a block's largest element
// and reach down to 2^-14 and 2^-16 of it.  A v that is not zero keeps a code that is not zero: the update it divides stays
// small.  The update itself uses the moments before they are rounded.  Every operation behind a code is rounded on its own
// (no contraction), so that codes repeat on any implementation of the same float32 operations.
//
// Bound: HBM.  Each thread holds eight consecutive elements of every stream, a warp a block of 256; the tensors' addresses travel in the
// kernel parameters, so nothing is copied to the device.
#include <math.h>

#include "act_pairs.cuh"
#include "common.cuh"

namespace mc {
namespace adamw {

constexpr int THREADS = 256, CHUNK = THREADS * 8, BLOCK8 = 256;
constexpr int SMALL = 32, LARGE = 256;  // tensors per launch: a short list keeps the parameters of small calls small
constexpr float MOST_M = 16129.f, MOST_V = 65025.f;

template <int N>
struct Table {
  void *p[N], *master[N], *m[N], *v[N];
  const void* g[N];
  float *ms[N], *vs[N];
  long long numel[N];
  double rate[N], inv_root[N];
  int first[N + 1];  // first chunk of each tensor
  bool aligned[N];   // every stream starts on 16 bytes
  int n;
};
struct Hyper {
  double b1, c1, b2, c2, eps, keep;  // c = 1 - b, keep = 1 - lr decay
};

// Eight elements from `i` on, those behind the n-th as zeros.
template <typename CT>
__device__ __forceinline__ void load8(const float* p, int i, int n, bool vec, CT (&v)[8]) {
  if (vec && i + 8 <= n) {
    const float4 a = __ldcs(reinterpret_cast<const float4*>(p + i)), b = __ldcs(reinterpret_cast<const float4*>(p + i) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < n ? p[i + j] : 0.f;
  }
}
__device__ __forceinline__ void load8(const bf16* p, int i, int n, bool vec, float (&v)[8]) {
  if (vec && i + 8 <= n) {
    const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p + i));
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < n ? __bfloat162float(p[i + j]) : 0.f;
  }
}
__device__ __forceinline__ void load8(const double* p, int i, int n, bool vec, double (&v)[8]) {
  if (vec && i + 8 <= n) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double2 a = __ldcs(reinterpret_cast<const double2*>(p + i) + j);
      v[2 * j] = a.x, v[2 * j + 1] = a.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < n ? p[i + j] : 0.0;
  }
}
__device__ __forceinline__ void store8(float* p, int i, int n, bool vec, const float (&v)[8]) {
  if (vec && i + 8 <= n) {
    __stcs(reinterpret_cast<float4*>(p + i), make_float4(v[0], v[1], v[2], v[3]));
    __stcs(reinterpret_cast<float4*>(p + i) + 1, make_float4(v[4], v[5], v[6], v[7]));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n) p[i + j] = v[j];
  }
}
__device__ __forceinline__ void store8(double* p, int i, int n, bool vec, const double (&v)[8]) {
  if (vec && i + 8 <= n) {
#pragma unroll
    for (int j = 0; j < 4; ++j) __stcs(reinterpret_cast<double2*>(p + i) + j, make_double2(v[2 * j], v[2 * j + 1]));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n) p[i + j] = v[j];
  }
}
__device__ __forceinline__ void store8(bf16* p, int i, int n, bool vec, const float (&v)[8]) {
  if (vec && i + 8 <= n) {
    __align__(16) bf16 o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = __float2bfloat16_rn(v[j]);
    __stcs(reinterpret_cast<uint4*>(p + i), *reinterpret_cast<const uint4*>(o));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n) p[i + j] = __float2bfloat16_rn(v[j]);
  }
}
__device__ __forceinline__ void load_codes(const uint8_t* p, int i, int n, bool vec, uint32_t (&c)[2]) {
  if (vec && i + 8 <= n) {
    const uint2 a = __ldcs(reinterpret_cast<const uint2*>(p + i));
    c[0] = a.x, c[1] = a.y;
  } else {
    c[0] = c[1] = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n) c[j / 4] |= (uint32_t)p[i + j] << (8 * (j % 4));
  }
}
__device__ __forceinline__ void store_codes(uint8_t* p, int i, int n, bool vec, const uint32_t (&c)[2]) {
  if (vec && i + 8 <= n) {
    __stcs(reinterpret_cast<uint2*>(p + i), make_uint2(c[0], c[1]));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n) p[i + j] = (uint8_t)(c[j / 4] >> (8 * (j % 4)));
  }
}
// ---- 8 bits -------------------------------------------------------------------------------------------------
// (instructions bound this path, not memory: packed float32 pairs, codes taken from and put into the last bits of floats)
using mix::add2;
using mix::fma2;
using mix::mul2;
using mix::two;
// Byte j of c as a float, by way of a float whose last bits it is: 2^23 + c, or 2^23 + 128 + c for a signed one.
__device__ __forceinline__ float byte_of(uint32_t c, int j) { return __uint_as_float(__byte_perm(c, 0x4B000000, 0x7540 + j)); }
__device__ __forceinline__ float2 pair_of(uint32_t (&c)[2], int j) {
  return make_float2(byte_of(c[j / 2], 2 * j % 4), byte_of(c[j / 2], 2 * j % 4 + 1));
}
__device__ __forceinline__ void values_of(uint32_t (&cm)[2], uint32_t (&cv)[2], float s, float q, float2 (&m)[4], float2 (&v)[4]) {
  uint32_t c[2] = {cm[0] ^ 0x80808080u, cm[1] ^ 0x80808080u};
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // (squares of codes are whole numbers: exact)
    const float2 k = add2(pair_of(c, j), two(-8388736.f)), l = add2(pair_of(cv, j), two(-8388608.f));
    m[j] = mul2(make_float2(k.x * fabsf(k.x), k.y * fabsf(k.y)), two(s));
    const float2 r = mul2(mul2(l, l), two(q));
    v[j] = mul2(r, r);
  }
}
__device__ __forceinline__ float sqrt_near(float v) {  // within 2^-22 of the root; zero below 2^-126
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// Largest of magnitudes, as bits: those of NaN are above all others.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
// (below 2^-126 the reciprocal of a scale can overflow: such blocks are zero)
__device__ __forceinline__ float scale_of(float a, float most, float* inverse) {
  float s = __fmul_rn(a, 1.f / most);
  if (s < 1.17549435e-38f) s = 0.f;
  *inverse = s == 0.f ? 0.f : __frcp_rn(s);
  return s;
}

__device__ __forceinline__ float mul(float a, float b) { return __fmul_rn(a, b); }
__device__ __forceinline__ double mul(double a, double b) { return __dmul_rn(a, b); }
__device__ __forceinline__ float root_of(float a) { return __fsqrt_rn(a); }
__device__ __forceinline__ double root_of(double a) { return sqrt(a); }
__device__ __forceinline__ float quotient(float a, float b) { return __fdiv_rn(a, b); }
__device__ __forceinline__ double quotient(double a, double b) { return a / b; }

// The codes of a block from its moments, in registers of a warp.
// Codes are whole numbers nearest to correctly rounded roots of correctly rounded products.  Approximate roots, 2^-21 off with what
// goes into them, give the same codes but near the middle of two (256 2^-21 < 2e-4), where the exact ones are computed.
// force: roots in reach of the type's smallest values, or a scale that is not finite.
constexpr float SIGNED = 12582912.f, PLAIN = 8388608.f;  // 1.5 2^23 + a code, 2^23 + a code: the code is the last bits
__device__ __forceinline__ void encode(const float2 (&m)[4], const float2 (&v)[4], const float2 (&r)[4], float s, float q, float im,
                                       float iv, bool force, uint32_t (&cm)[2], uint32_t (&cv)[2]) {
  const bool some = q > 0.f;
  float a[8], b[8], least[8];
  uint32_t ca[8], cb[8];
  float off = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 z = mul2(r[j], two(iv));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = 2 * j + h;
      const float x = h ? m[j].y : m[j].x;
      a[e] = copysignf(sqrt_near(fabsf(x) * im), x);
      b[e] = sqrt_near(h ? z.y : z.x);
      least[e] = some && (h ? v[j].y : v[j].x) > 0.f ? 1.f : 0.f;  // (a v that is not zero keeps a code that is not zero)
    }
    const float2 ta = add2(make_float2(a[2 * j], a[2 * j + 1]), two(SIGNED)), tb = add2(make_float2(b[2 * j], b[2 * j + 1]), two(PLAIN));
    const float2 ra = add2(ta, two(-SIGNED)), rb = add2(tb, two(-PLAIN));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = 2 * j + h;
      off = fmaxf(off, fmaxf(fabsf(a[e] - (h ? ra.y : ra.x)), fabsf(b[e] - (h ? rb.y : rb.x))));
    }
  }
  if (__any_sync(~0u, off > 0.4998f) || force) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = e & 1 ? m[e / 2].y : m[e / 2].x, y = e & 1 ? v[e / 2].y : v[e / 2].x;
      if (force || fabsf(a[e] - rintf(a[e])) > 0.4998f) a[e] = copysignf(__fsqrt_rn(__fmul_rn(fabsf(x), im)), x);
      if (force || fabsf(b[e] - rintf(b[e])) > 0.4998f) b[e] = __fsqrt_rn(__fmul_rn(__fsqrt_rn(y), iv));
      if (force && !(fabsf(a[e]) < 127.5f)) a[e] = 0.f;  // (a scale that is not finite)
      if (force && !(b[e] < 255.5f)) b[e] = 0.f;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) ca[e] = __float_as_uint(a[e] + SIGNED), cb[e] = __float_as_uint(fmaxf(b[e], least[e]) + PLAIN);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    cm[h] = __byte_perm(__byte_perm(ca[4 * h], ca[4 * h + 1], 0x0040), __byte_perm(ca[4 * h + 2], ca[4 * h + 3], 0x0040), 0x5410);
    cv[h] = __byte_perm(__byte_perm(cb[4 * h], cb[4 * h + 1], 0x0040), __byte_perm(cb[4 * h + 2], cb[4 * h + 3], 0x0040), 0x5410);
  }
}

// P: the parameters' type, G: the gradients', M: with float32 copies of bf16 parameters, B8: moments in 8 bits
// (8 bits: 48 warps an SM.  32: 125 us for 33.6 M bf16 parameters instead of 108, 40: 113.)
template <int N, typename P, typename G, bool M, bool B8>
__global__ void __launch_bounds__(THREADS, B8 ? 6 : 1) step_kernel(const __grid_constant__ Table<N> t, const Hyper h) {
  typedef typename Traits<P>::CT CT;
  const CT b1 = (CT)h.b1, c1 = (CT)h.c1, b2 = (CT)h.b2, c2 = (CT)h.c2, eps = (CT)h.eps, keep = (CT)h.keep;
  const int total = t.first[t.n];
  for (int c = blockIdx.x; c < total; c += gridDim.x) {
    int k = 0, hi = t.n - 1;  // first[k] <= c < first[k + 1]
    while (k < hi) {
      const int mid = (k + hi + 1) / 2;
      if (t.first[mid] <= c) k = mid;
      else hi = mid - 1;
    }
    const long long at = (long long)(c - t.first[k]) * CHUNK, left = t.numel[k] - at;
    const int n = left < CHUNK ? (int)left : CHUNK, i = threadIdx.x * 8;
    const bool vec = t.aligned[k];
    const CT rate = (CT)t.rate[k], inv_root = (CT)t.inv_root[k];
    P* p = (P*)t.p[k] + at;
    float* master = (float*)t.master[k] + at;
    CT g[8], w[8];
    load8((const G*)t.g[k] + at, i, n, vec, g);
    if constexpr (M) load8(master, i, n, vec, w);
    else load8((const P*)p, i, n, vec, w);
    if constexpr (B8) {
      uint32_t cm[2], cv[2];
      load_codes((const uint8_t*)t.m[k] + at, i, n, vec, cm);
      load_codes((const uint8_t*)t.v[k] + at, i, n, vec, cv);
      float *ms = nullptr, *vs = nullptr;
      if (i < n) ms = t.ms[k] + (at + i) / BLOCK8, vs = t.vs[k] + (at + i) / BLOCK8;
      float2 m[4], v[4], r[4];
      values_of(cm, cv, ms ? *ms : 0.f, vs ? *vs : 0.f, m, v);
      uint32_t am = 0, av = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // (not in pairs: packed products and sums came out as one operation, a last bit off)
        m[j].x = add_rn(mul(m[j].x, b1), mul(g[2 * j], c1)), m[j].y = add_rn(mul(m[j].y, b1), mul(g[2 * j + 1], c1));
        v[j].x = add_rn(mul(v[j].x, b2), mul(mul(g[2 * j], g[2 * j]), c2));
        v[j].y = add_rn(mul(v[j].y, b2), mul(mul(g[2 * j + 1], g[2 * j + 1]), c2));
        am = max(am, max(magnitude(m[j].x), magnitude(m[j].y)));  // (elements behind the end are zeros)
        av = max(av, max(magnitude(v[j].x), magnitude(v[j].y)));
      }
      av = __reduce_max_sync(~0u, av);
      // Approximate roots take those below 2^-63 for zero.  That changes no code where the block's largest is 2^-45 or more, and the
      // divisor by less than 2^-24 of it where eps is 2^-39 inv_root or more (5.7e-11 at a first step with beta2 = 0.999).  Approximate
      // reciprocals are zero from 2^126 on, which only an eps reaches: roots end at 2^64.
      const bool small = av < __float_as_uint(0x1p-90f) || eps < 0x1p-39f * inv_root || eps > 0x1p125f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        r[j] = small ? make_float2(__fsqrt_rn(v[j].x), __fsqrt_rn(v[j].y)) : make_float2(sqrt_near(v[j].x), sqrt_near(v[j].y));
        const float2 d = fma2(r[j], two(inv_root), two(eps));
        float2 u;
        if (small) u = make_float2(m[j].x / d.x, m[j].y / d.y);
        else u = mul2(m[j], mix::rcp2(d));
        const float2 x = fma2(u, two(-rate), mul2(make_float2(w[2 * j], w[2 * j + 1]), two(keep)));
        w[2 * j] = x.x, w[2 * j + 1] = x.y;
      }
      if constexpr (M) store8(master, i, n, vec, w);
      store8(p, i, n, vec, w);
      float im, iv;
      const float s = scale_of(__uint_as_float(__reduce_max_sync(~0u, am)), MOST_M, &im);
      const float q = scale_of(__fsqrt_rn(__uint_as_float(av)), MOST_V, &iv);  // (roots keep their order)
      encode(m, v, r, s, q, im, iv, small || !(s < INFINITY) || !(q < INFINITY), cm, cv);
      store_codes((uint8_t*)t.m[k] + at, i, n, vec, cm);
      store_codes((uint8_t*)t.v[k] + at, i, n, vec, cv);
      __syncwarp();  // (every lane has read the old scales)
      if (ms && threadIdx.x % 32 == 0) *ms = s, *vs = q;
    } else {
      CT m[8], v[8];
      load8((const CT*)t.m[k] + at, i, n, vec, m);
      load8((const CT*)t.v[k] + at, i, n, vec, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        m[j] = add_rn(mul(m[j], b1), mul(g[j], c1));
        v[j] = add_rn(mul(v[j], b2), mul(mul(g[j], g[j]), c2));
        const CT u = quotient(m[j], root_of(v[j]) * inv_root + eps);
        w[j] = w[j] * keep - rate * u;
      }
      if constexpr (M) store8(master, i, n, vec, w);
      store8(p, i, n, vec, w);
      store8((CT*)t.m[k] + at, i, n, vec, m);
      store8((CT*)t.v[k] + at, i, n, vec, v);
    }
  }
}

// What the codes stand for: m and v of the table are the codes, p and master the float32 results.
template <int N>
__global__ void __launch_bounds__(THREADS) values_kernel(const __grid_constant__ Table<N> t) {
  const int total = t.first[t.n];
  for (int c = blockIdx.x; c < total; c += gridDim.x) {
    int k = 0, hi = t.n - 1;
    while (k < hi) {
      const int mid = (k + hi + 1) / 2;
      if (t.first[mid] <= c) k = mid;
      else hi = mid - 1;
    }
    const long long at = (long long)(c - t.first[k]) * CHUNK, left = t.numel[k] - at;
    const int n = left < CHUNK ? (int)left : CHUNK, i = threadIdx.x * 8;
    if (i >= n) continue;
    const bool vec = t.aligned[k];
    const float s = t.ms[k][(at + i) / BLOCK8], q = t.vs[k][(at + i) / BLOCK8];
    uint32_t cm[2], cv[2];
    load_codes((const uint8_t*)t.m[k] + at, i, n, vec, cm);
    load_codes((const uint8_t*)t.v[k] + at, i, n, vec, cv);
    float2 m[4], v[4];
    values_of(cm, cv, s, q, m, v);
    float o[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[2 * j] = m[j].x, o[2 * j + 1] = m[j].y;
    store8((float*)t.p[k] + at, i, n, vec, o);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[2 * j] = v[j].x, o[2 * j + 1] = v[j].y;
    store8((float*)t.master[k] + at, i, n, vec, o);
  }
}

static bool placed(const mc_adamw_tensor& t) {
  const void* all[] = {t.p, t.g, t.master, t.m, t.v};
  for (const void* p : all)
    if ((uintptr_t)p % 16) return false;
  return true;
}
template <int N>
static void add(Table<N>& t, const mc_adamw_tensor& a, double rate, double inv_root) {
  const int k = t.n++;
  t.p[k] = a.p, t.master[k] = a.master, t.m[k] = a.m, t.v[k] = a.v, t.g[k] = a.g, t.ms[k] = a.m_scale, t.vs[k] = a.v_scale;
  t.numel[k] = a.numel, t.rate[k] = rate, t.inv_root[k] = inv_root, t.aligned[k] = placed(a);
  t.first[k + 1] = t.first[k] + (int)((a.numel + CHUNK - 1) / CHUNK);
}
// Chunks are counted in int.  (No sum is formed that could overflow.)
static bool too_many(int n, const mc_adamw_tensor* ts) {
  long long chunks = 0;
  for (int i = 0; i < n; ++i) {
    const long long more = ts[i].numel / CHUNK + 1;
    if (more >= (1 << 30) || chunks + more >= (1 << 30)) return true;
    chunks += more;
  }
  return false;
}
static int blocks_for(int chunks) { return chunks < 148 * 64 ? chunks : 148 * 64; }

template <int N>
static int launch(const Table<N>& t, const Hyper& h, const mc_adamw_tensor& like, cudaStream_t st) {
  const int blocks = blocks_for(t.first[t.n]);
#define MC_ADAMW(P, G, M, B8) step_kernel<N, P, G, M, B8><<<blocks, THREADS, 0, st>>>(t, h)
  const bool gb = like.g_dtype == MC_BF16, b8 = like.bits == 8;
  if (like.p_dtype == MC_F64) MC_ADAMW(double, double, false, false);
  else if (like.p_dtype == MC_F32) {
    if (gb) b8 ? MC_ADAMW(float, bf16, false, true) : MC_ADAMW(float, bf16, false, false);
    else b8 ? MC_ADAMW(float, float, false, true) : MC_ADAMW(float, float, false, false);
  } else if (like.master) {
    if (gb) b8 ? MC_ADAMW(bf16, bf16, true, true) : MC_ADAMW(bf16, bf16, true, false);
    else b8 ? MC_ADAMW(bf16, float, true, true) : MC_ADAMW(bf16, float, true, false);
  } else {
    if (gb) b8 ? MC_ADAMW(bf16, bf16, false, true) : MC_ADAMW(bf16, bf16, false, false);
    else b8 ? MC_ADAMW(bf16, float, false, true) : MC_ADAMW(bf16, float, false, false);
  }
#undef MC_ADAMW
  MC_COUNT(1);
  MC_CHECK_LAUNCH();
  return MC_OK;
}
static bool same_kind(const mc_adamw_tensor& a, const mc_adamw_tensor& b) {
  return a.p_dtype == b.p_dtype && a.g_dtype == b.g_dtype && !a.master == !b.master && a.bits == b.bits;
}

// One launch for up to N tensors of the same types; tensors of other types wait for a launch of their own.
template <int N>
static int run(int n, const mc_adamw_tensor* ts, const mc_adamw_hyper* h, const Hyper& k, cudaStream_t st) {
  Table<N> t;
  for (int i = 0; i < n; ++i) {
    if (ts[i].numel == 0) continue;
    bool seen = false;
    for (int j = 0; j < i && !seen; ++j) seen = ts[j].numel && same_kind(ts[i], ts[j]);
    if (seen) continue;
    t.n = 0, t.first[0] = 0;
    for (int j = i; j < n; ++j) {
      if (!ts[j].numel || !same_kind(ts[i], ts[j])) continue;
      add(t, ts[j], h->lr / (1 - pow(h->beta1, (double)ts[j].step)), 1 / sqrt(1 - pow(h->beta2, (double)ts[j].step)));
      if (t.n < N) continue;
      const int rc = launch(t, k, ts[i], st);
      if (rc) return rc;
      t.n = 0;
    }
    if (t.n) {
      const int rc = launch(t, k, ts[i], st);
      if (rc) return rc;
    }
  }
  return MC_OK;
}
template <int N>
static int run_values(int n, const mc_adamw_tensor* ts, cudaStream_t st) {
  Table<N> t;
  t.n = 0, t.first[0] = 0;
  for (int j = 0; j < n; ++j) {
    if (ts[j].numel) add(t, ts[j], 0, 0);
    if (t.n == N || (j + 1 == n && t.n)) {
      values_kernel<N><<<blocks_for(t.first[t.n]), THREADS, 0, st>>>(t), MC_COUNT(1);
      MC_CHECK_LAUNCH();
      t.n = 0;
    }
  }
  return MC_OK;
}

static bool on(const void* p, size_t n) { return (uintptr_t)p % n == 0; }
static size_t size_of(int dtype) { return dtype == MC_F64 ? 8 : dtype == MC_F32 ? 4 : 2; }
static bool known(int t) { return t == MC_F32 || t == MC_F64 || t == MC_BF16; }

static int check_tensor(const mc_adamw_tensor& t) {
  if (t.numel < 0 || t.step < 1 || (t.bits != 32 && t.bits != 8) || !known(t.p_dtype) || !known(t.g_dtype)) return MC_ERR_BAD_ARG;
  if ((t.p_dtype == MC_F64) != (t.g_dtype == MC_F64)) return MC_ERR_UNSUPPORTED;
  if (t.p_dtype == MC_F64 && t.bits == 8) return MC_ERR_UNSUPPORTED;
  if (t.master && t.p_dtype != MC_BF16) return MC_ERR_UNSUPPORTED;
  if (!t.numel) return MC_OK;
  if (!t.p || !t.g || !t.m || !t.v || (t.bits == 8 && (!t.m_scale || !t.v_scale))) return MC_ERR_BAD_ARG;
  const size_t e = t.bits == 8 ? 1 : t.p_dtype == MC_F64 ? 8 : 4;
  if (!on(t.p, size_of(t.p_dtype)) || !on(t.g, size_of(t.g_dtype)) || !on(t.master, 4) || !on(t.m, e) || !on(t.v, e) ||
      !on(t.m_scale, 4) || !on(t.v_scale, 4))
    return MC_ERR_BAD_ARG;
  return MC_OK;
}

}  // namespace adamw
}  // namespace mc
using namespace mc;

extern "C" {

int mc_adamw_step(int32_t n, const mc_adamw_tensor* tensors, const mc_adamw_hyper* h, void* stream) {
  if (n < 0 || (n && !tensors) || !h) return MC_ERR_BAD_ARG;
  if (!(h->beta1 >= 0 && h->beta1 < 1) || !(h->beta2 >= 0 && h->beta2 < 1) || !(h->lr >= 0) || !(h->eps >= 0) ||
      !(h->weight_decay >= 0))
    return MC_ERR_BAD_ARG;
  for (int i = 0; i < n; ++i)
    if (const int rc = adamw::check_tensor(tensors[i])) return rc;
  if (adamw::too_many(n, tensors)) return MC_ERR_TOO_LARGE;
  const adamw::Hyper k{h->beta1, 1 - h->beta1, h->beta2, 1 - h->beta2, h->eps, 1 - h->lr * h->weight_decay};
  return n <= adamw::SMALL ? adamw::run<adamw::SMALL>(n, tensors, h, k, (cudaStream_t)stream)
                           : adamw::run<adamw::LARGE>(n, tensors, h, k, (cudaStream_t)stream);
}

int mc_adamw_moments(int32_t n, const mc_adamw_tensor* tensors, void* stream) {
  if (n < 0 || (n && !tensors)) return MC_ERR_BAD_ARG;
  for (int i = 0; i < n; ++i) {
    const mc_adamw_tensor& t = tensors[i];
    if (t.numel < 0 || t.bits != 8) return MC_ERR_BAD_ARG;
    if (t.numel && (!t.p || !t.master || !t.m || !t.v || !t.m_scale || !t.v_scale)) return MC_ERR_BAD_ARG;
    if (!adamw::on(t.p, 4) || !adamw::on(t.master, 4) || !adamw::on(t.m_scale, 4) || !adamw::on(t.v_scale, 4)) return MC_ERR_BAD_ARG;
  }
  if (adamw::too_many(n, tensors)) return MC_ERR_TOO_LARGE;
  return n <= adamw::SMALL ? adamw::run_values<adamw::SMALL>(n, tensors, (cudaStream_t)stream)
                           : adamw::run_values<adamw::LARGE>(n, tensors, (cudaStream_t)stream);
}

}  // extern "C"
