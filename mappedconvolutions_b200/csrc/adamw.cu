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
__device__ __forceinline__ float value_m(uint32_t c, int j, float s) {
  const int k = (int)(int8_t)(c >> (8 * j));
  return __fmul_rn((float)(k * abs(k)), s);
}
__device__ __forceinline__ float value_v(uint32_t c, int j, float s) {
  const int k = (int)(c >> (8 * j) & 255);
  const float r = __fmul_rn((float)(k * k), s);
  return __fmul_rn(r, r);
}
// The larger of two magnitudes; NaN if one is.
__device__ __forceinline__ float larger(float a, float b) { return (b > a || b != b) ? b : a; }
__device__ __forceinline__ float warp_largest(float a) {
#pragma unroll
  for (int o = 16; o; o >>= 1) a = larger(a, __shfl_xor_sync(~0u, a, o));
  return a;
}
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
__device__ __forceinline__ float quotient(float a, float b) { return __fdividef(a, b); }  // (2 ulp; b < 2^126, sqrt(v) ends at 2^64)
__device__ __forceinline__ double quotient(double a, double b) { return a / b; }

// P: the parameters' type, G: the gradients', M: with float32 copies of bf16 parameters, B8: moments in 8 bits
template <int N, typename P, typename G, bool M, bool B8>
__global__ void __launch_bounds__(THREADS) step_kernel(const __grid_constant__ Table<N> t, const Hyper h) {
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
    CT g[8], w[8], m[8], v[8];
    load8((const G*)t.g[k] + at, i, n, vec, g);
    if constexpr (M) load8(master, i, n, vec, w);
    else load8((const P*)p, i, n, vec, w);
    uint32_t cm[2], cv[2];
    float* ms = nullptr;
    float* vs = nullptr;
    if constexpr (B8) {
      const long long block = (at + i) / BLOCK8;
      if (i < n) ms = t.ms[k] + block, vs = t.vs[k] + block;
      load_codes((const uint8_t*)t.m[k] + at, i, n, vec, cm);
      load_codes((const uint8_t*)t.v[k] + at, i, n, vec, cv);
      const float s = ms ? *ms : 0.f, q = vs ? *vs : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) m[j] = value_m(cm[j / 4], j % 4, s), v[j] = value_v(cv[j / 4], j % 4, q);
    } else {
      load8((const CT*)t.m[k] + at, i, n, vec, m);
      load8((const CT*)t.v[k] + at, i, n, vec, v);
    }
    CT r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = add_rn(mul(m[j], b1), mul(g[j], c1));
      v[j] = add_rn(mul(v[j], b2), mul(mul(g[j], g[j]), c2));
      r[j] = root_of(v[j]);
      const CT u = quotient(m[j], r[j] * inv_root + eps);
      w[j] = w[j] * keep - rate * u;
    }
    if constexpr (M) store8(master, i, n, vec, w);
    store8(p, i, n, vec, w);
    if constexpr (B8) {
      float am = 0.f, av = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) am = larger(am, fabsf(m[j])), av = larger(av, r[j]);  // (elements behind the end are zeros)
      float im, iv;
      const float s = scale_of(warp_largest(am), MOST_M, &im), q = scale_of(warp_largest(av), MOST_V, &iv);
      cm[0] = cm[1] = cv[0] = cv[1] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        int a = (int)rintf(__fsqrt_rn(__fmul_rn(fabsf(m[j]), im)));  // (NaN: zero; the scale is NaN)
        if (a > 127) a = 127;
        if (m[j] < 0.f) a = -a;
        cm[j / 4] |= (uint32_t)(a & 255) << (8 * (j % 4));
        int b = (int)rintf(__fsqrt_rn(__fmul_rn(r[j], iv)));
        if (b > 255) b = 255;
        if (b == 0 && r[j] > 0.f && q > 0.f) b = 1;
        cv[j / 4] |= (uint32_t)b << (8 * (j % 4));
      }
      store_codes((uint8_t*)t.m[k] + at, i, n, vec, cm);
      store_codes((uint8_t*)t.v[k] + at, i, n, vec, cv);
      __syncwarp();  // (every lane has read the old scales)
      if (ms && threadIdx.x % 32 == 0) *ms = s, *vs = q;
    } else {
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
    float m[8], v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = value_m(cm[j / 4], j % 4, s), v[j] = value_v(cv[j / 4], j % 4, q);
    store8((float*)t.p[k] + at, i, n, vec, m);
    store8((float*)t.master[k] + at, i, n, vec, v);
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
