// Norm of many gradients together, and the gradients scaled by it.
//
//   n = (sum |v|^2)^(1/2)  |  max |v|  |  sum |v|,     dst = src * min(1, max_norm / (n + 1e-6))
//
// Bound: HBM, one read for the norm, one read and one write for the scaling; launch latency for small sets.  Two
// launches however many tensors there are (up to 512 per launch): the tensors' addresses travel in the kernel
// parameters, so nothing is copied to the device and the call can be captured.  A block takes chunks of 8192 elements
// of whichever tensor they belong to and leaves one partial result; every block of the second kernel adds all partial
// results up itself, in the same order, instead of a third launch or a counter that somebody has to clear.  The second
// kernel walks the chunks backwards: what the first one read last is still in L2.
#include <math.h>

#include "common.cuh"

namespace mc {
namespace grad {

constexpr int CHUNK = 8192, THREADS = 256, MAX_BLOCKS = 148 * 8;
// Tensors per launch; a short list keeps the parameters small: 8 tensors 10.9 us a call, 13.8 us with the long list (32: 15.7 and
// 18.6), nearly all of it on the host (the kernels: 4.8 and 5.0).
constexpr int SMALL = 32, LARGE = 512;

template <int N>
struct Table {
  const void* src[N];
  void* dst[N];
  long long numel[N];
  int first[N + 1];  // first chunk of each tensor
  unsigned char src_type[N], dst_type[N];
  int n;
};

enum { P1 = 1, P2 = 2, PINF = 3 };

// Eight elements of a tensor as floats or doubles.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = __ldcg(reinterpret_cast<const float4*>(p)), b = __ldcg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(const double* p, double (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double2 a = __ldcg(reinterpret_cast<const double2*>(p) + i);
    v[2 * i] = a.x, v[2 * i + 1] = a.y;
  }
}
__device__ __forceinline__ void load8(const bf16* p, float (&v)[8]) {
  const uint4 a = __ldcg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
}
template <typename CT>
__device__ __forceinline__ void store8(float* p, const CT (&v)[8]) {
  __stcs(reinterpret_cast<float4*>(p), make_float4((float)v[0], (float)v[1], (float)v[2], (float)v[3]));
  __stcs(reinterpret_cast<float4*>(p) + 1, make_float4((float)v[4], (float)v[5], (float)v[6], (float)v[7]));
}
template <typename CT>
__device__ __forceinline__ void store8(double* p, const CT (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) __stcs(reinterpret_cast<double2*>(p) + i, make_double2((double)v[2 * i], (double)v[2 * i + 1]));
}
__device__ __forceinline__ bf16 to_bf16(float v) { return __float2bfloat16_rn(v); }
__device__ __forceinline__ bf16 to_bf16(double v) { return __double2bfloat16(v); }
template <typename CT>
__device__ __forceinline__ void store8(bf16* p, const CT (&v)[8]) {
  __align__(16) bf16 o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = to_bf16(v[i]);
  __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(o));
}
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(float* p, double v) { *p = (float)v; }
__device__ __forceinline__ void store1(double* p, double v) { *p = v; }
template <typename CT>
__device__ __forceinline__ void store1(bf16* p, CT v) { *p = to_bf16(v); }

__device__ __forceinline__ double combine(int kind, double a, double b) {
  if (kind == PINF) return (b > a || b != b) ? b : a;  // (a NaN stays: nothing compares greater)
  return a + b;
}
template <int KIND>
__device__ __forceinline__ double part8(const double (&v)[8]) {
  double s = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    s = KIND == P2 ? fma(v[i], v[i], s) : combine(KIND, s, fabs(v[i]));
  return s;
}
// In float32 where that loses nothing but rounding: a sum of squares of ordinary size (the squares that fall below the
// normal range are then 1e-11 of it), a finite sum.  Otherwise - large, tiny, zero or not finite - in double.
template <int KIND>
__device__ __forceinline__ double part8(const float (&v)[8]) {
  float s = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(v[i]);
    if (KIND == P2) s = fmaf(a, a, s);
    else if (KIND == P1) s += a;
    else s = (a > s || a != a) ? a : s;
  }
  if (KIND == PINF || s == 0.f && KIND == P1) return s;
  if (s >= (KIND == P2 ? 1e-26f : 0.f) && s <= 1e38f) return s;
  double d = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) d = KIND == P2 ? fma((double)v[i], (double)v[i], d) : d + fabs((double)v[i]);
  return d;
}

template <int KIND, typename T>
__device__ __forceinline__ double norm_chunk(const T* p, int n) {
  typedef typename Traits<T>::CT CT;
  double s = 0;
  int i = threadIdx.x * 8;
  if (((uintptr_t)p & 15) == 0) {
    CT v[8];
#pragma unroll 4
    for (; i + 8 <= n; i += THREADS * 8) {
      load8(p + i, v);
      s = combine(KIND, s, part8<KIND>(v));
    }
  }
  // a last incomplete group of eight, or a tensor that does not start on 16 bytes: consecutive elements per thread
  for (; i < n; i += THREADS * 8) {
    CT v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < n ? (CT)ldv(p + i + j) : CT(0);
    s = combine(KIND, s, part8<KIND>(v));
  }
  return s;
}

template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& t, int chunk) {  // first[i] <= chunk < first[i + 1]
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// the block's value, in thread 0: fixed order
__device__ __forceinline__ double block_combine(int kind, double s) {
  __shared__ double warp[THREADS / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) s = combine(kind, s, __shfl_down_sync(~0u, s, o));
  if (threadIdx.x % 32 == 0) warp[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int i = 1; i < THREADS / 32; ++i) s = combine(kind, s, warp[i]);
  __syncthreads();
  return s;
}

template <int N, int KIND>
__global__ void __launch_bounds__(THREADS) norm_kernel(const __grid_constant__ Table<N> t, double* part) {
  asm volatile("griddepcontrol.launch_dependents;");
  double s = 0;
  const int total = t.first[t.n];
  for (int c = blockIdx.x; c < total; c += gridDim.x) {
    const int i = tensor_of(t, c);
    const long long at = (long long)(c - t.first[i]) * CHUNK;
    const long long left = t.numel[i] - at;
    const int n = left < CHUNK ? (int)left : CHUNK;
    double v;
    switch (t.src_type[i]) {
      case MC_F32: v = norm_chunk<KIND>((const float*)t.src[i] + at, n); break;
      case MC_F64: v = norm_chunk<KIND>((const double*)t.src[i] + at, n); break;
      default: v = norm_chunk<KIND>((const bf16*)t.src[i] + at, n); break;
    }
    s = combine(KIND, s, v);
  }
  s = block_combine(KIND, s);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ __forceinline__ double finish(int kind, const double* part, int n) {
  double s = 0;
  for (int i = threadIdx.x; i < n; i += THREADS) s = combine(kind, s, __ldcg(part + i));
  s = block_combine(kind, s);
  return kind == P2 ? sqrt(s) : s;
}
__global__ void __launch_bounds__(THREADS) finish_kernel(int kind, const double* part, int n, double* norm, float* norm32) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const double v = finish(kind, part, n);
  if (threadIdx.x == 0) {
    if (norm) *norm = v;
    if (norm32) *norm32 = (float)v;
  }
}

// A coefficient as c 2^e: where float32 would hold it with fewer bits, or as zero (a norm of 1e38, say, scaled to 1e-3), c has
// the bits and 2^e the size, and v c 2^e is rounded once, as v c is otherwise (2^e = 1).
struct Coefficient {
  double c, power;
  __device__ explicit Coefficient(double v) : c(v), power(1.0) {
    if (v > 0 && v < 1e-30) {
      const int e = max(ilogb(v) + 1, -126);  // c < 1: no product overflows
      c = ldexp(v, -e), power = ldexp(1.0, e);
    }
  }
};
template <typename S, typename D>
__device__ __forceinline__ void scale_chunk(const S* p, D* q, int n, double factor, double power) {
  typedef typename Traits<S>::CT CT;
  constexpr int ROUND = sizeof(CT) == 4 ? 4 : 2;
  const CT c = (CT)factor, c2 = (CT)power;
  int i = threadIdx.x * 8;
  if ((((uintptr_t)p | (uintptr_t)q) & 15) == 0) {
    // (all loads of a round before its stores: the compiler may not move them across, p and q can be the same)
    for (; i + (ROUND - 1) * THREADS * 8 + 8 <= n; i += ROUND * THREADS * 8) {
      CT v[ROUND][8];
#pragma unroll
      for (int r = 0; r < ROUND; ++r) load8(p + i + r * THREADS * 8, v[r]);
#pragma unroll
      for (int r = 0; r < ROUND; ++r) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[r][j] = v[r][j] * c * c2;
        store8(q + i + r * THREADS * 8, v[r]);
      }
    }
    for (; i + 8 <= n; i += THREADS * 8) {
      CT v[8];
      load8(p + i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = v[j] * c * c2;
      store8(q + i, v);
    }
  }
  for (; i < n; i += THREADS * 8)
    for (int j = 0; j < 8 && i + j < n; ++j) store1(q + i + j, (CT)ldv(p + i + j) * c * c2);
}
template <typename S>
__device__ __forceinline__ void scale_from(const S* p, void* q, int type, long long at, int n, double c, double c2) {
  switch (type) {
    case MC_F32: scale_chunk(p + at, (float*)q + at, n, c, c2); break;
    case MC_F64: scale_chunk(p + at, (double*)q + at, n, c, c2); break;
    default: scale_chunk(p + at, (bf16*)q + at, n, c, c2); break;
  }
}

template <int N>
__global__ void __launch_bounds__(THREADS) scale_kernel(const __grid_constant__ Table<N> t, int kind, const double* part,
                                                        int nparts, double max_norm, double* norm, float* norm32) {
  __shared__ double shared_c, shared_c2;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const double v = finish(kind, part, nparts);
  if (threadIdx.x == 0) {
    if (blockIdx.x == 0) {
      if (norm) *norm = v;
      if (norm32) *norm32 = (float)v;
    }
    const double c = max_norm / (v + 1e-6);
    const Coefficient k(c > 1.0 ? 1.0 : c);  // (NaN stays NaN)
    shared_c = k.c, shared_c2 = k.power;
  }
  __syncthreads();
  const double c = shared_c, c2 = shared_c2;
  for (int k = t.first[t.n] - 1 - (int)blockIdx.x; k >= 0; k -= gridDim.x) {
    const int i = tensor_of(t, k);
    const long long at = (long long)(k - t.first[i]) * CHUNK;
    const long long left = t.numel[i] - at;
    const int n = left < CHUNK ? (int)left : CHUNK;
    switch (t.src_type[i]) {
      case MC_F32: scale_from((const float*)t.src[i], t.dst[i], t.dst_type[i], at, n, c, c2); break;
      case MC_F64: scale_from((const double*)t.src[i], t.dst[i], t.dst_type[i], at, n, c, c2); break;
      default: scale_from((const bf16*)t.src[i], t.dst[i], t.dst_type[i], at, n, c, c2); break;
    }
  }
}

struct Lists {
  int n;
  const void* const* src;
  const int32_t* src_type;
  void* const* dst;
  const int32_t* dst_type;
  const int64_t* numel;
};
static int kind_of(double norm_type) { return norm_type == 2 ? P2 : norm_type == 1 ? P1 : isinf(norm_type) && norm_type > 0 ? PINF : 0; }
static int blocks_for(int chunks) { return chunks < MAX_BLOCKS ? chunks : MAX_BLOCKS; }

// The tensors from `at` on that one launch takes, empty ones left out; returns the next one.
template <int N>
static int fill(Table<N>& t, const Lists& l, int at) {
  t.n = 0;
  t.first[0] = 0;
  for (; at < l.n && t.n < N; ++at) {
    const long long chunks = (l.numel[at] + CHUNK - 1) / CHUNK;
    if (chunks == 0) continue;
    t.src[t.n] = l.src[at];
    t.dst[t.n] = l.dst ? l.dst[at] : nullptr;
    t.numel[t.n] = l.numel[at];
    t.src_type[t.n] = (unsigned char)l.src_type[at];
    t.dst_type[t.n] = l.dst ? (unsigned char)l.dst_type[at] : 0;
    t.first[t.n + 1] = t.first[t.n] + (int)chunks;
    ++t.n;
  }
  return at;
}

static int check_lists(const Lists& l, bool scale) {
  if (l.n < 0 || (l.n && (!l.src || !l.src_type || !l.numel || (scale && (!l.dst || !l.dst_type))))) return MC_ERR_BAD_ARG;
  const auto known = [](int t) { return t == MC_F32 || t == MC_F64 || t == MC_BF16; };
  constexpr long long MOST = 1 << 30;  // chunks, which are counted in int
  long long chunks = 0;
  bool many = false;  // (no sum is formed that could overflow; what is wrong with a later tensor is still reported first)
  for (int i = 0; i < l.n; ++i) {
    if (l.numel[i] < 0 || !known(l.src_type[i]) || (scale && !known(l.dst_type[i]))) return MC_ERR_BAD_ARG;
    if (l.numel[i] && (!l.src[i] || (scale && !l.dst[i]))) return MC_ERR_BAD_ARG;
    const long long more = l.numel[i] / CHUNK + (l.numel[i] % CHUNK != 0);
    many = many || more >= MOST || chunks + more >= MOST;
    if (!many) chunks += more;
  }
  return many ? MC_ERR_TOO_LARGE : MC_OK;
}

template <typename... A>
static int launch_behind(void (*kern)(A...), int blocks, cudaStream_t st, bool overlap, A... args) {
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = overlap ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kern, args...) != cudaSuccess) return MC_ERR_LAUNCH;
  MC_COUNT(1);
  return MC_OK;
}

template <int N>
static int run(const Lists& l, bool scale, int kind, double max_norm, double* norm, float* norm32, double* part,
               cudaStream_t st) {
  Table<N> t;
  int nparts = 0;
  for (int at = 0; at < l.n;) {
    at = fill(t, l, at);
    if (t.n == 0) break;
    const int blocks = blocks_for(t.first[t.n]);
    if (kind == P2) norm_kernel<N, P2><<<blocks, THREADS, 0, st>>>(t, part + nparts), MC_COUNT(1);
    else if (kind == P1) norm_kernel<N, P1><<<blocks, THREADS, 0, st>>>(t, part + nparts), MC_COUNT(1);
    else norm_kernel<N, PINF><<<blocks, THREADS, 0, st>>>(t, part + nparts), MC_COUNT(1);
    MC_CHECK_LAUNCH();
    nparts += blocks;
  }
  if (!scale || nparts == 0)
    return launch_behind(finish_kernel, 1, st, nparts > 0, kind, (const double*)part, nparts, norm, norm32);
  bool first = true;
  for (int at = 0; at < l.n;) {
    at = fill(t, l, at);
    if (t.n == 0) break;
    const int rc = launch_behind(scale_kernel<N>, blocks_for(t.first[t.n]), st, first, (const Table<N>)t, kind,
                                 (const double*)part, nparts, max_norm, first ? norm : (double*)nullptr,
                                 first ? norm32 : (float*)nullptr);
    if (rc) return rc;
    first = false;
  }
  return MC_OK;
}

static int run_sized(const Lists& l, bool scale, double norm_type, double max_norm, double* norm, float* norm32, void* ws,
                     size_t ws_bytes, void* stream) {
  const int rc = check_lists(l, scale), kind = kind_of(norm_type);
  if (rc) return rc;
  if (kind == 0) return MC_ERR_UNSUPPORTED;
  if (scale && !(max_norm >= 0)) return MC_ERR_BAD_ARG;
  if (!ws || ws_bytes < mc_grad_workspace_bytes(l.n)) return MC_ERR_WORKSPACE;
  if ((uintptr_t)ws % sizeof(double)) return MC_ERR_BAD_ARG;
  return l.n <= SMALL ? run<SMALL>(l, scale, kind, max_norm, norm, norm32, (double*)ws, (cudaStream_t)stream)
                      : run<LARGE>(l, scale, kind, max_norm, norm, norm32, (double*)ws, (cudaStream_t)stream);
}

}  // namespace grad
}  // namespace mc
using namespace mc;

extern "C" {

size_t mc_grad_workspace_bytes(int32_t n) {
  // one double per block of the first kernel, for each launch of up to LARGE tensors
  return (1 + (size_t)(n > 0 ? n : 0) / grad::LARGE) * grad::MAX_BLOCKS * sizeof(double);
}
int mc_grad_norm(int32_t n, const void* const* src, const int64_t* numel, const int32_t* dtype, double norm_type,
                 double* norm, float* norm32, void* ws, size_t ws_bytes, void* stream) {
  const grad::Lists l{n, src, dtype, nullptr, nullptr, numel};
  return grad::run_sized(l, false, norm_type, 0, norm, norm32, ws, ws_bytes, stream);
}
int mc_grad_clip(int32_t n, const void* const* src, const int32_t* src_dtype, void* const* dst, const int32_t* dst_dtype,
                 const int64_t* numel, double norm_type, double max_norm, double* norm, float* norm32, void* ws,
                 size_t ws_bytes, void* stream) {
  const grad::Lists l{n, src, src_dtype, dst, dst_dtype, numel};
  return grad::run_sized(l, true, norm_type, max_norm, norm, norm32, ws, ws_bytes, stream);
}

}  // extern "C"
