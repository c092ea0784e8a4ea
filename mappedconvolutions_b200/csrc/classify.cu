// Softmax cross entropy of a pointwise classifier.
//
// With P = B * S pixels, row vectors x_p, class scores z_p = x_p W^T + b (V of them) and labels t_p:
//   top_p = max_v z_pv,   rest_p = log sum_v exp(z_pv - top_p),   loss_p = (top_p - z_p,t_p) + rest_p,   loss = scale sum_p loss_p
//   gz_pv = g scale exp((z_pv - top_p) - rest_p),  of the label g scale (e^-loss_p - 1),   gx = gz W,   gW = gz^T x,   gb = sum_p gz
// with scale = 1 / labelled pixels, or 1.  (top + rest is never formed: see Softmax.)
// A pixel whose label is `ignore` counts nothing: its top is kept as +infinity, its gz is zero and its features are read as
// zeros, whatever they are.  A label outside [0, V) makes the loss NaN, and the gradients that the pixel takes part in: its top is kept as NaN.
//
// bf16 (tensor cores): the scores of 256 pixels x up to 256 classes stand in TMEM; the forward call keeps their largest and the
// sum of their exponentials, the backward call computes them again, rounds gz to bf16 - which the next two products' operand is -
// and multiplies it, a piece of the pixels at a time.
// float32 with many products (tensor cores): the same kernels on three bf16 parts of every value, six products of parts for one
// (FloatCores below has the rule and both sides measured).  Bound: the products; the parts' copies where channels are few.
// float64, and float32 otherwise (CUDA cores), with the kernels of the channel-mixing layers: up to 128 classes stand in a block's
// registers, whose threads add up the softmax; scores of more classes go through the workspace, a piece of the pixels at a time.
// Bound: the products (FMA issue).
#include "act_pairs.cuh"
#include "mix_work.cuh"

namespace mc {
namespace classify {
using mix::RowsArgs;
using mix::View;

// What a forward call keeps: the number of labelled pixels (a double), from byte 256 on top, rest (in base 2 where the tensor cores read it)
// and miss of every pixel, and behind them the input as rows of channels where it lies in another way (bf16).
constexpr size_t KEPT_HEAD = 256;
using mix::Softmax;
template <typename T>
static size_t kept_bytes(long long pixels) { return KEPT_HEAD + 3 * mix::up256((size_t)pixels * sizeof(T)); }
template <typename T>
static Softmax<T> softmax_of(void* kept, long long pixels) {
  char* p = (char*)kept + KEPT_HEAD;
  const size_t n = mix::up256((size_t)pixels * sizeof(T));
  return Softmax<T>{(T*)p, (T*)(p + n), (T*)(p + 2 * n)};
}
constexpr size_t PIECE = 256u << 20;     // bytes of scores or gz at a time, CUDA cores
constexpr int FEW = 128;                 // classes that the CUDA-core kernels keep in registers
constexpr size_t PIECE_TC = 1024u << 20; // bytes of gz at a time, tensor cores
constexpr int THREADS = 256;
constexpr int SUM_BLOCKS = 296;          // blocks that add losses up

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
__device__ __forceinline__ float log_of(float v) { return logf(v); }
__device__ __forceinline__ double log_of(double v) { return log(v); }
__device__ __forceinline__ float expm1_of(float v) { return expm1f(v); }
__device__ __forceinline__ double expm1_of(double v) { return expm1(v); }

// The kernels that this is called in start while the one before them runs; here they wait until all that it wrote can be read.
__device__ __forceinline__ void behind_previous_kernel() {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... A>
static int launch_behind(void (*kern)(A...), int blocks, cudaStream_t st, A... args) {
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, args...) != cudaSuccess) return MC_ERR_LAUNCH;
  MC_COUNT(1);
  return MC_OK;
}

template <typename CT>
__device__ __forceinline__ CT warp_sum(CT v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

template <typename T> struct alignas(16) Four { T v[4]; };
// what is kept of the rows of a piece, and their losses, one warp to a row of ld (a multiple of 4) scores
template <typename T>
__global__ void __launch_bounds__(THREADS) softmax_kernel(const T* __restrict__ z, int ld, const int64_t* __restrict__ target,
                                                          long long n, int V, long long ignore, Softmax<T> kept, T* __restrict__ value) {
  const long long row = blockIdx.x * (long long)(THREADS / 32) + threadIdx.x / 32;
  if (row >= n) return;
  const int lane = threadIdx.x % 32;
  const long long t = target[row];
  T top = -T(INFINITY), rest = T(0), loss = T(0);
  if (t == ignore) {
    top = T(INFINITY);
  } else if (t < 0 || t >= V) {
    top = loss = T(NAN);
  } else {
    const T* r = z + row * ld;
    T sum = T(0);
#pragma unroll 4
    for (int v = lane * 4; v < V; v += 128) {
      const Four<T> q = *reinterpret_cast<const Four<T>*>(r + v);
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmax(top, v + e < V ? q.v[e] : -T(INFINITY));  // (a NaN shows in the sum)
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmax(top, __shfl_xor_sync(~0u, top, o));
#pragma unroll 4
    for (int v = lane * 4; v < V; v += 128) {
      const Four<T> q = *reinterpret_cast<const Four<T>*>(r + v);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += v + e < V ? exp_of(q.v[e] - top) : T(0);
    }
    rest = log_of(warp_sum(sum));
    loss = top - r[t] + rest;
  }
  if (lane == 0) kept.top[row] = top, kept.rest[row] = rest, kept.miss[row] = expm1_of(-loss), value[row] = loss;
}

// z <- gz
template <typename T>
__global__ void __launch_bounds__(THREADS) score_grad_kernel(T* __restrict__ z, int ld, const int64_t* __restrict__ target,
                                                             Softmax<T> kept, long long n, int V, const double* count, const T* grad) {
  const T scale = count ? (T)((double)*grad / *count) : *grad;
  for (long long row = blockIdx.x * (long long)(THREADS / 32) + threadIdx.x / 32; row < n; row += gridDim.x * (long long)(THREADS / 32)) {
    const T top = kept.top[row], rest = kept.rest[row], miss = kept.miss[row];
    const long long t = target[row];
    T* r = z + row * ld;
#pragma unroll 2
    for (int v = threadIdx.x % 32 * 4; v < V; v += 128) {
      Four<T> q = *reinterpret_cast<const Four<T>*>(r + v);
#pragma unroll
      for (int e = 0; e < 4; ++e) q.v[e] = top == T(INFINITY) ? T(0) : scale * (v + e == t ? miss : exp_of(q.v[e] - top - rest));
      *reinterpret_cast<Four<T>*>(r + v) = q;
    }
  }
}

// (images of n pixels, C) wherever they lie -> rows; those of pixels without a label are zero
template <typename T>
__global__ void __launch_bounds__(THREADS) rows_kernel(const T* __restrict__ src, long long img, long long pix, long long ch, long long n,
                                                       int C, const T* __restrict__ top, T* __restrict__ dst) {
  src += blockIdx.z * img, top += blockIdx.z * n, dst += blockIdx.z * n * C;
  __shared__ T tile[32][33];
  // 32 pixels x 32 channels, read along whichever direction is contiguous
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  const long long p0 = blockIdx.x * 32ll;
  for (int c0 = blockIdx.y * 32; c0 < C; c0 += gridDim.y * 32) {
    __syncthreads();
    for (int k = ty; k < 32; k += THREADS / 32) {
      const long long p = p0 + (ch == 1 ? k : tx);
      const int c = c0 + (ch == 1 ? tx : k);
      tile[ch == 1 ? k : tx][ch == 1 ? tx : k] = p < n && c < C && top[p] != T(INFINITY) ? src[p * pix + (long long)c * ch] : T(0);
    }
    __syncthreads();
    for (int k = ty; k < 32; k += THREADS / 32)
      if (p0 + k < n && c0 + tx < C) dst[(p0 + k) * C + c0 + tx] = tile[k][tx];
  }
}
// acc (+)= the shares of one piece, in order; the last piece's sums go to `out`
template <typename T>
__global__ void __launch_bounds__(THREADS) gather_kernel(const T* __restrict__ part, long long n, int splits, T* __restrict__ acc,
                                                         bool first, T* __restrict__ out) {
  for (long long i = blockIdx.x * (long long)THREADS + threadIdx.x; i < n; i += gridDim.x * (long long)THREADS) {
    T s = first ? T(0) : acc[i];
    for (int j = 0; j < splits; ++j) s += part[j * n + i];
    (out ? out : acc)[i] = s;
  }
}

template <typename CT>
__global__ void __launch_bounds__(THREADS) loss_part_kernel(const CT* __restrict__ value, const int64_t* __restrict__ target,
                                                            long long P, long long ignore, double* part) {
  __shared__ double sm[2][THREADS / 32];
  double s = 0, n = 0;
  for (long long p = blockIdx.x * (long long)THREADS + threadIdx.x; p < P; p += gridDim.x * (long long)THREADS)
    if (target[p] != ignore) s += (double)value[p], n += 1;
  s = warp_sum(s), n = warp_sum(n);
  if (threadIdx.x % 32 == 0) sm[0][threadIdx.x / 32] = s, sm[1][threadIdx.x / 32] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < THREADS / 32; ++i) s += sm[0][i], n += sm[1][i];
    part[2 * blockIdx.x] = s, part[2 * blockIdx.x + 1] = n;
  }
}
template <typename CT>
__global__ void __launch_bounds__(THREADS) loss_kernel(const double* part, int blocks, bool mean, double* count, CT* loss) {
  __shared__ double sm[2][THREADS / 32];
  behind_previous_kernel();
  double s = 0, n = 0;
  for (int i = threadIdx.x; i < blocks; i += THREADS) s += part[2 * i], n += part[2 * i + 1];
  s = warp_sum(s), n = warp_sum(n);
  if (threadIdx.x % 32 == 0) sm[0][threadIdx.x / 32] = s, sm[1][threadIdx.x / 32] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < THREADS / 32; ++i) s += sm[0][i], n += sm[1][i];
    *count = n;
    *loss = (CT)(mean ? s / n : s);  // (no labelled pixel: 0 / 0)
  }
}
// ---- bf16 -----------------------------------------------------------------------------------------------
// The tiles' sums of a pixel become what is kept of it; the blocks' losses and labelled pixels go to `part`.
// (It starts while the kernel that writes those sums still runs, and a later piece's sums take the same place: read behind L1, never
// through the read-only path.)
__global__ void __launch_bounds__(THREADS) finish_kernel(mix::Scores s, int tiles, long long P, int V, Softmax<float> kept, double* part) {
  __shared__ double sm[2][THREADS / 32];
  behind_previous_kernel();
  double sum = 0, n = 0;
  for (long long p = blockIdx.x * (long long)THREADS + threadIdx.x; p < P; p += gridDim.x * (long long)THREADS) {
    const long long t = s.target[p];
    if (t == s.ignore) {
      kept.top[p] = INFINITY, kept.rest[p] = kept.miss[p] = 0.f;
      continue;
    }
    n += 1;
    float top = NAN, rest = 0.f, loss = NAN;
    if (t >= 0 && t < V) {
      top = -INFINITY;
#pragma unroll 8
      for (int k = 0; k < tiles; ++k) top = fmaxf(top, __ldcg(&s.part[k * P + p].x));  // (a NaN shows in the sum)
      float all = 0.f;
#pragma unroll 8
      for (int k = 0; k < tiles; ++k) {
        const float2 v = __ldcg(s.part + k * P + p);
        all += v.y * exp2f((v.x - top) * mix::LOG2E);
      }
      rest = log2f(all);
      loss = top - __ldcg(s.hit + p) + rest * 0.69314718056f;
    }
    sum += (double)loss;
    kept.top[p] = top, kept.rest[p] = rest, kept.miss[p] = expm1f(-loss);
  }
  sum = warp_sum(sum), n = warp_sum(n);
  if (threadIdx.x % 32 == 0) sm[0][threadIdx.x / 32] = sum, sm[1][threadIdx.x / 32] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < THREADS / 32; ++i) sum += sm[0][i], n += sm[1][i];
    part[2 * blockIdx.x] = sum, part[2 * blockIdx.x + 1] = n;
  }
}
// rows of `per` 16-byte vectors: those of pixels without a label become zeros, the others are copied (or stay, in place)
__global__ void __launch_bounds__(THREADS) labelled_rows_kernel(const uint4* src, uint4* dst, const int64_t* __restrict__ target,
                                                                long long ignore, long long n, int per) {
  for (long long i = blockIdx.x * (long long)THREADS + threadIdx.x; i < n; i += gridDim.x * (long long)THREADS) {
    const bool off = target[i / per] == ignore;
    if (off) dst[i] = make_uint4(0, 0, 0, 0);
    else if (src != dst) dst[i] = __ldg(src + i);
  }
}
// n pixels of images of S pixels, wherever they lie -> rows of three bf16 parts of float32 values, 8 bits each, zeros behind the last
// channel of a part of Cp; pixels without a label are zeros if top is given.  (An infinity would leave NaN in the lower parts: they
// are zero there.)
// A block takes 32 pixels x 64 channels, eight values to a thread either way (one at a time: 40 us instead of 15 for 131 072 pixels of
// 50 channels).
// Up to three such jobs a launch: weights, their transposes and pixels.
struct Split {
  const float* src;
  long long S, img, pix, ch, p1, n;
  int C, Cp;
  const float* top;
  bf16* dst;
  unsigned blocks;
};
struct Splits { Split s[3]; };
__global__ void __launch_bounds__(THREADS) parts_kernel(const __grid_constant__ Splits all) {
  __shared__ float tile[32][65];
  unsigned block = blockIdx.x;
  int job = 0;
  while (job < 2 && block >= all.s[job].blocks) block -= all.s[job++].blocks;
  const Split& a = all.s[job];
  const float *src = a.src, *top = a.top;
  const long long S = a.S, img = a.img, pix = a.pix, ch = a.ch, p1 = a.p1, n = a.n;
  const int C = a.C, Cp = a.Cp, tx = threadIdx.x % 32, ty = threadIdx.x / 32, c0 = block % (Cp / 64) * 64;
  const long long p0 = block / (Cp / 64) * 32ll;
  const bool along = ch == 1;  // neighbouring threads read neighbouring channels, else pixels
  float v[8];
  if (along) {  // (one image)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = c0 + tx + 32 * (k / 4);
      const long long p = p0 + ty + 8 * (k % 4);
      v[k] = p < n && c < C && !(top && top[p] == INFINITY) ? __ldg(src + (p1 + p) * pix + c) : 0.f;
    }
  } else {
    const long long p = p0 + tx, b = (p1 + p) / S;
    const bool on = p < n && !(top && top[p] == INFINITY);
    const float* from = src + b * img + (p1 + p - b * S) * pix;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = on && c0 + ty + 8 * k < C ? __ldg(from + (c0 + ty + 8 * k) * ch) : 0.f;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) tile[along ? ty + 8 * (k % 4) : tx][along ? tx + 32 * (k / 4) : ty + 8 * k] = v[k];
  __syncthreads();
  const int r = threadIdx.x / 8, c = threadIdx.x % 8 * 8;
  if (p0 + r >= n) return;
  bf16* to = a.dst + (p0 + r) * 3 * Cp + c0 + c;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = tile[r][c + k];
#pragma unroll
  for (int part = 0; part < 3; ++part) {
    __align__(16) bf16 h[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      h[k] = __float2bfloat16_rn(v[k]);
      float f = __bfloat162float(h[k]);
      if (fabsf(f) == INFINITY && fabsf(v[k]) < INFINITY) h[k] = __float2bfloat16_rz(v[k]), f = __bfloat162float(h[k]);  // (largest values)
      v[k] = fabsf(f) < INFINITY ? v[k] - f : 0.f;
    }
    *reinterpret_cast<uint4*>(to + part * Cp) = *reinterpret_cast<const uint4*>(h);
  }
}

// (V, C) -> (C, 2 pad): every channel's weights twice, zeros behind the last class of each (pad: a multiple of 8)
__global__ void __launch_bounds__(THREADS) twice_transposed_kernel(const bf16* __restrict__ w, bf16* __restrict__ dst, int V, int C, int pad) {
  const int c = blockIdx.x * THREADS + threadIdx.x;
  if (c >= C) return;
  for (int v0 = 0; v0 < pad; v0 += 8) {
    __align__(16) bf16 q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = v0 + e < V ? w[(long long)(v0 + e) * C + c] : bf16(0.f);
#pragma unroll
    for (int part = 0; part < 2; ++part)
      *reinterpret_cast<uint4*>(dst + (long long)c * 2 * pad + part * pad + v0) = *reinterpret_cast<const uint4*>(q);
  }
}
// acc (+)= the shares of one piece, in order: sums (V, C) in rows of ldn (a multiple of 4), and V column sums, of shares of R rows; the
// last piece's go to gw and gb, rounded.  Four sums to a thread.
template <typename T>
__global__ void __launch_bounds__(THREADS) add_piece_kernel(const float* __restrict__ part, const float* __restrict__ csum, int splits,
                                                            int V, int R, int C, int ldn, float* __restrict__ acc, bool first,
                                                            bool last, T* gw, T* gb) {
  const long long nw = (long long)V * (ldn / 4), step = (long long)R * (ldn / 4), i = blockIdx.x * (long long)THREADS + threadIdx.x;
  if (i < nw) {
    float4 s = first ? make_float4(0.f, 0.f, 0.f, 0.f) : reinterpret_cast<const float4*>(acc)[i];
#pragma unroll 8
    for (int j = 0; j < splits; ++j) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(part) + j * step + i);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    if (!last) {
      reinterpret_cast<float4*>(acc)[i] = s;
    } else if (gw) {
      const int row = (int)(i / (ldn / 4)), c = (int)(i % (ldn / 4)) * 4;
      const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < C) stv(gw + (long long)row * C + c + e, v[e]);
    }
  } else if (i < nw + V) {
    const long long v = i - nw;
    float s = first ? 0.f : acc[4 * nw + v];
    for (int j = 0; j < splits; ++j) s += csum[j * (long long)R + v];
    if (!last) acc[4 * nw + v] = s;
    else if (gb) stv(gb + v, s);
  }
}

// ---- host -----------------------------------------------------------------------------------------------
using mix::up256;
static size_t csize(int dtype) { return dtype == MC_F64 ? 8 : 4; }
static size_t esize(int dtype) { return dtype == MC_F64 ? 8 : dtype == MC_F32 ? 4 : 2; }
static bool on(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

static int check_desc(const mc_ce_desc* d) {
  if (!d || d->B <= 0 || d->S <= 0 || d->C <= 0 || d->V <= 0) return MC_ERR_BAD_ARG;
  if (d->dtype != MC_F32 && d->dtype != MC_F64 && d->dtype != MC_BF16) return MC_ERR_BAD_ARG;
  if (d->layout != MC_NCHW && d->layout != MC_NHWC) return MC_ERR_BAD_ARG;
  if (d->reduction != MC_REDUCE_SUM && d->reduction != MC_REDUCE_MEAN) return MC_ERR_BAD_ARG;
  if (d->S >= (1ll << 31) || d->B >= (1ll << 31) || d->B * d->S > (1ll << 31) - 256) return MC_ERR_TOO_LARGE;
  if (d->C > (1 << 20) || d->V > (1 << 20) || (long long)d->C * d->V > (1ll << 31)) return MC_ERR_TOO_LARGE;
  return MC_OK;
}

// The pixels in pieces: several images, or part of one.
struct Pieces {
  long long S, B;    // pixels of an "image": channels-last batches are one
  long long images, run;  // of a piece: images > 1 or a run of an image
  Pieces(const mc_ce_desc* d) {
    const bool whole = d->layout == MC_NHWC || d->S == 1 || d->B == 1;
    S = whole ? d->B * d->S : d->S, B = whole ? 1 : d->B;
    const size_t row = (size_t)((d->V > d->C ? d->V : d->C) + 3) / 4 * 4 * csize(d->dtype);
    long long n = (long long)(PIECE / row);
    n = n < 32 ? 32 : n / 32 * 32;
    images = n >= S ? n / S : 1;
    if (images > B) images = B;
    run = images > 1 || n >= S ? S : n;
  }
  long long most() const { return images * run; }
};

// Lays a call's memory out; without a base it only adds up.
struct Memory {
  char* base;
  size_t used = 0;
  explicit Memory(void* b) : base((char*)b) {}
  void* take(size_t n) {
    void* p = base ? base + used : nullptr;
    used += up256(n);
    return p;
  }
};
struct Shares {
  long long share;
  int splits;
  Shares(long long n, int V, int C) {
    const long long tiles = (long long)((V + 127) / 128) * ((C + 127) / 128);
    long long want = (2 * 148 + tiles - 1) / tiles, most = (n + 255) / 256;
    if (want > most) want = most;
    share = ((n + want - 1) / want + 15) / 16 * 16;
    splits = (int)((n + share - 1) / share);
  }
};

// The way of float32 and float64 layers.
template <typename T>
struct General {
  const mc_ce_desc* d;
  Pieces pieces;
  Memory m;
  cudaStream_t st;
  const bool few;
  const int ld;  // of a row of scores
  T *z = nullptr, *rows = nullptr, *value = nullptr, *part = nullptr, *csum = nullptr, *acc = nullptr;
  double* sums = nullptr;

  General(const mc_ce_desc* desc, void* ws, bool backward, cudaStream_t s)
      : d(desc), pieces(desc), m(ws), st(s), few(desc->V <= FEW), ld((desc->V + 3) / 4 * 4) {
    const size_t n = pieces.most(), C = d->C, V = d->V;
    if (backward || !few) z = (T*)m.take(n * ld * sizeof(T));
    if (!backward) {
      value = (T*)m.take((size_t)d->B * d->S * sizeof(T));
      sums = (double*)m.take(SUM_BLOCKS * 16);
    } else {
      rows = (T*)m.take(n * C * sizeof(T));
      int splits = 1;
      each([&](long long, long long, long long k) {
        const Shares sh(k, d->V, d->C);
        if (sh.splits > splits) splits = sh.splits;
      });
      part = (T*)m.take((size_t)splits * V * C * sizeof(T));
      csum = (T*)m.take((size_t)splits * V * sizeof(T));
      acc = (T*)m.take((long long)n < d->B * d->S ? (V * C + V) * sizeof(T) : 0);
    }
  }
  // f(image, first pixel of it, pixels in all)
  template <typename F>
  void each(F f) const {
    for (long long i = 0; i < pieces.B; i += pieces.images) {
      const long long images = pieces.B - i < pieces.images ? pieces.B - i : pieces.images;
      for (long long s = 0; s < pieces.S; s += pieces.run) f(i, s, images * (pieces.S - s < pieces.run ? pieces.S - s : pieces.run));
    }
  }
  bool planes() const { return !(d->layout == MC_NHWC || d->S == 1) && d->C > 1; }
  template <typename X>
  View view(X* p, long long i, long long s) const {
    View v;
    v.img = pieces.S * d->C;
    if (planes()) v.pix = 1, v.ch = d->S;
    else v.pix = d->C, v.ch = 1;
    v.ptr = p + i * v.img + s * v.pix;
    return v;
  }
  View flat(const T* p, long long n, int wide) const { return View{p, n * wide, wide, 1}; }
  // labelled pixels of a piece as rows (several images one after the other)
  void gather(const T* x, long long i, long long s, long long n, const T* top) {
    const long long per = n < pieces.S ? n : pieces.S;
    const View v = view(x, i, s);
    for (long long k = 0; k * per < n; k += 32768) {  // (images are the grid's third dimension)
      const long long images = n / per - k < 32768 ? n / per - k : 32768;
      const dim3 tiles((unsigned)((per + 31) / 32), (unsigned)((d->C + 31) / 32 < 64 ? (d->C + 31) / 32 : 64), (unsigned)images);
      rows_kernel<T><<<tiles, THREADS, 0, st>>>((const T*)v.ptr + k * v.img, v.img, v.pix, v.ch, per, d->C, top + k * per,
                                                rows + k * per * d->C), MC_COUNT(1);
    }
  }
  // x W^T + b of n pixels
  RowsArgs product(const View& x, long long n, long long S, const T* w, const T* b) const {
    RowsArgs r{};
    r.a = x, r.w = w, r.wn = d->C, r.wk = 1, r.bias = b, r.y = View{z, S * (long long)ld, ld, 1}, r.P = n, r.S = (int)S, r.N = d->V, r.K = d->C;
    return r;
  }

  int forward(const T* x, const T* w, const T* b, const int64_t* target, T* loss, void* kept) {
    const long long P = d->B * d->S;
    const Softmax<T> soft = softmax_of<T>(kept, P);
    int rc = MC_OK;
    if (few) {
      RowsArgs r = product(view(x, 0, 0), P, pieces.S, w, b);
      r.y.ptr = nullptr;
      r.labels = mix::Labels{target, d->ignore_index, soft.top, soft.rest, soft.miss, value};
      rc = mix::simt_rows_launch(d->dtype, mix::EPI_SCORE_SUM, r, st);
    } else {
      each([&](long long i, long long s, long long n) {
        if (rc) return;
        const long long p = i * pieces.S + s;
        if ((rc = mix::simt_rows_launch(d->dtype, mix::EPI_LAYER, product(view(x, i, s), n, n < pieces.S ? n : pieces.S, w, b), st))) return;
        softmax_kernel<T><<<(unsigned)((n + 7) / 8), THREADS, 0, st>>>(z, ld, target + p, n, d->V, d->ignore_index, soft.at(p), value + p);
        MC_COUNT(1);
      });
    }
    if (rc) return rc;
    const int blocks = grid_for(P, 4 * THREADS, SUM_BLOCKS);
    loss_part_kernel<T><<<blocks, THREADS, 0, st>>>(value, target, P, d->ignore_index, sums), MC_COUNT(1);
    MC_CHECK_LAUNCH();
    return launch_behind(loss_kernel<T>, 1, st, (const double*)sums, (int)blocks, d->reduction == MC_REDUCE_MEAN, (double*)kept, (T*)loss);
  }

  int backward(const T* grad, const T* x, const T* w, const T* b, const int64_t* target, const void* kept, T* gx, T* gw, T* gb) {
    const long long P = d->B * d->S;
    const Softmax<T> soft = softmax_of<T>((void*)kept, P);
    const double* count = d->reduction == MC_REDUCE_MEAN ? (const double*)kept : nullptr;
    const long long VC = (long long)d->V * d->C;
    int rc = MC_OK;
    each([&](long long i, long long s, long long n) {
      if (rc) return;
      const long long p = i * pieces.S + s, S = n < pieces.S ? n : pieces.S;
      gather(x, i, s, n, soft.top + p);
      RowsArgs r = product(flat(rows, n, d->C), n, n, w, b);
      r.labels = mix::Labels{target + p, d->ignore_index, soft.top + p, soft.rest + p, soft.miss + p, nullptr, grad, count};
      if ((rc = mix::simt_rows_launch(d->dtype, few ? mix::EPI_SCORE_GRAD : mix::EPI_LAYER, r, st))) return;
      if (!few)
        score_grad_kernel<T><<<grid_for(n, 8, 148 * 8), THREADS, 0, st>>>(z, ld, target + p, soft.at(p), n, d->V, count, grad), MC_COUNT(1);
      if (gx) {
        r = RowsArgs{};
        r.a = View{z, S * (long long)ld, ld, 1}, r.w = w, r.wn = 1, r.wk = d->C, r.P = n, r.N = d->C, r.K = d->V, r.S = (int)S;
        r.y = view(gx, i, s);
        if ((rc = mix::simt_rows_launch(d->dtype, mix::EPI_LAYER, r, st))) return;
      }
      if (gw || gb) {
        const Shares sh(n, d->V, d->C);
        const mix::OuterArgs o{flat(z, n, ld), flat(rows, n, d->C), part, csum, n, sh.share, d->V, d->C, 1, 1, sh.splits, sh.splits};
        if ((rc = mix::simt_outer_launch(d->dtype, o, st))) return;
        const bool first = p == 0, last = p + n == P;
        if (first && last) {
          mix::add_shares<T, T>(part, d->V, d->C, d->C, gw, csum, gb, sh.splits, st);
        } else {
          if (gw) gather_kernel<T><<<grid_for(VC, THREADS, 1184), THREADS, 0, st>>>(part, VC, sh.splits, acc, first, last ? gw : nullptr), MC_COUNT(1);
          if (gb) gather_kernel<T><<<grid_for(d->V, THREADS, 1184), THREADS, 0, st>>>(csum, d->V, sh.splits, acc + VC, first, last ? gb : nullptr), MC_COUNT(1);
        }
      }
    });
    if (rc) return rc;
    MC_CHECK_LAUNCH();
    return MC_OK;
  }
};

// The way of bf16 layers.
struct TensorCores {
  const mc_ce_desc* d;
  mc_mix_desc like;  // the same tensors as the channel-mixing kernels describe them
  explicit TensorCores(const mc_ce_desc* desc) : d(desc) {
    like = mc_mix_desc{d->B, d->S, d->C, d->V, 0, MC_ACT_NONE, MC_BF16, d->layout};
  }
  long long pixels() const { return d->B * d->S; }
  bool in_place() const { return mix::Work::in_place(&like, d->C); }
  int parts() const { return d->V <= 32 ? 2 : 1; }  // of gz, see backward
  size_t saved_bytes() const {
    return kept_bytes<float>(pixels()) + (in_place() ? 0 : up256((size_t)pixels() * mix::pad8(d->C) * 2));
  }
  mix::TcRows rows_of(const void* p, long long n) const { return mix::TcRows{p, n, d->C, mix::pad8(d->C)}; }
  void labelled(const void* src, const mix::TcRows& r, const int64_t* target, cudaStream_t st) const {
    const int per = r.ld / 8;
    const long long n = r.rows * per;
    labelled_rows_kernel<<<grid_for(n, THREADS, 148 * 16), THREADS, 0, st>>>((const uint4*)src, (uint4*)r.p, target, d->ignore_index, n,
                                                                             per), MC_COUNT(1);
  }

  int forward(mix::Work& k, const bf16* x, const bf16* w, const bf16* bias, const int64_t* target, float* loss, char* kept) const {
    mix::TcRows xr = rows_of(x, pixels());
    if (!in_place()) {
      xr.p = kept ? kept + kept_bytes<float>(pixels()) : nullptr;
      k.lay_out(&like, x, xr, target, d->ignore_index);
      if (k.run() && !mix::Work::as_planes(&like, d->C)) labelled(xr.p, xr, target, k.st);
    }
    const mix::TcRows wr = k.weight(w, d->V, d->C);
    // (the tiles' sums of very many scores: a piece of the pixels at a time)
    const long long P = pixels(), piece = sum_piece(), last = (P - 1) % piece + 1, pieces = (P + piece - 1) / piece;
    const auto tiles = [&](long long n) { return mix::tc_scores_tiles(n, d->C, d->V); };
    const size_t one = (size_t)tiles(piece) * piece, other = (size_t)tiles(last) * last;
    mix::Scores s{target, d->ignore_index};
    s.part = (float2*)k.take((one > other ? one : other) * 8);
    s.hit = (float*)k.take((size_t)piece * 4);
    double* part = (double*)k.take((size_t)pieces * SUM_BLOCKS * 16);
    if (!k.run()) return k.rc;
    int blocks = 0;
    for (long long p = 0; p < P; p += piece) {
      const long long n = P - p < piece ? P - p : piece;
      s.target = target + p;
      k.did(mix::tc_scores_sum(rows_of((const bf16*)xr.p + p * xr.ld, n), wr, bias, s, k.st));
      if (k.rc) return k.rc;
      const int more = grid_for(n, THREADS, SUM_BLOCKS);
      k.did(launch_behind(finish_kernel, more, k.st, (mix::Scores)s, (int)tiles(n), (long long)n, (int)d->V,
                          softmax_of<float>(kept, P).at(p), (double*)(part + 2 * blocks)));
      if (k.rc) return k.rc;
      blocks += more;
    }
    return launch_behind(loss_kernel<float>, 1, k.st, (const double*)part, (int)blocks, d->reduction == MC_REDUCE_MEAN, (double*)kept,
                         (float*)loss);
  }
  long long sum_piece() const {
    const long long most = (long long)(PIECE_TC / 8) / ((d->V + 63) / 64) / 256 * 256;  // (tiles are 64 classes wide at least)
    return most >= pixels() ? pixels() : most < 256 ? 256 : most;
  }

  // Pixels of a piece: whole images, or part of one.
  struct Cut {
    long long images, run;
    Cut(const TensorCores& t) {
      const mc_ce_desc* d = t.d;
      const bool whole = !mix::Work::as_planes(&t.like, d->C);  // (the output need not be cut at images)
      const long long S = whole ? d->B * d->S : d->S, B = whole ? 1 : d->B;
      long long n = (long long)(PIECE_TC / ((size_t)mix::pad8(d->V) * 2 * t.parts())) / 256 * 256;
      if (n < 256) n = 256;
      images = n >= S ? n / S : 1;
      if (images > B) images = B;
      run = n >= S ? S : n;
    }
  };
  int backward(mix::Work& k, const float* grad, const bf16* x, const bf16* w, const bf16* bias, const int64_t* target,
               const char* kept, bf16* gx, bf16* gw, bf16* gb) const {
    const long long P = pixels();
    const Cut cut(*this);
    const bool planes = mix::Work::as_planes(&like, d->C);
    const long long S = planes ? d->S : P, B = planes ? d->B : 1, most = cut.images * cut.run;
    mix::TcRows xr = rows_of(kept ? kept + kept_bytes<float>(P) : nullptr, P);
    if (in_place()) {
      xr = k.fresh(P, d->C);
      if (k.run()) labelled(x, xr, target, k.st);
    }
    const mix::TcRows wr = k.weight(w, d->V, d->C);
    // Up to 32 classes: gz in two bf16 parts side by side, against every weight twice.  Both products' stages hold 64 columns in any case:
    // gx and gW are rounded once, not twice, at no cost.  (More classes: see read_scores.)
    const int pad = mix::pad8(d->V), parts = this->parts(), across = parts * (parts > 1 ? pad : d->V);
    mix::TcRows wt{nullptr, d->C, across, parts * pad};
    if (parts > 1) {
      wt.p = k.take((size_t)d->C * wt.ld * 2);
      if (k.run() && gx) twice_transposed_kernel<<<(d->C + THREADS - 1) / THREADS, THREADS, 0, k.st>>>(w, (bf16*)wt.p, d->V, d->C, pad), MC_COUNT(1);
    } else {
      wt = k.weight_t(w, d->V, d->C);
    }
    // (up to 64 classes are one block across: rows of their own length are shorter)
    mix::TcRows gz{nullptr, most, across, d->V > 64 ? 64 : parts * pad, 0, d->V > 64};
    gz.p = k.take(gz.blocks ? gz.block_bytes() : (size_t)most * gz.ld * 2);
    mix::TcRows out = rows_of(nullptr, most);
    if (!planes && !in_place()) out = k.fresh(most, d->C);
    // (shares of the largest piece; the last one can have other numbers of them)
    int splits = 0, ldn = 0;
    size_t floats = 0, sums = 0;
    const auto each = [&](auto f) {
      for (long long i = 0; i < B; i += cut.images)
        for (long long s = 0; s < S; s += cut.run) {
          const long long images = B - i < cut.images ? B - i : cut.images, run = S - s < cut.run ? S - s : cut.run;
          f(i, s, images * run);
        }
    };
    long long seen[2] = {0, 0};  // (there are at most a few sizes of pieces)
    each([&](long long, long long, long long n) {
      if (n == seen[0] || n == seen[1]) return;
      seen[1] = seen[0], seen[0] = n;
      const size_t f = mix::tc_outer_floats(n, across, 1, d->C, &splits, &ldn);
      if (f > floats) floats = f;
      if ((size_t)splits * across > sums) sums = (size_t)splits * across;
    });
    float* part = (float*)k.take(floats * 4);
    float* csum = (float*)k.take(sums * 4);
    const long long sums_all = (long long)d->V * (ldn / 4) + d->V;  // threads of add_piece_kernel
    float* acc = (float*)k.take(most < P ? ((size_t)d->V * ldn + d->V) * 4 : 0);
    if (!k.run()) return k.rc;
    const Softmax<float> soft = softmax_of<float>((void*)kept, P);
    each([&](long long i, long long s, long long n) {
      if (k.rc) return;
      const long long p = i * S + s;
      mix::Scores sc{target + p, d->ignore_index, nullptr, nullptr, {soft.top + p, soft.rest + p, soft.miss + p}, grad,
                     d->reduction == MC_REDUCE_MEAN ? (const double*)kept : nullptr, parts > 1 ? pad / 8 : 0};
      const mix::TcRows xp = rows_of((const bf16*)xr.p + p * xr.ld, n), gp{gz.p, n, across, gz.ld, 0, gz.blocks};
      k.did(mix::tc_scores_grad(xp, wr, bias, sc, gp, k.st));
      if (gx && !k.rc) {
        mix::TcRows to = rows_of(out.p, n);
        if (planes) to = mix::TcRows{gx + i * S * d->C + s, n, d->C, 0, d->S};
        else if (in_place()) to = mix::TcRows{gx + p * d->C, n, d->C, d->C};
        k.did(mix::tc_input_grad(gp, wt, mix::TcRows{}, mix::TcRows{}, to, k.st));
        if (!planes && !in_place() && !k.rc) k.did(mix::copy_rows(to.p, gx + p * d->C, n, to.ld, d->C, k.st));
      }
      if ((gw || gb) && !k.rc) {
        mix::tc_outer_floats(n, across, 1, d->C, &splits, &ldn);
        k.did(mix::tc_outer(gp, mix::TcRows{}, xp, part, csum, k.st));
        if (k.rc) return;
        // (a part's sums are a share of their own)
        const int shares = splits * parts, rows = across / parts;
        // (many shares of few sums: several threads for each)
        if (shares >= 64 && p == 0 && n == P) mix::add_shares<bf16, float>(part, d->V, d->C, ldn, gw, csum, gb, shares, k.st, rows);
        else add_piece_kernel<bf16><<<(unsigned)((sums_all + THREADS - 1) / THREADS), THREADS, 0, k.st>>>(
            part, csum, shares, d->V, rows, d->C, ldn, acc, p == 0, p + n == P, gw, gb), MC_COUNT(1);
        k.did(cudaGetLastError() == cudaSuccess ? MC_OK : MC_ERR_LAUNCH);
      }
    });
    return k.rc;
  }
};
// The way of float32 layers with many products: the tensor cores, on three bf16 parts of every value (see PRODUCTS in mix_tc.cu).
struct FloatCores {
  const mc_ce_desc* d;
  const long long P;
  const int Cp, Vp;
  explicit FloatCores(const mc_ce_desc* desc)
      : d(desc), P(desc->B * desc->S), Cp((desc->C + 63) / 64 * 64), Vp((desc->V + 63) / 64 * 64) {}
  // Sums over channels and over classes are one accumulator's, which truncates up to 2^-23 of what it holds for every sixteen: up to
  // 1024 channels (scores within 2^-17 of their terms, whose differences the exponential takes) and 4096 classes (2^-15 of a sum of
  // one sign).  2^20 channels: a loss 7e-4 off.
  // Forward and backward together, us, tensor cores / CUDA cores: 131 072 pixels, classes x channels 13 x 64 172 / 194, 40 x 64 176 /
  // 228, 99 x 50 208 / 314, 128 x 128 280 / 544; 40 962 pixels, 13 x 64 80 / 101, 40 x 64 82 / 116, 99 x 50 97 / 159, 300 x 96 201 /
  // 468; 10 242 pixels, 40 x 32 61 / 55, 99 x 50 70 / 88, 300 x 64 83 / 125, 700 x 128 122 / 336; 2 562 pixels, 99 x 50 56 / 83,
  // 300 x 64 64 / 94; 1 000 pixels, 40 x 64 52 / 65; 327 684 pixels, 20 x 32 386 / 308, 6 x 16 378 / 255.  (A stage has 64 channels:
  // fewer are paid for in whole.)
  static bool takes(const mc_ce_desc* d) {
    const double each = (double)d->V * d->C;
    return d->dtype == MC_F32 && d->C <= 1024 && d->V <= 4096 && each >= (d->C >= 48 ? 768 : 2048) && each * d->B * d->S >= 2.5e6;
  }
  bool planes() const { return !(d->layout == MC_NHWC || d->S == 1) && d->C > 1; }
  mix::TcRows parts_of(const void* p, long long rows, int cols, int wide) const { return mix::TcRows{p, rows, cols, 3 * wide, 0, false, 3}; }
  static size_t bytes(long long rows, int wide) { return (size_t)rows * 3 * wide * 2; }
  static Split job(const float* src, long long S, long long img, long long pix, long long ch, long long p1, long long n, int C, int wide,
                   const float* top, void* dst) {
    return Split{src, S, img, pix, ch, p1, n, C, wide, top, (bf16*)dst, (unsigned)((n + 31) / 32 * (wide / 64))};
  }
  Split pixels(const float* x, long long p, long long n, const float* top, void* dst) const {
    if (planes()) return job(x, d->S, d->S * d->C, 1, d->S, p, n, d->C, Cp, top, dst);
    return job(x, P, P * d->C, d->C, 1, p, n, d->C, Cp, top, dst);
  }
  Split weights(const float* w, void* dst) const { return job(w, d->V, 0, d->C, 1, 0, d->V, d->C, Cp, nullptr, dst); }
  Split transposed(const float* w, void* dst) const { return job(w, d->C, 0, 1, d->C, 0, d->C, d->V, Vp, nullptr, dst); }
  static int split(const Splits& s, cudaStream_t st) {
    parts_kernel<<<s.s[0].blocks + s.s[1].blocks + s.s[2].blocks, THREADS, 0, st>>>(s), MC_COUNT(1);
    return cudaGetLastError() == cudaSuccess ? MC_OK : MC_ERR_LAUNCH;
  }

  int forward(mix::Work& k, const float* x, const float* w, const float* bias, const int64_t* target, float* loss, char* kept) const {
    long long piece = (long long)(PIECE_TC / ((size_t)((d->V + 63) / 64) * 8 + bytes(1, Cp))) / 256 * 256;
    if (piece < 256) piece = 256;
    if (piece > P) piece = P;
    const long long last = (P - 1) % piece + 1, pieces = (P + piece - 1) / piece;
    const auto tiles = [&](long long n) { return mix::tc_scores_tiles(n, d->C, d->V, 3); };
    const size_t one = (size_t)tiles(piece) * piece, other = (size_t)tiles(last) * last;
    void* x3 = k.take(bytes(piece, Cp));
    void* w3 = k.take(bytes(d->V, Cp));
    mix::Scores s{target, d->ignore_index};
    s.bias32 = bias;
    s.part = (float2*)k.take((one > other ? one : other) * 8);
    s.hit = (float*)k.take((size_t)piece * 4);
    double* part = (double*)k.take((size_t)pieces * SUM_BLOCKS * 16);
    if (!k.run()) return k.rc;
    int blocks = 0;
    for (long long p = 0; p < P; p += piece) {
      const long long n = P - p < piece ? P - p : piece;
      k.did(split(Splits{{pixels(x, p, n, nullptr, x3), p ? Split{} : weights(w, w3)}}, k.st));
      if (k.rc) return k.rc;
      s.target = target + p;
      k.did(mix::tc_scores_sum(parts_of(x3, n, d->C, Cp), parts_of(w3, d->V, d->C, Cp), nullptr, s, k.st));
      if (k.rc) return k.rc;
      const int more = grid_for(n, THREADS, SUM_BLOCKS);
      k.did(launch_behind(finish_kernel, more, k.st, (mix::Scores)s, (int)tiles(n), (long long)n, (int)d->V,
                          softmax_of<float>(kept, P).at(p), (double*)(part + 2 * blocks)));
      if (k.rc) return k.rc;
      blocks += more;
    }
    MC_CHECK_LAUNCH();
    return launch_behind(loss_kernel<float>, 1, k.st, (const double*)part, (int)blocks, d->reduction == MC_REDUCE_MEAN, (double*)kept, loss);
  }

  int backward(mix::Work& k, const float* grad, const float* x, const float* w, const float* bias, const int64_t* target,
               const char* kept, float* gx, float* gw, float* gb) const {
    // pieces of pixels: whole images, or part of one, where the output lies in planes
    const long long S = planes() ? d->S : P, B = planes() ? d->B : 1;
    long long most = (long long)(PIECE_TC / (bytes(1, Vp) + bytes(1, Cp))) / 256 * 256;
    if (most < 256) most = 256;
    const long long run = most < S ? most : S, images = most < S ? 1 : most / S < B ? most / S : B;
    most = images * run;
    const auto each = [&](auto f) {
      for (long long i = 0; i < B; i += images)
        for (long long s = 0; s < S; s += run) f(i, s, (B - i < images ? B - i : images) * (S - s < run ? S - s : run));
    };
    void* x3 = k.take(bytes(most, Cp));
    void* w3 = k.take(bytes(d->V, Cp));
    void* wt3 = k.take(bytes(d->C, Vp));
    mix::TcRows gz{nullptr, most, d->V, 64, 0, true, 3};
    gz.p = k.take(gz.block_bytes());
    int splits = 0, ldn = 0;
    size_t floats = 0, sums = 0;
    long long seen[2] = {0, 0};  // (there are at most a few sizes of pieces)
    each([&](long long, long long, long long n) {
      if (n == seen[0] || n == seen[1]) return;
      seen[1] = seen[0], seen[0] = n;
      const size_t f = mix::tc_outer_floats(n, d->V, 1, d->C, &splits, &ldn, 3);
      if (f > floats) floats = f;
      if ((size_t)splits * d->V > sums) sums = (size_t)splits * d->V;
    });
    float* part = (float*)k.take(floats * 4);
    float* csum = (float*)k.take(sums * 4);
    float* acc = (float*)k.take(most < P ? ((size_t)d->V * ldn + d->V) * 4 : 0);
    if (!k.run()) return k.rc;
    const long long threads = (long long)d->V * (ldn / 4) + d->V;
    const Softmax<float> soft = softmax_of<float>((void*)kept, P);
    each([&](long long i, long long s, long long n) {
      if (k.rc) return;
      const long long p = i * S + s;
      k.did(split(Splits{{pixels(x, p, n, soft.top + p, x3), p ? Split{} : weights(w, w3), p || !gx ? Split{} : transposed(w, wt3)}}, k.st));
      if (k.rc) return;
      mix::Scores sc{target + p, d->ignore_index, nullptr, nullptr, {soft.top + p, soft.rest + p, soft.miss + p}, grad,
                     d->reduction == MC_REDUCE_MEAN ? (const double*)kept : nullptr, 0, bias};
      const mix::TcRows xp = parts_of(x3, n, d->C, Cp), gp{gz.p, n, d->V, 64, 0, true, 3};
      k.did(mix::tc_scores_grad(xp, parts_of(w3, d->V, d->C, Cp), nullptr, sc, gp, k.st));
      if (gx && !k.rc) {
        float* to = planes() ? gx + i * S * d->C + s : gx + p * d->C;
        k.did(mix::tc_input_grad32(gp, parts_of(wt3, d->C, d->V, Vp), to, planes() ? 0 : d->C, d->S, k.st));
      }
      if ((gw || gb) && !k.rc) {
        mix::tc_outer_floats(n, d->V, 1, d->C, &splits, &ldn, 3);
        k.did(mix::tc_outer(gp, mix::TcRows{}, xp, part, csum, k.st));
        if (k.rc) return;
        // (many shares of few sums: several threads for each)
        if (splits >= 64 && p == 0 && n == P) mix::add_shares<float, float>(part, d->V, d->C, ldn, gw, csum, gb, splits, k.st);
        else add_piece_kernel<float><<<(unsigned)((threads + THREADS - 1) / THREADS), THREADS, 0, k.st>>>(
            part, csum, splits, d->V, d->V, d->C, ldn, acc, p == 0, p + n == P, gw, gb), MC_COUNT(1);
        k.did(cudaGetLastError() == cudaSuccess ? MC_OK : MC_ERR_LAUNCH);
      }
    });
    return k.rc;
  }
};
template <typename F>
static size_t work_size(F f) {
  mix::Work k{};
  k.sizes = true;
  f(k);
  return k.used;
}

// f of the layer's arithmetic type: float32 or float64
template <typename F>
static auto by_type(int dtype, F f) {
  if (dtype == MC_F64) return f(double());
  return f(float());
}

}  // namespace classify
}  // namespace mc
using namespace mc;

extern "C" {

size_t mc_cross_entropy_saved_bytes(const mc_ce_desc* d) {
  if (classify::check_desc(d)) return 0;
  if (d->dtype == MC_BF16) return classify::TensorCores(d).saved_bytes();
  const long long pixels = d->B * d->S;
  return d->dtype == MC_F64 ? classify::kept_bytes<double>(pixels) : classify::kept_bytes<float>(pixels);
}
size_t mc_cross_entropy_workspace_bytes(const mc_ce_desc* d, int32_t phase) {
  if (classify::check_desc(d)) return 0;
  if (d->dtype == MC_BF16)
    return classify::work_size([&](mix::Work& k) {
      const classify::TensorCores t(d);
      if (phase == MC_PHASE_BACKWARD) t.backward(k, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
      else t.forward(k, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
    });
  if (classify::FloatCores::takes(d))
    return classify::work_size([&](mix::Work& k) {
      const classify::FloatCores t(d);
      if (phase == MC_PHASE_BACKWARD) t.backward(k, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
      else t.forward(k, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
    });
  return classify::by_type(d->dtype, [&](auto t) {
    return classify::General<decltype(t)>(d, nullptr, phase == MC_PHASE_BACKWARD, nullptr).m.used;
  });
}
int mc_cross_entropy_fwd(const mc_ce_desc* d, const void* x, const void* w, const void* bias, const int64_t* target, void* loss,
                         void* saved, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = classify::check_desc(d)) return rc;
  if (!x || !w || !target || !loss || !saved) return MC_ERR_BAD_ARG;
  const size_t e = classify::esize(d->dtype);
  if (!classify::on(x, 16) || !classify::on(w, 16) || !classify::on(bias, e) || !classify::on(target, 8) ||
      !classify::on(loss, classify::csize(d->dtype)) || !classify::on(saved, 16) || !classify::on(ws, 16))
    return MC_ERR_BAD_ARG;
  if (!ws || ws_bytes < mc_cross_entropy_workspace_bytes(d, MC_PHASE_FORWARD)) return MC_ERR_WORKSPACE;
  if (d->dtype == MC_BF16) {
    mix::Work k{(char*)ws, (cudaStream_t)stream};
    return classify::TensorCores(d).forward(k, (const bf16*)x, (const bf16*)w, (const bf16*)bias, target, (float*)loss, (char*)saved);
  }
  if (classify::FloatCores::takes(d)) {
    mix::Work k{(char*)ws, (cudaStream_t)stream};
    return classify::FloatCores(d).forward(k, (const float*)x, (const float*)w, (const float*)bias, target, (float*)loss, (char*)saved);
  }
  return classify::by_type(d->dtype, [&](auto t) {
    typedef decltype(t) T;
    return classify::General<T>(d, ws, false, (cudaStream_t)stream)
        .forward((const T*)x, (const T*)w, (const T*)bias, target, (T*)loss, saved);
  });
}
int mc_cross_entropy_bwd(const mc_ce_desc* d, const void* grad_loss, const void* x, const void* w, const void* bias,
                         const int64_t* target, const void* saved, void* gx, void* gw, void* gb, void* ws, size_t ws_bytes,
                         void* stream) {
  if (const int rc = classify::check_desc(d)) return rc;
  if (!grad_loss || !x || !w || !target || !saved) return MC_ERR_BAD_ARG;
  const size_t e = classify::esize(d->dtype);
  if (!classify::on(x, 16) || !classify::on(w, 16) || !classify::on(bias, e) || !classify::on(target, 8) ||
      !classify::on(grad_loss, classify::csize(d->dtype)) || !classify::on(saved, 16) || !classify::on(gx, 16) ||
      !classify::on(gw, e) || !classify::on(gb, e) || !classify::on(ws, 16))
    return MC_ERR_BAD_ARG;
  if (!ws || ws_bytes < mc_cross_entropy_workspace_bytes(d, MC_PHASE_BACKWARD)) return MC_ERR_WORKSPACE;
  if (d->dtype == MC_BF16) {
    mix::Work k{(char*)ws, (cudaStream_t)stream};
    return classify::TensorCores(d).backward(k, (const float*)grad_loss, (const bf16*)x, (const bf16*)w, (const bf16*)bias, target,
                                             (const char*)saved, (bf16*)gx, (bf16*)gw, (bf16*)gb);
  }
  if (classify::FloatCores::takes(d)) {
    mix::Work k{(char*)ws, (cudaStream_t)stream};
    return classify::FloatCores(d).backward(k, (const float*)grad_loss, (const float*)x, (const float*)w, (const float*)bias, target,
                                            (const char*)saved, (float*)gx, (float*)gw, (float*)gb);
  }
  return classify::by_type(d->dtype, [&](auto t) {
    typedef decltype(t) T;
    return classify::General<T>(d, ws, true, (cudaStream_t)stream)
        .backward((const T*)grad_loss, (const T*)x, (const T*)w, (const T*)bias, target, saved, (T*)gx, (T*)gw, (T*)gb);
  });
}

}  // extern "C"
