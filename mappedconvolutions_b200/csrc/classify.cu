// Softmax cross entropy of a pointwise classifier: entry points, and the way of float32, float64 and wide bf16 layers.
//
// Class scores are never kept: a call takes the pixels in pieces whose scores fit the workspace (PIECE bytes, which stay in L2),
// multiplies with the kernels of the channel-mixing layers and reduces the piece's rows; the backward call computes the scores again.
// Bound: the products (FMA issue).
#include <initializer_list>

#include "classify.cuh"

namespace mc {
namespace classify {
using mix::RowsArgs;
using mix::View;

constexpr size_t PIECE = 48u << 20;
constexpr int THREADS = 256;

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
__device__ __forceinline__ float log_of(float v) { return logf(v); }
__device__ __forceinline__ double log_of(double v) { return log(v); }

template <typename CT>
__device__ __forceinline__ CT warp_sum(CT v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// lse and loss of the rows of a piece, one warp to a row
template <typename CT>
__global__ void __launch_bounds__(THREADS) lse_kernel(const CT* __restrict__ z, const int64_t* __restrict__ target, long long n,
                                                      int V, long long ignore, CT* __restrict__ lse, CT* __restrict__ value) {
  const long long row = blockIdx.x * (long long)(THREADS / 32) + threadIdx.x / 32;
  if (row >= n) return;
  const int lane = threadIdx.x % 32;
  const long long t = target[row];
  CT out, loss;
  if (t == ignore) {
    out = CT(INFINITY), loss = CT(0);
  } else if (t < 0 || t >= V) {
    out = loss = CT(NAN);
  } else {
    const CT* r = z + row * V;
    CT top = -CT(INFINITY), sum = CT(0);
    for (int v = lane; v < V; v += 32) top = fmax(top, r[v]);  // (a NaN shows in the sum)
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmax(top, __shfl_xor_sync(~0u, top, o));
    for (int v = lane; v < V; v += 32) sum += exp_of(r[v] - top);
    out = top + log_of(warp_sum(sum));
    loss = out - r[t];
  }
  if (lane == 0) lse[row] = out, value[row] = loss;
}

// z <- gz
template <typename CT>
__global__ void __launch_bounds__(THREADS) score_grad_kernel(CT* __restrict__ z, const int64_t* __restrict__ target,
                                                             const CT* __restrict__ lse, long long n, int V,
                                                             const double* count, const CT* grad, bool mean) {
  const CT scale = mean ? (CT)((double)*grad / *count) : *grad;
  for (long long row = blockIdx.x * (long long)(THREADS / 32) + threadIdx.x / 32; row < n; row += gridDim.x * (long long)(THREADS / 32)) {
    const CT l = lse[row];
    const long long t = target[row];
    CT* r = z + row * V;
    for (int v = threadIdx.x % 32; v < V; v += 32)
      r[v] = l == CT(INFINITY) ? CT(0) : scale * (exp_of(r[v] - l) - (v == t ? CT(1) : CT(0)));
  }
}

// (pixels, C) wherever they lie -> rows of CT; those of pixels without a label are zero if lse is given
template <typename T, typename CT>
__global__ void __launch_bounds__(THREADS) rows_kernel(const T* __restrict__ src, long long pix, long long ch, long long n, int C,
                                                       const CT* __restrict__ lse, CT* __restrict__ dst) {
  __shared__ CT tile[32][33];
  // 32 pixels x 32 channels, read along whichever direction is contiguous
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  const long long p0 = blockIdx.x * 32ll;
  for (int c0 = blockIdx.y * 32; c0 < C; c0 += gridDim.y * 32) {
    __syncthreads();
    for (int k = ty; k < 32; k += THREADS / 32) {
      const long long p = p0 + (ch == 1 ? k : tx);
      const int c = c0 + (ch == 1 ? tx : k);
      CT v = CT(0);
      if (p < n && c < C && !(lse && lse[p] == CT(INFINITY))) v = (CT)ldv(src + p * pix + (long long)c * ch);
      tile[ch == 1 ? k : tx][ch == 1 ? tx : k] = v;
    }
    __syncthreads();
    for (int k = ty; k < 32; k += THREADS / 32)
      if (p0 + k < n && c0 + tx < C) dst[(p0 + k) * C + c0 + tx] = tile[k][tx];
  }
}
// and back
template <typename T, typename CT>
__global__ void __launch_bounds__(THREADS) unrows_kernel(const CT* __restrict__ src, T* __restrict__ dst, long long pix,
                                                         long long ch, long long n, int C) {
  __shared__ CT tile[32][33];
  const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
  const long long p0 = blockIdx.x * 32ll;
  for (int c0 = blockIdx.y * 32; c0 < C; c0 += gridDim.y * 32) {
    __syncthreads();
    for (int k = ty; k < 32; k += THREADS / 32)
      if (p0 + k < n && c0 + tx < C) tile[k][tx] = src[(p0 + k) * C + c0 + tx];
    __syncthreads();
    for (int k = ty; k < 32; k += THREADS / 32) {
      const int r = ch == 1 ? k : tx, q = ch == 1 ? tx : k;
      if (p0 + r < n && c0 + q < C) stv(dst + (p0 + r) * pix + (long long)(c0 + q) * ch, tile[r][q]);
    }
  }
}
template <typename T, typename CT>
__global__ void __launch_bounds__(THREADS) convert_kernel(const T* __restrict__ src, CT* __restrict__ dst, long long n) {
  for (long long i = blockIdx.x * (long long)THREADS + threadIdx.x; i < n; i += gridDim.x * (long long)THREADS) stv(dst + i, (CT)ldv(src + i));
}
// acc (+)= the shares of one piece, in order; the last piece's call rounds to `out`
template <typename T, typename CT>
__global__ void __launch_bounds__(THREADS) gather_kernel(const CT* __restrict__ part, long long n, int splits, CT* __restrict__ acc,
                                                         bool first, T* __restrict__ out) {
  for (long long i = blockIdx.x * (long long)THREADS + threadIdx.x; i < n; i += gridDim.x * (long long)THREADS) {
    CT s = first ? CT(0) : acc[i];
    for (int j = 0; j < splits; ++j) s += part[j * n + i];
    if (out) stv(out + i, s);
    else acc[i] = s;
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
template <typename CT>
int sum_loss(const CT* value, const int64_t* target, long long P, long long ignore, bool mean, double* part, double* count,
             CT* loss, cudaStream_t st) {
  const int blocks = grid_for(P, 4 * THREADS, SUM_BLOCKS);
  loss_part_kernel<CT><<<blocks, THREADS, 0, st>>>(value, target, P, ignore, part), MC_COUNT(1);
  loss_kernel<CT><<<1, THREADS, 0, st>>>(part, blocks, mean, count, loss), MC_COUNT(1);
  MC_CHECK_LAUNCH();
  return MC_OK;
}

// ---- host -----------------------------------------------------------------------------------------------
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
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
    const size_t row = (size_t)(d->V > d->C ? d->V : d->C) * csize(d->dtype);
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

template <typename T>
struct General {
  typedef typename Traits<T>::CT CT;
  static constexpr bool CONVERT = sizeof(T) != sizeof(CT);
  const mc_ce_desc* d;
  Pieces pieces;
  Memory m;
  cudaStream_t st;
  CT *z, *rows, *value, *w, *b, *gx, *part, *csum, *acc;
  double* sums;

  General(const mc_ce_desc* desc, void* ws, bool backward, cudaStream_t s) : d(desc), pieces(desc), m(ws), st(s) {
    const size_t n = pieces.most(), C = d->C, V = d->V, P = d->B * d->S;
    z = (CT*)m.take(n * V * sizeof(CT));
    rows = (CT*)(CONVERT || backward ? m.take(n * C * sizeof(CT)) : nullptr);
    w = (CT*)(CONVERT ? m.take(V * C * sizeof(CT)) : nullptr);
    b = (CT*)(CONVERT ? m.take(V * sizeof(CT)) : nullptr);
    if (!backward) {
      value = (CT*)m.take(P * sizeof(CT));
      sums = (double*)m.take(SUM_BLOCKS * 16);
    } else {
      gx = (CT*)(CONVERT ? m.take(n * C * sizeof(CT)) : nullptr);
      int splits = 1;
      each([&](long long, long long, long long k) { if (Shares(k, d->V, d->C).splits > splits) splits = Shares(k, d->V, d->C).splits; });
      part = (CT*)m.take((size_t)splits * V * C * sizeof(CT));
      csum = (CT*)m.take((size_t)splits * V * sizeof(CT));
      acc = (CT*)m.take((V * C + V) * sizeof(CT));
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
  View flat(const CT* p, long long n, int C) const { return View{p, n * C, C, 1}; }
  dim3 tiles(long long n) const { return dim3((unsigned)((n + 31) / 32), (unsigned)((d->C + 31) / 32 < 64 ? (d->C + 31) / 32 : 64)); }
  // pixels of a piece as rows of CT (several images one after the other)
  void gather(const T* x, long long i, long long s, long long n, const CT* lse) {
    const long long per = n < pieces.S ? n : pieces.S;
    for (long long k = 0; k * per < n; ++k) {
      const View v = view(x, i + k, s);
      rows_kernel<T, CT><<<tiles(per), THREADS, 0, st>>>((const T*)v.ptr, v.pix, v.ch, per, d->C, lse ? lse + k * per : nullptr,
                                                         rows + k * per * d->C), MC_COUNT(1);
    }
  }
  const CT* weights(const T* p, CT* to, long long n) {
    if (!CONVERT || !p) return (const CT*)(const void*)p;
    convert_kernel<T, CT><<<grid_for(n, THREADS, 1184), THREADS, 0, st>>>(p, to, n), MC_COUNT(1);
    return to;
  }
  // z = x W^T + b of a piece
  int scores(const View& x, long long n, long long S, const CT* wc, const CT* bc) {
    RowsArgs r{};
    r.a = x, r.w = wc, r.wn = d->C, r.wk = 1, r.bias = bc, r.y = View{z, S * (long long)d->V, d->V, 1}, r.P = n, r.S = (int)S, r.N = d->V, r.K = d->C;
    return mix::simt_rows_launch(d->dtype, mix::EPI_LAYER, r, st);
  }

  int forward(const T* x, const T* wt, const T* bt, const int64_t* target, CT* loss, void* kept) {
    CT* lse = (CT*)((char*)kept + KEPT_HEAD);
    const CT *wc = weights(wt, w, (long long)d->V * d->C), *bc = weights(bt, b, d->V);
    int rc = MC_OK;
    each([&](long long i, long long s, long long n) {
      if (rc) return;
      const long long p = i * pieces.S + s, S = n < pieces.S ? n : pieces.S;
      if (CONVERT) gather(x, i, s, n, nullptr), rc = scores(flat(rows, n, d->C), n, n, wc, bc);
      else rc = scores(view(x, i, s), n, S, wc, bc);
      if (rc) return;
      lse_kernel<CT><<<(unsigned)((n + 7) / 8), THREADS, 0, st>>>(z, target + p, n, d->V, d->ignore_index, lse + p, value + p);
      MC_COUNT(1);
    });
    if (rc) return rc;
    return sum_loss<CT>(value, target, d->B * d->S, d->ignore_index, d->reduction == MC_REDUCE_MEAN, sums, (double*)kept, loss, st);
  }

  int backward(const CT* grad, const T* x, const T* wt, const T* bt, const int64_t* target, const void* kept, T* gxt, T* gw, T* gb) {
    const CT* lse = (const CT*)((const char*)kept + KEPT_HEAD);
    const CT *wc = weights(wt, w, (long long)d->V * d->C), *bc = weights(bt, b, d->V);
    const long long P = d->B * d->S, VC = (long long)d->V * d->C;
    int rc = MC_OK;
    each([&](long long i, long long s, long long n) {
      if (rc) return;
      const long long p = i * pieces.S + s, S = n < pieces.S ? n : pieces.S;
      gather(x, i, s, n, lse + p);
      if ((rc = scores(flat(rows, n, d->C), n, n, wc, bc))) return;
      score_grad_kernel<CT><<<grid_for(n, 8, 148 * 8), THREADS, 0, st>>>(z, target + p, lse + p, n, d->V, (const double*)kept, grad,
                                                                        d->reduction == MC_REDUCE_MEAN), MC_COUNT(1);
      if (gxt) {
        RowsArgs r{};
        r.a = flat(z, n, d->V), r.w = wc, r.wn = 1, r.wk = d->C, r.P = n, r.N = d->C, r.K = d->V, r.S = (int)S;
        r.a.img = S * (long long)d->V;
        r.y = CONVERT ? View{gx, S * (long long)d->C, d->C, 1} : view(gxt, i, s);
        if ((rc = mix::simt_rows_launch(d->dtype, mix::EPI_LAYER, r, st))) return;
        for (long long k = 0; CONVERT && k * S < n; ++k) {
          const View v = view(gxt, i + k, s);
          unrows_kernel<T, CT><<<tiles(S), THREADS, 0, st>>>(gx + k * S * d->C, (T*)v.ptr, v.pix, v.ch, S, d->C), MC_COUNT(1);
        }
      }
      if (gw || gb) {
        const Shares sh(n, d->V, d->C);
        const mix::OuterArgs o{flat(z, n, d->V), flat(rows, n, d->C), part, csum, n, sh.share, d->V, d->C, 1, 1, sh.splits, sh.splits};
        if ((rc = mix::simt_outer_launch(d->dtype, o, st))) return;
        const bool first = p == 0, last = p + n == P;
        if (gw) gather_kernel<T, CT><<<grid_for(VC, THREADS, 1184), THREADS, 0, st>>>(part, VC, sh.splits, acc, first, last ? gw : nullptr), MC_COUNT(1);
        if (gb) gather_kernel<T, CT><<<grid_for(d->V, THREADS, 1184), THREADS, 0, st>>>(csum, d->V, sh.splits, acc + VC, first, last ? gb : nullptr), MC_COUNT(1);
      }
    });
    if (rc) return rc;
    MC_CHECK_LAUNCH();
    return MC_OK;
  }
};

template <typename F>
static auto by_type(int dtype, F f) {
  if (dtype == MC_F64) return f(double());
  if (dtype == MC_F32) return f(float());
  return f(bf16());
}

}  // namespace classify
}  // namespace mc
using namespace mc;

extern "C" {

size_t mc_cross_entropy_saved_bytes(const mc_ce_desc* d) {
  if (classify::check_desc(d)) return 0;
  return classify::KEPT_HEAD + classify::up256((size_t)d->B * d->S * classify::csize(d->dtype));
}
size_t mc_cross_entropy_workspace_bytes(const mc_ce_desc* d, int32_t phase) {
  if (classify::check_desc(d)) return 0;
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
  return classify::by_type(d->dtype, [&](auto t) {
    typedef decltype(t) T;
    typedef typename Traits<T>::CT CT;
    return classify::General<T>(d, ws, false, (cudaStream_t)stream)
        .forward((const T*)x, (const T*)w, (const T*)bias, target, (CT*)loss, saved);
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
  return classify::by_type(d->dtype, [&](auto t) {
    typedef decltype(t) T;
    typedef typename Traits<T>::CT CT;
    return classify::General<T>(d, ws, true, (cudaStream_t)stream)
        .backward((const CT*)grad_loss, (const T*)x, (const T*)w, (const T*)bias, target, saved, (T*)gx, (T*)gw, (T*)gb);
  });
}

}  // extern "C"
