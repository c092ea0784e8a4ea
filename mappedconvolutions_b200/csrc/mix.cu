// C-ABI entry points of the channel-mixing layers: argument checks, workspace layout, and the sequence of products
// behind each call.
#include <initializer_list>
#include <type_traits>

#include "mix.cuh"

namespace mc {
namespace mix {

static int esize(int dtype) { return dtype == MC_F64 ? 8 : dtype == MC_F32 ? 4 : 2; }
static int acc_size(int dtype) { return dtype == MC_F64 ? 8 : 4; }
static bool aligned(size_t n, std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p % n) return false;
  return true;
}
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

static int check_desc(const mc_mix_desc* d, bool gated) {
  if (!d || d->B <= 0 || d->S <= 0 || d->C_in <= 0 || d->C_out <= 0) return MC_ERR_BAD_ARG;
  if (gated ? d->hidden <= 0 : d->hidden != 0) return MC_ERR_BAD_ARG;
  if (d->dtype != MC_F32 && d->dtype != MC_F64 && d->dtype != MC_BF16) return MC_ERR_BAD_ARG;
  if (d->layout != MC_NCHW && d->layout != MC_NHWC) return MC_ERR_BAD_ARG;
  if (d->act < MC_ACT_NONE || d->act > MC_ACT_SIGMOID) return MC_ERR_BAD_ARG;
  // pixel indices are 32-bit (element offsets are not); channel tiles are a grid's second dimension
  if (d->S >= (1ll << 31) || d->B >= (1ll << 31) || d->B * d->S > (1ll << 31) - 256) return MC_ERR_TOO_LARGE;
  if (d->C_in > (1 << 20) || d->C_out > (1 << 20) || d->hidden > (1 << 19)) return MC_ERR_TOO_LARGE;
  return MC_OK;
}

// Activations and weights on 16 bytes for MC_BF16 (TMA), everything else on its elements, memory of calls on 16 bytes.
static bool placed(const mc_mix_desc* d, std::initializer_list<const void*> tensors, std::initializer_list<const void*> vectors,
                   std::initializer_list<const void*> memory) {
  return aligned(d->dtype == MC_BF16 ? 16 : esize(d->dtype), tensors) && aligned(esize(d->dtype), vectors) && aligned(16, memory);
}

static long long pixels(const mc_mix_desc* d) { return d->B * d->S; }

// Shares of the pixels that a parameter gradient is summed in: about a wave of blocks (two to an SM), at least 256 pixels
// each where images are that large; parts of an image or groups of images (channels-last batches are one image).
struct Shares {
  long long S, share;
  int B, group, per_image, splits;
  size_t part, csum;  // bytes
};
static Shares shares_of(const mc_mix_desc* d, int M, int N) {
  Shares s;
  const bool whole = d->layout == MC_NHWC || d->S == 1 || d->B == 1;
  s.B = whole ? 1 : (int)d->B;
  s.S = whole ? d->B * d->S : d->S;
  const long long tiles = (long long)((M + 127) / 128) * ((N + 127) / 128);
  long long want = (2 * 148 + tiles - 1) / tiles, most = (s.B * s.S + 255) / 256;
  if (want > most) want = most;
  s.group = (int)((s.B + want - 1) / want);
  const long long n = s.group > 1 ? 1 : (want + s.B - 1) / s.B;
  s.share = ((s.S + n - 1) / n + 15) / 16 * 16;
  s.per_image = (int)((s.S + s.share - 1) / s.share);
  s.splits = (s.B + s.group - 1) / s.group * s.per_image;
  s.part = up256((size_t)s.splits * M * N * acc_size(d->dtype));
  s.csum = up256((size_t)s.splits * M * acc_size(d->dtype));
  return s;
}

// gw (M, N) and gb (M), either of which may be null: the shares' sums, rounded once.  Rows of part have ldn elements.
// A block takes 32 sums; G threads for each add every G-th share, and their results are added in order.
template <typename T, typename CT, int G>
__global__ void __launch_bounds__(32 * G) add_shares_kernel(const CT* __restrict__ part, int M, int N, int ldn,
                                                            T* __restrict__ gw, const CT* __restrict__ csum,
                                                            T* __restrict__ gb, int splits) {
  __shared__ CT sums[G][32];
  const long long nw = (long long)M * N, i = blockIdx.x * 32ll + threadIdx.x % 32;
  const bool w = i < nw, in = i < nw + M && (w ? (void*)gw : (void*)gb);
  const int j0 = threadIdx.x / 32;
  CT s = CT(0);
  if (in) {
    const CT* src = w ? part + i / N * ldn + i % N : csum + (i - nw);
    const long long step = w ? (long long)M * ldn : M;
#pragma unroll 8
    for (int j = j0; j < splits; j += G) s += src[j * step];
  }
  sums[j0][threadIdx.x % 32] = s;
  __syncthreads();
  if (j0 || !in) return;
#pragma unroll
  for (int j = 1; j < G; ++j) s += sums[j][threadIdx.x];
  stv(w ? gw + i : gb + (i - nw), s);
}
// Many shares of few sums: 32 threads for each (296 shares of 99 x 50 sums: 6 us instead of 10), as long as the blocks run
// at one time (74 shares of 256 x 128 sums: 10 us instead of 6).
template <typename T, typename CT>
static void add_shares(const CT* part, int M, int N, int ldn, T* gw, const CT* csum, T* gb, int splits, cudaStream_t st) {
  const unsigned blocks = (unsigned)(((long long)M * N + M + 31) / 32);
  if (splits >= 64 && blocks <= 2 * 148) add_shares_kernel<T, CT, 32><<<blocks, 1024, 0, st>>>(part, M, N, ldn, gw, csum, gb, splits);
  else add_shares_kernel<T, CT, 8><<<blocks, 256, 0, st>>>(part, M, N, ldn, gw, csum, gb, splits);
  MC_COUNT(1);
}

// gz = gy act'(z), sixteen bytes at a time (vec: gy starts on a multiple of them, as the others do)
template <typename T>
__global__ void __launch_bounds__(256) act_bwd_kernel(const T* __restrict__ gy, const T* __restrict__ z,
                                                      T* __restrict__ gz, long long n, int act, bool vec) {
  constexpr int V = 16 / sizeof(T);
  for (long long i = (blockIdx.x * 256ll + threadIdx.x) * V; i < n; i += gridDim.x * 256ll * V) {
    __align__(16) T g[V], v[V];
    if (vec && i + V <= n) {
      *reinterpret_cast<uint4*>(g) = __ldcs(reinterpret_cast<const uint4*>(gy + i));
      *reinterpret_cast<uint4*>(v) = __ldcs(reinterpret_cast<const uint4*>(z + i));
#pragma unroll
      for (int e = 0; e < V; ++e) g[e] *= act_slope<T>(act, v[e]);
      *reinterpret_cast<uint4*>(gz + i) = *reinterpret_cast<const uint4*>(g);
    } else {
      for (int e = 0; e < V && i + e < n; ++e) gz[i + e] = gy[i + e] * act_slope<T>(act, z[i + e]);
    }
  }
}

template <typename F>
static int by_type(int dtype, F f) {
  if (dtype == MC_F64) f(double());
  else f(float());
  MC_CHECK_LAUNCH();
  return MC_OK;
}

static int param_grads(int dtype, View g, int M, View x, int N, const Shares& s, char* part, char* csum, void* gw,
                       void* gb, cudaStream_t st) {
  const OuterArgs o{g, x, part, csum, s.S, s.share, M, N, s.B, s.group, s.per_image, s.splits};
  const int rc = simt_outer_launch(dtype, o, st);
  if (rc) return rc;
  return by_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    typedef typename Traits<T>::CT CT;
    add_shares<T, CT>((const CT*)part, M, N, N, (T*)gw, (const CT*)csum, (T*)gb, s.splits, st);
  });
}

// ---- bf16: the tensor-core kernels, on rows of channels --------------------------------------------------------------
// Rows whose length is a multiple of 8 channels (16 bytes) are read and written where they lie; anything else - other
// channel counts, NCHW - is copied to padded rows in the workspace and back.
static int pad8(int c) { return (c + 7) / 8 * 8; }

// (R, C) without gaps <-> rows of ld elements (zeros behind the last one).  A block takes `chunk` rows (a multiple of 8, so
// that both sides start on 16 bytes) through shared memory, as they lie without gaps, and moves 16 bytes per access in
// global memory on both sides.  410 channels of 327 684 pixels from rows: 277 us with one element per thread.
constexpr int PACK_BYTES = 16 * 1024;
__global__ void __launch_bounds__(256) pack_rows_kernel(const bf16* __restrict__ src, bf16* __restrict__ dst, long long R,
                                                        int C, int ld, int chunk) {
  extern __shared__ __align__(16) bf16 flat[];
  const long long r0 = blockIdx.x * (long long)chunk;
  const int rows = R - r0 < chunk ? (int)(R - r0) : chunk, n = rows * C;
  const bf16* from = src + r0 * C;
  for (int i = threadIdx.x * 8; i < n; i += 256 * 8) {
    if (i + 8 <= n) *reinterpret_cast<uint4*>(flat + i) = __ldcs(reinterpret_cast<const uint4*>(from + i));
    else for (int j = i; j < n; ++j) flat[j] = from[j];
  }
  __syncthreads();
  const int per = ld / 8;
  for (int i = threadIdx.x; i < rows * per; i += 256) {
    const int r = i / per, c = (i - r * per) * 8;
    __align__(16) bf16 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < C ? flat[r * C + c + j] : bf16(0.f);
    *reinterpret_cast<uint4*>(dst + (r0 + r) * ld + c) = *reinterpret_cast<const uint4*>(v);
  }
}
__global__ void __launch_bounds__(256) unpack_rows_kernel(const bf16* __restrict__ src, bf16* __restrict__ dst, long long R,
                                                          int C, int ld, int chunk) {
  extern __shared__ __align__(16) bf16 flat[];
  const long long r0 = blockIdx.x * (long long)chunk;
  const int rows = R - r0 < chunk ? (int)(R - r0) : chunk, n = rows * C, per = ld / 8;
  for (int i = threadIdx.x; i < rows * per; i += 256) {
    const int r = i / per, c = (i - r * per) * 8;
    const uint4 q = __ldcs(reinterpret_cast<const uint4*>(src + (r0 + r) * ld + c));
    __align__(16) bf16 v[8];
    *reinterpret_cast<uint4*>(v) = q;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < C) flat[r * C + c + j] = v[j];
  }
  __syncthreads();
  bf16* to = dst + r0 * C;
  for (int i = threadIdx.x * 8; i < n; i += 256 * 8) {
    if (i + 8 <= n) *reinterpret_cast<uint4*>(to + i) = *reinterpret_cast<const uint4*>(flat + i);
    else for (int j = i; j < n; ++j) to[j] = flat[j];
  }
}
// Rows longer than a block's shared memory (of eight of them): element by element, rows as the grid's second dimension.
__global__ void __launch_bounds__(256) long_rows_kernel(const bf16* __restrict__ src, bf16* __restrict__ dst, long long R,
                                                        int from, int to) {
  const int n = from < to ? from : to;
  for (long long r = blockIdx.y; r < R; r += gridDim.y)
    for (int c = blockIdx.x * 256 + threadIdx.x; c < to; c += gridDim.x * 256)
      dst[r * to + c] = c < n ? src[r * from + c] : bf16(0.f);
}
// rows of `from` elements -> rows of `to`, one of which is the other's padded length
static int copy_rows(const void* src, void* dst, long long R, int from, int to, cudaStream_t st) {
  const int C = from < to ? from : to, ld = from < to ? to : from;
  int chunk = PACK_BYTES / 2 / ld / 8 * 8;
  if (chunk > 512) chunk = 512;
  const long long blocks = chunk ? (R + chunk - 1) / chunk : 0;
  if (chunk == 0 || blocks >= (1ll << 31)) {
    const dim3 grid((unsigned)((to + 255) / 256 < 64 ? (to + 255) / 256 : 64), (unsigned)(R < 65535 ? R : 65535));
    long_rows_kernel<<<grid, 256, 0, st>>>((const bf16*)src, (bf16*)dst, R, from, to), MC_COUNT(1);
  } else if (from < to) {
    pack_rows_kernel<<<(unsigned)blocks, 256, PACK_BYTES, st>>>((const bf16*)src, (bf16*)dst, R, C, ld, chunk), MC_COUNT(1);
  } else {
    unpack_rows_kernel<<<(unsigned)blocks, 256, PACK_BYTES, st>>>((const bf16*)src, (bf16*)dst, R, C, ld, chunk), MC_COUNT(1);
  }
  MC_CHECK_LAUNCH();
  return MC_OK;
}
// (B, C, S) -> rows of ld channels (zeros behind the last one): CT channels x 4096 / CT pixels at a time through shared
// memory.  The planes are read value by value, neighbouring threads at neighbouring pixels, because with an
// odd number of pixels they start anywhere; sixteen values per thread are on their way at once.  64 channels of
// 8 x 125 x 251 pixels to rows: 35 us with the general transpose.
template <int CT>
__global__ void __launch_bounds__(256) planes_to_rows_kernel(const bf16* __restrict__ src, bf16* __restrict__ dst,
                                                             long long S, int C, int ld, int tiles_s, int tiles_c) {
  constexpr int PX = 4096 / CT, PITCH = CT + 2;
  __shared__ __align__(16) bf16 tile[PX * PITCH];
  const int tc = blockIdx.x % tiles_c, ts = blockIdx.x / tiles_c % tiles_s, c0 = tc * CT;
  const long long b = blockIdx.x / tiles_c / tiles_s, s0 = (long long)ts * PX;
  const int s = threadIdx.x % PX, c = threadIdx.x / PX;
  const bf16* from = src + (b * C + c0 + c) * S + s0 + s;
  bf16 v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    v[i] = s0 + s < S && c0 + c + i * (256 / PX) < C ? __ldcs(from + (long long)i * (256 / PX) * S) : bf16(0.f);
#pragma unroll
  for (int i = 0; i < 16; ++i) tile[s * PITCH + c + i * (256 / PX)] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = threadIdx.x; i < 512; i += 256) {
    const int r = i / (CT / 8), j = i % (CT / 8) * 8;
    if (s0 + r >= S || c0 + j >= ld) continue;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(tile + r * PITCH + j);
    *reinterpret_cast<uint4*>(dst + (b * S + s0 + r) * ld + c0 + j) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
// Lays a call's temporary tensors out in the workspace; with `sizes` set it only adds up what they need.
struct Work {
  char* base;
  cudaStream_t st;
  bool sizes = false;
  size_t used = 0;
  int rc = MC_OK;
  bool run() const { return !sizes && rc == MC_OK; }
  char* take(size_t n) {
    char* p = sizes ? nullptr : base + used;
    used += up256(n);
    return p;
  }
  void did(int r) { if (rc == MC_OK) rc = r; }
  static bool in_place(const mc_mix_desc* d, int C) { return C % 8 == 0 && (d->layout == MC_NHWC || d->S == 1); }
  TcRows fresh(long long rows, int C) { return TcRows{take((size_t)rows * pad8(C) * 2), rows, C, pad8(C)}; }
  // an activation as rows
  TcRows in(const mc_mix_desc* d, const void* p, int C) {
    const long long P = pixels(d);
    if (in_place(d, C)) return TcRows{p, P, C, C};
    const TcRows r = fresh(P, C);
    if (!p && !sizes) return TcRows{nullptr, P, C, C};
    lay_out(d, p, r);
    return r;
  }
  void lay_out(const mc_mix_desc* d, const void* p, const TcRows& r) {
    if (!run()) return;
    const int C = r.cols;
    if (d->layout == MC_NHWC || d->S == 1 || C == 1) {
      did(copy_rows(p, (void*)r.p, r.rows, C, r.ld, st));
    } else {
      planes(d, C, [&](auto ct, unsigned blocks, int ts, int tc) {
        planes_to_rows_kernel<decltype(ct)::value><<<blocks, 256, 0, st>>>((const bf16*)p, (bf16*)r.p, d->S, C, r.ld, ts, tc);
      });
    }
  }
  // f(channels of a tile, blocks, tiles along S, tiles along C): 16 channels where there are no more
  template <typename F>
  void planes(const mc_mix_desc* d, int C, F f) {
    const int ct = C <= 16 ? 16 : 64, px = 4096 / ct;
    const long long ts = (d->S + px - 1) / px, tc = (C + ct - 1) / ct, blocks = d->B * ts * tc;
    if (blocks >= (1ll << 31)) return did(MC_ERR_TOO_LARGE);
    if (ct == 16) f(std::integral_constant<int, 16>(), (unsigned)blocks, (int)ts, (int)tc);
    else f(std::integral_constant<int, 64>(), (unsigned)blocks, (int)ts, (int)tc);
    MC_COUNT(1);
    did(cudaGetLastError() == cudaSuccess ? MC_OK : MC_ERR_LAUNCH);
  }
  TcRows weight(const void* p, int R, int C) {
    if (C % 8 == 0) return TcRows{p, R, C, C};
    const TcRows r = fresh(R, C);
    if (run()) did(copy_rows(p, (void*)r.p, R, C, r.ld, st));
    return r;
  }
  // n matrices (R, C) on top of each other -> their transposes (C, R); the first one is returned, the others follow
  TcRows weight_t(const void* p, int R, int C, int n = 1) {
    const TcRows r = fresh((long long)n * C, R);
    if (run()) did(mc_transpose(2, n, R, C, p, (void*)r.p, r.ld, st));
    return TcRows{r.p, C, R, r.ld};
  }
  // where a layer leaves an activation: where it belongs (rows in place, planes), or rows that put() brings there
  static bool as_planes(const mc_mix_desc* d, int C) { return d->layout == MC_NCHW && d->S > 1 && C > 1; }
  TcRows out(const mc_mix_desc* d, void* p, int C) {
    if (in_place(d, C)) return TcRows{p, pixels(d), C, C};
    return as_planes(d, C) ? TcRows{p, pixels(d), C, 0, d->S} : fresh(pixels(d), C);
  }
  void put(const mc_mix_desc* d, const TcRows& r, void* p, int C) {
    if (!run() || r.p == p) return;
    did(copy_rows(r.p, p, r.rows, r.ld, C, st));
  }
  void param_grads(const TcRows& g0, const TcRows& g1, int segs, const TcRows& x, void* gw, void* gb) {
    int splits, ldn;
    const size_t n = tc_outer_floats(x.rows, g0.cols, segs, x.cols, &splits, &ldn);
    const int M = segs * g0.cols;
    float* part = (float*)take(n * 4);
    float* csum = (float*)take((size_t)splits * M * 4);
    if (!run() || (!gw && !gb)) return;
    did(tc_outer(g0, g1, x, part, csum, st));
    if (rc) return;
    add_shares<bf16, float>(part, M, x.cols, ldn, (bf16*)gw, csum, (bf16*)gb, splits, st);
    did(cudaGetLastError() == cudaSuccess ? MC_OK : MC_ERR_LAUNCH);
  }
};

static size_t input_rows_bytes(const mc_mix_desc* d) {
  return Work::in_place(d, d->C_in) ? 0 : up256((size_t)pixels(d) * pad8(d->C_in) * 2);
}
// The input as rows: laid out at `kept` by a forward call (which may be null), found there by a backward call.
static TcRows input_rows(Work& k, const mc_mix_desc* d, const void* x, void* kept) {
  if (Work::in_place(d, d->C_in) || !kept) return k.in(d, x, d->C_in);
  const TcRows r{kept, pixels(d), d->C_in, pad8(d->C_in)};
  k.lay_out(d, x, r);
  return r;
}
static TcRows kept_rows(const mc_mix_desc* d, const void* x, const void* kept) {
  if (Work::in_place(d, d->C_in)) return TcRows{x, pixels(d), d->C_in, d->C_in};
  return TcRows{kept, pixels(d), d->C_in, pad8(d->C_in)};
}

static void tc_pointwise_fwd(Work& k, const mc_mix_desc* d, const void* x, const void* w, const void* bias,
                             const void* residual, void* y, void* saved) {
  const TcRows xr = input_rows(k, d, x, saved), wr = k.weight(w, d->C_out, d->C_in), rr = k.in(d, residual, d->C_out);
  const TcRows yr = k.out(d, y, d->C_out);
  if (k.run()) k.did(tc_layer(xr, wr, (const bf16*)bias, d->act, rr, yr, false, k.st));
  k.put(d, yr, y, d->C_out);
}

static void tc_pointwise_bwd(Work& k, const mc_mix_desc* d, const void* gy, const void* x, const void* w,
                             const void* bias, const void* saved, void* gx, void* gw, void* gb) {
  const TcRows xr = kept_rows(d, x, saved), gyr = k.in(d, gy, d->C_out);
  TcRows gz = gyr;
  if (d->act != MC_ACT_NONE) {
    const TcRows wr = k.weight(w, d->C_out, d->C_in);
    gz = k.fresh(pixels(d), d->C_out);
    if (k.run()) k.did(tc_layer(xr, wr, (const bf16*)bias, d->act, gyr, gz, true, k.st));
  }
  if (gx || k.sizes) {
    const TcRows wt = k.weight_t(w, d->C_out, d->C_in), gxr = k.out(d, gx, d->C_in);
    if (k.run()) k.did(tc_input_grad(gz, wt, TcRows{}, TcRows{}, gxr, k.st));
    k.put(d, gxr, gx, d->C_in);
  }
  k.param_grads(gz, TcRows{}, 1, xr, gw, gb);
}

static void tc_gated_fwd(Work& k, const mc_mix_desc* d, const void* x, const void* w_in, const void* b_in,
                         const void* w_out, const void* b_out, const void* residual, void* y, void* saved) {
  const int H = d->hidden;
  const size_t hb = up256((size_t)pixels(d) * pad8(H) * 2);
  const TcRows xr = input_rows(k, d, x, saved ? (char*)saved + hb : nullptr);
  const TcRows wi = k.weight(w_in, 2 * H, d->C_in), wo = k.weight(w_out, d->C_out, H);
  const TcRows h = saved ? TcRows{saved, pixels(d), H, pad8(H)} : k.fresh(pixels(d), H);
  if (k.run()) k.did(tc_gate(xr, wi, (const bf16*)b_in, d->act, h, k.st));
  const TcRows rr = k.in(d, residual, d->C_out), yr = k.out(d, y, d->C_out);
  if (k.run()) k.did(tc_layer(h, wo, (const bf16*)b_out, MC_ACT_NONE, rr, yr, false, k.st));
  k.put(d, yr, y, d->C_out);
}

static void tc_gated_bwd(Work& k, const mc_mix_desc* d, const void* gy, const void* x, const void* w_in, const void* b_in,
                         const void* w_out, const void* saved, void* gx, void* gw_in, void* gb_in, void* gw_out,
                         void* gb_out) {
  const int H = d->hidden;
  const TcRows xr = kept_rows(d, x, (const char*)saved + up256((size_t)pixels(d) * pad8(H) * 2));
  const TcRows wi = k.weight(w_in, 2 * H, d->C_in), wot = k.weight_t(w_out, d->C_out, H);
  const TcRows gyr = k.in(d, gy, d->C_out), gg = k.fresh(pixels(d), H), gu = k.fresh(pixels(d), H);
  if (k.run() && (gx || gw_in || gb_in)) k.did(tc_gate_bwd(xr, wi, (const bf16*)b_in, d->act, gyr, wot, gg, gu, k.st));
  if (gx || k.sizes) {
    const TcRows gxr = k.out(d, gx, d->C_in), wg = k.weight_t(w_in, H, d->C_in, 2);
    TcRows wu = wg;
    wu.p = (const char*)wg.p + (size_t)d->C_in * wg.ld * 2;
    if (k.run()) k.did(tc_input_grad(gg, wg, gu, wu, gxr, k.st));
    k.put(d, gxr, gx, d->C_in);
  }
  k.param_grads(gg, gu, 2, xr, gw_in, gb_in);
  k.param_grads(gyr, TcRows{}, 1, TcRows{saved, pixels(d), H, pad8(H)}, gw_out, gb_out);
}

// workspace of the whole call, for any choice of optional arguments
template <typename F>
static size_t work_size(F f) {
  Work k{nullptr, nullptr, true};
  f(k);
  return k.used;
}

}  // namespace mix
}  // namespace mc
using namespace mc;
using namespace mc::mix;

extern "C" {

int mc_mix_plan(const mc_mix_desc* d, int32_t product, int32_t sms, int32_t* plan) {
  const int rc = check_desc(d, d && d->hidden != 0);
  if (rc) return rc;
  if (!plan || sms < 0) return MC_ERR_BAD_ARG;
  if (d->dtype != MC_BF16) return MC_ERR_UNSUPPORTED;
  return tc_plan(d, product, sms, plan) ? MC_OK : MC_ERR_BAD_ARG;
}

// ---- pointwise layer ----------------------------------------------------------------------------------------

// kept for the backward pass: z in y's layout; bf16: the input as rows, where it is not rows already
size_t mc_pointwise_saved_bytes(const mc_mix_desc* d) {
  if (check_desc(d, false)) return 0;
  if (d->dtype == MC_BF16) return input_rows_bytes(d);
  if (d->act == MC_ACT_NONE) return 0;
  return up256((size_t)pixels(d) * d->C_out * esize(d->dtype));
}

size_t mc_pointwise_workspace_bytes(const mc_mix_desc* d, int32_t phase) {
  const bool backward = phase == MC_PHASE_BACKWARD;
  if (check_desc(d, false)) return 0;
  if (d->dtype == MC_BF16)
    return work_size([&](Work& k) {
      if (backward) tc_pointwise_bwd(k, d, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
      else
        tc_pointwise_fwd(k, d, nullptr, nullptr, nullptr, nullptr, nullptr,
                         phase == MC_PHASE_KEEP ? (void*)256 : nullptr);  // (not touched: only sizes are added up)
    });
  if (!backward) return 0;
  const Shares s = shares_of(d, d->C_out, d->C_in);
  return mc_pointwise_saved_bytes(d) + s.part + s.csum;
}

int mc_pointwise_fwd(const mc_mix_desc* d, const void* x, const void* w, const void* bias, const void* residual, void* y,
                     void* saved, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check_desc(d, false);
  if (rc) return rc;
  if (!x || !w || !y) return MC_ERR_BAD_ARG;
  const size_t need = mc_pointwise_workspace_bytes(d, saved ? MC_PHASE_KEEP : MC_PHASE_FORWARD);
  if (need && (!ws || ws_bytes < need)) return MC_ERR_WORKSPACE;
  if (!placed(d, {x, w, residual, y}, {bias}, {saved, ws})) return MC_ERR_BAD_ARG;
  if (d->dtype == MC_BF16) {
    Work k{(char*)ws, (cudaStream_t)stream};
    tc_pointwise_fwd(k, d, x, w, bias, residual, y, input_rows_bytes(d) ? saved : nullptr);
    return k.rc;
  }
  RowsArgs r{};
  r.a = image_view(x, d->layout, d->S, d->C_in);
  r.w = w, r.wn = d->C_in, r.wk = 1, r.bias = bias;
  r.res = image_view(residual, d->layout, d->S, d->C_out);
  r.y = image_view(y, d->layout, d->S, d->C_out);
  r.z = image_view(d->act == MC_ACT_NONE ? nullptr : saved, d->layout, d->S, d->C_out);
  r.P = pixels(d), r.S = (int)d->S, r.N = d->C_out, r.K = d->C_in, r.act = d->act;
  return simt_rows_launch(d->dtype, EPI_LAYER, r, (cudaStream_t)stream);
}

int mc_pointwise_bwd(const mc_mix_desc* d, const void* gy, const void* x, const void* w, const void* bias,
                     const void* saved, void* gx, void* gw, void* gb, void* ws, size_t ws_bytes, void* stream) {
  int rc = check_desc(d, false);
  if (rc) return rc;
  if (!gy || !x || !w || (mc_pointwise_saved_bytes(d) && !saved)) return MC_ERR_BAD_ARG;
  const size_t need = mc_pointwise_workspace_bytes(d, MC_PHASE_BACKWARD);
  if (need && (!ws || ws_bytes < need)) return MC_ERR_WORKSPACE;
  if (!placed(d, {gy, x, w, gx}, {bias, gw, gb}, {saved, ws})) return MC_ERR_BAD_ARG;
  if (d->dtype == MC_BF16) {
    Work k{(char*)ws, (cudaStream_t)stream};
    tc_pointwise_bwd(k, d, gy, x, w, bias, saved, gx, gw, gb);
    return k.rc;
  }
  cudaStream_t st = (cudaStream_t)stream;
  const long long P = pixels(d), n = P * d->C_out;
  const Shares s = shares_of(d, d->C_out, d->C_in);
  char* gz = (char*)ws;
  char* part = gz + mc_pointwise_saved_bytes(d);
  const void* g = gy;
  if (d->act != MC_ACT_NONE) {
    rc = by_type(d->dtype, [&](auto t) {
      typedef decltype(t) T;
      act_bwd_kernel<T><<<grid_for(n / (16 / (long)sizeof(T)) + 1, 256), 256, 0, st>>>(
          (const T*)gy, (const T*)saved, (T*)gz, n, d->act, aligned(16, {gy})), MC_COUNT(1);
    });
    if (rc) return rc;
    g = gz;
  }
  if (gx) {
    RowsArgs r{};
    r.a = image_view(g, d->layout, d->S, d->C_out);
    r.w = w, r.wn = 1, r.wk = d->C_in;
    r.y = image_view(gx, d->layout, d->S, d->C_in);
    r.P = P, r.S = (int)d->S, r.N = d->C_in, r.K = d->C_out, r.act = MC_ACT_NONE;
    rc = simt_rows_launch(d->dtype, EPI_LAYER, r, st);
    if (rc) return rc;
  }
  if (gw || gb)
    rc = param_grads(d->dtype, image_view(g, d->layout, d->S, d->C_out), d->C_out,
                     image_view(x, d->layout, d->S, d->C_in), d->C_in, s, part, part + s.part, gw, gb, st);
  return rc;
}

// ---- gated feed-forward block -----------------------------------------------------------------------------------

// kept for the backward pass: [g|u] (P, 2 H), then h (P, H); bf16: h in padded rows, then the input as
// rows where it is not rows already
size_t mc_gated_saved_bytes(const mc_mix_desc* d) {
  if (check_desc(d, true)) return 0;
  if (d->dtype == MC_BF16) return up256((size_t)pixels(d) * pad8(d->hidden) * 2) + input_rows_bytes(d);
  const size_t h = (size_t)pixels(d) * d->hidden * esize(d->dtype);
  return up256(2 * h) + up256(h);
}

size_t mc_gated_workspace_bytes(const mc_mix_desc* d, int32_t phase) {
  const bool backward = phase == MC_PHASE_BACKWARD;
  if (check_desc(d, true)) return 0;
  if (d->dtype == MC_BF16)
    return work_size([&](Work& k) {
      if (backward)
        tc_gated_bwd(k, d, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
      else
        tc_gated_fwd(k, d, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr,
                     phase == MC_PHASE_KEEP ? (void*)256 : nullptr);  // (not touched: only sizes are added up)
    });
  const size_t h = (size_t)pixels(d) * d->hidden * esize(d->dtype);
  if (!backward) return phase == MC_PHASE_KEEP ? 0 : up256(h);
  const Shares a = shares_of(d, 2 * d->hidden, d->C_in);
  const Shares b = shares_of(d, d->C_out, d->hidden);
  const size_t sa = a.part + a.csum, sb = b.part + b.csum;
  return up256(2 * h) + (sa > sb ? sa : sb);
}

int mc_gated_fwd(const mc_mix_desc* d, const void* x, const void* w_in, const void* b_in, const void* w_out,
                 const void* b_out, const void* residual, void* y, void* saved, void* ws, size_t ws_bytes,
                 void* stream) {
  int rc = check_desc(d, true);
  if (rc) return rc;
  if (!x || !w_in || !w_out || !y) return MC_ERR_BAD_ARG;
  const size_t need = mc_gated_workspace_bytes(d, saved ? MC_PHASE_KEEP : MC_PHASE_FORWARD);
  if (need && (!ws || ws_bytes < need)) return MC_ERR_WORKSPACE;
  if (!placed(d, {x, w_in, w_out, residual, y}, {b_in, b_out}, {saved, ws})) return MC_ERR_BAD_ARG;
  if (d->dtype == MC_BF16) {
    Work k{(char*)ws, (cudaStream_t)stream};
    tc_gated_fwd(k, d, x, w_in, b_in, w_out, b_out, residual, y, saved);
    return k.rc;
  }
  cudaStream_t st = (cudaStream_t)stream;
  const int H = d->hidden;
  const long long P = pixels(d);
  char* h = saved ? (char*)saved + up256((size_t)P * 2 * H * esize(d->dtype)) : (char*)ws;
  RowsArgs r{};
  r.a = image_view(x, d->layout, d->S, d->C_in);
  r.w = w_in, r.wn = d->C_in, r.wk = 1, r.bias = b_in;
  r.y = row_view(h, d->S, H);
  r.z = row_view(saved, d->S, 2ll * H);
  r.P = P, r.S = (int)d->S, r.N = H, r.K = d->C_in, r.act = d->act;
  rc = simt_rows_launch(d->dtype, EPI_GATE, r, st);
  if (rc) return rc;
  RowsArgs o{};
  o.a = row_view(h, d->S, H);
  o.w = w_out, o.wn = H, o.wk = 1, o.bias = b_out;
  o.res = image_view(residual, d->layout, d->S, d->C_out);
  o.y = image_view(y, d->layout, d->S, d->C_out);
  o.P = P, o.S = (int)d->S, o.N = d->C_out, o.K = H, o.act = MC_ACT_NONE;
  return simt_rows_launch(d->dtype, EPI_LAYER, o, st);
}

int mc_gated_bwd(const mc_mix_desc* d, const void* gy, const void* x, const void* w_in, const void* b_in,
                 const void* w_out, const void* saved, void* gx, void* gw_in, void* gb_in, void* gw_out, void* gb_out,
                 void* ws, size_t ws_bytes, void* stream) {
  int rc = check_desc(d, true);
  if (rc) return rc;
  if (!gy || !x || !w_in || !w_out || !saved) return MC_ERR_BAD_ARG;
  if (!ws || ws_bytes < mc_gated_workspace_bytes(d, MC_PHASE_BACKWARD)) return MC_ERR_WORKSPACE;
  if (!placed(d, {gy, x, w_in, w_out, gx}, {b_in, gw_in, gb_in, gw_out, gb_out}, {saved, ws})) return MC_ERR_BAD_ARG;
  if (d->dtype == MC_BF16) {
    Work k{(char*)ws, (cudaStream_t)stream};
    tc_gated_bwd(k, d, gy, x, w_in, b_in, w_out, saved, gx, gw_in, gb_in, gw_out, gb_out);
    return k.rc;
  }
  cudaStream_t st = (cudaStream_t)stream;
  const int H = d->hidden;
  const long long P = pixels(d);
  const size_t n2 = up256((size_t)P * 2 * H * esize(d->dtype));
  const char* h = (const char*)saved + n2;
  char* gz = (char*)ws;
  char* part = gz + n2;
  const View vgy = image_view(gy, d->layout, d->S, d->C_out), vgz = row_view(gz, d->S, 2ll * H);
  if (gx || gw_in || gb_in) {
    RowsArgs r{};
    r.a = vgy;
    r.w = w_out, r.wn = 1, r.wk = H;
    r.res = row_view(saved, d->S, 2ll * H);
    r.y = vgz;
    r.P = P, r.S = (int)d->S, r.N = H, r.K = d->C_out, r.act = d->act;
    rc = simt_rows_launch(d->dtype, EPI_GATE_BWD, r, st);
    if (rc) return rc;
  }
  if (gx) {
    RowsArgs r{};
    r.a = vgz;
    r.w = w_in, r.wn = 1, r.wk = d->C_in;
    r.y = image_view(gx, d->layout, d->S, d->C_in);
    r.P = P, r.S = (int)d->S, r.N = d->C_in, r.K = 2 * H, r.act = MC_ACT_NONE;
    rc = simt_rows_launch(d->dtype, EPI_LAYER, r, st);
    if (rc) return rc;
  }
  if (gw_in || gb_in) {
    const Shares s = shares_of(d, 2 * H, d->C_in);
    rc = param_grads(d->dtype, vgz, 2 * H, image_view(x, d->layout, d->S, d->C_in), d->C_in, s, part,
                     part + s.part, gw_in, gb_in, st);
    if (rc) return rc;
  }
  if (gw_out || gb_out) {
    const Shares s = shares_of(d, d->C_out, H);
    rc = param_grads(d->dtype, vgy, d->C_out, row_view(h, d->S, H), H, s, part, part + s.part, gw_out, gb_out, st);
  }
  return rc;
}

}  // extern "C"
