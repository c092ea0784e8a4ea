// What the entry points of the channel-mixing and classification kernels share: the layout of a call's memory, tensors brought
// to rows of channels and back, shares of a sum added up.
#pragma once
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

static long long pixels(const mc_mix_desc* d) { return d->B * d->S; }

// gw (M, N) and gb (M), either of which may be null: the shares' sums, rounded once.  Shares have R rows (M or more) of ldn elements.
// A block takes 32 sums; G threads for each add every G-th share, and their results are added in order.
template <typename T, typename CT, int G>
__global__ void __launch_bounds__(32 * G) add_shares_kernel(const CT* __restrict__ part, int M, int R, int N, int ldn,
                                                            T* __restrict__ gw, const CT* __restrict__ csum,
                                                            T* __restrict__ gb, int splits) {
  __shared__ CT sums[G][32];
  const long long nw = (long long)M * N, i = blockIdx.x * 32ll + threadIdx.x % 32;
  const bool w = i < nw, in = i < nw + M && (w ? (void*)gw : (void*)gb);
  const int j0 = threadIdx.x / 32;
  CT s = CT(0);
  if (in) {
    const CT* src = w ? part + i / N * ldn + i % N : csum + (i - nw);
    const long long step = w ? (long long)R * ldn : R;
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
static void add_shares(const CT* part, int M, int N, int ldn, T* gw, const CT* csum, T* gb, int splits, cudaStream_t st, int R = 0) {
  if (!R) R = M;
  const unsigned blocks = (unsigned)(((long long)M * N + M + 31) / 32);
  if (splits >= 64 && blocks <= 2 * 148) add_shares_kernel<T, CT, 32><<<blocks, 1024, 0, st>>>(part, M, R, N, ldn, gw, csum, gb, splits);
  else add_shares_kernel<T, CT, 8><<<blocks, 256, 0, st>>>(part, M, R, N, ldn, gw, csum, gb, splits);
  MC_COUNT(1);
}

// ---- bf16: the tensor-core kernels, on rows of channels --------------------------------------------------------------
// Rows whose length is a multiple of 8 channels (16 bytes) are read and written where they lie; anything else - other
// channel counts, NCHW - is copied to padded rows in the workspace and back.
static int pad8(int c) { return (c + 7) / 8 * 8; }

// (R, C) without gaps <-> rows of ld elements (zeros behind the last one).  A block takes `chunk` rows (a multiple of 8, so
// that both sides start on 16 bytes) through shared memory, as they lie without gaps, and moves 16 bytes per access in
// global memory on both sides.  410 channels of 327 684 pixels from rows: 277 us with one element per thread.
constexpr int PACK_BYTES = 16 * 1024;
static __global__ void __launch_bounds__(256) pack_rows_kernel(const bf16* __restrict__ src, bf16* __restrict__ dst, long long R,
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
static __global__ void __launch_bounds__(256) unpack_rows_kernel(const bf16* __restrict__ src, bf16* __restrict__ dst, long long R,
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
static __global__ void __launch_bounds__(256) long_rows_kernel(const bf16* __restrict__ src, bf16* __restrict__ dst, long long R,
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
// LABELS: pixels whose label is `ignore` become rows of zeros.  (A kernel of its own: with a test for a null target in the only one,
// layers without labels took 13 % longer here, 16.5 -> 19.1 us for 64 channels of 8 x 125 x 251 pixels.)
template <int CT, bool LABELS>
__global__ void __launch_bounds__(256) planes_to_rows_kernel(const bf16* __restrict__ src, bf16* __restrict__ dst,
                                                             long long S, int C, int ld, int tiles_s, int tiles_c,
                                                             const int64_t* __restrict__ target, long long ignore) {
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
  const bool off = LABELS && s0 + s < S && target[b * S + s0 + s] == ignore;
#pragma unroll
  for (int i = 0; i < 16; ++i) tile[s * PITCH + c + i * (256 / PX)] = off ? bf16(0.f) : v[i];
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
  // (a label `ignore` makes zeros of its pixel's row; rows that are planes no more only)
  void lay_out(const mc_mix_desc* d, const void* p, const TcRows& r, const int64_t* target = nullptr, long long ignore = 0) {
    if (!run()) return;
    const int C = r.cols;
    if (d->layout == MC_NHWC || d->S == 1 || C == 1) {
      did(copy_rows(p, (void*)r.p, r.rows, C, r.ld, st));
    } else {
      planes(d, C, [&](auto ct, unsigned blocks, int ts, int tc) {
        const auto go = [&](auto labels) {
          planes_to_rows_kernel<decltype(ct)::value, decltype(labels)::value><<<blocks, 256, 0, st>>>(
              (const bf16*)p, (bf16*)r.p, d->S, C, r.ld, ts, tc, target, ignore);
        };
        target ? go(std::true_type()) : go(std::false_type());
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

}  // namespace mix
}  // namespace mc
