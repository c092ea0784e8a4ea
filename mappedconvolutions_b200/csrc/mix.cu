// C-ABI entry points of the channel-mixing layers: argument checks, workspace layout, and the sequence of products
// behind each call.
#include "mix.cuh"

namespace mc {
namespace mix {

static int esize(int dtype) { return dtype == MC_F64 ? 8 : dtype == MC_F32 ? 4 : 2; }
static int acc_size(int dtype) { return dtype == MC_F64 ? 8 : 4; }
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

static int check_desc(const mc_mix_desc* d, bool gated) {
  if (!d || d->B <= 0 || d->S <= 0 || d->C_in <= 0 || d->C_out <= 0) return MC_ERR_BAD_ARG;
  if (gated ? d->hidden <= 0 : d->hidden != 0) return MC_ERR_BAD_ARG;
  if (d->dtype != MC_F32 && d->dtype != MC_F64 && d->dtype != MC_BF16) return MC_ERR_BAD_ARG;
  if (d->layout != MC_NCHW && d->layout != MC_NHWC) return MC_ERR_BAD_ARG;
  if (d->act < MC_ACT_NONE || d->act > MC_ACT_SIGMOID) return MC_ERR_BAD_ARG;
  // pixel indices are 32-bit (element offsets are not); channel tiles are a grid's second dimension
  if (d->S >= (1ll << 31) || d->B >= (1ll << 31) || d->B * d->S >= (1ll << 31)) return MC_ERR_TOO_LARGE;
  if (d->C_in > (1 << 20) || d->C_out > (1 << 20) || d->hidden > (1 << 19)) return MC_ERR_TOO_LARGE;
  return MC_OK;
}

static long long pixels(const mc_mix_desc* d) { return d->B * d->S; }

// Shares of the pixels that a parameter gradient is summed in: about two waves of blocks, at least 256 pixels each.
struct Shares {
  long long share;
  int splits;
  size_t part, csum;  // bytes
};
static Shares shares_of(long long P, int M, int N, int dtype) {
  const long long tiles = (long long)((M + 127) / 128) * ((N + 127) / 128);
  long long n = (2 * 148 + tiles - 1) / tiles, most = (P + 255) / 256;
  if (n > most) n = most;
  Shares s;
  s.share = ((P + n - 1) / n + 15) / 16 * 16;
  s.splits = (int)((P + s.share - 1) / s.share);
  s.part = up256((size_t)s.splits * M * N * acc_size(dtype));
  s.csum = up256((size_t)s.splits * M * acc_size(dtype));
  return s;
}

// gw and gb: the shares' sums added in order and rounded once.  gw may be null, gb may be null.
template <typename T, typename CT>
__global__ void __launch_bounds__(256) add_shares_kernel(const CT* __restrict__ part, long long nw, T* __restrict__ gw,
                                                         const CT* __restrict__ csum, int nb, T* __restrict__ gb,
                                                         int splits) {
  const long long total = nw + nb;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const bool w = i < nw;
    if (!(w ? (void*)gw : (void*)gb)) continue;
    const CT* src = w ? part + i : csum + (i - nw);
    const long long step = w ? nw : nb;
    CT s = CT(0);
    for (int j = 0; j < splits; ++j) s += src[j * step];
    stv(w ? gw + i : gb + (i - nw), s);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) act_bwd_kernel(const T* __restrict__ gy, const T* __restrict__ z,
                                                      T* __restrict__ gz, long long n, int act) {
  typedef typename Traits<T>::CT CT;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll)
    stv(gz + i, (CT)ldv(gy + i) * act_slope<CT>(act, (CT)ldv(z + i)));
}

template <typename F>
static int by_type(int dtype, F f) {
  switch (dtype) {
    case MC_F32: f(float()); break;
    case MC_F64: f(double()); break;
    default: f(bf16()); break;
  }
  MC_CHECK_LAUNCH();
  return MC_OK;
}

static int param_grads(int dtype, long long P, long long S, View g, int M, View x, int N, const Shares& s, char* part,
                       char* csum, void* gw, void* gb, cudaStream_t st) {
  OuterArgs o{g, x, part, csum, P, s.share, (int)S, M, N, s.splits};
  const int rc = simt_outer_launch(dtype, o, st);
  if (rc) return rc;
  const long long nw = (long long)M * N;
  return by_type(dtype, [&](auto t) {
    typedef decltype(t) T;
    typedef typename Traits<T>::CT CT;
    add_shares_kernel<T, CT><<<grid_for(nw + M, 256), 256, 0, st>>>((const CT*)part, nw, (T*)gw, (const CT*)csum, M,
                                                                    (T*)gb, s.splits), MC_COUNT(1);
  });
}

}  // namespace mix
}  // namespace mc
using namespace mc;
using namespace mc::mix;

extern "C" {

// ---- pointwise layer ----------------------------------------------------------------------------------------

size_t mc_pointwise_saved_bytes(const mc_mix_desc* d) {
  if (check_desc(d, false) || d->act == MC_ACT_NONE) return 0;
  return up256((size_t)pixels(d) * d->C_out * esize(d->dtype));
}

size_t mc_pointwise_workspace_bytes(const mc_mix_desc* d, int32_t backward) {
  if (check_desc(d, false) || !backward) return 0;
  const Shares s = shares_of(pixels(d), d->C_out, d->C_in, d->dtype);
  return mc_pointwise_saved_bytes(d) + s.part + s.csum;
}

int mc_pointwise_fwd(const mc_mix_desc* d, const void* x, const void* w, const void* bias, const void* residual, void* y,
                     void* saved, void* ws, size_t ws_bytes, void* stream) {
  const int rc = check_desc(d, false);
  if (rc) return rc;
  if (!x || !w || !y) return MC_ERR_BAD_ARG;
  if (ws_bytes < mc_pointwise_workspace_bytes(d, 0)) return MC_ERR_WORKSPACE;
  (void)ws;
  RowsArgs r{};
  r.a = image_view(x, d->layout, d->S, d->C_in);
  r.w = w, r.wn = d->C_in, r.wk = 1, r.bias = bias;
  r.res = image_view(residual, d->layout, d->S, d->C_out);
  r.y = image_view(y, d->layout, d->S, d->C_out);
  r.z = image_view(d->act == MC_ACT_NONE ? nullptr : saved, d->layout, d->S, d->C_out);
  r.P = pixels(d), r.S = (int)d->S, r.N = d->C_out, r.K = d->C_in, r.act = d->act;
  return simt_rows_launch(d->dtype, EPI_LAYER, r, (cudaStream_t)stream);
}

int mc_pointwise_bwd(const mc_mix_desc* d, const void* gy, const void* x, const void* w, const void* saved, void* gx,
                     void* gw, void* gb, void* ws, size_t ws_bytes, void* stream) {
  int rc = check_desc(d, false);
  if (rc) return rc;
  if (!gy || !x || !w || (d->act != MC_ACT_NONE && !saved)) return MC_ERR_BAD_ARG;
  if (!ws || ws_bytes < mc_pointwise_workspace_bytes(d, 1)) return MC_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t)stream;
  const long long P = pixels(d), n = P * d->C_out;
  const Shares s = shares_of(P, d->C_out, d->C_in, d->dtype);
  char* gz = (char*)ws;
  char* part = gz + mc_pointwise_saved_bytes(d);
  const void* g = gy;
  if (d->act != MC_ACT_NONE) {
    rc = by_type(d->dtype, [&](auto t) {
      typedef decltype(t) T;
      act_bwd_kernel<T><<<grid_for(n, 256), 256, 0, st>>>((const T*)gy, (const T*)saved, (T*)gz, n, d->act), MC_COUNT(1);
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
    rc = param_grads(d->dtype, P, d->S, image_view(g, d->layout, d->S, d->C_out), d->C_out,
                     image_view(x, d->layout, d->S, d->C_in), d->C_in, s, part, part + s.part, gw, gb, st);
  return rc;
}

// ---- gated feed-forward block -----------------------------------------------------------------------------------

// kept for the backward pass: [g|u] (P, 2 H), then h (P, H)
size_t mc_gated_saved_bytes(const mc_mix_desc* d) {
  if (check_desc(d, true)) return 0;
  const size_t h = (size_t)pixels(d) * d->hidden * esize(d->dtype);
  return up256(2 * h) + up256(h);
}

size_t mc_gated_workspace_bytes(const mc_mix_desc* d, int32_t backward) {
  if (check_desc(d, true)) return 0;
  const size_t h = (size_t)pixels(d) * d->hidden * esize(d->dtype);
  if (!backward) return up256(h);
  const Shares a = shares_of(pixels(d), 2 * d->hidden, d->C_in, d->dtype);
  const Shares b = shares_of(pixels(d), d->C_out, d->hidden, d->dtype);
  const size_t sa = a.part + a.csum, sb = b.part + b.csum;
  return up256(2 * h) + (sa > sb ? sa : sb);
}

int mc_gated_fwd(const mc_mix_desc* d, const void* x, const void* w_in, const void* b_in, const void* w_out,
                 const void* b_out, const void* residual, void* y, void* saved, void* ws, size_t ws_bytes,
                 void* stream) {
  int rc = check_desc(d, true);
  if (rc) return rc;
  if (!x || !w_in || !b_in || !w_out || !y) return MC_ERR_BAD_ARG;
  if (!saved && (!ws || ws_bytes < mc_gated_workspace_bytes(d, 0))) return MC_ERR_WORKSPACE;
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

int mc_gated_bwd(const mc_mix_desc* d, const void* gy, const void* x, const void* w_in, const void* w_out,
                 const void* saved, void* gx, void* gw_in, void* gb_in, void* gw_out, void* gb_out, void* ws,
                 size_t ws_bytes, void* stream) {
  int rc = check_desc(d, true);
  if (rc) return rc;
  if (!gy || !x || !w_in || !w_out || !saved) return MC_ERR_BAD_ARG;
  if (!ws || ws_bytes < mc_gated_workspace_bytes(d, 1)) return MC_ERR_WORKSPACE;
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
    const Shares s = shares_of(P, 2 * H, d->C_in, d->dtype);
    rc = param_grads(d->dtype, P, d->S, vgz, 2 * H, image_view(x, d->layout, d->S, d->C_in), d->C_in, s, part,
                     part + s.part, gw_in, gb_in, st);
    if (rc) return rc;
  }
  if (gw_out || gb_out) {
    const Shares s = shares_of(P, d->C_out, H, d->dtype);
    rc = param_grads(d->dtype, P, d->S, vgy, d->C_out, row_view(h, d->S, H), H, s, part, part + s.part, gw_out, gb_out, st);
  }
  return rc;
}

}  // extern "C"
