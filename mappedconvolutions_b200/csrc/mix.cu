// C-ABI entry points of the channel-mixing layers: argument checks, workspace layout, and the sequence of products
// behind each call.
#include "mix_work.cuh"

namespace mc {
namespace mix {

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
