// Channel mixing at every pixel: shared declarations of the pointwise layer and the gated feed-forward block.
//
// With P = B * S pixels (S = H * W) and row vectors per pixel:
//   pointwise   z = x W^T + b,  y = act(z) + r;   gz = gy act'(z),  gx = gz W,  gW = gz^T x,  gb = sum_p gz
//   gated       [g|u] = x W_in^T + b_in,  h = act(g) u,  y = h W_out^T + b_out + r;
//               gh = gy W_out,  [gg|gu] = [gh u act'(g) | gh act(g)],  gx = [gg|gu] W_in,
//               gW_in = [gg|gu]^T x,  gb_in = sum_p [gg|gu],  gW_out = gy^T h,  gb_out = sum_p gy
#pragma once
#include "common.cuh"

namespace mc {
namespace mix {

// A (pixels, channels) matrix: element (p, c) with p = b * S + s at ptr + b * img + s * pix + c * ch.
struct View {
  const void* ptr;
  long long img, pix, ch;
};
inline View image_view(const void* p, int layout, long long S, int C) {
  View v;
  v.ptr = p;
  v.img = (long long)C * S;
  if (layout == MC_NHWC || S == 1) { v.pix = C; v.ch = 1; } else { v.pix = 1; v.ch = S; }
  return v;
}
// (P, C) rows of ld elements, whatever the number of images
inline View row_view(const void* p, long long S, long long ld) { return View{p, S * ld, ld, 1}; }

// Pixel index -> (image, pixel of the image); both below 2^31.  q = floor(p / S) by one multiplication with
// m = ceil(2^(31+l) / S), 2^(l-1) < S <= 2^l: exact for p < 2^31 (the error of m is below 2^l / 2^(31+l)).
struct PixDiv {
  uint32_t S, m;
  int l;
  PixDiv() = default;
  __host__ explicit PixDiv(uint32_t s) : S(s), l(0) {
    while ((1ull << l) < s) ++l;
    m = (uint32_t)(((1ull << (31 + l)) + s - 1) / s);
  }
  __device__ __forceinline__ void split(uint32_t p, uint32_t& b, uint32_t& s) const {
    b = (uint32_t)(((unsigned long long)p * m) >> (31 + l));
    s = p - b * S;
  }
};

// ---- activations ---------------------------------------------------------------------------------------
__device__ __forceinline__ float exp_(float v) { return expf(v); }
__device__ __forceinline__ double exp_(double v) { return exp(v); }
__device__ __forceinline__ float erf_(float v) { return erff(v); }
__device__ __forceinline__ double erf_(double v) { return erf(v); }
__device__ __forceinline__ float tanh_(float v) { return tanhf(v); }
__device__ __forceinline__ double tanh_(double v) { return tanh(v); }

template <typename CT>
__device__ __forceinline__ CT act_value(int act, CT z) {
  switch (act) {
    case MC_ACT_RELU: return z < CT(0) ? CT(0) : z;  // (NaN stays NaN)
    case MC_ACT_GELU: return CT(0.5) * z * (CT(1) + erf_(z * CT(0.70710678118654752440)));
    case MC_ACT_GELU_TANH: {
      const CT t = tanh_(CT(0.79788456080286535588) * (z + CT(0.044715) * z * z * z));
      return CT(0.5) * z * (CT(1) + t);
    }
    case MC_ACT_SILU: return z / (CT(1) + exp_(-z));
    case MC_ACT_SIGMOID: return CT(1) / (CT(1) + exp_(-z));
    default: return z;
  }
}
template <typename CT>
__device__ __forceinline__ CT act_slope(int act, CT z) {
  switch (act) {
    case MC_ACT_RELU: return z > CT(0) ? CT(1) : (z == z ? CT(0) : z);
    case MC_ACT_GELU:
      return CT(0.5) * (CT(1) + erf_(z * CT(0.70710678118654752440))) +
             z * exp_(CT(-0.5) * z * z) * CT(0.39894228040143267794);
    case MC_ACT_GELU_TANH: {
      const CT c = CT(0.79788456080286535588), z2 = z * z;
      const CT t = tanh_(c * (z + CT(0.044715) * z2 * z));
      // (z^2 can overflow where 1 - t^2 is zero: kept finite, the product is zero as it should be)
      return CT(0.5) * (CT(1) + t) + CT(0.5) * z * (CT(1) - t * t) * c * fmin(CT(1) + CT(0.134145) * z2, CT(3e38));
    }
    case MC_ACT_SILU: {
      const CT s = CT(1) / (CT(1) + exp_(-z));
      return s * (CT(1) + z * (CT(1) - s));
    }
    case MC_ACT_SIGMOID: {  // s(z) s(-z) with e = exp(-|z|): 1 - s(z) would cancel
      const CT e = exp_(-fabs(z)), q = CT(1) / (CT(1) + e);
      return e * q * q;
    }
    default: return CT(1);
  }
}

// The same as calls, for kernels whose threads hold many values in registers: inlined for each of them the elementary
// functions would be more code than the instruction cache holds (a 50 -> 99 channel layer of 131 072 pixels took 196 us
// instead of 117).  W values per call, whose latencies overlap: 90 us instead of 106.
template <typename CT, int W>
struct Values {
  CT v[W];
};
template <typename CT, int W>
struct ActBoth {
  Values<CT, W> value, slope;
};
template <typename CT, int W>
__device__ __noinline__ Values<CT, W> act_value_call(int act, Values<CT, W> z) {
  Values<CT, W> o;
#define MC_ACT_CASE(A)                                        \
  case A:                                                     \
    _Pragma("unroll") for (int e = 0; e < W; ++e) o.v[e] = act_value<CT>(A, z.v[e]); \
    break;
  switch (act) {
    MC_ACT_CASE(MC_ACT_RELU)
    MC_ACT_CASE(MC_ACT_GELU)
    MC_ACT_CASE(MC_ACT_GELU_TANH)
    MC_ACT_CASE(MC_ACT_SILU)
    MC_ACT_CASE(MC_ACT_SIGMOID)
    default: o = z;
  }
#undef MC_ACT_CASE
  return o;
}
template <typename CT, int W>
__device__ __noinline__ ActBoth<CT, W> act_both_call(int act, Values<CT, W> z) {
  ActBoth<CT, W> o;
#define MC_ACT_CASE(A)                                        \
  case A:                                                     \
    _Pragma("unroll") for (int e = 0; e < W; ++e) {           \
      o.value.v[e] = act_value<CT>(A, z.v[e]);                \
      o.slope.v[e] = act_slope<CT>(A, z.v[e]);                \
    }                                                         \
    break;
  switch (act) {
    MC_ACT_CASE(MC_ACT_RELU)
    MC_ACT_CASE(MC_ACT_GELU)
    MC_ACT_CASE(MC_ACT_GELU_TANH)
    MC_ACT_CASE(MC_ACT_SILU)
    MC_ACT_CASE(MC_ACT_SIGMOID)
    MC_ACT_CASE(MC_ACT_NONE)
  }
#undef MC_ACT_CASE
  return o;
}

// ---- kernels on the CUDA cores (mix_simt.cu) -----------------------------------------------------------------
// out[p, n] = sum_k a[p, k] w[n, k] with an epilogue:
enum Epilogue {
  EPI_LAYER = 0,  // z = acc + bias; y = act(z) + res; z kept where z.ptr is set
  EPI_GATE = 1,   // two sums per output, rows n and N + n of w: g, u; y = h = act(g) u; z = [g|u] kept
  EPI_GATE_BWD = 2  // acc = gh; g, u read from res (= [g|u]); y = [gh u act'(g) | gh act(g)]
};
struct RowsArgs {
  View a;
  const void* w;
  long long wn, wk;  // strides of w[n, k]
  const void* bias;
  View res, y, z;  // ptr == nullptr: absent
  long long P;
  int S, N, K, act;
};
int simt_rows_launch(int dtype, Epilogue epi, const RowsArgs& a, cudaStream_t st);

// part[s][m][n] = sum over the s-th share of the pixels of g[p, m] x[p, n]; csum[s][m] = sum of g[p, m] over it.  Sums are
// float (double for MC_F64).  A share is `share` pixels (or what is left of them) of one of B images of S pixels, or
// `group` whole images; per_image shares to an image (1 where group > 1).
struct OuterArgs {
  View g, x;
  void *part, *csum;
  long long S, share;
  int M, N, B, group, per_image, splits;
};
int simt_outer_launch(int dtype, const OuterArgs& a, cudaStream_t st);

// ---- kernels on the tensor cores (mix_tc.cu): bf16 rows of ld elements (a multiple of 8), 16-byte aligned ------------
struct TcRows {
  const void* p;
  long long rows;
  int cols, ld;  // ld == 0: an NCHW tensor with S pixels an image, as output of a layer or input gradient only
  long long S = 0;
};
// y = act(a w^T + bias) + r, or with backward y = r act'(a w^T + bias); w (N, K), r.p may be null (not with backward)
int tc_layer(const TcRows& a, const TcRows& w, const bf16* bias, int act, const TcRows& r, const TcRows& y, bool backward,
             cudaStream_t st);
// gx = g0 w0^T + g1 w1^T, w (N, K); g1.p may be null
int tc_input_grad(const TcRows& g0, const TcRows& w0, const TcRows& g1, const TcRows& w1, const TcRows& gx,
                  cudaStream_t st);
// h = act(g) u, [g|u] = x w_in^T + b_in
int tc_gate(const TcRows& x, const TcRows& w_in, const bf16* b_in, int act, const TcRows& h, cudaStream_t st);
// gg = gh u act'(g), gu = gh act(g), gh = gy w_out, w_out_t = w_out^T (H, C_out)
int tc_gate_bwd(const TcRows& x, const TcRows& w_in, const bf16* b_in, int act, const TcRows& gy, const TcRows& w_out_t,
                const TcRows& gg, const TcRows& gu, cudaStream_t st);
// part[s] = the s-th share of [g0|g1]^T x (rows of *ldn floats), csum[s] = its column sums of [g0|g1]; g1.p may be null
size_t tc_outer_floats(long long P, int M, int segs, int N, int* splits, int* ldn);
int tc_outer(const TcRows& g0, const TcRows& g1, const TcRows& x, float* part, float* csum, cudaStream_t st);
// mc_mix_plan for a checked bf16 description; false: no such product
bool tc_plan(const mc_mix_desc* d, int product, int sms, int32_t* out);

}  // namespace mix
}  // namespace mc
