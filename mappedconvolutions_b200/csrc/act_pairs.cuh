// Activations of bf16 kernels: fast forms on pairs of float32 values.
#pragma once
#include "common.cuh"

namespace mc {
namespace mix {

// ---- activations: fast forms, two values at a time ------------------------------------------------------------------
// (packed float32 instructions: the read-out warps are short of issue slots, not of arithmetic)
// Against 64 bits over [-100, 100] (half a bf16 step is 2^-8): values within 2^-16 of themselves for z >= -13 (GELU, 2^-17.3
// for |z| < 5), -10 (tanh form, 2^-18.5) and -87 (SiLU, sigmoid, 2^-21.4), zero within 2e-36 below; slopes, where they are
// sums that cross zero, within 2^-18 of one, the sigmoid's within 2^-17 of itself.
__device__ __forceinline__ unsigned long long& bits(float2& v) { return reinterpret_cast<unsigned long long&>(v); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(bits(d)) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(bits(d)) : "l"(bits(a)), "l"(bits(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(bits(d)) : "l"(bits(a)), "l"(bits(b)));
  return d;
}
__device__ __forceinline__ float2 two(float v) { return make_float2(v, v); }
__device__ __forceinline__ float rcp_(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float exp2_(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float2 rcp2(float2 v) { return make_float2(rcp_(v.x), rcp_(v.y)); }
__device__ __forceinline__ float2 exp2_2(float2 v) { return make_float2(exp2_(v.x), exp2_(v.y)); }
constexpr float LOG2E = 1.44269504f;
// The functions below take NV pairs at a time, one step for all of them after the other: elementary functions answer
// after tens of cycles, and with two read-out warps per scheduler nobody else fills the time.
#define MC_EACH _Pragma("unroll") for (int j = 0; j < NV; ++j)
// v <- 1 / (1 + 2^v): the logistic function of z for v = -z log2(e)
template <int NV>
__device__ __forceinline__ void logistic(float2 (&v)[NV]) {
  MC_EACH v[j] = exp2_2(v[j]);
  MC_EACH v[j] = add2(v[j], two(1.f));
  MC_EACH v[j] = rcp2(v[j]);
}
// value: z <- act(z).  both: z <- act(z), s = act'(z)
struct ActNone {
  template <int NV>
  __device__ static void value(float2 (&)[NV]) {}
  template <int NV>
  __device__ static void both(float2 (&)[NV], float2 (&s)[NV]) { MC_EACH s[j] = two(1.f); }
};
struct ActRelu {
  __device__ static float value1(float z) { return z < 0.f ? 0.f : z; }  // (NaN stays NaN)
  __device__ static float slope1(float z) { return z > 0.f ? 1.f : (z == z ? 0.f : z); }
  template <int NV>
  __device__ static void value(float2 (&z)[NV]) { MC_EACH z[j] = make_float2(value1(z[j].x), value1(z[j].y)); }
  template <int NV>
  __device__ static void both(float2 (&z)[NV], float2 (&s)[NV]) {
    MC_EACH s[j] = make_float2(slope1(z[j].x), slope1(z[j].y));
    value(z);
  }
};
struct ActGelu {
  // p = Phi(z), e = exp(-z^2 / 2).  With x = |z| / sqrt(2), t = 1 / (1 + 0.44 x): exp(x^2) erfc(x) / 2 = t q(t), q a
  // least-squares fit of the relative error over x in [0, 10] (at most 5.2e-6; e alone decays beyond).
  template <int NV>
  __device__ static void phi(const float2 (&z)[NV], float2 (&p)[NV], float2 (&e)[NV]) {
    float2 t[NV];
    MC_EACH t[j] = fma2(two(0.31112698f), make_float2(fabsf(z[j].x), fabsf(z[j].y)), two(1.f));
    MC_EACH e[j] = mul2(mul2(z[j], two(-0.5f * LOG2E)), z[j]);
    MC_EACH t[j] = rcp2(t[j]);
    MC_EACH e[j] = exp2_2(e[j]);
    MC_EACH p[j] = fma2(two(-0.07305045425891876f), t[j], two(0.1753196418285370f));
    MC_EACH p[j] = fma2(p[j], t[j], two(0.020372465252876282f));
    MC_EACH p[j] = fma2(p[j], t[j], two(0.1317897737026215f));
    MC_EACH p[j] = fma2(p[j], t[j], two(0.12128554284572601f));
    MC_EACH p[j] = fma2(p[j], t[j], two(0.12428044527769089f));
    MC_EACH p[j] = mul2(mul2(p[j], t[j]), e[j]);
    MC_EACH {
      const float2 d = fma2(p[j], two(-1.f), two(1.f));
      p[j] = make_float2(z[j].x < 0.f ? p[j].x : d.x, z[j].y < 0.f ? p[j].y : d.y);
    }
  }
  template <int NV>
  __device__ static void value(float2 (&z)[NV]) {
    float2 p[NV], e[NV];
    phi(z, p, e);
    MC_EACH z[j] = mul2(z[j], p[j]);
  }
  template <int NV>
  __device__ static void both(float2 (&z)[NV], float2 (&s)[NV]) {
    float2 p[NV], e[NV];
    phi(z, p, e);
    MC_EACH s[j] = fma2(mul2(z[j], two(0.39894228f)), e[j], p[j]);
    MC_EACH z[j] = mul2(z[j], p[j]);
  }
};
struct ActGeluTanh {  // (1 + tanh(a)) / 2 is the logistic function of 2 a
  template <int NV>
  __device__ static void part(const float2 (&z)[NV], float2 (&p)[NV]) {
    MC_EACH p[j] = mul2(mul2(z[j], two(-1.59576912f * LOG2E)), fma2(mul2(z[j], two(0.044715f)), z[j], two(1.f)));
    logistic(p);
  }
  template <int NV>
  __device__ static void value(float2 (&z)[NV]) {
    float2 p[NV];
    part(z, p);
    MC_EACH z[j] = mul2(z[j], p[j]);
  }
  template <int NV>
  __device__ static void both(float2 (&z)[NV], float2 (&s)[NV]) {
    float2 p[NV];
    part(z, p);
    MC_EACH {  // (z^2 can overflow where p or 1 - p is zero: kept finite, the product is zero as it should be)
      const float2 v = mul2(z[j], p[j]);
      float2 d = fma2(mul2(z[j], two(1.59576912f * 0.134145f)), z[j], two(1.59576912f));
      d = make_float2(fminf(d.x, 3e38f), fminf(d.y, 3e38f));
      s[j] = fma2(mul2(v, fma2(p[j], two(-1.f), two(1.f))), d, p[j]);
      z[j] = v;
    }
  }
};
struct ActSilu {
  template <int NV>
  __device__ static void value(float2 (&z)[NV]) {
    float2 p[NV];
    MC_EACH p[j] = mul2(z[j], two(-LOG2E));
    logistic(p);
    MC_EACH z[j] = mul2(z[j], p[j]);
  }
  template <int NV>
  __device__ static void both(float2 (&z)[NV], float2 (&s)[NV]) {
    float2 p[NV];
    MC_EACH p[j] = mul2(z[j], two(-LOG2E));
    logistic(p);
    MC_EACH z[j] = mul2(z[j], p[j]);
    MC_EACH s[j] = fma2(z[j], fma2(p[j], two(-1.f), two(1.f)), p[j]);
  }
};
struct ActSigmoid {
  template <int NV>
  __device__ static void value(float2 (&z)[NV]) {
    MC_EACH z[j] = mul2(z[j], two(-LOG2E));
    logistic(z);
  }
  template <int NV>
  __device__ static void both(float2 (&z)[NV], float2 (&s)[NV]) {  // slope s(z) s(-z), e = 2^(-|z| log2 e): 1 - s(z) would cancel
    float2 e[NV];
    MC_EACH e[j] = mul2(make_float2(fabsf(z[j].x), fabsf(z[j].y)), two(-LOG2E));
    MC_EACH e[j] = exp2_2(e[j]);
    MC_EACH s[j] = rcp2(add2(e[j], two(1.f)));
    MC_EACH {
      const float2 q = s[j], m = mul2(e[j], q);
      s[j] = mul2(m, q);
      z[j] = make_float2(z[j].x < 0.f ? m.x : q.x, z[j].y < 0.f ? m.y : q.y);
    }
  }
};
#undef MC_EACH

}  // namespace mix
}  // namespace mc
