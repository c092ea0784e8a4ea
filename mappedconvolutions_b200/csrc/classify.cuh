// Softmax cross entropy of a pointwise classifier: shared declarations.
//
// With P = B * S pixels, row vectors x_p, class scores z_p = x_p W^T + b (V of them) and labels t_p:
//   lse_p = log sum_v exp(z_pv),   loss = scale sum_p (lse_p - z_p,t_p),   scale = 1 / labelled pixels, or 1
//   gz_pv = g scale (exp(z_pv - lse_p) - [v = t_p]),   gx = gz W,   gW = gz^T x,   gb = sum_p gz
// A pixel whose label is `ignore` counts nothing: its lse is kept as +infinity, and its gz is zero whatever its features are.
// A label outside [0, V) makes the loss NaN, and the gradients that the pixel takes part in: its lse is kept as NaN.
#pragma once
#include "mix.cuh"

namespace mc {
namespace classify {

// What a forward call keeps: the labelled pixels' count, lse of every pixel (float; double for MC_F64) from byte 256 on.
constexpr size_t KEPT_HEAD = 256;

// Sums of what pixels leave: value[p] (NaN or not) of labelled pixels.  `part`: SUM_BLOCKS * 2 doubles.
constexpr int SUM_BLOCKS = 296;
template <typename CT>
int sum_loss(const CT* value, const int64_t* target, long long P, long long ignore, bool mean, double* part, double* count,
             CT* loss, cudaStream_t st);

}  // namespace classify
}  // namespace mc
