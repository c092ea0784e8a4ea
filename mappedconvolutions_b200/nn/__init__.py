from .layers import (Convolution, GatedFeedForward, GroupNorm, MappedAvgPool, MappedAvgUnpool, MappedConvolution, MappedMaxPool,
                     MappedTransposedConvolution, PointwiseConvolution, PointwiseCrossEntropy, Resample, TransposedConvolution,
                     Unresample)

__all__ = ["Convolution", "TransposedConvolution", "MappedConvolution", "MappedTransposedConvolution",
           "MappedMaxPool", "MappedAvgPool", "MappedAvgUnpool", "Resample", "Unresample", "PointwiseConvolution",
           "GatedFeedForward", "GroupNorm", "PointwiseCrossEntropy"]
