from .layers import (Convolution, GatedFeedForward, MappedAvgPool, MappedAvgUnpool, MappedConvolution, MappedMaxPool,
                     MappedTransposedConvolution, PointwiseConvolution, Resample, TransposedConvolution, Unresample)

__all__ = ["Convolution", "TransposedConvolution", "MappedConvolution", "MappedTransposedConvolution",
           "MappedMaxPool", "MappedAvgPool", "MappedAvgUnpool", "Resample", "Unresample", "PointwiseConvolution",
           "GatedFeedForward"]
