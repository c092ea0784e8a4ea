"""nn.Module layer API, constructor and forward signatures as in the reference's
package/layers/nn/__init__.py:6-10."""
import math

import torch
import torch.nn as nn

from . import functions as F
from .checks import (REDUCTIONS, activation_code, check_args, check_input_map_shape, check_mix_args, check_norm_args,
                     check_target, interp_code)


class _ConvBase(nn.Module):
    """Parameters and initialisation shared by the two convolution layers:
    weight U(-s, s), bias U(-s, s) with s = 1/sqrt(in_channels * kernel_size); bias=False keeps a
    zero, still trainable, bias parameter (package/layers/nn/mapped_convolution_layer.py:90-108)."""

    def __init__(self, in_channels, out_channels, kernel_size, interpolation, bias, transposed):
        super().__init__()
        self.in_channels = in_channels
        self.out_channels = out_channels
        self.kernel_size = kernel_size
        self.interp = interp_code(interpolation)
        wshape = (in_channels, out_channels, kernel_size) if transposed else \
            (out_channels, in_channels, kernel_size)
        self.weight = nn.Parameter(torch.empty(*wshape))
        self.bias = nn.Parameter(torch.empty(out_channels))
        self.reset_parameters()
        if not bias:
            self.bias = nn.Parameter(torch.zeros(out_channels))

    def reset_parameters(self):
        s = 1.0 / math.sqrt(self.in_channels * self.kernel_size)
        with torch.no_grad():
            self.weight.uniform_(-s, s)
            self.bias.uniform_(-s, s)


class MappedConvolution(_ConvBase):
    """out[b, :, p] = W . [interp(x[b], sample_map[p, k]) for every channel and tap k] + bias.

    forward(x (B,C,IH,IW), sample_map (OH,OW,K,2) of (x, y) locations,
            interp_weights=None | (OH,OW,K,P) with sample_map (OH,OW,K,P,2)) -> (B,Cout,OH,OW)
    package/layers/nn/mapped_convolution_layer.py:62-121
    """

    def __init__(self, in_channels, out_channels, kernel_size=1, interpolation='bilinear',
                 bias=True, *, activation=None):
        """activation (keyword only, not in the reference): None, or 'relu' to get
        max(0, conv(x) + bias) from the convolution kernel itself instead of a separate
        element-wise pass; the layer then stands for conv followed by nn.ReLU."""
        super().__init__(in_channels, out_channels, kernel_size, interpolation, bias, False)
        assert activation in (None, 'relu'), 'activation must be None or "relu"'
        self.activation = activation

    def forward(self, x, sample_map, interp_weights=None):
        check_args(x, sample_map, interp_weights, self.in_channels, self.kernel_size)
        return F.conv(x, self.weight, self.bias, sample_map, self.kernel_size, self.interp, interp_weights,
                      self.activation == 'relu')


class MappedTransposedConvolution(_ConvBase):
    """The map has the input's size and points into the (oh, ow) output.

    forward(x (B,C,IH,IW), oh, ow, sample_map (IH,IW,K,2), interp_weights=None) -> (B,Cout,oh,ow)
    package/layers/nn/mapped_transposed_convolution_layer.py:64-121
    """

    def __init__(self, in_channels, out_channels, kernel_size=1, interpolation='bilinear',
                 bias=True):
        super().__init__(in_channels, out_channels, kernel_size, interpolation, bias, True)

    def forward(self, x, oh, ow, sample_map, interp_weights=None):
        check_args(x, sample_map, interp_weights, self.in_channels, self.kernel_size)
        check_input_map_shape(x, sample_map)
        return F.tconv(x, self.weight, self.bias, sample_map, oh, ow, self.kernel_size, self.interp, interp_weights)


class _PoolBase(nn.Module):
    def __init__(self, kernel_size, interpolation):
        super().__init__()
        self.kernel_size = kernel_size
        self.interp = interp_code(interpolation)


class MappedMaxPool(_PoolBase):
    """package/layers/nn/mapped_max_pooling_layer.py:58-90"""

    def __init__(self, kernel_size, interpolation='bilinear', return_indices=False):
        super().__init__(kernel_size, interpolation)
        self.return_indices = return_indices

    def forward(self, x, sample_map, interp_weights=None):
        check_args(x, sample_map, interp_weights, None, self.kernel_size)
        y, idx = F.max_pool(x, sample_map, int(self.kernel_size), self.interp, interp_weights)
        return (y, idx) if self.return_indices else y


class MappedAvgPool(_PoolBase):
    """package/layers/nn/mapped_avg_pooling_layer.py:56-77"""

    def __init__(self, kernel_size, interpolation='bilinear'):
        super().__init__(kernel_size, interpolation)

    def forward(self, x, sample_map, interp_weights=None):
        check_args(x, sample_map, interp_weights, None, self.kernel_size)
        return F.avg_pool(x, sample_map, int(self.kernel_size), self.interp, interp_weights)


class MappedAvgUnpool(_PoolBase):
    """package/layers/nn/mapped_avg_pooling_layer.py:124-154"""

    def __init__(self, kernel_size, interpolation='bilinear'):
        super().__init__(kernel_size, interpolation)

    def forward(self, x, oh, ow, sample_map, interp_weights=None):
        check_args(x, sample_map, interp_weights, None, self.kernel_size)
        check_input_map_shape(x, sample_map)
        return F.avg_unpool(x, oh, ow, sample_map, int(self.kernel_size), self.interp, interp_weights)


class Resample(nn.Module):
    """Scatter: every input element is added at its mapped real-valued output location.
    forward(x, sample_map (IH,IW,2), output_shape (OH,OW), interp_weights=None)
    package/layers/nn/resample_layer.py:51-79"""

    def __init__(self, interpolation='bilinear'):
        super().__init__()
        self.interp = interp_code(interpolation)

    def forward(self, x, sample_map, output_shape, interp_weights=None):
        check_args(x, sample_map, interp_weights, None, None)
        check_input_map_shape(x, sample_map)
        return F.resample(x, sample_map, (int(output_shape[0]), int(output_shape[1])), self.interp, interp_weights)


class Unresample(nn.Module):
    """Gather: a mapped convolution with unit weight, no bias and one tap.
    forward(x, sample_map (OH,OW,2), interp_weights=None)
    package/layers/nn/resample_layer.py:113-140"""

    def __init__(self, interpolation='bilinear'):
        super().__init__()
        self.interp = interp_code(interpolation)

    def forward(self, x, sample_map, interp_weights=None):
        check_args(x, sample_map, interp_weights, None, None)
        return F.unresample(x, sample_map, self.interp, interp_weights)


def _pair(v):
    return tuple(v) if isinstance(v, (tuple, list)) else (v, v)


class _GridConvBase(nn.Module):
    """The reference's two ordinary grid convolutions - its own im2col + GEMM code, kept there as
    a yardstick for the mapped layers (package/layers/nn/convolution_layer.py:34-75,
    transposed_convolution_layer.py:33-74).  Here they are the same modules (constructor,
    parameter shapes, initialisation, output sizes) on top of torch's convolutions: a grid
    convolution is not part of the mapped-convolution path and the library convolution is the
    right tool for it.

    Initialisation as in the reference: the weight is drawn once per kernel dimension (the last
    draw, U(-s, s) with s = 1/sqrt(in_channels * kh * kw), stays), then the bias with the same s,
    so that a seeded construction yields the reference's parameters."""

    def __init__(self, in_channels, out_channels, kernel_size, stride, padding, dilation, transposed):
        super().__init__()
        self.in_channels = in_channels
        self.out_channels = out_channels
        self.kernel_size = _pair(kernel_size)
        self.padding = _pair(padding)
        self.stride = _pair(stride)
        self.dilation = _pair(dilation)
        first = (in_channels, out_channels) if transposed else (out_channels, in_channels)
        self.weight = nn.Parameter(torch.empty(*first, *self.kernel_size))
        self.bias = nn.Parameter(torch.empty(out_channels))
        self.reset_parameters()

    def reset_parameters(self):
        n = self.in_channels
        with torch.no_grad():
            for k in self.kernel_size:
                n *= k
                s = 1.0 / math.sqrt(n)
                self.weight.uniform_(-s, s)
            self.bias.uniform_(-s, s)


class Convolution(_GridConvBase):
    """forward(x (B, C_in, H, W)) -> (B, C_out, (H + 2 p - d (k - 1) - 1) / s + 1, ...), the output size of
    src/nn/cpp/convolution_layer.cpp:17-24.  package/layers/nn/convolution_layer.py:34-75"""

    def __init__(self, in_channels, out_channels, kernel_size=1, stride=1, padding=0, dilation=1):
        super().__init__(in_channels, out_channels, kernel_size, stride, padding, dilation, False)

    def forward(self, x):
        return torch.nn.functional.conv2d(x, self.weight, self.bias, self.stride, self.padding, self.dilation)


class TransposedConvolution(_GridConvBase):
    """forward(x (B, C_in, H, W)) -> (B, C_out, s (H - 1) + d (k - 1) + 1 - 2 p, ...), the output size of
    src/nn/cpp/transposed_convolution_layer.cpp:54-57; weight (C_in, C_out, kh, kw).
    package/layers/nn/transposed_convolution_layer.py:33-74"""

    def __init__(self, in_channels, out_channels, kernel_size=1, stride=1, padding=0, dilation=1):
        super().__init__(in_channels, out_channels, kernel_size, stride, padding, dilation, True)

    def forward(self, x):
        return torch.nn.functional.conv_transpose2d(x, self.weight, self.bias, self.stride, self.padding, 0, 1,
                                                    self.dilation)


class PointwiseConvolution(_ConvBase):
    """act(W x + bias) + residual at every pixel or mesh vertex, in one kernel: a convolution with one tap and no sample
    map.  Parameters and their initialisation are those of MappedConvolution with kernel_size=1.  Not in the reference.

    forward(x (B,C_in,H,W), residual=None | (B,C_out,H,W)) -> (B,C_out,H,W) in x's layout
    activation: None, 'relu', 'gelu', 'gelu_tanh', 'silu' or 'sigmoid'; the residual is added behind it.
    """

    def __init__(self, in_channels, out_channels, bias=True, *, activation=None):
        super().__init__(in_channels, out_channels, 1, 'nearest', bias, False)
        self.activation = activation
        self._act = activation_code(activation)

    def forward(self, x, residual=None):
        check_mix_args(x, self.in_channels, self.out_channels, residual)
        return F.pointwise(x, self.weight, self.bias, residual, self._act)


class GatedFeedForward(nn.Module):
    """W_out (act(W_g x + b_g) * (W_u x + b_u)) + bias_out + residual at every pixel or mesh vertex: both inner
    projections, the activation and the product are one kernel, the outer projection with bias and residual a second.
    weight_in (2 * hidden, in, 1) and bias_in hold the gate's rows first, then the factor's.  Not in the reference.

    forward(x (B,C_in,H,W), residual=None | (B,C_out,H,W)) -> (B,C_out,H,W) in x's layout; out_channels defaults to
    in_channels.  Initialisation: U(-s, s) with s = 1/sqrt(number of inputs) for each projection; bias=False keeps zero,
    still trainable, biases.
    """

    def __init__(self, in_channels, hidden_channels, out_channels=None, bias=True, *, activation='silu'):
        super().__init__()
        self.in_channels = in_channels
        self.hidden_channels = hidden_channels
        self.out_channels = in_channels if out_channels is None else out_channels
        self.activation = activation
        self._act = activation_code(activation)
        self.weight_in = nn.Parameter(torch.empty(2 * hidden_channels, in_channels, 1))
        self.bias_in = nn.Parameter(torch.empty(2 * hidden_channels))
        self.weight_out = nn.Parameter(torch.empty(self.out_channels, hidden_channels, 1))
        self.bias_out = nn.Parameter(torch.empty(self.out_channels))
        self.reset_parameters()
        if not bias:
            self.bias_in = nn.Parameter(torch.zeros(2 * hidden_channels))
            self.bias_out = nn.Parameter(torch.zeros(self.out_channels))

    def reset_parameters(self):
        with torch.no_grad():
            for n, params in ((self.in_channels, (self.weight_in, self.bias_in)),
                              (self.hidden_channels, (self.weight_out, self.bias_out))):
                s = 1.0 / math.sqrt(n)
                for p in params:
                    p.uniform_(-s, s)

    def forward(self, x, residual=None):
        check_mix_args(x, self.in_channels, self.out_channels, residual)
        return F.gated(x, self.weight_in, self.bias_in, self.weight_out, self.bias_out, residual, self._act)


class GroupNorm(nn.Module):
    """act((x - mean) / sqrt(var + eps) * weight + bias), mean and variance over a group of neighbouring channels at all
    pixels of an image: torch.nn.GroupNorm of an image or mesh, its parameters, their names and their initialisation, with the
    activation in the same pass.  Not in the reference.

    forward(x (B,C,H,W)) -> (B,C,H,W) in x's layout
    activation: None, 'relu', 'gelu', 'gelu_tanh', 'silu' or 'sigmoid'.
    """

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, *, activation=None):
        super().__init__()
        assert num_groups > 0 and num_channels > 0 and num_channels % num_groups == 0, \
            'num_groups must divide num_channels ({}, {})'.format(num_groups, num_channels)
        assert eps >= 0, 'eps must not be negative ({})'.format(eps)
        self.num_groups = num_groups
        self.num_channels = num_channels
        self.eps = eps
        self.affine = affine
        self.activation = activation
        self._act = activation_code(activation)
        if affine:
            self.weight = nn.Parameter(torch.empty(num_channels))
            self.bias = nn.Parameter(torch.empty(num_channels))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)
        self.reset_parameters()

    def reset_parameters(self):
        if self.affine:
            nn.init.ones_(self.weight)
            nn.init.zeros_(self.bias)

    def forward(self, x):
        check_norm_args(x, self.num_channels)
        return F.group_norm(x, self.weight, self.bias, self.num_groups, self.eps, self._act)


class PointwiseCrossEntropy(_ConvBase):
    """Softmax cross entropy of the class scores W x + bias at every pixel or mesh vertex against a label each, without the
    scores in memory: for many classes, the vertices of a reference mesh say.  Parameters and their initialisation are those
    of PointwiseConvolution, which gives the scores themselves.  Not in the reference.

    forward(x (B,C_in,H,W), target (B,H,W) int64) -> 0-dim loss, float32 (float64 of a float64 input)
    Pixels whose target is ignore_index are left out, whatever their features are; any other target outside
    [0, num_classes) makes the loss NaN.  reduction: 'mean' over the other pixels (NaN if there are none) or 'sum'.
    """

    def __init__(self, in_channels, num_classes, bias=True, *, ignore_index=-100, reduction='mean'):
        super().__init__(in_channels, num_classes, 1, 'nearest', bias, False)
        assert reduction in REDUCTIONS, 'Unsupported reduction ({} is none of {})'.format(reduction, list(REDUCTIONS))
        self.num_classes = num_classes
        self.ignore_index = ignore_index
        self.reduction = reduction

    def forward(self, x, target):
        check_mix_args(x, self.in_channels, self.out_channels, None)
        check_target(x, target)
        return F.cross_entropy(x, self.weight, self.bias, target, self.ignore_index, REDUCTIONS[self.reduction])
