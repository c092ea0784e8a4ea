"""Operator surface of the reference's pybind modules, bound to the sm_100a C-ABI library.

Function names, argument order and return values follow the reference's
`_mapped_convolution_ext.<module>` functions (include/nn/layers/*.h, include/util/layers/knn_layer.h
of the reference's package/ext_modules); each docstring cites the one it mirrors.  As in the
reference, outputs are freshly allocated and returned, and inputs must be contiguous and on one
device.  Differences: tensors must be CUDA tensors (there is no CPU path), bf16 activations are
accepted (with a float32 sample map), and a 4-D activation may be channels_last, in which case
the outputs are channels_last too.
"""
import weakref

import torch

from . import _lib
from ._lib import McDesc, check, lib

_DT = {torch.float32: _lib.MC_F32, torch.float64: _lib.MC_F64, torch.bfloat16: _lib.MC_BF16}


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _need_cuda(*ts):
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("mapped convolution ops are CUDA only: got a CPU tensor "
                               "(this build has no CPU path)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError("all tensors must be on the same device")
    return dev


def _layout(x):
    if x.is_contiguous():
        return _lib.MC_NCHW
    if x.dim() == 4 and x.is_contiguous(memory_format=torch.channels_last):
        return _lib.MC_NHWC
    raise RuntimeError("input must be contiguous")


def _as_layout(t, layout):
    if layout == _lib.MC_NHWC:
        return t.contiguous(memory_format=torch.channels_last)
    return t.contiguous()


def _empty(shape, like, layout, dtype=None):
    fmt = torch.channels_last if layout == _lib.MC_NHWC else torch.contiguous_format
    return torch.empty(shape, dtype=dtype or like.dtype, device=like.device, memory_format=fmt)


def _map_args(x, sample_map, interp_weights):
    """Checks the map / weights tensors; returns (map, weights-or-None)."""
    want = torch.float64 if x.dtype == torch.float64 else torch.float32
    if sample_map.dtype != want:
        if x.dtype == torch.bfloat16 and sample_map.dtype == torch.bfloat16:
            raise RuntimeError("sample map of a bfloat16 input must be float32")
        raise RuntimeError("sample map dtype %s does not match input dtype %s"
                           % (sample_map.dtype, x.dtype))
    if not sample_map.is_contiguous():
        raise RuntimeError("sample_map must be contiguous")
    if interp_weights is not None:
        if interp_weights.dtype != want:
            raise RuntimeError("interp_weights dtype must match the sample map")
        if not interp_weights.is_contiguous():
            raise RuntimeError("interp_weights must be contiguous")
    return sample_map, interp_weights


def _check_conv_args(input, sample_map, weight, bias, w0, w1, n_bias, kernel_size, grad_output=None,
                     grad_shape=None):
    """The C ABI takes raw pointers: parameter / gradient dtypes must equal the input's (the
    reference raises through weight.data<scalar_t>(), src/nn/cuda/mapped_convolution_layer.cu:57-65)
    and the shapes must be the ones the descriptor is built from."""
    if input.dim() != 4:
        raise RuntimeError("input must be 4-D (B, C, H, W)")
    if sample_map.dim() < 4 or sample_map.shape[-1] != 2:
        raise RuntimeError("sample_map must be (OH, OW, K, 2) or (OH, OW, K, P, 2)")
    if weight.dtype != input.dtype:
        raise RuntimeError("weight dtype %s does not match input dtype %s" % (weight.dtype, input.dtype))
    if bias.dtype != input.dtype:
        raise RuntimeError("bias dtype %s does not match input dtype %s" % (bias.dtype, input.dtype))
    if tuple(weight.shape) != (w0, w1, kernel_size):
        raise RuntimeError("weight must have shape (%d, %d, %d), got %s"
                           % (w0, w1, kernel_size, tuple(weight.shape)))
    if bias.numel() != n_bias:
        raise RuntimeError("bias must have %d elements, got %d" % (n_bias, bias.numel()))
    if sample_map.shape[2] != kernel_size:
        raise RuntimeError("sample_map.size(2) = %d does not match kernel_size %d"
                           % (sample_map.shape[2], kernel_size))
    if not weight.is_contiguous() or not bias.is_contiguous():
        raise RuntimeError("weight and bias must be contiguous")
    if grad_output is not None:
        if grad_output.dtype != input.dtype:
            raise RuntimeError("grad_output dtype %s does not match input dtype %s"
                               % (grad_output.dtype, input.dtype))
        if tuple(grad_output.shape) != tuple(grad_shape):
            raise RuntimeError("grad_output must have shape %s, got %s"
                               % (tuple(grad_shape), tuple(grad_output.shape)))


def _desc(x_dtype, layout, B, C_in, C_out, IH, IW, OH, OW, K, P, interp):
    if x_dtype not in _DT:
        raise RuntimeError("unsupported dtype %s (float32, float64, bfloat16)" % x_dtype)
    return McDesc(int(B), int(C_in), int(C_out), int(IH), int(IW), int(OH), int(OW), int(K), int(P),
                  int(interp), _DT[x_dtype], layout)


def _ws(nbytes, device):
    if nbytes == 0:
        return None, 0, None
    t = torch.empty(int(nbytes), dtype=torch.uint8, device=device)
    return t, int(nbytes), t.data_ptr()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _P(interp_weights):
    return 0 if interp_weights is None else int(interp_weights.shape[-1])


# ------------------------------------------------------------------------------------------
# inverse-map cache
# ------------------------------------------------------------------------------------------
# The inverse map depends only on the sample map tensor and the image sizes.  A layer is called
# with the same map tensor step after step, so the last few are kept, keyed by the tensor's
# identity and version counter (an in-place edit of the map invalidates its entry).
_INV_CACHE = []
_INV_CACHE_SIZE = 8


def _cached(kind, d, sample_map, build):
    key = (kind, sample_map.data_ptr(), sample_map._version, tuple(sample_map.shape), d.IH, d.IW,
           d.interp, sample_map.device.index)
    for i, (k, ref, buf) in enumerate(_INV_CACHE):
        if k == key and ref() is sample_map:
            if i:
                _INV_CACHE.insert(0, _INV_CACHE.pop(i))
            return buf
    buf = build()
    _INV_CACHE.insert(0, (key, weakref.ref(sample_map), buf))
    del _INV_CACHE[_INV_CACHE_SIZE:]
    return buf


def _inverse_map(d, sample_map):
    """Inverse map (+ its tap table) of a sample map, built once per map tensor."""
    def build():
        L = lib()
        dev = sample_map.device
        nbytes = L.mc_invmap_bytes(d)
        inv = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        wst, wsn, wsp = _ws(L.mc_invmap_build_workspace_bytes(d), dev)
        check(L.mc_invmap_build(d, sample_map.data_ptr(), inv.data_ptr(), nbytes, wsp, wsn,
                                _stream()))
        return inv
    return _cached("inv", d, sample_map, build)


def _tap_map(d, sample_map):
    """Forward tap table of a sample map (None if the descriptor has no tensor-core path)."""
    L = lib()
    nbytes = L.mc_tapmap_bytes(d)
    if nbytes == 0:
        return None

    def build():
        tab = torch.empty(nbytes, dtype=torch.uint8, device=sample_map.device)
        check(L.mc_tapmap_build(d, sample_map.data_ptr(), tab.data_ptr(), nbytes, _stream()))
        return tab
    return _cached("tap", d, sample_map, build)


def clear_inverse_map_cache():
    del _INV_CACHE[:]


# ------------------------------------------------------------------------------------------
# convolution
# ------------------------------------------------------------------------------------------

def _cl(t):
    return t.contiguous(memory_format=torch.channels_last)


def _a16(t):
    """The tensor-core kernels read rows with 16-byte vector loads: a view that starts off a 16-byte
    boundary (a batch slice, say) is copied into a fresh, aligned allocation."""
    return t if t is None or t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.preserve_format)


def _tensor_core_via_channels_last(input, interp_weights, make_desc):
    """bfloat16 tensors in the reference's NCHW layout: the tensor-core kernels want channels-last,
    and two extra layout passes cost far less than the generic kernels (a factor of ten and more at
    64 channels).  True if the call should be rerouted through channels-last copies."""
    if interp_weights is not None or input.dtype != torch.bfloat16 or input.dim() != 4:
        return False
    if _layout(input) != _lib.MC_NCHW:
        return False
    return lib().mc_conv_fwd_workspace_bytes(make_desc(_lib.MC_NHWC)) > 0


def _conv_forward(input, sample_map, interp_weights, weight, bias, kernel_size, interpolation,
                  _nhwc=False):
    input, sample_map = _a16(input), _a16(sample_map)
    _check_conv_args(input, sample_map, weight, bias, weight.shape[0] if weight.dim() else 0,
                     input.shape[1] if input.dim() > 1 else 0, weight.shape[0] if weight.dim() else 0,
                     kernel_size)
    dev = _need_cuda(input, sample_map, interp_weights, weight, bias)
    if not _nhwc and _tensor_core_via_channels_last(
            input, interp_weights,
            lambda lay: _desc(input.dtype, lay, input.shape[0], input.shape[1], weight.shape[0],
                              input.shape[2], input.shape[3], sample_map.shape[0], sample_map.shape[1],
                              kernel_size, 0, interpolation)):
        return _conv_forward(_cl(input), sample_map, None, weight, bias, kernel_size,
                             interpolation, _nhwc=True).contiguous()
    layout = _lib.MC_NHWC if _nhwc else _layout(input)
    sample_map, interp_weights = _map_args(input, sample_map, interp_weights)
    if not weight.is_contiguous() or not bias.is_contiguous():
        raise RuntimeError("weight and bias must be contiguous")
    B, Cin, IH, IW = input.shape
    Cout = weight.shape[0]
    OH, OW = sample_map.shape[0], sample_map.shape[1]
    d = _desc(input.dtype, layout, B, Cin, Cout, IH, IW, OH, OW, kernel_size, _P(interp_weights),
              interpolation)
    y = _empty((B, Cout, OH, OW), input, layout)
    with torch.cuda.device(dev):
        wst, wsn, wsp = _ws(lib().mc_conv_fwd_workspace_bytes(d), dev)
        tab = _tap_map(d, sample_map) if wsn and interp_weights is None else None
        if tab is not None:  # tensor-core path with the map decoded once per map tensor
            check(lib().mc_conv_fwd_tap(d, input.data_ptr(), tab.data_ptr(), weight.data_ptr(),
                                        bias.data_ptr(), y.data_ptr(), wsp, wsn, _stream()))
        else:
            check(lib().mc_conv_fwd(d, input.data_ptr(), sample_map.data_ptr(),
                                    _ptr(interp_weights), weight.data_ptr(), bias.data_ptr(),
                                    y.data_ptr(), wsp, wsn, _stream()))
    return y


def _contract_first(d):
    """Input gradient as GEMM + gather-sum (mc_conv_dgrad_tapsum) instead of gather-in-the-GEMM: when
    the layer has more output than input channels and the product z fits comfortably.  z is bf16: only for
    layers whose gathered sums are bf16 in the other path as well (whole 64-channel blocks)."""
    if d.C_in % 64 or d.C_out % 64:
        return False
    lanes = d.C_in // 8
    # (also square wide layers with a nearest map, where the gather inside the GEMM kernel is slow)
    wider = d.C_out > d.C_in or (d.C_out == d.C_in and d.C_in >= 128 and d.interp not in (1, 2))
    return (d.dtype == _lib.MC_BF16 and d.layout == _lib.MC_NHWC and d.P == 0 and wider
            and lanes & (lanes - 1) == 0
            and d.B * d.OH * d.OW * d.K * d.C_in * 2 <= 8 << 30)


def _conv_backward(grad_output, sample_map, interp_weights, input, weight, bias, kernel_size,
                   interpolation, need_input_grad=True, _nhwc=False):
    input, sample_map = _a16(input), _a16(sample_map)
    _check_conv_args(input, sample_map, weight, bias, weight.shape[0] if weight.dim() else 0,
                     input.shape[1] if input.dim() > 1 else 0, weight.shape[0] if weight.dim() else 0,
                     kernel_size, grad_output,
                     (input.shape[0], weight.shape[0], sample_map.shape[0], sample_map.shape[1]))
    dev = _need_cuda(grad_output, sample_map, interp_weights, input, weight, bias)
    if not _nhwc and _tensor_core_via_channels_last(
            input, interp_weights,
            lambda lay: _desc(input.dtype, lay, input.shape[0], input.shape[1], weight.shape[0],
                              input.shape[2], input.shape[3], sample_map.shape[0], sample_map.shape[1],
                              kernel_size, 0, interpolation)):
        g = _conv_backward(_cl(grad_output), sample_map, None, _cl(input), weight, bias, kernel_size,
                           interpolation, need_input_grad, _nhwc=True)
        return [g[0].contiguous() if g[0] is not None else None, g[1], g[2]]
    layout = _lib.MC_NHWC if _nhwc else _layout(input)
    grad_output = _a16(_as_layout(grad_output, layout))
    sample_map, interp_weights = _map_args(input, sample_map, interp_weights)
    B, Cin, IH, IW = input.shape
    Cout = weight.shape[0]
    OH, OW = sample_map.shape[0], sample_map.shape[1]
    d = _desc(input.dtype, layout, B, Cin, Cout, IH, IW, OH, OW, kernel_size, _P(interp_weights),
              interpolation)
    acc = torch.float64 if input.dtype == torch.float64 else torch.float32
    gx = _empty(input.shape, input, layout) if need_input_grad else None
    gw = torch.empty(weight.shape, dtype=acc, device=dev)
    gb = torch.empty((Cout,), dtype=acc, device=dev)
    L = lib()
    with torch.cuda.device(dev):
        inv = _inverse_map(d, sample_map) if need_input_grad and L.mc_conv_dgrad_inv_supported(d) else None
        wst, wsn, wsp = _ws(max(L.mc_conv_dgrad_workspace_bytes(d) if inv is None else
                                L.mc_conv_dgrad_inv_workspace_bytes(d),
                                L.mc_conv_wgrad_workspace_bytes(d)), dev)
        if not need_input_grad:
            pass
        elif inv is not None and _contract_first(d):
            # more output than input channels: contract with the weights first (one dense GEMM), then
            # gather-sum the narrow rows through the inverse map
            g2 = grad_output.permute(0, 2, 3, 1).reshape(B * OH * OW, Cout)   # a view of channels-last
            wr = weight.permute(0, 2, 1).reshape(Cout, kernel_size * Cin)
            z = torch.matmul(g2, wr)
            check(L.mc_conv_dgrad_tapsum(d, z.data_ptr(), inv.data_ptr(), gx.data_ptr(), _stream()))
        elif inv is not None:
            check(L.mc_conv_dgrad_inv(d, grad_output.data_ptr(), inv.data_ptr(), weight.data_ptr(),
                                      None, gx.data_ptr(), wsp, wsn, _stream()))
        else:
            check(L.mc_conv_dgrad(d, grad_output.data_ptr(), sample_map.data_ptr(),
                                  _ptr(interp_weights), weight.data_ptr(), None, gx.data_ptr(), wsp,
                                  wsn, _stream()))
        tab = _tap_map(d, sample_map) if interp_weights is None else None
        rc = -2
        if tab is not None:  # weight / bias gradient on the tensor cores from the prebuilt table
            rc = L.mc_conv_wgrad_tap(d, grad_output.data_ptr(), input.data_ptr(), tab.data_ptr(),
                                     gw.data_ptr(), gb.data_ptr(), _stream())
        if rc != -2:
            check(rc)
        else:  # MC_ERR_UNSUPPORTED: shapes only the generic kernels take
            check(L.mc_conv_wgrad(d, grad_output.data_ptr(), input.data_ptr(),
                                  sample_map.data_ptr(), _ptr(interp_weights), gw.data_ptr(),
                                  gb.data_ptr(), wsp, wsn, _stream()))
    return [gx, gw.to(weight.dtype), gb.to(bias.dtype)]


def mapped_conv_forward(input, sample_map, weight, bias, kernel_size, interpolation):
    """MappedConvForward, include/nn/layers/mapped_convolution_layer.h:64-88."""
    return _conv_forward(input, sample_map, None, weight, bias, kernel_size, interpolation)


def mapped_conv_backward(grad_output, sample_map, input, weight, bias, kernel_size, interpolation,
                         need_input_grad=True, need_weight_grad=True, relu_output=None):
    """MappedConvBackward, include/nn/layers/mapped_convolution_layer.h:90-135.
    Returns [grad_input, grad_weight, grad_bias].  need_input_grad=False (not in the reference's
    signature) skips the input gradient and returns None in its place.  relu_output: the layer's
    output behind a fused ReLU - grad_output is then masked by relu_output > 0 first."""
    if relu_output is not None:
        grad_output = torch.ops.aten.threshold_backward(grad_output, relu_output, 0)
    g = _conv_backward(grad_output, sample_map, None, input, weight, bias, kernel_size,
                       interpolation, need_input_grad)
    return g if need_weight_grad else [g[0], None, None]


def weighted_mapped_conv_forward(input, sample_map, interp_weights, weight, bias, kernel_size,
                                 interpolation):
    """WeightedMappedConvForward, include/nn/layers/weighted_mapped_convolution_layer.h:65-93."""
    return _conv_forward(input, sample_map, interp_weights, weight, bias, kernel_size,
                         interpolation)


def weighted_mapped_conv_backward(grad_output, sample_map, interp_weights, input, weight, bias,
                                  kernel_size, interpolation):
    """WeightedMappedConvBackward, include/nn/layers/weighted_mapped_convolution_layer.h:95-149."""
    return _conv_backward(grad_output, sample_map, interp_weights, input, weight, bias,
                          kernel_size, interpolation)


# ------------------------------------------------------------------------------------------
# transposed convolution
# ------------------------------------------------------------------------------------------

def _tconv_forward(input, sample_map, interp_weights, weight, bias, output_height, output_width,
                   kernel_size, interpolation, _nhwc=False):
    input, sample_map = _a16(input), _a16(sample_map)
    _check_conv_args(input, sample_map, weight, bias, input.shape[1] if input.dim() > 1 else 0,
                     weight.shape[1] if weight.dim() > 1 else 0,
                     weight.shape[1] if weight.dim() > 1 else 0, kernel_size)
    if tuple(sample_map.shape[:2]) != tuple(input.shape[2:]):
        raise RuntimeError("the sample map of a transposed convolution has the size of the input")
    dev = _need_cuda(input, sample_map, interp_weights, weight, bias)
    if not _nhwc and _tensor_core_via_channels_last(
            input, interp_weights,
            lambda lay: _desc(input.dtype, lay, input.shape[0], weight.shape[1], input.shape[1],
                              output_height, output_width, input.shape[2], input.shape[3],
                              kernel_size, 0, interpolation)):
        return _tconv_forward(_cl(input), sample_map, None, weight, bias, output_height, output_width,
                              kernel_size, interpolation, _nhwc=True).contiguous()
    layout = _lib.MC_NHWC if _nhwc else _layout(input)
    sample_map, interp_weights = _map_args(input, sample_map, interp_weights)
    if not weight.is_contiguous() or not bias.is_contiguous():
        raise RuntimeError("weight and bias must be contiguous")
    B, Cin, H, W = input.shape
    Cout = weight.shape[1]
    d = _desc(input.dtype, layout, B, Cin, Cout, output_height, output_width, H, W, kernel_size,
              _P(interp_weights), interpolation)
    y = _empty((B, Cout, int(output_height), int(output_width)), input, layout)
    L = lib()
    # The same layer seen as a convolution: the sampled image carries C_out channels, the map grid
    # C_in.  Its input gradient IS this forward pass, so the gather-form tensor-core dgrad serves.
    ds = _desc(input.dtype, layout, B, Cout, Cin, output_height, output_width, H, W, kernel_size,
               _P(interp_weights), interpolation)
    with torch.cuda.device(dev):
        if interp_weights is None and L.mc_conv_dgrad_inv_supported(ds):
            inv = _inverse_map(ds, sample_map)
            wst, wsn, wsp = _ws(L.mc_conv_dgrad_inv_workspace_bytes(ds), dev)
            check(L.mc_conv_dgrad_inv(ds, input.data_ptr(), inv.data_ptr(), weight.data_ptr(),
                                      bias.data_ptr(), y.data_ptr(), wsp, wsn, _stream()))
            return y
        wst, wsn, wsp = _ws(L.mc_tconv_workspace_bytes(d), dev)
        check(L.mc_tconv_fwd(d, input.data_ptr(), sample_map.data_ptr(), _ptr(interp_weights),
                             weight.data_ptr(), bias.data_ptr(), y.data_ptr(), wsp, wsn, _stream()))
    return y


def _tconv_backward(grad_output, sample_map, interp_weights, input, weight, bias, kernel_size,
                    interpolation, _nhwc=False):
    input, sample_map = _a16(input), _a16(sample_map)
    if grad_output.dim() != 4:
        raise RuntimeError("grad_output must be 4-D")
    _check_conv_args(input, sample_map, weight, bias, input.shape[1] if input.dim() > 1 else 0,
                     weight.shape[1] if weight.dim() > 1 else 0,
                     weight.shape[1] if weight.dim() > 1 else 0, kernel_size, grad_output,
                     (input.shape[0], weight.shape[1], grad_output.shape[2], grad_output.shape[3]))
    if tuple(sample_map.shape[:2]) != tuple(input.shape[2:]):
        raise RuntimeError("the sample map of a transposed convolution has the size of the input")
    dev = _need_cuda(grad_output, sample_map, interp_weights, input, weight, bias)
    if not _nhwc and _tensor_core_via_channels_last(
            input, interp_weights,
            lambda lay: _desc(input.dtype, lay, input.shape[0], weight.shape[1], input.shape[1],
                              grad_output.shape[2], grad_output.shape[3], input.shape[2],
                              input.shape[3], kernel_size, 0, interpolation)):
        g = _tconv_backward(_cl(grad_output), sample_map, None, _cl(input), weight, bias, kernel_size,
                            interpolation, _nhwc=True)
        return [g[0].contiguous(), g[1], g[2]]
    layout = _lib.MC_NHWC if _nhwc else _layout(input)
    grad_output = _a16(_as_layout(grad_output, layout))
    sample_map, interp_weights = _map_args(input, sample_map, interp_weights)
    B, Cin, H, W = input.shape
    Cout = weight.shape[1]
    OHt, OWt = grad_output.shape[2], grad_output.shape[3]
    d = _desc(input.dtype, layout, B, Cin, Cout, OHt, OWt, H, W, kernel_size, _P(interp_weights),
              interpolation)
    acc = torch.float64 if input.dtype == torch.float64 else torch.float32
    gx = _empty(input.shape, input, layout)
    gw = torch.empty(weight.shape, dtype=acc, device=dev)
    gb = torch.empty((Cout,), dtype=acc, device=dev)
    L = lib()
    ds = _desc(input.dtype, layout, B, Cout, Cin, OHt, OWt, H, W, kernel_size, _P(interp_weights),
               interpolation)
    with torch.cuda.device(dev):
        tab = _tap_map(ds, sample_map) if interp_weights is None else None
        if tab is not None and L.mc_conv_fwd_workspace_bytes(ds):
            # tensor-core path: input gradient = forward of the equivalent convolution applied to
            # grad_output; weight gradient = its weight gradient with the two tensors swapped
            wst, wsn, wsp = _ws(L.mc_conv_fwd_workspace_bytes(ds), dev)
            check(L.mc_conv_fwd_tap(ds, grad_output.data_ptr(), tab.data_ptr(), weight.data_ptr(),
                                    None, gx.data_ptr(), wsp, wsn, _stream()))
            rc = L.mc_conv_wgrad_tap(ds, input.data_ptr(), grad_output.data_ptr(), tab.data_ptr(),
                                     gw.data_ptr(), None, _stream())
            if rc == -2:
                rc = L.mc_conv_wgrad(ds, input.data_ptr(), grad_output.data_ptr(),
                                     sample_map.data_ptr(), None, gw.data_ptr(), None, wsp, wsn,
                                     _stream())
            check(rc)
            db = _desc(input.dtype, layout, B, Cout, Cout, OHt, OWt, OHt, OWt, 1, 0, interpolation)
            check(L.mc_bias_grad(db, grad_output.data_ptr(), gb.data_ptr(), _stream()))
            return [gx, gw.to(weight.dtype), gb.to(bias.dtype)]
        wst, wsn, wsp = _ws(L.mc_tconv_workspace_bytes(d), dev)
        check(L.mc_tconv_dgrad(d, grad_output.data_ptr(), sample_map.data_ptr(),
                               _ptr(interp_weights), weight.data_ptr(), gx.data_ptr(), wsp, wsn,
                               _stream()))
        check(L.mc_tconv_wgrad(d, grad_output.data_ptr(), input.data_ptr(), sample_map.data_ptr(),
                               _ptr(interp_weights), gw.data_ptr(), gb.data_ptr(), wsp, wsn,
                               _stream()))
    return [gx, gw.to(weight.dtype), gb.to(bias.dtype)]


def mapped_transposed_conv_forward(input, sample_map, weight, bias, output_height, output_width,
                                   kernel_size, interpolation):
    """MappedTransposedConvForward, include/nn/layers/mapped_transposed_convolution_layer.h:64-92."""
    return _tconv_forward(input, sample_map, None, weight, bias, output_height, output_width,
                          kernel_size, interpolation)


def mapped_transposed_conv_backward(grad_output, sample_map, input, weight, bias, kernel_size,
                                    interpolation):
    """MappedTransposedConvBackward, include/nn/layers/mapped_transposed_convolution_layer.h:94-143."""
    return _tconv_backward(grad_output, sample_map, None, input, weight, bias, kernel_size,
                           interpolation)


def weighted_mapped_transposed_conv_forward(input, sample_map, interp_weights, weight, bias,
                                            output_height, output_width, kernel_size,
                                            interpolation):
    """include/nn/layers/weighted_mapped_transposed_convolution_layer.h:66-98."""
    return _tconv_forward(input, sample_map, interp_weights, weight, bias, output_height,
                          output_width, kernel_size, interpolation)


def weighted_mapped_transposed_conv_backward(grad_output, sample_map, interp_weights, input,
                                             weight, bias, kernel_size, interpolation):
    """include/nn/layers/weighted_mapped_transposed_convolution_layer.h:100-155."""
    return _tconv_backward(grad_output, sample_map, interp_weights, input, weight, bias,
                           kernel_size, interpolation)


# ------------------------------------------------------------------------------------------
# pooling
# ------------------------------------------------------------------------------------------

def _pool_desc(x, sample_map, interp_weights, kernel_size, interpolation, img_hw=None):
    """Descriptor for pooling: x lives on the image for forward, on the map grid for backward."""
    layout = _layout(x)
    B, C = x.shape[0], x.shape[1]
    OH, OW = sample_map.shape[0], sample_map.shape[1]
    IH, IW = (x.shape[2], x.shape[3]) if img_hw is None else img_hw
    return layout, _desc(x.dtype, layout, B, C, C, IH, IW, OH, OW, kernel_size, _P(interp_weights),
                         interpolation)


def _max_pool(input, sample_map, interp_weights, kernel_size, interpolation):
    dev = _need_cuda(input, sample_map, interp_weights)
    sample_map, interp_weights = _map_args(input, sample_map, interp_weights)
    layout, d = _pool_desc(input, sample_map, interp_weights, kernel_size, interpolation)
    shape = (d.B, d.C_in, d.OH, d.OW)
    y = _empty(shape, input, layout)
    idx = _empty(shape, input, layout, dtype=torch.int64)
    with torch.cuda.device(dev):
        check(lib().mc_pool_max_fwd(d, input.data_ptr(), sample_map.data_ptr(),
                                    _ptr(interp_weights), y.data_ptr(), idx.data_ptr(), _stream()))
    return [y, idx]


def _max_unpool(grad_output, idx_mask, sample_map, interp_weights, input_height, input_width,
                kernel_size, interpolation):
    if idx_mask.dtype != torch.int64:
        raise RuntimeError("idx_mask must be int64, got %s" % idx_mask.dtype)
    if tuple(idx_mask.shape) != tuple(grad_output.shape):
        raise RuntimeError("idx_mask shape %s does not match grad_output shape %s"
                           % (tuple(idx_mask.shape), tuple(grad_output.shape)))
    if grad_output.dim() != 4 or tuple(grad_output.shape[2:]) != tuple(sample_map.shape[:2]):
        raise RuntimeError("grad_output must live on the map grid")
    dev = _need_cuda(grad_output, idx_mask, sample_map, interp_weights)
    layout = _layout(idx_mask) if idx_mask.dim() == 4 else _lib.MC_NCHW
    grad_output = _as_layout(grad_output, layout)
    sample_map, interp_weights = _map_args(grad_output, sample_map, interp_weights)
    IH, IW = int(input_height), int(input_width)
    _, d = _pool_desc(grad_output, sample_map, interp_weights, kernel_size, interpolation, (IH, IW))
    gx = _empty((d.B, d.C_in, IH, IW), grad_output, layout)
    L = lib()
    with torch.cuda.device(dev):
        wst, wsn, wsp = _ws(L.mc_scatter_workspace_bytes(d), dev)
        check(L.mc_pool_max_bwd(d, grad_output.data_ptr(), idx_mask.data_ptr(),
                                sample_map.data_ptr(), _ptr(interp_weights), gx.data_ptr(), wsp,
                                wsn, _stream()))
    return gx


def _avg_pool(input, sample_map, interp_weights, kernel_size, interpolation):
    dev = _need_cuda(input, sample_map, interp_weights)
    sample_map, interp_weights = _map_args(input, sample_map, interp_weights)
    layout, d = _pool_desc(input, sample_map, interp_weights, kernel_size, interpolation)
    y = _empty((d.B, d.C_in, d.OH, d.OW), input, layout)
    with torch.cuda.device(dev):
        check(lib().mc_pool_avg_fwd(d, input.data_ptr(), sample_map.data_ptr(),
                                    _ptr(interp_weights), y.data_ptr(), _stream()))
    return y


def _avg_unpool(grad_output, sample_map, interp_weights, input_height, input_width, kernel_size,
                interpolation):
    dev = _need_cuda(grad_output, sample_map, interp_weights)
    layout = _layout(grad_output)
    sample_map, interp_weights = _map_args(grad_output, sample_map, interp_weights)
    IH, IW = int(input_height), int(input_width)
    _, d = _pool_desc(grad_output, sample_map, interp_weights, kernel_size, interpolation, (IH, IW))
    gx = _empty((d.B, d.C_in, IH, IW), grad_output, layout)
    L = lib()
    with torch.cuda.device(dev):
        rc = -2
        if interp_weights is None and L.mc_invmap_bytes(d) > 0:
            # gather through the inverse map (built once per map tensor): no atomics
            inv = _inverse_map(d, sample_map)
            rc = L.mc_pool_avg_bwd_inv(d, grad_output.data_ptr(), inv.data_ptr(), gx.data_ptr(),
                                       _stream())
        if rc != -2:
            check(rc)
        else:
            wst, wsn, wsp = _ws(L.mc_scatter_workspace_bytes(d), dev)
            check(L.mc_pool_avg_bwd(d, grad_output.data_ptr(), sample_map.data_ptr(),
                                    _ptr(interp_weights), gx.data_ptr(), wsp, wsn, _stream()))
    return gx


def mapped_max_pool(input, sample_map, kernel_size, interpolation):
    """MappedMaxPoolForward, include/nn/layers/mapped_max_pooling_layer.h:46-71 -> [out, idx]."""
    return _max_pool(input, sample_map, None, kernel_size, interpolation)


def mapped_max_unpool(grad_output, idx_mask, sample_map, input_height, input_width, kernel_size,
                      interpolation):
    """MappedMaxPoolBackward, include/nn/layers/mapped_max_pooling_layer.h:73-98."""
    return _max_unpool(grad_output, idx_mask, sample_map, None, input_height, input_width,
                       kernel_size, interpolation)


def weighted_mapped_max_pool(input, sample_map, interp_weights, kernel_size, interpolation):
    """include/nn/layers/weighted_mapped_max_pooling_layer.h:42-70."""
    return _max_pool(input, sample_map, interp_weights, kernel_size, interpolation)


def weighted_mapped_max_unpool(grad_output, idx_mask, sample_map, interp_weights, input_height,
                               input_width, kernel_size, interpolation):
    """include/nn/layers/weighted_mapped_max_pooling_layer.h:72-101."""
    return _max_unpool(grad_output, idx_mask, sample_map, interp_weights, input_height,
                       input_width, kernel_size, interpolation)


def mapped_avg_pool(input, sample_map, kernel_size, interpolation):
    """MappedAvgPoolForward, include/nn/layers/mapped_avg_pooling_layer.h:42-64."""
    return _avg_pool(input, sample_map, None, kernel_size, interpolation)


def mapped_avg_unpool(grad_output, sample_map, input_height, input_width, kernel_size,
                      interpolation):
    """MappedAvgPoolBackward, include/nn/layers/mapped_avg_pooling_layer.h:66-88."""
    return _avg_unpool(grad_output, sample_map, None, input_height, input_width, kernel_size,
                       interpolation)


def weighted_mapped_avg_pool(input, sample_map, interp_weights, kernel_size, interpolation):
    """include/nn/layers/weighted_mapped_avg_pooling_layer.h:45-72."""
    return _avg_pool(input, sample_map, interp_weights, kernel_size, interpolation)


def weighted_mapped_avg_unpool(grad_output, sample_map, interp_weights, input_height, input_width,
                               kernel_size, interpolation):
    """include/nn/layers/weighted_mapped_avg_pooling_layer.h:74-107."""
    return _avg_unpool(grad_output, sample_map, interp_weights, input_height, input_width,
                       kernel_size, interpolation)


# ------------------------------------------------------------------------------------------
# resample
# ------------------------------------------------------------------------------------------

def _resample_to_map(input, sample_map, interp_weights, output_height, output_width,
                     interpolation):
    dev = _need_cuda(input, sample_map, interp_weights)
    layout = _layout(input)
    sample_map, interp_weights = _map_args(input, sample_map, interp_weights)
    B, C, H, W = input.shape
    OH, OW = int(output_height), int(output_width)
    d = _desc(input.dtype, layout, B, C, C, OH, OW, H, W, 1, _P(interp_weights), interpolation)
    y = _empty((B, C, OH, OW), input, layout)
    L = lib()
    with torch.cuda.device(dev):
        rc = -2
        if interp_weights is None and L.mc_invmap_bytes(d) > 0:
            inv = _inverse_map(d, sample_map)
            rc = L.mc_resample_scatter_inv(d, input.data_ptr(), inv.data_ptr(), y.data_ptr(),
                                           _stream())
        if rc != -2:
            check(rc)
        else:
            wst, wsn, wsp = _ws(L.mc_scatter_workspace_bytes(d), dev)
            check(L.mc_resample_scatter(d, input.data_ptr(), sample_map.data_ptr(),
                                        _ptr(interp_weights), y.data_ptr(), wsp, wsn, _stream()))
    return y


def _resample_from_map(input, sample_map, interp_weights, interpolation):
    dev = _need_cuda(input, sample_map, interp_weights)
    layout = _layout(input)
    sample_map, interp_weights = _map_args(input, sample_map, interp_weights)
    B, C, H, W = input.shape
    OH, OW = sample_map.shape[0], sample_map.shape[1]
    d = _desc(input.dtype, layout, B, C, C, H, W, OH, OW, 1, _P(interp_weights), interpolation)
    y = _empty((B, C, OH, OW), input, layout)
    with torch.cuda.device(dev):
        check(lib().mc_resample_gather(d, input.data_ptr(), sample_map.data_ptr(),
                                       _ptr(interp_weights), y.data_ptr(), _stream()))
    return y


def resample_to_map(input, sample_map, output_height, output_width, interpolation):
    """ResampleToMap (scatter), include/nn/layers/resample_layer.h:38-60."""
    return _resample_to_map(input, sample_map, None, output_height, output_width, interpolation)


def resample_from_map(input, sample_map, interpolation):
    """ResampleFromMap (gather), include/nn/layers/resample_layer.h:62-80."""
    return _resample_from_map(input, sample_map, None, interpolation)


def weighted_resample_to_map(input, sample_map, interp_weights, output_height, output_width,
                             interpolation):
    """include/nn/layers/weighted_resample_layer.h:49-77."""
    return _resample_to_map(input, sample_map, interp_weights, output_height, output_width,
                            interpolation)


def weighted_resample_from_map(input, sample_map, interp_weights, interpolation):
    """include/nn/layers/weighted_resample_layer.h:79-103."""
    return _resample_from_map(input, sample_map, interp_weights, interpolation)


# ------------------------------------------------------------------------------------------
# knn
# ------------------------------------------------------------------------------------------

def knn_forward(ref, query, k):
    """KNNForward, include/util/layers/knn_layer.h:25-35 -> [idx (B,k,N) int64 1-based, dist]."""
    dev = _need_cuda(ref, query)
    if not ref.is_contiguous() or not query.is_contiguous():
        raise RuntimeError("ref and query must be contiguous")
    if ref.dtype != torch.float32 or query.dtype != torch.float32:
        raise RuntimeError("knn works on float32 points")
    B, D, M = ref.shape
    N = query.shape[2]
    idx = torch.empty((B, k, N), dtype=torch.int64, device=dev)
    dist = torch.empty((B, k, N), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        wst, wsn, wsp = _ws(lib().mc_knn_workspace_bytes(B, D, M, N, int(k)), dev)
        check(lib().mc_knn_ws(ref.data_ptr(), query.data_ptr(), B, D, M, N, int(k), idx.data_ptr(),
                              dist.data_ptr(), wsp, wsn, _stream()))
    return [idx, dist]


# ------------------------------------------------------------------------------------------
# cube map -> equirectangular image, voting resample
# ------------------------------------------------------------------------------------------

def cube2rect(cubemap, rect_height, rect_width, interpolation):
    """Cube2RectForward, include/util/layers/cube2rect_layer.h:14-45 (src/util/cuda/cube2rect_layer.cu:11-29):
    cubemap (C, D, 6 D) float32 / float64 with faces -z, -x, +z, +x, +y, -y -> (C, rect_height, rect_width)."""
    dev = _need_cuda(cubemap)
    if cubemap.dim() != 3 or cubemap.shape[2] != 6 * cubemap.shape[1]:
        raise RuntimeError("cubemap must be (channels, cube_dim, 6 * cube_dim)")
    if cubemap.dtype not in (torch.float32, torch.float64):
        raise RuntimeError("cube2rect works on float32 / float64 images")
    if interpolation not in (0, 1):
        raise RuntimeError("interpolation must be 0 (nearest) or 1 (bilinear)")
    cubemap = cubemap.contiguous()
    C, D = cubemap.shape[0], cubemap.shape[1]
    rect = torch.empty((C, int(rect_height), int(rect_width)), dtype=cubemap.dtype, device=dev)
    with torch.cuda.device(dev):
        check(lib().mc_cube2rect(_DT[cubemap.dtype], cubemap.data_ptr(), C, D,
                                 int(rect_height), int(rect_width), int(interpolation), rect.data_ptr(), _stream()))
    return rect


def voting_resample_to_map(input, sample_map, output_height, output_width, num_candidates):
    """VotingResampleToMap, include/nn/layers/voting_resample_layer.h:34-58: input (B, C, IH, IW) int64
    labels, sample_map (IH, IW, 2) int64 target (x, y) of every input pixel -> (B, C, OH, OW) int64, the
    label most input pixels brought to each output pixel."""
    dev = _need_cuda(input, sample_map)
    if input.dtype != torch.int64 or sample_map.dtype != torch.int64:
        raise RuntimeError("voting resample works on int64 labels and an int64 map")
    if input.dim() != 4 or tuple(sample_map.shape) != (input.shape[2], input.shape[3], 2):
        raise RuntimeError("input must be (B, C, IH, IW) and sample_map (IH, IW, 2)")
    if num_candidates <= 0:
        raise RuntimeError("num_candidates must be positive")
    input, sample_map = input.contiguous(), sample_map.contiguous()
    B, C, IH, IW = input.shape
    OH, OW, NC = int(output_height), int(output_width), int(num_candidates)
    out = torch.empty((B, C, OH, OW), dtype=torch.int64, device=dev)
    # (vote counters for a slice of the batch at a time: at most ~1 GiB of scratch)
    per_image = lib().mc_voting_resample_workspace(1, C, OH, OW, NC)
    step = max(1, min(B, (1 << 30) // max(1, per_image)))
    ws = torch.empty(per_image * step, dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        for b0 in range(0, B, step):
            nb = min(step, B - b0)
            check(lib().mc_voting_resample(input[b0:].data_ptr(), sample_map.data_ptr(), nb, C, IH, IW, OH, OW, NC,
                                           ws.data_ptr(), per_image * nb, out[b0:].data_ptr(), _stream()))
    return out


# ------------------------------------------------------------------------------------------
# channel mixing: pointwise layer, gated feed-forward block (no counterpart in the reference)
# ------------------------------------------------------------------------------------------

def _check_like(t, name, shape, x):
    if t.dtype != x.dtype:
        raise RuntimeError("%s dtype %s does not match input dtype %s" % (name, t.dtype, x.dtype))
    if tuple(t.shape) != tuple(shape):
        raise RuntimeError("%s must have shape %s, got %s" % (name, tuple(shape), tuple(t.shape)))


def _check_mix(x, params, residual, c_out, grad_output=None):
    """params: (name, tensor, shape).  Same checks and messages as the compiled binding."""
    if x.dim() != 4:
        raise RuntimeError("input must be 4-D (B, C, H, W)")
    for name, t, shape in params:
        _check_like(t, name, shape, x)
        if not t.is_contiguous():
            raise RuntimeError("%s must be contiguous" % name)
    out = (x.shape[0], c_out, x.shape[2], x.shape[3])
    if residual is not None:
        _check_like(residual, "residual", out, x)
    if grad_output is not None:
        _check_like(grad_output, "grad_output", out, x)
    return out


def _mix_desc(x, layout, c_out, hidden, activation):
    if x.dtype not in _DT:
        raise RuntimeError("unsupported dtype %s (float32, float64, bfloat16)" % x.dtype)
    if max(x.shape[1], c_out, hidden) >= 1 << 31:  # (of what the description can hold; the library's limit is lower)
        raise RuntimeError("size beyond a fixed limit: more than 2^31 channels")
    return _lib.McMixDesc(x.shape[0], x.shape[2] * x.shape[3], x.shape[1], c_out, hidden, int(activation),
                          _DT[x.dtype], layout)


def _bytes(n, dev):
    return torch.empty(int(n), dtype=torch.uint8, device=dev) if n else None


def _check_saved(saved, n):
    """What a forward call kept is memory that the kernels read without further checks."""
    if n and (saved is None or saved.dtype != torch.uint8 or not saved.is_contiguous() or saved.numel() < n):
        raise RuntimeError("saved must be what the forward call of the same input, parameters and activation kept")


def _weight_dims(weight, name):
    if weight.dim() != 3 or weight.shape[2] != 1:
        raise RuntimeError("%s must be 3-D (out channels, in channels, 1)" % name)
    return weight.shape[0], weight.shape[1]


def pointwise_forward(input, weight, bias, residual=None, activation=0, keep=False):
    """act(W x + bias) + residual at every pixel -> [output, what pointwise_backward needs (keep) or None]"""
    dev = _need_cuda(input, weight, bias, residual)
    c_out, _ = _weight_dims(weight, "weight")
    shape = _check_mix(input, [("weight", weight, (c_out, input.shape[1] if input.dim() > 1 else 0, 1)), ("bias", bias, (c_out,))],
                       residual, c_out)
    layout = _layout(input)
    y = _empty(shape, input, layout)
    d = _mix_desc(input, layout, c_out, 0, activation)
    if y.numel() == 0:
        return [y, None]
    if residual is not None:
        residual = _as_layout(residual, layout)
    with torch.cuda.device(dev):
        L = lib()
        saved = _bytes(L.mc_pointwise_saved_bytes(d), dev) if keep else None
        wst, wsn, wsp = _ws(L.mc_pointwise_workspace_bytes(d, 2 if keep else 0), dev)
        input, weight, residual = _a16(input), _a16(weight), _a16(residual)
        check(L.mc_pointwise_fwd(d, input.data_ptr(), weight.data_ptr(), bias.data_ptr(), _ptr(residual), y.data_ptr(),
                                 _ptr(saved), wsp, wsn, _stream()))
    return [y, saved]


def pointwise_backward(grad_output, saved, input, weight, bias, activation=0, need_input_grad=True, need_weight_grad=True):
    """-> [grad_input, grad_weight, grad_bias]; the residual's gradient is grad_output"""
    dev = _need_cuda(grad_output, input, weight, bias, saved)
    c_out, c_in = _weight_dims(weight, "weight")
    _check_mix(input, [("weight", weight, (c_out, input.shape[1] if input.dim() > 1 else 0, 1)), ("bias", bias, (c_out,))],
               None, c_out, grad_output)
    layout = _layout(input)
    gx = _empty(input.shape, input, layout) if need_input_grad else None
    nothing = input.numel() == 0 or grad_output.numel() == 0  # no pixels, or no output channels: zeros
    make = torch.zeros if nothing else torch.empty
    gw = make(weight.shape, dtype=weight.dtype, device=dev) if need_weight_grad else None
    gb = make((c_out,), dtype=weight.dtype, device=dev) if need_weight_grad else None
    if nothing:
        return [gx if gx is None else gx.zero_(), gw, gb]
    grad_output = _as_layout(grad_output, layout)
    d = _mix_desc(input, layout, c_out, 0, activation)
    with torch.cuda.device(dev):
        L = lib()
        _check_saved(saved, L.mc_pointwise_saved_bytes(d))
        wst, wsn, wsp = _ws(L.mc_pointwise_workspace_bytes(d, 1), dev)
        input, weight, grad_output = _a16(input), _a16(weight), _a16(grad_output)
        check(L.mc_pointwise_bwd(d, grad_output.data_ptr(), input.data_ptr(), weight.data_ptr(), bias.data_ptr(), _ptr(saved),
                                 _ptr(gx), _ptr(gw), _ptr(gb), wsp, wsn, _stream()))
    return [gx, gw, gb]


def _gated_dims(x, weight_in, weight_out):
    c_out, hidden = _weight_dims(weight_out, "weight_out")
    _weight_dims(weight_in, "weight_in")
    return c_out, hidden, [("weight_in", weight_in, (2 * hidden, x.shape[1] if x.dim() > 1 else 0, 1)),
                           ("weight_out", weight_out, (c_out, hidden, 1))]


def gated_forward(input, weight_in, bias_in, weight_out, bias_out, residual=None, activation=4, keep=False):
    """W_out (act(g) * u) + bias_out + residual with [g; u] = W_in x + bias_in at every pixel
    -> [output, what gated_backward needs (keep) or None]"""
    dev = _need_cuda(input, weight_in, bias_in, weight_out, bias_out, residual)
    c_out, hidden, params = _gated_dims(input, weight_in, weight_out)
    shape = _check_mix(input, params + [("bias_in", bias_in, (2 * hidden,)), ("bias_out", bias_out, (c_out,))], residual, c_out)
    layout = _layout(input)
    y = _empty(shape, input, layout)
    d = _mix_desc(input, layout, c_out, hidden, activation)
    if y.numel() == 0:
        return [y, None]
    if residual is not None:
        residual = _as_layout(residual, layout)
    with torch.cuda.device(dev):
        L = lib()
        saved = _bytes(L.mc_gated_saved_bytes(d), dev) if keep else None
        wst, wsn, wsp = _ws(L.mc_gated_workspace_bytes(d, 2 if keep else 0), dev)
        input, weight_in, weight_out, residual = _a16(input), _a16(weight_in), _a16(weight_out), _a16(residual)
        check(L.mc_gated_fwd(d, input.data_ptr(), weight_in.data_ptr(), bias_in.data_ptr(), weight_out.data_ptr(),
                             bias_out.data_ptr(), _ptr(residual), y.data_ptr(), _ptr(saved), wsp, wsn, _stream()))
    return [y, saved]


def gated_backward(grad_output, saved, input, weight_in, bias_in, weight_out, activation=4, need_input_grad=True,
                   need_weight_grad=True):
    """-> [grad_input, grad_weight_in, grad_bias_in, grad_weight_out, grad_bias_out]"""
    dev = _need_cuda(grad_output, input, weight_in, bias_in, weight_out, saved)
    c_out, hidden, params = _gated_dims(input, weight_in, weight_out)
    _check_mix(input, params + [("bias_in", bias_in, (2 * hidden,))], None, c_out, grad_output)
    layout = _layout(input)
    gx = _empty(input.shape, input, layout) if need_input_grad else None
    nothing = input.numel() == 0 or grad_output.numel() == 0  # no pixels, or no output channels: zeros
    make = torch.zeros if nothing else torch.empty
    grads = [make(s, dtype=input.dtype, device=dev) if need_weight_grad else None
             for s in (weight_in.shape, (2 * hidden,), weight_out.shape, (c_out,))]
    if nothing:
        return [gx if gx is None else gx.zero_()] + grads
    grad_output = _as_layout(grad_output, layout)
    d = _mix_desc(input, layout, c_out, hidden, activation)
    with torch.cuda.device(dev):
        L = lib()
        _check_saved(saved, L.mc_gated_saved_bytes(d))
        wst, wsn, wsp = _ws(L.mc_gated_workspace_bytes(d, 1), dev)
        input, weight_in, weight_out, grad_output = _a16(input), _a16(weight_in), _a16(weight_out), _a16(grad_output)
        check(L.mc_gated_bwd(d, grad_output.data_ptr(), input.data_ptr(), weight_in.data_ptr(), bias_in.data_ptr(),
                             weight_out.data_ptr(), _ptr(saved), _ptr(gx), *[_ptr(g) for g in grads], wsp, wsn, _stream()))
    return [gx] + grads


# ------------------------------------------------------------------------------------------
# gradient norm and clipping (no counterpart in the reference)
# ------------------------------------------------------------------------------------------

def _dense(t):
    """Every element of one block of memory exactly once, in any order of the dimensions."""
    n = 1
    for size, stride in sorted(((s, st) for s, st in zip(t.shape, t.stride()) if s != 1), key=lambda p: p[1]):
        if stride != n:
            return False
        n *= size
    return True


def _array(ctype, values):
    return (ctype * max(1, len(values)))(*values)


def _check_gradients(tensors, norm_type):
    if not tensors:
        raise RuntimeError("no tensor given")
    _need_cuda(*tensors)
    for t in tensors:
        if t.dtype not in _DT:
            raise RuntimeError("unsupported dtype %s (float32, float64, bfloat16)" % t.dtype)
    if norm_type not in (1, 2, float("inf")):
        raise RuntimeError("norm_type must be 1, 2 or infinity")


def _check_apart(pairs, outs, strided=()):
    """No destination may share memory with another tensor of the call, no dense result with another result.  Of strided
    results only the first elements are compared: what lies between the others may belong to anyone."""
    finals = sorted((o.data_ptr(), o.data_ptr() + (o.numel() if _dense(o) else 1) * o.element_size()) for o in outs if o.numel())
    if any(b[0] < a[1] for a, b in zip(finals, finals[1:])):
        raise RuntimeError("gradients to scale must not share memory with each other")
    spans = [(t.data_ptr(), t.data_ptr() + t.element_size(), True) for t in strided if t.numel()]
    for src, dst in pairs:
        if dst.numel():
            spans.append((dst.data_ptr(), dst.data_ptr() + dst.numel() * dst.element_size(), True))
            if src.data_ptr() != dst.data_ptr() or src.dtype != dst.dtype:
                spans.append((src.data_ptr(), src.data_ptr() + src.numel() * src.element_size(), False))
    end_any = end_dst = 0
    for begin, end, is_dst in sorted(spans):
        if begin < (end_any if is_dst else end_dst):
            raise RuntimeError("gradients to scale must not share memory with each other")
        end_any = max(end_any, end)
        if is_dst:
            end_dst = max(end_dst, end)


def _norm_out(tensors, dev):
    wide = any(t.dtype == torch.float64 for t in tensors)
    norm = torch.empty((), dtype=torch.float64 if wide else torch.float32, device=dev)
    return norm, (norm.data_ptr() if wide else None), (None if wide else norm.data_ptr())


def gradient_norm(tensors, norm_type=2.0):
    """Norm of all elements of all tensors, a 0-dim float32 tensor (float64 if one of them is)."""
    tensors = [t.detach() for t in tensors]
    _check_gradients(tensors, norm_type)
    dev = tensors[0].device
    norm, p64, p32 = _norm_out(tensors, dev)
    src = [t if _dense(t) else t.contiguous() for t in tensors]
    ct, n = _lib.ctypes, len(src)
    with torch.cuda.device(dev):
        wst, wsn, wsp = _ws(lib().mc_grad_workspace_bytes(n), dev)
        check(lib().mc_grad_norm(n, _array(ct.c_void_p, [t.data_ptr() for t in src]),
                                 _array(ct.c_int64, [t.numel() for t in src]), _array(ct.c_int32, [_DT[t.dtype] for t in src]),
                                 float(norm_type), p64, p32, wsp, wsn, _stream()))
    return norm


def clip_gradients(tensors, max_norm, norm_type=2.0, out=None):
    """out[i] = tensors[i] * min(1, max_norm / (norm + 1e-6)), in place without out -> the norm before scaling"""
    grads = [t.detach() for t in tensors]
    _check_gradients(grads, norm_type)
    if not max_norm >= 0:
        raise RuntimeError("max_norm must not be negative")
    outs = grads if out is None else [t.detach() for t in out]
    if len(outs) != len(grads):
        raise RuntimeError("out must have as many tensors as there are gradients")
    _check_gradients(outs, norm_type)
    if any(o.is_inference() for o in (tensors if out is None else out)) and not torch.is_inference_mode_enabled():
        raise RuntimeError("a tensor made in inference mode can be scaled in place in inference mode only")
    dev = _need_cuda(*grads, *outs)
    src, dst, back = [], [], []
    for g, o in zip(grads, outs):
        if g.shape != o.shape:
            raise RuntimeError("out must have the gradients' shapes")
        if _dense(g) and _dense(o) and (g.stride() == o.stride() or (g.is_contiguous() and o.is_contiguous())):
            src.append(g)
            dst.append(o)
            continue
        if any(s > 1 and st == 0 for s, st in zip(o.shape, o.stride())):
            raise RuntimeError("a gradient to scale must not share memory with itself")
        src.append(g.contiguous())
        dst.append(torch.empty(g.shape, dtype=o.dtype, device=dev))
        back.append((o, dst[-1]))
    _check_apart(list(zip(src, dst)), outs, [o for o, _ in back])
    norm, p64, p32 = _norm_out(grads, dev)
    ct, n = _lib.ctypes, len(src)
    with torch.cuda.device(dev):
        wst, wsn, wsp = _ws(lib().mc_grad_workspace_bytes(n), dev)
        check(lib().mc_grad_clip(n, _array(ct.c_void_p, [t.data_ptr() for t in src]),
                                 _array(ct.c_int32, [_DT[t.dtype] for t in src]),
                                 _array(ct.c_void_p, [t.data_ptr() for t in dst]),
                                 _array(ct.c_int32, [_DT[t.dtype] for t in dst]),
                                 _array(ct.c_int64, [t.numel() for t in src]), float(norm_type), float(max_norm), p64, p32,
                                 wsp, wsn, _stream()))
        for o, t in back:
            o.copy_(t)
    for t in (tensors if out is None else out):
        torch.autograd.graph.increment_version(t)
    return norm


# ------------------------------------------------------------------------------------------
# group normalisation with an activation (no counterpart in the reference)
# ------------------------------------------------------------------------------------------

def _norm_args(x, weight, bias, groups, eps, activation):
    if x.dim() != 4:
        raise RuntimeError("input must be 4-D (B, C, H, W)")
    c = x.shape[1]
    if not (groups > 0 and c % groups == 0):
        raise RuntimeError("groups must divide the channels (%d, %d)" % (groups, c))
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _check_like(t, name, (c,), x)
            if not t.is_contiguous():
                raise RuntimeError("%s must be contiguous" % name)
    if x.dtype not in _DT:
        raise RuntimeError("unsupported dtype %s (float32, float64, bfloat16)" % x.dtype)
    if c >= 1 << 31:
        raise RuntimeError("size beyond a fixed limit: more than 2^31 channels")
    layout = _layout(x)
    return layout, _lib.McNormDesc(x.shape[0], x.shape[2] * x.shape[3], c, int(groups), int(activation), _DT[x.dtype], layout,
                                   float(eps))


def group_norm_forward(input, weight, bias, groups, eps=1e-5, activation=0):
    """act(group norm) -> [output, the statistics that group_norm_backward needs]; weight and bias may be None"""
    dev = _need_cuda(input, weight, bias)
    layout, d = _norm_args(input, weight, bias, groups, eps, activation)
    y = _empty(input.shape, input, layout)
    if y.numel() == 0:
        return [y, None]
    with torch.cuda.device(dev):
        L = lib()
        stats = _bytes(L.mc_group_norm_stats_bytes(d), dev)
        wst, wsn, wsp = _ws(L.mc_group_norm_workspace_bytes(d, 0), dev)
        input = _a16(input)
        check(L.mc_group_norm_fwd(d, input.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), _ptr(stats), wsp, wsn, _stream()))
    return [y, stats]


def group_norm_backward(grad_output, stats, input, weight, bias, groups, eps=1e-5, activation=0, need_input_grad=True,
                        need_weight_grad=True):
    """-> [grad_input, grad_weight, grad_bias]; the latter two None where there is no weight or bias"""
    dev = _need_cuda(grad_output, stats, input, weight, bias)
    layout, d = _norm_args(input, weight, bias, groups, eps, activation)
    _check_like(grad_output, "grad_output", input.shape, input)
    nothing = input.numel() == 0
    gx = _empty(input.shape, input, layout) if need_input_grad else None
    make = torch.zeros_like if nothing else torch.empty_like
    gw, gb = (make(t) if need_weight_grad and t is not None else None for t in (weight, bias))
    if nothing:
        return [gx, gw, gb]
    with torch.cuda.device(dev):
        L = lib()
        _check_saved(stats, L.mc_group_norm_stats_bytes(d))
        wst, wsn, wsp = _ws(L.mc_group_norm_workspace_bytes(d, 1), dev)
        input, grad_output = _a16(input), _a16(_as_layout(grad_output, layout))
        check(L.mc_group_norm_bwd(d, grad_output.data_ptr(), input.data_ptr(), _ptr(weight), _ptr(bias), _ptr(stats), _ptr(gx),
                                  _ptr(gw), _ptr(gb), wsp, wsn, _stream()))
    return [gx, gw, gb]


# ------------------------------------------------------------------------------------------
# softmax cross entropy of a pointwise classifier (no counterpart in the reference)
# ------------------------------------------------------------------------------------------

def _ce_args(x, weight, bias, target, ignore_index, mean):
    if x.dim() != 4:
        raise RuntimeError("input must be 4-D (B, C, H, W)")
    classes, _ = _weight_dims(weight, "weight")
    _check_mix(x, [("weight", weight, (classes, x.shape[1], 1)), ("bias", bias, (classes,))], None, classes)
    if target.dtype != torch.int64:
        raise RuntimeError("target must be int64")
    want = (x.shape[0], x.shape[2], x.shape[3])
    if tuple(target.shape) != want:
        raise RuntimeError("target must have shape %s, got %s" % (want, tuple(target.shape)))
    if x.dtype not in _DT:
        raise RuntimeError("unsupported dtype %s (float32, float64, bfloat16)" % x.dtype)
    if x.shape[1] == 0 or classes == 0:
        raise RuntimeError("there must be a channel and a class")
    if max(x.shape[1], classes) >= 1 << 31:
        raise RuntimeError("size beyond a fixed limit: more than 2^31 channels")
    layout = _layout(x)
    loss = torch.float64 if x.dtype == torch.float64 else torch.float32
    return layout, loss, _lib.McCeDesc(x.shape[0], x.shape[2] * x.shape[3], int(ignore_index), x.shape[1], classes,
                                       1 if mean else 0, _DT[x.dtype], layout)


def cross_entropy_forward(input, weight, bias, target, ignore_index=-100, mean=True):
    """softmax cross entropy of the class scores W x + bias at every pixel -> [loss, what cross_entropy_backward needs]"""
    dev = _need_cuda(input, weight, bias, target)
    layout, dtype, d = _ce_args(input, weight, bias, target, ignore_index, mean)
    if target.numel() == 0:
        return [torch.full((), float("nan") if mean else 0.0, dtype=dtype, device=dev), None]
    loss = torch.empty((), dtype=dtype, device=dev)
    with torch.cuda.device(dev):
        L = lib()
        saved = _bytes(L.mc_cross_entropy_saved_bytes(d), dev)
        wst, wsn, wsp = _ws(L.mc_cross_entropy_workspace_bytes(d, 0), dev)
        input, weight, target = _a16(input), _a16(weight), target.contiguous()
        check(L.mc_cross_entropy_fwd(d, input.data_ptr(), weight.data_ptr(), bias.data_ptr(), target.data_ptr(), loss.data_ptr(),
                                     _ptr(saved), wsp, wsn, _stream()))
    return [loss, saved]


def cross_entropy_backward(grad_loss, saved, input, weight, bias, target, ignore_index=-100, mean=True, need_input_grad=True,
                           need_weight_grad=True):
    """-> [grad_input, grad_weight, grad_bias]"""
    dev = _need_cuda(grad_loss, saved, input, weight, bias, target)
    layout, dtype, d = _ce_args(input, weight, bias, target, ignore_index, mean)
    if grad_loss.dtype != dtype or grad_loss.numel() != 1:
        raise RuntimeError("grad_loss must be one value of the loss's type")
    nothing = target.numel() == 0
    gx = _empty(input.shape, input, layout) if need_input_grad else None
    make = torch.zeros if nothing else torch.empty
    gw, gb = (make(t.shape, dtype=t.dtype, device=dev) if need_weight_grad else None for t in (weight, bias))
    if nothing:
        return [gx, gw, gb]
    with torch.cuda.device(dev):
        L = lib()
        _check_saved(saved, L.mc_cross_entropy_saved_bytes(d))
        wst, wsn, wsp = _ws(L.mc_cross_entropy_workspace_bytes(d, 1), dev)
        input, weight, target = _a16(input), _a16(weight), target.contiguous()
        check(L.mc_cross_entropy_bwd(d, grad_loss.data_ptr(), input.data_ptr(), weight.data_ptr(), bias.data_ptr(),
                                     target.data_ptr(), _ptr(saved), _ptr(gx), _ptr(gw), _ptr(gb), wsp, wsn, _stream()))
    return [gx, gw, gb]


# ------------------------------------------------------------------------------------------
# AdamW over many tensors (no counterpart in the reference)
# ------------------------------------------------------------------------------------------

def _same_order(a, b):
    """Element i of a's memory belongs to element i of b's."""
    if a.shape != b.shape or not _dense(a) or not _dense(b):
        return False
    return all(s <= 1 or x == y for s, x, y in zip(a.shape, a.stride(), b.stride())) or (a.is_contiguous() and b.is_contiguous())


def _adamw_check(params, grads, exp_avgs, exp_avg_sqs, scales, sq_scales, masters, steps):
    if not params:
        raise RuntimeError("no tensor given")
    if len({len(v) for v in (params, grads, exp_avgs, exp_avg_sqs, scales, sq_scales, masters, steps)}) != 1:
        raise RuntimeError("all lists must have as many entries as there are parameters")
    dev = _need_cuda(*[t for v in (params, grads, exp_avgs, exp_avg_sqs, scales, sq_scales, masters) for t in v])
    ready, written = [], []
    for p, g, m, v, s, q, w, step in zip(params, grads, exp_avgs, exp_avg_sqs, scales, sq_scales, masters, steps):
        if p.dtype not in _DT:
            raise RuntimeError("unsupported dtype %s (float32, float64, bfloat16)" % p.dtype)
        if g.layout != torch.strided or g.shape != p.shape or g.dtype not in _DT or \
                (g.dtype == torch.float64) != (p.dtype == torch.float64):
            raise RuntimeError("a gradient must be a dense tensor of its parameter's shape: float64 for float64 parameters, float32 or "
                               "bfloat16 for the others")
        if not _dense(p):
            raise RuntimeError("a parameter must lie in memory without gaps and overlaps")
        wide = torch.float64 if p.dtype == torch.float64 else torch.float32
        eight = m.dtype == torch.int8
        if not (_same_order(m, p) and _same_order(v, p) and
                ((m.dtype, v.dtype) == (torch.int8, torch.uint8) if eight else m.dtype == v.dtype == wide)):
            raise RuntimeError("moments must lie as their parameter does: float32 (float64 for float64 parameters), or int8 and uint8")
        if eight and p.dtype == torch.float64:
            raise RuntimeError("moments of float64 parameters are float64")
        if eight:
            want = ((p.numel() + 255) // 256,)
            if any(t is None or t.dtype != torch.float32 or tuple(t.shape) != want or not t.is_contiguous() for t in (s, q)):
                raise RuntimeError("moments in 8 bits need a float32 scale for 256 elements each")
        elif s is not None or q is not None:
            raise RuntimeError("moments in 32 bits have no scales")
        if w is not None and (p.dtype != torch.bfloat16 or w.dtype != torch.float32 or not _same_order(w, p)):
            raise RuntimeError("master weights are float32 copies of bfloat16 parameters that lie as these do")
        if step < 1:
            raise RuntimeError("steps are counted from 1")
        mine = [t for t in (p, m, v, s, q, w) if t is not None]
        if any(t.is_inference() for t in mine) and not torch.is_inference_mode_enabled():
            raise RuntimeError("a tensor made in inference mode can be updated in inference mode only")
        written += mine
        if not _same_order(g, p):
            g = torch.empty_strided(p.shape, p.stride(), dtype=g.dtype, device=dev).copy_(g)
        ready.append(g)
    spans = sorted([(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), True) for t in written if t.numel()] +
                   [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), False) for t in ready if t.numel()])
    end_any = end_dst = 0
    for begin, end, is_dst in spans:
        if begin < (end_any if is_dst else end_dst):
            raise RuntimeError("tensors of a step must not share memory with each other")
        end_any = max(end_any, end)
        if is_dst:
            end_dst = max(end_dst, end)
    return dev, ready, written


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, masters, steps, lr, beta1, beta2, eps,
               weight_decay):
    """One AdamW step over all tensors, in place; `steps` counts this one.  Moments are float32 (float64), or int8 and uint8
    codes with a float32 scale for 256 elements; scales and masters are None where there are none."""
    lists = [[None if t is None else t.detach() for t in v]
             for v in (params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, masters)]
    dev, grads, written = _adamw_check(*lists, steps)
    params, _, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, masters = lists
    ts = (_lib.McAdamwTensor * len(params))()
    for t, p, g, m, v, s, q, w, step in zip(ts, params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, masters,
                                            steps):
        t.p, t.g, t.master, t.m, t.v, t.m_scale, t.v_scale = (_ptr(x) for x in (p, g, w, m, v, s, q))
        t.numel, t.step, t.p_dtype, t.g_dtype = p.numel(), int(step), _DT[p.dtype], _DT[g.dtype]
        t.bits = 8 if m.dtype == torch.int8 else 32
    with torch.cuda.device(dev):
        check(lib().mc_adamw_step(len(params), ts, _lib.McAdamwHyper(lr, beta1, beta2, eps, weight_decay), _stream()))
    for t in written:
        torch.autograd.graph.increment_version(t)


def adamw_moments(exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales):
    """What moments in 8 bits stand for -> (list of float32 exp_avg, list of float32 exp_avg_sq)"""
    lists = (exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales)
    if not exp_avgs:
        raise RuntimeError("no tensor given")
    if len({len(v) for v in lists}) != 1:
        raise RuntimeError("all lists must have as many entries")
    dev = _need_cuda(*[t for v in lists for t in v])
    ts, out = (_lib.McAdamwTensor * len(exp_avgs))(), ([], [])
    for t, m, v, s, q in zip(ts, *lists):
        want = ((m.numel() + 255) // 256,)
        if m.dtype != torch.int8 or v.dtype != torch.uint8 or not _same_order(m, v) or \
                any(x.dtype != torch.float32 or tuple(x.shape) != want or not x.is_contiguous() for x in (s, q)):
            raise RuntimeError("moments in 8 bits are int8 and uint8 tensors that lie alike, with a float32 scale for 256 elements each")
        for o in out:
            o.append(torch.empty_strided(m.shape, m.stride(), dtype=torch.float32, device=dev))
        t.p, t.master, t.m, t.v, t.m_scale, t.v_scale = (_ptr(x) for x in (out[0][-1], out[1][-1], m, v, s, q))
        t.numel, t.bits = m.numel(), 8
    with torch.cuda.device(dev):
        check(lib().mc_adamw_moments(len(exp_avgs), ts, _stream()))
    return out
