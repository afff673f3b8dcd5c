"""What stands between a residual stream and the FP8 products: the norm that
makes their operands, the router's product, and the adapters added beside a
projection; and the two places where a model calls them together.

Serving only: nothing here records gradients (:mod:`hkmoe.train` does).
"""
import torch

import tk_kernel

from .layer import F8, GROUP, MoELayer, MoELayerMX, _check_dev, _like, _written, gemm_fp8, gemm_mx, mx_pack_scales

_MODES = {"group": tk_kernel.SCALE_BLOCK, "mx": tk_kernel.SCALE_MX, "tensor": tk_kernel.SCALE_TENSOR}


def rms_norm_quant(x, weight, residual=None, scales="group", scale=None, eps=1e-6, with_norm=False,
                   residual_out=None):
    """RMS norm of ``x`` (+ ``residual``) as an e4m3 operand.

    x [R, C] bf16 or fp32, weight [C] bf16 or fp32, residual like x.  Returns
    ``(q, s, r, n)``: q e4m3 [R, C]; s its scales, for ``scales`` "group" fp32
    [R, C/128], "mx" e8m0 uint8 [R, C/32], "tensor" fp32 [1] (``scale``, one
    fp32 value on the device, is used as it is and returned where given); r the
    new residual stream x + residual in x's type (x itself without a residual,
    ``residual_out`` where given: it may be x or residual); n the norm in bf16
    with ``with_norm``, else None."""
    if scales not in _MODES:
        raise RuntimeError(f"rms_norm_quant: scales must be one of {sorted(_MODES)}, got {scales!r}")
    if x.dim() != 2:
        raise RuntimeError("rms_norm_quant: x must be [R, C]")
    rows, cols = x.shape
    ws = None
    if scales == "group":
        s = x.new_empty((rows, cols // GROUP), dtype=torch.float32)
    elif scales == "mx":
        s = x.new_empty((rows, cols // 32), dtype=torch.uint8)
    elif scale is None:
        s = x.new_empty((1,), dtype=torch.float32)
        need = tk_kernel.rms_norm_quant_workspace_size(rows, tk_kernel.SCALE_TENSOR, 0)
        ws = x.new_empty((need,), dtype=torch.uint8) if need else None
    else:
        s = None
    if scale is not None and s is not None:
        raise RuntimeError('rms_norm_quant: a given scale is for scales="tensor"')
    q = _like(x, F8)
    n = _like(x, torch.bfloat16) if with_norm else None
    given = residual_out
    if residual is None:
        if residual_out is not None:
            raise RuntimeError("rms_norm_quant: residual_out needs a residual")
        r = x
    else:
        r = residual_out = _like(x, x.dtype) if residual_out is None else residual_out
    tk_kernel.dispatch_rms_norm_quant(x, residual, weight, eps, _MODES[scales], q, s, scale, residual_out, n, ws)
    _written(given)
    return q, scale if s is None else s, r, n


def router_logits(x, w, out=None):
    """fp32 [T, E] router logits of bf16 x [T, H] and the router's bf16 weight w [E, H]."""
    given = out
    if out is None:
        out = x.new_empty((x.shape[0], w.shape[0]), dtype=torch.float32)
    tk_kernel.dispatch_router_logits(x, w, out)
    _written(given)
    return out


def lora_add(y, x, a, b, ids, scaling=None, out=None, workspace=None):
    """y[t] + scaling[l] * (x[t] A_l^T) B_l^T with l = ids[t]; rows whose id is
    outside [0, L), for instance -1, have no adapter and keep y.

    y [T, N] bf16 or fp32 and x [T, H] bf16 may be column slices of wider
    buffers; a [L, R, H], b [L, N, R] bf16; ids int32 [T]; scaling fp32 [L].
    ``out`` may be y itself (in place).  ``workspace``: uint8, at least
    tk_kernel.lora_workspace_size(T, H, R) bytes, allocated per call if None."""
    if a.dim() != 3:
        raise RuntimeError("lora_add: a must be [L, R, H]")
    given = out
    if out is None:
        out = _like(y, y.dtype)
    if workspace is None:
        _, rank, hidden = a.shape
        need = tk_kernel.lora_workspace_size(y.shape[0], hidden, rank)
        workspace = a.new_empty((need,), dtype=torch.uint8) if need else None
    tk_kernel.dispatch_lora_add(y, x, a, b, ids, scaling, out, workspace)
    _written(given)
    return out


class LoraLinear:
    """An FP8 projection with low-rank adapters beside it: e4m3 weights [N, K]
    with one fp32 scale ([1]; gemm_fp8) or 1x32 e8m0 exponents (uint8 [N, K/32],
    packed here; gemm_mx), adapters a [L, R, K] and b [L, N, R] in bf16.

    A call takes what rms_norm_quant returns: the e4m3 tokens and their scales
    for the projection, the bf16 norm for the adapters, and each row's adapter."""

    def __init__(self, w_q, w_scale, a, b, scaling=None):
        _check_dev(w_q, w_scale, a, b, scaling)
        if w_q.dtype != F8 or w_q.dim() != 2:
            raise RuntimeError("LoraLinear: weights must be float8_e4m3fn [N, K]")
        if a.dim() != 3 or b.dim() != 3 or a.shape[2] != w_q.shape[1] or b.shape[1] != w_q.shape[0]:
            raise RuntimeError("LoraLinear: a must be [L, R, K] and b [L, N, R]")
        self.mx = w_scale.dtype == torch.uint8
        self.w_q = w_q.contiguous()
        self.w_scale = mx_pack_scales(w_scale) if self.mx else w_scale.contiguous()
        self.a, self.b, self.scaling = a.contiguous(), b.contiguous(), scaling

    def __call__(self, x_q, x_scale, x, ids, out_dtype=torch.bfloat16):
        if self.mx:
            y = gemm_mx(x_q, mx_pack_scales(x_scale), self.w_q, self.w_scale, out_dtype=out_dtype)
        else:
            y = gemm_fp8(x_q, self.w_q, x_scale, self.w_scale, out_dtype=out_dtype)
        return lora_add(y, x, self.a, self.b, ids, self.scaling, out=y)


class MoEBlock:
    """A MoE layer from the residual stream on: norm and quantisation, router,
    layer.  ``layer`` is a MoELayer or MoELayerMX; its scales choose the norm's."""

    def __init__(self, norm_weight, router_weight, layer, eps=1e-6):
        if not isinstance(layer, (MoELayer, MoELayerMX)):
            raise RuntimeError("MoEBlock: layer must be a MoELayer or MoELayerMX")
        if tuple(router_weight.shape) != (layer.num_experts, layer.hidden) or norm_weight.numel() != layer.hidden:
            raise RuntimeError("MoEBlock: norm_weight must be [H] and router_weight [E, H]")
        self.norm_weight, self.router_weight, self.layer, self.eps = norm_weight, router_weight, layer, eps
        self.scales = "mx" if isinstance(layer, MoELayerMX) else "group" if layer.block else "tensor"

    def __call__(self, x, residual=None, out=None):
        """x [T, H] (what the previous sublayer added, or the stream itself) ->
        (bf16 layer output [T, H], the new residual stream)."""
        q, s, r, n = rms_norm_quant(x, self.norm_weight, residual, scales=self.scales, eps=self.eps, with_norm=True)
        # a workspace per call, as in the calls before it: the layer's cached one would be shared by
        # calls on several streams and by captured graphs
        ws = q.new_empty((self.layer.workspace_size(q.shape[0]),), dtype=torch.uint8)
        return self.layer(q, s, router_logits(n, self.router_weight), out=out, workspace=ws), r
