"""GroupInt4Layout: a weight of 4-bit codes with a scale (and, in checkpoints that have them, a zero
point) for each row and group of inputs, multiplied by 16-bit activations as they are.

2-D tensors [N, K]; K is padded with zeros to a multiple of 32.  Storage [N, K / 2] uint8 (the even
input in the low nibble), scales [N, ceil(K / group_size)] in the tensor's dtype, zero points uint8 of
the same shape or None (8 everywhere).  State-dict keys "" (codes), "_scale" and, where there are
zero points, "_zero".  `t()` is a flag flip; linear / mm / addmm of a plain f16 / bf16 activation with
such a weight run `ck.linear_int4`; anything else dequantizes.
"""
from __future__ import annotations

import logging
from dataclasses import dataclass

import torch

from ..float_utils import roundup
from .base import BaseLayoutParams, QuantizedLayout, QuantizedTensor, dequantize_args, register_layout_op

logger = logging.getLogger(__name__)
aten = torch.ops.aten
_FAILURES = (RuntimeError, TypeError, ValueError)
NAME = "GroupInt4Layout"


class GroupInt4Layout(QuantizedLayout):
    """w ~= (code - zero) * scale, one scale and zero point for `group_size` inputs of a row."""

    @dataclass(frozen=True)
    class Params(BaseLayoutParams):
        group_size: int = 128
        zero: torch.Tensor | None = None
        transposed: bool = False

    @classmethod
    def quantize(cls, tensor: torch.Tensor, group_size: int = 128, **kwargs):
        import comfy_kitchen as ck

        if tensor.dim() != 2:
            raise ValueError(f"GroupInt4Layout requires a 2D tensor, got {tensor.dim()}D")
        shape = tuple(tensor.shape)
        pad = roundup(shape[1], 32) - shape[1]
        if pad:
            tensor = torch.nn.functional.pad(tensor, (0, pad))
        qdata, scale = ck.quantize_int4(tensor, group_size)
        return qdata, cls.Params(scale=scale, orig_dtype=tensor.dtype, orig_shape=shape, group_size=group_size)

    @classmethod
    def dequantize(cls, qdata: torch.Tensor, params: Params) -> torch.Tensor:
        import comfy_kitchen as ck

        return ck.dequantize_int4(qdata, params.scale, params.zero, params.group_size, params.orig_dtype)

    @classmethod
    def get_plain_tensors(cls, qtensor: QuantizedTensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
        return qtensor._qdata, qtensor._params.scale, qtensor._params.zero

    @classmethod
    def state_dict_tensors(cls, qdata: torch.Tensor, params: Params) -> dict[str, torch.Tensor]:
        tensors = {"": qdata, "_scale": params.scale}
        if params.zero is not None:
            tensors["_zero"] = params.zero
        return tensors

    @classmethod
    def get_padded_shape(cls, orig_shape: tuple[int, ...]) -> tuple[int, ...]:
        if len(orig_shape) != 2:
            raise ValueError(f"GroupInt4Layout requires a 2D shape, got {len(orig_shape)}D")
        return (orig_shape[0], roundup(orig_shape[1], 32))

    @classmethod
    def get_storage_shape(cls, orig_shape: tuple[int, ...]) -> tuple[int, ...]:
        rows, cols = cls.get_padded_shape(orig_shape)
        return (rows, cols // 2)

    @classmethod
    def get_logical_shape_from_storage(cls, storage_shape: tuple[int, ...]) -> tuple[int, ...]:
        return (storage_shape[0], storage_shape[1] * 2)


def _is_weight(w, transposed: bool) -> bool:
    return (isinstance(w, QuantizedTensor) and w._layout_cls == NAME and w._params.transposed is transposed
            and w._qdata.dim() == 2)


def _product(x: torch.Tensor, w: QuantizedTensor, bias) -> torch.Tensor:
    """x @ w_stored.T + bias."""
    import comfy_kitchen as ck

    codes, scale, zero = GroupInt4Layout.get_plain_tensors(w)
    pad = 2 * codes.shape[1] - x.shape[-1]
    if pad:  # the weight's padding multiplies zeros
        x = torch.nn.functional.pad(x, (0, pad))
    return ck.linear_int4(x, codes, scale, zero, bias, w._params.group_size)


def _plain(x, *tensors):
    """The arguments dequantized; weights in x's dtype, which its kernel did not take."""
    x = dequantize_args(x)
    return (x, *(t.dequantize().to(x.dtype) if isinstance(t, QuantizedTensor) else t for t in tensors))


@register_layout_op(aten.t.default, GroupInt4Layout)
def _t(qt, args, kwargs):
    x = args[0]
    p = x._params
    params = GroupInt4Layout.Params(scale=p.scale, orig_dtype=p.orig_dtype, orig_shape=tuple(p.orig_shape)[::-1],
                                    group_size=p.group_size, zero=p.zero, transposed=not p.transposed)
    return QuantizedTensor(x._qdata, NAME, params)


@register_layout_op(aten.linear.default, GroupInt4Layout)
def _linear(qt, args, kwargs):
    x, w = args[0], args[1]
    bias = args[2] if len(args) > 2 else kwargs.get("bias")
    if isinstance(x, QuantizedTensor) or not _is_weight(w, False) or x.shape[-1] != w._params.orig_shape[1]:
        return torch.nn.functional.linear(*_plain(x, w, bias))
    try:
        return _product(x, w, bias)
    except _FAILURES as e:
        logger.warning("int4 linear failed (%s); dequantizing", e)
        return torch.nn.functional.linear(*_plain(x, w, bias))


@register_layout_op(aten.mm.default, GroupInt4Layout)
def _mm(qt, args, kwargs):
    a, b = args[0], args[1]
    if isinstance(a, QuantizedTensor) or not _is_weight(b, True) or a.shape[-1] != b._params.orig_shape[0]:
        return torch.mm(*_plain(a, b))
    try:
        return _product(a, b, None)
    except _FAILURES as e:
        logger.warning("int4 mm failed (%s); dequantizing", e)
        return torch.mm(*_plain(a, b))


@register_layout_op(aten.addmm.default, GroupInt4Layout)
def _addmm(qt, args, kwargs):
    bias, a, b = args[0], args[1], args[2]
    plain = kwargs.get("beta", 1) == 1 and kwargs.get("alpha", 1) == 1 and bias.dim() == 1
    if (not plain or isinstance(a, QuantizedTensor) or not _is_weight(b, True)
            or a.shape[-1] != b._params.orig_shape[0]):
        return torch.addmm(dequantize_args(bias), *_plain(a, b), **kwargs)
    try:
        return _product(a, b, bias)
    except _FAILURES as e:
        logger.warning("int4 addmm failed (%s); dequantizing", e)
        return torch.addmm(bias, *_plain(a, b))
