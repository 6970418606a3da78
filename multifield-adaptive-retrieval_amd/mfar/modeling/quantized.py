"""8-bit linear layers for inference on the GPU (mfar_quantize_rows / mfar_int8_linear of include/mfar_hip.h).

One scale per token, computed on the fly, one per output channel, laid out once; exact integer sums on the matrix units at twice the rate of
16-bit types.  There is no CPU form and no gradient: the layers serve forwards under `torch.no_grad()`.
"""
import contextlib
from typing import Iterator, Optional, Tuple

import torch

from mfar import _native

MAX_K = 131072


def _rows(x: torch.Tensor) -> torch.Tensor:
    """[..., K] as a 2-D view of rows with contiguous elements."""
    r = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    return r if r.stride(1) == 1 or r.size(1) == 1 else r.contiguous()


def _check(x: torch.Tensor) -> None:
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_K:
        raise ValueError(f"expected [..., K] with K in 1..{MAX_K}, got {tuple(x.shape)}")
    _native.op_dtype(x)
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError("the 8-bit layers have no gradient: call them under torch.no_grad()")


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [..., K] float32 / float16 / bfloat16 -> (q int8 [..., K], scale fp32 [...]): scale = max|row| times 1 / 127 (both rounded to fp32),
    q = rint(row / scale), ties to even.  A row of zeros has scale 0; a row with an infinity or NaN has scale NaN and zeros."""
    dev = _native.op_device(x)
    _check(x)
    K = x.shape[-1]
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    r = _rows(x)
    _native.check(_native.lib().mfar_quantize_rows(dev, r.data_ptr(), _native.op_dtype(x), r.stride(0), r.shape[0], K, q.data_ptr(), K, scale.data_ptr(),
                                                   _native.op_stream(dev)))
    return q, scale


def int8_linear(x: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x [..., K] times 8-bit weights wq [N, K] with one scale per channel w_scale [N] (+ bias [N]) -> [..., N] of out_dtype (x's type if not
    given), every token quantised by its own scale on the way (`quantize_rows`).  The integer sums are exact; their conversion to fp32, the products
    with both scales and the sum with the bias each round to fp32, the result to its type."""
    dev = _native.op_device(x, wq, w_scale, bias)
    _check(x)
    K = x.shape[-1]
    if wq.dtype != torch.int8 or wq.dim() != 2 or wq.shape[1] != K:
        raise ValueError(f"expected int8 weights [N, {K}], got {wq.dtype} {tuple(wq.shape)}")
    N = wq.shape[0]
    if w_scale.dtype != torch.float32 or w_scale.shape != (N,):
        raise ValueError(f"expected float32 scales [{N}], got {w_scale.dtype} {tuple(w_scale.shape)}")
    if bias is not None:
        if not bias.is_floating_point() or bias.shape != (N,):
            raise ValueError(f"expected a float bias [{N}], got {bias.dtype} {tuple(bias.shape)}")
        bias = bias.detach().float().contiguous()
    wq, w_scale = wq.contiguous(), w_scale.contiguous()
    if wq.data_ptr() % 16:
        wq = wq.clone()
    y = torch.empty(x.shape[:-1] + (N,), dtype=out_dtype or x.dtype, device=x.device)
    r = _rows(x)
    L = _native.lib()
    n = L.mfar_int8_linear_workspace_bytes(r.shape[0], K, N)
    work = torch.empty(n, dtype=torch.uint8, device=x.device) if n > 0 else None
    _native.check(L.mfar_int8_linear(dev, r.data_ptr(), _native.op_dtype(x), r.stride(0), r.shape[0], K, N, wq.data_ptr(), w_scale.data_ptr(),
                                     None if bias is None else bias.data_ptr(), y.data_ptr(), _native.op_dtype(y), None if work is None else work.data_ptr(), n, _native.op_stream(dev)))
    return y


class Int8Linear(torch.nn.Module):
    """Inference form of a `torch.nn.Linear`: its weights as 8-bit rows (`weight`, `weight_scale`), its bias shared.  Under autocast the result has
    autocast's type, as a Linear's has; the input is quantised from whatever type it arrives in."""

    def __init__(self, linear: torch.nn.Linear):
        super().__init__()
        q, scale = quantize_rows(linear.weight.detach())
        # (parameters, not buffers: what watches where an encoder's parameters live sees these too)
        self.weight = torch.nn.Parameter(q, requires_grad=False)
        self.weight_scale = torch.nn.Parameter(scale, requires_grad=False)
        self.bias = linear.bias
        self.in_features, self.out_features = linear.in_features, linear.out_features

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        out = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype
        return int8_linear(x, self.weight, self.weight_scale, self.bias, out_dtype=out)


@contextlib.contextmanager
def int8_linears(module: torch.nn.Module) -> Iterator[int]:
    """While the context is open, every `torch.nn.Linear` below `module` is its `Int8Linear` (weights quantised as they are on entry); yields how
    many.  For forwards under `torch.no_grad()`."""
    swapped = []
    try:
        for parent in list(module.modules()):
            for name, child in list(parent.named_children()):
                if type(child) is torch.nn.Linear:
                    swapped.append((parent, name, child))
                    setattr(parent, name, Int8Linear(child))
        yield len(swapped)
    finally:
        for parent, name, child in swapped:
            setattr(parent, name, child)
