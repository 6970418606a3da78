"""Attention with a learned relative position bias by buckets, on the GPU (mfar_attention_* of include/mfar_hip.h).

The attention of the gtr-t5 encoders (reference mfar/modeling/util.py:22-36 builds them from a pre-trained T5): no position in the inputs,
one learned number per (bucket of key - query, head) added to the scores.  One pass over the keys, nothing of size queries x keys in memory,
forward and backward; the bias table's gradient comes out of the same backward pass.  There is no CPU form.
"""
import ctypes
import functools
from typing import Optional, Union

import torch

from mfar import _native


@functools.lru_cache(maxsize=64)
def bucket_borders(num_buckets: int, causal: bool, max_distance: int):
    """First distance of every shared bucket after the first, as a C array.  Half of a side's buckets (`each`) hold one distance each; distance
    d >= each falls into bucket each + floor(log(d / each) / log(max_distance / each) * (side - each)), the last bucket holding the rest.
    In whole numbers: the floor is >= j exactly when d^n >= max_distance^j each^(n - j), n = side - each."""
    side = num_buckets if causal else num_buckets // 2
    each = side // 2
    if num_buckets > 256 or each < 1 or (not causal and num_buckets % 2):
        raise ValueError(f"num_buckets must be at most 256, at least {2 if causal else 4}{'' if causal else ' and even'}, got {num_buckets}")
    if max_distance <= each:
        raise ValueError(f"max_distance must be over {each} for {num_buckets} buckets, got {max_distance}")
    n = side - each
    out, d = [], each
    for j in range(1, n):
        need = max_distance ** j * each ** (n - j)
        while d ** n < need:
            d += 1
            if d > 1023:
                raise ValueError(f"max_distance {max_distance}: the last bucket must begin at a distance of at most 1023")
        out.append(d)
    return (ctypes.c_int32 * len(out))(*out)


def relative_buckets(distance: torch.Tensor, num_buckets: int, causal: bool, max_distance: int) -> torch.Tensor:
    """Bucket of each key position - query position (any integer tensor, any device): what the kernels add the table's row of."""
    borders = torch.tensor(list(bucket_borders(num_buckets, causal, max_distance)), device=distance.device, dtype=torch.int64)
    side = num_buckets if causal else num_buckets // 2
    far = (-distance).clamp(min=0) if causal else distance.abs()
    shared = side // 2 + torch.searchsorted(borders, far.contiguous().to(torch.int64), right=True)
    b = torch.where(far < side // 2, far, shared)
    return b if causal else b + side * (distance > 0).to(b.dtype)


@functools.lru_cache(maxsize=64)
def _borders(num_buckets: int, causal: bool, max_distance: int):
    b = bucket_borders(num_buckets, causal, max_distance)
    return ctypes.cast(b, ctypes.POINTER(ctypes.c_int32)), len(b)      # (the pointer keeps the array alive)


def _layout(x: torch.Tensor):
    """(x as the kernels can read it, its strides over batch, rows and heads): last dim contiguous, rows and base on 16-byte boundaries, row
    strides of at most 2^22 elements; copied where it is not."""
    b, l, h, d = x.stride()
    es = x.element_size()
    if d == 1 and l <= 4194304 and not ((b | l | h) * es | x.data_ptr()) & 15:
        return x, b, (l if x.size(1) > 1 else 0), h
    n = x.size()
    b, l, h = (0 if n[i] == 1 else s for i, s in enumerate((b, l, h)))    # (a dim of one element may have any stride)
    if (d != 1 and n[3] != 1) or l > 4194304 or ((b | l | h) * es | x.data_ptr()) & 15:
        x = x.contiguous()
        b, l, h = n[1] * n[2] * n[3], n[2] * n[3], n[3]
        if x.data_ptr() & 15:
            x = x.clone()
    return x, b, l, h


def _call(q, k, v, table, key_mask, q_start, causal, borders, scale):
    """(the C struct of one call's inputs, the tensors that must outlive it)."""
    q, q_b, q_l, q_h = _layout(q)
    k, k_b, k_l, k_h = _layout(k)
    v, v_b, v_l, v_h = _layout(v)
    B, Lq, H, D = q.shape
    each = torch.is_tensor(q_start)
    a = _native.Attention(_native.op_dtype(q), B, Lq, k.shape[1], H, D, causal, table.shape[0], borders[1], scale, borders[0], table.data_ptr(),
                          q.data_ptr(), k.data_ptr(), v.data_ptr(), q_b, q_l, q_h, k_b, k_l, k_h, v_b, v_l, v_h,
                          None if key_mask is None else key_mask.data_ptr(), 0 if key_mask is None or B == 1 else key_mask.stride(0),
                          q_start.data_ptr() if each else None, 0 if each else q_start)
    return a, (q, k, v)


def _workspace(a, backward, device):
    n = _native.lib().mfar_attention_workspace_bytes(a, backward)
    if n < 0:
        _native.check(int(n))
    if n == 0:
        return None
    w = torch.empty(n, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = w.data_ptr(), n
    return w


def _forward(q, k, v, table, key_mask, q_start, causal, borders, scale, keep):
    a, (q, k, v) = _call(q, k, v, table, key_mask, q_start, causal, borders, scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lo = lse = None
    a.out = out.data_ptr()
    if keep:
        lse = torch.empty(q.shape[0], q.shape[2], q.shape[1], dtype=torch.float32, device=q.device)
        a.lse = lse.data_ptr()
        if q.dtype != torch.float32:
            lo = torch.empty_like(out)
            a.out_lo = lo.data_ptr()
    work = _workspace(a, False, q.device)      # noqa: F841 -- alive until the call is enqueued
    dev = q.get_device()
    _native.check(_native.lib().mfar_attention_forward(dev, a, _native.op_stream(dev)))
    return out, lo, lse, (q, k, v)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, key_mask, q_start, causal, borders, scale):
        out, lo, lse, (q, k, v) = _forward(q, k, v, table, key_mask, q_start, causal, borders, scale, True)
        start = q_start if torch.is_tensor(q_start) else None
        ctx.save_for_backward(q, k, v, table, key_mask, start, out, lo, lse)
        ctx.rest = (None if start is not None else q_start, causal, borders, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, table, key_mask, start, out, lo, lse = ctx.saved_tensors
        q_start, causal, borders, scale = ctx.rest
        dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
        if q.numel() == 0 or k.numel() == 0:
            return dq.zero_(), dk.zero_(), dv.zero_(), torch.zeros_like(table), None, None, None, None, None
        a, keep = _call(q, k, v, table, key_mask, q_start if start is None else start, causal, borders, scale)      # noqa: F841
        dout, a.do_b, a.do_l, a.do_h = _layout(dout)
        a.out, a.lse, a.dout = out.data_ptr(), lse.data_ptr(), dout.data_ptr()
        if lo is not None:
            a.out_lo = lo.data_ptr()
        a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        dtable = None
        if ctx.needs_input_grad[3]:
            dtable = torch.empty_like(table)
            a.dtable = dtable.data_ptr()
        work = _workspace(a, True, q.device)      # noqa: F841
        dev = q.get_device()
        _native.check(_native.lib().mfar_attention_backward(dev, a, _native.op_stream(dev)))
        return dq, dk, dv, dtable, None, None, None, None, None


def relative_bias_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, *, key_mask: Optional[torch.Tensor] = None,
                            causal: bool = False, max_distance: int = 128, q_start: Union[int, torch.Tensor] = 0, scale: float = 1.0) -> torch.Tensor:
    """softmax(scale q k' + table[bucket(key position - query position)]) v per head -> [B, Lq, H, D], differentiable in q, k, v and table.

    q [B, Lq, H, D], k and v [B, Lk, H, D], float32 / float16 / bfloat16 on one GPU, D <= 128 (any strides; copied where the last dim is not
    contiguous or rows do not start on 16 bytes).  table [num_buckets, H]: the weight of the bias embedding, of any float type (used in fp32; numbers of
    up to 1e38 or -infinity).  Scores and their rows' logarithms are fp32 numbers: a probability in the backward pass is off by up to 2^-18 of the row's
    largest score, relative, so a table is no place for masks by large negative numbers where a row may hold nothing else.
    key_mask [B, Lk] bool or uint8: False hides a key from every query.  A query that sees no key gets zeros.  Keys that no query sees may hold
    anything; those that some query sees hold finite numbers.
    causal: keys behind a query's position are hidden and all buckets serve the distances back.  q_start: position of the first query among the
    keys, one number or one int32 / int64 [B] tensor -- a decoder's next token over a cache of n keys sits at n - 1.
    max_distance: distances from there on share the last bucket (at most 1023 may be told apart).  scale: 1 as the T5 family has it.
    """
    dev = _native.op_device(q, k, v, table, key_mask, q_start if torch.is_tensor(q_start) else None)
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"expected q [B, Lq, H, D] and k, v [B, Lk, H, D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, Lq, H, D = q.shape
    if k.shape[0] != B or k.shape[2] != H or k.shape[3] != D:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in batch, heads or head size")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f"q, k and v must share a type, got {q.dtype}, {k.dtype}, {v.dtype}")
    _native.op_dtype(q)
    if not 1 <= D <= 128:
        raise ValueError(f"head sizes 1 to 128, got {D}")
    if table.dim() != 2 or table.shape[1] != H or not table.is_floating_point():
        raise ValueError(f"expected a float table [num_buckets, {H}], got {table.dtype} {tuple(table.shape)}")
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8) or key_mask.shape != (B, k.shape[1]):
            raise ValueError(f"expected a bool or uint8 key_mask [{B}, {k.shape[1]}], got {key_mask.dtype} {tuple(key_mask.shape)}")
        if key_mask.stride(1) != 1 and key_mask.size(1) > 1:
            key_mask = key_mask.contiguous()
    if torch.is_tensor(q_start):
        if q_start.dtype not in (torch.int32, torch.int64) or q_start.shape != (B,):
            raise ValueError(f"expected an int32 or int64 q_start [{B}], got {q_start.dtype} {tuple(q_start.shape)}")
        q_start = q_start.clamp(-2 ** 30, 2 ** 30).to(torch.int32) if q_start.dtype == torch.int64 else q_start.contiguous()
    elif not -2 ** 30 <= q_start <= 2 ** 30:
        raise ValueError(f"q_start {q_start} is out of range")
    borders = _borders(table.shape[0], bool(causal), int(max_distance))
    if table.dtype != torch.float32 or not table.is_contiguous():
        table = table.float().contiguous()
    pad = -D % 8
    if pad:
        q, k, v = (torch.nn.functional.pad(x, (0, pad)) for x in (q, k, v))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or table.requires_grad):
        out = _Attention.apply(q, k, v, table, key_mask, q_start, bool(causal), borders, float(scale))
    else:
        out = _forward(q, k, v, table, key_mask, q_start, bool(causal), borders, float(scale), False)[0]
    return out[..., :D] if pad else out
