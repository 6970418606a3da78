"""The encoder / training operators from their definitions in 64 bits, and how far a kernel may be from them.

Bounds: u is half a step of the outputs' type (a rounding's largest relative error).  The kernels round the probabilities P and the score gradients
dS to the inputs' type before the second product, and every output once: u times the product of absolute values for each.  What stays in fp32
(scores, exponentials, sums) is allowed 64 half steps of fp32, times 1 + the largest score for what passes through exp."""
import math

import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def bucket_of(d, num_buckets, causal, max_distance):
    """One distance's bucket, in whole numbers, border by border."""
    side = num_buckets if causal else num_buckets // 2
    each, far = side // 2, (max(0, -d) if causal else abs(d))
    b = far
    if far >= each:
        n, b = side - each, each
        while b < side - 1 and far ** n >= max_distance ** (b + 1 - each) * each ** (n - (b + 1 - each)):
            b += 1
    return b + (side if d > 0 and not causal else 0)


def attention_ref(q, k, v, table, key_mask, causal, max_distance, start, scale, dout=None):
    """{name: (value, bound)} of out and, with dout, the gradients; float64, on the tensors' device."""
    dt = q.dtype
    u = half_step(dt)
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0                   # half a step of fp16's smallest numbers
    qd, kd, vd = (x.detach().double().transpose(1, 2).contiguous() for x in (q, k, v))
    td = table.detach().double()
    B, H, Lq, D = qd.shape
    Lk, dev = kd.shape[2], q.device
    st = start.to(torch.int64) if torch.is_tensor(start) else torch.full((B,), int(start), device=dev)
    rel = torch.arange(Lk, device=dev)[None, None, :] - (st[:, None] + torch.arange(Lq, device=dev)[None, :])[:, :, None]
    lo, hi = (int(rel.min()), int(rel.max())) if rel.numel() else (0, 0)
    lut = torch.tensor([bucket_of(d, table.shape[0], causal, max_distance) for d in range(lo, hi + 1)], device=dev)
    at = lut[rel - lo]                                                   # [B, Lq, Lk]
    seen = torch.ones(B, Lq, Lk, dtype=torch.bool, device=dev)
    if causal:
        seen &= rel <= 0
    if key_mask is not None:
        seen &= key_mask.bool()[:, None, :]
        hide = ~key_mask.bool()[:, None, :, None]
        kd, vd = kd.masked_fill(hide, 0.0), vd.masked_fill(hide, 0.0)    # hidden keys may hold anything
    seen = seen[:, None]
    S = scale * (qd @ kd.transpose(2, 3).contiguous()) + td[at].permute(0, 3, 1, 2)
    S = S.masked_fill(~seen, -math.inf)
    P = torch.nan_to_num(torch.softmax(S, 3)) if Lk else S
    out = P @ vd
    big = 1.0 + (float(S[seen.expand_as(S)].abs().max()) if bool(seen.any()) else 0.0)
    f = 64 * U32 * big
    back = lambda x: x.transpose(1, 2)   # noqa: E731
    res = {"out": (back(out), back((u + tiny) * out.abs() + (u + f) * (P @ vd.abs()) + tiny * (1 + vd.abs().sum(2, keepdim=True))))}
    if dout is None:
        return res
    g = dout.detach().double().transpose(1, 2).contiguous()
    dP = g @ vd.transpose(2, 3).contiguous()
    Dr = (P * dP).sum(3, keepdim=True)
    dS = P * (dP - Dr)
    # what dS may be off before its rounding: fp32 throughout, and D = <dO, O> from an O whose P was kept in two parts of the type (each p is
    # off by u of what its first rounding dropped, u p, so u^2 p, and O by u^2 P|V|) and which is itself kept in two parts (u^2 |O| <= u^2 P|V|)
    kept = 0.0 if dt == torch.float32 else 2 * u * u
    eD = (kept + f) * (g.abs() * (P @ vd.abs())).sum(3, keepdim=True) + 2 * tiny * (g.abs() * (1 + vd.abs().sum(2, keepdim=True))).sum(3, keepdim=True)
    raw = f * P * (g.abs() @ vd.abs().transpose(2, 3).contiguous() + Dr.abs()) + P * eD
    eS = raw + u * dS.abs() + tiny
    dq, dk, dv = scale * (dS @ kd), scale * (dS.transpose(2, 3).contiguous() @ qd), P.transpose(2, 3).contiguous() @ g
    res["dq"] = (back(dq), back(u * dq.abs() + scale * (eS @ kd.abs()) + f * scale * (dS.abs() @ kd.abs()) + tiny))
    res["dk"] = (back(dk), back(u * dk.abs() + scale * (eS.transpose(2, 3).contiguous() @ qd.abs()) + f * scale * (dS.abs().transpose(2, 3).contiguous() @ qd.abs()) + tiny))
    res["dv"] = (back(dv), back(u * dv.abs() + (((u + f) * P + tiny).transpose(2, 3).contiguous() @ g.abs()) + tiny))
    def summed(x):                                                       # [buckets, H]
        return torch.stack([torch.bincount(at.reshape(-1), weights=x.masked_fill(~seen, 0.0)[:, h].reshape(-1), minlength=table.shape[0]) for h in range(H)], 1)
    res["dtable"] = (summed(dS), summed(raw + f * dS.abs()) + 1e-30)
    return res


def check(name, got, want, bound):
    got = got.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    over = (got - want).abs() - bound
    bad = ~(over <= 0)
    if bool(bad.any()):
        i = int(torch.argmax(torch.nan_to_num(over, nan=math.inf).reshape(-1)))
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} values off; at flat place {i}: {float(got.reshape(-1)[i])} for "
                             f"{float(want.reshape(-1)[i])}, allowed {float(bound.expand_as(want).reshape(-1)[i])}")


def distillation_ref(x, ids, scores, tau, dloss):
    """(loss, its bound, gradient, its bound) in float64; no bad ids."""
    u = half_step(x.dtype)
    z = x.detach().double() / tau
    lse = torch.logsumexp(z, 1, keepdim=True)
    live = ids >= 0
    t = (scores.double() / tau).masked_fill(~live, -math.inf)
    p = torch.nan_to_num(torch.softmax(t, 1))
    logp = torch.where(p > 0, torch.log(p.clamp(min=1e-300)), torch.zeros_like(p))
    cols = ids.clamp(min=0).long()
    logq = torch.where(p > 0, z.gather(1, cols) - lse, torch.zeros_like(p))
    loss = tau * tau * (p * (logp - logq)).sum(1)
    finite = torch.where(torch.isfinite(z), z.abs(), torch.zeros_like(z)).amax(1)
    f = 64 * U32 * (1 + finite + torch.where(live, (scores.double() / tau).abs(), torch.zeros_like(p)).amax(1))
    e_loss = tau * tau * f * (1 + (p * (logp.abs() + logq.abs())).sum(1))
    q = torch.exp(z - lse) * (p.sum(1, keepdim=True) > 0.5)
    pj = torch.zeros_like(z).scatter_add_(1, cols, p)
    g = (tau * dloss.double())[:, None]
    d = g * (q - pj)
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 1e-37
    return loss, e_loss, d, u * d.abs() + f[:, None] * g.abs() * (q + pj) + tiny
