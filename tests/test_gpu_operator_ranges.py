"""GPU tests of the attention's gradients and outputs over the range of fp16's exponents: values that are large, probabilities that are small, keys that
no query sees.  Held to the formula in 64 bits.

Bounds: u is half a step of the type, f the 64 half steps of fp32 times 1 + the largest score that tests/helpers/operator_refs.py allows what stays in
fp32.  P and dS are rounded to the type on their way into a product, each column of them (a query's for dQ, a key's for dK and dV) under a power of two of
its own that puts its largest entry at 2^6 or more: entries in fp16's smallest numbers, whose half step is 2^-25, are off by at most 2^-31 of
the column's largest.  No entry is allowed an absolute error; results alone are, half of fp16's smallest step."""
import math

import pytest
import torch

from helpers.operator_refs import U32, bucket_of, check, half_step

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _reference(q, k, v, table, dout, causal=False, scale=1.0, start=0):
    """{name: (value, bound)} of out, dq, dk and dv in 64 bits; no masks.  Heads first inside."""
    dt = q.dtype
    u, small = half_step(dt), 2.0 ** -31 if dt == torch.float16 else 0.0
    tiny = 2.0 ** -25 if dt == torch.float16 else 1e-37
    t = lambda x: x.transpose(-1, -2).contiguous()   # noqa: E731
    qd, kd, vd, g = (x.detach().double().transpose(1, 2).contiguous() for x in (q, k, v, dout))
    Lq, Lk = qd.shape[2], kd.shape[2]
    rel = torch.arange(Lk, device=q.device)[None] - torch.arange(Lq, device=q.device)[:, None] - start
    lut = torch.tensor([bucket_of(d, table.shape[0], causal, 128) for d in range(-start - Lq, Lk + 1)], device=q.device)
    S = scale * (qd @ t(kd)) + table.double()[lut[rel + start + Lq]].permute(2, 0, 1)
    if causal:
        S = S.masked_fill(rel > 0, -math.inf)
    P = torch.softmax(S, 3)
    f = 64 * U32 * (1 + float(S[torch.isfinite(S)].abs().max()))
    out, dP = P @ vd, g @ t(vd)
    D = (P * dP).sum(3, keepdim=True)
    dS = P * (dP - D)
    twice = 0.0 if dt == torch.float32 else 2 * u * u                     # D: from P in two parts and an output kept in two parts
    eD = (twice + f) * (g.abs() * (P @ vd.abs())).sum(3, keepdim=True)
    if dt == torch.float16:                                               # ... whose second parts may lie in the smallest numbers
        eD = eD + 2 * (g.abs() * (2.0 ** -25 + 2.0 ** -31 * vd.abs().sum(2, keepdim=True))).sum(3, keepdim=True)
    raw = f * P * (g.abs() @ t(vd.abs()) + D.abs()) + P * eD
    e_q = raw + u * dS.abs() + small * (dS.abs() + raw).amax(3, keepdim=True)
    e_k = raw + u * dS.abs() + small * (dS.abs() + raw).amax(2, keepdim=True)
    e_p = (u + f) * P + small * P.amax(2, keepdim=True)
    dq, dk, dv = scale * (dS @ kd), scale * (t(dS) @ qd), t(P) @ g
    back = lambda x: x.transpose(1, 2)   # noqa: E731
    return {"out": (back(out), back((u + small) * out.abs() + (u + f + small) * (P @ vd.abs()) + tiny)),
            "dq": (back(dq), back(u * dq.abs() + scale * (e_q @ kd.abs() + f * (dS.abs() @ kd.abs())) + tiny)),
            "dk": (back(dk), back(u * dk.abs() + scale * (t(e_k) @ qd.abs() + f * (t(dS.abs()) @ qd.abs())) + tiny)),
            "dv": (back(dv), back(u * dv.abs() + t(e_p) @ g.abs() + tiny))}


def _run(q, k, v, table, dout, **kw):
    from mfar.modeling.attention import relative_bias_attention
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v, table)]
    out = relative_bias_attention(*leaves, **kw)
    return dict(zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(), *torch.autograd.grad(out, leaves, dout))))


def _hold(q, k, v, table, dout, **kw):
    got = _run(q, k, v, table, dout, causal=kw.get("causal", False), scale=kw.get("scale", 1.0), q_start=kw.get("start", 0))
    for name, (want, bound) in _reference(q, k, v, table, dout, **kw).items():
        check(name, got[name], want, bound)
    return got


@pytest.mark.parametrize("D", [40, 64, 128])
@pytest.mark.parametrize("size", [2000.0, 60000.0])
def test_fp16_gradients_under_large_values(D, size):
    """Two equally likely keys with values of opposite sign and a small gradient along them: dP is D times value times gradient, past fp16's largest number
    once dO alone is brought near 1, while every gradient is an ordinary number."""
    L, H = 2, 3
    q, k = torch.zeros(1, L, H, D, device="cuda"), torch.full((1, L, H, D), 0.01, device="cuda")
    q[..., 0] = 0.25
    k[:, 1] *= -1
    k[..., 0] = 0.0                                                       # equal scores
    v = torch.full((1, L, H, D), size, device="cuda")
    v[:, 1] *= -1
    dout = torch.full((1, L, H, D), 2.0 / size, device="cuda")
    x = [y.half() for y in (q, k, v)]
    got = _hold(*x, torch.zeros(32, H, device="cuda"), dout.half())
    assert all(bool(got[n].isfinite().all()) for n in got)
    assert float(got["dq"].abs().max()) > 0.1 and float(got["dk"].abs().max()) > 1


@pytest.mark.parametrize("B,Lq,Lk", [(2, 150, 150), (1, 300, 70), (1, 33, 200)])
def test_fp16_gradients_of_rows_that_differ_in_size(B, Lq, Lk):
    """Gradients from 2^-14 to 2^14 from query to query and values from 2^-10 to 2^10 from key to key, in any order along the tiles: every query's dQ and
    every key's dK is held to its own size."""
    H, D = 2, 64
    g = _gen(31)
    q = torch.randn(B, Lq, H, D, generator=g, device="cuda") * (1.0 / math.sqrt(D))
    k, v, dout = (torch.randn(B, n, H, D, generator=g, device="cuda") for n in (Lk, Lk, Lq))
    v = v * torch.exp2(torch.rand(B, Lk, H, 1, generator=g, device="cuda") * 20 - 10)
    dout = dout * torch.exp2(torch.rand(B, Lq, H, 1, generator=g, device="cuda") * 28 - 14)
    dout = dout * 2.0 ** -6                                               # (nothing past the type in the results themselves)
    table = torch.randn(32, H, generator=g, device="cuda")
    _hold(*(x.half() for x in (q, k * 0.05, v * 2.0 ** -4)), table, dout.half(), scale=20.0)


@pytest.mark.parametrize("bias", [-8.0, -10.0, -12.0, -16.0, -30.0])
@pytest.mark.parametrize("B,L,D", [(1, 512, 64), (1, 300, 128), (40, 200, 64)])
def test_fp16_gradients_of_keys_with_small_probabilities(bias, B, L, D):
    """Keys behind a learned bias that all but hides them still get gradients as exact as the type: P and dS of such a key are all small, none of them large
    beside them.  dO is what a gradient scaler hands over (2^10 over a mean's)."""
    H = 2
    g = _gen(32)
    q = torch.randn(B, L, H, D, generator=g, device="cuda") * (1.0 / math.sqrt(D))
    k, v, dout = (torch.randn(B, L, H, D, generator=g, device="cuda") for _ in range(3))
    table = torch.randn(32, H, generator=g, device="cuda")
    table[16:] += bias                                                    # every key past the query, from near ones to the last bucket
    x = [y.half() for y in (q, k, v, dout * 2.0 ** 10)]
    x[3][:, L // 2:] = 0.0                                                # (the second half's queries count for nothing: its keys are seen through the bias only)
    got = _hold(x[0], x[1], x[2], table, x[3])
    want = _reference(x[0], x[1], x[2], table, x[3])
    # ... and by norm: a row of dV is a sum of products whose operands are rounded once, so it is off by well under a step of the type, as far as fp16 can
    # show the result at all
    for name in ("dk", "dv"):
        w = want[name][0][:, L // 2:].transpose(1, 2)
        e = (got[name].double()[:, L // 2:].transpose(1, 2) - w).norm(dim=-1)
        assert bool((e <= 4 * half_step(torch.float16) * w.norm(dim=-1) + math.sqrt(D) * 2.0 ** -25).all()), (name, float((e / w.norm(dim=-1)).max()))


def test_fp16_gradients_of_a_long_uniform_attention():
    """Probabilities of 1 / 40000, under fp16's smallest normal number."""
    H, D, Lq, Lk = 1, 32, 40, 40000
    g = _gen(33)
    q = torch.randn(1, Lq, H, D, generator=g, device="cuda") * 0.01
    k, v = (torch.randn(1, Lk, H, D, generator=g, device="cuda") for _ in range(2))
    dout = torch.randn(1, Lq, H, D, generator=g, device="cuda") * 2.0 ** 12
    _hold(*(x.half() for x in (q, k, v)), torch.zeros(32, H, device="cuda"), dout.half())


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("Lq,Lk,start", [(40, 100, 0), (130, 300, 20), (70, 129, 58), (3, 200, 60)])
def test_keys_past_every_query_may_hold_anything(dtype, Lq, Lk, start):
    """Causal: what lies behind the last query's position reaches nothing, and gets zero gradients."""
    B, H, D = 2, 2, 64
    g = _gen(34)
    q = (torch.randn(B, Lq, H, D, generator=g, device="cuda") * 0.2).to(TYPES[dtype])
    k, v = (torch.randn(B, Lk, H, D, generator=g, device="cuda").to(TYPES[dtype]) for _ in range(2))
    dout = torch.randn(B, Lq, H, D, generator=g, device="cuda").to(TYPES[dtype])
    table = torch.randn(32, H, generator=g, device="cuda")
    end = start + Lq
    k[:, end:], v[:, end:] = 0.0, 0.0
    want = _run(q, k, v, table, dout, causal=True, q_start=start)
    k[:, end:], v[:, end:] = float("nan"), float("inf")
    got = _run(q, k, v, table, dout, causal=True, q_start=start)
    assert all(torch.equal(got[n], want[n]) for n in got)
    assert not got["dk"][:, end:].any() and not got["dv"][:, end:].any() and bool(got["dk"].isfinite().all())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("B,Lq", [(4, 9), (140, 130)])
def test_outputs_of_a_query_with_one_key_ahead_of_the_rest(dtype, B, Lq):
    """Two visible keys a tile apart, the second 2^4 to 2^7.9 times as likely as the first, which set the softmax's base.  Probabilities are multiplied as the type
    holds them (p1', p2') and divided by the sum of just those, so with w = p2' / (p1' + p2') the roundings of both all but cancel: w is off by at
    most 2 u w (1 - w), and the output beside that by its own rounding."""
    H, D, Lk = 2, 64, 160
    u = half_step(TYPES[dtype])
    g = _gen(35)
    mask = torch.zeros(B, Lk, dtype=torch.bool, device="cuda")
    mask[:, 3], mask[:, 140] = True, True
    q, k = torch.zeros(B, Lq, H, D, device="cuda"), torch.zeros(B, Lk, H, D, device="cuda")
    q[..., 0] = (torch.rand(B, Lq, H, generator=g, device="cuda") * 3.9 + 4) * math.log(2)
    k[:, 140, :, 0] = 1.0
    v = torch.randn(B, Lk, H, D, generator=g, device="cuda")
    q, k, v = (x.to(TYPES[dtype]) for x in (q, k, v))
    from mfar.modeling.attention import relative_bias_attention
    with torch.no_grad():
        got = relative_bias_attention(q, k, v, torch.zeros(32, H, device="cuda"), key_mask=mask).double()
    w = torch.sigmoid(q[..., :1].double())                               # of the second key
    a, b = v[:, 3].double()[:, None], v[:, 140].double()[:, None]
    want = a + w * (b - a)
    f = 64 * U32 * 7
    check("out", got, want, u * want.abs() * (1 + 4 * u) + (2 * u * (1 + 4 * u) * w * (1 - w) + f) * (a.abs() + b.abs()) + (2.0 ** -25 if dtype == "fp16" else 0.0))


@pytest.mark.parametrize("dtype,D", [("fp32", 64), ("fp32", 128), ("fp16", 128), ("bf16", 64)])
@pytest.mark.parametrize("causal", [False, True])
def test_large_batches_over_more_than_4096_keys(dtype, D, causal):
    """The kernels of large batches across a group of 4096 keys, forward and backward, in fp32 and wide heads too, where LDS holds one step of tiles alone: keys
    hidden on either side of the border, up to it, behind it, and all of a group."""
    from helpers.operator_refs import attention_ref
    B, H, Lq, Lk = 64, 2, 35, 4230
    print(f"attention {dtype} {D} {causal}", flush=True)
    g = _gen(36)
    q = (torch.randn(B, Lq, H, D, generator=g, device="cuda") * (1.5 / math.sqrt(D))).to(TYPES[dtype])
    k, v = (torch.randn(B, Lk, H, D, generator=g, device="cuda").to(TYPES[dtype]) for _ in range(2))
    dout = torch.randn(B, Lq, H, D, generator=g, device="cuda").to(TYPES[dtype])
    table = torch.randn(32, H, generator=g, device="cuda")
    mask = torch.rand(B, Lk, generator=g, device="cuda") < 0.7
    mask[0] = True
    mask[1, 4096:], mask[2, :4096], mask[3, 4095:4097] = False, False, False
    mask[4], mask[5, :] = False, False
    mask[5, 4096] = True
    mask[6, 4090:], mask[6, 4100] = False, True
    start = Lk - Lq - 3 if causal else 0
    got = _run(q, k, v, table, dout, key_mask=mask, causal=causal, q_start=start)
    for name, (want, bound) in attention_ref(q, k, v, table, mask, causal, 128, start, 1.0, dout).items():
        check(name, got[name], want, bound)
    assert not got["out"][4].any() and not got["dk"][4].any()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("B,Lq,Lk,causal", [(1, 12, 12, False), (5, 1, 4097, True), (3, 31, 300, False), (2, 200, 200, False)])
def test_outputs_of_few_queries_are_rounded_once(dtype, B, Lq, Lk, causal):
    """Short texts, single tokens over a cache and small batches: P is multiplied in two parts of the type (u^2 each), so an output is off by its own rounding and
    what fp32 leaves, element by element, however much of P|V| cancels in it."""
    from helpers.operator_refs import attention_ref
    from mfar.modeling.attention import relative_bias_attention
    H, D = 3, 64
    g = _gen(37)
    q = (torch.randn(B, Lq, H, D, generator=g, device="cuda") * (1.5 / math.sqrt(D))).to(TYPES[dtype])
    k, v = (torch.randn(B, Lk, H, D, generator=g, device="cuda").to(TYPES[dtype]) for _ in range(2))
    table = torch.randn(32, H, generator=g, device="cuda")
    start = Lk - Lq if causal else 0
    with torch.no_grad():
        got = relative_bias_attention(q, k, v, table, causal=causal, q_start=start)
    u = half_step(TYPES[dtype])
    want, loose = attention_ref(q, k, v, table, None, causal, 128, start, 1.0)["out"]
    # P|V| from above: `loose` holds it at least u times; scores are under 9, fp16's two parts miss 2^-31 of the largest P at most
    f = (4 * u * u + 64 * 10 * U32) * loose / u
    check("out", got, want, u * want.abs() + f + (2.0 ** -24 if dtype == "fp16" else 0.0))
