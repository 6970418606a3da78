"""GPU tests of the encoder / training operators (include/mfar_hip.h, last section) against their definitions in 64 bits
(tests/helpers/operator_refs.py, which also derives the tolerances)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _attention_inputs(seed, B, Lq, Lk, H, D, dtype, nb=32):
    g = _gen(seed)
    mk = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    q = (mk(B, Lq, H, D) * (1.5 / math.sqrt(D))).to(TYPES[dtype])
    return q, mk(B, Lk, H, D).to(TYPES[dtype]), mk(B, Lk, H, D).to(TYPES[dtype]), mk(nb, H), mk(B, Lq, H, D).to(TYPES[dtype])


def _run_attention(q, k, v, table, dout=None, **kw):
    from mfar.modeling.attention import relative_bias_attention
    if dout is None:
        return {"out": relative_bias_attention(q, k, v, table, **kw)}
    leaves = [x.detach().clone().requires_grad_(True) if x.is_contiguous() else x.detach().requires_grad_(True) for x in (q, k, v, table)]
    out = relative_bias_attention(*leaves, **kw)
    grads = torch.autograd.grad(out, leaves, dout)
    return dict(zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(), *grads)))


def _check_attention(q, k, v, table, dout, mask=None, causal=False, max_distance=128, start=0, scale=1.0):
    from helpers.operator_refs import attention_ref, check
    got = _run_attention(q, k, v, table, dout, key_mask=mask, causal=causal, max_distance=max_distance, q_start=start, scale=scale)
    want = attention_ref(q, k, v, table, mask, causal, max_distance, start, scale, dout)
    for name, (w, b) in want.items():
        check(name, got[name], w, b)
    serving = _run_attention(q, k, v, table, key_mask=mask, causal=causal, max_distance=max_distance, q_start=start, scale=scale)["out"]
    check("out without gradients", serving, *want["out"])
    return got


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("B,Lq,Lk,H,D,causal", [
    (1, 1, 1, 1, 64, False), (2, 12, 12, 3, 64, False), (1, 33, 33, 2, 32, True), (2, 64, 64, 2, 128, False), (1, 65, 129, 2, 16, False),
    (1, 130, 257, 2, 64, False), (2, 200, 200, 2, 40, True), (1, 513, 513, 1, 64, False), (1, 300, 300, 2, 128, True), (1, 5, 700, 2, 64, False),
])
def test_attention_and_gradients(dtype, B, Lq, Lk, H, D, causal):
    print(f"attention {dtype} {B} {Lq} {Lk} {H} {D} {causal}", flush=True)
    q, k, v, table, dout = _attention_inputs(1, B, Lq, Lk, H, D, dtype)
    _check_attention(q, k, v, table, dout, causal=causal)


@pytest.mark.parametrize("D", [1, 7, 33, 100])
def test_attention_head_sizes_that_fill_no_chunk(D):
    q, k, v, table, dout = _attention_inputs(2, 2, 40, 40, 2, D, "fp16")
    _check_attention(q, k, v, table, dout)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("B,Lq,Lk,H,D,causal", [(130, 150, 150, 1, 64, False), (40, 213, 213, 4, 40, True), (3, 300, 200, 40, 128, False), (270, 40, 70, 1, 32, True),
                                                (1, 8200, 4300, 4, 64, False)])
def test_attention_of_batches_that_fill_the_gpu(dtype, B, Lq, Lk, H, D, causal):
    """256 blocks of 128 queries and more: the kernel of large batches, forward and backward, with ragged key masks and over 4096 keys."""
    print(f"attention {dtype} {B} {Lq} {Lk} {H} {D} {causal}", flush=True)
    if dtype == "fp32" and Lk > 4096:
        pytest.skip("the 64-bit reference of 4 x 8200 x 4300 is made for two types only")
    q, k, v, table, dout = _attention_inputs(17, B, Lq, Lk, H, D, dtype)
    lens = torch.randint(0, Lk + 1, (B,), generator=_gen(18), device="cuda")
    lens[0] = Lk
    mask = torch.arange(Lk, device="cuda") < lens[:, None]
    if not causal:
        mask[:, 5] = False
    _check_attention(q, k, v, table, dout, mask=mask, causal=causal)
    if Lk <= 4096:
        _check_attention(q, k, v, table, dout, causal=causal, start=3)
    k2, v2 = k.clone(), v.clone()
    k2[~mask], v2[~mask] = float("nan"), float("inf")
    a = _run_attention(q, k, v, table, dout, key_mask=mask, causal=causal)
    b = _run_attention(q, k2, v2, table, dout, key_mask=mask, causal=causal)
    assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("B", [5, 300])
def test_attention_layouts_give_the_same_bits_in_large_batches(B):
    L, H, D = 70, 3, 32
    q, k, v, table, dout = _attention_inputs(19, B, L, L, H, D, "bf16")
    want = _run_attention(q, k, v, table, dout)
    packed = torch.stack([q, k, v], dim=2)
    got = _run_attention(packed[:, :, 0], packed[:, :, 1], packed[:, :, 2], table, dout)
    heads = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    got2 = _run_attention(*heads, table, dout.transpose(1, 2).contiguous().transpose(1, 2))
    mask = torch.rand(B, L, generator=_gen(20), device="cuda") < 0.6
    shifted = torch.zeros(B, L + 3, dtype=torch.bool, device="cuda")
    shifted[:, 3:] = mask                                                  # rows that start on no particular byte
    m1, m2 = _run_attention(q, k, v, table, dout, key_mask=mask), _run_attention(q, k, v, table, dout, key_mask=shifted[:, 3:])
    for a, b in ((want, got), (want, got2), (m1, m2)):
        assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_attention_masks_holes_empty_rows_and_poison(dtype):
    """Right-padded, scattered, fully hidden and single-key masks; hidden keys hold NaN, infinities and the type's lowest value."""
    B, L, H, D = 5, 150, 2, 64
    q, k, v, table, dout = _attention_inputs(3, B, L, L, H, D, dtype)
    mask = torch.ones(B, L, dtype=torch.bool, device="cuda")
    mask[0, 70:] = False
    mask[1] = torch.rand(L, generator=_gen(4), device="cuda") < 0.3
    mask[2] = False
    mask[3] = False
    mask[3, 64] = True
    got = _check_attention(q, k, v, table, dout, mask=mask)
    assert not got["out"][2].any() and not got["dq"][2].any() and not got["dk"][2].any() and not got["dv"][2].any()
    k2, v2 = k.clone(), v.clone()
    for x in (k2, v2):
        x[~mask] = float("nan")
        x[0, 100:] = float("inf")
        x[2, :50] = torch.finfo(x.dtype).min
    again = _run_attention(q, k2, v2, table, dout, key_mask=mask)
    for n in got:
        assert torch.equal(got[n], again[n]), n
    as_bytes = _run_attention(q, k, v, table, dout, key_mask=mask.to(torch.uint8) * 3)
    assert all(torch.equal(got[n], as_bytes[n]) for n in got)
    wide = torch.zeros(B, 2 * L, dtype=torch.bool, device="cuda")          # a mask whose rows and elements lie apart
    wide[:, ::2] = mask
    strided = _run_attention(q, k, v, table, dout, key_mask=wide[:, ::2])
    assert all(torch.equal(got[n], strided[n]) for n in got)


def test_attention_causal_rows_before_the_first_key_and_masks():
    B, L, H, D = 3, 90, 2, 32
    q, k, v, table, dout = _attention_inputs(5, B, L, L, H, D, "bf16")
    mask = torch.ones(B, L, dtype=torch.bool, device="cuda")
    mask[1, :40] = False                                                 # left padding: the first 40 queries see nothing
    got = _check_attention(q, k, v, table, dout, mask=mask, causal=True)
    assert not got["out"][1, :40].any()
    _check_attention(q, k, v, table, dout, causal=True, start=-10)        # queries before the first key


@pytest.mark.parametrize("Lk,Lq", [(1, 1), (31, 1), (64, 1), (1000, 1), (4097, 1), (517, 3)])
def test_attention_single_tokens_over_caches(Lk, Lq):
    """A decoder's next token(s): every sequence at its own place, what lies behind it in the cache not initialised."""
    B, H, D = 4, 3, 64
    q, k, v, table, _ = _attention_inputs(6, B, Lq, Lk, H, D, "fp16")
    lens = torch.tensor([Lk, max(Lq, Lk // 2), max(Lq, Lk - 1), Lq], device="cuda")
    start = (lens - Lq).to(torch.int32)
    from helpers.operator_refs import attention_ref, check
    dead = torch.arange(Lk, device="cuda")[None] >= lens[:, None]
    kz, vz = k.masked_fill(dead[..., None, None], 0.0), v.masked_fill(dead[..., None, None], 0.0)
    want = attention_ref(q, kz, vz, table, None, True, 128, start, 1.0)["out"]
    for x in (k, v):
        x[dead] = float("nan")
    check("out", _run_attention(q, k, v, table, causal=True, q_start=start)["out"], *want)
    check("out", _run_attention(q, k, v, table, causal=True, q_start=start.long())["out"], *want)
    cache = torch.stack([k.transpose(1, 2), v.transpose(1, 2)]).contiguous()       # [2, B, H, Lk, D]
    kc, vc = cache[0].transpose(1, 2), cache[1].transpose(1, 2)
    check("out", _run_attention(q, kc, vc, table, causal=True, q_start=start)["out"], *want)


def test_attention_layouts_and_strides():
    """Packed projections, heads first, odd offsets, an expanded batch and an expanded gradient give the contiguous call's bits."""
    B, L, H, D = 2, 70, 3, 32
    q, k, v, table, dout = _attention_inputs(7, B, L, L, H, D, "fp16")
    want = _run_attention(q, k, v, table, dout)
    packed = torch.stack([q, k, v], dim=2)                                         # [B, L, 3, H, D]
    got = _run_attention(packed[:, :, 0], packed[:, :, 1], packed[:, :, 2], table, dout)
    heads = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    got2 = _run_attention(*heads, table, dout.transpose(1, 2).contiguous().transpose(1, 2))
    odd = []
    for x in (q, k, v):
        y = torch.empty(x.numel() + 3, dtype=x.dtype, device="cuda")[3:].view_as(x)
        odd.append(y.copy_(x))
    got3 = _run_attention(*odd, table, dout)
    last = [torch.empty(B, L, D, H, dtype=x.dtype, device="cuda").copy_(x.transpose(2, 3)).transpose(2, 3) for x in (q, k, v)]
    got4 = _run_attention(*last, table, dout)
    for other in (got, got2, got3, got4):
        assert all(torch.equal(want[n], other[n]) for n in want)
    one = q[:1].expand(B, L, H, D).detach().requires_grad_(True)
    from mfar.modeling.attention import relative_bias_attention
    leaf = k[:1].detach().clone().requires_grad_(True)
    out = relative_bias_attention(one, leaf.expand(B, L, H, D), v, table)
    (gk,) = torch.autograd.grad(out.sum(), [leaf])                                  # the gradient of sum() is an expanded scalar
    ref = _run_attention(q[:1].expand(B, L, H, D).contiguous(), k[:1].expand(B, L, H, D).contiguous(), v, table, torch.ones_like(dout))
    assert torch.equal(out.detach(), ref["out"])
    assert torch.allclose(gk[0].float(), ref["dk"].float().sum(0), rtol=2 ** -10, atol=1e-3)      # one more rounding of a sum of two


@pytest.mark.parametrize("nb,max_distance,causal", [(32, 128, False), (4, 3, False), (2, 9, True), (8, 20, True), (64, 1000, False), (255, 1000, True)])
def test_attention_bucket_layouts(nb, max_distance, causal):
    q, k, v, table, dout = _attention_inputs(8, 1, 260, 260, 2, 32, "fp32", nb)
    _check_attention(q, k, v, table, dout, causal=causal, max_distance=max_distance, scale=0.5)


def test_attention_largest_table_and_heads():
    q, k, v, table, dout = _attention_inputs(14, 1, 140, 140, 1, 128, "fp32", 255)
    _check_attention(q, k, v, table, dout, causal=True, max_distance=1020)


def test_attention_gradients_against_differences():
    """Directional derivatives in fp32: the loss's difference quotient along a random direction of every input."""
    from mfar.modeling.attention import relative_bias_attention
    q, k, v, table, dout = _attention_inputs(9, 1, 37, 37, 2, 32, "fp32")
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v, table)]
    grads = torch.autograd.grad(relative_bias_attention(*leaves, causal=False), leaves, dout)
    f = lambda xs: float((relative_bias_attention(*xs).double() * dout.double()).sum())   # noqa: E731
    for i, x in enumerate((q, k, v, table)):
        d = torch.randn(x.shape, generator=_gen(20 + i), device="cuda")
        h = 2.0 ** -6 / float(d.abs().max())
        xs = [q, k, v, table]
        vals = []
        for s in (2, 1, -1, -2):
            ys = list(xs)
            ys[i] = x + s * h * d
            vals.append(f(ys))
        quotient = (-vals[0] + 8 * vals[1] - 8 * vals[2] + vals[3]) / (12 * h)        # error h^4
        along = float((grads[i].double() * d.double()).sum())
        size = float(grads[i].double().norm() * d.double().norm())
        assert abs(quotient - along) < 1e-3 * size, (i, quotient, along, size)


@pytest.mark.parametrize("size", [2.0 ** -10, 2.0 ** 8])
def test_attention_gradients_of_small_and_large_losses(size):
    """A power of two on dout is a power of two on every gradient, fp16's own rounding apart: the score gradients of a small loss do not drown in fp16's
    smallest numbers, those of a large one do not overflow on the way.  (2^-10: dS near 2^-17, of which fp16 by itself would keep 7 bits.)"""
    q, k, v, table, dout = _attention_inputs(15, 2, 150, 150, 2, 64, "fp16")
    dout = (dout.float().clamp(-4, 4) * 0.25).half()
    dout = torch.where(dout.abs() < 2.0 ** -4, dout.sign() * 2.0 ** -4, dout)          # exact after scaling: no subnormal numbers in dout itself
    one = _run_attention(q, k, v, table, (dout.float() * 2.0 ** -2).half())
    got = _run_attention(q, k, v, table, (dout.float() * size).half())
    f = size * 4
    assert torch.equal(got["dtable"], one["dtable"] * f)
    for n in ("dq", "dk", "dv"):
        a, b = got[n].double() / f, one[n].double()
        # one rounding each; what lies in fp16's smallest numbers is off by half their step
        tol = 2.0 ** -11 * (a.abs() + b.abs()) + 2.0 ** -25 / f + 2.0 ** -25
        assert bool(((a - b).abs() <= tol).all()), n


@pytest.mark.parametrize("dtype,B,Lq", [("fp16", 32, 300), ("bf16", 32, 300), ("fp16", 8, 300), ("fp16", 200, 20)])
def test_attention_output_is_kept_to_twice_its_type(dtype, B, Lq):
    """What the forward pass leaves for the backward one: out and what its rounding dropped, together as exact as P in two parts makes them (u^2 of P|V|,
    fp32 elsewhere) -- for every single element."""
    from helpers.operator_refs import U32, attention_ref, half_step
    from mfar.modeling.attention import _borders, _forward
    q, k, v, table, _ = _attention_inputs(16, B, Lq, 24, 3, 64, dtype)          # few keys: an output is not much smaller than P|V|
    out, lo, lse, _ = _forward(q, k, v, table, None, 0, False, _borders(32, False, 128), 1.0, True)
    want, loose = attention_ref(q, k, v, table, None, False, 128, 0, 1.0)["out"]
    u = half_step(q.dtype)
    # the reference's bound without its two roundings to the type: 64 half steps of fp32 times 1 + the largest score (under 9 here), of P|V|, which
    # `loose` = u |out| + (u + f) P|V| + .. holds at least u times
    pv = loose / u
    tiny = 2.0 ** -24 if dtype == "fp16" else 0.0
    err = (out.double() + lo.double() - want).abs()
    assert bool((err <= (4 * u * u + 64 * 10 * U32) * pv + tiny).all()), float((err / pv).max())


def test_attention_is_reproducible_and_follows_the_current_stream():
    q, k, v, table, dout = _attention_inputs(10, 3, 300, 300, 4, 64, "bf16")
    a = _run_attention(q, k, v, table, dout)
    b = _run_attention(q, k, v, table, dout)
    assert all(torch.equal(a[n], b[n]) for n in a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = _run_attention(q, k, v, table, dout)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a[n], c[n]) for n in a)


def test_attention_captured_and_replayed():
    """Forward and backward in one graph, replayed between eager calls; two graphs do not share a workspace."""
    from mfar.modeling.attention import relative_bias_attention
    graphs = []
    for seed, L in ((11, 200), (12, 77)):
        q, k, v, table, dout = _attention_inputs(seed, 2, L, L, 2, 64, "fp16")
        leaves = [x.clone().requires_grad_(True) for x in (q, k, v, table)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(relative_bias_attention(*leaves), leaves, dout)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = relative_bias_attention(*leaves)
            grads = torch.autograd.grad(out, leaves, dout)
        graphs.append((g, leaves, dout, out.detach(), grads, seed, L))
    for turn in range(4):
        for g, leaves, dout, out, grads, seed, L in graphs:
            fresh = _attention_inputs(100 * turn + seed, 2, L, L, 2, 64, "fp16")
            with torch.no_grad():
                for x, y in zip(leaves, fresh[:4]):
                    x.copy_(y)
                dout.copy_(fresh[4])
        for g, *_ in graphs:
            g.replay()
        for g, leaves, dout, out, grads, seed, L in graphs:
            want = _run_attention(*[x.detach() for x in leaves], dout)
            assert torch.equal(out, want["out"]), turn
            assert all(torch.equal(a, want[n]) for a, n in zip(grads, ("dq", "dk", "dv", "dtable"))), turn


def test_attention_empty_sizes():
    for B, Lq, Lk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q, k, v, table, dout = _attention_inputs(13, B, Lq, Lk, 2, 32, "fp16")
        got = _run_attention(q, k, v, table, dout)
        assert got["out"].shape == q.shape and not got["out"].any()
        assert not any(got[n].any() for n in ("dq", "dk", "dv", "dtable"))


# ---- 8-bit linear -----------------------------------------------------------------------------------------------------------------------
def _quantize_ref(x):
    # the product and the quotient rounded to fp32 once: a quotient of two fp32 numbers in 64 bits, rounded to 32, is the correctly rounded one
    # (53 >= 2 * 24 + 2 bits)
    xd = x.double()
    s = (xd.abs().amax(-1, keepdim=True) * float(torch.tensor(1.0) / 127)).float()      # (exact in 64 bits, then rounded)
    n = (xd / torch.where(s > 0, s, torch.ones_like(s)).double()).float()
    return torch.round(n).clamp(-127, 127).to(torch.int8), s[..., 0]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (5, 64), (130, 768), (9, 1001), (2, 5000), (1, 131072)])
def test_quantize_rows(dtype, M, K):
    from mfar.modeling.quantized import quantize_rows
    x = (torch.randn(M, K, generator=_gen(30), device="cuda") * torch.exp(torch.randn(K, generator=_gen(31), device="cuda"))).to(TYPES[dtype])
    q, s = quantize_rows(x)
    wq, ws = _quantize_ref(x)
    assert torch.equal(s, ws) and torch.equal(q, wq)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_quantize_rows_as_elementary_operations_do(dtype):
    """The same bytes and scales: one that fell on the other side of a tie would be a whole step off."""
    from mfar.modeling.quantized import quantize_rows
    x = torch.randn(20000, 1003, generator=_gen(33), device="cuda").to(TYPES[dtype])
    q, s = quantize_rows(x)
    scale = x.float().abs().amax(1) / 127
    assert torch.equal(s, scale) and torch.equal(q, torch.round(x.float() / scale[:, None]).to(torch.int8))


def test_quantize_rows_ties_zeros_and_poison():
    from mfar.modeling.quantized import quantize_rows
    x = torch.zeros(7, 130, device="cuda")
    x[0, :128] = torch.arange(-63.5, 64.5, 1.0, device="cuda")               # scale 0.5: whole numbers, twice each value
    x[1, 0], x[1, 1:] = 127.0, torch.arange(129, device="cuda") + 0.5 - 64   # scale 1: halves go to the even neighbour
    x[3, 5] = float("nan")
    x[4, 6] = float("-inf")
    x[5] = 1e-44                                                             # a scale below the smallest normal number
    x[6] = 3.0e38
    q, s = quantize_rows(x)
    good = [0, 1, 2, 6]
    wq, ws = _quantize_ref(x[good])
    assert torch.equal(q[good], wq) and torch.equal(s[good], ws)
    assert torch.isnan(s[3:5]).all() and not q[3:5].any() and s[2] == 0
    assert torch.equal(quantize_rows(x.t().contiguous().t())[0][good], wq)
    assert quantize_rows(x[:0])[0].shape == (0, 130)


def _int8_case(M, K, N, dtype, bias, seed=40):
    g = _gen(seed)
    x = (torch.randn(M, K, generator=g, device="cuda") * torch.exp(0.5 * torch.randn(K, generator=g, device="cuda"))).to(TYPES[dtype])
    w = torch.randn(N, K, generator=g, device="cuda") / math.sqrt(K)
    ws = w.abs().amax(1) / 127
    wq = torch.round(w / ws[:, None]).to(torch.int8)
    return x, wq, ws, torch.randn(N, generator=g, device="cuda") if bias else None


def _int8_check(x, wq, ws, b, got):
    from helpers.operator_refs import U32, check, half_step
    xq, xs = _quantize_ref(x)
    y = xq.double().reshape(-1, x.shape[-1]) @ wq.double().t() * xs.double().reshape(-1, 1) * ws.double()
    z = y + (b.double() if b is not None else 0.0)
    # exact sums; the sum's conversion, two scales and the bias round in fp32, the result once more
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 1e-37
    check("y", got.reshape(-1, wq.shape[0]), z, half_step(x.dtype) * z.abs() + 5 * U32 * (y.abs() + z.abs()) + tiny)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 768, 768), (12, 768, 769), (32, 2048, 65), (31, 2000, 100), (32, 2049, 40), (33, 64, 96), (129, 1001, 519), (300, 130, 257), (1000, 1536, 768), (70, 4096, 33),
                                   (513, 17, 1030), (3000, 200, 1500), (2049, 1000, 1025), (1700, 136, 1700), (4100, 144, 4200), (4000, 300, 4097)])
def test_int8_linear(dtype, M, K, N):
    from mfar.modeling.quantized import int8_linear
    print(f"int8 {dtype} {M} {K} {N}", flush=True)
    x, wq, ws, b = _int8_case(M, K, N, dtype, (M + N) % 2 == 0)
    _int8_check(x, wq, ws, b, int8_linear(x, wq, ws, b))


@pytest.mark.parametrize("M", [5, 300])
def test_int8_linear_result_types(M):
    from mfar.modeling.quantized import int8_linear
    x, wq, ws, b = _int8_case(M, 130, 72, "fp16", True)
    exact = int8_linear(x, wq, ws, b, out_dtype=torch.float32)
    for t in (torch.float16, torch.bfloat16, torch.float32):
        got = int8_linear(x, wq, ws, b, out_dtype=t)
        assert got.dtype == t and torch.equal(got, exact.to(t))
        assert torch.equal(int8_linear(x.float(), wq, ws, b, out_dtype=t), got)
    with pytest.raises(TypeError):
        int8_linear(x, wq, ws, b, out_dtype=torch.float64)


def test_int8_linear_layouts_extremes_and_poison():
    from mfar.modeling.quantized import int8_linear
    x, wq, ws, b = _int8_case(60, 200, 70, "fp16", True)
    want = int8_linear(x, wq, ws, b)
    assert torch.equal(int8_linear(x.view(3, 4, 5, 200), wq, ws, b).view(60, 70), want)
    wide = torch.full((60, 333), float("nan"), dtype=torch.float16, device="cuda")
    wide[:, 7:207] = x
    assert torch.equal(int8_linear(wide[:, 7:207], wq, ws, b), want)               # rows apart, not on 16 bytes
    assert torch.equal(int8_linear(x.t().contiguous().t(), wq, ws, b), want)
    shifted = torch.empty(wq.numel() + 5, dtype=torch.int8, device="cuda")[5:].view_as(wq).copy_(wq)
    assert torch.equal(int8_linear(x, shifted, ws, b), want)
    assert int8_linear(x[:0], wq, ws, b).shape == (0, 70) and int8_linear(x, wq[:0], ws[:0]).shape == (60, 0)
    x2 = x.clone()
    x2[3], x2[5, 9], x2[6, 1] = 0.0, float("inf"), float("nan")
    got = int8_linear(x2, wq, ws, b)
    assert torch.equal(got[3], b.half()) and torch.isnan(got[5:7]).all()
    rest = [i for i in range(60) if i not in (3, 5, 6)]
    assert torch.equal(got[rest], want[rest])
    big, wmax = torch.ones(2, 131072, device="cuda"), torch.full((3, 131072), 127, dtype=torch.int8, device="cuda")
    y = int8_linear(big, wmax, torch.ones(3, device="cuda"))                        # the largest sum: 127 * 127 * 131072 < 2^31
    scale = float(torch.tensor(1.0) / 127)
    assert torch.allclose(y.double(), torch.full((2, 3), 127.0 * 127 * 131072 * scale, dtype=torch.float64, device="cuda"), rtol=4 * 2.0 ** -24, atol=0)


def test_int8_linear_captured_and_on_another_stream():
    from mfar.modeling.quantized import int8_linear
    x, wq, ws, b = _int8_case(200, 300, 150, "bf16", True)
    want = int8_linear(x, wq, ws, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = int8_linear(x, wq, ws, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    static = x.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = int8_linear(static, wq, ws, b)
    for turn in range(3):
        fresh = _int8_case(200, 300, 150, "bf16", False, seed=50 + turn)[0]
        static.copy_(fresh)
        g.replay()
        assert torch.equal(y, int8_linear(fresh, wq, ws, b)), turn


# ---- distillation -----------------------------------------------------------------------------------------------------------------------
def _distill_case(seed, T, N, K, dtype):
    g = _gen(seed)
    x = (torch.randn(T, N, generator=g, device="cuda") * 2).to(TYPES[dtype])
    ids = torch.randint(0, N, (T, K), generator=g, device="cuda")                   # repeats among them
    ids = torch.where(torch.rand(T, K, generator=g, device="cuda") < 0.2, torch.full_like(ids, -1), ids)
    return x, ids, torch.randn(T, K, generator=g, device="cuda") * 3, torch.rand(T, generator=g, device="cuda") - 0.3


def _distill_check(x, ids, scores, tau, dloss):
    from helpers.operator_refs import check, distillation_ref
    from mfar.modeling.losses import topk_distillation
    leaf = x.detach().requires_grad_(True)
    loss = topk_distillation(leaf, ids, scores, temperature=tau)
    (dx,) = torch.autograd.grad(loss, [leaf], dloss)
    want, e, d, ed = distillation_ref(x, ids, scores, tau, dloss)
    check("loss", loss.detach(), want, e)
    check("gradient", dx, d, ed)
    return loss.detach(), dx


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("T,N,K,tau", [(1, 1, 1, 1.0), (3, 2, 5, 0.5), (16, 32, 8, 1.0), (5, 255, 100, 2.0), (33, 1001, 50, 1.0), (2, 70003, 1024, 4.0), (300, 4099, 7, 0.05)])
def test_distillation(dtype, T, N, K, tau):
    print(f"distillation {dtype} {T} {N} {K} {tau}", flush=True)
    _distill_check(*_distill_case(60, T, N, K, dtype)[:3], tau, _distill_case(60, T, N, K, dtype)[3])


@pytest.mark.parametrize("N", [50, 9000])
def test_distillation_edges(N):
    """Rows without a teacher, hidden columns, ids past the end, strided rows, int32 ids, 16-bit teacher scores."""
    from mfar.modeling.losses import TopKDistillationLoss, topk_distillation
    x, ids, scores, dloss = _distill_case(61, 8, N, 10, "fp32")
    ids[1] = -1
    ids[4] = 7
    x[2, 20:] = float("-inf")
    ids[2] = torch.arange(10, device="cuda")
    x[1] = float("-inf")
    x[5] = 1e30
    ids[5, 0] = 3
    rows = [0, 2, 3, 4, 6, 7]
    _distill_check(x[rows], ids[rows], scores[rows], 1.0, dloss[rows])
    leaf = x.clone().requires_grad_(True)
    loss = topk_distillation(leaf, ids, scores)
    (dx,) = torch.autograd.grad(loss, [leaf], dloss)
    assert loss[1] == 0 and not dx[1].any()
    assert torch.isfinite(dx[5]).all()
    bad = ids.clone()
    bad[3, 2] = N
    leaf = x.clone().requires_grad_(True)
    l2 = topk_distillation(leaf, bad, scores)
    (d2,) = torch.autograd.grad(l2, [leaf], dloss)
    assert torch.isnan(l2[3]) and torch.isnan(d2[3]).all()
    keep = [i for i in range(8) if i != 3]
    assert torch.equal(l2[keep], loss.detach()[keep]) and torch.equal(d2[keep], dx[keep])
    wide = torch.full((8, N + 5), float("nan"), device="cuda")
    wide[:, 3:N + 3] = x
    w = wide.requires_grad_(True)
    l3 = topk_distillation(w[:, 3:N + 3], ids.to(torch.int32), scores)
    (d3,) = torch.autograd.grad(l3, [w], dloss)
    assert torch.equal(l3, loss) and torch.equal(d3[:, 3:N + 3], dx) and not d3[:, :3].any()
    assert torch.equal(topk_distillation(x.t().contiguous().t(), ids, scores), loss.detach())
    mean, total, each = (TopKDistillationLoss(reduction=r)(x[rows], ids[rows], scores[rows]) for r in ("mean", "sum", "none"))
    assert torch.allclose(mean * len(rows), total) and torch.equal(total, each.sum())
    empty = x[:0].clone().requires_grad_(True)
    le = topk_distillation(empty, ids[:0], scores[:0])
    assert le.shape == (0,) and torch.autograd.grad(le.sum(), [empty])[0].shape == (0, N)


def test_distillation_captured_and_replayed():
    from mfar.modeling.losses import topk_distillation
    x, ids, scores, dloss = _distill_case(62, 6, 20011, 30, "fp16")
    leaf = x.clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(topk_distillation(leaf, ids, scores), [leaf], dloss)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss = topk_distillation(leaf, ids, scores)
        (dx,) = torch.autograd.grad(loss, [leaf], dloss)
    for turn in range(3):
        fresh = _distill_case(70 + turn, 6, 20011, 30, "fp16")
        with torch.no_grad():
            leaf.copy_(fresh[0])
            ids.copy_(fresh[1])
            scores.copy_(fresh[2])
        g.replay()
        other = leaf.detach().clone().requires_grad_(True)
        l2 = topk_distillation(other, ids, scores)
        (d2,) = torch.autograd.grad(l2, [other], dloss)
        assert torch.equal(loss.detach(), l2.detach()) and torch.equal(dx, d2), turn


# ---- refusals -----------------------------------------------------------------------------------------------------------------------------
def test_refusals():
    from mfar.modeling.attention import relative_bias_attention as attend
    from mfar.modeling.losses import topk_distillation
    from mfar.modeling.quantized import int8_linear, quantize_rows
    z = lambda *s, t=torch.float16: torch.zeros(*s, dtype=t, device="cuda")   # noqa: E731
    q, table = z(2, 3, 4, 64), z(32, 4)
    for bad in (dict(k=z(2, 3, 4, 32)), dict(k=z(1, 3, 4, 64)), dict(k=z(2, 3, 2, 64), v=z(2, 3, 2, 64)), dict(q=z(2, 3, 256)), dict(table=z(32, 5)),
                dict(table=z(32, 4, t=torch.int32)), dict(table=z(31, 4)), dict(key_mask=z(2, 4, t=torch.bool)), dict(key_mask=z(2, 3)),
                dict(q_start=z(3, t=torch.int32)), dict(q_start=z(2)), dict(q_start=2 ** 31), dict(max_distance=5), dict(key_mask=torch.ones(2, 3, dtype=torch.bool))):
        args = dict(q=q, k=q, v=q, table=table)
        if "k" in bad and "v" not in bad:
            bad["v"] = bad["k"]
        args.update(bad)
        with pytest.raises(ValueError):
            attend(args.pop("q"), args.pop("k"), args.pop("v"), args.pop("table"), **args)
    with pytest.raises(ValueError):
        attend(z(1, 2, 1, 136), z(1, 2, 1, 136), z(1, 2, 1, 136), z(32, 1))
    with pytest.raises(TypeError):
        attend(q, q.float(), q.float(), table)
    with pytest.raises(TypeError):
        attend(q.double(), q.double(), q.double(), table)
    x, w, s = z(5, 16), z(7, 16, t=torch.int8), z(7, t=torch.float32)
    for args in ((x, w[:, :8], s), (x, w.float(), s), (x, w, s[:3]), (x, w, s.half()), (x, w, s, z(6)), (x, w, s, z(7, t=torch.int32))):
        with pytest.raises(ValueError):
            int8_linear(*args)
    with pytest.raises(TypeError):
        quantize_rows(x.double())
    with pytest.raises(ValueError):
        quantize_rows(z(3, 0))
    with pytest.raises(RuntimeError, match="no_grad"):
        int8_linear(z(5, 16).requires_grad_(True), w, s)
    st, ids, sc = z(3, 20), z(3, 4, t=torch.int64), z(3, 4)
    for args in ((st[0], ids, sc), (st, ids[:2], sc), (st, ids.half(), sc), (st, ids, sc[:, :3]), (st, ids, ids), (st, z(3, 1025, t=torch.int64), z(3, 1025)),
                 (st, ids[:, :0], sc[:, :0])):
        with pytest.raises(ValueError):
            topk_distillation(*args)
    for tau in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            topk_distillation(st, ids, sc, temperature=tau)
