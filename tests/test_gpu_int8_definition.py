"""GPU tests of the 8-bit operators against their definition in 64 bits, scale = max|row| / 127 unrounded, with no step of the kernels' own arithmetic.

u = 2^-24.  1 / 127 in fp32 is 0.0625 u off, its product with the maximum rounds once: the scale is within 1.07 u.  The quotient rounds once more, so what is
rounded to a whole number is within 2.08 u of row / scale, relative: a byte may differ from the definition's, by one step, only where row / scale lies that
close to a half.  (Over 4 x 10^7 random numbers of each type 59, 341 and 1832 bytes do, in fp32, fp16 and bf16; under the correctly rounded quotient
max / 127 as the scale 61, 727 and 4577 would.)"""
import math

import pytest
import torch

from helpers.operator_refs import U32, check, half_step

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _definition(x):
    """(whole numbers, scale, where a whole number may fall to either side) in float64"""
    xd = x.double()
    top = xd.abs().amax(-1, keepdim=True)
    v = xd * 127 / torch.where(top > 0, top, torch.ones_like(top))
    return torch.round(v), top / 127, (v.abs() - v.abs().floor() - 0.5).abs() <= 2.1 * U32 * v.abs()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_quantize_rows_against_the_definition(dtype):
    from mfar.modeling.quantized import quantize_rows
    x = torch.randn(9000, 1003, generator=_gen(80), device="cuda").to(TYPES[dtype])
    q, s = quantize_rows(x)
    n, scale, either = _definition(x)
    assert bool(((s.double() - scale[:, 0]).abs() <= 1.07 * U32 * scale[:, 0]).all())
    off = (q.double() - n).abs()
    assert float(off.max()) <= 1 and not bool((off > 0)[~either].any())
    # (so that the test says something.  bf16: a maximum of significand 254 = 2 * 127, one row in some 128, makes x 127 / max a multiple of 2^-k of the 8-bit
    # significand of x: exactly a half for about one in 4 of the usual sizes; 1 / 512 in all)
    assert float(either.double().mean()) < (2.0 ** -8 if dtype == "bf16" else 2.0 ** -10)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("M,K,N", [(12, 768, 769), (1003, 1001, 519), (4100, 768, 1500), (300, 4096, 96)])
def test_int8_linear_against_the_definition(dtype, M, K, N):
    from mfar.modeling.quantized import int8_linear
    print(f"int8 {dtype} {M} {K} {N}", flush=True)
    g = _gen(81)
    x = (torch.randn(M, K, generator=g, device="cuda") * torch.exp(0.5 * torch.randn(K, generator=g, device="cuda"))).to(TYPES[dtype])
    wq = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    ws = torch.rand(N, generator=g, device="cuda") / (127 * math.sqrt(K))
    b = torch.randn(N, generator=g, device="cuda")
    n, scale, either = _definition(x)
    wt = wq.double().t().contiguous()
    y = (n @ wt) * scale * ws.double()
    z = y + b.double()
    # exact sums; then the sum's conversion, both scales (one of them 1.07 u off) and the bias round in fp32, the result once more; a byte that fell to the
    # other side of a half moves its row by one of its weights
    moved = (either.double() @ wt.abs()) * scale * ws.double()
    tiny = 2.0 ** -25 if dtype == "fp16" else 1e-37
    check("y", int8_linear(x, wq, ws, b), z, half_step(x.dtype) * (z.abs() + moved) + 5 * U32 * (y.abs() + z.abs() + moved) + moved + tiny)
