"""CPU tests of the encoder / training operators: what their entry points refuse (in Python and at the C ABI, where nothing needs a device), and the
bucket layout of the relative position bias."""
import ctypes
import math

import pytest
import torch


def _c_attention(**kw):
    """A valid struct over made-up addresses (never dereferenced: every call here is refused before anything is enqueued)."""
    from mfar import _native
    from mfar.modeling.attention import bucket_borders
    a = _native.Attention()
    a.dtype, a.B, a.Lq, a.Lk, a.H, a.D = _native.DTYPE_F16, 2, 8, 8, 4, 64
    a.n_buckets, a.scale = 32, 1.0
    b = bucket_borders(32, False, 128)
    a.n_borders, a.borders = len(b), ctypes.cast(b, ctypes.POINTER(ctypes.c_int32))
    for n in ("table", "q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv"):
        setattr(a, n, 4096)
    for x in ("q", "k", "v", "do"):
        setattr(a, x + "_b", 8 * 256)
        setattr(a, x + "_l", 256)
        setattr(a, x + "_h", 64)
    a._keep = b
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _borders(*values):
    return (ctypes.c_int32 * len(values))(*values)


@pytest.mark.parametrize("change,what", [
    (dict(dtype=9), "dtype"), (dict(B=-1), "B, Lq"), (dict(B=65536), "65535"), (dict(H=0), "H >= 1"), (dict(H=65536), "65535"), (dict(D=0), "D must"),
    (dict(D=12), "D must"), (dict(D=136), "D must"), (dict(Lq=2 ** 30 + 1), "2\\^30"), (dict(q_start=2 ** 30 + 1), "q_start"), (dict(n_buckets=1), "n_buckets"),
    (dict(n_buckets=31), "n_buckets"), (dict(n_buckets=258), "n_buckets"), (dict(n_borders=6), "n_borders"), (dict(causal=1), "n_borders"), (dict(q=None), "NULL"),
    (dict(table=None), "NULL"), (dict(v=None), "NULL"), (dict(out=None), "NULL"), (dict(k_l=4), "strides"), (dict(v_h=65), "strides"), (dict(q=4104), "aligned"),
    (dict(out_lo=4100), "aligned"), (dict(Lk=2 ** 30), "2\\^30"), (dict(B=65535, H=257), "2\\^24"), (dict(B=128, H=16, Lq=2 ** 21), "2\\^24"),
])
def test_attention_refusals_at_the_c_abi(change, what):
    from mfar import _native
    L = _native.lib()
    a = _c_attention(**change)
    assert L.mfar_attention_forward(0, ctypes.byref(a), None) == -1
    import re
    assert re.search(what, L.mfar_last_error().decode()), L.mfar_last_error()
    assert L.mfar_attention_workspace_bytes(ctypes.byref(a), 0) == -1


def test_attention_borders_and_backward_refusals_at_the_c_abi():
    from mfar import _native
    L = _native.lib()
    for values in ((7, 12, 16, 23, 32, 46, 64), (12, 11, 16, 23, 32, 46, 64), (12, 16, 23, 32, 46, 64, 1024)):
        b = _borders(*values)
        a = _c_attention(borders=ctypes.cast(b, ctypes.POINTER(ctypes.c_int32)))
        assert L.mfar_attention_forward(0, ctypes.byref(a), None) == -1, values
    assert L.mfar_attention_forward(0, None, None) == -1 and L.mfar_attention_backward(0, None, None) == -1
    need = L.mfar_attention_workspace_bytes(ctypes.byref(_c_attention(dtable=4096)), 1)
    assert need > 0
    assert L.mfar_attention_workspace_bytes(ctypes.byref(_c_attention(B=0)), 1) == 0
    for change in (dict(dout=None), dict(dq=None), dict(lse=None), dict(dk=None), dict(do_l=3), dict(dv=4097), dict(workspace=None, workspace_bytes=need),
                   dict(workspace=4096, workspace_bytes=need - 1, dtable=4096)):
        a = _c_attention(**change)
        assert L.mfar_attention_backward(0, ctypes.byref(a), None) == -1, change
    assert L.mfar_attention_forward(0, ctypes.byref(_c_attention(B=0, q=None)), None) == 0      # nothing to do


def test_int8_and_distillation_refusals_at_the_c_abi():
    from mfar import _native
    L, P = _native.lib(), 4096
    F16 = _native.DTYPE_F16
    assert L.mfar_quantize_rows(0, P, 7, 64, 4, 64, P, 64, P, None) == -1                          # type
    assert L.mfar_quantize_rows(0, P, F16, 64, -1, 64, P, 64, P, None) == -1
    assert L.mfar_quantize_rows(0, P, F16, 64, 4, 0, P, 64, P, None) == -1
    assert L.mfar_quantize_rows(0, P, F16, 64, 4, 131073, P, 131073, P, None) == -1
    assert L.mfar_quantize_rows(0, P, F16, 64, 4, 64, P, 63, P, None) == -1
    assert L.mfar_quantize_rows(0, P, F16, -64, 4, 64, P, 64, P, None) == -1
    assert L.mfar_quantize_rows(0, None, F16, 64, 4, 64, P, 64, P, None) == -1
    assert L.mfar_quantize_rows(0, None, F16, 64, 0, 64, None, 64, None, None) == 0
    n = L.mfar_int8_linear_workspace_bytes(40, 100, 20)
    assert n >= 40 * 100 + 40 * 4 and L.mfar_int8_linear_workspace_bytes(10, 100, 20) == 0 and L.mfar_int8_linear_workspace_bytes(-1, 5, 5) == -1
    ok = [0, P, F16, 100, 40, 100, 20, P, P, None, P, F16, P, n, None]
    for i, v in ((2, 5), (3, -1), (4, -1), (5, 0), (6, -1), (6, 2 ** 23 + 1), (7, None), (7, P + 4), (8, None), (10, None), (11, 4), (12, None), (12, P + 8), (13, n - 1)):
        args = list(ok)
        args[i] = v
        assert L.mfar_int8_linear(*args) == -1, (i, v)
    assert L.mfar_int8_linear(*[0 if i in (4,) else v for i, v in enumerate(ok)]) == 0
    assert L.mfar_distill_workspace_bytes(4, 0) == -1 and L.mfar_distill_workspace_bytes(2, 10 ** 6) > 0 and L.mfar_distill_workspace_bytes(5000, 100) == 0
    ok = [0, P, 0, 1000, 4, 1000, P, P, 8, 1.0, P, P, P, P, 1 << 20, None]
    for i, v in ((1, None), (2, 4), (3, -5), (4, -1), (4, 2 ** 31), (4, 2 ** 24), (5, 0), (5, 2 ** 30 + 1), (6, None), (7, None), (8, 0), (8, 1025), (9, 0.0), (9, -1.0),
                 (9, math.inf), (9, math.nan), (9, 1e-19), (9, 2e18), (10, None), (11, None), (12, None)):
        args = list(ok)
        args[i] = v
        assert L.mfar_distill_forward(*args) == -1, (i, v)
    args = list(ok)
    args[3], args[5], args[13] = 10 ** 6, 10 ** 6, None
    assert L.mfar_distill_forward(*args) == -1                                                       # a workspace is needed here
    ok = [0, P, 0, 1000, 4, 1000, P, 8, 1.0, P, P, P, P, None]
    for i in (1, 6, 9, 10, 11, 12):
        args = list(ok)
        args[i] = None
        assert L.mfar_distill_backward(*args) == -1, i


def test_there_is_no_cpu_form():
    from mfar.modeling.attention import relative_bias_attention
    from mfar.modeling.losses import topk_distillation
    from mfar.modeling.quantized import int8_linear, quantize_rows
    q = torch.zeros(1, 2, 2, 8)
    with pytest.raises(ValueError, match="GPU"):
        relative_bias_attention(q, q, q, torch.zeros(32, 2))
    with pytest.raises(ValueError, match="GPU"):
        quantize_rows(torch.zeros(2, 4))
    with pytest.raises(ValueError, match="GPU"):
        int8_linear(torch.zeros(2, 4), torch.zeros(3, 4, dtype=torch.int8), torch.zeros(3))
    with pytest.raises(ValueError, match="GPU"):
        topk_distillation(torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1))


@pytest.mark.parametrize("nb,max_distance,causal", [(32, 128, False), (32, 128, True), (4, 3, False), (2, 9, True), (8, 20, True), (64, 1000, False), (255, 1000, True), (256, 1000, False)])
def test_buckets_of_all_distances(nb, max_distance, causal):
    from helpers.operator_refs import bucket_of
    from mfar.modeling.attention import relative_buckets
    d = torch.arange(-1500, 1501)
    got = relative_buckets(d, nb, causal, max_distance)
    assert got.tolist() == [bucket_of(int(x), nb, causal, max_distance) for x in d]
    assert int(got.min()) == 0 and int(got.max()) <= nb - 1


@pytest.mark.parametrize("causal", [False, True])
def test_buckets_are_those_of_the_t5_family(causal):
    """The default layout (32 buckets, distances up to 128) against the T5 implementation the stock encoder runs."""
    from transformers.models.t5.modeling_t5 import T5Attention
    from mfar.modeling.attention import relative_buckets
    d = torch.arange(-600, 601)
    want = T5Attention._relative_position_bucket(d, bidirectional=not causal, num_buckets=32, max_distance=128)
    assert torch.equal(relative_buckets(d, 32, causal, 128), want)


@pytest.mark.parametrize("nb,causal,max_distance", [(33, False, 128), (2, False, 128), (1, True, 128), (258, False, 1000), (32, False, 8), (32, False, 100000), (255, True, 1100)])
def test_bucket_layouts_that_are_refused(nb, causal, max_distance):
    from mfar.modeling.attention import bucket_borders
    with pytest.raises(ValueError):
        bucket_borders(nb, causal, max_distance)


def test_distillation_reduction_is_checked():
    from mfar.modeling.losses import TopKDistillationLoss
    with pytest.raises(ValueError):
        TopKDistillationLoss(reduction="max")
