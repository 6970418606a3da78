"""GPU tests of the encoder's operators where the framework uses them: the fused T5 forward against the stock one (values and gradients), the 8-bit
corpus encode, and a training step that distils an index's top lists into a student through all three."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _texts(n, longest, seed=0):
    import random
    rng = random.Random(seed)
    words = ["alpha", "beta", "query", "field", "document", "7", "x1", "retrieval", "of", "and"]
    return [" ".join(rng.choice(words) for _ in range(rng.randint(1, longest))) for _ in range(n)]


def _t5(spec="random-init-t5:128x3"):
    from mfar.modeling.util import prepare_model
    _, enc, _ = prepare_model(spec)
    torch.manual_seed(5)
    with torch.no_grad():      # a table that matters (random-init tables are near zero against the scores)
        enc.auto_model.encoder.block[0].layer[0].SelfAttention.relative_attention_bias.weight.normal_(std=1.0)
    return enc.cuda()


def _features(enc, texts):
    return {k: v.cuda() for k, v in enc.tokenize(texts).items() if k in ("input_ids", "attention_mask")}


def test_fused_t5_forward_is_the_stock_forward():
    """fp32, padded batch.  Both run the same projections; attention and its sums differ in order only: a layer's relative error stays near 2^-22 and
    the norms in between keep it there, so 1e-5 of the largest value is far above it and far below any wrong bias, mask or scale."""
    enc = _t5()
    f = _features(enc, _texts(9, 60))
    with torch.no_grad():
        want = enc(f)
        enc.use_fused_attention()
        got = enc(f)
        enc.use_fused_attention(False)
        again = enc(f)
    m = f["attention_mask"].bool()
    a, b = got["token_embeddings"][m], want["token_embeddings"][m]
    assert float((a - b).abs().max()) <= 1e-5 * float(b.abs().max())
    assert float((got["sentence_embedding"] - want["sentence_embedding"]).abs().max()) <= 1e-5 * float(want["sentence_embedding"].abs().max())
    assert torch.equal(again["sentence_embedding"], want["sentence_embedding"])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_fused_t5_forward_under_autocast(dtype):
    """Held to the fp32 forward: the fused forward may be no further from it than twice the stock one under the same autocast."""
    enc = _t5()
    f = _features(enc, _texts(12, 80, 1))
    with torch.no_grad():
        exact = enc(f)["sentence_embedding"]
        with torch.autocast("cuda", dtype=dtype):
            stock = enc(f)["sentence_embedding"].float()
            enc.use_fused_attention()
            fused = enc(f)["sentence_embedding"].float()
    err = lambda x: float((x - exact).norm() / exact.norm())   # noqa: E731
    assert err(fused) <= 2 * err(stock) + 1e-6, (err(fused), err(stock))


def test_fused_t5_in_fp16_stays_within_the_type():
    """An fp16 model whose sums of hidden states pass the type's largest value: held there, as the stock blocks hold them, not infinite and then NaN."""
    enc = _t5().half().eval()
    seen = []
    with torch.no_grad():
        for block in enc.auto_model.encoder.block[:2]:
            o = block.layer[0].SelfAttention.o
            o.weight.fill_(6e4)
            o.register_forward_hook(lambda m, i, out: seen.append(bool(out.isinf().any())))
        f = _features(enc, _texts(9, 60))
        stock = enc(f)["sentence_embedding"]
        enc.use_fused_attention()
        seen.clear()
        fused = enc(f)["sentence_embedding"]
    assert any(seen) and bool(stock.isfinite().all()) and bool(fused.isfinite().all())


def test_fused_t5_gradients_are_the_stock_gradients():
    """Every parameter's gradient, the bias table's among them, in fp32 (no dropout)."""
    enc = _t5()
    f = _features(enc, _texts(7, 50, 2))
    dout = torch.randn(7, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    params = dict(enc.named_parameters())
    enc.eval()
    grads = {}
    for fused in (False, True):
        enc.use_fused_attention(fused)
        enc.zero_grad()
        enc(f)["sentence_embedding"].backward(dout)
        grads[fused] = {n: p.grad.clone() for n, p in params.items() if p.grad is not None}
    assert grads[True].keys() == grads[False].keys() and any("relative_attention_bias" in n for n in grads[True])
    for n, want in grads[False].items():
        got = grads[True][n]
        assert float((got - want).norm()) <= 2e-5 * float(want.norm()) + 1e-9, n


def test_fused_attention_training_with_dropout_stays_stock_and_other_encoders_refuse_it():
    from mfar.modeling.util import prepare_model
    enc = _t5()
    enc.use_fused_attention()
    f = _features(enc, _texts(4, 20, 3))
    enc.train()                                                            # dropout_rate 0.1
    torch.manual_seed(9)
    a = enc(f)["sentence_embedding"]
    enc.use_fused_attention(False)
    torch.manual_seed(9)
    assert torch.equal(a, enc(f)["sentence_embedding"])
    _, bert, _ = prepare_model("random-init:64x2")
    with pytest.raises(ValueError, match="T5"):
        bert.use_fused_attention()


def test_fused_t5_state_dict_and_capture():
    """The switch adds no parameter; a captured forward replays the eager one."""
    enc = _t5().eval()
    keys = list(enc.state_dict())
    enc.use_fused_attention()
    assert list(enc.state_dict()) == keys
    f = _features(enc, _texts(6, 40, 4))
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            enc(f)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = enc(f)["sentence_embedding"]
        for turn in range(3):
            ids = f["input_ids"]
            ids.copy_(torch.where(f["attention_mask"].bool(), (ids + turn) % 40 + 5, ids))
            g.replay()
            want = enc(f)["sentence_embedding"]
            assert float((out - want).abs().max()) <= 1e-6 * float(want.abs().max()), turn


@pytest.mark.parametrize("spec", ["random-init:128x3", "random-init-t5:128x3"])
def test_int8_encoder_and_its_restoration(spec):
    """Under int8_linears the transformer's products run in 8 bits; behind it the encoder is bit for bit what it was.  Each product rounds both operands to
    steps of max / 127: relative errors of about 1 / 127 / sqrt(3) per operand and row, through 3 layers with residuals -- 5 % is far above that
    and far below an unrelated embedding."""
    from mfar.modeling.quantized import Int8Linear, int8_linears
    from mfar.modeling.util import prepare_model
    _, enc, _ = prepare_model(spec)
    enc = enc.cuda().eval()
    f = _features(enc, _texts(10, 40, 6))
    with torch.no_grad():
        want = enc(f)["sentence_embedding"]
        with int8_linears(enc[0]) as n:
            assert n == sum(isinstance(m, Int8Linear) for m in enc.modules()) and n >= 3 * 6
            got = enc(f)["sentence_embedding"]
            with torch.autocast("cuda", dtype=torch.float16):
                half = enc(f)["sentence_embedding"].float()
        assert not any(isinstance(m, Int8Linear) for m in enc.modules())
        assert torch.equal(enc(f)["sentence_embedding"], want)
    for x in (got, half):
        assert float((x - want).norm() / want.norm()) < 0.05
    with pytest.raises(KeyError):
        with int8_linears(enc[0]):
            raise KeyError
    assert not any(isinstance(m, Int8Linear) for m in enc.modules())


@pytest.mark.parametrize("graphs", ["0", "1"])
def test_int8_corpus_encode(tmp_path, monkeypatch, graphs):
    """on_eval_start with encode precision int8: the slab's rows are the 8-bit encoder's, near the fp32 ones; the encoder is left as it was."""
    from mfar.data.schema import resolve_fields
    from mfar.modeling.contrastive import RetrievalTrainingModule
    from mfar.modeling.util import prepare_model, read_and_create_indices
    import json
    monkeypatch.setenv("MFAR_ENCODE_GRAPHS", graphs)
    n = 300
    with open(tmp_path / "corpus", "w") as f:
        for i, t in enumerate(_texts(n, 30, 8)):
            f.write(f"{i}\t{json.dumps({'title': t})}\n")
    _, enc, _ = prepare_model("random-init:128x2")
    enc = enc.cuda()
    fields = resolve_fields(["title_dense"], "mag")
    corpus, vectors, indices = read_and_create_indices(str(tmp_path / "corpus"), "mag", fields, str(tmp_path / "t"), enc)
    mod = RetrievalTrainingModule(encoder=enc, model_id="m", decoder=None, corpus_path=str(tmp_path / "corpus"), corpus=corpus, dataset_name="mag",
                                  dev_qrels_path=str(tmp_path / "q"), out_dir=str(tmp_path / "o"), field_info=fields, indices_dict=indices, vectors_dict=vectors,
                                  weights_learning_rate=1e-3)
    rows = {}
    for mode in ("fp32", "int8", "int8"):
        mod.encode_precision = mode
        mod.mark_encoder_updated()
        mod.on_eval_start()
        got = mod.slab.read_rows(0, 0, n)
        if mode in rows:
            assert abs(rows[mode] - got).max() <= 4e-3 * abs(got).max()      # (replayed or eager, the same products)
        rows[mode] = got
    import numpy as np
    err = float(np.linalg.norm(rows["int8"] - rows["fp32"]) / np.linalg.norm(rows["fp32"]))
    assert 0 < err < 0.05, err


def test_distillation_of_an_index_into_a_student():
    """As they would be used together: a corpus encoded in 8 bits into an index, the teacher's top lists from its search, a T5 student trained on them
    through the fused attention; the student's gradients are those of the stock encoder and an fp64 loss, and a step along them lowers the loss of the
    linearised objective (checked as a directional derivative, not by how far a loss falls)."""
    from mfar.data.index import MultiFieldIndex
    from mfar.modeling.losses import TopKDistillationLoss
    from mfar.modeling.quantized import int8_linears
    docs, queries = _texts(400, 25, 10), _texts(6, 8, 11)
    teacher, student = _t5().eval(), _t5("random-init-t5:128x2").eval()
    with torch.no_grad():
        with int8_linears(teacher[0]):
            vec = torch.cat([teacher(_features(teacher, docs[b:b + 100]))["sentence_embedding"] for b in range(0, 400, 100)]).float()
        tq = teacher(_features(teacher, queries))["sentence_embedding"].float().contiguous()
    ix = MultiFieldIndex(400, 1, 128, device=0)
    ix.write_rows(0, 0, vec.contiguous())
    ids, scores = ix.retrieve_fields(tq, 20, False)
    ids, scores = ids[:, 0], scores[:, 0]
    loss_fn = TopKDistillationLoss(temperature=2.0)
    f = _features(student, queries)
    grads = {}
    for fused in (False, True):
        student.use_fused_attention(fused)
        student.zero_grad()
        x = student(f)["sentence_embedding"] @ vec.t()
        if fused:
            loss = loss_fn(x, ids, scores)
        else:                                                              # the definition in 64 bits
            z = x.double() / 2
            p = torch.softmax(scores.double().masked_fill(ids < 0, -math.inf) / 2, 1)
            q = (z - torch.logsumexp(z, 1, keepdim=True)).gather(1, ids.clamp(min=0))
            loss = (4 * (torch.special.xlogy(p, p) - p * q).sum(1)).mean()
        loss.backward()
        grads[fused] = (float(loss.detach()), {n: p.grad.clone() for n, p in student.named_parameters() if p.grad is not None})
    (l0, g0), (l1, g1) = grads[False], grads[True]
    assert abs(l0 - l1) <= 1e-4 * abs(l0) + 1e-6
    assert g0.keys() == g1.keys()
    for n in g0:
        assert float((g1[n] - g0[n]).norm()) <= 1e-3 * float(g0[n].norm()) + 1e-8, n
    assert sum(float((g1[n].double() * g0[n].double()).sum()) for n in g0) > 0
    ix.close()
