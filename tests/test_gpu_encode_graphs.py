"""GPU tests of the opt-in corpus encodes through captured forwards: graphs are captured and replayed; they follow weights that change and 8-bit copies that
move between encodes, and do not outlive a switch of the attention."""
import json

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _module(tmp_path, monkeypatch, spec, n):
    """A module over n texts of one token count, and its encode of the corpus: (precision, captured forwards or not) -> rows."""
    from mfar.data.schema import resolve_fields
    from mfar.modeling.contrastive import RetrievalTrainingModule
    from mfar.modeling.util import prepare_model, read_and_create_indices
    monkeypatch.setenv("MFAR_ENCODE_TOKEN_BUDGET", "0")                      # batches of dev_batch_size texts: few shapes
    rng = np.random.default_rng(3)
    with open(tmp_path / "corpus", "w") as f:
        for i in range(n):
            f.write(f"{i}\t{json.dumps({'title': ' '.join(rng.choice(list('abcdefgh'), 12))})}\n")       # one token a letter: all of one length
    _, enc, _ = prepare_model(spec)
    enc = enc.cuda()
    fields = resolve_fields(["title_dense"], "mag")
    corpus, vectors, indices = read_and_create_indices(str(tmp_path / "corpus"), "mag", fields, str(tmp_path / "t"), enc)
    mod = RetrievalTrainingModule(encoder=enc, model_id="m", decoder=None, corpus_path=str(tmp_path / "corpus"), corpus=corpus, dataset_name="mag",
                                  dev_qrels_path=str(tmp_path / "q"), out_dir=str(tmp_path / "o"), field_info=fields, indices_dict=indices, vectors_dict=vectors,
                                  weights_learning_rate=1e-3, dev_batch_size=16)

    def encode(mode, graphs):
        monkeypatch.setenv("MFAR_ENCODE_GRAPHS", graphs)
        mod.encode_precision = mode
        mod.mark_encoder_updated()
        mod.on_eval_start()
        return mod.slab.read_rows(0, 0, n)
    return mod, encode


@pytest.mark.parametrize("spec", ["random-init:128x2", "random-init-t5:128x2"])
def test_int8_corpus_encode_replays_captured_forwards(tmp_path, monkeypatch, spec):
    mod, encode = _module(tmp_path, monkeypatch, spec, 240)
    enc = mod.encoder
    held, rows = [], []
    for turn in range(4):
        got = encode("int8", "1")
        g = mod._graphed
        before = g.n_replays
        assert before > 0 and g.graphs and not g.failed and not g.rejected, turn
        again = encode("int8", "1")
        assert mod._graphed is g and g.n_replays > before and not g.failed and not g.rejected, turn
        full = encode("fp16", "1")                                           # the same shapes, other layers: no graph of the 8-bit ones is taken for it
        assert mod._graphed is g and not g.failed
        want, want_full = encode("int8", "0"), encode("fp16", "0")           # eager; the graphs are gone
        for a, b in ((got, want), (again, want), (full, want_full)):
            assert abs(a - b).max() <= 4e-3 * abs(b).max(), turn
        assert abs(want - want_full).max() > 0
        rows.append(want)
        if turn:
            assert abs(rows[turn] - rows[turn - 1]).max() > 2e-2 * abs(want).max(), turn
        # other weights in place, and (from the second turn on) memory taken between the encodes, so that the 8-bit copies lie elsewhere
        with torch.no_grad():
            for p in enc.parameters():
                p.add_(torch.randn(p.shape, device=p.device, generator=torch.Generator("cuda").manual_seed(turn)) * 0.05 * p.std())
        if turn:
            held += [torch.empty(s, dtype=torch.uint8, device="cuda") for s in (1 << 14, 1 << 16, 128 * 128, 128 * 512, 1 << 20)]
    # without the eager encodes between them: weights change, the graphs of the encode before are kept or dropped as the copies' addresses have it
    encode("int8", "1")
    g = mod._graphed
    for turn in range(3):
        with torch.no_grad():
            for p in enc.parameters():
                p.add_(torch.randn(p.shape, device=p.device, generator=torch.Generator("cuda").manual_seed(9 + turn)) * 0.05 * p.std())
        if turn == 1:
            held += [torch.empty(s, dtype=torch.uint8, device="cuda") for s in (128 * 128, 128 * 512, 512 * 4, 128 * 4)]
        before = g.n_replays
        got = encode("int8", "1")
        assert mod._graphed is g and g.n_replays > before and not g.failed and not g.rejected, turn
        rows.append(got)
    want = encode("int8", "0")
    assert abs(rows[-1] - want).max() <= 4e-3 * abs(want).max()
    assert abs(rows[-2] - want).max() > 2e-2 * abs(want).max()


@pytest.mark.parametrize("precision", ["fp32", "fp16"])
def test_switched_attention_is_the_one_that_is_replayed(tmp_path, monkeypatch, precision):
    """Each attention's replayed encode gives the bits of its own graphs' first replays and lies by its own eager encode, whichever ran before."""
    mod, encode = _module(tmp_path, monkeypatch, "random-init-t5:128x2", 160)
    with torch.no_grad():                                                    # a table that matters, and attention that is far from uniform
        mod.encoder.auto_model.encoder.block[0].layer[0].SelfAttention.relative_attention_bias.weight.normal_(std=3.0)
    from mfar.modeling import t5
    inner, calls = t5.t5_encoder_forward, []

    def spy(*a):
        calls.append(1)
        return inner(*a)
    monkeypatch.setattr(t5, "t5_encoder_forward", spy)
    for turn in range(2):
        for fused in (False, True):
            mod.encoder.use_fused_attention(fused)
            calls.clear()
            got = encode(precision, "1")
            g = mod._graphed
            assert g.n_replays > 0 and g.graphs and not g.failed and not g.rejected
            assert bool(calls) == fused                                      # captured anew after the switch, by the attention that is on
            calls.clear()
            again = encode(precision, "1")
            assert mod._graphed is g and not calls                           # replays alone
            assert abs(again - got).max() <= (2e-5 if precision == "fp32" else 4e-3) * abs(got).max()
    want = encode(precision, "0")
    assert abs(got - want).max() <= (2e-5 if precision == "fp32" else 4e-3) * abs(want).max()
