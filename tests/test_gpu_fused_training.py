"""GPU tests of MFAR_FUSED_ATTENTION=1 through the `train` command: which attention a training step and the corpus encode run, and that the
user is told where it is not the fused one."""
import json
import warnings

import pytest

from test_gpu_cli import _write_dataset

pytestmark = pytest.mark.gpu


def _t5_directory(path, dropout):
    """A gtr-t5 checkpoint directory (encoder, tokenizer, 2_Dense) with random weights."""
    import torch
    from safetensors.torch import save_file
    from mfar.modeling.util import prepare_model
    tokenizer, enc, _ = prepare_model("random-init-t5:64x2")
    enc.auto_model.config.dropout_rate = dropout
    enc.auto_model.save_pretrained(path)
    tokenizer.save_pretrained(path)
    (path / "2_Dense").mkdir()
    save_file({"linear.weight": torch.eye(64)}, str(path / "2_Dense" / "model.safetensors"))
    (path / "2_Dense" / "config.json").write_text(json.dumps({"in_features": 64, "out_features": 64, "bias": False}))
    return str(path)


@pytest.mark.parametrize("dropout", [0.1, 0.0])
def test_train_command_with_the_fused_attention(tmp_path, monkeypatch, dropout):
    from mfar.commands import train
    from mfar.modeling import t5
    runs = []
    inner = t5.t5_encoder_forward

    def spy(stack, *args):
        runs.append(stack.training)
        return inner(stack, *args)
    monkeypatch.setattr(t5, "t5_encoder_forward", spy)
    monkeypatch.setenv("MFAR_FUSED_ATTENTION", "1")
    data = str(tmp_path / "data")
    _write_dataset(data, n_docs=300, n_q=8)
    with warnings.catch_warnings(record=True) as told:
        warnings.simplefilter("always")
        m = train.main(dataset_name="amazon", lexical_index="unused", out=str(tmp_path / "out"), temp_dir=str(tmp_path / "tmp"), data=data,
                       model_name=_t5_directory(tmp_path / "model", dropout), field_names="title_dense,brand_dense", weights_lr=1e-2, encoder_lr=1e-4,
                       train_batch_size=4, dev_batch_size=16, max_epochs=1, run_one_iteration=True, precision="32")
    told = [str(w.message) for w in told if "fused attention" in str(w.message)]
    assert False in runs                                                   # the corpus encode and the validation
    if dropout:
        assert True not in runs and len(told) == 1 and "drops attention weights" in told[0], (runs, told)
    else:
        assert True in runs and not told, (runs, told)
        table = m.encoder.auto_model.encoder.block[0].layer[0].SelfAttention.relative_attention_bias.weight
        assert table.requires_grad and bool(table.isfinite().all())


def test_hooks_on_attention_modules_run():
    """A forward hook on an attention module sees its outputs, the fused attention switched on or not."""
    import torch
    from mfar.modeling.util import prepare_model
    _, enc, _ = prepare_model("random-init-t5:64x2")
    enc = enc.cuda()
    f = {k: v.cuda() for k, v in enc.tokenize(["alpha beta", "gamma"]).items() if k in ("input_ids", "attention_mask")}
    with torch.no_grad():
        want = enc(f)["sentence_embedding"]
    enc.use_fused_attention()
    seen = []
    handle = enc.auto_model.encoder.block[1].layer[0].SelfAttention.register_forward_hook(lambda m, i, o: seen.append(1))
    with torch.no_grad(), pytest.warns(UserWarning, match="T5Attention"):
        assert torch.equal(enc(f)["sentence_embedding"], want)
    assert seen == [1]
    handle.remove()
    with torch.no_grad():
        enc(f)
    assert seen == [1]
