"""CPU tests of the switches around the fused T5 forward: captured forwards do not outlive a switch, and what the fused forward would pass by."""
import torch


def _t5():
    from mfar.modeling.util import prepare_model
    return prepare_model("random-init-t5:64x2")[1]


def test_captured_forwards_are_dropped_when_the_attention_is_switched():
    from mfar.modeling.graphed import GraphedForward
    enc = _t5()
    graphed = GraphedForward(enc, torch.device("cpu"))
    for on in (False, True, True, False):
        before = bool(enc[0].fused_stack)
        enc.use_fused_attention(on)
        graphed.graphs[(1, 8, None)] = ("graph", {}, None)
        if graphed.sig is None:
            graphed.sig = graphed.signature()
        graphed.begin()
        assert bool(graphed.graphs) == (on == before), on


def test_why_a_forward_stays_stock():
    from mfar.modeling.t5 import attention_dropout, stays_stock, t5_stack
    model = _t5().auto_model
    stack = t5_stack(model)
    assert attention_dropout(stack) > 0 and not stack.training and not stays_stock(model, stack)
    stack.train()
    assert "drops attention weights" in stays_stock(model, stack)
    for block in stack.block:
        block.layer[0].SelfAttention.dropout = 0.0
    assert not stays_stock(model, stack)                                   # (the dropout of hidden states is the stock modules' own)
    assert "another" in stays_stock(_t5().auto_model, stack)


def test_hooks_and_checkpointing_stay_stock():
    """The fused forward calls neither the blocks nor the attention modules: what is hung on them would not run."""
    from mfar.modeling.t5 import stays_stock, t5_stack
    model = _t5().auto_model
    stack = t5_stack(model)
    first = stack.block[0].layer[0].SelfAttention
    for m in (model, stack, stack.block[1], stack.block[1].layer[0], stack.block[1].layer[0].SelfAttention, first.relative_attention_bias):
        for register in (m.register_forward_hook, m.register_forward_pre_hook, m.register_full_backward_hook):
            handle = register(lambda *a: None)
            assert type(m).__name__ in stays_stock(model, stack)
            handle.remove()
            assert not stays_stock(model, stack)
    inner = stack.block[0].forward
    stack.block[0].forward = lambda *a, **k: inner(*a, **k)
    assert "forward of its own" in stays_stock(model, stack)
    del stack.block[0].forward
    for m in (first.q, first.o, stack.block[0].layer[0].layer_norm, stack.block[0].layer[-1], stack.final_layer_norm, stack.embed_tokens):
        m.register_forward_hook(lambda *a: None)                           # called as ever
    assert not stays_stock(model, stack)
    model.gradient_checkpointing_enable()
    assert not stays_stock(model, stack)
    model.train()
    for block in stack.block:
        block.layer[0].SelfAttention.dropout = 0.0
    assert "checkpointing" in stays_stock(model, stack)
    model.gradient_checkpointing_disable()
    assert not stays_stock(model, stack)
