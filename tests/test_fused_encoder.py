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
    stack = t5_stack(_t5().auto_model)
    assert attention_dropout(stack) > 0 and not stack.training and not stays_stock(stack)
    stack.train()
    assert "drops attention weights" in stays_stock(stack)
    for block in stack.block:
        block.layer[0].SelfAttention.dropout = 0.0
    assert not stays_stock(stack)                                          # (the dropout of hidden states is the stock modules' own)
