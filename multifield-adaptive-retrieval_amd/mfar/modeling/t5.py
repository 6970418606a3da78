"""Forward pass of a T5 encoder with the fused attention (mfar/modeling/attention.py), over the modules and parameters of the stock model.

The stock attention materialises a bias and a score tensor of heads x queries x keys per layer and adds the mask to them; here each layer is three
projections, one kernel and the output projection, and the bias table's gradient comes out of the attention's backward pass.  Parameters,
checkpoints and everything around the attention (norms, feed-forward, dropout of the hidden states) are the stock model's.
"""
import torch

from mfar.modeling.attention import relative_bias_attention


def t5_stack(auto_model: torch.nn.Module) -> torch.nn.Module:
    """The encoder stack of a T5 model whose layers this forward can run; ValueError for anything else."""
    stack = getattr(auto_model, "encoder", auto_model)
    blocks = getattr(stack, "block", None)
    try:
        first = blocks[0].layer[0].SelfAttention
        ok = first.has_relative_attention_bias and not first.is_decoder and hasattr(stack, "embed_tokens") and hasattr(stack, "final_layer_norm")
    except (AttributeError, IndexError, TypeError):
        ok = False
    if not ok:
        raise ValueError(f"{type(auto_model).__name__} is no T5 encoder with a relative attention bias")
    return stack


def attention_dropout(stack: torch.nn.Module) -> float:
    """Probability that the layers drop attention weights with while training."""
    return max(float(b.layer[0].SelfAttention.dropout) for b in stack.block)


def stays_stock(auto_model: torch.nn.Module, stack: torch.nn.Module) -> str:
    """Why a forward of this model, as it stands, is the stock model's to run; empty: the fused one runs it."""
    if getattr(auto_model, "encoder", auto_model) is not stack:
        return "the encoder's model is another than the one it was switched on for"
    if stack.training and attention_dropout(stack) > 0:
        return "the encoder is in training mode and drops attention weights, which the kernel does not"
    if stack.training and any(getattr(m, "gradient_checkpointing", False) for m in (stack, *stack.block)):
        return "gradient checkpointing is on, which goes through the stock blocks"
    for m in (auto_model, *_passed_by(stack)):
        if m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks or "forward" in vars(m):
            return f"a {type(m).__name__} that it passes by has hooks or a forward of its own"
    return ""


def _passed_by(stack: torch.nn.Module):
    """The modules whose own forward the fused one does not call."""
    yield stack
    for block in stack.block:
        yield block
        yield block.layer[0]
        yield block.layer[0].SelfAttention
    yield stack.block[0].layer[0].SelfAttention.relative_attention_bias


def _held(h: torch.Tensor) -> torch.Tensor:
    """Hidden states of an fp16 model stay within the type, as the stock blocks keep them: a sum past the largest value would be infinite, and NaN
    from the next norm on."""
    return h if h.dtype != torch.float16 else h.clamp(-65504.0, 65504.0)


def t5_encoder_forward(stack: torch.nn.Module, input_ids: torch.Tensor, attention_mask: torch.Tensor) -> torch.Tensor:
    """Token ids [B, L] and their mask (0: padding) -> hidden states [B, L, d].  No attention weight is dropped."""
    mask = attention_mask.ne(0)
    B, L = input_ids.shape
    h = stack.dropout(stack.embed_tokens(input_ids))
    first = stack.block[0].layer[0].SelfAttention
    table = first.relative_attention_bias.weight                          # [buckets, heads], shared by all layers
    max_distance = int(first.relative_attention_max_distance)
    for block in stack.block:
        layer = block.layer[0]
        att = layer.SelfAttention
        x = layer.layer_norm(h)
        heads = (B, L, att.n_heads, att.key_value_proj_dim)
        o = relative_bias_attention(att.q(x).view(heads), att.k(x).view(heads), att.v(x).view(heads), table, key_mask=mask, max_distance=max_distance)
        h = _held(h + layer.dropout(att.o(o.reshape(B, L, -1))))
        h = _held(block.layer[-1](h))                                          # the feed-forward with its norm, dropout and residual
    return stack.dropout(stack.final_layer_norm(h))
