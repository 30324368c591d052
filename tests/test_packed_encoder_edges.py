"""Edges of the encoder's packed forward (ah_rag.packed_encoder)."""
import pytest
import torch

from oracle import packed_ref as ref
from test_packed_encoder import _ids, _off, causal, post

DEV = torch.device("cuda", 0)


# ---- without a GPU -----------------------------------------------------------------------------


@pytest.mark.parametrize("make", ["post", "causal"])
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_gradients_of_the_biases_alone(make, which):
    """The projections of a model whose biases alone are trained (all weights frozen): their gradients in 64 bits."""
    from ah_rag.packed_encoder import PackedTransformer
    if make == "post":
        m = post()
        name = "encoder.layer.1.attention.self.%s.bias" % {"q": "query", "k": "key", "v": "value"}[which]
    else:
        m = causal()
        for p in "qkv":
            at = getattr(m.layers._modules["1"].self_attn, p + "_proj")
            at.register_parameter("bias", torch.nn.Parameter(torch.zeros(at.weight.shape[0], dtype=torch.bfloat16)))
        name = f"layers.1.self_attn.{which}_proj.bias"
    m.requires_grad_(False)
    t = PackedTransformer(m, DEV)
    bias = dict(m.named_parameters())[name].requires_grad_()
    x = torch.randn(7, m.config.hidden_size, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    with torch.no_grad():
        t._qkv(1, x)  # (a forward without gradients before)
    y = t._qkv(1, x)["qkv".index(which)]
    d = torch.randn(y.shape, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    got, = torch.autograd.grad(y, bias, d)
    want = d.double().flatten(1).sum(0)
    # a sum of 7 values in fp32 at least, or in bf16 at worst: 7 roundings of the absolute sum
    assert ((got.double() - want).abs() <= 7 * ref.half_step(torch.bfloat16) * d.double().flatten(1).abs().sum(0)).all()
