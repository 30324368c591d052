"""The encoder's packed forward (ah_rag.packed_encoder): the operators in the order in which a model uses them,
against the padded forward of the same weights and against a 64-bit restatement."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from oracle import packed_ref as ref


class Weights(torch.nn.Module):
    """A module that holds parameters under dotted names, with a config."""

    def __init__(self, cfg, shapes, seed, dtype, scale=0.08):
        super().__init__()
        self.config = SimpleNamespace(**cfg)
        g = torch.Generator().manual_seed(seed)
        for name, shape in shapes.items():
            at = self
            *path, leaf = name.split(".")
            for part in path:
                if not hasattr(at, part):
                    at.add_module(part, torch.nn.Module())
                at = getattr(at, part)
            x = torch.randn(shape, generator=g) * scale
            if "norm" in name:
                x = x + 1
            at.register_parameter(leaf, torch.nn.Parameter(x.to(dtype)))


def causal(heads=4, kv_heads=2, dim=64, hidden=192, ff=320, layers=2, vocab=500, dtype=torch.bfloat16, **more):
    cfg = dict(num_attention_heads=heads, num_key_value_heads=kv_heads, head_dim=dim, hidden_size=hidden, num_hidden_layers=layers,
               rms_norm_eps=1e-6, hidden_act="silu", rope_parameters={"rope_type": "default", "rope_theta": 1e6}, **more)
    s = {"embed_tokens.weight": (vocab, hidden), "norm.weight": (hidden,)}
    for i in range(layers):
        b = f"layers.{i}."
        s.update({b + "self_attn.q_proj.weight": (heads * dim, hidden), b + "self_attn.k_proj.weight": (kv_heads * dim, hidden),
                  b + "self_attn.v_proj.weight": (kv_heads * dim, hidden), b + "self_attn.o_proj.weight": (hidden, heads * dim),
                  b + "self_attn.q_norm.weight": (dim,), b + "self_attn.k_norm.weight": (dim,), b + "input_layernorm.weight": (hidden,),
                  b + "post_attention_layernorm.weight": (hidden,), b + "mlp.gate_proj.weight": (ff, hidden),
                  b + "mlp.up_proj.weight": (ff, hidden), b + "mlp.down_proj.weight": (hidden, ff)})
    return Weights(cfg, s, 5, dtype)


def causal64(model, ids, weights):
    """Mean of the last hidden states, from the definitions, in 64 bits, one sequence at a time."""
    c, w = model.config, weights
    out = []
    rms = lambda x, g: x * torch.rsqrt((x * x).mean(-1, keepdim=True) + c.rms_norm_eps) * g  # noqa: E731
    half = c.head_dim // 2
    for s in ids:
        n = len(s)
        a = torch.arange(n, dtype=torch.float64)[:, None] * c.rope_parameters["rope_theta"] ** (-torch.arange(half, dtype=torch.float64) / half)
        cos, sin = a.cos()[:, None], a.sin()[:, None]
        turn = lambda x: torch.cat((x[..., :half] * cos - x[..., half:] * sin, x[..., half:] * cos + x[..., :half] * sin), -1)  # noqa: E731
        x = w["embed_tokens.weight"][torch.tensor(s)]
        hide = ~ref.visible(n, n, True)
        for i in range(c.num_hidden_layers):
            b = f"layers.{i}."
            y = rms(x, w[b + "input_layernorm.weight"])
            q, k, v = ((y @ w[b + f"self_attn.{m}_proj.weight"].T).view(n, -1, c.head_dim) for m in "qkv")
            q, k = turn(rms(q, w[b + "self_attn.q_norm.weight"])), turn(rms(k, w[b + "self_attn.k_norm.weight"]))
            g = c.num_attention_heads // c.num_key_value_heads
            k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
            p = torch.einsum("ihd,jhd->hij", q, k) * c.head_dim ** -0.5
            o = torch.einsum("hij,jhd->ihd", torch.softmax(p.masked_fill(hide, -torch.inf), -1), v)
            x = x + o.flatten(1) @ w[b + "self_attn.o_proj.weight"].T
            y = rms(x, w[b + "post_attention_layernorm.weight"])
            x = x + (torch.nn.functional.silu(y @ w[b + "mlp.gate_proj.weight"].T) * (y @ w[b + "mlp.up_proj.weight"].T)) @ w[b + "mlp.down_proj.weight"].T
        out.append(rms(x, w["norm.weight"]).mean(0))
    return torch.stack(out)


def _ids(lens, seed=1, vocab=500, prefix=()):
    rng = np.random.default_rng(seed)
    return [list(prefix) + rng.integers(0, vocab, n).tolist() for n in lens]


def _off(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


# ---- without a GPU -----------------------------------------------------------------------------


def test_common_prefix():
    from ah_rag.packed_encoder import common_prefix
    assert common_prefix([]) == 0 and common_prefix([[1, 2, 3]]) == 0
    assert common_prefix([[1, 2, 3], [1, 2, 4], [1, 2, 3, 9]]) == 2
    assert common_prefix([[1, 2], [1, 2, 4]]) == 1  # each keeps a token of its own
    assert common_prefix([[5], [5]]) == 0 and common_prefix([[1, 2], [3]]) == 0 and common_prefix([[], [1]]) == 0


def test_unknown_layouts_are_refused():
    from ah_rag.packed_encoder import PackedTransformer, UnsupportedLayoutError
    dev = torch.device("cuda", 0)
    PackedTransformer(causal(), dev)  # (weights are only looked at)
    bad = [causal(dtype=torch.float32), causal(dim=68), causal(dim=160), causal(heads=3), causal(use_sliding_window=True, sliding_window=64)]
    m = causal()
    m.config.rope_parameters = {"rope_type": "yarn", "rope_theta": 1e4}
    bad.append(m)
    m = causal()
    m.config.hidden_act = "mish"
    bad.append(m)
    m = causal()
    m.layers._modules["0"].self_attn.q_norm.weight = torch.nn.Parameter(torch.ones(256, dtype=torch.bfloat16))  # of all heads at once
    bad.append(m)
    bad.append(Weights(dict(num_attention_heads=2, num_hidden_layers=1, hidden_size=8), {"some.other.weight": (3, 3)}, 1, torch.bfloat16))
    for m in bad:
        with pytest.raises(UnsupportedLayoutError):
            PackedTransformer(m, dev)


def post(hidden=64, heads=2, layers=2, vocab=50, positions=20, dtype=torch.bfloat16, more=(), **cfg):
    """Parameters of the bidirectional layout; `more`: further ones, name -> shape."""
    names = ("attention.self.query", "attention.self.key", "attention.self.value", "attention.output.dense", "attention.output.LayerNorm",
             "intermediate.dense", "output.dense", "output.LayerNorm")
    s = {"embeddings.word_embeddings.weight": (vocab, hidden), "embeddings.position_embeddings.weight": (positions, hidden),
         "embeddings.LayerNorm.weight": (hidden,), "embeddings.LayerNorm.bias": (hidden,)}
    for i in range(layers):
        for n in names:
            shape = (hidden,) if "Norm" in n else (hidden, hidden)
            s.update({f"encoder.layer.{i}.{n}.weight": shape, f"encoder.layer.{i}.{n}.bias": (hidden,)})
    s.update(more)
    return Weights(dict(num_attention_heads=heads, num_hidden_layers=layers, hidden_size=hidden, layer_norm_eps=1e-12, hidden_act="gelu", **cfg),
                   s, 4, dtype)


def test_parameters_and_settings_that_the_forward_does_not_have_are_refused():
    from ah_rag.packed_encoder import PackedTransformer, UnsupportedLayoutError
    dev = torch.device("cuda", 0)
    PackedTransformer(post(), dev)
    PackedTransformer(post(more={"pooler.dense.weight": (64, 64), "embeddings.token_type_embeddings.weight": (2, 64)}), dev)
    PackedTransformer(causal(layer_types=["full_attention"] * 2, residual_multiplier=1.0), dev)
    bad = [post(more={"embeddings_project.weight": (64, 64)}), post(more={"encoder.layer.0.crossattention.self.query.weight": (64, 64)}),
           post(layers=1, more={"encoder.layer.1.output.dense.weight": (64, 64)}), post(is_decoder=True), post(position_embedding_type="relative_key"),
           causal(layer_types=["full_attention", "sliding_attention"]), causal(residual_multiplier=0.2), causal(attn_logit_softcapping=30.0),
           causal(is_causal=False), causal(use_bidirectional_attention=True)]
    m = causal()
    m.layers._modules["1"].register_parameter("layer_scale", torch.nn.Parameter(torch.ones(3, dtype=torch.bfloat16)))
    bad.append(m)
    m = causal()
    del m.layers._modules["1"]._modules["input_layernorm"]
    bad.append(m)
    for m in bad:
        with pytest.raises(UnsupportedLayoutError):
            PackedTransformer(m, dev)


def test_ids_and_lengths_past_the_tables_are_refused():
    from ah_rag.packed_encoder import PackedTransformer
    dev = torch.device("cuda", 0)
    for m, ids in ((causal(), [[3, 500]]), (causal(), [[3], [-1, 2]]), (post(), [[50]]), (post(), [[1] * 21, [2]]),
                   (causal(), [[7] * 30 + [1], [7] * 30 + [900]])):
        with torch.inference_mode(), pytest.raises(ValueError, match="must lie|longer"):
            PackedTransformer(m, dev).pooled(ids, False)


# ---- on the GPU --------------------------------------------------------------------------------


def _texts(n=120, seed=3):
    rng = np.random.default_rng(seed)
    words = ["film", "director", "Tim", "Burton", "river", "city", "album", "band", "war", "novel", "Paris", "bridge", "1984", "of", "the"]
    return ["Entity: " + " ".join(rng.choice(words, size=int(rng.integers(1, 90)))) + "." for _ in range(n)]


@pytest.mark.gpu
@pytest.mark.parametrize("model", ["all-MiniLM-L6-v2", "all-mpnet-base-v2"])
def test_packed_encode_is_the_padded_one(cuda, model):
    """The same weights and texts through both forwards: 16-bit rounding apart. Order and batch size regroup rows only."""
    from ah_rag.encoder import TorchEncoder
    texts = _texts()
    a, b = TorchEncoder(model, cuda), TorchEncoder(model, cuda, packed=True)
    va, vb = (e.encode(texts, normalize_embeddings=True) for e in (a, b))
    assert vb.shape == va.shape and vb.dtype == np.float32 and np.abs(np.linalg.norm(vb, axis=1) - 1).max() < 1e-5
    assert (np.sum(va * vb, axis=1) > 0.999).all()
    rev = b.encode(texts[::-1], normalize_embeddings=True, batch_size=7)[::-1]
    assert (np.sum(vb * rev, axis=1) > 0.999).all()
    one = b.encode(texts[0], normalize_embeddings=True)
    assert one.shape == (b.dim,) and float(np.dot(one, vb[0])) > 0.999
    u, w = b.encode(texts[:4]), a.encode(texts[:4])
    assert np.linalg.norm(u - w) < 0.05 * np.linalg.norm(w)
    # a prompt is text in front
    p = b.encode(texts[:5], prompt="query: ", convert_to_tensor=True)
    q = b.encode(["query: " + t for t in texts[:5]], convert_to_tensor=True)
    assert torch.equal(p, q) and b.encode([]).shape == (0, b.dim)


@pytest.mark.gpu
def test_packed_mode_of_load_encoder(cuda, monkeypatch):
    from ah_rag.embeddings import load_encoder
    monkeypatch.setenv("AHR_ENCODER", "packed")
    enc = load_encoder("all-MiniLM-L6-v2")
    assert enc.packed is not None and enc is load_encoder("all-MiniLM-L6-v2")
    monkeypatch.setenv("AHR_ENCODER", "torch")
    assert load_encoder("all-MiniLM-L6-v2").packed is None


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(4, 2, 64, torch.bfloat16), (6, 1, 40, torch.float16), (4, 4, 128, torch.float16)])
def test_causal_model_against_64_bits(cuda, heads, kv_heads, dim, dtype):
    """Two layers: each rounds about a dozen intermediate rows to the type, half a step each, which at random add up
    like their square root: 16 half steps are far above that and far below any wrong term (of order one)."""
    from ah_rag.packed_encoder import PackedTransformer
    m = causal(heads, kv_heads, dim, dtype=dtype)
    w64 = {n: p.detach().double() for n, p in m.named_parameters()}
    t = PackedTransformer(m.to(cuda), cuda)
    bound = 16 * ref.half_step(dtype)
    for ids in (_ids([1]), _ids([5, 33, 1, 64, 130]), _ids([9, 1, 20, 70], prefix=range(40)), _ids([3, 3], prefix=range(200))):
        want = causal64(m, ids, w64)
        with torch.inference_mode():
            assert _off(t.pooled(ids, False), want) < bound
            y = t.pooled(ids, True)
        assert _off(y, want / want.norm(dim=1, keepdim=True)) < bound
        assert (y.norm(dim=1) - 1).abs().max() < 1e-5
    # the shared prefix is what it is without sharing
    ids = _ids([9, 1, 20, 70], prefix=range(40))
    with torch.no_grad():
        h, layout = t.hidden_states(ids)
        from ah_rag.packed import packed_mean_pool
        a, b = t.pooled(ids, False), packed_mean_pool(h, layout)
    assert _off(a, b.double().cpu()) < bound


@pytest.mark.gpu
def test_gradients_of_a_training_step(cuda):
    """A loss on the pooled vectors: the gradients of all the parameters against 64 bits, after an encode() in
    inference mode that shares the caches, and the joint projections after refresh()."""
    from ah_rag.packed_encoder import PackedTransformer
    m = causal(4, 2, 64, dtype=torch.bfloat16)
    w64 = {n: p.detach().double().requires_grad_() for n, p in m.named_parameters()}
    t = PackedTransformer(m.to(cuda), cuda)
    ids = _ids([7, 40, 65, 1, 100])
    with torch.inference_mode():
        before = t.pooled(ids, False)
    d = torch.randn(len(ids), 192, generator=torch.Generator().manual_seed(2))
    loss = (t.pooled(ids, True) * d.to(cuda)).sum()
    names = [n for n, _ in m.named_parameters()]
    grads = torch.autograd.grad(loss, [p for _, p in m.named_parameters()])
    want = causal64(m, ids, w64)
    loss64 = (want / want.norm(dim=1, keepdim=True) * d.double()).sum()
    grads64 = torch.autograd.grad(loss64, [w64[n] for n in names])
    for n, a, b in zip(names, grads, grads64):
        # the forward's roundings and as many of the backward's: 32 half steps
        assert _off(a, b) < 32 * ref.half_step(torch.bfloat16), n
    with torch.no_grad():
        for _, p in m.named_parameters():
            p.mul_(1.25)
    t.refresh()
    w64 = {n: p.detach().double().cpu() for n, p in m.named_parameters()}
    with torch.inference_mode():
        after = t.pooled(ids, False)
    assert _off(after, causal64(m, ids, w64)) < 16 * ref.half_step(torch.bfloat16) and not torch.equal(after, before)


@pytest.mark.gpu
@pytest.mark.parametrize("make", [causal, post])
def test_written_weights_are_noticed(cuda, make):
    """The joint projections follow writes to the weights: an optimizer's, and a loaded state dict."""
    from ah_rag.packed_encoder import PackedTransformer
    m = make().to(cuda)
    t = PackedTransformer(m, cuda)
    ids = _ids([7, 12, 1], vocab=50)
    old = {n: p.detach().clone() for n, p in m.named_parameters()}
    with torch.inference_mode():
        before = t.pooled(ids, False)
    opt = torch.optim.SGD(m.parameters(), lr=0.5)
    t.pooled(ids, True).square().sum(0)[:8].sum().backward()
    opt.step()
    with torch.inference_mode():
        after = t.pooled(ids, False)
        t.refresh()
        assert torch.equal(after, t.pooled(ids, False)) and not torch.equal(after, before)
    m.load_state_dict(old)
    with torch.inference_mode():
        assert torch.equal(t.pooled(ids, False), before)


@pytest.mark.gpu
def test_embed_of_the_bidirectional_encoder(cuda):
    """embed() gives encode()'s vectors, with gradients to the embeddings and every layer."""
    from ah_rag.encoder import TorchEncoder
    enc = TorchEncoder("all-MiniLM-L6-v2", cuda, packed=True)
    texts = _texts(12)
    y = enc.embed(texts, normalize_embeddings=True)
    v = enc.encode(texts, normalize_embeddings=True, convert_to_tensor=True)
    assert ((y.detach() * v).sum(1) > 0.999).all()
    (y * torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(cuda)).sum().backward()
    for n, p in enc.model.named_parameters():
        assert p.grad is not None and p.grad.isfinite().all(), n
    with pytest.raises(ValueError, match="packed"):
        TorchEncoder("all-MiniLM-L6-v2", cuda).embed(texts)
