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


def _tiny(model_type, **more):
    """A model of that type with random weights, small enough for the CPU."""
    from transformers import AutoConfig, AutoModel
    c = AutoConfig.for_model(model_type)
    small = dict(hidden_size=64, num_hidden_layers=2, num_attention_heads=4, intermediate_size=96, vocab_size=50, max_position_embeddings=40,
                 num_key_value_heads=2, head_dim=16, embedding_size=64)
    for n, x in {**{n: x for n, x in small.items() if hasattr(c, n)}, **more}.items():
        setattr(c, n, x)
    if getattr(c, "layer_types", None):
        c.layer_types = ["full_attention"] * 2
    c._attn_implementation = "eager"
    torch.manual_seed(7)
    m = AutoModel.from_config(c)
    with torch.no_grad():
        for p in m.parameters():  # (biases and norms too, so that none goes unseen)
            p.add_(0.05 * torch.randn(p.shape))
    return m.to(torch.bfloat16).eval()


class _Layout:
    """What the forward reads of a layout, on the host."""

    def __init__(self, lengths):
        self.lengths = torch.tensor(lengths).numpy()

    def __len__(self):
        return len(self.lengths)

    def positions(self):
        return torch.cat([torch.arange(n, dtype=torch.int32) for n in self.lengths.tolist()])


def _plain_operators(monkeypatch):
    """The forward on the CPU: the operators' 64-bit restatement in the place of the kernels."""
    from ah_rag import packed_encoder

    def attention(q, k, v, layout, causal=False):
        lens = layout.lengths.tolist()
        return ref.attention(q, k, v, lens, lens, causal, q.shape[2] ** -0.5)[0].to(q.dtype)

    def rope(q, k, wq, wk, cos, sin, positions, eps):
        return tuple(ref.rotate(x, w, cos, sin, positions, eps, False).to(x.dtype) for x, w in ((q, wq), (k, wk)))

    monkeypatch.setattr(packed_encoder, "packed_attention", attention)
    monkeypatch.setattr(packed_encoder, "qk_norm_rope", rope)


@pytest.mark.parametrize("model_type", ["bert", "bert-generation", "electra", "ernie", "splinter", "qwen3", "qwen3_vl_text"])
def test_accepted_models_give_their_own_hidden_states(monkeypatch, model_type):
    """The forward over packed tokens against the model's own, one sequence at a time. Both round some twenty rows of
    each layer to bf16 (half a step each), which at random add up like their square root: 16 half steps are well above
    that and far below a wrong position, norm or mask (of order one)."""
    from ah_rag.packed_encoder import PackedTransformer
    m = _tiny(model_type)
    _plain_operators(monkeypatch)
    t = PackedTransformer(m, torch.device("cpu"))
    ids = _ids([5, 17, 1, 33], vocab=50)
    with torch.no_grad():
        x = (t._post if t.kind == "post" else t._causal)(torch.tensor([i for s in ids for i in s]), _Layout([len(s) for s in ids]))
        want = torch.cat([m(input_ids=torch.tensor([s])).last_hidden_state[0] for s in ids])
    assert _off(x, want.double()) < 16 * ref.half_step(torch.bfloat16)


@pytest.mark.parametrize("model_type", ["roberta", "xlm-roberta", "camembert", "data2vec-text", "ibert", "mra", "yoso", "big_bird"])
def test_models_with_other_positions_or_attention_are_refused(model_type):
    """Their parameters have the names of the bidirectional layout, but their positions do not start at 0 (or their
    attention is another)."""
    from ah_rag.packed_encoder import PackedTransformer, UnsupportedLayoutError
    with pytest.raises(UnsupportedLayoutError):
        PackedTransformer(_tiny(model_type), DEV)


def test_a_padded_position_table_is_refused():
    """A position table with a padding row gives the first token a position after it, whatever the model calls itself."""
    from ah_rag.packed_encoder import PackedTransformer, UnsupportedLayoutError
    m = post()
    w = m.embeddings.position_embeddings.weight
    m.embeddings.position_embeddings = torch.nn.Embedding(*w.shape, padding_idx=1, dtype=w.dtype)
    with pytest.raises(UnsupportedLayoutError, match="positions"):
        PackedTransformer(m, DEV)


def _frozen(model):
    return model.requires_grad_(False)


@pytest.mark.parametrize("joins", [False, True])
@pytest.mark.parametrize("make", [causal, post])
def test_projections_follow_every_write_to_the_weights(monkeypatch, make, joins):
    """In place, through .data, to inference tensors, by a loaded state dict: the next forward computes with what stands in
    the weights, with each layer's projections joined for it or apart."""
    from ah_rag import packed_encoder
    from ah_rag.packed_encoder import PackedTransformer
    if not joins:
        monkeypatch.setattr(packed_encoder, "JOIN_UP_TO", 0)
    with torch.inference_mode():
        held = _frozen(make())
    for m in (_frozen(make()), held):
        t = PackedTransformer(m, torch.device("cpu"))
        prefix, names = t.fused[1]
        w, b = (dict(m.named_parameters()).get(prefix + names[1] + s) for s in (".weight", ".bias"))
        x = torch.randn(5, m.config.hidden_size, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)

        def keys():
            with torch.inference_mode():
                joined = t._joined()
                assert (joined is not None) == joins
                got = t._qkv(1, x, joined)[1].clone()
                assert _off(got.flatten(1), x.double() @ w.double().T + (0 if b is None else b.double())) < 2 * ref.half_step(torch.bfloat16)
                return got

        first = keys()
        with torch.inference_mode():
            w.add_(0.5)
        second = keys()
        w.data.mul_(2.0)
        third = keys()
        assert not torch.equal(first, second) and not torch.equal(second, third)
        if m is not held:
            m.load_state_dict({n: p.detach() * 0.5 for n, p in m.named_parameters()})
            assert not torch.equal(third, keys())


@pytest.mark.parametrize("make", [causal, post])
def test_joined_projections_give_what_three_products_give(make):
    """One product over the three projections of a layer, or three: each value a sum in fp32 that is rounded once."""
    from ah_rag.packed_encoder import PackedTransformer
    m = make()
    t = PackedTransformer(m, torch.device("cpu"))
    assert t._joined() is None  # (the weights' gradients are wanted)
    x = torch.randn(5, m.config.hidden_size, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    with torch.no_grad():
        for i in range(t.layers):
            for a, b in zip(t._qkv(i, x, t._joined()), t._qkv(i, x)):
                assert a.shape == b.shape and _off(a, b.double()) < 2 * ref.half_step(torch.bfloat16)
    m.requires_grad_(False)
    assert t._joined() is not None
    list(m.parameters())[-1].requires_grad_()
    assert t._joined() is not None
    t.w[t.fused[0][0] + t.fused[0][1][1] + ".weight"].requires_grad_()
    assert t._joined() is None
    if make is causal:  # a bias in one layer alone: three products
        m.layers._modules["0"].self_attn.k_proj.register_parameter("bias", torch.nn.Parameter(torch.ones(128, dtype=torch.bfloat16)))
        t = PackedTransformer(m, torch.device("cpu"))
        with torch.no_grad():
            assert t._joined() is None and _off(t._qkv(0, x)[1].flatten(1) - 1, (x @ t.w["layers.0.self_attn.k_proj.weight"].T).double()) < 0.02


@pytest.mark.parametrize("make", [causal, post])
def test_replaced_parameters_are_used(make):
    """Parameters that other ones have taken the place of (a state dict assigned, an attribute set): the forward reads and
    trains the model's, not those that it had first."""
    from ah_rag.packed_encoder import PackedTransformer
    m = make()
    t = PackedTransformer(m, torch.device("cpu"))
    old = t.w[t.fused[1][0] + t.fused[1][1][0] + ".weight"]
    m.load_state_dict({n: p.detach() * 2 for n, p in m.named_parameters()}, assign=True)
    assert all(t.w[n] is p for n, p in m.named_parameters()) and set(t.w) == {n for n, _ in m.named_parameters()}
    x = torch.randn(5, m.config.hidden_size, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    y = t._qkv(1, x)[0]
    d = torch.randn(y.shape, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    new = t.w[t.fused[1][0] + t.fused[1][1][0] + ".weight"]
    grad, = torch.autograd.grad(y, new, d)
    assert new is not old and _off(grad, d.double().flatten(1).T @ x.double()) < 2 * ref.half_step(torch.bfloat16)
    with torch.no_grad():
        assert _off(t._qkv(1, x, t._joined())[0], y.double()) < 2 * ref.half_step(torch.bfloat16)


def test_a_rotary_table_is_long_enough_whatever_another_thread_stores():
    """Another thread stores a shorter table between the look at its length and its use: the call goes on with one of the
    length that it asked for (rows past a shorter one would be NaN)."""
    from ah_rag.packed_encoder import PackedTransformer
    t = PackedTransformer(causal(), torch.device("cpu"))
    t._rotary(700)
    long, short = t._table, (torch.zeros(512, 32), torch.zeros(512, 32), *t._table[2:])

    for swap_at in (1, 2, 3):
        class Swapped(PackedTransformer):
            looks = 0

            @property
            def _table(self):
                self.looks += 1
                return long if self.looks < swap_at else short

            @_table.setter
            def _table(self, new):
                pass

        t.__dict__.pop("_table", None)
        t.__dict__.pop("looks", None)
        t.__class__ = Swapped
        assert all(x.shape[0] >= 650 for x in t._rotary(650)[:2]), swap_at


@pytest.mark.parametrize("make", [causal, post])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("ids", [[], [[]], [[], []]], ids=str)
def test_batches_without_tokens(monkeypatch, make, grad, ids):
    """No text, or texts without a token (an empty string, where the tokenizer adds none): no rows."""
    from ah_rag.packed_encoder import PackedTransformer
    _plain_operators(monkeypatch)
    m = make()
    t = PackedTransformer(m, torch.device("cpu"))

    class Layout(_Layout):
        def positions(self):
            return torch.zeros(0, dtype=torch.int32)

    with torch.set_grad_enabled(grad):
        x = (t._post if t.kind == "post" else t._causal)(torch.zeros(0, dtype=torch.int64), Layout([0] * len(ids)))
    assert x.shape == (0, m.config.hidden_size)


def test_rotary_settings_that_the_forward_does_not_have_are_refused():
    from ah_rag.packed_encoder import PackedTransformer, UnsupportedLayoutError
    m = causal()
    m.config.rope_parameters = {"full_attention": {"rope_type": "default", "rope_theta": 1e4}}  # for each type of layer
    for bad in (m, causal(partial_rotary_factor=0.5)):
        with pytest.raises(UnsupportedLayoutError, match="rotary"):
            PackedTransformer(bad, DEV)
    PackedTransformer(causal(partial_rotary_factor=1.0), DEV)


def test_embed_of_one_string_is_refused():
    """(It would be taken for a list of its letters.)"""
    from ah_rag.encoder import TorchEncoder
    enc = object.__new__(TorchEncoder)
    enc.packed = object()
    with pytest.raises(ValueError, match="list of texts"):
        enc.embed("a river")


# ---- on the GPU --------------------------------------------------------------------------------


@pytest.mark.gpu
def test_a_fresh_encoder_on_two_streams(cuda):
    """The first calls of an encoder at once from two threads, each on a stream of its own, with writes to the weights
    between rounds: every result is that of one call alone."""
    import threading

    from ah_rag.encoder import TorchEncoder
    texts = ["Entity: " + "river city album " * (1 + i % 20) for i in range(60)]
    for rnd in range(3):
        enc = TorchEncoder("all-MiniLM-L6-v2", cuda, packed=True)
        with torch.inference_mode():
            assert enc.packed._joined() is not None
        for change in range(3):
            if change:
                with torch.no_grad():
                    for p in enc.model.parameters():
                        p.data.mul_(1.0 + 0.01 * change)
                torch.cuda.synchronize()
            got, errors = {}, []

            def work(i):
                try:
                    s = torch.cuda.Stream()
                    with torch.cuda.stream(s):
                        y = enc.encode(texts, normalize_embeddings=True, convert_to_tensor=True)
                        s.synchronize()
                        got[i] = y.cpu()
                except Exception as e:  # noqa: BLE001
                    errors.append(e)

            threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
            for t in threads:
                t.start()
            for t in threads:
                t.join()
            assert not errors, errors
            want = enc.encode(texts, normalize_embeddings=True, convert_to_tensor=True).cpu()
            for y in got.values():
                assert torch.equal(y, want)


@pytest.mark.gpu
def test_a_replaced_rotary_table_outlives_its_readers(cuda):
    """A longer text on one stream replaces the table that another stream still waits to read: its memory is not handed out
    before."""
    from ah_rag.packed_encoder import PackedTransformer
    t = PackedTransformer(causal(layers=1).to(cuda), cuda)
    side = torch.cuda.Stream()
    with torch.inference_mode():
        want = torch.cat(t._rotary(300))
        fresh = [torch.full((512, 32), 1.0, device=cuda) for _ in range(64)]
        del fresh
        torch.cuda.synchronize()
        old = {x.data_ptr() for x in t._rotary(300)}
        with torch.cuda.stream(side):
            torch.cat(t._rotary(300))
            torch.cuda._sleep(1_000_000_000)  # (a finite wait on the device's clock)
            got = torch.cat(t._rotary(300))
        t._rotary(900)  # a longer table here, which lets the old one go
        # memory of the old table's size: none of it may be the old table's while the side stream still reads that
        fresh = [torch.full((512, 32), float("nan"), device=cuda) for _ in range(64)]
        assert not side.query() and not {f.data_ptr() for f in fresh} & old
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("make", [causal, post])
def test_texts_without_tokens(cuda, make):
    """Zeros for a text without tokens (the mean of no rows), alone or among others, and zero gradients."""
    from ah_rag.packed_encoder import PackedTransformer
    m = make().to(cuda)
    t = PackedTransformer(m, cuda)
    some = _ids([4, 7], vocab=50)
    for ids in ([], [[]], [[], []], [[], some[0], [], some[1]]):
        with torch.inference_mode():
            y = t.pooled(ids, True)
            alone = t.pooled([s for s in ids if s], True)
        assert y.shape == (len(ids), m.config.hidden_size) and y.dtype == torch.float32
        assert torch.equal(y[[i for i, s in enumerate(ids) if s]], alone) and not y[[i for i, s in enumerate(ids) if not s]].any()
        grads = torch.autograd.grad(t.pooled(ids, False).sum(), list(m.parameters()), allow_unused=True)
        assert all(g is None or g.isfinite().all() for g in grads)
