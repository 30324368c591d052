"""Packed-sequence operators on the GPU against their 64-bit restatement (oracle/packed_ref.py), within
bounds that the restatement derives from the roundings the arithmetic allows."""
import math

import pytest
import torch

from oracle import packed_ref as ref

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16

# (query lengths, key lengths or None, heads, key heads, head_dim, causal, type)
SHAPES = [
    ([1], None, 1, 1, 8, False, BF),
    ([1], None, 3, 1, 64, True, HF),
    ([5, 0, 17], None, 12, 12, 32, False, BF),
    ([31, 32, 33], None, 2, 2, 32, True, HF),
    ([63, 64, 65, 1], None, 4, 4, 64, False, BF),
    ([129, 7, 200], None, 12, 12, 64, False, HF),
    ([129, 7, 200], None, 6, 2, 64, True, BF),
    ([300, 1, 2], None, 5, 1, 128, True, BF),
    ([250], None, 4, 2, 128, False, HF),
    ([70, 130], None, 6, 3, 96, True, HF),
    ([70, 130], None, 4, 1, 80, False, BF),
    ([33, 100], None, 4, 4, 48, True, BF),
    ([65, 40], None, 2, 1, 112, True, BF),
    ([77, 40], None, 2, 1, 40, True, HF),
    ([20], None, 40, 1, 64, True, BF),       # a group wider than one wave's rows
    ([9, 3], None, 100, 1, 32, True, HF),    # and than two waves'
    ([1, 1, 1], [2000, 0, 1301], 8, 2, 128, True, HF),   # single tokens, keys split and joined
    ([1, 2, 5, 1], [700, 3, 1030, 64], 7, 1, 64, True, BF),
    ([3, 1], [500, 900], 4, 4, 32, False, BF),
    ([40, 3, 0], [20, 0, 7], 4, 2, 64, True, BF),        # rows that read no key
    ([40, 3], [20, 0], 4, 2, 64, False, HF),
    ([90, 5], [150, 65], 3, 3, 128, True, HF),           # keys from before the queries
]


def _ids(s):
    return "q%s-k%s-h%d.%d-d%d-%s-%s" % (s[0], s[1], *s[2:5], "causal" if s[5] else "full", str(s[6])[6:])


def _make(shape, seed, dev, fused=True):
    ql, kl, hq, hk, d, causal, dt = shape
    g = torch.Generator().manual_seed(seed)
    t, tk = sum(ql), sum(kl or ql)

    def normal(*s):
        return torch.randn(*s, generator=g).to(dt).to(dev)

    if kl is None and fused:  # views of one projection's output
        qkv = normal(t, hq + 2 * hk, d)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    else:
        q, k, v = normal(t, hq, d), normal(tk, hk, d), normal(tk, hk, d)
    return q, k, v, normal(t, hq, d)


def _within(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol).nan_to_num(1e9).max()):.3g} x the bound"


@pytest.mark.parametrize("shape", SHAPES, ids=_ids)
def test_attention_and_gradients(cuda, shape):
    from ah_rag.packed import PackedLayout, packed_attention
    ql, kl, hq, hk, d, causal, dt = shape
    q, k, v, d_o = _make(shape, 1, cuda)
    lay = PackedLayout(ql, kl, cuda)
    o = packed_attention(q, k, v, lay, causal=causal)
    w_o, t_o, w_g, t_g = ref.attention(q, k, v, ql, kl or ql, causal, d ** -0.5, d_o=d_o)
    _within(o, w_o, t_o, "o")
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    o2 = packed_attention(*leaves, lay, causal=causal)
    _within(o2, w_o, t_o, "o with gradients")
    grads = torch.autograd.grad(o2, leaves, d_o)
    for name, a, w, t in zip(("dq", "dk", "dv"), grads, w_g, t_g):
        assert a.dtype == dt
        _within(a, w, t, name)
    # the same bits again
    again = torch.autograd.grad(packed_attention(*leaves, lay, causal=causal), leaves, d_o)
    for a, b in zip(grads, again):
        assert torch.equal(a, b)


@pytest.mark.parametrize("shape,prefix", [
    (([5, 0, 17, 1], None, 4, 2, 64, True, BF), 1),
    (([5, 9, 17, 1], None, 12, 12, 32, True, HF), 63),
    (([3] * 40, None, 8, 4, 64, True, BF), 700),
    (([1] * 50, [7] * 49 + [0], 16, 4, 128, True, HF), 1500),
    (([200, 190], None, 4, 4, 128, True, BF), 130),
    (([600, 650, 300], None, 24, 12, 96, True, BF), 65),
    (([40, 3], [20, 0], 2, 1, 40, True, BF), 100),
    (([40, 3], [20, 0], 2, 1, 64, False, BF), 0),
    (([2, 2], None, 3, 1, 80, False, HF), 4000),
    (([3] * 40, None, 8, 4, 64, True, BF), 1300),
    (([2, 0, 5, 1] * 20, None, 12, 12, 40, True, HF), 700),
    (([4] * 30, [2] * 30, 4, 2, 64, False, BF), 2000),   # rows that read the prefix alone, and keys short of the queries
    (([4] * 30, [2] * 30, 4, 2, 64, True, BF), 2000),
], ids=lambda x: _ids(x) if isinstance(x, tuple) else "prefix%d" % x)
def test_prefix_attention(cuda, shape, prefix):
    from ah_rag.packed import PackedLayout, prefix_attention
    ql, kl, hq, hk, d, causal, dt = shape
    q, k, v, _ = _make(shape, 2, cuda)
    g = torch.Generator().manual_seed(3)
    both = torch.randn(prefix, 2, hk, d, generator=g).to(dt).to(cuda)
    lay = PackedLayout(ql, kl, cuda)
    o = prefix_attention(q, k, v, both[:, 0], both[:, 1], lay, causal=causal)
    w, t = ref.attention(q, k, v, ql, kl or ql, causal, d ** -0.5, both[:, 0], both[:, 1])
    _within(o, w, t, "o")


@pytest.mark.parametrize("dim,heads,kv_heads,causal", [(64, 12, 12, False), (32, 12, 12, True), (128, 8, 2, True)])
def test_a_batch_of_many_texts(cuda, dim, heads, kv_heads, causal):
    """64 texts of 1 to 384 tokens, as an encoder's batch: tiles of every fill, workgroups at different tiles at once.
    The reference padded, in 64 bits on the GPU; the bound that of the small cases for values of size one."""
    from ah_rag.packed import PackedLayout, packed_attention
    rng = torch.Generator().manual_seed(8)
    lens = torch.randint(1, 385, (64,), generator=rng).tolist()
    q, k, v, d_o = _make((lens, None, heads, kv_heads, dim, causal, BF), 9, cuda)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    o = packed_attention(*leaves, PackedLayout(lens, device=cuda), causal=causal)
    grads = torch.autograd.grad(o, leaves, d_o)
    n = torch.tensor(lens, device=cuda)
    at = torch.arange(384, device=cuda)
    real = at < n[:, None]
    idx = torch.where(real, (torch.cumsum(n, 0) - n)[:, None] + at, 0)
    L = [x.detach().double().requires_grad_() for x in (q, k, v)]
    Q, K, V = (x[idx].transpose(1, 2) for x in L)
    K, V = (x.repeat_interleave(heads // kv_heads, 1) for x in (K, V))
    see = real[:, None, None, :] & (~torch.ones(384, 384, dtype=torch.bool, device=cuda).triu(1) | (not causal))
    p = torch.softmax((Q @ K.transpose(2, 3) * dim ** -0.5).masked_fill(~see, -math.inf), -1)
    w = (p @ V).transpose(1, 2)[real]
    wg = torch.autograd.grad(w, L, d_o.double())
    u = ref.half_step(BF)
    # o: the weights' rounding (u of sum p |v|, here at most u max |v|) and its own; gradients: twice as many roundings of
    # terms that are sums over up to 384 rows of such size
    assert ((o - w).abs() <= u * (w.abs() + 6.0)).all()
    for a, b in zip(grads, wg):
        assert float((a - b).norm() / b.norm()) < 4 * u


def test_one_long_sequence(cuda):
    """Many tiles, a length that ends inside one; the reference by blocks in 64 bits."""
    from ah_rag.packed import PackedLayout, packed_attention
    shape = ([2501, 40], None, 2, 1, 128, True, BF)
    q, k, v, d_o = _make(shape, 5, cuda)
    lay = PackedLayout(shape[0], device=cuda)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    o = packed_attention(*leaves, lay, causal=True)
    g = torch.autograd.grad(o, leaves, d_o)
    w_o, t_o, w_g, t_g = ref.attention(q, k, v, *shape[:1], shape[0], True, 128 ** -0.5, d_o=d_o)
    _within(o, w_o, t_o, "o")
    for name, a, w, t in zip(("dq", "dk", "dv"), g, w_g, t_g):
        _within(a, w, t, name)


@pytest.mark.parametrize("what", ["transposed", "expanded", "odd rows", "strided last", "misaligned"])
def test_attention_takes_any_strides(cuda, what):
    from ah_rag.packed import PackedLayout, packed_attention
    shape = ([33, 70], None, 4, 2, 64, True, BF)
    q, k, v, d_o = _make(shape, 7, cuda, fused=False)
    lay = PackedLayout(shape[0], device=cuda)
    if what == "transposed":  # [heads, tokens, dim] in memory
        q2, k2, v2 = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    elif what == "expanded":  # one head for all
        q, k, v = q[:, :1].expand(-1, 4, -1), k[:, :1].expand(-1, 2, -1), v[:1].expand(103, -1, -1)
        q2, k2, v2 = q, k, v
    elif what == "odd rows":
        q2, k2, v2 = (torch.nn.functional.pad(x.flatten(1), (0, 3))[:, :-3].view(x.shape) for x in (q, k, v))
    elif what == "strided last":
        q2, k2, v2 = (torch.stack((x, x), -1)[..., 0] for x in (q, k, v))
    else:
        q2, k2, v2 = (torch.nn.functional.pad(x.flatten(), (1, 0))[1:].view(x.shape) for x in (q, k, v))
    leaves = [x.detach().requires_grad_() for x in (q2, k2, v2)]
    o = packed_attention(*leaves, lay, causal=True)
    g = torch.autograd.grad(o, leaves, d_o.transpose(0, 1).contiguous().transpose(0, 1))
    w_o, t_o, w_g, t_g = ref.attention(q, k, v, shape[0], shape[0], True, 0.125, d_o=d_o)
    _within(o, w_o, t_o, "o")
    for name, a, w, t in zip(("dq", "dk", "dv"), g, w_g, t_g):
        _within(a, w, t, name)


def test_gradients_of_shared_and_broadcast_inputs(cuda):
    """A broadcast query and one tensor as keys and values: autograd sums what the kernels return."""
    from ah_rag.packed import PackedLayout, packed_attention
    lens, d = [9, 30], 32
    g = torch.Generator().manual_seed(1)
    one = torch.randn(39, 1, d, generator=g).to(BF).to(cuda).requires_grad_()
    kv = torch.randn(39, 2, d, generator=g).to(BF).to(cuda).requires_grad_()
    d_o = torch.randn(39, 4, d, generator=g).to(BF).to(cuda)
    lay = PackedLayout(lens, device=cuda)
    o = packed_attention(one.expand(-1, 4, -1), kv, kv, lay)
    g1, g2 = torch.autograd.grad(o, (one, kv), d_o)
    q = one.detach().expand(-1, 4, -1)
    _, _, (wq, wk, wv), (tq, tk, tv) = ref.attention(q, kv, kv, lens, lens, False, d ** -0.5, d_o=d_o)
    u = ref.half_step(BF)
    _within(g1, wq.sum(1, keepdim=True), tq.sum(1, keepdim=True) + 4 * u * wq.abs().sum(1, keepdim=True), "dq summed over heads")
    _within(g2, wk + wv, tk + tv + u * (wk + wv).abs() * 1.01, "dk + dv")


def test_gradient_against_differences(cuda):
    """d/dt of <o, d_o> along a direction, by differences of the 64-bit oracle around the same inputs."""
    from ah_rag.packed import PackedLayout, packed_attention
    shape = ([23, 41], None, 4, 2, 32, True, BF)
    q, k, v, d_o = _make(shape, 11, cuda)
    lay = PackedLayout(shape[0], device=cuda)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(packed_attention(*leaves, lay, causal=True), leaves, d_o)
    gen = torch.Generator().manual_seed(2)
    _, _, _, t_g = ref.attention(q, k, v, shape[0], shape[0], True, 32 ** -0.5, d_o=d_o)
    for i, name in enumerate("qkv"):
        x = [y.detach().cpu().double() for y in (q, k, v)]
        r = torch.randn(x[i].shape, generator=gen, dtype=torch.float64)
        h = 1e-5
        f = []
        for s in (h, -h):
            y = list(x)
            y[i] = x[i] + s * r
            f.append(float((_plain64(*y, shape[0], True) * d_o.cpu().double()).sum()))
        num = (f[0] - f[1]) / (2 * h)
        got = float((grads[i].cpu().double() * r).sum())
        assert abs(got - num) <= float((t_g[i] * r.abs()).sum()) + 1e-6 * abs(num) + 1e-6, name


def _plain64(q, k, v, lens, causal):
    out, at = torch.zeros_like(q), 0
    for n in lens:
        for h in range(q.shape[1]):
            hk = h * k.shape[1] // q.shape[1]
            s = q[at:at + n, h] @ k[at:at + n, hk].T * q.shape[2] ** -0.5
            if causal:
                s = s.masked_fill(~ref.visible(n, n, True), -math.inf)
            out[at:at + n, h] = torch.softmax(s, 1) @ v[at:at + n, hk]
        at += n
    return out


@pytest.mark.parametrize("scale", [1e-3, 3.0])
def test_scales_and_large_scores(cuda, scale):
    """Flat and peaked rows: scores up to several hundred."""
    from ah_rag.packed import PackedLayout, packed_attention
    shape = ([100, 40], None, 2, 2, 64, True, BF)
    q, k, v, d_o = _make(shape, 13, cuda)
    lay = PackedLayout(shape[0], device=cuda)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    o = packed_attention(*leaves, lay, causal=True, scale=scale)
    g = torch.autograd.grad(o, leaves, d_o)
    w_o, t_o, w_g, t_g = ref.attention(q, k, v, shape[0], shape[0], True, scale, d_o=d_o)
    _within(o, w_o, t_o, "o")
    for name, a, w, t in zip(("dq", "dk", "dv"), g, w_g, t_g):
        _within(a, w, t, name)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("lens,causal", [([1, 2, 3, 8, 64, 33], False), ([1, 5, 40, 2], True)])
def test_few_keys_keep_the_small_gradients(cuda, lens, causal, dt):
    """Where one key takes nearly all the weight, ds = p (dp - delta) is far smaller than delta, and a delta from the
    rounded output would drown it. The kernel's is exact to 32 bits where a row's keys lie in one tile: with u half a
    step of the type, p off by 2^-17 (the roundings of c s and of the stored logarithm, each below 2^7, 2^-17 in
    exp2's argument, times ln 2), ds_j is off by u |ds_j| + 2^-16 p_j (|dp_j| + sum_i p_i |dp_i|), and dq by the sum of
    these times |k_j| and its own rounding. (f16 holds ds times a power of two, so it has no smallest value here.)"""
    from ah_rag.packed import PackedLayout, packed_attention
    hq, hk, d = 4, 2, 64
    q, k, v, do = _make((lens, None, hq, hk, d, causal, dt), 5, cuda)
    q, k, v = (x.detach().clone().requires_grad_() for x in (q, k, v))
    packed_attention(q, k, v, PackedLayout(lens, device=cuda), scale=1.0, causal=causal).backward(do)
    u = torch.finfo(dt).eps / 2
    q64, k64, v64, do64 = (x.detach().cpu().double() for x in (q, k, v, do))
    k64, v64 = (x.repeat_interleave(hq // hk, 1) for x in (k64, v64))
    at = 0
    for n in lens:
        Q, K, V, D = (x[at:at + n].transpose(0, 1) for x in (q64, k64, v64, do64))
        s = Q @ K.transpose(1, 2)
        assert float(s.abs().max()) * 1.4427 < 128
        if causal:
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf)
        p, dp = torch.softmax(s, 2), D @ V.transpose(1, 2)
        ds = p * (dp - (p * dp).sum(2, keepdim=True))
        off = u * ds.abs() + 2.0 ** -16 * p * (dp.abs() + (p * dp.abs()).sum(2, keepdim=True))
        want = (ds @ K).transpose(0, 1)
        _within(q.grad[at:at + n], want, (off @ K.abs()).transpose(0, 1) * 1.01 + u * want.abs() + 1e-7, "dq of %d tokens" % n)
        at += n


@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** 9])
def test_small_and_large_f16_gradients(cuda, size):
    """f16 holds neither ds of a long row with small gradients nor that of large ones by itself."""
    from ah_rag.packed import PackedLayout, packed_attention
    shape = ([700], None, 2, 1, 64, True, HF)
    q, k, v, d_o = _make(shape, 17, cuda)
    d_o = (d_o.float() * size).to(HF)
    lay = PackedLayout(shape[0], device=cuda)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    g = torch.autograd.grad(packed_attention(*leaves, lay, causal=True), leaves, d_o)
    _, _, w_g, t_g = ref.attention(q, k, v, shape[0], shape[0], True, 0.125, d_o=d_o)
    for name, a, w, t in zip(("dq", "dk", "dv"), g, w_g, t_g):
        _within(a, w, t, name)


def test_other_sequences_never_leak(cuda):
    """NaN and infinities in one sequence (keys, values, queries, gradients) stay there."""
    from ah_rag.packed import PackedLayout, packed_attention, prefix_attention
    for causal in (False, True):
        lens = [40, 70, 25]
        shape = (lens, None, 4, 2, 64, causal, BF)
        q, k, v, d_o = _make(shape, 19, cuda)
        bad = [x.clone() for x in (q, k, v, d_o)]
        for x, val in zip(bad, (math.nan, math.inf, -math.inf, math.nan)):
            x[40:110] = val
        lay = PackedLayout(lens, device=cuda)
        o, o2 = packed_attention(q, k, v, lay, causal=causal), packed_attention(*bad[:3], lay, causal=causal)
        l1 = [x.detach().requires_grad_() for x in (q, k, v)]
        l2 = [x.detach().requires_grad_() for x in bad[:3]]
        g1 = torch.autograd.grad(packed_attention(*l1, lay, causal=causal), l1, d_o)
        g2 = torch.autograd.grad(packed_attention(*l2, lay, causal=causal), l2, bad[3])
        pk = k[:5].contiguous()
        p1, p2 = (prefix_attention(*x, pk, pk, lay, causal=causal) for x in ((q, k, v), bad[:3]))
        for a, b in ((o, o2), (p1, p2), *zip(g1, g2)):
            for s in (slice(0, 40), slice(110, None)):
                assert torch.equal(a[s], b[s])


@pytest.mark.parametrize("dim,dt", [(64, BF), (40, HF), (128, BF)])
@pytest.mark.parametrize("val", [math.nan, math.inf, -math.inf])
def test_hidden_values_never_reach_a_row(cuda, dim, dt, val):
    """A causal sequence whose token 37 holds such keys and values: the rows before it keep their bits, the rows
    that read it have what the definition gives."""
    from ah_rag.packed import PackedLayout, packed_attention, prefix_attention
    lens = [100]
    q, k, v, _ = _make((lens, None, 4, 2, dim, True, dt), 37, cuda)
    lay = PackedLayout(lens, device=cuda)
    want, tol = ref.attention(q, k, v, lens, lens, True, dim ** -0.5)
    pk = k[:70].clone()
    k2, v2 = k.clone(), v.clone()
    k2[37] = val
    v2[37] = val
    o = packed_attention(q, k2, v, lay, causal=True)
    _within(o[:37], want[:37], tol[:37], "behind a hidden key")
    o = packed_attention(q, k, v2, lay, causal=True)
    _within(o[:37], want[:37], tol[:37], "behind a hidden value")
    assert (o[37:].isnan().all() if math.isnan(val) else (o[37:] == val).all())
    w2, t2 = ref.attention(q, k, v, lens, lens, True, dim ** -0.5, pk, pk)
    o = prefix_attention(q, k, v2, pk, pk, lay)
    _within(o[:37], w2[:37], t2[:37], "behind a hidden value, with a prefix")
    # the last key of a tile that is not full
    v3 = v.clone()
    v3[99] = val
    o = packed_attention(q, k, v3, lay, causal=True)
    _within(o[:99], want[:99], tol[:99], "before the last key")
    single = PackedLayout([1], [100], cuda)
    o = packed_attention(q[:1], k, v3, single, causal=True)
    assert (o.isnan().all() if math.isnan(val) else (o == val).all())


def test_rows_outside_are_left_alone(cuda):
    """out is a slice of a larger buffer: nothing around it is written."""
    from ah_rag.packed import PackedLayout, packed_attention
    shape = ([33, 0, 18], None, 2, 2, 40, True, BF)
    q, k, v, _ = _make(shape, 23, cuda)
    lay = PackedLayout(shape[0], device=cuda)
    big = torch.full((60, 3, 56), 7.0, dtype=BF, device=cuda)
    out = big[4:55, :2, 8:48]
    got = packed_attention(q, k, v, lay, causal=True, out=out)
    assert got is out and torch.equal(out, packed_attention(q, k, v, lay, causal=True))
    big[4:55, :2, 8:48] = 7.0
    assert (big == 7.0).all()


def test_far_offsets(cuda):
    """Rows whose byte offsets pass 32 bits: the keys of the last sequence lie beyond 4 GiB."""
    from ah_rag.packed import PackedLayout, packed_attention
    rows, wide = 600, (1 << 22) - 64  # 8 MiB from token to token: 4.7 GiB
    buf = torch.empty(rows * wide, dtype=BF, device=cuda)
    g = torch.Generator().manual_seed(4)
    small = torch.randn(3, rows, 1, 64, generator=g).to(BF).to(cuda)
    views = [buf.view(rows, wide)[:, 64 * i:64 * i + 64].unsqueeze(1) for i in range(3)]
    for a, b in zip(views, small):
        a.copy_(b)
    lay = PackedLayout([450, 150], device=cuda)
    leaves = [x.detach().requires_grad_() for x in views]
    dense = [x.detach().requires_grad_() for x in small]
    o, w = packed_attention(*leaves, lay, causal=True), packed_attention(*dense, lay, causal=True)
    assert torch.equal(o, w)
    d_o = torch.randn(rows, 1, 64, generator=g).to(BF).to(cuda)
    for a, b in zip(torch.autograd.grad(o, leaves, d_o), torch.autograd.grad(w, dense, d_o)):
        assert torch.equal(a, b)


def test_streams_and_two_calls_at_once(cuda):
    from ah_rag.packed import PackedLayout, packed_attention, packed_mean_pool
    shape = ([1, 1, 1, 1], [3000, 2500, 100, 900], 8, 2, 64, True, BF)  # split: a workspace each
    q, k, v, _ = _make(shape, 29, cuda)
    lay = PackedLayout(shape[0], shape[1], cuda)
    want = packed_attention(q, k, v, lay, causal=True)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [packed_attention(q, k, v, lay, causal=True, stream=s) for s in streams for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    with torch.cuda.stream(streams[0]):  # a layout made and dropped on another stream than its use
        streams[0].wait_stream(torch.cuda.default_stream())
        o = packed_attention(q, k, v, PackedLayout(shape[0], shape[1], cuda), causal=True)
        m = packed_mean_pool(k[:, 0], PackedLayout([3000, 2500, 100, 900], device=cuda))
    torch.cuda.synchronize()
    assert torch.equal(o, want) and torch.equal(m, packed_mean_pool(k[:, 0], PackedLayout([3000, 2500, 100, 900], device=cuda)))


def test_captured_step_replays(cuda):
    """Forward and backward of the operators in one graph, replayed on new inputs with eager work between."""
    from ah_rag.packed import PackedLayout, packed_attention, packed_mean_pool, prefix_attention, qk_norm_rope, rotary_table
    shape = ([30, 0, 71, 4], None, 6, 2, 64, True, BF)
    q, k, v, d_o = _make(shape, 31, cuda)
    lay = PackedLayout(shape[0], device=cuda)
    cos, sin = rotary_table(80, 64, device=cuda)
    wq, wk = torch.rand(64, device=cuda) + 0.5, torch.rand(64, device=cuda) + 0.5
    d_y = torch.randn(4, 6 * 64, device=cuda)
    pk, pv = k[:20].clone(), v[:20].clone()
    single = PackedLayout([1] * 4, [30, 0, 71, 4], device=cuda)

    def step(q, k, v, d_y):
        leaves = [x.detach().requires_grad_() for x in (q, k, v, wq, wk)]
        a, b = qk_norm_rope(leaves[0], leaves[1], leaves[3], leaves[4], cos, sin, lay.positions())
        o = packed_attention(a, b, leaves[2], lay, causal=True)
        y = packed_mean_pool(o.flatten(1), lay, normalize=True)
        g = torch.autograd.grad(y, leaves, d_y)
        p = prefix_attention(q, k, v, pk, pv, lay)
        s = packed_attention(q[:4], k, v, single, causal=True)  # split keys: a workspace
        return [y.detach(), p, s, *g]

    static = [x.clone() for x in (q, k, v, d_y)]
    step(*static)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*static)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*static)
    for i in range(4):
        new = [*_make(shape, 40 + i, cuda)[:3], torch.randn(4, 6 * 64, device=cuda)]
        want = step(*new)
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_graph_outlives_its_layout(cuda):
    """Nothing but the graph holds the work lists when it is replayed."""
    import gc
    from ah_rag.packed import PackedLayout, packed_attention, packed_mean_pool
    shape = ([50, 3, 80], None, 4, 2, 64, True, BF)
    q, k, v, d_o = _make(shape, 43, cuda)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]

    def step(lay):
        o = packed_attention(*leaves, lay, causal=True)
        return [o.detach(), packed_mean_pool(o.detach().flatten(1), lay), *torch.autograd.grad(o, leaves, d_o)]

    lay = PackedLayout(shape[0], device=cuda)
    want = step(lay)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        outs = step(lay)
    del lay
    gc.collect()
    junk = [torch.full((1 << n,), -1, dtype=torch.int32, device=cuda) for n in range(4, 16) for _ in range(8)]
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    assert len(junk) == 96


def test_layout_during_capture_is_refused(cuda):
    """Copying work lists is no work for a graph: the call says so."""
    from ah_rag.packed import PackedLayout
    lay = PackedLayout([3], device=cuda)
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device=cuda)
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before the capture"):
            lay.positions()
        x += 1
    graph.replay()
    torch.cuda.synchronize()
    assert float(x[0]) == 1.0


def test_empty_batches(cuda):
    from ah_rag.packed import PackedLayout, packed_attention, packed_mean_pool, prefix_attention, qk_norm_rope, rotary_table
    cos, sin = rotary_table(4, 64, device=cuda)
    for lens in ([], [0, 0]):
        lay = PackedLayout(lens, device=cuda)
        x = torch.empty(0, 2, 64, dtype=BF, device=cuda, requires_grad=True)
        o = packed_attention(x, x, x, lay)
        assert o.shape == (0, 2, 64)
        assert torch.autograd.grad(o, x, o.detach())[0].shape == (0, 2, 64)
        with torch.no_grad():
            assert prefix_attention(x, x, x, torch.zeros(3, 2, 64, dtype=BF, device=cuda), torch.zeros(3, 2, 64, dtype=BF, device=cuda),
                                    lay).shape == (0, 2, 64)
        r = torch.empty(0, 8, dtype=BF, device=cuda, requires_grad=True)
        y = packed_mean_pool(r, lay, normalize=True)
        assert y.shape == (len(lens), 8) and not y.any()
        assert torch.autograd.grad(y, r, torch.ones_like(y))[0].shape == (0, 8)
        w = torch.ones(64, device=cuda, requires_grad=True)
        a, b = qk_norm_rope(x, x, w, w, cos, sin, torch.empty(0, dtype=torch.int32, device=cuda))
        assert a.shape == b.shape == (0, 2, 64)
        assert not torch.autograd.grad((a, b), w, (a.detach(), b.detach()))[0].any()


def test_second_derivatives_are_refused(cuda):
    from ah_rag.packed import PackedLayout, packed_attention, packed_mean_pool, qk_norm_rope, rotary_table
    lay = PackedLayout([4], device=cuda)
    x = torch.randn(4, 2, 64, dtype=BF, device=cuda, requires_grad=True)
    cos, sin = rotary_table(4, 64, device=cuda)
    for y in (packed_attention(x, x, x, lay), packed_mean_pool(x.flatten(1), lay), qk_norm_rope(x, x, None, None, cos, sin, lay.positions())[0]):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_gpu_refusals(cuda):
    from ah_rag.packed import PackedLayout, packed_attention, prefix_attention
    lay = PackedLayout([4], device=cuda)
    x = torch.zeros(4, 2, 64, dtype=BF, device=cuda)
    p = x.clone().requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        prefix_attention(x, x, x, p, p, lay)
    with pytest.raises(ValueError, match="out cannot"):
        packed_attention(p, x, x, lay, out=torch.empty_like(x))
    with pytest.raises(ValueError, match="out must"):
        packed_attention(x, x, x, lay, out=torch.empty_like(x).half())
    with pytest.raises(ValueError, match="out's rows"):
        packed_attention(x, x, x, lay, out=torch.empty(4, 2, 65, dtype=BF, device=cuda)[..., 1:])
    with pytest.raises(ValueError, match="expanded"):
        packed_attention(x, x, x, lay, out=torch.empty(1, 2, 64, dtype=BF, device=cuda).expand(4, 2, 64))
    with pytest.raises(ValueError, match="read-only"):
        lay.lengths[0] = 3
    for s in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            packed_attention(x, x, x, lay, scale=s)
    with pytest.raises(ValueError, match="must be on"):
        packed_attention(x.cpu(), x.cpu(), x.cpu(), lay)
    with pytest.raises(ValueError, match="on the host"):
        PackedLayout(torch.tensor([4], device=cuda))


# ---- q/k norm with rotation ------------------------------------------------------------------

ROPE = [
    (1, 1, 1, 2, 2, False, torch.float32), (7, 3, 1, 32, 32, False, BF), (102, 16, 8, 128, 128, False, BF),
    (33, 4, 2, 64, 64, True, HF), (40, 5, 3, 256, 256, False, HF), (600, 2, 1, 128, 128, True, torch.float32),
    (19, 6, 2, 96, 96, False, BF), (19, 2, 2, 80, 40, False, HF), (19, 2, 1, 80, 40, True, BF), (9, 3, 2, 6, 4, True, torch.float32),
    (5, 2, 1, 512, 512, False, BF), (2100, 3, 1, 64, 64, False, BF),
    # rows that do not divide a wave, and heads whose halves are no multiples of 8
    (50, 8, 1, 48, 48, False, HF), (33, 13, 5, 80, 80, True, BF), (700, 20, 4, 80, 80, False, BF), (21, 11, 10, 112, 112, False, torch.float32),
    (9, 7, 7, 160, 160, True, HF), (40, 5, 3, 40, 40, False, BF), (40, 23, 2, 24, 24, True, HF), (65, 70, 9, 8, 8, False, BF),
    (17, 3, 3, 104, 104, False, torch.float32), (3, 2, 1, 504, 504, True, BF), (5, 3, 2, 480, 480, False, HF),
]


@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("shape", ROPE, ids=lambda s: "t%d-h%d.%d-d%d-r%d-%s-%s" % (*s[:5], "il" if s[5] else "half", str(s[6])[6:]))
def test_qk_norm_rope(cuda, shape, normed):
    """Bounds: fp32 arithmetic of about a dozen steps on values of the row's size (dim / 2 more for the sums
    of squares and of dn w x, which enter relatively), one rounding to the type; weight gradients: fp32 sums
    of tokens * heads terms, in any order off by at most their number's half steps, here sqrt-like, bounded
    by 2^-19 of the sum of absolute values."""
    from ah_rag.packed import qk_norm_rope, rotary_table
    t, hq, hk, d, rot, il, dt = shape
    g = torch.Generator().manual_seed(t)
    qkv = torch.randn(t, hq + 2 * hk, d, generator=g).to(dt).to(cuda)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    wq, wk = ((torch.rand(d, generator=g) + 0.5).to(cuda) if normed else None for _ in range(2))
    cos, sin = rotary_table(5000, rot, device=cuda)
    pos = torch.randint(0, 5000, (t,), generator=g).to(cuda)
    pos[-1] = 4999
    eps = 1e-6
    dyq, dyk = (torch.randn(t, h, d, generator=g).to(dt).to(cuda) for h in (hq, hk))
    plain = qk_norm_rope(q, k, wq, wk, cos, sin, pos, eps=eps, interleaved=il)
    leaves = [x.detach().requires_grad_() for x in (q, k, wq, wk) if x is not None]
    lw = leaves[2:] or [None, None]
    yq, yk = qk_norm_rope(leaves[0], leaves[1], *lw, cos, sin, pos.int(), eps=eps, interleaved=il)
    assert torch.equal(yq, plain[0]) and torch.equal(yk, plain[1])
    grads = torch.autograd.grad((yq, yk), leaves, (dyq, dyk))
    u = ref.half_step(dt)
    f = (16 + d / 2) * ref.F32
    for i, (x, w, y, dy) in enumerate(((q, wq, yq, dyq), (k, wk, yk, dyk))):
        wy, wdx, wdw = ref.rotate(x, w, cos, sin, pos, eps if normed else None, il, dy)
        pair = wy.abs().amax(-1, keepdim=True)
        _within(y, wy, u * wy.abs() * 1.01 + 2 * f * pair + 1e-30 + u * torch.finfo(dt).tiny, "y")
        x64 = x.cpu().double()
        r = 1 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + eps) if normed else torch.ones(t, 1, 1, dtype=torch.float64)
        dn = dy.cpu().double().abs().amax(-1, keepdim=True) * 3 * (1.5 if normed else 1.0)
        _within(grads[i], wdx, u * wdx.abs() * 1.01 + 2 * f * dn * r * (1 + (x64.abs() * r if normed else 0) * d ** 0.5) + u * torch.finfo(dt).tiny, "dx")
        if normed:
            size = (dy.cpu().double().abs().amax(-1, keepdim=True) * 2 * x64.abs() * r).sum((0, 1))
            _within(grads[2 + i], wdw, 2.0 ** -19 * size, "dw")


def test_rope_positions_outside_the_table(cuda):
    from ah_rag.packed import qk_norm_rope, rotary_table
    cos, sin = rotary_table(10, 64, device=cuda)
    for d in (64, 72):  # both kernels
        q = torch.randn(4, 2, d, device=cuda, dtype=BF).requires_grad_()
        pos = torch.tensor([9, 10, -1, 2 ** 32 + 3], device=cuda)
        y, z = qk_norm_rope(q, q, None, None, cos, sin, pos)
        assert y[0].isfinite().all() and y[1:].isnan().all() and z[1:].isnan().all()
        g, = torch.autograd.grad((y, z), q, (torch.ones_like(y), torch.ones_like(z)))
        assert g[0].isfinite().all() and g[1:].isnan().all()


def test_rope_weight_types_and_strides(cuda):
    from ah_rag.packed import qk_norm_rope, rotary_table
    cos, sin = rotary_table(50, 64, device=cuda)
    pos = torch.arange(50, device=cuda, dtype=torch.int32)
    q, k = torch.randn(50, 4, 64, device=cuda).to(BF), torch.randn(50, 2, 64, device=cuda).to(BF)
    w = (torch.rand(64, device=cuda) + 0.5).to(BF)
    a = qk_norm_rope(q, k, w, w, cos, sin, pos)
    b = qk_norm_rope(q.transpose(0, 1).contiguous().transpose(0, 1), torch.stack((k, k), -1)[..., 1], w.float(), w.float(),
                     torch.cat((cos, cos), 1)[:, :32], torch.cat((sin, sin), 1)[:, :32], torch.stack((pos, pos), 1)[:, 0])
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    w1 = w.detach().requires_grad_()
    y, z = qk_norm_rope(q, k, w1, w1, cos, sin, pos)
    g, = torch.autograd.grad((y, z), w1, (torch.ones_like(y), torch.ones_like(z)))
    assert g.dtype == BF and g.isfinite().all()
    odd = torch.nn.functional.pad(q.flatten(), (1, 0))[1:].view(q.shape)  # rows that start off 16 bytes
    c = qk_norm_rope(odd, k, w, w, cos, sin, pos)
    _within(c[0], a[0].cpu().double(), 2.1 * ref.half_step(BF) * a[0].cpu().double().abs() + 1e-6, "unaligned")


# ---- mean pooling ----------------------------------------------------------------------------


@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("lens,width,dt", [
    ([1], 1, BF), ([3, 0, 64, 65, 1], 384, BF), ([300, 2], 770, HF), ([129], 33, torch.float32), ([0, 5], 2048, torch.float32),
    ([2000, 40, 7], 1024, HF), ([5, 6], 9000, BF),
])
def test_mean_pool(cuda, lens, width, dt, normalize):
    """Bounds: sums of n values in fp32, off by at most n 2^-24 of the sum of absolute values; the norm and
    division 8 steps more; gradients the same and one rounding to the type."""
    from ah_rag.packed import PackedLayout, packed_mean_pool
    g = torch.Generator().manual_seed(len(lens) + width)
    wide = (torch.randn(sum(lens), width + 16, generator=g) + 0.3).to(dt).to(cuda)
    for rows in (wide[:, :width], wide[:, 5:5 + width], wide[:, :width].contiguous()):
        lay = PackedLayout(lens, device=cuda)
        leaf = rows.detach().requires_grad_()
        y = packed_mean_pool(leaf, lay, normalize=normalize)
        assert y.dtype == torch.float32 and torch.equal(y, packed_mean_pool(rows, lay, normalize=normalize))
        dy = torch.randn(y.shape, generator=g).to(cuda)
        d, = torch.autograd.grad(y, leaf, dy)
        assert d.dtype == dt
        wy, wd = ref.mean_pool(rows, lens, normalize, dy)
        n = max(lens) + 8
        size = ref.mean_pool(rows.abs(), lens, False)
        norm = ref.mean_pool(rows, lens, False).norm(dim=1, keepdim=True).clamp_min(1e-12) if normalize else torch.ones(len(lens), 1, dtype=torch.float64)
        t_y = n * ref.F32 * size / norm * 2 + (n + width / 8) * ref.F32 * wy.abs() + 1e-30
        _within(y, wy, t_y, "mean")
        each = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
        sz = ((dy.cpu().double().abs() + (wy.abs() * (dy.cpu().double().abs() * wy.abs()).sum(1, keepdim=True) if normalize else 0)) / norm
              / torch.tensor(lens).clamp_min(1)[:, None])[each]
        extra = (t_y.norm(dim=1) * dy.cpu().double().norm(dim=1) / norm[:, 0] / torch.tensor(lens).clamp_min(1))[each][:, None] * 2 if normalize else 0
        _within(d, wd, ref.half_step(dt) * wd.abs() * 1.01 + (n + width / 8) * ref.F32 * sz * 2 + extra + torch.finfo(dt).tiny * ref.half_step(dt), "rows' gradient")


def test_mean_pool_of_zero_rows_and_nan(cuda):
    from ah_rag.packed import PackedLayout, packed_mean_pool
    lay = PackedLayout([3, 4, 2], device=cuda)
    rows = torch.zeros(9, 64, dtype=BF, device=cuda)
    rows[3:7] = math.nan
    rows[7:] = 1.0
    y = packed_mean_pool(rows, lay, normalize=True)
    assert not y[0].any() and y[1].isnan().all() and torch.allclose(y[2], torch.full((64,), 0.125, device=cuda), rtol=1e-6)
