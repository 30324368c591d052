"""Edges of the packed-sequence operators on the GPU, against the 64-bit restatement (oracle/packed_ref.py) and the
bounds that it derives."""
import math

import pytest
import torch

from oracle import packed_ref as ref

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _normal(shape, seed, dtype, dev):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(dev)


def _within(got, want, tol, what):
    """Within tol where `want` is finite; the same infinity, or NaN, where it is not."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    fin = torch.isfinite(want)
    off = (got - want).abs()[fin]
    bad = ~(off <= tol[fin])
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol[fin]).nan_to_num(1e9).max()):.3g} x the bound"
    a, b = got[~fin], want[~fin]
    assert ((a == b) | (a.isnan() & b.isnan())).all(), f"{what}: values that are not finite differ"


# A value that is not finite in ONE column of one row of v: the columns of a row's output lie in two halves of a wave
# (columns with d & 4, and the others), which have to take the same weights and the same sum.


@pytest.mark.parametrize("dim,dt", [(24, BF), (32, HF), (64, BF), (56, HF), (96, HF), (80, BF), (128, BF), (128, HF)])
@pytest.mark.parametrize("col", [0, 3, 4, 7, -1])
@pytest.mark.parametrize("val", [math.nan, math.inf])
def test_one_bad_column_of_a_value(cuda, dim, dt, col, val):
    from ah_rag.packed import PackedLayout, packed_attention, prefix_attention
    scale = dim ** -0.5
    lens = [100, 30]
    q, k, v, pv = (_normal((130, h, dim), 40 + i, dt, cuda) for i, h in enumerate((4, 2, 2, 2)))
    pk, pv = k[20:90].clone(), pv[:70].clone()
    bad = v.clone()
    bad[37, 1, col] = val
    lay = PackedLayout(lens, device=cuda)
    _within(packed_attention(q, k, bad, lay, causal=True), *ref.attention(q, k, bad, lens, lens, True, scale), "causal")
    _within(packed_attention(q, k, bad, lay), *ref.attention(q, k, bad, lens, lens, False, scale), "full")
    _within(prefix_attention(q, k, bad, pk, pv, lay), *ref.attention(q, k, bad, lens, lens, True, scale, pk, pv), "own value, with a prefix")
    pv[50, 0, col] = val
    _within(prefix_attention(q, k, v, pk, pv, lay), *ref.attention(q, k, v, lens, lens, True, scale, pk, pv), "a prefix value")


@pytest.mark.parametrize("dim,dt", [(64, BF), (40, HF), (128, BF), (96, HF)])
@pytest.mark.parametrize("col", [0, 3, 4, 7, -1])
def test_one_bad_column_in_split_plans(cuda, dim, dt, col):
    """Keys in pieces that are joined: the piece with the bad value, hidden from the first query and read by the second;
    and a prefix that is read apart."""
    from ah_rag.packed import _CODES, PackedLayout, packed_attention, prefix_attention
    scale = dim ** -0.5
    ql, kl = [2, 1], [2000, 700]
    q, k, v = (_normal((n, h, dim), 50 + i, dt, cuda) for i, (n, h) in enumerate(((3, 8), (2700, 2), (2700, 2))))
    v[1999, 0, col] = math.nan
    v[1000, 1, col] = math.inf
    lay = PackedLayout(ql, kl, cuda)
    assert lay._plan(_CODES[dt], 8, 2, dim, True, False, 0)[0].n_join > 0
    _within(packed_attention(q, k, v, lay, causal=True), *ref.attention(q, k, v, ql, kl, True, scale), "pieces")
    lens, prefix = [3] * 40, 1300
    q, k, v, pk, pv = (_normal((n, h, dim), 60 + i, dt, cuda) for i, (n, h) in enumerate(((120, 8), (120, 4), (120, 4), (prefix, 4), (prefix, 4))))
    v[61, 2, col] = math.inf
    lay = PackedLayout(lens, device=cuda)
    assert lay._plan(_CODES[dt], 8, 4, dim, True, False, prefix)[0].n_join > 0
    _within(prefix_attention(q, k, v, pk, pv, lay), *ref.attention(q, k, v, lens, lens, True, scale, pk, pv), "a prefix read apart")
    pv[777, 1, col] = math.nan
    _within(prefix_attention(q, k, v, pk, pv, lay), *ref.attention(q, k, v, lens, lens, True, scale, pk, pv), "its values")


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("col", [0, 5])
def test_values_that_overflow_one_half_of_a_row(cuda, dim, col):
    """Large finite values in one column: weights relative to a reference that is raised late reach 2^8, so one half's
    sums pass fp32 before they are divided. Output, log-sum and gradients are what finite inputs give."""
    from ah_rag import packed
    scale = dim ** -0.5
    n = 150
    q = torch.zeros(n, 1, dim)
    q[:, 0, 1] = dim ** 0.5
    k = torch.zeros(n, 1, dim)
    k[140, 0, 1] = 5.0  # its score is 5 and the others' 0: 2^7.2 of the first tiles' reference
    q, k, v, d_o = q.to(BF).to(cuda), k.to(BF).to(cuda), _normal((n, 1, dim), 70, BF, cuda), _normal((n, 1, dim), 71, BF, cuda)
    v[140, 0, col] = 3e38
    d_o[..., col] = 0.0
    lay = packed.PackedLayout([n], device=cuda)
    want, tol, w_g, t_g = ref.attention(q, k, v, [n], [n], False, scale, d_o=d_o)
    assert torch.isfinite(want).all()
    lse = torch.empty(n, 1, device=cuda)
    _within(packed._attention(q, k, v, lay, False, scale, lse), want, tol, "o")
    # (in fp32: the scores' error of (dim + 4) 2^-24 of sum |q k|, and a few steps of a value below 16 for the logarithm and the sum)
    w_lse = math.log2(149 + math.exp(float(q[0, 0, 1].double() * 5 * scale)))
    assert (lse.double() - w_lse).abs().max() < (dim + 4) * 2.0 ** -24 * 5 * 1.5 + 8 * 2.0 ** -21
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(packed.packed_attention(*leaves, lay), leaves, d_o)
    for name, a, w, t in zip(("dq", "dk", "dv"), grads, w_g, t_g):
        _within(a, w, t, name)


def test_a_write_to_out_is_noticed(cuda):
    """out behaves as what torch writes in place: a graph that saved it refuses its backward pass afterwards, and one that
    wants a gradient is refused."""
    from ah_rag.packed import PackedLayout, packed_attention, prefix_attention
    q, k, v = (_normal((9, 2, 16), 80 + i, BF, cuda) for i in range(3))
    lay = PackedLayout([9], device=cuda)
    for call in (lambda out: packed_attention(q, k, v, lay, out=out), lambda out: prefix_attention(q, k, v, k, v, lay, out=out)):
        buf, leaf = torch.ones_like(q), torch.ones_like(q, requires_grad=True)
        y = (leaf * buf).sum()
        call(buf)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        with pytest.raises(ValueError, match="require a gradient"):
            call(torch.ones_like(q, requires_grad=True))
        with torch.no_grad():
            own = torch.ones_like(q, requires_grad=True)
            assert torch.equal(call(own), call(None))
        with torch.inference_mode():
            assert torch.equal(call(torch.ones_like(q)), call(None))


@pytest.mark.parametrize("q_len,few,many,dt,dim", [(1, 70, 6000, HF, 128), (1, 1, 3000, BF, 64), (3, 40, 4001, BF, 40)])
def test_one_long_sequence_in_a_large_batch(cuda, q_len, few, many, dt, dim):
    """More than 512 workgroups, one sequence's keys in pieces that are joined, the others whole."""
    from ah_rag.packed import _CODES, PackedLayout, packed_attention
    n, heads, hk = 80, 8, 8
    ql, kl = [q_len] * n, [few] * n
    kl[33] = many
    q, k, v = (_normal((sum(x), h, dim), 90 + i, dt, cuda) for i, (x, h) in enumerate(((ql, heads), (kl, hk), (kl, hk))))
    lay = PackedLayout(ql, kl, cuda)
    plan = lay._plan(_CODES[dt], heads, hk, dim, True, False, 0)[0]
    assert plan.n_rows * hk > 512 and plan.n_join == 1
    _within(packed_attention(q, k, v, lay, causal=True), *ref.attention(q, k, v, ql, kl, True, dim ** -0.5), "o")


@pytest.mark.parametrize("dt,dim,heads,kv_heads", [(HF, 128, 8, 1), (BF, 64, 16, 2)])
def test_long_sequences_in_a_large_batch_behind_a_prefix(cuda, dt, dim, heads, kv_heads):
    """Most tokens read the prefix apart, the long sequences in their own tiles, with partial rows of their own."""
    from ah_rag.packed import _CODES, PackedLayout, prefix_attention
    n, prefix, long = 6000, 2000, {0: 40000, 3001: 70000}
    ql = [1 + i % 2 for i in range(n)]
    kl = [long.get(i, 2 + i % 3) for i in range(n)]
    q, k, v, pk, pv = (_normal((m, h, dim), 100 + i, dt, cuda) for i, (m, h) in enumerate(
        ((sum(ql), heads), (sum(kl), kv_heads), (sum(kl), kv_heads), (prefix, kv_heads), (prefix, kv_heads))))
    lay = PackedLayout(ql, kl, cuda)
    plan = lay._plan(_CODES[dt], heads, kv_heads, dim, True, False, prefix)[0]
    assert plan.far_rows == sum(ql[i] for i in long) and plan.ws_bytes < 500e6
    o = prefix_attention(q, k, v, pk, pv, lay)
    q0, k0 = [0], [0]
    for a, b in zip(ql, kl):
        q0.append(q0[-1] + a)
        k0.append(k0[-1] + b)
    some = sorted({*long, 1, 2, 2999, 3000, 3002, 3003, n - 2, n - 1, *range(100, n, 371)})
    qi = torch.cat([torch.arange(q0[i], q0[i + 1]) for i in some])
    ki = torch.cat([torch.arange(k0[i], k0[i + 1]) for i in some])
    want, tol = ref.attention(q.cpu()[qi], k.cpu()[ki], v.cpu()[ki], [ql[i] for i in some], [kl[i] for i in some], True, dim ** -0.5, pk, pv)
    _within(o.cpu()[qi], want, tol, "o")
    assert o.isfinite().all()


def test_positions_outlive_their_layout(cuda):
    """A layout's positions read by a captured rotation, and by one that another stream still waits to run, after the layout
    and they themselves have been dropped and their memory asked for again."""
    from ah_rag.packed import PackedLayout, qk_norm_rope, rotary_table
    n = 700
    q, k = _normal((n, 4, 32), 110, BF, cuda), _normal((n, 2, 32), 111, BF, cuda)
    cos, sin = rotary_table(n, 32, device=cuda)
    want = qk_norm_rope(q, k, None, None, cos, sin, PackedLayout([n], device=cuda).positions())

    def fill():
        junk = [torch.full((n,), n + 5, dtype=torch.int32, device=cuda) for _ in range(200)]
        torch.cuda.synchronize()
        return junk

    pos = PackedLayout([n], device=cuda).positions()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = qk_norm_rope(q, k, None, None, cos, sin, pos)
    del pos
    for _ in range(3):
        junk = fill()
        for x in got:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del junk
    lay = PackedLayout([n], device=cuda)
    lay.positions()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)  # (a finite wait on the device's clock)
        got = qk_norm_rope(q, k, None, None, cos, sin, lay.positions())
    at = lay.positions().data_ptr()
    del lay
    junk = [torch.full((n,), n + 5, dtype=torch.int32, device=cuda) for _ in range(200)]
    assert not side.query() and at not in {x.data_ptr() for x in junk}
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def _bounds(dt):
    return {BF: 1e17, HF: 6e4}[dt]


@pytest.mark.parametrize("dt,dim", [(BF, 64), (BF, 128), (BF, 40), (HF, 32), (HF, 96)])
def test_scores_of_any_size(cuda, dt, dim):
    """Scores far beyond what fp32 tells apart by one (2^24): the largest takes the whole weight, whatever its size and sign."""
    from ah_rag.packed import PackedLayout, packed_attention, prefix_attention
    size = _bounds(dt)
    for sign in (1.0, -1.0):
        for case, (ql, kl, heads, hk, prefix) in enumerate((([70, 1], [200, 150], 4, 2, 0), ([2], [3000], 8, 2, 0), ([3] * 40, [3] * 40, 8, 4, 1300))):
            g = torch.Generator().manual_seed(120 + case)
            q = torch.zeros(sum(ql), heads, dim)
            q[..., :5] = size * (1 + torch.rand(sum(ql), heads, 5, generator=g)) * sign / 2
            k = torch.zeros(sum(kl) + prefix, hk, dim)
            k[..., :5] = size * (1 + torch.rand(sum(kl) + prefix, hk, 5, generator=g)) / 2
            q, k = q.to(dt).to(cuda), k.to(dt).to(cuda)
            v = _normal((sum(kl) + prefix, hk, dim), 130, dt, cuda)
            lay = PackedLayout(ql, kl, cuda)
            pk, pv, k, v = k[:prefix], v[:prefix], k[prefix:], v[prefix:]
            o = prefix_attention(q, k, v, pk, pv, lay, causal=False) if prefix else packed_attention(q, k, v, lay)
            qd, kd, vd, pkd, pvd = (x.cpu().double() for x in (q, k, v, pk, pv))
            q0 = k0 = 0
            for a, b in zip(ql, kl):
                for h in range(heads):
                    K, V = torch.cat((pkd[:, h * hk // heads], kd[k0:k0 + b, h * hk // heads])), torch.cat((pvd[:, h * hk // heads], vd[k0:k0 + b, h * hk // heads]))
                    s = qd[q0:q0 + a, h] @ K.T
                    top = s.topk(2, 1).values
                    # (rows whose best two are told apart by more than the fp32 sums may be off)
                    clear = (top[:, 0] - top[:, 1]) * dim ** -0.5 > 8 * 2.0 ** -24 * s.abs().amax(1) * dim ** -0.5 + 200
                    want = V[s.argmax(1)]
                    assert torch.equal(o[q0:q0 + a, h].cpu().double()[clear], want[clear]) and clear.any()
                q0, k0 = q0 + a, k0 + b


@pytest.mark.parametrize("dt,dim", [(BF, 64), (HF, 96)])
def test_rows_whose_scores_are_all_minus_infinity(cuda, dt, dim):
    """They have no softmax (NaN, as the definition gives); rows that read no key give zeros; others are untouched."""
    from ah_rag.packed import PackedLayout, packed_attention, prefix_attention
    scale = dim ** -0.5
    for ql, kl, heads, hk in (([5, 3, 2], [5, 0, 130], 4, 2), ([2, 1], [2000, 700], 8, 2)):
        q, k, v = (_normal((n, h, dim), 140 + i, dt, cuda) for i, (n, h) in enumerate(((sum(ql), heads), (sum(kl), hk), (sum(kl), hk))))
        q[..., 0] = q[..., 0].abs() + 0.1
        first = 5 if len(ql) == 3 else 2000
        k[:first, 1, 0] = -math.inf  # every key of the first sequence, for half the heads
        lay = PackedLayout(ql, kl, cuda)
        o = packed_attention(q, k, v, lay).cpu()
        want, tol = ref.attention(q[:, :heads // 2], k[:, :1], v[:, :1], ql, kl, False, scale)
        _within(o[:, :heads // 2], want, tol, "heads without")
        assert o[:ql[0], heads // 2:].isnan().all() and o[ql[0]:].isfinite().all()
        if len(ql) == 3:
            assert not o[5:8].any()
        one = k[:1].clone()  # a prefix of one key that is read: its value alone
        one[:, :, 0] = 0.0
        p = prefix_attention(q, k, v, one, v[:1].clone(), lay, causal=False).cpu()
        assert torch.equal(p[:ql[0], heads // 2:], v[:1, 1:].cpu().expand(ql[0], heads // 2, dim))


@pytest.mark.parametrize("dim,dt", [(32, BF), (64, HF), (96, BF), (128, HF)])
@pytest.mark.parametrize("col", [0, 4, -1])
def test_log_sums_and_gradients_beside_a_bad_column(cuda, dim, dt, col):
    """The log-sums that the backward pass reads are those of the rows' keys, whatever one column of a value holds, and the
    gradients of the other sequence keep their bits."""
    from ah_rag import packed
    scale, lens = dim ** -0.5, [100, 30]
    q, k, v, d_o = (_normal((130, h, dim), 150 + i, dt, cuda) for i, h in enumerate((4, 2, 2, 4)))
    bad = v.clone()
    bad[37, 1, col] = math.nan
    lay = packed.PackedLayout(lens, device=cuda)
    lse = torch.empty(130, 4, device=cuda)
    packed._attention(q, k, bad, lay, True, scale, lse)
    for h in range(4):
        for a, b in ((0, 100), (100, 130)):
            s = scale * (q[a:b, h].double() @ k[a:b, h // 2].double().T)
            s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), -math.inf)
            # scores in fp32 ((dim + 4) half steps of sum |q k|), the logarithm and the sum a few half steps of 16
            off = ((q[a:b, h].double().abs() @ k[a:b, h // 2].double().abs().T).amax(1) * scale * (dim + 4) + 16 * 8) * 2.0 ** -24 * 1.5
            assert ((lse[a:b, h].double() - torch.logsumexp(s, 1) / math.log(2)).abs() <= off).all()
    grads = []
    for x in (v, bad):
        leaves = [t.detach().requires_grad_() for t in (q, k, x)]
        grads.append(torch.autograd.grad(packed.packed_attention(*leaves, lay, causal=True), leaves, d_o))
    for a, b in zip(*grads):
        assert torch.equal(a[100:], b[100:]) and a.isfinite().all()


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("lens,kls", [([300], None), ([130, 64, 65], None), ([200], [150]), ([100], [130])])
def test_early_rows_of_long_causal_sequences_keep_the_small_gradients(cuda, dt, lens, kls):
    """Rows that read at most one tile's keys, 128 of them in a tile of rows whose last ones read more: their delta is exact
    too. Bounds as where all rows of a sequence read one tile: with u half a step of the type, ds_j is off by u |ds_j| +
    2^-16 p_j (|dp_j| + sum_i p_i |dp_i|), and dq by the sum of these times |k_j| and its own rounding."""
    from ah_rag.packed import PackedLayout, packed_attention
    h, d = 4, 64
    kls = kls or lens
    q, do = (_normal((sum(lens), h, d), 160 + i, dt, cuda) for i in range(2))
    k, v = (_normal((sum(kls), h, d), 162 + i, dt, cuda) for i in range(2))
    leaf = q.clone().requires_grad_()
    packed_attention(leaf, k, v, PackedLayout(lens, kls, cuda), scale=1.0, causal=True).backward(do)
    u = torch.finfo(dt).eps / 2
    q0 = k0 = 0
    for n, m in zip(lens, kls):
        # the rows of whole waves (32 rows) whose last one reads at most 64 keys
        rows = max(0, (min(n, 64 - (m - n)) // 32) * 32)
        Q, D = (x[q0:q0 + rows].transpose(0, 1).cpu().double() for x in (q, do))
        K, V = (x[k0:k0 + m].transpose(0, 1).cpu().double() for x in (k, v))
        s = Q @ K.transpose(1, 2)
        assert rows == 0 or float(s.abs().max()) * 1.4427 < 128
        see = ref.visible(n, m, True)[:rows]
        p = torch.softmax(s.masked_fill(~see, -math.inf), 2).nan_to_num(0.0)
        dp = D @ V.transpose(1, 2)
        ds = p * (dp - (p * dp).sum(2, keepdim=True))
        off = u * ds.abs() + 2.0 ** -16 * p * (dp.abs() + (p * dp.abs()).sum(2, keepdim=True))
        want = (ds @ K).transpose(0, 1)
        _within(leaf.grad[q0:q0 + rows], want, (off @ K.abs()).transpose(0, 1) * 1.01 + u * want.abs() + 1e-7, "dq of %d over %d" % (n, m))
        q0, k0 = q0 + n, k0 + m
    assert leaf.grad.isfinite().all()
