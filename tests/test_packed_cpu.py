"""Packed-sequence operators on the host: the work lists cover every (token, key) pair exactly once, and
bad arguments are refused before anything is launched."""
import ctypes

import numpy as np
import pytest

ROW = ("q0", "nq", "k0", "klen", "koff", "kb", "ke", "pb", "pe", "plane", "prow", "pad")
KEY = ("k0", "nk", "kpos", "klen", "q0", "qlen", "t0", "t1", "plane", "prow", "pad", "pad2")


def _plan(q_lens, k_lens=None, heads=12, kv_heads=12, dim=64, causal=0, backward=0, prefix=0, dtype=2):
    from ah_rag import _native as nat
    lib = nat.lib()
    q = np.asarray(q_lens, np.int32)
    k = None if k_lens is None else np.asarray(k_lens, np.int32)
    shape = nat.AttnShape(dtype, heads, kv_heads, dim, causal, backward, prefix)
    plan = nat.AttnPlan()
    args = (q.ctypes.data, None if k is None else k.ctypes.data, len(q), ctypes.byref(shape), ctypes.byref(plan))
    nat.check(lib.ahr_attn_plan_build(*args, None, 0))
    buf = np.full(plan.ints + 1, -7, np.int32)
    nat.check(lib.ahr_attn_plan_build(*args, buf.ctypes.data, plan.ints))
    assert buf[-1] == -7
    r, kk = plan.n_rows * len(ROW), plan.n_keys * len(KEY)
    assert r + kk + plan.n_join * 4 == plan.ints
    rows = [dict(zip(ROW, map(int, x))) for x in buf[:r].reshape(-1, len(ROW))]
    keys = [dict(zip(KEY, map(int, x))) for x in buf[r:r + kk].reshape(-1, len(KEY))]
    join = [tuple(map(int, x)) for x in buf[r + kk:-1].reshape(-1, 4)]
    return plan, rows, keys, join


CASES = [
    dict(q_lens=[5]),
    dict(q_lens=[0, 3, 0, 1]),
    dict(q_lens=[300, 1, 64, 65], causal=1),
    dict(q_lens=[130, 7, 500], heads=20, kv_heads=4, causal=1),
    dict(q_lens=[40, 3], k_lens=[20, 0], causal=1),
    dict(q_lens=[40, 3], k_lens=[20, 0]),
    dict(q_lens=[1, 1, 2], k_lens=[5000, 0, 1300], heads=32, kv_heads=8, dim=128, causal=1),
    dict(q_lens=[1], k_lens=[100000], heads=7, kv_heads=1, causal=1),
    dict(q_lens=[900], heads=100, kv_heads=1, causal=1),
    dict(q_lens=[6, 1, 9, 0, 2], prefix=1000, heads=16, kv_heads=8, causal=1),
    dict(q_lens=[1] * 60, k_lens=[3] * 59 + [0], prefix=5000, heads=16, kv_heads=4, causal=1),
    dict(q_lens=[2000, 1900], prefix=70, heads=16, kv_heads=8, causal=1),
    dict(q_lens=[700] * 20, prefix=1, heads=32, kv_heads=8, causal=1),
    dict(q_lens=[3, 0], k_lens=[0, 0], prefix=65),
    dict(q_lens=[]),
    dict(q_lens=[4000, 300], heads=16, kv_heads=4, dim=128, causal=1),
    dict(q_lens=[3000], k_lens=[700], heads=6, kv_heads=2),
    dict(q_lens=[2, 0, 5, 1] * 20, prefix=700, causal=1),
    dict(q_lens=[4] * 30, k_lens=[2] * 30, prefix=2000, heads=4, kv_heads=2),
]


@pytest.mark.parametrize("case", CASES)
def test_row_lists_cover_every_pair_once(case):
    plan, rows, _, join = _plan(**case)
    ql = case["q_lens"]
    kl = case.get("k_lens") or ql
    prefix, causal = case.get("prefix", 0), case.get("causal", 0)
    group = case.get("heads", 12) // case.get("kv_heads", 12)
    T, starts = sum(ql), np.concatenate(([0], np.cumsum(ql))).astype(int)
    kstarts = np.concatenate(([0], np.cumsum(kl))).astype(int)
    seq_of = np.repeat(np.arange(len(ql)), ql)
    own = [np.zeros(kl[s], int) for s in seq_of]
    pre = [np.zeros(prefix, int) for _ in range(T)]
    planes, final = [set() for _ in range(T)], np.zeros(T, int)
    for r in rows:
        assert 0 < r["nq"] and r["nq"] * group <= 128
        assert 0 <= r["q0"] and r["q0"] + r["nq"] <= T
        assert 0 <= r["pb"] <= r["pe"] <= prefix and 0 <= r["kb"] <= r["ke"]
        if r["ke"] > r["kb"]:
            s = seq_of[r["q0"]]
            assert seq_of[r["q0"] + r["nq"] - 1] == s and r["k0"] == kstarts[s] and r["ke"] <= r["klen"] == kl[s]
            assert r["kb"] % 64 == 0
        for i in range(r["nq"]):
            t = r["q0"] + i
            lim = min(r["klen"], r["koff"] + i + 1) if causal else r["klen"]
            own[t][r["kb"]:max(r["kb"], min(r["ke"], lim))] += 1
            pre[t][r["pb"]:r["pe"]] += 1
            if r["plane"] < 0:
                final[t] += 1
            else:
                assert r["plane"] < plan.planes and r["prow"] + i < plan.part_rows
                assert (r["plane"], r["prow"] + i) not in planes[t]
                planes[t].add((r["plane"], r["prow"] + i))
    for t in range(T):
        s = seq_of[t]
        lim = min(kl[s], t - starts[s] + kl[s] - ql[s] + 1) if causal else kl[s]
        want = (np.arange(kl[s]) < lim).astype(int)
        assert np.array_equal(own[t], want) and (pre[t] == 1).all()
    joined = {}
    for q0, nq, prow, n in join:
        for i in range(nq):
            assert q0 + i not in joined
            joined[q0 + i] = {(j, prow + i) for j in range(n)}
    for t in range(T):  # a token is either written once, or joined from exactly its partial rows
        assert (final[t] == 1 and not planes[t] and t not in joined) or (final[t] == 0 and planes[t] == joined[t])
    # no partial row belongs to two tokens
    flat = [x for p in planes for x in p]
    assert len(flat) == len(set(flat))
    assert plan.ws_bytes == plan.planes * plan.part_rows * case.get("heads", 12) * (case.get("dim", 64) + 1) * 4


@pytest.mark.parametrize("case,apart", [
    (dict(q_lens=[2, 0, 5, 1] * 20, prefix=700, causal=1), True), (dict(q_lens=[4] * 30, k_lens=[2] * 30, prefix=2000, heads=4, kv_heads=2), True),
    (dict(q_lens=[1] * 60, k_lens=[3] * 59 + [0], prefix=5000, heads=16, kv_heads=4, causal=1), True),
    (dict(q_lens=[2, 0, 5, 1] * 20, prefix=60, causal=1), False), (dict(q_lens=[128] * 30, prefix=5000), False),
    (dict(q_lens=[5], prefix=100000), False)])
def test_a_prefix_is_read_apart_where_that_saves_tiles(case, apart):
    _, rows, _, _ = _plan(**case)
    seq_of = np.repeat(np.arange(len(case["q_lens"])), case["q_lens"])
    across = [r for r in rows if seq_of[r["q0"]] != seq_of[r["q0"] + r["nq"] - 1]]
    assert bool(across) == apart and all(r["ke"] == r["kb"] and r["pe"] > r["pb"] for r in across)


@pytest.mark.parametrize("case", [c for c in CASES if "prefix" not in c])
def test_key_lists_cover_every_pair_once(case):
    plan, rows, keys, join = _plan(**case, backward=1)
    ql = case["q_lens"]
    kl = case.get("k_lens") or ql
    causal = case.get("causal", 0)
    kstarts = np.concatenate(([0], np.cumsum(kl))).astype(int)
    starts = np.concatenate(([0], np.cumsum(ql))).astype(int)
    seen, final = [np.zeros(ql[s], int) for s in np.repeat(np.arange(len(kl)), kl)], np.zeros(sum(kl), int)
    planes = [set() for _ in range(sum(kl))]
    for k in keys:
        s = int(np.searchsorted(kstarts, k["k0"], side="right") - 1)
        assert k["klen"] == kl[s] and k["qlen"] == ql[s] and k["q0"] == starts[s] and k["kpos"] == k["k0"] - kstarts[s]
        assert 0 < k["nk"] <= 128 and k["kpos"] + k["nk"] <= kl[s] and 0 <= k["t0"] <= k["t1"] <= ql[s]
        for i in range(k["k0"], k["k0"] + k["nk"]):
            seen[i][k["t0"]:k["t1"]] += 1
            if k["plane"] < 0:
                final[i] += 1
            else:
                assert k["plane"] < plan.planes and k["prow"] + k["nk"] <= plan.part_rows
                planes[i].add((k["plane"], k["prow"] + i - k["k0"]))
    for s in range(len(kl)):
        for j in range(kl[s]):
            got = seen[kstarts[s] + j]
            first = max(0, j - (kl[s] - ql[s])) if causal else 0  # the first token that reads key j
            assert (got[first:] == 1).all() and (got <= 1).all()
    joined = {k0 + i: {(j, prow + i) for j in range(n)} for k0, nk, prow, n in join for i in range(nk)}
    for i in range(sum(kl)):
        assert (final[i] == 1 and not planes[i] and i not in joined) or (final[i] == 0 and planes[i] == joined[i])
    flat = [x for p in planes for x in p]
    assert len(flat) == len(set(flat))
    assert all(r["plane"] < 0 and r["kb"] == 0 and r["pe"] == 0 for r in rows)
    assert sum(r["nq"] for r in rows) == sum(ql)


def test_plan_refusals():
    from ah_rag import _native as nat
    bad = [dict(dtype=0), dict(heads=12, kv_heads=5), dict(kv_heads=0), dict(heads=256, kv_heads=1), dict(dim=68), dict(dim=136),
           dict(dim=0), dict(causal=2), dict(prefix=-1), dict(prefix=5, backward=1)]
    for b in bad:
        with pytest.raises(nat.NativeLibraryError):
            _plan([3], **b)
    with pytest.raises(nat.NativeLibraryError, match="negative"):
        _plan([3, -1])
    with pytest.raises(nat.NativeLibraryError, match="2\\^30"):
        _plan([2 ** 30, 2 ** 30])


def test_launch_refusals_without_a_device():
    """Every check comes before the first HIP call."""
    from ah_rag import _native as nat
    lib = nat.lib()
    assert lib.ahr_attn_forward(None, None) == nat.AHR_EINVAL
    plan, *_ = _plan([4, 2], heads=4, kv_heads=2)
    a = nat.AttnArgs()
    a.plan, a.scale, a.lists = ctypes.pointer(plan), 1.0, 4096
    assert lib.ahr_attn_forward(ctypes.byref(a), None) == nat.AHR_EINVAL and b"q: null" in lib.ahr_last_error()
    for t in (a.q, a.k, a.v, a.o):
        t.p, t.ts, t.hs = 4096, 256, 64
    a.scale = 0.0
    assert lib.ahr_attn_forward(ctypes.byref(a), None) == nat.AHR_EINVAL and b"scale" in lib.ahr_last_error()
    a.scale, a.k.p = 1.0, 4098
    assert lib.ahr_attn_forward(ctypes.byref(a), None) == nat.AHR_EINVAL and b"16 bytes" in lib.ahr_last_error()
    a.k.p, a.k.ts = 4096, 257
    assert lib.ahr_attn_forward(ctypes.byref(a), None) == nat.AHR_EINVAL
    a.k.ts = 1 << 24
    assert lib.ahr_attn_forward(ctypes.byref(a), None) == nat.AHR_EUNSUP
    a.k.ts, a.lists = 256, None
    assert lib.ahr_attn_forward(ctypes.byref(a), None) == nat.AHR_EINVAL and b"lists" in lib.ahr_last_error()
    a.lists = 4096
    assert lib.ahr_attn_backward(ctypes.byref(a), None) == nat.AHR_EINVAL and b"backward plan" in lib.ahr_last_error()
    plan, *_ = _plan([4, 2], heads=4, kv_heads=2, backward=1)
    a.plan = ctypes.pointer(plan)
    assert lib.ahr_attn_backward(ctypes.byref(a), None) == nat.AHR_EINVAL and b"workspace" in lib.ahr_last_error()
    r = nat.RopeArgs()
    assert lib.ahr_qk_norm_rope(None, None) == nat.AHR_EINVAL
    r.dtype, r.heads, r.kv_heads, r.head_dim, r.rot = 2, 2, 1, 63, 2
    assert lib.ahr_qk_norm_rope(ctypes.byref(r), None) == nat.AHR_EUNSUP
    r.head_dim, r.rot = 64, 66
    assert lib.ahr_qk_norm_rope(ctypes.byref(r), None) == nat.AHR_EINVAL
    r.rot, r.tokens = 64, 3
    assert lib.ahr_qk_norm_rope(ctypes.byref(r), None) == nat.AHR_EINVAL and b"table" in lib.ahr_last_error()
    n = ctypes.c_int()
    bad = np.asarray([3, -2], np.int32)
    assert lib.ahr_pool_plan_build(bad.ctypes.data, 2, None, 0, ctypes.byref(n)) == nat.AHR_EINVAL
    assert lib.ahr_pool_mean(9, None, 0, 4, None, 0, 0, 0, None, None, None, 0, None) == nat.AHR_EINVAL
    assert lib.ahr_pool_mean(2, None, 0, 4, None, 0, 0, 0, None, None, None, 0, None) == nat.AHR_OK  # empty batch


@pytest.mark.parametrize("lens", [[0, 1, 64, 65, 0, 200], [0], [], [100000, 3, 0, 700]])
def test_pool_lists(lens):
    from ah_rag import _native as nat
    lens = np.asarray(lens, np.int32)
    n = ctypes.c_int()
    nat.check(nat.lib().ahr_pool_plan_build(lens.ctypes.data, len(lens), None, 0, ctypes.byref(n)))
    buf = np.full((n.value + len(lens)) * 4 + 1, -7, np.int32)
    nat.check(nat.lib().ahr_pool_plan_build(lens.ctypes.data, len(lens), buf.ctypes.data, buf.size - 1, ctypes.byref(n)))
    assert buf[-1] == -7
    chunks, seqs = buf[:n.value * 4].reshape(-1, 4), buf[n.value * 4:-1].reshape(-1, 4)
    assert chunks[:, 1].sum() == lens.sum() and (chunks[:, 1] > 0).all()
    assert (chunks[:, 0] == np.concatenate(([0], np.cumsum(chunks[:, 1])))[:-1]).all()
    assert (seqs[:, 0] == lens).all()
    for i, m in enumerate(lens):
        mine = chunks[seqs[i, 1]:seqs[i, 1] + seqs[i, 2]]
        assert (mine[:, 2] == i).all() and mine[:, 1].sum() == m
    assert seqs[:, 2].sum() == n.value
    if buf.size > 2:
        assert nat.lib().ahr_pool_plan_build(lens.ctypes.data, len(lens), buf.ctypes.data, buf.size - 2, ctypes.byref(n)) == nat.AHR_EINVAL


def test_layout_refusals():
    import torch
    from ah_rag.packed import PackedLayout
    for bad in ([1, -1], [1.5], [[1, 2]], [2 ** 30, 1]):
        with pytest.raises(ValueError):
            PackedLayout(bad, device="cuda:0")
    with pytest.raises(ValueError, match="one key length"):
        PackedLayout([1, 2], [3], device="cuda:0")
    with pytest.raises(ValueError, match="ROCm GPU"):
        PackedLayout([1], device="cpu")
    lay = PackedLayout(torch.tensor([2, 0, 3]), [4, 1, 3], device="cuda:0")
    assert (len(lay), lay.tokens, lay.key_tokens) == (3, 5, 8)
    assert PackedLayout([], device="cuda:0").tokens == 0
    mine = np.array([4, 5], np.int32)
    lay = PackedLayout(mine, device="cuda:0")
    mine[:] = 9
    assert lay.lengths.tolist() == [4, 5]


def test_call_refusals():
    import torch
    from ah_rag.packed import PackedLayout, packed_attention, packed_mean_pool, prefix_attention, qk_norm_rope, rotary_table
    lay = PackedLayout([2, 3], device="cuda:0")
    b = torch.bfloat16
    q, k = torch.zeros(5, 4, 64, dtype=b), torch.zeros(5, 2, 64, dtype=b)
    for args in ((q[0], k, k), (q[:4], k, k), (q, k[:4], k[:4]), (q, k, k[:, :1]), (q.float(), k.float(), k.float()),
                 (q, k.half(), k.half()), (q[:, :3], k, k), (q[..., :60], k[..., :60], k[..., :60]), (q, k, k)):
        with pytest.raises(ValueError):  # (the last: tensors on the CPU)
            packed_attention(*args, lay)
    with pytest.raises(ValueError):
        prefix_attention(q, k, k, k[:, :1], k[:, :1], lay)
    cos, sin = rotary_table(7, 64)
    pos = torch.zeros(5, dtype=torch.int32)
    w = torch.ones(64)
    for args in ((q, k[:4], w, w, cos, sin, pos), (q, k, w, None, cos, sin, pos), (q, k, w[:3], w[:3], cos, sin, pos),
                 (q, k, w, w, cos.double(), sin.double(), pos), (q, k, w, w, cos[:, :3], sin, pos), (q, k, w, w, cos, sin, pos.float()),
                 (q, k, w, w, cos, sin, pos[:2]), (q[..., :30], k[..., :30], None, None, cos, sin, pos)):
        with pytest.raises(ValueError):
            qk_norm_rope(*args)
    with pytest.raises(ValueError):
        packed_mean_pool(q, lay)
    with pytest.raises(ValueError):
        packed_mean_pool(q[:4, 0], lay)
    with pytest.raises(ValueError):
        rotary_table(3, 7)


def test_a_table_that_wants_a_gradient_is_refused():
    import torch
    from ah_rag.packed import qk_norm_rope
    x, pos = torch.zeros(3, 2, 8), torch.zeros(3, dtype=torch.int32)
    cos, sin = torch.ones(4, 4), torch.zeros(4, 4)
    for pair in ((cos.clone().requires_grad_(), sin), (cos, sin.clone().requires_grad_())):
        with pytest.raises(ValueError, match="no gradient"):
            qk_norm_rope(x, x, None, None, *pair, pos)


def test_rotary_table_is_exact_far_out():
    import math
    from ah_rag.packed import rotary_table
    cos, sin = rotary_table(100001, 4, 10000.0)
    for p in (0, 1, 99999, 100000):
        for i in range(2):
            a = p * 10000.0 ** (-i / 2)
            assert abs(float(cos[p, i]) - math.cos(a)) < 2 ** -24 and abs(float(sin[p, i]) - math.sin(a)) < 2 ** -24
