"""Edges of the packed-sequence operators and of the encoder on them that need no GPU."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from test_packed_cpu import _plan


@pytest.mark.parametrize("path", [["."], ["ah-rag_amd"], [".", "ah-rag_amd"], ["ah-rag_amd", "."]], ids="+".join)
def test_the_package_imports_from_the_repository_root(path):
    """With the root, the package's folder or both on the path, in either order: the same package, once."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    prog = ("import sys; sys.path[:0] = %r\n"
            "import ah_rag, ah_rag.packed, importlib\n"
            "from ah_rag.packed import packed_attention\n"
            "assert sys.modules['ah_rag'] is ah_rag and ah_rag.packed is sys.modules['ah_rag.packed']\n"
            "assert packed_attention is ah_rag.packed.packed_attention and importlib.import_module('ah_rag') is ah_rag\n"
            "print(ah_rag.__file__, ah_rag.packed.__file__, list(ah_rag.__path__))" % [os.path.join(root, p) for p in path])
    # (-I: neither the working folder nor PYTHONPATH)
    out = subprocess.run([sys.executable, "-I", "-c", prog], capture_output=True, text=True, timeout=300, cwd="/")
    assert out.returncode == 0, out.stderr
    init, packed, _ = (os.path.normpath(x) for x in out.stdout.split()[:3])
    pkg = os.path.join(root, "ah-rag_amd", "ah_rag")
    assert init == os.path.join(pkg, "__init__.py") and packed == os.path.join(pkg, "packed.py")


def test_forward_mode_derivatives_are_refused():
    """A tangent of any input is refused, whether or not a gradient is wanted too, and before anything else is looked at."""
    import torch.autograd.forward_ad as fwd
    from ah_rag.packed import PackedLayout, packed_attention, packed_mean_pool, prefix_attention, qk_norm_rope
    lay = PackedLayout([3], device="cuda:0")

    def new(*shape, dtype=torch.bfloat16):
        return torch.ones(shape, dtype=dtype)

    x, w, table, pos = new(3, 2, 16), new(16, dtype=torch.float32), new(8, 8, dtype=torch.float32), torch.zeros(3, dtype=torch.int32)
    calls = [(lambda *a: packed_attention(*a, lay), [x, x, x]), (lambda *a: prefix_attention(*a, lay), [x, x, x, x, x]),
             (lambda *a: qk_norm_rope(*a, pos), [x, x, w, w, table, table]), (lambda a: packed_mean_pool(a, lay), [new(3, 16)])]
    with fwd.dual_level():
        for call, args in calls:
            for i, a in enumerate(args):
                for wants in (False, True):
                    dual = fwd.make_dual(a.clone().requires_grad_(wants), torch.ones_like(a))
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        call(*args[:i], dual, *args[i + 1:])
            with pytest.raises((ValueError, RuntimeError)) as e:  # without a tangent: the host tensors are refused
                call(*args)
            assert "forward-mode" not in str(e.value)


@pytest.mark.parametrize("lengths", [[2 ** 62] * 4, [1 << 33], np.array([2 ** 63], np.uint64), np.array([2 ** 64 - 1, 1], np.uint64),
                                     [2 ** 30, 1]], ids=str)
def test_lengths_whose_sum_wraps_are_refused(lengths):
    from ah_rag.packed import PackedLayout
    for a, b in ((lengths, None), ([1] * len(lengths), lengths)):
        with pytest.raises(ValueError, match="2\\*\\*30"):
            PackedLayout(a, b, device="cuda:0")


def test_a_stream_of_another_device_is_refused():
    """(It was left aside, and the call ran on the tensors' device's current stream.)"""
    from types import SimpleNamespace

    from ah_rag.packed import _on
    with pytest.raises(ValueError, match="a stream of cuda:1"):
        _on(SimpleNamespace(device=torch.device("cuda", 1)), torch.device("cuda", 0))


def _tiles(row):
    return -(-(row["pe"] - row["pb"]) // 64) + -(-(row["ke"] - row["kb"]) // 64)


@pytest.mark.parametrize("n", [40, 63, 64, 65, 128, 300, 2000])
@pytest.mark.parametrize("few,many,q", [(1000, 32768, 1), (300, 100000, 1), (1, 9000, 1), (500, 20000, 9)])
@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (12, 12), (8, 1)])
def test_no_row_item_is_left_running_alone(n, few, many, q, heads, kv_heads):
    """One sequence with many keys among others with few: its rows are cut into pieces of no more than one and a half times
    what each of 512 resident workgroups has to do on average (or six tiles), however many sequences there are."""
    kl = [few] * n
    kl[n // 3] = many
    plan, rows, _, join = _plan([q] * n, kl, heads=heads, kv_heads=kv_heads, dim=128, causal=1)
    work = sum(map(_tiles, rows)) * kv_heads
    assert max(map(_tiles, rows)) <= max(6, 1.5 * (work / 512 + 1))
    if n * kv_heads >= 512:  # the others stay whole
        assert len(join) <= 1


@pytest.mark.parametrize("n,keys", [(64, 1000), (128, 4000), (512, 70), (1000, 10000)])
def test_even_batches_take_no_join(n, keys):
    plan, rows, _, join = _plan([1] * n, [keys] * n, heads=32, kv_heads=8, dim=128, causal=1)
    assert not join and plan.ws_bytes == 0 and len(rows) == n


def _part_address(plan, heads, dim, plane, row):
    """Where a partial row lies among the plan's, as the kernels compute it."""
    parts = plan.ws_bytes // (heads * (dim + 1) * 4)
    near = plan.part_rows - plan.far_rows
    at = plane * near + row if row < near else parts - (plane + 1) * plan.far_rows + row - near
    assert 0 <= at < parts
    return at


@pytest.mark.parametrize("q_lens,k_lens,prefix,heads,kv_heads,dim,most", [
    ([1] * 16000, [2] * 8000 + [131072] + [2] * 7999, 2000, 8, 1, 128, 300e6),   # 22 planes for all were 1.45 GB
    ([1] * 4000, [1] * 3999 + [100000], 4000, 8, 1, 128, 150e6),                 # 40 planes, 660 MB
    ([3] * 2000, [90000] + [3] * 1998 + [50000], 3000, 16, 2, 128, 600e6),       # at both ends, several tokens
    ([2, 0, 1] * 3000, ([2, 0, 70000] + [2, 0, 1] * 999) * 3, 1000, 32, 8, 64, 700e6),
    ([1] * 5000, [2] * 5000, 2000, 8, 1, 128, 200e6),                            # none is long: one grid
    ([1] * 60, [3] * 50 + [9000] * 10, 5000, 16, 4, 64, 256e6),                  # long, but a small batch: one grid
])
def test_long_sequences_behind_a_prefix_keep_the_workspace_small(q_lens, k_lens, prefix, heads, kv_heads, dim, most):
    """Every token reads each of its keys and of the prefix's once, no partial row belongs to two of them, and one long
    sequence does not add its planes to every token of a large batch."""
    plan, rows, _, join = _plan(q_lens, k_lens, heads=heads, kv_heads=kv_heads, dim=dim, causal=1, prefix=prefix)
    T, seq_of = sum(q_lens), np.repeat(np.arange(len(q_lens)), q_lens)
    first, k_first = np.cumsum(q_lens) - q_lens, np.cumsum(k_lens) - k_lens
    pre, own, parts, final = ([[] for _ in range(T)] for _ in range(4))
    for r in rows:
        assert 0 < r["nq"] and r["nq"] * heads // kv_heads <= 128 and r["q0"] + r["nq"] <= T
        for i in range(r["nq"]):
            t = r["q0"] + i
            s = seq_of[t]
            if r["pe"] > r["pb"]:
                pre[t].append((r["pb"], r["pe"]))
            if r["ke"] > r["kb"]:
                assert r["k0"] == k_first[s] and r["klen"] == k_lens[s] and r["koff"] + i == k_lens[s] - q_lens[s] + t - first[s]
                own[t].append((r["kb"], r["ke"]))
            (final if r["plane"] < 0 else parts)[t].append((r["plane"], r["prow"] + i))
    used, joined = set(), {}
    for q0, nq, prow, n in join:
        for i in range(nq):
            assert q0 + i not in joined
            joined[q0 + i] = [(j, prow + i) for j in range(n)]
            at = [_part_address(plan, heads, dim, j, prow + i) for j in range(n)]
            near = plan.part_rows - plan.far_rows
            step = near if prow < near else -plan.far_rows
            assert all(b - a == step for a, b in zip(at, at[1:])) and not used.intersection(at)
            used.update(at)
    for t in range(T):
        lim = k_lens[seq_of[t]] - q_lens[seq_of[t]] + t - first[seq_of[t]] + 1
        for spans, stop in ((sorted(pre[t]), prefix), (sorted(own[t]), max(0, lim))):
            end = 0
            for a, b in spans:
                assert a == end or a >= stop  # (a tile's later tokens read further: its pieces past `lim` are hidden)
                end = b
            assert end >= stop
        assert (len(final[t]) == 1 and not parts[t] and t not in joined) or (not final[t] and sorted(parts[t]) == joined[t])
    assert plan.ws_bytes <= most
    work = sum(map(_tiles, rows)) * kv_heads
    assert max(map(_tiles, rows)) <= max(6, 1.5 * (work / 512 + 1))


def test_batches_past_a_launch_are_refused():
    """More workgroups than a launch takes, or a scale whose base-2 form is no number: refused on the host."""
    import ctypes

    from ah_rag import _native as nat
    lib = nat.lib()
    n = (1 << 24) // 12 + 1
    for backward in (0, 1):
        with pytest.raises(nat.NativeLibraryError, match="too many"):
            _plan([1] * n, backward=backward)
    with pytest.raises(nat.NativeLibraryError, match="too many"):  # a prefix apart, whose join has more rows than a launch takes
        _plan([40] * 30, heads=4000, kv_heads=2000, dim=128, prefix=5000)
    many = np.ones(1 << 22, np.int32)
    chunks = ctypes.c_int()
    assert lib.ahr_pool_plan_build(many.ctypes.data, len(many), None, 0, ctypes.byref(chunks)) == nat.AHR_OK
    for call in (lambda: lib.ahr_pool_mean(2, 4096, 8, 8, 4096, chunks.value, len(many), 0, 4096, None, 4096, 1 << 40, None),
                 lambda: lib.ahr_pool_mean_backward(2, 4096, 8, 4096, chunks.value, len(many), 0, 4096, 4096, 4096, None)):
        assert call() == nat.AHR_EUNSUP and b"too many" in lib.ahr_last_error()
    plan, *_ = _plan([4, 2], heads=4, kv_heads=2)
    a = nat.AttnArgs()
    a.plan, a.lists = ctypes.pointer(plan), 4096
    for t in (a.q, a.k, a.v, a.o):
        t.p, t.ts, t.hs = 4096, 256, 64
    a.scale = 2.9e38
    assert lib.ahr_attn_forward(ctypes.byref(a), None) == nat.AHR_EINVAL and b"scale" in lib.ahr_last_error()
