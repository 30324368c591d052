"""Cases of the packed-sequence operators of ah_rag.packed, their plain forms and their exact values.

A packed batch holds the tokens of all its sequences behind each other, with no padding. The operators:

  attention        packed_attention: softmax(scale q k^T) v within each sequence, full or causal, grouped heads
  attention_train  the same with the gradients of q, k and v
  prefix           prefix_attention: every sequence also reads one prefix that the whole batch shares
  rotate           qk_norm_rope: RMS norm of each query and key head and the rotation by its position, one pass
  rotate_train     the same with the gradients of q, k and both norm weights
  pool             packed_mean_pool: the mean of each sequence's rows, L2-normalised
  pool_train       the same with the gradient of the rows

`own` False: elementary torch operations in 32 bits on padded batches. `own` True: the framework's calls.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
BASE = 10000.0


def listed():
    return [
        # a handful of search queries through the smaller sentence encoder's heads: latency counts
        dict(name="attention queries", op="attention", dtype="bf16", n=16, lo=3, hi=14, keys_lo=0, keys_hi=0, heads=12,
             kv_heads=12, dim=32, causal=False),
        # one batch of node texts of the corpus encode (256 texts, up to 384 tokens, 12 heads of 64)
        dict(name="attention corpus", op="attention", dtype="bf16", n=256, lo=8, hi=384, keys_lo=0, keys_hi=0, heads=12,
             kv_heads=12, dim=64, causal=False),
        # whole documents through a causal encoder with grouped heads
        dict(name="attention documents", op="attention", dtype="bf16", n=4, lo=1500, hi=8191, keys_lo=0, keys_hi=0,
             heads=32, kv_heads=8, dim=128, causal=True),
        # one new token for each of a batch of sequences over the keys that they hold
        dict(name="attention single tokens", op="attention", dtype="f16", n=24, lo=1, hi=1, keys_lo=1000, keys_hi=32768,
             heads=32, kv_heads=8, dim=128, causal=True),
        # a fine-tuning step's attention on short texts
        dict(name="attention train texts", op="attention_train", dtype="bf16", n=64, lo=8, hi=384, keys_lo=0, keys_hi=0,
             heads=12, kv_heads=12, dim=64, causal=False),
        # a fine-tuning step's attention on documents, causal, grouped heads
        dict(name="attention train documents", op="attention_train", dtype="bf16", n=3, lo=700, hi=4100, keys_lo=0,
             keys_hi=0, heads=16, kv_heads=4, dim=128, causal=True),
        # queries that all begin with the same instruction
        dict(name="prefix queries", op="prefix", dtype="bf16", prefix=900, n=64, lo=4, hi=40, keys_lo=0, keys_hi=0,
             heads=16, kv_heads=8, dim=64, causal=True),
        # one new token for each of many sequences that share a long retrieved context
        dict(name="prefix single tokens", op="prefix", dtype="f16", prefix=16000, n=200, lo=1, hi=1, keys_lo=1,
             keys_hi=200, heads=32, kv_heads=8, dim=128, causal=True),
        # the heads of a few queries
        dict(name="rotate queries", op="rotate", dtype="bf16", n=16, lo=3, hi=14, heads=16, kv_heads=8, dim=128),
        # the heads of a batch of documents, with gradients
        dict(name="rotate train documents", op="rotate_train", dtype="bf16", n=5, lo=1000, hi=8000, heads=32, kv_heads=8,
             dim=128),
        # the encoder's last step for one batch of node texts
        dict(name="pool corpus", op="pool", dtype="bf16", n=256, lo=8, hi=384, width=768),
        # the same for documents, with its gradient
        dict(name="pool train documents", op="pool_train", dtype="f16", n=12, lo=100, hi=8000, width=1024),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "attention_train", "attention_train", "prefix", "prefix",
                     "rotate", "rotate_train", "pool", "pool_train"))
    case = dict(op=op, dtype=rng.choice(("bf16", "bf16", "f16")))
    n = _spread(rng, 1, 256)
    if op.startswith("pool"):
        hi = _spread(rng, 8, 8000)
        width = _spread(rng, 100, 2048)
        cap = 48000000  # values of the rows
        n = max(1, min(n, cap // (hi * width)))
        return dict(case, n=n, lo=min(hi, _spread(rng, 1, 64)), hi=hi, width=width)
    dim = rng.choice((32, 48, 64, 64, 80, 96, 128, 128))
    kv_heads = rng.choice((1, 2, 3, 4, 6, 8, 12))
    heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 5, 8)) if kv_heads < 5 else kv_heads * rng.choice((1, 1, 2, 4))
    if op.startswith("rotate"):
        hi = _spread(rng, 8, 8000)
        cap = 100000000  # values of the heads
        n = max(1, min(n, cap // (hi * (heads + kv_heads) * dim)))
        return dict(case, n=n, lo=min(hi, _spread(rng, 1, 1000)), hi=hi, heads=heads, kv_heads=kv_heads, dim=dim)
    case.update(heads=heads, kv_heads=kv_heads, dim=dim, causal=True)
    if op == "prefix":
        hi = _spread(rng, 1, 64)
        keys = _spread(rng, hi, 400) if rng.random() < 0.4 else 0
        return dict(case, prefix=_spread(rng, 100, 16000), n=max(1, min(n, 6400 // (hi * heads))), lo=rng.randint(1, hi),
                    hi=hi, keys_lo=min(hi, keys), keys_hi=keys)
    if op == "attention" and rng.random() < 0.3:  # a few tokens over long keys
        hi = rng.choice((1, 1, 1, 2, 5))
        keys = _spread(rng, 64, 32768)
        n = max(1, min(n, 24 * 32768 // keys))
        return dict(case, n=n, lo=1, hi=hi, keys_lo=max(hi, keys // 30), keys_hi=keys)
    hi = _spread(rng, 8, 8191 if op == "attention" else 4100)
    cap = 3.0e9 if op == "attention" else 5.0e8  # scores of the padded batch
    n = max(1, min(n, int(cap // (heads * hi * hi))))
    return dict(case, n=n, lo=min(hi, _spread(rng, 1, 1500)), hi=hi, keys_lo=0, keys_hi=0, causal=rng.random() < 0.5)


def _lengths(n, lo, hi):
    """Ragged lengths from lo to hi, both among them where n allows: short ones are more frequent, the order is mixed."""
    got = [lo + int((hi - lo) * ((i * 0.6180339887498949) % 1.0) ** 1.6) for i in range(n)]
    got[n // 2] = hi
    return got


def _key_lengths(case):
    """Of each sequence: as many keys as queries, or (where the case says so) its own number, never fewer."""
    q = _lengths(case["n"], case["lo"], case["hi"])
    if not case["keys_hi"]:
        return q, q
    return q, [max(a, b) for a, b in zip(q, _lengths(case["n"], case["keys_lo"], case["keys_hi"]))]


def _pad_index(lengths, device):
    """[n, longest] places in the packed rows, and which of them are rows of the sequence."""
    n = torch.tensor(lengths, device=device)
    at = torch.arange(max(lengths), device=device)
    real = at < n[:, None]
    start = torch.cumsum(n, 0) - n
    return torch.where(real, start[:, None] + at, 0), real


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    op = case["op"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    s = {"case": case}
    if op.startswith("pool"):
        lengths = _lengths(case["n"], case["lo"], case["hi"])
        # hidden states: each width entry has an offset of its own, as after a norm with a learnt shift
        rows = (normal(sum(lengths), case["width"]) + 0.5 * normal(case["width"])).to(dt)
        s["rows"] = rows.requires_grad_(op == "pool_train")
        s["d_out"] = normal(case["n"], case["width"])
        s["at"], s["real"] = _pad_index(lengths, dev)
        s["lengths"] = torch.tensor(lengths, device=dev)
        s["layout"] = _layout(lengths, None, dev)
        return s
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if op.startswith("rotate"):
        lengths = _lengths(case["n"], case["lo"], case["hi"])
        t = sum(lengths)
        qkv = normal(t, (hq + 2 * hk) * d).to(dt)  # one projection's output: the heads are views of it
        s["q"] = qkv[:, :hq * d].view(t, hq, d)
        s["k"] = qkv[:, hq * d:(hq + hk) * d].view(t, hk, d)
        s["wq"], s["wk"] = 1 + 0.1 * normal(d), 1 + 0.1 * normal(d)
        angle = torch.arange(max(lengths), device=dev, dtype=torch.float64)[:, None] * BASE ** (
            -torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        at, real = _pad_index(lengths, dev)
        s["positions"] = torch.arange(max(lengths), device=dev, dtype=torch.int32).expand(at.shape)[real].contiguous()
        if op == "rotate_train":
            for name in ("q", "k", "wq", "wk"):
                s[name] = s[name].detach().requires_grad_()
            s["dq"], s["dk"] = normal(t, hq, d).to(dt), normal(t, hk, d).to(dt)
        return s
    lq, lk = _key_lengths(case)
    t, tk = sum(lq), sum(lk)
    if case["keys_hi"]:
        s["q"], s["k"], s["v"] = normal(t, hq, d).to(dt), normal(tk, hk, d).to(dt), normal(tk, hk, d).to(dt)
    else:
        qkv = normal(t, (hq + 2 * hk) * d).to(dt)  # one projection's output: the heads are views of it
        s["q"] = qkv[:, :hq * d].view(t, hq, d)
        s["k"] = qkv[:, hq * d:(hq + hk) * d].view(t, hk, d)
        s["v"] = qkv[:, (hq + hk) * d:].view(t, hk, d)
    if op == "prefix":
        s["prefix_k"], s["prefix_v"] = normal(case["prefix"], hk, d).to(dt), normal(case["prefix"], hk, d).to(dt)
    if op == "attention_train":
        for name in ("q", "k", "v"):
            s[name] = s[name].detach().requires_grad_()
        s["d_out"] = normal(t, hq, d).to(dt)
    s["at_q"], s["real_q"] = _pad_index(lq, dev)
    s["at_k"], s["real_k"] = _pad_index(lk, dev)
    # [n, 1, 1, queries, keys]: which keys a query may read
    allowed = s["real_k"][:, None, :].expand(-1, max(lq), -1)
    if case["causal"]:
        past = torch.tensor(lk, device=dev) - torch.tensor(lq, device=dev)
        i, j = torch.arange(max(lq), device=dev), torch.arange(max(lk), device=dev)
        allowed = allowed & (j <= i[:, None] + past[:, None, None])
    s["allowed"] = allowed[:, None, None]
    s["layout"] = _layout(lq, lk, dev)
    return s


def _layout(lengths, key_lengths, dev):
    """The handle that a program keeps for a batch: made once, used by every layer."""
    if own:
        from ah_rag.packed import PackedLayout
        return PackedLayout(lengths, key_lengths=key_lengths, device=dev)
    return None


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        op = state["case"]["op"]
        if op.startswith("pool"):
            return _plain_pool(state)
        if op.startswith("rotate"):
            return _plain_rotate(state)
        return _plain_attention(state)


def _run_own(s):
    from ah_rag.packed import packed_attention, packed_mean_pool, prefix_attention, qk_norm_rope
    case = s["case"]
    op = case["op"]
    if op == "attention":
        return packed_attention(s["q"], s["k"], s["v"], s["layout"], causal=case["causal"])
    if op == "attention_train":
        out = packed_attention(s["q"], s["k"], s["v"], s["layout"], causal=case["causal"])
        return out.detach(), torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["d_out"])
    if op == "prefix":
        return prefix_attention(s["q"], s["k"], s["v"], s["prefix_k"], s["prefix_v"], s["layout"], causal=case["causal"])
    if op == "rotate":
        return qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["positions"], eps=EPS)
    if op == "rotate_train":
        out = qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["cos"], s["sin"], s["positions"], eps=EPS)
        grads = torch.autograd.grad(out, (s["q"], s["k"], s["wq"], s["wk"]), (s["dq"], s["dk"]))
        return tuple(x.detach() for x in out), grads
    if op == "pool":
        return packed_mean_pool(s["rows"], s["layout"], normalize=True)
    out = packed_mean_pool(s["rows"], s["layout"], normalize=True)
    return out.detach(), torch.autograd.grad(out, (s["rows"],), s["d_out"])


# ---- plain forms -----------------------------------------------------------------------------


def _plain_attention(s):
    case = s["case"]
    hk, d = case["kv_heads"], case["dim"]
    group = case["heads"] // hk
    scale = d ** -0.5
    n, rows = s["at_q"].shape

    def padded(x, at, per):  # [n, kv heads, per, rows, dim], in 32 bits
        return x[at].float().view(*at.shape, hk, per, d).permute(0, 2, 3, 1, 4)

    def packed(x, real, dtype):
        x = x.permute(0, 3, 1, 2, 4)
        return x.reshape(*x.shape[:2], -1, d)[real].to(dtype)

    q = padded(s["q"], s["at_q"], group)
    k, v = padded(s["k"], s["at_k"], 1), padded(s["v"], s["at_k"], 1)
    dtype = s["q"].dtype
    # one product for each sequence and key head, with its group's query heads as further rows
    flat = q.reshape(n, hk, group * rows, d)
    score = torch.matmul(flat, k[:, :, 0].transpose(-1, -2)).view(n, hk, group, rows, -1)
    score.mul_(scale).masked_fill_(~s["allowed"], -math.inf)
    if case["op"] == "prefix":
        pk, pv = s["prefix_k"].float().permute(1, 0, 2), s["prefix_v"].float().permute(1, 0, 2)
        every = q.permute(1, 0, 2, 3, 4).reshape(hk, -1, d)
        before = torch.matmul(every, pk.transpose(-1, -2)).mul_(scale)
        before = before.view(hk, n, group, rows, -1).permute(1, 0, 2, 3, 4)
        top = torch.maximum(score.amax(-1, keepdim=True), before.amax(-1, keepdim=True))
        p, b = torch.exp(score - top), torch.exp(before - top)
        total = p.sum(-1, keepdim=True) + b.sum(-1, keepdim=True)
        out = torch.matmul(p.view(n, hk, group * rows, -1), v[:, :, 0]).view(n, hk, group, rows, d)
        shared = torch.matmul(b.permute(1, 0, 2, 3, 4).reshape(hk, n * group * rows, -1), pv)
        out = (out + shared.view(hk, n, group, rows, d).permute(1, 0, 2, 3, 4)) / total
        return packed(out, s["real_q"], dtype)
    p = torch.exp(score.sub_(score.amax(-1, keepdim=True)))
    p /= p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(n, hk, group * rows, -1), v[:, :, 0]).view(n, hk, group, rows, d)
    if case["op"] == "attention":
        return packed(out, s["real_q"], dtype)
    d_out = padded(s["d_out"], s["at_q"], group) * s["real_q"][:, None, None, :, None]
    d_flat = d_out.reshape(n, hk, group * rows, d)
    p_flat = p.view(n, hk, group * rows, -1)
    d_v = torch.matmul(p_flat.transpose(-1, -2), d_flat)
    d_p = torch.matmul(d_flat, v[:, :, 0].transpose(-1, -2))
    d_s = p_flat * (d_p - (d_out * out).sum(-1).view(n, hk, group * rows, 1)) * scale
    d_q = torch.matmul(d_s, k[:, :, 0]).view(n, hk, group, rows, d)
    d_k = torch.matmul(d_s.transpose(-1, -2), flat)
    return packed(out, s["real_q"], dtype), (packed(d_q, s["real_q"], dtype), packed(d_k[:, :, None], s["real_k"], dtype),
                                             packed(d_v[:, :, None], s["real_k"], dtype))


def _plain_rotate(s):
    cos, sin = s["cos"][s["positions"].long()][:, None], s["sin"][s["positions"].long()][:, None]

    def forward(x, w):
        x = x.float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        a, b = (x * r * w).chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    def backward(x, w, dy):
        x, dy = x.float(), dy.float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        a, b = dy.chunk(2, -1)
        dn = torch.cat((a * cos + b * sin, b * cos - a * sin), -1)  # the rotation the other way
        dw = (dn * x * r).sum((0, 1))
        dn = dn * w
        return r * (dn - x * r * r * (dn * x).mean(-1, keepdim=True)), dw

    dt = s["q"].dtype
    out = forward(s["q"], s["wq"]).to(dt), forward(s["k"], s["wk"]).to(dt)
    if s["case"]["op"] == "rotate":
        return out
    dq, dwq = backward(s["q"], s["wq"], s["dq"])
    dk, dwk = backward(s["k"], s["wk"], s["dk"])
    return out, (dq.to(dt), dk.to(dt), dwq, dwk)


def _plain_pool(s):
    rows = s["rows"][s["at"]].float() * s["real"][..., None]
    mean = rows.sum(1) / s["lengths"][:, None]
    norm = mean.square().sum(-1, keepdim=True).sqrt().clamp_min(1e-12)
    out = mean / norm
    if s["case"]["op"] == "pool":
        return out
    d_mean = (s["d_out"] - out * (out * s["d_out"]).sum(-1, keepdim=True)) / norm / s["lengths"][:, None]
    d_rows = d_mean[:, None].expand(rows.shape)[s["real"]].to(s["rows"].dtype)
    return out, (d_rows,)


# ---- what a pass cannot do without -----------------------------------------------------------


def _pairs(case):
    """Queries times the keys that they may read, of one head."""
    lq, lk = _key_lengths(case)
    if not case["causal"]:
        return sum(a * b for a, b in zip(lq, lk))
    return sum(a * (b - a) + a * (a + 1) // 2 for a, b in zip(lq, lk))


def work(case):
    op, size = case["op"], 2
    if op.startswith("pool"):
        rows = sum(_lengths(case["n"], case["lo"], case["hi"])) * case["width"]
        out = case["n"] * case["width"] * 4
        train = op == "pool_train"
        return {"bytes": rows * size * (2 if train else 1) + out * (2 if train else 1), "flops": rows * (2 if train else 1)}
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if op.startswith("rotate"):
        t = sum(_lengths(case["n"], case["lo"], case["hi"]))
        values = t * (hq + hk) * d
        train = op == "rotate_train"
        return {"bytes": values * size * (4 if train else 2) + t * 4 + case["hi"] * d * 4, "flops": values * (20 if train else 7)}
    lq, lk = _key_lengths(case)
    t, tk = sum(lq), sum(lk)
    pairs = _pairs(case) + (t * case["prefix"] if op == "prefix" else 0)
    moved = (2 * t * hq + 2 * tk * hk) * d * size
    if op == "prefix":
        moved += 2 * case["prefix"] * hk * d * size
    if op == "attention_train":
        return {"bytes": moved + (2 * t * hq + 2 * tk * hk) * d * size, "flops": 14.0 * d * hq * pairs}
    return {"bytes": moved, "flops": 4.0 * d * hq * pairs}


# ---- the definitions in 64 bits --------------------------------------------------------------


def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    op = case["op"]
    with torch.no_grad():
        if op.startswith("pool"):
            outs, grads, first = [], [], 0
            for i, length in enumerate(_lengths(case["n"], case["lo"], case["hi"])):
                x = s["rows"][first:first + length].double()
                first += length
                mean = x.sum(0) / length
                norm = torch.linalg.vector_norm(mean)
                y = mean / norm
                outs.append(y)
                # d(mean / |mean|) = (I - y y^T) / |mean|, the same for each of the rows
                dy = s["d_out"][i].double()
                grads.append(((dy - y * torch.dot(y, dy)) / (norm * length)).expand(length, -1))
            return torch.stack(outs) if op == "pool" else (torch.stack(outs), (torch.cat(grads),))
        if op.startswith("rotate"):
            outs, gx, gw = [], [], []
            c, z = s["cos"].double()[s["positions"].long()], s["sin"].double()[s["positions"].long()]
            turn = torch.complex(c, z)[:, None]
            half = case["dim"] // 2
            for x, w, name in ((s["q"], s["wq"], "dq"), (s["k"], s["wk"], "dk")):
                x, w = x.double(), w.double()
                length = (x.square().sum(-1, keepdim=True) / case["dim"] + EPS).sqrt()
                u = x / length
                y = u * w
                y = torch.complex(y[..., :half], y[..., half:]) * turn
                outs.append(torch.cat((y.real, y.imag), -1))
                if op == "rotate_train":
                    e = s[name].double()
                    e = torch.complex(e[..., :half], e[..., half:]) * turn.conj()
                    e = torch.cat((e.real, e.imag), -1)
                    gw.append((e * u).sum((0, 1)))
                    e = e * w
                    gx.append((e - u * (e * u).sum(-1, keepdim=True) / case["dim"]) / length)
            return tuple(outs) if op == "rotate" else (tuple(outs), (*gx, *gw))
        lq, lk = _key_lengths(case)
        group, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["dim"])
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        train = op == "attention_train"
        g_q = torch.zeros_like(out) if train else None
        g_k = torch.zeros(s["k"].shape, dtype=torch.float64, device=out.device) if train else None
        g_v = torch.zeros_like(g_k) if train else None
        for h in range(case["heads"]):
            hk, q0, k0 = h // group, 0, 0
            keys, vals = s["k"][:, hk].double(), s["v"][:, hk].double()
            queries = s["q"][:, h].double()
            more = (s["prefix_k"][:, hk].double(), s["prefix_v"][:, hk].double()) if op == "prefix" else None
            for a, b in zip(lq, lk):
                q, k, v = queries[q0:q0 + a], keys[k0:k0 + b], vals[k0:k0 + b]
                w = scale * (q @ k.T)
                if case["causal"]:
                    w = w + torch.full((a, b), -math.inf, dtype=torch.float64, device=w.device).triu_(b - a + 1)
                if more:
                    w = torch.cat((scale * (q @ more[0].T), w), 1)
                    v = torch.cat((more[1], v))
                p = torch.softmax(w, 1)
                o = p @ v
                out[q0:q0 + a, h] = o
                if train:
                    do = s["d_out"][q0:q0 + a, h].double()
                    g = do @ v.T
                    g = scale * p * (g - (p * g).sum(1, keepdim=True))
                    g_q[q0:q0 + a, h] = g @ k
                    g_k[k0:k0 + b, hk] += g.T @ q
                    g_v[k0:k0 + b, hk] += p.T @ do
                q0, k0 = q0 + a, k0 + b
        return (out, (g_q, g_k, g_v)) if train else out
