"""64-bit restatement of the packed-sequence operators (ah_rag.packed), with bounds of the rounding that
their arithmetic allows. Plain loops over sequences and heads; test infrastructure only."""
from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24  # half a step of fp32


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def visible(nq: int, nk: int, causal: bool) -> torch.Tensor:
    i, j = torch.arange(nq)[:, None], torch.arange(nk)[None, :]
    return (j <= i + nk - nq) if causal else torch.ones(nq, nk, dtype=torch.bool)


def attention(q, k, v, q_lens, k_lens, causal, scale, prefix_k=None, prefix_v=None, d_o=None):
    """(o, tol_o[, (dq, dk, dv), (tol_dq, tol_dk, tol_dv)]) in 64 bits.

    Bounds, with u half a step of the tensors' type. Scores: fp32 sums of dim products, off by at most
    e = (dim + 4) 2^-24 scale sum|q k| in the exponent, so p and the sum of p by a factor e^(2e) at most
    (16 2^-24 more for exp2 and the sum). p is rounded to the type for the second product (u p; below the
    type's normal numbers by an absolute half step, `tiny`, of the row's largest p), o once at the end.
    Gradients: p again (relative to its final value), ds rounded (u), delta from the rounded o (u sum|do o|),
    products in fp32 ((dim + 4) 2^-24 of their absolute sums)."""
    dt = q.dtype
    u = half_step(dt)
    tiny = torch.finfo(dt).tiny * u if dt == torch.float16 else 0.0
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    heads, dim = q.shape[1], q.shape[2]
    group = heads // k.shape[1]
    pk = prefix_k.detach().cpu().double() if prefix_k is not None else None
    pv = prefix_v.detach().cpu().double() if prefix_v is not None else None
    o, tol = torch.zeros_like(q), torch.zeros_like(q)
    if d_o is not None:
        d_o = d_o.detach().cpu().double()
        g = [torch.zeros_like(x) for x in (q, k, v)]
        gt = [torch.zeros_like(x) for x in (q, k, v)]
    q0 = k0 = 0
    for nq, nk in zip(q_lens, k_lens):
        see = visible(nq, nk, causal)
        if pk is not None:
            see = torch.cat((torch.ones(nq, pk.shape[0], dtype=torch.bool), see), 1)
        for h in range(heads):
            hk = h // group
            Q, K, V = q[q0:q0 + nq, h], k[k0:k0 + nk, hk], v[k0:k0 + nk, hk]
            if pk is not None:
                K, V = torch.cat((pk[:, hk], K)), torch.cat((pv[:, hk], V))
            if K.shape[0] == 0 or nq == 0:
                continue
            s = torch.where(see, scale * (Q @ K.T), -math.inf)
            e = (torch.where(see, Q.abs() @ K.abs().T, 0.0).amax(1, keepdim=True) * scale * (dim + 4) + 16) * F32
            m = s.amax(1, keepdim=True)
            any_ = torch.isfinite(m)
            p = torch.where(see, torch.exp(s - torch.where(any_, m, 0.0)), 0.0)
            total = p.sum(1, keepdim=True)
            p = torch.where(any_, p / total, 0.0)
            V_ = torch.where(torch.isfinite(V), V, 0.0)
            out = torch.stack([(p[i][see[i]] @ V[see[i]]) for i in range(nq)])
            o[q0:q0 + nq, h] = out
            # p / sum p: the largest p of a row is 1 / total
            low = tiny * torch.where(any_, 1 / total, 0.0) * see.double() @ V_.abs()
            tol[q0:q0 + nq, h] = (u + 4 * e) * (p @ V_.abs()) + low + u * out.abs() * 1.01 + torch.finfo(dt).tiny * u
            if d_o is None:
                continue
            D = d_o[q0:q0 + nq, h]
            dp = D @ V.T
            delta = (D * out).sum(1, keepdim=True)
            ds = p * (dp - delta)
            f = (dim + 4) * F32
            t_p = p * (u + 4 * e) + tiny
            t_ds = ds.abs() * (u + 4 * e) + p * (f * (D.abs() @ V.abs().T) + 1.01 * u * (D * out).abs().sum(1, keepdim=True)
                                                + (D.abs() * tol[q0:q0 + nq, h]).sum(1, keepdim=True))
            t_ds = torch.where(see, t_ds + ds.abs().max() * u * 2.0 ** -10, 0.0)  # ds is scaled to the type's range
            t_p = torch.where(see, t_p, 0.0)
            g[0][q0:q0 + nq, h] = scale * (ds @ K)
            g[1][k0:k0 + nk, hk] += scale * (ds.T @ Q)
            g[2][k0:k0 + nk, hk] += p.T @ D
            gt[0][q0:q0 + nq, h] = scale * (t_ds @ K.abs())
            gt[1][k0:k0 + nk, hk] += scale * (t_ds.T @ Q.abs())
            gt[2][k0:k0 + nk, hk] += t_p.T @ D.abs()
        q0, k0 = q0 + nq, k0 + nk
    if d_o is None:
        return o, tol
    gt = [t + 1.01 * u * x.abs() + torch.finfo(dt).tiny * u for t, x in zip(gt, g)]
    return o, tol, g, gt


def rotate(x, w, cos, sin, positions, eps, interleaved, dy=None):
    """(y[, dx, dw]) of the norm and rotation of one tensor [tokens, heads, dim], 64 bits."""
    x = x.detach().cpu().double().requires_grad_(dy is not None)
    dim, half = x.shape[2], cos.shape[1]
    w = torch.ones(dim, dtype=torch.float64) if w is None else w.detach().cpu().double()
    w.requires_grad_(dy is not None)
    n = x * w / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) if eps is not None else x * w
    c = cos.cpu().double()[positions.cpu().long()][:, None]
    s = sin.cpu().double()[positions.cpu().long()][:, None]
    if interleaved:
        a, b = n[..., 0:2 * half:2], n[..., 1:2 * half:2]
        r = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = n[..., :half], n[..., half:2 * half]
        r = torch.cat((a * c - b * s, b * c + a * s), -1)
    y = torch.cat((r, n[..., 2 * half:]), -1)
    if dy is None:
        return y.detach()
    dx, dw = torch.autograd.grad(y, (x, w), dy.detach().cpu().double())
    return y.detach(), dx, dw


def mean_pool(rows, lengths, normalize, d_out=None):
    """(out[, d_rows]) in 64 bits."""
    rows = rows.detach().cpu().double()
    out, grad, at = [], torch.zeros_like(rows), 0
    for i, n in enumerate(lengths):
        x = rows[at:at + n]
        m = x.sum(0) / n if n else torch.zeros(rows.shape[1], dtype=torch.float64)
        norm = m.norm().clamp_min(1e-12) if normalize else torch.tensor(1.0, dtype=torch.float64)
        y = m / norm
        out.append(y)
        if d_out is not None and n:
            d = d_out[i].detach().cpu().double()
            if normalize and m.norm() >= 1e-12:
                d = d - y * (y * d).sum()
            grad[at:at + n] = d / norm / n
        at += n
    out = torch.stack(out) if out else torch.zeros(0, rows.shape[1], dtype=torch.float64)
    return out if d_out is None else (out, grad)
