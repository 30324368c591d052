"""ah_rag.packed — operators of a transformer over packed sequences, on the MI355X.

A packed batch holds the tokens of all its sequences behind each other: [tokens, heads, head_dim], no
padding. A sentence encoder's batches are texts of very different lengths, so padding them to the
longest costs both the padded tokens' projections and the square of the padded length in attention.

  PackedLayout       the lengths of one batch and the kernels' work lists for them: made once, used by
                     every layer and by the backward pass
  packed_attention   softmax(scale q k^T) v within each sequence: full or causal, grouped heads, more keys
                     than queries (single tokens over long keys among them); differentiable
  prefix_attention   the same where every sequence also reads one prefix that the batch shares
  qk_norm_rope       RMS norm of each query and key head and the rotation by its position, in one pass;
                     differentiable
  rotary_table       cos and sin of that rotation's angles, computed in 64 bits
  packed_mean_pool   mean of each sequence's rows in fp32, optionally L2-normalised; differentiable

Everything runs in libahr_hip.so (include/ahr.h); there is no CPU fallback. Calls are enqueued on the
current stream of the tensors' device (or `stream`), synchronise nothing and may be captured into a
hipGraph once a layout has served a call of the same shape (its work lists are copied to the device
then). Tensors that the kernels cannot read in place (rows that do not start at multiples of 16
bytes, a strided last dimension) are copied first.

Replaces, behind the reference's SentenceTransformer.encode seam
(src/ah_rag/graph/hierarchical_graph.py:655-656, :709-712), that library's padded attention and
pooling.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
from typing import Dict, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _native as nat

_CODES = {torch.float32: nat.AHR_F32, torch.float16: nat.AHR_F16, torch.bfloat16: nat.AHR_BF16}
Lengths = Union[Sequence[int], np.ndarray, torch.Tensor]


def _host_lengths(x: Lengths, what: str) -> np.ndarray:
    if isinstance(x, torch.Tensor):
        if x.device.type != "cpu":
            raise ValueError(f"{what} must be on the host (the work lists are laid out there)")
        x = x.numpy()
    a = np.asarray(x)
    if a.size == 0:
        a = a.astype(np.int64).reshape(-1)
    if a.ndim != 1 or a.dtype.kind not in "iu":
        raise ValueError(f"{what} must be a list of whole numbers")
    if a.size and (a.min() < 0 or int(a.sum(dtype=np.int64)) > 1 << 30):
        raise ValueError(f"{what} must be >= 0 and sum to at most 2**30")
    return np.ascontiguousarray(a, dtype=np.int32)


class PackedLayout:
    """Lengths of a batch of packed sequences: `lengths[i]` tokens (queries), `key_lengths[i]` keys
    (default: as many). Zero lengths are allowed. The layout keeps the device work lists of each head
    shape that it has served; it may be used on any stream."""

    def __init__(self, lengths: Lengths, key_lengths: Optional[Lengths] = None,
                 device: Optional[Union[int, str, torch.device]] = None) -> None:
        self.lengths = _host_lengths(lengths, "lengths")
        self.key_lengths = self.lengths if key_lengths is None else _host_lengths(key_lengths, "key_lengths")
        if len(self.key_lengths) != len(self.lengths):
            raise ValueError("one key length per sequence")
        if device is None or isinstance(device, int):
            device = torch.device("cuda", torch.cuda.current_device() if device is None else device)
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("a PackedLayout serves a ROCm GPU")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.tokens = int(self.lengths.sum(dtype=np.int64))
        self.key_tokens = int(self.key_lengths.sum(dtype=np.int64))
        self._plans: Dict[tuple, Tuple[nat.AttnPlan, Optional[torch.Tensor]]] = {}
        self._pool: Optional[Tuple[int, torch.Tensor]] = None
        self._positions: Optional[torch.Tensor] = None

    def __len__(self) -> int:
        return len(self.lengths)

    def _upload(self, host: np.ndarray) -> torch.Tensor:
        with torch.cuda.device(self.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a layout's first call for a shape copies its work lists to the device: make it "
                                   "before the capture")
            # a blocking copy: the lists are complete for every stream
            return torch.from_numpy(host).to(self.device)

    def positions(self) -> torch.Tensor:
        """int32 [tokens] on the device: each token's position among its sequence's keys (0, 1, ... where
        there are as many keys as queries; with more keys the queries are the last ones)."""
        if self._positions is None:
            n = self.lengths.astype(np.int64)
            first = np.cumsum(n) - n
            past = self.key_lengths.astype(np.int64) - n
            self._positions = self._upload((np.arange(self.tokens) + np.repeat(past - first, n)).astype(np.int32))
        return self._positions

    def _plan(self, dtype: int, heads: int, kv_heads: int, dim: int, causal: bool, backward: bool,
              prefix: int) -> Tuple[nat.AttnPlan, Optional[torch.Tensor]]:
        key = (dtype, heads, kv_heads, dim, causal, backward, prefix)
        got = self._plans.get(key)
        if got is None:
            lib = nat.lib()
            shape = nat.AttnShape(dtype, heads, kv_heads, dim, int(causal), int(backward), prefix)
            plan = nat.AttnPlan()
            args = (self.lengths.ctypes.data, self.key_lengths.ctypes.data, len(self.lengths), ctypes.byref(shape),
                    ctypes.byref(plan))
            nat.check(lib.ahr_attn_plan_build(*args, None, 0), "ahr_attn_plan_build")
            lists = None
            if plan.ints:
                buf = np.empty(plan.ints, np.int32)
                nat.check(lib.ahr_attn_plan_build(*args, buf.ctypes.data, buf.size), "ahr_attn_plan_build")
                lists = self._upload(buf)
            got = self._plans[key] = (plan, lists)
        return got

    def _pool_lists(self) -> Tuple[int, torch.Tensor]:
        if self._pool is None:
            n = ctypes.c_int()
            args = (self.lengths.ctypes.data, len(self.lengths))
            nat.check(nat.lib().ahr_pool_plan_build(*args, None, 0, ctypes.byref(n)), "ahr_pool_plan_build")
            buf = np.zeros(max(4, n.value * 4 + 2 * len(self.lengths)), np.int32)
            nat.check(nat.lib().ahr_pool_plan_build(*args, buf.ctypes.data, buf.size, ctypes.byref(n)), "ahr_pool_plan_build")
            self._pool = (n.value, self._upload(buf))
        return self._pool


# ---- shared checks ---------------------------------------------------------------------------


def _heads(t: torch.Tensor, what: str, like: Optional[torch.Tensor] = None, tokens: Optional[int] = None) -> None:
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"{what} must be a [tokens, heads, head_dim] tensor")
    if like is not None and (t.dtype != like.dtype or t.device != like.device or t.shape[2] != like.shape[2]):
        raise ValueError(f"{what} must have q's dtype, device and head_dim")
    if tokens is not None and t.shape[0] != tokens:
        raise ValueError(f"{what} has {t.shape[0]} tokens, the layout {tokens}")


def _on_device(device: torch.device, *tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"tensors must be on {device}, got one on {t.device}")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy whose rows start at multiples of 16 bytes and are contiguous."""
    per = 16 // t.element_size()
    n, h, d = t.shape
    ts, hs, es = t.stride()
    if ((es == 1 or d == 1) and t.data_ptr() % 16 == 0 and (n < 2 or (ts % per == 0 and ts <= 1 << 23))
            and (h < 2 or (hs % per == 0 and hs * h <= 1 << 29))):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _tensor3(to: nat.Tensor3, t: torch.Tensor) -> None:
    to.p = t.data_ptr()
    # (the stride of an axis of one element is arbitrary)
    to.ts = t.stride(0) if t.shape[0] > 1 else 0
    to.hs = t.stride(1) if t.shape[1] > 1 else 0


@contextlib.contextmanager
def _on(stream: Optional[torch.cuda.Stream], device: torch.device, *tensors: Optional[torch.Tensor]):
    """Run on the tensors' device and, if given, on `stream`, after the current stream's work."""
    with torch.cuda.device(device):
        if stream is None or stream == torch.cuda.current_stream(device):
            yield
            return
        stream.wait_stream(torch.cuda.current_stream(device))
        for t in tensors:
            if t is not None:
                t.record_stream(stream)
        with torch.cuda.stream(stream):
            yield


def _keep(lists: Optional[torch.Tensor], device: torch.device) -> None:
    """The layout may be dropped while the current stream still reads its lists."""
    if lists is not None and not torch.cuda.is_current_stream_capturing():
        lists.record_stream(torch.cuda.current_stream(device))


# ---- attention -------------------------------------------------------------------------------


def _attention(q, k, v, layout, causal, scale, lse, prefix_k=None, prefix_v=None, out=None) -> torch.Tensor:
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    tokens, heads, dim = q.shape
    plan, lists = layout._plan(_CODES[q.dtype], heads, k.shape[1], dim, causal, False,
                               0 if prefix_k is None else prefix_k.shape[0])
    o = torch.empty((tokens, heads, dim), dtype=q.dtype, device=q.device) if out is None else out
    a = nat.AttnArgs()
    a.plan = ctypes.pointer(plan)
    a.lists = nat.ptr(lists)
    a.scale = scale
    for to, t in ((a.q, q), (a.k, k), (a.v, v), (a.o, o)):
        _tensor3(to, t)
    if prefix_k is not None:
        prefix_k, prefix_v = _aligned(prefix_k), _aligned(prefix_v)
        _tensor3(a.prefix_k, prefix_k)
        _tensor3(a.prefix_v, prefix_v)
    a.lse = nat.ptr(lse)
    if plan.ws_bytes:
        ws = torch.empty(plan.ws_bytes, dtype=torch.uint8, device=q.device)
        a.ws, a.ws_bytes = ws.data_ptr(), plan.ws_bytes
    nat.check(nat.lib().ahr_attn_forward(ctypes.byref(a), nat.stream_ptr(device_index=q.device.index)), "ahr_attn_forward")
    _keep(lists, q.device)
    return o


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, layout, causal, scale):
        q, k, v = _aligned(q), _aligned(k), _aligned(v)
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
        o = _attention(q, k, v, layout, causal, scale, lse)
        # the backward pass's lists too: its first call may be inside a capture
        layout._plan(_CODES[q.dtype], q.shape[1], k.shape[1], q.shape[2], causal, True, 0)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.layout, ctx.causal, ctx.scale = layout, causal, scale
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o):
        q, k, v, o, lse = ctx.saved_tensors
        with torch.cuda.device(q.device):
            plan, lists = ctx.layout._plan(_CODES[q.dtype], q.shape[1], k.shape[1], q.shape[2], ctx.causal, True, 0)
            d_o, o = _aligned(d_o), _aligned(o)
            dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
            a = nat.AttnArgs()
            a.plan = ctypes.pointer(plan)
            a.lists = nat.ptr(lists)
            a.scale = ctx.scale
            for to, t in ((a.q, q), (a.k, k), (a.v, v), (a.o, o), (a.d_o, d_o), (a.dq, dq), (a.dk, dk), (a.dv, dv)):
                _tensor3(to, t)
            a.lse = lse.data_ptr()
            if plan.ws_bytes:
                ws = torch.empty(plan.ws_bytes, dtype=torch.uint8, device=q.device)
                a.ws, a.ws_bytes = ws.data_ptr(), plan.ws_bytes
            nat.check(nat.lib().ahr_attn_backward(ctypes.byref(a), nat.stream_ptr(device_index=q.device.index)),
                      "ahr_attn_backward")
            _keep(lists, q.device)
        return dq, dk, dv, None, None, None


def _check_attention(q, k, v, layout, scale) -> float:
    _heads(q, "q", tokens=layout.tokens)
    _heads(k, "k", q, layout.key_tokens)
    _heads(v, "v", q, layout.key_tokens)
    if v.shape != k.shape:
        raise ValueError("v must have k's shape")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"attention takes float16 and bfloat16, got {q.dtype}")
    if k.shape[1] < 1 or q.shape[1] < 1 or q.shape[1] % k.shape[1] or q.shape[1] // k.shape[1] > 128:
        raise ValueError(f"{q.shape[1]} query heads do not share {k.shape[1]} key heads (a multiple, at most 128 each)")
    dim = q.shape[2]
    if dim < 8 or dim % 8 or dim > 128:
        raise ValueError(f"head_dim must be a multiple of 8, at most 128, got {dim}")
    _on_device(layout.device, q, k, v)
    scale = dim ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    return scale


def _check_out(out: Optional[torch.Tensor], q: torch.Tensor) -> None:
    if out is None:
        return
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError("out must have q's shape, dtype and device")
    if _aligned(out) is not out:
        raise ValueError("out's rows must be contiguous and start at multiples of 16 bytes")


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, layout: PackedLayout, causal: bool = False,
                     scale: Optional[float] = None, stream: Optional[torch.cuda.Stream] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q k^T) v within each sequence of the layout -> [tokens, heads, head_dim].

    q [tokens, heads, head_dim], k and v [key_tokens, kv_heads, head_dim] in float16 or bfloat16; heads a
    multiple of kv_heads (query head i reads key head i * kv_heads // heads); head_dim a multiple of 8 up
    to 128; any strides. scale: default head_dim ** -0.5. causal: query i of a sequence with n queries
    and m keys reads the keys j <= i + m - n (the last query reads all). A row that reads no key gives
    zeros, and zero gradients. Scores, sums and accumulators are fp32; the weights p are rounded to the
    tensors' type for the product with v, and o once at the end.

    Differentiable in q, k and v (no atomics: repeated runs give the same bits). `out`, where no gradient
    is wanted: written in place of a new tensor; it must not overlap the inputs. `stream`: runs there,
    after the current stream's work; the caller orders what follows. A value that is not finite stays
    within its own sequence."""
    scale = _check_attention(q, k, v, layout, scale)
    _check_out(out, q)
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if grad and out is not None:
        raise ValueError("out cannot be given where a gradient is wanted")
    with _on(stream, layout.device, q, k, v, out):
        if grad:
            return _PackedAttention.apply(q, k, v, layout, bool(causal), scale)
        return _attention(q, k, v, layout, bool(causal), scale, None, out=out)


def prefix_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor,
                     layout: PackedLayout, causal: bool = True, scale: Optional[float] = None,
                     stream: Optional[torch.cuda.Stream] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """packed_attention where every query of every sequence also reads the keys of one shared prefix
    (an instruction or a context in front of every text): softmax over [prefix keys, own keys].

    prefix_k, prefix_v: [prefix, kv_heads, head_dim]. The prefix is read for tiles of rows of all
    sequences together where sequences are short, so its cost does not grow with their number. causal
    concerns the own keys alone. No gradient: inputs that require one are refused while gradients are
    enabled."""
    scale = _check_attention(q, k, v, layout, scale)
    _check_out(out, q)
    _heads(prefix_k, "prefix_k", q)
    _heads(prefix_v, "prefix_v", q)
    if prefix_k.shape != prefix_v.shape or prefix_k.shape[1] != k.shape[1]:
        raise ValueError("prefix_k and prefix_v must have the same shape and k's heads")
    _on_device(layout.device, prefix_k, prefix_v)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, prefix_k, prefix_v)):
        raise ValueError("prefix_attention has no gradient")
    with _on(stream, layout.device, q, k, v, prefix_k, prefix_v, out):
        return _attention(q, k, v, layout, bool(causal), scale, None, prefix_k, prefix_v, out)


# ---- q/k norm with rotation ------------------------------------------------------------------


def rotary_table(n_positions: int, dim: int, base: float = 10000.0,
                 device: Optional[Union[str, torch.device]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin, float32 [n_positions, dim // 2], of the angles position * base ** (-2 i / dim); the
    angles are computed in 64 bits (in 32 a far position's angle is off by position * 2^-24)."""
    if n_positions < 0 or dim < 2 or dim % 2:
        raise ValueError("n_positions must be >= 0 and dim even")
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    angle = torch.arange(n_positions, dtype=torch.float64)[:, None] * float(base) ** (-i / dim)
    return angle.cos().float().to(device), angle.sin().float().to(device)


def _rope_args(q, k, cos, sin, positions, eps, interleaved, wq, wk) -> nat.RopeArgs:
    a = nat.RopeArgs()
    a.dtype, a.heads, a.kv_heads, a.head_dim = _CODES[q.dtype], q.shape[1], k.shape[1], q.shape[2]
    a.rot, a.interleaved = 2 * cos.shape[1], int(interleaved)
    a.tokens, a.n_pos, a.eps = q.shape[0], cos.shape[0], eps
    _tensor3(a.q, q)
    _tensor3(a.k, k)
    a.wq, a.wk = nat.ptr(wq), nat.ptr(wk)
    a.cos, a.sin, a.positions = cos.data_ptr(), sin.data_ptr(), positions.data_ptr()
    return a


def _rope_forward(q, k, wq, wk, cos, sin, positions, eps, interleaved):
    yq, yk = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
    a = _rope_args(q, k, cos, sin, positions, eps, interleaved, wq, wk)
    _tensor3(a.yq, yq)
    _tensor3(a.yk, yk)
    nat.check(nat.lib().ahr_qk_norm_rope(ctypes.byref(a), nat.stream_ptr(device_index=q.device.index)), "ahr_qk_norm_rope")
    return yq, yk


def _unit(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, cos, sin, positions, eps, interleaved):
        w = [None if x is None else x.detach().float().contiguous() for x in (wq, wk)]
        ctx.save_for_backward(q, k, w[0], w[1], cos, sin, positions)
        ctx.eps, ctx.interleaved = eps, interleaved
        ctx.w_dtype = None if wq is None else (wq.dtype, wk.dtype)
        return _rope_forward(q, k, w[0], w[1], cos, sin, positions, eps, interleaved)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dyq, dyk):
        q, k, wq, wk, cos, sin, positions = ctx.saved_tensors
        with torch.cuda.device(q.device):
            dyq, dyk = _unit(dyq), _unit(dyk)
            dq, dk = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
            a = _rope_args(q, k, cos, sin, positions, ctx.eps, ctx.interleaved, wq, wk)
            for to, t in ((a.yq, dyq), (a.yk, dyk), (a.dq, dq), (a.dk, dk)):
                _tensor3(to, t)
            dw = None
            if wq is not None:
                n = ctypes.c_int64()
                nat.check(nat.lib().ahr_rope_ws_bytes(q.shape[0], q.shape[2], ctypes.byref(n)), "ahr_rope_ws_bytes")
                ws = torch.empty(n.value, dtype=torch.uint8, device=q.device)
                dw = torch.empty((2, q.shape[2]), dtype=torch.float32, device=q.device)
                a.dwq, a.dwk, a.ws, a.ws_bytes = dw[0].data_ptr(), dw[1].data_ptr(), ws.data_ptr(), n.value
            nat.check(nat.lib().ahr_qk_norm_rope_backward(ctypes.byref(a), nat.stream_ptr(device_index=q.device.index)),
                      "ahr_qk_norm_rope_backward")
        gq, gk = (None, None) if dw is None else (dw[0].to(ctx.w_dtype[0]), dw[1].to(ctx.w_dtype[1]))
        return dq, dk, gq, gk, None, None, None, None, None


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                 cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, eps: float = 1e-6,
                 interleaved: bool = False, stream: Optional[torch.cuda.Stream] = None
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Each head of q and k: x * weight / sqrt(mean(x^2) + eps), then rotated by its token's position.

    q [tokens, heads, head_dim], k [tokens, kv_heads, head_dim] in float32, float16 or bfloat16, any
    strides; weights [head_dim], or both None for the rotation alone; cos, sin float32 [n, rot / 2] with
    rot <= head_dim even (elements from rot on are only normed); positions int32 or int64 [tokens], one
    outside [0, n) gives NaN rows. Pairs: element i with i + rot / 2, or with interleaved 2 i with
    2 i + 1. head_dim even, at most 512. Computed in fp32, rounded once. Differentiable in q, k and the
    weights (whose gradients are summed in a fixed order)."""
    _heads(q, "q")
    _heads(k, "k", q, q.shape[0])
    if q.dtype not in _CODES:
        raise ValueError(f"qk_norm_rope takes float32, float16 and bfloat16, got {q.dtype}")
    dim = q.shape[2]
    if dim < 2 or dim % 2 or dim > 512:
        raise ValueError(f"head_dim must be even, at most 512, got {dim}")
    if q.shape[1] < 1 or k.shape[1] < 1:
        raise ValueError("q and k need a head each")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("one norm weight without the other")
    for w in (q_weight, k_weight):
        if w is not None and (w.shape != (dim,) or not w.is_floating_point()):
            raise ValueError("a norm weight must be a floating [head_dim] tensor")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be float32 tensors of the same [positions, rot / 2]")
    if cos.shape[1] < 1 or 2 * cos.shape[1] > dim or (cos.shape[0] < 1 and q.shape[0] > 0):
        raise ValueError("the table must have a row, and at most head_dim / 2 columns")
    if positions.shape != (q.shape[0],) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64 [tokens]")
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError("eps must be finite and not negative")
    if q.device.type != "cuda":
        raise nat.NativeLibraryError("qk_norm_rope needs tensors on a ROCm GPU")
    _on_device(q.device, k, q_weight, k_weight, cos, sin, positions)
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight))
    with _on(stream, q.device, q, k, q_weight, k_weight, cos, sin, positions):
        if positions.dtype == torch.int64:  # (a position beyond 32 bits must not wrap into the table)
            positions = positions.clamp(-1, 2 ** 31 - 1).to(torch.int32)
        cos, sin, positions = cos.contiguous(), sin.contiguous(), positions.contiguous()
        q, k = _unit(q), _unit(k)
        if grad:
            return _QkNormRope.apply(q, k, q_weight, k_weight, cos, sin, positions, float(eps), bool(interleaved))
        w = [None if x is None else x.detach().float().contiguous() for x in (q_weight, k_weight)]
        return _rope_forward(q, k, w[0], w[1], cos, sin, positions, float(eps), bool(interleaved))


# ---- mean pooling ----------------------------------------------------------------------------


def _pool_forward(rows, layout, normalize, norm):
    n_chunks, lists = layout._pool_lists()
    n, width = len(layout), rows.shape[1]
    out = torch.empty((n, width), dtype=torch.float32, device=rows.device)
    ws = torch.empty(max(1, n_chunks * width), dtype=torch.float32, device=rows.device)
    nat.check(nat.lib().ahr_pool_mean(_CODES[rows.dtype], rows.data_ptr(), rows.stride(0), width, lists.data_ptr(), n_chunks, n,
                                      int(normalize), out.data_ptr(), nat.ptr(norm), ws.data_ptr(), ws.numel() * 4,
                                      nat.stream_ptr(device_index=rows.device.index)), "ahr_pool_mean")
    _keep(lists, rows.device)
    return out


class _PackedMeanPool(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, layout, normalize):
        norm = torch.empty(len(layout), dtype=torch.float32, device=rows.device)
        out = _pool_forward(rows, layout, normalize, norm)
        ctx.save_for_backward(out, norm)
        ctx.layout, ctx.normalize, ctx.shape, ctx.dtype = layout, normalize, rows.shape, rows.dtype
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        out, norm = ctx.saved_tensors
        with torch.cuda.device(out.device):
            n_chunks, lists = ctx.layout._pool_lists()
            d_out = d_out.contiguous()
            d_rows = torch.empty(ctx.shape, dtype=ctx.dtype, device=out.device)
            nat.check(nat.lib().ahr_pool_mean_backward(_CODES[ctx.dtype], d_rows.data_ptr(), ctx.shape[1], lists.data_ptr(),
                                                       n_chunks, len(ctx.layout), int(ctx.normalize), d_out.data_ptr(),
                                                       out.data_ptr(), norm.data_ptr(),
                                                       nat.stream_ptr(device_index=out.device.index)),
                      "ahr_pool_mean_backward")
            _keep(lists, out.device)
        return d_rows, None, None


def packed_mean_pool(rows: torch.Tensor, layout: PackedLayout, normalize: bool = False,
                     stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """float32 [sequences, width]: the mean of each sequence's rows, summed in fp32; with normalize divided
    by max(its L2 norm, 1e-12). rows [tokens, width] in float32, float16 or bfloat16, any row stride. A
    sequence without rows gives zeros. Differentiable in rows."""
    if not isinstance(rows, torch.Tensor) or rows.dim() != 2 or rows.shape[1] < 1 or rows.shape[1] > 1 << 20:
        raise ValueError("rows must be a [tokens, width] tensor")
    if rows.dtype not in _CODES:
        raise ValueError(f"packed_mean_pool takes float32, float16 and bfloat16, got {rows.dtype}")
    if rows.shape[0] != layout.tokens:
        raise ValueError(f"rows has {rows.shape[0]} tokens, the layout {layout.tokens}")
    _on_device(layout.device, rows)
    with _on(stream, layout.device, rows):
        if rows.stride(1) != 1 and rows.shape[1] > 1:
            rows = rows.contiguous()
        if torch.is_grad_enabled() and rows.requires_grad:
            return _PackedMeanPool.apply(rows, layout, bool(normalize))
        return _pool_forward(rows, layout, bool(normalize), None)
