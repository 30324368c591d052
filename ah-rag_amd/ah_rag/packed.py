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
then; a captured backward pass also needs leaves without a living graph from outside the capture, whose
gradients torch accumulates on the stream of that graph). Tensors that the kernels cannot read in place
(rows that do not start at multiples of 16 bytes, a strided last dimension) are copied first.

Replaces, behind the reference's SentenceTransformer.encode seam
(src/ah_rag/graph/hierarchical_graph.py:655-656, :709-712), that library's padded attention and
pooling.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import struct
from types import SimpleNamespace
from typing import Dict, Optional, Sequence, Tuple, Union

import numpy as np
import torch
from torch.autograd import forward_ad

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
    # (each, then the sum: that of large values would wrap)
    if a.size and (int(a.min()) < 0 or int(a.max()) > 1 << 30 or int(a.sum(dtype=np.int64)) > 1 << 30):
        raise ValueError(f"{what} must be >= 0 and sum to at most 2**30")
    own = np.array(a, dtype=np.int32)  # (a copy, and read-only: the work lists are made from it once)
    own.setflags(write=False)
    return own


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
        self._index = self.device.index
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
            # a blocking copy: the lists are complete for every stream (and no inference tensor, whatever mode the
            # first call runs in: later ones may save it for their backward pass)
            with torch.inference_mode(False):
                t = torch.from_numpy(host).to(self.device)
            t.ahr_stream = nat.stream_ptr(device_index=self._index)
            return t

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
            buf = np.zeros(max(1, n.value + len(self.lengths)) * 4, np.int32)
            nat.check(nat.lib().ahr_pool_plan_build(*args, buf.ctypes.data, buf.size, ctypes.byref(n)), "ahr_pool_plan_build")
            self._pool = (n.value, self._upload(buf))
        return self._pool


# ---- shared checks ---------------------------------------------------------------------------


def _heads(t: torch.Tensor, what: str) -> None:
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"{what} must be a [tokens, heads, head_dim] tensor")


def _like(t: torch.Tensor, what: str, q: torch.Tensor) -> None:
    _heads(t, what)
    if t.dtype != q.dtype or t.device != q.device or t.shape[2] != q.shape[2]:
        raise ValueError(f"{what} must have q's dtype, device and head_dim")


def _on_device(device: torch.device, *tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"tensors must be on {device}, got one on {t.device}")


def _no_tangent(*tensors: Optional[torch.Tensor]) -> None:
    """Forward-mode derivatives are refused: past autograd's function, a tangent would be dropped and read as zero."""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("the packed operators have no forward-mode derivative")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy whose rows start at multiples of 16 bytes and are contiguous (16-bit types)."""
    n, h, d = t.shape
    ts, hs, es = t.stride()
    if ((es == 1 or d == 1) and t.data_ptr() % 16 == 0 and (n < 2 or (ts % 8 == 0 and ts < 1 << 22))
            and (h < 2 or (hs % 8 == 0 and hs * h <= 1 << 29))):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _new(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor of t's kind (half the host time of torch.empty with its arguments)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _rows(t: Optional[torch.Tensor]) -> Tuple[int, int, int]:
    """A struct ahr_tensor3: address and strides of tokens and heads (of an axis of one element arbitrary)."""
    if t is None:
        return 0, 0, 0
    n, h, _ = t.shape
    ts, hs, _ = t.stride()
    return t.data_ptr(), ts if n > 1 else 0, hs if h > 1 else 0


def _calls() -> SimpleNamespace:
    """The entry points that take an argument struct, as (bytes, stream) -> status."""
    global _CALLS
    if _CALLS is None:
        lib = nat.lib()
        kind = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_char_p, ctypes.c_void_p)
        _CALLS = SimpleNamespace(**{n: kind((f, lib)) for n, f in (
            ("attn_forward", "ahr_attn_forward"), ("attn_backward", "ahr_attn_backward"), ("rope", "ahr_qk_norm_rope"),
            ("rope_backward", "ahr_qk_norm_rope_backward"))})
    return _CALLS


_CALLS: Optional[SimpleNamespace] = None

# The argument structs of include/ahr.h, packed in one step (field by field through ctypes costs more than
# a small kernel).
_ATTN_ARGS = struct.Struct("@PPfi 3q3q3q 3q3q 3q P 3q3q3q3q Pq".replace(" ", ""))
_ROPE_ARGS = struct.Struct("@iiiiii qqfi 3q3q 3q3q 3q3q PPPPP PP Pq".replace(" ", ""))
assert _ATTN_ARGS.size == ctypes.sizeof(nat.AttnArgs) and _ROPE_ARGS.size == ctypes.sizeof(nat.RopeArgs)


@contextlib.contextmanager
def _side(stream: torch.cuda.Stream, device: torch.device, *tensors: Optional[torch.Tensor]):
    """Run on `stream`, after the current stream's work."""
    with torch.cuda.device(device):
        stream.wait_stream(torch.cuda.current_stream(device))
        for t in tensors:
            if t is not None:
                t.record_stream(stream)
        with torch.cuda.stream(stream):
            yield


def _elsewhere(stream: Optional[torch.cuda.Stream], device: torch.device) -> bool:
    """Whether the call has to leave the current device or stream."""
    return stream is not None or torch.cuda.current_device() != device.index


def _on(stream: Optional[torch.cuda.Stream], device: torch.device, *tensors: Optional[torch.Tensor]):
    if stream is None:
        return torch.cuda.device(device)
    if stream.device != device:
        raise ValueError(f"a stream of {stream.device} for tensors on {device}")
    return _side(stream, device, *tensors)


def _keep(lists: Optional[torch.Tensor], stream: int, device: torch.device) -> None:
    """The layout may be dropped while another stream than the one that made its lists still reads them, or
    while a graph that captured the call can still be replayed (such lists, a few KB, are never freed)."""
    if lists is None:
        return
    if torch.cuda.is_current_stream_capturing():
        _CAPTURED[id(lists)] = lists
    elif lists.ahr_stream != stream:
        lists.record_stream(torch.cuda.current_stream(device))


_CAPTURED: Dict[int, torch.Tensor] = {}


# ---- attention -------------------------------------------------------------------------------


def _once() -> None:
    """The gradients are not differentiable again. (torch's once_differentiable says the same at the cost of a
    small kernel.)"""
    if torch.is_grad_enabled():
        raise RuntimeError("the packed operators have no second derivative (backward with create_graph=True)")


def _launch_attention(call, name, plan, lists, scale, q, k, v, pk, pv, o, lse, d_o, dq, dk, dv) -> None:
    ws = q.new_empty(plan.ws_bytes, dtype=torch.uint8) if plan.ws_bytes else None
    stream = nat.stream_ptr(device_index=q.device.index)
    args = _ATTN_ARGS.pack(ctypes.addressof(plan), 0 if lists is None else lists.data_ptr(), scale, 0, *_rows(q), *_rows(k), *_rows(v),
                           *_rows(pk), *_rows(pv), *_rows(o), 0 if lse is None else lse.data_ptr(), *_rows(d_o), *_rows(dq), *_rows(dk),
                           *_rows(dv), 0 if ws is None else ws.data_ptr(), plan.ws_bytes)
    if call(args, stream):
        nat.check(-1, name)
    _keep(lists, stream, q.device)


def _attention(q, k, v, layout, causal, scale, lse, prefix_k=None, prefix_v=None, out=None) -> torch.Tensor:
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    shape = q.shape
    if prefix_k is not None:
        prefix_k, prefix_v = _aligned(prefix_k), _aligned(prefix_v)
    plan, lists = layout._plan(_CODES[q.dtype], shape[1], k.shape[1], shape[2], causal, False, 0 if prefix_k is None else prefix_k.shape[0])
    o = _new(q) if out is None else out
    _launch_attention(_calls().attn_forward, "ahr_attn_forward", plan, lists, scale, q, k, v, prefix_k, prefix_v, o, lse, None, None, None, None)
    if out is not None and not out.is_inference():
        torch.autograd.graph.increment_version(out)  # (a graph that saved out has to notice the write)
    return o


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, layout, causal, scale):
        q, k, v = _aligned(q), _aligned(k), _aligned(v)
        lse = q.new_empty(q.shape[:2], dtype=torch.float32)
        o = _attention(q, k, v, layout, causal, scale, lse)
        # the backward pass's lists too: its first call may be inside a capture
        ctx.plan = layout._plan(_CODES[q.dtype], q.shape[1], k.shape[1], q.shape[2], causal, True, 0)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.scale = scale
        return o

    @staticmethod
    def backward(ctx, d_o):  # (on the device and stream of the forward call)
        _once()
        q, k, v, o, lse = ctx.saved_tensors
        plan, lists = ctx.plan
        dq, dk, dv = _new(q), _new(k), _new(k)
        _launch_attention(_calls().attn_backward, "ahr_attn_backward", plan, lists, ctx.scale, q, k, v, None, None, o, lse,
                          _aligned(d_o), dq, dk, dv)
        return dq, dk, dv, None, None, None


def _check_attention(q, k, v, layout, scale) -> float:
    _heads(q, "q")
    _like(k, "k", q)
    _like(v, "v", q)
    tokens, heads, dim = q.shape
    keys, kv_heads, _ = k.shape
    if tokens != layout.tokens or keys != layout.key_tokens:
        raise ValueError(f"q has {tokens} and k {keys} tokens, the layout {layout.tokens} and {layout.key_tokens}")
    if v.shape != k.shape:
        raise ValueError("v must have k's shape")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"attention takes float16 and bfloat16, got {q.dtype}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads or heads // kv_heads > 128:
        raise ValueError(f"{heads} query heads do not share {kv_heads} key heads (a multiple, at most 128 each)")
    if dim < 8 or dim % 8 or dim > 128:
        raise ValueError(f"head_dim must be a multiple of 8, at most 128, got {dim}")
    if q.device != layout.device:
        raise ValueError(f"tensors must be on {layout.device}, got one on {q.device}")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0 < scale < 3e38:
        raise ValueError("scale must be positive and finite")
    return scale


def _check_out(out: Optional[torch.Tensor], q: torch.Tensor) -> None:
    if out is None:
        return
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError("out must have q's shape, dtype and device")
    if torch.is_grad_enabled() and out.requires_grad:
        raise ValueError("out must not require a gradient")
    if any(n > 1 and st == 0 for n, st in zip(out.shape, out.stride())):
        raise ValueError("out must not be expanded")
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
    zeros, and zero gradients; one whose scores are all minus infinity NaN. Scores, sums and accumulators are
    fp32; the weights p are rounded to the tensors' type for the product with v, and o once at the end. The
    gradients use a row's log-sum in fp32, whose rounding shows in them where scaled scores pass 2^14.

    Differentiable in q, k and v (no atomics: repeated runs give the same bits). `out`, where no gradient
    is wanted: written in place of a new tensor; it must not overlap the inputs. `stream`: runs there,
    after the current stream's work; the caller orders what follows. A key or value that a row's mask
    hides never reaches that row's output, whatever it holds; in the gradients a value that is not finite may
    reach any row of its own sequence, and none of another."""
    _no_tangent(q, k, v)
    scale = _check_attention(q, k, v, layout, scale)
    _check_out(out, q)
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if grad and out is not None:
        raise ValueError("out cannot be given where a gradient is wanted")
    if _elsewhere(stream, layout.device):
        with _on(stream, layout.device, q, k, v, out):
            return packed_attention(q, k, v, layout, causal, scale, None, out)
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
    _no_tangent(q, k, v, prefix_k, prefix_v)
    scale = _check_attention(q, k, v, layout, scale)
    _check_out(out, q)
    _like(prefix_k, "prefix_k", q)
    _like(prefix_v, "prefix_v", q)
    if prefix_k.shape != prefix_v.shape or prefix_k.shape[1] != k.shape[1]:
        raise ValueError("prefix_k and prefix_v must have the same shape and k's heads")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, prefix_k, prefix_v)):
        raise ValueError("prefix_attention has no gradient")
    if _elsewhere(stream, layout.device):
        with _on(stream, layout.device, q, k, v, prefix_k, prefix_v, out):
            return prefix_attention(q, k, v, prefix_k, prefix_v, layout, causal, scale, None, out)
    return _attention(q, k, v, layout, bool(causal), scale, None, prefix_k, prefix_v, out)


# ---- q/k norm with rotation ------------------------------------------------------------------


def rotary_table(n_positions: int, dim: int, base: float = 10000.0,
                 device: Optional[Union[str, torch.device]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin, float32 [n_positions, dim // 2], of the angles position * base ** (-2 i / dim); the
    angles are computed in 64 bits (in 32 a far position's angle is off by position * 2^-24)."""
    if n_positions < 0 or dim < 2 or dim % 2:
        raise ValueError("n_positions must be >= 0 and dim even")
    with torch.inference_mode(False):
        i = torch.arange(0, dim, 2, dtype=torch.float64)
        angle = torch.arange(n_positions, dtype=torch.float64)[:, None] * float(base) ** (-i / dim)
        return angle.cos().float().to(device), angle.sin().float().to(device)


def _launch_rope(call, name, q, k, cos, sin, positions, eps, interleaved, wq, wk, yq, yk, dq=None, dk=None, dwq=None, dwk=None, ws=None) -> None:
    tokens, heads, dim = q.shape
    n_pos, half = cos.shape
    args = _ROPE_ARGS.pack(_CODES[q.dtype], heads, k.shape[1], dim, 2 * half, interleaved, tokens, n_pos, eps, 0, *_rows(q), *_rows(k),
                           *_rows(yq), *_rows(yk), *_rows(dq), *_rows(dk), 0 if wq is None else wq.data_ptr(),
                           0 if wk is None else wk.data_ptr(), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(),
                           0 if dwq is None else dwq.data_ptr(), 0 if dwk is None else dwk.data_ptr(),
                           0 if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel())
    stream = nat.stream_ptr(device_index=q.device.index)
    if call(args, stream):
        nat.check(-1, name)
    if getattr(positions, "ahr_stream", None) is not None:  # a layout's own
        _keep(positions, stream, q.device)


@functools.lru_cache(maxsize=64)
def _rope_ws(dim: int) -> int:
    """Bytes of the backward pass's workspace (the same for any number of tokens)."""
    n = ctypes.c_int64()
    nat.check(nat.lib().ahr_rope_ws_bytes(0, dim, ctypes.byref(n)), "ahr_rope_ws_bytes")
    return n.value


def _rope_forward(q, k, wq, wk, cos, sin, positions, eps, interleaved):
    yq, yk = _new(q), _new(k)
    _launch_rope(_calls().rope, "ahr_qk_norm_rope", q, k, cos, sin, positions, eps, interleaved, wq, wk, yq, yk)
    return yq, yk


def _unit(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _weight(w: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if w is None or (w.dtype == torch.float32 and w.is_contiguous()):
        return w
    return w.detach().float().contiguous()


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
        wq, wk = _weight(q_weight), _weight(k_weight)
        ctx.save_for_backward(q, k, wq, wk, cos, sin, positions)
        ctx.eps, ctx.interleaved = eps, interleaved
        ctx.w_dtype = None if wq is None else (q_weight.dtype, k_weight.dtype)
        return _rope_forward(q, k, wq, wk, cos, sin, positions, eps, interleaved)

    @staticmethod
    def backward(ctx, dyq, dyk):
        _once()
        q, k, wq, wk, cos, sin, positions = ctx.saved_tensors
        dq, dk = _new(q), _new(k)
        ws = gq = gk = None
        if wq is not None:
            ws = q.new_empty(_rope_ws(q.shape[2]), dtype=torch.uint8)
            gq, gk = _new(wq), _new(wk)
        _launch_rope(_calls().rope_backward, "ahr_qk_norm_rope_backward", q, k, cos, sin, positions, ctx.eps, ctx.interleaved, wq, wk,
                     _unit(dyq), _unit(dyk), dq, dk, gq, gk, ws)
        if gq is not None:
            if ctx.w_dtype != (torch.float32, torch.float32):
                gq, gk = gq.to(ctx.w_dtype[0]), gk.to(ctx.w_dtype[1])
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
    _no_tangent(q, k, q_weight, k_weight, cos, sin)
    _heads(q, "q")
    _like(k, "k", q)
    if q.dtype not in _CODES:
        raise ValueError(f"qk_norm_rope takes float32, float16 and bfloat16, got {q.dtype}")
    tokens, heads, dim = q.shape
    if k.shape[0] != tokens:
        raise ValueError("q and k must have the same tokens")
    if dim < 2 or dim % 2 or dim > 512:
        raise ValueError(f"head_dim must be even, at most 512, got {dim}")
    if heads < 1 or k.shape[1] < 1:
        raise ValueError("q and k need a head each")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("one norm weight without the other")
    for w in (q_weight, k_weight):
        if w is not None and (w.shape != (dim,) or not w.is_floating_point()):
            raise ValueError("a norm weight must be a floating [head_dim] tensor")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be float32 tensors of the same [positions, rot / 2]")
    n_pos, half = cos.shape
    if half < 1 or 2 * half > dim or (n_pos < 1 and tokens > 0):
        raise ValueError("the table must have a row, and at most head_dim / 2 columns")
    if positions.shape != (tokens,) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64 [tokens]")
    if not 0 <= eps < 3e38:
        raise ValueError("eps must be finite and not negative")
    if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad):
        raise ValueError("the table has no gradient")
    device = q.device
    if device.type != "cuda":
        raise nat.NativeLibraryError("qk_norm_rope needs tensors on a ROCm GPU")
    _on_device(device, q_weight, k_weight, cos, sin, positions)
    if _elsewhere(stream, device):
        with _on(stream, device, q, k, q_weight, k_weight, cos, sin, positions):
            return qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    if positions.dtype == torch.int64:  # (a position beyond 32 bits must not wrap into the table)
        positions = positions.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    cos, sin, positions = cos.contiguous(), sin.contiguous(), positions.contiguous()
    q, k = _unit(q), _unit(k)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or (q_weight is not None and (q_weight.requires_grad or k_weight.requires_grad))):
        return _QkNormRope.apply(q, k, q_weight, k_weight, cos, sin, positions, float(eps), bool(interleaved))
    return _rope_forward(q, k, _weight(q_weight), _weight(k_weight), cos, sin, positions, float(eps), bool(interleaved))


# ---- mean pooling ----------------------------------------------------------------------------


def _pool_forward(rows, layout, normalize, norm):
    n_chunks, lists = layout._pool_lists()
    n, width = len(layout), rows.shape[1]
    out = rows.new_empty((n, width), dtype=torch.float32)
    ws = rows.new_empty(max(1, n_chunks * ((width + 3) // 4 * 4)), dtype=torch.float32)
    stream = nat.stream_ptr(device_index=rows.device.index)
    nat.check(nat.lib().ahr_pool_mean(_CODES[rows.dtype], rows.data_ptr(), rows.stride(0), width, lists.data_ptr(), n_chunks, n,
                                      int(normalize), out.data_ptr(), nat.ptr(norm), ws.data_ptr(), ws.numel() * 4, stream), "ahr_pool_mean")
    _keep(lists, stream, rows.device)
    return out


class _PackedMeanPool(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, layout, normalize):
        norm = rows.new_empty(len(layout), dtype=torch.float32)
        out = _pool_forward(rows, layout, normalize, norm)
        ctx.save_for_backward(out, norm)
        ctx.layout, ctx.normalize, ctx.shape, ctx.dtype = layout, normalize, rows.shape, rows.dtype
        return out

    @staticmethod
    def backward(ctx, d_out):
        _once()
        out, norm = ctx.saved_tensors
        layout = ctx.layout
        n_chunks, lists = layout._pool_lists()
        d_out = d_out.contiguous()
        d_rows = out.new_empty(ctx.shape, dtype=ctx.dtype)
        stream = nat.stream_ptr(device_index=out.device.index)
        nat.check(nat.lib().ahr_pool_mean_backward(_CODES[ctx.dtype], d_rows.data_ptr(), ctx.shape[1], lists.data_ptr(), n_chunks,
                                                   len(layout), ctx.normalize, d_out.data_ptr(), out.data_ptr(), norm.data_ptr(), stream),
                  "ahr_pool_mean_backward")
        _keep(lists, stream, out.device)
        return d_rows, None, None


def packed_mean_pool(rows: torch.Tensor, layout: PackedLayout, normalize: bool = False,
                     stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """float32 [sequences, width]: the mean of each sequence's rows, summed in fp32; with normalize divided
    by max(its L2 norm, 1e-12). rows [tokens, width] in float32, float16 or bfloat16, any row stride. A
    sequence without rows gives zeros. Differentiable in rows."""
    _no_tangent(rows)
    if not isinstance(rows, torch.Tensor) or rows.dim() != 2 or rows.shape[1] < 1 or rows.shape[1] > 1 << 20:
        raise ValueError("rows must be a [tokens, width] tensor")
    if rows.dtype not in _CODES:
        raise ValueError(f"packed_mean_pool takes float32, float16 and bfloat16, got {rows.dtype}")
    if rows.shape[0] != layout.tokens:
        raise ValueError(f"rows has {rows.shape[0]} tokens, the layout {layout.tokens}")
    _on_device(layout.device, rows)
    if _elsewhere(stream, layout.device):
        with _on(stream, layout.device, rows):
            return packed_mean_pool(rows, layout, normalize)
    if rows.stride(1) != 1 and rows.shape[1] > 1:
        rows = rows.contiguous()
    if torch.is_grad_enabled() and rows.requires_grad:
        return _PackedMeanPool.apply(rows, layout, bool(normalize))
    return _pool_forward(rows, layout, bool(normalize), None)
