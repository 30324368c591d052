"""ah_rag.packed_encoder — a transformer's forward over packed sequences (no padding), on ah_rag.packed.

PackedTransformer takes the weights of a loaded model (any module with the state dict and config of one of
two layer layouts) and runs them over the tokens of a batch lying behind each other:

  "post":   absolute positions, bidirectional attention with as many key heads as query heads, layer norm
            after each residual (the architectures of ah_rag.encoder.ARCHS);
  "causal": rotary positions, causal attention with grouped heads and a norm of each query and key head,
            RMS norm before each block, gated feed-forward (decoder-style embedding checkpoints).

Projections, norms of whole rows and activations are torch / hipBLASLt calls; attention, the heads' norm
with the rotation, and pooling are this library's kernels. Other layouts are refused when the object is
made, never approximated. Dropout is not applied, in training either.

In a causal model the hidden states of a prefix do not depend on what follows, so tokens that all texts of
a batch begin with (an instruction in front of every query) are run once, and the rest of each text reads
their keys through prefix_attention.

Reference seam: SentenceTransformer.encode, src/ah_rag/graph/hierarchical_graph.py:655-656, :709-712.
"""
from __future__ import annotations

from typing import List, Mapping, Optional, Sequence, Tuple

import numpy as np
import torch
import torch.nn.functional as F

from .packed import PackedLayout, packed_attention, packed_mean_pool, prefix_attention, qk_norm_rope, rotary_table

# Bytes of all layers' projections up to which each layer's three are joined for a forward, by a copy of them. 6 layers
# of 384 (5 MB): one text / 256 texts 0.99 / 1.28 ms, with three products 1.16 / 1.40; 12 of 768 (42 MB) 1.84 / 3.66 and
# 2.24 / 3.56; 28 causal layers of 1024 (224 MB) 5.43 / 14.00 and 6.05 / 13.99: larger copies would cost more than launches.
JOIN_UP_TO = 256 << 20
SHARE_FROM = 16  # a common prefix of at least this many tokens is run once (a causal model, two texts or more)


class UnsupportedLayoutError(ValueError):
    """The model's layers are neither of the two layouts that the packed forward runs."""


def _get(cfg, *names, default=None):
    for n in names:
        v = getattr(cfg, n, None)
        if v is not None:
            return v
    return default


_POST = ("attention.self.query", "attention.self.key", "attention.self.value", "attention.output.dense", "attention.output.LayerNorm",
         "intermediate.dense", "output.dense", "output.LayerNorm")
_CAUSAL = ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")
# Model types whose forward is that of their layout (None: a module that names no type). Others share the parameters' names
# and settings, but start their positions elsewhere or compute attention in another way.
_TYPES = {"post": (None, "bert", "bert-generation", "electra", "ernie", "splinter"), "causal": (None, "qwen3", "qwen3_vl_text")}
_CAUSAL_NORMS = ("self_attn.q_norm", "self_attn.k_norm", "input_layernorm", "post_attention_layernorm")


class _Parameters(Mapping):
    """A model's parameters by name, each looked up in its module when it is read, so that one which another has taken the
    place of is not used on."""

    def __init__(self, model) -> None:
        self._at = {}
        for name, _ in model.named_parameters():
            path, _, leaf = name.rpartition(".")
            self._at[name] = (model.get_submodule(path)._parameters, leaf)

    def __getitem__(self, name: str) -> torch.Tensor:
        held, leaf = self._at[name]
        return held[leaf]

    def __iter__(self):
        return iter(self._at)

    def __len__(self) -> int:
        return len(self._at)


class PackedTransformer:
    """Weights are the model's own tensors (parameters receive gradients); `model` stays referenced, with the modules that
    it has now."""

    def __init__(self, model, device: torch.device) -> None:
        self.model, self.device = model, device
        cfg = model.config
        self.w = w = _Parameters(model)
        self.heads = int(cfg.num_attention_heads)
        self.layers = int(cfg.num_hidden_layers)
        self.hidden = int(cfg.hidden_size)
        if "encoder.layer.0.attention.self.query.weight" in w and "embeddings.position_embeddings.weight" in w:
            self.kind = "post"
            self.kv_heads, self.head_dim = self.heads, self.hidden // self.heads
            self.eps = float(cfg.layer_norm_eps)
            known = ["embeddings.%s_embeddings.weight" % n for n in ("word", "position", "token_type")]
            known += ["embeddings.LayerNorm.weight", "embeddings.LayerNorm.bias"]
            known += ["encoder.layer.%d.%s.%s" % (i, n, t) for i in range(self.layers) for n in _POST for t in ("weight", "bias")]
            self._names(known, optional=("embeddings.token_type_embeddings.weight",), unused="pooler.")
            if _get(cfg, "is_decoder", default=False):
                raise UnsupportedLayoutError("packed forward: a decoder's masks")
            if _get(cfg, "position_embedding_type", default="absolute") != "absolute":
                raise UnsupportedLayoutError("packed forward: positions other than absolute ones")
            table = getattr(getattr(model, "embeddings", None), "position_embeddings", None)
            if getattr(table, "padding_idx", None) is not None:  # (the first token's row is the one after it)
                raise UnsupportedLayoutError("packed forward: this model's positions are not those of its tokens")
            self.act = self._activation(cfg.hidden_act)
            self.fused = [("encoder.layer.%d.attention.self." % i, ("query", "key", "value")) for i in range(self.layers)]
        elif "layers.0.self_attn.q_norm.weight" in w and "layers.0.mlp.gate_proj.weight" in w:
            self.kind = "causal"
            self.kv_heads = int(_get(cfg, "num_key_value_heads", default=self.heads))
            self.head_dim = int(_get(cfg, "head_dim", default=self.hidden // self.heads))
            self.eps = float(cfg.rms_norm_eps)
            known = ["embed_tokens.weight", "norm.weight"]
            known += ["layers.%d.%s.weight" % (i, n) for i in range(self.layers) for n in _CAUSAL + _CAUSAL_NORMS]
            biases = ["layers.%d.%s.bias" % (i, n) for i in range(self.layers) for n in _CAUSAL]
            self._names(known + biases, optional=biases)
            # (settings that change the forward without a parameter of their own)
            if any(_get(cfg, n, default=1.0) != 1.0 for n in ("embedding_multiplier", "residual_multiplier", "attention_multiplier")):
                raise UnsupportedLayoutError("packed forward: scaled embeddings, residuals or scores")
            if (_get(cfg, "attn_logit_softcapping") is not None or _get(cfg, "is_causal", default=True) is False
                    or _get(cfg, "use_bidirectional_attention", default=False)
                    or any(t != "full_attention" for t in _get(cfg, "layer_types", default=()))):
                raise UnsupportedLayoutError("packed forward: attention other than causal softmax over all earlier tokens")
            if w["layers.0.self_attn.q_norm.weight"].shape != (self.head_dim,):
                raise UnsupportedLayoutError("packed forward: the query norm is not one of single heads")
            if _get(cfg, "use_sliding_window", default=False) and _get(cfg, "sliding_window") is not None:
                raise UnsupportedLayoutError("packed forward: sliding windows")
            rope = dict(_get(cfg, "rope_parameters", "rope_scaling", default={}) or {})
            if any(isinstance(v, dict) for v in rope.values()):
                raise UnsupportedLayoutError("packed forward: rotary positions that differ from layer to layer")
            if (rope.get("rope_type", rope.get("type", "default")) != "default"
                    or float(rope.get("partial_rotary_factor", _get(cfg, "partial_rotary_factor", default=1.0))) != 1.0):
                raise UnsupportedLayoutError("packed forward: scaled or partial rotary positions")
            self.theta = float(rope.get("rope_theta", _get(cfg, "rope_theta", default=10000.0)))
            self.act = self._activation(cfg.hidden_act)
            self.fused = [("layers.%d.self_attn." % i, ("q_proj", "k_proj", "v_proj")) for i in range(self.layers)]
            self._table: Optional[Tuple[torch.Tensor, torch.Tensor, Optional[torch.cuda.Stream]]] = None  # cos, sin, made on
        else:
            raise UnsupportedLayoutError("packed forward: unknown layer layout")
        if _get(cfg, "model_type") not in _TYPES[self.kind]:
            raise UnsupportedLayoutError(f"packed forward: a model of type {cfg.model_type!r}")
        p = next(iter(w.values()))
        if p.dtype not in (torch.float16, torch.bfloat16):
            raise UnsupportedLayoutError(f"packed forward: weights in float16 or bfloat16, got {p.dtype}")
        if self.head_dim % 8 or self.head_dim > 128 or self.heads % self.kv_heads:
            raise UnsupportedLayoutError(f"packed forward: {self.heads}/{self.kv_heads} heads of {self.head_dim}")

    def _names(self, known: Sequence[str], optional: Sequence[str] = (), unused: Optional[str] = None) -> None:
        """Every parameter of the model takes part in the forward here, and none is missing."""
        more = sorted(n for n in self.w if n not in set(known) and not (unused and n.startswith(unused)))
        less = sorted(set(known) - set(optional) - set(self.w))
        if more or less:
            raise UnsupportedLayoutError(f"packed forward: {'unknown' if more else 'no'} parameter {(more or less)[0]!r}")

    @staticmethod
    def _activation(name: str):
        acts = {"gelu": F.gelu, "silu": F.silu, "swish": F.silu, "relu": F.relu,
                "gelu_new": lambda x: F.gelu(x, approximate="tanh"), "gelu_pytorch_tanh": lambda x: F.gelu(x, approximate="tanh")}
        if name not in acts:
            raise UnsupportedLayoutError(f"packed forward: activation {name!r}")
        return acts[name]

    # ---- layers --------------------------------------------------------------------------------

    def _joined(self) -> Optional[List[Tuple[torch.Tensor, Optional[torch.Tensor]]]]:
        """Each layer's three projections as one weight and bias, for one forward: copied from the weights as they stand
        (two launches), so that every write to them counts and nothing is shared between streams. None where three
        products are taken instead: a gradient of the projections is wanted, or the copy costs more than it saves."""
        names = [prefix + n for prefix, all_ in self.fused for n in all_]
        ws = [self.w[n + ".weight"] for n in names]
        bs = [self.w.get(n + ".bias") for n in names]
        some = [b for b in bs if b is not None]
        if not self.layers or len(some) not in (0, len(bs)) or sum(w.numel() for w in ws) * ws[0].element_size() > JOIN_UP_TO:
            return None
        if torch.is_grad_enabled() and any(t.requires_grad for t in (*ws, *some)):
            return None
        rows = [sum(w.shape[0] for w in ws[i:i + 3]) for i in range(0, len(ws), 3)]
        w = torch.cat(ws).split(rows)
        return list(zip(w, torch.cat(some).split(rows) if some else [None] * len(rows)))

    def _qkv(self, i: int, x: torch.Tensor, joined: Optional[List[Tuple[torch.Tensor, Optional[torch.Tensor]]]] = None
             ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Queries, keys and values [tokens, heads, head_dim]: views of one product's output, or three products."""
        h, hk, d = self.heads, self.kv_heads, self.head_dim
        if joined is not None:
            y = F.linear(x, *joined[i]).view(x.shape[0], h + 2 * hk, d)
            return y[:, :h], y[:, h:h + hk], y[:, h + hk:]
        prefix, names = self.fused[i]
        return tuple(self._lin(prefix + n, x).view(x.shape[0], m, d) for n, m in zip(names, (h, hk, hk)))

    def refresh(self) -> None:
        """Nothing to do, for programs that call it after writing to the weights: nothing made from them is kept."""

    def _lin(self, name: str, x: torch.Tensor) -> torch.Tensor:
        return F.linear(x, self.w[name + ".weight"], self.w.get(name + ".bias"))

    def _ln(self, name: str, x: torch.Tensor) -> torch.Tensor:
        return F.layer_norm(x, (self.hidden,), self.w[name + ".weight"], self.w[name + ".bias"], self.eps)

    def _rms(self, name: str, x: torch.Tensor) -> torch.Tensor:
        return F.rms_norm(x, (self.hidden,), self.w[name + ".weight"], self.eps)

    def _post(self, ids: torch.Tensor, layout: PackedLayout) -> torch.Tensor:
        e = "embeddings."
        x = F.embedding(ids, self.w[e + "word_embeddings.weight"]) + F.embedding(layout.positions(), self.w[e + "position_embeddings.weight"])
        if e + "token_type_embeddings.weight" in self.w:
            x = x + self.w[e + "token_type_embeddings.weight"][0]
        x = self._ln(e + "LayerNorm", x)
        joined = self._joined()
        for i in range(self.layers):
            b = "encoder.layer.%d." % i
            q, k, v = self._qkv(i, x, joined)
            o = packed_attention(q, k, v, layout).flatten(1)
            x = self._ln(b + "attention.output.LayerNorm", x + self._lin(b + "attention.output.dense", o))
            y = self._lin(b + "output.dense", self.act(self._lin(b + "intermediate.dense", x)))
            x = self._ln(b + "output.LayerNorm", x + y)
        return x

    def _rotary(self, n: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """A table of n positions at least. It is complete when rotary_table returns (a blocking copy), and a stream that did
        not make it is noted as its reader, since a longer one may take its place while that stream still reads it."""
        held = self._table
        if held is None or held[0].shape[0] < n:
            table = rotary_table(max(512, n), self.head_dim, self.theta, self.device)
            self._table = held = (*table, self._stream())
        cos, sin, made_on = held
        stream = self._stream()
        if stream != made_on:
            cos.record_stream(stream)
            sin.record_stream(stream)
        return cos, sin

    def _stream(self) -> Optional[torch.cuda.Stream]:
        return torch.cuda.current_stream(self.device) if self.device.type == "cuda" else None

    def _causal(self, ids: torch.Tensor, layout: PackedLayout, first: int = 0, shared: Optional[List[tuple]] = None,
                keep: Optional[List[tuple]] = None) -> torch.Tensor:
        """shared: (keys, values) of a common prefix of `first` tokens, one pair a layer; keep: appended to, for such."""
        cos, sin = self._rotary(first + (int(layout.lengths.max()) if len(layout) else 0))
        pos = layout.positions() + first if first else layout.positions()
        x = F.embedding(ids, self.w["embed_tokens.weight"])
        joined = self._joined()
        for i in range(self.layers):
            b = "layers.%d." % i
            q, k, v = self._qkv(i, self._rms(b + "input_layernorm", x), joined)
            q, k = qk_norm_rope(q, k, self.w[b + "self_attn.q_norm.weight"], self.w[b + "self_attn.k_norm.weight"], cos, sin, pos, eps=self.eps)
            if keep is not None:
                keep.append((k, v))
            o = packed_attention(q, k, v, layout, causal=True) if shared is None else prefix_attention(q, k, v, *shared[i], layout)
            x = x + self._lin(b + "self_attn.o_proj", o.flatten(1))
            y = self._rms(b + "post_attention_layernorm", x)
            x = x + self._lin(b + "mlp.down_proj", self.act(self._lin(b + "mlp.gate_proj", y)) * self._lin(b + "mlp.up_proj", y))
        return self._rms("norm", x)

    # ---- batches -------------------------------------------------------------------------------

    def _flat(self, ids: Sequence[Sequence[int]]) -> Tuple[np.ndarray, np.ndarray]:
        """Token ids behind each other, and the lengths; indexes past a table, which on the device would be a fault, are
        refused here."""
        lens = np.fromiter((len(s) for s in ids), np.int64, len(ids))
        flat = np.fromiter((t for s in ids for t in s), np.int64, int(lens.sum()))
        table = self.w["embeddings.word_embeddings.weight" if self.kind == "post" else "embed_tokens.weight"]
        if flat.size and (flat.min() < 0 or flat.max() >= table.shape[0]):
            raise ValueError(f"token ids must lie in [0, {table.shape[0]})")
        if self.kind == "post" and lens.size:
            most = self.w["embeddings.position_embeddings.weight"].shape[0]
            if lens.max() > most:
                raise ValueError(f"a sequence is longer than the model's {most} positions")
        return flat, lens

    def _tokens(self, flat: np.ndarray, lens: np.ndarray) -> Tuple[torch.Tensor, PackedLayout]:
        return torch.from_numpy(flat).to(self.device), PackedLayout(lens, device=self.device)

    def hidden_states(self, ids: Sequence[Sequence[int]]) -> Tuple[torch.Tensor, PackedLayout]:
        """Last hidden states [tokens, hidden] of token id sequences, and their layout."""
        tok, layout = self._tokens(*self._flat(ids))
        return (self._post if self.kind == "post" else self._causal)(tok, layout), layout

    def pooled(self, ids: Sequence[Sequence[int]], normalize: bool) -> torch.Tensor:
        """float32 [n, hidden]: the mean of each sequence's last hidden states."""
        share = 0 if self.kind == "post" or torch.is_grad_enabled() else common_prefix(ids)
        if share < SHARE_FROM:
            h, layout = self.hidden_states(ids)
            return packed_mean_pool(h, layout, normalize=normalize)
        first, rest = self._flat([ids[0][:share]]), self._flat([s[share:] for s in ids])
        kept: List[tuple] = []
        tok, layout = self._tokens(*first)
        head = self._causal(tok, layout, keep=kept).float().sum(0)
        tok, layout = self._tokens(*rest)
        mean = packed_mean_pool(self._causal(tok, layout, share, kept), layout)
        n = torch.tensor([len(s) for s in ids], dtype=torch.float32, device=self.device)[:, None]
        y = (mean * (n - share) + head) / n
        return F.normalize(y, dim=1) if normalize else y


def common_prefix(ids: Sequence[Sequence[int]]) -> int:
    """Tokens that all sequences begin with; each keeps one of its own. 0 for fewer than two sequences."""
    if len(ids) < 2:
        return 0
    a, b = min(ids), max(ids)  # in order, what the first and the last share, all share
    n = 0
    for x, y in zip(a, b):
        if x != y:
            break
        n += 1
    return max(0, min(n, min(len(s) for s in ids) - 1))
