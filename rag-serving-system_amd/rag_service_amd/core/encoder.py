"""The embedding model's forward pass on the HIP operators, in 8 bits.

``HipEncoder`` stands where the reference's embedding model stands (``embedding_model["model"]``, called at
``batch_processor.py:89-91``): built from an XLM-R model (the reference's ``intfloat/multilingual-e5-large-instruct`` is one,
``main.py:26-28``), moved with ``.to(device)``, called with the tokenizer's tensors, it returns ``last_hidden_state``
(batch, length, hidden) in fp32. The linear layers run in 8-bit integers (weights rounded once, a scale a channel;
activations as they come, a scale a row), everything between them in `dtype` with fp32 arithmetic: an approximation of the fp32
model, which is why it is asked for by name (``BatchProcessor(..., encoder="hip")``) and not the default.

Padding. The reference averages over all positions, pads included (``batch_processor.py:91``), so the pads' hidden states
count; but no key is a pad, and an XLM-R pad has one token id and one position id wherever it stands, so all pads of a
sequence have the same hidden state. The batch is therefore packed: each sequence keeps its real tokens and ONE pad row (if it
has any), len + 1 queries against len keys, and the result is spread to (batch, length, hidden) at the end.
"""
from __future__ import annotations

import sys
import warnings

import numpy as np

from .. import ops

MODEL_TYPES = ("xlm-roberta", "roberta")      # position ids count from the pad's own: every pad has the same


def _torch():
    return sys.modules["torch"]               # (the model handed over is torch's)


def look(ids, mask, types, pad, words, kinds):
    """The batch as the host has to know it, in one read: every sequence's number of tokens, as a list and on the device
    (int32). Refuses batches that are not padded on the right by the pad token, sequences without tokens, and ids and token
    types (None: all 0) that the embedding tables do not hold."""
    torch = _torch()
    real = mask.sum(1)
    right = ((torch.arange(ids.shape[1], device=ids.device) < real[:, None]) == mask).all() & ((ids != pad) == mask).all()
    seen = [real, torch.stack([right.long(), *(x.long() for x in torch.aminmax(ids))])]
    if types is not None:
        seen.append(torch.stack([*torch.aminmax(types), types.masked_fill(mask, 0).abs().amax()]).long())
    lengths = torch.cat(seen).tolist()
    if types is not None:
        *lengths, low, high, pads = lengths
        if low < 0 or high >= kinds or pads:
            raise ValueError(f"HipEncoder: token types {low} to {high} of {kinds}; those of pads are 0")
    *lengths, good, low, high = lengths
    if low < 0 or high >= words:
        raise ValueError(f"HipEncoder: token ids {low} to {high} of {words}")
    if not all(lengths):
        raise ValueError("HipEncoder: a sequence without tokens")
    if not good:
        raise ValueError("HipEncoder takes batches padded on the right with the pad token, and no pads elsewhere")
    return lengths, real.to(torch.int32)


class EncoderOutput:
    def __init__(self, last_hidden_state):
        self.last_hidden_state = last_hidden_state


def pack(lengths, length):
    """How a right-padded batch is packed: for sequences of `lengths` real tokens padded to `length`, (offsets, source,
    place, spread): the packed rows of sequence b are [offsets[b], offsets[b + 1]), row r is position source[r] of the
    flattened batch and the place[r]-th real token of its sequence (-1: its pad), and position p of the flattened batch is
    packed row spread[p]."""
    n = np.asarray(lengths, dtype=np.int64)
    rows = n + (n < length)
    offsets = np.concatenate([[0], np.cumsum(rows)])
    which = np.repeat(np.arange(len(n)), rows)
    at = np.arange(offsets[-1]) - offsets[which]
    place = np.where(at < n[which], at, -1)
    spread = offsets[:-1, None] + np.minimum(np.arange(length)[None, :], n[:, None])
    return offsets.astype(np.int32), which * length + at, place, spread.reshape(-1)


class HipEncoder:
    """An XLM-R model's forward pass in 8-bit products on the MI355X (inference only)."""

    def __init__(self, model, dtype: str = "bf16"):
        """model: a transformers XLMRobertaModel (or RobertaModel), whose tensors are read, not changed, and
        copied by ``to()``. dtype: what stands between the products, "bf16", "fp16" or "fp32"."""
        cfg = model.config
        if cfg.model_type not in MODEL_TYPES:
            raise ValueError(f"HipEncoder runs {' / '.join(MODEL_TYPES)} models, not {cfg.model_type}")
        if cfg.hidden_act != "gelu":
            raise ValueError(f"HipEncoder has the gelu activation only, not {cfg.hidden_act!r}")
        if getattr(cfg, "position_embedding_type", "absolute") not in ("absolute", None):
            raise ValueError(f"HipEncoder has absolute positions only, not {cfg.position_embedding_type!r}")
        if getattr(cfg, "is_decoder", False) or getattr(cfg, "add_cross_attention", False):
            raise ValueError("HipEncoder runs encoders, not decoders")
        head = cfg.hidden_size // cfg.num_attention_heads
        if head % 8 or head > 128:
            raise ValueError(f"HipEncoder needs a head size that is a multiple of 8 up to 128, not {head}")
        if dtype not in ("bf16", "fp16", "fp32"):
            raise ValueError("dtype must be 'bf16', 'fp16' or 'fp32'")
        self.config, self.dtype = cfg, dtype
        self.pad = int(cfg.pad_token_id)
        self._model = model
        self._device = None

    # -- weights -----------------------------------------------------------------------------------
    def to(self, device):
        """Lays the weights out on `device` (8-bit weights, fp32 biases, norms in `dtype`, the embedding tables as they are), all
        of them copies: a model that changes needs a new HipEncoder. Needs a GPU."""
        torch = _torch()
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"HipEncoder runs on the GPU only, not on {device}")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        if self._device == device:
            return self
        t = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[self.dtype]

        def linear(*parts):
            w = torch.cat([p.weight.detach().to(device, torch.float32) for p in parts])
            b = torch.cat([p.bias.detach().to(device, torch.float32) for p in parts])
            return (*ops.quantize_rows(w), b)

        def norm(p, dtype):
            return p.weight.detach().to(device, dtype, copy=True), p.bias.detach().to(device, dtype, copy=True)

        with torch.no_grad():
            e = self._model.embeddings
            tables = [x.weight.detach().to(device, copy=True)
                      for x in (e.word_embeddings, e.position_embeddings, e.token_type_embeddings)]
            embedding_norm = norm(e.LayerNorm, torch.float32)
            layers = [{"q": linear(x.attention.self.query), "kv": linear(x.attention.self.key, x.attention.self.value),
                       "o": linear(x.attention.output.dense), "norm1": norm(x.attention.output.LayerNorm, t),
                       "up": linear(x.intermediate.dense), "down": linear(x.output.dense),
                       "norm2": norm(x.output.LayerNorm, t)} for x in self._model.encoder.layer]
        self._words, self._positions, self._types = tables      # (all of it, or nothing)
        self._embedding_norm, self._layers = embedding_norm, layers
        self._t, self._device = t, device
        return self

    # -- forward -----------------------------------------------------------------------------------
    def __call__(self, input_ids, attention_mask=None, token_type_ids=None):
        """The tokenizer's tensors, (batch, length) each. Without attention_mask the tokens that are not pads are the mask; a
        transformers model would take all of them, pads too, as keys, so a batch with pads then warns."""
        torch = _torch()
        if self._device is None:
            raise RuntimeError("HipEncoder: call .to(device) first")
        if input_ids.dim() != 2:
            raise ValueError(f"input_ids has shape {tuple(input_ids.shape)}; expected (batch, length)")
        batch, length = input_ids.shape
        if length + self.pad + 1 > self._positions.shape[0]:
            raise ValueError(f"{length} tokens, but the model has positions for {self._positions.shape[0] - self.pad - 1}")
        for name, t in (("attention_mask", attention_mask), ("token_type_ids", token_type_ids)):
            if t is not None and t.shape != input_ids.shape:
                raise ValueError(f"{name} has shape {tuple(t.shape)}; expected {tuple(input_ids.shape)}")
        if batch == 0 or length == 0:
            return EncoderOutput(torch.zeros(batch, length, self.config.hidden_size, device=self._device))
        with torch.no_grad(), torch.cuda.device(self._device):
            ids = input_ids.to(self._device)
            mask = ids != self.pad if attention_mask is None else attention_mask.to(self._device) != 0
            types = None if token_type_ids is None else token_type_ids.to(self._device)
            lengths, lens = look(ids, mask, types, self.pad, self._words.shape[0], self._types.shape[0])
            if attention_mask is None and min(lengths) < length:
                warnings.warn("HipEncoder: no attention_mask, and there are pads: they are left out as keys (the model itself would "
                              "attend to them)", stacklevel=2)
            offsets, source, place, spread = pack(lengths, length)
            move = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(self._device)  # noqa: E731
            rows = move(np.stack([source, np.where(place < 0, self.pad, self.pad + 1 + place)]))
            offs, spread = move(offsets), move(spread)
            tokens = ids.reshape(-1)[rows[0]]
            other = self._positions[rows[1]].float()
            kind = 0 if token_type_ids is None else types.reshape(-1)[rows[0]]
            other = other + self._types[kind].float()
            h = self._forward(self._words[tokens].float(), other, offs, lens, int(np.diff(offsets).max()), max(lengths))
            return EncoderOutput(h.float()[spread].view(batch, length, -1))

    def _forward(self, words, other, offsets, lengths, max_q, max_k):
        """Packed rows: word embeddings plus the other embeddings, through the layers."""
        heads = self.config.num_attention_heads
        eps = float(self.config.layer_norm_eps)
        rows, hidden = words.shape
        t = self._t
        w, b = self._embedding_norm
        n = ops.block_norm(words, other, next_weight=w, next_bias=b, eps=eps, stream=False, rows8=True)
        x, x8, scale = n.normed.to(t), n.rows8, n.scale

        def product(rows8, scales, weights, act="none"):
            return ops.linear_int8(rows8, weights[0], weights[1], x_scale=scales, bias=weights[2], act=act, out_dtype=t)

        for i, y in enumerate(self._layers):
            q = product(x8, scale, y["q"]).view(rows, heads, -1)
            kv = product(x8, scale, y["kv"]).view(rows, 2, heads, -1)
            c = ops.cross_attention(q, kv[:, 0], kv[:, 1], q_offsets=offsets, k_offsets=offsets, key_lengths=lengths,
                                    max_q=max_q, max_k=max_k).view(rows, hidden)
            a = ops.linear_int8(c, y["o"][0], y["o"][1], bias=y["o"][2])
            n = ops.block_norm(a, x, next_weight=y["norm1"][0], next_bias=y["norm1"][1], eps=eps, stream=False, rows8=True)
            f = product(n.rows8, n.scale, y["up"], "gelu")
            f = ops.linear_int8(f, y["down"][0], y["down"][1], bias=y["down"][2])
            n = ops.block_norm(f, n.normed, next_weight=y["norm2"][0], next_bias=y["norm2"][1], eps=eps, stream=False,
                               rows8=i + 1 < len(self._layers))
            x, x8, scale = n.normed, n.rows8, n.scale
        return x
