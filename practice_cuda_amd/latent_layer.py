"""A latent-attention layer served in fp8: the package's operators in their order of use.

One token's keys and values come from one latent vector; only that and a shared
rotary key are kept. ``LatentAttention`` runs

    x + residual -> rms_norm_quant -> query and latent projections (block-scaled
    products) -> rotary positions -> latent_append into the paged cache

and then, for prompts (``prefill``), expands keys and values and attends with
``latent_prefill``, or, for new tokens (``decode``), moves the queries into the
latent space with a head-batched block-scaled product, attends over the cache
with ``latent_decode`` and applies the value maps the same way. Weights are
quantized once, in 128 x 128 blocks; activations in 1 x 128 groups.

The head-batched products are those of the reference's BMM benchmarks
(fp8_training/fp8_bench, kernels/fp8_bmm); the layer around them has no
counterpart there.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from .impls._common import without_gradient
from .impls.hip_latent import LatentCache, hip_latent_append, hip_latent_decode, hip_latent_prefill
from .impls.hip_per_block import hip_per_block_quant
from .impls.hip_rms_norm import hip_rms_norm_quant
from .modules import _block_scaled_bmm
from .registry import QuantResult


def _quant(x: torch.Tensor, block_m: int = 1) -> QuantResult:
    return hip_per_block_quant(x, block_m=block_m, block_n=128, cache_outputs=True)


def _product(a: QuantResult, w: QuantResult) -> torch.Tensor:
    """``a @ w^T`` per batch: a [B, M, K] in 1 x 128 groups, w [B, N, K] in 128 x 128 blocks."""
    return _block_scaled_bmm(a.tensor, a.dequant_scale, w.tensor.transpose(1, 2), w.dequant_scale.transpose(1, 2),
                             None, 1, 128, 128, torch.bfloat16)


class LatentAttention(nn.Module):
    """hidden -> heads x (head_dim + rope_dim) queries, one latent_dim + rope_dim vector a token.

    Widths as the attention kernels take them: latent 512, rotary 64, head 128,
    or 256, 32 and 64. Inputs are bfloat16 [tokens, hidden]; residual may be
    None (a stack's first layer). Both calls return (the layer's output, the
    residual to add to it)."""

    def __init__(self, hidden: int, heads: int, *, latent_dim: int = 512, rope_dim: int = 64, head_dim: int = 128,
                 norm_eps: float = 1e-6, rope_base: float = 10000.0, device=None) -> None:
        super().__init__()
        self.hidden, self.heads = hidden, heads
        self.latent_dim, self.rope_dim, self.head_dim = latent_dim, rope_dim, head_dim
        self.norm_eps = norm_eps
        self.softmax_scale = 1.0 / math.sqrt(head_dim + rope_dim)

        def weight(*shape):
            w = torch.empty(shape, dtype=torch.bfloat16, device=device)
            return nn.Parameter(nn.init.normal_(w, std=shape[-1] ** -0.5), requires_grad=False)

        kw = {"dtype": torch.bfloat16, "device": device}
        self.norm = nn.Parameter(torch.ones(hidden, **kw), requires_grad=False)
        self.latent_norm = nn.Parameter(torch.ones(latent_dim, **kw), requires_grad=False)
        self.w_query = weight(1, heads * (head_dim + rope_dim), hidden)
        self.w_latent = weight(1, latent_dim + rope_dim, hidden)
        self.w_key = weight(heads, head_dim, latent_dim)    # key of head h: w_key[h] c
        self.w_value = weight(heads, head_dim, latent_dim)  # value: w_value[h] c
        self.w_out = weight(1, hidden, heads * head_dim)
        freq = rope_base ** (-torch.arange(0, rope_dim, 2, device=device).float() / rope_dim)
        self.register_buffer("freq", freq, persistent=False)
        self._fp8 = self._made_from = None

    def quantize(self) -> "LatentAttention":
        """The weights' fp8 forms. The layer's calls make them where they are missing, or older than a weight that was
        loaded, replaced, moved or changed in place since. Edits that torch does not count (through ``.data``, or of
        weights made in inference mode) need a call of this. New codes take the old ones' places, so a captured graph
        reads them; they are there when this returns, for any stream."""
        codes, old = self._codes(), self._fp8
        capturing = torch.cuda.is_current_stream_capturing()
        if old is None or any(old[n].tensor.shape != c.tensor.shape or old[n].tensor.device != c.tensor.device
                              for n, c in codes.items()):
            if capturing:
                raise RuntimeError("quantize() in a captured graph renews codes: make them before the capture")
            self._fp8 = codes
        else:
            with torch.inference_mode():  # the old ones may be inference tensors
                for name, new in codes.items():
                    old[name].tensor.copy_(new.tensor)
                    old[name].dequant_scale.copy_(new.dequant_scale)
        if not capturing:
            # with torch's count of their changes in place, which inference tensors do not have
            self._made_from = [(n, w, None if w.is_inference() else w._version) for n, w in self._weights()]
            torch.cuda.current_stream(self.w_out.device).synchronize()
        return self

    def _codes(self) -> dict:
        both = torch.cat([self.w_key, self.w_value], 1).reshape(1, -1, self.latent_dim)
        return {
            "query": _quant(self.w_query, 128), "latent": _quant(self.w_latent, 128),
            "key_value": _quant(both, 128),  # [1, H * 2 head, latent], head after head
            "absorb": _quant(self.w_key.transpose(1, 2).contiguous(), 128),  # [H, latent, head]
            "value": _quant(self.w_value, 128), "out": _quant(self.w_out, 128),
        }

    def _weights(self):
        return [(name, getattr(self, name)) for name in ("w_query", "w_latent", "w_key", "w_value", "w_out")]

    def _current(self) -> bool:
        """Whether the codes are those of the weights as they are."""
        if self._fp8 is None:
            return False
        own = self._parameters  # the module's own lookup of a parameter takes half a microsecond
        for name, weight, count in self._made_from:
            if own.get(name) is not weight or count is not None and weight._version != count:
                return False
        return True

    def _apply(self, fn, recurse=True):
        """Moves and type changes put other data behind the same parameters."""
        def places():
            return [(w.data_ptr(), w.dtype, w.device) for _, w in self._weights()]

        before, freq = places(), self.freq
        super()._apply(fn, recurse)
        if self.freq.dtype != freq.dtype:  # 16 bits of a frequency are not enough at any distance
            self.freq = freq.to(self.freq.device)
        if places() != before:
            self._fp8 = self._made_from = None
        return self

    def _angles(self, positions: torch.Tensor):
        angle = positions.float()[:, None] * self.freq
        return angle.cos(), angle.sin()

    def _rotate(self, x: torch.Tensor, positions: torch.Tensor, angles=None) -> torch.Tensor:
        """Rotary positions over the halves of the last dimension; x [T, .., rope]; angles: those of the positions."""
        shape = (x.shape[0],) + (1,) * (x.ndim - 2) + (x.shape[-1] // 2,)
        cos, sin = (t.view(shape) for t in angles or self._angles(positions))
        a, b = x.float().chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(x.dtype)

    def _project(self, x, residual, cache, slots, positions):
        """(queries [T, H, head + rope], latents, rotary keys, residual); the tokens are in the cache."""
        normed, total = hip_rms_norm_quant(x[None], self.norm, residual=None if residual is None else residual[None],
                                           norm_eps=self.norm_eps)
        q = _product(normed, self._fp8["query"])[0].view(x.shape[0], self.heads, self.head_dim + self.rope_dim)
        both = _product(normed, self._fp8["latent"])[0]
        angles = self._angles(positions)
        latent, rope = both[:, :self.latent_dim], self._rotate(both[:, self.latent_dim:], positions, angles)
        q[..., self.head_dim:] = self._rotate(q[..., self.head_dim:], positions, angles)
        hip_latent_append(cache, latent, rope, slots, weight=self.latent_norm, norm_eps=self.norm_eps)
        return q, latent, rope, x if total is None else total[0]

    def _output(self, o: torch.Tensor) -> torch.Tensor:  # [T, H, head]
        return _product(_quant(o.reshape(1, o.shape[0], self.heads * self.head_dim)), self._fp8["out"])[0]

    def prefill(self, x, residual, cache: LatentCache, slots, positions, cu_seqlens):
        """Whole prompts, packed: sequence i holds tokens cu_seqlens[i] .. cu_seqlens[i + 1] - 1 (int32)."""
        return self._served(self._prefill, x, residual, cache, slots, positions, cu_seqlens)

    def decode(self, x, residual, cache: LatentCache, slots, positions, block_table, seq_lens):
        """New tokens, [B * S, hidden] for B = seq_lens.numel() sequences of S each; seq_lens counts them."""
        return self._served(self._decode, x, residual, cache, slots, positions, block_table, seq_lens)

    def _served(self, form, x, residual, *args):
        """Both forms are for inference: what requires a gradient gets the same results, and an error backward."""
        if torch.is_grad_enabled():
            inputs = [x, residual, *self._parameters.values()]
            for t in inputs:
                if t is not None and t.requires_grad:
                    with torch.no_grad():
                        results = self._with_codes(form, x, residual, *args)
                    return without_gradient(type(self).__name__, inputs, *results)
        return self._with_codes(form, x, residual, *args)

    def _with_codes(self, form, *args):
        if self._current():
            return form(*args)
        if not torch.cuda.is_current_stream_capturing():
            self.quantize()
            return form(*args)
        # A captured call is recorded and not run: its codes are the graph's own, made at every replay.
        held, self._fp8 = self._fp8, self._codes()
        try:
            return form(*args)
        finally:
            self._fp8 = held

    def _prefill(self, x, residual, cache, slots, positions, cu_seqlens):
        q, latent, rope, residual = self._project(x, residual, cache, slots, positions)
        c, _ = hip_rms_norm_quant(latent[None], self.latent_norm, norm_eps=self.norm_eps)
        both = _product(c, self._fp8["key_value"])[0].view(x.shape[0], self.heads, 2 * self.head_dim)
        o = hip_latent_prefill(q, both[..., :self.head_dim], rope, both[..., self.head_dim:], cu_seqlens, cu_seqlens,
                               softmax_scale=self.softmax_scale)
        return self._output(o), residual

    def _decode(self, x, residual, cache, slots, positions, block_table, seq_lens):
        tokens, batch, heads = x.shape[0], seq_lens.shape[0], self.heads
        new = tokens // batch if batch else 0
        if new * batch != tokens:
            raise ValueError(f"{tokens} tokens cannot be as many for each of {batch} sequences")
        q, _, _, residual = self._project(x, residual, cache, slots, positions)
        nope = _quant(q[..., :self.head_dim].transpose(0, 1).contiguous())  # [H, T, head]
        q_latent = _product(nope, self._fp8["absorb"])                      # [H, T, latent]
        shape = (heads, batch, new, self.latent_dim)
        o = torch.empty_like(q_latent)
        hip_latent_decode(q_latent.view(shape).permute(1, 2, 0, 3),
                          q[..., self.head_dim:].view(batch, new, heads, self.rope_dim), cache,
                          block_table, seq_lens, softmax_scale=self.softmax_scale,
                          out=o.view(shape).permute(1, 2, 0, 3))
        values = _product(_quant(o), self._fp8["value"])                    # [H, T, head]
        return self._output(values.transpose(0, 1)), residual


__all__ = ["LatentAttention"]
