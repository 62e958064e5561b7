"""Conditioning around the DiT stream on the few-row operators: INT4 weights
for the projections of a timestep or a prompt, and a cross-attention adapter
(an image prompt) next to the block stack.  No reference counterpart.

* ``W4Linear`` -- a plain linear's weight as INT4 codes with group-128 scales,
  run by ``ops.w4_linear`` on unquantised rows.  ``k2b.dit`` takes one in the
  place of any of its small linears: at Krea2 widths the six modulation
  vectors of one latent then read 117 MB instead of 453.
* ``CrossAdapter`` -- decoupled cross attention: x + strength * W_o attn(W_q x;
  K, V of an encoder's states).  The keys and values are made once per prompt
  (``keys``: two few-row products and the key head norms) and kept over the
  denoising steps; a step (``add``) projects, norms and rotates the stream's
  queries, attends, and adds the projection through the W4A4 GEMM's gated
  residual.

    adapter = synthetic_adapter(cfg, width=1280)
    kept = adapter.keys(states, lengths)              # once per prompt
    for t in timesteps:
        x = adapter.add(x, kept, freqs=freqs, strength=0.6)
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import ops
from .model import ModelConfig, quantize_weight
from .ops import PreparedWeight


def pack_w4(w: torch.Tensor):
    """[n, k] -> packed INT4 (uint8 [n, k/2]) + fp16 group-128 scales, without
    rotation: codes clamp(rne(w / s), -8, 7), s = absmax / 7."""
    n, k = w.shape
    g = w.float().view(n, k // 128, 128)
    s = (g.abs().amax(-1) / 7).to(torch.float16)
    step = torch.where(s > 0, s.float(), 1.0)[..., None]
    c = torch.round(g / step).clamp_(-8, 7).to(torch.int8).view(n, k)
    packed = (c[:, 0::2] & 15) | ((c[:, 1::2] & 15) << 4)
    return packed.view(torch.uint8).contiguous(), s.contiguous()


@dataclass
class W4Linear:
    packed: torch.Tensor            # uint8 [n, k/2]
    scales: torch.Tensor            # fp16 [n, k/128]
    bias: Optional[torch.Tensor] = None
    rotate: bool = True             # the weight was rotated along k (quantize_weight)
    dense: Optional[torch.Tensor] = None  # bf16 [n, k]: the same weight for calls of many rows (k2b.dit)

    @classmethod
    def of(cls, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, dense: bool = False) -> "W4Linear":
        """Quantises a plain linear's weight [n, k]; rotated where the library's
        quantiser takes the width (k a multiple of 512).  ``dense``: keeps what
        the codes stand for in bf16 as well."""
        rotate = weight.shape[1] % 512 == 0
        packed, scales = quantize_weight(weight) if rotate else pack_w4(weight)
        made = cls(packed, scales, bias, rotate)
        if dense:
            made.dense = made.expand()
        return made

    def expand(self) -> torch.Tensor:
        """The weight that the codes and scales stand for, unrotated, bf16 [n, k]."""
        n, k = self.packed.shape[0], 2 * self.packed.shape[1]
        codes = torch.stack([self.packed & 15, self.packed >> 4], -1).view(n, k // 128, 128).float()
        w = torch.where(codes > 7, codes - 16, codes) * self.scales.float()[..., None]
        if self.rotate:
            h = torch.ones(1, 1, device=w.device)
            while h.shape[0] < 128:
                h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)])
            w = w @ (h * 128 ** -0.5)
        return w.view(n, k).to(torch.bfloat16)

    def __call__(self, x: torch.Tensor, act: str = "none") -> torch.Tensor:
        """x [..., k]; rows that are not evenly spaced (a slice of a batch of
        sequences) are copied together."""
        rows = x if x.is_contiguous() else x.reshape(-1, x.shape[-1])
        y = ops.w4_linear(rows, self.packed, self.scales, self.bias, rotate=self.rotate, act=act)
        return y.view(*x.shape[:-1], y.shape[-1])


@dataclass
class EncoderKeys:
    """One prompt's keys and values, kept between denoising steps."""

    k: torch.Tensor                  # bf16 [B|1, kvheads, L, 128], normed
    v: torch.Tensor
    lengths: Optional[torch.Tensor]  # int32 [B]
    bias: Optional[torch.Tensor]     # fp32 [B|1, L]


@dataclass
class CrossAdapter:
    heads: int
    kvheads: int
    wq: PreparedWeight    # [heads * 128, hidden], W4A4 like the block stack's
    wo: PreparedWeight    # [hidden, heads * 128]
    wk: W4Linear          # [kvheads * 128, width]
    wv: W4Linear
    qnorm: torch.Tensor   # fp32 [128] ("w+1" form)
    knorm: torch.Tensor
    eps: float = 1e-6

    def keys(self, states: torch.Tensor, lengths: Optional[torch.Tensor] = None,
             emphasis: Optional[torch.Tensor] = None) -> EncoderKeys:
        """states bf16 [B|1, L, width] of an encoder, the first lengths[b] of
        each real; emphasis fp32 [B|1, L]: positive weights of the tokens."""
        B, L, _ = states.shape
        split = lambda t: t.view(B, L, self.kvheads, 128).transpose(1, 2)  # noqa: E731
        k, v = split(self.wk(states)), split(self.wv(states))
        k, _ = ops.qk_norm_rope(k, None, self.knorm, None, eps_q=self.eps)
        return EncoderKeys(k, v, lengths, None if emphasis is None else torch.log(emphasis))

    def attend(self, x: torch.Tensor, kept: EncoderKeys, freqs: Optional[torch.Tensor] = None,
               mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x bf16 [B, L, hidden] -> attention output bf16 [B, L, heads * 128].
        freqs: the stream's rotation table, or None; mask as in
        ops.cross_attention (regional prompts)."""
        B, L, hidden = x.shape
        q = ops.gemm_bf16(*ops.rotate_quant(x.reshape(B * L, hidden)), self.wq)
        q, _ = ops.qk_norm_rope(q.view(B, L, self.heads, 128).transpose(1, 2), None, self.qnorm, None, freqs,
                                eps_q=self.eps)
        return ops.cross_attention(q, kept.k, kept.v, lengths=kept.lengths, mask=mask, bias=kept.bias)

    def add(self, x: torch.Tensor, kept: EncoderKeys, *, freqs: Optional[torch.Tensor] = None, strength: float = 1.0,
            mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x + strength * W_o attend(x), bf16 [B, L, hidden].  The strength is the
        gate of the W4A4 GEMM's residual, which is bf16: 0.6 acts as 0.6016."""
        B, L, hidden = x.shape
        o = self.attend(x, kept, freqs, mask)
        oq, os_ = ops.rotate_quant(o.view(B * L, self.heads * 128))
        gate = torch.full((B, hidden), strength, dtype=torch.bfloat16, device=x.device)
        return ops.gated_residual(oq, os_, self.wo, gate, x.reshape(B * L, hidden), length=L).view(B, L, hidden)


def synthetic_adapter(cfg: ModelConfig, width: int, seed: int = 0, device="cuda") -> CrossAdapter:
    """Seeded random-init adapter for a stream of cfg.hidden and an encoder of
    ``width``: N(0, 0.02) weights, norm multipliers ~U(0.9, 1.1)."""
    gen = torch.Generator(device=device).manual_seed(seed + 104729)

    def weight(n, k):
        return (torch.randn((n, k), generator=gen, device=device) * 0.02).to(torch.bfloat16)

    def norm():
        return (torch.rand(128, generator=gen, device=device) * 0.2 - 0.1).contiguous()

    return CrossAdapter(cfg.heads, cfg.kvheads,
                        wq=ops.prepare_weight(*quantize_weight(weight(cfg.heads * 128, cfg.hidden))),
                        wo=ops.prepare_weight(*quantize_weight(weight(cfg.hidden, cfg.heads * 128))),
                        wk=W4Linear.of(weight(cfg.kvheads * 128, width)),
                        wv=W4Linear.of(weight(cfg.kvheads * 128, width)), qnorm=norm(), knorm=norm(), eps=cfg.qk_eps)
