"""Self-attention of a video that arrives in chunks of frames.

A layer keeps the keys and values of the tokens so far in a ``StreamCache``
with a sliding window and sinks: the first tokens (usually the first frame)
and the newest ones stay, the others' slots are taken again, so a stream holds
a fixed amount of memory however long it is. It ends where its rotary table
does, and with its int32 lengths, 2^31 - 256 tokens. ``Wan_Stream_Processor`` drives an
attention module (the members ``Wan_DFSAttn_Processor2_0`` uses) over such a
cache: ``linear`` for the projections, ``qkv_cache`` for norms, rotation and
append, ``window_attention`` over the cache.

A chunk may pass through the model several times (denoising steps, guidance)
before it is done: each pass writes the chunk's keys and values to the same
slots, and ``advance`` moves on behind them. A conditional and an unconditional
pass have caches of their own.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from . import ops
from .replace_wan import Wan_DFSAttn_Processor2_0, _norm_args, rms_norm_like, rope_tables


class StreamCache:
    """Keys and values of ``batch`` streams: ``heads`` key heads of ``head_dim``
    channels, the first ``sinks`` tokens and at least ``left`` tokens before
    a chunk of up to ``chunk`` tokens."""

    MOST = 0x7fffff00  # keys that window_attention counts

    def __init__(self, batch: int, heads: int, head_dim: int, left: int, chunk: int, sinks: int = 0, device="cuda",
                 dtype: torch.dtype = torch.bfloat16):
        for name, n in (("batch", batch), ("heads", heads), ("left", left + 1), ("chunk", chunk), ("sinks", sinks + 1)):
            if n <= 0:
                raise ValueError(f"StreamCache: {name} is too small")
        self.left, self.chunk, self.sinks = left, chunk, sinks
        shape = (batch, heads, sinks + left + chunk, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        with torch.inference_mode(False):  # an inference tensor would not count its changes
            self.lens = torch.zeros(batch, dtype=torch.int32, device=device)  # tokens behind which the chunk stands
        self._keep(0)

    def _keep(self, position: Optional[int]) -> None:
        """What lens holds, by the host's count (None: not known, as under a
        capture, whose replays move lens unseen)."""
        if self.lens.is_cuda and torch.cuda.is_current_stream_capturing():
            position = None
        self._known = (self.lens, self.lens._version, position)

    def _position(self) -> Optional[int]:
        """The host's count, None where lens was moved otherwise than by
        ``advance`` and ``reset``."""
        lens, version, position = self._known
        return position if self.lens is lens and lens._version == version else None

    def attend(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
               k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
               table: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
               right: Optional[int] = None) -> torch.Tensor:
        """Writes a chunk's keys and values behind the tokens so far and
        attends over them all: q [B, T, H, D], k and v [B, T, G, D] as the
        projections leave them (see ``ops.qkv_cache``), out [B, H, T, D] in
        token-major storage. right: how far a token sees ahead within the
        chunk (None: all of it, 0: causal). A chunk past the table's last row
        is refused; where the host does not know the place (lens moved by hand
        or by a replayed graph), the rows past it are NaN."""
        tokens = q.shape[1]
        if tokens > self.chunk:
            raise ValueError(f"StreamCache: a chunk of {tokens} tokens, made for {self.chunk}")
        at = self._position()
        if at is not None and table is not None and at + tokens > table[0].shape[0]:
            raise ValueError(f"StreamCache: tokens {at} to {at + tokens - 1} of a stream whose rotary table has "
                             f"{table[0].shape[0]} rows")
        if at is not None and at + tokens > self.MOST:
            raise ValueError(f"StreamCache: a stream holds up to 2^31 - 256 tokens, this chunk ends at {at + tokens}")
        q = ops.qkv_cache(q, k, v, self.k, self.v, self.lens, q_weight, k_weight, eps, table, sinks=self.sinks,
                          rolling=True)
        return ops.window_attention(q, self.k, self.v, self.left, right, self.sinks, kv_lens=self.lens + tokens,
                                    rolling=True)

    def advance(self, tokens: int) -> None:
        """The chunk's ``tokens`` are final; the next one follows them."""
        if not 0 <= tokens <= self.chunk:
            raise ValueError(f"StreamCache: advance by {tokens} of a chunk of up to {self.chunk} tokens")
        at = self._position()
        self.lens += tokens
        self._keep(None if at is None else at + tokens)

    def reset(self) -> None:
        self.lens.zero_()
        self._keep(0)


class Wan_Stream_Processor:
    """Processor of a self-attention module over a ``StreamCache``: hidden
    states are a chunk's tokens [B, T, C], rotary_emb the complex table of all
    positions (as the model's blocks pass it)."""

    takes_chunks = True  # the tokens need not be the whole table's

    def __init__(self, cache: StreamCache, right: Optional[int] = None):
        self.cache = cache
        self.right = right

    def __call__(self, attn, hidden_states: torch.Tensor, encoder_hidden_states: Optional[torch.Tensor] = None,
                 attention_mask: Optional[torch.Tensor] = None,
                 rotary_emb: Optional[torch.Tensor] = None) -> torch.Tensor:
        if encoder_hidden_states is not None or attention_mask is not None or attn.add_k_proj is not None:
            raise NotImplementedError("a stream's processor runs self-attention without a mask")
        heads = attn.heads
        q, k, v = (ops.linear(hidden_states, p.weight, p.bias).unflatten(2, (heads, -1))
                   for p in (attn.to_q, attn.to_k, attn.to_v))
        channels = heads * q.shape[3]
        if not (rms_norm_like(attn.norm_q, channels) and rms_norm_like(attn.norm_k, channels)):
            raise NotImplementedError("a stream's processor takes RMS norms over all heads or none")
        wq, eq = _norm_args(attn.norm_q, channels, q)
        wk, ek = _norm_args(attn.norm_k, channels, k)
        if wq is not None and wk is not None and eq != ek:
            raise NotImplementedError(f"norm_q and norm_k have different eps ({eq} and {ek})")
        out = self.cache.attend(q, k, v, wq, wk, eq if wq is not None else ek,
                                None if rotary_emb is None else rope_tables(rotary_emb), self.right)
        to_out = attn.to_out[0]
        return attn.to_out[1](ops.linear(out.transpose(1, 2).flatten(2), to_out.weight, to_out.bias))


def install_stream_processors(model, left: int, chunk: int, sinks: int = 0, right: Optional[int] = None,
                              batch: int = 1) -> List[StreamCache]:
    """A ``Wan_Stream_Processor`` with its own cache on every self-attention
    module of a WanLikeDiT, dense attention on the text modules; returns the
    caches. ``model(latent, timestep, context)`` then takes the next frames'
    latent alone; advance the caches once the frames are done."""
    caches = []
    for i, (name, module) in enumerate(model.attention_modules()):
        if "attn2" in name:
            module.set_processor(Wan_DFSAttn_Processor2_0("full", 0.0, 16, 128, None, i, [], 0, 1, 0.0, False, True))
            continue
        weight = module.to_k.weight
        caches.append(StreamCache(batch, module.heads, weight.shape[0] // module.heads, left, chunk, sinks,
                                  weight.device, weight.dtype))
        module.set_processor(Wan_Stream_Processor(caches[-1], right))
    return caches
