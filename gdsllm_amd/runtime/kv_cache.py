"""Keys and values of the requests in flight, in 8 bits, over the gfx950 kernels.

Plays the part of the reference's KVCache (runtime/kv_cache.py: fp16 tensors
[layers, batch, heads, max_len, head_dim], every request as long as the
longest), with the state on the device: blocks of tokens that requests take
from a pool and give back, codes of 8 bits with one scale for each block and
head, and lengths that a captured step reads and advances by itself.

    cache = KVCache8(layers=32, requests=64, max_len=4096, kv_heads=8, head_dim=128)
    cache.begin_step(delta, max_tokens=64, max_new=1)      # once a step
    h = llama.cached_attention(x, weights, cache, layer, cos, sin)   # every layer
    cache.begin_step(-cache.lens * ended)                  # drop requests: no rows
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ext

BLOCK_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256)


class KVCache8:
    """The 8-bit KV cache of `layers` layers and up to `requests` requests of at
    most max_len tokens each (rounded up to whole blocks).

    num_blocks: blocks of block_size tokens in the pool all requests share
    (None: as many as hold every request at max_len); a request that needs a
    block when none is free is not served in that step (served()).  codes:
    torch.float8_e4m3fn or torch.int8.
    """

    def __init__(self, layers: int, requests: int, max_len: int, kv_heads: int, head_dim: int, block_size: int = 64,
                 num_blocks: Optional[int] = None, codes: torch.dtype = torch.float8_e4m3fn, device="cuda"):
        if layers < 1 or not 1 <= requests <= 8192 or max_len < 1 or kv_heads < 1:
            raise ValueError("KVCache8: layers, max_len and kv_heads must be positive, requests in [1, 8192]")
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"KVCache8: block_size must be one of {BLOCK_SIZES}, got {block_size}")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"KVCache8: head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if codes not in (torch.float8_e4m3fn, torch.int8):
            raise ValueError(f"KVCache8: codes must be float8_e4m3fn or int8, got {codes}")
        width = -(-max_len // block_size)
        num_blocks = requests * width if num_blocks is None else num_blocks
        if not 1 <= num_blocks <= (2 ** 31 - 1) // block_size:
            raise ValueError("KVCache8: num_blocks must be positive and num_blocks * block_size below 2^31")
        self.layers, self.requests, self.max_len = layers, requests, width * block_size
        self.kv_heads, self.head_dim, self.block_size, self.num_blocks = kv_heads, head_dim, block_size, num_blocks
        shape = (num_blocks, kv_heads, block_size, head_dim)
        # blocks are read only behind tokens that were written: no codes need a value
        self.k = [torch.empty(shape, dtype=codes, device=device) for _ in range(layers)]
        self.v = [torch.empty(shape, dtype=codes, device=device) for _ in range(layers)]
        self.k_scale = [torch.ones(shape[:2], dtype=torch.float32, device=device) for _ in range(layers)]
        self.v_scale = [torch.ones(shape[:2], dtype=torch.float32, device=device) for _ in range(layers)]
        i32 = dict(dtype=torch.int32, device=device)
        self.lens = torch.zeros(requests, **i32)
        self.block_tables = torch.zeros(requests, width, **i32)
        self.free_ring = torch.arange(num_blocks, **i32)
        self.free_state = torch.tensor([0, num_blocks], **i32)
        self.slots = self.positions = self.starts = None
        self._before = torch.zeros_like(self.lens)
        self._delta = torch.zeros_like(self.lens)
        self._max_new = self._max_len = 0

    @property
    def nbytes(self) -> int:
        """Bytes of codes and scales."""
        return sum(t.numel() * t.element_size() for ts in (self.k, self.v, self.k_scale, self.v_scale) for t in ts)

    def begin_step(self, delta: torch.Tensor, max_tokens: int = 0, max_new: int = 0, max_len: int = 0) -> None:
        """The blocks and slots of a step in which request r's tokens change by
        delta[r] (int32 [requests] on the device; positive: that many new tokens,
        negative: dropped from its end, all of them ends it).

        max_tokens: rows of the step's packed tensors, request after request
        (starts[r] .. starts[r + 1] - 1 are request r's).  max_new and max_len:
        bounds on a request's new tokens and length that the host knows (0: none),
        which attend() splits its work by.  Leaves lens, slots, positions and
        starts for the layers; asynchronous, and fit for a captured graph: lens and
        the blocks are then advanced by each replay, while slots, positions, starts
        and last_rows() stay those of the begin_step that Python ran last.
        """
        slots, positions, starts, lens, state = ext().kv_assign(
            self.lens, delta, self.block_tables, self.free_ring, self.free_state, self.block_size, max_tokens)
        self._before.copy_(self.lens)
        self._delta.copy_(delta)
        self.lens.copy_(lens)
        self.free_state.copy_(state)
        self.slots, self.positions, self.starts = slots, positions, starts
        self._max_new, self._max_len = max_new, min(max_len, self.max_len) if max_len else self.max_len

    def served(self) -> torch.Tensor:
        """bool [requests]: whether the last step gave the request what it asked
        for.  Rows of one that was not served are not written and their results
        mean nothing; it can ask again in a later step."""
        return (self._delta <= 0) | (self.lens != self._before)

    def last_rows(self) -> torch.Tensor:
        """int64 [requests]: the row of each request's last new token in this
        step's packed tensors; -1 for a request without one.  Of a captured step:
        taken within the capture."""
        last = self.starts[1:]
        return torch.where(last > self.starts[:-1], last - 1, -1).long()

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, q: Optional[torch.Tensor] = None,
               cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Write this step's keys and values (fp16 [max_tokens, kv_heads,
        head_dim]) into a layer's cache, turned by cos and sin (fp32 [positions,
        rotary / 2]) where they are given; returns q [max_tokens, heads,
        head_dim] turned the same way."""
        if self.slots is None:
            raise RuntimeError("KVCache8.append: begin_step comes first")
        if cos is not None and cos.shape[0] < self.max_len:
            # a token past the table would not be written, and read later all the same
            raise ValueError(f"KVCache8.append: cos and sin must reach position {self.max_len - 1}")
        return ext().kv_append(k, v, self.slots, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                               q, self.positions if cos is not None else None, cos, sin)

    def attend(self, layer: int, q: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
        """Causal attention of this step's rows q [max_tokens, heads, head_dim]
        over the tokens their requests hold; scale None: head_dim ** -0.5."""
        if self.slots is None:
            raise RuntimeError("KVCache8.attend: begin_step comes first")
        return ext().kv_attention(q, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                                  self.block_tables, self.lens, self.starts,
                                  self.head_dim ** -0.5 if scale is None else scale, self._max_new, self._max_len)


def rope_table(max_pos: int, rotary: int, theta: float = 10000.0, inv_freq: Optional[torch.Tensor] = None,
               device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), fp32 [max_pos, rotary / 2], of position * inv_freq (None:
    theta ** (-2 i / rotary)), the angles of runtime/llama.py:27-57 taken in 64
    bits (in 32, those at position 100000 are off by up to 0.005).
    Channels i and i + rotary / 2 of a head turn together."""
    if inv_freq is None:
        inv_freq = theta ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    if inv_freq.shape != (rotary // 2,):
        raise ValueError(f"rope_table: inv_freq must hold {rotary // 2} values")
    angle = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv_freq.double().cpu()
    return angle.cos().float().to(device), angle.sin().float().to(device)
