"""Keys and values of the requests in flight, in 8 or 4 bits, over the gfx950 kernels.

Plays the part of the reference's KVCache (runtime/kv_cache.py: fp16 tensors
[layers, batch, heads, max_len, head_dim], every request as long as the
longest), with the state on the device: blocks of tokens that requests take
from a pool and give back, codes of 8 bits with one scale for each block and
head (KVCache8) or of 4 bits with a scale and bias for each token and group of
channels (KVCache4), and lengths that a captured step reads and advances by itself.

    cache = KVCache8(layers=32, requests=64, max_len=4096, kv_heads=8, head_dim=128)
    cache.begin_step(delta, max_tokens=64, max_new=1)      # once a step
    h = llama.cached_attention(x, weights, cache, layer, cos, sin)   # every layer
    cache.begin_step(-cache.lens * ended)                  # drop requests: no rows
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import ext

BLOCK_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256)
GROUP_SIZES = (32, 64, 128)


class _PagedCache:
    """What the caches share: the requests' lengths and blocks on the device."""

    _MOST_RUNS = None  # of a block and a kv head, where the kernels count them in 32 bits

    def __init__(self, layers: int, requests: int, max_len: int, kv_heads: int, head_dim: int, block_size: int,
                 num_blocks: Optional[int], device):
        me = type(self).__name__
        if layers < 1 or not 1 <= requests <= 8192 or max_len < 1:
            raise ValueError(f"{me}: layers and max_len must be positive, requests in [1, 8192]")
        if not 1 <= kv_heads <= 1024:
            raise ValueError(f"{me}: kv_heads must be in [1, 1024], got {kv_heads}")
        if block_size not in BLOCK_SIZES:
            raise ValueError(f"{me}: block_size must be one of {BLOCK_SIZES}, got {block_size}")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"{me}: head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        width = -(-max_len // block_size)
        if width * block_size > 2 ** 31 - 8192:
            raise ValueError(f"{me}: max_len must be at most 2^31 - 8192, got {max_len}")
        num_blocks = requests * width if num_blocks is None else num_blocks
        if not 1 <= num_blocks <= (2 ** 31 - 1) // block_size:
            raise ValueError(f"{me}: num_blocks must be positive and num_blocks * block_size below 2^31")
        if self._MOST_RUNS and num_blocks * kv_heads > self._MOST_RUNS:
            raise ValueError(f"{me}: num_blocks * kv_heads must be at most {self._MOST_RUNS}")
        self.layers, self.requests, self.max_len = layers, requests, width * block_size
        self.kv_heads, self.head_dim, self.block_size, self.num_blocks = kv_heads, head_dim, block_size, num_blocks
        i32 = dict(dtype=torch.int32, device=device)
        self.lens = torch.zeros(requests, **i32)
        self.block_tables = torch.zeros(requests, width, **i32)
        self.free_ring = torch.arange(num_blocks, **i32)
        self.free_state = torch.tensor([0, num_blocks], **i32)
        self.slots = self.positions = self.starts = None
        self._before = torch.zeros_like(self.lens)
        self._delta = torch.zeros_like(self.lens)
        self._max_new = self._max_len = 0

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

    def _begun(self, what: str) -> None:
        if self.slots is None:
            raise RuntimeError(f"{type(self).__name__}.{what}: begin_step comes first")

    def _reaches(self, cos: Optional[torch.Tensor]) -> None:
        # a token past the table would not be written, and read later all the same
        if cos is not None and cos.shape[0] < self.max_len:
            raise ValueError(f"{type(self).__name__}.append: cos and sin must reach position {self.max_len - 1}")

    def _scale(self, scale: Optional[float]) -> float:
        return self.head_dim ** -0.5 if scale is None else scale


class KVCache8(_PagedCache):
    """The 8-bit KV cache of `layers` layers and up to `requests` requests of at
    most max_len tokens each (rounded up to whole blocks).

    num_blocks: blocks of block_size tokens in the pool all requests share
    (None: as many as hold every request at max_len); a request that needs a
    block when none is free is not served in that step (served()).  codes:
    torch.float8_e4m3fn or torch.int8.
    """

    def __init__(self, layers: int, requests: int, max_len: int, kv_heads: int, head_dim: int, block_size: int = 64,
                 num_blocks: Optional[int] = None, codes: torch.dtype = torch.float8_e4m3fn, device="cuda"):
        if codes not in (torch.float8_e4m3fn, torch.int8):
            raise ValueError(f"KVCache8: codes must be float8_e4m3fn or int8, got {codes}")
        super().__init__(layers, requests, max_len, kv_heads, head_dim, block_size, num_blocks, device)
        shape = (self.num_blocks, kv_heads, block_size, head_dim)
        # blocks are read only behind tokens that were written: no codes need a value
        self.k = [torch.empty(shape, dtype=codes, device=device) for _ in range(layers)]
        self.v = [torch.empty(shape, dtype=codes, device=device) for _ in range(layers)]
        self.k_scale = [torch.ones(shape[:2], dtype=torch.float32, device=device) for _ in range(layers)]
        self.v_scale = [torch.ones(shape[:2], dtype=torch.float32, device=device) for _ in range(layers)]

    @property
    def nbytes(self) -> int:
        """Bytes of codes and scales."""
        return sum(t.numel() * t.element_size() for ts in (self.k, self.v, self.k_scale, self.v_scale) for t in ts)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, q: Optional[torch.Tensor] = None,
               cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
               neighbours: bool = False) -> Optional[torch.Tensor]:
        """Write this step's keys and values (fp16 [max_tokens, kv_heads,
        head_dim]) into a layer's cache, turned by cos and sin (fp32 [positions,
        rotary / 2]) where they are given; returns q [max_tokens, heads,
        head_dim] turned the same way.  neighbours: channels 2i and 2i + 1 of a
        head turn together (rope, a launch of its own), else i and i + rotary / 2."""
        self._begun("append")
        self._reaches(cos)
        positions = self.positions if cos is not None else None
        if neighbours and cos is not None:
            # rope has no slots: a row that is not served has no position either
            turned, other = ext().rope(k if q is None else q, None if q is None else k, positions, cos, sin, True)
            k, q = (turned, None) if q is None else (other, turned)
            ext().kv_append(k, v, self.slots, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer])
            return q
        return ext().kv_append(k, v, self.slots, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                               q, positions, cos, sin)

    def attend(self, layer: int, q: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
        """Causal attention of this step's rows q [max_tokens, heads, head_dim]
        over the tokens their requests hold; scale None: head_dim ** -0.5."""
        self._begun("attend")
        return ext().kv_attention(q, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                                  self.block_tables, self.lens, self.starts, self._scale(scale), self._max_new, self._max_len)


class KVCache4(_PagedCache):
    """KVCache8's cache in 4 bits, the affine format of 4-bit weights: codes of
    each token and head with an fp16 scale and bias for every group_size (32, 64
    or 128) channels, 4.25 to 5 bits an element.  A token is quantized by itself: what other tokens of
    its block hold stays.  Same methods, and values()."""

    _MOST_RUNS = 2 ** 31 - 1

    def __init__(self, layers: int, requests: int, max_len: int, kv_heads: int, head_dim: int, block_size: int = 64,
                 num_blocks: Optional[int] = None, group_size: int = 64, device="cuda"):
        if group_size not in GROUP_SIZES or group_size > head_dim:
            raise ValueError(f"KVCache4: group_size must be one of {GROUP_SIZES} and at most head_dim, got {group_size}")
        super().__init__(layers, requests, max_len, kv_heads, head_dim, block_size, num_blocks, device)
        self.group_size = group_size
        codes = (self.num_blocks, kv_heads, block_size, head_dim // 2)
        affine = (self.num_blocks, kv_heads, head_dim // group_size, block_size, 2)
        # blocks are read only behind tokens that were written: nothing needs a value
        self.k = [torch.empty(codes, dtype=torch.uint8, device=device) for _ in range(layers)]
        self.v = [torch.empty(codes, dtype=torch.uint8, device=device) for _ in range(layers)]
        self.k_affine = [torch.empty(affine, dtype=torch.float16, device=device) for _ in range(layers)]
        self.v_affine = [torch.empty(affine, dtype=torch.float16, device=device) for _ in range(layers)]

    @property
    def nbytes(self) -> int:
        """Bytes of codes, scales and biases."""
        return sum(t.numel() * t.element_size() for ts in (self.k, self.v, self.k_affine, self.v_affine) for t in ts)

    def _layer(self, layer: int) -> tuple:
        return self.k[layer], self.v[layer], self.k_affine[layer], self.v_affine[layer]

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, q: Optional[torch.Tensor] = None,
               cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
               neighbours: bool = False) -> Optional[torch.Tensor]:
        """KVCache8.append, in one launch for both ways of pairing channels."""
        self._begun("append")
        self._reaches(cos)
        return ext().kv4_append(k, v, self.slots, *self._layer(layer), q, self.positions if cos is not None else None, cos, sin,
                                neighbours)

    def attend(self, layer: int, q: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
        """Causal attention of this step's rows q [max_tokens, heads, head_dim]
        over the tokens their requests hold; scale None: head_dim ** -0.5."""
        self._begun("attend")
        return ext().kv4_attention(q, *self._layer(layer), self.block_tables, self.lens, self.starts, self._scale(scale),
                                   self._max_new, self._max_len)

    def values(self, layer: int, request: int, tokens: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """(k, v), fp16 [tokens, kv_heads, head_dim]: what the cache holds of a
        request's first `tokens` tokens (the keys as they were turned), to move it
        into another cache; zeros past its length."""
        if not 0 <= request < self.requests or not 0 <= tokens <= self.max_len:
            raise ValueError(f"KVCache4.values: request must be in [0, {self.requests}), tokens in [0, {self.max_len}]")
        at = torch.arange(tokens, dtype=torch.int32, device=self.lens.device)
        slots = self.block_tables[request][at // self.block_size] * self.block_size + at % self.block_size
        return ext().kv4_values(torch.where(at < self.lens[request], slots, -1).int(), *self._layer(layer))


def rope_frequencies(rotary: int, theta: float = 10000.0, scaling: Optional[dict] = None) -> Tuple[torch.Tensor, float]:
    """(inv_freq, factor): the rotary / 2 angles of a position, theta ** (-2 i /
    rotary) scaled for contexts longer than the model was trained on, in 64 bits,
    and what cos and sin are multiplied by (1 but for "yarn").

    scaling, as a checkpoint's configuration spells it (its type under
    "rope_type" or "type"; None or "default": none), s = factor, L =
    original_max_position_embeddings, w = 2 pi / inv_freq:
      "linear"  inv_freq / s
      "ntk"     theta * s ** (rotary / (rotary - 2)) in theta's place
      "llama3"  inv_freq / s where w > L / low_freq_factor, as it is where w < L /
                high_freq_factor, between them the mean of both weighted by (L / w -
                low) / (high - low)
      "yarn"    inv_freq / s for pairs past beta_slow turns in L positions, as it
                is for those before beta_fast (32 and 1 where they are not given), a
                line in i between them, from and to whole pairs unless truncate is
                false; factor = attention_factor, or t(mscale) / t(mscale_all_dim)
                with t(m) = 0.1 m ln s + 1 where both are given, or t(1).  (Models
                that give mscale_all_dim also multiply the scale of their scores by
                t(mscale_all_dim) ** 2: attend's `scale`.)
    A key that its kind does not use is refused, but for those that say what the
    arguments say or what the model is: rope_theta (must be theta),
    partial_rotary_factor, original_max_position_embeddings, finetuned.  A key
    with None is not given.
    """
    if rotary < 2 or rotary % 2:
        raise ValueError(f"rope_frequencies: rotary must be even and positive, got {rotary}")
    scaling = {key: v for key, v in (scaling or {}).items() if v is not None}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if scaling.get("type", kind) != kind:
        raise ValueError(f"rope_frequencies: rope_type {kind!r} and type {scaling['type']!r} differ")
    if kind not in _SCALING_KEYS:
        raise ValueError(f"rope_frequencies: unknown scaling {kind!r}")
    other = sorted(set(scaling) - _SCALING_KEYS[kind] - _MODEL_KEYS)
    if other:
        raise ValueError(f"rope_frequencies: {kind} does not use {', '.join(map(repr, other))}")
    if float(scaling.get("rope_theta", theta)) != theta:
        raise ValueError(f"rope_frequencies: rope_theta is {scaling['rope_theta']}, theta {theta}")
    i = torch.arange(rotary // 2, dtype=torch.float64)

    def need(key: str, low: float) -> float:
        v = scaling.get(key)
        if v is None or not float(v) >= low:
            raise ValueError(f"rope_frequencies: {kind} needs {key} >= {low}, got {v}")
        return float(v)

    if kind == "ntk":
        if rotary == 2:
            raise ValueError("rope_frequencies: ntk needs more than one pair")
        return (theta * need("factor", 1.0) ** (rotary / (rotary - 2))) ** (-2 * i / rotary), 1.0
    f = theta ** (-2 * i / rotary)
    if kind == "default":
        return f, 1.0
    s = need("factor", 1.0)
    if kind == "linear":
        return f / s, 1.0
    length = need("original_max_position_embeddings", 1.0)
    if kind == "llama3":
        low, high = need("low_freq_factor", 0.0), need("high_freq_factor", 0.0)
        if not high > low:
            raise ValueError("rope_frequencies: llama3 needs high_freq_factor > low_freq_factor")
        keep = ((length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return (1 - keep) * f / s + keep * f, 1.0
    if not theta > 1:
        raise ValueError(f"rope_frequencies: yarn needs theta > 1, got {theta}")

    def pair_of(turns: float) -> float:
        """The pair (a real number) that turns so often in `length` positions."""
        return rotary * math.log(length / (2 * math.pi * turns)) / (2 * math.log(theta))

    fast, slow = float(scaling.get("beta_fast") or 32.0), float(scaling.get("beta_slow") or 1.0)
    if not fast >= slow > 0:
        raise ValueError(f"rope_frequencies: yarn needs beta_fast >= beta_slow > 0, got {fast} and {slow}")
    first, last = pair_of(fast), pair_of(slow)
    if scaling.get("truncate", True):
        first, last = math.floor(first), math.ceil(last)
    first, last = max(first, 0), min(last, rotary - 1)
    slowed = ((i - first) / (last - first)).clamp(0, 1) if last > first else (i > first).double()
    return slowed * f / s + (1 - slowed) * f, _yarn_factor(scaling, s)


# Keys that a dictionary of any kind may hold, and those that a kind's formula reads.
_MODEL_KEYS = {"rope_type", "type", "rope_theta", "partial_rotary_factor", "original_max_position_embeddings", "finetuned"}
_SCALING_KEYS = {
    "default": set(),
    "linear": {"factor"},
    "ntk": {"factor"},
    "llama3": {"factor", "low_freq_factor", "high_freq_factor"},
    "yarn": {"factor", "beta_fast", "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim"},
}


def _yarn_factor(scaling: dict, s: float) -> float:
    """What yarn multiplies cos and sin by."""
    if "attention_factor" in scaling:
        return float(scaling["attention_factor"])
    m, all_dim = float(scaling.get("mscale") or 0.0), float(scaling.get("mscale_all_dim") or 0.0)
    if m < 0 or all_dim < 0:
        raise ValueError("rope_frequencies: mscale and mscale_all_dim must not be negative")
    if not all_dim and m in (0.0, 1.0):
        return 0.1 * math.log(s) + 1
    if not m or not all_dim:  # programs differ in what one without the other means
        raise ValueError("rope_frequencies: yarn needs mscale and mscale_all_dim together")
    return (0.1 * m * math.log(s) + 1) / (0.1 * all_dim * math.log(s) + 1)


def rope_table(max_pos: int, rotary: int, theta: float = 10000.0, inv_freq: Optional[torch.Tensor] = None,
               device="cuda", scaling: Optional[dict] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), fp32 [max_pos, rotary / 2], of position * inv_freq (None:
    those of rope_frequencies, with its scaling for long contexts), the angles of
    runtime/llama.py:27-57 taken in 64 bits (in 32, those at position 100000 are
    off by up to 0.005)."""
    factor = 1.0
    if inv_freq is None:
        inv_freq, factor = rope_frequencies(rotary, theta, scaling)
    elif scaling is not None:
        raise ValueError("rope_table: scaling is for the frequencies that inv_freq replaces")
    if inv_freq.shape != (rotary // 2,):
        raise ValueError(f"rope_table: inv_freq must hold {rotary // 2} values")
    angle = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv_freq.double().cpu()
    return (factor * angle.cos()).float().to(device), (factor * angle.sin()).float().to(device)
