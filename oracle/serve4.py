"""Plain 64-bit forms of the 4-bit cache's operators (test infrastructure only):
rotation of both pairings, the affine codes, attention over the elements they
stand for.  CPU torch."""

from __future__ import annotations

import numpy as np
import torch

from .serve import blocks


def rotate(x, positions, cos, sin, neighbours=False):
    """fp16 [T, H, D] turned by positions -> (the fp16 values gdsllm_rope writes, through fp32; the 64-bit ones).  Zeros
    where there is no position."""
    half = cos.shape[1]
    live = ((positions >= 0) & (positions < cos.shape[0]))[:, None, None]
    c, s = (t.double()[positions.clamp(0, cos.shape[0] - 1).long()][:, None, :] for t in (cos, sin))
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if neighbours else (slice(0, half), slice(half, 2 * half))
    y = x.double()
    y[..., a], y[..., b] = x[..., a].double() * c - x[..., b].double() * s, x[..., b].double() * c + x[..., a].double() * s
    y = torch.where(live, y, 0.0)
    return y.float().half(), y


def quantize(x, group):
    """fp16 [..., D] -> codes uint8 [..., D], scale and bias fp16 [..., D / group]."""
    y = x.double().unflatten(-1, (-1, group))
    finite = y.isfinite()
    some = finite.any(-1)
    bias = torch.where(some, torch.where(finite, y, torch.inf).amin(-1), 0.0)
    top = torch.where(some, torch.where(finite, y, -torch.inf).amax(-1), 0.0)
    scale = ((top - bias) / 15).half()
    below = (scale.view(torch.int16) - 1).view(torch.float16)
    scale = torch.where(15 * scale.double() + bias >= 65520, below, scale)  # what would round to infinity
    s = scale.double()[..., None]
    code = torch.where(s > 0, (y - bias[..., None]) / torch.where(s > 0, s, 1.0), 0.0).round().clamp(0, 15)
    code = torch.where(finite, code, torch.where((y == torch.inf) & (s > 0), 15.0, 0.0))
    return code.to(torch.uint8).flatten(-2), scale, bias.half() + 0.0


def pack(code):
    return code[..., ::2] | (code[..., 1::2] << 4)


def unpack(packed):
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


def elements(packed, affine):
    """float64 [N, H, bs, D] that codes [N, H, bs, D / 2] and pairs [N, H, groups, bs, 2] stand for, rounded to fp16 once."""
    code = unpack(packed).double()
    a = affine.double().repeat_interleave(code.shape[-1] // affine.shape[2], 2).transpose(2, 3)
    with np.errstate(over="ignore", invalid="ignore"):
        return torch.from_numpy((code * a[..., 0] + a[..., 1]).numpy().astype(np.float16).astype(np.float64))


def append(x, slots, packed, affine):
    """Writes x fp16 [T, H, D] into packed codes and affine pairs in place; of rows with one slot the last counts."""
    groups, bs = affine.shape[2], packed.shape[2]
    code, scale, bias = quantize(x, x.shape[-1] // groups)
    code = pack(code)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < packed.shape[0] * bs:
            page, off = divmod(s, bs)
            packed[page, :, off] = code[t]
            affine[page, :, :, off] = torch.stack((scale[t], bias[t]), -1)


def values(slots, packed, affine):
    """float64 rows [n, H, D] of slots; zeros outside the cache."""
    rows = elements(packed, affine).transpose(1, 2).flatten(0, 1)
    ok = (slots >= 0) & (slots < rows.shape[0])
    return torch.where(ok[:, None, None], rows[slots.clamp(0, rows.shape[0] - 1).long()], 0.0)


def attention(q, k_val, v_val, tables, lens, starts, scale, heads=None):
    """q fp16 [T, Hq, D]; k_val, v_val float64 [N, Hkv, bs, D].  (out, bound), float64 [T, Hq, D]: zero where nothing is
    seen and in rows of no request; a block outside the cache has no weight; bound, how far a row computed with fp32 sums, fp16 weights and an fp16 result may be off:
      * scores: D products summed in fp32 and scaled: |dx| <= D 2^-24 sum|q k| scale + 3 * 2^-24 |x|, the exponential
        2^-22 more; so dp / p <= d = that, twice (numerator, sum)
      * a weight in the product with v: half an fp16 step, 2^-11 of itself, or 2^-25 where the largest is 2^7 at least
        (2^-32 of the largest)
      * sums of n terms over waves and parts: n 2^-24 of their magnitudes, numerator and denominator
      * the result: half an fp16 step, 2^-11, or 2^-25 for subnormals
    heads: the kv heads to compute (the others' rows stay zero)."""
    T, Hq, D = q.shape
    Hkv, bs = k_val.shape[1], k_val.shape[2]
    G = Hq // Hkv
    out, bound = (torch.zeros(T, Hq, D, dtype=torch.float64) for _ in range(2))
    for b, held in enumerate(lens.tolist()):
        lo, hi = int(starts[b]), int(starts[b + 1])
        n = hi - lo
        if not n or not held:
            continue
        ids = tables[b, :blocks(held, bs)].long()
        last = held - n + torch.arange(n)
        there = (ids >= 0) & (ids < k_val.shape[0])
        see = (torch.arange(held) <= last[:, None]) & there.repeat_interleave(bs)[:held]  # [n, held]
        for h in range(Hkv) if heads is None else heads:
            k, v = (t[torch.where(there, ids, 0), h].reshape(-1, D)[:held] for t in (k_val, v_val))
            for j in range(h * G, (h + 1) * G):
                qq = q[lo:hi, j].double()
                x = (qq @ k.T * scale).masked_fill(~see, -torch.inf)
                p = torch.softmax(x, 1).nan_to_num(0.0)
                o = p @ v
                mags = (qq.abs() @ k.abs().T * abs(scale)).masked_fill(~see, 0.0).amax(1)
                top = x.masked_fill(~see, 0.0).abs().amax(1)
                d = (D * 2.0 ** -24 * mags + 3 * 2.0 ** -24 * top + 2.0 ** -21)[:, None]
                a = p @ v.abs()
                count = (last + 1).clamp(min=0)[:, None].double()
                biggest = v.abs().amax() * p.amax(1, keepdim=True)
                out[lo:hi, j] = o
                bound[lo:hi, j] = ((2.0 ** -11 + 2 * d + count * 2.0 ** -23) * a + count * 2.0 ** -32 * biggest
                                   + 2.0 ** -11 * o.abs() + 2.0 ** -25) * (count > 0)
    return out, bound
