"""Plain 64-bit forms of the serving operators (test infrastructure only):
block assignment, 8-bit cache writes, attention over the cache, sampling.  CPU
torch and Python integers, element by element where that is clearer."""

from __future__ import annotations

import math

import torch

QMAX = {"e4m3": 448.0, "int8": 127.0}
DTYPE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
MIN_SCALE = 2.0 ** -32


def blocks(tokens: int, bs: int) -> int:
    return -(-tokens // bs)


def assign(lens, delta, tables, ring, state, bs, max_tokens):
    """gdsllm_kv_assign on Python lists; tables and ring are changed in place."""
    R, (head, count), width = len(ring), state, len(tables[0])
    slots, positions, starts = [-1] * max_tokens, [-1] * max_tokens, [0]
    out, wanted, taken, back = [], 0, 0, []
    total = 0
    old = [list(row) for row in tables]
    for r, (n, d) in enumerate(zip(lens, delta)):
        add, drop = max(d, 0), min(max(-d, 0), n)
        t0 = total
        total += add
        starts.append(min(total, max_tokens))
        fits = add == 0 or (blocks(n + add, bs) <= width and total <= max_tokens)
        need = blocks(n + add, bs) - blocks(n, bs) if fits else 0
        wanted += need
        served = fits and (need == 0 or wanted <= count)
        if served:
            for j in range(need):
                tables[r][blocks(n, bs) + j] = ring[(head + wanted - need + j) % R]
            taken += need
            for i in range(add):
                slots[t0 + i] = tables[r][(n + i) // bs] * bs + (n + i) % bs
                positions[t0 + i] = n + i
        back += old[r][blocks(n - drop, bs):blocks(n, bs)] if drop else []
        out.append(n + add - drop if served else n)
    for i, b in enumerate(back):
        ring[(head + count + i) % R] = b
    return slots, positions, starts, out, [(head + taken) % R, count - taken + len(back)]


def codes64(x: torch.Tensor, fmt: str) -> torch.Tensor:
    """The nearest 8-bit value (ties to the even code), float64; NaN as kv_append stores it."""
    if fmt == "int8":
        return torch.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0).clamp(-127, 127).round()
    y = torch.nan_to_num(x, nan=math.nan, posinf=448.0, neginf=-448.0).clamp(-448, 448)
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(y / step) * step


def want_scale(amax: float, fmt: str) -> float:
    """Smallest power of two s >= 2^-32 with amax <= QMAX * s."""
    s = MIN_SCALE
    while amax > QMAX[fmt] * s:
        s *= 2
    return s


def rotate(x, positions, cos, sin):
    """fp16 [T, H, D] -> the values kv_append writes (fp16, through fp32), and the 64-bit ones."""
    half = cos.shape[1]
    c, s = (t.double()[positions.clamp(0, cos.shape[0] - 1).long()][:, None, :] for t in (cos, sin))
    a, b = x[..., :half].double(), x[..., half:2 * half].double()
    y = torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:].double()], -1)
    return y.float().half(), y


def append(x, slots, cache, scale, fmt):
    """Writes x fp16 [T, H, D] into cache (float64 code values [N, H, bs, D]) and scale (float64 [N, H]) in place."""
    bs, H = cache.shape[2], cache.shape[1]
    rows: dict = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < cache.shape[0] * bs:
            rows.setdefault(s // bs, []).append((s % bs, t))
    for page, ot in rows.items():
        low = min(o for o, _ in ot)
        for h in range(H):
            v = torch.stack([x[t, h] for _, t in ot]).double()
            fin = v[v.isfinite()]
            now = want_scale(float(fin.abs().max()) if fin.numel() else 0.0, fmt)
            if low > 0:
                was = float(scale[page, h])
                now = max(now, was)
                if now != was:
                    cache[page, h, :low] = codes64(cache[page, h, :low] * (was / now), fmt)
            for o, t in ot:
                cache[page, h, o] = codes64(x[t, h].double() / now, fmt)
            scale[page, h] = now


def attention(q, k_val, v_val, v_scale, tables, lens, starts, scale):
    """q fp16 [T, Hq, D]; k_val, v_val float64 values (scale * code) [N, Hkv, bs, D]; v_scale [N, Hkv].  Returns (out,
    bound): float64 rows [T, Hq, D] (zero where nothing is seen; rows behind the last request too) and how far a row
    computed with fp32 sums, fp16 weights and an fp16 result may be from it:
      * scores: D products summed in fp32, scaled and shifted by a maximum: |dx| <= D 2^-24 sum|q k| scale + 3 * 2^-24 |x|
        (times ln 2 and log2 e, which cancel), the exponential 2^-22 more; so dp/p <= d = that, twice (numerator, sum)
      * weights: half an fp16 step, 2^-11 relative, or 2^-25 of the largest weight (of any row value 448 * v_scale)
      * accumulation of n terms over at most 4 waves and the units: n 2^-24 relative
      * the result: half an fp16 step, or 2^-25 for subnormals."""
    T, Hq, D = q.shape
    N, Hkv, bs, _ = k_val.shape
    G = Hq // Hkv
    out, bound = torch.zeros(T, Hq, D, dtype=torch.float64), torch.full((T, Hq, D), 0.0, dtype=torch.float64)
    for b, n_held in enumerate(lens.tolist()):
        lo, hi = int(starts[b]), int(starts[b + 1])
        n = hi - lo
        ids = tables[b, :blocks(n_held, bs)].long()
        for i in range(n):
            seen = n_held - n + i + 1
            if seen <= 0:
                continue
            for h in range(Hq):
                k = k_val[ids, h // G].reshape(-1, D)[:seen]
                v = v_val[ids, h // G].reshape(-1, D)[:seen]
                vs = v_scale[ids, h // G].repeat_interleave(bs)[:seen]
                qq = q[lo + i, h].double()
                x = (k @ qq) * scale
                mags = (k.abs() @ qq.abs()) * abs(scale)
                p = torch.softmax(x, 0)
                o = p @ v
                out[lo + i, h] = o
                d = D * 2.0 ** -24 * float(mags.max()) + 3 * 2.0 ** -24 * float(x.abs().max()) + 2.0 ** -21
                a = p @ v.abs()
                top = float(vs[torch.argmax(x + torch.log(vs.clamp(min=2.0 ** -64)))])
                bound[lo + i, h] = ((2.0 ** -11 + 2 * d + seen * 2.0 ** -23) * a + seen * 2.0 ** -25 * 448.0 * top
                                    + 2.0 ** -11 * o.abs() + 2.0 ** -25)
    return out, bound


def sample_row(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row of gdsllm_sample_tokens.  Returns (token, border): border is how near (relative to the kept mass) a
    cut or the draw came to going the other way; masses are exactly rounded sums."""
    x = logits.double()
    x = torch.where(x.isnan(), torch.tensor(-math.inf, dtype=torch.float64), x)
    value, index = torch.sort(x, descending=True, stable=True)
    live = int((value > -math.inf).sum())
    if not live:
        return -1, 1.0
    if not temperature > 0:
        return int(index[0]), 1.0
    value, index = value[:live].tolist(), index[:live].tolist()
    w = [1.0 if v == value[0] else 0.0 if value[0] == math.inf else math.exp((v - value[0]) / temperature) for v in value]
    n, border = live, 1.0
    if 0 < top_k < n:
        n = top_k
    mass = math.fsum(w[:n])
    cut = n
    if top_p < 1:
        run = 0.0
        cut = 0
        for j in range(n):
            if j and not run < max(top_p, 0.0) * mass:
                break
            cut = j + 1
            run = math.fsum((run, w[j]))
            border = min(border, abs(run - top_p * mass) / mass)
    while cut > 1 and w[cut - 1] < min_p:
        cut -= 1
    kept = math.fsum(w[:cut])
    uu = min(max(u, 0.0), 1.0)
    run = 0.0
    for j in range(cut):
        run = math.fsum((run, w[j]))
        border = min(border, abs(run - uu * kept) / kept) if run < kept else border
        if run > uu * kept:
            return index[j], border
    return index[cut - 1], border
