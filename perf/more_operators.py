"""What the operators of a 4-bit KV cache are timed on.

`rope` rotates q and k by their positions, pairs of neighbouring channels
(2i, 2i + 1) or of halves (i, i + rotary / 2); `kv4_append` rotates and writes a
step's keys and values into a paged cache of 4-bit codes; `kv4_attention`
attends over it; `kv4_values` reads rows of it back.  Head counts and widths are
those of the LLaMA-7B (32 query and 32 key heads of 128), LLaMA-70B (64 and 8 of
128) and Qwen-MoE (32 and 2 of 256) layers.

The cache holds, for each token, head and group of channels, a scale and a bias
in fp16 and codes 0 .. 15; an element is fp16(code * scale + bias).  The bias is
the group's smallest finite value, the scale a 15th of its finite range rounded
to fp16 (the next smaller fp16 value where 15 * scale + bias would leave fp16),
the code round((x - bias) / scale), ties to even, NaN as the smallest value.

Where `own` is false every operator is computed in elementary torch operations
in 32 bits (64 for rotary angles, scales and codes, which lie next to a
border), rounded once; where it is true, by the framework's kernels.
"""

import math

import torch

own = False

_PHI = 0.6180339887498949


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # A decode batch whose checkpoint pairs halves: latency counts.
        dict(name="rope_decode_64", kind="rope", tokens=64, heads=64, kv_heads=8, dim=128, rotary=128, pairs=0, pad=0),
        # A prompt of no round length whose checkpoint pairs neighbouring channels.
        dict(name="rope_prompt_4001_pairs", kind="rope", tokens=4001, heads=32, kv_heads=32, dim=128, rotary=128,
             pairs=1, pad=7),
        # 32 sequences decoded together over a grouped-query layer: one token each, into blocks half full.
        dict(name="append4_decode_32x8", kind="append", group=64, requests=32, new=1, held=1000, heads=64, kv_heads=8,
             dim=128, block=64, rotary=128, pairs=0, pad=0),
        # Prompts of no round length into the small blocks of a multi-head layer, neighbouring channels paired.
        dict(name="append4_prompt_2x1000_pairs", kind="append", group=32, requests=2, new=1000, held=37, heads=32,
             kv_heads=32, dim=128, block=16, rotary=128, pairs=1, pad=3),
        # A long prompt, wide heads of which a quarter is rotated.
        dict(name="append4_prompt_8192", kind="append", group=128, requests=1, new=8192, held=0, heads=32, kv_heads=2,
             dim=256, block=128, rotary=64, pairs=0, pad=0),
        # A conversation handed to another server.
        dict(name="values4_777x8", kind="values", group=64, tokens=777, kv_heads=8, dim=128, block=64),
        # A long one of a multi-head layer.
        dict(name="values4_8192x32", kind="values", group=32, tokens=8192, kv_heads=32, dim=128, block=32),
        # A single conversation of some hundred tokens, every head with its own keys: latency counts.
        dict(name="attend4_decode_1x777", kind="attend", group=32, requests=1, new=1, longest=777, heads=32,
             kv_heads=32, dim=128, block=16),
        # A ragged decode batch over a grouped-query layer, an idle request among them.
        dict(name="attend4_decode_32x8192", kind="attend", group=64, requests=32, new=1, longest=8192, heads=64,
             kv_heads=8, dim=128, block=64),
        # One very long sequence over two wide key heads: the work is split along it.
        dict(name="attend4_decode_1x131072", kind="attend", group=128, requests=1, new=1, longest=131072, heads=32,
             kv_heads=2, dim=256, block=128),
        # Prompt chunks of several requests behind what their caches hold.
        dict(name="attend4_chunk_4x300", kind="attend", group=64, requests=4, new=300, longest=5000, heads=64,
             kv_heads=8, dim=128, block=32),
        # A whole prompt at once, every head with its own keys: bound by the matrix cores.
        dict(name="attend4_prompt_4096", kind="attend", group=64, requests=1, new=4096, longest=4096, heads=32,
             kv_heads=32, dim=128, block=64),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _drawn(rng):
    kind = rng.choice(["rope", "append", "append", "values", "attend", "attend", "attend"])
    kv = rng.choice([1, 2, 4, 5, 8, 32])
    dim = rng.choice([64, 128, 128, 256])
    heads = kv * rng.choice([1, 2, 4, 7, 8, 16])
    pairs, pad = rng.choice([0, 1]), rng.choice([0, 0, 1, 13])
    if kind == "rope":
        # wider choices of heads, and parts of a head of no round size, than the cache takes
        dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
        return dict(kind=kind, tokens=_log_int(rng, 1, 8000), heads=heads, kv_heads=kv, dim=dim,
                    rotary=rng.choice([dim, dim, dim // 2, dim // 4]), pairs=pairs, pad=pad)
    group = rng.choice([g for g in (32, 64, 128) if g <= dim])
    block = rng.choice([16, 32, 64, 128, 256])
    if kind == "values":
        return dict(kind=kind, group=group, tokens=_log_int(rng, 1, 20000), kv_heads=kv, dim=dim, block=block)
    case = dict(kind=kind, group=group, requests=_log_int(rng, 1, 64), new=rng.choice([1, 1, 2, 5, _log_int(rng, 3, 2100)]),
                heads=heads, kv_heads=kv, dim=dim, block=block)
    if kind == "append":
        return dict(case, held=_log_int(rng, 1, 2000) - 1, rotary=rng.choice([0, dim // 2, dim]), pairs=pairs, pad=pad)
    return dict(case, longest=max(case["new"], _log_int(rng, 1, 40000)))


def draw(rng):
    most = [max(work(c)[k] for c in listed()) for k in ("bytes", "flops")]
    while True:
        case = _drawn(rng)
        w = work(case)
        plain = 0
        if case["kind"] == "attend":
            plain = case["requests"] * case["heads"] * case["new"] * case["longest"]
        if w["bytes"] <= most[0] and w["flops"] <= most[1] and plain <= 2 ** 30:
            return case


# ------------------------------------------------- sizes that a case stands for

def _spread(n, lo, hi, shift=0.0):
    """n whole numbers in [lo, hi], spread evenly in no order, the first at `hi`."""
    return [hi - int((hi - lo) * ((i * _PHI + (shift if i else 0.0)) % 1.0)) for i in range(n)]


def _lengths(case):
    """(tokens held after this step's, tokens new in it) of each request of an append or attend case."""
    n = case["requests"]
    if case["new"] == 1:
        new = [1] * n
    else:
        new = _spread(n, max(1, case["new"] // 3), case["new"])
    if case["kind"] == "append":
        return [h + t for h, t in zip(_spread(n, case["held"] // 2, case["held"]), new)], new
    total = [max(a, t) for a, t in zip(_spread(n, max(1, case["longest"] // 16), case["longest"], 0.37), new)]
    if n >= 8:  # a slot of the batch that nobody uses
        total[n // 2], new[n // 2] = 0, 0
    return total, new


def _blocks(tokens, block):
    return -(-tokens // block)


# ------------------------------------------------- inputs, from the seed alone

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, g, std=1.0):
    return torch.randn(shape, dtype=torch.float32, device="cuda", generator=g) * std


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _heads(tokens, heads, dim, g):
    """Keys of a layer: a few channels of every head much larger than the others, all of them off zero."""
    x = _normal((tokens, heads, dim), g)
    gain = torch.exp(_normal((heads, dim), g, 0.6))
    return ((x + _normal((heads, dim), g, 0.5)) * gain).half()


def _cache(case, pool, g):
    """A filled cache: packed codes [pool, heads, block, dim / 2], affine [pool, heads, groups, block, 2]."""
    x = _normal((pool, case["kv_heads"], case["block"], case["dim"]), g)
    x = x * torch.exp(_normal((1, case["kv_heads"], 1, case["dim"]), g, 0.4))
    x = x.half().unflatten(-1, (-1, case["group"]))
    bias, top = x.amin(-1), x.amax(-1)
    scale = ((top.float() - bias.float()) / 15).half()
    code = ((x.float() - bias.float()[..., None]) / scale.float().clamp(min=1e-8)[..., None]).round().clamp(0, 15)
    code = code.to(torch.uint8).flatten(-2)
    return code[..., ::2] | (code[..., 1::2] << 4), torch.stack((scale, bias), -1).transpose(2, 3).contiguous()


def _tables(case, totals, g):
    """Block tables over a pool in no order, and the pool's size."""
    bs = case["block"]
    counts = [_blocks(t, bs) for t in totals]
    width, pool = max(1, max(counts)), sum(counts) + 3
    ids = torch.randperm(pool, device="cuda", generator=g).to(torch.int32)
    rows = torch.arange(width, device="cuda") < _ints(counts)[:, None]
    tables = torch.zeros(len(totals), width, dtype=torch.int32, device="cuda")
    tables[rows] = ids[:sum(counts)]
    return tables, pool


def _angles(positions, rotary):
    """cos and sin of position * frequency, as a model's program holds them."""
    half = rotary // 2
    at = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None]
    angle = at * 500000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    return {"cos": angle.cos().float(), "sin": angle.sin().float()}


def _inputs(case, seed):
    """Inputs by name; the same for both sides and for the 64-bit one."""
    g, kind = _gen(seed), case["kind"]
    hk, d = case["kv_heads"], case["dim"]
    if kind == "rope":
        n, pad = case["tokens"], case["pad"]
        # q and k as they leave one projection: heads of one packed row
        row = _heads(n + pad, case["heads"] + 2 * hk, d, g)
        pos = torch.randint(0, 9000, (n + pad,), dtype=torch.int32, device="cuda", generator=g)
        pos[n:] = -1
        return {"q": row[:, :case["heads"]], "k": row[:, case["heads"]:case["heads"] + hk], "positions": pos,
                **_angles(9000, case["rotary"])}
    if kind == "values":
        n, bs = case["tokens"], case["block"]
        tables, pool = _tables(case, [n], g)
        (kc, ka), (vc, va) = _cache(case, pool, g), _cache(case, pool, g)
        i = torch.arange(n, device="cuda")
        slots = tables[0][i // bs].long() * bs + i % bs
        return {"k_cache": kc, "k_affine": ka, "v_cache": vc, "v_affine": va, "slots": slots.int()}
    totals, new = _lengths(case)
    tables, pool = _tables(case, totals, g)
    starts = _ints([0] + new).cumsum(0, dtype=torch.int32)
    rows, pad = sum(new), case.get("pad", 0)
    (kc, ka), (vc, va) = _cache(case, pool, g), _cache(case, pool, g)
    got = {"k_cache": kc, "k_affine": ka, "v_cache": vc, "v_affine": va}
    q = _normal((rows + pad, case["heads"], d), g, 1.5).half()
    if kind == "attend":
        return dict(got, q=q, scale=d ** -0.5, tables=tables, lens=_ints(totals), starts=starts, block=case["block"],
                    new=max(new), longest=max(totals))
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), _ints(new).long())
    pos = (_ints(totals) - _ints(new))[seq] + torch.arange(rows, device="cuda") - starts[seq]
    slot = tables[seq, (pos // case["block"]).long()] * case["block"] + pos % case["block"]
    none = torch.full((pad,), -1, dtype=torch.int32, device="cuda")
    got |= {"k": _heads(rows + pad, hk, d, g), "v": _heads(rows + pad, hk, d, g), "q": q,
            "slots": torch.cat([slot.int(), none]), "positions": torch.cat([pos.int(), none]), "cos": None, "sin": None}
    if case["rotary"]:
        got |= _angles(max(totals), case["rotary"])
    return got


def prepare(case, seed):
    return dict(_inputs(case, seed), kind=case["kind"], pairs=bool(case.get("pairs", 0)))


# ------------------------------------------------------------ plain forms

def _rotate(x, s):
    """Pairs of the first channels turned by the position's angle, one rounding; zeros where there is no position."""
    if s["cos"] is None:
        return x
    live = (s["positions"] >= 0)[:, None, None]
    at = s["positions"].long().clamp(min=0)
    c, n = (t[at].double()[:, None, :] for t in (s["cos"], s["sin"]))
    half = c.shape[-1]
    turned = x[..., :2 * half].double()
    if s["pairs"]:
        a, b = turned[..., ::2], turned[..., 1::2]
        y = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        y = torch.cat([a * c - b * n, b * c + a * n], -1)
    return torch.where(live, torch.cat([y.half(), x[..., 2 * half:]], -1), 0.0)


def _rope(s):
    return {"q": _rotate(s["q"], s), "k": _rotate(s["k"], s)}


def _element(code, affine):
    """code * scale + bias, rounded to fp16; code [..., groups, channels], affine [..., groups, 2]."""
    return (code.float() * affine[..., :1].float() + affine[..., 1:].float()).half()


def _unpack(codes, groups):
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (groups, -1))


def _read(cache, affine, slots):
    """fp16 rows [n, heads, dim] of slots [n]; zeros for slots below 0."""
    groups, bs = affine.shape[2], affine.shape[3]
    page, off = slots.long().clamp(min=0) // bs, slots.long().clamp(min=0) % bs
    x = _element(_unpack(cache[page, :, off], groups), affine[page, :, :, off])
    return torch.where((slots >= 0)[:, None, None], x.flatten(-2), 0.0)


def _values(s):
    return {c: _read(s[c + "_cache"], s[c + "_affine"], s["slots"]) for c in "kv"}


def _write(x, cache, affine, slots):
    """x fp16 [n, heads, dim] into the cache's slots, each token and group for itself."""
    live = slots >= 0
    x, slots = x[live], slots[live].long()
    groups, bs = affine.shape[2], affine.shape[3]
    x = x.unflatten(-1, (groups, -1)).double()
    bias, top = x.amin(-1), x.amax(-1)  # what the cases hold is finite
    scale = ((top - bias) / 15).half()
    lower = (scale.view(torch.int16) - 1).view(torch.float16)
    scale = torch.where(15 * scale.double() + bias >= 65520.0, lower, scale)
    step = scale.double()[..., None]
    code = torch.where(step > 0, (x - bias[..., None]) / step, 0.0).round().clamp(0, 15).to(torch.uint8).flatten(-2)
    page, off = slots // bs, slots % bs
    cache[page, :, off] = code[..., ::2] | (code[..., 1::2] << 4)
    affine[page, :, :, off] = torch.stack((scale, bias.half()), -1)


def _append(s):
    _write(_rotate(s["k"], s), s["k_cache"], s["k_affine"], s["slots"])
    _write(s["v"], s["v_cache"], s["v_affine"], s["slots"])
    # what the cache holds of the step's tokens: the values that its codes stand for
    out = _values(s)
    return out if s["cos"] is None else dict(out, q=_rotate(s["q"], s))


def _rows_of(s):
    """Token rows as a padded batch: (row of each [request, i], whether it is there)."""
    new = s["starts"].diff()
    i = torch.arange(s["new"], device=new.device)
    there = i < new[:, None]
    return torch.where(there, s["starts"][:-1, None] + i, 0).long(), there


def _attend(s):
    q, bs, d = s["q"].float(), s["block"], s["q"].shape[-1]
    row, there = _rows_of(s)
    pages = s["tables"][:, :_blocks(s["longest"], bs)].long()
    n, width, hk = pages.shape[0], pages.shape[1], s["k_cache"].shape[1]

    def held(cache, affine):  # [n, Hkv, tokens, D]
        x = _element(_unpack(cache, affine.shape[2]), affine.transpose(2, 3)).flatten(-2)[pages].float()
        return x.transpose(1, 2).reshape(n, hk, width * bs, d)

    group, m = q.shape[1] // hk, s["new"]
    qb = q[row].view(n, m, hk, group, d).permute(0, 2, 1, 3, 4).reshape(n, hk, m * group, d)
    k = held(s["k_cache"], s["k_affine"])
    sc = torch.matmul(qb * s["scale"], k.transpose(2, 3).contiguous()).view(n, hk, m, group, width * bs)
    del k
    last = s["lens"].long()[:, None] - there.sum(1, keepdim=True) + torch.arange(m, device=q.device)
    seen = torch.arange(width * bs, device=q.device) <= last[..., None]
    sc = sc.masked_fill(~seen[:, None, :, None, :], float("-inf"))
    p = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-3e38))
    del sc
    v = held(s["v_cache"], s["v_affine"]).masked_fill(
        (torch.arange(width * bs, device=q.device) >= s["lens"][:, None])[:, None, :, None], 0.0)
    o = torch.matmul(p.reshape(n, hk, m * group, width * bs), v)
    o = o / p.sum(-1).view(n, hk, m * group, 1).clamp(min=1e-30)
    o = o.view(n, hk, m, group, d).permute(0, 2, 1, 3, 4).reshape(n, m, hk * group, d)
    out = torch.zeros_like(s["q"])
    out[row[there]] = o[there].half()
    return out


_PLAIN = {"rope": _rope, "append": _append, "values": _values, "attend": _attend}


# ------------------------------------------------------------ the framework's side

def _own(s):
    from gdsllm_amd.runtime import ext

    if s["kind"] == "rope":
        q, k = ext().rope(s["q"], s["k"], s["positions"], s["cos"], s["sin"], s["pairs"])
        return {"q": q, "k": k}
    cache = (s["k_cache"], s["v_cache"], s["k_affine"], s["v_affine"])
    if s["kind"] == "attend":
        return ext().kv4_attention(s["q"], *cache, s["tables"], s["lens"], s["starts"], s["scale"], s["new"],
                                   s["longest"])
    out = {}
    if s["kind"] == "append":
        turns = s["cos"] is not None
        q = ext().kv4_append(s["k"], s["v"], s["slots"], *cache, s["q"] if turns else None, s["positions"], s["cos"],
                             s["sin"], s["pairs"])
        out = {"q": q} if turns else {}
    k, v = ext().kv4_values(s["slots"], *cache)
    return {"k": k, "v": v, **out}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["kind"]](state)


# ------------------------------------------------------------ what a pass needs

def work(case):
    kind, hk, d = case["kind"], case["kv_heads"], case["dim"]
    if kind == "rope":
        t, h = case["tokens"], case["heads"] + hk
        return {"bytes": 4 * t * h * d + 2 * case["pad"] * h * d + 4 * t + 4 * case["rotary"] * min(t, 9000),
                "flops": 3 * t * h * case["rotary"]}
    held = d + 8 * d // case["group"]  # bytes of a token's keys and values in one head
    if kind == "values":
        t = case["tokens"]
        return {"bytes": t * hk * (held + 4 * d) + 4 * t, "flops": 4 * t * hk * d}
    totals, new = _lengths(case)
    h, bs = case["heads"], case["block"]
    if kind == "append":
        t = sum(new)
        by = t * hk * (4 * d + held + 4 * d) + 4 * t  # and the values that the written codes stand for
        if case["rotary"]:
            by += 4 * t * h * d + 4 * t + 4 * case["rotary"] * min(t, max(totals))
        return {"bytes": by, "flops": t * d * (20 * hk + 3 * h)}
    by = sum(a * hk * held + 4 * _blocks(a, bs) for a in totals) + 4 * sum(new) * h * d
    pairs = sum(b * (a - b) + b * (b + 1) // 2 for a, b in zip(totals, new))
    return {"bytes": by, "flops": 4 * pairs * h * d}


# --------------------------------------------------------- the same in 64 bits

def _round16(x):
    """The fp16 value nearest to a float64 one (ties to even), as float64: 10 bits behind the leading one."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -14)))
    step = torch.exp2(e - 10)
    return torch.round(x / step) * step


def _turned64(x, name, pairs):
    y = x[name].double()
    if x["cos"] is None:
        return y
    half = x["cos"].shape[1]
    at = x["positions"].long().clamp(min=0)
    w = torch.complex(*(x[t].double()[at].unsqueeze(1) for t in ("cos", "sin")))
    if pairs:
        z = torch.view_as_complex(y[..., :2 * half].unflatten(-1, (-1, 2)).contiguous()) * w
        y = torch.cat([torch.view_as_real(z).flatten(-2), y[..., 2 * half:]], -1)
    else:
        z = torch.complex(y[..., :half], y[..., half:2 * half]) * w
        y = torch.cat([z.real, z.imag, y[..., 2 * half:]], -1)
    return y * (x["positions"] >= 0)[:, None, None]


def _held64(x, name, group):
    """Every element of a cache, float64 [pool, heads, block, dim]."""
    byte = x[name + "_cache"].long()
    n, h, bs, half = byte.shape
    code = torch.empty(n, h, bs, 2 * half, dtype=torch.float64, device=byte.device)
    code[..., 0::2] = (byte % 16).double()
    code[..., 1::2] = (byte // 16).double()
    a = x[name + "_affine"].double().repeat_interleave(group, 2).transpose(2, 3)
    return _round16(code * a[..., 0] + a[..., 1])


def exact(case, seed):
    x, kind = _inputs(case, seed), case["kind"]

    if kind == "rope":
        return {name: _turned64(x, name, case["pairs"]) for name in "qk"}

    if kind == "values":
        out = {}
        for c in "kv":
            rows = _held64(x, c, case["group"]).transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])
            out[c] = rows[x["slots"].long()]
        return out

    if kind == "append":
        out = {"q": _turned64(x, "q", case["pairs"])} if case["rotary"] else {}
        live = (x["slots"] >= 0)[:, None, None].double()
        for c, y in (("k", _round16(_turned64(x, "k", case["pairs"]))), ("v", x["v"].double())):
            y = y.view(*y.shape[:2], -1, case["group"])
            low, high = y.min(3, keepdim=True).values, y.max(3, keepdim=True).values
            s = _round16((high - low) / 15)
            n = torch.where(s > 0, torch.round((y - low) / s.clamp(min=2.0 ** -24)), 0.0).clamp(0, 15)
            out[c] = (n * s + low).flatten(2) * live
        return out

    hk, bs, d = case["kv_heads"], case["block"], case["dim"]
    q, out = x["q"].double(), torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    starts, lens = x["starts"].tolist(), x["lens"].tolist()
    keys, vals = _held64(x, "k", case["group"]), _held64(x, "v", case["group"])
    for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
        n, held = hi - lo, lens[b]
        if not n or not held:
            continue
        ids = x["tables"][b, :_blocks(held, bs)].long()
        k, v = (t[ids].transpose(0, 1).reshape(hk, -1, d)[:, :held] for t in (keys, vals))
        for h in range(hk):
            group = case["heads"] // hk
            for r in range(0, n, 1024):
                m = min(1024, n - r)
                qs = q[lo + r:lo + r + m, h * group:(h + 1) * group].transpose(0, 1)  # [group, m, d]
                s = qs @ k[h].t().contiguous() * x["scale"]
                last = held - n + r + torch.arange(m, device="cuda")
                s.masked_fill_(torch.arange(held, device="cuda") > last[:, None], float("-inf"))
                p = torch.softmax(s, -1).nan_to_num(0.0)
                out[lo + r:lo + r + m, h * group:(h + 1) * group] = (p @ v[h]).transpose(0, 1)
    return out
