"""What the operators around a decode step's projections are timed on.

Between the q/k/v projections and o_proj a serving step gives each request
its cache blocks (`kv_assign`), rotates q and k and writes k and v into the
8-bit cache (`kv_append`), and attends over it (`kv_attention`); after lm_head
it draws the next tokens (`sample_tokens`).  Head counts and widths are those of
the LLaMA-7B (32 query and 32 key heads of 128), LLaMA-70B (64 and 8 of 128) and
Qwen-MoE (32 and 2 of 256) layers, vocabularies 32000 and larger.

Where `own` is false every operator is computed in elementary torch operations
in 32 bits (64 for rotary angles, softmax weights of the sampler and their
running sums), rounded once; where it is true, by the framework's kernels.
"""

import math

import torch

own = False

_PHI = 0.6180339887498949
_QMAX = {"e4m3": 448.0, "int8": 127.0}
_CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_MIN_SCALE = 2.0 ** -32


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One step of a small batch of decoding requests: most add one token, a few end.
        dict(name="assign_decode_64", kind="assign", requests=64, block=16, longest=4096, prompts=0, prompt=0),
        # A large server's step: decoding requests, ended ones, and new prompts of up to 1024 tokens.
        dict(name="assign_mixed_2048", kind="assign", requests=2048, block=64, longest=8192, prompts=128,
             prompt=1024),
        # 32 sequences decoded together over a grouped-query layer: one token each, into blocks half full.
        dict(name="append_decode_32x8", kind="append", codes="e4m3", requests=32, new=1, held=1000, heads=64,
             kv_heads=8, dim=128, block=64, rotary=128),
        # Prompts of no round length into the small blocks of a multi-head layer.
        dict(name="append_prompt_2x1000", kind="append", codes="e4m3", requests=2, new=1000, held=37, heads=32,
             kv_heads=32, dim=128, block=16, rotary=128),
        # A long prompt in int8, wide heads of which a quarter is rotated.
        dict(name="append_prompt_8192_int8", kind="append", codes="int8", requests=1, new=8192, held=0, heads=32,
             kv_heads=2, dim=256, block=128, rotary=64),
        # A single conversation of some hundred tokens, every head with its own keys: latency counts.
        dict(name="attend_decode_1x777", kind="attend", codes="e4m3", requests=1, new=1, longest=777, heads=32,
             kv_heads=32, dim=128, block=16),
        # A ragged decode batch over a grouped-query layer, an idle request among them.
        dict(name="attend_decode_32x8192", kind="attend", codes="e4m3", requests=32, new=1, longest=8192, heads=64,
             kv_heads=8, dim=128, block=64),
        # One very long sequence over two wide key heads: the work is split along it.
        dict(name="attend_decode_1x131072", kind="attend", codes="int8", requests=1, new=1, longest=131072,
             heads=32, kv_heads=2, dim=256, block=128),
        # Prompt chunks of several requests behind what their caches hold.
        dict(name="attend_chunk_4x300", kind="attend", codes="int8", requests=4, new=300, longest=5000, heads=64,
             kv_heads=8, dim=128, block=32),
        # A whole prompt at once, every head with its own keys: bound by the matrix cores.
        dict(name="attend_prompt_4096", kind="attend", codes="e4m3", requests=1, new=4096, longest=4096, heads=32,
             kv_heads=32, dim=128, block=64),
        # The next token of one conversation.
        dict(name="sample_1x32000", kind="sample", rows=1, vocab=32000, bits=16, greedy=0),
        # A decode batch over a large vocabulary of no round size.
        dict(name="sample_64x128257", kind="sample", rows=64, vocab=128257, bits=16, greedy=1),
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def _drawn(rng):
    kind = rng.choice(["assign", "append", "append", "attend", "attend", "attend", "sample", "sample"])
    if kind == "assign":
        n = _log_int(rng, 1, 4096)
        return dict(kind=kind, requests=n, block=rng.choice([16, 32, 64, 128]), longest=_log_int(rng, 100, 8192),
                    prompts=rng.randint(0, min(n, 64)), prompt=_log_int(rng, 1, 1500))
    if kind == "sample":
        return dict(kind=kind, rows=_log_int(rng, 1, 128), vocab=_log_int(rng, 1000, 200003),
                    bits=rng.choice([16, 16, 32]), greedy=rng.choice([0, 0, 1]))
    kv = rng.choice([1, 2, 4, 5, 8, 32])
    dim = rng.choice([64, 128, 128, 256])
    group = rng.choice([1, 2, 4, 7, 8, 16])
    case = dict(kind=kind, codes=rng.choice(["e4m3", "int8"]), requests=_log_int(rng, 1, 64),
                new=rng.choice([1, 1, 2, 5, _log_int(rng, 3, 2100)]), heads=kv * group, kv_heads=kv, dim=dim,
                block=rng.choice([16, 32, 64, 128]))
    if kind == "append":
        return dict(case, held=_log_int(rng, 1, 2000) - 1, rotary=rng.choice([0, dim // 2, dim]))
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


def _deltas(case):
    """(tokens held, change) of each request of an assign case."""
    n = case["requests"]
    held = _spread(n, 0, case["longest"], 0.21)
    every = max(1, n // max(1, case["prompts"]))
    sizes = dict(zip(range(0, n, every), _spread(case["prompts"], 1, case["prompt"])))
    held = [0 if i in sizes else h for i, h in enumerate(held)]

    def change(i):
        if i in sizes:
            return sizes[i]  # a new prompt
        if i % 16 == 3:
            return -held[i]  # ended
        if i % 16 == 7:
            return 0  # idle
        if i % 32 == 11:
            return -min(5, held[i])  # takes back a few tokens that it had guessed
        return 1

    return held, [change(i) for i in range(n)]


def _blocks(tokens, block):
    return -(-tokens // block)


# ------------------------------------------------- inputs, from the seed alone

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, g, std=1.0):
    return torch.randn(shape, dtype=torch.float32, device="cuda", generator=g) * std


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


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


def _heads(tokens, heads, dim, g):
    """Keys of a layer: a few channels of every head much larger than the others."""
    x = _normal((tokens, heads, dim), g)
    gain = torch.exp(_normal((heads, dim), g, 0.6))
    return (x * gain).half()


def _cache(case, pool, g):
    """A filled cache: codes with a power-of-two scale for each block and head."""
    shape = (pool, case["kv_heads"], case["block"], case["dim"])
    x = _normal(shape, g) * torch.exp(_normal((1, case["kv_heads"], 1, case["dim"]), g, 0.4))
    s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / _QMAX[case["codes"]])))
    x = x / s[:, :, None, None]
    return (x if case["codes"] == "e4m3" else x.round()).to(_CODES[case["codes"]]), s


def _inputs(case, seed):
    """Inputs by name; the same for both sides and for the 64-bit one."""
    g, kind = _gen(seed), case["kind"]
    if kind == "sample":
        n, v = case["rows"], case["vocab"]
        # a peaked head over a long tail, as a language model's logits are
        x = _normal((n, v), g, 2.0) + 9.0 * torch.rand((n, v), device="cuda", generator=g) ** 24
        x = x.to(torch.float16 if case["bits"] == 16 else torch.float32)
        some = torch.arange(n, device="cuda")
        temperature = 0.6 + 0.1 * (some % 5).float()
        if case["greedy"]:
            temperature[some % 8 == 5] = 0.0
        return {"logits": x, "u": torch.rand(n, device="cuda", generator=g), "temperature": temperature,
                "top_k": _ints([(50, 0, 200, 1000, 40)[i % 5] for i in range(n)]),
                "top_p": torch.where(some % 3 == 1, 1.0, 0.8 + 0.05 * (some % 4)).float(),
                "min_p": torch.where(some % 2 == 1, 0.02, 0.0).float()}
    if kind == "assign":
        held, delta = _deltas(case)
        bs = case["block"]
        need = sum(_blocks(h + max(d, 0), bs) for h, d in zip(held, delta))
        tables, _ = _tables(case, held, g)
        width = max(_blocks(h + max(d, 0), bs) for h, d in zip(held, delta)) + 1
        wide = torch.zeros(len(held), max(width, tables.shape[1]), dtype=torch.int32, device="cuda")
        wide[:, :tables.shape[1]] = tables
        used = sum(_blocks(h, bs) for h in held)
        pool = used + 3 + 2 * (need - used) + 64
        ring = torch.zeros(pool, dtype=torch.int32, device="cuda")
        head = int(torch.randint(0, pool, (1,), device="cuda", generator=g))
        spare = torch.arange(used + 3, pool, dtype=torch.int32, device="cuda")
        at = (head + torch.arange(spare.numel(), device="cuda")) % pool
        ring[at] = spare[torch.randperm(spare.numel(), device="cuda", generator=g)]
        tokens = sum(max(d, 0) for d in delta)
        return {"lens": _ints(held), "delta": _ints(delta), "tables": wide, "ring": ring,
                "state": _ints([head, spare.numel()]), "block": bs, "rows": -(-max(1, tokens) // 64) * 64}
    totals, new = _lengths(case)
    tables, pool = _tables(case, totals, g)
    starts = _ints([0] + new).cumsum(0, dtype=torch.int32)
    rows = sum(new)
    (kc, ks), (vc, vs) = _cache(case, pool, g), _cache(case, pool, g)
    got = {"k_cache": kc, "k_scale": ks, "v_cache": vc, "v_scale": vs, "tables": tables, "lens": _ints(totals),
           "starts": starts, "block": case["block"], "new": max(new), "longest": max(totals)}
    q = _normal((rows, case["heads"], case["dim"]), g, 1.5).half()
    if kind == "attend":
        return dict(got, q=q, scale=case["dim"] ** -0.5)
    seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), _ints(new).long())
    pos = (got["lens"] - _ints(new))[seq] + torch.arange(rows, device="cuda") - starts[seq]
    slot = tables[seq, (pos // case["block"]).long()] * case["block"] + pos % case["block"]
    got |= {"k": _heads(rows, case["kv_heads"], case["dim"], g), "v": _heads(rows, case["kv_heads"], case["dim"], g),
            "q": q, "slots": slot.to(torch.int32), "positions": pos.to(torch.int32), "cos": None, "sin": None}
    if case["rotary"]:
        half = case["rotary"] // 2
        at = torch.arange(max(totals), device="cuda", dtype=torch.float64)[:, None]
        angle = at * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        got |= {"cos": angle.cos().float(), "sin": angle.sin().float()}
    return got


def prepare(case, seed):
    return dict(_inputs(case, seed), kind=case["kind"], codes=case.get("codes"))


# ------------------------------------------------------------ plain forms

def _assign(s):
    lens, delta, bs, rows = s["lens"].long(), s["delta"].long(), s["block"], s["rows"]
    ring, (head, count) = s["ring"], s["state"].long().unbind()
    size, n = ring.numel(), lens.numel()
    add = delta.clamp(min=0)
    drop = torch.minimum((-delta).clamp(min=0), lens)
    ends = add.cumsum(0)
    have = (lens + bs - 1) // bs
    after = (lens + add + bs - 1) // bs
    fits = (add == 0) | ((after <= s["tables"].shape[1]) & (ends <= rows))
    need = torch.where(fits, after - have, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= count))
    first = upto - need
    need = torch.where(served, need, 0)
    # new blocks of the served requests, in request order
    row = torch.repeat_interleave(torch.arange(n, device=lens.device), need)
    j = torch.arange(row.numel(), device=lens.device) - (need.cumsum(0) - need)[row]
    s["tables"][row, have[row] + j] = ring[(head + first[row] + j) % size]
    # tokens
    t = torch.arange(rows, device=lens.device)
    req = torch.searchsorted(ends, t, right=True).clamp(max=n - 1)
    ok = (t < ends[-1]) & served[req]
    pos = lens[req] + t - (ends - add)[req]
    width = s["tables"].shape[1]
    slot = s["tables"][req, (pos // bs).clamp(0, width - 1)].long() * bs + pos % bs
    # blocks given back
    kept = (lens - drop + bs - 1) // bs
    back = have - kept
    row = torch.repeat_interleave(torch.arange(n, device=lens.device), back)
    j = torch.arange(row.numel(), device=lens.device) - (back.cumsum(0) - back)[row]
    at = head + count + torch.arange(row.numel(), device=lens.device)
    ring[at % size] = s["tables"][row, kept[row] + j]
    taken = need.sum()
    return {"slots": torch.where(ok, slot, -1).int(), "positions": torch.where(ok, pos, -1).int(),
            "starts": torch.cat([ends.new_zeros(1), ends.clamp(max=rows)]).int(),
            "lens": torch.where(served, lens + add - drop, lens).int(),
            "state": torch.stack([(head + taken) % size, count - taken + back.sum()]).int(),
            "tables": s["tables"], "ring": ring}


def _rotate(x, s):
    """Pairs (i, i + R/2) of the first R channels turned by the position's angle; one rounding."""
    if s["cos"] is None:
        return x
    c, n = (t[s["positions"].long()].double()[:, None, :] for t in (s["cos"], s["sin"]))
    half = c.shape[-1]
    a, b = x[..., :half].double(), x[..., half:2 * half].double()
    return torch.cat([(a * c - b * n).half(), (b * c + a * n).half(), x[..., 2 * half:]], -1)


def _write(x, cache, scale, s):
    """x into the pages of its slots: one power-of-two scale for each page and head, old codes rescaled to it."""
    bs, top = s["block"], _QMAX[s["codes"]]
    page, off = s["slots"].long() // bs, s["slots"].long() % bs
    pages, at = torch.unique(page, return_inverse=True)
    first = torch.full_like(pages, bs).scatter_reduce(0, at, off, "amin")
    x = x.float()
    big = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)  # [T, H]
    amax = torch.zeros(pages.numel(), big.shape[1], device=x.device)
    amax = amax.scatter_reduce(0, at[:, None].expand_as(big), big, "amax")
    mant, expo = torch.frexp(amax / top)
    want = torch.where(amax > 0, torch.exp2((expo - (mant == 0.5).int()).float()), 0.0).clamp(min=_MIN_SCALE)
    was = scale[pages]
    kept = (first > 0)[:, None]
    now = torch.where(kept, torch.maximum(was, want), want)
    old = cache[pages].float() * (was / now)[:, :, None, None]
    stays = torch.arange(bs, device=x.device) < first[:, None]
    old = _code(torch.where(stays[:, None, :, None], old, 0.0), s)
    fresh = _code(x * (1.0 / now[at])[..., None], s)
    codes = torch.where(stays[:, None, :, None], old.view(torch.uint8), cache[pages].view(torch.uint8))
    codes = codes.transpose(1, 2)  # [pages, bs, H, D]
    codes[at, off] = fresh.view(torch.uint8)
    cache.view(torch.uint8)[pages] = codes.transpose(1, 2)
    scale[pages] = now


def _code(x, s):
    top = _QMAX[s["codes"]]
    if s["codes"] == "int8":
        return torch.nan_to_num(x, nan=0.0, posinf=top, neginf=-top).round().clamp(-top, top).to(torch.int8)
    return x.clamp(-top, top).to(torch.float8_e4m3fn)


def _append(s):
    q, k = _rotate(s["q"], s), _rotate(s["k"], s)
    _write(k, s["k_cache"], s["k_scale"], s)
    _write(s["v"], s["v_cache"], s["v_scale"], s)
    return _cache_of(s, q if s["cos"] is not None else None)


def _cache_of(s, q):
    # the cache is the state's own: 8-bit values, and beside them the scales that multiply them
    out = {"k_cache": s["k_cache"], "k_scale": s["k_scale"], "v_cache": s["v_cache"], "v_scale": s["v_scale"]}
    return out if q is None else dict(out, q=q)


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

    def held(cache, scale):  # [n, Hkv, tokens, D]
        x = cache[pages].float() * scale[pages][..., None, None]
        return x.transpose(1, 2).reshape(n, hk, width * bs, d)

    group, m = q.shape[1] // hk, s["new"]
    qb = q[row].view(n, m, hk, group, d).permute(0, 2, 1, 3, 4).reshape(n, hk, m * group, d)
    k = held(s["k_cache"], s["k_scale"])
    sc = torch.matmul(qb * s["scale"], k.transpose(2, 3).contiguous()).view(n, hk, m, group, width * bs)
    del k
    last = s["lens"].long()[:, None] - there.sum(1, keepdim=True) + torch.arange(m, device=q.device)
    seen = torch.arange(width * bs, device=q.device) <= last[..., None]
    sc = sc.masked_fill(~seen[:, None, :, None, :], float("-inf"))
    top = sc.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(sc - top)
    del sc
    v = held(s["v_cache"], s["v_scale"]).masked_fill(
        (torch.arange(width * bs, device=q.device) >= s["lens"][:, None])[:, None, :, None], 0.0)
    o = torch.matmul(p.reshape(n, hk, m * group, width * bs), v)
    o = o / p.sum(-1).view(n, hk, m * group, 1).clamp(min=1e-30)
    o = o.view(n, hk, m, group, d).permute(0, 2, 1, 3, 4).reshape(n, m, hk * group, d)
    out = torch.zeros_like(s["q"])
    out[row[there]] = o[there].half()
    return out


def _sample(s):
    x = s["logits"].double()
    x = torch.where(x.isnan(), float("-inf"), x)
    n, v = x.shape
    t = s["temperature"].double()[:, None]
    value, index = torch.sort(x, dim=1, descending=True, stable=True)
    top = value[:, :1]
    w = torch.where(value == top, 1.0, torch.exp((value - top) / torch.where(t > 0, t, 1.0)))
    at = torch.arange(v, device=x.device)
    k = s["top_k"].long()[:, None]
    w = torch.where((k <= 0) | (at < k), w, 0.0)
    before = w.cumsum(1) - w
    p = s["top_p"].double()[:, None]
    keep = (p >= 1) | (before < p * w.sum(1, keepdim=True)) | (at == 0)
    keep &= (w >= s["min_p"].double()[:, None]) | (at == 0)
    upto = torch.where(keep, w, 0.0).cumsum(1)
    u = s["u"].double()[:, None].clamp(0, 1)
    past = keep & (upto > u * upto[:, -1:])
    # the first token, in falling order, whose running mass passes u; the last kept one where rounding hides it
    at = torch.where(past.any(1), past.int().argmax(1), keep.sum(1) - 1)
    pick = index.gather(1, at[:, None])[:, 0]
    pick = torch.where(t[:, 0] > 0, pick, index[:, 0])
    return torch.where(top[:, 0] == float("-inf"), -1, pick)


_PLAIN = {"assign": _assign, "append": _append, "attend": _attend, "sample": _sample}


# ------------------------------------------------------------ the framework's side

def _own(s):
    from gdsllm_amd.runtime import ext

    if s["kind"] == "assign":
        slots, positions, starts, lens, state = ext().kv_assign(
            s["lens"], s["delta"], s["tables"], s["ring"], s["state"], s["block"], s["rows"])
        return {"slots": slots, "positions": positions, "starts": starts, "lens": lens, "state": state,
                "tables": s["tables"], "ring": s["ring"]}
    if s["kind"] == "append":
        q = ext().kv_append(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                            s["q"] if s["cos"] is not None else None, s["positions"], s["cos"], s["sin"])
        return _cache_of(s, q)
    if s["kind"] == "attend":
        return ext().kv_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["tables"],
                                  s["lens"], s["starts"], s["scale"], s["new"], s["longest"])
    return ext().sample_tokens(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["kind"]](state)


# ------------------------------------------------------------ what a pass needs

def work(case):
    kind = case["kind"]
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * case["bits"] // 8 + 28 * case["rows"], "flops": 4 * n}
    if kind == "assign":
        held, delta = _deltas(case)
        bs, n = case["block"], case["requests"]
        moved = sum(abs(_blocks(h + d, bs) - _blocks(h, bs)) for h, d in zip(held, delta))
        tokens = -(-max(1, sum(max(d, 0) for d in delta)) // 64) * 64
        return {"bytes": 4 * (4 * n + 2 * moved + 2 * tokens + n), "flops": 8 * (n + tokens)}
    totals, new = _lengths(case)
    h, hk, d, bs = case["heads"], case["kv_heads"], case["dim"], case["block"]
    if kind == "append":
        t = sum(new)
        pages = sum(_blocks(a, bs) - (a - b) // bs for a, b in zip(totals, new))
        by = 2 * t * hk * d * (2 + 1) + 8 * pages * hk + 4 * t
        if case["rotary"]:
            by += 4 * t * h * d + 4 * t + 4 * case["rotary"] * min(t, max(totals))
        return {"bytes": by, "flops": t * d * (6 * hk + 3 * h)}
    by = sum(2 * a * hk * d + 8 * _blocks(a, bs) * hk + 4 * _blocks(a, bs) for a in totals) + 4 * sum(new) * h * d
    pairs = sum(b * (a - b) + b * (b + 1) // 2 for a, b in zip(totals, new))
    return {"bytes": by, "flops": 4 * pairs * h * d}


# --------------------------------------------------------- the same in 64 bits

def _codes64(x, codes):
    """The nearest value that the 8-bit type has (ties to the even code), float64."""
    if codes == "int8":
        return torch.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0).clamp(-127, 127).round()
    x = x.clamp(-448, 448)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))  # 3 bits behind the leading one, subnormals below 2^-6
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    """Whole-number outputs (block tables, slots, tokens) have no value of this kind."""
    if case["kind"] not in ("append", "attend"):
        return None
    x = _inputs(case, seed)

    def append():
        half = case["rotary"] // 2
        turned = {}
        for name in ("q", "k"):
            y = x[name].double()
            if half:
                c, n = (x[t].double()[x["positions"].long()].unsqueeze(1) for t in ("cos", "sin"))
                z = torch.complex(y[..., :half], y[..., half:2 * half]) * torch.complex(c, n)
                y = torch.cat([z.real, z.imag, y[..., 2 * half:]], -1)
            turned[name] = y
        out = {"q": turned["q"]} if half else {}
        bs, top = case["block"], _QMAX[case["codes"]]
        for name, y in (("k", turned["k"].half().double()), ("v", x["v"].double())):
            codes, scale = x[name + "_cache"].double(), x[name + "_scale"].double()
            slots, starts = x["slots"].tolist(), x["starts"].tolist()
            for a, b in zip(starts, starts[1:]):
                t = a
                while t < b:  # the tokens of one page
                    page, o = divmod(slots[t], bs)
                    m = min(b - t, bs - o)
                    part = y[t:t + m].transpose(0, 1)  # [H, m, D]
                    s = torch.clamp(torch.exp2(torch.ceil(torch.log2(part.abs().amax((1, 2)) / top))), min=2.0 ** -32)
                    if o:
                        s = torch.maximum(s, scale[page])
                        r = (scale[page] / s)[:, None, None]
                        codes[page, :, :o] = _codes64(codes[page, :, :o] * r, case["codes"])
                    codes[page, :, o:o + m] = _codes64(part / s[:, None, None], case["codes"])
                    scale[page] = s
                    t += m
            out |= {name + "_cache": codes, name + "_scale": scale}
        return out

    def attend():
        hk, bs, d = case["kv_heads"], case["block"], case["dim"]
        q, out = x["q"].double(), torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
        starts, lens = x["starts"].tolist(), x["lens"].tolist()
        for b, (lo, hi) in enumerate(zip(starts, starts[1:])):
            n, held = hi - lo, lens[b]
            if not n or not held:
                continue
            ids = x["tables"][b, :_blocks(held, bs)].long()
            k, v = ((x[c + "_cache"][ids].double() * x[c + "_scale"][ids].double()[..., None, None])
                    .transpose(0, 1).reshape(hk, -1, d)[:, :held] for c in "kv")
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

    return append() if case["kind"] == "append" else attend()
