"""Block assignment and 8-bit cache writes against the plain 64-bit forms
(oracle/serve.py).  Everything kv_assign writes is a whole number and has to be
equal; scales are powers of two and codes one rounding of an exact quotient, so
caches have to be equal too; a rotated q is within half an fp16 step (and the
half fp32 step it passes through) of its 64-bit value."""

import pytest
import torch

from gdsllm_amd.runtime import ext
from helpers import gen
from oracle import serve as sv

pytestmark = pytest.mark.gpu


def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------ kv_assign

def _pool(lens, bs, width, spare, g, head=None):
    """Block tables of requests holding `lens` tokens, and a ring with `spare` free blocks."""
    used = [sv.blocks(n, bs) for n in lens]
    ids = torch.randperm(sum(used) + spare, generator=g).tolist()
    tables, at = [], 0
    for u in used:
        tables.append(ids[at:at + u] + [-7] * (width - u))
        at += u
    R = sum(used) + spare
    ring = [-9] * R
    head = R - 1 if head is None else head  # the ring's contents wrap
    for i, b in enumerate(ids[at:]):
        ring[(head + i) % R] = b
    return tables, ring, [head, spare]


def _check_assign(dev, lens, delta, tables, ring, state, bs, max_tokens, again=1):
    want_t, want_r = [list(r) for r in tables], list(ring)
    want = sv.assign(lens, delta, want_t, want_r, state, bs, max_tokens)
    wide = torch.full((len(lens), len(tables[0]) + 3), 77, dtype=torch.int32, device=dev)  # rows further apart than used
    t = wide[:, :len(tables[0])]
    t.copy_(_ints(tables, dev))
    r, st = _ints(ring, dev), _ints(state, dev)
    ln, dl = _ints(lens, dev), _ints(delta, dev)
    for _ in range(again):  # inputs stay, so a second call gives the same
        got = ext().kv_assign(ln, dl, t, r, st, bs, max_tokens)
        for name, g, w in zip(("slots", "positions", "starts", "lens", "state"), got, want):
            assert g.tolist() == w, name
        assert t.tolist() == want_t and r.tolist() == want_r
    assert bool((wide[:, len(tables[0]):] == 77).all()) and ln.tolist() == lens and st.tolist() == state


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 256, 257, 1025, 8192])
@pytest.mark.parametrize("bs", [16, 128])
def test_assign(gpu, n, bs):
    g = gen(100 + n + bs)
    lens = torch.randint(0, 5 * bs, (n,), generator=g).tolist()
    delta = torch.randint(-2 * bs, 2 * bs, (n,), generator=g).tolist()
    delta[n // 2] = -10 ** 9  # ended, asked for more than it holds
    delta[n // 3] = 0
    rows = sum(max(d, 0) for d in delta)
    need = sum(sv.blocks(l + max(d, 0), bs) - sv.blocks(l, bs) for l, d in zip(lens, delta))
    tables, ring, state = _pool(lens, bs, 7, need + 5, g)
    _check_assign(gpu, lens, delta, tables, ring, state, bs, rows + 13, again=2)


def test_assign_every_length_across_a_block(gpu):
    bs = 16
    lens = list(range(0, 40))
    for d in (1, 15, 16, 17, -1, -16, -17):
        tables, ring, state = _pool(lens, bs, 5, 100, gen(1), head=3)
        _check_assign(gpu, lens, [d] * 40, tables, ring, state, bs, 40 * 17)


def test_assign_refuses_requests_that_do_not_fit(gpu):
    bs = 16
    # the third needs the last block and one more; the ones behind it that need none are still served
    lens, delta = [16, 31, 16, 5, 32, 16], [1, 1, 33, 3, -32, 1]
    tables, ring, state = _pool(lens, bs, 5, 2, gen(2))
    _check_assign(gpu, lens, delta, tables, ring, state, bs, 64, again=2)
    # a row that is too short for its request; tokens behind max_tokens
    lens, delta = [70, 3, 4, 5], [20, 5, 9, -2]
    tables, ring, state = _pool(lens, bs, 5, 20, gen(3))
    _check_assign(gpu, lens, delta, tables, ring, state, bs, 40)
    _check_assign(gpu, lens, delta, tables, ring, state, bs, 26)
    _check_assign(gpu, lens, delta, tables, ring, state, bs, 0)
    # no free block at all
    tables, ring, state = _pool([16, 8], bs, 5, 0, gen(4))
    _check_assign(gpu, [16, 8], [1, 1], tables, ring, state, bs, 2)


def test_assign_many_steps(gpu):
    """A pool used up and given back over many steps: no block is ever held twice, none is lost."""
    bs, n, width, pool = 16, 12, 8, 40
    g = gen(5)
    ring = _ints(list(range(pool)), gpu)
    tables = torch.zeros(n, width, dtype=torch.int32, device=gpu)
    lens, state = _ints([0] * n, gpu), _ints([0, pool], gpu)
    for step in range(60):
        delta = torch.randint(-30, 40, (n,), generator=g)
        delta[step % n] = -1000
        _, _, _, lens, state = ext().kv_assign(lens, delta.int().to(gpu), tables, ring, state, bs, 512)
        held = [b for r, m in zip(tables.tolist(), lens.tolist()) for b in r[:sv.blocks(m, bs)]]
        head, count = state.tolist()
        free = [ring.tolist()[(head + i) % pool] for i in range(count)]
        assert sorted(held + free) == list(range(pool))


# ------------------------------------------------------------------ kv_append

class Cache:
    """A device cache with random codes in it, and the oracle's copy in float64."""

    def __init__(self, fmt, blocks, heads, bs, dim, dev, seed):
        g = gen(seed)
        x = torch.randn(blocks, heads, bs, dim, generator=g) * 100
        x = x.clamp(-sv.QMAX[fmt], sv.QMAX[fmt])
        self.codes = (x.round() if fmt == "int8" else x).to(sv.DTYPE[fmt])
        self.scale = torch.exp2(torch.randint(-9, -3, (blocks, heads), generator=g).float())
        self.fmt, self.dev = fmt, (self.codes.to(dev), self.scale.to(dev))
        self.ref = (self.codes.double(), self.scale.double())

    def check(self, what):
        torch.testing.assert_close(self.dev[1].cpu().double(), self.ref[1], rtol=0, atol=0, msg=lambda m: f"{what} scale: {m}")
        torch.testing.assert_close(self.dev[0].cpu().double(), self.ref[0], rtol=0, atol=0, equal_nan=True,
                                   msg=lambda m: f"{what} codes: {m}")


def _append(kc, vc, k, v, slots, q=None, positions=None, cos=None, sin=None):
    dev = kc.dev[0].device
    mv = lambda t: None if t is None else t.to(dev)  # noqa: E731
    out = ext().kv_append(mv(k), mv(v), mv(slots), kc.dev[0], vc.dev[0], kc.dev[1], vc.dev[1], mv(q), mv(positions),
                          mv(cos), mv(sin))
    kr = k if cos is None else sv.rotate(k, positions, cos, sin)[0]
    s = slots.clone()
    if cos is not None:
        s[(positions < 0) | (positions >= cos.shape[0])] = -1
    sv.append(kr, s, *kc.ref, kc.fmt)
    sv.append(v, s, *vc.ref, vc.fmt)
    kc.check("k")
    vc.check("v")
    if q is not None:
        _, want = sv.rotate(q, positions, cos, sin)
        n_blocks, bs = kc.codes.shape[0], kc.codes.shape[2]
        live = (s >= 0) & (s < n_blocks * bs)
        want[~live] = 0
        err = (out.cpu().double() - want).abs()
        # to nearest through fp32: half a step of each; 2^-25 is half the step of fp16's subnormals
        assert bool((err <= (2.0 ** -11 + 2.0 ** -24) * want.abs() + 2.0 ** -25).all())
    return out


def _rope(n, half):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    return a.cos().float(), a.sin().float()


def _requests(spans, bs, blocks, g):
    """Slots of requests that add tokens [a, b) to what they hold, in blocks of their own."""
    ids = torch.randperm(blocks, generator=g).tolist()
    slots, pos = [], []
    for a, b in spans:
        mine = [ids.pop() for _ in range(sv.blocks(b, bs))]
        slots += [mine[i // bs] * bs + i % bs for i in range(a, b)]
        pos += list(range(a, b))
    return torch.tensor(slots, dtype=torch.int32), torch.tensor(pos, dtype=torch.int32)


SPANS = {
    "one": [(0, 1)],
    "last_of_block": [(15, 16)],
    "decode": [(i, i + 1) for i in range(0, 70, 5)],
    "prompts": [(0, 37), (5, 130), (16, 32), (63, 66), (0, 16)],
    "long": [(3, 700), (0, 129)],
}


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim,heads,q_heads,rotary", [(64, 3, 6, 32), (128, 2, 14, 128), (256, 1, 4, 64), (128, 8, 0, 0)])
@pytest.mark.parametrize("bs", [16, 64, 128])
@pytest.mark.parametrize("spans", list(SPANS))
def test_append(gpu, fmt, dim, heads, q_heads, rotary, bs, spans):
    g = gen(hash((dim, bs)) % 1000)
    blocks = sum(sv.blocks(b, bs) for _, b in SPANS[spans]) + 2
    kc, vc = (Cache(fmt, blocks, heads, bs, dim, gpu, s) for s in (11, 12))
    slots, pos = _requests(SPANS[spans], bs, blocks, g)
    T = slots.numel()
    # rows of a fused projection: q, k and v side by side
    fused = torch.randn(T, (q_heads + 2 * heads) * dim, generator=g).half() * 3
    q, k, v = (t.unflatten(1, (-1, dim)) for t in fused.split([q_heads * dim, heads * dim, heads * dim], 1))
    if rotary:
        cos, sin = _rope(int(pos.max()) + 1, rotary // 2)
        _append(kc, vc, k, v, slots, q, pos, cos, sin)
        _append(kc, vc, k * 2, v / 4, slots, q, pos, cos, sin)  # over what the first call wrote
    else:
        _append(kc, vc, k, v, slots)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_extreme_values(gpu, fmt):
    """Zeros, subnormals, the largest fp16, infinities and NaN; scales that grow by many powers of two and do not shrink."""
    dim, bs = 64, 16
    kc, vc = (Cache(fmt, 3, 1, bs, dim, gpu, s) for s in (21, 22))
    rows = [torch.zeros(dim), torch.full((dim,), 2.0 ** -24), torch.linspace(-1, 1, dim), torch.full((dim,), 65504.0),
            torch.tensor([float("inf"), float("-inf"), float("nan"), 1.0] * 16), torch.full((dim,), float("nan")),
            torch.full((dim,), 448.0), torch.full((dim,), 127.0), torch.full((dim,), 448.5), -torch.zeros(dim)]
    for i, r in enumerate(rows):
        x = r.half().view(1, 1, dim)
        _append(kc, vc, x, -x, torch.tensor([16 + i], dtype=torch.int32))
    order = [3, 1, 2, 0, 6, 4]
    for i, j in enumerate(order):
        x = rows[j].half().view(1, 1, dim)
        _append(kc, vc, x, x, torch.tensor([32 + i], dtype=torch.int32))


def test_append_padding_and_repeated_slots(gpu):
    dim, bs, heads = 128, 16, 2
    g = gen(31)
    cos, sin = _rope(50, dim // 2)
    kc, vc = (Cache("e4m3", 6, heads, bs, dim, gpu, s) for s in (32, 33))
    mk = lambda h: torch.randn(len(slots), h, dim, generator=g).half()  # noqa: E731
    # padding before, between and behind; slots past the cache; positions outside the table
    slots = torch.tensor([-1, 3, 4, -1, 16, 96, 2 ** 31 - 1, 40, 41, -5, 80, 81, -1], dtype=torch.int32)
    pos = torch.tensor([0, 3, 4, 0, 49, 1, 1, 50, 1, 1, -1, 7, 0], dtype=torch.int32)
    q = mk(4)
    out = _append(kc, vc, mk(heads), mk(heads), slots, q, pos, cos, sin)
    assert bool((out[[0, 3, 5, 6, 7, 9, 10, 12]] == 0).all())
    # the last of several rows with one slot stays; offsets in falling order; a rewind to offset 2
    for s in ([5, 5], [18, 17, 16, 17], [34, 35, 33, 34, 35], list(range(48, 64)) + [50, 49]):
        slots = torch.tensor(s, dtype=torch.int32)
        _append(kc, vc, mk(heads), mk(heads), slots)


def test_append_strides_and_alignment(gpu):
    """k off the 16-byte grid, transposed heads, no tokens at all."""
    dim, bs, heads, T = 64, 16, 2, 5
    g = gen(41)
    slots = torch.tensor([0, 1, 2, 20, 21], dtype=torch.int32)
    x = torch.randn(T, heads, dim, generator=g).half()
    got = []
    raw = torch.empty(T * heads * dim + 8, dtype=torch.float16, device=gpu)
    odd = raw[1:1 + x.numel()].view(x.shape).copy_(x)
    turned = x.to(gpu).transpose(0, 1).contiguous().transpose(0, 1)
    for k in (x.to(gpu), odd, turned):
        kc, vc = (Cache("int8", 2, heads, bs, dim, gpu, 42) for _ in range(2))
        ext().kv_append(k, k, slots.to(gpu), kc.dev[0], vc.dev[0], kc.dev[1], vc.dev[1])
        got.append(kc.dev[0].cpu())
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    none = torch.empty(0, heads, dim, dtype=torch.float16, device=gpu)
    assert ext().kv_append(none, none, slots[:0].to(gpu), kc.dev[0], vc.dev[0], kc.dev[1], vc.dev[1]) is None
    assert torch.equal(kc.dev[0].cpu(), got[0])


def test_append_offsets_past_32_bits(gpu):
    """Blocks whose bytes lie behind 4 GiB."""
    dim, bs, heads = 256, 256, 8
    blocks = (2 ** 32) // (heads * bs * dim) + 3
    codes = [torch.zeros(blocks, heads, bs, dim, dtype=torch.int8, device=gpu) for _ in range(2)]
    scale = [torch.ones(blocks, heads, device=gpu) for _ in range(2)]
    slots = torch.tensor([(blocks - 1) * bs + i for i in range(3)] + [7], dtype=torch.int32)
    x = torch.randn(4, heads, dim, generator=gen(51)).half()
    ext().kv_append(x.to(gpu), x.to(gpu), slots.to(gpu), *codes, *scale)
    ref_c, ref_s = torch.zeros(2, heads, bs, dim, dtype=torch.float64), torch.ones(2, heads, dtype=torch.float64)
    near = torch.tensor([bs, bs + 1, bs + 2, 7], dtype=torch.int32)
    sv.append(x, near, ref_c, ref_s, "int8")
    for c, s in zip(codes, scale):
        assert torch.equal(c[[0, -1]].cpu().double(), ref_c) and torch.equal(s[[0, -1]].cpu().double(), ref_s)
        assert not bool(c[1:-1].any())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim,heads,rotary", [(64, 5, 64), (256, 2, 128)])
@pytest.mark.parametrize("spans", ["prompts", "long"])
def test_append_largest_blocks(gpu, fmt, dim, heads, rotary, spans):
    """Blocks of 256 tokens, pages longer than their threads hold; a second call that grows the scales."""
    bs = 256
    blocks = sum(sv.blocks(b, bs) for _, b in SPANS[spans]) + 2
    kc, vc = (Cache(fmt, blocks, heads, bs, dim, gpu, s) for s in (61, 62))
    slots, pos = _requests(SPANS[spans], bs, blocks, gen(63))
    q, k, v = (torch.randn(slots.numel(), h, dim, generator=gen(64 + i)).half() for i, h in enumerate((3 * heads, heads, heads)))
    cos, sin = _rope(int(pos.max()) + 1, rotary // 2)
    _append(kc, vc, k, v, slots, q, pos, cos, sin)
    _append(kc, vc, k * 300, v * 5, slots, q, pos, cos, sin)


@pytest.mark.parametrize("bs", [16, 128])
def test_append_large_decode_batch(gpu, bs):
    """More tokens than a workgroup to each would leave room for, every one in a block of its own."""
    n, heads, dim = 700, 2, 128
    kc, vc = (Cache("e4m3", n + 3, heads, bs, dim, gpu, s) for s in (71, 72))
    slots = torch.randperm(n + 3, generator=gen(73))[:n].int() * bs + torch.randint(0, bs, (n,), generator=gen(74)).int()
    slots[::41] = -1
    q, k, v = (torch.randn(n, h, dim, generator=gen(75 + h)).half() for h in (8, heads, heads))
    cos, sin = _rope(90, 64)
    _append(kc, vc, k, v, slots, q, torch.randint(0, 90, (n,), generator=gen(78)).int(), cos, sin)


def test_append_turns_keys_without_queries(gpu):
    """A rotation without q, and on a stream of the caller's."""
    kc, vc = (Cache("e4m3", 9, 2, 16, 128, gpu, s) for s in (81, 82))
    slots, pos = _requests([(0, 40), (7, 60)], 16, 9, gen(83))
    k, v = (torch.randn(slots.numel(), 2, 128, generator=gen(84 + i)).half() for i in range(2))
    cos, sin = _rope(64, 48)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert _append(kc, vc, k, v, slots, None, pos, cos, sin) is None


def test_append_long_prompt_in_large_blocks(gpu):
    """Past 2048 tokens the queries of large blocks are turned by a launch of their own."""
    bs, dim = 256, 64
    kc, vc = (Cache("int8", 12, 1, bs, dim, gpu, s) for s in (91, 92))
    slots, pos = _requests([(0, 2100), (5, 80)], bs, 12, gen(93))
    slots, pos = (torch.cat([t[:2100], torch.tensor([-1, -1], dtype=torch.int32), t[2100:]]) for t in (slots, pos))
    q, k, v = (torch.randn(slots.numel(), h, dim, generator=gen(94 + h)).half() for h in (3, 1, 1))
    cos, sin = _rope(2100, 16)
    _append(kc, vc, k, v, slots, q, pos, cos, sin)
