"""Writes into the 4-bit cache and reads of it against the 64-bit forms
(oracle/serve4.py).  Scales, biases and codes are roundings of exact quotients, an
element one rounding: everything has to be equal, bit for bit."""

import pytest
import torch

from gdsllm_amd.runtime import ext
from helpers import gen
from oracle import serve4 as s4

pytestmark = pytest.mark.gpu


class Cache:
    """A device cache with arbitrary bytes in it, and the oracle's copy."""

    def __init__(self, dev, blocks, heads, bs, dim, group, seed):
        g = gen(seed)
        shape = (blocks, heads, bs, dim // 2)
        self.ref = [torch.randint(0, 256, shape, generator=g).to(torch.uint8) for _ in range(2)]
        self.ref += [torch.randn(blocks, heads, dim // group, bs, 2, generator=g).half() for _ in range(2)]
        self.dev = [t.to(dev) for t in self.ref]

    def check(self):
        for name, a, b in zip(("k", "v", "k_affine", "v_affine"), self.dev, self.ref):
            assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8)), name

    def append(self, k, v, slots, q=None, pos=None, cos=None, sin=None, neighbours=False):
        mv = lambda t: None if t is None else t.to(self.dev[0].device)  # noqa: E731
        out = ext().kv4_append(mv(k), mv(v), mv(slots), *self.dev, mv(q), mv(pos), mv(cos), mv(sin), neighbours)
        s = slots.clone()
        if cos is not None:
            s[(pos < 0) | (pos >= cos.shape[0])] = -1
            k = s4.rotate(k, pos, cos, sin, neighbours)[0]
        s4.append(k, s, self.ref[0], self.ref[2])
        s4.append(v, s, self.ref[1], self.ref[3])
        if q is None:
            assert out is None
        else:
            ok = (s >= 0) & (s < self.ref[0].shape[0] * self.ref[0].shape[2])
            want = torch.where(ok[:, None, None], s4.rotate(q, pos, cos, sin, neighbours)[0], 0.0)
            assert torch.equal(out.cpu(), want)
        self.check()


def rows(tokens, heads, dim, g):
    return (torch.randn(tokens, heads, dim, generator=g) * torch.exp(torch.randn(heads, dim, generator=g))).half()


def angles(positions, rotary, g):
    a = torch.rand(positions, rotary // 2, generator=g) * 6.3
    return a.cos(), a.sin()


SHAPES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)]


@pytest.mark.parametrize("dim,group", SHAPES, ids=[f"d{d}_g{g}" for d, g in SHAPES])
@pytest.mark.parametrize("heads", [1, 3, 8])
@pytest.mark.parametrize("rotary,neighbours", [(0, False), (16, False), (16, True), (64, False), (64, True)])
def test_append(gpu, dim, group, heads, rotary, neighbours):
    """Runs of rows in blocks in no order, padding between the runs, slots outside the cache."""
    g = gen(dim + group + heads + rotary)
    c = Cache(gpu, 7, heads, 16, dim, group, 1)
    slots = torch.cat([torch.arange(80, 96), torch.tensor([-1, 3, 4, 5, -1, -1, 112, 10 ** 9, 47]), torch.arange(16, 27)]).int()
    n = slots.numel()
    k, v = rows(n, heads, dim, g), rows(n, heads, dim, g)
    if not rotary:
        return c.append(k, v, slots)
    pos = torch.randint(0, 50, (n,), generator=g).int()
    pos[5], pos[20] = -1, 50
    c.append(k, v, slots, rows(n, 2 * heads, dim, g), pos, *angles(50, rotary, g), neighbours)


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("tokens", [1, 2, 63, 64, 65, 200])
def test_block_sizes(gpu, bs, tokens):
    """Whole blocks and their ends, over blocks in falling order."""
    g = gen(bs + tokens)
    c = Cache(gpu, 9 + 200 // bs, 2, bs, 128, 64, 2)
    t = torch.arange(tokens) + bs - 3
    pages = torch.arange(8 + 200 // bs, -1, -1)
    c.append(rows(tokens, 2, 128, g), rows(tokens, 2, 128, g), (pages[t // bs] * bs + t % bs).int())


@pytest.mark.parametrize("dim,rotary", [(128, 128), (256, 256), (256, 48), (64, 32)])
@pytest.mark.parametrize("neighbours", [False, True])
def test_prompts(gpu, dim, rotary, neighbours):
    """Many rows, so that a wave takes several heads of a token, and the whole head or a part of it turns."""
    g = gen(dim + rotary)
    c = Cache(gpu, 70, 12, 64, dim, 64, 3)
    n = 4200
    c.append(rows(n, 12, dim, g), rows(n, 12, dim, g), (torch.arange(n) + 17).int(), rows(n, 13, dim, g),
             torch.arange(n).int(), *angles(n, rotary, g), neighbours)


@pytest.mark.parametrize("order", ["twice", "falling", "all"])
def test_rows_with_one_slot(gpu, order):
    """The last row of a slot counts, wherever in its block's run of rows the others stand."""
    g = gen(4)
    slots = {"twice": [32, 33, 32, 34, 33, 48, -1, 40, 40, 41], "falling": list(range(255, 128, -1)) + [140, 255],
             "all": [70] * 300}[order]
    bs = {"twice": 16, "falling": 128, "all": 64}[order]
    c = Cache(gpu, 5, 2, bs, 64, 32, 5)
    n = len(slots)
    c.append(rows(n, 2, 64, g), rows(n, 2, 64, g), torch.tensor(slots, dtype=torch.int32))


@pytest.mark.parametrize("group", [32, 64, 128])
def test_values_at_the_edges(gpu, group):
    """Equal values, zeros of both signs, subnormals, the type's whole range, ties between codes, infinities and NaN,
    groups without any number."""
    g = gen(6)
    n, dim = 64, 128
    x = torch.randn(n, 1, dim, generator=g)
    x[0], x[1], x[2] = 3.25, 0.0, -0.0
    x[3] *= 2.0 ** -24
    x[4] = torch.where(x[4] > 0, 65504.0, -65504.0)
    x[5] = torch.where(x[5] > 0, 65504.0, 2.0 ** -24)
    x[6] = torch.arange(dim) % 16  # whole codes
    x[7] = (torch.arange(dim) % 31) / 2  # every other value lies between two codes
    x[8] = 1000 + x[8] / 16
    x[9] = 2.0 ** -24
    x[9, :, ::3] = 3 * 2.0 ** -24
    x[10, :, 5], x[11, :, 7], x[12, :, ::2] = float("inf"), float("-inf"), float("nan")
    x[13], x[14], x[15] = float("nan"), float("inf"), float("-inf")
    x[16, :, ::2], x[16, :, 1::2] = float("inf"), float("nan")
    x[17] = 65504.0
    x[18], x[18, :, ::9] = float("inf"), 2.0
    x[19] = torch.tensor([0.0, 2.0 ** -24])[torch.arange(dim) % 2]
    x[20] = torch.tensor([-65504.0, 2.0 ** -24, 65504.0 / 15, 30000.0])[torch.arange(dim) % 4]
    for i in range(21, n):
        x[i] *= torch.exp(4 * torch.randn(dim, generator=g))
    x = x.half()
    c = Cache(gpu, 4, 1, 16, dim, group, 7)
    c.append(x, x.flip(0), torch.arange(n).int())
    k, v = ext().kv4_values(torch.arange(n, dtype=torch.int32, device=gpu), *c.dev)
    assert bool(k.isfinite().all()) and bool(v.isfinite().all())


def test_every_exponent(gpu):
    """Groups of every range and offset that fp16 has."""
    g = gen(8)
    n, dim = 4096, 64
    at = torch.exp2(torch.randint(-24, 16, (n, 1, 1), generator=g).float())
    spread = torch.exp2(torch.randint(-24, 16, (n, 1, 1), generator=g).float())
    x = (at * torch.randn(n, 1, 1, generator=g) + spread * torch.randn(n, 1, dim, generator=g)).clamp(-65504, 65504).half()
    c = Cache(gpu, n // 64, 1, 64, dim, 32, 9)
    c.append(x, x.flip(0), torch.arange(n).int())


def test_values_next_to_ties(gpu):
    """Groups of values in the middle between two codes of theirs, or one fp16 step off it, of every range and offset;
    signalling NaNs among them."""
    g = gen(10)
    n, dim, group = 4096, 64, 32
    low = (torch.exp2(torch.randint(-24, 15, (n, 2, 1), generator=g).float()) * torch.randn(n, 2, 1, generator=g)).half().double()
    span = 15 * torch.exp2(torch.randint(-24, 11, (n, 2, 1), generator=g).double()) * (1 + torch.rand(n, 2, 1, generator=g).double())
    high = (low + span).clamp(max=65504).half().double()
    scale = ((high - low) / 15).float().half().double()
    x = (low + (torch.randint(0, 15, (n, 2, group), generator=g) + 0.5) * scale).clamp(-65504, 65504).half()
    x = (x.view(torch.int16) + torch.randint(-1, 2, x.shape, generator=g).to(torch.int16)).view(torch.float16)
    x = torch.minimum(torch.maximum(x.double(), low), high)
    x[:, :, :1], x[:, :, 1:2] = low, high
    x = x.half().reshape(n, 1, dim)
    x.view(torch.int16)[::7, 0, 9] = 0x7C01
    c = Cache(gpu, n // 64, 1, 64, dim, group, 11)
    c.append(x, x.flip(0), torch.arange(n).int())


def test_append_and_values_in_a_graph(gpu):
    """A replay takes what its inputs hold then, as the eager calls do."""
    g = gen(12)
    n, heads, dim = 37, 3, 128
    a, b = Cache(gpu, 6, heads, 16, dim, 64, 13), Cache(gpu, 6, heads, 16, dim, 64, 13)
    cos, sin = (t.to(gpu) for t in angles(50, dim, g))
    k, v, slots, pos = (torch.zeros(s, dtype=d, device=gpu) for s, d in (((n, heads, dim), torch.float16),) * 2 +
                        (((n,), torch.int32),) * 2)

    def step(c):
        q = ext().kv4_append(k, v, slots, *c.dev, k, pos, cos, sin, True)
        return (q, *ext().kv4_values(slots, *c.dev))

    step(Cache(gpu, 6, heads, 16, dim, 64, 14))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(a)
    for i in range(4):
        k.copy_(rows(n, heads, dim, g))
        v.copy_(rows(n, heads, dim, g))
        slots.copy_(torch.randperm(96, generator=g)[:n].sort().values.int())
        pos.copy_(torch.randint(-1, 51, (n,), generator=g).int())
        graph.replay()
        want = step(b)
        torch.cuda.synchronize()
        assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(got, want))
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a.dev, b.dev))


def test_strided_rows_and_another_stream(gpu):
    """q, k and v inside one projection's rows, on a stream of the caller's."""
    g = gen(10)
    n, c = 21, Cache(gpu, 4, 2, 16, 128, 64, 11)
    wide = rows(n, 10, 128, g)
    cos, sin = angles(40, 128, g)
    pos, slots = torch.arange(n).int(), torch.arange(5, 5 + n).int()
    d = [t.to(gpu) for t in (wide, slots, pos, cos, sin)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ext().kv4_append(d[0][:, 4:6], d[0][:, 7:9], d[1], *c.dev, d[0][:, :4], *d[2:])
    s.synchronize()
    s4.append(s4.rotate(wide[:, 4:6], pos, cos, sin)[0], slots, c.ref[0], c.ref[2])
    s4.append(wide[:, 7:9], slots, c.ref[1], c.ref[3])
    c.check()
    assert torch.equal(got.cpu(), s4.rotate(wide[:, :4], pos, cos, sin)[0])


def test_no_rows(gpu):
    c = Cache(gpu, 2, 1, 16, 64, 32, 12)
    none = torch.zeros(0, 1, 64).half()
    c.append(none, none, torch.zeros(0, dtype=torch.int32))
    c.append(rows(3, 1, 64, gen(1)), rows(3, 1, 64, gen(2)), torch.tensor([-1, -5, 32], dtype=torch.int32))


@pytest.mark.parametrize("dim,group", SHAPES, ids=[f"d{d}_g{g}" for d, g in SHAPES])
@pytest.mark.parametrize("heads,bs", [(1, 16), (5, 64), (32, 256)])
def test_values(gpu, dim, group, heads, bs):
    g = gen(20 + dim + group)
    c = Cache(gpu, 6, heads, bs, dim, group, 13)
    slots = torch.randint(0, 6 * bs, (77,), generator=g).int()
    slots[3], slots[4], slots[76] = -1, 6 * bs, 2 ** 31 - 1
    got = ext().kv4_values(slots.to(gpu), *c.dev)
    for x, code, pair in zip(got, c.ref[:2], c.ref[2:]):
        assert torch.equal(x.cpu().double(), s4.values(slots, code, pair))
    assert ext().kv4_values(slots[:0].to(gpu), *c.dev)[0].shape == (0, heads, dim)


def test_blocks_past_32_bits(gpu):
    """Blocks whose codes lie behind 4 GiB."""
    heads, bs, dim = 16, 256, 256
    blocks = 2 ** 32 // (heads * bs * dim // 2) + 2
    codes = [torch.zeros(blocks, heads, bs, dim // 2, dtype=torch.uint8, device=gpu) for _ in range(2)]
    pairs = [torch.zeros(blocks, heads, 8, bs, 2, dtype=torch.float16, device=gpu) for _ in range(2)]
    g = gen(30)
    k, v = rows(3, heads, dim, g), rows(3, heads, dim, g)
    slots = torch.tensor([blocks * bs - 1, blocks * bs - 2, 7], dtype=torch.int32)
    ext().kv4_append(k.to(gpu), v.to(gpu), slots.to(gpu), *codes, *pairs)
    got = ext().kv4_values(slots.to(gpu), *codes, *pairs)
    for x, y in zip(got, (k, v)):
        code, scale, bias = s4.quantize(y, 32)
        want = s4.elements(s4.pack(code)[:, :, None], torch.stack((scale, bias), -1)[:, :, :, None])
        assert torch.equal(x.cpu().double(), want[:, :, 0])
    assert not bool(codes[0][1].any()) and not bool(codes[0][blocks - 2].any())


def test_refusals(gpu):
    c = Cache(gpu, 2, 2, 16, 64, 32, 14)
    k = torch.zeros(3, 2, 64, dtype=torch.float16, device=gpu)
    s = torch.zeros(3, dtype=torch.int32, device=gpu)
    kc, vc, ka, va = c.dev
    cs = torch.zeros(4, 16, device=gpu)
    bad = [((k.float(), k, s, kc, vc, ka, va), "k must be"), ((k, k[:2], s, kc, vc, ka, va), "differ"),
           ((k, k[:, :1], s, kc, vc, ka, va), "v must be"), ((k, k, s[:2], kc, vc, ka, va), "slots"),
           ((k, k, s.long(), kc, vc, ka, va), "slots"), ((k, k, s, kc.view(torch.int8), vc, ka, va), "k_cache"),
           ((k, k, s, kc, vc[:1], ka, va), "v_cache"), ((k, k, s, kc, vc, ka.float(), va), "affine"),
           ((k, k, s, kc, vc, ka, va[:, :, :1]), "affine"), ((k, k, s, kc, vc, ka.transpose(2, 3), va), "affine"),
           ((k, k, s, kc, vc, ka, va, k), "without cos"), ((k, k, s, kc, vc, ka, va, k, s, cs), "together"),
           ((k, k, s, kc, vc, ka, va, k, None, cs, cs), "positions"), ((k, k, s, kc, vc, ka, va, k, s, cs, cs[:2]), "sin"),
           ((k, k, s, kc, vc, ka, va, k[:2], s, cs, cs), "differ"), ((k, k, s, kc, vc, ka, va, k, s, cs[:, :12], cs[:, :12]), "rotary")]
    for args, word in bad:
        with pytest.raises(RuntimeError, match=word):
            ext().kv4_append(*args)
    with pytest.raises(RuntimeError, match="slots"):
        ext().kv4_values(s.long(), *c.dev)
    c.check()


def test_gradients_are_refused(gpu):
    """There is no backward pass: rows that autograd would follow are refused before anything is written."""
    g = gen(71)
    c = Cache(gpu, 3, 2, 16, 64, 32, 72)
    k, v, q = (rows(3, h, 64, g).to(gpu) for h in (2, 2, 4))
    slots, pos = (torch.tensor(t, dtype=torch.int32, device=gpu) for t in ([5, 6, 7], [0, 1, 2]))
    cos, sin = (t.to(gpu) for t in angles(9, 64, g))
    for i, name in enumerate("kvq"):
        rows_ = [k, v, q]
        rows_[i] = rows_[i].clone().requires_grad_()
        with pytest.raises(RuntimeError, match=f"kv4_append: {name} needs a gradient"):
            ext().kv4_append(*rows_[:2], slots, *c.dev, rows_[2], pos, cos, sin)
        c.check()
    with torch.no_grad():
        ext().kv4_append(k.clone().requires_grad_(), v, slots, *c.dev, q, pos, cos, sin)
    c.append(k.cpu(), v.cpu(), slots.cpu(), q.cpu(), pos.cpu(), cos.cpu(), sin.cpu())
