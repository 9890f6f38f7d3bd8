"""Attention over the 8-bit cache against the plain 64-bit form
(oracle/serve.py attention, which derives the bound its results are held to)."""

import ctypes
import math

import pytest
import torch

from gdsllm_amd import KvCache8, capi
from gdsllm_amd.runtime import ext
from helpers import gen
from oracle import serve as sv

pytestmark = pytest.mark.gpu


class Problem:
    def __init__(self, dev, fmt, dim, heads, kv_heads, bs, lens, new, seed, extra_rows=0, spread=1.0, qscale=1.0):
        g = gen(seed)
        counts = [sv.blocks(n, bs) for n in lens]
        pool = sum(counts) + 2
        x = torch.randn(2, pool, kv_heads, bs, dim, generator=g) * 100
        x = x.clamp(-sv.QMAX[fmt], sv.QMAX[fmt])
        self.codes = (x.round() if fmt == "int8" else x).to(sv.DTYPE[fmt])
        # any positive scale: those kv_append writes are powers of two
        self.scales = 0.01 * torch.exp(spread * torch.randn(2, pool, kv_heads, generator=g))
        ids = torch.randperm(pool, generator=g)
        width = max(1, max(counts))
        self.tables = torch.full((len(lens), width), -1, dtype=torch.int32)
        at = 0
        for b, c in enumerate(counts):
            self.tables[b, :c] = ids[at:at + c].int()
            at += c
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.starts = torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32)
        self.q = (torch.randn(sum(new) + extra_rows, heads, dim, generator=g) * qscale).half()
        self.scale, self.dev, self.fmt, self.bs = dim ** -0.5, dev, fmt, bs
        self.new, self.longest = max(new), max(lens)

    def poison(self):
        """Everything behind a request's last token, and blocks nobody holds, is no number (e4m3) or large."""
        held = torch.zeros(self.codes.shape[1], self.bs, dtype=torch.bool)
        for row, n in zip(self.tables.tolist(), self.lens.tolist()):
            for i in range(n):
                held[row[i // self.bs], i % self.bs] = True
        bad = 0x7F
        c = self.codes.view(torch.uint8)
        c.copy_(torch.where(held[None, :, None, :, None], c, torch.tensor(bad, dtype=torch.uint8)))
        free = ~held.any(1)
        self.scales[:, free] = float("nan")

    def run(self, max_new=None, max_len=None, **kw):
        d = lambda t: t.to(self.dev)  # noqa: E731
        return ext().kv_attention(d(self.q), d(self.codes[0]), d(self.codes[1]), d(self.scales[0]), d(self.scales[1]),
                                  d(self.tables), d(self.lens), d(self.starts), self.scale,
                                  self.new if max_new is None else max_new,
                                  self.longest if max_len is None else max_len, **kw)

    def check(self, got):
        s = self.scales.double().nan_to_num(1.0)
        vals = self.codes.double() * s[..., None, None]
        want, bound = sv.attention(self.q, vals[0], vals[1], s[1], self.tables, self.lens, self.starts, self.scale)
        err = (got.cpu().double() - want).abs()
        assert bool((err <= bound).all()), f"worst {float((err / bound.clamp(min=2.0 ** -25)).max()):.3f} of the bound"


HEADS = [(64, 4, 4), (128, 8, 1), (128, 6, 2), (256, 16, 1), (128, 7, 7), (64, 40, 2)]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim,heads,kv_heads", HEADS, ids=[f"d{d}_{h}x{k}" for d, h, k in HEADS])
@pytest.mark.parametrize("bs", [16, 32, 64, 256])
def test_decode(gpu, fmt, dim, heads, kv_heads, bs):
    """One new token a request: lengths about a block's and a tile's edge, an idle slot among them."""
    lens = [1, 15, 16, 17, 0, 31, 33, 63, 64, 65, 127, 129, 255, 257, 300]
    p = Problem(gpu, fmt, dim, heads, kv_heads, bs, lens, [0 if n == 0 else 1 for n in lens], 200 + dim + bs)
    p.poison()
    p.check(p.run())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim,heads,kv_heads,bs", [(128, 4, 1, 64), (64, 8, 8, 16), (256, 4, 2, 128)])
def test_decode_split(gpu, fmt, dim, heads, kv_heads, bs):
    """Sequences long enough to be split, the last unit short; the bound on the length loose, right and too small."""
    p = Problem(gpu, fmt, dim, heads, kv_heads, bs, [2100, 513, 5, 1024], [1, 1, 1, 1], 300 + dim)
    p.poison()
    outs = [p.run(), p.run(max_len=0), p.run(max_len=300), p.run(max_new=0)]
    for o in outs:
        p.check(o)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim,heads,kv_heads,bs", [(128, 4, 1, 64), (64, 3, 3, 16), (256, 4, 2, 128), (128, 14, 2, 32)])
@pytest.mark.parametrize("lens,new", [([5, 300, 64, 129], [5, 2, 64, 100]), ([200], [200]), ([17, 0, 40], [1, 0, 33]),
                                      ([400, 3], [3, 3])], ids=["ragged", "whole", "mixed", "few"])
def test_prompts(gpu, fmt, dim, heads, kv_heads, bs, lens, new):
    """Several new tokens a request, behind what its cache holds; rows see the tokens up to their own."""
    p = Problem(gpu, fmt, dim, heads, kv_heads, bs, lens, new, 400 + dim + bs)
    p.poison()
    p.check(p.run())


def test_rows_that_see_nothing_and_rows_behind_the_last(gpu):
    """More rows than tokens (a request that was not served): the first rows see nothing and are zero.  Rows behind
    the last request are zero in a new tensor and left alone in a given one."""
    p = Problem(gpu, "e4m3", 128, 4, 2, 16, [3, 0, 20], [5, 2, 1], 500, extra_rows=6)
    p.poison()
    got = p.run()
    p.check(got)
    assert bool((got[:2] == 0).all()) and bool((got[5:7] == 0).all()) and bool((got[8:] == 0).all())
    wide = torch.full((14, 4 * 128 + 64), 7.0, dtype=torch.float16, device=gpu)
    out = wide[:, :4 * 128].unflatten(1, (4, 128))
    assert p.run(output=out).data_ptr() == out.data_ptr()
    p.check(torch.cat([out[:8], torch.zeros_like(out[8:])]))
    assert bool((wide[8:] == 7).all()) and bool((wide[:, 512:] == 7).all())


def test_scales_far_apart(gpu):
    """Value scales of neighbouring blocks 2^40 apart, a block of zeros with a tiny scale, large scores."""
    p = Problem(gpu, "e4m3", 64, 2, 1, 16, [200, 64], [1, 3], 600, spread=0.0, qscale=6.0)
    e = torch.arange(p.scales.shape[1]) % 3
    p.scales[1] *= torch.exp2(torch.tensor([0.0, -40.0, -20.0]))[e][:, None]
    p.codes[1].view(torch.uint8)[p.tables[0, 3]] = 0
    p.check(p.run())


def test_blocks_outside_the_cache_have_no_weight(gpu):
    p = Problem(gpu, "int8", 64, 2, 1, 16, [40], [1], 700)
    want = Problem(gpu, "int8", 64, 2, 1, 16, [40], [1], 700)
    keep = p.tables.clone()
    p.tables[0, 1] = 10 ** 9
    got = p.run()
    # the same as with the block's tokens left out: one softmax over the rest
    vals = want.codes.double() * want.scales.double()[..., None, None]
    ids = keep[0].long()
    ids = torch.stack([ids[0], ids[2]])
    k, v = (vals[i][ids, 0].reshape(-1, 64)[:24] for i in range(2))
    for h in range(2):
        o = torch.softmax((k @ want.q[0, h].double()) * want.scale, 0) @ v
        assert float((got[0, h].cpu().double() - o).norm() / o.norm()) < 2e-3


def test_special_values(gpu):
    """A NaN key reaches its row alone; q without any number gives none; int8 zeros give zeros."""
    p = Problem(gpu, "e4m3", 64, 2, 2, 16, [20, 20], [1, 1], 800)
    p.codes[0].view(torch.uint8)[p.tables[0, 0], 0, 3, 5] = 0x7F
    got = p.run()
    assert bool(got[0, 0].isnan().all()) and bool(got[0, 1].isfinite().all()) and bool(got[1].isfinite().all())
    z = Problem(gpu, "int8", 64, 2, 2, 16, [20, 20], [1, 1], 801)
    z.codes.zero_()
    assert bool((z.run() == 0).all())


def test_strided_q_and_tables_on_another_stream(gpu):
    """q inside a fused projection's rows, tables inside a wider tensor, on a stream of the caller's."""
    p = Problem(gpu, "e4m3", 128, 4, 2, 32, [100, 7], [2, 1], 900)
    wide = torch.randn(3, 8 * 128).half().to(gpu)
    wide[:, :512] = p.q.flatten(1).to(gpu)
    tabs = torch.full((2, 9), -3, dtype=torch.int32, device=gpu)
    tabs[:, :p.tables.shape[1]] = p.tables.to(gpu)
    d = lambda t: t.to(gpu)  # noqa: E731
    args = [wide[:, :512].unflatten(1, (4, 128)), d(p.codes[0]), d(p.codes[1]), d(p.scales[0]), d(p.scales[1]),
            tabs[:, :p.tables.shape[1]], d(p.lens), d(p.starts)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ext().kv_attention(*args, p.scale)
    s.synchronize()
    p.check(got)


def test_long_cache_past_32_bits(gpu):
    """Blocks whose bytes lie behind 4 GiB."""
    dim, bs, heads = 256, 256, 8
    blocks = (2 ** 32) // (heads * bs * dim) + 2
    codes = [torch.zeros(blocks, heads, bs, dim, dtype=torch.int8, device=gpu) for _ in range(2)]
    x = torch.randint(-127, 128, (2, heads, bs, dim), generator=gen(1000)).to(torch.int8)
    for c, y in zip(codes, x):
        c[-1] = y.to(gpu)
    scale = torch.full((blocks, heads), 0.01, device=gpu)
    q = torch.randn(1, heads, dim, generator=gen(1001)).half()
    got = ext().kv_attention(q.to(gpu), *codes, scale, scale, torch.tensor([[blocks - 1]], dtype=torch.int32, device=gpu),
                             torch.tensor([200], dtype=torch.int32, device=gpu),
                             torch.tensor([0, 1], dtype=torch.int32, device=gpu), dim ** -0.5)
    s = torch.full((1, heads), 0.01).double()
    vals = x.double() * scale[0, 0].cpu().double()
    want, bound = sv.attention(q, vals[:1], vals[1:], s, torch.tensor([[0]]), torch.tensor([200]), torch.tensor([0, 1]),
                               dim ** -0.5)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


def repeated(p, dev, lens, new, seed):
    """The problem's blocks, in any order and again and again, as long sequences."""
    width = max(sv.blocks(n, p.bs) for n in lens)
    p.tables = torch.randint(0, p.codes.shape[1], (len(lens), width), generator=gen(seed)).int()
    p.lens = torch.tensor(lens, dtype=torch.int32)
    p.starts = torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32)
    p.q = torch.randn(sum(new), *p.q.shape[1:], generator=gen(seed + 1)).half()
    p.new, p.longest = max(new), max(lens)


def check_heads(p, got, kv_heads):
    """check() of some kv heads and their query heads."""
    G, sel = p.q.shape[1] // p.codes.shape[2], torch.tensor(kv_heads)
    heads = (sel[:, None] * G + torch.arange(G)).flatten()
    s = p.scales[:, :, sel].double()
    vals = p.codes[:, :, sel].double() * s[..., None, None]
    want, bound = sv.attention(p.q[:, heads], vals[0], vals[1], s[1], p.tables, p.lens, p.starts, p.scale)
    assert bool(((got[:, heads.to(got.device)].cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("max_new,max_len", [(1, 0), (0, 4000), (2, 3000), (17, 2500), (1, 16)])
def test_bounds_smaller_than_the_requests(gpu, max_new, max_len):
    """The host's bounds only say how the work is split: requests with more rows and tokens than they say, where
    sequences are shared out and where not."""
    p = Problem(gpu, "e4m3", 64, 4, 2, 32, [2500, 40, 0, 3000, 700], [7, 20, 0, 1, 33], 1200)
    p.poison()
    p.check(p.run(max_new=max_new, max_len=max_len))


def test_more_requests_than_a_step_of_the_sums(gpu):
    """More than 256 requests share one line of work."""
    lens = [(37 * i) % 90 for i in range(299)] + [2600, 5]
    p = Problem(gpu, "int8", 64, 2, 1, 64, lens, [min(1, n) for n in lens], 1300)
    p.poison()
    p.check(p.run())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim,heads,kv_heads,bs", [(64, 4, 2, 16), (128, 2, 2, 64), (256, 6, 2, 128)])
def test_long_prompts_share_the_work(gpu, fmt, dim, heads, kv_heads, bs):
    """Few sequences past 2048 tokens: every tile's keys lie in several workgroups' shares, rows that see none of
    a share among them; requests of few rows beside them."""
    p = Problem(gpu, fmt, dim, heads, kv_heads, bs, [2300, 70, 2100, 180], [150, 2, 1, 180], 1400 + dim)
    p.poison()
    p.check(p.run())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_sequences_take_the_widest_tiles(gpu, fmt, dim):
    """512 and more (request, kv head, 256 rows): the last rows of a tile ragged, a request with few rows."""
    p = Problem(gpu, fmt, dim, 512, 128, 16, [130, 65, 7], [100, 65, 2], 1500 + dim)
    p.poison()
    check_heads(p, p.run(), [0, 77, 127])


def test_whole_sequences_past_a_segment(gpu):
    """Many sequences, so that each has a workgroup of its own, longer than the block table it holds at once."""
    p = Problem(gpu, "int8", 256, 1024, 1024, 64, [100, 3], [1, 1], 1600)
    repeated(p, gpu, [8300, 3], [1, 1], 1601)
    check_heads(p, p.run(), [0, 500, 1023])
    p = Problem(gpu, "e4m3", 64, 256, 256, 16, [60], [2], 1602)
    repeated(p, gpu, [4200], [40], 1603)
    check_heads(p, p.run(), [0, 255])


def test_a_sequence_in_more_parts_than_threads_that_join(gpu):
    """One long sequence among short ones, in about 470 parts; 256 threads add a row's."""
    lens = [120000] + list(range(1, 32))
    p = Problem(gpu, "e4m3", 64, 16, 1, 256, [1000] * 32, [1] * 32, 1700)
    repeated(p, gpu, lens, [1] * 32, 1701)
    p.q *= 0.5
    check_heads(p, p.run(), [0])


def test_two_graphs_on_two_streams(gpu):
    """Captured calls that share their work out keep workspaces apart: replayed side by side, each gives what it
    gives alone."""
    ps = [Problem(gpu, "e4m3", 128, 4, 1, 64, [5000, 3000 + i], [1, 1], 1800 + i) for i in range(2)]
    graphs, outs, args = [], [], []
    for p in ps:
        d = lambda t: t.to(gpu)  # noqa: E731
        a = [d(p.q), d(p.codes[0]), d(p.codes[1]), d(p.scales[0]), d(p.scales[1]), d(p.tables), d(p.lens), d(p.starts)]
        ext().kv_attention(*a, p.scale)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = ext().kv_attention(*a, p.scale)
        graphs.append(g), outs.append(o), args.append(a)
    streams = [torch.cuda.Stream() for _ in ps]
    for _ in range(5):
        for o in outs:
            o.fill_(9.0)
        torch.cuda.synchronize()
        for _ in range(4):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for p, o, a in zip(ps, outs, args):
            p.check(o)
            assert torch.equal(o, ext().kv_attention(*a, p.scale))


def test_one_key_head_for_many_query_heads(gpu):
    """128 query heads over one key head: a single new token fills a tile of 128 rows."""
    p = Problem(gpu, "e4m3", 64, 128, 1, 32, [2500, 100, 0, 3], [1, 1, 0, 1], 1900)
    p.poison()
    p.check(p.run())


def test_no_rows(gpu):
    p = Problem(gpu, "int8", 64, 4, 2, 16, [5, 40], [0, 0], 2000)
    assert p.run(max_new=0).shape == (0, 4, 64)
    p = Problem(gpu, "int8", 64, 4, 2, 16, [5, 40], [0, 0], 2000, extra_rows=3)
    assert bool((p.run(max_new=0) == 0).all())


@pytest.mark.parametrize("seed", range(24))
def test_drawn_sizes(gpu, seed):
    """Any sizes together: requests idle, decoding and with prompts, bounds given, loose or not at all."""
    g = gen(3000 + seed)
    pick = lambda *v: v[int(torch.randint(len(v), (1,), generator=g))]  # noqa: E731
    kv, group = pick(1, 2, 3), pick(1, 2, 5, 8)
    n, longest = pick(1, 2, 5, 9), pick(40, 300, 1100, 2600)
    lens = [int(v) for v in torch.randint(0, longest + 1, (n,), generator=g)]
    new = [min(pick(0, 1, 1, 2, 9, 70), m) for m in lens]
    p = Problem(gpu, pick("e4m3", "int8"), pick(64, 128, 256), kv * group, kv, pick(16, 32, 64, 128, 256), lens, new, seed,
                extra_rows=pick(0, 2))
    p.poison()
    p.check(p.run(max_new=pick(0, p.new, p.new + 3), max_len=pick(0, p.longest, 4 * p.longest)))


PROMPT_TILES = [("whole", 128, 2, 1, 64, [300], [100]), ("whole", 256, 4, 2, 16, [200, 90], [60, 90]),
                ("shared", 64, 2, 1, 32, [2300], [80]), ("shared", 128, 3, 1, 128, [2100, 40], [40, 1]),
                ("wide", 64, 512, 128, 16, [300, 140], [70, 110]), ("wide", 128, 512, 128, 64, [300, 140], [70, 110])]


@pytest.mark.parametrize("values", ["apart", "zeros"])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("tiles,dim,heads,kv_heads,bs,lens,new", PROMPT_TILES,
                         ids=[f"{t[0]}_{t[1]}" for t in PROMPT_TILES])
def test_prompts_with_value_scales_far_apart(gpu, values, fmt, tiles, dim, heads, kv_heads, bs, lens, new):
    """Prompts' tiles, one workgroup to a sequence and shared out, of 128 and 256 rows: a block whose values are
    small or zero has its whole share of the softmax's sum.  "apart": value scales 2^20 and 2^40 apart; "zeros": all
    blocks behind each request's first hold zeros at the scale kv_append gives them."""
    p = Problem(gpu, fmt, dim, heads, kv_heads, bs, lens, new, 2100 + dim, spread=0.0)
    if values == "apart":
        e = torch.arange(p.scales.shape[1]) % 3
        p.scales[1] *= torch.exp2(torch.tensor([0.0, -40.0, -20.0]))[e][:, None]
    else:
        small = p.tables[:, 1:].flatten()
        small = small[small >= 0].long()
        p.codes[1].view(torch.uint8)[small] = 0
        p.scales[1, small] = sv.MIN_SCALE
    p.poison()
    if tiles == "wide":
        check_heads(p, p.run(), [0, 127])
    else:
        p.check(p.run())


@pytest.mark.parametrize("lens,new", [([3000], [64]), ([3000, 40], [1, 1]), ([2500, 700, 0], [70, 3, 0]), ([90], [1])])
def test_workspace_of_the_largest_step(gpu, lens, new):
    """C callers size their workspace once: a call with the same bounds and fewer tokens, or with bounds of its own,
    finds it large enough and writes nothing behind it."""
    p = Problem(gpu, "e4m3", 128, 4, 2, 64, lens, new, 2200 + sum(lens))
    p.poison()
    lib = capi()
    size = lib.gdsllm_kv_attention_workspace_size(4, 4, 2, 128, 4096, 4096)
    t = [x.to(gpu) for x in (p.q, p.codes[0], p.codes[1], p.scales[0], p.scales[1], p.tables, p.lens, p.starts)]
    q, k, v, ks, vs, tables, lens_d, starts = t
    cache = KvCache8(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), k.shape[0], 2, 64, 128, 0)
    for max_new, max_len in ((4096, 4096), (p.new, p.longest), (0, 0)):
        ws, out = torch.full((size + 4096,), 0x5A, dtype=torch.uint8, device=gpu), torch.full_like(q, 9.0)
        torch.cuda.synchronize()
        rc = lib.gdsllm_kv_attention(ctypes.byref(cache), q.data_ptr(), 512, out.data_ptr(), 512, q.shape[0], 4,
                                     tables.data_ptr(), tables.shape[1], tables.shape[1], lens_d.data_ptr(),
                                     starts.data_ptr(), len(lens), p.scale, max_new, max_len, 1, ws.data_ptr(), size,
                                     torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.gdsllm_last_error().decode()
        p.check(out)
        assert bool((ws[size:] == 0x5A).all())


LONG_TAILS = [("decode", 64, 2, 1, 16, [1000], [1]), ("decode_shared", 128, 2, 2, 64, [3000, 500], [1, 1]),
              ("prompt", 128, 2, 1, 64, [900], [80]), ("prompt_shared", 256, 2, 1, 32, [2200], [70]),
              ("prompt_wide", 64, 512, 128, 16, [200, 100], [70, 70])]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim,heads,kv_heads,bs,lens,new", [t[1:] for t in LONG_TAILS], ids=[t[0] for t in LONG_TAILS])
def test_many_small_weights(gpu, fmt, dim, heads, kv_heads, bs, lens, new):
    """Keys 2^-25.1 of the largest weight, 31 of every 32, with all of the values: they count by their share.  The
    largest weight is taken as 2^7 at least, so theirs are 2^-18.1 and off by half a step of fp16's least, 2^-25;
    the scores' and sums' fp32 and the result add 2^-20 and half an fp16 step."""
    p = Problem(gpu, fmt, dim, heads, kv_heads, bs, lens, new, 2300 + dim, spread=0.0)
    codes = torch.zeros(p.codes.shape)
    codes[0, :, :, 0::32 if bs >= 32 else bs, 0] = 64
    codes[1] = 100 * (codes[0, ..., :1] == 0)
    if bs < 32:  # every other block of 16
        odd = p.tables[:, 1::2].flatten()
        codes[0, odd[odd >= 0].long()], codes[1, odd[odd >= 0].long()] = 0, 100
    p.codes = codes.to(sv.DTYPE[fmt])
    p.scales[0], p.scales[1], p.scale = 1.0, 2.0 ** 8, 1.0
    p.q.zero_()
    p.q[..., 0] = 17.4 / 64
    got = p.run().cpu().double()
    sel = [0] if kv_heads == 128 else range(kv_heads)
    G = heads // kv_heads
    for h in sel:
        vals = p.codes[:, :, h:h + 1].double() * p.scales[:, :, h:h + 1, None, None].double()
        want, _ = sv.attention(p.q[:, h * G:(h + 1) * G], vals[0], vals[1], p.scales[1, :, h:h + 1].double(), p.tables, p.lens,
                               p.starts, p.scale)
        assert float(want.max()) > 0.01
        err = (got[:, h * G:(h + 1) * G] - want).abs()
        weight = 2.0 ** (7 - float(p.q[0, 0, 0]) * 64 * math.log2(math.e))
        assert bool((err <= (2.0 ** -25 / weight + 2.0 ** -11 + 2.0 ** -20) * want + 2.0 ** -25).all()), float((err / want).max())


@pytest.mark.parametrize("lens,new,max_len", [([100, 7], [2, 1], 0), ([2500, 30], [1, 1], 0), ([200], [90], 0)],
                         ids=["whole", "shared", "prompt"])
def test_rows_before_the_first_request(gpu, lens, new, max_len):
    """Some of a batch's requests: the rows of none of them are zero in a new tensor and left alone in a given one."""
    p = Problem(gpu, "e4m3", 64, 4, 2, 32, lens, new, 2400, extra_rows=5)
    p.poison()
    p.starts += 3
    used = [torch.full(p.q.shape, 9.0, dtype=torch.float16, device=gpu) for _ in range(1024)]
    del used  # what a new tensor holds is no zero by chance
    got = p.run(max_len=max_len)
    p.check(got)
    rest = torch.ones(p.q.shape[0], dtype=torch.bool)
    rest[3:3 + sum(new)] = False
    assert bool((got[rest.to(gpu)] == 0).all())
    out = torch.full_like(got, 7.0)
    p.run(max_len=max_len, output=out)
    assert bool((out[rest.to(gpu)] == 7).all()) and torch.equal(out[~rest.to(gpu)], got[~rest.to(gpu)])


@pytest.mark.parametrize("power", [20, 23, 24, 25, 26])
@pytest.mark.parametrize("lens,new", [([700], [1]), ([3000], [1]), ([700], [150]), ([2100], [40])],
                         ids=["decode", "decode_shared", "prompt", "prompt_shared"])
def test_large_scores(gpu, power, lens, new):
    """Scores of 2^power, where fp32 tells neighbours apart by up to 8, that rise a little from one block of 64 tokens to
    the next and then by more than any weight's range: results are means of the values, so no larger than the largest,
    and where one token is far ahead they are its values.  Half an fp16 step for the weight in the product with the
    values (the sum has it unrounded), half a step for the result, 2^-20 for fp32 sums and quotients."""
    heads, bs = 8, 64
    p = Problem(gpu, "int8", 128, 2 * heads, heads, bs, lens, new, 2500, spread=0.0)
    n, step = lens[0], torch.arange(heads)
    codes = torch.zeros(p.codes.shape)
    codes[0, ..., 0] = 100
    for i, page in enumerate(p.tables[0].tolist()):
        codes[0, page, :, :, 1] = i % 16
    codes[1] = p.codes[1].float()
    codes[0, p.tables[0, n // 2 // bs], :, n // 2 % bs, 2] = 127
    p.codes = codes.to(torch.int8)
    p.scales[0] = 16.0
    p.scales[1] = torch.exp2(0.37 * step - 6)
    p.scale = 1.0
    p.q.zero_()
    p.q[..., 0] = 2.0 ** power / 1600
    p.q[..., 1] = (0.05 + 0.04 * torch.arange(2 * heads)).half()  # 1 to 16 in log2 from block to block
    got = p.run().cpu().double()
    top = 127 * p.scales[1, 0].double().repeat_interleave(2)[None, :, None]
    assert bool((got.abs() <= top * (1 + 2.0 ** -9)).all())
    p.q[..., 2] = 1000.0
    got = p.run().cpu().double()
    page, at = int(p.tables[0, n // 2 // bs]), n // 2 % bs
    want = (p.codes[1, page, :, at].double() * p.scales[1, page].double()[:, None]).repeat_interleave(2, 0)
    seen = torch.arange(new[0]) + n - new[0] >= n // 2
    assert bool(((got[seen] - want).abs() <= (2.0 ** -10 + 2.0 ** -20) * want.abs() + 2.0 ** -25).all()) and bool(seen.any())
