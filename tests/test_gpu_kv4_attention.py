"""Attention over the 4-bit cache against the plain 64-bit form
(oracle/serve4.py attention, which derives the bound its results are held to)."""

import ctypes
import math

import pytest
import torch

from gdsllm_amd import KvCache4, capi
from gdsllm_amd.runtime import ext
from helpers import gen
from oracle import serve as sv
from oracle import serve4 as s4

pytestmark = pytest.mark.gpu


class Problem:
    def __init__(self, dev, group, dim, heads, kv_heads, bs, lens, new, seed, extra_rows=0, qscale=1.0):
        g = gen(seed)
        counts = [sv.blocks(n, bs) for n in lens]
        pool = sum(counts) + 2
        self.k, self.v = (torch.randint(0, 256, (pool, kv_heads, bs, dim // 2), generator=g).to(torch.uint8) for _ in range(2))
        pairs = torch.randn(2, pool, kv_heads, dim // group, bs, 2, generator=g)
        pairs[..., 0] = 0.2 * torch.exp(0.5 * pairs[..., 0])  # a range of 15 scales about zero
        pairs[..., 1] = -7.5 * pairs[..., 0] + 0.3 * pairs[..., 1]
        self.ka, self.va = pairs.half()
        ids = torch.randperm(pool, generator=g)
        self.tables = torch.full((len(lens), max(1, max(counts))), -1, dtype=torch.int32)
        at = 0
        for b, c in enumerate(counts):
            self.tables[b, :c] = ids[at:at + c].int()
            at += c
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.starts = torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32)
        self.q = (torch.randn(sum(new) + extra_rows, heads, dim, generator=g) * qscale).half()
        self.scale, self.dev, self.bs = dim ** -0.5, dev, bs
        self.new, self.longest = max(new), max(lens)

    def poison(self):
        """Everything behind a request's last token, and blocks nobody holds: pairs that are no numbers."""
        held = torch.zeros(self.k.shape[0], self.bs, dtype=torch.bool)
        for row, n in zip(self.tables.tolist(), self.lens.tolist()):
            for i in range(n):
                held[row[i // self.bs], i % self.bs] = True
        for pair, bad in ((self.ka, float("nan")), (self.va, float("inf"))):
            pair.copy_(torch.where(held[:, None, None, :, None], pair, torch.tensor(bad).half()))

    def args(self):
        return [t.to(self.dev) for t in (self.q, self.k, self.v, self.ka, self.va, self.tables, self.lens, self.starts)]

    def run(self, max_new=None, max_len=None, **kw):
        return ext().kv4_attention(*self.args(), self.scale, self.new if max_new is None else max_new,
                                   self.longest if max_len is None else max_len, **kw)

    def check(self, got, heads=None):
        kv, vv = (torch.nan_to_num(s4.elements(c, p), 0.0, 0.0, 0.0) for c, p in ((self.k, self.ka), (self.v, self.va)))
        want, bound = s4.attention(self.q, kv, vv, self.tables, self.lens, self.starts, self.scale, heads)
        got = got.cpu().double()
        if heads is not None:
            G = self.q.shape[1] // self.k.shape[1]
            sel = (torch.tensor(heads)[:, None] * G + torch.arange(G)).flatten()
            got, want, bound = got[:, sel], want[:, sel], bound[:, sel]
        err = (got - want).abs()
        assert bool((err <= bound).all()), f"worst {float((err / bound.clamp(min=2.0 ** -25)).max()):.3f} of the bound"


HEADS = [(64, 4, 4, 32), (128, 8, 1, 64), (128, 6, 2, 32), (256, 16, 1, 128), (128, 7, 7, 128), (64, 40, 2, 64), (256, 2, 2, 32)]


@pytest.mark.parametrize("dim,heads,kv_heads,group", HEADS, ids=[f"d{d}_{h}x{k}_g{g}" for d, h, k, g in HEADS])
@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
def test_decode(gpu, dim, heads, kv_heads, group, bs):
    """One new token a request: lengths about a block's and a tile's edge, an idle slot among them."""
    lens = [1, 15, 16, 17, 0, 31, 33, 63, 64, 65, 127, 129, 255, 257, 300]
    p = Problem(gpu, group, dim, heads, kv_heads, bs, lens, [0 if n == 0 else 1 for n in lens], 200 + dim + bs)
    p.poison()
    p.check(p.run())


@pytest.mark.parametrize("dim,heads,kv_heads,bs,group", [(128, 4, 1, 64, 64), (64, 8, 8, 16, 32), (256, 4, 2, 128, 128),
                                                         (256, 4, 1, 32, 64)])
def test_decode_split(gpu, dim, heads, kv_heads, bs, group):
    """Sequences long enough to be split, the last unit short; the bound on the length loose, right and too small."""
    p = Problem(gpu, group, dim, heads, kv_heads, bs, [2100, 513, 5, 1024], [1, 1, 1, 1], 300 + dim)
    p.poison()
    for o in [p.run(), p.run(max_len=0), p.run(max_len=300), p.run(max_new=0)]:
        p.check(o)


@pytest.mark.parametrize("dim,heads,kv_heads,bs,group", [(128, 4, 1, 64, 64), (64, 3, 3, 16, 32), (256, 4, 2, 128, 128),
                                                         (128, 14, 2, 32, 32), (256, 3, 1, 64, 32)])
@pytest.mark.parametrize("lens,new", [([5, 300, 64, 129], [5, 2, 64, 100]), ([200], [200]), ([17, 0, 40], [1, 0, 33]),
                                      ([400, 3], [3, 3])], ids=["ragged", "whole", "mixed", "few"])
def test_prompts(gpu, dim, heads, kv_heads, bs, group, lens, new):
    """Several new tokens a request, behind what its cache holds; rows see the tokens up to their own."""
    p = Problem(gpu, group, dim, heads, kv_heads, bs, lens, new, 400 + dim + bs)
    p.poison()
    p.check(p.run())


def test_rows_that_see_nothing_and_rows_behind_the_last(gpu):
    """More rows than tokens (a request that was not served): the first rows see nothing and are zero.  Rows behind
    the last request are zero in a new tensor and left alone in a given one."""
    p = Problem(gpu, 64, 128, 4, 2, 16, [3, 0, 20], [5, 2, 1], 500, extra_rows=6)
    p.poison()
    got = p.run()
    p.check(got)
    assert bool((got[:2] == 0).all()) and bool((got[5:7] == 0).all()) and bool((got[8:] == 0).all())
    wide = torch.full((14, 4 * 128 + 64), 7.0, dtype=torch.float16, device=gpu)
    out = wide[:, :4 * 128].unflatten(1, (4, 128))
    assert p.run(output=out).data_ptr() == out.data_ptr()
    p.check(torch.cat([out[:8], torch.zeros_like(out[8:])]))
    assert bool((wide[8:] == 7).all()) and bool((wide[:, 512:] == 7).all())


def test_blocks_outside_the_cache_have_no_weight(gpu):
    p = Problem(gpu, 32, 64, 2, 1, 16, [40], [1], 700)
    keep = p.tables.clone()
    p.tables[0, 1] = 10 ** 9
    got = p.run()
    # the same as with the block's tokens left out: one softmax over the rest
    ids = torch.stack([keep[0, 0], keep[0, 2]]).long()
    k, v = (s4.elements(c, a)[ids, 0].reshape(-1, 64)[:24] for c, a in ((p.k, p.ka), (p.v, p.va)))
    for h in range(2):
        o = torch.softmax((k @ p.q[0, h].double()) * p.scale, 0) @ v
        assert float((got[0, h].cpu().double() - o).norm() / o.norm()) < 2e-3


def test_equal_keys_and_special_values(gpu):
    """Zero queries take the mean; groups without a range; q without any number gives none."""
    p = Problem(gpu, 64, 64, 2, 2, 16, [20, 20], [1, 1], 800)
    p.q[0] = 0.0
    p.va[..., 0] = 0.0
    p.q[1, 0, 5] = float("nan")
    got = p.run()
    assert bool(got[1, 0].isnan().all()) and bool(got[1, 1].isfinite().all())
    p.q[1, 0, 5] = 0.0
    p.check(p.run())
    assert torch.equal(p.run()[0], got[0])


def test_strided_q_and_tables_on_another_stream(gpu):
    """q inside a fused projection's rows, tables inside a wider tensor, on a stream of the caller's."""
    p = Problem(gpu, 32, 128, 4, 2, 32, [100, 7], [2, 1], 900)
    wide = torch.randn(3, 8 * 128).half().to(gpu)
    wide[:, :512] = p.q.flatten(1).to(gpu)
    tabs = torch.full((2, 9), -3, dtype=torch.int32, device=gpu)
    tabs[:, :p.tables.shape[1]] = p.tables.to(gpu)
    a = p.args()
    a[0], a[5] = wide[:, :512].unflatten(1, (4, 128)), tabs[:, :p.tables.shape[1]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ext().kv4_attention(*a, p.scale)
    s.synchronize()
    p.check(got)


def test_long_cache_past_32_bits(gpu):
    """Blocks whose codes lie behind 4 GiB."""
    dim, bs, heads = 256, 256, 16
    blocks = 2 ** 32 // (heads * bs * dim // 2) + 2
    small = Problem(gpu, 32, dim, heads, heads, bs, [200], [1], 1000)
    big = [torch.zeros(blocks, *t.shape[1:], dtype=t.dtype, device=gpu) for t in (small.k, small.v, small.ka, small.va)]
    for b, t in zip(big, (small.k, small.v, small.ka, small.va)):
        b[-1] = t[small.tables[0, 0].item()].to(gpu)
    a = small.args()
    tables = torch.tensor([[blocks - 1]], dtype=torch.int32, device=gpu)
    small.check(ext().kv4_attention(a[0], *big, tables, a[6], a[7], small.scale))


def repeated(p, lens, new, seed):
    """The problem's blocks, in any order and again and again, as long sequences."""
    width = max(sv.blocks(n, p.bs) for n in lens)
    p.tables = torch.randint(0, p.k.shape[0], (len(lens), width), generator=gen(seed)).int()
    p.lens = torch.tensor(lens, dtype=torch.int32)
    p.starts = torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32)
    p.q = torch.randn(sum(new), *p.q.shape[1:], generator=gen(seed + 1)).half()
    p.new, p.longest = max(new), max(lens)


@pytest.mark.parametrize("max_new,max_len", [(1, 0), (0, 4000), (2, 3000), (17, 2500), (1, 16)])
def test_bounds_smaller_than_the_requests(gpu, max_new, max_len):
    """The host's bounds only say how the work is split: requests with more rows and tokens than they say, where
    sequences are shared out and where not."""
    p = Problem(gpu, 64, 64, 4, 2, 32, [2500, 40, 0, 3000, 700], [7, 20, 0, 1, 33], 1200)
    p.poison()
    p.check(p.run(max_new=max_new, max_len=max_len))


def test_more_requests_than_a_step_of_the_sums(gpu):
    """More than 256 requests share one line of work."""
    lens = [(37 * i) % 90 for i in range(299)] + [2600, 5]
    p = Problem(gpu, 32, 64, 2, 1, 64, lens, [min(1, n) for n in lens], 1300)
    p.poison()
    p.check(p.run())


@pytest.mark.parametrize("dim,heads,kv_heads,bs,group", [(64, 4, 2, 16, 32), (128, 2, 2, 64, 64), (256, 6, 2, 128, 128)])
def test_long_prompts_share_the_work(gpu, dim, heads, kv_heads, bs, group):
    """Few sequences past 2048 tokens: every tile's keys lie in several workgroups' shares, rows that see none of
    a share among them; requests of few rows beside them."""
    p = Problem(gpu, group, dim, heads, kv_heads, bs, [2300, 70, 2100, 180], [150, 2, 1, 180], 1400 + dim)
    p.poison()
    p.check(p.run())


@pytest.mark.parametrize("dim,group", [(64, 32), (128, 64)])
def test_many_sequences_take_the_widest_tiles(gpu, dim, group):
    """512 and more (request, kv head, 256 rows): the last rows of a tile ragged, a request with few rows."""
    p = Problem(gpu, group, dim, 512, 128, 16, [130, 65, 7], [100, 65, 2], 1500 + dim)
    p.poison()
    p.check(p.run(), [0, 77, 127])


@pytest.mark.parametrize("dim,group,bs,lens,new", [(128, 64, 32, [1300, 900], [70, 65]), (64, 32, 16, [1100, 5, 1500], [80, 3, 33]),
                                                   (128, 128, 256, [1029], [200]), (64, 64, 64, [70, 2100], [70, 129])])
def test_the_widest_tiles_share_the_work(gpu, dim, group, bs, lens, new):
    """128 to 511 (request, kv head, 256 rows) past 1024 tokens: parts of 256-row tiles, which begin and end inside
    the tiles of tokens, rows that see none of a part, ragged last rows, a request with few rows beside them."""
    p = Problem(gpu, group, dim, 256, 64, bs, lens, new, 1550 + dim + len(lens))
    p.poison()
    p.check(p.run(), [0, 31, 63])


@pytest.mark.parametrize("dim,max_new,max_len", [(128, 20, 0), (64, 20, 1500), (128, 0, 1100), (128, 30, 40000)])
def test_the_widest_tiles_under_other_bounds(gpu, dim, max_new, max_len):
    """More rows, and longer requests, than the caller said, over work that is shared out in 256-row tiles."""
    p = Problem(gpu, 64, dim, 256, 64, 64, [1700, 1200, 3], [70, 130, 1], 1570 + dim)
    p.poison()
    p.check(p.run(max_new=max_new, max_len=max_len), [0, 31, 63])


def test_whole_sequences_past_a_segment(gpu):
    """Many sequences, so that each has a workgroup of its own, longer than the block table it holds at once."""
    p = Problem(gpu, 128, 256, 1024, 1024, 64, [100, 3], [1, 1], 1600)
    repeated(p, [8300, 3], [1, 1], 1601)
    p.check(p.run(), [0, 500, 1023])
    p = Problem(gpu, 32, 64, 256, 256, 16, [60], [2], 1602)
    repeated(p, [4200], [40], 1603)
    p.check(p.run(), [0, 255])


def test_a_sequence_in_more_parts_than_threads_that_join(gpu):
    """One long sequence among short ones, in hundreds of parts; 256 threads add a row's."""
    lens = [120000] + list(range(1, 32))
    p = Problem(gpu, 64, 64, 16, 1, 256, [1000] * 32, [1] * 32, 1700)
    repeated(p, lens, [1] * 32, 1701)
    p.q *= 0.5
    p.check(p.run(), [0])


def test_two_graphs_on_two_streams(gpu):
    """Captured calls that share their work out keep workspaces apart: replayed side by side, each gives what it
    gives alone."""
    ps = [Problem(gpu, 64, 128, 4, 1, 64, [5000, 3000 + i], [1, 1], 1800 + i) for i in range(2)]
    graphs, outs, args = [], [], []
    for p in ps:
        a = p.args()
        ext().kv4_attention(*a, p.scale)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = ext().kv4_attention(*a, p.scale)
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
            assert torch.equal(o, ext().kv4_attention(*a, p.scale))


def test_one_key_head_for_many_query_heads(gpu):
    """128 query heads over one key head: a single new token fills a tile of 128 rows."""
    p = Problem(gpu, 64, 64, 128, 1, 32, [2500, 100, 0, 3], [1, 1, 0, 1], 1900)
    p.poison()
    p.check(p.run())


def test_no_rows(gpu):
    p = Problem(gpu, 64, 64, 4, 2, 16, [5, 40], [0, 0], 2000)
    assert p.run(max_new=0).shape == (0, 4, 64)
    p = Problem(gpu, 64, 64, 4, 2, 16, [5, 40], [0, 0], 2000, extra_rows=3)
    assert bool((p.run(max_new=0) == 0).all())


@pytest.mark.parametrize("seed", range(32))
def test_drawn_sizes(gpu, seed):
    """Any sizes together: requests idle, decoding and with prompts, bounds given, loose or not at all."""
    g = gen(3000 + seed)
    pick = lambda *v: v[int(torch.randint(len(v), (1,), generator=g))]  # noqa: E731
    kv, heads = pick(1, 2, 3), pick(1, 2, 5, 8)
    n, longest = pick(1, 2, 5, 9), pick(40, 300, 1100, 2600)
    lens = [int(v) for v in torch.randint(0, longest + 1, (n,), generator=g)]
    new = [min(pick(0, 1, 1, 2, 9, 70), m) for m in lens]
    dim = pick(64, 128, 256)
    p = Problem(gpu, min(dim, pick(32, 64, 128)), dim, kv * heads, kv, pick(16, 32, 64, 128, 256), lens, new, seed,
                extra_rows=pick(0, 2))
    p.poison()
    p.check(p.run(max_new=pick(0, p.new, p.new + 3), max_len=pick(0, p.longest, 4 * p.longest)))


@pytest.mark.parametrize("lens,new", [([3000], [64]), ([3000, 40], [1, 1]), ([2500, 700, 0], [70, 3, 0]), ([90], [1])])
def test_workspace_of_the_largest_step(gpu, lens, new):
    """C callers size their workspace once: a call with the same bounds and fewer tokens, or with bounds of its own,
    finds it large enough and writes nothing behind it."""
    p = Problem(gpu, 64, 128, 4, 2, 64, lens, new, 2200 + sum(lens))
    p.poison()
    lib = capi()
    size = lib.gdsllm_kv4_attention_workspace_size(4, 4, 2, 128, 4096, 4096)
    q, k, v, ka, va, tables, lens_d, starts = p.args()
    cache = KvCache4(k.data_ptr(), v.data_ptr(), ka.data_ptr(), va.data_ptr(), k.shape[0], 2, 64, 128, 64)
    for max_new, max_len in ((4096, 4096), (p.new, p.longest), (0, 0)):
        ws, out = torch.full((size + 4096,), 0x5A, dtype=torch.uint8, device=gpu), torch.full_like(q, 9.0)
        torch.cuda.synchronize()
        rc = lib.gdsllm_kv4_attention(ctypes.byref(cache), q.data_ptr(), 512, out.data_ptr(), 512, q.shape[0], 4,
                                      tables.data_ptr(), tables.shape[1], tables.shape[1], lens_d.data_ptr(),
                                      starts.data_ptr(), len(lens), p.scale, max_new, max_len, 1, ws.data_ptr(), size,
                                      torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.gdsllm_last_error().decode()
        p.check(out)
        assert bool((ws[size:] == 0x5A).all())


LONG_TAILS = [("decode", 64, 2, 1, 16, [1000], [1]), ("decode_shared", 128, 2, 2, 64, [3000, 500], [1, 1]),
              ("prompt", 128, 2, 1, 64, [900], [80]), ("prompt_shared", 256, 2, 1, 32, [2200], [70]),
              ("prompt_wide", 64, 512, 128, 16, [200, 100], [70, 70])]


@pytest.mark.parametrize("dim,heads,kv_heads,bs,lens,new", [t[1:] for t in LONG_TAILS], ids=[t[0] for t in LONG_TAILS])
def test_many_small_weights(gpu, dim, heads, kv_heads, bs, lens, new):
    """Keys 2^-25.1 of the largest weight, 15 of every 16, with all of the values: they count by their share.  The
    largest weight is taken as 2^7 at least, so theirs are 2^-18.1 and off by half a step of fp16's least, 2^-25;
    the scores' and sums' fp32 and the result add 2^-20 and half an fp16 step."""
    p = Problem(gpu, 64, dim, heads, kv_heads, bs, lens, new, 2300 + dim)
    code = torch.zeros(2, *p.k.shape[:3], dim)
    code[0, :, :, 0::16, 0] = 15
    code[1] = 10.0 * (code[0, ..., :1] == 0)
    p.k, p.v = s4.pack(code[0].to(torch.uint8)), s4.pack(code[1].to(torch.uint8))
    p.ka[..., 0], p.ka[..., 1], p.va[..., 0], p.va[..., 1] = 4.0, 0.0, 1024.0, 0.0
    p.scale = 1.0
    p.q.zero_()
    p.q[..., 0] = 17.4 / 60
    got = p.run().cpu().double()
    sel = [0] if kv_heads == 128 else list(range(kv_heads))
    G = heads // kv_heads
    want, _ = s4.attention(p.q, s4.elements(p.k, p.ka), s4.elements(p.v, p.va), p.tables, p.lens, p.starts, 1.0, sel)
    cols = (torch.tensor(sel)[:, None] * G + torch.arange(G)).flatten()
    got, want = got[:, cols], want[:, cols]
    assert float(want.max()) > 0.001
    weight = 2.0 ** (7 - float(p.q[0, 0, 0]) * 60 * math.log2(math.e))
    assert bool(((got - want).abs() <= (2.0 ** -25 / weight + 2.0 ** -11 + 2.0 ** -20) * want + 2.0 ** -25).all())


@pytest.mark.parametrize("lens,new,max_len", [([100, 7], [2, 1], 0), ([2500, 30], [1, 1], 0), ([200], [90], 0)],
                         ids=["whole", "shared", "prompt"])
def test_rows_before_the_first_request(gpu, lens, new, max_len):
    """Some of a batch's requests: the rows of none of them are zero in a new tensor and left alone in a given one."""
    p = Problem(gpu, 32, 64, 4, 2, 32, lens, new, 2400, extra_rows=5)
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


@pytest.mark.parametrize("power", [14, 18, 22, 26])
@pytest.mark.parametrize("lens,new", [([700], [1]), ([3000], [1]), ([700], [150]), ([2100], [40])],
                         ids=["decode", "decode_shared", "prompt", "prompt_shared"])
def test_large_scores(gpu, power, lens, new):
    """Scores of 2^power, where fp32 tells neighbours apart by up to 8, that rise from one block of 64 tokens to the
    next: results are means of the values, so no larger than the largest, and where one token is far ahead they are
    its values.  Half an fp16 step for the weight in the product with the values (the sum has it unrounded), half a
    step for the result, 2^-20 for fp32 sums and quotients."""
    heads, bs = 8, 64
    p = Problem(gpu, 64, 128, 2 * heads, heads, bs, lens, new, 2500)
    n = lens[0]
    code = torch.zeros(*p.k.shape[:3], 128)
    code[..., 0] = 10
    for i, page in enumerate(p.tables[0].tolist()):
        code[page, :, :, 1] = i % 16
    code[p.tables[0, n // 2 // bs], :, n // 2 % bs, 2] = 15
    p.k = s4.pack(code.to(torch.uint8))
    p.ka[..., 0], p.ka[..., 1] = 160.0, 0.0
    p.va[..., 1] = 0.0
    p.va[..., 0] = p.va[..., 0].abs().clamp(max=2.0)
    p.scale = 1.0
    p.q.zero_()
    p.q[..., 0] = 2.0 ** power / 1600
    p.q[..., 1] = (0.05 + 0.04 * torch.arange(2 * heads)).half()
    got = p.run().cpu().double()
    assert bool(got.isfinite().all()) and float(got.abs().max()) <= 30 * (1 + 2.0 ** -9)
    p.q[..., 2] = 1000.0
    got = p.run().cpu().double()
    page, at = int(p.tables[0, n // 2 // bs]), n // 2 % bs
    want = s4.elements(p.v, p.va)[page, :, at].repeat_interleave(2, 0)
    seen = torch.arange(new[0]) + n - new[0] >= n // 2
    assert bool(((got[seen] - want).abs() <= (2.0 ** -10 + 2.0 ** -20) * want.abs() + 2.0 ** -25).all()) and bool(seen.any())


def test_refusals(gpu):
    p = Problem(gpu, 32, 64, 4, 2, 16, [20, 20], [1, 1], 2600)
    q, k, v, ka, va, t, n, st = p.args()
    bad = [((q.float(), k, v, ka, va, t, n, st), "q must be"), ((q[..., :32], k, v, ka, va, t, n, st), "q must be"),
           ((q[:, :3], k, v, ka, va, t, n, st), "multiple of kv_heads"), ((q, k[..., :16], v, ka, va, t, n, st), "k_cache"),
           ((q, k, v, ka[:1], va, t, n, st), "affine"), ((q, k, v, ka, va, t.long(), n, st), "block_tables"),
           ((q, k, v, ka, va, t[:1], n, st), "block_tables"), ((q, k, v, ka, va, t, n.cpu(), st), "lens"),
           ((q, k, v, ka, va, t, n, st[:2]), "starts")]
    for args, word in bad:
        with pytest.raises(RuntimeError, match=word):
            ext().kv4_attention(*args, 0.1)
    with pytest.raises(RuntimeError, match="scale"):
        ext().kv4_attention(q, k, v, ka, va, t, n, st, 0.0)
    with pytest.raises(RuntimeError, match="output"):
        ext().kv4_attention(q, k, v, ka, va, t, n, st, 0.1, output=torch.empty_like(q)[:1])


def test_gradients_and_versions(gpu):
    """There is no backward pass: a q that autograd would follow is refused, and it learns of a written output."""
    p = Problem(gpu, 32, 64, 4, 2, 16, [20, 20], [1, 1], 2700)
    a = p.args()
    for q in (a[0].clone().requires_grad_(), a[0].clone().requires_grad_() * 1.0):
        with pytest.raises(RuntimeError, match="kv4_attention: q needs a gradient"):
            ext().kv4_attention(q, *a[1:], p.scale)
        with torch.no_grad():
            p.check(ext().kv4_attention(q, *a[1:], p.scale))
    out = torch.ones_like(a[0])
    z = out * torch.ones(64, dtype=torch.float16, device=gpu, requires_grad=True)
    ext().kv4_attention(*a, p.scale, output=out)
    p.check(out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.float().sum().backward()


BAD_IDS = (-1, 10 ** 9, -2 ** 31)


def lose(p, *places):
    """Table entries (request, block) that name no block of the cache.  Block 0, which lies where a bad index is taken
    to, is nobody's and its pairs are no numbers."""
    used = set(p.tables[p.tables >= 0].tolist())
    free = next((i for i in range(1, p.k.shape[0]) if i not in used), 1)  # (blocks that occur again and again: any)
    if 0 in used and free not in used:
        for t in (p.k, p.v, p.ka, p.va):
            t[free] = t[0]
    p.tables[p.tables == 0] = free
    p.ka[0], p.va[0] = float("nan"), float("inf")
    for i, (b, block) in enumerate(places):
        p.tables[b, block] = (*BAD_IDS, p.k.shape[0])[i % 4]


# dim, heads, kv_heads, bs, group, lens, new, max_len, lost (request, block)
LOST = {
    "decode": (128, 4, 1, 64, 64, [300, 64, 17, 140], [1] * 4, None, [(0, 2), (1, 0), (2, 0), (3, 2), (0, 4)]),
    "decode_256": (256, 4, 2, 16, 128, [300, 16, 33], [1] * 3, None, [(0, 0), (1, 0), (2, 2), (0, 7)]),
    "decode_shared": (128, 4, 1, 32, 32, [2100, 513], [1, 1], None, [(0, 0), (0, 9), (0, 40), (0, 65), (1, 16), (1, 3)]),
    "decode_shared_256": (256, 4, 2, 128, 64, [2100, 700], [1, 2], None, [(0, 3), (0, 16), (1, 0), (1, 5)]),
    "decode_segments": (64, 8, 8, 16, 32, [4500], [1], 500, [(0, 255), (0, 256), (0, 270)]),
    "prompt_64": (64, 4, 1, 16, 32, [300, 129, 20], [200, 100, 20], None, [(0, 0), (0, 5), (0, 12), (0, 18), (1, 0), (1, 1), (2, 1)]),
    "prompt_128": (128, 6, 2, 64, 128, [300, 129], [200, 100], None, [(0, 1), (0, 4), (1, 0)]),
    "prompt_256": (256, 6, 2, 32, 64, [300, 129], [200, 100], None, [(0, 0), (0, 4), (0, 8), (1, 2), (1, 4)]),
    "prompt_wide_64": (64, 512, 128, 16, 64, [130, 65, 7], [100, 65, 2], None, [(0, 0), (0, 5), (0, 8), (1, 0), (2, 0)]),
    "prompt_wide_128": (128, 512, 128, 64, 64, [130, 65, 7], [100, 65, 2], None, [(0, 1), (1, 1)]),
    "prompt_shared_64": (64, 4, 2, 16, 64, [2300, 70, 2100, 180], [150, 2, 1, 180], None,
                         [(0, 0), (0, 60), (0, 64), (0, 140), (1, 4), (2, 7), (3, 1)]),
    "prompt_shared_128": (128, 2, 2, 128, 32, [2300, 70, 2100, 180], [150, 2, 1, 180], None, [(0, 0), (0, 8), (0, 17), (2, 16), (3, 0)]),
    "prompt_shared_256": (256, 6, 2, 32, 128, [2300, 70, 2100, 180], [150, 2, 1, 180], None, [(0, 2), (0, 33), (0, 71), (2, 0), (3, 5)]),
    "prompt_wide_shared_64": (64, 256, 64, 16, 32, [1100, 5, 1500], [80, 3, 33], None, [(0, 0), (0, 33), (0, 68), (2, 50), (2, 93)]),
    "prompt_wide_shared_128": (128, 256, 64, 32, 64, [1300, 900], [70, 65], None, [(0, 0), (0, 20), (0, 40), (1, 27), (1, 3)]),
}


@pytest.mark.parametrize("case", LOST.values(), ids=LOST)
def test_lost_blocks(gpu, case):
    """Blocks outside the cache, the first, the last and some between, have no weight in any kind of tile, whole or
    shared out; rows that see no other block are zero."""
    dim, heads, kv_heads, bs, group, lens, new, max_len, lost = case
    p = Problem(gpu, group, dim, heads, kv_heads, bs, lens, new, 2800 + len(lost))
    p.poison()
    lose(p, *lost)
    p.check(p.run(max_len=max_len), None if kv_heads < 64 else [0, 31, kv_heads - 1])


def mark(p, blocks):
    """Equal keys, and no values but 1024 in one block, request r's number blocks[r]: a row that sees m of its tokens
    among n gets 1024 m / n.  Gives those: [rows, 1, 1]."""
    p.q.zero_()
    p.va.zero_()
    marked = p.k.shape[0] - 1
    p.va[marked, ..., 1] = 1024.0
    p.tables[p.tables == marked] = 0
    want = []
    for r, block in enumerate(blocks):
        p.tables[r, block] = marked
        n = int(p.starts[r + 1] - p.starts[r])
        seen = torch.arange(int(p.lens[r]) - n + 1, int(p.lens[r]) + 1).double()
        want.append(1024 * (seen - block * p.bs).clamp(0, p.bs) / seen)
    return torch.cat(want)[:, None, None]


def check_marks(p, blocks, **kw):
    """Weights are equal powers of two and sums whole numbers of them, exact in fp32; the quotient and its product are
    off by 2^-22, the result by half an fp16 step."""
    want = mark(p, blocks)
    got = p.run(**kw).cpu().double()
    assert bool(((got - want).abs() <= (2.0 ** -11 + 2.0 ** -21) * want + 2.0 ** -25).all()), blocks


SEGMENTS = [(64, 2, 32), (128, 2, 64), (256, 2, 128), (64, 64, 64), (128, 64, 128)]


@pytest.mark.parametrize("bs", [16, 256])
@pytest.mark.parametrize("dim,kv_heads,group", SEGMENTS, ids=[f"d{d}_{'wide' if h > 2 else 'tall'}" for d, h, _ in SEGMENTS])
def test_prompts_past_a_segment(gpu, dim, kv_heads, group, bs):
    """Prompt tiles, of 128 rows (tall) and of 256 (wide), over more tokens than a workgroup holds a block table of at
    once: twice and three times as many.  (The bound of 1000 tokens leaves each sequence to one workgroup.)"""
    lens, new = [4200, 8300, 4096, 4097], [70, 66, 33, 40]
    p = Problem(gpu, group, dim, 2 * kv_heads, kv_heads, bs, [2 * bs] * 4, new, 2900 + dim + bs)
    repeated(p, lens, new, 2901)
    p.check(p.run(max_len=1000), [0, kv_heads - 1])
    lose(p, (0, 4096 // bs), (1, 4096 // bs + 1), (1, 8192 // bs), (3, 0), (2, 4095 // bs))
    p.check(p.run(max_len=1000), [0, kv_heads - 1])


@pytest.mark.parametrize("max_len", [1000, 0], ids=["whole", "shared"])
@pytest.mark.parametrize("bs", [16, 256])
@pytest.mark.parametrize("dim,kv_heads,group", SEGMENTS, ids=[f"d{d}_{'wide' if h > 2 else 'tall'}" for d, h, _ in SEGMENTS])
def test_every_block_counts_once(gpu, dim, kv_heads, group, bs, max_len):
    """In prompt tiles, whole and shared out: the first block, those about a segment's edge, the last, and others
    between count by their share, each row's by the tokens that it sees."""
    lens, new = [4200, 8300, 4097, 8190, 300], [70, 66, 40, 35, 34]
    p = Problem(gpu, group, dim, 2 * kv_heads, kv_heads, bs, [2 * bs] * 5, new, 3000 + dim + bs)
    repeated(p, lens, new, 3001)
    tables, at = p.tables.clone(), [sv.blocks(n, bs) for n in lens]
    edge = 4096 // bs
    for blocks in ([0] * 5, [n - 1 for n in at], [edge - 1, edge - 1, edge, edge, 0], [edge, 2 * edge, 1, edge - 1, at[4] - 1],
                   [at[0] - 2, 2 * edge - 1, edge - 2, edge + 1, at[4] // 2], [at[0] // 2, at[1] // 3, 3, at[3] - 3, 0]):
        p.tables = tables.clone()
        check_marks(p, blocks, max_len=max_len)


def test_every_part_of_a_long_sequence_counts_once(gpu):
    """Hundreds of parts of 256 tokens, a block each, joined by 256 threads (one long sequence among short ones) and by
    1024 (alone): parts about the 256th and the 512th, the first and the last."""
    for lens, blocks in (([120000] + list(range(1, 32)), (0, 1, 63, 64, 255, 256, 257, 300, 467, 468)),
                         ([131000], (0, 1, 16, 255, 256, 257, 500, 510, 511))):
        n = len(lens)
        p = Problem(gpu, 64, 64, 16, 1, 256, [1000] * n, [1] * n, 3100)
        repeated(p, lens, [1] * n, 3101)
        tables = p.tables.clone()
        for block in blocks:
            p.tables = tables.clone()
            check_marks(p, [block] + [0] * (n - 1))


@pytest.mark.parametrize("lens,new", [([2100, 700, 5], [1, 1, 1]), ([1500, 0, 1100], [2, 0, 3]), ([1300, 1030], [4, 1])])
def test_full_tiles_of_wide_heads(gpu, lens, new):
    """16 and more rows of 256 channels over sequences that are shared out, in workgroups of four waves."""
    p = Problem(gpu, 128, 256, 32, 2, 64, lens, new, 3200 + sum(new))
    p.poison()
    p.check(p.run())
    p.check(p.run(max_len=0))


def test_full_tiles_of_wide_heads_in_four_and_eight_waves(gpu):
    """On both sides of the number of tokens to a workgroup that the choice goes by: every part counts once."""
    for lens, blocks in (([30000, 999], (0, 1, 58, 116, 117)), ([140000, 999], (0, 4, 5, 273, 545, 546)),
                         ([60000], (0, 1, 2, 117, 233, 234)), ([100000], (0, 1, 3, 4, 200, 389, 390))):
        n = len(lens)
        p = Problem(gpu, 64, 256, 32, 2, 256, [300] * n, [1] * n, 3300)
        repeated(p, lens, [1] * n, 3301)
        tables = p.tables.clone()
        for block in blocks:
            p.tables = tables.clone()
            check_marks(p, [block, 3][:n])
