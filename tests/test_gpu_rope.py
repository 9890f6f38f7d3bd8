"""The rotation of q and k against its 64-bit form (oracle/serve4.py), whose
values it must have bit for bit: products are exact in 64 bits, and both go
from there to fp32 and to fp16."""

import pytest
import torch

from gdsllm_amd.runtime import ext
from helpers import gen
from oracle import serve4 as s4

pytestmark = pytest.mark.gpu


def problem(tokens, heads, kv_heads, dim, rotary, seed, table=300, pad=True):
    g = gen(seed)
    q, k = (torch.randn(tokens, h, dim, generator=g).half() for h in (heads, kv_heads))
    angle = torch.rand(table, rotary // 2, generator=g) * 6.3
    pos = torch.randint(0, table, (tokens,), generator=g).int()
    if pad and tokens > 2:
        pos[1], pos[tokens - 1] = -1, table  # neither has a position
    return q, k, pos, angle.cos(), angle.sin()


def check(gpu, q, k, pos, cos, sin, neighbours, **kw):
    d = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    got = ext().rope(d(q), d(k), d(pos), d(cos), d(sin), neighbours, **kw)
    for x, y in zip((q, k), got):
        assert (x is None) == (y is None)
        if x is not None:
            assert torch.equal(y.cpu(), s4.rotate(x, pos, cos, sin, neighbours)[0])


SIZES = [(128, 128), (128, 64), (64, 64), (256, 64), (80, 32), (96, 24), (80, 20), (192, 192), (64, 2), (10, 6), (1024, 1024),
         (2, 2), (256, 16)]


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("dim,rotary", SIZES, ids=[f"{a}_{b}" for a, b in SIZES])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (3, 8, 1), (37, 5, 3), (300, 64, 8)])
def test_sizes(gpu, neighbours, dim, rotary, tokens, heads, kv_heads):
    if dim * tokens * heads > 2 ** 22:
        heads, kv_heads = 5, 2
    check(gpu, *problem(tokens, heads, kv_heads, dim, rotary, dim + rotary + tokens), neighbours)


@pytest.mark.parametrize("neighbours", [False, True])
def test_without_k_and_without_tokens(gpu, neighbours):
    q, _, pos, cos, sin = problem(5, 3, 1, 64, 64, 1)
    check(gpu, q, None, pos, cos, sin, neighbours)
    check(gpu, q[:0], None, pos[:0], cos, sin, neighbours)
    check(gpu, q[:0], q[:0], pos[:0], cos, sin, neighbours)
    check(gpu, q, q[:, :0], pos, cos, sin, neighbours)


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_rows_of_one_projection(gpu, neighbours, shift):
    """q and k as parts of wider rows, on the 16-byte grid and off it; in place, what lies beside them stays."""
    q, k, pos, cos, sin = problem(40, 6, 2, 64, 32, 7)
    wide = torch.full((40, 16 * 64 + 16), 5.0, dtype=torch.float16)
    wide[:, shift:shift + 384] = q.flatten(1)
    wide[:, shift + 384:shift + 512] = k.flatten(1)
    row = wide.to(gpu)
    qv, kv = row[:, shift:shift + 384].unflatten(1, (6, 64)), row[:, shift + 384:shift + 512].unflatten(1, (2, 64))
    args = [t.to(gpu) for t in (pos, cos, sin)]
    want = [s4.rotate(x, pos, cos, sin, neighbours)[0] for x in (q, k)]
    got = ext().rope(qv, kv, *args, neighbours)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want)) and torch.equal(row.cpu(), wide)
    got = ext().rope(qv, kv, *args, neighbours, True)
    assert got[0].data_ptr() == qv.data_ptr() and got[1].data_ptr() == kv.data_ptr()
    assert all(torch.equal(a.cpu(), b) for a, b in zip((qv, kv), want))
    wide[:, shift:shift + 384], wide[:, shift + 384:shift + 512] = want[0].flatten(1), want[1].flatten(1)
    assert torch.equal(row.cpu(), wide)


def test_in_place_needs_rows_to_write(gpu):
    q, k, pos, cos, sin = (t.to(gpu) for t in problem(4, 2, 2, 64, 64, 9))
    for bad in (q.transpose(0, 1).contiguous().transpose(0, 1), q[:, :, ::2], q[:1].expand(4, 2, 64)):
        c = cos if bad.shape[2] == 64 else cos[:, :16].contiguous()
        s = sin if bad.shape[2] == 64 else sin[:, :16].contiguous()
        with pytest.raises(RuntimeError, match="in place"):
            ext().rope(bad, None, pos, c, s, False, True)
        assert torch.equal(ext().rope(bad, None, pos, c, s)[0].cpu(), s4.rotate(bad.cpu(), pos.cpu(), c.cpu(), s.cpu())[0])


def test_special_values(gpu):
    """Infinities and NaN stay in their pairs; small and large values; a rotation that cancels."""
    q, k, pos, cos, sin = problem(6, 2, 1, 64, 64, 11, pad=False)
    q[0, 0, 3], q[1, 1, 40] = float("inf"), float("nan")
    q[2] *= 2.0 ** -14
    k[3] = 65504.0
    k[4] = 1.0
    cos[pos[4].long()], sin[pos[4].long()] = 0.70710677, 0.70710677
    for nb in (False, True):
        got = ext().rope(*(t.to(gpu) for t in (q, k, pos, cos, sin)), nb)
        for x, y in zip((q, k), got):
            want = s4.rotate(x, pos, cos, sin, nb)[0]
            assert torch.equal(y.cpu().nan_to_num(7), want.nan_to_num(7)) and torch.equal(y.cpu().isnan(), want.isnan())


def test_another_stream_and_a_graph(gpu):
    q, k, pos, cos, sin = problem(33, 8, 2, 128, 128, 13)
    d = [t.to(gpu) for t in (q, k, pos, cos, sin)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = ext().rope(*d, True)
    s.synchronize()
    assert torch.equal(out[0].cpu(), s4.rotate(q, pos, cos, sin, True)[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ext().rope(*d)
    for i in range(3):
        pos = (pos + 1) % 300
        d[2].copy_(pos)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0].cpu(), s4.rotate(q, pos, cos, sin)[0]) and torch.equal(out[1].cpu(), s4.rotate(k, pos, cos, sin)[0])


def test_refusals(gpu):
    q, k, pos, cos, sin = (t.to(gpu) for t in problem(4, 2, 2, 64, 64, 15))
    bad = [((q.float(), k, pos, cos, sin), "q must be"), ((q, k[:3], pos, cos, sin), "k must be"),
           ((q, k, pos.long(), cos, sin), "positions"), ((q, k, pos[:3], cos, sin), "positions"),
           ((q, k, pos, cos.half(), sin), "cos"), ((q, k, pos, cos[0], sin), "cos"), ((q, k, pos, cos, sin[:9]), "sin"),
           ((q, k, pos, cos, sin.view(-1, 150)), "differ"), ((q[:, :0], k, pos, cos, sin), "no heads"),
           ((q, k, pos.cpu(), cos, sin), "positions"), ((q[..., :32], k[..., :32], pos, cos, sin), "rotary")]
    for args, word in bad:
        with pytest.raises(RuntimeError, match=word):
            ext().rope(*args)


@pytest.mark.parametrize("neighbours", [False, True])
def test_in_place_k_is_not_q(gpu, neighbours):
    """q and k that share memory are refused in place; rows between each other's, from either side, are not."""
    q, _, pos, cos, sin = problem(9, 4, 4, 64, 64, 17)
    d = [t.to(gpu) for t in (q, pos, cos, sin)]
    with pytest.raises(RuntimeError, match="overlap"):
        ext().rope(d[0], d[0], *d[1:], neighbours, True)
    with pytest.raises(RuntimeError, match="overlap"):
        ext().rope(d[0][:, :3], d[0][:, 2:], *d[1:], neighbours, True)
    assert torch.equal(d[0].cpu(), q)
    want = s4.rotate(q, pos, cos, sin, neighbours)[0]
    for cut in (1, 2, 3):
        for first in (True, False):
            x = q.to(gpu)
            a, b = (x[:, :cut], x[:, cut:]) if first else (x[:, cut:], x[:, :cut])
            ext().rope(a, b, *d[1:], neighbours, True)
            assert torch.equal(x.cpu(), want)
    # the same heads twice, into new tensors
    assert all(torch.equal(y.cpu(), want) for y in ext().rope(d[0], d[0], *d[1:], neighbours))


def test_gradients_and_versions(gpu):
    """There is no backward pass: what autograd would follow is refused, and in place it learns of the write."""
    q, k, pos, cos, sin = problem(5, 3, 1, 64, 64, 19)
    d = [t.to(gpu) for t in (q, k, pos, cos, sin)]
    for i, name in enumerate("qk"):
        for inplace in (False, True):
            a = list(d)
            a[i] = (a[i].clone().requires_grad_() * 1.0)
            with pytest.raises(RuntimeError, match=f"rope: {name} needs a gradient"):
                ext().rope(*a, False, inplace)
            with torch.no_grad():
                got = ext().rope(*a)
            assert not got[i].requires_grad and torch.equal(got[i].cpu(), s4.rotate((q, k)[i], pos, cos, sin)[0])
    w = torch.ones(64, dtype=torch.float16, device=gpu, requires_grad=True)
    x, y = d[0].clone(), d[1].clone()
    z, u = x * w, y * w
    ext().rope(x, y, *d[2:], False, True)
    for t in (z, u):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            t.float().sum().backward()
    z = d[0] * w
    ext().rope(d[0], d[1], *d[2:])  # into new tensors: q stays
    z.float().sum().backward()
    with torch.inference_mode():
        x = d[0] * 1.0
    ext().rope(x, None, *d[2:], False, True)
    assert torch.equal(x.cpu(), s4.rotate(q, pos, cos, sin)[0])
