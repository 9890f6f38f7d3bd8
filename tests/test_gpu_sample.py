"""Sampling against the plain 64-bit form (oracle/serve.py sample_row): the
same token, except where the form itself says that a cut or the draw lies
within 2^-40 of the kept mass of going the other way (64-bit sums of up to 2^17
weights in another order, each of 2^-52, and whole-number masses of 2^-45)."""

import math

import pytest
import torch

from gdsllm_amd.runtime import ext
from helpers import gen
from oracle import serve as sv

pytestmark = pytest.mark.gpu
NEAR = 2.0 ** -40


def _check(dev, logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    n = logits.shape[0]
    mk = lambda v, t: None if v is None else torch.tensor(v, dtype=t, device=dev)  # noqa: E731
    args = [mk(temperature, torch.float32), mk(top_k, torch.int32), mk(top_p, torch.float32), mk(min_p, torch.float32)]
    ut = torch.tensor(u, dtype=torch.float32)
    got = ext().sample_tokens(logits.to(dev), ut.to(dev), *args)
    assert got.dtype == torch.int64 and got.shape == (n,)
    f32 = lambda v, i, d: d if v is None else float(torch.tensor(v[i], dtype=torch.float32))  # noqa: E731
    for i in range(n):
        want, border = sv.sample_row(logits[i], float(ut[i]), f32(temperature, i, 1.0), 0 if top_k is None else top_k[i],
                                     f32(top_p, i, 1.0), f32(min_p, i, 0.0))
        assert int(got[i]) == want or border < NEAR, (i, int(got[i]), want, border)
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 63, 64, 65, 1000, 1025, 8191, 32000])
def test_sample(gpu, dtype, vocab):
    g = gen(vocab)
    n = 12
    x = (torch.randn(n, vocab, generator=g) * 2 + 9 * torch.rand(n, vocab, generator=g) ** 20).to(dtype)
    u = torch.rand(n, generator=g).tolist()
    k = [0, 1, 5, vocab, vocab + 3, -1, 40, 2, 0, 7, 1000, 50]
    p = [1.0, 0.9, 0.5, 0.0, 0.999, 1.5, 0.95, -1.0, 0.3, 0.8, 0.9, 1.0]
    m = [0.0, 0.05, 0.5, 0.0, 1.0, 0.0, 0.1, 0.0, 2.0, 0.0, 0.01, -1.0]
    t = [1.0, 0.7, 1.5, 0.2, 1.0, 0.9, 2.0, 0.8, 100.0, 0.0, 0.6, -1.0]
    _check(gpu, x, u)
    _check(gpu, x, u, t)
    _check(gpu, x, u, None, k)
    _check(gpu, x, u, None, None, p)
    _check(gpu, x, u, None, None, None, m)
    _check(gpu, x, u, t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_ties(gpu, dtype):
    """Equal logits stand in the order of their index, in every cut and in the draw."""
    vocab, n = 700, 16
    x = torch.zeros(n, vocab, dtype=dtype)
    x[1::2] = (torch.arange(vocab) % 3).to(dtype)
    x[2, ::2] = -0.0
    u = [i / n for i in range(n)]
    _check(gpu, x, u)
    _check(gpu, x, u, None, [0, 3, 500, 233, 234, 235, 466, 467, 1, 2, 10, 699, 700, 701, 0, 0])
    _check(gpu, x, u, None, None, [0.5, 0.25, 0.75, 0.1, 0.9, 0.3, 0.01, 0.99] * 2)
    got = _check(gpu, x, u, [0.0] * n)
    assert got.tolist() == [0, 2] * 8


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_special_values(gpu, dtype):
    inf, nan = math.inf, math.nan
    rows = [[nan, -inf, nan, -inf], [nan, 1.0, -inf, nan], [inf, 1.0, inf, -inf], [-inf, -65504.0, 65504.0, nan],
            [1.0, 1.0, nan, nan], [-0.0, 0.0, -inf, -inf], [inf, inf, inf, inf], [6e-8, 0.0, -6e-8, -inf]]
    x = torch.tensor(rows).to(dtype)
    for u in (0.0, 0.3, 0.6, 0.99999994):
        for t in (None, [0.5] * 8, [1e-30] * 8, [float("inf")] * 8, [nan] * 8, [0.0] * 8):
            got = _check(gpu, x, [u] * 8, t)
            assert int(got[0]) == -1 and int(got[1]) == 1
    # uniforms outside [0, 1) are taken as its ends
    one = torch.randn(6, 50, generator=gen(1)).to(dtype)
    ends = ext().sample_tokens(one.to(gpu), torch.tensor([-1.0, nan, 0.0, 1.0, 7.0, 1.0], device=gpu))
    first, last = one.argmax(1), one.argmin(1)
    assert ends.tolist() == torch.cat([first[:3], last[3:]]).tolist()


@pytest.mark.parametrize("vocab", [65535, 65536, 70001, 131072])
def test_more_equal_logits_than_a_counter_holds(gpu, vocab):
    """All equal, all but one equal: 65536 tokens of one value and more."""
    n = 4
    x = torch.full((n, vocab), 1.5).half()
    x[1, vocab // 2] = 3.0
    x[2, 5] = -math.inf
    x[3] = torch.randn(vocab, generator=gen(vocab)).half()
    u = [0.999, 0.7, 0.25, 0.5]
    _check(gpu, x, u)
    _check(gpu, x, u, [0.7] * 4, [65000, 66000, 0, 100], [0.99, 0.5, 0.9, 0.9])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_strides_and_shapes(gpu, dtype):
    g = gen(77)
    wide = torch.randn(9, 1111, generator=g).to(dtype).to(gpu)
    u = torch.rand(9, generator=g).to(gpu)
    want = ext().sample_tokens(wide[:, 3:1004].contiguous(), u)
    assert torch.equal(ext().sample_tokens(wide[:, 3:1004], u), want)  # rows off the 16-byte grid
    assert torch.equal(ext().sample_tokens(wide[:, 3:1004].t().contiguous().t(), u), want)
    got = ext().sample_tokens(wide[:, 3:1004].reshape(3, 3, 1001), u.view(3, 3))
    assert got.shape == (3, 3) and torch.equal(got.view(-1), want)
    assert ext().sample_tokens(wide[:0], u[:0]).shape == (0,)
    many = wide[:1, :40].expand(5000, 40).contiguous()
    uu = torch.rand(5000, generator=g).to(gpu)
    got = ext().sample_tokens(many, uu)
    for i in range(0, 5000, 500):
        assert int(got[i]) == sv.sample_row(many[0].cpu(), float(uu[i]))[0]


def test_frequencies(gpu):
    """Over an even grid of uniforms every kept token is drawn as often as its weight says, to one draw."""
    vocab, n = 50, 4096
    x = torch.randn(vocab, generator=gen(88)).half()
    u = (torch.arange(n) + 0.5) / n
    got = ext().sample_tokens(x.expand(n, vocab).contiguous().to(gpu), u.float().to(gpu))
    share = torch.bincount(got.cpu(), minlength=vocab).double()
    want = torch.softmax(x.double(), 0) * n
    assert bool(((share - want).abs() <= 1.0 + 1e-3).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [32752, 32753, 40000, 128257, 200003, 2 ** 20])
def test_large_vocabularies(gpu, dtype, vocab):
    """Rows in registers and not, and fp32 rows of which a 4096th of the keys' range holds more than the list."""
    x = torch.randn(4, vocab, generator=gen(vocab))
    x[1] = 1.0 + 1e-4 * x[1]
    x[2] *= 0.05
    u = [0.5, 0.123, 0.999, 0.25]
    _check(gpu, x.to(dtype), u)
    _check(gpu, x.to(dtype), u, [0.8, 1.0, 0.3, 0.0], [0, 20000, 5, 0], [0.95, 0.9, 1.0, 1.0], [0.0, 0.0, 0.01, 0.5])
