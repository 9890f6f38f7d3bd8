"""What pins oracle/serve.py (CPU): torch's own float64 attention, fp8 cast and
complex products, and brute force."""

import math

import pytest
import torch
import torch.nn.functional as F

from oracle import serve as sv


def gen(seed):
    return torch.Generator().manual_seed(seed)


def test_codes_are_torchs_casts():
    x = torch.cat([torch.randn(4000, generator=gen(1)) * s for s in (1e-3, 0.02, 1.0, 200.0, 3000.0)]).double()
    x = torch.cat([x, torch.arange(-32, 33).double() * 2.0 ** -10, torch.tensor([0.0, 448.0, 464.0, 465.0, 1e9]).double()])
    want = x.float().clamp(-448, 448).to(torch.float8_e4m3fn).double()
    assert torch.equal(sv.codes64(x.float().double(), "e4m3"), want)
    assert sv.codes64(torch.tensor([2.5, 3.5, -0.5, 1e9, math.nan, -math.inf]).double(), "int8").tolist() == \
        [2.0, 4.0, -0.0, 127.0, 0.0, -127.0]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_scales(fmt):
    top = sv.QMAX[fmt]
    assert sv.want_scale(0.0, fmt) == 2.0 ** -32
    for e in (-8, 0, 3):
        assert sv.want_scale(top * 2.0 ** e, fmt) == 2.0 ** e
        assert sv.want_scale(top * 2.0 ** e * (1 + 2.0 ** -20), fmt) == 2.0 ** (e + 1)


def test_rotation_is_a_complex_product():
    half, T = 8, 5
    x = torch.randn(T, 2, 24, generator=gen(2)).half()
    angle = torch.randn(9, half, generator=gen(3)).double()
    pos = torch.tensor([0, 8, 3, 3, 1])
    y = sv.rotate(x, pos, angle.cos(), angle.sin())[1]
    z = torch.complex(x[..., :half].double(), x[..., half:16].double()) * torch.polar(torch.ones_like(angle), angle)[pos][:, None]
    torch.testing.assert_close(y, torch.cat([z.real, z.imag, x[..., 16:].double()], -1), rtol=0, atol=1e-14)


@pytest.mark.parametrize("G", [1, 3])
def test_attention_is_torchs(G):
    """Blocks in any order; causal over the last rows; grouped heads."""
    bs, D, Hkv, lens, new = 4, 8, 2, [9, 3], [4, 3]
    k, v = torch.randn(2, 6, Hkv, bs, D, generator=gen(4), dtype=torch.float64)
    tables = torch.tensor([[5, 0, 2], [3, -1, -1]])
    q = torch.randn(sum(new), Hkv * G, D, generator=gen(5)).half()
    out, bound = sv.attention(q, k, v, torch.ones(6, Hkv).double(), tables, torch.tensor(lens), torch.tensor([0, 4, 7]), 0.3)
    at = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        ids = tables[b, :sv.blocks(n, bs)]
        kk, vv = (t[ids].transpose(0, 1).reshape(Hkv, -1, D)[:, :n].repeat_interleave(G, 0) for t in (k, v))
        mask = torch.ones(n, n).tril().bool()[n - m:]
        want = F.scaled_dot_product_attention(q[at:at + m].transpose(0, 1).double(), kk, vv, attn_mask=mask, scale=0.3)
        torch.testing.assert_close(out[at:at + m], want.transpose(0, 1), rtol=1e-12, atol=1e-12)
        at += m
    assert bool((bound > 0).all()) and float(bound.max()) < 0.05


def test_assign_by_hand():
    ring, state = [4, 5, 6, 0, 0], [0, 3]
    tables = [[1, -1, -1], [2, 3, -1], [-1, -1, -1]]
    slots, pos, starts, lens, state = sv.assign([4, 7, 0], [1, -4, 9], tables, ring, state, 4, 12)
    # request 0 takes block 4; request 1 gives block 3 back; request 2 needs three blocks and two are left
    assert slots == [16] + [-1] * 11 and pos == [4] + [-1] * 11
    assert starts == [0, 1, 1, 10] and lens == [5, 3, 0] and state == [1, 3]
    assert tables[0] == [1, 4, -1] and ring == [4, 5, 6, 3, 0]


def test_sampling_by_counting():
    """Each token's share of u is its share of the kept mass, cut by cut."""
    x = torch.tensor([1.0, 3.0, 2.0, 3.0, -math.inf, 0.0])
    w = [math.exp(v - 3.0) for v in (3.0, 3.0, 2.0, 1.0, 0.0)]
    order = [1, 3, 2, 0, 5]
    for kw, n in (({}, 5), ({"top_k": 2}, 2), ({"top_p": 0.85}, 3), ({"min_p": 0.3}, 3), ({"top_p": 0.0}, 1)):
        mass = sum(w[:n])
        run = 0.0
        for j in range(n):
            assert sv.sample_row(x, (run + 0.01 * w[j]) / mass, **kw)[0] == order[j], (kw, j)
            assert sv.sample_row(x, (run + 0.99 * w[j]) / mass, **kw)[0] == order[j], (kw, j)
            run += w[j]
    assert sv.sample_row(x, 0.9, temperature=0.0)[0] == 1
    assert sv.sample_row(torch.full((3,), math.nan), 0.5)[0] == -1
