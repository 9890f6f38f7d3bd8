"""What pins oracle/serve4.py (CPU): codes are the nearest of sixteen by exact
fractions, elements one rounding to fp16, rotations those of complex numbers,
attention a softmax over the tokens a row sees."""

import cmath
from fractions import Fraction

import numpy as np
import pytest
import torch

from helpers import gen
from oracle import serve4 as s4


def nearest16(v: Fraction) -> float:
    """The fp16 value nearest to v (ties to even), by search."""
    lo, hi = -0x7BFF, 0x7BFF
    val = lambda i: Fraction(float(np.uint16(abs(i)).view(np.float16))) * (1 if i >= 0 else -1)  # noqa: E731
    while lo < hi:
        mid = (lo + hi + 1) // 2
        lo, hi = (mid, hi) if val(mid) <= v else (lo, mid - 1)
    a, b = val(lo), val(min(lo + 1, 0x7BFF))
    if v - a == b - v:
        return float(a if lo % 2 == 0 else b)
    return float(a if v - a < b - v else b)


@pytest.mark.parametrize("kind", ["normal", "wide", "tiny", "equal", "offset", "largest"])
def test_codes_are_the_nearest(kind):
    g = gen(1)
    x = torch.randn(6, 64, generator=g)
    x = {"normal": x, "wide": x * torch.exp(3 * torch.randn(6, 64, generator=g)), "tiny": x * 2.0 ** -22,
         "equal": torch.full((6, 64), -3.25), "offset": 1000 + x, "largest": x.sign() * 65504}[kind].half()
    code, scale, bias = s4.quantize(x, 32)
    for r in range(6):
        for j in range(2):
            row = [Fraction(float(v)) for v in x[r, 32 * j:32 * j + 32]]
            s, b = Fraction(float(scale[r, j])), Fraction(float(bias[r, j]))
            want = nearest16((max(row) - min(row)) / 15)
            assert b == min(row) and (s == want or (15 * Fraction(want) + b >= 65520 and s < want))
            for v, c in zip(row, code[r, 32 * j:32 * j + 32].tolist()):
                exact = (v - b) / s if s else Fraction(0)
                assert c == min(max(round(exact), 0), 15)  # Python rounds fractions half to even
                assert abs(c * s + b) < 65520


def test_special_values():
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(3, 32).half()
    x[0, :6] = torch.tensor([1.0, inf, -inf, nan, 16.0, 2.0])
    x[1] = nan
    x[2] = -0.0
    code, scale, bias = s4.quantize(x, 32)
    assert scale[0].item() == torch.tensor(16 / 15).half() and bias[0].item() == 0
    assert code[0, :6].tolist() == [1, 15, 0, 0, 15, 2] and code[1:].sum() == 0 and scale[1:].sum() == 0 and bias[1:].sum() == 0


def test_elements_round_once():
    g = gen(2)
    packed = torch.randint(0, 256, (2, 2, 16, 32), generator=g).to(torch.uint8)
    affine = torch.randn(2, 2, 2, 16, 2, generator=g) * torch.exp2(torch.randint(-12, 12, (2, 2, 2, 16, 2), generator=g).float())
    affine = affine.half()
    e = s4.elements(packed, affine)
    for _ in range(200):
        n, h, t, c = (int(torch.randint(m, (1,), generator=g)) for m in (2, 2, 16, 64))
        byte = int(packed[n, h, t, c // 2])
        s, b = (Fraction(float(v)) for v in affine[n, h, c // 32, t])
        assert e[n, h, t, c].item() == nearest16((byte >> 4 if c % 2 else byte & 15) * s + b)


@pytest.mark.parametrize("neighbours", [False, True])
def test_rotation(neighbours):
    g = gen(3)
    x, angle = torch.randn(3, 2, 10, generator=g).half(), torch.randn(5, 3, generator=g)
    got16, got = s4.rotate(x, torch.tensor([4, 0, 5]), angle.cos(), angle.sin(), neighbours)
    for t, p in ((0, 4), (1, 0)):
        for h in range(2):
            for i in range(3):
                a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + 3)
                w = complex(x[t, h, a], x[t, h, b]) * complex(angle[p, i].cos(), angle[p, i].sin())
                assert cmath.isclose(complex(got[t, h, a], got[t, h, b]), w, rel_tol=1e-12, abs_tol=1e-12)
            assert torch.equal(got16[t, h, 6:], x[t, h, 6:])
    assert bool((got[2] == 0).all())


def test_append_and_values():
    g = gen(4)
    packed, affine = torch.randint(0, 256, (3, 2, 16, 32), generator=g).to(torch.uint8), torch.randn(3, 2, 2, 16, 2, generator=g).half()
    before = packed.clone(), affine.clone()
    x = torch.randn(4, 2, 64, generator=g).half()
    s4.append(x, torch.tensor([17, -1, 40, 17]), packed, affine)
    got = s4.values(torch.tensor([17, 40, 48, -1]), packed, affine)
    step = affine[1, :, :, 1, 0].double()
    err = (got[0] - x[3].double()).abs().unflatten(-1, (2, 32))
    # half a step and the element's rounding, and what the top code falls short by where the scale was rounded down
    assert bool((err <= (0.5 + 15 * 2.0 ** -11) * step[..., None] + 2.0 ** -11 * x[3].abs().max()).all())
    assert bool((got[2:] == 0).all())
    packed[1, :, 1], affine[1, :, :, 1] = before[0][1, :, 1], before[1][1, :, :, 1]
    packed[2, :, 8], affine[2, :, :, 8] = before[0][2, :, 8], before[1][2, :, :, 8]
    assert torch.equal(packed, before[0]) and torch.equal(affine, before[1])


def test_attention():
    g = gen(5)
    k, v = (torch.randn(4, 2, 16, 64, generator=g).double() for _ in range(2))
    q = torch.randn(5, 4, 64, generator=g).half()
    tables, lens, starts = torch.tensor([[2, 0], [1, 3], [0, 0]]), torch.tensor([20, 3, 0]), torch.tensor([0, 1, 5, 5])
    out, bound = s4.attention(q, k, v, tables, lens, starts, 0.125)
    kk, vv = (torch.cat([t[2, 1], t[0, 1]])[:20] for t in (k, v))
    want = torch.softmax(kk @ q[0, 3].double() * 0.125, 0) @ vv
    assert torch.allclose(out[0, 3], want, rtol=1e-12)
    assert bool((out[1] == 0).all()) and torch.allclose(out[2, 0], v[1, 0, 0])  # four rows of three tokens: the first sees none
    assert bool((bound >= 0).all()) and float((bound / out.abs().clamp(min=0.05)).max()) < 0.02


def test_attention_without_blocks_outside_the_cache():
    """A block that is not there has no weight: the same as a table without it, for rows that stand behind it; nothing
    but zeros where no other is seen."""
    g = gen(9)
    k, v = torch.randn(2, 6, 2, 4, 8, generator=g).double()
    q = torch.randn(5, 4, 8, generator=g).half()
    tables, i32 = torch.tensor([[3, 1, 5, 0]], dtype=torch.int32), dict(dtype=torch.int32)
    starts = torch.tensor([0, 5], **i32)
    for lost in (-1, 6, 10 ** 9, -2 ** 31):
        t = tables.clone()
        t[0, 1] = lost
        got = s4.attention(q, k, v, t, torch.tensor([15], **i32), starts, 0.3)
        want = s4.attention(q, k, v, tables[:, [0, 2, 3]], torch.tensor([11], **i32), starts, 0.3)
        assert torch.allclose(got[0], want[0], rtol=1e-12, atol=1e-14) and bool((got[1] >= want[1] * (1 - 1e-12)).all())
        t = torch.tensor([[lost, 2]], **i32)
        got = s4.attention(q, k, v, t, torch.tensor([6], **i32), starts, 0.3)[0]
        assert bool((got[:3] == 0).all()) and bool((got[3:].abs().amax(-1) > 0).all())
