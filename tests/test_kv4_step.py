"""The 4-bit cache a serving loop keeps (CPU): runtime/kv_cache.py KVCache4 and
cached_attention over it with the operators replaced by oracle/serve4.py, both
pairings of channels, and the angles of scaled contexts."""

import math

import pytest
import torch

from gdsllm_amd.runtime import kv_cache, llama
from oracle import serve as sv
from oracle import serve4 as s4


class Oracle:
    """The operators on CPU tensors."""

    def kv_assign(self, lens, delta, tables, ring, state, bs, max_tokens):
        t, r = tables.tolist(), ring.tolist()
        out = sv.assign(lens.tolist(), delta.tolist(), t, r, state.tolist(), bs, max_tokens)
        tables.copy_(torch.tensor(t))
        ring.copy_(torch.tensor(r))
        return tuple(torch.tensor(o, dtype=torch.int32) for o in out)

    def rope(self, q, k, positions, cos, sin, neighbours=False):
        self.turned = neighbours
        turn = lambda x: None if x is None else s4.rotate(x, positions, cos, sin, neighbours)[0]  # noqa: E731
        return turn(q), turn(k)

    def kv4_append(self, k, v, slots, kc, vc, ka, va, q=None, positions=None, cos=None, sin=None, neighbours=False):
        if cos is not None:
            k = s4.rotate(k, positions, cos, sin, neighbours)[0]
            q = None if q is None else s4.rotate(q, positions, cos, sin, neighbours)[0]
        s4.append(k, slots, kc, ka)
        s4.append(v, slots, vc, va)
        return q

    def kv4_values(self, slots, kc, vc, ka, va):
        return tuple(s4.values(slots, *c).half() for c in ((kc, ka), (vc, va)))

    def kv4_attention(self, q, kc, vc, ka, va, tables, lens, starts, scale, max_new=0, max_len=0):
        self.bounds = (max_new, max_len)
        return s4.attention(q, s4.elements(kc, ka), s4.elements(vc, va), tables, lens, starts, scale)[0].half()

    def kv_append(self, k, v, slots, kc, vc, ks, vs, q=None, positions=None, cos=None, sin=None):
        assert cos is None and q is None
        for x, c, s in ((k, kc, ks), (v, vc, vs)):
            c64, s64 = c.double(), s.double()
            sv.append(x, slots, c64, s64, "int8")
            c.copy_(c64.to(c.dtype))
            s.copy_(s64)


@pytest.fixture
def ops(monkeypatch):
    o = Oracle()
    for m in (kv_cache, llama):
        monkeypatch.setattr(m, "ext", lambda: o)
    return o


def cache(**kw):
    kw = {**dict(layers=1, requests=3, max_len=64, kv_heads=2, head_dim=64, block_size=16, group_size=32, device="cpu"), **kw}
    c = kv_cache.KVCache4(**kw)
    for t in c.k + c.v + c.k_affine + c.v_affine:
        t.zero_()
    return c


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def model(g, H=256, D=64, heads=4, kv=2):
    w = {f"self_attn.{n}_proj.weight": (torch.randint(-1, 2, (m, H), generator=g) / 8).half()
         for n, m in (("q", heads * D), ("k", kv * D), ("v", kv * D))}
    w["self_attn.o_proj.weight"] = torch.eye(H).half()
    return w


def test_bytes():
    a, b = cache(group_size=64), cache(group_size=32)
    n = a.num_blocks * 2 * 16
    assert a.nbytes == 2 * n * (32 + 4) and b.nbytes == 2 * n * (32 + 8)


@pytest.mark.parametrize("neighbours", [False, True])
def test_a_step_of_rows_equals_the_tokens_one_by_one(ops, neighbours):
    """A prompt at once and token by token, bit for bit: a token's codes are its own; the projections are exact (small
    whole numbers, o_proj the identity)."""
    g = torch.Generator().manual_seed(1)
    w = model(g)
    x = torch.randint(-2, 3, (9, 256), generator=g).half()
    cos, sin = kv_cache.rope_table(64, 64, device="cpu")
    a, b = cache(), cache()
    a.begin_step(i32(0, 9, 0), 9, max_new=9, max_len=20)
    whole = llama.cached_attention(x, w, a, 0, cos, sin, neighbours=neighbours)
    assert ops.bounds == (9, 20) and whole.shape == (9, 256)
    single = []
    for t in range(9):
        b.begin_step(i32(0, 1, 0), 1)
        single.append(llama.cached_attention(x[t:t + 1], w, b, 0, cos, sin, neighbours=neighbours))
    assert torch.equal(whole, torch.cat(single)) and float(whole.abs().max()) > 1
    for t in ("k", "v", "k_affine", "v_affine"):
        assert torch.equal(*(getattr(c, t)[0][c.block_tables[1, 0].item()] for c in (a, b)))
    k, v = a.values(0, 1, 12)
    assert k.shape == (12, 2, 64) and bool((k[9:] == 0).all()) and bool((v[:9] != 0).any())
    want = torch.nn.functional.linear(x, w["self_attn.v_proj.weight"]).view(9, 2, 64)
    assert float((v[:9].float() - want.float()).abs().max()) <= float(want.float().abs().max()) / 14


def test_both_pairings_attend_alike(ops):
    """A checkpoint whose channels are paired (2i, 2i + 1) is one paired (i, i + D/2) with its rows in another order."""
    g = torch.Generator().manual_seed(2)
    w = model(g)
    x = torch.randint(-2, 3, (5, 256), generator=g).half()
    cos, sin = kv_cache.rope_table(64, 64, device="cpu")
    order = torch.arange(64).view(32, 2).T.flatten()  # halves from neighbours
    other = {n: t if "o_proj" in n or "v_proj" in n else t.view(-1, 64, 256)[:, order].reshape(t.shape) for n, t in w.items()}
    outs = []
    for weights, neighbours in ((w, True), (other, False)):
        c = cache(group_size=64)  # one group a head: the same values in it
        c.begin_step(i32(5, 0, 0), 5)
        outs.append(llama.cached_attention(x, weights, c, 0, cos, sin, neighbours=neighbours))
    # the same numbers, summed in another order before an fp16 result: half a step, and twice what 64 bits leave
    assert bool(((outs[0] - outs[1]).abs() <= 2.0 ** -10 * outs[0].abs() + 2.0 ** -24).all())


def test_the_8_bit_cache_takes_neighbours(ops):
    g = torch.Generator().manual_seed(3)
    c = kv_cache.KVCache8(1, 2, 32, 2, 64, 16, codes=torch.int8, device="cpu")
    for t in c.k + c.v:
        t.zero_()
    cos, sin = kv_cache.rope_table(32, 64, device="cpu")
    k, v, q = (torch.randn(4, 2, 64, generator=g).half() for _ in range(3))
    c.begin_step(i32(3, 0), 4)
    got = c.append(0, k, v, q, cos, sin, neighbours=True)
    want = s4.rotate(q, c.positions, cos, sin, True)[0]
    assert ops.turned and torch.equal(got, want) and bool((got[3] == 0).all())
    page = c.block_tables[0, 0].item()
    held = c.k[0][page, :, :3].double() * c.k_scale[0][page].double()[:, None, None]
    turned = s4.rotate(k, c.positions, cos, sin, True)[1][:3].transpose(0, 1)
    # half a step of the code, and before it half an fp16 step of the turned key, which the first bound of 0.51 steps left out
    # (keys of up to 3.97: 2^-11 of them is 0.062 steps of 2^-5)
    assert bool(((held - turned).abs() <= 0.5 * c.k_scale[0][page].double()[:, None, None] + 2.0 ** -11 * turned.abs()).all())
    assert c.append(0, k, v, None, cos, sin, neighbours=True) is None


def test_order_and_arguments(ops):
    c = cache()
    x = torch.zeros(2, 2, 64).half()
    with pytest.raises(RuntimeError, match="KVCache4.append: begin_step"):
        c.append(0, x, x)
    with pytest.raises(RuntimeError, match="KVCache4.attend: begin_step"):
        c.attend(0, x)
    c.begin_step(i32(1, 0, 0), 1)
    with pytest.raises(ValueError, match="position 63"):
        c.append(0, x[:1], x[:1], x[:1], *kv_cache.rope_table(50, 64, device="cpu"))
    for request, tokens in ((-1, 1), (3, 1), (0, -1), (0, 65)):
        with pytest.raises(ValueError, match="KVCache4.values"):
            c.values(0, request, tokens)


# ------------------------------------------------------- angles of long contexts

def test_frequencies_without_scaling():
    for scaling in (None, {}, {"rope_type": "default"}):
        f, m = kv_cache.rope_frequencies(64, 500000.0, scaling)
        assert m == 1.0 and all(abs(f[i].item() - 500000.0 ** (-i / 32)) < 1e-15 for i in range(32))


def test_linear_and_ntk():
    f, m = kv_cache.rope_frequencies(32, 10000.0, {"type": "linear", "factor": 4.0})
    assert m == 1.0 and f[0] == 0.25 and abs(f[8].item() - 10000.0 ** -0.5 / 4) < 1e-16
    f, m = kv_cache.rope_frequencies(32, 10000.0, {"rope_type": "ntk", "factor": 4.0})
    # the slowest pair turns a factor slower, the fastest as before
    assert f[0] == 1 and abs(f[15].item() * 4 - 10000.0 ** (-30 / 32)) < 1e-15


def test_llama3():
    s, low, high, length = 8.0, 1.0, 4.0, 8192
    f, m = kv_cache.rope_frequencies(128, 500000.0, dict(rope_type="llama3", factor=s, low_freq_factor=low,
                                                         high_freq_factor=high, original_max_position_embeddings=length))
    kinds = set()
    for i in range(64):
        plain = 500000.0 ** (-i / 64)
        w = 2 * math.pi / plain
        if w < length / high:
            want, kind = plain, "kept"
        elif w > length / low:
            want, kind = plain / s, "slow"
        else:
            a = (length / w - low) / (high - low)
            want, kind = (1 - a) * plain / s + a * plain, "between"
        kinds.add(kind)
        assert abs(f[i].item() / want - 1) < 1e-12
    assert m == 1.0 and kinds == {"kept", "slow", "between"}


def test_yarn():
    cfg = dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096)
    f, m = kv_cache.rope_frequencies(128, 10000.0, cfg)
    assert abs(m - (0.1 * math.log(16) + 1)) < 1e-15
    turns = lambda i: 4096 * 10000.0 ** (-i / 64) / (2 * math.pi)  # noqa: E731
    # pairs that turn 32 times and more stay, those that turn less than once are slowed; whole pairs at the borders
    first = max(i for i in range(64) if turns(i) >= 32)
    last = min(i for i in range(64) if turns(i) <= 1)
    for i in range(64):
        slowed = min(max((i - first) / (last - first), 0), 1)
        want = 10000.0 ** (-i / 64) * (slowed / 16 + 1 - slowed)
        assert abs(f[i].item() / want - 1) < 1e-12
    assert kv_cache.rope_frequencies(128, 10000.0, dict(cfg, attention_factor=1.5))[1] == 1.5
    cos, sin = kv_cache.rope_table(3, 128, scaling=cfg, device="cpu")
    assert abs(cos[0, 0].item() - m) < 1e-6 and abs(sin[2, 5].item() - m * math.sin(2 * f[5].item())) < 1e-6


@pytest.mark.parametrize("scaling,word", [
    (dict(type="dynamic", factor=2.0), "unknown"), (dict(type="linear"), "factor"), (dict(type="linear", factor=0.5), "factor"),
    (dict(type="llama3", factor=2.0), "original"), (dict(type="yarn", factor=2.0), "original"),
    (dict(type="llama3", factor=2.0, original_max_position_embeddings=10, low_freq_factor=2, high_freq_factor=2), "high_freq")])
def test_scaling_refusals(scaling, word):
    with pytest.raises(ValueError, match=word):
        kv_cache.rope_frequencies(64, 10000.0, scaling)
    with pytest.raises(ValueError, match="inv_freq"):
        kv_cache.rope_table(4, 64, inv_freq=torch.ones(32), scaling=scaling, device="cpu")


def test_rotary_refusals():
    for r in (0, 3):
        with pytest.raises(ValueError, match="rotary"):
            kv_cache.rope_frequencies(r)
    with pytest.raises(ValueError, match="one pair"):
        kv_cache.rope_frequencies(2, 10000.0, dict(type="ntk", factor=2.0))


YARN = dict(rope_type="yarn", factor=40.0, original_max_position_embeddings=4096)


@pytest.mark.parametrize("keys,want", [
    (dict(mscale=1.0, mscale_all_dim=1.0), 1.0), (dict(mscale=0.707, mscale_all_dim=0.707), 1.0),
    (dict(mscale=2.0, mscale_all_dim=0.5), (0.2 * math.log(40) + 1) / (0.05 * math.log(40) + 1)),
    (dict(mscale=1.0), 0.1 * math.log(40) + 1), (dict(mscale=1.0, mscale_all_dim=0), 0.1 * math.log(40) + 1),
    (dict(mscale=None, mscale_all_dim=None, attention_factor=None), 0.1 * math.log(40) + 1),
    (dict(mscale=0.0, mscale_all_dim=0.0), 0.1 * math.log(40) + 1),
    (dict(mscale=1.0, mscale_all_dim=1.0, attention_factor=0.75), 0.75)])
def test_yarn_factor(keys, want):
    f, m = kv_cache.rope_frequencies(64, 10000.0, dict(YARN, **keys))
    assert abs(m - want) < 1e-15
    assert torch.equal(f, kv_cache.rope_frequencies(64, 10000.0, YARN)[0])


def test_yarn_between_whole_pairs_or_not():
    """truncate: whether the line between the pairs that stay and those that are slowed begins and ends at whole pairs."""
    turns = lambda i: 4096 * 10000.0 ** (-i / 32) / (2 * math.pi)  # noqa: E731
    first, last = (32 * math.log(4096 / (2 * math.pi * b)) / math.log(10000.0) for b in (32, 1))
    assert abs(turns(first) - 32) < 1e-9 and abs(turns(last) - 1) < 1e-9 and first % 1 and last % 1
    for truncate, lo, hi in ((True, math.floor(first), math.ceil(last)), (False, first, last)):
        f, _ = kv_cache.rope_frequencies(64, 10000.0, dict(YARN, truncate=truncate))
        for i in range(32):
            slowed = min(max((i - lo) / (hi - lo), 0), 1)
            assert abs(f[i].item() / (10000.0 ** (-i / 32) * (slowed / 40 + 1 - slowed)) - 1) < 1e-12


def test_keys_that_say_what_the_model_is():
    own = {"rope_theta": 500000, "partial_rotary_factor": 0.5, "original_max_position_embeddings": 8192, "type": "linear",
           "rope_type": "linear", "factor": 2.0, "finetuned": True, "beta_fast": None}
    assert torch.equal(kv_cache.rope_frequencies(64, 500000.0, own)[0],
                       kv_cache.rope_frequencies(64, 500000.0, dict(type="linear", factor=2.0))[0])


@pytest.mark.parametrize("scaling,word", [
    (dict(YARN, mscale=0.707), "together"), (dict(YARN, mscale_all_dim=1.0), "together"), (dict(YARN, mscale=-1.0), "negative"),
    (dict(YARN, beta_fast=1.0, beta_slow=2.0), "beta_fast"), (dict(YARN, beta_slow=-1.0), "beta_slow"),
    (dict(YARN, attn_factor=1.0), "attn_factor"), (dict(YARN, low_freq_factor=1.0), "low_freq_factor"),
    (dict(type="linear", factor=2.0, mscale=1.0), "'mscale'"), (dict(type="ntk", factor=2.0, alpha=1.0), "'alpha'"),
    (dict(rope_type="default", factor=2.0), "'factor'"), (dict(factor=2.0), "'factor'"),
    (dict(rope_type="llama3", factor=2.0, original_max_position_embeddings=10, low_freq_factor=1, high_freq_factor=4, short_factor=[1.0]),
     "short_factor"),
    (dict(rope_type="linear", type="mrope", factor=2.0), "differ"), (dict(type="linear", factor=2.0, rope_theta=1e6), "rope_theta")])
def test_scaling_keys_are_not_dropped(scaling, word):
    with pytest.raises(ValueError, match=word):
        kv_cache.rope_frequencies(64, 10000.0, scaling)
