"""The cache a serving loop keeps and its step (CPU): runtime/kv_cache.py
KVCache8, cached_attention and next_tokens, with the operators replaced by
oracle/serve.py."""

import math

import pytest
import torch

from gdsllm_amd.runtime import kv_cache, llama, scheduler
from oracle import serve as sv


class Oracle:
    """The four operators on CPU tensors."""

    def kv_assign(self, lens, delta, tables, ring, state, bs, max_tokens):
        t, r = tables.tolist(), ring.tolist()
        out = sv.assign(lens.tolist(), delta.tolist(), t, r, state.tolist(), bs, max_tokens)
        tables.copy_(torch.tensor(t))
        ring.copy_(torch.tensor(r))
        return tuple(torch.tensor(o, dtype=torch.int32) for o in out)

    def kv_append(self, k, v, slots, kc, vc, ks, vs, q=None, positions=None, cos=None, sin=None):
        fmt = "int8" if kc.dtype == torch.int8 else "e4m3"
        if cos is not None:
            k = sv.rotate(k, positions, cos, sin)[0]
            q = None if q is None else torch.where(slots[:, None, None] >= 0, sv.rotate(q, positions, cos, sin)[0], 0)
        for x, c, s in ((k, kc, ks), (v, vc, vs)):
            c64, s64 = c.double(), s.double()
            sv.append(x, slots, c64, s64, fmt)
            c.copy_(c64.to(c.dtype))
            s.copy_(s64)
        return q

    def kv_attention(self, q, kc, vc, ks, vs, tables, lens, starts, scale, max_new=0, max_len=0):
        self.bounds = (max_new, max_len)
        ks, vs = ks.double(), vs.double()
        return sv.attention(q, kc.double() * ks[..., None, None], vc.double() * vs[..., None, None], vs, tables, lens, starts,
                            scale)[0].half()

    def sample_tokens(self, logits, u, temperature, top_k, top_p, min_p):
        pick = lambda t, i, d: d if t is None else t[i].item()  # noqa: E731
        return torch.tensor([sv.sample_row(logits[i], u[i].item(), pick(temperature, i, 1.0), pick(top_k, i, 0),
                                           pick(top_p, i, 1.0), pick(min_p, i, 0.0))[0] for i in range(len(logits))])


@pytest.fixture
def ops(monkeypatch):
    o = Oracle()
    for m in (kv_cache, llama, scheduler):
        monkeypatch.setattr(m, "ext", lambda: o)
    return o


def cache(**kw):
    kw = {**dict(layers=1, requests=3, max_len=64, kv_heads=2, head_dim=64, block_size=16, device="cpu"), **kw}
    c = kv_cache.KVCache8(**kw)
    for t in c.k + c.v:
        t.zero_()
    return c


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("kw,word", [
    (dict(layers=0), "layers"), (dict(requests=0), "requests"), (dict(requests=8193), "requests"), (dict(max_len=0), "max_len"),
    (dict(kv_heads=0), "kv_heads"), (dict(block_size=24), "block_size"), (dict(head_dim=96), "head_dim"),
    (dict(codes=torch.float16), "codes"), (dict(num_blocks=0), "num_blocks"), (dict(num_blocks=2 ** 27), "num_blocks")])
def test_refusals(kw, word):
    with pytest.raises(ValueError, match=word):
        cache(**kw)


def test_state_over_steps(ops):
    """Requests begin, grow, end and begin again in the blocks that others gave back."""
    c = cache(num_blocks=5)
    c.begin_step(i32(20, 0, 3), 24)
    assert c.lens.tolist() == [20, 0, 3] and c.starts.tolist() == [0, 20, 20, 23] and c.free_state.tolist() == [3, 2]
    assert c.last_rows().tolist() == [19, -1, 22] and c.served().tolist() == [True] * 3
    held = set(c.block_tables[0, :2].tolist()) | {c.block_tables[2, 0].item()}
    assert len(held) == 3
    # 33 tokens need three blocks and two are left; the third request goes on in its block
    c.begin_step(i32(1, 33, 1), 40)
    assert c.lens.tolist() == [21, 0, 4] and c.served().tolist() == [True, False, True]
    assert c.slots[1:34].tolist() == [-1] * 33 and c.slots[34].item() == c.block_tables[2, 0] * 16 + 3
    c.begin_step(i32(-21, 0, 0))
    assert c.lens.tolist() == [0, 0, 4] and c.free_state[1].item() == 4 and c.served().all()
    c.begin_step(i32(0, 33, 0), 33)
    assert c.lens.tolist() == [0, 33, 4] and c.free_state[1].item() == 1
    assert len(set(c.block_tables[1, :3].tolist()) | {c.block_tables[2, 0].item()}) == 4


def test_a_step_of_rows_equals_the_tokens_one_by_one(ops):
    """A prompt at once and token by token, bit for bit: its first token has the largest keys and values, so no scale
    grows later; the projections are exact (small whole numbers, o_proj the identity)."""
    g = torch.Generator().manual_seed(1)
    H, D, heads, kv = 256, 64, 4, 2
    w = {f"self_attn.{n}_proj.weight": (torch.randint(-1, 2, (m, H), generator=g) / 8).half()
         for n, m in (("q", heads * D), ("k", kv * D), ("v", kv * D))}
    w["self_attn.o_proj.weight"] = torch.eye(H).half()
    x = torch.randint(-2, 3, (9, H), generator=g).half()
    x[0] *= 16
    cos, sin = kv_cache.rope_table(64, D, device="cpu")
    a, b = cache(codes=torch.int8), cache(codes=torch.int8)
    a.begin_step(i32(0, 9, 0), 9, max_new=9, max_len=20)
    whole = llama.cached_attention(x, w, a, 0, cos, sin)
    assert ops.bounds == (9, 20) and whole.shape == (9, H)
    single = []
    for t in range(9):
        b.begin_step(i32(0, 1, 0), 1)
        single.append(llama.cached_attention(x[t:t + 1], w, b, 0, cos, sin))
    assert ops.bounds == (0, 64)
    assert torch.equal(whole, torch.cat(single)) and float(whole.abs().max()) > 1
    for t in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(*(getattr(c, t)[0][c.block_tables[1, 0].item()] for c in (a, b)))


def test_order_and_arguments(ops):
    c = cache()
    x = torch.zeros(2, 2, 64).half()
    with pytest.raises(RuntimeError, match="begin_step"):
        c.append(0, x, x)
    with pytest.raises(RuntimeError, match="begin_step"):
        c.attend(0, x)
    with pytest.raises(ValueError, match="rows"):
        llama.cached_attention(torch.zeros(2, 64).half(), {}, c, 0, None, None)
    c.begin_step(i32(1, 1, 0), 2)
    with pytest.raises(ValueError, match="rows"):
        llama.cached_attention(torch.zeros(3, 64).half(), {}, c, 0, None, None)
    with pytest.raises(RuntimeError, match="gradients"):
        llama.cached_attention(torch.zeros(2, 64, dtype=torch.float16, requires_grad=True), {}, c, 0, None, None)
    c.begin_step(i32(0, 0, 0))
    assert llama.cached_attention(torch.zeros(0, 64).half(), {}, c, 0, None, None).shape == (0, 64)


def test_the_rotation_reaches_every_position(ops):
    """max_len counts whole blocks, and a table that ends before it is refused."""
    c = cache(max_len=50)
    assert c.max_len == 64 and c.block_tables.shape == (3, 4)
    c.begin_step(i32(1, 0, 0), 1)
    x = torch.zeros(1, 2, 64).half()
    with pytest.raises(ValueError, match="position 63"):
        c.append(0, x, x, x, *kv_cache.rope_table(50, 64, device="cpu"))
    c.append(0, x, x, x, *kv_cache.rope_table(64, 64, device="cpu"))


def test_rope_table():
    cos, sin = kv_cache.rope_table(100001, 64, theta=500000.0, device="cpu")
    for p, i in ((0, 0), (1, 0), (100000, 0), (100000, 31), (777, 5)):
        a = p * 500000.0 ** (-2 * i / 64)
        assert abs(cos[p, i].item() - math.cos(a)) <= 2.0 ** -24 + 1e-10 and abs(sin[p, i].item() - math.sin(a)) <= 2.0 ** -24 + 1e-10
    with pytest.raises(ValueError, match="inv_freq"):
        kv_cache.rope_table(4, 64, inv_freq=torch.ones(3))


@pytest.mark.parametrize("rows", [1, 8, 9])
def test_next_tokens(ops, rows):
    g = torch.Generator().manual_seed(rows)
    h, w = torch.randn(rows, 32, generator=g).half(), torch.randn(50, 32, generator=g).half()
    u = torch.rand(rows, generator=g)
    got = scheduler.next_tokens(h, {"lm_head.weight": w}, u, temperature=torch.zeros(rows))
    assert torch.equal(got, torch.nn.functional.linear(llama.packed_rows(h), w).reshape(rows, 50).argmax(-1))
    assert scheduler.next_tokens(h[:0], {"lm_head.weight": w}, u[:0]).shape == (0,)
    with pytest.raises(ValueError, match="rows"):
        scheduler.next_tokens(h[None], {"lm_head.weight": w}, u)
