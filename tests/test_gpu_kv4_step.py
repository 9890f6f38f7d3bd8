"""The operators of the 4-bit cache run together, as a server runs them
(runtime/kv_cache.py KVCache4 under the two-layer model of test_gpu_kv_step.py):

* every call of an operator is held to oracle/serve4.py on the inputs it got, for
  both pairings of channels;
* the decode step captured into a graph and replayed, with eager work and
  synchronizations between the replays, gives the eager step's tokens, lengths and
  cache bytes, each time;
* what a request's cache holds moves to another cache through values()."""

import pytest
import torch

import test_gpu_kv_step as base
from gdsllm_amd.runtime import kv_cache, llama, scheduler
from helpers import gen
from oracle import serve4 as s4

pytestmark = pytest.mark.gpu

LAYERS, REQ, VOCAB, KV, D, BS = base.LAYERS, base.REQ, base.VOCAB, base.KV, base.D, base.BS
NAMES = ("k", "v", "k_affine", "v_affine")


class Model(base.Model):
    def __init__(self, dev, neighbours):
        super().__init__(dev)
        self.neighbours = neighbours
        self.cos, self.sin = kv_cache.rope_table(256, D, device=dev, scaling=dict(type="linear", factor=2.0))

    def step(self, cache, ids, u, temperature, top_p):
        h = scheduler._embed_tokens(ids[None], self.tensors)[0]
        for i, w in enumerate(self.layers):
            h = h + llama.cached_attention(self.norm(h), w, cache, i, self.cos, self.sin, neighbours=self.neighbours)
            h = h + llama.mlp(llama.packed_rows(self.norm(h)), w).reshape(h.shape)
        rows = self.norm(h)[cache.last_rows().clamp(min=0)]
        return scheduler.next_tokens(rows, self.tensors, u, temperature=temperature, top_p=top_p)


class Held:
    """The extension, with every call of the cache's operators held to the oracle."""

    def __init__(self, real):
        self.real, self.calls = real, []

    def __getattr__(self, name):
        return getattr(self.real, name)

    def rope(self, q, k, positions, cos, sin, neighbours):
        got = self.real.rope(q, k, positions, cos, sin, neighbours)
        for x, y in zip((q, k), got):
            assert torch.equal(y.cpu(), s4.rotate(x.cpu(), positions.cpu(), cos.cpu(), sin.cpu(), neighbours)[0])
        self.calls.append("rope")
        return got

    def kv4_append(self, k, v, slots, kc, vc, ka, va, q, positions, cos, sin, neighbours):
        want = [t.cpu() for t in (kc, vc, ka, va)]
        got = self.real.kv4_append(k, v, slots, kc, vc, ka, va, q, positions, cos, sin, neighbours)
        p, c, s = positions.cpu(), cos.cpu(), sin.cpu()
        s4.append(s4.rotate(k.cpu(), p, c, s, neighbours)[0], slots.cpu(), want[0], want[2])
        s4.append(v.cpu(), slots.cpu(), want[1], want[3])
        for t, w in zip((kc, vc, ka, va), want):
            assert torch.equal(t.cpu().view(torch.uint8), w.view(torch.uint8))
        assert torch.equal(got.cpu(), s4.rotate(q.cpu(), p, c, s, neighbours)[0])
        self.calls.append("append")
        return got

    def kv4_attention(self, q, kc, vc, ka, va, tables, lens, starts, scale, max_new, max_len):
        got = self.real.kv4_attention(q, kc, vc, ka, va, tables, lens, starts, scale, max_new, max_len)
        vals = [s4.elements(c.cpu(), a.cpu()) for c, a in ((kc, ka), (vc, va))]
        want, bound = s4.attention(q.cpu(), *vals, tables.cpu(), lens.cpu(), starts.cpu(), scale)
        assert bool(((got.cpu().double() - want).abs() <= bound).all())
        self.calls.append("attend")
        return got


def new_cache(dev, group, **kw):
    c = kv_cache.KVCache4(LAYERS, REQ, 200, KV, D, BS, group_size=group, device=dev, **kw)
    for n in NAMES:
        for t in getattr(c, n):
            t.zero_()
    return c


@pytest.mark.parametrize("group,neighbours", [(32, False), (64, True)])
def test_a_server_of_four_requests(gpu, monkeypatch, group, neighbours):
    m, held = Model(gpu, neighbours), Held(kv_cache.ext())
    for module in (kv_cache, llama, scheduler):
        monkeypatch.setattr(module, "ext", lambda: held)
    c = new_cache(gpu, group, num_blocks=20)
    t, p = base.settings(gpu)
    g = gen(12)
    # prompts; a slot that is idle; decoding; one that ends while another begins; a prompt of one token
    steps = [[5, 70, 0, 33], [1, 1, 0, 1], [1, 1, 0, 1], [-7, 1, 40, 1], [1, 1, 1, 1], [3, 0, 1, -36], [1, 1, 1, 1]]
    last, total = torch.zeros(REQ, dtype=torch.int64), [0] * REQ
    for delta in steps:
        rows = sum(max(d, 0) for d in delta) + 2  # two rows of no request behind the last
        ids = torch.cat([last[r:r + 1] if d == 1 else torch.randint(0, VOCAB, (max(d, 0),), generator=g)
                         for r, d in enumerate(delta)] + [torch.zeros(2, dtype=torch.int64)])
        total = [n + d for n, d in zip(total, delta)]
        c.begin_step(base.i32(gpu, delta), rows, max(delta), max(total))
        assert c.lens.tolist() == total and c.served().all()
        last = m.step(c, ids.to(gpu), torch.rand(REQ, generator=g).to(gpu), t, p).cpu()
        assert bool(((last >= 0) & (last < VOCAB)).all())
    assert held.calls == ["append", "attend"] * (LAYERS * len(steps))


def test_the_8_bit_cache_with_neighbours(gpu, monkeypatch):
    """KVCache8 turns neighbouring channels by rope ahead of its append."""
    held = Held(kv_cache.ext())
    monkeypatch.setattr(kv_cache, "ext", lambda: held)
    g = gen(20)
    caches = [kv_cache.KVCache8(1, 2, 64, KV, D, BS, codes=torch.int8, device=gpu) for _ in range(2)]
    cos, sin = kv_cache.rope_table(64, D, device=gpu)
    q, k, v = (torch.randn(12, h, D, generator=g).half().to(gpu) for h in (8, KV, KV))
    order = torch.arange(D, device=gpu).view(-1, 2).T.flatten()  # halves from neighbours
    outs = []
    for c, neighbours in zip(caches, (True, False)):
        for t in c.k + c.v:
            t.zero_()
        c.begin_step(base.i32(gpu, [9, 2]), 12)
        turned = c.append(0, k if neighbours else k[..., order], v, q if neighbours else q[..., order], cos, sin, neighbours=neighbours)
        outs.append(turned)
        assert bool((turned[11] == 0).all())
    assert held.calls == ["rope"] and torch.equal(outs[0][..., order], outs[1])
    assert torch.equal(caches[0].k[0][..., order], caches[1].k[0]) and torch.equal(caches[0].k_scale[0], caches[1].k_scale[0])


@pytest.mark.parametrize("group,neighbours", [(32, True), (64, False)])
def test_the_decode_step_as_a_graph(gpu, group, neighbours):
    m = Model(gpu, neighbours)
    t, p = base.settings(gpu)
    g = gen(13)
    prompt = torch.randint(0, VOCAB, (5 + 63 + 1 + 16,), generator=g).to(gpu)
    us = [torch.rand(REQ, generator=g).to(gpu) for _ in range(8)]
    eager, graph, trial = (new_cache(gpu, group) for _ in range(3))
    one = base.i32(gpu, [1] * REQ)

    def decode(c, ids, u):
        c.begin_step(one, REQ, max_new=1)
        return m.step(c, ids, u, t, p)

    firsts = []
    for c in (eager, graph, trial):
        c.begin_step(base.i32(gpu, [5, 63, 1, 16]), 85, 63, 63)
        firsts.append(m.step(c, prompt, us[0], t, p))
    assert torch.equal(firsts[0], firsts[1])
    decode(trial, firsts[2], us[1])  # loads every kernel outside the capture
    torch.cuda.synchronize()
    ids, u = firsts[1].clone(), us[1].clone()
    recorded = torch.cuda.CUDAGraph()
    with torch.cuda.graph(recorded):
        ids.copy_(decode(graph, ids, u))
    want = firsts[0]
    for step in us[1:]:
        u.copy_(step)
        recorded.replay()
        want = decode(eager, want, step)
        torch.cuda.synchronize()
        assert torch.equal(ids, want) and torch.equal(graph.lens, eager.lens)
        assert torch.equal(graph.free_state, eager.free_state) and torch.equal(graph.block_tables, eager.block_tables)
        for name in NAMES:
            for a, b in zip(getattr(graph, name), getattr(eager, name)):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert eager.lens.tolist() == [12, 70, 8, 23]


def test_a_request_moves_to_another_cache(gpu):
    """The values of a request, appended to an empty 4-bit cache with other blocks, are the values again: the codes of
    sixteen equidistant values are exact but for the roundings of the scale and the elements."""
    g = gen(14)
    a, b = new_cache(gpu, 32), new_cache(gpu, 32, num_blocks=9)
    k, v = (torch.randn(50, KV, D, generator=g).half().to(gpu) for _ in range(2))
    a.begin_step(base.i32(gpu, [0, 50, 0, 0]), 50)
    a.append(1, k, v)
    held = a.values(1, 1, 60)
    assert held[0].shape == (60, KV, D) and bool((held[0][50:] == 0).all()) and bool((held[1][50:] == 0).all())
    b.begin_step(base.i32(gpu, [0, 0, 0, 50]), 50)
    b.append(1, held[0][:50], held[1][:50])
    again = b.values(1, 3, 50)
    for x, y, orig in zip(again, held, (k, v)):
        # a value moves by the second scale's rounding (2^-11 of up to 15 steps) and half an fp16 step, twice
        top = orig.float().abs().amax()
        assert float((x.float() - y[:50].float()).abs().max()) <= 4 * 2.0 ** -11 * 2 * float(top)
        spread = orig.float().unflatten(-1, (-1, 32))
        half = (spread.amax(-1) - spread.amin(-1)) / 30
        # half a step of the code, the scale's rounding over 15 steps, the element's
        err = (y[:50].float() - orig.float()).abs().unflatten(-1, (-1, 32)).amax(-1)
        assert bool((err <= half * (1 + 2.0 ** -6) + 2.0 ** -11 * top).all())
