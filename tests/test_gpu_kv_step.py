"""The serving operators run together, as a server runs them (runtime/kv_cache.py
KVCache8, runtime/llama.py cached_attention and mlp, runtime/scheduler.py
next_tokens): a small two-layer Q4_0 model with grouped query heads through
prompts, decoding, an ended request and a new one.

* every call of an operator is held to oracle/serve.py on the inputs it got;
* the decode step captured into a graph and replayed, with eager work and
  synchronizations between the replays, gives the eager step's tokens, lengths
  and cache bytes, each time."""

import pytest
import torch

from gdsllm_amd.runtime import kv_cache, llama, scheduler
from helpers import gen, syn
from oracle import serve as sv

pytestmark = pytest.mark.gpu

H, FFN, VOCAB, LAYERS, HEADS, KV, D, BS, REQ = 512, 768, 1000, 2, 8, 2, 64, 16, 4
PROJ = (("self_attn.q_proj", HEADS * D, H), ("self_attn.k_proj", KV * D, H), ("self_attn.v_proj", KV * D, H),
        ("self_attn.o_proj", H, HEADS * D), ("mlp.gate_proj", FFN, H), ("mlp.up_proj", FFN, H), ("mlp.down_proj", H, FFN))


class Model:
    def __init__(self, dev):
        g = torch.Generator(device=dev).manual_seed(11)
        self.layers = []
        for _ in range(LAYERS):
            mats = [syn.q4_0_weights(m, k, g) for _, m, k in PROJ]
            buf, offs = syn.pack_buffer(mats)
            handle = kv_cache.ext().GdsBufferHandle.from_tensor(buf)
            self.layers.append({f"{p}.weight": {"buffer": handle, "shape": [m, k], "gguf_type": "q4_0", "offset": o}
                                for (p, m, k), o in zip(PROJ, offs)})
        self.tensors = {"model.embed_tokens.weight": torch.randn(VOCAB, H, generator=g, device=dev).half(),
                        "lm_head.weight": (torch.randn(VOCAB, H, generator=g, device=dev) / 8).half()}
        self.cos, self.sin = kv_cache.rope_table(256, D, device=dev)

    @staticmethod
    def norm(h):
        f = h.float()
        return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-5)).half()

    def step(self, cache, ids, u, temperature, top_p):
        """Tokens of the rows ids [T], one for each request (of its last row; the first row's where it has none)."""
        h = scheduler._embed_tokens(ids[None], self.tensors)[0]
        for i, w in enumerate(self.layers):
            h = h + llama.cached_attention(self.norm(h), w, cache, i, self.cos, self.sin)
            h = h + llama.mlp(llama.packed_rows(self.norm(h)), w).reshape(h.shape)
        rows = self.norm(h)[cache.last_rows().clamp(min=0)]
        return scheduler.next_tokens(rows, self.tensors, u, temperature=temperature, top_p=top_p)


class Held:
    """The extension, with every call of the four operators held to the oracle."""

    def __init__(self, real):
        self.real, self.calls = real, []

    def __getattr__(self, name):
        return getattr(self.real, name)

    def kv_assign(self, lens, delta, tables, ring, state, bs, max_tokens):
        t, r = tables.tolist(), ring.tolist()
        want = sv.assign(lens.tolist(), delta.tolist(), t, r, state.tolist(), bs, max_tokens)
        got = self.real.kv_assign(lens, delta, tables, ring, state, bs, max_tokens)
        assert [g.tolist() for g in got] == [list(w) for w in want] and tables.tolist() == t and ring.tolist() == r
        self.calls.append("assign")
        return got

    def kv_append(self, k, v, slots, kc, vc, ks, vs, q, positions, cos, sin):
        before = [t.cpu().double() for t in (kc, vc, ks, vs)]
        got = self.real.kv_append(k, v, slots, kc, vc, ks, vs, q, positions, cos, sin)
        p, c, s, sl = positions.cpu(), cos.cpu(), sin.cpu(), slots.cpu()
        fmt = "int8" if kc.dtype == torch.int8 else "e4m3"
        sv.append(sv.rotate(k.cpu(), p, c, s)[0], sl, before[0], before[2], fmt)
        sv.append(v.cpu(), sl, before[1], before[3], fmt)
        for t, w in zip((kc, vc, ks, vs), before):
            assert torch.equal(t.cpu().double().nan_to_num(999), w.nan_to_num(999))
        assert torch.equal(got.cpu(), torch.where(sl[:, None, None] >= 0, sv.rotate(q.cpu(), p, c, s)[0], 0))
        self.calls.append("append")
        return got

    def kv_attention(self, q, kc, vc, ks, vs, tables, lens, starts, scale, max_new, max_len):
        got = self.real.kv_attention(q, kc, vc, ks, vs, tables, lens, starts, scale, max_new, max_len)
        s = [t.cpu().double() for t in (ks, vs)]
        vals = [t.cpu().double() * w[..., None, None] for t, w in zip((kc, vc), s)]
        want, bound = sv.attention(q.cpu(), *vals, s[1], tables.cpu(), lens.cpu(), starts.cpu(), scale)
        assert bool(((got.cpu().double() - want).abs() <= bound).all())
        self.calls.append("attend")
        return got

    def sample_tokens(self, logits, u, temperature, top_k, top_p, min_p):
        got = self.real.sample_tokens(logits, u, temperature, top_k, top_p, min_p)
        for i, t in enumerate(got.tolist()):
            want, border = sv.sample_row(logits[i].cpu(), u[i].item(), temperature[i].item(), 0, top_p[i].item())
            assert t == want or border < 1e-12
        self.calls.append("sample")
        return got


def new_cache(dev, codes, **kw):
    c = kv_cache.KVCache8(LAYERS, REQ, 200, KV, D, BS, codes=codes, device=dev, **kw)
    for t in c.k + c.v:
        t.zero_()
    return c


def settings(dev):
    return torch.tensor([0.0, 1.0, 0.7, 1.5], device=dev), torch.tensor([1.0, 0.9, 1.0, 0.5], device=dev)


def i32(dev, v):
    return torch.tensor(v, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("codes", [torch.float8_e4m3fn, torch.int8], ids=["e4m3", "int8"])
def test_a_server_of_four_requests(gpu, monkeypatch, codes):
    m, held = Model(gpu), Held(kv_cache.ext())
    for module in (kv_cache, llama, scheduler):
        monkeypatch.setattr(module, "ext", lambda: held)
    c = new_cache(gpu, codes, num_blocks=20)
    t, p = settings(gpu)
    g = gen(12)
    # prompts; a slot that is idle; decoding; one that ends while another begins; a prompt of one token
    steps = [[5, 70, 0, 33], [1, 1, 0, 1], [1, 1, 0, 1], [-7, 1, 40, 1], [1, 1, 1, 1], [3, 0, 1, -36], [1, 1, 1, 1]]
    last, total = torch.zeros(REQ, dtype=torch.int64), [0] * REQ
    for delta in steps:
        rows = sum(max(d, 0) for d in delta)
        ids = torch.cat([last[r:r + 1] if d == 1 else torch.randint(0, VOCAB, (max(d, 0),), generator=g)
                         for r, d in enumerate(delta)])
        total = [n + d for n, d in zip(total, delta)]
        c.begin_step(i32(gpu, delta), rows, max(delta), max(total))
        assert c.lens.tolist() == total and c.served().all()
        last = m.step(c, ids.to(gpu), torch.rand(REQ, generator=g).to(gpu), t, p).cpu()
        assert bool(((last >= 0) & (last < VOCAB)).all())
    n = len(steps)
    assert held.calls == (["assign"] + ["append", "attend"] * LAYERS + ["sample"]) * n


@pytest.mark.parametrize("codes", [torch.float8_e4m3fn, torch.int8], ids=["e4m3", "int8"])
def test_the_decode_step_as_a_graph(gpu, codes):
    m = Model(gpu)
    t, p = settings(gpu)
    g = gen(13)
    prompt = torch.randint(0, VOCAB, (5 + 63 + 1 + 16,), generator=g).to(gpu)
    us = [torch.rand(REQ, generator=g).to(gpu) for _ in range(8)]
    eager, graph, trial = (new_cache(gpu, codes) for _ in range(3))
    one = i32(gpu, [1] * REQ)

    def decode(c, ids, u):
        c.begin_step(one, REQ, max_new=1)
        return m.step(c, ids, u, t, p)

    firsts = []
    for c in (eager, graph, trial):
        c.begin_step(i32(gpu, [5, 63, 1, 16]), 85, 63, 63)
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
        for name in ("k", "v", "k_scale", "v_scale"):
            for a, b in zip(getattr(graph, name), getattr(eager, name)):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert eager.lens.tolist() == [12, 70, 8, 23]
