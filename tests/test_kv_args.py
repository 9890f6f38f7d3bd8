"""Refusals of the serving operators on the CPU: every call here is rejected
before anything touches a device, with a message that names what is wrong."""

import ctypes

import pytest
import torch

from gdsllm_amd import KvCache8, capi
from gdsllm_amd.runtime import ext

BAD = 1


def _err():
    return capi().gdsllm_last_error().decode()


def _cache(**kw):
    base = dict(k=16, v=16, k_scale=16, v_scale=16, num_blocks=4, kv_heads=2, block_size=16, head_dim=64, format=0)
    c = KvCache8(**dict(base, **kw))
    return ctypes.byref(c)


CACHES = [(dict(k=0), "null"), (dict(v_scale=0), "null"), (dict(k=8), "misaligned"), (dict(k_scale=18), "misaligned"),
          (dict(block_size=8), "block_size"), (dict(block_size=48), "block_size"), (dict(block_size=512), "block_size"),
          (dict(head_dim=80), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(kv_heads=0), "kv_heads"),
          (dict(num_blocks=0), "num_blocks"), (dict(num_blocks=2 ** 28), "num_blocks"), (dict(format=2), "format")]


@pytest.mark.parametrize("kw,word", CACHES, ids=[str(i) for i in range(len(CACHES))])
def test_cache_descriptor(kw, word):
    lib = capi()
    assert lib.gdsllm_kv_append(_cache(**kw), 16, 128, 16, 128, 16, 1, None, 0, None, 0, None, None, None, 0, 0, None) == BAD
    assert word in _err()
    assert lib.gdsllm_kv_attention(_cache(**kw), 16, 128, 16, 128, 1, 2, 16, 1, 1, 16, 16, 1, 1.0, 1, 1, 0, None, 0, None) == BAD
    assert word in _err()


def test_null_cache():
    lib = capi()
    assert lib.gdsllm_kv_append(None, 16, 128, 16, 128, 16, 1, None, 0, None, 0, None, None, None, 0, 0, None) == BAD


def test_append_refusals():
    def call(c=None, k=16, ldk=128, v=16, ldv=128, slots=16, n=1, q=None, ldq=0, qo=None, hq=0, pos=None, cos=None, sin=None,
             rot=0, mp=0):
        return capi().gdsllm_kv_append(c or _cache(), k, ldk, v, ldv, slots, n, q, ldq, qo, hq, pos, cos, sin, rot, mp, None)

    assert call(n=0) == 0 and call(n=0, k=None, v=None, slots=None) == 0
    assert call(n=-1) == BAD and "token" in _err()
    for name in ("k", "v", "slots"):
        assert call(**{name: None}) == BAD and "null" in _err()
    assert call(ldk=64) == BAD and "stride" in _err()
    assert call(ldv=132) == BAD and "multiples of 8" in _err()
    assert call(k=24) == BAD and "aligned" in _err()
    assert call(slots=18) == BAD and "misaligned" in _err()
    rope = dict(pos=16, cos=16, sin=16, rot=32, mp=9)
    assert call(**dict(rope, rot=24)) == BAD and "rotary" in _err()
    assert call(**dict(rope, rot=80)) == BAD and "rotary" in _err()
    assert call(**dict(rope, pos=None)) == BAD and "positions" in _err()
    assert call(**dict(rope, mp=0)) == BAD and "positions" in _err()
    assert call(q=16, qo=16, hq=2, ldq=128) == BAD and "rotation" in _err()
    assert call(**rope, q=16, qo=None, hq=2, ldq=128) == BAD and "null" in _err()
    assert call(**rope, q=16, qo=16, hq=0, ldq=128) == BAD and "q_heads" in _err()
    assert call(**rope, q=16, qo=16, hq=4, ldq=128) == BAD and "stride" in _err()


def test_attention_refusals():
    def call(c=None, q=16, ldq=128, o=16, ldo=128, n=1, hq=2, tab=16, w=1, ldt=1, lens=16, st=16, b=1, new=1, ml=16, ws=None,
             wb=0, scale=1.0):
        return capi().gdsllm_kv_attention(c or _cache(), q, ldq, o, ldo, n, hq, tab, w, ldt, lens, st, b, scale, new, ml, 0,
                                          ws, wb, None)

    assert call(n=0) == 0
    for name in ("q", "o", "tab", "lens", "st"):
        assert call(**{name: None}) == BAD and "null" in _err()
    assert call(hq=3) == BAD and "multiple of kv_heads" in _err()
    assert call(hq=0) == BAD
    assert call(ldq=64) == BAD and "stride" in _err()
    assert call(ldo=130) == BAD and "multiples of 8" in _err()
    assert call(q=24) == BAD and "aligned" in _err()
    assert call(st=18) == BAD and "misaligned" in _err()
    assert call(ldt=0) == BAD and call(w=0) == BAD
    assert call(w=2 ** 28, ldt=2 ** 28) == BAD and "table_width" in _err()
    assert call(b=70000) == BAD and "requests" in _err()
    assert call(b=0) == BAD and "requests" in _err()
    assert call(new=-1) == BAD and call(ml=-1) == BAD
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert call(scale=scale) == BAD and "scale" in _err()
    # a sequence long enough to be split needs its workspace
    lib = capi()
    need = lib.gdsllm_kv_attention_workspace_size(1, 2, 2, 64, 1, 16 * 1000)
    assert need > 0 and call(w=1000, ldt=1000, ml=0) == BAD and f"{need} bytes" in _err()
    assert call(w=1000, ldt=1000, ml=0, ws=16, wb=need - 1) == BAD
    assert lib.gdsllm_kv_attention_workspace_size(1, 3, 2, 64, 1, 100) == 0
    assert lib.gdsllm_kv_attention_workspace_size(-1, 2, 2, 64, 1, 100) == 0


def test_assign_refusals():
    def call(lens=4, delta=4, n=1, tab=4, w=1, ldt=1, ring=4, r=1, st=4, bs=16, mt=1, sl=4, pos=4, starts=4, lo=8, so=8):
        return capi().gdsllm_kv_assign(lens, delta, n, tab, w, ldt, ring, r, st, bs, mt, sl, pos, starts, lo, so, None)

    for name in ("lens", "delta", "tab", "ring", "st", "sl", "pos", "starts", "lo", "so"):
        assert call(**{name: None}) == BAD and "null" in _err()
        assert call(**{name: 6}) == BAD and "misaligned" in _err()
    assert call(n=0) == BAD and call(n=8193) == BAD and "requests" in _err()
    assert call(bs=24) == BAD and "block_size" in _err()
    assert call(w=0) == BAD and call(w=2, ldt=1) == BAD
    assert call(r=0) == BAD and call(r=2 ** 28) == BAD and "ring_size" in _err()
    assert call(mt=-1) == BAD and "max_tokens" in _err()
    assert call(lo=4) == BAD and "must not be the inputs" in _err()
    assert call(so=4) == BAD


def test_sample_refusals():
    def call(l=8, bits=16, rows=1, v=10, ld=10, u=8, t=None, k=None, p=None, m=None, out=8):
        return capi().gdsllm_sample_tokens(l, bits, rows, v, ld, u, t, k, p, m, out, None)

    assert call(rows=0) == 0
    assert call(bits=8) == BAD and "fp16 or fp32" in _err()
    assert call(rows=-1) == BAD and call(v=0) == BAD and call(v=2 ** 20 + 1, ld=2 ** 21) == BAD and "vocab" in _err()
    assert call(ld=9) == BAD and "ld" in _err()
    assert call(l=None) == BAD and call(out=None) == BAD and "null" in _err()
    assert call(u=None) == BAD and "uniform" in _err()
    assert call(l=9) == BAD and call(l=10, bits=32) == BAD and call(out=12) == BAD and call(t=6) == BAD and "misaligned" in _err()


def test_calls_too_large_for_one_launch():
    """Grids count threads in 32 bits and rows in 31."""
    lib = capi()
    assert lib.gdsllm_sample_tokens(8, 16, 2 ** 22, 10, 10, 8, None, None, None, None, 8, None) == BAD and "rows" in _err()
    wide = _cache(kv_heads=1024, num_blocks=4)
    assert lib.gdsllm_kv_append(wide, 16, 2 ** 16, 16, 2 ** 16, 16, 2 ** 30, None, 0, None, 0, None, None, None, 0, 0, None) == BAD
    assert "too many" in _err()
    n = 2 ** 30
    assert lib.gdsllm_kv_attention(_cache(), 16, 256, 16, 256, n, 4, 16, 1, 1, 16, 16, 1, 1.0, 1, 16, 0, None, 0, None) == BAD
    assert "2^30" in _err()


def test_q_out_apart_from_q():
    rope = (16, 16, 16, 32, 9, None)
    assert capi().gdsllm_kv_append(_cache(), 16, 128, 16, 128, 16, 1, 32, 128, 32, 2, *rope) == BAD and "q_out" in _err()


def test_extension_refuses_host_tensors():
    """The torch entry points name the argument that is not where or what it has to be."""
    e = ext()
    i, f = torch.zeros(2, dtype=torch.int32), torch.zeros(2)
    cache = torch.zeros(1, 1, 16, 64, dtype=torch.int8)
    row = torch.zeros(2, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="kv_assign: lens must be on a GPU"):
        e.kv_assign(i, i, i.view(2, 1), i, i, 16, 4)
    with pytest.raises(RuntimeError, match="kv_append: k_cache must be"):
        e.kv_append(row, row, i, cache, cache, f, f)
    with pytest.raises(RuntimeError, match="kv_attention: k_cache must be"):
        e.kv_attention(row, cache, cache, f, f, i.view(2, 1), i, i, 1.0)
    with pytest.raises(RuntimeError, match="sample_tokens: logits must be"):
        e.sample_tokens(torch.zeros(2, 5), f)


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 32, 128), (64, 8, 128), (32, 2, 256), (8, 1, 64), (128, 1, 64)])
def test_attention_workspace_serves_smaller_calls(heads, kv_heads, dim):
    """A workspace sized for the largest step is enough for every step with fewer requests, rows or tokens."""
    size = capi().gdsllm_kv_attention_workspace_size
    steps = [(r, new, length) for r in (1, 4, 64, 300) for new in (0, 1, 3, 33, 64, 70, 300, 4096)
             for length in (16, 1024, 1025, 2048, 4096, 4097, 131072)]
    sizes = {s: size(s[0], heads, kv_heads, dim, s[1], s[2]) for s in steps}
    for big in steps:
        for small in steps:
            if all(a <= b for a, b in zip(small, big)):
                assert sizes[small] <= sizes[big], (small, big)


def test_assign_outputs_apart_from_every_input():
    """Workgroups read all of lens, delta and free_state while the first writes lens_out and state_out."""
    base = [16, 32, 1, 48, 1, 1, 64, 1, 80, 16, 1, 96, 112, 128]  # lens, delta, ..., free_state, ..., slots, positions, starts
    for lens_out, state_out in ((16, 144), (32, 144), (80, 144), (144, 16), (144, 32), (144, 80), (144, 144)):
        assert capi().gdsllm_kv_assign(*base, lens_out, state_out, None) == BAD
        assert "must not be" in _err()


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
def test_attention_tables_end_before_32_bits(bs):
    """Kernels step up to 4096 tokens past a request's last one in 32 bits: a table that long has to end before."""
    def call(w):
        return capi().gdsllm_kv_attention(_cache(block_size=bs), 16, 128, None, 128, 1, 2, 16, w, w, 16, 16, 1, 1.0, 1, 16, 0, None,
                                          0, None)

    most = (2 ** 31 - 8192) // bs
    assert call(most) == BAD and "null" in _err()
    assert call(most + 1) == BAD and "table_width" in _err()
