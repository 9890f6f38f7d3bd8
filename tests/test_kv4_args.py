"""Refusals of the 4-bit cache's operators on the CPU: every call here is rejected
before anything touches a device, with a message that names what is wrong."""

import ctypes
import re

import pytest
import torch

from gdsllm_amd import KvCache4, capi
from gdsllm_amd.runtime import ext, kv_cache

BAD = 1


def _err():
    return capi().gdsllm_last_error().decode()


def _cache(**kw):
    base = dict(k=16, v=16, k_affine=16, v_affine=16, num_blocks=4, kv_heads=2, block_size=16, head_dim=64, group_size=32)
    return ctypes.byref(KvCache4(**dict(base, **kw)))


CACHES = [(dict(k=0), "null"), (dict(v_affine=0), "null"), (dict(k=8), "misaligned"), (dict(k_affine=24), "misaligned"),
          (dict(block_size=8), "block_size"), (dict(block_size=48), "block_size"), (dict(block_size=512), "block_size"),
          (dict(head_dim=80), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(kv_heads=0), "kv_heads"),
          (dict(kv_heads=1025), "kv_heads"), (dict(num_blocks=0), "num_blocks"), (dict(num_blocks=2 ** 28), "num_blocks"), (dict(num_blocks=2 ** 21, kv_heads=1024), "kv_heads"),
          (dict(group_size=16), "group_size"), (dict(group_size=48), "group_size"), (dict(group_size=128), "group_size")]


def append(c=None, k=16, ldk=128, v=16, ldv=128, slots=16, n=1, q=None, ldq=0, qo=None, hq=0, pos=None, cos=None, sin=None,
           rot=0, mp=0, nb=0):
    return capi().gdsllm_kv4_append(c or _cache(), k, ldk, v, ldv, slots, n, q, ldq, qo, hq, pos, cos, sin, rot, mp, nb, None)


def attention(c=None, q=16, ldq=128, o=16, ldo=128, n=1, hq=2, tab=16, w=1, ldt=1, lens=16, st=16, b=1, new=1, ml=16, ws=None,
              wb=0, scale=1.0):
    return capi().gdsllm_kv4_attention(c or _cache(), q, ldq, o, ldo, n, hq, tab, w, ldt, lens, st, b, scale, new, ml, 0, ws,
                                       wb, None)


def values(c=None, slots=16, n=1, k=16, v=16):
    return capi().gdsllm_kv4_values(c or _cache(), slots, n, k, v, None)


@pytest.mark.parametrize("kw,word", CACHES, ids=[str(i) for i in range(len(CACHES))])
def test_cache_descriptor(kw, word):
    for call in (append, attention, values):
        assert call(c=_cache(**kw)) == BAD and word in _err()


def test_null_cache():
    lib = capi()
    assert lib.gdsllm_kv4_values(None, 16, 1, 16, 16, None) == BAD and "null cache" in _err()


def test_append_refusals():
    assert append(n=0) == 0 and append(n=0, k=None, v=None, slots=None) == 0
    assert append(n=-1) == BAD and "token" in _err()
    for name in ("k", "v", "slots"):
        assert append(**{name: None}) == BAD and "null" in _err()
    assert append(ldk=64) == BAD and "stride" in _err()
    assert append(ldv=132) == BAD and "multiples of 8" in _err()
    assert append(k=24) == BAD and "aligned" in _err()
    assert append(slots=18) == BAD and "misaligned" in _err()
    for nb in (0, 1):
        rope = dict(pos=16, cos=16, sin=16, rot=32, mp=9, nb=nb)
        assert append(**dict(rope, rot=24)) == BAD and "rotary" in _err()
        assert append(**dict(rope, rot=80)) == BAD and "rotary" in _err()
        assert append(**dict(rope, rot=-16)) == BAD and "rotary" in _err()
        assert append(**dict(rope, pos=None)) == BAD and "positions" in _err()
        assert append(**dict(rope, cos=24)) == BAD and "misaligned" in _err()
        assert append(**dict(rope, mp=0)) == BAD and "positions" in _err()
        assert append(**rope, q=16, qo=None, hq=2, ldq=128) == BAD and "null" in _err()
        assert append(**rope, q=16, qo=32, hq=0, ldq=128) == BAD and "q_heads" in _err()
        assert append(**rope, q=16, qo=32, hq=4, ldq=128) == BAD and "stride" in _err()
        assert append(**rope, q=32, qo=32, hq=2, ldq=128) == BAD and "q_out" in _err()
    assert append(q=16, qo=16, hq=2, ldq=128) == BAD and "rotation" in _err()
    wide = _cache(kv_heads=1024)
    assert append(c=wide, ldk=2 ** 16, ldv=2 ** 16, n=2 ** 30) == BAD and "too many" in _err()


def test_values_refusals():
    assert values(n=0) == 0 and values(n=0, slots=None, k=None, v=None) == 0
    assert values(n=-1) == BAD and "row" in _err()
    for name in ("slots", "k", "v"):
        assert values(**{name: None}) == BAD and "null" in _err()
    assert values(slots=18) == BAD and values(k=24) == BAD and "misaligned" in _err()
    assert values(c=_cache(kv_heads=1024), n=2 ** 30) == BAD and "too many" in _err()


def test_attention_refusals():
    assert attention(n=0) == 0
    for name in ("q", "o", "tab", "lens", "st"):
        assert attention(**{name: None}) == BAD and "null" in _err()
    assert attention(hq=3) == BAD and "multiple of kv_heads" in _err()
    assert attention(hq=0) == BAD
    assert attention(ldq=64) == BAD and "stride" in _err()
    assert attention(ldo=130) == BAD and "multiples of 8" in _err()
    assert attention(q=24) == BAD and "aligned" in _err()
    assert attention(st=18) == BAD and "misaligned" in _err()
    assert attention(ldt=0) == BAD and attention(w=0) == BAD
    assert attention(w=2 ** 28, ldt=2 ** 28) == BAD and "table_width" in _err()
    assert attention(b=70000) == BAD and "requests" in _err()
    assert attention(b=0) == BAD and "requests" in _err()
    assert attention(new=-1) == BAD and attention(ml=-1) == BAD
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert attention(scale=scale) == BAD and "scale" in _err()
    assert attention(n=2 ** 30, hq=4, ldq=256, ldo=256) == BAD and "2^30" in _err()
    lib = capi()
    need = lib.gdsllm_kv4_attention_workspace_size(1, 2, 2, 64, 1, 16 * 1000)
    assert need > 0 and attention(w=1000, ldt=1000, ml=0) == BAD and f"{need} bytes" in _err()
    assert attention(w=1000, ldt=1000, ml=0, ws=16, wb=need - 1) == BAD
    assert lib.gdsllm_kv4_attention_workspace_size(1, 3, 2, 64, 1, 100) == 0


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 32, 128), (64, 8, 128), (32, 2, 256), (8, 1, 64), (128, 1, 64)])
def test_attention_workspace_serves_smaller_calls(heads, kv_heads, dim):
    """A workspace sized for the largest step is enough for every step with fewer requests, rows or tokens."""
    size = capi().gdsllm_kv4_attention_workspace_size
    steps = [(r, new, length) for r in (1, 4, 64, 300) for new in (0, 1, 3, 33, 64, 70, 300, 4096)
             for length in (16, 512, 513, 1024, 1025, 2048, 2049, 4096, 4097, 131072)]
    sizes = {s: size(s[0], heads, kv_heads, dim, s[1], s[2]) for s in steps}
    for big in steps:
        for small in steps:
            if all(a <= b for a, b in zip(small, big)):
                assert sizes[small] <= sizes[big], (small, big)


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 32, 128), (64, 8, 128), (32, 2, 256), (8, 1, 64), (256, 64, 64), (7, 7, 128)])
def test_attention_workspace_covers_the_plan(heads, kv_heads, dim):
    """What a call says that it needs is within the workspace's size for the same step, in every form of the plan (the
    call is refused for its 2^30 tokens in any case)."""
    size, c, shared = capi().gdsllm_kv4_attention_workspace_size, _cache(kv_heads=kv_heads, head_dim=dim, group_size=64), 0
    for r in (1, 2, 3, 4, 5, 16, 40, 300):
        for new in (1, 2, 9, 33, 64, 65, 70, 129, 300, 1000, 4096):
            for length in (512, 1024, 1025, 1300, 2048, 2049, 5000, 131072):
                assert attention(c=c, n=2 ** 30, hq=heads, ldq=heads * dim, ldo=heads * dim, w=8192, ldt=8192, b=r, new=new,
                                 ml=length, ws=None, wb=0) == BAD
                need = re.search(r"workspace of (\d+) bytes", _err())
                assert need or "2^30" in _err(), _err()
                if need:
                    shared += 1
                    assert int(need[1]) <= size(r, heads, kv_heads, dim, new, length), (r, new, length)
    assert shared > 50


def rope(q=16, ldq=128, qo=32, ldqo=128, hq=2, k=16, ldk=64, ko=48, ldko=64, hk=1, d=64, n=2, pos=16, cos=16, sin=16, rot=64,
         mp=9, nb=0):
    return capi().gdsllm_rope(q, ldq, qo, ldqo, hq, k, ldk, ko, ldko, hk, d, n, pos, cos, sin, rot, mp, nb, None)


def test_rope_refusals():
    assert rope(n=0) == 0 and rope(n=0, q=None, pos=None) == 0
    assert rope(n=-1) == BAD and "token" in _err()
    assert rope(d=0) == BAD and rope(d=1025, rot=64) == BAD and "head_dim" in _err()
    for rot in (0, -2, 63, 66):
        assert rope(rot=rot) == BAD and "rotary" in _err()
    assert rope(hq=0) == BAD and "q_heads" in _err()
    assert rope(hk=-1) == BAD and "k_heads" in _err()
    for name in ("q", "qo", "k", "ko", "pos", "cos", "sin"):
        assert rope(**{name: None}) == BAD and "null" in _err()
    assert rope(mp=0) == BAD and "positions" in _err()
    for name in ("ldq", "ldqo", "ldk", "ldko"):
        assert rope(**{name: 63}) == BAD and "stride" in _err()
    assert rope(q=17) == BAD and rope(pos=18) == BAD and rope(cos=18) == BAD and "misaligned" in _err()
    assert rope(qo=16, ldqo=136) == BAD and "in place" in _err()


def test_extension_refuses_host_tensors():
    """The torch entry points name the argument that is not where or what it has to be."""
    e = ext()
    i, f = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 32)
    codes, pairs = torch.zeros(1, 1, 16, 32, dtype=torch.uint8), torch.zeros(1, 1, 2, 16, 2, dtype=torch.float16)
    row = torch.zeros(2, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="rope: q must be"):
        e.rope(row, row, i, f, f)
    with pytest.raises(RuntimeError, match="kv4_append: k_cache must be"):
        e.kv4_append(row, row, i, codes, codes, pairs, pairs)
    with pytest.raises(RuntimeError, match="kv4_values: k_cache must be"):
        e.kv4_values(i, codes, codes, pairs, pairs)
    with pytest.raises(RuntimeError, match="kv4_attention: k_cache must be"):
        e.kv4_attention(row, codes, codes, pairs, pairs, i.view(2, 1), i, i, 1.0)


@pytest.mark.parametrize("kw,word", [
    (dict(layers=0), "layers"), (dict(requests=0), "requests"), (dict(max_len=0), "max_len"), (dict(kv_heads=0), "kv_heads"),
    (dict(block_size=24), "block_size"), (dict(head_dim=96), "head_dim"), (dict(group_size=16), "group_size"),
    (dict(group_size=128), "group_size"), (dict(num_blocks=0), "num_blocks"), (dict(num_blocks=2 ** 27), "num_blocks")])
def test_cache_refusals(kw, word):
    base = dict(layers=1, requests=3, max_len=64, kv_heads=2, head_dim=64, block_size=16, device="cpu")
    with pytest.raises(ValueError, match=word):
        kv_cache.KVCache4(**dict(base, **kw))


@pytest.mark.parametrize("bs", [16, 32, 64, 128, 256])
def test_attention_tables_end_before_32_bits(bs):
    """Kernels step up to 4096 tokens past a request's last one in 32 bits: a table that long has to end before."""
    most = (2 ** 31 - 8192) // bs
    assert attention(c=_cache(block_size=bs), w=most, ldt=most, o=None) == BAD and "null" in _err()
    assert attention(c=_cache(block_size=bs), w=most + 1, ldt=most + 1, o=None) == BAD and "table_width" in _err()
    with pytest.raises(ValueError, match="max_len"):
        kv_cache.KVCache4(1, 1, bs * most + 1, 1, 64, bs, num_blocks=2, group_size=32, device="meta")
    assert kv_cache.KVCache4(1, 1, bs * most, 1, 64, bs, num_blocks=2, group_size=32, device="meta").max_len == bs * most


def test_caches_refuse_what_their_kernels_refuse():
    """Before they allocate anything: more key heads than a call takes, more (block, head) than the 4-bit kernels count."""
    for cls in (kv_cache.KVCache8, kv_cache.KVCache4):
        with pytest.raises(ValueError, match="kv_heads"):
            cls(1, 1, 64, 1025, 64, 16, device="meta")
        assert cls(1, 1, 64, 1024, 64, 16, device="meta").kv_heads == 1024
    with pytest.raises(ValueError, match="num_blocks . kv_heads"):
        kv_cache.KVCache4(1, 1, 64, 1024, 64, 16, num_blocks=2 ** 21, group_size=32, device="meta")
    with pytest.raises(ValueError, match="num_blocks . kv_heads"):
        kv_cache.KVCache4(1, 8192, 4096, 1024, 64, 16, group_size=32, device="meta")
    kv_cache.KVCache4(1, 1, 64, 1023, 64, 16, num_blocks=2 ** 21, group_size=32, device="meta")


def test_rope_outputs_apart():
    """Rows of 128 and 64 halves (256 and 128 bytes) 512 bytes apart: outputs may lie between the inputs' rows, not on them."""
    ld = dict(ldq=256, ldqo=256, ldk=256, ldko=256, n=3)
    far = dict(q=2 ** 20, qo=2 ** 21, k=2 ** 22, ko=2 ** 23)
    def refused(**kw):
        return rope(**{**ld, **far, **kw}) == BAD and "overlap" in _err()

    q = far["q"]
    assert refused(qo=q + 16) and refused(qo=q - 16) and refused(qo=q + 240) and refused(qo=q + 512) and refused(qo=q + 2 * 512 + 240)
    assert refused(ko=q) and refused(ko=q + 240) and refused(k=q, qo=q) and refused(k=q, ko=q, qo=q)
    assert refused(k=q + 128, ko=q + 128, qo=q) and refused(ko=far["qo"]) and refused(ko=far["qo"] + 512 - 112)
    assert refused(ko=far["k"] + 64) and refused(k=far["qo"] + 128)
    # rows of other distances, in the same memory; a single row
    assert refused(ldqo=384, qo=q + 256) and refused(n=1, qo=q + 16) and refused(n=1, k=q + 128, ko=q + 128, qo=q)
