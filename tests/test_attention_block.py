"""CPU: the attention block's entry points (head norms with rotation, packed
prompt attention, the 4-bit KV cache) reject bad arguments on the host, before
any device work, with a status and a message that names the call."""
import ctypes as C
from importlib import import_module

import pytest

P = C.c_void_p(64)    # 16-byte aligned, never dereferenced
ODD = C.c_void_p(68)  # not 16-byte aligned


def refused(pkg, rc, text, kind=RuntimeError):
    with pytest.raises(kind) as e:
        pkg.check(rc)
    assert text in str(e.value), str(e.value)


def rope(pkg, **kw):
    a = dict(q=P, ldq=256, k=P, ldk=128, n=3, h=4, kv=2, d=64, qw=P, kw=P, eps=1e-6, pos=P,
             theta=1e6, neox=1, qo=P, ldqo=256, ko=P, ldko=128)
    a.update(kw)
    return pkg.lib().dqmk_qk_norm_rope(*a.values(), None)


@pytest.mark.parametrize("change,text", [
    (dict(n=-1), "counts must not be negative"), (dict(h=-1), "counts must not be negative"),
    (dict(d=63), "positive and even"), (dict(d=0), "positive and even"),
    (dict(d=258, ldq=2000, ldk=2000, ldqo=2000, ldko=2000), "larger than 256"),
    (dict(theta=0.0), "theta"), (dict(theta=float("nan")), "theta"),
    (dict(theta=float("inf")), "theta"),
    (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(ldq=255), "row stride"), (dict(ldko=127), "row stride"),
    (dict(q=None), "null pointer"), (dict(kw=None), "null pointer"),
    (dict(pos=None), "null pointer"), (dict(ko=None), "null pointer"),
])
def test_qk_norm_rope_refusals(pkg, change, text):
    refused(pkg, rope(pkg, **change), text)
    assert pkg.lib().dqmk_last_error().decode().startswith("QkNormRope: ")


def test_qk_norm_rope_nothing_to_do(pkg):
    assert rope(pkg, n=0) == 0
    assert rope(pkg, h=0, kv=0, q=None, k=None) == 0


def prompt(pkg, **kw):
    a = dict(q=P, ldq=256, k=P, ldk=128, v=P, ldv=128, starts=P, seqs=2, n=10, h=4, kv=2, d=64,
             out=P, ldo=256, work=P, size=1 << 30)
    a.update(kw)
    return pkg.lib().dqmk_attention_prompt(*a.values(), None)


@pytest.mark.parametrize("change,text", [
    (dict(n=-1), "counts must not be negative"), (dict(seqs=-1), "counts must not be negative"),
    (dict(h=5), "invalid head configuration"), (dict(kv=0), "invalid head configuration"),
    (dict(d=0), "invalid head configuration"),
    (dict(d=66, ldq=1000, ldk=1000, ldv=1000, ldo=1000), "multiple of 4"),
    (dict(d=132, ldq=1000, ldk=1000, ldv=1000, ldo=1000), "at most 128"),
    (dict(ldq=252), "row stride"), (dict(ldv=124), "row stride"), (dict(ldo=100), "row stride"),
    (dict(v=None), "null pointer"), (dict(starts=None), "null pointer"),
    (dict(work=None), "null pointer"),
    (dict(q=ODD), "16-byte aligned"), (dict(out=ODD), "16-byte aligned"),
    (dict(ldk=130), "16-byte aligned"), (dict(size=8), "workspace of 8 bytes"),
])
def test_attention_prompt_refusals(pkg, change, text):
    refused(pkg, prompt(pkg, **change), text)
    assert pkg.lib().dqmk_last_error().decode().startswith("AttentionPrompt: ")


def test_attention_prompt_nothing_to_do(pkg):
    assert prompt(pkg, n=0) == 0
    assert prompt(pkg, seqs=0) == 0
    assert pkg.lib().dqmk_attention_prompt_workspace(0, 1, 4, 2, 64) == 0
    assert pkg.lib().dqmk_attention_prompt_workspace(10, 1, 5, 2, 64) == 0
    assert pkg.lib().dqmk_attention_prompt_workspace(10, 1, 4, 2, 64) > 0


def cache(pkg, **kw):
    a = dict(keys=64, values=128, layers=2, slots=3, seq=40, kv=2, dim=64)
    a.update(kw)
    return import_module(pkg.__name__ + "._lib").KvQ40(*a.values())


def write(pkg, kv=None, **kw):
    a = dict(layer=1, k=P, ldk=128, v=P, ldv=128, slots=P, pos=P, n=5)
    a.update(kw)
    return pkg.lib().dqmk_kv_q40_write(C.byref(kv or cache(pkg)), *a.values(), None)


def read(pkg, kv=None, **kw):
    a = dict(layer=1, slots=P, pos=P, n=5, k=P, ldk=128, v=P, ldv=128)
    a.update(kw)
    return pkg.lib().dqmk_kv_q40_read(C.byref(kv or cache(pkg)), *a.values(), None)


def decode(pkg, kv=None, **kw):
    a = dict(layer=1, q=P, ldq=256, slots=P, lengths=P, n=5, h=4, out=P, ldo=256, work=P,
             size=1 << 30)
    a.update(kw)
    return pkg.lib().dqmk_kv_q40_attention(C.byref(kv or cache(pkg)), *a.values(), None)


CACHES = [
    (dict(keys=None), "null pointer", RuntimeError), (dict(values=None), "null pointer", RuntimeError),
    (dict(layers=0), "invalid cache shape", RuntimeError),
    (dict(slots=-1), "invalid cache shape", RuntimeError),
    (dict(seq=0), "invalid cache shape", RuntimeError),
    (dict(kv=0), "invalid cache shape", RuntimeError),
    (dict(dim=48), "multiple of 32", RuntimeError), (dict(dim=160), "at most 128", RuntimeError),
    (dict(keys=72), "16-byte aligned", RuntimeError),
]


@pytest.mark.parametrize("change,text,kind", CACHES)
def test_cache_refusals(pkg, change, text, kind):
    kv = cache(pkg, **change)
    for call, name in ((write, "KvQ40Write"), (read, "KvQ40Read"), (decode, "KvQ40Attention")):
        refused(pkg, call(pkg, kv), text, kind)
        assert pkg.lib().dqmk_last_error().decode().startswith(name + ": ")


@pytest.mark.parametrize("call", [write, read, decode])
def test_cache_layer_out_of_range(pkg, call):
    for layer in (-1, 2):
        refused(pkg, call(pkg, layer=layer), "layer out of range", pkg.OutOfRange)


@pytest.mark.parametrize("call", [write, read])
@pytest.mark.parametrize("change,text", [
    (dict(n=-1), "negative token count"), (dict(ldk=127), "row stride"),
    (dict(ldv=127), "row stride"), (dict(k=None), "null pointer"), (dict(v=None), "null pointer"),
    (dict(pos=None), "null pointer"),
])
def test_cache_rows_refusals(pkg, call, change, text):
    refused(pkg, call(pkg, **change), text)
    assert call(pkg, n=0) == 0


@pytest.mark.parametrize("change,text", [
    (dict(h=3), "invalid head configuration"), (dict(h=0), "invalid head configuration"),
    (dict(n=-1), "negative column count"), (dict(ldq=255), "row stride"),
    (dict(ldo=10), "row stride"), (dict(q=None), "null pointer"),
    (dict(lengths=None), "null pointer"), (dict(out=None), "null pointer"),
    (dict(work=None), "null pointer"), (dict(work=ODD), "16-byte aligned"),
    (dict(size=4), "workspace of 4 bytes"),
])
def test_cache_attention_refusals(pkg, change, text):
    refused(pkg, decode(pkg, **change), text)
    assert decode(pkg, n=0) == 0


def test_cache_bytes(pkg):
    L = pkg.lib()
    # 18 bytes for 32 values, positions padded to whole tiles of 32
    assert L.dqmk_kv_q40_bytes(2, 3, 40, 4, 128) == 2 * 3 * 4 * 64 * 4 * 18
    assert L.dqmk_kv_q40_bytes(1, 1, 1, 1, 32) == 32 * 18
    for bad in ((0, 1, 1, 1, 32), (1, 1, 1, 1, 16), (1, 1, 1, 1, 160), (1, -1, 1, 1, 32)):
        assert L.dqmk_kv_q40_bytes(*bad) == 0
    # more than 32 bits of bytes
    assert L.dqmk_kv_q40_bytes(28, 64, 65536, 4, 128) == 28 * 64 * 65536 * 4 * 4 * 18
    kv = cache(pkg)
    assert L.dqmk_kv_q40_attention_workspace(C.byref(kv), 5, 4) > 0
    assert L.dqmk_kv_q40_attention_workspace(C.byref(kv), 5, 3) == 0
    assert L.dqmk_kv_q40_attention_workspace(C.byref(kv), 0, 4) == 0


def test_python_wrappers_refuse_host_tensors(pkg):
    import torch
    x = torch.zeros(2, 4, 64)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="QkNormRope: q must be"):
        pkg.qk_norm_rope(x, x, x[0, 0], x[0, 0], i, 1e6, 1e-6)
    with pytest.raises(RuntimeError, match="AttentionPrompt: q must be"):
        pkg.attention_prompt(x, x, x, i)
    with pytest.raises(RuntimeError, match="KvCacheQ40: unsupported shape"):
        pkg.KvCacheQ40(1, 1, 8, 1, 48)


def test_attention_prompt_heads_that_share_keys(pkg):
    heads = (1 << 20) + 1
    refused(pkg, prompt(pkg, n=1, seqs=1, h=heads, kv=1, d=4, ldq=4 * heads, ldo=4 * heads,
                        size=1 << 40), "too many query heads")


def test_attention_prompt_output_is_no_input(pkg):
    for name in "qkv":
        inputs = {x: P if x == name else C.c_void_p(8192) for x in "qkv"}
        refused(pkg, prompt(pkg, **inputs), "out must not be an input")


def test_kv_q40_bytes_past_64_bits(pkg):
    big, odd = 1 << 30, (1 << 30) + 1  # the product keeps low bits when it wraps
    assert pkg.lib().dqmk_kv_q40_bytes(odd, odd, odd, 1, 32) == 0
    kv = cache(pkg, layers=odd, slots=odd, seq=odd, kv=1, dim=32)
    for call in (write, read, decode):
        refused(pkg, call(pkg, kv), "too large")
    assert pkg.lib().dqmk_kv_q40_bytes(1, 1, big, 1, 32) == 18 * big
