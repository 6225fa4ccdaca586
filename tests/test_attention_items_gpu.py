"""GPU: packed prompts whose items exceed the CTAs, so that a CTA takes several
items of several key tiles each, in every build of the kernel; and the 4-bit
cache's bytes behind a length."""
import pytest

from test_attention_block_gpu import check_prompt, fill, gen, i32, randn  # noqa: F401

pytestmark = pytest.mark.gpu

# the 128-wide build; the 64-wide one with one CTA an SM (up to 4 items each), with two
PACKS = [((28, 4, 128), [600] * 4 + [1, 130, 64, 65] * 6), ((12, 3, 80), [700, 600, 600, 500] * 2 + [0, 1, 129] * 9),
         ((14, 2, 64), [1024, 500, 700]), ((8, 8, 64), [800, 700, 900, 500, 450, 410]), ((9, 3, 36), [600] * 8 + [3, 65]),
         ((14, 2, 64), [600] * 16), ((3, 1, 20), [1300] * 20)]


@pytest.mark.parametrize("heads,lengths", PACKS, ids=lambda x: "_".join(map(str, x)) if len(x) == 3 else f"{len(x)}x{max(x)}")
def test_attention_prompt_several_items_a_cta(pkg, cuda, gen, heads, lengths):  # noqa: F811
    torch = cuda
    h, kv, d = heads
    starts = [0]
    for x in lengths:
        starts.append(starts[-1] + x)
    n = starts[-1]
    items = kv * sum(-(-x * (h // kv) // 128) for x in lengths)
    assert items > 148
    q, k, v = (randn(torch, gen, n, x, d) for x in (h, kv, kv))
    v[:starts[1]] *= 2.0 ** 20
    k[starts[1]:starts[2]] *= torch.exp2(torch.randint(-5, 6, (lengths[1], 1, 1), generator=gen, device="cuda").float())
    out = pkg.attention_prompt(q, k, v, i32(torch, starts))
    for a, b in zip(starts[:-1], starts[1:]):
        # scores of hundreds in the second sequence
        check_prompt(torch, out[a:b], q[a:b], k[a:b], v[a:b], [0, b - a], f"from {a}",
                     norm=2.0 ** -14 if a == starts[1] else 2.0 ** -19)
    for _ in range(3):
        assert torch.equal(out, pkg.attention_prompt(q, k, v, i32(torch, starts)))


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (5, 1, 32), (6, 2, 96)], ids=lambda h: "h%d_kv%d_d%d" % h)
def test_cache_attention_bytes_behind_the_length(pkg, cuda, gen, heads):  # noqa: F811
    """The same rows in a cache whose other bytes are 0xff and in one that holds
    other rows behind them: the same bits."""
    torch = cuda
    h, kv, d = heads
    lengths = [70, 199, 1, 32]
    full, _, _ = fill(pkg, torch, gen, 1, 4, 300, kv, d, 0, poison=False)
    bare = pkg.KvCacheQ40(1, 4, 300, kv, d)
    bare.keys.fill_(255)
    bare.values.fill_(255)
    for s, n in enumerate(lengths):
        k, v = randn(torch, gen, n, kv, d), randn(torch, gen, n, kv, d)
        p = torch.arange(n, device="cuda", dtype=torch.int32)
        for cache in (full, bare):
            cache.write(0, k, v, p, torch.full_like(p, s))
        for x, y in zip(full.read(0, p, torch.full_like(p, s)), bare.read(0, p, torch.full_like(p, s))):
            assert torch.equal(x, y)
    q = randn(torch, gen, 4, h, d)
    n = i32(torch, lengths)
    out = bare.attention(q, 0, n)
    assert bool(out.isfinite().all())
    assert torch.equal(full.attention(q, 0, n), out)


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_cache_rows_written_back_stay(pkg, cuda, gen, dim):  # noqa: F811
    """The values that a row holds quantize to themselves: the largest of a block
    of codes 1..15 is 7 steps away at most, 7 d is exact and divided by 7 is d."""
    torch = cuda
    n, kv = 300, 2
    a, b = (pkg.KvCacheQ40(1, 1, n, kv, dim) for _ in "ab")
    p = torch.arange(n, device="cuda", dtype=torch.int32)
    k, v = (randn(torch, gen, n, kv, dim).clamp(-3, 3) for _ in "kv")
    a.write(0, k, v, p, torch.zeros_like(p))
    held = a.read(0, p, torch.zeros_like(p))
    b.write(0, *held, p, torch.zeros_like(p))
    for x, y in zip(held, b.read(0, p, torch.zeros_like(p))):
        assert torch.equal(x, y)
