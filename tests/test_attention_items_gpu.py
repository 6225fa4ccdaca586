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


def spread(torch, gen, n, bits):  # noqa: F811
    return torch.exp2(-torch.rand(n, generator=gen, device="cuda") * bits)


def off_by(torch, x):
    """How far a key or value may be off: 2^-22 of itself or 2^-23 r c / t, the
    largest of its row, its channel and its tile of 64 tokens."""
    a = x.abs().double()
    out = torch.zeros_like(a)
    for t in range(0, x.shape[0], 64):
        b = a[t:t + 64]
        r, c, top = b.amax(2), b.amax(0), b.amax((0, 2)).clamp(min=1e-300)
        out[t:t + 64] = torch.maximum(b * 2.0 ** -22, 2.0 ** -23 * r[:, :, None] * c[None] / top[None, :, None])
    return out


@pytest.mark.parametrize("seed", range(12))
def test_attention_prompt_stated_bounds(pkg, cuda, seed):
    """Rows and channels of random sizes on both sides of what marks a tile:
    outputs within what follows from the errors stated for queries (2^-22, or
    2^-34 of the row's largest), keys, values and weights (2^-22, or 2^-39 of the
    row's largest), with f32 sums (6 e a term and addition, as in the tests of
    the attention block) and 2^-22 of a score for its scaling and exponent."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(seed)  # noqa: F811
    h, kv, d = [(14, 2, 64), (6, 2, 128), (9, 1, 36), (5, 5, 100)][seed % 4]
    lengths = [[200, 1, 33], [64, 65, 3, 130], [500]][seed % 3]
    starts = [0]
    for x in lengths:
        starts.append(starts[-1] + x)
    n = starts[-1]
    size, channels = 2.0 ** (0, -12, 7, -40)[seed % 4], spread(torch, gen, d, (0, 7, 12)[seed % 3])
    q = randn(torch, gen, n, h, d) * channels * size
    k = randn(torch, gen, n, kv, d) / channels / size * spread(torch, gen, n, (0, 6, 20)[seed % 3])[:, None, None]
    v = randn(torch, gen, n, kv, d) * spread(torch, gen, n, (3, 12, 25, 0)[seed % 4])[:, None, None]
    v = v * spread(torch, gen, d, (9, 0, 5, 20, 3)[seed % 5])
    k[n // 2] = 0
    out = pkg.attention_prompt(q, k, v, i32(torch, starts))
    e = 2.0 ** -24
    for a, b in zip(starts[:-1], starts[1:]):
        qs = q[a:b].double().permute(1, 0, 2)
        ks, vs, dk, dv = (x.double().permute(1, 0, 2).repeat_interleave(h // kv, 0)
                          for x in (k[a:b], v[a:b], off_by(torch, k[a:b]), off_by(torch, v[a:b])))
        dq = torch.maximum(qs.abs() * 2.0 ** -22, 2.0 ** -34 * qs.abs().amax(-1, keepdim=True))
        seen = torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").tril()
        root = d ** 0.5
        s = qs @ ks.transpose(-1, -2) / root
        ds = (qs.abs() @ dk.transpose(-1, -2) + dq @ ks.abs().transpose(-1, -2)
              + (6 * d + 8) * e * (qs.abs() @ ks.abs().transpose(-1, -2))) / root + 4 * e * s.abs()
        p = torch.softmax(s.masked_fill(~seen, -float("inf")), -1)
        ds = ds.masked_fill(~seen, 0).amax(-1, keepdim=True)
        bound = ((p @ vs.abs()) * (2 * torch.expm1(ds) + (16 + 6 * (b - a)) * e) + (p * torch.exp(ds)) @ dv
                 + 2.0 ** -38 * p.amax(-1, keepdim=True) * (seen.double() @ vs.abs()))
        off = (out[a:b].double().permute(1, 0, 2) - p @ vs).abs()
        assert bool((off <= bound + 1e-37).all()), float((off / (bound + 1e-37)).max())


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128)], ids=lambda h: "h%d_kv%d_d%d" % h)
def test_attention_prompt_replayed_with_other_sequences(pkg, cuda, gen, heads):  # noqa: F811
    """A captured call replayed with other offsets, rows and sizes in the same
    memory, two graphs in turn on two streams: the bits of plain calls."""
    torch = cuda
    h, kv, d = heads
    n = 400
    q, k, v = (randn(torch, gen, n, x, d) for x in (h, kv, kv))
    starts = i32(torch, [0, 100, 100, 350])
    graphs = []
    for _ in range(2):
        pkg.attention_prompt(q, k, v, starts)
        out = torch.zeros_like(q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            pkg.attention_prompt(q, k, v, starts, out=out)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for offsets, far in (([0, 100, 100, 350], 0), ([0, 1, 2, 3], 0), ([7, 7, 7, 7], 0), ([0, 0, 0, 400], 1),
                         ([2, 66, 131, 400], 2)):
        starts.copy_(i32(torch, offsets))
        k.copy_(randn(torch, gen, n, kv, d))
        v.copy_(randn(torch, gen, n, kv, d))
        if far:
            (k if far == 1 else v)[100] *= 1e-9
        want = pkg.attention_prompt(q, k, v, starts)
        for _, out in graphs:
            out.zero_()
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want)
        check_prompt(torch, want, q, k, v, offsets)
    assert pkg.lib().dqmk_device_error(0) == 0
