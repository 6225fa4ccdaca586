"""GPU: attention whose operands are far from 1, or far from each other, in size.
References and bounds are those of the attention block's tests: a score is off
by at most (16 + 6 D) e sum |q k| / sqrt(D), e = 2^-24, whatever the sizes."""
import pytest

from test_attention_block_gpu import (attend, check_close, check_decode, check_prompt, gen, i32,  # noqa: F401
                                      randn)

pytestmark = pytest.mark.gpu

HEADS = [(14, 2, 64), (28, 4, 128)]


@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "h%d_kv%d_d%d" % h)
@pytest.mark.parametrize("qs,ks", [(1e-18, 1e-18), (1e-25, 1e-25), (1e-38, 1e-38), (1e-30, 1e-5),
                                   (1e18, 1e-18), (1e-30, 1e30), (1e36, 1e-36), (1e-12, 1.0)])
def test_attention_prompt_far_from_one(pkg, cuda, gen, heads, qs, ks):  # noqa: F811
    """Queries and keys of any size: products of their sizes that leave a
    float's range downwards are scores of zero, a plain mean."""
    torch = cuda
    h, kv, d = heads
    starts = [0, 70, 71, 200]
    q, k, v = (randn(torch, gen, 200, x, d) for x in (h, kv, kv))
    q, k = q * qs, k * ks
    out = pkg.attention_prompt(q, k, v, i32(torch, starts))
    check_prompt(torch, out, q, k, v, starts)


@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "h%d_kv%d_d%d" % h)
@pytest.mark.parametrize("which", [1, 2], ids=["key", "value"])
def test_attention_prompt_large_queries_before_an_infinity(pkg, cuda, gen, heads, which):  # noqa: F811
    """A later token's infinity, in the same tile of keys, reaches no earlier
    token, however large their queries are."""
    torch = cuda
    h, kv, d = heads
    n, at = 100, 90
    for size in (2.0 ** 33, 2.0 ** 40, 2.0 ** 100):
        x = [randn(torch, gen, n, y, d) for y in (h, kv, kv)]
        x[0] *= size
        x[1] /= size
        x[which][at, 1, 3] = float("inf")
        out = pkg.attention_prompt(*x, i32(torch, [0, n]))
        check_prompt(torch, out[:at], *(y[:at] for y in x), [0, at], f"{size} before")
        g = h // kv
        check_prompt(torch, out[:, :g], x[0][:, :g], x[1][:, :1], x[2][:, :1], [0, n], f"{size} beside")


def spread(torch, gen, n, bits):  # noqa: F811
    """n powers of two, 2^-bits among them, and 1."""
    e = -torch.randint(0, bits + 1, (n,), generator=gen, device="cuda").float()
    e[n // 3], e[n // 2] = -bits, 0
    return torch.exp2(e)


@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "h%d_kv%d_d%d" % h)
@pytest.mark.parametrize("rows", [0, 8, 12, 15])
@pytest.mark.parametrize("channels", [0, 5, 7, 10, 14])
def test_attention_prompt_keys_of_many_sizes(pkg, cuda, gen, heads, rows, channels):  # noqa: F811
    """Channels of the keys that differ in size, the queries' the other way
    round, so that each counts the same in a score; and among the rows of a tile
    of keys some that are 2^rows larger and weigh nothing: their scores are far
    below the others', or they come behind the tokens that are looked at."""
    torch = cuda
    h, kv, d = heads
    n = 130
    q, k, v = (randn(torch, gen, n, x, d) for x in (h, kv, kv))
    c = spread(torch, gen, d, channels)
    q[..., 0] = q[..., 0].abs() + 1.0
    for large in (20, 85):
        k[large] *= 2.0 ** rows
        if rows:
            k[large] *= 0.01
            k[large, :, 0] = -8.0 * 2.0 ** rows  # a score of about -2^rows or less
    k[60] *= 2.0 ** rows
    k[128] *= 2.0 ** rows
    q, k = q / c, k * c
    starts = [0, n]
    out = pkg.attention_prompt(q, k, v, i32(torch, starts))
    # tokens up to the first large key see none, those up to key 60 one of no weight
    check_prompt(torch, out[:20], q[:20], k[:20], v[:20], [0, 20], f"{rows} {channels} first")
    check_prompt(torch, out[:60], q[:60], k[:60], v[:60], [0, 60], f"{rows} {channels}", norm=0)
    check_prompt(torch, out, q, k, v, starts, f"{rows} {channels} all", norm=0)


@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "h%d_kv%d_d%d" % h)
@pytest.mark.parametrize("rows,channels", [(0, 10), (0, 14), (7, 7), (0, 20), (0, 24), (0, 40), (12, 12),
                                           (15, 10), (15, 1)])
def test_attention_prompt_values_of_many_sizes(pkg, cuda, gen, heads, rows, channels):  # noqa: F811
    """Channels of the values that differ by up to 2^40, and rows: every output
    channel to its own precision, whatever the others' size."""
    torch = cuda
    h, kv, d = heads
    starts = [0, 1, 33, 163]
    q, k, v = (randn(torch, gen, 163, x, d) for x in (h, kv, kv))
    v *= spread(torch, gen, d, channels)
    v *= spread(torch, gen, 163, rows)[:, None, None]
    out = pkg.attention_prompt(q, k, v, i32(torch, starts))
    check_prompt(torch, out, q, k, v, starts, f"{rows} {channels}")


@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** -9, 2.0 ** -1, 1.0, 2.0 ** 4, 2.0 ** 7, 2.0 ** 12])
@pytest.mark.parametrize("channels", [6, 10, 13])
def test_attention_prompt_queries_of_many_sizes(pkg, cuda, gen, size, channels):  # noqa: F811
    """Query rows of any size whose channels differ, the keys' the other way round."""
    torch = cuda
    n, h, kv, d = 140, 14, 2, 64
    q, k, v = (randn(torch, gen, n, x, d) for x in (h, kv, kv))
    c = spread(torch, gen, d, channels)
    c[-8:] = 2.0 ** -channels
    q = q * c * size
    q[::7, 1:] *= 0.01  # rows whose largest channel stands out
    k = k / c / size
    starts = [0, n]
    out = pkg.attention_prompt(q, k, v, i32(torch, starts))
    check_prompt(torch, out, q, k, v, starts, f"{size} {channels}", norm=0)


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (3, 3, 36), (6, 1, 80), (130, 1, 32)],
                         ids=lambda h: "h%d_kv%d_d%d" % h)
@pytest.mark.parametrize("which", ["keys", "values", "both"])
@pytest.mark.parametrize("lengths", [[300, 1, 70], [40, 64, 65, 3], [600] * 20], ids=lambda n: f"{len(n)}x{max(n)}")
def test_attention_prompt_marked_tiles(pkg, cuda, gen, heads, which, lengths):  # noqa: F811
    """Rows of almost nothing (not zeros) in some tiles of the keys, of the
    values, or of both: the tiles taken in f32 between others, first and last
    ones among them, give what the formula gives, the same each time."""
    torch = cuda
    h, kv, d = heads
    starts = [0]
    for x in lengths:
        starts.append(starts[-1] + x)
    n = starts[-1]
    q, k, v = (randn(torch, gen, n, x, d) for x in (h, kv, kv))
    for s, x in zip(starts, lengths):
        for at in (0, 130, x - 1):
            if at < x and x > 1:
                if which != "values":
                    k[s + at] *= 1e-9
                if which != "keys":
                    v[s + at] *= 1e-9
    if which == "both":
        v[starts[-2] + lengths[-1] // 2:, :, 0] *= 2.0 ** 40
    out = pkg.attention_prompt(q, k, v, i32(torch, starts))
    check_prompt(torch, out, q, k, v, starts)
    assert torch.equal(out, pkg.attention_prompt(q, k, v, i32(torch, starts)))


def blocks(torch, d, bits):
    """A power of two for each channel, the same in a block of 32: 1, and 2^-bits in every other block."""
    c = torch.ones(d, device="cuda")
    c.view(-1, 32)[1::2] = 2.0 ** -bits
    return c


def cache_of(pkg, torch, k, v):
    """One sequence's cache of these rows, and the values it holds."""
    n, kv, d = k.shape
    cache = pkg.KvCacheQ40(1, 1, n, kv, d)
    p = torch.arange(n, device="cuda", dtype=torch.int32)
    cache.write(0, k, v, p, torch.zeros_like(p))
    ks, vs = cache.read(0, p, torch.zeros_like(p))
    return cache, ks[None], vs[None]


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (5, 1, 96)], ids=lambda h: "h%d_kv%d_d%d" % h)
@pytest.mark.parametrize("bits", [6, 10, 14, 18, 22])
@pytest.mark.parametrize("size", [1.0, 100.0, 2.0 ** -5])
def test_cache_attention_value_blocks_of_many_sizes(pkg, cuda, gen, heads, bits, size):  # noqa: F811
    """Blocks of the values that differ by up to 2^22, also where the large ones
    come late or in few rows.  Beside the bound of any attention here, a
    product of a weight and a scale is off by 2^-32 of the largest weight times the
    largest scale, and a value is up to 8 times its scale (its block's largest at
    least 7 times)."""
    torch = cuda
    h, kv, d = heads
    n = 1100
    for late in (0, 1, 700):
        k, v = (randn(torch, gen, n, kv, d) for _ in "kv")
        v *= size * blocks(torch, d, bits)
        v[:late, :, :32] *= 2.0 ** -bits  # all small at first
        v[40:48] = 0
        v[300:420, :, -32:] *= 2.0 ** -4
        cache, ks, vs = cache_of(pkg, torch, k, v)
        q = randn(torch, gen, 1, h, d)
        for length in (1, 2, 33, 45, 140, 701, 1100):
            out = cache.attention(q, 0, i32(torch, [length]), i32(torch, [0]))
            kk, vv = (x[0, :length].permute(1, 0, 2).repeat_interleave(h // kv, 0).double() for x in (ks, vs))
            seen = torch.ones(1, length, dtype=torch.bool, device="cuda")
            ref, bound = attend(torch, q[0][:, None], kk, vv, seen)
            p = torch.softmax(q[0].double()[:, None] @ kk.transpose(-1, -2) / d ** 0.5, -1)
            largest = p.amax(-1, keepdim=True) * vv.abs().amax((1, 2))[:, None, None] / 7
            check_close(out[0][:, None], ref, bound + 8 * length * 2.0 ** -32 * largest,
                        f"{bits} {size} {late} {length}")


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128)], ids=lambda h: "h%d_kv%d_d%d" % h)
@pytest.mark.parametrize("bits", [6, 10, 12])
def test_cache_attention_key_blocks_of_many_sizes(pkg, cuda, gen, heads, bits):  # noqa: F811
    """Blocks of the keys that differ in size, the queries' the other way round."""
    torch = cuda
    h, kv, d = heads
    k, v = (randn(torch, gen, 700, kv, d) for _ in "kv")
    c = blocks(torch, d, bits)
    cache, ks, vs = cache_of(pkg, torch, k * c, v)
    q = randn(torch, gen, 1, h, d) / c
    for length in (1, 45, 700):
        out = cache.attention(q, 0, i32(torch, [length]), i32(torch, [0]))
        check_decode(torch, out, q, ks, vs, [length], [0], f"{bits}")
