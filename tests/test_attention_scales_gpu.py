"""GPU: attention whose operands are far from 1, or far from each other, in size.
References and bounds are those of the attention block's tests: a score is off
by at most (16 + 6 D) e sum |q k| / sqrt(D), e = 2^-24, whatever the sizes."""
import pytest

from test_attention_block_gpu import check_prompt, gen, i32, randn  # noqa: F401

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
