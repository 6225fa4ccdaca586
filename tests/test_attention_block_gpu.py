"""GPU: the attention block of many tokens against its formulas in 64 bits:
head norms with the rotary rotation, causal attention over packed prompts, the
4-bit KV cache's write, read-back and decode attention, and all of them in a row.

Tolerances (e = 2^-24, half a step of a float, relative):

norm and rotation: the sum of squares takes at most 16 additions in a lane and
5 across lanes, and enters under a root (11 e); mean, eps, root, quotient and
the two products 6 e; the angle is rounded to 2^-25 half turns (pi / 2 e),
sine and cosine to 2 e, the rotation 3 e.  Under 32 e of the pair's length.

attention: a score is a sum of D products of operands of 22 bits (three
products of 2^-22 = 12 e, at most 6 D e for the order of 3 D additions, 4 e for
scaling), so it is off by at most (16 + 6 D) e sum |q k| / sqrt(D); a weight by
that much of itself, the norm likewise, and the weighted sum of values by
another (16 + 6 n) e in the worst order of n additions.  That is the bound for
each value.  Errors of such sums are independent in fact: over a whole output
they come to a few 2^-22, and 2^-19 of its norm is asked for.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


@pytest.fixture()
def gen(cuda):
    return cuda.Generator(device="cuda").manual_seed(1234)


def randn(torch, gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def i32(torch, values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------ norm and rotation
def rope_reference(torch, x, w, pos, theta, eps, neox):
    x = x.double()
    d = x.shape[-1]
    n = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + eps) * w.double()
    freq = torch.tensor([theta ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64,
                        device="cuda")
    a = (pos.double()[:, None] * freq)[:, None]
    p, q = (n[..., :d // 2], n[..., d // 2:]) if neox else (n[..., 0::2], n[..., 1::2])
    y = (p * a.cos() - q * a.sin(), p * a.sin() + q * a.cos())
    out = torch.cat(y, -1) if neox else torch.stack(y, -1).flatten(-2)
    size = torch.hypot(p, q)
    size = torch.cat([size, size], -1) if neox else torch.stack([size, size], -1).flatten(-2)
    return out, size


def check_rope(torch, y, x, w, pos, theta, eps, neox):
    ref, size = rope_reference(torch, x, w, pos, theta, eps, neox)
    off = (y.double() - ref).abs() - 32 * E * size
    assert bool((off <= 1e-37).all()), float(off.max())


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("dim", [2, 6, 32, 64, 80, 96, 128, 200, 256])
@pytest.mark.parametrize("heads", [(14, 2), (5, 1), (3, 3), (40, 8)])
def test_qk_norm_rope(pkg, cuda, gen, heads, dim, neox):
    torch = cuda
    h, kv = heads
    for n, theta, eps in ((1, 1e6, 1e-6), (7, 1e4, 1e-5)):
        q, k = randn(torch, gen, n, h, dim) * 3, randn(torch, gen, n, kv, dim)
        qw, kw = 1 + 0.1 * randn(torch, gen, dim), 1 + 0.1 * randn(torch, gen, dim)
        pos = torch.randint(-5, 1_000_000, (n,), generator=gen, device="cuda", dtype=torch.int32)
        qo, ko = pkg.qk_norm_rope(q, k, qw, kw, pos, theta, eps, neox)
        check_rope(torch, qo, q, qw, pos, theta, eps, neox)
        check_rope(torch, ko, k, kw, pos, theta, eps, neox)


@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_qk_norm_rope_views_in_place(pkg, cuda, gen, dim, shift):
    """Heads inside the rows of one fused product, at any alignment, in place:
    the same bits as from separate tensors, and nothing else of the rows changes."""
    torch = cuda
    n, h, kv = 5, 6, 2
    width = (h + 2 * kv) * dim + 4
    flat = randn(torch, gen, n * width + shift)
    rows = flat[shift:].view(n, width)
    q = rows[:, :h * dim].view(n, h, dim)
    k = rows[:, h * dim:(h + kv) * dim].view(n, kv, dim)
    w = 1 + 0.1 * randn(torch, gen, dim)
    pos = i32(torch, [0, 3, 2047, 2 ** 31 - 1, -(2 ** 31)])
    want = [t.clone() for t in (q, k, rows[:, (h + kv) * dim:], flat[:shift])]
    apart = pkg.qk_norm_rope(want[0], want[1], w, w, pos, 1e6, 1e-6)
    pkg.qk_norm_rope(q, k, w, w, pos, 1e6, 1e-6, q_out=q, k_out=k)
    check_rope(torch, q, want[0], w, pos, 1e6, 1e-6, True)
    check_rope(torch, k, want[1], w, pos, 1e6, 1e-6, True)
    if shift != 1:  # the same variant
        assert torch.equal(q, apart[0]) and torch.equal(k, apart[1])
    assert torch.equal(rows[:, (h + kv) * dim:], want[2]) and torch.equal(flat[:shift], want[3])


def test_qk_norm_rope_special_rows(pkg, cuda, gen):
    """A zero row stays zero, a row with a NaN is NaN by itself, no heads of one kind."""
    torch = cuda
    q, k = randn(torch, gen, 3, 4, 64), randn(torch, gen, 3, 2, 64)
    q[0, 1] = 0
    q[1, 2, 5] = float("nan")
    w = torch.ones(64, device="cuda")
    pos = i32(torch, [1, 2, 3])
    qo, ko = pkg.qk_norm_rope(q, k, w, w, pos, 1e6, 1e-6)
    assert float(qo[0, 1].abs().max()) == 0.0
    assert bool(qo[1, 2].isnan().all())
    qo[1, 2] = 0
    assert bool(qo.isfinite().all()) and bool(ko.isfinite().all())
    none = torch.empty(3, 0, 64, device="cuda")
    qo2, _ = pkg.qk_norm_rope(q, none, w, w, pos, 1e6, 1e-6)
    assert torch.equal(qo2[0], qo[0])
    _, ko2 = pkg.qk_norm_rope(none, k, w, w, pos, 1e6, 1e-6)
    assert torch.equal(ko2, ko)


# ------------------------------------------------------------ attention reference
def attend(torch, q, k, v, seen):
    """(out, bound) of softmax(q k^T / sqrt(D)) v in 64 bits; rows that see nothing are 0."""
    q, k, v = q.double(), k.double(), v.double()
    d, n = q.shape[-1], k.shape[-2]
    s = (q @ k.transpose(-1, -2)) / math.sqrt(d)
    size = (q.abs() @ k.abs().transpose(-1, -2)) / math.sqrt(d)
    s = s.masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    p = torch.where(seen.any(-1, keepdim=True), p, torch.zeros_like(p))
    worst = (size.masked_fill(~seen, 0).amax(-1, keepdim=True)) * (16 + 6 * d) * E
    return p @ v, (p @ v.abs()) * (2 * torch.expm1(worst) + (16 + 6 * n) * E)


def check_close(out, ref, bound, label="", norm=2.0 ** -19):
    off = (out.double() - ref).abs()
    assert bool((off <= bound + 1e-37).all()), f"{label}: {float((off - bound).max()):.3e} over"
    size = float(ref.norm())
    if size and norm:
        assert float(off.norm()) <= norm * size, f"{label}: {float(off.norm()) / size:.3e}"


# ------------------------------------------------------------ packed prompts
def check_prompt(torch, out, q, k, v, starts, label="", norm=2.0 ** -19):
    group = q.shape[1] // k.shape[1]
    for a, b in zip(starts[:-1], starts[1:]):
        n = b - a
        if n == 0:
            continue
        seen = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        qs = q[a:b].permute(1, 0, 2)
        ks, vs = (x[a:b].permute(1, 0, 2).repeat_interleave(group, 0) for x in (k, v))
        ref, bound = attend(torch, qs, ks, vs, seen)
        check_close(out[a:b].permute(1, 0, 2), ref, bound, f"{label} {a}..{b}", norm)


LENGTHS = [[1], [2], [17], [63, 64, 65], [127, 128, 129], [0, 5, 0, 0, 31, 0], [300, 1, 1, 40],
           [1] * 70, [602]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda n: f"{len(n)}x{max(n)}")
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (3, 3, 80), (40, 8, 32)],
                         ids=lambda h: "h%d_kv%d_d%d" % h)
def test_attention_prompt(pkg, cuda, gen, heads, lengths):
    torch = cuda
    h, kv, d = heads
    starts = np.concatenate([[0], np.cumsum(lengths)]).tolist()
    n = starts[-1]
    q, k, v = randn(torch, gen, n, h, d), randn(torch, gen, n, kv, d), randn(torch, gen, n, kv, d)
    out = pkg.attention_prompt(q, k, v, i32(torch, starts))
    check_prompt(torch, out, q, k, v, starts)
    assert torch.equal(out, pkg.attention_prompt(q, k, v, i32(torch, starts)))


@pytest.mark.parametrize("dim", [4, 20, 36, 60, 64, 68, 96, 100, 124, 128])
@pytest.mark.parametrize("heads", [(1, 1), (9, 1), (6, 3)])
def test_attention_prompt_head_sizes(pkg, cuda, gen, heads, dim):
    torch = cuda
    h, kv = heads
    starts = [0, 40, 41, 190]
    q, k, v = (randn(torch, gen, 190, x, dim) for x in (h, kv, kv))
    check_prompt(torch, pkg.attention_prompt(q, k, v, i32(torch, starts)), q, k, v, starts)


def test_attention_prompt_views_and_tail(pkg, cuda, gen):
    """Views into fused rows; rows before the first and behind the last sequence stay."""
    torch = cuda
    n, h, kv, d = 200, 4, 2, 64
    rows = randn(torch, gen, n, h + 2 * kv, d)
    q, k, v = rows[:, :h], rows[:, h:h + kv], rows[:, h + kv:]
    wide = torch.full((n, h + 1, d), 7.0, device="cuda")
    starts = [3, 80, 80, 171]
    out = pkg.attention_prompt(q, k, v, i32(torch, starts), out=wide[:, :h])
    check_prompt(torch, out, q, k, v, starts)
    assert bool((wide[:3] == 7).all() and (wide[171:] == 7).all() and (wide[:, h] == 7).all())


def test_attention_prompt_offsets_out_of_range(pkg, cuda, gen):
    """Sequences with offsets out of order or out of range are skipped and recorded."""
    torch = cuda
    n, h, kv, d = 64, 2, 1, 64
    q, k, v = randn(torch, gen, n, h, d), randn(torch, gen, n, kv, d), randn(torch, gen, n, kv, d)
    pkg.lib().dqmk_device_error(1)
    for starts, fine in (([0, 20, 10, 40], [(0, 20), (10, 40)]), ([-4, 8, 30], [(8, 30)]),
                         ([0, 30, 65], [(0, 30)]), ([70, 80], [])):
        out = pkg.attention_prompt(q, k, v, i32(torch, starts),
                                   out=torch.full((n, h, d), 9.0, device="cuda"))
        assert pkg.lib().dqmk_device_error(1) == 8
        kept = torch.ones(n, dtype=torch.bool)
        for a, b in fine:
            kept[a:b] = False
        if len(fine) == 1 or not fine:
            for a, b in fine:
                check_prompt(torch, out, q, k, v, [a, b])
        assert bool((out[kept.cuda()] == 9).all())
    assert pkg.lib().dqmk_device_error(1) == 0


def test_attention_prompt_magnitudes(pkg, cuda, gen):
    """Sequences whose values differ by 2^40 in one pack, rows that differ by
    2^20 in one sequence, and scores of hundreds: each output to the precision
    of its own values."""
    torch = cuda
    h, kv, d = 4, 2, 64
    starts = [0, 150, 300, 450]
    q, k, v = (randn(torch, gen, 450, x, d) for x in (h, kv, kv))
    v[:150] *= 2.0 ** 20
    v[150:300] *= 2.0 ** -20
    v[300:] *= torch.exp2(torch.randint(-10, 11, (150, 1, 1), generator=gen, device="cuda").float())
    k[150:300] *= 30.0
    out = pkg.attention_prompt(q, k, v, i32(torch, starts))
    for a, b in zip(starts[:-1], starts[1:]):
        # scores of hundreds make weights of one: their error is the score's, not 2^-19
        check_prompt(torch, out[a:b], q[a:b], k[a:b], v[a:b], [0, b - a], f"from {a}",
                     norm=2.0 ** -19 if a != 150 else 2.0 ** -14)


def test_attention_prompt_one_key_is_its_value(pkg, cuda, gen):
    """The first token of a sequence sees itself alone: its output is v, to v's
    rounding as two 11-bit terms (2^-22) and the quotient's (2^-24)."""
    torch = cuda
    starts = list(range(0, 40))
    q, k, v = randn(torch, gen, 39, 6, 128), randn(torch, gen, 39, 3, 128), randn(torch, gen, 39, 3, 128)
    out = pkg.attention_prompt(q, k, v, i32(torch, starts))
    ref = v.repeat_interleave(2, 1)
    assert bool(((out - ref).abs() <= 6 * E * ref.abs()).all())


def test_attention_prompt_many_sequences(pkg, cuda, gen):
    """More sequences than a CTA has threads, most of them short or empty."""
    torch = cuda
    h, kv, d = 6, 2, 64
    r = np.random.RandomState(5)
    lengths = r.randint(0, 12, 700)
    lengths[[3, 256, 511, 699]] = [130, 0, 70, 1]
    starts = np.concatenate([[0], np.cumsum(lengths)]).tolist()
    n = starts[-1]
    q, k, v = randn(torch, gen, n, h, d), randn(torch, gen, n, kv, d), randn(torch, gen, n, kv, d)
    out = pkg.attention_prompt(q, k, v, i32(torch, starts))
    # one dense masked product over the whole pack
    seq = torch.searchsorted(i32(torch, starts), torch.arange(n, device="cuda", dtype=torch.int32),
                             right=True)
    at = torch.arange(n, device="cuda")
    seen = (seq[:, None] == seq[None]) & (at[None] <= at[:, None])
    ks, vs = (x.permute(1, 0, 2).repeat_interleave(h // kv, 0) for x in (k, v))
    ref, bound = attend(torch, q.permute(1, 0, 2), ks, vs, seen)
    check_close(out.permute(1, 0, 2), ref, bound)


@pytest.mark.parametrize("heads", [(130, 1), (300, 2)])
def test_attention_prompt_wide_groups(pkg, cuda, gen, heads):
    """Groups of more heads than an item has rows."""
    torch = cuda
    h, kv = heads
    starts = [0, 3, 75]
    q, k, v = (randn(torch, gen, 75, x, 32) for x in (h, kv, kv))
    check_prompt(torch, pkg.attention_prompt(q, k, v, i32(torch, starts)), q, k, v, starts)


def test_attention_prompt_not_finite(pkg, cuda, gen):
    """An infinity or a NaN in a later token's key or value, or in another
    sequence, leaves a token's output as it is without; a NaN query its row's."""
    torch = cuda
    h, kv, d = 4, 2, 64
    starts = [0, 100, 200]
    q, k, v = (randn(torch, gen, 200, x, d) for x in (h, kv, kv))
    want = pkg.attention_prompt(q, k, v, i32(torch, starts))
    for bad in (float("nan"), float("inf"), -float("inf")):
        for which in (1, 2):
            x = [q, k.clone(), v.clone()]
            x[which][70, 1, 3] = bad
            out = pkg.attention_prompt(*x, i32(torch, starts))
            # heads of the other group and tokens before the bad one
            check_prompt(torch, out[:70], q[:70], k[:70], v[:70], [0, 70], "before")
            check_prompt(torch, out[:100, :2], q[:100, :2], k[:100, :1], v[:100, :1], [0, 100], "beside")
            assert torch.equal(out[100:], want[100:])
            if bad != bad:
                assert bool(out[70:100, 2:, 3].isnan().all())
    x = q.clone()
    x[50, 2] = float("nan")
    out = pkg.attention_prompt(x, k, v, i32(torch, starts))
    assert bool(out[50, 2].isnan().all())
    out[50, 2] = want[50, 2]
    assert torch.equal(out, want)


def test_row_strides_past_32_bits(pkg, cuda, gen):
    """Rows so far apart that a token's offset needs more than 32 bits."""
    torch = cuda
    n, h, kv, d = 70, 2, 1, 64
    step = 2 ** 31 // 64 + 4  # elements: row 64 starts past 2^31
    if torch.cuda.mem_get_info()[0] < 40 * 2 ** 30:
        pytest.skip("needs 28 GB of device memory")
    flat = [torch.empty(n * step, device="cuda") for _ in range(3)]
    q, k, v = (f.as_strided((n, x, d), (step, d, 1)) for f, x in zip(flat, (h, kv, kv)))
    small = [randn(torch, gen, n, x, d) for x in (h, kv, kv)]
    for a, b in zip((q, k, v), small):
        a.copy_(b)
    w = torch.ones(d, device="cuda")
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    starts = i32(torch, [0, n])
    want = pkg.qk_norm_rope(small[0], small[1], w, w, pos, 1e6, 1e-6)
    got = pkg.qk_norm_rope(q, k, w, w, pos, 1e6, 1e-6)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(pkg.attention_prompt(q, k, v, starts), pkg.attention_prompt(*small, starts))
    caches = [pkg.KvCacheQ40(1, 1, n, kv, d) for _ in range(2)]
    zero = torch.zeros_like(pos)
    caches[0].write(0, k, v, pos, zero)
    caches[1].write(0, small[1], small[2], pos, zero)
    assert torch.equal(caches[0].keys, caches[1].keys)
    assert torch.equal(caches[0].values, caches[1].values)
    del flat, q, k, v
    torch.cuda.empty_cache()


# ------------------------------------------------------------ 4-bit cache
def fill(pkg, torch, gen, layers, slots, room, kv, d, layer, scale=1.0, poison=True):
    """A cache with random rows at every position of one layer, every other
    byte 0xff (scales that are NaN), and the rows' values."""
    cache = pkg.KvCacheQ40(layers, slots, room, kv, d)
    if poison:
        cache.keys.fill_(255)
        cache.values.fill_(255)
    k, v = (randn(torch, gen, slots * room, kv, d) * scale for _ in "kv")
    s = torch.arange(slots, device="cuda", dtype=torch.int32).repeat_interleave(room)
    p = torch.arange(room, device="cuda", dtype=torch.int32).repeat(slots)
    cache.write(layer, k, v, p, s)
    ks, vs = cache.read(layer, p, s)
    return cache, ks.view(slots, room, kv, d), vs.view(slots, room, kv, d)


def check_decode(torch, out, q, ks, vs, lengths, slots, label="", norm=2.0 ** -19):
    group = q.shape[1] // ks.shape[2]
    for c, (n, s) in enumerate(zip(lengths, slots)):
        if n == 0:
            assert float(out[c].abs().max()) == 0.0
            continue
        kk, vv = (x[s, :n].permute(1, 0, 2).repeat_interleave(group, 0) for x in (ks, vs))
        seen = torch.ones(1, n, dtype=torch.bool, device="cuda")
        ref, bound = attend(torch, q[c][:, None], kk, vv, seen)
        check_close(out[c][:, None], ref, bound, f"{label} column {c} length {n}", norm)


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("rows", ["normal", "wide", "zero", "tiny", "ties"])
def test_cache_write_is_the_block_format(pkg, cuda, gen, dim, rows):
    """What a row reads back as is what QuantizeToQ40 and DequantizeFromQ40 make
    of it, bit for bit; other rows stay."""
    torch = cuda
    n, kv = 50, 3
    k, v = randn(torch, gen, n, kv, dim), randn(torch, gen, n, kv, dim)
    if rows == "wide":
        k *= torch.exp(8 * randn(torch, gen, n, kv, 1))
    elif rows == "zero":
        k[::2] = 0
        v[:, :, :32] = 0
    elif rows == "tiny":
        k *= 1e-6
        v *= 1e-9
    elif rows == "ties":
        k = (k * 4).round() / 2
        k[..., 0] = 7.0
    cache = pkg.KvCacheQ40(2, 4, 20, kv, dim)
    order = torch.randperm(80, generator=gen, device="cuda")[:n].to(torch.int32)
    slots, pos = order // 20, order % 20
    cache.write(1, k, v, pos, slots)
    got = cache.read(1, pos, slots)
    for x, y in zip((k, v), got):
        want = pkg.DequantizeFromQ40(pkg.QuantizeToQ40(x), tuple(x.shape))
        assert torch.equal(y.view(torch.int32), want.view(torch.int32))
    every = torch.arange(80, device="cuda", dtype=torch.int32)
    all_k, all_v = cache.read(1, every % 20, every // 20)
    other = torch.ones(80, dtype=torch.bool, device="cuda")
    other[order.long()] = False
    assert float(all_k[other].abs().max()) == 0.0 and float(all_v[other].abs().max()) == 0.0
    for x in cache.read(0, every % 20, every // 20):
        assert float(x.abs().max()) == 0.0


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_cache_write_of_many_rows(pkg, cuda, gen, dim):
    """Enough rows that a CTA takes several tokens, their number not a multiple:
    the block format bit for bit, infinities and NaN among the values."""
    torch = cuda
    n, kv = 1501, 3
    k, v = randn(torch, gen, n, kv, dim), randn(torch, gen, n, kv, dim)
    k[5, 1, 3], k[6, 2, 31], v[7, 0, 0] = float("inf"), -float("inf"), float("nan")
    v[8, 1] = float("nan")
    k[9:20] *= 1e6  # scales that overflow fp16
    cache = pkg.KvCacheQ40(1, 3, 501, kv, dim)
    order = torch.randperm(3 * 501, generator=gen, device="cuda")[:n].to(torch.int32)
    slots, pos = order % 3, order // 3
    pos[[0, 700, n - 1]] = -1
    cache.write(0, k, v, pos, slots)
    live = pos >= 0
    for x, y in zip((k, v), cache.read(0, pos, slots)):
        want = pkg.DequantizeFromQ40(pkg.QuantizeToQ40(x), tuple(x.shape))
        same = (y == want) | (y.isnan() & want.isnan())
        assert bool(same[live].all())
        assert float(y[~live].abs().max()) == 0.0


def test_cache_offsets_past_32_bits(pkg, cuda, gen):
    """A cache whose last layer starts more than 2^32 bytes in."""
    torch = cuda
    if torch.cuda.mem_get_info()[0] < 20 * 2 ** 30:
        pytest.skip("needs 10 GB of device memory")
    room, kv, d = 1 << 20, 8, 128
    cache = pkg.KvCacheQ40(4, 2, room, kv, d)
    assert cache.keys.numel() > 2 ** 32
    small = pkg.KvCacheQ40(1, 1, 300, kv, d)
    k, v = randn(torch, gen, 300, kv, d), randn(torch, gen, 300, kv, d)
    p = torch.arange(300, device="cuda", dtype=torch.int32)
    cache.write(3, k, v, p, torch.ones_like(p))
    small.write(0, k, v, p, torch.zeros_like(p))
    q = randn(torch, gen, 1, 16, d)
    n, one = i32(torch, [300]), i32(torch, [1])
    # other cuts of the same work: sums of 300 weighted values in another order
    want = small.attention(q, 0, n, i32(torch, [0]))
    got = cache.attention(q, 3, n, one)
    assert float((got - want).abs().max()) <= 2.0 ** -20 * float(want.abs().max())
    # positions at the end of the room
    last = p + (room - 300)
    cache.write(3, k, v, last, torch.ones_like(p))
    assert all(torch.equal(a, b) for a, b in zip(cache.read(3, last, torch.ones_like(p)),
                                                 small.read(0, p, torch.zeros_like(p))))
    del cache
    torch.cuda.empty_cache()


def test_cache_rows_strides_padding_and_bad_indices(pkg, cuda, gen):
    torch = cuda
    kv, d, n = 2, 64, 9
    for shift in (0, 1):  # rows at any alignment
        flat = randn(torch, gen, n * 300 + shift)
        rows = flat[shift:].view(n, 300)
        k = rows[:, 4:4 + kv * d].view(n, kv, d)
        v = rows[:, 150:150 + kv * d].view(n, kv, d)
        cache = pkg.KvCacheQ40(1, n, 10, kv, d)
        pos = i32(torch, [0, 1, -1, 9, 4, -1, 2, 3, 8])
        cache.write(0, k, v, pos)
        out = torch.full((n, 300), 5.0, device="cuda")
        ko, vo = cache.read(0, pos, k_out=out[:, 8:8 + kv * d].view(n, kv, d),
                            v_out=out[:, 160:160 + kv * d].view(n, kv, d))
        live = pos >= 0
        for x, y in ((k, ko), (v, vo)):
            want = pkg.DequantizeFromQ40(pkg.QuantizeToQ40(x.contiguous()), (n, kv, d))
            assert torch.equal(y[live], want[live]) and bool((y[~live] == 5).all())
        assert bool((out[:, :8] == 5).all() and (out[:, 288:] == 5).all())
    pkg.lib().dqmk_device_error(1)
    before = cache.keys.clone(), cache.values.clone()
    for p, s in ((10, 0), (-2, 0), (2 ** 31 - 1, 0), (0, n), (0, -1)):
        cache.write(0, k[:1], v[:1], i32(torch, [p]), i32(torch, [s]))
        assert pkg.lib().dqmk_device_error(1) == 8
    assert torch.equal(cache.keys, before[0]) and torch.equal(cache.values, before[1])
    # a padding row's slot is not looked at
    cache.write(0, k[:1], v[:1], i32(torch, [-1]), i32(torch, [99]))
    assert pkg.lib().dqmk_device_error(1) == 0


@pytest.mark.parametrize("heads", [(1, 1), (14, 2), (28, 4), (6, 3), (9, 1), (16, 1), (40, 8)],
                         ids=lambda h: "h%d_kv%d" % h)
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_cache_attention(pkg, cuda, gen, heads, dim):
    torch = cuda
    h, kv = heads
    room = 517
    cache, ks, vs = fill(pkg, torch, gen, 3, 4, room, kv, dim, 2)
    lengths = [0, 1, 2, 31, 32, 33, 63, 100, 127, 128, 129, 256, 257, 500, 516, 517]
    slots = [c % 4 for c in range(len(lengths))]
    q = randn(torch, gen, len(lengths), h, dim)
    args = (q, 2, i32(torch, lengths), i32(torch, slots))
    out = cache.attention(*args)
    check_decode(torch, out, q, ks, vs, lengths, slots)
    assert torch.equal(out, cache.attention(*args))
    # one at a time: other cuts of the same work
    for c in (1, 5, 13, 15):
        one = cache.attention(q[c:c + 1], 2, args[2][c:c + 1], args[3][c:c + 1])
        check_decode(torch, one, q[c:c + 1], ks, vs, lengths[c:c + 1], slots[c:c + 1])


@pytest.mark.parametrize("room", [1, 31, 32, 128, 129, 2048])
def test_cache_attention_rooms(pkg, cuda, gen, room):
    """Caches of every size, unwritten bytes NaN, default slots, strided rows."""
    torch = cuda
    h, kv, d, n = 7, 1, 64, 5
    cache, ks, vs = fill(pkg, torch, gen, 1, n, room, kv, d, 0)
    lengths = [room, max(1, room // 2), 0, 1, room]
    rows = randn(torch, gen, n, h + 2, d)
    wide = torch.full((n, h + 1, d), 3.0, device="cuda")
    out = cache.attention(rows[:, 1:1 + h], 0, i32(torch, lengths), out=wide[:, :h])
    check_decode(torch, out, rows[:, 1:1 + h], ks, vs, lengths, range(n))
    assert bool((wide[:, h] == 3).all())


@pytest.mark.parametrize("columns", [128, 129, 300])
def test_cache_attention_many_columns(pkg, cuda, gen, columns):
    """More columns than a CTA has threads, a prompt's tokens one by one among
    them: several columns of a slot with growing lengths."""
    torch = cuda
    h, kv, d, room = 14, 2, 64, 700
    cache, ks, vs = fill(pkg, torch, gen, 1, 5, room, kv, d, 0)
    r = np.random.RandomState(columns)
    lengths = r.randint(0, room + 1, columns)
    lengths[:40] = np.arange(40)
    lengths[-1] = room
    slots = r.randint(0, 5, columns)
    slots[:40] = 2
    q = randn(torch, gen, columns, h, d)
    out = cache.attention(q, 0, i32(torch, lengths.tolist()), i32(torch, slots.tolist()))
    check_decode(torch, out, q, ks, vs, lengths.tolist(), slots.tolist())


def test_cache_attention_not_finite(pkg, cuda, gen):
    """A query with a NaN or an infinity spoils its own head alone."""
    torch = cuda
    cache, ks, vs = fill(pkg, torch, gen, 1, 2, 400, 2, 64, 0)
    q = randn(torch, gen, 2, 14, 64)
    n = i32(torch, [400, 33])
    want = cache.attention(q, 0, n)
    for bad in (float("nan"), float("inf")):
        x = q.clone()
        x[0, 4, 9] = bad
        out = cache.attention(x, 0, n)
        assert not bool(out[0, 4].isfinite().any())
        out[0, 4] = want[0, 4]
        assert torch.equal(out, want)


def test_cache_attention_behind_the_length_is_never_read(pkg, cuda, gen):
    """Bytes behind the length (stale rows, NaN scales) do not change a bit."""
    torch = cuda
    h, kv, d = 14, 2, 64
    a, ks, vs = fill(pkg, torch, gen, 1, 2, 300, kv, d, 0, poison=False)
    b = pkg.KvCacheQ40(1, 2, 300, kv, d)
    b.keys.fill_(255)
    b.values.fill_(255)
    lengths = [70, 199]
    for s, n in enumerate(lengths):
        b.write(0, ks[s, :n], vs[s, :n], torch.arange(n, device="cuda", dtype=torch.int32),
                torch.full((n,), s, device="cuda", dtype=torch.int32))
        p = torch.arange(n, device="cuda", dtype=torch.int32)
        kb, vb = b.read(0, p, torch.full_like(p, s))
        a.write(0, kb, vb, p, torch.full_like(p, s))
        # quantizing quantized values again may move them: both caches hold the same now
        kb, vb = a.read(0, p, torch.full_like(p, s))
        b.write(0, kb, vb, p, torch.full_like(p, s))
        for x, y in zip(a.read(0, p, torch.full_like(p, s)), b.read(0, p, torch.full_like(p, s))):
            if not torch.equal(x, y):
                pytest.skip("values did not settle")
    q = randn(torch, gen, 2, h, d)
    n = i32(torch, lengths)
    assert torch.equal(a.attention(q, 0, n), b.attention(q, 0, n))


def test_cache_attention_out_of_range(pkg, cuda, gen):
    torch = cuda
    cache, ks, vs = fill(pkg, torch, gen, 1, 2, 50, 2, 64, 0)
    q = randn(torch, gen, 4, 4, 64)
    pkg.lib().dqmk_device_error(1)
    for lengths, slots in (([51, 50, 3, 0], [0, 1, 0, 1]), ([-1, 50, 3, 0], [0, 1, 0, 1]),
                           ([5, 50, 3, 0], [2, 1, 0, 1]), ([5, 50, 3, 0], [-1, 1, 0, 1])):
        out = cache.attention(q, 0, i32(torch, lengths), i32(torch, slots))
        assert pkg.lib().dqmk_device_error(1) == 8
        check_decode(torch, out, q, ks, vs, [0] + lengths[1:], [0] + slots[1:])
    assert pkg.lib().dqmk_device_error(1) == 0


def test_cache_attention_weights(pkg, cuda, gen):
    """Equal weights over a long history (the small mean of many values),
    scores of hundreds, a query of zeros or of large and small heads, values
    whose scales differ by 2^20 from position to position."""
    torch = cuda
    h, kv, d, room = 8, 2, 128, 5000
    cache, ks, vs = fill(pkg, torch, gen, 1, 1, room, kv, d, 0)
    n = [room]
    q = torch.zeros(1, h, d, device="cuda")
    out = cache.attention(q, 0, i32(torch, n))
    # a mean of 5000 values is 1/70 of them: its error is that of the sum of sizes
    check_decode(torch, out, q, ks, vs, n, [0], "equal", norm=2.0 ** -15)
    q = randn(torch, gen, 1, h, d) * 40
    check_decode(torch, cache.attention(q, 0, i32(torch, n)), q, ks, vs, n, [0], "sharp",
                 norm=2.0 ** -14)
    q = randn(torch, gen, 1, h, d) * torch.tensor([1.0, 1e-20, 1e-3, 0.5, 1, 2, 0, 1e-30],
                                                  device="cuda")[None, :, None]
    check_decode(torch, cache.attention(q, 0, i32(torch, n)), q, ks, vs, n, [0], "heads",
                 norm=2.0 ** -15)
    e = torch.randint(-10, 11, (room, 1, 1), generator=gen, device="cuda").float()
    p = torch.arange(room, device="cuda", dtype=torch.int32)
    cache.write(0, ks[0], randn(torch, gen, room, kv, d) * torch.exp2(e), p, torch.zeros_like(p))
    ks, vs = (x[None] for x in cache.read(0, p, torch.zeros_like(p)))
    q = randn(torch, gen, 1, h, d)
    check_decode(torch, cache.attention(q, 0, i32(torch, n)), q, ks, vs, n, [0], "scales")


# ------------------------------------------------------------ streams and graphs
def test_attention_block_on_streams_and_in_graphs(pkg, cuda, gen):
    """Another stream than torch's current one, two streams at once, a captured
    and replayed run: the bits of the plain calls."""
    torch = cuda
    h, kv, d, n = 14, 2, 64, 150
    starts = i32(torch, [0, 100, 150])
    q, k, v = randn(torch, gen, n, h, d), randn(torch, gen, n, kv, d), randn(torch, gen, n, kv, d)
    w = torch.ones(d, device="cuda")
    pos = i32(torch, list(range(100)) + list(range(50)))
    slots = i32(torch, [0] * 100 + [1] * 50)
    cache = pkg.KvCacheQ40(1, 2, 160, kv, d)
    qd = randn(torch, gen, 2, h, d)
    lengths = i32(torch, [100, 50])
    torch.cuda.synchronize()

    def block(stream=None):
        qr, kr = pkg.qk_norm_rope(q, k, w, w, pos, 1e6, 1e-6, stream=stream)
        out = pkg.attention_prompt(qr, kr, v, starts, stream=stream)
        cache.write(0, kr, v, pos, slots, stream=stream)
        return out, cache.attention(qd, 0, lengths, stream=stream)

    want = block()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = [block(streams[0]), block(streams[1].cuda_stream)]
        torch.cuda.synchronize()
        for a in got:
            assert all(torch.equal(x, y) for x, y in zip(a, want))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = block()
        graphs.append((g, out))
    for _ in range(3):
        for g, out in graphs:
            for x in out:
                x.zero_()
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(x, y) for x, y in zip(out, want))
    # new inputs in the same memory
    lengths.copy_(i32(torch, [7, 0]))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1][1], cache.attention(qd, 0, lengths))


# ------------------------------------------------------------ together
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128)], ids=lambda h: "h%d_kv%d_d%d" % h)
def test_attention_block_serves_prompts_and_decodes(pkg, cuda, gen, heads):
    """Prompts of three sequences, then tokens one at a time for all of them,
    one of which has ended: every output against the whole computation in 64
    bits from the rows the cache holds."""
    torch = cuda
    h, kv, d = heads
    lens = [5, 130, 40]
    theta, eps = 1e6, 1e-6
    qw, kw = 1 + 0.1 * randn(torch, gen, d), 1 + 0.1 * randn(torch, gen, d)
    starts = np.concatenate([[0], np.cumsum(lens)]).tolist()
    total = starts[-1]
    cache = pkg.KvCacheQ40(2, 3, 200, kv, d)
    rows = randn(torch, gen, total, h + 2 * kv, d)
    q, k, v = rows[:, :h], rows[:, h:h + kv], rows[:, h + kv:]
    slots = i32(torch, sum(([s] * n for s, n in enumerate(lens)), []))
    pos = i32(torch, sum((list(range(n)) for n in lens), []))
    qr, kr = pkg.qk_norm_rope(q, k, qw, kw, pos, theta, eps)
    check_rope(torch, kr, k, kw, pos, theta, eps, True)
    out = pkg.attention_prompt(qr, kr, v, i32(torch, starts))
    check_prompt(torch, out, qr, kr, v, starts)
    cache.write(1, kr, v, pos, slots)
    for step in range(3):
        rows = randn(torch, gen, 3, h + 2 * kv, d)
        q, k, v = rows[:, :h], rows[:, h:h + kv], rows[:, h + kv:]
        at = [n + step for n in lens]
        at[0] = -1  # the first sequence has ended
        qr, kr = pkg.qk_norm_rope(q, k, qw, kw, i32(torch, at), theta, eps)
        cache.write(1, kr, v, i32(torch, at))
        seen = [p + 1 for p in at]
        out = cache.attention(qr, 1, i32(torch, seen))
        every = torch.arange(600, device="cuda", dtype=torch.int32)
        ks, vs = (x.view(3, 200, kv, d) for x in cache.read(1, every % 200, every // 200))
        check_decode(torch, out, qr, ks, vs, seen, range(3), f"step {step}")
    assert pkg.lib().dqmk_device_error(1) == 0


@pytest.mark.parametrize("columns", [1, 70])
def test_cache_attention_in_place(pkg, cuda, gen, columns):
    """Output over the queries: groups of one CTA and of several, zero rows."""
    torch = cuda
    h, kv, d, room = 20, 2, 64, 3000
    cache, _, _ = fill(pkg, torch, gen, 1, 3, room, kv, d, 0)
    lengths = [room] if columns == 1 else [(c * 677) % (room + 1) for c in range(columns)]
    q = randn(torch, gen, columns, h, d)
    args = (0, i32(torch, lengths), i32(torch, [c % 3 for c in range(columns)]))
    want = cache.attention(q, *args)
    assert cache.attention(q, *args, out=q) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("heads", [(14, 2, 64), (12, 3, 36), (40, 8, 32)], ids=lambda h: "h%d_kv%d_d%d" % h)
def test_attention_prompt_full_machine(pkg, cuda, gen, heads):
    """More items than the SMs take at once, several key tiles each, a sequence
    whose rows differ by 2^20 and, in another, sizes of 2^20 throughout; twice."""
    torch = cuda
    h, kv, d = heads
    lengths = [600] * 8 + [1, 0, 130, 64, 65] * 60
    starts = np.concatenate([[0], np.cumsum(lengths)]).tolist()
    n = starts[-1]
    q, k, v = (randn(torch, gen, n, x, d) for x in (h, kv, kv))
    v[:600] *= torch.exp2(torch.randint(-10, 11, (600, 1, 1), generator=gen, device="cuda").float())
    v[600:1200] *= 2.0 ** 20
    out = pkg.attention_prompt(q, k, v, i32(torch, starts))
    for a, b in zip(starts[:40], starts[1:41]):
        check_prompt(torch, out[a:b], q[a:b], k[a:b], v[a:b], [0, b - a], f"from {a}")
    check_prompt(torch, out[starts[-6]:], *(x[starts[-6]:] for x in (q, k, v)),
                 [s - starts[-6] for s in starts[-6:]])
    assert torch.equal(out, pkg.attention_prompt(q, k, v, i32(torch, starts)))
