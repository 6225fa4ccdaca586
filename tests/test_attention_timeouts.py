"""CPU: how the decode attention over the 4-bit cache cuts its work, restated:
the runs of the CTAs, and the span (first and last CTA) of each group whose
partial sums the join kernel reads.  Every CTA of a span must hold chunks of the
group, and none outside it may, or a partial sum would be missed or one that was
never written be read."""
import ctypes as C

import numpy as np
import pytest

CHUNK, EXTRA, GRID = 128, 1, 444


def held(chunks, grid):
    """For groups of these chunks: [(cta, group, first chunk, chunks taken)] and the spans."""
    first = np.concatenate([[0], np.cumsum([c + EXTRA for c in chunks])])
    total = int(first[-1])
    n = min(grid, total)
    pieces = []
    for cta in range(n):
        u, u1 = cta * total // n, (cta + 1) * total // n
        while u < u1:
            g = int(np.searchsorted(first, u, side="right")) - 1
            r = u - int(first[g])
            take = min(chunks[g] + EXTRA - r, u1 - u)
            lo, hi = max(r - EXTRA, 0), max(r + take - EXTRA, 0)
            if hi > lo:
                pieces.append((cta, g, lo, hi - lo))
            u += take
    spans = {g: (cta, ((int(first[g]) + EXTRA + chunks[g] - 1 + 1) * n - 1) // total)
             for cta, g, lo, _ in pieces if lo == 0}
    return pieces, spans, n


@pytest.mark.parametrize("grid", [1, 7, GRID])
@pytest.mark.parametrize("seed", range(6))
def test_spans_name_the_ctas_that_hold_a_group(grid, seed):
    r = np.random.RandomState(seed)
    lengths = r.randint(1, (200, 5000, 60000)[seed % 3], r.randint(1, 60))
    chunks = [int(-(-n // CHUNK)) for n in lengths]
    pieces, spans, n = held(chunks, grid)
    for g, count in enumerate(chunks):
        mine = [(cta, lo, take) for cta, gg, lo, take in pieces if gg == g]
        assert sum(take for _, _, take in mine) == count
        x, y = spans[g]
        assert 0 <= x <= y < n
        assert [cta for cta, _, _ in mine] == list(range(x, y + 1))
        # the slot of a CTA's partial sum: 1 where the group starts, 0 behind
        assert [lo == 0 for _, lo, _ in mine] == [cta == x for cta, _, _ in mine]


def test_rows_past_32_bits_are_refused(pkg):
    """Rows whose heads or elements are counted past 31 bits."""
    from importlib import import_module
    L, p = pkg.lib(), C.c_void_p(64)
    big = 1 << 30
    with pytest.raises(RuntimeError, match="QkNormRope: too many heads"):
        pkg.check(L.dqmk_qk_norm_rope(p, 2 * big, p, 2 * big, 1, big, big, 2, p, p, 1e-6, p, 1e6, 1, p,
                                      2 * big, p, 2 * big, None))
    kv = import_module(pkg.__name__ + "._lib").KvQ40(64, 128, 1, 1, 40, 1, 128)
    with pytest.raises(RuntimeError, match="KvQ40Attention: too many heads"):
        pkg.check(L.dqmk_kv_q40_attention(C.byref(kv), 0, p, 1 << 31, p, p, 1, 1 << 24, p, 1 << 31, p,
                                          1 << 40, None))


def test_withheld_copies_refusals(pkg):
    from importlib import import_module
    kv = import_module(pkg.__name__ + "._lib").KvQ40(64, 128, 2, 3, 40, 2, 64)
    p = C.c_void_p(64)
    call = pkg.lib().dqmk_kv_q40_attention_withhold_tile
    for layer, heads, text in ((2, 4, "layer out of range"), (1, 3, "invalid head configuration")):
        with pytest.raises(RuntimeError if heads == 3 else pkg.OutOfRange, match=text):
            pkg.check(call(C.byref(kv), layer, p, 256, p, p, 5, heads, p, 256, p, 1 << 30, 0, 0, None))
    prompt = pkg.lib().dqmk_attention_prompt_withhold_tile
    with pytest.raises(RuntimeError, match="AttentionPrompt: invalid head configuration"):
        pkg.check(prompt(p, 256, p, 128, p, 128, p, 2, 10, 5, 2, 64, p, 256, p, 1 << 30, 0, None))
