"""GPU: the attention kernels' bounded waits.  A test hook withholds the copies
of one tile, so that the waits for it run out: the kernels must record it and
exit, read nothing but their own results from a workspace that holds anything,
and leave the context usable.  Nothing here faults, traps or hangs the GPU."""
import ctypes as C
import time

import pytest

pytestmark = pytest.mark.gpu


def withheld(pkg, torch, cache, q, lengths, column, tile, fill):
    """(out, seconds) of a call whose copies of one tile never come; out starts as 7."""
    L = pkg.lib()
    n, h, d = q.shape
    out = torch.full_like(q, 7.0)
    size = L.dqmk_kv_q40_attention_workspace(cache._ref, n, h)
    work = torch.full((size // 4,), fill, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    t0 = time.time()
    pkg.check(L.dqmk_kv_q40_attention_withhold_tile(
        cache._ref, 0, q.data_ptr(), h * d, None, lengths.data_ptr(), n, h, out.data_ptr(), h * d,
        work.data_ptr(), size, column, tile, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    return out, time.time() - t0


# column 1 over all CTAs, its first tile or one in the middle; many short columns, several to a CTA
CASES = [([100, 30000, 90], 1, 0), ([100, 30000, 90], 1, 500), ([100, 30000, 90], 1, 937),
         ([100 + c % 60 for c in range(900)], 450, 1)]


@pytest.mark.parametrize("lengths,column,tile", CASES, ids=["start", "middle", "end", "short"])
@pytest.mark.parametrize("fill", [0x7f7f7f7f, -3, 1], ids=["large", "negative", "small"])
def test_cache_attention_wait_runs_out(pkg, cuda, lengths, column, tile, fill):
    torch = cuda
    L = pkg.lib()
    h, kv, d = 14, 2, 64
    n, room = len(lengths), max(lengths)
    g = torch.Generator(device="cuda").manual_seed(5)
    cache = pkg.KvCacheQ40(1, n, room, kv, d)
    for s, length in enumerate(lengths):
        k, v = (torch.randn(length, kv, d, generator=g, device="cuda") for _ in "kv")
        p = torch.arange(length, device="cuda", dtype=torch.int32)
        cache.write(0, k, v, p, torch.full_like(p, s))
    q = torch.randn(n, h, d, generator=g, device="cuda")
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = cache.attention(q, 0, lens)
    assert L.dqmk_device_error(1) == 0
    out, seconds = withheld(pkg, torch, cache, q, lens, column, tile, fill)
    assert seconds < 30
    assert L.dqmk_device_error(1) == 1  # recorded, and cleared by the read
    # every row of a head is what it would be, or was left, or is NaN
    same = (out == want).all(-1)
    kept = (out == 7.0).all(-1)
    lost = out.isnan().all(-1)
    assert bool((same | kept | lost).all())
    assert not bool(same[column].any())
    # a CTA that stopped holds few groups: the others' rows are all there
    assert int(same.sum()) >= n * h - (h if n == 3 else 60 * h)
    assert torch.equal(cache.attention(q, 0, lens), want)
    assert L.dqmk_device_error(0) == 0


# one item a CTA; many items a CTA, two CTAs an SM; many items of the 128-wide build
PROMPTS = [((14, 2, 64), [600, 300, 64, 5], 12, 0), ((8, 8, 64), [64] * 400, 5, 3),
           ((28, 4, 128), [200] * 40, 4 * 7 + 2, 3)]


@pytest.mark.parametrize("heads,lengths,tile,ahead", PROMPTS, ids=["one", "many", "wide"])
@pytest.mark.parametrize("fill", [0x7f7f7f7f, -3])
def test_attention_prompt_wait_runs_out(pkg, cuda, heads, lengths, tile, ahead, fill):
    torch = cuda
    L = pkg.lib()
    h, kv, d = heads
    g = torch.Generator(device="cuda").manual_seed(6)
    starts = [0]
    for x in lengths:
        starts.append(starts[-1] + x)
    n = starts[-1]
    q, k, v = (torch.randn(n, x, d, generator=g, device="cuda") for x in (h, kv, kv))
    st = torch.tensor(starts, dtype=torch.int32, device="cuda")
    want = pkg.attention_prompt(q, k, v, st)
    assert L.dqmk_device_error(1) == 0
    out = torch.full_like(q, 7.0)
    size = L.dqmk_attention_prompt_workspace(n, len(lengths), h, kv, d)
    work = torch.full((size // 4,), fill, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    t0 = time.time()
    pkg.check(L.dqmk_attention_prompt_withhold_tile(
        q.data_ptr(), h * d, k.data_ptr(), kv * d, v.data_ptr(), kv * d, st.data_ptr(), len(lengths), n,
        h, kv, d, out.data_ptr(), h * d, work.data_ptr(), size, tile,
        torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert time.time() - t0 < 30
    assert L.dqmk_device_error(1) == 1
    same, kept = (out == want).all(-1), (out == 7.0).all(-1)
    assert bool((same | kept).all())
    # tokens of the withheld tile, and those behind it in its sequence
    s, first = 0, tile
    while first >= -(-lengths[s] // 64):
        first -= -(-lengths[s] // 64)
        s += 1
    assert bool(kept[starts[s] + 64 * first:starts[s + 1]].all())
    # a CTA that stops loses its item and those that it had taken ahead
    items = kv * (-(-lengths[s] * (h // kv) // 128))
    assert int(kept.sum()) <= items * (1 + ahead) * 128
    if not ahead:
        assert bool(same[:starts[s]].all() and same[starts[s + 1]:].all())
        assert bool(same[starts[s]:starts[s] + 64 * first - 128 * kv // h - 1].all())
    assert torch.equal(pkg.attention_prompt(q, k, v, st), want)
    assert L.dqmk_device_error(0) == 0
