"""Page bounds of sequences that end at their own lengths, and what depends on them: bounds exactly,
selection and attention after a compaction as before it."""
import numpy as np
import pytest

from kv_reads import PAGE, Cache, page_bounds, queries

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def reef():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import reef_amd
    reef_amd.lib()
    return reef_amd


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D,T,starts,lens", [
    (128, 160, [0, 0, 0, 0, 0], [100, 1, 160, 0, 64]),   # every page that holds tokens
    (64, 160, [0, 0, 0, 0, 0], [159, 16, 17, 33, 15]),
    (64, 20, [90, 17, 139, 0, 60], [100, 30, 160, 0, 60]),  # ends before, at and behind a range
    (128, 1, [99, 31, 144, 5, 63], [100, 32, 160, 3, 64]),  # (a length before the start: nothing)
])
def test_bounds_up_to_each_length(reef, paged, bits, D, T, starts, lens):
    """Behind a length lie codes of the largest size, scales that are no numbers and, in a table, no
    pages."""
    rng = np.random.default_rng(T + D + bits)
    B, H, L = 5, 2, 160
    cache = Cache(rng, bits, B, H, D, L, lens, paged)
    lead = (cache.tensors[0].shape[0], H) if paged else (B, H, L // PAGE)
    bounds = torch.from_numpy(rng.integers(-127, 128, (*lead, 2, D)).astype(np.int8)).cuda()
    scales = torch.rand(lead, device="cuda")
    want, want_s = bounds.cpu().numpy(), scales.cpu().numpy()
    table = None
    if paged:
        empty = np.arange(L // PAGE) * PAGE >= np.asarray(lens)[:, None]
        table = ints(np.where(empty, -1, cache.table))
    reef.kv_page_bounds(ints(starts), T, cache.tensors[0], cache.tensors[2], bounds, scales,
                        block_table=table, context_lens=ints(lens))
    for b in range(B):
        end = min(starts[b] + T, lens[b])
        if end <= starts[b]:
            continue
        for p in range(starts[b] // PAGE, (end - 1) // PAGE + 1):
            live = slice(p * PAGE, min(p * PAGE + PAGE, end))
            for h in range(H):
                x = cache.k[b, h, live].astype(np.float32) * cache.ks[b, h, live, None]
                at = (cache.table[b, p], h) if paged else (b, h, p)
                want[at], want_s[at] = page_bounds(x)
    assert np.array_equal(scales.cpu().numpy(), want_s)
    assert np.array_equal(bounds.cpu().numpy(), want)


def test_lengths_outside_the_cache(reef):
    k = torch.ones(3, 1, 32, 64, dtype=torch.int8, device="cuda")
    ks = torch.ones(3, 1, 32, device="cuda")
    for lens in ([-1, 32, 7], [33, 32, 7]):
        bounds = torch.full((3, 1, 2, 2, 64), 5, dtype=torch.int8, device="cuda")
        scales = torch.full((3, 1, 2), 9.0, device="cuda")
        with pytest.raises(reef.InvalidArgument):
            reef.kv_page_bounds(ints([0, 0, 0]), 32, k, ks, bounds, scales, context_lens=ints(lens))
        one = float(np.float32(1) / np.float32(127))
        assert scales.tolist() == [[[9, 9]], [[one, one]], [[one, 9]]]
        assert (bounds[0] == 5).all() and (bounds[2, 0, 1] == 5).all() and (bounds[1] == 127).all()
    with pytest.raises(reef.InvalidArgument):
        reef.kv_page_bounds(ints([0, 0, 0]), 32, k, ks, bounds, scales, context_lens=ints([1, 2]))
    with pytest.raises(reef.CapacityError):
        reef.kv_page_bounds(ints([0, 1, 0]), 32, k, ks, bounds, scales, context_lens=ints([1, 2, 3]))


@pytest.mark.parametrize("bits", [4, 8])
def test_selection_after_a_compaction(reef, bits):
    """Sequences of unequal lengths whose pages move into the places of freed ones: the lists and the
    attention are those of before, bit for bit."""
    rng = np.random.default_rng(40 + bits)
    B, H, G, D, L = 6, 2, 4, 128, 640
    lens = [640, 333, 17, 500, 161, 609]
    cache = Cache(rng, bits, B, H, D, L, lens, True, key_drift=0.3)
    pages = cache.tensors[0].shape[0]
    empty = np.arange(L // PAGE) * PAGE >= np.asarray(lens)[:, None]
    rows = np.where(empty, -1, cache.table)
    refs = np.zeros(pages, np.int32)
    refs[rows[rows >= 0]] = 1
    table, lengths, refs = ints(rows), ints(lens), torch.from_numpy(refs).cuda()
    bounds = torch.zeros((pages, H, 2, D), dtype=torch.int8, device="cuda")
    scales = torch.zeros((pages, H), device="cuda")
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")

    def measure():
        reef.kv_page_bounds(zero, L, cache.tensors[0], cache.tensors[2], bounds, scales,
                            block_table=table, context_lens=lengths)

    q, qs = (torch.from_numpy(a).cuda() for a in queries(rng, B, H * G, D))
    left = torch.tensor([1, 3, 4, 5], device="cuda")
    decode = reef.attention_decode_int4 if bits == 4 else reef.attention_decode_selected

    def step():
        where = dict(block_table=table[left].contiguous())
        chosen = reef.kv_select_pages(q[left], qs[left], bounds, scales, lengths[left], 6, sinks=1,
                                      recent=2, **where)
        return [*chosen, decode(q[left], qs[left], *cache.tensors, lengths[left], selected=chosen, **where)]

    measure()
    want = step()
    reef.kv_free(ints([0, 2]), table, lengths, refs)
    source, place, live = reef.kv_compact(table, refs)
    copy = reef.kv_copy_pages_int4 if bits == 4 else reef.kv_copy_pages
    copy(source, place, *cache.tensors)
    assert int((source >= 0).sum()) > 10 and int(live) == int((~empty[[1, 3, 4, 5]]).sum())
    stale = step()
    assert not torch.equal(stale[0], want[0])  # (the bounds did not move)
    measure()
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
