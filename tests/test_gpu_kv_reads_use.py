"""The 4-bit cache and the page selection as a server calls them: captured chunks beside eager
ones, graphs replayed at the same time, pools and caches whose offsets pass 31 bits, windows that
leave a list nothing."""
import numpy as np
import pytest

from kv_reads import PAGE, Cache, attention, queries

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
    return torch.tensor(list(x), dtype=torch.int32).cuda()


def captured(call):
    """(graph, what the call returned while it was recorded)."""
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            held = call()
    torch.cuda.current_stream().wait_stream(stream)
    return graph, held


@pytest.mark.parametrize("T,n", [(5, 900), (128, 4100)])
def test_captured_chunk(reef, T, n):
    """As columns of the decode kernel, and through the copy of the cache."""
    rng = np.random.default_rng(T)
    cache = Cache(rng, 4, 2, 2, 128, -(-n // PAGE) * PAGE, [n] * 2, True)
    G = 4 if T == 5 else 8
    word = reef.StatusWord("cuda")
    q = torch.empty((2, 2 * G, T, 128), dtype=torch.int8, device="cuda")
    qs = torch.rand(2 * G, device="cuda") * 0.01 + 0.01

    def call():
        return reef.attention_prefill_cache_int4(q, qs, *cache.tensors, n, status=word,
                                                 block_table=cache.block_table)

    q.zero_()
    graph, held = captured(call)
    for _ in range(4):
        q.copy_(torch.randint(-127, 128, q.shape, device="cuda", dtype=torch.int8))
        want = call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want)
    word.check("chunk")


def test_graphs_at_the_same_time(reef):
    """Recorded on one stream, replayed on two: each has its workspace."""
    rng = np.random.default_rng(5)
    word = reef.StatusWord("cuda")
    jobs = []
    for i in range(2):
        lens = [4000, 1700]
        cache = Cache(rng, 4, 2, 2, 128, 4096, lens, True)
        q, qs = (torch.from_numpy(a).cuda() for a in queries(rng, 2, 8, 128))
        rows = torch.from_numpy(rng.integers(-127, 128, (2, 8, 4, 128)).astype(np.int8)).cuda()

        def call(cache=cache, q=q, qs=qs, rows=rows):
            return (reef.attention_decode_int4(q, qs, *cache.tensors, cache.context_lens, status=word,
                                               block_table=cache.block_table),
                    reef.attention_prefill_cache_int4(rows, qs[0], *cache.tensors, 1700, status=word,
                                                      block_table=cache.block_table))

        want = [t.clone() for t in call()]
        jobs.append((*captured(call), want, call))  # (call: a graph's inputs have to live)
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(10):
        for (graph, *_), s in zip(jobs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, held, want, _ in jobs:
            assert all(torch.equal(a, b) for a, b in zip(held, want))
    word.check("graphs")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("paged", [False, True])
def test_offsets_past_31_bits(reef, bits, paged):
    """Caches, and their bounds, of more than 2^31 bytes hold what small ones hold at the same
    places of a sequence: the same results, bit for bit."""
    B, H, G, D, T, budget = 2, 64, 2, 128, 77, 3
    code = torch.uint8 if bits == 4 else torch.int8
    word = reef.StatusWord("cuda")
    x = torch.randn(B, H, T, D, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randint(-127, 128, (B, H * G, D), generator=g, device="cuda", dtype=torch.int8)
    rows = torch.randint(-127, 128, (B, H * G, 3, D), generator=g, device="cuda", dtype=torch.int8)
    qs = torch.rand((B, H * G), generator=g, device="cuda") * 0.01 + 0.01
    start, lens = ints([0, 0]), ints([T, T])

    def run(blocks, pages):
        """blocks: of a sequence; pages: the pool's (0: contiguous)."""
        lead = (pages, H) if pages else (B, H, blocks)
        cache = [torch.empty((*lead, PAGE, D * bits // 8), dtype=code, device="cuda"),
                 torch.empty((*lead, D, 2 * bits), dtype=code, device="cuda"),
                 torch.empty((*lead, PAGE), device="cuda"), torch.empty((*lead, PAGE), device="cuda")]
        bounds = torch.empty((*lead, 2, D), dtype=torch.int8, device="cuda")
        scales = torch.empty(lead, device="cuda")
        table = None
        if pages:
            table = torch.arange(pages - 1, pages - 1 - B * blocks, -1, device="cuda",
                                 dtype=torch.int32).reshape(B, blocks)
        else:
            cache = [cache[0].view(B, H, blocks * PAGE, D * bits // 8), cache[1],
                     *(t.view(B, H, blocks * PAGE) for t in cache[2:])]
        if bits == 4:
            reef.kv_append_int4(x, x, start, *cache, block_table=table, status=word)
        elif pages:
            reef.kv_append_paged(x, x, start, table, *cache, status=word)
        else:
            reef.kv_append(x, x, start, *cache, status=word)
        reef.kv_page_bounds(start, T, cache[0], cache[2], bounds, scales, block_table=table, status=word)
        chosen = reef.kv_select_pages(q, qs, bounds, scales, lens, budget, block_table=table, status=word)
        results = [*chosen]
        if bits == 4:
            for selected in (None, chosen):
                results.append(reef.attention_decode_int4(q, qs, *cache, lens, selected=selected,
                                                          block_table=table, status=word))
            results.append(reef.attention_prefill_cache_int4(rows, qs[0], *cache, T, block_table=table,
                                                             status=word))
        else:
            results.append(reef.attention_decode_selected(q, qs, *cache, lens, selected=chosen,
                                                          block_table=table, status=word))
        torch.cuda.synchronize()
        word.check("calls")
        return results

    blocks = -(-T // PAGE)
    small = run(blocks, 2 * B * blocks if paged else 0)
    # the last sequence's or page's heads lie past 2^31 bytes of keys, values and bounds
    large = run(blocks, 140_000) if paged else run(140_000, 0)
    assert 140_000 * H * 2 * D > 1 << 31 and 140_000 * H * PAGE * D * bits // 8 > 1 << 31
    for a, b in zip(small, large):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [4, 8])
def test_window_that_leaves_a_list_nothing(reef, bits):
    rng = np.random.default_rng(bits)
    cache = Cache(rng, bits, 2, 1, 64, 640, [640, 630], True)
    q, qs = queries(rng, 2, 4, 64)
    listed = torch.tensor([[[0, 3, 20]], [[1, 39, 5]]], dtype=torch.int32).cuda()
    call = reef.attention_decode_int4 if bits == 4 else reef.attention_decode_selected
    got = call(torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda(), *cache.tensors,
               cache.context_lens, selected=(listed, torch.full((2, 1), 3, dtype=torch.int32).cuda()),
               block_table=cache.block_table, window=10)
    want, tol = attention(cache, q, qs, lambda b, h: range(624, 630) if b else [])
    assert np.abs(got.double().cpu().numpy() - want).max() <= tol
    assert not got[0].any()


@pytest.mark.parametrize("B,H,splits", [(40, 8, 9), (33, 8, 4), (33, 8, 1), (70, 1, 30), (300, 8, 7)])
def test_asked_for_splits_of_many_sequences(reef, B, H, splits):
    """num_splits with more items than a wave's plan holds, and than a workgroup's."""
    rng = np.random.default_rng(B + splits)
    lens = [int(n) for n in rng.integers(1, 641, B)]
    cache = Cache(rng, 4, B, H, 64, 640, lens, True)
    q, qs = queries(rng, B, H, 64)
    want, tol = attention(cache, q, qs, lambda b, h: range(lens[b]))
    tq, tqs = torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda()
    for _ in range(2):
        got = reef.attention_decode_int4(tq, tqs, *cache.tensors, cache.context_lens,
                                         block_table=cache.block_table, num_splits=splits)
        assert np.abs(got.double().cpu().numpy() - want).max() <= tol
    listed = torch.arange(39, -1, -1, dtype=torch.int32).cuda().expand(B, H, 40).contiguous()
    counts = torch.full((B, H), 40, dtype=torch.int32)
    for b in range(B):
        counts[b] = -(-lens[b] // PAGE)
    # (a list in descending order holds the pages at its end: the rest is left out by a negative entry)
    listed = torch.where(listed < counts.cuda()[..., None], listed, -1).contiguous()
    got = reef.attention_decode_int4(tq, tqs, *cache.tensors, cache.context_lens, num_splits=splits,
                                     selected=(listed, torch.full((B, H), 40, dtype=torch.int32).cuda()),
                                     block_table=cache.block_table)
    assert np.abs(got.double().cpu().numpy() - want).max() <= tol
