"""Bounds of pages, the pages that a query selects and decode over them: bounds, scores' order and
lists exactly, attention against the formula in 64 bits (kv_reads.attention's tolerance)."""
import math

import numpy as np
import pytest

from kv_reads import PAGE, Cache, attention, page_bounds, queries

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


# --- bounds ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("B,H,D,T,starts", [
    (1, 1, 64, 1, [0]), (3, 2, 128, 1, [0, 15, 47]), (2, 3, 64, 7, [12, 3]),
    (2, 1, 128, 16, [16, 8]), (2, 2, 64, 33, [0, 31]), (1, 2, 128, 144, [0]),
])
def test_bounds(reef, paged, bits, B, H, D, T, starts):
    rng = np.random.default_rng(T + D + bits)
    lens = [s + T for s in starts]
    cache = Cache(rng, bits, B, H, D, 144, lens, paged)
    blocks = 144 // PAGE
    lead = (cache.tensors[0].shape[0], H) if paged else (B, H, blocks)
    bounds = torch.from_numpy(rng.integers(-127, 128, (*lead, 2, D)).astype(np.int8)).cuda()
    scales = torch.rand(lead, device="cuda")
    want, want_s = bounds.cpu().numpy(), scales.cpu().numpy()
    reef.kv_page_bounds(ints(starts), T, cache.tensors[0], cache.tensors[2], bounds, scales,
                        block_table=cache.block_table)
    for b in range(B):
        for p in range(starts[b] // PAGE, (lens[b] - 1) // PAGE + 1):
            live = slice(p * PAGE, min(p * PAGE + PAGE, lens[b]))
            for h in range(H):
                x = cache.k[b, h, live].astype(np.float32) * cache.ks[b, h, live, None]
                at = (cache.table[b, p], h) if paged else (b, h, p)
                want[at], want_s[at] = page_bounds(x)
    assert np.array_equal(scales.cpu().numpy(), want_s)
    assert np.array_equal(bounds.cpu().numpy(), want)


def test_bounds_of_zeros_and_refusals(reef):
    k = torch.zeros(2, 1, 32, 64, dtype=torch.int8, device="cuda")
    ks = torch.ones(2, 1, 32, device="cuda")
    bounds = torch.full((2, 1, 2, 2, 64), 5, dtype=torch.int8, device="cuda")
    scales = torch.zeros(2, 1, 2, device="cuda")
    reef.kv_page_bounds(ints([0, 20]), 3, k, ks, bounds, scales)
    assert scales.tolist() == [[[1, 0]], [[0, 1]]]
    assert (bounds[0, 0, 0] == 0).all() and (bounds[0, 0, 1] == 5).all()
    for starts, error in (([-1, 0], reef.InvalidArgument), ([0, 30], reef.CapacityError)):
        with pytest.raises(error):
            reef.kv_page_bounds(ints(starts), 3, k, ks, bounds, scales)
    with pytest.raises(reef.InvalidArgument):  # a page that is not there
        reef.kv_page_bounds(ints([0]), 3, k[:, :, :16], ks[:, :, :16].contiguous(),
                            bounds[:, :, 0].contiguous(), scales[:, :, 0].contiguous(),
                            block_table=ints([[2]]))


# --- selection ------------------------------------------------------------------------------------

def chosen(q, qs, bounds, scales, n, budget, sinks, recent, dead=()):
    """The pages of one (sequence, kv head): codes q [G, D], bounds [n, 2, D]; products in
    whole numbers, the scores' two roundings in float32."""
    q = q.astype(np.int64)
    high, low = bounds[:n, 0].astype(np.int64), bounds[:n, 1].astype(np.int64)
    total = np.maximum(q, 0) @ high.T + np.minimum(q, 0) @ low.T
    score = (total.astype(np.float32) * (qs[:, None] * scales[None, :n])).max(0).astype(np.float64)
    score[:sinks] = np.inf
    score[max(0, n - recent):] = np.inf
    order = [p for p in np.argsort(-score, kind="stable") if p not in dead]
    return sorted(order[:budget])


def selection(rng, B, H, G, D, N, paged, coarse=False):
    """Random bounds of N pages a sequence, in their layout, and queries."""
    bounds = np.sort(rng.integers(-127, 128, (B, H, N, 2, D)), axis=3)[:, :, :, ::-1].astype(np.int8)
    scales = rng.uniform(0.1, 1.0, (B, H, N)).astype(np.float32)
    if coarse:  # few different pages: many ties
        kinds = rng.integers(0, 3, (B, H, N))
        bounds = np.take_along_axis(bounds, kinds[..., None, None], 2)
        scales[:] = 0.25
    q, qs = queries(rng, B, H * G, D)
    tb, ts, table = bounds, scales, None
    if paged:
        P = B * N + 2
        rows = rng.permutation(P)[:B * N].reshape(B, N).astype(np.int32)
        tb, ts = np.zeros((P, H, 2, D), np.int8), np.ones((P, H), np.float32)
        tb[rows], ts[rows] = np.swapaxes(bounds, 1, 2), np.swapaxes(scales, 1, 2)
        table = torch.from_numpy(rows).cuda()
    on_gpu = [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (q, qs, tb, ts)]
    return q, qs, bounds, scales, on_gpu, table


def compare(got, q, qs, bounds, scales, lens, budget, sinks, recent, dead={}):
    pages, counts = (x.cpu().numpy() for x in got)
    B, H = counts.shape
    G = q.shape[1] // H
    for b in range(B):
        n = -(-lens[b] // PAGE)
        for h in range(H):
            g = slice(h * G, h * G + G)
            want = chosen(q[b, g], qs[b, g], bounds[b, h], scales[b, h], n, budget, sinks, recent,
                          dead.get(b, ()))
            assert counts[b, h] == len(want)
            assert pages[b, h].tolist() == want + [-1] * (budget - len(want)), (b, h)


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("B,H,G,D,N,lens,budget,sinks,recent,coarse", [
    (1, 1, 1, 64, 1, [1], 1, 0, 1, False), (2, 2, 4, 128, 40, [640, 333], 8, 1, 2, False),
    (3, 1, 16, 64, 70, [1, 1120, 900], 13, 0, 1, False), (1, 2, 7, 128, 300, [4800], 64, 4, 4, False),
    (2, 3, 2, 128, 257, [4112, 4100], 100, 2, 3, True), (1, 1, 8, 64, 1500, [23999], 500, 0, 1, True),
    (2, 1, 4, 128, 20, [320, 100], 64, 1, 1, False), (1, 1, 1, 128, 1025, [16400], 1, 0, 1, False),
    (1, 8, 4, 128, 8192, [131071], 256, 4, 16, False), (1, 1, 1, 64, 20001, [320016], 37, 1, 2, False),
    (1, 1, 2, 64, 33000, [528000], 4000, 1, 2, True), (2, 2, 1, 64, 64, [1024, 512], 9, 4, 5, False),
])
def test_select(reef, paged, B, H, G, D, N, lens, budget, sinks, recent, coarse):
    rng = np.random.default_rng(N + budget + paged)
    q, qs, bounds, scales, gpu, table = selection(rng, B, H, G, D, N, paged, coarse)
    for _ in range(2):
        got = reef.kv_select_pages(*gpu, ints(lens), budget, block_table=table, sinks=sinks,
                                   recent=recent)
        compare(got, q, qs, bounds, scales, lens, budget, sinks, recent)


def test_select_scale_forms_and_extreme_codes(reef):
    rng = np.random.default_rng(2)
    q, qs, bounds, scales, gpu, _ = selection(rng, 1, 2, 3, 64, 50, False)
    q[0, 0], q[0, 1] = -128, 127
    q[0, 2] = 0                        # scores of zero, of either sign
    gpu[0] = torch.from_numpy(q).cuda()
    for form, s in ((reef.PER_TENSOR, np.float32([0.01])),
                    (reef.PER_HEAD, rng.uniform(0.005, 0.02, 6).astype(np.float32))):
        got = reef.kv_select_pages(gpu[0], torch.from_numpy(s).cuda(), *gpu[2:], ints([790]), 11,
                                   q_granularity=form)
        compare(got, q, np.broadcast_to(s, (1, 6)), bounds, scales, [790], 11, 0, 1)


def test_select_bad_pages_and_lengths(reef):
    rng = np.random.default_rng(4)
    q, qs, bounds, scales, gpu, table = selection(rng, 3, 2, 2, 128, 30, True)
    table[0, 0], table[0, 29], table[2, 7] = -1, 1 << 20, 92
    status = reef.StatusWord("cuda")
    for budget in (6, 29, 64):
        got = reef.kv_select_pages(*gpu, ints([480, 0, 480]), budget, block_table=table, sinks=1,
                                   recent=2, status=status)
        with pytest.raises(reef.InvalidArgument):
            status.check("select")
        dead = {0: (0, 29), 1: range(30), 2: (7,)}
        compare(got, q, qs, bounds, scales, [480, 0, 480], budget, 1, 2, dead)


# --- decode over selected pages --------------------------------------------------------------------

SPARSE = [  # B, kv heads, group, D, L, lens
    (1, 1, 1, 64, 16, [1]), (2, 2, 4, 128, 160, [160, 77]), (1, 1, 16, 128, 640, [639]),
    (3, 2, 2, 64, 320, [320, 1, 161]), (2, 4, 8, 128, 4096, [4090, 300]),
]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("B,H,G,D,L,lens", SPARSE)
def test_decode_listed(reef, bits, paged, B, H, G, D, L, lens):
    """Any list: unordered, with gaps, pages twice, empty."""
    rng = np.random.default_rng(L + bits + paged)
    cache = Cache(rng, bits, B, H, D, L, lens, paged)
    q, qs = queries(rng, B, H * G, D)
    most = 3 * (L // PAGE)
    listed = np.full((B, H, most), 1 << 20, np.int32)  # behind the count: not read
    counts = np.zeros((B, H), np.int32)
    for b in range(B):
        for h in range(H):
            counts[b, h] = rng.integers(0, most + 1) if (b, h) != (0, 0) else most
            listed[b, h, :counts[b, h]] = rng.integers(-1, -(-lens[b] // PAGE), counts[b, h])
    listed[0, 0, :2] = -7, 0
    selected = torch.from_numpy(listed).cuda(), torch.from_numpy(counts).cuda()
    call = reef.attention_decode_int4 if bits == 4 else reef.attention_decode_selected
    tq, tqs = torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda()
    for window, splits in ((0, 0), (40, 0), (0, 5)):
        def seen(b, h):
            t = [PAGE * p + i for p in listed[b, h, :counts[b, h]] if p >= 0 for i in range(PAGE)]
            return [x for x in t if x < lens[b] and (not window or x >= lens[b] - window)]
        want, tol = attention(cache, q, qs, seen)
        got = call(tq, tqs, *cache.tensors, cache.context_lens, selected=selected,
                   block_table=cache.block_table, window=window, num_splits=splits)
        assert np.abs(got.double().cpu().numpy() - want).max() <= tol, (window, splits)


@pytest.mark.parametrize("bits", [4, 8])
def test_decode_listed_more_sequences_than_a_plan(reef, bits):
    rng = np.random.default_rng(bits)
    lens = [int(n) for n in rng.integers(1, 129, 520)]
    cache = Cache(rng, bits, 520, 4, 64, 128, lens, True)
    q, qs = queries(rng, 520, 4, 64)
    listed = np.stack([rng.permutation(8)[:5] for _ in range(520 * 4)]).reshape(520, 4, 5)
    listed = np.where(listed < -(-np.array(lens)[:, None, None] // PAGE), listed, -1).astype(np.int32)
    selected = torch.from_numpy(listed).cuda(), torch.full((520, 4), 5, dtype=torch.int32).cuda()
    call = reef.attention_decode_int4 if bits == 4 else reef.attention_decode_selected
    want, tol = attention(cache, q, qs, lambda b, h: [
        t for p in listed[b, h] if p >= 0 for t in range(PAGE * p, min(PAGE * p + PAGE, lens[b]))])
    got = call(torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda(), *cache.tensors,
               cache.context_lens, selected=selected, block_table=cache.block_table)
    assert np.abs(got.double().cpu().numpy() - want).max() <= tol


@pytest.mark.parametrize("B,H", [(1, 3), (40, 8), (130, 8)])
@pytest.mark.parametrize("bits", [4, 8])
def test_decode_lists_longer_than_the_cache(reef, bits, B, H):
    """A few pages named many times, by some sequences: parts of long lists next to short ones."""
    rng = np.random.default_rng(bits + B)
    L = 592  # 10 blocks of 64 keys: more than a part has at least
    lens = [L if i % 2 else 16 for i in range(B)]
    cache = Cache(rng, bits, B, H, 64, L, lens, False)
    q, qs = queries(rng, B, H, 64)
    listed = np.stack([rng.integers(0, -(-lens[i // H] // PAGE), 300) for i in range(B * H)])
    listed = listed.reshape(B, H, 300).astype(np.int32)
    counts = np.where(rng.random((B, H)) < 0.2, 300, rng.integers(0, 20, (B, H))).astype(np.int32)
    counts[0, 0] = 300
    call = reef.attention_decode_int4 if bits == 4 else reef.attention_decode_selected
    want, tol = attention(cache, q, qs, lambda b, h: [
        t for p in listed[b, h, :counts[b, h]] for t in range(PAGE * p, min(PAGE * p + PAGE, lens[b]))])
    for _ in range(2):
        got = call(torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda(), *cache.tensors,
                   cache.context_lens,
                   selected=(torch.from_numpy(listed).cuda(), torch.from_numpy(counts).cuda()))
        assert np.abs(got.double().cpu().numpy() - want).max() <= tol


@pytest.mark.parametrize("bits", [4, 8])
def test_decode_listed_bad_entries(reef, bits):
    rng = np.random.default_rng(bits)
    cache = Cache(rng, bits, 4, 1, 128, 96, [50, 50, 50, 50], True)
    q, qs = queries(rng, 4, 2, 128)
    tq, tqs = torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda()
    call = reef.attention_decode_int4 if bits == 4 else reef.attention_decode_selected
    listed = np.array([[[0, 4, 2]], [[1 << 30, 3, 1]], [[0, 1, 2]], [[0, 1, 2]]], np.int32)
    counts = np.array([[3], [2], [4], [-1]], np.int32)  # a page past the end, counts outside
    status = reef.StatusWord("cuda")
    got = call(tq, tqs, *cache.tensors, cache.context_lens, status=status,
               selected=(torch.from_numpy(listed).cuda(), torch.from_numpy(counts).cuda()),
               block_table=cache.block_table)
    with pytest.raises(reef.InvalidArgument):
        status.check("decode")
    pages = {0: [0, 2], 1: [3], 2: [], 3: []}
    want, tol = attention(cache, q, qs, lambda b, h: [
        t for p in pages[b] for t in range(PAGE * p, min(PAGE * p + PAGE, 50))])
    assert np.abs(got.double().cpu().numpy() - want).max() <= tol


# --- a serving step ------------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("paged", [False, True])
def test_steps(reef, bits, paged):
    """Prompt, then tokens one by one: append, bounds, selection, attention. The whole budget is
    the dense step; a smaller one reads what its list says. A captured step replays them."""
    rng = np.random.default_rng(bits + paged)
    B, H, G, D, L, T = 2, 2, 2, 64, 512, 300
    cache = Cache(rng, bits, B, H, D, L, [L] * B, paged)
    tensors, table = cache.tensors, cache.block_table
    lead = (tensors[0].shape[0], H) if paged else (B, H, L // PAGE)
    bounds = torch.zeros((*lead, 2, D), dtype=torch.int8, device="cuda")
    scales = torch.zeros(lead, device="cuda")
    status = reef.StatusWord("cuda")

    def append(x, start, lens):
        if bits == 4:
            reef.kv_append_int4(x, x, start, *tensors, lens, block_table=table, status=status)
        elif paged:
            reef.kv_append_paged(x, x, start, table, *tensors, lens, status=status)
        else:
            reef.kv_append(x, x, start, *tensors, lens, status=status)
        reef.kv_page_bounds(start, x.shape[2], tensors[0], tensors[2], bounds, scales,
                            block_table=table, status=status)

    sparse = reef.attention_decode_int4 if bits == 4 else reef.attention_decode_selected

    def dense(q, qs, lens):
        if bits == 4:
            return reef.attention_decode_int4(q, qs, *tensors, lens, block_table=table, status=status)
        if paged:
            return reef.attention_decode_paged(q, qs, *tensors, table, lens, status=status)
        return reef.attention_decode(q, qs, *tensors, lens, status=status)

    def step(x, q, qs, start, lens, budget):
        append(x, start, lens)
        chosen = reef.kv_select_pages(q, qs, bounds, scales, lens, budget, block_table=table, sinks=1,
                                      recent=2, status=status)
        return chosen, sparse(q, qs, *tensors, lens, selected=chosen, block_table=table, status=status)

    start, lens = ints([0, 0]), ints([0, 0])
    append(torch.randn(B, H, T, D, device="cuda"), start, lens)
    x = torch.randn(B, H, 1, D, device="cuda")
    q, qs = (torch.from_numpy(a).cuda() for a in queries(rng, B, H * G, D))
    start.copy_(lens)
    _, out = step(x, q, qs, start, lens, L // PAGE)
    # all pages: the same sums in another order of blocks at most
    n, top = T + 1, tensors[3].nan_to_num().max().item() * (7 if bits == 4 else 127)
    assert (out - dense(q, qs, lens)).abs().max() <= 2 * top * (n + 64) * 2.0 ** -24 * 2

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            step(x, q, qs, start, lens, 7)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            held = step(x, q, qs, start, lens, 7)
    torch.cuda.current_stream().wait_stream(stream)
    for _ in range(20):  # across a page's end
        x.normal_()
        start.copy_(lens)
        q.copy_(torch.randint(-127, 128, q.shape, device="cuda", dtype=torch.int8))
        (pages, counts), want = step(x, q, qs, start, lens, 7)
        torch.cuda.synchronize()
        want, pages, counts = want.clone(), pages.clone(), counts.clone()
        graph.replay()  # the same tokens once more, at the same places
        torch.cuda.synchronize()
        assert torch.equal(held[0][0], pages) and torch.equal(held[0][1], counts)
        assert torch.equal(held[1], want)
    status.check("steps")
    assert lens.tolist() == [T + 21] * B


@pytest.mark.parametrize("bits", [4, 8])
def test_two_streams(reef, bits):
    """Calls in flight at the same time share no workspace."""
    rng = np.random.default_rng(30 + bits)
    call = reef.attention_decode_int4 if bits == 4 else reef.attention_decode_selected
    jobs = []
    for i in range(2):
        cache = Cache(rng, bits, 4, 4, 128, 4096, [4096, 3000, 2000, 1000], True)
        q, qs, *_ = (torch.from_numpy(a).cuda() for a in queries(rng, 4, 16, 128))
        bounds = torch.zeros((cache.tensors[0].shape[0], 4, 2, 128), dtype=torch.int8, device="cuda")
        scales = torch.ones(bounds.shape[:2], device="cuda")
        reef.kv_page_bounds(ints([0] * 4), 1000, cache.tensors[0], cache.tensors[2], bounds, scales,
                            block_table=cache.block_table)
        jobs.append((cache, q, qs, bounds, scales))

    def run(job):
        cache, q, qs, bounds, scales = job
        chosen = reef.kv_select_pages(q, qs, bounds, scales, cache.context_lens, 40,
                                      block_table=cache.block_table, status=word)
        return [*chosen, call(q, qs, *cache.tensors, cache.context_lens, selected=chosen,
                              block_table=cache.block_table, status=word)]

    word = reef.StatusWord("cuda")
    want = [run(j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(jobs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))
