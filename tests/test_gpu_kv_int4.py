"""The KV cache held in 4 bits: append, unpack, copies of pages, decode and prefill over it,
against their definitions in 64 bits (codes, scales and bytes exactly)."""
import math

import numpy as np
import pytest

from kv_reads import (PAGE, U, Cache, attention, pack_keys, pack_values, quantized, queries,
                      unpack_keys, unpack_values)

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


# --- append, unpack, copies ------------------------------------------------------------------

@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("B,H,D,T,starts", [
    (1, 1, 64, 1, [0]), (3, 2, 128, 1, [0, 15, 47]), (2, 3, 128, 7, [12, 3]),
    (2, 1, 64, 16, [16, 8]), (2, 2, 128, 33, [0, 31]), (1, 2, 64, 64, [0]),
])
def test_append(reef, paged, B, H, D, T, starts):
    rng = np.random.default_rng(T + D + paged)
    cache = Cache(rng, 4, B, H, D, 64, [64] * B, paged)
    x, y = (rng.normal(0, 1, (B, T, H, D)).astype(np.float32) for _ in range(2))
    x[0, 0, 0] = 0                                  # a row of zeros
    x[-1, -1, -1, :8] = [3.5, -3.5, 7, -7, 0.5, 1.5, 2.5, -0.5]  # ties of scale 1
    x[-1, -1, -1, 8:] = 0
    new = [torch.from_numpy(a).cuda().transpose(1, 2) for a in (x, y)]  # as a projection lies
    k, v, ks, vs = (t.clone() for t in cache.tensors)
    lens = torch.full((B,), -1, dtype=torch.int32).cuda()
    reef.kv_append_int4(*new, ints(starts), k, v, ks, vs, lens, block_table=cache.block_table)
    assert lens.tolist() == [s + T for s in starts]
    want = []
    for a, codes, scales in ((x, cache.k.copy(), cache.ks.copy()), (y, cache.v.copy(), cache.vs.copy())):
        c, s = quantized(a, 7)
        for b in range(B):
            codes[b, :, starts[b]:starts[b] + T] = np.swapaxes(c[b], 0, 1)
            scales[b, :, starts[b]:starts[b] + T] = s[b].T
        want += [codes, scales]
    wk, wks, wv, wvs = want
    wv = wv.reshape(B, H, -1, PAGE, D)

    def seen(t, rows):  # back by sequences
        t = t.cpu().numpy()
        if paged:
            t = np.swapaxes(t[cache.table], 1, 2)  # [B, H, blocks, ...]
            return t.reshape(B, H, 64, *t.shape[4:]) if rows else t
        return t

    assert np.array_equal(seen(k, True), pack_keys(wk))
    assert np.array_equal(seen(v, False), pack_values(wv))
    assert np.array_equal(seen(ks, True), wks) and np.array_equal(seen(vs, True), wvs)
    if paged:  # other sequences' pages
        others = np.setdiff1d(np.arange(k.shape[0]), cache.table)
        for a, b in zip((k, v, ks, vs), cache.tensors):
            assert torch.equal(a[others], b[others])
    fk, fv = reef.kv_unpack_int4(k, v, ks, vs)
    for f, codes, s in ((fk, unpack_keys(k.cpu().numpy()), ks), (fv, unpack_values(v.cpu().numpy()), vs)):
        s = s.cpu().numpy()
        codes = codes.reshape(*f.shape).astype(np.float32)
        assert np.array_equal(f.cpu().numpy(), codes * s.reshape(*f.shape[:-1], 1))


def test_append_in_place_lengths_and_what_is_refused_leaves_the_cache(reef):
    rng = np.random.default_rng(5)
    cache = Cache(rng, 4, 3, 2, 64, 32, [32] * 3, True)
    before = [t.clone() for t in cache.tensors]
    new = [torch.randn(3, 2, 5, 64, device="cuda") for _ in range(2)]
    lens = ints([-1, 28, 6])
    with pytest.raises((reef.InvalidArgument, reef.CapacityError)):
        reef.kv_append_int4(*new, lens, *cache.tensors, lens, block_table=cache.block_table)
    assert lens.tolist() == [-1, 28, 11]  # the third sequence's tokens went in
    keep = cache.block_table[:2].long().flatten()
    for a, b in zip(cache.tensors, before):
        assert torch.equal(a[keep], b[keep])
    table = cache.block_table.clone()
    table[0, 0] = 99
    with pytest.raises(reef.InvalidArgument):
        reef.kv_append_int4(*new, ints([0, 0, 0]), *cache.tensors, block_table=table)
    new[0][1, 1, 2, 3] = math.inf
    with pytest.raises(reef.NonFiniteInput):
        reef.kv_append_int4(*new, ints([0, 0, 0]), *cache.tensors, block_table=cache.block_table)


@pytest.mark.parametrize("H,D", [(1, 64), (3, 128)])
def test_copy_pages(reef, H, D):
    g = torch.Generator(device="cuda").manual_seed(3)
    pool = [torch.randint(0, 256, s, generator=g, device="cuda", dtype=torch.uint8)
            for s in ((9, H, 16, D // 2), (9, H, D, 8))]
    pool += [torch.rand((9, H, 16), generator=g, device="cuda") for _ in range(2)]
    want = [t.clone() for t in pool]
    for t in want:
        t[[4, 0]] = t[[1, 8]]
    reef.kv_copy_pages_int4(ints([1, -1, 8]), ints([4, 2, 0]), *pool)
    for a, b in zip(pool, want):
        assert torch.equal(a, b)
    with pytest.raises(reef.InvalidArgument):
        reef.kv_copy_pages_int4(ints([9]), ints([0]), *pool)


# --- decode ---------------------------------------------------------------------------------------

DECODE = [  # B, kv heads, group, D, L, lens, window
    (1, 1, 1, 64, 16, [1], 0), (2, 2, 4, 128, 16, [16, 15], 0), (3, 1, 16, 128, 144, [1, 17, 143], 0),
    (1, 12, 1, 64, 208, [200], 0), (4, 2, 7, 64, 1024, [1, 63, 64, 1000], 0),
    (2, 8, 4, 128, 512, [511, 65], 0), (3, 2, 2, 128, 512, [512, 100, 40], 48),
    (2, 1, 8, 64, 4096, [4095, 2049], 0), (2, 1, 1, 128, 4096, [4096, 129], 1000),
]


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("B,H,G,D,L,lens,window", DECODE)
def test_decode(reef, paged, B, H, G, D, L, lens, window):
    rng = np.random.default_rng(L + B + paged)
    cache = Cache(rng, 4, B, H, D, L, lens, paged)
    q, qs = queries(rng, B, H * G, D)
    want, tol = attention(cache, q, qs, lambda b, h: range(max(0, lens[b] - window) if window else 0,
                                                           lens[b]))
    tq, tqs = torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda()
    for splits in (0, 1, 9):
        got = reef.attention_decode_int4(tq, tqs, *cache.tensors, cache.context_lens,
                                         block_table=cache.block_table, window=window,
                                         num_splits=splits)
        assert np.abs(got.double().cpu().numpy() - want).max() <= tol, splits


def test_decode_scale_forms_and_a_full_cache(reef):
    rng = np.random.default_rng(11)
    cache = Cache(rng, 4, 2, 2, 128, 80, [80, 80], False)
    q, _ = queries(rng, 2, 6, 128)
    tq = torch.from_numpy(q).cuda()
    for form, s in ((reef.PER_TENSOR, np.float32([0.01])),
                    (reef.PER_HEAD, rng.uniform(0.005, 0.02, 6).astype(np.float32))):
        qs = np.broadcast_to(s, (2, 6))
        want, tol = attention(cache, q, qs, lambda b, h: range(80))
        got = reef.attention_decode_int4(tq, torch.from_numpy(s).cuda(), *cache.tensors,
                                         q_granularity=form)
        assert np.abs(got.double().cpu().numpy() - want).max() <= tol


@pytest.mark.parametrize("B,H,L", [(20, 8, 1040), (48, 8, 1040), (256, 8, 704), (2, 1, 6000)])
def test_decode_lengths_far_apart(reef, B, H, L):
    """One or a few long sequences among short ones: items of several parts and of one, few and many
    of them, the same bits on every run."""
    rng = np.random.default_rng(B)
    lens = [int(n) for n in rng.integers(1, 200, B)]
    for i in rng.choice(B, max(1, B // 16), replace=False):
        lens[i] = L - int(rng.integers(0, 100))
    cache = Cache(rng, 4, B, H, 64, L, lens, True)
    q, qs = queries(rng, B, 2 * H, 64)
    tq, tqs = torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda()
    want, tol = attention(cache, q, qs, lambda b, h: range(lens[b]))
    runs = [reef.attention_decode_int4(tq, tqs, *cache.tensors, cache.context_lens,
                                       block_table=cache.block_table) for _ in range(4)]
    assert np.abs(runs[0].double().cpu().numpy() - want).max() <= tol
    assert all(torch.equal(r, runs[0]) for r in runs)


def test_decode_more_sequences_than_a_plan(reef):
    """Beyond 2048 (sequence, kv head) pairs a launch deals out whole sequences."""
    rng = np.random.default_rng(12)
    lens = [int(n) for n in rng.integers(1, 65, 300)]
    cache = Cache(rng, 4, 300, 8, 64, 64, lens, True)
    q, qs = queries(rng, 300, 8, 64)
    want, tol = attention(cache, q, qs, lambda b, h: range(lens[b]))
    got = reef.attention_decode_int4(torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda(),
                                     *cache.tensors, cache.context_lens, block_table=cache.block_table)
    assert np.abs(got.double().cpu().numpy() - want).max() <= tol


def test_decode_bad_lengths_and_pages(reef):
    rng = np.random.default_rng(13)
    cache = Cache(rng, 4, 3, 2, 64, 64, [40, 40, 40], True)
    q, qs = queries(rng, 3, 4, 64)
    tq, tqs = torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda()
    status = reef.StatusWord("cuda")
    got = reef.attention_decode_int4(tq, tqs, *cache.tensors, ints([0, 40, 65]),
                                     block_table=cache.block_table, status=status)
    with pytest.raises(reef.InvalidArgument):
        status.check("decode")
    want, tol = attention(cache, q, qs, lambda b, h: range(40) if b == 1 else [])
    assert np.abs(got.double().cpu().numpy() - want).max() <= tol
    table = cache.block_table.clone()
    table[0, 1], table[2, 0] = -1, table.numel() + 3
    got = reef.attention_decode_int4(tq, tqs, *cache.tensors, cache.context_lens, block_table=table,
                                     status=status)
    with pytest.raises(reef.InvalidArgument):
        status.check("decode")
    dead = {0: range(16, 32), 2: range(16)}
    want, tol = attention(cache, q, qs, lambda b, h: [t for t in range(40) if t not in dead.get(b, ())])
    assert np.abs(got.double().cpu().numpy() - want).max() <= tol


# --- prefill over the cache -------------------------------------------------------------------------

@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("B,H,G,D,T,n,window", [
    (1, 1, 1, 64, 1, 1, 0), (2, 2, 2, 128, 5, 21, 0), (1, 3, 4, 64, 33, 33, 0),
    (2, 1, 8, 128, 77, 333, 0), (1, 2, 1, 64, 130, 1021, 0), (2, 1, 2, 128, 40, 200, 64),
])
def test_chunk(reef, paged, B, H, G, D, T, n, window):
    """Row by row, whichever way the chunk runs: the prefill's own tolerance is 1e-3."""
    rng = np.random.default_rng(T + n + paged)
    L = -(-n // PAGE) * PAGE
    cache = Cache(rng, 4, B, H, D, L, [n] * B, paged)
    q = rng.integers(-127, 128, (B, H * G, T, D)).astype(np.int8)
    qs = rng.uniform(0.005, 0.02, H * G).astype(np.float32)
    got = reef.attention_prefill_cache_int4(torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda(),
                                            *cache.tensors, n, block_table=cache.block_table,
                                            window=window).double().cpu().numpy()
    for i in range(T):
        last = n - T + i
        want, tol = attention(cache, q[:, :, i], np.broadcast_to(qs, (B, H * G)),
                              lambda b, h: range(max(0, last + 1 - window) if window else 0, last + 1))
        assert np.abs(got[:, :, i] - want).max() <= max(tol, 1e-3), i


def test_long_chunk_is_the_int8_prefill_on_the_same_codes(reef):
    """Where the codes are widened they are the int8 cache's: the same results, bit for bit."""
    rng = np.random.default_rng(15)
    cache = Cache(rng, 4, 2, 2, 128, 4112, [4100, 4100], True)
    k, v, ks, vs = cache.tensors
    wide_k = torch.from_numpy(unpack_keys(k.cpu().numpy()).astype(np.int8)).cuda()
    wide_v = torch.from_numpy(np.ascontiguousarray(
        np.swapaxes(unpack_values(v.cpu().numpy()), -1, -2)).astype(np.int8)).cuda()
    q = torch.from_numpy(rng.integers(-127, 128, (2, 16, 128, 128)).astype(np.int8)).cuda()
    qs = torch.rand(16, device="cuda") * 0.01 + 0.01
    a = reef.attention_prefill_cache_int4(q, qs, *cache.tensors, 4100, block_table=cache.block_table)
    b = reef.attention_prefill_cache(q, qs, wide_k, wide_v, ks, vs, 4100, block_table=cache.block_table)
    assert torch.equal(a, b)


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("B,H,G,D,T,n,window,form", [
    (1, 1, 1, 64, 3, 3, 0, 2), (2, 1, 3, 128, 1, 130, 0, 2), (1, 2, 4, 128, 2, 700, 100, 1),
    (3, 2, 1, 64, 17, 65, 0, 0), (1, 1, 7, 64, 9, 1500, 0, 2), (2, 3, 5, 128, 10, 64, 20, 1),
    (1, 1, 40, 64, 2, 300, 0, 2), (2, 2, 2, 64, 300, 300, 0, 1), (1, 1, 2, 128, 64, 5000, 0, 2),
])
def test_short_chunk(reef, paged, B, H, G, D, T, n, window, form):
    """Rows as columns: groups that end inside a tile of them, strided rows, every form of scales,
    a query of its own place (query_start). Tolerance: kv_reads.attention's."""
    rng = np.random.default_rng(T + n + paged)
    L = -(-n // PAGE) * PAGE + 16
    cache = Cache(rng, 4, B, H, D, L, [n] * B, paged)
    q = rng.integers(-127, 128, (B, T, H * G, D)).astype(np.int8)  # as a projection lays them out
    shape = {0: (1,), 1: (H * G,), 2: (B, H * G, T)}[form]
    qs = rng.uniform(0.005, 0.02, shape).astype(np.float32)
    full = np.broadcast_to(qs.reshape({0: (1, 1, 1), 1: (1, H * G, 1), 2: shape}[form]), (B, H * G, T))
    tq = torch.from_numpy(q).cuda().transpose(1, 2)
    out = torch.full((B, T, H * G, D), 9.0, device="cuda").transpose(1, 2)
    for start in (n - T, (n - T) // 2):
        reef.attention_prefill_cache_int4(tq, torch.from_numpy(qs).cuda(), *cache.tensors, n,
                                          block_table=cache.block_table, window=window,
                                          query_start=start, q_granularity=form, out=out)
        got = out.double().cpu().numpy()
        for i in range(T):
            end = start + i + 1
            want, tol = attention(cache, q[:, i], full[:, :, i],
                                  lambda b, h: range(max(0, end - window) if window else 0, end))
            assert np.abs(got[:, :, i] - want).max() <= tol, (start, i)


def test_short_chunk_bad_pages_read_as_zero_codes(reef):
    rng = np.random.default_rng(17)
    cache = Cache(rng, 4, 2, 2, 64, 96, [90, 90], True)
    q = rng.integers(-127, 128, (2, 4, 5, 64)).astype(np.int8)
    qs = rng.uniform(0.005, 0.02, 4).astype(np.float32)
    table = cache.block_table.clone()
    table[0, 1], table[1, 3] = -1, 1 << 20
    cache.k[0, :, 16:32] = cache.v[0, :, 16:32] = 0
    cache.k[1, :, 48:64] = cache.v[1, :, 48:64] = 0
    status = reef.StatusWord("cuda")
    got = reef.attention_prefill_cache_int4(torch.from_numpy(q).cuda(), torch.from_numpy(qs).cuda(),
                                            *cache.tensors, 90, block_table=table, status=status)
    with pytest.raises(reef.InvalidArgument):
        status.check("chunk")
    for i in range(5):
        want, tol = attention(cache, q[:, :, i], np.broadcast_to(qs, (2, 4)), lambda b, h: range(86 + i))
        assert np.abs(got[:, :, i].double().cpu().numpy() - want).max() <= tol
