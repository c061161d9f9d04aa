"""The forms of launch that the sizes of the other tests do not reach: chunks over the 4-bit cache
through its copy (both head_dims, contiguous and paged, bad pages, scales on 4 bytes, an asked-for
schedule), bounds of several pages a wave, appends with pages first, unpacking over several rows of
workgroups. All bit for bit."""
import ctypes as C

import numpy as np
import pytest

from kv_reads import PAGE, Cache, unpack_keys, unpack_values

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


def widened(cache):
    """The int8 cache of the same codes."""
    k, v, ks, vs = cache.tensors
    wide_k = unpack_keys(k.cpu().numpy()).astype(np.int8)
    wide_v = np.swapaxes(unpack_values(v.cpu().numpy()), -1, -2).astype(np.int8)
    return [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (wide_k, wide_v)] + [ks, vs]


def on_4_bytes(t):
    """The same values 4 bytes behind a 16-byte address."""
    held = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    held[1:] = t.flatten()
    return held[1:].view(t.shape)


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("B,H,G,D,T,n,window", [
    (1, 1, 16, 64, 2064, 2070, 0), (1, 1, 16, 128, 2064, 2077, 0),  # too many rows for a short chunk
    (2, 3, 1, 64, 37, 333, 0), (2, 2, 3, 128, 37, 333, 100), (3, 1, 2, 64, 1, 16, 0),
    (1, 2, 4, 128, 5, 5, 0),
])
def test_chunk_through_the_copy(reef, paged, B, H, G, D, T, n, window):
    """The int8 prefill's result on the same codes."""
    rng = np.random.default_rng(T + n + paged)
    cache = Cache(rng, 4, B, H, D, -(-n // PAGE) * PAGE, [n] * B, paged)
    q = torch.from_numpy(rng.integers(-127, 128, (B, H * G, T, D)).astype(np.int8)).cuda()
    qs = torch.rand(H * G, device="cuda") * 0.01 + 0.01
    k, v, ks, vs = cache.tensors
    if T < 100:  # a short chunk: through the copy with scales that are not on 16 bytes
        ks, vs = on_4_bytes(ks), on_4_bytes(vs)
        assert ks.data_ptr() % 16 and vs.data_ptr() % 16
    where = dict(block_table=cache.block_table, window=window)
    got = reef.attention_prefill_cache_int4(q, qs, k, v, ks, vs, n, **where)
    assert torch.equal(got, reef.attention_prefill_cache(q, qs, *widened(cache), n, **where))
    assert got.isfinite().all()


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_chunk_of_an_asked_for_schedule(reef, paged, D):
    rng = np.random.default_rng(D + paged)
    B, H, G, T, n = 2, 2, 2, 40, 200
    cache = Cache(rng, 4, B, H, D, 208, [n] * B, paged)
    q = torch.from_numpy(rng.integers(-127, 128, (B, H * G, T, D)).astype(np.int8)).cuda()
    qs = torch.rand(H * G, device="cuda") * 0.01 + 0.01
    lib = reef.lib()
    table = cache.block_table
    for schedule in (reef.SCHED_ONE_ITEM, reef.SCHED_BALANCED):
        p = reef.AttentionParams(B, H * G, H, T, n, D, n - T, 0, D ** -0.5, reef.PER_HEAD,
                                 reef.PER_TOKEN, schedule)
        size = lib.reef_attention_prefill_cache_workspace_bytes(C.byref(p))
        ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
        outs = []
        for call, tensors in ((lib.reef_attention_prefill_int4_cache, cache.tensors),
                              (lib.reef_attention_prefill_int8_cache, widened(cache))):
            out = torch.full((B, H * G, T, D), 7.0, device="cuda")
            assert call(C.byref(p), q.data_ptr(), None, qs.data_ptr(), *(t.data_ptr() for t in tensors),
                        208, table.data_ptr() if paged else None, 13 if paged else 0,
                        cache.tensors[0].shape[0] if paged else 0, out.data_ptr(), None, ws.data_ptr(),
                        size, None, torch.cuda.current_stream().cuda_stream) == reef.OK
            torch.cuda.synchronize()
            outs.append(out)
        assert torch.equal(*outs)


@pytest.mark.parametrize("D", [64, 128])
def test_copy_of_bad_pages(reef, D):
    rng = np.random.default_rng(D)
    n = 333
    cache = Cache(rng, 4, 2, 2, D, 336, [n] * 2, True)
    q = torch.from_numpy(rng.integers(-127, 128, (2, 4, 9, D)).astype(np.int8)).cuda()
    qs = torch.rand(4, device="cuda") * 0.01 + 0.01
    table = cache.block_table.clone()
    table[0, 1], table[1, 20], table[1, 3] = -1, 1 << 20, cache.tensors[0].shape[0]
    k, v, ks, vs = cache.tensors
    outs = []
    for call, tensors in ((reef.attention_prefill_cache_int4, [k, v, on_4_bytes(ks), on_4_bytes(vs)]),
                          (reef.attention_prefill_cache, widened(cache))):
        status = reef.StatusWord("cuda")
        outs.append(call(q, qs, *tensors, n, block_table=table, status=status))
        with pytest.raises(reef.InvalidArgument):
            status.check("chunk")
    assert torch.equal(*outs) and outs[0].isfinite().all()


@pytest.mark.parametrize("bits,paged,D", [(8, False, 64), (8, True, 128), (4, False, 128), (4, True, 64)])
def test_bounds_of_several_pages_a_wave(reef, bits, paged, D):
    """More than 32768 (page, head, sequence) triples; ranges that begin in a page and end inside a
    wave's run of four, and a page that is not there in the middle of one."""
    g = torch.Generator(device="cuda").manual_seed(bits + D)
    B, H, T = 2, 16, 16403
    starts = [5, 37]
    blocks = -(-(max(starts) + T) // PAGE)
    pages = B * blocks + 1
    assert (-(-T // PAGE) + 1) * B * H > 32768 and (starts[0] + T) % (4 * PAGE)
    lead = (pages, H) if paged else (B, H, blocks)
    if bits == 8:
        codes = torch.randint(-127, 128, (*lead, PAGE, D), generator=g, device="cuda", dtype=torch.int8)
        k = codes
    else:
        k = torch.randint(0, 256, (*lead, PAGE, D // 2), generator=g, device="cuda", dtype=torch.uint8)
        codes = torch.cat([k & 15, k >> 4], -1).to(torch.int8) - 8
    ks = torch.rand((*lead, PAGE), generator=g, device="cuda") + 0.1
    bounds = torch.full((*lead, 2, D), 3, dtype=torch.int8, device="cuda")
    scales = torch.full(lead, 2.0, device="cuda")
    want, want_s = bounds.clone(), scales.clone()
    table = torch.randperm(pages, generator=g, device="cuda")[:B * blocks].view(B, blocks)
    bad = 517  # of the first sequence: third of a wave's four
    for b in range(B):
        end = starts[b] + T
        block = torch.arange(starts[b] // PAGE, (end - 1) // PAGE + 1, device="cuda")
        at = table[b, block] if paged else (b, slice(None), block)
        x, s = codes[at], ks[at]                       # paged: [n, H, 16, D]; else [H, n, 16, D]
        if not paged:
            x, s = x.transpose(0, 1), s.transpose(0, 1)
        x = x.float() * s[..., None]
        live = (block[:, None] * PAGE + torch.arange(PAGE, device="cuda") < end)[:, None, :, None]
        most = x.masked_fill(~live, 0).abs().amax((-1, -2))
        scale = most / torch.full_like(most, 127)
        high = x.masked_fill(~live, -np.inf).amax(-2) / scale[..., None]
        low = x.masked_fill(~live, np.inf).amin(-2) / scale[..., None]
        codes_of = torch.stack([high.ceil().clamp(max=127), low.floor().clamp(min=-127)], -2).to(torch.int8)
        if paged:
            keep = block != bad if b == 0 else slice(None)
            want[at[keep]], want_s[at[keep]] = codes_of[keep], scale[keep]
        else:
            want[at], want_s[at] = codes_of.transpose(0, 1), scale.t()
    held = table.int()
    status = reef.StatusWord("cuda")
    if paged:
        held[0, bad] = -1
    cache = (k, ks) if paged else (k.flatten(2, 3), ks.flatten(2, 3))
    reef.kv_page_bounds(ints(starts), T, *cache, bounds, scales, status=status,
                        block_table=held if paged else None)
    if paged:
        with pytest.raises(reef.InvalidArgument):
            status.check("bounds")
    else:
        status.check("bounds")
    assert torch.equal(scales, want_s)
    assert torch.equal(bounds, want)


def test_append_with_pages_first(reef):
    """More pages than a grid's second dimension has: as two appends of half the rows."""
    T, H, D = 65535 * PAGE + 7, 2, 64
    half = 600_001
    L = T + 9
    assert L % PAGE == 0
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn((1, T, H, D), generator=g, device="cuda").transpose(1, 2) for _ in range(2))

    def empty():
        return [torch.full((1, H, L, D // 2), 0x5a, dtype=torch.uint8, device="cuda"),
                torch.full((1, H, L // PAGE, D, 8), 0x5a, dtype=torch.uint8, device="cuda"),
                torch.zeros(1, H, L, device="cuda"), torch.zeros(1, H, L, device="cuda")]

    one, two = empty(), empty()
    lens = ints([0])
    reef.kv_append_int4(k, v, ints([3]), *one, lens)
    reef.kv_append_int4(k[:, :, :half], v[:, :, :half], ints([3]), *two)
    reef.kv_append_int4(k[:, :, half:], v[:, :, half:], ints([3 + half]), *two)
    assert lens.tolist() == [3 + T]
    for a, b in zip(one, two):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128])
def test_unpack_many_pages(reef, D):
    """More pages than one row of workgroups has."""
    pages, some = (1 << 21) + 5, 33
    g = torch.Generator(device="cuda").manual_seed(D)
    k = torch.randint(0, 256, (pages, 1, PAGE, D // 2), generator=g, device="cuda", dtype=torch.uint8)
    v = torch.randint(0, 256, (pages, 1, D, 8), generator=g, device="cuda", dtype=torch.uint8)
    ks, vs = (torch.rand((pages, 1, PAGE), generator=g, device="cuda") for _ in range(2))
    whole = reef.kv_unpack_int4(k, v, ks, vs)
    for at in (0, (1 << 20) + 3, (1 << 21) - some + 2, pages - some):
        part = reef.kv_unpack_int4(*(t[at:at + some].clone() for t in (k, v, ks, vs)))
        assert all(torch.equal(a[at:at + some], b) for a, b in zip(whole, part))
