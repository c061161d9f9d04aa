"""Refusals of the drafted-token, page, norm and epilogue calls, without a GPU: the C entry
points on the host before any launch, and the Python wrappers."""
import ctypes as C

import pytest

import reef_amd
from reef_amd import Epilogue, KvAppendParams, Strides, TreeParams

OK, INVALID, CAPACITY, UNSUPPORTED = (reef_amd.OK, reef_amd.INVALID_ARGUMENT, reef_amd.CAPACITY,
                                      reef_amd.UNSUPPORTED)


def at(n=1, offset=0):
    # Non-null, 256-byte aligned host addresses: validation never dereferences them.
    return C.c_void_p(0x10000 * n + offset)


# --- attention of drafted tokens ------------------------------------------------------------

def tree_params(**kw):
    d = dict(batch=2, q_heads=8, kv_heads=2, head_dim=128, draft_len=5, max_context=64, window=0,
             softmax_scale=0.1, q_granularity=2, flags=0, reserved=0)
    d.update(kw)
    return TreeParams(**d)


def tree(p, q=at(1), q_strides=None, mask=at(9), out=at(10), out_strides=None, ws=at(11),
         ws_bytes=1 << 40, ks=at(5)):
    return reef_amd.lib().reef_attention_decode_tree_int8(
        p, q, q_strides, at(2), at(3), at(4), ks, at(6), at(7), mask, out, out_strides, ws,
        ws_bytes, None, None)


def tree_paged(p, table=at(8), blocks=4, pages=9, lens=at(7), ws_bytes=1 << 40):
    return reef_amd.lib().reef_attention_decode_tree_int8_paged(
        p, at(1), None, at(2), at(3), at(4), at(5), at(6), table, blocks, pages, lens, at(9),
        at(10), None, at(11), ws_bytes, None, None)


@pytest.mark.parametrize("change,status", [
    (dict(batch=0), INVALID), (dict(draft_len=0), INVALID), (dict(q_heads=3), INVALID),
    (dict(max_context=60), INVALID), (dict(window=-1), INVALID), (dict(flags=1), INVALID),
    (dict(softmax_scale=0.0), INVALID), (dict(softmax_scale=float("inf")), INVALID),
    (dict(softmax_scale=float("nan")), INVALID), (dict(q_granularity=3), INVALID),
    (dict(head_dim=96), UNSUPPORTED), (dict(draft_len=65, max_context=128), UNSUPPORTED),
    (dict(q_heads=2050), UNSUPPORTED),              # 1025 query heads of a key head
    (dict(max_context=1 << 30), UNSUPPORTED), (dict(batch=65536), UNSUPPORTED),
    (dict(draft_len=17, max_context=16), CAPACITY),
    (dict(batch=2048, max_context=1 << 24, kv_heads=8), UNSUPPORTED),  # 2^31 pages and more
    # fewer pages than that, but more units of work: 2048 column ranges a key head
    (dict(batch=2048, q_heads=1024, kv_heads=1, draft_len=64, max_context=1 << 16), UNSUPPORTED),
])
def test_tree_sizes(change, status):
    assert tree(tree_params(**change)) == status
    if "max_context" not in change:
        assert tree_paged(tree_params(**change)) == status


def test_tree_pointers_strides_and_workspace():
    p = tree_params()
    assert tree(p, q=None) == INVALID
    assert tree(p, q=at(1, 8)) == INVALID                      # rows not on 16 bytes
    assert tree(p, q_strides=Strides(0, 120, 128)) == INVALID
    assert tree(p, q_strides=Strides(0, -128, 128)) == INVALID
    assert tree(p, out=at(10, 4)) == INVALID
    assert tree(p, out_strides=Strides(0, 130, 128)) == INVALID
    assert tree(p, mask=at(9, 4)) == INVALID                   # 8-byte words
    assert tree(p, ks=at(5, 2)) == INVALID
    assert tree(p, ws=None) == INVALID
    assert tree(p, ws=at(11, 8)) == INVALID
    need = reef_amd.lib().reef_attention_decode_tree_workspace_bytes(p)
    assert tree(p, ws_bytes=need - 1) == INVALID
    assert tree(None) == INVALID
    assert tree_paged(p, table=None) == INVALID
    assert tree_paged(p, blocks=3) == INVALID                  # 48 tokens of 64
    assert tree_paged(p, pages=0) == INVALID
    assert tree_paged(p, pages=1 << 31) == INVALID
    assert tree_paged(p, pages=1 << 30) == UNSUPPORTED         # 2^31 pages of a head
    assert tree_paged(p, lens=None) == INVALID


def test_tree_workspace_bytes():
    """2048 counters, then two part slots a workgroup, at most two workgroups a unit (256
    without a GPU) and one for each 64-key block of an item: a tile's 16 columns of D floats and
    a (maximum, sum) for each of 64 lanes, one tile where the columns fit, otherwise two."""
    size = reef_amd.lib().reef_attention_decode_tree_workspace_bytes
    slot = {64: (64 // 8 + 1) * 64 * 8, 128: (128 // 8 + 1) * 64 * 8}
    assert size(tree_params(draft_len=4)) == 8192 + 4 * 2 * slot[128]
    assert size(tree_params(draft_len=5)) == 8192 + 4 * 2 * 2 * slot[128]
    assert size(tree_params(draft_len=4, head_dim=64, max_context=4096, batch=64)) == \
        8192 + 512 * 2 * slot[64]
    # slices of 2048 sequences: the largest counts
    assert size(tree_params(batch=2049, draft_len=1)) == 8192 + 512 * 2 * slot[128]
    for bad in (dict(head_dim=96), dict(batch=0), dict(draft_len=65)):
        assert size(tree_params(**bad)) == 0
    assert size(None) == 0
    with pytest.raises(C.ArgumentError):
        size(KvAppendParams(1, 1, 64, 1, 16))


# --- pages ------------------------------------------------------------------------------------

def test_page_table_calls():
    lib = reef_amd.lib()

    def free(sequences=at(1), n=1, table=at(2), blocks=10, lens=at(3), batch=4, refs=at(4), pages=9):
        return lib.reef_kv_free(sequences, n, table, blocks, lens, batch, refs, pages, None, None)

    def fork(parents=at(1), children=at(5), n=1, table=at(2), blocks=10, lens=at(3), batch=4,
             refs=at(4), pages=9):
        return lib.reef_kv_fork(parents, children, n, table, blocks, lens, batch, refs, pages, None,
                                None)

    for call in (free, fork):
        for bad in (dict(n=0), dict(n=-1), dict(table=None), dict(blocks=0), dict(lens=None),
                    dict(batch=0), dict(refs=None), dict(pages=0)):
            assert call(**bad) == INVALID, (call, bad)
        for big in (dict(n=65536), dict(batch=65536), dict(blocks=1 << 26), dict(pages=1 << 31)):
            assert call(**big) == UNSUPPORTED, (call, big)
    assert free(sequences=None) == INVALID
    assert fork(parents=None) == INVALID and fork(children=None) == INVALID


def test_reserve_and_compact():
    lib = reef_amd.lib()

    def reserve(new=5, blocks=10, batch=4, src=at(5), dst=at(6), ws=at(7), ws_bytes=1 << 40,
                lens=at(3), pages=9):
        return lib.reef_kv_reserve(at(2), blocks, lens, batch, new, at(4), pages, src, dst, ws,
                                   ws_bytes, None, None)

    for bad in (dict(new=0), dict(new=-3), dict(blocks=0), dict(batch=0), dict(src=None),
                dict(dst=None), dict(ws=None), dict(ws=at(7, 2)), dict(lens=None), dict(pages=0)):
        assert reserve(**bad) == INVALID, bad
    assert reserve(new=161) == CAPACITY and reserve(new=1 << 62) == CAPACITY
    assert reserve(batch=65536) == UNSUPPORTED
    assert reserve(new=1 << 29, blocks=1 << 25, batch=65535) == UNSUPPORTED
    # 5 tokens touch at most two blocks, 17 at most two, 18 three: two words an item
    size = lib.reef_kv_reserve_workspace_bytes
    assert [size(4, n) for n in (1, 2, 5, 17, 18)] == [32, 64, 64, 64, 96]
    assert size(0, 5) == 0 and size(4, 0) == 0
    assert reserve(ws_bytes=63) == INVALID

    def compact(pages=100, src=at(5), dst=at(6), ws=at(7), ws_bytes=1 << 40, batch=4, table=at(2)):
        return lib.reef_kv_compact(table, 10, batch, at(4), pages, src, dst, None, ws, ws_bytes,
                                   None, None)

    for bad in (dict(pages=0), dict(src=None), dict(dst=None), dict(ws=None), dict(ws=at(7, 2)),
                dict(batch=0), dict(table=None)):
        assert compact(**bad) == INVALID, bad
    assert compact(pages=1 << 31) == UNSUPPORTED
    size = lib.reef_kv_compact_workspace_bytes
    assert size(100) == 4 * (100 + 1 + 1) and size(4097) == 4 * (4097 + 5 + 1) and size(0) == 0
    assert compact(ws_bytes=size(100) - 1) == INVALID


def test_copy_and_keep():
    lib = reef_amd.lib()

    def copy(n=3, heads=2, D=128, pages=9, k=at(3), ks=at(5), src=at(1)):
        return lib.reef_kv_copy_pages(src, at(2), n, heads, D, k, at(4), ks, at(6), pages, None,
                                      None)

    for bad in (dict(n=0), dict(heads=0), dict(pages=0), dict(k=None), dict(k=at(3, 8)),
                dict(ks=at(5, 4)), dict(src=None)):
        assert copy(**bad) == INVALID, bad
    for big in (dict(D=96), dict(heads=65536), dict(n=1 << 31), dict(pages=1 << 31)):
        assert copy(**big) == UNSUPPORTED, big

    def keep(p, kept=at(1), lens=at(3), k=at(4), new_lens=None):
        return lib.reef_kv_keep_int8(p, kept, at(2), lens, k, at(5), at(6), at(7), new_lens, None,
                                     None)

    def keep_paged(p, table=at(8), blocks=4, pages=9):
        return lib.reef_kv_keep_int8_paged(p, at(1), at(2), at(3), table, blocks, pages, at(4),
                                           at(5), at(6), at(7), None, None, None)

    def params(**kw):
        d = dict(batch=2, kv_heads=2, head_dim=128, new_tokens=5, max_context=64)
        d.update(kw)
        return KvAppendParams(**d)

    for change, status in ((dict(batch=0), INVALID), (dict(new_tokens=0), INVALID),
                           (dict(max_context=40), INVALID), (dict(new_tokens=65), CAPACITY),
                           (dict(new_tokens=65, max_context=80), UNSUPPORTED),
                           (dict(head_dim=32), UNSUPPORTED), (dict(batch=65536), UNSUPPORTED),
                           (dict(kv_heads=65536), UNSUPPORTED)):
        assert keep(params(**change)) == status, change
        assert keep_paged(params(**change), blocks=1 << 20) == status, change
    p = params()
    assert keep(p, kept=None) == INVALID and keep(p, lens=None) == INVALID
    assert keep(p, k=at(4, 8)) == INVALID
    # every workgroup of a sequence reads its length: the new ones go elsewhere
    assert keep(p, new_lens=at(3)) == INVALID and keep(p, new_lens=at(3, 4)) == INVALID
    assert keep_paged(p, table=None) == INVALID and keep_paged(p, blocks=3) == INVALID
    assert keep_paged(p, pages=0) == INVALID and keep_paged(p, blocks=1 << 26) == INVALID


@pytest.mark.parametrize("paged", [False, True])
def test_keep_writes_no_lengths_over_what_it_reads(paged):
    """The workgroups of a sequence's other kv heads read its kept rows and their number, too."""
    lib, p = reef_amd.lib(), KvAppendParams(batch=3, kv_heads=2, head_dim=64, new_tokens=5, max_context=64)

    def keep(new_lens):
        if paged:
            return lib.reef_kv_keep_int8_paged(p, at(1), at(2), at(3), at(8), 4, 9, at(4), at(5), at(6),
                                               at(7), new_lens, None, None)
        return lib.reef_kv_keep_int8(p, at(1), at(2), at(3), at(4), at(5), at(6), at(7), new_lens, None,
                                     None)

    for n, rows in ((1, 15), (2, 3), (3, 3)):  # kept [3, 5], kept_lens [3], context_lens [3]
        for offset in (-8, 0, 4 * (rows - 1)):
            assert keep(at(n, offset)) == INVALID, (n, offset)


# --- norm, product ----------------------------------------------------------------------------

def test_norm():
    lib = reef_amd.lib()

    def norm(x=at(1), rows=4, width=16, stride=16, residual=at(2), r_stride=16, weight=at(3),
             eps=1e-6, q=at(4), scales=at(5), total=at(6), s_stride=16):
        return lib.reef_rmsnorm_quantize_int8(x, rows, width, stride, residual, r_stride, weight,
                                              eps, q, scales, total, s_stride, None, None)

    for bad in (dict(x=None), dict(q=None), dict(scales=None), dict(rows=0), dict(width=0),
                dict(stride=15), dict(r_stride=15), dict(s_stride=15), dict(residual=None),
                dict(eps=-1e-9), dict(eps=float("nan")), dict(eps=float("inf")), dict(x=at(1, 2)),
                dict(weight=at(3, 1)), dict(total=at(6, 2))):
        assert norm(**bad) == INVALID, bad
    assert norm(rows=1 << 31) == UNSUPPORTED
    wide = 1 << 30
    assert norm(width=wide, stride=wide, r_stride=wide, s_stride=wide) == UNSUPPORTED


def test_epilogue():
    lib = reef_amd.lib()

    def gemm(epilogue, out=8, y_stride=8):
        return lib.reef_gemm_w8a8_epilogue(at(1), at(2), 4, 16, at(3), at(4), None, epilogue, out,
                                           at(5), y_stride, None, None)

    def linear(epilogue, ws_bytes=1 << 20):
        return lib.reef_linear_w8a8_epilogue(at(1), 4, 16, 16, at(3), at(4), None, epilogue, 8,
                                             at(5), 8, at(6), ws_bytes, None, None)

    residual = 0x70000
    for bad in (Epilogue(None, 0, 5), Epilogue(None, 0, -1), Epilogue(None, 0, 1 << 32),
                Epilogue(residual, 7, 0), Epilogue(residual, -8, 0), Epilogue(residual, 0, 0),
                Epilogue(residual + 2, 8, 0)):
        assert gemm(bad) == INVALID and linear(bad) == INVALID, (bad.residual, bad.activation)
    assert gemm(Epilogue(None, 0, 1), y_stride=7) == INVALID
    assert linear(Epilogue(None, 0, 1), ws_bytes=79) == INVALID
    with pytest.raises(C.ArgumentError):
        gemm(Strides(0, 0, 0))


def test_wrappers_refuse_what_is_not_on_the_gpu():
    torch = pytest.importorskip("torch")
    r = reef_amd
    f, b, i = torch.zeros(4, 16), torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4).int()
    table, refs = torch.zeros(4, 4).int(), torch.zeros(9).int()
    cache = torch.zeros(4, 2, 16, 64, dtype=torch.int8)
    scales = torch.zeros(4, 2, 16)
    kv = (cache, cache.view(4, 2, 1, 64, 16), scales, scales)
    pool = (cache, cache.view(4, 2, 64, 16), scales, scales)
    q = torch.zeros(4, 8, 2, 64, dtype=torch.int8)
    for call in (lambda: r.rmsnorm_quantize(f), lambda: r.rmsnorm_quantize([1.0]),
                 lambda: r.gemm_w8a8(b, f[:, 0], b, f[:, 0]),
                 lambda: r.linear_w8a8(f, b, f[:, 0], activation="silu"),
                 lambda: r.attention_decode_tree(q, torch.zeros(4, 8, 2), *kv, i),
                 lambda: r.attention_decode_tree_paged(q, torch.zeros(4, 8, 2), *pool, table, i),
                 lambda: r.kv_free(i, table, i, refs), lambda: r.kv_fork(i, i, table, i, refs),
                 lambda: r.kv_reserve(table, i, refs, 1), lambda: r.kv_compact(table, refs),
                 lambda: r.kv_copy_pages(i, i, *pool), lambda: r.kv_keep(table, i, i, *kv),
                 lambda: r.kv_keep_paged(table, i, i, table, *pool)):
        with pytest.raises(r.InvalidArgument):
            call()
