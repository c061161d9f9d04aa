"""Refusals of the 4-bit cache's and the page selection's calls, without a GPU: the C entry points on
the host before any launch, their C++ face and the Python wrappers."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import reef_amd
from reef_amd import AttentionParams, DecodeParams, KvAppendParams, PageSelection, Strides

OK, INVALID, CAPACITY, UNSUPPORTED = (reef_amd.OK, reef_amd.INVALID_ARGUMENT, reef_amd.CAPACITY,
                                      reef_amd.UNSUPPORTED)
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def at(n=1, offset=0):
    # Non-null, 256-byte aligned host addresses: validation never dereferences them.
    return C.c_void_p(0x10000 * n + offset)


def rows(**kw):
    d = dict(batch=2, kv_heads=2, head_dim=128, new_tokens=5, max_context=64)
    d.update(kw)
    return KvAppendParams(**d)


def steps(**kw):
    d = dict(batch=2, q_heads=8, kv_heads=2, head_dim=128, max_context=64, window=0,
             softmax_scale=0.1, q_granularity=2, num_splits=0, flags=0)
    d.update(kw)
    return DecodeParams(**d)


def append(p, k=at(1), ks=None, start=at(3), table=None, blocks=0, pages=0, kc=at(4), vs=at(7)):
    return reef_amd.lib().reef_kv_append_int4(p, k, ks, at(2), None, start, table, blocks, pages, kc,
                                              at(5), at(6), vs, None, None, None)


def bounds(p, bits=8, k=at(4), ks=at(6), start=at(3), table=None, blocks=0, pages=0, out=at(8),
           scales=at(9)):
    lib = reef_amd.lib()
    f = lib.reef_kv_page_bounds_int8 if bits == 8 else lib.reef_kv_page_bounds_int4
    return f(p, start, k, ks, table, blocks, pages, out, scales, None, None)


def test_append_int4():
    for change, status in ((dict(batch=0), INVALID), (dict(new_tokens=0), INVALID),
                           (dict(max_context=40), INVALID), (dict(new_tokens=65), CAPACITY),
                           (dict(head_dim=32), UNSUPPORTED), (dict(batch=65536), UNSUPPORTED),
                           (dict(kv_heads=65536), UNSUPPORTED), (dict(max_context=1 << 30), UNSUPPORTED)):
        assert append(rows(**change)) == status, change
        assert append(rows(**change), table=at(9), blocks=1 << 20, pages=9) == status, change
    p = rows()
    for bad in (dict(k=None), dict(start=None), dict(kc=None), dict(vs=None), dict(kc=at(4, 4)),
                dict(ks=Strides(0, -1, 0)), dict(table=at(9), blocks=3, pages=9),
                dict(table=at(9), blocks=4, pages=0), dict(table=at(9), blocks=1 << 26, pages=9),
                dict(table=at(9), blocks=4, pages=1 << 31)):
        assert append(p, **bad) == INVALID, bad
    assert append(None) == INVALID


def test_unpack_and_copies():
    lib = reef_amd.lib()

    def unpack(k=at(1), v=at(2), ks=at(3), vs=at(4), pages=3, D=64, ko=at(5), vo=at(6)):
        return lib.reef_kv_unpack_int4(k, v, ks, vs, pages, D, ko, vo, None)

    for bad in (dict(pages=0), dict(D=0), dict(ko=None, vo=None), dict(k=None), dict(vs=None),
                dict(k=at(1, 8)), dict(vo=at(6, 4)), dict(ks=at(3, 2)), dict(vs=at(4, 8))):
        assert unpack(**bad) == INVALID, bad
    assert unpack(D=96) == UNSUPPORTED and unpack(pages=1 << 40) == UNSUPPORTED

    def copy(n=3, heads=2, D=128, pages=9, k=at(3), ks=at(5), src=at(1)):
        return lib.reef_kv_copy_pages_int4(src, at(2), n, heads, D, k, at(4), ks, at(6), pages, None,
                                           None)

    for bad in (dict(n=0), dict(heads=0), dict(pages=0), dict(k=None), dict(k=at(3, 8)),
                dict(ks=at(5, 4)), dict(src=None)):
        assert copy(**bad) == INVALID, bad
    for big in (dict(D=96), dict(heads=65536), dict(n=1 << 31), dict(pages=1 << 31)):
        assert copy(**big) == UNSUPPORTED, big


def decode(p, bits=4, k=at(3), ks=at(5), table=None, blocks=0, pages=0, lens=at(7), selection=None,
           out=at(8), ws=at(9), ws_bytes=1 << 40):
    lib = reef_amd.lib()
    f = lib.reef_attention_decode_int4 if bits == 4 else lib.reef_attention_decode_int8_selected
    return f(p, at(1), at(2), k, at(4), ks, at(6), table, blocks, pages, lens, selection, out, ws,
             ws_bytes, None, None)


@pytest.mark.parametrize("bits", [4, 8])
def test_decode(bits):
    chosen = PageSelection(at(10).value, at(11).value, 4)
    need = reef_amd.lib().reef_attention_decode_workspace_bytes(steps())
    for change, status in ((dict(batch=0), INVALID), (dict(q_heads=3), INVALID),
                           (dict(max_context=60), INVALID), (dict(window=-1), INVALID),
                           (dict(q_granularity=3), INVALID), (dict(softmax_scale=float("nan")), INVALID),
                           (dict(head_dim=96), UNSUPPORTED), (dict(q_heads=34), UNSUPPORTED),
                           (dict(max_context=1 << 30), UNSUPPORTED)):
        assert decode(steps(**change), bits, selection=chosen) == status, change
    p = steps()
    for bad in (dict(k=None), dict(k=at(3, 8)), dict(ks=at(5, 4)), dict(out=at(8, 8)), dict(ws=None),
                dict(ws=at(9, 8)), dict(ws_bytes=need - 1), dict(lens=None),
                dict(table=at(12), blocks=3, pages=9), dict(table=at(12), blocks=4, pages=0),
                dict(table=at(12), blocks=4, pages=1 << 31), dict(table=at(12), blocks=4, pages=9, lens=None)):
        assert decode(p, bits, **{"selection": chosen, **bad}) == INVALID, bad
    for bad in (PageSelection(None, at(11).value, 4), PageSelection(at(10).value, None, 4),
                PageSelection(at(10).value, at(11).value, 0), PageSelection(at(10, 2).value, at(11).value, 4)):
        assert decode(p, bits, selection=bad) == INVALID
    assert decode(p, bits, selection=PageSelection(at(10).value, at(11).value, 1 << 26)) == UNSUPPORTED
    if bits == 8:  # the whole int8 cache is reef_attention_decode_int8's
        assert decode(p, 8) == INVALID


def test_prefill_over_the_cache():
    lib = reef_amd.lib()

    def chunk(ws_bytes=1 << 40, tokens=64, table=None, blocks=0, pages=0, k=at(3), q=at(1), out=at(7),
              q_strides=None, out_strides=None, **kw):
        d = dict(batch=2, q_heads=8, kv_heads=2, q_len=8, kv_len=40, head_dim=128, query_start=32,
                 window=0, softmax_scale=0.1, q_granularity=1, kv_granularity=2, flags=0)
        d.update(kw)
        return lib.reef_attention_prefill_int4_cache(
            AttentionParams(**d), q, q_strides, at(2), k, at(4), at(5), at(6), tokens, table, blocks, pages,
            out, out_strides, at(8), ws_bytes, None, None)

    for bad in (dict(kv_granularity=1), dict(query_start=33), dict(tokens=32), dict(tokens=72),
                dict(ws_bytes=1000), dict(k=None), dict(k=at(3, 8)), dict(q_heads=3),
                dict(table=at(9), blocks=2, pages=9), dict(table=at(9), blocks=3, pages=0),
                dict(window=-1), dict(softmax_scale=0.0), dict(softmax_scale=float("nan")),
                dict(q_granularity=3), dict(q=at(1, 8)), dict(out=at(7, 4)),
                dict(q_strides=Strides(0, 120, 128)), dict(q_strides=Strides(0, -128, 128)),
                dict(out_strides=Strides(0, 130, 128)), dict(out_strides=Strides(0, 128, -4))):
        assert chunk(**bad) == INVALID, bad
    assert chunk(head_dim=96) == UNSUPPORTED and chunk(window=1 << 30) == UNSUPPORTED


def test_the_widest_window():
    """The widest 64-bit window is refused like others past 2^30, on the way of a short chunk too."""
    for q_len in (1, 8):
        p = AttentionParams(batch=2, q_heads=8, kv_heads=2, q_len=q_len, kv_len=4096, head_dim=128,
                            query_start=4096 - q_len, window=(1 << 63) - 1, softmax_scale=0.1,
                            q_granularity=1, kv_granularity=2, flags=0)
        assert reef_amd.lib().reef_attention_prefill_int4_cache(
            p, at(1), None, at(2), at(3), at(4), at(5), at(6), 4096, None, 0, 0, at(7), None, at(8),
            1 << 40, None, None) == UNSUPPORTED


@pytest.mark.parametrize("bits", [4, 8])
def test_bounds(bits):
    for change, status in ((dict(batch=0), INVALID), (dict(new_tokens=0), INVALID),
                           (dict(max_context=40), INVALID), (dict(new_tokens=65), CAPACITY),
                           (dict(head_dim=96), UNSUPPORTED), (dict(batch=65536), UNSUPPORTED),
                           (dict(kv_heads=65536), UNSUPPORTED), (dict(max_context=1 << 30), UNSUPPORTED)):
        assert bounds(rows(**change), bits) == status, change
    p = rows()
    for bad in (dict(k=None), dict(ks=None), dict(start=None), dict(out=None), dict(scales=None),
                dict(k=at(4, 8)), dict(out=at(8, 8)), dict(scales=at(9, 2)),
                dict(table=at(10), blocks=3, pages=9), dict(table=at(10), blocks=4, pages=0),
                dict(table=at(10), blocks=1 << 26, pages=9)):
        assert bounds(p, bits, **bad) == INVALID, bad
    assert bounds(None, bits) == INVALID


def test_selection():
    lib = reef_amd.lib()
    size = lib.reef_kv_select_pages_workspace_bytes

    def select(p, q=at(1), b=at(3), bs=at(4), table=None, blocks=0, pages=0, lens=at(5), budget=3,
               sinks=1, recent=1, out=at(6), counts=at(7), ws=at(8), ws_bytes=1 << 40):
        return lib.reef_kv_select_pages(p, q, at(2), b, bs, table, blocks, pages, lens, budget, sinks,
                                        recent, out, counts, ws, ws_bytes, None, None)

    assert size(steps()) == 2 * 2 * 4 * 4  # a word a page, sequence and kv head
    assert size(steps(batch=65535, kv_heads=1)) == 65535 * 4 * 4
    for bad in (dict(batch=0), dict(max_context=60), dict(q_heads=3), dict(batch=65536, kv_heads=1),
                dict(max_context=1 << 30)):
        assert size(steps(**bad)) == 0, bad
    assert size(None) == 0
    for change, status in ((dict(batch=0), INVALID), (dict(q_heads=3), INVALID),
                           (dict(max_context=60), INVALID), (dict(q_granularity=3), INVALID),
                           (dict(head_dim=96), UNSUPPORTED), (dict(q_heads=34), UNSUPPORTED),
                           (dict(batch=32768), UNSUPPORTED), (dict(max_context=1 << 30), UNSUPPORTED)):
        assert select(steps(**change)) == status, change
    p = steps()
    for bad in (dict(q=None), dict(b=None), dict(bs=None), dict(lens=None), dict(out=None),
                dict(counts=None), dict(ws=None), dict(q=at(1, 8)), dict(b=at(3, 8)), dict(ws=at(8, 8)),
                dict(ws_bytes=63), dict(budget=0), dict(sinks=-1), dict(recent=0), dict(sinks=2, recent=2),
                dict(sinks=(1 << 63) - 1), dict(table=at(9), blocks=3, pages=9),
                dict(table=at(9), blocks=4, pages=0)):
        assert select(p, **bad) == INVALID, bad
    assert select(p, budget=1 << 26) == UNSUPPORTED


def test_wrappers_refuse_what_is_not_on_the_gpu():
    torch = pytest.importorskip("torch")
    r = reef_amd
    q, qs, i = torch.zeros(4, 8, 64, dtype=torch.int8), torch.zeros(4, 8), torch.zeros(4).int()
    new = torch.zeros(4, 2, 1, 64)
    b = dict(dtype=torch.uint8)
    cache4 = (torch.zeros(4, 2, 16, 32, **b), torch.zeros(4, 2, 1, 64, 8, **b), torch.zeros(4, 2, 16),
              torch.zeros(4, 2, 16))
    cache8 = (torch.zeros(4, 2, 16, 64).char(), torch.zeros(4, 2, 1, 64, 16).char(), *cache4[2:])
    bounds_ = torch.zeros(4, 2, 1, 2, 64).char(), torch.zeros(4, 2, 1)
    chosen = torch.zeros(4, 2, 1).int(), torch.zeros(4, 2).int()
    for call in (lambda: r.kv_append_int4(new, new, i, *cache4), lambda: r.kv_unpack_int4(*cache4),
                 lambda: r.kv_copy_pages_int4(i, i, *cache4),
                 lambda: r.attention_decode_int4(q, qs, *cache4, i),
                 lambda: r.attention_decode_int4(q, qs, [1], *cache4[1:], i),
                 lambda: r.attention_decode_selected(q, qs, *cache8, i, selected=chosen),
                 lambda: r.attention_decode_selected(q, qs, *cache8, i, selected=None),
                 lambda: r.attention_prefill_cache_int4(q[:, :, None], qs, *cache4, 16),
                 lambda: r.kv_page_bounds(i, 1, cache8[0], cache8[2], *bounds_),
                 lambda: r.kv_select_pages(q, qs, *bounds_, i, 1)):
        with pytest.raises(r.InvalidArgument):
            call()


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_cxx_wrappers_throw(tmp_path):
    reef_amd.lib()  # the library must be built
    exe = tmp_path / "kv_reads_check"
    libdir = os.path.dirname(reef_amd.LIB_PATH)
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__",
           "-I", os.path.join(ROOT, "include"), "-isystem", "/opt/rocm/include",
           os.path.join(ROOT, "tests", "cxx", "kv_reads_check.cpp"),
           "-L", libdir, "-lreef_hip", f"-Wl,-rpath,{libdir}", "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    print(r.stdout)
    assert r.returncode == 0, r.stdout + r.stderr
