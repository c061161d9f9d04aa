"""What the 4-bit cache's and the page selection's wrappers make of their arguments: missing ones are
refused by name, as every other call of the library refuses them, and sizes that are kept are those of
the device."""
import os
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")

import reef_amd as r


def calls(device):
    """(name, call, required tensors, other arguments) of every wrapper."""
    def ints(*shape):
        return torch.zeros(shape, dtype=torch.int32, device=device)

    f32 = dict(device=device)
    new = torch.zeros(2, 2, 1, 64, **f32)
    four = [torch.zeros(2, 2, 16, 32, dtype=torch.uint8, **f32),
            torch.zeros(2, 2, 1, 64, 8, dtype=torch.uint8, **f32)]
    eight = [torch.zeros(2, 2, 16, 64, dtype=torch.int8, **f32),
             torch.zeros(2, 2, 1, 64, 16, dtype=torch.int8, **f32)]
    scales = [torch.ones(2, 2, 16, **f32), torch.ones(2, 2, 16, **f32)]
    q, qs = torch.zeros(2, 4, 64, dtype=torch.int8, **f32), torch.ones(2, 4, **f32)
    bounds = [torch.zeros(2, 2, 1, 2, 64, dtype=torch.int8, **f32), torch.ones(2, 2, 1, **f32)]

    def selected(call):
        return lambda *t: call(*t[:-2], selected=t[-2:])

    return [
        ("append", r.kv_append_int4, [new, new, ints(2), *four, *scales]),
        ("unpack", r.kv_unpack_int4, [*four, *scales]),
        ("copy", r.kv_copy_pages_int4, [ints(1), ints(1), *four, *scales]),
        ("decode", r.attention_decode_int4, [q, qs, *four, *scales]),
        ("decode listed", selected(r.attention_decode_int4),
         [q, qs, *four, *scales, ints(2), ints(2, 2, 1), ints(2, 2)]),
        ("decode selected", selected(r.attention_decode_selected),
         [q, qs, *eight, *scales, ints(2), ints(2, 2, 1), ints(2, 2)]),
        ("chunk", lambda *t: r.attention_prefill_cache_int4(*t, 16, q_granularity=r.PER_TENSOR),
         [q[:, :, None], torch.ones(1, **f32), *four, *scales]),
        ("bounds", lambda start, *t: r.kv_page_bounds(start, 1, *t),
         [ints(2), eight[0], scales[0], *bounds]),
        ("bounds of 4 bits", lambda start, *t: r.kv_page_bounds(start, 1, *t),
         [ints(2), four[0], scales[0], *bounds]),
        ("select", lambda *t: r.kv_select_pages(*t, 1), [q, qs, *bounds, ints(2)]),
    ]


@pytest.mark.parametrize("i", range(10))
def test_nothing_but_none(i):
    name, call, tensors = calls("cpu")[i]
    with pytest.raises(r.InvalidArgument):
        call(*[None] * len(tensors))


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(10))
def test_each_tensor_missing(i):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    name, call, tensors = calls("cuda")[i]
    for at in range(len(tensors)):
        with pytest.raises(r.InvalidArgument):
            call(*tensors[:at], None, *tensors[at + 1:])


def test_workspace_bytes_are_the_devices(monkeypatch):
    """A size that is kept from one device is not another's, which may have more compute units."""
    class Library:
        current = 0

        def reef_attention_decode_workspace_bytes(self, p):
            return (1000, 4000)[self.current]

    lib = Library()
    monkeypatch.setattr(r, "_lib", lambda: lib)
    monkeypatch.setattr(r, "_DECODE_BYTES", {})
    sizes = b"the packed sizes of a call"
    for _ in range(2):
        for lib.current in (0, 1):
            assert r._decode_workspace_bytes(sizes, lib.current) == (1000, 4000)[lib.current]


@pytest.mark.parametrize("bits", [4, 8])
def test_bounds_up_to_lengths_refuses(bits):
    """The refusals of the call without lengths, and of lengths that are not there."""
    def at(n, offset=0):  # host addresses: validation never dereferences them
        return 0x10000 * n + offset

    lib = r.lib()
    f = lib.reef_kv_page_bounds_int4_ragged if bits == 4 else lib.reef_kv_page_bounds_int8_ragged

    def call(lens=at(2), k=at(3), out=at(5), table=None, blocks=0, pages=0, **kw):
        sizes = dict(batch=2, kv_heads=2, head_dim=128, new_tokens=5, max_context=64)
        return f(r.KvAppendParams(**{**sizes, **kw}), at(1), lens, k, at(4), table, blocks, pages, out,
                 at(6), None, None)

    for bad in (dict(lens=None), dict(k=None), dict(k=at(3, 8)), dict(out=None), dict(batch=0),
                dict(new_tokens=0), dict(max_context=40), dict(table=at(7), blocks=3, pages=9),
                dict(table=at(7), blocks=4, pages=0)):
        assert call(**bad) == r.INVALID_ARGUMENT, bad
    assert call(new_tokens=65) == r.CAPACITY
    assert call(head_dim=96) == r.UNSUPPORTED and call(batch=65536) == r.UNSUPPORTED


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_bounds_up_to_lengths_in_cxx(tmp_path):
    r.lib()  # the library must be built
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe, libdir = tmp_path / "kv_bounds_check", os.path.dirname(r.LIB_PATH)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__",
                    "-I", os.path.join(root, "include"), "-isystem", "/opt/rocm/include",
                    os.path.join(root, "tests", "cxx", "kv_bounds_check.cpp"), "-L", libdir, "-lreef_hip",
                    f"-Wl,-rpath,{libdir}", "-o", str(exe)], check=True, capture_output=True, text=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout + done.stderr
