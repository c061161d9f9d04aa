"""Captured chunks over the int8 cache beside eager ones over either cache, which share their
stream's workspace."""
import numpy as np
import pytest

from kv_reads import Cache

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def reef():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import reef_amd
    reef_amd.lib()
    return reef_amd


@pytest.mark.parametrize("D,T,n", [(128, 40, 300), (64, 130, 1021)])
def test_a_captured_chunk_holds_its_workspace(reef, monkeypatch, D, T, n):
    """The stream's workspace may be replaced by a larger one, of the 4-bit cache's chunks too: a graph
    takes one of its own. Its replays are the eager call, with such calls between them."""
    rng = np.random.default_rng(T)
    eight = Cache(rng, 8, 2, 2, D, -(-n // 16) * 16, [n] * 2, True)
    four = Cache(rng, 4, 2, 2, D, 2064, [2050] * 2, True)
    q = torch.zeros((2, 8, T, D), dtype=torch.int8, device="cuda")
    rows = torch.from_numpy(rng.integers(-127, 128, (2, 8, 40, D)).astype(np.int8)).cuda()
    qs = torch.rand(8, device="cuda") * 0.01 + 0.01
    word = reef.StatusWord("cuda")
    used = []
    plain = reef._lib()

    class Library:
        def __getattr__(self, name):
            return getattr(plain, name)

        def reef_attention_prefill_int8_cache(self, *args):
            used.append(args[-4])
            return plain.reef_attention_prefill_int8_cache(*args)

    monkeypatch.setattr(reef, "_lib", lambda: library)
    library = Library()

    def call():
        return reef.attention_prefill_cache(q, qs, *eight.tensors, n, status=word,
                                            block_table=eight.block_table)

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            held = call()
        eager, captured = used
        assert eager != captured
        for _ in range(4):
            q.copy_(torch.randint(-127, 128, q.shape, device="cuda", dtype=torch.int8))
            want = call().clone()
            reef.attention_prefill_cache_int4(rows, qs, *four.tensors, 2050, status=word,
                                              block_table=four.block_table)
            graph.replay()
            stream.synchronize()
            assert torch.equal(held, want)
    torch.cuda.current_stream().wait_stream(stream)
    word.check("chunks")
