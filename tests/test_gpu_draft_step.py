"""A layer's steps over trees of drafted tokens, from the residual stream back to it: norm,
QKV product, room in the page pool, append, attention of the trees, output product with the
residual, norm, the MLP's products, and the accepted tokens kept; between steps a sequence
ends, another is forked onto its place, and the pool is compacted.

Every operator is held to its formula in 64 bits on the inputs it was given (the int8 codes
between them are the device's own: a code at a half would come out either way). The cache is
held, byte for byte, to a plain list of each sequence's rows.

Tolerances, u = 2^-24. The products: float(sum) exact below 2^24, three roundings, and bias
and residual one each; the activation's own as its formula has them (v rounded three times:
u (|x| + 4 |y|)), its slope at most 1.13. The norm's code: half a step, and 1e-4 for the
scale's rounding (127 u / 2 and the 64-bit steps). Attention: an exponent of X log2 units
rounded four times, exp2, the weight's two parts and its fp16 floor, twice, and 14 u for the
merges and the quotient."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

PAGE, U = 16, 2.0 ** -24


@pytest.fixture(scope="module")
def reef():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import reef_amd
    reef_amd.lib()
    return reef_amd


class Layer:
    def __init__(self, seed, W, F, Hq, H, D):
        self.W, self.F, self.Hq, self.H, self.D = W, F, Hq, H, D
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(out, fin):
            return (torch.randint(-127, 128, (out, fin), generator=g, device="cuda").to(torch.int8),
                    (0.5 + torch.rand(out, generator=g, device="cuda")) / (73 * math.sqrt(fin)),
                    0.1 * torch.randn(out, generator=g, device="cuda"))

        self.qkv, self.o = weight((Hq + 2 * H) * D, W), weight(W, Hq * D)
        self.up, self.down = weight(F, W), weight(W, F)
        self.norms = [0.5 + torch.rand(W, generator=g, device="cuda") for _ in range(2)]


class Cache:
    """A page pool with its table; lens count the kept tokens."""

    def __init__(self, layer, batch, blocks, pages):
        H, D = layer.H, layer.D
        z = lambda dtype, *s: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
        self.pool = [z(torch.int8, pages, H, PAGE, D), z(torch.int8, pages, H, D, PAGE),
                     z(torch.float32, pages, H, PAGE), z(torch.float32, pages, H, PAGE)]
        for s in self.pool[2:]:
            s.fill_(float("nan"))
        self.table = torch.full((batch, blocks), -1, dtype=torch.int32, device="cuda")
        self.lens, self.refs = z(torch.int32, batch), z(torch.int32, pages)

    def tensors(self):
        return [*self.pool, self.table, self.lens, self.refs]

    def clone(self):
        other = object.__new__(Cache)
        other.pool = [t.clone() for t in self.pool]
        other.table, other.lens, other.refs = (t.clone() for t in (self.table, self.lens, self.refs))
        return other


def step(reef, layer, cache, x, mask, kept, kept_lens, status, seen=None):
    """One step in place on the residual stream x [B * T, W] and the cache. seen: a dict that
    takes what every operator was given and gave."""
    B, T = mask.shape
    Hq, H, D = layer.Hq, layer.H, layer.D
    note = (lambda **kw: None) if seen is None else seen.update

    def project(rows, w, **kw):
        return reef.gemm_w8a8(*rows, w[0], w[1], w[2], status, **kw)

    rows = reef.rmsnorm_quantize(x, layer.norms[0], status=status)
    note(x0=x.clone(), norm0=rows)
    qkv = project(rows, layer.qkv)
    note(qkv=qkv)
    heads = qkv.view(B, T, Hq + 2 * H, D).transpose(1, 2)
    q, k, v = heads[:, :Hq], heads[:, Hq:Hq + H], heads[:, Hq + H:]
    src, dst = reef.kv_reserve(cache.table, cache.lens, cache.refs, T, status=status)
    reef.kv_copy_pages(src, dst, *cache.pool, status=status)
    reef.kv_append_paged(k, v, cache.lens, cache.table, *cache.pool, status=status)
    qq, qs = reef.quantize_rows(q, status)
    note(k=k, v=v, q=(qq, qs))
    lens = cache.lens + T
    o = torch.empty((B, T, Hq, D), dtype=torch.float32, device="cuda")
    reef.attention_decode_tree_paged(qq, qs, *cache.pool, cache.table, lens, tree_mask=mask,
                                     status=status, out=o.transpose(1, 2))
    rows = reef.quantize_rows(o.view(B * T, Hq * D), status)
    project(rows, layer.o, residual=x, out=x)
    note(o=o, o_rows=rows, x1=x.clone())
    rows = reef.rmsnorm_quantize(x, layer.norms[1], status=status)
    y = project(rows, layer.up, activation="gelu_tanh")
    note(norm1=rows, y=y)
    x.copy_(reef.linear_w8a8(y, layer.down[0], layer.down[1], layer.down[2], status, residual=x))
    note(x2=x.clone(), y_rows=reef.quantize_rows(y, status))
    cache.lens.copy_(reef.kv_keep_paged(kept, kept_lens, lens, cache.table, *cache.pool,
                                        status=status))


def f64(t):
    return t.cpu().numpy().astype(np.float64)


def check_product(rows, w, y, residual=None, gelu=False):
    total = f64(rows[0]) @ f64(w[0]).T
    product = total * f64(rows[1])[:, None] * f64(w[1])
    ref = product + f64(w[2])
    tol = U * (3 * np.abs(product) + np.abs(ref))
    if gelu:
        d = ref
        ref = d / (1 + np.exp(-2 * math.sqrt(2 / math.pi) * (d + 0.044715 * d ** 3)))
        tol = 1.13 * tol + U * (np.abs(d) + 4 * np.abs(ref))
    if residual is not None:
        ref = ref + f64(residual)
        tol = tol + U * np.abs(ref)
    assert (np.abs(f64(y) - ref) <= tol * (1 + 1e-6)).all()


def check_norm(x, weight, rows):
    d = f64(x)
    y = d * f64(weight) / np.sqrt((d * d).mean(1, keepdims=True) + 1e-6)
    q, s = f64(rows[0]), f64(rows[1])[:, None]
    assert (np.abs(np.abs(y).max(1, keepdims=True) / 127 - s) <= U * s * (1 + 1e-6)).all()
    assert (np.abs(y / s - q) <= 0.5 + 1e-4).all()


def check_attention(layer, past, new, q, seen, o):
    """past: per sequence (k, v) codes and scales as float64 [H, n, D] products; new the same
    for the drafted tokens; o [B, T, Hq, D]."""
    qd = f64(q[0]) * f64(q[1])[..., None]
    B, Hq, T, D = qd.shape
    G = Hq // layer.H
    o = f64(o)
    for b in range(B):
        for h in range(Hq):
            k, v = (np.concatenate([past[b][i][h // G], new[b][i][h // G]]) for i in (0, 1))
            P = len(k) - T
            s = qd[b, h] @ k.T / math.sqrt(D)
            X = np.abs(s).max() / math.log(2)
            vis = np.concatenate([np.ones((T, P), bool), seen[b]], 1)
            s = np.where(vis, s, -np.inf)
            some = vis.any(1) & seen[b].any(1)
            ref = np.zeros((T, D))
            p = np.exp(s[some] - s[some].max(1, keepdims=True))
            ref[some] = p @ v / p.sum(1, keepdims=True)
            tol = np.abs(v).max() * (2 * (2.8 * X * U + 6 * U + len(k) * 2.0 ** -33) + 14 * U)
            assert np.abs(o[b, :, h] - ref).max() <= tol


def cached(cache, layer):
    """Every sequence's kept rows in the pool, as float64 [H, n, D]: (k, v) each."""
    k, v, ks, vs = (f64(t) for t in cache.pool)
    table, lens = cache.table.cpu().numpy(), cache.lens.cpu().numpy()
    out = []
    for b, n in enumerate(lens):
        pages = table[b, :-(-n // PAGE)]
        assert (pages >= 0).all()
        kk = (k * ks[..., None])[pages].transpose(1, 0, 2, 3).reshape(layer.H, -1, layer.D)
        vv = (v.transpose(0, 1, 3, 2) * vs[..., None])[pages].transpose(1, 0, 2, 3)
        out.append((kk[:, :n], vv.reshape(layer.H, -1, layer.D)[:, :n]))
    return out


def trees(rng, B, T):
    """(bool [B, T, T], accepted rows [B, T], their numbers): a random tree a sequence, the
    last ones with fewer tokens, and a path of each."""
    m = np.zeros((B, T, T), bool)
    kept, n = np.zeros((B, T), np.int32), np.zeros(B, np.int32)
    for b in range(B):
        count = T if b % 3 else int(rng.integers(1, T + 1))
        for i in range(count):
            p = int(rng.integers(-1, i))
            if p >= 0:
                m[b, i] = m[b, p]
            m[b, i, i] = True
        path = np.flatnonzero(m[b, int(rng.integers(0, count))])
        kept[b, :len(path)], n[b] = path, len(path)
    return m, kept, n


def on_gpu(m, kept, n):
    w = (m.astype(np.uint64) << np.arange(m.shape[2], dtype=np.uint64)).sum(2, dtype=np.uint64)
    return tuple(torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (w.view(np.int64), kept, n))


SHAPES = [(5, 7, 256, 512, 4, 2, 64), (3, 33, 512, 768, 8, 1, 128), (4, 1, 384, 400, 3, 3, 128)]


@pytest.mark.parametrize("B,T,W,F,Hq,H,D", SHAPES)
def test_steps_over_drafted_tokens(reef, B, T, W, F, Hq, H, D):
    rng = np.random.default_rng(T)
    layer, cache = Layer(T, W, F, Hq, H, D), None
    cache = Cache(layer, B, 12, 12 * B)
    status = reef.StatusWord()
    rows = [(np.zeros((H, 0, D)), np.zeros((H, 0, D))) for _ in range(B)]
    for i in range(4):
        print(f"\n[case] step {i}: {B} x {T} tokens, width {W}, {Hq}/{H} heads of {D}", flush=True)
        m, kept, n = trees(rng, B, T)
        x = torch.from_numpy(rng.standard_normal((B * T, W)).astype(np.float32)).cuda()
        seen = {}
        step(reef, layer, cache, x, *on_gpu(m, kept, n), status, seen)
        status.check("step")
        check_norm(seen["x0"], layer.norms[0], seen["norm0"])
        check_product(seen["norm0"], layer.qkv, seen["qkv"])
        new = []
        for name in ("k", "v"):
            codes, scales = reef.quantize_rows(seen[name].contiguous())
            new.append(f64(codes) * f64(scales)[..., None])
        new = [(new[0][b], new[1][b]) for b in range(B)]
        check_attention(layer, rows, new, seen["q"], m, seen["o"])
        check_product(seen["o_rows"], layer.o, seen["x1"], residual=seen["x0"])
        check_norm(seen["x1"], layer.norms[1], seen["norm1"])
        check_product(seen["norm1"], layer.up, seen["y"], gelu=True)
        check_product(seen["y_rows"], layer.down, seen["x2"], residual=seen["x1"])
        rows = [tuple(np.concatenate([rows[b][j], new[b][j][:, kept[b, :n[b]]]], 1) for j in (0, 1))
                for b in range(B)]
        # a sequence ends and another is forked onto its place; then the pool is compacted
        ends, parent = int(rng.integers(0, B)), int(rng.integers(0, B - 1))
        parent += parent >= ends
        ids = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        reef.kv_free(ids(ends), cache.table, cache.lens, cache.refs, status)
        reef.kv_fork(ids(parent), ids(ends), cache.table, cache.lens, cache.refs, status)
        rows[ends] = rows[parent]
        if i % 2:
            src, dst, live = reef.kv_compact(cache.table, cache.refs, status)
            reef.kv_copy_pages(src, dst, *cache.pool, status=status)
            assert int(live) == int((cache.refs > 0).sum()) == int((cache.refs[:int(live)] > 0).sum())
        status.check("pages")
        for (k, v), (gk, gv) in zip(rows, cached(cache, layer)):
            assert np.array_equal(k, gk) and np.array_equal(v, gv)


def test_captured_steps(reef):
    """The whole step in a graph, replayed with new inputs between the program's own eager
    steps on a twin: the same bytes."""
    print("\n[case] a captured step", flush=True)
    B, T, W, F, Hq, H, D = 4, 9, 256, 512, 8, 2, 64
    rng = np.random.default_rng(99)
    layer = Layer(5, W, F, Hq, H, D)
    twin = Cache(layer, B, 12, 80)
    status = reef.StatusWord()
    m, kept, n = trees(rng, B, T)
    ins = [t.clone() for t in on_gpu(m, kept, n)]
    x = torch.zeros((B * T, W), device="cuda")
    spare = twin.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(reef, layer, spare, x.normal_(), *ins, status)
    torch.cuda.current_stream().wait_stream(side)
    captured = twin.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(reef, layer, captured, x, *ins, status)
    for _ in range(4):
        for t, new in zip(ins, on_gpu(*trees(rng, B, T))):
            t.copy_(new)
        fresh = torch.from_numpy(rng.standard_normal((B * T, W)).astype(np.float32)).cuda()
        x.copy_(fresh)
        graph.replay()
        step(reef, layer, twin, fresh, *ins, status)
        torch.cuda.synchronize()
        assert torch.equal(x, fresh)
        for a, b in zip(captured.tensors(), twin.tensors()):
            assert torch.equal(a.view(torch.int8) if a.is_floating_point() else a,
                               b.view(torch.int8) if b.is_floating_point() else b)
    status.check("graph")
