"""Attention of drafted tokens over the int8 cache against the formula in 64 bits.

Tolerance, relative to the largest |value| of the cache, u = 2^-24: an exponent of X log2
units is rounded four times (key scale, query scale with the softmax scale, log2 e, the
difference), which moves a weight by 4 ln2 X u; exp2 adds 2 u, a weight's hi + lo parts 4 u,
and a weight below 2^-14 in fp16 at most 2^-25 of units of 2^-8: 2^-33 a key. Numerator and
row sum can both be off by that, so twice: 2 (2.8 X u + 6 u + keys 2^-33), and u for each
of the roundings of up to 6 merges and the quotient: 14 u."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

PAGE = 16
U = 2.0 ** -24


@pytest.fixture(scope="module")
def reef():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import reef_amd
    reef_amd.lib()
    return reef_amd


def tree_masks(rng, B, T, kind):
    """bool [B, T, T]: what each drafted token sees of the drafted ones."""
    m = np.zeros((B, T, T), bool)
    for b in range(B):
        n = T if kind != "padded" else int(rng.integers(0, T + 1))
        for i in range(n):
            p = i - 1 if kind == "chain" else int(rng.integers(-1, i))
            if p >= 0:
                m[b, i] = m[b, p]
            m[b, i, i] = True
        if kind == "any":  # whatever a caller sets
            m[b] = rng.random((T, T)) < 0.4
            m[b, rng.integers(0, T)] = False
    return m


def words(m):
    w = (m.astype(np.uint64) << np.arange(m.shape[2], dtype=np.uint64)).sum(2, dtype=np.uint64)
    return torch.from_numpy(w.view(np.int64)).cuda()


def problem(rng, B, Hq, H, D, T, lens, L):
    q = rng.integers(-127, 128, (B, Hq, T, D)).astype(np.int8)
    k = rng.integers(-127, 128, (B, H, L, D)).astype(np.int8)
    v = rng.integers(-127, 128, (B, H, L, D)).astype(np.int8)
    qs = rng.uniform(0.005, 0.02, (B, Hq, T)).astype(np.float32)
    ks, vs = (rng.uniform(0.005, 0.03, (B, H, L)).astype(np.float32) for _ in range(2))
    return q, k, v, qs, ks, vs


def reference(q, k, v, qs, ks, vs, lens, m, window, scale):
    """(out, tolerance) in 64 bits; rows that see nothing are zeros."""
    B, Hq, T, D = q.shape
    G = Hq // k.shape[1]
    out = np.zeros((B, Hq, T, D))
    most, X = 0.0, 0.0
    for b in range(B):
        n = int(lens[b])
        P = n - T
        depth = m[b].sum(1) - 1
        pos = np.concatenate([np.arange(P), P + depth])
        seen = np.concatenate([np.ones((T, P), bool), m[b]], 1)
        if window:
            seen &= pos[None, :] > (P + depth)[:, None] - window
        seen[m[b].sum(1) == 0] = False
        some = seen.any(1)
        for h in range(Hq):
            kk, vv = (x[b, h // G, :n].astype(np.float64) * s[b, h // G, :n, None]
                      for x, s in ((k, ks), (v, vs)))
            s = (q[b, h] * qs[b, h][:, None].astype(np.float64)) @ kk.T * scale
            X = max(X, np.abs(s).max() / math.log(2))
            s = np.where(seen, s, -np.inf)[some]
            p = np.exp(s - s.max(1, keepdims=True))
            out[b, h, some] = p @ vv / p.sum(1, keepdims=True)
            most = max(most, np.abs(vv).max())
    return out, most * (2 * (2.8 * X * U + 6 * U + max(lens) * 2.0 ** -33) + 14 * U)


def gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def contiguous(k, v, ks, vs):
    B, H, L, D = k.shape
    vp = v.reshape(B, H, L // PAGE, PAGE, D).transpose(0, 1, 2, 4, 3)
    return [gpu(k), gpu(vp), gpu(ks), gpu(vs)]


def paged(rng, k, v, ks, vs, lens):
    """The same cache in scattered pages; entries of blocks past a sequence's end are -1."""
    B, H, L, D = k.shape
    n = L // PAGE
    P = B * n + 5
    order = rng.permutation(P)[:B * n].reshape(B, n)
    kp = rng.integers(-127, 128, (P, H, PAGE, D)).astype(np.int8)
    vp = rng.integers(-127, 128, (P, H, D, PAGE)).astype(np.int8)
    ksp, vsp = (np.full((P, H, PAGE), np.nan, np.float32) for _ in range(2))
    for b in range(B):
        for i in range(n):
            at = slice(i * PAGE, (i + 1) * PAGE)
            kp[order[b, i]], vp[order[b, i]] = k[b, :, at], v[b, :, at].transpose(0, 2, 1)
            ksp[order[b, i]], vsp[order[b, i]] = ks[b, :, at], vs[b, :, at]
    table = np.where(np.arange(n)[None, :] * PAGE < np.asarray(lens)[:, None], order, -1)
    return [gpu(kp), gpu(vp), gpu(ksp), gpu(vsp)], gpu(table.astype(np.int32))


def poison(k, v, ks, vs, lens):
    """What lies behind a sequence's last token is anything: scales NaN and infinite."""
    ks, vs = ks.copy(), vs.copy()
    for b, n in enumerate(lens):
        ks[b, :, n:] = np.nan
        vs[b, :, n:] = np.inf
    return k, v, ks, vs


CASES = [
    # B, Hq, Hkv, D, T, lens, window, masks
    (1, 1, 1, 64, 1, [1], 0, "chain"),
    (1, 1, 1, 128, 1, [17], 0, "chain"),
    (2, 12, 12, 64, 8, [200, 8], 0, "tree"),
    (3, 8, 2, 128, 7, [1000, 63, 64], 0, "tree"),
    (2, 32, 8, 128, 3, [700, 450], 0, "chain"),
    (3, 10, 2, 64, 13, [129, 65, 500], 0, "padded"),
    (2, 8, 1, 128, 64, [900, 64], 0, "tree"),
    (1, 16, 1, 64, 64, [333], 0, "tree"),
    (2, 5, 1, 128, 33, [80, 41], 0, "any"),
    (2, 33, 1, 64, 31, [222, 31], 0, "padded"),
    (4, 4, 4, 128, 16, [1500, 16, 17, 777], 0, "any"),
    (2, 8, 2, 128, 9, [1000, 300], 64, "tree"),
    (3, 4, 1, 64, 20, [500, 20, 30], 5, "tree"),
    (2, 4, 2, 128, 64, [640, 65], 1, "chain"),
    (2, 2, 2, 64, 6, [320, 100], 100000, "padded"),
    (3, 16, 16, 128, 5, [2000, 1000, 5], 300, "chain"),
    (40, 2, 1, 64, 4, list(range(4, 164, 4)), 0, "tree"),
]


@pytest.mark.parametrize("layout", ["contiguous", "paged"])
@pytest.mark.parametrize("B,Hq,H,D,T,lens,window,kind", CASES)
def test_tree_matches_formula(reef, B, Hq, H, D, T, lens, window, kind, layout):
    print(f"\n[case] tree {layout} {B}x{Hq}/{H}x{D} T {T} lens {lens[:4]} window {window} {kind}",
          flush=True)
    rng = np.random.default_rng(B * 1000 + T * 10 + D + window)
    L = -(-max(lens) // PAGE) * PAGE + 16
    q, k, v, qs, ks, vs = problem(rng, B, Hq, H, D, T, lens, L)
    m = tree_masks(rng, B, T, kind)
    ref, tol = reference(q, k, v, qs, ks, vs, lens, m, window, 1 / math.sqrt(D))
    cache = poison(k, v, ks, vs, lens)
    mask = None if kind == "chain" else words(m)
    ln = gpu(np.array(lens, np.int32))
    for _ in range(2):  # the workspace serves again
        if layout == "paged":
            pools, table = paged(rng, *cache, lens)
            out = reef.attention_decode_tree_paged(gpu(q), gpu(qs), *pools, table, ln,
                                                   tree_mask=mask, window=window)
        else:
            out = reef.attention_decode_tree(gpu(q), gpu(qs), *contiguous(*cache), ln,
                                             tree_mask=mask, window=window)
        err = np.abs(out.cpu().numpy().astype(np.float64) - ref).max()
        assert err <= tol, (err, tol)
        if kind in ("padded", "any"):
            empty = ~m.any(2)
            assert not out.cpu().numpy().transpose(0, 2, 1, 3)[empty].any()


@pytest.mark.parametrize("D,Hq,H", [(128, 32, 8), (64, 12, 12), (128, 8, 1)])
def test_one_token_is_the_decode_step(reef, D, Hq, H):
    """T = 1: what attention_decode computes, within both kernels' roundings."""
    print(f"\n[case] tree of one against decode {Hq}/{H}x{D}", flush=True)
    rng = np.random.default_rng(D + Hq)
    B, L = 5, 1040
    lens = [1, 1040, 333, 64, 1000]
    q, k, v, qs, ks, vs = problem(rng, B, Hq, H, D, 1, lens, L)
    cache, ln = contiguous(k, v, ks, vs), gpu(np.array(lens, np.int32))
    for window in (0, 100):
        one = reef.attention_decode(gpu(q[:, :, 0]), gpu(qs[:, :, 0]), *cache, ln, window=window)
        tree = reef.attention_decode_tree(gpu(q), gpu(qs), *cache, ln, window=window)
        m = np.ones((B, 1, 1), bool)
        _, tol = reference(q, k, v, qs, ks, vs, lens, m, window, 1 / math.sqrt(D))
        assert float((tree[:, :, 0] - one).abs().max()) <= 2 * tol


def test_chain_is_a_prefill_chunk(reef):
    """A chain over equally long caches: attention_prefill_cache's chunk."""
    print("\n[case] chain against the prefill over the cache", flush=True)
    rng = np.random.default_rng(77)
    B, Hq, H, D, T, n = 2, 8, 2, 128, 24, 300
    L = 304
    q, k, v, qs, ks, vs = problem(rng, B, Hq, H, D, T, [n] * B, L)
    cache, ln = contiguous(k, v, ks, vs), gpu(np.full(B, n, np.int32))
    for window in (0, 40):
        chunk = reef.attention_prefill_cache(gpu(q), gpu(qs), *cache, n, window=window,
                                             q_granularity=reef.PER_TOKEN)
        tree = reef.attention_decode_tree(gpu(q), gpu(qs), *cache, ln, window=window)
        m = np.tril(np.ones((T, T), bool))[None].repeat(B, 0)
        _, tol = reference(q, k, v, qs, ks, vs, [n] * B, m, window, 1 / math.sqrt(D))
        assert float((tree - chunk).abs().max()) <= 2 * tol


@pytest.mark.parametrize("gran", ["tensor", "head", "token"])
def test_granularities_and_strides(reef, gran):
    """q and out as a projection lays them out; one scale per tensor, head or row; softmax
    scale 1; no lengths (every sequence full)."""
    print(f"\n[case] tree strides, scales per {gran}", flush=True)
    rng = np.random.default_rng(4)
    B, Hq, H, D, T, L = 3, 6, 2, 64, 10, 160
    q, k, v, _, ks, vs = problem(rng, B, Hq, H, D, T, [L] * B, L)
    g = {"tensor": 0, "head": 1, "token": 2}[gran]
    qs = rng.uniform(1e-4, 1e-3, [(1,), (Hq,), (B, Hq, T)][g]).astype(np.float32)
    full = np.broadcast_to(qs if g == 2 else qs.reshape(1, -1, 1), (B, Hq, T))
    m = tree_masks(rng, B, T, "tree")
    ref, tol = reference(q, k, v, full, ks, vs, [L] * B, m, 0, 1.0)
    qt = gpu(q.transpose(0, 2, 1, 3)).transpose(1, 2)  # [B, T, Hq, D] seen as [B, Hq, T, D]
    store = torch.full((B, T, Hq + 1, D), 3.0, device="cuda")
    out = store[:, :, :Hq].transpose(1, 2)
    got = reef.attention_decode_tree(qt, gpu(qs), *contiguous(k, v, ks, vs), tree_mask=words(m),
                                     softmax_scale=1.0, q_granularity=g, out=out)
    assert got is out
    assert np.abs(out.cpu().numpy() - ref).max() <= tol
    assert (store[:, :, Hq] == 3).all()


@pytest.mark.parametrize("D,Hq,H,T", [(128, 4, 1, 3), (64, 16, 2, 40)])
def test_long_sequences_merge_over_workgroups(reef, D, Hq, H, T):
    """Few long sequences: their blocks are cut into many runs. The result does not depend on
    the order in which they end: equal bits each time."""
    print(f"\n[case] tree of long sequences {Hq}/{H}x{D} T {T}", flush=True)
    rng = np.random.default_rng(D)
    lens = [20000, 77, 9001]
    L = 20016
    q, k, v, qs, ks, vs = problem(rng, 3, Hq, H, D, T, lens, L)
    m = tree_masks(rng, 3, T, "tree")
    ref, tol = reference(q, k, v, qs, ks, vs, lens, m, 0, 1 / math.sqrt(D))
    cache, ln = contiguous(k, v, ks, vs), gpu(np.array(lens, np.int32))
    first = None
    for _ in range(5):
        out = reef.attention_decode_tree(gpu(q), gpu(qs), *cache, ln, tree_mask=words(m))
        assert np.abs(out.cpu().numpy() - ref).max() <= tol
        assert first is None or torch.equal(first, out)
        first = out


def test_peaked_and_flat_rows(reef):
    """Scores that rise by hundreds along the keys (every block rescales), and all equal; value
    scales from 1e-6 to 1e3 along the keys."""
    print("\n[case] tree peaked and flat rows", flush=True)
    rng = np.random.default_rng(6)
    B, Hq, H, D, T, n = 2, 4, 1, 64, 5, 900
    L = 912
    q, k, v, qs, ks, vs = problem(rng, B, Hq, H, D, T, [n] * B, L)
    q[0] = 127
    k[0] = 1 + np.arange(L)[None, :, None] % 100
    k[0, :, :, D // 2:] = (np.arange(L) // 8)[None, :, None].clip(0, 127)
    q[1] = 0
    ks[:] = 0.02
    vs[:] = 10.0 ** np.linspace(-6, 3, L)[None, None, :]
    m = tree_masks(rng, B, T, "tree")
    ref, tol = reference(q, k, v, qs, ks, vs, [n] * B, m, 0, 1.0)
    out = reef.attention_decode_tree(gpu(q), gpu(qs), *contiguous(k, v, ks, vs),
                                     gpu(np.full(B, n, np.int32)), tree_mask=words(m), softmax_scale=1.0)
    assert np.abs(out.cpu().numpy() - ref).max() <= tol


def test_pages_behind_the_window_may_be_given_back(reef):
    """Table entries of pages that no row's window reaches are not looked up."""
    print("\n[case] tree with evicted pages", flush=True)
    rng = np.random.default_rng(12)
    B, Hq, H, D, T, window = 2, 4, 2, 128, 4, 50
    lens = [400, 111]
    q, k, v, qs, ks, vs = problem(rng, B, Hq, H, D, T, lens, 400)
    m = tree_masks(rng, B, T, "tree")
    ref, tol = reference(q, k, v, qs, ks, vs, lens, m, window, 1 / math.sqrt(D))
    pools, table = paged(rng, *poison(k, v, ks, vs, lens), lens)
    for b in range(B):
        first = lens[b] - T + 1 - window  # the shallowest row's
        gone = table[b, :first // PAGE].long()
        pools[2][gone], pools[3][gone] = float("nan"), float("inf")
        table[b, :first // PAGE] = -1
    out = reef.attention_decode_tree_paged(gpu(q), gpu(qs), *pools, table,
                                           gpu(np.array(lens, np.int32)), tree_mask=words(m), window=window)
    assert np.abs(out.cpu().numpy() - ref).max() <= tol


def test_bad_lengths_and_pages(reef):
    """A length outside gives zeros for that sequence, a page outside takes no part: both are
    flagged and the neighbours are right."""
    print("\n[case] tree bad lengths and pages", flush=True)
    rng = np.random.default_rng(13)
    B, Hq, H, D, T = 4, 8, 2, 64, 6
    lens = [100, 90, 80, 70]
    q, k, v, qs, ks, vs = problem(rng, B, Hq, H, D, T, lens, 112)
    m = tree_masks(rng, B, T, "tree")
    ref, tol = reference(q, k, v, qs, ks, vs, lens, m, 0, 1 / math.sqrt(D))
    for bad in (5, 113, 0, -3):
        status = reef.StatusWord()
        ln = np.array(lens, np.int32)
        ln[1] = bad
        out = reef.attention_decode_tree(gpu(q), gpu(qs), *contiguous(k, v, ks, vs), gpu(ln),
                                         tree_mask=words(m), status=status).cpu().numpy()
        with pytest.raises(reef.InvalidArgument):
            status.check("tree")
        assert not out[1].any()
        assert np.abs(out - ref)[[0, 2, 3]].max() <= tol
    for bad in (-1, 10 ** 6):
        status = reef.StatusWord()
        pools, table = paged(rng, k, v, ks, vs, lens)
        table[2, 1] = bad
        out = reef.attention_decode_tree_paged(gpu(q), gpu(qs), *pools, table,
                                               gpu(np.array(lens, np.int32)), tree_mask=words(m),
                                               status=status).cpu().numpy()
        with pytest.raises(reef.InvalidArgument):
            status.check("tree")
        assert np.isfinite(out).all()
        assert np.abs(out - ref)[[0, 1, 3]].max() <= tol


@pytest.mark.parametrize("D,Hq,H,T", [(64, 2, 2, 7), (128, 8, 1, 20)])
@pytest.mark.parametrize("what", ["nan key", "nan value", "inf value"])
def test_a_drafted_token_that_is_not_finite(reef, D, Hq, H, T, what):
    """Its scale reaches the rows that see it, which are not finite, and no other."""
    print(f"\n[case] tree with a drafted token that is not finite: {what} {Hq}/{H}x{D} T {T}",
          flush=True)
    rng = np.random.default_rng(D)
    B, L = 2, 720
    lens = [700, T]
    q, k, v, qs, ks, vs = problem(rng, B, Hq, H, D, T, lens, L)
    m = tree_masks(rng, B, T, "tree")
    ref, tol = reference(q, k, v, qs, ks, vs, lens, m, 0, 1 / math.sqrt(D))
    bad = 1
    for b in range(B):
        (ks if what == "nan key" else vs)[b, :, lens[b] - T + bad] = float(what[:3])
    out = reef.attention_decode_tree(gpu(q), gpu(qs), *contiguous(k, v, ks, vs),
                                     gpu(np.array(lens, np.int32)), tree_mask=words(m)).cpu().numpy()
    sees = np.broadcast_to(m[:, None, :, bad], out.shape[:3])
    assert sees.any() and not sees.all()
    assert not np.isfinite(out[sees]).any()
    assert np.abs(out - ref)[~sees].max() <= tol


@pytest.mark.parametrize("D,Hq,H,T", [(64, 2, 2, 7), (128, 8, 1, 20)])
@pytest.mark.parametrize("value", [np.inf, -np.inf])
def test_a_drafted_token_with_an_infinite_key_scale(reef, D, Hq, H, T, value):
    """Its score is an infinity of either sign: the rows that see it are not finite whichever,
    and the others are right. The token lies in a sequence's last block, or in its only one."""
    print(f"\n[case] tree with a key scale of {value} {Hq}/{H}x{D} T {T}", flush=True)
    rng = np.random.default_rng(D + T)
    B, L = 3, 720
    lens = [700, T, 64]
    q, k, v, qs, ks, vs = problem(rng, B, Hq, H, D, T, lens, L)
    m = tree_masks(rng, B, T, "tree")
    ref, tol = reference(q, k, v, qs, ks, vs, lens, m, 0, 1 / math.sqrt(D))
    bad = 1
    at = [n - T + bad for n in lens]
    signs = [(q[b, h, t].astype(int) @ k[b, h // (Hq // H), at[b]].astype(int)) * value > 0
             for b in range(B) for h in range(Hq) for t in range(T) if m[b, t, bad]]
    assert any(signs) and not all(signs)
    for b in range(B):
        ks[b, :, at[b]] = value
    out = reef.attention_decode_tree(gpu(q), gpu(qs), *contiguous(k, v, ks, vs),
                                     gpu(np.array(lens, np.int32)), tree_mask=words(m)).cpu().numpy()
    sees = np.broadcast_to(m[:, None, :, bad], out.shape[:3])
    assert sees.any() and not sees.all()
    assert not np.isfinite(out[sees]).any()
    assert np.abs(out - ref)[~sees].max() <= tol


def reference_by_row(q, k, v, qs, ks, vs, lens, m, window, scale):
    """(out, tolerance [B, Hq, T, 1]): the tolerance of the file's head from what each row sees
    alone, its exponents and 127 times its largest value scale. (A weight is off by 2^-33 of a
    power of two that is less than twice that scale, or 2^-112; the row sum does not share this.)"""
    out, _ = reference(q, k, v, qs, ks, vs, lens, m, window, scale)
    B, Hq, T, D = q.shape
    tol = np.zeros((B, Hq, T, 1))
    for b in range(B):
        n = int(lens[b])
        depth = m[b].sum(1) - 1
        pos = np.concatenate([np.arange(n - T), n - T + depth])
        seen = np.concatenate([np.ones((T, n - T), bool), m[b]], 1)
        if window:
            seen &= pos[None, :] > (n - T + depth)[:, None] - window
        seen[m[b].sum(1) == 0] = False
        for h in range(Hq):
            kk = k[b, h * k.shape[1] // Hq, :n] * ks[b, h * k.shape[1] // Hq, :n, None].astype(np.float64)
            s = np.abs((q[b, h] * qs[b, h][:, None].astype(np.float64)) @ kk.T) * scale / math.log(2)
            for t in np.flatnonzero(seen.any(1)):
                X = s[t, seen[t]].max()
                top = float(vs[b, h * k.shape[1] // Hq, :n][seen[t]].max())
                tol[b, h, t] = 127.0 * (top * (2 * (2.8 * X * U + 6 * U) + 14 * U)
                                        + max(top, 2.0 ** -112) * 2 * n * 2.0 ** -33)
    return out, tol


@pytest.mark.parametrize("D,Hq,H,T", [(64, 2, 2, 7), (128, 8, 1, 20), (128, 3, 3, 64)])
@pytest.mark.parametrize("large", [1e4, 1e8, 1e30, 1e36])
def test_large_values_of_a_hidden_token(reef, D, Hq, H, T, large):
    """A token whose values are finite and far above all others' changes nothing for the rows that
    do not see it: a drafted one in a sequence's last block or its only one, and one that
    only the shallow rows' windows reach."""
    print(f"\n[case] tree with value scales of {large} {Hq}/{H}x{D} T {T}", flush=True)
    rng = np.random.default_rng(D + T + 1)
    B, L = 3, 720
    lens = [700, 64, max(T, 33)]
    q, k, v, qs, ks, vs = problem(rng, B, Hq, H, D, T, lens, L)
    m = tree_masks(rng, B, T, "tree")
    for window in (0, 25):
        scales = vs.copy()
        for b in range(B):
            scales[b, :, lens[b] - T + 1] = large
            if window and lens[b] - T >= window:
                scales[b, :, lens[b] - T + 1 - window] = large
        ref, tol = reference_by_row(q, k, v, qs, ks, scales, lens, m, window, 1 / math.sqrt(D))
        sees = tol[..., 0] > large * 1e-7
        assert sees.any() and (tol[~sees] < 1e-3).all() and not sees.all()
        cache, ln = contiguous(k, v, ks, scales), gpu(np.array(lens, np.int32))
        out = reef.attention_decode_tree(gpu(q), gpu(qs), *cache, ln, tree_mask=words(m), window=window)
        assert (np.abs(out.cpu().numpy() - ref) <= tol).all()


@pytest.mark.parametrize("size", [1e-30, 1e-36, 1e-37])
def test_small_values(reef, size):
    """Value scales whose inverse times 2^8 is beyond fp32; beside them drafted tokens of
    ordinary ones, which some rows see."""
    print(f"\n[case] tree with value scales of {size}", flush=True)
    rng = np.random.default_rng(31)
    B, Hq, H, D, T, lens = 2, 4, 1, 64, 12, [300, 30]
    q, k, v, qs, ks, vs = problem(rng, B, Hq, H, D, T, lens, 304)
    m = tree_masks(rng, B, T, "tree")
    vs = (rng.uniform(0.5, 1.0, vs.shape) * size).astype(np.float32)
    for mixed in (False, True):
        if mixed:
            for b in range(B):
                vs[b, :, lens[b] - T + 1] = 0.01
        ref, tol = reference_by_row(q, k, v, qs, ks, vs, lens, m, 0, 1 / math.sqrt(D))
        out = reef.attention_decode_tree(gpu(q), gpu(qs), *contiguous(k, v, ks, vs),
                                         gpu(np.array(lens, np.int32)), tree_mask=words(m))
        assert (np.abs(out.cpu().numpy().astype(np.float64) - ref) <= tol).all()


@pytest.mark.parametrize("D,Hq,H,T,window", [(64, 2, 2, 7, 0), (128, 8, 1, 20, 0), (64, 4, 2, 6, 30)])
def test_query_scales_of_zero(reef, D, Hq, H, T, window):
    """Rows whose scale is 0 (so are their scores): the mean of the values that they see. A row
    whose mask is 0 too stays zeros."""
    print(f"\n[case] tree with query scales of 0 {Hq}/{H}x{D} T {T}", flush=True)
    rng = np.random.default_rng(D + T + 2)
    lens = [300, T, 64]
    q, k, v, qs, ks, vs = problem(rng, 3, Hq, H, D, T, lens, 304)
    qs[:, :, ::2] = 0
    m = tree_masks(rng, 3, T, "tree")
    m[1, T - 1] = False
    ref, tol = reference(q, k, v, qs, ks, vs, lens, m, window, 1 / math.sqrt(D))
    cache = contiguous(*poison(k, v, ks, vs, lens))
    out = reef.attention_decode_tree(gpu(q), gpu(qs), *cache, gpu(np.array(lens, np.int32)),
                                     tree_mask=words(m), window=window).cpu().numpy()
    assert np.abs(out - ref).max() <= tol
    assert not out[1, :, T - 1].any()


def test_workspace_serves_every_shape(reef):
    """One explicit workspace, sized for the largest, through calls of several shapes."""
    print("\n[case] tree workspace over shapes", flush=True)
    rng = np.random.default_rng(14)
    ws = reef.tree_workspace(reef.TreeParams(4, 32, 1, 128, 64, 4096, 0, 0.1, 2, 0, 0), "cuda")
    for B, Hq, H, D, T, lens in ((1, 8, 1, 128, 64, [4000]), (3, 8, 2, 64, 3, [3000, 10, 500]),
                                 (1, 2, 2, 64, 1, [4000]), (1, 8, 1, 128, 64, [4000])):
        q, k, v, qs, ks, vs = problem(rng, B, Hq, H, D, T, lens, 4000)
        m = tree_masks(rng, B, T, "tree")
        ref, tol = reference(q, k, v, qs, ks, vs, lens, m, 0, 1 / math.sqrt(D))
        out = reef.attention_decode_tree(gpu(q), gpu(qs), *contiguous(k, v, ks, vs),
                                         gpu(np.array(lens, np.int32)), tree_mask=words(m), workspace=ws)
        assert np.abs(out.cpu().numpy() - ref).max() <= tol


def test_refuses_what_lies_elsewhere(reef):
    """A workspace in host memory, q and scales that do not match: refused before a launch."""
    print("\n[case] tree refusals", flush=True)
    rng = np.random.default_rng(17)
    q, k, v, qs, ks, vs = problem(rng, 1, 2, 1, 64, 3, [40], 48)
    cache = contiguous(k, v, ks, vs)
    p = reef.TreeParams(1, 2, 1, 64, 3, 48, 0, 0.1, 2, 0, 0)
    ws = reef.tree_workspace(p, "cuda")
    for call in (lambda: reef.attention_decode_tree(gpu(q), gpu(qs), *cache, workspace=ws.cpu()),
                 lambda: reef.attention_decode_tree(gpu(q), gpu(qs), *cache, workspace=ws[:100]),
                 lambda: reef.attention_decode_tree(gpu(q), gpu(qs), *cache,
                                                    workspace=torch.stack([ws, ws])[:, ::2]),
                 lambda: reef.attention_decode_tree(gpu(q), gpu(qs[:, :1]), *cache),
                 lambda: reef.attention_decode_tree(gpu(q)[..., :32], gpu(qs), *cache),
                 lambda: reef.attention_decode_tree(gpu(q), gpu(qs), *cache, out=gpu(qs)),
                 lambda: reef.attention_decode_tree(gpu(q), gpu(qs), *cache, window=-1),
                 lambda: reef.attention_decode_tree(
                     gpu(q), gpu(qs), *cache, tree_mask=torch.zeros((1, 2), dtype=torch.int64, device="cuda")),
                 lambda: reef.attention_decode_tree(
                     gpu(q), gpu(qs), *cache, torch.zeros(2, dtype=torch.int32, device="cuda"))):
        with pytest.raises(reef.InvalidArgument):
            call()


def test_two_streams_and_a_large_batch(reef):
    """Calls on two streams at once have a workspace each; over 2048 sequences run in slices."""
    print("\n[case] tree on two streams, 2100 sequences", flush=True)
    rng = np.random.default_rng(15)
    B, Hq, H, D, T, L = 2100, 2, 1, 64, 2, 32
    lens = rng.integers(T, L + 1, B)
    q, k, v, qs, ks, vs = problem(rng, B, Hq, H, D, T, lens, L)
    m = tree_masks(rng, B, T, "tree")
    ref, tol = reference(q, k, v, qs, ks, vs, lens, m, 0, 1 / math.sqrt(D))
    cache, ln, mask, tq, tqs = contiguous(k, v, ks, vs), gpu(lens.astype(np.int32)), words(m), gpu(q), gpu(qs)
    pools, table = paged(rng, k, v, ks, vs, lens)
    torch.cuda.synchronize()
    status = [reef.StatusWord() for _ in range(2)]
    outs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            if i % 2:
                outs.append(reef.attention_decode_tree(tq, tqs, *cache, ln, tree_mask=mask, status=status[1]))
            else:
                outs.append(reef.attention_decode_tree_paged(tq, tqs, *pools, table, ln, tree_mask=mask,
                                                             status=status[0]))
    torch.cuda.synchronize()
    for s in status:
        s.check("tree")
    for out in outs:
        assert np.abs(out.cpu().numpy() - ref).max() <= tol


def test_tree_in_graphs(reef):
    """Two captured graphs and eager calls in turn, each equal to the eager result."""
    print("\n[case] tree in graphs", flush=True)
    rng = np.random.default_rng(16)
    B, Hq, H, D, T, L = 3, 8, 2, 128, 12, 1600
    lens = [1600, 12, 801]
    q, k, v, qs, ks, vs = problem(rng, B, Hq, H, D, T, lens, L)
    m = tree_masks(rng, B, T, "tree")
    cache, ln, mask, tq, tqs = contiguous(k, v, ks, vs), gpu(np.array(lens, np.int32)), words(m), gpu(q), gpu(qs)
    status = reef.StatusWord()

    def step():
        return reef.attention_decode_tree(tq, tqs, *cache, ln, tree_mask=mask, status=status)

    eager = step().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for _ in range(3):
        for graph, out in graphs:
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, eager) for _, out in graphs)
        assert torch.equal(step(), eager)
    status.check("graphs")


@pytest.mark.parametrize("layout", ["contiguous", "paged"])
def test_offsets_past_32_bits(reef, layout):
    """The last tokens of a cache of 2.2 GB of keys and as much of values: attention within a
    window, and the kept rows."""
    print(f"\n[case] tree and keep past 2^31 bytes, {layout}", flush=True)
    rng = np.random.default_rng(18)
    Hq, H, D, T, window, L = 4, 1, 128, 5, 100, 17_200_000
    n, tail = L - 3, 192  # the last `tail` places hold something
    q, k, v, qs, ks, vs = problem(rng, 1, Hq, H, D, T, [tail - 3], tail)
    m = tree_masks(rng, 1, T, "tree")
    ref, tol = reference(q, k, v, qs, ks, vs, [tail - 3], m, window, 1 / math.sqrt(D))
    P = L // PAGE
    small = contiguous(k, v, ks, vs)
    if layout == "contiguous":
        cache = [torch.zeros((1, H, L, D), dtype=torch.int8, device="cuda"),
                 torch.zeros((1, H, P, D, PAGE), dtype=torch.int8, device="cuda"),
                 *(torch.full((1, H, L), float("nan"), device="cuda") for _ in range(2))]
        ends = [t[:, :, -s.shape[2]:] for t, s in zip(cache, small)]
    else:
        cache = [torch.zeros((P, H, PAGE, D), dtype=torch.int8, device="cuda"),
                 torch.zeros((P, H, D, PAGE), dtype=torch.int8, device="cuda"),
                 *(torch.full((P, H, PAGE), float("nan"), device="cuda") for _ in range(2))]
        ends = [t[-(tail // PAGE):].view(s.shape) for t, s in zip(cache, small)]
    for end, s in zip(ends, small):
        end.copy_(s)
    lens = gpu(np.array([n], np.int32))
    args = [lens]
    if layout == "paged":
        args = [torch.arange(P, dtype=torch.int32, device="cuda")[None], lens]
    call = reef.attention_decode_tree if layout == "contiguous" else reef.attention_decode_tree_paged
    out = call(gpu(q), gpu(qs), *cache, *args, tree_mask=words(m), window=window)
    assert np.abs(out.cpu().numpy() - ref).max() <= tol
    kept, some = np.array([[1, 3, 4, 0, 0]], np.int32), gpu(np.array([3], np.int32))
    if layout == "contiguous":
        new = reef.kv_keep(gpu(kept), some, lens, *cache)
    else:
        new = reef.kv_keep_paged(gpu(kept), some, lens, args[0], *cache)
    assert int(new) == n - T + 3
    first = tail - 3 - T
    for a, s, to in ((k, small[0], ends[0]), (ks, small[2], ends[2]), (vs, small[3], ends[3])):
        want = a.copy()
        want[:, :, first:first + 3] = a[:, :, first + kept[0, :3]]
        assert np.array_equal(want, to.cpu().numpy(), equal_nan=False)
    want = v.copy()
    want[:, :, first:first + 3] = v[:, :, first + kept[0, :3]]
    assert np.array_equal(contiguous(k, want, ks, vs)[1].cpu().numpy(), ends[1].cpu().numpy())
