"""Pages of the int8 cache against a sequential model of the same rules on the host: every
table, count, length and copy list equal, and the pools byte for byte. Each case prints its
name before touching the GPU."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

PAGE = 16


@pytest.fixture(scope="module")
def reef():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import reef_amd
    reef_amd.lib()
    return reef_amd


def gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def host(t):
    return t.cpu().numpy()


def i32(a):
    return np.array(a, np.int32)


class Model:
    """Table, lengths and counts, one sequence after the other."""

    def __init__(self, batch, blocks, pages):
        self.table = np.full((batch, blocks), -1, np.int32)
        self.lens = np.zeros(batch, np.int32)
        self.refs = np.zeros(pages, np.int32)

    def device(self):
        return gpu(self.table), gpu(self.lens), gpu(self.refs)

    def free(self, sequences):
        for b in sequences:
            if b < 0:
                continue
            for i, p in enumerate(self.table[b]):
                if p >= 0:
                    self.refs[p] -= 1
                    self.table[b, i] = -1
            self.lens[b] = 0

    def fork(self, parents, children):
        for p, c in zip(parents, children):
            if p < 0 or c < 0 or p == c:
                continue
            row = np.where(np.arange(self.table.shape[1]) * PAGE < self.lens[p], self.table[p], -1)
            for x in row[row >= 0]:
                self.refs[x] += 1
            for x in self.table[c][self.table[c] >= 0]:
                self.refs[x] -= 1
            self.table[c], self.lens[c] = row, self.lens[p]

    def reserve(self, n):
        """(source, destination, whether every block was served)"""
        src, dst = np.full(len(self.lens), -1, np.int32), np.full(len(self.lens), -1, np.int32)
        free, given_up, served = list(np.flatnonzero(self.refs == 0)), [], True
        before = self.refs.copy()
        for b, length in enumerate(self.lens):
            if length < 0 or length + n > self.table.shape[1] * PAGE:
                served = False
                continue
            for i in range(length // PAGE, -(-(length + n) // PAGE)):
                old = self.table[b, i]
                if old >= 0 and before[old] <= 1:
                    continue
                if not free:
                    served = False
                    continue
                new = free.pop(0)
                self.table[b, i], self.refs[new] = new, 1
                if old >= 0:
                    given_up.append(old)
                    if i * PAGE < length:
                        src[b], dst[b] = old, new
        for p in given_up:
            self.refs[p] -= 1
        return src, dst, served

    def compact(self):
        P = len(self.refs)
        live = np.flatnonzero(self.refs > 0)
        L = len(live)
        movers, holes = live[live >= L][::-1], np.flatnonzero(self.refs[:L] <= 0)
        src, dst = np.full(P // 2, -1, np.int32), np.full(P // 2, -1, np.int32)
        src[:len(movers)], dst[:len(movers)] = movers, holes
        to = np.arange(P)
        to[movers] = holes
        self.table = np.where(self.table >= 0, to[self.table], -1).astype(np.int32)
        self.refs[holes], self.refs[movers] = self.refs[movers], 0
        return src, dst, L

    def check(self, table, lens, refs):
        assert np.array_equal(host(table), self.table)
        assert np.array_equal(host(refs), self.refs)
        if lens is not None:
            assert np.array_equal(host(lens), self.lens)
        named = self.table[self.table >= 0]
        assert np.array_equal(np.bincount(named, minlength=len(self.refs)), self.refs)


@pytest.mark.parametrize("seed,batch,blocks,pages", [(0, 6, 9, 64), (1, 1, 1, 1), (2, 70, 40, 2100),
                                                     (3, 300, 5, 900), (4, 13, 700, 5000),
                                                     (5, 40, 30, 20011)])
def test_a_servers_life(reef, seed, batch, blocks, pages):
    """Sequences come, grow by one or many tokens, fork, end; the pool is compacted. Whenever
    pages run out, the blocks served are the first ones and CAPACITY is set."""
    print(f"\n[case] pages seed {seed} batch {batch} blocks {blocks} pages {pages}", flush=True)
    rng = np.random.default_rng(seed)
    m = Model(batch, blocks, pages)
    table, lens, refs = m.device()
    for step in range(40):
        what = rng.integers(0, 8)
        if what <= 3:
            n = int(rng.choice([1, 1, 5, 16, 17, min(blocks * PAGE, 200)]))
            n = min(n, blocks * PAGE)
            src, dst, served = m.reserve(n)
            status = reef.StatusWord()
            s, d = reef.kv_reserve(table, lens, refs, n, status=status)
            if served:
                status.check("reserve")
            else:
                with pytest.raises(reef.CapacityError):
                    status.check("reserve")
            assert np.array_equal(host(s), src) and np.array_equal(host(d), dst)
            # the sequences that have the room take the tokens
            for b in range(batch):
                end = m.lens[b] + n
                if end <= blocks * PAGE and (m.table[b, :-(-end // PAGE)] >= 0).all() and rng.random() < 0.9:
                    m.lens[b] = end
            lens.copy_(gpu(m.lens))
        elif what <= 4:
            some = i32(rng.permutation(batch)[:rng.integers(1, batch + 1)])
            some = i32(np.concatenate([some, [-1], some[:1]]))  # padding, and one twice
            m.free(some[:-1])
            reef.kv_free(gpu(some), table, lens, refs)
        elif what <= 6 and batch > 1:
            children = rng.permutation(batch)[:rng.integers(1, batch)]
            parents = rng.choice(np.setdiff1d(np.arange(batch), children), len(children))
            parents[0] = parents[0] if rng.random() < 0.8 else -1
            m.fork(parents, children)
            reef.kv_fork(gpu(i32(parents)), gpu(i32(children)), table, lens, refs)
        else:
            src, dst, live = m.compact()
            s, d, n = reef.kv_compact(table, refs)
            assert int(n) == live
            assert np.array_equal(host(s), src) and np.array_equal(host(d), dst)
        m.check(table, lens, refs)


def pool(rng, shape, D):
    k = rng.integers(-127, 128, (*shape, PAGE, D)).astype(np.int8)
    v = rng.integers(-127, 128, (*shape, D, PAGE)).astype(np.int8)
    ks, vs = (rng.random((*shape, PAGE)).astype(np.float32) for _ in range(2))
    return k, v, ks, vs


@pytest.mark.parametrize("heads,D", [(1, 64), (3, 128), (8, 128), (5, 64), (37, 64)])
def test_copy_pages(reef, heads, D):
    print(f"\n[case] copy pages heads {heads} dim {D}", flush=True)
    rng = np.random.default_rng(heads + D)
    P = 90
    pools = pool(rng, (P, heads), D)
    order = rng.permutation(P)
    src, dst = i32(order[:30]), i32(order[30:60])
    src[3], dst[7], src[9], dst[9] = -1, -1, 11, 11
    src[20] = src[21]  # one page to two places
    t = [gpu(x) for x in pools]
    reef.kv_copy_pages(gpu(src), gpu(dst), *t)
    for got, was in zip(t, pools):
        want = was.copy()
        for s, d in zip(src, dst):
            if s >= 0 and d >= 0:
                want[d] = was[s]
        assert np.array_equal(host(got), want)
    reef.kv_copy_pages(gpu(src[:0]), gpu(dst[:0]), *t)  # nothing


def test_copy_of_very_long_lists(reef):
    """As many workgroups as have 2^32 threads, and some: the pairs at the end are copied too."""
    print("\n[case] copy pages, 2^24 + 3 pairs", flush=True)
    rng = np.random.default_rng(24)
    n = (1 << 24) + 3
    pools = pool(rng, (8, 1), 64)
    src = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    dst = src.clone()
    for i, (s, d) in enumerate(((0, 1), (2, 3), (4, 5), (6, 7))):
        at = (0, 1 << 21, (1 << 24) - 1, n - 1)[i]
        src[at], dst[at] = s, d
    t = [gpu(x) for x in pools]
    reef.kv_copy_pages(src, dst, *t)
    for got, was in zip(t, pools):
        want = was.copy()
        want[1::2] = was[::2]
        assert np.array_equal(host(got), want)


def test_copy_on_write_keeps_the_parent(reef):
    """A fork's next token lands in a copy: the parent's bytes stay, also on two layers."""
    print("\n[case] copy on write", flush=True)
    rng = np.random.default_rng(8)
    B, H, D, P = 4, 2, 64, 40
    m = Model(B, 4, P)
    table, lens, refs = m.device()
    one = reef.kv_reserve(table, lens, refs, 23)
    lens[:2] = 23
    layers = [[gpu(x) for x in pool(rng, (P, H), D)] for _ in range(2)]
    before = [[x.clone() for x in layer] for layer in layers]
    reef.kv_fork(gpu(i32([0, 0])), gpu(i32([2, 3])), table, lens, refs)
    src, dst = reef.kv_reserve(table, lens, refs, 1)
    for layer in layers:
        reef.kv_copy_pages(src, dst, *layer)
    tb = host(table)
    assert len({tb[0, 1], tb[2, 1], tb[3, 1]}) == 3 and tb[0, 0] == tb[2, 0] == tb[3, 0]
    for layer, was in zip(layers, before):
        for x, y in zip(layer, was):
            for b in (2, 3):
                assert torch.equal(x[tb[b, 1]], y[host(src)[b]])
            assert torch.equal(x[tb[1, 1]], y[tb[1, 1]])
    k_new, v_new = (torch.randn(B, H, 1, D, device="cuda") for _ in range(2))
    start = lens.clone()
    start[1] = 23
    parent = [x[tb[0, 0]].clone() for x in layers[0]]
    reef.kv_append_paged(k_new, v_new, start, table, *layers[0])
    for x, y in zip(layers[0], parent):
        assert torch.equal(x[tb[0, 0]], y)
    assert one is not None


@pytest.mark.parametrize("who", [[0, 2, 3], [2, 3], [0], [3]])
def test_tokens_after_a_fork_stay_apart(reef, who):
    """Two forks of a sequence whose last page is partial, then a token for some of the three: each
    finds the seven tokens from before the fork and its own, and the others' pages stay as they
    were, byte for byte."""
    print(f"\n[case] copy on write, tokens of sequences {who}", flush=True)
    rng = np.random.default_rng(9)
    B, H, D, P, n = 4, 2, 64, 40, 23
    m = Model(B, 4, P)
    table, lens, refs = m.device()
    reef.kv_reserve(table, lens, refs, n)
    lens[:2] = n
    layer = [gpu(x) for x in pool(rng, (P, H), D)]
    shared = int(table[0, 1])
    before = [host(x[shared]) for x in layer]
    reef.kv_fork(gpu(i32([0, 0])), gpu(i32([2, 3])), table, lens, refs)
    src, dst = reef.kv_reserve(table, lens, refs, 1)
    reef.kv_copy_pages(src, dst, *layer)
    tb = host(table)
    assert len(set(tb[:, 1])) == B and len({tb[0, 0], tb[2, 0], tb[3, 0]}) == 1
    whole = [host(x) for x in layer]
    k_new, v_new = (torch.randn(len(who), H, 1, D, generator=torch.Generator().manual_seed(i)).cuda()
                    for i in range(2))
    reef.kv_append_paged(k_new, v_new, lens[gpu(i32(who)).long()], table[gpu(i32(who)).long()], *layer)
    (kq, ks), (vq, vs) = (reef.quantize_rows(x.view(-1, D)) for x in (k_new, v_new))
    new = [host(x).reshape(len(who), H, -1) for x in (kq, vq, ks, vs)]
    slot = n % PAGE
    for i, x in enumerate(layer):
        got, want = host(x), whole[i].copy()
        value = i == 1  # [pages, heads, head_dim, 16]: the slot is last
        for b in (0, 2, 3):
            page = got[tb[b, 1]]
            if not value:
                assert np.array_equal(page[:, :slot], before[i][:, :slot])
            else:
                assert np.array_equal(page[..., :slot], before[i][..., :slot])
        for j, b in enumerate(who):
            row = new[i][j] if i < 2 else new[i][j][:, 0]
            if value:
                want[tb[b, 1]][..., slot] = row
            else:
                want[tb[b, 1]][:, slot] = row
        assert np.array_equal(got, want)


@pytest.mark.parametrize("sharers,free,short", [(2, 1, False), (2, 0, True), (5, 4, False), (5, 3, True),
                                                (2, 2, False), (1300, 1299, False), (1300, 1298, True)])
def test_the_last_sharer_needs_no_page(reef, sharers, free, short):
    """With one free page fewer than sharers of a page, the last of them is left with it alone:
    every block has a page of its own, nothing is missing. With fewer still, some lack one."""
    print(f"\n[case] reserve {sharers} sharers {free} free pages", flush=True)
    m = Model(sharers, 2, 1 + free)
    m.table[:, 0], m.lens[:], m.refs[0] = 0, 5, sharers
    table, lens, refs = m.device()
    src, dst, _ = m.reserve(1)
    status = reef.StatusWord()
    s, d = reef.kv_reserve(table, lens, refs, 1, status=status)
    assert np.array_equal(host(s), src) and np.array_equal(host(d), dst)
    m.check(table, lens, refs)
    if short:
        with pytest.raises(reef.CapacityError):
            status.check("reserve")
        assert m.refs.max() > 1
    else:
        status.check("reserve")
        assert (m.refs[m.table[:, 0]] == 1).all()
        if free < sharers:  # again: there is nothing left to do
            reef.kv_reserve(table, lens, refs, 1)
            m.check(table, lens, refs)


def test_no_page_for_an_absent_block(reef):
    """Beside a last sharer that needs none, a sequence without a page lacks one."""
    print("\n[case] reserve a last sharer and an absent block", flush=True)
    m = Model(3, 2, 2)
    m.table[:2, 0], m.lens[:2], m.refs[0] = 0, 5, 2
    table, lens, refs = m.device()
    m.reserve(1)
    status = reef.StatusWord()
    reef.kv_reserve(table, lens, refs, 1, status=status)
    m.check(table, lens, refs)
    assert m.table[2, 0] == -1
    with pytest.raises(reef.CapacityError):
        status.check("reserve")


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("B,H,D,T", [(1, 1, 64, 1), (5, 3, 128, 7), (9, 2, 64, 64), (3, 8, 128, 33),
                                     (66, 1, 128, 16)])
def test_keep(reef, paged, B, H, D, T):
    print(f"\n[case] keep paged {paged} {B}x{H}x{D} T {T}", flush=True)
    rng = np.random.default_rng(B * T + D + paged)
    blocks = 12
    L = blocks * PAGE
    lens = i32(rng.integers(T, L + 1, B))
    lens[0] = T  # nothing before the drafts
    lens[-1] = L
    kept, n = np.full((B, T), 10 ** 6, np.int32), np.zeros(B, np.int32)
    for b in range(B):
        n[b] = rng.integers(0, T + 1) if b else T  # all, none, some
        kept[b, :n[b]] = np.sort(rng.permutation(T)[:n[b]])
    if B > 2:
        kept[1, :1], n[1] = T - 1, 1
        n[2] = 0
    if paged:
        pools = pool(rng, (B * blocks + 7, H), D)
        table = i32(rng.permutation(B * blocks + 7)[:B * blocks].reshape(B, blocks))
    else:
        pools = pool(rng, (B, H, blocks), D)
    want = [x.copy() for x in pools]

    def at(x, b, pos, value):
        i = (table[b, pos // PAGE], slice(None)) if paged else (b, slice(None), pos // PAGE)
        return x[i][..., pos % PAGE] if value else x[i][:, pos % PAGE]

    for b in range(B):
        for i in range(n[b]):
            for x, was, value in zip(want, pools, (False, True, False, False)):
                at(x, b, lens[b] - T + i, value)[:] = at(was, b, lens[b] - T + kept[b, i], value)
    if paged:
        t = [gpu(x) for x in pools]
        new = reef.kv_keep_paged(gpu(kept), gpu(n), gpu(lens), gpu(table), *t)
    else:
        k, v, ks, vs = pools
        t = [gpu(k.reshape(B, H, L, D)), gpu(v), gpu(ks.reshape(B, H, L)), gpu(vs.reshape(B, H, L))]
        new = reef.kv_keep(gpu(kept), gpu(n), gpu(lens), *t)
    assert np.array_equal(host(new), lens - T + n)
    for got, x in zip(t, want):
        assert np.array_equal(host(got).reshape(x.shape), x)


@pytest.mark.parametrize("paged", [False, True])
def test_keep_leaves_a_bad_sequence(reef, paged):
    """Rows that do not ascend or lie outside, lengths outside, a page outside: that sequence
    stays, its neighbours are served, and the status says so."""
    print(f"\n[case] keep refusals paged {paged}", flush=True)
    rng = np.random.default_rng(5)
    B, H, D, T, blocks = 8, 2, 64, 4, 6
    lens = i32([40, 40, 40, 40, 3, 97, 40, 40])
    kept = i32([[1, 3, 0, 0], [3, 1, 0, 0], [1, 4, 0, 0], [-1, 2, 0, 0], [1, 2, 0, 0], [1, 2, 0, 0],
                [1, 2, 0, 0], [2, 2, 0, 0]])
    n = i32([2, 2, 2, 2, 2, 2, 5, 2])
    table = i32(rng.permutation(60)[:B * blocks].reshape(B, blocks))
    if paged:
        pools = pool(rng, (60, H), D)
    else:
        pools = pool(rng, (B, H, blocks), D)
    status = reef.StatusWord()
    if paged:
        t = [gpu(x) for x in pools]
        new = reef.kv_keep_paged(gpu(kept), gpu(n), gpu(lens), gpu(table), *t, status=status)
    else:
        k, v, ks, vs = pools
        t = [gpu(k.reshape(B, H, -1, D)), gpu(v), gpu(ks.reshape(B, H, -1)), gpu(vs.reshape(B, H, -1))]
        new = reef.kv_keep(gpu(kept), gpu(n), gpu(lens), *t, status=status)
    assert host(new).tolist() == [38] + lens[1:].tolist()
    with pytest.raises(reef.InvalidArgument):
        status.check("keep")
    k0 = host(t[0]).reshape(pools[0].shape)
    for b in range(1, B):
        rows = table[b] if paged else b
        assert np.array_equal(k0[rows], pools[0][rows])
    rows = table[0] if paged else 0
    assert not np.array_equal(k0[rows], pools[0][rows])
    if paged:
        status = reef.StatusWord()
        table[0, 2] = 60
        t = [gpu(x) for x in pools]
        new = reef.kv_keep_paged(gpu(kept[:1]), gpu(n[:1]), gpu(lens[:1]), gpu(table[:1]), *t, status=status)
        assert int(new) == 40 and np.array_equal(host(t[0]), pools[0])
        with pytest.raises(reef.InvalidArgument):
            status.check("keep")


def test_what_is_past_the_ends_is_flagged(reef):
    print("\n[case] page bookkeeping: indices and pages past the ends", flush=True)
    m = Model(3, 4, 10)
    m.table[0, :2], m.lens[0], m.refs[:2] = [0, 1], 20, 1
    table, lens, refs = m.device()

    def refused(f, error):
        status = reef.StatusWord()
        out = f(status)
        with pytest.raises(error):
            status.check("pages")
        m.check(table, lens, refs)
        return out

    refused(lambda s: reef.kv_free(gpu(i32([3])), table, lens, refs, status=s), reef.InvalidArgument)
    refused(lambda s: reef.kv_fork(gpu(i32([0, 7])), gpu(i32([3, 1])), table, lens, refs, status=s),
            reef.InvalidArgument)
    lens[0] = m.lens[0] = 65  # beyond the table
    refused(lambda s: reef.kv_fork(gpu(i32([0])), gpu(i32([1])), table, lens, refs, status=s),
            reef.InvalidArgument)
    m.lens[:] = [65, 64, -1]
    lens.copy_(gpu(m.lens))
    refused(lambda s: reef.kv_reserve(table, lens, refs, 1, status=s), reef.CapacityError)
    pools = [gpu(x) for x in pool(np.random.default_rng(0), (10, 2), 64)]
    was = [x.clone() for x in pools]
    refused(lambda s: reef.kv_copy_pages(gpu(i32([0, 10])), gpu(i32([10, 0])), *pools, status=s),
            reef.InvalidArgument)
    assert all(torch.equal(x, y) for x, y in zip(pools, was))
    # a page that the counts do not know is not given back
    t2, r2 = gpu(i32([[5, 11, -1, -1]])), gpu(np.zeros(10, np.int32))
    status = reef.StatusWord()
    reef.kv_free(gpu(i32([0])), t2, gpu(i32([17])), r2, status=status)
    assert not host(r2).any() and (host(t2) == -1).all()
    with pytest.raises(reef.InvalidArgument):
        status.check("free")


def test_a_step_of_a_search_in_a_graph(reef):
    """free, fork, reserve and copy captured once: replays on the restored state give the
    eager result each time."""
    print("\n[case] search step in a graph", flush=True)
    rng = np.random.default_rng(3)
    B, H, D, P = 12, 2, 64, 120
    m = Model(B, 8, P)
    m.lens[:6] = [5, 16, 31, 40, 64, 77]
    for b in range(6):
        n = -(-m.lens[b] // PAGE)
        m.table[b, :n] = rng.permutation(np.flatnonzero(m.refs == 0))[:n]
        m.refs[m.table[b, :n]] = 1
    start, pools = m.device(), [gpu(x) for x in pool(rng, (P, H), D)]
    state = [x.clone() for x in start]
    work = [x.clone() for x in pools]
    parents, children = gpu(i32([0, 0, 3, 4, 5, 1])), gpu(i32([6, 7, 8, 9, 10, 11]))
    status = reef.StatusWord()

    def step():
        table, lens, refs = state
        reef.kv_free(children, table, lens, refs, status=status)
        reef.kv_fork(parents, children, table, lens, refs, status=status)
        src, dst = reef.kv_reserve(table, lens, refs, 2, status=status)
        reef.kv_copy_pages(src, dst, *work, status=status)

    def restore():
        for x, y in zip(state + work, list(start) + pools):
            x.copy_(y)

    step()
    eager = [x.clone() for x in state + work]
    m.free(host(children))
    m.fork(host(parents), host(children))
    m.reserve(2)
    m.check(*state)
    restore()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        restore()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(state + work, eager))
        restore()
        step()
        assert all(torch.equal(x, y) for x, y in zip(state + work, eager))
    status.check("graph")


@pytest.mark.parametrize("pages,entries", [(300_001, 180_000), (1_048_576, 400_000), (262_144, 262_144)])
def test_compact_of_a_large_pool(reef, pages, entries):
    """More chunks of pages than a workgroup has threads; a tenth of the entries shared; the last
    pool is full."""
    print(f"\n[case] compact {pages} pages, {entries} entries", flush=True)
    rng = np.random.default_rng(pages)
    m = Model(64, -(-entries // 64), pages)
    flat = m.table.reshape(-1)
    flat[:entries] = rng.permutation(pages)[:entries]
    if entries < pages:
        flat[rng.permutation(entries)[:entries // 10]] = flat[0]
    rng.shuffle(flat)
    m.refs[:] = np.bincount(flat[flat >= 0], minlength=pages)
    table, _, refs = m.device()
    for _ in range(2):  # the second time there is nothing to move
        src, dst, live = m.compact()
        s, d, n = reef.kv_compact(table, refs)
        assert int(n) == live
        assert np.array_equal(host(s), src) and np.array_equal(host(d), dst)
        m.check(table, None, refs)


def test_page_calls_without_work_and_refusals(reef):
    """Empty lists do nothing; what does not match is refused before a launch."""
    print("\n[case] page refusals", flush=True)
    m = Model(4, 3, 20)
    m.reserve(5)
    m.lens[:] = 5
    table, lens, refs = m.device()
    none, one = gpu(i32([])), gpu(i32([1]))
    reef.kv_free(none, table, lens, refs)
    reef.kv_fork(none, none, table, lens, refs)
    m.check(table, lens, refs)
    for n in (0, -1):
        with pytest.raises(reef.InvalidArgument):
            reef.kv_reserve(table, lens, refs, n)
    for n in (49, 1 << 40):
        with pytest.raises(reef.CapacityError):
            reef.kv_reserve(table, lens, refs, n)
    for call in (lambda: reef.kv_free(one.long(), table, lens, refs),
                 lambda: reef.kv_free(one, table[:, ::2], lens, refs),
                 lambda: reef.kv_free(one, table, lens[:3], refs),
                 lambda: reef.kv_free(one, table.view(-1), lens, refs),
                 lambda: reef.kv_fork(one, gpu(i32([2, 3])), table, lens, refs),
                 lambda: reef.kv_reserve(table, lens, refs.view(4, 5), 1),
                 lambda: reef.kv_compact(table, refs.cpu())):
        with pytest.raises(reef.InvalidArgument):
            call()
    m.check(table, lens, refs)
