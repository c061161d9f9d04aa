"""Operators of a layer's step over drafted tokens in int8, timed in their plain form and
as the library runs them:

  tree     attention of a tree of drafted tokens over a filled int8 cache
  keep     the accepted tokens' rows moved to their places in the cache
  beams    a step of a search: the losers' pages freed, the winners forked, room made
           for the next token, and the shared last pages copied
  compact  a page pool's live pages moved to its front
  norm     root-mean-square norm of a residual sum, as int8 rows with scales
  product  the W8A8 product with bias, activation and residual

`run` takes elementary torch operations where `own` is false and the library's calls
where it is true. Cache pages are moved, not computed: they come back as the bytes they
are. The norm's int8 rows come back as the values they stand for.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 16
ACTIVATIONS = ("none", "relu", "gelu_tanh", "gelu_erf", "silu")
# Drawn cases cost no more than the largest listed ones of their kind.
_CACHE = {"bytes": 6e8, "flops": 4e10}  # 64 sequences x 8 heads x 4096 tokens x 128
MOST = {"tree": _CACHE, "keep": _CACHE, "beams": _CACHE, "compact": _CACHE,
        "norm": {"bytes": 1.1e9, "flops": 1e9}, "product": {"bytes": 6e8, "flops": 5.6e11}}


def listed():
    return [
        # One conversation of a small model: eight drafted tokens, a short cache, one launch.
        {"name": "tree_1x12x64_t8_l200", "kind": "tree", "batch": 1, "q_heads": 12,
         "kv_heads": 12, "head_dim": 64, "drafts": 8, "context": 200, "min_context": 200,
         "window": 0, "paged": False, "chain": False, "padded": False},
        # A chain of three drafted tokens for a full batch over long caches: bound by the
        # cache's bytes, as a decode step is.
        {"name": "tree_64x32x128_t3_l4096", "kind": "tree", "batch": 64, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "drafts": 3, "context": 4096, "min_context": 4096,
         "window": 0, "paged": False, "chain": True, "padded": False},
        # Trees of sixteen over pages, sequences of very different lengths, some with
        # fewer drafted tokens.
        {"name": "tree_paged_16x32x128_t16", "kind": "tree", "batch": 16, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "drafts": 16, "context": 8192, "min_context": 512,
         "window": 0, "paged": True, "chain": False, "padded": True},
        # Wide trees on one tensor-parallel rank of a 70B-sized layer: 512 query rows a
        # key head, bound by the products and the softmax.
        {"name": "tree_paged_32x8x128_t64", "kind": "tree", "batch": 32, "q_heads": 8,
         "kv_heads": 1, "head_dim": 128, "drafts": 64, "context": 8192, "min_context": 512,
         "window": 0, "paged": True, "chain": False, "padded": False},
        # The accepted tokens of those trees, on one layer's cache.
        {"name": "keep_paged_64x8x128_t16", "kind": "keep", "batch": 64, "kv_heads": 8,
         "head_dim": 128, "drafts": 16, "context": 4096, "min_context": 512, "paged": True},
        # A search step of 64 beams, and the pool of a long-running server after many
        # sequences have ended: the ends of the page operators' range.
        {"name": "beams_64x8x128", "kind": "beams", "pairs": 64, "kv_heads": 8, "head_dim": 128,
         "context": 1024, "min_context": 77, "tokens": 1},
        {"name": "compact_8192x8x128", "kind": "compact", "pages": 8192, "live": 0.55,
         "batch": 64, "kv_heads": 8, "head_dim": 128},
        # A decode batch's rows, a prompt's rows, and rows of an odd width.
        {"name": "norm_7x2048", "kind": "norm", "rows": 7, "width": 2048, "residual": True},
        {"name": "norm_8192x8192", "kind": "norm", "rows": 8192, "width": 8192, "residual": True},
        {"name": "norm_1021x5003", "kind": "norm", "rows": 1021, "width": 5003, "residual": False},
        # The projections of an MLP: up with its activation for a batch of drafted tokens,
        # down with the residual for a prompt.
        {"name": "product_48x4096x6144_gelu", "kind": "product", "rows": 48, "in": 4096,
         "out": 6144, "bias": True, "activation": "gelu_tanh", "residual": False},
        {"name": "product_4096x8192x8192_residual", "kind": "product", "rows": 4096, "in": 8192,
         "out": 8192, "bias": True, "activation": "none", "residual": True},
    ]


def draw(rng):
    def spread(low, high):
        x = math.exp(rng.uniform(math.log(low), math.log(high + 1)))
        return min(high, max(low, int(x)))

    kind = rng.choice(["tree", "tree", "tree", "keep", "beams", "compact", "norm", "norm",
                       "product", "product"])
    while True:
        kv = rng.choice([1, 1, 2, 4, 8, 12, 16])
        heads = kv * (rng.choice([1, 2, 4, 8]) if kv <= 8 else 1)
        case = {"kind": kind, "kv_heads": kv, "head_dim": rng.choice([64, 128, 128])}
        if kind in ("tree", "keep"):
            drafts = spread(1, 64)
            top = max(drafts, spread(64, 8192))
            case.update(batch=spread(1, 64), drafts=drafts, context=top,
                        min_context=rng.choice([top, max(drafts, spread(1, top))]),
                        paged=rng.random() < 0.6)
            if kind == "tree":
                case.update(q_heads=heads, window=rng.choice([0, 0, 0, spread(16, 2048)]),
                            chain=rng.random() < 0.3, padded=rng.random() < 0.3)
        elif kind == "beams":
            top = spread(32, 4096)
            case.update(pairs=spread(1, 128), context=top, min_context=spread(1, top),
                        tokens=rng.choice([1, 1, 3, spread(1, 64)]))
        elif kind == "compact":
            case.update(pages=spread(64, 8192), live=round(rng.uniform(0.2, 0.9), 3),
                        batch=spread(1, 64))
        elif kind == "norm":
            case = {"kind": kind, "rows": spread(1, 8192), "width": spread(48, 16384),
                    "residual": rng.random() < 0.7}
        else:
            case = {"kind": kind, "rows": spread(1, 8192), "in": 16 * spread(16, 512),
                    "out": spread(64, 8192), "bias": rng.random() < 0.6,
                    "activation": rng.choice(ACTIVATIONS), "residual": rng.random() < 0.5}
        cost, most = work(case), MOST[kind]
        pages = case.get("pages", 0)
        if kind in ("tree", "keep", "beams"):  # the cache, where a pass reads a part of it
            sequences = 2 * case["pairs"] if kind == "beams" else case["batch"]
            pages = sequences * (case["context"] // PAGE + 1)
        held = pages * _page_bytes(case) if pages else 0
        if max(held, cost["bytes"]) <= most["bytes"] and cost["flops"] <= most["flops"]:
            return case


# --- inputs ---------------------------------------------------------------------------

def _page_bytes(case):
    return PAGE * case["kv_heads"] * (2 * case["head_dim"] + 8)


def _codes(x, dims):
    scale = x.abs().amax(dim=dims, keepdim=True) / 127.0
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return torch.round(x / scale).clamp_(-127, 127).to(torch.int8), scale


def _pool(g, case, lead):
    """Keys, values (transposed pages) and their scales of pages [*lead, H]."""
    H, D = case["kv_heads"], case["head_dim"]
    k, ks = _codes(torch.randn((*lead, H, PAGE, D), generator=g, device="cuda"), (-1,))
    v, vs = _codes(torch.randn((*lead, H, PAGE, D), generator=g, device="cuda"), (-1,))
    return {"k": k, "v": v.transpose(-1, -2).contiguous(), "ks": ks.squeeze(-1).contiguous(),
            "vs": vs.squeeze(-1).contiguous()}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 32))
    kind = case["kind"]
    st = {"case": case}

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).cuda()

    if kind == "norm":
        # a sublayer's output and the residual stream, whose channels differ in size
        shape = (case["rows"], case["width"])
        size = 0.5 + torch.rand(case["width"], generator=g, device="cuda")
        st["x"] = torch.randn(shape, generator=g, device="cuda") * 0.3
        if case["residual"]:
            st["r"] = torch.randn(shape, generator=g, device="cuda") * size
        st["w"] = 0.5 + torch.rand(case["width"], generator=g, device="cuda")
        return st
    if kind == "product":
        rows, fin, fout = case["rows"], case["in"], case["out"]
        st["x"], xs = _codes(torch.randn((rows, fin), generator=g, device="cuda"), (1,))
        w = torch.randn((fout, fin), generator=g, device="cuda") / math.sqrt(fin)
        st["w"], ws = _codes(w, (1,))
        st["xs"], st["ws"] = xs.reshape(-1).contiguous(), ws.reshape(-1).contiguous()
        st["bias"] = torch.randn(fout, generator=g, device="cuda") if case["bias"] else None
        st["r"] = (torch.randn((rows, fout), generator=g, device="cuda") if case["residual"]
                   else None)
        return st
    if kind == "beams":
        # rows 0 .. n - 1 of the table are the beams that go on, the others their forks
        n, top = case["pairs"], case["context"]
        lens = host.randint(case["min_context"], top + 1, n)
        blocks = -(-(top + case["tokens"]) // PAGE) + 1
        used = -(-lens // PAGE)
        pages = n * -(-top // PAGE) + 2 * n * (case["tokens"] // PAGE + 3)
        order = host.permutation(pages)[:int(used.sum())]
        table = np.full((2 * n, blocks), -1, np.int32)
        table[:n][np.arange(blocks)[None, :] < used[:, None]] = order
        refs = np.zeros(pages, np.int32)
        refs[order] = 1
        st.update(_pool(g, case, (pages,)), table=ints(table), refs=ints(refs),
                  lens=ints(np.concatenate([lens, np.zeros(n, lens.dtype)])),
                  parents=ints(host.randint(0, n, n)), children=ints(n + np.arange(n)))
        return st
    if kind == "compact":
        # sequences of unequal lengths whose pages are scattered over the pool; a few are
        # shared by two sequences
        pages, n = case["pages"], case["batch"]
        live = max(1, int(case["live"] * pages))
        order = host.permutation(pages)[:live]
        shared = host.permutation(live)[:live // 16]
        entries = np.concatenate([order, order[shared]])
        entries = entries[host.permutation(len(entries))]
        blocks = -(-len(entries) // n)
        table = np.full(n * blocks, -1, np.int32)
        table[:len(entries)] = entries
        refs = np.zeros(pages, np.int32)
        np.add.at(refs, entries, 1)
        st.update(_pool(g, case, (pages,)), table0=ints(table.reshape(n, blocks)),
                  refs0=ints(refs), table=ints(table.reshape(n, blocks)), refs=ints(refs))
        return st

    # tree, keep: a filled cache with every sequence's drafted tokens at its end
    B, H, T = case["batch"], case["kv_heads"], case["drafts"]
    lens = host.randint(case["min_context"], case["context"] + 1, B)
    blocks = -(-case["context"] // PAGE)
    st["lens"] = ints(lens)
    if case["paged"]:
        used = B * blocks
        pages = used + max(1, used // 4)
        st.update(_pool(g, case, (pages,)), table=ints(host.permutation(pages)[:used]).view(B, blocks))
    else:
        c = _pool(g, case, (B, blocks))
        c = {n: t.transpose(1, 2).contiguous() for n, t in c.items()}  # [B, H, blocks, ...]
        L = blocks * PAGE
        st.update(k=c["k"].view(B, H, L, -1), v=c["v"], ks=c["ks"].view(B, H, L),
                  vs=c["vs"].view(B, H, L), table=None)
    # every drafted token continues an earlier one, or the last of the cached tokens
    counts = host.randint(1, T + 1, B) if case.get("padded") else np.full(B, T)
    parent = np.array([[host.randint(-1, max(0, i)) if i else -1 for i in range(T)] for _ in range(B)])
    if case.get("chain"):
        parent = np.tile(np.arange(T) - 1, (B, 1))
    masks = np.zeros((B, T), np.uint64)
    for b in range(B):
        for i in range(counts[b]):
            up = masks[b, parent[b, i]] if parent[b, i] >= 0 else np.uint64(0)
            masks[b, i] = up | (np.uint64(1) << np.uint64(i))
    if kind == "tree":
        q, qs = _codes(torch.randn((B, case["q_heads"], T, case["head_dim"]), generator=g,
                                   device="cuda"), (-1,))
        st["q"], st["qs"] = q, qs.squeeze(-1).contiguous()
        st["mask"] = torch.from_numpy(masks.view(np.int64)).cuda()
        return st
    # keep: the path to a random drafted token was accepted
    kept, count = np.full((B, T), -1), np.zeros(B)
    for b in range(B):
        last = int(masks[b, host.randint(T)])
        path = [j for j in range(T) if last >> j & 1]
        kept[b, :len(path)] = path
        count[b] = len(path)
    st["kept"], st["count"] = ints(kept), ints(count)
    return st


# --- the plain forms -------------------------------------------------------------------

def _softmax_scale(case):
    return 1.0 / math.sqrt(case["head_dim"])


def _token_major(st, B, H, D):
    """The cache's keys and values, float32 [B, H, tokens, D], with their scales applied."""
    k, v, ks, vs, table = st["k"], st["v"], st["ks"], st["vs"], st["table"]
    if table is None:
        v = v.transpose(3, 4).reshape(B, H, -1, D)
    else:
        at = table.long()
        k = k[at].transpose(1, 2).reshape(B, H, -1, D)
        v = v[at].permute(0, 2, 1, 4, 3).reshape(B, H, -1, D)
        ks, vs = ks[at].transpose(1, 2).reshape(B, H, -1), vs[at].transpose(1, 2).reshape(B, H, -1)
    return k.float() * ks[..., None], v.float() * vs[..., None]


def _bits(mask, T):
    return (mask[:, :, None] >> torch.arange(T, device=mask.device)) & 1


def _plain_tree(st):
    case = st["case"]
    B, Hq, H, D, T = (case["batch"], case["q_heads"], case["kv_heads"], case["head_dim"],
                      case["drafts"])
    k, v = _token_major(st, B, H, D)
    L = k.shape[2]
    q = (st["q"].float() * st["qs"][..., None]).view(B, H, Hq // H * T, D)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * _softmax_scale(case)
    seen = _bits(st["mask"], T)                             # [B, T, T]
    depth = seen.sum(2)
    key = torch.arange(L, device=q.device)
    draft = key[None, :] - (st["lens"].long() - T)[:, None]  # [B, L]: drafted token of a key
    at = draft.clamp(0, T - 1)
    drafted = torch.gather(seen, 2, at[:, None, :].expand(B, T, L)) == 1
    visible = (draft < 0)[:, None, :] | ((draft < T)[:, None, :] & drafted)
    if case["window"]:
        # positions behind the last token before the drafts
        pos = torch.where(draft < 0, draft, torch.gather(depth, 1, at) - 1)
        visible &= pos[:, None, :] > (depth - 1)[:, :, None] - case["window"]
    visible &= (depth > 0)[:, :, None]
    s = s.view(B, H, Hq // H, T, L).masked_fill(~visible[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    return torch.matmul(p.view(B, H, -1, L), v).view(B, Hq, T, D)


def _plain_keep(st):
    case = st["case"]
    T = case["drafts"]
    first = (st["lens"] - T).long()[:, None]
    i = torch.arange(T, device=first.device)[None, :]
    valid = i < st["count"][:, None]
    source, place = first + torch.where(valid, st["kept"].long(), i), first + i
    if st["table"] is None:
        b = torch.arange(case["batch"], device=first.device)[:, None]
        k, ks, vs = st["k"][b, :, source], st["ks"][b, :, source], st["vs"][b, :, source]
        v = st["v"][b, :, source // PAGE, :, source % PAGE]
        st["k"][b, :, place], st["ks"][b, :, place], st["vs"][b, :, place] = k, ks, vs
        st["v"][b, :, place // PAGE, :, place % PAGE] = v
    else:
        table = st["table"].long()
        sp, ss = torch.gather(table, 1, source // PAGE), source % PAGE
        pp, ps = torch.gather(table, 1, place // PAGE), place % PAGE
        k, ks, vs = st["k"][sp, :, ss], st["ks"][sp, :, ss], st["vs"][sp, :, ss]
        v = st["v"][sp, :, :, ss]
        st["k"][pp, :, ps], st["ks"][pp, :, ps], st["vs"][pp, :, ps] = k, ks, vs
        st["v"][pp, :, :, ps] = v
    return st["lens"] - T + st["count"]


def _count_pages(refs, pages, by):
    """refs[p] += by for every page of `pages` that is one (-1: none)."""
    pages = pages.reshape(-1)
    at = torch.where(pages >= 0, pages, torch.zeros_like(pages)).long()
    refs.index_add_(0, at, torch.where(pages >= 0, by, 0).to(torch.int32))


def _copy_pages(st, source, place):
    """Page source[i] to place[i] where place[i] is a page. The other pairs repeat the first
    one that is (page 0 onto itself where none is): the same bytes once more."""
    valid = place >= 0
    first = valid.int().argmax()
    source = torch.where(valid, source, source[first]).clamp(min=0).long()
    place = torch.where(valid, place, place[first]).clamp(min=0).long()
    source = torch.where(valid.any(), source, place)
    for name in ("k", "v", "ks", "vs"):
        st[name][place] = st[name][source]


def _plain_beams(st):
    case, table, refs, lens = st["case"], st["table"], st["refs"], st["lens"]
    parents, children = st["parents"].long(), st["children"].long()
    # free the children of the last step
    _count_pages(refs, table[children], -1)
    table[children] = -1
    lens[children] = 0
    # fork
    block = torch.arange(table.shape[1], device=table.device)
    rows = table[parents]
    rows = torch.where(block[None, :] < ((lens[parents] + PAGE - 1) // PAGE)[:, None], rows, -1)
    _count_pages(refs, rows, 1)
    table[children] = rows
    lens[children] = lens[parents]
    # room for the next tokens: the blocks from the one that the next token falls in; an
    # absent or shared page is replaced, lowest free pages first
    nb = (case["tokens"] + PAGE - 2) // PAGE + 1
    at = lens.long()[:, None] // PAGE + torch.arange(nb, device=table.device)[None, :]
    due = at * PAGE < lens.long()[:, None] + case["tokens"]
    at = at.clamp(max=table.shape[1] - 1)
    old = torch.gather(table, 1, at)
    shared = (old >= 0) & (refs[old.clamp(min=0).long()] > 1)
    due &= (old < 0) | shared
    rank = torch.cumsum(due.reshape(-1).long(), 0).view(due.shape) - 1
    free = refs == 0
    order = torch.where(free, torch.cumsum(free.long(), 0) - 1, refs.numel())
    pages = torch.full((refs.numel() + 1,), -1, dtype=torch.int32, device=table.device)
    pages.scatter_(0, order, torch.arange(refs.numel(), dtype=torch.int32, device=table.device))
    new = torch.where(due, pages[rank.clamp(0, refs.numel() - 1)], -1)
    table.scatter_(1, at, torch.where(due, new, old))
    _count_pages(refs, new, 1)
    _count_pages(refs, torch.where(due & shared, old, -1), -1)
    holds = due & shared & (at * PAGE < lens.long()[:, None])
    _copy_pages(st, old[:, 0], torch.where(holds[:, 0], new[:, 0], -1))
    return [table, refs, lens, st["k"], st["v"], st["ks"], st["vs"]]


def _plain_compact(st):
    table, refs = st["table"].copy_(st["table0"]), st["refs"].copy_(st["refs0"])
    page = torch.arange(refs.numel(), device=refs.device)
    live = refs > 0
    before = torch.cumsum(live.long(), 0)
    count = before[-1]
    # the k-th live page from the pool's end takes the k-th free place from its front
    moves, hole = live & (page >= count), ~live & (page < count)
    spare = refs.numel()
    source = torch.full((spare + 1,), -1, dtype=torch.int32, device=refs.device)
    place = torch.full((spare + 1,), -1, dtype=torch.int32, device=refs.device)
    source.scatter_(0, torch.where(moves, count - before, spare), page.int())
    place.scatter_(0, torch.where(hole, page - before, spare), page.int())
    source, place = source[:spare // 2], place[:spare // 2]
    to = torch.where(moves, place[(count - before).clamp(0, max(spare // 2 - 1, 0))], page.int())
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], -1))
    there = torch.where(hole, refs[source[(page - before).clamp(0, max(spare // 2 - 1, 0))].clamp(min=0).long()], refs)
    refs.copy_(torch.where(moves, 0, there))
    _copy_pages(st, source, place)
    return [table, refs, st["k"], st["v"], st["ks"], st["vs"]]


def _plain_norm(st):
    h = st["x"] + st["r"] if "r" in st else st["x"]
    # the codes are whole numbers: 64 bits up to their rounding, so that none falls on the
    # other side of a half
    d = h.double()
    y = d * st["w"].double() * torch.rsqrt((d * d).mean(1, keepdim=True) + 1e-6)
    scale = (y.abs().amax(1, keepdim=True) / 127).float()
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    values = torch.round(y / scale.double()).float() * scale
    return [values, scale.reshape(-1), h] if "r" in st else [values, scale.reshape(-1)]


def _plain_product(st):
    activation = st["case"]["activation"]
    y = torch.matmul(st["x"].float(), st["w"].float().t()) * (st["xs"][:, None] * st["ws"])
    if st["bias"] is not None:
        y = y + st["bias"]
    if activation == "relu":
        y = torch.where(y > 0, y, torch.zeros_like(y))
    elif activation == "gelu_tanh":
        y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    elif activation == "gelu_erf":
        y = 0.5 * y * torch.erfc(y * -math.sqrt(0.5))
    elif activation == "silu":
        y = y / (1 + torch.exp(-y))
    return y if st["r"] is None else y + st["r"]


# --- the library's calls -----------------------------------------------------------------

def _own(st):
    import reef_amd as reef

    case, kind = st["case"], st["case"]["kind"]
    if "status" not in st:
        st["status"] = reef.StatusWord("cuda")
    status = st["status"]
    if kind == "tree":
        cache = [st[n] for n in ("k", "v", "ks", "vs")]
        if st["table"] is None:
            return reef.attention_decode_tree(st["q"], st["qs"], *cache, st["lens"],
                                              tree_mask=st["mask"], window=case["window"],
                                              status=status)
        return reef.attention_decode_tree_paged(st["q"], st["qs"], *cache, st["table"], st["lens"],
                                                tree_mask=st["mask"], window=case["window"],
                                                status=status)
    if kind == "keep":
        if st["table"] is None:
            lens = reef.kv_keep(st["kept"], st["count"], st["lens"], st["k"], st["v"], st["ks"],
                                st["vs"], status=status)
        else:
            lens = reef.kv_keep_paged(st["kept"], st["count"], st["lens"], st["table"], st["k"],
                                      st["v"], st["ks"], st["vs"], status=status)
        return [lens, st["k"], st["v"], st["ks"], st["vs"]]
    if kind == "beams":
        table, refs, lens = st["table"], st["refs"], st["lens"]
        reef.kv_free(st["children"], table, lens, refs, status=status)
        reef.kv_fork(st["parents"], st["children"], table, lens, refs, status=status)
        source, place = reef.kv_reserve(table, lens, refs, case["tokens"], status=status)
        reef.kv_copy_pages(source, place, st["k"], st["v"], st["ks"], st["vs"], status=status)
        return [table, refs, lens, st["k"], st["v"], st["ks"], st["vs"]]
    if kind == "compact":
        table, refs = st["table"].copy_(st["table0"]), st["refs"].copy_(st["refs0"])
        source, place, _ = reef.kv_compact(table, refs, status=status)
        reef.kv_copy_pages(source, place, st["k"], st["v"], st["ks"], st["vs"], status=status)
        return [table, refs, st["k"], st["v"], st["ks"], st["vs"]]
    if kind == "norm":
        q, scale, *h = reef.rmsnorm_quantize(st["x"], st["w"], residual=st.get("r"), eps=1e-6,
                                             status=status)
        return [reef.dequantize(q, scale, case["width"]), scale, *h]
    return reef.gemm_w8a8(st["x"], st["xs"], st["w"], st["ws"], st["bias"],
                          activation=case["activation"], residual=st["r"], status=status)


def run(st):
    if own:
        return _own(st)
    kind = st["case"]["kind"]
    if kind == "tree":
        return _plain_tree(st)
    if kind == "keep":
        return [_plain_keep(st), st["k"], st["v"], st["ks"], st["vs"]]
    if kind == "beams":
        return _plain_beams(st)
    if kind == "compact":
        return _plain_compact(st)
    return _plain_norm(st) if kind == "norm" else _plain_product(st)


# --- what a pass cannot do without -------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "norm":  # values, the row scales, and the sum where there is a residual
        n = case["rows"] * case["width"]
        return {"bytes": n * (16 if case["residual"] else 8) + 4 * case["rows"] + 4 * case["width"],
                "flops": 8 * n}
    if kind == "product":
        r, i, o = case["rows"], case["in"], case["out"]
        return {"bytes": r * i + o * i + 4 * (r + o) + (4 * o if case["bias"] else 0)
                + 4 * r * o * (2 if case["residual"] else 1), "flops": 2 * r * i * o}
    H, D = case["kv_heads"], case["head_dim"]
    if kind == "compact":
        moved = (case["live"] - case["live"] ** 2) * case["pages"]  # the live ones at the back
        return {"bytes": 2 * moved * _page_bytes(case) + 16 * case["pages"] * (1 + case["live"]),
                "flops": 0}
    mean = (case["context"] + case["min_context"]) / 2
    if kind == "beams":
        n = case["pairs"]
        copied = 2 * n * 15 / 16  # both sharers' last pages, unless full
        tables = 4 * n * (mean / PAGE) * 8
        return {"bytes": 2 * copied * _page_bytes(case) + tables, "flops": 0}
    B, T = case["batch"], case["drafts"]
    if kind == "keep":  # about the logarithm of the tree's size are kept
        return {"bytes": 2 * B * H * (2 * D + 8) * math.log(T + 1) + 8 * B * T, "flops": 0}
    tokens = B * (min(mean, T + case["window"]) if case["window"] else mean)
    return {"bytes": tokens * H * (2 * D + 8) + B * case["q_heads"] * T * (5 * D + 4) + 8 * B * T,
            "flops": 4 * tokens * case["q_heads"] * T * D}


# --- the same in 64 bits -----------------------------------------------------------------

def exact(case, seed):
    kind = case["kind"]
    if kind in ("keep", "beams", "compact"):
        return None  # bytes and whole numbers, computed from no others
    st = prepare(case, seed)
    if kind == "norm":
        h = st["x"].double() + st["r"].double() if "r" in st else st["x"].double()
        total = h.float().double()  # the sum as the residual stream holds it
        length = (total.square().sum(1) / case["width"] + 1e-6).sqrt()
        y = total / length[:, None] * st["w"].double()
        scale = (y.abs().max(1).values / 127).float().double()
        values = torch.round(y / scale[:, None]) * scale[:, None]
        return [values, y.abs().max(1).values / 127] + ([h] if "r" in st else [])
    if kind == "product":
        y = (st["x"].double() @ st["w"].double().t()) * st["xs"].double()[:, None] * st["ws"].double()
        y = y + st["bias"].double() if case["bias"] else y
        if case["activation"] == "relu":
            y = y.clamp(min=0)
        elif case["activation"] == "gelu_tanh":
            y = torch.nn.functional.gelu(y, approximate="tanh")
        elif case["activation"] == "gelu_erf":
            y = torch.nn.functional.gelu(y)
        elif case["activation"] == "silu":
            y = torch.nn.functional.silu(y)
        return y + st["r"].double() if case["residual"] else y
    # tree: sequence by sequence, key head by key head, over the keys that it has
    B, Hq, H, D, T = (case["batch"], case["q_heads"], case["kv_heads"], case["head_dim"],
                      case["drafts"])
    G, lens, masks = Hq // H, st["lens"].tolist(), st["mask"].tolist()
    out = torch.zeros((B, Hq, T, D), dtype=torch.float64, device="cuda")
    for b in range(B):
        n, prefix = lens[b], lens[b] - T
        depth = [bin(m & (1 << T) - 1).count("1") - 1 for m in masks[b]]
        tail = torch.tensor([[bool(m >> j & 1) and (not case["window"] or depth[j] > depth[i] - case["window"])
                              for j in range(T)] for i, m in enumerate(masks[b])], device="cuda")
        where = torch.arange(prefix, device="cuda")[None, :] - prefix
        first = torch.tensor(depth, device="cuda")[:, None] - (case["window"] or 1 << 40)
        shown = torch.cat([(where > first), tail], 1)
        shown &= torch.tensor(masks[b], device="cuda")[:, None] != 0
        hidden = torch.zeros((T, n), dtype=torch.float64, device="cuda").masked_fill_(~shown, -math.inf)
        some = shown.any(1)
        if not bool(some.any()):
            continue
        if case["paged"]:
            pages = st["table"][b, :-(-n // PAGE)].long()
        for h in range(H):
            if case["paged"]:
                k, v = st["k"][pages, h].reshape(-1, D)[:n], st["v"][pages, h].transpose(1, 2).reshape(-1, D)[:n]
                ks, vs = st["ks"][pages, h].reshape(-1)[:n], st["vs"][pages, h].reshape(-1)[:n]
            else:
                k, ks, vs = st["k"][b, h, :n], st["ks"][b, h, :n], st["vs"][b, h, :n]
                v = st["v"][b, h].transpose(1, 2).reshape(-1, D)[:n]
            k, v = k.double() * ks.double()[:, None], v.double() * vs.double()[:, None]
            q = st["q"][b, h * G:(h + 1) * G].double() * st["qs"][b, h * G:(h + 1) * G, :, None].double()
            s = (q.reshape(G * T, D) @ k.t() / math.sqrt(D)).view(G, T, n) + hidden
            p = torch.softmax(s[:, some], 2)
            out[b, h * G:(h + 1) * G, some] = (p.view(-1, n) @ v).view(G, -1, D)
    return out
