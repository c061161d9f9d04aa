"""Operators of steps that read less of the cache, timed in their plain form and as the
library runs them:

  append  new tokens quantized to 4 bits into the cache, read back
  decode  attention of one token per sequence over a cache held in 4 bits
  chunk   attention of a prompt's chunk over the 4-bit cache that holds it
  bounds  largest and least key of every channel of the pages that new tokens fall in
  step    the pages that a query's score against those bounds selects, and attention over
          them alone, in 8 and 4 bits

`run` takes elementary torch operations where `own` is false and the library's calls where
it is true. Cache rows and bounds come back as the values they stand for.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 16
# Drawn cases cost no more than the largest listed ones of their kind. (A cache of 64
# sequences x 8 heads x 4096 tokens x 128 in 4 bits, one of 16 x 8 x 32768 in 8.)
MOST = {"append": {"bytes": 3e8, "flops": 1e9}, "decode": {"bytes": 3.2e8, "flops": 4e10},
        "chunk": {"bytes": 2e8, "flops": 1.6e11}, "bounds": {"bytes": 1.8e8, "flops": 1e9},
        "step": {"bytes": 1.2e9, "flops": 4e10}}


def listed():
    return [
        # A decode step's new tokens of a full batch, into pages.
        {"name": "append_paged_64x8x128_t1", "kind": "append", "batch": 64, "kv_heads": 8,
         "head_dim": 128, "tokens": 1, "context": 64, "paged": True},
        # Prompts, an odd number of tokens behind an earlier turn.
        {"name": "append_4x8x128_t4095", "kind": "append", "batch": 4, "kv_heads": 8,
         "head_dim": 128, "tokens": 4095, "context": 4112, "paged": False},
        # One conversation of a small model: latency.
        {"name": "decode_1x12x64_l200", "kind": "decode", "batch": 1, "q_heads": 12,
         "kv_heads": 12, "head_dim": 64, "context": 200, "min_context": 200, "window": 0,
         "paged": False},
        # A full batch over long caches: the cache's bytes.
        {"name": "decode_64x32x128_l4096", "kind": "decode", "batch": 64, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "context": 4096, "min_context": 4096, "window": 0,
         "paged": False},
        # One tensor-parallel rank of a 70B-sized layer, sequences of very different lengths.
        {"name": "decode_paged_128x8x128_ragged", "kind": "decode", "batch": 128, "q_heads": 8,
         "kv_heads": 1, "head_dim": 128, "context": 8192, "min_context": 512, "window": 0,
         "paged": True},
        # One very long document.
        {"name": "decode_paged_1x32x128_l131071", "kind": "decode", "batch": 1, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "context": 131071, "min_context": 131071, "window": 0,
         "paged": True},
        # A short second turn of a small model, and a prompt's last chunk.
        {"name": "chunk_2x12x64_c77_l1021", "kind": "chunk", "batch": 2, "q_heads": 12,
         "kv_heads": 12, "head_dim": 64, "tokens": 77, "context": 1021, "paged": False},
        {"name": "chunk_paged_4x32x128_c512_l4608", "kind": "chunk", "batch": 4, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "tokens": 512, "context": 4608, "paged": True},
        # Prompts that fill the int8 cache, and a decode step's tokens in the 4-bit one.
        {"name": "bounds_8x8x128_t16384", "kind": "bounds", "batch": 8, "kv_heads": 8,
         "head_dim": 128, "bits": 8, "tokens": 16384, "context": 16384, "paged": False},
        {"name": "bounds4_paged_64x8x128_t1", "kind": "bounds", "batch": 64, "kv_heads": 8,
         "head_dim": 128, "bits": 4, "tokens": 1, "context": 64, "paged": True},
        # Steps that read 2048 of 32768 tokens for sixteen sequences, and 4096 of 131071 for one.
        {"name": "step_paged_16x32x128_l32768", "kind": "step", "batch": 16, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "bits": 8, "context": 32768, "min_context": 16384,
         "budget": 128, "sinks": 1, "recent": 4, "paged": True},
        {"name": "step4_1x32x128_l131071", "kind": "step", "batch": 1, "q_heads": 32,
         "kv_heads": 8, "head_dim": 128, "bits": 4, "context": 131071, "min_context": 131071,
         "budget": 256, "sinks": 4, "recent": 16, "paged": False},
    ]


def draw(rng):
    def spread(low, high):
        x = math.exp(rng.uniform(math.log(low), math.log(high + 1)))
        return min(high, max(low, int(x)))

    kind = rng.choice(["append", "append", "decode", "decode", "decode", "chunk", "chunk",
                       "bounds", "step", "step", "step"])
    while True:
        kv = rng.choice([1, 1, 2, 4, 8, 12, 16])
        heads = kv * (rng.choice([1, 2, 4, 7, 8]) if kv <= 8 else 1)
        case = {"kind": kind, "batch": spread(1, 128), "kv_heads": kv,
                "head_dim": rng.choice([64, 128, 128]), "paged": rng.random() < 0.6}
        if kind in ("append", "bounds"):
            tokens = spread(1, 16384)
            case.update(tokens=tokens, context=tokens + spread(1, 256) - 1)
            if kind == "bounds":
                case["bits"] = rng.choice([4, 8])
        elif kind == "chunk":
            tokens = spread(1, 1024)
            case.update(batch=spread(1, 8), q_heads=heads, tokens=tokens,
                        context=tokens + spread(1, 8192))
        else:
            top = spread(16, 131072)
            case.update(q_heads=heads, context=top,
                        min_context=rng.choice([top, spread(1, top)]))
            if kind == "decode":
                case["window"] = rng.choice([0, 0, 0, spread(16, 2048)])
            else:
                budget = spread(4, 512)
                case.update(bits=rng.choice([4, 8]), budget=budget,
                            sinks=rng.randint(0, min(4, budget // 4)),
                            recent=rng.randint(1, max(1, budget // 4)))
        cost, most = work(case), MOST[kind]
        held = _held(case)
        if max(held, cost["bytes"]) <= most["bytes"] and cost["flops"] <= most["flops"]:
            return case


def _held(case):
    """Bytes of the cache."""
    bits = case.get("bits", 4)
    return (case["batch"] * (case["context"] // PAGE + 1) * PAGE * case["kv_heads"]
            * (case["head_dim"] * bits // 4 + 8))


# --- the cache's layouts ------------------------------------------------------------------
#
# A 4-bit code c is held as c + 8. A key's byte j holds channel j in its low half and channel
# j + D/2 in its high half. A page's values are transposed, 8 bytes a channel: token t's code
# is nibble 8 (t / 8) + (t % 8) / 2 + 4 (t % 2), low halves first.

def _key_codes(k):
    """[..., D/2] bytes -> [..., D] codes, float32."""
    return torch.cat([k & 15, k >> 4], -1).float() - 8


def _value_codes(v):
    """Transposed pages [..., D, 8] -> [..., 16, D] codes, float32."""
    half = torch.stack([v & 15, v >> 4], -1).unflatten(-2, (2, 4)).flatten(-2)  # [.., D, 2, 8]
    codes = half.unflatten(-1, (2, 4)).transpose(-1, -2).flatten(-3)
    return codes.transpose(-1, -2).float() - 8


def _pack_keys(codes):
    u = (codes + 8).to(torch.uint8)
    D = u.shape[-1]
    return u[..., :D // 2] | u[..., D // 2:] << 4


def _pack_values(codes):
    u = (codes + 8).to(torch.uint8).transpose(-1, -2)                      # [..., D, 16]
    u = u.unflatten(-1, (2, 4, 2)).transpose(-1, -2).flatten(-3)           # nibbles in order
    return u[..., 0::2] | u[..., 1::2] << 4


def _quantized(x, most):
    top = x.abs().amax(-1, keepdim=True)
    scale = top / torch.full_like(top, most)  # (by a number, torch multiplies by its inverse)
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return torch.round(x / scale).clamp_(-most, most), scale.squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 32))
    kind, bits = case["kind"], case.get("bits", 4)
    B, H, D = case["batch"], case["kv_heads"], case["head_dim"]
    st = {"case": case}

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).cuda()

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    blocks = -(-case["context"] // PAGE)
    pages = B * blocks + (max(1, B * blocks // 4) if case["paged"] else 0)
    lead = (pages, H) if case["paged"] else (B, H, blocks)
    # keys whose channels differ in size and that drift from page to page, and values
    size = 0.5 + torch.rand((H, 1, D), generator=g, device="cuda")
    if not case["paged"]:
        size = size[:, None]
    k = (normal(*lead, PAGE, D) + normal(*lead, 1, D)) * size
    v = normal(*lead, PAGE, D)
    most = 127 if bits == 8 else 7
    (kc, ks), (vc, vs) = _quantized(k, most), _quantized(v, most)
    del k, v
    if bits == 8:
        kc, vc = kc.to(torch.int8), vc.to(torch.int8).transpose(-1, -2).contiguous()
    else:
        kc, vc = _pack_keys(kc), _pack_values(vc)
    if not case["paged"]:  # keys and scales lie by tokens
        kc, ks, vs = kc.flatten(2, 3), ks.flatten(2, 3), vs.flatten(2, 3)
    st.update(k=kc, v=vc, ks=ks.contiguous(), vs=vs.contiguous(), table=None)
    if case["paged"]:
        st["table"] = ints(host.permutation(pages)[:B * blocks]).view(B, blocks)

    if kind in ("append", "bounds"):
        T = case["tokens"]
        st["start"] = ints(host.randint(0, case["context"] - T + 1, B))
        if kind == "append":
            # rows as a projection lays them out
            st["k_new"] = (normal(B, T, H, D) * size.reshape(H, D)).transpose(1, 2)
            st["v_new"] = normal(B, T, H, D).transpose(1, 2)
        else:
            st["bounds"] = torch.zeros((*lead, 2, D), dtype=torch.int8, device="cuda")
            st["bs"] = torch.ones(lead, device="cuda")
        return st
    if kind == "chunk":
        Hq, T = case["q_heads"], case["tokens"]
        q = normal(B, Hq, T, D)
        scale = q.abs().amax((0, 2, 3)) / 127
        st["q"] = torch.round(q / scale[:, None, None]).clamp_(-127, 127).to(torch.int8)
        st["qs"] = scale
        return st
    st["lens"] = ints(host.randint(case["min_context"], case["context"] + 1, B))
    q, st["qs"] = _quantized(normal(B, case["q_heads"], D), 127)
    st["q"] = q.to(torch.int8)
    if kind == "step":
        # the bounds of every page, as kv_page_bounds leaves them
        keys = st["k"] if case["paged"] else st["k"].unflatten(2, (blocks, PAGE))
        scales = st["ks"] if case["paged"] else st["ks"].unflatten(2, (blocks, PAGE))
        live = torch.full((*lead, PAGE), True, device="cuda")
        inside = (torch.arange(blocks * PAGE, device="cuda").view(1, blocks, PAGE)
                  < st["lens"][:, None, None])
        if case["paged"]:
            live[st["table"].long()] = inside[:, :, None].expand(B, blocks, H, PAGE)
        else:
            live[:] = inside[:, None]
        bounds, st["bs"] = _page_bounds(_keys(keys, scales, case), live)
        st["bounds"] = bounds.to(torch.int8)
    return st


# --- the plain forms -------------------------------------------------------------------

def _keys(k, ks, case):
    """Keys in float32 from their codes and scales."""
    codes = k.float() if case.get("bits", 4) == 8 else _key_codes(k)
    return codes * ks[..., None]


def _values(v, vs, case):
    """Token-major values in float32 from transposed pages and scales."""
    codes = v.transpose(-1, -2).float() if case.get("bits", 4) == 8 else _value_codes(v)
    return codes * vs[..., None]


def _token_major(st):
    """The cache's keys and values of every sequence, float32 [B, H, tokens, D]."""
    case, table = st["case"], st["table"]
    if table is None:
        v = _values(st["v"], st["vs"].unflatten(2, (-1, PAGE)), case)
        return _keys(st["k"], st["ks"], case), v.flatten(2, 3)
    at = table.long()
    k = _keys(st["k"][at], st["ks"][at], case).transpose(1, 2).flatten(2, 3)
    v = _values(st["v"][at], st["vs"][at], case).transpose(1, 2).flatten(2, 3)
    return k, v


def _attend(q, k, v, visible, scale):
    """Softmax attention of rows q [..., R, D] over k and v [..., L, D]."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    s = s.masked_fill(~visible, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    return torch.matmul(p, v)


def _plain_decode(st):
    case = st["case"]
    B, H, D = case["batch"], case["kv_heads"], case["head_dim"]
    k, v = _token_major(st)
    key = torch.arange(k.shape[2], device=k.device)[None, :]
    lens = st["lens"].long()[:, None]
    visible = key < lens
    if case["window"]:
        visible &= key >= lens - case["window"]
    q = (st["q"].float() * st["qs"][..., None]).view(B, H, -1, D)
    out = _attend(q, k, v, visible[:, None, None], 1 / math.sqrt(D))
    return out.view(B, -1, D)


def _plain_chunk(st):
    case = st["case"]
    B, H, D, T, L = (case["batch"], case["kv_heads"], case["head_dim"], case["tokens"],
                     case["context"])
    k, v = _token_major(st)
    k, v = k[:, :, :L], v[:, :, :L]
    key = torch.arange(L, device=k.device)
    visible = key[None, :] <= key[L - T:, None]
    q = st["q"].float() * st["qs"][:, None, None]
    G = case["q_heads"] // H
    out = _attend(q.view(B, H, G * T, D), k, v, visible.repeat(G, 1), 1 / math.sqrt(D))
    return out.view(B, H * G, T, D)


def _touched(st):
    """The pages [B, n] that the new tokens fall in (their number in the sequence; the last
    one repeated where a sequence has fewer), and an index of them into the cache."""
    case = st["case"]
    start, T = st["start"].long(), case["tokens"]
    n = (T + PAGE - 2) // PAGE + 1
    block = start[:, None] // PAGE + torch.arange(n, device=start.device)
    block = torch.minimum(block, (start[:, None] + T - 1) // PAGE)
    if st["table"] is not None:
        return block, (torch.gather(st["table"], 1, block).long(),)
    b = torch.arange(case["batch"], device=start.device)[:, None]
    return block, (b, slice(None), block)


def _by_pages(st):
    """The cache's keys and scales by pages, as views."""
    if st["table"] is not None:
        return st["k"], st["ks"], st["vs"]
    return tuple(st[n].unflatten(2, (-1, PAGE)) for n in ("k", "ks", "vs"))


def _plain_append(st):
    case = st["case"]
    T = case["tokens"]
    block, at = _touched(st)
    k, ks, vs = _by_pages(st)
    token = (block[:, :, None] * PAGE + torch.arange(PAGE, device=block.device)
             - st["start"].long()[:, None, None])                 # [B, n, 16]
    fresh = ((token >= 0) & (token < T))[:, :, None]               # over heads
    b = torch.arange(case["batch"], device=block.device)[:, None, None]
    token = token.clamp(0, T - 1)
    (kc, knew), (vc, vnew) = _quantized(st["k_new"], 7), _quantized(st["v_new"], 7)

    def rows(x):  # [B, H, T, ...] -> [B, n, H, 16, ...]
        return x[b, :, token].transpose(2, 3)

    knew = torch.where(fresh, rows(knew), ks[at])
    vnew = torch.where(fresh, rows(vnew), vs[at])
    fresh = fresh[..., None]
    kc = torch.where(fresh, rows(kc), _key_codes(k[at]))
    vc = torch.where(fresh, rows(vc), _value_codes(st["v"][at]))
    k[at], st["v"][at] = _pack_keys(kc), _pack_values(vc)
    ks[at], vs[at] = knew, vnew
    return [_keys(k, ks, case), _values(st["v"], vs, case), st["ks"], st["vs"], st["start"] + T]


def _page_bounds(x, live):
    """Codes [..., 2, D] (largest, least) and scales [...] of pages of keys [..., 16, D]."""
    top = (x.abs() * live[..., None]).amax((-1, -2))
    scale = top / torch.full_like(top, 127)
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    high = x.masked_fill(~live[..., None], -math.inf).amax(-2) / scale[..., None]
    low = x.masked_fill(~live[..., None], math.inf).amin(-2) / scale[..., None]
    some = live.any(-1)[..., None]
    high = torch.where(some, torch.ceil(high), 0.0).clamp_(-127, 127)
    low = torch.where(some, torch.floor(low), 0.0).clamp_(-127, 127)
    return torch.stack([high, low], -2), scale


def _plain_bounds(st):
    case = st["case"]
    block, at = _touched(st)
    k, ks, _ = _by_pages(st)
    place = block[:, :, None] * PAGE + torch.arange(PAGE, device=block.device)
    live = (place < st["start"].long()[:, None, None] + case["tokens"])[:, :, None]
    x = _keys(k[at], ks[at], case)
    bounds, scale = _page_bounds(x, live.expand(*x.shape[:-1]))
    st["bounds"][at], st["bs"][at] = bounds.to(torch.int8), scale
    return [st["bounds"].float() * st["bs"][..., None, None], st["bs"]]


def _plain_step(st):
    case = st["case"]
    B, H, D, K = case["batch"], case["kv_heads"], case["head_dim"], case["budget"]
    table = st["table"]
    bounds, bs = st["bounds"], st["bs"]
    if table is not None:
        bounds, bs = bounds[table.long()].transpose(1, 2), bs[table.long()].transpose(1, 2)
    N = bs.shape[2]
    q, qs = st["q"].float().view(B, H, -1, D), st["qs"].view(B, H, -1, 1)
    high = bounds[..., 0, :].float().transpose(2, 3).contiguous()
    low = bounds[..., 1, :].float().transpose(2, 3).contiguous()
    total = torch.matmul(q.clamp(min=0), high) + torch.matmul(q.clamp(max=0), low)
    score = (total * (qs * bs[:, :, None]) + 0.0).amax(2)            # [B, H, N]
    page = torch.arange(N, device=q.device)
    count = ((st["lens"].long() + PAGE - 1) // PAGE)[:, None, None]  # pages that hold tokens
    always = (page < case["sinks"]) | (page >= count - case["recent"])
    score = torch.where(always, math.inf, score).masked_fill(page >= count, -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :K]
    kept = torch.where(torch.arange(best.shape[-1], device=q.device) < count, best, N)
    kept = torch.sort(kept, dim=-1).values
    kept = torch.where(kept == N, -1, kept)
    if K > N:
        kept = torch.nn.functional.pad(kept, (0, K - N), value=-1)
    counts = count.clamp(max=K).expand(B, H, 1).squeeze(-1)

    # attention over those pages
    some = kept.clamp(min=0)
    b = torch.arange(B, device=q.device)[:, None, None]
    h = torch.arange(H, device=q.device)[None, :, None]
    at = (table.long()[b, some], h) if table is not None else (b, h, some)
    k, ks, vs = _by_pages(st)
    keys = _keys(k[at], ks[at], case).flatten(2, 3)
    values = _values(st["v"][at], vs[at], case).flatten(2, 3)
    place = some[..., None] * PAGE + torch.arange(PAGE, device=q.device)
    visible = (kept >= 0)[..., None] & (place < st["lens"].long()[:, None, None, None])
    out = _attend(q * qs, keys, values, visible.flatten(2)[:, :, None], 1 / math.sqrt(D))
    return [kept.int(), counts.int(), out.view(B, -1, D)]


# --- the library's calls -----------------------------------------------------------------

def _own(st):
    import reef_amd as reef

    case, kind = st["case"], st["case"]["kind"]
    if "status" not in st:
        st["status"] = reef.StatusWord("cuda")
    status, table = st["status"], st["table"]
    cache = [st[n] for n in ("k", "v", "ks", "vs")]
    if kind == "append":
        lens = torch.empty_like(st["start"])
        reef.kv_append_int4(st["k_new"], st["v_new"], st["start"], *cache, context_lens=lens,
                            block_table=table, status=status)
        return [*reef.kv_unpack_int4(*cache), st["ks"], st["vs"], lens]
    if kind == "decode":
        return reef.attention_decode_int4(st["q"], st["qs"], *cache, st["lens"],
                                          block_table=table, window=case["window"],
                                          status=status)
    if kind == "chunk":
        return reef.attention_prefill_cache_int4(st["q"], st["qs"], *cache, case["context"],
                                                 block_table=table, status=status)
    if kind == "bounds":
        reef.kv_page_bounds(st["start"], case["tokens"], st["k"], st["ks"], st["bounds"],
                            st["bs"], block_table=table, status=status)
        return [reef.dequantize(st["bounds"], st["bs"], 2 * case["head_dim"]), st["bs"]]
    selected = reef.kv_select_pages(st["q"], st["qs"], st["bounds"], st["bs"], st["lens"],
                                    case["budget"], block_table=table, sinks=case["sinks"],
                                    recent=case["recent"], status=status)
    attend = reef.attention_decode_selected if case["bits"] == 8 else reef.attention_decode_int4
    out = attend(st["q"], st["qs"], *cache, st["lens"], selected=selected, block_table=table,
                 status=status)
    return [*selected, out]


def run(st):
    if own:
        return _own(st)
    return {"append": _plain_append, "decode": _plain_decode, "chunk": _plain_chunk,
            "bounds": _plain_bounds, "step": _plain_step}[st["case"]["kind"]](st)


# --- what a pass cannot do without -------------------------------------------------------

def work(case):
    kind, bits = case["kind"], case.get("bits", 4)
    B, H, D = case["batch"], case["kv_heads"], case["head_dim"]
    row = D * bits // 4 + 8  # a token's keys and values of one head, and their scales
    if kind == "append":  # the rows into the cache, and the cache's values out of it
        rows, held = B * H * case["tokens"], _held(case) // row
        return {"bytes": rows * (8 * D + row) + held * (row + 8 * D), "flops": 4 * rows * D}
    if kind == "bounds":
        # the keys of the touched pages; every page's bounds come out as values
        touched = B * H * (case["tokens"] + 15)
        return {"bytes": touched * (D * bits // 8 + 4) + _held(case) // row // PAGE * (10 * D + 4),
                "flops": 3 * touched * D}
    mean = (case["context"] + case.get("min_context", case["context"])) / 2
    if kind == "chunk":
        T = case["tokens"]
        pairs = B * case["q_heads"] * T * (mean - (T - 1) / 2)
        return {"bytes": B * mean * H * row + B * case["q_heads"] * T * 5 * D, "flops": 4 * pairs * D}
    io = B * case["q_heads"] * (5 * D + 4)
    if kind == "decode":
        tokens = B * (min(mean, case["window"]) if case["window"] else mean)
        return {"bytes": tokens * H * row + io, "flops": 4 * tokens * case["q_heads"] * D}
    pages = B * mean / PAGE
    tokens = B * min(mean, PAGE * case["budget"])
    return {"bytes": pages * H * (2 * D + 4) + tokens * H * row + 2 * io + 8 * B * H * case["budget"],
            "flops": 4 * pages * case["q_heads"] * D + 4 * tokens * case["q_heads"] * D}


# --- the same in 64 bits -----------------------------------------------------------------

def _exact_rows(packed, scales, case, values):
    """float64 rows [n, D] of one head's pages: keys [n, row bytes] or value pages
    [pages, D, bytes], with their scales [n]."""
    bits, D = case.get("bits", 4), case["head_dim"]
    if bits == 8:
        codes = packed.transpose(1, 2).reshape(-1, D) if values else packed
    elif not values:
        codes = torch.empty((packed.shape[0], D), dtype=torch.int64, device="cuda")
        codes[:, :D // 2], codes[:, D // 2:] = packed % 16, packed // 16
        codes -= 8
    else:
        codes = torch.empty((packed.shape[0], PAGE, D), dtype=torch.int64, device="cuda")
        for t in range(PAGE):
            n = 8 * (t // 8) + t % 8 // 2 + 4 * (t % 2)
            byte = packed[:, :, n // 2].long()
            codes[:, t] = (byte // 16 if n % 2 else byte % 16) - 8
        codes = codes.reshape(-1, D)
    return codes.double() * scales.double()[:, None]


def _exact_head(st, b, h, n):
    """float64 keys and values of the first n tokens' pages of one sequence and head."""
    case, blocks = st["case"], -(-n // PAGE)
    if st["table"] is not None:
        at = st["table"][b, :blocks].long()
        k, v = st["k"][at, h].flatten(0, 1), st["v"][at, h]
        ks, vs = st["ks"][at, h].flatten(), st["vs"][at, h].flatten()
    else:
        k, ks, vs = (st[x][b, h, :blocks * PAGE] for x in ("k", "ks", "vs"))
        v = st["v"][b, h, :blocks]
    return _exact_rows(k, ks, case, False), _exact_rows(v, vs, case, True)


def _exact_bounds(x, n):
    """Of pages [blocks, 16, D] of keys, the first n of them live: codes [blocks, 2, D] (largest,
    least) and scales [blocks]."""
    past = (torch.arange(x.shape[0] * PAGE, device="cuda") >= n).view(-1, PAGE, 1)
    high, low = (x.masked_fill(past, far).sort(1).values[:, end]
                 for far, end in ((-math.inf, -1), (math.inf, 0)))
    top = torch.maximum(high, -low).max(1, keepdim=True).values
    scale = torch.where(top > 0, (top / 127).float().double(), 1.0)
    # the quotients as 32 bits round them (rounding twice changes nothing here)
    high, low = (high / scale).float().double(), (low / scale).float().double()
    return torch.stack([high.ceil(), low.floor()], 1).clamp(-127, 127), scale[:, 0]


def exact(case, seed):
    kind = case["kind"]
    B, H, D = case["batch"], case["kv_heads"], case["head_dim"]
    st = prepare(case, seed)
    paged = case["paged"]
    if kind == "append":
        if B * H * case["context"] > 1 << 20:
            return None
        k = torch.empty((*st["v"].shape[:-2], PAGE, D), dtype=torch.float64, device="cuda")
        v, ks, vs = torch.empty_like(k), st["ks"].double(), st["vs"].double()
        flat_k, flat_v = k.view(-1, PAGE, D), v.view(-1, PAGE, D)
        n = flat_k.shape[0]
        flat_k[:] = _exact_rows(st["k"].reshape(n * PAGE, -1), st["ks"].reshape(-1), case,
                                False).view(n, PAGE, D)
        flat_v[:] = _exact_rows(st["v"].reshape(n, D, 8), st["vs"].reshape(-1), case,
                                True).view(n, PAGE, D)
        for new, rows, scales in ((st["k_new"], k, ks), (st["v_new"], v, vs)):
            x = new.double()
            scale = (x.abs().max(-1).values / 7).float().double()
            scale[scale == 0] = 1
            # the quotient as 32 bits round it (rounding twice changes nothing here)
            y = torch.round((x / scale[..., None]).float()).double() * scale[..., None]
            for b in range(B):
                place = int(st["start"][b]) + torch.arange(case["tokens"], device="cuda")
                if paged:
                    at = st["table"][b].long()[place // PAGE]
                    rows[at, :, place % PAGE] = y[b].transpose(0, 1)
                    scales[at, :, place % PAGE] = scale[b].t()
                else:
                    rows[b, :, place // PAGE, place % PAGE] = y[b]
                    scales[b, :, place] = scale[b]
        return [k, v, ks, vs, None]
    if kind == "bounds":
        if B * H > 2048:
            return None
        values, scales = (st["bounds"].double() * st["bs"].double()[..., None, None],
                          st["bs"].double())
        for b in range(B):
            first, end = int(st["start"][b]) // PAGE, int(st["start"][b]) + case["tokens"]
            for h in range(H):
                x, _ = _exact_head(st, b, h, end)
                x = x[first * PAGE:].float().double()  # a key is the product as 32 bits hold it
                codes, scale = _exact_bounds(x.view(-1, PAGE, D), end - first * PAGE)
                block = torch.arange(first, first + len(scale), device="cuda")
                at = (st["table"][b, block].long(), h) if paged else (b, h, block)
                values[at], scales[at] = codes * scale[:, None, None], scale
        return [values, scales]
    Hq = case["q_heads"]
    G = Hq // H
    if kind == "chunk":
        T, L = case["tokens"], case["context"]
        out = torch.empty((B, Hq, T, D), dtype=torch.float64, device="cuda")
        hidden = torch.ones((T, L), dtype=torch.bool, device="cuda").triu(L - T + 1)
        for b in range(B):
            for h in range(H):
                k, v = _exact_head(st, b, h, L)
                for head in range(h * G, (h + 1) * G):
                    s = st["q"][b, head].double() @ k[:L].t() * (st["qs"][head].double() / math.sqrt(D))
                    out[b, head] = torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ v[:L]
        return out
    lens = st["lens"].tolist()
    if B * H > 2048:
        return None
    out = torch.empty((B, Hq, D), dtype=torch.float64, device="cuda")
    for b in range(B):
        n = lens[b]
        for h in range(H):
            k, v = _exact_head(st, b, h, n)
            at = torch.arange(n, device="cuda")
            codes = st["q"][b, h * G:(h + 1) * G]
            scale = st["qs"][b, h * G:(h + 1) * G]
            if kind == "decode":
                if case["window"]:
                    at = at[max(0, n - case["window"]):]
            else:
                at = _exact_tokens(st, b, h, n, codes, scale)
            q = codes.double() * scale.double()[:, None]
            p = torch.softmax(q @ k[at].t() / math.sqrt(D), 1)
            out[b, h * G:(h + 1) * G] = p @ v[at]
    return out if kind == "decode" else [None, None, out]


def _exact_tokens(st, b, h, n, codes, scale):
    """The tokens of the pages that one key head's queries select, in whole numbers up to the
    scores' two roundings."""
    case, pages = st["case"], -(-n // PAGE)
    if st["table"] is not None:
        at = st["table"][b, :pages].long()
        bounds, bs = st["bounds"][at, h], st["bs"][at, h]
    else:
        bounds, bs = st["bounds"][b, h, :pages], st["bs"][b, h, :pages]
    q = codes.cpu().numpy().astype(np.int64)
    high, low = (bounds[:, i].cpu().numpy().astype(np.int64) for i in (0, 1))
    total = np.maximum(q[:, None] * high, q[:, None] * low).sum(-1)
    unit = scale.cpu().numpy()[:, None] * bs.cpu().numpy()[None, :]
    score = (total.astype(np.float32) * unit).max(0)
    score[:case["sinks"]] = np.inf
    score[max(0, pages - case["recent"]):] = np.inf
    best = np.sort(np.argsort(-score, kind="stable")[:case["budget"]])
    tokens = (best[:, None] * PAGE + np.arange(PAGE)).reshape(-1)
    return torch.from_numpy(tokens[tokens < n]).cuda()
