"""Caches in 8 and 4 bits, laid out by the definitions of the C header, for the tests of the calls
that read less of a cache."""
import math

import numpy as np

PAGE = 16
U = 2.0 ** -24


def pack_keys(c):
    """Codes [..., D] -> bytes [..., D/2]: channel j low, channel j + D/2 high."""
    u, half = (c + 8).astype(np.uint8), c.shape[-1] // 2
    return u[..., :half] | u[..., half:] << 4


def pack_values(c):
    """Codes by tokens [..., 16, D] -> bytes [..., D, 8]."""
    u = np.moveaxis((c + 8).astype(np.uint8), -2, -1)
    out = np.zeros((*u.shape[:-1], 8), np.uint8)
    for t in range(PAGE):
        n = 8 * (t // 8) + t % 8 // 2 + 4 * (t % 2)
        out[..., n // 2] |= u[..., t] << (4 * (n % 2))
    return out


def unpack_keys(b):
    return np.concatenate([b & 15, b >> 4], -1).astype(np.int64) - 8


def unpack_values(b):
    out = np.empty((*b.shape[:-2], PAGE, b.shape[-2]), np.int64)
    for t in range(PAGE):
        n = 8 * (t // 8) + t % 8 // 2 + 4 * (t % 2)
        out[..., t, :] = (b[..., n // 2] >> (4 * (n % 2)) & 15).astype(np.int64) - 8
    return out


def quantized(x, most):
    """(codes, scales) of rows [..., D] in float32, as the append writes them."""
    scale = np.abs(x).max(-1) / np.float32(most)
    scale[scale == 0] = 1
    return np.clip(np.rint(x / scale[..., None]), -most, most).astype(np.int64), scale


class Cache:
    """Random codes [B, H, L, D] and scales [B, H, L] of `bits`, and their image on the GPU:
    contiguous, or a pool with pages of other sequences between them. What lies behind a
    sequence's end is of the largest codes, with scales that are no numbers."""

    def __init__(self, rng, bits, B, H, D, L, lens, paged, key_drift=0.0):
        import torch
        most = 127 if bits == 8 else 7
        self.bits, self.B, self.H, self.D, self.L, self.lens = bits, B, H, D, L, lens
        shape = (B, H, L, D)
        self.k, self.v = (rng.integers(-most, most + 1, shape) for _ in range(2))
        if key_drift:  # pages whose keys differ from one another
            page = rng.normal(0, key_drift * most, (B, H, L // PAGE, 1, D))
            self.k = np.clip(np.rint(self.k.reshape(B, H, -1, PAGE, D) * 0.4 + page), -most,
                             most).astype(np.int64).reshape(shape)
        self.ks, self.vs = (rng.uniform(0.2, 1.0, shape[:3]).astype(np.float32) / most
                            for _ in range(2))
        past = np.arange(L) >= np.asarray(lens)[:, None]
        k, v, ks, vs = (x.copy() for x in (self.k, self.v, self.ks, self.vs))
        for x in (k, v):
            x[np.broadcast_to(past[:, None, :, None], shape)] = most
        for x in (ks, vs):
            x[np.broadcast_to(past[:, None], shape[:3])] = np.nan
        v = v.reshape(B, H, L // PAGE, PAGE, D)
        if bits == 8:
            k, v = k.astype(np.int8), np.ascontiguousarray(np.moveaxis(v, -2, -1)).astype(np.int8)
        else:
            k, v = pack_keys(k), pack_values(v)
        self.table = self.block_table = None
        if paged:
            blocks = L // PAGE
            pages = B * blocks + 3
            self.table = rng.permutation(pages)[:B * blocks].reshape(B, blocks).astype(np.int32)
            self.block_table = torch.from_numpy(self.table).cuda()

            def pool(x):  # [B, H, blocks, ...] -> [P, H, ...]
                out = np.full((pages, H, *x.shape[3:]), 1, x.dtype)
                out[self.table] = np.swapaxes(x, 1, 2)
                return out

            k, ks, vs = (x.reshape(B, H, blocks, PAGE, *x.shape[3:]) for x in (k, ks, vs))
            k, v, ks, vs = pool(k), pool(v), pool(ks), pool(vs)
        self.tensors = [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (k, v, ks, vs)]
        self.context_lens = torch.tensor(list(lens), dtype=torch.int32).cuda()

    def keys(self, b, h):
        return self.k[b, h] * self.ks[b, h, :, None].astype(np.float64)

    def values(self, b, h):
        return self.v[b, h] * self.vs[b, h, :, None].astype(np.float64)


def queries(rng, B, Hq, D):
    return (rng.integers(-127, 128, (B, Hq, D)).astype(np.int8),
            rng.uniform(0.005, 0.02, (B, Hq)).astype(np.float32))


def attention(cache, q, qs, seen):
    """(out [B, Hq, D], tolerance) in 64 bits; seen(b, kv head) gives the tokens, with repeats.

    The tolerance, relative to the largest |value|, u = 2^-24: an exponent of X log2 units is
    rounded four times (key scale, query scale with the softmax scale, log2 e, the difference),
    which moves a weight by 4 ln2 X u; exp2 adds 2 u, a weight's two fp16 parts 4 u, and a weight
    below 2^-14 at most 2^-33 a key. Sums of n terms are off by n u. Numerator and row sum can both
    be off by all that; 14 u for up to 6 merges and the quotient."""
    B, Hq, D = q.shape
    G = Hq // cache.H
    out = np.zeros((B, Hq, D))
    most = X = 0.0
    n = 0
    for b in range(B):
        for h in range(cache.H):
            at = np.asarray(seen(b, h), np.int64)
            if len(at) == 0:
                continue
            n = max(n, len(at))
            k, v = cache.keys(b, h)[at], cache.values(b, h)[at]
            most = max(most, np.abs(v).max())
            for head in range(h * G, h * G + G):
                s = (q[b, head] * np.float64(qs[b, head])) @ k.T / math.sqrt(D)
                X = max(X, np.abs(s).max() / math.log(2))
                p = np.exp(s - s.max())
                out[b, head] = p @ v / p.sum()
    return out, most * (2 * (2.8 * X * U + 6 * U + n * (U + 2.0 ** -33)) + 14 * U)


def page_bounds(x):
    """Bounds of keys [n, D], products in float32: codes [2, D] and the scale."""
    x = x.astype(np.float32)
    scale = np.abs(x).max() / np.float32(127)
    if scale == 0:
        scale = np.float32(1)
    high = np.minimum(np.ceil(x.max(0) / scale), 127)
    low = np.maximum(np.floor(x.min(0) / scale), -127)
    return np.stack([high, low]).astype(np.int8), scale
