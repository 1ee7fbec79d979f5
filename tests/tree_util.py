"""Pages, trees and 64-bit restatements for the tests of drafted decoding and of
the bounded cache.  Everything here runs on the CPU; tests copy to the GPU."""
import math
import random

import torch

import pyvcpp

KV = {"f32": pyvcpp.KV_F32, "f16": pyvcpp.KV_F16, "i8": pyvcpp.KV_I8, "fp8": pyvcpp.KV_FP8}


class Pool:
    """A KV pool of `layers` layers in one block, with tables for `lens`."""

    def __init__(self, kv, lens, hkv, D, bs=16, layers=1, seed=0, std=1.0, extra=3):
        g = torch.Generator().manual_seed(seed)
        used = [-(-n // bs) for n in lens]
        self.nb = sum(used) + extra
        self.kv, self.bs, self.hkv, self.D, self.layers = kv, bs, hkv, D, layers
        perm = torch.randperm(self.nb, generator=g)
        self.tables = torch.full((len(lens), max(used + [1])), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(used):
            self.tables[i, :n] = perm[at:at + n]
            at += n
        self.spare = perm[at:].tolist()
        shape = (self.nb, layers, bs, hkv, D)
        self.k, self.ks = self._values(shape, g, std)
        self.v, self.vs = self._values(shape, g, std)

    def _values(self, shape, g, std):
        x = torch.randn(shape, generator=g) * std
        if self.kv == "f32":
            return x, None
        if self.kv == "f16":
            return x.half(), None
        if self.kv == "fp8":
            return x.to(torch.float8_e4m3fn).view(torch.uint8), None
        scale = (x.abs().amax(-1) / 127).half()
        q = torch.round(x / scale.float().unsqueeze(-1)).clamp(-127, 127).to(torch.int8)
        return q, scale.transpose(2, 3).contiguous()

    def to(self, device):
        """(descriptor of layer 0, buffers) on a device; the buffers keep it alive."""
        b = {n: t.to(device) for n, t in (("k", self.k), ("v", self.v), ("ks", self.ks), ("vs", self.vs)) if t is not None}
        page = self.bs * self.hkv * self.D
        pages = pyvcpp.kv_pages(KV[self.kv], b["k"], b["v"], self.bs, self.hkv, self.D, self.nb, self.layers * page,
                                b.get("ks"), b.get("vs"), self.layers * self.hkv * self.bs if self.kv == "i8" else 0)
        return pages, b

    def rows(self, s, n, which, layer=0):
        """[n][hkv][D] in 64 bits and which of the positions exist."""
        x, sc = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        out = torch.zeros(n, self.hkv, self.D, dtype=torch.float64)
        ok = torch.zeros(n, dtype=torch.bool)
        for b in range(-(-n // self.bs)):
            bid = int(self.tables[s, b]) if b < self.tables.shape[1] else -1
            if not 0 <= bid < self.nb:
                continue
            m = min(self.bs, n - b * self.bs)
            y = x[bid, layer, :m]
            y = (y.view(torch.float8_e4m3fn).float() if self.kv == "fp8" else y).double()
            if sc is not None:
                y = y * sc[bid, layer, :, :m].double().t()[..., None]
            out[b * self.bs:b * self.bs + m] = y
            ok[b * self.bs:b * self.bs + m] = True
        return out, ok


FAR = 1 << 30  # elements between the blocks of `far`


def far(pool, device):
    """(descriptor, buffers) of one layer's pool with its blocks FAR elements apart."""
    b = {}
    for n in ("k", "v", "ks", "vs"):
        t = getattr(pool, n)
        if t is None:
            continue
        t = t.to(device).reshape(pool.nb, -1)
        b[n] = torch.empty((pool.nb - 1) * FAR + t.shape[1], dtype=t.dtype, device=device)
        for i in range(pool.nb):
            b[n][i * FAR:i * FAR + t.shape[1]] = t[i]
    return pyvcpp.kv_pages(KV[pool.kv], b["k"], b["v"], pool.bs, pool.hkv, pool.D, pool.nb, FAR, b.get("ks"), b.get("vs"),
                           FAR if pool.kv == "i8" else 0), b


def near(buffers, n, pool):
    """The blocks of a buffer of `far`."""
    size = getattr(pool, n).reshape(pool.nb, -1).shape[1]
    return [buffers[n][i * FAR:i * FAR + size] for i in range(pool.nb)]


def tree_bits(n, seed, kind="tree"):
    """Ancestor sets as integers: a random tree, a chain, or arbitrary rows
    (some empty)."""
    r = random.Random(seed)
    if kind == "chain":
        return [(2 << i) - 1 for i in range(n)]
    if kind == "any":
        return [0 if r.random() < 0.2 else r.getrandbits(n) for _ in range(n)]
    bits = []
    for i in range(n):
        bits.append((bits[r.randrange(max(0, i - 6), i)] if i else 0) | 1 << i)
    return bits


def mask_words(bits, words):
    rows = [[(x >> 64 * w) & ((1 << 64) - 1) for w in range(words)] for x in bits]
    return torch.tensor([[w - (1 << 64) if w >> 63 else w for w in r] for r in rows], dtype=torch.int64).reshape(-1, words)


def starts(nodes):
    at = [0]
    for n in nodes:
        at.append(at[-1] + n)
    return at


def reference(pool, q, prefix, nodes, bits):
    """(out, lse, visible weights per sequence [H][n][len]) in 64 bits; a key
    that a row does not see takes no part, whatever it holds."""
    rows, H, D = q.shape
    G = H // pool.hkv
    out = torch.zeros(rows, H, D, dtype=torch.float64)
    lse = torch.full((rows, H), -math.inf, dtype=torch.float64)
    weights, at = [], 0
    for s, (p, n) in enumerate(zip(prefix, nodes)):
        k, ok = pool.rows(s, p + n, "k")
        v, _ = pool.rows(s, p + n, "v")
        see = torch.ones(n, p + n, dtype=torch.bool)
        for i in range(n):
            for j in range(n):
                see[i, p + j] = bool(bits[at + i] >> j & 1)
        see &= ok
        w = torch.zeros(H, n, p + n, dtype=torch.float64)
        for h in range(H):
            kh, vh = k[:, h // G], v[:, h // G]
            x = (q[at:at + n, h].double() @ kh.t()) / math.sqrt(D)
            x = torch.where(see, x, -math.inf)
            m = x.amax(-1, keepdim=True) if p + n else torch.full((n, 1), -math.inf, dtype=torch.float64)
            e = torch.where(see, torch.exp(x - torch.where(torch.isfinite(m), m, 0.0)), 0.0)
            tot = e.sum(-1, keepdim=True)
            w[h] = torch.where(tot > 0, e / tot, 0.0) if not torch.isnan(tot).any() else e / tot
            # rows that see a key which is not finite take its part; others never touch it
            bad = ~torch.isfinite(vh).all(-1)
            out[at:at + n, h] = w[h][:, ~bad] @ vh[~bad] if bad.any() else w[h] @ vh
            for j in torch.nonzero(bad).flatten().tolist():
                hit = see[:, j]
                out[at:at + n, h][hit] += w[h][hit, j, None] * vh[j]
            lse[at:at + n, h] = torch.where(tot[:, 0] > 0, m[:, 0] + torch.log(tot[:, 0]), -math.inf)
        weights.append((w, see))
        at += n
    return out, lse, weights
