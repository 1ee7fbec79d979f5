"""Operators of drafted decoding and of a bounded KV cache, over the paged cache
of libvcpp_attn.so: what a serving engine calls beside its decode and prefill.

A case is a dict of plain values; `op` names the operator:

  tree    vcpp_paged_tree_attention: attention of a tree of drafted tokens over
          a paged prefix, with each row's log-sum-exp
  mass    vcpp_attention_mass: the softmax weights of a step's queries added up
          per kv head and cache position
  plan    vcpp_kv_evict_plan: which positions a bounded cache keeps, and the
          moves that close the gaps
  apply   vcpp_kv_evict_apply: those moves on the K and V pages
  commit  vcpp_kv_commit: an accepted path's rows moved into place, all layers

Lengths, tree sizes and move counts come from a case's bounds through its `lens`
seed, so that a case is the same work whatever its inputs hold.
"""
import math
import os
import random
import sys

import torch

own = False
DEV = "cuda:0"
ESIZE = {"f32": 4, "f16": 2, "i8": 1, "fp8": 1}
DTYPE = {"f32": torch.float32, "f16": torch.float16, "i8": torch.int8, "fp8": torch.float8_e4m3fn}
KV_CODE = {"f32": 0, "f16": 1, "i8": 2, "fp8": 3}


def _lib():
    """This repository's binding (a directory whose name is no package name)."""
    at = os.path.join(os.getcwd(), "vllm-cpp_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import pyvcpp
    return pyvcpp


def listed():
    return [
        # One chat with a short history verifies a small draft tree: the
        # smallest call, where latency counts.
        dict(name="tree_f16_single", op="tree", kv="f16", seqs=1, prefix_min=200, prefix_max=200, nodes_min=8,
             nodes_max=8, heads=64, kv_heads=8, dim=80, block=16, lens=1),
        # A loaded server's speculative step: the headline decode batch's
        # contexts, 16 drafted tokens each.
        dict(name="tree_f16_batch", op="tree", kv="f16", seqs=32, prefix_min=128, prefix_max=4096, nodes_min=16,
             nodes_max=16, heads=64, kv_heads=8, dim=80, block=16, lens=2),
        # Uneven trees on an int8 cache, wide heads and larger pages.
        dict(name="tree_i8_ragged", op="tree", kv="i8", seqs=24, prefix_min=300, prefix_max=6000, nodes_min=5,
             nodes_max=27, heads=32, kv_heads=8, dim=128, block=32, lens=3),
        # Few long documents with wide trees: the largest, bound by the matrix cores.
        dict(name="tree_fp8_long", op="tree", kv="fp8", seqs=8, prefix_min=8000, prefix_max=16384, nodes_min=64,
             nodes_max=64, heads=64, kv_heads=8, dim=80, block=16, lens=4),
        # Every decode step of a bounded cache: one query a sequence adds its weights.
        dict(name="mass_f16_decode", op="mass", kv="f16", seqs=64, prefix_min=128, prefix_max=4096, nodes_min=1,
             nodes_max=1, heads=64, kv_heads=8, dim=80, block=16, lens=5),
        # After a long prompt: the last 32 queries' weights choose what stays.
        dict(name="mass_i8_window", op="mass", kv="i8", seqs=4, prefix_min=4000, prefix_max=16000, nodes_min=32,
             nodes_max=32, heads=32, kv_heads=8, dim=128, block=16, lens=6),
        # A batch that runs at its budget: some steps past it, back to it.
        dict(name="plan_steady", op="plan", seqs=64, len_min=2049, len_max=2064, budget=2048, first=4, last=256,
             kv_heads=8, lens=7),
        # Long prompts cut to a budget for the first time.
        dict(name="plan_prompt", op="plan", seqs=4, len_min=8000, len_max=16384, budget=2048, first=4, last=128,
             kv_heads=8, lens=8),
        # The rows of the steady batch: a few moves in each head.
        dict(name="apply_steady", op="apply", kv="f16", seqs=64, len_min=2049, len_max=2064, budget=2048,
             heads=64, kv_heads=8, dim=80, block=16, lens=9),
        # The rows of a cut prompt: most of the kept ones move.
        dict(name="apply_prompt", op="apply", kv="f16", seqs=4, len_min=8000, len_max=16384, budget=4096,
             heads=64, kv_heads=8, dim=80, block=16, lens=10),
        # One chat's accepted tokens, every layer of a deep model at once.
        dict(name="commit_single", op="commit", kv="f16", seqs=1, layers=64, prefix_min=200, prefix_max=200,
             nodes_min=8, nodes_max=8, depth=4, heads=64, kv_heads=8, dim=80, block=16, lens=11),
        # A batch's accepted paths.
        dict(name="commit_batch", op="commit", kv="f16", seqs=32, layers=16, prefix_min=20, prefix_max=90,
             nodes_min=16, nodes_max=48, depth=8, heads=64, kv_heads=8, dim=80, block=16, lens=12),
    ]


# (query heads, kv heads): group sizes 1 to 8, 2 to 16 kv heads
HEADS = [(64, 8), (32, 8), (28, 4), (16, 8), (32, 4), (12, 2), (16, 16), (24, 8)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges: any operator, page type, head
    shape and page size, batch sizes and lengths spread over their logarithm."""
    limit = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("tree", "mass", "plan", "apply", "commit")}
    while True:
        op = rng.choice(["tree", "tree", "tree", "mass", "mass", "plan", "apply", "commit"])
        heads, kv_heads = rng.choice(HEADS)
        case = dict(op=op, seqs=_log_int(rng, 1, 64), kv_heads=kv_heads, lens=rng.randrange(1 << 20))
        if op != "plan":
            kv = rng.choice(["f16", "f16", "i8", "fp8"] + (["f32"] if op in ("apply", "commit") else []))
            case.update(kv=kv, heads=heads, dim=rng.choice([64, 80, 80, 128, 128]), block=rng.choice([16, 16, 32]))
        if op in ("tree", "mass", "commit"):
            hi = _log_int(rng, 16, 128 if op == "commit" else 32768)
            case.update(prefix_max=hi, prefix_min=int(hi * rng.uniform(0.02, 1.0)))
            hi = _log_int(rng, 1, 128)
            case.update(nodes_max=hi, nodes_min=max(1, int(hi * rng.uniform(0.3, 1.0))))
        if op == "commit":
            case.update(layers=_log_int(rng, 1, 64), depth=rng.randint(1, 12))
        if op in ("plan", "apply"):
            hi = _log_int(rng, 64, 32768)
            case.update(len_max=hi, len_min=max(1, int(hi * rng.uniform(0.3, 1.0))))
            case["budget"] = max(8, int(case["len_max"] * rng.choice([0.1, 0.25, 0.5, 0.9, 0.99])))
        if op == "plan":
            case.update(first=rng.choice([0, 4]), last=int(case["budget"] * rng.uniform(0.0, 0.9)))
            case["first"] = min(case["first"], case["budget"] - case["last"])
        if _cost(case) <= limit[op]:
            return case


def _lens(case):
    """(prefix lengths, tree sizes) of a case, or (lengths, moves per sequence)."""
    r = random.Random(case["lens"])
    S = case["seqs"]
    if "len_min" in case:
        n = [r.randint(case["len_min"], case["len_max"]) for _ in range(S)]
        # kept rows behind the budget, if every row were as likely to be kept
        return n, [max(0, min(case["budget"], x - case["budget"], round(case["budget"] * (x - case["budget"]) / x)))
                   for x in n]
    prefix = [r.randint(case["prefix_min"], case["prefix_max"]) for _ in range(S)]
    return prefix, [r.randint(case["nodes_min"], case["nodes_max"]) for _ in range(S)]


def _row_bytes(case):
    """Bytes of one token's K (or V) row of all kv heads, int8 with its scales."""
    return case["kv_heads"] * (case["dim"] * ESIZE[case["kv"]] + (2 if case["kv"] == "i8" else 0))


def work(case):
    """Bytes read or written once and multiply-add flops of one pass."""
    a, b = _lens(case)
    S, hkv = case["seqs"], case["kv_heads"]
    if case["op"] == "plan":  # scores and positions in and out, the moves
        return {"bytes": hkv * (16 * sum(a) + 8 * sum(b) + 4 * S) + 12 * S, "flops": 0}
    if case["op"] == "apply":  # each moved row's K and V read and written, its move, the table
        table = sum(-(-n // case["block"]) for n in a)
        return {"bytes": sum(b) * (4 * _row_bytes(case) + 8 * hkv) + 4 * S * hkv + 4 * table, "flops": 0}
    if case["op"] == "commit":
        d = sum(min(case["depth"], n) for n in b)
        return {"bytes": case["layers"] * d * 4 * _row_bytes(case) + 4 * d + 8 * S, "flops": 0}
    H, D = case["heads"], case["dim"]
    words = (max(b) + 63) // 64
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in zip(a, b))
    small = sum(b) * (H * D * 2 + H * 4 + 8 * words) + sum(4 * -(-(p + n) // case["block"]) for p, n in zip(a, b)) + 8 * S
    rows = sum(a) + sum(b)
    if case["op"] == "mass":
        return {"bytes": rows * (_row_bytes(case) + 8 * hkv) + small, "flops": pairs * 2 * D * H}
    return {"bytes": rows * 2 * _row_bytes(case) + small + sum(b) * H * D * 4, "flops": pairs * 4 * D * H}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 8e12, w["flops"] / 2.5e15)


# ---- inputs -----------------------------------------------------------------


class _Pool:
    """Pages of a paged KV cache and random block tables for the given lengths.
    `layers` > 1: every layer in one block, as an engine that allocates a block
    for all layers holds it.  The last block belongs to no table."""

    def __init__(self, case, lens, gen, layers=1):
        bs, hkv, D = case["block"], case["kv_heads"], case["dim"]
        used = [-(-n // bs) for n in lens]
        nb = max(1, (sum(used) * 9 + 7) // 8) + 1
        self.kv, self.bs, self.nb, self.layers = case["kv"], bs, nb, layers
        perm = torch.randperm(nb - 1, generator=gen, device=DEV).to(torch.int32)
        at, rows = 0, []
        for n in used:
            rows.append(torch.nn.functional.pad(perm[at:at + n], (0, max(used) - n), value=-1))
            at += n
        self.tables = torch.stack(rows).contiguous()
        self.ks = self.vs = None
        self.k, self.ks = self._values((nb, layers, bs, hkv, D), gen)
        self.v, self.vs = self._values((nb, layers, bs, hkv, D), gen)
        self.hkv, self.D = hkv, D

    def _values(self, shape, gen):
        if self.kv == "f16":
            return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float16), None
        x = torch.randn(shape, generator=gen, device=DEV)
        if self.kv == "f32":
            return x, None
        if self.kv == "fp8":
            return x.to(torch.float8_e4m3fn), None
        scale = (x.abs().amax(-1) / 127).to(torch.float16)
        q = torch.round(x / scale.float().unsqueeze(-1)).clamp_(-127, 127).to(torch.int8)
        return q, scale.transpose(2, 3).contiguous()

    def pages(self):
        """The descriptor of layer 0."""
        lib = _lib()
        page = self.bs * self.hkv * self.D
        return lib.kv_pages(KV_CODE[self.kv], self.k, self.v, self.bs, self.hkv, self.D, self.nb, self.layers * page,
                            self.ks, self.vs, self.layers * self.hkv * self.bs if self.kv == "i8" else 0)

    def buffers(self):
        out = {"k": self.k, "v": self.v}
        if self.kv == "i8":
            out.update(ks=self.ks, vs=self.vs)
        return out

    def dense(self, which, dtype=torch.float32):
        """K or V of every sequence's table, [S][kv heads][positions][dim] (layer 0)."""
        x, s = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        ids = self.tables.long().clamp_min(0)
        x = self._take(x, ids).to(dtype)  # [S][blocks][bs][hkv][D]
        if s is not None:
            x = x * s[ids, 0].to(dtype).transpose(2, 3).unsqueeze(-1)
        S = ids.shape[0]
        return x.reshape(S, -1, self.hkv, self.D).permute(0, 2, 1, 3)

    def _take(self, x, ids):
        """Layer 0 of the blocks `ids`."""
        return x.view(torch.uint8)[ids, 0].view(x.dtype) if self.kv == "fp8" else x[ids, 0]

    def slots(self, pos):
        """Physical slots (block * block size + place) of positions [S][...] through the tables."""
        S, width = self.tables.shape  # (places that are not used may lie behind the table)
        b = (pos // self.bs).clamp_max(width - 1).reshape(S, -1)
        b = torch.gather(self.tables.long(), 1, b).reshape(pos.shape)
        return b * self.bs + pos % self.bs


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(n):
    at = [0]
    for x in n:
        at.append(at[-1] + x)
    return at


def _tree_bits(rng, n):
    """Ancestor sets (own node included) of a random draft tree as it is grown:
    every node's parent is one of the eight before it."""
    bits = []
    for i in range(n):
        bits.append((bits[rng.randrange(max(0, i - 8), i)] if i else 0) | 1 << i)
    return bits


def _words(bits, words):
    """Integers as rows of 64-bit words (two's complement)."""
    rows = [[(x >> 64 * w & (1 << 64) - 1) for w in range(words)] for x in bits]
    return torch.tensor([[w - (1 << 64) if w >> 63 else w for w in r] for r in rows], dtype=torch.int64, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    a, b = _lens(case)
    s = {"case": case, "op": case["op"]}
    if case["op"] == "plan":
        return _prepare_plan(case, s, gen, a)
    if case["op"] == "apply":
        return _prepare_apply(case, s, gen, a, b)
    if case["op"] == "commit":
        s["pool"] = _Pool(case, [p + n for p, n in zip(a, b)], gen, case["layers"])
        path = torch.full((len(a), case["depth"]), -1, dtype=torch.int32)
        for i, n in enumerate(b):
            d = min(case["depth"], n)
            path[i, :d] = torch.tensor(sorted(rng.sample(range(n), d)), dtype=torch.int32)
        s["path"], s["taken"] = path.to(DEV), _ints([min(case["depth"], n) for n in b])
        s["prefix"], s["max_nodes"] = _ints(a), max(b)
        return s
    H, D = case["heads"], case["dim"]
    s["pool"] = _Pool(case, [p + n for p, n in zip(a, b)], gen)
    s["start"], s["prefix"] = _ints(_starts(b)), _ints(a)
    s["max_nodes"], s["max_prefix"], s["H"] = max(b), max(a), H
    s["q"] = torch.randn(sum(b), H, D, generator=gen, device=DEV, dtype=torch.float16)
    words = (max(b) + 63) // 64
    if case["op"] == "mass":  # a window of consecutive tokens: a tree that is a chain
        s["mask"] = _words([(2 << i) - 1 for n in b for i in range(n)], words)
        s["lse"] = _softmax_of(s)[2]
        L = s["max_prefix"] + s["max_nodes"]
        s["scores"] = torch.rand(len(a), case["kv_heads"], L, generator=gen, device=DEV)
        s["scores"] *= 4.0 * H // case["kv_heads"] * max(b) / L  # some steps' weights are there already
        return s
    s["mask"] = _words([x for n in b for x in _tree_bits(rng, n)], words)
    s["out"] = torch.zeros(sum(b), H, D, device=DEV)
    s["lse"] = torch.zeros(sum(b), H, device=DEV)
    return s


def _prepare_plan(case, s, gen, n):
    S, hkv, top = len(n), case["kv_heads"], case["len_max"]
    s["lens"] = _ints(n)
    # Weights as attention leaves them: most positions nearly none, a few much.
    s["scores"] = torch.randn(S, hkv, top, generator=gen, device=DEV).mul_(2.5).exp_()
    s["scores"] *= torch.arange(top, device=DEV) < s["lens"][:, None, None]
    # Half of the sequences have been cut before: what lies in front of the
    # budget is out of order, what came after it is marked as new.
    seen = [x + (x // 2 if i % 2 else 0) for i, x in enumerate(n)]
    s["seen"] = _ints(seen)
    s["positions"] = torch.full((S, hkv, top), -1, dtype=torch.int32, device=DEV)
    for i in range(1, S, 2):
        m = min(case["budget"], n[i])
        old = torch.rand(hkv, seen[i] - (n[i] - m), generator=gen, device=DEV).argsort(-1)[:, :m]
        s["positions"][i, :, :m] = old.to(torch.int32)
    most = max(1, min(case["budget"], top - case["budget"]))
    s["moves"] = torch.full((S, hkv, most, 2), -1, dtype=torch.int32, device=DEV)
    s["counts"] = torch.zeros(S, hkv, dtype=torch.int32, device=DEV)
    s["new_lens"] = torch.zeros(S, dtype=torch.int32, device=DEV)
    s["scores_out"], s["positions_out"] = torch.zeros_like(s["scores"]), torch.zeros_like(s["positions"])
    return s


def _prepare_apply(case, s, gen, n, moves):
    S, hkv, budget = len(n), case["kv_heads"], case["budget"]
    s["pool"] = _Pool(case, n, gen)
    most = max(1, max(moves))
    s["moves"] = torch.full((S, hkv, most, 2), -1, dtype=torch.int32, device=DEV)
    for i, m in enumerate(moves):
        if m:  # holes in front of the budget, kept rows behind it
            to = torch.rand(hkv, budget, generator=gen, device=DEV).argsort(-1)[:, :m].sort(-1)[0]
            of = torch.rand(hkv, n[i] - budget, generator=gen, device=DEV).argsort(-1)[:, :m].sort(-1)[0] + budget
            s["moves"][i, :, :m] = torch.stack([to, of], -1).to(torch.int32)
    s["counts"] = _ints(moves)[:, None].expand(S, hkv).contiguous()
    return s


# ---- one pass ---------------------------------------------------------------


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    lib, op = _lib(), s["op"]
    if "pool" in s and "pages" not in s:
        s["pages"] = s["pool"].pages()  # the descriptor, once per pool
    if op == "tree":
        if "ws" not in s:  # scratch that an engine keeps
            need = lib.tree_workspace_size(s["pages"], s["prefix"].shape[0], s["max_nodes"], s["max_prefix"], s["H"])
            s["ws"] = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
        lib.paged_tree_attention(s["pages"], s["q"], s["out"], s["pool"].tables, s["start"], s["prefix"], s["max_nodes"],
                                 s["max_prefix"], s["H"], tree_mask=s["mask"], lse=s["lse"], workspace=s["ws"])
        return {"out": s["out"], "lse": s["lse"]}
    if op == "mass":
        lib.attention_mass(s["pages"], s["q"], s["lse"], s["scores"], s["pool"].tables, s["start"], s["prefix"],
                           s["max_nodes"], s["max_prefix"], s["H"], tree_mask=s["mask"])
        return {"scores": s["scores"]}
    if op == "plan":
        c = s["case"]
        lib.kv_evict_plan(s["scores"], s["lens"], c["len_max"], c["budget"], s["moves"], s["counts"], s["new_lens"],
                          s["scores_out"], keep_first=c["first"], keep_last=c["last"], seen_lens=s["seen"],
                          positions=s["positions"], positions_out=s["positions_out"])
        return {x: s[x] for x in ("moves", "counts", "new_lens", "scores_out", "positions_out")}
    if op == "apply":
        lib.kv_evict_apply(s["pages"], s["pool"].tables, s["moves"], s["counts"])
        return s["pool"].buffers()
    pool = s["pool"]
    lib.kv_commit(s["pages"], pool.tables, s["prefix"], s["path"], s["taken"], s["max_nodes"], num_layers=pool.layers,
                  layer_stride=pool.bs * pool.hkv * pool.D, scale_layer_stride=pool.hkv * pool.bs)
    return pool.buffers()


def _plain(s):
    if s["op"] == "tree":
        p, _, lse, take = _softmax_of(s, rows=True)
        S, hkv = p.shape[:2]
        out = torch.matmul(p, s["pool"].dense("v"))
        out = out.reshape(S, hkv, -1, s["H"] // hkv, out.shape[-1]).permute(0, 2, 1, 3, 4)
        return {"out": out.reshape(-1, s["H"], out.shape[-1])[take], "lse": lse}
    if s["op"] == "mass":
        p, visible, _ = _softmax_of(s, s["lse"])
        reach = min(p.shape[3], s["scores"].shape[2])  # whole blocks reach past it, or the longest table falls short
        s["scores"][:, :, :reach] += p.sum(2)[:, :, :reach]
        return {"scores": s["scores"]}
    if s["op"] == "plan":
        return _plain_plan(s)
    if s["op"] == "apply":
        pos = s["moves"].clamp_min(0).long()
        used = torch.arange(pos.shape[2], device=DEV)[None, None] < s["counts"][:, :, None]
        _move(s["pool"], pos[..., 1], pos[..., 0], used, True)
        return s["pool"].buffers()
    d = torch.arange(s["path"].shape[1], device=DEV)[None]
    prefix = s["prefix"].long()[:, None]
    _move(s["pool"], prefix + s["path"].clamp_min(0), (prefix + d).expand_as(s["path"]), d < s["taken"][:, None], False)
    return s["pool"].buffers()


def _softmax_of(s, lse=None, rows=False):
    """Softmax weights [S][kv heads][nodes * group][positions] in 32 bits, the
    visible places, and the rows' log-sum-exp [rows][heads] (or weights by the
    given one); rows: also the packed rows' places in the padded ones."""
    pool, H = s["pool"], s["H"]
    q, mask, start, prefix = s["q"], s["mask"], s["start"].long(), s["prefix"].long()
    N, S, hkv, D = s["max_nodes"], prefix.numel(), pool.hkv, pool.D
    G = H // hkv
    count = start[1:] - start[:-1]
    i = torch.arange(N, device=DEV)
    live = i[None] < count[:, None]
    at = torch.where(live, start[:-1, None] + i[None], 0)
    k = pool.dense("k")
    L = k.shape[2]
    node = torch.arange(L, device=DEV)[None] - prefix[:, None]  # [S][L]
    inside = (node >= 0) & (node < count[:, None])
    j = torch.where(inside, node, 0)
    word = mask[at].gather(2, (j >> 6)[:, None].expand(S, N, L))
    seen = ((word >> (j & 63)[:, None]) & 1).bool() & inside[:, None]
    has = pool.tables.ge(0).repeat_interleave(pool.bs, 1)
    visible = ((node < 0)[:, None] | seen) & has[:, None] & live[:, :, None]  # [S][N][L]
    qs = q[at].float().reshape(S, N, hkv, G, D).permute(0, 2, 1, 3, 4).reshape(S, hkv, N * G, D)
    x = torch.matmul(qs, k.transpose(2, 3)).mul_(1.0 / math.sqrt(D))
    hide = ~visible[:, None, :, None].expand(S, 1, N, G, L).reshape(S, 1, N * G, L)
    x.masked_fill_(hide, -math.inf)
    take = live.reshape(-1).nonzero().reshape(-1) if lse is None else None
    if lse is not None:
        ref = lse[at].reshape(S, N, hkv, G).permute(0, 2, 1, 3).reshape(S, hkv, N * G, 1)
        return x.sub_(ref).exp_(), visible, lse
    m = x.amax(-1, keepdim=True).clamp_min(-1e30)
    p = x.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    out = (m + total.log()).reshape(S, hkv, N, G).permute(0, 2, 1, 3).reshape(S * N, H)[take]
    if not rows:
        return p, visible, out
    return p.div_(total + 1e-9), visible, out, take


def _plain_plan(s):
    c, scores = s["case"], s["scores"]
    S, hkv, top = scores.shape
    budget = c["budget"]
    n = s["lens"].long()[:, None, None]
    slot = torch.arange(top, device=DEV)[None, None]
    valid = slot < n
    seen = s["seen"].long()[:, None, None]
    place = torch.where(s["positions"] >= 0, s["positions"].long(), seen - n + slot)
    safe = (place < c["first"]) | (place >= seen - c["last"])
    key = torch.where(safe, math.inf, scores).masked_fill(~valid, -math.inf)
    order = key.sort(dim=-1, descending=True, stable=True)[1]
    rank = torch.empty_like(order).scatter_(-1, order, slot.expand_as(order))
    kept = (rank < budget) & valid
    hole, filler = ~kept & (slot < budget) & valid, kept & (slot >= budget)
    most = s["moves"].shape[2]
    to = (~hole).to(torch.int8).sort(dim=-1, stable=True)[1][..., :most]
    of = (~filler).to(torch.int8).sort(dim=-1, stable=True)[1][..., :most]
    count = hole.sum(-1)
    used = torch.arange(most, device=DEV)[None, None] < count[..., None]
    moves = torch.where(used[..., None], torch.stack([to, of], -1), -1).to(torch.int32)
    new = n.clamp_max(budget)
    source = slot.expand_as(order).scatter(-1, torch.where(used, to, top - 1), torch.where(used, of, top - 1))
    stays = (slot < new).expand_as(order)
    # (a move slot that is not used writes the last place's own index)
    scores_out = torch.where(stays, scores.gather(-1, source), 0.0)
    places = torch.where(stays, place.gather(-1, source), -1).to(torch.int32)
    return {"moves": moves, "counts": count.to(torch.int32), "new_lens": new[:, 0, 0].to(torch.int32),
            "scores_out": scores_out, "positions_out": places}


def _move(pool, of, to, used, by_head):
    """Rows of positions `of` to positions `to`, all read before any is written;
    what is not used writes the spare block's first row onto itself."""
    spare = (pool.nb - 1) * pool.bs
    of, to = (torch.where(used, pool.slots(x), spare) for x in (of, to))
    bs = pool.bs
    if by_head:
        h = torch.arange(pool.hkv, device=DEV)[None, :, None].expand_as(of)
    for x in (pool.k, pool.v):
        y = x.view(torch.uint8) if pool.kv == "fp8" else x
        if by_head:
            y[to // bs, 0, to % bs, h] = y[of // bs, 0, of % bs, h]
        else:
            y[to // bs, :, to % bs] = y[of // bs, :, of % bs]
    if pool.kv == "i8":
        for x in (pool.ks, pool.vs):
            if by_head:
                x[to // bs, 0, h, to % bs] = x[of // bs, 0, h, of % bs]
            else:
                x[to // bs, :, :, to % bs] = x[of // bs, :, :, of % bs]


# ---- the same in 64 bits ----------------------------------------------------


def _rows64(pool, i, n, which):
    """K or V of the first n positions of sequence i (layer 0), [n][kv heads][dim]."""
    x, scale = (pool.k, pool.ks) if which == "k" else (pool.v, pool.vs)
    ids = pool.tables[i, :-(-n // pool.bs)].long()
    y = pool._take(x, ids).double()
    if scale is not None:
        y = y * scale[ids, 0].double().transpose(1, 2)[..., None]
    return y.reshape(-1, pool.hkv, pool.D)[:n]


def _bits64(words):
    """[n][words] 64-bit words as truth values [n][64 * words]."""
    j = torch.arange(64 * words.shape[1], device=DEV)
    return (words[:, j // 64] >> (j % 64) & 1).bool()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return _exact_plan(s)
    if case["op"] in ("apply", "commit"):
        return _exact_move(s)
    pool, H, hkv, D = s["pool"], s["H"], s["pool"].hkv, s["pool"].D
    G = H // hkv
    prefix, nodes = _lens(case)
    out, lse, scores, at = [], [], s["scores"].double() if case["op"] == "mass" else None, 0
    for i, (p, n) in enumerate(zip(prefix, nodes)):
        k = _rows64(pool, i, p + n, "k")
        allowed = torch.ones(n, p + n, dtype=torch.bool, device=DEV)
        allowed[:, p:] = _bits64(s["mask"][at:at + n])[:, :n]
        o = torch.zeros(n, H, D, dtype=torch.float64, device=DEV)
        z = torch.zeros(n, H, dtype=torch.float64, device=DEV)
        v = _rows64(pool, i, p + n, "v") if case["op"] == "tree" else None
        for h in range(H):
            x = (s["q"][at:at + n, h].double() @ k[:, h // G].t().contiguous()) / math.sqrt(D)
            x = torch.where(allowed, x, -math.inf)
            if case["op"] == "mass":
                w = torch.exp(x - s["lse"][at:at + n, h, None].double())
                scores[i, h // G, :p + n] += w.sum(0)
                continue
            z[:, h] = torch.logsumexp(x, -1)
            o[:, h] = torch.exp(x - z[:, h, None]) @ v[:, h // G].contiguous()
        out.append(o)
        lse.append(z)
        at += n
    return {"scores": scores} if case["op"] == "mass" else {"out": torch.cat(out), "lse": torch.cat(lse)}


def _exact_plan(s):
    c = s["case"]
    S, hkv, top = s["scores"].shape
    scores, places = s["scores"].double().cpu(), s["positions"].cpu()
    seen, lens = s["seen"].tolist(), s["lens"].tolist()
    moves = torch.full(s["moves"].shape, -1, dtype=torch.int32)
    counts = torch.zeros(S, hkv, dtype=torch.int32)
    scores_out = torch.zeros(S, hkv, top, dtype=torch.float64)
    places_out = torch.full((S, hkv, top), -1, dtype=torch.int32)
    for i, n in enumerate(lens):
        for h in range(hkv):
            at, weight = places[i, h, :n].tolist(), scores[i, h, :n].tolist()
            at = [x if x >= 0 else seen[i] - n + j for j, x in enumerate(at)]
            weight = [math.inf if x < c["first"] or x >= seen[i] - c["last"] else w for x, w in zip(at, weight)]
            best = set(sorted(range(n), key=lambda j: (-weight[j], j))[:c["budget"]])
            to = [j for j in range(min(n, c["budget"])) if j not in best]
            of = [j for j in range(c["budget"], n) if j in best]
            row = list(range(min(n, c["budget"])))
            for x, y in zip(to, of):
                row[x] = y
            counts[i, h] = len(to)
            if to:
                moves[i, h, :len(to)] = torch.tensor([to, of], dtype=torch.int32).t()
            scores_out[i, h, :len(row)] = scores[i, h][row]
            places_out[i, h, :len(row)] = torch.tensor([at[j] for j in row], dtype=torch.int32)
    new = torch.tensor([min(n, c["budget"]) for n in lens], dtype=torch.int32)
    return {"moves": moves, "counts": counts, "new_lens": new, "scores_out": scores_out, "positions_out": places_out}


def _exact_move(s):
    """Each moved row by itself, from a copy of the pages as they were."""
    pool, case = s["pool"], s["case"]
    a, b = _lens(case)
    got = {}
    for name, x in pool.buffers().items():
        if case["kv"] == "fp8":
            x = x.view(torch.uint8)
        # [block][layer][place][head][...]
        x = x.transpose(2, 3) if name in ("ks", "vs") else x
        new = x.clone()
        for i, n in enumerate(a):
            table = pool.tables[i].tolist()
            if case["op"] == "commit":
                pairs = [(n + j, n + x0) for j, x0 in enumerate(s["path"][i].tolist()[:min(case["depth"], b[i])])]
                for to, of in pairs:
                    new[table[to // pool.bs], :, to % pool.bs] = x[table[of // pool.bs], :, of % pool.bs]
                continue
            for h in range(pool.hkv):
                if not b[i]:
                    continue
                to, of = s["moves"][i, h, :b[i]].long().unbind(-1)
                t = pool.tables[i].long()
                new[t[to // pool.bs], 0, to % pool.bs, h] = x[t[of // pool.bs], 0, of % pool.bs, h]
        new = new.view(torch.float8_e4m3fn) if case["kv"] == "fp8" else new
        new = new.transpose(2, 3) if name in ("ks", "vs") else new
        got[name] = new.double() if new.is_floating_point() else new
    return got
