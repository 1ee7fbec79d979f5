"""The bounded cache and the commit of an accepted path on the GPU:
vcpp_attention_mass against its definition in 64 bits, vcpp_kv_evict_plan,
vcpp_kv_evict_apply and vcpp_kv_commit against plain restatements, exactly."""
import math

import pytest
import torch

import pyvcpp
import tree_util as U

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# A weight exp(s - lse) is off by what the exponent is: the fp32 score (at most
# about 16 here, some roundings of 2^-24 each: 4e-6) and the fp32 lse (at most
# 16: 1e-6), exp2's 2 ulp, and the sums' roundings.
REL = 6e-6


def dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


# ---- attention mass ---------------------------------------------------------


def mass(pool, q, lse, scores, prefix, nodes, mask, H, max_prefix=None, max_nodes=None):
    pages, keep = pool.to(DEV)
    s = scores.to(DEV)
    pyvcpp.attention_mass(pages, q.to(DEV), lse.to(DEV), s, pool.tables.to(DEV), dev(U.starts(nodes)), dev(prefix),
                          max(nodes) if max_nodes is None else max_nodes, max(prefix) if max_prefix is None else max_prefix, H,
                          tree_mask=None if mask is None else mask.to(DEV))
    torch.cuda.synchronize()
    return s.cpu()


def check_mass(kv, H, hkv, D, bs, prefix, nodes, kind="tree", seed=1, extra=0, **kw):
    pool = U.Pool(kv, [p + n for p, n in zip(prefix, nodes)], hkv, D, bs, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(sum(nodes), H, D, generator=g).half()
    bits = [b for i, n in enumerate(nodes) for b in U.tree_bits(n, seed + i, kind)]
    _, lse, weights = U.reference(pool, q, prefix, nodes, bits)
    stride = kw.get("max_prefix", max(prefix)) + kw.get("max_nodes", max(nodes)) + extra
    before = torch.rand(len(prefix), hkv, stride, generator=g) * 0.01
    got = mass(pool, q, lse.float(), before, prefix, nodes, U.mask_words(bits, (max(nodes) + 63) // 64), H, **kw)
    want = before.double()
    for s, (w, see) in enumerate(weights):
        L = w.shape[2]
        want[s, :, :L] += w.reshape(hkv, H // hkv, -1, L).sum((1, 2)) if w.shape[1] else 0
        assert torch.equal(got[s, :, L:], before[s, :, L:]), "positions behind the sequence changed"
    d = got.double() - want
    assert float(d.norm()) <= REL * float(want.norm()), float(d.norm() / want.norm())
    assert float(d.abs().max()) <= 8 * REL * max(1.0, float(want.max()))
    return pool, q, bits, lse, got


@pytest.mark.parametrize("kv", ["f16", "i8", "fp8"])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("H,hkv", [(8, 8), (6, 2), (7, 1), (16, 1)])
def test_mass_types_and_heads(kv, D, H, hkv):
    check_mass(kv, H, hkv, D, 16, [37, 0, 130], [9, 5, 16])


@pytest.mark.parametrize("kv", ["f16", "i8"])
@pytest.mark.parametrize("n", [1, 2, 15, 33, 64, 65, 130, 256])
def test_mass_rows(kv, n):
    check_mass(kv, 8, 2, 80, 16, [100], [n], seed=n)


@pytest.mark.parametrize("p", [0, 1, 15, 16, 63, 64, 65, 255, 256, 257, 1000, 3001])
def test_mass_prefix_lengths(p):
    check_mass("f16", 8, 2, 80, 16, [p], [3], seed=p)
    check_mass("fp8", 8, 2, 128, 32, [p], [1], seed=p, kind="chain")


@pytest.mark.parametrize("kv", ["f16", "i8", "fp8"])
def test_mass_ragged_with_empty_sequences(kv):
    check_mass(kv, 8, 2, 80, 16, [100, 33, 0, 700, 5], [3, 0, 17, 6, 0], max_prefix=2000, max_nodes=40, extra=7)


@pytest.mark.parametrize("p", [0, 20])
def test_mass_any_mask_and_rows_that_see_nothing(p):
    """Rows whose lse is -inf add nothing."""
    check_mass("f16", 8, 2, 80, 16, [p, 10], [40, 3], kind="any", seed=5)


@pytest.mark.parametrize("kv", ["f16", "i8", "fp8"])
@pytest.mark.parametrize("hkv", [1, 2, 3, 4, 6, 12])
def test_mass_of_a_decode_step(kv, hkv):
    """One query a sequence, head counts that fill a workgroup's waves and do not."""
    check_mass(kv, 2 * hkv, hkv, 80, 16, [300, 0, 64, 1025, 17], [1, 1, 1, 1, 0], seed=hkv)


@pytest.mark.parametrize("kv", ["f16", "i8"])
def test_mass_moves_and_commit_past_32_bits(kv):
    """Blocks 2^30 elements apart: byte offsets past 2^32, the dense pool's bits."""
    pool = U.Pool(kv, [70], 2, 80, 16, seed=2, extra=0)
    q, lse = torch.randn(10, 8, 80).half(), torch.full((10, 8), 5.0)
    base = torch.rand(1, 2, 70)
    want = mass(pool, q, lse, base, [60], [10], None, 8)
    got, tables = base.to(DEV), pool.tables.to(DEV)
    far, room = U.far(pool, DEV)
    pyvcpp.attention_mass(far, q.to(DEV), lse.to(DEV), got, tables, dev([0, 10]), dev([60]), 10, 60, 8)
    assert torch.equal(got.cpu(), want)
    pages, b = pool.to(DEV)
    moves, counts = dev([[[[1, 69], [17, 40]], [[0, 33], [2, 65]]]]), dev([[2, 2]])
    for x in (pages, far):
        pyvcpp.kv_evict_apply(x, tables, moves, counts)
        pyvcpp.kv_commit(x, tables, dev([40]), dev([[3, 29, 20]]), dev([3]), 30)
    torch.cuda.synchronize()
    for n in b:
        assert not torch.equal(b[n].cpu(), getattr(pool, n))
        assert torch.equal(torch.stack([r.view(b[n].dtype) for r in U.near(room, n, pool)]).reshape(b[n].shape), b[n])


def test_mass_missing_blocks_and_masked_rows():
    """Positions of missing blocks keep their scores; a drafted K row of NaN
    counts only where it is seen."""
    p, n = 100, 10
    pool = U.Pool("f16", [p + n], 2, 80, 16, seed=3)
    pool.tables[0, 2] = -1
    pool.tables[0, 4] = pool.nb + 1
    q = torch.randn(n, 8, 80).half()
    bits = [1 << i for i in range(n)]
    bits[3] = 0
    for j in range(n):
        bits[j] &= ~(1 << 6)  # nobody sees node 6
    pool.k[int(pool.tables[0, (p + 6) // 16]), 0, (p + 6) % 16] = float("nan")
    _, lse, weights = U.reference(pool, q, [p], [n], bits)
    before = torch.rand(1, 2, p + n)
    got = mass(pool, q, lse.float(), before, [p], [n], U.mask_words(bits, 1), 8)
    w, see = weights[0]
    w = torch.nan_to_num(w)
    want = before.double() + w.reshape(2, 4, n, p + n).sum((1, 2))
    assert float((got.double() - want).abs().max()) <= 8 * REL * float(want.max())
    hidden = list(range(32, 48)) + list(range(64, 80)) + [p + 6]
    assert torch.equal(got[..., hidden], before[..., hidden])


def test_mass_is_reproducible_and_replays():
    prefix, nodes = [900, 35], [12, 30]
    pool = U.Pool("i8", [a + b for a, b in zip(prefix, nodes)], 2, 80, 16, seed=2)
    pages, keep = pool.to(DEV)
    q = torch.randn(42, 8, 80).half().to(DEV)
    lse = torch.full((42, 8), 7.0, device=DEV)
    st, pf, tables = dev(U.starts(nodes)), dev(prefix), pool.tables.to(DEV)
    base = torch.rand(2, 2, 930, device=DEV)

    def go(s):
        pyvcpp.attention_mass(pages, q, lse, s, tables, st, pf, 30, 900, 8)

    want = base.clone()
    go(want)
    torch.cuda.synchronize()
    s = base.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go(s)
    side.synchronize()
    assert torch.equal(s, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(s)
    for _ in range(3):
        s.copy_(base)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(s, want)


# ---- plan -------------------------------------------------------------------


def plan_reference(scores, lens, budget, first, last, seen=None, positions=None):
    S, hkv, stride = scores.shape
    moves, new_scores, new_pos = {}, scores.clone(), torch.full((S, hkv, stride), -1, dtype=torch.int32)
    for s in range(S):
        n, total = lens[s], lens[s] if seen is None else seen[s]
        for h in range(hkv):
            w = scores[s, h, :n].tolist()
            at = [positions[s, h, j].item() if positions is not None and positions[s, h, j] >= 0 else total - n + j for j in range(n)]
            key = [math.inf if x < first or x >= total - last else (-math.inf if math.isnan(y) else y) for x, y in zip(at, w)]
            tier = [2 if x < first or x >= total - last else (0 if math.isnan(y) else 1) for x, y in zip(at, w)]
            best = set(sorted(range(n), key=lambda j: (-tier[j], -key[j], j))[:budget])
            to = [j for j in range(min(n, budget)) if j not in best]
            of = [j for j in range(budget, n) if j in best]
            assert len(to) == len(of)
            moves[s, h] = list(zip(to, of))
            row = list(range(min(n, budget)))
            for x, y in moves[s, h]:
                row[x] = y
            new_scores[s, h] = 0
            for i, j in enumerate(row):
                new_scores[s, h, i] = scores[s, h, j]
                new_pos[s, h, i] = at[j]
    return moves, new_scores, new_pos


def run_plan(scores, lens, budget, first=0, last=0, seen=None, positions=None, top=None, in_place=False, pos_out=True):
    S, hkv, stride = scores.shape
    top = max(lens + [1]) if top is None else top
    most = max(1, min(budget, top - budget))
    moves = torch.full((S, hkv, most, 2), -7, dtype=torch.int32, device=DEV)
    counts, new = torch.full((S, hkv), -7, dtype=torch.int32, device=DEV), torch.full((S,), -7, dtype=torch.int32, device=DEV)
    sc = scores.to(DEV)
    pos = None if positions is None else positions.to(DEV)
    so = sc if in_place else torch.full_like(sc, 9.0)
    po = (pos if in_place and pos is not None else torch.full((S, hkv, stride), 9, dtype=torch.int32, device=DEV)) if pos_out else None
    pyvcpp.kv_evict_plan(sc, dev(lens), top, budget, moves, counts, new, so, keep_first=first, keep_last=last,
                         seen_lens=None if seen is None else dev(seen), positions=pos, positions_out=po)
    torch.cuda.synchronize()
    return moves.cpu(), counts.cpu(), new.cpu(), so.cpu(), None if po is None else po.cpu()


def check_plan(scores, lens, budget, first=0, last=0, seen=None, positions=None, top=None, in_place=False):
    top = max(lens + [1]) if top is None else top
    moves, counts, new, so, po = run_plan(scores, lens, budget, first, last, seen, positions, top, in_place)
    want, ws, wp = plan_reference(scores, lens, budget, first, last, seen, positions)
    S, hkv, stride = scores.shape
    for s in range(S):
        assert int(new[s]) == min(lens[s], budget)
        for h in range(hkv):
            n = int(counts[s, h])
            assert [tuple(x) for x in moves[s, h, :n].tolist()] == want[s, h], (s, h)
            assert bool((moves[s, h, n:] == -7).all())
    assert torch.equal(so[..., :top].nan_to_num(77.0), ws[..., :top].nan_to_num(77.0))
    assert torch.equal(po[..., :top], wp[..., :top])
    if not in_place:
        assert bool((so[..., top:] == 9).all()) and bool((po[..., top:] == 9).all())
    return moves, counts, new, so, po


def some_scores(S, hkv, n, seed=0):
    return torch.randn(S, hkv, n, generator=torch.Generator().manual_seed(seed)).mul(2.5).exp()


@pytest.mark.parametrize("lens,budget", [
    ([1], 1), ([2], 1), ([63, 64, 65], 64), ([64, 65, 66, 130], 63), ([255, 256, 257], 255), ([100, 5, 0, 64], 32),
    ([1000, 700, 1], 999), ([1024], 700), ([1025], 700), ([2049, 2050, 2064, 2048], 2048), ([4096, 4097, 3000], 500), ([9000, 4097], 4096)])
def test_plan_lengths(lens, budget):
    check_plan(some_scores(len(lens), 3, max(lens) + 5), lens, budget)


@pytest.mark.parametrize("first,last", [(4, 0), (0, 16), (4, 60), (0, 64), (64, 0), (64, 36)])
def test_plan_protection(first, last):
    check_plan(some_scores(2, 2, 300, 1), [300, 180], 100, first, last)


def test_plan_after_earlier_cuts():
    """Slots out of order keep their token positions; appended ones are marked -1."""
    S, hkv, n, budget = 3, 2, 220, 200
    g = torch.Generator().manual_seed(3)
    lens, seen = [220, 210, 150], [900, 210, 5000]
    pos = torch.full((S, hkv, 230), -1, dtype=torch.int32)
    for h in range(hkv):
        pos[0, h, :budget] = torch.randperm(880, generator=g)[:budget].int()
        pos[2, h, :150] = torch.randperm(5000, generator=g)[:150].int()
    for in_place in (False, True):
        check_plan(some_scores(S, hkv, 230, 2), lens, budget, 4, 50, seen, pos, in_place=in_place)


@pytest.mark.parametrize("kind", ["equal", "two", "zeros", "denormal", "special", "negative"])
def test_plan_ties_and_odd_scores(kind):
    """Equal scores stay in slot order; NaN goes first, -0 counts as 0,
    infinities and subnormal numbers have their places."""
    s = some_scores(2, 2, 500, 4)
    if kind == "equal":
        s[:] = 0.25
    elif kind == "two":
        s = (s > 1).float()
    elif kind == "zeros":
        s[:] = 0.0
        s[..., ::3] = -0.0
        s[..., 7] = 1.0
    elif kind == "denormal":
        s = (torch.arange(500) % 37).float().expand(2, 2, 500) * 1e-44
        s = s.contiguous()
    elif kind == "special":
        s[..., ::5] = float("nan")
        s[..., 1::7] = float("inf")
        s[..., 2::11] = -float("inf")
    else:
        s = -s
    check_plan(s, [500, 333], 200, 3, 9)
    check_plan(s, [500, 333], 450, 0, 0)


@pytest.mark.parametrize("n", [32768, 32769, 50000])
def test_plan_long(n):
    """Rows that fill LDS, and rows that do not fit it."""
    check_plan(some_scores(1, 2, n, n), [n], n // 3, 4, 64)


def test_plan_in_place_and_loose_bounds():
    check_plan(some_scores(3, 2, 700, 5), [300, 600, 10], 256, 4, 32, top=700, in_place=True)
    check_plan(some_scores(3, 2, 700, 5), [300, 600, 10], 256, 4, 32, top=650)


def test_plan_without_positions_out_and_a_length_past_the_bound():
    s = some_scores(1, 2, 400, 6)
    a = run_plan(s, [400], 100, pos_out=False)
    b = run_plan(s, [400], 100)
    assert torch.equal(a[0], b[0]) and torch.equal(a[3], b[3])
    # (a longer context counts as the bound)
    moves, counts, new, so, po = run_plan(s, [400], 100, top=300)
    c = run_plan(s, [300], 100, top=300)
    assert torch.equal(moves, c[0]) and torch.equal(counts, c[1])


# ---- moves ------------------------------------------------------------------


def bytes_of(t):
    return t.cpu().contiguous().view(torch.uint8)


@pytest.mark.parametrize("kv", ["f32", "f16", "i8", "fp8"])
@pytest.mark.parametrize("D,hkv,bs", [(64, 8, 16), (80, 3, 16), (128, 2, 32)])
def test_apply_moves_rows(kv, D, hkv, bs):
    lens, budget = [300, 90, 40, 200], 64
    pool = U.Pool(kv, lens, hkv, D, bs, seed=1)
    pool.tables[3, 2] = -1  # rows of a missing block do not move
    scores = some_scores(4, hkv, 300, 2)
    want, _, _ = plan_reference(scores, lens, budget, 2, 8)
    moves, counts, new, _, _ = run_plan(scores, lens, budget, 2, 8)
    pages, b = pool.to(DEV)
    before = {n: t.clone().cpu() for n, t in b.items()}
    pyvcpp.kv_evict_apply(pages, pool.tables.to(DEV), moves.to(DEV), counts.to(DEV))
    torch.cuda.synchronize()
    expect = {n: t.clone() for n, t in before.items()}
    for (s, h), pairs in want.items():
        for to, of in pairs:
            x, y = int(pool.tables[s, to // bs]), int(pool.tables[s, of // bs])
            if x < 0 or y < 0:
                continue
            for n in ("k", "v"):
                expect[n][x, 0, to % bs, h] = before[n][y, 0, of % bs, h]
            if kv == "i8":
                for n in ("ks", "vs"):
                    expect[n][x, 0, h, to % bs] = before[n][y, 0, h, of % bs]
    for n in expect:
        assert torch.equal(bytes_of(b[n]), bytes_of(expect[n])), n


def test_apply_ignores_what_is_no_move():
    """Counts past max_moves, negative slots and slots past the table: skipped, nothing out of range is touched."""
    pool = U.Pool("f16", [64], 2, 80, 16, seed=1)
    pages, b = pool.to(DEV)
    before = {n: t.clone() for n, t in b.items()}
    moves = torch.tensor([[[[-1, 20], [3, 64], [2**31 - 1, 1]], [[5, -2**31], [70, 3], [-5, -5]]]], dtype=torch.int32, device=DEV)
    pyvcpp.kv_evict_apply(pages, pool.tables.to(DEV), moves, dev([[1000, 3]]))
    pyvcpp.kv_evict_apply(pages, pool.tables.to(DEV), moves, dev([[-1, 0]]))
    torch.cuda.synchronize()
    for n in b:
        assert torch.equal(b[n], before[n])


def commit_reference(pool, before, prefix, path, taken, max_nodes):
    out = {n: t.clone() for n, t in before.items()}
    bs = pool.bs
    for s, p in enumerate(prefix):
        for j in range(min(max(taken[s], 0), len(path[s]))):
            a = path[s][j]
            if not 0 <= a < max_nodes:
                continue
            to, of = p + j, p + a
            if max(to, of) // bs >= pool.tables.shape[1]:
                continue
            x, y = int(pool.tables[s, to // bs]), int(pool.tables[s, of // bs])
            if x < 0 or y < 0:
                continue
            for n in ("k", "v"):
                out[n][x, :, to % bs] = before[n][y, :, of % bs]
            if pool.kv == "i8":
                for n in ("ks", "vs"):
                    out[n][x, :, :, to % bs] = before[n][y, :, :, of % bs]
    return out


@pytest.mark.parametrize("kv", ["f32", "f16", "i8", "fp8"])
@pytest.mark.parametrize("D,hkv,bs,layers", [(64, 8, 16, 1), (80, 3, 16, 5), (128, 2, 32, 2)])
def test_commit_moves_an_accepted_path(kv, D, hkv, bs, layers):
    prefix, nodes = [30, 0, 47, 16, 100], 40
    pool = U.Pool(kv, [p + nodes for p in prefix], hkv, D, bs, layers=layers, seed=1)
    pool.tables[4, (100 + 20) // bs] = -1
    path = [[0, 2, 5, 9, 33], [1, 2, 3, 4, 39], [7, 7, 7, 7, 7], [0, -1, 40, 3, 2**31 - 1], [20, 3, 18, 22, 1]]
    taken = [5, 3, 5, 5, 9]
    pages, b = pool.to(DEV)
    before = {n: t.clone().cpu() for n, t in b.items()}
    pyvcpp.kv_commit(pages, pool.tables.to(DEV), dev(prefix), dev(path), dev(taken), nodes, num_layers=layers,
                     layer_stride=bs * hkv * D, scale_layer_stride=hkv * bs)
    torch.cuda.synchronize()
    want = commit_reference(pool, before, prefix, path, taken, nodes)
    for n in want:
        assert torch.equal(bytes_of(b[n]), bytes_of(want[n])), n


@pytest.mark.parametrize("kv", ["f16", "i8"])
@pytest.mark.parametrize("n", [1, 63, 200, 256])
def test_commit_reads_all_before_it_writes(kv, n):
    """A permutation of the whole tree: every source is another row's target."""
    pool = U.Pool(kv, [300], 4, 80, 16, layers=2, seed=n)
    path = [torch.randperm(n, generator=torch.Generator().manual_seed(n)).tolist()]
    pages, b = pool.to(DEV)
    before = {k: t.clone().cpu() for k, t in b.items()}
    pyvcpp.kv_commit(pages, pool.tables.to(DEV), dev([37]), dev(path), dev([n]), n, num_layers=2, layer_stride=16 * 4 * 80,
                     scale_layer_stride=64)
    torch.cuda.synchronize()
    want = commit_reference(pool, before, [37], path, [n], n)
    for k in want:
        assert torch.equal(bytes_of(b[k]), bytes_of(want[k])), k


def test_commit_past_the_table_and_empty():
    pool = U.Pool("f16", [64, 64], 2, 80, 16, seed=1)
    pages, b = pool.to(DEV)
    before = {n: t.clone() for n, t in b.items()}
    pyvcpp.kv_commit(pages, pool.tables.to(DEV), dev([60, 10]), dev([[9, 12, 30], [4, 5, 6]]), dev([3, 0]), 40)
    pyvcpp.kv_commit(pages, pool.tables.to(DEV), dev([2**31 - 1, -5]), dev([[9, 12, 30], [0, 1, 2]]), dev([3, 3]), 40)
    torch.cuda.synchronize()
    for n in b:
        assert torch.equal(b[n], before[n])


def test_plan_apply_and_commit_replay():
    """Captured together; replays give the eager result each time."""
    pool = U.Pool("f16", [200, 120], 2, 80, 16, seed=1)
    pages, b = pool.to(DEV)
    start = {n: t.clone() for n, t in b.items()}
    scores = some_scores(2, 2, 200, 3).to(DEV)
    lens, tables, prefix = dev([200, 120]), pool.tables.to(DEV), dev([150, 90])
    path, taken = dev([[3, 5, 9], [1, 2, 20]]), dev([3, 2])
    moves = torch.full((2, 2, 64, 2), -1, dtype=torch.int32, device=DEV)
    counts, new, so = torch.zeros(2, 2, dtype=torch.int32, device=DEV), dev([0, 0]), torch.zeros_like(scores)

    def go():
        pyvcpp.kv_commit(pages, tables, prefix, path, taken, 30)
        pyvcpp.kv_evict_plan(scores, lens, 200, 64, moves, counts, new, so, keep_last=8)
        pyvcpp.kv_evict_apply(pages, tables, moves, counts)

    go()
    torch.cuda.synchronize()
    want = [t.clone() for t in (b["k"], b["v"], moves, counts, new, so)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for _ in range(3):
        for n in b:
            b[n].copy_(start[n])
        so.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip((b["k"], b["v"], moves, counts, new, so), want):
            assert torch.equal(x, y)


# ---- together ---------------------------------------------------------------


@pytest.mark.parametrize("kv", ["f16", "i8", "fp8"])
def test_drafted_decoding_on_a_bounded_cache(kv):
    """Some steps as an engine runs them: draft rows written, the tree verified,
    the accepted path committed, its weights added, the cache cut to a budget,
    and a decode on what is left -- each against 64 bits on a plain mirror of
    what every kv head holds."""
    H, hkv, D, bs, budget = 8, 2, 80, 16, 96
    ctx = [130, 60]
    top = 200
    pool = U.Pool(kv, [top, top], hkv, D, bs, seed=1)
    pages, b = pool.to(DEV)
    tables = pool.tables.to(DEV)
    g = torch.Generator().manual_seed(5)
    scores = torch.zeros(2, hkv, top, device=DEV)
    positions = torch.full((2, hkv, top), -1, dtype=torch.int32, device=DEV)
    seen, lens = list(ctx), list(ctx)
    kc, vc = ([pool.rows(s, top, w)[0] for s in range(2)] for w in ("k", "v"))  # mirrors [slot][head][D]
    mirror_scores = torch.zeros(2, hkv, top, dtype=torch.float64)
    for step in range(4):
        nodes = [7, 12]
        n = sum(nodes)
        bits = [x for i, m in enumerate(nodes) for x in U.tree_bits(m, 10 * step + i)]
        new_k, new_v = torch.randn(n, hkv, D, generator=g), torch.randn(n, hkv, D, generator=g)
        slots = [int(pool.tables[s, (lens[s] + i) // bs]) * bs + (lens[s] + i) % bs for s in range(2) for i in range(nodes[s])]
        pyvcpp.write_kv(pages, new_k.to(DEV), new_v.to(DEV), dev(slots, torch.int64), fp16_round_nearest=True)
        torch.cuda.synchronize()
        for name in b:
            setattr(pool, name, b[name].cpu())
        for s in range(2):  # the written rows as the pages hold them
            kr, vr = pool.rows(s, top, "k")[0], pool.rows(s, top, "v")[0]
            kc[s][lens[s]:lens[s] + nodes[s]] = kr[lens[s]:lens[s] + nodes[s]]
            vc[s][lens[s]:lens[s] + nodes[s]] = vr[lens[s]:lens[s] + nodes[s]]
            assert torch.equal(kr[:lens[s]], kc[s][:lens[s]])
        q = torch.randn(n, H, D, generator=g).half()
        out, lse = torch.zeros(n, H, D, device=DEV), torch.zeros(n, H, device=DEV)
        st = dev(U.starts(nodes))
        pyvcpp.paged_tree_attention(pages, q.to(DEV), out, tables, st, dev(lens), 12, top - 12, H,
                                    tree_mask=U.mask_words(bits, 1).to(DEV), lse=lse)
        want, zw, _ = U.reference(pool, q, lens, nodes, bits)
        torch.cuda.synchronize()
        assert float((out.cpu().double() - want).norm()) <= REL * float(want.norm())
        # the longest branch is accepted
        path, taken, at = [], [], 0
        for m in nodes:
            leaf = max(range(m), key=lambda i: (bin(bits[at + i]).count("1"), i))
            p = [j for j in range(m) if bits[at + leaf] >> j & 1]
            path.append(p + [-1] * (12 - len(p)))
            taken.append(len(p))
            at += m
        pyvcpp.kv_commit(pages, tables, dev(lens), dev(path), dev(taken), 12)
        acc = [U.starts(nodes)[s] + j for s in range(2) for j in path[s][:taken[s]]]
        ast = dev(U.starts(taken))
        pyvcpp.attention_mass(pages, q.to(DEV)[acc].contiguous(), lse[acc].contiguous(), scores, tables, ast, dev(lens), 12,
                              top - 12, H)
        for s in range(2):
            keep = [lens[s] + j for j in path[s][:taken[s]]]
            for x in (kc[s], vc[s]):
                x[lens[s]:lens[s] + taken[s]] = x[keep].clone()
            rows = [U.starts(nodes)[s] + j for j in path[s][:taken[s]]]
            for i, r in enumerate(rows):
                L = lens[s] + i + 1
                for h in range(H):
                    x = kc[s][:L, h // 4] @ q[r, h].double() / math.sqrt(D)
                    mirror_scores[s, h // 4, :L] += torch.softmax(x, 0)
            lens[s] += taken[s]
            seen[s] += taken[s]
        torch.cuda.synchronize()
        got = scores.cpu().double()
        assert float((got - mirror_scores).norm()) <= 4 * REL * float(mirror_scores.norm())
        # cut back
        moves = torch.zeros(2, hkv, top, 2, dtype=torch.int32, device=DEV)
        counts, new = torch.zeros(2, hkv, dtype=torch.int32, device=DEV), dev([0, 0])
        was = scores.cpu()
        ref, ws, wp = plan_reference(was, lens, budget, 2, 24, seen, positions.cpu())
        pyvcpp.kv_evict_plan(scores, dev(lens), top, budget, moves, counts, new, scores, keep_first=2, keep_last=24,
                             seen_lens=dev(seen), positions=positions, positions_out=positions)
        pyvcpp.kv_evict_apply(pages, tables, moves, counts)
        torch.cuda.synchronize()
        assert torch.equal(scores.cpu(), ws) and torch.equal(positions.cpu(), wp)
        order = mirror_scores.clone()
        for (s, h), pairs in ref.items():
            for to, of in pairs:
                kc[s][to, h], vc[s][to, h] = kc[s][of, h].clone(), vc[s][of, h].clone()
                order[s, h, to] = mirror_scores[s, h, of]
            order[s, h, min(lens[s], budget):] = 0
        mirror_scores = order
        lens = [min(x, budget) for x in lens]
        assert new.tolist() == lens
        # a decode on what is left
        dq = torch.randn(2, H, D, generator=g)
        dout = torch.zeros(2, H, D, device=DEV)
        pyvcpp.paged_decode(pages, dq.to(DEV), dout, tables, dev(lens), max(lens), H)
        torch.cuda.synchronize()
        for s in range(2):
            for h in range(H):
                x = torch.softmax(kc[s][:lens[s], h // 4] @ dq[s, h].double() / math.sqrt(D), 0)
                w = x @ vc[s][:lens[s], h // 4]
                assert float((dout[s, h].cpu().double() - w).norm()) <= 2e-5 * float(w.norm()) + 1e-9
