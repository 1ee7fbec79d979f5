"""vcpp_paged_tree_attention on the GPU against its definition in 64 bits.

Tolerance.  K, Q and V enter the matrix products exactly (fp16 values, or int8
and FP8 codes widened to fp16), and products of two fp16 numbers are exact in
fp32.  What is rounded: the fp32 sums of head_dim products and the scaled score
(a few 2^-24 of a magnitude of at most 16 in these inputs: 16 * 4 * 2^-24 =
3.8e-6 on the exponent, and as much relative on a weight), exp2 (2 ulp), P as
two fp16 numbers (half a step of the low one: 2^-11 * 2^-12 = 1.2e-7), and the
sums of the outputs (some 2^-24 each).  5e-6 normwise covers their sum; an
element, up to 4 times the outputs' size, 4e-5."""
import ctypes
import math

import pytest
import torch

import pyvcpp
import tree_util as U

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
REL, ABS = 5e-6, 4e-5


def call(pool, q, prefix, nodes, mask, H, max_prefix=None, max_nodes=None, out=None, lse=True, workspace=None,
         tables=None):
    pages, keep = pool.to(DEV)
    rows = q.shape[0]
    o = torch.full((rows, H, pool.D), float("nan"), device=DEV) if out is None else out
    z = torch.full((rows, H), float("nan"), device=DEV) if lse is True else lse
    pyvcpp.paged_tree_attention(
        pages, q.to(DEV), o, (pool.tables if tables is None else tables).to(DEV),
        torch.tensor(U.starts(nodes), dtype=torch.int32, device=DEV), torch.tensor(prefix, dtype=torch.int32, device=DEV),
        max(nodes) if max_nodes is None else max_nodes, max(prefix) if max_prefix is None else max_prefix, H,
        tree_mask=None if mask is None else mask.to(DEV), lse=z, workspace=workspace)
    torch.cuda.synchronize()
    return o.cpu(), None if z is None else z.cpu()


def close(got, want, what=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin), "%s: finite elsewhere" % what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "%s: NaN elsewhere" % what
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)])
    d = (got - want)[fin]
    if d.numel():
        assert float(d.abs().max()) <= ABS * max(1.0, float(want[fin].abs().max())), "%s: max %.3g" % (what, float(d.abs().max()))
        n = float(want[fin].norm())
        assert float(d.norm()) <= REL * n if n else float(d.norm()) == 0.0, "%s: rel %.3g" % (what, float(d.norm()) / max(n, 1e-300))


def check(kv, H, hkv, D, bs, prefix, nodes, kind="tree", seed=1, std=1.0, words=None, **kw):
    pool = U.Pool(kv, [p + n for p, n in zip(prefix, nodes)], hkv, D, bs, seed=seed, std=std)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(sum(nodes), H, D, generator=g).half()
    bits = [b for i, n in enumerate(nodes) for b in U.tree_bits(n, seed + i, kind)]
    words = (max(nodes) + 63) // 64 if words is None else words
    out, lse = call(pool, q, prefix, nodes, U.mask_words(bits, words), H, **kw)
    want, zw, _ = U.reference(pool, q, prefix, nodes, bits)
    close(out, want, "out")
    close(lse, zw, "lse")
    return pool, q, bits, out, lse


@pytest.mark.parametrize("kv", ["f16", "i8", "fp8"])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("H,hkv", [(8, 8), (6, 2), (7, 1), (16, 2), (16, 1)])
def test_types_and_heads(kv, D, H, hkv):
    """Every page type and head size, group sizes 1 to 16."""
    check(kv, H, hkv, D, 16, [37, 0, 130], [9, 5, 16])


@pytest.mark.parametrize("kv", ["f16", "i8", "fp8"])
@pytest.mark.parametrize("n", [1, 2, 3, 8, 9, 31, 33, 64, 65, 100, 128, 129, 256])
def test_tree_sizes(kv, n):
    """One node to the most (row tiles of every size, one to four mask words)."""
    check(kv, 8, 2, 80, 16, [50], [n], seed=n)


@pytest.mark.parametrize("kv,D", [("f16", 80), ("i8", 128), ("fp8", 64)])
@pytest.mark.parametrize("p", [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 127, 128, 129, 255, 1000, 4097])
def test_prefix_lengths(kv, D, p):
    """Prefixes around pages, key blocks and parts."""
    check(kv, 8, 1, D, 16, [p], [7], seed=p)


@pytest.mark.parametrize("bs", [16, 32, 48, 64])
def test_page_sizes(bs):
    check("f16", 8, 2, 80, bs, [3, 200, 77], [4, 12, 1])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [17, 40, 90])
def test_row_tiles_other_dims(D, n):
    check("f16", 8, 2, D, 16, [70], [n], seed=n)
    check("i8", 8, 2, D, 16, [70], [n], seed=n)


@pytest.mark.parametrize("kv", ["f16", "i8", "fp8"])
def test_ragged_batch_with_empty_sequences(kv):
    """Sequences without nodes between others, prefix 0, loose bounds."""
    prefix, nodes = [100, 33, 0, 700, 5, 0], [3, 0, 17, 6, 0, 1]
    check(kv, 8, 2, 80, 16, prefix, nodes, max_prefix=3000, max_nodes=40, words=1)


@pytest.mark.parametrize("kv", ["f16", "i8", "fp8"])
@pytest.mark.parametrize("seqs", [64, 65, 150])
def test_many_sequences(kv, seqs):
    """More sequences than lanes, most of them short, some empty, one long."""
    prefix = [(37 * s) % 90 for s in range(seqs)]
    prefix[seqs - 2] = 1500
    check(kv, 4, 2, 80, 16, prefix, [(5 * s) % 7 for s in range(seqs)], seed=4)


@pytest.mark.parametrize("kv", ["f16", "i8", "fp8"])
@pytest.mark.parametrize("p", [0, 20, 64])
def test_any_mask_and_empty_rows(kv, p):
    """Masks that are no trees, rows that see no node; at prefix 0 those are zeros with lse -inf."""
    _, _, bits, out, lse = check(kv, 8, 2, 80, 16, [p, 10], [40, 3], kind="any", seed=5)
    if p == 0:
        empty = [i for i in range(40) if bits[i] == 0]
        assert empty
        assert bool((out[empty] == 0).all()) and bool((lse[empty] == -math.inf).all())


@pytest.mark.parametrize("kv", ["f16", "i8", "fp8"])
def test_missing_blocks(kv):
    """Table entries of -1 and past the pool are skipped, in the prefix and in the tree."""
    pool = U.Pool(kv, [200, 90], 2, 80, 16, seed=3)
    pool.tables[0, 2] = -1
    pool.tables[0, 7] = pool.nb + 5
    pool.tables[1, 5] = -1  # the tree's own block
    prefix, nodes = [190, 80], [10, 10]
    bits = [b for i, n in enumerate(nodes) for b in U.tree_bits(n, i)]
    q = torch.randn(20, 8, 80, generator=torch.Generator().manual_seed(1)).half()
    out, lse = call(pool, q, prefix, nodes, U.mask_words(bits, 1), 8)
    want, zw, _ = U.reference(pool, q, prefix, nodes, bits)
    close(out, want)
    close(lse, zw)


def test_table_shorter_than_context():
    """Positions past the table are skipped."""
    pool = U.Pool("f16", [100], 2, 80, 16, seed=3)
    pool.tables = pool.tables[:, :4].contiguous()
    bits = U.tree_bits(10, 1)
    q = torch.randn(10, 8, 80).half()
    out, lse = call(pool, q, [90], [10], U.mask_words(bits, 1), 8)
    want, zw, _ = U.reference(pool, q, [90], [10], bits)
    close(out, want)
    close(lse, zw)


@pytest.mark.parametrize("kv,what", [("f16", "v"), ("f16", "k"), ("i8", "vs"), ("i8", "ks"), ("fp8", "v"), ("fp8", "k")])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_not_finite_in_masked_places(kv, what, value):
    """A drafted row of NaN or inf reaches only the rows that see it: the others
    keep the bits they have without it."""
    if kv == "fp8" and value == float("inf"):
        pytest.skip("FP8 pages hold no infinity")
    p, n = 50, 20
    pool = U.Pool(kv, [p + n], 2, 80, 16, seed=9)
    bits = U.tree_bits(n, 4)
    q = torch.randn(n, 8, 80, generator=torch.Generator().manual_seed(2)).half()
    mask = U.mask_words(bits, 1)
    out0, lse0 = call(pool, q, [p], [n], mask, 8)
    bad = 7
    bid, at = int(pool.tables[0, (p + bad) // 16]), (p + bad) % 16
    t = getattr(pool, what)
    if what in ("ks", "vs"):
        t[bid, 0, :, at] = value
    else:
        t[bid, 0, at, :, ::3] = 0x7F if kv == "fp8" else value
    out, lse = call(pool, q, [p], [n], mask, 8)
    for i in range(n):
        if bits[i] >> bad & 1:
            assert not torch.isfinite(out[i]).all()
        else:
            assert torch.equal(out[i], out0[i]) and torch.equal(lse[i], lse0[i]), i


def test_not_finite_behind_the_tree():
    """Whatever lies in the last page behind the tree is not read."""
    pool = U.Pool("f16", [64], 2, 80, 16, seed=9)
    bits = U.tree_bits(5, 4)
    q = torch.randn(5, 8, 80).half()
    mask = U.mask_words(bits, 1)
    a = call(pool, q, [40], [5], mask, 8)
    b = int(pool.tables[0, 2])
    pool.k[b, 0, 13:] = float("nan")
    pool.v[b, 0, 13:] = float("inf")
    c = call(pool, q, [40], [5], mask, 8)
    assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


@pytest.mark.parametrize("kv", ["f16", "i8"])
@pytest.mark.parametrize("scale", [1e-3, 30.0])
def test_wide_scores_and_scales(kv, scale):
    """Tiny and large values: int8 scales from subnormal fp16 to far above 1,
    scores whose maximum moves in almost every block (a weight's relative
    error grows with its score's size: 300 here, 20 times the 16 above)."""
    pool = U.Pool(kv, [700], 2, 80, 16, seed=3, std=scale)
    if kv == "i8":
        pool.vs *= 100.0 if scale > 1 else 0.01
    bits = U.tree_bits(12, 1)
    q = torch.randn(12, 8, 80, generator=torch.Generator().manual_seed(1)).half()
    out, lse = call(pool, q, [688], [12], U.mask_words(bits, 1), 8)
    want, zw, _ = U.reference(pool, q, [688], [12], bits)
    f = 20 if scale > 1 else 1
    d = (out.double() - want)
    assert float(d.norm()) <= f * REL * float(want.norm())
    assert float((lse.double() - zw).abs().max()) <= f * ABS


def test_one_heavy_key_among_many_light_ones():
    """A weight of 1 beside thousands of 2^-14 each: the light ones together
    weigh as much, and none of them may lose its low bits."""
    p, n = 16384, 4
    pool = U.Pool("f16", [p + n], 1, 64, 16, seed=3)
    pool.k.zero_()
    b = int(pool.tables[0, 3])
    pool.k[b, 0, 5, 0, 0] = 8.0
    q = torch.zeros(n, 2, 64)
    q[..., 0] = 14 * math.log(2)  # q k / 8 = ln 2^14
    q = q.half()
    bits = U.tree_bits(n, 1)
    out, lse = call(pool, q, [p], [n], U.mask_words(bits, 1), 2)
    want, zw, _ = U.reference(pool, q, [p], [n], bits)
    close(out, want)
    close(lse, zw)


@pytest.mark.parametrize("kv", ["f16", "i8", "fp8"])
def test_chain_without_a_mask(kv):
    """No mask: the chain, bit for bit as its explicit mask, with and without lse."""
    prefix, nodes = [300, 0, 61], [33, 70, 1]
    pool = U.Pool(kv, [a + b for a, b in zip(prefix, nodes)], 2, 80, 16, seed=2)
    q = torch.randn(sum(nodes), 8, 80).half()
    bits = [b for n in nodes for b in U.tree_bits(n, 0, "chain")]
    a = call(pool, q, prefix, nodes, U.mask_words(bits, 2), 8)
    b = call(pool, q, prefix, nodes, None, 8)
    c = call(pool, q, prefix, nodes, None, 8, lse=None)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(c[0], b[0])


def test_one_token_is_a_decode():
    """One node without drafts: the decode of that token (fp32 q rounded to
    fp16 beforehand, the same logits in both)."""
    ctx = [1, 17, 300, 2000]
    pool = U.Pool("f16", ctx, 8, 80, 16, seed=2)
    q = torch.randn(4, 64, 80).half()
    out, _ = call(pool, q, [c - 1 for c in ctx], [1] * 4, None, 64)
    pages, keep = pool.to(DEV)
    want = torch.zeros(4, 64, 80, device=DEV)
    pyvcpp.paged_decode(pages, q.float().to(DEV), want, pool.tables.to(DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV),
                        max(ctx), 64)
    torch.cuda.synchronize()
    close(out, want.cpu().double())


def test_rows_behind_the_last_sequence_stay():
    """q and out may have more rows than the trees: they are left as they were."""
    prefix, nodes = [30, 45], [5, 9]
    pool = U.Pool("f16", [60, 60], 2, 80, 16, seed=2)
    q = torch.randn(18, 8, 80).half()
    out = torch.full((18, 8, 80), 7.0, device=DEV)
    lse = torch.full((18, 8), 7.0, device=DEV)
    bits = [b for n in nodes for b in U.tree_bits(n, 0)]
    mask = torch.zeros(18, 1, dtype=torch.int64)
    mask[:14] = U.mask_words(bits, 1)
    o, z = call(pool, q, prefix, nodes, mask, 8, out=out, lse=lse)
    want, zw, _ = U.reference(pool, q[:14], prefix, nodes, bits)
    close(o[:14], want)
    close(z[:14], zw)
    assert bool((o[14:] == 7).all()) and bool((z[14:] == 7).all())


def test_layer_slab_of_a_pool_of_layers():
    """A layer inside blocks of several layers (block_stride of all of them)."""
    pool = U.Pool("i8", [120], 2, 80, 16, layers=3, seed=2)
    pages, b = pool.to(DEV)
    page = 16 * 2 * 80
    view = pyvcpp.KVPages(pages.dtype, 16, 2, 80, pool.nb, 3 * page, 3 * 2 * 16, pages.k + 2 * page, pages.v + 2 * page,
                          pages.k_scale + 2 * 2 * 16 * 2, pages.v_scale + 2 * 2 * 16 * 2)
    q = torch.randn(6, 8, 80).half()
    out, lse = torch.zeros(6, 8, 80, device=DEV), torch.zeros(6, 8, device=DEV)
    pyvcpp.paged_tree_attention(view, q.to(DEV), out, pool.tables.to(DEV), torch.tensor([0, 6], dtype=torch.int32, device=DEV),
                                torch.tensor([114], dtype=torch.int32, device=DEV), 6, 114, 8, lse=lse)
    for name in ("k", "v", "ks", "vs"):
        setattr(pool, name, getattr(pool, name)[:, 2:3].contiguous())
    want, zw, _ = U.reference(pool, q, [114], [6], U.tree_bits(6, 0, "chain"))
    close(out.cpu(), want)
    close(lse.cpu(), zw)


@pytest.mark.parametrize("kv", ["f16", "i8", "fp8"])
def test_pages_past_32_bits(kv):
    """Blocks 2^30 elements apart: byte offsets past 2^32, the dense pool's bits."""
    prefix, nodes = [60, 9], [10, 4]
    pool = U.Pool(kv, [70, 13], 2, 80, 16, seed=2, extra=0)
    q = torch.randn(14, 8, 80).half()
    want = call(pool, q, prefix, nodes, None, 8)
    pages, keep = U.far(pool, DEV)
    out, lse = torch.zeros(14, 8, 80, device=DEV), torch.zeros(14, 8, device=DEV)
    pyvcpp.paged_tree_attention(pages, q.to(DEV), out, pool.tables.to(DEV),
                                torch.tensor([0, 10, 14], dtype=torch.int32, device=DEV),
                                torch.tensor(prefix, dtype=torch.int32, device=DEV), 10, 60, 8, lse=lse)
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), want[0]) and torch.equal(lse.cpu(), want[1])


def test_byte_pages_on_8_byte_bases():
    """FP8 pages need 8-byte bases only: the aligned pool's bits."""
    pool = U.Pool("fp8", [300], 2, 80, 16, seed=2)
    q = torch.randn(10, 8, 80).half()
    want = call(pool, q, [290], [10], None, 8)
    pages, b = pool.to(DEV)
    room = {n: torch.zeros(b[n].numel() + 16, dtype=torch.uint8, device=DEV) for n in ("k", "v")}
    for n in room:
        room[n][8:8 + b[n].numel()] = b[n].flatten()
    view = pyvcpp.KVPages(pages.dtype, 16, 2, 80, pool.nb, 16 * 2 * 80, 0, room["k"].data_ptr() + 8, room["v"].data_ptr() + 8,
                          None, None)
    out, lse = torch.zeros(10, 8, 80, device=DEV), torch.zeros(10, 8, device=DEV)
    pyvcpp.paged_tree_attention(view, q.to(DEV), out, pool.tables.to(DEV), torch.tensor([0, 10], dtype=torch.int32, device=DEV),
                                torch.tensor([290], dtype=torch.int32, device=DEV), 10, 290, 8, lse=lse)
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), want[0]) and torch.equal(lse.cpu(), want[1])


def test_given_stream_without_a_workspace():
    """`stream` other than the current one: the scratch that the call allocates
    stays its own while tensors come and go on the current stream."""
    pool = U.Pool("f16", [5000], 2, 80, 16, seed=2)
    q = torch.randn(9, 8, 80).half()
    want = call(pool, q, [4991], [9], None, 8)
    pages, keep = pool.to(DEV)
    args = (q.to(DEV), pool.tables.to(DEV), torch.tensor([0, 9], dtype=torch.int32, device=DEV),
            torch.tensor([4991], dtype=torch.int32, device=DEV))
    need = pyvcpp.tree_workspace_size(pages, 1, 9, 4991, 8)
    outs = [torch.zeros(9, 8, 80, device=DEV) for _ in range(8)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for o in outs:
        pyvcpp.paged_tree_attention(pages, args[0], o, args[1], args[2], args[3], 9, 4991, 8, stream=side)
        torch.full((need,), 255, dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o.cpu(), want[0])


def test_workspace_exact_and_garbage():
    """The stated bytes suffice, and what the buffer held does not matter."""
    pool = U.Pool("f16", [5000], 2, 80, 16, seed=2)
    pages, _ = pool.to(DEV)
    need = pyvcpp.tree_workspace_size(pages, 1, 9, 4991, 8)
    assert need > 0
    q = torch.randn(9, 8, 80).half()
    big = torch.full((need + 4096,), 255, dtype=torch.uint8, device=DEV)
    a = call(pool, q, [4991], [9], None, 8, workspace=big[:need])
    assert bool((big[need:] == 255).all())
    b = call(pool, q, [4991], [9], None, 8)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_side_stream_and_graph_replays():
    """On another stream, and captured: three replays with eager work between
    them give the eager call's bits."""
    prefix, nodes = [900, 35, 0], [12, 30, 3]
    pool = U.Pool("fp8", [a + b for a, b in zip(prefix, nodes)], 2, 80, 16, seed=2)
    pages, keep = pool.to(DEV)
    q = torch.randn(45, 8, 80).half().to(DEV)
    st, pf = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (U.starts(nodes), prefix))
    bits = [b for i, n in enumerate(nodes) for b in U.tree_bits(n, i)]
    mask, tables = U.mask_words(bits, 1).to(DEV), pool.tables.to(DEV)
    ws = torch.empty(max(16, pyvcpp.tree_workspace_size(pages, 3, 30, 900, 8)), dtype=torch.uint8, device=DEV)

    def go(out, lse):
        pyvcpp.paged_tree_attention(pages, q, out, tables, st, pf, 30, 900, 8, tree_mask=mask, lse=lse, workspace=ws)

    want, zw = torch.zeros(45, 8, 80, device=DEV), torch.zeros(45, 8, device=DEV)
    go(want, zw)
    torch.cuda.synchronize()
    out, lse = torch.zeros_like(want), torch.zeros_like(zw)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        go(out, lse)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, zw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(out, lse)
    for _ in range(3):
        out.fill_(-1.0)
        lse.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, zw)


def test_refuses_what_it_would_misread():
    """The binding refuses strided, wrongly typed and misplaced tensors."""
    pool = U.Pool("f16", [64], 2, 80, 16)
    pages, _ = pool.to(DEV)
    t, st, pf = pool.tables.to(DEV), torch.tensor([0, 4], dtype=torch.int32, device=DEV), torch.tensor([60], dtype=torch.int32, device=DEV)
    q, out = torch.randn(4, 8, 80, device=DEV).half(), torch.zeros(4, 8, 80, device=DEV)
    for bad in (dict(q=q.float()), dict(q=torch.randn(4, 80, 8, device=DEV).half().transpose(1, 2)), dict(out=out.half()),
                dict(st=st.long()), dict(lse=torch.zeros(4, 9, device=DEV)), dict(q=q.cpu()),
                dict(mask=torch.zeros(4, 1, dtype=torch.int32, device=DEV)), dict(mask=torch.zeros(3, 1, dtype=torch.int64, device=DEV))):
        with pytest.raises(ValueError):
            pyvcpp.paged_tree_attention(pages, bad.get("q", q), bad.get("out", out), t, bad.get("st", st), pf, 4, 60, 8,
                                        tree_mask=bad.get("mask"), lse=bad.get("lse"))
    with pytest.raises(pyvcpp.VcppError):
        pyvcpp.paged_tree_attention(pages, q, out, t, st, pf, 300, 60, 8)  # more nodes than a tree may have
