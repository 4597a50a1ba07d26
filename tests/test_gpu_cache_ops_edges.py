"""The cache operators at their edges: values that are no numbers, scales and queries of very
different size, masks and nodes beyond what a step names, graphs and streams."""
import numpy as np
import pytest
import torch

from test_gpu_cache_ops import F16, F32, NP, Q8, Cache, attend, check, dev, plain, random_tree

pytestmark = pytest.mark.gpu


def set_rows(c, which, index, row, slot=0, layer=0):
    """K (0) or V (1) of place `index` of a slot becomes `row` [hd], or one number, for every head; on an
    8-bit cache the place's scale becomes `row`."""
    raw = c.raw().copy()
    page, t = c.table[slot, index // 16], index % 16
    if c.kv == Q8:
        raw[layer, page, which, :, 4 * t:4 * t + 4] = np.array([row], np.float32).view(np.uint8)
    else:
        b = c.hd * (2 if c.kv == F16 else 4)
        raw[layer, page, which, :, t * b:(t + 1) * b] = np.broadcast_to(np.asarray(row, NP[c.kv]), (c.hd,)).copy().view(np.uint8)
    c.pool.copy_(torch.from_numpy(raw.reshape(-1)))


# nodes, nq, nkv, hd: up to 8, 16, 32, 64 and more rows a kv head, and any head_dim
ROWS = [(5, 2, 2, 64), (6, 2, 2, 128), (12, 2, 2, 64), (13, 1, 1, 128), (14, 4, 2, 64), (14, 4, 2, 128), (20, 6, 2, 64), (40, 8, 2, 128),
        (9, 4, 2, 40)]


@pytest.mark.parametrize("kv", [F32, F16])
@pytest.mark.parametrize("nodes,nq,nkv,hd", ROWS)
@pytest.mark.parametrize("ctx", [0, 5, 31, 120])
def test_infinities_in_v_of_many_nodes(sb, ctx, nodes, nq, nkv, hd, kv):
    """Every second node's V holds infinities and is seen by that node alone: the other rows are the same
    bits as without them, wherever in a tile the nodes lie, in every call."""
    rng = np.random.default_rng(ctx + nodes)
    c = Cache(sb, kv, 1, nkv, hd, [ctx + nodes], seed=2)
    bad = np.arange(1, nodes, 2)
    masks = np.array([(1 << i) | (1 if i else 0) for i in range(nodes)], np.uint64)      # itself and the root
    q = rng.normal(0, 1, (nodes, nq, hd)).astype(np.float32)
    clean = attend(sb, c, 0, [nodes], [ctx], masks, q, 0.1)
    for b in bad:
        set_rows(c, 1, ctx + b, np.where(np.arange(hd) % 3 == 0, np.inf, 1.0))
    others = np.arange(nodes) % 2 == 0
    for _ in range(3):
        dirty = attend(sb, c, 0, [nodes], [ctx], masks, q, 0.1)
        assert np.array_equal(dirty[others], clean[others])
        assert not np.isfinite(dirty[bad][..., ::3]).any()


def test_accept_of_more_sequences_than_32_bits_of_outputs(sb):
    """The last of 2^25 + 3 sequences: its outputs lie beyond 2^31 elements."""
    n = (1 << 25) + 3
    if torch.cuda.mem_get_info()[0] < 4 * (2 * 64 * n) + (4 << 30):
        pytest.skip("needs 21 GB")
    c = Cache(sb, F16, 1, 1, 4, [8])
    off = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    off[n] = 2                                           # two nodes of the last sequence, the second one matches
    slot, ctx, cnt = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(3))
    mask, parent = dev(np.array([1, 3], np.int64)), dev(np.array([-1, 0], np.int32))
    token, target = dev(np.array([5, 6], np.int32)), dev(np.array([6, 7], np.int32))
    node, new = (torch.full((n, 64), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    tree = sb.TreeBatch(n_seq=n, rows=2, max_nodes=2, row_off=off.data_ptr(), slot=slot.data_ptr(), ctx=ctx.data_ptr(), mask=mask.data_ptr())
    sb.tree_accept(c.desc, tree, parent.data_ptr(), token.data_ptr(), target.data_ptr(), cnt.data_ptr(), node.data_ptr(), new.data_ptr())
    assert cnt[:3].tolist() == [0, 0, 0] and cnt[-2:].tolist() == [0, 2]
    assert node[-1].tolist() == [0, 1] + [-1] * 62 and new[-1].tolist() == [6, 7] + [-1] * 62
    assert bool((node[:5] == -1).all()) and bool((new[-9:-1] == -1).all())


# ------------------------------------------------------------- scales of any size
def dim0(c, index, k, which=0, slot=0):
    """The key at `index` becomes k in dim 0 and 0 elsewhere (for every head)."""
    raw = c.raw().copy()
    page, t = c.table[slot, index // 16], index % 16
    row = np.zeros(c.hd)
    row[0] = k
    if c.kv == Q8:
        raw[0, page, which, :, 64 + t * c.hd:64 + (t + 1) * c.hd] = np.where(np.arange(c.hd) == 0, 100, 0).astype(np.int8).view(np.uint8)
        raw[0, page, which, :, 4 * t:4 * t + 4] = np.array([k / 100], np.float32).view(np.uint8)
    else:
        b = c.hd * (2 if c.kv == F16 else 4)
        raw[0, page, which, :, t * b:(t + 1) * b] = row.astype(NP[c.kv]).view(np.uint8)
    c.pool.copy_(torch.from_numpy(raw.reshape(-1)))


@pytest.mark.parametrize("nodes,nq,nkv,hd", ROWS)
@pytest.mark.parametrize("size", [1e3, 1e6, 1e12, 1e30])
@pytest.mark.parametrize("ctx", [40, 700])
def test_a_large_v_scale_that_a_row_does_not_see(sb, ctx, size, nodes, nq, nkv, hd):
    """8 bits: a finite scale of a masked node, of any size, takes nothing from the other rows; the row
    that sees it gets its own sum right."""
    rng = np.random.default_rng(nodes + ctx)
    c = Cache(sb, Q8, 1, nkv, hd, [ctx + nodes], seed=3)
    bad = nodes // 2
    masks = sb.tree_masks(random_tree(rng, nodes))
    masks[np.arange(nodes) != bad] &= ~np.uint64(1 << bad)
    q = rng.normal(0, 1, (nodes, nq, hd)).astype(np.float32)
    set_rows(c, 1, ctx + bad, size)
    got = attend(sb, c, 0, [nodes], [ctx], masks, q, hd ** -0.5)
    want, n = plain(c, 0, [nodes], [ctx], masks, q, hd ** -0.5)
    others = np.arange(nodes) != bad
    check(got[others], want[others], n)
    check(got[bad], want[bad], n)


@pytest.mark.parametrize("nodes,nq,nkv,hd", ROWS)
@pytest.mark.parametrize("size,score", [(1e6, -60.0), (1e12, -80.0), (1e30, -150.0), (1e30, -95.0)])
@pytest.mark.parametrize("at", [0, 77, 390])
def test_a_large_v_scale_of_little_weight(sb, at, size, score, nodes, nq, nkv, hd):
    """8 bits: a token of the context with a large scale and a weight so small that it does not count
    leaves the others' sum as exact as ever, wherever it lies."""
    rng = np.random.default_rng(nodes + at)
    ctx = 391
    c = Cache(sb, Q8, 1, nkv, hd, [ctx + nodes], seed=3)
    masks = sb.tree_masks(random_tree(rng, nodes))
    q = (rng.normal(0, 1, (nodes, nq, hd)) * hd ** -0.5).astype(np.float32)
    q[..., 0] = 1.0
    dim0(c, at, score)
    set_rows(c, 1, at, size)
    got = attend(sb, c, 0, [nodes], [ctx], masks, q, 1.0)
    check(got, *plain(c, 0, [nodes], [ctx], masks, q, 1.0))


@pytest.mark.parametrize("nodes,nq,nkv,hd", ROWS)
@pytest.mark.parametrize("slope", [0.05, -0.05, 0.012, -0.012])
@pytest.mark.parametrize("level", [False, True])
def test_v_scales_that_grow_along_the_context(sb, level, slope, nodes, nq, nkv, hd):
    """8 bits: scales of 2^(slope i); `level`: with scores that fall as they rise, so that every token's
    part of the sum is alike."""
    rng = np.random.default_rng(nodes)
    ctx = 1100
    c = Cache(sb, Q8, 1, nkv, hd, [ctx + nodes], seed=7)
    e, s = c.parts()
    for i in range(ctx + nodes):
        page, t = c.table[0, i // 16], i % 16
        up = slope * (i if slope > 0 else i - ctx)          # from 2^0 up, or down to 2^0
        s[0, page, 1, :, t] *= np.float32(2.0 ** up)
        if level:
            e[0, page, 0, :, t, 0] = -100
            s[0, page, 0, :, t] = np.float32(up * np.log(2.0) / 100 + 1e-3)
    raw = c.raw().copy()
    raw[..., 64:], raw[..., :64] = e.view(np.uint8).reshape(raw[..., 64:].shape), s.view(np.uint8)
    c.pool.copy_(torch.from_numpy(raw.reshape(-1)))
    masks = sb.tree_masks(random_tree(rng, nodes))
    q = (rng.normal(0, 1, (nodes, nq, hd)) * (0.001 if level else hd ** -0.5)).astype(np.float32)
    q[..., 0] = 1.0 if level else q[..., 0]
    check(attend(sb, c, 0, [nodes], [ctx], masks, q, 1.0), *plain(c, 0, [nodes], [ctx], masks, q, 1.0))
