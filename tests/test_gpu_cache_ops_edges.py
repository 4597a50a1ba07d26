"""The cache operators at their edges: values that are no numbers, scales and queries of very
different size, masks and nodes beyond what a step names, graphs and streams."""
import numpy as np
import pytest
import torch

from test_gpu_cache_ops import F16, F32, NP, Q8, Cache, attend, check, dev, f32_rotate, plain, random_tree

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


@pytest.mark.parametrize("nodes,nq,nkv,hd", [(1, 4, 1, 128), (4, 4, 1, 64), (8, 4, 1, 64), (5, 4, 1, 128), (16, 4, 1, 128), (11, 4, 1, 64), (30, 4, 1, 64)])
def test_v_scales_of_many_sequences(sb, nodes, nq, nkv, hd):
    """8 bits: sequences of even scales beside others whose scales spread over 2^20, more of them than workers: what
    one leaves in a worker does not reach the next."""
    rng = np.random.default_rng(nodes)
    n = 170
    counts = [nodes - s % 2 * (nodes // 2) for s in range(n)]
    ctx = [int(x) for x in rng.integers(100, 420, n)]
    c = Cache(sb, Q8, 1, nkv, hd, [x + k for x, k in zip(ctx, counts)], seed=8)
    e, s = c.parts()
    for i in range(0, n, 3):
        for page in c.table[i, :-(-(ctx[i] + counts[i]) // 16)]:
            s[0, page, 1] *= np.exp2(rng.uniform(0, 20, 16)).astype(np.float32)
    raw = c.raw().copy()
    raw[..., :64] = s.view(np.uint8)
    c.pool.copy_(torch.from_numpy(raw.reshape(-1)))
    masks = np.concatenate([sb.tree_masks(random_tree(rng, k)) for k in counts])
    q = rng.normal(0, 1, (sum(counts), nq, hd)).astype(np.float32)
    got = attend(sb, c, 0, counts, ctx, masks, q, hd ** -0.5)
    want, size = plain(c, 0, counts, ctx, masks, q, hd ** -0.5)
    at = np.repeat(np.arange(n) % 3 == 0, counts)                # apart: their outputs differ in size
    check(got[at], want[at], size)
    check(got[~at], want[~at], size)


# ------------------------------------------------------------- infinities that a row sees
def formula(c, nodes, ctx, masks, q, scale):
    """The formula in f64 with infinities and NaN: a key of score -inf is as if not seen; one of +inf or NaN
    makes the row NaN; an infinity or NaN in v of a key that is seen makes that dim it (NaN: where signs differ)."""
    out, r = np.zeros(q.shape), 0
    values = c.values()
    with np.errstate(all="ignore"):
        for s, n in enumerate(nodes):
            K, V = c.rows(0, s, ctx[s] + n, values)
            for i in range(n):
                see = np.r_[np.arange(ctx[s]), ctx[s] + np.array([j for j in range(n) if int(masks[r]) >> j & 1], int)].astype(int)
                for h in range(q.shape[1]):
                    k, v = K[see, h // (q.shape[1] // c.nkv)], V[see, h // (q.shape[1] // c.nkv)]
                    z = (k * q[r, h].astype(np.float64)).sum(-1) * scale
                    v, z = v[z != -np.inf], z[z != -np.inf]
                    if not len(z):
                        continue
                    p = np.exp(z - z.max())
                    fin = np.isfinite(v)
                    out[r, h] = (p @ np.where(fin, v, 0)) / p.sum() + np.where(fin, 0, v).sum(0)
                r += 1
    return out


def check_values(got, want, size):
    """The same infinities and NaN, and the numbers beside them within the usual bound."""
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isposinf(got), np.isposinf(want)) and np.array_equal(np.isneginf(got), np.isneginf(want))
    fin = np.isfinite(want)
    check(np.where(fin, got, 0), np.where(fin, want, 0), size)


def edge_case(sb, kv, nodes, nq, nkv, hd, ctx=150):
    rng = np.random.default_rng(nodes + hd)
    c = Cache(sb, kv, 1, nkv, hd, [ctx + nodes], seed=3)
    masks = sb.tree_masks(random_tree(rng, nodes))
    q = (rng.normal(0, 1, (nodes, nq, hd)) * hd ** -0.5).astype(np.float32)
    q[..., 0] = 1.0
    size = plain(c, 0, [nodes], [ctx], masks, q, 1.0)[1]
    return c, masks, q, size


@pytest.mark.parametrize("kv", [F32, F16])
@pytest.mark.parametrize("nodes,nq,nkv,hd", ROWS)
@pytest.mark.parametrize("at", [3, 149, 152])
def test_a_key_of_score_minus_infinity_weighs_nothing(sb, at, nodes, nq, nkv, hd, kv):
    """In the context and among the nodes; its v, an infinity too, does not count either."""
    c, masks, q, size = edge_case(sb, kv, nodes, nq, nkv, hd)
    for inf_v in (False, True):
        set_rows(c, 0, at, np.where(np.arange(hd) == 0, -np.inf, 1.0))
        if inf_v:
            set_rows(c, 1, at, -np.inf)
        want = formula(c, [nodes], [150], masks, q, 1.0)
        assert np.isfinite(want).all()
        check_values(attend(sb, c, 0, [nodes], [150], masks, q, 1.0), want, size)


@pytest.mark.parametrize("kv", [F32, F16])
@pytest.mark.parametrize("nodes,nq,nkv,hd", ROWS)
def test_infinite_v_that_rows_see(sb, nodes, nq, nkv, hd, kv):
    """Dims of v that are infinite in the context, in one node, in tokens of opposite signs, in tokens whose weight
    is too small for f32: each shows where the row sees it, the other dims keep their sums."""
    c, masks, q, size = edge_case(sb, kv, nodes, nq, nkv, hd)
    v = np.full(hd, 0.5)
    v[3], v[5], v[7] = np.inf, -np.inf, np.nan
    set_rows(c, 1, 20, v)
    w = np.full(hd, -0.25)
    w[5], w[9], w[11] = np.inf, np.inf, -np.inf
    set_rows(c, 1, 140, w)
    u = np.full(hd, 0.125)
    u[13], u[9] = -np.inf, np.inf
    set_rows(c, 1, 152, u)                              # a node
    dim0(c, 100, -300.0)                                # weights that f32 does not hold, in the context ...
    set_rows(c, 1, 100, np.where(np.arange(hd) == 15, np.inf, 1.0))
    dim0(c, 153, -300.0)                                # ... and in a node
    set_rows(c, 1, 153, np.where(np.arange(hd) == 2, -np.inf, 1.0))
    check_values(attend(sb, c, 0, [nodes], [150], masks, q, 1.0), formula(c, [nodes], [150], masks, q, 1.0), 2 * size)


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("nodes,nq,nkv,hd", ROWS)
@pytest.mark.parametrize("x", [np.inf, np.nan])
def test_scores_that_are_no_numbers(sb, x, nodes, nq, nkv, hd, kv):
    """A score of +inf or NaN makes the rows that see it NaN and no others."""
    c, masks, q, size = edge_case(sb, kv, nodes, nq, nkv, hd)
    set_rows(c, 0, 152, x if kv == Q8 else np.where(np.arange(hd) == 0, x, 1.0))
    want = formula(c, [nodes], [150], masks, q, 1.0)
    sees = masks >> np.uint64(2) & np.uint64(1) > 0
    if kv == Q8:                                        # an infinite scale: infinities of both signs
        want[sees] = np.nan
    assert np.isnan(want[sees]).all() and np.isfinite(want[~sees]).all()
    check_values(attend(sb, c, 0, [nodes], [150], masks, q, 1.0), want, size)


@pytest.mark.parametrize("nodes,nq,nkv,hd", ROWS)
@pytest.mark.parametrize("x", [np.inf, np.nan])
@pytest.mark.parametrize("score", [0.0, -300.0])
def test_8_bit_v_that_is_no_number(sb, score, x, nodes, nq, nkv, hd):
    """A v row that the append wrote from an infinity or NaN (such a scale, integers of 0) makes the rows that see it
    NaN, whatever their weight."""
    c, masks, q, size = edge_case(sb, Q8, nodes, nq, nkv, hd)
    dim0(c, 152, score)
    dim0(c, 152, 1.0, which=1)
    e, s = c.parts()
    e[0, c.table[0, 9], 1, :, 8] = 0
    raw = c.raw().copy()
    raw[..., 64:] = e.view(np.uint8).reshape(raw[..., 64:].shape)
    c.pool.copy_(torch.from_numpy(raw.reshape(-1)))
    set_rows(c, 1, 152, x)
    want = formula(c, [nodes], [150], masks, q, 1.0)
    check_values(attend(sb, c, 0, [nodes], [150], masks, q, 1.0), want, size)


# ------------------------------------------------------------- queries
@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("nodes,nq,nkv,hd", ROWS)
@pytest.mark.parametrize("e", [-120, -104, 101, 112, 120])
def test_queries_of_any_exponent(sb, e, nodes, nq, nkv, hd, kv):
    c, masks, q, size = edge_case(sb, kv, nodes, nq, nkv, hd)
    s = 0.1 * 2.0 ** -e
    check(attend(sb, c, 0, [nodes], [150], masks, (q * np.float32(2.0 ** e)).astype(np.float32), s),
          plain(c, 0, [nodes], [150], masks, q, 0.1)[0], size)


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("nodes,nq,nkv,hd", ROWS)
@pytest.mark.parametrize("outlier", [1e3, 2e4])
def test_queries_with_one_large_dim(sb, outlier, nodes, nq, nkv, hd, kv):
    """A dim that is `outlier` times the others and meets keys of 0 there: the others' products keep f32's exactness."""
    rng = np.random.default_rng(nodes)
    ctx = 600
    c = Cache(sb, kv, 1, nkv, hd, [ctx + nodes], seed=3)
    e, s = c.parts()
    e[:, :, 0, :, :, 5] = 0
    raw = c.raw().copy()
    if kv == Q8:
        raw[..., 64:] = e.view(np.uint8).reshape(raw[..., 64:].shape)
    else:
        raw = np.ascontiguousarray(e).view(np.uint8).reshape(raw.shape)
    c.pool.copy_(torch.from_numpy(raw.reshape(-1)))
    masks = sb.tree_masks(random_tree(rng, nodes))
    q = rng.normal(0, 1, (nodes, nq, hd)).astype(np.float32)
    q[..., 5] = outlier
    check(attend(sb, c, 0, [nodes], [ctx], masks, q, hd ** -0.5), *plain(c, 0, [nodes], [ctx], masks, q, hd ** -0.5))


# ------------------------------------------------------------- nodes and masks beyond what a step names
@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("hd,nq", [(64, 2), (128, 16), (64, 32), (24, 4)])
def test_rows_of_nodes_beyond_max_nodes_stay_as_they_are(sb, hd, nq, kv):
    rng = np.random.default_rng(1)
    c = Cache(sb, kv, 1, 2, hd, [60, 60], seed=1)
    masks = np.concatenate([sb.tree_masks(random_tree(rng, n)) for n in (9, 1)])
    q = rng.normal(0, 1, (10, nq, hd)).astype(np.float32)
    got = attend(sb, c, 0, [9, 1], [40, 50], masks, q, 0.1, max_nodes=5)
    assert (got[5:9] == 9).all() and (got[:5] != 9).all() and (got[9] != 9).all()


def accept(sb, c, nodes, ctx, masks, parents, tokens, targets, max_nodes):
    off = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    keep = [dev(off), dev(np.arange(len(nodes), dtype=np.int32)), dev(np.array(ctx, np.int32)), dev(np.asarray(masks, np.uint64).view(np.int64)),
            *(dev(np.asarray(x, np.int32)) for x in (parents, tokens, targets))]
    tree = sb.TreeBatch(n_seq=len(nodes), rows=int(off[-1]), max_nodes=max_nodes, row_off=keep[0].data_ptr(), slot=keep[1].data_ptr(),
                        ctx=keep[2].data_ptr(), mask=keep[3].data_ptr())
    cnt = torch.full((len(nodes),), -7, dtype=torch.int32, device="cuda")
    node, tok = (torch.full((len(nodes), 64), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    sb.tree_accept(c.desc, tree, *(k.data_ptr() for k in keep[4:]), cnt.data_ptr(), node.data_ptr(), tok.data_ptr())
    return cnt.tolist(), node.cpu().numpy(), tok.cpu().numpy()


def test_accept_leaves_out_nodes_beyond_max_nodes(sb):
    """A chain of seven nodes that all match, of which the step names four (one more sequence keeps
    rows within n_seq * max_nodes)."""
    c = Cache(sb, F16, 2, 1, 64, [40, 40])
    parents = np.arange(7) - 1
    cnt, node, tok = accept(sb, c, [7, 1], [20, 30], np.r_[sb.tree_masks(parents), [np.uint64(1)]], np.r_[parents, -1], np.r_[np.arange(7), 3],
                            np.r_[np.arange(1, 8), 4], 4)
    assert cnt == [4, 1] and node[0, :5].tolist() == [0, 1, 2, 3, -1] and tok[0, :5].tolist() == [1, 2, 3, 4, -1]


def test_accept_of_a_node_whose_mask_does_not_name_it(sb):
    """The node itself has to match too, whether or not its mask has its own bit."""
    c = Cache(sb, F16, 1, 1, 64, [40])
    masks = np.array([0b1, 0b11, 0b011, 0b011], np.uint64)               # nodes 2 and 3: their ancestors alone
    parents, targets = [-1, 0, 1, 1], [5, 6, 7, 8]
    cnt, node, _ = accept(sb, c, [4], [20], masks, parents, [1, 9, 6, 4], targets, 4)      # node 1 fails: the root alone
    assert cnt == [1] and node[0, 0] == 0
    cnt, node, _ = accept(sb, c, [4], [20], np.array([0b1, 0b10, 0b1, 0b1], np.uint64), [-1, 0, 0, 0], [1, 9, 4, 3], targets, 4)
    assert cnt == [1] and node[0, 0] == 0
    masks = np.array([0b1, 0b11, 0b1011, 0b0011], np.uint64)             # the deepest by its mask does not match itself
    cnt, node, _ = accept(sb, c, [4], [20], masks, [-1, 0, 1, 1], [1, 5, 4, 6], targets, 4)
    assert cnt == [2] and node[0, :2].tolist() == [0, 1]


# ------------------------------------------------------------- buffers, graphs, streams
@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("hd,rot,layout,odd", [(64, 64, 0, 1), (128, 64, 1, 1), (256, 256, 0, 0), (20, 14, 1, 3), (128, 128, 0, 0)])
def test_rope_append_in_place(sb, hd, rot, layout, odd, kv):
    """q_out = q, a part of the row that k and v come from, on strides that vectors take and on others."""
    nq, nkv, rows = 6, 2, 37
    c = Cache(sb, kv, 1, nkv, hd, [rows], seed=3, fill=False)
    rng = np.random.default_rng(hd)
    ld = (nq + 2 * nkv) * hd + odd
    x = rng.normal(0, 1, (rows, ld)).astype(np.float32)
    cos, sin = sb.rope_tables(500, rot, 1e4)
    pos = rng.integers(0, 500, rows).astype(np.int32)
    d, dc, ds, dp, i = dev(x), dev(cos), dev(sin), dev(pos), dev(np.arange(rows, dtype=np.int32))
    z = torch.zeros(rows, dtype=torch.int32, device="cuda")
    rope = sb.Rope(cos=dc.data_ptr(), sin=ds.data_ptr(), n_pos=500, rot_dim=rot, layout=layout)
    p = d.data_ptr()
    sb.rope_append(c.desc, 0, rope, rows, nq, p, ld, p, ld, p + 4 * nq * hd, ld, p + 4 * (nq + nkv) * hd, ld, z.data_ptr(), i.data_ptr(),
                   dp.data_ptr())
    want = x.copy()
    want[:, :nq * hd] = f32_rotate(x[:, :nq * hd].reshape(rows, nq, hd), cos[pos], sin[pos], rot, layout).reshape(rows, -1)
    assert np.array_equal(d.cpu().numpy(), want)


class Step:
    """A layer's calls over device buffers that a graph can hold: append the nodes, attend, accept, read back."""

    def __init__(self, sb, kv, hd, nq, nodes, ctx, seed):
        rng = np.random.default_rng(seed)
        self.sb, self.nq, self.hd, self.nkv = sb, nq, hd, 2
        self.rows = sum(nodes)
        self.c = Cache(sb, kv, 1, 2, hd, [x + n + 40 for x, n in zip(ctx, nodes)], seed=seed)
        parents = [random_tree(rng, n) for n in nodes]
        cos, sin = sb.rope_tables(3000, hd, 1e4)
        i32 = lambda a: dev(np.asarray(a, np.int32))  # noqa: E731
        self.off, self.slot, self.ctx = i32(np.concatenate([[0], np.cumsum(nodes)])), i32(np.arange(len(nodes))), i32(ctx)
        self.mask = dev(np.concatenate([sb.tree_masks(p) for p in parents]).view(np.int64))
        self.parent, self.token, self.target = i32(np.concatenate(parents)), i32(rng.integers(0, 3, self.rows)), i32(rng.integers(0, 3, self.rows))
        self.row_slot = i32(np.repeat(np.arange(len(nodes)), nodes))
        self.index = i32(np.concatenate([x + np.arange(n) for x, n in zip(ctx, nodes)]))
        self.cos, self.sin = dev(cos), dev(sin)
        self.qkv = dev(rng.normal(0, 1, (self.rows, (nq + 4) * hd)).astype(np.float32))
        self.q, self.out = (torch.zeros(self.rows, nq * hd, device="cuda") for _ in range(2))
        self.K, self.V = (torch.zeros(self.rows, 2 * hd, device="cuda") for _ in range(2))
        self.cnt = torch.zeros(len(nodes), dtype=torch.int32, device="cuda")
        self.node, self.new = (torch.zeros(len(nodes), 64, dtype=torch.int32, device="cuda") for _ in range(2))
        self.rope = sb.Rope(cos=self.cos.data_ptr(), sin=self.sin.data_ptr(), n_pos=3000, rot_dim=hd, layout=0)
        self.tree = sb.TreeBatch(n_seq=len(nodes), rows=self.rows, max_nodes=max(nodes), row_off=self.off.data_ptr(), slot=self.slot.data_ptr(),
                                 ctx=self.ctx.data_ptr(), mask=self.mask.data_ptr())
        self.ws = torch.empty(sb.attention_tree_workspace(self.c.desc, nq, len(nodes), self.rows, max(nodes)), dtype=torch.uint8, device="cuda")
        self.pool0 = self.c.pool.clone()
        torch.cuda.synchronize()

    def reset(self):
        self.c.pool.copy_(self.pool0)
        for x in (self.q, self.out, self.K, self.V, self.cnt, self.node, self.new):
            x.zero_()

    def run(self, stream):
        sb, p, ld, nq, hd = self.sb, self.qkv.data_ptr(), (self.nq + 4) * self.hd, self.nq, self.hd
        sb.rope_append(self.c.desc, 0, self.rope, self.rows, nq, self.q.data_ptr(), nq * hd, p, ld, p + 4 * nq * hd, ld, p + 4 * (nq + 2) * hd,
                       ld, self.row_slot.data_ptr(), self.index.data_ptr(), self.index.data_ptr(), stream)
        sb.attention_tree(self.c.desc, 0, self.tree, nq, self.out.data_ptr(), nq * hd, self.q.data_ptr(), nq * hd, hd ** -0.5,
                          self.ws.data_ptr(), self.ws.numel(), stream)
        sb.tree_accept(self.c.desc, self.tree, self.parent.data_ptr(), self.token.data_ptr(), self.target.data_ptr(), self.cnt.data_ptr(),
                       self.node.data_ptr(), self.new.data_ptr(), stream)
        sb.kv_read(self.c.desc, 0, 1, self.rows, self.row_slot.data_ptr(), self.index.data_ptr(), self.K.data_ptr(), self.V.data_ptr(), F32,
                   stream)

    def results(self):
        torch.cuda.synchronize()
        return [x.cpu().numpy() for x in (self.q, self.out, self.K, self.V, self.cnt, self.node, self.new, self.c.pool)]


def same(a, b):
    return all(np.array_equal(x, y) for x, y in zip(a, b))


STEPS = [(64, 4, [1, 1, 1], [700, 3, 90]), (128, 8, [5, 2], [333, 0]), (64, 8, [16, 9], [1200, 31]), (128, 16, [40, 13], [260, 1001]),
         (80, 4, [6], [100])]


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("hd,nq,nodes,ctx", STEPS)
def test_a_captured_step(sb, hd, nq, nodes, ctx, kv):
    """A graph of all four operators gives what the calls give, and reads lengths, places, masks and
    inputs anew at every replay."""
    s = Step(sb, kv, hd, nq, nodes, ctx, 5)
    s.run(torch.cuda.current_stream().cuda_stream)
    first = s.results()
    s.reset()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        s.run(torch.cuda.current_stream().cuda_stream)
    s.reset()
    graph.replay()
    assert same(first, s.results())
    # longer contexts, other masks and values, in the same buffers
    s.ctx += 17
    s.index += 17
    s.qkv.mul_(-0.5)
    s.token.copy_(s.token.flip(0))
    s.mask.copy_(s.mask & -2 | 1)
    s.reset()
    s.run(torch.cuda.current_stream().cuda_stream)
    second = s.results()
    assert not same(first, second)
    s.reset()
    graph.replay()
    assert same(second, s.results())
    del graph


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("hd,nq,nodes,ctx", STEPS[:4])
def test_steps_on_two_streams(sb, hd, nq, nodes, ctx, kv):
    """Two sequences of calls at the same time, with a cache and a workspace each, give the bits of either alone."""
    steps = [Step(sb, kv, hd, nq, nodes, ctx, 5), Step(sb, kv, hd, nq, nodes[::-1], ctx[::-1], 6)]
    alone = []
    for s in steps:
        s.run(torch.cuda.current_stream().cuda_stream)
        alone.append(s.results())
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(8):
        for s in steps:
            s.reset()
        torch.cuda.synchronize()
        for s, st in zip(steps, streams):
            s.run(st.cuda_stream)
        for s, a in zip(steps, alone):
            assert same(a, s.results())
