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
