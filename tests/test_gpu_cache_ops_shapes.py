"""The cache operators where their kernels change form: rows on 16 bytes (vector
kernels), outputs that are not, many sequences, maxima that grow, long contexts."""
import numpy as np
import pytest
import torch

import test_gpu_cache_ops as ops
from test_gpu_cache_ops import F16, F32, NP, Q8, Cache, attend, check, dev, f32_quant, f32_rotate, plain, random_tree

pytestmark = pytest.mark.gpu


# rows, nq, nkv, hd, rot, layout: every lane count (head_dim to 32, 64, 128), both numbers of
# heads a warp holds, heads that do not fill the last warp, head_dims that do not fill their lanes
VECTORS = [(1, 1, 1, 4, 0, 0), (1, 32, 8, 128, 128, 0), (16, 32, 8, 128, 64, 1), (33, 5, 3, 128, 128, 1), (5, 8, 2, 64, 64, 0),
           (7, 9, 3, 64, 32, 1), (6, 6, 2, 32, 32, 0), (3, 7, 1, 32, 8, 1), (9, 2, 2, 96, 48, 0), (4, 3, 1, 20, 16, 1),
           (11, 4, 2, 112, 112, 0), (2, 5, 5, 80, 80, 1), (700, 32, 8, 128, 128, 0), (900, 16, 8, 64, 64, 1), (1500, 32, 16, 32, 16, 0)]


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("rows,nq,nkv,hd,rot,layout", VECTORS)
def test_rope_append_rows_on_16_bytes(sb, rows, nq, nkv, hd, rot, layout, kv):
    """Bit for bit the f32 formula, on aligned strides; half of the values lie on or beside a
    boundary between two 8-bit integers."""
    rot = rot or 2                                    # (rot 2 takes the scalar kernel)
    rng = np.random.default_rng(rows + hd + rot)
    x = rng.normal(0, 2, (rows, nq + 2 * nkv, hd)).astype(np.float32)
    ties = rng.integers(-126, 127, x.shape) + np.float32(0.5)
    ties = (ties * np.exp2(rng.integers(-3, 4, x.shape[:2] + (1,)))).astype(np.float32)
    ties[..., 0] = np.abs(ties).max(-1) * np.float32(127) / np.float32(126.5)
    x[::2] = np.nextafter(ties, np.where(rng.random(x.shape) < 0.5, ties, np.inf).astype(np.float32))[::2]
    c = Cache(sb, kv, 2, nkv, hd, [rows + 3], seed=rows, fill=False)
    before = c.raw().copy()
    index = rng.permutation(rows + 3)[:rows].astype(np.int32)
    pos = rng.integers(0, 300, rows).astype(np.int32)
    pos[::2] = 0                                      # position 0 turns nothing: the ties stay ties
    cos, sin = sb.rope_tables(300, rot, 1e4)
    ld = (nq + 2 * nkv) * hd + 8
    xp = np.zeros((rows, ld), np.float32)
    xp[:, :ld - 8] = x.reshape(rows, -1)
    d, dc, ds, di, dp = dev(xp), dev(cos), dev(sin), dev(index), dev(pos)
    z = torch.zeros(rows, dtype=torch.int32, device="cuda")
    rope = sb.Rope(cos=dc.data_ptr(), sin=ds.data_ptr(), n_pos=300, rot_dim=rot, layout=layout)
    out = torch.full((rows, nq * hd + 4), 7.0, device="cuda")
    p = d.data_ptr()
    sb.rope_append(c.desc, 1, rope, rows, nq, out.data_ptr(), nq * hd + 4, p, ld, p + 4 * nq * hd, ld, p + 4 * (nq + nkv) * hd, ld,
                   z.data_ptr(), di.data_ptr(), dp.data_ptr())
    turned = f32_rotate(x[:, :nq + nkv], cos[pos], sin[pos], rot, layout)
    got = out.cpu().numpy()
    assert np.array_equal(got[:, :-4].reshape(rows, nq, hd), turned[:, :nq]) and (got[:, -4:] == 7).all()
    e, s = c.parts(before)
    page = c.table[0, index // 16]
    for w, y in ((0, turned[:, nq:]), (1, x[:, nq + nkv:])):
        if kv == Q8:
            e[1, page, w, :, index % 16], s[1, page, w, :, index % 16] = f32_quant(y)
        else:
            e[1, page, w, :, index % 16] = y.astype(NP[kv])
    ge, gs = c.parts()
    assert np.array_equal(ge, e) and (kv != Q8 or np.array_equal(gs, s))
    assert np.array_equal(d.cpu().numpy(), xp)


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("out", [F32, F16])
@pytest.mark.parametrize("rows,nkv,hd", [(1, 1, 4), (17, 2, 64), (40, 3, 128), (9, 2, 20)])
def test_read_into_any_alignment(sb, rows, nkv, hd, out, kv):
    """K and V that start one element off a 16-byte boundary, and nothing beside them is written."""
    c = Cache(sb, kv, 2, nkv, hd, [rows])
    i = np.random.default_rng(rows).permutation(rows).astype(np.int32)
    z, di = torch.zeros(rows, dtype=torch.int32, device="cuda"), dev(i)
    n = 2 * rows * nkv * hd
    K, V = (torch.full((n + 2,), 3.0, dtype=torch.float32 if out == F32 else torch.float16, device="cuda") for _ in range(2))
    sz = K.element_size()
    sb.kv_read(c.desc, 0, 2, rows, z.data_ptr(), di.data_ptr(), K.data_ptr() + sz, V.data_ptr() + sz, out)
    e, s = c.parts()
    full = e.astype(np.float32) * (np.float32(1) if s is None else s[..., None])
    for w, g in ((0, K), (1, V)):
        g = g.cpu().numpy()
        want = np.moveaxis(full[:, c.table[0, i // 16], w][:, np.arange(rows), :, i % 16], 0, 1)
        assert np.array_equal(g[1:-1].reshape(want.shape), want.astype(g.dtype)) and g[0] == 3 and g[-1] == 3


# sequences, nodes at most, nq, nkv, hd: the plan of up to 32, up to 128 and more sequences, with
# each of the kernels for few and for many rows
MANY = [(33, 2, 8, 2, 64), (130, 1, 4, 4, 128), (300, 1, 2, 2, 64), (33, 3, 8, 2, 128), (150, 3, 8, 2, 64), (40, 8, 16, 4, 128),
        (150, 7, 16, 2, 64), (1000, 1, 1, 1, 64)]


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("n,most,nq,nkv,hd", MANY)
def test_attention_tree_many_sequences(sb, n, most, nq, nkv, hd, kv):
    rng = np.random.default_rng(n + hd)
    nodes = [int(x) for x in rng.integers(0, most + 1, n)]          # many are empty
    nodes[:2], nodes[-1] = [0, 0], most
    ctx = [int(x) for x in rng.integers(0, 60, n)]
    ctx[n // 2] = 700
    c = Cache(sb, kv, 1, nkv, hd, [x + k for x, k in zip(ctx, nodes)], seed=n)
    masks = np.concatenate([sb.tree_masks(random_tree(rng, k)) for k in nodes])
    q = rng.normal(0, 1, (sum(nodes), nq, hd)).astype(np.float32)
    check(attend(sb, c, 0, nodes, ctx, masks, q, hd ** -0.5, max_nodes=most), *plain(c, 0, nodes, ctx, masks, q, hd ** -0.5))


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("nodes,nq,nkv,hd", [(1, 4, 1, 128), (3, 4, 1, 64), (8, 4, 1, 64), (20, 8, 1, 128), (40, 8, 1, 64)])
@pytest.mark.parametrize("step", [0.5, 40.0, -40.0])
def test_attention_tree_maxima_that_grow(sb, nodes, nq, nkv, hd, step, kv):
    """Scores that rise (or fall) by `step` every 16 tokens: the running maximum moves within a
    tile, at every tile and seldom, and what was summed before is scaled down to nothing."""
    rng = np.random.default_rng(nodes)
    ctx = 1400
    c = Cache(sb, kv, 1, nkv, hd, [ctx + nodes], seed=7)
    e, s = c.parts()
    for i, page in enumerate(c.table[0, :-(-(ctx + nodes) // 16)]):
        if kv == Q8:
            e[0, page, 0, :, :, 0] = 100
            s[0, page, 0] = np.float32(i / 100)
        else:
            e[0, page, 0, :, :, 0] = i
    raw = c.raw().copy()
    if kv == Q8:
        raw[..., 64:], raw[..., :64] = e.view(np.uint8).reshape(raw[..., 64:].shape), s.view(np.uint8)
    else:
        raw = e.view(np.uint8).reshape(raw.shape)
    c.pool.copy_(torch.from_numpy(np.ascontiguousarray(raw).reshape(-1)))
    masks = sb.tree_masks(random_tree(rng, nodes))
    q = (rng.normal(0, 1, (nodes, nq, hd)) * (0.01 if kv == Q8 else 1)).astype(np.float32)
    q[..., 0] = step
    check(attend(sb, c, 0, [nodes], [ctx], masks, q, 1.0), *plain(c, 0, [nodes], [ctx], masks, q, 1.0))


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("nodes,ctx,nq,nkv,hd", [([64], [30011], 4, 1, 64), ([50, 3], [12001, 20000], 4, 1, 128),
                                                 ([7, 7], [30000, 9], 8, 4, 64), ([1], [40003], 4, 1, 128)])
def test_attention_tree_long_contexts(sb, nodes, ctx, nq, nkv, hd, kv):
    """Items that many workers share, over several row tiles."""
    rng = np.random.default_rng(sum(ctx))
    c = Cache(sb, kv, 1, nkv, hd, [x + n for x, n in zip(ctx, nodes)], seed=9)
    masks = np.concatenate([sb.tree_masks(random_tree(rng, n)) for n in nodes])
    q = rng.normal(0, 1, (sum(nodes), nq, hd)).astype(np.float32)
    check(attend(sb, c, 0, nodes, ctx, masks, q, hd ** -0.5), *plain(c, 0, nodes, ctx, masks, q, hd ** -0.5))


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("hd,nodes", [(64, 8), (64, 16), (64, 20), (64, 32), (128, 9), (128, 16), (128, 32), (64, 64), (128, 64)])
def test_attention_tree_ignores_what_it_does_not_see_at_every_row_count(sb, hd, nodes, kv):
    """16 to 128 rows a kv head: each kernel and its limits."""
    ops.test_attention_tree_ignores_what_it_does_not_see(sb, kv=kv, hd=hd, nodes=nodes)


@pytest.mark.parametrize("kv", [F16, Q8])
@pytest.mark.parametrize("nodes,nq,nkv,hd", [(10, 8, 2, 128), (16, 8, 2, 64), (13, 4, 1, 64), (20, 8, 2, 128)])
@pytest.mark.parametrize("q_size,v_size,scale", [(1e5, 1.0, 1e-6), (1e-5, 1.0, 1e4), (30.0, 1.0, 0.2), (1.0, 1e-3, 0.1), (1.0, 200.0, 0.1)])
def test_attention_tree_sizes_of_values_with_many_rows(sb, nodes, nq, nkv, hd, q_size, v_size, scale, kv):
    rng = np.random.default_rng(nodes)
    ctx = 500
    c = Cache(sb, kv, 1, nkv, hd, [ctx + nodes], seed=4)
    raw = c.raw().copy()
    if kv == Q8:
        raw[:, :, 1, :, :64] = (raw[:, :, 1, :, :64].copy().view(np.float32) * np.float32(v_size)).view(np.uint8)
    else:
        raw[:, :, 1] = (raw[:, :, 1].copy().view(NP[kv]).astype(np.float32) * np.float32(v_size)).astype(NP[kv]).view(np.uint8)
    c.pool.copy_(torch.from_numpy(raw.reshape(-1)))
    masks = sb.tree_masks(random_tree(rng, nodes))
    q = (rng.normal(0, 1, (nodes, nq, hd)) * q_size).astype(np.float32)
    check(attend(sb, c, 0, [nodes], [ctx], masks, q, scale), *plain(c, 0, [nodes], [ctx], masks, q, scale))


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("nodes,nq,hd", [(10, 4, 128), (16, 4, 64), (9, 4, 64)])
@pytest.mark.parametrize("step", [0.5, 40.0, -40.0])
def test_attention_tree_maxima_that_grow_on_two_lanes(sb, nodes, nq, hd, step, kv):
    test_attention_tree_maxima_that_grow(sb, nodes, nq, 1, hd, step, kv)


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("nodes,ctx,nq,nkv,hd", [([16], [20011], 4, 1, 64), ([13, 3, 16], [9001, 0, 127], 4, 1, 128), ([12], [1], 8, 2, 128),
                                                 ([11], [0], 8, 2, 64), ([16, 16], [128, 63], 4, 1, 64)])
def test_attention_tree_up_to_64_rows(sb, nodes, ctx, nq, nkv, hd, kv):
    rng = np.random.default_rng(sum(ctx))
    c = Cache(sb, kv, 1, nkv, hd, [x + n for x, n in zip(ctx, nodes)], seed=11)
    masks = np.concatenate([sb.tree_masks(random_tree(rng, n)) for n in nodes])
    q = rng.normal(0, 1, (sum(nodes), nq, hd)).astype(np.float32)
    check(attend(sb, c, 0, nodes, ctx, masks, q, hd ** -0.5), *plain(c, 0, nodes, ctx, masks, q, hd ** -0.5))


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("hd,nq", [(64, 2), (128, 16), (24, 4)])
def test_attention_tree_leaves_out_nodes_beyond_max_nodes(sb, hd, nq, kv):
    rng = np.random.default_rng(1)
    c = Cache(sb, kv, 1, 2, hd, [60, 60], seed=1)
    masks = np.concatenate([sb.tree_masks(random_tree(rng, n)) for n in (9, 1)])
    q = rng.normal(0, 1, (10, nq, hd)).astype(np.float32)
    got = attend(sb, c, 0, [9, 1], [40, 50], masks, q, 0.1, max_nodes=5)
    want, size = plain(c, 0, [5, 1], [40, 50], np.r_[masks[:5], masks[9:]], np.concatenate([q[:5], q[9:]]), 0.1)
    check(np.concatenate([got[:5], got[9:]]), want, size)
