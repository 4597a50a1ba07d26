"""The cache operators on the GPU against plain numpy: rotary append, read-back,
tree attention, tree acceptance, over the cache's three element types."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, Q8 = 0, 1, 2
NP = {F32: np.float32, F16: np.float16}


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Cache:
    """A paged cache on the device and what it holds, as f64 rows."""

    def __init__(self, sb, kv, layers, nkv, hd, lengths, seed=0, slack=1, fill=True):
        rng = np.random.default_rng(seed)
        self.sb, self.kv, self.layers, self.nkv, self.hd = sb, kv, layers, nkv, hd
        need = [-(-max(n, 1) // 16) for n in lengths]
        self.n_pages = sum(need) + 2
        perm = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(lengths), max(need) + slack), -1, np.int32)
        at = 0
        for s, k in enumerate(need):
            self.table[s, :k] = perm[at:at + k]
            at += k
        self.block = 64 + 16 * hd if kv == Q8 else 16 * hd * (2 if kv == F16 else 4)
        assert sb.kv_pool_bytes(kv, self.n_pages, layers, nkv, hd) == layers * self.n_pages * 2 * nkv * self.block
        n = layers * self.n_pages * 2 * nkv
        if kv == Q8:
            raw = np.zeros((n, self.block), np.uint8)
            if fill:
                raw[:, :64] = (rng.uniform(0.5, 2.0, (n, 16)).astype(np.float32) / 127).view(np.uint8)
                raw[:, 64:] = rng.integers(-127, 128, (n, 16 * hd)).astype(np.int8).view(np.uint8)
        else:
            raw = (rng.normal(0, 1, (n, 16 * hd)) if fill else np.zeros((n, 16 * hd))).astype(NP[kv]).view(np.uint8)
        self.pool = dev(raw.reshape(-1))
        self.d_table = dev(self.table)
        self.desc = sb.KVCache(pool=self.pool.data_ptr(), page_table=self.d_table.data_ptr(), n_pages=self.n_pages,
                               n_slots=len(lengths), max_pages=self.table.shape[1], n_layers=layers, n_kv_heads=nkv,
                               head_dim=hd, kv_dtype=kv)

    def raw(self):
        torch.cuda.synchronize()
        return self.pool.cpu().numpy().reshape(self.layers, self.n_pages, 2, self.nkv, self.block)

    def parts(self, raw=None):
        """(elements [layers, pages, 2, nkv, 16, hd], scales or None) of the pool."""
        raw = self.raw() if raw is None else raw
        shape = raw.shape[:4] + (16, self.hd)
        if self.kv == Q8:
            return raw[..., 64:].copy().view(np.int8).reshape(shape), raw[..., :64].copy().view(np.float32)
        return raw.copy().view(NP[self.kv]).reshape(shape), None

    def values(self):
        e, s = self.parts()
        return e.astype(np.float64) * (1.0 if s is None else s.astype(np.float64)[..., None])

    def rows(self, layer, slot, n, values=None):
        """K, V [n, nkv, hd] f64 of a slot's first n places."""
        v = self.values() if values is None else values
        i = np.arange(n)
        b = v[layer, self.table[slot, i // 16]]                      # [n, 2, nkv, 16, hd]
        b = b[i, :, :, i % 16]
        return b[:, 0], b[:, 1]


def f32_rotate(x, cos, sin, rot, layout):
    """The rotation in f32, each product and sum rounded once."""
    y = x.copy()
    a, b = (np.s_[..., :rot // 2], np.s_[..., rot // 2:rot]) if layout == 0 else (np.s_[..., 0:rot:2], np.s_[..., 1:rot:2])
    c, s = cos[:, None], sin[:, None]
    y[a] = x[a] * c - x[b] * s
    y[b] = x[a] * s + x[b] * c
    return y


def f32_quant(x):
    """(int8, scale) by the rule at slate_kv_cache_t, in f32."""
    with np.errstate(all="ignore"):
        scale = np.abs(x).max(-1) * np.float32(1.0 / 127.0)
        q = x / scale[..., None]
        q = np.where(np.isfinite(scale)[..., None] & (scale > 0)[..., None], q, 0)
        return np.clip(np.rint(q), -127, 127).astype(np.int8), scale


APPEND = [  # rows, nq, nkv, hd, rot, layout
    (1, 1, 1, 4, 2, 0), (1, 32, 8, 128, 128, 0), (5, 8, 2, 64, 64, 1), (33, 4, 4, 128, 64, 0), (17, 7, 1, 128, 32, 1),
    (3, 6, 2, 20, 14, 0), (3, 6, 2, 20, 14, 1), (9, 2, 2, 96, 48, 1), (4, 3, 1, 256, 256, 0), (2, 5, 5, 80, 80, 1),
    (300, 4, 2, 32, 32, 0), (6, 2, 1, 16, 8, 0), (40, 16, 2, 112, 56, 0), (3, 4, 2, 128, 6, 0), (70, 9, 3, 64, 48, 0)]


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("rows,nq,nkv,hd,rot,layout", APPEND)
def test_rope_append_and_read(sb, rows, nq, nkv, hd, rot, layout, kv):
    """Every bit of what is written, against the f32 formula step by step; the
    rotation against f64; read-back of both output types."""
    rng = np.random.default_rng(rows + hd + rot)
    slots = min(rows, 4)
    slot = rng.integers(0, slots, rows).astype(np.int32)
    index = np.zeros(rows, np.int32)
    for s in range(slots):                       # distinct places, in no order
        at = np.flatnonzero(slot == s)
        index[at] = rng.permutation(len(at) + 5)[:len(at)]
    c = Cache(sb, kv, 3, nkv, hd, [rows + 5] * slots, seed=rows)
    before = c.raw().copy()
    pos = rng.integers(0, 5000, rows).astype(np.int32)
    cos, sin = sb.rope_tables(5000, rot, 10000.0)
    x = rng.normal(0, 2, (rows, (nq + 2 * nkv) * hd + 3)).astype(np.float32)    # one row [q | k | v], odd stride
    d, dc, ds = dev(x), dev(cos), dev(sin)
    rope = sb.Rope(cos=dc.data_ptr(), sin=ds.data_ptr(), n_pos=5000, rot_dim=rot, layout=layout)
    out = torch.full((rows, nq * hd + 1), 7.0, device="cuda")
    d_slot, d_index, d_pos = dev(slot), dev(index), dev(pos)
    p, ld = d.data_ptr(), x.shape[1]
    sb.rope_append(c.desc, 1, rope, rows, nq, out.data_ptr(), nq * hd + 1, p, ld, p + 4 * nq * hd, ld, p + 4 * (nq + nkv) * hd, ld,
                   d_slot.data_ptr(), d_index.data_ptr(), d_pos.data_ptr())
    q = x[:, :nq * hd].reshape(rows, nq, hd)
    k = x[:, nq * hd:(nq + nkv) * hd].reshape(rows, nkv, hd)
    v = x[:, (nq + nkv) * hd:(nq + 2 * nkv) * hd].reshape(rows, nkv, hd)
    wq, wk = f32_rotate(q, cos[pos], sin[pos], rot, layout), f32_rotate(k, cos[pos], sin[pos], rot, layout)
    got = out.cpu().numpy()
    assert np.array_equal(got[:, :-1].reshape(q.shape), wq) and (got[:, -1] == 7).all()
    # and against f64: two products and a sum, each within 2^-24 of at most |a| + |b|
    q64 = f32_rotate(q.astype(np.float64), cos[pos].astype(np.float64), sin[pos].astype(np.float64), rot, layout)
    assert np.max(np.abs(wq - q64)) <= 3 * 2.0 ** -24 * 2 * np.abs(q).max()
    want = before.copy()
    e, s = c.parts(want)
    page = c.table[slot, index // 16]
    for r in range(rows):
        for w, y in ((0, wk[r]), (1, v[r])):
            if kv == Q8:
                e[1, page[r], w, :, index[r] % 16], s[1, page[r], w, :, index[r] % 16] = f32_quant(y)
            else:
                e[1, page[r], w, :, index[r] % 16] = y.astype(NP[kv])
    ge, gs = c.parts()
    assert np.array_equal(ge, e)
    if kv == Q8:
        assert np.array_equal(gs, s)
        # half a step of the row's scale, the scale's own rounding and the division's added
        vals = ge[1, page, 1][np.arange(rows), :, index % 16] * gs[1, page, 1][np.arange(rows), :, index % 16][..., None]
        assert np.all(np.abs(vals - v) <= np.abs(v).max(-1, keepdims=True) / 127 * (0.5 + 1e-4))
    assert np.array_equal(d.cpu().numpy(), x)
    # read back, all layers, both types
    full = e.astype(np.float32) * (np.float32(1) if s is None else s[..., None])
    for od, dt in ((F32, torch.float32), (F16, torch.float16)):
        K = torch.full((2, rows, nkv, hd), 3.0, dtype=dt, device="cuda")
        V = torch.full_like(K, 3.0)
        sb.kv_read(c.desc, 1, 2, rows, d_slot.data_ptr(), d_index.data_ptr(), K.data_ptr(), V.data_ptr(), od)
        for w, g in ((0, K), (1, V)):
            b = full[1:3, page, w][:, np.arange(rows), :, index % 16]            # [rows, 2, nkv, hd]
            assert np.array_equal(g.cpu().numpy(), np.moveaxis(b, 0, 1).astype(g.cpu().numpy().dtype))


@pytest.mark.parametrize("kv", [F32, F16, Q8])
def test_rope_append_in_place_and_skipped_rows(sb, kv):
    """q_out = q; rows with a negative index or a position outside the tables
    leave everything as it is; a slot or place without a page leaves the cache."""
    nq, nkv, hd, rows = 4, 2, 64, 8
    c = Cache(sb, kv, 1, nkv, hd, [20, 20], seed=3)
    rng = np.random.default_rng(0)
    x = rng.normal(0, 1, (rows, nq * hd)).astype(np.float32)
    kx = rng.normal(0, 1, (rows, nkv * hd)).astype(np.float32)
    cos, sin = sb.rope_tables(50, hd, 1e4)
    slot = np.array([0, 0, 0, 0, 2, -1, 0, 1], np.int32)
    index = np.array([3, -1, 4, 5, 1, 1, 40, 19], np.int32)
    pos = np.array([9, 9, -1, 50, 9, 9, 9, 49], np.int32)
    skipped = [1, 2, 3]                          # rows 4 to 6: turned, but there is no page to write
    before = c.raw().copy()
    d, dk, dc, ds = dev(x), dev(kx), dev(cos), dev(sin)
    arr = [dev(a) for a in (slot, index, pos)]
    rope = sb.Rope(cos=dc.data_ptr(), sin=ds.data_ptr(), n_pos=50, rot_dim=hd, layout=0)
    sb.rope_append(c.desc, 0, rope, rows, nq, d.data_ptr(), nq * hd, d.data_ptr(), nq * hd, dk.data_ptr(), nkv * hd, dk.data_ptr(),
                   nkv * hd, *(a.data_ptr() for a in arr))
    p = np.clip(pos, 0, 49)
    want = f32_rotate(x.reshape(rows, nq, hd), cos[p], sin[p], hd, 0)
    want[skipped] = x.reshape(rows, nq, hd)[skipped]
    assert np.array_equal(d.cpu().numpy().reshape(want.shape), want)
    changed = np.argwhere((c.raw() != before).any((2, 3, 4)))
    assert {tuple(a) for a in changed} == {(0, c.table[0, 0]), (0, c.table[1, 1])}


def test_q8_rows_of_zeros_and_nonfinite_values(sb):
    """Zeros read back as zeros, a row with an infinity or NaN as NaN, the
    smallest numbers within the grid."""
    c = Cache(sb, Q8, 1, 1, 32, [16], fill=False)
    x = np.zeros((6, 32), np.float32)
    x[1, 5] = np.inf
    x[2, 31] = np.nan
    x[3, 0] = 190 * 2.0 ** -149
    x[4, :] = np.linspace(-3e38, 3e38, 32)
    x[5, 7] = 1e-45
    cos, sin = sb.rope_tables(8, 2, 1e4)
    d, dc, ds, i = dev(x), dev(cos), dev(sin), dev(np.arange(6, dtype=np.int32))
    z = torch.zeros(6, dtype=torch.int32, device="cuda")
    rope = sb.Rope(cos=dc.data_ptr(), sin=ds.data_ptr(), n_pos=8, rot_dim=2, layout=0)
    sb.rope_append(c.desc, 0, rope, 6, 1, torch.empty_like(d).data_ptr(), 32, d.data_ptr(), 32, d.data_ptr(), 32, d.data_ptr(), 32,
                   z.data_ptr(), i.data_ptr(), z.data_ptr())
    V = torch.empty(6, 32, device="cuda")
    sb.kv_read(c.desc, 0, 1, 6, z.data_ptr(), i.data_ptr(), torch.empty_like(V).data_ptr(), V.data_ptr(), F32)
    e, s = f32_quant(x)
    with np.errstate(all="ignore"):
        want = e.astype(np.float32) * s[:, None]
    got = V.cpu().numpy()
    assert np.array_equal(got, want, equal_nan=True)
    assert (got[0] == 0).all() and np.isnan(got[1]).all() and np.isnan(got[2]).all()


def test_read_of_places_without_a_page(sb):
    for kv in (F32, F16, Q8):
        c = Cache(sb, kv, 1, 2, 64, [20, 5])
        slot, index = dev(np.array([0, 0, 1, 7, -1, 0, 1], np.int32)), dev(np.array([19, 32, 16, 0, 0, -3, 4], np.int32))
        K = torch.full((7, 2, 64), 5.0, device="cuda")
        V = torch.full_like(K, 5.0)
        sb.kv_read(c.desc, 0, 1, 7, slot.data_ptr(), index.data_ptr(), K.data_ptr(), V.data_ptr(), F32)
        k = K.cpu().numpy()
        assert (k[1:6] == 0).all() and (V.cpu().numpy()[1:6] == 0).all()
        assert np.array_equal(k[0], c.rows(0, 0, 20)[0][19].astype(np.float32))
        assert np.array_equal(k[6], c.rows(0, 1, 5)[0][4].astype(np.float32))


# ---------------------------------------------------------------- attention
def random_tree(rng, n):
    return np.array([-1] + [int(rng.integers(-1 if i % 5 == 4 else 0, i)) for i in range(1, n)][:max(n - 1, 0)], np.int32)[:n]


def attend(sb, c, layer, nodes, ctx, masks, q, scale, slot=None, ld_extra=0, max_nodes=None, stream=None):
    """slate_cuda_attention_tree; q [rows, nq, hd].  Returns out [rows, nq, hd]."""
    off = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    rows, nq, hd = q.shape
    ldq = nq * hd + ld_extra
    qp = np.full((max(rows, 1), ldq), np.nan, np.float32)
    qp[:rows, :nq * hd] = q.reshape(rows, -1)
    keep = [dev(off), dev(np.asarray(slot if slot is not None else np.arange(len(nodes)), np.int32)), dev(np.asarray(ctx, np.int32)),
            dev(np.asarray(masks, np.uint64).view(np.int64)), dev(qp)]
    tree = sb.TreeBatch(n_seq=len(nodes), rows=rows, max_nodes=max_nodes or max(max(nodes), 1), row_off=keep[0].data_ptr(),
                        slot=keep[1].data_ptr(), ctx=keep[2].data_ptr(), mask=keep[3].data_ptr())
    out = torch.full((max(rows, 1), ldq), 9.0, device="cuda")
    n = sb.attention_tree_workspace(c.desc, nq, len(nodes), rows, tree.max_nodes)
    ws = torch.full((n + 64,), 255, dtype=torch.uint8, device="cuda")         # whatever it holds before
    torch.cuda.synchronize()
    sb.attention_tree(c.desc, layer, tree, nq, out.data_ptr(), ldq, keep[4].data_ptr(), ldq, scale, ws.data_ptr(), n, stream)
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert (got[:, nq * hd:] == 9).all() and (ws[n:] == 255).all()
    return got[:rows, :nq * hd].reshape(q.shape)


def plain(c, layer, nodes, ctx, masks, q, scale, slot=None, values=None):
    """The formula in f64, and per row the sum of |q||k| that bounds a score's error."""
    values = c.values() if values is None else values
    out, size = np.zeros(q.shape), 0.0
    r = 0
    for s, n in enumerate(nodes):
        K, V = c.rows(layer, slot[s] if slot is not None else s, ctx[s] + n, values)
        for i in range(n):
            see = np.r_[np.arange(ctx[s]), ctx[s] + np.array([j for j in range(n) if int(masks[r]) >> j & 1], int)].astype(int)
            for h in range(q.shape[1] if len(see) else 0):
                k, v = K[see, h // (q.shape[1] // c.nkv)], V[see, h // (q.shape[1] // c.nkv)]
                z = k @ q[r, h].astype(np.float64) * scale
                size = max(size, abs(scale) * float((np.abs(k) @ np.abs(q[r, h])).mean()))
                p = np.exp(z - z.max())
                out[r, h] = (p @ v) / p.sum()
            r += 1
    return out, size


def check(got, want, size):
    """A score carries at most ~2^-21 of sum |q||k| (22-bit operands, f32 sums), which
    moves p and so the output by the same share; the sums of p and p v add their own
    few 2^-24: 2^-20 (1 + size) of the output's size."""
    assert np.isfinite(got).all()
    err = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30)
    assert err <= 2.0 ** -20 * (1 + size), (err, size)
    assert np.abs(got - want).max() <= 2.0 ** -17 * (1 + size) * max(np.abs(want).max(), 1e-30)


ATTEND = [  # nodes of each sequence, ctx of each, nq, nkv, hd
    ([1], [0], 1, 1, 64), ([1], [1], 4, 2, 128), ([1], [15], 8, 8, 64), ([1, 1, 1], [16, 0, 333], 32, 8, 128),
    ([5], [0], 8, 2, 64), ([7, 1, 16], [1500, 31, 32], 8, 2, 128), ([64, 33], [700, 65], 16, 2, 128), ([3, 0, 2], [40, 9, 17], 7, 1, 64),
    ([13], [4097], 8, 1, 128), ([64], [129], 8, 8, 64), ([17, 2], [255, 1023], 4, 4, 64), ([1] * 9, list(range(9)), 8, 4, 128),
    ([2, 3], [5, 70], 12, 4, 32), ([4, 9], [63, 64], 6, 2, 16), ([5], [90], 4, 2, 96), ([6], [35], 3, 1, 256), ([3], [50], 2, 2, 20),
    ([2], [33], 2, 1, 4), ([9, 30], [100, 300], 33, 1, 80), ([40], [47], 64, 2, 112), ([1], [20000], 8, 2, 128), ([31], [9001], 4, 1, 64)]


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("nodes,ctx,nq,nkv,hd", ATTEND, ids=[str(i) for i in range(len(ATTEND))])
def test_attention_tree(sb, nodes, ctx, nq, nkv, hd, kv):
    rng = np.random.default_rng(len(nodes) + hd + sum(ctx))
    c = Cache(sb, kv, 2, nkv, hd, [x + n for x, n in zip(ctx, nodes)], seed=hd)
    masks = np.concatenate([sb.tree_masks(random_tree(rng, n)) for n in nodes])
    q = rng.normal(0, 1.5, (sum(nodes), nq, hd)).astype(np.float32)
    scale = hd ** -0.5
    got = attend(sb, c, 1, nodes, ctx, masks, q, scale)
    check(got, *plain(c, 1, nodes, ctx, masks, q, scale))


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("hd", [64, 128, 24])
def test_attention_tree_odd_masks_strides_and_shared_slots(sb, kv, hd):
    """Masks that are no trees, a row that sees nothing, sequences that read one
    slot, strides beyond the row, a max_nodes above every sequence's."""
    rng = np.random.default_rng(hd)
    nodes, ctx, slot = [6, 4, 5], [0, 37, 16], [0, 1, 1]
    c = Cache(sb, kv, 1, 2, hd, [6, 41], seed=1)
    masks = rng.integers(0, 2 ** 62, 15).astype(np.uint64) * np.uint64(5)      # bits beyond the nodes are ignored
    masks[1] = 0                                                             # ctx 0: sees nothing
    masks[8] = 0
    masks = np.where(np.arange(15) == 3, np.uint64(0xFFFFFFFFFFFFFFC0), masks)   # names no node of its sequence
    q = rng.normal(0, 1, (15, 6, hd)).astype(np.float32)
    got = attend(sb, c, 0, nodes, ctx, masks, q, 0.3, slot=slot, ld_extra=5, max_nodes=64)
    check(got, *plain(c, 0, nodes, ctx, masks, q, 0.3, slot=slot))
    assert (got[1] == 0).all() and (got[3] == 0).all()


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("hd,nodes", [(64, 12), (128, 3), (128, 40), (40, 9)])
def test_attention_tree_ignores_what_it_does_not_see(sb, kv, hd, nodes):
    """Infinities and NaN in K and V of masked nodes, behind the last node and in
    free pages: rows that do not see them are the same bits as without them."""
    rng = np.random.default_rng(nodes)
    ctx = 45
    c = Cache(sb, kv, 1, 2, hd, [ctx + nodes], seed=2)
    parent = random_tree(rng, nodes)
    bad = 1
    masks = sb.tree_masks(parent)
    masks[2:] &= ~np.uint64(1 << bad)                   # node 1 is seen by itself alone
    masks[0] = 1
    q = rng.normal(0, 1, (nodes, 4, hd)).astype(np.float32)
    clean = attend(sb, c, 0, [nodes], [ctx], masks, q, 0.1)
    raw = c.raw().copy()
    pages = [c.table[0, i // 16] for i in range(ctx + nodes)]
    used = np.zeros((c.n_pages, 16), bool)
    for i, p in enumerate(pages):
        used[p, i % 16] = i != ctx + bad
    for p in range(c.n_pages):
        for t in range(16):
            if used[p, t]:
                continue
            for w, x in ((0, np.nan), (1, np.inf if t % 2 else np.nan)):
                if kv == Q8:
                    raw[0, p, w, :, 4 * t:4 * t + 4] = np.array([x], np.float32).view(np.uint8)
                else:
                    b = raw.dtype.itemsize * hd * (2 if kv == F16 else 4)
                    raw[0, p, w, :, t * b:(t + 1) * b] = np.full(hd, x, NP[kv]).view(np.uint8)
    c.pool.copy_(torch.from_numpy(raw.reshape(-1)))
    dirty = attend(sb, c, 0, [nodes], [ctx], masks, q, 0.1)
    others = np.arange(nodes) != bad
    assert np.array_equal(dirty[others], clean[others])
    assert not np.isfinite(dirty[bad]).any()            # what it does see, it shows


@pytest.mark.parametrize("kv", [F32, F16, Q8])
def test_attention_tree_sizes_of_values(sb, kv):
    """Large and small queries and values: no overflow or loss in the 16-bit
    halves, peaked and flat rows."""
    hd, nq, nkv, nodes, ctx = 128, 8, 2, 5, 500
    rng = np.random.default_rng(5)
    for qs, vs, scale in ((1e5, 1.0, 1e-6), (1e-5, 1.0, 1e4), (30.0, 1.0, 0.2), (1.0, 1e-3, 0.1), (1.0, 200.0 if kv == F16 else 1e6, 0.1)):
        c = Cache(sb, kv, 1, nkv, hd, [ctx + nodes], seed=4)
        raw = c.raw().copy()
        if kv == Q8:
            raw[:, :, 1, :, :64] = (raw[:, :, 1, :, :64].copy().view(np.float32) * np.float32(vs)).view(np.uint8)
        else:
            raw[:, :, 1] = (raw[:, :, 1].copy().view(NP[kv]).astype(np.float32) * np.float32(vs)).astype(NP[kv]).view(np.uint8)
        c.pool.copy_(torch.from_numpy(raw.reshape(-1)))
        masks = sb.tree_masks(random_tree(rng, nodes))
        q = (rng.normal(0, 1, (nodes, nq, hd)) * qs).astype(np.float32)
        got = attend(sb, c, 0, [nodes], [ctx], masks, q, scale)
        check(got, *plain(c, 0, [nodes], [ctx], masks, q, scale))


def test_attention_tree_missing_pages_and_bad_slots(sb):
    """A sequence whose slot or page does not exist sees what there is: nothing is
    read outside the pool."""
    for kv in (F32, F16, Q8):
        c = Cache(sb, kv, 1, 2, 64, [40, 40])
        c.d_table[0, 1] = -1
        c.d_table[1, 0] = c.n_pages
        c.table[0, 1] = c.table[0, 0]                   # not read below
        q = np.random.default_rng(0).normal(0, 1, (4, 4, 64)).astype(np.float32)
        got = attend(sb, c, 0, [1, 1, 1, 1], [20, 10, 12, 9], [1, 1, 1, 1], q, 0.1, slot=[0, 1, 5, -1])
        assert np.isfinite(got).all() and (got[1:] == 0).all()
        cut, _ = plain(c, 0, [0, 1], [0, 15], [1], q[:1], 0.1, slot=[0, 0])       # the first page alone
        assert np.allclose(got[0], cut[0], atol=1e-5)


def test_attention_tree_repeats_bit_for_bit_on_another_stream(sb):
    rng = np.random.default_rng(8)
    nodes, ctx = [9, 30, 1], [3000, 77, 1200]
    for kv in (F32, F16, Q8):
        c = Cache(sb, kv, 1, 2, 128, [x + n for x, n in zip(ctx, nodes)])
        masks = np.concatenate([sb.tree_masks(random_tree(rng, n)) for n in nodes])
        q = rng.normal(0, 1, (40, 8, 128)).astype(np.float32)
        a = attend(sb, c, 0, nodes, ctx, masks, q, 0.1)
        st = torch.cuda.Stream()
        for _ in range(3):
            assert np.array_equal(a, attend(sb, c, 0, nodes, ctx, masks, q, 0.1, stream=st.cuda_stream))


# --------------------------------------------------------------- acceptance
def plain_accept(parent, mask, token, target):
    best, node = [], -1
    for i in range(len(parent)):
        anc = [j for j in range(len(parent)) if int(mask[i]) >> j & 1]
        if all(parent[j] < 0 or (parent[j] < len(parent) and token[j] == target[parent[j]]) for j in anc) and len(anc) > len(best):
            best, node = anc, i
    return best


@pytest.mark.parametrize("kv", [F32, F16, Q8])
@pytest.mark.parametrize("hd", [64, 128, 20, 4])
def test_tree_accept(sb, kv, hd):
    rng = np.random.default_rng(hd + kv)
    nodes = [1, 0, 5, 64, 33, 16, 40, 7, 64]
    ctx = [0, 3, 17, 100, 31, 15, 16, 0, 70]
    c = Cache(sb, kv, 3, 2, hd, [x + n for x, n in zip(ctx, nodes)], seed=5)
    parents = [random_tree(rng, n) for n in nodes]
    masks = [sb.tree_masks(p) for p in parents]
    # few token values: several nodes match, paths of every length and ties among them
    tokens = [rng.integers(0, 3, n).astype(np.int32) for n in nodes]
    targets = [rng.integers(0, 3, n).astype(np.int32) for n in nodes]
    parents[3] = np.arange(64, dtype=np.int32) - 1                       # a chain that is accepted whole
    masks[3] = sb.tree_masks(parents[3])
    tokens[3][1:] = targets[3][:-1]
    parents[8] = np.r_[-1, 0, np.arange(31), np.arange(31, 62)].astype(np.int32)[:64]   # two children a node
    masks[8] = sb.tree_masks(parents[8])
    tokens[8] = np.r_[0, targets[8][parents[8][1:]]].astype(np.int32)    # every node matches: the deepest wins
    parents[5] = parents[5].copy()
    parents[5][3] = 99                                                   # no such parent: never accepted
    off = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    before = c.raw().copy()
    keep = [dev(off), dev(np.arange(len(nodes), dtype=np.int32)), dev(np.array(ctx, np.int32)),
            dev(np.concatenate(masks).view(np.int64)), *(dev(np.concatenate(x).astype(np.int32)) for x in (parents, tokens, targets))]
    tree = sb.TreeBatch(n_seq=len(nodes), rows=int(off[-1]), max_nodes=64, row_off=keep[0].data_ptr(), slot=keep[1].data_ptr(),
                        ctx=keep[2].data_ptr(), mask=keep[3].data_ptr())
    cnt = torch.full((len(nodes),), -7, dtype=torch.int32, device="cuda")
    node, tok = (torch.full((len(nodes), 64), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    sb.tree_accept(c.desc, tree, *(k.data_ptr() for k in keep[4:]), cnt.data_ptr(), node.data_ptr(), tok.data_ptr())
    e0, s0 = c.parts(before)
    we, ws = e0.copy(), None if s0 is None else s0.copy()
    wn, wt = np.full((len(nodes), 64), -1), np.full((len(nodes), 64), -1)
    for s in range(len(nodes)):
        path = plain_accept(parents[s], masks[s], tokens[s], targets[s])
        assert len(path) == int(cnt[s])
        for k, a in enumerate(path):
            wn[s, k], wt[s, k] = a, targets[s][a]
            i, j = ctx[s] + a, ctx[s] + k
            we[:, c.table[s, j // 16], :, :, j % 16] = e0[:, c.table[s, i // 16], :, :, i % 16]
            if ws is not None:
                ws[:, c.table[s, j // 16], :, :, j % 16] = s0[:, c.table[s, i // 16], :, :, i % 16]
    assert int(cnt[3]) == 64 and int(cnt[1]) == 0
    assert np.array_equal(node.cpu().numpy(), wn) and np.array_equal(tok.cpu().numpy(), wt)
    ge, gs = c.parts()
    assert np.array_equal(ge.view(np.uint8), we.view(np.uint8))
    assert ws is None or np.array_equal(gs, ws)


def test_place_beyond_32_bits(sb):
    """A pool of more than 4 GB: the last page of the last layer is addressed in 64 bits."""
    pages, nkv, hd = 8192, 8, 128
    layers = (5 << 30) // sb.kv_pool_bytes(Q8, pages, 1, nkv, hd) + 1
    pool = torch.zeros(sb.kv_pool_bytes(Q8, pages, layers, nkv, hd), dtype=torch.uint8, device="cuda")
    assert pool.numel() > 1 << 32
    table = dev(np.array([[pages - 1]], np.int32))
    c = sb.KVCache(pool=pool.data_ptr(), page_table=table.data_ptr(), n_pages=pages, n_slots=1, max_pages=1, n_layers=layers,
                   n_kv_heads=nkv, head_dim=hd, kv_dtype=Q8)
    x = torch.randn(16, nkv * hd, device="cuda")
    cos, sin = sb.rope_tables(16, 2, 1e4)
    dc, ds, z, i = dev(cos), dev(sin), torch.zeros(16, dtype=torch.int32, device="cuda"), dev(np.arange(16, dtype=np.int32))
    rope = sb.Rope(cos=dc.data_ptr(), sin=ds.data_ptr(), n_pos=16, rot_dim=2, layout=0)
    sb.rope_append(c, layers - 1, rope, 16, 8, torch.empty_like(x).data_ptr(), nkv * hd, x.data_ptr(), nkv * hd, x.data_ptr(), nkv * hd,
                   x.data_ptr(), nkv * hd, z.data_ptr(), i.data_ptr(), i.data_ptr())
    K, V = torch.empty_like(x), torch.empty_like(x)
    sb.kv_read(c, layers - 1, 1, 16, z.data_ptr(), i.data_ptr(), K.data_ptr(), V.data_ptr(), F32)
    e, s = f32_quant(x.cpu().numpy().reshape(16, nkv, hd))
    assert np.array_equal(V.cpu().numpy().reshape(16, nkv, hd), e.astype(np.float32) * s[..., None])
    off, ctx, mask = dev(np.array([0, 1], np.int32)), dev(np.array([15], np.int32)), dev(np.array([1], np.int64))
    tree = sb.TreeBatch(n_seq=1, rows=1, max_nodes=1, row_off=off.data_ptr(), slot=z.data_ptr(), ctx=ctx.data_ptr(), mask=mask.data_ptr())
    n = sb.attention_tree_workspace(c, nkv, 1, 1, 1)
    ws, out = torch.empty(n, dtype=torch.uint8, device="cuda"), torch.empty(1, nkv, hd, device="cuda")
    sb.attention_tree(c, layers - 1, tree, nkv, out.data_ptr(), nkv * hd, x.data_ptr(), nkv * hd, 0.0, ws.data_ptr(), n)
    want = V.view(16, nkv, hd).double().mean(0)                     # scale 0: the mean of V
    assert float((out[0] - want).norm() / want.norm()) < 2.0 ** -19
