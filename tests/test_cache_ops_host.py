"""Host side of the cache operators, without a GPU: rotary tables, tree masks,
pool sizes, and what every entry refuses before it touches a device."""
import ctypes as C
import math

import numpy as np
import pytest


def angles(n_pos, rot, theta, kind=0, factor=1.0, low=1.0, high=4.0, trained=64):
    """[n_pos, rot/2] angles in f64, by the definitions at slate_rope_scaling_t."""
    j = np.arange(rot // 2, dtype=np.float64)
    if kind == 2:
        theta = theta * factor ** (rot / (rot - 2))
    w = theta ** (-2 * j / rot)
    if kind == 1:
        w = w / factor
    if kind == 3:
        wave = 2 * math.pi / w
        out = []
        for wi, la in zip(w, wave):
            if la > trained / low:
                out.append(wi / factor)
            elif la < trained / high:
                out.append(wi)
            else:
                keep = (trained / la - low) / (high - low)
                out.append((1 - keep) * wi / factor + keep * wi)
        w = np.array(out)
    return np.arange(n_pos)[:, None] * w[None]


@pytest.mark.parametrize("kind", [0, 1, 2, 3])
@pytest.mark.parametrize("rot,n_pos", [(4, 1), (64, 700), (128, 33)])
def test_rope_tables(sb, kind, rot, n_pos):
    f32 = np.float32
    theta, factor, low, high, trained, mag = 500000.0, 4.0, 1.0, 4.0, 256, 1.25
    sc = sb.RopeScaling(kind, factor, low, high, trained, mag)
    cos, sin = sb.rope_tables(n_pos, rot, theta, sc)
    a = angles(n_pos, rot, theta, kind, factor, low, high, trained)
    # one rounding to f32 of values up to 1.25; the f64 angle is good to ~1e-13 here
    assert np.max(np.abs(cos - mag * np.cos(a))) < 1.25 * 2.0 ** -24 + 1e-10
    assert np.max(np.abs(sin - mag * np.sin(a))) < 1.25 * 2.0 ** -24 + 1e-10
    assert cos.dtype == f32 and cos.shape == (n_pos, rot // 2)


def test_rope_tables_far_positions(sb):
    """Angles beyond 10^5 turns keep f32 accuracy (a product in f32 would not)."""
    cos, sin = sb.rope_tables(131072, 4, 10000.0)
    a = angles(131072, 4, 10000.0)
    assert np.max(np.abs(cos - np.cos(a))) < 2.0 ** -23
    assert np.max(np.abs(sin - np.sin(a))) < 2.0 ** -23


@pytest.mark.parametrize("bad", [dict(n_pos=0), dict(rot=3), dict(rot=0), dict(theta=0.0), dict(theta=float("nan")),
                                 dict(kind=4), dict(kind=1, factor=0.5), dict(kind=1, factor=float("inf")),
                                 dict(kind=2, rot=2), dict(kind=3, low=0.0), dict(kind=3, low=4.0, high=4.0),
                                 dict(kind=3, trained=0), dict(mag=-1.0), dict(mag=float("nan"))])
def test_rope_tables_refusals(sb, bad):
    a = dict(n_pos=4, rot=8, theta=1e4, kind=0, factor=2.0, low=1.0, high=4.0, trained=64, mag=1.0)
    a.update(bad)
    with pytest.raises(ValueError, match="rope_tables"):
        sb.rope_tables(a["n_pos"], a["rot"], a["theta"],
                       sb.RopeScaling(a["kind"], a["factor"], a["low"], a["high"], a["trained"], a["mag"]))


def test_tree_masks(sb):
    parent = [-1, 0, 0, 1, 3, 2, -1, 6]
    want = []
    for i, p in enumerate(parent):
        m, a = 0, i
        while a >= 0:
            m |= 1 << a
            a = parent[a]
        want.append(m)
    assert list(sb.tree_masks(parent)) == want
    chain = sb.tree_masks(np.arange(64) - 1)
    assert int(chain[63]) == (1 << 64) - 1
    assert len(sb.tree_masks([])) == 0
    for bad in ([0], [-1, 1], [-1, -2], list(range(-1, 64))):
        with pytest.raises(ValueError, match="tree_masks"):
            sb.tree_masks(bad)


def test_kv_pool_bytes(sb):
    assert sb.kv_pool_bytes(sb.KV_F32, 3, 2, 4, 64) == 3 * 2 * 2 * 4 * 16 * 64 * 4
    assert sb.kv_pool_bytes(sb.KV_F16, 3, 2, 4, 64) == 3 * 2 * 2 * 4 * 16 * 64 * 2
    assert sb.kv_pool_bytes(sb.KV_Q8, 3, 2, 4, 64) == 3 * 2 * 2 * 4 * (16 * 64 + 64)
    assert sb.kv_pool_bytes(3, 3, 2, 4, 64) == 0 and sb.kv_pool_bytes(0, 0, 2, 4, 64) == 0
    assert sb.kv_pool_bytes(sb.KV_F32, 1 << 24, 80, 8, 128) == (1 << 24) * 80 * 2 * 8 * 16 * 128 * 4


GOOD_CACHE = dict(pool=4096, page_table=4096, n_pages=8, n_slots=2, max_pages=4, n_layers=2, n_kv_heads=2,
                  head_dim=64, kv_dtype=2)
BAD_CACHES = [dict(pool=None), dict(pool=4100), dict(page_table=None), dict(n_pages=0), dict(n_slots=0), dict(max_pages=0),
              dict(n_layers=0), dict(n_kv_heads=0), dict(head_dim=0), dict(head_dim=66), dict(head_dim=260),
              dict(kv_dtype=3), dict(kv_dtype=-1)]
GOOD_TREE = dict(n_seq=2, rows=3, max_nodes=2, row_off=4096, slot=4096, ctx=4096, mask=4096)
BAD_TREES = [dict(n_seq=0), dict(rows=-1), dict(rows=5), dict(max_nodes=0), dict(max_nodes=65), dict(row_off=None),
             dict(slot=None), dict(ctx=None), dict(mask=None)]
GOOD_ROPE = dict(cos=4096, sin=4096, n_pos=16, rot_dim=64, layout=0)
BAD_ROPES = [dict(cos=None), dict(sin=None), dict(n_pos=0), dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=66), dict(layout=2)]
D = 4096     # stands for a device address: every refusal comes before any device work


def _rope_append(sb, cache=None, rope=None, **kw):
    a = dict(layer=1, rows=3, n_heads=4, q_out=D, ld_q_out=256, q=D, ld_q=256, k=D, ld_k=128, v=D, ld_v=128, row_slot=D,
             row_index=D, row_pos=D)
    a.update(kw)
    sb.rope_append(sb.KVCache(**{**GOOD_CACHE, **(cache or {})}), a["layer"], sb.Rope(**{**GOOD_ROPE, **(rope or {})}), a["rows"],
                   a["n_heads"], a["q_out"], a["ld_q_out"], a["q"], a["ld_q"], a["k"], a["ld_k"], a["v"], a["ld_v"],
                   a["row_slot"], a["row_index"], a["row_pos"])


def _kv_read(sb, cache=None, **kw):
    a = dict(layer0=0, n_layers=2, rows=3, row_slot=D, row_index=D, K=D, V=D, out=0)
    a.update(kw)
    sb.kv_read(sb.KVCache(**{**GOOD_CACHE, **(cache or {})}), a["layer0"], a["n_layers"], a["rows"], a["row_slot"], a["row_index"],
               a["K"], a["V"], a["out"])


def _attend(sb, cache=None, tree=None, **kw):
    a = dict(layer=1, n_heads=4, out=D, ld_out=256, q=D, ld_q=256, scale=0.125, ws=D, ws_bytes=1 << 40)
    a.update(kw)
    sb.attention_tree(sb.KVCache(**{**GOOD_CACHE, **(cache or {})}), a["layer"], sb.TreeBatch(**{**GOOD_TREE, **(tree or {})}),
                      a["n_heads"], a["out"], a["ld_out"], a["q"], a["ld_q"], a["scale"], a["ws"], a["ws_bytes"])


def _accept(sb, cache=None, tree=None, **kw):
    a = dict(parent=D, token=D, target=D, count=D, node=D, out=D)
    a.update(kw)
    sb.tree_accept(sb.KVCache(**{**GOOD_CACHE, **(cache or {})}), sb.TreeBatch(**{**GOOD_TREE, **(tree or {})}), a["parent"],
                   a["token"], a["target"], a["count"], a["node"], a["out"])


REFUSALS = (
    [(f, dict(cache=b)) for f in (_rope_append, _kv_read, _attend, _accept) for b in BAD_CACHES]
    + [(f, dict(tree=b)) for f in (_attend, _accept) for b in BAD_TREES]
    + [(_rope_append, dict(rope=b)) for b in BAD_ROPES]
    + [(_rope_append, {k: v}) for k, v in dict(layer=2, rows=-1, n_heads=0, q_out=None, ld_q_out=255, q=None, ld_q=255, k=None,
                                               ld_k=127, v=None, ld_v=127, row_slot=None, row_index=None, row_pos=None).items()]
    + [(_kv_read, {k: v}) for k, v in dict(layer0=1, n_layers=0, rows=-1, row_slot=None, row_index=None, K=None, V=None,
                                           out=2).items()]
    + [(_attend, {k: v}) for k, v in dict(layer=-1, n_heads=3, out=None, ld_out=255, q=None, ld_q=255, scale=float("inf"),
                                          ws=None, ws_bytes=0).items()]
    + [(_attend, dict(n_heads=0)), (_attend, dict(ws=D + 8)), (_attend, dict(scale=float("nan")))]
    + [(_accept, {k: None}) for k in ("parent", "token", "target", "count", "node", "out")])


@pytest.mark.parametrize("call,bad", REFUSALS, ids=[f"{f.__name__[1:]}-{i}" for i, (f, _) in enumerate(REFUSALS)])
def test_refusals(sb, call, bad):
    with pytest.raises(RuntimeError, match=call.__name__[1:].replace("attend", "attention_tree").replace("accept", "tree_accept")):
        call(sb, **bad)
    assert sb.last_error()


def test_refusals_of_null_descriptors(sb):
    none = C.POINTER(sb.KVCache)()
    assert sb.F["slate_cuda_kv_read"](none, 0, 1, 1, D, D, D, D, 0, None) == -1
    assert sb.F["slate_cuda_attention_tree"](none, 0, None, 1, D, 64, D, 64, 1.0, D, 16, None) == -1
    assert sb.F["slate_cuda_attention_tree_workspace"](none, 4, 1, 1, 1) == 0


def test_empty_calls_do_nothing(sb):
    """No rows: accepted, and nothing is launched (this runs without a GPU)."""
    _rope_append(sb, rows=0)
    _kv_read(sb, rows=0)
    _attend(sb, tree=dict(rows=0))
