"""Cases for the operators that serve a paged KV cache held in 8 bits and trees of drafted tokens over it.

Four operators, as a decoder's layer and its step call them:

  append   rotary positions (half or interleaved pairs, the whole head or its first dims, cos/sin tables that may
           carry a long-context scaling) applied to query and key heads; keys and values written into the paged
           cache, for the 8-bit cache quantised as they are written (one scale for each token and head)
  read     rows of the cache read back as f32 or f16, dequantised
  attend   attention of the nodes of a token tree over the cache: a node sees its sequence's context and, of the
           tree's own tokens (which follow the context in the cache), those that its 64-bit mask names; one node a
           sequence is the ordinary single-token decode
  accept   greedy verification of a drafted tree: the deepest node all of whose ancestors match the model's
           tokens, the tokens that the path yields, and the path's K/V rows moved up behind the context

The paged cache: pool[layer][page][K|V][kv head] blocks of 16 tokens. f32/f16 block: [16][head_dim]. 8-bit block: 16
f32 scales, then [16][head_dim] int8, a value standing for int8 * scale.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
ELEM = {"f32": 4, "f16": 2, "q8": 1}
DEV = "cuda"


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # sixteen sequences write one token each into the 8-bit cache (the 8B-shape heads) and the step reads it back: latency
        {"name": "append 16 tokens 8-bit", "op": "append", "rows": 16, "slots": 16, "start": 300, "nq": 32, "nkv": 8, "hd": 128,
         "rot": 128, "layout": "half", "kv": "q8"},
        # a server's batch of 256 sequences on the f16 cache, narrow heads
        {"name": "append 256 tokens f16", "op": "append", "rows": 256, "slots": 256, "start": 60, "nq": 32, "nkv": 8, "hd": 64,
         "rot": 64, "layout": "half", "kv": "f16"},
        # a long prompt's rows into the 8-bit cache, interleaved pairs over half of the head, read back for dense use
        {"name": "append 8191 rows 8-bit", "op": "append", "rows": 8191, "slots": 1, "start": 5, "nq": 32, "nkv": 8, "hd": 128,
         "rot": 64, "layout": "interleaved", "kv": "q8"},
        # a short session's rows of two layers, as f16 (what a prefix store keeps)
        {"name": "read 517 rows f16 out", "op": "read", "rows": 517, "slots": 3, "nkv": 8, "hd": 64, "kv": "q8", "out": "f16",
         "layers": 2},
        # a long session's rows of four layers back to f32
        {"name": "read 32760 rows f32 out", "op": "read", "rows": 32760, "slots": 1, "nkv": 8, "hd": 128, "kv": "q8", "out": "f32",
         "layers": 4},
        # one sequence, one token: the smallest decode, where latency counts
        {"name": "attend 1 x 1 over 700", "op": "attend", "seqs": 1, "nodes": 1, "ctx": 700, "nq": 32, "nkv": 8, "hd": 128, "kv": "q8"},
        # a server's decode of 64 ragged sequences on the 8-bit cache
        {"name": "attend 64 x 1 over 4096", "op": "attend", "seqs": 64, "nodes": 1, "ctx": 4096, "nq": 32, "nkv": 8, "hd": 128,
         "kv": "q8"},
        # drafted trees of up to 7 nodes, f32 cache, narrow heads
        {"name": "attend 16 x 7 over 1501 f32", "op": "attend", "seqs": 16, "nodes": 7, "ctx": 1501, "nq": 32, "nkv": 8, "hd": 64,
         "kv": "f32"},
        # drafted trees of up to 16 nodes, f16 cache
        {"name": "attend 8 x 16 over 8000 f16", "op": "attend", "seqs": 8, "nodes": 16, "ctx": 8000, "nq": 32, "nkv": 8, "hd": 128,
         "kv": "f16"},
        # wide trees over long contexts, 64 query heads on 8: the most arithmetic for each byte
        {"name": "attend 4 x 64 over 32000", "op": "attend", "seqs": 4, "nodes": 64, "ctx": 32000, "nq": 64, "nkv": 8, "hd": 128,
         "kv": "q8"},
        # one drafted tree of a small model: latency
        {"name": "accept 1 x 13", "op": "accept", "seqs": 1, "nodes": 13, "ctx": 100, "layers": 16, "nkv": 8, "hd": 64, "kv": "f32"},
        # a server's batch of drafted trees over all layers
        {"name": "accept 48 x 40", "op": "accept", "seqs": 48, "nodes": 40, "ctx": 70, "layers": 32, "nkv": 8, "hd": 128, "kv": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "accept"])
    hd = rng.choice([64, 128])
    nkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 7, 8])
    if op == "append":
        rows = _log(rng, 1, 6000)
        slots = rng.choice([1, rows, max(1, rows // rng.randint(2, 40))])
        return {"op": op, "rows": rows, "slots": slots, "start": _log(rng, 1, 700), "nq": nkv * group if nkv * group <= 32 else 32,
                "nkv": nkv, "hd": hd, "rot": rng.choice([hd, hd, hd // 2, 3 * hd // 4]), "layout": rng.choice(["half", "interleaved"]),
                "kv": rng.choice(["q8", "q8", "f16", "f32"])}
    if op == "read":
        layers = rng.randint(1, 4)
        rows = _log(rng, 1, 32000)
        return {"op": op, "rows": rows, "slots": rng.randint(1, min(rows, 64)), "nkv": nkv, "hd": hd,
                "kv": rng.choice(["q8", "q8", "f16", "f32"]), "out": rng.choice(["f32", "f16"]), "layers": layers}
    if op == "attend":
        nodes = rng.choice([1, 1, _log(rng, 2, 64)])
        ctx = _log(rng, 17, 32000)
        seqs = _log(rng, 1, max(1, min(128, 8 * 128000 // (ctx * nkv), 4 * 64 * 64 * 32000 // (ctx * nodes * nkv * group))))
        return {"op": op, "seqs": seqs, "nodes": nodes, "ctx": ctx, "nq": nkv * group, "nkv": nkv, "hd": hd,
                "kv": rng.choice(["q8", "q8", "f16", "f32"])}
    return {"op": op, "seqs": _log(rng, 1, 48), "nodes": _log(rng, 1, 40), "ctx": rng.randint(0, 120), "layers": rng.randint(1, 16), "nkv": nkv,
            "hd": hd, "kv": rng.choice(["f16", "f32"])}


# ------------------------------------------------------------------------------------- shapes that follow from a case
def _nodes(c):
    """Nodes of each sequence's tree: the case's number and down to half of it."""
    return [c["nodes"] - (5 * s) % (c["nodes"] // 2 + 1) for s in range(c["seqs"])]


def _contexts(c):
    """Context length of each sequence: the case's number and down to half of it."""
    return [c["ctx"] - (7919 * s) % (c["ctx"] // 2 + 1) for s in range(c["seqs"])]


def _depth(n):
    """Nodes on the drafted path that the model agrees with."""
    return n // 4 + 1


def _block(c):
    """Bytes of one (page, K or V, head) block."""
    return 64 + PAGE * c["hd"] if c["kv"] == "q8" else PAGE * c["hd"] * ELEM[c["kv"]]


def _row_bytes(c):
    """Bytes of one token's K and V in one layer."""
    return 2 * c["nkv"] * (c["hd"] + 4 if c["kv"] == "q8" else c["hd"] * ELEM[c["kv"]])


def work(case):
    c = case
    if c["op"] == "append":
        q, kv = 4 * c["rows"] * c["nq"] * c["hd"], 8 * c["rows"] * c["nkv"] * c["hd"]
        b = 2 * q + kv + c["rows"] * (_row_bytes(c) + 12 + 4 * c["rot"])
        if c["kv"] == "q8":
            b += kv + c["rows"] * _row_bytes(c)  # read back
        return {"bytes": b, "flops": 3 * c["rows"] * (c["nq"] + c["nkv"]) * c["rot"]}
    if c["op"] == "read":
        out = 4 if c["out"] == "f32" else 2
        return {"bytes": c["rows"] * (8 + c["layers"] * (_row_bytes(c) + 2 * out * c["nkv"] * c["hd"])),
                "flops": 2 * c["rows"] * c["layers"] * c["nkv"] * c["hd"]}
    n, x = _nodes(c), _contexts(c)
    if c["op"] == "attend":
        b = sum((xi + ni) * _row_bytes(c) + ni * (8 * c["nq"] * c["hd"] + 8) for ni, xi in zip(n, x))
        return {"bytes": b, "flops": sum(4 * c["hd"] * c["nq"] * ni * (xi + 1) for ni, xi in zip(n, x))}
    return {"bytes": sum(_depth(ni) * (2 * c["layers"] * _row_bytes(c) + 8) + 20 * ni for ni in n), "flops": 0}


# ---------------------------------------------------------------------------------------------------- inputs
def _i32(a):
    return torch.tensor(np.ascontiguousarray(a, dtype=np.int32), device=DEV)


def _normal(g, shape, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV) * scale


def _pool(c, g, n_pages, layers):
    """A pool whose every row holds what a model leaves there: normal values, heads and tokens of different size."""
    n = layers * n_pages * 2 * c["nkv"]
    size = torch.exp(0.5 * _normal(g, (n, PAGE, 1)))
    if c["kv"] == "q8":
        p = torch.empty(n, _block(c), dtype=torch.uint8, device=DEV)
        p[:, :64] = (size.view(n, PAGE) * (3.0 / 127)).contiguous().view(torch.uint8)
        p[:, 64:] = (_normal(g, (n, PAGE * c["hd"]), 40.0).round_().clamp_(-127, 127).to(torch.int8)).view(torch.uint8)
        return p.view(layers, n_pages, 2, c["nkv"], _block(c))
    p = _normal(g, (n, PAGE, c["hd"])) * size
    return p.to(torch.float16 if c["kv"] == "f16" else torch.float32).view(layers, n_pages, 2, c["nkv"], PAGE, c["hd"])


def _pages(r, lengths):
    """Shuffled pages for sequences of these lengths: the table, and the number of pages in the pool."""
    need = [-(-max(1, n) // PAGE) for n in lengths]
    ids = r.permutation(sum(need) + 3).astype(np.int32)
    table = np.full((len(lengths), max(need) + 1), -1, np.int32)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = ids[at:at + k]
        at += k
    return table, len(ids)


def _trees(r, counts):
    """Random trees: parents, masks (bit j: the node sees node j, itself included) and the path that the model will agree with."""
    parent, mask, path = [], [], []
    for n in counts:
        on = np.concatenate([[0], np.sort(r.permutation(n - 1)[:_depth(n) - 1] + 1)]).astype(np.int64) if n > 1 else np.zeros(1, np.int64)
        p = np.array([-1] + [int(r.randint(0, i)) for i in range(1, n)])
        p[on[1:]] = on[:-1]
        m = [0] * n
        for i in range(n):
            m[i] = (m[p[i]] if p[i] >= 0 else 0) | (1 << i)
        parent.append(p)
        mask.append(np.array(m, np.uint64))
        path.append(on)
    return parent, mask, path


def prepare(case, seed):
    c = case
    r = np.random.RandomState((seed * 2654435761 + 12345) % (1 << 32))
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    st = {"case": c}
    if c["op"] in ("append", "read"):
        rows, slots = c["rows"], c["slots"]
        slot = np.arange(rows) * slots // rows
        first = np.searchsorted(slot, np.arange(slots))
        start = c.get("start", 0)
        begin = np.array([start - (31 * s) % (start // 2 + 1) for s in range(slots)])
        index = begin[slot] + np.arange(rows) - first[slot]
        lengths = [int(b + n) for b, n in zip(begin, np.bincount(slot, minlength=slots))]
        layers = c.get("layers", 2)
    else:
        nodes, ctx = _nodes(c), _contexts(c)
        lengths = [x + n for x, n in zip(ctx, nodes)]
        layers = c.get("layers", 1)
    table, n_pages = _pages(r, lengths)
    st.update(table=torch.tensor(table, device=DEV), n_pages=n_pages, layers=layers, layer=layers - 1)
    st["pool"] = _pool(c, g, n_pages, layers)
    if c["op"] in ("append", "read"):
        st.update(slot=_i32(slot), index=_i32(index))
    if c["op"] == "append":
        half = c["rot"] // 2
        far = int(max(lengths)) + 7
        inv = 500000.0 ** (-np.arange(half) / half) / (4.0 if c["layout"] == "interleaved" else 1.0)  # positions compressed four times
        ang = torch.tensor(np.arange(far)[:, None] * inv[None, :], device=DEV)
        st.update(pos=_i32(index), cos=ang.cos().float().contiguous(), sin=ang.sin().float().contiguous())
        st["q"] = _normal(g, (rows, c["nq"], c["hd"]))
        st["k"] = _normal(g, (rows, c["nkv"], c["hd"]), 2.0)
        st["v"] = _normal(g, (rows, c["nkv"], c["hd"]))
        st["q_out"] = torch.empty_like(st["q"])
    if c["op"] == "read" or (c["op"] == "append" and c["kv"] == "q8"):
        dt = torch.float16 if c.get("out") == "f16" else torch.float32
        n_read = c["layers"] if c["op"] == "read" else 1
        st["K"] = torch.empty(n_read, rows, c["nkv"], c["hd"], dtype=dt, device=DEV)
        st["V"] = torch.empty_like(st["K"])
    if c["op"] in ("attend", "accept"):
        parent, mask, path = _trees(r, nodes)
        off = np.concatenate([[0], np.cumsum(nodes)])
        rows = int(off[-1])
        st.update(rows=rows, off=_i32(off), seq=_i32(np.arange(c["seqs"])), ctx=_i32(ctx), longest=max(lengths),
                  mask=torch.tensor(np.concatenate(mask).view(np.int64), device=DEV))
    if c["op"] == "attend":
        st["q"] = _normal(g, (rows, c["nq"], c["hd"]), 1.5)
        st["out"] = torch.empty_like(st["q"])
    if c["op"] == "accept":
        tokens, target = [], []
        for n, p, on in zip(nodes, parent, path):
            t = r.permutation(32000)[:n]  # distinct: what is off the path never matches
            w = 32000 + r.randint(0, 32000, n)
            w[on[:-1]] = t[on[1:]]
            tokens.append(t)
            target.append(w)
        st.update(parent=_i32(np.concatenate(parent)), tokens=_i32(np.concatenate(tokens)), target=_i32(np.concatenate(target)))
        for name, shape in (("count", (c["seqs"],)), ("node", (c["seqs"], 64)), ("next", (c["seqs"], 64))):
            st[name] = torch.empty(shape, dtype=torch.int32, device=DEV)
    if own:
        _handles(st)
    return st


# ---------------------------------------------------------------------------------------- the framework's operators
def _handles(st):
    """The descriptors that a program keeps beside its cache: they hold addresses and sizes."""
    import slate_b200 as sb
    c, t = st["case"], st["table"]
    st["sb"] = sb
    st["cache"] = sb.KVCache(pool=st["pool"].data_ptr(), page_table=t.data_ptr(), n_pages=st["n_pages"], n_slots=t.shape[0],
                             max_pages=t.shape[1], n_layers=st["layers"], n_kv_heads=c["nkv"], head_dim=c["hd"],
                             kv_dtype={"f32": sb.KV_F32, "f16": sb.KV_F16, "q8": sb.KV_Q8}[c["kv"]])
    if c["op"] == "append":
        st["rope"] = sb.Rope(cos=st["cos"].data_ptr(), sin=st["sin"].data_ptr(), n_pos=st["cos"].shape[0], rot_dim=c["rot"],
                             layout=sb.ROPE_HALF if c["layout"] == "half" else sb.ROPE_INTERLEAVED)
    if c["op"] in ("attend", "accept"):
        st["tree"] = sb.TreeBatch(n_seq=c["seqs"], rows=st["rows"], max_nodes=c["nodes"], row_off=st["off"].data_ptr(),
                                  slot=st["seq"].data_ptr(), ctx=st["ctx"].data_ptr(), mask=st["mask"].data_ptr())
    if c["op"] == "attend":
        st["ws"] = torch.empty(sb.attention_tree_workspace(st["cache"], c["nq"], c["seqs"], st["rows"], c["nodes"]), dtype=torch.uint8,
                               device=DEV)


def _own(st):
    sb, c, stream = st["sb"], st["case"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "append":
        qd, kd = c["nq"] * c["hd"], c["nkv"] * c["hd"]
        sb.rope_append(st["cache"], st["layer"], st["rope"], c["rows"], c["nq"], st["q_out"].data_ptr(), qd, st["q"].data_ptr(), qd,
                       st["k"].data_ptr(), kd, st["v"].data_ptr(), kd, st["slot"].data_ptr(), st["index"].data_ptr(),
                       st["pos"].data_ptr(), stream)
        if c["kv"] != "q8":
            return st["q_out"], st["pool"]
        sb.kv_read(st["cache"], st["layer"], 1, c["rows"], st["slot"].data_ptr(), st["index"].data_ptr(), st["K"].data_ptr(),
                   st["V"].data_ptr(), sb.KV_F32, stream)
        return st["q_out"], st["K"], st["V"]
    if c["op"] == "read":
        sb.kv_read(st["cache"], 0, c["layers"], c["rows"], st["slot"].data_ptr(), st["index"].data_ptr(), st["K"].data_ptr(),
                   st["V"].data_ptr(), sb.KV_F16 if c["out"] == "f16" else sb.KV_F32, stream)
        return st["K"], st["V"]
    if c["op"] == "attend":
        qd = c["nq"] * c["hd"]
        sb.attention_tree(st["cache"], st["layer"], st["tree"], c["nq"], st["out"].data_ptr(), qd, st["q"].data_ptr(), qd,
                          c["hd"] ** -0.5, st["ws"].data_ptr(), st["ws"].numel(), stream)
        return st["out"]
    sb.tree_accept(st["cache"], st["tree"], st["parent"].data_ptr(), st["tokens"].data_ptr(), st["target"].data_ptr(),
                   st["count"].data_ptr(), st["node"].data_ptr(), st["next"].data_ptr(), stream)
    return st["count"], st["node"], st["next"], st["pool"]


# ------------------------------------------------------------------------------------------------- the plain forms
def _rotate(x, cos, sin, rot, layout):
    """The pairs of the first `rot` dims turned by their angles; the rest as it is. x [rows, heads, hd], cos/sin [rows, 1, rot / 2]."""
    y = x.clone()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


def _write(st, which, x):
    """Rows x [rows, heads, hd] into the cache's K (0) or V (1)."""
    c, pool = st["case"], st["pool"][st["layer"]]
    index = st["index"].long()
    page = st["table"][st["slot"].long(), index // PAGE].long()[:, None]
    t, head = (index % PAGE)[:, None], torch.arange(c["nkv"], device=DEV)[None]
    if c["kv"] != "q8":
        pool[page, which, head, t] = x.to(pool.dtype)
        return
    scale = x.abs().amax(-1, keepdim=True) * (1.0 / 127.0)
    v = torch.where(scale > 0, x / scale, torch.zeros_like(x)).round().clamp(-127, 127).to(torch.int8)
    at = torch.arange(c["hd"], device=DEV) + 64 + c["hd"] * t[..., None]
    pool.view(torch.int8)[page[..., None], which, head[..., None], at] = v
    pool[..., :64].view(torch.float32)[page, which, head, t] = scale[..., 0]


def _values(blocks, c):
    """Cache blocks [..., block bytes] (8 bits) or [..., 16, hd] as f32 [..., 16, hd]."""
    if c["kv"] != "q8":
        return blocks.float()
    v = blocks[..., 64:].view(torch.int8).float().unflatten(-1, (PAGE, c["hd"]))
    return v * blocks[..., :64].contiguous().view(torch.float32)[..., None]


def _read(st, layers, dtype):
    c = st["case"]
    index = st["index"].long()
    page, t = st["table"][st["slot"].long(), index // PAGE].long(), index % PAGE
    head = torch.arange(c["nkv"], device=DEV)[None]
    pool = st["pool"][layers]
    if c["kv"] != "q8":
        return tuple(pool[:, page[:, None], w, head, t[:, None]].to(dtype) for w in (0, 1))
    at = torch.arange(c["hd"], device=DEV) + 64 + c["hd"] * t[:, None, None]
    scale = pool[..., :64].view(torch.float32)
    return tuple((pool.view(torch.int8)[:, page[:, None, None], w, head[..., None], at].float()
                  * scale[:, page[:, None], w, head, t[:, None]][..., None]).to(dtype) for w in (0, 1))


def _padded(st):
    """Row numbers of each sequence's nodes padded to one length, which of them are nodes, and their masks as truth values."""
    off, n = st["off"].long(), st["case"]["nodes"]
    i = torch.arange(n, device=DEV)
    row = off[:-1, None] + i
    live = row < off[1:, None]
    row = row.clamp(max=st["rows"] - 1)
    sees = (st["mask"][row][..., None] >> i) & 1 > 0
    return row, live, sees & live[..., None]


def _attend(st):
    c = st["case"]
    S, nq, nkv, hd, n = c["seqs"], c["nq"], c["nkv"], c["hd"], c["nodes"]
    G = nq // nkv
    row, live, sees = _padded(st)
    P = -(-st["longest"] // PAGE)
    blocks = st["pool"][st["layer"]][st["table"][st["seq"].long(), :P].long().clamp(min=0)]  # [S, P, 2, nkv, ...]
    kv = _values(blocks, c).permute(2, 0, 3, 1, 4, 5).reshape(2, S, nkv, P * PAGE, hd)
    q = st["q"][row].view(S, n, nkv, G, hd).permute(0, 2, 3, 1, 4).reshape(S, nkv, G * n, hd)
    s = torch.matmul(q, kv[0].transpose(-1, -2)).view(S, nkv, G, n, P * PAGE) * hd ** -0.5
    key = torch.arange(P * PAGE, device=DEV)[None] - st["ctx"].long()[:, None]  # below 0: the context
    inside = (key >= 0) & (key < n)
    vis = torch.where(inside[:, None], sees.gather(2, key.clamp(0, n - 1)[:, None].expand(S, n, -1)), (key < 0)[:, None])
    s = s.masked_fill_(~vis[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    l = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(S, nkv, G * n, -1), kv[1]).view(S, nkv, G, n, hd)
    o = torch.where(l > 0, o / l, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(S, n, nq, hd)
    st["out"][row[live]] = o[live]
    return st["out"]


def _accept(st):
    c, n = st["case"], st["case"]["nodes"]
    row, live, sees = _padded(st)
    off = st["off"].long()
    parent = st["parent"][row].long()
    said = st["target"].long()[(off[:-1, None] + parent).clamp(0, st["rows"] - 1)]
    good = (parent < 0) | (st["tokens"][row] == said)
    whole = live & (good[:, None, :] | ~sees).all(-1)
    depth = sees.sum(-1)
    score = torch.where(whole, depth * 64 + (63 - torch.arange(n, device=DEV)), torch.zeros_like(depth))
    best = score.argmax(-1)
    on = sees.gather(1, best[:, None, None].expand(-1, 1, n))[:, 0]  # the path, in order of nodes
    on = on & (score.amax(-1, keepdim=True) > 0)
    count = on.sum(-1)
    node = torch.where(on, torch.arange(n, device=DEV), 64).sort(-1).values
    kept = node < 64
    token = torch.where(kept, st["target"].long().gather(0, (off[:-1, None] + node).clamp(max=st["rows"] - 1).flatten()).view_as(node), -1)
    st["count"].copy_(count)
    st["node"].fill_(-1)[:, :n] = torch.where(kept, node, -1).int()
    st["next"].fill_(-1)[:, :n] = token.int()
    # the path's rows, all layers, gathered before any is written
    s, k = kept.nonzero(as_tuple=True)
    src, dst = (st["ctx"].long()[s] + node[s, k], st["ctx"].long()[s] + k)
    at = lambda i: (st["table"][s, i // PAGE].long(), i % PAGE)  # noqa: E731
    (p0, t0), (p1, t1) = at(src), at(dst)
    st["pool"][:, p1, :, :, t1] = st["pool"][:, p0, :, :, t0]
    return st["count"], st["node"], st["next"], st["pool"]


def run(state):
    if own:
        return _own(state)
    st, c = state, state["case"]
    if c["op"] == "attend":
        return _attend(st)
    if c["op"] == "accept":
        return _accept(st)
    if c["op"] == "read":
        K, V = _read(st, slice(0, c["layers"]), st["K"].dtype)
        return K, V
    pos = st["pos"].long()
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]
    q = _rotate(st["q"], cos, sin, c["rot"], c["layout"])
    _write(st, 0, _rotate(st["k"], cos, sin, c["rot"], c["layout"]))
    _write(st, 1, st["v"])
    if c["kv"] != "q8":
        return q, st["pool"]
    K, V = _read(st, slice(st["layer"], st["layer"] + 1), torch.float32)
    return q, K, V


# ----------------------------------------------------------------------------------------------------- in 64 bits
def _row64(st, which, layer, slot, index):
    """One cache row's values [nkv, hd] in 64 bits for each of the given places."""
    c = st["case"]
    b = st["pool"][layer, st["table"][slot, index // PAGE].long(), which]
    n = torch.arange(len(index), device=DEV)
    if c["kv"] != "q8":
        return b[n, :, index % PAGE].double()
    raw = b[..., 64:].view(torch.int8).reshape(len(index), c["nkv"], PAGE, c["hd"])[n, :, index % PAGE].double()
    return raw * b[..., :64].contiguous().view(torch.float32)[n, :, index % PAGE].double()[..., None]


def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["op"] == "read":
        slot, index = st["slot"].long(), st["index"].long()
        return tuple(torch.stack([_row64(st, w, l, slot, index) for l in range(c["layers"])]) for w in (0, 1))
    if c["op"] == "append":
        ang = st["pos"].long()
        cs, sn = st["cos"].double()[ang][:, None, :], st["sin"].double()[ang][:, None, :]
        h = c["rot"] // 2

        def turn(x):
            x = x.double()
            head, rest = x[..., :c["rot"]], x[..., c["rot"]:]
            z = head.unflatten(-1, (2, h)).transpose(-1, -2) if c["layout"] == "half" else head.unflatten(-1, (h, 2))
            z = torch.view_as_complex(z.contiguous()) * torch.complex(cs, sn)
            z = torch.view_as_real(z)
            z = (z.transpose(-1, -2) if c["layout"] == "half" else z).flatten(-2)
            return torch.cat([z, rest], -1)

        q, k, v = turn(st["q"]), turn(st["k"]), st["v"].double()
        if c["kv"] == "q8":
            back = []
            for x in (k, v):
                unit = x.abs().max(-1, keepdim=True).values / 127
                back.append((torch.round(x / unit) * unit)[None])
            return (q, *back)
        pool = st["pool"].double()
        for w, x in ((0, k), (1, v)):
            for r in range(c["rows"]) if c["rows"] <= 300 else ():
                s, i = int(st["slot"][r]), int(st["index"][r])
                pool[st["layer"], int(st["table"][s, i // PAGE]), w, :, i % PAGE] = x[r]
        return q, pool if c["rows"] <= 300 else None
    off = st["off"].tolist()
    ctx = st["ctx"].tolist()
    mask = st["mask"].tolist()
    if c["op"] == "attend":
        out = torch.zeros(st["rows"], c["nq"], c["hd"], dtype=torch.float64, device=DEV)
        G = c["nq"] // c["nkv"]
        for s in range(c["seqs"]):
            n = off[s + 1] - off[s]
            i = torch.arange(ctx[s] + n, device=DEV)
            K, V = (_row64(st, w, st["layer"], torch.full_like(i, s), i) for w in (0, 1))
            sees = torch.tensor([[mask[off[s] + a] >> b & 1 for b in range(n)] for a in range(n)], dtype=torch.bool, device=DEV)
            for h in range(c["nq"]):
                z = st["q"][off[s]:off[s + 1], h].double() @ K[:, h // G].T / math.sqrt(c["hd"])
                z[:, ctx[s]:][~sees] = -math.inf
                out[off[s]:off[s + 1], h] = torch.softmax(z, -1) @ V[:, h // G]
        return out
    parent, tok, want = st["parent"].tolist(), st["tokens"].tolist(), st["target"].tolist()
    pool, table = st["pool"].clone(), st["table"].tolist()
    for s in range(c["seqs"]):
        best = []
        for i in range(off[s + 1] - off[s]):
            path, a = [], i
            while a >= 0:
                path.insert(0, a)
                a = parent[off[s] + a]
            if all(tok[off[s] + b] == want[off[s] + a] for a, b in zip(path, path[1:])) and len(path) > len(best):
                best = path
        for k, a in enumerate(best):
            i, j = ctx[s] + a, ctx[s] + k
            pool[:, table[s][j // PAGE], :, :, j % PAGE] = st["pool"][:, table[s][i // PAGE], :, :, i % PAGE]
    return None, None, None, pool.double()
