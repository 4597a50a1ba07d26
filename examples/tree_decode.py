"""Greedy decoding that verifies a tree of drafted tokens a step, on an 8-bit (or f16, f32)
paged cache.

    python examples/tree_decode.py [model.gguf] [--kv q8|f16|f32] [--seqs 4] [--new 128]

The model is a LLaMA GGUF with f32 weights (a small synthetic one is written when none is
named); its projections are torch matrix products, and everything that touches the cache is
an operator of this library:

  rope_append      turns q and k, writes k and v, quantised as they are written
  attention_tree   every drafted node against the context and its own ancestors
  tree_accept      the longest drafted path that the model agrees with; its rows move up
  kv_read          a prompt's rows out of the cache, to start other sequences from them

Drafts come from the sequence itself: what followed earlier occurrences of its last tokens.
A step runs the model once over all nodes of all sequences, and yields one token a sequence
at least, as plain decoding does, and one more for each drafted node that was right.
"""
import argparse
import ctypes as C
import os
import sys
import tempfile
import time

import numpy as np
import torch
import torch.nn.functional as nnf

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import slate_b200 as sb  # noqa: E402

KV = {"f32": sb.KV_F32, "f16": sb.KV_F16, "q8": sb.KV_Q8}


def i32(a):
    return torch.as_tensor(np.asarray(a, np.int32)).cuda()


class Model:
    """The weights of an f32 LLaMA GGUF on the device."""

    def __init__(self, path):
        d = sb.LlamaDesc()
        h = sb.F["slate_gguf_model_open"](path.encode(), C.byref(d))
        if not h:
            raise OSError(f"{path}: {sb.last_error()}")
        for f in ("n_layers", "d_model", "ffn_hidden", "n_heads", "n_kv_heads", "head_dim", "max_seq", "vocab", "theta_base", "rms_eps"):
            setattr(self, f, getattr(d, f))

        def weight(at, *shape, dtype=0):
            if dtype != 0:
                raise ValueError(f"{path}: this example reads f32 weights")
            n = int(np.prod(shape))
            return torch.from_numpy(np.ctypeslib.as_array((C.c_float * n).from_address(at)).reshape(shape).copy()).cuda()

        D, F, kvd = d.d_model, d.ffn_hidden, d.n_kv_heads * d.head_dim
        self.embd = weight(d.token_embd, d.vocab, D, dtype=d.token_embd_dtype)
        self.norm = weight(d.output_norm, D)
        self.out = weight(d.output, d.vocab, D, dtype=d.output_dtype)
        self.layers = []
        for i in range(d.n_layers):
            x = d.layers[i].contents
            self.layers.append((
                weight(x.attn_norm, D),
                torch.cat([weight(x.attn_q, D, D, dtype=x.attn_q_dtype), weight(x.attn_k, kvd, D, dtype=x.attn_k_dtype),
                           weight(x.attn_v, kvd, D, dtype=x.attn_v_dtype)]),
                weight(x.attn_output, D, D, dtype=x.attn_output_dtype), weight(x.ffn_norm, D),
                weight(x.ffn_gate, F, D, dtype=x.ffn_gate_dtype), weight(x.ffn_up, F, D, dtype=x.ffn_up_dtype),
                weight(x.ffn_down, D, F, dtype=x.ffn_down_dtype)))
        sb.F["slate_gguf_model_close"](h)


class Decoder:
    """`seqs` sequences over a paged cache, each fed by step() with a tree of nodes."""

    def __init__(self, model, seqs, kv=sb.KV_Q8):
        m = self.m = model
        per = -(-m.max_seq // 16)
        # pages in no order, as an allocator would have handed them out
        self.table = i32(np.random.default_rng(0).permutation(seqs * per).reshape(seqs, per))
        self.pool = torch.zeros(sb.kv_pool_bytes(kv, seqs * per, m.n_layers, m.n_kv_heads, m.head_dim), dtype=torch.uint8, device="cuda")
        self.cache = sb.KVCache(pool=self.pool.data_ptr(), page_table=self.table.data_ptr(), n_pages=seqs * per, n_slots=seqs,
                                max_pages=per, n_layers=m.n_layers, n_kv_heads=m.n_kv_heads, head_dim=m.head_dim, kv_dtype=kv)
        cos, sin = sb.rope_tables(m.max_seq, m.head_dim, m.theta_base)
        self.tables = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
        self.rope = sb.Rope(cos=self.tables[0].data_ptr(), sin=self.tables[1].data_ptr(), n_pos=m.max_seq, rot_dim=m.head_dim,
                            layout=sb.ROPE_HALF)
        # one workspace for the largest step: calls on one stream take turns with it
        n = sb.attention_tree_workspace(self.cache, m.n_heads, seqs, seqs * sb.TREE_MAX_NODES, sb.TREE_MAX_NODES)
        self.ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        self.ctx = [0] * seqs

    def step(self, seqs, parents, tokens, given=False):
        """One pass over a tree of nodes for each of `seqs` (parents[i]: -1 or an earlier node;
        tokens[i]).  Returns per sequence the tokens that the model adds along the longest path of
        nodes it agrees with (`given`: of nodes as they stand); that path's rows stay in the cache."""
        m, stream = self.m, torch.cuda.current_stream().cuda_stream
        nodes = [len(p) for p in parents]
        depth = []
        for p in parents:
            for i, up in enumerate(p):
                depth.append(0 if up < 0 else depth[len(depth) - i + up] + 1)
        rows = sum(nodes)
        slot = i32(np.repeat(seqs, nodes))
        index = i32(np.concatenate([self.ctx[s] + np.arange(n) for s, n in zip(seqs, nodes)]))
        pos = i32(np.repeat([self.ctx[s] for s in seqs], nodes) + np.array(depth))
        off, of, ctx = i32(np.concatenate([[0], np.cumsum(nodes)])), i32(seqs), i32([self.ctx[s] for s in seqs])
        mask = torch.from_numpy(np.concatenate([sb.tree_masks(p) for p in parents]).view(np.int64)).cuda()
        tree = sb.TreeBatch(n_seq=len(seqs), rows=rows, max_nodes=max(nodes), row_off=off.data_ptr(), slot=of.data_ptr(),
                            ctx=ctx.data_ptr(), mask=mask.data_ptr())
        token = i32(np.concatenate(tokens))
        D, kvd = m.n_heads * m.head_dim, m.n_kv_heads * m.head_dim
        x, att = m.embd[token.long()], torch.empty(rows, D, device="cuda")
        for layer, (an, qkv, wo, fn, gate, up, down) in enumerate(m.layers):
            y = nnf.rms_norm(x, (m.d_model,), an, m.rms_eps) @ qkv.T           # [rows, q | k | v]
            p, ld = y.data_ptr(), D + 2 * kvd
            sb.rope_append(self.cache, layer, self.rope, rows, m.n_heads, p, ld, p, ld, p + 4 * D, ld, p + 4 * (D + kvd), ld,
                           slot.data_ptr(), index.data_ptr(), pos.data_ptr(), stream)
            sb.attention_tree(self.cache, layer, tree, m.n_heads, att.data_ptr(), D, p, ld, m.head_dim ** -0.5, self.ws.data_ptr(),
                              self.ws.numel(), stream)
            x = x + att @ wo.T
            y = nnf.rms_norm(x, (m.d_model,), fn, m.rms_eps)
            x = x + (nnf.silu(y @ gate.T) * (y @ up.T)) @ down.T
        target = (nnf.rms_norm(x, (m.d_model,), m.norm, m.rms_eps) @ m.out.T).argmax(1).int()
        parent = i32(np.full(rows, -1) if given else np.concatenate(parents))
        count = torch.empty(len(seqs), dtype=torch.int32, device="cuda")
        node, new = (torch.empty(len(seqs), sb.TREE_MAX_NODES, dtype=torch.int32, device="cuda") for _ in range(2))
        sb.tree_accept(self.cache, tree, parent.data_ptr(), token.data_ptr(), target.data_ptr(), count.data_ptr(), node.data_ptr(),
                       new.data_ptr(), stream)
        count, new = count.tolist(), new.tolist()
        for s, n in zip(seqs, count):
            self.ctx[s] += n
        return [row[:n] for row, n in zip(new, count)]

    def prompt(self, s, tokens):
        """Appends a prompt, up to 64 tokens a step, each following the one before.  Returns the
        token after it."""
        for i in range(0, len(tokens), sb.TREE_MAX_NODES):
            part = tokens[i:i + sb.TREE_MAX_NODES]
            new, = self.step([s], [np.arange(len(part)) - 1], [part], given=True)
        return new[-1]

    def save(self, s):
        """The sequence's rows, K and V [n_layers, n, n_kv_heads * head_dim] f32."""
        m, n = self.m, self.ctx[s]
        K = torch.empty(m.n_layers, n, m.n_kv_heads * m.head_dim, device="cuda")
        V = torch.empty_like(K)
        slot, index = i32([s] * n), i32(np.arange(n))
        sb.kv_read(self.cache, 0, m.n_layers, n, slot.data_ptr(), index.data_ptr(), K.data_ptr(), V.data_ptr(), sb.KV_F32,
                   torch.cuda.current_stream().cuda_stream)
        return K, V

    def load(self, s, K, V):
        """Rows that save() returned into sequence s.  They are turned already: position 0."""
        m, n = self.m, K.shape[1]
        slot, index, pos = i32([s] * n), i32(np.arange(n)), i32(np.zeros(n))
        kvd = m.n_kv_heads * m.head_dim
        q = torch.empty(n, kvd, device="cuda")       # (the query is not needed: k stands in for it)
        for layer in range(m.n_layers):
            sb.rope_append(self.cache, layer, self.rope, n, m.n_kv_heads, q.data_ptr(), kvd, K[layer].data_ptr(), kvd,
                           K[layer].data_ptr(), kvd, V[layer].data_ptr(), kvd, slot.data_ptr(), index.data_ptr(), pos.data_ptr(),
                           torch.cuda.current_stream().cuda_stream)
        self.ctx[s] = n


def draft(text, most=sb.TREE_MAX_NODES, depth=12, branches=6):
    """(parents, tokens) of a tree over the last token of `text`: what followed the latest
    occurrences of its last two tokens (or one), merged where they begin alike."""
    parents, tokens, child = [-1], [text[-1]], {}
    for n in (2, 1):
        tail, found = text[-n:], 0
        for i in range(len(text) - n - 1, -1, -1):
            if found == branches or len(tokens) == most:
                break
            if text[i:i + n] != tail:
                continue
            found += 1
            at = 0
            for t in text[i + n:i + n + depth]:
                if (at, t) not in child and len(tokens) < most:
                    child[at, t] = len(tokens)
                    parents.append(at)
                    tokens.append(t)
                if (at, t) not in child:
                    break
                at = child[at, t]
        if found:
            break
    return np.array(parents), tokens


def generate(dec, texts, new, trees=True):
    """Extends each text (its last token not in the cache yet) by `new` tokens; returns the steps taken."""
    ends, steps = [len(t) + new for t in texts], 0
    while True:
        live = [s for s, t in enumerate(texts) if len(t) < ends[s]]
        if not live:
            return steps
        # a node beyond the wanted length would be thrown away
        trees_ = [draft(texts[s], depth=min(12, ends[s] - len(texts[s]) - 1)) if trees else (np.array([-1]), texts[s][-1:]) for s in live]
        for s, more in zip(live, dec.step(live, [p for p, _ in trees_], [t for _, t in trees_])):
            texts[s] += more
        steps += 1


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("model", nargs="?")
    ap.add_argument("--kv", choices=KV, default="q8")
    ap.add_argument("--seqs", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=200)
    ap.add_argument("--new", type=int, default=128)
    a = ap.parse_args()
    with tempfile.TemporaryDirectory() as tmp:
        if not a.model:
            a.model = os.path.join(tmp, "synthetic.gguf")
            sb.synth_gguf(a.model, n_layers=4, d_model=512, ffn_hidden=1024, n_heads=8, n_kv_heads=2, vocab=1000, max_seq=2048, q4k=False)
        model = Model(a.model)
    prompt = np.random.default_rng(1).integers(0, model.vocab, a.prompt).tolist()
    out = {}
    for trees in (False, True, False, True):         # the first two warm up
        dec = Decoder(model, a.seqs, KV[a.kv])
        first = dec.prompt(0, prompt)
        K, V = dec.save(0)
        for s in range(1, a.seqs):                    # the others begin from the same prompt's rows
            dec.load(s, K, V)
        # ... and go on with another token each
        texts = [prompt + [first if s == 0 else (first + 17 * s) % model.vocab] for s in range(a.seqs)]
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        steps = generate(dec, texts, a.new, trees)
        torch.cuda.synchronize()
        out[trees] = texts, steps, time.perf_counter() - t0
    for trees, name in ((False, "one token a step"), (True, "trees")):
        texts, steps, sec = out[trees]
        n = a.seqs * a.new
        print(f"{name}: {n} tokens in {steps} steps, {n / steps / a.seqs:.2f} tokens a sequence and step, {sec / steps * 1e3:.2f} ms a step, "
              f"{n / sec:.0f} tokens/s")
    same = sum(x == y for t, u in zip(out[False][0], out[True][0]) for x, y in zip(t[a.prompt:], u[a.prompt:]))
    print(f"equal tokens: {same} of {a.seqs * (a.new + 1)}")


if __name__ == "__main__":
    main()
