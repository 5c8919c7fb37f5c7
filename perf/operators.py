"""Workloads of the KV-cache row operators and of attention over a tree of drafted tokens.

A cache layer holds K and V rows [positions, n_kv_heads, head_dim], as f16 or as
int8 with one f32 scale per position and head (value = int8 x scale).  A
sequence owns consecutive rows from `starts[b]`: `lens[b]` rows of context,
then one row per drafted token of the step (its node j sits at row
starts + lens + j).

  store   quantise rows into an int8 cache as they are written, and read them back
  read    read rows back by index, as f32 or f16
  move    close the accepted branch of each drafted tree up behind the context
  attend  attention of every drafted token over its context and its ancestors;
          one node per sequence is plain single-token decode

`run` computes them in elementary torch operations, or with the library's
kernels where `own` is true.
"""
import math

import torch

own = False


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one decoded token of a 0.5B-size model enters its cache: pure latency
        {"name": "store one token", "op": "store", "n": 1, "n_kv": 2, "hd": 64, "positions": 2303, "src": "f32"},
        # a batch prefill of 2048 tokens of an 8B-size model
        {"name": "store a prompt", "op": "store", "n": 2048, "n_kv": 8, "hd": 128, "positions": 4096, "src": "f32"},
        # an f16 cache of several long sequences turned into an int8 one, odd row count
        {"name": "store many prompts", "op": "store", "n": 40961, "n_kv": 8, "hd": 128, "positions": 65536, "src": "f16"},
        # a shared prefix of 777 scattered rows read back for a check or a hand-over
        {"name": "read a prefix", "op": "read", "n": 777, "n_kv": 2, "hd": 64, "positions": 4096, "dst": "f32"},
        # a whole long cache turned back into f16 rows
        {"name": "read a long cache", "op": "read", "n": 32768, "n_kv": 8, "hd": 128, "positions": 32768, "dst": "f16"},
        # one sequence's accepted branch of an eight-token tree
        {"name": "move one branch", "op": "move", "kind": "q8", "n_seq": 1, "ctx": 1024, "nodes": 8, "n_kv": 2, "hd": 64},
        # the accepted branches of a batch, 64 drafted tokens each, over an f16 cache
        {"name": "move a batch of branches", "op": "move", "kind": "f16", "n_seq": 128, "ctx": 333, "nodes": 64, "n_kv": 8, "hd": 128},
        # single-token decode at a short context: latency
        {"name": "decode, short", "op": "attend", "kind": "q8", "n_seq": 1, "ctx": 255, "nodes": 1, "n_heads": 14, "n_kv": 2, "hd": 64, "tree": False},
        # 16 sequences, one token each, ragged contexts up to 4096
        {"name": "decode, 16 sequences", "op": "attend", "kind": "q8", "n_seq": 16, "ctx": 4095, "nodes": 1, "n_heads": 32, "n_kv": 8, "hd": 128, "tree": False},
        # one sequence at a very long context: the cache's bytes
        {"name": "decode, long", "op": "attend", "kind": "q8", "n_seq": 1, "ctx": 131000, "nodes": 1, "n_heads": 32, "n_kv": 8, "hd": 128, "tree": False},
        # one sequence verifies a 16-token tree over the model's f16 cache
        {"name": "tree, one sequence", "op": "attend", "kind": "f16", "n_seq": 1, "ctx": 4096, "nodes": 16, "n_heads": 32, "n_kv": 8, "hd": 128, "tree": True},
        # a batch verifies trees of up to 60 tokens over int8 caches
        {"name": "tree, batch", "op": "attend", "kind": "q8", "n_seq": 24, "ctx": 6001, "nodes": 60, "n_heads": 32, "n_kv": 8, "hd": 128, "tree": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    # head layouts: this repository's model shapes and their kin
    n_heads, n_kv, hd = rng.choice([(14, 2, 64), (32, 8, 128), (32, 4, 128), (12, 2, 128), (6, 6, 48), (9, 3, 96)])
    op = rng.choice(["store", "read", "move", "attend", "attend", "attend"])
    if op in ("store", "read"):
        n = _log_int(rng, 1, 30000)
        way = {"src" if op == "store" else "dst": rng.choice(["f32", "f16"])}
        return {"op": op, "n": n, "n_kv": n_kv, "hd": hd, "positions": n + _log_int(rng, 1, 8000), **way}
    kind = rng.choice(["q8", "f16"])
    if op == "move":
        return {"op": op, "kind": kind, "n_seq": _log_int(rng, 1, 128), "ctx": _log_int(rng, 1, 2000), "nodes": rng.randint(2, 64), "n_kv": n_kv, "hd": hd}
    nodes = rng.choice([1, 1, rng.randint(2, 8), rng.randint(9, 60)])
    ctx = _log_int(rng, 1, 100000)
    n_seq = _log_int(rng, 1, max(1, min(64, 120000 // (ctx + nodes))))
    return {"op": op, "kind": kind, "n_seq": n_seq, "ctx": ctx, "nodes": nodes, "n_heads": n_heads, "n_kv": n_kv, "hd": hd,
            "tree": nodes > 1 and rng.random() < 0.8}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _kv_rows(shape, g):
    """K or V rows as a model makes them: normal values on a per-channel offset, rows of differing size."""
    x = torch.randn(shape, generator=g, device="cuda")
    x = x + torch.randn(shape[1:], generator=g, device="cuda") * 0.5
    return x * torch.exp(torch.randn(shape[:2] + (1,), generator=g, device="cuda") * 0.3)


def _cache(kind, positions, n_kv, hd, g):
    """One layer's cache tensors, every row holding values."""
    k, v = _kv_rows((positions, n_kv, hd), g), _kv_rows((positions, n_kv, hd), g)
    if kind == "f16":
        return {"k": k.half(), "v": v.half(), "k_scale": None, "v_scale": None}
    ks, vs = k.abs().amax(-1) / 127, v.abs().amax(-1) / 127
    k, v = torch.round(k / ks[..., None]).to(torch.int8), torch.round(v / vs[..., None]).to(torch.int8)
    # scales lie head by head: shape [positions, n_kv], a head's positions next to each other
    return {"k": k, "v": v, "k_scale": ks.t().contiguous().t(), "v_scale": vs.t().contiguous().t()}


def _lens(case, g):
    """Contexts of a batch: the longest, then between a quarter of it and it."""
    n, ctx = case["n_seq"], case["ctx"]
    lens = (ctx * (0.25 + 0.75 * torch.rand(n, generator=g, device="cuda"))).int()
    lens[0] = ctx
    return lens


def _trees(n_seq, nodes, tree, g):
    """parents [n_seq, nodes] (-1: the root) and ancestor-or-self sets [n_seq, nodes, nodes]."""
    j = torch.arange(nodes, device="cuda")
    up = torch.rand(n_seq, nodes, generator=g, device="cuda") ** 0.5 if tree else torch.ones(n_seq, nodes, device="cuda")
    parents = torch.minimum((up * j).long(), j - 1)  # a tree that tends to be deep, or a chain
    see = torch.eye(nodes, device="cuda").expand(n_seq, -1, -1).clone()
    for i in range(1, nodes):  # a parent comes before its children
        see[:, i] += see[torch.arange(n_seq, device="cuda"), parents[:, i]]
    return parents, see > 0


def prepare(case, seed):
    g = _gen(seed)
    op, s = case["op"], {"case": case}
    if op == "store":
        s.update(_cache("q8", case["positions"], case["n_kv"], case["hd"], g))
        dt = torch.float32 if case["src"] == "f32" else torch.float16
        shape = (case["n"], case["n_kv"], case["hd"])
        s["new_k"], s["new_v"] = _kv_rows(shape, g).to(dt), _kv_rows(shape, g).to(dt)
        first = (case["positions"] - case["n"]) // 2
        s["rows"] = first + torch.arange(case["n"], device="cuda", dtype=torch.int32)
        return s
    if op == "read":
        s.update(_cache("q8", case["positions"], case["n_kv"], case["hd"], g))
        s["rows"] = torch.randperm(case["positions"], generator=g, device="cuda")[: case["n"]].int()
        return s
    n_seq, nodes = case["n_seq"], case["nodes"]
    lens = _lens(case, g)
    room = lens + nodes + 17  # each sequence's rows, some of them not in use yet
    starts = (torch.cumsum(room, 0) - room).int()
    positions = n_seq * (case["ctx"] + nodes + 17)
    s.update(_cache(case["kind"], positions, case["n_kv"], case["hd"], g))
    s["starts"], s["lens"] = starts, lens
    parents, see = _trees(n_seq, nodes, case.get("tree", True), g)
    if op == "move":
        # the accepted branch: a random node and its ancestors, in order
        leaf = torch.randint(0, nodes, (n_seq,), generator=g, device="cuda")
        on = see[torch.arange(n_seq, device="cuda"), leaf]
        s["counts"] = on.sum(1).int()
        s["path"] = torch.sort(torch.where(on, torch.arange(nodes, device="cuda"), nodes), dim=1)[0].int() % nodes
        return s
    s["q"] = torch.randn(n_seq * nodes, case["n_heads"] * case["hd"], generator=g, device="cuda") * 1.5
    s["offsets"] = torch.arange(n_seq + 1, device="cuda", dtype=torch.int32) * nodes
    bits = see.long() << torch.arange(nodes, device="cuda")
    s["masks"] = bits.sum(2).reshape(-1) if case["tree"] else None
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    case = s["case"]
    if own:
        from prana_b200 import kernels as K

        cache = K.KvRows(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if case["op"] == "store":
            K.kv_rows_write(cache, s["rows"], s["new_k"], s["new_v"])
            return K.kv_rows_read(cache, s["rows"])
        if case["op"] == "read":
            return K.kv_rows_read(cache, s["rows"], torch.float32 if case["dst"] == "f32" else torch.float16)
        if case["op"] == "move":
            K.kv_rows_move(cache, s["starts"], s["lens"], s["path"], s["counts"])
            return s["k"], s["v"], s["k_scale"], s["v_scale"]
        return K.attention_tree(s["q"], cache, s["starts"], s["lens"], s["offsets"], case["nodes"], case["n_heads"], s["masks"])
    if case["op"] == "store":
        _plain_write(s["k"], s["k_scale"], s["rows"].long(), s["new_k"].float())
        _plain_write(s["v"], s["v_scale"], s["rows"].long(), s["new_v"].float())
        return _plain_values(s["k"], s["k_scale"], s["rows"]), _plain_values(s["v"], s["v_scale"], s["rows"])
    if case["op"] == "read":
        dt = torch.float32 if case["dst"] == "f32" else torch.float16
        return _plain_values(s["k"], s["k_scale"], s["rows"]).to(dt), _plain_values(s["v"], s["v_scale"], s["rows"]).to(dt)
    if case["op"] == "move":
        return tuple(_plain_move(s, s[name]) for name in ("k", "v", "k_scale", "v_scale"))
    return _plain_attend(s, case)


def _plain_write(x, scale, rows, new):
    amax = new.abs().amax(-1)
    sc = amax / torch.full_like(amax, 127)
    sc = torch.where(amax > 0, sc, torch.ones_like(sc))
    t = new * (torch.ones_like(sc) / sc)[..., None]
    t = torch.copysign(torch.floor(t.abs() + 0.5), t)  # to the nearest, halves away from zero
    x[rows] = t.clamp(-127, 127).to(torch.int8)
    scale[rows] = sc


def _plain_values(x, scale, rows):
    x = x[rows].float()
    return x if scale is None else x * scale[rows][..., None]


def _plain_move(s, x):
    if x is None:
        return None
    i = torch.arange(s["path"].shape[1], device=x.device)
    base = (s["starts"] + s["lens"]).long()[:, None]
    use = i < s["counts"][:, None]
    x[(base + i)[use]] = x[(base + s["path"].long())[use]]
    return x


def _plain_attend(s, case):
    n_seq, nodes, nh, nkv, hd = case["n_seq"], case["nodes"], case["n_heads"], case["n_kv"], case["hd"]
    # whole stretches of 512 places, summed one by one and then together: one f32 sum over a long context would lose digits
    lens, total = s["lens"].long(), (case["ctx"] + nodes + 511) // 512 * 512
    at = torch.arange(total, device="cuda")
    rows = (s["starts"].long()[:, None] + at).clamp(max=s["k"].shape[0] - 1)
    node = at - lens[:, None]  # which drafted token sits at this place, if one does
    there = (node < nodes)[:, None, :, None]
    k = _plain_values(s["k"], s["k_scale"], rows).transpose(1, 2).masked_fill(~there, 0)
    v = _plain_values(s["v"], s["v_scale"], rows).transpose(1, 2).masked_fill(~there, 0)
    i = torch.arange(nodes, device="cuda")
    see = (i[None, :, None] >= node[:, None]) if s["masks"] is None else ((s["masks"].view(n_seq, nodes, 1) >> node.clamp(0, 63)[:, None]) & 1).bool()
    see = ((node < 0)[:, None] | (see & (node < nodes)[:, None]))[:, None, :, None]  # [seq, 1, nodes, 1, total]
    q = s["q"].view(n_seq, nodes, nkv, nh // nkv, hd).permute(0, 2, 1, 3, 4)
    sc = torch.matmul(q.reshape(n_seq, nkv, -1, hd), k.transpose(2, 3)) / math.sqrt(hd)
    sc = sc.view(n_seq, nkv, nodes, nh // nkv, total).masked_fill(~see, -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isfinite(top), top, 0))
    sums = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n_seq, nkv, -1, total // 512, 512).transpose(2, 3), v.reshape(n_seq, nkv, -1, 512, hd)).sum(2)
    o = o.view(n_seq, nkv, nodes, nh // nkv, hd)
    o = torch.where(sums > 0, o / sums, 0)
    return o.permute(0, 2, 1, 3, 4).reshape(n_seq * nodes, nh * hd)


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "move":
        return None  # rows are copied: nothing is computed
    rows = s.get("rows")
    if case["op"] == "read":
        i = rows.long()
        return tuple(s[n].index_select(0, i).double().mul(s[n + "_scale"].index_select(0, i).double().unsqueeze(2)) for n in ("k", "v"))
    if case["op"] == "store":
        out = []
        for new in (s["new_k"], s["new_v"]):
            x = new.double()
            step = (x.abs().max(dim=2, keepdim=True).values / 127).float()  # the scale is held in f32, and its inverse taken there
            out.append(step.double() * (torch.sign(x) * torch.floor(x.abs() * step.reciprocal().double() + 0.5)))
        return tuple(out)
    nh, nkv, hd, nodes = case["n_heads"], case["n_kv"], case["hd"], case["nodes"]
    q, out = s["q"].double().view(case["n_seq"], nodes, nh, hd), []
    for b, (start, n) in enumerate(zip(s["starts"].tolist(), s["lens"].tolist())):
        end = start + n + nodes
        k, v = s["k"][start:end].double(), s["v"][start:end].double()
        if s["k_scale"] is not None:
            k, v = k * s["k_scale"][start:end, :, None].double(), v * s["v_scale"][start:end, :, None].double()
        see = torch.ones(nodes, n + nodes, dtype=torch.bool, device="cuda")
        for i in range(nodes):
            mask = (2 << i) - 1 if s["masks"] is None else int(s["masks"][b * nodes + i]) & (2 ** 64 - 1)
            see[i, n:] = torch.tensor([bool(mask >> j & 1) for j in range(nodes)], device="cuda")
        o = torch.empty(nodes, nh, hd, dtype=torch.float64, device="cuda")
        for h in range(nh):
            c = h // (nh // nkv)
            w = torch.where(see, q[b, :, h] @ k[:, c].t() / hd ** 0.5, -math.inf)
            o[:, h] = torch.softmax(w, dim=1) @ v[:, c]
        out.append(o.view(nodes, nh * hd))
    return torch.cat(out)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op, n_kv, hd = case["op"], case["n_kv"], case["hd"]
    if op in ("store", "read"):
        n = case["n"] * n_kv
        row_q8 = 2 * (hd + 4)  # K and V: int8 values and a scale
        wide = 2 * hd * (4 if case.get("src", case.get("dst")) == "f32" else 2)
        if op == "read":
            return {"bytes": n * (row_q8 + wide) + 4 * case["n"], "flops": n * 2 * hd}
        # the rows in, the int8 rows out; then those in and the f32 values out
        return {"bytes": n * (wide + 2 * row_q8 + 2 * hd * 4) + 8 * case["n"], "flops": n * 2 * hd * 5}
    n_seq, nodes = case["n_seq"], case["nodes"]
    row = n_kv * 2 * (hd + 4 if case["kind"] == "q8" else 2 * hd)
    if op == "move":  # about half of the nodes lie on the accepted branch
        return {"bytes": n_seq * (2 * row * max(1, nodes // 2) + 4 * nodes + 12), "flops": 0}
    total = case["ctx"] + (n_seq - 1) * 0.625 * case["ctx"] + n_seq * nodes  # contexts spread from a quarter to all
    q_out = 2 * 4 * n_seq * nodes * case["n_heads"] * hd
    return {"bytes": total * row + q_out + 12 * n_seq + 8 * n_seq * nodes, "flops": 4 * nodes * case["n_heads"] * hd * total}
