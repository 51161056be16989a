"""Measured cases of the operators that search over continuations on the KV ring.

    tree_attend   attention of a tree of drafted tokens over a stream's ring and the tree's own rows
    tree_commit   the accepted path of such a tree written into the rings of several layers
    beam_select   one beam-search step: the best continuations over beams and codes
    ring_reorder  the rings of a beam group permuted to the selected parents, in place

`run` computes them with elementary torch operations, or, where `own` is true, with the calls a user makes of
this package.  `exact` computes the same outputs from the definitions in 64 bits.

A ring holds kv[layer][stream][K|V][head][slot][64] and slot_pos[layer][stream][slot] (-1: empty); the position p
lives in slot p % capacity.  A drafted node's parent is an earlier node of its tree, -1 (it follows the ring's last
position) or -2 (absent: padding, its output row is not written).
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HD = 64
THETA = 10000.0


# ---------------------------------------------------------------- cases

def _tree(name, n, heads, nodes, capacity, lo, hi, dtype, wrap, ragged):
    return {"name": name, "op": "tree_attend", "n": n, "heads": heads, "nodes": nodes, "capacity": capacity, "lo": lo,
            "hi": hi, "dtype": dtype, "wrap": wrap, "ragged": ragged}


def _commit(name, layers, n, heads, nodes, capacity, lo, hi, dtype, wrap):
    return {"name": name, "op": "tree_commit", "layers": layers, "n": n, "heads": heads, "nodes": nodes,
            "capacity": capacity, "lo": lo, "hi": hi, "dtype": dtype, "wrap": wrap}


def _beam(name, groups, beams, codes, stride, dtype, first, end, penalty):
    return {"name": name, "op": "beam_select", "groups": groups, "beams": beams, "codes": codes, "stride": stride,
            "dtype": dtype, "first": first, "end": end, "penalty": penalty}


def _reorder(name, layers, groups, beams, heads, capacity, lo, hi, dtype):
    return {"name": name, "op": "ring_reorder", "layers": layers, "groups": groups, "beams": beams, "heads": heads,
            "capacity": capacity, "lo": lo, "hi": hi, "dtype": dtype}


def listed():
    return [
        # one utterance on the engine's global ring (570 slots, 300 filled), eight drafted frames: latency
        _tree("tree one stream f32", 1, 12, 8, 570, 300, 300, "f32", False, False),
        # 64 streams on 512-slot fp32 rings, past the wrap or not, five drafted frames each
        _tree("tree 64 streams f32", 64, 12, 5, 512, 100, 1500, "f32", True, False),
        # 64 streams on long bf16 rings, ragged lengths, trees of up to 16 nodes with padding
        _tree("tree 64 streams bf16", 64, 12, 16, 4096, 1, 6000, "bf16", True, True),
        # a few streams with wide trees over fp16 rings
        _tree("tree wide f16", 16, 12, 64, 2048, 500, 2000, "f16", True, False),
        # the accepted frames of one utterance into its 12 layers
        _commit("commit one stream f32", 12, 1, 12, 8, 570, 300, 300, "f32", False),
        # the accepted frames of 64 streams, some across the wrap
        _commit("commit 64 streams bf16", 12, 64, 12, 16, 256, 10, 700, "bf16", True),
        # the first step of one utterance: an audio codebook, one live beam of four
        _beam("beam one utterance f32", 1, 4, 1024, 1024, "f32", True, -1, 1.0),
        # 64 utterances over an audio codebook with the repetition penalty
        _beam("beam 64 penalty f32", 64, 8, 1024, 1024, "f32", False, 7, 1.2),
        # a text vocabulary of odd size in padded bf16 rows, some beams finished
        _beam("beam vocabulary bf16", 32, 8, 50021, 50048, "bf16", False, 2, 1.0),
        # the largest vocabulary and beam count
        _beam("beam vocabulary f32", 16, 16, 131071, 131071, "f32", False, -1, 1.0),
        # four beams of one utterance on the engine's global ring
        _reorder("reorder one utterance f32", 12, 1, 4, 12, 570, 300, 300, "f32"),
        # eight utterances of eight beams on 1024-slot bf16 rings, past the wrap or not
        _reorder("reorder 8 groups bf16", 12, 8, 8, 12, 1024, 300, 3000, "bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree_attend", "tree_attend", "tree_commit", "beam_select", "beam_select", "ring_reorder"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "beam_select":
        codes = _log(rng, 64, 131071)
        beams = rng.randint(1, 16)
        groups = _log(rng, 1, max(1, min(64, 16 * 16 * 131071 // (beams * codes))))
        penalty = 1.0
        if codes <= 4096 and rng.random() < 0.5:
            codes, penalty = 32 * max(1, codes // 32), round(rng.uniform(1.05, 1.6), 2)
        stride = codes + rng.choice([0, 0, 1, 5, 64])
        end = rng.choice([-1, rng.randrange(codes)])
        c = _beam("", groups, beams, codes, stride, dtype, rng.random() < 0.2, end, penalty)
    else:
        heads = rng.choice([1, 4, 8, 12, 16])
        wrap = op == "ring_reorder" or rng.random() < 0.6
        capacity = _log(rng, 17, 4096)
        nodes = _log(rng, 1, 64)
        if not wrap:
            capacity = max(capacity, nodes + 2)
        top = 2 * capacity if wrap else capacity - nodes
        a, b = sorted((rng.randint(0, top), rng.randint(0, top)))
        size = 12 * 64 * 4096 // (heads * capacity)
        if op == "tree_attend":
            n = _log(rng, 1, max(1, min(64, size)))
            c = _tree("", n, heads, nodes, capacity, a, b, dtype, wrap, rng.random() < 0.4)
        elif op == "tree_commit":
            layers = rng.randint(1, 12)
            n = _log(rng, 1, max(1, min(64, size // (4 * layers))))
            c = _commit("", layers, n, heads, nodes, capacity, a, b, dtype, wrap)
        else:
            layers, beams = rng.randint(1, 12), rng.randint(1, 16)
            groups = _log(rng, 1, max(1, min(16, 2 * size // (4 * layers * beams))))
            c = _reorder("", layers, groups, beams, heads, capacity, a, b, dtype)
    c.pop("name")
    return c


# ---------------------------------------------------------------- inputs

def _positions(c, n):
    """One position per item, spread evenly over [lo, hi] in a mixed order."""
    at = [c["lo"] + (c["hi"] - c["lo"]) * i // max(1, n - 1) for i in range(n)]
    random.Random(n).shuffle(at)
    return at


def _counts(c, n):
    """Nodes present in each item's tree."""
    t = c["nodes"]
    return [max(1, t - (i * 5) % (t // 2 + 1)) if c.get("ragged") else t for i in range(n)]


def _accepted(c, n):
    """Length of each item's accepted path: none, some or all of its drafts."""
    return [min((i * 3 + 4) % (c["nodes"] + 1), c["capacity"]) for i in range(n)]


def _trees(n, nodes, counts, chains, r):
    """parents[n][nodes]: the first chains[i] nodes of item i follow one another, the others hang anywhere."""
    return [[-2 if t >= counts[i] else t - 1 if t < chains[i] else r.randrange(-1, t) for t in range(nodes)]
            for i in range(n)]


def _filled(layers, streams, heads, capacity, positions, dtype, g):
    """Rings that hold the last `capacity` positions below each stream's position."""
    kv = torch.empty(layers, streams, 2, heads, capacity, HD, dtype=DTYPES[dtype], device="cuda")
    kv.normal_(generator=g)
    p = torch.tensor(positions, dtype=torch.int64, device="cuda")[:, None] - 1
    j = torch.arange(capacity, device="cuda")[None, :]
    sp = p - (p - j) % capacity
    sp = torch.where((p >= 0) & (sp >= 0), sp, -1).to(torch.int32)
    return kv, sp[None].expand(layers, -1, -1).contiguous()


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _inputs(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = random.Random(seed)
    if c["op"] == "beam_select":
        G, B, V = c["groups"], c["beams"], c["codes"]
        rows = torch.empty(G, B, c["stride"], device="cuda").normal_(generator=g).mul_(3.0).to(DTYPES[c["dtype"]])
        s = {"logits": rows[:, :, :V], "scores": -20.0 * torch.rand(G, B, device="cuda", generator=g)}
        if c["first"]:
            s["scores"][:, 1:] = -math.inf
            s["scores"][:, 0] = 0.0
        s["finished"] = s["seen"] = None
        if c["end"] >= 0:
            s["finished"] = (torch.rand(G, B, device="cuda", generator=g) < (0.0 if c["first"] else 0.2)).to(torch.int32)
        if c["penalty"] != 1.0:
            s["penalty"] = torch.tensor(c["penalty"], device="cuda")
            bits = (torch.rand(G, B, V // 32, 32, device="cuda", generator=g) < 0.1).to(torch.int64)
            words = (bits << torch.arange(32, device="cuda")).sum(-1)
            s["seen"] = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
        return s
    H = c["heads"]
    if c["op"] == "ring_reorder":
        G, B = c["groups"], c["beams"]
        at = [p for p in _positions(c, G) for _ in range(B)]
        kv, sp = _filled(c["layers"], G * B, H, c["capacity"], at, c["dtype"], g)
        ids = list(range(G * B))
        r.shuffle(ids)
        sp = sp[:, torch.argsort(torch.tensor(ids, device="cuda"))].contiguous()  # entry k is stream ids[k]
        return {"kv": kv, "slot_pos": sp, "streams": _ints(ids).view(G, B),
                "parents": _ints([r.randrange(B) for _ in range(G * B)]).view(G, B), "last": max(at)}
    n, T, L = c["n"], c["nodes"], c.get("layers", 1)
    at = _positions(c, n)
    counts = _counts(c, n)
    took = _accepted(c, n) if c["op"] == "tree_commit" else [r.randrange(counts[i] + 1) for i in range(n)]
    ids = list(range(n))
    r.shuffle(ids)  # item i is on stream ids[i]
    by_stream = [0] * n
    for i in range(n):
        by_stream[ids[i]] = at[i]
    kv, sp = _filled(L, n, H, c["capacity"], by_stream, c["dtype"], g)
    s = {"kv": kv, "slot_pos": sp, "streams": _ints(ids), "positions": _ints(at),
         "parents": _ints(_trees(n, T, counts, took, r)), "last": max(at) + T,
         "qkv": torch.empty(L, n, T, 3 * H * HD, device="cuda").normal_(generator=g)}
    if c["op"] == "tree_attend":
        s["qkv"] = s["qkv"][0]
        s["out"] = torch.zeros(n, T, H * HD, device="cuda")
    else:
        s["leaves"] = _ints([a - 1 for a in took])
        s["next"] = torch.zeros(n, dtype=torch.int32, device="cuda")
    return s


class _View:
    """A ring's device memory for torch, which keeps the ring alive as long as the tensor."""

    def __init__(self, ring, address, shape, kind):
        self.ring = ring
        self.__cuda_array_interface__ = {"data": (address, False), "shape": shape, "typestr": kind, "version": 3}


def prepare(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    s["case"] = c
    if c["op"] == "beam_select" or not own:
        return s
    # the ring is the handle that a program keeps: made once, then filled with the state drawn above
    from mockbird_b200 import KvRing

    L, S, _, H, C, _ = s["kv"].shape
    ring = KvRing(layers=L, heads=H, capacity=C, streams=S, dtype=c["dtype"], wrap=c.get("wrap", True),
                  max_position=s["last"] + 1)
    info = ring.info
    kind = {"f32": "<f4", "bf16": "<i2", "f16": "<f2"}[c["dtype"]]
    kv = torch.as_tensor(_View(ring, info.kv, (L, S, 2, H, C, HD), kind), device="cuda").view(DTYPES[c["dtype"]])
    sp = torch.as_tensor(_View(ring, info.slot_pos, (L, S, C), "<i4"), device="cuda")
    kv.copy_(s["kv"])
    sp.copy_(s["slot_pos"])
    s["ring"], s["kv"], s["slot_pos"] = ring, kv, sp
    return s


# ---------------------------------------------------------------- one pass

def _rope(x, pos):
    """x [..., 64] fp32 at positions pos (broadcast over the leading axes): interleaved pairs, angles in 64 bits."""
    inv = THETA ** (-torch.arange(0, HD, 2, dtype=torch.float64, device=x.device) / HD)
    a = pos.to(torch.float64)[..., None] * inv
    cos, sin = a.cos().float(), a.sin().float()
    u, v = x[..., 0::2], x[..., 1::2]
    return torch.stack((u * cos - v * sin, v * cos + u * sin), -1).flatten(-2)


def _ancestors(parents):
    """reach [n][T][T]: whether node j lies on the path from the root to node t, t itself included."""
    n, T = parents.shape
    j = torch.arange(T, device=parents.device)
    step = (parents[:, :, None] == j).float() + torch.eye(T, device=parents.device)
    return (torch.matrix_power(step, max(1, T)) > 0.5) & (parents != -2)[:, :, None]


def _tree_attend(s):
    c = s["case"]
    n, T, H, C = c["n"], c["nodes"], c["heads"], c["capacity"]
    store = DTYPES[c["dtype"]]
    reach = _ancestors(s["parents"])
    present = s["parents"] != -2
    depth = reach.sum(-1) - 1
    pos = torch.where(present, s["positions"][:, None] + depth, 0)
    q, k, v = s["qkv"].view(n, T, 3, H, HD).permute(2, 0, 3, 1, 4)  # each [n][H][T][64]
    q = _rope(q, pos[:, None])
    k = _rope(k, pos[:, None]).to(store).float()
    v = v.to(store).float()
    ids = s["streams"].long()
    rk, rv = s["kv"][0, ids, 0].float(), s["kv"][0, ids, 1].float()
    sp = s["slot_pos"][0, ids][:, None, :]  # [n][1][C]
    seen = (sp >= 0) & (sp < s["positions"][:, None, None]) & (pos[:, :, None] - sp < C)
    own_ = reach & (depth[:, :, None] - depth[:, None, :] < C)
    score = torch.cat((q @ rk.transpose(-1, -2), q @ k.transpose(-1, -2)), -1) * 0.125
    mask = torch.cat((seen, own_), -1)[:, None]
    score = torch.where(mask, score, -math.inf)
    w = torch.exp(score - score.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = w[..., :C] @ rv + w[..., C:] @ v
    o = o.permute(0, 2, 1, 3).reshape(n, T, H * HD)
    s["out"].copy_(torch.where(present[:, :, None], o, s["out"]))
    return s["out"]


def _tree_commit(s):
    c = s["case"]
    L, n, T, H, C = c["layers"], c["n"], c["nodes"], c["heads"], c["capacity"]
    reach = _ancestors(s["parents"])
    depth = reach.sum(-1) - 1
    pos = s["positions"][:, None] + depth
    leaf = s["leaves"].long()
    took = reach[torch.arange(n, device="cuda"), leaf.clamp_min(0)] & (leaf >= 0)[:, None]  # [n][T]
    length = took.sum(-1)
    took = took & (length[:, None] - depth <= C)
    i, t = took.nonzero(as_tuple=True)
    stream, p = s["streams"].long()[i], pos[i, t]
    rows = s["qkv"].view(L, n, T, 3, H, HD)[:, i, t]  # [L][m][3][H][64]
    kv = torch.stack((_rope(rows[:, :, 1], p[:, None]), rows[:, :, 2]), 2).to(DTYPES[c["dtype"]])
    s["kv"][:, stream, :, :, p % C] = kv.transpose(0, 1)
    s["slot_pos"][:, stream, p % C] = p.to(torch.int32)
    s["next"].copy_(s["positions"] + length)
    return [s["kv"], s["slot_pos"], s["next"]]


def _beam_select(s):
    c = s["case"]
    G, B, V = c["groups"], c["beams"], c["codes"]
    x = s["logits"].float()
    if s["seen"] is not None:
        bit = (s["seen"][..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x = torch.where(bit.view(G, B, V) == 1, torch.where(x >= 0, x / s["penalty"], x * s["penalty"]), x)
    x = x.double()
    m = x.amax(-1, keepdim=True)
    value = s["scores"].double()[..., None] + (x - (m + torch.exp(x - m).sum(-1, keepdim=True).log()))
    if s["finished"] is not None:
        only = torch.arange(V, device="cuda") == c["end"]
        done = (s["finished"] != 0)[..., None]
        value = torch.where(done, torch.where(only, s["scores"].double()[..., None], -math.inf), value)
    value = torch.where(torch.isfinite(value), value, -math.inf).view(G, B * V)
    value, order = torch.sort(value, dim=-1, descending=True, stable=True)
    value, order = value[:, :B], order[:, :B]
    there = value > -math.inf
    parents = torch.where(there, order // V, -1).to(torch.int32)
    tokens = torch.where(there, order % V, -1).to(torch.int32)
    got = [parents, tokens, value.float()]
    up = parents.clamp_min(0).long()
    if s["finished"] is not None:
        was = s["finished"].gather(1, up) != 0
        got.append(torch.where(there, (was | (tokens == c["end"])).to(torch.int32), s["finished"]))
    if s["seen"] is not None:
        rows = s["seen"].gather(1, up[..., None].expand(-1, -1, V // 32))
        add = there if s["finished"] is None else there & ~was
        word = tokens.clamp_min(0).long() // 32
        bit = torch.ones_like(word) << (tokens.clamp_min(0).long() % 32)
        bit = torch.where(bit >= 2 ** 31, bit - 2 ** 32, bit).to(torch.int32)
        hot = torch.where((torch.arange(V // 32, device="cuda") == word[..., None]) & add[..., None], bit[..., None], 0)
        s["seen"].copy_(torch.where(there[..., None], rows | hot, s["seen"]))
        got.append(s["seen"])
    return got


def _ring_reorder(s):
    ids, parents = s["streams"].long(), s["parents"].long()
    source = torch.where(parents < 0, ids, ids.gather(1, parents.clamp_min(0)))
    ids, source = ids.flatten(), source.flatten()
    live = s["slot_pos"][:, source] >= 0  # [L][m][C]
    s["kv"][:, ids] = torch.where(live[:, :, None, None, :, None], s["kv"][:, source], s["kv"][:, ids])
    s["slot_pos"][:, ids] = s["slot_pos"][:, source]
    return [s["kv"], s["slot_pos"]]


def _own(s):
    c = s["case"]
    if c["op"] == "tree_attend":
        return s["ring"].tree_attend(0, s["streams"], s["positions"], s["parents"], s["qkv"], out=s["out"])
    if c["op"] == "tree_commit":
        s["ring"].tree_commit(0, s["streams"], s["positions"], s["parents"], s["leaves"], s["qkv"],
                              next_positions=s["next"])
        return [s["kv"], s["slot_pos"], s["next"]]
    if c["op"] == "ring_reorder":
        s["ring"].reorder(s["streams"], s["parents"])
        return [s["kv"], s["slot_pos"]]
    from mockbird_b200 import beam_select

    got = beam_select(s["logits"], s["scores"], finished=s["finished"], end_id=c["end"], seen=s["seen"],
                      penalty=c["penalty"])
    return [x for x in got if x is not None] + ([] if s["seen"] is None else [s["seen"]])


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return (_tree_attend if op == "tree_attend" else _tree_commit if op == "tree_commit"
            else _beam_select if op == "beam_select" else _ring_reorder)(state)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    if c["op"] == "beam_select":
        G, B, V = c["groups"], c["beams"], c["codes"]
        e = 4 if c["dtype"] == "f32" else 2
        rows = G * (1 if c["first"] else B) * (0.8 if c["end"] >= 0 and not c["first"] else 1.0)  # dead and finished beams propose nothing
        seen = 0 if c["penalty"] == 1.0 else (rows + 2 * G * B) * V / 8
        return {"bytes": rows * V * e + seen + G * B * 20, "flops": rows * V * 4}
    e = 4 if c["dtype"] == "f32" else 2
    H, C = c["heads"], c["capacity"]
    if c["op"] == "ring_reorder":
        G, B, L = c["groups"], c["beams"], c["layers"]
        row = L * (2 * H * HD * e + 4)
        live = sum(min(p, C) for p in _positions(c, G))
        moved, read = B - 1, B * (1 - (1 - 1 / B) ** (B - 1))  # expected over parents drawn evenly
        return {"bytes": live * row * (moved + read) + 8 * G * B, "flops": 0}
    n, T = c["n"], c["nodes"]
    if c["op"] == "tree_commit":
        rows = sum(_accepted(c, n)) * c["layers"]
        return {"bytes": rows * (2 * H * HD * (4 + e) + 4) + n * (16 + 4 * T), "flops": rows * H * HD * 3}
    at, counts = _positions(c, n), _counts(c, n)
    live = [min(p, C) for p in at]
    bytes_ = sum(w * (2 * H * HD * e + 4) for w in live) + sum(counts) * 4 * H * HD * 4 + n * (8 + 4 * T)
    return {"bytes": bytes_, "flops": sum(4 * HD * H * m * (w + 1) for m, w in zip(counts, live))}


# ---------------------------------------------------------------- the same outputs in 64 bits

def _path(parents, t):
    got = []
    while t >= 0:
        got.append(t)
        t = parents[t]
    return got[::-1]


def _turn(x, p):
    """x [..., 64] in 64 bits turned by position p, as complex numbers."""
    i = torch.arange(HD // 2, dtype=torch.float64, device=x.device)
    z = torch.view_as_complex(x.reshape(*x.shape[:-1], HD // 2, 2).contiguous())
    z = z * torch.polar(torch.ones_like(i), p * THETA ** (-2 * i / HD))
    return torch.view_as_real(z).flatten(-2)


def _exact_attend(c, s):
    n, T, H, C = c["n"], c["nodes"], c["heads"], c["capacity"]
    store, out = DTYPES[c["dtype"]], torch.zeros(n, T, H * HD, dtype=torch.float64, device="cuda")
    parents, at, ids = s["parents"].tolist(), s["positions"].tolist(), s["streams"].tolist()
    for i in range(n):
        row = s["qkv"][i].double().view(T, 3, H, HD)
        paths = [_path(parents[i], t) if parents[i][t] != -2 else [] for t in range(T)]
        pos = [at[i] + max(0, len(x) - 1) for x in paths]
        there = [t for t in range(T) if paths[t]]
        turned = torch.stack([_turn(row[t, :2], pos[t]) for t in range(T)])  # [T][2][H][64]
        keys = torch.cat((s["kv"][0, ids[i], 0].double(), turned[:, 1].to(store).double().transpose(0, 1)), 1)
        vals = torch.cat((s["kv"][0, ids[i], 1].double(), row[:, 2].to(store).double().transpose(0, 1)), 1)
        sp = s["slot_pos"][0, ids[i]].long()
        mask = torch.zeros(T, C + T, dtype=torch.bool)
        for t in there:
            mask[t, [C + u for u in paths[t] if pos[t] - pos[u] < C]] = True
        mask = mask.cuda()
        p = torch.tensor(pos, device="cuda")[:, None]
        mask[:, :C] = (sp >= 0) & (sp < at[i]) & (p - sp < C)
        score = torch.einsum("thd,hjd->htj", turned[:, 0], keys) / 8
        w = torch.softmax(score.masked_fill(~mask, -math.inf), -1)
        o = torch.einsum("htj,hjd->thd", w, vals).reshape(T, H * HD)
        out[i, there] = o[there]
    return out


def _exact_commit(c, s):
    T, H, C = c["nodes"], c["heads"], c["capacity"]
    kv, sp, nxt = s["kv"], s["slot_pos"], s["positions"].clone()
    parents, at, ids, leaves = (s[k].tolist() for k in ("parents", "positions", "streams", "leaves"))
    for i in range(c["n"]):
        path = _path(parents[i], leaves[i])
        for d, t in enumerate(path):
            if len(path) - d <= C:
                row = s["qkv"][:, i, t].double().view(-1, 3, H, HD)
                kv[:, ids[i], 0, :, (at[i] + d) % C] = _turn(row[:, 1], at[i] + d).to(kv.dtype)
                kv[:, ids[i], 1, :, (at[i] + d) % C] = row[:, 2].to(kv.dtype)
                sp[:, ids[i], (at[i] + d) % C] = at[i] + d
        nxt[i] += len(path)
    return [kv, sp, nxt]


def _exact_beam(c, s):
    G, B, V = c["groups"], c["beams"], c["codes"]
    parents = torch.full((G, B), -1, dtype=torch.int32)
    tokens, scores = parents.clone(), torch.full((G, B), -math.inf, dtype=torch.float64)
    done = None if s["finished"] is None else s["finished"].cpu().clone()
    seen = None if s["seen"] is None else s["seen"].cpu()
    after = None if seen is None else seen.clone()
    for g in range(G):
        found = []
        for b in range(B):
            start = float(s["scores"][g, b])
            if done is not None and int(s["finished"][g, b]):
                if math.isfinite(start):
                    found.append((-start, b * V + c["end"]))
                continue
            x = s["logits"][g, b].double()
            if seen is not None:
                on = (seen[g, b].to(torch.int64)[:, None] >> torch.arange(32)) & 1
                on = on.flatten().bool().cuda()
                x = torch.where(on & (x >= 0), x / c["penalty"], torch.where(on, x * c["penalty"], x))
            lp = start + (x - torch.logsumexp(x, 0))
            cut = torch.topk(lp, min(B, V)).values[-1]
            at = (lp >= cut).nonzero().flatten()
            found += [(-v, b * V + j) for v, j in zip(lp[at].tolist(), at.tolist()) if math.isfinite(v)]
        for k, (v, j) in enumerate(sorted(found)[:B]):
            parents[g, k], tokens[g, k], scores[g, k] = j // V, j % V, -v
            was = done is not None and bool(s["finished"][g, j // V])
            if done is not None:
                done[g, k] = int(was or j % V == c["end"])
            if seen is not None:
                after[g, k] = seen[g, j // V]
                if not was:
                    word = int(after[g, k, j % V // 32]) & 0xFFFFFFFF | 1 << j % 32
                    after[g, k, j % V // 32] = word - (1 << 32) if word >> 31 else word
    return [x for x in (parents, tokens, scores, done, after) if x is not None]


def _exact_reorder(c, s):
    kv, sp = s["kv"].clone(), s["slot_pos"].clone()
    for ids, up in zip(s["streams"].tolist(), s["parents"].tolist()):
        for k, stream in enumerate(ids):
            source = ids[up[k]]
            live = (s["slot_pos"][:, source] >= 0)[:, None, None, :, None]
            kv[:, stream] = torch.where(live, s["kv"][:, source], s["kv"][:, stream])
            sp[:, stream] = s["slot_pos"][:, source]
    return [kv, sp]


def exact(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    op = c["op"]
    return (_exact_attend if op == "tree_attend" else _exact_commit if op == "tree_commit"
            else _exact_beam if op == "beam_select" else _exact_reorder)(c, s)
