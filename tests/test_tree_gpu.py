"""Attention of a tree of drafted tokens over the ring, and the commit of an accepted path, against the plain
64-bit form (search_util) and against append_attend one node after another."""
import ctypes
import os
import random

import numpy as np
import pytest
import torch

from mockbird_b200 import KvRing, MockbirdError, beam_select
from search_util import HD, TORCH_DT, attend_tree, path_to

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def tree_of(kind, T, seed=0):
    r = random.Random(seed)
    if kind == "chain":
        return [t - 1 for t in range(T)]
    if kind == "star":
        return [-1] * T
    if kind == "ragged":  # random, every third node absent
        par = []
        for t in range(T):
            ok = [-1] + [u for u in range(t) if par[u] != -2]
            par.append(-2 if t % 3 == 2 else r.choice(ok))
        return par
    return [r.randrange(-1, t) for t in range(T)]


def normal(shape, seed, scale=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.empty(shape, device=DEV).normal_(generator=g).mul_(scale)


def fill(ring, layer, stream, base, seed):
    """The positions below `base` that a ring of this capacity still holds, through ring_write."""
    first = max(0, base - ring.capacity)
    if base == first:
        return
    k = normal((ring.heads, base - first, HD), seed).to(ring.torch_dtype)
    v = normal((ring.heads, base - first, HD), seed + 1).to(ring.torch_dtype)
    ring.ring_write(layer, stream, first, k, v)


class Held:
    """A ring's memory, read and written through its addresses."""

    def __init__(self, ring):
        self.ring = ring
        i = ring.info
        L, S, H, C = ring.layers, ring.streams, ring.heads, ring.capacity
        kind = {"f32": "<f4", "bf16": "<i2", "f16": "<f2"}[ring.dtype]
        self.kv = self.view(i.kv, (L, S, 2, H, C, HD), kind).view(ring.torch_dtype)
        self.slot_pos = self.view(i.slot_pos, (L, S, C), "<i4")

    @staticmethod
    def view(address, shape, kind):
        class A:
            __cuda_array_interface__ = {"data": (address, False), "shape": shape, "typestr": kind, "version": 3}
        return torch.as_tensor(A(), device=DEV)

    def item(self, layer, stream):
        kv = self.kv[layer, stream].double().cpu().numpy()
        return kv[0], kv[1], self.slot_pos[layer, stream].cpu().numpy()


def check(ring, layer, streams, bases, trees, qkv, out, before=None):
    held = Held(ring)
    got = out.double().cpu().numpy()
    rows = qkv.cpu().numpy()
    for i, (s, b, par) in enumerate(zip(streams, bases, trees)):
        k, v, sp = held.item(layer, s)
        want, bound = attend_tree(k, v, sp, b, par, rows[i], ring.dtype, ring.heads)
        for t, p in enumerate(par):
            if p == -2:
                assert before is None or torch.equal(out[i, t], before[i, t])
                continue
            off = np.abs(got[i, t] - want[t])
            assert np.isfinite(got[i, t]).all(), (i, t)
            assert (off <= bound[t]).all(), (i, t, off.max(), bound[t][off.argmax()], (off / bound[t]).max())


# node counts around the query tiles (16, 32, 64) and windows around the slot tiles and splits
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,C,bases,wrap,kind", [
    (1, 17, [0, 1, 16, 17, 40], True, "chain"),
    (2, 33, [31, 32, 33, 34, 66], True, "star"),
    (5, 64, [0, 15, 16, 17, 59], False, "random"),
    (8, 570, [300, 562, 0, 1], False, "random"),
    (15, 130, [127, 128, 129, 130, 131, 259, 260], True, "ragged"),
    (16, 512, [511, 512, 513, 1030, 3], True, "chain"),
    (17, 300, [255, 256, 257, 299, 600], True, "random"),
    (33, 200, [10, 150, 199, 200, 345], True, "ragged"),
    (64, 1100, [1023, 1024, 1025, 2300, 0], True, "random"),
    (64, 40, [0, 39, 40, 41, 100], True, "chain"),     # a path longer than the ring
    (48, 2, [0, 1, 2, 3, 77], True, "random"),
    (7, 1, [0, 1, 5], True, "chain"),
])
def test_tree_against_64_bits(dtype, T, C, bases, wrap, kind):
    n, H = len(bases), 3
    ring = KvRing(layers=2, heads=H, streams=n + 2, capacity=C, dtype=dtype, wrap=wrap, max_position=4096)
    streams = [(3 * i + 1) % (n + 2) for i in range(n)] if (n + 2) % 3 else [n + 1 - i for i in range(n)]
    for i in range(n):
        fill(ring, 1, streams[i], bases[i], 100 * T + i)
    trees = [tree_of(kind, T, i) for i in range(n)]
    qkv = normal((n, T, 3 * H * HD), T)
    before = torch.full((n, T, H * HD), 7.5, device=DEV)
    held = Held(ring)
    kv, sp = held.kv.clone(), held.slot_pos.clone()
    out = ring.tree_attend(1, streams, bases, trees, qkv, out=before.clone())
    ring.sync()
    check(ring, 1, streams, bases, trees, qkv, out, before)
    assert torch.equal(held.slot_pos, sp) and torch.equal(held.kv, kv)  # the rings are only read


@pytest.mark.parametrize("T", [5, 9, 33])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_large_scores_and_skewed_rows(dtype, T):
    """Scores of some hundreds (one slot takes the whole weight) and rows of very different size."""
    H, C = 2, 257
    ring = KvRing(layers=1, heads=H, streams=1, capacity=C, dtype=dtype, wrap=True, max_position=1024)
    held = Held(ring)
    fill(ring, 0, 0, 400, 5)
    held.kv.mul_(torch.logspace(-3, 1.2, C, device=DEV)[:, None].to(held.kv.dtype))
    qkv = normal((1, T, 3 * H * HD), 6) * torch.logspace(-4, 1.5, T, device=DEV)[None, :, None]
    trees = [tree_of("random", T, 1)]
    out = ring.tree_attend(0, [0], [400], trees, qkv)
    ring.sync()
    check(ring, 0, [0], [400], trees, qkv, out)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("C,start,T", [(64, 0, 20), (64, 50, 33), (300, 299, 16), (24, 100, 40)])
def test_chain_is_append_attend_in_sequence(dtype, C, start, T):
    """A chain of drafts gives what append_attend gives node by node, and committing it leaves the same ring."""
    H, L = 12, 2
    a = KvRing(layers=L, heads=H, streams=2, capacity=C, dtype=dtype, wrap=True, max_position=1024)
    b = KvRing(layers=L, heads=H, streams=2, capacity=C, dtype=dtype, wrap=True, max_position=1024)
    for layer in range(L):
        for ring in (a, b):
            fill(ring, layer, 1, start, 11 + layer)
    qkv = normal((L, 1, T, 3 * H * HD), 12)
    tree = [tree_of("chain", T)]
    for layer in range(L):
        out = a.tree_attend(layer, [1], [start], tree, qkv[layer])
        check(a, layer, [1], [start], tree, qkv[layer], out)
        for t in range(T):
            row = b.append_attend(layer, [1], [start + t], qkv[layer, :, t].contiguous())
            # each side is within 1e-5 of the formula at unit inputs (the bound of `check` is tighter)
            assert (row[0] - out[0, t]).abs().max() < 2e-5, (layer, t)
    nxt = a.tree_commit(0, [1], [start], tree, [T - 1], qkv)
    a.sync(), b.sync()
    assert nxt.tolist() == [start + T]
    ha, hb = Held(a), Held(b)
    assert torch.equal(ha.slot_pos, hb.slot_pos)
    live = (hb.slot_pos >= 0)[:, :, None, None, :, None]
    assert torch.equal(torch.where(live, ha.kv, 0), torch.where(live, hb.kv, 0))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("T,H,n", [(7, 2, 1), (13, 2, 1), (20, 2, 1), (50, 2, 1), (20, 64, 5)])
def test_what_is_masked_does_not_matter(dtype, bad, T, H, n):
    """NaN and infinities in empty slots, in slots of positions the query may not see (later ones, and expired
    ones that another node still sees), in absent nodes and in nodes off the path."""
    C, base = 90, 150
    ring = KvRing(layers=1, heads=H, streams=1, capacity=C, dtype=dtype, wrap=True, max_position=1024, max_batch=n)
    held = Held(ring)
    fill(ring, 0, 0, base, 3)
    sp = held.slot_pos[0, 0]
    kv = held.kv[0, 0]
    for j in (0, 17, 33, 89):          # empty
        sp[j] = -1
    sp[5], sp[40] = base, base + 3     # left over from a longer run: not below the base
    for j in (0, 17, 33, 89, 5, 40):
        kv[:, :, j] = bad
    # 0 - 1 - 2 - 3 a chain, 4.. hang on the ring; node 4 absent, node 5 (and the last) off every other path
    tree = [-1, 0, 1, 2] + [-1] * (T - 4)
    tree[4] = -2
    qkv = normal((1, T, 3 * H * HD), 4)
    for t in (4, 5, T - 1):
        qkv[0, t] = bad
    # the slot of position base - C + 1 is seen at depth 0, expired for depth >= 1
    edge = (base - C + 1) % C
    kv[1, :, edge] = bad
    # (n equal items: from 296 heads in all on, 16-bit rings take two tiles of rows per warp)
    many = qkv.expand(n, -1, -1).contiguous()
    out = ring.tree_attend(0, [0] * n, [base] * n, [tree] * n, many, out=torch.zeros(n, T, H * HD, device=DEV))
    ring.sync()
    for i in range(1, n):
        assert torch.equal(out[i].nan_to_num(7.0), out[0].nan_to_num(7.0))
    got = out[0].double().cpu().numpy()
    k, v, s = held.item(0, 0)
    want, bound = attend_tree(k, v, s, base, tree, qkv[0].cpu().numpy(), dtype, H)
    for t in (1, 2, 3):  # depth >= 1: nothing bad is visible
        assert np.isfinite(got[t]).all(), t
        assert (np.abs(got[t] - want[t]) <= bound[t]).all(), t
    # without the bad value at the edge the siblings are clean too, whatever nodes 5 and T - 1 hold
    kv[1, :, edge] = 0.5
    out = ring.tree_attend(0, [0] * n, [base] * n, [tree] * n, many)
    ring.sync()
    got = out[0].double().cpu().numpy()
    k, v, s = held.item(0, 0)
    want, bound = attend_tree(k, v, s, base, tree, qkv[0].cpu().numpy(), dtype, H)
    for t in range(T):
        if t in (4, 5, T - 1):
            continue
        assert np.isfinite(got[t]).all(), t
        assert (np.abs(got[t] - want[t]) <= bound[t]).all(), t


def test_partly_filled_ring_and_repeated_stream():
    """Holes all over the window, whole tiles of them; two trees on one stream; order of the streams."""
    H, C, T = 4, 700, 12
    ring = KvRing(layers=1, heads=H, streams=3, capacity=C, dtype="f32", wrap=True, max_position=4096, max_batch=4)
    held = Held(ring)
    for s in range(3):
        fill(ring, 0, s, 650 + 40 * s, s)
    keep = normal((C,), 9) < -0.25
    keep[64:256] = False
    held.slot_pos[0, 2][~keep] = -1
    held.slot_pos[0, 1] = -1  # nothing
    streams, bases = [2, 0, 2, 1], [730, 650, 729, 690]
    trees = [tree_of(k, T, i) for i, k in enumerate(("random", "star", "chain", "ragged"))]
    qkv = normal((4, T, 3 * H * HD), 8)
    out = ring.tree_attend(0, streams, bases, trees, qkv)
    ring.sync()
    check(ring, 0, streams, bases, trees, qkv, out)


def test_rejected_and_absent_items_leave_their_rows():
    H, C, T = 2, 50, 6
    ring = KvRing(layers=1, heads=H, streams=4, capacity=C, dtype="f32", wrap=False, max_position=60)
    for s in range(4):
        fill(ring, 0, s, 20, s)
    ok = tree_of("random", T, 1)
    cases = [  # (stream, base, tree, what it says)
        (4, 20, ok, "stream"), (-1, 20, ok, "stream"), (0, -1, ok, "position"), (0, 60, [-1] * T, "position"),
        (0, 50, [-1] * T, "capacity|ring"), (0, 46, tree_of("chain", T), "ring"),
        (0, 20, [-1, 1, 0, 0, 0, 0], "tree"), (0, 20, [-1, 0, 7, 0, 0, 0], "tree"), (0, 20, [-3] + [-1] * 5, "tree"),
        (0, 20, [-1, -2, 1, -1, -1, -1], "tree"), (0, 20, [-1, 2 ** 31 - 1, 0, 0, 0, 0], "tree"),
    ]
    qkv = normal((3, T, 3 * H * HD), 2)
    for stream, base, tree, word in cases:
        before = torch.full((3, T, H * HD), 3.25, device=DEV)
        out = ring.tree_attend(0, [1, stream, 2], [20, base, 20], [ok, tree, ok], qkv, out=before.clone())
        with pytest.raises(MockbirdError, match=word):
            ring.sync()
        ring.sync()
        assert torch.equal(out[1], before[1]), (stream, base, tree)
        check(ring, 0, [1, 2], [20, 20], [ok, ok], qkv[[0, 2]], out[[0, 2]])
        with pytest.raises(MockbirdError, match=word):
            nxt = torch.tensor([-7, -7, -7], dtype=torch.int32, device=DEV)
            ring.tree_commit(0, [1, stream, 2], [20, base, 20], [ok, tree, ok], [-1, T - 1, -1], qkv[None], nxt)
            ring.sync()
        assert nxt.tolist() == [20, -7, 20]
    # the last base a chain of T fits at
    out = ring.tree_attend(0, [0], [44], [tree_of("chain", T)], qkv[:1])
    ring.sync()
    # a padding item: no node present, its stream and position are not looked at
    before = torch.full((3, T, H * HD), 3.25, device=DEV)
    out = ring.tree_attend(0, [1, -5, 2], [20, 10 ** 6, 20], [ok, [-2] * T, ok], qkv, out=before.clone())
    ring.sync()
    assert torch.equal(out[1], before[1])
    for leaf in (-2, T, 2 ** 30, 2):  # the last: an absent node
        tree = [-1, 0, -2, 0, 0, 0]
        with pytest.raises(MockbirdError, match="tree"):
            ring.tree_commit(0, [1], [20], [tree], [leaf], qkv[None, :1].contiguous())
            ring.sync()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("C,wrap,T,H", [(20, True, 33, 5), (200, True, 64, 1), (400, False, 9, 12), (100, True, 64, 64)])
def test_commit_is_rope_append_along_the_path(dtype, C, wrap, T, H):
    L, n = 3, 4
    bases = [0, 7, C - T - 1 if not wrap else C - 3, 2 * C + 5 if wrap else 3]
    a = KvRing(layers=L, heads=H, streams=6, capacity=C, dtype=dtype, wrap=wrap, max_position=1024)
    b = KvRing(layers=L, heads=H, streams=6, capacity=C, dtype=dtype, wrap=wrap, max_position=1024)
    streams = [5, 0, 3, 2]
    for ring in (a, b):
        for layer in range(L):
            for i in range(n):
                fill(ring, layer, streams[i], bases[i], 10 * layer + i)
    trees = [tree_of(k, T, i) for i, k in enumerate(("chain", "random", "ragged", "star"))]
    leaves = [T - 1, T - 1, max(t for t in range(T) if trees[2][t] != -2), -1]
    qkv = normal((2, n, T, 3 * H * HD), 1)
    nxt = a.tree_commit(1, streams, bases, trees, leaves, qkv)  # layers 1 and 2
    a.sync()
    for i in range(n):
        path = path_to(trees[i], leaves[i])
        assert nxt[i].item() == bases[i] + len(path)
        for d, t in enumerate(path):
            for layer in (1, 2):
                b.rope_split_ring(layer, [streams[i]], [bases[i] + d], qkv[layer - 1, i:i + 1, t].clone())
    b.sync()
    ha, hb = Held(a), Held(b)
    assert torch.equal(ha.slot_pos, hb.slot_pos)
    assert torch.equal(ha.kv, hb.kv)


def test_drafting_loop_gives_the_plain_decode():
    """Trees verified and committed step after step leave the ring, the positions and the attention of a run that
    decodes the accepted tokens one by one."""
    L, H, C, n, T = 2, 4, 48, 3, 10
    a = KvRing(layers=L, heads=H, streams=n, capacity=C, dtype="bf16", wrap=True, max_position=1024)
    b = KvRing(layers=L, heads=H, streams=n, capacity=C, dtype="bf16", wrap=True, max_position=1024)
    ids = torch.arange(n, dtype=torch.int32, device=DEV)
    pos = torch.zeros(n, dtype=torch.int32, device=DEV)
    r = random.Random(3)
    for step in range(14):
        trees = [tree_of("random", T, 10 * step + i) for i in range(n)]
        leaves = [r.randrange(-1, T) for _ in range(n)]
        qkv = normal((L, n, T, 3 * H * HD), step)
        outs = [a.tree_attend(layer, ids, pos, trees, qkv[layer]) for layer in range(L)]
        nxt = a.tree_commit(0, ids, pos, trees, leaves, qkv)
        for i in range(n):
            for d, t in enumerate(path_to(trees[i], leaves[i])):
                p = int(pos[i]) + d
                for layer in range(L):
                    row = b.append_attend(layer, [i], [p], qkv[layer, i:i + 1, t].contiguous())
                    assert (row[0] - outs[layer][i, t]).abs().max() < 2e-5, (step, i, t)
        pos = nxt
        a.sync(), b.sync()
    ha, hb = Held(a), Held(b)
    assert torch.equal(ha.slot_pos, hb.slot_pos) and torch.equal(ha.kv, hb.kv)
    x = normal((n, 3 * H * HD), 99)
    assert torch.equal(a.append_attend(0, ids, pos, x), b.append_attend(0, ids, pos, x))
    a.sync(), b.sync()


def test_capture_streams_and_determinism():
    """Replayed from a graph with new inputs in place, and two streams of one context at once: tree_attend keeps
    nothing between calls and shares nothing among them, so results are the same bits."""
    H, C, T, n = 12, 1024, 16, 4
    ring = KvRing(layers=1, heads=H, streams=n, capacity=C, dtype="bf16", wrap=True, max_position=4096)
    for s in range(n):
        fill(ring, 0, s, 1500 + s, s)
    ids = torch.arange(n, dtype=torch.int32, device=DEV)
    pos = torch.tensor([1500, 1501, 1502, 1503], dtype=torch.int32, device=DEV)
    trees = torch.tensor([tree_of("random", T, i) for i in range(n)], dtype=torch.int32, device=DEV)
    qa, qb = normal((n, T, 3 * H * HD), 1), normal((n, T, 3 * H * HD), 2)
    wa, wb = (ring.tree_attend(0, ids, pos, trees, q) for q in (qa, qb))
    ring.sync()
    buf, out = qa.clone(), torch.zeros_like(wa)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ring.tree_attend(0, ids, pos, trees, buf, out=out)
    for q, w in ((qa, wa), (qb, wb), (qa, wa)):
        buf.copy_(q)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        got.append((ring.tree_attend(0, ids, pos, trees, qa, stream=s1),
                    ring.tree_attend(0, ids, pos, trees, qb, stream=s2.cuda_stream)))
    torch.cuda.synchronize()
    ring.sync()
    assert all(torch.equal(x, wa) and torch.equal(y, wb) for x, y in got)


def test_outputs_of_another_stream_are_not_memory_in_use():
    """A call on another stream does not get memory that work queued on the current stream still uses."""
    H, C, T = 4, 64, 8
    ring = KvRing(layers=1, heads=H, streams=1, capacity=C, dtype="f32", wrap=True, max_position=256)
    fill(ring, 0, 0, 50, 1)
    trees, qkv = [tree_of("chain", T)], normal((1, T, 3 * H * HD), 2)
    x, s = normal((1, 4, 1000), 3), torch.zeros(1, 4, device=DEV)
    want, chosen = ring.tree_attend(0, [0], [50], trees, qkv), beam_select(x, s)
    ring.sync()
    other = torch.cuda.Stream()
    torch.cuda._sleep(200_000_000)
    held = [torch.empty(1, T, H * HD, device=DEV).fill_(3.0) for _ in range(4)]
    held += [torch.empty(1, 4, dtype=torch.int32, device=DEV).fill_(3) for _ in range(8)]
    busy = {t.data_ptr() for t in held}
    del held
    got = ring.tree_attend(0, [0], [50], trees, qkv, stream=other)
    picked = beam_select(x, s, stream=other.cuda_stream)
    assert not busy & {t.data_ptr() for t in (got, *picked[:3])}
    other.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(picked[:3], chosen[:3]))
    ring.sync()


def test_bounded_wait_runs_out_and_the_context_recovers():
    """mb_set_wait_limit's probe: the waits for copies run out, the call returns, the next sync says so, and the
    context goes on."""
    H, C, T = 2, 300, 9
    ring = KvRing(layers=1, heads=H, streams=2, capacity=C, dtype="f32", wrap=True, max_position=1024)
    for s in range(2):
        fill(ring, 0, s, 200, s)
    trees = [tree_of("random", T, i) for i in range(2)]
    qkv = normal((2, T, 3 * H * HD), 1)
    want = ring.tree_attend(0, [0, 1], [200, 200], trees, qkv)
    ring.sync()
    ring.set_wait_limit(-20000)
    ring.tree_attend(0, [0, 1], [200, 200], trees, qkv)
    with pytest.raises(MockbirdError, match="TIMEOUT"):
        ring.sync()
    ring.set_wait_limit(0)
    assert torch.equal(ring.tree_attend(0, [0, 1], [200, 200], trees, qkv), want)
    ring.sync()


@pytest.mark.parametrize("H", [1, 64])
def test_head_counts(H):
    """The fewest and the most heads."""
    C, T = 70, 21
    ring = KvRing(layers=1, heads=H, streams=2, capacity=C, dtype="bf16", wrap=True, max_position=512)
    for s in range(2):
        fill(ring, 0, s, 60 + 30 * s, s)
    trees = [tree_of("random", T, i) for i in range(2)]
    qkv = normal((2, T, 3 * H * HD), 3)
    out = ring.tree_attend(0, [0, 1], [60, 90], trees, qkv)
    ring.sync()
    check(ring, 0, [0, 1], [60, 90], trees, qkv, out)


def test_first_calls_may_be_captured():
    """Nothing has to run before a capture: the first call of every operator of a process, in a graph."""
    import subprocess
    import sys

    code = """
import torch
from mockbird_b200 import KvRing, beam_select
H, T, n = 2, 5, 2
ring = KvRing(layers=2, heads=H, streams=n, capacity=40, dtype="f16", wrap=True, max_position=128)
ids = torch.arange(n, dtype=torch.int32, device="cuda")
pos = torch.zeros(n, dtype=torch.int32, device="cuda")
tree = torch.tensor([[-1, 0, 1, 1, -1]] * n, dtype=torch.int32, device="cuda")
leaf = torch.tensor([2, 4], dtype=torch.int32, device="cuda")
qkv = torch.randn(2, n, T, 3 * H * 64, device="cuda")
x, s = torch.randn(1, n, 5000, device="cuda"), torch.zeros(1, n, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = ring.tree_attend(0, ids, pos, tree, qkv[0])
    nxt = ring.tree_commit(0, ids, pos, tree, leaf, qkv)
    parents, tokens, scores, _ = beam_select(x, s)
    ring.reorder(ids.view(1, n), parents)
g.replay()
ring.sync()
assert nxt.tolist() == [3, 1] and torch.isfinite(out).all() and torch.isfinite(scores).all(), (nxt, scores)
want = beam_select(x, s)
assert torch.equal(want[0], parents) and torch.equal(want[1], tokens) and torch.equal(want[2], scores)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("n,T,dtype", [(40, 16, "bf16"), (130, 5, "f32"), (70, 20, "f16"), (70, 31, "bf16"),
                                       (60, 32, "f32"), (50, 64, "bf16")])
def test_many_ragged_items(n, T, dtype):
    """More blocks than run at once (their items are then taken longest window first), equal windows and empty
    ones among them; every row against a call of its own."""
    H, C = 12, 384
    ring = KvRing(layers=1, heads=H, streams=n, capacity=C, dtype=dtype, wrap=True, max_position=2048)
    r = random.Random(n)
    bases = [r.choice([0, 7, 100, r.randrange(900)]) for _ in range(n)]
    ids = list(range(n))
    r.shuffle(ids)
    for s, b in zip(ids, bases):
        fill(ring, 0, s, b, s)
    trees = [tree_of("random", T, i) for i in range(n)]
    qkv = normal((n, T, 3 * H * HD), 5)
    out = ring.tree_attend(0, ids, bases, trees, qkv)
    for i in range(0, n, 3):
        one = ring.tree_attend(0, ids[i:i + 1], bases[i:i + 1], trees[i:i + 1], qkv[i:i + 1])
        # each side is within 1e-5 of the formula at unit inputs
        assert (one[0] - out[i]).abs().max() < 2e-5, i
    ring.sync()
    check(ring, 0, ids[:4], bases[:4], trees[:4], qkv[:4], out[:4])


def test_offsets_past_32_bits():
    """A stream whose rows start more than 2^31 elements (4 GB) into the ring."""
    H, C, S, T = 16, 1024, 1100, 9
    ring = KvRing(layers=1, heads=H, streams=S, capacity=C, dtype="bf16", wrap=True, max_position=4096, max_batch=4)
    assert (S - 1) * 2 * H * C * HD > 2 ** 31
    for s in (0, S - 1):
        fill(ring, 0, s, 1500, s)
    trees = [tree_of("random", T, i) for i in range(2)]
    qkv = normal((2, T, 3 * H * HD), 7)
    out = ring.tree_attend(0, [S - 1, 0], [1500, 1500], trees, qkv)
    ring.sync()
    check(ring, 0, [S - 1, 0], [1500, 1500], trees, qkv, out)
    held = Held(ring)
    ring.tree_commit(0, [S - 1, 0], [1500, 1500], trees, [T - 1, -1], qkv[None])
    ring.reorder([[0, S - 1]], [[-1, 0]])
    ring.sync()
    assert torch.equal(held.kv[0, 0], held.kv[0, S - 1]) and torch.equal(held.slot_pos[0, 0], held.slot_pos[0, S - 1])


def test_refusals():
    H, C, T = 2, 32, 4
    ring = KvRing(layers=2, heads=H, streams=3, capacity=C, dtype="f32", wrap=True, max_position=128)
    q = normal((2, T, 3 * H * HD), 0)
    tree = [tree_of("chain", T)] * 2
    good = dict(layer=0, streams=[0, 1], positions=[0, 0], parents=tree, qkv=q)

    def refused(kind, match, fn=ring.tree_attend, **kw):
        with pytest.raises(kind, match=match):
            fn(**{**(good if fn == ring.tree_attend else commit), **kw})

    refused(MockbirdError, "LAYER", layer=2)
    refused(MockbirdError, "LAYER", layer=-1)
    refused(ValueError, "streams", streams=[0])
    refused(ValueError, "positions", positions=[0, 0, 0])
    refused(ValueError, "parents", parents=[[-1] * 3] * 2)
    refused(ValueError, "qkv", qkv=q[0])
    refused(ValueError, "qkv", qkv=q[..., :64].contiguous())
    refused(TypeError, "qkv", qkv=q.double())
    refused(TypeError, "qkv", qkv=q.cpu())
    refused(TypeError, "qkv", qkv=q.transpose(0, 1))
    refused(TypeError, "streams", streams=torch.zeros(2, dtype=torch.int64, device=DEV))
    refused(ValueError, "out", out=torch.zeros(2, T, H * HD + 1, device=DEV))
    refused(TypeError, "out", out=torch.zeros(2, T, H * HD, dtype=torch.float64, device=DEV))
    refused(MockbirdError, "out overlaps", out=q.view(-1)[:2 * T * H * HD].view(2, T, H * HD))
    refused(MockbirdError, "out overlaps", out=q.view(-1)[-2 * T * H * HD:].view(2, T, H * HD))
    many = normal((4, T, 3 * H * HD), 0)
    refused(MockbirdError, "max_batch", streams=[0, 1, 2, 0], positions=[0] * 4, parents=[tree[0]] * 4, qkv=many)
    wide = normal((1, 65, 3 * H * HD), 0)
    refused(MockbirdError, "node count", streams=[0], positions=[0], parents=[tree_of("chain", 65)], qkv=wide)
    refused(MockbirdError, "node count", streams=[0], positions=[0], parents=np.zeros((1, 0)), qkv=wide[:, :0])
    flat = torch.zeros(2 * T * 3 * H * HD + 1, device=DEV)
    refused(MockbirdError, "misaligned", qkv=flat[1:].view(2, T, 3 * H * HD))
    lay = normal((2, 2, T, 3 * H * HD), 0)
    commit = dict(layer=0, streams=[0, 1], positions=[0, 0], parents=tree, leaves=[0, 0], qkv=lay)
    refused(MockbirdError, "LAYER", fn=ring.tree_commit, layer=1)
    refused(ValueError, "leaves", fn=ring.tree_commit, leaves=[0])
    p = torch.zeros(2, dtype=torch.int32, device=DEV)
    refused(MockbirdError, "overlaps", fn=ring.tree_commit, positions=p, next_positions=p)
    assert ring.lib.mb_tree_attend(ring.ctx, 0, 1, 1, None, None, None, None, None, None) == 1
    assert ring.lib.mb_tree_commit(ring.ctx, 0, 1, 1, 1, None, None, None, None, None, None, None) == 1
    assert ring.lib.mb_tree_commit(ring.ctx, 0, 0, 1, 1, None, None, None, None, None, None, None) == 3
    # no items: nothing runs
    assert ring.lib.mb_tree_attend(ring.ctx, 0, 0, 1, None, None, None, None, None, ctypes.c_void_p()) == 0
    ring.sync()
