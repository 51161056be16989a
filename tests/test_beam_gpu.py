"""Beam search: the selection over beams and codes, and the reordering of the beams' rings, against the plain
64-bit form (search_util)."""
import math
import random

import numpy as np
import pytest
import torch

from mockbird_b200 import KvRing, MockbirdError, argmax_penalty, beam_select
from search_util import HD, TORCH_DT, select
from test_tree_gpu import Held, fill, normal, tree_of

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
INF = math.inf


def case(G, B, V, dtype, seed, pad=0, shift=0, scale=3.0):
    """Rows of V logits, V + pad apart, the first `shift` elements behind an aligned address."""
    flat = torch.zeros(G * B * (V + pad) + shift, device=DEV, dtype=TORCH_DT[dtype])
    rows = flat[shift:].view(G, B, V + pad)[:, :, :V]
    rows.copy_(normal((G, B, V), seed, scale).to(TORCH_DT[dtype]))
    scores = -20 * torch.rand(G, B, generator=torch.Generator().manual_seed(seed)).to(DEV)
    return rows, scores


def masks(shape, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randint(-2 ** 31, 2 ** 31, shape, device=DEV, dtype=torch.int64, generator=g).to(torch.int32)


def check(logits, scores, finished=None, end_id=-1, seen=None, penalty=1.0):
    x, s = logits.float().cpu().numpy(), scores.cpu().numpy()
    f = None if finished is None else finished.cpu().numpy()
    m = None if seen is None else seen.cpu().numpy()
    kept = [t.clone() for t in (logits, scores) if t is not None]
    p, t, o, d = beam_select(logits, scores, finished, end_id, seen, penalty)
    torch.cuda.synchronize()
    assert all(torch.equal(a.nan_to_num(1e9), b.nan_to_num(1e9)) for a, b in zip(kept, (logits, scores)))
    p, t, o = p.cpu().numpy(), t.cpu().numpy(), o.cpu().numpy()
    for g in range(x.shape[0]):
        wp, wt, wo, wd, ws = select(x[g], s[g], None if f is None else f[g], end_id, None if m is None else m[g],
                                    penalty)
        assert np.array_equal(p[g], wp) and np.array_equal(t[g], wt), (g, p[g], wp, t[g], wt, o[g], wo)
        fin = np.isfinite(wo)
        assert np.array_equal(np.isfinite(o[g]), fin) and (o[g][~fin] == -INF).all()
        # the value in 64 bits but for a sum in 32 (its logarithm off by at most 5e-6), rounded once
        assert (np.abs(o[g][fin] - wo[fin]) <= 5e-6 + np.abs(wo[fin]) * 2.0 ** -24).all(), (o[g], wo)
        if f is not None:
            assert np.array_equal(d[g].cpu().numpy(), wd)
        if m is not None:
            assert np.array_equal(seen[g].cpu().numpy(), ws)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("G,B,V,pad,shift", [
    (1, 1, 1, 0, 0), (3, 1, 7, 0, 0), (2, 16, 1, 0, 0), (2, 5, 3, 2, 1), (1, 4, 1024, 0, 0), (65, 8, 1024, 0, 0),
    (7, 3, 2048, 64, 0), (2, 16, 997, 3, 3), (5, 8, 16385, 7, 1), (1, 16, 50021, 27, 5), (1, 1, 131071, 0, 0),
    (300, 2, 33, 0, 0), (2, 13, 8191, 1, 2),
])
def test_select_against_64_bits(dtype, G, B, V, pad, shift):
    rows, scores = case(G, B, V, dtype, 7 * V + B, pad, shift)
    check(rows, scores)
    end = (V - 1) // 2
    finished = (normal((G, B), 70) < -0.5).to(torch.int32)
    check(rows, scores, finished, end)


@pytest.mark.parametrize("V", [32, 1024, 4096])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_select_with_the_repetition_penalty(V, dtype):
    G, B = 9, 6
    rows, scores = case(G, B, V, dtype, V)
    words = masks((G, B, V // 32), 31)
    words[0] = 0
    words[1] = -1
    words[2] &= 0x0F0F0F0F
    check(rows, scores, seen=words, penalty=1.2)
    finished = (normal((G, B), 71) < -0.25).to(torch.int32)
    check(rows, scores, finished, 5, words, 0.8)


def test_one_beam_is_the_greedy_argmax():
    """With one beam the token is argmax_penalty's, and the seen masks end alike."""
    n, V = 40, 1024
    rows, _ = case(n, 1, V, "f32", 3)
    seen = masks((n, 1, V // 32), 31)
    other = seen.clone().view(n, V // 32)
    want = argmax_penalty(rows.reshape(n, V).contiguous(), other, 1.2)
    p, t, o, d = beam_select(rows, torch.zeros(n, 1, device=DEV), seen=seen, penalty=1.2)
    torch.cuda.synchronize()
    assert torch.equal(t.flatten(), want) and torch.equal(seen.view(n, -1), other) and (p == 0).all() and d is None


def test_rows_past_32_bits():
    """Rows that start more than 2^31 elements behind the first."""
    G, B, V, stride = 5, 7, 700, 1 << 26
    flat = torch.empty(G * B * stride, device=DEV, dtype=torch.bfloat16)
    rows = flat.view(G, B, stride)[:, :, :V]
    rows.copy_(normal((G, B, V), 8, 3.0))
    check(rows, -normal((G, B), 9).abs())


@pytest.mark.parametrize("where", ["rising", "falling", "last", "first"])
def test_where_the_largest_stand(where):
    """Rows sorted either way (the reference of the sum moves, every batch beats the last) and rows whose largest
    codes stand in the first or last few places."""
    G, B, V = 2, 9, 70001
    rows, scores = case(G, B, V, "f32", 4, 3, 1)
    if where in ("rising", "falling"):
        rows.copy_(rows.sort(-1, descending=where == "falling").values * 20)
    else:
        at = slice(V - 12, V) if where == "last" else slice(0, 12)
        rows[:, :, at] += 60
    check(rows, scores)


def test_ties_go_to_the_lowest_index():
    G, B, V = 4, 5, 1500
    rows = torch.zeros(G, B, V, device=DEV)
    scores = torch.zeros(G, B, device=DEV)
    rows[1] = torch.finfo(torch.float32).min          # every code at the type's lowest value: an even row
    rows[2, :, 700:720] = 2.0
    rows[3] = normal((V,), 1).round()                 # the same row, full of ties, in every beam
    check(rows, scores)
    check(rows.to(torch.bfloat16), scores)


def test_nothing_to_propose():
    """Rows masked altogether, rows holding NaN or +inf, dead beams, and groups with too few candidates."""
    G, B, V = 8, 4, 600
    rows, scores = case(G, B, V, "f32", 5)
    rows[0, 1] = -INF
    rows[1] = -INF
    rows[2, 0, 300] = math.nan
    rows[2, 3, 599] = INF
    rows[3, :, 3:] = -INF              # three codes a beam
    rows[4, 1:] = -INF
    rows[4, 0, 2:] = -INF              # two candidates for four beams
    scores[5, 1:] = -INF               # a first step
    scores[6, 2] = math.nan
    scores[6, 1] = INF
    rows[7, :, ::2] = torch.finfo(torch.float32).min
    check(rows, scores)
    finished = torch.zeros(G, B, dtype=torch.int32, device=DEV)
    finished[:, 0] = 1
    finished[1] = 1
    scores[1, 2] = -INF
    check(rows, scores, finished, 17)
    finished[6] = 1                    # finished hypotheses with scores that are none
    finished[5, 1] = 1
    check(rows, scores, finished, 17)
    seen = masks((G, B, 19), 31)
    check(rows[:, :, :576], scores, finished, 17, seen[:, :, :18].contiguous(), 1.3)


@pytest.mark.parametrize("V", [50, 4096, 40000])
def test_near_ties_across_beams_are_ordered_in_64_bits(V):
    """Beams whose candidates differ by less than a 32-bit sum resolves: equal rows in another order, with scores a
    few 32-bit steps apart.  The order is that of the 64-bit values."""
    G, B = 16, 8
    base = normal((G, 1, V), V, 2.0)
    rows = torch.cat([base[:, :, torch.randperm(V, generator=torch.Generator().manual_seed(b)).to(DEV)]
                      for b in range(B)], 1).contiguous()
    step = torch.randperm(B, generator=torch.Generator().manual_seed(1)).to(DEV)
    # near -1 a 32-bit step is 2^-24: far above what separates two orders of a 64-bit sum
    scores = (-1.0 + step * 2.0 ** -24).expand(G, B).contiguous().float()
    check(rows, scores)
    rows[:, 0, 0] = 12.0  # a peaked beam among them
    check(rows, scores)


def test_select_in_place_and_captured():
    """The C entry with scores_out = scores and finished_out = finished, and a captured step replayed."""
    G, B, V = 6, 4, 1024
    rows, scores = case(G, B, V, "f32", 9)
    fin = (normal((G, B), 70) < -0.5).to(torch.int32)
    p, t, o, d = beam_select(rows, scores, fin, 3)
    from mockbird_b200 import load
    lib = load()
    p2, t2, s2, f2 = torch.empty_like(p), torch.empty_like(t), scores.clone(), fin.clone()
    st = torch.cuda.current_stream().cuda_stream
    assert lib.mb_beam_select(G, B, V, 0, rows.data_ptr(), V, s2.data_ptr(), s2.data_ptr(), f2.data_ptr(),
                              f2.data_ptr(), 3, None, 1.0, p2.data_ptr(), t2.data_ptr(), st) == 0
    torch.cuda.synchronize()
    assert torch.equal(p, p2) and torch.equal(t, t2) and torch.equal(o, s2) and torch.equal(d, f2)
    x, s = rows.clone(), scores.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = beam_select(x, s, fin, 3)
    for seed in (10, 11):
        y, z = case(G, B, V, "f32", seed)
        x.copy_(y), s.copy_(z)
        g.replay()
        want = beam_select(y, z, fin, 3, stream=torch.cuda.current_stream())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def snapshot(ring):
    h = Held(ring)
    return h, h.kv.clone(), h.slot_pos.clone()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("G,B,C,L,H", [(1, 1, 5, 1, 1), (1, 2, 17, 2, 3), (3, 4, 130, 2, 12), (2, 5, 64, 3, 1),
                                       (2, 8, 257, 1, 4), (2, 16, 100, 2, 2), (1, 11, 33, 1, 5)])
def test_reorder(dtype, G, B, C, L, H):
    ring = KvRing(layers=L, heads=H, streams=G * B + 3, capacity=C, dtype=dtype, wrap=True, max_position=2048)
    r = random.Random(C)
    held, _, _ = snapshot(ring)
    held.kv.copy_(normal(held.kv.shape, C).to(held.kv.dtype))
    ids = list(range(G * B + 3))
    r.shuffle(ids)
    for i, s in enumerate(ids):
        base = [0, 3, C // 2, C, 2 * C + 1][i % 5]
        for layer in range(L):
            for p in range(max(0, base - C), base):
                held.slot_pos[layer, s, p % C] = p
    held.slot_pos[0, ids[0], ::3] = -1
    for trial in range(3):
        kv, sp = held.kv.clone(), held.slot_pos.clone()
        streams = [ids[g * B:(g + 1) * B] for g in range(G)]
        if trial == 0:
            parents = [[(k + 1) % B for k in range(B)] for _ in range(G)]       # a cycle
        else:
            parents = [[r.randrange(-1, B) for _ in range(B)] for _ in range(G)]
        ring.reorder(streams, parents)
        ring.sync()
        for row, up in zip(streams, parents):
            for k, s in enumerate(row):
                src = row[up[k]] if up[k] >= 0 else s
                live = (sp[:, src] >= 0)[:, None, None, :, None]
                kv_want = torch.where(live, kv[:, src], kv[:, s])
                assert torch.equal(held.kv[:, s], kv_want) and torch.equal(held.slot_pos[:, s], sp[:, src])
        for s in ids[G * B:]:
            assert torch.equal(held.kv[:, s], kv[:, s]) and torch.equal(held.slot_pos[:, s], sp[:, s])


def test_reorder_refusals():
    ring = KvRing(layers=1, heads=1, streams=8, capacity=20, dtype="f32", wrap=True, max_position=64)
    for s in range(8):
        fill(ring, 0, s, 12, s)
    held, kv, sp = snapshot(ring)
    for streams, parents, word in [([[0, 1], [2, 8]], [[1, 0], [1, 0]], "stream"),
                                   ([[0, 1], [2, -1]], [[1, 0], [1, 0]], "stream"),
                                   ([[0, 1], [2, 2]], [[1, 0], [1, 0]], "stream"),
                                   ([[0, 1], [2, 3]], [[1, 0], [1, 2]], "parent"),
                                   ([[0, 1], [2, 3]], [[1, 0], [-2, 0]], "parent")]:
        ring.reorder(streams, parents)
        with pytest.raises(MockbirdError, match=word):
            ring.sync()
        # the group that was right has moved, the other has not
        assert torch.equal(held.slot_pos[:, 2:], sp[:, 2:]) and torch.equal(held.kv[:, 2:], kv[:, 2:])
        ring.reorder([[0, 1]], [[1, 0]])  # and back
        ring.sync()
        assert torch.equal(held.kv, kv)
    with pytest.raises(MockbirdError, match="beam count"):
        ring.reorder([list(range(8)) + [0] * 9], [[0] * 17])
    with pytest.raises(MockbirdError, match="exceed"):
        ring.reorder([[0, 1, 2], [3, 4, 5], [6, 7, 0]], [[0] * 3] * 3)
    with pytest.raises(ValueError, match="streams"):
        ring.reorder([0, 1], [0, 1])
    with pytest.raises(ValueError, match="parents"):
        ring.reorder([[0, 1]], [[0]])
    with pytest.raises(TypeError):
        ring.reorder(torch.zeros(1, 2, dtype=torch.int64, device=DEV), [[0, 0]])
    assert ring.lib.mb_ring_reorder(ring.ctx, 1, 2, None, None, None) == 1
    ring.reorder(np.zeros((0, 2)), np.zeros((0, 2)))
    ring.sync()


def test_select_refusals():
    rows, scores = case(2, 3, 64, "f32", 0)
    fin = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    seen = torch.zeros(2, 3, 2, dtype=torch.int32, device=DEV)
    for kind, args in [(TypeError, (rows[0], scores)), (TypeError, (rows.double(), scores)),
                       (TypeError, (rows.cpu(), scores)), (TypeError, (rows.transpose(0, 1), scores)),
                       (TypeError, (rows.transpose(1, 2).contiguous().transpose(1, 2), scores)),
                       (TypeError, (rows, scores[:, :2])), (TypeError, (rows, scores.double())),
                       (TypeError, (rows, scores.cpu())), (TypeError, (rows, scores, fin.long(), 1)),
                       (TypeError, (rows, scores, None, -1, seen[:, :, :1], 1.2)),
                       (MockbirdError, (rows, scores, fin)), (MockbirdError, (rows, scores, fin, 64)),
                       (MockbirdError, (rows, scores, None, -2)), (MockbirdError, (rows, scores, None, -1, seen, 0.0)),
                       (MockbirdError, (rows, scores, None, -1, seen, math.nan)),
                       (TypeError, (rows[:, :1].expand(2, 3, 64), scores)),
                       (MockbirdError, (rows[0, 0].expand(2, 3, 64), scores)),
                       (MockbirdError, (torch.zeros(1, 17, 64, device=DEV), torch.zeros(1, 17, device=DEV))),
                       (MockbirdError, (rows[:, :, :40], scores, None, -1, seen[:, :, :1].contiguous(), 1.2))]:
        with pytest.raises(kind):
            beam_select(*args)


def test_beam_search_over_the_rings():
    """A beam search over rings, selection and reordering together, against a search that keeps whole sequences and
    attends them from scratch in 64 bits."""
    H, V, B, G, steps, L, end = 2, 48, 4, 3, 12, 2, 7
    ring = KvRing(layers=L, heads=H, streams=G * B, capacity=9, dtype="f32", wrap=True, max_position=64)
    w = H * HD
    emb = normal((L, V, 3 * w), 1)                      # a code's qkv row in each layer
    head = normal((L * w, V), 2, 0.4)
    ids = torch.arange(G * B, dtype=torch.int32, device=DEV).view(G, B)
    tok = torch.arange(G, device=DEV, dtype=torch.int64)[:, None].expand(G, B).contiguous()
    scores = torch.full((G, B), -INF, device=DEV)
    scores[:, 0] = 0
    fin = torch.zeros(G, B, dtype=torch.int32, device=DEV)
    seqs = [[([g], 0.0, 0)] + [([g], -INF, 0)] * (B - 1) for g in range(G)]
    e64, h64 = emb.double().cpu().numpy(), head.double().cpu().numpy()
    inv = 10000.0 ** (-np.arange(0, HD, 2) / HD)

    def turn(x, p):
        z = (x[:, 0::2] + 1j * x[:, 1::2]) * np.exp(1j * p * inv)
        return np.stack((z.real, z.imag), -1).reshape(x.shape)

    def logits64(seq):
        outs = []
        for layer in range(L):
            rows = e64[layer][seq].reshape(len(seq), 3, H, HD)
            q = turn(rows[-1, 0], len(seq) - 1)
            k = np.stack([turn(rows[p, 1], p) for p in range(max(0, len(seq) - 9), len(seq))])
            v = rows[max(0, len(seq) - 9):, 2]
            for h in range(H):
                s = np.exp(k[:, h] @ q[h] / 8)
                outs.append((s / s.sum()) @ v[:, h])
        return np.concatenate(outs) @ h64

    for step in range(steps):
        pos = torch.full((G * B,), step, dtype=torch.int32, device=DEV)
        ctx = [ring.append_attend(layer, ids.view(-1), pos, emb[layer][tok.view(-1)].contiguous())
               for layer in range(L)]
        logits = (torch.cat(ctx, -1).double() @ head.double()).float().view(G, B, V)
        parents, tokens, scores, fin = beam_select(logits, scores, fin, end)
        ring.reorder(ids, parents)
        tok = tokens.long().clamp_min(0)
        for g in range(G):
            found = []
            for b, (seq, score, done) in enumerate(seqs[g]):
                if not math.isfinite(score):
                    continue
                if done:
                    found.append((score, b, end, seq, 1))
                    continue
                x = logits64(seq)
                lp = score + x - (x.max() + math.log(np.exp(x - x.max()).sum()))
                found += [(lp[j], b, j, seq, int(j == end)) for j in range(V)]
            found.sort(key=lambda f: -f[0])
            seqs[g] = [(seq + [j], s, d) for s, b, j, seq, d in found[:B]]
            # gaps between neighbours are far above the 32-bit attention's error, so the choices agree
            gaps = [found[i][0] - found[i + 1][0] for i in range(min(B, len(found) - 1))]
            assert min(gaps) > 1e-4, "inputs with a near tie"
            assert [f[2] for f in found[:B]] == tokens[g].tolist() and [f[1] for f in found[:B]] == parents[g].tolist()
            assert np.allclose(scores[g].cpu().numpy(), [f[0] for f in found[:B]], rtol=0, atol=1e-3)
    ring.sync()


def test_trees_on_reordered_beams():
    """The operators together: hypotheses reordered, then a tree of drafts verified and committed on each."""
    H, B, T, C = 3, 3, 6, 24
    ring = KvRing(layers=1, heads=H, streams=B, capacity=C, dtype="f16", wrap=True, max_position=256)
    for s in range(B):
        fill(ring, 0, s, 30, s)
    ring.reorder([[0, 1, 2]], [[2, 2, 0]])
    trees = [tree_of("random", T, i) for i in range(B)]
    qkv = normal((B, T, 3 * H * HD), 4)
    qkv[1] = qkv[0]
    trees[1] = trees[0]
    out = ring.tree_attend(0, [0, 1, 2], [30] * B, trees, qkv)
    nxt = ring.tree_commit(0, [0, 1, 2], [30] * B, trees, [T - 1, T - 1, -1], qkv[None])
    ring.sync()
    assert torch.equal(out[0], out[1]) and not torch.equal(out[0], out[2])
    held = Held(ring)
    assert torch.equal(held.kv[:, 0], held.kv[:, 1]) and nxt[0] == nxt[1] and nxt[2] == 30
