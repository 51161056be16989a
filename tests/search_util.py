"""Plain 64-bit forms of the operators that search over continuations."""
import math

import numpy as np
import torch

import oracle

HD = 64
TORCH_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def rounded(a, dtype):
    """a (fp32 numpy) rounded to the storage type, as fp64."""
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(TORCH_DT[dtype]).double().numpy()


def path_to(parents, t):
    got = []
    while t >= 0:
        got.append(t)
        t = parents[t]
    return got[::-1]


def roped(rows, pos):
    """rows [m][H*64] fp32 at positions [m]: the table and the roundings every kernel uses (fp32, bit for bit)."""
    tab = oracle.rope_table(max(pos) + 1)
    return oracle.rope_rows(np.ascontiguousarray(rows, np.float32), list(pos), tab)


def attend_tree(k, v, slot_pos, base, parents, qkv, dtype, heads):
    """One item in 64 bits: k, v [H][C][64] fp64 (what the ring holds), qkv [T][3*H*64] fp32.

    Returns (out [T][H*64], bound [T][H*64]): the context, and a bound of an fp32 kernel's error of it.  The bound:
    a product of 64 terms, whatever its order and with operands held as parts that leave 2^-21 of each product,
    is within (64 + 8) 2^-24 of sum |q k|; so each weight is within e = 2 * 72 * 2^-24 * 0.125 * max sum |q k|
    (of the row and of its maximum) + 8 * 2^-24 (the scaling, the exponential) relative, the normalised weight
    within 2 e, and the sum over the slots adds (slots) roundings, at worst 2^-24 each, of partial sums whose
    magnitude is at most sum w |v|.
    """
    T, C = len(parents), slot_pos.shape[0]
    H = heads
    out = np.zeros((T, H * HD))
    bound = np.zeros((T, H * HD))
    there = [t for t in range(T) if parents[t] != -2]
    if not there:
        return out, bound
    paths = {t: path_to(parents, t) for t in there}
    pos = [base + (len(paths[t]) - 1 if t in paths else 0) for t in range(T)]
    q = roped(qkv[:, :H * HD], pos).reshape(T, H, HD).astype(np.float64)
    kd = rounded(roped(qkv[:, H * HD:2 * H * HD], pos), dtype).reshape(T, H, HD)
    vd = rounded(qkv[:, 2 * H * HD:], dtype).reshape(T, H, HD)
    for t in there:
        sel = [j for j in range(C) if 0 <= slot_pos[j] < base and pos[t] - slot_pos[j] < C]
        anc = [u for u in paths[t] if pos[t] - pos[u] < C]
        for h in range(H):
            kk = np.concatenate((k[h, sel], kd[anc, h]))
            vv = np.concatenate((v[h, sel], vd[anc, h]))
            s = kk @ q[t, h] * 0.125
            w = np.exp(s - s.max())
            w /= w.sum()
            out[t, h * HD:(h + 1) * HD] = w @ vv
            e = (2 * 72 * 0.125 * (np.abs(kk) @ np.abs(q[t, h])).max() + 8) * 2.0 ** -24
            bound[t, h * HD:(h + 1) * HD] = (2 * e + (len(w) + 4) * 2.0 ** -24) * (w @ np.abs(vv)) + 1e-30
    return out, bound


def select(logits, scores, finished=None, end_id=-1, seen=None, penalty=1.0):
    """One group in 64 bits: logits [B][V] fp32, scores [B].  Returns (parents, tokens, scores, finished, seen)."""
    B, V = logits.shape
    found = []
    for b in range(B):
        start = float(scores[b])
        if finished is not None and finished[b]:
            if math.isfinite(start):
                found.append((-start, b * V + end_id))
            continue
        x = logits[b].astype(np.float32)
        if seen is not None:
            on = ((seen[b].astype(np.int64)[:, None] >> np.arange(32)) & 1).reshape(-1).astype(bool)
            p = np.float32(penalty)
            with np.errstate(invalid="ignore", over="ignore"):
                x = np.where(on, np.where(x >= 0, x / p, x * p), x)
        x = x.astype(np.float64)
        if np.isnan(x).any() or np.isposinf(x).any() or np.isneginf(x).all():
            continue
        m = x.max()
        val = start + (x - (m + math.log(math.fsum(np.exp(x - m)))))
        with np.errstate(over="ignore"):
            ok = np.isfinite(val.astype(np.float32))
        at = np.nonzero(ok)[0]
        at = at[np.argsort(-val[at], kind="stable")][:B]
        found += [(-val[j], b * V + int(j)) for j in at]
    found = sorted(found)[:B]
    parents, tokens = np.full(B, -1, np.int32), np.full(B, -1, np.int32)
    out = np.full(B, -np.inf)
    done = None if finished is None else np.array(finished, np.int32)
    after = None if seen is None else np.array(seen)
    for k, (v, f) in enumerate(found):
        b, j = divmod(f, V)
        parents[k], tokens[k], out[k] = b, j, -v
        was = finished is not None and bool(finished[b])
        if done is not None:
            done[k] = int(was or j == end_id)
        if after is not None:
            after[k] = seen[b]
            if not was:
                after[k] = after[k].copy()
                after.view(np.uint32)[k, j // 32] |= np.uint32(1 << (j % 32))
    return parents, tokens, out, done, after
