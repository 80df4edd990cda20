"""4-bit matrices, logit rules and sampling restated in 64 bits for the tests."""
from __future__ import annotations

import numpy as np


def quantize(rng, rows, cols, group, scale_dtype="f16", zero=False, scale=0.04):
    """Packed bytes [rows, cols / 2], scales and zero points of random weights, and the float64
    matrix that they stand for. Scales are numpy float32/float16, or bfloat16 as float32."""
    groups = -(-cols // group)
    q = rng.integers(0, 16, (rows, cols), dtype=np.uint8)
    s = (rng.random((rows, groups)) * scale + scale / 4).astype(np.float32)
    if scale_dtype == "f16":
        s = s.astype(np.float16)
    elif scale_dtype == "bf16":
        s = (s.view(np.uint32) & 0xFFFF0000).view(np.float32)
    z = rng.integers(0, 16, (rows, groups), dtype=np.uint8) if zero else None
    return (q[:, 0::2] | (q[:, 1::2] << 4)), s, z, dense(q, s, z, group)


def dense(q, s, z, group):
    cols = q.shape[1]
    wide = lambda a: np.repeat(a.astype(np.float64), group, 1)[:, :cols]
    return (q.astype(np.float64) - (8.0 if z is None else wide(z))) * wide(s)


def sum_tolerance(cols, group, w, x):
    """How far an f32 sum of w . x may be from the exact one, per output [T, rows]: roundings of
    2^-24 of the sum of |w x| each. A group is 4 steps x 2 parts of matrix products, counted as 4
    roundings each at most; then one fma per group of a slot and one sum per slot; 2 for the
    activations' 23 bits, 2 for scale and output."""
    blocks = -(-cols // 128)
    depth = 32 + -(-blocks // 8) * (128 // group) + 8 + 4
    return depth * 2.0 ** -24 * (np.abs(x).astype(np.float64) @ np.abs(w).T)


def adjust(logits, rules, dtype=np.float32):
    """The rules of ie_hip_adjust_logits step by step in `dtype`."""
    out = logits.astype(dtype).copy()
    R, n = out.shape
    get = lambda k, r, d: dtype(d) if rules.get(k) is None else dtype(rules[k][r])
    for r in range(R):
        if rules.get("history") is not None:
            ids, start, length = rules["history"]
            plen = 0 if rules.get("prompt_len") is None else int(rules["prompt_len"][r])
            count, seen = {}, set()
            for i in range(int(length[r])):
                e = int(start[r]) + i
                if not 0 <= e < ids.size:
                    continue
                t = int(ids.flat[e])
                if not 0 <= t < n:
                    continue
                seen.add(t)
                if i >= plen:
                    count[t] = count.get(t, 0) + 1
            rep, pres, freq = get("repetition", r, 1), get("presence", r, 0), get("frequency", r, 0)
            for t in seen:
                l, c = out[r, t], count.get(t, 0)
                l = l / rep if l > 0 else l * rep
                l = l - freq * dtype(c)
                out[r, t] = l - (pres if c else dtype(0))
        if rules.get("bias") is not None:
            tok, val, start, length = rules["bias"]
            last = {}
            for i in range(int(length[r])):
                e = int(start[r]) + i
                if 0 <= e < tok.size and 0 <= int(tok.flat[e]) < n:
                    last[int(tok.flat[e])] = dtype(val.flat[e])
            for t, v in last.items():
                out[r, t] = out[r, t] + v
        if rules.get("mask") is not None:
            m = r if rules.get("mask_row") is None else int(rules["mask_row"][r])
            if 0 <= m < rules["mask"].shape[0]:
                on = np.unpackbits(rules["mask"][m].view(np.uint8), bitorder="little")[:n]
                out[r, on == 0] = -np.inf
    return out


def sample(l, temperature, u, top_k=0, top_p=1.0, min_p=0.0):
    """One row's token by the definition, in 64 bits over a sorted row."""
    l = np.where(np.isnan(l), -np.inf, l).astype(np.float64) + 0.0
    n = l.size
    order = np.argsort(-l, kind="stable")
    top = l[order[0]]
    if not temperature > 0 or top == -np.inf:
        return int(order[0])
    if top == np.inf:
        w = (l == np.inf).astype(np.float64)
    else:
        with np.errstate(over="ignore"):
            w = np.where(l == -np.inf, 0.0, np.exp((l - top) / np.float64(np.float32(temperature))))
    keep = n if top_k <= 0 or top_k >= n else int(top_k)
    if min_p > 0:
        keep = min(keep, int((w >= min(float(np.float32(min_p)), 1.0)).sum()))
    if top_p < 1:
        if top_p <= 0:
            keep = 1
        else:
            sums = np.concatenate(([0.0], np.cumsum(w[order[:keep]])))
            keep = int((sums[:-1] < float(np.float32(top_p)) * sums[-1]).sum())
    kept = np.zeros(n, bool)
    kept[order[:keep]] = True
    sums = np.cumsum(np.where(kept, w, 0.0))
    u = float(np.float32(u))
    u = 0.0 if not u > 0 else min(u, 1 - 2.0 ** -24)
    return int((sums <= u * sums[-1]).sum())
