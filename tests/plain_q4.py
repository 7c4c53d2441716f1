"""Plain forms, in 64 bits on the CPU, of general routing and of the products with 4-bit weights in groups, with bounds on
how far a 32-bit evaluation may be from them."""
from __future__ import annotations

import torch

HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}  # half a step of each type
U = 2.0**-23  # one fp32 addition inside a matrix instruction, whose rounding is not documented: a whole step


# ---- weights --------------------------------------------------------------------------------------------------------

def matrix(gen, shape, group, s_dtype, symmetric=False):
    """Random words int32 [.., n, k / 8], scales and biases [.., n, k / group] (biases None with `symmetric`)."""
    *lead, n, k = shape
    words = torch.randint(-(2**31), 2**31, (*lead, n, k // 8), generator=gen, dtype=torch.int64).to(torch.int32)
    scales = (0.01 * (0.5 + torch.rand((*lead, n, k // group), generator=gen))).to(s_dtype)
    biases = None if symmetric else (-0.08 + 0.02 * torch.randn((*lead, n, k // group), generator=gen)).to(s_dtype)
    return words, scales, biases


def values(words):
    """The integers [.., n, k] of words int32 [.., n, k / 8]."""
    w = words.to(torch.int64) & 0xFFFFFFFF
    return torch.stack([(w >> (4 * i)) & 15 for i in range(8)], dim=-1).flatten(-2)


def _spread(words, scales, biases):
    q = values(words).double()
    group = q.shape[-1] // scales.shape[-1]
    s = scales.double().repeat_interleave(group, -1)
    b = -8 * s if biases is None else biases.double().repeat_interleave(group, -1)
    return q, s, b, group


def dense(words, scales, biases):
    q, s, b, _ = _spread(words, scales, biases)
    return s * q + b


def product(x, m, dx=0.0):
    """x @ W^T in 64 bits, and the bound of its evaluation as s (sum of q x) + b (sum of x): every addition (a group's, the
    two a group that apply s and b, up to 16 partial sums) off by a step of the largest sum there can be; dx: a bound on the
    error of x itself."""
    q, s, b, group = _spread(*m)
    k = q.shape[-1]
    size = (s.abs() * q + b.abs()).t()
    steps = group + 2 * (k // group) + 16
    w = s * q + b
    err = steps * U * (x.abs() @ size)
    if not isinstance(dx, float):
        err = err + dx @ size
    return x @ w.t(), err


def experts(x, pick, wts, gate, up, down, out_dtype):
    """The routed experts of rows x in 64 bits, and the bound of the library's evaluation."""
    E, terms = gate[0].shape[0], {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}[out_dtype]
    at = lambda m, e: tuple(None if t is None else t[e] for t in m)  # noqa: E731
    out = torch.zeros(x.shape, dtype=torch.float64)
    err = torch.zeros(x.shape, dtype=torch.float64)
    for e in range(E):
        rows, slot = torch.nonzero(pick == e, as_tuple=True)
        if not rows.numel():
            continue
        g, dg = product(x[rows], at(gate, e))
        u, du = product(x[rows], at(up, e))
        act = g * torch.sigmoid(g)
        h = act * u
        # silu's slope is below 1.1; the exponential, the sum, the division and the product: 8 half steps; the terms
        dh = (1.1 * dg) * (u.abs() + du) + act.abs() * du + (8 * 2.0**-24 + HALF[torch.bfloat16] ** terms) * h.abs()
        y, dy = product(h, at(down, e), dh)
        w = wts[rows, slot].double()[:, None]
        out.index_add_(0, rows, w * y)
        err.index_add_(0, rows, w.abs() * (dy + (pick.shape[1] + 1) * 2.0**-24 * y.abs()))
    return out, err


def close(got, want, err, what=""):
    """got, of its type, within err of want and its own rounding's half step (a value below the smallest normal number:
    half of the smallest step)."""
    t = got.dtype
    tiny = torch.finfo(t).tiny * torch.finfo(t).eps
    room = err + HALF[t] * (want.abs() + err) + tiny
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all(), what
    assert (off <= room).all(), f"{what}: off by {float((off / room).max()):.3g} of what is allowed"


# ---- routing --------------------------------------------------------------------------------------------------------

def _ranked(c, out):
    """Positions by choice: numbers from the largest, then NaN, then what is out; the lower one where equal."""
    big = sorted(range(len(c)), key=lambda i: (2 if out[i] else 1 if c[i] != c[i] else 0, 0.0 if out[i] or c[i] != c[i] else -c[i], i))
    return big


def route(logits, bias, slots, softmax, groups, top_groups, best, renorm, scale):
    x = logits.double().cpu()
    R, E = x.shape
    pick, wts = torch.full((R, slots), -1, dtype=torch.int32), torch.zeros((R, slots), dtype=torch.float64)
    for r in range(R):
        row = x[r]
        out = [v == float("-inf") for v in row.tolist()]
        if softmax:
            top = row.max()
            p = torch.exp(row - (0.0 if top == float("-inf") else top))
            score = p / p.sum()
        else:
            score = 1 / (1 + torch.exp(-row))
        c = (score if bias is None else score + bias.double().cpu()).tolist()
        size = E // groups
        if groups > 1:
            rank, empty = [], []
            for g in range(groups):
                lead = [i for i in _ranked(c[g * size:(g + 1) * size], out[g * size:(g + 1) * size])[:best]
                        if not out[g * size + i]]
                rank.append(sum(c[g * size + i] for i in lead))
                empty.append(not lead)
            kept = set(_ranked(rank, empty)[:top_groups])
            out = [o or i // size not in kept for i, o in enumerate(out)]
        got = [i for i in _ranked(c, out)[:slots] if not out[i]]
        w = score[got]
        if renorm:
            w = w / (w.sum() + 1e-20)
        pick[r, :len(got)] = torch.tensor(got, dtype=torch.int32)
        wts[r, :len(got)] = w * scale
    return pick, wts
