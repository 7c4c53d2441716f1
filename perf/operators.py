"""Routing to experts in its general form, products with 4-bit weights in groups, and routed experts with such weights, as
cases that can be timed and checked.

    own                    False: run() computes the plain forms; True: it calls ea_exl3
    listed()               the cases
    draw(rng)              one more case of the ranges they stand for
    prepare(case, seed)    inputs on the GPU, and the weights as the program keeps them
    run(state)             one pass; its outputs
    work(case)             the bytes and operations a pass cannot do without
    exact(case, seed)      the same outputs in 64-bit arithmetic

4-bit weights are stored as affine checkpoints have them: words int32 [N, K / 8] with value k of a row in bits
4 (k % 8) .. + 3 of word k / 8, scales and biases [N, K / group] in bf16 or fp16, W[n, k] = scale * q + bias.
"""
import math
import os
import sys

import torch

own = False

DTYPE = {"f16": 0, "bf16": 1, "f32": 2}
TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SCALE = 2.5  # the routed experts' factor


# ---- the cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # The routing of one decode step: 256 experts by sigmoid and a balance bias, 8 kept. Latency is all there is.
        dict(name="route_1row", kind="route", rows=1, experts=256, slots=8, score="sigmoid", bias=True, groups=1, top_groups=1,
             best=1, renorm=True, logits="f32", out=0, empty=0),
        # A decode window whose model limits a token to 4 of 8 groups of experts, each ranked by its two best.
        dict(name="route_groups_128rows", kind="route", rows=128, experts=256, slots=8, score="sigmoid", bias=True, groups=8,
             top_groups=4, best=2, renorm=True, logits="f32", out=0, empty=0),
        # A prompt on a softmax router with 16-bit logits and an odd number of experts, some of them not resident (their
        # logits -inf), the last rows of the batch empty.
        dict(name="route_softmax_777rows", kind="route", rows=777, experts=60, slots=4, score="softmax", bias=False, groups=1,
             top_groups=1, best=1, renorm=False, logits="bf16", out=7, empty=9),
        # A long prompt.
        dict(name="route_4096rows", kind="route", rows=4096, experts=256, slots=8, score="sigmoid", bias=True, groups=1,
             top_groups=1, best=1, renorm=True, logits="f32", out=0, empty=0),
        # The gate and up projections of a shared expert's share in a short window: the smallest weights.
        dict(name="linear_5rows_2x256", kind="linear", rows=5, k=6144, n=256, jobs=2, group=64, x="f16", y="f32", scales="f16"),
        # One projection of a decode step.
        dict(name="linear_1row_2048", kind="linear", rows=1, k=6144, n=2048, jobs=1, group=64, x="bf16", y="bf16", scales="bf16"),
        # A draft model's output head: one token, the weights' bandwidth.
        dict(name="linear_1row_65521", kind="linear", rows=1, k=6144, n=65521, jobs=1, group=64, x="bf16", y="f32", scales="bf16"),
        # A projection of a prompt chunk of an odd size.
        dict(name="linear_301rows_6144", kind="linear", rows=301, k=2048, n=6144, jobs=1, group=128, x="bf16", y="bf16",
             scales="bf16"),
        # The routed experts of one decode step: one of eight ranks' share of a layer (256 columns of every expert).
        dict(name="experts_1row", kind="experts", rows=1, experts=256, slots=8, dims=6144, width=256, group=64, x="bf16",
             y="f32", scales="bf16", skew=False, pad=0),
        # A speculative window: four sequences of four tokens, about a hundred distinct experts.
        dict(name="experts_16rows", kind="experts", rows=16, experts=256, slots=8, dims=6144, width=256, group=64, x="bf16",
             y="f32", scales="bf16", skew=False, pad=0),
        # A wider window, padded: the last rows pick nothing.
        dict(name="experts_67rows", kind="experts", rows=67, experts=256, slots=8, dims=6144, width=256, group=32, x="f16",
             y="f16", scales="f16", skew=False, pad=6),
        # A prompt chunk, unevenly routed.
        dict(name="experts_2048rows", kind="experts", rows=2048, experts=256, slots=8, dims=6144, width=256, group=64, x="bf16",
             y="bf16", scales="bf16", skew=True, pad=0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["route", "linear", "experts"])
    x = rng.choice(["bf16", "f16"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * max(2, _log_int(rng, 8, 512) // groups)
        top_groups = rng.randint(1, groups)
        slots = rng.randint(1, min(12, experts // groups * top_groups))
        rows = _log_int(rng, 1, 4096)
        return dict(kind=kind, rows=rows, experts=experts, slots=slots, score=rng.choice(["sigmoid", "softmax"]),
                    bias=rng.random() < 0.5, groups=groups, top_groups=top_groups, best=rng.choice([1, 2]),
                    renorm=rng.random() < 0.6, logits=rng.choice(["f32", "bf16", "f16"]),
                    out=rng.choice([0, 0, experts // 5]), empty=rng.choice([0, 0, rows // 7]))
    group = rng.choice([32, 64, 128])
    scales = rng.choice(["bf16", x])
    y = rng.choice(["f32", x])
    if kind == "linear":
        rows, jobs = _log_int(rng, 1, 512), rng.choice([1, 1, 2, 3])
        return dict(kind=kind, rows=rows, k=group * _log_int(rng, 2, 8192 // group), n=_log_int(rng, 1, 12000), jobs=jobs,
                    group=group, x=x, y=y, scales=scales)
    experts = _log_int(rng, 4, 256)
    rows = _log_int(rng, 1, 1024)
    return dict(kind=kind, rows=rows, experts=experts, slots=rng.randint(1, min(8, experts)),
                dims=group * _log_int(rng, 2, 6144 // group), width=group * _log_int(rng, 1, 512 // group), group=group, x=x,
                y=y, scales=scales, skew=rng.random() < 0.5, pad=rng.choice([0, rows // 5]))


# ---- inputs and weights ---------------------------------------------------------------------------------------------

def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + what) & 0x7FFFFFFF)
    return g


def _quantize(gen, rows, k, group, scales):
    """N(0, 0.02) weights [rows, k] in 4 bits: words int32 [rows, k / 8], scales and biases [rows, k / group]."""
    words, sc, bi = [], [], []
    step = max(1, (1 << 26) // k)
    for r in range(0, rows, step):
        w = 0.02 * torch.randn((min(step, rows - r), k // group, group), device="cuda", generator=gen)
        lo, hi = w.amin(2, keepdim=True), w.amax(2, keepdim=True)
        s, b = ((hi - lo) / 15).to(TORCH[scales]), lo.to(TORCH[scales])
        q = ((w - b.float()) / s.float()).round_().clamp_(0, 15).to(torch.uint8).reshape(-1, k // 2, 2)
        words.append((q[..., 0] | (q[..., 1] << 4)).view(torch.int32))  # bytes in order, low half first
        sc.append(s[..., 0])
        bi.append(b[..., 0])
    return torch.cat(words), torch.cat(sc), torch.cat(bi)


def _linear_weights(case, seed):
    gen = _gen(seed, 31)
    return [_quantize(gen, case["n"], case["k"], case["group"], case["scales"]) for _ in range(case["jobs"])]


def _expert_weights(case, seed):
    """gate, up [E, I, D] and down [E, D, I], each as words, scales and biases."""
    gen, E = _gen(seed, 33), case["experts"]
    mats = []
    for n, k in ((case["width"], case["dims"]), (case["width"], case["dims"]), (case["dims"], case["width"])):
        w, s, b = _quantize(gen, E * n, k, case["group"], case["scales"])
        mats.append((w.reshape(E, n, -1), s.reshape(E, n, -1), b.reshape(E, n, -1)))
    return mats


def _activations(case, seed, k):
    return torch.randn((case["rows"], k), device="cuda", generator=_gen(seed, 11)).to(TORCH[case["x"]])


def _logits(case, seed):
    """Router logits ~ N(0, 1.5), a bias ~ N(0, 0.05); the logits of `out` experts -inf, and whole rows at the end."""
    gen, E = _gen(seed, 21), case["experts"]
    x = (1.5 * torch.randn((case["rows"], E), device="cuda", generator=gen)).to(TORCH[case["logits"]])
    if case["out"]:
        x[:, torch.randperm(E, device="cuda", generator=gen)[:case["out"]]] = -math.inf
    if case["empty"]:
        x[case["rows"] - case["empty"]:] = -math.inf
    return x, (0.05 * torch.randn(E, device="cuda", generator=gen) if case["bias"] else None)


def _picks(case, seed):
    """Distinct experts int32 [rows, slots] and weights [rows, slots] that sum to SCALE; with `skew` by a Zipf(1.1)
    popularity. The last `pad` rows pick nothing (-1)."""
    gen, R, E = _gen(seed, 22), case["rows"], case["experts"]
    u = torch.rand((R, E), device="cuda", generator=gen).clamp_min(1e-20)
    score = -torch.log(-torch.log(u))
    if case["skew"]:
        rank = torch.randperm(E, device="cuda", generator=gen)
        score -= 1.1 * torch.log(1.0 + rank.float())
    pick = torch.topk(score, case["slots"], dim=1).indices.to(torch.int32).contiguous()
    w = torch.rand((R, case["slots"]), device="cuda", generator=gen) * 0.95 + 0.05
    w = (w / w.sum(1, keepdim=True) * SCALE).contiguous()
    if case["pad"]:
        pick[R - case["pad"]:] = -1
        w[R - case["pad"]:] = 0
    return pick, w


class _State:
    """What one case keeps, by name."""

    def __init__(self, case):
        self.case = case


def prepare(case, seed):
    s, kind, R = _State(case), case["kind"], case["rows"]
    if kind == "route":
        s.logits, s.bias = _logits(case, seed)
        s.pick = torch.zeros((R, case["slots"]), dtype=torch.int32, device="cuda")
        s.wts = torch.zeros((R, case["slots"]), device="cuda")
    elif kind == "linear":
        s.x = _activations(case, seed, case["k"])
        s.weights = _linear_weights(case, seed)
        s.y = [torch.zeros((R, case["n"]), dtype=TORCH[case["y"]], device="cuda") for _ in s.weights]
    else:
        s.x = _activations(case, seed, case["dims"])
        s.pick, s.wts = _picks(case, seed)
        s.weights = _expert_weights(case, seed)
        s.out = torch.zeros((R, case["dims"]), dtype=TORCH[case["y"]], device="cuda")
    if own:
        _library(s)
    return s


def _library(s):
    """The weights in the library's layout, as a program makes them when it loads a model, instead of the checkpoint's."""
    sys.path.insert(0, os.path.join(os.getcwd(), "expertatlas-glm5.3_amd"))
    from ea_exl3 import device, q4

    device.init(0)
    case = s.case
    if case["kind"] == "linear":
        s.weights = [q4.Linear(*w) for w in s.weights]
    elif case["kind"] == "experts":
        s.weights = q4.Experts(*s.weights)
        s.scratch = q4.Scratch(s.weights, case["rows"], case["slots"])


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _call(s)
    kind = s.case["kind"]
    return _plain_route(s) if kind == "route" else _plain_linear(s) if kind == "linear" else _plain_experts(s)


def _call(s):
    from ea_exl3 import device, ops, q4

    case, q, R = s.case, device.stream(), s.case["rows"]
    if case["kind"] == "route":
        ops.route(q, s.logits.data_ptr(), DTYPE[case["logits"]], case["experts"], device.addr(s.bias), s.pick.data_ptr(),
                  s.wts.data_ptr(), R, case["experts"], case["slots"],
                  score=ops.SIGMOID if case["score"] == "sigmoid" else ops.SOFTMAX, groups=case["groups"],
                  top_groups=case["top_groups"], group_best=case["best"], renorm=case["renorm"], scale=SCALE)
        return {"pick": s.pick, "wts": s.wts}
    if case["kind"] == "linear":
        q4.call(q, s.weights, s.x.data_ptr(), DTYPE[case["x"]], case["k"], R, [y.data_ptr() for y in s.y],
                [DTYPE[case["y"]]] * len(s.y))
        return s.y
    q4.routed(q, s.x.data_ptr(), DTYPE[case["x"]], case["dims"], s.pick.data_ptr(), s.wts.data_ptr(), s.weights, s.scratch,
              s.out.data_ptr(), DTYPE[case["y"]], R)
    return s.out


def _plain_route(s):
    # in 64 bits: neighbouring choices can lie closer than a 32-bit sigmoid's error, and the picks are whole numbers
    case = s.case
    R, E, G = s.logits.shape[0], s.logits.shape[1], case["groups"]
    x = s.logits.double()
    off = x == -math.inf
    if case["score"] == "sigmoid":
        score = 1 / (1 + torch.exp(-x))
    else:
        top = x.amax(1, keepdim=True)
        p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
        score = p / p.sum(1, keepdim=True)
    choice = score if s.bias is None else score + s.bias.double()
    choice = torch.where(off, -math.inf, choice)
    if G > 1:
        lead = torch.sort(choice.reshape(R, G, E // G), dim=2, descending=True).values[:, :, :case["best"]]
        rank = torch.where(lead == -math.inf, 0.0, lead).sum(2)
        rank = torch.where(lead[:, :, 0] == -math.inf, -math.inf, rank)
        kept = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        mask = torch.zeros((R, G), dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        choice = torch.where(mask[:, :, None], choice.reshape(R, G, E // G), -math.inf).reshape(R, E)
    best, pick = torch.sort(choice, dim=1, descending=True, stable=True)  # the lower expert first where equal
    best, pick = best[:, :case["slots"]], pick[:, :case["slots"]]
    w = torch.where(best == -math.inf, 0.0, torch.gather(score, 1, pick))
    if case["renorm"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return {"pick": torch.where(best == -math.inf, -1, pick).to(torch.int32), "wts": (w * SCALE).float()}


def _dense(words, scales, biases):
    """4-bit weights [.., N, K] in fp32."""
    shift = torch.arange(0, 32, 4, dtype=torch.int32, device=words.device)
    q = ((words.unsqueeze(-1) >> shift) & 15).reshape(*scales.shape, -1).float()
    return (scales.float().unsqueeze(-1) * q + biases.float().unsqueeze(-1)).flatten(-2)


def _plain_linear(s):
    return [(s.x.float() @ _dense(*w).t()).to(y.dtype) for w, y in zip(s.weights, s.y)]


def _plain_experts(s):
    x, E = s.x.float(), s.case["experts"]
    out = torch.zeros(s.out.shape, device=x.device)
    if s.pick.numel() <= E:  # few picks: each one's matrices
        for j in range(s.pick.shape[1]):
            e = s.pick[:, j].long()
            at = e.clamp_min(0)
            gate, up, down = (_dense(*(t[at] for t in m)) for m in s.weights)
            g, u = torch.matmul(gate, x[:, :, None]), torch.matmul(up, x[:, :, None])
            y = torch.matmul(down, g / (1 + torch.exp(-g)) * u)[:, :, 0]
            out += torch.where((e >= 0)[:, None], s.wts[:, j, None] * y, 0.0)
        return out.to(s.out.dtype)
    for e in range(E):  # many: every expert on every row, weighted where the row picked it
        gate, up, down = (_dense(*(t[e] for t in m)) for m in s.weights)
        g, u = x @ gate.t(), x @ up.t()
        out += torch.where(s.pick == e, s.wts, 0.0).sum(1)[:, None] * ((g / (1 + torch.exp(-g)) * u) @ down.t())
    return out.to(s.out.dtype)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

_SIZE = {"f16": 2, "bf16": 2, "f32": 4}


def _matrix_bytes(n, k, group):
    return n * k // 2 + n * (k // group) * 4


def work(case):
    R = case["rows"]
    if case["kind"] == "route":
        E = case["experts"]
        return {"bytes": R * (E * _SIZE[case["logits"]] + case["slots"] * 8) + (E * 4 if case["bias"] else 0),
                "flops": R * E * 8}
    if case["kind"] == "linear":
        k, n, j = case["k"], case["n"], case["jobs"]
        return {"bytes": j * _matrix_bytes(n, k, case["group"]) + R * k * 2 + j * R * n * _SIZE[case["y"]],
                "flops": 2 * j * R * k * n}
    live, E, S = R - case["pad"], case["experts"], case["slots"]
    if case["skew"]:  # experts that `live` rows are expected to touch
        p = [(1.0 + r) ** -1.1 for r in range(E)]
        touched = sum(1 - max(0.0, 1 - S * v / sum(p)) ** live for v in p)
    else:
        touched = E * (1 - (1 - S / E) ** live)
    D, I, g = case["dims"], case["width"], case["group"]
    return {"bytes": int(touched * (2 * _matrix_bytes(I, D, g) + _matrix_bytes(D, I, g))) + R * (D * (2 + _SIZE[case["y"]]) + S * 8),
            "flops": 6 * live * S * D * I}


# ---- the same in 64-bit arithmetic ----------------------------------------------------------------------------------

def _values(words, scales, biases):
    """The weights in float64 from the words' bytes (two values a byte, the low half first)."""
    byte = words.contiguous().view(torch.uint8)
    q = torch.stack([byte & 15, byte >> 4], dim=-1).flatten(-2).double()
    group = q.shape[-1] // scales.shape[-1]
    return q * scales.double().repeat_interleave(group, -1) + biases.double().repeat_interleave(group, -1)


def _exact_route(case, logits, bias):
    x = logits.double().cpu()
    b = torch.zeros(case["experts"], dtype=torch.float64) if bias is None else bias.double().cpu()
    live = torch.isfinite(x)
    score = torch.special.expit(x)
    if case["score"] == "softmax":
        score = torch.exp(x - torch.logsumexp(torch.where(live.any(1, keepdim=True), x, torch.zeros(())), 1, keepdim=True))
    key = torch.where(live, score + b, torch.full_like(x, -1e300))
    if case["groups"] > 1:
        member = torch.arange(case["experts"]) // (case["experts"] // case["groups"])
        value = torch.empty((x.shape[0], case["groups"]), dtype=torch.float64)
        for g in range(case["groups"]):
            k, n = key[:, member == g], live[:, member == g].sum(1)
            first = k.amax(1)
            second = k.scatter(1, k.argmax(1, keepdim=True), -1e300).amax(1)
            value[:, g] = first + (torch.where(n > 1, second, torch.zeros(())) if case["best"] == 2 else 0)
        # a group is kept if fewer than top_groups others rank before it
        before = (value[:, None, :] > value[:, :, None]) | ((value[:, None, :] == value[:, :, None])
                                                           & (torch.arange(case["groups"])[None, :] < torch.arange(case["groups"])[:, None]))
        live = live & (before.sum(2) < case["top_groups"])[:, member]
        key = torch.where(live, key, torch.full_like(x, -1e300))
    picks, weights = [], []
    for _ in range(case["slots"]):
        e = key.argmax(1)  # equal choices to the last bit do not occur in the inputs, but among the experts left out
        ok = live.gather(1, e[:, None])[:, 0]
        picks.append(torch.where(ok, e, -1))
        weights.append(torch.where(ok, score.gather(1, e[:, None])[:, 0], torch.zeros((), dtype=torch.float64)))
        key.scatter_(1, e[:, None], -2e300)
        live = live.scatter(1, e[:, None], False)
    w = torch.stack(weights, 1)
    if case["renorm"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    # 16-bit logits do tie, and the picks are compared with the plain form's: only the weights, the same either way, are given
    return {"pick": None, "wts": (w * SCALE).cuda()}


def exact(case, seed):
    if case["kind"] == "route":
        return _exact_route(case, *_logits(case, seed))
    if case["kind"] == "linear":
        x = _activations(case, seed, case["k"]).double()
        return [torch.matmul(_values(*w), x.t()).t() for w in _linear_weights(case, seed)]
    x = _activations(case, seed, case["dims"]).double()
    pick, wts = _picks(case, seed)
    mats = _expert_weights(case, seed)
    out = torch.zeros_like(x)
    for e in range(case["experts"]):
        rows, slot = torch.nonzero(pick == e, as_tuple=True)
        if rows.numel():
            gate, up, down = (_values(*(t[e] for t in m)) for m in mats)
            v = x[rows]
            h = torch.nn.functional.silu(v @ gate.t()) * (v @ up.t())
            out.index_add_(0, rows, (h @ down.t()) * wts[rows, slot].double()[:, None])
    return out
