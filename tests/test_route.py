"""ops.route (ea_route) against a plain form in 64 bits: the picks and empty slots exactly, the weights to their rounding."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

import plain_q4 as plain  # noqa: E402

INF, NAN = float("inf"), float("nan")


def _case(rows, experts, dtype, seed, bias=True, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn((rows, experts), generator=g)).to(dtype)
    return x, 0.1 * torch.randn(experts, generator=g) if bias else None


# ---- the plain form itself --------------------------------------------------------------------------------------------

def test_plain_route_by_hand():
    x = torch.tensor([[0.0, 2.0, 2.0, -INF, 1.0, NAN]])
    pick, w = plain.route(x, None, 6, False, 1, 1, 1, False, 1.0)
    assert pick.tolist() == [[1, 2, 4, 0, 5, -1]]  # a tie by the lower expert, NaN after every number, -inf never
    assert w[0, 5] == 0 and math.isnan(w[0, 4]) and abs(float(w[0, 3]) - 0.5) < 1e-15
    x = torch.tensor([[1.0, 0.0, 0.9, 0.8, -INF, 5.0, -INF, -INF]])
    # two best of runs of two: .73 + .5, .71 + .69, sigmoid(5) alone, nothing: run 1 and run 0
    pick, _ = plain.route(x, None, 4, False, 4, 2, 2, True, 1.0)
    assert pick.tolist() == [[0, 2, 3, 1]]
    pick, _ = plain.route(x, None, 2, False, 4, 1, 1, True, 1.0)  # by their best: run 2, which has one expert
    assert pick.tolist() == [[5, -1]]


# ---- refusals: all before anything runs ---------------------------------------------------------------------------------

def _refused(**kw):
    from ea_exl3._lib import EaError
    from ea_exl3 import ops

    a = dict(stream=0, logits=4096, l_dtype=2, l_stride=64, bias=0, pick=4096, wts=4096, rows=1, experts=64, slots=8)
    a.update(kw)
    with pytest.raises(EaError) as e:
        ops.route(**a)
    return e.value.code


@pytest.mark.parametrize("kw,code", [
    (dict(logits=0), 18), (dict(pick=0), 18), (dict(wts=0), 18), (dict(l_dtype=3), 18), (dict(l_dtype=-1), 18),
    (dict(score=2), 18), (dict(experts=0, l_stride=8), 18), (dict(slots=0), 18), (dict(experts=1025, l_stride=1025), 5),
    (dict(slots=33), 6), (dict(l_stride=63), 9), (dict(groups=0), 18), (dict(groups=65), 18), (dict(top_groups=2), 18),
    (dict(groups=4, top_groups=0), 18), (dict(groups=4, top_groups=2, group_best=3), 18),
    (dict(groups=4, top_groups=2, group_best=0), 18), (dict(groups=7, top_groups=2), 8),
    (dict(groups=16, top_groups=1, slots=5), 6), (dict(experts=7, slots=8), 6),
])
def test_route_refuses(kw, code):
    assert _refused(**kw) == code


def test_route_needs_init():
    if not torch.cuda.is_available():
        assert _refused() == 17


# ---- the kernel -----------------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def ea():
    from ea_exl3 import device, ops

    device.init(0)
    return device, ops


def _run(ea, x, bias, slots, softmax=False, groups=1, top_groups=1, best=1, renorm=True, scale=2.5, stride=None):
    device, ops = ea
    rows, E = x.shape
    stride = stride or E
    buf = torch.full((rows, stride), 77.0, dtype=x.dtype, device="cuda")  # what lies between rows would win every choice
    buf[:, :E] = x.cuda()
    db = None if bias is None else bias.float().cuda()
    pick = torch.full((rows + 1, slots), -5, dtype=torch.int32, device="cuda")
    wts = torch.full((rows + 1, slots), -5.0, device="cuda")
    code = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}[x.dtype]
    print(f"route {tuple(x.shape)} {x.dtype} slots={slots} softmax={softmax} groups={groups}/{top_groups}/{best}", flush=True)
    ops.route(device.stream(), buf.data_ptr(), code, stride, device.addr(db), pick.data_ptr(), wts.data_ptr(), rows, E,
              slots, ops.SOFTMAX if softmax else ops.SIGMOID, groups, top_groups, best, renorm, scale)
    torch.cuda.synchronize()
    assert (pick[rows] == -5).all() and (wts[rows] == -5).all()  # nothing behind the last row
    return pick[:rows].cpu(), wts[:rows].cpu()


def _check(ea, x, bias, slots, softmax=False, groups=1, top_groups=1, best=1, renorm=True, scale=2.5, stride=None):
    pick, wts = _run(ea, x, bias, slots, softmax, groups, top_groups, best, renorm, scale, stride)
    want_p, want_w = plain.route(x, bias, slots, softmax, groups, top_groups, best, renorm, scale)
    assert torch.equal(pick, want_p)
    nan = torch.isnan(want_w)
    assert torch.equal(torch.isnan(wts), nan)
    # 64-bit scores, rounded once: half an fp32 step and, far below it, the exponential's and the sums' 64-bit errors
    room = 2.0**-24 * want_w.abs() * (1 + 1e-6) + 1e-44
    assert ((wts.double() - want_w).abs()[~nan] <= room[~nan]).all()


ROWS = [1, 2, 5, 64]
EXPERTS = [1, 7, 60, 64, 65, 128, 200, 256, 384, 512, 1000, 1024]


@pytest.mark.gpu
@pytest.mark.parametrize("experts", EXPERTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("softmax", [False, True])
def test_gpu_route(ea, experts, dtype, softmax):
    for i, rows in enumerate(ROWS):
        x, bias = _case(rows, experts, dtype, experts + i, bias=i % 2 == 0)
        _check(ea, x, bias, min(experts, 8 if i else 32), softmax, renorm=i < 3, stride=experts + 3 * i)


@pytest.mark.gpu
@pytest.mark.parametrize("experts,groups,top,best,slots", [
    (256, 8, 4, 2, 8), (256, 8, 4, 1, 8), (60, 4, 1, 2, 15), (64, 64, 9, 2, 9), (1024, 64, 3, 2, 32), (6, 2, 1, 2, 3),
    (160, 8, 3, 1, 6), (12, 3, 3, 2, 12), (36, 12, 5, 2, 4)])
@pytest.mark.parametrize("softmax", [False, True])
def test_gpu_route_groups(ea, experts, groups, top, best, slots, softmax):
    for seed, rows in enumerate([1, 37]):
        x, bias = _case(rows, experts, torch.float32, 50 + seed)
        if seed:  # experts out: whole runs, runs with one left, whole rows
            g = torch.Generator().manual_seed(9)
            x[torch.rand(x.shape, generator=g) < 0.3] = -INF
            x[3] = -INF
            x[4, : experts - experts // groups] = -INF
            x[5, 1:] = -INF
        _check(ea, x, bias, slots, softmax, groups, top, best)


@pytest.mark.gpu
@pytest.mark.parametrize("softmax", [False, True])
def test_gpu_route_special_values(ea, softmax):
    E = 96
    x, bias = _case(12, E, torch.float32, 3)
    low = torch.finfo(torch.float32).min
    x[0] = 0.0                     # all equal: the lowest experts in order
    x[1] = -INF                    # nothing left
    x[2, 5:] = -INF                # fewer than the slots
    x[3] = low                     # the lowest number is a number
    x[4, ::2] = low
    x[5, 7] = NAN
    x[6] = NAN
    x[7, 90:] = NAN
    x[7, :85] = -INF
    x[8] = -900.0                  # scores of zero
    x[9] = 60.0                    # a sigmoid of one
    x[10, 11] = INF
    x[11, ::3] = -0.0
    for b in (None, bias, torch.zeros(E)):
        for groups, top, best in ((1, 1, 1), (4, 2, 2), (4, 4, 1)):
            _check(ea, x, b, 8, softmax, groups, top, best)
    b = bias.clone()
    b[3], b[4], b[5] = INF, -INF, NAN
    _check(ea, x, b, 32, softmax)
    _check(ea, x, b, 24, softmax, 4, 2, 2)


@pytest.mark.gpu
def test_gpu_route_choices_closer_than_32_bits(ea):
    """Choices that one 32-bit sigmoid could swap: logits a step apart under a bias that takes the difference back."""
    E = 64
    base = torch.linspace(-2, 2, E, dtype=torch.float64)
    up = torch.nextafter(base.float(), torch.tensor(9.0))
    x = torch.stack([base.float(), up, base.float().flip(0)])
    bias = (-torch.sigmoid(base.float().double())).float()  # every choice within 1e-7 of zero
    _check(ea, x, bias, 32)


@pytest.mark.gpu
def test_gpu_route_as_topk(ea):
    """The reference's router (sigmoid, bias, 8 of 256, renormalised): the same picks as ops.topk."""
    device, ops = ea
    x, bias = _case(333, 256, torch.float32, 8)
    pick, wts = _run(ea, x, bias, 8)
    dx, db = x.cuda(), bias.cuda()
    p, w = torch.zeros((333, 8), dtype=torch.int32, device="cuda"), torch.zeros((333, 8), device="cuda")
    ops.topk(device.stream(), dx.data_ptr(), db.data_ptr(), p.data_ptr(), w.data_ptr(), 333, 2.5)
    assert torch.equal(p.cpu(), pick)
    assert (w.cpu() - wts).abs().max() <= 16 * 2.0**-24 * 2.5  # its scores, sum and division are 32-bit
