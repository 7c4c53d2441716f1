"""Routing of many rows, which half a wave takes each, and scores at the ends of their range."""
import pytest

torch = pytest.importorskip("torch")

import plain_q4 as plain  # noqa: E402
from test_route import _case, _check, _run  # noqa: E402
from test_route import ea  # noqa: E402, F401  (the module's fixture)

INF, NAN = float("inf"), float("nan")


def _sampled(x, pick, wts, rows, bias, slots, softmax, renorm):
    """The plain form at some rows: picks exactly, weights as in test_route."""
    want_p, want_w = plain.route(x[rows], bias, slots, softmax, 1, 1, 1, renorm, 2.5)
    got = wts[rows].double()
    assert torch.equal(pick[rows], want_p)
    nan = torch.isnan(want_w)
    assert torch.equal(torch.isnan(got), nan)
    room = 2.0**-24 * want_w.abs() * (1 + 1e-6) + 1e-44
    assert ((got - want_w).abs()[~nan] <= room[~nan]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,experts,slots", [(4096, 256, 8), (4097, 256, 32), (4103, 200, 8), (4096, 128, 1), (5001, 65, 32),
                                                (4099, 64, 9), (4098, 33, 32), (6000, 7, 5), (4097, 1, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("softmax", [False, True])
def test_gpu_route_many_rows(ea, rows, experts, slots, dtype, softmax):  # noqa: F811
    """Rows of equal logits, of NaN, with experts out, with nothing left and with ties, each beside ordinary ones; every row also
    as fewer rows give it, where a wave takes one."""
    bias = experts % 2 == 0
    x, b = _case(rows, experts, dtype, rows + experts, bias=bias)
    x[5::31] = 0.5                                      # ties all through
    x[7::37, ::2] = -INF
    x[9::41] = -INF
    x[10::43, 0] = NAN
    x[12::47] = NAN
    x[13::53, -1] = INF if not softmax else 40.0
    x[14::59] = (x[14::59] * 2).round() / 2             # a few values each, many times
    x[rows - 1] = -x[rows - 2]
    renorm = dtype != torch.bfloat16
    pick, wts = _run(ea, x, b, slots, softmax, renorm=renorm, stride=experts + 5)
    few = torch.unique(torch.cat([torch.arange(0, 66), torch.arange(rows - 9, rows), torch.arange(66, rows, 97)]))
    _sampled(x, pick, wts, few, b, slots, softmax, renorm)
    for lo in range(0, rows, 2000):
        p, w = _run(ea, x[lo:lo + 2000], b, slots, softmax, renorm=renorm)
        assert torch.equal(pick[lo:lo + 2000], p)
        nan = torch.isnan(w)
        assert torch.equal(torch.isnan(wts[lo:lo + 2000]), nan)
        # both within half a step of the 64-bit value
        assert ((wts[lo:lo + 2000].double() - w.double()).abs()[~nan] <= 2.0**-23 * w.double().abs()[~nan] * (1 + 1e-6) + 1e-44).all()


@pytest.mark.gpu
def test_gpu_route_scores_at_the_ends(ea):  # noqa: F811
    """Sigmoids down to the smallest numbers that 64 bits hold are still in order, and softmax's scores as far apart."""
    E = 64
    g = torch.Generator().manual_seed(17)
    order = torch.stack([torch.randperm(E, generator=g) for _ in range(6)])
    lows = torch.stack([torch.linspace(-709.782, -709.0, E), torch.linspace(-709.0, -690.0, E), torch.linspace(-720.0, -100.0, E),
                        torch.linspace(-100.0, 0.0, E), torch.linspace(-40.0, 30.0, E), torch.linspace(5.0, 33.0, E)])
    x = torch.gather(lows.float(), 1, order)
    x[2][x[2] < -709.78] = -INF
    for renorm in (False, True):
        _check(ea, x, None, 32, False, renorm=renorm)
    _check(ea, x, None, 32, True)
