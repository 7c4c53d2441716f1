"""Routing of scores at the ends of their range."""
import pytest

torch = pytest.importorskip("torch")

from test_route import _check  # noqa: E402
from test_route import ea  # noqa: E402, F401  (the module's fixture)

INF = float("inf")


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
