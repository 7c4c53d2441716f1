"""Forms of the 4-bit products that sizes, types and jobs far from the usual ones select."""
import pytest

torch = pytest.importorskip("torch")

from test_q4 import _linear  # noqa: E402
from test_q4 import ea  # noqa: E402, F401  (the module's fixture)

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("ns", [[26000, 17], [26000, 48], [26000, 33, 5], [9000, 32, 26000], [9000, 40]])
@pytest.mark.parametrize("m", [1, 7, 16, 40])
def test_gpu_linear_narrow_job_beside_wide(ea, ns, m):  # noqa: F811
    """Linears of very different widths in one call: the widest one sets the tiles a block takes, and the others have fewer."""
    _linear(ea, m, 288, ns, 32, BF16, BF16, [F32, BF16, F16][:len(ns)], seed=sum(ns))
