"""Forms of the 4-bit products that sizes, types and jobs far from the usual ones select, and refusals of their weights."""
import pytest

torch = pytest.importorskip("torch")

import plain_q4 as plain  # noqa: E402
from test_q4 import _cuda, _experts, _layer, _linear, _routing  # noqa: E402
from test_q4 import ea  # noqa: E402, F401  (the module's fixture)

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("ns", [[26000, 17], [26000, 48], [26000, 33, 5], [9000, 32, 26000], [9000, 40]])
@pytest.mark.parametrize("m", [1, 7, 16, 40])
def test_gpu_linear_narrow_job_beside_wide(ea, ns, m):  # noqa: F811
    """Linears of very different widths in one call: the widest one sets the tiles a block takes, and the others have fewer."""
    _linear(ea, m, 288, ns, 32, BF16, BF16, [F32, BF16, F16][:len(ns)], seed=sum(ns))


@pytest.mark.gpu
@pytest.mark.parametrize("R", [1, 2, 5, 16, 23, 90, 12000])
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
def test_gpu_experts_narrowest(ea, R, out_dtype):  # noqa: F811
    """32 dims and 32 columns: two tiles of the output, one chunk that is a quarter full; from one row to long items."""
    g = torch.Generator().manual_seed(R)
    mats = _layer(g, 5, 32, 32, 32, BF16)
    x = torch.randn((R, 32), generator=g).to(BF16)
    pick, wts = _routing(g, R, 5, 3)
    out, _, _ = _experts(ea, x, pick, wts, mats, out_dtype, pad=4)
    want, err = plain.experts(x.double(), pick, wts, *mats, out_dtype)
    plain.close(out, want, err)


@pytest.mark.gpu
@pytest.mark.parametrize("E", [1023, 1024, 1025, 2048, 2500, 4096])
@pytest.mark.parametrize("R", [16, 40, 700])
def test_gpu_experts_many(ea, E, R):  # noqa: F811
    """More experts than the grouping scans in one step, picked on both sides of each step's border and at the last one."""
    g = torch.Generator().manual_seed(E + R)
    mats = _layer(g, E, 32, 32, 32, BF16)
    x = torch.randn((R, 32), generator=g).to(BF16)
    pick, wts = _routing(g, R, E, 4)
    edges = torch.tensor([e for e in (0, 1022, 1023, 1024, 1025, 2047, 2048, 4095, E - 1) if e < E], dtype=torch.int32)
    pick[:, 0] = edges[torch.arange(R) % len(edges)]
    pick[R // 2:, 1] = E - 1
    if R > 600:
        pick[100:600, 2] = 1023  # many full items before the border
    for r in range(R):  # an expert once a row
        seen = set()
        for s in range(4):
            e = int(pick[r, s])
            pick[r, s] = -1 if e in seen else e
            seen.add(e)
    out, _, _ = _experts(ea, x, pick, wts, mats, F32)
    want, err = plain.experts(x.double(), pick, wts, *mats, F32)
    plain.close(out, want, err)


@pytest.mark.gpu
@pytest.mark.parametrize("x_dtype,s_dtype", [(BF16, F16), (F16, BF16)])
@pytest.mark.parametrize("E,D,I,group,slots,R", [
    (6, 256, 64, 64, 3, 1), (6, 320, 96, 32, 3, 7), (5, 384, 128, 128, 3, 16), (12, 256, 160, 32, 4, 50),
    (16, 256, 512, 64, 4, 1200), (16, 256, 512, 32, 4, 1200), (24, 128, 512, 128, 3, 1400), (8, 160, 1056, 32, 4, 900)])
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
def test_gpu_experts_scales_of_another_type(ea, x_dtype, s_dtype, E, D, I, group, slots, R, out_dtype):  # noqa: F811, E741
    g = torch.Generator().manual_seed(E + R)
    mats = _layer(g, E, D, I, group, s_dtype)
    x = torch.randn((R, D), generator=g).to(x_dtype)
    pick, wts = _routing(g, R, E, slots)
    out, _, _ = _experts(ea, x, pick, wts, mats, out_dtype, pad=4)
    want, err = plain.experts(x.double(), pick, wts, *mats, out_dtype)
    plain.close(out, want, err)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [2, 7, 16, 17, 90])
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
def test_gpu_experts_rows_in_another_order(ea, R, out_dtype):  # noqa: F811
    """A row's bits do not depend on the rows beside it or on their order, whichever place of an item its pairs get; nor on a
    smaller batch, down to two rows. Some rows name an expert twice."""
    g = torch.Generator().manual_seed(R)
    mats = _layer(g, 8, 256, 96, 32, BF16)
    x = torch.randn((R, 256), generator=g).to(BF16)
    pick, wts = _routing(g, R, 8, 3)
    pick[::3, 2] = pick[::3, 0]
    a, ex, sc = _experts(ea, x, pick, wts, mats, out_dtype)
    want, err = plain.experts(x.double(), pick, wts, *mats, out_dtype)
    plain.close(a, want, err)
    for _ in range(3):
        order = torch.randperm(R, generator=g)
        b, _, _ = _experts(ea, x[order], pick[order], wts[order], mats, out_dtype, ex=ex, sc=sc)
        assert torch.equal(a[order.cuda()], b)
    for n in (2, 3, 16, 17):
        if n < R:
            b, _, _ = _experts(ea, x[:n], pick[:n], wts[:n], mats, out_dtype, ex=ex, sc=sc)
            assert torch.equal(a[:n], b)


# ---- refusals of weights ------------------------------------------------------------------------------------------------

def _linear_source(**kw):
    g = torch.Generator().manual_seed(5)
    m = dict(zip(("words", "scales", "biases"), plain.matrix(g, (16, 256), 64, F16)))
    return {k: None if v is None else v.cuda() for k, v in (m | {k: f(m) for k, f in kw.items()}).items()}


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [
    dict(words=lambda m: m["words"][0]), dict(words=lambda m: m["words"].long()), dict(words=lambda m: m["words"][:8]),
    dict(scales=lambda m: m["scales"].float()), dict(scales=lambda m: m["scales"][:, :3]),
    dict(scales=lambda m: m["scales"][:, :1], biases=lambda m: m["biases"][:, :1]),
    dict(scales=lambda m: m["scales"].repeat(1, 4), biases=lambda m: m["biases"].repeat(1, 4)),
    dict(scales=lambda m: m["scales"][:, :0], biases=lambda m: m["biases"][:, :0]),
    dict(scales=lambda m: m["scales"][:9], biases=lambda m: m["biases"][:9]),
    dict(biases=lambda m: m["biases"].bfloat16()), dict(biases=lambda m: m["biases"][:, :2]),
    dict(biases=lambda m: m["biases"].T.contiguous())])
def test_gpu_linear_refuses_sources(ea, bad):  # noqa: F811
    q4 = ea[2]
    q4.Linear(**_linear_source())
    with pytest.raises(ValueError):
        q4.Linear(**_linear_source(**bad))


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2])
def test_gpu_linear_refuses_host_tensors(ea, which):  # noqa: F811
    m = list(_linear_source().values())
    m[which] = m[which].cpu()
    with pytest.raises(ValueError):
        ea[2].Linear(*m)


@pytest.mark.gpu
def test_gpu_experts_refuse_sources(ea):  # noqa: F811
    q4, g = ea[2], torch.Generator().manual_seed(6)
    E, D, I = 4, 128, 64  # noqa: E741

    def source(shape, group=64, t=BF16, symmetric=False):
        return _cuda(plain.matrix(g, shape, group, t, symmetric))

    gate, up, down = source((E, I, D)), source((E, I, D)), source((E, D, I))
    q4.Experts(gate, up, down)
    for bad in ((source((E, I, 2 * D)), up, down), (gate, source((E, 2 * I, D)), down), (gate, source((E - 1, I, D)), down),
                (gate, up, source((E + 1, D, I))), (gate, up, source((E, I, D))), (gate, up, source((E, D, 2 * I))),
                (gate, source((E, I, D), 32), down), (gate, up, source((E, D, I), 32)), (gate, source((E, I, D), t=F16), down),
                (gate, up, source((E, D, I), t=F16)), (gate, source((E, I, D), symmetric=True), down),
                (tuple(t[0] for t in gate), up, down), (gate, up, (down[0], down[1].cpu(), down[2]))):
        with pytest.raises(ValueError):
            q4.Experts(*bad)
    q4.Experts(gate, up, source((E, D, I), symmetric=True))  # down's are its own
