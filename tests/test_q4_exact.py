"""Routed experts with 4-bit weights on integers whose every product and sum is exact in fp32, so that the result is the
integers' own: a rounding that the library does not state, of the activated values above all, shows as another number."""
import pytest

torch = pytest.importorskip("torch")

import plain_q4 as plain  # noqa: E402
from test_q4 import _cuda, _experts  # noqa: E402
from test_q4 import ea  # noqa: E402, F401  (the module's fixture)

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TERMS = {BF16: 2, F16: 2, F32: 3}  # bf16 numbers that an activated value is held as, by the output's type


def _ints(gen, shape, group, lo, hi, bias, scale, s_dtype):
    """Weights scale * (q + bias) with q in lo .. hi, as words, scales and biases."""
    *lead, n, k = shape
    q = torch.randint(lo, hi + 1, shape, generator=gen, dtype=torch.int64)
    nibble = q.reshape(*lead, n, k // 8, 8) << torch.arange(0, 32, 4)
    word = nibble.sum(-1)
    words = torch.where(word >= 2**31, word - 2**32, word).to(torch.int32)
    s = torch.full((*lead, n, k // group), scale, dtype=s_dtype)
    return words, s, torch.full_like(s, bias * scale)


LOUD = slice(8, 16)  # columns of x, and what they hold: 8 bits each, their sum 19
LOUD_X = torch.tensor([255 * 256, 253 * 256, 191 * 256, 129 * 256, 251 * 128, 247 * 64, 243 * 32, 239 * 16])


def _fill(m, columns, q):
    """The integers of some columns, in whole words, set to q."""
    words = m[0].clone()
    words[..., columns.start // 8:columns.stop // 8] = sum(q << (4 * i) for i in range(8)) - (2**32 if q >= 8 else 0)
    return words, m[1], m[2]


def _case(seed, E, D, I, group, slots, R, s_dtype, out_dtype, loud=False):
    """x in 0 .. 2, gate sums large and positive (silu(g) = g there: 1 + exp(-g) is 1 from g = 18 on), up sums of either sign
    in a few of the columns and zero in the others; down weights -1, 0 and 1 over 256. With fp32 out the activated values have up
    to 20 bits, else up to 14. With `loud`, half of the rows have eight large columns, whose weights are zero: s (sum of q x)
    and b (sum of x) cancel there, numbers of 19 bits and more."""
    g = torch.Generator().manual_seed(seed)
    wide = out_dtype == F32
    x = torch.randint(0, 3, (R, D), generator=g) * (torch.rand((R, D), generator=g) < (64 if wide else 160) / D)
    x[:, ::max(1, D // 32)] = 1  # no row's gate sum is small
    gate = _ints(g, (E, I, D), group, 2, 15 if wide else 3, -1, 1.0, s_dtype) if loud else \
        _ints(g, (E, I, D), group, 0, 15 if wide else 1, 1, 1.0, s_dtype)
    up = _ints(g, (E, I, D), group, 0, 14 if wide else 2, -7 if wide else -1, 1.0, s_dtype)
    if loud:
        x[::2, LOUD] = LOUD_X
        gate, up = _fill(gate, LOUD, 1), _fill(up, LOUD, 7 if wide else 1)
    up_zero = torch.ones(I, dtype=torch.bool)
    live = 4 if wide else 16
    up_zero[torch.arange(live) * I // live] = False
    for t in (up[1], up[2]):  # q s + b with both zero: none of these columns' values
        t[:, up_zero] = 0
    down = _ints(g, (E, D, I), group, 0, 2, -1, 2.0**-8, s_dtype)
    pick = torch.stack([torch.randperm(E, generator=g)[:slots] for _ in range(R)]).to(torch.int32)
    wts = 2.0 ** torch.randint(-1, 2, (R, slots), generator=g).float()
    x, mats = x.to(s_dtype), [gate, up, down]
    if wide:  # as large as the sums allow: times an odd number, which adds to the bits
        size = _plain(x, pick, wts, mats)[3]
        odd = max(v for v in range(1, 16, 2) if v * size < 2**24)
        for t in gate[1:]:
            t *= odd
    return x, pick, wts, mats


def _plain(x, pick, wts, mats, terms=None):
    """The experts in 64 bits, with h rounded to `terms` bf16 numbers that add up to it (None: not rounded), and the sizes that
    exactness needs: the smallest gate sum, the largest h, the largest sum of |q h|, |b| |h| or |out| of any order."""
    out = torch.zeros(x.shape, dtype=torch.float64)
    low, large, size = float("inf"), 0.0, 0.0
    total = torch.zeros(x.shape, dtype=torch.float64)
    for e in range(mats[0][0].shape[0]):
        rows, slot = torch.nonzero(pick == e, as_tuple=True)
        if not rows.numel():
            continue
        gate, up, down = (plain.dense(*(t[e] for t in m)) for m in mats)
        v = x[rows].double()
        g, u = v @ gate.t(), v @ up.t()
        h = g * u
        low, large = min(low, float(g.min())), max(large, float(h.abs().max()))
        size = max(size, float((h.abs() @ (2.0 * torch.ones(h.shape[1], dtype=torch.float64))).max()))
        if terms:
            rest, h = h.float(), torch.zeros_like(h)
            for _ in range(terms):
                b = rest.to(BF16)
                h, rest = h + b.double(), rest - b.float()
        w = wts[rows, slot].double()[:, None]
        out.index_add_(0, rows, w * (h @ down.t()))
        total.index_add_(0, rows, w * (h.abs() @ down.abs().t()))
    return out, low, large, max(size, 512 * float(total.max()))


SHAPES = [  # E, D, I, group, slots, R
    (6, 64, 32, 32, 3, 1), (6, 256, 256, 64, 3, 1), (12, 1152, 128, 128, 4, 1), (5, 512, 192, 64, 3, 2), (6, 64, 32, 32, 2, 7),
    (12, 256, 256, 32, 4, 16), (9, 384, 384, 128, 4, 16), (12, 256, 160, 32, 4, 40), (40, 512, 256, 64, 8, 90),
    (16, 128, 256, 64, 4, 2300), (16, 256, 512, 64, 4, 1200), (8, 160, 1056, 32, 4, 900), (12, 64, 128, 32, 8, 2100),
    (4, 128, 2048, 128, 2, 1100)]


def _seed(shape):
    return sum(v * p for v, p in zip(shape, (1, 3, 7, 11, 13, 17)))


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[-1] <= 40])
@pytest.mark.parametrize("s_dtype", [BF16, F16])
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
def test_integers_need_every_term(shape, s_dtype, out_dtype):
    """The inputs do what the next test takes of them: sums stay below 2^24, silu(g) = g, and the result is that of the terms
    that the library holds, but not of one fewer."""
    x, pick, wts, mats = _case(_seed(shape), *shape, s_dtype, out_dtype)
    want, low, large, size = _plain(x, pick, wts, mats)
    assert low >= 18 and size < 2**24 and float(want.abs().max()) < 65504
    assert 2**8 < large < 2**16 if out_dtype != F32 else 2**16 < large < 2**24
    assert torch.equal(_plain(x, pick, wts, mats, TERMS[out_dtype])[0], want)
    fewer = _plain(x, pick, wts, mats, TERMS[out_dtype] - 1)[0]
    assert not torch.equal(fewer.float().to(out_dtype), want.float().to(out_dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("s_dtype", [BF16, F16])
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
def test_gpu_experts_exact_on_integers(ea, shape, s_dtype, out_dtype):  # noqa: F811
    """One row, few rows, items of 16 and long ones that stay in LDS or not: every value is the integers', rounded once to the
    output's type."""
    x, pick, wts, mats = _case(_seed(shape), *shape, s_dtype, out_dtype)
    want, low, _, size = _plain(x, pick, wts, mats)
    assert low >= 18 and size < 2**24
    out, _, _ = _experts(ea, x, pick, wts, mats, out_dtype, pad=4)
    assert torch.equal(out.cpu(), want.float().to(out_dtype))


@pytest.mark.parametrize("shape", [s for s in SHAPES if s[-1] <= 40])
@pytest.mark.parametrize("s_dtype", [BF16, F16])
def test_loud_columns_need_every_term(shape, s_dtype):
    """The sums of x over the loud columns' group are exact in fp32 and need all three bf16 terms (of some row, where there are several)."""
    for out_dtype in (BF16, F32):
        x, pick, wts, mats = _case(_seed(shape), *shape, s_dtype, out_dtype, True)
        _, low, _, size = _plain(x, pick, wts, mats)
        assert low >= 18 and size < 2**24
        sums = x[::2, :shape[3]].double().sum(1)
        assert float(sums.max()) * 15 < 2**24
        two = sums.float().to(BF16).double()
        two = two + (sums - two).float().to(BF16).double()
        assert (two != sums).any() or len(sums) < 2


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("s_dtype", [BF16, F16])
@pytest.mark.parametrize("out_dtype", [BF16, F32])
def test_gpu_experts_exact_beside_loud_columns(ea, shape, s_dtype, out_dtype):  # noqa: F811
    """Biases times sums of x that are far larger than what is left: every bit of the sums counts."""
    x, pick, wts, mats = _case(_seed(shape), *shape, s_dtype, out_dtype, True)
    want, low, _, size = _plain(x, pick, wts, mats)
    assert low >= 18 and size < 2**24
    out, _, _ = _experts(ea, x, pick, wts, mats, out_dtype)
    assert torch.equal(out.cpu(), want.float().to(out_dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 16, 40, 300])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gpu_linear_exact_beside_loud_columns(ea, m, dtype):  # noqa: F811
    device, _, q4 = ea
    g = torch.Generator().manual_seed(m)
    w = _fill(_ints(g, (83, 2112), 64, 0, 15, -7, 1.0, dtype), LOUD, 7)
    x = torch.randint(-3, 4, (m, 2112), generator=g)
    x[::2, LOUD] = LOUD_X
    x = x.to(dtype)
    out, dx = torch.zeros((m, 83), device="cuda"), x.cuda()
    q4.call(device.stream(), [q4.Linear(*_cuda(w))], dx.data_ptr(), {F16: 0, BF16: 1}[dtype], 2112, m, [out.data_ptr()], [2])
    assert torch.equal(out.cpu().double(), x.double() @ plain.dense(*w).t())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 16, 40, 300])
@pytest.mark.parametrize("group", [32, 128])
def test_gpu_linear_exact_on_the_largest_rows(ea, m, group):  # noqa: F811
    """bf16 rows up to 2^116, where a group's sum of q x still is a number: 15 x 128 x 2^116 < 2^127."""
    device, _, q4 = ea
    g = torch.Generator().manual_seed(m + group)
    w = _ints(g, (83, 1152), group, 0, 15, -7, 2.0**-20, BF16)
    x = (torch.randint(-1, 2, (m, 1152), generator=g) * 2.0**116).to(BF16)
    x[0], w[0][0] = 2.0**116, -1  # the largest sum: q = 15 throughout
    out, dx = torch.zeros((m, 83), device="cuda"), x.cuda()
    q4.call(device.stream(), [q4.Linear(*_cuda(w))], dx.data_ptr(), 1, 1152, m, [out.data_ptr()], [2])
    assert torch.equal(out.cpu().double(), x.double() @ plain.dense(*w).t())
