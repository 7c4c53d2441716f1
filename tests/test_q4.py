"""4-bit weights in groups (q4.Linear / call, q4.Experts / routed) against plain forms in 64 bits, within bounds that count
the additions and roundings of their evaluation (plain_q4)."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import plain_q4 as plain  # noqa: E402

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
CODE = {F16: 0, BF16: 1, F32: 2}


# ---- the plain form and the refusals, without a GPU ----------------------------------------------------------------------

def test_plain_values_by_hand():
    words = torch.tensor([[0x76543210, -0x12345679]], dtype=torch.int32)  # the second: 0xEDCBA987
    assert plain.values(words).tolist() == [[0, 1, 2, 3, 4, 5, 6, 7, 7, 8, 9, 10, 11, 12, 13, 14]]


def test_bytes():
    from ea_exl3._lib import lib

    b = lib().ea_q4_bytes
    assert b(16, 128, 128) == 1024 + 64 and b(16, 128, 64) == 1024 + 128 and b(16, 128, 32) == 1024 + 256
    assert b(17, 160, 32) == 4 * 1280 and b(1, 64, 64) == 1152
    for bad in ((16, 128, 16), (16, 128, 256), (16, 96, 64), (0, 128, 64), (16, 0, 64)):
        assert b(*bad) == 0


def _lin(**kw):
    from ea_exl3._lib import Q4Linear

    a = dict(words=4096, k=128, n=16, group=64, s_dtype=1)
    a.update(kw)
    return Q4Linear(a["words"], a["k"], a["n"], a["group"], a["s_dtype"])


def _call(ls, x=4096, x_dtype=1, x_stride=128, m=1, outs=None, dts=None):
    from ea_exl3._lib import lib

    n = len(ls)
    arr = (C.c_uint64 * n)(*[C.addressof(l) for l in ls])
    o = (C.c_uint64 * n)(*(outs or [4096] * n))
    d = (C.c_int * n)(*(dts or [2] * n))
    return lib().ea_q4_call(0, arr, n, x, x_dtype, x_stride, m, o, d)


def test_call_refuses():
    assert _call([_lin()] * 4) == 14
    assert _call([_lin(), _lin(k=256)], x_stride=256) == 14
    assert _call([_lin(), _lin(group=32)]) == 14
    assert _call([_lin(), _lin(s_dtype=0)]) == 14
    assert _call([_lin(group=16)]) == 11
    assert _call([_lin(k=96)]) == 8
    assert _call([_lin()], x_stride=124) == 9 and _call([_lin()], x_stride=130) == 9
    for bad in (dict(x=0), dict(x=4098), dict(x=4100), dict(x_dtype=2), dict(outs=[0]), dict(dts=[3]), dict(m=65537)):
        assert _call([_lin()], **bad) == 18, bad
    for bad in (dict(words=0), dict(words=4104), dict(n=0), dict(k=0), dict(s_dtype=2)):
        assert _call([_lin(**bad)]) == 18, bad
    if not torch.cuda.is_available():
        assert _call([_lin()]) == 17


def _ex(**kw):
    from ea_exl3._lib import Q4Experts

    a = dict(gu=4096, down=4096, count=4, dims=256, width=64, group=64, s_dtype=1, reserved=0)
    a.update(kw)
    return Q4Experts(*a.values())


def test_experts_refuse():
    from ea_exl3._lib import Q4Scratch, lib

    L = lib()
    ex, sc = _ex(), Q4Scratch()
    n = L.ea_q4_scratch_bytes(C.byref(ex), 8, 2)
    assert n > 0
    init = lambda e=ex, base=4096, size=n, rows=8, slots=2: L.ea_q4_scratch_init(  # noqa: E731
        C.byref(sc), base, size, C.byref(e), rows, slots)
    assert init(size=n - 1) == 12 and init(base=0) == 18 and init(base=4097) == 18 and init(slots=33) == 6
    assert init(slots=0) == 6 and init(rows=0) == 18 and init(rows=262145, size=1 << 60) == 18
    for e, code in ((_ex(group=48), 11), (_ex(dims=224), 8), (_ex(width=96), 8), (_ex(count=0), 18), (_ex(count=4097), 5),
                    (_ex(gu=0), 18), (_ex(down=0), 18), (_ex(gu=4104), 18), (_ex(down=4100), 18), (_ex(s_dtype=2), 18), (_ex(dims=0), 18)):
        assert init(e) == code
        assert L.ea_q4_scratch_bytes(C.byref(e), 8, 2) == 0
    assert init() == 0

    def call(e=ex, x=4096, x_dtype=1, stride=256, pick=4096, wts=4096, s=sc, out=4096, dt=2, R=1):
        return L.ea_q4_routed(0, x, x_dtype, stride, pick, wts, C.byref(e), C.byref(s), out, dt, R)

    assert call(R=9) == 12 and call(_ex(count=5)) == 12 and call(_ex(dims=320), stride=320) == 12 and call(_ex(width=128)) == 12
    assert call(stride=252) == 9 and call(stride=258) == 9
    for bad in (dict(x=0), dict(x=4100), dict(x_dtype=2), dict(pick=0), dict(wts=0), dict(out=0), dict(dt=3),
                dict(s=Q4Scratch())):
        assert call(**bad) in (18, 12), bad
    if not torch.cuda.is_available():
        assert call() == 17


# ---- on the GPU -------------------------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def ea():
    from ea_exl3 import device, ops, q4

    device.init(0)
    return device, ops, q4


def _cuda(m):
    return tuple(None if t is None else t.cuda() for t in m)


def _guarded(rows, n, dtype):
    """An output with a row of marks on either side."""
    return torch.full((rows + 2, n), 7.0, dtype=dtype, device="cuda")


def _linear(ea, m, k, ns, group, x_dtype, s_dtype, dts, seed=0, symmetric=False, pad=0, x=None):
    device, ops, q4 = ea
    g = torch.Generator().manual_seed(1000 * seed + k + m)
    mats = [plain.matrix(g, (n, k), group, s_dtype, symmetric) for n in ns]
    x = torch.randn((m, k), generator=g).to(x_dtype) if x is None else x
    dx = torch.full((m, k + pad), float("nan"), dtype=x_dtype, device="cuda")
    dx[:, :k] = x.cuda()
    ls = [q4.Linear(*_cuda(w)) for w in mats]
    outs = [_guarded(m, n, t) for n, t in zip(ns, dts)]
    print(f"linear m={m} k={k} ns={ns} group={group} x={x_dtype} s={s_dtype} out={dts}", flush=True)
    q4.call(device.stream(), ls, dx.data_ptr(), CODE[x_dtype], k + pad, m, [o[1:].data_ptr() for o in outs],
            [CODE[t] for t in dts])
    torch.cuda.synchronize()
    for o, w, t in zip(outs, mats, dts):
        assert (o[0] == 7).all() and (o[m + 1] == 7).all()
        want, err = plain.product(x.double(), w)
        plain.close(o[1:m + 1], want, err, f"n={want.shape[1]}")
    return [o[1:m + 1] for o in outs]


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("x_dtype", [F16, BF16])
@pytest.mark.parametrize("s_dtype", [F16, BF16])
def test_gpu_linear_values(ea, group, x_dtype, s_dtype):
    """One-hot rows give the weights themselves: every integer, scale and bias in its place."""
    k, n = 2 * 128 + group, 40
    x = torch.zeros((k, k), dtype=x_dtype)
    x[torch.arange(k), torch.arange(k)] = 1
    device, ops, q4 = ea
    g = torch.Generator().manual_seed(group)
    m = plain.matrix(g, (n, k), group, s_dtype)
    out = torch.zeros((k, n), device="cuda")
    dx = x.cuda()
    q4.call(device.stream(), [q4.Linear(*_cuda(m))], dx.data_ptr(), CODE[x_dtype], k, k, [out.data_ptr()], [2])
    want = plain.dense(*m).t()
    # one multiply by s and one addition of b, each rounded once, and sums with zeros
    assert ((out.cpu().double() - want).abs() <= 2.0**-23 * 0.3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 3, 5, 8, 15, 16, 17, 31, 33, 64, 65, 100, 128, 129, 200])
def test_gpu_linear_rows(ea, m):
    _linear(ea, m, 512, [48], 64, BF16, BF16, [F32])
    _linear(ea, m, 256, [33], 32, F16, F16, [F16], pad=4)


@pytest.mark.gpu
@pytest.mark.parametrize("k,group", [(32, 32), (64, 64), (96, 32), (128, 128), (160, 32), (192, 64), (1024, 128),
                                     (2112, 32), (6144, 64)])
@pytest.mark.parametrize("n", [1, 7, 16, 17, 250])
def test_gpu_linear_sizes(ea, k, group, n):
    for m, t in ((1, BF16), (6, F32), (40, F16)):
        _linear(ea, m, k, [n], group, BF16 if t != F16 else F16, BF16, [t])


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(17, 1024, 2080), (47, 83, 6144), (256, 256, 2176), (257, 250, 6144), (300, 250, 2048),
                                   (129, 4200, 2112), (600, 1000, 320), (40, 9000, 256), (16, 9000, 4096), (3, 26000, 2080)])
def test_gpu_linear_many_blocks(ea, m, n, k):
    """Rows and columns on both sides of each change of the kernels' form."""
    _linear(ea, m, k, [n], 32, BF16, BF16, [F32], seed=m)
    _linear(ea, m, k, [n], 32, F16, F16, [BF16], pad=4)


@pytest.mark.gpu
@pytest.mark.parametrize("k,group", [(32, 32), (320, 64), (1152, 128), (6144, 64)])
@pytest.mark.parametrize("m", [1, 4, 16, 20, 64, 100, 300])
def test_gpu_linear_exact_on_integers(ea, m, k, group):
    """Small integers everywhere: every sum is exact in fp32 in whatever order, so the result is the integers' own."""
    device, ops, q4 = ea
    g = torch.Generator().manual_seed(k + m)
    n = 83
    words = torch.randint(-(2**31), 2**31, (n, k // 8), generator=g, dtype=torch.int64).to(torch.int32)
    s = (2.0 ** torch.randint(-1, 2, (n, k // group), generator=g)).to(BF16)
    b = torch.randint(-20, 5, (n, k // group), generator=g).to(BF16)
    x = torch.randint(-3, 4, (m, k), generator=g).to(BF16)
    out, dx = torch.zeros((m, n), device="cuda"), x.cuda()
    q4.call(device.stream(), [q4.Linear(words.cuda(), s.cuda(), b.cuda())], dx.data_ptr(), 1, k, m, [out.data_ptr()], [2])
    assert torch.equal(out.cpu().double(), x.double() @ plain.dense(words, s, b).t())


@pytest.mark.gpu
@pytest.mark.parametrize("ns,dts", [([48, 17], [F32, BF16]), ([5, 64, 200], [F16, F32, BF16]), ([256, 256], [BF16, BF16])])
@pytest.mark.parametrize("m", [1, 9, 70])
def test_gpu_linear_jobs(ea, ns, dts, m):
    _linear(ea, m, 768, ns, 128, BF16, F16, dts, symmetric=m == 9, pad=12)


@pytest.mark.gpu
def test_gpu_linear_large_values(ea):
    """The largest finite inputs and scales: no intermediate leaves fp32, and other rows keep their values beside a row of NaN
    or infinities."""
    device, ops, q4 = ea
    x = torch.randn((5, 256)).to(F16)
    x[1] = 65504.0
    x[2] = float("nan")
    x[3, 7] = float("inf")
    g = torch.Generator().manual_seed(5)
    m = plain.matrix(g, (32, 256), 64, F16)
    out = torch.zeros((5, 32), device="cuda")
    dx = x.cuda()
    q4.call(device.stream(), [q4.Linear(*_cuda(m))], dx.data_ptr(), 0, 256, 5, [out.data_ptr()], [2])
    want, err = plain.product(x.double(), m)
    for r in (0, 1, 4):
        plain.close(out[r], want[r], err[r], f"row {r}")
    assert torch.isnan(out[2]).all() and not torch.isfinite(out[3]).any()


@pytest.mark.gpu
def test_gpu_linear_nothing_to_do(ea):
    device, ops, q4 = ea
    g = torch.Generator().manual_seed(5)
    l = q4.Linear(*_cuda(plain.matrix(g, (32, 256), 64, F16)))
    out = torch.full((4, 32), 3.0, device="cuda")
    q4.call(device.stream(), [l], out.data_ptr(), 0, 256, 0, [out.data_ptr()], [2])
    assert (out == 3).all()


@pytest.mark.parametrize("bad", ["group", "scales", "biases", "dims", "host"])
def test_linear_sources_refused(bad):
    if not torch.cuda.is_available() and bad != "host":
        pytest.skip("needs device tensors to get past the device check")
    from ea_exl3 import q4

    g = torch.Generator().manual_seed(5)
    w, s, b = plain.matrix(g, (16, 256), 64, F16)
    if bad != "host":
        w, s, b = w.cuda(), s.cuda(), b.cuda()
    elif not torch.cuda.is_available():
        pytest.skip("the current device is asked for")
    if bad == "group":
        s, b = s[:, :1].contiguous(), b[:, :1].contiguous()
    if bad == "scales":
        s = s.float()
    if bad == "biases":
        b = b.bfloat16()
    if bad == "dims":
        w = w[0]
    with pytest.raises(ValueError):
        q4.Linear(w, s, b)


# ---- experts ----------------------------------------------------------------------------------------------------------

def _layer(gen, E, D, I, group, s_dtype, symmetric=False):
    return [plain.matrix(gen, shape, group, s_dtype, symmetric) for shape in ((E, I, D), (E, I, D), (E, D, I))]


def _experts(ea, x, pick, wts, mats, out_dtype, pad=0, ex=None, sc=None):
    device, ops, q4 = ea
    R, D = x.shape
    ex = ex or q4.Experts(*(_cuda(m) for m in mats))
    sc = sc or q4.Scratch(ex, R, pick.shape[1])
    sc.buf.fill_(255)  # NaN wherever it is read before it is written
    dx = torch.full((R, D + pad), float("nan"), dtype=x.dtype, device="cuda")
    dx[:, :D] = x.cuda()
    dp, dw = pick.cuda(), wts.cuda()
    out = _guarded(R, D, out_dtype)
    print(f"experts R={R} {ex.count}x{D}x{ex.width} group={ex.group} slots={pick.shape[1]} {x.dtype} -> {out_dtype}", flush=True)
    q4.routed(device.stream(), dx.data_ptr(), CODE[x.dtype], D + pad, dp.data_ptr(), dw.data_ptr(), ex, sc,
              out[1:].data_ptr(), CODE[out_dtype], R)
    torch.cuda.synchronize()
    assert (out[0] == 7).all() and (out[R + 1] == 7).all()
    return out[1:R + 1], ex, sc


def _routing(gen, R, E, slots):
    pick = torch.stack([torch.randperm(E, generator=gen)[:slots] for _ in range(R)]).to(torch.int32)
    return pick, torch.rand((R, slots), generator=gen) + 0.1


@pytest.mark.gpu
@pytest.mark.parametrize("R", [1, 2, 3, 7, 15, 16, 17, 40, 65, 130, 300])
@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
def test_gpu_experts_rows(ea, R, out_dtype):
    g = torch.Generator().manual_seed(R)
    E, D, I, S = 12, 256, 64, 4
    mats = _layer(g, E, D, I, 64, BF16)
    x = torch.randn((R, D), generator=g).to(F16 if out_dtype == F16 else BF16)
    pick, wts = _routing(g, R, E, S)
    out, _, _ = _experts(ea, x, pick, wts, mats, out_dtype)
    want, err = plain.experts(x.double(), pick, wts, *mats, out_dtype)
    plain.close(out, want, err)


@pytest.mark.gpu
@pytest.mark.parametrize("E,D,I,group,slots", [
    (1, 128, 128, 128, 1), (3, 64, 32, 32, 3), (9, 96, 160, 32, 2), (5, 1024, 192, 64, 5), (40, 384, 512, 128, 32),
    (300, 64, 64, 64, 8), (2, 2112, 96, 32, 2), (20, 6144, 256, 64, 8)])
@pytest.mark.parametrize("R", [1, 5, 16, 23, 90])
def test_gpu_experts_sizes(ea, E, D, I, group, slots, R):
    g = torch.Generator().manual_seed(E + R)
    dt = F16 if R == 5 else BF16
    mats = _layer(g, E, D, I, group, dt, symmetric=R == 16)
    x = torch.randn((R, D), generator=g).to(dt)
    pick, wts = _routing(g, R, E, slots)
    out_dtype = dt if R in (1, 90) else F32
    out, _, _ = _experts(ea, x, pick, wts, mats, out_dtype, pad=4)
    want, err = plain.experts(x.double(), pick, wts, *mats, out_dtype)
    plain.close(out, want, err)


@pytest.mark.gpu
@pytest.mark.parametrize("E,D,I,group,slots,R,dt,out_dtype", [
    (16, 256, 512, 64, 4, 1200, BF16, BF16), (16, 256, 512, 32, 4, 1200, F16, F32), (24, 128, 512, 128, 3, 1400, BF16, F32),
    (8, 160, 1056, 32, 4, 900, BF16, F16), (4, 384, 2048, 128, 2, 1100, F16, F16), (40, 96, 320, 32, 8, 1000, F16, BF16),
    (24, 1152, 384, 64, 3, 1700, BF16, BF16), (16, 128, 256, 64, 4, 2300, BF16, F16), (16, 192, 256, 32, 4, 2300, F16, F32),
    (12, 64, 128, 32, 8, 2100, BF16, BF16), (16, 256, 512, 64, 4, 500, BF16, BF16)])
def test_gpu_experts_long_items(ea, E, D, I, group, slots, R, dt, out_dtype):
    """Prompts: items of up to 64 pairs of experts picked more and less often (some by nobody, some rows empty), widths whose
    rows stay in LDS and wider ones; the same bits again, and for the rows in another order."""
    g = torch.Generator().manual_seed(E + R)
    mats = _layer(g, E, D, I, group, dt)
    x = torch.randn((R, D), generator=g).to(dt)
    heat = torch.rand((R, E), generator=g).log() / torch.linspace(3.0, 0.05, E)
    heat[:, 1] = float("-inf")
    pick = heat.topk(slots, dim=1).indices.to(torch.int32)
    wts = torch.rand((R, slots), generator=g) + 0.1
    pick[R - 20:] = -1
    out, ex, sc = _experts(ea, x, pick, wts, mats, out_dtype, pad=8)
    want, err = plain.experts(x.double(), pick, wts, *mats, out_dtype)
    plain.close(out, want, err)
    assert (out[R - 20:] == 0).all()
    again, _, _ = _experts(ea, x, pick, wts, mats, out_dtype, ex=ex, sc=sc)
    assert torch.equal(out, again)
    order = torch.randperm(R, generator=g)
    turned, _, _ = _experts(ea, x[order], pick[order], wts[order], mats, out_dtype, ex=ex, sc=sc)
    assert torch.equal(out[order.cuda()], turned)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [1, 6, 16, 17, 150])
def test_gpu_experts_odd_picks(ea, R):
    """Empty slots and rows, picks outside the experts, one expert for all, an expert twice in a row; NaN weights and rows
    where nothing is picked do not reach the output, and a row of NaN only its own."""
    g = torch.Generator().manual_seed(R)
    E, D, I, S = 6, 192, 64, 3
    mats = _layer(g, E, D, I, 64, BF16)
    x = torch.randn((R, D), generator=g).to(BF16)
    pick, wts = _routing(g, R, E, S)
    pick[:, 0] = 4                      # everyone's
    pick[R // 2] = -1                   # a row without experts
    wts[R // 2] = float("nan")
    x[R // 2] = float("nan")
    if R > 3:
        pick[1, 1] = E                  # outside
        wts[1, 1] = float("inf")
        pick[2] = torch.tensor([3, 3, 3])
        pick[3, 2] = -(2**31)
        x[R - 1, 5] = float("nan")
    out, _, _ = _experts(ea, x, pick, wts, mats, F32)
    clean = torch.where(torch.isnan(x), 0, x)
    live = (pick >= 0) & (pick < E)
    want, err = plain.experts(clean.double(), torch.where(live, pick, -1), torch.where(live, wts, 0), *mats, F32)
    if R > 3 and live[R - 1].any():
        assert torch.isnan(out[R - 1]).all()
        out[R - 1] = want[R - 1].float().cuda()
    plain.close(out, want, err)
    assert (out[R // 2] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [BF16, F32])
def test_gpu_experts_odd_picks_in_long_items(ea, out_dtype):
    """The same where items are long: rows of NaN between others of their items, an infinite activation, rows without experts,
    picks outside, an expert named twice."""
    g = torch.Generator().manual_seed(11)
    E, D, I, S, R = 6, 192, 512, 3, 1500
    mats = _layer(g, E, D, I, 64, BF16)
    x = torch.randn((R, D), generator=g).to(BF16)
    pick, wts = _routing(g, R, E, S)
    pick[::7] = torch.tensor([2, -1, 2], dtype=torch.int32)
    pick[::11] = -1
    wts[::11], x[::11] = float("nan"), float("nan")
    pick[5::13, 1] = E
    wts[5::13, 1] = float("inf")
    bad = torch.arange(1, R, 37)
    bad = bad[(bad % 7 != 0) & (bad % 11 != 0)]
    pick[bad] = torch.tensor([0, 3, 5], dtype=torch.int32)
    wts[bad] = 0.5
    x[bad[::2]] = float("nan")
    x[bad[1::2], 4] = float("inf")
    out, _, _ = _experts(ea, x, pick, wts, mats, out_dtype)
    assert not torch.isfinite(out[bad.cuda()]).any()
    assert (out[::11] == 0).all()
    live = (pick >= 0) & (pick < E)
    clean = torch.where(torch.isfinite(x), x, 0)
    want, err = plain.experts(clean.double(), torch.where(live, pick, -1), torch.where(live, wts, 0), *mats, out_dtype)
    rest = torch.ones(R, dtype=torch.bool)
    rest[bad] = False
    plain.close(out[rest.cuda()], want[rest], err[rest])


@pytest.mark.gpu
def test_gpu_experts_scratch_serves_smaller_calls(ea):
    """A scratch made for more rows and a larger layer, used again and again: the same bits as with one of its own."""
    device, ops, q4 = ea
    g = torch.Generator().manual_seed(77)
    big = _layer(g, 10, 512, 128, 64, BF16)
    small = _layer(g, 7, 256, 64, 64, BF16)
    exb, exs = (q4.Experts(*(_cuda(m) for m in t)) for t in (big, small))
    sc = q4.Scratch(exb, 120, 3)
    for R in (120, 1, 16, 50, 3):
        for mats, ex in ((big, exb), (small, exs)):
            x = torch.randn((R, ex.dims), generator=g).to(BF16)
            pick, wts = _routing(g, R, ex.count, 3)
            a, _, _ = _experts(ea, x, pick, wts, mats, BF16, ex=ex, sc=sc)
            b, _, _ = _experts(ea, x, pick, wts, mats, BF16, ex=ex)
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [1, 16, 70])
def test_gpu_experts_same_bits_again(ea, R):
    """The same call gives the same bits; above 16 rows, where pairs are summed alone, a row's bits do not depend on the batch
    around it either (up to 16 rows the experts are added in the batch's order)."""
    g = torch.Generator().manual_seed(R)
    mats = _layer(g, 8, 256, 64, 64, BF16)
    x = torch.randn((R, 256), generator=g).to(BF16)
    pick, wts = _routing(g, R, 8, 3)
    a, ex, sc = _experts(ea, x, pick, wts, mats, F32)
    for _ in range(3):
        b, _, _ = _experts(ea, x, pick, wts, mats, F32, ex=ex, sc=sc)
        assert torch.equal(a, b)
    if R > 16:
        order = torch.randperm(R, generator=g)
        b, _, _ = _experts(ea, x[order], pick[order], wts[order], mats, F32, ex=ex, sc=sc)
        assert torch.equal(a[order.cuda()], b)


@pytest.mark.gpu
def test_gpu_experts_on_two_streams(ea):
    """Two layers at once, each with a stream and a scratch of its own, from one row to long items; and a captured prompt pass
    replayed between eager ones on the same scratch."""
    device, ops, q4 = ea
    g = torch.Generator().manual_seed(3)
    E, D, I, S = 16, 256, 512, 4
    exs = [q4.Experts(*(_cuda(m) for m in _layer(g, E, D, I, 64, BF16))) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for R in (1, 16, 100, 1200):
        scs = [q4.Scratch(ex, R, S) for ex in exs]
        xs = [torch.randn((R, D), generator=g).to(BF16).cuda() for _ in exs]
        routing = [[t.cuda() for t in _routing(g, R, E, S)] for _ in exs]
        outs = [torch.zeros((R, D), device="cuda") for _ in exs]

        def run(i, stream):
            q4.routed(stream, xs[i].data_ptr(), 1, D, routing[i][0].data_ptr(), routing[i][1].data_ptr(), exs[i], scs[i],
                      outs[i].data_ptr(), 2, R)

        torch.cuda.synchronize()
        want = []
        for i in range(2):
            run(i, device.stream())
            want.append(outs[i].clone())
        torch.cuda.synchronize()
        for o in outs:
            o.fill_(5)
        torch.cuda.synchronize()
        for _ in range(4):
            for i in range(2):
                run(i, device.stream(streams[i]))
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[0]):
            run(0, device.stream())
        for _ in range(3):
            outs[0].fill_(5)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want[0])
            xs[0].neg_()
            run(0, device.stream())
            xs[0].neg_()
            torch.cuda.synchronize()


# ---- the set together -----------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("R", [1, 16, 60])
def test_gpu_layer_together(ea, R):
    """A 4-bit MoE layer as a program issues it: the router's logits, routing with groups, routed experts, the shared expert
    (gate|up, SwiGLU, down) and their sum, eager and replayed from a graph, on a stream of its own."""
    device, ops, q4 = ea
    g = torch.Generator().manual_seed(R)
    E, D, I, S = 16, 512, 128, 4
    mats = _layer(g, E, D, I, 64, BF16)
    shared = [plain.matrix(g, s, 64, BF16) for s in ((I, D), (I, D), (D, I))]
    ex = q4.Experts(*(_cuda(m) for m in mats))
    gate, up, down = (q4.Linear(*_cuda(m)) for m in shared)
    sc = q4.Scratch(ex, R, S)
    wr = (0.05 * torch.randn((E, D), generator=g)).to(BF16).cuda()
    bias = (0.1 * torch.randn(E, generator=g)).cuda()
    x = torch.empty((R, D), dtype=BF16, device="cuda")
    logits, pick = torch.zeros((R, E), device="cuda"), torch.zeros((R, S), dtype=torch.int32, device="cuda")
    wts, out, sy = torch.zeros((R, S), device="cuda"), torch.zeros((R, D), device="cuda"), torch.zeros((R, D), device="cuda")
    hg, hu, act = (torch.zeros((R, I), dtype=BF16, device="cuda") for _ in range(3))

    def layer(s):
        ops.router(s, x.data_ptr(), D, wr.data_ptr(), 0, logits.data_ptr(), R, D, E)
        ops.route(s, logits.data_ptr(), 2, E, bias.data_ptr(), pick.data_ptr(), wts.data_ptr(), R, E, S, groups=4,
                  top_groups=2, group_best=2, scale=2.5)
        q4.routed(s, x.data_ptr(), 1, D, pick.data_ptr(), wts.data_ptr(), ex, sc, out.data_ptr(), 2, R)
        q4.call(s, [gate, up], x.data_ptr(), 1, D, R, [hg.data_ptr(), hu.data_ptr()], [1, 1])
        ops.swiglu2(s, hg.data_ptr(), hu.data_ptr(), act.data_ptr(), R, I)
        q4.call(s, [down], act.data_ptr(), 1, I, R, [sy.data_ptr()], [2])
        ops.add_f32(s, out.data_ptr(), sy.data_ptr(), R * D)

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    xs = [torch.randn((R, D), generator=g).to(BF16) for _ in range(3)]
    with torch.cuda.stream(side):
        x.copy_(xs[0])
        layer(device.stream())
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            layer(device.stream())
    torch.cuda.synchronize()
    for v in xs + xs[:1]:
        x.copy_(v)
        torch.cuda.synchronize()
        layer(device.stream())
        eager = out.clone()
        ep, ew, el = pick.clone(), wts.clone(), logits.cpu()
        out.fill_(9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        want_p, want_w = plain.route(el, bias.cpu(), S, False, 4, 2, 2, True, 2.5)
        assert torch.equal(ep.cpu(), want_p)
        want, err = plain.experts(v.double(), want_p, ew.cpu(), *mats, F32)
        h = {}
        for name, m in (("g", shared[0]), ("u", shared[1])):
            t, e = plain.product(v.double(), m)
            h[name] = t, e + plain.HALF[BF16] * (t.abs() + e)  # gate and up are rounded to bf16
        (tg, eg), (tu, eu) = h["g"], h["u"]
        s = tg * torch.sigmoid(tg)
        es = 1.1 * eg + (plain.HALF[BF16] + 2.0**-20) * (s.abs() + 1.1 * eg)  # silu's slope, its rounding to bf16
        ha, ea_ = s * tu, es * (tu.abs() + eu) + s.abs() * eu
        y, ey = plain.product(ha, shared[2], ea_ + plain.HALF[BF16] * (ha.abs() + ea_))
        plain.close(eager, want + y, err + ey + 2.0**-23 * (want.abs() + y.abs()))
