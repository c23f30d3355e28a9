"""Fully connected layers (``linear``) against their formulas in 64 bits.

Most inputs are small integers times powers of two: then every product and every sum of the layer is exact in fp32, and what the
kernels return is the exact value rounded once -- equality is asked for, not closeness.  With the smooth activations the tolerance
counts, per element, the rounding of the result (half a step: ``eps / 2`` relative) and 2^-18 of what an fp32 activation is made
of (its exponential and division are good to a few 2^-22, the arguments of the exponential lose up to 2^-23 times their size,
which is below 16 where the slope is not flat), and for products of a rounded gradient half a step of each of its values."""
import ctypes

import pytest
import torch

from pytorch_winoconv_b200 import capi, checkpoint, linear as lin

gpu = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]
F = torch.nn.functional


def ints(shape, seed, span, step, dtype, device="cuda"):
    """Integers of -span..span times step."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-span, span + 1, shape, generator=g).double() * step).to(dtype).to(device)


def act64(z, name):
    return {None: lambda t: t, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"), "silu": F.silu}[name](z)


def half_step(t, dtype):
    """Half a step of the type at each value, and of its subnormals."""
    info = torch.finfo(dtype)
    return t.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def make(rows, k, n, dtype, seed=0, bias=True, residual=True):
    """Layer inputs whose sums are exact: |x| <= 2, |w| <= 1/2 in steps of 1/4 and 1/8, so sums are multiples of 2^-5 below 2^15."""
    x = ints((rows, k), seed, 8, 0.25, dtype)
    w = ints((n, k), seed + 1, 4, 0.125, dtype)
    b = ints((n,), seed + 2, 8, 0.25, dtype) if bias else None
    r = ints((rows, n), seed + 3, 8, 0.25, dtype) if residual else None
    return x, w, b, r


def forward64(x, w, b, r, act):
    z = x.double() @ w.double().t()
    if b is not None:
        z = z + b.double()
    y = act64(z, act)
    return z, y if r is None else y + r.double()


def check(got, want, act, dtype, extra=None):
    """Equal to the exact value rounded once, or within the tolerance of a smooth activation."""
    if act in (None, "relu") and extra is None:
        assert torch.equal(got, want.to(dtype))
        return
    tol = half_step(want, dtype) + want.abs() * 2.0 ** -18 + (0 if extra is None else extra)
    off = (got.double() - want).abs()
    assert (off <= tol).all(), ((off - tol).max().item(), off.max().item())


SHAPES = [(1, 64, 128), (1, 1, 1), (1, 1000, 1531), (1, 4103, 130), (2, 33, 7), (2, 4608, 1001), (3, 4096, 250), (16, 72, 136), (17, 129, 131), (31, 520, 2048), (64, 2048, 129),
          (127, 40, 64), (128, 64, 128), (129, 65, 129), (130, 777, 1000), (257, 200, 520), (1000, 136, 96), (1025, 100, 300), (513, 1024, 768),
          (1301, 72, 1531), (2000, 129, 1100), (1281, 1801, 1537), (1536, 1600, 1792),
          (300, 2056, 4001), (510, 712, 8000), (4100, 520, 264)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_forward_is_the_exact_value_rounded_once(rows, k, n, dtype):
    for i, (act, bias, residual) in enumerate([(None, False, False), ("relu", True, False), (None, True, True), ("relu", False, True)]):
        x, w, b, r = make(rows, k, n, dtype, 10 * i, bias, residual)
        y = lin.linear(x, w, b, r, activation=act)
        assert y.shape == (rows, n) and y.dtype == dtype
        check(y, forward64(x, w, b, r, act)[1], act, dtype)
    assert capi.read_device_error() == 0


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows,k,n", [(1, 64, 128), (17, 129, 131), (300, 40, 520)])
def test_smooth_activations(rows, k, n, act, dtype):
    x, w, b, r = make(rows, k, n, dtype)
    z, y = forward64(x, w, b, r, act)
    # fp32 error of the activation (relative to z: 1 + erf cancels for negative z), then of the sum
    check(lin.linear(x, w, b, r, activation=act), y, act, dtype, extra=(z.abs() + 1) * 2.0 ** -20)
    y = act64(z, act)
    check(lin.linear(x, w, b, activation=act), y, act, dtype, extra=(z.abs() + 1) * 2.0 ** -20)


def reference_backward(x, w, gy, z, act, dtype, bits8):
    """dz, and the gradients from what was kept."""
    if bits8:
        kept_x, kept_z = values8(x.double(), dtype), values8(z, dtype)
    else:
        kept_x, kept_z = x.double(), z.to(dtype).double()
    kept_z.requires_grad_()
    dz, = torch.autograd.grad(act64(kept_z, act), kept_z, gy.double())
    return dz, kept_x


def values8(x, dtype):
    """The values that eight bits hold, in 64 bits: rounding to the step at each value, half to even."""
    out = torch.empty_like(x)
    for c in range(0, x.shape[-1], 32):
        v = x[..., c:c + 32]
        top = torch.where(v.abs() < float("inf"), v.abs(), torch.zeros_like(v)).nan_to_num(0.0).amax(-1, keepdim=True)
        m, e = torch.frexp(top)
        e = torch.where(top > 0, e - 9 + (m > 0.875).int(), torch.full_like(e, -127)).clamp_min(-127).double()
        t = v / torch.exp2(e)
        _, at = torch.frexp(t.abs().clamp_min(2.0 ** -6))
        step = torch.exp2((at - 4).double())
        q = torch.where(t.abs() < float("inf"), torch.round(t / step) * step, torch.full_like(t, float("nan")))
        out[..., c:c + 32] = q * torch.exp2(e)
    most = torch.finfo(dtype).max
    return out.clamp(-most, most)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pack", [None, "e4m3"])
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_gradients_are_exact_values_rounded_once(rows, k, n, pack, dtype):
    """Integer gradients of 9 values: dz is exact, and so are the sums of the three products."""
    for act in (None, "relu"):
        x, w, b, r = make(rows, k, n, dtype, 5)
        gy = ints((rows, n), 9, 4, 2.0 ** -6, dtype)
        for t in (x, w, b, r):
            t.requires_grad_()
        y = lin.linear(x, w, b, r, activation=act, checkpoint=pack)
        z, want = forward64(x.detach(), w.detach(), b.detach(), r.detach(), act)
        check(y.detach(), want, act, dtype)
        dx, dw, db, dr = torch.autograd.grad(y, (x, w, b, r), gy)
        dz, kept = reference_backward(x.detach(), w.detach(), gy, z, act, dtype, pack)
        assert torch.equal(dx, (dz @ w.detach().double()).to(dtype))
        assert torch.equal(dw, (dz.t() @ kept).to(dtype))
        assert torch.equal(db, dz.sum(0).to(dtype))
        assert torch.equal(dr, gy)
    assert capi.read_device_error() == 0


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pack", [None, "e4m3"])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows,k,n", [(1, 64, 128), (33, 72, 130), (200, 129, 264)])
def test_gradients_through_smooth_activations(rows, k, n, act, pack, dtype):
    x, w, b, _ = make(rows, k, n, dtype, 7)
    gy = ints((rows, n), 9, 4, 2.0 ** -3, dtype)
    for t in (x, w, b):
        t.requires_grad_()
    y = lin.linear(x, w, b, activation=act, checkpoint=pack)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), gy)
    wd, xd = w.detach().double(), x.detach().double()
    z = xd @ wd.t() + b.detach().double()
    dz, kept = reference_backward(xd, wd, gy, z, act, dtype, pack)
    # dz: fp32 slope (at most 1.13) times gy, then half a step of the type; the sums of n and of rows such values in fp32
    off = gy.double().abs() * 2.0 ** -18
    tol_dz = off + half_step(dz, dtype) + off * torch.finfo(dtype).eps
    sums = 2.0 ** -23
    check(dx, dz @ wd, act, dtype, extra=tol_dz @ wd.abs() + (dz.abs() @ wd.abs()) * (n / 16 + 8) * sums)
    check(dw, dz.t() @ kept, act, dtype, extra=tol_dz.t() @ kept.abs() + (dz.abs().t() @ kept.abs()) * (rows / 16 + 8) * sums)
    check(db, dz.sum(0), act, dtype, extra=off.sum(0) + dz.abs().sum(0) * (rows / 8 + 16) * sums)


@gpu
@pytest.mark.parametrize("act", [None, "gelu", "silu"])
def test_gradients_against_differences(act):
    """The derivative of sum(gy y) along a direction of each input, by central differences of the 64-bit layer."""
    x, w, b, r = (t.detach().requires_grad_() for t in make(20, 40, 48, torch.float16, 3))
    gy = ints((20, 48), 4, 8, 0.125, torch.float16)
    grads = torch.autograd.grad(lin.linear(x, w, b, r, activation=act), (x, w, b, r), gy)
    leaves = [t.detach().double() for t in (x, w, b, r)]
    for i, g in enumerate(grads):
        d = torch.randn(leaves[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).cuda()

        def value(h):
            at = [t + h * d if j == i else t for j, t in enumerate(leaves)]
            return (forward64(*at, act)[1] * gy.double()).sum().item()

        slope = (value(1e-5) - value(-1e-5)) / 2e-5
        got = (g.double() * d).sum().item()
        # every value of g is within two half steps (dz and the result) and z's own rounding: 2^-11 each, |act''| <= 0.8 and |z| < 64
        assert abs(got - slope) <= (g.double() * d).abs().sum().item() * 2.0 ** -9 + 1e-6 + abs(slope) * 2.0 ** -8


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_views_strides_and_types_of_the_arguments(dtype):
    rows, k, n = 48, 72, 104
    x, w, b, r = make(rows, k, n, dtype)
    want = forward64(x, w, b, r, None)[1].to(dtype)
    wide = torch.full((rows, k + 24), float("nan"), dtype=dtype, device="cuda")
    wide[:, 8:8 + k] = x
    assert torch.equal(lin.linear(wide[:, 8:8 + k], w, b, r), want)                     # rows apart, read as they lie
    wide[:, 3:3 + k] = x
    assert torch.equal(lin.linear(wide[:, 3:3 + k], w, b, r), want)                     # not on 16 bytes: copied
    assert torch.equal(lin.linear(x.t().contiguous().t(), w.t().contiguous().t(), b, r.t().contiguous().t()), want)
    both = torch.stack([b, b], 1)[:, 0]
    assert both.stride(0) == 2 and torch.equal(lin.linear(x, w, both, r), want)
    shifted = torch.cat([torch.zeros(1, dtype=dtype, device="cuda"), b])[1:]
    assert torch.equal(lin.linear(x, w, shifted, r), want)
    rw = torch.full((rows, n + 5), float("nan"), dtype=dtype, device="cuda")
    rw[:, 1:n + 1] = r
    assert torch.equal(lin.linear(x, w, b, rw[:, 1:n + 1]), want)                       # a residual anywhere
    assert torch.equal(lin.linear(x, w.float(), b.float(), r), want)
    y = lin.linear(x.reshape(4, 3, 4, k), w, b, r.reshape(4, 3, 4, n))
    assert y.shape == (4, 3, 4, n) and torch.equal(y.reshape(rows, n), want)
    assert torch.equal(lin.linear(x[5], w, b, r[5]), want[5])                           # one row without a batch
    one = x[:1].expand(rows, k)
    assert torch.equal(lin.linear(one, w, b, r[:1].expand(rows, n)), want[:1].expand(rows, n))
    turned = x.reshape(6, 8, k).transpose(0, 1)
    assert torch.equal(lin.linear(turned, w, b), lin.linear(x, w, b).reshape(6, 8, n).transpose(0, 1))


@gpu
@pytest.mark.parametrize("pack", [None, "e4m3"])
def test_gradients_of_views_and_of_float_parameters(pack):
    rows, k, n, dtype = 40, 36, 50, torch.bfloat16
    x, w, b, _ = make(rows, k, n, dtype)
    gy = ints((rows, n), 9, 4, 2.0 ** -6, dtype)
    xd, wd, gd = x.double(), w.double(), gy.double()
    kept = values8(xd, dtype) if pack else xd
    base = torch.zeros(rows, k + 3, dtype=dtype, device="cuda")
    base[:, 2:2 + k] = x
    base.requires_grad_()
    wf, bf = w.float().requires_grad_(), b.float().requires_grad_()
    y = lin.linear(base[:, 2:2 + k], wf, bf, checkpoint=pack)
    spread = torch.zeros(rows, 2 * n, dtype=dtype, device="cuda")
    spread[:, ::2] = gy
    dbase, dw, db = torch.autograd.grad(y, (base, wf, bf), spread[:, ::2])              # a gradient with gaps
    assert torch.equal(dbase[:, 2:2 + k], (gd @ wd).to(dtype)) and dbase[:, :2].abs().sum() == 0
    assert dw.dtype == torch.float32 and torch.equal(dw, (gd.t() @ kept).float())
    assert db.dtype == torch.float32 and torch.equal(db, gd.sum(0).float())
    # the gradient behind a sum: one value with strides of zero
    y = lin.linear(x.requires_grad_(), w, b, checkpoint=pack)
    dx, = torch.autograd.grad(y.sum(), x)
    assert torch.equal(dx, wd.sum(0).expand(rows, k).to(dtype))
    # a row used many times over
    one = x.detach()[:1].clone().requires_grad_()
    y = lin.linear(one.expand(rows, k), w, b, checkpoint=pack)
    dx, = torch.autograd.grad(y, one, gy)
    parts = (gd @ wd).to(dtype).double()
    assert ((dx.double() - parts.sum(0)).abs() <= half_step(parts.sum(0), dtype) + parts.abs().sum(0) * 2.0 ** -23 * rows).all()


@gpu
def test_only_what_is_asked_for_is_kept_and_computed():
    rows, k, n, dtype = 256, 512, 1024, torch.bfloat16
    x, w, b, r = make(rows, k, n, dtype)

    def kept(wanted, **kw):
        leaves = {"x": x, "w": w, "b": b, "r": r}
        for name, t in leaves.items():
            t.requires_grad_(name in wanted)
        size = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: size.append(t.numel() * t.element_size()) or t, lambda t: t):
            y = lin.linear(x, w, b, r, **kw)
        grads = torch.autograd.grad(y, [leaves[i] for i in wanted], torch.ones_like(y))
        assert all(g.shape == leaves[i].shape for g, i in zip(grads, wanted))
        return sum(size)

    w_, x_, z_ = 2 * n * k, 2 * rows * k, 2 * rows * n
    assert kept("x") == w_
    assert kept("w") == x_
    assert kept("b") == 0 and kept("r") == 0
    assert kept("xwbr", activation="gelu") == w_ + x_ + z_
    assert kept("r", activation="gelu") == 0
    assert kept("xwbr", activation="gelu", checkpoint="e4m3") == w_ + (x_ + z_) // 2 + (x_ + z_) // 64
    for t in (x, w, b, r):
        t.requires_grad_(False)
    assert lin.linear(x, w, b, r).grad_fn is None
    x.requires_grad_()
    with torch.no_grad():
        assert lin.linear(x, w, b, r).grad_fn is None


@gpu
def test_no_rows():
    x, w, b, r = (t.requires_grad_() for t in make(2, 24, 40, torch.float16))
    y = lin.linear(x[:0], w, b, r[:0], activation="gelu", checkpoint="e4m3")
    assert y.shape == (0, 40)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert dx.abs().sum() == 0 and dw.abs().sum() == 0 and db.abs().sum() == 0


@gpu
@pytest.mark.parametrize("rows", [1, 70, 300])
def test_infinities_and_nan_stay_in_their_rows(rows):
    dtype = torch.bfloat16
    x, w, b, r = make(rows, 200, 260, dtype)
    want = lin.linear(x, w, b, r, activation="relu")
    bad = x.clone()
    bad[rows // 2, 7] = float("inf")
    bad[0, 199] = float("nan")
    y = lin.linear(bad, w, b, r, activation="relu")
    ok = torch.ones(rows, dtype=torch.bool)
    ok[0] = ok[rows // 2] = False
    assert torch.equal(y[ok.cuda()], want[ok.cuda()])
    assert y[0].isnan().all()
    # operands end at their last value: what lies behind them in memory takes no part
    pool = torch.full((rows + 3, 208 + 16), float("nan"), dtype=dtype, device="cuda")
    pool[:rows, :200] = x
    assert torch.equal(lin.linear(pool[:rows, :200], w, b, r, activation="relu"), want)
    gpool = torch.full((rows + 3, 264), float("nan"), dtype=dtype, device="cuda")
    gpool[:rows, :260] = 0.5
    leaves = [t.detach().requires_grad_() for t in (x, w)]
    for got, g in ((gpool[:rows, :260], torch.full((rows, 260), 0.5, dtype=dtype, device="cuda")),):
        a = torch.autograd.grad(lin.linear(*leaves), leaves, got)
        c = torch.autograd.grad(lin.linear(*leaves), leaves, g)
        assert all(torch.equal(i, j) for i, j in zip(a, c))


@gpu
@pytest.mark.parametrize("rows,k,n", [(1, 4096, 4096), (24, 2048, 8192), (300, 1000, 1531), (2048, 1024, 1024)])
def test_the_same_bits_every_time(rows, k, n):
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w, gy = (torch.randn(*s, device="cuda", generator=g).bfloat16() for s in ((rows, k), (n, k), (rows, n)))
    b = torch.randn(n, device="cuda", generator=g).bfloat16()
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def once():
        y = lin.linear(x, w, b, activation="silu", checkpoint="e4m3")
        return [y.detach(), *torch.autograd.grad(y, leaves, gy)]

    first = once()
    for _ in range(3):
        assert all(torch.equal(i, j) for i, j in zip(first, once()))
    # and close to the exact values: sums of k, n and rows products in fp32, once or twice rounded
    z = x.detach().double() @ w.detach().double().t() + b.detach().double()
    y = F.silu(z)
    err = ((first[0].double() - y).norm() / y.norm()).item()
    assert err < 2.0 ** -8, err


@gpu
def test_nothing_beyond_the_outputs_is_written():
    """Through the C ABI: an output with gaps between its rows and rows behind its last."""
    lib = capi.lib()
    for dtype, code in ((torch.float16, capi.F16), (torch.bfloat16, capi.BF16)):
        for rows, k, n in ((3, 64, 130), (300, 72, 200), (257, 136, 31)):
            x, w, b, _ = make(rows, k, n, dtype)
            y = torch.full((rows + 2, n + 6), 7.0, dtype=dtype, device="cuda")
            z8 = torch.full((rows + 1, n), 9, dtype=torch.uint8, device="cuda")
            zs = torch.full((rows + 1, (n + 31) // 32), 9, dtype=torch.uint8, device="cuda")
            d = capi.LinearDesc(rows=rows, in_features=k, out_features=n, dtype=code, activation=0, y_stride=n + 6)
            capi.check(lib.winoconv_linear_forward(ctypes.byref(d), x.data_ptr(), w.data_ptr(), b.data_ptr(), None, y.data_ptr(), None, z8.data_ptr(), zs.data_ptr(),
                                                   torch.cuda.current_stream().cuda_stream), "forward")
            z, want = forward64(x, w, b, None, None)
            assert torch.equal(y[:rows, :n], want.to(dtype))
            assert (y[rows:] == 7).all() and (y[:, n:] == 7).all()
            assert (z8[rows:] == 9).all() and (zs[rows:] == 9).all()
            # sums are exact in fp32, so the eight bits are those of the exact z
            q = z8[:rows].view(torch.float8_e4m3fn).double()
            s = zs[:rows].view(torch.float8_e8m0fnu).float().double().repeat_interleave(32, 1)[:, :n]
            assert torch.equal((q * s), values8(z, torch.bfloat16))


@gpu
def test_streams_and_graphs():
    rows, k, n, dtype = 200, 264, 392, torch.bfloat16
    x, w, b, r = make(rows, k, n, dtype)
    gy = ints((rows, n), 9, 4, 2.0 ** -6, dtype)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        y = lin.linear(*leaves, activation="silu", checkpoint="e4m3")
        return [y.detach(), *torch.autograd.grad(y, leaves, gy)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(i, j) for i, j in zip(got, want))
    # two graphs, replayed with other values and in turn: nothing is shared between them or kept from the capture
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    x.copy_(ints(x.shape, 77, 8, 0.25, dtype))
    w.copy_(ints(w.shape, 78, 4, 0.125, dtype))
    want = step()
    for g, _ in graphs:
        g.replay()
    graphs[0][0].replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(i, j) for i, j in zip(out, want))
    assert capi.read_device_error() == 0


@gpu
def test_more_values_than_32_bits_count():
    """2^31 outputs and more: the last rows are those of a call on them alone, forward and backward."""
    rows, k, n, dtype = 262_147, 64, 8_200, torch.bfloat16
    assert rows * n > 2 ** 31
    x, w, b, _ = make(rows, k, n, dtype, residual=False)
    part = x[-300:].clone()
    x.requires_grad_()
    y = lin.linear(x, w, b, activation="relu", checkpoint="e4m3")
    want, = (lin.linear(part.requires_grad_(), w, b, activation="relu", checkpoint="e4m3"),)
    assert torch.equal(y[-300:], want)
    gy = torch.zeros_like(y)
    gy[-300:] = ints((300, n), 9, 4, 2.0 ** -6, dtype)
    dx, = torch.autograd.grad(y, x, gy)
    dp, = torch.autograd.grad(want, part, gy[-300:].clone())
    assert torch.equal(dx[-300:], dp) and dx[:-300].abs().max() == 0
    assert capi.read_device_error() == 0


@gpu
@pytest.mark.parametrize("rows,k,n", [(40_000, 72, 130), (33_000, 1030, 515), (50_001, 31, 65)])
def test_float_weight_gradients_of_many_rows(rows, k, n):
    """Added up over runs of rows: exact where every sum is (below 2^24 of the smallest step), and without the drift of one long
    chain where it is not: a run of 16384 rows is 1024 additions, each cuts off less than a step of 2^-23 of a sum that is half the
    last one on average, so sums of one sign are within 1024 x 2^-24."""
    x = ints((rows, k), 1, 4, 0.25, torch.float16)
    gy = ints((rows, n), 2, 4, 2.0 ** -6, torch.float16)
    w = torch.zeros(n, k, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(lin.linear(x, w), w, gy)
    assert torch.equal(dw, (gy.double().t() @ x.double()).float())
    x, gy = (torch.rand(rows, c, device="cuda", generator=torch.Generator(device="cuda").manual_seed(c)).half() for c in (k, n))
    dw, = torch.autograd.grad(lin.linear(x, w), w, gy)
    want = gy.double().t() @ x.double()
    assert ((dw.double() - want).abs() <= want * 1024 * 2.0 ** -24).all()
    assert capi.read_device_error() == 0


@gpu
def test_a_first_call_that_is_captured():
    """A fresh process whose first calls of the layer are in a capture, forward and backward: kernels are loaded and attributes set
    without a word to the stream, and the replay gives the eager values."""
    code = """
import torch
from pytorch_winoconv_b200 import capi, linear
torch.manual_seed(0)
x = torch.randn(40, 72, device="cuda").half()
w = torch.randn(104, 72, device="cuda").half().requires_grad_()
gy = torch.randn(40, 104, device="cuda").half()
def step():
    leaf = x.detach().requires_grad_()
    y = linear.linear(leaf, w, activation="gelu", checkpoint="e4m3")
    return [y.detach(), *torch.autograd.grad(y, (leaf, w), gy)]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = step()
g2 = torch.cuda.CUDAGraph()
with torch.cuda.graph(g2):
    out2 = step()
g.replay(); g2.replay(); torch.cuda.synchronize()
want = step()
assert all(torch.equal(a, b) for a, b in zip(out, want)) and all(torch.equal(a, b) for a, b in zip(out2, want))
assert capi.read_device_error() == 0
print("captured")
"""
    import os
    import subprocess
    import sys
    done = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


@gpu
def test_threads_inference_mode_and_hooks_on_saved_tensors():
    import threading
    x, w, b, r = make(130, 136, 264, torch.float16)
    gy = ints((130, 264), 9, 4, 2.0 ** -6, torch.float16)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        y = lin.linear(*leaves, activation="silu", checkpoint="e4m3")
        return [y.detach(), *torch.autograd.grad(y, leaves, gy)]

    want, got = step(), {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = [step() for _ in range(20)][-1]
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 3 and all(torch.equal(a, c) for v in got.values() for a, c in zip(v, want))
    with torch.inference_mode():
        y = lin.linear(x.clone(), w, b, r, activation="silu")
    assert torch.equal(y, want[0])
    with torch.autograd.graph.save_on_cpu():      # what is kept goes to the host and comes back
        assert all(torch.equal(a, c) for a, c in zip(step(), want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.stack([t.view(torch.uint8)] * 2, -1)[..., 0].view(t.dtype)
                                                  if t.element_size() == 1 else t):      # laid out with gaps
        assert all(torch.equal(a, c) for a, c in zip(step(), want))
    # one tensor in several places: as the input and the residual, and as the input and the weight
    s = ints((64, 64), 3, 4, 0.25, torch.float16).requires_grad_()
    g = ints((64, 64), 4, 4, 2.0 ** -6, torch.float16)
    ds, = torch.autograd.grad(lin.linear(s, s, None, s), s, g)
    gd, sd = g.double(), s.detach().double()
    parts = [gd @ sd, gd.t() @ sd, gd]
    assert ((ds.double() - sum(parts)).abs() <= 3 * sum(half_step(p, torch.float16) for p in parts) + half_step(sum(parts), torch.float16)).all()


@gpu
def test_gradients_accumulate_and_chain():
    """A feed-forward block as it would be used: two layers, the skip connection in the second's epilogue, shared weights."""
    dtype = torch.float16
    torch.manual_seed(0)
    up = lin.Linear(64, 256, activation="gelu", checkpoint="e4m3", dtype=dtype).cuda()
    down = lin.Linear(256, 64, dtype=dtype).cuda()
    x = (torch.randn(50, 64, device="cuda") * 0.5).to(dtype).requires_grad_()
    for _ in range(2):
        h = x
        for _ in range(2):                       # the same weights twice: gradients of both uses add up
            h = down(up(h), h)
        h.float().square().mean().backward()
    names = [x, *up.parameters(), *down.parameters()]
    got = [t.grad.double() / 2 for t in names]
    ref = [t.detach().double().requires_grad_() for t in names]
    h = ref[0]
    for _ in range(2):
        h = F.linear(F.gelu(F.linear(h, ref[1], ref[2])), ref[3], ref[4]) + h
    h.square().mean().backward()
    for g, t in zip(got, ref):
        # four significant bits of x and z: 2^-4 of each at most, a third of that in the mean square of many
        assert (g - t.grad).norm() <= 2.0 ** -4 * t.grad.norm()


@gpu
def test_module_follows_its_parameters():
    layer = lin.Linear(40, 24, activation="relu").cuda()
    ref = torch.nn.Linear(40, 24).cuda()
    ref.load_state_dict(layer.state_dict())
    x = torch.randn(10, 40, device="cuda", requires_grad=True)
    y = layer(x)
    assert y.dtype == torch.float16
    z64 = F.linear(x.detach().half().double(), layer.weight.detach().half().double(), layer.bias.detach().double())
    assert ((y.double() - F.relu(z64)).abs() <= half_step(z64, torch.float16) + 2.0 ** -20).all()
    y.float().sum().backward()
    assert x.grad.dtype == torch.float32 and layer.weight.grad.dtype == torch.float32 and layer.bias.grad.dtype == torch.float32
    with torch.no_grad():
        layer.weight.zero_()
        layer.bias.fill_(0.5)
    assert (layer(x) == 0.5).all()
    assert lin.Linear(8, 8, compute_dtype=None, dtype=torch.bfloat16).cuda()(torch.ones(2, 8, device="cuda", dtype=torch.bfloat16)).dtype == torch.bfloat16
    assert "activation=relu" in repr(layer)


@gpu
def test_refusals_on_the_device():
    x, w, b, r = make(4, 16, 24, torch.float16)
    for args, kw, text in (((x.float(), w), {}, "float16 or bfloat16"), ((x, w[:, :8]), {}, "input features"), ((x, w.bfloat16()), {}, "weight must be"),
                           ((x, w, b[:8]), {}, "bias must be"), ((x, w, b.double()), {}, "bias must be"), ((x, w, b, r[:1]), {}, "residual must have"),
                           ((x, w, b, r.float()), {}, "residual must be"), ((x, w.cpu()), {}, "weight is on"), ((x, w, b.cpu()), {}, "bias is on"),
                           ((x, w[:0]), {}, "not be empty"), ((x, w[0]), {}, "weight must be")):
        with pytest.raises(RuntimeError, match=text):
            lin.linear(*args, **kw)
    with pytest.raises(RuntimeError, match="not differentiable again"):
        leaf = x.clone().requires_grad_()
        torch.autograd.grad(lin.linear(leaf, w).float().sum(), leaf, create_graph=True)
    leaf = x.clone().requires_grad_()
    wl = w.clone().requires_grad_()
    y = lin.linear(leaf * 1, wl)
    with torch.no_grad():
        wl.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()


# ---- without a GPU -------------------------------------------------------------------------------------------------------
def test_refusals_of_the_python_layer():
    x, w = torch.zeros(2, 8, dtype=torch.float16), torch.zeros(4, 8, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        lin.linear(x, w)
    with pytest.raises(ValueError, match="activation must be one of"):
        lin.linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="checkpoint must be"):
        lin.linear(x, w, checkpoint="int8")
    with pytest.raises(ValueError, match="compute_dtype"):
        lin.Linear(8, 8, compute_dtype=torch.float32)
    with pytest.raises(ValueError, match="activation"):
        lin.Linear(8, 8, activation=["relu"])
    with pytest.raises(RuntimeError, match="no CPU path"):
        checkpoint.pack(x)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        checkpoint.unpack(x.to(torch.float8_e4m3fn), torch.zeros(2, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu))
    layer = lin.Linear(8, 4, activation="silu", checkpoint="e4m3")
    assert list(layer.state_dict()) == list(torch.nn.Linear(8, 4).state_dict())


def test_refusals_of_the_c_abi():
    lib = capi.lib()
    p = 1 << 20      # never dereferenced: every call is refused before a launch

    def desc(**kw):
        return ctypes.byref(capi.LinearDesc(**{**dict(rows=4, in_features=16, out_features=24, dtype=capi.F16), **kw}))

    def fwd(d, x=p, w=p, bias=None, res=None, y=p, z=None, z8=None, zs=None):
        return lib.winoconv_linear_forward(d, x, w, bias, res, y, z, z8, zs, None)

    bad, unsupported = capi.ERR_INVALID_ARGUMENT, capi.ERR_UNSUPPORTED
    for status, want in ((fwd(None), bad), (fwd(desc(dtype=capi.F32)), unsupported), (fwd(desc(activation=5)), bad), (fwd(desc(activation=-1)), bad),
                         (fwd(desc(rows=0)), bad), (fwd(desc(in_features=-1)), bad), (fwd(desc(out_features=0)), bad),
                         (fwd(desc(rows=1 << 33)), unsupported), (fwd(desc(rows=(1 << 31) - 2000, out_features=(1 << 31) - 2000)), unsupported),
                         (fwd(desc(x_stride=8)), bad), (fwd(desc(y_stride=23)), bad), (fwd(desc(z_stride=1)), bad), (fwd(desc(residual_stride=1)), bad),
                         (fwd(desc(x_stride=17)), bad), (fwd(desc(w_stride=20)), bad), (fwd(desc(in_features=15)), bad), (fwd(desc(x_stride=1 << 40)), unsupported),
                         (fwd(desc(), x=None), bad), (fwd(desc(), w=None), bad), (fwd(desc(), y=None), bad), (fwd(desc(), x=p + 8), bad),
                         (fwd(desc(), w=p + 2), bad), (fwd(desc(), y=p + 1), bad), (fwd(desc(), bias=p + 1), bad), (fwd(desc(bias_f32=1), bias=p + 2), bad),
                         (fwd(desc(), res=p + 1), bad), (fwd(desc(), z=p + 1), bad), (fwd(desc(), z8=p), bad), (fwd(desc(), zs=p), bad),
                         (fwd(desc(), z8=p + 8, zs=p), bad)):
        assert status == want, capi.last_error()
    one = desc(rows=1)      # read as they lie, but for z8
    for status, want in ((fwd(one, x=p + 1), bad), (fwd(one, w=p + 1), bad), (fwd(one, x=None), bad), (fwd(one, w=None), bad), (fwd(one, y=None), bad),
                         (fwd(one, x=p + 2, z8=p, zs=p), bad)):
        assert status == want, capi.last_error()

    def act(d, gy=p, gs=0, z=None, z8=None, zs=None, dz=p, dzs=0, db=None, dbt=0, ws=None, n=0):
        return lib.winoconv_linear_backward_activation(d, gy, gs, z, z8, zs, dz, dzs, db, dbt, ws, n, None)

    relu = desc(activation=1)
    for status, want in ((act(relu), bad), (act(relu, z=p, z8=p, zs=p), bad), (act(relu, z8=p), bad), (act(relu, z=p, gy=None), bad), (act(relu, z=p, dz=None), bad),
                         (act(relu, z=p, gs=3), bad), (act(relu, z=p, dzs=3), bad), (act(relu, z=p, db=p, dbt=9, ws=p, n=1 << 20), bad),
                         (act(relu, z=p, db=p), bad), (act(relu, z=p, db=p, ws=p, n=8), capi.ERR_WORKSPACE), (act(relu, z=p + 1), bad), (act(relu, z=p, gy=p + 1), bad)):
        assert status == want, capi.last_error()
    need = ctypes.c_uint64(0)
    assert lib.winoconv_linear_backward_ws(desc(), ctypes.byref(need)) == capi.OK and need.value >= 24 * 4
    assert lib.winoconv_linear_backward_ws(desc(), None) == bad
    data, weight = lib.winoconv_linear_backward_data, lib.winoconv_linear_backward_weight
    for status, want in ((data(desc(), p, 0, p, None, 0, None), bad), (data(desc(), p + 2, 0, p, p, 0, None), bad), (data(desc(), p, 25, p, p, 0, None), bad),
                         (data(desc(), p, 0, p, p, 8, None), bad), (data(desc(out_features=23), p, 0, p, p, 0, None), bad), (data(desc(), p, 0, None, p, 0, None), bad),
                         (weight(desc(), p, 0, p, None, 0, None), bad), (weight(desc(), p, 0, p, p, capi.BF16, None), unsupported),
                         (weight(desc(), p, 0, p + 4, p, 0, None), bad), (weight(desc(), p, 0, p, p + 2, 0, None), bad)):
        assert status == want, capi.last_error()
    def pad(count=1, **kw):
        m = (capi.Rows * 2)()
        for i in range(2):
            m[i] = capi.Rows(**{**dict(x=p, y=p, y_stride=8, rows=1, cols=8, in_dtype=capi.F16, dtype=capi.F16), **(kw if i == count - 1 else {})})
        return lib.winoconv_pad_rows(m, count, None)

    for count in (1, 2):
        for kw, want in ((dict(x=None), bad), (dict(y=None), bad), (dict(y_stride=9), bad), (dict(cols=9), bad), (dict(y=p + 8), bad), (dict(x_stride=4), bad), (dict(rows=0), bad),
                         (dict(x=p + 1), bad), (dict(x=p + 2, in_dtype=capi.F32), bad), (dict(in_dtype=capi.BF16), unsupported), (dict(dtype=capi.F32), unsupported)):
            assert pad(count, **kw) == want, capi.last_error()
    assert pad(0) == bad and pad(3) == bad and lib.winoconv_pad_rows(None, 1, None) == bad


def test_the_c_abi_reports_a_missing_device():
    if torch.cuda.is_available():
        pytest.skip("a device is there")
    p = 1 << 20
    d = capi.LinearDesc(rows=4, in_features=16, out_features=24, dtype=capi.F16)
    assert capi.lib().winoconv_linear_forward(ctypes.byref(d), p, p, None, None, p, None, None, None, None) == capi.ERR_NO_DEVICE


# ---- calls that would be recorded or differentiated as something else ---------------------------------------------------
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_recorded_calls_and_forward_mode_are_refused(device):
    """A tracer sees nothing of a layer but its empty output, and a forward-mode gradient would be lost: both are errors, on every device."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, b, r = (ints(s, i, 4, 0.25, torch.float16, device) for i, s in enumerate([(4, 40), (24, 40), (24,), (4, 24)]))
    layer = lin.Linear(40, 24, device=device, dtype=torch.float16)
    for leaves in (False, True):
        for p in layer.parameters():
            p.requires_grad_(leaves)
        for call in (lambda t: lin.linear(t, w, b, activation="gelu"), layer):
            with pytest.raises(RuntimeError, match="cannot be recorded"):
                torch.jit.trace(call, x)
            with pytest.raises(RuntimeError, match="cannot be recorded"):
                make_fx(call)(x)
    for i, t in enumerate((x, w, b, r)):
        with torch.autograd.forward_ad.dual_level():
            args = [torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) if j == i else s for j, s in enumerate((x, w, b, r))]
            with pytest.raises(RuntimeError, match="forward-mode"):
                lin.linear(*args)
    if device == "cuda":      # and nothing of it lasts
        assert torch.equal(lin.linear(x, w, b, r), forward64(x, w, b, r, None)[1].half())


# ---- how good an activation is, relative to its value --------------------------------------------------------------------
def smooth64(z, act):
    """Value, slope, the size of what the slope is a sum of, and the relative error that fp32 leaves of either.

    The exponential's argument t carries about three roundings of 2^-24 relative each (eight with the cubic), which are as many of |t|
    relative to the result; 2^-18 stands for the rest: 2^x and 1/x to a few 2^-22, a fitted tail to 2^-20, some products."""
    if act == "gelu":
        tail, density = 0.5 * torch.special.erfc(-z * 0.5 ** 0.5), torch.exp(-z * z / 2) * (2 * torch.pi) ** -0.5
        return z * tail, tail + z * density, tail + (z * density).abs(), 2.0 ** -18 + z * z * 2.0 ** -23
    if act == "gelu_tanh":
        c, a = 2 * (2 / torch.pi) ** 0.5, 0.044715
        t, dt = c * (z + a * z ** 3), c * (1 + 3 * a * z * z)
        s, off = torch.sigmoid(t), 2.0 ** -18 + t.abs() * 2.0 ** -21
    else:
        t, dt, s, off = z, 1.0, torch.sigmoid(z), 2.0 ** -18 + z.abs() * 2.0 ** -22
    bend = z * s * torch.sigmoid(-t) * dt
    return z * s, s + bend, s + bend.abs(), off


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_activations_keep_their_relative_precision(act, dtype):
    """Every value of the type up to 30 as a pre-activation, through each of the kernels: the far side of zero too is good to half a step
    of the result (and to 2^-126, below which the hardware's 2^x is zero)."""
    z = torch.arange(65536, dtype=torch.int32).to(torch.int16).cuda().view(dtype)
    z = z[z.abs() <= 30][:, None].contiguous()      # (NaN compares as false)
    one = torch.ones(1, 1, dtype=dtype, device="cuda")
    zd = z.double()
    y, slope, size, off = smooth64(zd, act)
    floor = (1 + zd.abs() + zd.abs() ** 3) * 2.0 ** -126
    check(lin.linear(z, one, activation=act), y, act, dtype, extra=y.abs() * off + floor)                                    # clusters
    check(lin.linear(one, z, activation=act), y.t(), act, dtype, extra=(y.abs() * off + floor).t())                          # one row
    many = lin.linear(z, one.expand(264, 1).contiguous(), activation=act)                                                    # pairs
    check(many[:, :1], y, act, dtype, extra=y.abs() * off + floor)
    assert torch.equal(many, many[:, :1].expand_as(many))
    for cols in (1, 8):      # the gradient's pass by single values and by vectors; each of eight equal columns gives an eighth, rounded by itself
        leaf = z.clone().requires_grad_()
        w = torch.ones(cols, 1, dtype=dtype, device="cuda")
        dx, = torch.autograd.grad(lin.linear(leaf, w, activation=act), leaf, torch.full((len(z), cols), 1 / cols, dtype=dtype, device="cuda"))
        check(dx, slope, act, dtype, extra=size * off + floor + (0 if cols == 1 else 8 * half_step(slope / 8, dtype)))
    assert capi.read_device_error() == 0


# ---- reductions longer than the tensor cores' accumulators are good for --------------------------------------------------
def halves(rows, cols, seed, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand(rows, cols, device="cuda", generator=g).mul_(scale).to(dtype)


# A run: 4096 values for float results, 16384 for f16 and 65536 for bf16.  An MMA adds 16 products to a sum; each of the 17 is cut off at
# 2^-25 of the power of two that leads the largest (two bits below the sum's last place), so a sum that grows to S evenly loses at most
# 17/2 x 2^-25 = 4.25 x 2^-24 of S for each 16 values (3.0 has been seen, of constant columns).  The runs are added in fp32, half a step
# each: at most 256 of them here, 2^-16, and so are the eight parts of a cluster.
def check_long(got, want):
    run = {torch.float32: 4096, torch.float16: 16384, torch.bfloat16: 65536}[got.dtype]
    long = run / 16 * 4.25 * 2.0 ** -24 + 2.0 ** -16
    tol = want * long + (0 if got.dtype == torch.float32 else half_step(want, got.dtype) * (1 + long))
    off = (got.double() - want).abs()
    assert (off <= tol).all(), (off / want).max().item()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,n", [(2 ** 20, 40, 24), (2 ** 20 + 17, 72, 130), (2 ** 18, 1024, 1024), (2 ** 18 + 5, 515, 1030)])
def test_weight_gradients_of_very_many_rows(rows, k, n, dtype):
    """Sums of one sign, in clusters and in pairs, by vectors and by single values."""
    x, gy = halves(rows, k, 1, dtype), halves(rows, n, 2, dtype, 2.0 ** -6)
    want = torch.zeros(n, k, dtype=torch.float64, device="cuda")
    for i in range(0, rows, 2 ** 16):
        want += gy[i:i + 2 ** 16].double().t() @ x[i:i + 2 ** 16].double()
    for w in (torch.zeros(n, k, dtype=dtype, device="cuda", requires_grad=True), torch.zeros(n, k, device="cuda", requires_grad=True)):
        dw, = torch.autograd.grad(lin.linear(x, w), w, gy)
        assert dw.dtype == w.dtype
        check_long(dw, want)
    assert capi.read_device_error() == 0


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 5, 40, 300, 2100])
def test_very_many_features(rows, dtype):
    """A long reduction in the forward pass and one in the data gradient."""
    many, few = 262_152, 264
    x, w = halves(rows, many, 1, dtype), halves(few, many, 2, dtype, 2.0 ** -4)
    want = sum(x[:, i:i + 2 ** 16].double() @ w[:, i:i + 2 ** 16].double().t() for i in range(0, many, 2 ** 16))
    check_long(lin.linear(x, w), want)
    check_long(lin.linear(x, w, halves(1, few, 3, dtype)[0] * 0, activation="relu"), want)
    w = w.t().contiguous()
    leaf = halves(rows, few, 4, dtype).requires_grad_()
    dx, = torch.autograd.grad(lin.linear(leaf, w), leaf, x)
    check_long(dx, want)
    assert capi.read_device_error() == 0


@gpu
@pytest.mark.parametrize("rows,k,n", [(33_000, 2048, 1024), (33_001, 1023, 2049), (70_000, 1024, 1024)])
def test_float_weight_gradients_of_many_rows_in_pairs(rows, k, n):
    """The same over runs in the pair kernel: exact where every sum is, and without the drift where it is not."""
    x, gy = ints((rows, k), 1, 4, 0.25, torch.float16), ints((rows, n), 2, 4, 2.0 ** -6, torch.float16)
    w = torch.zeros(n, k, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(lin.linear(x, w), w, gy)
    assert torch.equal(dw, (gy.double().t() @ x.double()).float())
    x, gy = halves(rows, k, 1, torch.float16), halves(rows, n, 2, torch.float16)
    dw, = torch.autograd.grad(lin.linear(x, w), w, gy)
    check_long(dw, gy.double().t() @ x.double())
    assert capi.read_device_error() == 0


@gpu
def test_the_longest_reduction():
    """The most rows that the C ABI takes: a tile's sum takes about the second after which a wait gives up, none of its runs does."""
    rows, dtype = (1 << 31) - 1152, torch.float16
    v = torch.arange(1, 9, device="cuda").mul(2.0 ** -12).to(dtype)
    x = v.expand(rows, 8).contiguous()
    dw = torch.full((8, 8), float("nan"), dtype=dtype, device="cuda")
    d = capi.LinearDesc(rows=rows, in_features=8, out_features=8, dtype=capi.F16)
    capi.check(capi.lib().winoconv_linear_backward_weight(ctypes.byref(d), x.data_ptr(), 0, x.data_ptr(), dw.data_ptr(), capi.F16, torch.cuda.current_stream().cuda_stream),
               "weight gradient")
    assert capi.read_device_error() == 0
    want = rows * torch.outer(v.double(), v.double())
    # 2^14 runs to each of a cluster's eight parts: as many fp32 additions, off by 2^-24 at most of sums that are half the last one on average
    assert ((dw.double() - want).abs() <= half_step(want, dtype) + want * (16384 / 16 * 4.25 * 2.0 ** -24 + 2.0 ** 14 * 2.0 ** -25)).all()


# ---- the pair kernel's forms ---------------------------------------------------------------------------------------------
# whole and odd widths with 256, 128 and 64 columns to a tile (the planner's choice for these sizes)
PAIRS = [(2000, 64, 2000), (2001, 72, 1999), (1025, 520, 1000), (1500, 64, 1111), (900, 512, 1104), (700, 512, 1100), (509, 1000, 1531)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pack", [None, "e4m3"])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows,k,n", PAIRS)
def test_smooth_layers_of_many_rows(rows, k, n, act, pack, dtype):
    """Each value of the result and of the gradients; z is exact, so what is kept of it is known too."""
    x, w, b, r = make(rows, k, n, dtype, 11)
    gy = ints((rows, n), 9, 4, 2.0 ** -3, dtype)
    for t in (x, w, b, r):
        t.requires_grad_()
    y = lin.linear(x, w, b, r, activation=act, checkpoint=pack)
    dx, dw, db, dr = torch.autograd.grad(y, (x, w, b, r), gy)
    xd, wd, rd = (t.detach().double() for t in (x, w, r))
    z = forward64(xd, wd, b.detach(), None, None)[0]
    value, _, _, off = smooth64(z, act)
    # the sum with the residual is rounded in fp32 before the result's type
    check(y.detach(), value + rd, act, dtype, extra=value.abs() * off + 2.0 ** -120 + (value + rd).abs() * 2.0 ** -24)
    kept_z, kept_x = (values8(z, dtype), values8(xd, dtype)) if pack else (z.to(dtype).double(), xd)
    _, slope, size, off = smooth64(kept_z, act)
    dz, gd = slope * gy.double(), gy.double().abs()
    raw = gd * (size * off + 2.0 ** -120)                                   # of a value of dz before its rounding
    tol_dz, sums = raw + half_step(dz, dtype) + raw * torch.finfo(dtype).eps, 2.0 ** -23
    check(dx, dz @ wd, act, dtype, extra=tol_dz @ wd.abs() + (dz.abs() @ wd.abs()) * (n / 16 + 8) * sums)
    check(dw, dz.t() @ kept_x, act, dtype, extra=tol_dz.t() @ kept_x.abs() + (dz.abs().t() @ kept_x.abs()) * (rows / 16 + 8) * sums)
    check(db, dz.sum(0), act, dtype, extra=raw.sum(0) + dz.abs().sum(0) * (rows / 8 + 16) * sums)
    assert torch.equal(dr, gy)
    assert capi.read_device_error() == 0


@gpu
@pytest.mark.parametrize("rows", [1, 40])
def test_lazily_negated_tensors(rows):
    """Tensors whose memory holds minus their values (the imaginary part of a conjugate is one) give what their copies give."""
    x, w, b, r = make(rows, 40, 24, torch.float16)
    gy = ints((rows, 24), 9, 4, 2.0 ** -6, torch.float16)
    part = torch.view_as_complex(torch.stack([torch.zeros_like(x), x], -1)).conj().imag
    assert part.is_neg() and torch.equal(part, -x)
    assert torch.equal(lin.linear(part, w, b, r), lin.linear(-x, w, b, r))
    turned = torch._neg_view
    assert torch.equal(lin.linear(x, turned(w), turned(b), turned(r)), lin.linear(x, -w, -b, -r))
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    got = torch.autograd.grad(lin.linear(turned(x), turned(w), b, r, activation="silu", checkpoint="e4m3"), leaves, turned(gy))
    want = torch.autograd.grad(lin.linear(-x, -w, b, r, activation="silu", checkpoint="e4m3"), leaves, -gy)
    assert all(torch.equal(i, j) for i, j in zip(got, want))
    with torch.no_grad():
        q, scale = checkpoint.pack(turned(x))
        assert torch.equal(checkpoint.unpack(q, scale, x.dtype), -checkpoint.unpack(*checkpoint.pack(x), x.dtype))


@gpu
@pytest.mark.parametrize("pack", [None, "e4m3"])
@pytest.mark.parametrize("rows,k,n", [(2048, 20_000, 2048), (2001, 20_000, 1999), (2304, 20_000, 1000), (1500, 20_000, 1111), (600, 20_000, 1100)])
def test_layers_with_a_long_reduction(rows, k, n, pack):
    """More than one run (f16), in pairs with 256 and 128 columns and in clusters: the whole epilogue, with sums that are exact."""
    dtype = torch.float16
    x, w, b, r = make(rows, k, n, dtype, 13)
    z = forward64(x, w, b, None, None)[0]
    for act in (None, "relu", "gelu", "gelu_tanh", "silu"):
        w.requires_grad_(act == "relu")
        y = lin.linear(x, w, b, r, activation=act, checkpoint=pack)
        want = act64(z, act) + r.double()
        off = 0 if act in (None, "relu") else smooth64(z, act)[3]
        check(y.detach(), want, act, dtype, extra=None if act in (None, "relu") else act64(z, act).abs() * off + want.abs() * 2.0 ** -24 + 2.0 ** -120)
        if act == "relu":      # through what was kept of z
            gy = ints((rows, n), 9, 4, 2.0 ** -6, dtype)
            dw, = torch.autograd.grad(y, w, gy)
            dz, kept = reference_backward(x, w.detach(), gy, z, act, dtype, pack)
            assert torch.equal(dw, (dz.t() @ kept).to(dtype))
    assert capi.read_device_error() == 0


@gpu
@pytest.mark.parametrize("pack", [None, "e4m3"])
def test_layers_that_are_computed_again_in_the_backward_pass(pack):
    """torch.utils.checkpoint runs the forward pass again from within the backward pass of the layer that asks for its saved tensors first:
    the gradients are those of the layers without it, with other operators between them and a float input before them."""
    from torch.utils.checkpoint import checkpoint as again
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.LayerNorm(64), lin.Linear(64, 96, activation="gelu", checkpoint=pack), torch.nn.Tanh(),
                              lin.Linear(96, 40, checkpoint=pack)).cuda()
    x = torch.randn(30, 64, device="cuda", requires_grad=True)
    gy = ints((30, 40), 1, 4, 2.0 ** -3, torch.float16)
    names = [x, *net.parameters()]
    want = torch.autograd.grad(net(x), names, gy)
    for reentrant in (False, True):
        for t in names:
            t.grad = None
        again(net, x, use_reentrant=reentrant).backward(gy)
        assert all(torch.equal(t.grad, g) for t, g in zip(names, want))
    hooked = []

    def unpack(t):
        with torch.enable_grad():      # (a backward pass runs without)
            hooked.append((t.detach().float().requires_grad_() * 2).requires_grad)
        return t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = net[1](x)
    y.backward(torch.ones_like(y))
    assert hooked and all(hooked)      # a hook's own operators are differentiable
