"""Activations in eight bits (``checkpoint``) against their definition in 64 bits: equality everywhere."""
import pytest
import torch

from pytorch_winoconv_b200 import capi, checkpoint, conv
from tests.test_linear import values8

gpu = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


def check(x):
    q, scale = checkpoint.pack(x)
    assert q.shape == x.shape and q.dtype == torch.float8_e4m3fn and q.is_contiguous()
    assert scale.shape == (*x.shape[:-1], -(-x.shape[-1] // 32)) and scale.dtype == torch.float8_e8m0fnu
    want = values8(x.double(), x.dtype)
    for dtype in DTYPES:
        got = checkpoint.unpack(q, scale, dtype)
        assert got.dtype == dtype and got.shape == x.shape
        if dtype == x.dtype:
            assert torch.equal(got.double().nan_to_num(12345.0), want.nan_to_num(12345.0))
    # what is held, times the scale
    s = scale.float().double().repeat_interleave(32, -1)[..., :x.shape[-1]]
    most = torch.finfo(x.dtype).max
    assert torch.equal((q.double() * s).clamp(-most, most).nan_to_num(12345.0), want.nan_to_num(12345.0))
    return q, scale


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33), (7, 64), (2, 3, 40), (100, 72), (1001, 777), (64, 4096), (1, 100003), (5000, 8), (2048, 1)])
def test_values_and_scales(shape, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(shape, device="cuda", generator=g) * torch.exp2(torch.randint(-14, 6, shape, device="cuda", generator=g).float())
    q, scale = check(x.to(dtype))
    # the smallest power of two that holds the block: half of it would not
    pad = torch.nn.functional.pad(x.to(dtype).double(), (0, -shape[-1] % 32)).reshape(*shape[:-1], -1, 32)
    top, s = pad.abs().amax(-1), scale.float().double()
    assert (top <= 448 * s).all() and ((top > 224 * s) | (s == 2.0 ** -127)).all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_value_of_the_type(dtype):
    """All 65536 bit patterns: as the only value of a block, and next to a large one."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).cuda()
    every = bits.view(dtype)
    alone = torch.zeros(65536, 32, dtype=dtype, device="cuda")
    alone[:, 5] = every
    check(alone)
    alone[:, 9] = 1.75
    check(alone)
    check(every.reshape(-1, 64))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_borders_and_special_values(dtype):
    inf, nan, most = float("inf"), float("nan"), torch.finfo(dtype).max
    rows = [[0.0] * 32, [-0.0, 0.0] * 16, [448.0] + [k / 16 + 1 / 32 for k in range(16, 47)], [1.75] * 32, [1.7578125] + [1.0] * 31, [inf] + [1.0] * 31, [nan] + [3.0] * 31,
            [inf] * 32, [nan] * 32, [-inf, nan, inf] + [2.0 ** -10] * 29, [most] + [1.0] * 31, [-most] * 32, [torch.finfo(dtype).smallest_normal] * 32,
            [torch.finfo(dtype).tiny * torch.finfo(dtype).eps] * 32]
    x = torch.tensor(rows, dtype=torch.float64).to(dtype).cuda()
    q, scale = check(x)
    got = checkpoint.unpack(q, scale, dtype)
    assert got[0].abs().sum() == 0 and got[10, 0] == most and (got[11] == -most).all()      # no infinity where there was none
    assert got[5, 0].isnan() and (got[5, 1:] == 1).all()                                    # and none kept: an overflow stays visible as NaN
    assert torch.equal(got[3], x[3]) and got[7].isnan().all()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_views(dtype):
    g = torch.Generator(device="cuda").manual_seed(2)
    base = torch.randn(60, 200, device="cuda", generator=g).to(dtype)
    for x in (base[:, 8:104], base[:, 3:100], base[::3, :64], base.t(), base[:, ::2], base[7:8, 1:], base[0], base[:1].expand(5, 200), base.reshape(3, 20, 200).transpose(0, 1),
              base[:, :64][:, None, :]):
        q, scale = check(x)
        again = checkpoint.pack(x.contiguous())
        assert torch.equal(q.view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(scale.view(torch.uint8), again[1].view(torch.uint8))
    q, scale = checkpoint.pack(base)
    part = checkpoint.unpack(q[5:40], scale[5:40], dtype)
    assert torch.equal(part, checkpoint.unpack(q, scale, dtype)[5:40])
    assert torch.equal(checkpoint.unpack(q[:, 1:30], scale[:, :1], dtype), checkpoint.unpack(q, scale, dtype)[:, 1:30])      # a copy not on 16 bytes


@gpu
def test_more_values_than_32_bits_count():
    for cols in (4104, 4099):      # by vectors and one by one
        rows = 2 ** 31 // cols + 100
        x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
        x[-50:] = torch.randn(50, cols, device="cuda").bfloat16()
        q, scale = checkpoint.pack(x)
        part = checkpoint.pack(x[-50:].clone())
        assert torch.equal(q[-50:].view(torch.uint8), part[0].view(torch.uint8)) and torch.equal(scale[-50:].view(torch.uint8), part[1].view(torch.uint8))
        del x
        got = checkpoint.unpack(q, scale)
        assert torch.equal(got[-50:], checkpoint.unpack(*part)) and got[:50].abs().max() == 0
        del got, q, scale


@gpu
def test_empty_streams_and_graphs():
    q, scale = checkpoint.pack(torch.empty(0, 40, dtype=torch.float16, device="cuda"))
    assert q.shape == (0, 40) and scale.shape == (0, 2) and checkpoint.unpack(q, scale).shape == (0, 40)
    x = torch.randn(64, 96, device="cuda").bfloat16().requires_grad_()
    q, scale = checkpoint.pack(x)
    assert not q.requires_grad
    want = checkpoint.unpack(q, scale)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = checkpoint.unpack(*checkpoint.pack(x))
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = checkpoint.unpack(*checkpoint.pack(x))
    with torch.no_grad():
        x.mul_(-2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, -2 * want)


@gpu
def test_refusals_on_the_device():
    x = torch.zeros(4, 40, dtype=torch.float16, device="cuda")
    q, scale = checkpoint.pack(x)
    for call, text in ((lambda: checkpoint.pack(x.float()), "float16 or bfloat16"), (lambda: checkpoint.pack(x[:, :0]), "not empty"),
                       (lambda: checkpoint.pack(x[0, 0]), "not empty"), (lambda: checkpoint.unpack(q, scale, torch.float32), "float16 or bfloat16"),
                       (lambda: checkpoint.unpack(q, scale[:, :1]), "scale must be"), (lambda: checkpoint.unpack(q[:3], scale), "scale must be"),
                       (lambda: checkpoint.unpack(x, scale), "float8_e4m3fn"), (lambda: checkpoint.unpack(q, scale.cpu()), "same one")):
        with pytest.raises(RuntimeError, match=text):
            call()


# ---- convolution layers that keep their input in eight bits ----------------------------------------------------------------
LAYERS = [(conv.Conv2d, (2, 16, 9, 11), 24, 3, 1, 1, True), (conv.Conv2d, (3, 5, 14, 10), 8, 3, 2, 1, True), (conv.Conv2d, (2, 72, 12, 8), 40, 5, 1, 2, False),
          (conv.Conv2d, (4, 64, 7, 7), 31, 1, 1, 0, True), (conv.Conv3d, (2, 8, 5, 6, 7), 16, 3, 1, 1, True)]


def rounded(x):
    """x as eight bits hold it, per pixel over the channels."""
    return checkpoint.unpack(*checkpoint.pack(x.movedim(1, -1)), x.dtype).movedim(-1, 1)


@gpu
@pytest.mark.parametrize("cls,shape,k,ks,stride,pad,bias", LAYERS)
@pytest.mark.parametrize("activation", [None, "relu"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_convolution_layers(cls, shape, k, ks, stride, pad, bias, activation, dtype):
    """Result, data and bias gradient are those of the layer without it, to the bit; the weight gradient is that of the rounded input."""
    torch.manual_seed(3)
    args, kw = (shape[1], k, ks), dict(stride=stride, padding=pad, bias=bias, compute_dtype=dtype)
    plain = cls(*args, activation=activation, **kw).cuda()
    kept = cls(*args, activation=activation, checkpoint="e4m3", **kw).cuda()
    linear = cls(*args, **kw).cuda()
    for m in (kept, linear):
        m.load_state_dict(plain.state_dict())
    x = torch.randn(shape, device="cuda").to(dtype).requires_grad_()

    def run(m, t, gy=None):
        y = m(t)
        gy = torch.randn(y.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype) if gy is None else gy
        return y.detach(), gy, torch.autograd.grad(y, [t, *m.parameters()], gy)

    y0, gy, g0 = run(plain, x)
    y1, _, g1 = run(kept, x)
    assert torch.equal(y0, y1) and torch.equal(g0[0], g1[0])
    if bias:
        assert torch.equal(g0[2], g1[2])
    masked = gy * (y0 > 0).to(dtype) if activation else gy
    _, _, g2 = run(linear, rounded(x.detach()).requires_grad_(), masked)
    assert torch.equal(g1[1], g2[1])
    assert not torch.equal(g1[1], g0[1])
    assert capi.read_device_error() == 0


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 1000, 8192, 100_003])
def test_signs(n, dtype):
    lib, code = capi.lib(), capi.F16 if dtype == torch.float16 else capi.BF16
    y = torch.randn(n + 8, device="cuda").to(dtype)
    y[:n:5] = 0
    y[:n:11] = -0.0
    y[n // 2] = float("nan")
    gy = torch.randn(n, device="cuda").to(dtype)
    bits = torch.full(((n + 7) // 8 + 3,), 0xAA, dtype=torch.uint8, device="cuda")
    gx = torch.full((n + 8,), 7.0, dtype=dtype, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    capi.check(lib.winoconv_sign_pack(code, y.data_ptr(), n, bits.data_ptr(), s), "sign_pack")
    capi.check(lib.winoconv_sign_apply(code, gy.data_ptr(), bits.data_ptr(), n, gx.data_ptr(), s), "sign_apply")
    on = torch.stack([(bits[:(n + 7) // 8].int() >> i) & 1 for i in range(8)], 1).flatten()
    assert torch.equal(on[:n].bool(), y[:n] > 0) and on[n:].sum() == 0 and (bits[(n + 7) // 8:] == 0xAA).all()
    assert torch.equal(gx[:n], gy * (y[:n] > 0).to(dtype)) and (gx[n:] == 7).all()
    assert capi.read_device_error() == 0


@gpu
def test_what_a_convolution_layer_keeps():
    layer = conv.Conv2d(64, 32, 3, padding=1, activation="relu", checkpoint="e4m3").cuda()
    x = torch.randn(4, 64, 20, 20, device="cuda", requires_grad=True)      # float input: kept as the rounded operand's eight bits
    size = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: size.append(t.numel() * t.element_size()) or t, lambda t: t):
        y = layer(x)
    assert sorted(size) == sorted([x.numel(), x.numel() // 32, y.numel() // 8])
    y.float().sum().backward()
    assert x.grad.dtype == torch.float32 and layer.weight.grad is not None
    layer.weight.requires_grad_(False)
    size.clear()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: size.append(t.numel() * t.element_size()) or t, lambda t: t):
        y = layer(x)
    assert size == [y.numel() // 8]
    plain = conv.Conv2d(64, 32, 3, padding=1, activation="relu").cuda()
    plain.load_state_dict(layer.state_dict())
    dx, db = torch.autograd.grad(y.float().sum(), (x, layer.bias))
    dx2, db2 = torch.autograd.grad(plain(x).float().sum(), (x, plain.bias))
    # (the bias gradient without the weight gradient beside it is another order of the same sum of ones)
    assert torch.equal(dx, dx2) and torch.equal(db, db2)
    assert layer.eval()(x).grad_fn is not None and "checkpoint=e4m3" in repr(layer)


@gpu
def test_a_convolution_and_a_linear_layer_in_a_captured_step():
    """A small network as it would be trained, both layers keeping eight bits: the captured step gives the eager one's gradients."""
    from pytorch_winoconv_b200 import linear
    torch.manual_seed(0)
    body = conv.Conv2d(8, 32, 3, padding=1, activation="relu", checkpoint="e4m3").cuda()
    head = linear.Linear(32 * 36, 10, checkpoint="e4m3").cuda()
    x = torch.randn(6, 8, 6, 6, device="cuda")
    params = [*body.parameters(), *head.parameters()]

    def step():
        y = head(body(x).flatten(1))
        return [y.detach(), *torch.autograd.grad(y.float().square().mean(), params)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x.copy_(torch.randn(6, 8, 6, 6, device="cuda"))
    with torch.no_grad():
        for p in params:
            p.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))
    assert capi.read_device_error() == 0


@gpu
def test_convolution_refusals_on_the_device():
    layer = conv.Conv2d(4, 8, 3, compute_dtype=None, checkpoint="e4m3").cuda()
    with pytest.raises(NotImplementedError, match="checkpoint"):
        layer(torch.randn(1, 4, 8, 8, device="cuda", requires_grad=True))      # computes in float32
    with torch.no_grad():
        assert layer(torch.randn(1, 4, 8, 8, device="cuda")).shape == (1, 8, 6, 6)      # nothing to keep


def test_convolution_refusals():
    with pytest.raises(ValueError, match="checkpoint"):
        conv.Conv2d(4, 8, 3, checkpoint="int8")
    with pytest.raises(NotImplementedError, match="checkpoint"):
        conv.Conv3d(4, 8, 3, compute_dtype=torch.float32, checkpoint="e4m3")


def test_refusals_of_the_c_abi():
    lib, p = capi.lib(), 1 << 20
    bad = capi.ERR_INVALID_ARGUMENT
    for f in (lambda dt, x, xs, r, c, q, s: lib.winoconv_e4m3_pack(dt, x, xs, r, c, q, s, None),
              lambda dt, x, xs, r, c, q, s: lib.winoconv_e4m3_unpack(dt, q, s, r, c, x, xs, None)):
        for args, want in (((capi.F32, p, 0, 1, 8, p, p), capi.ERR_UNSUPPORTED), ((capi.F16, None, 0, 1, 8, p, p), bad), ((capi.F16, p, 0, 1, 8, None, p), bad),
                           ((capi.F16, p, 0, 1, 8, p, None), bad), ((capi.F16, p, 0, 0, 8, p, p), bad), ((capi.F16, p, 0, 1, 0, p, p), bad), ((capi.BF16, p, 7, 1, 8, p, p), bad),
                           ((capi.BF16, p + 1, 0, 1, 8, p, p), bad), ((capi.BF16, p, 0, 1 << 40, 8, p, p), capi.ERR_UNSUPPORTED)):
            assert f(*args) == want, capi.last_error()
    for f in (lambda dt, a, n, bits: lib.winoconv_sign_pack(dt, a, n, bits, None), lambda dt, a, n, bits: lib.winoconv_sign_apply(dt, a, bits, n, p, None),
              lambda dt, a, n, bits: lib.winoconv_sign_apply(dt, p, bits, n, a, None)):
        for args, want in (((capi.F32, p, 8, p), capi.ERR_UNSUPPORTED), ((capi.F16, None, 8, p), bad), ((capi.F16, p, 8, None), bad), ((capi.F16, p, 0, p), bad),
                           ((capi.F16, p + 2, 8, p), bad), ((capi.F16, p, 1 << 41, p), capi.ERR_UNSUPPORTED)):
            assert f(*args) == want, capi.last_error()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_recorded_calls_and_forward_mode_are_refused(device):
    from torch.fx.experimental.proxy_tensor import make_fx
    x = torch.randn(4, 40, device=device).half()
    q, scale = torch.zeros(4, 40, device=device).to(torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
    for call, args in ((lambda t: checkpoint.pack(t)[0].view(torch.uint8), (x,)), (lambda a, s: checkpoint.unpack(a, s), (q, scale))):
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            torch.jit.trace(call, args)
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            make_fx(call)(*args)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            checkpoint.pack(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))


@gpu
def test_gradients_of_convolutions_in_eight_bits_are_not_differentiable_again():
    """They would come back as constants, and a penalty on them would be left out of a loss without a word."""
    layer = conv.Conv2d(8, 16, 3, activation="relu", checkpoint="e4m3").cuda()
    x = torch.randn(2, 8, 9, 9, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="not differentiable again"):
        torch.autograd.grad(layer(x).float().square().sum(), x, create_graph=True)


@gpu
@pytest.mark.parametrize("activation", [None, "relu"])
def test_convolutions_computed_again_and_kept_on_the_host(activation):
    from torch.utils.checkpoint import checkpoint as again
    torch.manual_seed(0)
    net = torch.nn.Sequential(conv.Conv2d(8, 40, 3, padding=1, activation=activation, checkpoint="e4m3"), torch.nn.Tanh(),
                              conv.Conv2d(40, 12, 3, activation=activation, checkpoint="e4m3")).cuda()
    x = torch.randn(3, 8, 11, 9, device="cuda", requires_grad=True)
    names = [x, *net.parameters()]
    want = torch.autograd.grad(net(x).float().square().sum(), names)
    again(net, x, use_reentrant=False).float().square().sum().backward()
    assert all(torch.equal(t.grad, g) for t, g in zip(names, want))
    with torch.autograd.graph.save_on_cpu():
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(net(x).float().square().sum(), names), want))
    crop = torch.randn(3, 12, 13, 14, device="cuda")[:, 2:10, 1:12, 3:12].requires_grad_()
    whole = crop.detach().clone().requires_grad_()
    assert torch.equal(*(torch.autograd.grad(net(t).float().square().sum(), t)[0] for t in (crop, whole)))
