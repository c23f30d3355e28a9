"""Activations in eight bits (``checkpoint``) against their definition in 64 bits: equality everywhere."""
import pytest
import torch

from pytorch_winoconv_b200 import capi, checkpoint
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


def test_refusals_of_the_c_abi():
    lib, p = capi.lib(), 1 << 20
    bad = capi.ERR_INVALID_ARGUMENT
    for f in (lambda dt, x, xs, r, c, q, s: lib.winoconv_e4m3_pack(dt, x, xs, r, c, q, s, None),
              lambda dt, x, xs, r, c, q, s: lib.winoconv_e4m3_unpack(dt, q, s, r, c, x, xs, None)):
        for args, want in (((capi.F32, p, 0, 1, 8, p, p), capi.ERR_UNSUPPORTED), ((capi.F16, None, 0, 1, 8, p, p), bad), ((capi.F16, p, 0, 1, 8, None, p), bad),
                           ((capi.F16, p, 0, 1, 8, p, None), bad), ((capi.F16, p, 0, 0, 8, p, p), bad), ((capi.F16, p, 0, 1, 0, p, p), bad), ((capi.BF16, p, 7, 1, 8, p, p), bad),
                           ((capi.BF16, p + 1, 0, 1, 8, p, p), bad), ((capi.BF16, p, 0, 1 << 40, 8, p, p), capi.ERR_UNSUPPORTED)):
            assert f(*args) == want, capi.last_error()
