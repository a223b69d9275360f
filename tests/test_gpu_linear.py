"""The output head on the GPU against 64 bits.

Products of bf16 are exact in fp32.  With small whole numbers every partial sum is exact too, whatever its
order, so that results are equal to the last bit.  With real numbers a partial sum is cut off once per 16
products, by less than 2^-23 of itself (rms of all outputs: (K/16 + 2) 2^-23), and inside such a step each of
the 17 addends by less than 2^-23 of the largest: K 2^-22 of sum |x w| bounds any single output.  The
epilogue's functions are within 8 ulp (8 * 2^-23) and do not enlarge differences by more than 1.2; the result is rounded once.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module")
def s(lib):
    from born_b200 import Sampler
    with Sampler(device=0, max_batch=64, max_vocab=65536) as h:
        yield h


def whole(shape, seed, lo=-2, hi=3):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(lo, hi, shape, generator=g, device="cuda").to(torch.bfloat16)


@pytest.mark.parametrize("M,K,V", [(1, 8, 1), (1, 16, 7), (2, 56, 127), (3, 64, 128), (15, 72, 129), (16, 128, 1000), (17, 1000, 515),
                                   (64, 512, 18944), (65, 136, 18945), (255, 264, 900), (256, 2048, 640), (257, 64, 300), (300, 192, 19100),
                                   (512, 320, 400), (700, 64, 257), (1, 8192, 300), (40, 4096, 40000),
                                   (1, 8192, 1024), (16, 4104, 128), (33, 8000, 130), (128, 2048, 2000), (300, 3200, 1500), (512, 4096, 4096),
                                   # two tiles a CTA: alone, in pairs, with single ones behind them
                                   (9, 520, 32000), (50, 72, 32001), (128, 200, 37000), (100, 72, 45001), (70, 640, 80001),
                                   # K over clusters of two to eight, tiles of every width, lone CTAs of 256 columns
                                   (200, 2048, 1000), (256, 8192, 2001), (130, 1032, 3001), (512, 4104, 1001), (256, 520, 4096), (150, 4096, 100),
                                   (256, 2048, 128), (8, 2048, 513), (128, 4096, 1024), (1, 2048, 2048), (1, 520, 1)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_whole_numbers_are_exact(s, M, K, V, dtype):
    import torch
    x, w = whole((M, K), M + K), whole((V, K), V)
    y = s.linear(x, w, out_dtype=getattr(torch, dtype))
    want = (x.double() @ w.double().t()).to(getattr(torch, dtype))
    assert torch.equal(y, want)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strides_bias_and_residual(s, dtype):
    """Rows inside larger tensors, at any alignment of the output; what lies between them stays."""
    import torch
    M, K, V, t = 21, 200, 333, getattr(torch, dtype)
    xs, ws = whole((M, K + 24), 1), whole((V, K + 8), 2)
    x, w = xs[:, 8:8 + K], ws[:, :K]
    bias = torch.randint(-9, 9, (V,), device="cuda").float()
    for lead in (0, 1, 3):
        buf = torch.full((M * (V + 5) + 8,), -77.0, dtype=t, device="cuda")
        out = buf[lead:lead + M * (V + 5)].view(M, V + 5)[:, :V]
        res = whole((M, V + 2), 3).to(t)[:, 1:1 + V]
        assert s.linear(x, w, bias=bias, residual=res, out=out) is out
        y = x.double() @ w.double().t() + bias.double() + res.double()
        assert torch.equal(out, y.to(t))
        rest = buf.clone()
        rest[lead:lead + M * (V + 5)].view(M, V + 5)[:, :V] = -77.0
        assert (rest == -77.0).all()
        # the residual in place
        s.linear(x, w, residual=res, out=res)
        assert torch.equal(res, (y - bias.double()).to(t))


def reference(y, activation, scale):
    import torch
    if activation == "relu":
        return y.clamp(min=0)
    if activation == "sigmoid":
        return torch.sigmoid(y)
    if activation == "tanh":
        return scale * torch.tanh(y / scale)
    if activation == "gelu":
        return 0.5 * y * torch.erfc(-y / math.sqrt(2))
    if activation == "silu":
        return y * torch.sigmoid(y)
    return y


@pytest.mark.parametrize("activation,scale", [("none", 1.0), ("relu", 1.0), ("sigmoid", 1.0), ("tanh", 1.0), ("tanh", 30.0), ("gelu", 1.0), ("silu", 1.0)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,K,V", [(1, 2048, 3000), (37, 1000, 5025), (256, 4096, 2000), (3, 48, 130)])
def test_real_numbers(s, M, K, V, dtype, activation, scale):
    import torch
    g = torch.Generator(device="cuda").manual_seed(M + K)
    t = getattr(torch, dtype)
    x = torch.randn((M, K), generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn((V, K), generator=g, device="cuda") * (3 / math.sqrt(K))).to(torch.bfloat16)
    bias = torch.randn(V, generator=g, device="cuda")
    res = torch.randn((M, V), generator=g, device="cuda").to(t)
    got = s.linear(x, w, bias=bias, residual=res, activation=activation, scale=scale, out_dtype=t).double()
    lin = x.double() @ w.double().t()
    act = reference(lin + bias.double(), activation, scale)
    want = act + res.double()
    u, h = 2.0 ** -23, HALF_STEP[dtype]
    size = x.double().abs() @ w.double().abs().t()
    # sum, bias addition, function, residual addition, result
    most = 1.2 * (K * 2 * u * size + u * (lin + bias).abs()) + 8 * u * (act.abs() + 1e-30) + u * want.abs() + h * want.abs()
    if activation in ("gelu", "silu"):
        most += 8 * u * (lin + bias).abs()  # (1 + erf(y) cancels towards -inf)
    assert ((got - want).abs() <= most).all()
    rms = lambda v: float(v.square().mean().sqrt())  # noqa: E731
    assert rms(got - want) <= 1.2 * (K / 16 + 2) * u * rms(lin) + 10 * u * rms(act) + (u + h) * rms(want) + u * rms(lin + bias)


def test_one_row_does_not_touch_another(s):
    """Infinities and NaN of a row of x stay in its row of the result, those of a weight in its column."""
    import torch
    x, w = whole((20, 96), 5), whole((400, 96), 6)
    clean = s.linear(x, w)
    x[3, 5], w[7, 9] = math.nan, math.nan
    x[19, 95] = math.inf
    y = s.linear(x, w)
    assert y[3].isnan().all() and y[:, 7].isnan().all()
    assert not y[19, w[:, 95] > 0].isfinite().any()
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[3] = keep[19] = False
    keep[:, 7] = False
    assert torch.equal(y[keep], clean[keep])
    r = s.linear(x, w, activation="relu")
    assert r[3].isnan().all()


def test_offsets_past_32_bits(s):
    import torch
    K, V = 8192, 270000  # 2.2e9 weights
    w = torch.zeros((V, K), dtype=torch.bfloat16, device="cuda")
    w[-1] = 1
    w[123456, :7] = 2
    x = whole((2, K), 7)
    out = torch.empty((1 << 31) + V, dtype=torch.float32, device="cuda").as_strided((2, V), (1 << 31, 1))
    s.linear(x, w, out=out)
    assert torch.equal(out[:, -1], x.double().sum(1).float())
    assert torch.equal(out[:, 123456], 2 * x[:, :7].double().sum(1).float())
    assert int((out != 0).sum()) <= 4


def test_results_do_not_depend_on_the_run(s):
    """Parts of K are added in their order, whichever CTA comes last."""
    import torch
    for M, K, V in [(1, 8192, 1024), (100, 4096, 900)]:
        x, w = torch.randn((M, K), device="cuda").to(torch.bfloat16), torch.randn((V, K), device="cuda").to(torch.bfloat16)
        y = s.linear(x, w)
        for _ in range(5):
            assert torch.equal(s.linear(x, w), y)


def test_graph_and_stream(s):
    import torch
    x, w = whole((33, 256), 8), whole((2000, 256), 9)
    want = (x.double() @ w.double().t()).float()
    out = torch.zeros((33, 2000), device="cuda")
    call = s.prepare_linear(x, w, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        call.run(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        out.zero_()
        x.copy_(-x)
        g.replay()
        want = -want
        assert torch.equal(out, want)
    s.check_error()


def test_refusals(s):
    import torch
    from born_b200 import InvalidArgument, SamplerError, _lib as L
    x, w = whole((4, 64), 1), whole((100, 64), 2)

    def bad(error, code, f, *a, **kw):
        with pytest.raises(error) as e:
            f(*a, **kw)
        assert e.value.code == code, e.value

    inv, uns = (InvalidArgument, L.ERR_INVALID_ARGUMENT), (SamplerError, L.ERR_UNSUPPORTED)
    bad(*inv, s.linear, x.float(), w)
    bad(*inv, s.linear, x, w.half())
    bad(*inv, s.linear, x.cpu(), w)
    bad(*inv, s.linear, x[0], w)
    bad(*inv, s.linear, x, w[:, :56])
    bad(*inv, s.linear, x.t(), w)
    bad(*inv, s.linear, x, w, activation="swish")
    bad(*inv, s.linear, x, w, scale=-1.0)
    bad(*inv, s.linear, x, w, scale=math.nan)
    bad(*inv, s.linear, x, w, bias=torch.zeros(99, device="cuda"))
    bad(*inv, s.linear, x, w, bias=torch.zeros(100, device="cuda", dtype=torch.bfloat16))
    bad(*inv, s.linear, x, w, residual=torch.zeros((4, 100), device="cuda", dtype=torch.bfloat16))
    bad(*inv, s.linear, x, w, residual=torch.zeros((4, 99), device="cuda"))
    bad(*inv, s.linear, x, w, out=torch.zeros((4, 200), device="cuda")[:, ::2])
    bad(*inv, s.linear, x, w, out_dtype=torch.float16)
    bad(*inv, s.linear, x[:0], w)
    bad(*uns, s.linear, x[:, :60], w[:, :60])                       # no multiple of 8
    bad(*uns, s.linear, whole((4, 72), 1)[:, 1:65], w)              # rows off the 16-byte boundaries
    bad(*uns, s.linear, whole((4, 68), 1)[:, :64], w)
    call = s.prepare_linear(x, w)
    for field, value, err in [("struct_size", 4, inv), ("memory", L.MEM_HOST, uns), ("rows", 0, inv), ("out_dtype", 3, inv), ("activation", 6, inv),
                              ("out", None, inv), ("out_row_stride", 99, inv), ("weight_row_stride", 63, inv)]:
        keep = getattr(call.args, field)
        setattr(call.args, field, value)
        bad(*err, call.run)
        setattr(call.args, field, keep)


def test_sizes_that_are_refused(s):
    from born_b200 import InvalidArgument, SamplerError, _lib as L
    call = s.prepare_linear(whole((4, 64), 1), whole((100, 64), 2), activation="tanh")
    for field in ("rows", "hidden", "features"):
        keep = getattr(call.args, field)
        setattr(call.args, field, 2 ** 31 - 1000)
        with pytest.raises(SamplerError) as e:
            call.run()
        assert e.value.code == L.ERR_UNSUPPORTED
        setattr(call.args, field, keep)
    call.args.scale = 1e-40  # whose inverse is no number
    with pytest.raises(InvalidArgument):
        call.run()
