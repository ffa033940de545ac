"""8-bit rows and their product on sm_100a against the 64-bit oracle.

Codes and scales are exact (the definition rounds the exact quotient), the
values read back are one fp32 rounding and one to the output's type.  A
product's integer sum is exact; on its way out it is rounded to fp32, scaled
twice and (with a bias) added once, 2^-24 each relative to the scaled sum or
the result, then rounded to the output's type (half a step: eps / 2, and half
the smallest subnormal)."""
import numpy as np
import pytest
import torch

import memboost_b200 as mb
from memboost_b200 import gptq
from oracle import serving

pytestmark = pytest.mark.gpu

TYPES = [torch.float16, torch.bfloat16, torch.float32]
IDS = ["fp16", "bf16", "fp32"]


def _x(rows, K, dtype, seed=0, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, K), generator=g)
    if spread:  # rows of very different size
        x = x * torch.exp2(torch.randint(-12, 8, (rows, 1), generator=g).float())
    return x.to(dtype)


def _np(t):
    return t.detach().cpu().double().numpy()


def _check_rows(t, x):
    codes, scales = serving.quantize_rows(_np(x))
    assert np.array_equal(t.codes.cpu().numpy(), codes)
    assert np.array_equal(t.scales.cpu().numpy(), scales, equal_nan=True)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 17), (3, 16), (5, 33), (70, 8), (129, 1000),
                                    (7, 1024), (4, 1025), (9, 4096), (3, 5000), (2, 8193),
                                    (3, 16391), (1, 40000), (2, 131072)])
def test_rows_exact(rows, K, dtype):
    x = _x(rows, K, dtype, seed=rows * 1000 + K)
    t = mb.quantize_int8(x.cuda())
    assert t.codes.stride(0) % 16 == 0 and t.scales.dtype == torch.float32
    _check_rows(t, x)
    for out in TYPES:
        got = mb.dequantize_int8(t, out)
        want = torch.from_numpy(serving.dequantize_rows(t.codes.cpu().numpy(),
                                                        t.scales.cpu().numpy())).to(out)
        assert torch.equal(got.cpu(), want)


def test_rows_ties_and_borders():
    """scale 1: every half is a tie (to even); scales that put many quotients
    within an fp32 rounding of a border."""
    x = torch.cat((torch.arange(-126.5, 127), torch.tensor([127.0]))).unsqueeze(0)
    _check_rows(mb.quantize_int8(x.cuda()), x)
    g = torch.Generator().manual_seed(5)
    amax = torch.rand((512, 1), generator=g) + 1
    s = amax.double() / 127
    half = torch.randint(-127, 127, (512, 255), generator=g).double() + 0.5
    x = (half * s).float()  # rounds to either side of the border
    x = torch.cat((amax, x.clamp(-1, 1) * amax.abs().clamp(max=1)), 1).float()
    _check_rows(mb.quantize_int8(x.cuda()), x)


def test_rows_of_zeros_nan_infinity_and_tiny():
    x = _x(9, 200, torch.float32, seed=2, spread=False)
    x[1] = 0
    x[2, 150] = float("nan")
    x[3, 7] = float("inf")
    x[4, 199] = -float("inf")
    x[5] *= 1e-38                 # a subnormal scale
    x[6] = 0
    x[6, 3] = 1e-45               # the scale underflows to 0
    x[7] = 3e38 * torch.sign(x[7])
    x[8] *= 1e-33                 # 1 / scale near the end of fp32
    t = mb.quantize_int8(x.cuda())
    _check_rows(t, x)
    y = mb.dequantize_int8(t, torch.float32).cpu()
    assert torch.isnan(y[2:5]).all() and (y[1] == 0).all() and (y[6] == 0).all()
    assert torch.isfinite(y[7]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_rows_strides(dtype):
    x = _x(40, 121, dtype, seed=3).cuda()
    for view in (x[:, 1:], x[::3, 5:70], x[1:, :64], x.t(), x[7], x.view(4, 10, 121),
                 x[:1].expand(5, 121), x[:, :1].expand(40, 30), x.view(4, 10, 121)[:, ::2],
                 x.view(4, 10, 121).transpose(0, 1), x[:, :1], x.t()[:, :1]):
        t = mb.quantize_int8(view)
        _check_rows(t, view.reshape(-1, view.shape[-1]))


def test_rows_empty_and_out():
    assert mb.quantize_int8(torch.zeros((0, 40), dtype=torch.float16, device="cuda")).shape \
        == (0, 40)
    t = mb.quantize_int8(torch.zeros((3, 2, 0), dtype=torch.float16, device="cuda"))
    assert t.shape == (6, 0) and (t.scales == 0).all()
    t = mb.quantize_int8(_x(5, 40, torch.float16).cuda())
    out = torch.full((7, 40), 9.0, dtype=torch.float16, device="cuda")
    assert mb.dequantize_int8(t, torch.float16, out=out[1:6]).data_ptr() == out[1].data_ptr()
    assert (out[0] == 9).all() and (out[6] == 9).all()
    assert torch.equal(out[1:6], mb.dequantize_int8(t))
    for bad in (out, out[1:6].float(), out[:5, :20]):
        with pytest.raises(RuntimeError, match="out must be"):
            mb.dequantize_int8(t, torch.float16, out=bad)


def _check_product(y, a, w, bias=None):
    want, mag = serving.matmul(a.codes.cpu().numpy(), a.scales.cpu().numpy(),
                               w.codes.cpu().numpy(), w.scales.cpu().numpy(),
                               None if bias is None else _np(bias))
    f = torch.finfo(y.dtype)
    u = 2.0 ** -24
    work = mag * ((1 + u) ** 3 - 1) + (0 if bias is None else u * (np.abs(want) + 4 * u * mag))
    tol = work + (f.eps / 2) * (np.abs(want) + work) + f.tiny * f.eps / 2
    err = np.abs(_np(y).reshape(want.shape) - want)
    assert np.all(err <= tol), (err - tol).max()


SIZES = [(1, 1, 1), (1, 16, 16), (2, 8, 33), (3, 130, 64), (17, 4096, 1000), (16, 257, 128),
         (33, 65, 129), (64, 64, 4096), (65, 4100, 40), (100, 1000, 1001), (129, 129, 257),
         (128, 256, 512), (257, 513, 300), (300, 40, 2050), (1, 5000, 11008), (520, 768, 1024),
         (1000, 3, 70), (7, 40, 20000), (2300, 2100, 300),
         (4100, 1300, 40), (300, 19100, 1700), (2049, 2561, 2049)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(M, N, K, dtype):
    x = _x(M, K, dtype, seed=M + N + K).cuda()
    w = mb.quantize_int8(_x(N, K, torch.float32, seed=N, spread=False).cuda() * 0.02)
    a = mb.quantize_int8(x)
    y = mb.int8_matmul(x, w)
    assert y.dtype == dtype and tuple(y.shape) == (M, N)
    _check_product(y, a, w)
    bias = _x(1, N, dtype, seed=9, spread=False)[0].cuda()
    _check_product(mb.int8_matmul(x, w, bias=bias), a, w, bias)
    for out in TYPES:  # given codes: the same product
        assert torch.equal(mb.int8_matmul(a, w, out_dtype=out),
                           mb.int8_matmul(x, w, out_dtype=out))


@pytest.mark.parametrize("M", [1, 16, 64, 65, 256])
@pytest.mark.parametrize("N,K", [(19100, 300), (32000, 1024)])
def test_product_few_tokens_over_many_channels(M, N, K):
    """On either side of where the kernel changes: the sums are whole numbers,
    so a wide product equals its parts'."""
    x = _x(M, K, torch.bfloat16, seed=M).cuda()
    w = mb.quantize_int8(_x(N, K, torch.float32, seed=N, spread=False).cuda() * 0.02)
    y = mb.int8_matmul(x, w)
    parts = [mb.Int8Tensor(w.codes[n:n + 3000], w.scales[n:n + 3000]) for n in range(0, N, 3000)]
    assert torch.equal(y, torch.cat([mb.int8_matmul(x, p) for p in parts], 1))
    some = slice(N - 500, N)
    _check_product(y[:, some], mb.quantize_int8(x), mb.Int8Tensor(w.codes[some], w.scales[some]))


@pytest.mark.parametrize("M", [1, 20, 150, 600])
def test_product_largest_sums(M):
    """All codes +-127 over the longest K: sums next to 2^31."""
    K, N = 131072, 40
    codes = torch.full((M + N, K), 127, dtype=torch.int8, device="cuda")
    codes[M + 1] = -127
    one = torch.ones(M + N, device="cuda")
    y = mb.int8_matmul(mb.Int8Tensor(codes[:M], one[:M]), mb.Int8Tensor(codes[M:], one[M:]),
                       out_dtype=torch.float32)
    want = torch.full((M, N), 127.0 * 127.0 * K)
    want[:, 1] *= -1
    assert torch.equal(y.cpu(), want.float())


def test_product_not_finite_rows():
    x = _x(40, 300, torch.float16, seed=1, spread=False).cuda()
    x[3, 5], x[39, 0] = float("nan"), float("inf")
    w = mb.quantize_int8(_x(50, 300, torch.float16, seed=2, spread=False).cuda())
    w.scales[7] = float("nan")
    y = mb.int8_matmul(x, w)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[3], bad[39], bad[:, 7] = True, True, True
    assert torch.equal(torch.isnan(y), bad)


def test_product_layouts():
    """Leading dimensions, strided inputs, a slice of a weight's rows, an
    output given, empty batches."""
    x = _x(24, 200, torch.bfloat16, seed=4).cuda()
    w = mb.quantize_int8(_x(96, 200, torch.float32, seed=5, spread=False).cuda())
    full = mb.int8_matmul(x, w)
    assert torch.equal(mb.int8_matmul(x.view(2, 3, 4, 200), w).view(24, 96), full)
    assert torch.equal(mb.int8_matmul(x[5], w), full[5])
    assert torch.equal(mb.int8_matmul(x[::2], w), full[::2])
    assert torch.equal(mb.int8_matmul(x.t().contiguous().t(), w), full)
    part = mb.Int8Tensor(w.codes[32:64], w.scales[32:64])
    assert torch.equal(mb.int8_matmul(x, part), full[:, 32:64])
    every = mb.Int8Tensor(w.codes[::3], w.scales[::3])
    assert torch.equal(mb.int8_matmul(x, every), full[:, ::3])
    out = torch.full((26, 96), 7.0, dtype=torch.bfloat16, device="cuda")
    mb.int8_matmul(x, w, out=out[1:25])
    assert torch.equal(out[1:25], full) and (out[0] == 7).all() and (out[25] == 7).all()
    assert mb.int8_matmul(x[:0], w).shape == (0, 96)
    assert mb.int8_matmul(x, mb.Int8Tensor(w.codes[:0], w.scales[:0])).shape == (24, 0)
    moved = w.to("cuda")
    assert torch.equal(mb.int8_matmul(x, moved), full)


def test_product_refusals():
    x = _x(4, 64, torch.float16).cuda()
    w = mb.quantize_int8(_x(8, 64, torch.float16).cuda())
    cases = [
        (dict(x=x[:, :32]), "64 columns"), (dict(x=x.double()), "float16 or bfloat16 or float32"),
        (dict(x=x.cpu()), "device of w"), (dict(bias=x[0]), r"bias must be \[8\]"),
        (dict(bias=torch.zeros(8, device="cuda", dtype=torch.int32)), "bias must be float16"),
        (dict(out=torch.empty((4, 8), device="cuda")), "out must be"),
        (dict(out_dtype=torch.int32), "out_dtype must be"),
        (dict(w=mb.Int8Tensor(w.codes[:, 1:], w.scales)), "16-byte"),
        (dict(w=mb.Int8Tensor(w.codes.t().contiguous().t(), w.scales)), "16-byte"),
        (dict(w=mb.Int8Tensor(w.codes, w.scales[:4])), "w.scales must be"),
        (dict(w=mb.Int8Tensor(w.codes.float(), w.scales)), "2D int8"),
        (dict(x=mb.Int8Tensor(w.codes, w.scales.half())), "x.scales must be"),
    ]
    for change, msg in cases:
        a = dict(dict(x=x, w=w), **change)
        with pytest.raises(RuntimeError, match=msg):
            mb.int8_matmul(**a)


def test_product_on_a_stream_and_in_a_graph():
    xs = [_x(m, 512, torch.float16, seed=m).cuda() for m in (3, 90)]
    w = mb.quantize_int8(_x(700, 512, torch.float32, seed=8, spread=False).cuda())
    want = [mb.int8_matmul(x, w) for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [mb.int8_matmul(x, w) for x in xs]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    held = [x.clone() for x in xs]
    for x in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = mb.int8_matmul(x, w)
        graphs.append((g, y))
    for rounds in range(3):
        for x, h in zip(xs, held):
            h.copy_(x if rounds != 1 else -x)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, y), t in zip(graphs, want):
            assert torch.equal(y, t if rounds != 1 else -t)


def test_two_products_at_once():
    """Two streams, each with its own product, over and over."""
    w = mb.quantize_int8(_x(512, 2048, torch.float32, seed=8, spread=False).cuda())
    xs = [_x(m, 2048, torch.bfloat16, seed=m).cuda() for m in (8, 200)]
    want = [mb.int8_matmul(x, w) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(mb.int8_matmul(xs[i], w))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_clusters_of_two_streams_at_once():
    """Products on pairs of CTAs, which take all of an SM's TMEM, and small ones
    split over clusters, side by side and starting together."""
    wide = mb.quantize_int8(_x(2100, 300, torch.float32, seed=8, spread=False).cuda() * 0.02)
    small = [mb.quantize_int8(_x(4096, 1024, torch.float32, seed=i, spread=False).cuda() * 0.02)
             for i in range(2)]
    many = _x(2300, 300, torch.bfloat16, seed=1).cuda()
    few = [_x(m, 1024, torch.bfloat16, seed=m).cuda() for m in (1, 40)]
    want = mb.int8_matmul(many, wide), [mb.int8_matmul(x, w) for x, w in zip(few, small)]
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        got, go = [], torch.cuda.Event()
        torch.cuda._sleep(200000)  # the three start when this ends
        go.record()
        for s in streams:
            s.wait_event(go)
        for _ in range(4):
            with torch.cuda.stream(streams[0]):
                got.append((mb.int8_matmul(many, wide), want[0]))
            for s, x, w, y in zip(streams[1:], few, small, want[1]):
                with torch.cuda.stream(s):
                    got.append((mb.int8_matmul(x, w), y))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in got)


def test_int8_linear_from_a_quantized_weight():
    """Int8Linear of a 2/4-bit weight: the product of its dequantised matrix
    held in 8 bits."""
    g = torch.Generator().manual_seed(3)
    W = (torch.randn((96, 256), generator=g) * 0.02).half().cuda()
    qt = mb.quantize(W, ratio_4bit=0.25,
                     hessian_diag=torch.rand(256, generator=g).add(0.1).cuda())
    lin = gptq.Int8Linear.from_quantized(qt)
    x = torch.randn((2, 5, 256), generator=g).half().cuda()
    y = lin(x)
    w8 = mb.quantize_int8(mb.dequantize(qt))
    assert torch.equal(y, mb.int8_matmul(x, w8))
    _check_product(y.view(10, 96), mb.quantize_int8(x), w8)


class _Subclass(torch.Tensor):
    pass


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_every_way_into_a_call_agrees(dtype):
    """Parameters, subclasses, transposed and strided tensors, leading dimensions,
    a stride of one row, given outputs: the same codes and products."""
    g = torch.Generator().manual_seed(11)
    x = torch.randn((6, 80), generator=g).to(dtype).cuda()
    w = mb.quantize_int8(torch.randn((24, 80), generator=g).cuda())
    bias = torch.randn(24, generator=g).cuda()
    a = mb.quantize_int8(x)
    want = mb.int8_matmul(x, w, bias)
    assert want.dtype == dtype
    wide = torch.zeros((6, 100), dtype=dtype, device="cuda")
    wide[:, :80] = x
    for same in (torch.nn.Parameter(x), x.as_subclass(_Subclass), x.t().contiguous().t(),
                 wide[:, :80], x.view(2, 3, 80), x.view(1, 6, 1, 80), wide.double()[:, :80].to(dtype)):
        b = mb.quantize_int8(same)
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
        y = mb.int8_matmul(same, w, bias)
        assert y.shape == same.shape[:-1] + (24,) and not y.requires_grad
        assert torch.equal(y.reshape(6, 24), want)
        assert torch.equal(mb.int8_matmul(same, w, torch.stack([bias, bias], 1)[:, 0]).reshape(6, 24),
                           want)
        out = torch.empty_like(want).view(y.shape)
        assert mb.int8_matmul(same, w, bias, out=out) is out and torch.equal(out, y)
    for to in (torch.float16, torch.bfloat16, torch.float32):
        out = torch.empty((6, 80), dtype=to, device="cuda")
        assert torch.equal(mb.dequantize_int8(a, to), mb.dequantize_int8(a, to, out=out))
        y = mb.int8_matmul(a, w, bias, out_dtype=to)
        assert y.dtype == to and torch.equal(y, mb.int8_matmul(x, w, bias, out_dtype=to))
    assert mb.int8_matmul(a, w).dtype == torch.float16
    # the rows of another scales' tensor, and one row of many
    spread = torch.stack([a.scales, a.scales], 1)[:, 0]
    assert torch.equal(mb.dequantize_int8(mb.Int8Tensor(a.codes, spread)), mb.dequantize_int8(a))
    one = mb.quantize_int8(x[2:3])
    assert torch.equal(one.codes[0], a.codes[2]) and torch.equal(one.scales, a.scales[2:3])
    assert torch.equal(mb.int8_matmul(x[2:3], w, bias), want[2:3])


def test_allocation_failures_are_torch_errors():
    w = mb.quantize_int8(torch.zeros((1 << 20, 16), device="cuda"))
    x = torch.zeros((1 << 22, 16), dtype=torch.float16, device="cuda")
    with pytest.raises(torch.OutOfMemoryError):  # 8 TB of outputs
        mb.int8_matmul(x, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("M,N", [(1, 200), (40, 300), (300, 1000), (2300, 2100)])
def test_product_of_very_large_and_very_small_tokens(M, N, dtype):
    """Tokens next to the ends of fp32 whose products are of ordinary size: the
    sum times the token's scale alone would be infinite, or subnormal."""
    g = torch.Generator().manual_seed(M)
    x = torch.randn((M, 4096), generator=g)
    big = torch.arange(M) % 3
    x = x * torch.tensor([4e37, 1.0, 1e-40])[big].unsqueeze(1)  # the third: subnormal scales
    x = x.clamp(-3e38, 3e38).to(dtype).cuda()
    for size in (1e-3, 1e-30, 1e30):
        w = mb.quantize_int8(torch.randn((N, 4096), generator=g).cuda() * size)
        y = mb.int8_matmul(x, w)
        a = mb.quantize_int8(x)
        with np.errstate(over="ignore"):
            want, mag = serving.matmul(a.codes.cpu().numpy(), a.scales.cpu().numpy(),
                                       w.codes.cpu().numpy(), w.scales.cpu().numpy())
        f = torch.finfo(dtype)
        u = 2.0 ** -24
        work = mag * ((1 + u) ** 3 - 1) + 2.0 ** -149
        tol = work + (f.eps / 2) * (np.abs(want) + work) + f.tiny * f.eps / 2
        got = _np(y)
        fits = np.abs(want) + tol <= f.max
        assert np.all(np.abs(got - want)[fits] <= tol[fits])
        beyond = np.abs(want) - tol > f.max * (1 + f.eps / 2)
        assert np.all(np.isinf(got[beyond])) and not np.isnan(got).any()
        for rest in ([1], [0, 1], [1, 2]):  # a token's results are its own
            some = [i for i in range(M) if i % 3 in rest]
            assert torch.equal(mb.int8_matmul(x[some], w), y[some])
