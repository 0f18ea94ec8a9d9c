"""mxfp4.quantize / dequantize / matmul on the GPU against the 64-bit references of tests/_operators.py."""
import numpy as np
import pytest
import torch

from tests import _operators as O

pytestmark = pytest.mark.gpu

BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def _check_quantize(x):
    from speech_to_text_amd import mxfp4
    codes, scales = O.quantize_reference(x.double().cpu().numpy())
    t = mxfp4.quantize(x)
    got_s, got_c = t.scales.cpu().numpy(), O.unpack(t.codes.cpu().numpy())
    assert np.array_equal(got_s, scales)
    fine = np.repeat(scales != 255, 32, axis=1)
    assert np.array_equal(got_c[fine], codes[fine])
    want = O.values_of(codes, scales)
    for dt in (FF, BF):
        assert np.array_equal(t.dequantize(dt).double().cpu().numpy(), want, equal_nan=True)


@pytest.mark.parametrize("dtype", [FF, BF, HF])
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 64), (9, 1280), (7, 96), (300, 160), (33, 5120), (2049, 32)])
def test_quantize_shapes_and_types(dtype, rows, k):
    g = torch.Generator().manual_seed(rows + k)
    x = torch.randn(rows, k, generator=g) * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g).float())
    _check_quantize(x.to(dtype).cuda())


@pytest.mark.parametrize("dtype", [FF, BF, HF])
def test_quantize_ties_zeros_and_extremes(dtype):
    """Every tie of the grid under several scales (the block's maximum fixes the scale), signed zeros, values just
    beside the ties, the smallest and largest magnitudes of the type, infinities and NaN."""
    info = torch.finfo(dtype)
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.0, -0.0, 6.0, 7.0, 7.75, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0]
    base = torch.tensor(ties + [-t for t in ties[:7]] + [4.0] * 7)
    blocks = [base * 2.0 ** e for e in ((-10, -3, 0, 5, 12) if dtype == HF else (-120, -60, 0, 31, 125))]
    for near in (1 + info.eps, 1 - info.eps):
        b = base.clone()
        b[:7] *= near
        blocks.append(b)
    tiny = torch.zeros(32)
    tiny[0] = info.smallest_normal * info.eps                      # the type's smallest subnormal
    tiny[1], tiny[2] = -info.smallest_normal, info.smallest_normal * 1.5
    only_sub = torch.zeros(32)
    only_sub[3], only_sub[4] = info.smallest_normal * info.eps, -info.smallest_normal / 2
    top = torch.full((32,), info.max)
    top[1], top[2], top[3] = -info.max, info.max / 3, info.tiny
    nan, inf, both = torch.ones(32), torch.ones(32), torch.zeros(32)
    nan[31], inf[0], both[5], both[6] = float("nan"), -float("inf"), float("inf"), float("nan")
    blocks += [tiny, only_sub, top, nan, inf, both, torch.zeros(32), torch.full((32,), -0.0)]
    _check_quantize(torch.stack(blocks).to(dtype).view(-1, 32).cuda())
    _check_quantize(torch.cat(blocks[:-1] if len(blocks) % 2 else blocks).to(dtype).view(-1, 64).cuda())


def test_quantize_strided_rows_and_empty():
    from speech_to_text_amd import mxfp4
    g = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn(21, 640, generator=g, device="cuda")
    _check_quantize(wide[:, 64:256])
    _check_quantize(wide.to(BF)[::3, 8:40])
    assert mxfp4.quantize(wide[:0]).codes.shape == (0, 320)
    assert mxfp4.quantize(wide[:, :0]).scales.shape == (21, 0)
    assert mxfp4.quantize(wide[:0]).dequantize().shape == (0, 640)


def _weight(n, k, seed):
    from speech_to_text_amd import mxfp4
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 256, (n, k // 2), dtype=np.uint8)
    scales = rng.integers(117, 123, (n, k // 32), dtype=np.uint8)
    w = torch.from_numpy(O.values_of(O.unpack(codes), scales))
    return mxfp4.Mxfp4Weight(mxfp4.Mxfp4Tensor(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda())), w


def _check_product(m, n, k, x4=False, bias=True, gelu=None, out_dtype=BF, seed=0):
    from speech_to_text_amd import mxfp4
    g = torch.Generator().manual_seed(seed)
    weight, w = _weight(n, k, seed)
    x = torch.randn(m, k, generator=g).to(BF)
    b = torch.randn(n, generator=g) if bias else None
    if x4:
        xq = mxfp4.quantize(x.cuda())
        xd = torch.from_numpy(O.values_of(*O.quantize_reference(x.double().numpy())))
    else:
        xq, xd = x.cuda(), x.double()
    y = mxfp4.matmul(xq, weight, bias=b.cuda() if bias else None, gelu=gelu, out_dtype=out_dtype)
    assert y.dtype == out_dtype and y.shape == (m, n)
    want, bound = O.product_reference(xd.cuda(), w.cuda(), b.cuda() if bias else None, gelu, out_dtype)
    err = (y.double() - want).abs()
    assert (err <= bound).all(), "off by %g, %.2f of the bound" % (float(err.max()), float((err / bound).max()))


@pytest.mark.parametrize("x4", [False, True])
@pytest.mark.parametrize("m", [1, 2, 9, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 640])
def test_product_rows(m, x4):
    _check_product(m, 80, 320, x4=x4, seed=m)


@pytest.mark.parametrize("x4", [False, True])
@pytest.mark.parametrize("n", [1, 3, 15, 16, 17, 31, 33, 63, 65, 127, 129, 255, 257, 511])
def test_product_columns(n, x4):
    _check_product(5, n, 256, x4=x4, seed=n, out_dtype=FF)
    _check_product(130, n, 128, x4=x4, seed=n)


@pytest.mark.parametrize("x4", [False, True])
@pytest.mark.parametrize("k", [32, 64, 96, 128, 160, 224, 256, 480, 512, 544, 1280, 5120])
def test_product_depths(k, x4):
    for m in (1, 9, 150):
        _check_product(m, 48, k, x4=x4, seed=k + m, out_dtype=FF)


@pytest.mark.parametrize("x4", [False, True])
@pytest.mark.parametrize("gelu", [None, "tanh", "erf"])
@pytest.mark.parametrize("out_dtype", [BF, FF])
@pytest.mark.parametrize("bias", [False, True])
def test_product_epilogues(x4, gelu, out_dtype, bias):
    for m in (3, 70, 300):
        _check_product(m, 208, 192, x4=x4, gelu=gelu, out_dtype=out_dtype, bias=bias, seed=m)


@pytest.mark.parametrize("x4", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 5120, 1280), (9, 1280, 5120), (600, 1280, 1280), (1500, 640, 256), (2000, 1000, 96), (700, 5120, 160)])
def test_product_layer_sizes(m, n, k, x4):
    _check_product(m, n, k, x4=x4, seed=m + n)


@pytest.mark.parametrize("x4", [False, True])
@pytest.mark.parametrize("m,n,k,gelu,out_dtype", [(5001, 1310, 256, None, BF), (4100, 1283, 1280, "tanh", BF), (12300, 520, 128, None, FF),
                                                  (8193, 769, 384, "erf", FF), (6000, 1300, 160, None, BF)])
def test_product_many_rows(m, n, k, gelu, out_dtype, x4):
    _check_product(m, n, k, x4=x4, gelu=gelu, out_dtype=out_dtype, seed=m)


@pytest.mark.parametrize("x4", [False, True])
@pytest.mark.parametrize("k", [160, 192, 224, 288, 480, 1120])
def test_product_many_rows_any_depth(k, x4):
    _check_product(4099, 1300, k, x4=x4, seed=k, out_dtype=FF)


@pytest.mark.parametrize("k", [160, 224, 256])
def test_product_reads_nothing_behind_a_row(k):
    from speech_to_text_amd import mxfp4
    weight, _ = _weight(1300, k, 3)
    wide = torch.full((4099, k + 40), float("nan"), dtype=BF, device="cuda")
    wide[:, :k] = torch.randn(4099, k, generator=torch.Generator().manual_seed(k)).to(BF).cuda()
    x = wide[:, :k]
    a, b = mxfp4.matmul(x, weight), mxfp4.matmul(x.contiguous(), weight)
    assert torch.isfinite(a).all() and torch.equal(a, b)


@pytest.mark.parametrize("m", [7, 6000])
def test_product_of_a_slice_of_quantised_rows(m):
    """Rows taken out of a larger quantised matrix (scales that start at any byte)."""
    from speech_to_text_amd import mxfp4
    weight, w = _weight(1290, 128, 4)
    x = mxfp4.quantize(torch.randn(m + 3, 128, device="cuda").to(BF))
    for first in (1, 2, 3):
        part = mxfp4.Mxfp4Tensor(x.codes[first: first + m], x.scales[first: first + m])
        y = mxfp4.matmul(part, weight)
        want, bound = O.product_reference(part.dequantize().double(), w.cuda(), None, None, BF)
        assert ((y.double() - want).abs() <= bound).all()
    odd = torch.empty(x.scales.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(x.scales.shape)
    odd.copy_(x.scales)
    assert torch.equal(mxfp4.matmul(mxfp4.Mxfp4Tensor(x.codes, odd), weight), mxfp4.matmul(x, weight))


@pytest.mark.parametrize("x4", [False, True])
def test_product_accumulated_into_many_rows(x4):
    from speech_to_text_amd import mxfp4
    weight, w = _weight(1290, 128, 5)
    x = torch.randn(6000, 128, device="cuda").to(BF)
    xq = mxfp4.quantize(x) if x4 else x
    start = torch.randn(6000, 1290, device="cuda")
    out = start.clone()
    mxfp4.matmul(xq, weight, out=out, accumulate=True)
    want, bound = O.product_reference((xq.dequantize() if x4 else x).double(), w.cuda(), None, None, FF)
    assert ((out.double() - (want + start)).abs() <= bound + 2.0 ** -24 * (want + start).abs()).all()


@pytest.mark.parametrize("x4", [False, True])
@pytest.mark.parametrize("m", [4, 90, 400])
def test_product_into_given_rows_and_accumulated(m, x4):
    """`out` with a row stride, nothing written beside its columns; accumulate adds to what is there."""
    from speech_to_text_amd import mxfp4
    weight, w = _weight(70, 160, 3)
    x = torch.randn(m, 160, generator=torch.Generator().manual_seed(3)).to(BF)
    xq = mxfp4.quantize(x.cuda()) if x4 else x.cuda()
    xd = (xq.dequantize() if x4 else xq).double()
    b = torch.randn(70, device="cuda")
    want, bound = O.product_reference(xd, w.cuda(), b, None, FF)
    for pad in (70, 72, 75):
        buf = torch.full((m, pad + 9), 5.0, device="cuda")
        view = buf[:, 4: 74]
        assert mxfp4.matmul(xq, weight, bias=b, out=view) is view
        assert ((view.double() - want).abs() <= bound).all()
        mxfp4.matmul(xq, weight, bias=b, out=view, accumulate=True)
        assert ((view.double() - 2 * want).abs() <= 2 * bound + 2.0 ** -23 * want.abs()).all()
        assert (buf[:, :4] == 5).all() and (buf[:, 74:] == 5).all()
    half = torch.full((m, 91), 5.0, device="cuda", dtype=BF)
    mxfp4.matmul(xq, weight, out=half[:, 1: 71])
    assert (half[:, 0] == 5).all() and (half[:, 71:] == 5).all()
    want, bound = O.product_reference(xd, w.cuda(), None, None, BF)
    assert ((half[:, 1: 71].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("m", [1, 20, 200])
def test_product_nan_and_infinity_stay_in_their_row_and_column(m):
    from speech_to_text_amd import mxfp4
    rng = np.random.default_rng(5)
    n, k = 100, 224
    codes = rng.integers(0, 256, (n, k // 2), dtype=np.uint8)
    scales = rng.integers(117, 123, (n, k // 32), dtype=np.uint8)
    scales[40, 3] = 255
    w = mxfp4.Mxfp4Weight(mxfp4.Mxfp4Tensor(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()))
    x = torch.randn(m, k).to(BF)
    row = m // 2
    if m > 1:
        x[row, 7] = float("nan")
        x[m - 1, 9] = float("inf")
    y = mxfp4.matmul(x.cuda(), w).cpu()
    rows = torch.ones(m, dtype=torch.bool)
    if m > 1:
        rows[row] = rows[m - 1] = False
        assert torch.isnan(y[row]).all() and not torch.isfinite(y[m - 1]).any()
    cols = torch.ones(n, dtype=torch.bool)
    cols[40] = False
    assert torch.isnan(y[:, 40]).all()
    assert torch.isfinite(y[rows][:, cols]).all()
    xq = mxfp4.quantize(x.cuda())
    y = mxfp4.matmul(xq, w).cpu()
    assert torch.isnan(y[:, 40]).all() and torch.isfinite(y[rows][:, cols]).all()
    if m > 1:
        assert torch.isnan(y[row]).all() and torch.isnan(y[m - 1]).all()


def test_product_small_scales_are_exact():
    """Weights whose values are subnormal in bfloat16 still enter the product exactly."""
    from speech_to_text_amd import mxfp4
    for s in (0, 1, 3, 130, 200):
        codes = torch.randint(0, 256, (16, 16), dtype=torch.uint8, generator=torch.Generator().manual_seed(s))
        scales = torch.full((16, 1), s, dtype=torch.uint8)
        w = torch.from_numpy(O.values_of(O.unpack(codes.numpy()), scales.numpy()))
        x = torch.zeros(4, 32, dtype=BF)
        x[torch.arange(4), torch.tensor([0, 5, 17, 31])] = torch.tensor([1.0, -2.0, 0.5, 8.0]).to(BF)
        y = mxfp4.matmul(x.cuda(), mxfp4.Mxfp4Weight(mxfp4.Mxfp4Tensor(codes.cuda(), scales.cuda())), out_dtype=FF)
        assert torch.equal(y.double().cpu(), x.double() @ w.t()), s


def test_product_rows_are_independent_of_their_number():
    """A row's result does not depend on how many rows share the call, as far as one kernel serves them."""
    from speech_to_text_amd import mxfp4
    weight, _ = _weight(256, 512, 9)
    x = torch.randn(64, 512, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(BF)
    whole = mxfp4.matmul(x[:16], weight, out_dtype=FF)
    for m in (1, 2, 9, 15):
        assert torch.equal(mxfp4.matmul(x[:m], weight, out_dtype=FF), whole[:m])


def test_product_empty_batches_streams_and_graphs():
    from speech_to_text_amd import mxfp4
    weight, _ = _weight(96, 256, 11)
    x = torch.randn(40, 256, device="cuda").to(BF)
    assert mxfp4.matmul(x[:0], weight).shape == (0, 96)
    assert mxfp4.matmul(mxfp4.quantize(x[:0]), weight).shape == (0, 96)
    step = lambda: (mxfp4.matmul(x, weight, gelu="tanh"), mxfp4.matmul(mxfp4.quantize(x), weight, out_dtype=FF))
    eager = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        for t in out:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        assert all(torch.equal(a, b) for a, b in zip(step(), eager))
