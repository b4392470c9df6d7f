"""The linear layer in 8-bit integers on the GPU (lmx_linear_i8) against 64 bits."""
import numpy as np
import pytest
import torch

import lutmac_amd as L
from lutmac_amd import synth

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def reference(x, w, scale, bias):
    """(y, most) in 64 bits: the sum of products is exact, its conversion to fp32, the
    two scales' products and the bias' sum (and amax / 127) round once each, then
    the result to its type."""
    xd = x.double().cpu()
    top = xd.abs().amax(1, keepdim=True)
    codes = torch.where(top > 0, (xd * 127 / top).round(), torch.zeros(()).double())
    p = codes @ w.double().cpu().T * (top / 127) * scale.double().cpu()
    y = p if bias is None else p + bias.double().cpu()
    most = 6 * 2.0 ** -24 * (p.abs() + y.abs()) + y.abs() * HALF_STEP[x.dtype] + (2.0 ** -24 if x.dtype == torch.float16 else 1e-40)
    return y, most


def make(rows, cols, batch, dtype, seed, width=None, bias=True):
    g = torch.Generator().manual_seed(seed)
    width = width or -(-cols // 16) * 16
    w = torch.randint(-128, 128, (rows, width), generator=g, dtype=torch.int8).cuda()[:, :cols]
    x = torch.randn(batch, cols, generator=g)
    x[:, :: max(1, cols // 3)] *= 15
    scale = (0.001 * (0.5 + torch.rand(rows, generator=g))).cuda()
    b = torch.randn(rows, generator=g).to(dtype).cuda() if bias else None
    return x.to(dtype).cuda(), w, scale, b


def check(x, w, scale, bias, y):
    want, most = reference(x, w, scale, bias)
    got, top = y.double().cpu().view_as(want), torch.finfo(x.dtype).max
    # a result past the type's largest value rounds to infinity, its sum in fp32 perhaps just before it
    past = want.abs() - most > top
    assert torch.equal(got[past], want[past].sign() * float("inf"))
    got, want, most = got[~past], want[~past], most[~past]
    sure = want.abs() + most < top
    over = ((got - want).abs() - most)[sure]
    assert over.max() <= 0, f"off by {over.max().item()} more than the bound"


@pytest.mark.parametrize("dtype", sorted(HALF_STEP, key=str))
@pytest.mark.parametrize("rows,cols", [(1, 1), (16, 128), (33, 100), (300, 2048), (259, 1400), (1030, 8960)])
@pytest.mark.parametrize("batch", [1, 3, 16, 17, 48, 64, 65, 200, 300])
def test_linear_i8(cuda, dtype, rows, cols, batch):
    a = make(rows, cols, batch, dtype, rows + cols + batch, bias=batch % 2 == 1)
    check(*a, L.linear_i8(a[0], a[1], a[2], bias=a[3]))


# workgroups of 16, 32 and 64 weight rows, the last one in part; tiles of just one round of the CUs
@pytest.mark.parametrize("rows,cols", [(4101, 700), (7001, 2048), (14000, 128), (20003, 300), (33000, 256)])
@pytest.mark.parametrize("batch", [2, 4, 20, 37, 64])
def test_linear_i8_many_weight_rows(cuda, rows, cols, batch):
    a = make(rows, cols, batch, torch.bfloat16, rows + batch)
    check(*a, L.linear_i8(a[0], a[1], a[2], bias=a[3]))


@pytest.mark.parametrize("rows,cols,batch", [(4096, 512, 4100), (4100, 260, 4097), (8190, 1400, 2200), (16384, 128, 1100)])
def test_linear_i8_large(cuda, rows, cols, batch):
    a = make(rows, cols, batch, torch.bfloat16, 7)
    check(*a, L.linear_i8(a[0], a[1], a[2], bias=a[3]))


@pytest.mark.parametrize("rows,cols,batch", [(70, 131072, 2), (64, 20000, 70)])
def test_linear_i8_long(cuda, rows, cols, batch):
    """Rows longer than a workgroup keeps in registers, up to the longest: the sum of
    the largest codes still fits 32 bits."""
    a = make(rows, cols, batch, torch.float32, 8)
    check(*a, L.linear_i8(a[0], a[1], a[2], bias=a[3]))
    x, w, scale, b = a
    x.fill_(2.0)
    w.fill_(-128)
    check(x, w, scale, b, L.linear_i8(x, w, scale, bias=b))


def test_linear_i8_borders(cuda):
    """Codes exactly between two whole numbers go to the even one, whatever the
    largest value: x = amax (2 n + 1) / 254."""
    for top in (127.0, 254.0 * 3, 127 * 9.0, 1.0):
        x = torch.tensor([[top] + [top * (2 * n + 1) / 254 for n in range(127)]], dtype=torch.float64)
        x = torch.cat([x, -x]).float().cuda()
        w = torch.eye(128, dtype=torch.int8).cuda()
        scale = torch.ones(128).cuda()
        check(x, w, scale, None, L.linear_i8(x, w, scale))


def test_linear_i8_special_rows(cuda):
    """A row with a value that is not finite gives NaN, rows of zeros the bias, tiny
    and huge rows their products; the others are untouched by it."""
    for batch in (5, 100):
        x, w, scale, b = make(70, 300, batch, torch.float32, 9)
        x[0, 3], x[1, 299], x[2], x[3], x[4] = float("nan"), -float("inf"), 0.0, x[3] * 1e-38, x[4] * 1e36
        y = L.linear_i8(x, w, scale, bias=b)
        assert torch.isnan(y[:2]).all() and torch.isfinite(y[2:4]).all()
        assert torch.equal(y[2], b)
        check(x[5:] if batch > 5 else x[4:], w, scale, b, y[5:] if batch > 5 else y[4:])


def test_linear_i8_views(cuda):
    """Rows of weights far apart, x, y and bias at odd elements, leading dimensions."""
    for batch in (2, 90):
        x, w, scale, b = make(101, 77, batch, torch.float16, 10, width=208)
        keep = w.clone()
        xo, bo = torch.empty(batch * 77 + 1, dtype=x.dtype, device="cuda")[1:].view(batch, 77), torch.empty(102, dtype=x.dtype, device="cuda")[1:]
        xo.copy_(x), bo.copy_(b)
        buf = torch.full((batch * 101 + 3,), 5.0, dtype=x.dtype, device="cuda")
        y = buf[1:-2].view(batch, 101)
        L.linear_i8(xo, w, scale, bias=bo, y=y)
        check(x, w, scale, b, y)
        assert (buf[0] == 5) and (buf[-2:] == 5).all() and torch.equal(w, keep)
        assert torch.equal(L.linear_i8(xo.view(1, batch, 77), w, scale, bias=bo)[0], y)


def test_linear_i8_graph_and_stream(cuda):
    for batch in (3, 40, 130):
        x, w, scale, b = make(200, 500, batch, torch.bfloat16, 11)
        y = torch.empty(batch, 200, dtype=x.dtype, device="cuda")
        work = torch.empty(L.linear_i8_workspace(200, 500, batch), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            L.linear_i8(x, w, scale, bias=b, y=y, workspace=work)
        for step in range(4):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(step)).cuda())
            graph.replay()
            eager = L.linear_i8(x, w, scale, bias=b)
            torch.cuda.synchronize()
            assert torch.equal(y, eager)
            check(x, w, scale, b, y)
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            z = L.linear_i8(x, w, scale, bias=b)
        other.synchronize()
        assert torch.equal(z, y)


@pytest.mark.parametrize("rows,cols", [(70, 256), (300, 1400)])
def test_linear_i8_of_a_handle(cuda, rows, cols):
    """The codes of an 8-bit weight handle with one scale per row, and their product
    beside the handle's own (fp32 activations): they differ by the codes' half
    steps."""
    planes, scales, _ = L.quantize(L.FMT_INT8, L.synth_normal(3, 0, rows, cols, 0.02), cols)   # one group a row
    w = L.Weight.from_planes(L.FMT_INT8, planes, scales, rows, cols, 0)
    codes, sc = w.codes_i8()
    bits = np.unpackbits(planes.reshape(8, rows, -1), axis=-1)[:, :, :cols]
    want = sum(bits[p].astype(np.uint8) << p for p in range(8)).astype(np.uint8).view(np.int8)
    np.testing.assert_array_equal(codes.cpu().numpy(), want)
    np.testing.assert_array_equal(sc.cpu().numpy(), scales.reshape(-1)[:rows])
    x = torch.randn(4, cols, generator=torch.Generator().manual_seed(1)).cuda()
    y, full = L.linear_i8(x, codes, sc), w.gemv(x).view(4, rows)
    check(x, codes, sc, None, y)
    half = x.abs().amax(1, keepdim=True) / 254
    most = half * codes.float().abs().sum(1) * sc
    assert ((y - full).abs() <= most + 1e-4 * full.abs().max()).all()
    grouped, s2, g2 = synth.make_weights(L.FMT_INT8, rows, 512, seed=3, group=128)
    with pytest.raises(L.LmxError):
        L.Weight.from_planes(L.FMT_INT8, grouped, s2, rows, 512, g2).codes_i8()
