"""The linear layer in 8-bit floating point on the GPU (lmx_linear_f8) against 64 bits.

Tolerances, from A = sum of |products| with their scales: fp32 sums round at most
once a product, a block and a scale, 2^-24 each of at most A.  In the 16-bit types a
product may lose 2^-13 of the largest of its instruction, so at most 128 * 2^-13 of
a block's largest |x| times |w|; where all products of a block are whole multiples of 2^-12 of
the largest they lose nothing.  The result is rounded to its type, half a step."""
import pytest
import torch

import lutmac_amd as L

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = sorted(HALF_STEP, key=str)


def blocks(t):   # [rows, cols] -> [rows, blocks, 128]
    return torch.nn.functional.pad(t, (0, -t.shape[1] % 128)).view(t.shape[0], -1, 128)


def power(e):   # 2^e, exactly
    return ((e + 1023) << 52).view(torch.float64)


def rounded(x):
    """x as the codes and their powers of two hold it, in 64 bits."""
    b = blocks(x.double())
    top = b.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -126, dtype=torch.int64)
    for n in range(-126, 121):
        e += (top > 448.0 * 2.0 ** n).long()
    v = b / power(e)
    # e4m3: 3 bits behind the first, down to 2^-9
    step = power((v.abs().clamp_min(2.0 ** -6).view(torch.int64) >> 52) - 1023 - 3)
    return ((v / step).round() * step * power(e)).view(x.shape[0], -1)[:, :x.shape[1]]


def make(rows, cols, batch, dtype, seed, bias=True, narrow=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = -(-cols // 16) * 16

    def normal(*s):
        return torch.randn(*s, generator=g, device="cuda")
    if narrow:   # magnitudes 0.5 .. 4 of 4 bits: products lose nothing
        def some(*s):
            t = (8 + torch.randint(0, 8, s, generator=g, device="cuda")) * 2.0 ** torch.randint(-4, -1, s, generator=g, device="cuda")
            return t * (1 - 2 * torch.randint(0, 2, s, generator=g, device="cuda"))
        x, w = some(batch, cols), some(rows, width)
    else:
        x, w = normal(batch, cols), normal(rows, width) * 100
        x[:, :: max(1, cols // 3)] *= 15
    w = w.clamp(-448, 448).to(torch.float8_e4m3fn)
    # what lies behind the columns is not read as numbers
    w.view(torch.uint8)[:, cols:] = 0x7F
    scale = 0.001 * (0.5 + torch.rand(-(-rows // 128), -(-cols // 128), generator=g, device="cuda"))
    return x.to(dtype), w[:, :cols], scale, normal(rows).to(dtype) if bias else None


def check(x, w, scale, bias, y, narrow=False):
    rows, cols = w.shape
    steps = scale.shape[1]
    ws = scale.double().repeat_interleave(128, 0)[:rows]
    wd = w.float().double() * ws.repeat_interleave(128, 1)[:, :cols]
    xd = rounded(x)
    want = xd @ wd.T
    most = (xd.abs() @ wd.abs().T) * ((128 + steps + 4) * 2.0 ** -24)
    if x.dtype != torch.float32 and not narrow:
        most += 2.0 ** -6 * (blocks(xd).abs().amax(-1) @ blocks(wd).abs().amax(-1).T)
    if bias is not None:
        want = want + bias.double()
        most = most + want.abs() * 2.0 ** -24
    most = most + want.abs() * HALF_STEP[x.dtype] + (2.0 ** -24 if x.dtype == torch.float16 else 1e-40)
    got = y.double().view_as(want)
    fits = want.abs() + most < torch.finfo(x.dtype).max
    over = ((got - want).abs() - most)[fits]
    assert over.max() <= 0, f"off by {over.max().item()} more than the bound"
    norm = (got - want)[fits].norm() / want[fits].norm()
    assert norm < HALF_STEP[x.dtype] + (1e-3 if x.dtype != torch.float32 else 2e-6), norm


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols", [(1, 1), (16, 128), (33, 100), (300, 2048), (259, 1400), (1030, 8960)])
@pytest.mark.parametrize("batch", [1, 2, 3, 4, 5, 16, 17, 48, 64, 65, 200, 300])
def test_linear_f8(cuda, dtype, rows, cols, batch):
    narrow = batch % 2 == 0
    a = make(rows, cols, batch, dtype, rows + cols + batch, bias=batch % 3 == 1, narrow=narrow)
    check(*a, L.linear_f8(a[0], a[1], a[2], bias=a[3]), narrow)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols,batch", [(4096, 512, 4100), (4100, 260, 2049), (8190, 1400, 1100), (16384, 128, 1100),
                                             (16500, 300, 1), (20003, 300, 4), (33000, 256, 37), (7001, 2048, 64)])
def test_linear_f8_large(cuda, dtype, rows, cols, batch):
    a = make(rows, cols, batch, dtype, 7, narrow=True)
    check(*a, L.linear_f8(a[0], a[1], a[2], bias=a[3]), True)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols,batch", [(70, 131072, 2), (64, 20000, 70), (16, 131071, 1), (130, 60001, 20),
                                             (1000, 8300, 33), (17, 30001, 64), (300, 5000, 9)])
def test_linear_f8_long(cuda, dtype, rows, cols, batch):
    a = make(rows, cols, batch, dtype, 8)
    check(*a, L.linear_f8(a[0], a[1], a[2], bias=a[3]))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("batch", [1, 5, 70])
def test_activation_codes(cuda, dtype, batch):
    """Values between two codes go to the nearer, of two equally near to the even one;
    blocks whose largest is just at, above and below 448 of a power of two; with a
    unit weight each code comes out alone."""
    code = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float().double()
    mid = (code[1:] + code[:-1]) / 2
    x = torch.cat([mid, torch.tensor([448.0, 0.0], dtype=torch.float64)])
    x = torch.stack([x, -x, x * 2.0 ** -20 if dtype != torch.float16 else x / 4, x.clamp(max=447.0), x.clamp(max=224.0)])
    x = x.to(dtype)[torch.arange(batch) % 5].cuda()
    w = torch.eye(128).to(torch.float8_e4m3fn).cuda()
    y = L.linear_f8(x, w, torch.ones(1, 1).cuda())
    assert torch.equal(y.double(), rounded(x).to(dtype).double())


@pytest.mark.parametrize("batch", [1, 3, 40, 100])
def test_extreme_values(cuda, batch):
    """The smallest and largest powers of two, zeros, and values that are not finite,
    which reach their own row only."""
    for value in (1e-45, 2.0 ** -130, 2.0 ** -120, 1e30, 3e38):
        x = torch.full((batch, 256), value).cuda()
        x[:, 128:] = 0
        w = torch.full((20, 256), 2.0 ** -6).to(torch.float8_e4m3fn).cuda()
        y = L.linear_f8(x, w, torch.ones(1, 2).cuda())
        want = (rounded(x) @ w.float().double().T).float()
        assert torch.allclose(y.double(), want.double(), rtol=1e-6, atol=0.0), value
    for dtype in TYPES:
        for value in (float("inf"), float("-inf"), float("nan")):
            x = torch.randn(batch, 300).to(dtype).cuda()
            clean = x.clone()
            x[batch // 2, 7] = value
            w, scale = L.blocks_f8(torch.randn(40, 300).cuda())
            y, z = L.linear_f8(x, w, scale), L.linear_f8(clean, w, scale)
            assert y[batch // 2].isnan().all()
            keep = torch.arange(batch) != batch // 2
            assert torch.equal(y[keep], z[keep])


@pytest.mark.parametrize("batch", [1, 30, 300])
def test_weight_nan(cuda, batch):
    """A weight that is NaN makes NaN of its output alone."""
    w, scale = L.blocks_f8(torch.randn(200, 500).cuda())
    w.view(torch.uint8)[77, 300] = 0x7F
    y = L.linear_f8(torch.randn(batch, 500).cuda(), w, scale)
    bad = torch.zeros(200, dtype=torch.bool)
    bad[77] = True
    assert torch.equal(y.isnan().cpu(), bad.expand(batch, -1))


def test_strides_shapes_and_outputs(cuda):
    x, w, scale, bias = make(50, 200, 6, torch.float16, 3)
    want = L.linear_f8(x, w, scale, bias=bias)
    wide = torch.empty(50, 1024, dtype=torch.uint8, device="cuda").fill_(0x7F)
    wide[:, 16:216] = w.view(torch.uint8)
    assert torch.equal(L.linear_f8(x, wide.view(torch.float8_e4m3fn)[:, 16:216], scale, bias=bias), want)
    assert torch.equal(L.linear_f8(x.view(2, 3, 200), w, scale, bias=bias), want.view(2, 3, 50))
    odd = torch.empty(6 * 200 + 1, dtype=torch.float16, device="cuda")[1:].view(6, 200).copy_(x)
    out = torch.full((6 * 50 + 2,), 7.0, dtype=torch.float16, device="cuda")
    y = out[1:-1].view(6, 50)
    assert L.linear_f8(odd, w, scale, bias=bias, y=y) is y
    assert torch.equal(y, want) and out[0] == 7.0 and out[-1] == 7.0
    n = L.linear_f8_workspace(50, 200, 6, torch.float16)
    work = torch.full((n + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    assert torch.equal(L.linear_f8(x, w, scale, bias=bias, workspace=work), want)
    assert (work[n:] == 0xFF).all()
    for bad in (work[: n - 1], work[4: n + 4]):
        with pytest.raises(L.LmxError):
            L.linear_f8(x, w, scale, workspace=bad)
    assert L.linear_f8(x[:0], w, scale).shape == (0, 50)
    # weights that start at no multiple of 16 bytes
    with pytest.raises(L.LmxError):
        L.linear_f8(x, wide.view(torch.float8_e4m3fn)[:, 8:208], scale)


@pytest.mark.parametrize("batch", [1, 4, 40, 300])
def test_replays_and_streams(cuda, batch):
    """A captured call follows its inputs at every replay; calls on another stream are
    the same."""
    x, w, scale, bias = make(600, 1000, batch, torch.bfloat16, 5)
    stream, graph, y = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.empty(batch, 600, dtype=torch.bfloat16, device="cuda")
    work = torch.empty(L.linear_f8_workspace(600, 1000, batch, torch.bfloat16), dtype=torch.uint8, device="cuda")
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        L.linear_f8(x, w, scale, bias=bias, y=y, workspace=work)
    for i in range(4):
        x.copy_(torch.randn(batch, 1000) * 3 ** i)
        work.fill_(0xFF)
        graph.replay()
        want = L.linear_f8(x, w, scale, bias=bias)
        torch.cuda.synchronize()
        assert torch.equal(y, want), i
    other = L.linear_f8(x, w, scale, bias=bias, stream=stream)
    stream.synchronize()
    assert torch.equal(other, want)


def test_blocks_f8(cuda):
    w = torch.randn(300, 200).cuda() * torch.exp(torch.randn(300, 1).cuda())
    w[128:256, 128:] = 0
    codes, scale = L.blocks_f8(w)
    back = codes.float() * scale.repeat_interleave(128, 0)[:300].repeat_interleave(128, 1)[:, :200]
    # half a step of e4m3, below 2^-6 of the code half of 2^-9; and the quotient's rounding
    assert ((back - w).abs() <= w.abs() * (2.0 ** -4 + 1e-6) + scale.max() * 2.0 ** -10).all()
    assert codes.stride(0) % 16 == 0 and scale[1, 1] == 1.0
