"""The sums of the 8-bit float linear layer (lmx_linear_f8) against 64 bits, as tightly as
fp32 sums allow.

Tolerance of an output: half a step of its type there, and with A = sum of |products| with
their scales 2^-24 A for each product of a block, each block, and four more (scales, bias).
Norm of the error in fp16: fp32 sums are off by d <= 2e-6 of the norm (the bound of the
fp32 results); an output is rounded otherwise where it lies within d of a border, which
adds 2 d^2 to a squared error of u^2 / 12 at a step u >= 2^-11: a share of 24 (2e-6 2^11)^2 =
4e-4 of it, 2e-4 of the norm."""
import pytest
import torch

import lutmac_amd as L
from test_gpu_f8 import check, make, rounded

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# one for each way a call goes: a launch of its own for few rows, k among waves (16 and 32
# weight rows a workgroup, k in parts), tiles of 64 (k in parts and not) and of 128
WAYS = [(300, 2048, 1), (333, 1000, 3), (300, 8960, 16), (300, 400, 9), (5000, 600, 48), (300, 8960, 100), (700, 300, 300), (2100, 200, 2049)]


def half_step(want, dtype):
    """Half the distance of dtype's numbers at want."""
    tiny = torch.finfo(dtype).smallest_normal
    e = torch.frexp(want.abs().clamp_min(tiny))[1] - 1
    return torch.ldexp(torch.full_like(want, torch.finfo(dtype).eps / 2), e)


def tight(x, w, scale, bias, y):
    rows, cols = w.shape
    ws = scale.double().repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
    wd, xd = w.float().double() * ws, rounded(x)
    want = xd @ wd.T + (0.0 if bias is None else bias.double())
    size = xd.abs() @ wd.abs().T + (0.0 if bias is None else bias.double().abs())
    off = (y.double() - want).abs()
    most = half_step(want, x.dtype) + (128 + scale.shape[1] + 4) * 2.0 ** -24 * size
    fits = want.abs() + most < torch.finfo(x.dtype).max
    assert (off - most)[fits].max() <= 0
    if x.dtype == torch.float16 and want.numel() > 10000:
        least = (want.to(x.dtype).double() - want)[fits].norm()
        assert off[fits].norm() <= 1.0002 * least


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols,batch", WAYS)
def test_small_products_beside_large_ones(cuda, dtype, rows, cols, batch):
    """Of every eight products one is large and seven lie just below 2^-13 of it: together
    8e-4 of the sum, whatever the border between two results that it lies next to."""
    k = torch.arange(cols, device="cuda")
    x = torch.where(k % 8 == (k // 8 + torch.arange(batch, device="cuda")[:, None]) % 8, 256.0, 15.0 / 512).to(dtype)
    w = torch.ones(rows, -(-cols // 16) * 16, device="cuda").to(torch.float8_e4m3fn)[:, :cols]
    scale = torch.full((-(-rows // 128), -(-cols // 128)), 2.0 ** -8, device="cuda")
    bias = (torch.arange(rows, device="cuda") / rows).to(dtype)
    y = L.linear_f8(x, w, scale, bias=bias)
    want = rounded(x).sum(1, keepdim=True) / 256 + bias.double()
    most = half_step(want, dtype) + (scale.shape[1] + 4) * 2.0 ** -24 * want
    assert ((y.double() - want).abs() - most).max() <= 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols,batch", WAYS)
def test_general_values(cuda, dtype, rows, cols, batch):
    a = make(rows, cols, batch, dtype, 31, bias=batch % 2 == 0)
    tight(*a, L.linear_f8(*a[:3], bias=a[3]))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols,batch", [(4099, 1400, 3100), (8191, 260, 1700), (2563, 1100, 1029)])
def test_large_odd_sizes(cuda, dtype, rows, cols, batch):
    """Largest tiles with odd rows, a last block that is not whole and several steps of k."""
    a = make(rows, cols, batch, dtype, 32)
    tight(*a, L.linear_f8(*a[:3], bias=a[3]))


def test_slices_past_32_bits(cuda):
    """Rows of 2.3e9 outputs against 64 bits."""
    x, w, scale, bias = make(70000, 100, 32768, torch.bfloat16, 33)
    y = L.linear_f8(x, w, scale, bias=bias)
    for rows in (slice(0, 64), slice(30650, 30714), slice(32704, 32768)):
        tight(x[rows], w, scale, bias, y[rows])
        check(x[rows], w, scale, bias, y[rows])
