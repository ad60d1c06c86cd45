"""The weight gradient on sizes that take its 256 x 256 tiles (those of the other
tests stay on 128 x 128 ones), and at the ends of the kept values' range.

Bars as for the small sizes: products are exact and sums FP32, so each element is
within (rows + 8) 2^-24 of the sum of its terms' magnitudes, plus one place of the
output type.  An FP32 cotangent's bits below BF16's smallest step, 2^-133, are in
none of its three parts: that much of each kept value's magnitude."""
import math

import pytest
import torch

from sandmuon_amd import act8

pytestmark = pytest.mark.gpu

PLACE = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


def make(device, rows, cols, dtype, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(rows, cols, device=device, generator=g)
    return (x * torch.exp(torch.randn(1, cols, device=device, generator=g))).to(dtype)


def check(delta, saved, out):
    """Against the values that the bytes read back as (compared with their definition elsewhere)."""
    dw, db = act8.linear_backward(delta, saved, out)
    d, k = delta.double(), act8.decode(saved, torch.float32).double()
    rows = d.shape[0]
    tiny = 2.0 ** -25 if out == torch.float16 else 0
    dropped = 2.0 ** -133 * k.abs().sum(0) if delta.dtype == torch.float32 else torch.zeros_like(k[0])
    for got, want, size, rest in ((dw, d.t().contiguous() @ k, d.abs().t().contiguous() @ k.abs(), dropped),
                                  (db, d.sum(0), d.abs().sum(0), 0)):
        assert got.dtype == out and got.shape == want.shape
        off = (got.double() - want).abs()
        assert (off <= (rows + 8) * 2.0 ** -24 * size + PLACE[out] * want.abs() + tiny + rest).all()


# 16 x 16 tiles with no split, 6 x 6 in 7 splits: odd edges in every direction
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,k,n", [(515, 4001, 4090), (4100, 1500, 1300), (3, 4100, 4095)])
def test_wide_tiles(device, rows, k, n, dtype, fmt):
    saved = act8.encode(make(device, rows, k, dtype, 1), fmt)
    delta = make(device, rows, n, dtype, 2) * 0.1
    check(delta, saved, torch.float32)
    check(delta, saved, dtype)
    wide = make(device, rows, n + 5, dtype, 3)
    check(wide[:, 3:n + 3], saved, torch.float32)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,k,n", [(96, 64, 48), (515, 4001, 4090)])
def test_infinities_and_nans(device, rows, k, n, dtype, fmt):
    x, delta = make(device, rows, k, dtype, 4), make(device, rows, n, dtype, 5)
    x[5, 3], x[7, 40] = math.nan, -math.inf
    delta[7, 9] = math.inf
    delta[11, 12] = math.nan
    dw, db = act8.linear_backward(delta, act8.encode(x, fmt), torch.float32)
    assert torch.isnan(dw[:, :64]).all()
    rest = torch.ones(n, dtype=torch.bool, device=device)
    rest[9] = rest[12] = False
    assert torch.isnan(dw[12]).all() and not torch.isfinite(dw[9]).any()
    assert torch.isfinite(dw[rest][:, 64:]).all()
    assert db[9] == math.inf and torch.isnan(db[12]) and torch.isfinite(db[rest]).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n", [(40, 96, 24), (515, 4001, 4090)])
def test_blocks_at_the_ends_of_the_range(device, rows, k, n, dtype, fmt):
    # the largest exponent (3e38) and the least (1e-38) in blocks of their own, beside ordinary ones
    x = make(device, rows, k, torch.float32, 6)
    x[3, :32] = torch.linspace(-1, 1, 32, device=device) * 3.3e38
    x[4, 32:64] = torch.linspace(-1, 1, 32, device=device) * 1.6e38
    x[5, :32] = torch.linspace(-1, 1, 32, device=device) * 1e-38
    delta = make(device, rows, n, dtype, 7)
    delta[3] *= 1e-36
    delta[4] *= 1e-36
    delta[3, ::2] = 0
    check(delta, act8.encode(x.to(dtype), fmt), torch.float32)
