"""The residual norm's loop over rows: more rows than a launch's workgroups hold, twice and a remainder, all of them different, for
every number of threads to a row.  Tolerances: test_residual_norm_gpu.py."""

from __future__ import annotations

import pytest
import torch

from test_residual_norm_gpu import BF16, F16, F32, _check_fp8, _compare, _inputs

pytestmark = pytest.mark.gpu

# rows past twice what a forward's workgroups hold: 8192 rows of 64 threads, 4096 of 128, 2048 of 256, 1024 of 512, 512 of 1024
WIDE16 = [(17001, 384), (8195, 768), (4099, 2048), (2051, 4096), (1031, 8192), (1031, 9000)]
WIDE32 = [(17001, 200), (8195, 512), (4099, 1000), (2051, 2048), (1031, 4096), (1031, 8192), (1031, 9000)]
SINGLE = [(17001, 41), (4099, 1001), (1031, 4001), (1031, 5001)]


def _rows(shape, dtype, stream, wdt, seed):
    """Rows of different sizes: another row's statistics would show."""
    x, r, w, gy, gh = _inputs(shape, dtype, stream, wdt, seed)
    f = 2.0 ** (torch.arange(shape[0], device="cuda") % 7 - 3)[:, None]
    return (x * f).to(dtype), None if r is None else (r * f).to(r.dtype), w, gy, gh


@pytest.mark.parametrize("types", [(BF16, BF16), (F16, F32), (BF16, None)])
@pytest.mark.parametrize("shape", WIDE16 + SINGLE)
def test_rows_one_after_another(shape, types):
    print(f"rows {shape} {types}", flush=True)
    _compare(*_rows(shape, *types, F32, 11), eps=1e-5)


@pytest.mark.parametrize("shape", WIDE32 + SINGLE)
def test_rows_one_after_another_float32(shape):
    print(f"rows {shape}", flush=True)
    _compare(*_rows(shape, F32, F32, F32, 12), eps=1e-5)


@pytest.mark.parametrize("types,shape,group", [
    *[((BF16, BF16), s, g) for s, g in zip(WIDE16, (128, 32, 64, 128, 32, None))], *[((F16, F32), s, None) for s in WIDE16],
    *[((F32, F32), s, g) for s, g in zip(WIDE32, (None, 32, None, 64, 128, None, None))],
    *[((F32, None), s, g) for s, g in zip(WIDE32, (None, None, None, None, None, 128, None))],
    *[((BF16, F32), s, None) for s in SINGLE]])
def test_rows_one_after_another_in_eight_bits(types, shape, group):
    print(f"8 bits {shape} {types} {group}", flush=True)
    x, r, w, _, _ = _rows(shape, *types, F32, 13)
    _check_fp8(x, r, w, group)


def test_different_rows_past_2_31_elements():
    from hclsm_amd.kernels import residual_rms_norm
    n = (1 << 17) + 3
    row = torch.randn(1, 16384, device="cuda").bfloat16()
    x = row * (2.0 ** (torch.arange(n, device="cuda") % 11 - 5)[:, None]).bfloat16()
    y, h = residual_rms_norm(x, row.expand(n, 16384))
    for i in (0, 511, 512, 1025, 65537, n - 2, n - 1):
        a, b = residual_rms_norm(x[i:i + 1], row)
        assert torch.equal(y[i:i + 1], a) and torch.equal(h[i:i + 1], b), i
