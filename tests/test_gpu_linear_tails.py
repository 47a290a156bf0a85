"""GPU tests of ``linear``'s activations over the whole range of their
arguments: zero, tiny, far negative (where the result leaves the range of
normal numbers), huge, infinite and NaN.

The operands' codes are zero, so that the argument is the bias, exactly.

Tolerance: half a step of C's type (half its smallest subnormal below the
normal range), and before that rounding, in fp32: an exponent t (the power of
two that the quotient's denominator or erfc's value has) is off by 2^-22 |t|
from its constants and products and by 2^-21 from the shift that keeps the
denominator's reciprocal in range, both of which enter the result by ln 2; the
exponential, the reciprocal, erfcf and the last products are off by
2^-20 together; and a factor that is subnormal is off by 2^-148, absolutely."""
import numpy as np
import pytest
import torch

import nvfp4_dual_gemm_b200 as dg
from nvfp4_dual_gemm_b200 import _lib

pytestmark = pytest.mark.gpu

INF = float("inf")
POINTS = [0.0, 1e-45, 1e-40, 2.0 ** -126, 3e-38, 1e-30, 1e-10, 2.0 ** -12,
          0.03, 0.5, 1.0, 2.5, 5.0, 7.5, 9.0, 10.0, 10.02, 10.1, 10.2, 10.25,
          10.3, 10.4, 10.45, 10.5, 10.8, 11.5, 12.9, 13.1, 13.3, 13.6, 16.0, 40.0, 80.0, 86.9, 87.4, 88.0, 88.5, 88.8, 89.5,
          90.5, 91.5, 92.0, 93.0, 95.0, 97.0, 103.0, 104.5, 150.0, 1e3, 7e4,
          1e9, 1e18, 3e19, 1e30, 3e38, INF]
TILES = {"auto": 0, "t32": _lib.LINEAR_TOKENS32, "t128": _lib.LINEAR_TOKENS128,
         "pair": _lib.LINEAR_PAIR}


def reference(x, act):
    """(act(x), the exponent t of its far side) in 64 bits, in forms that do
    not cancel."""
    if act == "relu":
        return np.where(x < 0, 0.0, x), np.zeros_like(x)
    if act == "silu":
        return x / (1 + np.exp(-x)), np.abs(x) * np.log2(np.e)
    if act == "gelu_tanh":
        u = 2 * np.sqrt(2 / np.pi) * (x + 0.044715 * x ** 3)
        return x / (1 + np.exp(-u)), np.abs(u) * np.log2(np.e)
    v = torch.from_numpy(x)
    return ((0.5 * v * torch.erfc(-v * 0.5 ** 0.5)).numpy(),
            x * x * np.log2(np.e))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tile", list(TILES))
@pytest.mark.parametrize("act", ["relu", "silu", "gelu_tanh", "gelu"])
def test_arguments_of_any_size(act, tile, dtype):
    x = np.float32(POINTS + [-v for v in POINTS] + [float("nan")] * 8)
    n, m, k = len(x), 3, 64
    zero = torch.zeros
    u8 = dict(dtype=torch.uint8, device="cuda")
    got = dg.linear(zero(m, k // 2, **u8), zero(n, k // 2, **u8),
                    zero(512, **u8), zero(512, **u8), dtype=dtype,
                    bias=torch.from_numpy(x).cuda(), activation=act,
                    flags=TILES[tile])
    got = got.double().cpu().numpy()
    with np.errstate(all="ignore"):
        want, t = reference(x.astype(np.float64), act)
        info = torch.finfo(dtype)
        half, least = info.eps / 2, info.smallest_normal * info.eps
        t = np.minimum(t, 200.0)
        err = np.abs(want) * (2.0 ** -20 + np.log(2) * (
            2.0 ** -22 * t + 2.0 ** -21)) if act != "relu" else 0 * t
        err = err + np.minimum(np.abs(x), 200.0) * 2.0 ** -148
        tol = err + half * (np.abs(want) + err) + least / 2
        # past the largest value and half a step: an infinity
        want = np.where(np.abs(want) >= info.max * (1 + info.eps / 4),
                        np.sign(want) * INF, want)
        for row in got:
            same = (np.isnan(row) & np.isnan(want)) | (row == want)
            bad = ~(same | (np.abs(row - want) <= tol))
            assert not bad.any(), [
                (float(x[i]), row[i], want[i]) for i in np.nonzero(bad)[0]]
