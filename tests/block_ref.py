"""64-bit references of the block operators and random NVFP4 operands.

Tolerances: an output rounded once to a type of spacing eps is off by at most
half a step, eps / 2 relative.  A sum of K products of NVFP4 values
(each exact in fp32) that is accumulated 64 products at a time in fp32 is off by at
most one rounding or truncation, 2^-22 relative to the sum of the magnitudes,
for each of its K / 64 steps and again for each split-K partial; the epilogue
adds a few fp32 roundings (2^-24 each) of its intermediate values."""
import numpy as np
import torch

E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4,
                 -6])


def random_nvfp4(rows, k, rng, lo=0x28, hi=0x3C):
    """Random codes [rows, K/2], plain scale bytes [rows, K/16] between two
    e4m3 bit patterns, and the 64-bit values they stand for."""
    codes = rng.integers(0, 256, (rows, k // 2), dtype=np.uint8)
    sf = rng.integers(lo, hi, (rows, k // 16), dtype=np.uint8)
    return codes, sf, values(codes, sf)


def e4m3(b):
    e, f = (b >> 3 & 15).astype(np.float64), (b & 7).astype(np.float64)
    return np.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * 2.0 ** (e - 7))


def values(codes, sf):
    v = np.empty((codes.shape[0], 2 * codes.shape[1]))
    v[:, 0::2] = E2M1[codes & 15]
    v[:, 1::2] = E2M1[codes >> 4]
    return v * np.repeat(e4m3(sf), 16, axis=1)


def blocked(sf):
    """Plain scale bytes -> the blocked layout; padding rows get 0x7F, the
    e4m3 NaN, which no output of a valid row may see."""
    rows, c = sf.shape
    p = np.full(((rows + 127) // 128 * 128, c), 0x7F, np.uint8)
    p[:rows] = sf
    return np.ascontiguousarray(
        p.reshape(-1, 4, 32, c // 4, 4).transpose(0, 3, 2, 1, 4)).ravel()


def act64(v, act):
    if act == "relu":
        return np.maximum(v, 0)
    if act == "silu":
        return v / (1 + np.exp(-v))
    if act == "gelu_tanh":
        u = np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)
        return 0.5 * v * (1 + np.tanh(u))
    if act == "gelu":
        return (0.5 * torch.from_numpy(v)
                * torch.erfc(torch.from_numpy(-v) * 0.5 ** 0.5)).numpy()
    return v


def linear64(a, b, bias=None, act=None, residual=None, row_scale=None,
             alpha=1.0):
    """(reference, error bound before the final rounding)."""
    k = a.shape[1]
    s = a @ b.T * alpha
    # 8 more steps for the partials of a split K range
    err = (k / 64 + 8) * 2.0 ** -22 * (np.abs(a) @ np.abs(b).T) * abs(alpha)
    if bias is not None:
        s = s + bias
        err = err + 2.0 ** -23 * np.abs(s)
    v = act64(s, act)
    # slopes of the activations stay below 1.13; the fast exponential is off
    # by 2^-21 relative for the arguments here, the quotient by 2^-22
    err = 1.13 * err + (2.0 ** -20 * np.abs(s) if act else 0)
    if row_scale is not None:
        v = v * row_scale[:, None]
        err = err * np.abs(row_scale[:, None]) + 2.0 ** -24 * np.abs(v)
    if residual is not None:
        v = v + residual
        err = err + 2.0 ** -24 * np.abs(v)
    return v, err


def assert_linear(got, want, err, what=""):
    """`got` (fp16 / bf16) against linear64's pair."""
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * 2 * half
    # the bound before rounding, the half step of the rounded value, and the
    # half step of the subnormals
    tol = err + half * (np.abs(want) + err) + tiny / 2
    off = np.abs(got.double().cpu().numpy() - want)
    bad = ~(off <= tol)
    assert not bad.any(), (
        f"{what}: {bad.sum()} of {bad.size} outside; worst "
        f"{np.nanmax(np.where(bad, off / tol, 0)):.3g} x the tolerance at "
        f"{np.argwhere(bad)[0]}")
