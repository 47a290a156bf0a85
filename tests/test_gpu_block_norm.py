"""GPU tests of ``block_norm`` and ``block_norm_nvfp4`` against the formulas in
64 bits.

Tolerances: R is one fp32 fma of exact inputs (and a few fp32 roundings of u)
rounded once, so half a step of its type plus the error of u.  A norm's fp32
sum of D terms, added in a tree of threads after at most 32 serial terms, is
off by at most (32 + 10) 2^-24 relative (all terms of the sum of squares are
positive), which enters the result by half; rsqrt and the products add 6
roundings of 2^-23.  The layer norm's mean is off by 42 * 2^-24 of the mean
magnitude, which the centred values carry as an absolute error."""
import numpy as np
import pytest
import torch

import nvfp4_dual_gemm_b200 as dg

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
REL = 21 * 2.0 ** -24 + 6 * 2.0 ** -23


def norm64(v, kind, w, b, eps):
    """(norm, absolute error bound of the fp32 computation)."""
    mean = v.mean(1, keepdim=True) if kind == "layer" else 0.0
    c = v - mean
    inv = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    shift = 42 * 2.0 ** -24 * v.abs().mean(1, keepdim=True) \
        if kind == "layer" else 0.0
    err = (c.abs() * REL + 2 * shift) * inv
    z = c * inv
    if w is not None:
        z, err = z * w.double(), err * w.double().abs()
    if b is not None:
        z = z + b.double()
        err = err + 2.0 ** -23 * z.abs()
    return z, err


def check(got, want, err, what):
    f = torch.finfo(got.dtype)
    tol = err + f.eps / 2 * (want.abs() + err) + f.smallest_normal * f.eps / 2
    off = (got.double() - want).abs()
    assert (off <= tol).all(), \
        f"{what}: worst {(off / tol).max().item():.3g} x the tolerance"


def problem(rows, d, dtype, seed, gates=0, layer_bias=False, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*s):
        return torch.randn(s, generator=g, device="cuda")
    t = {"x": (rnd(rows, d) * spread).to(dtype), "y": rnd(rows, d).to(dtype),
         "weight": 1 + 0.3 * rnd(d), "post_weight": 1 + 0.3 * rnd(d),
         "bias": 0.2 * rnd(d) if layer_bias else None,
         "post_bias": 0.2 * rnd(d) if layer_bias else None,
         "gate": rnd(gates, d).to(dtype) if gates else None}
    return t


def reference(t, got_r, kind="rms", scale=1.0, eps=1e-6, post=True):
    """Checks R against its formula, and returns Z's from R as it is."""
    u, err = t["y"].double(), 0.0
    if post:
        u, err = norm64(u, kind, t.get("post_weight"), t.get("post_bias"),
                        eps)
    if t.get("gate") is not None:
        f = t["gate"].double().repeat_interleave(
            u.shape[0] // t["gate"].shape[0], 0)
        u, err = u * f, err * f.abs() + 2.0 ** -24 * (u * f).abs()
    r = t["x"].double() + scale * u
    check(got_r, r, abs(scale) * err + 2.0 ** -24 * r.abs(), "R")
    return norm64(got_r.double(), kind, t.get("weight"), t.get("bias"), eps)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,d", [(1, 8), (3, 64), (37, 248), (5, 256),
                                    (700, 264), (9, 512), (2, 1032),
                                    (130, 4096), (4, 4104), (3, 8192),
                                    (2, 8200), (1, 32768)])
def test_norms(rows, d, kind, dtype):
    t = problem(rows, d, dtype, rows + d, gates=1, layer_bias=kind == "layer")
    r, z = dg.block_norm(**t, kind=kind, scale=0.5)
    want, err = reference(t, r, kind, 0.5)
    check(z, want, err, "Z")


@pytest.mark.parametrize("gates", [0, 1, 4, 12])
@pytest.mark.parametrize("post", [False, True])
def test_gates(gates, post):
    t = problem(12, 320, torch.bfloat16, gates, gates)
    if not post:
        t["post_weight"] = None
    r, z = dg.block_norm(**t, scale=-1.5)
    want, err = reference(t, r, scale=-1.5, post=post)
    check(z, want, err, "Z")


def test_pre_only_and_post_only():
    t = problem(50, 640, torch.float16, 1)
    r, z = dg.block_norm(t["x"], weight=t["weight"])
    assert r is t["x"]
    want, err = norm64(t["x"].double(), "rms", t["weight"], None, 1e-6)
    check(z, want, err, "pre")
    r, z = dg.block_norm(t["x"], t["y"], post=True, pre=False)
    assert z is None
    reference({"x": t["x"], "y": t["y"]}, r)


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_of_the_streams_type(dtype):
    t = problem(6, 512, dtype, 2, layer_bias=True)
    for k in ("weight", "post_weight", "bias", "post_bias"):
        t[k] = t[k].to(dtype)
    r, z = dg.block_norm(**t, kind="layer")
    want, err = reference(t, r, "layer")
    check(z, want, err, "Z")


def test_strides_in_place_and_leading_dimensions():
    t = problem(24, 384, torch.bfloat16, 3, gates=4)
    want_r, want_z = dg.block_norm(**t)
    wide = torch.zeros(24, 512, dtype=torch.bfloat16, device="cuda")
    wide[:, 64:448] = t["x"]
    view = wide[:, 64:448]
    r, z = dg.block_norm(**{**t, "x": view}, R=view)
    assert r.data_ptr() == view.data_ptr()
    assert torch.equal(view, want_r) and torch.equal(z, want_z)
    assert (wide[:, :64] == 0).all() and (wide[:, 448:] == 0).all()
    y = t["y"].clone()
    r, _ = dg.block_norm(**{**t, "y": y}, R=y)
    assert torch.equal(y, want_r)
    r, z = dg.block_norm(**{**t, "x": t["x"].view(4, 6, 384),
                            "y": t["y"].view(4, 6, 384),
                            "gate": t["gate"].view(4, 1, 384)})
    assert r.shape == z.shape == (4, 6, 384)
    assert torch.equal(r.view(24, 384), want_r)
    assert torch.equal(z.view(24, 384), want_z)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", [(1, 64), (3, 192), (129, 320), (37, 1024),
                                    (200, 1088), (5, 7168), (2, 16384)])
def test_nvfp4_equals_the_quantiser(rows, d, dtype):
    t = problem(rows, d, dtype, rows * d, gates=1, spread=3.0)
    r, z = dg.block_norm(**t)
    r2, codes, sf = dg.block_norm_nvfp4(**t)
    want = dg.quantize_nvfp4(z, plain=False)
    assert torch.equal(r, r2)
    assert torch.equal(codes, want[0])
    assert torch.equal(sf, want[2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,d,gates", [(301, 1088, 7), (903, 2048, 903),
                                          (640, 4160, 0), (1201, 7168, 1),
                                          (299, 8192, 299)])
def test_many_wide_rows(rows, d, gates, kind, dtype):
    """More rows than the CTAs of a launch, in pairs, the last one alone."""
    t = problem(rows, d, dtype, rows, gates, layer_bias=kind == "layer")
    r, z = dg.block_norm(**t, kind=kind, scale=0.25)
    want, err = reference(t, r, kind, 0.25)
    check(z, want, err, "Z")
    r2, codes, sf = dg.block_norm_nvfp4(**t, kind=kind, scale=0.25)
    quant = dg.quantize_nvfp4(z, plain=False)
    assert torch.equal(r, r2)
    assert torch.equal(codes, quant[0]) and torch.equal(sf, quant[2])
    t["x"] = t["x"].clone()
    dg.block_norm(**t, kind=kind, scale=0.25, R=t["x"], Z=z)
    assert torch.equal(t["x"], r)
    _, z = dg.block_norm(r, weight=t["weight"], bias=t["bias"], kind=kind)
    want, err = norm64(r.double(), kind, t["weight"], t["bias"], 1e-6)
    check(z, want, err, "pre only")
    r, none = dg.block_norm(t["y"], r, post=True, pre=False, kind=kind)
    assert none is None


def test_nvfp4_special_values():
    """NaN and infinite elements, zero rows and huge ones: the same bytes as
    the quantiser gives for Z."""
    x = torch.randn(8, 256, device="cuda").half()
    x[1, 5] = float("nan")
    x[2, 40] = float("inf")
    x[3] = 0
    x[4] = 65504
    x[5] = 6e-8
    for kind in ("rms", "layer"):
        _, z = dg.block_norm(x, kind=kind)
        _, codes, sf = dg.block_norm_nvfp4(x, kind=kind)
        want = dg.quantize_nvfp4(z, plain=False)
        assert torch.equal(codes, want[0]) and torch.equal(sf, want[2])
        rows = [0, 3, 4, 5, 6, 7]
        want, err = norm64(x[rows].double(), kind, None, None, 1e-6)
        check(z[rows], want, err, kind)


def test_mean_far_from_zero():
    """Layer norm of values whose mean is far above their spread."""
    x = 1000 + torch.randn(16, 2048, device="cuda")
    _, z = dg.block_norm(x, kind="layer")
    want, err = norm64(x.double(), "layer", None, None, 1e-6)
    check(z, want, err, "Z")


def test_streams_and_graph():
    t = problem(40, 1536, torch.bfloat16, 5)
    r0, z0 = dg.block_norm(**t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        r1, z1 = dg.block_norm(**t)
    s.synchronize()
    assert torch.equal(r0, r1) and torch.equal(z0, z1)
    g = torch.cuda.CUDAGraph()
    R, Z = torch.empty_like(r0), torch.empty_like(z0)
    with torch.cuda.graph(g):
        dg.block_norm(**t, R=R, Z=Z)
        dg.block_norm(R, t["y"], weight=t["weight"], Z=Z, R=R)
    g.replay()
    r2, z2 = dg.block_norm(r0, t["y"], weight=t["weight"])
    torch.cuda.synchronize()
    assert torch.equal(R, r2) and torch.equal(Z, z2)


@pytest.mark.parametrize("rows,d", [(1, 7168), (40, 512), (800, 2048)])
def test_every_in_place_form(rows, d):
    t = problem(rows, d, torch.bfloat16, rows)
    w = dict(weight=t["weight"], post_weight=t["post_weight"])
    x, y = t["x"], t["y"]
    r0, z0 = dg.block_norm(x, y, **w)
    for r_at, z_at in (("x", "y"), ("y", "x"), ("x", None), (None, "x"),
                       (None, "y")):
        c = {"x": x.clone(), "y": y.clone(), None: None}
        r, z = dg.block_norm(c["x"], c["y"], R=c[r_at], Z=c[z_at], **w)
        assert torch.equal(r, r0) and torch.equal(z, z0)
    z0 = dg.block_norm(x, weight=t["weight"])[1]
    c = x.clone()
    assert torch.equal(dg.block_norm(c, weight=t["weight"], Z=c)[1], z0)
    with pytest.raises(ValueError):
        dg.block_norm(x, y, R=c, Z=c)
    wide = torch.zeros(rows + 1, d, dtype=x.dtype, device="cuda")
    if rows > 1:
        with pytest.raises(ValueError):
            dg.block_norm(wide[1:], y, R=wide[:-1])
