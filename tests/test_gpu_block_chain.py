"""GPU tests of the block operators together, as a transformer block and a
mixture of experts use them, and of the refusals of their Python entry points.

Each step is compared with 64-bit arithmetic on the values its inputs stand
for (the step before it as it came out), so that every tolerance is one
operator's own."""
import numpy as np
import pytest
import torch

import nvfp4_dual_gemm_b200 as dg
from tests.block_ref import (assert_linear, blocked, linear64, random_nvfp4,
                             values)

pytestmark = pytest.mark.gpu


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def weights(n, k, seed):
    rng = np.random.default_rng(seed)
    c, s, v = random_nvfp4(n, k, rng, 0x10, 0x24)
    return dev(c), dev(blocked(s)), v


def stands_for(codes, sf, rows, k):
    """64-bit values of device codes and blocked scales."""
    plain = dg.scales_from_blocked(sf, rows, k).cpu().numpy()
    return values(codes.cpu().numpy(), plain)


def block(t, w):
    """norm -> gate and up -> down + residual -> norm."""
    r, a, sfa = dg.block_norm_nvfp4(t["x"], t["y"], weight=t["w1"],
                                    post_weight=t["w0"], scale=0.5)
    h, sfh = dg.dual_gemm_nvfp4(a, w["b1"][0], w["b2"][0], sfa, w["b1"][1],
                                w["b2"][1])
    out = dg.linear(h, w["down"][0], sfh, w["down"][1], residual=r,
                    bias=t["bias"])
    s, z = dg.block_norm(out, weight=t["w1"])
    return {"r": r, "a": a, "sfa": sfa, "h": h, "sfh": sfh, "out": out,
            "z": z, "s": s}


@pytest.mark.parametrize("rows", [1, 37, 300])
def test_ffn_block(rows):
    d, f = 512, 1024
    g = torch.Generator(device="cuda").manual_seed(rows)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    t = {"x": rnd(rows, d).half(), "y": rnd(rows, d).half(),
         "w0": 1 + 0.1 * rnd(d), "w1": 1 + 0.1 * rnd(d), "bias": rnd(d)}
    w = {"b1": weights(f, d, 1), "b2": weights(f, d, 2),
         "down": weights(d, f, 3)}
    o = block(t, w)
    a = stands_for(o["a"], o["sfa"], rows, d)
    _, z = dg.block_norm(o["r"], weight=t["w1"])
    want = dg.quantize_nvfp4(z, plain=False)
    assert torch.equal(o["a"], want[0]) and torch.equal(o["sfa"], want[2])
    gate, up = a @ w["b1"][2].T, a @ w["b2"][2].T
    h64 = gate / (1 + np.exp(-gate)) * up
    h = stands_for(o["h"], o["sfh"], rows, f)
    # e2m1 steps are at most 2 of 6 wide and the scale is half a step of e4m3
    # off, so a block's values are within (1 / 6 + 1 / 16) of its largest
    top = np.abs(h64.reshape(rows, -1, 16)).max(2).repeat(16, 1)
    assert (np.abs(h - h64) <= (1 / 6 + 1 / 16) * top + 1e-3).all()
    ref, err = linear64(h, w["down"][2], t["bias"].double().cpu().numpy(),
                        residual=o["r"].double().cpu().numpy())
    assert_linear(o["out"], ref, err, "down")
    assert o["s"] is o["out"]
    # captured and replayed on other inputs of the same shape
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        p = block(t, w)
    t["x"].copy_(rnd(rows, d))
    t["y"].copy_(rnd(rows, d))
    gr.replay()
    eager = block(t, w)
    torch.cuda.synchronize()
    for k in eager:
        assert torch.equal(eager[k], p[k]), k


def test_mixture_of_experts():
    tokens, d, f, experts, top = 50, 256, 512, 6, 2
    rng = np.random.default_rng(7)
    x = torch.randn(tokens, d, device="cuda").half()
    # expert 4 gets nothing
    pick = torch.from_numpy(np.stack([rng.choice([0, 1, 2, 3, 5], top,
                                                 replace=False)
                                      for _ in range(tokens)])).cuda()
    share = torch.softmax(torch.randn(tokens, top, device="cuda"), -1)
    order = torch.argsort(pick.flatten(), stable=True)
    counts = torch.bincount(pick.flatten(), minlength=experts)
    rows = counts.tolist()
    row0 = dg.group_offsets(rows)
    R = row0[-1] + 128
    at = torch.cat([torch.arange(r, r + n) for r, n in zip(row0, rows)]).cuda()
    xs = torch.zeros(R, d, dtype=torch.float16, device="cuda")
    xs[at] = x[order // top]
    scale = torch.zeros(R, device="cuda")
    scale[at] = share.flatten()[order]
    w1 = [weights(f, d, 10 + e) for e in range(experts)]
    w2 = [weights(f, d, 20 + e) for e in range(experts)]
    w3 = [weights(d, f, 30 + e) for e in range(experts)]

    def stack(ws):
        return (torch.stack([w[0] for w in ws]).permute(1, 2, 0),
                torch.cat([w[1] for w in ws]))
    (b1, s1), (b2, s2), (b3, s3) = stack(w1), stack(w2), stack(w3)
    a, _, sfa = dg.quantize_nvfp4(xs)
    h = torch.zeros(R, f, dtype=torch.float16, device="cuda")
    dg.dual_gemm_grouped(a, b1, b2, sfa, s1, s2, h, rows)
    hq, plain, sfh = dg.quantize_nvfp4(h)
    out = torch.full((R, d), float("nan"), dtype=torch.bfloat16,
                     device="cuda")
    dg.linear_grouped(hq, b3, sfh, s3, out, counts.int(), row_scale=scale)
    h64 = values(hq.cpu().numpy(), plain.view(torch.uint8).cpu().numpy())
    for e, (r, n) in enumerate(zip(row0, rows)):
        if n:
            s = slice(r, r + n)
            ref, err = linear64(h64[s], w3[e][2],
                                row_scale=scale[s].double().cpu().numpy())
            assert_linear(out[s], ref, err, f"expert {e}")
    other = torch.ones(R, dtype=torch.bool, device="cuda")
    other[at] = False
    assert torch.isnan(out[other]).all()
    # combined back to the tokens
    y = torch.zeros(tokens, d, device="cuda")
    y.index_add_(0, order // top, out[at].float())
    assert torch.isfinite(y).all()


def operands(m=4, n=128, k=128):
    a, sfa, _ = weights(m, k, 1)
    b, sfb, _ = weights(n, k, 2)
    return a, b, sfa, sfb


def test_linear_refusals():
    a, b, sfa, sfb = operands()
    f16 = dict(dtype=torch.float16, device="cuda")
    bad = [
        dict(activation="tanh"), dict(dtype=torch.float32),
        dict(bias=torch.zeros(127, device="cuda")),
        dict(bias=torch.zeros(128, dtype=torch.bfloat16, device="cuda")),
        dict(bias=torch.zeros(128)),
        dict(residual=torch.zeros(4, 64, **f16)),
        dict(residual=torch.zeros(4, 128, device="cuda"),
             dtype=torch.float16),
        dict(residual=torch.zeros(1, 128, **f16).expand(4, 128)),
        dict(residual=torch.zeros(128, 4, **f16).t()),
        dict(row_scale=torch.zeros(4, **f16)),
        dict(row_scale=torch.zeros(5, device="cuda")),
        dict(C=torch.zeros(5, 128, **f16)),
        dict(C=torch.zeros(4, 128, **f16), dtype=torch.bfloat16),
        dict(C=torch.zeros(4, 132, **f16)[:, 4:]),
        dict(flags=1 << 12),
        dict(residual=torch.zeros(4, 128, requires_grad=True, **f16)),
    ]
    for kw in bad:
        with pytest.raises(ValueError):
            dg.linear(a, b, sfa, sfb, **kw)
    with pytest.raises(ValueError):
        dg.linear(a.float(), b, sfa, sfb)
    with pytest.raises(ValueError):
        dg.linear(a, b[:, :32], sfa, sfb)
    with pytest.raises(ValueError):
        dg.linear(a, b, sfa[:-1], sfb)
    with pytest.raises(ValueError):
        dg.linear(a.cpu(), b, sfa, sfb)
    with pytest.raises(ValueError):
        dg.linear(a, b[:100], sfa, sfb)  # N % 8
    with torch.no_grad():
        dg.linear(a, b, sfa, sfb,
                  residual=torch.zeros(4, 128, requires_grad=True, **f16))
    assert dg.linear(a[:0], b, sfa[:0], sfb).shape == (0, 128)


def test_linear_grouped_refusals():
    a, b, sfa, sfb = operands(m=256)
    b3 = b.unsqueeze(0).expand(2, -1, -1).contiguous().permute(1, 2, 0)
    sf3 = torch.cat([sfb, sfb])
    c = torch.zeros(256, 128, dtype=torch.float16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    calls = [
        ([4, 4, 4], None, {}), ([4], None, {}), ([4, 129], None, {}),
        ([-1, 4], None, {}), ([4, 4], [0], {}), ([4, 4], [0, 64], {}),
        (torch.tensor([4, 4], device="cuda"), None, {}),  # int64
        (torch.tensor([4, 4], **i32), [0, 128], {}),
        ([4, 4], torch.tensor([0, 128], **i32), {}),
        (torch.tensor([[4, 4]], **i32), None, {}),
        ([4, 4], None, dict(bias=torch.zeros(128, device="cuda"))),
        ([4, 4], None, dict(row_scale=torch.zeros(255, device="cuda"))),
    ]
    for rows, row0, kw in calls:
        with pytest.raises(ValueError):
            dg.linear_grouped(a, b3, sfa, sf3, c, rows, row0, **kw)
    with pytest.raises(ValueError):
        dg.linear_grouped(a, b3, sfa, sfb, c, [4, 4])  # one SFB
    with pytest.raises(ValueError):
        dg.linear_grouped(a, b3, sfa, sf3, c[:, :64], [4, 4])
    assert (c == 0).all()


def test_block_norm_refusals():
    x = torch.zeros(6, 128, dtype=torch.float16, device="cuda")
    y, w = torch.zeros_like(x), torch.ones(128, device="cuda")
    bad = [
        dict(y=y[:5]), dict(y=y.float()), dict(y=y.cpu()),
        dict(weight=w[:64]), dict(weight=w.bfloat16()),
        dict(weight=w, bias=w.half()), dict(kind="group"), dict(eps=-1.0),
        dict(gate=x), dict(post=True), dict(R=y),
        dict(y=y, gate=x[:4]), dict(y=y, gate=x.float()),
        dict(pre=False, weight=w), dict(pre=False, Z=y),
        dict(weight=w.cpu()), dict(weight=w.clone().requires_grad_()),
        dict(weight=torch.ones(132, device="cuda")[1:129]),  # alignment
    ]
    for kw in bad:
        with pytest.raises(ValueError):
            dg.block_norm(x, **kw)
    for t in (x.cpu(), x.double(), x[:, :100], x.t(), x[:, :0]):
        with pytest.raises(ValueError):
            dg.block_norm(t)
    with pytest.raises(ValueError):
        dg.block_norm_nvfp4(x[:, :72])
    r, z = dg.block_norm(x[:0], y[:0])
    assert r.shape == z.shape == (0, 128)
    r, codes, sf = dg.block_norm_nvfp4(x[:0])
    assert codes.shape == (0, 64) and sf.numel() == 0


def test_two_streams_at_once():
    """Calls on two streams share no state of the library's."""
    a, b, sfa, sfb = operands(m=40, n=512, k=2048)
    want = dg.linear(a, b, sfa, sfb)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                outs.append(dg.linear(a, b, sfa, sfb))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)


FIRST_IN_CAPTURE = """
import torch
import nvfp4_dual_gemm_b200 as dg
x = torch.randn(5, 256, device="cuda").half()
b = torch.randint(0, 256, (64, 128), dtype=torch.uint8, device="cuda")
sfb = torch.full((128 * 16,), 0x30, dtype=torch.uint8, device="cuda")
w = torch.ones(256, device="cuda")
counts = torch.tensor([5], dtype=torch.int32, device="cuda")
c2 = torch.zeros(5, 64, dtype=torch.float16, device="cuda")
def step():
    _, a, sfa = dg.block_norm_nvfp4(x, weight=w)
    dg.linear_grouped(a, b, sfa, sfb, c2, counts)
    return dg.linear(a, b, sfa, sfb)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    c = step()
g.replay()
torch.cuda.synchronize()
assert torch.equal(c, step()) and torch.equal(c, c2)
print("same")
"""


def test_first_calls_of_a_process_inside_a_capture():
    import subprocess
    import sys
    out = subprocess.run([sys.executable, "-c", FIRST_IN_CAPTURE],
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "same" in out.stdout, out.stderr[-2000:]


def test_scales_that_ask_for_a_gradient_are_refused():
    a, b, sfa, sfb = operands()
    f8 = sfb.view(torch.float8_e4m3fn)
    dg.linear(a, b, sfa, f8)
    with pytest.raises(ValueError, match="inference only"):
        dg.linear(a, b, sfa, f8.detach().requires_grad_())
