"""GPU tests of what the block operators' documentation allows at its edges:
outputs beside their inputs in one buffer, tensors that autograd knows,
schedules where a CTA's tiles belong to several groups, and many wide rows."""
import subprocess
import sys

import pytest
import torch

import nvfp4_dual_gemm_b200 as dg
from nvfp4_dual_gemm_b200 import _lib
from tests.test_gpu_block_norm import check, problem, reference
from tests.test_gpu_linear import TILES, Groups

pytestmark = pytest.mark.gpu


def linear_operands(m, n, k, seed=0):
    """Random codes and scales of 0.25 to 0.5 for A [m, k] and B [n, k]."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    u8 = dict(dtype=torch.uint8, device="cuda")

    def matrix(rows):
        return (torch.randint(0, 256, (rows, k // 2), generator=g, **u8),
                torch.randint(0x28, 0x30, ((rows + 127) // 128 * 8 * k,),
                              generator=g, **u8))
    (a, sfa), (b, sfb) = matrix(m), matrix(n)
    return a, b, sfa, sfb


def test_c_beside_the_bias_in_one_buffer():
    """The bias in the columns that a strided C leaves out is no overlap; in
    C's own it is."""
    m, n, k = 9, 64, 128
    ops = linear_operands(m, n, k)
    both = torch.randn(m, 2 * n, device="cuda").half()
    bias = both[0, n:]
    want = dg.linear(*ops, bias=bias.clone())
    keep = both[:, n:].clone()
    got = dg.linear(*ops, both[:, :n], bias=bias)
    assert torch.equal(got, want) and torch.equal(both[:, n:], keep)
    with pytest.raises(ValueError, match="must not overlap bias"):
        dg.linear(*ops, both[:, :n], bias=both[3, :n])
    assert torch.equal(got, want)


def test_norm_outputs_beside_gate_and_weight_in_one_buffer():
    """Gate and weights in the columns that a strided R leaves out are no
    overlap; in its own they are."""
    rows, d = 7, 128
    x, y = (torch.randn(rows, d, device="cuda").half() for _ in range(2))
    both = torch.randn(rows, 2 * d, device="cuda").half()
    gate, w = both[0, d:], both[5, d:]
    want = dg.block_norm(x, y, gate=gate.clone(), weight=w.clone())
    keep = both[:, d:].clone()
    r, z = dg.block_norm(x, y, gate=gate, weight=w, R=both[:, :d])
    assert torch.equal(r, want[0]) and torch.equal(z, want[1])
    assert torch.equal(both[:, d:], keep)
    for kw in (dict(gate=both[2, :d]), dict(weight=both[2, :d]),
               dict(post_bias=both[6, :d])):
        with pytest.raises(ValueError, match="must not overlap R or Z"):
            dg.block_norm(x, y, R=both[:, :d], **kw)
    assert torch.equal(r, want[0])


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fw

    def refused():
        return pytest.raises(ValueError, match="inference only")
    n, half = 128, dict(dtype=torch.float16, device="cuda")
    ops = linear_operands(4, n, 128)
    f8 = ops[3].view(torch.float8_e4m3fn)
    x, y, w = (torch.randn(4, n, **half), torch.randn(4, n, **half),
               torch.ones(n, device="cuda"))
    want, norm = dg.linear(*ops, residual=x), dg.block_norm(x, y, weight=w)
    with fw.dual_level():
        def dual(t):
            return fw.make_dual(t, torch.ones_like(t))
        for kw in (dict(bias=dual(w)), dict(residual=dual(x)),
                   dict(row_scale=dual(torch.ones(4, device="cuda")))):
            with torch.no_grad(), refused():
                dg.linear(*ops, **kw)
        with refused():
            dg.linear(*ops, dual(x.clone()))
        with refused():
            dg.linear_grouped(*ops, x.clone(), [4], bias=dual(w[None]))
        for args, kw in (((dual(x),), {}), ((x, dual(y)), {}),
                         ((x,), dict(weight=dual(w))),
                         ((x,), dict(bias=dual(w))),
                         ((x, y), dict(post_weight=dual(w))),
                         ((x, y), dict(gate=dual(x[0].clone()))),
                         ((x, y), dict(R=dual(x.clone())))):
            with refused():
                dg.block_norm(*args, **kw)
            with refused():
                dg.block_norm_nvfp4(*args, **kw)
        # with the tangent taken off, or with forward mode off as inside a
        # custom function's forward
        assert torch.equal(dg.linear(*ops[:3], f8,
                                     residual=fw.unpack_dual(dual(x)).primal),
                           want)

        class Norm(torch.autograd.Function):
            @staticmethod
            def forward(ctx, v):
                return dg.block_norm(v, y, weight=w)[1]

            @staticmethod
            def jvp(ctx, t):
                return t
        assert torch.equal(fw.unpack_dual(Norm.apply(dual(x))).primal,
                           norm[1])


def test_outputs_of_the_callers_raise_their_version():
    n, half = 256, dict(dtype=torch.float16, device="cuda")
    ops = linear_operands(4, n, n)
    x, y = torch.randn(4, n, **half), torch.randn(4, n, **half)
    d = dg.generate_input(4, n, 2 * n)
    a, b1, b2, sfa, sfb1, sfb2 = (d[i] for i in (0, 1, 2, 6, 7, 8))
    c = d[9].squeeze(2)
    cq, sfc = dg.dual_gemm_nvfp4(a, b1, b2, sfa, sfb1, sfb2)
    host = [t.cpu().pin_memory() for t in (*(t.view(torch.uint8) for t in (
        a, b1, b2, sfa, sfb1, sfb2)), d[9])]
    calls = {
        "linear": (lambda t: dg.linear(*ops, t), x.clone()),
        "in place": (lambda t: dg.linear(*ops, t, residual=t), x.clone()),
        "linear_grouped": (lambda t: dg.linear_grouped(*ops, t, [4]),
                           x.clone()),
        "R": (lambda t: dg.block_norm(x, y, R=t), x.clone()),
        "Z": (lambda t: dg.block_norm(x, y, Z=t), x.clone()),
        "R of nvfp4": (lambda t: dg.block_norm_nvfp4(t, y, R=t), x.clone()),
        "dual_gemm": (lambda t: dg.dual_gemm(a, b1, b2, sfa, sfb1, sfb2, t),
                      c.clone()),
        "custom_kernel": (lambda t: dg.custom_kernel((*d[:9], t)), c.clone()),
        "dual_gemm_grouped": (lambda t: dg.dual_gemm_grouped(
            a, b1, b2, sfa, sfb1, sfb2, t, [4]), c.clone()),
        "Cq": (lambda t: dg.dual_gemm_nvfp4(a, b1, b2, sfa, sfb1, sfb2, t),
               cq),
        "SFC": (lambda t: dg.dual_gemm_nvfp4(a, b1, b2, sfa, sfb1, sfb2,
                                             SFC=t), sfc),
        "dual_gemm_host": (lambda t: dg.dual_gemm_host(*host[:6], t),
                           host[6]),
    }
    for name, (call, t) in calls.items():
        before, reads = t._version, (x._version, y._version)
        call(t)
        assert t._version > before, name
        assert (x._version, y._version) == reads, name
        view = t[:2]
        call(t)
        assert view._version == t._version, name
    with torch.inference_mode():
        t = x.clone()
        dg.linear(*ops, t, residual=t)
        dg.block_norm(t, y, R=t)
    dg.linear(*ops, t)  # and outside of it: an inference tensor has no version
    torch.cuda.synchronize()


def test_a_saved_tensor_that_is_overwritten_fails_its_backward():
    w = torch.randn(4, 64, device="cuda", requires_grad=True)
    s = torch.exp(w)  # backward reads s
    dg.block_norm(s.detach(), torch.ones(4, 64, device="cuda"),
                  R=s.detach())
    with pytest.raises(RuntimeError, match="inplace"):
        s.sum().backward()


@pytest.mark.parametrize("flags", [1 << 32, (1 << 32) + 4, -1])
def test_flags_beyond_32_bits_are_refused(flags):
    ops = linear_operands(4, 256, 256)
    x = torch.randn(4, 256, device="cuda").half()
    for call in (lambda: dg.linear(*ops, flags=flags),
                 lambda: dg.linear_grouped(*ops, x, [4], flags=flags),
                 lambda: dg.block_norm(x, flags=flags),
                 lambda: dg.block_norm_nvfp4(x, flags=flags),
                 lambda: dg.dual_gemm(ops[0], ops[1], ops[1], ops[2], ops[3],
                                      ops[3], x, flags=flags)):
        with pytest.raises(ValueError, match="32 bits"):
            call()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_without_its_pair_kernel_the_other_tiles_compute(dtype):
    """A build whose pair kernel cannot be launched leaves its problems to the
    128-token tiles, which round the same sums the same way."""
    m, n, k = 2048, 2056, 2048
    ops = linear_operands(m, n, k)
    assert dg.linear_plan(m, n, k)["tokens"] == 256
    flags = _lib.LINEAR_TEST_NO_PAIR | _lib.FLAG_SYNC_CHECK
    want = dg.linear(*ops, dtype=dtype, flags=_lib.LINEAR_TOKENS128)
    got = dg.linear(*ops, dtype=dtype, flags=flags)
    assert torch.equal(got, want)
    b, sfb = ops[1][None].permute(1, 2, 0), ops[3]
    for counts in ([m], torch.tensor([m], dtype=torch.int32, device="cuda")):
        got.zero_()
        dg.linear_grouped(ops[0], b, ops[2], sfb, got, counts, flags=flags)
        assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="pair kernel"):
        dg.linear(*ops, dtype=dtype, flags=flags | _lib.LINEAR_PAIR)


# boxed and row-by-row stores, groups that end within a tile and empty ones
# alternate among the tiles of one CTA
MIXED = [0, 300, 37, 128, 513, 0, 255, 129]


@pytest.mark.parametrize("where", ["host", "device"])
@pytest.mark.parametrize("tile", ["auto", "t32", "t64", "t128", "pair"])
def test_grouped_tiles_of_several_groups_in_one_cta(tile, where):
    """More tiles than workers: 162 of pairs, 490 of 128 tokens and more of
    the others."""
    p = Groups(MIXED, 4360, 576, seed=21)
    rows = MIXED if where == "host" else torch.tensor(
        MIXED, dtype=torch.int32, device="cuda")
    p.run(rows, flags=TILES[tile])
    p.check()


def test_grouped_pairs_replayed_with_other_counts():
    p = Groups(MIXED, 2312, 320, seed=22, cap=2304)
    counts = torch.tensor(MIXED, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dg.linear_grouped(p.A, p.B, p.SFA, p.SFB, p.C, counts, bias=p.bias,
                          activation="silu", row_scale=p.w,
                          flags=_lib.LINEAR_PAIR)
    for new in (MIXED, MIXED[::-1], [257, 1, 0, 511, 128, 64, 256, 5],
                [0] * 7 + [1500], MIXED):
        counts.copy_(torch.tensor(new, dtype=torch.int32))
        p.C.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        p.check(new, dg.group_offsets(new))


def test_grouped_pairs_on_two_streams():
    p = Groups(MIXED, 2312, 320, seed=23)
    args = (p.A, p.B, p.SFA, p.SFB)
    kw = dict(bias=p.bias, activation="silu", row_scale=p.w,
              flags=_lib.LINEAR_PAIR)
    counts = torch.tensor(MIXED, dtype=torch.int32, device="cuda")
    p.C.zero_()
    dg.linear_grouped(*args, p.C, counts, **kw)
    outs = [torch.zeros_like(p.C) for _ in range(16)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i, c in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            dg.linear_grouped(*args, c, counts, **kw)
    torch.cuda.synchronize()
    assert all(torch.equal(c, p.C) for c in outs)


FIRST_PAIR_IN_CAPTURE = """
import torch
import nvfp4_dual_gemm_b200 as dg
from nvfp4_dual_gemm_b200 import _lib
u8 = dict(dtype=torch.uint8, device="cuda")
a = torch.randint(0, 256, (300, 128), **u8)
b = torch.randint(0, 256, (520, 128), **u8)
sfa, sfb = torch.full((3 * 2048,), 0x30, **u8), torch.full((5 * 2048,), 0x30,
                                                           **u8)
x = torch.randn(400, 2048, device="cuda").half()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    c = dg.linear(a, b, sfa, sfb, flags=_lib.LINEAR_PAIR)
    z = dg.block_norm(x, x)[1]
g.replay()
torch.cuda.synchronize()
assert torch.equal(c, dg.linear(a, b, sfa, sfb, flags=_lib.LINEAR_PAIR))
assert torch.equal(z, dg.block_norm(x, x)[1])
print("same")
"""


def test_first_pair_and_ring_calls_of_a_process_inside_a_capture():
    out = subprocess.run([sys.executable, "-c", FIRST_PAIR_IN_CAPTURE],
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "same" in out.stdout, out.stderr[-2000:]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,d,gates", [(301, 8256, 7), (700, 16384, 0),
                                          (310, 20032, 310), (300, 32768, 1)])
def test_many_rows_wider_than_8192(rows, d, gates, kind, dtype):
    t = problem(rows, d, dtype, rows, gates, layer_bias=kind == "layer")
    r, z = dg.block_norm(**t, kind=kind, scale=0.25)
    want, err = reference(t, r, kind, 0.25)
    check(z, want, err, "Z")
    r2, codes, sf = dg.block_norm_nvfp4(**t, kind=kind, scale=0.25)
    quant = dg.quantize_nvfp4(z, plain=False)
    assert torch.equal(r, r2)
    assert torch.equal(codes, quant[0]) and torch.equal(sf, quant[2])


def test_mixed_operators_on_two_streams():
    """Norms with a ring, few-token and pair products of two streams at once
    give the bits that each gives alone."""
    m, d, n = 400, 2048, 1032
    x, y = (torch.randn(m, d, device="cuda").bfloat16() for _ in range(2))
    b, sfb = linear_operands(1, n, d)[1::2]
    w = torch.ones(d, device="cuda")

    def step(rows):
        r, a, sfa = dg.block_norm_nvfp4(x[:rows], y[:rows], weight=w,
                                        post_weight=w)
        return r, a, sfa, dg.linear(a, b, sfa, sfb, dtype=x.dtype)
    sizes = (1, 40, 400)
    want = {rows: step(rows) for rows in sizes}
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(60):
        rows = sizes[i % 3]
        with torch.cuda.stream(streams[i * 7 // 3 % 2]):
            got.append((rows, step(rows)))
    torch.cuda.synchronize()
    for rows, out in got:
        for a, e in zip(out, want[rows]):
            assert torch.equal(a, e)
