"""CPU tests of the block operators' C ABI: every argument that must be
refused is refused before anything touches a GPU, empty problems are no-ops,
and the schedule of ``linear`` covers what it must."""
import ctypes

import pytest
import torch

import nvfp4_dual_gemm_b200 as dg
from nvfp4_dual_gemm_b200 import _lib

P = 0x1000  # an aligned address that no refused call may follow


def linear_args(**kw):
    a = dict(A=P, B=P, SFA=P, SFB=P, C=P, ldc=256, M=4, N=256, K=128,
             c_dtype=_lib.DTYPE_BF16, alpha=1.0)
    a.update(kw)
    return _lib.LinearArgs(**a)


def run_linear(**kw):
    return _lib.load().nvfp4_linear_run(ctypes.byref(linear_args(**kw)), None)


@pytest.mark.parametrize("kw,word", [
    (dict(M=-1), "non-negative"), (dict(N=252), "multiple of 8"),
    (dict(K=96), "multiple of 64"), (dict(K=0), "multiple of 64"),
    (dict(c_dtype=_lib.DTYPE_F32), "F16 or BF16"), (dict(c_dtype=9), "F16"),
    (dict(bias=P, bias_dtype=_lib.DTYPE_F16), "bias"),
    (dict(activation=5), "activation"), (dict(activation=-1), "activation"),
    (dict(alpha=float("nan")), "alpha"),
    (dict(flags=1 << 12), "flag"), (dict(flags=3), "exclusive"),
    (dict(flags=0x500), "split"), (dict(C=None), "NULL"),
    (dict(A=None), "NULL"), (dict(SFB=None), "NULL"),
    (dict(ldc=248), "pitch"), (dict(residual=P, ldr=0), "pitch"),
    (dict(ldc=1 << 23), "pitch"), (dict(M=(1 << 30) + 1), "too"),
    (dict(M=1 << 30, N=1 << 20, ldc=1 << 20), "tiles"),
])
def test_linear_refuses(kw, word):
    assert run_linear(**kw) == _lib.ERR_INVALID
    assert word in _lib.last_error()


@pytest.mark.parametrize("kw", [
    dict(A=P + 8), dict(SFA=P + 4), dict(C=P + 2), dict(ldc=260),
    dict(residual=P + 8, ldr=256), dict(residual=P, ldr=262),
    dict(bias=P + 2, bias_dtype=_lib.DTYPE_F32), dict(row_scale=P + 2),
])
def test_linear_refuses_misaligned(kw):
    assert run_linear(**kw) == _lib.ERR_ALIGN


def test_empty_problems_touch_nothing():
    lib = _lib.load()
    assert run_linear(M=0, A=None, C=None) == _lib.OK
    assert run_linear(N=0, B=None, C=None) == _lib.OK
    assert lib.nvfp4_linear_run(None, None) == _lib.ERR_INVALID
    a = norm_args(rows=0, x=None)
    assert lib.nvfp4_block_norm_run(ctypes.byref(a), None) == _lib.OK
    # r is x and nothing else is asked for
    a = norm_args(Z=None)
    assert lib.nvfp4_block_norm_run(ctypes.byref(a), None) == _lib.OK


def run_grouped(rows, row0=None, groups=None, **kw):
    g = len(rows) if groups is None else groups
    r = (ctypes.c_int * max(len(rows), 1))(*rows)
    o = None if row0 is None else (ctypes.c_int * len(row0))(*row0)
    return _lib.load().nvfp4_linear_run_grouped(
        ctypes.byref(linear_args(**{"M": 512, **kw})), r, o, g, 0, None)


@pytest.mark.parametrize("rows,row0,word", [
    ([-1, 3], None, ">= 0"), ([3, 4], [0, 64], "128"),
    ([3, 4], [-128, 128], "128"), ([130, 4], [0, 128], "overlaps"),
    ([4, 4], [128, 0], "overlaps"), ([513], None, "past"),
    ([1, 1, 1, 1, 1], None, "past"), ([4, 129], [0, 384], "past"),
])
def test_linear_grouped_refuses_host_groups(rows, row0, word):
    assert run_grouped(rows, row0) == _lib.ERR_INVALID
    assert word in _lib.last_error()


def test_linear_grouped_refuses_counts_of_groups_and_residual():
    assert run_grouped([1], groups=0) == _lib.ERR_INVALID
    assert run_grouped([1] * 257) == _lib.ERR_INVALID
    assert "256" in _lib.last_error()
    assert run_grouped([1], residual=P, ldr=256) == _lib.ERR_INVALID
    assert run_grouped([0, 0]) == _lib.OK  # every group empty
    lib = _lib.load()
    assert lib.nvfp4_linear_run_grouped(ctypes.byref(linear_args()), None,
                                        None, 1, 1, None) == _lib.ERR_INVALID


def norm_args(**kw):
    a = dict(x=P, Z=P, ldx=64, ldy=64, ldr=64, ldz=64, rows=4, D=64,
             dtype=_lib.DTYPE_BF16, eps=1e-6, scale=1.0)
    a.update(kw)
    return _lib.BlockNormArgs(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(rows=-1), "rows"), (dict(D=60), "D %"), (dict(D=0), "D %"),
    (dict(D=32776), "32768"), (dict(dtype=7), "dtype"),
    (dict(w_dtype=_lib.DTYPE_F16), "weights"), (dict(kind=2), "norm"),
    (dict(eps=-1e-6), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(flags=1), "flag"), (dict(x=None), "x is NULL"),
    (dict(y=P), "R is required"), (dict(post=1), "need y"),
    (dict(gate=P, gate_rows=1), "need y"),
    (dict(y=P, R=P, gate=P, gate_rows=3), "divide"),
    (dict(y=P, R=P, gate=P, gate_rows=0), "divide"),
    (dict(codes=P), "together"), (dict(sf=P), "together"),
    (dict(D=72, ldx=72, ldz=72, codes=P, sf=P), "64"), (dict(ldx=56), "least"),
])
def test_block_norm_refuses(kw, word):
    a = norm_args(**kw)
    assert _lib.load().nvfp4_block_norm_run(ctypes.byref(a), None) == \
        _lib.ERR_INVALID
    assert word in _lib.last_error()


@pytest.mark.parametrize("kw", [
    dict(x=P + 8), dict(Z=P + 2), dict(weight=P + 4), dict(ldx=68),
    dict(y=P, R=P, ldr=65),
])
def test_block_norm_refuses_misaligned(kw):
    a = norm_args(**kw)
    assert _lib.load().nvfp4_block_norm_run(ctypes.byref(a), None) == \
        _lib.ERR_ALIGN


@pytest.mark.parametrize("sms", [2, 20, 132, 148])
@pytest.mark.parametrize("m,n,k", [(1, 8, 64), (1, 4096, 4096),
                                   (16, 4096, 14336), (333, 1480, 1344),
                                   (8192, 8192, 28672), (5, 72, 320)])
def test_plan_is_launchable(m, n, k, sms):
    for residual in (False, True):
        pl = dg.linear_plan(m, n, k, residual, num_sms=sms)
        assert pl["tokens"] in (32, 64, 128, 256)
        assert pl["split"] in (1, 2, 4, 8)
        block = 512 if pl["tokens"] <= 64 else 256
        assert pl["split"] <= -(-k // block)  # a K block for every CTA
        assert 1 <= pl["grid"] <= sms
        assert pl["grid"] % pl["split"] == 0
        if pl["tokens"] == 256:
            assert pl["grid"] % 2 == 0 and pl["split"] == 1


def test_plan_follows_the_flags():
    for flag, tokens in ((_lib.LINEAR_TOKENS32, 32),
                         (_lib.LINEAR_TOKENS64, 64),
                         (_lib.LINEAR_TOKENS128, 128),
                         (_lib.LINEAR_PAIR, 256)):
        for split in (1, 2, 4, 8):
            pl = dg.linear_plan(40, 256, 4096, False,
                                flag | _lib.linear_split(split))
            assert pl["tokens"] == tokens
            assert pl["split"] == (1 if tokens == 256 else split)
    with pytest.raises(ValueError):
        dg.linear_plan(4, 12, 64)


@pytest.mark.parametrize("kw", [
    dict(residual=P + 16, ldr=256),            # shifted within the rows
    dict(residual=P + 512, ldr=256),           # by a row
    dict(residual=P + 2 * 3 * 256, ldr=256),   # the last row
    dict(residual=P, ldr=264),                 # another pitch
    dict(ldc=504, residual=P + 512, ldr=504),  # rows that meet in a gap of N-8
    dict(ldc=1024, residual=P + 256, ldr=1024),
])
def test_linear_refuses_a_residual_that_overlaps_c_in_part(kw):
    assert run_linear(**kw) == _lib.ERR_INVALID
    assert "overlap" in _lib.last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(Z=P + 16), "Z must each"), (dict(Z=P + 128), "Z must each"),
    (dict(Z=P, ldz=128), "Z must each"),
    (dict(x=P + 4096, y=P, R=P + 128, Z=None), "Z must each"),
    (dict(x=P + 4096, y=P + 8192, R=P, Z=P), "one another"),
    (dict(x=P + 4096, y=P + 8192, R=P, Z=P + 384), "one another"),
    (dict(x=P, y=P + 8192, R=P, Z=None, gate=P + 384, gate_rows=1), "gate"),
    (dict(x=P + 4096, y=P + 8192, R=P + 4096, Z=P, gate=P - 384,
          gate_rows=4), "gate"),
])
def test_block_norm_refuses_outputs_that_overlap(kw, word):
    a = norm_args(**kw)
    assert _lib.load().nvfp4_block_norm_run(ctypes.byref(a), None) == \
        _lib.ERR_INVALID
    assert {"one another": "R and Z must not"}.get(word, word) in \
        _lib.last_error()


def test_plan_refuses_what_the_call_refuses():
    for flags in (3, 0x500, 1 << 12):
        with pytest.raises(ValueError):
            dg.linear_plan(4, 128, 256, flags=flags)
    with pytest.raises(ValueError):
        dg.linear_plan(4, 128, 256, flags=_lib.LINEAR_PAIR, num_sms=1)
    assert dg.linear_plan(4, 128, 256, num_sms=1)["grid"] == 1


@pytest.mark.parametrize("rows,row0,word", [
    ([-1], None, ">= 0"), ([5], [64], "128"), ([5], [-128], "128"),
    ([130, 4], [0, 128], "overlaps"), ([513], None, "past"),
])
def test_empty_grouped_problems_check_their_groups(rows, row0, word):
    assert run_grouped(rows, row0, N=0, B=None, C=None) == _lib.ERR_INVALID
    assert word in _lib.last_error()
    # (without rows of A, a group's reach past them comes before its overlap)
    assert run_grouped(rows, row0, M=0, A=None, C=None) == _lib.ERR_INVALID
    assert word in _lib.last_error() or "past" in _lib.last_error()


def test_grouped_rows_need_rows_of_a():
    empty = dict(M=0, A=None, C=None)
    assert run_grouped([5], **empty) == _lib.ERR_INVALID
    assert "past" in _lib.last_error()
    assert run_grouped([0, 0], [0, 0], **empty) == _lib.OK
    assert run_grouped([5], N=0, B=None, C=None) == _lib.OK


@pytest.mark.parametrize("counts", [
    [1.5], ["1"], "12", [2 ** 70], [2 ** 31], [[1, 2]], [None],
    torch.tensor([1.5]), torch.tensor([[1, 2]]),
])
def test_counts_that_are_no_integers_are_refused(counts):
    t = torch.zeros(4, 64, dtype=torch.uint8)
    for kw in (dict(group_rows=counts),
               dict(group_rows=[1], group_row0=counts)):
        with pytest.raises(ValueError, match="group_row.*32 bits"):
            dg.linear_grouped(t, t, t, t, t, **kw)


FAR = 1 << 20  # apart from every other operand of these tests


@pytest.mark.parametrize("where", [0, 512, 3 * 512 + 496, -16])
@pytest.mark.parametrize("name", ["A", "B", "SFA", "SFB", "bias",
                                  "row_scale"])
def test_linear_refuses_a_c_that_meets_its_inputs(name, where):
    c = 16 * FAR
    kw = dict(A=FAR, B=2 * FAR, SFA=3 * FAR, SFB=4 * FAR, bias=5 * FAR,
              row_scale=6 * FAR, C=c)
    kw[name] = c + where
    if name == "row_scale" and where < 0:
        kw[name] = c - 4  # its last row
    if name == "bias" and where == 0:
        kw.update(bias=c - 4, bias_dtype=_lib.DTYPE_F32)
    assert run_linear(**kw) == _lib.ERR_INVALID
    assert "C must not overlap " + name in _lib.last_error()


def test_linear_grouped_refuses_a_c_that_meets_a_later_groups_weights():
    c = 16 * FAR
    kw = dict(A=FAR, B=2 * FAR, SFA=3 * FAR, SFB=4 * FAR, bias=5 * FAR, C=c)
    for name, size in (("B", 256 * 64), ("SFB", 2 * 2 * 512),
                       ("bias", 256 * 4)):
        # two groups: the second one's last 16 bytes are C's first
        a = {**kw, name: c + 16 - 2 * size}
        assert run_grouped([1, 1], **a) == _lib.ERR_INVALID
        assert "C must not overlap " + name in _lib.last_error()


@pytest.mark.parametrize("out", ["R", "Z"])
@pytest.mark.parametrize("where", [0, 128, 384, -16])
@pytest.mark.parametrize("name", ["weight", "bias", "post_weight",
                                  "post_bias"])
def test_block_norm_refuses_outputs_over_its_weights(name, where, out):
    kw = dict(x=FAR, y=2 * FAR, R=3 * FAR, Z=4 * FAR, post=1)
    kw[name] = kw[out] + where
    a = norm_args(**kw)
    assert _lib.load().nvfp4_block_norm_run(ctypes.byref(a), None) == \
        _lib.ERR_INVALID
    assert name + " must not overlap" in _lib.last_error()


@pytest.mark.parametrize("out,size", [("codes", 4 * 32), ("sf", 512)])
@pytest.mark.parametrize("name", ["x", "y", "R", "Z", "weight", "bias",
                                  "post_weight", "post_bias", "gate"])
def test_block_norm_refuses_codes_over_anything_else(name, out, size):
    kw = dict(x=FAR, y=2 * FAR, R=3 * FAR, Z=4 * FAR, codes=5 * FAR,
              sf=6 * FAR, weight=7 * FAR, bias=8 * FAR, post_weight=9 * FAR,
              post_bias=10 * FAR, gate=11 * FAR, gate_rows=2, post=1)
    for at in (kw[name], kw[name] - size + 16):
        a = norm_args(**{**kw, out: at})
        assert _lib.load().nvfp4_block_norm_run(ctypes.byref(a), None) == \
            _lib.ERR_INVALID
        assert "codes and sf must not overlap" in _lib.last_error()
    a = norm_args(**{**kw, "sf": kw["codes"] + 112})
    assert _lib.load().nvfp4_block_norm_run(ctypes.byref(a), None) == \
        _lib.ERR_INVALID


@pytest.mark.parametrize("flags", [1 << 32, (1 << 32) + 1, -1, -(1 << 32)])
def test_flags_beyond_32_bits_are_refused(flags):
    for call in (lambda: dg.linear_plan(4, 128, 256, flags=flags),
                 lambda: dg.plan(128, 256, 512, flags),
                 lambda: dg.plan_work(128, 256, 512, 0, flags),
                 lambda: dg.grouped_workspace_size([4], 128, 256, flags)):
        with pytest.raises(ValueError, match="32 bits"):
            call()


def test_plan_refuses_sizes_beyond_32_bits():
    for size in ((4 + (1 << 32), 128, 256), (4, 128 + (1 << 32), 256),
                 (4, 128, 256 + (1 << 32))):
        with pytest.raises(ValueError):
            dg.linear_plan(*size)
    with pytest.raises(ValueError):
        dg.linear_plan(4, 128, 256, num_sms=148 + (1 << 32))


def test_plan_without_pairs_takes_other_tiles():
    for m, n, k in ((4096, 4096, 14336), (500, 8192, 7168), (2048, 2056, 2048)):
        assert dg.linear_plan(m, n, k)["tokens"] == 256
        pl = dg.linear_plan(m, n, k, flags=_lib.LINEAR_TEST_NO_PAIR)
        assert pl["tokens"] in (32, 64, 128) and 1 <= pl["grid"] <= 148
