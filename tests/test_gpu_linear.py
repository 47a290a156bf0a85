"""GPU tests of ``linear`` and ``linear_grouped`` against 64-bit products of
the values the operands stand for (tests/block_ref.py derives the tolerance):
every tile and split schedule, sizes around the tiles' and blocks' edges,
types, epilogues, strides, ragged groups from the host and the device, and
rows and columns that must stay as they were."""
import numpy as np
import pytest
import torch

import nvfp4_dual_gemm_b200 as dg
from nvfp4_dual_gemm_b200 import _lib
from tests.block_ref import (assert_linear, blocked, linear64, random_nvfp4)

pytestmark = pytest.mark.gpu

SYNC = _lib.FLAG_SYNC_CHECK
TILES = {"auto": 0, "t32": _lib.LINEAR_TOKENS32, "t64": _lib.LINEAR_TOKENS64,
         "t128": _lib.LINEAR_TOKENS128, "pair": _lib.LINEAR_PAIR}


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


class Problem:
    def __init__(self, m, n, k, seed, dtype=torch.float16, bias=None,
                 residual=False, row_scale=False):
        rng = np.random.default_rng(seed)
        ca, sa, self.a = random_nvfp4(m, k, rng)
        cb, sb, self.b = random_nvfp4(n, k, rng, 0x10, 0x24)
        self.A, self.SFA = dev(ca), dev(blocked(sa))
        self.B, self.SFB = dev(cb), dev(blocked(sb))
        self.kw, self.ref = {}, {}
        if bias is not None:
            t = dev(rng.standard_normal(n).astype(np.float32)).to(bias)
            self.kw["bias"], self.ref["bias"] = t, t.double().cpu().numpy()
        if residual:
            t = dev(rng.standard_normal((m, n)).astype(np.float32)).to(dtype)
            self.kw["residual"] = t
            self.ref["residual"] = t.double().cpu().numpy()
        if row_scale:
            t = dev(rng.random(m).astype(np.float32))
            self.kw["row_scale"] = t
            self.ref["row_scale"] = t.double().cpu().numpy()

    def run(self, C=None, flags=0, **kw):
        return dg.linear(self.A, self.B, self.SFA, self.SFB, C,
                         flags=flags | SYNC, **self.kw, **kw)

    def check(self, got, what="", act=None, alpha=1.0):
        want, err = linear64(self.a, self.b, act=act, alpha=alpha, **self.ref)
        assert_linear(got, want, err, what)


@pytest.mark.parametrize("split", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("tile", list(TILES))
@pytest.mark.parametrize("m,n,k", [(1, 8, 64), (33, 136, 2368),
                                   (130, 264, 2048)])
def test_every_schedule(m, n, k, tile, split):
    p = Problem(m, n, k, seed=m + n + k, residual=True, bias=torch.float32,
                row_scale=True)
    flags = TILES[tile] | (_lib.linear_split(split) if split else 0)
    p.check(p.run(flags=flags), f"{tile} split {split}")


@pytest.mark.parametrize("m", [1, 2, 5, 31, 32, 33, 63, 64, 65, 127, 128, 129,
                               255, 257, 500])
def test_rows(m):
    p = Problem(m, 200, 512, seed=m)
    p.check(p.run(), f"m {m}")
    p.check(p.run(flags=_lib.LINEAR_PAIR), f"pair, m {m}")


@pytest.mark.parametrize("n", [8, 16, 72, 120, 128, 136, 256, 1000])
@pytest.mark.parametrize("m", [3, 140])
def test_columns(m, n):
    p = Problem(m, n, 320, seed=n, residual=True)
    p.check(p.run(), f"n {n}")
    p.check(p.run(flags=_lib.LINEAR_PAIR), f"pair, n {n}")
    for split in (1, 2):
        p.check(p.run(flags=_lib.LINEAR_TOKENS128 | _lib.linear_split(split)),
                f"t128 split {split}, n {n}")


@pytest.mark.parametrize("k", [64, 128, 192, 256, 320, 448, 512, 1088, 4096])
@pytest.mark.parametrize("m", [1, 200])
def test_depth(m, k):
    p = Problem(m, 144, k, seed=k)
    p.check(p.run(), f"k {k}")
    p.check(p.run(flags=_lib.LINEAR_PAIR), f"pair, k {k}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu_tanh", "gelu"])
@pytest.mark.parametrize("m", [7, 150, 300])
def test_epilogue(m, act, dtype):
    p = Problem(m, 264, 384, seed=5, dtype=dtype, bias=dtype, residual=True,
                row_scale=True)
    got = p.run(dtype=dtype, activation=act, alpha=0.375,
                flags=_lib.LINEAR_PAIR if m == 300 else 0)
    p.check(got, f"{act}", act=act, alpha=0.375)


def test_many_tiles_per_cta():
    """Several tiles for each CTA: both accumulators, every ring phase."""
    p = Problem(700, 4360, 576, seed=9, residual=True)
    p.check(p.run(flags=_lib.LINEAR_TOKENS32 | _lib.linear_split(1)))
    p.check(p.run(flags=_lib.LINEAR_TOKENS128 | _lib.linear_split(1)))
    p = Problem(2100, 4360, 576, seed=10, residual=True, bias=torch.float32)
    p.check(p.run(flags=_lib.LINEAR_PAIR))


@pytest.mark.parametrize("tile", ["auto", "pair"])
def test_output_given_strided_and_in_place(tile):
    m, n, k = 45, 200, 256
    p = Problem(m, n, k, seed=3, residual=True)
    wide = torch.full((m, n + 56), float("nan"), dtype=torch.float16,
                      device="cuda")
    wide[:, 8:n + 8] = p.kw["residual"]
    view = wide[:, 8:n + 8]
    p.kw["residual"] = view
    out = p.run(C=view, flags=TILES[tile])  # residual and output are the same strided rows
    assert out.data_ptr() == view.data_ptr()
    p.check(view, "in place")
    assert torch.isnan(wide[:, :8]).all() and torch.isnan(wide[:, n + 8:]).all()


def test_same_bits_every_run():
    p = Problem(4, 512, 4096, seed=12, residual=True)
    first = p.run()
    for _ in range(5):
        assert torch.equal(first, p.run())


def test_other_stream_and_graph():
    p = Problem(9, 256, 1024, seed=4, residual=True)
    want = p.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = p.run()
    s.synchronize()
    assert torch.equal(got, want)
    C = torch.empty_like(want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dg.linear(p.A, p.B, p.SFA, p.SFB, C, **p.kw)
        dg.linear(p.A, p.B, p.SFA, p.SFB, C, **p.kw)
    for _ in range(3):
        C.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(C, want)


# ------------------------------------------------------------------ grouped
class Groups:
    def __init__(self, rows, n, k, seed, row0=None, cap=None):
        rng = np.random.default_rng(seed)
        self.rows = rows
        self.row0 = dg.group_offsets(rows) if row0 is None else row0
        R = max([r + (m + 127) // 128 * 128
                 for r, m in zip(self.row0, rows)] + [1])
        R = R if cap is None else cap
        ca, sa, self.a = random_nvfp4(R, k, rng)
        bs = [random_nvfp4(n, k, rng, 0x10, 0x24) for _ in rows]
        self.A, self.SFA = dev(ca), dev(blocked(sa))
        self.B = dev(np.stack([b[0] for b in bs])).permute(1, 2, 0)
        self.SFB = dev(np.concatenate([blocked(b[1]) for b in bs]))
        self.b = [b[2] for b in bs]
        self.bias = dev(rng.standard_normal((len(rows), n))
                        .astype(np.float32))
        self.w = dev(rng.random(R).astype(np.float32))
        self.C = torch.full((R, n), float("nan"), dtype=torch.bfloat16,
                            device="cuda")

    def run(self, rows, row0=None, flags=0, **kw):
        return dg.linear_grouped(self.A, self.B, self.SFA, self.SFB, self.C,
                                 rows, row0, bias=self.bias,
                                 activation="silu", row_scale=self.w,
                                 flags=flags | SYNC, **kw)

    def check(self, rows=None, row0=None):
        rows = self.rows if rows is None else rows
        row0 = self.row0 if row0 is None else row0
        covered = np.zeros(self.C.shape[0], bool)
        for g, (r, m) in enumerate(zip(row0, rows)):
            if m <= 0:
                continue
            s = slice(r, r + m)
            want, err = linear64(
                self.a[s], self.b[g], self.bias[g].double().cpu().numpy(),
                "silu", row_scale=self.w[s].double().cpu().numpy())
            assert_linear(self.C[s], want, err, f"group {g}")
            covered[s] = True
        rest = self.C[torch.from_numpy(~covered).cuda()]
        assert torch.isnan(rest).all()


ROWS = {"ragged": [0, 37, 128, 300, 5, 0], "ones": [1] * 9,
        "one": [129], "empty": [0, 0, 0], "many": [3, 0] * 60}


@pytest.mark.parametrize("where", ["host", "device"])
@pytest.mark.parametrize("tile", list(TILES))
@pytest.mark.parametrize("rows", list(ROWS))
def test_grouped(rows, tile, where):
    r = ROWS[rows]
    p = Groups(r, 200, 448, seed=len(r))
    given = r if where == "host" else torch.tensor(r, dtype=torch.int32,
                                                   device="cuda")
    p.run(given, flags=TILES[tile])
    p.check()


@pytest.mark.parametrize("where", ["host", "device"])
def test_grouped_given_first_rows(where):
    rows, row0 = [130, 0, 7, 128], [128, 0, 512, 640]
    p = Groups(rows, 136, 256, seed=8, row0=row0)
    if where == "host":
        p.run(torch.tensor(rows), row0)
    else:
        p.run(torch.tensor(rows, dtype=torch.int32, device="cuda"),
              torch.tensor(row0, dtype=torch.int32, device="cuda"))
    p.check()


def test_grouped_256_groups():
    rows = [(7 * g) % 5 for g in range(256)]
    p = Groups(rows, 64, 128, seed=1)
    p.run(torch.tensor(rows, dtype=torch.int32, device="cuda"))
    p.check()


def test_grouped_device_counts_out_of_place():
    """Counts that the host cannot check: negative, past the rows, first rows
    outside the matrix or off the 128 grid."""
    p = Groups([5, 100, 60, 9, 4], 72, 192, seed=6, cap=400)
    i32 = dict(dtype=torch.int32, device="cuda")
    p.run(torch.tensor([-3, 100, 2 ** 31 - 1, 9, 4], **i32))
    p.check([0, 100, 400 - 128, 0, 0], [0, 0, 128, 0, 0])
    p.C.fill_(float("nan"))
    p.run(torch.tensor([5, 100, 60, 9, 4], **i32),
          torch.tensor([-128, 128, 384, 512, 65], **i32))
    p.check([0, 100, 16, 0, 0], [0, 128, 384, 0, 0])


def test_grouped_replay_reads_new_counts():
    rows = [40, 0, 90]
    p = Groups(rows, 128, 256, seed=2, cap=512)
    counts = torch.tensor(rows, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dg.linear_grouped(p.A, p.B, p.SFA, p.SFB, p.C, counts, bias=p.bias,
                          activation="silu", row_scale=p.w)
    for new in ([40, 0, 90], [0, 200, 1], [0, 0, 0], [128, 128, 128]):
        counts.copy_(torch.tensor(new, dtype=torch.int32))
        p.C.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        p.check(new, dg.group_offsets(new))


@pytest.mark.parametrize("tile", ["t32", "t128", "pair"])
def test_residual_beside_c_in_one_matrix(tile):
    """C and residual as the halves of one matrix, either way round."""
    m, n, k = 300, 136, 320
    rng = np.random.default_rng(5)
    (a, sfa, _), (b, sfb, _) = (random_nvfp4(r, k, rng, 0x10, 0x24)
                                for r in (m, n))
    ops = (dev(a), dev(b), dev(blocked(sfa)), dev(blocked(sfb)))
    flags = {"t32": _lib.LINEAR_TOKENS32, "t128": _lib.LINEAR_TOKENS128,
             "pair": _lib.LINEAR_PAIR}[tile]
    both = torch.randn(m, 2 * n, device="cuda").half()
    halves = both[:, :n], both[:, n:]
    for c, r in (halves, halves[::-1]):
        keep = r.clone()
        want = dg.linear(*ops, residual=keep, flags=flags)
        got = dg.linear(*ops, c, residual=r, flags=flags)
        assert torch.equal(got, want) and torch.equal(r, keep)
    with pytest.raises(ValueError):
        dg.linear(*ops, both[:-1, :n], residual=both[1:, :n], flags=flags)
    with pytest.raises(ValueError):
        dg.linear(*ops, both[:, :n], residual=both[:, 8:n + 8], flags=flags)
