"""The decoder steps (include/urb_step.h) against their definitions in 64 bits.

Tolerances are derived per value, before any run: u = 2^-24 for an f32 rounding, a chain of n f32
additions of terms t_i is off by at most n * 2u * sum |t_i| (MFMA sums may truncate, hence 2u), and
the output's own rounding is half a step (BF16 2^-8, f32 2^-24, relative)."""

import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest

from urbilateria_amd import configs as C
from urbilateria_amd import native as N
from urbilateria_amd import synth

from .test_gpu_parity import _small_layer, moe_mod

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F32: U}
FMTS = {"bf16": C.FMT_BF16, "mxfp4": C.FMT_MXFP4, "mxfp8": C.FMT_MXFP8}


@pytest.fixture(scope="module", autouse=True)
def _gpu(require_gpu):
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()


def step():
    from urbilateria_amd import step as s
    return s


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _status(call):
    try:
        call()
    except N.UrbError as e:
        return e.status
    return N.OK


# ---- projections --------------------------------------------------------------------------------

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def _weight(fmt, rows, cols, g):
    """(data, scales, the matrix in f64) in the checkpoint layout, on the host."""
    if fmt == "bf16":
        w = (torch.randn(rows, cols, generator=g) * 0.05).to(BF16)
        return w, None, w.double()
    scales = torch.randint(117, 123, (rows, cols // 32), generator=g, dtype=torch.uint8)
    by = torch.exp2(scales.double() - 127).repeat_interleave(32, 1)
    if fmt == "mxfp4":
        data = torch.randint(0, 256, (rows, cols // 2), generator=g, dtype=torch.uint8)
        codes = torch.stack((data & 15, data >> 4), 2).view(rows, cols).long()
        v = E2M1[codes & 7] * torch.where(codes > 7, -1.0, 1.0)
    else:
        data = torch.randint(0, 256, (rows, cols), generator=g, dtype=torch.uint8)
        data = torch.where((data & 0x7F) == 0x7F, data - 1, data)   # no NaN codes
        v = data.view(torch.float8_e4m3fn).double()
    return data, scales, v * by


class Proj:
    """A projection with adapters of the given ranks, and its definition in 64 bits."""

    def __init__(self, fmt, rows, cols, max_tokens, dtype, out_dtype=None, ranks=(), seed=1,
                 max_rank=None, host=False):
        g = _gen(seed)
        self.g, self.cols, self.out_dtype = g, cols, out_dtype or dtype
        data, scales, self.w = _weight(fmt, rows, cols, g)
        up = lambda t: t if t is None or host else t.cuda()
        self.dtype = dtype
        self.p = step().AdaptedProjection(up(data), up(scales), FMTS[fmt], rows, cols, max_tokens,
                                          dtype, out_dtype, slots=len(ranks),
                                          max_rank=max_rank or max(ranks, default=0))
        self.adapters = {}
        for i, r in enumerate(ranks):
            if r:
                self.fill(i, r)

    def fill(self, slot, rank, scale=None, host=False):
        a = (torch.randn(rank, self.cols, generator=self.g) * self.cols ** -0.5).to(BF16)
        b = torch.randn(self.w.shape[0], rank, generator=self.g).to(BF16)
        scale = 0.5 + 0.25 * slot if scale is None else scale
        self.p.set_adapter(slot, a if host else a.cuda(), b if host else b.cuda(), scale)
        self.adapters[slot] = (a.double(), b.double(), float(np.float32(scale)))

    def rows_of(self, T, values="normal"):
        x = torch.randn(T, self.cols, generator=self.g)
        if values == "bf16":
            x = x.to(BF16).float()
        elif values == "wide":     # magnitudes 2^-30 .. 2^30
            x = x * torch.exp2(torch.randint(-30, 31, x.shape, generator=self.g).float())
        return x.to(self.dtype)

    def check(self, got, x, ids=None):
        x = x.cpu().double()
        want, size = x @ self.w.T, x.abs() @ self.w.abs().T
        # chains of cols / 32 MFMAs, their 32 terms and the split parts' sums
        chain = 2 * U * (self.cols / 32 + 64)
        off = chain * size
        for slot, (a, b, s) in self.adapters.items():
            at = torch.zeros(len(x), dtype=torch.bool) if ids is None else ids.cpu() == slot
            u, usize = x[at] @ a.T, x[at].abs() @ a.abs().T
            want[at] += s * (u @ b.T)
            # u's own chain; its planes (16 bits for BF16 outputs); the second product's chain
            planes = 2.0 ** -16 if self.out_dtype == BF16 else 0.0
            off[at] += abs(s) * ((chain + planes + 40 * U) * usize) @ b.abs().T
        tol = off + HALF_STEP[self.out_dtype] * (want.abs() + off)
        got = got.cpu().double()
        assert got.shape == want.shape and bool(torch.isfinite(got).all())
        bad = (got - want).abs() > tol
        assert not bool(bad.any()), (int(bad.sum()), float(((got - want).abs() / tol).max()),
                                     bad.nonzero()[:4].tolist())


def _mixed(T, slots, g, idle=0.3):
    ids = torch.randint(0, slots, (T,), generator=g, dtype=torch.int32)
    return torch.where(torch.rand(T, generator=g) < idle, torch.full_like(ids, -1), ids).cuda()


@pytest.mark.parametrize("fmt", sorted(FMTS))
@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (F32, F32), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 33, 64, 65, 130])
def test_projection_with_adapters(fmt, dtype, out, T):
    p = Proj(fmt, 208, 640, T, dtype, out, ranks=(16, 1, 7, 8, 33))
    x, ids = p.rows_of(T).cuda(), _mixed(T, 5, p.g)
    p.check(p.p.forward(x, ids), x, ids)


@pytest.mark.parametrize("rows,cols", [(16, 128), (32, 8192), (48, 32768), (1040, 256)])
@pytest.mark.parametrize("T", [1, 20, 200])
def test_projection_shapes(rows, cols, T):
    p = Proj("mxfp8", rows, cols, T, BF16, F32, ranks=(4, 64))
    x, ids = p.rows_of(T).cuda(), _mixed(T, 2, p.g)
    p.check(p.p.forward(x, ids), x, ids)


@pytest.mark.parametrize("rank", [1, 8, 9, 31, 32, 100, 256])
@pytest.mark.parametrize("out", [BF16, F32])
def test_adapter_ranks(rank, out):
    p = Proj("bf16", 96, 256, 40, BF16, out, ranks=(rank, 2), max_rank=256)
    x, ids = p.rows_of(40).cuda(), _mixed(40, 2, p.g, idle=0.0)
    p.check(p.p.forward(x, ids), x, ids)


@pytest.mark.parametrize("values", ["bf16", "wide"])
@pytest.mark.parametrize("T", [3, 150])
def test_f32_rows_keep_all_their_bits(values, T):
    p = Proj("mxfp4", 64, 512, T, F32, ranks=(12,))
    x, ids = p.rows_of(T, values).cuda(), _mixed(T, 1, p.g)
    p.check(p.p.forward(x, ids), x, ids)


@pytest.mark.parametrize("T,slots", [(1, 1), (40, 64), (700, 3), (1300, 40), (1300, 600)])
def test_many_rows_and_many_adapters(T, slots):
    # more rows than a scan takes at once; more slots than rows and fewer
    p = Proj("mxfp4", 320, 256, T, BF16, F32, ranks=tuple(1 + i % 5 for i in range(slots)))
    x = p.rows_of(T).cuda()
    for ids in (_mixed(T, slots, p.g), _mixed(T, slots, p.g).sort().values,
                torch.full((T,), slots - 1, dtype=torch.int32, device="cuda"),
                torch.full((T,), -1, dtype=torch.int32, device="cuda"), None):
        p.check(p.p.forward(x, ids), x, ids)


@pytest.mark.parametrize("fmt", sorted(FMTS))
@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("T,rank", [(1, 1), (1, 9), (1, 16), (1, 17), (1, 32), (1, 33), (2, 16), (2, 5),
                                    (2, 17), (3, 16)])
def test_single_tokens_of_low_rank(fmt, dtype, out, T, rank):
    # the sizes around which a tile computes its first products itself
    p = Proj(fmt, 80, 1152, T, dtype, out, ranks=(rank, max(1, rank // 2), rank, 0), max_rank=rank)
    x = p.rows_of(T).cuda()
    for ids in ([0, 1, 0], [2, 2, 1], [-1, 0, -1], [-1, -1, -1]):
        ids = torch.tensor(ids[:T], dtype=torch.int32, device="cuda")
        p.check(p.p.forward(x, ids), x, ids)
    y = torch.empty(T, 80, dtype=p.out_dtype, device="cuda")
    for bad in (3, 4):     # an empty slot, none
        ids = torch.tensor([bad, 0, 0][:T], dtype=torch.int32, device="cuda")
        p.p.forward_into(x, y, ids)
        assert _status(p.p.sync) == N.ERR_ARGUMENT
        p.check(y, x, torch.where(ids == bad, -1, ids))


@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("T,cols,rank", [(1, 256, 8), (1, 256, 24), (2, 256, 8), (3, 256, 20), (16, 512, 40),
                                         (40, 256, 24), (131, 384, 70), (40, 5120, 24), (131, 5248, 40),
                                         (1100, 256, 9)])
def test_adapters_that_cancel_the_matrix(dtype, out, T, cols, rank):
    # W = -scale B A but for one value per row: y is that column of x.  All values are whole numbers (and
    # halves), all sums below 2^24 of them, so nothing is rounded while A x keeps its 20 bits and more
    g = _gen(T + cols)
    rows, most = 208, 127 if cols <= 512 else 31
    whole = lambda *shape: torch.randint(1, most + 1, shape, generator=g).double()
    proj = step().AdaptedProjection
    a, x = whole(rank, cols), whole(T, cols)
    r, c = torch.randint(0, rank, (rows,), generator=g), torch.randint(0, cols, (rows,), generator=g)
    sign = torch.randint(0, 2, (rows,), generator=g).double() * 2 - 1
    b = torch.zeros(rows, rank, dtype=torch.float64)
    b[torch.arange(rows), r] = sign
    assert cols * most * most < 2 ** 24
    for scale in (1.0, -0.5):
        w = -scale * (b @ a)
        w[torch.arange(rows), c] += 1.0
        wb = w.to(BF16)
        assert torch.equal(wb.double(), w)
        p = proj(wb.cuda(), None, C.FMT_BF16, rows, cols, T, dtype, out, slots=3, max_rank=rank)
        p.set_adapter(1, a.to(BF16).cuda(), b.to(BF16).cuda(), scale)
        got = p.forward(x.to(dtype).cuda(), torch.ones(T, dtype=torch.int32, device="cuda"))
        assert torch.equal(got.cpu().double(), x[:, c])


def test_calls_longer_than_one_pass():
    T = 8192 + 77
    p = Proj("bf16", 16, 128, T, BF16, F32, ranks=(3, 2))
    x, ids = p.rows_of(T).cuda(), _mixed(T, 2, p.g)
    p.check(p.p.forward(x, ids), x, ids)


@pytest.mark.parametrize("fmt", sorted(FMTS))
@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("T,rows,cols", [(100, 784, 384), (90, 2064, 1152), (65, 272, 5120), (400, 528, 640),
                                         (512, 48, 5248), (513, 48, 5248)])
def test_tiles_of_every_height_and_slices_of_the_long_axis(fmt, dtype, out, T, rows, cols):
    # rows and columns that end inside a tile, few tiles and long sums, rows that share first products
    p = Proj(fmt, rows, cols, T, dtype, out, ranks=(24, 3, 40, 0), max_rank=48)
    x, ids = p.rows_of(T).cuda(), _mixed(T, 3, p.g)
    p.check(p.p.forward(x, ids), x, ids)
    p.check(p.p.forward(x[:T // 3], ids[:T // 3]), x[:T // 3], ids[:T // 3])
    p.check(p.p.forward(x), x)


def test_f32_rows_of_more_than_one_pass():
    T = 2048 + 40
    p = Proj("mxfp8", 144, 384, T, F32, ranks=(5, 17))
    x, ids = p.rows_of(T).cuda(), _mixed(T, 2, p.g)
    p.check(p.p.forward(x, ids), x, ids)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("stride", [(1 << 22) - 8, 1 << 22])
def test_rows_far_apart(dtype, stride):
    T, cols = 37, 256
    p = Proj("bf16", 80, cols, T, dtype, F32, ranks=(8, 9))
    x, ids = p.rows_of(T).cuda(), _mixed(T, 2, p.g)
    far = torch.empty((T - 1) * stride + cols, dtype=dtype, device="cuda").as_strided((T, cols), (stride, 1))
    far.copy_(x)
    p.check(p.p.forward(far, ids), x, ids)
    y = torch.empty((T - 1) * stride + 80, device="cuda").as_strided((T, 80), (stride, 1))
    p.p.forward_into(x, y, ids)
    p.p.sync()
    p.check(y, x, ids)


def test_many_rows_farther_apart_than_32_bit_offsets():
    T, cols, stride = 600, 128, (1 << 22) - 8
    p = Proj("bf16", 48, cols, T, BF16, F32, ranks=(8, 9, 20))
    x, ids = p.rows_of(T).cuda(), _mixed(T, 3, p.g)
    far = torch.empty((T - 1) * stride + cols, dtype=BF16, device="cuda").as_strided((T, cols), (stride, 1))
    far.copy_(x)
    p.check(p.p.forward(far, ids), x, ids)


def test_a_matrix_of_more_than_4_gib():
    rows, cols = 65536 + 64, 32768
    w = torch.randn(rows, cols, device="cuda", dtype=BF16,
                    generator=torch.Generator("cuda").manual_seed(1))
    some = list(range(16)) + list(range(rows - 64, rows))
    for T in (1, 18):
        proj = step().AdaptedProjection(w, None, C.FMT_BF16, rows, cols, T, BF16, F32, slots=2, max_rank=8)
        g = _gen(T)
        a = (torch.randn(8, cols, generator=g) * cols ** -0.5).to(BF16)
        b = torch.randn(rows, 8, generator=g).to(BF16)
        proj.set_adapter(1, a.cuda(), b.cuda(), 0.5)
        x = torch.randn(T, cols, generator=g).to(BF16)
        got = proj.forward(x.cuda(), torch.ones(T, dtype=torch.int32, device="cuda"))[:, some].cpu().double()
        xd, wd, bd = x.double(), w[some].cpu().double(), b[some].double()
        want = xd @ wd.T + 0.5 * (xd @ a.double().T) @ bd.T
        chain = 2 * U * (cols / 32 + 64)
        size = xd.abs() @ wd.abs().T + 0.5 * ((xd.abs() @ a.double().abs().T) @ bd.abs().T)
        # the chains of both products (u and the matrix), the second product's, the output's rounding
        assert bool(((got - want).abs() <= 2 * (chain + 40 * U) * size).all())
        del proj


def test_every_slot_there_is():
    p = Proj("bf16", 32, 128, 300, F32, ranks=(0,) * 4096, max_rank=4)
    for slot in (0, 1, 2047, 4094, 4095):
        p.fill(slot, 1 + slot % 4, scale=1.5)
    x = p.rows_of(300).cuda()
    ids = torch.tensor([0, 1, 2047, 4094, 4095, -1], dtype=torch.int32)
    ids = ids[torch.randint(0, 6, (300,), generator=p.g)].cuda()
    for T in (1, 3, 40, 300):
        p.check(p.p.forward(x[:T], ids[:T].contiguous()), x[:T], ids[:T])


@pytest.mark.parametrize("T,rows,cols,dtype", [(1, 64, 256, BF16), (12, 64, 1024, F32), (40, 272, 5120, F32),
                                               (200, 528, 1024, BF16), (200, 528, 5120, F32)])
def test_captured_projections_replay_on_new_inputs(T, rows, cols, dtype):
    # rows, ids and a slot's content change between the replays; eager calls of the context stand between
    p = Proj("mxfp4", rows, cols, T, dtype, F32, ranks=(16, 3, 20), max_rank=32)
    x, ids = p.rows_of(T).cuda(), _mixed(T, 3, p.g)
    y = torch.empty(T, rows, device="cuda")
    p.p.forward_into(x, y, ids)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        p.p.forward_into(x, y, ids)
    for i in range(4):
        x.copy_(p.rows_of(T))
        ids.copy_(_mixed(T, 3, p.g))
        p.fill(i % 3, 1 + 7 * i)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        p.check(y, x, ids)
        assert torch.equal(p.p.forward(x, ids), y)
    p.p.sync()


def test_projections_on_two_streams():
    both = [Proj("mxfp8", 784, 1152, 150, dtype, F32, ranks=(9, 30), seed=i)
            for i, dtype in enumerate((BF16, F32))]
    ins = [(p.rows_of(150).cuda(), _mixed(150, 2, p.g)) for p in both]
    outs = [torch.empty(150, 784, device="cuda") for _ in both]
    streams = [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()
    for _ in range(5):
        for p, (x, ids), y, s in zip(both, ins, outs, streams):
            with torch.cuda.stream(s):
                p.p.forward_into(x, y, ids)
    torch.cuda.synchronize()
    for p, (x, ids), y in zip(both, ins, outs):
        p.check(y, x, ids)
        p.p.sync()


def test_outputs_of_padded_rows_are_left():
    # a call over the first rows of a buffer writes nothing behind them
    p = Proj("bf16", 272, 640, 80, BF16, ranks=(8,))
    x = p.rows_of(80).cuda()
    for T in (1, 16, 17, 33, 64, 70):
        y = torch.full((80, 272), 5.0, dtype=BF16, device="cuda")
        ids = torch.zeros(80, dtype=torch.int32, device="cuda")
        ids[T:] = 99     # not read
        p.p.forward_into(x[:T], y[:T], ids[:T])
        p.p.sync()
        p.check(y[:T], x[:T], ids[:T])
        assert bool((y[T:] == 5.0).all())


@pytest.mark.parametrize("T", [5, 140])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strided_rows_and_outputs_leave_the_rest(T, dtype):
    p = Proj("bf16", 48, 256, T, dtype, ranks=(8, 8))
    wide = torch.randn(T, 256 + 8 + 16, generator=p.g).to(dtype).cuda()
    x, ids = wide[:, 8:264], _mixed(T, 2, p.g)
    for start in (0, 1, 8):    # outputs at any value
        y = torch.full((T + 1, 61), 7.0, dtype=dtype, device="cuda")
        p.p.forward_into(x, y[:T, start:start + 48], ids)
        p.p.sync()
        p.check(y[:T, start:start + 48], x, ids)
        rest = torch.ones_like(y, dtype=torch.bool)
        rest[:T, start:start + 48] = False
        assert bool((y[rest] == 7.0).all())


def test_a_row_of_infinities_touches_no_other():
    for dtype in (BF16, F32):
        p = Proj("bf16", 64, 256, 20, dtype, F32, ranks=(4, 4))
        x, ids = p.rows_of(20), _mixed(20, 2, p.g, idle=0.0)
        clean = p.p.forward(x.cuda(), ids)
        x[3, 7], x[9, 100], x[9, 101] = math.inf, math.nan, -math.inf
        got = p.p.forward(x.cuda(), ids)
        rows = [i for i in range(20) if i not in (3, 9)]
        assert torch.equal(got[rows], clean[rows])
        assert not bool(torch.isfinite(got[[3, 9]]).any())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [2, 12, 60, 140])
def test_infinities_among_rows_with_and_without_an_adapter(dtype, T):
    # few rows and tiles; adapters of the bad row, of others and none
    p = Proj("mxfp4", 272, 5120, T, dtype, ranks=(20, 4))
    x, ids = p.rows_of(T), _mixed(T, 2, p.g)
    clean = p.p.forward(x.cuda(), ids)
    for bad, value in ((0, math.inf), (T - 1, -math.inf), (T // 2, math.nan)):
        for id_ in (-1, 0, 1):
            ids[bad] = id_
            here = x.clone()
            here[bad, 4000] = 1.0
            want = p.p.forward(here.cuda(), ids)
            here[bad, 4000] = value
            got = p.p.forward(here.cuda(), ids)
            rows = [i for i in range(T) if i != bad]
            assert torch.equal(got[rows], want[rows])
            assert not bool(torch.isfinite(got[bad]).any())
    assert bool(torch.isfinite(clean).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,cols,rank", [(1, 256, 1), (1, 256, 9), (1, 256, 17), (2, 256, 7), (5, 256, 3), (40, 256, 20),
                                         (40, 5120, 20), (200, 384, 33), (1100, 128, 5)])
def test_infinite_values_stay_infinite_beside_padded_ranks(dtype, T, cols, rank):
    # all weights above zero: a row with an infinity is infinite, of its sign, not NaN
    g = _gen(T + rank)
    w = (torch.rand(80, cols, generator=g) + 0.5).to(BF16)
    a, b = ((torch.rand(s, generator=g) + 0.5).to(BF16) for s in ((rank, cols), (80, rank)))
    p = step().AdaptedProjection(w.cuda(), None, C.FMT_BF16, 80, cols, T, dtype, slots=2, max_rank=rank)
    p.set_adapter(1, a.cuda(), b.cuda(), 0.5)
    x = torch.rand(T, cols, generator=g)
    bad = {0: math.inf, T // 2: -math.inf, T - 1: math.inf}
    for t, v in bad.items():
        x[t, (37 * t + 5) % cols] = v
    for ids in (torch.ones(T, dtype=torch.int32), torch.arange(T, dtype=torch.int32) % 2 * 2 - 1):
        y = p.forward(x.to(dtype).cuda(), ids.cuda()).cpu()
        for t in range(T):
            if t in bad:
                assert bool((y[t] == bad[t]).all()), (t, y[t])
        assert bool(torch.isfinite(y[[t for t in range(T) if t not in bad]]).all())


def test_results_do_not_depend_on_the_other_rows():
    p = Proj("mxfp8", 64, 512, 16, BF16, F32, ranks=(8, 8, 8))
    x, ids = p.rows_of(16).cuda(), _mixed(16, 3, p.g)
    first = p.p.forward(x, ids)
    for _ in range(3):
        assert torch.equal(p.p.forward(x, ids), first)
    order = torch.randperm(16, generator=p.g).cuda()
    assert torch.equal(p.p.forward(x[order].contiguous(), ids[order].contiguous()), first[order])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [60, 200, 1300])
def test_tiles_give_a_row_the_same_among_any_others(T, dtype):
    p = Proj("bf16", 272, 5120, T, dtype, F32, ranks=(8, 40, 0, 17), max_rank=64)
    x, ids = p.rows_of(T).cuda(), _mixed(T, 4, p.g)
    ids[ids == 2] = 3
    x[::3] = x[::3].bfloat16().to(dtype)     # rows of one plane among rows of three
    first = p.p.forward(x, ids)
    p.check(first, x, ids)
    for _ in range(3):
        assert torch.equal(p.p.forward(x, ids), first)
        order = torch.randperm(T, generator=p.g).cuda()
        assert torch.equal(p.p.forward(x[order].contiguous(), ids[order].contiguous()), first[order])


def test_a_captured_slot_change_follows_its_source():
    p = Proj("mxfp8", 80, 256, 70, BF16, F32, ranks=(0, 4), max_rank=16)
    x, ids = p.rows_of(70).cuda(), _mixed(70, 2, p.g)
    ids[0] = 0
    a, b = torch.zeros(9, 256, dtype=BF16, device="cuda"), torch.zeros(80, 9, dtype=BF16, device="cuda")
    y = torch.empty(70, 80, device="cuda")
    p.p.set_adapter(0, a, b, 0.5)
    p.p.forward_into(x, y, ids)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        p.p.set_adapter(0, a, b, 0.5)
        p.p.forward_into(x, y, ids)
    for i in range(3):
        a.copy_(torch.randn(9, 256, generator=p.g) / 16)
        b.copy_(torch.randn(80, 9, generator=p.g))
        p.adapters[0] = (a.cpu().double(), b.cpu().double(), 0.5)
        graph.replay()
        p.p.sync()
        p.check(y, x, ids)
    b[3, 3] = math.inf          # the slot becomes empty, its rows W x alone
    graph.replay()
    assert _status(p.p.sync) == N.ERR_NONFINITE
    del p.adapters[0]
    p.check(y, x, ids)
    # (the rows that named the emptied slot had been latched with it)
    assert _status(p.p.sync) == N.OK


def test_slots_change_in_stream_order():
    p = Proj("bf16", 64, 256, 8, F32, ranks=(4, 6), max_rank=16)
    x = p.rows_of(8).cuda()
    ids = torch.tensor([0, 1, -1, 0, 1, 0, 1, -1], dtype=torch.int32, device="cuda")
    p.check(p.p.forward(x, ids), x, ids)
    y0, old = torch.empty(8, 64, device="cuda"), dict(p.adapters)
    p.p.forward_into(x, y0, ids)          # before the change, not waited for
    p.fill(1, 16, scale=-2.0)
    y1 = p.p.forward(x, ids)
    p.check(y1, x, ids)
    p.fill(0, 5, host=True)
    p.check(p.p.forward(x, ids), x, ids)
    p.adapters = old
    p.check(y0, x, ids)


def test_ids_without_an_adapter_are_reported_and_projected_alone():
    p = Proj("bf16", 64, 256, 6, F32, ranks=(4, 0), max_rank=8)
    x = p.rows_of(6).cuda()
    for bad in (1, 2, 2**31 - 1):
        ids = torch.tensor([0, bad, -1, -2**31, 0, -7], dtype=torch.int32, device="cuda")
        y = torch.empty(6, 64, device="cuda")
        p.p.forward_into(x, y, ids)
        assert _status(p.p.sync) == N.ERR_ARGUMENT
        assert _status(p.p.sync) == N.OK
        p.check(y, x, torch.where(ids == bad, -1, ids))
    p.p.clear_adapter(0)
    p.adapters = {}
    assert _status(lambda: p.p.forward(x, torch.zeros(6, dtype=torch.int32, device="cuda"))) \
        == N.ERR_ARGUMENT
    without = Proj("bf16", 64, 256, 6, F32)
    y = torch.empty(6, 64, device="cuda")
    without.p.forward_into(x, y, torch.zeros(6, dtype=torch.int32, device="cuda"))
    assert _status(without.p.sync) == N.ERR_ARGUMENT
    without.check(y, x)


@pytest.mark.parametrize("T", [16, 17, 64, 65, 200, 1024, 1025, 1300])
def test_ids_without_an_adapter_among_many_rows(T):
    p = Proj("bf16", 80, 256, T, BF16, F32, ranks=(4, 0, 20), max_rank=24)
    x = p.rows_of(T).cuda()
    for bad in (1, 3, 2**31 - 1):
        ids = _mixed(T, 3, p.g)
        ids[ids == 1] = 0
        assert _status(lambda: p.p.forward(x, ids)) == N.OK
        ids[torch.randint(0, T, (1 + T // 50,), generator=p.g).cuda()] = bad
        ids[T - 1] = -2**31
        ids[T // 2] = bad
        y = torch.empty(T, 80, device="cuda")
        p.p.forward_into(x, y, ids)
        assert _status(p.p.sync) == N.ERR_ARGUMENT and _status(p.p.sync) == N.OK
        p.check(y, x, torch.where(ids == bad, -1, ids))
    without = Proj("mxfp4", 80, 256, T, F32)
    x, y = without.rows_of(T).cuda(), torch.empty(T, 80, device="cuda")
    without.p.forward_into(x, y, torch.zeros(T, dtype=torch.int32, device="cuda"))
    assert _status(without.p.sync) == N.ERR_ARGUMENT
    without.check(y, x)
    without.p.forward_into(x, y, torch.full((T,), -3, dtype=torch.int32, device="cuda"))
    assert _status(without.p.sync) == N.OK
    without.check(y, x)


def test_projection_payloads_are_validated():
    w = torch.zeros(16, 128, dtype=BF16)
    w[3, 5] = math.inf
    make = lambda d, s, f: step().AdaptedProjection(d, s, f, 16, 128, 4, F32)
    assert _status(lambda: make(w.cuda(), None, C.FMT_BF16)) == N.ERR_NONFINITE
    assert _status(lambda: make(w, None, C.FMT_BF16)) == N.ERR_NONFINITE
    s = torch.full((16, 4), 127, dtype=torch.uint8)
    s[2, 1] = 255
    assert _status(lambda: make(torch.zeros(16, 64, dtype=torch.uint8).cuda(), s.cuda(),
                                C.FMT_MXFP4)) == N.ERR_INVALID_SCALE
    p = Proj("bf16", 16, 128, 4, F32, ranks=(2,))
    for where in "ab":
        a, b = torch.zeros(2, 128, dtype=BF16), torch.zeros(16, 2, dtype=BF16)
        (a if where == "a" else b)[1, 1] = math.nan
        p.p.set_adapter(0, a.cuda(), b.cuda())
        assert _status(p.p.sync) == N.ERR_NONFINITE
        x = p.rows_of(4).cuda()
        y = torch.empty(4, 16, device="cuda")
        p.p.forward_into(x, y, torch.zeros(4, dtype=torch.int32, device="cuda"))
        assert _status(p.p.sync) == N.ERR_ARGUMENT   # the slot is empty
        p.adapters = {}
        p.check(y, x)
    p.fill(0, 2)
    p.check(p.p.forward(x, torch.zeros(4, dtype=torch.int32, device="cuda")), x,
            torch.zeros(4, dtype=torch.int32))


def test_projection_refuses_calls():
    p = Proj("bf16", 64, 256, 4, F32, ranks=(4,))
    lib, ctx = N.moe_lib(), p.p._ctx
    x, y = torch.zeros(8, 256, device="cuda"), torch.zeros(8, 64, device="cuda")
    call = lambda T=4, xp=x.data_ptr(), xs=256, ys=64, yp=y.data_ptr(): lib.urb_proj_forward(
        ctx, xp, xs, None, T, yp, ys, None)
    assert call() == N.OK
    assert call(T=0) == call(T=5) == call(xs=252) == call(ys=63) == N.ERR_SHAPE
    assert call(xp=x.data_ptr() + 4) == call(xs=258) == call(yp=y.data_ptr() + 2) == N.ERR_ARGUMENT
    assert call(xp=None) == call(yp=None) == N.ERR_ARGUMENT
    a, b = torch.zeros(4, 256, dtype=BF16, device="cuda"), torch.zeros(64, 4, dtype=BF16, device="cuda")
    assert _status(lambda: p.p.set_adapter(1, a, b)) == N.ERR_SHAPE
    assert _status(lambda: p.p.set_adapter(0, a, b, math.inf)) == N.ERR_NONFINITE
    wide = Proj("bf16", 64, 256, 4, F32, ranks=(4,)).p
    big = torch.zeros(5, 256, dtype=BF16, device="cuda"), torch.zeros(64, 5, dtype=BF16, device="cuda")
    assert _status(lambda: wide.set_adapter(0, *big)) == N.ERR_SHAPE
    ad = N.Adapter(a.data_ptr(), b.data_ptr(), 4, 1.0)
    assert lib.urb_proj_set_adapter(ctx, 0, ctypes.byref(ad), N.SOURCE_DEVICE_BORROW, None) \
        == N.ERR_ARGUMENT
    for bad in (dict(x=x.half()), dict(x=x[:, ::2]), dict(y=y[:4]), dict(ids=[1, 2]),
                dict(ids=torch.zeros(8, dtype=torch.int64, device="cuda"))):
        with pytest.raises((ValueError, AttributeError)):
            p.p.forward_into(bad.get("x", x), bad.get("y", y), bad.get("ids"))
    with pytest.raises(ValueError):
        step().AdaptedProjection(torch.zeros(64, 255, dtype=BF16), None, 0, 64, 256, 4)
    torch.cuda.synchronize()


def test_adapters_and_matrices_on_another_device_are_refused(monkeypatch):
    # (a context of device 1: nothing is called that would read memory of device 0 there)
    p = Proj("bf16", 64, 256, 4, F32, ranks=(4,)).p
    a, b = torch.zeros(4, 256, dtype=BF16, device="cuda"), torch.zeros(64, 4, dtype=BF16, device="cuda")
    p.set_adapter(0, a, b)
    p.device = 1
    with pytest.raises(ValueError, match="cuda:1"):
        p.set_adapter(0, a, b)
    p.device = 0
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for source in (None, N.SOURCE_DEVICE_BORROW):
        with pytest.raises(ValueError, match="cuda:1"):
            step().AdaptedProjection(torch.zeros(64, 256, dtype=BF16, device="cuda"), None, C.FMT_BF16, 64, 256, 4,
                                     source=source)


def test_borrowed_panels_and_host_matrices_give_the_same():
    g = _gen(5)
    data, scales, _ = _weight("mxfp4", 64, 256, g)
    x = torch.randn(9, 256, generator=g).cuda()
    make = lambda d, s, src=None: step().AdaptedProjection(d, s, C.FMT_MXFP4, 64, 256, 9, F32,
                                                           source=src)
    want = make(data.cuda(), scales.cuda()).forward(x)
    pd, ps = moe_mod().pack_matrix(C.FMT_MXFP4, data.cuda(), scales.cuda(), 64, 256)
    torch.cuda.synchronize()
    borrowed = make(pd, ps, N.SOURCE_DEVICE_BORROW)
    assert torch.equal(borrowed.forward(x), want)
    assert torch.equal(make(data, scales).forward(x), want)
    assert borrowed.memory()[0] == 0 and make(data, scales).memory()[0] >= 64 * 256 // 2


@pytest.mark.parametrize("source", [N.SOURCE_DEVICE_COPY, N.SOURCE_DEVICE_BORROW])
def test_matrices_that_a_side_stream_still_writes(source):
    # creating waits for the matrix, whatever stream it comes from
    g = _gen(6)
    data, _, _ = _weight("bf16", 64, 256, g)
    x = torch.randn(9, 256, generator=g).cuda()
    make = lambda d, src=None: step().AdaptedProjection(d, None, C.FMT_BF16, 64, 256, 9, F32, source=src)
    want = make(data.cuda()).forward(x)
    ready = data.cuda()
    if source == N.SOURCE_DEVICE_BORROW:
        ready, _ = moe_mod().pack_matrix(C.FMT_BF16, ready, None, 64, 256)
    late, side = torch.full_like(ready.view(torch.uint8), 0xFF), torch.cuda.Stream()    # all NaN
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        late.copy_(ready.view(torch.uint8))
    assert torch.equal(make(late, source).forward(x), want)


# ---- norms and rotation ------------------------------------------------------------------------

def _turned(h, w, positions, freq, eps, zero_centered, interleaved):
    """(the definition in f64, the size its rounding errors are relative to)."""
    x = h.cpu().double()
    n = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * (w.cpu().double() + zero_centered)
    out, size = n.clone(), n.abs()
    r = 2 * freq.numel()
    if r:
        a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2),
                                                                     slice(r // 2, r))
        angle = torch.outer(positions.cpu().double(), freq.cpu().double()).unsqueeze(1)
        c, s = angle.cos(), angle.sin()
        out[..., a], out[..., b] = (n[..., a] * c - n[..., b] * s, n[..., b] * c + n[..., a] * s)
        both = n[..., a].abs() + n[..., b].abs()
        size[..., a], size[..., b] = both, both
    return out, size


def _check_turned(got, h, w, positions, freq, eps=1e-6, zero_centered=True, interleaved=False):
    want, size = _turned(h, w, positions, freq, eps, zero_centered, interleaved)
    # the row's sum (16 terms per lane and six steps of the tree; half of it after the root), the
    # mean, root, reciprocal, weight and products, cosine and sine and two FMAs: under 32 roundings
    tol = 32 * U * size + HALF_STEP[h.dtype] * want.abs() * (1 + 2.0 ** -10)
    bad = (got.cpu().double() - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())


def _freq(r):
    half = r // 2
    return (1e4 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))).float().cuda()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(64, 64), (128, 128), (256, 64), (80, 80), (80, 32), (96, 24),
                                 (2, 2), (34, 34), (34, 6), (192, 0), (1024, 1024), (16, 16),
                                 (576, 96), (112, 112)])
def test_heads_normed_and_turned(dtype, interleaved, D, R):
    g = _gen(D + R)
    for T, hq, hk in ((1, 1, 0), (1, 16, 2), (7, 5, 3), (130, 4, 1)):
        q, k = (torch.randn(T, h, D, generator=g).mul(3.0).to(dtype).cuda() for h in (hq, hk))
        wq, wk = (torch.randn(D, generator=g).mul(0.2).cuda() for _ in range(2))
        pos = torch.randint(0, 1 << 20, (T,), generator=g).cuda()
        qo, ko = step().qk_norm_rope(q, k if hk else None, wq, wk, pos, _freq(R), 1e-6,
                                     zero_centered=True, interleaved=interleaved)
        _check_turned(qo, q, wq, pos, _freq(R), interleaved=interleaved)
        if hk:
            _check_turned(ko, k, wk, pos, _freq(R), interleaved=interleaved)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_strided_heads_in_place_and_beside(dtype, shift):
    # heads of a fused q/k/v row, at any value of it; out of place, then in place
    g = _gen(3)
    T, hq, hk, D = 33, 6, 2, 64
    row = torch.randn(T, shift + (hq + 2 * hk) * D + 8, generator=g).to(dtype).cuda()
    q = row[:, shift:shift + hq * D].unflatten(1, (hq, D))
    k = row[:, shift + hq * D:shift + (hq + hk) * D].unflatten(1, (hk, D))
    w, pos = torch.rand(D, generator=g).cuda(), torch.arange(T).cuda() + 5000
    before, q0, k0 = row.clone(), q.clone(), k.clone()
    # head-major outputs
    qo, ko = (torch.empty(h, T, D, dtype=dtype, device="cuda").transpose(0, 1) for h in (hq, hk))
    call = lambda out: step().qk_norm_rope(q, k, w, w, pos, _freq(32), 1e-5, out=out)
    call((qo, ko))
    _check_turned(qo, q0, w, pos, _freq(32), 1e-5, False)
    _check_turned(ko, k0, w, pos, _freq(32), 1e-5, False)
    assert torch.equal(row, before)
    call((q, k))
    assert torch.equal(q, qo) and torch.equal(k, ko)
    rest = torch.ones_like(row, dtype=torch.bool)
    rest[:, shift:shift + (hq + hk) * D] = False
    assert torch.equal(row[rest], before[rest])


def test_angles_of_far_positions():
    D = 64
    h = torch.randn(5, 1, D, generator=_gen(1)).cuda()
    w = torch.ones(D, device="cuda")
    # exact products up to 2^29; the sign of a position turns the other way
    pos = torch.tensor([0, -1, (1 << 24) + 1, (1 << 29) - 1, -(1 << 28) - 3]).cuda()
    got, _ = step().qk_norm_rope(h, None, w, None, pos, _freq(D), 1e-6)
    _check_turned(got, h, w, pos, _freq(D), zero_centered=False)


def test_norms_alone():
    h, w = torch.randn(9, 3, 96, generator=_gen(16)).cuda(), torch.rand(96, device="cuda")
    got, none = step().qk_norm_rope(h, None, w, None, None, None, 1e-6)
    assert none is None
    _check_turned(got, h, w, torch.zeros(9), _freq(0), zero_centered=False)


def test_rotation_of_rows_with_zeros_and_nan():
    h = torch.randn(3, 2, 64, generator=_gen(2)).cuda()
    h[0] = 0.0
    h[1, 0, 5] = math.nan
    w, pos = torch.ones(64, device="cuda"), torch.arange(3).cuda()
    got, _ = step().qk_norm_rope(h, None, w, None, pos, _freq(64), 1e-6)
    assert bool((got[0] == 0).all()) and bool(got[1, 0].isnan().all())
    rest = torch.stack((h[1, 1], h[2, 0], h[2, 1])).unsqueeze(1)
    _check_turned(torch.stack((got[1, 1], got[2, 0], got[2, 1])).unsqueeze(1), rest, w,
                  torch.tensor([1, 2, 2]), _freq(64), zero_centered=False)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_same_heads_in_wide_and_in_single_steps(dtype):
    # aligned heads and the same ones off every boundary: two kernels, one definition
    g = _gen(13)
    T, H, D = 70, 3, 128
    h = torch.randn(T, H, D, generator=g).to(dtype).cuda()
    w, pos = torch.rand(D, generator=g).cuda(), torch.arange(T).cuda() * 1000
    odd = torch.empty(T, H * D + 3, dtype=dtype, device="cuda")[:, 1:1 + H * D].unflatten(1, (H, D))
    odd.copy_(h)
    for inter in (False, True):
        a, _ = step().qk_norm_rope(h, None, w, None, pos, _freq(64), 1e-6, interleaved=inter)
        b, _ = step().qk_norm_rope(odd, None, w, None, pos, _freq(64), 1e-6, interleaved=inter)
        for got in (a, b):
            _check_turned(got, h, w, pos, _freq(64), zero_centered=False, interleaved=inter)


def test_captured_rotation_replays_on_new_positions():
    g = _gen(14)
    q = torch.randn(1, 8, 128, generator=g).to(BF16).cuda()
    w, pos, freq = torch.rand(128, generator=g).cuda(), torch.tensor([5]).cuda(), _freq(64)
    out = torch.empty_like(q)
    call = lambda: step().qk_norm_rope(q, None, w, None, pos, freq, 1e-6, out=(out, None))
    call()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        call()
    for at in (6, 1000, 123456):
        q.copy_(torch.randn(1, 8, 128, generator=g))
        pos.fill_(at)
        graph.replay()
        torch.cuda.synchronize()
        _check_turned(out, q, w, pos, freq, zero_centered=False)


def test_heads_of_more_than_4_gib():
    # the last token's heads lie past 32-bit byte offsets, in a fused buffer
    T, H, D, row = 66000, 2, 64, 33000
    wide = torch.zeros(T, row, dtype=BF16, device="cuda")
    q = wide[:, :H * D].unflatten(1, (H, D))
    q.copy_(torch.randn(T, H, D, generator=_gen(15)))
    before, w, pos = q.clone(), torch.ones(D, device="cuda"), torch.arange(T).cuda()
    step().qk_norm_rope(q, None, w, None, pos, _freq(D), 1e-6, out=(q, None))
    some = [0, 1, 40000, 65999]
    _check_turned(q[some], before[some], w, pos[some], _freq(D), zero_centered=False)
    assert bool((wide[-1, H * D:] == 0).all())


@pytest.mark.parametrize("T,hq,hk,D,R,interleaved,start", [
    ((1 << 20) + 5, 60, 4, 2, 2, True, 0),          # single values
    (140000, 56, 8, 16, 16, False, 0), (140000, 62, 2, 16, 8, True, 0), (140000, 56, 8, 16, 16, False, 1),
    ((1 << 27) + 77, 1, 0, 16, 16, False, 0),
])
def test_more_head_rows_than_a_launch_holds(T, hq, hk, D, R, interleaved, start):
    # 2^23 head rows are a launch of either kernel; 2^26 of 64 threads, or 2^24 groups of 256, would be 2^32
    # threads, more than there may be
    g = torch.Generator("cuda").manual_seed(T)
    wide = torch.randn(T, start + (hq + hk) * D, dtype=BF16, device="cuda", generator=g)
    q = wide[:, start:start + hq * D].unflatten(1, (hq, D))
    k = wide[:, start + hq * D:].unflatten(1, (hk, D))
    wq, wk = (torch.rand(D, generator=_gen(i)).cuda() for i in (1, 2))
    pos = torch.arange(T, device="cuda") * 3 - T
    out = tuple(torch.full((T, h, D), math.nan, dtype=BF16, device="cuda") for h in (hq, hk))
    step().qk_norm_rope(q, k if hk else None, wq, wk, pos, _freq(R), 1e-6, interleaved=interleaved, out=out)
    assert all(bool(o.isfinite().all()) for o in out)
    per = (1 << 23) // (hq + hk)
    some = sorted({t for n in range(0, T, per) for t in (n - 1, n, n + 1) if 0 <= t < T} | {T // 2, T - 1})
    for o, h, w in ((out[0], q, wq), (out[1], k, wk)):
        if h.shape[1]:
            _check_turned(o[some], h[some], w, pos[some], _freq(R), zero_centered=False, interleaved=interleaved)


def test_outputs_that_overlap_themselves_are_refused():
    q, w = torch.zeros(4, 3, 64, device="cuda"), torch.ones(64, device="cuda")
    pos, buf = torch.arange(4).cuda(), torch.zeros(4 * 3 * 64, device="cuda")
    call = lambda strides, q=q: _status(lambda: step().qk_norm_rope(
        q, None, w, None, pos[:len(q)], _freq(64), 1e-6, out=(buf.as_strided(q.shape, strides), None)))
    for strides in ((192, 64, 1), (64, 256, 1)):
        assert call(strides) == N.OK
    for strides in ((0, 64, 1), (192, 0, 1), (191, 64, 1), (192, 63, 1), (64, 255, 1), (64, 64, 1), (63, 256, 1)):
        assert call(strides) == N.ERR_SHAPE
    assert call((0, 64, 1), q[:1]) == N.OK and call((64, 0, 1), q[:, :1]) == N.OK
    torch.cuda.synchronize()


def test_new_outputs_belong_to_the_stream_of_the_call():
    # memory that the current stream has freed but still writes is not handed to another stream
    g = _gen(18)
    T = 6000     # outputs of 12 MB, which the allocator keeps one by one
    q = torch.randn(T, 4, 128, generator=g).cuda()
    w, pos, side = torch.rand(128, generator=g).cuda(), torch.arange(T).cuda(), torch.cuda.Stream()
    freq = _freq(64)
    torch.cuda.synchronize()
    freed = [torch.empty_like(q) for _ in range(4)]
    torch.cuda._sleep(100_000_000)
    for t in freed:
        t.fill_(7.0)
    del freed, t
    got, got_k = step().qk_norm_rope(q, q, w, w, pos, freq, 1e-6, stream=side)
    torch.cuda.synchronize()
    for o in (got, got_k):
        _check_turned(o, q, w, pos, freq, zero_centered=False)


def test_rotation_wrapper_refuses():
    q, w = torch.zeros(2, 3, 64, device="cuda"), torch.ones(64, device="cuda")
    pos = torch.arange(2).cuda()
    call = lambda **c: step().qk_norm_rope(c.get("q", q), c.get("k"), c.get("w", w), w,
                                           c.get("pos", pos), _freq(64), 1e-6, out=c.get("out"))
    for c in (dict(q=q[0]), dict(k=q[:1]), dict(w=w[:32]), dict(w=w.double()), dict(pos=pos.int()),
              dict(out=(q[:, :2], None)), dict(q=q.transpose(1, 2)), dict(k=q.bfloat16())):
        with pytest.raises(ValueError):
            call(**c)
    assert _status(lambda: call(q=q.half())) == N.ERR_ARGUMENT


# ---- sampling ------------------------------------------------------------------------------------

def _drawn(row, tau=1.0, k=0, p=1.0, min_p=0.0, u=0.5):
    """(id, probability) by the definition: e in f64, its sums in whole multiples of 2^-shift.  (In
    f64 a sum of many ones loses the small masses that decide a border between equal tokens.)"""
    shift = min(51, 62 - math.ceil(math.log2(row.numel())))
    row = row.cpu().double().numpy()
    at = np.flatnonzero(row > -np.inf)
    if not at.size:
        return -1, 0.0
    order = at[np.lexsort((at, -row[at]))]
    if tau == 0:
        return int(order[0]), 1.0
    top = row[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        e = np.exp(np.where(row[order] == top, 0.0, (row[order] - top) / tau))
    q = np.floor(e * 2.0 ** shift + 0.5).astype(np.int64)
    n = min(k, e.size) if k > 0 else e.size
    if p < 1:
        mass = np.cumsum(q[:n])
        want = math.ceil(Fraction(p) * int(mass[-1]))
        n = 1 + int(np.searchsorted(mass[:-1], want, side="left"))
    n = max(1, min(n, int(np.count_nonzero(e >= min_p))))
    kept = np.argsort(order[:n])
    mass = np.cumsum(q[kept])
    target = math.floor(Fraction(u) * int(mass[-1]))
    i = int(np.searchsorted(mass, target, side="right"))
    return int(order[kept[i]]), float(e[kept[i]] / (int(mass[-1]) / 2.0 ** shift))


def _check_drawn(logits, uniform, sampler=None, **params):
    T, V = logits.shape
    sampler = sampler or step().Sampler(V, T, logits.dtype)
    names = {"tau": "temperature", "k": "top_k", "p": "top_p", "min_p": "min_p"}
    dev = {names[n]: torch.tensor(v, dtype=torch.int32 if n == "k" else F32).cuda()
           for n, v in params.items()}
    u = torch.tensor(uniform, dtype=F32).cuda()
    ids, probs = sampler.sample(logits, u, **dev)
    ids, probs, u = ids.tolist(), probs.tolist(), u.tolist()
    host = {n: dev[names[n]].tolist() for n in params}
    for t in range(T):
        id_, prob = _drawn(logits[t], u=u[t], **{n: host[n][t] for n in params})
        assert ids[t] == id_, (t, ids[t], id_, {n: host[n][t] for n in params}, u[t])
        # one rounding to f32, and sums that are exact to 2^-20 of it
        assert abs(probs[t] - prob) <= (U + 2.0 ** -40) * prob, (t, probs[t], prob)


def _logits(T, V, g, dtype=F32, spread=3.0):
    x = torch.randn(T, V, generator=g) * spread
    x[torch.rand(T, V, generator=g) < 0.05] = -math.inf
    return x.to(dtype).cuda()


GRID = [dict(), dict(tau=0.7), dict(tau=0.0), dict(k=1), dict(k=7), dict(k=300), dict(p=0.9),
        dict(p=0.2), dict(p=1e-9), dict(p=0.9999), dict(min_p=0.1), dict(min_p=1.0),
        dict(tau=1.7, k=40, p=0.8), dict(tau=0.5, k=500, p=0.95, min_p=0.02),
        dict(p=0.99, min_p=0.001), dict(tau=100.0, p=0.9), dict(tau=0.01), dict(k=20000, p=0.5)]


@pytest.mark.parametrize("V", [1, 2, 63, 64, 1000, 4097, 32000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_draws_under_every_filter(V, dtype):
    g = _gen(V)
    T = 3 * len(GRID)
    x = _logits(T, V, g, dtype)
    full = [dict(dict(tau=1.0, k=0, p=1.0, min_p=0.0), **d) for d in GRID for _ in range(3)]
    params = {n: [d[n] for d in full] for n in ("tau", "k", "p", "min_p")}
    _check_drawn(x, torch.rand(T, generator=g).tolist(), **params)


@pytest.mark.parametrize("V", [129280, 262144 + 3, 1 << 20])
def test_draws_from_large_vocabularies(V):
    g = _gen(V)
    x = _logits(6, V, g)
    _check_drawn(x, torch.rand(6, generator=g).tolist(), tau=[1.0, 0.8, 1.0, 2.0, 0.0, 1.0],
                 k=[0, 50, 0, 100000, 0, 3000], p=[1.0, 0.9, 0.95, 0.9, 1.0, 0.97],
                 min_p=[0.0, 0.0, 0.01, 0.0, 0.0, 0.0])


@pytest.mark.parametrize("V", [5, 900, 40000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_ties_go_to_the_lowest_index(V, dtype):
    g = _gen(V)
    same = torch.full((V,), 1.5)
    few = torch.randint(0, 3, (V,), generator=g).float()          # three values
    signed = torch.zeros(V)
    signed[::2] = -0.0                                            # equal to +0
    two = torch.where(torch.arange(V) % 2 == 0, 4.0, -30.0)
    rows = [same, few, signed, two]
    cases = [(r, k, p, u) for r in rows for k, p in ((0, 1.0), (3, 1.0), (0, 0.5), (V // 2 + 1, 0.7))
             for u in (0.0, 0.3, 1.0 - 2.0 ** -24)]
    x = torch.stack([c[0] for c in cases]).to(dtype).cuda()
    _check_drawn(x, [c[3] for c in cases], k=[c[1] for c in cases], p=[c[2] for c in cases])
    _check_drawn(x, [c[3] for c in cases], tau=[0.0] * len(cases))


@pytest.mark.parametrize("V", [3, 700, 33000])
def test_masked_rows(V):
    inf, nan, low = math.inf, math.nan, torch.finfo(F32).min
    base = torch.randn(V, generator=_gen(V))
    rows = []
    for change in ({0: -inf}, {0: nan}, {1: inf}, {1: inf, 2: inf}, {0: low, 1: low}, {0: nan, 1: -inf}):
        r = base.clone()
        for i, v in change.items():
            r[i] = v
        rows.append(r)
    rows += [torch.full((V,), v) for v in (-inf, nan, low, inf)]
    only = torch.full((V,), -inf)
    only[V - 1] = -5.0
    rows.append(only)
    x = torch.stack(rows).cuda()
    T = len(rows)
    for params in (dict(), dict(tau=[0.0] * T), dict(p=[0.9] * T), dict(k=[2] * T),
                   dict(k=[V - 1] * T, p=[0.5] * T, min_p=[0.3] * T)):
        for u in (0.0, 0.6, 1.0 - 2.0 ** -24):
            _check_drawn(x, [u] * T, **params)


def test_strided_and_unaligned_logits_and_extra_rows():
    g = _gen(8)
    for dtype in (BF16, F32):
        wide = _logits(9, 1003 + 5, g, dtype)
        sampler = step().Sampler(1003, 12, dtype)
        _check_drawn(wide[:, 3:1006], torch.rand(9, generator=g).tolist(), sampler, p=[0.9] * 9)
        _check_drawn(wide[:1, 1:1004], [0.4], sampler)
        _check_drawn(wide[::2, :1003], [0.1, 0.2, 0.3, 0.4, 0.5], sampler, k=[0, 1, 2, 30, 4000])


def test_more_rows_than_one_pass():
    g = _gen(21)
    T, V = 2 * 512 + 3, 1500
    x = _logits(T, V, g)
    pick = lambda values: [values[i % len(values)] for i in range(T)]
    _check_drawn(x, torch.rand(T, generator=g).tolist(), tau=pick([1.0, 0.0, 0.6]), k=pick([0, 5, 0, 70]),
                 p=pick([0.9, 1.0, 0.5, 0.99, 1.0]), min_p=pick([0.0, 0.05]))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [1025, 8192 * 3 + 5, 70001])
def test_crowded_bins_and_rows_off_the_boundary(V, dtype):
    # flat rows, whose cut lies among more tokens than a list holds, beside rows whose cut's bin alone
    # does, rows without a cut, and rows of one value; each from every start within 16 bytes
    g = _gen(V)
    near = lambda at, n: torch.cat((torch.full((n,), at), torch.full((V - n,), at - 8.0)))[
        torch.randperm(V, generator=g)]
    rows = [torch.randn(V, generator=g) * spread for spread in (1e-4, 0.02, 0.5, 6.0)]
    rows += [near(3.0, 5), near(3.0, 1024), near(3.0, min(V, 1030)), torch.full((V,), -2.0)]
    wide = torch.zeros(len(rows), V + 17, dtype=dtype, device="cuda")
    lists = [dict(p=0.5), dict(k=1000), dict(k=1024, p=0.7), dict(p=0.9, min_p=0.3), dict()]
    for start in range(0, 8, 3):
        view = wide[:, start:start + V]
        view.copy_(torch.stack(rows))
        for params in lists:
            _check_drawn(view, torch.rand(len(rows), generator=g).tolist(),
                         **{n: [v] * len(rows) for n, v in params.items()})


@pytest.mark.parametrize("T,V", [(1, 700), (3, 9000), (40, 33000)])
def test_captured_draws_replay_on_new_inputs(T, V):
    g = _gen(T)
    sampler = step().Sampler(V, T)
    x, u = _logits(T, V, g), torch.rand(T, generator=g).cuda()
    p = torch.full((T,), 0.9, device="cuda")
    ids, probs = torch.empty(T, dtype=torch.int32, device="cuda"), torch.empty(T, device="cuda")
    call = lambda: sampler.sample_into(x, u, ids, probs, top_p=p)
    call()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        call()
    for i in range(4):
        x.copy_(_logits(T, V, g))
        u.copy_(torch.rand(T, generator=g))
        p.fill_(0.3 + 0.2 * i)
        ids.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        got = ids.clone(), probs.clone()
        for t in range(T):
            id_, prob = _drawn(x[t], p=float(p[t]), u=float(u[t]))
            assert int(got[0][t]) == id_ and abs(float(got[1][t]) - prob) <= (U + 2.0 ** -40) * prob
        call()
        assert torch.equal(got[0], ids) and torch.equal(got[1], probs)
    sampler.sync()


def test_samplers_on_two_streams():
    g = _gen(31)
    both = [step().Sampler(40000, 20) for _ in range(2)]
    ins = [(_logits(20, 40000, g), torch.rand(20, generator=g).cuda()) for _ in both]
    p, tau = torch.full((20,), 0.8, device="cuda"), torch.full((20,), 0.7, device="cuda")
    outs = [(torch.empty(20, dtype=torch.int32, device="cuda"), torch.empty(20, device="cuda")) for _ in both]
    streams = [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()
    for _ in range(5):
        for sampler, (x, u), (ids, probs), s in zip(both, ins, outs, streams):
            with torch.cuda.stream(s):
                sampler.sample_into(x, u, ids, probs, top_p=p, temperature=tau)
    torch.cuda.synchronize()
    for (x, u), (ids, probs) in zip(ins, outs):
        for t in range(20):
            id_, prob = _drawn(x[t], tau=float(tau[t]), p=float(p[t]), u=float(u[t]))
            assert int(ids[t]) == id_ and abs(float(probs[t]) - prob) <= (U + 2.0 ** -40) * prob


@pytest.mark.parametrize("V", [65, 130, 700, 1024])
@pytest.mark.parametrize("kept", [1, 5, 33, 64])
def test_small_vocabularies_with_a_heavy_mask(V, kept):
    # at most 64 tokens left, spread over all the waves that hold the row: the first wave orders them
    # by itself while the others still take the row's largest logit
    g = _gen(V + kept)
    T = 512
    x = torch.full((T, V), -math.inf)
    for t in range(T):
        at = torch.randperm(V, generator=g)[:kept]
        x[t, at] = torch.randn(len(at), generator=g) * 2.0
    pick = lambda values: [values[i % len(values)] for i in range(T)]
    wide = torch.zeros(T, V + 9, device="cuda")
    for start in (0, 3):
        view = wide[:, start:start + V]
        view.copy_(x)
        _check_drawn(view, torch.rand(T, generator=g).tolist(), tau=pick([1.0, 0.6, 2.0]), k=pick([0, 3, 0, 40, 0]),
                     p=pick([1.0, 0.9, 0.5, 0.99]), min_p=pick([0.0, 0.0, 0.05]))


def test_draws_on_another_stream_are_waited_for():
    # behind work of that stream, and after what the current one still does to the inputs
    g = _gen(32)
    s, side = step().Sampler(700, 4), torch.cuda.Stream()
    x, u = _logits(4, 700, g), torch.rand(4, generator=g).cuda()
    want = s.sample(x, u)
    later, bad = torch.zeros_like(x), torch.full((4,), -1.0, device="cuda")
    torch.cuda.synchronize()
    for busy in (side, torch.cuda.current_stream()):
        later.zero_()
        with torch.cuda.stream(busy):
            torch.cuda._sleep(100_000_000)
        later.copy_(x)
        ids, probs = s.sample(later, u, stream=side)
        other = torch.cuda.Stream()
        with torch.cuda.stream(other):     # done: another stream may read them at once
            assert torch.equal(ids, want[0]) and torch.equal(probs, want[1])
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
    assert _status(lambda: s.sample(x, u, stream=side, temperature=bad)) == N.ERR_ARGUMENT
    assert _status(s.sync) == N.OK
    torch.cuda.synchronize()


def test_probabilities_may_be_left_out():
    g = _gen(22)
    for V in (700, 20000):
        s, x, u = step().Sampler(V, 5), _logits(5, V, g), torch.rand(5, generator=g).cuda()
        ids = torch.empty(5, dtype=torch.int32, device="cuda")
        s.sample_into(x, u, ids)
        s.sync()
        assert torch.equal(ids, s.sample(x, u)[0])


def test_rows_behind_the_last_are_left():
    s = step().Sampler(2000, 8)
    x, u = _logits(8, 2000, _gen(5)), torch.full((8,), 0.5, device="cuda")
    ids, probs = torch.full((8,), 77, dtype=torch.int32, device="cuda"), torch.full((8,), 7.0, device="cuda")
    s.sample_into(x[:3], u[:3], ids[:3], probs[:3])
    s.sync()
    assert bool((ids[3:] == 77).all()) and bool((probs[3:] == 7.0).all()) and bool((ids[:3] < 2000).all())


def test_logits_of_more_than_4_gib():
    V, T = 1 << 20, 1100
    x = torch.zeros(T, V, device="cuda")
    x[T - 1, V - 1] = x[T - 2, 12345] = x[0, 7] = 60.0
    ids, probs = step().Sampler(V, T).sample(x, torch.full((T,), 0.5, device="cuda"),
                                             temperature=torch.full((T,), 0.5, device="cuda"))
    assert [int(ids[i]) for i in (T - 1, T - 2, 0)] == [V - 1, 12345, 7]
    # the middle of a flat row: the smallest index i at which i + 1 > V / 2
    assert int(ids[1]) == V // 2 and bool((ids[1:T - 2] == V // 2).all())
    assert bool((probs[1:T - 2] == 1.0 / V).all()) and bool((probs[[0, T - 1]] == 1.0).all())


def test_extreme_temperatures():
    x = _logits(6, 500, _gen(4))
    _check_drawn(x, [0.9] * 6, tau=[1e-45, 1e-30, 1e30, 3e38, 1e-3, 1e3])


@pytest.mark.parametrize("V", [64, 3000])
def test_extreme_temperatures_of_extreme_logits(V):
    # differences that f32 cannot hold, and multiples of them that it cannot, of tokens with mass
    tiny, low, high = 2.0 ** -149, torch.finfo(F32).min, torch.finfo(F32).max
    g = _gen(V)
    small = tiny * torch.randint(-6, 7, (V,), generator=g)
    large = torch.where(torch.rand(V, generator=g) < 0.5, low, high)
    x = torch.stack((small, large, large.clone().fill_(low), small)).cuda()
    x[2, 5] = high
    for tau in ([tiny, 3e38, 3e38, 4 * tiny], [2e-38, 1.5e38, 2e30, 1e-30]):
        for u in (0.0, 0.4, 1.0 - 2.0 ** -24):
            _check_drawn(x, [u] * 4, tau=tau)
            _check_drawn(x, [u] * 4, tau=tau, p=[0.8, 0.9, 0.95, 0.5])
            _check_drawn(x, [u] * 4, tau=tau, k=[V - 1] * 4, min_p=[0.2, 0.1, 0.0, 0.5])


def test_parameters_out_of_range_are_reported():
    g = _gen(6)
    x = _logits(4, 300, g)
    s = step().Sampler(300, 4)
    good = dict(temperature=[1.0] * 4, top_p=[0.9] * 4, min_p=[0.0] * 4, uniform=[0.5] * 4)
    bad = dict(temperature=[-1.0, math.nan, math.inf], top_p=[0.0, -0.5, math.nan],
               min_p=[-0.1, 1.5, math.nan], uniform=[-0.1, 1.0, math.nan])
    for name, values in bad.items():
        for v in values:
            p = {n: torch.tensor([v if (n == name and t == 2) else q for t, q in enumerate(c)]).cuda()
                 for n, c in good.items()}
            u = p.pop("uniform")
            ids = torch.empty(4, dtype=torch.int32, device="cuda")
            probs = torch.empty(4, device="cuda")
            s.sample_into(x, u, ids, probs, **p)
            assert _status(s.sync) == N.ERR_ARGUMENT and _status(s.sync) == N.OK
            assert ids[2] == -1 and probs[2] == 0
            for t in (0, 1, 3):
                assert int(ids[t]) == _drawn(x[t], p=float(np.float32(0.9)))[0]


def test_sampler_refuses_calls():
    s = step().Sampler(300, 4)
    lib = N.moe_lib()
    x, v = torch.zeros(8, 300, device="cuda"), torch.zeros(8, dtype=torch.int32, device="cuda")
    u = torch.zeros(8, device="cuda")
    call = lambda rows=4, stride=300, at=0, uni=u.data_ptr(), ids=v.data_ptr(): lib.urb_sample(
        s._ctx, x.data_ptr() + at, stride, rows, None, uni, ids, None, None)
    assert call() == N.OK
    assert call(rows=0) == call(rows=5) == call(stride=299) == N.ERR_SHAPE
    assert call(at=2) == call(uni=None) == call(ids=None) == N.ERR_ARGUMENT
    with pytest.raises(ValueError):
        s.sample(x[:4].half(), u[:4])
    with pytest.raises(ValueError):
        s.sample(x[:4], u[:4], top_k=u[:4])
    torch.cuda.synchronize()


# ---- together, and under capture ----------------------------------------------------------------

class TokenStep:
    """A decoder's token step around one MoE block: fused q/k/v projection of the residual stream with
    adapters, norm and rotation of its heads, the block call, the vocabulary projection and the draw."""

    HQ, HK, D, V = 4, 2, 64, 1008

    def __init__(self, T):
        self.T, self.host = T, _small_layer("c1_bf16_decode")
        H = self.H = self.host.spec.hidden
        self.layer = moe_mod().MoeLayer(self.host, max_tokens=T)
        self.qkv = Proj("bf16", (self.HQ + 2 * self.HK) * self.D, H, T, F32, BF16, ranks=(8, 4), seed=2)
        self.head = Proj("mxfp8", self.V, H, T, F32, ranks=(8,), seed=3)
        self.sampler = step().Sampler(self.V, T)
        g = _gen(9)
        self.h = torch.empty(T, H, device="cuda")
        self.norm = torch.from_numpy(synth.activations("norm", 1, H)[0] * np.float32(0.1)).cuda()
        self.ids = torch.tensor([(t % 3) - 1 for t in range(T)], dtype=torch.int32, device="cuda")
        self.head_ids = torch.clamp(self.ids, max=0)
        self.w = torch.randn(self.D, generator=g).mul(0.1).cuda()
        self.pos = torch.randint(0, 100000, (T,), generator=g).cuda()
        self.u = torch.rand(T, generator=g).cuda()
        self.p = torch.full((T,), 0.9, device="cuda")
        self.freq = _freq(self.D)
        rows = (self.HQ + 2 * self.HK) * self.D
        self.out = dict(qkv=torch.empty(T, rows, dtype=BF16, device="cuda"),
                        block=torch.empty(T, H, device="cuda"),
                        logits=torch.empty(T, self.V, device="cuda"),
                        tokens=torch.empty(T, dtype=torch.int32, device="cuda"),
                        probs=torch.empty(T, device="cuda"))

    def heads(self):
        row, a, b = self.out["qkv"], self.HQ * self.D, (self.HQ + self.HK) * self.D
        return (row[:, :a].unflatten(1, (self.HQ, self.D)),
                row[:, a:b].unflatten(1, (self.HK, self.D)))

    def run(self):
        o = self.out
        s = torch.cuda.current_stream()
        self.qkv.p.forward_into(self.h, o["qkv"], self.ids)
        q, k = self.heads()
        step().qk_norm_rope(q, k, self.w, self.w, self.pos, self.freq, 1e-6,
                            zero_centered=True, out=(q, k))
        N.check(N.moe_lib().urb_moe_forward_block(
            self.layer._ctx, self.h.data_ptr(), self.norm.data_ptr(), 1e-6, self.T,
            o["block"].data_ptr(), None, None, s.cuda_stream or None), "block")
        self.head.p.forward_into(o["block"], o["logits"], self.head_ids)
        self.sampler.sample_into(o["logits"], self.u, o["tokens"], o["probs"], top_p=self.p)

    def results(self):
        torch.cuda.synchronize()
        for c in (self.qkv.p, self.head.p, self.sampler, self.layer):
            c.sync()
        return {n: t.clone() for n, t in self.out.items()}

    def check(self, got):
        # each step against its definition on the step before's output
        raw = self.qkv.p.forward(self.h, self.ids)
        self.qkv.check(raw, self.h, self.ids)
        a, b = self.HQ * self.D, (self.HQ + self.HK) * self.D
        for lo, hi, n in ((0, a, self.HQ), (a, b, self.HK)):
            _check_turned(got["qkv"][:, lo:hi].unflatten(1, (n, self.D)),
                          raw[:, lo:hi].unflatten(1, (n, self.D)), self.w, self.pos, _freq(self.D))
        assert torch.equal(got["qkv"][:, b:], raw[:, b:])
        block, _, _ = self.layer.forward_block(self.h, self.norm, 1e-6)
        assert torch.equal(got["block"], block)
        self.head.check(got["logits"], block, self.head_ids)
        for t in range(self.T):
            id_, prob = _drawn(got["logits"][t], p=float(self.p[t]), u=float(self.u[t]))
            assert int(got["tokens"][t]) == id_ and abs(float(got["probs"][t]) - prob) < 1e-6


@pytest.mark.parametrize("T", [1, 5, 40])
def test_a_token_step_around_the_block(T):
    run = TokenStep(T)
    run.h.copy_(torch.from_numpy(synth.activations("h", T, run.H)))
    run.run()
    run.check(run.results())


@pytest.mark.parametrize("T", [1, 21])
def test_a_captured_token_step_replays_on_new_inputs(T):
    run, other = TokenStep(T), TokenStep(T)
    inputs = [torch.from_numpy(synth.activations(f"h.{i}", T, run.H)).cuda() for i in range(4)]
    run.h.copy_(inputs[0])
    run.run()
    run.results()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        run.run()
    for x in inputs[1:]:
        for t in run.out.values():
            t.zero_()
        run.h.copy_(x)
        graph.replay()
        got = run.results()
        other.h.copy_(x)      # eager work of the same program between the replays
        other.run()
        want = other.results()
        for n in got:
            assert torch.equal(got[n], want[n]), n
    run.check(got)


def test_steps_on_a_stream_of_their_own():
    run, side = TokenStep(9), torch.cuda.Stream()
    x = torch.from_numpy(synth.activations("h.side", 9, run.H)).cuda()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run.h.copy_(x)
        run.run()
    side.synchronize()
    run.check(run.results())
