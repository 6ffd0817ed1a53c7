"""The paged cache (include/urb_cache.h) and beam search's selection against their definitions.

Whole numbers and copies are equal to those of plain loops.  Attention is held to 64 bits with a
tolerance per value, derived before any run: u = 2^-24 for an f32 rounding; a product over head_dim is a
chain of head_dim / 32 MFMAs of 32 terms, off by at most 2u (head_dim / 32 + 64) sum |q k| (MFMA sums may
truncate, hence 2u); the output's own rounding is half a step (BF16 2^-8, f32 2^-24, relative)."""

import math

import numpy as np
import pytest

from urbilateria_amd import native as N

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
BF16, F32, F8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
HALF_STEP = {BF16: 2.0 ** -8, F32: U}
NAN = float("nan")


@pytest.fixture(scope="module", autouse=True)
def _gpu(require_gpu):
    torch.cuda.set_device(0)
    yield
    torch.cuda.synchronize()


def cache_mod():
    from urbilateria_amd import cache
    return cache


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


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _same(got, want):
    got = got.cpu()
    want = torch.as_tensor(want).to(got.dtype).reshape(got.shape)
    assert torch.equal(got, want), (got != want).nonzero()[:5].tolist()


# ---- plans --------------------------------------------------------------------------------------

def _plan_by_hand(lengths, added, tables, free, count, page, pages, max_blocks, tokens):
    """(tables, lengths, starts, rows, positions, slots, count, status), row by row."""
    tables = [list(r) for r in tables]
    bits = set()
    if not 0 <= count <= pages:
        bits.add(N.ERR_ARGUMENT)
        count = 0
    out, starts, rows, positions, slots = [], [], [], [], []
    wanted, left = 0, count
    for r, (have, add) in enumerate(zip(lengths, added)):
        starts.append(min(len(rows), tokens))
        if have < 0 or add < 0 or have + add > max_blocks * page:
            bits.add(N.ERR_ARGUMENT)
            out.append(have)
            continue
        held, after = -(-have // page), -(-(have + add) // page)
        over = len(rows) + add > tokens
        if over:
            bits.add(N.ERR_ARGUMENT)
        need = 0 if over else after - held
        enough = need == 0 or wanted + need <= count
        if not enough:
            bits.add(N.ERR_OUT_OF_MEMORY)
        wanted += need
        served = enough and not over
        if served:
            for j in range(need):
                left -= 1
                tables[r][held + j] = free[left]
        out.append(have + add if served else have)
        for i in range(have, have + add):
            rows.append(r)
            positions.append(i)
            entry = tables[r][i // page] if served else -1
            if served and not 0 <= entry < pages:
                bits.add(N.ERR_ARGUMENT)
                entry = -1
            slots.append(entry * page + i % page if entry >= 0 else -1)
    starts.append(min(len(rows), tokens))
    pad = tokens - len(rows)
    fill = lambda v, x: (v + [x] * pad)[:tokens]
    status = N.ERR_ARGUMENT if N.ERR_ARGUMENT in bits else (
        N.ERR_OUT_OF_MEMORY if bits else N.OK)
    return (tables, out, starts, fill(rows, -1), fill(positions, 0), fill(slots, -1), left, status)


class Steps:
    """Random rows of a pager, with tables that lie in a wider buffer."""

    def __init__(self, rows, page, max_blocks, most, seed, room=None, spare=10, tokens=None, idle=0.3):
        g = np.random.default_rng(seed)
        self.rows, self.page, self.max_blocks = rows, page, max_blocks
        top = max_blocks * page
        self.added = np.where(g.random(rows) < idle, 0, g.integers(0, most + 1, rows))
        self.lengths = np.maximum(g.integers(0, top + 1, rows) - self.added, 0)
        self.added = np.minimum(self.added, top - self.lengths)
        held = -(-self.lengths // page)
        need = -(-(self.lengths + self.added) // page) - held
        self.pages = int(held.sum() + need.sum()) + spare
        ids = g.permutation(self.pages)
        self.tables = np.full((rows, max_blocks), -7)
        at = 0
        for r in range(rows):
            self.tables[r, :held[r]] = ids[at:at + held[r]]
            at += held[r]
        self.count = int(need.sum()) + spare if room is None else room
        self.free = np.full(self.pages, -9)
        self.free[:self.count] = ids[at:at + self.count]
        self.tokens = int(self.added.sum()) + 5 if tokens is None else tokens

    def check(self, in_place=False, optional=True, added=True):
        P = cache_mod().Pager(self.pages, self.page, self.rows, self.max_blocks, self.tokens + 3)
        wide = torch.full((self.rows, self.max_blocks + 3), -5, dtype=torch.int32, device="cuda")
        tables = wide[:, 1:-2]
        tables.copy_(torch.from_numpy(self.tables))
        lengths, free, count = _i32(self.lengths), _i32(self.free), _i32([self.count])
        plan = P.new_plan(self.rows, self.tokens)
        if in_place:
            plan.lengths, plan.count = lengths, count
        if not optional:
            plan.starts = plan.rows = plan.positions = None
        steps = self.added if added else np.ones_like(self.added)
        want = _plan_by_hand(self.lengths.tolist(), steps.tolist(), self.tables.tolist(),
                             self.free.tolist(), self.count, self.page, self.pages, self.max_blocks,
                             self.tokens)
        P.plan_into(lengths, _i32(self.added) if added else None, tables, free, count, plan)
        assert _status(P.sync) == want[7]
        _same(tables, want[0])
        _same(plan.lengths, want[1])
        _same(plan.slots, want[5])
        _same(plan.count, [want[6]])
        if optional:
            _same(plan.starts, want[2])
            _same(plan.rows, want[3])
            _same(plan.positions, want[4])
        assert bool((wide[:, 0] == -5).all()) and bool((wide[:, -2:] == -5).all())
        assert _status(P.sync) == N.OK
        return want


@pytest.mark.parametrize("rows,page,max_blocks,most", [
    (1, 16, 4, 1), (1, 1, 3, 2), (3, 7, 5, 9), (200, 16, 40, 1), (1000, 3, 20, 4), (1024, 16, 8, 3),
    (1025, 16, 8, 3), (3000, 64, 6, 100), (2100, 1, 50, 30), (17, 1024, 3, 2000)])
def test_plans(rows, page, max_blocks, most):
    for seed in (1, 2):
        assert Steps(rows, page, max_blocks, most, seed).check()[7] == N.OK
    Steps(rows, page, max_blocks, most, 3).check(in_place=True, optional=False)


def test_plans_of_one_token_each():
    s = Steps(300, 16, 9, 0, 4)
    s.lengths = np.minimum(s.lengths, 9 * 16 - 1)
    s.count = len(s.free)      # entries past the filled ones are no pages
    assert s.check(added=False)[7] in (N.OK, N.ERR_ARGUMENT)


@pytest.mark.parametrize("rows,page", [(1, 1), (300, 16), (300, 1), (1024, 7), (2000, 4)])
def test_plans_of_one_token_each_take_pages(rows, page):
    s = Steps(rows, page, 9, 1, 5, idle=0.0)
    s.lengths = np.arange(rows) % (9 * page)        # every place in a page, and whole pages, among them
    s.added[:] = 1
    held, need = -(-s.lengths // page), -(-(s.lengths + 1) // page)
    s.pages, s.count = int(need.sum()) + 3, int((need - held).sum()) + 3
    assert s.count > 3
    ids, at = np.random.default_rng(6).permutation(s.pages), 0
    s.tables[:] = -7
    for r in range(rows):
        s.tables[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    s.free = np.full(s.pages, -9)
    s.free[:s.count] = ids[at:]
    s.tokens = rows + 2
    want = s.check(added=False)
    assert want[7] == N.OK and want[6] == 3 and want[5].count(-1) == 2
    s.check(in_place=True, added=False)


def test_plans_with_many_rows_that_bring_nothing():
    s = Steps(9000, 16, 4, 3, 5, idle=0.95, tokens=6000)
    assert s.check()[7] == N.OK


@pytest.mark.parametrize("room", [0, 1, 7, 30])
@pytest.mark.parametrize("rows", [60, 1500])
def test_plans_without_enough_pages(rows, room):
    s = Steps(rows, 4, 12, 9, 6, room=room)
    assert s.check()[7] == N.ERR_OUT_OF_MEMORY
    s.check(in_place=True)


@pytest.mark.parametrize("tokens", [1, 40, 5000])
def test_plans_of_more_tokens_than_the_step_has(tokens):
    s = Steps(1300, 16, 10, 12, 7, tokens=tokens)
    assert s.check()[7] == N.ERR_ARGUMENT


def test_plans_of_rows_that_cannot_be():
    for rows in (50, 1100):
        s = Steps(rows, 16, 10, 12, 8)
        s.lengths[3], s.lengths[7], s.added[9] = -1, 161, -4
        s.lengths[11], s.added[11] = 150, 11
        s.lengths[12] = 2 ** 31 - 1
        s.lengths[13], s.added[13] = 5, 2 ** 31 - 1
        s.lengths[20], s.added[20], s.tables[20, 2] = 40, 3, s.pages      # a page that is none
        s.free[s.count - 2] = -3
        s.tokens = 12 * rows
        assert s.check()[7] == N.ERR_ARGUMENT


@pytest.mark.parametrize("count", [-1, 10 ** 6])
def test_plans_with_a_count_out_of_range(count):
    s = Steps(20, 16, 10, 12, 9)
    s.count = count
    assert s.check()[7] == N.ERR_ARGUMENT


def test_captured_plans_go_on_from_step_to_step():
    rows, page, blocks = 9, 4, 30
    P = cache_mod().Pager(400, page, rows, blocks, 64)
    free, count = P.new_stack()
    lengths = _i32([0, 1, 3, 4, 5, 7, 8, 9, 11])
    tables = torch.full((rows, blocks), -1, dtype=torch.int32, device="cuda")
    first = P.plan(torch.zeros_like(lengths), lengths, tables, free, count, 64)
    count.copy_(first.count)
    plan = P.new_plan(rows, 64)
    plan.lengths, plan.count = lengths, count
    added = torch.zeros_like(lengths)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        P.plan_into(lengths, added, tables, free, count, plan)
    for i in range(5):
        some = [(i * r) % 5 for r in range(rows)]
        added.copy_(_i32(some))
        want = _plan_by_hand(lengths.tolist(), some, tables.tolist(), free.tolist(), count.item(), page, 400,
                             blocks, 64)
        graph.replay()
        P.sync()
        for got, w in zip((tables, lengths, plan.starts, plan.rows, plan.positions, plan.slots, count), want):
            _same(got, w)


# ---- appends ------------------------------------------------------------------------------------

LAYOUTS = {   # how [pages, heads, page, dim] lies in memory
    "pages": lambda n, h, p, d, t: torch.zeros(n, h, p, d, dtype=t, device="cuda"),
    "tokens": lambda n, h, p, d, t: torch.zeros(n, p, h, d, dtype=t, device="cuda").transpose(1, 2),
    "padded": lambda n, h, p, d, t: torch.zeros(n, h, p, d + 16, dtype=t, device="cuda")[..., :d],
    "heads": lambda n, h, p, d, t: torch.zeros(h, n, p, d, dtype=t, device="cuda").transpose(0, 1),
}


def _make_cache(pages, heads, page, dim, dtype, layout="pages"):
    raw = torch.uint8 if dtype == F8 else dtype
    k, v = (LAYOUTS[layout](pages, heads, page, dim, raw).view(dtype) for _ in range(2))
    if dtype != F8:
        return cache_mod().PagedCache(k, v)
    return cache_mod().PagedCache(k, v, *(torch.full((pages, heads, page), 127, dtype=torch.uint8,
                                                     device="cuda") for _ in range(2)))


def _bits(t):
    return t.contiguous().view(torch.uint8 if t.dtype == F8 else torch.int16 if t.dtype == BF16
                               else torch.int32).cpu()


def _quantized(x):
    """(codes, scale exponents + 127) of rows x in f64."""
    x = x.double()
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    fine = torch.where(bad, 1.0, top)
    e = torch.ceil(torch.log2((fine / 448).clamp(min=2.0 ** -100)))
    e = torch.where(448 * torch.exp2(e - 1) >= fine.clamp(min=448 * 2.0 ** -100), e - 1, e)  # log2's rounding
    e = torch.where(448 * torch.exp2(e) < fine, e + 1, e).clamp(min=-100)
    codes = (torch.where(bad.unsqueeze(-1), 0.0, x) * torch.exp2(-e).unsqueeze(-1)).float().to(F8)
    codes = torch.where(bad.unsqueeze(-1), torch.full_like(codes.view(torch.uint8), 0x7f),
                        codes.view(torch.uint8))
    return codes, torch.where(bad, 127, e + 127).to(torch.uint8)


@pytest.mark.parametrize("layout", sorted(LAYOUTS))
@pytest.mark.parametrize("dtype,rows", [(BF16, BF16), (BF16, F32), (F8, BF16), (F8, F32)])
@pytest.mark.parametrize("T,heads,dim,page", [(1, 1, 16, 1), (5, 3, 80, 7), (70, 8, 128, 16), (33, 2, 256, 24),
                                              (300, 5, 48, 64)])
def test_appends(layout, dtype, rows, T, heads, dim, page):
    g = _gen(T + dim)
    pages = T // page + 9
    c = _make_cache(pages, heads, page, dim, dtype, layout)
    was = [_bits(t).clone() for t in (c.k, c.v)]
    qkv = (torch.randn(T, 4 * heads * dim, generator=g) * 3).to(rows).cuda()
    k = qkv[:, heads * dim:2 * heads * dim].unflatten(1, (heads, dim))
    v = qkv[:, 3 * heads * dim:].unflatten(1, (heads, dim))
    slots = torch.randperm(pages * page, generator=g)[:T]
    slots[torch.rand(T, generator=g) < 0.1] = -1
    if T > 4:
        slots[:4] = torch.tensor([pages * page, -5, 1 << 40, -(1 << 63)])
    c.append(k, v, slots.cuda())
    torch.cuda.synchronize()
    real = (slots >= 0) & (slots < pages * page)
    p, at = slots[real] // page, slots[real] % page
    for t, x, old, scales in ((c.k, k, was[0], c.k_scales), (c.v, v, was[1], c.v_scales)):
        x = x.cpu()[real]
        if dtype == F8:
            codes, e = _quantized(x)
            old[p, :, at] = codes
            want = torch.full((pages, heads, page), 127, dtype=torch.uint8)
            want[p, :, at] = e
            _same(scales, want)
        else:
            old[p, :, at] = x.to(BF16).view(torch.int16)
        if dtype == F8:   # a zero's sign is not part of the definition
            a, b = _bits(t), old
            assert torch.equal(torch.where(a == 128, 0, a), torch.where(b == 128, 0, b))
        else:
            assert torch.equal(_bits(t), old)


@pytest.mark.parametrize("rows", [BF16, F32])
def test_quantized_rows_at_the_ends_of_the_range(rows):
    values = [0.0, 1e-45, 1e-38, 3e-31, 448 * 2.0 ** -100, 448 * 2.0 ** -99, 1e-20, 448.0, 449.0, 447.0, 1.75,
              1.7500001, 1.76, 3.3e38, -3.3e38, math.inf, -math.inf, NAN]
    g = _gen(1)
    x = torch.randn(len(values), 1, 64, generator=g)
    for i, top in enumerate(values):
        x[i] = x[i].clamp(-1, 1) * (top if math.isfinite(top) else 1.0)
        x[i, 0, 5 * i % 64] = top
    x = x.to(rows)
    c = _make_cache(2, 1, 16, 64, F8)
    c.append(x.cuda(), x.cuda(), torch.arange(len(values), device="cuda"))
    codes, e = _quantized(x)
    n = len(values)
    got = _bits(c.k).view(32, 64)[:n]
    got, codes = (torch.where(t == 128, 0, t) for t in (got, codes[:, 0]))
    # (f32 rows below 2^-126 are subnormal; their products with 2^100 are exact all the same)
    assert torch.equal(got, codes)
    _same(c.k_scales.view(-1)[:n], e[:, 0])
    _same(c.v_scales.view(-1)[:n], e[:, 0])
    assert bool(torch.isnan(c.v.view(32, 64)[15:18].float()).all())


def test_appends_of_many_heads_in_several_launches():
    # 2^26 / 1024 = 65536 tokens of a launch
    T, heads = 65536 + 3, 1024
    c = _make_cache(1, heads, 8, 16, BF16)
    base = torch.arange(16, device="cuda", dtype=torch.float32)
    x = base.to(BF16).expand(T, heads, 16)
    slots = torch.full((T,), -1, device="cuda")
    slots[0], slots[65535], slots[65536], slots[T - 1] = 0, 3, 4, 7
    c.append(x, x, slots)
    want = torch.zeros(8, 16)
    want[[0, 3, 4, 7]] = base.cpu()
    for t in (c.k, c.v):
        assert torch.equal(t[0].float().cpu(), want.expand(heads, 8, 16))


@pytest.mark.parametrize("dtype", [BF16, F8])
def test_a_caches_tensors_stay(dtype):
    c = _make_cache(2, 1, 4, 16, dtype)
    for name in ("k", "v", "k_scales", "v_scales", "heads", "dtype"):
        was = getattr(c, name)
        with pytest.raises(AttributeError):
            setattr(c, name, None if was is None else was.clone() if torch.is_tensor(was) else was)
        assert getattr(c, name) is was
    for c.layer in (1, 2):     # what is not the cache's own
        pass


# ---- attention ----------------------------------------------------------------------------------

class Cached:
    """A cache that holds rows of the given lengths, and NaN wherever none of them reaches."""

    def __init__(self, lengths, q_heads, heads, dim, page, dtype=BF16, rows=BF16, queries=1, window=0, seed=1,
                 layout="pages", max_length=None, sharp=1.5, sinks=False, scale=None):
        g = _gen(seed)
        self.g, self.lengths, self.queries, self.window = g, list(lengths), queries, window
        self.heads, self.q_heads, self.dim, self.page, self.rows = heads, q_heads, dim, page, rows
        self.scale = dim ** -0.5 if scale is None else scale
        R = len(lengths)
        self.max_length = max(max(lengths), 1) if max_length is None else max_length
        width = -(-self.max_length // page)
        held = [-(-n // page) for n in lengths]
        pages = sum(held) + 3
        ids = torch.randperm(pages, generator=g)
        self.tables = torch.randint(-(1 << 31), 1 << 31, (R, width + 2), generator=g).int()
        self.cache = _make_cache(pages, heads, page, dim, dtype, layout)
        whole = {n: torch.full((pages, heads, page, dim), NAN) for n in "kv"}
        scales = {n: torch.full((pages, heads, page), 120, dtype=torch.uint8) for n in "kv"}
        self.k, self.v, at = [], [], 0
        for r, n in enumerate(lengths):
            mine = ids[at:at + held[r]]
            at += held[r]
            first = max(0, n - (queries - 1) - window) if window else 0
            some = first // page       # pages before the first token in reach may be gone
            self.tables[r, some:held[r]] = mine[some:].int()
            for name, rows_of in (("k", self.k), ("v", self.v)):
                x = torch.randn(heads, n, dim, generator=g)
                if dtype == F8:
                    e = torch.randint(115, 123, (heads, n), generator=g)
                    c = (x * 100).clamp(-448, 448).to(F8).float()
                    exact = c.double() * torch.exp2(e.double() - 127).unsqueeze(2)
                else:
                    c = x.to(BF16).float()
                    exact = c.double()
                rows_of.append(exact)
                t = torch.arange(first, n)
                whole[name][mine[t // page], :, t % page] = c[:, first:].transpose(0, 1)
                if dtype == F8:
                    scales[name][mine[t // page], :, t % page] = e[:, first:].T.to(torch.uint8)
        for name, t, s in (("k", self.cache.k, self.cache.k_scales), ("v", self.cache.v, self.cache.v_scales)):
            x = whole[name].to(dtype)
            (t.view(torch.uint8) if dtype == F8 else t).copy_(x.view(torch.uint8) if dtype == F8 else x)
            if s is not None:
                s.copy_(scales[name])
        self.q = (sharp * torch.randn(R, queries, q_heads, dim, generator=g)).to(rows)
        self.sinks = torch.randn(q_heads, generator=g) if sinks else None
        self.attention = cache_mod().PagedAttention(q_heads, self.cache, R, self.max_length, rows, queries,
                                                    window, scale)

    def run(self, q=None, out=None, lse=True, stream=None):
        q = self.q.cuda() if q is None else q
        out = torch.full(self.q.shape, 7.0, dtype=self.rows, device="cuda") if out is None else out
        lse = torch.full(self.q.shape[:3], 7.0, device="cuda") if lse else None
        self.attention.attend_into(q, self.cache, self.tables.cuda(), _i32(self.lengths), out, lse,
                                   None if self.sinks is None else self.sinks.cuda(), stream)
        return out, lse

    def check(self, out, lse=None, some=None):
        G, D, n = self.q_heads // self.heads, self.dim, self.queries
        dot = 2 * U * (D / 32 + 64)
        weights = {BF16: 2.0 ** -16, F32: U}[self.rows]
        for r in range(len(self.lengths)) if some is None else some:
            for i in range(n):
                end = max(0, self.lengths[r] - (n - 1 - i))
                begin = max(0, end - self.window) if self.window else 0
                k, v = (t[r][:, begin:end].repeat_interleave(G, 0) for t in (self.k, self.v))
                q = self.q[r, i].double().unsqueeze(1)
                x = (q * k).sum(2) * self.scale
                size = (q * k).abs().sum(2) * self.scale
                if self.sinks is not None:
                    x = torch.cat((x, self.sinks.double().unsqueeze(1)), 1)
                got = out[r, i].cpu().double()
                if x.shape[1] == 0:
                    assert bool((got == 0).all())
                    assert lse is None or bool((lse[r, i] == -math.inf).all())
                    continue
                m = x.amax(1, keepdim=True)
                e = (x - m).exp()
                z = e.sum(1, keepdim=True)
                p = (e / z)[:, :end - begin]
                want, spread = (p.unsqueeze(2) * v).sum(1), (p.unsqueeze(2) * v.abs()).sum(1)
                # a weight's relative error: the products of it and of the maximum, the steps from there to
                # exp2 (of values up to |x - m|), exp2's own
                off = 2 * dot * size.amax(1) if size.shape[1] else torch.zeros(self.q_heads)
                off = (off + 8 * U * ((m - x).amax(1) + m.squeeze(1).abs() + 2)).unsqueeze(1)
                # sums over the length: a step per tile, with its rescaling, and the joins
                steps = 2 * U * (2 * (end - begin) / 32 + 200)
                tol = (2 * off + 2 * weights + 2 * steps) * spread
                tol = tol + HALF_STEP[self.rows] * (want.abs() + tol)
                assert bool(torch.isfinite(got).all())
                bad = (got - want).abs() > tol
                assert not bool(bad.any()), (r, i, int(bad.sum()), float(((got - want).abs() / tol).max()),
                                             bad.nonzero()[:4].tolist())
                if lse is not None:
                    exact = (m + z.log()).squeeze(1)
                    far = off.squeeze(1) + steps + 4 * U * (exact.abs() + m.squeeze(1).abs() + 2)
                    assert bool(((lse[r, i].cpu().double() - exact).abs() <= far).all()), (r, i)


KINDS = [(BF16, BF16), (F8, BF16), (BF16, F32), (F8, F32)]
ENDS = [1, 2, 31, 32, 33, 0, 127, 128, 129, 255, 300, 16, 17]


@pytest.mark.parametrize("dtype,rows", KINDS)
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128, 160, 192, 208, 256])
def test_attention_of_every_head_dim(dtype, rows, dim):
    c = Cached(ENDS, 8, 2, dim, 16, dtype, rows)
    c.check(*c.run())
    assert _status(c.attention.sync) == N.OK


@pytest.mark.parametrize("dtype,rows", KINDS)
@pytest.mark.parametrize("page", [1, 3, 16, 24, 32, 64, 100, 1024])
@pytest.mark.parametrize("layout", sorted(LAYOUTS))
def test_attention_over_pages_of_any_size_and_layout(dtype, rows, page, layout):
    c = Cached([1, 200, 33, 97, 1500, 0], 4, 2, 64, page, dtype, rows, layout=layout)
    c.check(*c.run())
    assert _status(c.attention.sync) == N.OK


@pytest.mark.parametrize("dtype,rows", KINDS)
@pytest.mark.parametrize("q_heads,heads", [(1, 1), (2, 2), (5, 1), (16, 1), (17, 1), (40, 8), (64, 2), (33, 3)])
@pytest.mark.parametrize("queries", [1, 3])
def test_attention_of_shared_heads(dtype, rows, q_heads, heads, queries):
    c = Cached([300, 1, 2, 0, 65, 129], q_heads, heads, 64, 16, dtype, rows, queries=queries)
    c.check(*c.run())


@pytest.mark.parametrize("dtype,rows", KINDS)
@pytest.mark.parametrize("queries", [1, 2, 5, 16])
@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 257, 2 ** 32 - 1])
def test_windows(dtype, rows, queries, window):
    c = Cached([1, 3, 16, 64, 300, 0, 700, 129], 6, 2, 96, 24, dtype, rows, queries=queries, window=window)
    c.check(*c.run())
    assert _status(c.attention.sync) == N.OK


@pytest.mark.parametrize("dtype,rows", KINDS)
@pytest.mark.parametrize("lengths", [[0], [5], [3000, 0, 1]])
def test_sinks(dtype, rows, lengths):
    c = Cached(lengths, 8, 2, 128, 16, dtype, rows, sinks=True, queries=2)
    out, lse = c.run()
    c.check(out, lse)
    c.sinks = torch.full((8,), -math.inf)     # as none
    out, lse = c.run()
    c.sinks = None
    c.check(out, lse)
    c.sinks = torch.full((8,), 1e4)           # takes all
    out, lse = c.run()
    assert bool((out == 0).all()) and bool((lse == 1e4).all())


@pytest.mark.parametrize("lengths", [[0], [40], [5, 0, 9000]])
def test_infinite_sinks(lengths):
    c = Cached(lengths, 4, 2, 64, 16, seed=8)
    want, want_lse = c.run()
    c.sinks = torch.tensor([math.inf, -math.inf, -math.inf, math.inf])
    out, lse = c.run()
    for h, s in enumerate(c.sinks.tolist()):
        if s > 0:
            assert bool((out[:, :, h] == 0).all()) and bool((lse[:, :, h] == math.inf).all())
        else:
            assert torch.equal(_bits(out[:, :, h].contiguous()), _bits(want[:, :, h].contiguous()))
            assert torch.equal(lse[:, :, h], want_lse[:, :, h])


@pytest.mark.parametrize("lengths", [[1, 1, 1], [3, 40, 2], [1, 9000]])
def test_sinks_beside_scores_past_the_range(lengths):
    # scores of 2^127 products: the largest is past f32's range (its lse +-inf), and the weights are 1 or 0
    c = Cached(lengths, 8, 2, 64, 16, sharp=100.0, scale=2.0 ** 127, seed=12)
    plain, plain_lse = c.run()
    c.sinks = torch.tensor([0.5, -3.0, -math.inf, math.inf] * 2)
    out, lse = c.run()
    signs = set()
    for r, n in enumerate(lengths):
        top = (c.q[r, 0].double().unsqueeze(1) * c.k[r].repeat_interleave(4, 0)).sum(2).amax(1)
        assert bool((top.abs() > 2).all())
        for h, s in enumerate(c.sinks.tolist()):
            over = top[h] > 0
            signs.add(bool(over))
            assert plain_lse[r, 0, h] == (math.inf if over else -math.inf)
            takes_all = s == math.inf or (s > -math.inf and not over)
            want = torch.zeros_like(plain[r, 0, h]) if takes_all else plain[r, 0, h]
            assert torch.equal(out[r, 0, h], want), (r, h)      # (a zero's sign is not part of the definition)
            assert lse[r, 0, h] == (s if takes_all else plain_lse[r, 0, h]), (r, h)
    assert max(lengths) > 1 or len(signs) == 2


@pytest.mark.parametrize("dtype,rows", KINDS)
@pytest.mark.parametrize("lengths,q_heads,heads,dim", [
    ([20000], 16, 2, 256), ([131071], 4, 1, 64), ([5000, 3, 40, 9000, 0, 777], 32, 8, 128),
    ([64] * 97 + [30000], 4, 4, 64), (list(range(1, 130)), 8, 8, 80)])
def test_lengths_shared_out_over_the_chip(dtype, rows, lengths, q_heads, heads, dim):
    c = Cached(lengths, q_heads, heads, dim, 64, dtype, rows)
    out, lse = c.run()
    c.check(out, lse, some=range(0, len(lengths), max(1, len(lengths) // 12)))
    again = c.run()
    assert torch.equal(_bits(out), _bits(again[0])) and torch.equal(_bits(lse), _bits(again[1]))


@pytest.mark.parametrize("dtype,rows,dim,page,queries", [
    (BF16, BF16, 128, 24, 1), (BF16, F32, 96, 16, 3), (BF16, BF16, 80, 64, 1), (F8, BF16, 128, 7, 2),
    (F8, F32, 192, 100, 1)])
def test_more_than_the_caches_of_the_chip_hold(dtype, rows, dim, page, queries):
    size = 1 if dtype == F8 else 2
    n = (160 << 20) // (2 * 8 * dim * size)
    lengths = [n // 2, 0, 1, n // 4 + 5, 33, n // 8, n // 8 + 130, 127]
    c = Cached(lengths, 16, 8, dim, page, dtype, rows, queries)
    out, lse = c.run()
    c.check(out, lse, some=[1, 2, 4, 5, 6, 7])
    again = c.run()
    assert torch.equal(_bits(out), _bits(again[0])) and torch.equal(_bits(lse), _bits(again[1]))


def test_more_rows_than_a_launch_takes():
    lengths = [(7 * r) % 50 for r in range(2100)]
    c = Cached(lengths, 2, 1, 32, 16)
    out, lse = c.run()
    c.check(out, lse, some=list(range(0, 2100, 97)) + [1023, 1024, 1025, 2047, 2048, 2099])


@pytest.mark.parametrize("sharp,scale", [(30.0, None), (1.0, 5.0), (1e-3, 1e-3), (1e18, 1e-18)])
@pytest.mark.parametrize("dtype,rows", KINDS)
def test_scores_of_any_size(dtype, rows, sharp, scale):
    c = Cached([1, 700, 64, 33], 8, 2, 64, 16, dtype, rows, sharp=sharp, scale=scale)
    c.check(*c.run())


def test_rows_whose_scores_are_all_far_below_zero():
    # every product is -1e4 and less: nothing underflows before the maximum is taken off
    c = Cached([200, 40], 4, 1, 64, 16, sharp=0.0)
    c.q = torch.full_like(c.q, -100.0)
    for r in range(2):
        c.k[r] = c.k[r].abs() + 2
    g = c.cache.k.float()
    c.cache.k.copy_((g.abs() + 2).to(BF16))
    for r in range(2):
        pages = c.tables[r, :-(-c.lengths[r] // 16)].long()
        c.k[r] = c.cache.k[pages].cpu().double().transpose(0, 1).flatten(1, 2)[:, :c.lengths[r]]
    c.check(*c.run())


@pytest.mark.parametrize("rows", [BF16, F32])
def test_outputs_in_place_and_strided(rows):
    c = Cached([5, 300, 64], 8, 2, 64, 16, rows=rows, queries=2)
    want, lse = c.run()
    fused = torch.full((3, 2, 8 * 64 + 128 + 32), 3.0, dtype=rows, device="cuda")
    q = fused[..., 64:64 + 512].unflatten(2, (8, 64))
    q.copy_(c.q)
    out, _ = c.run(q=q, out=q)
    assert torch.equal(_bits(out), _bits(want))
    assert bool((fused[..., :64] == 3).all()) and bool((fused[..., 576:] == 3).all())
    turned = torch.full((8, 3, 2, 80), 3.0, dtype=rows, device="cuda").permute(1, 2, 0, 3)[..., :64]
    c.run(out=turned, lse=False)
    assert torch.equal(_bits(turned), _bits(want))


def test_a_cache_of_more_than_4_gib():
    pages, stride = 48, 1 << 27
    raw = torch.empty(pages * stride, dtype=BF16, device="cuda")
    c = Cached([600, 37], 4, 1, 64, 16, seed=3)
    n = c.cache.pages
    k, v = (torch.as_strided(raw, (pages, 1, 16, 64), (stride, 1 << 20, 64, 1), at) for at in (0, 1 << 25))
    far = cache_mod().PagedCache(k, v)
    order = torch.randperm(pages, generator=c.g)[:n]
    k[order.cuda()], v[order.cuda()] = c.cache.k, c.cache.v
    want = c.run()
    t = c.tables
    inside = (t >= 0) & (t < n)
    c.tables = torch.where(inside, order[t.clamp(0, n - 1).long()].int(), t)
    c.cache = far
    got = c.run()
    assert torch.equal(_bits(got[0]), _bits(want[0])) and torch.equal(_bits(got[1]), _bits(want[1]))
    x = torch.randn(3, 1, 64, generator=c.g).to(BF16).cuda()
    slots = torch.tensor([39 * 16 + 15, 20 * 16, 1], device="cuda")
    far.append(x, x, slots)
    for i, s in enumerate(slots.tolist()):
        assert torch.equal(k[s // 16, 0, s % 16], x[i, 0]) and torch.equal(v[s // 16, 0, s % 16], x[i, 0])


def test_infinities_and_nans_stay_in_their_rows():
    c = Cached([40, 50, 60], 4, 2, 64, 16)
    want, lse = c.run()
    page = int(c.tables[1, 1])
    c.cache.k[page, 0, 3] = math.inf
    c.cache.v[page, 1, 2, 7] = NAN
    out, lse2 = c.run()
    for r in (0, 2):
        assert torch.equal(_bits(out[r]), _bits(want[r])) and torch.equal(_bits(lse2[r]), _bits(lse[r]))
    # heads 2, 3 read cache head 1: only value 7 is touched
    rest = [d for d in range(64) if d != 7]
    assert torch.equal(_bits(out[1, 0, 2:][:, rest]), _bits(want[1, 0, 2:][:, rest]))
    assert bool(torch.isnan(out[1, 0, 2:, 7]).all())


@pytest.mark.parametrize("lengths", [[40], [9000], [5, 0, 9000]])
@pytest.mark.parametrize("rows", [BF16, F32])
def test_queries_of_nan_stay_nan(lengths, rows):
    # in a row of one workgroup and in one that several share
    c = Cached(lengths, 8, 2, 64, 16, rows=rows, queries=2)
    want, want_lse = c.run()
    c.q[-1, 1, 3], c.q[-1, 0, 6, 5] = NAN, NAN
    out, lse = c.run()
    hit = torch.zeros(out.shape[:3], dtype=torch.bool)
    hit[-1, 1, 3] = hit[-1, 0, 6] = True
    assert bool(torch.isnan(out.cpu()[hit].float()).all()) and bool(torch.isnan(lse.cpu()[hit]).all())
    assert torch.equal(_bits(out)[~hit], _bits(want)[~hit])
    assert torch.equal(_bits(lse)[~hit], _bits(want_lse)[~hit])


def test_lengths_and_pages_out_of_range():
    c = Cached([100, 40, 64, 90], 4, 2, 64, 16, max_length=100)
    want, lse = c.run()
    good = list(c.lengths)
    for bad in (-1, 101, 2 ** 31 - 1, -2 ** 31):
        c.lengths = [good[0], bad, good[2], good[3]]
        out, lse2 = c.run()
        assert _status(c.attention.sync) == N.ERR_ARGUMENT
        assert _status(c.attention.sync) == N.OK
        assert bool((out[1] == 0).all()) and bool((lse2[1] == -math.inf).all())
        c.lengths[1] = 0
        c.check(out, lse2)
    c.lengths = good
    for entry in (-1, c.cache.pages, 2 ** 31 - 1):
        tables = c.tables.clone()
        c.tables[2, 1] = entry                 # tokens 16 .. 31 of row 2
        out, lse2 = c.run()
        assert _status(c.attention.sync) == N.ERR_ARGUMENT
        c.tables = tables
        d = Cached([100, 40, 64, 90], 4, 2, 64, 16, max_length=100)
        left = [t for t in range(64) if not 16 <= t < 32]
        d.k[2], d.v[2], d.lengths = d.k[2][:, left], d.v[2][:, left], [100, 40, 48, 90]
        d.check(out, lse2)


@pytest.mark.parametrize("lengths,dim,rows", [([1], 64, BF16), ([700, 3], 128, BF16), ([90000], 64, F32)])
def test_captured_attention_replays(lengths, dim, rows):
    c = Cached(lengths, 8, 2, dim, 16, rows=rows)
    q, out = c.q.cuda(), torch.empty(c.q.shape, dtype=rows, device="cuda")
    lse = torch.empty(c.q.shape[:3], device="cuda")
    tables, n = c.tables.cuda(), _i32(c.lengths)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        c.attention.attend_into(q, c.cache, tables, n, out, lse)
    full = list(lengths)
    k, v = list(c.k), list(c.v)
    for i in range(4):
        c.q = (1.5 * torch.randn(c.q.shape, generator=c.g)).to(rows)
        c.lengths = [max(0, m - 29 * i) for m in full]
        c.k, c.v = ([t[r][:, :m] for r, m in enumerate(c.lengths)] for t in (k, v))
        q.copy_(c.q)
        n.copy_(_i32(c.lengths))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        c.check(out, lse)
        eager, _ = c.run()
        assert torch.equal(_bits(eager), _bits(out))


def test_attention_on_another_stream():
    c = Cached([3000, 40], 8, 2, 64, 16)
    want, lse = c.run()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    q, out = c.q.cuda(), torch.empty_like(want)
    s.wait_stream(torch.cuda.current_stream())
    c.run(q=q, out=out, stream=s)
    c.attention.sync(s)
    torch.cuda.synchronize()
    assert torch.equal(_bits(out), _bits(want))


def test_two_contexts_at_once():
    cases = [Cached([9000, 40, 0, 700], 8, 2, 128, 16, seed=5), Cached([6000, 1, 3000], 4, 4, 64, 24, F8, F32, seed=6)]
    want = [c.run() for c in cases]
    tensors = [(c.q.cuda(), c.tables.cuda(), _i32(c.lengths), torch.empty_like(w[0]), torch.empty_like(w[1]))
               for c, w in zip(cases, want)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, (q, tables, n, out, lse), s in zip(cases, tensors, streams):
            c.attention.attend_into(q, c.cache, tables, n, out, lse, stream=s)
    torch.cuda.synchronize()
    for c, (_, _, _, out, lse), w, s in zip(cases, tensors, want, streams):
        c.attention.sync(s)
        assert torch.equal(_bits(out), _bits(w[0])) and torch.equal(_bits(lse), _bits(w[1]))


def test_a_step_on_another_stream():
    C, g = cache_mod(), _gen(9)
    rows, page, blocks = 6, 4, 8
    k, v = (torch.randn(rows, 2, 64, generator=g).to(BF16).cuda() for _ in range(2))
    q = torch.randn(rows, 1, 8, 64, generator=g).to(BF16).cuda()
    results = []
    for stream in (None, torch.cuda.Stream()):
        cache = C.PagedCache.zeros(40, 2, page, 64)
        pager = C.Pager(40, page, rows, blocks, rows)
        attention = C.PagedAttention(8, cache, rows, page * blocks)
        (free, count), plan = pager.new_stack(), pager.new_plan(rows, rows)
        plan.count, plan.lengths = count, torch.zeros(rows, dtype=torch.int32, device="cuda")
        tables, other = (torch.zeros(rows, blocks, dtype=torch.int32, device="cuda") for _ in range(2))
        out, parents = torch.empty_like(q), _i32([[1, 1, -1], [0, 2, 0]])
        torch.cuda.synchronize()
        for _ in range(6):
            pager.plan_into(plan.lengths, None, tables, free, count, plan, stream)
            cache.append(k, v, plan.slots, stream)
            attention.attend_into(q, cache, tables, plan.lengths, out, stream=stream)
            pager.fork_into(parents, tables, plan.lengths, free, count, other, plan.lengths, count, [cache], stream)
            tables, other = other, tables
        for c in (pager, attention):
            c.sync(stream)
        results.append([t.cpu() for t in (plan.lengths, plan.slots, count, _bits(out), _bits(cache.k), _bits(cache.v))])
    for one, two in zip(*results):
        assert torch.equal(one, two)
    assert results[0][0].tolist() == [6, 6, 0, 6, 6, 6]


def test_attention_refuses():
    c = Cached([40], 4, 2, 64, 16)
    att, q = c.attention, c.q.cuda()
    out, tables, n = torch.empty_like(q), c.tables.cuda(), _i32([40])
    call = lambda **k: att.attend_into(**{**dict(q=q, cache=c.cache, tables=tables, lengths=n, out=out), **k})
    call()
    for change in (dict(q=q.float()), dict(out=out.float()), dict(q=q[:, :, :3]), dict(tables=tables[:, :2]),
                   dict(tables=tables.long()), dict(lengths=n.long()), dict(lengths=n.cpu()),
                   dict(lse=torch.empty(1, device="cuda")), dict(sinks=torch.empty(3, device="cuda")),
                   dict(out=torch.empty(1, 1, 64, 4, dtype=BF16, device="cuda").transpose(2, 3))):
        with pytest.raises(ValueError):
            call(**change)
    odd = torch.empty(1 * 4 * 64 + 1, dtype=BF16, device="cuda")[1:].view(1, 1, 4, 64)
    assert _status(lambda: call(q=odd)) == N.ERR_ARGUMENT
    assert _status(lambda: call(out=odd)) == N.ERR_ARGUMENT
    assert _status(lambda: call(out=torch.empty(64, dtype=BF16, device="cuda").expand(1, 1, 4, 64))) == N.ERR_SHAPE
    for other in (_make_cache(3, 2, 8, 64, BF16), _make_cache(3, 1, 16, 64, BF16),
                  _make_cache(3, 2, 16, 80, BF16), _make_cache(3, 2, 16, 64, F8)):
        assert _status(lambda: call(cache=other)) == N.ERR_SHAPE
    many = q.expand(2, 1, 4, 64).contiguous()
    assert _status(lambda: call(q=many, out=torch.empty_like(many), tables=tables.expand(2, -1).contiguous(),
                                lengths=_i32([1, 1]))) == N.ERR_SHAPE


# ---- forks --------------------------------------------------------------------------------------

def _fork_by_hand(parents, tables, out, lengths, free, count, page, pages, max_blocks):
    """(tables, lengths, free, count, copies, status): copies (from, to, tokens)."""
    R, W = parents.shape
    out, free = [list(r) for r in out], list(free)
    bits = set()
    if not 0 <= count <= pages:
        bits.add(N.ERR_ARGUMENT)
        count = 0
    n = np.array(lengths).reshape(R, W)
    if ((n < 0) | (n > max_blocks * page)).any():
        bits.add(N.ERR_ARGUMENT)
    n = np.where((n < 0) | (n > max_blocks * page), 0, n)
    if (parents >= W).any():
        bits.add(N.ERR_ARGUMENT)
    parents = np.where((parents < 0) | (parents >= W), -1, parents)
    new_lengths = [0] * (R * W)
    blocks = -(-n // page)
    for r in range(R):
        for j in range(blocks[r].max()):
            column = [tables[r * W + i][j] if j < blocks[r, i] else None for i in range(W)]
            held = {column[p] for p in parents[r] if p >= 0}
            for i in range(W):
                if column[i] is None or i in parents[r]:
                    continue
                if not 0 <= column[i] < pages:
                    bits.add(N.ERR_ARGUMENT)
                elif column[i] not in held:
                    held.add(column[i])
                    if count < pages:
                        free[count] = column[i]
                        count += 1
                    else:
                        bits.add(N.ERR_ARGUMENT)
    copies = []
    for r in range(R):
        seen = set()
        for i in range(W):
            p = parents[r, i]
            if p < 0:
                continue
            row, m = r * W + i, int(n[r, p])
            out[row][:blocks[r, p]] = tables[r * W + p][:blocks[r, p]]
            new_lengths[row] = m
            if p in seen and m % page:
                source = out[row][m // page]
                if count == 0:
                    bits.add(N.ERR_OUT_OF_MEMORY)
                    new_lengths[row] = 0
                else:
                    count -= 1
                    out[row][m // page] = free[count]
                    if 0 <= free[count] < pages and 0 <= source < pages:
                        copies.append((source, free[count], m % page))
                    else:
                        bits.add(N.ERR_ARGUMENT)
            seen.add(p)
    status = N.ERR_ARGUMENT if N.ERR_ARGUMENT in bits else N.ERR_OUT_OF_MEMORY if bits else N.OK
    return out, new_lengths, free, count, copies, status


class Beams:
    """Rows of requests that share the pages of a beginning, and caches of them."""

    def __init__(self, requests, width, page, max_blocks, seed, spare=None, layers=1, dtype=BF16, heads=2, dim=32,
                 ragged=False):
        g = np.random.default_rng(seed)
        self.page, self.max_blocks, self.shape = page, max_blocks, (requests, width)
        top = max_blocks * page
        length = np.repeat(g.integers(0, top + 1, (requests, 1)), width, 1)
        if ragged:
            length = g.integers(0, top + 1, (requests, width))
        common = np.minimum(g.integers(0, max_blocks + 1, (requests, 1)), length.min(1, keepdims=True) // page)
        blocks = -(-length // page)
        total = int(blocks.sum()) + (requests * width if spare is None else spare)
        ids = list(g.permutation(total))
        self.tables = np.full((requests * width, max_blocks), -3)
        for r in range(requests):
            first = [ids.pop() for _ in range(int(common[r, 0]))]
            for i in range(width):
                row = first + [ids.pop() for _ in range(int(blocks[r, i] - common[r, 0]))]
                self.tables[r * width + i, :len(row)] = row
        self.pages = total
        self.count = len(ids) if spare is None else min(spare, len(ids))
        self.free = np.full(total, -4)
        self.free[:self.count] = ids[:self.count]
        self.lengths = length.reshape(-1)
        self.parents = g.integers(0, width, (requests, width))
        self.layers = [self._filled(total, heads, page, dim, dtype, seed + i) for i in range(layers)]

    @staticmethod
    def _filled(pages, heads, page, dim, dtype, seed):
        c = _make_cache(pages, heads, page, dim, dtype)
        g = torch.Generator("cuda").manual_seed(seed)
        for t in (c.k, c.v):
            t.view(torch.uint8).random_(0, 256, generator=g)
        for t in (c.k_scales, c.v_scales):
            if t is not None:
                t.random_(0, 256, generator=g)
        return c

    def check(self, in_place=False, stream=None):
        R, W = self.shape
        P = cache_mod().Pager(self.pages, self.page, R * W, self.max_blocks)
        wide = torch.full((R * W, self.max_blocks + 2), -8, dtype=torch.int32, device="cuda")
        out, tables = wide[:, 1:-1], _i32(self.tables)
        lengths, free, count = _i32(self.lengths), _i32(self.free), _i32([self.count])
        new_lengths, new_count = (lengths, count) if in_place else (
            torch.empty_like(lengths), torch.empty_like(count))
        want = _fork_by_hand(self.parents, self.tables.tolist(), out.tolist(), self.lengths, self.free.tolist(),
                             self.count, self.page, self.pages, self.max_blocks)
        held = [[_bits(t) for t in (c.k, c.v)] + [s.cpu() for s in (c.k_scales, c.v_scales) if s is not None]
                for c in self.layers]
        for tensors in held:
            for t in tensors:
                for source, to, tokens in want[4]:
                    t[to, :, :tokens] = t[source, :, :tokens].clone()
        P.fork_into(_i32(self.parents), tables, lengths, free, count, out, new_lengths, new_count, self.layers)
        assert _status(P.sync) == want[5]
        _same(out, want[0])
        _same(new_lengths, want[1])
        _same(free, want[2])
        _same(new_count, [want[3]])
        _same(tables, self.tables)
        assert bool((wide[:, 0] == -8).all()) and bool((wide[:, -1] == -8).all())
        for c, tensors in zip(self.layers, held):
            for t, w in zip([c.k, c.v, c.k_scales, c.v_scales], tensors):
                assert torch.equal(_bits(t) if t.dtype != torch.uint8 else t.cpu(), w)
        return want


@pytest.mark.parametrize("dtype", [BF16, F8])
@pytest.mark.parametrize("requests,width,page,blocks", [
    (1, 1, 16, 4), (1, 4, 16, 5), (7, 5, 3, 9), (32, 8, 16, 12), (3, 64, 7, 6), (300, 2, 1, 5), (5, 3, 100, 2),
    (2, 4, 2, 700), (600, 3, 16, 4)])
def test_forks(dtype, requests, width, page, blocks):
    for seed in (1, 2):
        want = Beams(requests, width, page, blocks, seed, dtype=dtype).check(in_place=seed == 2)
        assert want[5] == N.OK


@pytest.mark.parametrize("dtype", [BF16, F8])
@pytest.mark.parametrize("width,page,blocks", [
    (4, 2, 700), (64, 7, 6), (9, 3, 300), (8, 16, 43), (63, 1, 513), (64, 2, 257), (2, 100, 3)])
def test_forks_of_a_single_request(dtype, width, page, blocks):
    # more than 256 columns, more than eight rows, all of the LDS
    for seed in (1, 2):
        assert Beams(1, width, page, blocks, seed, dtype=dtype).check(in_place=seed == 2)[5] == N.OK
    b = Beams(1, width, page, blocks, 3, dtype=dtype, ragged=True)
    b.lengths[0] = blocks * page            # (its pages in all the passes over columns, and dropped)
    b.tables[0] = np.arange(blocks) + b.pages
    b.pages += blocks
    b.free = np.concatenate((b.free, np.full(blocks, -4)))
    b.layers = [b._filled(b.pages, 2, page, 32, dtype, 1)]
    b.parents[:] = np.where(np.arange(width) % 3, width - 1, -1)
    want = b.check()
    assert want[5] == N.OK and want[3] >= b.count + blocks - (width - 1)
    b.parents[:] = -1
    want = b.check(in_place=True)
    assert want[5] == N.OK and not want[4]


def test_forks_of_every_layer():
    for layers in (0, 16, 17, 35):
        Beams(4, 3, 5, 6, layers, layers=layers, dim=16).check()


@pytest.mark.parametrize("requests,width", [(6, 4), (40, 2)])
def test_rows_that_end(requests, width):
    b = Beams(requests, width, 8, 7, 3, ragged=True)
    b.parents = np.where(np.random.default_rng(1).random(b.parents.shape) < 0.4, -1, b.parents)
    assert b.check()[5] == N.OK
    b.parents[:] = -1
    want = b.check()
    assert want[3] == len({p for r, n in zip(b.tables, b.lengths) for p in r[:-(-n // 8)]}) + b.count
    b = Beams(requests, width, 8, 7, 3)
    b.parents[:] = np.arange(width)     # nothing changes hands
    want = b.check()
    assert want[3] == b.count and not want[4]


def test_a_search_that_begins_from_one_row():
    b = Beams(5, 6, 16, 4, 4, ragged=True)
    b.parents[:] = 0
    assert b.check()[5] == N.OK


@pytest.mark.parametrize("spare", [0, 1, 4])
def test_forks_without_enough_pages(spare):
    # rows of no length with one that has all the children: nothing is dropped
    b = Beams(6, 4, 16, 3, 5)
    b.lengths = np.where(np.arange(24) % 4 == 0, 21, 0)
    b.parents[:] = 0
    b.tables[::4, :2] = np.arange(12).reshape(6, 2)
    b.pages = 12 + spare
    b.free, b.count = np.arange(12 + spare) + 12, spare
    b.layers = [b._filled(b.pages, 2, 16, 32, BF16, 1)]
    assert b.check()[5] == N.ERR_OUT_OF_MEMORY
    b.check(in_place=True)


@pytest.mark.parametrize("spare", [0, 1, 2])
def test_a_single_request_without_enough_pages(spare):
    b = Beams(1, 4, 16, 3, 5)
    b.lengths = np.array([21, 0, 0, 0])
    b.parents[:] = 0
    b.tables[0, :2] = [0, 1]
    b.pages = 2 + spare
    b.free, b.count = np.arange(2 + spare) + 2, spare
    b.layers = [b._filled(b.pages, 2, 16, 32, BF16, 1)]
    assert b.check()[5] == N.ERR_OUT_OF_MEMORY
    b.check(in_place=True)


def test_a_single_request_that_cannot_be():
    b = Beams(1, 4, 16, 3, 6)
    b.parents[0, 1], b.lengths[2] = 4, -1
    assert b.check()[5] == N.ERR_ARGUMENT
    for seed in (6, 7):
        for count in (-1, 10 ** 6):
            b = Beams(1, 4, 16, 3, seed)
            b.count = count
            assert b.check(in_place=True)[5] == N.ERR_ARGUMENT
    # two pages dropped on a stack with room for one, and one that is none
    b = Beams(1, 3, 16, 3, 7)
    b.lengths[:], b.parents[:] = 32, [0, 0, 0]
    b.tables[:, :2] = [[0, 1], [2, 3], [4, 10 ** 6]]
    b.count = b.pages - 1
    assert b.check()[5] == N.ERR_ARGUMENT


def test_forks_of_rows_that_cannot_be():
    b = Beams(6, 4, 16, 3, 6)
    b.parents[0, 1], b.parents[2, 0] = 4, 2 ** 31 - 1
    b.lengths[9], b.lengths[14] = -1, 49
    assert b.check()[5] == N.ERR_ARGUMENT
    for count in (-1, 10 ** 6):
        b = Beams(6, 4, 16, 3, 6)
        b.count = count
        assert b.check()[5] == N.ERR_ARGUMENT
    b = Beams(6, 4, 16, 3, 7)
    b.lengths[:] = 40
    b.tables[:, :3] = np.arange(72).reshape(24, 3)
    b.parents[:] = [0, 0, 1, 1]
    b.tables[2, 1], b.tables[5, 2], b.tables[7, 2] = -1, b.pages, 2 ** 31 - 1
    b.count, b.pages = 5, max(b.pages, 80)
    b.free = np.full(b.pages, -4)
    b.free[:5] = [72, 73, 74, 75, 76]
    b.layers = [b._filled(b.pages, 2, 16, 32, BF16, 1)]
    assert b.check()[5] == N.ERR_ARGUMENT
    b.pages, b.layers = 74, []      # a stack that cannot take all the dropped
    b.free = b.free[:74]
    b.count = 72
    assert b.check()[5] == N.ERR_ARGUMENT


@pytest.mark.parametrize("width", [2, 4, 16, 17, 64])
@pytest.mark.parametrize("requests", [1, 3])
def test_rows_with_children_that_share_a_page_filled_in_part(requests, width):
    rows, page, last = requests * width, 4, width - 1
    common = [[0, 1, 2 + i] for i in range(width)]      # the first two pages are all rows'
    stay = list(range(width))
    for status, lengths, parents, tables in (
            (N.OK, [8] * width, stay, common),                                   # whole pages
            (N.OK, [11] * width, stay, common),                                  # and one in part for each
            (N.ERR_ARGUMENT, [7] * width, stay, common),                         # a prompt that all go on with
            (N.OK, [7] * width, [last] + [-1] * last, common),                   # ... one does
            (N.OK, [7] * width, [last] * width, common),                         # ... with all the children
            (N.ERR_ARGUMENT, [7] * width, [0, last] + [-1] * (width - 2), common),
            (N.ERR_ARGUMENT, [8] * last + [6], stay, common),                    # whole in the others
            (N.ERR_ARGUMENT, [6] + [12] * last, stay, common),
            (N.OK, [4] * last + [6], stay, common),                              # the others end before it
            (N.OK, [7] * width, stay, [[0, -1, 2]] * width)):                    # no page
        own = width + 2
        tables = np.array([[p + r * own if p >= 0 else p for p in row] for r in range(requests) for row in tables])
        lengths, parents = np.array(lengths * requests), np.array([parents] * requests)
        free = list(range(requests * own, requests * own + rows)) + [-4] * 7
        pages = len(free) + requests * own
        free += [-4] * (pages - len(free))
        P = cache_mod().Pager(pages, page, rows, 3)
        out, n, stack, count = torch.full((rows, 3), -8, dtype=torch.int32, device="cuda"), _i32(lengths), _i32(
            free), _i32([rows])
        want = _fork_by_hand(parents, tables.tolist(), out.tolist(), lengths, free, rows, page, pages, 3)
        assert want[5] == N.OK
        P.fork_into(_i32(parents), _i32(tables), n, stack, count, out, n, count)
        assert _status(P.sync) == status, (lengths, parents)
        for got, w in zip((out, n, stack, count), want):
            _same(got, w)
        assert _status(P.sync) == N.OK


def test_forks_refuse():
    P = cache_mod().Pager(20, 16, 8, 3)
    t, n, one = torch.zeros(8, 3, dtype=torch.int32, device="cuda"), _i32([0] * 8), _i32([0])
    free, out = torch.zeros(20, dtype=torch.int32, device="cuda"), torch.zeros_like(t)
    call = lambda parents=_i32([[0, 1], [0, 1], [0, 1], [0, 1]]), **k: P.fork_into(
        parents, *[k.get(name, v) for name, v in (("tables", t), ("lengths", n), ("free", free), ("count", one),
                                                  ("out", out), ("new", n), ("left", one))], k.get("caches", ()))
    call()
    assert _status(lambda: call(out=t)) == N.ERR_ARGUMENT
    assert _status(lambda: call(caches=[_make_cache(20, 1, 8, 16, BF16)])) == N.ERR_SHAPE
    assert _status(lambda: call(caches=[_make_cache(19, 1, 16, 16, BF16)])) == N.ERR_SHAPE
    for change in (dict(parents=_i32([0])), dict(tables=t[:, :2]), dict(out=out[:4]), dict(lengths=n[:4]),
                   dict(free=free[:5]), dict(count=n)):
        with pytest.raises(ValueError):
            call(**change)
    big = cache_mod().Pager(20, 16, 65, 1)
    t, n = torch.zeros(65, 1, dtype=torch.int32, device="cuda"), _i32([0] * 65)
    assert _status(lambda: big.fork_into(_i32([[0] * 65]), t, n, free, one, torch.zeros_like(t), n,
                                         one)) == N.ERR_SHAPE


def test_forks_of_the_most_requests_and_caches():
    rows = 4097
    P = cache_mod().Pager(rows, 4, rows, 1)
    t, n, one = torch.arange(rows, dtype=torch.int32, device="cuda").view(-1, 1), _i32([3] * rows), _i32([0])
    free, out = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.full_like(t, -1)
    def call(R, W=1, caches=()):
        k = R * W
        P.fork_into(torch.zeros(R, W, dtype=torch.int32, device="cuda"), t[:k], n[:k].clone(), free, one, out[:k],
                    torch.empty_like(n[:k]), torch.empty_like(one), caches)
    call(4096)
    assert _status(P.sync) == N.OK and torch.equal(out[:4096], t[:4096]) and int(out[4096]) == -1
    assert _status(lambda: call(4097)) == N.ERR_SHAPE
    layers = [_make_cache(rows, 1, 4, 16, BF16) for _ in range(3)]
    for c in layers:
        c.k.view(-1)[:] = torch.arange(c.k.numel(), device="cuda").to(BF16)
    was = layers[0].k.clone()
    few = [layers[i % 3] for i in range(4096)]
    n[0], n[1], one[0] = 3, 0, 1
    free[0] = rows - 1
    P.fork_into(_i32([[0, 0]]), t[:2], n[:2], free, one, out[:2], torch.empty_like(n[:2]), torch.empty_like(one), few)
    assert _status(P.sync) == N.OK
    was[rows - 1, :, :3] = was[0, :, :3]
    assert all(torch.equal(c.k, was) for c in layers)
    assert _status(lambda: call(1, caches=few + few[:1])) == N.ERR_SHAPE


def test_forks_of_tables_that_overlap_refuse():
    P = cache_mod().Pager(20, 16, 4, 3)
    n, one, parents = _i32([0] * 4), _i32([0]), _i32([[0, 1], [0, 1]])
    free = torch.zeros(20, dtype=torch.int32, device="cuda")
    raw = torch.zeros(200, dtype=torch.int32, device="cuda")
    table = lambda at, stride, columns=3: torch.as_strided(raw, (4, columns), (stride, 1), at)
    call = lambda a, b: _status(lambda: P.fork_into(parents, a, n, free, one, b, n, one))
    for a, b in ((table(0, 3), table(12, 3)), (table(20, 3), table(8, 3)),            # one behind the other
                 (table(0, 6), table(3, 6)), (table(3, 6), table(0, 6)),              # rows by turns
                 (table(0, 7), table(24, 10)), (table(0, 8, 5), table(3, 8, 5)),      # more columns than blocks
                 (table(0, 40), table(3, 5)), (table(3, 5), table(43, 40))):
        assert call(a, b) == N.OK
    for a, b in ((table(0, 3), table(11, 3)), (table(0, 3), table(3, 3)), (table(1, 3), table(0, 3)),
                 (table(0, 6), table(2, 6)), (table(0, 6), table(4, 6)), (table(0, 7), table(23, 10)),
                 (table(0, 40), table(38, 5)), (table(37, 5), table(0, 40)), (table(0, 20), table(60, 3))):
        assert call(a, b) == N.ERR_ARGUMENT and call(b, a) == N.ERR_ARGUMENT


# ---- beam search's selection ----------------------------------------------------------------------

def _select_by_hand(logits, scores, picks, ended, end_token):
    """(scores, tokens, parents) in f64 from host tensors."""
    R, W = scores.shape
    V = logits.shape[1]
    x = logits.double().view(R, W, V)
    x = torch.where(x.isnan(), -math.inf, x)
    m = x.amax(2, keepdim=True)
    gap = torch.where(x == m, 0.0, x - m)
    p = torch.where(x == -math.inf, -math.inf, gap - gap.exp().sum(2, keepdim=True).log())
    if ended is not None:
        only = torch.full((V,), -math.inf, dtype=torch.float64)
        if end_token >= 0:
            only[end_token] = 0.0
        p = torch.where(ended.unsqueeze(2) != 0, only, p)
    c = scores.double()
    c = torch.where(c.isnan() | (c == math.inf), -math.inf, c)
    total = (c.unsqueeze(2) + p).flatten(1)
    total, at = total.sort(dim=1, descending=True, stable=True)
    pad = max(0, picks - W * V)
    total = torch.cat((total[:, :picks], torch.full((R, pad), -math.inf, dtype=torch.float64)), 1)
    at = torch.cat((at[:, :picks], torch.zeros((R, pad), dtype=torch.long)), 1)
    none = total == -math.inf
    return total, torch.where(none, -1, at % V), torch.where(none, -1, at // V)


def _check_beams(logits, scores, picks, ended=None, end_token=-1, width=None, status=N.OK, strided=False):
    R, W = scores.shape
    V = logits.shape[1]
    s = step().BeamSelector(V, W, picks, R, logits.dtype)
    x = logits.cuda()
    if strided:
        x = torch.full((R * W, V + 5), 50.0, dtype=logits.dtype, device="cuda")
        x[:, 3:-2] = logits.cuda()
        x = x[:, 3:-2]
    out = (torch.empty(R, picks, device="cuda"), torch.empty(R, picks, dtype=torch.int32, device="cuda"),
           torch.empty(R, picks, dtype=torch.int32, device="cuda"))
    over = torch.empty(R, picks, dtype=torch.int32, device="cuda")
    s.select_into(x, scores.cuda(), *out, ended=None if ended is None else ended.int().cuda(),
                  end_token=end_token, ended_out=over)
    assert _status(s.sync) == status
    total, tokens, parents = _select_by_hand(logits, scores, picks, ended, end_token)
    _same(out[1], tokens)
    _same(out[2], parents)
    # the sums in f64 are off by far less than an f32's half step; a midpoint may fall to either side
    got = out[0].cpu().double()
    fine = torch.isfinite(total)
    assert torch.equal(fine, torch.isfinite(got))
    assert bool(((got - total).abs()[fine] <= 1.01 * U * total.abs()[fine]).all())
    was = torch.zeros(R, W, dtype=torch.bool) if ended is None else ended != 0
    done = was.gather(1, parents.clamp(min=0)) | (parents < 0) | ((tokens == end_token) & (tokens >= 0))
    _same(over, done.int())
    return out


def _beam_case(R, W, V, dtype, seed, dead=0.2, over=0.2):
    g = _gen(seed)
    logits = 3 * torch.randn(R * W, V, generator=g)
    logits[torch.rand(R * W, V, generator=g) < 0.05] = -math.inf
    scores = -5 * torch.rand(R, W, generator=g)
    scores[torch.rand(R, W, generator=g) < dead] = -math.inf
    return logits.to(dtype), scores, torch.rand(R, W, generator=g) < over


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("R,W,picks,V", [
    (1, 1, 1, 1), (1, 1, 4, 3), (3, 4, 4, 1), (2, 4, 8, 50257), (5, 8, 16, 32000), (1, 32, 64, 262144),
    (9, 3, 7, 8192), (4, 5, 5, 8193), (40, 16, 32, 999), (2, 2, 64, 40), (3, 32, 64, 20000)])
def test_beams(dtype, R, W, picks, V):
    logits, scores, ended = _beam_case(R, W, V, dtype, R + W + V)
    _check_beams(logits, scores, picks)
    _check_beams(logits, scores, picks, ended, end_token=V // 2)
    _check_beams(logits, scores, picks, ended, end_token=V - 1, strided=True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [40, 9000, 70000])
def test_candidates_that_tie(dtype, V):
    # equal logits in a beam, equal beams in a request: the lowest beam and token
    logits = torch.zeros(6, V)
    logits[:, 7::3] = 1.0
    _check_beams(logits.to(dtype), torch.zeros(2, 3), 64)
    _check_beams(torch.full((6, V), 2.0).to(dtype), torch.zeros(2, 3), 64)
    _check_beams(torch.full((6, V), -3.0).to(dtype), torch.tensor([[0.0, 0.0, 0.5]] * 2), 5,
                 torch.tensor([[True, False, True]] * 2), end_token=3)


# beam scores and logits [n] that differ but whose scores, in f64, do not: the lowest tokens, not the largest logits
ONE_SCORE = {
    "nearly 0": (-1.0, lambda n, g: 1e-20 * torch.arange(n)),
    "falling": (-2.0, lambda n, g: 1e-25 * torch.arange(n, 0, -1)),
    "subnormal": (0.0, lambda n, g: torch.randint(0, 200, (n,), generator=g) * 1e-44),
    "either sign": (-3.0, lambda n, g: 1e-30 * torch.randn(n, generator=g)),
    "a few larger": (-1.0, lambda n, g: torch.where(torch.rand(n, generator=g) < 4 / n, 1.0, 1e-20) * torch.rand(
        n, generator=g)),
    "neighbours": (-1e9, lambda n, g: 0.5 + 2.0 ** -24 * torch.randint(0, 40, (n,), generator=g)),
    "far below": (-1e12, lambda n, g: 1e-3 * torch.randn(n, generator=g)),
    "lowest": (-3.4e38, lambda n, g: 5 * torch.randn(n, generator=g)),
}


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [5, 3000, 8195, 70000])
@pytest.mark.parametrize("kind", sorted(ONE_SCORE))
def test_logits_that_differ_under_one_score(dtype, V, kind):
    g = _gen(V)
    score, make = ONE_SCORE[kind]
    logits = torch.stack([make(V, g).float() for _ in range(8)])
    logits[torch.rand(8, V, generator=g) < 0.2] = -math.inf
    logits = logits.to(dtype)
    for picks in (1, 4, 64):
        _check_beams(logits, torch.full((2, 4), score), picks)
        # (other beams' few candidates before and behind them, and some that have ended)
        some = logits.clone()
        some[[0, 6], 2:] = -math.inf
        scores = torch.full((2, 4), score)
        scores[0, 0] = scores[1, 2] = score / 2 + 1
        _check_beams(some, scores, picks, torch.tensor([[0, 1, 0, 0], [0, 0, 0, 1]]), end_token=V - 2, strided=True)


def test_one_score_in_place():
    V, R, W = 5000, 3, 4
    s = step().BeamSelector(V, W, W, R)
    logits = 1e-20 * torch.randn(R * W, V, generator=_gen(3))
    scores, ended = -torch.ones(R, W), torch.tensor([[0, 0, 0, 0], [1, 0, 0, 0], [0, 0, 1, 1]], dtype=torch.int32)
    want, tokens, parents = _select_by_hand(logits, scores, W, ended, 7)
    c, e, t, p = scores.cuda(), ended.cuda(), ended.clone().cuda(), ended.clone().cuda()
    s.select_into(logits.cuda(), c, c, t, p, ended=e, end_token=7, ended_out=e)
    s.sync()
    _same(t, tokens)
    _same(p, parents)
    _same(c, want.float())
    _same(e, (ended.gather(1, parents.long()) != 0) | (tokens == 7))


@pytest.mark.parametrize("V", [4, 9000, 70000])
def test_scores_below_the_range_of_f32(V):
    # masks of f32's lowest value: a beam that took one has nothing but its first token
    low = torch.finfo(F32).min
    logits = torch.full((6, V), -math.inf)
    logits[:, [0, 2, V - 1]] = torch.tensor([1.0, low, low])
    scores = torch.tensor([[low, 0.9 * low, -math.inf], [low, -1.0, low / 2]])
    for picks in (1, 3, 8, 64):
        total, tokens, parents = _select_by_hand(logits, scores, min(picks, 3 * V), None, -1)
        none = total.float() == -math.inf
        assert picks < 5 or bool((none & (total > -math.inf)).any())
        got = step().BeamSelector(V, 3, picks, 2).select(logits.cuda(), scores.cuda())
        n = total.shape[1]
        _same(got[0][:, :n], total.float())
        _same(got[1][:, :n], torch.where(none, -1, tokens))
        _same(got[2][:, :n], torch.where(none, -1, parents))
        assert bool((got[1][:, n:] == -1).all()) and bool((got[0][:, n:] == -math.inf).all())


def test_few_candidates():
    V = 30000
    logits = torch.full((4, V), -math.inf)
    logits[0, 29999], logits[0, 3], logits[1, 5] = 1.0, 1.0, -2.0     # beam 3 has none
    logits[3, :] = NAN
    scores = torch.tensor([[0.0, -1.0], [-math.inf, 0.0]])
    _check_beams(logits, scores, 6)
    _check_beams(logits, scores, 6, torch.tensor([[False, True], [True, False]]), end_token=0)


def test_infinite_logits_and_zeros_of_either_sign():
    g = _gen(1)
    logits = torch.randn(4, 20000, generator=g)
    logits[0, [5, 17000]] = math.inf
    logits[1, 9] = math.inf
    logits[2] = torch.where(torch.rand(20000, generator=g) < 0.5, 0.0, -0.0)
    logits[3, ::2] = NAN
    _check_beams(logits, torch.tensor([[0.0, -0.5], [0.0, -0.1]]), 9)


def test_candidates_all_from_one_place():
    # one thread's neighbours hold all the best of a slice, one slice of a beam all of a request
    V = 262144
    logits = torch.randn(64, V, generator=_gen(2))
    logits[3, 8192 * 5 + 40:8192 * 5 + 140] = torch.arange(100).float() + 20
    logits[40, 100::1024] += 50
    _check_beams(logits, torch.zeros(2, 32), 64)


def test_scores_that_cannot_be():
    logits, scores, _ = _beam_case(3, 4, 500, F32, 3, dead=0.0)
    scores[1, 2], scores[2, 0] = NAN, math.inf
    _check_beams(logits, scores, 4, status=N.ERR_ARGUMENT)


def test_beams_in_place_and_captured():
    R, W, V = 3, 4, 3000
    s = step().BeamSelector(V, W, W, R)
    logits = torch.empty(R * W, V, device="cuda")
    scores, ended = torch.empty(R, W, device="cuda"), torch.empty(R, W, dtype=torch.int32, device="cuda")
    tokens, parents = torch.empty_like(ended), torch.empty_like(ended)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        s.select_into(logits, scores, scores, tokens, parents, ended=ended, end_token=5, ended_out=ended)
    for i in range(4):
        x, c, e = _beam_case(R, W, V, F32, i)
        want = _check_beams(x, c, W, e, end_token=5)
        logits.copy_(x)
        scores.copy_(c)
        ended.copy_(e.int())
        graph.replay()
        s.sync()
        for got, w in zip((scores, tokens, parents), want):
            assert torch.equal(got, w)


@pytest.mark.parametrize("R,W,picks,V", [(20, 4, 8, 50257), (21, 4, 16, 50257), (32, 4, 64, 32000), (3, 8, 16, 129280)])
def test_beams_on_either_side_of_the_short_slices(R, W, picks, V):
    logits, scores, ended = _beam_case(R, W, V, BF16, R + W)
    _check_beams(logits, scores, picks, ended, end_token=7)


@pytest.mark.parametrize("first,n", [(0, 40), (250, 300), (2000, 100), (8190, 4), (15000, 1900)])
def test_few_logits_that_are_not_masked(first, n):
    logits, scores, _ = _beam_case(3, 4, 17000, F32, 11)
    logits[:, :first] = -math.inf
    logits[:, first + n:] = -math.inf
    for picks in (1, 5, 64):
        _check_beams(logits, scores, picks)


def test_beams_of_many_requests():
    logits, scores, ended = _beam_case(2500, 32, 60, F32, 4)
    _check_beams(logits, scores, 32, ended, end_token=1)


def test_beams_refuse():
    s = step().BeamSelector(100, 4, 8, 2)
    x, c = torch.zeros(8, 100, device="cuda"), torch.zeros(2, 4, device="cuda")
    out = lambda: [torch.empty(2, 8, dtype=t, device="cuda") for t in (F32, torch.int32, torch.int32)]
    ended = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    for end in (-1, 100, -2):
        assert _status(lambda: s.select_into(x, c, *out(), ended=ended, end_token=end)) == N.ERR_ARGUMENT
    assert _status(lambda: s.select_into(x, c, *out(), end_token=100)) == N.ERR_ARGUMENT
    more = torch.zeros(12, 100, device="cuda")
    three = [torch.empty(3, 8, dtype=t, device="cuda") for t in (F32, torch.int32, torch.int32)]
    assert _status(lambda: s.select_into(more, torch.zeros(3, 4, device="cuda"), *three)) == N.ERR_SHAPE
    for change in (dict(logits=x[:7]), dict(logits=x.bfloat16()), dict(logits=x[:, :99]), dict(scores=c[:1])):
        with pytest.raises(ValueError):
            s.select_into(**{**dict(logits=x, scores=c), **change}, scores_out=out()[0], tokens=out()[1],
                          parents=out()[2])


# ---- a run of them together -----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F8])
@pytest.mark.parametrize("captured", [False, True])
def test_a_beam_search_over_a_paged_cache(dtype, captured):
    """Prompts, then steps of plan, append, attention, selection and fork, held step by step to plain copies of
    every beam's keys and values; at the end all pages are free."""
    cm, R, W, page, heads, D, V, steps = cache_mod(), 3, 4, 4, 2, 32, 500, 9
    g, rows, blocks, pages = _gen(7), 12, 12, 200
    prompts = [5, 1, 8]
    pager = cm.Pager(pages, page, rows, blocks, 64)
    free, count = pager.new_stack()
    layer = _make_cache(pages, heads, page, D, dtype)
    att = cm.PagedAttention(4, layer, rows, blocks * page, F32)
    chooser = step().BeamSelector(V, W, W, R)
    tables = [torch.zeros(rows, blocks, dtype=torch.int32, device="cuda") for _ in range(2)]
    lengths = _i32([0] * rows)
    # the prompts go into the first row of each request
    added = [0] * rows
    added[::W] = prompts
    plan = pager.plan(lengths, _i32(added), tables[0], free, count, 64)
    k, v = (torch.randn(64, heads, D, generator=g).to(BF16) for _ in range(2))
    layer.append(k.cuda(), v.cuda(), plan.slots)
    lengths.copy_(plan.lengths)
    count.copy_(plan.count)

    def stored(x):       # what the cache holds of a row
        if dtype == BF16:
            return x.double()
        codes, e = _quantized(x)
        return codes.view(F8).double() * torch.exp2(e.double() - 127).unsqueeze(-1)

    beams = [([], []) for _ in range(rows)]
    at = 0
    for r, n in enumerate(prompts):
        beams[r * W] = tuple([stored(t[at + i]) for i in range(n)] for t in (k, v))
        at += n
    scores = torch.full((R, W), -math.inf, device="cuda")
    scores[:, 0] = 0.0
    tokens, parents = (torch.empty(R, W, dtype=torch.int32, device="cuda") for _ in range(2))
    logits = torch.empty(rows, V, device="cuda")
    q, kn, vn = (torch.empty(s, dtype=t, device="cuda") for s, t in (
        ((rows, 1, 4, D), F32), ((rows, heads, D), BF16), ((rows, heads, D), BF16)))
    out = torch.empty_like(q)
    step_plan = pager.new_plan(rows, 16)
    step_plan.lengths, step_plan.count = lengths, count

    def choose(i):       # selection and the pages that follow it, from tables i to the others
        chooser.select_into(logits, scores, scores, tokens, parents)
        pager.fork_into(parents, tables[i], lengths, free, count, tables[1 - i], lengths, count, [layer])

    def extend(i):       # a new token of every beam
        pager.plan_into(lengths, None, tables[i], free, count, step_plan)
        layer.append(kn, vn, step_plan.slots[:rows])
        att.attend_into(q, layer, tables[i], lengths, out)

    graphs = []
    if captured:
        torch.cuda.synchronize()
        for i in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                choose(i)
                extend(1 - i)
            graphs.append(graph)
    for n in range(steps):
        x, qh = 2 * torch.randn(rows, V, generator=g), torch.randn(rows, 1, 4, D, generator=g)
        kh, vh = (torch.randn(rows, heads, D, generator=g).to(BF16) for _ in range(2))
        for device, host in ((logits, x), (q, qh), (kn, kh), (vn, vh)):
            device.copy_(host)
        was = scores.cpu()
        if captured:
            graphs[n % 2].replay()
        else:
            choose(n % 2)
            extend(1 - n % 2)
        pager.sync()
        att.sync()
        _, want_tokens, want_parents = _select_by_hand(x, was, W, None, -1)
        _same(tokens, want_tokens)
        _same(parents, want_parents)
        beams = [tuple(list(t) for t in beams[r // W * W + p]) for r, p in enumerate(
            want_parents.flatten().tolist())]
        for r in range(rows):
            beams[r][0].append(stored(kh[r]))
            beams[r][1].append(stored(vh[r]))
        assert lengths.tolist() == [len(b[0]) for b in beams]
        c = Cached.__new__(Cached)
        c.lengths, c.queries, c.window, c.heads, c.q_heads, c.dim, c.rows = (
            lengths.tolist(), 1, 0, heads, 4, D, F32)
        c.scale, c.sinks, c.q = D ** -0.5, None, qh
        c.k, c.v = ([torch.stack(b[i], 1) for b in beams] for i in range(2))
        c.check(out)
        # no page is free twice, and none that is in use is free
        used = {p for t, m in zip(tables[1 - n % 2].tolist(), lengths.tolist()) for p in t[:-(-m // page)]}
        left = free[:count.item()].tolist()
        assert len(set(left)) == len(left) and not used & set(left) and len(used) + len(left) == pages
    pager.fork_into(torch.full_like(parents, -1), tables[steps % 2], lengths, free, count, tables[1 - steps % 2],
                    lengths, count)
    pager.sync()
    assert count.item() == pages and sorted(free.tolist()) == list(range(pages))


def test_a_decoder_layer_around_the_cache():
    """Rotated heads of a fused projection into the cache, attention over it, the output projection: one chain
    on one stream, against the same chain in 64 bits."""
    s, cm = step(), cache_mod()
    T, H, HK, D, page, hidden = 37, 8, 2, 64, 16, 256
    g = _gen(11)
    qkv = torch.randn(T, (H + 2 * HK) * D, generator=g).to(BF16)
    wq, wk = (1 + 0.1 * torch.randn(D, generator=g) for _ in range(2))
    inv_freq = 1e4 ** (-torch.arange(D // 2).float() / (D // 2))
    w = (torch.randn(hidden, H * D, generator=g) * 0.05).to(BF16)
    out_proj = s.AdaptedProjection(w.cuda(), None, 0, hidden, H * D, 8, BF16)
    pager = cm.Pager(40, page, 4, 8, 64)
    free, count = pager.new_stack()
    layer = cm.PagedCache.zeros(40, HK, page, D)
    tables = torch.zeros(1, 8, dtype=torch.int32, device="cuda")
    plan = pager.plan(_i32([0]), _i32([T]), tables, free, count, 64)
    dev = qkv.cuda()
    heads = lambda t, a, b: t[:, a * D:b * D].unflatten(1, (b - a, D))
    q, k = s.qk_norm_rope(heads(dev, 0, H), heads(dev, H, H + HK), wq.cuda(), wk.cuda(), plan.positions[:T],
                          inv_freq.cuda(), 1e-6)
    layer.append(k, heads(dev, H + HK, H + 2 * HK), plan.slots[:T])
    att = cm.PagedAttention(H, layer, 1, 128, BF16)
    last = att.attend(q[-1:].unsqueeze(0), layer, tables, plan.lengths)
    got = out_proj.forward(last.view(1, H * D)).cpu().double()
    # from the rotated heads as they were rounded: attention's rounding and the projection's
    qd, kd = q[-1].cpu().double(), k.cpu().double().repeat_interleave(H // HK, 1)
    vd = heads(qkv, H + HK, H + 2 * HK).double().repeat_interleave(H // HK, 1)
    p = torch.softmax((qd.unsqueeze(0) * kd).sum(2) / math.sqrt(D), 0)
    mid = (p.unsqueeze(2) * vd).sum(0).flatten()
    off = 2.0 ** -8 * mid.abs() + 2.0 ** -14 * (p.unsqueeze(2) * vd.abs()).sum(0).flatten()
    want = w.double() @ mid
    size = w.double().abs()
    tol = size @ off + 2 * U * (H * D / 32 + 64) * (size @ mid.abs())
    tol = tol + 2.0 ** -8 * (want.abs() + tol)
    assert bool(((got[0] - want).abs() <= tol).all())
