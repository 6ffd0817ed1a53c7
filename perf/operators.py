"""The steps of a decoder on either side of the MoE block call, as they are timed: projections with
low-rank adapters of many requests, norms of queries and keys with the position rotation, and
sampling from logits.

Each has a plain form in elementary torch operations (``own`` false), the framework's call (``own``
true) and its definition in 64 bits (``exact``).
"""

import math

import numpy as np
import torch

own = False

FMT = {"bf16": 0, "mxfp4": 1, "mxfp8": 2}
DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


# ---- cases -------------------------------------------------------------------------------------

def _project(name, fmt, tokens, rows, cols, slots, rank, order="mixed", idle=0.0, dtype="bf16"):
    """tokens rows of `cols` values times a [rows, cols] matrix; `slots` adapters of up to `rank`;
    a share `idle` of the rows has no adapter."""
    return {"name": name, "op": "project", "fmt": fmt, "tokens": tokens, "rows": rows, "cols": cols,
            "slots": slots, "rank": rank, "order": order, "idle": idle, "dtype": dtype}


def _rotate(name, tokens, q_heads, k_heads, dim, rotary, interleaved=False, fused=True,
            reach=40000, dtype="bf16"):
    return {"name": name, "op": "rotate", "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads,
            "dim": dim, "rotary": rotary, "interleaved": interleaved, "fused": fused,
            "reach": reach, "dtype": dtype}


def _sample(name, rows, vocab, filters="mixed", dtype="f32"):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "filters": filters,
            "dtype": dtype}


def listed():
    return [
        # one token of one request through a BF16 output projection: launches and latency
        _project("project_1", "bf16", 1, 2048, 4096, 4, 16),
        # a decode batch of 24 requests, most with an adapter of their own, MXFP8 matrix
        _project("project_mxfp8_24", "mxfp8", 24, 9232, 6144, 20, 64, idle=0.2),
        # a short prompt beside decoding requests, f32 rows as the layer call leaves them
        _project("project_f32_131", "mxfp4", 131, 4096, 7168, 6, 32, idle=0.4, dtype="f32"),
        # a chunked prefill of many short prompts, one adapter per prompt, in order of request
        _project("project_1000", "mxfp4", 1000, 6144, 4096, 17, 24, order="sorted", idle=0.1),
        # the largest prefill step: 4096 tokens of a few requests, BF16 matrix
        _project("project_4096", "bf16", 4096, 7168, 7168, 8, 16, order="sorted", idle=0.2),
        # one token's heads, rotation of a quarter of the 256 values
        _rotate("rotate_1", 1, 16, 2, 256, 64),
        # a long decode batch over far positions, all values rotated, pairs of neighbours
        _rotate("rotate_515", 515, 64, 8, 128, 128, interleaved=True, reach=1 << 24),
        # a long prompt's chunk, f32 rows
        _rotate("rotate_f32_2000", 2000, 40, 8, 80, 80, dtype="f32", fused=False),
        # the largest: every head of a 32768-token prefill step
        _rotate("rotate_32768", 32768, 16, 2, 256, 64),
        # one token's choice from the whole vocabulary
        _sample("sample_1", 1, 129280),
        # a decode batch over a vocabulary of odd size, BF16 logits
        _sample("sample_bf16_37", 37, 50257, dtype="bf16"),
        # the largest: every request of a large decode batch
        _sample("sample_256", 256, 129280),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("project", "project", "rotate", "sample"))
    if op == "project":
        dtype = rng.choice(("bf16", "bf16", "f32"))
        rows, cols = 16 * _spread(rng, 32, 1024), 128 * _spread(rng, 8, 64)
        most = min(4096, (4096 * 7168 * 7168) // (rows * cols * (4 if dtype == "f32" else 1)))
        c = _project("", rng.choice(sorted(FMT)), _spread(rng, 1, most), rows, cols,
                     rng.randint(1, 32), rng.choice((4, 7, 8, 16, 24, 32, 64)),
                     rng.choice(("mixed", "sorted")), round(rng.choice((0.0, rng.random())), 2),
                     dtype)
    elif op == "rotate":
        dim = rng.choice((64, 80, 96, 128, 192, 256))
        rotary = rng.choice((dim, dim, dim // 2, dim // 4))
        heads = rng.choice((8, 14, 16, 32, 40, 64))
        k_heads = rng.choice((1, 2, 4, 8))
        most = min(32768, 32768 * 18 * 256 // ((heads + k_heads) * dim * 2))
        c = _rotate("", _spread(rng, 1, most), heads, k_heads, dim, rotary,
                    rng.random() < 0.4, rng.random() < 0.7, rng.choice((4096, 40000, 1 << 20)),
                    rng.choice(("bf16", "bf16", "f32")))
    else:
        vocab = rng.choice((32000, 50257, 64000 + rng.randint(0, 999), 129280))
        c = _sample("", _spread(rng, 1, 256), vocab, rng.choice(("mixed", "top_p", "none")),
                    rng.choice(("f32", "f32", "bf16")))
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _matrix(g, fmt, rows, cols):
    """(data, scales) in the checkpoint layout, weights of about 0.02 standard deviation."""
    if fmt == "bf16":
        return _normal(g, rows, cols).mul_(0.02).to(torch.bfloat16), None
    if fmt == "mxfp4":
        data = torch.randint(0, 256, (rows, cols // 2), generator=g, dtype=torch.uint8,
                             device="cuda")
        low, high = 118, 122
    else:
        z = _normal(g, rows, cols).mul_(120.0).clamp_(-448.0, 448.0)
        data = z.to(torch.float8_e4m3fn).view(torch.uint8)
        low, high = 113, 116
    scales = torch.randint(low, high, (rows, cols // 32), generator=g, dtype=torch.uint8,
                           device="cuda")
    return data, scales


def _ranks(case):
    """The adapters' ranks: up to `rank`, unlike each other as tenants' adapters are."""
    return [max(1, case["rank"] // (1 + i % 3)) for i in range(case["slots"])]


def _prepare_project(case, g):
    T, N, K = case["tokens"], case["rows"], case["cols"]
    dtype = DTYPE[case["dtype"]]
    data, scales = _matrix(g, case["fmt"], N, K)
    x = _normal(g, T, K).to(dtype)
    ranks = _ranks(case)
    a = [(_normal(g, r, K) * K ** -0.5).to(torch.bfloat16) for r in ranks]
    b = [(_normal(g, N, r) * 0.3).to(torch.bfloat16) for r in ranks]
    alphas = [0.5 + 0.25 * (i % 5) for i in range(case["slots"])]
    ids = torch.randint(0, case["slots"], (T,), generator=g, dtype=torch.int32, device="cuda")
    idle = torch.rand(T, generator=g, device="cuda") < case["idle"]
    ids = torch.where(idle, torch.full_like(ids, -1), ids)
    if case["order"] == "sorted":
        ids = ids.sort().values
    state = {"case": case, "x": x, "ids": ids, "data": data, "scales": scales, "a": a, "b": b,
             "alphas": alphas}
    if own:
        from urbilateria_amd import step
        p = step.AdaptedProjection(data, scales, FMT[case["fmt"]], N, K, max_tokens=T, dtype=dtype,
                                   slots=case["slots"], max_rank=max(ranks))
        for i in range(case["slots"]):
            p.set_adapter(i, a[i], b[i], alphas[i])
        state["projection"] = p
        state["y"] = torch.empty((T, N), dtype=dtype, device="cuda")
    else:
        # every adapter's rows under one another, as a program without the operator keeps them
        owner = torch.tensor([i for i, r in enumerate(ranks) for _ in range(r)], device="cuda")
        state.update(down=torch.cat(a), up=torch.cat(b, 1), owner=owner,
                     alpha=torch.tensor(alphas, device="cuda")[owner])
    return state


def _prepare_rotate(case, g):
    T, D, dtype = case["tokens"], case["dim"], DTYPE[case["dtype"]]
    hq, hk = case["q_heads"], case["k_heads"]
    if case["fused"]:
        # one buffer of queries, keys and values per token, as a fused projection writes it
        qkv = _normal(g, T, (hq + 2 * hk) * D).mul_(2.0).to(dtype)
        q = qkv[:, :hq * D].unflatten(1, (hq, D))
        k = qkv[:, hq * D:(hq + hk) * D].unflatten(1, (hk, D))
    else:
        q = _normal(g, T, hq, D).to(dtype)
        k = _normal(g, T, hk, D).to(dtype)
    wq, wk = _normal(g, D) * 0.1, _normal(g, D) * 0.1
    start = torch.randint(0, case["reach"], (1,), generator=g, device="cuda")
    positions = start + torch.arange(T, device="cuda")
    half = case["rotary"] // 2
    inv_freq = (1e6 ** (-torch.arange(half, dtype=torch.float64) / half)).float().cuda()
    state = {"case": case, "q": q, "k": k, "wq": wq, "wk": wk, "positions": positions,
             "inv_freq": inv_freq}
    if own:
        state["out"] = (torch.empty((T, hq, D), dtype=dtype, device="cuda"),
                        torch.empty((T, hk, D), dtype=dtype, device="cuda"))
    return state


def _prepare_sample(case, g):
    T, V = case["rows"], case["vocab"]
    # a bulk of unlikely tokens and a tail of likely ones, more or less sharp by row; some tokens
    # masked, as a grammar masks them
    sharp = 1.0 + 2.0 * torch.rand((T, 1), generator=g, device="cuda")
    z = _normal(g, T, V)
    logits = sharp * z + 0.5 * z.clamp(min=2.5).sub_(2.5).square_()
    logits[torch.rand((T, V), generator=g, device="cuda") < 0.02] = -math.inf
    logits = logits.to(DTYPE[case["dtype"]])
    pick = lambda v: torch.tensor(v, device="cuda")[
        torch.randint(0, len(v), (T,), generator=g, device="cuda")]
    kind = case["filters"]
    temperature = pick([0.6, 0.8, 1.0, 1.3] + ([0.0] if kind == "mixed" else []))
    top_k = pick([0, 0, 20, 50, 400] if kind == "mixed" else [0]).int()
    top_p = pick([1.0] if kind == "none" else [0.9, 0.95, 0.99] + [1.0] * (kind == "mixed"))
    min_p = pick([0.0, 0.0, 0.02, 0.1] if kind == "mixed" else [0.0])
    uniform = torch.rand(T, generator=g, device="cuda")
    state = {"case": case, "logits": logits, "temperature": temperature, "top_k": top_k,
             "top_p": top_p, "min_p": min_p, "uniform": uniform}
    if own:
        from urbilateria_amd import step
        state["sampler"] = step.Sampler(V, max_rows=T, dtype=logits.dtype)
        state["out"] = (torch.empty(T, dtype=torch.int32, device="cuda"),
                        torch.empty(T, dtype=torch.float32, device="cuda"))
    return state


def prepare(case, seed):
    make = {"project": _prepare_project, "rotate": _prepare_rotate, "sample": _prepare_sample}
    return make[case["op"]](case, _generator(seed))


# ---- one pass ----------------------------------------------------------------------------------

def _e2m1(codes):
    """Values of E2M1 codes 0..15: sign, two exponent bits, one mantissa bit."""
    m, e = (codes & 1).float(), (codes >> 1 & 3).float()
    v = torch.where(e == 0, m * 0.5, (1 + 0.5 * m) * torch.exp2(e - 1))
    return torch.where(codes > 7, -v, v)


def _weights(data, scales, fmt, rows, cols):
    """The matrix in 32 bits."""
    if fmt == "bf16":
        return data.float()
    if fmt == "mxfp4":
        v = _e2m1(torch.stack((data & 15, data >> 4), -1)).view(rows, cols // 32, 32)
    else:
        v = data.view(torch.float8_e4m3fn).float().view(rows, cols // 32, 32)
    return (v * torch.exp2(scales.float() - 127).unsqueeze(-1)).view(rows, cols)


def _plain_project(s):
    case = s["case"]
    x = s["x"].float()
    w = _weights(s["data"], s["scales"], case["fmt"], case["rows"], case["cols"])
    u = x @ s["down"].float().T
    u = torch.where(s["owner"] == s["ids"].unsqueeze(1), u * s["alpha"], 0.0)
    return (x @ w.T + u @ s["up"].float().T).to(s["x"].dtype)


def _plain_heads(h, w, cos, sin, interleaved):
    x = h.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1 + w)
    r = 2 * cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., r:]), -1).to(h.dtype)


def _plain_rotate(s):
    # in 64 bits: an angle of a far position has no fraction left in 32
    angle = s["positions"].double().unsqueeze(1) * s["inv_freq"].double()
    cos, sin = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)
    turn = s["case"]["interleaved"]
    return (_plain_heads(s["q"], s["wq"], cos, sin, turn),
            _plain_heads(s["k"], s["wk"], cos, sin, turn))


def _plain_sample(s):
    # in 64 bits: a border between two tokens decides which of them is drawn
    x = s["logits"].double()
    x = torch.where(x.isnan(), -math.inf, x)
    T, V = x.shape
    top = x.max(1, keepdim=True).values
    empty, greedy = (top == -math.inf).squeeze(1), s["temperature"] <= 0
    tau = torch.where(greedy, 1.0, s["temperature"]).double().unsqueeze(1)
    e = torch.where(x == top, 0.0, (x - top) / tau).exp()
    order = x.sort(dim=1, descending=True, stable=True).indices
    es = e.gather(1, order)
    mass = es.cumsum(1)
    before = torch.cat((torch.zeros_like(mass[:, :1]), mass[:, :-1]), 1)
    place = torch.arange(V, device=x.device)
    n = torch.where(s["top_k"] <= 0, V, s["top_k"]).clamp(max=V).long().unsqueeze(1)
    p = s["top_p"].double().unsqueeze(1)
    keep = (place < n) & (es >= s["min_p"].double().unsqueeze(1))
    keep &= (p >= 1) | (before < p * mass.gather(1, n - 1))
    keep[:, 0] = True
    w = torch.zeros_like(e).scatter_(1, order, torch.where(keep, es, 0.0))
    cdf = w.cumsum(1)
    total = cdf[:, -1:]
    ids = (cdf <= s["uniform"].double().unsqueeze(1) * total).sum(1)
    first = torch.where(x == top, place, V).min(1).values
    ids = torch.where(greedy, first, ids).clamp(max=V - 1)
    prob = torch.where(greedy, 1.0, (w.gather(1, ids.unsqueeze(1)) / total).squeeze(1))
    ids = torch.where(empty, -1, ids)
    return ids.int(), torch.where(empty, 0.0, prob).float()


def run(state):
    op = state["case"]["op"]
    if not own:
        plain = {"project": _plain_project, "rotate": _plain_rotate, "sample": _plain_sample}
        return plain[op](state)
    if op == "project":
        state["projection"].forward_into(state["x"], state["y"], state["ids"])
        return state["y"]
    if op == "rotate":
        from urbilateria_amd import step
        return step.qk_norm_rope(state["q"], state["k"], state["wq"], state["wk"],
                                 state["positions"], state["inv_freq"], eps=EPS,
                                 zero_centered=True, interleaved=state["case"]["interleaved"],
                                 out=state["out"])
    ids, prob = state["out"]
    state["sampler"].sample_into(state["logits"], state["uniform"], ids, prob,
                                 temperature=state["temperature"], top_k=state["top_k"],
                                 top_p=state["top_p"], min_p=state["min_p"])
    return ids, prob


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    if case["op"] == "project":
        T, N, K = case["tokens"], case["rows"], case["cols"]
        size = 2 if case["dtype"] == "bf16" else 4
        weight = {"bf16": N * K * 2, "mxfp4": N * K // 2 + N * K // 32,
                  "mxfp8": N * K + N * K // 32}[case["fmt"]]
        ranks = _ranks(case)
        busy = T * (1.0 - case["idle"])
        # adapters that some row uses, if rows choose among the slots evenly
        used = 1.0 - (1.0 - 1.0 / case["slots"]) ** busy
        rank = sum(ranks) / len(ranks)
        return {"bytes": weight + int(used * sum(ranks) * (N + K) * 2) + T * (N + K) * size,
                "flops": 2 * T * N * K + int(2 * busy * rank * (N + K))}
    if case["op"] == "rotate":
        n = case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        return {"bytes": 2 * n * (2 if case["dtype"] == "bf16" else 4), "flops": 6 * n}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * (2 if case["dtype"] == "bf16" else 4), "flops": 4 * n}


# ---- the definitions in 64 bits ------------------------------------------------------------------

def _exact_project(s):
    case = s["case"]
    N, K = case["rows"], case["cols"]
    if case["fmt"] == "bf16":
        w = s["data"].double()
    else:
        if case["fmt"] == "mxfp4":
            table = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
            codes = torch.empty((N, K), dtype=torch.long, device="cuda")
            codes[:, 0::2], codes[:, 1::2] = s["data"] % 16, s["data"] // 16
        else:
            table = [(c & 7) / 8 * 2.0 ** -6 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7)
                     for c in range(128)]
            codes = s["data"].long()
        table = torch.tensor(table + [-v for v in table], dtype=torch.float64, device="cuda")
        w = table[codes]
        w *= torch.pow(2.0, s["scales"].double() - 127).repeat_interleave(32, 1)
    x = s["x"].double()
    y = x @ w.T
    for i, (a, b) in enumerate(zip(s["a"], s["b"])):
        rows = (s["ids"] == i).nonzero().squeeze(1)
        y[rows] += s["alphas"][i] * ((x[rows] @ a.double().T) @ b.double().T)
    return y


def _exact_heads(h, w, turn, interleaved):
    x = h.double()
    x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * (w.double() + 1)
    r = 2 * turn.shape[-1]
    out = x.clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2),
                                                                          slice(r // 2, r))
    z = torch.complex(x[..., first], x[..., second]) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_rotate(s):
    angle = torch.outer(s["positions"].double(), s["inv_freq"].double())
    turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)
    return (_exact_heads(s["q"], s["wq"], turn, s["case"]["interleaved"]),
            _exact_heads(s["k"], s["wk"], turn, s["case"]["interleaved"]))


def _exact_sample(s):
    host = {n: s[n].double().cpu().numpy() for n in
            ("logits", "temperature", "top_k", "top_p", "min_p", "uniform")}
    ids, probs = [], []
    for t, row in enumerate(host["logits"]):
        at = np.flatnonzero(row > -np.inf)         # NaN and -inf are never drawn
        if not at.size:
            ids.append(-1)
            probs.append(0.0)
            continue
        rank = at[np.lexsort((at, -row[at]))]
        if host["temperature"][t] <= 0:
            ids.append(rank[0])
            probs.append(1.0)
            continue
        with np.errstate(invalid="ignore"):
            gap = row[rank] - row[rank[0]]
        e = np.exp(np.where(row[rank] == row[rank[0]], 0.0, gap / host["temperature"][t]))
        n = int(host["top_k"][t])
        n = e.size if n <= 0 else min(n, e.size)
        if host["top_p"][t] < 1:
            mass = np.cumsum(e[:n])
            n = 1 + int(np.searchsorted(mass[:-1], host["top_p"][t] * mass[-1], side="left"))
        n = max(1, min(n, int(np.count_nonzero(e >= host["min_p"][t]))))
        kept = np.argsort(rank[:n])
        mass = np.cumsum(e[kept])
        i = min(int(np.searchsorted(mass, host["uniform"][t] * mass[-1], side="right")), n - 1)
        ids.append(rank[kept[i]])
        probs.append(e[kept[i]] / mass[-1])
    return (torch.tensor(ids, dtype=torch.int32, device="cuda"),
            torch.tensor(probs, dtype=torch.float64, device="cuda"))


def exact(case, seed):
    global own
    mode, own = own, False     # the inputs alone
    try:
        state = prepare(case, seed)
    finally:
        own = mode
    return {"project": _exact_project, "rotate": _exact_rotate, "sample": _exact_sample}[
        case["op"]](state)
