"""The calls on a paged key-value cache, as they are timed: planning a step's pages and slots from the
requests' lengths, writing keys and values into the pages, attention of each request's new tokens over
them, the choice of beam search, and the pages that follow its beams.

Each has a plain form in elementary torch operations (``own`` false), the framework's call (``own``
true) and, where it computes numbers, its definition in 64 bits (``exact``).
"""

import math

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "f32": torch.float32}
F8 = torch.float8_e4m3fn


# ---- cases -------------------------------------------------------------------------------------

def _plan(name, requests, most, context, page):
    """`requests` of up to `context` cached tokens, each with 1 .. `most` new ones while the step
    has room for them (half of what all could bring)."""
    return {"name": name, "op": "plan", "requests": requests, "most": most, "context": context,
            "page": page}


def _append(name, tokens, heads, dim, page, cache="bf16", dtype="bf16", runs=True):
    """`tokens` rows into pages; runs: in order within a page, as a prompt's are."""
    return {"name": name, "op": "append", "tokens": tokens, "heads": heads, "dim": dim,
            "page": page, "cache": cache, "dtype": dtype, "runs": runs}


def _attend(name, requests, longest, q_heads, heads, dim, page, cache="bf16", dtype="bf16",
            drafted=1, window=0, sinks=False, ragged=True):
    return {"name": name, "op": "attend", "requests": requests, "longest": longest,
            "q_heads": q_heads, "heads": heads, "dim": dim, "page": page, "cache": cache,
            "dtype": dtype, "drafted": drafted, "window": window, "sinks": sinks,
            "ragged": ragged}


def _beam(name, requests, width, picks, vocab, dtype="f32"):
    return {"name": name, "op": "beam", "requests": requests, "width": width, "picks": picks,
            "vocab": vocab, "dtype": dtype}


def _fork(name, requests, width, prompt, grown, layers, heads, dim, page, cache="bf16"):
    """Beams that share a prompt of up to `prompt` tokens and have grown `grown` of their own."""
    return {"name": name, "op": "fork", "requests": requests, "width": width, "prompt": prompt,
            "grown": grown, "layers": layers, "heads": heads, "dim": dim, "page": page,
            "cache": cache}


def listed():
    return [
        # a decode step: one new token for each of 200 requests, some at the end of a page
        _plan("plan_200", 200, 1, 8191, 16),
        # a large chunked prefill: prompts and parts of prompts beside decoding requests
        _plan("plan_prefill_1500", 1500, 400, 5000, 64),
        # the new keys and values of a decode batch, each into another page
        _append("append_33", 33, 2, 256, 16, runs=False),
        # an 8190-token prefill step, quantized on its way into the cache
        _append("append_f8_8190", 8190, 8, 128, 64, cache="f8"),
        # one token of one request of 1000 tokens: launches and latency
        _attend("attend_1", 1, 1000, 16, 2, 256, 16, ragged=False),
        # three drafted tokens of 24 requests, f32 rows, a sliding window with sinks
        _attend("attend_f32_24", 24, 6000, 40, 8, 80, 24, dtype="f32", drafted=3, window=2000,
                sinks=True),
        # one request over a very long cache of E4M3
        _attend("attend_f8_131071", 1, 131071, 64, 8, 128, 64, cache="f8", ragged=False),
        # the largest: a full decode batch of ragged lengths
        _attend("attend_200", 200, 12000, 32, 8, 128, 16),
        # one request's four beams over a vocabulary of odd size
        _beam("beam_1", 1, 4, 8, 50257, dtype="bf16"),
        # a batch of beam searches over a large vocabulary
        _beam("beam_32", 32, 8, 16, 129280),
        # the beams of one request, a few layers' caches
        _fork("fork_1", 1, 4, 900, 37, 2, 2, 256, 16),
        # the beams of a batch
        _fork("fork_32", 32, 8, 2500, 260, 6, 4, 128, 64),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("plan", "append", "attend", "attend", "attend", "beam", "fork"))
    page = rng.choice((16, 16, 24, 32, 64, 128))
    cache = rng.choice(("bf16", "bf16", "f8"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    dim = rng.choice((64, 80, 96, 128, 128, 192, 256))
    heads = rng.choice((1, 2, 4, 8, 8))
    if op == "plan":
        requests = _spread(rng, 1, 1500)
        c = _plan("", requests, _spread(rng, 1, 400), _spread(rng, 16, 8000), page)
    elif op == "append":
        tokens = _spread(rng, 1, max(2, 8190 * 1024 // (heads * dim)) // 2)
        c = _append("", tokens, heads, dim, page, cache, dtype, rng.random() < 0.6)
    elif op == "attend":
        longest = _spread(rng, 30, 100000)
        ragged = rng.random() < 0.8
        most = 200 * 12000 * 1024 // (longest * heads * dim * (2 if ragged else 10))
        c = _attend("", _spread(rng, 1, max(1, min(200, most))), longest,
                    heads * rng.choice((1, 4, 5, 7, 8, 16)), heads, dim, page, cache, dtype,
                    rng.choice((1, 1, 1, 2, 5)), rng.choice((0, 0, 0, 128, 1000)),
                    rng.random() < 0.2, ragged)
    elif op == "beam":
        width = rng.choice((2, 4, 5, 8, 16))
        c = _beam("", _spread(rng, 1, 256 // width), width, rng.choice((width, 2 * width)),
                  rng.choice((32000, 50257, 64000 + rng.randint(0, 999), 129280)), dtype)
    else:
        width = rng.choice((2, 4, 5, 8))
        c = _fork("", _spread(rng, 1, 32), width, _spread(rng, 20, 2500), _spread(rng, 1, 260),
                  rng.randint(1, 6), min(heads, 4), min(dim, 128), page, cache)
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _whole(g, low, high, n):
    """n numbers of low .. high."""
    return torch.randint(low, high + 1, (n,), generator=g, device="cuda")


def _lengths(g, low, high, n):
    """n lengths, spread over their logarithm."""
    u = torch.rand(n, generator=g, device="cuda")
    return (math.log(low) + u * math.log(high / low)).exp().round().long().clamp(low, high)


def _order(g, n):
    return torch.randperm(n, generator=g, device="cuda")


def _pages(g, kind, pages, heads, page, dim):
    """(k, v, their scales or None) of a cache that holds something everywhere, as one in use."""
    out, scales = [], []
    for _ in range(2):
        if kind == "bf16":
            t = torch.empty((pages, heads, page, dim), dtype=torch.bfloat16, device="cuda")
            t.normal_(generator=g)
            scales.append(None)
        else:
            t = torch.empty((pages, heads, page, dim), dtype=F8, device="cuda")
            for i in range(0, pages, 1024):     # (in parts: the 32-bit values take four times the room)
                part = t[i:i + 1024]
                part.copy_(_normal(g, *part.shape).mul_(120.0).clamp_(-448.0, 448.0))
            scales.append(torch.randint(117, 122, (pages, heads, page), generator=g,
                                        dtype=torch.uint8, device="cuda"))
        out.append(t)
    return (*out, *scales)


def _cache(case, g, pages):
    state = dict(zip(("k", "v", "k_scales", "v_scales"),
                     _pages(g, case["cache"], pages, case["heads"], case["page"], case["dim"])))
    if own:
        from urbilateria_amd import cache
        state["cache"] = cache.PagedCache(**state)
    return state


def _prepare_plan(case, g):
    R, P = case["requests"], case["page"]
    have = _whole(g, 0, case["context"], R)
    added = _whole(g, 1, case["most"], R)
    room = R * (1 + case["most"]) // 2
    added = added.minimum((room - (added.cumsum(0) - added)).clamp(min=0))
    tokens = (room + 63) // 64 * 64       # a padded batch
    held = (have + P - 1) // P
    width = (case["context"] + case["most"] + P - 1) // P
    pages = R * width + 100
    used = int(held.sum())
    ids = _order(g, pages).int()
    tables = torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    tables[torch.arange(width, device="cuda") < held.unsqueeze(1)] = ids[:used]
    free = torch.zeros(pages, dtype=torch.int32, device="cuda")
    free[:pages - used] = ids[used:]
    count = torch.tensor([pages - used], dtype=torch.int32, device="cuda")
    state = {"case": case, "lengths": have.int(), "added": added.int(), "tables": tables,
             "free": free, "count": count, "tokens": tokens}
    if own:
        from urbilateria_amd import cache
        state["pager"] = cache.Pager(pages, P, max_rows=R, max_blocks=width, max_tokens=tokens)
        state["plan"] = state["pager"].new_plan(R, tokens)
    return state


def _prepare_append(case, g):
    T, H, D, P = case["tokens"], case["heads"], case["dim"], case["page"]
    pages = (T + P - 1) // P + 40 if case["runs"] else T + 40
    t, ids = torch.arange(T, device="cuda"), _order(g, pages)
    slots = ids[t // P] * P + t % P if case["runs"] else ids[t] * P + _whole(g, 0, P - 1, T)
    slots[torch.rand(T, generator=g, device="cuda") < 0.02] = -1     # a batch's padding
    # queries, keys and values of a token in one row, as a fused projection writes them
    qkv = _normal(g, T, 6 * H * D).to(DTYPE[case["dtype"]])
    state = {"case": case, "slots": slots,
             "rows_k": qkv[:, 4 * H * D:5 * H * D].unflatten(1, (H, D)),
             "rows_v": qkv[:, 5 * H * D:].unflatten(1, (H, D))}
    state.update(_cache(case, g, pages))
    return state


def _prepare_attend(case, g):
    R, P, n = case["requests"], case["page"], case["drafted"]
    longest = max(case["longest"], n)
    lengths = _lengths(g, n, longest, R) if case["ragged"] else torch.full((R,), longest,
                                                                           device="cuda")
    if case["ragged"]:
        lengths[0] = longest
        if R > 4:
            lengths[R // 2] = 0           # a row of a padded batch
    held = (lengths + P - 1) // P
    width = (longest + P - 1) // P
    used = int(held.sum())
    tables = torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    tables[torch.arange(width, device="cuda") < held.unsqueeze(1)] = _order(g, used + 7)[:used].int()
    dtype = DTYPE[case["dtype"]]
    q = (1.5 * _normal(g, R, n, case["q_heads"], case["dim"])).to(dtype)
    sinks = _normal(g, case["q_heads"]) if case["sinks"] else None
    state = {"case": case, "q": q, "tables": tables, "lengths": lengths.int(), "sinks": sinks}
    state.update(_cache(case, g, used + 7))
    if own:
        from urbilateria_amd import cache
        state["attention"] = cache.PagedAttention(
            case["q_heads"], state["cache"], max_rows=R, max_length=longest, dtype=dtype,
            queries=n, window=case["window"])
        state["out"] = torch.empty_like(q)
        state["lse"] = torch.empty((R, n, case["q_heads"]), device="cuda")
    return state


def _prepare_beam(case, g):
    R, W, V = case["requests"], case["width"], case["vocab"]
    sharp = 1.0 + 2.0 * torch.rand((R * W, 1), generator=g, device="cuda")
    z = _normal(g, R * W, V)
    logits = sharp * z + 0.5 * z.clamp(min=2.5).sub_(2.5).square_()
    logits[torch.rand((R * W, V), generator=g, device="cuda") < 0.02] = -math.inf
    # beams of one search lie close together; some searches have just begun, some beams have ended
    scores = -20.0 * torch.rand((R, 1), generator=g, device="cuda") - 3.0 * torch.rand(
        (R, W), generator=g, device="cuda")
    begun = torch.rand((R, 1), generator=g, device="cuda") < 0.8
    first = torch.arange(W, device="cuda") == 0
    scores = torch.where(begun | first, scores, -math.inf)
    ended = (torch.rand((R, W), generator=g, device="cuda") < 0.1).int()
    state = {"case": case, "logits": logits.to(DTYPE[case["dtype"]]), "scores": scores,
             "ended": ended, "end_token": V - 1}
    if own:
        from urbilateria_amd import step
        N = case["picks"]
        state["selector"] = step.BeamSelector(V, W, N, max_requests=R, dtype=DTYPE[case["dtype"]])
        state["out"] = (torch.empty((R, N), device="cuda"),
                        torch.empty((R, N), dtype=torch.int32, device="cuda"),
                        torch.empty((R, N), dtype=torch.int32, device="cuda"))
    return state


def _prepare_fork(case, g):
    R, W, P = case["requests"], case["width"], case["page"]
    prompt = _lengths(g, min(20, case["prompt"]), case["prompt"], R).unsqueeze(1)
    lengths = (prompt + case["grown"]).expand(R, W)
    width = (case["prompt"] + case["grown"] + P - 1) // P + 1
    col = torch.arange(width, device="cuda")
    # the whole pages of the prompt are one for all beams, the later ones each beam's
    shared = (col < prompt // P).unsqueeze(1).expand(R, W, width)
    held = col < ((lengths + P - 1) // P).unsqueeze(2)
    first = (torch.arange(W, device="cuda") == 0).view(1, W, 1)
    owned = held & (~shared | first)
    used = int(owned.sum())
    own_blocks = (case["grown"] + P - 1) // P + 1
    pages = R * (case["prompt"] // P + W * own_blocks) + R * W + 9
    ids = _order(g, pages).int()
    tables = torch.full((R, W, width), -1, dtype=torch.int32, device="cuda")
    tables[owned] = ids[:used]
    tables = torch.where(held & shared, tables[:, :1], tables)
    free = torch.zeros(pages, dtype=torch.int32, device="cuda")
    free[:pages - used] = ids[used:]
    # good beams have several children
    parents = (W * torch.rand((R, W), generator=g, device="cuda") ** 2).int().clamp(max=W - 1)
    state = {"case": case, "parents": parents, "tables": tables.view(R * W, width),
             "lengths": lengths.reshape(-1).int(), "free": free,
             "count": torch.tensor([pages - used], dtype=torch.int32, device="cuda"),
             "caches": [_cache(case, g, pages) for _ in range(case["layers"])]}
    if own:
        from urbilateria_amd import cache
        state["pager"] = cache.Pager(pages, P, max_rows=R * W, max_blocks=width)
        state["layers"] = [c["cache"] for c in state["caches"]]
        state["out"] = (torch.full_like(state["tables"], -1),
                        torch.empty_like(state["lengths"]), torch.empty_like(state["count"]))
    return state


def prepare(case, seed):
    make = {"plan": _prepare_plan, "append": _prepare_append, "attend": _prepare_attend,
            "beam": _prepare_beam, "fork": _prepare_fork}
    return make[case["op"]](case, _generator(seed))


# ---- one pass ----------------------------------------------------------------------------------

def _plain_plan(s):
    P, T = s["case"]["page"], s["tokens"]
    have, added = s["lengths"].long(), s["added"].long()
    held = (have + P - 1) // P
    need = (have + added + P - 1) // P - held
    taken = need.cumsum(0)
    ends = added.cumsum(0)
    starts = torch.cat((torch.zeros_like(ends[:1]), ends))
    # the pages on top of the stack, in the order of the requests
    tables, col = s["tables"], torch.arange(s["tables"].shape[1], device="cuda")
    nth = (taken - need - held).unsqueeze(1) + col
    new = (col >= held.unsqueeze(1)) & (col < (held + need).unsqueeze(1))
    top = s["count"].long() - 1
    tables = torch.where(new, s["free"][(top - nth).clamp(min=0)], tables)
    s["tables"].copy_(tables)
    t = torch.arange(T, device="cuda")
    rows = torch.searchsorted(ends, t, right=True)
    real = rows < have.numel()
    r = rows.clamp(max=have.numel() - 1)
    position = torch.where(real, have[r] + t - starts[r], 0)
    slots = torch.where(real, tables[r, position // P].long() * P + position % P, -1)
    return (tables, (have + added).int(), starts.int(), torch.where(real, rows, -1).int(), position,
            slots, (s["count"] - taken[-1:]).int())


def _plain_append(s):
    P = s["case"]["page"]
    real = (s["slots"] >= 0).nonzero().squeeze(1)
    page, at = s["slots"][real] // P, s["slots"][real] % P
    for name in ("k", "v"):
        x = s["rows_" + name][real].float()
        if s[name].dtype == F8:
            # the power of two at or above a 448th of the largest value, 2^-100 at least
            top = x.abs().amax(-1).clamp(min=448.0 * 2.0 ** -100) / 448.0
            m, e = torch.frexp(top)
            e = torch.where(m == 0.5, e - 1, e)
            x = x / torch.exp2(e.float()).unsqueeze(-1)
            s[name + "_scales"][page, :, at] = (e + 127).to(torch.uint8)
        s[name].view(torch.uint8 if s[name].dtype == F8 else s[name].dtype)[page, :, at] = (
            x.to(F8).view(torch.uint8) if s[name].dtype == F8 else x.to(s[name].dtype))
    return [t for t in (s["k"], s["v"], s["k_scales"], s["v_scales"]) if t is not None]


def _gathered(s, name, wide):
    """The cached rows of every request, [R, heads, blocks * page, dim], in type `wide`."""
    at = s["tables"].clamp(min=0).long()
    if s[name].dtype == F8:
        t = s[name].view(torch.uint8)[at].view(F8).to(wide)
        t *= torch.exp2(s[name + "_scales"][at].to(wide) - 127).unsqueeze(-1)
    else:
        t = s[name][at].to(wide)
    return t.transpose(1, 2).flatten(2, 3)


def _mask(s, tokens):
    """[R, drafted, tokens]: what each new token sees."""
    n, window = s["case"]["drafted"], s["case"]["window"]
    end = s["lengths"].long().unsqueeze(1) - torch.arange(n - 1, -1, -1, device="cuda")
    at = torch.arange(tokens, device="cuda")
    seen = at < end.unsqueeze(2)
    return seen & (at >= end.unsqueeze(2) - window) if window else seen


def _grouped(s, q):
    """[R, drafted, q_heads, D] -> [R, heads, drafted * group, D]."""
    H = s["case"]["heads"]
    return q.unflatten(2, (H, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3)


def _ungrouped(s, t):
    """The way back, whatever follows the third axis."""
    n = s["case"]["drafted"]
    return t.unflatten(2, (n, -1)).transpose(1, 2).flatten(2, 3)


def _plain_attend(s):
    R, G = s["q"].shape[0], s["case"]["q_heads"] // s["case"]["heads"]
    k, v = _gathered(s, "k", torch.float32), _gathered(s, "v", torch.float32)
    seen = _mask(s, k.shape[2]).repeat_interleave(G, 1).unsqueeze(1)
    x = _grouped(s, s["q"].float() * s["case"]["dim"] ** -0.5) @ k.transpose(2, 3)
    x = torch.where(seen, x, -math.inf)
    v = torch.where(seen.any(2).unsqueeze(3), v, 0.0)
    m = x.amax(3, keepdim=True)
    if s["sinks"] is not None:
        sink = _grouped(s, s["sinks"].view(1, 1, -1, 1).expand(R, s["case"]["drafted"], -1, 1))
        m = torch.maximum(m, sink)
    m = torch.where(m == -math.inf, 0.0, m)
    e = (x - m).exp()
    z = e.sum(3, keepdim=True)
    if s["sinks"] is not None:
        z = z + (sink - m).exp()
    out = torch.where(z > 0, (e @ v) / z, 0.0)
    return (_ungrouped(s, out).to(s["q"].dtype), _ungrouped(s, (m + z.log()).squeeze(3)))


def _plain_beam(s):
    # in 64 bits: a border between two candidates decides which of them is taken
    R, W = s["scores"].shape
    x = s["logits"].double()
    x = torch.where(x.isnan(), -math.inf, x).view(R, W, -1)
    V = x.shape[2]
    top = x.amax(2, keepdim=True)
    gap = torch.where(x == top, 0.0, x - top)
    p = gap - gap.exp().sum(2, keepdim=True).log()
    p = torch.where(x == -math.inf, -math.inf, p)
    only = torch.where(torch.arange(V, device="cuda") == s["end_token"], 0.0, -math.inf).double()
    p = torch.where(s["ended"].unsqueeze(2) != 0, only, p)
    total = (s["scores"].double().unsqueeze(2) + p).flatten(1)
    total, at = total.sort(dim=1, descending=True, stable=True)
    total, at = total[:, :s["case"]["picks"]], at[:, :s["case"]["picks"]]
    none = total == -math.inf
    return (total.float(), torch.where(none, -1, at % V).int(), torch.where(none, -1, at // V).int())


def _plain_fork(s):
    R, W = s["parents"].shape
    P = s["case"]["page"]
    old = s["tables"].view(R, W, -1)
    width = old.shape[2]
    length = s["lengths"].view(R, W).long()
    col = torch.arange(width, device="cuda")
    held = col < ((length + P - 1) // P).unsqueeze(2)
    parent = s["parents"].long()
    new_length = length.gather(1, parent)
    take = parent.unsqueeze(2).expand(-1, -1, width)
    new_held = held.gather(1, take)
    tables = torch.where(new_held, old.gather(1, take), -1)
    # pages that no beam holds any more, each once, in the order of requests, columns and beams
    was = torch.where(held, old, -2)
    kept = (was.unsqueeze(2) == tables.unsqueeze(1)).any(2)
    lower = torch.ones((W, W), dtype=torch.bool, device="cuda").tril(-1).unsqueeze(2)
    again = ((was.unsqueeze(2) == was.unsqueeze(1)) & lower).any(2)
    dropped = (held & ~kept & ~again).transpose(1, 2)
    pages = old.transpose(1, 2)[dropped]
    count = s["count"].long()
    free = s["free"]
    free[count + torch.arange(pages.numel(), device="cuda")] = pages
    size = count + pages.numel()
    # a partial page stays with the lowest child, the others take copies
    later = ((parent.unsqueeze(2) == parent.unsqueeze(1)) & lower[..., 0]).any(2)
    copies = later & (new_length % P != 0)
    r, b = copies.nonzero(as_tuple=True)
    last = (new_length // P)[r, b]
    source = tables[r, b, last].long()
    target = free[size - 1 - torch.arange(r.numel(), device="cuda")].long()
    tables[r, b, last] = target.int()
    within = torch.arange(P, device="cuda") < (new_length % P)[r, b].unsqueeze(1)
    outputs = []
    for c in s["caches"]:
        for name in ("k", "v"):
            t = c[name].view(torch.uint8) if c[name].dtype == F8 else c[name]
            t[target] = torch.where(within[:, None, :, None], t[source], t[target])
            if c[name + "_scales"] is not None:
                t = c[name + "_scales"]
                t[target] = torch.where(within[:, None], t[source], t[target])
                outputs.append(t)
            outputs.append(c[name])
    return (tables.view(R * W, width), new_length.view(-1).int(), (size - r.numel()).int(), free,
            outputs)


def run(state):
    op = state["case"]["op"]
    if not own:
        plain = {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend,
                 "beam": _plain_beam, "fork": _plain_fork}
        return plain[op](state)
    if op == "plan":
        plan = state["plan"]
        state["pager"].plan_into(state["lengths"], state["added"], state["tables"], state["free"],
                                 state["count"], plan)
        return (state["tables"], plan.lengths, plan.starts, plan.rows, plan.positions, plan.slots,
                plan.count)
    if op == "append":
        state["cache"].append(state["rows_k"], state["rows_v"], state["slots"])
        return [t for t in (state["k"], state["v"], state["k_scales"], state["v_scales"])
                if t is not None]
    if op == "attend":
        state["attention"].attend_into(state["q"], state["cache"], state["tables"],
                                       state["lengths"], state["out"], lse=state["lse"],
                                       sinks=state["sinks"])
        return state["out"], state["lse"]
    if op == "beam":
        scores, tokens, parents = state["out"]
        state["selector"].select_into(state["logits"], state["scores"], scores, tokens, parents,
                                      ended=state["ended"], end_token=state["end_token"])
        return state["out"]
    tables, lengths, count = state["out"]
    state["pager"].fork_into(state["parents"], state["tables"], state["lengths"], state["free"],
                             state["count"], tables, lengths, count, state["layers"])
    outputs = []
    for c in state["caches"]:
        for name in ("k", "v"):
            if c[name + "_scales"] is not None:
                outputs.append(c[name + "_scales"])
            outputs.append(c[name])
    return tables, lengths, count, state["free"], outputs


# ---- what a pass cannot do without --------------------------------------------------------------

def _mean_length(case):
    """The average of the lengths that _lengths spreads over their logarithm."""
    low, high = case["drafted"], max(case["longest"], case["drafted"])
    return (high - low) / math.log(high / low) if case["ragged"] and high > low else high


def work(case):
    op = case["op"]
    if op == "plan":
        R, T = case["requests"], case["requests"] * (1 + case["most"]) // 2
        # lengths, added, starts and lengths out; row, position and slot of a token; pages
        return {"bytes": R * 16 + T * 20 + 8 * max(1, T // case["page"]), "flops": 10 * (R + T)}
    if op == "append":
        n = 2 * case["tokens"] * case["heads"] * case["dim"]
        size = {"bf16": 2, "f32": 4}[case["dtype"]]
        return {"bytes": n * (size + {"bf16": 2, "f8": 1}[case["cache"]]), "flops": 4 * n}
    if op == "attend":
        seen = _mean_length(case) + case["drafted"]
        if case["window"]:
            seen = min(seen, case["window"] + case["drafted"] - 1)
        n = case["requests"] * seen * case["dim"]
        rows = 2 * case["requests"] * case["drafted"] * case["q_heads"] * case["dim"]
        return {"bytes": int(2 * n * case["heads"] * {"bf16": 2, "f8": 1}[case["cache"]]
                             + rows * {"bf16": 2, "f32": 4}[case["dtype"]]),
                "flops": int(4 * n * case["q_heads"] * case["drafted"])}
    if op == "beam":
        n = case["requests"] * case["width"] * case["vocab"]
        return {"bytes": n * {"bf16": 2, "f32": 4}[case["dtype"]], "flops": 4 * n}
    rows = case["requests"] * case["width"]
    blocks = (case["prompt"] // 2 + case["grown"]) // case["page"] + 1
    copied = rows // 3 * case["page"] // 2 * case["heads"] * case["dim"]
    return {"bytes": 8 * rows * blocks
            + 4 * case["layers"] * copied * {"bf16": 2, "f8": 1}[case["cache"]],
            "flops": rows * blocks * case["width"]}


# ---- the definitions in 64 bits ------------------------------------------------------------------

def _exact_append(s):
    P = s["case"]["page"]
    real = s["slots"] >= 0
    page, at = torch.div(s["slots"][real], P, rounding_mode="floor"), s["slots"][real].remainder(P)
    out = []
    for name in ("k", "v"):
        x, t = s["rows_" + name][real].double(), s[name].double()
        if s["k_scales"] is not None:
            largest = x.abs().max(dim=-1).values.clamp(min=448 * 2.0 ** -100)
            x = x / torch.pow(2.0, torch.ceil(torch.log2(largest / 448))).unsqueeze(2)
        t[page, :, at] = x
        out.append(t)
    return out + [None, None] if s["k_scales"] is not None else out


def _exact_attend(s):
    """One request and key head at a time, over the pages as they are."""
    case = s["case"]
    n, D, P, G = case["drafted"], case["dim"], case["page"], case["q_heads"] // case["heads"]
    q = s["q"].double()
    out = torch.zeros_like(q)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    values = {}
    for r, length in enumerate(s["lengths"].tolist()):
        pages = s["tables"][r, :-(-length // P)].long()
        for name in ("k", "v"):
            t = s[name].view(torch.uint8)[pages].view(s[name].dtype).double()
            if s["k_scales"] is not None:
                t = t * torch.pow(2.0, s[name + "_scales"][pages].double() - 127).unsqueeze(3)
            values[name] = t.permute(1, 0, 2, 3).reshape(case["heads"], len(pages) * P, D)
        for i in range(n):
            end = length - (n - 1 - i)
            begin = max(0, end - case["window"]) if case["window"] else 0
            if end <= 0 and s["sinks"] is None:
                continue
            k, v = (values[name][:, begin:max(end, begin)] for name in ("k", "v"))
            z = q[r, i].view(case["heads"], G, D) @ k.transpose(1, 2) / math.sqrt(D)
            if s["sinks"] is not None:
                z = torch.cat((z, s["sinks"].double().view(case["heads"], G, 1)), 2)
                v = torch.cat((v, torch.zeros_like(v[:, :1]) if v.shape[1] else v.new_zeros(
                    case["heads"], 1, D)), 1)
            lse[r, i] = torch.logsumexp(z, 2).flatten()
            out[r, i] = (torch.softmax(z, 2) @ v).reshape(-1, D)
    return out, lse


def _exact_beam(s):
    R, W = s["scores"].shape
    best = []
    for r in range(R):
        x = s["logits"].view(R, W, -1)[r].double()
        x = s["scores"][r].double().unsqueeze(1) + torch.log_softmax(x, 1)
        x[s["ended"][r] != 0] = -math.inf
        stay = torch.where(s["ended"][r] != 0, s["scores"][r].double(), -math.inf)
        best.append(torch.cat((x.flatten(), stay)).topk(s["case"]["picks"]).values)
    return torch.stack(best), None, None


def exact(case, seed):
    global own
    if case["op"] in ("plan", "fork"):
        return None                # whole numbers and copies
    mode, own = own, False         # the inputs alone
    try:
        state = prepare(case, seed)
    finally:
        own = mode
    return {"append": _exact_append, "attend": _exact_attend, "beam": _exact_beam}[case["op"]](state)
