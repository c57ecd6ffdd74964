"""Attention over pages of keys and values that many requests share, and over packed prompts, as measurable cases.

    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program holds before the call
    run(state)          one pass: through the framework's operators when `own` is set, in plain torch operations otherwise
    work(case)          bytes and operations the pass cannot do without
    exact(case, seed)   the outputs of run() in 64 bits, from the definitions

Kinds of cases:
  plan    the rows, positions, places and pages of a step, from the requests' lengths (a decode step, an admission of prompts)
  write   the projected rows of a step: query and key norms, temperature, value mixing, keys and values to their pages
  paged   causal grouped-query attention of a step's rows (single tokens, chunks of prompts, both) over the pages
  packed  causal grouped-query attention of whole prompts that lie behind one another, without a cache

How many tokens each request holds and brings follows from the case alone, so that the work of a case is one number; the seed
shuffles the requests, their pages and all values.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"


def _up16(n):
    return (n + 15) // 16 * 16


def _up64(n):
    return (n + 63) // 64 * 64


def _heads(heads, kv_heads, dim, vdim=None):
    return dict(heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim or dim)


def listed():
    return [
        # A decode step of 256 requests, each one token further; some start a page.
        dict(name="plan_step", kind="plan", requests=256, page=16, ctx=32768, chunk=1, chunks=0, done=0, idle=3, pad=0),
        # Admission: 64 prompts (or parts of them) beside decoding requests, finished ones give their pages back; rows are padded.
        dict(name="plan_admission", kind="plan", requests=2000, page=32, ctx=4096, chunk=1024, chunks=64, done=100, idle=200, pad=1111),
        # A decode step in true 32 bits, values mixed with those of an earlier layer, two rows of padding.
        dict(name="write_step_f32", kind="write", requests=6, page=16, ctx=1500, chunk=1, chunks=0, pad=2, f32=True, mix=True,
             **_heads(4, 1, 256)),
        # Prompts of 8000 tokens in all.
        dict(name="write_prompts", kind="write", requests=16, page=64, ctx=512, chunk=800, chunks=16, pad=0, f32=False, mix=False,
             **_heads(32, 8, 128)),
        # One token of one request: the smallest call, all latency. Heads as in the 1152-wide decoder.
        dict(name="paged_row", kind="paged", requests=1, page=16, ctx=500, chunk=1, chunks=0, idle=0, pad=0, f32=False, **_heads(4, 1, 256)),
        # A decode step of 64 requests of very different lengths: the stream of keys and values.
        dict(name="paged_step", kind="paged", requests=64, page=16, ctx=16384, chunk=1, chunks=0, idle=2, pad=4, f32=False,
             **_heads(32, 8, 128)),
        # A decode step in true 32 bits, heads as in the 768-wide decoder.
        dict(name="paged_step_f32", kind="paged", requests=24, page=32, ctx=1500, chunk=1, chunks=0, idle=0, pad=0, f32=True,
             **_heads(12, 4, 64)),
        # Chunks of six prompts beside 34 decoding requests, seven query heads per key head.
        dict(name="paged_mixed", kind="paged", requests=40, page=64, ctx=4000, chunk=600, chunks=6, idle=0, pad=100, f32=False,
             **_heads(28, 4, 128)),
        # The last chunk of a long document.
        dict(name="paged_long", kind="paged", requests=1, page=128, ctx=30000, chunk=2048, chunks=1, idle=0, pad=0, f32=False,
             **_heads(8, 2, 256)),
        # Prompts of different lengths scored together.
        dict(name="packed_prompts", kind="packed", sequences=24, longest=2048, empty=1, pad=77, f32=False, **_heads(32, 8, 128)),
        # One document at once: the largest product.
        dict(name="packed_long", kind="packed", sequences=1, longest=16384, empty=0, pad=0, f32=False, **_heads(16, 4, 128)),
        # Short texts in true 32 bits, heads that fill no tile.
        dict(name="packed_f32_odd", kind="packed", sequences=7, longest=700, empty=1, pad=0, f32=True, **_heads(6, 2, 80, 48)),
    ]


HEADS = (_heads(12, 4, 64), _heads(8, 2, 128), _heads(4, 1, 256), _heads(32, 8, 128), _heads(8, 8, 64), _heads(28, 4, 128),
         _heads(6, 2, 80, 48), _heads(16, 1, 128), _heads(5, 5, 72, 104), _heads(24, 8, 192, 128))


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("plan", "write", "paged", "paged", "paged", "packed", "packed"))
    while True:
        f32 = rng.random() < 0.25
        if kind == "packed":
            case = dict(kind=kind, sequences=_log(rng, 1, 40), longest=_log(rng, 1, 700 if f32 else 16384), empty=rng.randint(0, 2),
                        pad=rng.choice((0, rng.randint(1, 200))), f32=f32, **rng.choice(HEADS))
        else:
            page = rng.choice((16, 32, 64, 128))
            requests = _log(rng, 1, 2000 if kind == "plan" else 64)
            chunks = rng.choice((0, rng.randint(0, requests)))
            chunk = _log(rng, 2, 300 if f32 else 2048) if chunks else 1
            rest = requests - chunks
            case = dict(kind=kind, requests=requests, page=page, ctx=_log(rng, 1, 3000 if f32 else 30000), chunk=chunk, chunks=chunks,
                        pad=rng.choice((0, rng.randint(1, 100))))
            if kind == "plan":
                case.update(done=rng.randint(0, rest // 2), idle=rng.randint(0, rest // 4))
            elif kind == "write":
                case.update(f32=f32, mix=rng.random() < 0.3, **rng.choice(HEADS))
            else:
                case.update(idle=rng.randint(0, rest // 4), f32=f32, **rng.choice(HEADS))
        w = work(case)
        if w["flops"] <= (1.2e12 if not f32 else 1e11) and w["bytes"] <= 2.5e9 and _plain_floats(case) <= 4.3e9:
            return case


def _plain_floats(case):
    """Floats of the largest array of the plain form."""
    if case["kind"] == "packed":
        lens = _lengths(case)
        return len(lens) * max(lens) ** 2 * case["heads"]
    if case["kind"] == "paged":
        requests = _requests(case)
        longest, most = max(o + max(n, 0) for o, n in requests), max(max(n, 0) for _, n in requests)
        return len(requests) * longest * max(most * case["heads"], case["kv_heads"] * (case["dim"] + case["vdim"]))
    return 0


# ---- what a case's requests hold and bring ---------------------------------------------------------------------------
def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _requests(case):
    """(tokens held, tokens brought) of every request; -1 brought: the request is done."""
    rng, out = _rng(case), []
    for i in range(case["requests"]):
        held = case["ctx"] if i == 0 else _log(rng, max(1, case["ctx"] // 32), case["ctx"])
        if i < case["chunks"]:
            out.append((held if rng.random() < 0.7 or i == 0 else 0, case["chunk"] if i == 0 else rng.randint((case["chunk"] + 1) // 2, case["chunk"])))
        elif i < case["chunks"] + case.get("done", 0):
            out.append((held, -1))
        elif i < case["chunks"] + case.get("done", 0) + case.get("idle", 0):
            out.append((held, 0))
        else:
            out.append((held, 1))
    return out


def _lengths(case):
    rng = _rng(case)
    return [case["longest"]] + [0] * case["empty"] + [_log(rng, max(1, case["longest"] // 32), case["longest"])
                                                      for _ in range(case["sequences"] - 1)]


def _rows(case):
    if case["kind"] == "packed":
        return sum(_lengths(case)) + case["pad"]
    return sum(max(n, 0) for _, n in _requests(case)) + case["pad"]


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _from_zero(counts):
    return torch.cat([counts.new_zeros(1), counts.cumsum(0)])


def _step(case, g):
    """Requests in the seed's order with their pages: everything that a step starts from."""
    P, requests = case["page"], _requests(case)
    order = torch.randperm(len(requests), generator=g, device=DEVICE)
    held, new = (_i32(v)[order] for v in zip(*requests))
    used = sum(-(-h // P) for h, _ in requests)
    wanted = sum(-(-(h + max(n, 0)) // P) - -(-h // P) for h, n in requests)
    pages = used + wanted + max(8, used // 8)
    most = max(-(-(h + max(n, 0)) // P) for h, n in requests) + 1
    scattered = torch.randperm(pages, generator=g, device=DEVICE, dtype=torch.int32)
    count = (held + P - 1) // P
    first = _from_zero(count)[:-1]
    j = torch.arange(most, device=DEVICE)
    at = (first[:, None] + j).clamp(max=pages - 1).long()
    tables = torch.where(j < count[:, None], scattered[at], -1).to(torch.int32)
    free = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
    start = int(torch.randint(pages, (1,), generator=g, device=DEVICE))
    free[(start + torch.arange(pages - used, device=DEVICE)) % pages] = scattered[used:]
    span = _i32([start, pages - used])
    return dict(new=new, lens=held, tables=tables, free=free, span=span, pages=pages)


def _randn(g, dtype, *shape):
    out = torch.empty(*shape, dtype=dtype, device=DEVICE)
    flat, piece = out.view(-1), 1 << 28
    for at in range(0, flat.numel(), piece):
        flat[at:at + piece] = torch.randn(min(piece, flat.numel() - at), generator=g, device=DEVICE)
    return out


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case=case, rows=_rows(case), f32=case.get("f32", False))
    if case["kind"] == "packed":
        return _prepare_packed(case, g, s)
    s.update(_step(case, g))
    if case["kind"] == "plan":
        return s
    H, G, D, V, P = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case["page"]
    dtype = torch.float32 if s["f32"] else torch.bfloat16
    # what the step's plan says: requests behind their new tokens, with pages for them
    planned = _plan(s, case)
    s.update(lens=planned["lens"], tables=planned["tables"], row_start=planned["row_start"], pos=planned["pos"], places=planned["places"])
    s["real"] = s["rows"] - case["pad"]
    cache = None
    if own:
        from zignn_b200 import api
        cache = api.PagedCache(H, G, D, V, s["pages"], P, D ** -0.5, temp_coef=0.1, temp_every=512.0, f32=s["f32"])
        s.update(cache=cache, k=cache.k, v=cache.v)
    else:
        s["k"] = torch.zeros(s["pages"], P, G, _up16(D), dtype=dtype, device=DEVICE)
        s["v"] = torch.zeros(s["pages"], P, G, _up16(V), dtype=dtype, device=DEVICE)
    s["k"][..., :D] = _randn(g, dtype, s["pages"], P, G, D)
    s["v"][..., :V] = _randn(g, dtype, s["pages"], P, G, V)
    if case["kind"] == "write":
        s["qkv"] = _randn(g, torch.float32, s["rows"], (H + G) * D + G * V)
        s["q_norm"], s["k_norm"] = (1 + 0.1 * _randn(g, torch.float32, D) for _ in range(2))
        s["vmix"] = _randn(g, torch.float32, 1) * 0.1 + 0.5 if case["mix"] else None
        s["v_first"] = _randn(g, torch.float32, s["rows"], G * V) if case["mix"] else None
    else:
        s["q"] = torch.zeros(s["rows"], H, _up16(D), dtype=dtype, device=DEVICE)
        s["q"][..., :D] = _randn(g, dtype, s["rows"], H, D)
        s["out"] = torch.zeros(s["rows"], _up64(H * V), dtype=dtype, device=DEVICE)
    return s


def _prepare_packed(case, g, s):
    H, G, D, V = case["heads"], case["kv_heads"], case["dim"], case["vdim"]
    dp, vp, dtype = _up16(D), _up16(V), torch.float32 if case["f32"] else torch.bfloat16
    lens = _i32(_lengths(case))
    lens = lens[torch.randperm(lens.numel(), generator=g, device=DEVICE)]
    qkv = torch.zeros(s["rows"], (H + G) * dp + G * vp, dtype=dtype, device=DEVICE)
    q, k, v = qkv[:, :H * dp].view(-1, H, dp), qkv[:, H * dp:(H + G) * dp].view(-1, G, dp), qkv[:, (H + G) * dp:].view(-1, G, vp)
    for t, n in ((q, D), (k, D), (v, V)):
        t[..., :n] = _randn(g, dtype, t.shape[0], t.shape[1], n)
    s.update(q=q, k=k, v=v, row_start=_from_zero(lens).to(torch.int32), longest=case["longest"], scale=D ** -0.5,
             out=torch.zeros(s["rows"], _up64(H * V), dtype=dtype, device=DEVICE))
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(s):
    return {"plan": _run_plan, "write": _run_write, "paged": _run_paged, "packed": _run_packed}[s["case"]["kind"]](s)


def _run_plan(s):
    if own:
        from zignn_b200 import api
        p = api.page_plan(s["new"], s["lens"], s["tables"], s["free"], s["span"], s["case"]["page"], s["rows"])
        return dict(lens=p.lens, tables=s["tables"], free=s["free"], span=p.span, row_start=p.row_start, pos=p.pos, places=p.places,
                    status=p.status)
    return _plan(s, s["case"])


def _plan(s, case):
    P, pages, rows = case["page"], s["pages"], s["rows"]
    new, lens, tables, free, span = s["new"], s["lens"], s["tables"], s["free"], s["span"]
    done, more = new < 0, new.clamp(min=0)
    have = (lens + P - 1) // P
    after = torch.where(done, 0, lens + more)
    want = (lens + more + P - 1) // P - have
    row_start = _from_zero(more)
    take, give = _from_zero(want), _from_zero(torch.where(done, have, 0))
    j = torch.arange(tables.shape[1], device=DEVICE)
    fresh = (j >= have[:, None]) & (j < (have + want)[:, None])
    from_free = ((span[0] + take[:-1, None] + j - have[:, None]) % pages).long()
    # pages given back go behind the free ones; one place more takes what is no page
    back = torch.where(done[:, None] & (j < have[:, None]), (span[0] + span[1] + give[:-1, None] + j) % pages, pages).long()
    new_free = torch.cat([free, free.new_zeros(1)]).scatter(0, back.view(-1), tables.view(-1))[:pages]
    new_tables = torch.where(fresh, free[from_free], tables)
    row = torch.arange(rows, device=DEVICE)
    of = (torch.searchsorted(row_start, row, right=True) - 1).clamp(max=new.numel() - 1)
    real = row < row_start[-1]
    pos = torch.where(real, lens[of] + row - row_start[of], 0)
    places = torch.where(real, new_tables[of, pos // P] * P + pos % P, -1)
    i32 = torch.int32
    return dict(lens=after.to(i32), tables=new_tables, free=new_free,
                span=torch.stack([(span[0] + take[-1]) % pages, span[1] - take[-1] + give[-1]]).to(i32), row_start=row_start.to(i32),
                pos=pos.to(i32), places=places.to(i32), status=torch.zeros(1, dtype=i32, device=DEVICE))


def _norm(x, w, eps=1e-6):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w


def _run_write(s):
    if own:
        q = s["cache"].write(s["qkv"], s["q_norm"], s["k_norm"], s["pos"], s["places"], s["vmix"], s["v_first"])
        return dict(q=q, k=s["k"], v=s["v"])
    H, G, D, V = (s["case"][n] for n in ("heads", "kv_heads", "dim", "vdim"))
    q, k, v = s["qkv"].split([H * D, G * D, G * V], 1)
    temperature = 1 + 0.1 * torch.log(torch.floor((s["pos"] + 1) / 512.0) + 1)
    q = _norm(q.view(-1, H, D), s["q_norm"]) * temperature[:, None, None]
    k = _norm(k.view(-1, G, D), s["k_norm"])
    if s["vmix"] is not None:
        v = (1 - s["vmix"]) * v + s["vmix"] * s["v_first"]
    out = torch.zeros(s["rows"], H, _up16(D), dtype=s["k"].dtype, device=DEVICE)
    out[..., :D] = q.to(out.dtype)
    real, P = s["real"], s["case"]["page"]
    at = s["places"][:real].long()
    s["k"][at // P, at % P, :, :D] = k[:real].to(out.dtype)
    s["v"][at // P, at % P, :, :V] = v.reshape(-1, G, V)[:real].to(out.dtype)
    return dict(q=out, k=s["k"], v=s["v"])


def _run_paged(s):
    if own:
        return s["cache"].attend(s["q"], s["row_start"], s["lens"], s["tables"], out=s["out"])
    case, P = s["case"], s["case"]["page"]
    requests = _requests(case)
    longest, most = max(h + max(n, 0) for h, n in requests), max(1, max(n for _, n in requests))
    key = torch.arange(longest, device=DEVICE)
    page = s["tables"][:, key // P].clamp(0, s["pages"] - 1).long()
    k, v = s["k"][page, key % P], s["v"][page, key % P]
    row = torch.arange(most, device=DEVICE)
    count = s["row_start"][1:] - s["row_start"][:-1]
    q = s["q"][(s["row_start"][:-1, None] + row).clamp(max=s["rows"] - 1).long()]
    see = (s["lens"] - count)[:, None] + row + 1
    return _spread(s, _attention(case, q, k, v, see, case["dim"] ** -0.5), count)


def _run_packed(s):
    if own:
        from zignn_b200 import api
        return api.packed_attention(s["q"], s["k"], s["v"], s["row_start"], s["scale"], vdim=s["case"]["vdim"], out=s["out"])
    row = torch.arange(s["longest"], device=DEVICE)
    at = (s["row_start"][:-1, None] + row).clamp(max=s["rows"] - 1).long()
    count = s["row_start"][1:] - s["row_start"][:-1]
    see = (row + 1).expand(count.numel(), -1)
    return _spread(s, _attention(s["case"], s["q"][at], s["k"][at], s["v"][at], see, s["scale"]), count)


def _attention(case, q, k, v, see, scale):
    """[requests, rows, heads, vdim] of q [requests, rows, heads, .] over keys 0 .. see - 1 of [requests, keys, kv_heads, .], f32."""
    n, most, H, G = q.shape[0], q.shape[1], case["heads"], case["kv_heads"]
    q, k, v = (t.float() for t in (q, k, v[..., :case["vdim"]]))
    q = q.view(n, most, G, H // G, -1).permute(0, 2, 3, 1, 4).reshape(n, G, H // G * most, -1)
    p = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(scale).view(n, G, H // G, most, -1)
    p.masked_fill_(torch.arange(k.shape[1], device=DEVICE) >= see[:, None, None, :, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp(min=1e-30))
    o = torch.matmul(p.view(n, G, H // G * most, -1), v.permute(0, 2, 1, 3))
    return o.view(n, G, H // G, most, -1).permute(0, 3, 1, 2, 4).reshape(n, most, H, -1)


def _spread(s, o, count):
    """The real rows of o [requests, rows, heads, vdim] behind one another, zeros in the columns of the pitch and in the padding."""
    row = torch.arange(s["rows"], device=DEVICE)
    of = (torch.searchsorted(s["row_start"], row, right=True) - 1).clamp(max=count.numel() - 1)
    y = o[of, (row - s["row_start"][of]).clamp(max=o.shape[1] - 1)].reshape(s["rows"], -1)
    y = torch.where(row[:, None] < s["row_start"][-1], y, 0.0)
    out = torch.zeros(s["rows"], _up64(y.shape[1]), dtype=s["q"].dtype, device=DEVICE)
    out[:, :y.shape[1]] = y.to(out.dtype)
    return out


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    rows = _rows(case) - case["pad"]
    if case["kind"] == "plan":
        requests, P = _requests(case), case["page"]
        moved = sum(-(-h // P) if n < 0 else -(-(h + n) // P) - -(-h // P) for h, n in requests)
        # lengths in and out, new tokens, row starts; pages taken or given (read, written); position and place of every row
        return dict(bytes=16 * len(requests) + 8 * moved + 8 * (rows + case["pad"]) + 20, flops=0)
    H, G, D, V = case["heads"], case["kv_heads"], case["dim"], case["vdim"]
    size = 4 if case["f32"] else 2
    if case["kind"] == "write":
        values, n = (H + G) * D + G * V, rows + case["pad"]
        return dict(bytes=n * (4 * values + size * H * D + 8) + rows * G * (D + V) * size + (4 * n * G * V if case["mix"] else 0),
                    flops=n * 4 * values)
    if case["kind"] == "paged":
        requests = [(h, n) for h, n in _requests(case) if n > 0]
        keys = sum(h + n for h, n in requests)
        pairs = sum(n * h + n * (n + 1) // 2 for h, n in requests)
        index = sum(-(-(h + n) // case["page"]) for h, n in requests) * 4
    else:
        keys, pairs, index = rows, sum(n * (n + 1) // 2 for n in _lengths(case)), 0
    return dict(bytes=size * (rows * H * (D + V) + keys * G * (D + V)) + index, flops=2 * pairs * H * (D + V))


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "plan":
        return None
    s, f64 = prepare(case, seed), torch.float64
    H, G, D, V = case["heads"], case["kv_heads"], case["dim"], case["vdim"]
    if case["kind"] == "write":
        x = s["qkv"].to(f64)
        unit = lambda t, w: t / torch.sqrt(t.pow(2).sum(-1, keepdim=True) / D + 1e-6) * w.to(f64)
        heads = x[:, :(H + G) * D].reshape(-1, H + G, D)
        steps = torch.div(s["pos"] + 1, 512, rounding_mode="floor").to(f64)
        q = torch.zeros(s["rows"], H, _up16(D), dtype=f64, device=DEVICE)
        q[..., :D] = unit(heads[:, :H], s["q_norm"]) * (1 + 0.1 * torch.log1p(steps))[:, None, None]
        value = x[:, (H + G) * D:]
        if case["mix"]:
            share = s["vmix"].to(f64)
            value = value + share * (s["v_first"].to(f64) - value)
        k, v = (t.to(f64).view(-1, G, t.shape[-1]) for t in (s["k"], s["v"]))
        at = s["places"][:s["real"]].long()
        k[at, :, :D] = unit(heads[:, H:], s["k_norm"])[:s["real"]]
        v[at, :, :V] = value.reshape(-1, G, V)[:s["real"]]
        return dict(q=q, k=k.view(s["k"].shape), v=v.view(s["v"].shape))
    out = torch.zeros(s["rows"], _up64(H * V), dtype=f64, device=DEVICE)
    starts = s["row_start"].tolist()
    held = s["lens"].tolist() if case["kind"] == "paged" else [b - a for a, b in zip(starts, starts[1:])]
    for i, (a, b) in enumerate(zip(starts, starts[1:])):
        if a == b:
            continue
        if case["kind"] == "paged":
            pages = s["tables"][i, :-(-held[i] // case["page"])].long()
            k, v = (s[n][pages].flatten(0, 1)[:held[i]] for n in ("k", "v"))
        else:
            k, v = s["k"][a:b], s["v"][a:b]
        for h in range(H):
            keys, values = k[:, h // (H // G), :D].to(f64), v[:, h // (H // G), :V].to(f64)
            for r in range(a, b, 1024):
                e = min(r + 1024, b)
                z = s["q"][r:e, h, :D].to(f64) @ keys.T / math.sqrt(D)
                last = torch.arange(held[i] - (b - r), held[i] - (b - e), device=DEVICE)
                z = z.masked_fill(torch.arange(held[i], device=DEVICE)[None] > last[:, None], -math.inf)
                out[r:e, h * V:(h + 1) * V] = torch.softmax(z, 1) @ values
    return out
