"""The batched-serving operators, measured: a step's page plan, the rotary append by slot, and the decode attention of
many sequences over one paged pool. `run` computes them in plain torch, or, with `own` set, through the library."""
import ctypes
import math

import torch

own = False

PAGE = 64                                    # positions per page
THETA = 1e6
FORMATS = {"fp16": 0, "e4m3": 1, "e5m2": 2}  # vv_kv_format_t
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
# (query heads, KV heads, head_dim): the 7B decoder; the narrower ones of its family; a plain multi-head and a
# four-to-one layout.
HEADS = ((28, 4, 128), (12, 2, 128), (14, 2, 64), (8, 8, 128), (32, 8, 128), (16, 16, 64))


class KvView(ctypes.Structure):
    """One layer of a KV cache as the attention entry points take it."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_meta", ctypes.c_void_p),
                ("v_meta", ctypes.c_void_p), ("page_table", ctypes.c_void_p), ("format", ctypes.c_int),
                ("n_kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int)]


def listed():
    seven = {"q_heads": 28, "kv_heads": 4, "head_dim": 128}
    return [
        # one decode step of 64 requests, each a token longer: the smallest call, once per step
        {"name": "plan 64 decoding", "op": "plan", "decoding": 64, "prompts": 0, "prompt_rows": 0, "longest": 14449,
         "pad_rows": 0, "short": False},
        # decoding requests beside two prompt chunks that fill a step's budget, padded to a captured graph's rows
        {"name": "plan 193 mixed", "op": "plan", "decoding": 193, "prompts": 2, "prompt_rows": 2048 - 193,
         "longest": 8192, "pad_rows": 2048, "short": False},
        # many prompts at once with too few free pages: the last ones are turned away
        {"name": "plan 31 prompts", "op": "plan", "decoding": 7, "prompts": 31, "prompt_rows": 31 * 1031,
         "longest": 14449, "pad_rows": 100, "short": True},
        # a decode step of 16 requests through one layer: latency
        {"name": "append 16 rows", "op": "append", "rows": 16, "skipped": 0, "format": "fp16", "bias": True, **seven},
        # a streaming step: a prefill chunk and decoding rows together, packed cache, some padding rows
        {"name": "append 2161 rows e4m3", "op": "append", "rows": 2161, "skipped": 113, "format": "e4m3", "bias": True,
         **seven},
        # a whole hour-long prompt's rows
        {"name": "append 14449 rows", "op": "append", "rows": 14449, "skipped": 0, "format": "fp16", "bias": True,
         **seven},
        # one request on a filled cache
        {"name": "attend 1 x 14449", "op": "attend", "seqs": 1, "shortest": 14449, "longest": 14449, "format": "fp16",
         **seven},
        # a slot pool of requests at every stage
        {"name": "attend 24 ragged", "op": "attend", "seqs": 24, "shortest": 0, "longest": 14449, "format": "fp16",
         **seven},
        # many short requests, the narrow decoder
        {"name": "attend 193 short", "op": "attend", "seqs": 193, "shortest": 1, "longest": 700, "format": "fp16",
         "q_heads": 12, "kv_heads": 2, "head_dim": 128},
        # heads of 64 channels
        {"name": "attend 48 hd64", "op": "attend", "seqs": 48, "shortest": 100, "longest": 4099, "format": "fp16",
         "q_heads": 14, "kv_heads": 2, "head_dim": 64},
        # a full card of long requests on the packed cache
        {"name": "attend 64 e4m3", "op": "attend", "seqs": 64, "shortest": 6001, "longest": 8192, "format": "e4m3",
         **seven},
        # the largest: hour-long requests on the FP16 cache
        {"name": "attend 32 long", "op": "attend", "seqs": 32, "shortest": 12345, "longest": 14449, "format": "fp16",
         **seven},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    op = rng.choice(("plan", "append", "attend", "attend"))
    if op == "plan":
        decoding, prompts = _log(rng, 1, 1024), rng.choice((0, 1, 3, 17, 40))
        return {"op": op, "decoding": decoding, "prompts": prompts,
                "prompt_rows": _log(rng, prompts, 30000) if prompts else 0, "longest": _log(rng, 64, 16384),
                "pad_rows": _log(rng, 1, 2048) - 1, "short": rng.random() < 0.3}
    nq, nkv, hd = rng.choice(HEADS)
    fmt = rng.choice(("fp16", "e4m3", "e5m2")) if hd == 128 else "fp16"
    c = {"op": op, "format": fmt, "q_heads": nq, "kv_heads": nkv, "head_dim": hd}
    if op == "append":
        rows = _log(rng, 1, 14449 * 32 // (nq + nkv) // 2)
        return {**c, "rows": rows, "skipped": rng.randrange(rows // 4 + 1), "bias": rng.random() < 0.5}
    longest = _log(rng, 1, 16384)
    most = 13400 * 32 * 4 * 128 // (nkv * hd * longest)      # no more cache than the largest listed case reads
    return {**c, "seqs": _log(rng, 1, max(1, min(512, most // 2))), "shortest": rng.randrange(longest + 1),
            "longest": longest}


# ── inputs ──────────────────────────────────────────────────────────────────

def _spread(lo, hi, n):
    """n whole numbers evenly from lo to hi (hi alone where n is 1): the same ones whatever the seed."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _plan_sizes(case):
    """(new tokens, cached tokens) of every request, before the seed orders them."""
    p, rows, top = case["prompts"], case["prompt_rows"], case["longest"]
    new = [1] * case["decoding"]
    done = 0
    for i in range(p):                                       # chunks of unlike sizes that add up to prompt_rows
        upto = rows if i == p - 1 else rows * (i + 1) * (i + 2) // (p * (p + 1))
        new.append(upto - done)
        done = upto
    return new, _spread(1, top, case["decoding"]) + [0 if i % 2 == 0 else top * i // (4 * p) for i in range(p)]


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _tables(lens, width, gen, spare):
    """Page tables of that width for these lengths from a shuffled pool with `spare` pages more; -1 where no page is."""
    have = (lens + PAGE - 1) // PAGE
    total = int(have.sum())
    perm = torch.randperm(total + spare, generator=gen, device="cuda").to(torch.int32)
    tables = torch.full((lens.numel(), width), -1, dtype=torch.int32, device="cuda")
    tables[torch.arange(width, device="cuda")[None, :] < have[:, None]] = perm[:total]
    return tables, perm[total:].contiguous(), total + spare


def _encode(x, fmt):
    if fmt == "fp16":
        return x.half()
    return x.clamp(-LARGEST[fmt], LARGEST[fmt]).to(FP8[fmt]).view(torch.uint8)


def _pool(n_pages, row, fmt, gen):
    return _encode(torch.randn(n_pages * PAGE, row, generator=gen, device="cuda", dtype=torch.float16), fmt)


def _addresses(state):
    return {k: t.data_ptr() for k, t in state.items() if isinstance(t, torch.Tensor)}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).half()

    if case["op"] == "plan":
        new, cached = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in _plan_sizes(case))
        order = torch.randperm(new.numel(), generator=gen, device="cuda")
        new, cached = new[order].contiguous(), cached[order].contiguous()
        need = sum(_pages(c + n) - _pages(c) for n, c in zip(*_plan_sizes(case)))
        width = max(_pages(c + n) for n, c in zip(*_plan_sizes(case)))
        rows = sum(_plan_sizes(case)[0]) + case["pad_rows"]
        spare = max(1, need * 3 // 4 if case["short"] else need + 16)
        tables, free, _ = _tables(cached, width, gen, spare)
        s = {"new_lens": new, "cache_lens": cached, "tables": tables, "free": free,
             "n_free": torch.tensor([spare], dtype=torch.int32, device="cuda"),
             "lens": torch.empty_like(cached),
             "row_starts": torch.empty(new.numel() + 1, dtype=torch.int32, device="cuda"),
             "positions": torch.empty(rows, dtype=torch.int32, device="cuda"),
             "slots": torch.empty(rows, dtype=torch.int64, device="cuda"),
             "counts": torch.empty(3, dtype=torch.int32, device="cuda")}
        return {**s, "case": case, "n": new.numel(), "width": width, "rows": rows, "at": _addresses(s)}
    nq, nkv, hd, fmt = case["q_heads"], case["kv_heads"], case["head_dim"], case["format"]
    if case["op"] == "append":
        rows, n_pages = case["rows"], _pages(case["rows"]) + 9
        slots = torch.randperm(n_pages * PAGE, generator=gen, device="cuda")[:rows].contiguous()
        if case["skipped"]:
            slots[torch.randperm(rows, generator=gen, device="cuda")[:case["skipped"]]] = -1
        s = {"q": normal(rows, nq, hd), "k": normal(rows, nkv, hd), "v": normal(rows, nkv, hd),
             "positions": torch.randint(0, 16384, (rows,), generator=gen, device="cuda", dtype=torch.int32),
             "slots": slots, "q_out": torch.zeros(rows, nq, hd, dtype=torch.float16, device="cuda"),
             "k_pool": _pool(n_pages, nkv * hd, fmt, gen), "v_pool": _pool(n_pages, nkv * hd, fmt, gen)}
        if case["bias"]:
            s.update(q_bias=normal(nq, hd, std=0.5), k_bias=normal(nkv, hd, std=0.5), v_bias=normal(nkv, hd, std=0.1))
        return {**s, "case": case, "n_pages": n_pages, "at": {"q_bias": None, "k_bias": None, "v_bias": None, **_addresses(s)}}
    lens = torch.tensor(_spread(case["shortest"], case["longest"], case["seqs"]), dtype=torch.int32, device="cuda")
    lens = lens[torch.randperm(case["seqs"], generator=gen, device="cuda")].contiguous()
    width = max(1, _pages(case["longest"]))
    tables, _, n_pages = _tables(lens, width, gen, 5)
    s = {"q": normal(case["seqs"], nq, hd, std=1.5), "k_pool": _pool(n_pages, nkv * hd, fmt, gen),
         "v_pool": _pool(n_pages, nkv * hd, fmt, gen), "tables": tables, "lens": lens,
         "out": torch.empty(case["seqs"], nq, hd, dtype=torch.float16, device="cuda")}
    at = _addresses(s)
    view = KvView(at["k_pool"], at["v_pool"], None, None, at["tables"], FORMATS[fmt], nkv, hd)
    return {**s, "case": case, "n_pages": n_pages, "width": width, "at": at, "view": view, "scratch": {}}


# ── the plain forms ─────────────────────────────────────────────────────────

def _plan(s):
    new, cached, rows, width = s["new_lens"].long(), s["cache_lens"].long(), s["rows"], s["width"]
    new = new.clamp(min=0)
    row_end = new.cumsum(0)
    had = (cached + PAGE - 1) // PAGE
    fits = (new > 0) & (cached >= 0) & (cached + new <= width * PAGE) & (row_end <= rows)
    need = torch.where(fits, (cached + new + PAGE - 1) // PAGE - had, 0)
    taken = need.cumsum(0)
    served = fits & ((need == 0) | (taken <= s["n_free"]))
    r = torch.arange(rows, device="cuda")
    seq = (row_end[None, :] <= r[:, None]).sum(1)            # the request a row belongs to; past the last: none
    inside = seq < s["n"]
    seq = seq.clamp(max=s["n"] - 1)
    live = inside & served[seq]
    position = torch.where(live, cached[seq] + r - (row_end - new)[seq], 0)
    index = position // PAGE
    fresh = (s["n_free"] - 1 - (taken - need)[seq] - (index - had[seq])).clamp(0, s["free"].numel() - 1)
    old = s["tables"][seq, index].long()
    page = torch.where(index < had[seq], old, s["free"][fresh].long())
    first = live & (index >= had[seq]) & (position % PAGE == 0)
    flat = torch.cat([s["tables"].flatten(), s["tables"].new_zeros(1)])
    flat[torch.where(first, seq * width + index, s["n"] * width)] = page.int()
    s["tables"].copy_(flat[:-1].view_as(s["tables"]))
    left = s["n_free"].long() - torch.where(served, taken, 0).max()
    counts = torch.cat([left, row_end[-1:].clamp(max=rows), ((new > 0) & ~served).sum()[None]])
    return {"tables": s["tables"], "lens": (cached + torch.where(served, new, 0)).int(),
            "row_starts": torch.cat([row_end.new_zeros(1), row_end]).clamp(max=rows).int(),
            "positions": position.int(), "slots": torch.where(live, page * PAGE + position % PAGE, -1),
            "counts": counts.int()}


def _as_values(pool, fmt):
    return pool if fmt == "fp16" else pool.view(FP8[fmt])


def _append(s):
    case, fmt, hd = s["case"], s["case"]["format"], s["case"]["head_dim"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if case["bias"]:
        q, k, v = q + s["q_bias"].float(), k + s["k_bias"].float(), v + s["v_bias"].float()
    turn = torch.arange(hd // 2, device="cuda", dtype=torch.float64) * (-2.0 * math.log(THETA) / hd)
    angle = s["positions"].double()[:, None] * turn.exp()
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]

    def rope(x):
        a, b = x[..., : hd // 2], x[..., hd // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    keep = s["slots"] >= 0
    s["q_out"].copy_(torch.where(keep[:, None, None], rope(q).half(), s["q_out"]))
    to = s["slots"][keep]
    s["k_pool"][to] = _encode(rope(k)[keep].flatten(1), fmt)
    s["v_pool"][to] = _encode(v[keep].flatten(1), fmt)
    return {"q": s["q_out"], "k": _as_values(s["k_pool"], fmt), "v": _as_values(s["v_pool"], fmt)}


def _attend(s):
    case, fmt = s["case"], s["case"]["format"]
    n, nq, nkv, hd = case["seqs"], case["q_heads"], case["kv_heads"], case["head_dim"]
    pages, length = s["tables"].long().clamp(min=0), s["width"] * PAGE

    def gathered(pool):
        return _as_values(pool.view(-1, PAGE, nkv * hd)[pages], fmt).float().view(n, length, nkv, hd)

    seen = torch.arange(length, device="cuda")[None, :] < s["lens"][:, None]
    q = s["q"].float().view(n, nkv, nq // nkv, hd) * hd ** -0.5
    scores = q @ gathered(s["k_pool"]).permute(0, 2, 3, 1).contiguous()
    scores = scores.masked_fill(~seen[:, None, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)     # a request without positions: zeros, not NaN
    p = (scores - top).exp()
    o = p @ gathered(s["v_pool"]).permute(0, 2, 1, 3).contiguous()
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, o / total, 0.0).view(n, nq, hd).half()


# ── one pass ────────────────────────────────────────────────────────────────

def _ok(status):
    if status != 0:
        raise RuntimeError("status %d" % status)


def _own(s):
    from __graft_entry__ import load_device
    dev, case, at = load_device(), s["case"], s["at"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "plan":
        _ok(dev.vv_kv_page_plan_dev(at["new_lens"], at["cache_lens"], s["n"], at["tables"], s["width"], at["free"],
                                    at["n_free"], at["lens"], at["row_starts"], at["positions"], at["slots"], s["rows"],
                                    None, at["counts"], stream))
        return {k: s[k] for k in ("tables", "lens", "row_starts", "positions", "slots", "counts")}
    nq, nkv, hd, fmt = case["q_heads"], case["kv_heads"], case["head_dim"], case["format"]
    if case["op"] == "append":
        _ok(dev.vv_rope_kv_append_dev(at["q"], at["k"], at["v"], at["q_bias"], at["k_bias"], at["v_bias"],
                                      at["positions"], at["slots"], at["q_out"], at["k_pool"], at["v_pool"],
                                      case["rows"], nq, nkv, hd, s["n_pages"], FORMATS[fmt], THETA, stream))
        return {"q": s["q_out"], "k": _as_values(s["k_pool"], fmt), "v": _as_values(s["v_pool"], fmt)}
    if not s["scratch"]:                                     # the context's buffer, allocated at its first step
        size = dev.vv_attn_decode_batch_scratch_bytes(case["seqs"], nq, nkv, hd)
        s["scratch"].update(size=size, held=torch.empty(max(size, 16), dtype=torch.uint8, device="cuda"))
    _ok(dev.vv_attn_decode_batch(2, at["q"], ctypes.addressof(s["view"]), at["out"], nq, case["seqs"], at["lens"],
                                 s["width"], s["n_pages"], s["scratch"]["held"].data_ptr(), s["scratch"]["size"],
                                 stream))
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"plan": _plan, "append": _append, "attend": _attend}[state["case"]["op"]](state)


# ── what a pass cannot do without ───────────────────────────────────────────

def work(case):
    if case["op"] == "plan":
        new, cached = _plan_sizes(case)
        rows, n = sum(new), len(new)
        fresh = sum(_pages(c + k) - _pages(c) for k, c in zip(new, cached))
        # lengths in and out, row starts, an old page id for each request, new ids read and written, rows written
        return {"bytes": 4 * (3 * n + n + 1 + n + 2 * fresh + 4) + 12 * (rows + case["pad_rows"]), "flops": 0}
    nq, nkv, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    unit = 2 if case["format"] == "fp16" else 1
    if case["op"] == "append":
        rows = case["rows"] - case["skipped"]
        row = hd * (4 * nq + 4 * nkv + 2 * nkv * unit) + 12
        bias = 2 * hd * (nq + 2 * nkv) if case["bias"] else 0
        return {"bytes": rows * row + bias, "flops": rows * hd * (3 * (nq + nkv) + (nq + 2 * nkv if case["bias"] else 0))}
    seen = sum(_spread(case["shortest"], case["longest"], case["seqs"]))
    pages = sum(_pages(x) for x in _spread(case["shortest"], case["longest"], case["seqs"]))
    return {"bytes": seen * nkv * hd * 2 * unit + 4 * case["seqs"] * nq * hd + 4 * (pages + case["seqs"]),
            "flops": 4 * seen * nq * hd}


# ── the same in 64 bits, from the definitions ───────────────────────────────

def exact(case, seed):
    if case["op"] == "plan":
        return None                                          # whole numbers throughout
    s = prepare(case, seed)
    fmt, nkv, hd = case["format"], case["kv_heads"], case["head_dim"]

    def wide(pool):
        return _as_values(pool, fmt).to(torch.float32).double()

    if case["op"] == "append":
        live = (s["slots"] >= 0).nonzero().flatten()
        where = s["slots"][live]
        place = torch.arange(hd // 2, dtype=torch.float64, device="cuda")
        rate = torch.pow(torch.tensor(THETA, dtype=torch.float64, device="cuda"), -2.0 * place / hd)
        unit = torch.exp(1j * s["positions"][live].double()[:, None, None] * rate)

        def rotated(x, bias):
            x = x[live].double() + (bias.double() if bias is not None else 0.0)
            z = torch.complex(x[..., : hd // 2], x[..., hd // 2:]) * unit
            return torch.cat([z.real, z.imag], -1)

        q, k, v = s["q_out"].double(), wide(s["k_pool"]), wide(s["v_pool"])
        top = LARGEST.get(fmt, math.inf)
        q[live] = rotated(s["q"], s.get("q_bias"))
        k[where] = rotated(s["k"], s.get("k_bias")).flatten(1).clamp(-top, top)
        plain = s["v"][live].double() + (s["v_bias"].double() if case["bias"] else 0.0)
        v[where] = plain.flatten(1).clamp(-top, top)
        if fmt == "e5m2":                                    # two bits of mantissa: its own rounding is 5 % of the values,
            return {"q": q, "k": None, "v": None}            # which says nothing about how exactly they were computed
        return {"q": q, "k": k, "v": v}
    out = torch.zeros(case["seqs"], case["q_heads"], hd, dtype=torch.float64, device="cuda")
    group = case["q_heads"] // nkv
    lens, tables = s["lens"].tolist(), s["tables"].long()
    for b, n in enumerate(lens):
        if n == 0:
            continue
        at = torch.arange(n, device="cuda")
        rows = tables[b][at // PAGE] * PAGE + at % PAGE
        k, v = (wide(s[x][rows]).view(n, nkv, hd) for x in ("k_pool", "v_pool"))
        for h in range(nkv):
            keys, values = k[:, h].t().contiguous(), v[:, h].contiguous()
            weight = torch.softmax(s["q"][b, h * group:(h + 1) * group].double() @ keys / math.sqrt(hd), -1)
            out[b, h * group:(h + 1) * group] = weight @ values
    return out
