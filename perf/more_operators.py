"""The attention sublayer's operators, as cases that can be timed.

  page_slots       the page table, positions and cache slots of a batch's new
                   tokens from the sequences' lengths (Context.page_slots)
  norm_rotate      the norm of every query and key head and the position
                   rotation in one pass; serving, keys and values go to the
                   paged cache in the same pass (Context.norm_rotate)
  norm_rotate_backward  the gradients of the heads and of the norms' weights
                   (Context.norm_rotate_backward)
  paged_attention  new tokens' attention over the paged cache, with a window
                   and first tokens that stay visible
                   (Context.paged_attention_bf16)

With `own` false a case runs in plain torch operations; with `own` true
through the public entry points of `tiler_amd`.  Device storage is torch's;
the framework's launches go to the bound context's stream.
"""
import math
import random

import torch

own = False

EPS_BITS = 0x358637BD  # 1e-6 as binary32
EPS = 9.999999974752427e-07

_context = _workspace = None


def context():
    """The program's one bound context."""
    global _context
    if _context is None:
        from tiler_amd import Context
        _context = Context(0)
    return _context


def workspace(nbytes):
    """The program's one workspace, as large as its calls have needed so far (they follow one another on one stream)."""
    global _workspace
    if _workspace is None or _workspace.numel() < nbytes:
        context().synchronize()  # nothing reads the smaller one any more
        _workspace = torch.empty(max(nbytes, 1), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
    return _workspace


def listed():
    return [
        # A decode step of 64 sequences: one new token each.
        {"name": "slots_decode", "kind": "slots", "sequences": 64, "fresh_low": 1, "fresh_high": 1, "kept_low": 0,
         "kept_high": 4000, "page": 16, "pad": 0, "spread": 1},
        # A serving step of 512 sequences, decodes and chunks of prompts, rows padded to a graph's size.
        {"name": "slots_mixed", "kind": "slots", "sequences": 512, "fresh_low": 0, "fresh_high": 130, "kept_low": 0,
         "kept_high": 9000, "page": 64, "pad": 37, "spread": 2},
        # A decode step of 16 sequences: queries rotated, keys and values stored.
        {"name": "rotate_decode", "kind": "rotate", "tokens": 16, "heads": 32, "kv_heads": 8, "dim": 128, "rotary":
         128, "pairing": "halves", "norm": True, "dtype": "bf16", "cache": "tokens", "page": 16, "pad": 0, "far":
         5000},
        # A training step's queries and keys, slices of one projection.
        {"name": "rotate_train", "kind": "rotate", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "rotary":
         128, "pairing": "halves", "norm": True, "dtype": "bf16", "cache": "none", "page": 1, "pad": 0, "far": 8192},
        # The gradients of the same.
        {"name": "rotate_grad", "kind": "rotate_backward", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "pairing": "halves", "norm": True, "dtype": "bf16", "far": 8192},
        # A small model in binary32: a part of each head rotated, neighbours paired, everything ragged.
        {"name": "rotate_grad_ragged", "kind": "rotate_backward", "tokens": 1237, "heads": 7, "kv_heads": 1, "dim":
         90, "rotary": 34, "pairing": "neighbours", "norm": True, "dtype": "f32", "far": 100000},
        # A decode step of a small model, short contexts: latency.
        {"name": "attend_decode", "kind": "attend", "sequences": 16, "fresh_low": 1, "fresh_high": 1, "kept_low": 100,
         "kept_high": 1000, "heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "layout": "tokens", "window": 0,
         "sinks": 0, "pad": 0, "spread": 3},
        # A decode step over long contexts: the cache's bytes.
        {"name": "attend_decode_long", "kind": "attend", "sequences": 8, "fresh_low": 1, "fresh_high": 1, "kept_low":
         20000, "kept_high": 32000, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "layout": "heads", "window": 0,
         "sinks": 0, "pad": 0, "spread": 4},
        # A chunk of one prompt behind 8000 cached tokens.
        {"name": "attend_chunk", "kind": "attend", "sequences": 1, "fresh_low": 512, "fresh_high": 512, "kept_low":
         8000, "kept_high": 8000, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "layout": "tokens", "window": 0,
         "sinks": 0, "pad": 0, "spread": 5},
        # Two whole prompts: the products.
        {"name": "attend_prompt", "kind": "attend", "sequences": 2, "fresh_low": 4096, "fresh_high": 4096, "kept_low":
         0, "kept_high": 0, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "layout": "tokens", "window": 0,
         "sinks": 0, "pad": 0, "spread": 6},
        # Chunks of four long prompts under a sliding window, the first tokens visible.
        {"name": "attend_window", "kind": "attend", "sequences": 4, "fresh_low": 1000, "fresh_high": 1100, "kept_low":
         5000, "kept_high": 20000, "heads": 16, "kv_heads": 8, "dim": 64, "page": 32, "layout": "tokens", "window":
         1024, "sinks": 4, "pad": 0, "spread": 7},
        # A serving step of decodes, drafts under verification and chunks, every size ragged, rows padded.
        {"name": "attend_ragged", "kind": "attend", "sequences": 24, "fresh_low": 0, "fresh_high": 150, "kept_low": 0,
         "kept_high": 3000, "heads": 35, "kv_heads": 5, "dim": 80, "page": 24, "layout": "heads", "window": 0, "sinks":
         0, "pad": 21, "spread": 8},
    ]


def _log(rng, lo, hi):
    """A size between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("slots", "rotate", "rotate", "rotate_backward", "attend", "attend", "attend", "attend"))
    if kind == "slots":
        fresh = rng.choice(((1, 1), (0, 3), (0, _log(rng, 4, 200))))
        kept = rng.randrange(2000)
        return {"kind": kind, "sequences": _log(rng, 1, 1000), "fresh_low": fresh[0], "fresh_high": fresh[1],
                "kept_low": kept, "kept_high": kept + _log(rng, 1, 9000),
                "page": rng.choice((1, 16, 32, 64, 128, rng.randrange(5, 100))), "pad": rng.randrange(1, 100),
                "spread": rng.randrange(1 << 20)}
    if kind in ("rotate", "rotate_backward"):
        dim = rng.choice((64, 128, 128, 256, 80, 2 * _log(rng, 8, 130)))
        kv_heads = rng.choice((1, 2, 4, 8, _log(rng, 1, 16)))
        heads = kv_heads * rng.choice((1, 2, 4, 5, 8))
        case = {"kind": kind, "tokens": _log(rng, 1, min(8192, (1 << 25) // (dim * (heads + kv_heads)))), "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "rotary": rng.choice((dim, dim, dim // 4 * 2, 2 * rng.randrange(dim // 2))),
                "pairing": rng.choice(("halves", "halves", "neighbours")), "norm": rng.random() < 0.7,
                "dtype": rng.choice(("bf16", "bf16", "f32")), "far": rng.choice((1000, 100000, 2000000))}
        if kind == "rotate":
            case["cache"] = rng.choice(("none", "tokens", "heads")) if case["dtype"] == "bf16" else "none"
            case["page"] = rng.choice((1, 16, 64, rng.randrange(5, 100)))
            case["pad"] = min(case["tokens"] - 1, rng.randrange(5)) if case["cache"] != "none" else 0
        return case
    kv_heads = rng.choice((1, 2, 4, 8, 8, rng.randrange(1, 12)))
    case = {"kind": kind, "heads": kv_heads * rng.choice((1, 2, 4, 4, 8, rng.randrange(1, 17))), "kv_heads": kv_heads,
            "dim": rng.choice((64, 128, 128, 128, 256, 8 * rng.randrange(2, 32))),
            "page": rng.choice((16, 16, 32, 64, 128, rng.randrange(1, 100))), "layout": rng.choice(("tokens", "heads")),
            "window": rng.choice((0, 0, _log(rng, 1, 4096))), "sinks": 0, "pad": rng.choice((0, rng.randrange(50))),
            "spread": rng.randrange(1 << 20)}
    if case["window"] and rng.random() < 0.7:
        case["sinks"] = rng.choice((1, 4, rng.randrange(100)))
    most = max(work(c)["flops"] for c in listed())
    while True:  # no more than the two whole prompts cost
        what = rng.choice(("decode", "drafts", "chunks", "mixed"))
        case["sequences"] = _log(rng, 1, 48 if what in ("decode", "drafts", "mixed") else 4)
        hi = _log(rng, 1, 2000)
        fresh = {"decode": (1, 1), "drafts": (1, 8), "chunks": (hi, hi + hi // 7), "mixed": (0, 1 + hi // 8)}[what]
        case["fresh_low"], case["fresh_high"] = fresh
        kept = rng.choice((0, _log(rng, 1, 24000), _log(rng, 100, 24000)))
        case["kept_low"], case["kept_high"] = kept // 3, kept
        if 0 < work(case)["flops"] <= most and work(case)["bytes"] < 1 << 30:
            return case


# ---------------------------------------------------------------------------
# Inputs

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _batch(case):
    """The sequences' cached and new tokens, as a scheduler's host lists."""
    rng = random.Random(case["spread"])
    kept = [rng.randint(case["kept_low"], case["kept_high"]) for _ in range(case["sequences"])]
    lo, hi = case["fresh_low"], case["fresh_high"]
    # half of a mixed step's sequences decode
    fresh = [1 if hi > 8 >= lo and rng.random() < 0.5 else rng.randint(lo, hi) for _ in kept]
    return kept, fresh


def _pages(case, kept, fresh):
    return [-(-(a + b) // case["page"]) for a, b in zip(kept, fresh)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sums(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def _normal(g, shape, std=1.0, dtype=torch.bfloat16, mean=0.0):
    """Seeded normal values (made in binary32, then narrowed)."""
    return torch.randn(shape, generator=g, device="cuda").mul_(std).add_(mean).to(dtype)


def _cache(g, case, pages, dim, heads, layout):
    """(k, v) of a page pool, [pages, page, heads, dim] or [pages, heads, page, dim]."""
    shape = (pages, case["page"], heads, dim) if layout == "tokens" else (pages, heads, case["page"], dim)
    return _normal(g, shape), _normal(g, shape)


def _tokens_view(case, cache, layout):
    """[pages, page, heads, dim] of either layout."""
    return cache if layout == "tokens" else cache.transpose(1, 2)


def _placed(g, pages, width, spare=7):
    """Every sequence's pages at random places of a pool: (table, pages of the pool)."""
    total = sum(pages) + spare
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(pages), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(pages):
        table[s, :n] = order[at:at + n]
        at += n
    return table, total


def _frequencies(rotary):
    """Radians a position, for each pair."""
    return 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / max(rotary, 1))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "slots":
        kept, fresh = _batch(case)
        need, have = _pages(case, kept, fresh), _pages(case, kept, [0] * len(kept))
        width = max(max(need), 1) + 3
        table, total = _placed(g, have, width)
        taken = sum(need) - sum(have)
        tokens, count = sum(fresh) + case["pad"], len(kept)
        return {"case": case, "kept": _ints(kept), "fresh": _ints(fresh), "table": table, "width": width,
                "free": (total + torch.randperm(taken + 5, generator=g, device="cuda")).to(torch.int32), "tokens": tokens,
                "starts": _ints([0] * (count + 1)), "lengths": _ints([0] * count), "positions": _ints([0] * tokens),
                "slots": _ints([0] * tokens), "taken": _ints([0])}
    if kind in ("rotate", "rotate_backward"):
        t, h, hk, dim, dtype = (case[x] for x in ("tokens", "heads", "kv_heads", "dim", "dtype"))
        dtype = _DTYPES[dtype]
        # one projection's output: queries, keys and values side by side
        row = _normal(g, (t, (h + 2 * hk) * dim), dtype=dtype) * torch.exp(_normal(g, (t, 1), 0.5, torch.float32)).to(dtype)
        s = {"case": case, "row": row, "q": row[:, :h * dim], "k": row[:, h * dim:(h + hk) * dim],
             "v": row[:, (h + hk) * dim:],
             "positions": torch.randint(0, case["far"], (t,), generator=g, device="cuda", dtype=torch.int32),
             "frequencies": _frequencies(case["rotary"]), "wq": None, "wk": None}
        if case["norm"]:
            s["wq"], s["wk"] = _normal(g, (dim,), 0.1, dtype, 1.0), _normal(g, (dim,), 0.1, dtype, 1.0)
        s["q_out"] = torch.zeros((t, h * dim), dtype=dtype, device="cuda")
        if kind == "rotate":
            if case["cache"] != "none":
                pages = 2 * (-(-t // case["page"])) + 3
                s["kc"], s["vc"] = _cache(g, case, pages, dim, hk, case["cache"])
                slots = torch.randperm(pages * case["page"], generator=g, device="cuda")[:t].to(torch.int32)
                slots[t - case["pad"]:] = -1  # rows that pad the batch
                s.update(slots=slots, pages=pages)
            else:
                s["k_out"] = torch.zeros((t, hk * dim), dtype=dtype, device="cuda")
            return s
        s["dq_out"], s["dk_out"] = _normal(g, (t, h * dim), 0.02, dtype), _normal(g, (t, hk * dim), 0.02, dtype)
        s["drow"] = torch.zeros_like(row)
        s["dq"], s["dk"] = s["drow"][:, :h * dim], s["drow"][:, h * dim:(h + hk) * dim]
        if case["norm"]:
            s["dwq"], s["dwk"] = torch.zeros_like(s["wq"]), torch.zeros_like(s["wk"])
        return s
    kept, fresh = _batch(case)
    h, hk, dim = case["heads"], case["kv_heads"], case["dim"]
    pages = _pages(case, kept, fresh)
    table, total = _placed(g, pages, max(pages) + 1)
    tokens = sum(fresh) + case["pad"]
    s = {"case": case, "kept": kept, "fresh": fresh, "at": _sums(fresh), "table": table, "pages": total, "tokens": tokens,
         "starts": _ints(_sums(fresh)), "lengths": _ints([a + b for a, b in zip(kept, fresh)]),
         "q": _normal(g, (tokens, h * dim), 1.5), "out": torch.zeros((tokens, h * dim), dtype=torch.bfloat16, device="cuda")}
    s["kc"], s["vc"] = _cache(g, case, total, dim, hk, case["layout"])
    return s


# ---------------------------------------------------------------------------
# One pass

def _own_cache(s, layout):
    from tiler_amd import _lib as L
    case = s["case"]
    hk, dim, page = case["kv_heads"], case["dim"], case["page"]
    token, head = (hk * dim, dim) if layout == "tokens" else (dim, page * dim)
    return L.PagedCache(k=s["kc"].data_ptr(), v=s["vc"].data_ptr(), pages=s["pages"], page=page, heads=hk, head_dim=dim,
                        page_stride=page * hk * dim, token_stride=token, head_stride=head)


def _own_heads(case):
    from tiler_amd import _lib as L
    h, hk, dim = case["heads"], case["kv_heads"], case["dim"]
    row = (h + 2 * hk) * dim
    return L.HeadLayout(tokens=case["tokens"], q_heads=h, kv_heads=hk, head_dim=dim, rotary=case["rotary"],
                        pairing=L.ROTATE_HALVES if case["pairing"] == "halves" else L.ROTATE_NEIGHBOURS,
                        eps_bits=EPS_BITS if case["norm"] else 0, q_stride=row, k_stride=row, v_stride=row,
                        q_out_stride=h * dim, k_out_stride=hk * dim)


def _run_own(s):
    from tiler_amd import _lib as L
    case, ctx = s["case"], context()
    at = {name: v.data_ptr() for name, v in s.items() if isinstance(v, torch.Tensor)}
    kind = case["kind"]
    if kind == "slots":
        ctx.page_slots(at["kept"], at["fresh"], case["sequences"], case["page"], at["free"], s["free"].numel(), at["table"],
                       s["width"], s["tokens"], at["starts"], at["lengths"], at["positions"], at["slots"], at["taken"])
        return {name: s[name] for name in ("table", "starts", "lengths", "positions", "slots", "taken")}
    if kind == "rotate":
        dtype = L.BF16 if case["dtype"] == "bf16" else L.F32
        cache = _own_cache(s, case["cache"]) if case["cache"] != "none" else None
        ctx.norm_rotate(dtype, _own_heads(case), at["q"], at["k"], at["v"] if cache else None, at.get("wq"), at.get("wk"),
                        at["positions"], at["frequencies"], at["q_out"], at.get("k_out"), cache, at.get("slots"))
        return {name: s[name] for name in ("q_out", "k_out", "kc", "vc") if name in s}
    if kind == "rotate_backward":
        dtype, heads = L.BF16 if case["dtype"] == "bf16" else L.F32, _own_heads(case)
        space = workspace(ctx.norm_rotate_backward_workspace(dtype, heads))
        ctx.norm_rotate_backward(dtype, heads, at["dq_out"], at["dk_out"], at["q"], at["k"], at.get("wq"), at.get("wk"),
                                 at["positions"], at["frequencies"], at["dq"], at["dk"], at.get("dwq"), at.get("dwk"),
                                 workspace=space.data_ptr(), workspace_bytes=space.numel())
        return {name: s[name] for name in ("dq", "dk", "dwq", "dwk") if name in s}
    shape = L.AttentionShape(tokens=s["tokens"], sequences=case["sequences"], q_heads=case["heads"],
                             scale=case["dim"] ** -0.5, q_stride=case["heads"] * case["dim"],
                             out_stride=case["heads"] * case["dim"], table_width=s["table"].shape[1],
                             window=case["window"], sinks=case["sinks"], max_fresh=max(s["fresh"]),
                             max_length=max(a + b for a, b in zip(s["kept"], s["fresh"])))
    cache = _own_cache(s, case["layout"])
    space = workspace(ctx.paged_attention_bf16_workspace(shape, cache))
    ctx.paged_attention_bf16(shape, at["q"], cache, at["table"], at["starts"], at["lengths"], at["out"],
                             workspace=space.data_ptr(), workspace_bytes=space.numel())
    return {"out": s["out"]}


def _plain_slots(s):
    page, width, tokens = s["case"]["page"], s["width"], s["tokens"]
    kept, fresh = s["kept"].long(), s["fresh"].long()
    lengths = kept + fresh
    have = (kept + page - 1) // page
    new = ((lengths + page - 1) // page).clamp(max=width) - have
    ends, bases = fresh.cumsum(0), new.cumsum(0) - new
    j = torch.arange(width, device="cuda") - have[:, None]
    at = bases[:, None] + j
    wanted = (j >= 0) & (j < new[:, None])
    page_of = torch.where(at < s["free"].numel(), s["free"][at.clamp(0, s["free"].numel() - 1)], -1)
    s["table"].copy_(torch.where(wanted, page_of, s["table"]))
    token = torch.arange(tokens, device="cuda")
    of = torch.searchsorted(ends, token, right=True)
    inside = of < len(kept)
    of = of.clamp(max=len(kept) - 1)
    positions = torch.where(inside, kept[of] + token - (ends - fresh)[of], 0)
    pages = s["table"].long()[of, (positions // page).clamp(max=width - 1)]
    slots = torch.where(inside & (pages >= 0) & (positions < width * page), pages * page + positions % page, -1)
    return {"table": s["table"], "starts": torch.cat((ends.new_zeros(1), ends)).int(), "lengths": lengths.int(),
            "positions": positions.int(), "slots": slots.int(), "taken": new.sum().int().reshape(1)}


def _angles(s):
    # angles in 64 bits: 32 lose the places of far positions
    a = s["positions"].double()[:, None] * s["frequencies"]
    return torch.cos(a).float()[:, None, :], torch.sin(a).float()[:, None, :]


def _turn(case, x, cos, sin):
    """Each head's first `rotary` elements turned in pairs; the rest as they are."""
    r = case["rotary"]
    if case["pairing"] == "halves":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., r:]), -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat((torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2), x[..., r:]), -1)


def _plain_rotate(s):
    case = s["case"]
    t, dim, dtype = case["tokens"], case["dim"], _DTYPES[case["dtype"]]
    cos, sin = _angles(s)

    def heads(x, w):
        x = x.float().reshape(t, -1, dim)
        if w is not None:
            x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * w.float()
        return _turn(case, x, cos, sin).to(dtype)

    q, k = heads(s["q"], s["wq"]), heads(s["k"], s["wk"])
    if case["cache"] == "none":
        return {"q_out": q.reshape(t, -1), "k_out": k.reshape(t, -1)}
    stored = t - case["pad"]
    slots = s["slots"][:stored].long()
    for cache, x in ((s["kc"], k), (s["vc"], s["v"].reshape(t, -1, dim))):
        _tokens_view(case, cache, case["cache"])[slots // case["page"], slots % case["page"]] = x[:stored]
    return {"q_out": q.reshape(t, -1), "kc": s["kc"], "vc": s["vc"]}


def _plain_rotate_backward(s):
    case = s["case"]
    t, dim, dtype = case["tokens"], case["dim"], _DTYPES[case["dtype"]]
    cos, sin = _angles(s)
    out = {}
    for name in ("q", "k"):
        g = _turn(case, s["d" + name + "_out"].float().reshape(t, -1, dim), cos, -sin)
        w = s["w" + name]
        if w is not None:
            x = s[name].float().reshape(t, -1, dim)
            r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
            xh = x * r
            out["dw" + name] = (g * xh).sum((0, 1)).to(dtype)
            g = g * w.float()
            g = r * (g - xh * (g * xh).mean(-1, keepdim=True))
        out["d" + name] = g.reshape(t, -1).to(dtype)
    return out


def _plain_attend(s):
    case = s["case"]
    hk, dim, page = case["kv_heads"], case["dim"], case["page"]
    group = case["heads"] // hk
    for i, (kept, fresh) in enumerate(zip(s["kept"], s["fresh"])):
        if not fresh:
            continue
        length, rows = kept + fresh, slice(s["at"][i], s["at"][i] + fresh)
        pages = s["table"][i, :-(-length // page)].long()

        def keys(cache):  # [heads, length, dim]
            x = _tokens_view(case, cache, case["layout"])[pages].reshape(-1, hk, dim)[:length]
            return x.float().transpose(0, 1).contiguous()

        q = s["q"][rows].float().reshape(fresh, hk, group, dim).permute(1, 0, 2, 3).reshape(hk, fresh * group, dim)
        p = torch.arange(kept, length, device="cuda").repeat_interleave(group)[:, None]
        j = torch.arange(length, device="cuda")
        seen = j <= p
        if case["window"]:
            seen = seen & ((j > p - case["window"]) | (j < case["sinks"]))
        scores = (q @ keys(s["kc"]).transpose(1, 2).contiguous() * dim ** -0.5).masked_fill(~seen, -math.inf)
        e = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = (e / e.sum(-1, keepdim=True)) @ keys(s["vc"])
        s["out"][rows] = o.reshape(hk, fresh, group, dim).transpose(0, 1).reshape(fresh, -1).bfloat16()
    return {"out": s["out"]}


def run(s):
    if own:
        return _run_own(s)
    return {"slots": _plain_slots, "rotate": _plain_rotate, "rotate_backward": _plain_rotate_backward,
            "attend": _plain_attend}[s["case"]["kind"]](s)


# ---------------------------------------------------------------------------
# What a pass cannot do without

def _seen(case, kept, fresh):
    """(pairs of a query and a key it sees, keys that any of the queries sees) of one sequence."""
    pairs = 0
    window, sinks = case["window"], case["sinks"]
    for p in range(kept, kept + fresh):
        pairs += p + 1 if not window else min(window, p + 1) + min(sinks, max(p + 1 - window, 0))
    keys = kept + fresh
    if window and fresh:
        first = max(kept + 1 - window, 0)  # of the first query's window
        keys -= first - min(sinks, first)
    return pairs, keys if fresh else 0


def work(case):
    kind = case["kind"]
    if kind == "slots":
        kept, fresh = _batch(case)
        taken = sum(_pages(case, kept, fresh)) - sum(_pages(case, kept, [0] * len(kept)))
        return {"bytes": 4 * (4 * len(kept) + 2 * (sum(fresh) + case["pad"]) + 2 * taken), "flops": 0}
    if kind in ("rotate", "rotate_backward"):
        t, h, hk, dim = (case[x] for x in ("tokens", "heads", "kv_heads", "dim"))
        e = 2 if case["dtype"] == "bf16" else 4
        n = t * (h + hk) * dim
        small = 4 * t + 4 * case["rotary"] + (2 * e * dim if case["norm"] else 0)
        if kind == "rotate":
            return {"bytes": 2 * e * (n + (t * hk * dim if case["cache"] != "none" else 0)) + small, "flops": 8 * n}
        return {"bytes": (3 if case["norm"] else 2) * e * n + 2 * small, "flops": 16 * n}
    kept, fresh = _batch(case)
    pairs = keys = 0
    for a, b in zip(kept, fresh):
        p, k = _seen(case, a, b)
        pairs, keys = pairs + p, keys + k
    h, hk, dim = case["heads"], case["kv_heads"], case["dim"]
    return {"bytes": 4 * (sum(fresh) * h + keys * hk) * dim + 4 * -(-keys // case["page"]), "flops": 4 * dim * h * pairs}


# ---------------------------------------------------------------------------
# The same results from the definitions, in 64 bits

def _exact_turn(case, x, angle):
    """The pairs as complex numbers, times e^(i angle)."""
    r = case["rotary"]
    pairs = (torch.complex(x[..., :r // 2], x[..., r // 2:r]) if case["pairing"] == "halves"
             else torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()))
    pairs = pairs * torch.polar(torch.ones_like(angle), angle)[:, None, :]
    turned = (torch.cat((pairs.real, pairs.imag), -1) if case["pairing"] == "halves"
              else torch.view_as_real(pairs).flatten(-2))
    return torch.cat((turned, x[..., r:]), -1)


def _exact_rotate(s):
    case = s["case"]
    t, dim = case["tokens"], case["dim"]
    angle = torch.outer(s["positions"].double(), s["frequencies"])
    y = {}
    for name in ("q", "k"):
        x = s[name].double().reshape(t, -1, dim)
        if s["w" + name] is not None:
            x = x * (torch.linalg.vecdot(x, x)[..., None] / dim + EPS) ** -0.5 * s["w" + name].double()
        y[name] = _exact_turn(case, x, angle)
    if case["cache"] == "none":
        return {"q_out": y["q"].flatten(1), "k_out": y["k"].flatten(1)}
    out = {"q_out": y["q"].flatten(1)}
    for name, new in (("kc", y["k"]), ("vc", s["v"].double().reshape(t, -1, dim))):
        cache = s[name].double()
        for i, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                where = (slot // case["page"], slot % case["page"])
                if case["cache"] == "tokens":
                    cache[where[0], where[1]] = new[i]
                else:
                    cache[where[0], :, where[1]] = new[i]
        out[name] = cache
    return out


def _exact_rotate_backward(s):
    case = s["case"]
    t, dim = case["tokens"], case["dim"]
    angle = -torch.outer(s["positions"].double(), s["frequencies"])
    out = {}
    for name in ("q", "k"):
        g = _exact_turn(case, s["d" + name + "_out"].double().reshape(t, -1, dim), angle)
        if s["w" + name] is not None:
            x = s[name].double().reshape(t, -1, dim)
            square = torch.linalg.vecdot(x, x)[..., None] / dim + EPS
            out["dw" + name] = torch.einsum("thd,thd->d", g, x * square ** -0.5)
            g = g * s["w" + name].double()
            # the norm's Jacobian: (I - x x^T / (N square)) / sqrt(square)
            g = (g - x * (torch.linalg.vecdot(g, x)[..., None] / (dim * square))) * square ** -0.5
        out["d" + name] = g.flatten(1)
    return out


def _exact_attend(s):
    case = s["case"]
    hk, dim, page = case["kv_heads"], case["dim"], case["page"]
    group = case["heads"] // hk
    out = s["out"].double()
    for i, (kept, fresh) in enumerate(zip(s["kept"], s["fresh"])):
        if not fresh:
            continue
        length, first = kept + fresh, s["at"][i]
        j = torch.arange(length, device="cuda")
        slot = s["table"][i].long()[j // page]
        for head in range(hk):
            if case["layout"] == "tokens":
                k, v = (s[c][slot, j % page, head].double() for c in ("kc", "vc"))
            else:
                k, v = (s[c][slot, head, j % page].double() for c in ("kc", "vc"))
            for m in range(group):
                at = (head * group + m) * dim
                logits = torch.mm(s["q"][first:first + fresh, at:at + dim].double(), k.t()) / math.sqrt(dim)
                back = torch.arange(kept, length, device="cuda")[:, None] - j  # how far behind the query
                hidden = back < 0
                if case["window"]:
                    hidden |= (back >= case["window"]) & (j >= case["sinks"])
                logits[hidden] = -math.inf
                out[first:first + fresh, at:at + dim] = torch.mm(torch.softmax(logits, -1), v)
    return {"out": out}


def exact(case, seed):
    if case["kind"] == "slots":
        return None  # whole numbers
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "rotate_backward": _exact_rotate_backward, "attend": _exact_attend}[case["kind"]](s)
