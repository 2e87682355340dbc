"""Cases that time three operators over a paged KV cache, with their plain forms.

  varlen  attention of ragged new tokens over the paged cache, with optional distance bias (one
          slope per head), prefix mask, per-token first visible position, sliding window, soft-cap
  shared  decode attention of a batch whose groups of sequences share a long prefix
  gather  rows of the cache read back, dequantised, as contiguous keys and values

Lengths are fixed by the case alone; page tables and values come from the seed.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
QUANT = ("i8", "i4")


# ------------------------------------------------------------------------------------- cases

def _varlen(name, kv, q, seqs, ctx, new, heads, dim, page=16, **more):
    case = {"name": name, "op": "varlen", "kv": kv, "q": q, "seqs": seqs, "ctx_min": ctx[0], "ctx_max": ctx[1],
            "new_min": new[0], "new_max": new[1], "hq": heads[0], "hkv": heads[1], "dim": dim, "page": page,
            "causal": True, "bias": False, "prefix": 0, "docs": False, "window": 0, "cap": 0.0, "lens": 1}
    case.update(more)
    return case


def _shared(name, kv, q, groups, seqs, prefix, ctx, heads, dim, page=16, **more):
    case = {"name": name, "op": "shared", "kv": kv, "q": q, "groups": groups, "seqs": seqs, "pre_min": prefix[0],
            "pre_max": prefix[1], "ctx_min": ctx[0], "ctx_max": ctx[1], "hq": heads[0], "hkv": heads[1], "dim": dim,
            "page": page, "cap": 0.0, "lens": 1}
    case.update(more)
    return case


def _gather(name, kv, to, seqs, ctx, heads, dim, page=16, **more):
    case = {"name": name, "op": "gather", "kv": kv, "to": to, "seqs": seqs, "ctx_min": ctx[0], "ctx_max": ctx[1],
            "hkv": heads, "dim": dim, "page": page, "per_page": False, "lens": 1}
    case.update(more)
    return case


def listed():
    return [
        # one decode step of a few short conversations of a model with distance-biased scores: latency counts
        _varlen("decode_few", "bf16", "bf16", 4, (37, 512), (1, 1), (8, 8), 64, bias=True),
        # a full serving batch of the same kind, one new token each, the contexts of the repository's decode workload
        _varlen("decode_batch", "bf16", "bf16", 64, (512, 8192), (1, 1), (32, 8), 128, bias=True),
        # the same with an int8 cache whose rows carry their own scales, as the append writes them
        _varlen("decode_int8", "i8", "bf16", 48, (512, 8192), (1, 1), (32, 8), 128, bias=True),
        # continuous batching: prompt chunks of uneven length beside decode steps, capped scores and a window
        _varlen("mixed_chunks", "bf16", "bf16", 16, (200, 4096), (1, 512), (32, 8), 128, cap=30.0, window=1024),
        # packed documents behind a bidirectional prefix (image or instruction tokens): odd sizes, f16
        _varlen("prefix_docs", "f16", "f16", 5, (300, 1900), (150, 1700), (12, 4), 64, prefix=257, docs=True, page=32),
        # long prompt chunks: the compute-bound end
        _varlen("prompt_long", "bf16", "bf16", 2, (8000, 8192), (2000, 2048), (32, 8), 128, bias=True),
        # a handful of requests behind one short system prompt: latency counts
        _shared("shared_few", "bf16", "bf16", 1, 8, (500, 500), (1, 60), (32, 8), 128),
        # a chat batch behind one system prompt with examples
        _shared("shared_chat", "bf16", "bf16", 1, 64, (4096, 4096), (16, 1024), (32, 8), 128),
        # three prompts of uneven length over uneven groups, capped scores, f16, odd sizes
        _shared("shared_groups", "f16", "f16", 3, 77, (700, 5001), (1, 700), (16, 2), 64, page=32, cap=50.0),
        # many answers over one long document
        _shared("shared_long", "bf16", "bf16", 1, 256, (32768, 32768), (64, 2048), (64, 8), 128),
        # one request's int8 rows read back
        _gather("read_one", "i8", "bf16", 1, (301, 301), 8, 128),
        # a batch's int8 cache read back for a dense pass
        _gather("read_batch", "i8", "bf16", 32, (512, 8192), 8, 128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {op: max(w["bytes"] + w["flops"] / 200 for w in (work(c) for c in listed() if c["op"] == op))
            for op in ("varlen", "shared", "gather")}
    while True:
        op = rng.choice(("varlen", "varlen", "shared", "gather"))
        page = rng.choice((16, 16, 32, 64))
        lens = rng.randrange(1 << 20)
        if op == "gather":
            kv = rng.choice(("i8", "i8", "i4", "bf16", "f16", "f32"))
            top = _log(rng, 16, 8192)
            case = _gather("", kv, rng.choice(("bf16", "f32", "f16")), _log(rng, 1, 40), (max(1, top // rng.choice((1, 4, 16))), top),
                           rng.choice((1, 2, 4, 8, 8, 12)), rng.choice((64, 128, 128, 96)), page, per_page=rng.random() < 0.3 and kv in QUANT, lens=lens)
        elif op == "shared":
            kv = rng.choice(("bf16", "bf16", "f16", "i8"))
            pre, ctx = _log(rng, 64, 32768), _log(rng, 1, 2048)
            case = _shared("", kv, "f16" if kv == "f16" else "bf16", rng.choice((1, 1, 2, 5)), _log(rng, 5, 256), (max(1, pre // rng.choice((1, 3))), pre),
                           (max(1, ctx // 8), ctx), rng.choice(((32, 8), (64, 8), (16, 2), (8, 8), (12, 4))), rng.choice((64, 128, 128)), page,
                           cap=rng.choice((0.0, 0.0, 50.0)), lens=lens)
        else:
            kv = rng.choice(("bf16", "bf16", "bf16", "f16", "i8", "f32"))
            q = "bf16" if kv == "i8" else kv
            heads = rng.choice(((32, 8), (32, 8), (64, 8), (8, 8), (12, 4), (20, 4)))
            seqs = _log(rng, 1, 64)
            top = _log(rng, 16, 8192)
            new = (1, 1) if rng.random() < 0.4 or kv == "i8" else (1, _log(rng, 2, 2048))
            if kv == "f32":
                top, new, seqs = min(top, 1500), (1, min(new[1], 96)), min(seqs, 8)
            case = _varlen("", kv, q, seqs, (max(1, top // rng.choice((1, 4, 16))), top), (new[0], min(new[1], top)), heads,
                           rng.choice((64, 128, 128)), page, bias=rng.random() < 0.5, docs=rng.random() < 0.25,
                           prefix=rng.choice((0, 0, 0, 100)), window=rng.choice((0, 0, 0, 700)), cap=rng.choice((0.0, 0.0, 30.0)),
                           causal=rng.random() < 0.9, lens=lens)
            if not case["causal"]:
                case["window"] = 0
        del case["name"]
        w = work(case)
        if w["bytes"] + w["flops"] / 200 <= most[op] and _plain_bytes(case) < 9e9:
            return case


# ------------------------------------------------------------------------------- what is in a case

def _lengths(case):
    """Everything about a case that its sizes alone fix: lists of plain integers."""
    r = random.Random(case["lens"])
    ctx = [r.randint(case["ctx_min"], case["ctx_max"]) for _ in range(case["seqs"])]
    ctx[-1] = case["ctx_max"]
    d = {"ctx": ctx}
    if case["op"] == "varlen":
        new = [min(c, r.randint(case["new_min"], case["new_max"])) for c in ctx]
        new[-1] = min(ctx[-1], case["new_max"])
        d["new"] = new
        d["prefix"] = [min(c, r.randint(0, 2 * case["prefix"])) if case["prefix"] else 0 for c in ctx]
        # documents of 64 .. 600 positions, packed one behind the other in each sequence
        d["starts"] = []
        if case["docs"]:
            for c, n in zip(ctx, new):
                at, cuts = 0, [0] * c
                while at < c:
                    size = r.randint(64, 600)
                    cuts[at:at + size] = [at] * len(cuts[at:at + size])
                    at += size
                d["starts"] += cuts[c - n:]
    if case["op"] == "shared":
        g = min(case["groups"], case["seqs"])
        d["starts"] = [0] + sorted(r.sample(range(1, case["seqs"]), g - 1)) + [case["seqs"]]
        d["prefix"] = [r.randint(case["pre_min"], case["pre_max"]) for _ in range(g)]
        d["prefix"][-1] = case["pre_max"]
    return d


def _plain_bytes(case):
    """Bytes of the largest intermediate of the plain form (its scores, or the gathered cache)."""
    n = _lengths(case)
    if case["op"] == "gather":
        return 0
    top = max(n["ctx"])
    if case["op"] == "varlen":
        return 4 * case["seqs"] * max(case["hq"] * max(n["new"]) * top, top * case["hkv"] * case["dim"])
    widest = max(b - a for a, b in zip(n["starts"], n["starts"][1:]))
    return 4 * max(len(n["prefix"]) * widest * case["hq"] * max(n["prefix"]), case["seqs"] * top * case["hkv"] * case["dim"])


def _row_bytes(kind, dim, per_page=False, page=16):
    return {"f32": 4 * dim, "bf16": 2 * dim, "f16": 2 * dim, "i8": dim, "i4": dim / 2}[kind] + (4 / (page if per_page else 1) if kind in QUANT else 0)


def _visible(case, n):
    """Query-key pairs that are attended, and the cache rows that at least one query attends, over all sequences."""
    pairs, rows, at = 0, 0, 0
    for c, m, p in zip(n["ctx"], n["new"], n["prefix"]):
        low, high = c, 0
        for i in range(m):
            pos = c - m + i
            hi = min(c, max(pos + 1, p)) if case["causal"] else c
            lo = max(0, pos - case["window"] + 1 if case["window"] else 0, n["starts"][at + i] if case["docs"] else 0)
            if lo < hi:
                pairs, low, high = pairs + hi - lo, min(low, lo), max(high, hi)
        rows, at = rows + max(0, high - low), at + m
    return pairs, rows


def work(case):
    n = _lengths(case)
    row = 2 * case["hkv"] * _row_bytes(case["kv"], case["dim"], case.get("per_page", False), case["page"])
    if case["op"] == "gather":
        tokens = sum(n["ctx"])
        return {"bytes": tokens * (row + 2 * case["hkv"] * _row_bytes(case["to"], case["dim"]) + 8), "flops": 2 * tokens * case["hkv"] * case["dim"]}
    q = 2 * case["hq"] * _row_bytes(case["q"], case["dim"])
    if case["op"] == "varlen":
        pairs, rows = _visible(case, n)
        return {"bytes": rows * (row + 4 / case["page"]) + sum(n["new"]) * q, "flops": 4 * pairs * case["hq"] * case["dim"]}
    widths = [b - a for a, b in zip(n["starts"], n["starts"][1:])]
    rows = sum(n["ctx"]) + sum(n["prefix"])
    pairs = sum(n["ctx"]) + sum(w * p for w, p in zip(widths, n["prefix"]))
    return {"bytes": rows * (row + 4 / case["page"]) + case["seqs"] * q, "flops": 4 * pairs * case["hq"] * case["dim"]}


def _tables(lens, page, perm, at):
    """[len(lens), widest] page ids taken from `perm` at `at`, -1 behind each sequence's last page."""
    need = torch.tensor([-(-c // page) for c in lens], device=perm.device)
    width = max(1, -(-max(lens) // page))
    first = at + torch.cumsum(need, 0) - need
    col = torch.arange(width, device=perm.device)
    ids = perm[(first[:, None] + col).clamp(max=perm.numel() - 1)]
    return torch.where(col < need[:, None], ids, -1).to(torch.int32).contiguous(), at + sum(-(-c // page) for c in lens)


def prepare(case, seed):
    """A paged pool with its tables, as an engine holds them, and the new tokens' queries: q ~ N(0, 1), K and V ~ N(0, 0.5^2)."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    n = _lengths(case)
    page, hkv, dim = case["page"], case["hkv"], case["dim"]
    lists = [n["ctx"]] + ([n["prefix"]] if case["op"] == "shared" else [])
    pages = sum(-(-c // page) for one in lists for c in one) + 3
    perm = torch.randperm(pages, device=dev, generator=g)
    s = {"case": case, "pages": pages, "top": max(n["ctx"])}
    s["table"], at = _tables(n["ctx"], page, perm, 0)
    s["ctx"] = torch.tensor(n["ctx"], dtype=torch.int32, device=dev)

    def pool():
        shape = (pages, hkv, page, dim)
        if case["kv"] not in QUANT:
            return torch.randn(shape, dtype=DTYPES[case["kv"]], device=dev, generator=g).mul_(0.5), None, (0, 0, 0)
        x = torch.randn(shape, dtype=torch.float32, device=dev, generator=g).mul_(0.5)
        big = x.abs().amax(dim=(2, 3) if case.get("per_page") else 3)
        scale = big / (127 if case["kv"] == "i8" else 7)
        whole = torch.floor(x.div_(scale[:, :, None, None] if case.get("per_page") else scale[..., None]).add_(0.5))
        strides = (hkv, 1, 0) if case.get("per_page") else (hkv * page, page, 1)
        if case["kv"] == "i8":
            return whole.clamp_(-127, 127).to(torch.int8), scale, strides
        half = whole.clamp_(-8, 7).add_(8).to(torch.uint8).view(pages, -1, 2)
        return (half[..., 0] | (half[..., 1] << 4)).contiguous(), scale, strides

    s["k"], s["ks"], s["strides"] = pool()
    s["v"], s["vs"], _ = pool()
    if case["op"] == "gather":
        s["seq"] = torch.repeat_interleave(torch.arange(case["seqs"], device=dev), s["ctx"].long()).to(torch.int32)
        s["pos"] = torch.cat([torch.arange(c, device=dev) for c in n["ctx"]]).to(torch.int32)
        return s
    rows = sum(n["new"]) if case["op"] == "varlen" else case["seqs"]
    s["q"] = torch.randn((rows, case["hq"], dim), device=dev, generator=g).to(DTYPES[case["q"]])
    if case["op"] == "varlen":
        s["cu"] = torch.tensor([0] + n["new"], device=dev).cumsum(0).to(torch.int32)
        s["most"] = max(n["new"])
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, case["hq"] + 1, device=dev) / case["hq"]) if case["bias"] else None
        s["prefix"] = torch.tensor(n["prefix"], dtype=torch.int32, device=dev) if case["prefix"] else None
        s["starts"] = torch.tensor(n["starts"], dtype=torch.int32, device=dev) if case["docs"] else None
    else:
        s["ptable"], _ = _tables(n["prefix"], page, perm, at)
        s["plen"] = torch.tensor(n["prefix"], dtype=torch.int32, device=dev)
        s["starts"] = torch.tensor(n["starts"], dtype=torch.int32, device=dev)
        s["ptop"] = max(n["prefix"])
        s["most"] = max(b - a for a, b in zip(n["starts"], n["starts"][1:]))
    return s


# ------------------------------------------------------------------------------------- plain forms

def _rows(s, which, pages, slots):
    """Cache rows [..., hkv, dim] in 32 bits of the given pages and slots (two integer tensors of one shape)."""
    case = s["case"]
    pool, scale = s[which], s[which + "s"]
    if case["kv"] == "i4":
        both = pool.view(s["pages"], case["hkv"], case["page"], case["dim"] // 2)[pages, :, slots]
        x = torch.stack((both & 15, both >> 4), -1).flatten(-2).float() - 8
    else:
        x = pool[pages, :, slots].float()
    if scale is None:
        return x
    return x * (scale[pages] if case.get("per_page") else scale[pages, :, slots])[..., None]


def _context(s, which, table, top):
    """[sequences, top, hkv, dim] in 32 bits: the first `top` positions of each table row, zeros where it has no page."""
    page = s["case"]["page"]
    pos = torch.arange(top, device=table.device)
    pages = table[:, pos // page].long()
    x = _rows(s, which, pages.clamp(min=0), (pos % page).expand_as(pages))
    return x.masked_fill_((pages < 0)[..., None, None], 0)


def _scores(s, q, k, eq):
    x = torch.einsum(eq, q, k).mul_(1.0 / math.sqrt(s["case"]["dim"]))
    cap = s["case"]["cap"]
    return x.div_(cap).tanh_().mul_(cap) if cap else x


def _plain_varlen(s):
    case, q, ctx = s["case"], s["q"], s["ctx"].long()
    hkv, grp, dim = case["hkv"], case["hq"] // case["hkv"], case["dim"]
    cu = s["cu"].long()
    new = cu[1:] - cu[:-1]
    i = torch.arange(s["most"], device=q.device)
    live = i < new[:, None]
    at = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)
    x = _scores(s, q[at].float().view(case["seqs"], s["most"], hkv, grp, dim), _context(s, "k", s["table"], s["top"]), "sqhgd,slhd->shgql")
    pos = (ctx - new)[:, None] + i
    key = torch.arange(s["top"], device=q.device)
    hi = ctx[:, None].expand_as(pos)
    if case["causal"]:
        hi = torch.minimum(hi, pos + 1 if s["prefix"] is None else torch.maximum(pos + 1, s["prefix"].long()[:, None]))
    lo = torch.zeros_like(pos)
    if case["window"]:
        lo = torch.maximum(lo, pos - case["window"] + 1)
    if s["starts"] is not None:
        lo = torch.maximum(lo, s["starts"].long()[at])
    seen = (key >= lo[..., None]) & (key < hi[..., None]) & live[..., None]
    if s["slopes"] is not None:
        far = (pos[..., None] - key).abs().float()
        x -= s["slopes"].view(1, hkv, grp, 1, 1) * far[:, None, None]
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x.sub_(x.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    x.div_(x.sum(-1, keepdim=True).clamp(min=1e-30))
    y = torch.einsum("shgql,slhd->sqhgd", x, _context(s, "v", s["table"], s["top"]))
    row = torch.arange(q.shape[0], device=q.device)
    seq = torch.searchsorted(cu[1:], row, right=True)
    return y.reshape(case["seqs"], s["most"], case["hq"], dim)[seq, row - cu[seq]].to(q.dtype)


def _plain_shared(s):
    case, q = s["case"], s["q"]
    hkv, grp, dim, seqs = case["hkv"], case["hq"] // case["hkv"], case["dim"], case["seqs"]
    starts = s["starts"].long()
    row = torch.arange(seqs, device=q.device)
    group = torch.searchsorted(starts[1:], row, right=True)
    q = q.float().view(seqs, hkv, grp, dim)
    at = (starts[:-1, None] + torch.arange(s["most"], device=q.device)).clamp(max=seqs - 1)
    # the prefix once for all sequences of its group, then each sequence's own positions
    a = _scores(s, q[at], _context(s, "k", s["ptable"], s["ptop"]), "gnhrd,glhd->gnhrl")
    a.masked_fill_((torch.arange(s["ptop"], device=q.device) >= s["plen"][:, None])[:, None, None, None], -math.inf)
    b = _scores(s, q, _context(s, "k", s["table"], s["top"]), "shrd,slhd->shrl")
    b.masked_fill_((torch.arange(s["top"], device=q.device) >= s["ctx"][:, None])[:, None, None], -math.inf)
    mine = (group, row - starts[group])
    most = torch.maximum(a.amax(-1)[mine], b.amax(-1)).clamp(min=-3e38)
    shift = torch.zeros(a.shape[:4], device=q.device)
    shift[mine] = most
    a.sub_(shift[..., None]).exp_()
    b.sub_(most[..., None]).exp_()
    total = a.sum(-1)[mine] + b.sum(-1)
    y = torch.einsum("gnhrl,glhd->gnhrd", a, _context(s, "v", s["ptable"], s["ptop"]))[mine]
    y = y + torch.einsum("shrl,slhd->shrd", b, _context(s, "v", s["table"], s["top"]))
    return (y / total.clamp(min=1e-30)[..., None]).view(seqs, case["hq"], dim).to(s["q"].dtype)


def _plain_gather(s):
    page = s["case"]["page"]
    pages = s["table"][s["seq"].long(), (s["pos"] // page).long()].long()
    slots = (s["pos"] % page).long()
    to = DTYPES[s["case"]["to"]]
    return _rows(s, "k", pages, slots).to(to), _rows(s, "v", pages, slots).to(to)


def run(state):
    s, case = state, state["case"]
    if own:
        from gollek_b200 import ops
        pool = dict(num_kv_heads=case["hkv"], block_size=case["page"], num_blocks=s["pages"], k_scales=s["ks"], v_scales=s["vs"],
                    scale_strides=s["strides"], int4=case["kv"] == "i4")
        if case["op"] == "varlen":
            return ops.paged_attention_varlen(s["q"], s["k"], s["v"], s["table"], s["cu"], s["ctx"], causal=case["causal"], soft_cap=case["cap"],
                                              sliding_window=case["window"], alibi_slopes=s["slopes"], prefix_lens=s["prefix"],
                                              token_starts=s["starts"], **pool)
        if case["op"] == "shared":
            return ops.paged_attention_shared_prefix(s["q"], s["k"], s["v"], s["ptable"], s["plen"], s["starts"], s["table"], s["ctx"],
                                                     soft_cap=case["cap"], **pool)
        return ops.kv_gather(s["k"], s["v"], s["pos"], s["table"], head_dim=case["dim"], token_seq=s["seq"], dtype=DTYPES[case["to"]], **pool)
    return {"varlen": _plain_varlen, "shared": _plain_shared, "gather": _plain_gather}[case["op"]](s)


# ------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    """The operators from their definitions in 64 bits, one sequence at a time."""
    s, n = prepare(case, seed), _lengths(case)
    page, hkv, dim = case["page"], case["hkv"], case["dim"]

    def read(which, table, count):
        """[count, hkv, dim]: positions 0 .. count - 1 of one table row."""
        ids = table[: -(-count // page)].long()
        x = s[which][ids]
        if case["kv"] == "i4":
            x = x.view(-1, hkv, page, dim // 2).to(torch.int64)
            x = torch.cat(((x & 15).unsqueeze(-1), (x >> 4).unsqueeze(-1)), -1).reshape(-1, hkv, page, dim) - 8
        x = x.double()
        if s[which + "s"] is not None:
            f = s[which + "s"][ids].double()
            x = x * (f.view(-1, hkv, 1, 1) if case.get("per_page") else f.unsqueeze(-1))
        return x.transpose(1, 2).reshape(-1, hkv, dim)[:count]

    if case["op"] == "gather":
        return tuple(torch.cat([read(w, s["table"][i], c) for i, c in enumerate(n["ctx"])]) for w in ("k", "v"))

    grp, out, at = case["hq"] // hkv, [], 0
    for i, c in enumerate(n["ctx"]):
        k, v = read("k", s["table"][i], c), read("v", s["table"][i], c)
        if case["op"] == "shared":
            g = max(j for j, a in enumerate(n["starts"][:-1]) if a <= i)
            k = torch.cat((read("k", s["ptable"][g], n["prefix"][g]), k))
            v = torch.cat((read("v", s["ptable"][g], n["prefix"][g]), v))
        m = n["new"][i] if case["op"] == "varlen" else 1
        q = s["q"][at:at + m].double()
        seen = torch.ones((m, k.shape[0]), dtype=torch.bool, device=k.device)
        where = torch.arange(c - m, c, device=k.device)[:, None]
        key = torch.arange(k.shape[0], device=k.device)[None]
        if case["op"] == "varlen":
            if case["causal"]:
                seen &= (key <= where) | (key < n["prefix"][i])
            if case["window"]:
                seen &= key > where - case["window"]
            if case["docs"]:
                seen &= key >= torch.tensor(n["starts"][at:at + m], device=k.device)[:, None]
        one = torch.empty((m, case["hq"], dim), dtype=torch.float64, device=k.device)
        for h in range(case["hq"]):
            x = q[:, h] @ k[:, h // grp].T / math.sqrt(dim)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["op"] == "varlen" and case["bias"]:
                x = x - s["slopes"][h].double() * (where - key).abs()
            x = x.masked_fill(~seen, -math.inf)
            one[:, h] = torch.nan_to_num(torch.softmax(x, -1)) @ v[:, h // grp]
        out.append(one)
        at += m
    return torch.cat(out)
