"""Measured cases of the paged-cache operators: the norm and rotation of new
queries and keys on their way into the cache, attention of a chunk of new
tokens over the cache, the attention weight that each cached token collects,
and the eviction of the tokens that collected least.

Each operator has a plain form (elementary torch operations in 32 bits) and
the framework's call of the same name; ``own`` selects which one ``run``
takes.  ``exact`` gives the operator's definition in 64 bits.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f16": 0, "bf16": 1}
EPS = 1e-6
THETA = 10000.0


def listed():
    return [
        # one new token of one sequence: the call between two decode steps, where latency counts
        {"name": "norm_rope_1_token", "op": "norm_rope", "type": "f16", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "halves": True, "page": 16, "table": 4096},
        # one decode step of 253 sequences; small heads of which half the columns turn, in neighbouring pairs
        {"name": "norm_rope_253_tokens", "op": "norm_rope", "type": "bf16", "tokens": 253, "heads": 20, "kv_heads": 4, "dim": 64, "rot": 32,
         "halves": False, "page": 32, "table": 32768},
        # the prompts of one prefill step
        {"name": "norm_rope_16384_tokens", "op": "norm_rope", "type": "bf16", "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "halves": True, "page": 16, "table": 32768},
        # one decode step of one sequence
        {"name": "attn_1x777", "op": "attn", "type": "f16", "batch": 1, "q_max": 1, "kv_max": 777, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "causal": True},
        # one decode step of 96 sequences, 1 to 16384 cached tokens each
        {"name": "attn_96x16384", "op": "attn", "type": "bf16", "batch": 96, "q_max": 1, "kv_max": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "causal": True},
        # a mixed step without shared heads: chunks of 1 to 301 new tokens, short heads
        {"name": "attn_11x301_of_4099", "op": "attn", "type": "bf16", "batch": 11, "q_max": 301, "kv_max": 4099, "heads": 16, "kv_heads": 16, "dim": 64,
         "page": 32, "causal": True},
        # the last 4096 tokens of a prompt of 16384
        {"name": "attn_4096_of_16384", "op": "attn", "type": "f16", "batch": 1, "q_max": 4096, "kv_max": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "causal": True},
        # the weight that one decode step of 64 sequences gives to up to 8192 tokens each
        {"name": "scores_64x8192", "op": "scores", "type": "f16", "batch": 64, "q_max": 1, "kv_max": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "causal": True},
        # the weight that prompts' last chunks of up to 1000 tokens give to what is cached
        {"name": "scores_3x1000_of_6000", "op": "scores", "type": "bf16", "batch": 3, "q_max": 1000, "kv_max": 6000, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "causal": True},
        # one long conversation cut to a quarter
        {"name": "evict_1x4099", "op": "evict", "type": "f16", "batch": 1, "kv_max": 4099, "kv_heads": 8, "dim": 128, "page": 16, "budget": 1024, "sink": 4,
         "recent": 128},
        # a serving batch cut to 2048 tokens a sequence; some are shorter and only move
        {"name": "evict_32x8192", "op": "evict", "type": "bf16", "batch": 32, "kv_max": 8192, "kv_heads": 8, "dim": 128, "page": 16, "budget": 2048, "sink": 4,
         "recent": 256},
        # one very long document cut to a sixteenth
        {"name": "evict_1x131072", "op": "evict", "type": "f16", "batch": 1, "kv_max": 131072, "kv_heads": 8, "dim": 64, "page": 64, "budget": 8192, "sink": 16,
         "recent": 1024},
    ]


def draw(rng):
    def size(low, high):
        return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))

    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("norm_rope", "attn", "scores", "evict")}
    while True:
        op = rng.choice(("norm_rope", "attn", "attn", "scores", "evict"))
        kv_heads = rng.choice((1, 2, 4, 8, 16))
        case = {"op": op, "type": rng.choice(("f16", "bf16")), "kv_heads": kv_heads, "dim": rng.choice((64, 128)), "page": rng.choice((16, 32, 64, 128))}
        if op != "evict":
            case["heads"] = kv_heads * rng.choice((1, 2, 4, 5, 7, 8))
        if op == "norm_rope":
            case |= {"tokens": size(1, 16384), "rot": case["dim"] // rng.choice((1, 1, 2)), "halves": rng.random() < 0.5, "table": 32768}
        elif op == "evict":
            budget = size(64, 8192)
            case |= {"batch": size(1, 32), "kv_max": size(budget, 131072), "budget": budget, "sink": rng.randrange(0, 17), "recent": rng.randrange(1, budget // 2)}
        else:
            q_max = 1 if rng.random() < 0.5 else size(2, 4096 if op == "attn" else 1000)
            case |= {"batch": size(1, 96 if op == "attn" else 64), "q_max": q_max, "kv_max": size(q_max, 16384), "causal": rng.random() < 0.85}
        if _cost(case) <= most[op]:
            return case


def _cost(case):
    """What the plain form of a case handles: padded score entries and cached values."""
    if case["op"] == "norm_rope":
        return case["tokens"] * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
    cached = case["batch"] * case["kv_max"] * case["kv_heads"] * case["dim"]
    return cached + 8 * case["batch"] * case["kv_max"] * case.get("heads", 0) * case.get("q_max", 0)


def _lengths(case):
    """Cached and new tokens of each sequence: spread over the range, the longest first, the same for every seed."""
    n = case["batch"]
    kv = [max(1, case["kv_max"] - (case["kv_max"] - 1) * ((b * 7) % n) // n) for b in range(n)]
    q_max = case.get("q_max", 0)
    q = [min(kv[b], max(1, q_max - (q_max - 1) * ((b * 5) % n) // n)) for b in range(n)] if q_max else []
    return kv, q


def _seen(case):
    """Pairs of a new token and a cached one that it sees, over the batch."""
    kv, q = _lengths(case)
    if not case["causal"]:
        return sum(a * b for a, b in zip(kv, q))
    return sum(b * (a - b) + b * (b + 1) // 2 for a, b in zip(kv, q))


def work(case):
    size, dim, kv_heads = 2, case["dim"], case["kv_heads"]
    if case["op"] == "norm_rope":
        rows = case["tokens"] * (case["heads"] + 2 * kv_heads)
        turned = case["tokens"] * (case["heads"] + kv_heads)
        return {"bytes": 2 * rows * dim * size + case["tokens"] * (case["rot"] * 4 + 8), "flops": turned * (4 * dim + 3 * case["rot"])}
    kv, q = _lengths(case)
    if case["op"] == "evict":
        kept = sum(min(n, case["budget"]) for n in kv)
        return {"bytes": sum(kv) * kv_heads * 4 + kept * kv_heads * (4 * dim * size + 8), "flops": 0}
    pairs, rows = _seen(case) * case["heads"], sum(q) * case["heads"]
    if case["op"] == "attn":
        return {"bytes": 2 * sum(kv) * kv_heads * dim * size + rows * (2 * dim * size + 4), "flops": 4 * pairs * dim}
    return {"bytes": sum(kv) * kv_heads * (dim * size + 8) + rows * (dim * size + 4), "flops": 2 * pairs * dim}


def _table(lengths, page, spare, gen):
    """A block table over shuffled pages, and how many pages there are."""
    counts = [-(-n // page) for n in lengths]
    wide, pages = max(counts), sum(counts) + spare
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(lengths), wide, dtype=torch.int32)
    first = 0
    at = []
    for b, n in enumerate(counts):
        at.append((b, first, n))
        first += n
    host = order.cpu()
    for b, f, n in at:
        table[b, :n] = host[f:f + n]
    return table.cuda(), pages, order[first:]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, dim, kv_heads, page = TYPES[case["type"]], case["dim"], case["kv_heads"], case["page"]

    def normal(*shape, dtype=kind, by=1.0):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype) * by

    s = {"case": dict(case)}
    if case["op"] == "norm_rope":
        n, heads, rot = case["tokens"], case["heads"], case["rot"]
        wide = (heads + 2 * kv_heads) * dim
        packed = normal(n, wide, by=1.5)  # one projection's output: queries, keys and values side by side
        s["q"], s["k"], s["v"] = packed[:, :heads * dim], packed[:, heads * dim:(heads + kv_heads) * dim], packed[:, (heads + kv_heads) * dim:]
        s["stride"] = wide
        s["q_gain"], s["k_gain"] = 1 + normal(dim, by=0.1), 1 + normal(dim, by=0.1)
        turns = torch.arange(case["table"], device="cuda", dtype=torch.float64)[:, None] * THETA ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        s["cos"], s["sin"] = turns.cos().float(), turns.sin().float()
        s["positions"] = torch.randint(0, case["table"], (n,), generator=gen, device="cuda", dtype=torch.int32)
        pages = -(-n // page) + 3
        s["slots"] = torch.randperm(pages * page, generator=gen, device="cuda")[:n].to(torch.int32)
        s["q_out"] = torch.empty(n, heads * dim, device="cuda", dtype=kind)
        s["k_pages"] = torch.zeros(pages, kv_heads, page, dim, device="cuda", dtype=kind)
        s["v_pages"] = torch.zeros_like(s["k_pages"])
        s["scores"] = torch.ones(pages, kv_heads, page, device="cuda")
        return s
    kv, q = _lengths(case)
    s["kv_lens"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    if case["op"] == "evict":
        new = [min(n, case["budget"]) for n in kv]
        s["table"], pages, left = _table(kv, page, sum(-(-n // page) for n in new), gen)
        counts = [-(-n // page) for n in new]
        dst = torch.zeros(len(kv), -(-case["budget"] // page), dtype=torch.int32)
        host, first = left.cpu(), 0
        for b, n in enumerate(counts):
            dst[b, :n] = host[first:first + n]
            first += n
        s["dst"] = dst.cuda()
        # collected weight has a long tail, many equal small values among it
        s["scores"] = (normal(pages, kv_heads, page, dtype=torch.float32, by=1.5).exp() * 64).round() / 64
        s["new_lens"] = torch.empty_like(s["kv_lens"])
        s["kept"] = torch.empty(len(kv), kv_heads, case["budget"], dtype=torch.int32, device="cuda")
    else:
        s["table"], pages, _ = _table(kv, page, 2, gen)
        offs = [0]
        for n in q:
            offs.append(offs[-1] + n)
        s["q_offs"] = torch.tensor(offs, dtype=torch.int32, device="cuda")
        s["q"] = normal(offs[-1], case["heads"], dim, by=1.5)
        s["scale"] = dim ** -0.5
    s["k_pages"] = normal(pages, kv_heads, page, dim)
    if case["op"] == "scores":
        s["scores"] = normal(pages, kv_heads, page, dtype=torch.float32).exp()
        s["lse"] = _log_sums(s)
    else:
        s["v_pages"] = normal(pages, kv_heads, page, dim)
    if case["op"] == "attn":
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(s["q"].shape[:2], device="cuda")
    return s


_calls = {}


def _framework():
    """The framework's launcher, bound to torch's stream, and a workspace for the calls that take one."""
    if not _calls:
        from hexkernels_b200 import device, load, ops

        ops.init(1)
        load().hexcuda_set_timing(0)
        device.bind_stream(0)
        _calls["launch"] = device.launch
        _calls["space"] = torch.empty(device.paged_attn_workspace(0), dtype=torch.uint8, device="cuda")
    return _calls["launch"], _calls["space"]


def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"norm_rope": _norm_rope, "attn": _attn, "scores": _scores, "evict": _evict}[op](s)
    launch, space = _framework()
    code, dim, kv_heads, page = CODES[case["type"]], case["dim"], case["kv_heads"], case["page"]
    pages = s["k_pages"].shape[0]
    if op == "norm_rope":
        launch("qk_norm_rope", 0, code, s["q"], s["stride"], s["k"], s["stride"], s["v"], s["stride"], s["q_gain"], s["k_gain"], s["cos"], s["sin"],
               s["positions"], s["slots"], s["q_out"], s["k_pages"], s["v_pages"], s["scores"], case["tokens"], case["heads"], kv_heads, dim, case["rot"],
               int(case["halves"]), 1, case["table"], pages, page, EPS)
        return {k: s[k] for k in ("q_out", "k_pages", "v_pages", "scores")}
    batch, wide = s["table"].shape
    if op == "attn":
        launch("paged_attn", 0, code, s["q"], s["k_pages"], s["v_pages"], s["table"], s["kv_lens"], s["q_offs"], s["out"], s["lse"], space, space.numel(),
               batch, s["q"].shape[0], case["q_max"], case["heads"], kv_heads, dim, pages, page, wide, s["scale"], int(case["causal"]))
        return {"out": s["out"], "lse": s["lse"]}
    if op == "scores":
        launch("cache_scores", 0, code, s["q"], s["lse"], s["k_pages"], s["table"], s["kv_lens"], s["q_offs"], s["scores"], batch, s["q"].shape[0],
               case["q_max"], case["heads"], kv_heads, dim, pages, page, wide, s["scale"], int(case["causal"]))
        return {"scores": s["scores"]}
    launch("cache_evict", 0, s["k_pages"], s["v_pages"], s["scores"], s["table"], s["dst"], s["kv_lens"], s["new_lens"], s["kept"], batch, kv_heads, dim,
           pages, page, wide, s["dst"].shape[1], case["budget"], case["sink"], case["recent"])
    return {k: s[k] for k in ("kept", "new_lens", "k_pages", "v_pages", "scores")}


# ------------------------------------------------------------- plain forms

def _norm_rope(s):
    case = s["case"]
    n, dim, kv_heads, page, half = case["tokens"], case["dim"], case["kv_heads"], case["page"], case["rot"] // 2
    at = s["positions"].long()
    c, t = s["cos"][at][:, None], s["sin"][at][:, None]

    def turned(x, gain):
        x = x.reshape(n, -1, dim).float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain.float()
        r = x[..., :2 * half]
        a, b = (r[..., :half], r[..., half:]) if case["halves"] else (r[..., 0::2], r[..., 1::2])
        u, w = a * c - b * t, a * t + b * c
        r = torch.cat((u, w), -1) if case["halves"] else torch.stack((u, w), -1).flatten(-2)
        return torch.cat((r, x[..., 2 * half:]), -1)

    kind = s["q"].dtype
    s["q_out"].copy_(turned(s["q"], s["q_gain"]).to(kind).reshape(n, -1))
    where, off = s["slots"].long() // page, s["slots"].long() % page
    s["k_pages"][where, :, off] = turned(s["k"], s["k_gain"]).to(kind)
    s["v_pages"][where, :, off] = s["v"].reshape(n, kv_heads, dim)
    s["scores"][where, :, off] = 0.0
    return {k: s[k] for k in ("q_out", "k_pages", "v_pages", "scores")}


def _cached(pages, table):
    """The cached rows of every sequence, padded to the longest, in 32 bits: [batch, kv_heads, tokens, dim]."""
    x = pages[table.long()]
    return x.transpose(1, 2).flatten(2, 3).float()


def _padded(s):
    """The new tokens' queries, padded, in 32 bits [batch, kv_heads, new * group, dim], their rows, and which exist."""
    case, offs = s["case"], s["q_offs"].long()
    at = offs[:-1, None] + torch.arange(case["q_max"], device="cuda")
    there = at < offs[1:, None]
    at = at.clamp(max=s["q"].shape[0] - 1)
    group = case["heads"] // case["kv_heads"]
    q = s["q"][at].unflatten(2, (case["kv_heads"], group)).permute(0, 2, 1, 3, 4).flatten(2, 3).float()
    return q, at, there


def _hidden(s, there):
    """[batch, 1, new, tokens]: cached tokens that a new token does not see."""
    kv, offs = s["kv_lens"].long(), s["q_offs"].long()
    wide = s["table"].shape[1] * s["case"]["page"]
    key = torch.arange(wide, device="cuda")
    last = kv[:, None].expand(-1, s["case"]["q_max"])
    if s["case"]["causal"]:
        new = torch.arange(s["case"]["q_max"], device="cuda")
        last = torch.minimum(last, kv[:, None] - (offs[1:] - offs[:-1])[:, None] + new + 1)
    return (key >= last[..., None])[:, None]


def _scored(s):
    """The scaled scores of all pairs, minus infinity where hidden [batch, kv_heads, new, group, tokens]."""
    q, at, there = _padded(s)
    x = q @ _cached(s["k_pages"], s["table"]).transpose(-1, -2)
    x = x.unflatten(2, (s["case"]["q_max"], -1)).mul_(s["scale"])
    return x.masked_fill_(_hidden(s, there).unsqueeze(3), -math.inf), at, there


def _log_sums(s):
    x, at, there = _scored(s)
    top = x.amax(-1, keepdim=True)
    lse = (x.sub_(top).exp_().sum(-1).log() + top[..., 0]).permute(0, 2, 1, 3).flatten(2)
    out = torch.empty(s["q"].shape[:2], device="cuda")
    out[at[there]] = lse[there]
    return out


def _attn(s):
    x, at, there = _scored(s)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(top).exp_()
    sums = x.sum(-1, keepdim=True)
    y = (x.flatten(2, 3) @ _cached(s["v_pages"], s["table"])).unflatten(2, (s["case"]["q_max"], -1)) / sums
    y = y.permute(0, 2, 1, 3, 4).flatten(2, 3)
    lse = (sums.log() + top)[..., 0].permute(0, 2, 1, 3).flatten(2)
    s["out"][at[there]] = y[there].to(s["out"].dtype)
    s["lse"][at[there]] = lse[there]
    return {"out": s["out"], "lse": s["lse"]}


def _scores(s):
    x, at, there = _scored(s)
    case = s["case"]
    lse = s["lse"][at].unflatten(2, (case["kv_heads"], -1)).permute(0, 2, 1, 3)
    x = x.sub_(lse[..., None]).exp_().masked_fill_(~there[:, None, :, None, None], 0.0)
    got = x.sum((2, 3)).unflatten(2, (-1, case["page"])).transpose(1, 2)
    used = torch.arange(s["table"].shape[1], device="cuda") * case["page"] < s["kv_lens"][:, None]
    s["scores"].index_add_(0, s["table"][used].long(), got[used])
    return {"scores": s["scores"]}


def _evict(s):
    case, page, kv = s["case"], s["case"]["page"], s["kv_lens"].long()
    budget, table, dst = case["budget"], s["table"].long(), s["dst"].long()
    x = s["scores"][table].transpose(1, 2).flatten(2)
    wide = x.shape[-1]
    key = torch.arange(wide, device="cuda")
    n = kv[:, None, None]
    rank = torch.where(key >= n, 0, torch.where((key < case["sink"]) | (key >= n - case["recent"]), 2, 1)).expand_as(x)
    order = x.sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, rank.gather(-1, order).sort(dim=-1, descending=True, stable=True).indices)
    new = n.clamp(max=budget)
    if wide < budget:
        order = torch.nn.functional.pad(order, (0, budget - wide))
    place = torch.arange(budget, device="cuda")
    kept = torch.where(place < new, order[..., :budget], wide).sort(dim=-1).values
    b, h, j = torch.nonzero(place < new.expand(-1, x.shape[1], -1), as_tuple=True)
    i = kept[b, h, j]
    source, to = (table[b, i // page], h, i % page), (dst[b, j // page], h, j % page)
    s["kept"].copy_(torch.where(place < new, kept, -1))
    s["new_lens"].copy_(new[:, 0, 0])
    s["k_pages"][to] = s["k_pages"][source]
    s["v_pages"][to] = s["v_pages"][source]
    s["scores"][to] = s["scores"][source]
    return {k: s[k] for k in ("kept", "new_lens", "k_pages", "v_pages", "scores")}


# ------------------------------------------------- definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm_rope":
        return _exact_norm_rope(case, s)
    if case["op"] == "evict":
        return _exact_evict(case, s)
    kv, q = _lengths(case)
    group, page, first = case["heads"] // case["kv_heads"], case["page"], 0
    out, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    scores = s["scores"].double() if case["op"] == "scores" else None
    for b, (n, m) in enumerate(zip(kv, q)):
        used = s["table"][b, :-(-n // page)].long()
        for h in range(case["kv_heads"]):
            k = s["k_pages"][used, h].reshape(-1, case["dim"])[:n].double()
            total = torch.zeros(len(used) * page, dtype=torch.float64, device="cuda")
            for lo in range(0, m, 1024):
                hi = min(m, lo + 1024)
                x = s["q"][first + lo:first + hi, h * group:(h + 1) * group].double() @ k.T * float(s["scale"])
                if case["causal"]:
                    ahead = torch.arange(n, device="cuda")[None] - torch.arange(n - m + lo, n - m + hi, device="cuda")[:, None]
                    x[(ahead > 0)[:, None].expand_as(x)] = -math.inf
                if scores is not None:
                    total[:n] += torch.exp(x - s["lse"][first + lo:first + hi, h * group:(h + 1) * group, None].double()).sum((0, 1))
                    continue
                z = torch.logsumexp(x, -1, keepdim=True)
                v = s["v_pages"][used, h].reshape(-1, case["dim"])[:n].double()
                out[first + lo:first + hi, h * group:(h + 1) * group] = torch.exp(x - z) @ v
                lse[first + lo:first + hi, h * group:(h + 1) * group] = z[..., 0]
            if scores is not None:
                scores[used, h] += total.view(-1, page)
        first += m
    return {"scores": scores} if scores is not None else {"out": out, "lse": lse}


def _exact_norm_rope(case, s):
    n, dim, rot, page, kv_heads = case["tokens"], case["dim"], case["rot"], case["page"], case["kv_heads"]
    cos, sin = s["cos"].double()[s["positions"].long()], s["sin"].double()[s["positions"].long()]
    pairs = [(i, i + rot // 2) if case["halves"] else (2 * i, 2 * i + 1) for i in range(rot // 2)]

    def turned(x, gain):
        y = x.reshape(n, -1, dim).double()
        y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / dim + EPS) * gain.double()
        z = y.clone()
        for i, (a, b) in enumerate(pairs):
            z[..., a] = cos[:, i, None] * y[..., a] - sin[:, i, None] * y[..., b]
            z[..., b] = sin[:, i, None] * y[..., a] + cos[:, i, None] * y[..., b]
        return z

    k, v, scores = s["k_pages"].double(), s["v_pages"].double(), s["scores"].double()
    slot = s["slots"].long()
    k.transpose(1, 2).reshape(-1, kv_heads, dim)  # layout only: rows are addressed by page and offset below
    k[slot // page, :, slot % page] = turned(s["k"], s["k_gain"])
    v[slot // page, :, slot % page] = s["v"].reshape(n, kv_heads, dim).double()
    scores[slot // page, :, slot % page] = 0
    return {"q_out": turned(s["q"], s["q_gain"]).reshape(n, -1), "k_pages": k, "v_pages": v, "scores": scores}


def _exact_evict(case, s):
    page, budget, kv_heads = case["page"], case["budget"], case["kv_heads"]
    table, dst, before = s["table"].long().cpu(), s["dst"].long().cpu(), s["scores"].double().cpu()
    kept = torch.full((case["batch"], kv_heads, budget), -1)
    source, to = [], []
    for b, n in enumerate(_lengths(case)[0]):
        m = min(n, budget)
        place = torch.arange(m)
        for h in range(kv_heads):
            key = torch.arange(n)
            x = before[table[b, key // page], h, key % page]
            forced = (key < case["sink"]) | (key >= n - case["recent"])
            if n > budget:
                free = key[~forced]
                best = free[(-x[free]).argsort(stable=True)][:m - int(forced.sum())]
                key = torch.cat((key[forced], best)).sort().values
            kept[b, h, :m] = key
            source.append(torch.stack((table[b, key // page], torch.full_like(key, h), key % page)))
            to.append(torch.stack((dst[b, place // page], torch.full_like(place, h), place % page)))
    source, to = torch.cat(source, 1).cuda(), torch.cat(to, 1).cuda()
    got = {"kept": kept, "new_lens": s["kv_lens"].clamp(max=budget)}
    for name in ("k_pages", "v_pages", "scores"):
        x = s[name].double()
        x[tuple(to)] = x[tuple(source)]
        got[name] = x
    return got
