"""What is measured of the operators that serve many continuations of a context: the 8-bit paged cache (written, read
back, attended over), attention of a batch over a prefix that its sequences share, and the verification of drafted tokens.

A case is a dict of plain values; `kind` names the operator:

  write   keys and values of new tokens into the 8-bit cache: each (token, head) row of D values gets the smallest power of
          two 2^e with which its largest value is at most 448, and holds round(x / 2^e) as float8_e4m3fn
  read    the values that places of that cache stand for
  attend  softmax(scale q k^T) v of a step's rows over that cache, causal
  prefix  the same for groups of rows that begin with the same tokens: their cache pages are the same ones
  verify  drafted tokens against the target's probabilities, from given random numbers

Cache layout of a page: keys [Hkv, P, D], values [Hkv, D, P], scales [2, Hkv, P]. Sizes are those of the Qwen3 shapes that the
benchmark runs (32, 40 and 64 heads over 8 of 128, 151,936 tokens) and generic ones."""
import math

import torch

own = False
DEV = "cuda"
BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
TYPES = {"bfloat16": BF, "float32": F32}


def listed():
    """Twelve cases, from a step's few tokens to whole prompts."""
    qwen = {"kv_heads": 8, "dim": 128, "page": 16, "type": "bfloat16"}
    return [
        # eight requests decode one token each: a launch's latency
        {"name": "write 8 tokens", "kind": "write", "tokens": 8, **qwen},
        # a prompt portion, keys and values as columns of the merged projection
        {"name": "write 4096 tokens", "kind": "write", "tokens": 4096, **qwen},
        # a short run of tokens of a smaller model in 32 bits, an odd number
        {"name": "read 333 tokens f32", "kind": "read", "tokens": 333, "kv_heads": 4, "dim": 64, "page": 32, "type": "float32"},
        # a long sequence's cache handed on
        {"name": "read 32768 tokens", "kind": "read", "tokens": 32768, **qwen},
        # one request early in its answer: latency
        {"name": "attend 1x300", "kind": "attend", "rows": 1, "len": 300, "query": 1, "long": 0, "heads": 32, "window": 0, **qwen},
        # eight requests behind long contexts
        {"name": "attend 8x32768", "kind": "attend", "rows": 8, "len": 32768, "query": 1, "long": 0, "heads": 32, "window": 0, **qwen},
        # a prompt portion of 2,048 tokens behind 6,144, seven decode rows beside it
        {"name": "attend portion 2048", "kind": "attend", "rows": 8, "len": 8192, "query": 1, "long": 2048, "heads": 32, "window": 0, **qwen},
        # four continuations of one short prompt, bfloat16 cache: latency
        {"name": "prefix 4x1000", "kind": "prefix", "groups": 1, "rows": 4, "prefix": 1000, "len": 60, "query": 1, "heads": 16, "cache8": False,
         "kv_heads": 8, "dim": 64, "page": 16, "type": "bfloat16"},
        # sixty-four answers to one long document, bfloat16 cache
        {"name": "prefix 64x16384", "kind": "prefix", "groups": 1, "rows": 64, "prefix": 16384, "len": 512, "query": 1, "heads": 32, "cache8": False, **qwen},
        # three system prompts, a dozen requests each, four drafted tokens checked a step, 8-bit cache
        {"name": "prefix 3x12x5 8-bit", "kind": "prefix", "groups": 3, "rows": 12, "prefix": 5000, "len": 700, "query": 5, "heads": 40, "cache8": True, **qwen},
        # one request, three drafted tokens: latency
        {"name": "verify 1x3", "kind": "verify", "requests": 1, "drafts": 3, "vocab": 151936, "probs": True},
        # a full batch, up to four drafted tokens each
        {"name": "verify 64x4", "kind": "verify", "requests": 64, "drafts": 4, "vocab": 151936, "probs": True},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["write", "read", "attend", "attend", "prefix", "prefix", "verify"])
    if kind == "verify":
        return {"kind": kind, "requests": log(1, 64), "drafts": rng.randint(1, 8), "vocab": rng.choice([log(900, 160000), 32000, 151936]),
                "probs": rng.random() < 0.7}
    kv_heads, group = rng.choice([(8, 4), (8, 5), (8, 8), (4, 7), (2, 16), (1, 8), (16, 1)])
    dim = rng.choice([64, 128, 128, 128, 256])
    base = {"kind": kind, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 16, 32, 64]), "type": "bfloat16"}
    if kind in ("write", "read"):
        return {**base, "tokens": log(1, 16384), "type": rng.choice(["bfloat16", "bfloat16", "float32"])}
    if kind == "attend":
        long, heads = rng.choice([0, 0, log(6, 1500)]), kv_heads * group
        length = max(long, log(20, 16384))
        if long:
            length = max(long, min(length, 44_000_000_000 // (long * heads * dim)))
        # the 32-bit path's steps: decode rows and a few tokens
        kind_of = "float32" if long == 0 and rng.random() < 0.3 else "bfloat16"
        return {**base, "rows": log(1, 24), "len": length, "query": rng.choice([1, 1, rng.randint(2, 9)]), "long": long, "heads": heads,
                "window": rng.choice([0, 0, 0, log(40, 4000)]), "type": kind_of}
    return {**base, "groups": rng.randint(1, 3), "rows": log(2, 24), "prefix": log(30, 12000), "len": log(2, 800), "query": rng.choice([1, 1, rng.randint(2, 6)]),
            "heads": kv_heads * group, "cache8": rng.random() < 0.5}


# -- inputs -----------------------------------------------------------------------------------------------------------------

def _spread(g, n, least, most):
    """n whole numbers over [least, most] with both ends among them (n > 1: the last one is `most`)."""
    x = least + torch.rand(n, generator=g) * (most - least)
    x = x.round().long().clamp(least, most)
    x[-1] = most
    return x


def _cache8(g, pages, kv_heads, page, dim):
    """Codes and scales as a cache holds them whose rows are about normal: rows' largest codes lie between 224 and 448."""
    codes = torch.empty((pages, 2, kv_heads, page * dim), dtype=E4M3, device=DEV)
    for at in range(0, pages, 4096):
        part = torch.randn((min(4096, pages - at), 2, kv_heads, page * dim), generator=g, device=DEV).mul_(110).clamp_(-448, 448)
        codes[at:at + part.shape[0]] = part.to(E4M3)
    scales = torch.randint(119, 122, (pages, 2, kv_heads, page), generator=g, device=DEV, dtype=torch.uint8).view(E8M0)
    return codes, scales


def prepare(case, seed):
    g, h = torch.Generator(device=DEV).manual_seed(seed), torch.Generator().manual_seed(seed)
    s = dict(case)
    if case["kind"] == "verify":
        b, k, v = case["requests"], case["drafts"], case["vocab"]
        counts = torch.randint(max(1, k - 1), k + 1, (b,), generator=h) + 1          # drafted tokens, and the place behind them
        counts[-1] = k + 1
        start = torch.cat((torch.zeros(1, dtype=torch.long), counts.cumsum(0)))
        n = int(start[-1])
        s["logits"] = torch.randn((n, v), generator=g, device=DEV) * 2.5
        probs = torch.softmax(s["logits"] + 0.7 * torch.randn((n, v), generator=g, device=DEV), -1)   # a smaller model's view
        s["drafted"] = torch.multinomial(probs, 1, generator=g)[:, 0].to(I32)
        s["draft_probs"] = probs if case["probs"] else None
        s["accept"] = torch.rand(n, generator=g, device=DEV)
        s["draw"] = torch.rand(b, generator=g, device=DEV)
        s["temperature"] = (0.6 + 0.5 * torch.rand(b, generator=g, device=DEV)) * (torch.rand(b, generator=g, device=DEV) > 0.12)
        s["start"] = start.to(DEV, I32)
        return s
    kv, dim, page, dtype = case["kv_heads"], case["dim"], case["page"], TYPES[case["type"]]
    if case["kind"] in ("write", "read"):
        t = case["tokens"]
        held = -(-t // page)
        n = held + max(4, held // 8) + 1
        order = torch.randperm(n - 1, generator=h)[:held]
        at = torch.arange(t)
        s["place_page"], s["place_off"] = order[at // page].to(DEV, I32), (at % page).to(DEV, I32)
        s["pages"], s["scales"] = _cache8(g, n, kv, page, dim)
        if case["kind"] == "write":
            rows = torch.randn((t, 6 * kv * dim), generator=g, device=DEV)               # a merged projection of 4 groups of queries
            rows *= torch.exp(0.5 * torch.randn((t, 1), generator=g, device=DEV))        # tokens differ in size
            rows = rows.to(dtype)
            s["k"] = rows[:, 4 * kv * dim: 5 * kv * dim].view(t, kv, dim)
            s["v"] = rows[:, 5 * kv * dim:].view(t, kv, dim)
        return s
    if case["kind"] == "attend":
        b = case["rows"]
        counts = torch.full((b,), case["query"])
        if case["long"]:
            counts[-1] = case["long"]
        least = max(int(counts[:-1].max()) if b > 1 else 1, case["len"] // 3)
        lens = _spread(h, b, min(least, case["len"]), case["len"])
        lens = torch.maximum(lens, counts)
        first = [[] for _ in range(b)]
        shared = torch.zeros(b, dtype=torch.long)
    else:
        b, groups = case["rows"] * case["groups"], case["groups"]
        counts = torch.full((b,), case["query"])
        prefix = _spread(h, groups, max(1, case["prefix"] // 2), case["prefix"])
        tail = _spread(h, b, case["query"], max(case["query"], case["len"]))
        group_of = torch.arange(b) // case["rows"]
        shared = prefix[group_of] // page                        # whole pages: what a prefix cache shares
        prefix = prefix // page * page
        lens = prefix[group_of] + tail
        s["group_start"] = (torch.arange(groups + 1) * case["rows"]).to(DEV, I32)
        s["group_lens"] = prefix.to(DEV, I32)
        s["max_prefix"], s["max_group_queries"] = int(prefix.max()), case["rows"] * case["query"]
        first = None
    wide = int((lens.max() + page - 1) // page) + 1
    need = (lens + page - 1) // page - shared
    starts = torch.cat((torch.zeros(1, dtype=torch.long), need.cumsum(0)))
    heads_of = []
    total = int(starts[-1])
    if first is None:
        for p in (prefix // page).tolist():
            heads_of.append(torch.arange(total, total + p))
            total += p
    n = total + 1                                                # and the null page
    order = torch.randperm(total, generator=h)
    table = torch.full((b + 1, wide), n - 1)
    slots = torch.randperm(b, generator=h)
    for i in range(b):
        mine = torch.arange(int(starts[i]), int(starts[i + 1]))
        if first is None:
            mine = torch.cat((heads_of[int(group_of[i])], mine))
        table[slots[i], : len(mine)] = order[mine]
    if case["kind"] == "attend" or case["cache8"]:
        s["pages"], s["scales"] = _cache8(g, n, kv, page, dim)
    else:
        s["pages"] = torch.empty((n, 2, kv, page * dim), dtype=dtype, device=DEV)
        for at in range(0, n, 4096):
            s["pages"][at:at + 4096] = torch.randn((min(4096, n - at), 2, kv, page * dim), generator=g, device=DEV).to(dtype)
        s["scales"] = None
    t = int(counts.sum())
    s["q"] = (1.5 * torch.randn((t, case["heads"], dim), generator=g, device=DEV)).to(dtype)
    s["table"], s["slots"], s["lens"] = table.to(DEV, I32), slots.to(DEV, I32), lens.to(DEV, I32)
    s["query_start"] = torch.cat((torch.zeros(1, dtype=torch.long), counts.cumsum(0))).to(DEV, I32)
    decode, chunk = torch.nonzero(counts == 1)[:, 0], torch.nonzero(counts > 1)[:, 0]
    s["decode_rows"], s["chunk_rows"] = decode.to(DEV, I32), chunk.to(DEV, I32)
    s["bounds"] = (len(decode), len(chunk), int(lens[decode].max()) if len(decode) else 0, int(counts[chunk].max()) if len(chunk) else 0,
                   int(lens[chunk].max()) if len(chunk) else 0, len(chunk) == 0)
    s["scale"] = dim ** -0.5
    return s


# -- the framework's calls ----------------------------------------------------------------------------------------------------

def _rows(s):
    from holon_amd.kernels.api import AttnRows
    return AttnRows(s["slots"], s["lens"], s["query_start"], s["decode_rows"], s["chunk_rows"], *s["bounds"])


def _run_own(s):
    from holon_amd.kernels import load_hip
    kernels, kind = load_hip(), s["kind"]
    if kind == "write":
        kernels.kv_write_q8(s["k"], s["v"], s["pages"], s["scales"], s["place_page"], s["place_off"], s["page"])
        return {"pages": s["pages"], "scales": s["scales"]}
    if kind == "read":
        k, v = kernels.kv_read_q8(s["pages"], s["scales"], s["place_page"], s["place_off"], s["page"], TYPES[s["type"]])
        return {"k": k, "v": v}
    if kind == "attend":
        return kernels.paged_attention_q8(s["q"], s["pages"], s["scales"], s["table"], _rows(s), s["page"], s["scale"], s["window"])
    if kind == "prefix":
        from holon_amd.kernels.api import SharedPrefix
        prefix = SharedPrefix(s["group_start"], s["group_lens"], s["groups"], s["max_group_queries"], s["max_prefix"])
        return kernels.prefix_attention(s["q"], s["pages"], s["table"], _rows(s), prefix, s["page"], s["scale"], scales=s["scales"])
    tokens, accepted = kernels.verify_drafts(s["logits"], s["drafted"], s["draft_probs"], s["accept"], s["draw"], s["temperature"],
                                             s["start"], s["drafts"])
    return {"tokens": tokens, "accepted": accepted}


# -- the plain forms ----------------------------------------------------------------------------------------------------------

def _power(scales):
    return torch.ldexp(torch.ones((), device=DEV), scales.view(torch.uint8).to(I32) - 127)


def _quantised(x):
    """x [..., D] -> (codes, exponents + 127): the smallest power of two that brings the row's largest value to 448 or less."""
    mantissa, power = torch.frexp(x.float().abs().amax(-1))
    e = torch.where(mantissa == 0, 0, power - 9 + (mantissa > 0.875).to(I32)).clamp(min=-126)
    return torch.ldexp(x.float(), -e[..., None]).to(E4M3), (e + 127).to(torch.uint8)


def _plain_write(s):
    (t, kv, dim), n, page = s["k"].shape, s["pages"].shape[0], s["page"]
    at_page, at_off = s["place_page"].long(), s["place_off"].long()
    (kc, ke), (vc, ve) = _quantised(s["k"]), _quantised(s["v"])
    codes = s["pages"].view(torch.uint8)
    codes[:, 0].view(n, kv, page, dim)[at_page, :, at_off] = kc.view(torch.uint8)
    codes[:, 1].view(n, kv, dim, page)[at_page, :, :, at_off] = vc.view(torch.uint8)
    scales = s["scales"].view(torch.uint8)
    scales[at_page, 0, :, at_off] = ke
    scales[at_page, 1, :, at_off] = ve
    return {"pages": s["pages"], "scales": s["scales"]}


def _plain_read(s):
    n, kv, dim, page = s["pages"].shape[0], s["kv_heads"], s["dim"], s["page"]
    at_page, at_off = s["place_page"].long(), s["place_off"].long()
    codes, scales = s["pages"].view(torch.uint8), s["scales"].view(torch.uint8)
    k = codes[:, 0].view(n, kv, page, dim)[at_page, :, at_off].view(E4M3).float()
    v = codes[:, 1].view(n, kv, dim, page)[at_page, :, :, at_off].view(E4M3).float()
    ke, ve = _power(scales[at_page, 0, :, at_off]), _power(scales[at_page, 1, :, at_off])
    return {"k": (k * ke[..., None]).to(TYPES[s["type"]]), "v": (v * ve[..., None]).to(TYPES[s["type"]])}


def _attend_rows(s, lo, hi, most):
    """Rows lo .. hi - 1 side by side, padded to `most` query tokens and the longest context; -> [tokens, heads, D], float32. What a
    mask leaves out leaves no trace."""
    page, kv, dim, (t, heads, _) = s["page"], s["kv_heads"], s["dim"], s["q"].shape
    b, group, wide = hi - lo, heads // kv, s["table"].shape[1]
    at = s["table"][s["slots"][lo:hi].long()].long()                                     # [B, pages]
    held = s["pages"].view(torch.uint8)[at].view(E4M3) if s["scales"] is not None else s["pages"][at]
    k = held[:, :, 0].reshape(b, wide, kv, page, dim).transpose(1, 2).reshape(b, kv, wide * page, dim).float()
    v = held[:, :, 1].reshape(b, wide, kv, dim, page).permute(0, 2, 1, 4, 3).reshape(b, kv, wide * page, dim).float()
    if s["scales"] is not None:
        e = _power(s["scales"].view(torch.uint8)[at])                                    # [B, pages, 2, kv, P]
        k = k * e[:, :, 0].transpose(1, 2).reshape(b, kv, wide * page, 1)
        v = v * e[:, :, 1].transpose(1, 2).reshape(b, kv, wide * page, 1)
    lens, start = s["lens"][lo:hi].long(), s["query_start"][lo:hi + 1].long()
    counts = start[1:] - start[:-1]
    place = torch.arange(most, device=DEV)
    token = (start[:-1, None] + place).clamp(max=t - 1)                                  # [B, most]
    q = s["q"][token].float().view(b, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, group * most, dim)
    key = torch.arange(wide * page, device=DEV)
    position = (lens - counts)[:, None] + place                                          # [B, most]
    seen = (key <= position[..., None]) & (key < lens[:, None, None])
    if s.get("window"):
        seen &= key > position[..., None] - s["window"]
    v = torch.where((key < lens[:, None])[:, None, :, None], v, 0.0)
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(b, kv, group, most, wide * page) * s["scale"]
    scores = torch.where(seen[:, None, None], scores, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights.view(b, kv, group * most, wide * page), v).view(b, kv, group, most, dim) / total.clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4).reshape(b, most, heads, dim)[place < counts[:, None]]


def _plain_attend(s):
    b = s["slots"].shape[0]
    if not s.get("long"):
        return _attend_rows(s, 0, b, s["query"]).to(s["q"].dtype)
    short = _attend_rows(s, 0, b - 1, s["query"]) if b > 1 else s["q"][:0].float()       # a portion is the last row
    return torch.cat((short, _attend_rows(s, b - 1, b, s["long"]))).to(s["q"].dtype)


def _plain_verify(s):
    start, b, n, vocab, most = s["start"].long(), s["requests"], s["logits"].shape[0], s["vocab"], s["drafts"]
    counts = start[1:] - start[:-1]
    row = torch.repeat_interleave(torch.arange(b, device=DEV), counts, output_size=n)
    logits, heat = s["logits"].double(), s["temperature"].double()
    greedy = heat <= 0
    z = logits / torch.where(greedy, 1.0, heat)[row, None]
    e = torch.exp(z - z.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    best = logits.argmax(-1)
    drafted = s["drafted"].long()
    mine = torch.arange(n, device=DEV)
    q = s["draft_probs"][mine, drafted].double() if s["draft_probs"] is not None else torch.ones(n, dtype=F64, device=DEV)
    good = torch.where(greedy[row], drafted == best, s["accept"].double() * q <= p[mine, drafted])
    place = torch.arange(most + 1, device=DEV)
    at = (start[:-1, None] + place).clamp(max=n - 1)                                     # [B, most + 1]
    held = (place < counts[:, None] - 1) & good[at]
    accepted = held.long().cumprod(-1).sum(-1)
    end = start[:-1] + accepted
    rest = p[end]
    judged = (accepted < counts - 1)[:, None]                                            # a draft was turned down there
    less = s["draft_probs"][end].double() if s["draft_probs"] is not None else torch.nn.functional.one_hot(drafted[end], vocab) * 2.0
    left = (rest - less).clamp(min=0)
    left = torch.where(judged & (left.sum(-1, keepdim=True) > 0), left, rest)
    cumulated = left.cumsum(-1)
    drawn = (cumulated > s["draw"].double()[:, None] * cumulated[:, -1:]).to(torch.uint8).argmax(-1)
    last = torch.where(greedy, best[end], drawn)
    tokens = torch.where(place < accepted[:, None], drafted[at], torch.where(place == accepted[:, None], last[:, None], -1))
    return {"tokens": tokens.to(I32), "accepted": accepted.to(I32)}


def run(state):
    if own:
        return _run_own(state)
    return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "prefix": _plain_attend, "verify": _plain_verify}[state["kind"]](state)


# -- what a pass cannot do without ----------------------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "verify":
        b, k, v = case["requests"], case["drafts"], case["vocab"]
        n = b * (k + 1)
        return {"bytes": 4 * v * (n + (b if case["probs"] else 0)) + 20 * n, "flops": 4 * v * n}
    kv, dim, size = case["kv_heads"], case["dim"], 2 if case["type"] == "bfloat16" else 4
    if case["kind"] in ("write", "read"):
        rows = 2 * kv * case["tokens"]
        return {"bytes": rows * (dim * size + dim + 1) + 8 * case["tokens"], "flops": 2 * rows * dim}
    heads, held = case["heads"], dim + 1 if case["kind"] == "attend" or case["cache8"] else 2 * dim
    if case["kind"] == "attend":
        rows, length, window = case["rows"], case["len"], case["window"] or case["len"]
        short = rows - 1 if case["long"] else rows
        mean = (length + length / 3) / 2 if rows > 1 else length
        near = min(mean, window + case["query"])
        queries = short * case["query"] + case["long"]
        seen = short * near + (min(length, window + case["long"]) if case["long"] else 0)
        pairs = short * case["query"] * min(mean, window) + case["long"] * min(max(length - case["long"] / 2, 1), window)
    else:
        rows = case["groups"] * case["rows"]
        queries, prefix = rows * case["query"], 0.75 * case["prefix"]
        seen = case["groups"] * prefix + rows * case["len"] / 2
        pairs = queries * (prefix + case["len"] / 2)
    return {"bytes": 2 * kv * held * seen + 2 * queries * heads * dim * size, "flops": 4 * pairs * heads * dim}


# -- the definitions in 64 bits ---------------------------------------------------------------------------------------------------

def _rounded(y):
    """The float8_e4m3fn value nearest to each y, ties to the even one: steps of 2^-3 of the value's power of two, 2^-9 the finest."""
    power = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    step = torch.exp2(power - 3)
    return torch.round(y / step) * step


def _exact_write(s):
    kv, dim, page = s["kv_heads"], s["dim"], s["page"]
    pages, scales = s["pages"].to(F64), s["scales"].to(F32).to(F64)
    where = (s["place_page"].long(), s["place_off"].long())
    for part, x in enumerate((s["k"].double(), s["v"].double())):
        e = torch.ceil(torch.log2(x.abs().amax(-1) / 448)).clamp(min=-126)
        code = _rounded(x / torch.exp2(e)[..., None])                                    # [T, kv, dim]
        scales[where[0], part, :, where[1]] = torch.exp2(e)
        for head in range(kv):
            inner = torch.arange(dim, device=DEV)
            flat = where[1][:, None] * dim + inner if part == 0 else inner * page + where[1][:, None]
            pages[where[0][:, None], part, head, flat] = code[:, head]
    return {"pages": pages, "scales": scales}


def _exact_read(s):
    kv, dim, page, got = s["kv_heads"], s["dim"], s["page"], {}
    inner = torch.arange(dim, device=DEV)
    for part, name in enumerate("kv"):
        off = s["place_off"].long()[:, None]
        flat = off * dim + inner if part == 0 else inner * page + off
        rows = [s["pages"][s["place_page"].long(), part, head].double().gather(1, flat)
                * s["scales"].to(F32).double()[s["place_page"].long(), part, head].gather(1, off) for head in range(kv)]
        got[name] = torch.stack(rows, 1)
    return got


def _exact_attend(s):
    kv, dim, page, start = s["kv_heads"], s["dim"], s["page"], s["query_start"].tolist()
    group = s["heads"] // kv
    out = torch.zeros(s["q"].shape, dtype=F64, device=DEV)
    for b, n in enumerate(s["lens"].tolist()):
        lo, hi = start[b], start[b + 1]
        at = s["table"][int(s["slots"][b])].long()[: -(-n // page)]
        position = torch.arange(n - (hi - lo), n, device=DEV)[:, None]
        key = torch.arange(n, device=DEV)[None]
        hidden = key > position
        if s.get("window"):
            hidden |= position - key >= s["window"]
        for head in range(kv):
            k = s["pages"][at, 0, head].double().view(-1, dim)[:n]
            v = s["pages"][at, 1, head].double().view(-1, dim, page).permute(1, 0, 2).reshape(dim, -1)[:, :n]
            if s["scales"] is not None:
                k = k * s["scales"][at, 0, head].to(F32).double().reshape(-1, 1)[:n]
                v = v * s["scales"][at, 1, head].to(F32).double().reshape(1, -1)[:, :n]
            for i in range(head * group, (head + 1) * group):
                x = (s["q"][lo:hi, i].double() @ k.T.contiguous()).mul_(s["scale"]).masked_fill_(hidden, -torch.inf)
                out[lo:hi, i] = torch.softmax(x, -1) @ v.T.contiguous()
    return out


def exact(case, seed):
    if case["kind"] == "verify":
        return None                                                                      # whole numbers
    s = prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read, "attend": _exact_attend, "prefix": _exact_attend}[case["kind"]](s)
