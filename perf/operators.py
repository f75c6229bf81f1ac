"""The calls that a serving step's operators are judged by: keys and values written into a paged
cache (as they are, or in 8 bits with a scale for each token and head), the cache read back into
the contiguous layout of the other attention calls, attention of each sequence's new tokens over
its pages, and the choice of the next tokens from the logits and given random numbers.

A case is a dict of plain values.  `op` names the operator:

  write, read, attention   batch; seq: cached positions of the longest sequence, its new tokens
                           among them; fresh: new tokens of the longest chunk; kind: how the
                           lengths are spread (_lengths); heads, kv_heads, head_dim, page; dtype:
                           of K, V, Q and O; cache: of the pages
  sample                   rows, vocab, dtype, cut: whether rows bring top-k, top-p and min-p

A page is [kv_heads][page][head_dim].  A token's K or V of one head is held in 8 bits as codes and
one f32 scale: with a the largest magnitude of its values and M that of the type (448 in e4m3, 127
in i8), scale = a / M and code = the type's nearest to x * (M / a), each product and quotient
rounded to f32; value = code * scale.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
          "e4m3": torch.float8_e4m3fn, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "i8": 1}
MOST = {"e4m3": 448.0, "i8": 127.0}


def _framework():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tile-rs_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import tilers_hip
    return tilers_hip


def listed():
    gqa = dict(heads=32, kv_heads=8, head_dim=128)
    return [
        # a decode step of a few short sequences: one launch's latency
        dict(name="attention step", op="attention", kind="even", batch=4, seq=500, fresh=1, **gqa,
             page=16, dtype="bf16", cache="bf16"),
        # a decode step of a full server, sequences of all ages: the cache's bandwidth
        dict(name="attention steps", op="attention", kind="ragged", batch=64, seq=8192, fresh=1,
             **gqa, page=64, dtype="bf16", cache="bf16"),
        # the same with the cache in 8 bits, few and long sequences
        dict(name="attention long e4m3", op="attention", kind="ragged", batch=3, seq=32001,
             fresh=1, **gqa, page=128, dtype="bf16", cache="e4m3"),
        # one chunk of a long prompt after what is cached already: the largest product
        dict(name="attention chunk", op="attention", kind="even", batch=1, seq=8192, fresh=512,
             **gqa, page=64, dtype="bf16", cache="bf16"),
        # prompts of any length at once, nothing cached before them, narrow heads
        dict(name="attention prompts e4m3", op="attention", kind="prompts", batch=5, seq=2000,
             fresh=2000, heads=16, kv_heads=2, head_dim=64, page=32, dtype="f16", cache="e4m3"),
        # a step that checks a few drafted tokens of each sequence, others idle
        dict(name="attention drafts i8", op="attention", kind="ragged", batch=17, seq=3001,
             fresh=5, **gqa, page=16, dtype="bf16", cache="i8"),
        # the step's own keys and values into the cache
        dict(name="write step e4m3", op="write", kind="ragged", batch=64, seq=2048, fresh=1,
             **gqa, page=64, dtype="bf16", cache="e4m3"),
        # the keys and values of whole prompts into the cache
        dict(name="write prompts i8", op="write", kind="prompts", batch=8, seq=4096, fresh=4096,
             **gqa, page=32, dtype="bf16", cache="i8"),
        # a cache in 8 bits back for an attention over contiguous 16-bit keys
        dict(name="read e4m3", op="read", kind="ragged", batch=8, seq=8192, fresh=1, **gqa,
             page=64, dtype="bf16", cache="e4m3"),
        # the cached part of a few sequences, a copy
        dict(name="read f16", op="read", kind="ragged", batch=3, seq=1999, fresh=1, heads=16,
             kv_heads=2, head_dim=64, page=16, dtype="f16", cache="f16"),
        # the next tokens of a few sequences, without cuts
        dict(name="sample step", op="sample", rows=8, vocab=128256, dtype="bf16", cut=False),
        # the next tokens of many sequences, rows that are not 16-byte aligned
        dict(name="sample batch", op="sample", rows=256, vocab=50257, dtype="f32", cut=True),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "write", "read", "sample"])
    if op == "sample":
        vocab = _log(rng, 1000, 152064)
        return dict(op=op, rows=_log(rng, 1, min(256, (1 << 24) // vocab)), vocab=vocab,
                    dtype=rng.choice(["f32", "bf16", "f16"]), cut=rng.random() < 0.7)
    heads, kv_heads = rng.choice([(32, 8), (32, 32), (16, 2), (8, 8)])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    case = dict(op=op, heads=heads, kv_heads=kv_heads, head_dim=rng.choice([128, 128, 64]),
                page=rng.choice([16, 32, 64, 128, 256]), dtype=dtype,
                cache=rng.choice([dtype, dtype, "e4m3", "i8"]))
    kind = rng.choice(["even", "ragged", "ragged", "prompts", "mixed"])
    batch = _log(rng, 1, 8 if kind == "prompts" else 16 if kind == "mixed" else 64)
    # values of K in the batch, and scores over all heads, at most
    values, scores = 1 << 28 if op == "attention" else 1 << 26, 1 << 26
    most = values // (batch * kv_heads * case["head_dim"])
    if kind == "prompts":
        seq = _log(rng, 16, max(16, min(4096, most, int((scores / (batch * heads)) ** 0.5))))
        return case | dict(kind=kind, batch=batch, seq=seq, fresh=seq)
    seq = _log(rng, 64, max(64, min(32768, most)))
    if kind == "mixed" or rng.random() < 0.3:
        fresh = _log(rng, 2, max(2, min(seq, 1024, scores // (batch * heads * seq))))
    else:
        fresh = rng.choice([1, 1, _log(rng, 2, 8)])
    return case | dict(kind=kind, batch=batch, seq=seq, fresh=fresh)


def _lengths(case):
    """Each sequence's new tokens and cached positions, the new ones among them.  even: all alike;
    ragged: from a quarter of the positions on, every eighth slot idle; prompts: nothing cached
    before the new tokens, from a quarter on; mixed: one long chunk, the others one token each."""
    n, kind, seq, fresh = case["batch"], case["kind"], case["seq"], case["fresh"]
    rng = random.Random(1000003 * n + seq)
    new, total = [fresh] * n, [seq] * n
    for b in range(n):
        if kind == "even" or b == 0:
            continue
        total[b] = rng.randint(max(1, seq // 4), seq)
        if kind == "prompts":
            new[b] = total[b]
        else:
            new[b] = min(total[b], 1 if kind == "mixed" else fresh)
        if kind == "ragged" and b % 8 == 7:
            new[b] = 0
    return new, total


def _paged(case, seed):
    """The pool of pages, the sequences' tables and lengths, and their new tokens' Q, K and V."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    new, total = _lengths(case)
    h, hk, d, page, cache = (case[k] for k in ("heads", "kv_heads", "head_dim", "page", "cache"))
    each = [-(-t // page) for t in total]
    used, width = sum(each), max(each)
    pages = used + 3   # a pool is a little larger than what is in use
    order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    place = torch.full((case["batch"], width), -1, dtype=torch.int32)
    at = 0
    order = order.cpu()
    for b, n in enumerate(each):
        place[b, :n] = order[at:at + n]
        at += n
    tokens = sum(new)

    def normal(*shape, dtype):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=g)

    s = dict(case=case, table=place.cuda(), tokens=tokens, pages=pages,
             start=torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32,
                                device="cuda"),
             length=torch.tensor(total, dtype=torch.int32, device="cuda"),
             most=(max(new), max(total)))
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "write":
        # one projection's output, Q before K and V: rows with a stride
        s["qkv"] = normal(tokens, (h + 2 * hk) * d, dtype=dtype)
    if case["op"] == "attention":
        s["q"] = normal(tokens, h, d, dtype=dtype)
        s["o"] = torch.zeros_like(s["q"])
    if case["op"] == "read":
        for name in ("k_out", "v_out"):
            s[name] = torch.zeros(case["batch"], hk, max(total), d, dtype=dtype, device="cuda")
    for name in ("k", "v"):
        shape = (pages, hk, page, d)
        if cache in MOST:
            if cache == "i8":
                code = torch.randint(-127, 128, shape, generator=g, device="cuda",
                                     dtype=torch.int8)
            else:
                code = normal(*shape, dtype=torch.bfloat16).mul_(150.0).clamp_(-448.0, 448.0)
            s[name] = code.to(DTYPES[cache])
            s[name + "_scale"] = torch.empty(shape[:3], device="cuda").uniform_(
                1.2 / MOST[cache], 3.0 / MOST[cache], generator=g)
        else:
            s[name] = normal(*shape, dtype=DTYPES[cache])
            s[name + "_scale"] = None
    return s


def _logits(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows = case["rows"]

    def uniform(lo, hi):
        return torch.empty(rows, device="cuda").uniform_(lo, hi, generator=g)

    x = torch.empty(rows, case["vocab"], device="cuda").normal_(0.0, 2.5, generator=g)
    s = dict(case=case, logits=x.to(DTYPES[case["dtype"]]), uniform=uniform(0.0, 1.0),
             temperature=uniform(0.5, 1.3), top_k=None, top_p=None, min_p=None,
             out=torch.empty(rows, dtype=torch.int32, device="cuda"))
    s["temperature"][3::16] = 0.0   # some rows ask for the likeliest token
    if case["cut"]:
        s["top_k"] = torch.randint(1, 1000, (rows,), generator=g, device="cuda",
                                   dtype=torch.int32)
        s["top_k"][1::4] = 0        # and some bring no limit
        s["top_p"] = uniform(0.5, 1.0)
        s["top_p"][2::4] = 1.0
        s["min_p"] = uniform(0.0, 0.1)
        s["min_p"][::2] = 0.0
    return s


def prepare(case, seed):
    if case["op"] == "sample":
        s = _logits(case, seed)
    else:
        s = _paged(case, seed)
    if own:
        th = s["th"] = _framework()
        types = {"f32": th.TileDtype.F32, "f16": th.TileDtype.F16, "bf16": th.TileDtype.BF16,
                 "e4m3": th.TileDtype.E4M3, "i8": th.TileDtype.I8}
        s["dtype"] = types[case["dtype"]]
        if case["op"] != "sample":
            s["cache"] = th.KvPages(
                s["k"].data_ptr(), s["v"].data_ptr(), s["pages"], case["page"], case["kv_heads"],
                case["head_dim"], types[case["cache"]],
                k_scale=None if s["k_scale"] is None else s["k_scale"].data_ptr(),
                v_scale=None if s["v_scale"] is None else s["v_scale"].data_ptr())
            s["seqs"] = th.KvBatch(s["table"].data_ptr(), s["start"].data_ptr(),
                                   s["length"].data_ptr(), case["batch"], s["table"].shape[1],
                                   s["tokens"])
        if case["op"] == "attention":
            s["room"] = th.attention_paged_workspace_size(s["cache"], s["seqs"], case["heads"])
            s["workspace"] = torch.empty(max(16, s["room"]), dtype=torch.uint8, device="cuda")
    return s


def _new_kv(s):
    """The new tokens' K and V, views into the projection's output."""
    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["head_dim"]
    k, v = (s["qkv"][:, (h + i * hk) * d:(h + (i + 1) * hk) * d] for i in range(2))
    return k, v


def _tokens(s):
    """Sequence and position of each new token."""
    start, tokens = s["start"].long(), s["tokens"]
    token = torch.arange(tokens, device="cuda")
    b = torch.searchsorted(start, token, right=True) - 1
    return b, s["length"][b].long() - (start[b + 1] - token)


def _write(s):
    c = s["case"]
    b, at = _tokens(s)
    page, row = s["table"][b, at // c["page"]].long(), at % c["page"]
    k, v = _new_kv(s)
    x = torch.stack([k, v]).float().unflatten(-1, (c["kv_heads"], c["head_dim"]))
    if c["cache"] in MOST:
        most = x.abs().amax(dim=-1)
        range_ = torch.full_like(most, MOST[c["cache"]])   # (a number would be multiplied by)
        code = x * (range_ / most).unsqueeze(-1)
        if c["cache"] == "i8":
            code = code.round()
        x = code.to(DTYPES[c["cache"]]).view(torch.uint8)
        scale = most / range_
        s["k_scale"][page, :, row], s["v_scale"][page, :, row] = scale[0], scale[1]
        s["k"].view(torch.uint8)[page, :, row], s["v"].view(torch.uint8)[page, :, row] = x[0], x[1]
    else:
        x = x.to(DTYPES[c["cache"]])
        s["k"][page, :, row], s["v"][page, :, row] = x[0], x[1]


def _gather(s, name):
    """K or V of every sequence in f32, [batch][kv_heads][positions][head_dim]."""
    table = s["table"].clamp(min=0).long()
    x = s[name].view(torch.uint8)[table].view(s[name].dtype).float()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][table].unsqueeze(-1)
    return x.transpose(1, 2).flatten(2, 3)[:, :, :s["most"][1]]


def _read(s):
    position = torch.arange(s["most"][1], device="cuda")
    held = (position < s["length"].unsqueeze(-1))[:, None, :, None]
    return [torch.where(held, _gather(s, a).to(s[b].dtype), s[b])
            for a, b in (("k", "k_out"), ("v", "v_out"))]


def _attention(s):
    c = s["case"]
    n, (new, total), hk, d = c["batch"], s["most"], c["kv_heads"], c["head_dim"]
    group = c["heads"] // hk
    start = s["start"].long()
    count = start[1:] - start[:-1]
    index = torch.arange(new, device="cuda")
    live = index < count.unsqueeze(-1)                       # [batch][new]
    token = (start[:-1].unsqueeze(-1) + index).clamp(max=s["tokens"] - 1)
    q = s["q"].float()[token].view(n, new, hk, group, d).permute(0, 2, 1, 3, 4)
    k, v = _gather(s, "k"), _gather(s, "v")
    position = torch.arange(total, device="cuda")
    last = (s["length"].long() - count).unsqueeze(-1) + index
    seen = (position <= last.unsqueeze(-1)) & live.unsqueeze(-1)   # [batch][new][total]
    seen = seen[:, None, :, None]
    score = q.flatten(2, 3) @ k.transpose(2, 3).contiguous() / math.sqrt(d)
    score = score.unflatten(2, (new, group)).masked_fill_(~seen, float("-inf"))
    top = score.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weight = score.sub_(top).exp_()
    total_weight = weight.sum(dim=-1)
    v = v.masked_fill((position >= s["length"].unsqueeze(-1))[:, None, :, None], 0.0)
    o = (weight.flatten(2, 3) @ v).unflatten(2, (new, group))
    o = torch.where(total_weight.unsqueeze(-1) > 0, o / total_weight.unsqueeze(-1), 0.0)
    return o.permute(0, 2, 1, 3, 4).reshape(n, new, c["heads"], d)[live].to(s["q"].dtype)


def _sample(s):
    # in 64 bits: cumulative masses next to the cuts and to the random number
    x, t = s["logits"].double(), s["temperature"].double().unsqueeze(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    weight = ((order.values - order.values[:, :1]) / t.clamp(min=1e-30)).exp()
    rank = torch.arange(x.shape[1], device="cuda")
    kept = torch.ones_like(x, dtype=torch.bool)
    if s["top_k"] is not None:
        limit = s["top_k"].unsqueeze(-1)
        kept = (rank < limit) | (limit <= 0)
    if s["top_p"] is not None:
        part = weight * kept
        before = part.cumsum(dim=-1) - part
        whole, most = part.sum(dim=-1, keepdim=True), s["top_p"].double().unsqueeze(-1)
        kept = kept & ((before < most * whole) | (most >= 1))
    if s["min_p"] is not None:
        kept = kept & (weight >= s["min_p"].double().unsqueeze(-1))
    kept = (kept | (rank == 0)) & ((t > 0) | (rank == 0))
    weight = torch.zeros_like(x).scatter_(1, order.indices, weight * kept)
    mass = weight.cumsum(dim=-1)
    over = mass > s["uniform"].double().unsqueeze(-1) * mass[:, -1:]
    return over.int().argmax(dim=-1).int()


def run(s):
    c, op = s["case"], s["case"]["op"]
    if own:
        th = s["th"]
        if op == "write":
            k, v = _new_kv(s)
            th.kv_cache_write(s["cache"], s["seqs"], k.data_ptr(), v.data_ptr(), s["dtype"],
                              stride=k.stride(0))
        elif op == "read":
            th.kv_cache_read(s["cache"], s["seqs"], s["k_out"].data_ptr(), s["v_out"].data_ptr(),
                             s["most"][1], s["dtype"])
            return [s["k_out"], s["v_out"]]
        elif op == "attention":
            th.attention_paged(s["q"].data_ptr(), s["cache"], s["seqs"], s["o"].data_ptr(),
                               c["heads"], s["dtype"], workspace=s["workspace"].data_ptr(),
                               workspace_bytes=s["room"])
            return s["o"]
        else:
            cuts = (None if x is None else x.data_ptr()
                    for x in (s["temperature"], s["top_k"], s["top_p"], s["min_p"]))
            th.sample(s["logits"].data_ptr(), s["out"].data_ptr(), c["rows"], c["vocab"],
                      s["dtype"], s["uniform"].data_ptr(), *cuts)
            return s["out"]
    elif op == "write":
        _write(s)
    else:
        return {"read": _read, "attention": _attention, "sample": _sample}[op](s)
    return [s[k] for k in ("k", "v", "k_scale", "v_scale") if s[k] is not None]


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZE[case["dtype"]] + 20 * case["rows"], "flops": 4 * n}
    new, total = _lengths(case)
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    held = hk * (d * SIZE[case["cache"]] + (4 if case["cache"] in MOST else 0))
    plain = SIZE[case["dtype"]] * d
    if case["op"] == "write":
        return {"bytes": 2 * sum(new) * (held + hk * plain), "flops": 4 * sum(new) * hk * d}
    if case["op"] == "read":
        return {"bytes": 2 * sum(total) * (held + hk * plain), "flops": 2 * sum(total) * hk * d}
    pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))
    return {"bytes": 2 * sum(new) * h * plain + 2 * sum(t for n, t in zip(new, total) if n) * held,
            "flops": 4 * h * d * pairs}


def _value(s, name, b, g):
    """K or V of head g of sequence b in 64 bits, [positions][head_dim]."""
    page, n = s["case"]["page"], int(s["length"][b])
    at = s["table"][b, :-(-n // page)].long()
    x = s[name].view(torch.uint8)[at, g].view(s[name].dtype).double()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][at, g].double().unsqueeze(-1)
    return x.reshape(-1, x.shape[-1])[:n]


def exact(case, seed):
    op = case["op"]
    if op == "sample":
        return None   # whole numbers
    s = _paged(case, seed)
    new, total = _lengths(case)
    if op == "attention":
        o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        group, at = case["heads"] // case["kv_heads"], 0
        for b, (n, t) in enumerate(zip(new, total)):
            if n == 0:
                continue
            hidden = torch.ones(n, t, dtype=torch.bool, device="cuda").triu(t - n + 1)
            for g in range(case["kv_heads"]):
                k, v = (_value(s, name, b, g) for name in ("k", "v"))
                for h in range(g * group, (g + 1) * group):
                    score = s["q"][at:at + n, h].double() @ k.t().contiguous()
                    score = (score / case["head_dim"] ** 0.5).masked_fill(hidden, -math.inf)
                    o[at:at + n, h] = torch.softmax(score, dim=-1) @ v
            at += n
        return o
    if op == "read":
        out = [s[k].double() for k in ("k_out", "v_out")]
        for b, t in enumerate(total):
            for g in range(case["kv_heads"]):
                for x, name in zip(out, ("k", "v")):
                    x[b, g, :t] = _value(s, name, b, g)
        return out
    # write: the pool with each new token's codes (or values) and scales in their places
    held, scales = [s[k].double() for k in ("k", "v")], []
    if case["cache"] in MOST:
        scales = [s[k].double() for k in ("k_scale", "v_scale")]
    at = 0
    for n, t, table in zip(new, total, s["table"]):
        where = torch.arange(t - n, t, device="cuda")
        page, row = table[where // case["page"]].long(), where % case["page"]
        for i, x in enumerate(_new_kv(s)):
            x = x[at:at + n].double().view(n, case["kv_heads"], case["head_dim"])
            if case["cache"] in MOST:
                a = x.abs().amax(dim=-1)
                scales[i][page, :, row] = a / MOST[case["cache"]]
                # the definition rounds the factor and the product to f32
                x = x * (torch.full_like(a, MOST[case["cache"]]) / a).float().double().unsqueeze(-1)
                x = x.float().double()
                if case["cache"] == "e4m3":   # steps of an eighth of the power of two below
                    step = torch.exp2(torch.frexp(x).exponent.clamp(min=-5).double() - 4)
                    x = (x / step).round() * step
                else:
                    x = x.round()
            held[i][page, :, row] = x
        at += n
    return held + scales
