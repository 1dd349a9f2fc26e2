"""Performance cases of the operators that serve many completions of shared prompts.

`shared`  decode attention of a batch whose sequences share long prefixes, each prefix read once per group
`fork`    new block-table rows that share their parent's KV pages (the unfinished last page is copied)
`retire`  finished sequences give their pages back, and the pages still held move to the front of the cache
`draw`    tokens from logits and given uniform numbers: temperature, top-k, top-p, min-p

`run` computes an operator in plain torch operations, or calls `bloom_b200.ops` where `own` is set.
"""
import math
import random

import torch

own = False

PAGE = 16
DEV = "cuda"


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # --- shared-prefix decode: one layer's attention of a decode step
        # four completions of one short prompt, just begun (the latency end)
        dict(name="shared-n4-p512", op="shared", heads=32, kv_heads=8, dim=128, groups=1, members=4, uneven=0,
             prefix=512, prefix_step=0, suffix_lo=1, suffix_hi=24, q_len=1),
        # 32 completions of one prompt, in mid-generation
        dict(name="shared-n32-p4096", op="shared", heads=32, kv_heads=8, dim=128, groups=1, members=32, uneven=0,
             prefix=4096, prefix_step=0, suffix_lo=33, suffix_hi=300, q_len=1),
        # a full batch of 256 requests behind one long system prompt
        dict(name="shared-n256-p8192", op="shared", heads=32, kv_heads=8, dim=128, groups=1, members=256, uneven=0,
             prefix=8192, prefix_step=0, suffix_lo=1, suffix_hi=511, q_len=1),
        # 64-wide heads in groups of three, several prompts of odd page counts, uneven groups
        dict(name="shared-d64-odd", op="shared", heads=9, kv_heads=3, dim=64, groups=7, members=9, uneven=5,
             prefix=1008, prefix_step=112, suffix_lo=1, suffix_hi=77, q_len=1),
        # 16 prompts with 8 completions each, verifying four proposed tokens per sequence
        dict(name="shared-g16-verify", op="shared", heads=64, kv_heads=8, dim=128, groups=16, members=8, uneven=0,
             prefix=2048, prefix_step=-64, suffix_lo=5, suffix_hi=260, q_len=4),
        # --- forks: bf16 pages, then int8 pages
        # four completions of one prompt on a small model
        dict(name="fork-n4", op="fork", layers=16, kv_heads=8, dim=64, kind="bf16", parents=1, children=4,
             len_lo=300, len_hi=300, spare=0),
        # a batch of prompts, eight completions each, on a pipeline stage of eight layers, int8 pages
        dict(name="fork-n128", op="fork", layers=8, kv_heads=8, dim=128, kind="int8", parents=16, children=128,
             len_lo=500, len_hi=2047, spare=64),
        # --- retiring: some sequences finish, the cache is compacted
        dict(name="retire-s8", op="retire", layers=16, kv_heads=8, dim=64, kind="bf16", seqs=8, done=3, shared=4,
             len_lo=40, len_hi=500, moved_pct=25, spare=64),
        # a large pool after half of a batch has finished
        dict(name="retire-s256", op="retire", layers=2, kv_heads=8, dim=128, kind="bf16", seqs=256, done=128,
             shared=16, len_lo=100, len_hi=1600, moved_pct=40, spare=2000),
        # --- drawing tokens
        # one request's next token
        dict(name="draw-b1", op="draw", rows=1, vocab=128256, draws=1, dtype="bf16", mix="nucleus"),
        # a full batch with every kind of request in it
        dict(name="draw-b256", op="draw", rows=256, vocab=128256, draws=1, dtype="bf16", mix="all"),
        # the first tokens of eight completions for each of 48 prompts, from fp32 logits
        dict(name="draw-b48-n8", op="draw", rows=48, vocab=151936, draws=8, dtype="f32", mix="all"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


HEADS = [(32, 8, 128), (32, 4, 128), (64, 8, 128), (4, 2, 128), (9, 3, 64), (32, 8, 64), (8, 2, 64)]


def draw(rng):
    op = rng.choice(["shared", "shared", "fork", "retire", "draw"])
    if op == "shared":
        top = work(listed()[2])
        while True:
            heads, kv, dim = rng.choice(HEADS)
            groups = _spread(rng, 1, 24)
            members = max(1, _spread(rng, 1, 256) // groups)
            q_len = rng.choice([1, 1, 1, 2, 4])
            lo = rng.randint(q_len, 40)
            c = dict(op=op, heads=heads, kv_heads=kv, dim=dim, groups=groups, members=members,
                     uneven=rng.randint(0, max(0, members - 1)), prefix=PAGE * _spread(rng, 1, 512),
                     prefix_step=PAGE * rng.randint(-3, 3), suffix_lo=lo, suffix_hi=lo + _spread(rng, 1, 800),
                     q_len=q_len)
            w = work(c)
            room = groups * members * (c["prefix"] + 48 * groups + c["suffix_hi"]) * kv * dim
            if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"] and room <= 256 * 8704 * 8 * 128:
                return c
    if op == "fork":
        parents = _spread(rng, 1, 24)
        lo = rng.randint(1, 900)
        dim = rng.choice([64, 128])
        return dict(op=op, layers=rng.randint(1, 8), kv_heads=rng.choice([2, 3, 4, 8]), dim=dim,
                    kind=rng.choice(["bf16", "int8"]) if dim == 128 else "bf16", parents=parents,
                    children=_spread(rng, 1, 128), len_lo=lo, len_hi=lo + rng.randint(0, 1000),
                    spare=rng.randint(0, 64))
    if op == "retire":
        seqs = _spread(rng, 2, 256)
        lo = rng.randint(1, 100)
        dim = rng.choice([64, 128])
        return dict(op=op, layers=rng.randint(1, 2), kv_heads=rng.choice([2, 3, 4, 8]), dim=dim,
                    kind=rng.choice(["bf16", "int8"]) if dim == 128 else "bf16", seqs=seqs,
                    done=rng.randint(0, seqs), shared=rng.choice([1, 2, 4, 8]), len_lo=lo,
                    len_hi=lo + _spread(rng, 1, 1400), moved_pct=rng.randint(0, 40), spare=rng.randint(0, 1000))
    vocab = rng.choice([49152, 128256, 151936, _spread(rng, 1, 262144)])
    return dict(op=op, rows=max(1, min(_spread(rng, 1, 256), 256 * 128256 // vocab)), vocab=vocab,
                draws=rng.choice([1, 1, 2, 8, 17]), dtype=rng.choice(["bf16", "f32"]),
                mix=rng.choice(["all", "nucleus", "plain", "top-k"]))


# ---------------------------------------------------------------- sizes that follow from a case
def _lens(n, lo, hi):
    """n lengths of [lo, hi], the same for every seed."""
    return [lo + (i * 7919 + 13) % (hi - lo + 1) for i in range(n)]


def _pages(tokens):
    return -(-tokens // PAGE)


def _shared_sizes(c):
    members = [max(1, c["members"] - (g * 3) % (c["uneven"] + 1)) for g in range(c["groups"])]
    prefix = [max(PAGE, c["prefix"] + g * c["prefix_step"]) for g in range(c["groups"])]
    suffix = _lens(sum(members), c["suffix_lo"], c["suffix_hi"])
    return members, prefix, suffix


def _page_words(c):
    """int32 words of one page of one layer: bf16 pages, or int8 pages with a 4-byte scale for each token and head."""
    return 2 * c["kv_heads"] * PAGE * (c["dim"] * 2 if c["kind"] == "bf16" else c["dim"] + 4) // 4


def _retire_sizes(c):
    """(lengths, groups that share their full prompt pages, pages held before, pages held after, pages to move).

    Sequence s belongs to group s // shared; a group shares the pages of `len_lo` tokens that are full."""
    lens = _lens(c["seqs"], c["len_lo"], c["len_hi"])
    common = c["len_lo"] // PAGE
    groups = -(-c["seqs"] // c["shared"])
    done = set(random.Random(c["seqs"] * 1009 + c["done"]).sample(range(c["seqs"]), c["done"]))
    alive = [s for s in range(c["seqs"]) if s not in done]
    before = groups * common + sum(_pages(n) - common for n in lens)
    after = len({s // c["shared"] for s in alive}) * common + sum(_pages(lens[s]) - common for s in alive)
    total = before + c["spare"]
    return lens, common, groups, sorted(done), before, after, min(after * c["moved_pct"] // 100, total - after), total


def work(case):
    c = case
    if c["op"] == "shared":
        members, prefix, suffix = _shared_sizes(c)
        kv = 2 * c["kv_heads"] * c["dim"] * 2
        rows = sum(members) * c["q_len"]
        keys = sum(prefix) + sum(suffix)
        seen = c["q_len"] * (sum(m * p for m, p in zip(members, prefix)) + sum(suffix))
        return {"bytes": keys * kv + 2 * rows * c["heads"] * c["dim"] * 2 + 4 * (_pages(keys) + sum(members)),
                "flops": 4 * seen * c["heads"] * c["dim"]}
    if c["op"] == "fork":
        lens = _lens(c["parents"], c["len_lo"], c["len_hi"])
        of = [i * c["parents"] // c["children"] for i in range(c["children"])]
        page = c["layers"] * _page_words(c) * 4
        read = len({p for p in of if lens[p] % PAGE})
        made = sum(1 for p in of if lens[p] % PAGE)
        entries = sum(_pages(lens[p]) for p in of)
        return {"bytes": (read + made) * page + 4 * entries * 4, "flops": 0}
    if c["op"] == "retire":
        lens, common, groups, done, before, after, moved, total = _retire_sizes(c)
        page = c["layers"] * _page_words(c) * 4
        return {"bytes": 2 * moved * page + 4 * (3 * total + 2 * sum(_pages(n) for n in lens)), "flops": 0}
    size = 2 if c["dtype"] == "bf16" else 4
    return {"bytes": c["rows"] * c["vocab"] * size + 8 * c["rows"] * c["draws"] + 16 * c["rows"],
            "flops": 6 * c["rows"] * c["vocab"]}


# ---------------------------------------------------------------- the inputs
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def prepare(case, seed):
    return {"shared": _prepare_shared, "fork": _prepare_fork, "retire": _prepare_retire,
            "draw": _prepare_draw}[case["op"]](case, seed)


def _prepare_shared(c, seed):
    members, prefix, suffix = _shared_sizes(c)
    host, gen = random.Random(seed), _gen(seed)
    need = sum(_pages(p) for p in prefix)
    rows, lens, b = [], [], 0
    seq_prefix = []
    for m, p in zip(members, prefix):
        for _ in range(m):
            lens.append(p + suffix[b])
            seq_prefix.append(p)
            need += _pages(suffix[b])
            b += 1
    blocks = need + 3
    free = list(range(blocks))
    host.shuffle(free)
    width = max(_pages(n) for n in lens)
    b = 0
    for m, p in zip(members, prefix):
        common = [free.pop() for _ in range(_pages(p))]
        for _ in range(m):
            row = common + [free.pop() for _ in range(_pages(suffix[b]))]
            rows.append(row + [0] * (width - len(row)))
            b += 1
    cache = torch.randn(2, blocks, 2, c["kv_heads"], PAGE, c["dim"], generator=gen, device=DEV, dtype=torch.bfloat16)
    q = torch.randn(len(lens) * c["q_len"], c["heads"], c["dim"], generator=gen, device=DEV, dtype=torch.bfloat16)
    s = dict(case=c, q=q, cache=cache, layer=1, table=_ints(rows), lens=_ints(lens), out=torch.empty_like(q),
             scale=c["dim"] ** -0.5, groups=members, prefix=prefix)
    if own:  # what a serving loop keeps for as long as the groups stay as they are
        from bloom_b200 import ops

        s["plan"] = ops.shared_prefix_plan(members, prefix, num_q_heads=c["heads"], num_kv_heads=c["kv_heads"],
                                           head_dim=c["dim"], q_len=c["q_len"], max_seq_len=max(lens), device=DEV)
    return s


def _cache(c, blocks, gen):
    """The pages of all layers, as the cache's own type; random bits that are finite numbers as bf16."""
    if c["kind"] == "bf16":
        return torch.randn(c["layers"], blocks, 2, c["kv_heads"], PAGE, c["dim"], generator=gen, device=DEV,
                           dtype=torch.bfloat16)
    return torch.randint(0, 256, (c["layers"], blocks, 4 * _page_words(c)), generator=gen, device=DEV,
                         dtype=torch.uint8)


def _seen(cache):
    """A cache as an output: bf16 values, or the bytes of int8 pages as whole numbers."""
    return cache if cache.dtype == torch.bfloat16 else cache.view(torch.int32)


def _prepare_fork(c, seed):
    host = random.Random(seed)
    lens = _lens(c["parents"], c["len_lo"], c["len_hi"])
    of = [i * c["parents"] // c["children"] for i in range(c["children"])]
    blocks = sum(_pages(n) for n in lens) + c["children"] + c["spare"]
    free = list(range(blocks))
    host.shuffle(free)
    width = max(_pages(n) for n in lens) + 4
    ref = [0] * blocks
    rows = []
    for n in lens:
        row = [free.pop() for _ in range(_pages(n))]
        for p in row:
            ref[p] = 1
        rows.append(row + [0] * (width - len(row)))
    return dict(case=c, cache=_cache(c, blocks, _gen(seed)), table=_ints(rows), lens=_ints(lens), parents=_ints(of),
                fresh=_ints([free.pop() for _ in of]), ref0=_ints(ref), ref=_ints(ref))


def _prepare_retire(c, seed):
    host = random.Random(seed)
    lens, common, groups, done, before, after, moved, total = _retire_sizes(c)
    kept_low = host.sample(range(after), after - moved)
    kept_high = host.sample(range(after, total), moved)
    kept = kept_low + kept_high
    host.shuffle(kept)
    rest = sorted(set(range(total)) - set(kept))
    host.shuffle(rest)
    gone = set(done)
    ref = [0] * total
    rows = []
    width = max(_pages(n) for n in lens)
    for g in range(groups):
        seqs = [s for s in range(g * c["shared"], min(c["seqs"], (g + 1) * c["shared"]))]
        pool = kept if any(s not in gone for s in seqs) else rest
        prompt = [pool.pop() for _ in range(common)]
        for s in seqs:
            row = prompt + [(rest if s in gone else kept).pop() for _ in range(_pages(lens[s]) - common)]
            for p in row:
                ref[p] += 1
            rows.append(row + [0] * (width - len(row)))
    return dict(case=c, cache=_cache(c, total, _gen(seed)), table0=_ints(rows), lens0=_ints(lens), ref0=_ints(ref),
                table=_ints(rows), lens=_ints(lens), ref=_ints(ref), done=_ints(done))


def _prepare_draw(c, seed):
    host, gen = random.Random(seed), _gen(seed)
    rows, vocab = c["rows"], c["vocab"]
    logits = torch.randn(rows, vocab, generator=gen, device=DEV) * 2.2
    # a few likely tokens in each row, as a trained model gives
    at = torch.randint(0, vocab, (rows, min(vocab, 24)), generator=gen, device=DEV)
    logits.scatter_(1, at, torch.rand(at.shape, generator=gen, device=DEV) * 9 + 5)
    temp, top_k, top_p, min_p, masked = [], [], [], [], []
    for r in range(rows):
        kind = c["mix"] if c["mix"] != "all" else ("nucleus", "plain", "top-k", "min-p", "greedy", "both",
                                                  "masked")[(r + host.randint(0, 1) * 3) % 7]
        temp.append(0.0 if kind == "greedy" else host.choice([0.6, 0.7, 0.8, 1.0, 1.0, 1.3]))
        top_k.append(host.choice([1, 20, 40, 50, 500]) if kind in ("top-k", "both") else 0)
        top_p.append(host.choice([0.5, 0.8, 0.9, 0.95]) if kind in ("nucleus", "both") else 1.0)
        min_p.append(host.choice([0.02, 0.05, 0.1]) if kind == "min-p" else 0.0)
        masked.append(kind == "masked")
    # constrained rows: a grammar leaves one token in sixteen
    hide = torch.tensor(masked, device=DEV)[:, None] & (torch.rand(rows, vocab, generator=gen, device=DEV) > 1 / 16)
    logits.masked_fill_(hide, float("-inf"))
    if c["dtype"] == "bf16":
        logits = logits.bfloat16()

    def f(v):
        return torch.tensor(v, dtype=torch.float32, device=DEV)

    return dict(case=c, logits=logits, u=torch.rand(rows, c["draws"], generator=gen, device=DEV), temperature=f(temp),
                top_k=_ints(top_k), top_p=f(top_p), min_p=f(min_p))


# ---------------------------------------------------------------- one pass
def run(state):
    return {"shared": _run_shared, "fork": _run_fork, "retire": _run_retire, "draw": _run_draw}[state["case"]["op"]](state)


def _run_shared(s):
    c = s["case"]
    if own:
        from bloom_b200 import ops

        return ops.shared_prefix_attention(s["q"], s["cache"], s["layer"], s["table"], s["lens"], s["out"],
                                           plan=s["plan"], scale=s["scale"])
    b, width = s["table"].shape
    kv, dim, q_len = c["kv_heads"], c["dim"], c["q_len"]
    per = c["heads"] // kv
    pages = s["cache"][s["layer"]][s["table"].long()].float()  # [B, W, 2, KVH, 16, D]
    k = pages[:, :, 0].permute(0, 2, 1, 3, 4).reshape(b, kv, width * PAGE, dim)
    v = pages[:, :, 1].permute(0, 2, 1, 3, 4).reshape(b, kv, width * PAGE, dim)
    at = torch.arange(width * PAGE, device=DEV)
    there = at[None, :] < s["lens"][:, None]
    v = torch.where(there[:, None, :, None], v, 0.0)
    q = s["q"].float().view(b, q_len, kv, per, dim).permute(0, 2, 1, 3, 4).reshape(b, kv, q_len * per, dim)
    scores = (q @ k.transpose(-1, -2)).view(b, kv, q_len, per, width * PAGE) * s["scale"]
    last = s["lens"][:, None] - q_len + torch.arange(q_len, device=DEV)[None, :]  # [B, q_len]
    sees = (at[None, None, :] <= last[:, :, None])[:, None, :, None, :]
    scores = torch.where(sees, scores, float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = p.view(b, kv, q_len * per, -1) @ v
    o = o / p.sum(-1).view(b, kv, q_len * per, 1)
    return o.view(b, kv, q_len, per, dim).permute(0, 2, 1, 3, 4).reshape(b * q_len, c["heads"], dim).bfloat16()


def _run_fork(s):
    s["ref"].copy_(s["ref0"])  # every pass starts from the same counts
    if own:
        from bloom_b200 import ops

        table, lens = ops.kv_fork(s["cache"], s["table"], s["lens"], s["parents"], s["fresh"], s["ref"])
        return {"table": table, "lens": lens, "ref": s["ref"], "cache": _seen(s["cache"])}
    parents, fresh = s["parents"].long(), s["fresh"].long()
    lens = s["lens"][parents]
    at = torch.arange(s["table"].shape[1], device=DEV)[None, :]
    table = torch.where(at < ((lens + PAGE - 1) // PAGE)[:, None], s["table"][parents], 0)
    full = (lens // PAGE).long()
    partial = lens % PAGE > 0
    last = table.gather(1, full[:, None].clamp(max=table.shape[1] - 1))[:, 0].long()
    s["cache"][:, fresh] = s["cache"][:, torch.where(partial, last, fresh)]
    table = torch.where((at == full[:, None]) & partial[:, None], s["fresh"][:, None], table)
    held = at < ((lens + PAGE - 1) // PAGE)[:, None]
    s["ref"].index_add_(0, table.reshape(-1), held.reshape(-1).int())
    return {"table": table, "lens": lens, "ref": s["ref"], "cache": _seen(s["cache"])}


def _run_retire(s):
    for name in ("table", "lens", "ref"):  # every pass starts from the same sequences
        s[name].copy_(s[name + "0"])
    if own:
        from bloom_b200 import ops

        ops.kv_free(s["table"], s["lens"], s["done"], s["ref"])
        moved, used = ops.kv_compact(s["cache"], s["table"], s["lens"], s["ref"])
        return {"table": s["table"], "lens": s["lens"], "ref": s["ref"], "moved": moved, "used": used,
                "cache": _seen(s["cache"])}
    table, lens, ref, done = s["table"], s["lens"], s["ref"], s["done"].long()
    at = torch.arange(table.shape[1], device=DEV)[None, :]
    held = at < ((lens[done] + PAGE - 1) // PAGE)[:, None]
    ref.index_add_(0, table[done].reshape(-1), -held.reshape(-1).int())
    lens[done] = 0
    taken = ref > 0
    used = taken.sum(dtype=torch.int32).reshape(1)
    index = torch.arange(ref.shape[0], device=DEV)
    high = taken & (index >= used)
    hole = ~taken & (index < used)
    src, dst = high.nonzero()[:, 0], hole.nonzero()[:, 0]
    s["cache"][:, dst] = s["cache"][:, src]
    moved = torch.where(taken, index, -1).int()
    moved[src] = dst.int()
    ref[dst] = ref[src]
    ref[src] = 0
    held = at < ((lens + PAGE - 1) // PAGE)[:, None]
    table.copy_(torch.where(held, moved[table.long()], table))
    return {"table": table, "lens": lens, "ref": ref, "moved": moved, "used": used, "cache": _seen(s["cache"])}


def _run_draw(s):
    if own:
        from bloom_b200 import ops

        return ops.sample_uniform(s["logits"], s["u"], s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                  min_p=s["min_p"])
    x = s["logits"].double()
    rows, vocab = x.shape
    x = torch.where(x.isnan(), float("-inf"), x)
    best = x.amax(-1, keepdim=True)
    t = s["temperature"].double()[:, None]
    w = torch.exp((x - best) / t)
    w = torch.where(x == best, 1.0, torch.where(x == float("-inf"), 0.0, w))
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1]
    ws = w.gather(1, order)
    at = torch.arange(vocab, device=DEV)[None, :]
    k = s["top_k"][:, None]
    keep = (at < k) | (k <= 0)
    cum = torch.cumsum(torch.where(keep, ws, 0.0), -1)
    ahead = torch.cat([torch.zeros(rows, 1, dtype=torch.float64, device=DEV), cum[:, :-1]], -1)
    p = s["top_p"].double()[:, None]
    keep = keep & ((ahead < p * cum[:, -1:]) | (p >= 1) | (p <= 0))
    keep = keep & (ws >= s["min_p"].double()[:, None].clamp(max=1.0))
    kept = torch.zeros_like(keep).scatter(1, order, keep) & (w > 0)
    cum = torch.cumsum(torch.where(kept, w, 0.0), -1)
    token = torch.searchsorted(cum, s["u"].double() * cum[:, -1:], right=True)
    token = torch.minimum(token, torch.where(kept, at, -1).amax(-1, keepdim=True))
    first = torch.where(x == best, at, vocab).amin(-1, keepdim=True)
    token = torch.where(t > 0, token, first)
    return torch.where(best == float("-inf"), -1, token).int()


# ---------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"shared": _exact_shared, "fork": _exact_fork, "retire": _exact_retire, "draw": _exact_draw}[case["op"]](s)


def _exact_shared(s):
    c = s["case"]
    per = c["heads"] // c["kv_heads"]
    cache = s["cache"][s["layer"]]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lens"].tolist()):
        pages = cache[s["table"][b, :_pages(n)].long()].double()
        kv = pages.permute(1, 2, 0, 3, 4).reshape(2, c["kv_heads"], -1, c["dim"])[:, :, :n]
        for i in range(c["q_len"]):
            sees = n - c["q_len"] + i + 1
            q = s["q"][b * c["q_len"] + i].double().view(c["kv_heads"], per, c["dim"])
            p = torch.softmax(torch.einsum("hgd,hkd->hgk", q, kv[0, :, :sees]) * s["scale"], -1)
            out[b * c["q_len"] + i] = torch.einsum("hgk,hkd->hgd", p, kv[1, :, :sees]).reshape(c["heads"], c["dim"])
    return out


def _exact_fork(s):
    table, lens, ref = s["table"].tolist(), s["lens"].tolist(), s["ref0"].tolist()
    rows, new_lens = [], []
    for p, f in zip(s["parents"].tolist(), s["fresh"].tolist()):
        n = lens[p]
        row = table[p][:n // PAGE]
        for page in row:
            ref[page] += 1
        if n % PAGE:
            s["cache"][:, f].copy_(s["cache"][:, table[p][n // PAGE]])
            row = row + [f]
            ref[f] += 1
        rows.append(row + [0] * (len(table[p]) - len(row)))
        new_lens.append(n)
    return {"table": _ints(rows), "lens": _ints(new_lens), "ref": _ints(ref), "cache": _seen(s["cache"])}


def _exact_retire(s):
    table, lens, ref = s["table0"].tolist(), s["lens0"].tolist(), s["ref0"].tolist()
    for d in s["done"].tolist():
        for page in table[d][:_pages(lens[d])]:
            ref[page] -= 1
        lens[d] = 0
    used = sum(1 for r in ref if r > 0)
    holes = [p for p in range(used) if ref[p] <= 0]
    moved = [p if r > 0 else -1 for p, r in enumerate(ref)]
    for src in range(used, len(ref)):
        if ref[src] > 0:
            dst = holes.pop(0)
            s["cache"][:, dst].copy_(s["cache"][:, src])
            moved[src] = dst
            ref[dst], ref[src] = ref[src], 0
    table = [[moved[p] for p in row[:_pages(n)]] + row[_pages(n):] for row, n in zip(table, lens)]
    return {"table": _ints(table), "lens": _ints(lens), "ref": _ints(ref), "moved": _ints(moved), "used": _ints([used]),
            "cache": _seen(s["cache"])}


def _exact_draw(s):
    import numpy as np

    tokens = []
    for r in range(s["logits"].shape[0]):
        x = s["logits"][r].double().cpu().numpy()
        x = np.where(np.isnan(x), -np.inf, x)
        t, k = float(s["temperature"][r]), int(s["top_k"][r])
        p, floor = float(s["top_p"][r]), min(1.0, float(s["min_p"][r]))
        best = int(np.argmax(x))
        if x[best] == -np.inf:
            tokens.append([-1] * s["u"].shape[1])
            continue
        if not t > 0:
            tokens.append([best] * s["u"].shape[1])
            continue
        by = np.argsort(-x, kind="stable")  # falling values, ties by index
        by = by[x[by] > -np.inf]
        if k > 0:
            by = by[:k]
        w = np.exp((x[by] - x[best]) / t)
        if 0 < p < 1:
            total = np.cumsum(w)
            by = by[:1 + int(np.searchsorted(total, p * total[-1], side="left"))]
            w = w[:by.size]
        by = np.sort(by[(w >= floor) & (w > 0)])
        total = np.cumsum(np.exp((x[by] - x[best]) / t))
        tokens.append([int(by[min(by.size - 1, int(np.searchsorted(total, float(u) * total[-1], side="right")))])
                       for u in s["u"][r].tolist()])
    return _ints(tokens)
