"""Timed cases of the prompt attention over packed sequences, the 4-bit paged
key/value cache, its attention and its page operations.

Every case is one pass through one operator as a serving loop makes it.  With
`own` false `run` computes it with elementary torch operations in 32 bits, with
`own` true through the package's entry points; both take the same state.

The cache (pool) of one layer is uint8 [pages, kv_heads, page_size, 5 * hd / 4];
the bytes of one (page, head) are, in this order: the keys' codes [page_size,
hd / 2], the keys' (scale, minimum) half pairs [page_size, hd / 32, 2], the
values' codes and the values' pairs.  A value is minimum + code * scale of its
group of 32 head columns.  With NG = hd / 32 groups, the four-byte word of
eight key codes that starts at column 32 g + 8 c sits at word c * NG + g of its
row, and the two-byte unit of four value codes that starts at column 32 g + 4 n
at unit n * NG + g; code i of a word or unit is its bits 4 i .. 4 i + 3.
"""
import math
import random

import torch

own = False

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one short prompt of the smallest configuration (128 wide, 4 heads): latency alone counts
        dict(op="prompt", name="prompt one fp32", type="fp32", seqs=1, longest=16, shortest=16, heads=4, kv=4, hd=32,
             prefix=0, fused=False, pattern=1),
        # a batch of ragged prompts at the 512-wide configuration, in the library's own fp32
        dict(op="prompt", name="prompts fp32 ragged", type="fp32", seqs=32, longest=511, shortest=9, heads=8, kv=8,
             hd=64, prefix=0, fused=True, pattern=2),
        # document prompts at the 1024-wide configuration's heads, in halves, odd lengths
        dict(op="prompt", name="prompts fp16 heads 16", type="fp16", seqs=48, longest=1537, shortest=31, heads=16,
             kv=16, hd=64, prefix=0, fused=False, pattern=3),
        # long prompts with grouped heads at the 4096-wide configuration's head size
        dict(op="prompt", name="prompts bf16 grouped", type="bf16", seqs=6, longest=4096, shortest=700, heads=32, kv=8,
             hd=128, prefix=0, fused=True, pattern=4),
        # chunks of prompts whose beginning has been run before: keys lead the queries
        dict(op="prompt", name="chunks bf16 after prefix", type="bf16", seqs=4, longest=512, shortest=100, heads=32,
             kv=8, hd=128, prefix=5000, fused=False, pattern=5),
        # the new rows of one decode step of 64 sequences written to the cache and read back
        dict(op="append", name="append one row each", type="bf16", seqs=64, longest=1, shortest=1, kv=16, hd=64,
             held=1599, page=64, pattern=6),
        # whole prompts written to the cache and read back
        dict(op="append", name="append prompts", type="bf16", seqs=16, longest=2048, shortest=129, kv=8, hd=128,
             held=0, page=64, pattern=7),
        # one sequence at the start of its decode, smallest configuration
        dict(op="decode", name="decode one fp32", type="fp32", seqs=1, longest=40, shortest=40, heads=4, kv=4, hd=32,
             page=16, pattern=8),
        # one step of 64 sequences at the 1024-wide configuration, in the library's own fp32
        dict(op="decode", name="decode 64 fp32", type="fp32", seqs=64, longest=1600, shortest=1537, heads=16, kv=16,
             hd=64, page=64, pattern=9),
        # a few long sequences of very different lengths, grouped heads
        dict(op="decode", name="decode long grouped", type="bf16", seqs=8, longest=65537, shortest=2000, heads=32,
             kv=8, hd=128, page=64, pattern=10),
        # four continuations of one prompt: the shared pages counted, the page in use copied
        dict(op="fork", name="fork one into four", layers=4, kv=4, hd=32, page=16, pages=64, parents=1, children=4,
             longest=57, shortest=57, pattern=11),
        # half of the sequences of a full cache end, and the rest is moved together
        dict(op="compact", name="free half and compact", layers=8, kv=8, hd=64, page=32, pages=2600, parents=64,
             children=0, longest=1600, shortest=600, pattern=12),
    ]


def _log(rng, lo, hi):
    """A whole number spread over [lo, hi] by its logarithm."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(max(v, lo), hi)


def _length(rng, lo, hi):
    v = _log(rng, lo, hi)
    return v - 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(["prompt", "prompt", "decode", "decode", "append", "fork", "compact"])
    heads, kv, hd = rng.choice([(4, 4, 32), (8, 8, 64), (16, 16, 64), (32, 8, 128), (8, 2, 64), (6, 2, 64), (8, 1, 128),
                                (32, 32, 128), (12, 4, 32)])
    kind, page, pattern = rng.choice(sorted(TYPES)), rng.choice([16, 32, 64, 128]), rng.randrange(1, 1 << 20)
    if op == "prompt":
        # the plain form holds seqs * heads * longest * (longest + prefix) scores: at most the largest listed case's
        longest = _length(rng, 1, 4096)
        prefix = _length(rng, 1, 4096) if rng.random() < 0.3 else 0
        most = 6 * 32 * 4096 * 4096 // (heads * longest * (longest + 2 * prefix))
        seqs = _log(rng, 1, max(1, min(64, most)))
        if most < 1:
            heads, kv, hd = 8, 2, 64
        return dict(op=op, type=kind, seqs=seqs, longest=longest, shortest=_length(rng, 1, longest), heads=heads, kv=kv,
                    hd=hd, prefix=prefix, fused=heads < 16 and rng.random() < 0.5, pattern=pattern)
    if op == "decode":
        longest = _length(rng, 1, 65536)
        most = 8 * 65537 * 8 * 128 // (longest * kv * hd)
        return dict(op=op, type=kind, seqs=_log(rng, 1, max(1, min(128, most))), longest=longest,
                    shortest=_length(rng, 1, longest), heads=heads, kv=kv, hd=hd, page=page, pattern=pattern)
    if op == "append":
        longest = rng.choice([1, 1, _length(rng, 2, 2048)])
        held = rng.choice([0, _length(rng, 1, 2000)])
        most = 16 * 2048 * 8 * 128 // ((longest + held) * kv * hd)
        return dict(op=op, type=kind, seqs=_log(rng, 1, max(1, min(128, most))), longest=longest,
                    shortest=_length(rng, 1, longest), kv=kv, hd=hd, held=held, page=page, pattern=pattern)
    longest, layers = _length(rng, 1, 1600), rng.choice([1, 4, 8, 12])
    parents = _log(rng, 1, 32)
    children = _log(rng, 1, 64) if op == "fork" else 0
    pages = parents * (-(-longest // page)) + children + rng.randrange(0, 40)
    most = int(8 * 2600 * 8 * 32 * 80 // (layers * kv * page * hd * 5 // 4))
    if pages > most:
        layers, kv, hd, parents = 1, 2, 64, min(parents, 8)
        pages = parents * (-(-longest // page)) + children + rng.randrange(0, 40)
    return dict(op=op, layers=layers, kv=kv, hd=hd, page=page, pages=pages, parents=parents, children=children,
                longest=longest, shortest=_length(rng, 1, longest), pattern=pattern)


def lengths(case, count=None, salt=0):
    """The sequences' lengths: by the case alone; the longest is among them."""
    rng = random.Random(case["pattern"] * 7 + salt)
    n = case["seqs"] if count is None else count
    got = [_length(rng, case["shortest"], case["longest"]) for _ in range(n)]
    got[rng.randrange(n)] = case["longest"]
    return got


def prefixes(case):
    rng = random.Random(case["pattern"] * 7 + 3)
    return [_log(rng, max(1, case["prefix"] // 2), case["prefix"]) if case["prefix"] else 0 for _ in range(case["seqs"])]


def work(case):
    op, hd = case["op"], case["hd"]
    if op == "prompt":
        es = 4 if case["type"] == "fp32" else 2
        lq, pre = lengths(case), prefixes(case)
        lk = [a + b for a, b in zip(lq, pre)]
        pairs = sum(a * (a + 1) // 2 + a * p for a, p in zip(lq, pre))
        return {"bytes": es * hd * (2 * sum(lq) * case["heads"] + 2 * sum(lk) * case["kv"]),
                "flops": 4 * hd * case["heads"] * pairs}
    if op == "append":
        es = 4 if case["type"] == "fp32" else 2
        values = 2 * sum(lengths(case)) * case["kv"] * hd
        return {"bytes": values * (es + 2 * 0.625 + 4), "flops": 0}
    if op == "decode":
        es = 4 if case["type"] == "fp32" else 2
        keys = sum(lengths(case))
        return {"bytes": keys * case["kv"] * hd * 1.25 + 2 * es * case["seqs"] * case["heads"] * hd,
                "flops": 4 * hd * case["heads"] * keys}
    page_bytes = case["layers"] * case["kv"] * case["page"] * hd * 5 // 4
    page, lens = case["page"], lengths(case, case["parents"])
    need = [-(-n // page) for n in lens]
    meta = 4 * (case["pages"] + sum(need))
    if op == "fork":
        copied = sum(lens[p] % page != 0 for p in _parents(case))
        meta += 4 * sum(need[p] for p in _parents(case))
        return {"bytes": 2 * copied * page_bytes + meta, "flops": 0}
    order, ended = _layout(case)
    live = {p for s in range(case["parents"]) if s not in ended for p in order[s]}
    return {"bytes": 2 * sum(p >= len(live) for p in live) * page_bytes + 2 * meta, "flops": 0}


# ------------------------------------------------------ what a program holds

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)


def _normal(shape, gen, kind, spread=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * spread).to(TYPES[kind])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _key_rows(shape, gen, kind):
    """Keys with a few head columns far from zero, as trained projections give them."""
    x = torch.randn(shape, generator=gen, device=DEV)
    shift = torch.randn(shape[-2:], generator=gen, device=DEV)
    return (x + 2.0 * shift * (shift.abs() > 1.8)).to(TYPES[kind])


def _pack_codes(codes, hd, unit):
    """Codes [..., hd] (whole numbers) as bytes [..., hd / 2] in the cache's order: `unit` codes stay together."""
    groups, inner = hd // 32, 32 // unit
    x = codes.to(torch.uint8).unflatten(-1, (groups, inner, unit)).transpose(-3, -2)
    x = x.reshape(*codes.shape[:-1], hd // 2, 2)
    return x[..., 0] | (x[..., 1] << 4)


def _unpack_codes(packed, hd, unit):
    groups, inner = hd // 32, 32 // unit
    x = torch.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], inner, groups, unit)
    return x.transpose(-3, -2).reshape(*packed.shape[:-1], hd)


def _quantise(x, unit):
    """Rows [..., hd] as (packed codes, the bytes of the half pairs)."""
    hd = x.shape[-1]
    g = x.float().clamp(-65504.0, 65504.0).unflatten(-1, (hd // 32, 32))
    low = g.amin(-1, keepdim=True).half()
    scale = ((g.amax(-1, keepdim=True) - low.float()) * (1.0 / 15.0)).half()
    s = scale.float()
    inv = torch.where(s == 0, torch.zeros_like(s), torch.reciprocal(s))
    codes = torch.nan_to_num(((g - low.float()) * inv).round().clamp(0, 15)).flatten(-2)
    return _pack_codes(codes, hd, unit), torch.cat([scale, low], -1).view(torch.uint8).flatten(-2)


def _views(pool, hd):
    """The key codes, key pairs, value codes and value pairs of a layer's pool, as views of its bytes."""
    pages, heads, page, _ = pool.shape
    flat = pool.view(pages, heads, -1)
    c, m = page * hd // 2, page * hd // 8
    at = [0, c, c + m, 2 * c + m, 2 * c + 2 * m]
    part = [flat[:, :, at[i]:at[i + 1]].unflatten(-1, (page, -1)) for i in range(4)]
    return part


def _halves(raw):
    return raw.contiguous().view(torch.float16).unflatten(-1, (-1, 2))


def _values(codes, pairs, hd, unit):
    """The values, in 32 bits, that codes and pairs stand for."""
    c = _unpack_codes(codes, hd, unit).float().unflatten(-1, (hd // 32, 32))
    m = _halves(pairs).float()
    return (m[..., 1:] + c * m[..., :1]).flatten(-2)


def _filled_pool(pages, kv, page, hd, gen, kind):
    pool = torch.empty(pages, kv, page, 5 * hd // 4, dtype=torch.uint8, device=DEV)
    part = _views(pool, hd)
    step = max(1, (1 << 26) // (kv * page * hd))
    for lo in range(0, pages, step):
        n = min(step, pages - lo)
        k, km = _quantise(_key_rows((n, page, kv, hd), gen, kind).transpose(1, 2), 8)
        v, vm = _quantise(_normal((n, page, kv, hd), gen, kind, 0.5).transpose(1, 2), 4)
        for dst, src in zip(part, (k, km, v, vm)):
            dst[lo:lo + n] = src
    return pool


def _table(lens, page, seed, spare=5):
    """A table of pages in no order, -1 past a sequence's last page, and how many pages there are."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    order = list(range(total))
    random.Random(seed).shuffle(order)
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [-1] * (max(need) - n))
        at += n
    return _ints(rows).reshape(len(lens), max(need)), total


def _parents(case):
    rng = random.Random(case["pattern"] * 7 + 5)
    return [rng.randrange(case["parents"]) for _ in range(case["children"])]


def _layout(case):
    """Each parent's pages, in no order over the whole pool, and the sequences that end (compact)."""
    rng = random.Random(case["pattern"] * 7 + 6)
    need = [-(-n // case["page"]) for n in lengths(case, case["parents"])]
    order = rng.sample(range(case["pages"]), sum(need))
    at = _starts(need)
    ended = rng.sample(range(case["parents"]), (case["parents"] + 1) // 2) if case["op"] == "compact" else []
    return [order[at[i]:at[i + 1]] for i in range(case["parents"])], ended


def prepare(case, seed):
    gen, op, hd = _gen(seed), case["op"], case["hd"]
    s = dict(case)
    if op == "prompt":
        lq, pre = lengths(case), prefixes(case)
        lk = [a + b for a, b in zip(lq, pre)]
        tq, tk, heads, kv = sum(lq), sum(lk), case["heads"], case["kv"]
        if case["fused"] and not case["prefix"]:  # the rows of one QKV product, used in place
            rows = _normal((tq, heads + 2 * kv, hd), gen, case["type"])
            rows[:, heads:heads + kv] = _key_rows((tq, kv, hd), gen, case["type"])
            s["q"], s["k"], s["v"] = rows[:, :heads], rows[:, heads:heads + kv], rows[:, heads + kv:]
        else:
            s["q"] = _normal((tq, heads, hd), gen, case["type"])
            s["k"] = _key_rows((tk, kv, hd), gen, case["type"])
            s["v"] = _normal((tk, kv, hd), gen, case["type"])
        s["q_starts"] = _ints(_starts(lq))
        s["k_starts"] = _ints(_starts(lk)) if case["prefix"] else None
        s["longest_k"] = max(lk)
        s["out"] = torch.empty(tq, heads, hd, dtype=TYPES[case["type"]], device=DEV)
        s["scale"] = 1.0 / math.sqrt(hd)
        return s
    if op == "append":
        new = lengths(case)
        lens = [n + case["held"] for n in new]
        s["table"], pages = _table(lens, case["page"], seed)
        s["pool"] = torch.zeros(pages, case["kv"], case["page"], 5 * hd // 4, dtype=torch.uint8, device=DEV)
        s["lens"], s["starts"], rows = _ints(lens), _ints(_starts(new)), sum(new)
        s["k"], s["v"] = _key_rows((rows, case["kv"], hd), gen, case["type"]), _normal((rows, case["kv"], hd), gen, case["type"], 0.5)
        s["k_out"] = torch.empty(rows, case["kv"], hd, device=DEV)
        s["v_out"] = torch.empty_like(s["k_out"])
        return s
    if op == "decode":
        lens = lengths(case)
        s["table"], pages = _table(lens, case["page"], seed)
        s["pool"], s["lens"] = _filled_pool(pages, case["kv"], case["page"], hd, gen, "fp32"), _ints(lens)
        s["q"] = _normal((case["seqs"], case["heads"], hd), gen, case["type"])
        s["out"] = torch.empty_like(s["q"])
        s["scale"] = 1.0 / math.sqrt(hd)
        return s
    # page operations: one int32 buffer [counts | lengths | tables | status] that the cache's owner keeps
    order, ended = _layout(case)
    seqs = case["parents"] + case["children"]
    width = -(-case["longest"] // case["page"])
    lens = lengths(case, case["parents"]) + [0] * case["children"]
    counts = [0] * case["pages"]
    for p in (p for o in order for p in o):
        counts[p] = 1
    table = [o + [-1] * (width - len(o)) for o in order] + [[-1] * width] * case["children"]
    s["meta"] = _ints(counts + lens + [p for r in table for p in r] + [0])
    s["at"] = (case["pages"], case["pages"] + seqs, case["pages"] + seqs + seqs * width)
    s["width"] = width
    s["pool"] = torch.randint(0, 256, (case["layers"], case["pages"], case["kv"], case["page"], 5 * hd // 4), generator=gen,
                              dtype=torch.uint8, device=DEV)
    s["ended"], s["from"] = _ints(ended), _ints(_parents(case))
    s["to"] = _ints(list(range(case["parents"], seqs)))
    return s


# ----------------------------------------------------------------- one pass

def run(state):
    return {"prompt": _prompt, "append": _append, "decode": _decode, "fork": _fork, "compact": _compact}[state["op"]](state)


def _prompt(s):
    if own:
        from freeml_b200 import matrix_ops
        matrix_ops.attention_packed(s["out"], s["q"], s["k"], s["v"], s["q_starts"], s["scale"], k_starts=s["k_starts"])
        return s["out"]
    heads, group, most_q, most_k = s["heads"], s["heads"] // s["kv"], s["longest"], s["longest_k"]
    qs = s["q_starts"].long()
    ks = qs if s["k_starts"] is None else s["k_starts"].long()
    lq, lk = (qs[1:] - qs[:-1])[:, None], (ks[1:] - ks[:-1])[:, None]
    i, j = torch.arange(most_q, device=DEV)[None], torch.arange(most_k, device=DEV)[None]
    take_q = torch.where(i < lq, qs[:-1, None] + i, 0)
    take_k = torch.where(j < lk, ks[:-1, None] + j, 0)
    q = s["q"][take_q].float().permute(0, 2, 1, 3).unflatten(1, (s["kv"], group)).flatten(2, 3)  # [B, kv, group * rows, hd]
    k, v = s["k"][take_k].float().permute(0, 2, 1, 3), s["v"][take_k].float().permute(0, 2, 1, 3)
    seen = (j[:, None] <= i[:, :, None] + (lk - lq)[:, :, None]) & (j < lk)[:, None]  # [B, rows, keys]
    x = torch.matmul(q, k.transpose(2, 3)).unflatten(2, (group, most_q)).mul_(s["scale"])
    x.masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.flatten(2, 3), v).unflatten(2, (group, most_q)) / torch.where(total == 0, 1.0, total)
    o = o.flatten(1, 2).permute(0, 2, 1, 3)  # [B, rows, heads, hd]
    s["out"][take_q[i < lq]] = o[i.expand(len(lq), -1) < lq].to(s["out"].dtype)
    return s["out"]


def _places(s, rows):
    """The page and the row within it of every new row."""
    starts, lens, page = s["starts"].long(), s["lens"].long(), s["page"]
    r = torch.arange(rows, device=DEV)
    b = torch.searchsorted(starts, r, right=True) - 1
    at = lens[b] - starts[b + 1] + r
    return s["table"][b, at // page].long(), at % page


def _store(x, codes, pairs, page, slot, unit, out):
    codes[page, :, slot], pairs[page, :, slot] = _quantise(x, unit)
    out.copy_(_values(codes[page, :, slot], pairs[page, :, slot], x.shape[-1], unit))


def _append(s):
    if own:
        from freeml_b200 import kv4
        kv4.append(s["pool"], s["table"], s["lens"], s["k"], s["v"], s["starts"])
        kv4.read(s["k_out"], s["v_out"], s["pool"], s["table"], s["lens"], s["starts"])
        return s["k_out"], s["v_out"]
    hd, (page, slot) = s["hd"], _places(s, len(s["k"]))
    kc, km, vc, vm = _views(s["pool"], hd)
    _store(s["k"], kc, km, page, slot, 8, s["k_out"])
    _store(s["v"], vc, vm, page, slot, 4, s["v_out"])
    return s["k_out"], s["v_out"]


def _decode(s):
    if own:
        from freeml_b200 import kv4
        kv4.attention(s["out"], s["q"], s["pool"], s["table"], s["lens"], s["scale"])
        return s["out"]
    hd, kv, group, pages = s["hd"], s["kv"], s["heads"] // s["kv"], s["table"].clamp(min=0).long()
    kc, km, vc, vm = _views(s["pool"], hd)
    keys = torch.arange(pages.shape[1] * s["page"], device=DEV)
    gone = keys[None, None, None] >= s["lens"][:, None, None, None]
    q = s["q"].float().unflatten(1, (kv, group))
    k = _values(kc[pages], km[pages], hd, 8).transpose(1, 2).flatten(2, 3)  # [B, kv, keys, hd]
    x = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).masked_fill_(gone, float("-inf"))
    del k
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    v = _values(vc[pages], vm[pages], hd, 4).transpose(1, 2).flatten(2, 3)
    o = torch.matmul(x, v) / torch.where(total == 0, 1.0, total)
    s["out"].copy_(o.flatten(1, 2))
    return s["out"]


def _parts(s, meta):
    a, b, c = s["at"]
    return meta[:a], meta[a:b], meta[b:c].view(b - a, s["width"]), meta[c:]


def _fork(s):
    meta, pool, page = s["meta"].clone(), s["pool"], s["page"]
    counts, lens, table, status = _parts(s, meta)
    if own:
        from freeml_b200 import kv4
        kv4.fork(pool, counts, table, lens, s["from"], s["to"], status)
        return meta, pool
    parent, child = s["from"].long(), s["to"].long()
    n, rows = lens[parent], table[parent]
    full, some = n // page, (n % page) != 0
    col = torch.arange(s["width"], device=DEV)[None]
    shared = col < full[:, None]
    counts.index_add_(0, torch.where(shared, rows, 0).flatten().long(), shared.flatten().int())
    fresh = torch.nonzero(counts == 0).flatten()[:int(some.sum())]
    last = full[some].long()
    pool[:, fresh] = pool[:, rows[some].gather(1, last[:, None]).flatten().long()]
    counts[fresh] = 1
    rows = torch.where(shared, rows, -1)
    rows[some.nonzero().flatten(), last] = fresh.int()
    table[child], lens[child] = rows, n
    return meta, pool


def _compact(s):
    meta, pool = s["meta"].clone(), s["pool"]
    counts, lens, table, status = _parts(s, meta)
    if own:
        from freeml_b200 import kv4
        kv4.free(counts, table, lens, s["ended"], status)
        kv4.compact(pool, counts, table)
        return meta, pool
    ended = s["ended"].long()
    rows = table[ended]
    counts.index_add_(0, rows.clamp(min=0).flatten().long(), -(rows >= 0).flatten().int())
    table[ended], lens[ended] = -1, 0
    live = counts > 0
    total, number = live.sum(), torch.arange(len(counts), device=DEV)
    holes, movers = torch.nonzero(~live & (number < total)).flatten(), torch.nonzero(live & (number >= total)).flatten()
    pool[:, holes] = pool[:, movers]
    counts[holes] = counts[movers]
    counts[movers] = 0
    number[movers] = holes
    table.copy_(torch.where(table >= 0, number[table.clamp(min=0).long()].int(), table))
    return meta, pool


# ---------------------------------------------- the definition, in 64 bits

def _attend64(q, k, v, scale, seen=None):
    """q [rows, hd], k / v [keys, hd]: softmax(scale q k^T) v over the keys that `seen` [rows, keys] leaves."""
    x = (q @ k.T) * scale
    if seen is not None:
        x = x.masked_fill(~seen, -math.inf)
    return torch.softmax(x, -1) @ v


def _group64(x):
    """Rows [..., hd] as the values their 4-bit groups stand for; only the stored pairs are rounded."""
    hd = x.shape[-1]
    g = x.double().clamp(-65504, 65504).reshape(*x.shape[:-1], hd // 32, 32)
    low = g.min(-1, keepdim=True).values.half().double()
    scale = ((g.max(-1, keepdim=True).values - low) / 15).half().double()
    code = torch.where(scale > 0, (g - low) / torch.where(scale > 0, scale, 1.0), 0.0).round().clamp(0, 15)
    return (low + code * scale).reshape(x.shape)


def _columns64(blocks, page, hd, values):
    """The bytes of one head's blocks, page after page, as [keys, hd] numbers: each column from the layout's words."""
    raw, groups = blocks.reshape(len(blocks), -1), hd // 32
    half = page * hd // 2 + page * hd // 8
    raw = raw[:, half:] if values else raw[:, :half]
    codes = raw[:, :page * hd // 2].reshape(-1, hd // 2)
    pairs = raw[:, page * hd // 2:].contiguous().view(torch.float16).reshape(-1, groups, 2).double()
    d = torch.arange(hd, device=raw.device)
    unit = 4 if values else 8
    g, u, i = d // 32, d % 32 // unit, d % unit
    nibble = (u * groups + g) * unit + i
    code = (codes[:, nibble // 2].int() >> (4 * (nibble % 2)).int()) & 15
    return pairs[:, g, 1] + code.double() * pairs[:, g, 0]


def exact(case, seed):
    op, hd = case["op"], case["hd"]
    if op in ("fork", "compact"):
        return None
    s = prepare(case, seed)
    if op == "append":
        return _group64(s["k"]), _group64(s["v"])
    group, out = case["heads"] // case["kv"], torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    if op == "prompt":
        lq, pre = lengths(case), prefixes(case)
        qs, ks = _starts(lq), _starts([a + b for a, b in zip(lq, pre)])
        for b in range(case["seqs"]):
            i = torch.arange(lq[b], device=DEV)[:, None]
            seen = torch.arange(lq[b] + pre[b], device=DEV)[None] <= i + pre[b]
            for h in range(case["heads"]):
                k, v = (s[n][ks[b]:ks[b + 1], h // group].double() for n in "kv")
                out[qs[b]:qs[b + 1], h] = _attend64(s["q"][qs[b]:qs[b + 1], h].double(), k, v, s["scale"], seen)
        return out
    for b, n in enumerate(lengths(case)):
        used = s["table"][b][:-(-n // case["page"])].long()
        for h in range(case["kv"]):
            k, v = (_columns64(s["pool"][used, h], case["page"], hd, w)[:n] for w in (False, True))
            out[b, h * group:(h + 1) * group] = _attend64(s["q"][b, h * group:(h + 1) * group].double(), k, v, s["scale"])
    return out
