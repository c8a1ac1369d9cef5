"""A cache of 8-bit pages and batches that share a prefix, as cases that can be timed and checked.

The heads are those of the 27B model whose geometry the loader checks (gguf_pq2.py), 24 query and 4
key/value heads of 256 with 64 rotated elements; some cases take heads of 128, drawn ones shards of
them and heads of 64 too.  A row (one key or value of one head) of an 8-bit page is whole numbers
-127 .. 127 and one fp32 scale, a page the rows of all its heads and behind them their scales.
Kinds of case:

* append: head norms, position rotation and the append of keys and values to 8-bit pages, and the
  rows that were written read back in 16 bits;
* read: rows of a cache read back by their slots;
* attn: attention of every sequence's new tokens over its 8-bit pages;
* shared: attention of a batch whose sequences, group by group, begin with the same keys.

Lengths of ragged batches come from the case alone (its "mix" number), values from the seed.
"""
import math
import os
import random
import sys

import torch

own = False

EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "q8": torch.int8}


def listed():
    return [
        # one token of a decode loop, handed on to a second cache: latency is all there is
        {"name": "append 1 token", "kind": "append", "n_tok": 1, "heads": 24, "kv_heads": 4, "dim": 256, "rot": 64,
         "page": 16, "q_type": "f32", "rows": "bf16", "columns": False, "far": 4096},
        # a prompt chunk as the prompt product leaves it, one row per feature, far into a long context
        {"name": "append 2048 tokens", "kind": "append", "n_tok": 2048, "heads": 24, "kv_heads": 4, "dim": 256,
         "rot": 64, "page": 64, "q_type": "bf16", "rows": "f16", "columns": True, "far": 200000},
        # one request's context taken out of the cache
        {"name": "read 1000 rows", "kind": "read", "n_tok": 1000, "kv_heads": 4, "dim": 256, "page": 16, "type": "q8",
         "rows": "bf16", "spare": 3},
        # a long document handed to a program that works in fp32
        {"name": "read 50001 rows", "kind": "read", "n_tok": 50001, "kv_heads": 4, "dim": 256, "page": 64, "type": "q8",
         "rows": "f32", "spare": 5},
        # a single user's decode step, in the activations' own type
        {"name": "attn decode 1x4000", "kind": "attn", "n_seq": 1, "new": 1, "ctx": 4000, "heads": 24, "kv_heads": 4,
         "dim": 256, "page": 16, "io": "f32", "mix": 0},
        # a serving batch of ragged contexts
        {"name": "attn decode 32x12000", "kind": "attn", "n_seq": 32, "new": 1, "ctx": 12000, "heads": 24,
         "kv_heads": 4, "dim": 256, "page": 16, "io": "bf16", "mix": 11},
        # a chunk of no round length after a long context
        {"name": "attn chunk 777 of 16000", "kind": "attn", "n_seq": 1, "new": 777, "ctx": 16000, "heads": 24,
         "kv_heads": 4, "dim": 256, "page": 16, "io": "f16", "mix": 0},
        # prompts and continuations of several users in one call, heads of 128
        {"name": "attn mixed 9 sequences", "kind": "attn", "n_seq": 9, "new": 300, "ctx": 5000, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 32, "io": "bf16", "mix": 5},
        # a few samples drawn for one prompt
        {"name": "shared 4x(1000+20)", "kind": "shared", "n_seq": 4, "groups": 1, "prefix": 1000, "own": 20, "new": 1,
         "heads": 24, "kv_heads": 4, "dim": 256, "page": 16, "type": "f16", "io": "f32", "mix": 0},
        # a serving batch behind one long system prompt
        {"name": "shared 64x(16000+500)", "kind": "shared", "n_seq": 64, "groups": 1, "prefix": 16000, "own": 500,
         "new": 1, "heads": 24, "kv_heads": 4, "dim": 256, "page": 64, "type": "bf16", "io": "bf16", "mix": 7},
        # the same from 8-bit pages, the prefix longer
        {"name": "shared 32x(40000+1500) 8 bits", "kind": "shared", "n_seq": 32, "groups": 1, "prefix": 40000,
         "own": 1500, "new": 1, "heads": 24, "kv_heads": 4, "dim": 256, "page": 16, "type": "q8", "io": "bf16",
         "mix": 9},
        # several documents with questions to each, a few new tokens a sequence
        {"name": "shared 5 groups of 40x(6007+300)", "kind": "shared", "n_seq": 40, "groups": 5, "prefix": 6007,
         "own": 300, "new": 12, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "type": "f16", "io": "f16",
         "mix": 3},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "read", "attn", "attn", "shared", "shared"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "append":
        heads, kv_heads, dim, rot = rng.choice([(24, 4, 256, 64), (18, 3, 256, 64), (32, 8, 128, 128), (10, 5, 64, 32)])
        return {"kind": kind, "n_tok": _log_int(rng, 1, 2048), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rot": rot, "page": page, "q_type": rng.choice(["f32", "f16", "bf16"]),
                "rows": rng.choice(["f16", "bf16"]), "columns": rng.random() < 0.5, "far": _log_int(rng, 4096, 1000000)}
    if kind == "read":
        kv_heads, dim = rng.choice([(4, 256), (1, 256), (8, 128), (2, 64)])
        return {"kind": kind, "n_tok": _log_int(rng, 1, 50000), "kv_heads": kv_heads, "dim": dim, "page": page,
                "type": rng.choice(["q8", "q8", "f16", "bf16"]), "rows": rng.choice(["f32", "f16", "bf16"]),
                "spare": rng.randint(0, 40)}
    heads, kv_heads, dim = rng.choice([(24, 4, 256), (24, 4, 256), (6, 1, 256), (32, 8, 128), (14, 2, 64)])
    if kind == "attn":
        n_seq = _log_int(rng, 1, 32)
        new = 1 if rng.random() < 0.5 else _log_int(rng, 2, 1024 // n_seq if n_seq < 4 else 128)
        ctx = max(new, _log_int(rng, 64, (40000 if n_seq < 4 else 8000) if new == 1 else 8000 if n_seq < 4 else 3000))
        return {"kind": kind, "n_seq": n_seq, "new": new, "ctx": ctx, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "page": page, "io": rng.choice(["f32", "f16", "bf16"]), "mix": rng.randint(1, 1000)}
    n_seq = _log_int(rng, 2, 64)
    t = rng.choice(["q8", "f16", "bf16"])
    new = 1 if rng.random() < 0.7 else rng.randint(2, 8)
    return {"kind": kind, "n_seq": n_seq, "groups": min(n_seq, rng.choice([1, 1, 2, 4])), "new": new,
            "prefix": _log_int(rng, 100, 16000), "own": new + _log_int(rng, 1, 500), "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "type": t,
            "io": rng.choice(["f32", "f16", "bf16"] if t == "q8" else ["f32", t]), "mix": rng.randint(1, 1000)}


# ------------------------------------------------------------------ inputs
def _spread(rng, most, least, count, ragged):
    """`count` lengths, the first of them `most`, the others below it where they are ragged."""
    return [most if i == 0 or not ragged else max(least, int(most * rng.uniform(0.05, 1))) for i in range(count)]


def _lengths(case):
    """New tokens and context (the new ones included) of every sequence."""
    rng = random.Random(case["mix"])
    new, kv = [], []
    for i in range(case["n_seq"]):
        n = case["new"] if i == 0 or not case["mix"] else max(1, int(case["new"] * rng.uniform(0, 1) ** 2))
        c = case["ctx"] if i == 0 or not case["mix"] else max(n, int(case["ctx"] * rng.uniform(0.05, 1)))
        new.append(n)
        kv.append(c)
    order = list(range(case["n_seq"]))
    rng.shuffle(order)
    return [new[i] for i in order], [kv[i] for i in order]


def _groups(case):
    """Where the groups begin among the sequences, the prefix of each, and new tokens and own keys (the new ones
    included) of every sequence."""
    rng = random.Random(case["mix"])
    cuts = sorted(rng.sample(range(1, case["n_seq"]), case["groups"] - 1))
    prefix = _spread(rng, case["prefix"], 1, case["groups"], case["mix"])
    new = _spread(rng, case["new"], 1, case["n_seq"], case["mix"])
    ends = _spread(rng, case["own"], 1, case["n_seq"], case["mix"])
    order = list(range(case["n_seq"]))
    rng.shuffle(order)
    return [0, *cuts, case["n_seq"]], prefix, [new[i] for i in order], [max(new[i], ends[i]) for i in order]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(lengths):
    c = [0]
    for n in lengths:
        c.append(c[-1] + n)
    return c


def _empty_pages(n, kv, page, d, kind):
    """Pages, and for 8-bit ones the scales that lie behind the rows of each."""
    if kind != "q8":
        return torch.zeros((n, kv, page, d), dtype=TYPES[kind], device="cuda"), None
    rows = kv * page * d
    memory = torch.zeros((n, rows + 4 * kv * page), dtype=torch.int8, device="cuda")
    return memory[:, :rows].unflatten(1, (kv, page, d)), memory[:, rows:].view(torch.float32).unflatten(1, (kv, page))


def _quantised(x):
    """Whole numbers and scales of rows: the largest of a row is 127."""
    scale = x.abs().amax(-1) / 127
    return torch.round(x / torch.where(scale > 0, scale, 1)[..., None]).clamp_(-127, 127), scale


def _filled_pages(g, s, name, n, kv, page, d, kind):
    pages, scales = _empty_pages(n, kv, page, d, kind)
    for i in range(0, n, 4096):                     # some at a time, as the fp32 values of a cache are many
        x = _randn(g, min(4096, n - i), kv, page, d)
        if kind == "q8":
            x *= torch.exp(_randn(g, *x.shape[:3], 1) * 0.3)
            x, scales[i:i + 4096] = _quantised(x)
        pages[i:i + 4096] = x
    s[name + "_pages"], s[name + "_scales"] = pages, scales


def _append_inputs(case, g):
    n, heads, kv, d = case["n_tok"], case["heads"], case["kv_heads"], case["dim"]
    # the query rows of the projection hold a head's queries and then its gates
    shape = [(heads, 2 * d), (kv, d), (kv, d)]
    x = [_randn(g, n, h, w) * 1.5 for h, w in shape]
    if case["columns"]:
        x = [t.permute(1, 2, 0).contiguous().permute(2, 0, 1) for t in x]
    s = {"q": x[0][:, :, :d], "k": x[1], "v": x[2], "hold": x}
    s["q_norm"], s["k_norm"] = _randn(g, d) * 0.1 + 1, _randn(g, d) * 0.1 + 1
    s["inv_freq"] = 1e7 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
    start = int(torch.randint(0, case["far"], (1,), generator=g, device="cuda"))
    s["pos"] = torch.arange(start, start + n, dtype=torch.int32, device="cuda")
    # pages anywhere in the cache, the first of them partly filled
    page, skip = case["page"], start % case["page"]
    pages = n // page + 3
    at = torch.randperm(pages, generator=g, device="cuda")
    i = torch.arange(n, device="cuda") + skip
    s["slots"] = at[i // page] * page + i % page
    for name in "kv":
        s[name + "_pages"], s[name + "_scales"] = _empty_pages(pages, kv, page, d, "q8")
        s[name + "_rows"] = torch.zeros((n, kv, d), dtype=TYPES[case["rows"]], device="cuda")
    s["q_out"] = torch.zeros((n, heads, d), dtype=TYPES[case["q_type"]], device="cuda")
    return s


def _read_inputs(case, g):
    n, kv, d, page = case["n_tok"], case["kv_heads"], case["dim"], case["page"]
    pages = -(-n // page) + case["spare"]
    s = {}
    for name in "kv":
        _filled_pages(g, s, name, pages, kv, page, d, case["type"])
        s[name + "_rows"] = torch.zeros((n, kv, d), dtype=TYPES[case["rows"]], device="cuda")
    at = torch.randperm(pages, generator=g, device="cuda")
    i = torch.arange(n, device="cuda")
    s["slots"] = at[i // page] * page + i % page
    return s


def _attn_inputs(case, g):
    new, kv = _lengths(case)
    heads, kvh, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    io, n = TYPES[case["io"]], sum(new)
    pages = [-(-c // page) for c in kv]
    total = sum(pages)
    s = {"q": (_randn(g, n, heads, d) * 1.2).to(io)}
    for name in "kv":
        _filled_pages(g, s, name, total + 1, kvh, page, d, "q8")
    perm = torch.randperm(total + 1, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((case["n_seq"], max(pages)), dtype=torch.int32, device="cuda")
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = perm[at:at + p]
        at += p
    s["table"], s["starts"], s["kv_len"] = table, _ints(_starts(new)), _ints(kv)
    s["max_kv"], s["max_new"] = max(kv), max(new)
    s["out"] = torch.zeros((n, heads, d), dtype=io, device="cuda")
    # memory that the program keeps for its calls
    s["work"] = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    return s


def _shared_inputs(case, g):
    first, prefix, new, tail = _groups(case)
    heads, kvh, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    io, n = TYPES[case["io"]], sum(new)
    lead = [p for i, p in enumerate(prefix) for _ in range(first[i], first[i + 1])]
    kv = [p + t for p, t in zip(lead, tail)]
    rows, total = [], 0
    for i, p in enumerate(prefix):
        whole = p // page                           # a page that holds the prefix's last keys and others is each one's own,
        front = list(range(total, total + -(-p // page)))     # but for the one that the prefix is read from
        total += len(front)
        for s in range(first[i], first[i + 1]):
            count = -(-kv[s] // page) - whole
            mine = list(range(total, total + count))
            total += count
            if s == first[i] and len(front) > whole:
                mine[0] = front[whole]
            rows.append(front[:whole] + mine)
    s = {"q": (_randn(g, n, heads, d) * 1.2).to(io)}
    for name in "kv":
        _filled_pages(g, s, name, total, kvh, page, d, case["type"])
    perm = torch.randperm(total, generator=g, device="cuda").cpu().tolist()
    longest = max(len(r) for r in rows)
    s["table"] = _ints([[perm[p] for p in r] + [0] * (longest - len(r)) for r in rows])
    s["starts"], s["kv_len"] = _ints(_starts(new)), _ints(kv)
    s["groups"], s["shared"] = _ints(first), _ints(prefix)
    s["max_kv"], s["max_new"], s["max_shared"], s["max_own"] = max(kv), max(new), max(prefix), max(tail)
    s["max_rows"] = max(sum(new[a:b]) for a, b in zip(first, first[1:]))
    s["out"] = torch.zeros((n, heads, d), dtype=io, device="cuda")
    s["work"] = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    return s


_INPUTS = {"append": _append_inputs, "read": _read_inputs, "attn": _attn_inputs, "shared": _shared_inputs}


def prepare(case, seed):
    s = _INPUTS[case["kind"]](case, _generator(seed))
    s["case"] = case
    return s


# ---------------------------------------------------------------- plain forms
def _plain_append(s):
    case = s["case"]
    rot = case["rot"]
    angle = s["pos"].double()[:, None] * s["inv_freq"][None]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, w):
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)

    s["q_out"].copy_(turned(s["q"], s["q_norm"]))
    page, off = s["slots"] // case["page"], s["slots"] % case["page"]
    k, k_scale = _quantised(turned(s["k"], s["k_norm"]))
    v, v_scale = _quantised(s["v"])
    s["k_pages"][page, :, off], s["k_scales"][page, :, off] = k.to(torch.int8), k_scale
    s["v_pages"][page, :, off], s["v_scales"][page, :, off] = v.to(torch.int8), v_scale
    s["k_rows"].copy_(k * k_scale[..., None])
    s["v_rows"].copy_(v * v_scale[..., None])
    return {"q": s["q_out"], "k": s["k_rows"], "v": s["v_rows"]}


def _plain_read(s):
    page, off = s["slots"] // s["case"]["page"], s["slots"] % s["case"]["page"]
    k, v = s["k_pages"][page, :, off].float(), s["v_pages"][page, :, off].float()
    if s["k_scales"] is not None:
        k, v = k * s["k_scales"][page, :, off][..., None], v * s["v_scales"][page, :, off][..., None]
    s["k_rows"].copy_(k)
    s["v_rows"].copy_(v)
    return {"k": s["k_rows"], "v": s["v_rows"]}


def _keys_of(s, name, table, first, count):
    """The rows of `count` keys from `first` (one for each row of the table) on: (rows of the table, kv heads, count,
    dim)."""
    pages, scales, page = s[name + "_pages"], s[name + "_scales"], s["case"]["page"]
    j = first[:, None] + torch.arange(count, device="cuda")
    at = table.long().gather(1, (j // page).clamp(max=table.shape[1] - 1))
    x = pages[at, :, j % page].float()
    if scales is not None:
        x = x * scales[at, :, j % page][..., None]
    return x.transpose(1, 2)


def _parts(q, k, v, seen):
    """Sums of weights, of weighted values, and the largest score of each row of q (batch, kv heads, rows, dim) over
    the keys that it sees (batch, 1 or rows, keys)."""
    score = torch.matmul(q, k.transpose(2, 3)).mul_(q.shape[-1] ** -0.5)
    score.masked_fill_(~seen[:, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(top.clamp(min=-1e30)).exp_()
    return score.sum(-1, keepdim=True), torch.matmul(score, v.masked_fill(~seen.any(1)[:, None, :, None], 0)), top


def _padded_rows(s, first, count, top):
    """Queries of `count` tokens from `first` on, padded to `top`: (batch, kv heads, tokens x heads of a group, dim),
    the tokens' places, and which of them there are."""
    case = s["case"]
    kvh, d = case["kv_heads"], case["dim"]
    t = torch.arange(top, device="cuda")
    rows = (first[:, None] + t).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().view(len(first), top, kvh, case["heads"] // kvh, d)
    return q.permute(0, 2, 1, 3, 4).reshape(len(first), kvh, -1, d), rows, t < count[:, None]


def _by_token(x, top):
    """(batch, kv heads, tokens x heads of a group, n) as (batch, tokens, heads, n)."""
    b, kvh, r, n = x.shape
    return x.view(b, kvh, top, r // top, n).permute(0, 2, 1, 3, 4).reshape(b, top, kvh * (r // top), n)


def _plain_attn(s):
    """All sequences at once, padded to the longest."""
    case, top = s["case"], s["max_new"]
    group = case["heads"] // case["kv_heads"]
    first = s["starts"][:-1].long()
    count = s["starts"][1:].long() - first
    kv_len = s["kv_len"].long()
    q, rows, keep = _padded_rows(s, first, count, top)
    zero = torch.zeros_like(kv_len)
    k, v = (_keys_of(s, name, s["table"], zero, s["max_kv"]) for name in "kv")
    t, j = torch.arange(top, device="cuda"), torch.arange(s["max_kv"], device="cuda")
    seen = j <= (kv_len - count)[:, None, None] + t[:, None]
    total, out, _ = _parts(q, k, v, (seen & (j < kv_len[:, None, None])).repeat_interleave(group, 1))
    s["out"][rows[keep]] = _by_token(out / total, top)[keep].to(s["out"].dtype)
    return s["out"]


def _plain_shared(s):
    """The prefixes with all rows of their groups, then every sequence's own keys, and the two joined."""
    case, top = s["case"], s["max_new"]
    heads, d = case["heads"], case["dim"]
    group = heads // case["kv_heads"]
    starts, lead, shared = s["starts"].long(), s["groups"][:-1].long(), s["shared"].long()
    n = s["q"].shape[0]
    weight, value, high = (torch.empty((2, n, heads, w), device="cuda") for w in (1, d, 1))

    first = starts[lead]
    q, rows, keep = _padded_rows(s, first, starts[s["groups"][1:].long()] - first, s["max_rows"])
    k, v = (_keys_of(s, name, s["table"][lead], torch.zeros_like(lead), s["max_shared"]) for name in "kv")
    seen = (torch.arange(s["max_shared"], device="cuda") < shared[:, None])[:, None]
    for to, x in zip((weight, value, high), _parts(q, k, v, seen)):
        to[0, rows[keep]] = _by_token(x, s["max_rows"])[keep]

    first = starts[:-1]
    count = starts[1:] - first
    size = s["groups"][1:].long() - lead
    behind = shared.repeat_interleave(size, output_size=case["n_seq"])
    q, rows, keep = _padded_rows(s, first, count, top)
    k, v = (_keys_of(s, name, s["table"], behind, s["max_own"]) for name in "kv")
    t, j = torch.arange(top, device="cuda"), torch.arange(s["max_own"], device="cuda")
    mine = s["kv_len"].long() - behind
    seen = (j <= (mine - count)[:, None, None] + t[:, None]) & (j < mine[:, None, None])
    for to, x in zip((weight, value, high), _parts(q, k, v, seen.repeat_interleave(group, 1))):
        to[1, rows[keep]] = _by_token(x, top)[keep]

    high = (high - high.amax(0)).exp()
    s["out"].copy_((value * high).sum(0) / (weight * high).sum(0))
    return s["out"]


_PLAIN = {"append": _plain_append, "read": _plain_read, "attn": _plain_attn, "shared": _plain_shared}


def _library():
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), os.pardir, "p40-kernel_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import bonsai_p40
    return bonsai_p40


def run(state):
    s = state
    kind = s["case"]["kind"]
    if not own:
        return _PLAIN[kind](s)
    B = _library()
    if kind == "append":
        B.qk_norm_rope(s["q"], s["k"], s["v"], s["q_norm"], s["k_norm"], EPS, s["pos"], s["inv_freq"], s["slots"],
                       s["k_pages"], s["v_pages"], s["q_out"])
        B.kv_read(s["k_pages"], s["v_pages"], s["slots"], s["k_rows"], s["v_rows"])
        return {"q": s["q_out"], "k": s["k_rows"], "v": s["v_rows"]}
    if kind == "read":
        B.kv_read(s["k_pages"], s["v_pages"], s["slots"], s["k_rows"], s["v_rows"])
        return {"k": s["k_rows"], "v": s["v_rows"]}
    if kind == "attn":
        B.attn_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["starts"], s["kv_len"], s["out"], s["work"],
                     max_kv=s["max_kv"])
    else:
        B.attn_shared(s["q"], s["k_pages"], s["v_pages"], s["table"], s["starts"], s["kv_len"], s["groups"],
                      s["shared"], s["out"], s["work"], max_kv=s["max_kv"], max_shared=s["max_shared"])
    return s["out"]


# ---------------------------------------------------------- work, exactness
def _size(name):
    return {"f32": 4, "q8": 1}.get(name, 2)


def _row_bytes(case, kind):
    """A key and a value of all heads."""
    return 2 * case["kv_heads"] * (case["dim"] * _size(kind) + (4 if kind == "q8" else 0))


def work(case):
    d = case["dim"]
    if case["kind"] in ("append", "read"):
        n, kv = case["n_tok"], 2 * case["kv_heads"] * d
        back = n * (_row_bytes(case, case.get("type", "q8")) + kv * _size(case["rows"]))
        if case["kind"] == "read":
            return {"bytes": back, "flops": n * kv}
        q = case["heads"] * d
        return {"bytes": n * (q * (4 + _size(case["q_type"])) + 4 * kv + _row_bytes(case, "q8")) + back,
                "flops": n * (q + 2 * kv) * 6}
    if case["kind"] == "attn":
        new, kv = _lengths(case)
        keys, kind = sum(kv), "q8"
    else:
        first, prefix, new, tail = _groups(case)
        lead = [p for i, p in enumerate(prefix) for _ in range(first[i], first[i + 1])]
        kv = [p + t for p, t in zip(lead, tail)]
        keys, kind = sum(prefix) + sum(tail), case["type"]
    pairs = sum(n * c - n * (n - 1) // 2 for n, c in zip(new, kv))
    q = sum(new) * case["heads"] * d
    return {"bytes": 2 * _size(case["io"]) * q + keys * _row_bytes(case, kind), "flops": 4 * d * case["heads"] * pairs}


def _exact_row(case, s, x, w):
    x = x.double()
    x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
    half = case["rot"] // 2
    y = x.clone()
    turn = torch.polar(torch.ones_like(s["inv_freq"]).expand(x.shape[0], half),
                       s["pos"].double()[:, None] * s["inv_freq"])[:, None]
    z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
    y[..., :half], y[..., half:2 * half] = z.real, z.imag
    return y


def _exact_append(case, s):
    def kept(x):
        step = x.abs().max(-1, keepdim=True).values / 127
        return (x / step).round() * step

    return {"q": _exact_row(case, s, s["q"], s["q_norm"]), "k": kept(_exact_row(case, s, s["k"], s["k_norm"])),
            "v": kept(s["v"].double())}


def _values(s, name):
    """Every slot's row in 64 bits."""
    x = s[name + "_pages"].double()
    if s[name + "_scales"] is not None:
        x = x * s[name + "_scales"].double().unsqueeze(-1)
    return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])


def _exact_read(case, s):
    return {name: _values(s, name)[s["slots"]] for name in "kv"}


def _exact_over(case, s, new, kv, slots_of):
    """Token rows of 64 bits; slots_of(sequence): the slots of its keys."""
    d, group = case["dim"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, c) in enumerate(zip(new, kv)):
        slots = slots_of(i)
        page, off = slots // case["page"], slots % case["page"]
        for h in range(case["kv_heads"]):
            k, v = (s[name + "_pages"][page, h, off].double() for name in "kv")
            if s["k_scales"] is not None:
                k, v = k * s["k_scales"][page, h, off].double()[:, None], v * s["v_scales"][page, h, off].double()[:, None]
            for r in range(0, n, 512):
                m = min(512, n - r)
                late = torch.arange(c, device="cuda")[None] > (c - n + r + torch.arange(m, device="cuda"))[:, None]
                for x in range(h * group, (h + 1) * group):
                    p = s["q"][at + r:at + r + m, x].double() @ k.t() / math.sqrt(d)
                    out[at + r:at + r + m, x] = torch.softmax(p.masked_fill(late, -math.inf), -1) @ v
        at += n
    return out


def _exact_attn(case, s):
    new, kv = _lengths(case)

    def slots_of(i):
        j = torch.arange(kv[i], device="cuda")
        return s["table"][i].long()[j // case["page"]] * case["page"] + j % case["page"]

    return _exact_over(case, s, new, kv, slots_of)


def _exact_shared(case, s):
    first, prefix, new, tail = _groups(case)
    of = [i for i in range(len(prefix)) for _ in range(first[i], first[i + 1])]
    kv = [prefix[of[i]] + t for i, t in enumerate(tail)]

    def slots_of(i):
        j = torch.arange(kv[i], device="cuda")
        row = torch.where(j < prefix[of[i]], first[of[i]], i)
        return s["table"].long()[row, j // case["page"]] * case["page"] + j % case["page"]

    return _exact_over(case, s, new, kv, slots_of)


def exact(case, seed):
    made = {"append": _exact_append, "read": _exact_read, "attn": _exact_attn, "shared": _exact_shared}
    return made[case["kind"]](case, prepare(case, seed))
