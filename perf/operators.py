"""The token mixers between a decoder layer's projections, as cases that can be timed and checked.

The heads are those of the 27B model whose geometry the loader checks (gguf_pq2.py): 24 query and 4
key/value heads of 256 with 64 rotated elements in the full-attention layers, 16 key and 48 value heads
of 128 in the linear-attention layers; drawn cases take shards of them and heads of 64 and 128 too.
Kinds of case:

* rope: RMSNorm of every query and key head, position rotation, and the append of keys and values to
  the pages of the cache, from the fp32 rows of the projections (one row per token, or one per
  feature as the prompt product writes them);
* attn: attention of every sequence's new tokens over its pages;
* gdn: the gated delta rule over every sequence's new tokens, with the state that it leaves.

Lengths of ragged batches come from the case alone (its "mix" number), values from the seed.
"""
import math
import os
import random
import sys

import torch

own = False

EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token of a decode loop: latency is all there is
        {"name": "rope 1 token", "kind": "rope", "n_tok": 1, "heads": 24, "kv_heads": 4, "dim": 256, "rot": 64,
         "page": 16, "type": "bf16", "q_type": "bf16", "columns": False, "far": 4096},
        # a prompt chunk as the prompt product leaves it, one row per feature, far into a long context
        {"name": "rope 2048 tokens", "kind": "rope", "n_tok": 2048, "heads": 24, "kv_heads": 4, "dim": 256,
         "rot": 64, "page": 64, "type": "f16", "q_type": "f16", "columns": True, "far": 200000},
        # a single user's decode step, in the activations' own type
        {"name": "attn decode 1x4000", "kind": "attn", "n_seq": 1, "new": 1, "ctx": 4000, "heads": 24, "kv_heads": 4,
         "dim": 256, "page": 16, "type": "f16", "io": "f32", "mix": 0},
        # a serving batch of ragged contexts
        {"name": "attn decode 32x12000", "kind": "attn", "n_seq": 32, "new": 1, "ctx": 12000, "heads": 24,
         "kv_heads": 4, "dim": 256, "page": 16, "type": "bf16", "io": "bf16", "mix": 11},
        # one long document
        {"name": "attn decode 1x131071", "kind": "attn", "n_seq": 1, "new": 1, "ctx": 131071, "heads": 24,
         "kv_heads": 4, "dim": 256, "page": 64, "type": "bf16", "io": "f32", "mix": 0},
        # a first prompt chunk
        {"name": "attn chunk 2048", "kind": "attn", "n_seq": 1, "new": 2048, "ctx": 2048, "heads": 24, "kv_heads": 4,
         "dim": 256, "page": 64, "type": "bf16", "io": "bf16", "mix": 0},
        # a chunk of no round length after a long context
        {"name": "attn chunk 777 of 16000", "kind": "attn", "n_seq": 1, "new": 777, "ctx": 16000, "heads": 24,
         "kv_heads": 4, "dim": 256, "page": 16, "type": "f16", "io": "f16", "mix": 0},
        # prompts and continuations of several users in one call, heads of 128
        {"name": "attn mixed 9 sequences", "kind": "attn", "n_seq": 9, "new": 300, "ctx": 5000, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 32, "type": "bf16", "io": "bf16", "mix": 5},
        # one token of a decode loop
        {"name": "gdn step 1", "kind": "gdn", "n_seq": 1, "new": 1, "k_heads": 16, "v_heads": 48, "dim": 128,
         "type": "f32", "mix": 0},
        # a serving batch, two tokens each (one of them a draft)
        {"name": "gdn step 48x2", "kind": "gdn", "n_seq": 48, "new": 2, "k_heads": 16, "v_heads": 48, "dim": 128,
         "type": "bf16", "mix": 0},
        # a prompt chunk
        {"name": "gdn chunk 2048", "kind": "gdn", "n_seq": 1, "new": 2048, "k_heads": 16, "v_heads": 48, "dim": 128,
         "type": "f32", "mix": 0},
        # prompts of several users, ragged
        {"name": "gdn chunk 6 sequences", "kind": "gdn", "n_seq": 6, "new": 1500, "k_heads": 16, "v_heads": 48,
         "dim": 128, "type": "bf16", "mix": 3},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "attn", "attn", "gdn"])
    if kind == "rope":
        heads, kv_heads, dim, rot = rng.choice([(24, 4, 256, 64), (12, 2, 256, 64), (32, 8, 128, 128), (10, 5, 64, 32)])
        return {"kind": kind, "n_tok": _log_int(rng, 1, 2048), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rot": rot, "page": rng.choice([16, 32, 64, 128]), "type": rng.choice(["f16", "bf16"]),
                "q_type": rng.choice(["f32", "f16", "bf16"]), "columns": rng.random() < 0.5,
                "far": _log_int(rng, 4096, 1000000)}
    if kind == "attn":
        heads, kv_heads, dim = rng.choice([(24, 4, 256), (24, 4, 256), (6, 1, 256), (32, 8, 128), (14, 2, 64)])
        n_seq = _log_int(rng, 1, 32)
        new = 1 if rng.random() < 0.5 else _log_int(rng, 2, 1024 // n_seq if n_seq < 4 else 128)
        ctx = max(new, _log_int(rng, 64, (40000 if n_seq < 4 else 8000) if new == 1 else 8000 if n_seq < 4 else 3000))
        t = rng.choice(["f16", "bf16"])
        return {"kind": kind, "n_seq": n_seq, "new": new, "ctx": ctx, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "page": rng.choice([16, 32, 64, 128]), "type": t, "io": rng.choice([t, "f32"]),
                "mix": rng.randint(1, 1000)}
    n_seq = _log_int(rng, 1, 24)
    k_heads, per = rng.choice([(16, 3), (8, 3), (4, 2), (5, 1)])
    return {"kind": kind, "n_seq": n_seq, "new": 1 if rng.random() < 0.3 else _log_int(rng, 2, 2048 // n_seq + 2),
            "k_heads": k_heads, "v_heads": k_heads * per, "dim": rng.choice([128, 128, 64]),
            "type": rng.choice(["f32", "f16", "bf16"]), "mix": rng.randint(1, 1000)}


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """New tokens and context (the new ones included) of every sequence: the largest first where "mix" is 0,
    else spread below it, one at least."""
    rng = random.Random(case["mix"])
    ctx = case.get("ctx", case["new"])
    new, kv = [], []
    for i in range(case["n_seq"]):
        n = case["new"] if i == 0 or not case["mix"] else max(1, int(case["new"] * rng.uniform(0, 1) ** 2))
        c = ctx if i == 0 or not case["mix"] else max(n, int(ctx * rng.uniform(0.05, 1)))
        new.append(n)
        kv.append(c)
    order = list(range(case["n_seq"]))
    rng.shuffle(order)
    return [new[i] for i in order], [kv[i] for i in order]


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


def _rope_inputs(case, g):
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
    t = TYPES[case["type"]]
    s["k_pages"], s["v_pages"] = (torch.zeros((pages, kv, page, d), dtype=t, device="cuda") for _ in range(2))
    s["q_out"] = torch.zeros((n, heads, d), dtype=TYPES[case["q_type"]], device="cuda")
    return s


def _attn_inputs(case, g):
    new, kv = _lengths(case)
    heads, kvh, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    t, io = TYPES[case["type"]], TYPES[case["io"]]
    n = sum(new)
    pages = [-(-c // page) for c in kv]
    total = sum(pages)
    s = {"q": (_randn(g, n, heads, d) * 1.2).to(io)}
    s["k_pages"] = torch.empty((total + 1, kvh, page, d), dtype=t, device="cuda")
    s["v_pages"] = torch.empty_like(s["k_pages"])
    s["k_pages"].normal_(generator=g)
    s["v_pages"].normal_(generator=g)
    perm = torch.randperm(total + 1, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((case["n_seq"], max(pages)), dtype=torch.int32, device="cuda")
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = perm[at:at + p]
        at += p
    s["table"], s["starts"], s["kv_len"] = table, _ints(_starts(new)), _ints(kv)
    s["max_kv"] = max(kv)
    s["max_new"] = max(new)
    s["out"] = torch.zeros((n, heads, d), dtype=io, device="cuda")
    # memory that the program keeps for its calls
    s["work"] = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    return s


def _gdn_inputs(case, g):
    new, _ = _lengths(case)
    kh, vh, d = case["k_heads"], case["v_heads"], case["dim"]
    n, t = sum(new), TYPES[case["type"]]
    # one row per token: queries, keys and values as the convolution before them leaves them
    x = _randn(g, n, (2 * kh + vh) * d)
    x = (x * torch.sigmoid(x)).to(t)
    s = {"hold": x, "q": x[:, :kh * d].view(n, kh, d), "k": x[:, kh * d:2 * kh * d].view(n, kh, d),
         "v": x[:, 2 * kh * d:].view(n, vh, d)}
    rate = torch.exp(_randn(g, vh) * 1.5 - 2)
    s["g"] = -rate * torch.log1p(torch.exp(_randn(g, n, vh)))
    s["beta"] = torch.sigmoid(_randn(g, n, vh))
    s["state"] = _randn(g, len(new), vh, d, d) * 0.2
    s["state_out"] = torch.zeros_like(s["state"])
    s["starts"], s["max_new"] = _ints(_starts(new)), max(new)
    s["out"] = torch.zeros((n, vh, d), dtype=t, device="cuda")
    chunks = -(-n // 64) + len(new)
    s["work"] = torch.empty((64 << 20) + chunks * vh * (80 << 10), dtype=torch.uint8, device="cuda")
    return s


_INPUTS = {"rope": _rope_inputs, "attn": _attn_inputs, "gdn": _gdn_inputs}


def prepare(case, seed):
    s = _INPUTS[case["kind"]](case, _generator(seed))
    s["case"] = case
    return s


# ---------------------------------------------------------------- plain forms
def _plain_rope(s):
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
    s["k_pages"][page, :, off] = turned(s["k"], s["k_norm"]).to(s["k_pages"].dtype)
    s["v_pages"][page, :, off] = s["v"].to(s["v_pages"].dtype)
    return {"q": s["q_out"], "k": s["k_pages"], "v": s["v_pages"]}


def _plain_attn(s):
    """All sequences at once, padded to the longest."""
    case = s["case"]
    kvh, d, page = case["kv_heads"], case["dim"], case["page"]
    group = case["heads"] // kvh
    n_seq, top, keys = case["n_seq"], s["max_new"], s["max_kv"]
    first = s["starts"][:-1].long()
    count = s["starts"][1:].long() - first
    kv_len = s["kv_len"].long()
    t = torch.arange(top, device="cuda")
    j = torch.arange(keys, device="cuda")
    k = s["k_pages"][s["table"].long()].transpose(2, 1).reshape(n_seq, kvh, -1, d)[:, :, :keys].float()
    v = s["v_pages"][s["table"].long()].transpose(2, 1).reshape(n_seq, kvh, -1, d)[:, :, :keys].float()
    rows = (first[:, None] + t).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().view(n_seq, top, kvh, group, d).permute(0, 2, 1, 3, 4).reshape(n_seq, kvh, top * group, d)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).view(n_seq, kvh, top, group, keys)
    seen = j <= (kv_len - count)[:, None, None] + t[:, None]
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    v = v.masked_fill_((j >= kv_len[:, None])[:, None, :, None], 0)
    out = torch.matmul(score.view(n_seq, kvh, top * group, keys), v).view(n_seq, kvh, top, group, d)
    out = out / score.sum(-1, keepdim=True)
    out = out.permute(0, 2, 1, 3, 4).reshape(n_seq, top, kvh * group, d)
    keep = t < count[:, None]
    s["out"][rows[keep]] = out[keep].to(s["out"].dtype)
    return s["out"]


def _unit(x):
    x = x.float()
    return x * torch.rsqrt(x.square().sum(-1, keepdim=True) + EPS)


def _plain_gdn(s):
    """In chunks of up to 64 tokens, all sequences at once, padded to the longest."""
    case = s["case"]
    n_seq, top, vh, kh, d = case["n_seq"], s["max_new"], case["v_heads"], case["k_heads"], case["dim"]
    c = min(64, top)
    steps = -(-top // c)
    first = s["starts"][:-1].long()
    count = s["starts"][1:].long() - first
    t = torch.arange(steps * c, device="cuda")
    keep = t < count[:, None]
    rows = torch.where(keep, first[:, None] + t, 0)

    def chunks(x):                                  # (n_seq, steps, heads, c, ...), zeros behind the end
        x = x[rows].float() * keep.view(n_seq, -1, *[1] * (x.dim() - 1))
        return x.view(n_seq, steps, c, *x.shape[2:]).transpose(2, 3)

    head = torch.arange(vh, device="cuda") % kh
    q, k = chunks(_unit(s["q"]))[:, :, head] * d ** -0.5, chunks(_unit(s["k"]))[:, :, head]
    v, beta = chunks(s["v"]), chunks(s["beta"][..., None])
    sums = chunks(s["g"][..., None])[..., 0].double().cumsum(-1)
    gaps = sums[..., :, None] - sums[..., None, :]
    below = torch.ones((c, c), dtype=torch.bool, device="cuda").tril()
    decay = torch.where(below, gaps, -math.inf).exp().float()
    mixed = torch.matmul(q, k.transpose(-1, -2)) * decay
    lower = (torch.matmul(k, k.transpose(-1, -2)) * decay * beta).tril(-1)
    inverse = torch.eye(c, device="cuda").expand_as(lower).clone()
    for i in range(1, c):                           # forward substitution, all chunks at once
        inverse[..., i, :] -= torch.matmul(lower[..., i:i + 1, :i], inverse[..., :i, :])[..., 0, :]
    inverse = inverse * beta.transpose(-1, -2)
    since = sums.exp().float()[..., None]
    left = (sums[..., -1:] - sums).exp().float()[..., None]
    last = sums[..., -1:].exp().float()[..., None]
    state, out = s["state"], []
    for i in range(steps):
        u = torch.matmul(inverse[:, i], v[:, i] - since[:, i] * torch.matmul(k[:, i], state))
        out.append(since[:, i] * torch.matmul(q[:, i], state) + torch.matmul(mixed[:, i], u))
        state = last[:, i] * state + torch.matmul((k[:, i] * left[:, i]).transpose(-1, -2), u)
    out = torch.stack(out, 1).transpose(2, 3).reshape(n_seq, steps * c, vh, d)
    s["out"].copy_(out[keep])
    s["state_out"].copy_(state)
    return {"out": s["out"], "state": s["state_out"]}


_PLAIN = {"rope": _plain_rope, "attn": _plain_attn, "gdn": _plain_gdn}


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
    if kind == "rope":
        B.qk_norm_rope(s["q"], s["k"], s["v"], s["q_norm"], s["k_norm"], EPS, s["pos"], s["inv_freq"], s["slots"],
                       s["k_pages"], s["v_pages"], s["q_out"])
        return {"q": s["q_out"], "k": s["k_pages"], "v": s["v_pages"]}
    if kind == "attn":
        B.attn_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["starts"], s["kv_len"], s["out"], s["work"],
                     max_kv=s["max_kv"])
        return s["out"]
    B.gdn(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s["state_out"], s["out"], s["starts"], s["work"],
          max_new=s["max_new"], l2_eps=EPS, tiled=True)
    return {"out": s["out"], "state": s["state_out"]}


# ---------------------------------------------------------- work, exactness
def _size(name):
    return 4 if name == "f32" else 2


def work(case):
    if case["kind"] == "rope":
        q, kv = case["heads"] * case["dim"], 2 * case["kv_heads"] * case["dim"]
        n = case["n_tok"]
        return {"bytes": n * (q * (4 + _size(case["q_type"])) + kv * (4 + 2)), "flops": n * (q + kv) * 6}
    new, kv = _lengths(case)
    if case["kind"] == "attn":
        pairs = sum(n * c - n * (n - 1) // 2 for n, c in zip(new, kv))
        q = sum(new) * case["heads"] * case["dim"]
        return {"bytes": 2 * _size(case["io"]) * q + sum(kv) * case["kv_heads"] * case["dim"] * 4,
                "flops": 4 * case["dim"] * case["heads"] * pairs}
    n, d, vh = sum(new), case["dim"], case["v_heads"]
    row = (2 * case["k_heads"] + 2 * vh) * d * _size(case["type"]) + 8 * vh
    return {"bytes": n * row + case["n_seq"] * vh * d * d * 8, "flops": 7 * d * d * vh * n}


def _exact_rope(case, s):
    def row(x, w):
        x = x.double()
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
        half = case["rot"] // 2
        y = x.clone()
        turn = torch.polar(torch.ones_like(s["inv_freq"]).expand(x.shape[0], half),
                           s["pos"].double()[:, None] * s["inv_freq"])[:, None]
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
        return y

    out = {"q": row(s["q"], s["q_norm"])}
    for name, x in (("k", row(s["k"], s["k_norm"])), ("v", s["v"].double())):
        pages = s[name + "_pages"].double()
        n_pages, kv, page, d = pages.shape
        flat = pages.transpose(1, 2).reshape(n_pages * page, kv, d)
        flat[s["slots"]] = x
        out[name] = flat.view(n_pages, page, kv, d).transpose(1, 2).contiguous()
    return out


def _exact_attn(case, s):
    new, kv = _lengths(case)
    d, page, group = case["dim"], case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, c) in enumerate(zip(new, kv)):
        used = s["table"][i, :-(-c // page)].long()
        for h in range(case["kv_heads"]):
            k = s["k_pages"][used, h].reshape(-1, d)[:c].double()
            v = s["v_pages"][used, h].reshape(-1, d)[:c].double()
            for r in range(0, n, 512):
                m = min(512, n - r)
                for x in range(h * group, (h + 1) * group):
                    p = s["q"][at + r:at + r + m, x].double() @ k.t() / math.sqrt(d)
                    late = torch.arange(c, device="cuda")[None] > (c - n + r + torch.arange(m, device="cuda"))[:, None]
                    p = torch.softmax(p.masked_fill(late, -math.inf), -1)
                    out[at + r:at + r + m, x] = p @ v
        at += n
    return out


def _exact_gdn(case, s):
    """Token by token."""
    new, _ = _lengths(case)
    kh, vh, d = case["k_heads"], case["v_heads"], case["dim"]
    q, k = (x.double() / (x.double().square().sum(-1, keepdim=True) + EPS).sqrt() for x in (s["q"], s["k"]))
    q, k = (x.repeat(1, vh // kh, 1)[..., None] for x in (q / math.sqrt(d), k))
    v, decay, beta = s["v"].double()[:, :, None], s["g"].double().exp(), s["beta"].double()
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    final = s["state"].double()
    # sequences that still have a token left step together
    starts = _starts(new)
    order = sorted(range(len(new)), key=lambda i: -new[i])
    state = final[order]
    firsts = torch.tensor([starts[i] for i in order], device="cuda")
    for t in range(max(new)):
        live = sum(new[i] > t for i in order)
        at = firsts[:live] + t
        S = state[:live] * decay[at][..., None, None]
        u = (v[at] - (k[at] * S).sum(-2, keepdim=True)) * beta[at][..., None, None]
        S = S + k[at] * u
        out[at] = (q[at] * S).sum(-2)
        state[:live] = S
    final[order] = state
    return {"out": out, "state": final}


def exact(case, seed):
    return {"rope": _exact_rope, "attn": _exact_attn, "gdn": _exact_gdn}[case["kind"]](case, prepare(case, seed))
