"""Attention over 8-bit pages where the scales of values are 0, tiny or large beside each other: a
weight counts in the softmax's sum whatever its value's scale is.

Reference: 64 bits; U = 2^-24 is a rounding of fp32."""
import pytest

import bonsai_p40 as B
from test_gpu_mixers import BF16, F16, F32, NAN, U, case, gen, half_step, ints, normwise
from test_gpu_q8_cache import pages_of

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")


def paged(codes, scales, page):
    """Rows (keys, heads, d) and their scales as pages in some order; (pages, their order)."""
    kv, kvh, d = codes.shape
    n = -(-kv // page)
    perm = torch.randperm(n, generator=gen(9))
    c, s = torch.zeros(n * page, kvh, d, dtype=torch.int8), torch.zeros(n * page, kvh)
    c[:kv], s[:kv] = codes, scales
    pc, ps = torch.empty(n, kvh, page, d, dtype=torch.int8), torch.empty(n, kvh, page)
    pc[perm], ps[perm] = c.view(n, page, kvh, d).transpose(1, 2), s.view(n, page, kvh).transpose(1, 2)
    return pages_of(pc, ps)[0], perm.int()


def check(got, ref, mag, top, io, keys, split, least=0.0):
    """q is whole.  A score of up to top is rounded 16 times (and its query's one element is off by 1.01 x 2^-15 or 1.6 x
    2^-23 of itself, as the header has it); a weight is rounded once to f16 (fp32: to 22 bits), or is off by 2^-36
    (2^-47) of the largest.  The sums over keys add a rounding a tile of 32, each U of a sum that is at most the whole:
    keys / 32 U in one part, where all may go the same way as the terms are alike.  least: more that a weight may be off
    by, of the largest, so that a sum of n of them is by that times n values."""
    assert torch.equal(torch.isfinite(got.double()), torch.isfinite(ref))
    e, p, tiny = (1.6 * 2.0 ** -23, 2.0 ** -22, 2.0 ** -47) if io == F32 else (1.01 * 2.0 ** -15, 2.0 ** -11, 2.0 ** -36)
    sums = (keys / 32 + 24) * U
    lim = mag * (2 * (e + 16 * U) * top + p + 2 * sums) + keys * max(tiny, least) * mag.amax(-1, keepdim=True) * 4
    lim = lim + half_step(io) * (ref.abs() + lim) + torch.finfo(io).tiny
    err = (got.double() - ref).abs()
    assert bool((err <= lim).all()), float((err - lim).max())
    rel = normwise(got, ref)
    assert rel <= (half_step(io) if io != F32 else 2.0 ** -18) + (0.0 if split else sums) + least * keys ** 0.5, rel


def attend(n, heads, d, score, vd, io, work, what, scale=1.0, seed=0, groups=None, tiny=0.0):
    """The last n tokens of one sequence whose key j has the score score[j] and values of scale vd[j]; groups: the keys
    that are the prefix of n sequences of one token each, of which the first has all the others."""
    kv = score.numel()
    case(f"q8 ranges {what} n={n} heads={heads} d={d} keys={kv} io={io} work={work} groups={groups}")
    g = gen(seed)
    q = torch.zeros(n, heads, d)
    q[..., 0] = 1.0                                         # (a whole number of any digits as it stands)
    q = q.to(io)
    kc = torch.zeros(kv, 1, d, dtype=torch.int8)
    kc[:, 0, 0] = 64
    ks = (score.float() / 64 / scale)[:, None]
    vc = torch.randint(-127, 128, (kv, 1, d), generator=g, dtype=torch.int8)
    vs = vd.float()[:, None]
    (kp, perm), (vp, _) = paged(kc, ks, 16), paged(vc, vs, 16)
    out = torch.full((n, heads, d), 7.0, dtype=io, device="cuda")
    x = (kc[:, 0, 0].double() * ks[:, 0].double() * scale)[None].expand(n, -1)
    if groups is None:
        args = [q.cuda(), kp, vp, perm.cuda()[None], ints([0, n]), ints([kv]), out]
        ws = torch.full((B.attn_paged_workspace_bytes(*args, max_kv=kv, scale=scale) + 16,), 255, dtype=torch.uint8, device="cuda") if work else None
        B.attn_paged(*args, ws, max_kv=kv, scale=scale)
        late = torch.arange(kv)[None] > (kv - n + torch.arange(n))[:, None]
    else:
        table = perm[None].repeat(n, 1)
        lens = [kv] + [groups] * (n - 1)
        args = [q.cuda(), kp, vp, table.cuda(), ints(range(n + 1)), ints(lens), ints([0, n]), ints([groups]), out]
        ws = torch.full((B.attn_shared_workspace_bytes(*args, max_kv=kv, max_shared=groups, scale=scale) + 16,), 255, dtype=torch.uint8, device="cuda")
        B.attn_shared(*args, ws, max_kv=kv, max_shared=groups, scale=scale)
        late = torch.arange(kv)[None] >= torch.tensor(lens)[:, None]
    torch.cuda.synchronize()
    p = torch.softmax(x.masked_fill(late, -INF), -1)
    v = vc[:, 0].double() * vs.double()
    ref, mag = p @ v, p @ v.abs()
    check(out.cpu(), ref[:, None].expand(n, heads, d), mag[:, None].expand(n, heads, d), float(x.abs().max()), io, kv, work, tiny)


LOG2 = 0.6931471805599453
SHAPES = [(1, 2, 256), (1, 1, 64), (40, 1, 128), (70, 2, 256)]


@pytest.mark.parametrize("n,heads,d", SHAPES)
@pytest.mark.parametrize("io", [BF16, F32])
@pytest.mark.parametrize("small", [0.0, 2.0 ** -100])
def test_scales_of_nothing_beside_large_ones(n, heads, d, io, small):
    """Equal scores: values of no or hardly any size count as keys all the same.  In one wave's tiles, in those of
    several, and in several parts; the large ones last, first, and in the middle."""
    for big in (2.0 ** 30, 2.0 ** 78):
        for lead, large, tail in ((32, 32, 0), (32, 33, 95), (256, 256, 0), (500, 40, 700), (0, 100, 400), (4000, 64, 4000)):
            if lead + large + tail < n:
                continue
            vd = torch.cat([torch.full((c,), x) for c, x in ((lead, small), (large, big), (tail, small))])
            for work in (True, False):
                attend(n, heads, d, torch.zeros(vd.numel()), vd, io, work, f"{lead} of {small}, {large} of {big}, {tail}")


@pytest.mark.parametrize("groups", [64, 5000])
@pytest.mark.parametrize("io", [BF16, F32])
def test_a_prefix_of_nothing_before_large_values(groups, io):
    """... with one in the prefix and the other among the own keys of the first sequence."""
    for n in (3, 40):
        for vd in ((0.0, 2.0 ** 60), (2.0 ** 60, 0.0)):
            vd = torch.cat([torch.full((groups,), vd[0]), torch.full((70,), vd[1])])
            attend(n, 2, 128, torch.zeros(vd.numel()), vd, io, True, "prefix and own keys", groups=groups)


@pytest.mark.parametrize("n,heads,d", SHAPES)
@pytest.mark.parametrize("small", [0.0, 2.0 ** -100])
def test_many_keys_without_values(n, heads, d, small):
    """40000 keys whose scores are 2.7 (3.9 in log2) above the first ones', all of values of no size, then 300 of
    ordinary ones that share the rest."""
    score = torch.cat([torch.zeros(256), torch.full((40000,), 2.7), torch.full((300,), 2.7)])
    vd = torch.cat([torch.full((40256,), small), torch.rand(300, generator=gen(2)) + 0.5])
    for io in (BF16, F32):
        for work in (True, False):
            attend(n, heads, d, score, vd, io, work, f"40000 of {small}")


def test_a_whole_long_cache_without_values():
    """600000 equal scores in one part: values of 2^-100 alone, and with some ordinary ones behind them."""
    score = torch.zeros(600000)
    vd = torch.full((600000,), 2.0 ** -100)
    for n in (1, 33):
        attend(n, 1, 64, score, vd, F32, False, "600000 of 2^-100")
    vd[-1000:] = 1.0
    for n in (1, 33):
        attend(n, 1, 64, score, vd, F32, False, "599000 of 2^-100")


@pytest.mark.parametrize("n,heads,d", SHAPES)
def test_weights_far_below_a_key_whose_value_is_large(n, heads, d):
    """Thousands of keys without values 27 (log2) below one that has one: their share of the sum is 2^-15."""
    score = torch.cat([torch.zeros(4000), torch.full((1,), 27 * LOG2), torch.zeros(80)])
    vd = torch.cat([torch.zeros(4000), torch.ones(1), torch.zeros(80)])
    for work in (True, False):
        attend(n, heads, d, score, vd, F32, work, "behind zeros")
        attend(n, heads, d, score.flip(0), vd.flip(0), F32, work, "before zeros")


@pytest.mark.parametrize("n,heads,d", SHAPES)
def test_large_scores_with_large_and_small_scales(n, heads, d):
    """Scores where fp32 has steps of 64 and more, equal or far apart, values of 2^-60 .. 2^60: the products of weight
    and scale stay within f16."""
    for size in (2.0 ** 21, 2.0 ** 30, 2.0 ** 80):
        score = torch.zeros(600)
        score[::3] = size
        for vd in (torch.full((600,), 2.0 ** 60), torch.full((600,), 2.0 ** -60), 2.0 ** torch.linspace(-60, 60, 600), 2.0 ** torch.linspace(60, -60, 600)):
            for io in (BF16, F32):
                attend(n, heads, d, score, vd, io, True, f"scores of {size}")


@pytest.mark.parametrize("d", [64, 256])
def test_scales_far_apart_in_16_bits(d):
    """Scales that grow or fall from key to key by many powers of two, bf16 rows: every row against its own size."""
    for n, kv in ((1, 300), (70, 200), (40, 40)):
        for low, high in ((-60, 60), (60, -60), (-110, -100), (70, 78)):
            vd = 2.0 ** torch.round(low + (high - low) * torch.arange(kv) / kv)
            attend(n, 2, d, torch.randn(kv, generator=gen(kv)), vd, BF16, True, f"2^{low} .. 2^{high}")
            if n > 1:
                continue
            # f16 holds the results of scales up to 2^8
            attend(n, 2, d, torch.randn(kv, generator=gen(kv)), 2.0 ** torch.linspace(-20, 8, kv), F16, True, "2^-20 .. 2^8")
            attend(n, 2, d, torch.randn(kv, generator=gen(kv)), 2.0 ** torch.linspace(8, -20, kv), F16, True, "2^8 .. 2^-20")


@pytest.mark.parametrize("kind", ["q8", F16, BF16])
@pytest.mark.parametrize("value", [0.0, 2.0 ** -112, 2.0 ** -140])
def test_scores_whose_factor_is_next_to_nothing(kind, value):
    """Queries of (next to) nothing and a scale of 1e-9 or less: every score is 0, and each token's result the mean of
    the values it sees."""
    d, kv = 64, 100
    g = gen(3)
    codes = torch.randint(-127, 128, (kv, 1, d), generator=g, dtype=torch.int8)
    one = torch.full((kv, 1), 2.0 ** -6)
    if kind == "q8":
        (kp, perm), (vp, _) = paged(codes, one, 16), paged(codes.flip(0), one, 16)
    else:
        perm = torch.arange(7, dtype=torch.int32)
        kp, vp = ((torch.cat([x, torch.zeros(12, 1, d)]).view(7, 16, 1, d).transpose(1, 2) * 2.0 ** -6).to(kind).cuda() for x in (codes, codes.flip(0)))
    v = codes.flip(0)[:, 0].double() * 2.0 ** -6
    for n in (1, 40):
        for scale in (1e-9, 1e-30, 1e-45):
            case(f"tiny scores {kind} value={value} n={n} scale={scale}")
            out = torch.zeros(n, 2, d, device="cuda")
            B.attn_paged(torch.full((n, 2, d), value, device="cuda"), kp, vp, perm.cuda()[None], ints([0, n]), ints([kv]), out, scale=scale)
            torch.cuda.synchronize()
            ref = torch.stack([v[:kv - n + t + 1].mean(0) for t in range(n)])[:, None].expand(n, 2, d)
            # weights of 22 bits or more, alike; sums of 100 terms
            assert bool(((out.cpu().double() - ref).abs() <= (2.0 ** -21 + 16 * U) * v.abs().max()).all()), (n, scale)


@pytest.mark.parametrize("io", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 256])
def test_queries_of_nan_that_see_no_key(io, d):
    """0, as of any query without keys: whole sequences, a chunk's first tokens beside others that see some, pages that
    are none; those that see a key are NaN."""
    case(f"q8 ranges queries of NaN without keys io={io} d={d}")
    pages = pages_of(torch.ones(9, 1, 16, d, dtype=torch.int8), torch.ones(9, 1, 16))[0]
    for starts, lens, table, seen in (
            ([0, 1, 2], [0, 5], [[0, 1, 2], [3, 4, 5]], [0, 1]),
            ([0, 40, 41], [3, 0], [[0, 1, 2], [3, 4, 5]], [0] * 37 + [1] * 3 + [0]),
            ([0, 70, 75], [48, 2], [[-1, -1, 7], [-1, 9, 8]], [0] * 54 + [1] * 16 + [0] * 5),
            ([0, 1, 2], [300, 300], [[-1] * 19, [-1] * 9 + [3] + [-1] * 9], [0, 1])):
        n = starts[-1]
        q = torch.full((n, 2, d), NAN, dtype=io)
        out = torch.full((n, 2, d), 7.0, dtype=io, device="cuda")
        for work in (True, False):
            args = [q.cuda(), pages, pages, ints(table), ints(starts), ints(lens), out.fill_(7.0)]
            ws = torch.full((B.attn_paged_workspace_bytes(*args) + 16,), 255, dtype=torch.uint8, device="cuda") if work else None
            B.attn_paged(*args, ws)
            torch.cuda.synchronize()
            some = torch.tensor(seen, dtype=torch.bool)
            assert bool(out.cpu()[some].isnan().all()) and bool((out.cpu()[~some] == 0).all()), (starts, lens, work)


@pytest.mark.parametrize("n,heads,d", SHAPES)
def test_values_as_small_as_the_append_writes(n, heads, d):
    """Scales of 2^-119, those of rows of 2^-112, alone and beside others: a weight is off by up to 2^-17 (fp32 rows
    2^-28) of the largest where all that a row sees are below 2^-100."""
    score = torch.randn(200, generator=gen(n))
    for low, high in ((-119, -119), (-119, -101), (-119, 0)):
        vd = 2.0 ** torch.round(low + (high - low) * torch.rand(200, generator=gen(1)))
        for io in (BF16, F32):
            attend(n, heads, d, score, vd, io, True, f"2^{low} .. 2^{high}", tiny=2.0 ** (-28 if io == F32 else -17) if high < -100 else 0.0)
