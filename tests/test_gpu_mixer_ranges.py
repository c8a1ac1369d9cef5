"""The token mixers where a row's values span many powers of two: what is small
keeps its digits beside what is large, as it does in fp32 sums.

Reference: 64 bits.  U = 2^-24 is a rounding of fp32."""
import pytest

import bonsai_p40 as B
from test_gpu_mixers import BF16, F16, F32, U, case, gen, half_step, ints, normwise, run_attn

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")


def attend(q, k, v, io, t, work=True, page=16):
    """attn_paged of the last tokens of one sequence; (result, the same in 64 bits)."""
    n, heads, d = q.shape
    kv, kvh, _ = k.shape
    pages = -(-kv // page)
    q, k, v = q.to(io), k.to(t), v.to(t)
    perm = torch.randperm(pages, generator=gen(9))
    both = []
    for x in (k, v):
        full = torch.zeros(pages * page, kvh, d, dtype=t)
        full[:kv] = x
        store = torch.empty(pages, kvh, page, d, dtype=t)
        store[perm] = full.view(pages, page, kvh, d).transpose(1, 2)
        both.append(store.cuda())
    out = torch.full((n, heads, d), 7.0, dtype=io, device="cuda")
    args = [q.cuda(), *both, perm.int().cuda()[None], ints([0, n]), ints([kv]), out]
    ws = torch.full((B.attn_paged_workspace_bytes(*args, max_kv=kv) + 16,), 255, dtype=torch.uint8, device="cuda") if work else None
    B.attn_paged(*args, ws, max_kv=kv)
    torch.cuda.synchronize()
    group = heads // kvh
    ref = torch.empty(n, heads, d, dtype=torch.float64)
    late = torch.arange(kv)[None] > (kv - n + torch.arange(n))[:, None]
    for h in range(heads):
        x = (q[:, h].double() @ k[:, h // group].double().t()) * d ** -0.5
        ref[:, h] = torch.softmax(x.masked_fill(late, -float("inf")), -1) @ v[:, h // group].double()
    return out.cpu(), ref


def sink_limit(io, gap, ref):
    store = 2.0 ** -25 * ref.numel() ** 0.5 / float(ref.norm()) if io == F16 else 0.0
    return (2.0 ** -18 if io == F32 else half_step(io)) + 2 * gap * 1.4427 * U + store


SHAPES = [(1, 4000, 6, 1, 256), (1, 3000, 4, 2, 128), (40, 1500, 6, 1, 256), (70, 900, 4, 2, 64), (50, 700, 2, 1, 128)]


@pytest.mark.parametrize("n,kv,heads,kvh,d", SHAPES)
@pytest.mark.parametrize("t,io", [(F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("gap", [10, 14, 18])
def test_attn_a_key_that_has_nearly_all_the_weight(n, kv, heads, kvh, d, t, io, gap):
    """One key's score is `gap` above thousands of others (an attention sink), and its value is 0 or small: the
    result is what the others, e^-gap of the weight each, make of it.

    The key's score is one product of numbers that the types hold, so it is exact.  Behind it, an exponent's
    argument of up to gap log2(e) is rounded twice; the rest is as with scores of one size.  A result below 2^-14,
    f16's smallest normal number, is stored to a multiple of 2^-24 and so off by up to 2^-25: of N results, by
    2^-25 sqrt(N) of the norm (gap 14: results of e^-14 30 = 2.5e-5 beside steps of 6e-8)."""
    case(f"sink n={n} kv={kv} heads={heads}/{kvh} d={d} {t} io={io} gap={gap}")
    g = gen(gap + n)
    q, k, v = torch.randn(n, heads, d, generator=g), torch.randn(kv, kvh, d, generator=g) * 0.5, torch.randn(kv, kvh, d, generator=g)
    q[..., 0] = 4.0
    k[..., 0] = 0.0
    k[0] = 0.0
    k[0, :, 0] = round(gap * d ** 0.5 / 4)
    for value, work in ((0.0, True), (0.0, False), (2.0 ** -12, True)):
        v[0] = value
        got, ref = attend(q, k, v, io, t, work)
        err, limit = normwise(got, ref), sink_limit(io, gap, ref)
        print(f"value {value}: {err:.2e} of {limit:.2e}", flush=True)
        assert err <= limit


@pytest.mark.parametrize("gap", [10, 18])
def test_attn_the_key_comes_late(gap):
    """The same with the key among the last: what was summed before it is scaled down, and counts."""
    for n, kv, d, at in ((1, 2000, 128, 1990), (1, 2000, 256, 700), (40, 600, 256, 400), (40, 600, 64, 540)):
        for io in (F32, F16):
            case(f"late sink n={n} kv={kv} d={d} at={at} io={io} gap={gap}")
            g = gen(at)
            q, k, v = torch.randn(n, 2, d, generator=g), torch.randn(kv, 1, d, generator=g) * 0.5, torch.randn(kv, 1, d, generator=g)
            q[..., 0] = 4.0
            k[..., 0] = 0.0
            k[at] = 0.0
            k[at, :, 0] = round(gap * d ** 0.5 / 4)
            v[at] = 0.0
            got, ref = attend(q, k, v, io, F16)
            err = normwise(got, ref)
            print(f"{err:.2e}", flush=True)
            assert err <= sink_limit(io, gap, ref)


@pytest.mark.parametrize("n,kv", [(1, 900), (40, 600)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("high", [2.0 ** 8, 2.0 ** 14])
def test_attn_query_elements_beside_a_large_one(n, kv, d, high):
    """Queries with one element far above the others, where every key is 0: the scores come of the others."""
    for t in (F16, BF16):
        case(f"large element n={n} d={d} high={high} {t}")
        g = gen(d)
        q, k, v = torch.randn(n, 4, d, generator=g), torch.randn(kv, 2, d, generator=g), torch.randn(kv, 2, d, generator=g)
        q[..., 5] = high
        k[..., 5] = 0.0
        got, ref = attend(q, k, v, F32, t)
        err = normwise(got, ref)
        print(f"{err:.2e}", flush=True)
        assert err <= 2.0 ** -18


@pytest.mark.parametrize("t,io", [(F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("n,kv,d", [(1, 50, 64), (1, 3000, 256), (40, 90, 128), (40, 700, 256)])
def test_attn_scores_of_minus_infinity(n, kv, d, t, io):
    """A key whose score is -inf has no weight, and where no other is seen the softmax is 0 / 0, not 0.  fp32 queries
    meet a key's infinity with each of their terms, of which one is 0: NaN."""
    g = gen(kv)
    for which in ("all", "some", "first"):
        case(f"-inf n={n} kv={kv} d={d} {t} {io} {which}")
        q, k, v = torch.randn(n, 2, d, generator=g), torch.randn(kv, 1, d, generator=g), torch.randn(kv, 1, d, generator=g)
        q[..., 3] = 300.0
        k[..., 3] = 0.0                                     # (300 times -inf is -inf)
        hit = slice(None) if which == "all" else slice(0, kv, 3) if which == "some" else slice(0, kv - n + 1)
        k[hit, :, 3] = -float("inf")
        for work in (True, False):
            got, ref = attend(q, k, v, io, t, work)
            # "first": the first token sees such keys only
            assert bool(ref.isnan().all()) if which == "all" else bool(ref[0].isnan().all()) == (which == "first")
            if io == F32:
                assert bool(got.isnan().all())
                continue
            assert torch.equal(got.isnan(), ref.isnan())
            fin = ~ref.isnan()
            assert normwise(got[fin], ref[fin]) <= half_step(io)


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("n,kv,d", [(1, 4000, 256), (1, 3000, 64), (30, 3000, 128)])
def test_attn_minus_infinity_in_whole_parts(n, kv, d, t):
    """Workgroups and waves that see keys of -inf only, beside others: they count for nothing in the join."""
    g = gen(kv + n)
    for hit in (slice(0, kv // 2), slice(kv // 2, kv - n), slice(64, kv - n - 64)):
        case(f"-inf part n={n} kv={kv} d={d} {t} {hit}")
        q, k, v = torch.randn(n, 4, d, generator=g), torch.randn(kv, 2, d, generator=g), torch.randn(kv, 2, d, generator=g)
        q[..., 3], k[..., 3] = 300.0, 0.0
        k[hit, :, 3] = -float("inf")
        for work in (True, False):
            got, ref = attend(q, k, v, t, t, work)
            assert normwise(got, ref) <= half_step(t)


@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_attn_what_is_not_seen_stays_out_of_f16(io, value):
    """Keys and values of later tokens of the same chunk, whatever they hold, with the terms of f16 pages."""
    for new, kv, heads, kvh, d in (([40], [40], 6, 1, 256), ([9], [50], 3, 1, 128), ([100, 30], [230, 30], 4, 1, 64)):
        def both(q, k, v, table):
            for s, (n, c) in enumerate(zip(new, kv)):
                for j in (c - 1, c - n // 2):
                    k[int(table[s, j // 16]), :, j % 16] = v[int(table[s, j // 16]), :, j % 16] = value
        run_attn(new, kv, heads, kvh, d, 16, F16, io, edit=both)

        def values_only(q, k, v, table):
            for s, (n, c) in enumerate(zip(new, kv)):
                v[int(table[s, (c - 2) // 16]), :, (c - 2) % 16, 3] = value
        run_attn(new, kv, heads, kvh, d, 16, F16, io, edit=values_only)


@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("n,kv", [(1, 2000), (40, 500)])
def test_attn_large_values(n, kv, io):
    """Values up to f16's largest, all of the weight on them or spread over all keys: sums stay inside fp32."""
    for d in (64, 256):
        for spread in (0.0, 1.0):
            case(f"large values n={n} kv={kv} d={d} {io} spread={spread}")
            g = gen(d)
            q, k = torch.randn(n, 2, d, generator=g) * spread, torch.randn(kv, 1, d, generator=g)
            v = torch.where(torch.rand(kv, 1, d, generator=g) < 0.5, -65504.0, 65504.0)
            v[..., 0] = 65504.0
            got, ref = attend(q, k, v, io, F16)
            err = (got.double() - ref).abs().max()
            # beside the mean of the magnitudes, 65504: 2^-18, or P's and the store's half steps
            assert float(err) <= 65504 * (2.0 ** -18 if io == F32 else 2 * half_step(io))


@pytest.mark.parametrize("t,io", [(F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("n,kv,d", [(1, 60, 64), (1, 3000, 256), (1, 2000, 128), (40, 300, 64), (40, 700, 256), (50, 600, 128)])
@pytest.mark.parametrize("high", [300.0, 3000.0, 60000.0])
def test_attn_scores_of_any_size(n, kv, d, t, io, high):
    """Queries and keys up to f16's largest: scores of up to 2^36, which fp32 holds to 2^12 of it.

    The largest score of a row is far above the next (where it is not, by 2^-18 of the largest and 40, the row is
    not looked at): its key has all the weight, and the row is that key's value."""
    case(f"scores n={n} kv={kv} d={d} {t} io={io} high={high}")
    g = gen(int(high) + d)
    q, k = (torch.rand(n, 2, d, generator=g) * 2 - 1) * high, (torch.rand(kv, 1, d, generator=g) * 2 - 1) * high
    v = torch.randn(kv, 1, d, generator=g)
    for work in (True, False):
        got, ref = attend(q, k, v, io, t, work)
        for h in range(2):
            x = (q[:, h].to(io).double() @ k[:, 0].to(t).double().t()) * d ** -0.5
            x = x.masked_fill(torch.arange(kv)[None] > (kv - n + torch.arange(n))[:, None], -float("inf"))
            top = x.topk(2, -1)
            clear = top.values[:, 0] - top.values[:, 1] > 40 + 2.0 ** -18 * x.masked_fill(x.isinf(), 0.0).abs().amax(-1)
            assert int(clear.sum()) >= (n + 1) // 2 or high < 1000
            want = v[top.indices[:, 0], 0].to(t).double()
            assert torch.equal(ref[clear, h], want[clear])
            # V's own value times P over l: one weight, of which P has the half step of 16 bits and the store another, or
            # 2^-22 (fp32), and l, 1 / l and the product 3 roundings
            off = (got[clear, h].double() - want[clear]).abs()
            step = 2 * half_step(io) if io != F32 else 2.0 ** -22
            assert bool((off <= want[clear].abs() * (step + 8 * U)).all())
            assert bool(torch.isfinite(got).all())


@pytest.mark.parametrize("t,io", [(F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("n,kv,d", [(1, 2000, 256), (1, 900, 64), (40, 600, 128), (40, 500, 256)])
def test_attn_scores_far_from_the_others(n, kv, d, t, io):
    """Keys whose scores are 2^22 and more below the others' count for nothing, wherever they come; one far above has
    all the weight.  (Powers of two in one element, so that those scores are exact; the others' are sums in fp32 of
    products of usual size.)"""
    g = gen(kv + d)
    for low in (slice(0, kv // 3), slice(kv // 4, kv // 2), slice(0, kv, 2)):
        case(f"far below n={n} kv={kv} d={d} {t} io={io} {low}")
        q, k, v = torch.randn(n, 2, d, generator=g), torch.randn(kv, 1, d, generator=g), torch.randn(kv, 1, d, generator=g)
        q[..., 0], k[..., 0] = 4096.0, 0.0
        k[low, :, 0] = -16384.0
        k[kv - n, :, 0] = 0.0
        for work in (True, False):
            got, ref = attend(q, k, v, io, t, work)
            assert normwise(got, ref) <= (2.0 ** -18 if io == F32 else half_step(io))
    for at in (0, kv // 2, kv - n):
        case(f"far above n={n} kv={kv} d={d} {t} io={io} at={at}")
        q, k, v = torch.randn(n, 2, d, generator=g), torch.randn(kv, 1, d, generator=g), torch.randn(kv, 1, d, generator=g)
        q[..., 0], k[..., 0] = 4096.0, 0.0
        k[at, :, 0] = 16384.0
        got, ref = attend(q, k, v, io, t)
        off, want = (got.double() - ref).abs(), v[at, 0].to(t).double()
        assert torch.equal(ref, want.expand_as(ref))
        # as with scores of any size: P's step and the store's
        step = 2 * half_step(io) if io != F32 else 2.0 ** -22
        assert bool((off <= want.abs() * (step + 8 * U)).all())


# -------------------------------------------------------------------- gdn
def delta(q, k, v, g, beta, state, t, eps, work=True, scale=None):
    """One sequence; ((outputs, state), the same in 64 bits).  Heads as they come."""
    n, heads, kd = q.shape
    q, k, v = q.to(t), k.to(t), v.to(t)
    out = torch.full(v.shape, 7.0, dtype=t, device="cuda")
    so = torch.zeros_like(state, device="cuda")
    args = (q.cuda(), k.cuda(), v.cuda(), g.cuda(), beta.cuda(), state.cuda(), so, out, ints([0, n]))
    kw = dict(l2_eps=eps, scale=scale)
    ws = torch.full((B.gdn_workspace_bytes(*args, **kw) + 16,), 255, dtype=torch.uint8, device="cuda") if work else None
    B.gdn(*args, ws, **kw)
    torch.cuda.synchronize()
    q, k, v, g, beta = (x.double() for x in (q, k, v, g, beta))
    if eps > 0:
        q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + eps) for x in (q, k))
    S, ref = state[0].double(), []
    for i in range(n):
        S = S * g[i].exp()[:, None, None]
        u = beta[i][:, None] * (v[i] - (k[i][:, :, None] * S).sum(1))
        S = S + k[i][:, :, None] * u[:, None]
        ref.append((q[i][:, :, None] * S).sum(1) * (kd ** -0.5 if scale is None else scale))
    return (out.cpu(), so.cpu()[0]), (torch.stack(ref), S)


def check_rows(got, ref, rows, tol, t):
    """Every (token, head) row by itself, beside the root mean square norm of its head's rows."""
    err = (got[rows].double() - ref[rows]).norm(dim=-1)
    norm = ref[rows].norm(dim=-1)
    rms = norm.square().mean(0, keepdim=True).sqrt()
    worst = float(((err - (half_step(t) * norm if t != F32 else 0)) / rms).max())
    print(f"{worst:.2e} of {tol:.2e}", flush=True)
    assert worst <= tol


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("kd,vd", [(128, 128), (64, 32)])
@pytest.mark.parametrize("work", [True, False])
@pytest.mark.parametrize("high", [2.0 ** 10, 2.0 ** 14, 2.0 ** 20])
def test_gdn_tokens_before_a_large_one(high, work, kd, vd, t):
    """One token's values far above the others': what comes before it does not lose by it.

    2^-18 as for values of one size, and what 2^-40 of a chunk's largest comes to, with 8 for the sums."""
    for n, at in ((138, 100), (60, 59), (70, 20)):
        case(f"gdn before high={high} work={work} {kd}x{vd} {t} n={n} at={at}")
        r = gen(n)
        q, k = torch.randn(n, 2, kd, generator=r), torch.randn(n, 2, kd, generator=r)
        v, state = torch.randn(n, 2, vd, generator=r), torch.randn(1, 2, kd, vd, generator=r) * 0.3
        v[at] *= high
        g, beta = -0.3 * torch.rand(n, 2, generator=r), torch.sigmoid(torch.randn(n, 2, generator=r))
        (out, _), (ref, _) = delta(q, k, v, g, beta, state, t, 1e-6, work)
        check_rows(out, ref, list(range(at)), 2.0 ** -18 + 8 * 2.0 ** -40 * high, t)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("work", [True, False])
@pytest.mark.parametrize("high", [2.0 ** 10, 2.0 ** 15])
def test_gdn_tokens_after_a_large_one_that_has_decayed(high, work, t):
    """Decay of e^-5 a token: 8 tokens later nothing of the large one is left, and nothing lost."""
    for n, at in ((60, 20), (140, 70)):
        case(f"gdn after high={high} work={work} {t} n={n} at={at}")
        r = gen(n)
        q, k = torch.randn(n, 2, 128, generator=r), torch.randn(n, 2, 128, generator=r)
        v, state = torch.randn(n, 2, 64, generator=r), torch.randn(1, 2, 128, 64, generator=r) * 0.3
        v[at] = torch.where(v[at] > 0, 1.0, -1.0) * high
        g, beta = torch.full((n, 2), -5.0), torch.sigmoid(torch.randn(n, 2, generator=r))
        (out, S), (ref, final) = delta(q, k, v, g, beta, state, t, 1e-6, work)
        rows = [i for i in range(n) if i < at or i >= at + 8]
        tol = 2.0 ** -18 + 8 * 2.0 ** -40 * high
        check_rows(out, ref, rows, tol, t)
        assert all(normwise(S[h], final[h]) <= tol for h in range(2))


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("work", [True, False])
def test_gdn_elements_of_a_row_beside_a_large_one(work, t):
    """Queries and keys with an element 2^18 above the others where the state is 0 (and the other side is): the
    others make the results.  2^-40 2^18 and the sums of 128: below 2^-18."""
    n = 100
    case(f"gdn row range work={work} {t}")
    for large in ("q", "k"):
        r = gen(3)
        q, k = torch.randn(n, 2, 128, generator=r), torch.randn(n, 2, 128, generator=r) / 16
        v, state = torch.randn(n, 2, 64, generator=r), torch.randn(1, 2, 128, 64, generator=r)
        state[:, :, 0] = 0.0
        q[..., 0], k[..., 0] = 0.0, 0.0
        if large == "q":
            q *= 2.0 ** -6
            q[..., 0] = 2.0 ** 12
            beta = torch.sigmoid(torch.randn(n, 2, generator=r))
        else:
            k *= 2.0 ** -6
            k[:1, :, 0] = 2.0 ** 8                         # one key: the others do not meet it
            beta = torch.sigmoid(torch.randn(n, 2, generator=r))
            beta[0] = 2.0 ** -40
        g = -0.01 * torch.rand(n, 2, generator=r)
        (out, S), (ref, final) = delta(q, k, v, g, beta, state, t, 0.0, work)
        check_rows(out, ref, list(range(n)), 2.0 ** -18, t)
        assert all(normwise(S[h], final[h]) <= 2.0 ** -18 for h in range(2))


@pytest.mark.parametrize("work", [True, False])
def test_gdn_rows_of_the_state_beside_a_large_one(work):
    """A state with one row 2^15 above the others, which no key or query meets: 2^-40 2^15 is below 2^-18."""
    n, r = 100, gen(6)
    case(f"gdn state range work={work}")
    q, k = torch.randn(n, 2, 128, generator=r), torch.randn(n, 2, 128, generator=r)
    v, state = torch.randn(n, 2, 64, generator=r), torch.randn(1, 2, 128, 64, generator=r)
    q[..., 7], k[..., 7] = 0.0, 0.0
    state[:, :, 7] *= 2.0 ** 15
    g, beta = -0.01 * torch.rand(n, 2, generator=r), torch.sigmoid(torch.randn(n, 2, generator=r))
    (out, S), (ref, final) = delta(q, k, v, g, beta, state, F32, 1e-6, work)
    check_rows(out, ref, list(range(n)), 2.0 ** -18, F32)
    rest = [i for i in range(128) if i != 7]
    assert all(normwise(S[h][rest], final[h][rest]) <= 2.0 ** -18 for h in range(2))

@pytest.mark.parametrize("work", [True, False])
def test_gdn_large_and_small_rows(work):
    """Rows of 2^60 and of 2^-60: each by itself, as sums of fp32 have them."""
    case(f"gdn powers work={work}")
    for power in (-60, 60):
        n, r = 80, gen(4)
        q, k = torch.randn(n, 2, 64, generator=r), torch.randn(n, 2, 64, generator=r)
        v = torch.randn(n, 2, 32, generator=r) * 2.0 ** power
        state = torch.randn(1, 2, 64, 32, generator=r) * 2.0 ** power
        g, beta = -0.3 * torch.rand(n, 2, generator=r), torch.sigmoid(torch.randn(n, 2, generator=r))
        (out, S), (ref, final) = delta(q, k, v, g, beta, state, F32, 1e-6, work)
        check_rows(out, ref, list(range(n)), 2.0 ** -18, F32)
        assert all(normwise(S[h], final[h]) <= 2.0 ** -18 for h in range(2))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta", "state"])
@pytest.mark.parametrize("work", [True, False])
def test_gdn_values_that_are_not_finite(work, name, value):
    """They reach their head of their sequence, from their chunk (token by token: from themselves) on, and nothing else."""
    case(f"gdn {name}={value} work={work}")
    n, heads, r = 200, 3, gen(5)
    x = dict(q=torch.randn(2 * n, heads, 64, generator=r), k=torch.randn(2 * n, heads, 64, generator=r),
             v=torch.randn(2 * n, heads, 32, generator=r), g=-0.1 * torch.rand(2 * n, heads, generator=r),
             beta=torch.rand(2 * n, heads, generator=r), state=torch.randn(2, heads, 64, 32, generator=r))
    at = 150                                               # in the third chunk of the first sequence

    def run():
        out, so = torch.zeros(2 * n, heads, 32, device="cuda"), torch.zeros(2, heads, 64, 32, device="cuda")
        args = (*(x[i].cuda() for i in ("q", "k", "v", "g", "beta", "state")), so, out, ints([0, n, 2 * n]))
        ws = torch.empty(B.gdn_workspace_bytes(*args, l2_eps=1e-6) + 16, dtype=torch.uint8, device="cuda") if work else None
        B.gdn(*args, ws, l2_eps=1e-6)
        torch.cuda.synchronize()
        return out.cpu(), so.cpu()
    out0, so0 = run()
    if name == "state":
        x["state"][0, 1, 7] = value                        # (a row: every column has one)
    elif x[name].dim() == 3:
        x[name][at, 1, 5 if name in "qk" else slice(None)] = value
    else:
        x[name][at, 1] = value
    out, so = run()
    # a decay of e^-inf is e^-10000, that is 0: nothing that is not finite comes of it
    if name == "g" and value < 0:
        assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(so).all())
        return
    assert torch.equal(out[:, [0, 2]], out0[:, [0, 2]]) and torch.equal(out[n:], out0[n:])
    assert torch.equal(so[1], so0[1]) and torch.equal(so[0, [0, 2]], so0[0, [0, 2]])
    first = 0 if name == "state" else at // 64 * 64 if work else at
    assert torch.equal(out[:first, 1], out0[:first, 1])
    row = 0 if name == "state" else at
    assert not bool(torch.isfinite(out[row, 1]).any())
    if name != "q":                                        # (a query is its own token's alone)
        assert not bool(torch.isfinite(out[row:n, 1]).any()) and not bool(torch.isfinite(so[0, 1]).any(0).any())
