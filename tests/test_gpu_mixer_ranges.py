"""The token mixers where a row's values span many powers of two: what is small
keeps its digits beside what is large, as it does in fp32 sums.

Reference: 64 bits.  U = 2^-24 is a rounding of fp32."""
import pytest

import bonsai_p40 as B
from test_gpu_mixers import BF16, F16, F32, U, case, gen, half_step, ints, normwise

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
