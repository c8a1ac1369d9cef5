"""The token mixers (qk_norm_rope, attn_paged, gdn) against plain implementations
in 64 bits, at the sizes and masks where they can go wrong.

Tolerances count roundings.  A store to a type t is off by at most
finfo(t).eps / 2 of the value; fp32 arithmetic by 2^-24 an operation."""
import ctypes as C
import math

import pytest

import bonsai_p40 as B

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24
NAN = float("nan")


def case(text):
    print("[case] " + text, flush=True)


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def half_step(t):
    return torch.finfo(t).eps / 2


def ints(v, t=torch.int32):
    return torch.tensor(v, dtype=t).cuda()


def normwise(got, ref):
    d = (got.double().cpu() - ref).norm()
    return float(d / ref.norm()) if ref.norm() > 0 else float(d)


# ------------------------------------------------------------ qk_norm_rope
def rope_ref(x, w, eps, pos, inv_freq, interleaved):
    """(result, sum of the magnitudes it is made of) in 64 bits."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    y, mag = x.clone(), x.abs()
    r = 2 * len(inv_freq)
    if r:
        a = (pos.double()[:, None] * inv_freq)[:, None]
        i, j = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
        y[..., i] = x[..., i] * a.cos() - x[..., j] * a.sin()
        y[..., j] = x[..., j] * a.cos() + x[..., i] * a.sin()
        mag = mag.clone()
        mag[..., i] = mag[..., j] = x[..., i].abs() + x[..., j].abs()
    return y, mag


def run_rope(n, heads, kv, d, rot, page, qt, ct, columns, far=5000, interleaved=False, norm=True, seed=0, extra=2,
             odd=False, slots=None):
    case(f"rope n={n} heads={heads}/{kv} d={d} rot={rot} page={page} {qt} {ct} columns={columns} il={interleaved}")
    g = gen(seed)
    full = [torch.randn(n, h, w + (1 if odd else 0), generator=g) * 2 for h, w in ((heads, 2 * d), (kv, d), (kv, d))]
    dev = []
    for t in full:
        t = t.cuda()
        dev.append(t.permute(1, 2, 0).contiguous().permute(2, 0, 1) if columns else t)
    q, k, v = (t[:, :, :d] for t in dev)
    wq, wk = (torch.randn(d, generator=g) * 0.2 + 1 for _ in range(2))
    inv = 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    pos = torch.randint(0, far, (n,), generator=g, dtype=torch.int32)
    pages = -(-n // page) + extra
    if slots is None:
        slots = torch.randperm(pages * page, generator=g)[:n]
    kp = torch.randn(pages, kv, page, d, generator=g).to(ct).cuda()
    vp = torch.randn(pages, kv, page, d, generator=g).to(ct).cuda()
    k0, v0 = kp.cpu(), vp.cpu()
    qo = torch.full((n, heads, d), NAN, dtype=qt, device="cuda")
    B.qk_norm_rope(q, k, v, wq.cuda() if norm else None, wk.cuda() if norm else None, 1e-6, pos.cuda(), inv.cuda(),
                   slots.cuda(), kp, vp, qo, interleaved)
    torch.cuda.synchronize()
    # the mean's sum (10 roundings), + eps, root, reciprocal and 2 products: 15; cos and sin: 2 and 3.2 for
    # the angle's own rounding; 2 in the rotation
    fp32 = 24 * U
    for name, got, src, w in (("q", qo, full[0], wq), ("k", kp, full[1], wk)):
        ref, mag = rope_ref(src[:, :, :d], w if norm else None, 1e-6, pos, inv, interleaved)
        if name == "k":
            got, whole = kp.cpu().transpose(1, 2).reshape(-1, kv, d), k0.transpose(1, 2).reshape(-1, kv, d).clone()
            ok = (slots >= 0) & (slots < pages * page)
            gone = torch.ones(pages * page, dtype=torch.bool)
            gone[slots[ok]] = False
            assert torch.equal(got[gone].view(torch.int16), whole[gone].view(torch.int16)), "a slot that was not named changed"
            got, ref, mag = got[slots[ok]], ref[ok], mag[ok]
        err = (got.cpu().double() - ref).abs()
        lim = half_step(got.dtype) * (ref.abs() + fp32 * mag) + fp32 * mag + torch.finfo(got.dtype).tiny
        assert bool((err <= lim).all()), (name, float((err - lim).max()))
    ok = (slots >= 0) & (slots < pages * page)
    gv = vp.cpu().transpose(1, 2).reshape(-1, kv, d)
    want = v0.transpose(1, 2).reshape(-1, kv, d).clone()
    want[slots[ok]] = full[2][ok][:, :, :d].to(ct)
    assert torch.equal(gv.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("d,rot", [(256, 64), (128, 128), (64, 32), (64, 8), (256, 256)])
def test_rope_shapes(d, rot, columns):
    for i, n in enumerate((1, 2, 5, 31, 33, 100)):
        run_rope(n, 3, 2, d, rot, 16, (F32, F16, BF16)[i % 3], (F16, BF16)[i % 2], columns, seed=i)


@pytest.mark.parametrize("d,rot", [(256, 64), (128, 16), (64, 64)])
def test_rope_interleaved(d, rot):
    run_rope(37, 2, 1, d, rot, 32, F32, BF16, False, interleaved=True)
    run_rope(37, 2, 1, d, rot, 32, BF16, F16, True, interleaved=True)


def test_rope_far_positions_and_plain_rows():
    run_rope(40, 24, 4, 256, 64, 64, F32, BF16, False, far=2 ** 31 - 1)
    run_rope(40, 4, 2, 128, 64, 64, F32, BF16, True, far=2 ** 31 - 1, norm=False)
    run_rope(3, 2, 2, 128, 0, 16, F32, F16, False, norm=False)
    run_rope(70, 2, 2, 128, 64, 1, F32, F16, False, odd=True)          # rows at any 4-byte place
    run_rope(70, 2, 2, 64, 64, 128, F32, F16, True, odd=True)


@pytest.mark.parametrize("d,rot", [(256, 64), (256, 256), (64, 64)])
def test_rope_every_tile(d, rot):
    """More tokens than 4 a workgroup pays for, and in columns than 16 (all of 256 rotated: 16 again)."""
    for columns, n in ((False, 65), (False, 301), (True, 65), (True, 512), (True, 513), (True, 547)):
        run_rope(n, 2, 1, d, rot, 64, BF16, F16, columns, seed=n)


def test_rope_slots_outside_are_not_written():
    pages, page = 4, 16
    slots = torch.tensor([-1, 3, 64, 2 ** 40, 63, -2 ** 40, 0, 17], dtype=torch.int64)
    run_rope(8, 2, 2, 128, 64, page, F16, F16, False, extra=pages - 1, slots=slots)
    run_rope(8, 2, 2, 128, 64, page, F16, F16, True, extra=pages - 1, slots=slots)


def test_rope_extreme_rows():
    """Zero rows (only eps is left), and large ones."""
    q = torch.zeros(3, 1, 128, device="cuda")
    q[1] = 1e15
    q[2] = 1e-20
    pages = torch.zeros(1, 1, 16, 128, dtype=BF16, device="cuda")
    out = torch.full((3, 1, 128), NAN, device="cuda")
    B.qk_norm_rope(q, q, q, None, None, 1e-6, ints([0, 1, 2]), B.rope_inv_freq(64, 1e4), ints([0, 1, -1], torch.int64),
                   pages, pages.clone(), out)
    ones = torch.ones(128, device="cuda")
    ref = torch.full((3, 1, 128), NAN, device="cuda")
    B.qk_norm_rope(q, q, q, ones, ones, 1e-6, ints([0, 0, 0]), None, ints([0, 1, -1], torch.int64), pages, pages.clone(), ref)
    assert bool((ref[0] == 0).all()) and bool(((ref[1] - 1).abs() < 1e-6).all()) and bool((ref[2].abs() < 1e-16).all())
    assert bool(torch.isfinite(out).all())


# ------------------------------------------------------------- attn_paged
def attn_ref(q, kp, vp, table, starts, kv_len, scale, out):
    """In 64 bits, token by token in the definition's order: (result, sum of p |v|, largest sum of |q| |k|)."""
    n, heads, d = q.shape
    n_pages, kvh, page, _ = kp.shape
    group = heads // kvh
    ref = out.double().clone()
    mag, top = torch.zeros(n, heads, d, dtype=torch.float64), torch.zeros(n, heads, 1, dtype=torch.float64)
    for s in range(len(kv_len)):
        a, b, kv = starts[s], starts[s + 1], min(kv_len[s], table.shape[1] * page)
        for t in range(a, b):
            seen = [j for j in range(max(0, min(kv, kv - (b - a) + (t - a) + 1)))
                    if 0 <= int(table[s, j // page]) < n_pages]
            if not seen:
                ref[t] = 0
                continue
            pg, off = table[s, [j // page for j in seen]].long(), torch.tensor([j % page for j in seen])
            for h in range(heads):
                k, v = kp[pg, h // group, off].double(), vp[pg, h // group, off].double()
                x = (k @ q[t, h].double()) * scale
                p = torch.softmax(x, 0)
                ref[t, h] = p @ v
                mag[t, h] = p @ v.abs()
                top[t, h] = (k.abs() @ q[t, h].double().abs()).max() * scale
    return ref, mag, top


def run_attn(new, kv, heads, kvh, d, page, t, io, seed=0, scale=None, work=True, max_kv=None, pad=0, table=None,
             edit=None, spread=1, check=True):
    case(f"attn new={new} kv={kv} heads={heads}/{kvh} d={d} page={page} {t} io={io} work={work} max_kv={max_kv} pad={pad}")
    g = gen(seed)
    starts = [pad]
    for x in new:
        starts.append(starts[-1] + x)
    n = starts[-1] + pad
    need = [-(-c // page) for c in kv]
    cols = max(max(need), 1)
    total = sum(need) + 2
    perm = torch.randperm(total, generator=g)
    if table is None:
        table = torch.full((len(kv), cols), -1, dtype=torch.int32)
        at = 0
        for i, c in enumerate(need):
            table[i, :c] = perm[at:at + c].int()
            at += c
    q = (torch.randn(n, heads, d, generator=g) * 1.3 * spread).to(io)
    kp, vp = (torch.randn(total, kvh, page, d, generator=g).to(t) for _ in range(2))
    # what lies behind the last key of a sequence is never read into a result
    for i, c in enumerate(kv):
        if c % page and need[i] <= table.shape[1]:
            p = int(table[i, c // page]) if c // page < table.shape[1] else -1
            if 0 <= p < total:
                kp[p, :, c % page:] = NAN
                vp[p, :, c % page:] = float("inf")
    if edit:
        edit(q, kp, vp, table)
    out = torch.full((n, heads, d), 7.0, dtype=io)
    scale = d ** -0.5 if scale is None else scale
    args = [q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), ints(starts), ints(kv), out.cuda()]
    mk = max(kv) if max_kv is None else max_kv
    ws = None
    if work:
        ws = torch.full((B.attn_paged_workspace_bytes(*args, max_kv=mk, scale=scale) + 16,), 255, dtype=torch.uint8, device="cuda")
    B.attn_paged(*args, ws, max_kv=mk, scale=scale)
    torch.cuda.synchronize()
    got = args[6].cpu()
    if not check:
        return got
    ref, mag, top = attn_ref(q, kp, vp, table, starts, kv, scale, out)
    check_attn(got, ref, mag, top, io, d, max(kv + [1]))
    return got


def check_attn(got, ref, mag, top, io, d, keys):
    assert torch.equal(torch.isfinite(got.double()), torch.isfinite(ref))
    fin = torch.isfinite(ref)
    # a score is a sum of d products, off by d + 2 roundings of its magnitudes (fp32 queries: and one of 2^-22 of
    # them); exp2 and its argument 8; P is rounded once to the pages' type (or 2^-22), the sums over keys add one
    # rounding a tile of 16 and one a part
    dx = (d + 8) * U * top
    p = half_step(io) if io != F32 else 2.0 ** -22
    lim = mag * (2 * dx + p + (keys / 16 + 24) * U)
    lim = lim + half_step(io) * (ref.abs() + lim) + torch.finfo(io).tiny
    err = (got.double() - ref).abs()
    bad = fin & ~(err <= lim)
    assert not bool(bad.any()), float((err - lim)[bad].max())
    # two roundings, each of them evenly spread: eps/2 sqrt(2/3) of the norm; fp32: 2^-18
    f = torch.where(fin, ref, 0.0)
    rel = normwise(torch.where(fin, got.double(), 0.0), f)
    assert rel <= (half_step(io) if io != F32 else 2.0 ** -18), rel


HEADS = [(6, 1, 256), (24, 4, 256), (4, 2, 128), (7, 1, 64), (3, 3, 64), (40, 1, 128)]


@pytest.mark.parametrize("heads,kvh,d", HEADS)
@pytest.mark.parametrize("t,io", [(BF16, BF16), (F16, F16), (F16, F32), (BF16, F32)])
def test_attn_decode(heads, kvh, d, t, io):
    run_attn([1], [1], heads, kvh, d, 16, t, io)
    run_attn([1, 1, 1], [33, 129, 700], heads, kvh, d, 16, t, io, seed=1)
    run_attn([1, 1], [300, 17], heads, kvh, d, 64, t, io, seed=2, work=False)


@pytest.mark.parametrize("heads,kvh,d", HEADS)
@pytest.mark.parametrize("t,io", [(BF16, BF16), (F16, F16), (F16, F32), (BF16, F32)])
def test_attn_chunks(heads, kvh, d, t, io):
    run_attn([64], [64], heads, kvh, d, 16, t, io)
    run_attn([75, 1, 0, 33], [75, 150, 40, 290], heads, kvh, d, 32, t, io, seed=1, pad=3)
    run_attn([50], [421], heads, kvh, d, 64, t, io, seed=2, work=False)


@pytest.mark.parametrize("io", [BF16, F32])
def test_attn_few_tokens(io):
    """Drafts: both shapes of workgroup, around the line between them."""
    for n in (2, 3, 5, 8, 10, 11, 12, 16, 22):
        run_attn([n], [n + 200], 6, 1, 128, 16, BF16, io, seed=n)
        run_attn([n, n + 1], [n, n + 130], 4, 4, 64, 16, BF16, io, seed=n)


@pytest.mark.parametrize("t,io", [(F16, F16), (BF16, F32), (F16, F32)])
def test_attn_few_tokens_of_a_long_context(t, io):
    """More rows than one tile of the decode shape, over as many workgroups as there are."""
    run_attn([8], [5000], 12, 2, 256, 64, t, io)
    run_attn([40], [1500], 8, 4, 64, 16, t, io, seed=1)
    run_attn([7, 9, 11], [900, 2000, 30], 6, 1, 128, 32, t, io, seed=2)


def test_attn_rows_without_keys():
    """More new tokens than keys: the first of them see nothing; no keys at all; no pages at all."""
    got = run_attn([5, 40], [2, 3], 4, 2, 128, 16, BF16, BF16)
    assert bool((got[:3] == 0).all()) and bool((got[5:42] == 0).all())
    got = run_attn([1, 1, 30], [0, 5, 0], 4, 2, 128, 16, F16, F32)
    assert bool((got[0] == 0).all()) and bool((got[2:] == 0).all())
    q = torch.ones(2, 2, 64, dtype=F16, device="cuda")
    pages = torch.zeros(0, 2, 16, 64, dtype=F16, device="cuda")
    out = torch.full_like(q, 3)
    B.attn_paged(q, pages, pages, torch.zeros(2, 0, dtype=torch.int32, device="cuda"), ints([0, 1, 2]), ints([4, 0]), out)
    assert bool((out == 0).all())


@pytest.mark.parametrize("new", [[1, 1], [60, 50]])
def test_attn_pages_that_are_no_pages(new):
    """Freed (-1) and wild entries hold no keys."""
    t = torch.tensor([[-1, 2, 10 ** 6, 3, 0], [1, -5, 2 ** 31 - 1, 4, -2 ** 31]], dtype=torch.int32)
    for io in (BF16, F32):
        run_attn(new, [80, 70], 6, 2, 128, 16, BF16, io, table=t)
        run_attn(new, [80, 70], 6, 2, 256, 16, BF16, io, table=t)
    t = torch.full((2, 5), -1, dtype=torch.int32)
    assert bool((run_attn(new, [80, 70], 6, 2, 128, 16, BF16, BF16, table=t) == 0).all())


def test_attn_lengths_beyond_the_table():
    """A kv_len past the last page of the table counts as the table's end; one below 0 as 0."""
    case("attn kv_len beyond the table")
    g = gen(5)
    pages = torch.randn(2, 2, 16, 64, generator=g).to(F16).cuda()
    table = ints([[1, 0]])
    for n in (1, 40):
        q = torch.randn(n, 4, 64, generator=g).to(F16).cuda()
        got = []
        for kv in (32, 33, 10 ** 6, 2 ** 31 - 1, 0, -1, -2 ** 31):
            out = torch.full_like(q, 5.0)
            B.attn_paged(q, pages, pages, table, ints([0, n]), ints([kv]), out, max_kv=32)
            got.append(out)
        assert all(torch.equal(x, got[0]) for x in got[1:4])
        assert all(bool((x == 0).all()) for x in got[4:])


@pytest.mark.parametrize("io", [BF16, F32])
@pytest.mark.parametrize("value", [NAN, float("inf"), -float("inf")])
def test_attn_what_is_not_seen_stays_out(io, value):
    """Keys and values of later tokens of the same chunk, whatever they hold."""
    for new, kv, heads, kvh, d in (([40], [40], 6, 1, 256), ([9], [50], 3, 1, 128), ([100, 30], [230, 30], 4, 1, 64)):
        def edit(q, k, v, table):
            for s, (n, c) in enumerate(zip(new, kv)):
                for j in (c - 1, c - n // 2):
                    v[int(table[s, j // 16]), :, j % 16] = value
                    k[int(table[s, j // 16]), :, j % 16] = value
        run_attn(new, kv, heads, kvh, d, 16, BF16, io, edit=edit)

        def values_only(q, k, v, table):
            for s, (n, c) in enumerate(zip(new, kv)):
                v[int(table[s, (c - 2) // 16]), :, (c - 2) % 16, 3] = value
        run_attn(new, kv, heads, kvh, d, 16, BF16, io, edit=values_only)


def test_attn_sharp_and_flat_rows():
    """Scores so large that one key has all the weight, and so small that all have the same."""
    for spread in (30.0, 1e-4):
        run_attn([1, 70], [900, 200], 4, 2, 128, 16, BF16, F32, spread=spread)
        run_attn([1, 70], [900, 200], 4, 2, 128, 16, F16, F16, spread=spread)
    run_attn([20], [100], 4, 2, 64, 16, F16, F32, spread=1e6, scale=1e-6)
    run_attn([20], [100], 4, 2, 64, 16, F16, F32, spread=1e-20, scale=1e18)


def test_attn_maximum_that_keeps_growing():
    """Later keys with larger scores: the running maximum moves at every tile, and jumps down never."""
    def edit(q, k, v, table):
        q[:] = 1.0
        for j in range(320):
            k[int(table[0, j // 16]), :, j % 16] = j / 60.0
    for io in (F16, F32):
        run_attn([1], [320], 4, 1, 64, 16, F16, io, edit=edit)
        run_attn([70], [320], 4, 1, 64, 16, F16, io, edit=edit)


def test_attn_strided_rows_and_pages():
    """Rows inside wider ones, and pages with room between them."""
    case("attn strides")
    g = gen(3)
    wide = torch.randn(40, 2, 4, 128, generator=g).to(BF16).cuda()
    store = torch.randn(6, 3, 2, 32, 128, generator=g).to(BF16).cuda()
    kp, vp = store[:, 0], store[:, 1]
    out = torch.full((40, 3, 4, 128), 5.0, dtype=BF16, device="cuda")
    table = ints([[3, 0, 5, -1], [1, 4, -1, -1]])
    for starts, kv in (([0, 1, 2], [90, 33]), ([0, 30, 40], [90, 33])):
        out.fill_(5.0)
        B.attn_paged(wide[:, 0], kp, vp, table, ints(starts), ints(kv), out[:, 1], max_kv=90)
        ref, mag, top = attn_ref(wide[:, 0].cpu(), kp.cpu(), vp.cpu(), table.cpu(), starts, kv, 128 ** -0.5, out[:, 1].cpu())
        check_attn(out[:, 1].cpu(), ref, mag, top, BF16, 128, 90)
        assert bool((out[:, 0] == 5).all()) and bool((out[:, 2] == 5).all()) and bool((out[starts[2]:] == 5).all())


def test_attn_any_hint_and_many_sequences():
    """max_kv places the work and nothing else; more sequences than lanes of a wave."""
    for mk in (0, 1, 128, 100000):
        run_attn([1, 1], [700, 130], 4, 2, 64, 16, F16, F16, max_kv=mk)
        run_attn([90], [700], 4, 2, 64, 16, F16, F16, max_kv=mk)
    run_attn([1] * 150, [(7 * i) % 61 for i in range(150)], 2, 1, 64, 16, F16, F16)
    run_attn([i % 4 for i in range(150)], [(7 * i) % 61 for i in range(150)], 2, 1, 64, 16, F16, F32)


@pytest.mark.parametrize("n_seq,new", [(1, 1), (2, 1), (1, 40)])
def test_attn_without_pages(n_seq, new):
    """No pages, or none that the table could name: nothing is seen, and table and pages may be NULL."""
    case(f"attn no pages {n_seq} {new}")
    n = n_seq * new
    for pages, cols in ((0, 3), (4, 0), (0, 0)):
        q, out = torch.ones(n, 4, 64, dtype=F16, device="cuda"), torch.ones(n, 4, 64, dtype=F16, device="cuda")
        kp = torch.zeros(pages, 2, 16, 64, dtype=F16, device="cuda")
        table = torch.zeros(n_seq, cols, dtype=torch.int32, device="cuda")
        args = B._attn_args(q, kp, kp, table, ints([i * new for i in range(n_seq + 1)]), ints([40] * n_seq), out, None, 40, None)
        a = B.AttnPagedArgs.from_buffer_copy(args)
        a.table = a.k_pages = a.v_pages = None
        assert B.lib().bonsai_p40_attn_paged(C.byref(a), B._stream(None)) == 0
        assert bool((out == 0).all())


def test_attn_pages_that_sequences_share():
    """A common prefix: the same pages in several rows of the table, and twice in one."""
    table = torch.tensor([[0, 1, 2], [0, 1, 3], [0, 0, 4]], dtype=torch.int32)
    for new in ([1, 1, 1], [40, 9, 33]):
        run_attn(new, [48, 41, 48], 4, 2, 64, 16, F16, F16, table=table)
        run_attn(new, [48, 41, 48], 4, 2, 64, 16, BF16, F32, table=table)


def test_attn_offsets_beyond_32_bits():
    """A page stride that puts pages more than 4 GiB apart."""
    case("attn pages beyond 4 GiB")
    g = gen(4)
    store = torch.empty(3, 1 << 30, dtype=F16, device="cuda")
    kp = store[:, :2 * 16 * 64].view(3, 2, 16, 64)
    vp = store[:, 4096:4096 + 2 * 16 * 64].view(3, 2, 16, 64)
    kp.copy_(torch.randn(3, 2, 16, 64, generator=g))
    vp.copy_(torch.randn(3, 2, 16, 64, generator=g))
    table = ints([[2, 0, 1]])
    for n in (1, 40):
        q = torch.randn(n, 4, 64, generator=g).to(F16).cuda()
        out = torch.zeros_like(q)
        B.attn_paged(q, kp, vp, table, ints([0, n]), ints([45]), out)
        ref, mag, top = attn_ref(q.cpu(), kp.cpu(), vp.cpu(), table.cpu(), [0, n], [45], 0.125, out.cpu())
        check_attn(out.cpu(), ref, mag, top, F16, 64, 45)


# -------------------------------------------------------------------- gdn
def gdn_ref(q, k, v, g, beta, state, starts, slots, scale, eps, tiled):
    q, k, v, g, beta = (x.double() for x in (q, k, v, g, beta))
    if eps > 0:
        q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + eps) for x in (q, k))
    vh, per = v.shape[1], v.shape[1] // q.shape[1]
    head = [h % q.shape[1] if tiled else h // per for h in range(vh)]
    out, final = {}, state.double().clone()
    for s in range(len(starts) - 1):
        i = slots[s] if slots is not None else s
        if not 0 <= i < state.shape[0]:
            continue
        S = final[i]
        for t in range(starts[s], starts[s + 1]):
            kk, qq = k[t, head], q[t, head]
            S = S * g[t].exp()[:, None, None]
            u = beta[t][:, None] * (v[t] - torch.einsum("hk,hkv->hv", kk, S))
            S = S + kk[:, :, None] * u[:, None]
            out[t] = torch.einsum("hk,hkv->hv", qq, S) * scale
        final[i] = S
    return out, final


def run_gdn(new, kh, vh, kd, vd, t, seed=0, eps=1e-6, tiled=True, work=True, max_new=None, pad=0, slots=None, states=None,
            in_place=False, gates=None, amp=1.0, tol=2.0 ** -18, scale=None):
    case(f"gdn new={new} heads={kh}/{vh} K={kd} V={vd} {t} eps={eps} tiled={tiled} work={work} max_new={max_new}")
    r = gen(seed)
    starts = [pad]
    for x in new:
        starts.append(starts[-1] + x)
    n = starts[-1] + pad
    x = torch.randn(n, (2 * kh + vh) * max(kd, vd), generator=r) * amp
    x = (x * torch.sigmoid(x)).to(t)
    row = x.cuda()
    k = row[:, kh * kd:2 * kh * kd].view(n, kh, kd)
    q = row[:, :kh * kd].view(n, kh, kd)
    v = row[:, 2 * kh * kd:2 * kh * kd + vh * vd].view(n, vh, vd)
    gg = -torch.rand(n, vh, generator=r) * 0.3 if gates is None else gates(n, vh, r)
    beta = torch.sigmoid(torch.randn(n, vh, generator=r))
    states = len(new) if states is None else states
    st = torch.randn(states, vh, kd, vd, generator=r) * 0.3
    sd = st.cuda()
    so = sd if in_place else torch.full_like(sd, 9.0)
    out = torch.full((n, vh, vd), 7.0, dtype=t, device="cuda")
    mn = max(new + [1]) if max_new is None else max_new
    kw = dict(max_new=mn, slots=ints(slots) if slots is not None else None, l2_eps=eps, tiled=tiled, scale=scale)
    args = (q, k, v, gg.cuda(), beta.cuda(), sd, so, out, ints(starts))
    ws = None
    if work:
        ws = torch.full((B.gdn_workspace_bytes(*args, **kw) + 16,), 255, dtype=torch.uint8, device="cuda")
    B.gdn(*args, ws, **kw)
    torch.cuda.synchronize()
    ref, final = gdn_ref(q.cpu(), k.cpu(), v.cpu(), gg, beta, st, starts, slots, kd ** -0.5 if scale is None else scale,
                         eps, tiled)
    got = out.cpu()
    quiet = [i for i in range(n) if i not in ref]
    assert bool((got[quiet] == 7).all()), "a row that belongs to no sequence changed"
    used = sorted(slots[s] if slots is not None else s for s in range(len(new)))
    used = [i for i in used if 0 <= i < states]
    rest = [i for i in range(states) if i not in used]
    assert torch.equal(so.cpu()[rest], (st if in_place else torch.full_like(st, 9.0))[rest])
    if used:
        assert normwise(so.cpu()[used], final[used]) <= tol, normwise(so.cpu()[used], final[used])
    if ref:
        order = sorted(ref)
        want = torch.stack([ref[i] for i in order])
        # fp32 sums, and the rounding of the store
        rel = normwise(got[order], want)
        assert rel <= tol + (half_step(t) if t != F32 else 0), rel
    return so, out


# five products in a row, each off by 2^-22 of its operands' norms or less, times what (I + L)^-1 adds: 2^-18
@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("kh,vh,kd,vd", [(2, 6, 128, 128), (3, 3, 64, 64), (1, 2, 128, 48), (2, 2, 64, 16)])
def test_gdn_shapes(kh, vh, kd, vd, t):
    run_gdn([1], kh, vh, kd, vd, t)
    run_gdn([1, 2, 0, 5], kh, vh, kd, vd, t, seed=1, tiled=False, pad=2)
    run_gdn([64], kh, vh, kd, vd, t, seed=2)
    run_gdn([17, 63, 65, 130, 1, 0], kh, vh, kd, vd, t, seed=3, pad=3, tiled=False)


@pytest.mark.parametrize("new", [1, 15, 16, 17, 33, 64, 127, 128, 129, 500])
def test_gdn_lengths_both_ways(new):
    a = run_gdn([new], 1, 2, 128, 64, F32, seed=new)
    b = run_gdn([new], 1, 2, 128, 64, F32, seed=new, work=False)
    assert normwise(a[0], b[0].double().cpu()) <= 2.0 ** -17


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("kh,vh,kd,vd", [(2, 6, 128, 128), (3, 9, 64, 48), (10, 10, 64, 16), (1, 2, 128, 144)])
def test_gdn_many_sequences(kh, vh, kd, vd, t):
    """More workgroups than CUs; key heads that are no multiple of 8; columns that end inside a workgroup's."""
    run_gdn([(11 * i) % 71 for i in range(45)], kh, vh, kd, vd, t, seed=7, pad=1)
    run_gdn([70], kh, vh, kd, vd, t, seed=8, tiled=False)


@pytest.mark.parametrize("n_seq", [2, 63, 64, 65])
def test_gdn_sequences_in_any_order(n_seq):
    """The longest go first, whatever their place: lengths up, down, alike and none, with a wave's lanes full and not."""
    up = [(i * 5) % 40 for i in range(n_seq - 1)] + [300]
    for new in (up, up[::-1], [20] * n_seq, [0] * (n_seq - 1) + [70]):
        run_gdn(new, 1, 2, 64, 16, F32, seed=n_seq)


@pytest.mark.parametrize("t", [F32, BF16])
def test_gdn_rows_of_out_at_any_element(t):
    case(f"gdn out strides {t}")
    n, r = 100, gen(5)
    q, k, v = (torch.randn(n, 2, 64, generator=r).to(t).cuda() for _ in range(3))
    g, beta = -torch.rand(n, 2, generator=r).cuda(), torch.rand(n, 2, generator=r).cuda()
    st = torch.randn(2, 2, 64, 64, generator=r).cuda()
    for starts in ([0, 1, 3], [0, 30, 99]):
        res = []
        for off, width in ((0, 128), (1, 131)):
            wide = torch.full((n * width + 8,), 5.0, dtype=t, device="cuda")
            out = wide[off:off + n * width].view(n, width)[:, :128].unflatten(1, (2, 64))
            args = (q, k, v, g, beta, st, torch.empty_like(st), out, ints(starts))
            ws = torch.empty(B.gdn_workspace_bytes(*args, l2_eps=1e-6) + 16, dtype=torch.uint8, device="cuda")
            B.gdn(*args, ws, l2_eps=1e-6)
            res.append(out.clone())
            assert bool((wide[off:off + n * width].view(n, width)[:, 128:] == 5).all()) and bool((wide[n * width + off:] == 5).all())
        assert torch.equal(*res) and bool((res[0][starts[-1]:] == 5).all())


def test_gdn_slots():
    for new in ([1, 2, 3], [40, 70, 1]):
        run_gdn(new, 1, 2, 64, 64, F32, slots=[4, 0, 2], states=6)
        run_gdn(new, 1, 2, 64, 64, F32, slots=[4, -1, 6], states=6, in_place=True)
        run_gdn(new, 1, 2, 64, 64, F32, states=2)          # the third has no state


def test_gdn_hints():
    for mn in (0, 1, 10, 1000):
        run_gdn([3, 90], 2, 2, 64, 64, F32, max_new=mn)


@pytest.mark.parametrize("new", [[5], [150]])
def test_gdn_gates_and_scales(new):
    """No decay, decay to nothing (also at once), growth; rows far from 1 without the L2 norm."""
    run_gdn(new, 1, 2, 64, 64, F32, gates=lambda n, h, r: torch.zeros(n, h))
    run_gdn(new, 1, 2, 64, 64, F32, gates=lambda n, h, r: torch.full((n, h), -30.0))
    run_gdn(new, 1, 2, 64, 64, F32, gates=lambda n, h, r: torch.where(torch.rand(n, h, generator=r) < 0.1, -float("inf"), -0.02))
    run_gdn(new, 1, 2, 64, 64, F32, gates=lambda n, h, r: torch.where(torch.rand(n, h, generator=r) < 0.1, -300.0, -1e-3))
    run_gdn(new, 1, 2, 64, 64, F32, gates=lambda n, h, r: torch.full((n, h), 0.01))
    run_gdn(new, 1, 2, 64, 64, F32, eps=0.0, amp=0.1)
    run_gdn(new, 1, 2, 128, 64, F32, eps=1e-6, amp=1e4)
    run_gdn(new, 1, 2, 128, 64, F32, eps=1e-30, amp=1e-6, scale=3.0)


def test_gdn_keys_that_repeat():
    """The same key at every token, beta near 1: the state's row is replaced each time."""
    case("gdn repeated keys")
    n = 130
    k = torch.randn(1, 1, 64, generator=gen(1)).expand(n, 1, 64).contiguous()
    q, v = torch.randn(n, 1, 64, generator=gen(2)), torch.randn(n, 1, 64, generator=gen(3))
    g, beta = torch.zeros(n, 1), torch.full((n, 1), 0.999)
    st = torch.randn(1, 1, 64, 64, generator=gen(4))
    out, so = torch.zeros(n, 1, 64, device="cuda"), torch.zeros(1, 1, 64, 64, device="cuda")
    args = (q.cuda(), k.cuda(), v.cuda(), g.cuda(), beta.cuda(), st.cuda(), so, out, ints([0, n]))
    ws = torch.empty(B.gdn_workspace_bytes(*args, l2_eps=1e-6) + 16, dtype=torch.uint8, device="cuda")
    B.gdn(*args, ws, l2_eps=1e-6)
    ref, final = gdn_ref(q, k, v, g, beta, st, [0, n], None, 0.125, 1e-6, False)
    assert normwise(so.cpu(), final) <= 2.0 ** -17
    assert normwise(out.cpu(), torch.stack([ref[i] for i in range(n)])) <= 2.0 ** -17


def test_gdn_in_place_equals_apart():
    for new in ([3], [100, 20]):
        a = run_gdn(new, 2, 4, 64, 64, BF16, in_place=True)
        b = run_gdn(new, 2, 4, 64, 64, BF16)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
