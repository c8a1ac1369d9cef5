"""8-bit pages of a cache (written by qk_norm_rope, read by attn_paged and back by
kv_read) against plain implementations in 64 bits, at the sizes and masks where
they can go wrong.

Tolerances count roundings: U = 2^-24 is one of fp32, finfo(t).eps / 2 a store to t."""
import ctypes as C

import pytest

import bonsai_p40 as B
from test_gpu_mixers import BF16, F16, F32, NAN, U, attn_ref, case, gen, half_step, ints, normwise, rope_ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")


def quantised(x):
    """The header's formula for rows, in fp32: (numbers, scales)."""
    top = x.abs().amax(-1)
    fine = torch.isfinite(x).all(-1)
    some = fine & (top >= 2.0 ** -112)
    r = torch.full_like(top, 127.0) / top                       # (127 / top would be 127 times a rounded 1 / top)
    n = torch.round(x * torch.where(some, r, 0.0)[..., None])
    d = torch.where(some, top / 127, torch.where(fine, 0.0, NAN))
    return torch.where(some[..., None], n, 0.0).to(torch.int8), d


def pages_of(codes, scales):
    """CPU numbers and scales as 8-bit pages on the device."""
    c, s = B.q8_pages(*codes.shape)
    c.copy_(codes)
    s.copy_(scales)
    return c, s


# ------------------------------------------------------------------ append
def run_append(n, heads, kv, d, rot, page, qt, columns, interleaved=False, norm=True, seed=0, slots=None, edit=None):
    case(f"q8 append n={n} heads={heads}/{kv} d={d} rot={rot} page={page} {qt} columns={columns} il={interleaved}")
    g = gen(seed)
    full = [torch.randn(n, h, w, generator=g) * 2 for h, w in ((heads, d), (kv, d), (kv, d))]
    if edit:
        edit(*full)
    q, k, v = (t.cuda().permute(1, 2, 0).contiguous().permute(2, 0, 1) if columns else t.cuda() for t in full)
    wq, wk = (torch.randn(d, generator=g) * 0.2 + 1 for _ in range(2))
    inv = 1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    pos = torch.randint(0, 5000, (n,), generator=g, dtype=torch.int32)
    pages = -(-n // page) + 2
    if slots is None:
        slots = torch.randperm(pages * page, generator=g)[:n]
    before = torch.randint(-127, 128, (pages, kv, page, d), generator=g, dtype=torch.int8), torch.rand(pages, kv, page, generator=g)
    (kc, ks), (vc, vs) = pages_of(*before), pages_of(*before)
    qo = torch.full((n, heads, d), NAN, dtype=qt, device="cuda")
    B.qk_norm_rope(q, k, v, wq.cuda() if norm else None, wk.cuda() if norm else None, 1e-6, pos.cuda(), inv.cuda(),
                   slots.cuda(), kc, vc, qo, interleaved)
    torch.cuda.synchronize()
    rows = [t.cpu().transpose(1, 2).reshape(pages * page, kv, -1) for t in (kc, ks[..., None], vc, vs[..., None])]
    ok = (slots >= 0) & (slots < pages * page)
    gone = torch.ones(pages * page, dtype=torch.bool)
    gone[slots[ok]] = False
    old = [t.transpose(1, 2).reshape(pages * page, kv, -1) for t in (before[0], before[1][..., None])]
    for got, want in zip(rows, old * 2):
        assert torch.equal(got[gone], want[gone]), "a slot that was not named changed"
    kn, kd, vn, vd = (t[slots[ok]] for t in rows)
    # values: the formula's bytes
    n_ref, d_ref = quantised(full[2][ok])
    assert torch.equal(vn, n_ref) and torch.equal(vd[..., 0].view(torch.int32)[~d_ref.isnan()], d_ref.view(torch.int32)[~d_ref.isnan()])
    assert torch.equal(vd[..., 0].isnan(), d_ref.isnan())
    # keys: 24 roundings of fp32 before them, then half a step and 0.00002 of one
    ref, mag = rope_ref(full[1], wk if norm else None, 1e-6, pos, inv, interleaved)
    ref, mag, fp32 = ref[ok], mag[ok], 24 * U
    fine = torch.isfinite(ref).all(-1)
    top = ref.abs().amax(-1)
    assert torch.equal(kd[..., 0].isnan(), ~fine)
    err = (kd.double() * kn.double() - ref).abs()[fine]
    lim = (0.50002 * kd.double() + fp32 * mag.amax(-1, keepdim=True))[fine] + 2.0 ** -112
    assert bool((err <= lim).all()), float((err - lim).max())
    off = (kd[..., 0].double() * 127 - top).abs()[fine]
    assert bool((off <= ((fp32 + 2 * U) * mag.amax(-1))[fine] + 2.0 ** -112).all())
    assert bool((kn.abs().amax(-1)[fine & (top > 1e-30)] == 127).all())
    # queries: as with 16-bit pages
    ref, mag = rope_ref(full[0], wq if norm else None, 1e-6, pos, inv, interleaved)
    fine = torch.isfinite(ref).all(-1)
    err = (qo.cpu().double() - ref).abs()[fine]
    lim = (half_step(qt) * (ref.abs() + fp32 * mag) + fp32 * mag + torch.finfo(qt).tiny)[fine]
    assert bool((err <= lim).all())


@pytest.mark.parametrize("columns", [False, True])
@pytest.mark.parametrize("d,rot", [(256, 64), (128, 128), (64, 32)])
def test_append_shapes(d, rot, columns):
    for i, n in enumerate((1, 2, 5, 31, 33, 70, 130, 530)):
        run_append(n, 3, 2, d, rot, (16, 1, 64)[i % 3], (F32, F16, BF16)[i % 3], columns, seed=i)


def test_append_interleaved_and_plain_rows():
    run_append(37, 2, 1, 256, 64, 32, F32, False, interleaved=True)
    run_append(37, 2, 3, 64, 64, 32, BF16, True, interleaved=True)
    run_append(40, 1, 5, 128, 64, 16, F32, False, norm=False)
    run_append(9, 2, 2, 128, 0, 16, F16, False, norm=False)


def test_append_slots_outside_are_not_written():
    slots = torch.tensor([5, -1, 200, 63, 64, -2 ** 62, 2 ** 62, 0])
    run_append(8, 2, 2, 64, 32, 16, F32, False, slots=slots)


@pytest.mark.parametrize("d", [64, 256])
def test_append_rows_of_nothing_and_of_anything(d):
    """Zeros, the smallest and the largest numbers, one element far above the rest, ties, infinities and NaN."""
    def edit(q, k, v):
        k[0], v[0] = 0.0, 0.0
        v[1], v[2], v[3] = 1e-40, 2.0 ** -112, 2.0 ** -113
        v[4] = torch.finfo(F32).max
        v[5] = -torch.finfo(F32).max
        v[6] = 1e-6
        v[6, :, 7] = 100.0
        v[7] = torch.arange(d) % 127 + 0.5
        v[7, :, 0] = 127.0
        for row, value in ((8, NAN), (9, INF), (10, -INF)):
            k[row, 1, d - 1] = v[row, 0, 3] = value
    run_append(12, 2, 2, d, 32, 16, F32, False, edit=edit)
    run_append(12, 2, 2, d, 0, 16, F32, False, norm=False, edit=edit)


# -------------------------------------------------------------------- read
@pytest.mark.parametrize("kind", ["q8", F16, BF16])
@pytest.mark.parametrize("out", [F32, F16, BF16])
@pytest.mark.parametrize("kv,d,page", [(4, 256, 16), (3, 128, 64), (1, 64, 1)])
def test_read_back(kind, out, kv, d, page):
    """Any slots, twice, in any order; those outside leave their rows; rows inside wider ones."""
    for n in (1, 3, 17, 64, 257):
        case(f"read {kind} -> {out} n={n} kv={kv} d={d} page={page}")
        g = gen(n)
        pages = 300 // page + 1
        x = torch.randn(2, pages, kv, page, d, generator=g) * 3
        if kind == "q8":
            codes = torch.randint(-128, 128, x.shape, generator=g, dtype=torch.int8)
            scales = torch.rand(x.shape[:-1], generator=g) * 10 ** torch.randint(-3, 3, x.shape[:-1], generator=g).float()
            scales[:, 0, 0, 0] = NAN
            dev = [pages_of(c, s)[0] for c, s in zip(codes, scales)]
            x = codes.float() * scales[..., None]
        else:
            x = x.to(kind)
            dev = [t.cuda() for t in x]
        slots = torch.randint(0, pages * page, (n,), generator=g)
        slots[n // 2] = slots[0]
        if n > 3:
            slots[1], slots[2], slots[3] = -1, pages * page, 2 ** 62
        wide = torch.full((2, n, kv + 1, d), 7.0, dtype=out, device="cuda")
        got = wide[:, :, :kv]
        B.kv_read(*dev, slots.cuda(), got[0], got[1])
        torch.cuda.synchronize()
        ok = (slots >= 0) & (slots < pages * page)
        want = torch.full((2, n, kv + 1, d), 7.0, dtype=out)
        for i in range(2):
            want[i, ok, :kv] = x[i].transpose(1, 2).reshape(pages * page, kv, d)[slots[ok]].to(out)
        assert torch.equal(wide.cpu().isnan(), want.isnan())
        assert torch.equal(wide.cpu().nan_to_num(0.0), want.nan_to_num(0.0))


def test_read_pages_far_apart():
    """Slots past 2^32 elements, and a page stride of more than 4 GiB."""
    case("read beyond 32 bits")
    big = torch.zeros((5 << 30) + 16384, dtype=torch.int8, device="cuda")
    stride, (kv, page, d) = 5 << 30, (1, 16, 64)
    rows = torch.randint(-127, 128, (2, 16, 64), generator=gen(1), dtype=torch.int8)
    scales = torch.rand(2, 16, generator=gen(2))
    for p in range(2):
        at = p * stride
        big[at:at + 1024] = rows[p].flatten().cuda()
        big[at + 1024:at + 1088].view(F32).copy_(scales[p])
    slots = torch.tensor([0, 17, 31, 5], device="cuda")
    out = torch.zeros(2, 4, 1, 64, device="cuda")
    a = B.KvReadArgs(k_pages=big.data_ptr(), v_pages=big.data_ptr(), n_pages=2, page_stride=stride, page_size=page, n_kv_head=kv,
                     head_dim=d, kv_type=B.Q8, slots=slots.data_ptr(), n_tok=4, k_out=out[0].data_ptr(), v_out=out[1].data_ptr(),
                     k_tok=64, v_tok=64, out_type=B.F32)
    assert B.lib().bonsai_p40_kv_read(C.byref(a), B._stream(None)) == 0
    want = (rows.float() * scales[..., None]).reshape(32, 64)[slots.cpu()]
    assert torch.equal(out[0, :, 0].cpu(), want) and torch.equal(out[1, :, 0].cpu(), want)


# --------------------------------------------------------------- attention
def check_q8(got, ref, mag, top, q, keys_abs, scale, io, keys, wmax=None):
    """keys_abs: the largest sum of a key's magnitudes.  A score is off by what its query's elements are (1.01 x 2^-15
    of the row's largest, fp32 1.6 x 2^-23) and by 16 roundings; a weight is rounded once to f16 (fp32: to 22 bits),
    or is off by 2^-36 (2^-47) of the largest; the sums over keys add a rounding a tile of 16 and one a part."""
    assert torch.equal(torch.isfinite(got.double()), torch.isfinite(ref))
    fin = torch.isfinite(ref)
    e = 1.01 * 2.0 ** -15 if io != F32 else 1.6 * 2.0 ** -23
    dx = e * q.double().abs().amax(-1, keepdim=True) * keys_abs * scale + 16 * U * top
    p = 2.0 ** -11 if io != F32 else 2.0 ** -22
    floor = keys * (2.0 ** -36 if io != F32 else 2.0 ** -47) * mag.abs().amax(-1, keepdim=True) * 4
    lim = mag * (2 * dx + p + (keys / 16 + 24) * U) + floor
    lim = lim + half_step(io) * (ref.abs() + lim) + torch.finfo(io).tiny
    err = (got.double() - ref).abs()
    bad = fin & ~(err <= lim)
    assert not bool(bad.any()), float((err - lim)[bad].max())
    f = torch.where(fin, ref, 0.0)
    rel = normwise(torch.where(fin, got.double(), 0.0), f)
    assert rel <= (half_step(io) if io != F32 else 2.0 ** -18), rel


def run_q8(new, kv, heads, kvh, d, page, io, seed=0, scale=None, work=True, max_kv=None, pad=0, table=None, edit=None, spread=1,
           check=True):
    case(f"q8 attn new={new} kv={kv} heads={heads}/{kvh} d={d} page={page} io={io} work={work} max_kv={max_kv} pad={pad}")
    g = gen(seed)
    starts = [pad]
    for x in new:
        starts.append(starts[-1] + x)
    n = starts[-1] + pad
    need = [-(-c // page) for c in kv]
    total = sum(need) + 2
    perm = torch.randperm(total, generator=g)
    if table is None:
        table = torch.full((len(kv), max(max(need), 1)), -1, dtype=torch.int32)
        at = 0
        for i, c in enumerate(need):
            table[i, :c] = perm[at:at + c].int()
            at += c
    q = (torch.randn(n, heads, d, generator=g) * 1.3 * spread).to(io)
    kc, ks = quantised(torch.randn(total, kvh, page, d, generator=g))
    vc, vs = quantised(torch.randn(total, kvh, page, d, generator=g) * torch.exp(torch.randn(total, kvh, page, 1, generator=g)))
    if edit:
        edit(q, kc, ks, vc, vs, table)
    kp, vp = kc.double() * ks.double()[..., None], vc.double() * vs.double()[..., None]
    # what lies behind the last key of a sequence is never read into a result
    for i, c in enumerate(kv):
        if c % page and c // page < table.shape[1] and 0 <= int(table[i, c // page]) < total:
            ks[int(table[i, c // page]), :, c % page:] = NAN
            vs[int(table[i, c // page]), :, c % page:] = INF
    out = torch.full((n, heads, d), 7.0, dtype=io)
    scale = d ** -0.5 if scale is None else scale
    args = [q.cuda(), pages_of(kc, ks)[0], pages_of(vc, vs)[0], table.cuda(), ints(starts), ints(kv), out.cuda()]
    mk = max(kv) if max_kv is None else max_kv
    ws = None
    if work:
        ws = torch.full((B.attn_paged_workspace_bytes(*args, max_kv=mk, scale=scale) + 16,), 255, dtype=torch.uint8, device="cuda")
    B.attn_paged(*args, ws, max_kv=mk, scale=scale)
    torch.cuda.synchronize()
    got = args[6].cpu()
    if check:
        ref, mag, top = attn_ref(q, kp, vp, table, starts, kv, scale, out)
        check_q8(got, ref, mag, top, q, float(kp.abs().sum(-1).nan_to_num(0, 0, 0).max()), scale, io, max(kv + [1]))
    return got


HEADS = [(6, 1, 256), (24, 4, 256), (4, 2, 128), (7, 1, 64), (3, 3, 64), (40, 1, 128)]


@pytest.mark.parametrize("heads,kvh,d", HEADS)
@pytest.mark.parametrize("io", [BF16, F16, F32])
def test_decode(heads, kvh, d, io):
    run_q8([1], [1], heads, kvh, d, 16, io)
    run_q8([1, 1, 1], [33, 129, 700], heads, kvh, d, 16, io, seed=1)
    run_q8([1, 1], [300, 17], heads, kvh, d, 64, io, seed=2, work=False)


@pytest.mark.parametrize("heads,kvh,d", HEADS)
@pytest.mark.parametrize("io", [BF16, F16, F32])
def test_chunks(heads, kvh, d, io):
    run_q8([64], [64], heads, kvh, d, 16, io)
    run_q8([75, 1, 0, 33], [75, 150, 40, 290], heads, kvh, d, 32, io, seed=1, pad=3)
    run_q8([50], [421], heads, kvh, d, 64, io, seed=2, work=False)


@pytest.mark.parametrize("io", [BF16, F32])
def test_few_tokens(io):
    for n in (2, 3, 5, 8, 10, 11, 12, 16, 22):
        run_q8([n], [n + 200], 6, 1, 128, 16, io, seed=n)
        run_q8([n, n + 1], [n, n + 130], 4, 4, 64, 16, io, seed=n)
    run_q8([8], [3000], 12, 2, 256, 64, io)


def test_rows_without_keys():
    got = run_q8([5, 40], [2, 3], 4, 2, 128, 16, BF16)
    assert bool((got[:3] == 0).all()) and bool((got[5:42] == 0).all())
    got = run_q8([1, 1, 30], [0, 5, 0], 4, 2, 128, 16, F32)
    assert bool((got[0] == 0).all()) and bool((got[2:] == 0).all())


@pytest.mark.parametrize("new", [[1, 1], [60, 50]])
def test_pages_that_are_no_pages(new):
    t = torch.tensor([[-1, 2, 10 ** 6, 3, 0], [1, -5, 2 ** 31 - 1, 4, -2 ** 31]], dtype=torch.int32)
    for io in (BF16, F32):
        run_q8(new, [80, 70], 6, 2, 128, 16, io, table=t)
        run_q8(new, [80, 70], 6, 2, 256, 16, io, table=t)
    t = torch.full((2, 5), -1, dtype=torch.int32)
    assert bool((run_q8(new, [80, 70], 6, 2, 128, 16, BF16, table=t) == 0).all())


@pytest.mark.parametrize("io", [BF16, F32])
def test_rows_of_nan_reach_those_that_see_them(io):
    """A key or value whose d is NaN makes the tokens NaN that see it, and no others."""
    for new, kv, heads, kvh, d in (([40], [40], 6, 1, 256), ([9], [50], 3, 1, 128), ([100, 30], [230, 30], 4, 1, 64), ([1], [300], 6, 1, 256)):
        for which in (0, 1):
            def edit(q, kc, ks, vc, vs, table):
                for s, (n, c) in enumerate(zip(new, kv)):
                    j = c - 1 - n // 2
                    (ks, vs)[which][int(table[s, j // 16]), :, j % 16] = NAN
            run_q8(new, kv, heads, kvh, d, 16, io, edit=edit)


@pytest.mark.parametrize("io", [BF16, F16, F32])
def test_queries_that_are_not_finite(io):
    """Their rows are NaN, the others are not touched (but for last bits: the rows of a wave are rescaled together)."""
    for new, kv in (([1, 1, 1], [40, 300, 9]), ([50], [200])):
        def edit(q, *rest):
            q[0, 1, 5], q[2, 0, 63] = NAN, INF
        got = run_q8(new, kv, 4, 2, 64, 16, io, edit=edit, check=False)
        plain = run_q8(new, kv, 4, 2, 64, 16, io)
        bad = torch.zeros(got.shape[:2], dtype=torch.bool)
        bad[0, 1] = bad[2, 0] = True
        assert bool(got[bad].isnan().all())
        # both are within the norm's limit of the exact result
        assert normwise(got[~bad], plain[~bad].double()) <= 2 * (half_step(io) if io != F32 else 2.0 ** -18)


def test_numbers_of_all_values():
    """-128 is read as it stands; scales may be 0 or below it."""
    def edit(q, kc, ks, vc, vs, table):
        kc[:] = torch.randint(-128, 128, kc.shape, generator=gen(3), dtype=torch.int8)
        vc[:] = torch.randint(-128, 128, vc.shape, generator=gen(4), dtype=torch.int8)
        kc[..., 0], vc[..., 1] = -128, -128
        vs[0], ks[1] = 0.0, 0.0
        vs[:, :, ::3] *= -1
    for io in (F16, F32):
        run_q8([1, 1], [90, 300], 4, 2, 128, 16, io, edit=edit)
        run_q8([60], [300], 4, 2, 256, 16, io, edit=edit)


@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("d", [64, 256])
def test_scales_far_apart(io, d):
    """Values whose scales grow or fall from key to key by many powers of two, so that each row's result is made by
    the few largest it sees; and all of them small, and all large.  Tokens before a large one are not touched by it."""
    for new, kv in (([1], [300]), ([70], [200]), ([40], [40])):
        for low, high in ((-60, 60), (60, -60), (-110, -100), (70, 78)):
            def edit(q, kc, ks, vc, vs, table):
                for j in range(kv[0]):
                    vs[int(table[0, j // 16]), :, j % 16] = 2.0 ** round(low + (high - low) * j / kv[0])
            got = run_q8(new, kv, 2, 1, d, 16, io, edit=edit, check=io == F32)
            assert got.shape[0] == new[0]


def attend(q, k, v, io, work=True, page=16):
    """attn_paged of the last tokens of one sequence over quantised rows; (result, the same in 64 bits)."""
    n, heads, d = q.shape
    kv, kvh, _ = k.shape
    pages = -(-kv // page)
    q, perm = q.to(io), torch.randperm(pages, generator=gen(9))
    dev, val = [], []
    for x in (k, v):
        c, s = quantised(x)
        val.append(c.double() * s.double()[..., None])
        full, sc = torch.zeros(pages * page, kvh, d, dtype=torch.int8), torch.zeros(pages * page, kvh)
        full[:kv], sc[:kv] = c, s
        store, scs = torch.empty(pages, kvh, page, d, dtype=torch.int8), torch.empty(pages, kvh, page)
        store[perm], scs[perm] = full.view(pages, page, kvh, d).transpose(1, 2), sc.view(pages, page, kvh).transpose(1, 2)
        dev.append(pages_of(store, scs)[0])
    out = torch.full((n, heads, d), 7.0, dtype=io, device="cuda")
    args = [q.cuda(), *dev, perm.int().cuda()[None], ints([0, n]), ints([kv]), out]
    ws = torch.full((B.attn_paged_workspace_bytes(*args, max_kv=kv) + 16,), 255, dtype=torch.uint8, device="cuda") if work else None
    B.attn_paged(*args, ws, max_kv=kv)
    torch.cuda.synchronize()
    ref = torch.empty(n, heads, d, dtype=torch.float64)
    late = torch.arange(kv)[None] > (kv - n + torch.arange(n))[:, None]
    for h in range(heads):
        x = (q[:, h].double() @ val[0][:, h // (heads // kvh)].t()) * d ** -0.5
        ref[:, h] = torch.softmax(x.masked_fill(late, -INF), -1) @ val[1][:, h // (heads // kvh)]
    return out.cpu(), ref


@pytest.mark.parametrize("n,kv,heads,kvh,d", [(1, 4000, 6, 1, 256), (1, 3000, 4, 2, 128), (40, 1500, 6, 1, 256), (70, 900, 4, 2, 64)])
@pytest.mark.parametrize("io", [F32, F16, BF16])
@pytest.mark.parametrize("gap", [10, 18])
def test_a_key_that_has_nearly_all_the_weight(n, kv, heads, kvh, d, io, gap):
    """One key's score is `gap` above thousands of others, and its value is 0 or small: the result is what the others
    make of it.  The one key is off by half a step of 8 bits as all are, but its row stands for what it stands for;
    scores are whole numbers' sums, rounded 4 times, an exponent's argument of up to gap log2(e) twice; q is off by
    1.01 x 2^-15 (1.6 x 2^-23) of its largest element, 4, and so the gap by that share of itself; results below f16's
    smallest normal number are off by up to 2^-25."""
    case(f"q8 sink n={n} kv={kv} heads={heads}/{kvh} d={d} io={io} gap={gap}")
    g = gen(gap + n)
    q, k, v = torch.randn(n, heads, d, generator=g), torch.randn(kv, kvh, d, generator=g) * 0.5, torch.randn(kv, kvh, d, generator=g)
    q.clamp_(-3.5, 3.5)
    q[..., 0] = 4.0
    k[..., 0] = 0.0
    k[0] = 0.0
    k[0, :, 0] = round(gap * d ** 0.5 / 4)
    for value, work in ((0.0, True), (0.0, False), (2.0 ** -12, True)):
        v[0] = value
        got, ref = attend(q, k, v, io, work)
        store = 2.0 ** -25 * ref.numel() ** 0.5 / float(ref.norm()) if io == F16 else 0.0
        e = 1.6 * 2.0 ** -23 if io == F32 else 1.01 * 2.0 ** -15
        err, limit = normwise(got, ref), (2.0 ** -18 if io == F32 else half_step(io)) + 6 * gap * 1.4427 * U + 2 * gap * e + store
        print(f"value {value}: {err:.2e} of {limit:.2e}", flush=True)
        assert err <= limit


def test_sharp_flat_and_growing_rows():
    for spread in (30.0, 1e-4):
        run_q8([1, 70], [900, 200], 4, 2, 128, 16, F32, spread=spread)
        run_q8([1, 70], [900, 200], 4, 2, 64, 16, F32, spread=spread)
    run_q8([20], [100], 4, 2, 64, 16, F32, spread=1e6, scale=1e-6)
    run_q8([20], [100], 4, 2, 64, 16, F32, spread=1e-20, scale=1e18)

    def edit(q, kc, ks, vc, vs, table):
        q[:] = 1.0
        for j in range(320):
            kc[int(table[0, j // 16]), :, j % 16] = 100
            ks[int(table[0, j // 16]), :, j % 16] = j / 6000.0
    for io in (F16, F32):
        run_q8([1], [320], 4, 1, 64, 16, io, edit=edit)
        run_q8([70], [320], 4, 1, 64, 16, io, edit=edit)


def test_any_hint_many_sequences_and_lengths_beyond_the_table():
    for mk in (0, 1, 128, 100000):
        run_q8([1, 1], [700, 130], 4, 2, 64, 16, F16, max_kv=mk)
        run_q8([90], [700], 4, 2, 64, 16, F16, max_kv=mk)
    run_q8([1] * 150, [(7 * i) % 61 for i in range(150)], 2, 1, 64, 16, F16)
    run_q8([i % 4 for i in range(150)], [(7 * i) % 61 for i in range(150)], 2, 1, 64, 16, F32)
    case("q8 kv_len beyond the table")
    pages = pages_of(*quantised(torch.randn(2, 2, 16, 64, generator=gen(5))))[0]
    for n in (1, 40):
        q = torch.randn(n, 4, 64, generator=gen(6)).to(F16).cuda()
        got = []
        for kv in (32, 33, 10 ** 6, 2 ** 31 - 1, 0, -1, -2 ** 31):
            out = torch.full_like(q, 5.0)
            B.attn_paged(q, pages, pages, ints([[1, 0]]), ints([0, n]), ints([kv]), out, max_kv=32)
            got.append(out)
        assert all(torch.equal(x, got[0]) for x in got[1:4]) and all(bool((x == 0).all()) for x in got[4:])


def test_strided_rows_and_other_streams():
    """Rows inside wider ones; the same bytes on another stream and on a second call."""
    case("q8 strides")
    g = gen(3)
    wide = torch.randn(40, 2, 4, 128, generator=g).to(BF16).cuda()
    kc, ks = quantised(torch.randn(6, 2, 32, 128, generator=g))
    vc, vs = quantised(torch.randn(6, 2, 32, 128, generator=g))
    kp, vp = pages_of(kc, ks)[0], pages_of(vc, vs)[0]
    table = ints([[3, 0, 5, -1], [1, 4, -1, -1]])
    kd, vd = kc.double() * ks.double()[..., None], vc.double() * vs.double()[..., None]
    side = torch.cuda.Stream()
    for starts, kv in (([0, 1, 2], [90, 33]), ([0, 30, 40], [90, 33])):
        out = torch.full((40, 3, 4, 128), 5.0, dtype=BF16, device="cuda")
        args = (wide[:, 0], kp, vp, table, ints(starts), ints(kv))
        B.attn_paged(*args, out[:, 1], max_kv=90)
        ref, mag, top = attn_ref(wide[:, 0].cpu(), kd, vd, table.cpu(), starts, kv, 128 ** -0.5, out[:, 1].cpu())
        check_q8(out[:, 1].cpu(), ref, mag, top, wide[:, 0].cpu(), float(kd.abs().sum(-1).max()), 128 ** -0.5, BF16, 90)
        assert bool((out[:, 0] == 5).all()) and bool((out[:, 2] == 5).all()) and bool((out[starts[2]:] == 5).all())
        torch.cuda.synchronize()
        again = torch.full_like(out, 5.0)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            B.attn_paged(*args, again[:, 1], max_kv=90)
        torch.cuda.synchronize()
        assert torch.equal(again, out)


def test_pages_far_apart():
    """A page stride of more than 4 GiB."""
    case("q8 attention beyond 32 bits")
    big = torch.zeros((5 << 30) + 16384, dtype=torch.int8, device="cuda")
    stride, d = 5 << 30, 64
    kc, ks = quantised(torch.randn(2, 1, 16, d, generator=gen(1)))
    for p in range(2):
        big[p * stride:p * stride + 1024] = kc[p].flatten().cuda()
        big[p * stride + 1024:p * stride + 1088].view(F32).copy_(ks[p, 0])
    table, kd = ints([[1, 0]]), kc.double() * ks.double()[..., None]
    for n in (1, 30):
        q = torch.randn(n, 40 // (1 if n > 1 else 10), d, generator=gen(n)).to(F16).cuda()
        out, st, kl = torch.zeros_like(q), ints([0, n]), ints([32])
        h = q.shape[1]
        a = B.AttnPagedArgs(q=q.data_ptr(), out=out.data_ptr(), q_tok=h * d, out_tok=h * d, n_tok=n, n_seq=1, n_head=h, n_kv_head=1,
                            head_dim=d, io_type=B.F16, kv_type=B.Q8, scale=d ** -0.5, k_pages=big.data_ptr(), v_pages=big.data_ptr(),
                            n_pages=2, page_stride=stride, page_size=16, max_pages=2, table=table.data_ptr(), table_stride=2,
                            starts=st.data_ptr(), kv_len=kl.data_ptr(), max_kv=32)
        assert B.lib().bonsai_p40_attn_paged(C.byref(a), B._stream(None)) == 0
        ref, mag, top = attn_ref(q.cpu(), kd, kd, table.cpu(), [0, n], [32], d ** -0.5, out.cpu())
        check_q8(out.cpu(), ref, mag, top, q.cpu(), float(kd.abs().sum(-1).max()), d ** -0.5, F16, 32)
