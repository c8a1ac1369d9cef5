"""attn_shared (batches that share a prefix) against a plain implementation in 64
bits, at the groups, lengths and masks where it can go wrong; tolerances are
those of attn_paged over the same pages."""
import pytest

import bonsai_p40 as B
from test_gpu_mixers import BF16, F16, F32, NAN, case, check_attn, gen, ints
from test_gpu_q8_cache import check_q8, pages_of, quantised

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")


def ref_of(q, kp, vp, table, starts, kv_len, groups, shared, scale, out):
    """attn_ref of tokens that see the shared keys of their group and then their own."""
    n, heads, d = q.shape
    n_pages, kvh, page, _ = kp.shape
    cap = table.shape[1] * page
    ref = out.double().clone()
    mag, top = torch.zeros(n, heads, d, dtype=torch.float64), torch.zeros(n, heads, 1, dtype=torch.float64)
    lead = {s: (max(min(groups[g], len(kv_len)), 0), max(0, min(shared[g], cap))) for g in range(len(shared))
            for s in range(groups[g], min(groups[g + 1], len(kv_len)))}
    for s in range(len(kv_len)):
        a, b, kv = starts[s], starts[s + 1], max(0, min(kv_len[s], cap))
        first, pre = lead.get(s, (s, 0))
        for t in range(a, b):
            keys = [(first, j) for j in range(pre)] + [(s, j) for j in range(pre, max(0, min(kv, kv - (b - a) + (t - a) + 1)))]
            keys = [(int(table[r, j // page]), j % page) for r, j in keys]
            keys = [x for x in keys if 0 <= x[0] < n_pages]
            if not keys:
                ref[t] = 0
                continue
            pg, off = (torch.tensor(x) for x in zip(*keys))
            for h in range(heads):
                k, v = kp[pg, h // (heads // kvh), off].double(), vp[pg, h // (heads // kvh), off].double()
                x = (k @ q[t, h].double()) * scale
                p = torch.softmax(x, 0)
                ref[t, h], mag[t, h] = p @ v, p @ v.abs()
                top[t, h] = (k.abs() @ q[t, h].double().abs()).max() * scale
    return ref, mag, top


def run_shared(new, own, groups, shared, heads, kvh, d, page, t, io, seed=0, pad=0, hints=True, edit=None, lengths=None, calls=1):
    """new tokens and own keys (the new ones included) of every sequence; lengths: kv_len instead."""
    case(f"shared new={new} own={own} groups={groups} shared={shared} heads={heads}/{kvh} d={d} page={page} {t} io={io} pad={pad} hints={hints}")
    g = gen(seed)
    starts = [pad]
    for x in new:
        starts.append(starts[-1] + x)
    n, n_seq = starts[-1] + pad, len(new)
    pre = [0] * n_seq
    for i, p in enumerate(shared):
        for s in range(groups[i], min(groups[i + 1], n_seq)):
            pre[s] = p
    kv = [p + o for p, o in zip(pre, own)] if lengths is None else lengths
    cols = max(-(-c // page) for c in kv + [1])
    total = n_seq * cols + 2
    table = torch.randperm(total, generator=g)[:n_seq * cols].view(n_seq, cols).int()
    kp, vp = torch.randn(2, total, kvh, page, d, generator=g)
    if t == "q8":
        (kc, ks), (vc, vs) = quantised(kp), quantised(vp)
    else:
        kc, vc = kp.to(t), vp.to(t)
        ks = vs = None
    q = (torch.randn(n, heads, d, generator=g) * 1.3).to(io)
    if edit:
        edit(q, kc, ks, vc, vs, table)
    kd, vd = (kc.double() * ks.double()[..., None], vc.double() * vs.double()[..., None]) if t == "q8" else (kc, vc)
    kd, vd = kd.clone(), vd.clone()
    # nothing is seen behind the last key, nor before its own ones in a sequence's pages that do not lead its group
    for s in range(n_seq):
        lead = any(groups[i] == s for i in range(len(shared)) if groups[i] < groups[i + 1])
        for j in ([] if lead else range(min(pre[s], cols * page))):
            spoil(kc, ks, vc, vs, int(table[s, j // page]), j % page)
        for j in range(max(kv[s], 0), cols * page):
            if not (lead and j < pre[s]):
                spoil(kc, ks, vc, vs, int(table[s, j // page]), j % page)
    dev = [pages_of(kc, ks)[0], pages_of(vc, vs)[0]] if t == "q8" else [kc.cuda(), vc.cuda()]
    out = torch.full((n, heads, d), 7.0, dtype=io)
    mk, ms = (max(kv + [1]), max(shared + [0])) if hints is True else hints
    args = [q.cuda(), *dev, table.cuda(), ints(starts), ints(kv), ints(groups), ints(shared), out.cuda()]
    ws = torch.full((B.attn_shared_workspace_bytes(*args, max_kv=mk, max_shared=ms) + 16,), 255, dtype=torch.uint8, device="cuda")
    for _ in range(calls):
        B.attn_shared(*args, ws, max_kv=mk, max_shared=ms)
    torch.cuda.synchronize()
    got = args[8].cpu()
    scale = d ** -0.5
    ref, mag, top = ref_of(q, kd, vd, table, starts, kv, groups, shared, scale, out)
    keys = max(kv + shared + [1])
    if t == "q8":
        check_q8(got, ref, mag, top, q, float(kd.abs().sum(-1).max()), scale, io, keys)
    else:
        check_attn(got, ref, mag, top, io, d, keys)
    return got


def spoil(kc, ks, vc, vs, page, slot):
    if ks is None:
        kc[page, :, slot], vc[page, :, slot] = NAN, INF
    else:
        ks[page, :, slot], vs[page, :, slot] = NAN, INF


KINDS = [(BF16, BF16), (F16, F16), (F16, F32), (BF16, F32), ("q8", BF16), ("q8", F16), ("q8", F32)]


@pytest.mark.parametrize("heads,kvh,d", [(6, 1, 256), (8, 2, 128), (7, 1, 64)])
@pytest.mark.parametrize("t,io", KINDS)
def test_decode_of_one_group(heads, kvh, d, t, io):
    run_shared([1], [1], [0, 1], [1], heads, kvh, d, 16, t, io)
    run_shared([1] * 3, [1, 20, 33], [0, 3], [100], heads, kvh, d, 16, t, io, seed=1)
    run_shared([1] * 12, [1 + 7 * i for i in range(12)], [0, 12], [256], heads, kvh, d, 32, t, io, seed=2)
    run_shared([1] * 30, [1 + i for i in range(30)], [0, 30], [333], heads, kvh, d, 16, t, io, seed=3, pad=2)


@pytest.mark.parametrize("heads,kvh,d", [(6, 1, 256), (4, 2, 128), (5, 1, 64)])
@pytest.mark.parametrize("t,io", KINDS)
def test_groups_and_several_tokens(heads, kvh, d, t, io):
    """Ragged groups, an empty one, sequences of none; drafts and chunks."""
    run_shared([1, 2, 1, 3, 1, 1, 1], [4, 9, 1, 40, 70, 5, 6], [1, 3, 3, 6], [37, 5, 64], heads, kvh, d, 16, t, io)
    run_shared([40, 0, 33, 75, 1], [45, 3, 33, 130, 9], [0, 2, 4], [90, 48], heads, kvh, d, 32, t, io, seed=1, pad=3)
    run_shared([5] * 9, [5 + i for i in range(9)], [0, 4, 9], [70, 129], heads, kvh, d, 16, t, io, seed=2)


@pytest.mark.parametrize("t,io", [(F16, F16), (BF16, F32), ("q8", F32)])
def test_every_place_where_a_prefix_can_end(t, io):
    """Against tiles of 32, the 16 keys of a page's share, and pages: the first own keys are in the middle of each."""
    for pre in (0, 1, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65):
        run_shared([1, 1], [1, 18], [0, 2], [pre], 4, 2, 64, 64, t, io, seed=pre)
        run_shared([34, 1], [40, 2], [0, 2], [pre], 4, 1, 128, 16, t, io, seed=pre)


@pytest.mark.parametrize("t,io", [(F16, F16), (F16, F32), ("q8", BF16)])
def test_lengths_that_do_not_fit_the_prefix(t, io):
    """A prefix longer than a sequence is seen whole; negative and too long ones are cut; no own keys at all."""
    for new, kv in (([1, 1, 1], [50, 20, 0]), ([40, 3, 1], [45, 2, 70])):
        run_shared(new, None, [0, 3], [48], 4, 2, 64, 16, t, io, lengths=kv)
        run_shared(new, None, [0, 3], [-5], 4, 2, 64, 16, t, io, lengths=kv)
    got = run_shared([1, 1], None, [0, 1, 2], [0, 0], 4, 2, 64, 16, t, io, lengths=[0, 0])
    assert bool((got == 0).all())

    def edit(q, kc, ks, vc, vs, table):
        table[:, -1] = -1
    run_shared([1, 30], None, [0, 2], [10 ** 6], 4, 2, 64, 16, t, io, lengths=[50, 80], edit=edit)


@pytest.mark.parametrize("t,io", [(BF16, BF16), ("q8", F32)])
def test_freed_pages(t, io):
    """Pages that are none, in the prefix, in the own keys, and everywhere."""
    def some(q, kc, ks, vc, vs, table):
        table[0, 1], table[1, 5], table[2, 6] = -1, 10 ** 6, -2 ** 31

    def none(q, kc, ks, vc, vs, table):
        table[:] = -1
    for new in ([1, 1, 1], [20, 40, 1]):
        run_shared(new, [60, 50, 45], [0, 3], [70], 6, 2, 128, 16, t, io, edit=some)
        got = run_shared(new, [60, 50, 45], [0, 3], [70], 6, 2, 128, 16, t, io, edit=none)
        assert bool((got == 0).all())


@pytest.mark.parametrize("t,io", [(F16, F16), ("q8", BF16)])
def test_many_groups_and_sequences(t, io):
    """More than a wave has lanes; groups outside the sequences are cut."""
    run_shared([1] * 150, [1 + i % 20 for i in range(150)], list(range(0, 150, 2)) + [150], [(5 * i) % 50 for i in range(75)],
               2, 1, 64, 16, t, io)
    run_shared([i % 3 for i in range(140)], [3 + i % 9 for i in range(140)], [0, 70, 139], [40, 20], 2, 1, 64, 16, t, io, seed=1)
    run_shared([1, 1, 1], [9, 8, 7], [1, 50], [20], 2, 1, 64, 16, t, io, seed=2)


@pytest.mark.parametrize("t,io", [(F16, F16), (F16, F32), ("q8", F16), ("q8", F32)])
def test_hints_place_the_work_only(t, io):
    for hints in ((0, 0), (1, 1), (5000, 4000), (700, 0), (0, 500)):
        run_shared([1] * 4, [30, 1, 200, 77], [0, 3, 4], [500, 300], 4, 2, 64, 16, t, io, hints=hints)
        run_shared([50, 60], [70, 60], [0, 2], [300], 4, 2, 64, 16, t, io, hints=hints)


def test_long_prefix_over_many_workgroups():
    for t, io in ((F16, F32), ("q8", F32), ("q8", BF16), (BF16, BF16)):
        run_shared([1] * 8, [1 + 9 * i for i in range(8)], [0, 8], [5000], 6, 1, 256, 64, t, io)
        run_shared([1] * 40, [3] * 40, [0, 40], [2000], 6, 1, 128, 16, t, io, seed=1)


@pytest.mark.parametrize("t,io", [(F16, F16), ("q8", F16)])
def test_values_that_are_not_finite(t, io):
    """A row of NaN in one sequence's own keys, or in one group's prefix, reaches those that see it."""
    for where, key in ((0, 7), (2, 50), (4, 10)):
        def edit(q, kc, ks, vc, vs, table):
            at = int(table[where, key // 16]), slice(None), key % 16
            if ks is None:
                vc[at] = NAN
            else:
                vs[at] = NAN
        for new in ([1] * 6, [20, 9, 5, 30, 1, 40]):
            run_shared(new, [40] * 6, [0, 4, 6], [33, 20], 4, 2, 64, 16, t, io, edit=edit)


def test_the_same_bytes_again_and_on_another_stream():
    g = gen(1)
    for t in (F16, "q8"):
        kp, vp = torch.randn(2, 40, 2, 16, 64, generator=g)
        dev = [pages_of(*quantised(x))[0] if t == "q8" else x.to(t).cuda() for x in (kp, vp)]
        q = torch.randn(6, 8, 64, generator=g).cuda().to(F16)
        table = torch.randperm(40, generator=g)[:36].view(6, 6).int().cuda()
        args = [q, *dev, table, ints(range(7)), ints([90, 70, 80, 96, 65, 66]), ints([0, 4, 6]), ints([64, 60])]
        outs = [torch.full_like(q, 5.0) for _ in range(3)]
        side = torch.cuda.Stream()
        for i, out in enumerate(outs):
            ws = torch.empty(B.attn_shared_workspace_bytes(*args, out), dtype=torch.uint8, device="cuda")
            torch.cuda.synchronize()
            with torch.cuda.stream(side if i == 2 else torch.cuda.current_stream()):
                B.attn_shared(*args, out, ws)
            torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]), t


def test_no_groups_is_attn_paged():
    q = torch.randn(3, 4, 64, generator=gen(2)).cuda().to(F16)
    kp, vp = torch.randn(2, 9, 2, 16, 64, generator=gen(3)).to(F16).cuda()
    args = [q, kp, vp, ints([[0, 1, 2], [3, 4, 5], [6, 7, 8]]), ints(range(4)), ints([40, 20, 48])]
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    B.attn_paged(*args, a)
    B.attn_shared(*args, ints([0]), torch.zeros(0, dtype=torch.int32, device="cuda"), b, None)
    assert torch.equal(a, b)


@pytest.mark.parametrize("heads,kvh", [(24, 4), (6, 1)])
@pytest.mark.parametrize("t,io", [("q8", F32), ("q8", BF16), (F16, F32), (BF16, BF16)])
def test_samples_of_a_long_prompt(t, io, heads, kvh):
    """Two samples of a prompt of 16000 keys: more parts than a wave has lanes."""
    part = 2 * heads * 258 * 4
    got = run_shared([1, 1], [40, 125], [0, 2], [16000], heads, kvh, 256, 64, t, io)
    q = torch.zeros(2, heads, 256, dtype=io, device="cuda")
    pages = B.q8_pages(1, kvh, 64, 256)[0] if t == "q8" else torch.zeros(1, kvh, 64, 256, dtype=t, device="cuda")
    table = torch.zeros(2, 252, dtype=torch.int32, device="cuda")
    args = [q, pages, pages, table, ints([0, 1, 2]), ints([1, 1]), ints([0, 2]), ints([16000]), got.cuda()]
    assert B.attn_shared_workspace_bytes(*args, max_kv=16125, max_shared=16000) // part > 64


@pytest.mark.parametrize("t,io", [("q8", BF16), (F16, F16), (F16, F32)])
def test_one_long_sequence_outside_the_groups(t, io):
    """Short own keys behind a prefix, and many of a sequence of no group, or of one behind a short prefix, whatever the hints."""
    for hints in (True, (700 + 3000, 700), (0, 0), (3100, 0), (1, 3000)):
        run_shared([1] * 5, [9, 20, 3, 15, 3000], [0, 4], [700], 4, 2, 64, 16, t, io, hints=hints)
        run_shared([1, 2, 1, 40], [9, 20, 1500, 60], [0, 2, 3], [700, 10], 6, 2, 256, 16, t, io, hints=hints)
