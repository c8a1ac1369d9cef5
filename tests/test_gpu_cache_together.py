"""8-bit pages and shared prefixes as they are used: between the projections of a
layer, a prompt in chunks and then token by token, samples of one prompt, captured in
graphs that are replayed while the lengths grow, and a cache handed on to another."""
import pytest

import bonsai_p40 as B
from test_gpu_attn_shared import ref_of
from test_gpu_mixers import BF16, F16, F32, U, attn_ref, case, check_attn, gen, half_step, ints, normwise, rope_ref
from test_gpu_mixers_together import AttnLayer, D, EMBD, HEADS, KVH, PAGE, scratch
from test_gpu_q8_cache import check_q8, pages_of, quantised

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    B.lib()
    yield
    torch.cuda.synchronize()


class Layer8(AttnLayer):
    """The same layer over 8-bit pages."""

    def __init__(self, seed, tokens):
        super().__init__(seed, F16, tokens)
        pages = self.kp.shape[0]
        (self.kp, self.ks), (self.vp, self.vs) = (B.q8_pages(pages, KVH, PAGE, D) for _ in range(2))

    def rows(self, slots):
        """What the pages hold: numbers times scales, in 64 bits."""
        c = [p.cpu().transpose(1, 2).reshape(-1, KVH, D)[slots.cpu()].double() for p in (self.kp, self.vp)]
        s = [p.cpu().transpose(1, 2).reshape(-1, KVH)[slots.cpu()].double()[..., None] for p in (self.ks, self.vs)]
        return c[0] * s[0], c[1] * s[1], s[0], s[1]

    def values(self):
        return (self.kp.cpu().double() * self.ks.cpu().double()[..., None], self.vp.cpu().double() * self.vs.cpu().double()[..., None])


def test_attention_between_its_projections():
    """A prompt of 70 tokens, 3 single ones, then 20 more; every stage against 64 bits."""
    case("layer over 8-bit pages")
    layer = Layer8(1, 100)
    fp32 = 24 * U
    for i, n in enumerate((70, 1, 1, 1, 20)):
        y = layer.project(torch.randn(n, EMBD, generator=gen(i)).cuda())
        q, k, v, pos, slots, qr, out = layer.mix(y)
        kr, vr, kd, vd = layer.rows(slots)
        ref, mag = rope_ref(k.cpu(), layer.norms[1].cpu(), 1e-6, pos.cpu(), layer.inv_freq.cpu(), False)
        assert bool(((kr - ref).abs() <= 0.50002 * kd + fp32 * mag.amax(-1, keepdim=True)).all())
        assert bool(((vr - v.cpu().double()).abs() <= 0.50002 * vd).all())
        kp, vp = layer.values()
        ref, mag, top = attn_ref(qr.cpu(), kp, vp, layer.table.cpu(), [0, n], [layer.seen], D ** -0.5, out.cpu())
        check_q8(out.cpu(), ref, mag, top, qr.cpu(), float(kp.abs().sum(-1).max()), D ** -0.5, F32, layer.seen)
        # read back in any type, they are the rows that attention saw
        for t in (F32, BF16):
            ko, vo = (torch.empty(n, KVH, D, dtype=t, device="cuda") for _ in range(2))
            B.kv_read(layer.kp, layer.vp, slots, ko, vo)
            assert torch.equal(ko.cpu(), kr.float().to(t)) and torch.equal(vo.cpu(), vr.float().to(t))


def test_a_chunk_equals_its_tokens():
    case("8-bit pages: chunk against steps")
    a, b = Layer8(2, 90), Layer8(2, 90)
    y = a.project(torch.randn(81, EMBD, generator=gen(0)).cuda())
    whole = a.mix(y)[-1]
    parts = [b.mix(y[:, i:j].contiguous())[-1] for i, j in [(0, 60)] + [(i, i + 1) for i in range(60, 81)]]
    assert torch.equal(a.kp, b.kp) and torch.equal(a.ks, b.ks) and torch.equal(a.vp, b.vp) and torch.equal(a.vs, b.vs)
    # each is within 2^-18 of the exact result for the same pages
    assert normwise(torch.cat(parts), whole.double().cpu()) <= 2.0 ** -17


def test_a_cache_handed_to_another():
    """16-bit pages read back and appended to 8-bit ones, and these to 16-bit ones again."""
    case("16 bits to 8 bits and back")
    n, g = 100, gen(4)
    kp, vp = torch.randn(2, 8, KVH, PAGE, D, generator=g).to(F16).cuda()
    slots = torch.randperm(8 * PAGE, generator=g)[:n].cuda()
    k, v = (torch.empty(n, KVH, D, device="cuda") for _ in range(2))
    B.kv_read(kp, vp, slots, k, v)
    (kc, ks), (vc, vs) = (B.q8_pages(8, KVH, PAGE, D) for _ in range(2))
    q, qo = torch.zeros(n, 1, D, device="cuda"), torch.empty(n, 1, D, device="cuda")
    B.qk_norm_rope(q, k, v, None, None, 1e-6, None, None, slots, kc, vc, qo)
    k8, v8 = (torch.empty(n, KVH, D, dtype=F16, device="cuda") for _ in range(2))
    B.kv_read(kc, vc, slots, k8, v8)
    for x, y in ((k, k8), (v, v8)):
        codes, d = quantised(x.cpu())
        assert torch.equal(y.cpu(), (codes.float() * d[..., None]).to(F16))
    back = torch.zeros_like(kp), torch.zeros_like(vp)
    B.qk_norm_rope(q, k8.float(), v8.float(), None, None, 1e-6, None, None, slots, *back, qo)
    k16, v16 = torch.empty_like(k8), torch.empty_like(v8)
    B.kv_read(*back, slots, k16, v16)
    assert torch.equal(k16, k8) and torch.equal(v16, v8)


@pytest.mark.parametrize("t", ["q8", F16])
def test_a_captured_decode_step_of_samples_of_one_prompt(t):
    """Append and attn_shared in a graph, replayed while every sequence grows: each replay against 64 bits, with
    other work and synchronisations between the replays.  Its prefix gets longer and its groups change, too."""
    case(f"captured shared step {t}")
    n_seq, heads, kvh, d, page, pages = 5, 6, 2, 64, 16, 40
    g = gen(7)
    base = torch.randn(2, pages, kvh, page, d, generator=g)
    if t == "q8":
        dev = [pages_of(*quantised(x)) for x in base]
        kp, vp = dev[0][0], dev[1][0]
    else:
        kp, vp = (x.to(t).cuda() for x in base)
    q, k, v = (torch.zeros(n_seq, h, d, device="cuda") for h in (heads, kvh, kvh))
    table = torch.zeros(n_seq, 7, dtype=torch.int32)
    free = torch.randperm(pages, generator=g).tolist()
    front = [free.pop() for _ in range(3)]                  # 48 keys of prefix
    for s in range(n_seq):
        table[s] = torch.tensor(front + [free.pop() for _ in range(4)])
    dtab, starts = table.cuda(), ints(range(n_seq + 1))
    kv, slots = ints([0] * n_seq), torch.full((n_seq,), -1, dtype=torch.int64, device="cuda")     # (-1: nothing is written yet)
    pos, inv = ints([0] * n_seq), B.rope_inv_freq(32, 1e4)
    groups, shared = ints([0, n_seq]), ints([48])
    qr, out = torch.empty_like(q), torch.empty_like(q)
    args = [qr, kp, vp, dtab, starts, kv, groups, shared, out]
    ws = torch.empty(B.attn_shared_workspace_bytes(*args, max_kv=112, max_shared=48) + 16, dtype=torch.uint8, device="cuda")

    def step():
        B.qk_norm_rope(q, k, v, None, None, 1e-6, pos, inv, slots, kp, vp, qr)
        B.attn_shared(*args, ws, max_kv=112, max_shared=48)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(6):
        length = [50 + i + 3 * s for s in range(n_seq)]
        kv.copy_(torch.tensor(length))
        pos.copy_(torch.tensor(length) - 1)
        slots.copy_(torch.tensor([int(table[s, (length[s] - 1) // page]) * page + (length[s] - 1) % page for s in range(n_seq)]))
        gr, sh = ([0, n_seq], [48]) if i < 4 else ([1, 4], [32])
        groups.copy_(torch.tensor(gr))
        shared.copy_(torch.tensor(sh))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        if t == "q8":
            kd, vd = (c.cpu().double() * s.cpu().double()[..., None] for c, s in dev)
        else:
            kd, vd = kp.cpu(), vp.cpu()
        ref, mag, top = ref_of(qr.cpu(), kd, vd, table, list(range(n_seq + 1)), length, gr, sh, d ** -0.5, out.cpu())
        if t == "q8":
            check_q8(out.cpu(), ref, mag, top, qr.cpu(), float(kd.abs().sum(-1).max()), d ** -0.5, F32, 112)
        else:
            check_attn(out.cpu(), ref, mag, top, F32, d, 112)
        eager = torch.empty_like(out)
        B.attn_shared(*args[:-1], eager, ws, max_kv=112, max_shared=48)
        assert torch.equal(eager, out)


def test_two_graphs_with_workspaces_of_their_own():
    """Replayed at the same time on two streams."""
    case("two graphs")
    g = gen(8)
    pages = [pages_of(*quantised(torch.randn(60, 2, 16, 64, generator=g)))[0] for _ in range(2)]
    table = torch.randperm(60, generator=g)[:56].view(8, 7).int().cuda()
    made = []
    for i in range(2):
        q = torch.randn(8, 6, 64, generator=g).cuda().to(BF16)
        args = [q, *pages, table, ints(range(9)), ints([100 + j for j in range(8)]), ints([0, 5, 8]), ints([64 + i, 48]), torch.empty_like(q)]
        ws = scratch(B.attn_shared_workspace_bytes(*args, max_kv=112, max_shared=65))
        B.attn_shared(*args, ws, max_kv=112, max_shared=65)
        want = args[-1].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            B.attn_shared(*args, ws, max_kv=112, max_shared=65)
        made.append((graph, args[-1], want, torch.cuda.Stream(), (args, ws)))     # (a graph keeps no tensors)
    for _ in range(5):
        for graph, out, want, stream, _ in made:
            out.zero_()
        torch.cuda.synchronize()
        for graph, out, want, stream, _ in made:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out, want, _, _ in made)


def test_a_shared_batch_equals_its_sequences():
    """attn_shared and attn_paged over the same tables: both within their limits of the exact result, and so of each other."""
    case("shared against paged")
    g = gen(9)
    for t, io in (("q8", F32), (F16, F32), (BF16, BF16)):
        raw = torch.randn(2, 50, KVH, PAGE, D, generator=g)
        dev = [pages_of(*quantised(x))[0] for x in raw] if t == "q8" else [x.to(t).cuda() for x in raw]
        rows = [list(range(6)) + [6 + 4 * s + j for j in range(4)] for s in range(8)]
        q = torch.randn(8 * 3, HEADS, D, generator=g).cuda().to(io)
        kv = [96 + 5 + 7 * s for s in range(8)]
        args = [q, *dev, ints(rows), ints([3 * s for s in range(9)]), ints(kv)]
        a, b = torch.empty_like(q), torch.empty_like(q)
        B.attn_paged(*args, a, max_kv=max(kv))
        ws = scratch(B.attn_shared_workspace_bytes(*args, ints([0, 8]), ints([96]), b))
        B.attn_shared(*args, ints([0, 8]), ints([96]), b, ws)
        assert normwise(b, a.double().cpu()) <= 2 * (half_step(io) if io != F32 else 2.0 ** -18)
