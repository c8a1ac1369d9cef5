"""The token mixers as they are used: between the projections of a layer, a prompt
in chunks and then token by token, captured in graphs that are replayed while
the lengths grow, and on several streams."""
import pytest

import bonsai_p40 as B
from test_gpu_chain import weights
from test_gpu_mixers import (BF16, F16, F32, U, attn_ref, case, check_attn, gdn_ref, gen, half_step, ints, normwise,
                             rope_ref)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU visible")
    B.lib()
    yield
    torch.cuda.synchronize()


HEADS, KVH, D, ROT, EMBD, PAGE = 8, 2, 64, 32, 1024, 16
Q_ROWS, KV_ROWS = HEADS * 2 * D, KVH * D                     # a head's queries are followed by its gates


def scratch(n):
    return torch.empty(n + 16, dtype=torch.uint8, device="cuda")


class AttnLayer:
    """Projection, head norms and rotation, pages, attention, projection: one sequence, n tokens a call."""

    def __init__(self, seed, t, tokens):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.w_in, self.w_out = weights(g, Q_ROWS + 2 * KV_ROWS, EMBD), weights(g, EMBD, HEADS * D)
        self.norms = [torch.rand(D, generator=g, device="cuda") + 0.5 for _ in range(2)]
        self.inv_freq = B.rope_inv_freq(ROT, 1e6)
        pages = -(-tokens // PAGE)
        self.kp, self.vp = (torch.zeros(pages + 1, KVH, PAGE, D, dtype=t, device="cuda") for _ in range(2))
        self.table = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int().cuda()[None]
        self.seen = 0

    def project(self, x):
        n = x.shape[0]
        xq = torch.empty(B.q8_bytes(EMBD, n), dtype=torch.uint8, device="cuda")
        y = torch.empty(Q_ROWS + 2 * KV_ROWS, n, device="cuda")
        B.quant_tokens(x, None, xq, EMBD, n, False)
        B.gemm(self.w_in, xq, y, Q_ROWS + 2 * KV_ROWS, EMBD, n)
        return y

    def mix(self, y):
        n = y.shape[1]
        q = y[:Q_ROWS].view(HEADS, 2 * D, n).permute(2, 0, 1)[:, :, :D]
        k = y[Q_ROWS:Q_ROWS + KV_ROWS].view(KVH, D, n).permute(2, 0, 1)
        v = y[Q_ROWS + KV_ROWS:].view(KVH, D, n).permute(2, 0, 1)
        pos = torch.arange(self.seen, self.seen + n, dtype=torch.int32, device="cuda")
        slots = self.table[0, (pos // PAGE).long()].long() * PAGE + pos % PAGE
        qr = torch.empty(n, HEADS, D, device="cuda")
        B.qk_norm_rope(q, k, v, *self.norms, 1e-6, pos, self.inv_freq, slots, self.kp, self.vp, qr)
        self.seen += n
        out = torch.empty_like(qr)
        args = (qr, self.kp, self.vp, self.table, ints([0, n]), ints([self.seen]), out)
        B.attn_paged(*args, scratch(B.attn_paged_workspace_bytes(*args, max_kv=self.seen)), max_kv=self.seen)
        return q, k, v, pos, slots, qr, out

    def finish(self, out):
        n = out.shape[0]
        xq = torch.empty(B.q8_bytes(HEADS * D, n), dtype=torch.uint8, device="cuda")
        y = torch.empty(EMBD, n, device="cuda")
        B.quant_tokens(out, None, xq, HEADS * D, n, False)
        B.gemm(self.w_out, xq, y, EMBD, HEADS * D, n)
        return y


@pytest.mark.parametrize("t", [F16, BF16])
def test_attention_between_its_projections(t):
    """A prompt of 70 tokens, 3 single ones, then 20 more; every stage against 64 bits."""
    case(f"layer {t}")
    layer = AttnLayer(1, t, 100)
    w = torch.empty(EMBD * HEADS * D, device="cuda")
    B.dequantize_pq2_0(layer.w_out, w, w.numel())
    w = w.view(EMBD, HEADS * D).double().cpu()
    fp32 = 24 * U                                            # as for the head rows by themselves
    for i, n in enumerate((70, 1, 1, 1, 20)):
        y = layer.project(torch.randn(n, EMBD, generator=gen(i)).cuda())
        q, k, v, pos, slots, qr, out = layer.mix(y)
        last = layer.finish(out)
        for got, src, norm in ((qr, q, layer.norms[0]), (layer.kp.transpose(1, 2).reshape(-1, KVH, D)[slots], k, layer.norms[1])):
            ref, mag = rope_ref(src.cpu(), norm.cpu(), 1e-6, pos.cpu(), layer.inv_freq.cpu(), False)
            lim = half_step(got.dtype) * (ref.abs() + fp32 * mag) + fp32 * mag + torch.finfo(got.dtype).tiny
            assert bool(((got.cpu().double() - ref).abs() <= lim).all())
        assert torch.equal(layer.vp.transpose(1, 2).reshape(-1, KVH, D)[slots], v.to(t))
        ref, mag, top = attn_ref(qr.cpu(), layer.kp.cpu(), layer.vp.cpu(), layer.table.cpu(), [0, n], [layer.seen], D ** -0.5, out.cpu())
        check_attn(out.cpu(), ref, mag, top, F32, D, layer.seen)
        # a block of 32 is rounded to steps of amax / 127, a scale that has 11 bits; 512 products and sums in fp32
        x = out.cpu().double().view(n, HEADS * D)
        step = x.abs().view(n, -1, 32).amax(-1, keepdim=True) * (1 / 254 + 2.0 ** -10)
        lim = (step.expand(-1, -1, 32).reshape(n, -1) + x.abs() * 1024 * U) @ w.abs().t()
        assert bool(((last.t().cpu().double() - x @ w.t()).abs() <= lim).all())


def test_a_chunk_equals_its_tokens():
    """The same tokens at once and one after another: attention and the gated delta rule."""
    case("chunk against steps")
    a, b = AttnLayer(2, BF16, 90), AttnLayer(2, BF16, 90)
    y = a.project(torch.randn(81, EMBD, generator=gen(0)).cuda())
    whole = a.mix(y)[-1]
    parts = [b.mix(y[:, i:j].contiguous())[-1] for i, j in [(0, 60)] + [(i, i + 1) for i in range(60, 81)]]
    # each is within 2^-18 of the exact result for the same pages
    assert torch.equal(a.kp, b.kp) and torch.equal(a.vp, b.vp)
    assert normwise(torch.cat(parts), whole.double().cpu()) <= 2.0 ** -17

    r, n, kh, vh, kd = gen(1), 150, 2, 4, 64
    q, k = (torch.randn(n, kh, kd, generator=r).cuda() for _ in range(2))
    v, g = torch.randn(n, vh, kd, generator=r).cuda(), -0.2 * torch.rand(n, vh, generator=r).cuda()
    beta = torch.sigmoid(torch.randn(n, vh, generator=r)).cuda()
    results = []
    for cuts in ([0, 150], [0, 100] + list(range(101, 151)), [0, 1, 2, 65, 66, 150]):
        state = torch.zeros(1, vh, kd, kd, device="cuda")
        out = torch.empty_like(v)
        for i, j in zip(cuts, cuts[1:]):
            args = (q[i:j], k[i:j], v[i:j], g[i:j], beta[i:j], state, state, out[i:j], ints([0, j - i]))
            B.gdn(*args, scratch(B.gdn_workspace_bytes(*args, l2_eps=1e-6)), l2_eps=1e-6)
        results.append((out, state))
    ref, final = gdn_ref(q.cpu(), k.cpu(), v.cpu(), g.cpu(), beta.cpu(), torch.zeros(1, vh, kd, kd), [0, n], None, kd ** -0.5, 1e-6, False)
    want = torch.stack([ref[i] for i in range(n)])
    for out, state in results:
        assert normwise(out, want) <= 2.0 ** -17 and normwise(state, final) <= 2.0 ** -17


class Step:
    """The three mixers on fixed buffers: sequences of `new` tokens each, more from call to call."""

    def __init__(self, new, room, seed=0, t=BF16):
        g, s = gen(seed), len(new)
        self.new, n = new, sum(new)
        self.qkv = [torch.randn(n, h, D, generator=g).cuda() for h in (HEADS, KVH, KVH)]
        self.rows = torch.randn(n, 3, HEADS, D, generator=g).to(t).cuda()
        self.g, self.beta = -torch.rand(n, HEADS, generator=g).cuda(), torch.rand(n, HEADS, generator=g).cuda()
        self.per = -(-room // PAGE)
        self.table = torch.randperm(s * self.per, generator=g).int().view(s, -1).cuda()
        self.kp, self.vp = (torch.zeros(s * self.per, KVH, PAGE, D, dtype=t, device="cuda") for _ in range(2))
        self.state = torch.zeros(s, HEADS, D, D, device="cuda")
        self.inv_freq, self.norm = B.rope_inv_freq(ROT, 1e4), torch.ones(D, device="cuda")
        self.starts = ints([sum(new[:i]) for i in range(s + 1)])
        self.qr, self.out = (torch.zeros(n, HEADS, D, dtype=t, device="cuda") for _ in range(2))
        self.mixed = torch.zeros(n, HEADS, D, dtype=t, device="cuda")
        self.kv_len, self.pos, self.slots = ints([0] * s), ints([0] * n), torch.zeros(n, dtype=torch.int64, device="cuda")
        self.room = room
        self.ws = [scratch(B.attn_paged_workspace_bytes(*self.attn(), max_kv=room)),
                   scratch(B.gdn_workspace_bytes(*self.delta(), **self.kw()))]

    def attn(self):
        return self.qr, self.kp, self.vp, self.table, self.starts, self.kv_len, self.out

    def delta(self):
        return self.rows[:, 0], self.rows[:, 1], self.rows[:, 2], self.g, self.beta, self.state, self.state, self.mixed, self.starts

    def kw(self):
        return dict(max_new=max(self.new), l2_eps=1e-6)

    def advance(self, i):
        """New inputs and lengths, in place: the i-th call's."""
        g = gen(100 + i)
        for x in (*self.qkv, self.rows):
            x.copy_(torch.randn(x.shape, generator=g))
        before = self.kv_len.cpu()
        pos = torch.cat([torch.arange(n) + int(before[s]) for s, n in enumerate(self.new)])
        seq = torch.cat([torch.full((n,), s) for s, n in enumerate(self.new)])
        self.pos.copy_(pos.int())
        self.slots.copy_(self.table.cpu()[seq, pos // PAGE].long() * PAGE + pos % PAGE)
        self.kv_len.copy_(before + torch.tensor(self.new))

    def run(self, stream=None):
        q, k, v = self.qkv
        B.qk_norm_rope(q, k, v, self.norm, self.norm, 1e-6, self.pos, self.inv_freq, self.slots, self.kp, self.vp, self.qr, stream=stream)
        B.attn_paged(*self.attn(), self.ws[0], max_kv=self.room, stream=stream)
        B.gdn(*self.delta(), self.ws[1], **self.kw(), stream=stream)

    def results(self):
        torch.cuda.synchronize()
        return [x.clone() for x in (self.qr, self.kp, self.vp, self.out, self.mixed, self.state)]


SHAPES = [([1], 3000), ([1, 1, 1], 200), ([90], 700), ([70, 1, 40], 500), ([8], 2000)]


@pytest.mark.parametrize("new,room", SHAPES)
def test_graphs_replayed_while_lengths_grow(new, room):
    case(f"graph new={new} room={room}")
    eager, twin = Step(new, room), Step(new, room)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        Step(new, room).run()
    torch.cuda.current_stream().wait_stream(warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        twin.run()
    other = Step([33], 100, seed=9)
    for i in range(5):
        eager.advance(i)
        eager.run()
        twin.advance(i)
        for w in twin.ws:
            w.fill_(255 - i)                                 # nothing is kept there
        torch.cuda.synchronize()
        graph.replay()
        for x, y in zip(twin.results(), eager.results()):
            assert torch.equal(x, y), f"replay {i}"
        other.advance(0) if i == 0 else None
        other.run()                                          # eager work between the replays
        torch.cuda.synchronize()


def test_two_graphs_that_share_a_workspace():
    """One after the other on one stream, as often as one likes."""
    case("two graphs, one workspace")
    steps, plain = [Step([60], 400, 1), Step([1, 1], 900, 2)], [Step([60], 400, 1), Step([1, 1], 900, 2)]
    ws = [max((s.ws[i] for s in steps), key=lambda w: w.numel()) for i in range(2)]
    graphs = []
    for s in steps:
        s.ws = ws
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            s.run()
    for i in range(4):
        for s in steps + plain:
            s.advance(i)
        torch.cuda.synchronize()
        for j in (0, 1):
            graphs[j].replay()
            plain[j].run()
        for s, p in zip(steps, plain):
            for x, y in zip(s.results(), p.results()):
                assert torch.equal(x, y), i


def test_streams_side_by_side():
    """Two streams at once, each with its workspaces, by argument and by context."""
    case("streams")
    steps = [Step([100, 7], 600, 3), Step([1, 1], 2500, 4)]
    plain = [Step([100, 7], 600, 3), Step([1, 1], 2500, 4)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(4):
        for s in steps + plain:
            s.advance(i)
        torch.cuda.synchronize()
        steps[0].run(stream=streams[0])
        with torch.cuda.stream(streams[1]):
            steps[1].run()
        torch.cuda.synchronize()
        for s, p in zip(steps, plain):
            p.run()
            for x, y in zip(s.results(), p.results()):
                assert torch.equal(x, y), i


def test_the_same_call_gives_the_same_bytes():
    case("again")
    for new, room in SHAPES:
        results = []
        for rep in range(3):
            s = Step(new, room, 6)
            s.advance(0)
            s.run()
            results.append(s.results())
        for r in results[1:]:
            for x, y in zip(r, results[0]):
                assert torch.equal(x, y)


def test_room_for_every_length():
    """Sequences without tokens and without keys beside others, and a batch padded behind the last sequence."""
    case("padded batch")
    s = Step([5, 0, 1], 60)
    s.advance(0)
    s.starts.copy_(ints([0, 4, 4, 5]))                       # the sixth row is padding
    s.kv_len.copy_(ints([4, 0, 1]))
    s.slots[5] = -1
    s.slots[4] = int(s.table[2, 0]) * PAGE
    s.slots[:4] = int(s.table[0, 0]) * PAGE + torch.arange(4, device="cuda")
    s.pos.copy_(ints([0, 1, 2, 3, 0, 0]))
    s.out.fill_(3.0), s.mixed.fill_(3.0)
    s.run()
    qr, kp, vp, out, mixed, state = s.results()
    ref, mag, top = attn_ref(qr.cpu(), kp.cpu(), vp.cpu(), s.table.cpu(), [0, 4, 4, 5], [4, 0, 1], D ** -0.5, out.cpu())
    check_attn(out.cpu(), ref, mag, top, BF16, D, 4)
    assert bool((out[5] == 3).all()) and bool((mixed[5] == 3).all()) and bool((state[1] == 0).all())


@pytest.mark.parametrize("new", [[20, 20, 20], [1, 1, 1]])
def test_starts_that_fall_stay_inside(new):
    """Sequences that overlap, or lie outside: nothing but their rows changes, and what they do not claim is as ever."""
    case(f"falling starts {new}")
    n = sum(new)
    s = Step(new, 200)
    s.advance(0)
    for starts in ([0, n, 1, n - 1], [-5, n - 1, n - 1, n - 1], [n - 1, 0, 0, 0], [0, n + 9, n + 9, n + 99], [2 ** 31 - 1, -2 ** 31, 0, 1]):
        s.starts.copy_(torch.tensor(starts, dtype=torch.int32))
        s.out.fill_(3.0), s.mixed.fill_(3.0)
        s.run()
        torch.cuda.synchronize()
        ends = [min(max(x, 0), n) for x in starts]
        rows = {t for a, b in zip(ends, ends[1:]) for t in range(a, b)}
        rest = [t for t in range(n) if t not in rows]
        assert bool((s.out[rest] == 3).all()) and bool((s.mixed[rest] == 3).all())
