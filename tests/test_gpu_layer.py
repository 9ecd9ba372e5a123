"""The attention-side operators as a decoder uses them: together with the
router and the routed experts, on one cache from prompts over chunks to single
tokens; in captured graphs, on several streams and from several threads.

Tolerance of the attention output against the exact result of the layer's
projection rows.  With h half a step of the cache's type, q and k are off by h
each (their norm and rotation round once; f32 roundings before are 2^-13 of
that), so a score by 2.1 h sum |q_d k_d| scale =: s and a weight by the factor
exp(2 s) at most (its own score and the sum's); a value is off by h, a weight's
rounding by h, the output's by h:
|got - want| <= sum_j p_j |v_j| (exp(2 s) - 1 + 2.1 h) + h |want|.
"""
from __future__ import annotations

import importlib
import math
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_attention import BF16, F16, F32, HALF, Batch, inv_freq, norm_rope64  # noqa: E402
from test_gpu_parity import Q4, _oracle_moe, _table, assert_ffn_close, make_expert, say  # noqa: E402

pytestmark = pytest.mark.gpu


class Pages:
    """Block tables that grow: hands out pages of a pool in a scattered order."""

    def __init__(self, n_pages, page, n_seqs, width):
        self.page, self.free = page, [(7 * i + 3) % n_pages for i in range(n_pages)]
        assert math.gcd(7, n_pages) == 1
        self.table = torch.full((n_seqs, width), -1, dtype=torch.int32)
        self.len = [0] * n_seqs

    def append(self, s, n):
        """Slots of n more tokens of sequence s."""
        slots = []
        for at in range(self.len[s], self.len[s] + n):
            if at % self.page == 0:
                self.table[s, at // self.page] = self.free.pop()
            slots.append(int(self.table[s, at // self.page]) * self.page + at % self.page)
        self.len[s] += n
        return slots


def attention_bound(q, k, v, first, scale, h):
    """(out, bound above) of one sequence; q [n, H, d], k and v [L, G, d], float64."""
    n, heads, d = q.shape
    groups = k.shape[1]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    seen = torch.arange(k.shape[0]) <= first + torch.arange(n)[:, None]
    for hd in range(heads):
        kk, vv, qq = k[:, hd * groups // heads], v[:, hd * groups // heads], q[:, hd]
        p = torch.softmax(torch.where(seen, qq @ kk.T * scale, -math.inf), 1)
        s = torch.where(seen, qq.abs() @ kk.abs().T * scale, 0.0).amax(1, keepdim=True) * 2.1 * h
        out[:, hd] = p @ vv
        bound[:, hd] = (torch.exp(2 * s) - 1 + 2.1 * h) * (p @ vv.abs()) + h * out[:, hd].abs()
    return out, bound


def test_decoder_layers(mer, oracle, gpu):
    """Two layers of projections, q/k norm and rotation, append, attention,
    output projection, router and experts, over two sequences: prompts
    together, a chunk beside a single token, then single tokens."""
    say("decoder layers")
    route = importlib.import_module(mer.__name__ + ".routing").route_linear_gate_gpu
    dm, dff, heads, kv, d, page, n_exp, top = 256, 256, 8, 2, 64, 16, 8, 2
    dt, layers, eps = F16, 2, 1e-6
    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g)
    freq = inv_freq(d)
    pages = Pages(20, page, 2, 8)
    per_layer = []
    for l in range(layers):
        blobs = [make_expert(oracle, Q4, dm, dff, 300 + l * n_exp + e) for e in range(n_exp)]
        w = dict(qkv=rnd(dm, (heads + 2 * kv) * d) * dm ** -0.5, out=rnd(heads * d, dm) * (heads * d) ** -0.5,
                 qn=1 + 0.1 * rnd(d), kn=1 + 0.1 * rnd(d), gate=rnd(n_exp, dm) * dm ** -0.5)
        per_layer.append(dict(blobs=blobs, table=_table(blobs, gpu), dev={n: t.to(gpu) for n, t in w.items()}, **w,
                              cache=mer.PagedKvCache(20, page, kv, d, dt), k64=[torch.zeros(0, kv, d).double()] * 2,
                              v64=[torch.zeros(0, kv, d).double()] * 2))
    up = lambda t, kind=torch.int32: torch.tensor(t, dtype=kind, device=gpu)
    for step, counts in enumerate([(37, 20), (5, 1), (1, 1), (1, 1)]):
        first = list(pages.len)
        slots = up(pages.append(0, counts[0]) + pages.append(1, counts[1]), torch.int64)
        pos_cpu = torch.tensor([first[s] + i for s in (0, 1) for i in range(counts[s])], dtype=torch.int32)
        pos, start, lens, table = pos_cpu.to(gpu), up([0, counts[0], sum(counts)]), up(pages.len), pages.table.to(gpu)
        n = sum(counts)
        x = rnd(n, dm).to(gpu)
        for l, w in enumerate(per_layer):
            dev = w["dev"]
            row = (x * torch.rsqrt(x.pow(2).mean(1, keepdim=True) + eps)) @ dev["qkv"]
            q = row[:, :heads * d].view(n, heads, d)
            k, v = (row[:, (heads + i * kv) * d:(heads + (i + 1) * kv) * d].view(n, kv, d) for i in (0, 1))
            f = freq.to(gpu)
            q16, _ = mer.qk_norm_rope(q, None, pos, f, q_norm=dev["qn"], eps=eps, out_dtype=dt)
            mer.kv_append(w["cache"], k, v, slots, positions=pos, inv_freq=f, k_norm=dev["kn"], eps=eps)
            a = mer.paged_attention(w["cache"], q16, table, start, lens, max_q_len=max(counts),
                                    max_kv_len=max(pages.len))
            x1 = x + a.view(n, heads * d).float() @ dev["out"]
            ids, scores = route(dev["gate"], x1, top)
            y = mer.moe_forward(mer.WeightDtype.Q4_0, dm, dff, w["table"][1], ids, scores, x1, residual=True)
            mer.take_device_status()

            row64 = row.cpu().double()
            q64, _ = norm_rope64(row64[:, :heads * d].view(n, heads, d), w["qn"], pos_cpu, freq, eps, False)
            k64, _ = norm_rope64(row64[:, heads * d:(heads + kv) * d].view(n, kv, d), w["kn"], pos_cpu, freq, eps, False)
            v64 = row64[:, (heads + kv) * d:].view(n, kv, d)
            at = 0
            for s in (0, 1):
                rows = slice(at, at + counts[s])
                at += counts[s]
                w["k64"][s] = torch.cat([w["k64"][s], k64[rows]])
                w["v64"][s] = torch.cat([w["v64"][s], v64[rows]])
                want, bound = attention_bound(q64[rows], w["k64"][s], w["v64"][s], first[s], d ** -0.5, HALF[dt])
                err = (a[rows].cpu().double() - want).abs()
                assert (err <= bound + 2.0 ** -24).all(), f"step {step} layer {l} sequence {s}"
            logits = x1.cpu().double() @ w["gate"].double().T
            best = logits.gather(1, ids.cpu().long()).amin(1)
            rest = logits.scatter(1, ids.cpu().long(), -math.inf).amax(1)
            off = 2 * dm * HALF[F32] * (x1.cpu().double().abs() @ w["gate"].double().abs().T).amax(1)  # f32 dot products
            assert (best >= rest - off).all(), f"step {step} layer {l}: not the largest logits"
            sure = slice(0, 4)  # a few rows: the oracle's experts run on the CPU
            x1c = x1[sure].cpu().numpy()
            assert_ffn_close(y[sure].cpu().numpy(), x1c + _oracle_moe(oracle, Q4, w["blobs"], ids[sure].cpu().numpy(),
                                                                      scores[sure].cpu().numpy(), x1c, dm, dff),
                             f"step {step} layer {l}")
            x = y


def test_chunks_of_a_prompt(mer, gpu):
    """A prompt in chunks of every kind gives what the whole prompt gives: the
    same keys, bit by bit, and outputs within both sides' rounding."""
    say("chunks of a prompt")
    heads, kv, d, page, n = 8, 2, 128, 16, 700
    g = torch.Generator().manual_seed(4)
    row = torch.randn(n, (heads + 2 * kv) * d, generator=g).to(BF16).to(gpu)
    q, k, v = row[:, :heads * d].view(n, heads, d), row[:, heads * d:-kv * d].view(n, kv, d), row[:, -kv * d:].view(n, kv, d)
    freq = inv_freq(d).to(gpu)
    caches, outs = [], []
    for cuts in ([n], [1, 1, 3, 4, 27, 128, 300, 236]):
        cache = mer.PagedKvCache.wrap(*(torch.zeros(50, kv, page, d, dtype=BF16, device=gpu) for _ in range(2)))
        pages = Pages(50, page, 1, 44)
        out = torch.empty(n, heads, d, dtype=BF16, device=gpu)
        at = 0
        for c in cuts:
            part = slice(at, at + c)
            at += c
            slots = torch.tensor(pages.append(0, c), device=gpu)
            pos = torch.arange(part.start, part.stop, dtype=torch.int32, device=gpu)
            qr, _ = mer.qk_norm_rope(q[part], None, pos, freq)
            mer.kv_append(cache, k[part], v[part], slots, positions=pos, inv_freq=freq)
            mer.paged_attention(cache, qr, pages.table.to(gpu), torch.tensor([0, c], dtype=torch.int32, device=gpu),
                                torch.tensor([at], dtype=torch.int32, device=gpu), out=out[part])
        caches.append(cache)
        outs.append(out.cpu().double())
    assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)
    # Weights and outputs round once each on both sides; the scores' f32 error,
    # 2 (d / 16 + 8) half steps of sum |q_d k_d| scale <= 16, is 512 of them.
    ids = pages.table[0, :44].long().to(gpu)
    vv = caches[0].v[ids].transpose(1, 2).reshape(-1, kv, d)[:n].abs().cpu().double().cummax(0).values
    h = HALF[BF16]
    bound = 2 * (h + 512 * HALF[F32]) * vv.repeat_interleave(heads // kv, 1) + 2 * h * outs[0].abs() + 1e-30
    assert ((outs[0] - outs[1]).abs() <= bound).all()


def test_sequences_that_share_pages(mer, gpu):
    """Two sequences over the same first pages, one of them twice in the call."""
    b = Batch([(1, 100), (3, 100), (1, 100)], 4, 2, 64, 16, F16, seed=21)
    for i in (1, 2):
        b.table[i] = b.table[0]
        b.kk[i], b.vv[i] = b.kk[0], b.vv[0]
    b.check(b.run(mer, gpu))


# ---- graphs ----------------------------------------------------------------

class Step:
    """A step of the three operators over buffers that stay where they are."""

    def __init__(self, mer, gpu, counts, heads, kv, d, page, width, seed):
        self.mer, self.n, self.shape = mer, sum(counts), (heads, kv, d)
        self.counts, self.page = counts, page
        seqs = len(counts)
        g = torch.Generator().manual_seed(seed)
        self.g = g
        pool = seqs * width
        self.cache = mer.PagedKvCache.wrap(*(torch.randn(pool, kv, page, d, generator=g).to(BF16).to(gpu)
                                             for _ in range(2)))
        self.table = torch.randperm(pool, generator=g).to(torch.int32).view(seqs, width)
        zeros = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype, device=gpu)
        self.row = zeros(self.n, (heads + 2 * kv) * d)
        self.slots, self.pos = zeros(self.n, dtype=torch.int64), zeros(self.n, dtype=torch.int32)
        self.start = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=gpu)
        self.lens, self.dev_table = zeros(seqs, dtype=torch.int32), self.table.to(gpu)
        self.q16 = zeros(self.n, heads, d, dtype=BF16)
        self.out = zeros(self.n, heads, d, dtype=BF16)
        self.freq, self.kn = inv_freq(d).to(gpu), (1 + 0.1 * torch.randn(d, generator=g)).to(gpu)
        self.width = width

    def load(self, lens):
        """New inputs: sequences of these lengths, the new tokens included."""
        slots, pos = [], []
        for i, (c, l) in enumerate(zip(self.counts, lens)):
            for at in range(l - c, l):
                pos.append(at)
                slots.append(int(self.table[i, at // self.page]) * self.page + at % self.page)
        self.slots.copy_(torch.tensor(slots))
        self.pos.copy_(torch.tensor(pos, dtype=torch.int32))
        self.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        self.row.copy_(torch.randn(self.row.shape, generator=self.g))

    def run(self, out):
        heads, kv, d = self.shape
        row, n = self.row, self.n
        k, v = (row[:, (heads + i * kv) * d:(heads + (i + 1) * kv) * d].view(n, kv, d) for i in (0, 1))
        self.mer.qk_norm_rope(row[:, :heads * d].view(n, heads, d), None, self.pos, self.freq, q_out=self.q16)
        self.mer.kv_append(self.cache, k, v, self.slots, positions=self.pos, inv_freq=self.freq, k_norm=self.kn)
        self.mer.paged_attention(self.cache, self.q16, self.dev_table, self.start, self.lens, out=out,
                                 max_q_len=max(self.counts), max_kv_len=self.width * self.page)


def test_two_graphs_on_one_stream(mer, gpu):
    """A decode step and a step with a long chunk, captured on one stream and
    replayed in turn over new inputs and growing lengths, with eager work of
    other sizes between; every replay equals the eager call."""
    say("two attention graphs on one stream")
    s = torch.cuda.Stream(device=gpu)
    steps = [Step(mer, gpu, (1, 1, 1, 1), 8, 2, 128, 16, 160, 31), Step(mer, gpu, (200, 1, 33), 8, 2, 64, 16, 160, 32)]
    other = Step(mer, gpu, (1, 3), 4, 1, 128, 8, 40, 33)
    graphs = []
    with torch.cuda.stream(s):
        for st in [*steps, other]:
            st.load([300] * len(st.counts))
            st.run(st.out)  # grows the workspace before capture
    s.synchronize()
    for st in steps:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            st.run(st.out)
        graphs.append(gr)
    for rep in range(4):
        for i, st in enumerate(steps):
            st.load([201 + 577 * rep + 37 * j for j in range(len(st.counts))])
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                graphs[i].replay()
                other.run(other.out)
            torch.cuda.synchronize()
            got, keys = st.out.clone(), st.cache.k.clone()
            want = torch.zeros_like(got)
            with torch.cuda.stream(s):
                st.run(want)
            torch.cuda.synchronize()
            assert torch.isfinite(want).all() and torch.equal(got, want), f"replay {rep} of graph {i}"
            assert torch.equal(keys, st.cache.k)
    mer.take_device_status()
    del graphs
    mer.stream_release(s)


def test_graph_of_a_stream_without_workspace_is_refused(mer, gpu):
    """Growth under capture is an error, not an allocation, and the stream
    works afterwards."""
    s = torch.cuda.Stream(device=gpu)
    st = Step(mer, gpu, (1,), 8, 1, 128, 16, 100, 34)
    st.load([1500])
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=s):
        st.out.add_(0)  # the graph is not empty
        with pytest.raises(mer.GpuExpertDispatchError) as e:
            mer.paged_attention(st.cache, st.q16, st.dev_table, st.start, st.lens, out=st.out)
    assert e.value.kind == mer.GpuExpertDispatchErrorKind.PhysicalCapacity
    del gr
    with torch.cuda.stream(s):
        st.run(st.out)
    s.synchronize()
    assert st.out.abs().sum() > 0
    mer.stream_release(s)


def test_streams_and_threads(mer, gpu):
    """Four threads, two of them on one stream, each with calls of its own."""
    say("attention from four threads")
    shapes = [((1,), 16, 1, 128, 16, 300, 4700), ((1, 1, 2), 8, 2, 64, 16, 100, 1500),
              ((150, 20), 8, 1, 128, 16, 80, 1200), ((1,) * 40, 4, 2, 128, 8, 30, 200)]
    steps = [Step(mer, gpu, c, h, kv, d, page, w, 40 + i) for i, (c, h, kv, d, page, w, _) in enumerate(shapes)]
    want = []
    for st, sh in zip(steps, shapes):
        st.load([sh[-1]] * len(st.counts))
        st.run(st.out)
        torch.cuda.synchronize()
        want.append(st.out.clone())
    streams = [torch.cuda.Stream(device=gpu) for _ in range(3)]
    outs = [[torch.zeros_like(w) for _ in range(5)] for w in want]
    torch.cuda.synchronize()
    errors = []

    def work(i):
        try:
            with torch.cuda.device(gpu), torch.cuda.stream(streams[min(i, 2)]):
                for out in outs[i]:
                    steps[i].run(out)
        except BaseException as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=60)
    assert not any(t.is_alive() for t in threads) and not errors, errors
    torch.cuda.synchronize()
    for i in range(4):
        for out in outs[i]:
            assert torch.equal(out, want[i]), f"thread {i}"
    for s in streams:
        mer.stream_release(s)


# ---- refusals of the Python entry points -------------------------------------

def test_python_refusals(mer, gpu):
    z = lambda *s, dtype=F16: torch.zeros(*s, dtype=dtype, device=gpu)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)
    cache = mer.PagedKvCache(4, 16, 2, 64, F16)
    q, kv, pos, f = z(3, 4, 64), z(3, 2, 64), i32(0, 1, 2), inv_freq(64).to(gpu)
    slots = torch.arange(3, device=gpu)
    table, start, lens = i32(0, 1).view(1, 2), i32(0, 3), i32(3)
    att = lambda **kw: mer.paged_attention(**{**dict(cache=cache, q=q, block_table=table, q_start=start, kv_len=lens), **kw})
    rope = lambda **kw: mer.qk_norm_rope(**{**dict(q=q, k=kv, positions=pos, inv_freq=f), **kw})
    app = lambda **kw: mer.kv_append(**{**dict(cache=cache, k=kv, v=kv, slots=slots), **kw})
    att(), rope(), app()
    bad = (ValueError, TypeError, mer.InvalidLayout, mer.Misaligned)
    cases = [
        (att, dict(q=q.cpu())), (att, dict(q=z(3, 4, 64, dtype=BF16))), (att, dict(q=z(3, 4, 32))), (att, dict(q=z(3, 256))),
        (att, dict(q=z(3, 3, 64))), (att, dict(q=z(3, 64, 4).transpose(1, 2))), (att, dict(block_table=i32(0, 1))),
        (att, dict(block_table=table.long())), (att, dict(block_table=table.cpu())), (att, dict(q_start=i32(0, 1, 3))),
        (att, dict(kv_len=lens.long())), (att, dict(kv_len=i32(3, 3))), (att, dict(window=-1)), (att, dict(max_q_len=-1)),
        (att, dict(max_kv_len=-5)), (att, dict(scale=0.0)), (att, dict(scale=math.nan)), (att, dict(sinks=z(4))),
        (att, dict(sinks=z(3, dtype=F32))), (att, dict(out=z(3, 4, 64, dtype=F32))), (att, dict(out=z(2, 4, 64))),
        (att, dict(block_table=i32(0, 9, 1, 9).view(2, 2)[:, :1])), (att, dict(q=z(3 * 256 + 1)[1:].view(3, 4, 64))),
        (rope, dict(q=q.double())), (rope, dict(q=q.cpu())), (rope, dict(positions=pos.long())), (rope, dict(positions=None)),
        (rope, dict(positions=i32(0, 1))), (rope, dict(inv_freq=f.double())), (rope, dict(inv_freq=inv_freq(68).to(gpu))),
        (rope, dict(inv_freq=inv_freq(128).to(gpu))), (rope, dict(k=kv.float())), (rope, dict(k=z(2, 2, 64))),
        (rope, dict(k=None, k_norm=z(64, dtype=F32))), (rope, dict(q_norm=z(32, dtype=F32))),
        (rope, dict(out_dtype=torch.int32)), (rope, dict(q_out=z(3, 4, 32))), (rope, dict(q_norm=z(64, dtype=F32), eps=-1.0)),
        (rope, dict(q=z(3, 4, 60), k=z(3, 2, 60), inv_freq=None)),
        (app, dict(k=z(3, 1, 64))), (app, dict(v=kv.float())), (app, dict(slots=slots.int())), (app, dict(slots=slots[:2])),
        (app, dict(inv_freq=f)), (app, dict(k=kv.cpu())), (app, dict(slots=slots.cpu())),
    ]
    for i, (call, kw) in enumerate(cases):
        with pytest.raises(bad):
            call(**kw)
            pytest.fail(f"case {i}: {kw.keys()} was taken")
    for args in ((z(2, 2, 16, 64), z(2, 2, 8, 64)), (z(2, 2, 16, 64, dtype=F32),) * 2, (z(2, 16, 64),) * 2,
                 (z(2, 16, 2, 64).transpose(1, 2),) * 2):
        with pytest.raises((ValueError, TypeError)):
            mer.PagedKvCache.wrap(*args)
    mer.take_device_status()


def test_nothing_to_do(mer, gpu):
    """No tokens, no sequences."""
    z = lambda *s, dtype=F16: torch.zeros(*s, dtype=dtype, device=gpu)
    cache = mer.PagedKvCache(4, 16, 2, 64, F16)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=gpu)
    assert mer.paged_attention(cache, z(0, 4, 64), i32(2, 3), i32(3), i32(2)).shape == (0, 4, 64)
    assert (mer.paged_attention(cache, z(3, 4, 64), i32(0, 3), i32(1), i32(0)) == 0).all()
    assert (mer.paged_attention(cache, z(3, 4, 64), i32(1, 0), i32(2) + torch.tensor([0, 3], dtype=torch.int32, device=gpu),
                                i32(1) + 3) == 0).all()  # a table without pages holds no keys
    mer.kv_append(cache, z(0, 2, 64), z(0, 2, 64), torch.zeros(0, dtype=torch.int64, device=gpu))
    q, k = mer.qk_norm_rope(z(0, 4, 64), z(0, 2, 64), i32(0), inv_freq(64).to(gpu))
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    mer.take_device_status()


def test_a_scale_that_float32_rounds_to_zero_is_refused(mer, gpu):
    """Zero means the default scale at the entry point: a scale below float32's
    least number must not turn into it."""
    cache = mer.PagedKvCache(4, 16, 2, 64, F16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)
    q = torch.ones(1, 4, 64, dtype=F16, device=gpu)
    for scale in (0, 0.0, -0.0, 1e-50, -1e-300):
        with pytest.raises(ValueError):
            mer.paged_attention(cache, q, i32(0).view(1, 1), i32(0, 1), i32(1), scale=scale)
