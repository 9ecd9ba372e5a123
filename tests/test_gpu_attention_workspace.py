"""An attention call that is no larger than an earlier one on its stream leaves
the stream's workspace where it is, into however many chunks its keys are cut,
so graphs captured on the stream stay valid."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_gpu_attention import BF16, HALF, attention64  # noqa: E402
from test_gpu_parity import say  # noqa: E402

pytestmark = pytest.mark.gpu


class Call:
    """One sequence of n new tokens over `keys` keys, in tensors that stay where they are."""

    def __init__(self, mer, gpu, n, keys, heads, kv, d, page, seed):
        g = torch.Generator().manual_seed(seed)
        pages = -(-keys // page)
        rnd = lambda *s: torch.randn(*s, generator=g).to(BF16).to(gpu)
        self.mer, self.n, self.keys = mer, n, keys
        self.cache = mer.PagedKvCache.wrap(rnd(pages, kv, page, d), rnd(pages, kv, page, d))
        i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)
        self.table = torch.randperm(pages, generator=g).to(torch.int32).view(1, pages).to(gpu)
        self.start, self.lens = i32(0, n), i32(keys)
        self.q, self.out = rnd(n, heads, d), torch.zeros(n, heads, d, dtype=BF16, device=gpu)

    def run(self, out=None):
        self.mer.paged_attention(self.cache, self.q, self.table, self.start, self.lens, max_q_len=self.n,
                                 max_kv_len=self.keys, out=self.out if out is None else out)


@pytest.mark.parametrize("heads,kv,d", [(16, 4, 128), (8, 8, 64), (8, 1, 256)])
def test_smaller_calls_keep_the_workspace(mer, gpu, heads, kv, d):
    say(f"attention workspace after smaller calls {heads}/{kv} heads of {d}")
    keys, page = 4096, 64
    calls = [Call(mer, gpu, n, keys, heads, kv, d, page, 50 + n) for n in (4096, 1, 2048, 1024, 512, 300, 128, 20, 5)]
    large, decode, small = calls[0], calls[1], calls[2:]
    news = [torch.randn(decode.q.shape, generator=torch.Generator().manual_seed(i)).to(BF16).to(gpu) for i in range(4)]
    want = torch.zeros_like(decode.out)
    s = torch.cuda.Stream(device=gpu)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        large.run()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info(gpu)[0]
    with torch.cuda.stream(s):
        decode.run()
    torch.cuda.synchronize()
    assert torch.cuda.mem_get_info(gpu)[0] == free, "a single token made the workspace grow"
    # calls of other sizes may be captured without a run of their own
    graphs = []
    for c in (decode, small[3]):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            c.run()
        graphs.append(gr)
    for i, new in enumerate(news):
        torch.cuda.synchronize()
        free = torch.cuda.mem_get_info(gpu)[0]
        with torch.cuda.stream(s):
            for c in small:
                c.run()
            decode.q.copy_(new)
        torch.cuda.synchronize()
        assert torch.cuda.mem_get_info(gpu)[0] == free, "a smaller call made the workspace grow"
        graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        chunk = small[3].out.clone()
        with torch.cuda.stream(s):
            decode.run(want)
            small[3].run()
        torch.cuda.synchronize()
        assert torch.isfinite(want).all() and torch.equal(decode.out, want), f"replay {i}"
        assert torch.equal(chunk, small[3].out), f"replay {i} of the chunk"
    # and the last answer is the right one
    flat = lambda t: t[decode.table[0].long()].transpose(1, 2).reshape(-1, kv, d)[:keys].cpu().double()
    exact, bound = attention64(decode.q.cpu().double(), flat(decode.cache.k), flat(decode.cache.v), keys - 1, 0, None,
                               d ** -0.5, HALF[BF16])
    assert ((want.cpu().double() - exact).abs() <= bound + 1e-30).all()
    mer.take_device_status()
    del graphs
    mer.stream_release(s)


def test_a_full_device_runs_fewer_chunks(mer, gpu):
    """A device that refuses what a chunk reserves still answers it, and the
    buffer that a captured decode step points to stays where it is."""
    say("attention workspace refused")
    heads, kv, d, keys = 16, 4, 128, 8192
    decode, chunk, less = (Call(mer, gpu, n, keys, heads, kv, d, 64, 70 + n) for n in (1, 1200, 300))  # the chunk reserves 256 MiB
    want, got = torch.zeros_like(chunk.out), torch.zeros_like(decode.out)
    s, other = torch.cuda.Stream(device=gpu), torch.cuda.Stream(device=gpu)
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        chunk.run(want)  # in chunks
        decode.run(got)
    with torch.cuda.stream(s):
        decode.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        decode.run()
    held = []
    for step in (8 << 30, 1 << 30, 128 << 20):  # until less than 256 MiB are left
        while torch.cuda.mem_get_info(gpu)[0] > step + (100 << 20):
            held.append(torch.empty(step, dtype=torch.uint8, device=gpu))
    free = torch.cuda.mem_get_info(gpu)[0]
    assert free < 250 << 20
    try:
        with torch.cuda.stream(s):
            for _ in range(2):
                chunk.run()
        torch.cuda.synchronize()
        # (the runtime may give back memory of its own when it refuses)
        assert torch.cuda.mem_get_info(gpu)[0] >= free, "nothing was there to take"
        decode.out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
    finally:
        held.clear()
        torch.cuda.empty_cache()
    assert torch.equal(decode.out, got)
    # with the memory back, a smaller call that would have reserved more than there is leaves the buffer, too
    free = torch.cuda.mem_get_info(gpu)[0]
    with torch.cuda.stream(s):
        less.run()
    torch.cuda.synchronize()
    assert torch.cuda.mem_get_info(gpu)[0] == free, "a smaller call moved the workspace"
    decode.out.zero_()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(decode.out, got)
    # both sides round the weights and the output once; 512 half steps of f32 cover the scores' sums
    h = HALF[BF16]
    flat = chunk.cache.v[chunk.table[0].long()].transpose(1, 2).reshape(-1, kv, d)[:keys]
    most = flat.float().abs().amax(0).repeat_interleave(heads // kv, 0)
    assert ((chunk.out.float() - want.float()).abs() <= 2 * (h + 512 * HALF[torch.float32]) * most + 2 * h * want.float().abs()).all()
    assert chunk.out.float().abs().sum() > 0
    mer.take_device_status()
    del graph
    for st in (s, other):
        mer.stream_release(st)
