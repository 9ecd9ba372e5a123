"""Calls whose pieces are counted by grids of other sizes, on one stream, eager
and replayed in turns: every answer has the bits of the first."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from test_gpu_attention import Batch, F16  # noqa: E402
from test_gpu_parity import say  # noqa: E402

pytestmark = pytest.mark.gpu


def test_grids_in_turns(mer, gpu):
    say("attention grids in turns")
    shapes = [([(1, 5000)], 8, 1, 128), ([(1, 4500), (1, 40)], 16, 2, 64), ([(1, 33000)], 9, 1, 256),
              ([(1, 90 + i % 150) for i in range(200)], 24, 6, 128), ([(1, 70 + i % 99) for i in range(150)], 16, 8, 64),
              ([(5, 4000)], 16, 4, 128), ([(200, 900)], 4, 1, 128)]
    s = torch.cuda.Stream(device=gpu)
    calls = []
    for i, (seqs, heads, kv, d) in enumerate(shapes):
        b = Batch(seqs, heads, kv, d, 16, F16, seed=90 + i)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)
        args = (mer.PagedKvCache.wrap(b.k.to(gpu), b.v.to(gpu)), b.q.to(gpu), b.table.to(gpu), i32(b.start),
                i32([l for _, l in seqs]))
        out = torch.zeros_like(args[1])
        run = lambda out=out, args=args, seqs=seqs: mer.paged_attention(
            *args, max_q_len=max(n for n, _ in seqs), max_kv_len=max(l for _, l in seqs), out=out)
        calls.append((b, run, out))
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _, run, _ in calls:
            run()
    torch.cuda.synchronize()
    want = [out.clone() for _, _, out in calls]
    for (b, _, _), w in zip(calls, want):
        got = w.cpu()
        b.check(got)
    graphs = []
    for _, run, _ in calls:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            run()
            run()
        graphs.append(gr)
    order = [0, 3, 3, 1, 4, 0, 2, 6, 5, 4, 2, 2, 5, 1, 0, 6, 3]
    for rep, i in enumerate(order * 2):
        _, run, out = calls[i]
        with torch.cuda.stream(s):
            out.zero_()
            graphs[i].replay() if rep % 3 else run()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), f"call {i}, turn {rep}"
    mer.take_device_status()
    del graphs
    mer.stream_release(s)
