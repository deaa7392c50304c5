"""Graphs that were recorded before their context's scratch grew."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_a_recorded_step_outlives_larger_calls(ctx):
    """Calls with scratch of their own size, recorded; then larger eager calls, whose scratch is another one; then the
    graph again, on new values, with the old scratch's place in memory asked for by others."""
    import torch
    from vokra_b200 import logits, ops
    from vokra_b200.blockkv import Batch, BlockKvCache, PagePool, PageState
    rng = np.random.default_rng(1)
    n_seq, heads, group, d, vocab, n_pages, ld = 5, 2, 2, 64, 3001, 400, 60
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        own = ops.Context(0)
        new = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
        status = new(1, dtype=torch.int32)
        cache = BlockKvCache.empty(own, 1, heads, d, n_pages)
        for t in (cache.k, cache.v):
            t.copy_(torch.from_numpy(rng.integers(-127, 128, t.shape).astype(np.int8)))
        for t in (cache.k_scale, cache.v_scale):
            t.copy_(torch.from_numpy((rng.random(t.shape) * 0.05).astype(np.float32)))
        pages = cache.pages(status)
        a, b, c = (PageState.empty(n_seq, ld, n_pages) for _ in range(3))
        grow = torch.from_numpy(rng.integers(1, ld * 16, n_seq).astype(np.int32)).cuda()
        start = torch.arange(n_seq + 1, dtype=torch.int32, device="cuda")
        q, x = new(n_seq, heads * group, d), new(n_seq, vocab)
        y, ids, lp = torch.empty_like(q), new(n_seq, 4, dtype=torch.int32), new(n_seq, 4)

        def step():
            pages.advance(a, b, None, grow)
            pages.compact(b, c)
            cache.attention(0, Batch(start, c.len, c.table, n_seq, 1, status), q, 0.125, out=y)
            logits.topk(own, x, 4, ids=ids, logprobs=lp)

        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    from vokra_b200 import _lib
    held = _lib.load().vkb_context_workspace_bytes(own.h)

    def many_rows():
        wide = BlockKvCache.empty(own, 1, 1, 128, 4)
        table = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
        one = Batch(torch.tensor([0, 9], dtype=torch.int32, device="cuda"), torch.tensor([9], dtype=torch.int32, device="cuda"), table, 9, 9)
        wide.attention(0, one, torch.zeros(9, 2, 128, dtype=torch.float16, device="cuda"))

    def many_pages():
        n = 5_000_000
        big = PagePool(own, [torch.zeros(1, n, 1, dtype=torch.uint8, device="cuda")], new(1, dtype=torch.int32))
        big.advance(PageState.empty(1, 2, n), PageState.empty(1, 2, n))

    with torch.cuda.stream(stream):
        for larger in (many_rows, many_pages):
            larger()
            assert _lib.load().vkb_context_workspace_bytes(own.h) > held
            held = _lib.load().vkb_context_workspace_bytes(own.h)
            noise = [torch.full((1 << 20,), float("nan"), device="cuda") for _ in range(40)]
            for t in (q, x):
                t.copy_(torch.from_numpy(rng.standard_normal(t.shape).astype(np.float32)))
            out = (y, ids, lp, b.table, b.len, b.refs, c.table, c.len, c.refs)
            for t in out:
                t.fill_(7)
            graph.replay()
            got = [t.clone() for t in out]
            for t in out:
                t.fill_(8)
            step()
            assert all(torch.equal(g, t) for g, t in zip(got, out))
            assert all(bool(t.isnan().all()) for t in noise)
            del noise
    assert int(status) == 0 and int(c.len.sum()) == int(grow.sum())
    del graph
