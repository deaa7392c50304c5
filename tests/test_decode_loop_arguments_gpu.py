"""What the decode loop's calls make of tensors that are parts of others, on another GPU, or of the wrong shape."""
import numpy as np
import pytest

from tests.test_logits_gpu import check_topk, dev, plain_rules

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", ["none", "within", "beyond"])
def test_history_that_is_part_of_longer_rows(ctx, lens):
    """Only the part counts, whatever the lengths say: what lies behind it is other data."""
    from vokra_b200 import logits
    rng = np.random.default_rng(1)
    rows, vocab, cols = 4, 700, 9
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    whole = rng.integers(0, vocab, (rows + 1, 30)).astype(np.int32)
    n = {"none": None, "within": rng.integers(0, cols + 1, rows), "beyond": np.array([cols + 1, cols + 5, 30, 1 << 30])}[lens]
    n = None if n is None else n.astype(np.int32)
    kw = {"presence": np.full(rows, 3, np.float32), "no_repeat_ngram": 2}
    rules = logits.LogitsRules(history=dev(whole)[:rows, 4:4 + cols], history_len=None if n is None else dev(n),
                               presence=dev(kw["presence"]), no_repeat_ngram=2)
    want = plain_rules(x, vocab, history=whole[:rows, 4:4 + cols], history_len=n, **kw)
    assert np.array_equal(logits.process(ctx, dev(x), rules).cpu().numpy(), want)
    check_topk(want, 5, *logits.topk(ctx, dev(x), 5, rules))


def test_tensors_of_another_gpu(ctx):
    """A stand-in for a context of GPU 1 meets tensors of GPU 0: refused before anything is launched."""
    import types
    import torch
    from vokra_b200 import _lib, blockkv, logits
    away = types.SimpleNamespace(h=ctx.h, device=1)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    x, q, kv = (torch.zeros(*s, device="cuda") for s in ((2, 100), (1, 4, 64), (1, 2, 64)))
    cache = blockkv.BlockKvCache.empty(ctx, 1, 2, 64, 4)
    pages = cache.pages(i(1))
    a, b = blockkv.PageState.empty(3, 4, 4), blockkv.PageState.empty(3, 4, 4)
    batch = blockkv.Batch(i(2), i(1), i(1, 4), 1, 1)
    cache.attention(0, batch, q)  # (as it should be)
    arenas = (cache.k, cache.v, cache.k_scale, cache.v_scale)
    with pytest.raises(blockkv.VkbError, match="GPU 0, the context is on GPU 1"):
        logits.LogitsRules(presence=torch.zeros(2, device="cuda")).check(2, 100, away.device)
    cache.ctx = pages.ctx = away
    launches = ctx.launch_count
    for n, call in enumerate([
        lambda: logits.process(away, x), lambda: logits.topk(away, x, 2), lambda: blockkv.BlockKvCache(away, *arenas),
        lambda: blockkv.PagePool(away, [cache.k], i(1)), lambda: cache.attention(0, batch, q), lambda: cache.append(0, batch, kv, kv),
        lambda: cache.read(0, batch), lambda: pages.advance(a, b), lambda: pages.compact(a, b),
    ]):
        with pytest.raises(blockkv.VkbError, match="GPU 0, the context is on GPU 1") as e:
            call()
        assert e.value.code == _lib.ERROR_INVALID_ARGUMENT, n
    assert ctx.launch_count == launches


def test_more_refusals(ctx):
    """Shapes that ended in errors of another kind, and a scale whose products leave fp32."""
    import torch
    from vokra_b200 import _lib, blockkv
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = blockkv.BlockKvCache.empty(ctx, 1, 2, 64, 4)
    batch = blockkv.Batch(i(2), i(1), i(1, 4), 1, 1)
    q = torch.zeros(1, 4, 64, device="cuda")
    for n, call in enumerate([
        lambda: cache.attention(0, batch, q[0, 0]), lambda: cache.attention(0, batch, q[0, 0, 0]), lambda: cache.attention(0, batch, q[None]),
        lambda: cache.append(0, batch, q[0, 0], q[0, 0]), lambda: cache.attention(0, batch, q, scale=2.5e38),
        lambda: blockkv.PagePool(ctx, [], i(1)), lambda: blockkv.PagePool(ctx, [torch.zeros(2, 0, 4, device="cuda")], i(1)),
        lambda: blockkv.PagePool(ctx, [torch.zeros(8, device="cuda")], i(1)),
    ]):
        with pytest.raises(blockkv.VkbError) as e:
            call()
        assert e.value.code == _lib.ERROR_INVALID_ARGUMENT, n
    cache.attention(0, batch, q, scale=1.9e38)
