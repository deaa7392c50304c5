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
