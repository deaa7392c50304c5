"""Penalties, biases and masks on logits and the choice of the best tokens, against plain numpy.

The rules are single fp32 operations in a fixed order, so processed logits are compared for equality.
Log-probabilities are compared with 64 bits: x - max is one rounding (2^-24 of values up to 64), the
exponents of the terms that count are below 32 in size and rounded once (2e-6 of a term), and the sum and
its logarithm add a few 2^-24: 1e-5 in all."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LOGPROB_TOL = 1e-5


def plain_rules(x, vocab, history=None, history_len=None, repetition=None, frequency=None, presence=None, no_repeat_ngram=0,
                bias=None, bias_row=None, mask=None, mask_row=None):
    x = x.astype(np.float32)
    rows = x.shape[0]
    one = np.float32
    for r in range(rows):
        y = x[r]
        banned = np.zeros(vocab, bool)
        if history is not None:
            h = history[r]
            if history_len is not None:
                h = h[:max(0, min(len(h), history_len[r]))]
            rep = one(1) if repetition is None else repetition[r]
            fr = one(0) if frequency is None else frequency[r]
            pr = one(0) if presence is None else presence[r]
            tok, n = np.unique(h[(h >= 0) & (h < vocab)], return_counts=True)
            z = y[tok]
            with np.errstate(all="ignore"):
                z = np.where(z > 0, z / rep, z * rep).astype(np.float32)
                y[tok] = z - (fr * n.astype(np.float32) + pr)
            m = no_repeat_ngram
            if m > 1:
                for i in range(m - 1, len(h)):
                    if np.array_equal(h[i - m + 1:i], h[len(h) - m + 1:]) and 0 <= h[i] < vocab:
                        banned[h[i]] = True
        if bias is not None:
            b = 0 if bias_row is None else bias_row[r]
            if 0 <= b < len(bias):
                with np.errstate(all="ignore"):
                    y += bias[b][:vocab]
        if mask is not None:
            b = 0 if mask_row is None else mask_row[r]
            if 0 <= b < len(mask):
                bits = np.unpackbits(np.ascontiguousarray(mask[b]).view(np.uint8), bitorder="little")[:vocab]
                banned |= bits == 0
        y[banned] = -np.inf
    return x


def plain_topk(x, k):
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    ids = np.full((len(x), k), -1, np.int32)
    lp = np.full((len(x), k), -np.inf)
    for r, y in enumerate(x):
        order = np.argsort(-(y + 0.0), kind="stable")[:k]
        order = order[y[order] > -np.inf]
        if not len(order):
            continue
        m = y.max()
        ids[r, :len(order)] = order
        if m == np.inf:
            lp[r, :len(order)] = np.where(y[order] == np.inf, -np.log((y == np.inf).sum()), -np.inf)
        else:
            lp[r, :len(order)] = y[order] - m - np.log(np.exp(y - m).sum())
    return ids, lp


def make(rng, rows, vocab, hist=0, ngram=0, n_bias=0, n_mask=0):
    kw = {"no_repeat_ngram": ngram}
    if hist:
        h = rng.integers(0, max(1, min(vocab, 7)), (rows, hist)).astype(np.int32)
        h[rng.random((rows, hist)) < 0.3] = -1
        h[rng.random((rows, hist)) < 0.2] = vocab - 1
        h[rng.random((rows, hist)) < 0.1] = vocab  # not a token
        kw["history"], kw["history_len"] = h, rng.integers(-1, hist + 3, rows).astype(np.int32)
        kw["repetition"] = (1 + rng.random(rows)).astype(np.float32)
        kw["frequency"] = rng.random(rows).astype(np.float32)
        kw["presence"] = rng.random(rows).astype(np.float32)
    if n_bias:
        b = rng.standard_normal((n_bias, vocab)).astype(np.float32)
        b[:, rng.integers(0, vocab, 3)] = -np.inf
        kw["bias"], kw["bias_row"] = b, rng.integers(-1, n_bias + 1, rows).astype(np.int32)
    if n_mask:
        m = rng.integers(-2**31, 2**31, (n_mask, (vocab + 31) // 32)).astype(np.int32)
        m[0] = 0  # allows nothing
        kw["mask"], kw["mask_row"] = m, rng.integers(-1, n_mask + 1, rows).astype(np.int32)
    return kw


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def rules_of(kw):
    from vokra_b200 import logits
    return logits.LogitsRules(**{k: v if isinstance(v, int) else dev(v) for k, v in kw.items()})


def check_topk(x, k, ids, lp):
    want_ids, want_lp = plain_topk(x, k)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    got = lp.cpu().numpy()
    assert not np.isnan(got).any()
    fin = np.isfinite(want_lp)
    assert np.array_equal(fin, np.isfinite(got)) and np.array_equal(got[~fin], want_lp[~fin].astype(np.float32))
    assert np.max(np.abs(got[fin] - want_lp[fin]), initial=0.0) <= LOGPROB_TOL


SHAPES = [(1, 1), (2, 3), (3, 31), (2, 33), (1, 1023), (3, 4095), (2, 4096), (2, 4097), (5, 8193), (4, 51866), (130, 1000)]


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_process_and_topk(ctx, rows, vocab, dtype):
    from vokra_b200 import logits
    rng = np.random.default_rng(rows * 100003 + vocab)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(dtype)
    for hist, ngram, n_bias, n_mask in [(0, 0, 0, 0), (40, 0, 0, 0), (40, 2, 2, 0), (300, 3, 1, 3), (0, 0, 3, 2)]:
        kw = make(rng, rows, vocab, hist, ngram, n_bias, n_mask)
        want = plain_rules(x, vocab, **kw)
        rules = rules_of(kw)
        got = logits.process(ctx, dev(x), rules).cpu().numpy()
        assert got.dtype == x.dtype and np.array_equal(got, want.astype(dtype))
        for k in (1, 5, 64):
            check_topk(want, k, *logits.topk(ctx, dev(x), k, rules))


def test_no_rules_is_a_copy_and_a_plain_topk(ctx):
    from vokra_b200 import logits
    rng = np.random.default_rng(3)
    x = rng.standard_normal((7, 5000)).astype(np.float32)
    assert np.array_equal(logits.process(ctx, dev(x)).cpu().numpy(), x)
    check_topk(x, 9, *logits.topk(ctx, dev(x), 9))


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("off", [0, 1, 2, 3, 5])
def test_rows_at_any_address_and_in_place(ctx, dtype, off):
    """Rows that start anywhere inside longer ones; what lies around them stays as it is."""
    from vokra_b200 import logits
    rng = np.random.default_rng(off)
    rows, vocab = 5, 4999
    big = (rng.standard_normal((rows, vocab + 11)) * 3).astype(dtype)
    kw = make(rng, rows, vocab, 50, 2, 2, 2)
    want = plain_rules(big[:, off:off + vocab], vocab, **kw)
    rules = rules_of(kw)
    x = dev(big)
    check_topk(want, 7, *logits.topk(ctx, x[:, off:off + vocab], 7, rules))
    other = dev(np.zeros((rows, vocab + 6), dtype))
    logits.process(ctx, x[:, off:off + vocab], rules, out=other[:, 4:4 + vocab])
    assert np.array_equal(other.cpu().numpy()[:, 4:4 + vocab], want.astype(dtype))
    assert not other[:, :4].any() and not other[:, 4 + vocab:].any()
    logits.process(ctx, x[:, off:off + vocab], rules, out=x[:, off:off + vocab])
    big[:, off:off + vocab] = want.astype(dtype)
    assert np.array_equal(x.cpu().numpy(), big)


@pytest.mark.parametrize("vocab", [10, 4096, 9000, 51866])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("k", [1, 3, 64])
def test_ties_go_to_the_lower_id(ctx, vocab, dtype, k):
    from vokra_b200 import logits
    rng = np.random.default_rng(vocab + k)
    x = np.zeros((6, vocab), dtype)
    x[1] = rng.integers(0, 3, vocab)          # many of each value
    x[2, :] = -np.inf
    x[2, rng.integers(0, vocab, 20)] = 1.0    # few left
    x[3] = -0.0
    x[3, ::2] = 0.0
    x[4] = np.arange(vocab) // 7              # ascending
    x[5] = -(np.arange(vocab) // 7)           # descending
    check_topk(x, k, *logits.topk(ctx, dev(x), k))


def test_rows_with_nothing_left_infinities_and_nan(ctx):
    from vokra_b200 import logits
    rng = np.random.default_rng(5)
    vocab = 6000
    x = rng.standard_normal((9, vocab)).astype(np.float32)
    x[0] = -np.inf
    x[1, 17] = np.inf
    x[2, [5, 4100, 5999]] = np.inf
    x[3] = np.nan
    x[4, ::2] = np.nan
    x[5] = np.finfo(np.float32).min
    x[6] = np.finfo(np.float32).max
    x[7, 1:] = -np.inf
    mask = np.full((1, (vocab + 31) // 32), -1, np.int32)
    mask[0, 0] &= ~(1 << 17)
    x[8, 17] = np.nan                         # masked: it counts for nothing
    row = np.full(9, -1, np.int32)
    row[8] = 0
    kw = {"mask": mask, "mask_row": row}
    want = plain_rules(x, vocab, **kw)
    got = logits.process(ctx, dev(x), rules_of(kw)).cpu().numpy()
    assert np.array_equal(got, want, equal_nan=True)
    ids, lp = logits.topk(ctx, dev(x), 6, rules_of(kw))
    check_topk(want, 6, ids, lp)
    assert (ids[0] == -1).all() and (ids[3] == -1).all() and ids[7].tolist() == [0, -1, -1, -1, -1, -1]
    assert abs(float(lp[7, 0])) <= LOGPROB_TOL and abs(float(lp[1, 0])) <= LOGPROB_TOL


@pytest.mark.parametrize("left", [1, 31, 100, 700, 5000])
@pytest.mark.parametrize("k", [1, 8, 32, 40, 64])
def test_masks_that_leave_a_stretch_of_the_vocabulary(ctx, left, k):
    """All candidates in a few neighbouring threads, in one window or over the border of two."""
    from vokra_b200 import logits
    rng = np.random.default_rng(left + k)
    vocab, rows = 20000, 4
    bits = np.zeros((rows, (vocab + 31) // 32 * 32), np.uint8)
    for r, first in enumerate([0, 4000, 12288, vocab - left]):
        bits[r, first:first + left] = 1
    mask = np.packbits(bits, axis=1, bitorder="little").view(np.int32)
    kw = {"mask": mask, "mask_row": np.arange(rows, dtype=np.int32)}
    for x in ((rng.standard_normal((rows, vocab)) * 3).astype(np.float32), np.zeros((rows, vocab), np.float16)):
        check_topk(plain_rules(x, vocab, **kw), k, *logits.topk(ctx, dev(x), k, rules_of(kw)))


def test_all_rows_masked_and_no_rows(ctx):
    import torch
    from vokra_b200 import logits
    x = np.random.default_rng(0).standard_normal((3, 300)).astype(np.float32)
    rules = rules_of({"mask": np.zeros((1, 10), np.int32)})
    assert (logits.process(ctx, dev(x), rules) == -np.inf).all()
    ids, lp = logits.topk(ctx, dev(x), 4, rules)
    assert (ids == -1).all() and (lp == -np.inf).all()
    none = torch.empty(0, 300, device="cuda")
    assert logits.process(ctx, none).shape == (0, 300) and logits.topk(ctx, none, 2)[0].shape == (0, 2)


def test_long_history_and_many_rows(ctx):
    """A history longer than the block, counts above 255, and rows that each split over several blocks, twice
    (the arrival counters of the first call are at rest again)."""
    from vokra_b200 import logits
    rng = np.random.default_rng(8)
    rows, vocab = 3, 40000
    x = (rng.standard_normal((rows, vocab)) * 2).astype(np.float32)
    h = rng.integers(0, 50, (rows, 30000)).astype(np.int32)
    kw = {"history": h, "repetition": np.full(rows, 1.2, np.float32), "frequency": np.full(rows, 0.01, np.float32), "no_repeat_ngram": 4}
    want = plain_rules(x, vocab, **kw)
    rules = rules_of(kw)
    assert np.array_equal(logits.process(ctx, dev(x), rules).cpu().numpy(), want)
    for _ in range(2):
        check_topk(want, 33, *logits.topk(ctx, dev(x), 33, rules))


def test_runs_on_the_stream_of_the_context(ctx):
    import torch
    from vokra_b200 import logits, ops
    rng = np.random.default_rng(9)
    x = rng.standard_normal((40, 51866)).astype(np.float32)
    st = torch.cuda.Stream()
    c = ops.Context(0)
    c.set_stream(st.cuda_stream)
    with torch.cuda.stream(st):
        t = dev(x) * 2.0
        ids, lp = logits.topk(c, t, 3)
        out = logits.process(c, t)
    st.synchronize()
    check_topk(x * np.float32(2), 3, ids, lp)
    assert np.array_equal(out.cpu().numpy(), x * np.float32(2))


def test_refusals(ctx):
    import torch
    from vokra_b200 import _lib, logits
    from vokra_b200.ops import VkbError
    x = torch.zeros(2, 100, device="cuda")
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    bad = [
        lambda: logits.topk(ctx, x, 0), lambda: logits.topk(ctx, x, 65), lambda: logits.process(ctx, x.double()),
        lambda: logits.process(ctx, x.cpu()), lambda: logits.process(ctx, x[0]), lambda: logits.process(ctx, x.t()),
        lambda: logits.process(ctx, x, out=f(2, 99)), lambda: logits.process(ctx, x, out=x.half()),
        lambda: logits.topk(ctx, x, 2, ids=i(2, 3)), lambda: logits.process(ctx, x[:1].expand(2, 100)),
        lambda: logits.process(ctx, x, logits.LogitsRules(history=i(1, 5))),
        lambda: logits.process(ctx, x, logits.LogitsRules(history=i(1, 5).expand(2, 5))),
        lambda: logits.process(ctx, x, logits.LogitsRules(bias=f(1, 99))),
        lambda: logits.process(ctx, x, logits.LogitsRules(mask=i(1, 3))),
        lambda: logits.process(ctx, x, logits.LogitsRules(mask=i(1, 4), mask_row=i(1))),
        lambda: logits.LogitsRules(repetition=i(2)), lambda: logits.LogitsRules(history=f(2, 3)),
        lambda: logits.process(ctx, x, logits.LogitsRules(no_repeat_ngram=-1)),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(VkbError) as e:
            call()
        assert e.value.code == _lib.ERROR_INVALID_ARGUMENT, n
    L = _lib.load()
    p = x.data_ptr()
    assert L.vkb_logits_process(ctx.h, p, _lib.DT_F16X2, 2, 100, 100, None, p, 100) == _lib.ERROR_UNSUPPORTED_OP
    assert L.vkb_logits_process(ctx.h, p, _lib.DT_F32, 2, 100, 99, None, p, 99) == _lib.ERROR_INVALID_ARGUMENT
    assert L.vkb_logits_process(ctx.h, p + 2, _lib.DT_F32, 1, 10, 10, None, p, 10) == _lib.ERROR_INVALID_ARGUMENT
    assert L.vkb_logits_topk(ctx.h, None, _lib.DT_F32, 2, 100, 100, None, 1, p, p) == _lib.ERROR_INVALID_ARGUMENT
    assert L.vkb_logits_topk(None, p, _lib.DT_F32, 2, 100, 100, None, 1, p, p) == _lib.ERROR_INVALID_ARGUMENT


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("hist", [60, 2100])
@pytest.mark.parametrize("what", ["repetition", "presence", "frequency"])
def test_penalties_that_raise(ctx, dtype, hist, what):
    """Penalties below their neutral value lift tokens into the k best."""
    import torch
    from vokra_b200 import logits
    rng = np.random.default_rng(hist)
    rows, vocab, k = 3, 5003, 9
    x = (rng.standard_normal((rows, vocab)) - 3).astype(dtype)
    kw = dict(history=rng.integers(0, vocab, (rows, hist)).astype(np.int32), no_repeat_ngram=2,
              **{what: np.full(rows, 0.01 if what == "repetition" else -2.5, np.float32)})
    ids, lp = logits.topk(ctx, torch.from_numpy(x).cuda(), k, rules_of(kw))
    torch.cuda.synchronize()
    y = plain_rules(x, vocab, **kw)
    want, _ = plain_topk(y, k)
    assert np.isin(want[0], kw["history"][0]).any()  # the case is what it says
    check_topk(y, k, ids, lp)


def test_offsets_above_32_bits_and_more_rows_than_a_launch(ctx):
    import torch
    from vokra_b200 import logits
    rng = np.random.default_rng(41)
    rows, vocab, k = 33000, 66001, 3
    x = torch.zeros(rows, vocab, dtype=torch.float16, device="cuda")
    assert x.numel() > 2**31
    some = [0, 32767, 32768, rows - 1]
    y = rng.standard_normal((len(some), vocab)).astype(np.float16)
    for r, row in zip(some, y):
        x[r] = dev(row)
    history = torch.full((rows, 2), -1, dtype=torch.int32, device="cuda")
    history[some] = dev(np.stack([np.argsort(-row.astype(np.float32), kind="stable")[:2] for row in y]).astype(np.int32))
    rules = logits.LogitsRules(history=history, presence=torch.full((rows,), 9.0, device="cuda"))
    ids, lp = logits.topk(ctx, x, k, rules)
    want = plain_rules(y, vocab, history=history[some].cpu().numpy(), presence=np.full(len(some), 9, np.float32))
    check_topk(want, k, ids[some], lp[some])
    logits.process(ctx, x, rules, out=x)
    assert np.array_equal(x[some].cpu().numpy(), want.astype(np.float16))
