"""Attention over the 8-bit cache where blocks, weights or rows of q differ by many powers of two, against 64 bits.

The measure is a row's own: the sum of its weights times the largest |v| of each key that it sees. With 32-bit rows
a weight is known to 4.4e-5 of itself (2e-4 of values up to 4.5 in test_blockkv_gpu.py); with 16-bit rows it is
rounded to 2^-11 of itself, the output too, and a score is off by less than 1e-4 for these q: 1.2e-3."""
import numpy as np
import pytest

from tests.test_blockkv_gpu import BLOCK, Plain, batch_of, cache_of, dev, filled, tables

pytestmark = pytest.mark.gpu

REL = {"float32": 4.4e-5, "float16": 1.2e-3}
# rows a stream, query heads of a KV head: 8 rows of a tile, 16 rows of a tile, tensor-core tiles of 128 rows
FORMS = [("float32", 6, 1), ("float32", 40, 2), ("float16", 6, 1), ("float16", 6, 4), ("float16", 90, 2)]


def exact(plain, table, start, lens, q, scale):
    """(out, measure [rows, heads], largest |v| seen [rows, heads]) in 64 bits; a row without keys is 0."""
    heads, group = plain.k.shape[1], q.shape[1] // plain.k.shape[1]
    out, size, most = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    for s, n in enumerate(lens):
        k, v, there = plain.rows(table, s, n)
        nq = start[s + 1] - start[s]
        for i in range(nq):
            see = there & (np.arange(n) <= n - nq + i)
            if not see.any():
                continue
            for h in range(q.shape[1]):
                w = k[see, h // group] @ q[start[s] + i, h].astype(np.float64) * scale
                w = np.exp(w - w.max())
                w /= w.sum()
                vs = v[see, h // group]
                out[start[s] + i, h] = w @ vs
                size[start[s] + i, h] = w @ np.abs(vs).max(1)
                most[start[s] + i, h] = np.abs(vs).max()
    return out, size, most


def run(ctx, plain, table, start, lens, q, scale=0.125, **kw):
    return cache_of(ctx, plain).attention(0, batch_of(table, start, lens), dev(q), scale=scale, **kw).cpu().numpy()


@pytest.mark.parametrize("dtype,new,group", FORMS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("factor", [2.0**12, 2.0**22, 2.0**60, 2.0**121])
def test_blocks_that_a_row_does_not_see_do_not_matter(ctx, dtype, new, group, d, factor):
    """V blocks behind a row's own position, in its tile and its step, have scales far above those that it sees."""
    rng = np.random.default_rng(d + new + group)
    heads = 2
    lens = [67, 160]
    new = [min(new, n) for n in lens]
    start = np.concatenate([[0], np.cumsum(new)])
    table, n_pages = tables(rng, lens)
    plain = filled(rng, n_pages, heads, d)
    plain.vs /= np.float32(64)
    first = [64, 144]  # positions from here on are in a block with a large scale
    for s, t in enumerate(first):
        plain.vs[table[s, t // BLOCK]] = np.float32(factor * 0.02)
    q = rng.standard_normal((start[-1], heads * group, d)).astype(dtype)
    got = run(ctx, plain, table, start, lens, q).astype(np.float64)
    want, size, _ = exact(plain, table, start, lens, q, 0.125)
    before = np.concatenate([np.arange(n - m, n) < t for n, m, t in zip(lens, new, first)])
    assert before.any() and not before.all()
    assert np.isfinite(got[before]).all()
    assert (np.abs(got - want).max(2)[before] <= REL[dtype] * size[before]).all()
    if dtype == "float32" and factor < 2.0**100:
        assert (np.abs(got - want).max(2) <= REL[dtype] * size).all()


@pytest.mark.parametrize("dtype,new,group", FORMS)
def test_an_infinity_in_a_later_token(ctx, dtype, new, group):
    """Stored as FLT_MAX, it is no business of the rows in front of its block."""
    rng = np.random.default_rng(5)
    heads, d, n = 2, 64, 100
    table, n_pages = tables(rng, [n])
    plain = Plain(n_pages, heads, d)
    k, v = (rng.standard_normal((n, heads, d)).astype(dtype) for _ in range(2))
    v[n - 1, 0, 3] = np.inf
    v[n - 2, 1, 0] = -np.inf
    cache = cache_of(ctx, plain)
    cache.append(0, batch_of(table, [0, n], [n]), dev(k), dev(v))
    plain.append(table, [0, n], [n], k, v)
    q = rng.standard_normal((new, heads * group, d)).astype(dtype)
    got = cache.attention(0, batch_of(table, [0, new], [n]), dev(q), 0.125).cpu().numpy().astype(np.float64)
    want, size, _ = exact(plain, table, [0, new], [n], q, 0.125)
    before = np.arange(n - new, n) < 96
    assert before.any()
    assert (np.abs(got - want).max(2)[before] <= REL[dtype] * size[before]).all()


@pytest.mark.parametrize("dtype,new,group", FORMS)
@pytest.mark.parametrize("factor", [2.0**10, 2.0**20, 2.0**30])
def test_large_blocks_of_no_weight(ctx, dtype, new, group, factor):
    """Blocks with large values and weights near 0 leave the others their bits."""
    rng = np.random.default_rng(7)
    heads, d, lens = 2, 64, [300]
    start = [0, new]
    table, n_pages = tables(rng, lens)
    plain = filled(rng, n_pages, heads, d)
    big = table[0, :18:2]
    plain.vs[big] *= np.float32(factor)
    plain.k[big] = 0
    plain.k[big, :, :, 0] = -127
    plain.ks[big] = np.float32(300 / 127)  # scores of these keys are 37 and more below 0: weights of 2^-53
    q = rng.standard_normal((new, heads * group, d)).astype(dtype)
    q[..., 0] = 1 + np.abs(q[..., 0])
    got = run(ctx, plain, table, start, lens, q).astype(np.float64)
    want, size, _ = exact(plain, table, start, lens, q, 0.125)
    assert (np.abs(got - want).max(2) <= REL[dtype] * size).all()


@pytest.mark.parametrize("dtype,new,group", FORMS)
def test_blocks_of_scale_zero_have_weight(ctx, dtype, new, group):
    """Values of 0 whatever the quants, beside small ones: they take their part of the softmax."""
    rng = np.random.default_rng(8)
    heads, d, lens = 2, 64, [300]
    table, n_pages = tables(rng, lens)
    plain = filled(rng, n_pages, heads, d)
    plain.vs[table[0, 1:19:2]] = 0
    q = rng.standard_normal((new, heads * group, d)).astype(dtype)
    got = run(ctx, plain, table, [0, new], lens, q).astype(np.float64)
    want, size, most = exact(plain, table, [0, new], lens, q, 0.125)
    assert (np.abs(got - want).max(2) <= REL[dtype] * np.maximum(size, most * 0.2)).all()


@pytest.mark.parametrize("dtype,new,group,n", [("float32", 1, 1, 40000), ("float16", 1, 1, 40000), ("float16", 3, 4, 40000), ("float16", 90, 1, 470)])
def test_many_small_weights(ctx, dtype, new, group, n):
    """One key of weight 1 and value 0, the others of weight 2^-26 and value 100 each."""
    rng = np.random.default_rng(9)
    heads, d = 1, 64
    table, n_pages = tables(rng, [n])
    plain = Plain(n_pages, heads, d)
    plain.k[..., 0] = -127
    plain.k[table[0, 0], :, 0, 0] = 127
    plain.ks[:] = np.float32(26 * np.log(2) / 254)
    plain.v[:] = 127
    plain.v[table[0, 0], :, :, 0] = 0
    plain.vs[:] = np.float32(100 / 127)
    q = np.zeros((new, heads * group, d), dtype)
    q[..., 0] = 1
    got = run(ctx, plain, table, [0, new], [n], q, scale=1.0).astype(np.float64)
    # every row sees the first key and n - new + 1 or more others
    others = n - new + np.arange(new)
    w = 2.0**-26 * others
    want = (100 * w / (1 + w))[:, None, None]
    # the smallest step of f16 is 6e-8; equal weights are rounded alike: 2^-11, and the output 2^-11
    assert (np.abs(got - want) <= REL[dtype] * want + (3e-8 if dtype == "float16" else 0)).all()


@pytest.mark.parametrize("n", [64, 65, 700, 5000])
def test_the_largest_values(ctx, n):
    """Values near the largest finite number: their average is finite, however the keys are shared out."""
    rng = np.random.default_rng(10)
    heads, d = 2, 64
    table, n_pages = tables(rng, [n])
    plain = filled(rng, n_pages, heads, d)
    plain.vs[:] = np.float32(np.finfo(np.float32).max / 130)
    q = rng.standard_normal((2, heads * 2, d)).astype(np.float32)
    got = run(ctx, plain, table, [0, 2], [n], q).astype(np.float64)
    want, size, _ = exact(plain, table, [0, 2], [n], q, 0.125)
    assert np.isfinite(got).all()
    assert (np.abs(got - want).max(2) <= REL["float32"] * size).all()


@pytest.mark.parametrize("dtype,new,group", FORMS)
@pytest.mark.parametrize("d", [64, 128])
def test_rows_with_an_infinity(ctx, dtype, new, group, d):
    """NaN, whatever the signs of the few keys that the row sees; a row without any key is 0, whatever it holds."""
    rng = np.random.default_rng(11)
    heads = 2
    lens, rows = [new, new - 3], [new, new]
    start = np.array([0, new, 2 * new])
    table, n_pages = tables(rng, lens)
    plain = filled(rng, n_pages, heads, d)
    plain.k[table[:, 0], :, 0] = -np.abs(plain.k[table[:, 0], :, 0]) - (plain.k[table[:, 0], :, 0] == 0)
    cache = cache_of(ctx, plain)
    b = batch_of(table, start, lens)
    q = rng.standard_normal((2 * new, heads * group, d)).astype(dtype)
    clean = cache.attention(0, b, dev(q), 0.125).cpu().numpy()
    bad = np.zeros(q.shape[:2], bool)
    none = np.zeros(q.shape[:2], bool)
    for r, h, x in ((0, 0, np.inf), (0, 1, -np.inf), (1, 0, np.inf), (new + 3, 1, np.inf), (new + 4, 0, np.nan)):
        q[r, h, 5] = x
        bad[r, h] = True
    for r, h, x in ((new, 0, np.inf), (new + 1, 1, np.nan), (new + 2, 0, -np.inf)):
        q[r, h, 7] = x
        none[r, h] = True
    got = cache.attention(0, b, dev(q), 0.125).cpu().numpy()
    assert np.isnan(got[bad]).all()
    assert (got[new:new + 3] == 0).all()
    assert np.array_equal(got[~(bad | none)], clean[~(bad | none)])


@pytest.mark.parametrize("size", [1e-33, 1e-36, 1e-39])
@pytest.mark.parametrize("d", [64, 96])
def test_rows_of_tiny_values(ctx, size, d):
    """Small rows of q over keys as large as they are small: scores of ordinary size. A q below 1.2e-38 has fewer bits
    itself (steps of 1.4e-45, exact in the plain form too)."""
    rng = np.random.default_rng(12)
    heads, lens = 2, [200]
    table, n_pages = tables(rng, lens)
    plain = filled(rng, n_pages, heads, d)
    up = min(1 / size, 1e37)
    plain.ks *= np.float32(up)
    q = (rng.standard_normal((5, heads * 2, d)) * size).astype(np.float32)
    got = run(ctx, plain, table, [0, 5], lens, q, scale=0.125 / (size * up)).astype(np.float64)
    want, size_of, _ = exact(plain, table, [0, 5], lens, q, np.float64(np.float32(0.125 / (size * up))))
    assert (np.abs(got - want).max(2) <= REL["float32"] * size_of).all()


@pytest.mark.parametrize("dtype,new,group", FORMS)
def test_rows_with_an_outlying_channel(ctx, dtype, new, group):
    """One channel of q is 200 and the others about 1. The kernel for few rows takes 16-bit rows of q to 2^-15.98 of the
    row's largest value and 32-bit rows to 2^-23.97, the tensor-core tiles take them as they are. Errors of a uniform
    distribution over 64 channels and |k| of 1.75 (root of the mean square), six times over, move a score by at most
    `off`, its weight by that part, and the sum of the weights too."""
    rng = np.random.default_rng(13)
    heads, d, lens = 2, 64, [300]
    table, n_pages = tables(rng, lens)
    plain = filled(rng, n_pages, heads, d)
    plain.k[:, :, :, 9] = 1
    q = rng.standard_normal((new, heads * group, d)).astype(dtype)
    q[..., 9] = 200
    got = run(ctx, plain, table, [0, new], lens, q).astype(np.float64)
    want, size, _ = exact(plain, table, [0, new], lens, q, 0.125)
    step = 2.0**-23.97 if dtype == "float32" else 2.0**-15.98 if new * group < 64 else 0.0
    off = 6 * 200 * step / np.sqrt(3) * np.sqrt(64) * 1.75 * 0.125
    assert (np.abs(got - want).max(2) <= (REL[dtype] + 2 * off) * size).all()


def test_a_wider_table_takes_the_same_kernel(ctx):
    """A table with room for more tokens than the streams have: same pages, same bits."""
    rng = np.random.default_rng(14)
    heads, group, d = 8, 4, 128
    lens, new = [2000, 700], [2000, 500]
    start = np.concatenate([[0], np.cumsum(new)])
    table, n_pages = tables(rng, lens)
    cache = cache_of(ctx, filled(rng, n_pages, heads, d))
    q = dev(rng.standard_normal((start[-1], heads * group, d)).astype(np.float16))
    first = cache.attention(0, batch_of(table, start, lens), q, d**-0.5).cpu().numpy()
    for times in (2, 8, 64):
        wide = np.full((2, times * table.shape[1]), -1, np.int32)
        wide[:, :table.shape[1]] = table
        assert np.array_equal(cache.attention(0, batch_of(wide, start, lens), q, d**-0.5).cpu().numpy(), first)


def test_a_wider_table_of_few_rows_with_a_hint(ctx):
    """Few enough rows that the number of keys decides: max_kv says it where the table does not."""
    from vokra_b200 import blockkv
    rng = np.random.default_rng(15)
    heads, group, d, n, new = 8, 4, 128, 1000, 100
    table, n_pages = tables(rng, [n])
    cache = cache_of(ctx, filled(rng, n_pages, heads, d))
    q = dev(rng.standard_normal((new, heads * group, d)).astype(np.float16))
    wide = np.full((1, 4096), -1, np.int32)
    wide[:, :table.shape[1]] = table
    i32 = lambda *x: dev(np.array(x, np.int32))  # noqa: E731
    got = [cache.attention(0, blockkv.Batch(i32(0, new), i32(n), dev(t), new, new, max_kv=kv), q, d**-0.5).cpu().numpy()
           for t, kv in ((table, 0), (wide, n), (wide, 0), (table, n))]
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[3])
    # without the hint it is another kernel, and the same values to its rounding (2 * 2^-11 of values up to 4.5)
    assert np.abs(got[0].astype(np.float64) - got[2]).max() <= 2 * 4.5e-3
    with pytest.raises(blockkv.VkbError):
        cache.attention(0, blockkv.Batch(i32(0, new), i32(n), dev(table), new, new, max_kv=-1), q)
