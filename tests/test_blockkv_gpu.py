"""The paged 8-bit KV cache with a scale per block of 16 tokens and head: append and read against plain numpy
(fp32, operation by operation: equal to the bit), attention against 64 bits.

Attention's bounds. Values are at most VMAX = 4.5 in size. With 32-bit rows q and the weights enter the
products in two f16 parts (2^-21 of a value): a score is off by at most scale * sum |q| |k| * 2^-21, below
1e-5 for the sizes here, so the weights by 2e-5 of themselves and an output by 2 * 2e-5 * VMAX < 2e-4. With
16-bit rows a weight is rounded to 2^-11 of itself and the output too: 2 * 2^-11 * VMAX < 4.5e-3."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

BLOCK = 16
TOL = {"float32": 2e-4, "float16": 4.5e-3}


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Plain:
    """The cache in numpy."""

    def __init__(self, n_pages, heads, d):
        self.k = np.zeros((n_pages, heads, BLOCK, d), np.int8)
        self.v = np.zeros((n_pages, heads, d, BLOCK), np.int8)
        self.ks = np.zeros((n_pages, heads), np.float32)
        self.vs = np.zeros((n_pages, heads), np.float32)

    def append(self, table, start, lens, k, v):
        one = np.float32
        for s, n in enumerate(lens):
            a, b = start[s], start[s + 1]
            pos0 = n - (b - a)
            for p in range(max(pos0, 0) // BLOCK, -(-n // BLOCK) if b > a else 0):
                if p >= table.shape[1] or not 0 <= table[s, p] < len(self.k):
                    continue
                t0, t1 = max(pos0 - p * BLOCK, 0), min(n - p * BLOCK, BLOCK)
                rows = slice(a + p * BLOCK + t0 - pos0, a + p * BLOCK + t1 - pos0)
                for x, q, sc in ((k[rows], self.k[table[s, p]], self.ks[table[s, p]]),
                                 (v[rows], self.v[table[s, p]].transpose(0, 2, 1), self.vs[table[s, p]])):
                    x = x.astype(np.float32).transpose(1, 0, 2)  # [heads, new, d]
                    with np.errstate(all="ignore"):
                        amax = np.minimum(np.fmax.reduce(np.fmax.reduce(np.abs(x), 2), 1), np.finfo(np.float32).max)
                        amax = np.fmax(amax, one(0))
                        old = sc.copy() if t0 > 0 else np.zeros_like(sc)
                        new = np.maximum(old, amax * (one(1) / one(127)))
                        inv = np.where(new > 0, one(1) / new, one(0)).astype(np.float32)
                        grown = (new > old)[:, None, None] & (t0 > 0)
                        ratio = np.where(new > 0, old / new, one(0)).astype(np.float32)
                        q[:, :t0] = np.where(grown, np.rint(q[:, :t0].astype(np.float32) * ratio[:, None, None]), q[:, :t0])
                        y = x * inv[:, None, None]
                        y = np.where(np.isnan(y), 0, np.clip(np.rint(y), -127, 127))
                    q[:, t0:t1] = y
                    sc[:] = new

    def rows(self, table, s, n):
        """(K, V) of the first n tokens in 64 bits, and which of them are there."""
        heads, d = self.k.shape[1], self.k.shape[3]
        k, v, there = np.zeros((n, heads, d)), np.zeros((n, heads, d)), np.zeros(n, bool)
        for t in range(n):
            p = table[s, t // BLOCK] if t // BLOCK < table.shape[1] else -1
            if 0 <= p < len(self.k):
                there[t] = True
                k[t] = self.k[p, :, t % BLOCK].astype(np.float64) * self.ks[p][:, None]
                v[t] = self.v[p, :, :, t % BLOCK].astype(np.float64) * self.vs[p][:, None]
        return k, v, there

    def attention(self, table, start, lens, q, scale):
        heads = self.k.shape[1]
        out = np.zeros(q.shape)
        group = q.shape[1] // heads
        for s, n in enumerate(lens):
            if n <= 0:
                continue
            k, v, there = self.rows(table, s, n)
            nq = start[s + 1] - start[s]
            for i in range(nq):
                see = there & (np.arange(n) <= n - nq + i)
                if not see.any():
                    continue
                for h in range(q.shape[1]):
                    w = k[see, h // group] @ q[start[s] + i, h].astype(np.float64) * scale
                    w = np.exp(w - w.max())
                    out[start[s] + i, h] = w @ v[see, h // group] / w.sum()
        return out


def tables(rng, lens, extra=2, missing=()):
    need = -(-np.maximum(np.asarray(lens), 0) // BLOCK)
    n_pages = int(need.sum()) + 3
    ids = rng.permutation(n_pages)
    table = np.full((len(lens), int(need.max(initial=0)) + extra), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    for s, p in missing:
        table[s, p] = -1
    return table, n_pages


def filled(rng, n_pages, heads, d, size=1.0):
    """A cache with random quants and scales everywhere, pages in no table with scales that are not numbers."""
    c = Plain(n_pages, heads, d)
    c.k[:] = rng.integers(-127, 128, c.k.shape)
    c.v[:] = rng.integers(-127, 128, c.v.shape)
    c.ks[:] = (rng.random(c.ks.shape) + 0.5) * (size * 3 / 127)
    c.vs[:] = (rng.random(c.vs.shape) + 0.5) * (3 / 127)
    return c


def cache_of(ctx, c, layers=1, layer=0):
    """The device cache holding c in one of its layers."""
    import torch
    from vokra_b200 import blockkv
    arenas = []
    for a in (c.k, c.v, c.ks, c.vs):
        t = torch.zeros((layers,) + a.shape, dtype=torch.from_numpy(a[:1]).dtype, device="cuda")
        t[layer] = dev(a)
        arenas.append(t)
    return blockkv.BlockKvCache(ctx, *arenas)


def batch_of(table, start, lens, status=None):
    from vokra_b200 import blockkv
    new = np.diff(start)
    return blockkv.Batch(dev(np.asarray(start, np.int32)), dev(np.asarray(lens, np.int32)), dev(table), int(start[-1]),
                         int(new.max(initial=0)), status)


def same_cache(cache, c, layer=0):
    for got, want in ((cache.k, c.k), (cache.v, c.v), (cache.k_scale, c.ks), (cache.v_scale, c.vs)):
        assert np.array_equal(got[layer].cpu().numpy(), want)


@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_append_and_read_equal_plain_to_the_bit(ctx, d, dtype):
    """Streams that grow in several calls: from nothing, inside a block, over block ends, by one and by many."""
    rng = np.random.default_rng(d)
    heads, layers, layer = 3, 2, 1
    final = [70, 1, 16, 33, 0, 48]
    table, n_pages = tables(rng, final, missing=[(0, 2)])
    plain = Plain(n_pages, heads, d)
    cache = cache_of(ctx, plain, layers, layer)
    lens = np.zeros(len(final), int)
    for step in range(5):
        grow = np.array([min(g, f - n) for g, f, n in zip(rng.integers(0, 30, len(final)) if step < 4 else final, final, lens)])
        lens = lens + grow
        start = np.concatenate([[0], np.cumsum(grow)])
        size = np.float32(10.0) ** rng.integers(-3, 4, (start[-1], heads, 1))  # scales grow and blocks are rounded anew
        k, v = ((rng.standard_normal((start[-1], heads, d)) * size).astype(dtype) for _ in range(2))
        if start[-1] == 0:
            continue
        cache.append(layer, batch_of(table, start, lens), dev(k), dev(v))
        plain.append(table, start, lens, k, v)
        same_cache(cache, plain, layer)
        assert not cache.k[0].any() and not cache.k_scale[0].any()
    rows = np.concatenate([[0], np.cumsum(lens)])
    got_k, got_v = cache.read(layer, batch_of(table, rows, lens))
    for s, n in enumerate(lens):
        k, v, _ = plain.rows(table, s, n)
        assert np.array_equal(got_k[rows[s]:rows[s + 1]].cpu().numpy(), k.astype(np.float32))
        assert np.array_equal(got_v[rows[s]:rows[s + 1]].cpu().numpy(), v.astype(np.float32))
    # the last rows only, one more than some streams have, in 16 bits
    start = np.arange(len(final) + 1) * 2
    import torch
    got_k, got_v = cache.read(layer, batch_of(table, start, lens), torch.float16)
    for s, n in enumerate(lens):
        k, v, _ = plain.rows(table, s, n)
        for got, want in ((got_k, k), (got_v, v)):
            want = np.concatenate([np.zeros((2, heads, d)), want])[-2:].astype(np.float32).astype(np.float16)
            assert np.array_equal(got[2 * s:2 * s + 2].cpu().numpy(), want)


def test_append_edge_values(ctx):
    """Zeros, values whose scale is subnormal, the largest finite ones, infinities and NaN."""
    rng = np.random.default_rng(1)
    heads, d = 2, 64
    table, n_pages = tables(rng, [16] * 6)
    plain = Plain(n_pages, heads, d)
    cache = cache_of(ctx, plain)
    k = rng.standard_normal((6 * 16, heads, d)).astype(np.float32)
    k[:16] = 0
    k[16:32] *= np.float32(1e-37)
    k[32:48] *= np.float32(8e37)
    k[48:64, :, ::5] = np.inf
    k[48:64, :, 1::5] = -np.inf
    k[64:80, :, ::3] = np.nan
    k[80:96] = np.nan
    start = np.arange(7) * 16
    b = batch_of(table, start, [16] * 6)
    cache.append(0, b, dev(k), dev(k * np.float32(0.5)))
    plain.append(table, start, [16] * 6, k, k * np.float32(0.5))
    same_cache(cache, plain)


def test_append_rewrites_a_block_from_its_first_slot(ctx):
    """A block that is begun again forgets its old scale; one that is continued keeps it."""
    rng = np.random.default_rng(2)
    heads, d = 1, 32
    table, n_pages = tables(rng, [32])
    plain = Plain(n_pages, heads, d)
    cache = cache_of(ctx, plain)
    for lens, n, size in ((20, 20, 100.0), (16, 16, 0.01), (18, 2, 0.01), (17, 1, 5.0), (32, 16, 1.0)):
        k = (rng.standard_normal((n, heads, d)) * size).astype(np.float32)
        cache.append(0, batch_of(table, [0, n], [lens]), dev(k), dev(-k))
        plain.append(table, [0, n], [lens], k, -k)
        same_cache(cache, plain)


def test_append_takes_any_row_stride_and_address(ctx):
    import torch
    rng = np.random.default_rng(3)
    heads, d = 2, 64
    lens, start = [19, 40], np.array([0, 19, 59])
    table, n_pages = tables(rng, lens)
    w = heads * d
    for dtype in ("float32", "float16"):
        for off, ld in ((0, 3 * w), (1, 3 * w + 1), (2, 3 * w + 6)):
            big = rng.standard_normal((59, ld + 2)).astype(dtype)
            plain = Plain(n_pages, heads, d)
            cache = cache_of(ctx, plain)
            t = dev(big)
            k, v = t[:, off:off + w], t[:, off + w:off + 2 * w]
            cache.append(0, batch_of(table, start, lens), k, v.view(59, heads, d) if v.is_contiguous() else v)
            plain.append(table, start, lens, big[:, off:off + w].reshape(59, heads, d), big[:, off + w:off + 2 * w].reshape(59, heads, d))
            same_cache(cache, plain)
            torch.cuda.synchronize()


def test_append_stores_nothing_after_a_failed_advance(ctx):
    import torch
    rng = np.random.default_rng(4)
    table, n_pages = tables(rng, [10])
    plain = Plain(n_pages, 1, 64)
    cache = cache_of(ctx, plain)
    k = dev(rng.standard_normal((10, 1, 64)).astype(np.float32))
    cache.append(0, batch_of(table, [0, 10], [10], torch.ones(1, dtype=torch.int32, device="cuda")), k, k)
    same_cache(cache, plain)


def check_attention(ctx, rng, lens, new, heads, group, d, dtype, missing=(), size=1.0, out_dtype=None, plain=None):
    start = np.concatenate([[0], np.cumsum(new)])
    table, n_pages = tables(rng, lens, missing=missing)
    plain = plain or filled(rng, n_pages, heads, d, size)
    unused = np.setdiff1d(np.arange(n_pages), table[table >= 0])
    cache = cache_of(ctx, plain)
    cache.k_scale[0, dev(unused).long()] = float("nan")
    cache.v_scale[0, dev(unused).long()] = float("nan")
    # pages in the table behind a stream's last token may hold anything
    if len(unused):
        for s in range(len(lens)):
            at = -(-max(lens[s], 0) // BLOCK)
            table[s, at:] = unused[0]
    q = rng.standard_normal((start[-1], heads * group, d)).astype(dtype)
    import torch
    out = torch.full((int(start[-1]), heads * group, d), 7.0, dtype=getattr(torch, out_dtype or dtype), device="cuda")
    got = cache.attention(0, batch_of(table, start, lens), dev(q), scale=d ** -0.5, out=out).cpu().numpy()
    table = np.where(np.arange(table.shape[1]) < -(-np.maximum(np.asarray(lens), 0) // BLOCK)[:, None], table, -1)
    want = plain.attention(table, start, lens, q, d ** -0.5)
    tol = max(TOL[dtype], TOL[out_dtype or dtype])
    assert np.isfinite(got).all()
    assert np.max(np.abs(got - want), initial=0.0) <= tol
    return got, want


@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 1), (2, 4), (1, 8), (2, 3)])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_decode_over_ragged_lengths(ctx, d, heads, group, dtype):
    rng = np.random.default_rng(d * 10 + heads + group)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129, 300]
    check_attention(ctx, rng, lens, [1] * len(lens), heads, group, d, dtype)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 5])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_several_rows_a_stream(ctx, d, group, dtype):
    """Checked tokens and prompt chunks, streams without rows, more rows than the stream has tokens."""
    rng = np.random.default_rng(d + group)
    lens = [40, 7, 64, 65, 3, 0, 200, 130, 16]
    new = [4, 7, 1, 9, 6, 2, 33, 0, 16]
    check_attention(ctx, rng, lens, new, 2, group, d, dtype)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("new,lens", [([130, 257], [130, 300]), ([200], [901]), ([64, 1, 500], [640, 64, 500])])
def test_prompt_chunks(ctx, d, dtype, new, lens):
    rng = np.random.default_rng(d + new[0])
    check_attention(ctx, rng, lens, new, 2, 2, d, dtype)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,group,new,lens", [
    (8, 4, [300, 1, 129, 0, 64], [300, 700, 1000, 50, 64]),    # tiles that end inside 128 and 256 rows, streams with few rows between
    (16, 1, [600, 513], [640, 4000]),
    (16, 3, [256, 100, 90], [255, 100, 91]),                   # more rows than tokens: rows without any key
])
def test_many_rows_of_16_bits(ctx, d, heads, group, new, lens):
    """Enough row tiles for the tensor-core kernel; against the kernel for few rows, which 32-bit rows take, and 64 bits on some heads."""
    import torch
    rng = np.random.default_rng(d + heads + group)
    start = np.concatenate([[0], np.cumsum(new)])
    table, n_pages = tables(rng, lens, missing=[(1, 2)])
    plain = filled(rng, n_pages, heads, d)
    plain.vs[rng.random(plain.vs.shape) < 0.2] *= np.float32(40)     # V scales rise along the way
    plain.vs /= np.float32(40)
    cache = cache_of(ctx, plain)
    b = batch_of(table, start, lens)
    q = rng.standard_normal((start[-1], heads * group, d)).astype(np.float16)
    got = cache.attention(0, b, dev(q), scale=d ** -0.5)
    few = cache.attention(0, b, dev(q.astype(np.float32)), scale=d ** -0.5)
    assert torch.isfinite(got).all()
    assert float((got.float() - few).abs().max()) <= TOL["float16"]
    sub = Plain(n_pages, 1, d)
    h = heads - 1
    sub.k, sub.v, sub.ks, sub.vs = plain.k[:, h:h + 1], plain.v[:, h:h + 1], plain.ks[:, h:h + 1], plain.vs[:, h:h + 1]
    want = sub.attention(table, start, lens, q[:, h * group:(h + 1) * group], d ** -0.5)
    assert np.max(np.abs(got[:, h * group:(h + 1) * group].cpu().numpy() - want)) <= TOL["float16"]
    again = cache.attention(0, b, dev(q), scale=d ** -0.5)
    assert torch.equal(got, again)


def test_rows_that_are_not_numbers(ctx):
    """A row of q with NaN or an infinity is NaN; the others are as they would be."""
    rng = np.random.default_rng(19)
    for dtype, heads, group, new in (("float32", 2, 2, [3, 1]), ("float16", 2, 2, [2, 1]), ("float16", 2, 8, [3, 2]), ("float16", 16, 4, [300, 200])):
        lens = [n + 70 for n in new]
        start = np.concatenate([[0], np.cumsum(new)])
        table, n_pages = tables(rng, lens)
        cache = cache_of(ctx, filled(rng, n_pages, heads, 64))
        b = batch_of(table, start, lens)
        q = rng.standard_normal((start[-1], heads * group, 64)).astype(dtype)
        want = cache.attention(0, b, dev(q)).cpu().numpy()
        bad = np.zeros(q.shape[:2], bool)
        for i, (r, h, x) in enumerate([(0, 0, np.nan), (0, 3, np.inf), (start[-1] - 1, 1, -np.inf), (1, 2, np.nan)]):
            q[r, h, 7 * i] = x
            bad[r, h] = True
        got = cache.attention(0, b, dev(q)).cpu().numpy()
        assert np.isnan(got[bad]).all()
        assert np.array_equal(got[~bad], want[~bad])


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_one_long_stream_and_many_short_ones(ctx, dtype):
    rng = np.random.default_rng(11)
    check_attention(ctx, rng, [20000], [1], 2, 4, 128, dtype)
    check_attention(ctx, rng, list(rng.integers(0, 90, 300)), [1] * 300, 2, 1, 64, dtype)


def test_mixed_types(ctx):
    rng = np.random.default_rng(12)
    for dtype, out in (("float32", "float16"), ("float16", "float32")):
        check_attention(ctx, rng, [33, 100], [1, 20], 2, 2, 64, dtype, out_dtype=out)


def test_pages_that_are_not_there(ctx):
    rng = np.random.default_rng(13)
    for dtype in ("float32", "float16"):
        check_attention(ctx, rng, [100, 20, 70], [1, 3, 20], 2, 2, 64, dtype, missing=[(0, 3), (1, 0), (1, 1), (2, 4)])


def test_sharp_scores_and_odd_scales(ctx):
    """Scores in the hundreds (one key takes all), blocks whose scale is 0, and V scales far apart."""
    rng = np.random.default_rng(14)
    for dtype in ("float32", "float16"):
        got, want = check_attention(ctx, rng, [500, 129], [1, 5], 2, 2, 64, dtype, size=0.05)
        heads, d, lens = 2, 64, [200, 333]
        table, n_pages = tables(np.random.default_rng(14), lens)
        plain = filled(rng, n_pages, heads, d)
        plain.ks[::3] = 0
        plain.vs[::2] *= np.float32(1e-9)
        plain.vs[1::4] = 0
        check_attention(ctx, np.random.default_rng(14), lens, [1, 1], heads, 2, d, dtype, plain=plain)


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e6, 1e30])
def test_values_of_any_size(ctx, scale):
    """The products do not leave their range whatever the V scales and the size of q."""
    rng = np.random.default_rng(15)
    heads, d, lens, new = 2, 64, [100, 65], [1, 10]
    start = np.array([0, 1, 11])
    table, n_pages = tables(rng, lens)
    plain = filled(rng, n_pages, heads, d)
    plain.vs *= np.float32(scale)
    plain.ks *= np.float32(1 / scale)
    cache = cache_of(ctx, plain)
    q = (rng.standard_normal((11, 4, d)) * scale).astype(np.float32)
    got = cache.attention(0, batch_of(table, start, lens), dev(q), scale=0.125).cpu().numpy().astype(np.float64)
    want = plain.attention(table, start, lens, q, 0.125)
    assert np.max(np.abs(got - want)) <= TOL["float32"] * scale


def test_strided_rows_of_a_fused_projection(ctx):
    import torch
    rng = np.random.default_rng(16)
    heads, group, d, lens, new = 2, 2, 64, [50, 90], [3, 1]
    start = np.array([0, 3, 4])
    table, n_pages = tables(rng, lens)
    plain = filled(rng, n_pages, heads, d)
    cache = cache_of(ctx, plain)
    w = heads * group * d
    for dtype in ("float32", "float16"):
        for off, ld in ((0, 2 * w), (1, 2 * w + 1), (3, 2 * w + 5)):
            big = rng.standard_normal((4, ld + 4)).astype(dtype)
            out = torch.full((4, ld + 3), 9.0, dtype=getattr(torch, dtype), device="cuda")
            cache.attention(0, batch_of(table, start, lens), dev(big)[:, off:off + w], scale=0.125, out=out[:, off:off + w])
            want = plain.attention(table, start, lens, big[:, off:off + w].reshape(4, heads * group, d), 0.125)
            got = out.cpu().numpy()
            assert np.max(np.abs(got[:, off:off + w].reshape(4, -1, d) - want)) <= TOL[dtype]
            assert (got[:, :off] == 9).all() and (got[:, off + w:] == 9).all()


def test_same_inputs_same_bits(ctx):
    rng = np.random.default_rng(17)
    lens = [700, 31, 2000]
    table, n_pages = tables(rng, lens)
    cache = cache_of(ctx, filled(rng, n_pages, 2, 64))
    q = dev(rng.standard_normal((3, 4, 64)).astype(np.float32))
    b = batch_of(table, [0, 1, 2, 3], lens)
    first = cache.attention(0, b, q).cpu().numpy()
    for _ in range(5):
        assert np.array_equal(cache.attention(0, b, q).cpu().numpy(), first)


def test_append_then_attend_in_a_recorded_step(ctx):
    """Append and attention recorded once and replayed on new values."""
    import torch
    from vokra_b200 import ops
    rng = np.random.default_rng(18)
    heads, d, lens = 2, 64, [37, 80]
    start = np.array([0, 1, 2])
    table, n_pages = tables(rng, lens)
    plain = filled(rng, n_pages, heads, d)
    st = torch.cuda.Stream()
    c = ops.Context(0)
    c.set_stream(st.cuda_stream)
    cache = cache_of(c, plain)
    b = batch_of(table, start, lens)
    k, v, q = (torch.zeros(2, heads, d, device="cuda") for _ in range(3))
    out = torch.zeros(2, heads, d, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        cache.attention(0, b, q, out=out)  # the context's scratch grows here
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        cache.append(0, b, k, v)
        cache.attention(0, b, q, scale=0.125, out=out)
    for _ in range(3):
        x = [rng.standard_normal((2, heads, d)).astype(np.float32) for _ in range(3)]
        for t, a in zip((k, v, q), x):
            t.copy_(dev(a))
        g.replay()
        torch.cuda.synchronize()
        plain.append(table, start, lens, x[0], x[1])
        same_cache(cache, plain)
        assert np.max(np.abs(out.cpu().numpy() - plain.attention(table, start, lens, x[2], 0.125))) <= TOL["float32"]


def test_refusals(ctx):
    import torch
    from vokra_b200 import _lib, blockkv
    from vokra_b200.ops import VkbError
    cache = blockkv.BlockKvCache.empty(ctx, 2, 2, 64, 4)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    b = blockkv.Batch(i(2), i(1), i(1, 4), 1, 1)
    q = torch.zeros(1, 4, 64, device="cuda")
    kv = torch.zeros(1, 2, 64, device="cuda")
    bad = [
        lambda: cache.append(2, b, kv, kv), lambda: cache.append(-1, b, kv, kv), lambda: cache.append(0, b, kv, kv.half()),
        lambda: cache.append(0, b, q, q), lambda: cache.append(0, b, kv.double(), kv.double()), lambda: cache.append(0, b, kv.cpu(), kv),
        lambda: cache.attention(0, b, torch.zeros(1, 3, 64, device="cuda")), lambda: cache.attention(0, b, q[:0]),
        lambda: cache.attention(0, b, q, scale=0.0), lambda: cache.attention(0, b, q, scale=float("nan")),
        lambda: cache.attention(0, b, q, scale=float("inf")), lambda: cache.attention(0, b, q, out=kv),
        lambda: cache.attention(0, b, q.transpose(1, 2)), lambda: cache.read(0, b, torch.float64),
        lambda: blockkv.Batch(i(1), i(1), i(1, 4), 1, 1), lambda: blockkv.Batch(i(2), i(1), i(2, 4), 1, 1),
        lambda: blockkv.Batch(i(2).long(), i(1), i(1, 4), 1, 1), lambda: blockkv.Batch(i(2), i(1), i(1, 8)[:, ::2], 1, 1),
        lambda: blockkv.BlockKvCache(ctx, cache.k, cache.k, cache.k_scale, cache.v_scale),
        lambda: blockkv.BlockKvCache(ctx, cache.k[:, :, :1], cache.v[:, :, :1], cache.k_scale[:, :, :1], cache.v_scale[:, :, :1]),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(VkbError) as e:
            call()
        assert e.value.code == _lib.ERROR_INVALID_ARGUMENT, n
    odd = blockkv.BlockKvCache.empty(ctx, 1, 1, 48, 2)
    with pytest.raises(VkbError) as e:
        odd.attention(0, b, torch.zeros(1, 1, 48, device="cuda"))
    assert e.value.code == _lib.ERROR_UNSUPPORTED_OP
    none = blockkv.Batch(i(1), i(0), i(0, 4), 0, 0)
    assert cache.attention(0, none, q[:0]).shape == (0, 4, 64)
    L = _lib.load()
    assert L.vkb_bkv_attention(None, cache.ref, 0, b.ref, 4, None, 256, 0, 1.0, None, 256, 0) == _lib.ERROR_INVALID_ARGUMENT
    assert L.vkb_bkv_append(ctx.h, None, 0, b.ref, None, 128, None, 128, 0) == _lib.ERROR_INVALID_ARGUMENT
    assert L.vkb_bkv_append(ctx.h, cache.ref, 0, b.ref, None, 128, None, 128, 0) == _lib.ERROR_INVALID_ARGUMENT
    assert L.vkb_bkv_read(ctx.h, cache.ref, 0, None, None, None, 0) == _lib.ERROR_INVALID_ARGUMENT


@pytest.mark.parametrize("d,dtype,most", [(64, "float32", 3), (64, "float16", 3), (128, "float16", 9), (256, "float32", 2), (32, "float16", 9)])
def test_many_short_streams_beside_long_ones(ctx, d, dtype, most):
    """Several steps for every warp of the GPU: shares count an item's fixed cost, ends of shares fall anywhere, in an
    item's last steps too; more streams than one launch takes."""
    rng = np.random.default_rng(d + most)
    heads, group, n_seq = 4, 2, 560
    lens = rng.integers(0, 260, n_seq)
    lens[[3, 250, 511, 540]] = [1500, 64, 2100, 1023]
    lens[20:40] = 0
    new = rng.integers(0, most + 1, n_seq)
    new[100:130] = 0
    start = np.concatenate([[0], np.cumsum(new)])
    table, n_pages = tables(rng, lens)
    plain = filled(rng, n_pages, heads, d)
    q = (rng.standard_normal((start[-1], heads * group, d)) * 0.5).astype(dtype)
    out = cache_of(ctx, plain).attention(0, batch_of(table, start, lens), dev(q), d**-0.5)
    want = plain.attention(table, start, lens, q, d**-0.5)
    assert np.abs(out.cpu().numpy() - want).max() <= TOL[dtype]


@pytest.mark.parametrize("dtype,new", [("float32", [1, 2]), ("float16", [200, 150])])
def test_offsets_above_32_bits(ctx, dtype, new):
    """Pages at the end of arenas of 2.3 GB: append, attention, read and a page that is copied on a write."""
    import torch
    from vokra_b200 import blockkv
    rng = np.random.default_rng(31)
    heads, group, d, n_pages = 8, 1, 128, 140000
    lens = [230, 170]
    start = np.concatenate([[0], np.cumsum(new)])
    table, few = tables(rng, lens)
    plain = filled(rng, few, heads, d)
    cache = blockkv.BlockKvCache.empty(ctx, 1, heads, d, n_pages)
    assert cache.k.numel() > 2**31
    at = n_pages - few
    for t, a in ((cache.k, plain.k), (cache.v, plain.v), (cache.k_scale, plain.ks), (cache.v_scale, plain.vs)):
        t[0, at:] = dev(a)
    high = np.where(table >= 0, table + at, -1).astype(np.int32)
    b = batch_of(high, start, lens)
    k, v = (rng.standard_normal((start[-1], heads, d)).astype(dtype) for _ in range(2))
    q = rng.standard_normal((start[-1], heads * group, d)).astype(dtype)
    cache.append(0, b, dev(k), dev(v))
    plain.append(table, start, lens, k, v)
    for t, a in ((cache.k, plain.k), (cache.v, plain.v), (cache.k_scale, plain.ks), (cache.v_scale, plain.vs)):
        assert np.array_equal(t[0, at:].cpu().numpy(), a)
    out = cache.attention(0, b, dev(q), d**-0.5).cpu().numpy()
    assert np.abs(out - plain.attention(table, start, lens, q, d**-0.5)).max() <= TOL[dtype]
    got, _ = cache.read(0, b)
    want, _, _ = plain.rows(table, 1, lens[1])
    assert np.array_equal(got[start[1]:].cpu().numpy(), want[-new[1]:].astype(np.float32))
    # stream 0 of a fork keeps its last page, stream 1 writes into a copy; every page in front is taken
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    pages = cache.pages(status)
    refs = np.ones(n_pages, np.int32)
    refs[at:] = 0
    own = high[0, :-(-lens[0] // BLOCK)]
    refs[own] = 1
    state = [np.stack([high[0], np.full_like(high[0], -1)]), np.array([lens[0], 0], np.int32), refs]
    a, c = blockkv.PageState(*map(dev, state)), blockkv.PageState(*map(dev, state))
    pages.advance(a, c, dev(np.zeros(2, np.int32)), dev(np.array([0, 1], np.int32)))
    pages.check()
    copy, last = int(c.table[1, lens[0] // BLOCK]), int(own[lens[0] // BLOCK])
    assert copy >= at and copy != last
    assert torch.equal(cache.k[0, copy], cache.k[0, last]) and torch.equal(cache.v_scale[0, copy], cache.v_scale[0, last])
