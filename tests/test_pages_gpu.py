"""Forking, freeing, growing and compacting the pages of a cache on the device, against a plain allocator.
Everything is whole numbers and moved bytes: compared for equality."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

PT = 16


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def plain_advance(table, lens, refs, arenas, parent, new):
    """(status, table, lens, refs); arenas change in place."""
    n, ld = table.shape
    t, ln = np.full_like(table, -1), np.zeros_like(lens)
    held = np.zeros_like(refs)
    live = np.zeros(n, bool)
    for s in range(n):
        p = s if parent is None else parent[s]
        if p >= n:
            return 3, table, lens, refs
        if p < 0:
            continue
        live[s] = True
        ln[s] = lens[p]
        have = -(-lens[p] // PT)
        t[s, :have] = table[p, :have]
        if ((t[s, :have] < 0) | (t[s, :have] >= len(refs))).any():
            return 3, table, lens, refs
        np.add.at(held, t[s, :have], 1)
    grow = np.where(live, 0 if new is None else new, 0)
    if (grow < 0).any():
        return 3, table, lens, refs
    if (-(-(ln + grow) // PT) > ld).any():
        return 2, table, lens, refs
    free = [i for i in range(len(refs)) if held[i] == 0 and refs[i] == 0]
    takes = []
    for s in range(n):
        have, want = -(-ln[s] // PT), -(-(ln[s] + grow[s]) // PT)
        if grow[s] > 0 and ln[s] % PT and held[t[s, have - 1]] > 1:
            takes.append((s, have - 1, t[s, have - 1]))
        takes += [(s, p, -1) for p in range(have, want)]
    if len(takes) > len(free):
        return 1, table, lens, refs
    for (s, p, src), dst in zip(takes, free):
        t[s, p] = dst
        if src >= 0:
            for a in arenas:
                a[:, dst] = a[:, src]
    out = np.zeros_like(refs)
    np.add.at(out, t[t >= 0], 1)
    return 0, t, ln + grow, out


def plain_compact(table, refs, arenas):
    used = int((refs > 0).sum())
    src = [i for i in range(used, len(refs)) if refs[i] > 0]
    dst = [i for i in range(used) if refs[i] == 0]
    to = {a: b for a, b in zip(src, dst)}
    out = np.where(np.arange(len(refs)) < used, refs, 0)
    for a, b in to.items():
        out[b] = refs[a]
        for x in arenas:
            x[:, b] = x[:, a]
    return np.vectorize(lambda i: to.get(i, i))(table).astype(np.int32), out, used


def make_arenas(rng, layers, n_pages, shapes=((2, 16, 8), (2, 1))):
    """One plane whose pages are a multiple of 16 bytes, one of 8, one of bytes that nothing divides."""
    a = [rng.integers(0, 255, (layers, n_pages) + s).astype(np.uint8) for s in shapes]
    return a + [rng.integers(0, 255, (layers, n_pages, 5)).astype(np.uint8), rng.standard_normal((layers, n_pages, 3)).astype(np.float32)]


class Both:
    """The device pages and the plain ones, side by side."""

    def __init__(self, ctx, rng, n, ld, n_pages, layers=2):
        import torch
        from vokra_b200 import blockkv
        self.plain = make_arenas(rng, layers, n_pages)
        self.dev = [dev(a) for a in self.plain]
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.pool = blockkv.PagePool(ctx, self.dev, self.status)
        self.a, self.b = blockkv.PageState.empty(n, ld, n_pages), blockkv.PageState.empty(n, ld, n_pages)
        self.table, self.lens, self.refs = np.full((n, ld), -1, np.int32), np.zeros(n, np.int32), np.zeros(n_pages, np.int32)

    def same(self, st=None):
        st = st or self.a
        assert np.array_equal(st.table.cpu().numpy(), self.table)
        assert np.array_equal(st.len.cpu().numpy(), self.lens)
        assert np.array_equal(st.refs.cpu().numpy(), self.refs)
        for a, b in zip(self.dev, self.plain):
            assert np.array_equal(a.cpu().numpy(), b)

    def advance(self, parent=None, new=None, status=0):
        i = lambda x: None if x is None else dev(np.asarray(x, np.int32))  # noqa: E731
        self.b.table.fill_(77)
        self.b.refs.fill_(77)
        self.pool.advance(self.a, self.b, i(parent), i(new))
        st, *state = plain_advance(self.table, self.lens, self.refs, self.plain, parent, new)
        assert st == status and int(self.status.cpu()[0]) == status
        self.table, self.lens, self.refs = (np.asarray(x, np.int32) for x in state)
        self.same(self.b)
        self.status.zero_()
        self.a, self.b = self.b, self.a

    def compact(self):
        import torch
        used = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.b.table.fill_(77)
        self.b.refs.fill_(77)
        self.pool.compact(self.a, self.b, used)
        self.table, self.refs, n = plain_compact(self.table, self.refs, self.plain)
        assert int(used.cpu()[0]) == n
        self.same(self.b)
        self.a, self.b = self.b, self.a


@pytest.mark.parametrize("n,ld,n_pages", [(1, 3, 5), (5, 9, 60), (40, 30, 1500), (3, 300, 9001)])
def test_random_histories(ctx, n, ld, n_pages):
    """Beam steps, prompts, finished streams and compactions in a row."""
    rng = np.random.default_rng(n)
    x = Both(ctx, rng, n, ld, n_pages)
    x.advance(new=rng.integers(0, ld * PT // 3, n))
    for step in range(8):
        parent = rng.integers(-1, n, n)
        x.advance(parent, (rng.random(n) < 0.8).astype(np.int64))
        if step == 3:
            x.advance(np.where(rng.random(n) < 0.5, -1, np.arange(n)), None)
            x.compact()
        if step == 5:
            x.advance(None, rng.integers(0, ld * PT // 4, n))
    x.compact()
    x.compact()


def test_many_streams_and_a_full_plan(ctx):
    """More streams than the planning block has threads."""
    rng = np.random.default_rng(4)
    x = Both(ctx, rng, 1500, 3, 9000, layers=1)
    x.advance(new=rng.integers(0, 20, 1500))
    x.advance(rng.integers(-1, 1500, 1500), rng.integers(0, 9, 1500))
    x.compact()


def test_shared_page_is_copied_by_each_writer(ctx):
    rng = np.random.default_rng(5)
    x = Both(ctx, rng, 4, 4, 20)
    x.advance(new=[20, 0, 0, 0])
    x.advance([0, 0, 0, -1])                # three streams share a full page and a partly filled one
    assert x.refs[x.table[0, 0]] == 3 and x.refs[x.table[0, 1]] == 3
    x.advance(new=[1, 1, 0, 0])             # two write: each gets its own copy, the third keeps the page
    assert len({x.table[0, 1], x.table[1, 1], x.table[2, 1]}) == 3 and x.refs[x.table[2, 1]] == 1
    x.advance(new=[12, 0, 0, 0])            # to the end of the block: nothing shared is written
    x.advance([0, 0, 0, 0], [1, 1, 1, 1])   # after a full block: new pages, no copies


def test_what_cannot_be_done_changes_nothing(ctx):
    rng = np.random.default_rng(6)
    x = Both(ctx, rng, 3, 4, 6)
    x.advance(new=[30, 30, 0])              # 4 of 6 pages
    x.advance(new=[16, 16, 16], status=1)   # 5 more: too many
    x.advance(new=[64, 0, 0], status=2)     # longer than its table
    x.advance([0, 3, 1], [1, 1, 1], status=3)
    x.advance(new=[1, -1, 0], status=3)
    x.advance([0, 0, -1], [0, 0, 0])        # frees a stream's pages
    x.advance([0, -1, -1], [0, 0, 0])
    x.advance(new=[2, 0, 16])               # and they are there again
    bad = x.a.table.clone()
    x.a.table[0, 0] = 99
    x.table[0, 0] = 99
    x.advance(status=3)
    x.a.table.copy_(bad)


def test_a_call_can_be_repeated(ctx):
    """The old state stays valid: the same call again gives the same new state."""
    rng = np.random.default_rng(7)
    x = Both(ctx, rng, 6, 5, 40)
    x.advance(new=[20, 21, 22, 5, 0, 40])
    par, new = dev(np.array([1, 1, 1, 5, 0, -1], np.int32)), dev(np.ones(6, np.int32))
    x.pool.advance(x.a, x.b, par, new)
    first = [t.clone() for t in (x.b.table, x.b.len, x.b.refs, *x.dev)]
    x.pool.advance(x.a, x.b, par, new)
    for t, f in zip((x.b.table, x.b.len, x.b.refs, *x.dev), first):
        assert (t == f).all()


def test_compact_full_and_empty_arenas(ctx):
    rng = np.random.default_rng(8)
    x = Both(ctx, rng, 2, 4, 8)
    x.compact()
    x.advance(new=[64, 64])
    x.compact()
    x.advance([1, -1])
    x.compact()
    assert (x.table[0] == np.arange(4)).sum() == 4 or x.table[0].max() == 3


def test_refusals(ctx):
    import torch
    from vokra_b200 import _lib, blockkv
    from vokra_b200.ops import VkbError
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    arena = torch.zeros(2, 8, 4, device="cuda")
    pool = blockkv.PagePool(ctx, [arena], i(1))
    a, b = blockkv.PageState.empty(3, 4, 8), blockkv.PageState.empty(3, 4, 8)
    bad = [
        lambda: pool.advance(a, a), lambda: pool.compact(a, a), lambda: pool.advance(a, blockkv.PageState(a.table, b.len, b.refs)),
        lambda: pool.advance(a, blockkv.PageState.empty(3, 5, 8)), lambda: pool.advance(a, b, i(2)), lambda: pool.advance(a, b, i(3).long()),
        lambda: pool.advance(blockkv.PageState.empty(3, 4, 9), blockkv.PageState.empty(3, 4, 9)),
        lambda: blockkv.PagePool(ctx, [arena, torch.zeros(2, 7, 4, device="cuda")], i(1)),
        lambda: blockkv.PagePool(ctx, [arena.transpose(0, 1)], i(1)), lambda: blockkv.PagePool(ctx, [arena], None),
        lambda: blockkv.PagePool(ctx, [arena] * 9, i(1)).advance(a, b), lambda: blockkv.PageState(i(3, 4), i(2), i(8)),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(VkbError) as e:
            call()
        assert e.value.code == _lib.ERROR_INVALID_ARGUMENT, n
    pool.check()
    pool.advance(a, b, None, i(3) + 100)
    with pytest.raises(VkbError) as e:
        pool.check()
    assert e.value.code == _lib.ERROR_INVALID_ARGUMENT
    pool.status.zero_()
    pool.advance(a, b, None, i(3) + 64)
    with pytest.raises(VkbError) as e:
        pool.check()
    assert e.value.code == _lib.ERROR_KV_CACHE_EXHAUSTED
