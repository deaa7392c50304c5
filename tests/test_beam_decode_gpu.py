"""The decode loop of examples/beam_decode.py: cache, page tables, rules and top-k together.

Each hypothesis is scored again alone, in 64 bits: the decoder's formulas in numpy over a plain cache (one stream,
pages in order) that takes the prompt in one chunk and then token by token, the rules and the log-probabilities of
the plain forms of the operators' own tests. Wrong parents, pages or lengths give other logits.

Bound: the products are exact to about 2^-21 of their terms, the operators to 2e-4 of values up to 4.5, so a
logit of size below 16 is off by about 1e-3 after two layers. An element of K or V whose rounding to 8 bits
falls the other way moves by 1 / 127 of its block's maximum: one of 2 * 64 channels of one of >= 3 tokens, with a
weight below 1, moves a head's output by less than 4.5 / 127 = 0.036 of one channel in 512, a logit by about
2 * 0.036 / sqrt(512) = 3e-3. A token's log-probability is taken to 1e-2."""
import numpy as np
import pytest
from scipy.special import erf

from tests.test_blockkv_gpu import Plain
from tests.test_logits_gpu import plain_rules

pytestmark = pytest.mark.gpu


class PlainDecoder:
    def __init__(self, model):
        from vokra_b200 import synth
        self.m = model
        self.w = {n: synth.dequantize(model.tag, p, rows * cols).reshape(rows, cols).astype(np.float64)
                  for n, (p, rows, cols) in model.payloads.items()}
        self.embed = model.embed.cpu().numpy().astype(np.float64)

    @staticmethod
    def norm(x):
        return x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-6)

    def start(self, max_len):
        pages = -(-max_len // 16)
        self.table = np.arange(pages, dtype=np.int32)[None]
        self.caches = [Plain(pages, self.m.n_kv_head, self.m.d_head) for _ in range(self.m.n_layer)]
        self.n = 0

    def step(self, tokens):
        m, n = self.m, len(tokens)
        self.n += n
        start, lens = [0, n], [self.n]
        x = self.embed[tokens]
        hq, hk = m.n_head * m.d_head, m.n_kv_head * m.d_head
        for i, cache in enumerate(self.caches):
            qkv = self.norm(x) @ self.w[f"qkv{i}"].T
            k, v = (t.reshape(n, m.n_kv_head, m.d_head) for t in (qkv[:, hq:hq + hk], qkv[:, hq + hk:]))
            cache.append(self.table, start, lens, k, v)
            y = cache.attention(self.table, start, lens, qkv[:, :hq].reshape(n, m.n_head, m.d_head), m.d_head**-0.5)
            x = x + y.reshape(n, hq) @ self.w[f"o{i}"].T
            h = self.norm(x) @ self.w[f"up{i}"].T
            x = x + (0.5 * h * (1 + erf(h / np.sqrt(2)))) @ self.w[f"down{i}"].T
        return self.norm(x[-1:]) @ self.w["head"].T


@pytest.mark.parametrize("n_head,n_kv_head,d_head,beams,steps", [(8, 2, 64, 4, 40), (4, 4, 32, 3, 19), (4, 1, 128, 1, 20)])
def test_scores_of_the_hypotheses(ctx, n_head, n_kv_head, d_head, beams, steps):
    from examples import beam_decode as bd
    vocab, eot, banned = 259, 7, (3, 4)
    model = bd.Decoder(ctx, vocab=vocab, d_model=128, n_layer=2, n_head=n_head, n_kv_head=n_kv_head, d_head=d_head, seed=5)
    rng = np.random.default_rng(6)
    prompts = [[int(t) for t in rng.integers(8, vocab, n)] for n in (3, 16, 37)]
    tokens, scores, (cache, state) = bd.beam_search(model, prompts, beams, steps, eot, banned=banned)
    tokens, scores = tokens.cpu().numpy(), scores.cpu().numpy()
    bias = np.zeros((1, vocab), np.float32)
    bias[0, eot] = -1
    mask = bd.allowed(vocab, [t for t in range(vocab) if t not in banned])[None]
    plain = PlainDecoder(model)
    for c, prompt in enumerate(prompts):
        assert (np.diff(scores[c]) <= 0).all()
        assert len({tuple(t) for t in tokens[c].tolist()}) == beams
        for b in range(beams):
            plain.start(len(prompt) + steps)
            told, total, n = list(prompt), 0.0, 0
            for i in range(steps):
                x = plain.step(told if i == 0 else told[-1:])
                y = plain_rules(x, vocab, np.array([told], np.int32), None, np.array([1.2], np.float32), no_repeat_ngram=3,
                                bias=bias, mask=mask)[0].astype(np.float64)
                t = int(tokens[c, b, i])
                total += y[t] - y.max() - np.log(np.exp(y - y.max()).sum())
                told.append(t)
                n += 1
                if t == eot:
                    assert (tokens[c, b, i:] == eot).all()
                    break
            assert abs(total - scores[c, b]) <= 1e-2 * n, (c, b, total, scores[c, b])
    # tables, lengths and counts agree
    table, length, refs = (t.cpu().numpy() for t in (state.table, state.len, state.refs))
    assert (length == np.repeat([len(p) + steps - 1 for p in prompts], beams)).all()
    listed = np.concatenate([row[:-(-n // 16)] for row, n in zip(table, length)])
    assert (np.bincount(listed, minlength=len(refs)) == refs).all()
    assert sum(-(-n // 16) for n in length) >= (refs > 0).sum()


def test_pages_that_run_out(ctx):
    from examples import beam_decode as bd
    from vokra_b200._lib import VkbError
    model = bd.Decoder(ctx, vocab=259, d_model=64, n_layer=1, n_head=2, n_kv_head=1, d_head=32)
    with pytest.raises(VkbError, match="exhausted"):
        bd.beam_search(model, [[9, 8, 7]], 4, 20, 0, n_pages=2)


def test_a_step_in_a_graph(ctx):
    """A recorded step reads tables, lengths, counts, history and masks when it runs."""
    import torch
    from vokra_b200 import logits, ops
    from vokra_b200.blockkv import Batch, BlockKvCache, PageState
    n_seq, heads, group, d, vocab, n_pages, ld = 3, 2, 4, 64, 999, 64, 8
    rng = np.random.default_rng(3)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        own = ops.Context(0)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        k, v = (torch.zeros(n_seq, heads, d, device="cuda", dtype=torch.float16) for _ in range(2))
        q = torch.zeros(n_seq, heads * group, d, device="cuda", dtype=torch.float16)
        x = torch.zeros(n_seq, vocab, device="cuda")
        history = torch.zeros(n_seq, 6, dtype=torch.int32, device="cuda")
        rules = logits.LogitsRules(history=history, frequency=torch.ones(n_seq, device="cuda"))
        parent = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
        one = torch.ones(n_seq, dtype=torch.int32, device="cuda")
        start = torch.arange(n_seq + 1, dtype=torch.int32, device="cuda")
        y, ids, lp = torch.empty_like(q), torch.empty(n_seq, 4, dtype=torch.int32, device="cuda"), torch.empty(n_seq, 4, device="cuda")

        def world():
            cache = BlockKvCache.empty(own, 1, heads, d, n_pages)
            return cache, cache.pages(status), PageState.empty(n_seq, ld, n_pages), PageState.empty(n_seq, ld, n_pages)

        def step(cache, pages, a, b):
            pages.advance(a, b, parent, one)
            batch = Batch(start, b.len, b.table, n_seq, 1, status)
            cache.append(0, batch, k, v)
            cache.attention(0, batch, q, 0.125, out=y)
            logits.topk(own, x, 4, rules, ids=ids, logprobs=lp)
            for s, t in ((b.table, a.table), (b.len, a.len), (b.refs, a.refs)):
                t.copy_(s)

        recorded, eager = world(), world()
        step(*world())  # sizes the scratch
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(*recorded)
    with torch.cuda.stream(stream):
        for i in range(40):
            for t in (k, v, q, x):
                t.copy_(torch.from_numpy(rng.standard_normal(t.shape).astype(np.float32)))
            history.copy_(torch.from_numpy(rng.integers(0, vocab, (n_seq, 6)).astype(np.int32)))
            parent.copy_(torch.from_numpy(rng.integers(0, n_seq, n_seq).astype(np.int32)))
            graph.replay()
            got = [t.clone() for t in (y, ids, lp)]
            step(*eager)
            assert all(torch.equal(g, t) for g, t in zip(got, (y, ids, lp))), i
    assert int(status) == 0 and int(recorded[2].len[0]) == 40
