"""Beam search with the whole decode loop on the device: paged 8-bit KV cache, page tables, logits rules, top-k.

A small decoder with random weights (grouped heads, RMS norms, GELU) continues a few prompts. In each step

    pages.advance     beams take over their parents' pages (a shared, partly filled page is copied) and grow by a token
    cache.append      the step's K and V rows, in 8 bits
    cache.attention   causal attention of the step's rows over their streams
    logits.topk       penalties, repeated n-grams, biases and masks, then the best tokens' log-probabilities

and the few numbers between them (which beam continues which) are torch tensors: nothing is read back before the
end, so the host only launches. Half-way the pages in use are moved to the front of the arenas (pages.compact).

    python examples/beam_decode.py --clips 4 --beams 5 --steps 40
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from vokra_b200 import _lib, logits, ops, synth  # noqa: E402
from vokra_b200.blockkv import Batch, BlockKvCache, PageState  # noqa: E402


class Decoder:
    """n_layer blocks x += Wo attention(rms(x)), x += W2 gelu(W1 rms(x)); tied to nothing, no positions."""

    def __init__(self, ctx, vocab=1009, d_model=256, n_layer=2, n_head=8, n_kv_head=2, d_head=64, tag=synth.Q8_0, seed=0):
        self.ctx, self.vocab, self.n_layer = ctx, vocab, n_layer
        self.n_head, self.n_kv_head, self.d_head = n_head, n_kv_head, d_head
        rng = np.random.default_rng(seed)
        self.tag, self.payloads, self.weights = tag, {}, {}

        def weight(name, n, k, gain=1.0):
            w = synth.quantize(tag, (gain * rng.standard_normal(n * k) / np.sqrt(k)).astype(np.float32))
            self.payloads[name] = (w, n, k)
            self.weights[name] = ops.Weight(ctx, tag, n, k, w)

        for i in range(n_layer):
            weight(f"qkv{i}", (n_head + 2 * n_kv_head) * d_head, d_model)
            weight(f"o{i}", d_model, n_head * d_head)
            weight(f"up{i}", 4 * d_model, d_model)
            weight(f"down{i}", d_model, 4 * d_model)
        weight("head", vocab, d_model, 2.0)
        self.embed = torch.from_numpy(rng.standard_normal((vocab, d_model)).astype(np.float32)).cuda()

    def linear(self, name, a, **kw):
        out = torch.empty(a.shape[0], self.weights[name].n, device=a.device)
        ops.linear(self.ctx, self.weights[name], a, out, **kw)
        return out

    @staticmethod
    def norm(x):
        return x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-6)

    def step(self, cache, batch, tokens, last):
        """Logits [len(last), vocab] of the rows `last` of the batch's tokens."""
        x = self.embed[tokens.long().clamp(0, self.vocab - 1)]
        hq, hk = self.n_head * self.d_head, self.n_kv_head * self.d_head
        for i in range(self.n_layer):
            qkv = self.linear(f"qkv{i}", self.norm(x))
            cache.append(i, batch, qkv[:, hq:hq + hk], qkv[:, hq + hk:])
            y = torch.empty(x.shape[0], hq, device=x.device)
            cache.attention(i, batch, qkv[:, :hq], self.d_head**-0.5, out=y)
            x = self.linear(f"o{i}", y, epilogue=_lib.EPI_RESIDUAL, residual=x)
            h = self.linear(f"up{i}", self.norm(x), epilogue=_lib.EPI_GELU)
            x = self.linear(f"down{i}", h, epilogue=_lib.EPI_RESIDUAL, residual=x)
        return self.linear("head", self.norm(x[last]))


def allowed(vocab, tokens):
    """A mask row with these tokens' bits."""
    bits = np.zeros(((vocab + 31) // 32) * 32, np.uint8)
    bits[tokens] = 1
    return np.packbits(bits, bitorder="little").view(np.int32)


def beam_search(model, prompts, beams, steps, eot, repetition=1.2, no_repeat_ngram=3, banned=(), n_pages=None):
    """(tokens int32 [clips, beams, steps], scores f32 [clips, beams], states): for each prompt (a list of tokens) the
    best continuations, the best first; a beam that has reached `eot` repeats it."""
    ctx, vocab, dev = model.ctx, model.vocab, "cuda"
    clips, n_seq = len(prompts), len(prompts) * beams
    max_len = max(len(p) for p in prompts) + steps
    max_pages = -(-max_len // 16)
    # a beam shares the whole pages in front of its fork: this is enough whatever happens
    n_pages = n_pages or n_seq * max_pages + n_seq
    cache = BlockKvCache.empty(ctx, model.n_layer, model.n_kv_head, model.d_head, n_pages)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    pages = cache.pages(status)
    a, b = PageState.empty(n_seq, max_pages, n_pages), PageState.empty(n_seq, max_pages, n_pages)

    # rules: live beams may take every token but the banned ones, finished ones only `eot` (which then costs nothing)
    history = torch.full((n_seq, max_len), -1, dtype=torch.int32, device=dev)
    history_len = torch.zeros(n_seq, dtype=torch.int32, device=dev)
    mask_row = torch.zeros(n_seq, dtype=torch.int32, device=dev)
    live = [t for t in range(vocab) if t not in banned]
    mask = torch.from_numpy(np.stack([allowed(vocab, live), allowed(vocab, [eot])])).to(dev)
    bias = torch.zeros(1, vocab, device=dev)
    bias[0, eot] = -1.0
    rules = logits.LogitsRules(history=history, history_len=history_len, no_repeat_ngram=no_repeat_ngram,
                               repetition=torch.full((n_seq,), repetition, device=dev), bias=bias, mask=mask, mask_row=mask_row)

    # ---- prompts: the first beam of each clip
    for c, p in enumerate(prompts):
        history[c * beams, :len(p)] = torch.tensor(p, dtype=torch.int32)
    lens = [len(prompts[i // beams]) if i % beams == 0 else 0 for i in range(n_seq)]
    start = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=dev)
    n_new = torch.tensor(lens, dtype=torch.int32, device=dev)
    history_len.copy_(n_new)
    pages.advance(a, b, None, n_new)
    batch = Batch(start, b.len, b.table, sum(lens), max(lens), status, max_kv=max(lens))
    tokens = torch.tensor([t for p in prompts for t in p], dtype=torch.int32, device=dev)
    last = (start[1:] - 1).clamp(min=0).long()
    x = model.step(cache, batch, tokens, last)
    a, b = b, a

    # ---- steps: rows of beam 0 count in the first one
    score = torch.full((clips, beams), -float("inf"), device=dev)
    score[:, 0] = 0
    first = torch.arange(clips, device=dev)[:, None] * beams
    one = torch.ones(n_seq, dtype=torch.int32, device=dev)
    start = torch.arange(n_seq + 1, dtype=torch.int32, device=dev)
    out = torch.full((n_seq, steps), eot, dtype=torch.int32, device=dev)
    seen = history_len.view(clips, beams)[:, :1].repeat(1, beams).view(-1).long()  # history slots of each beam
    done = torch.zeros(n_seq, dtype=torch.bool, device=dev)
    for i in range(steps):
        ids, lp = logits.topk(ctx, x, beams, rules)
        total = (score.view(-1, 1) + lp).view(clips, beams * beams)
        score, pick = total.topk(beams)
        parent = (first + pick // beams).view(-1)
        token = ids.view(clips, -1).gather(1, pick).view(-1)
        out = out[parent]
        out[:, i] = token
        done = done[parent] | (token == eot)
        history.copy_(history[parent])
        history.scatter_(1, seen[:, None], token[:, None])
        seen += 1
        history_len.copy_(torch.where(done, 0, seen))
        mask_row.copy_(done)
        if i + 1 == steps:
            break
        pages.advance(a, b, parent.to(torch.int32), one)
        if i == steps // 2:
            pages.compact(b, a)
        else:
            a, b = b, a
        x = model.step(cache, Batch(start, a.len, a.table, n_seq, 1, status), token, torch.arange(n_seq, device=dev))
    pages.check()
    return out.view(clips, beams, steps), score, (cache, a)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--clips", type=int, default=4)
    ap.add_argument("--beams", type=int, default=5)
    ap.add_argument("--steps", type=int, default=40)
    args = ap.parse_args()
    ctx = ops.Context(0)
    model = Decoder(ctx)
    rng = np.random.default_rng(1)
    prompts = [list(rng.integers(1, model.vocab, 3 + 17 * c)) for c in range(args.clips)]
    beam_search(model, prompts, args.beams, 4, eot=0)  # warm
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record()
    tokens, score, (cache, state) = beam_search(model, prompts, args.beams, args.steps, eot=0)
    t1.record()
    torch.cuda.synchronize()
    used = int((state.refs > 0).sum())
    held = int(((state.len + 15) // 16).sum())
    for c in range(args.clips):
        print(f"clip {c}: score {float(score[c, 0]):8.3f}  tokens {tokens[c, 0].tolist()[:12]} ...")
    print(f"{args.clips * args.beams} streams, {args.steps} steps: {t0.elapsed_time(t1):.1f} ms; "
          f"{used} pages of 16 tokens for {held} that the streams list")


if __name__ == "__main__":
    main()
