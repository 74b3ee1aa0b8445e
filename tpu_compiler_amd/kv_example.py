"""A language model that answers from a quantised cache: prompts of different lengths are read into it, then every sequence is continued a
token at a time.  The model is small and has random weights; its attention runs on the GPU, its products on the host with float32 weights, or on the
GPU with weights in 4 bits:

    python -m tpu_compiler_amd.kv_example [--bits 4|8] [--tokens N] [--window W --sinks S] [--weights f32|f4] [--pages host|gpu]

What a user of the cache does is in `Sequences`: pages are given out as sequences grow, the new tokens' rows are written to their slots, and
their queries attend to what the pages hold, prompts and single tokens by the same call.  `SequencesOnGpu` gives the pages out on the GPU,
`Model4` multiplies with weights in microscaled 4-bit floating point, and activations that are quantised on the way."""
import argparse

import numpy as np

from . import capi, mx
from .kv_cache import DeviceArray, KVCache, KVPages


class Sequences:
    """sequences of one model in a cache for each of its layers; all layers use the same pages"""

    def __init__(self, ctx, layers, heads, kv_heads, head_dim, bits, pages, page_tokens=64, window=0, sinks=0):
        self.ctx, self.heads, self.page_tokens, self.window, self.sinks = ctx, heads, page_tokens, window, sinks
        self.caches = [KVCache(ctx, pages, kv_heads, head_dim, bits, page_tokens) for _ in range(layers)]
        self.free = list(range(pages))[::-1]
        self.pages, self.lens = [], []

    def begin(self, new_tokens):
        """new_tokens[i] more tokens of sequence i: their slots, and what the layers' calls need"""
        while len(self.lens) < len(new_tokens):
            self.pages.append([])
            self.lens.append(0)
        more = [max(0, -(-(have + n) // self.page_tokens) - len(pages)) for have, n, pages in zip(self.lens, new_tokens, self.pages)]
        if sum(more) > len(self.free):
            raise ValueError("%d pages are wanted, %d are free" % (sum(more), len(self.free)))
        slots = []
        for i, n in enumerate(new_tokens):
            at = np.arange(self.lens[i], self.lens[i] + n)
            self.lens[i] += n
            while len(self.pages[i]) * self.page_tokens < self.lens[i]:
                self.pages[i].append(self.free.pop())
            slots.append(np.array(self.pages[i], np.int64)[at // self.page_tokens] * self.page_tokens + at % self.page_tokens)
        table = np.zeros((len(self.pages), max(map(len, self.pages))), np.int32)
        for row, pages in zip(table, self.pages):
            row[:len(pages)] = pages
        put = lambda v: DeviceArray.of(self.ctx, v, "i32")
        self.step = dict(slots=put(np.concatenate(slots)), starts=put(np.cumsum([0] + list(new_tokens))), lens=put(self.lens), table=put(table),
                         max_q=max(new_tokens), max_kv=max(self.lens))

    def attend(self, layer, q, k, v):
        """[tokens, heads, head_dim] of the new tokens, the sequences' one after the other -> the same of what they attend to"""
        s, cache, put = self.step, self.caches[layer], lambda x: DeviceArray.of(self.ctx, x, "bf16")
        q, k, v, out = put(q), put(k), put(v), DeviceArray(self.ctx, q.shape, "bf16")
        cache.write(k, v, s["slots"])
        cache.attention(q, out, s["starts"], s["lens"], s["table"], max_q=s["max_q"], max_kv=s["max_kv"], window=self.window, sinks=self.sinks)
        result = out.numpy()
        for a in (q, k, v, out):
            a.free()
        return result

    def end(self):
        for k in ("slots", "starts", "lens", "table"):
            self.step[k].free()

    def close(self):
        for c in self.caches:
            c.close()


class SequencesOnGpu(Sequences):
    """the same for a batch of `sequences`, whose pages, slots and starts are found on the GPU"""

    def __init__(self, ctx, layers, heads, kv_heads, head_dim, bits, pages, sequences, page_tokens=64, window=0, sinks=0):
        super().__init__(ctx, layers, heads, kv_heads, head_dim, bits, pages, page_tokens, window, sinks)
        self.batch, self.lens = KVPages(ctx, pages, sequences, pages, page_tokens), [0] * sequences

    def begin(self, new_tokens):
        put, p = lambda v: DeviceArray.of(self.ctx, v, "i32"), self.batch
        new, refused = put(new_tokens), DeviceArray(self.ctx, (1,), "i32")
        self.step = dict(slots=DeviceArray(self.ctx, (sum(new_tokens),), "i32"), starts=DeviceArray(self.ctx, (len(new_tokens) + 1,), "i32"))
        p.grow(new, self.step["starts"], self.step["slots"], refused)
        short = int(refused.numpy()[0])              # a loop on the GPU would go on instead, with those that got theirs
        new.free(), refused.free()
        if short:
            self.trim(self.lens)
            self.end()
            raise ValueError("pages for %d sequences are not there" % short)
        self.lens = [a + n for a, n in zip(self.lens, new_tokens)]
        self.step.update(lens=p.lens, table=p.table, max_q=max(new_tokens), max_kv=max(self.lens))

    def trim(self, keep):
        """the sequences' tokens behind keep[i] go, and their pages are free"""
        a = DeviceArray.of(self.ctx, keep, "i32")
        self.batch.trim(a)
        a.free()
        self.lens = [min(have, k) for have, k in zip(self.lens, keep)]

    def end(self):
        for k in ("slots", "starts"):
            self.step[k].free()

    def close(self):
        super().close()
        for a in (self.batch.lens, self.batch.table, self.batch.free, self.batch.n_free):
            a.free()


class Model:
    """embedding, `layers` of attention with a residual around it, logits"""

    def __init__(self, vocabulary=512, layers=3, heads=8, kv_heads=2, head_dim=64, seed=0):
        rng = np.random.default_rng(seed)
        width = heads * head_dim
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.embedding = rng.standard_normal((vocabulary, width)).astype(np.float32)
        self.logits = (rng.standard_normal((width, vocabulary)) / width ** 0.5).astype(np.float32)
        n = (heads + 2 * kv_heads) * head_dim
        self.qkv = [(rng.standard_normal((width, n)) / width ** 0.5).astype(np.float32) for _ in range(layers)]
        self.out = [(rng.standard_normal((width, width)) / width ** 0.5).astype(np.float32) for _ in range(layers)]

    def product(self, x, weights, residual=None):
        """x times weights (+ residual)"""
        y = x @ weights
        return y if residual is None else residual + y

    def __call__(self, tokens, attend):
        """tokens [n] -> logits [n, vocabulary]; attend(layer, q, k, v)"""
        x = self.embedding[tokens]
        for layer, (qkv, out) in enumerate(zip(self.qkv, self.out)):
            y = self.product(x / np.sqrt((x * x).mean(-1, keepdims=True)), qkv).reshape(len(x), -1, self.head_dim)
            q, k, v = np.split(y, [self.heads, self.heads + self.kv_heads], 1)
            x = self.product(attend(layer, q, k, v).reshape(len(x), -1), out, x)
        return self.product(x / np.sqrt((x * x).mean(-1, keepdims=True)), self.logits)


class Model4(Model):
    """the same with its weights in 4 bits on the GPU, where its products run"""

    def __init__(self, ctx, **sizes):
        super().__init__(**sizes)
        self.ctx = ctx
        self.qkv, self.out, self.logits = [self._quantized(w) for w in self.qkv], [self._quantized(w) for w in self.out], self._quantized(self.logits)

    def _quantized(self, weights):
        a = DeviceArray.of(self.ctx, weights.T, "f32")
        m = mx.MXMatrix(self.ctx, *a.shape).quantize(a)
        a.free()
        return m

    def product(self, x, weights, residual=None):
        put = lambda v: DeviceArray.of(self.ctx, v, "f32")
        a, out = put(x), DeviceArray(self.ctx, (len(x), weights.rows), "f32")
        more = None if residual is None else put(residual)
        mx.product(self.ctx, a, weights, out, residual=more)
        y = out.numpy()
        for v in (a, out) + (() if more is None else (more,)):
            v.free()
        return y

    def close(self):
        for m in self.qkv + self.out + [self.logits]:
            m.free()


def generate(ctx, model, prompts, tokens, bits=4, window=0, sinks=0, page_tokens=64, pages_on_gpu=False):
    """continues each prompt by `tokens` tokens, the likeliest one each time -> (lists of tokens, logits of every step, bytes of the cache)"""
    if not len(prompts) or not all(len(p) for p in prompts):
        raise ValueError("a prompt has a token at least")
    need = sum(-(-(len(p) + tokens) // page_tokens) for p in prompts)
    sizes = (ctx, len(model.qkv), model.heads, model.kv_heads, model.head_dim, bits, need)
    s = SequencesOnGpu(*sizes, len(prompts), page_tokens, window, sinks) if pages_on_gpu else Sequences(*sizes, page_tokens, window, sinks)
    answers, steps, new = [[] for _ in prompts], [], [list(p) for p in prompts]
    for _ in range(tokens):
        s.begin([len(n) for n in new])
        logits = model(np.concatenate(new).astype(np.int64), s.attend)
        s.end()
        last = logits[np.cumsum([len(n) for n in new]) - 1]
        steps.append(last)
        new = [[int(t)] for t in last.argmax(-1)]
        for a, n in zip(answers, new):
            a += n
    size = sum(c.nbytes for c in s.caches)
    s.close()
    return answers, steps, size


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--bits", type=int, default=4, choices=(4, 8))
    ap.add_argument("--tokens", type=int, default=16)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=0)
    ap.add_argument("--weights", default="f32", choices=("f32", "f4"))
    ap.add_argument("--pages", default="host", choices=("host", "gpu"))
    a = ap.parse_args()
    ctx = capi.Context()
    model = Model4(ctx) if a.weights == "f4" else Model()
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, len(model.embedding), n) for n in (5, 130, 64, 1)]
    answers, _, size = generate(ctx, model, prompts, a.tokens, a.bits, a.window, a.sinks, pages_on_gpu=a.pages == "gpu")
    for p, t in zip(prompts, answers):
        print("%4d tokens ->" % len(p), *t)
    print("%d bytes of cache in %d bits" % (size, a.bits))
    ctx.close()


if __name__ == "__main__":
    main()
