"""Answering over an index: passages are found by the flat search, their texts
stand as prompts before a small random decoder whose keys and values are held in
4 bits, and the decoder answers.

    python examples/answer.py [--layers 2] [--width 512] [--passages 4] [--tokens 16]

The decoder has random weights, so its answer means nothing; the program shows
the calls of a serving loop in their order, and returns what it computed.

  1. queries find their passages             Index.search
  2. the passages' tokens run as one pack    prompt_attention, extend, append
  3. each question continues its passages:   copy-on-write fork of the prefix,
     its own keys behind those read back     extend, append, read, prompt_attention
  4. answers, a token a step                 extend, append, attend
  5. drafted tokens, checked in one step,    attend with several rows, truncate
     kept as far as they agree
  6. what is no longer needed goes           free, compact
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from ultravec_ann_b200_loader import load  # noqa: E402


def ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def starts(counts):
    return ints([sum(counts[:i]) for i in range(len(counts) + 1)])


class Decoder:
    """A pre-norm decoder with grouped heads and rotary positions."""

    def __init__(self, layers, width, heads, kv_heads, vocab, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, width // heads

        def weight(*shape):
            w = torch.randn(*shape, generator=g, device="cuda") / math.sqrt(shape[-1])
            return w.bfloat16()

        self.embed = weight(vocab, width) * math.sqrt(width)
        self.qkv = [weight((heads + 2 * kv_heads) * self.dim, width) for _ in range(layers)]
        self.out = [weight(width, width) for _ in range(layers)]
        self.up = [weight(4 * width, width) for _ in range(layers)]
        self.down = [weight(width, 4 * width) for _ in range(layers)]

    @staticmethod
    def norm(x):
        return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).bfloat16()

    def rotary(self, x, position):
        half = self.dim // 2
        angle = position[:, None].float() * torch.exp(
            -math.log(10000.0) / half * torch.arange(half, device="cuda"))
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        a, b = x.float().split(half, -1)
        return torch.cat((a * c - b * s, a * s + b * c), -1).bfloat16()

    def __call__(self, tokens, position, attend):
        """Logits of packed tokens; attend(layer, q, k, v) is the attention."""
        x = self.embed[tokens]
        for i in range(len(self.qkv)):
            qkv = (self.norm(x) @ self.qkv[i].T).unflatten(-1, (-1, self.dim))
            q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), 1)
            a = attend(i, self.rotary(q, position), self.rotary(k, position), v)
            x = x + a.flatten(1) @ self.out[i].T
            x = x + torch.nn.functional.gelu(self.norm(x) @ self.up[i].T) @ self.down[i].T
        return (self.norm(x) @ self.embed.T).float()


def main(layers=2, width=512, passages=4, tokens=16, questions=3, seed=0):
    uv = load()
    g = torch.Generator(device="cuda").manual_seed(seed)
    heads, kv_heads, vocab, drafts = width // 128, max(1, width // 512), 1000, 4

    # 1. the index, and which passages each question gets
    rows = torch.randn(5000, 128, generator=g, device="cuda")
    index = uv.Index(uv.Codec(128, 2, 8))
    index.add_batch(rows)
    found, _ = index.search(torch.randn(questions, 128, generator=g, device="cuda"), passages)
    lengths = [40 + int(i) % 150 for i in found.flatten()]
    texts = [[int(x) for x in torch.randint(0, vocab, (sum(lengths[q * passages:(q + 1) * passages]),),
                                            generator=g, device="cuda")] for q in range(questions)]
    asked = [[int(x) for x in torch.randint(0, vocab, (7 + q,), generator=g, device="cuda")]
             for q in range(questions)]

    model = Decoder(layers, width, heads, kv_heads, vocab)
    longest = max(len(t) for t in texts) + max(len(a) for a in asked) + tokens + 2 * drafts + 2
    pages = 2 * sum(-(-(len(t) + longest) // 64) for t in texts)
    cache = uv.KvCache(model.dim, kv_heads, pages, 2 * questions, longest, layers=layers)
    base, live = list(range(questions)), list(range(questions, 2 * questions))
    used = {s: 0 for s in base + live}

    def grow(seqs, counts):
        cache.extend(ints(seqs), ints(counts))
        for s, n in zip(seqs, counts):
            used[s] += n

    def positions(seqs, counts):
        return torch.cat([torch.arange(used[s] - n, used[s], device="cuda")
                          for s, n in zip(seqs, counts)])

    # 2. the passages, packed, each question's as one prompt
    counts = [len(t) for t in texts]
    grow(base, counts)
    at = starts(counts)

    def prompt(i, q, k, v):
        cache.append(ints(base), k, v, at, layer=i)
        return uv.prompt_attention(q, k, v, at)

    model(torch.tensor(sum(texts, []), device="cuda"), positions(base, counts), prompt)

    # 3. the questions continue a shared prefix: a later question about the same
    #    passages would fork it again
    cache.fork(ints(base), ints(live))
    used.update({s: used[b] for s, b in zip(live, base)})
    new = [len(a) for a in asked]
    grow(live, new)
    whole = [used[s] for s in live]

    def question(i, q, k, v):
        cache.append(ints(live), k, v, starts(new), layer=i)
        k, v = cache.read(ints(live), starts(whole), sum(whole), layer=i)
        return uv.prompt_attention(q, k, v, starts(new), starts(whole))

    logits = model(torch.tensor(sum(asked, []), device="cuda"), positions(live, new), question)
    last = logits[torch.tensor([sum(new[:i + 1]) - 1 for i in range(questions)], device="cuda")]

    # 4. the answers
    answers = [[] for _ in live]
    pick = last.argmax(-1)
    for _ in range(tokens):
        for a, t in zip(answers, pick.tolist()):
            a.append(t)
        grow(live, [1] * questions)

        def step(i, q, k, v):
            cache.append(ints(live), k, v, layer=i)
            return cache.attend(ints(live), q, layer=i)

        logits = model(pick, positions(live, [1] * questions), step)
        pick = logits.argmax(-1)

    # 5. drafts: the same model is the drafter here, with its guesses spoilt at
    #    one place, so the check keeps the tokens before it
    guess = torch.randint(0, vocab, (questions, drafts), generator=g, device="cuda")
    guess[:, 0] = pick
    grow(live, [drafts] * questions)
    at = starts([drafts] * questions)

    def verify(i, q, k, v):
        cache.append(ints(live), k, v, at, layer=i)
        return cache.attend(ints(live), q, at, drafts, layer=i)

    logits = model(guess.flatten(), positions(live, [drafts] * questions), verify)
    says = logits.argmax(-1).view(questions, drafts)
    agree = (says[:, :-1] == guess[:, 1:]).cumprod(1).sum(1) + 1
    for s, n in zip(live, agree.tolist()):
        used[s] += n - drafts
    cache.truncate(ints(live), ints(used[s] for s in live))

    # 6. the passages go, the answers' pages close up
    cache.free(ints(base))
    cache.compact()
    cache.check()
    return dict(answers=answers, kept=agree.tolist(), lens=cache.lens.tolist(),
                used=[0] * questions + [used[s] for s in live],
                pages=int((cache.refs > 0).sum()), logits=last, cache=cache, model=model,
                texts=texts, asked=asked)


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("layers", 2), ("width", 512), ("passages", 4), ("tokens", 16), ("questions", 3)):
        p.add_argument("--" + name, type=int, default=value)
    got = main(**vars(p.parse_args()))
    for i, a in enumerate(got["answers"]):
        print(f"question {i}: {len(got['texts'][i])} tokens of passages, answer {a}, "
              f"{got['kept'][i]} drafted kept")
    print(f"{got['pages']} pages of {got['cache'].n_pages} in use, tokens {got['lens']}")
