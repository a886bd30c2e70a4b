#!/usr/bin/env python3
"""Several samples of one prompt over a paged 8-bit key/value cache (q38hip.kv).

A small attention-only model with random weights reads a prompt in one call,
is forked into samples that share the prompt's pages, and generates a token per
sample and step.  Half way the samples of lowest probability are dropped and
the others forked again; at the end the pool is compacted.

    python examples/parallel_samples.py [--samples 4] [--steps 24] [--prompt 300] [--kind int8]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3.8-27b-in-c_amd"))
from q38hip import kv  # noqa: E402

LAYERS, HEADS, KV_HEADS, DIM, WIDTH, WORDS = 3, 24, 4, 256, 512, 1000


class Model:
    def __init__(self, seed, device):
        g = torch.Generator(device="cpu").manual_seed(seed)
        weight = lambda rows, columns: (torch.randn(rows, columns, generator=g) * rows ** -0.5).to(device)  # noqa: E731
        self.words = (torch.randn(WORDS, WIDTH, generator=g)).to(device)
        self.layers = [(weight(WIDTH, HEADS * 2 * DIM), weight(WIDTH, 2 * KV_HEADS * DIM), weight(HEADS * DIM, WIDTH))
                       for _ in range(LAYERS)]
        self.out = weight(WIDTH, WORDS)

    def step(self, cache, tokens, sequences, row_starts=None):
        """log-probabilities behind each of `tokens`, the last rows of `sequences`"""
        x = self.words[tokens]
        for layer, (to_query, to_kv, back) in enumerate(self.layers):
            y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-6)
            both = (y @ to_query).unflatten(1, (HEADS, 2 * DIM))          # queries and gates, interleaved by head
            rows = (y @ to_kv).unflatten(1, (2, KV_HEADS, DIM))
            cache.append(layer, rows[:, 0], rows[:, 1], sequences, row_starts)
            out = cache.attention(layer, both[..., :DIM], sequences, row_starts, gate=both[..., DIM:])
            x = x + out.flatten(1) @ back
        x = x * torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-6)
        return torch.log_softmax(x @ self.out, 1)


def generate(model, prompt, samples, steps, kind, noise, device):
    """tokens [samples, steps], the last step's log-probabilities, and the cache"""
    words = lambda values: torch.tensor(values, dtype=torch.int32, device=device)  # noqa: E731
    tokens_most = len(prompt) + steps
    cache = kv.KVPages.allocate(LAYERS, pages=2 * samples * (tokens_most // 64 + 2), page_tokens=64, kv_heads=KV_HEADS,
                                head_dim=DIM, sequences=2 * samples, table_entries=tokens_most // 64 + 1, kind=kind,
                                device=device)
    cache.extend(words([0]), words([len(prompt)]))
    log_p = model.step(cache, prompt, words([0]))[-1:].expand(samples, -1)
    active = list(range(samples))
    if samples > 1:
        cache.fork(words([0] * (samples - 1)), words(active[1:]))
    taken, total = [], torch.zeros(samples, device=device)
    for step in range(steps):
        if step == steps // 2 and samples > 1:
            # the better half, and a second sample of each in place of the others
            order = torch.argsort(total, descending=True).tolist()
            keep = order[:(samples + 1) // 2]
            drop, fresh = order[len(keep):], [i for i in range(2 * samples) if i not in active][:samples - len(keep)]
            cache.truncate(words([active[i] for i in drop]), words([0] * len(drop)))
            parents = keep[:len(fresh)]
            cache.fork(words([active[i] for i in parents]), words(fresh))
            rows = torch.tensor(keep + parents, device=device)
            active = [active[i] for i in keep] + fresh
            log_p, total, taken = log_p[rows], total[rows], [t[rows] for t in taken]
        pick = (log_p + noise[step, :samples]).argmax(1)                  # Gumbel noise: a sample of the distribution
        total = total + log_p.gather(1, pick[:, None])[:, 0]
        taken.append(pick)
        ids = words(active)
        cache.extend(ids, torch.ones_like(ids))
        log_p = model.step(cache, pick, ids)
    moved = cache.compact()
    cache.check()
    return torch.stack(taken, 1), log_p, cache, active, moved.tolist()


def main(arguments=None):
    p = argparse.ArgumentParser()
    p.add_argument("--samples", type=int, default=4)
    p.add_argument("--steps", type=int, default=24)
    p.add_argument("--prompt", type=int, default=300)
    p.add_argument("--kind", choices=tuple(kv.KINDS), default="int8")
    p.add_argument("--seed", type=int, default=1)
    a = p.parse_args(arguments)
    device = torch.device("cuda:0")
    model = Model(a.seed, device)
    g = torch.Generator(device="cpu").manual_seed(a.seed + 1)
    prompt = torch.randint(0, WORDS, (a.prompt,), generator=g).to(device)
    noise = -torch.log(-torch.log(torch.rand(a.steps, a.samples, WORDS, generator=g).clamp(1e-9, 1 - 1e-7))).to(device)
    tokens, _, cache, active, moved = generate(model, prompt, a.samples, a.steps, a.kind, noise, device)
    for sequence, row in zip(active, tokens.tolist()):
        print("sequence %d: %s" % (sequence, " ".join(map(str, row))))
    print("pages in use %d of %d, %d moved to the front; %.1f MB for %d tokens of %d sequences"
          % (moved[1], cache.pages, moved[0], moved[1] * cache.data[:, 0].numel() / 1e6, int(cache.lengths.sum()), len(active)))


if __name__ == "__main__":
    main()
