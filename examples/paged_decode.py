"""Autoregressive decoding with the paged cache: draw several continuations of each prompt,
keep the best, with log probabilities from the same step.

A small random transformer stands in for the model. Each tick reserves a token's room in
every live slot, runs the layers with ``PagedCache.attend`` (which stores the new keys and
values), samples with ``sample_rows`` and scores the sampled tokens with ``token_logprobs``;
after the prompt every request is forked into ``--beams`` candidates that share its pages,
and at the end all but the most likely one are freed and the pool is packed.

    python examples/paged_decode.py --requests 4 --beams 3 --tokens 24
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from yapd_b200.logprobs import token_logprobs  # noqa: E402
from yapd_b200.paged import PagedCache  # noqa: E402
from yapd_b200.select import sample_rows  # noqa: E402

LAYERS, HEADS, KV_HEADS, DIM, VOCAB = 3, 8, 4, 64, 6563


class Model:
    """Random weights; the shapes of a small decoder."""

    def __init__(self, seed: int, device):
        g = torch.Generator(device=device).manual_seed(seed)
        width = HEADS * DIM
        init = lambda *s: torch.randn(*s, generator=g, device=device).mul_(s[-1] ** -0.5).to(torch.bfloat16)  # noqa: E731
        self.embed = init(VOCAB, width) * 16
        self.qkv = [init((HEADS + 2 * KV_HEADS) * DIM, width) for _ in range(LAYERS)]
        self.out = [init(width, width) for _ in range(LAYERS)]
        self.head = init(VOCAB, width)

    def __call__(self, cache: PagedCache, tokens: torch.Tensor, slots: torch.Tensor, window: int, sinks: int):
        """Logits after the last of each request's new tokens ``(B, T)``, which the slots hold already."""
        B, T = tokens.shape
        x = self.embed[tokens]
        for layer in range(LAYERS):
            h = torch.nn.functional.rms_norm(x, x.shape[-1:])
            q, k, v = (h @ self.qkv[layer].t()).view(B, T, -1, DIM).split([HEADS, KV_HEADS, KV_HEADS], 2)
            a = cache.attend(layer, q, k, v, slots=slots, causal=True, window=window, sinks=sinks)
            x = x + a.reshape(B, T, -1) @ self.out[layer].t()
        return (torch.nn.functional.rms_norm(x[:, -1], x.shape[-1:]) @ self.head.t()).float() * 4


def run(requests: int = 4, beams: int = 3, prompt: int = 40, tokens: int = 24, window: int = 64, sinks: int = 8,
        seed: int = 0, verbose: bool = False):
    """Returns each request's best continuation (token ids) and its total log probability."""
    dev = torch.device("cuda", torch.cuda.current_device())
    model = Model(seed, dev)
    slots = requests * beams
    cache = PagedCache.empty(LAYERS, pages=slots * (-(-(prompt + tokens) // 16) + 1), page_size=16, kv_heads=KV_HEADS,
                             head_dim=DIM, slots=slots, max_pages=-(-(prompt + tokens) // 16) + 1, device=dev)
    every = torch.arange(slots, dtype=torch.int32, device=dev)
    first = every[::beams].contiguous()                      # slot r * beams holds request r's prompt
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    text = torch.randint(0, VOCAB, (requests, prompt), generator=g, device=dev)

    # the prompt, up to 32 tokens a call
    for at in range(0, prompt, 32):
        part = text[:, at:at + 32]
        cache.reserve(part.shape[1], first)
        logits = model(cache, part, first, window, sinks)
    # every candidate starts as a copy of its request: pages are shared until they are written
    others = every[every % beams != 0].contiguous()
    cache.fork((others // beams * beams).contiguous(), others)
    logits = logits.repeat_interleave(beams, 0)

    seen = torch.zeros(slots, VOCAB, dtype=torch.bool, device=dev)
    total = torch.zeros(slots, device=dev)
    drawn = []
    for step in range(tokens):
        token = sample_rows(logits, temperature=0.9, top_k=40, rep_penalty=1.1, seen=seen, seed=seed, offset=step)
        scored = token_logprobs(logits, token, top_n=3)
        total += scored.logprob
        seen.scatter_(1, token.long()[:, None], True)
        drawn.append(token)
        cache.trim(window, sinks)                            # what the next token no longer sees
        cache.reserve(1)
        logits = model(cache, token.long()[:, None], every, window, sinks)

    best = total.view(requests, beams).argmax(1)
    keep = (first + best).to(torch.int32)
    losers = every[~torch.isin(every, keep)].contiguous()
    if len(losers):
        cache.free(losers)
    live = cache.compact()
    sequences = torch.stack(drawn, 1)[keep.long()]
    if verbose:
        for r in range(requests):
            print(f"request {r}: log probability {float(total[keep[r]]):.2f}, tokens {sequences[r].tolist()}")
        print(f"live pages {int(live)} of {cache.refs.numel()}, status {cache.status()}")
    return sequences, total[keep.long()], cache


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("requests", 4), ("beams", 3), ("prompt", 40), ("tokens", 24), ("window", 64), ("sinks", 8),
                        ("seed", 0)):
        ap.add_argument("--" + name, type=int, default=value)
    run(**vars(ap.parse_args()), verbose=True)
