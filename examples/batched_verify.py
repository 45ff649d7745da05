"""Speculative decoding of many requests from one NVFP4 pool.

    python examples/batched_verify.py [--requests R] [--steps N]

A toy model (one attention layer with random weights, 24/4/256 heads, whose
tokens tend to follow one another round blocks of sixteen) serves requests that join with prompts of different lengths, draft by repeating the
last occurrence of their last token, verify the drafts in windows, and leave.
Every step is the same four calls, with all lengths on the device:

    batch.build_tables     pages, block tables, slot map, row offsets
    batch.append           the step's K/V rows into their slots
    batch.attend           attention of all rows over their pages
    scoring.token_logprobs the drafted tokens' log probabilities, the entropy
                           and the model's own choice (top 1) for every row

The host reads back what a server needs to answer its clients: the top token of
every row, from which it counts the accepted drafts.
"""
from __future__ import annotations

import argparse
import random
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from qwarz_b200 import batch, scoring  # noqa: E402

HEADS, KV_HEADS, DIM, VOCAB, HIDDEN, DRAFTS, TOP = 24, 4, 256, 8192, 512, 6, 4


class Toy:
    """Embedding, one attention layer, unembedding; random BF16 weights."""

    KEEP = 0.1  # of the embedding beside what attention adds

    def __init__(self, device, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)

        def w(rows, cols):
            return (torch.randn(rows, cols, generator=g, device=device) / rows ** 0.5).bfloat16()

        self.embed = w(VOCAB, HIDDEN) * VOCAB ** 0.5
        self.unembed = self.embed.view(-1, 16, HIDDEN).roll(1, 1).view(VOCAB, HIDDEN)  # token t is followed by t + 1
        self.qkv, self.o = w(HIDDEN, (HEADS + 2 * KV_HEADS) * DIM), w(HEADS * DIM, HIDDEN)

    def project(self, tokens):
        """Rows of a packed projection: q, k and v are views of it."""
        rows = (self.embed[tokens] @ self.qkv).view(-1, HEADS + 2 * KV_HEADS, DIM)
        return rows[:, :HEADS], rows[:, HEADS:HEADS + KV_HEADS], rows[:, HEADS + KV_HEADS:]

    def logits(self, tokens, attended):
        return (self.KEEP * self.embed[tokens] + attended.flatten(1) @ self.o) @ self.unembed.T


class Server:
    """`requests` slots over a pool of `pages` pages; a step serves them all."""

    def __init__(self, device, requests, width, pages, rows):
        def i32(*shape):
            return torch.zeros(*shape, dtype=torch.int32, device=device)

        self.device, self.rows = device, rows
        self.lengths, self.held, self.table = i32(requests), i32(requests), i32(requests, width)
        self.ring = torch.arange(pages, dtype=torch.int32, device=device)
        self.ring_state = torch.tensor([0, pages], dtype=torch.int32, device=device)
        self.cu, self.kv = i32(requests + 1), i32(requests)
        self.held_out, self.ring_out = i32(requests), i32(2)
        self.slots, self.positions, self.request_of = i32(rows), i32(rows), i32(rows)
        pool = [torch.zeros(pages, 256, KV_HEADS, n, dtype=torch.uint8, device=device)
                for n in (DIM // 2, DIM // 2, DIM // 16, DIM // 16)]
        self.pool = pool[:2] + [s.view(torch.float8_e4m3fn) for s in pool[2:]]
        self.out = torch.zeros(rows, HEADS, DIM, dtype=torch.bfloat16, device=device)
        self.attend_ws = batch.attend_workspace(device, DIM)
        self.score_ws = scoring.workspace(device, rows, VOCAB, TOP)

    def step(self, model, new_rows, tokens, targets, max_rows):
        """Runs the step's rows (`tokens`, request by request; new_rows < 0 ends a
        request) and scores `targets`, the token drafted after each row (-1:
        none).  Returns per row: log probability, entropy, top tokens."""
        T = tokens.numel()
        batch.build_tables(self.lengths, new_rows, self.held, self.ring, self.ring_state, self.table, self.cu,
                           self.kv, self.held_out, self.ring_out, self.slots[:T], self.positions[:T],
                           self.request_of[:T])
        q, k, v = model.project(tokens)
        batch.append(k, v, *self.pool, self.slots[:T])
        batch.attend(q, *self.pool, self.table, self.cu, self.kv, self.out[:T], self.attend_ws, max_rows)
        logits = model.logits(tokens, self.out[:T])
        logprob, entropy = (torch.empty(T, device=self.device) for _ in range(2))
        top, ids = torch.empty(T, TOP, device=self.device), torch.empty(T, TOP, dtype=torch.int32, device=self.device)
        scoring.token_logprobs(logits, targets, logprob, entropy, top, ids, self.score_ws)
        return logprob, entropy, ids

    def commit(self, kept):
        """Keeps `kept` tokens of every request; the slots of rejected rows are
        simply written again."""
        self.lengths.copy_(kept)
        self.held.copy_(self.held_out)
        self.ring_state.copy_(self.ring_out)


def draft(text):
    """Up to DRAFTS tokens that followed the last earlier occurrence of the last one."""
    for i in range(len(text) - 2, -1, -1):
        if text[i] == text[-1]:
            return text[i + 1:i + 1 + DRAFTS]
    return []


def serve(requests=8, steps=20, seed=0, say=print):
    device = torch.device("cuda", torch.cuda.current_device())
    rng = random.Random(seed)
    model = Toy(device, seed)
    server = Server(device, requests, width=16, pages=requests * 4, rows=requests * 700)
    texts = [[] for _ in range(requests)]
    done = [0] * requests          # tokens of a request that are in the cache
    drafted = accepted = finished = 0
    surprise = 0.0
    for step in range(steps):
        new, tokens, targets, plan = [], [], [], []
        for r in range(requests):
            if len(texts[r]) > 900 or (texts[r] and rng.random() < 0.03):  # the request ends, another takes its slot
                new.append(-1)
                texts[r], done[r] = [], 0
                finished += 1
                plan.append(None)
                continue
            if not texts[r]:
                texts[r] = [rng.randrange(VOCAB // 64) for _ in range(rng.randint(1, 600))]
            row = texts[r][done[r]:]           # the prompt, or the last token
            guess = draft(texts[r]) if len(row) == 1 else []
            plan.append((len(tokens), len(row), guess))
            tokens += row + guess
            targets += [-1] * (len(row) - 1) + guess + [-1]
            new.append(len(row) + len(guess))
        out = server.step(model, torch.tensor(new, dtype=torch.int32, device=device),
                          torch.tensor(tokens, dtype=torch.long, device=device),
                          torch.tensor(targets, dtype=torch.long, device=device), max(max(new), 1))
        logprob, _, ids = (t.cpu() for t in out)
        for r, p in enumerate(plan):
            if p is None:
                continue
            at, n, guess = p
            choice = ids[at + n - 1:at + n + len(guess), 0].tolist()  # the model's token after each row
            good = 0
            while good < len(guess) and guess[good] == choice[good]:
                good += 1
            texts[r] += choice[:good + 1]
            done[r] = len(texts[r]) - 1
            drafted, accepted = drafted + len(guess), accepted + good
            surprise -= float(logprob[at + n - 1:at + n - 1 + len(guess)].sum())
        server.commit(torch.tensor(done, dtype=torch.int32, device=device))
        say(f"step {step}: {len(tokens)} rows, {sum(done)} tokens cached")
    free = int(server.ring_state[1])
    say(f"{finished} requests ended, {accepted} of {drafted} drafts accepted, "
        f"{surprise / max(drafted, 1):.2f} nats a draft, {free} pages free")
    return {"finished": finished, "drafted": drafted, "accepted": accepted, "free": free,
            "held": int(server.held.sum()), "pages": server.ring.numel(), "cached": sum(done),
            "lengths": server.lengths.tolist(), "done": done}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    serve(a.requests, a.steps)
