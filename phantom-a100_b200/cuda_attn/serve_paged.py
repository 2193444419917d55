"""A small serving loop over the paged cache: ragged prompts are taken in in chunks, tokens are decoded, sequences come and
go and their pages are used again.

    python -m cuda_attn.serve_paged --requests 12 --int8

One attention layer with random weights stands for the model: a token's query, key and value are rows of three tables, the
next token is the one whose output row it is nearest to. Every step packs the new tokens of all running sequences (a chunk
of a prompt, or one token), appends their keys and values and attends; whole finished sequences are read back from the cache
and their last outputs computed again by the dense kernel, as a check.
"""
from __future__ import annotations

import argparse
import sys
from dataclasses import dataclass, field

import torch


class PagePool:
    """Free pages of a pool, and which of them each sequence has."""

    def __init__(self, pages: int, page: int):
        self.page, self.pages = page, pages
        self.free = list(range(pages - 1, -1, -1))
        self.of: dict[int, list[int]] = {}

    def holds(self, tokens: int) -> bool:
        """Whether `tokens` tokens of a sequence fit when nothing else is there."""
        return -(-tokens // self.page) <= self.pages

    def reserve(self, seq: int, tokens: int) -> bool:
        """Give a sequence the pages that `tokens` tokens need; False, and nothing changed, if there are not enough."""
        have = self.of.setdefault(seq, [])
        want = -(-tokens // self.page) - len(have)
        if want > len(self.free):
            return False
        for _ in range(max(0, want)):
            have.append(self.free.pop())
        return True

    def release(self, seq: int) -> None:
        self.free += reversed(self.of.pop(seq, []))


@dataclass
class Request:
    prompt: list[int]
    want: int                                        # tokens to decode
    tokens: list[int] = field(default_factory=list)  # the prompt, then what was decoded
    done: int = 0                                    # of them in the cache


class Server:
    def __init__(self, heads: int = 8, group: int = 4, d: int = 128, page: int = 16, pages: int = 512, vocab: int = 1000,
                 dtype: torch.dtype = torch.bfloat16, int8: bool = False, chunk: int = 256, seed: int = 0, device: str = "cuda"):
        if chunk < 1:
            raise ValueError(f"a chunk has at least one token (got {chunk})")
        g = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.group, self.d, self.chunk, self.dtype, self.device = heads, group, d, chunk, dtype, device

        def table(n):
            return torch.randn(vocab, n, d, device=device, generator=g).to(dtype)

        self.wq, self.wk, self.wv = table(heads * group), table(heads), table(heads)
        self.out = torch.randn(vocab, heads * group * d, device=device, generator=g).to(dtype)
        kind = torch.int8 if int8 else dtype
        self.k_cache, self.v_cache = (torch.zeros(pages, heads, page, d, device=device, dtype=kind) for _ in "kv")
        self.scales = {}
        if int8:
            self.scales = {n: torch.zeros(pages, heads, page, device=device) for n in ("k_scale", "v_scale")}
        self.pool = PagePool(pages, page)
        self.waiting: list[int] = []
        self.running: list[int] = []
        self.requests: dict[int, Request] = {}

    def submit(self, prompt: list[int], want: int) -> int:
        """Queue a request for `want` tokens after a prompt; one that could never run is refused."""
        vocab = self.wq.shape[0]
        if not prompt or want < 1:
            raise ValueError(f"a request needs a prompt and at least one token to decode (got {len(prompt)} and {want})")
        if not all(0 <= t < vocab for t in prompt):
            raise ValueError(f"a prompt's tokens must be from 0 to {vocab - 1}")
        if not self.pool.holds(len(prompt) + want):
            raise ValueError(f"{len(prompt)} + {want} tokens exceed the pool of {self.pool.pages} pages of {self.pool.page} tokens")
        seq = len(self.requests)
        self.requests[seq] = Request(prompt, want, list(prompt))
        self.waiting.append(seq)
        return seq

    def tables(self, seqs: list[int], new: list[int]):
        """page_table, kv_lens (with the new tokens) and cu_new of some sequences, on the GPU."""
        width = max(len(self.pool.of[s]) for s in seqs)
        rows = [self.pool.of[s] + [-1] * (width - len(self.pool.of[s])) for s in seqs]
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        lens = [self.requests[s].done + n for s, n in zip(seqs, new)]
        return [torch.tensor(x, dtype=torch.int32, device=self.device) for x in (rows, lens, cu)]

    def step(self) -> list[int]:
        """One step of all sequences that have room; the finished ones, still in the cache until their pages are released."""
        from . import paged_append, paged_attn
        while self.waiting:
            r = self.requests[self.waiting[0]]
            if not self.pool.reserve(self.waiting[0], len(r.prompt) + r.want):
                break
            self.running.append(self.waiting.pop(0))
        if not self.running and self.waiting:
            raise RuntimeError("no room for the next request: finished sequences keep their pages until they are released")
        if not self.running:
            return []
        seqs, reqs = list(self.running), [self.requests[s] for s in self.running]
        new = [min(self.chunk, len(r.tokens) - r.done) for r in reqs]
        where = (self.k_cache, self.v_cache, *self.tables(seqs, new))
        ids = torch.tensor([t for r, n in zip(reqs, new) for t in r.tokens[r.done:r.done + n]], device=self.device)
        paged_append(self.wk[ids], self.wv[ids], *where, **self.scales)
        o = paged_attn(self.wq[ids], *where, **self.scales, max_new=max(new))
        last = torch.tensor([sum(new[:i + 1]) - 1 for i in range(len(new))], device=self.device)
        nxt = (o[last].flatten(1).float() @ self.out.float().T).argmax(-1).tolist()
        finished = []
        for seq, r, n, token in zip(seqs, reqs, new, nxt):
            r.done += n
            if r.done < len(r.tokens):
                continue  # more of the prompt to come
            r.tokens.append(token)
            if len(r.tokens) == len(r.prompt) + r.want:
                finished.append(seq)
                self.running.remove(seq)
        return finished

    def check(self, seq: int) -> float:
        """Relative distance of a finished sequence's last chunk of outputs from the dense kernel's on the tokens read back."""
        from . import fused, paged_attn, paged_read
        r = self.requests[seq]
        k, v = paged_read(self.k_cache, self.v_cache, *self._whole(seq), r.done, dtype=self.dtype, **self.scales)
        q = self.wq[torch.tensor(r.tokens[:r.done], device=self.device)]

        def dense(x):  # (tokens, heads, d) -> (1, query heads, tokens, d) in fp32
            return x.float().repeat_interleave(q.shape[1] // x.shape[1], 1).transpose(0, 1).unsqueeze(0).contiguous()

        want = fused(dense(q), dense(k), dense(v), True)[0].transpose(0, 1)
        got = paged_attn(q, self.k_cache, self.v_cache, *self._whole(seq), **self.scales)
        return ((got.float() - want).norm() / want.norm()).item()

    def _whole(self, seq: int):
        r = self.requests[seq]
        rows = torch.tensor([self.pool.of[seq]], dtype=torch.int32, device=self.device)
        return rows, torch.tensor([r.done], dtype=torch.int32, device=self.device), torch.tensor([0, r.done], dtype=torch.int32, device=self.device)


def run(requests: int = 12, seed: int = 0, **kw) -> tuple[Server, float, int]:
    """Serve random requests to their end; (server, the largest check, steps)."""
    import random
    rng = random.Random(seed)
    server = Server(seed=seed, **kw)
    for _ in range(requests):
        server.submit([rng.randrange(1000) for _ in range(rng.randint(1, 900))], rng.randint(1, 40))
    worst, steps, left = 0.0, 0, requests
    while left:
        finished = server.step()
        steps += 1
        for seq in finished:
            worst = max(worst, server.check(seq))
            server.pool.release(seq)
            left -= 1
    return server, worst, steps


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=12)
    ap.add_argument("--pages", type=int, default=512)
    ap.add_argument("--page", type=int, default=16)
    ap.add_argument("--chunk", type=int, default=256)
    ap.add_argument("--int8", action="store_true")
    ap.add_argument("--dtype", choices=["fp16", "bf16"], default="bf16")
    a = ap.parse_args(argv)
    from . import device_status
    try:
        server, worst, steps = run(a.requests, pages=a.pages, page=a.page, chunk=a.chunk, int8=a.int8,
                                   dtype={"fp16": torch.float16, "bf16": torch.bfloat16}[a.dtype])
    except ValueError as e:
        ap.error(str(e))
    tokens = sum(len(r.tokens) for r in server.requests.values())
    print(f"served {a.requests} requests, {tokens} tokens in {steps} steps; largest distance from the dense kernel {worst:.2e}, "
          f"{len(server.pool.free)} of {a.pages} pages free, device status {device_status()}")
    return 0 if worst < 1e-2 else 1


if __name__ == "__main__":
    sys.exit(main())
