"""Ragged sequences in a paged cache for the tests, and the operators' definitions in 64 bits (plain loops over sequences).

Bounds on the attention's outputs, from the kernels' arithmetic. Let u be the output type's unit roundoff (2^-8 for bf16's 8
significant bits, 2^-11 for fp16's 11) and A = sum_j p_j |v_j| / sum_j p_j the size of the terms that an output is the sum of. An output is off by

  u |o|            its own rounding,
  r A              the rounding of each p_j to 16 bits: at most r = 2^-8 (bf16) or 2^-11 (fp16, and all 8-bit caches) of p_j,
                   twice that to cover the sum of p_j, which takes them unrounded,
  2^-12 A          the scores: fp32 sums of at most 128 products of size up to about 8, and exp2 to 2^-13.7,

and the 2-norm of the error over all outputs is at most 1.5 times that of a correctly rounded result (1.66e-3 and 2.08e-4 of
the result for uniformly spread mantissas): the output's rounding and one more of the same size are sqrt(2) times.
"""
import random

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
REL_L2 = {torch.bfloat16: 1.5 * 1.66e-3, torch.float16: 1.5 * 2.08e-4}


def quantise64(x):
    """Whole numbers and fp32 scales of x (..., d), by the definition in 64 bits."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True).clamp_min(127 * 2.0 ** -100)
    return torch.round(127 * x / top).to(torch.int8), (top / 127).squeeze(-1).float()


class Case:
    """`new`, `kv`: new and all tokens of each sequence. The pool's unused places hold `stale` (NaN by default)."""

    def __init__(self, new, kv, heads, group, d, page, dtype, int8, seed=0, layout="plain", stale=float("nan"), scale=1.0):
        dev = "cuda"
        g = torch.Generator(device=dev).manual_seed(seed)
        self.new, self.kv, self.heads, self.group, self.d, self.page, self.dtype, self.int8 = new, kv, heads, group, d, page, dtype, int8
        need = [-(-max(t, 0) // page) for t in kv]
        pages = sum(need) + 2
        order = list(range(pages))
        random.Random(seed).shuffle(order)
        width = max(need) + 2
        table = torch.full((len(kv), width), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        self.table = table.to(dev)
        self.lens = torch.tensor(kv, dtype=torch.int32, device=dev)
        self.cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=dev)
        self.total = sum(new)
        ctype = torch.int8 if int8 else dtype

        def pool(fill):
            if layout == "interleaved":   # keys and values of a page beside each other
                base = torch.full((pages, 2, heads, page, d), fill, device=dev, dtype=ctype)
                return base[:, 0], base[:, 1]
            if layout == "token":         # (pages, tokens, heads, d)
                return tuple(torch.full((pages, page, heads, d), fill, device=dev, dtype=ctype).transpose(1, 2) for _ in "kv")
            return tuple(torch.full((pages, heads, page, d), fill, device=dev, dtype=ctype) for _ in "kv")

        self.k_cache, self.v_cache = pool(-77 if int8 else stale)
        self.k_scale = self.v_scale = None
        if int8:
            self.k_scale, self.v_scale = (torch.full((pages, heads, page), stale, device=dev) for _ in "kv")
        self.keys, self.values = [], []   # (tokens, heads, d) in 64 bits, as the cache stands for them
        self.written = []
        for b, t in enumerate(kv):
            t = max(t, 0)
            for cache, sc, held in ((self.k_cache, self.k_scale, self.keys), (self.v_cache, self.v_scale, self.values)):
                x = (torch.randn(t, heads, d, device=dev, generator=g) * scale).to(dtype)
                self.written.append(x)
                ids, place = self.places(b, t)
                if int8:
                    q, s = quantise64(x)
                    cache[ids, :, place] = q
                    sc[ids, :, place] = s
                    held.append(q.double() * s.double()[..., None])
                else:
                    cache[ids, :, place] = x
                    held.append(x.double())
        wide = torch.randn(self.total, heads * group + 2 * heads, d, device=dev, generator=g).to(dtype)
        self.q = wide[:, :heads * group] if layout != "plain" else wide[:, :heads * group].contiguous()

    def places(self, b, t):
        j = torch.arange(t, device=self.table.device)
        return self.table[b][(j // self.page)].long(), j % self.page

    def where(self):
        return self.k_cache, self.v_cache, self.table, self.lens, self.cu

    def scales(self):
        return {"k_scale": self.k_scale, "v_scale": self.v_scale}

    def attention64(self, causal, scale=None):
        """(o, A): outputs in 64 bits and the size of their terms."""
        scale = self.d ** -0.5 if scale is None else scale
        outs, sizes, at = [], [], 0
        for b, (n, t) in enumerate(zip(self.new, self.kv)):
            t = max(t, 0)
            k, v = (x.repeat_interleave(self.group, 1) for x in (self.keys[b], self.values[b]))
            q = self.q[at:at + n].double()
            at += n
            s = torch.einsum("ihd,jhd->hij", q, k) * scale
            if causal:
                i = torch.arange(n, device=s.device)[:, None]
                s = s.masked_fill(torch.arange(t, device=s.device) > t - n + i, -torch.inf)
            p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) if t else s
            outs.append(torch.einsum("hij,jhd->ihd", p, v))
            sizes.append(torch.einsum("hij,jhd->ihd", p, v.abs()))
        return torch.cat(outs), torch.cat(sizes)


def assert_attention(out, ref, size, dtype, int8=False):
    u = U[dtype]
    r = 2.0 ** -11 if int8 else u
    err = (out.double() - ref).abs()
    bound = u * ref.abs() + (2 * r + 2.0 ** -12) * size + 2.0 ** -24
    assert torch.isfinite(out).all(), "non-finite output"
    worst = (err / bound).max().item()
    assert worst <= 1.0, f"error {worst:.2f} times its bound"
    norm = ref.norm().item()
    rel = (out.double() - ref).norm().item() / norm if norm else 0.0
    assert rel <= REL_L2[dtype], f"relative L2 {rel:.2e} > {REL_L2[dtype]:.2e}"
