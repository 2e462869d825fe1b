"""Plain 64-bit implementations of the paged operators and of sampling, for the tests."""
import numpy as np
import torch

TYPES = {"f32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def half_step(name):
    """What rounding to a type is off by at most, relative to the value."""
    return torch.finfo(TYPES[name]).eps / 2


class Scene:
    """Sequences with pages of their own in shuffled order, a cache filled with a poison where nothing may be read, and rows."""

    def __init__(self, seed, heads, kv_heads, head_dim, rows, lengths, page_tokens=32, dtype="bf16", layout="head", causal=True, window=0, scale=None, spare_pages=2, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim, self.rows, self.lengths = heads, kv_heads, head_dim, list(rows), list(lengths)
        self.page_tokens, self.dtype, self.layout, self.causal, self.window = page_tokens, dtype, layout, causal, window
        self.scale = scale or head_dim ** -0.5
        held = [-(-n // page_tokens) for n in lengths]
        self.pages = sum(held) + spare_pages
        order = torch.randperm(self.pages, generator=g).numpy().astype(np.int32)
        self.table = np.full((len(rows), max(max(held), 1)), -7, np.int32)
        at = 0
        for s, n in enumerate(held):
            self.table[s, :n] = order[at:at + n]
            at += n
        t = TYPES[dtype]
        shape = (self.pages, kv_heads, page_tokens, head_dim) if layout == "head" else (self.pages, page_tokens, kv_heads, head_dim)
        k, v = torch.full(shape, float("nan"), dtype=t), torch.full(shape, float("nan"), dtype=t)
        self.tokens = []                                  # per sequence: keys and values [length][kv_heads][head_dim] in 64 bits
        for s, n in enumerate(lengths):
            keys, values = (torch.randn((n, kv_heads, head_dim), generator=g).to(t) for _ in range(2))
            self.tokens.append((keys.double(), values.double()))
            for cache, x in ((k, keys), (v, values)):
                view = cache if layout == "head" else cache.transpose(1, 2)
                for i in range(held[s]):
                    part = x[i * page_tokens:(i + 1) * page_tokens]
                    view[self.table[s, i], :, :part.shape[0]] = part.transpose(0, 1)
        self.total = sum(rows)
        self.q = (1.5 * torch.randn((self.total, heads, head_dim), generator=g)).to(t)
        self.k, self.v, self.dq = k.to(device), v.to(device), self.q.to(device)

    def paged(self, engine, cls, **more):
        return cls(engine, self.heads, self.kv_heads, self.head_dim, self.pages, page_tokens=self.page_tokens, dtype=self.dtype, layout=self.layout, causal=self.causal,
                   window=self.window, scale=self.scale, max_sequences=len(self.rows), max_rows=self.total, max_context=max(max(self.lengths), 1), **more)

    def expected(self):
        """(attention in 64 bits, the bound on what 16-bit probabilities and 32-bit sums may move it by), [rows][heads][head_dim].

        With p_j the exact weights, a relative error e_j of each moves the quotient sum p v / sum p by at most 2 max|e| sum p|v| / sum p. e has three parts: the probability's
        rounding (half a step, in the numerator only, so once), the error of a score (a dot product of head_dim fp32 products, error
        <= head_dim 2^-24 sum|q k| scale whatever the order of its sum; its exponent adds as much), and the exponential's and the sums' (2^-18 allowed)."""
        out, bound = torch.zeros((self.total, self.heads, self.head_dim), dtype=torch.float64), torch.zeros((self.total, self.heads, self.head_dim), dtype=torch.float64)
        at = 0
        group = self.heads // self.kv_heads
        for (keys, values), n, length in zip(self.tokens, self.rows, self.lengths):
            for i in range(n):
                position = length - n + i
                first = max(0, position + 1 - self.window) if self.window else 0
                last = position + 1 if self.causal else length
                for h in range(self.heads):
                    q = self.q[at + i, h].double()
                    k, v = keys[first:last, h // group], values[first:last, h // group]
                    s = (k @ q) * self.scale
                    wide = ((k.abs() @ q.abs()) * self.scale).max().item()
                    p = torch.exp(s - s.max())
                    p = p / p.sum()
                    out[at + i, h] = p @ v
                    e = half_step(self.dtype) + 2 * (self.head_dim * 2.0 ** -24 * wide + 2.0 ** -18)
                    bound[at + i, h] = e * (p @ v.abs())
            at += n
        return out, bound


def check_attention(scene, got, out_dtype):
    want, bound = scene.expected()
    if out_dtype != "f32":
        bound = bound + half_step(out_dtype) * (want.abs() + bound) + 2.0 ** -25      # and the output's rounding (a subnormal fp16's step is absolute)
    got = got.double().cpu()
    worst = ((got - want).abs() / bound).max().item()
    assert worst <= 1.0, f"{worst:.3f} of the bound"
    return worst


def sample(x, temperature, top_k, top_p, min_p, uniform):
    """One row of logits (numpy float32) -> the token, from the definition in 64 bits."""
    x = x.astype(np.float64)
    order = np.argsort(np.where(np.isnan(x), np.inf, -x), kind="stable")
    order = order[~np.isnan(x[order]) & (x[order] > -np.inf)]
    if len(order) == 0:
        return 0
    if not temperature > 0:
        return int(order[0])
    if top_k > 0:
        order = order[:top_k]
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / np.float64(temperature)))
    if top_p < 1:
        c = np.cumsum(w)
        n = int(np.searchsorted(c, np.float64(top_p) * c[-1], side="left")) + 1
        order, w = order[:n], w[:n]
    stays = w >= min(np.float64(min_p), 1.0)
    order, w = order[stays], w[stays]
    c = np.cumsum(w)
    return int(order[min(int(np.searchsorted(c, np.float64(uniform) * c[-1], side="left")), len(order) - 1)])
