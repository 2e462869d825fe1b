"""Plain 64-bit implementations for the tests: attention over a paged cache of e4m3 codes, or of sequences that share their first pages, and the test of drafted tokens."""
import numpy as np
import torch

from paged_reference import TYPES, half_step

E4M3, LARGEST, SCALE_MIN = torch.float8_e4m3fn, 448.0, 2.0 ** -100


def quantised(x):
    """Codes (float8) and scales of [..., channels] in fp32: scale = max / 448 (at least 2^-100)."""
    scale = (x.abs().amax(-1, keepdim=True) / LARGEST).clamp(min=SCALE_MIN)
    return (x / scale).to(E4M3), scale[..., 0]


class Scene:
    """Sequences with pages in shuffled order (the members of a group begin with the same ones), a poison where nothing may be read, and rows. dtype "bf16", "fp16" or "e4m3"."""

    def __init__(self, seed, heads, kv_heads, head_dim, rows, lengths, page_tokens=32, dtype="e4m3", layout="head", causal=True, window=0, groups=(), spare_pages=2, spread=0.5, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim, self.rows, self.lengths, self.groups = heads, kv_heads, head_dim, list(rows), list(lengths), list(groups)
        self.page_tokens, self.dtype, self.layout, self.causal, self.window = page_tokens, dtype, layout, causal, window
        self.scale = head_dim ** -0.5
        self.q_type = "bf16" if dtype == "e4m3" else dtype
        held = [-(-n // page_tokens) for n in lengths]
        leader, behind, at = list(range(len(rows))), [0] * len(rows), 0
        for n, shared in groups:
            leader[at:at + n], behind[at + 1:at + n], at = [at] * n, [shared // page_tokens] * (n - 1), at + n
        self.pages = sum(held) - sum(behind) + spare_pages
        order = torch.randperm(self.pages, generator=g).numpy().astype(np.int32)
        self.table = np.full((len(rows), max(max(held), 1)), -7, np.int32)
        t = E4M3 if dtype == "e4m3" else TYPES[dtype]
        shape = (self.pages, kv_heads, page_tokens, head_dim)
        k, v = (torch.full(shape, float("nan")).to(t) for _ in range(2))
        ks, vs = (torch.full(shape[:3], float("nan")) for _ in range(2))
        self.tokens, at = [], 0                           # per sequence: keys, values (as stored, 64 bits) and their scales
        for s, n in enumerate(lengths):
            lead, own = leader[s], behind[s]
            self.table[s, :own] = self.table[lead, :own]
            self.table[s, own:held[s]] = order[at:at + held[s] - own]
            at += held[s] - own
            pair = []
            for i, (cache, scales) in enumerate(((k, ks), (v, vs))):
                x = torch.randn((n, kv_heads, head_dim), generator=g) * torch.exp(spread * torch.randn((n, kv_heads, 1), generator=g))
                codes, scale = quantised(x) if dtype == "e4m3" else (x.to(t), torch.ones(n, kv_heads))
                if own:
                    codes, scale = codes.clone(), scale.clone()
                    codes[:own * page_tokens], scale[:own * page_tokens] = self.tokens[lead][2 * i][:own * page_tokens].to(t), self.tokens[lead][2 * i + 1][:own * page_tokens].float()
                for p in range(own, held[s]):
                    part = slice(p * page_tokens, min(n, (p + 1) * page_tokens))
                    count = part.stop - part.start
                    cache[self.table[s, p], :, :count], scales[self.table[s, p], :, :count] = codes[part].transpose(0, 1), scale[part].transpose(0, 1)
                pair += [codes.double(), scale.double()]
            self.tokens.append(pair)
        self.total = sum(rows)
        self.q = (1.5 * torch.randn((self.total, heads, head_dim), generator=g)).to(TYPES[self.q_type])
        if layout == "token":
            k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
        self.k, self.v, self.ks, self.vs, self.dq = k.to(device), v.to(device), ks.to(device), vs.to(device), self.q.to(device)

    def paged(self, engine, cls, **more):
        args = dict(page_tokens=self.page_tokens, dtype=self.dtype, layout=self.layout, causal=self.causal, window=self.window, scale=self.scale, max_sequences=len(self.rows), max_rows=self.total,
                    max_context=max(max(self.lengths), 1))
        return cls(engine, self.heads, self.kv_heads, self.head_dim, self.pages, **{**args, **more})

    def scales(self):
        return {"k_scale": self.ks.data_ptr(), "v_scale": self.vs.data_ptr()} if self.dtype == "e4m3" else {}

    def expected(self):
        """(attention in 64 bits, the bound on what its arithmetic may move it by), [rows][heads][head_dim].

        With w_j = p_j s_j the exact products of probability and value scale, o = sum w_j V_j / sum p_j; relative errors e_j of the p_j move it by at most 2 max|e| sum w|V|, and one of a w_j alone by e_j w|V|.
        Of 16-bit caches: the rounding of p (half a step), the score's error (head_dim products and sums in fp32, each half a step of what has been summed: head_dim 2^-24 sum|q k| scale; its exponent adds as much),
        and 2^-18 for exponentials and sums. Of e4m3: w is rounded to fp16 (2^-11), and below 2^-21 of the row's largest to that much 2^-11 of the largest; a bf16 query is the sum of two e4m3 of its row's largest times
        2^-7 at least: exact but for the smallest channels, which are off by at most 2^-10 of that 2^-7: 2^-17 of the largest."""
        out, bound = (torch.zeros((self.total, self.heads, self.head_dim), dtype=torch.float64) for _ in range(2))
        group, e4m3, at = self.heads // self.kv_heads, self.dtype == "e4m3", 0
        for (keys, k_scale, values, v_scale), n, length in zip(self.tokens, self.rows, self.lengths):
            position = torch.arange(length - n, length)[:, None]
            token = torch.arange(length)[None, :]
            hidden = token > position if self.causal else torch.zeros((n, length), dtype=torch.bool)
            if self.window:
                hidden = hidden | (token <= position - self.window)
            for h in range(self.heads if n else 0):
                kv = h // group
                q, k, v = self.q[at:at + n, h].double(), keys[:, kv] * k_scale[:, kv, None], values[:, kv] * v_scale[:, kv, None]
                s = (q @ k.T) * self.scale
                wide = (q.abs() @ k.abs().T) * self.scale
                s[hidden], wide[hidden] = -np.inf, 0.0
                p = torch.softmax(s, -1)
                e = 2 * (self.head_dim * 2.0 ** -24 * wide.amax(-1) + 2.0 ** -18)
                small = 0.0
                if e4m3:
                    e += 2 * 2.0 ** -17 * (q.abs().amax(-1, keepdim=True) * k.abs().sum(-1)[None, :] * self.scale).masked_fill(hidden, 0.0).amax(-1) + 2.0 ** -11
                    w = p * v_scale[:, kv]
                    small = 2.0 ** -32 * w.amax(-1, keepdim=True) * ((~hidden).double() @ values[:, kv].abs())
                else:
                    e += half_step(self.dtype)
                out[at:at + n, h] = p @ v
                bound[at:at + n, h] = e[:, None] * (p @ v.abs()) + small
            at += n
        return out, bound


def check(scene, got, out_dtype):
    want, bound = scene.expected()
    if out_dtype != "f32":
        bound = bound + half_step(out_dtype) * (want.abs() + bound) + 2.0 ** -25
    else:
        bound = bound + 2.0 ** -24 * want.abs()
    worst = ((got.double().cpu() - want).abs() / bound).max().item()
    assert worst <= 1.0, f"{worst:.3f} of the bound"
    return worst


def verify(x, temperature, top_k, top_p, min_p, draft, candidates, uniform):
    """One row of logits (numpy float32): -1 where the drafted token stays, else the token in its place, from the definition in 64 bits. `candidates`: (id, probability) pairs, or None where the
    draft was the only choice."""
    x = x.astype(np.float64)
    order = np.argsort(np.where(np.isnan(x), np.inf, -x), kind="stable")
    order = order[~np.isnan(x[order]) & (x[order] > -np.inf)]
    if len(order) == 0:
        return 0
    if not temperature > 0:
        order, w = order[:1], np.ones(1)
    else:
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
    # All in units of the weights: p W = w, and q W. (Over ties these are whole numbers; divided by W first, they would be rounded.)
    total, q = w.sum(), {}
    if draft >= 0:
        for i, one in ([(draft, 1.0)] if candidates is None else candidates):
            q.setdefault(int(i), np.float64(one))
        at = np.flatnonzero(order == draft)
        if np.float64(uniform[0]) * q.get(int(draft), 0.0) * total < (w[at[0]] if len(at) else 0.0):
            return -1
    rest = np.array([max(0.0, one - q.get(int(i), 0.0) * total) for i, one in zip(order, w)])
    if not rest.sum() > 0:
        rest = w
    c = np.cumsum(rest)
    return int(order[min(int(np.searchsorted(c, np.float64(uniform[1]) * c[-1], side="left")), int(np.flatnonzero(rest)[-1]))])
