"""The operators of a pass over the caller's own tensors that lie between its GEMMs and the next token, as a serving program
calls them: new keys and values into a paged cache with the rotation applied on the way, attention of the new rows over that
cache, and sampling from the logits.

Where `own` is false, `run` computes each operator from elementary torch operations; where it is true it makes the calls of
splosh_b200 (PagedAttention.append and .attend, Engine.pass_sample). The cache, its page table and the batch that says which
sequences have which rows are what a program has in hand before it runs its layers, so `prepare` makes them.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6                     # the norms' epsilon (the engine's geometry has the same)
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _paged(name, op, heads, kv_heads, head_dim, rows, lengths, page, dtype="bf16", layout="head", rotary=0, theta=1e7, norm=False, window=0, causal=True):
    """`rows` and `lengths` are texts of comma-separated numbers: a sequence's new tokens, and its tokens with them."""
    return {"name": name, "op": op, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "rows": _text(rows), "lengths": _text(lengths), "page": page,
            "dtype": dtype, "layout": layout, "rotary": rotary, "theta": theta, "norm": norm, "window": window, "causal": causal}


def _sample(name, rows, vocab, limit, settings, masked=0.0):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "limit": limit, "settings": settings, "masked": masked}


def _text(numbers):
    return ",".join(str(int(n)) for n in numbers)


def _numbers(text):
    return [int(n) for n in text.split(",")]


def _ragged(count, around):
    """Lengths around a mean, as sessions of a server have them: none a multiple of anything."""
    return [max(1, int(around * (0.9 + 0.2 * ((n * 0.618034) % 1.0))) + n) for n in range(count)]


def listed():
    return [
        # A decode step of eight short sessions on the tiny shape: one new token each. Launches and latency.
        _paged("append_decode_8", "append", 8, 2, 128, [1] * 8, _ragged(8, 1000), 16, rotary=32),
        # Eight verify blocks of eight rows on the 27B shape, heads normalised on the way.
        _paged("append_verify_64", "append", 24, 4, 256, [8] * 8, _ragged(8, 6000), 256, dtype="fp16", rotary=64, norm=True),
        # A prompt's chunk of 2,048 rows, a cache whose tokens hold all heads side by side.
        _paged("append_chunk_2048", "append", 24, 4, 256, [2048], [26624], 64, layout="token", rotary=64, norm=True),
        # The smallest attention: one session of the tiny shape, one token.
        _paged("attend_decode_1", "attend", 8, 2, 128, [1], [1024], 16),
        # Continuous batching: twelve sessions of chat length, a token each.
        _paged("attend_decode_12", "attend", 24, 4, 256, [1] * 12, _ragged(12, 3000), 256),
        # Verify blocks of eight rows over long contexts.
        _paged("attend_verify_8x8", "attend", 24, 4, 256, [8] * 8, _ragged(8, 39000), 256),
        # A block-diffusion draft: blocks of sixteen rows that see each other and a window of 2,048 tokens.
        _paged("attend_draft_8x16", "attend", 32, 8, 128, [16] * 8, _ragged(8, 9000), 64, dtype="fp16", layout="token", window=2048, causal=False),
        # A new session's question of 301 tokens beside six decoding sessions.
        _paged("attend_prompt_301", "attend", 24, 4, 256, [1] * 6 + [301], _ragged(6, 2500) + [301], 128, layout="token"),
        # A long prompt's chunk: 2,048 rows over 24K tokens already fed.
        _paged("attend_chunk_2048", "attend", 24, 4, 256, [2048], [26624], 256),
        # One session's next token on the tiny shape's vocabulary.
        _sample("sample_1", 1, 32000, 32000, "0.8:20:0.95:0"),
        # Twelve sessions on the 27B vocabulary (the last ids are not tokens), nucleus sampling over the whole of it.
        _sample("sample_12", 12, 248320, 248077, "1.0:0:0.95:0,0.7:0:0.9:0.02"),
        # Verify rows of many sessions with settings of their own, a grammar's mask on a part of the vocabulary.
        _sample("sample_64", 64, 248320, 248077, "1.0:0:1:0,0.7:50:0.9:0,1.2:0:1:0.05,0:0:1:0,0.9:1000:0.98:0.001,1.0:0:0.999:0", masked=0.3),
    ]


def draw(rng):
    most = max(map(_floor, listed()))
    while True:
        case = _drawn(rng)
        if _floor(case) <= most:
            del case["name"]
            return case


def _floor(case):
    """Roughly the seconds that a case cannot do without."""
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.4e15)


def _drawn(rng):
    def log(low, high):
        return int(round(low * (high / low) ** rng.random()))
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "sample", "sample"])
    if kind == "sample":
        vocab = log(1000, 248320)
        settings = ",".join("%g:%d:%g:%g" % (rng.choice([0.0, 0.6, 0.8, 1.0, 1.0, 1.5]), rng.choice([0, 0, log(1, 2000)]), rng.choice([1.0, 0.9, 0.95, 0.999]),
                                             rng.choice([0.0, 0.0, 0.02, 0.1])) for _ in range(rng.randint(1, 6)))
        return _sample("", log(1, 64), vocab, vocab - rng.choice([0, 0, rng.randint(1, 300)]), settings, masked=rng.choice([0.0, 0.0, 0.5]))
    kv_heads, group, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 6, 8]), rng.choice([64, 128, 128, 256])
    form = rng.choice(["decode", "verify", "prompt", "chunk", "mixed"])
    if form == "decode":
        rows = [1] * log(1, 32)
        lengths = [log(1, 20000) for _ in rows]
    elif form == "verify":
        rows = [rng.randint(2, 16) for _ in range(log(1, 8))]
        lengths = [n + log(1, 40000) for n in rows]
    elif form == "prompt":
        rows = [log(17, 1500) for _ in range(rng.randint(1, 3))]
        lengths = list(rows)
    elif form == "chunk":
        rows = [log(100, 2048)]
        lengths = [rows[0] + log(100, 16000)]
    else:
        rows = [1] * rng.randint(1, 12) + [log(20, 600)]
        lengths = [n + log(1, 6000) for n in rows]
    if kind == "append":
        lengths = [max(n, length // 8) for n, length in zip(rows, lengths)]      # new tokens alone are touched: a smaller cache says as much
    window = 0 if rng.random() < 0.75 else log(64, 4096)
    return _paged("", kind, kv_heads * group, kv_heads, head_dim, rows, lengths, rng.choice([16, 32, 64, 128, 256]), dtype=rng.choice(["bf16", "fp16"]),
                         layout=rng.choice(["head", "token"]), rotary=rng.choice([head_dim // 4, head_dim // 2, head_dim]), theta=rng.choice([1e4, 1e6, 1e7]),
                         norm=rng.random() < 0.5, window=window, causal=rng.random() < 0.8)


def _visible(case):
    """Tokens that the rows see, summed over the rows."""
    total = 0
    for n, length in zip(_numbers(case["rows"]), _numbers(case["lengths"])):
        for position in range(length - n, length):
            first = max(0, position + 1 - case["window"]) if case["window"] else 0
            total += (position + 1 if case["causal"] else length) - first
    return total


def work(case):
    if case["op"] == "sample":
        # A row's logits in, its token out; a comparison and an exponential a value.
        return {"bytes": case["rows"] * (case["limit"] * 4.0 + 24), "flops": 2.0 * case["rows"] * case["limit"]}
    rows, heads, kv_heads, d = sum(_numbers(case["rows"])), case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        # fp32 rows in, 16-bit queries, keys and values out.
        return {"bytes": rows * (heads + 2 * kv_heads) * d * 6.0, "flops": rows * (heads + kv_heads) * (3.0 * case["rotary"] + (4.0 * d if case["norm"] else 0.0))}
    tokens = 0
    for n, length in zip(_numbers(case["rows"]), _numbers(case["lengths"])):
        first = max(0, length - n + 1 - case["window"]) if case["window"] else 0
        tokens += length - first
    return {"bytes": (tokens * kv_heads * 2.0 + rows * heads * 2.0) * d * 2.0, "flops": 4.0 * heads * d * _visible(case)}


# ---- inputs --------------------------------------------------------------------------------------
class _State:
    pass


_engine = None


def _the_engine():
    global _engine
    if _engine is None:
        import splosh_b200 as S
        _engine = S.Engine(S.tiny_geometry(), S.EngineConfig(max_slots=1, max_rows=64, kv_pages=4, max_context=1024))
    return _engine


def _stream():
    return torch.cuda.current_stream().cuda_stream


def prepare(case, seed):
    s = _State()
    s.case = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "sample":
        return _prepare_sample(s, case, g)
    rows, lengths = _numbers(case["rows"]), _numbers(case["lengths"])
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    t = TYPES[case["dtype"]]
    total = sum(rows)
    held = [-(-length // page) for length in lengths]
    pages = sum(held) + 3                                    # a few pages belong to nobody
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).numpy().astype(np.int32)
    s.table = np.full((len(rows), max(held)), -1, np.int32)
    at = 0
    for n, count in enumerate(held):
        s.table[n, :count] = order[at:at + count]
        at += count
    shape = (pages, kv_heads, page, d) if case["layout"] == "head" else (pages, page, kv_heads, d)
    s.k = torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(t) if case["op"] == "attend" else torch.zeros(shape, device="cuda", dtype=t)
    s.v = torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).to(t) if case["op"] == "attend" else torch.zeros(shape, device="cuda", dtype=t)
    # Each row's sequence and position, and where the cache holds it.
    sequence = np.repeat(np.arange(len(rows)), rows)
    position = np.concatenate([np.arange(length - n, length) for n, length in zip(rows, lengths)])
    s.position = torch.from_numpy(position).cuda()
    s.page_of = torch.from_numpy(s.table[sequence, position // page].astype(np.int64)).cuda()
    s.slot_of = torch.from_numpy(position % page).cuda()
    s.pages_of = [torch.from_numpy(s.table[n, :count].astype(np.int64)).cuda() for n, count in enumerate(held)]
    s.rows, s.lengths = rows, lengths
    if case["op"] == "append":
        s.qkv = torch.randn((total, (heads + 2 * kv_heads) * d), device="cuda", generator=g)
        s.q_norm, s.k_norm = ((1.0 + 0.1 * torch.randn(d, device="cuda", generator=g)).to(torch.bfloat16) for _ in range(2))
        s.q = torch.zeros((total, heads, d), device="cuda", dtype=t)
    else:
        # Queries of models with normalised heads: scores spread over several units, a few tokens far above the rest.
        s.q = (1.5 * torch.randn((total, heads, d), device="cuda", generator=g)).to(t)
        s.out = torch.zeros((total, heads, d), device="cuda", dtype=t)
    if own:
        import splosh_b200 as S
        engine = _the_engine()
        s.paged = S.PagedAttention(engine, heads, kv_heads, d, pages, page_tokens=page, dtype=case["dtype"], layout=case["layout"], rotary_dim=case["rotary"],
                                   rope_theta=case["theta"], causal=case["causal"], window=case["window"], max_sequences=len(rows), max_rows=total,
                                   max_context=max(lengths))
        s.paged.batch(rows, lengths, s.table, stream=_stream())
        if case["op"] == "append" and case["norm"]:
            s.norms = [engine.tensor_vector(w.view(torch.int16).cpu().numpy().view(np.uint16)) for w in (s.q_norm, s.k_norm)]
    torch.cuda.synchronize()
    return s


def _prepare_sample(s, case, g):
    rows, vocab, limit = case["rows"], case["vocab"], case["limit"]
    # A language model's logits: a broad bell, and some dozens of likely tokens above it.
    x = 2.0 * torch.randn((rows, vocab), device="cuda", generator=g)
    likely = torch.randint(0, limit, (rows, 48), device="cuda", generator=g)
    x.scatter_add_(1, likely, 6.0 + 4.0 * torch.rand((rows, 48), device="cuda", generator=g))
    if case["masked"]:
        x[torch.rand((rows, vocab), device="cuda", generator=g) < case["masked"]] = -math.inf
    s.logits = x
    settings = [[float(v) for v in one.split(":")] for one in case["settings"].split(",")]
    per_row = np.array([settings[r % len(settings)] for r in range(rows)])
    s.temperature, s.top_p, s.min_p = (torch.tensor(per_row[:, n], dtype=torch.float32, device="cuda") for n in (0, 2, 3))
    s.top_k = torch.tensor(per_row[:, 1], dtype=torch.int32, device="cuda")
    s.uniform = torch.rand(rows, device="cuda", generator=g)
    s.ids = torch.zeros(rows, dtype=torch.int32, device="cuda")
    if own:
        s.engine = _the_engine()
    torch.cuda.synchronize()
    return s


# ---- the operators -------------------------------------------------------------------------------
def run(state):
    op = state.case["op"]
    if op == "append":
        return _append(state)
    if op == "attend":
        return _attend(state)
    return _sample_rows(state)


def _append(s):
    c = s.case
    heads, kv_heads, d = c["heads"], c["kv_heads"], c["head_dim"]
    if own:
        ld = (heads + 2 * kv_heads) * d
        base = s.qkv.data_ptr()
        q_norm, k_norm = s.norms if c["norm"] else (None, None)
        s.paged.append(base, base + 4 * heads * d, base + 4 * (heads + kv_heads) * d, s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), ld=ld,
                       q_norm=q_norm, k_norm=k_norm, stream=_stream())
        return {"q": s.q, "k": s.k, "v": s.v}
    q, k, v = s.qkv.split([heads * d, kv_heads * d, kv_heads * d], dim=1)
    half = c["rotary"] // 2
    frequency = c["theta"] ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = s.position.double()[:, None] * frequency
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(x, count, weight):
        x = x.reshape(-1, count, d)
        if c["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    t = TYPES[c["dtype"]]
    s.q.copy_(turned(q, heads, s.q_norm).to(t))
    for cache, x in ((s.k, turned(k, kv_heads, s.k_norm)), (s.v, v.reshape(-1, kv_heads, d))):
        if c["layout"] == "head":
            cache[s.page_of, :, s.slot_of] = x.to(t)
        else:
            cache[s.page_of, s.slot_of] = x.to(t)
    return {"q": s.q, "k": s.k, "v": s.v}


def _attend(s):
    c = s.case
    if own:
        s.paged.attend(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.out.data_ptr(), stream=_stream())
        return s.out
    heads, kv_heads, d = c["heads"], c["kv_heads"], c["head_dim"]
    group, at = heads // kv_heads, 0
    for n, (count, length) in enumerate(zip(s.rows, s.lengths)):
        q = s.q[at:at + count].float().reshape(count, kv_heads, group, d)
        token = torch.arange(length, device="cuda")
        position = torch.arange(length - count, length, device="cuda")[:, None]
        seen = token <= position if c["causal"] else token < length + 0 * position
        if c["window"]:
            seen = seen & (token > position - c["window"])
        for h in range(kv_heads):
            k, v = ((x[s.pages_of[n], h] if c["layout"] == "head" else x[s.pages_of[n], :, h]).reshape(-1, d)[:length].float() for x in (s.k, s.v))
            score = (q[:, h] @ k.T) * d ** -0.5
            score.masked_fill_(~seen[:, None], -math.inf)
            score = torch.exp(score - score.max(-1, keepdim=True).values)
            out = (score @ v) / score.sum(-1, keepdim=True)
            s.out[at:at + count, h * group:(h + 1) * group] = out.to(s.out.dtype)
        at += count
    return s.out


def _sample_rows(s):
    c = s.case
    if own:
        s.engine.pass_sample(s.logits.data_ptr(), c["rows"], c["vocab"], c["limit"], s.ids.data_ptr(), s.uniform.data_ptr(), temperature=s.temperature.data_ptr(),
                             top_k=s.top_k.data_ptr(), top_p=s.top_p.data_ptr(), min_p=s.min_p.data_ptr(), stream=_stream())
        return s.ids
    x = s.logits[:, :c["limit"]]
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    greedy = ~(s.temperature > 0)
    scaled = (x.double() - x[:, :1].double()) / torch.where(greedy, 1.0, s.temperature.double())[:, None]
    weight = torch.exp(scaled)                               # a masked value's is zero
    place = torch.arange(c["limit"], device="cuda")
    top_k = torch.where(s.top_k > 0, s.top_k, c["limit"])[:, None]
    weight = torch.where(place < top_k, weight, 0.0)
    total = weight.cumsum(1)
    kept = (total < s.top_p.double()[:, None] * total[:, -1:]).sum(1, keepdim=True)      # the place where the prefix is complete
    weight = torch.where((place <= kept) | (s.top_p >= 1)[:, None], weight, 0.0)
    weight = torch.where(weight >= s.min_p.double()[:, None], weight, 0.0)
    total = weight.cumsum(1)
    pick = (total < s.uniform.double()[:, None] * total[:, -1:]).sum(1)
    pick = torch.where(greedy, 0, torch.minimum(pick, (weight > 0).sum(1) - 1))
    s.ids.copy_(order.gather(1, pick[:, None])[:, 0])
    return s.ids


# ---- the definitions in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    return _exact_sample(case, s)


def _exact_append(case, s):
    heads, kv_heads, d, rot = case["heads"], case["kv_heads"], case["head_dim"], case["rotary"]
    x = s.qkv.cpu().numpy().astype(np.float64).reshape(-1, heads + 2 * kv_heads, d)
    position = s.position.cpu().numpy().astype(np.float64)
    y = x.copy()
    if case["norm"]:
        scale = 1.0 / np.sqrt(np.square(x).mean(axis=2, keepdims=True) + EPS)
        weights = np.ones((heads + 2 * kv_heads, d))
        weights[:heads] = s.q_norm.double().cpu().numpy()
        weights[heads:heads + kv_heads] = s.k_norm.double().cpu().numpy()
        scale[:, heads + kv_heads:] = 1.0
        y = x * scale * weights
    z = y.copy()
    for i in range(rot // 2):
        turn = position * case["theta"] ** (-2.0 * i / rot)
        pair = (y[:, :heads + kv_heads, i] + 1j * y[:, :heads + kv_heads, i + rot // 2]) * np.exp(1j * turn)[:, None]
        z[:, :heads + kv_heads, i], z[:, :heads + kv_heads, i + rot // 2] = pair.real, pair.imag
    out = {"q": z[:, :heads]}
    page, slot = s.page_of.cpu().numpy(), s.slot_of.cpu().numpy()
    for name, cache, first in (("k", s.k, heads), ("v", s.v, heads + kv_heads)):
        full = cache.double().cpu().numpy()
        view = full if case["layout"] == "head" else full.transpose(0, 2, 1, 3)
        for r in range(len(page)):
            view[page[r], :, slot[r]] = z[r, first:first + kv_heads]
        out[name] = full
    return out


def _exact_attend(case, s):
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    group = heads // kv_heads
    out = torch.zeros(tuple(s.q.shape), dtype=torch.float64)
    at = 0
    for n, (count, length) in enumerate(zip(s.rows, s.lengths)):
        for h in range(kv_heads):
            if case["layout"] == "head":
                k, v = s.k[s.pages_of[n]][:, h], s.v[s.pages_of[n]][:, h]
            else:
                k, v = s.k[s.pages_of[n]][:, :, h], s.v[s.pages_of[n]][:, :, h]
            k, v = k.flatten(0, 1).double(), v.flatten(0, 1).double()
            for r0 in range(0, count, 256):
                r1 = min(count, r0 + 256)
                q = s.q[at + r0:at + r1, h * group:(h + 1) * group].double()
                logit = torch.einsum("rgd,td->rgt", q, k) / math.sqrt(d)
                for r in range(r0, r1):
                    p = length - count + r
                    last = p + 1 if case["causal"] else length
                    first = max(0, p + 1 - case["window"]) if case["window"] else 0
                    logit[r - r0, :, :first] = -math.inf
                    logit[r - r0, :, last:] = -math.inf
                out[at + r0:at + r1, h * group:(h + 1) * group] = torch.einsum("rgt,td->rgd", torch.softmax(logit, -1), v).cpu()
        at += count
    return out


def _exact_sample(case, s):
    ids = np.zeros(case["rows"], np.int32)
    for r in range(case["rows"]):
        x = s.logits[r, :case["limit"]].double().cpu().numpy()
        t, k, p, m, u = (float(a[r]) for a in (s.temperature, s.top_k, s.top_p, s.min_p, s.uniform))
        order = np.argsort(-x, kind="stable")
        order = order[:int(np.isfinite(x).sum())]
        if t <= 0:
            ids[r] = order[0]
            continue
        if k > 0:
            order = order[:int(k)]
        w = np.exp((x[order] - x[order[0]]) / t)
        if p < 1:
            c = np.cumsum(w)
            n = int(np.searchsorted(c, p * c[-1], side="left")) + 1
            order, w = order[:n], w[:n]
        keep = w >= m
        order, w = order[keep], w[keep]
        c = np.cumsum(w)
        ids[r] = order[min(int(np.searchsorted(c, u * c[-1], side="left")), len(order) - 1)]
    return torch.from_numpy(ids)
