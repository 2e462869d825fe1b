"""More operators of a pass over the caller's own tensors, as a serving program that speculates calls them: new keys and values into a paged cache of
8-bit floating point, attention over that cache, attention of a batch whose sequences begin with the same tokens, and the test of drafted tokens against
the target's probabilities.

Where `own` is false, `run` computes each operator from elementary torch operations; where it is true it makes the calls of splosh_b200
(PagedAttention.append and .attend, Engine.pass_verify). The cache, its page table and the batch that says which sequences have which rows and which of
them share their first pages are what a program has in hand before it runs its layers, so `prepare` makes them.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6                     # the norms' epsilon (the engine's geometry has the same)
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn
LARGEST = 448.0                # of an e4m3 code
SCALE_MIN = 2.0 ** -100        # of a token's scale: a head of zeros has it


def _paged(name, op, heads, kv_heads, head_dim, rows, lengths, page, cache="e4m3", layout="head", rotary=0, theta=1e7, norm=False, window=0, causal=True, groups=""):
    """`rows` and `lengths` are texts of comma-separated numbers: a sequence's new tokens, and its tokens with them. `groups`: comma-separated "sequences:tokens",
    the next so many sequences share the pages of their first so many tokens."""
    return {"name": name, "op": op, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "rows": _text(rows), "lengths": _text(lengths), "page": page,
            "cache": cache, "layout": layout, "rotary": rotary, "theta": theta, "norm": norm, "window": window, "causal": causal, "groups": groups}


def _verify(name, drafts, vocab, limit, settings, candidates, noise=1.0, masked=0.0):
    """`drafts`: a sequence's drafted tokens. `candidates` a drafted token was picked from, with their probabilities (0: it was the drafter's only choice)."""
    return {"name": name, "op": "verify", "drafts": _text(drafts), "vocab": vocab, "limit": limit, "settings": settings, "candidates": candidates, "noise": noise, "masked": masked}


def _text(numbers):
    return ",".join(str(int(n)) for n in numbers)


def _numbers(text):
    return [int(n) for n in text.split(",")]


def _groups(text):
    return [tuple(int(n) for n in one.split(":")) for one in text.split(",")] if text else []


def _ragged(count, around):
    """Lengths around a mean, as sessions of a server have them: none a multiple of anything."""
    return [max(1, int(around * (0.9 + 0.2 * ((n * 0.618034) % 1.0))) + n) for n in range(count)]


def listed():
    return [
        # A decode step of eight short sessions on the tiny shape into an 8-bit cache: one new token each. Launches and latency.
        _paged("append_8bit_decode_8", "append", 8, 2, 128, [1] * 8, _ragged(8, 1000), 16, rotary=32),
        # A prompt's chunk of 2,048 rows on the 27B shape, heads normalised on the way, tokens that hold all heads side by side.
        _paged("append_8bit_chunk_2048", "append", 24, 4, 256, [2048], [26624], 64, layout="token", rotary=64, norm=True),
        # The smallest attention: one session of the tiny shape, one token.
        _paged("attend_8bit_decode_1", "attend", 8, 2, 128, [1], [1024], 16),
        # Continuous batching: twelve sessions of chat length, a token each.
        _paged("attend_8bit_decode_12", "attend", 24, 4, 256, [1] * 12, _ragged(12, 6000), 256),
        # Verify blocks of eight rows over long contexts.
        _paged("attend_8bit_verify_8x8", "attend", 24, 4, 256, [8] * 8, _ragged(8, 39000), 64, layout="token"),
        # A long prompt's chunk: 2,048 rows over 24K tokens already fed.
        _paged("attend_8bit_chunk_2048", "attend", 24, 4, 256, [2048], [26624], 256),
        # Twelve sessions behind one system prompt with its tools, a token each.
        _paged("shared_decode_12", "attend", 24, 4, 256, [1] * 12, [8192 + n for n in _ragged(12, 600)], 256, cache="bf16", groups="12:8192"),
        # Eight continuations of one 21K prompt, verify blocks of eight rows.
        _paged("shared_verify_8x8", "attend", 24, 4, 256, [8] * 8, [20992 + n for n in _ragged(8, 1500)], 256, cache="bf16", groups="8:20992"),
        # A busy server on the drafter's shape: two system prompts, a few sessions without one.
        _paged("shared_decode_48", "attend", 32, 8, 128, [1] * 48, [4096 + n for n in _ragged(24, 700)] + [2048 + n for n in _ragged(16, 900)] + _ragged(8, 1200), 64, cache="fp16",
               layout="token", groups="24:4096,16:2048"),
        # One session's verify block of four drafted tokens on the tiny shape's vocabulary.
        _verify("verify_1x4", [4], 32000, 32000, "0.8:20:0.95:0", 16),
        # Eight sessions, seven drafted tokens each from the drafter's sixteen candidates, nucleus sampling over the whole vocabulary (the last ids are not tokens).
        _verify("verify_8x7", [7] * 8, 248320, 248077, "1.0:0:0.95:0,0.7:0:0.9:0", 16),
        # Blocks of several lengths found by looking back in the text (no probabilities), settings of their own, a grammar's mask.
        _verify("verify_lookup", [15, 3, 0, 9, 15, 1, 12], 248320, 248077, "1.0:0:1:0,0.7:50:0.9:0,1.2:0:1:0.05,0:0:1:0,0.9:1000:0.98:0.001", 0, noise=0.5, masked=0.3),
    ]


def draw(rng):
    most = max(map(_floor, listed()))
    while True:
        case = _drawn(rng)
        if _floor(case) <= most and _values(case) <= 1.5e9:
            del case["name"]
            return case


def _values(case):
    """Scores, or keys and values, of the plain form's rectangle of sequences."""
    if case["op"] == "verify":
        return 0
    rows, longest = _numbers(case["rows"]), max(_numbers(case["lengths"]))
    return len(rows) * longest * max(max(rows) * case["heads"] if case["op"] == "attend" else 0, 3 * case["kv_heads"] * case["head_dim"])


def _floor(case):
    """Roughly the seconds that a case cannot do without."""
    w = work(case)
    return max(w["bytes"] / 6.5e12, w["flops"] / 1.4e15)


def _drawn(rng):
    def log(low, high):
        return int(round(low * (high / low) ** rng.random()))
    kind = rng.choice(["append", "attend", "attend", "attend", "shared", "shared", "verify", "verify"])
    if kind == "verify":
        vocab = log(1000, 248320)
        settings = ",".join("%g:%d:%g:%g" % (rng.choice([0.0, 0.6, 0.8, 1.0, 1.0, 1.5]), rng.choice([0, 0, log(1, 2000)]), rng.choice([1.0, 0.9, 0.95, 0.999]),
                                             rng.choice([0.0, 0.0, 0.02, 0.1])) for _ in range(rng.randint(1, 6)))
        return _verify("", [rng.randint(0, 15) for _ in range(log(1, 8))], vocab, vocab - rng.choice([0, 0, rng.randint(1, 300)]), settings, rng.choice([0, 1, 4, 16, 16, 64]),
                       noise=rng.choice([0.0, 0.3, 1.0, 2.0]), masked=rng.choice([0.0, 0.0, 0.5]))
    kv_heads, group, head_dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 6, 8]), rng.choice([64, 128, 128, 256])
    page, causal = rng.choice([16, 32, 64, 128, 256]), rng.random() < 0.8
    if kind == "shared":
        rows, lengths, groups = [], [], []
        for _ in range(rng.randint(1, 3)):
            n, each, shared = log(2, 24), rng.choice([1, 1, 1, log(2, 16)]), page * max(1, log(100, 24000) // page)
            rows += [each] * n
            lengths += [shared + each + log(1, 3000) for _ in range(n)]
            groups.append("%d:%d" % (n, shared))
        for _ in range(rng.choice([0, 0, 3])):                  # and some that share nothing
            rows.append(1)
            lengths.append(log(1, 5000))
        return _paged("", "attend", kv_heads * group, kv_heads, head_dim, rows, lengths, page, cache=rng.choice(["bf16", "fp16", "e4m3"]), layout=rng.choice(["head", "token"]),
                      causal=causal, groups=",".join(groups))
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
    return _paged("", kind, kv_heads * group, kv_heads, head_dim, rows, lengths, page, layout=rng.choice(["head", "token"]),
                  rotary=rng.choice([head_dim // 4, head_dim // 2, head_dim]), theta=rng.choice([1e4, 1e6, 1e7]), norm=rng.random() < 0.5, window=window, causal=causal)


def _visible(case):
    """Tokens that the rows see, summed over the rows."""
    total = 0
    for n, length in zip(_numbers(case["rows"]), _numbers(case["lengths"])):
        for position in range(length - n, length):
            first = max(0, position + 1 - case["window"]) if case["window"] else 0
            total += (position + 1 if case["causal"] else length) - first
    return total


def work(case):
    if case["op"] == "verify":
        # A row's logits in, its answer out; a comparison and an exponential a value.
        rows = sum(n + 1 for n in _numbers(case["drafts"]))
        return {"bytes": rows * (case["limit"] * 4.0 + 32 + 8.0 * case["candidates"]), "flops": 2.0 * rows * case["limit"]}
    rows, heads, kv_heads, d = sum(_numbers(case["rows"])), case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        # fp32 rows in; 16-bit queries, 8-bit keys and values with a scale a head out.
        return {"bytes": rows * (heads * d * 6.0 + 2 * kv_heads * (d * 5.0 + 4)), "flops": rows * (heads + kv_heads) * (3.0 * case["rotary"] + (4.0 * d if case["norm"] else 0.0))}
    tokens, at = 0, 0
    lengths = _numbers(case["lengths"])
    for n, length in zip(_numbers(case["rows"]), lengths):
        first = max(0, length - n + 1 - case["window"]) if case["window"] else 0
        tokens += length - first
    for n, shared in _groups(case["groups"]):
        tokens -= (n - 1) * shared                             # read once for all
        at += n
    token_bytes = d + 4.0 if case["cache"] == "e4m3" else d * 2.0
    return {"bytes": tokens * kv_heads * 2.0 * token_bytes + rows * heads * d * 4.0, "flops": 4.0 * heads * d * _visible(case)}


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
    if case["op"] == "verify":
        return _prepare_verify(s, case, g)
    rows, lengths, groups = _numbers(case["rows"]), _numbers(case["lengths"]), _groups(case["groups"])
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    t = TYPES.get(case["cache"], torch.bfloat16)             # of the queries
    total = sum(rows)
    held = [-(-length // page) for length in lengths]
    # Of a group's shared pages the first sequence's serve for all.
    leader, behind, at = list(range(len(rows))), [0] * len(rows), 0
    for n, shared in groups:
        leader[at:at + n], behind[at + 1:at + n], at = [at] * n, [shared // page] * (n - 1), at + n
    pages = sum(held) - sum(behind) + 3                      # a few pages belong to nobody
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).numpy().astype(np.int32)
    s.table = np.full((len(rows), max(held)), -1, np.int32)
    at = 0
    for n, count in enumerate(held):
        s.table[n, :behind[n]] = s.table[leader[n], :behind[n]]
        s.table[n, behind[n]:count] = order[at:at + count - behind[n]]
        at += count - behind[n]
    # Each row's sequence and position, and where the cache holds it; the rows as a rectangle, the shorter sequences' last row again.
    sequence = np.repeat(np.arange(len(rows)), rows)
    position = np.concatenate([np.arange(length - n, length) for n, length in zip(rows, lengths)])
    first = np.concatenate([[0], np.cumsum(rows)[:-1]])
    inside = np.arange(max(rows))
    rectangle = first[:, None] + np.minimum(inside, np.array(rows)[:, None] - 1)
    s.position = torch.from_numpy(position).cuda()
    s.page_of = torch.from_numpy(s.table[sequence, position // page].astype(np.int64)).cuda()
    s.slot_of = torch.from_numpy(position % page).cuda()
    s.pages_of = torch.from_numpy(np.maximum(s.table, 0).astype(np.int64)).cuda()
    s.rectangle, s.is_row = torch.from_numpy(rectangle).cuda(), torch.from_numpy(inside < np.array(rows)[:, None]).cuda()
    s.lengths = torch.tensor(lengths, device="cuda")
    shape = (pages, kv_heads, page, d) if case["layout"] == "head" else (pages, page, kv_heads, d)
    if case["op"] == "append":
        s.qkv = torch.randn((total, (heads + 2 * kv_heads) * d), device="cuda", generator=g)
        s.q_norm, s.k_norm = ((1.0 + 0.1 * torch.randn(d, device="cuda", generator=g)).to(torch.bfloat16) for _ in range(2))
        s.q = torch.zeros((total, heads, d), device="cuda", dtype=t)
        s.k, s.v = (torch.zeros(shape, device="cuda", dtype=torch.uint8) for _ in range(2))
        s.k_scale, s.v_scale = (torch.zeros((pages, kv_heads, page), device="cuda") for _ in range(2))
    else:
        # Queries of models with normalised heads: scores spread over several units, a few tokens far above the rest. Tokens' values are of several sizes.
        s.q = (1.5 * torch.randn((total, heads, d), device="cuda", generator=g)).to(t)
        s.out = torch.zeros((total, heads, d), device="cuda", dtype=t)
        k, v = (torch.randn(shape, device="cuda", generator=g) for _ in range(2))
        v *= torch.exp(0.5 * torch.randn(shape[:3] + (1,), device="cuda", generator=g))
        if case["cache"] == "e4m3":
            (s.k, s.k_scale), (s.v, s.v_scale) = (_quantised(x, case["layout"]) for x in (k, v))
        else:
            s.k, s.v = k.to(t), v.to(t)
        del k, v
    if own:
        import splosh_b200 as S
        engine = _the_engine()
        s.paged = S.PagedAttention(engine, heads, kv_heads, d, pages, page_tokens=page, dtype=case["cache"], layout=case["layout"], rotary_dim=case["rotary"],
                                   rope_theta=case["theta"], causal=case["causal"], window=case["window"], max_sequences=len(rows), max_rows=total,
                                   max_context=max(lengths))
        s.paged.batch(rows, lengths, s.table, groups=groups, stream=_stream())
        if case["op"] == "append" and case["norm"]:
            s.norms = [engine.tensor_vector(w.view(torch.int16).cpu().numpy().view(np.uint16)) for w in (s.q_norm, s.k_norm)]
    torch.cuda.synchronize()
    return s


def _quantised(x, layout):
    """Codes (as bytes) and scales [pages][kv heads][tokens] of keys or values."""
    scale = (x.abs().amax(-1, keepdim=True) / LARGEST).clamp(min=SCALE_MIN)
    codes = (x / scale).to(E4M3).view(torch.uint8)
    scale = scale[..., 0]
    return codes, (scale if layout == "head" else scale.transpose(1, 2)).contiguous()


def _prepare_verify(s, case, g):
    drafts, vocab, limit = _numbers(case["drafts"]), case["vocab"], case["limit"]
    s.first = np.concatenate([[0], np.cumsum([n + 1 for n in drafts])]).astype(np.int32)
    rows = int(s.first[-1])
    # A language model's logits: a broad bell, and some dozens of likely tokens above it.
    x = 2.0 * torch.randn((rows, vocab), device="cuda", generator=g)
    likely = torch.randint(0, limit, (rows, 48), device="cuda", generator=g)
    x.scatter_add_(1, likely, 6.0 + 4.0 * torch.rand((rows, 48), device="cuda", generator=g))
    if case["masked"]:
        x[torch.rand((rows, vocab), device="cuda", generator=g) < case["masked"]] = -math.inf
    s.logits = x
    # The drafter sees nearly the same: its candidates, their probabilities, and the one that it took. (Masked tokens may be among them, as a drafter knows no grammar.)
    y = torch.where(x > -math.inf, x, -2.0)[:, :limit] + case["noise"] * torch.randn((rows, limit), device="cuda", generator=g)
    value, ids = torch.topk(y, max(1, case["candidates"]), dim=1)
    p = torch.softmax(value, 1)
    taken = (p.cumsum(1) < torch.rand((rows, 1), device="cuda", generator=g)).sum(1, keepdim=True).clamp(max=p.shape[1] - 1)
    s.drafts = ids.gather(1, taken)[:, 0].to(torch.int32)
    s.drafts[torch.from_numpy(s.first[1:].astype(np.int64) - 1).cuda()] = -1          # a sequence's last row has none
    s.candidates, s.probabilities = ids.to(torch.int32).contiguous(), p.contiguous()
    settings = [[float(v) for v in one.split(":")] for one in case["settings"].split(",")]
    per_row = np.array([settings[n % len(settings)] for n in range(len(drafts)) for _ in range(drafts[n] + 1)])
    s.temperature, s.top_p, s.min_p = (torch.tensor(per_row[:, n], dtype=torch.float32, device="cuda") for n in (0, 2, 3))
    s.top_k = torch.tensor(per_row[:, 1], dtype=torch.int32, device="cuda")
    s.uniform = torch.rand((rows, 2), device="cuda", generator=g)
    s.sequence = torch.from_numpy(np.repeat(np.arange(len(drafts)), np.diff(s.first))).cuda()
    s.first = torch.from_numpy(s.first).cuda()
    s.ids = torch.zeros(rows, dtype=torch.int32, device="cuda")
    s.accepted, s.next = (torch.zeros(len(drafts), dtype=torch.int32, device="cuda") for _ in range(2))
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
    return _verify_rows(state)


def _append(s):
    c = s.case
    heads, kv_heads, d = c["heads"], c["kv_heads"], c["head_dim"]
    out = {"q": s.q, "k": s.k.view(E4M3), "v": s.v.view(E4M3), "k_scale": s.k_scale, "v_scale": s.v_scale}
    if own:
        ld = (heads + 2 * kv_heads) * d
        base = s.qkv.data_ptr()
        q_norm, k_norm = s.norms if c["norm"] else (None, None)
        s.paged.append(base, base + 4 * heads * d, base + 4 * (heads + kv_heads) * d, s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), ld=ld,
                       q_norm=q_norm, k_norm=k_norm, k_scale=s.k_scale.data_ptr(), v_scale=s.v_scale.data_ptr(), stream=_stream())
        return out
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

    def stored(x, cache, scales):
        scale = (x.abs().amax(-1, keepdim=True) / LARGEST).clamp(min=SCALE_MIN)
        codes = (x / scale).to(E4M3).view(torch.uint8)
        if c["layout"] == "head":
            cache[s.page_of, :, s.slot_of] = codes
        else:
            cache[s.page_of, s.slot_of] = codes
        scales[s.page_of, :, s.slot_of] = scale[..., 0]
    s.q.copy_(turned(q, heads, s.q_norm).to(s.q.dtype))
    stored(turned(k, kv_heads, s.k_norm), s.k, s.k_scale)
    stored(v.reshape(-1, kv_heads, d), s.v, s.v_scale)
    return out


def _attend(s):
    c = s.case
    if own:
        scales = {"k_scale": s.k_scale.data_ptr(), "v_scale": s.v_scale.data_ptr()} if c["cache"] == "e4m3" else {}
        s.paged.attend(s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.out.data_ptr(), stream=_stream(), **scales)
        return s.out
    heads, kv_heads, d = c["heads"], c["kv_heads"], c["head_dim"]
    sequences, most = s.rectangle.shape

    def of_sequences(cache, scales):
        x = cache[s.pages_of]                                  # [sequence][page] ...
        x = x if c["layout"] == "head" else x.transpose(2, 3)
        x = x.view(E4M3).float() * scales[s.pages_of][..., None] if scales is not None else x.float()
        return x.transpose(1, 2).reshape(sequences, kv_heads, -1, d)
    k, v = of_sequences(s.k, s.k_scale if c["cache"] == "e4m3" else None), of_sequences(s.v, s.v_scale if c["cache"] == "e4m3" else None)
    token, position = torch.arange(k.shape[2], device="cuda"), s.position[s.rectangle][..., None]
    seen = token <= position if c["causal"] else (token < s.lengths[:, None, None]).expand(-1, most, -1)
    if c["window"]:
        seen = seen & (token > position - c["window"])
    q = s.q[s.rectangle].float().reshape(sequences, most, kv_heads, -1, d).transpose(1, 2)       # [sequence][kv head][row][head of the group]
    score = (q.flatten(2, 3) @ k.transpose(2, 3)).view(*q.shape[:4], -1) * d ** -0.5
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    score = score.sub_(score.amax(-1, keepdim=True)).exp_()
    out = (score.flatten(2, 3) @ v) / score.sum(-1).flatten(2, 3)[..., None]
    out = out.view(q.shape).transpose(1, 2).reshape(sequences, most, heads, d)
    s.out.copy_(out[s.is_row].to(s.out.dtype))
    return s.out


def _verify_rows(s):
    c = s.case
    if own:
        candidates = {"candidates": c["candidates"], "candidate_ids": s.candidates.data_ptr(), "probabilities": s.probabilities.data_ptr()} if c["candidates"] else {}
        s.engine.pass_verify(s.logits.data_ptr(), s.accepted.shape[0], s.ids.shape[0], c["vocab"], c["limit"], s.first.data_ptr(), s.drafts.data_ptr(), s.uniform.data_ptr(),
                             s.ids.data_ptr(), s.accepted.data_ptr(), s.next.data_ptr(), temperature=s.temperature.data_ptr(), top_k=s.top_k.data_ptr(),
                             top_p=s.top_p.data_ptr(), min_p=s.min_p.data_ptr(), stream=_stream(), **candidates)
        return {"ids": s.ids, "accepted": s.accepted, "next": s.next}
    limit = c["limit"]
    x, order = torch.sort(s.logits[:, :limit], dim=1, descending=True, stable=True)
    greedy = ~(s.temperature > 0)
    weight = torch.exp((x.double() - x[:, :1].double()) / torch.where(greedy, 1.0, s.temperature.double())[:, None])          # a masked value's is zero
    place = torch.arange(limit, device="cuda")
    top_k = torch.where(s.top_k > 0, s.top_k, limit)[:, None]
    weight = torch.where(place < torch.where(greedy[:, None], 1, top_k), weight, 0.0)
    total = weight.cumsum(1)
    kept = (total < s.top_p.double()[:, None] * total[:, -1:]).sum(1, keepdim=True)      # the place where the prefix is complete
    weight = torch.where((place <= kept) | (s.top_p >= 1)[:, None], weight, 0.0)
    weight = torch.where((weight >= s.min_p.double()[:, None]) | greedy[:, None], weight, 0.0)
    p = weight / weight.sum(1, keepdim=True)
    # The drafter's probabilities at the places of the order: of its candidates, or one of its only choice.
    is_draft = s.drafts >= 0
    draft = torch.where(is_draft, s.drafts, 0).long()[:, None]
    q = torch.zeros((x.shape[0], limit), dtype=torch.float64, device="cuda")
    if c["candidates"]:
        q.scatter_(1, s.candidates.long(), s.probabilities.double())
    else:
        q.scatter_(1, draft, 1.0)
    q = torch.where(is_draft[:, None], q, 0.0).gather(1, order)
    here = order == draft
    p_draft, q_draft = (torch.where(here, y, 0.0).sum(1) for y in (p, q))
    stays = is_draft & (s.uniform[:, 0].double() * q_draft < p_draft)
    rest = (p - q).clamp(min=0.0)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p)
    total = rest.cumsum(1)
    pick = (total < s.uniform[:, 1:].double() * total[:, -1:]).sum(1, keepdim=True)
    last = torch.where(rest > 0, place, 0).amax(1, keepdim=True)
    pick = order.gather(1, torch.minimum(pick, last))[:, 0]
    s.ids.copy_(torch.where(stays, -1, pick))
    # A sequence's first row whose draft does not stay.
    row = torch.arange(s.ids.shape[0], device="cuda")
    end = s.first[1:].long()
    stop = end.scatter_reduce(0, s.sequence, torch.where(stays, s.ids.shape[0], row), "amin")
    s.accepted.copy_(stop - s.first[:-1])
    s.next.copy_(torch.where(stop < end, s.ids[stop.clamp(max=s.ids.shape[0] - 1)], -1))
    return {"ids": s.ids, "accepted": s.accepted, "next": s.next}


# ---- the definitions in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    return _exact_verify(case, s)


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
    pages, tokens = s.k_scale.shape[0], s.k_scale.shape[2]
    for name, first in (("k", heads), ("v", heads + kv_heads)):
        # What the codes stand for before they are rounded: the value over its token's scale.
        codes, scales = np.zeros((pages, kv_heads, tokens, d)), np.zeros((pages, kv_heads, tokens))
        for r in range(len(page)):
            scales[page[r], :, slot[r]] = np.maximum(np.abs(z[r, first:first + kv_heads]).max(axis=1) / LARGEST, SCALE_MIN)
            codes[page[r], :, slot[r]] = z[r, first:first + kv_heads] / scales[page[r], :, slot[r]][:, None]
        out[name] = codes if case["layout"] == "head" else np.ascontiguousarray(codes.transpose(0, 2, 1, 3))
        out[name + "_scale"] = scales
    return out


def _exact_attend(case, s):
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    group = heads // kv_heads
    out = torch.zeros(tuple(s.q.shape), dtype=torch.float64)
    at = 0
    for n, (count, length) in enumerate(zip(_numbers(case["rows"]), _numbers(case["lengths"]))):
        used = s.pages_of[n, :-(-length // page)]
        position = torch.arange(length - count, length, device="cuda")[:, None]
        token = torch.arange(length, device="cuda")[None, :]
        hidden = (token > position) if case["causal"] else torch.zeros((count, length), dtype=torch.bool, device="cuda")
        if case["window"]:
            hidden |= token + case["window"] <= position
        for h in range(kv_heads):
            pair = []
            for name in ("k", "v"):
                cache = getattr(s, name)[used]
                x = cache[:, h] if case["layout"] == "head" else cache[:, :, h]
                if case["cache"] == "e4m3":
                    x = x.contiguous().view(E4M3).double() * getattr(s, name + "_scale")[used][:, h, :, None].double()
                pair.append(x.double().flatten(0, 1)[:length])
            for r0 in range(0, count, 512):
                q = s.q[at + r0:min(at + count, at + r0 + 512), h * group:(h + 1) * group].double()
                logit = torch.einsum("rgd,td->rgt", q, pair[0]) / math.sqrt(d)
                logit[hidden[r0:r0 + 512, None].expand_as(logit)] = -math.inf
                out[at + r0:at + r0 + q.shape[0], h * group:(h + 1) * group] = torch.einsum("rgt,td->rgd", torch.softmax(logit, -1), pair[1]).cpu()
        at += count
    return out


def _exact_verify(case, s):
    first, drafts, uniform = (x.cpu().numpy() for x in (s.first, s.drafts, s.uniform))
    candidates, probabilities = s.candidates.cpu().numpy(), s.probabilities.double().cpu().numpy()
    ids = np.zeros(len(drafts), np.int32)
    for r in range(len(drafts)):
        x = s.logits[r, :case["limit"]].double().cpu().numpy()
        t, k, top_p, m = (float(a[r]) for a in (s.temperature, s.top_k, s.top_p, s.min_p))
        order = np.argsort(-x, kind="stable")
        order = order[:int(np.isfinite(x).sum())]
        if t <= 0:
            order, w = order[:1], np.ones(1)
        else:
            if k > 0:
                order = order[:int(k)]
            w = np.exp((x[order] - x[order[0]]) / t)
            if top_p < 1:
                c = np.cumsum(w)
                n = int(np.searchsorted(c, top_p * c[-1], side="left")) + 1
                order, w = order[:n], w[:n]
            keep = w >= m
            order, w = order[keep], w[keep]
        target = dict(zip(order.tolist(), (w / w.sum()).tolist()))
        drafted = {}
        if drafts[r] >= 0:
            drafted = dict(zip(candidates[r].tolist(), probabilities[r].tolist())) if case["candidates"] else {int(drafts[r]): 1.0}
            if float(uniform[r, 0]) * drafted.get(int(drafts[r]), 0.0) < target.get(int(drafts[r]), 0.0):
                ids[r] = -1
                continue
        rest = np.array([max(0.0, target[i] - drafted.get(i, 0.0)) for i in order.tolist()])
        if not rest.sum() > 0:
            rest = np.array(list(target.values()))
        c = np.cumsum(rest)
        ids[r] = order[min(int(np.searchsorted(c, float(uniform[r, 1]) * c[-1], side="left")), int(np.flatnonzero(rest)[-1]))]
    accepted, following = [], []
    for a, b in zip(first[:-1], first[1:]):
        n = next((r for r in range(a, b) if ids[r] >= 0), b)
        accepted.append(n - a)
        following.append(ids[n] if n < b else -1)
    return {"ids": torch.from_numpy(ids), "accepted": torch.tensor(accepted, dtype=torch.int32), "next": torch.tensor(following, dtype=torch.int32)}
