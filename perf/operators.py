"""Cases of the packed-token operators, with their plain forms.

Three operators serve the attention blocks when several requests of different sizes share one call:
``adapter_linear`` (a shared projection with each request's low-rank adapter beside it),
``rotary_axes`` (rotary positions along several axes) and ``attention`` (document, causal and prefix
masks, capped scores, a distance bias, grouped heads, a cache with lengths). ``run`` computes one of
them with elementary torch operations in 32 bits, or, with ``own``, by the package's own call.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _ops():
    import sys
    from pathlib import Path

    package = str(Path(__file__).resolve().parents[1] / "mlx-generate-ctmr_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from ctmr_b200 import ops

    return ops


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # Attention of the diffusion network's level-2 blocks (8 heads of 32) over the latent grids of
        # seven volumes of different extents packed in one call: 16x16x8 down to one of 5x7x3.
        dict(name="attn-volumes", op="attention", form="packed", dtype="fp16", heads=8, kv_heads=8, dim=32,
             q="2048,1024,2048,512,1183,105,2048", k="", causal=False, prefix="", cap=0.0, bias=False, lse=False),
        # One long latent sequence, both directions, with the distance bias: the largest product.
        dict(name="attn-long-bias", op="attention", form="packed", dtype="bf16", heads=8, kv_heads=8, dim=128,
             q="8192", k="", causal=False, prefix="", cap=0.0, bias=True, lse=False),
        # Conditioned generation: each request's condition tokens are a prefix that all its tokens see,
        # the rest causal; grouped heads, capped scores; odd lengths, one request of a single token.
        dict(name="attn-prefix-cap", op="attention", form="packed", dtype="bf16", heads=16, kv_heads=4, dim=128,
             q="1531,1,2300,264", k="", causal=True, prefix="200,0,777,264", cap=30.0, bias=False, lse=True),
        # New tokens against a shorter or longer context (queries without any key among them); head size 72.
        dict(name="attn-cross-ragged", op="attention", form="packed", dtype="fp16", heads=12, kv_heads=6, dim=72,
             q="300,513,64,77", k="900,100,0,1301", causal=True, prefix="", cap=0.0, bias=True, lse=True),
        # Serving, one new token for each of 16 requests over a cache of up to 8192 tokens.
        dict(name="attn-token-16", op="attention", form="cache", dtype="bf16", heads=16, kv_heads=4, dim=128,
             q="1", k="8192", batch=16, causal=True, prefix="", cap=0.0, bias=False, lse=False),
        # The smallest: one token of one request over a short cache.
        dict(name="attn-token-1", op="attention", form="cache", dtype="fp16", heads=8, kv_heads=8, dim=64,
             q="1", k="300", batch=1, causal=True, prefix="", cap=50.0, bias=True, lse=False),
        # Projection of the packed tokens of eight requests, ragged, two of them without an adapter: prompts.
        dict(name="lora-prompts", op="linear", dtype="bf16", inner=4096, outer=4096, rank=32, adapters=6, bias=True,
             rows="2048,1000,1,1777,512,1024,1333,497", index="0,3,1,-1,5,2,-1,0"),
        # The level-3 attention's stacked Q/K/V projection (512 channels) for three volumes of 256 tokens or fewer.
        dict(name="lora-volumes", op="linear", dtype="fp16", inner=512, outer=1536, rank=8, adapters=3, bias=True,
             rows="256,105,256", index="2,0,1"),
        # Serving, one row for each of 32 requests with 24 adapters among them.
        dict(name="lora-token-32", op="linear", dtype="bf16", inner=4096, outer=4096, rank=16, adapters=24, bias=False,
             rows=",".join(["1"] * 32), index=",".join(str((7 * i) % 25 - 1) for i in range(32))),
        # Positions of two large latent volumes and a small one: 24 query and key heads of 128, bf16.
        dict(name="rope-volumes", op="rotary", dtype="bf16", heads=24, dim=128, sections="16,24,24", interleaved=False,
             inverse=False, grids="16x32x32,12x28x20,5x7x3", spacing=0.0),
        # The gradient's direction (the inverse rotation) in 32 bits, positions in millimetres, partial rotation.
        dict(name="rope-mm-inverse", op="rotary", dtype="fp32", heads=8, dim=72, sections="10,11,11", interleaved=True,
             inverse=True, grids="16x16x8,9x11x13", spacing=1.17),
        # One small volume of the level-2 blocks: latency.
        dict(name="rope-small", op="rotary", dtype="fp16", heads=16, dim=32, sections="4,6,6", interleaved=False,
             inverse=False, grids="5x7x3", spacing=0.0),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _parts(rng, total, count):
    cuts = sorted(rng.randint(0, total) for _ in range(count - 1))
    return [b - a for a, b in zip([0, *cuts], [*cuts, total])]


def _text(values):
    return ",".join(str(v) for v in values)


def _ints(text):
    return [int(v) for v in text.split(",")] if text else []


def draw(rng):
    kind = rng.choice(["packed", "packed", "cache", "linear", "linear", "rotary"])
    half = rng.choice(["bf16", "fp16"])
    if kind == "packed":
        # Documents of any lengths, up to 6000 tokens in all; keys the queries' own or another context's.
        kv_heads, group, dim = rng.choice([(8, 1), (4, 2), (2, 4), (1, 8), (3, 2)]) + (8 * rng.randint(4, 16),)
        total, docs = _log_int(rng, 64, 6000), rng.randint(1, 9)
        causal = rng.random() < 0.5
        q = _parts(rng, total, docs)
        k = _parts(rng, _log_int(rng, 64, 6000), docs) if rng.random() < 0.3 else None
        lengths = k or q
        prefix = [rng.randint(0, n) for n in lengths] if causal and rng.random() < 0.5 else []
        return dict(op="attention", form="packed", dtype=half, heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    q=_text(q), k=_text(k or []), causal=causal, prefix=_text(prefix),
                    cap=rng.choice([0.0, 0.0, 15.0, 50.0]), bias=rng.random() < 0.4, lse=rng.random() < 0.5)
    if kind == "cache":
        kv_heads, group, dim = rng.choice([(8, 1), (4, 4), (8, 2), (2, 8), (1, 5)]) + (rng.choice([32, 64, 80, 128]),)
        return dict(op="attention", form="cache", dtype=half, heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    q=str(rng.choice([1, 1, 1, 2, 5])), k=str(_log_int(rng, 1, 16000)), batch=_log_int(rng, 1, 24),
                    causal=True, prefix="", cap=rng.choice([0.0, 0.0, 30.0]), bias=rng.random() < 0.4, lse=False)
    if kind == "linear":
        inner, outer = 8 * _log_int(rng, 8, 512), _log_int(rng, 64, 4096)
        total, adapters = _log_int(rng, 1, 8000), rng.randint(1, 24)
        rows = [1] * total if total <= 64 and rng.random() < 0.5 else _parts(rng, total, rng.randint(1, 10))
        return dict(op="linear", dtype=half, inner=inner, outer=outer, rank=8 * rng.choice([1, 2, 3, 4, 8, 16]),
                    adapters=adapters, bias=rng.random() < 0.5, rows=_text(rows),
                    index=_text(rng.randint(-1, adapters - 1) for _ in rows))
    dim = 8 * rng.randint(2, 20)
    axes = rng.randint(1, 4)
    sections = _parts(rng, rng.randint(axes, dim // 2), axes)
    grids = ["x".join(str(_log_int(rng, 1, 24)) for _ in range(axes)) for _ in range(rng.randint(1, 4))]
    return dict(op="rotary", dtype=rng.choice(["bf16", "fp16", "fp32"]), heads=rng.randint(1, 40 if axes < 4 else 2), dim=dim,
                sections=_text(sections), interleaved=rng.random() < 0.5, inverse=rng.random() < 0.3,
                grids=_text(grids), spacing=rng.choice([0.0, 0.0, 0.73, 2.5]))


# ---------------------------------------------------------------------------------------------- inputs
def _offsets(lengths, device):
    return torch.tensor([0, *lengths], dtype=torch.int32).cumsum(0, dtype=torch.int32).to(device)


def _inputs(case, seed, device):
    gen = torch.Generator(device=device).manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, to=dtype):
        return (torch.randn(shape, generator=gen, device=device) * std).to(to)

    if case["op"] == "attention":
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
        slopes = None
        if case["bias"]:  # slopes in a geometric row, 2^-1 down to 2^-8, each seed a little different
            slopes = torch.exp2(-8.0 * torch.arange(1, heads + 1, device=device) / heads) * (
                0.9 + 0.2 * torch.rand(heads, generator=gen, device=device))
        common = dict(scale=dim ** -0.5, causal=case["causal"], cap=case["cap"], slopes=slopes)
        if case["form"] == "cache":
            # The cache is filled up to a different length for each request.
            batch, lq, lk = case["batch"], int(case["q"]), int(case["k"])
            lengths = torch.randint((lk + 1) // 2, lk + 1, (batch,), generator=gen, device=device, dtype=torch.int32)
            return dict(common, q=randn(batch, lq, heads, dim), k=randn(batch, lk, kv_heads, dim),
                        v=randn(batch, lk, kv_heads, dim), k_lengths=lengths)
        q_len, k_len = _ints(case["q"]), _ints(case["k"]) or _ints(case["q"])
        prefix = torch.tensor(_ints(case["prefix"]), dtype=torch.int32).to(device) if case["prefix"] else None
        if not case["k"]:  # self-attention: Q, K and V are views of one projection's rows
            rows = randn(sum(q_len), heads + 2 * kv_heads, dim)
            q, k, v = rows.split((heads, kv_heads, kv_heads), dim=1)
        else:
            q, k, v = randn(sum(q_len), heads, dim), randn(sum(k_len), kv_heads, dim), randn(sum(k_len), kv_heads, dim)
        return dict(common, q=q, k=k, v=v, q_offsets=_offsets(q_len, device), k_offsets=_offsets(k_len, device),
                    prefix=prefix)
    if case["op"] == "linear":
        inner, outer, rank, n = case["inner"], case["outer"], case["rank"], case["adapters"]
        rows = _ints(case["rows"])
        return dict(x=randn(sum(rows), inner), weight=randn(outer, inner, std=inner ** -0.5),
                    bias=randn(outer, std=0.5) if case["bias"] else None,
                    down=randn(n, rank, inner, std=inner ** -0.5), up=randn(n, outer, rank, std=rank ** -0.5),
                    scale=0.25 + torch.rand(n, generator=gen, device=device), offsets=_offsets(rows, device),
                    index=torch.tensor(_ints(case["index"]), dtype=torch.int32).to(device))
    sections = tuple(_ints(case["sections"]))
    grids = []
    for text in case["grids"].split(","):
        extents = [torch.arange(int(n)) for n in text.split("x")]
        grids.append(torch.stack([a.reshape(-1) for a in torch.meshgrid(*extents, indexing="ij")], dim=1))
    positions = torch.cat(grids).to(device)
    positions = (positions.to(torch.float32) * case["spacing"] if case["spacing"] else positions.to(torch.int32)).contiguous()
    inv_freq = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in sections])
    return dict(x=randn(positions.shape[0], case["heads"], case["dim"]), positions=positions,
                inv_freq=inv_freq.to(torch.float32).to(device), sections=sections,
                interleaved=case["interleaved"], inverse=case["inverse"])


def prepare(case, seed):
    return dict(_inputs(case, seed, "cuda"), op=case["op"], lse=bool(case.get("lse", False)))


# ---------------------------------------------------------------------------------------------- plain forms
def _documents(offsets, total):
    """For each of `total` tokens its document and its place in it."""
    at = torch.arange(total, device=offsets.device, dtype=torch.int32)
    doc = torch.searchsorted(offsets[1:].contiguous(), at, right=True)
    return doc, at - offsets[doc]


def _softmax_values(scores, seen, v):
    """(out, lse) of scores over the last axis where `seen`; rows that see nothing give zeros and -inf."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    total = p.sum(dim=-1, keepdim=True)
    out = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)
    return out, (torch.log(total) + top).squeeze(-1)


def _scores(q, k, scale, cap):
    s = (q @ k.transpose(-1, -2)) * scale
    return torch.tanh(s / cap) * cap if cap else s


def _plain_attention(s):
    q, k, v = s["q"], s["k"], s["v"]
    group = q.shape[-2] // k.shape[-2]
    qf = q.float().transpose(-3, -2)
    kf, vf = (t.float().transpose(-3, -2).repeat_interleave(group, dim=-3) for t in (k, v))
    scores = _scores(qf, kf, s["scale"], s["cap"])
    if q.dim() == 4:
        lengths, lq = s["k_lengths"].view(-1, 1, 1), q.shape[1]
        key = torch.arange(k.shape[1], device=q.device).view(1, 1, -1)
        place = torch.arange(lq, device=q.device).view(1, -1, 1) + lengths - lq
        seen = (key < lengths) & (key <= place)
        gap, seen = (place - key).abs().unsqueeze(1), seen.unsqueeze(1)
    else:
        qo, ko = s["q_offsets"], s["k_offsets"]
        (q_doc, q_at), (k_doc, k_at) = _documents(qo, q.shape[0]), _documents(ko, k.shape[0])
        place = (q_at + (ko[1:] - ko[:-1] - qo[1:] + qo[:-1])[q_doc]).view(-1, 1)
        key = k_at.view(1, -1)
        seen = q_doc.view(-1, 1) == k_doc.view(1, -1)
        if s["causal"]:
            before = key <= place
            if s["prefix"] is not None:
                before = before | (key < s["prefix"][k_doc].view(1, -1))
            seen = seen & before
        gap = (place - key).abs()
    if s["slopes"] is not None:
        scores = scores - s["slopes"].view(-1, 1, 1) * gap
    out, lse = _softmax_values(scores, seen, vf)
    out = out.transpose(-3, -2).to(q.dtype)
    return (out, lse.transpose(-2, -1).contiguous()) if s["lse"] else out


def _plain_linear(s):
    x, index = s["x"].float(), s["index"]
    y = x @ s["weight"].float().T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    doc, _ = _documents(s["offsets"], x.shape[0])
    adapter = index[doc].view(-1, 1)
    n, rank, inner = s["down"].shape
    # All adapters' inner products side by side; each row keeps its own adapter's.
    t = (x @ s["down"].float().view(n * rank, inner).T).view(-1, n, rank) * s["scale"].view(1, n, 1)
    mine = adapter == torch.arange(n, device=x.device).view(1, n)
    t = torch.where(mine.unsqueeze(-1), t, torch.zeros_like(t)).view(-1, n * rank)
    return (y + t @ s["up"].float().permute(0, 2, 1).reshape(n * rank, -1)).to(s["x"].dtype)


def _rotate(x, cos, sin, interleaved):
    """x[..., :2 * pairs] rotated in pairs by angles of (tokens, 1, pairs); the rest as it is."""
    pairs = cos.shape[-1]
    turned, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = turned[..., :pairs], turned[..., pairs:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _angles(s, dtype):
    sections = torch.tensor(s["sections"], device=s["positions"].device)
    axis = torch.arange(len(s["sections"]), device=s["positions"].device).repeat_interleave(sections)
    angle = s["positions"].to(dtype)[:, axis] * s["inv_freq"].to(dtype)
    return (-angle if s["inverse"] else angle).unsqueeze(1)


def _plain_rotary(s):
    angle = _angles(s, torch.float32)
    return _rotate(s["x"].float(), torch.cos(angle), torch.sin(angle), s["interleaved"]).to(s["x"].dtype)


def _own_attention(s):
    ops = _ops()
    common = dict(scale=s["scale"], causal=s["causal"], cap=s["cap"], slopes=s["slopes"], return_lse=s["lse"])
    if s["q"].dim() == 4:
        return ops.attention(s["q"], s["k"], s["v"], k_lengths=s["k_lengths"], **common)
    return ops.attention(s["q"], s["k"], s["v"], q_offsets=s["q_offsets"], k_offsets=s["k_offsets"],
                         prefix=s["prefix"], **common)


def run(state):
    if state["op"] == "attention":
        return _own_attention(state) if own else _plain_attention(state)
    if state["op"] == "linear":
        if not own:
            return _plain_linear(state)
        return _ops().adapter_linear(state["x"], state["weight"], state["bias"], down=state["down"], up=state["up"],
                                     scale=state["scale"], offsets=state["offsets"], index=state["index"])
    if not own:
        return _plain_rotary(state)
    return _ops().rotary_axes(state["x"], state["positions"], state["inv_freq"], state["sections"],
                              interleaved=state["interleaved"], inverse=state["inverse"])


# ---------------------------------------------------------------------------------------------- work
def _seen_pairs(lq, lk, causal, prefix):
    """Query-key pairs of one document: a query at place p = i + lk - lq sees max(p + 1, prefix) keys, within [0, lk]."""
    if not causal:
        return lq * lk
    return sum(max(0, min(lk, max(i + lk - lq + 1, prefix))) for i in range(lq))


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attention":
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
        if case["form"] == "cache":
            lq, mean = int(case["q"]), 0.75 * int(case["k"])
            rows, keys, pairs = case["batch"] * lq, case["batch"] * mean, case["batch"] * lq * mean
        else:
            q_len, k_len = _ints(case["q"]), _ints(case["k"]) or _ints(case["q"])
            prefix = _ints(case["prefix"]) or [0] * len(q_len)
            rows, keys = sum(q_len), sum(k_len)
            pairs = sum(_seen_pairs(a, b, case["causal"], p) for a, b, p in zip(q_len, k_len, prefix))
        lse = 4 * rows * heads if case["lse"] else 0
        return {"bytes": size * dim * (2 * rows * heads + 2 * keys * kv_heads) + lse, "flops": 4 * pairs * heads * dim}
    if case["op"] == "linear":
        inner, outer, rank = case["inner"], case["outer"], case["rank"]
        rows, index = _ints(case["rows"]), _ints(case["index"])
        total, used = sum(rows), len({i for n, i in zip(rows, index) if n and i >= 0})
        adapted = sum(n for n, i in zip(rows, index) if i >= 0)
        return {"bytes": size * (total * (inner + outer) + inner * outer + used * rank * (inner + outer)),
                "flops": 2 * total * inner * outer + 2 * adapted * rank * (inner + outer)}
    tokens = sum(math.prod(int(n) for n in g.split("x")) for g in case["grids"].split(","))
    pairs = sum(_ints(case["sections"]))
    return {"bytes": 2 * size * tokens * case["heads"] * case["dim"] + 4 * tokens * len(_ints(case["sections"])),
            "flops": 6 * tokens * case["heads"] * pairs}


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_document(q, k, v, scale, cap, slopes, causal, prefix):
    """One document's attention in 64 bits: q (Lq, H, D), k and v (Lk, H, D) -> (Lq, H, D), (Lq, H)."""
    lq, lk = q.shape[0], k.shape[0]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    if lq == 0 or lk == 0:
        return out, lse
    place = torch.arange(lq, device=q.device)[:, None] + (lk - lq)
    key = torch.arange(lk, device=q.device)[None, :]
    seen = ((key <= place) | (key < prefix)) if causal else torch.ones((lq, lk), dtype=torch.bool, device=q.device)
    some = seen.any(dim=1)
    for h in range(q.shape[1]):
        s = torch.einsum("id,jd->ij", q[:, h], k[:, h]) * scale
        if cap:
            s = cap * torch.tanh(s / cap)
        if slopes is not None:
            s = s - slopes[h] * (place - key).abs()
        s = torch.where(seen, s, torch.full_like(s, -math.inf))[some]
        lse[some, h] = torch.logsumexp(s, dim=1)
        out[some, h] = torch.softmax(s, dim=1) @ v[:, h]
    return out, lse


def exact(case, seed):
    s = _inputs(case, seed, "cuda")
    if case["op"] == "attention":
        q, k, v = (s[n].double() for n in ("q", "k", "v"))
        group = q.shape[-2] // k.shape[-2]
        heads = torch.arange(q.shape[-2], device=q.device) // group
        k, v = k[..., heads, :], v[..., heads, :]
        slopes = s["slopes"].double() if s["slopes"] is not None else None
        rest = (s["scale"], s["cap"], slopes, s["causal"])
        if case["form"] == "cache":
            done = [_exact_document(q[b], k[b, :n], v[b, :n], *rest, 0) for b, n in enumerate(s["k_lengths"].tolist())]
            out, lse = torch.stack([o for o, _ in done]), torch.stack([m for _, m in done])
        else:
            qo, ko = s["q_offsets"].tolist(), s["k_offsets"].tolist()
            prefix = s["prefix"].tolist() if s["prefix"] is not None else [0] * (len(qo) - 1)
            done = [_exact_document(q[qo[i]:qo[i + 1]], k[ko[i]:ko[i + 1]], v[ko[i]:ko[i + 1]], *rest, prefix[i])
                    for i in range(len(qo) - 1)]
            out, lse = torch.cat([o for o, _ in done]), torch.cat([m for _, m in done])
        return (out, lse) if case["lse"] else out
    if case["op"] == "linear":
        x = s["x"].double()
        y = torch.einsum("ti,oi->to", x, s["weight"].double())
        if s["bias"] is not None:
            y += s["bias"].double()
        start = 0
        for n, a in zip(_ints(case["rows"]), _ints(case["index"])):
            if n and a >= 0:
                inner = torch.einsum("ti,ri->tr", x[start:start + n], s["down"][a].double())
                y[start:start + n] += float(s["scale"][a]) * torch.einsum("tr,or->to", inner, s["up"][a].double())
            start += n
        return y
    x, column = s["x"].double(), 0
    y = x.clone()
    pairs = sum(s["sections"])
    for axis, n in enumerate(s["sections"]):
        for c in range(column, column + n):
            angle = s["positions"][:, axis].double() * s["inv_freq"][c].double() * (-1.0 if s["inverse"] else 1.0)
            i, j = (2 * c, 2 * c + 1) if s["interleaved"] else (c, c + pairs)
            cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
            y[:, :, i] = x[:, :, i] * cos - x[:, :, j] * sin
            y[:, :, j] = x[:, :, i] * sin + x[:, :, j] * cos
        column += n
    return y
