"""Work of the ragged-batch decode operators: block tables and slot maps from
request lengths, writing and reading a paged cache of 8 bits with a scale for
each block of tokens and kv head, attention over that cache, and sampling with
temperature, top-k, top-p and min-p from given uniforms.

Each case is one pass through one operator on seeded data.  ``own`` selects
the framework's kernels; otherwise the plain forms below compute the same
results with elementary torch operations.  ``exact`` restates the operators in
64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one verify step of the large configuration: 32 requests, 4 drafts + 1 token each
        dict(name="plan verify 32", kind="plan", batch=32, q=5, len=3080, page=128, ragged=False),
        # a full server: thousands of requests, decode steps mixed with prompt chunks
        dict(name="plan mixed 2048", kind="plan", batch=2048, q=64, len=8192, page=128, ragged=True),
        # the same verify step's cache write, 32 heads of 128
        dict(name="append verify", kind="append", batch=32, q=5, len=3080, kv_heads=32, dim=128, page=128, block=16,
             dtype="bf16", ragged=False),
        # prompts written whole: 4 x 2,048 tokens
        dict(name="append prompt", kind="append", batch=4, q=2048, len=2048, kv_heads=32, dim=128, page=128, block=16,
             dtype="bf16", ragged=False),
        # the first tokens of small requests (4 heads of 64, fp32): latency
        dict(name="attend small", kind="attend", batch=8, q=1, len=100, heads=4, kv_heads=4, dim=64, page=128, block=16,
             dtype="f32", window=0, ragged=True),
        # a verify pass of the large configuration: 32 heads of 128, 5 query rows a request
        dict(name="attend verify", kind="attend", batch=32, q=5, len=3080, heads=32, kv_heads=32, dim=128, page=128,
             block=16, dtype="bf16", window=0, ragged=True),
        # decode with grouped heads over ragged caches
        dict(name="attend grouped", kind="attend", batch=64, q=1, len=4096, heads=32, kv_heads=8, dim=128, page=128,
             block=32, dtype="bf16", window=0, ragged=True),
        # two long documents, one token each: the cache axis is what there is to split
        dict(name="attend long", kind="attend", batch=2, q=1, len=131071, heads=32, kv_heads=8, dim=128, page=128,
             block=128, dtype="bf16", window=0, ragged=False),
        # a chunk of prompt over what is cached already
        dict(name="attend chunk", kind="attend", batch=4, q=509, len=4096, heads=32, kv_heads=8, dim=128, page=128,
             block=64, dtype="bf16", window=0, ragged=True),
        # the token of a single request
        dict(name="sample one", kind="sample", rows=1, vocab=32000, dtype="f32"),
        # one row for each verify position of the large configuration
        dict(name="sample verify", kind="sample", rows=160, vocab=32000, dtype="f32"),
        # a big batch over a big, odd vocabulary
        dict(name="sample wide", kind="sample", rows=256, vocab=128259, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "append", "attend", "attend", "attend", "sample", "sample"])
    page = rng.choice([16, 32, 64, 128, 128, 128])
    if kind == "plan":
        batch, q = _log_int(rng, 1, 2048), _log_int(rng, 1, 64)
        return dict(kind=kind, batch=batch, q=q, len=_log_int(rng, q, 8192), page=page, ragged=rng.random() < 0.7)
    block = rng.choice([b for b in (16, 32, 64, 128) if b <= page])
    heads, kv_heads = rng.choice([(4, 4), (4, 2), (4, 1), (12, 12), (16, 2), (24, 8), (32, 8), (32, 32)])
    dim = rng.choice([16, 32, 64, 64, 128, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "append":
        batch = _log_int(rng, 1, 64)
        row = kv_heads * dim * (2 if dtype == "bf16" else 4)
        q = _log_int(rng, 1, max(1, min(8192, (8192 * 32 * 128 * 2) // row) // batch))
        return dict(kind=kind, batch=batch, q=q, len=q + _log_int(rng, 1, 2048) - 1, kv_heads=kv_heads, dim=dim,
                    page=page, block=block, dtype=dtype, ragged=rng.random() < 0.7)
    if kind == "attend":
        window = 0 if rng.random() < 0.75 else _log_int(rng, 1, 2048)
        if rng.random() < 0.7:  # decode and verify
            batch, q = _log_int(rng, 1, 64), rng.choice([1, 1, 1, 2, 3, 5, 8, 16])
            most = min(131071, (20 * 3080 * 32 * 128) // (batch * kv_heads * dim))
        else:  # chunks
            batch, q = _log_int(rng, 1, 4), _log_int(rng, 16, 512)
            most = 4096
        most = min(most, 13_000_000_000 // (batch * q * heads * dim))
        return dict(kind=kind, batch=batch, q=q, len=_log_int(rng, q, max(q, most)), heads=heads, kv_heads=kv_heads,
                    dim=dim, page=page, block=block, dtype=dtype, window=window, ragged=rng.random() < 0.7)
    vocab = _log_int(rng, 100, 160000)
    return dict(kind=kind, rows=_log_int(rng, 1, min(512, (256 * 128259) // vocab)), vocab=vocab, dtype=dtype)


# ---------------------------------------------------------------------------
# inputs

def _lengths(c):
    """New tokens and total lengths of the requests: given by the case alone."""
    r = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    q = [r.randint(1, c["q"]) if c["ragged"] else c["q"] for _ in range(c["batch"])]
    q[0] = c["q"]
    ln = [max(n, int(c["len"] * (0.25 + 0.75 * r.random()))) if c["ragged"] else max(n, c["len"]) for n in q]
    ln[0] = max(c["q"], c["len"])
    return q, ln


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _tables(c, q, ln, g):
    """Pages of the requests, in no order, and the batch's row arrays."""
    P = c["page"]
    n = [-(-x // P) for x in ln]
    cols, n_pages = max(n), sum(n) + 3
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    need = _ints(n)
    col = torch.arange(cols, device="cuda")
    first = (torch.cumsum(need, 0) - need).long()
    at = (first[:, None] + col[None]).clamp_(max=n_pages - 1)
    table = torch.where(col[None] < need[:, None], perm[at], torch.full_like(perm[at], -1))
    cu = _ints([0] + q).cumsum(0).to(torch.int32)
    return dict(table=table.contiguous(), n_pages=n_pages, kv_len=_ints(ln), cu_q=cu, tokens=sum(q))


def _cache(c, n_pages, g):
    """A filled cache: codes about as a block's largest value leaves them, scales of a few sizes."""
    H, P, D = c["kv_heads"], c["page"], c["dim"]
    s = {}
    for name in ("k", "v"):
        codes = torch.empty(n_pages, H, P, D, dtype=torch.int8, device="cuda")
        step = max(1, (1 << 26) // (H * P * D))
        for i in range(0, n_pages, step):
            part = codes[i:i + step]
            part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(36.0).round_().clamp_(-127, 127))
        s[name] = codes
        s[name + "_scale"] = torch.rand(n_pages, H, P // c["block"], generator=g, device="cuda").mul_(0.03).add_(0.01)
    return s


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = c["kind"]
    if kind == "sample":
        return _prepare_sample(c, g)
    if kind == "plan":
        return _prepare_plan(c, g)
    q, ln = _lengths(c)
    s = dict(case=c, kind=kind, **_tables(c, q, ln, g))
    s.update(_cache(c, s["n_pages"], g))
    dt, T, D, H = DTYPES[c["dtype"]], s["tokens"], c["dim"], c["kv_heads"]
    heads = c.get("heads", H)
    # rows as a fused q/k/v projection leaves them
    qkv = torch.randn(T, (heads + 2 * H) * D, generator=g, device="cuda").to(dt)
    s["q"] = qkv[:, :heads * D].view(T, heads, D)
    s["new_k"] = qkv[:, heads * D:(heads + H) * D].view(T, H, D)
    s["new_v"] = qkv[:, (heads + H) * D:].view(T, H, D)
    if kind == "append":
        # the rows that a reader of the changed blocks wants: from the first changed block's start to the end
        rows = []
        P, t = c["page"], c["block"]
        table = s["table"].tolist()
        for b in range(c["batch"]):
            for pos in range((ln[b] - q[b]) // t * t, ln[b]):
                rows.append(table[b][pos // P] * P + pos % P)
        s["rows"] = torch.tensor(rows, dtype=torch.int64, device="cuda")
        s["out_k"] = torch.empty(len(rows), H, D, dtype=dt, device="cuda")
        s["out_v"] = torch.empty(len(rows), H, D, dtype=dt, device="cuda")
    else:
        s["max_q"] = max(q)
        s["scale"] = 1.0 / math.sqrt(D)
        s["out"] = torch.empty(T, heads, D, dtype=dt, device="cuda")
        s["lse"] = torch.empty(T, heads, dtype=torch.float32, device="cuda")
    if own:  # what a program keeps from step to step: the handle and the records of its own buffers
        sd = _package()
        s["handle"] = _handle(sd, heads, H, D, c["page"], c["block"], c["batch"])
        s["layer"] = sd.KV8Layer(s["k"], s["v"], s["k_scale"], s["v_scale"])
        s["batch"] = sd.KV8Batch(table=s["table"], kv_len=s["kv_len"], cu_q=s["cu_q"])
    return s


def _prepare_plan(c, g):
    P, B = c["page"], c["batch"]
    q, ln = _lengths(c)
    cols = -(-max(ln) // P) + 1
    rand = torch.rand(4, B, generator=g, device="cuda")
    q_len, most = _ints(q), _ints(ln)
    keep = ((most - q_len) * rand[0].sqrt()).to(torch.int32)
    keep = torch.where(rand[1] < 0.03, torch.zeros_like(keep), keep)  # a slot whose request ended: a new one starts
    held = keep + (rand[2] * 2 * c["q"]).to(torch.int32)
    held = torch.where(rand[1] < 0.03, (most * rand[3]).to(torch.int32), held).clamp_(max=cols * P)
    have = (held + P - 1) // P
    n_pages = B * cols + 7
    perm = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    col = torch.arange(cols, device="cuda")
    table = torch.where(col[None] < have[:, None], perm[:B * cols].view(B, cols), torch.full((B, cols), -1, dtype=torch.int32, device="cuda"))
    free_mask = torch.ones(n_pages, dtype=torch.int64, device="cuda")
    free_mask[:B * cols] = (col[None] >= have[:, None]).flatten().long()
    order = torch.argsort(free_mask, descending=True, stable=True)
    count = free_mask.sum()
    head = (rand[0, 0] * n_pages).long()
    ring = torch.empty(n_pages, dtype=torch.int32, device="cuda")
    ring[(head + torch.arange(n_pages, device="cuda")) % n_pages] = perm[order]
    T = sum(q)
    i32 = dict(dtype=torch.int32, device="cuda")
    s = dict(case=c, kind="plan", held=held, keep=keep, q_len=q_len, table=table.contiguous(), ring=ring,
             ring_state=torch.stack([head, count]).to(torch.int32), ring_out=torch.empty(2, **i32), tokens=T,
             kv_len=torch.empty(B, **i32), cu_q=torch.empty(B + 1, **i32), tok_req=torch.empty(T, **i32),
             tok_pos=torch.empty(T, **i32), slots=torch.empty(T, dtype=torch.int64, device="cuda"),
             status=torch.empty(1, **i32))
    if own:
        sd = _package()
        s["handle"] = _handle(sd, 1, 1, 64, P, P, B)
        s["batch"] = sd.KV8Batch(table=s["table"], kv_len=s["kv_len"], cu_q=s["cu_q"], tok_req=s["tok_req"],
                                 tok_pos=s["tok_pos"], slots=s["slots"], status=s["status"])
    return s


def _prepare_sample(c, g):
    B, V = c["rows"], c["vocab"]
    dt = DTYPES[c["dtype"]]
    # logits of a trained head: a wide bulk, a few likely tokens; some ids never allowed
    logits = torch.randn(B, V, generator=g, device="cuda").mul_(2.5)
    at = torch.randint(0, V, (B, 16), generator=g, device="cuda")
    logits.scatter_add_(1, at, torch.rand(B, 16, generator=g, device="cuda").mul_(14.0))
    logits = torch.where(torch.rand(1, V, generator=g, device="cuda") < 0.01, -math.inf, logits).to(dt)
    r = torch.rand(5, B, generator=g, device="cuda")
    f = dict(dtype=torch.float32, device="cuda")
    return dict(case=c, kind="sample", logits=logits,
                temperature=torch.where(r[0] < 0.1, 0.0, 0.4 + r[0]).to(**f),
                top_k=torch.where(r[1] < 0.4, 0.0, 1 + (r[1] * 200).floor()).to(torch.int32),
                top_p=torch.where(r[2] < 0.3, 1.0, 0.5 + 0.5 * r[2]).to(**f),
                min_p=torch.where(r[3] < 0.5, 0.0, 0.1 * r[3]).to(**f),
                u=torch.rand(B, generator=g, device="cuda"),
                tokens=torch.empty(B, dtype=torch.int32, device="cuda"), probs=torch.empty(B, **f))


# ---------------------------------------------------------------------------
# the framework's operators

_handles = {}


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "neural-network_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import specdec_b200

    return specdec_b200


def _handle(sd, heads, kv_heads, dim, page, block, batch):
    key = (heads, kv_heads, dim, page, block, batch)
    if key not in _handles:
        _handles[key] = sd.KV8(heads, kv_heads, dim, page_tokens=page, block_tokens=block, max_batch=batch)
    return _handles[key]


def run(state):
    s = state
    if s["kind"] == "plan":
        if own:
            s["handle"].plan(s["batch"], s["held"], s["keep"], s["q_len"], s["ring"], s["ring_state"], s["ring_out"])
        else:
            _plan(s)
        return {n: s[n] for n in ("table", "ring", "ring_out", "kv_len", "cu_q", "tok_req", "tok_pos", "slots",
                                  "status")}
    if s["kind"] == "append":
        if own:
            s["handle"].append(s["layer"], s["batch"], s["new_k"], s["new_v"])
            s["handle"].gather(s["layer"], s["rows"], s["out_k"], s["out_v"])
            return {"k": s["out_k"], "v": s["out_v"]}
        out = {}
        for name in ("k", "v"):
            _append(s, s[name], s[name + "_scale"], s["new_" + name])
            out[name] = _gather(s, s[name], s[name + "_scale"]).to(s["new_" + name].dtype)
        return out
    if s["kind"] == "attend":
        if own:
            s["handle"].attend(s["layer"], s["batch"], s["q"], s["out"], lse=s["lse"], max_q=s["max_q"],
                               scale=s["scale"], window=s["case"]["window"])
            return {"out": s["out"], "lse": s["lse"]}
        return _attend(s)
    if own:
        _package().sample(s["logits"], s["u"], s["tokens"], s["probs"], temperature=s["temperature"], top_k=s["top_k"],
                          top_p=s["top_p"], min_p=s["min_p"])
        return {"token": s["tokens"], "prob": s["probs"]}
    return _sample(s)


# ---------------------------------------------------------------------------
# plain forms

def _plan(s):
    P, table, ring, T = s["case"]["page"], s["table"], s["ring"], s["tokens"]
    B, cols = table.shape
    cap = ring.numel()
    held, keep, q = s["held"].long(), s["keep"].long(), s["q_len"].long()
    ring_head, count = s["ring_state"][0].long(), s["ring_state"][1].long()
    length = keep + q
    have, need = (held + P - 1) // P, (length + P - 1) // P
    take, give = (need - have).clamp(min=0), (have - need).clamp(min=0)
    bad = (held < 0) | (keep < 0) | (keep > held) | (q < 0) | (length > cols * P) | (held > cols * P)
    status = bad.any() * 2 + (q.sum() > T) * 4 + (take.sum() > count) * 1
    fine = status == 0
    col = torch.arange(cols, device=table.device)[None]
    take_at, give_at = torch.cumsum(take, 0) - take, torch.cumsum(give, 0) - give
    taken = (col >= have[:, None]) & (col < need[:, None]) & fine
    src = (ring_head + take_at[:, None] + col - have[:, None]) % cap
    given = (col >= need[:, None]) & (col < have[:, None]) & fine
    dst = torch.where(given, (ring_head + count + give_at[:, None] + col - need[:, None]) % cap, cap)
    new_table = torch.where(taken, ring[src], table)
    more = torch.cat([ring, ring[:1]]).scatter(0, dst.flatten(), table.flatten())
    table.copy_(new_table)
    ring.copy_(more[:cap])
    q = torch.where(fine, q, 0)
    s["kv_len"].copy_(torch.where(fine, length, held))
    ends = torch.cumsum(q, 0)
    s["cu_q"].copy_(torch.cat([torch.zeros_like(ends[:1]), ends]))
    moved = torch.stack([ring_head + take.sum(), count - take.sum() + give.sum()])
    moved[0] %= cap
    s["ring_out"].copy_(torch.where(fine, moved, s["ring_state"].long()))
    t = torch.arange(T, device=table.device)
    live = t < ends[-1]
    req = torch.searchsorted(ends, t, right=True).clamp(max=B - 1)
    pos = keep[req] + t - (ends - q)[req]
    page = table[req, (pos // P).clamp(0, cols - 1)].long()
    s["tok_req"].copy_(torch.where(live, req, -1))
    s["tok_pos"].copy_(torch.where(live, pos, -1))
    s["slots"].copy_(torch.where(live, page * P + pos % P, -1))
    s["status"].copy_(status)


def _append(s, codes, scales, x):
    c = s["case"]
    P, t, D = c["page"], c["block"], c["dim"]
    n_pages, H = codes.shape[:2]
    nb = P // t
    cu, ln = s["cu_q"].long(), s["kv_len"].long()
    q = cu[1:] - cu[:-1]
    tok = torch.arange(x.shape[0], device=x.device)
    req = torch.searchsorted(cu[1:], tok, right=True)
    start = ln - q
    pos = start[req] + tok - cu[req]
    page = s["table"][req, pos // P].long()
    blk = page * nb + pos % P // t  # [T]
    x = x.float()
    a = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)  # [T, H]
    high = torch.zeros(n_pages * nb, H, device=x.device).scatter_reduce(0, blk[:, None].expand(-1, H), a, "amax")
    flat = scales.permute(0, 2, 1).reshape(n_pages * nb, H)
    older = (pos // t * t < start[req])[:, None]
    old = torch.where(older, flat[blk], 0.0)  # [T, H]
    new = torch.maximum(old, high[blk] / 127.0)
    new = torch.where(new < 2.0 ** -126, 0.0, new)
    # rows that a first block of a request held before
    first = start // t * t
    at = first[:, None] + torch.arange(t, device=x.device)[None]  # [B, t]
    is_old = (at < start[:, None]) & (q > 0)[:, None]
    page0 = s["table"].long().gather(1, (at // P).clamp(max=s["table"].shape[1] - 1)).clamp(min=0)
    f = cu[:-1].clamp(max=x.shape[0] - 1)
    factor = torch.where(new[f] > old[f], old[f] / new[f], 1.0)  # [B, H]
    was = codes[page0, :, at % P]  # [B, t, H, D]
    now = torch.round(was.float() * factor[:, None, :, None]).to(torch.int8)
    codes[page0, :, at % P] = torch.where(is_old[:, :, None, None], now, was)
    # the new rows and the scales
    inv = torch.where(new > 0, 1.0 / new, 0.0)
    code = torch.round(x * inv[:, :, None]).nan_to_num(0.0).clamp(-127, 127)
    code = torch.where(new[:, :, None] > 0, code, 0.0)
    codes[page, :, pos % P] = code.to(torch.int8)
    scales[page, :, pos % P // t] = new


def _gather(s, codes, scales):
    P, t = s["case"]["page"], s["case"]["block"]
    page, off = s["rows"] // P, s["rows"] % P
    return codes[page, :, off].float() * scales[page, :, off // t][:, :, None]


def _attend(s):
    c, table = s["case"], s["table"]
    P, t, D, H = c["page"], c["block"], c["dim"], c["kv_heads"]
    B, cols = table.shape
    T, heads = s["q"].shape[:2]
    G, L = heads // H, cols * P
    cu, ln = s["cu_q"].long(), s["kv_len"].long()
    q_len = cu[1:] - cu[:-1]
    i = torch.arange(s["max_q"], device=table.device)
    at = (cu[:-1, None] + i[None]).clamp(max=T - 1)  # [B, Q]
    q = s["q"][at].float().view(B, -1, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, -1, D)
    page = table.long().clamp(min=0)

    def rows(codes, scales):
        x = codes[page].float().view(B, cols, H, P // t, t, D) * scales[page].view(B, cols, H, P // t, 1, 1)
        return x.view(B, cols, H, P, D).permute(0, 2, 1, 3, 4).reshape(B, H, L, D)

    score = torch.matmul(q, rows(s["k"], s["k_scale"]).transpose(2, 3)).mul_(s["scale"]).view(B, H, -1, G, L)
    j = torch.arange(L, device=table.device)
    own_pos = ln[:, None] - q_len[:, None] + i[None]  # [B, Q]
    seen = (j <= own_pos[:, :, None]) & (j < ln[:, None, None])
    if c["window"]:
        seen &= j > own_pos[:, :, None] - c["window"]
    score.masked_fill_(~seen[:, None, :, None], -math.inf)
    high = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(high == -math.inf, 0.0, high)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, H, -1, L), rows(s["v"], s["v_scale"])).view(B, H, -1, G, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3, 4).reshape(B, -1, heads, D)
    lse = (high + total.log()).permute(0, 2, 1, 3, 4).reshape(B, -1, heads)
    tok = torch.arange(T, device=table.device)
    req = torch.searchsorted(cu[1:], tok, right=True)
    return {"out": o[req, tok - cu[req]].to(s["q"].dtype), "lse": lse[req, tok - cu[req]]}


def _sample(s):
    x = s["logits"].float()
    B, V = x.shape
    x = torch.where(torch.isnan(x), -math.inf, x)
    T = s["temperature"][:, None]
    z = torch.where(T > 0, x / torch.where(T > 0, T, 1.0), x)
    high = z.amax(-1, keepdim=True)
    e = torch.where(z == high, 1.0, torch.exp(z - high))
    e = torch.where(high == -math.inf, 0.0, e)
    w = (e * 2.0 ** 31).long()
    zs, order = torch.sort(z, dim=-1, descending=True, stable=True)
    ws, es = w.gather(1, order), e.gather(1, order)
    rank = torch.arange(V, device=x.device)[None]
    k = s["top_k"].long()[:, None]
    ws = torch.where((k <= 0) | (rank < k), ws, 0)
    run_sum = ws.cumsum(-1)
    p24 = torch.round(s["top_p"].clamp(0.0, 1.0) * 2.0 ** 24).long()[:, None]
    mass = run_sum[:, -1:]
    most = (p24 * (mass >> 24) + (p24 * (mass & 0xFFFFFF) >> 24)).clamp(min=1)
    ws = torch.where((s["top_p"][:, None] >= 1) | (run_sum - ws < most), ws, 0)
    ws = torch.where(es >= s["min_p"].clamp(max=1.0)[:, None], ws, 0)
    kept = torch.zeros_like(w).scatter(1, order, ws)
    run_sum = kept.cumsum(-1)
    total = run_sum[:, -1]
    u24 = (s["u"] * 2.0 ** 24).long().clamp(0, (1 << 24) - 1)
    target = u24 * (total >> 24) + (u24 * (total & 0xFFFFFF) >> 24)
    token = (run_sum <= target[:, None]).sum(-1).clamp(max=V - 1)
    prob = kept.gather(1, token[:, None])[:, 0].float() / total.float()
    greedy = ~(s["temperature"] > 0)
    token = torch.where(greedy, (z == high).int().argmax(-1), token)
    prob = torch.where(greedy, 1.0, prob)
    empty = high[:, 0] == -math.inf
    return {"token": torch.where(empty, -1, token).to(torch.int32), "prob": torch.where(empty, 0.0, prob)}


# ---------------------------------------------------------------------------
# 64 bits

def exact(case, seed):
    if case["kind"] == "plan":
        return None
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](s)


def _exact_append(s):
    c = s["case"]
    P, t = c["page"], c["block"]
    table, cu, ln = s["table"].tolist(), s["cu_q"].tolist(), s["kv_len"].tolist()
    out = {}
    for name in ("k", "v"):
        parts = []
        for b in range(c["batch"]):
            start, end = ln[b] - (cu[b + 1] - cu[b]), ln[b]
            lead = start % t
            x = s["new_" + name][cu[b]:cu[b + 1]].double()
            n = lead + end - start
            whole = torch.zeros((n + t - 1) // t * t, *x.shape[1:], dtype=torch.float64, device=x.device)
            whole[lead:n] = x
            blocks = whole.view(-1, t, *x.shape[1:])
            new = blocks.abs().amax((1, 3)) / 127  # [blocks, H]
            if lead:  # rows that were there, with the scale they had
                page, off = table[b][start // P], start % P // t * t
                old = s[name + "_scale"][page, :, off // t].double()
                was = s[name][page, :, off:off + lead].double().permute(1, 0, 2)
                grown = torch.maximum(new[0], old)
                factor = torch.where(grown > old, old / grown, 1.0)
                blocks[0, :lead] = torch.round(was * factor[None, :, None]) * grown[None, :, None]
                new[0] = grown
            step = new[:, None, :, None].clamp(min=1e-300)
            codes = torch.round(blocks / step).clamp(-127, 127)
            parts.append((codes * step).view(-1, *x.shape[1:])[:n])
        out[name] = torch.cat(parts)
    return out


def _exact_attend(s):
    c = s["case"]
    P, t, D, H = c["page"], c["block"], c["dim"], c["kv_heads"]
    heads = s["q"].shape[1]
    G = heads // H
    table, cu, ln = s["table"].tolist(), s["cu_q"].tolist(), s["kv_len"].tolist()
    outs, lses = [], []
    for b in range(c["batch"]):
        n, L = cu[b + 1] - cu[b], ln[b]
        pages = s["table"][b, :-(-L // P)].long()

        def rows(codes, scales, h):
            x = codes[pages, h].double() * scales[pages, h].double().repeat_interleave(t, 1)[:, :, None]
            return x.reshape(-1, D)[:L]

        pos = torch.arange(L - n, L, device="cuda")[:, None]
        j = torch.arange(L, device="cuda")[None]
        seen = j <= pos
        if c["window"]:
            seen = seen & (j > pos - c["window"])
        o = torch.empty(n, heads, D, dtype=torch.float64, device="cuda")
        lse = torch.empty(n, heads, dtype=torch.float64, device="cuda")
        for h in range(H):
            k, v = rows(s["k"], s["k_scale"], h), rows(s["v"], s["v_scale"], h)
            for i in range(h * G, (h + 1) * G):
                score = (s["q"][cu[b]:cu[b + 1], i].double() @ k.T / math.sqrt(D)).masked_fill(~seen, -math.inf)
                lse[:, i] = torch.logsumexp(score, -1)
                o[:, i] = torch.softmax(score, -1) @ v
        outs.append(o)
        lses.append(lse)
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}


def _exact_sample(s):
    prob = []
    for b in range(s["case"]["rows"]):
        x = s["logits"][b].float()
        T, u = s["temperature"][b].item(), s["u"][b].item()
        if x.max().item() == -math.inf:
            prob.append(0.0)
            continue
        if T <= 0:
            prob.append(1.0)
            continue
        z = (x / s["temperature"][b]).double()  # the scaled logit is defined in 32 bits
        d = (z - z.max()).float().double()
        w = torch.floor(torch.exp(d) * 2.0 ** 31)
        k, top_p, min_p = s["top_k"][b].item(), s["top_p"][b].item(), s["min_p"][b].item()
        by = torch.argsort(d, descending=True, stable=True)
        if k > 0:
            by = by[:k]
        if top_p < 1:
            run_sum = torch.cumsum(w[by], 0)
            by = by[(run_sum - w[by]) < max(1.0, math.floor(round(top_p * 2 ** 24) * run_sum[-1].item() / 2 ** 24))]
        by = by[torch.exp(d[by]) >= min(1.0, min_p)]
        kept = torch.zeros_like(w)
        kept[by] = w[by]
        run_sum = torch.cumsum(kept, 0)
        total = run_sum[-1].item()
        target = math.floor(int(u * 2 ** 24) * total / 2 ** 24)
        token = int(torch.searchsorted(run_sum, torch.tensor(float(target), dtype=torch.float64, device="cuda"), right=True))
        prob.append((kept[token] / total).item())
    return {"token": None, "prob": torch.tensor(prob, dtype=torch.float64, device="cuda")}


# ---------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    c = case
    if c["kind"] == "sample":
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": c["rows"] * (c["vocab"] * size + 28), "flops": 4 * c["rows"] * c["vocab"]}
    q, ln = _lengths(c)
    T = sum(q)
    if c["kind"] == "plan":
        return {"bytes": T * 16 + c["batch"] * 20 + T / c["page"] * 8, "flops": 0}
    H, D = c["kv_heads"], c["dim"]
    size = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "append":
        t = c["block"]
        rows = sum(n - (n - m) // t * t for m, n in zip(q, ln))
        blocks = sum(-(-n // t) - (n - m) // t for m, n in zip(q, ln))
        return {"bytes": 2 * H * (T * D * (size + 1) + rows * D * (1 + size) + blocks * 8), "flops": 8 * T * H * D}
    heads, w = c["heads"], c["window"]
    seen = sum(n if not w else min(n, w + m - 1) for m, n in zip(q, ln))
    pairs = sum(sum(min(p + 1, w) if w else p + 1 for p in range(n - m, n)) for m, n in zip(q, ln))
    return {"bytes": seen * H * (2 * D + 8 / c["block"]) + T * heads * (2 * D * size + 4), "flops": 4 * D * heads * pairs}
