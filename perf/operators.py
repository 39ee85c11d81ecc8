"""The operators of a decoding step whose lengths live on the device, as a program that verifies drafted tokens uses them:

* `tables`: pages handed out and block tables, positions and cache slots built from the requests' lengths;
* `write`: the step's keys and values written to their slots of the paged cache;
* `attend`: attention of every request's few new tokens (or a chunk of hundreds) over its pages;
* `verify`: drafted tokens accepted or replaced against the target's probabilities, from given random numbers.

Each case is one call.  Lengths are spread evenly over the range that a case names, in scattered order; everything else is drawn
from the seed.  Cache slots that no token has written hold NaN, as a fresh pool of the engine does.
"""
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
VOCAB = 128256                      # of the Llama shapes that bench.py runs
FIXED = 2.0 ** 48                   # verification adds up weights in units of 2^-48

# Head layouts of the shapes that bench.py runs.
LLAMA_8B = dict(heads=32, kv_heads=8, head_dim=128)
LLAMA_3B = dict(heads=24, kv_heads=8, head_dim=128)
LLAMA_1B = dict(heads=32, kv_heads=8, head_dim=64)
WIDTH_2048 = dict(heads=16, kv_heads=4, head_dim=128)


def _attend(dtype, requests, cached, new, layout, page=16, window=0):
    return dict(op="attend", dtype=dtype, requests=requests, cached_lo=cached[0], cached_hi=cached[1], new_lo=new[0], new_hi=new[1],
                page=page, window=window, **layout)


def _verify(requests, drafts, vocab, draft_probs, ragged):
    return dict(op="verify", requests=requests, drafts=drafts, vocab=vocab, draft_probs=draft_probs, ragged=ragged)


def _tables(requests, cached, new, page, width, short, spare):
    return dict(op="tables", requests=requests, cached_lo=cached[0], cached_hi=cached[1], new_lo=new[0], new_hi=new[1], page=page,
                width=width, short=short, spare=spare)


def _write(tokens, rows, cache, kv_heads, head_dim, page, fused):
    return dict(op="write", tokens=tokens, rows=rows, cache=cache, kv_heads=kv_heads, head_dim=head_dim, page=page, fused=fused)


def listed():
    return [
        # one user's drafted tokens behind a short conversation: latency
        dict(_attend("bf16", 1, (1000, 1000), (5, 5), LLAMA_8B), name="attend_one"),
        # eight requests that verify four drafted tokens each
        dict(_attend("bf16", 8, (500, 2000), (5, 5), LLAMA_8B), name="attend_drafts"),
        # a full serving batch of the small model, drafts of unequal length
        dict(_attend("bf16", 56, (700, 4500), (1, 8), LLAMA_1B), name="attend_batch_head64"),
        # few requests with a long context each: the keys have to be shared out
        dict(_attend("bf16", 4, (30000, 33000), (6, 9), LLAMA_3B), name="attend_long"),
        # chunks of prompts behind cached ones, bound by the products
        dict(_attend("bf16", 4, (6000, 9000), (301, 513), LLAMA_8B), name="attend_chunks"),
        # the 32-bit path, which results are checked with
        dict(_attend("fp32", 8, (500, 3000), (3, 7), WIDTH_2048), name="attend_fp32"),
        # one user, four drafted tokens: latency
        dict(_verify(1, 4, VOCAB, True, False), name="verify_one"),
        # a serving batch whose requests drafted one to five tokens
        dict(_verify(64, 5, VOCAB, True, True), name="verify_batch"),
        # the tables of a small verification step
        dict(_tables(8, (500, 2000), (5, 5), 16, 256, False, 24), name="tables_drafts"),
        # the tables of a large step: long contexts, portions of prompts beside drafted tokens, pages run out before the last
        dict(_tables(512, (100, 32000), (1, 60), 16, 2048, True, 300), name="tables_batch"),
        # keys and values of a verification step, out of a fused float32 projection
        dict(_write(40, "fp32", "bf16", 8, 128, 16, True), name="write_drafts"),
        # keys and values of a step of prompt portions
        dict(_write(8191, "bf16", "bf16", 8, 128, 16, True), name="write_prompts"),
    ]


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def _range(rng, lo, hi):
    a, b = _log(rng, lo, hi), _log(rng, lo, hi)
    return min(a, b), max(a, b)


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "verify", "tables", "write"])
    if op == "attend":
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        layout = rng.choice([LLAMA_8B, LLAMA_3B, LLAMA_1B, WIDTH_2048, dict(heads=16, kv_heads=16, head_dim=64),
                             dict(heads=8, kv_heads=1, head_dim=128)])
        requests, cached, new = _log(rng, 1, 64), _range(rng, 1, 33000), _range(rng, 1, 513 if dtype == "bf16" else 40)
        page, window = rng.choice([8, 16, 16, 32, 64]), rng.choice([0, 0, 0, _log(rng, 16, 5000)])
        while True:
            c = _attend(dtype, requests, cached, new, layout, page, window)
            w, keys = work(c), cached[1] + new[1]
            padded = max(requests * new[1] * keys * layout["heads"] / 1e9, requests * keys * layout["kv_heads"] * layout["head_dim"] / 3e8)
            if w["bytes"] <= 5e8 and w["flops"] <= (2e11 if dtype == "bf16" else 1e10) and padded <= 1:
                return c
            if requests > 1:
                requests = (requests + 1) // 2
            else:
                cached, new = (cached[0] // 2 + 1, cached[1] // 2 + 1), (new[0] // 2 + 1, new[1] // 2 + 1)
    if op == "verify":
        return _verify(_log(rng, 1, 64), rng.randint(1, 5), rng.choice([VOCAB, VOCAB, _log(rng, 500, 128000)]),
                       rng.choice([True, True, False]), rng.choice([True, False]))
    if op == "tables":
        page, cached = rng.choice([8, 16, 16, 32, 64]), _range(rng, 1, 32000)
        requests, new = _log(rng, 1, 512), _range(rng, 1, 60)
        width = (cached[1] + new[1] + page - 1) // page + rng.randint(0, 40)
        return _tables(requests, cached, new, page, width, rng.choice([True, False]), rng.randint(0, 300))
    rows, cache = rng.choice([("fp32", "bf16"), ("bf16", "bf16"), ("fp32", "fp32")])
    return _write(_log(rng, 1, 8000), rows, cache, rng.choice([1, 4, 8]), rng.choice([64, 128]), rng.choice([8, 16, 16, 64]),
                  rng.choice([True, False]))


def _spread(lo, hi, n):
    return [lo + (hi - lo) * ((i * 7919) % n) // max(1, n - 1) for i in range(n)]


def _lengths(c):
    """(tokens cached, tokens brought) of every request."""
    return _spread(c["cached_lo"], c["cached_hi"], c["requests"]), _spread(c["new_lo"], c["new_hi"], c["requests"])[::-1]


def _draft_lengths(c):
    return _spread(1 if c["ragged"] else c["drafts"], c["drafts"], c["requests"])


def _seen(c):
    """(keys that any token of a request sees, (token, key) pairs), each summed over the requests."""
    keys = pairs = 0
    for cached, new in zip(*_lengths(c)):
        w = c["window"] or cached + new
        keys += min(cached + new, w + new - 1)
        pairs += sum(min(cached + i + 1, w) for i in range(new))
    return keys, pairs


def work(c):
    if c["op"] == "attend":
        size = 2 if c["dtype"] == "bf16" else 4
        keys, pairs = _seen(c)
        tokens = sum(_lengths(c)[1])
        return dict(bytes=size * c["head_dim"] * (2 * keys * c["kv_heads"] + 2 * tokens * c["heads"]) + 4 * keys // c["page"],
                    flops=4.0 * pairs * c["heads"] * c["head_dim"])
    if c["op"] == "verify":
        # the target's row behind the last accepted token, and the draft's row where that was a refusal (three in four here)
        rows = c["requests"] * (1 + (0.75 if c["draft_probs"] else 0))
        return dict(bytes=4 * rows * c["vocab"] + 4 * c["requests"] * (5 * c["drafts"] + 5), flops=2 * rows * c["vocab"])
    if c["op"] == "tables":
        cached, new = _lengths(c)
        pages, tokens = sum((n + c["page"] - 1) // c["page"] for n in cached), sum(new) + c["spare"]
        return dict(bytes=4 * (pages + c["requests"] * (c["width"] + 6) + 3 * tokens), flops=tokens + c["requests"])
    a, b = (2 if c[k] == "bf16" else 4 for k in ("rows", "cache"))
    return dict(bytes=2 * c["tokens"] * c["kv_heads"] * c["head_dim"] * (a + b) + 4 * c["tokens"], flops=0)


# ---------------------------------------------------------------------------
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(new):
    return _ints([sum(new[:i]) for i in range(len(new))])


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=g)
    uniform = lambda *s: torch.rand(*s, device=DEV, generator=g)
    s = dict(op=c["op"], err=torch.zeros(1, dtype=torch.int32, device=DEV))
    if c["op"] == "attend":
        dt, (cached, new) = DTYPES[c["dtype"]], _lengths(c)
        H, K, d, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
        held = [(a + b + P - 1) // P for a, b in zip(cached, new)]
        n_pages, width = sum(held) + 5, max(held)
        ids = torch.randperm(n_pages, device=DEV, generator=g).int()
        at = torch.arange(width, device=DEV)[None] + _starts(held)[:, None]
        there = torch.arange(width, device=DEV)[None] < _ints(held)[:, None]
        table = torch.where(there, ids[at.clamp(max=n_pages - 1)], -1).int()
        total = _ints([a + b for a, b in zip(cached, new)])
        filled = torch.zeros(n_pages, P, dtype=torch.bool, device=DEV)
        place = torch.arange(width * P, device=DEV).view(width, P)[None] < total[:, None, None]
        filled[table[there].long()] = place[there]
        pools = [torch.where(filled[:, None, :, None], randn(n_pages, K, P, d), float("nan")).to(dt) for _ in range(2)]
        s.update(q=(1.5 * randn(sum(new), H, d)).to(dt), k_pages=pools[0], v_pages=pools[1], table=table, q_start=_starts(new),
                 q_len=_ints(new), ctx_len=_ints(cached), scale=1 / math.sqrt(d), window=c["window"], new_hi=max(new),
                 keys_hi=max(a + b for a, b in zip(cached, new)))
    elif c["op"] == "verify":
        R, N, V, lens = c["requests"], c["drafts"], c["vocab"], _draft_lengths(c)
        rows = [n + 1 for n in lens]
        logits = 3 * randn(sum(rows), V)
        start = _starts(rows)
        row_of = (start[:, None] + torch.arange(N, device=DEV)).clamp(max=sum(rows) - 1)
        guess = torch.softmax(logits[row_of] + 0.7 * randn(R, N, V), dim=-1)      # the drafts come from a model that is near
        tokens = (guess / torch.empty_like(guess).exponential_(generator=g)).argmax(-1).int()
        s.update(target=torch.softmax(logits, dim=-1), q_start=start, tokens=tokens, lens=_ints(lens),
                 guess=guess if c["draft_probs"] else None, accept=uniform(R, N), pick=uniform(R))
    elif c["op"] == "tables":
        (cached, new), P, W, R = _lengths(c), c["page"], c["width"], c["requests"]
        # one request in three kept a page more than its tokens need, from drafts that were refused
        held = [min(W, (n + P - 1) // P + (1 if i % 3 == 1 else 0)) for i, n in enumerate(cached)]
        need = sum(max(0, (a + b + P - 1) // P - h) for a, b, h in zip(cached, new, held))
        free = max(0, need * 3 // 4 - 1) if c["short"] else need + 7
        n_pages = sum(held) + need + 9
        ids = torch.randperm(n_pages, device=DEV, generator=g).int()
        at = torch.arange(W, device=DEV)[None] + _starts(held)[:, None]
        table = torch.where(torch.arange(W, device=DEV)[None] < _ints(held)[:, None], ids[at.clamp(max=n_pages - 1)], -1).int()
        s.update(cached=_ints(cached), counts=_ints(new), held=_ints(held), table=table, free=ids[sum(held):].clone(),
                 free_count=_ints([free]), page=P, n_pages=n_pages, capacity=sum(new) + c["spare"])
    else:
        T, K, d, P = c["tokens"], c["kv_heads"], c["head_dim"], c["page"]
        n_pages = (T + P - 1) // P + 3
        if c["fused"]:      # the columns of keys and values of a fused projection, four query heads to a key head
            kv = randn(T, 6 * K, d).to(DTYPES[c["rows"]])[:, 4 * K:]
        else:
            kv = randn(T, 2 * K, d).to(DTYPES[c["rows"]])
        slots = torch.randperm(n_pages * P, device=DEV, generator=g)[:T].int()
        slots[uniform(T) < 0.02] = -1                                         # rows of requests that got no page
        pools = [randn(n_pages, K, P, d).to(DTYPES[c["cache"]]) for _ in range(2)]
        s.update(k=kv[:, :K], v=kv[:, K:], slots=slots, k_pages=pools[0], v_pages=pools[1])
    return s


# ---------------------------------------------------------------------------
def run(s):
    return {"attend": _run_attend, "verify": _run_verify, "tables": _run_tables, "write": _run_write}[s["op"]](s)


def _run_attend(s):
    if own:
        from ai_engine_b200.kernels import ops
        return ops.paged_attention_chunks(s["q"], s["k_pages"], s["v_pages"], s["q_start"], s["q_len"], s["ctx_len"], s["table"],
                                          s["scale"], s["window"], s["err"])
    q, table = s["q"], s["table"]
    (T, H, d), (N, K, P, _), R = q.shape, s["k_pages"].shape, table.shape[0]
    i, j = torch.arange(s["new_hi"], device=DEV), torch.arange(s["keys_hi"], device=DEV)
    total = s["ctx_len"] + s["q_len"]
    there = j[None] < total[:, None]                                           # [R, keys]
    page = table[:, j // P].clamp(min=0).long()
    k, v = (torch.where(there[:, :, None, None], t[page, :, j % P], 0).float() for t in (s["k_pages"], s["v_pages"]))
    mine = i[None] < s["q_len"][:, None]                                       # [R, new]
    rows = (s["q_start"][:, None] + i).clamp(max=T - 1)
    qs = q[rows].float().view(R, -1, K, H // K, d).permute(0, 2, 3, 1, 4).reshape(R, K, -1, d)
    scores = torch.matmul(qs, k.permute(0, 2, 3, 1)).view(R, K, H // K, -1, s["keys_hi"]) * s["scale"]
    pos = s["ctx_len"][:, None] + i                                            # [R, new]
    sees = j <= pos[..., None]
    if s["window"]:
        sees = sees & (j > pos[..., None] - s["window"])
    scores = scores.masked_fill_(~(sees & there[:, None])[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores.sub_(torch.where(top == -math.inf, 0, top)))
    mass = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(R, K, -1, s["keys_hi"]), v.transpose(1, 2)).view(R, K, H // K, -1, d)
    o = torch.where(mass > 0, o / mass, 0).permute(0, 3, 1, 2, 4).reshape(R, -1, H, d)
    out = torch.empty_like(q)
    out[rows[mine]] = o[mine].to(q.dtype)
    return out


def _run_verify(s):
    if own:
        from ai_engine_b200.sampling import verify_drafts
        return verify_drafts(s["target"], s["q_start"], s["tokens"], s["lens"], s["guess"], s["accept"], s["pick"], s["err"])
    target, tokens, lens, guess = s["target"], s["tokens"], s["lens"], s["guess"]
    (R, N), V = tokens.shape, target.shape[1]
    r, i = torch.arange(R, device=DEV), torch.arange(N, device=DEV)
    rows = (s["q_start"][:, None] + i).clamp(max=target.shape[0] - 1)
    p = target[rows, tokens.long()].double()
    q = guess[r[:, None], i, tokens.long()].double() if guess is not None else torch.ones_like(p)
    kept = (s["accept"].double() * q < p) & (i < lens[:, None])
    accepted = kept.int().cumprod(-1).sum(-1)
    last = target[s["q_start"] + accepted]
    at = accepted.clamp(max=N - 1)
    if guess is not None:
        minus = guess[r, at]
    else:
        minus = torch.zeros_like(last).scatter_(1, tokens[r, at][:, None].long(), math.inf)
    minus = torch.where((accepted < lens)[:, None], minus, 0)
    weight = lambda w: (w.clamp(0, 1) * FIXED).double().round().long()
    left = weight(last - minus)
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, weight(last))
    mass = left.sum(-1)
    goal = torch.minimum((s["pick"].double() * mass.double()).floor().long(), mass - 1)
    drawn = (left.cumsum(-1) <= goal[:, None]).sum(-1).int()
    both = torch.cat([tokens, tokens[:, :1]], dim=1)
    place = torch.arange(N + 1, device=DEV)
    out = torch.where(place < accepted[:, None], both, torch.where(place == accepted[:, None], drawn[:, None], -1)).int()
    return out, (accepted + 1).int()


def _run_tables(s):
    if own:
        from ai_engine_b200.cache import step_tables
        t = step_tables(s["cached"], s["counts"], s["held"], s["table"], s["free"], s["free_count"], s["page"], s["n_pages"],
                        s["capacity"], s["err"])
        return t.tables, t.held, t.free_count, t.q_start, t.q_len, t.positions, t.token_req, t.slots
    cached, counts, held, table, P = (s[k] for k in ("cached", "counts", "held", "table", "page"))
    R, W = table.shape
    want = torch.maximum((cached + counts + P - 1) // P, held)
    need = want - held
    upto = need.cumsum(0)
    granted = (need == 0) | (upto <= s["free_count"])
    first = s["free_count"] - 1 - (upto - need)                                # the free list is taken from its end
    now = torch.where(granted, want, held)
    w = torch.arange(W, device=DEV)[None]
    fresh = (w >= held[:, None]) & (w < now[:, None])
    place = (first[:, None] - (w - held[:, None])).clamp(0, s["free"].shape[0] - 1)
    tables = torch.where(w < held[:, None], table, torch.where(fresh, s["free"][place], -1)).int()
    start = counts.cumsum(0) - counts
    t = torch.arange(s["capacity"], device=DEV)
    req = torch.searchsorted(counts.cumsum(0), t, right=True)
    real, at = req < R, req.clamp(max=R - 1)
    pos = cached[at] + t - start[at]
    page = tables[at, (pos // P).clamp(max=W - 1)]
    slots = torch.where(real & granted[at], page * P + pos % P, -1).int()
    left = s["free_count"] - torch.where(granted, need, 0).sum()
    return (tables, now.int(), left.int(), start.int(), torch.where(granted, counts, 0).int(), torch.where(real, pos, -1).int(),
            torch.where(real, req, -1).int(), slots)


def _run_write(s):
    k_pages, v_pages, slots = s["k_pages"], s["v_pages"], s["slots"]
    if own:
        from ai_engine_b200.kernels import ops
        ops.write_kv_slots(s["k"], s["v"], k_pages, v_pages, slots, s["err"])
        return k_pages, v_pages
    P, there = k_pages.shape[2], slots >= 0
    to = slots[there].long()
    k_pages[to // P, :, to % P] = s["k"][there].float().to(k_pages.dtype)
    v_pages[to // P, :, to % P] = s["v"][there].float().to(v_pages.dtype)
    return k_pages, v_pages


# ---------------------------------------------------------------------------
def exact(c, seed):
    s = prepare(c, seed)
    return {"attend": _exact_attend, "verify": _exact_verify, "tables": _exact_tables, "write": _exact_write}[c["op"]](s)


def _exact_attend(s):
    """One request and key head at a time, softmax(q k^T) v in 64 bits."""
    H, K = s["q"].shape[1], s["k_pages"].shape[1]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for r, (a, n, c) in enumerate(zip(s["q_start"].tolist(), s["q_len"].tolist(), s["ctx_len"].tolist())):
        P = s["k_pages"].shape[2]
        pages = s["table"][r, :(c + n + P - 1) // P].long()
        pos = torch.arange(c, c + n, device=DEV)[:, None]
        key = torch.arange(c + n, device=DEV)[None]
        hidden = key > pos
        if s["window"]:
            hidden |= key <= pos - s["window"]
        for kh in range(K):
            k, v = (t[pages, kh].reshape(-1, t.shape[-1])[:c + n].double() for t in (s["k_pages"], s["v_pages"]))
            for h in range(kh * (H // K), (kh + 1) * (H // K)):
                x = (s["q"][a:a + n, h].double() @ k.T) * s["scale"]
                out[a:a + n, h] = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1) @ v
    return out


def _exact_verify(s):
    """Request by request, token by token."""
    target, guess = s["target"], s["guess"]
    R, N = s["tokens"].shape
    out, emitted = torch.full((R, N + 1), -1, dtype=torch.int32), []
    for r, (start, n, ids, us) in enumerate(zip(s["q_start"].tolist(), s["lens"].tolist(), s["tokens"].tolist(), s["accept"].tolist())):
        k, rest = 0, None
        while k < n and rest is None:
            p = target[start + k].double()
            q = guess[r, k].double() if guess is not None else torch.zeros_like(p).index_fill_(0, torch.tensor([ids[k]], device=DEV), 1)
            if us[k] * q[ids[k]].item() < p[ids[k]].item():
                out[r, k] = ids[k]
                k += 1
            else:
                rest = (p - q).clamp(min=0)
        upto = (target[start + n].double() if rest is None else rest).cumsum(0)
        out[r, k] = int((upto <= s["pick"][r].double() * upto[-1]).sum())
        emitted.append(k + 1)
    return out.to(DEV), _ints(emitted)


def _exact_tables(s):
    """Request by request, page by page."""
    cached, counts, held, free = (s[k].tolist() for k in ("cached", "counts", "held", "free"))
    P, W, table, left = s["page"], s["table"].shape[1], s["table"].tolist(), int(s["free_count"])
    stack, at, waiting = free[:left], 0, False
    q_start, q_len, positions, token_req, slots = [], [], [], [], []
    for r, (c, n) in enumerate(zip(cached, counts)):
        short = -(-(c + n) // P) - held[r]
        refused = short > 0 and (waiting or short > len(stack))
        waiting = waiting or refused                    # who comes later and wants pages waits too
        if not refused:
            for _ in range(short):
                table[r][held[r]] = stack.pop()
                held[r] += 1
        q_start.append(at)
        q_len.append(0 if refused else n)
        for pos in range(c, c + n):
            positions.append(pos)
            token_req.append(r)
            slots.append(-1 if refused else table[r][pos // P] * P + pos % P)
        at += n
    pad = [-1] * (s["capacity"] - at)
    return tuple(map(_ints, (table, held, [len(stack)], q_start, q_len, positions + pad, token_req + pad, slots + pad)))


def _exact_write(s):
    """Pools whose named rows hold the given keys and values."""
    done = []
    for rows, pages in ((s["k"], s["k_pages"]), (s["v"], s["v_pages"])):
        flat = pages.double().transpose(1, 2).reshape(-1, *rows.shape[1:])
        flat[s["slots"][s["slots"] >= 0].long()] = rows[s["slots"] >= 0].double()
        done.append(flat.view(pages.shape[0], pages.shape[2], *rows.shape[1:]).transpose(1, 2))
    return tuple(done)
