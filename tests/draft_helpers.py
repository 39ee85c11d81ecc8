"""Plain forms in 64 bits, and batches, for the tests of steps that verify drafted tokens."""
import math

import torch

U = 2.0 ** -24                       # half a step of float32, relative


def paged_batch(cached, new, H, K, d, P, dtype, seed, spare_pages=3, window=0, device="cuda", slack=0):
    """Random queries, pools and tables of requests with `cached` tokens that bring `new` more; pages scattered, slots without a token NaN,
    table entries without one -1, and, with a window, entries that every token's window has passed -1 too.  `slack` rows of q
    belong to nobody."""
    g = torch.Generator().manual_seed(seed)
    pages = [(c + n + P - 1) // P for c, n in zip(cached, new)]
    N, W, R = sum(pages) + spare_pages, max(pages + [1]), len(new)
    ids = torch.randperm(N, generator=g)
    table = torch.full((R, W), -1, dtype=torch.int32)
    k_pages, v_pages = torch.full((N, K, P, d), float("nan")), torch.full((N, K, P, d), float("nan"))
    at, rows = 0, []
    for r, (c, n) in enumerate(zip(cached, new)):
        mine = ids[at:at + pages[r]]
        at += pages[r]
        table[r, :pages[r]] = mine.int()
        k, v = torch.randn(c + n, K, d, generator=g), torch.randn(c + n, K, d, generator=g)
        k, v = k.to(dtype).float(), v.to(dtype).float()
        rows.append((k, v))
        for j in range(c + n):
            k_pages[mine[j // P], :, j % P] = k[j]
            v_pages[mine[j // P], :, j % P] = v[j]
        if window:
            table[r, :max(0, c - window + 1) // P] = -1
    T = sum(new)
    q = (1.5 * torch.randn(T + slack, H, d, generator=g)).to(dtype)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    start = [sum(new[:i]) for i in range(R)]
    return dict(q=q.to(device), k_pages=k_pages.to(dtype).to(device), v_pages=v_pages.to(dtype).to(device), table=table.to(device),
                q_start=ints(start), q_len=ints(new), ctx_len=ints(cached), rows=rows, cached=list(cached), new=list(new), start=start,
                scale=1 / math.sqrt(d), window=window)


def plain_attention(b, dtype):
    """(o, tolerance) in 64 bits for the rows that requests name.  What may be off, element by element: a score is a sum of d products in
    float32, off by at most 4 sqrt(d) roundings (U each) of |q||k| scale, the most that a partial sum can be, and 4 roundings of itself in
    the exponential; a change of all scores by up to t moves a weighted mean by at most 2 t max|v|; sums over n keys 4 sqrt(n) roundings.
    bfloat16: probabilities (2^-8 of sum p|v|) and the result (2^-8) are rounded once each."""
    q = b["q"].double().cpu()
    T, H, d = q.shape
    K = b["k_pages"].shape[1]
    out, tol = torch.zeros(T, H, d, dtype=torch.float64), torch.zeros(T, H, d, dtype=torch.float64)
    for r, (c, n) in enumerate(zip(b["cached"], b["new"])):
        if n == 0:
            continue
        k, v = (x.double() for x in b["rows"][r])
        pos, key = torch.arange(c, c + n)[:, None], torch.arange(c + n)[None]
        hidden = key > pos
        if b["window"]:
            hidden = hidden | (key <= pos - b["window"])
        for h in range(H):
            kh = h // (H // K)
            qs = q[b["start"][r]:b["start"][r] + n, h]
            x = (qs @ k[:, kh].T * b["scale"]).masked_fill(hidden, -math.inf)
            p = torch.softmax(x, dim=-1)
            o, size = p @ v[:, kh], p @ v[:, kh].abs()
            most = qs.norm(dim=-1).max() * k[:, kh].norm(dim=-1).max() * abs(b["scale"])      # a size, whatever the sign
            t = U * (4 * math.sqrt(d) + 4) * most
            e = 2 * t * v[:, kh].abs().max() + 4 * U * math.sqrt(c + n) * v[:, kh].abs().max()
            if dtype == torch.bfloat16:
                e = e + 2.0 ** -8 * (size + o.abs() + e)
            else:
                e = e + U * o.abs()
            out[b["start"][r]:b["start"][r] + n, h], tol[b["start"][r]:b["start"][r] + n, h] = o, e
    return out, tol


def plain_tables(cached, counts, held, table, free, free_count, P, max_tokens):
    """Request by request, page by page; the same order of outputs as StepTables."""
    table, held, stack, at, waits = [list(t) for t in table], list(held), list(free[:free_count]), 0, False
    q_start, q_len, positions, token_req, slots = [], [], [], [], []
    for r, (c, n) in enumerate(zip(cached, counts)):
        short = max(0, -(-(c + n) // P) - held[r]) if n > 0 else 0
        refused = short > 0 and (waits or short > len(stack))
        waits = waits or refused
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
    pad = [-1] * (max_tokens - at)
    return table, held, [len(stack)], q_start, q_len, positions + pad, token_req + pad, slots + pad


def plain_verify(target, q_start, tokens, lens, guess, accept, pick):
    """Request by request in 64 bits; weights as Python's whole numbers of 2^-48."""
    R, N = len(tokens), len(tokens[0]) if tokens else 0
    fixed = lambda row: [int(round(min(max(float(x), 0.0), 1.0) * 2.0 ** 48)) for x in row]
    out, emitted = [], []
    for r in range(R):
        row, n = [-1] * (N + 1), N if lens is None else lens[r]
        if n < 0:
            out.append(row)
            emitted.append(0)
            continue
        k, minus = 0, None
        while k < n:
            p, x = target[q_start[r] + k], tokens[r][k]
            q = torch.zeros_like(p).index_fill_(0, torch.tensor([x]), math.inf) if guess is None else guess[r, k]
            if accept[r][k] * (1.0 if guess is None else float(q[x])) < float(p[x]):
                row[k] = x
                k += 1
            else:
                minus = q
                break
        p = target[q_start[r] + k]
        w = fixed(p if minus is None else p - minus)
        if sum(w) == 0:
            w = fixed(p)
        goal, upto, t = min(int(pick[r] * sum(w)), sum(w) - 1), 0, 0
        for t, x in enumerate(w):
            upto += x
            if upto > goal:
                break
        row[k] = t
        out.append(row)
        emitted.append(k + 1)
    return out, emitted
