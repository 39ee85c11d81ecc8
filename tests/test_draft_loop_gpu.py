"""The operators together, as a program that verifies drafted tokens runs them: tables, keys and values into their slots, attention,
verification, and the lengths that come out of it into the next step, without a word from the host in between."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
V, WIDTH, H, K, d, P = 97, 64, 8, 2, 64, 8
PAGES, N = 26, 3


def model(seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64) / math.sqrt(s[0])
    return dict(embed=torch.randn(V, WIDTH, generator=g, dtype=torch.float64), qkv=r(WIDTH, (H + 2 * K) * d), o=r(H * d, WIDTH), head=3 * r(WIDTH, V))


def plain_logits(m, tokens):
    """One layer of attention in 64 bits: logits behind the last token."""
    x = m["embed"][tokens]
    q, k, v = (x @ m["qkv"]).split((H * d, K * d, K * d), dim=-1)
    q, k, v = q[-1].view(H, d), k.view(-1, K, d), v.view(-1, K, d)
    o = torch.stack([torch.softmax(q[h] @ k[:, h // (H // K)].T / math.sqrt(d), -1) @ v[:, h // (H // K)] for h in range(H)])
    return (x[-1] + o.reshape(-1) @ m["o"]) @ m["head"]


def greedy(m, prompt, n):
    tokens, least = list(prompt), math.inf
    for _ in range(n):
        top = plain_logits(m, tokens).topk(2)
        least = min(least, float(top.values[0] - top.values[1]))
        tokens.append(int(top.indices[0]))
    return tokens, least


class Loop:
    """Device state of R requests and one step over it; the step is a function of device memory alone."""

    def __init__(self, m, prompts, dtype):
        R = len(prompts)
        self.m = {k: v.float().to(DEV) for k, v in m.items()}
        self.dtype, self.R, self.longest = dtype, R, max(map(len, prompts))
        ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)
        self.cached, self.held, self.free_count, self.err = ints(R), ints(R), ints(1) + PAGES, ints(1)
        self.table = ints(R, PAGES) - 1
        self.free = torch.randperm(PAGES, generator=torch.Generator().manual_seed(3)).int().to(DEV)
        self.pools = [torch.full((PAGES, K, P, d), float("nan"), dtype=dtype, device=DEV) for _ in range(2)]
        self.last, self.drafts = ints(R), ints(R, N)
        self.tokens, self.emitted = ints(R, N + 1), ints(R)

    def _run(self, ids, counts, most):
        from ai_engine_b200.cache import step_tables
        from ai_engine_b200.kernels import ops

        t = step_tables(self.cached, counts, self.held, self.table, self.free, self.free_count, P, PAGES, most, self.err)
        x = self.m["embed"][ids.long()]
        qkv = x @ self.m["qkv"]
        k, v = (qkv[:, (H + i * K) * d:(H + (i + 1) * K) * d].view(-1, K, d) for i in range(2))
        ops.write_kv_slots(k, v, *self.pools, t.slots, self.err)
        q = qkv[:, :H * d].to(self.dtype).view(-1, H, d)
        a = ops.paged_attention_chunks(q, *self.pools, t.q_start, t.q_len, self.cached, t.tables, 1 / math.sqrt(d), 0, self.err,
                                       out=torch.zeros_like(q))
        return t, (x + a.float().view(-1, H * d) @ self.m["o"]) @ self.m["head"]

    def _keep(self, t, emitted):
        self.cached += torch.where(t.q_len > 0, emitted, 0)
        for mine, new in ((self.held, t.held), (self.table, t.tables), (self.free_count, t.free_count)):
            mine.copy_(new)

    def prompt(self, prompts):
        """Prompts as portions: the longest first in the batch's width, then the first token of each."""
        lens = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=DEV)
        ids = torch.tensor([x for p in prompts for x in p], dtype=torch.int32, device=DEV)
        t, logits = self._run(ids, lens, int(ids.numel()))
        self._keep(t, t.q_len)
        self.last.copy_(logits[(t.q_start + t.q_len - 1).long()].argmax(-1).int())

    def step(self):
        """Verifies self.drafts behind self.last."""
        from ai_engine_b200.sampling import verify_drafts

        ids = torch.cat([self.last[:, None], self.drafts], dim=1).reshape(-1)
        counts = torch.full_like(self.cached, N + 1)
        t, logits = self._run(ids, counts, self.R * (N + 1))
        certain = torch.zeros_like(logits).scatter_(1, logits.argmax(-1, keepdim=True), 1.0)
        lens = torch.where(t.q_len > 0, t.q_len - 1, -1).int()      # a request that waits for pages is idle
        draws = torch.full((self.R, N), 0.5, device=DEV)
        tokens, emitted = verify_drafts(certain, t.q_start, self.drafts, lens, None, draws, draws[:, 0].contiguous(), self.err)
        self._keep(t, emitted)
        new = tokens.gather(1, (emitted - 1).clamp(min=0)[:, None].long())[:, 0]
        self.last.copy_(torch.where(emitted > 0, new, self.last))
        self.tokens.copy_(tokens)
        self.emitted.copy_(emitted)


@pytest.mark.parametrize("captured", [False, True])
def test_drafts_are_verified_as_greedy_decoding_goes_on(captured):
    """Requests whose drafts are the true continuation up to a place that differs from step to step: tokens come out as greedy decoding in
    64 bits makes them one by one.  The pool is too small for all of them to the end, so the last one waits."""
    m = model(7)
    prompts = [[5, 9, 33, 60, 2], [71], [14, 3, 8, 8, 90, 41, 22, 17, 6, 50, 11]]
    wanted = [greedy(m, p, 90) for p in prompts]
    # No choice is nearer than float32 tells apart: sums of up to 512 products are off by about sqrt(512) roundings of the vectors' norms (22
    # and 1): 3e-5 an element of what the head multiplies, by columns of norm 3: 1e-4.
    assert min(least for _, least in wanted) > 1e-4
    loop = Loop(m, prompts, torch.float32)
    loop.prompt(prompts)
    got = [p + [x] for p, x in zip(prompts, loop.last.tolist())]
    graph, g = None, torch.Generator().manual_seed(1)
    waited = False
    for step in range(28):
        for r, have in enumerate(got):
            true = wanted[r][0][len(have):len(have) + N]
            right = int(torch.randint(0, N + 1, (1,), generator=g))
            drafts = [x if i < right else (x + 1 + i) % V for i, x in enumerate(true)] + [0] * (N - len(true))
            loop.drafts[r] = torch.tensor(drafts, dtype=torch.int32)
        if captured and step == 2:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                loop.step()
        if graph is not None:
            graph.replay()
        else:
            loop.step()
        for r, (row, n) in enumerate(zip(loop.tokens.tolist(), loop.emitted.tolist())):
            waited |= n == 0
            got[r] += row[:n]
            assert row[n:] == [-1] * (N + 1 - n)
    assert int(loop.err.item()) == 0 and waited
    for have, (true, _) in zip(got, wanted):
        n = min(len(have), len(true))
        assert have[:n] == true[:n] and n > 40
    # no page is anybody's twice, and the lengths are what came out
    held = [x for row, n in zip(loop.table.tolist(), loop.held.tolist()) for x in row[:n]]
    rest = loop.free.tolist()[:int(loop.free_count)]
    assert sorted(held + rest) == list(range(PAGES))
    assert [c + 1 for c in loop.cached.tolist()] == [len(h) for h in got]


def test_the_same_loop_in_bfloat16_stays_finite():
    """bfloat16 pools behind the same steps (tokens may part from 64 bits): nothing unwritten is read, nothing is flagged."""
    m = model(8)
    prompts = [[5, 9, 33], [71, 4, 4, 18, 2, 2, 60, 31, 9]]
    loop = Loop(m, prompts, torch.bfloat16)
    loop.prompt(prompts)
    for step in range(10):
        loop.drafts.copy_(torch.randint(0, V, (2, N), generator=torch.Generator().manual_seed(step)).int())
        loop.step()
        assert all(0 <= x < V for row, n in zip(loop.tokens.tolist(), loop.emitted.tolist()) for x in row[:n])
    assert int(loop.err.item()) == 0
