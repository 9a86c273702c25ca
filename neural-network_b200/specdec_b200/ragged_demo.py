"""A small server of ragged requests on the 8-bit paged cache: every step takes
prompt chunks of some requests and single tokens of others through
``KV8.plan``, ``KV8.append``, ``KV8.attend`` and ``sample``, requests come and
go, and their pages go back to the ring.  The model is a few layers of
attention with random weights.

    python -m specdec_b200.ragged_demo [requests] [new tokens]
"""
from __future__ import annotations

import sys
import time

import specdec_b200 as sd


class Model:
    """Embedding + position waves, layers of normalisation, attention and a residual, tied output rows."""

    def __init__(self, vocab=1000, layers=2, heads=8, kv_heads=2, dim=64, seed=0, dtype=None):
        import torch

        g = torch.Generator().manual_seed(seed)
        self.vocab, self.layers, self.heads, self.kv_heads, self.dim = vocab, layers, heads, kv_heads, dim
        self.dtype = dtype or torch.bfloat16
        width, kv = heads * dim, kv_heads * dim

        def weight(*shape):
            return (torch.randn(*shape, generator=g) * shape[-1] ** -0.5).to("cuda", self.dtype)

        self.embed = (torch.randn(vocab, width, generator=g)).to("cuda", self.dtype)
        self.wqkv = [weight(width + 2 * kv, width) for _ in range(layers)]
        self.wo = [weight(width, width) for _ in range(layers)]
        self.freq = torch.exp(-torch.arange(width // 2) * (9.0 / (width // 2))).cuda()

    def positions(self, pos):
        import torch

        a = pos[:, None].float() * self.freq
        return torch.cat([a.sin(), a.cos()], 1)

    def forward(self, ids, pos, attention):
        """Logit rows of tokens `ids` at `pos`; attention(layer, q, k, v) -> rows of q's shape."""
        import torch

        x = self.embed[ids].float() + self.positions(pos)
        width, kv = self.heads * self.dim, self.kv_heads * self.dim
        for i in range(self.layers):
            y = torch.nn.functional.layer_norm(x, (width,)).to(self.dtype)
            q, k, v = (y @ self.wqkv[i].T).split([width, kv, kv], 1)
            heads = [t.view(len(ids), -1, self.dim) for t in (q, k, v)]  # parts of one buffer, by stride
            x = x + (attention(i, *heads).reshape(len(ids), width) @ self.wo[i].T).float()
        y = torch.nn.functional.layer_norm(x, (width,)).to(self.dtype)
        return lambda rows: y[rows] @ self.embed.T * width ** -0.5


class Server:
    """Slots of requests over one pool of pages."""

    def __init__(self, model: Model, slots=8, max_len=512, pages=None, page_tokens=64, block_tokens=16, chunk=48):
        import torch

        self.m, self.slots, self.chunk, self.page_tokens = model, slots, chunk, page_tokens
        cols = -(-max_len // page_tokens)
        pages = pages or slots * cols
        self.kv = sd.KV8(model.heads, model.kv_heads, model.dim, page_tokens, block_tokens, max_batch=slots)
        codes = (pages, model.kv_heads, page_tokens, model.dim)
        scales = (pages, model.kv_heads, page_tokens // block_tokens)
        self.cache = [sd.KV8Layer(*(torch.zeros(codes, dtype=torch.int8, device="cuda") for _ in range(2)),
                                  *(torch.zeros(scales, device="cuda") for _ in range(2))) for _ in range(model.layers)]
        # a step reads the last step's lengths while it writes its own: two batches over one table take turns
        most = slots * chunk
        ints = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")
        table, status = torch.full((slots, cols), -1, dtype=torch.int32, device="cuda"), ints(1)
        self.kv_len = [ints(slots) for _ in range(2)]
        self.maps = dict(cu_q=ints(slots + 1), tok_req=ints(most), tok_pos=ints(most),
                         slots=torch.zeros(most, dtype=torch.int64, device="cuda"), status=status)
        self.batch = [sd.KV8Batch(table, self.kv_len[i], **self.maps) for i in range(2)]
        self.ring = torch.arange(pages, dtype=torch.int32, device="cuda")
        self.state = [torch.tensor([0, pages], dtype=torch.int32, device="cuda"), ints(2)]
        self.turn, self.free = 0, pages

    def serve(self, prompts, n_new, temperature=0.8, top_k=40, top_p=0.95, min_p=0.02, seed=0):
        """The prompts with n_new drawn tokens each."""
        import torch

        g = torch.Generator().manual_seed(seed)
        done, waiting = [list(p) for p in prompts], list(range(len(prompts)))
        if any(not p for p in done):
            raise ValueError("prompts must not be empty")
        need = [-(-(len(p) + n_new) // self.page_tokens) for p in done]
        if max(need, default=0) > min(self.batch[0]._keep[0].shape[1], self.ring.shape[0]):
            raise ValueError("a request does not fit the pool")
        total = [len(p) + n_new for p in done]
        at, held = [None] * self.slots, [0] * self.slots  # request of each slot; positions in the cache
        while waiting or any(r is not None for r in at) or any(held):
            keep, q, ids, last, given = list(held), [0] * self.slots, [], [], 0
            for s in range(self.slots):
                if at[s] is not None and len(done[at[s]]) == total[at[s]]:  # ended: its pages go back in this step
                    given += need[at[s]]  # to be had from the next step on
                    at[s], keep[s] = None, 0
                elif at[s] is None and waiting and held[s] == 0 and need[waiting[0]] <= self.free:
                    at[s] = waiting.pop(0)
                    self.free -= need[at[s]]
                if at[s] is not None:
                    new = done[at[s]][keep[s]:keep[s] + self.chunk]
                    q[s] = len(new)
                    ids += new
                    if keep[s] + q[s] == len(done[at[s]]):
                        last.append((s, len(ids) - 1))
            rows = self.step(keep, q, ids, [i for _, i in last])
            if last:
                n = len(last)
                tokens = torch.zeros(n, dtype=torch.int32, device="cuda")
                full = lambda v, t=torch.float32: torch.full((n,), v, dtype=t, device="cuda")
                sd.sample(rows, torch.rand(n, generator=g).cuda(), tokens, temperature=full(temperature),
                          top_k=full(top_k, torch.int32), top_p=full(top_p), min_p=full(min_p),
                          stream=torch.cuda.current_stream().cuda_stream)
                for (s, _), t in zip(last, tokens.tolist()):
                    done[at[s]].append(t)
            held = [k + n for k, n in zip(keep, q)]
            self.free += given
        return done

    def step(self, keep, q, ids, last):
        """One pass of the rows `ids` (q[s] of slot s, in order): logits of the rows `last`."""
        import torch

        st = torch.cuda.current_stream().cuda_stream
        t, self.turn = self.turn, self.turn ^ 1
        now = self.batch[t ^ 1]
        ints = lambda v, dt=torch.int32: torch.tensor(v, dtype=dt, device="cuda")
        self.kv.plan(now, self.kv_len[t], ints(keep), ints(q), self.ring, self.state[t], self.state[t ^ 1], stream=st)
        if not ids:
            return None

        def attention(layer, q_rows, k, v):
            out = torch.empty_like(q_rows, memory_format=torch.contiguous_format)
            self.kv.append(self.cache[layer], now, k, v, stream=st)
            self.kv.attend(self.cache[layer], now, q_rows, out, max_q=max(q), stream=st)
            return out

        logits = self.m.forward(ints(ids, torch.int64), self.maps["tok_pos"][:len(ids)], attention)
        self.kv.check(st)
        if int(self.maps["status"][0]):
            raise sd.SpecDecError(1, f"the step could not be planned: status {int(self.maps['status'][0])}")
        return logits(ints(last, torch.int64)) if last else None


def main(requests=20, n_new=40):
    import torch

    g = torch.Generator().manual_seed(1)
    model = Model()
    server = Server(model)
    prompts = [torch.randint(0, model.vocab, (int(n),), generator=g).tolist()
               for n in torch.randint(1, 200, (requests,), generator=g)]
    server.serve(prompts[:2], 2)
    t = time.perf_counter()
    out = server.serve(prompts, n_new)
    t = time.perf_counter() - t
    print(f"{requests} requests, {sum(map(len, prompts))} prompt tokens, {sum(map(len, out)) - sum(map(len, prompts))} new "
          f"tokens in {t:.2f} s; free pages {int(server.state[server.turn][1])} of {server.ring.shape[0]}")


if __name__ == "__main__":
    main(*(int(a) for a in sys.argv[1:]))
