"""A turn of several requests on mounted grafts and the 8-bit paged arena.

    python examples/paged_turn.py

Every request is admitted with routed grafts: packed INT4 keys and values that one
mount writes, re-RoPEd at their seats, as bf16 rows (``ArenaMount``).  Those rows
join the request's pages in the 8-bit arena (plan, append).  Then the requests
take a question of a few rows each, ragged, and a number of single tokens, all of
them together in one step (plan, append, attend).  At the end a request's own
turn is read back and packed as a graft again (read), and its pages go to whoever
comes next (release).

The model around it is a stand-in with random weights: projections, RoPE,
attention, a residual; nothing else.
"""

import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from graftrepository_b200 import graft_mount  # noqa: E402
from graftrepository_b200.paged_arena import PagedArena, PageTables  # noqa: E402


class PagedTurn:
    """Requests that share one arena, and a stand-in model of `layers` layers."""

    def __init__(self, requests=4, layers=2, kv_heads=8, group=4, head_dim=128, limit=2048,
                 page_tokens=64, device="cuda:0", seed=0):
        self.requests, self.layers, self.device = requests, layers, device
        self.heads = dict(kv_heads=kv_heads, query_heads=kv_heads * group, head_dim=head_dim)
        self.width = kv_heads * group * head_dim
        pages = requests * -(-limit // page_tokens)
        self.tables = PageTables(requests, pages, pages, page_tokens=page_tokens, device=device)
        self.arena = PagedArena(layers, pages, kv_heads, head_dim, page_tokens=page_tokens,
                                device=device)
        # a plan for single tokens, which the kernel for few rows serves, and one for more
        self.one = self.tables.make_plan(requests, max_fresh=1, **self.heads)
        self.many = self.tables.make_plan(limit, **self.heads)
        cos, sin = graft_mount.rope_tables(limit, head_dim)
        self.cos, self.sin = torch.from_numpy(cos).to(device), torch.from_numpy(sin).to(device)
        self.rope = graft_mount.RopeSpec(self.cos, self.sin, offset=0, dim=head_dim)
        gen = torch.Generator(device=device).manual_seed(seed)

        def weight(n, m):
            w = torch.randn((layers, n, m), device=device, generator=gen)
            return (w * n ** -0.5).to(torch.bfloat16)

        kv = kv_heads * head_dim
        self.wq, self.wo = weight(self.width, self.width), weight(self.width, self.width)
        self.wk, self.wv = weight(self.width, kv), weight(self.width, kv)

    def counts(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def rotate(self, x, positions):
        """RoPE of rows [tokens, heads, head_dim]; rows past the step's last have
        position -1 and are not used."""
        at = positions.clamp(min=0).long()
        half = x.shape[2] // 2
        turned = torch.cat([-x[:, :, half:], x[:, :, :half]], 2)
        return (x * self.cos[at][:, None] + turned * self.sin[at][:, None]).to(x.dtype)

    def admit(self, request, grafts):
        """`grafts`: for keys and for values (codes, scales) of packed INT4 grafts
        [n, layers * kv_heads, tokens * head_dim], keys without RoPE, and the
        tokens of one of them.  They become the request's first tokens."""
        keys, values, tokens = grafts
        n, dim = keys[0].shape[0], self.heads["head_dim"]
        kv_heads = self.heads["kv_heads"]
        seats = np.arange(n, dtype=np.int64) * tokens
        rows = []
        for (codes, scales), rope in ((keys, self.rope), (values, None)):
            mount = graft_mount.ArenaMount(self.layers * kv_heads, n * tokens, dim, self.device)
            mount.mount_packed(torch.from_numpy(codes).to(self.device),
                               torch.from_numpy(scales.view(np.uint16)).to(self.device), seats,
                               tokens, 4, rope=rope, stream=torch.cuda.current_stream())
            rows.append(mount.arena.view(self.layers, kv_heads, n * tokens, dim))
        fresh = self.counts([n * tokens if r == request else 0 for r in range(self.requests)])
        plan = self.tables.make_plan(n * tokens, **self.heads)
        self.tables.plan(plan, fresh)
        for layer in range(self.layers):  # [tokens, kv_heads, head_dim] as it stands, no copy
            self.arena.append(plan, *(x[layer].transpose(0, 1) for x in rows), layer=layer)
        self.tables.commit(plan)
        plan.check()

    def step(self, x, fresh):
        """Hidden rows `x` [tokens, width], the requests' `fresh` rows (a list of
        counts) one after another; returns the hidden rows after all layers."""
        plan = self.one if max(fresh) <= 1 else self.many
        rows = x.shape[0]
        if rows < plan.tokens:
            x = torch.cat([x, x.new_zeros((plan.tokens - rows, self.width))])
        self.tables.plan(plan, self.counts(fresh))
        for layer in range(self.layers):
            y = torch.nn.functional.rms_norm(x, (self.width,))
            q = self.rotate((y @ self.wq[layer]).view(plan.query_shape), plan.positions)
            k = self.rotate((y @ self.wk[layer]).view(plan.kv_shape), plan.positions)
            v = (y @ self.wv[layer]).view(plan.kv_shape)
            self.arena.append(plan, k, v, layer=layer)
            out = self.attend(plan, q, layer)
            x = x + out.view(plan.tokens, self.width) @ self.wo[layer]
        self.tables.commit(plan)
        plan.check()  # waits; the next plan call would clear what this step has to say
        return x[:rows]

    def attend(self, plan, q, layer):
        return self.arena.attend(plan, q, layer=layer)[0]

    def harvest(self, request, first, tokens):
        """Tokens `first` .. of a request as a packed INT4 graft (keys, values);
        the keys keep their RoPE."""
        page = self.tables.page_tokens
        at = torch.arange(first, first + tokens, device=self.device)
        slots = self.tables.table[request].long()[at // page] * page + at % page
        sides = ([], [])
        for layer in range(self.layers):
            for side, x in zip(sides, self.arena.read(slots, layer=layer, dtype=torch.float32)):
                side.append(x.transpose(0, 1))  # [kv_heads, tokens, head_dim]
        return tuple(graft_mount.quantize_packed(
            torch.cat(side).reshape(1, -1, tokens * self.heads["head_dim"]).cpu().numpy(), 4)
            for side in sides)

    def release(self, requests):
        self.tables.release(self.counts(requests))


def random_grafts(turn, n, tokens, seed):
    """Packed INT4 keys and values of n grafts."""
    rng = np.random.default_rng(seed)
    shape = (n, turn.layers * turn.heads["kv_heads"], tokens * turn.heads["head_dim"])
    return tuple(graft_mount.quantize_packed(rng.standard_normal(shape, np.float32), 4)
                 for _ in range(2)) + (tokens,)


def run(turn, question=(5, 40, 1, 17), answer=16, grafts=2, graft_tokens=128):
    """Admit every request, take the question (its rows for each of them), answer
    those that asked token by token; returns the last hidden row of each of these."""
    for r in range(turn.requests):
        turn.admit(r, random_grafts(turn, grafts, graft_tokens, seed=r))
    gen = torch.Generator(device=turn.device).manual_seed(1)
    x = torch.randn((sum(question), turn.width), device=turn.device, generator=gen)
    x = turn.step(x.to(torch.bfloat16), question)
    asked = torch.tensor(question) > 0
    x = x[(torch.tensor(question).cumsum(0) - 1)[asked].to(turn.device)]
    for _ in range(answer):  # the stand-in feeds its own result back
        x = turn.step(x, asked.int().tolist())
    return x


def main():
    turn = PagedTurn()
    x = run(turn)
    lens = turn.tables.lens.tolist()
    print(f"requests hold {lens} tokens; last rows {tuple(x.shape)}, finite: "
          f"{bool(torch.isfinite(x).all())}")
    keys, values = turn.harvest(1, 256, lens[1] - 256)
    print(f"request 1's own {lens[1] - 256} tokens as a graft: {keys[0].nbytes + values[0].nbytes} "
          "bytes of codes")
    turn.release([1])
    turn.admit(1, random_grafts(turn, 1, 128, seed=9))
    print(f"after its release and another admission: {turn.tables.lens.tolist()}")


if __name__ == "__main__":
    main()
