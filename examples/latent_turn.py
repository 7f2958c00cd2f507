"""A turn of several requests on mounted latent grafts and pages of latent rows.

    python examples/latent_turn.py

Every request is admitted with routed grafts: packed INT4 rows of a latent vector and
a positional part, which one mount writes, re-RoPEd at their seats, as bf16 rows
(``ArenaMount``).  Those rows join the request's pages (plan, append).  Then the
requests take a question of a few rows each, ragged, which attends in the expanded
form, and a number of single tokens, all of them together in one step, in the
absorbed form; positions are put on by ``Rotary`` and, for rows, on the way into their
pages.  At the end a request's own turn is packed as a graft again, its positions
taken off, and its pages go to whoever comes next (release).

The model around it is a stand-in with random weights: projections, positions,
attention, a residual; nothing else.
"""

import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from graftrepository_b200 import graft_mount  # noqa: E402
from graftrepository_b200.latent_arena import LatentArena  # noqa: E402
from graftrepository_b200.paged_arena import PageTables  # noqa: E402
from graftrepository_b200.rotary import Rotary  # noqa: E402


class LatentTurn:
    """Requests that share one arena, and a stand-in model of `layers` layers."""

    def __init__(self, requests=4, layers=2, heads=40, latent=256, rope=32, nope=64, width=640,
                 limit=2048, page_tokens=64, device="cuda:0", seed=0):
        self.requests, self.layers, self.heads, self.width = requests, layers, heads, width
        self.latent, self.rope, self.nope, self.device = latent, rope, nope, device
        self.scale = (nope + rope) ** -0.5
        pages = requests * -(-limit // page_tokens)
        self.tables = PageTables(requests, pages, pages, page_tokens=page_tokens, device=device)
        self.arena = LatentArena(layers, pages, latent, rope, page_tokens=page_tokens,
                                 device=device)
        # a plan for single tokens, which attend in the absorbed form, and one for more
        self.one = self.arena.make_plan(self.tables, requests, heads=heads, max_fresh=1)
        self.many = self.arena.make_plan(self.tables, limit, heads=heads, nope=nope, value=nope,
                                         expand_tokens=pages * page_tokens)
        cos, sin = graft_mount.rope_tables(limit, rope)
        cos, sin = torch.from_numpy(cos).to(device), torch.from_numpy(sin).to(device)
        self.mounts = graft_mount.RopeSpec(cos, sin, offset=latent, dim=rope)
        # the same frequencies for rows on their way in, for queries and for whole rows
        self.keys, self.queries, self.rows = (Rotary(rope, offset=at, device=device)
                                              for at in (0, nope, latent))
        gen = torch.Generator(device=device).manual_seed(seed)

        def weight(n, m):
            w = torch.randn((layers, n, m), device=device, generator=gen)
            return (w * n ** -0.5).to(torch.bfloat16)

        self.wq, self.wo = weight(width, heads * (nope + rope)), weight(heads * nope, width)
        self.wc, self.wr = weight(width, latent), weight(width, rope)
        # [layers, heads, nope + value, latent]: what makes a head's keys and values of a row
        wkv = weight(latent, heads * 2 * nope).mT.contiguous()
        self.wkv = wkv.view(layers, heads, 2 * nope, latent)

    def counts(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.device)

    def admit(self, request, grafts):
        """`grafts`: (codes, scales) of packed INT4 grafts [n, layers, tokens * (latent +
        rope)] without RoPE, and the tokens of one of them.  They become the
        request's first tokens."""
        (codes, scales), tokens = grafts
        n, wide = codes.shape[0], self.latent + self.rope
        seats = np.arange(n, dtype=np.int64) * tokens
        mount = graft_mount.ArenaMount(self.layers, n * tokens, wide, self.device)
        mount.mount_packed(torch.from_numpy(codes).to(self.device),
                           torch.from_numpy(scales.view(np.uint16)).to(self.device), seats, tokens,
                           4, rope=self.mounts, stream=torch.cuda.current_stream())
        rows = mount.arena.view(self.layers, n * tokens, wide)
        fresh = self.counts([n * tokens if r == request else 0 for r in range(self.requests)])
        plan = self.arena.make_plan(self.tables, n * tokens, heads=1)
        self.tables.plan(plan, fresh)
        for layer in range(self.layers):  # positions are on them
            self.arena.append(plan, *rows[layer].split([self.latent, self.rope], 1), layer=layer)
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
            self.arena.append(plan, y @ self.wc[layer], y @ self.wr[layer], layer=layer,
                              rotary=self.keys)
            q = (y @ self.wq[layer]).view(plan.tokens, self.heads, self.nope + self.rope)
            q = self.queries.rotate(q, plan.positions)
            attend = self.absorbed if plan is self.one else self.expanded
            x = x + attend(plan, q, layer).reshape(plan.tokens, -1) @ self.wo[layer]
        self.tables.commit(plan)
        plan.check()  # waits; the next plan call would clear what this step has to say
        return x[:rows]

    def absorbed(self, plan, q, layer):
        """Queries into the latent space, and results out of it again."""
        keys, values = self.wkv[layer].split(self.nope, 1)
        q_latent = torch.einsum("thn,hnc->thc", q[:, :, :self.nope], keys)
        out = self.attend(plan, q_latent, q[:, :, self.nope:], layer)
        return torch.einsum("thc,hvc->thv", out, values)

    def attend(self, plan, q_latent, q_rope, layer):
        return self.arena.attend(plan, q_latent, q_rope, scale=self.scale, layer=layer)[0]

    def expanded(self, plan, q, layer):
        return self.arena.attend_expanded(plan, q, self.wkv[layer], scale=self.scale,
                                          layer=layer)[0]

    def slots(self, request, first, tokens):
        """Rows of the arena that hold tokens `first` .. of a request."""
        page = self.tables.page_tokens
        at = torch.arange(first, first + tokens, device=self.device)
        return self.tables.table[request].long()[at // page] * page + at % page

    def harvest(self, request, first, tokens):
        """Tokens `first` .. of a request as a packed INT4 graft without RoPE, as
        ``admit`` takes it (an even number of them: groups are of 64 values)."""
        slots = self.slots(request, first, tokens)
        at = torch.arange(first, first + tokens, dtype=torch.int32, device=self.device)
        rows = [self.rows.rotate(x.flatten(0, 1)[slots][:, None], at, inverse=True)
                for x in self.arena.rows]
        return graft_mount.quantize_packed(
            torch.stack(rows).float().reshape(1, self.layers, -1).cpu().numpy(), 4), tokens

    def release(self, requests):
        self.tables.release(self.counts(requests))


def random_grafts(turn, n, tokens, seed):
    """Packed INT4 rows of n grafts."""
    rng = np.random.default_rng(seed)
    shape = (n, turn.layers, tokens * (turn.latent + turn.rope))
    return graft_mount.quantize_packed(rng.standard_normal(shape, np.float32), 4), tokens


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
    turn = LatentTurn()
    x = run(turn)
    lens = turn.tables.lens.tolist()
    print(f"requests hold {lens} tokens; last rows {tuple(x.shape)}, finite: "
          f"{bool(torch.isfinite(x).all())}")
    graft = turn.harvest(1, 256, lens[1] - 256)
    print(f"request 1's own {lens[1] - 256} tokens as a graft: {graft[0][0].nbytes} bytes of codes")
    turn.release([1])
    turn.admit(1, graft)
    print(f"after its release and the graft's admission: {turn.tables.lens.tolist()}")


if __name__ == "__main__":
    main()
