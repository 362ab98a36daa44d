"""A text decoder that writes lines token by token, on the library's operators: image tokens of many
lines as the prompt, then beam search over a paged 8-bit cache.

    python examples/text_decoder.py [lines] [steps]

The weights are random (the text is noise), the layers are ordinary: RMS norm, grouped-query
attention with normed and rotated heads, a gated product. Matrix products are torch's; what the
library adds is the attention of the packed prompts (every line's image tokens see each other), the
cache that keys and values are written to and attended to in 8 bits, and the choice of the beams with
the reordering of their pages.
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wgpu-ocr_amd"))
import ocrhip  # noqa: E402

VOCAB, EOS = 97, 0  # the ocrs alphabet and the end


class Decoder:
    """`layers` layers of width q_heads * dim, heads of `dim` values."""

    def __init__(self, ctx, layers=2, q_heads=8, heads=2, dim=64, dtype=torch.float16, seed=1):
        self.ctx, self.layers, self.q_heads, self.heads, self.dim, self.dtype = ctx, layers, q_heads, heads, dim, dtype
        self.width = width = q_heads * dim
        g = torch.Generator().manual_seed(seed)
        w = lambda *s: (torch.randn(*s, generator=g) * s[0] ** -0.5).to(dtype).cuda()  # noqa: E731
        self.qkv = [w(width, (q_heads + 2 * heads) * dim) for _ in range(layers)]
        self.out = [w(width, width) for _ in range(layers)]
        self.up, self.gate = ([w(width, 2 * width) for _ in range(layers)] for _ in range(2))
        self.down = [w(2 * width, width) for _ in range(layers)]
        self.q_norm, self.k_norm = ([torch.ones(dim).cuda() for _ in range(layers)] for _ in range(2))
        self.embed = torch.randn(VOCAB, width, generator=g).to(dtype).cuda()
        self.head = (w(width, VOCAB).float() * 3).to(dtype)

    def norm(self, x):
        y = x.float()
        return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)).to(self.dtype)

    def forward(self, x, attend):
        """x [n][width] through the layers; attend(layer, projections) gives the heads' outputs."""
        for i in range(self.layers):
            x = x + attend(i, self.norm(x) @ self.qkv[i]).flatten(1) @ self.out[i]
            y = self.norm(x)
            x = x + (torch.nn.functional.silu(y @ self.gate[i]) * (y @ self.up[i])) @ self.down[i]
        return x

    def logits(self, x):
        return (self.norm(x) @ self.head).float()


class Writer:
    """The state of a search: a cache a layer, all with the same pages; `beams` sequences a line."""

    def __init__(self, model, lines, beams, most, fmt="i8", page=16):
        self.model, self.lines, self.beams, self.page = model, lines, beams, page
        self.rows, self.ctx = lines * beams, model.ctx
        width = -(-most // page)
        # Enough pages that none has to come back: each sequence's own, and one a step for its copy.
        self.pages = self.rows * (width + most)
        self.caches = [ocrhip.KvCache(self.ctx, self.pages, page, model.heads, model.dim, fmt) for _ in range(model.layers)]
        self.table = torch.full((self.rows, width), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(self.rows, dtype=torch.int32, device="cuda")
        self.seq = torch.arange(self.rows, dtype=torch.int32, device="cuda")
        self.taken = 0
        self.scores = torch.full((lines, beams), -float("inf"), device="cuda")
        self.scores[:, 0] = 0
        self.finished = torch.zeros(lines, beams, dtype=torch.int32, device="cuda")
        self.text = torch.zeros(lines, beams, 0, dtype=torch.int32, device="cuda")

    def take(self, n):
        self.taken += n
        assert self.taken <= self.pages
        return torch.arange(self.taken - n, self.taken, dtype=torch.int32, device="cuda")

    def call(self, f, *args, **more):
        """A library call between torch's work, in torch's stream's order."""
        stream = torch.cuda.current_stream().cuda_stream
        self.ctx.acquire(stream)
        f(*args, **more)
        self.ctx.release(stream)

    def prompt(self, tokens, counts):
        """tokens [n][width]: the lines' image tokens one after another, counts[i] of line i. Their
        keys and values go to the pages of each line's first beam."""
        m = self.model
        n = len(tokens)
        count = torch.tensor(counts, device="cuda")
        docs = torch.cat([count.new_zeros(1), count.cumsum(0)]).to(torch.int32)
        line = torch.repeat_interleave(torch.arange(self.lines, device="cuda"), count)
        pos = (torch.arange(n, device="cuda") - docs[line]).to(torch.int32)
        for i, c in enumerate(counts):
            need = -(-c // self.page)
            self.table[i * self.beams, :need] = self.take(need)
            self.lens[i * self.beams] = c
        seq = (line * self.beams).to(torch.int32)

        def attend(i, qkv):
            q = torch.empty(n, m.q_heads, m.dim, dtype=m.dtype, device="cuda")
            k = torch.empty(n, m.heads, m.dim, dtype=m.dtype, device="cuda")
            v = qkv[:, (m.q_heads + m.heads) * m.dim:].unflatten(1, (m.heads, m.dim))
            out = torch.empty_like(q)
            self.call(self.caches[i].append, self.table, seq, pos, qkv, q, k, m.q_norm[i], m.k_norm[i])
            self.call(ocrhip.attention, self.ctx, q, k, v, out, docs, prefix=count.to(torch.int32))
            return out

        x = m.forward(tokens, attend)[(docs[1:] - 1).long()]
        # Every beam starts from its line's last image token.
        self.choose(m.logits(x).repeat_interleave(self.beams, 0))

    def step(self):
        """The beams' next tokens."""
        m = self.model
        fresh = (self.lens % self.page == 0).nonzero()[:, 0]
        if len(fresh):
            self.table[fresh, (self.lens[fresh] // self.page).long()] = self.take(len(fresh))
        pos, after = self.lens.clone(), self.lens + 1

        def attend(i, qkv):
            q = torch.empty(self.rows, m.q_heads, m.dim, dtype=m.dtype, device="cuda")
            out = torch.empty_like(q)
            self.call(self.caches[i].append, self.table, self.seq, pos, qkv, q, None, m.q_norm[i], m.k_norm[i])
            self.call(self.caches[i].attend, self.table, after, q, out)
            return out

        x = m.forward(m.embed[self.text[:, :, -1].flatten().long()], attend)
        self.lens = after
        self.choose(m.logits(x))

    def choose(self, logits):
        """The best continuations, and the pages that go with them."""
        parents, tokens = (torch.empty(self.lines, self.beams, dtype=torch.int32, device="cuda") for _ in range(2))
        self.call(ocrhip.beam_select, self.ctx, logits, self.scores, self.finished, EOS, self.scores, parents, tokens, self.finished)
        table, lens, used = torch.empty_like(self.table), torch.empty_like(self.lens), torch.empty_like(self.lens)
        spare = self.take(self.rows)
        for cache in self.caches:  # the same tables each time, and each cache's copies
            self.call(cache.fork, self.table, self.lens, parents, spare, table, lens, used)
        self.table, self.lens = table, lens
        self.text = torch.cat([self.text.gather(1, parents.long()[..., None].expand_as(self.text)), tokens[..., None]], 2)


def write(model, tokens, counts, beams, steps, fmt="i8"):
    """(text [lines][beams][steps], scores [lines][beams]) for the lines' image tokens."""
    w = Writer(model, len(counts), beams, max(counts) + steps, fmt)
    w.prompt(tokens, counts)
    for _ in range(steps - 1):
        w.step()
    return w.text, w.scores


def main():
    lines, steps = (int(a) for a in (sys.argv[1:] + ["6", "24"][len(sys.argv) - 1:])[:2])
    ctx = ocrhip.Context()
    model = Decoder(ctx)
    g = torch.Generator().manual_seed(2)
    counts = [int(c) for c in torch.randint(20, 110, (lines,), generator=g)]
    tokens = torch.randn(sum(counts), model.width, generator=g).to(model.dtype).cuda()
    text, scores = write(model, tokens, counts, 4, steps)
    alphabet = " 0123456789!\"#$%&'()*+,-./:;<=>?@[\\]^_`{|}~ABCDEFGHIJKLMNOPQRSTUVWXYZabcdefghijklmnopqrstuvwxyz"
    for t, s in zip(text[:, 0].tolist(), scores[:, 0].tolist()):
        t = t[: t.index(EOS)] if EOS in t else t
        print(f"{s:9.3f}  {''.join(alphabet[min(c, len(alphabet) - 1)] for c in t)}")


if __name__ == "__main__":
    main()
