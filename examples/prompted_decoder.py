"""A prompted decoder over the library's ops: packed prompts of frames and text in, tokens out.

The layer is the usual one (RMSNorm, q / k / v, attention, output, RMSNorm, gated
FFN) with W8A8 linears, q and k normed by head and turned by (time, row, column)
positions. A batch of prompts of different lengths runs packed through
prompt_attention, the frames of each seeing one another (prefix); its keys and
values go to the paged 4-bit cache, and every further token reads them from there
with kv4_attention. Weights are random: the point is the calls.

    python examples/prompted_decoder.py [--layers 4] [--tokens 16]
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from vla_simd_b200 import ops  # noqa: E402

SECTIONS = (8, 12, 12)   # rotated pairs of the time, row and column axes of a head of 64


class PromptedDecoder:
    """Defaults: SmolVLA's text tower (hidden 960, 15 query heads over 5 key heads of 64, FFN 2560)."""

    def __init__(self, layers=4, hidden=960, n_q=15, n_kv=5, d=64, ffn=2560, vocab=4096, batch=4, max_tokens=1024,
                 page=64, seed=0):
        self.n_q, self.n_kv, self.d, self.page, self.hidden = n_q, n_kv, d, page, hidden
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(n, k):
            return ops.pack_weights_i8(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)

        ones = torch.ones(hidden, device="cuda")
        self.embed = torch.randn(vocab, hidden, generator=g, device="cuda") * 0.5
        self.layers = [dict(norm1=ones, norm2=ones, q_norm=torch.ones(d, device="cuda"), k_norm=torch.ones(d, device="cuda"),
                            qkv=weight((n_q + 2 * n_kv) * d, hidden), o=weight(hidden, n_q * d),
                            gate=weight(ffn, hidden), up=weight(ffn, hidden), down=weight(hidden, ffn))
                       for _ in range(layers)]
        self.norm, self.head = ones, weight(vocab, hidden)
        pages = -(-max_tokens // page)
        self.batch, self.room, self.longest = batch, pages * page, 0
        self.caches = [ops.kv4_cache(batch * pages, n_kv, d, page) for _ in range(layers)]
        self.table = torch.arange(batch * pages, dtype=torch.int32, device="cuda").view(batch, pages)
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.next_pos = torch.zeros(batch, dtype=torch.int32, device="cuda")

    def need(self, tokens, sequences):
        """Refuses sequences and lengths (known on the host) that the page table has no place for: an index past it
        would stop the device."""
        if sequences != self.batch:
            raise ValueError(f"{sequences} sequences for a cache of {self.batch}")
        if tokens > self.room:
            raise ValueError(f"a sequence of {tokens} tokens does not fit the cache's {self.room}: raise max_tokens")

    def slots(self, seq, at):
        """Cache slots of positions `at` of sequences `seq`."""
        return self.table[seq, at // self.page].long() * self.page + at % self.page

    def _layers(self, x, pos, slots, attend):
        T = x.shape[0]
        for w, cache in zip(self.layers, self.caches):
            h = ops.rmsnorm(x, w["norm1"])
            qkv = ops.dense_linear_i8(h, *w["qkv"]).view(T, self.n_q + 2 * self.n_kv, self.d)
            q, k = ops.qk_norm_rope(qkv[:, :self.n_q], qkv[:, self.n_q:self.n_q + self.n_kv], pos, SECTIONS, w["q_norm"],
                                    w["k_norm"], out_dtype=torch.bfloat16)
            v = qkv[:, self.n_q + self.n_kv:].to(torch.bfloat16)
            ops.kv4_append(cache, k, v, slots)
            a = attend(q, k, v, cache).float().view(T, -1)
            x = x + ops.dense_linear_i8(a, *w["o"])
            h = ops.rmsnorm(x, w["norm2"])
            f = ops.activation("silu_gate", ops.dense_linear_i8(h, *w["gate"]), ops.dense_linear_i8(h, *w["up"]))
            x = x + ops.dense_linear_i8(f, *w["down"])
        return ops.rmsnorm(x, self.norm)

    def prompt(self, x, lens, pos, frames):
        """x [T, hidden]: the prompts' embeddings, one after another; lens: their lengths; pos [3, T]; frames
        [batch]: how many leading tokens of each are frames. Returns the logits after each prompt."""
        if min(lens, default=0) < 1 or x.shape[0] != sum(lens) or pos.shape != (3, sum(lens)):
            raise ValueError("x and pos have to hold the tokens of every prompt, at least one each")
        self.need(max(lens), len(lens))
        self.longest = max(lens)
        lens_t = torch.tensor(lens, device="cuda")
        cu = torch.nn.functional.pad(lens_t.cumsum(0), (1, 0)).int()
        seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), lens_t)
        at = torch.arange(x.shape[0], device="cuda") - cu[:-1].long()[seq]
        h = self._layers(x, pos, self.slots(seq, at),
                         lambda q, k, v, cache: ops.prompt_attention(q, k, v, cu, prefix=frames))
        self.lens.copy_(lens_t)
        last = cu[1:].long() - 1
        self.next_pos = pos.amax(0)[last] + 1
        return ops.dense_linear_i8(h[last].contiguous(), *self.head)

    def step(self, tokens):
        """One token for every sequence; returns the logits after it."""
        self.need(self.longest + 1, tokens.numel())
        self.longest += 1
        seq = torch.arange(tokens.numel(), device="cuda")
        slots = self.slots(seq, self.lens.long())
        self.lens += 1
        pos = self.next_pos.expand(3, -1).int().contiguous()
        self.next_pos = self.next_pos + 1
        table = self.table[:, :-(-self.longest // self.page)]   # the pages in use: the kernel plans by its width
        h = self._layers(self.embed[tokens], pos, slots,
                         lambda q, k, v, cache: ops.kv4_attention(q, cache, table, self.lens))
        return ops.dense_linear_i8(h, *self.head)


def prompt_positions(frames, rows, cols, text):
    """(time, row, column) of a prompt: frames of rows x cols patches, then text on all axes together."""
    n = rows * cols
    i = torch.arange(frames * n)
    vis = torch.stack([i // n, i % n // cols, i % cols])
    t = torch.arange(text) + (int(vis.max()) + 1 if frames else 0)
    return torch.cat([vis, t.expand(3, -1)], 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=16)
    a = ap.parse_args()
    shapes = [(2, 8, 8, 21), (1, 8, 8, 5), (3, 8, 8, 40), (0, 0, 0, 9)]   # frames, rows, columns, words
    pos = [prompt_positions(*s) for s in shapes]
    lens = [p.shape[1] for p in pos]
    dec = PromptedDecoder(layers=a.layers, batch=len(shapes), max_tokens=max(1024, max(lens) + a.tokens))
    x = torch.randn(sum(lens), dec.hidden, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    frames = torch.tensor([f * r * c for f, r, c, _ in shapes], dtype=torch.int32, device="cuda")
    logits = dec.prompt(x, lens, torch.cat(pos, 1).int().cuda(), frames)
    out = []
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(a.tokens):
        out.append(logits.argmax(-1))
        logits = dec.step(out[-1])
    torch.cuda.synchronize()
    ms = (time.perf_counter() - t0) / a.tokens * 1e3
    for b, row in enumerate(torch.stack(out, 1).tolist()):
        print(f"prompt of {lens[b]}: {row}")
    print(f"{ms:.2f} ms a token for {len(lens)} sequences, {a.layers} layers")
    if ops.device_status() != 0:
        raise SystemExit("device status is not 0")


if __name__ == "__main__":
    main()
