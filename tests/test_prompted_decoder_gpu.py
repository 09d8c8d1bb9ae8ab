"""examples/prompted_decoder.py: prompts and steps against the same layers with attention written out in 64 bits.

The linears are the library's own on both sides, so a difference can only come from positions, slots, tables,
lengths and attention. Attention is off by a bf16 rounding of its output and of its weights (2^-7 of its size at
most); int8 quantizers downstream turn such differences into steps of 1/127 of a row's largest value. Through two
layers the logits agree to a few per cent of their size, while a wrong slot, position or mask moves them by as much
as they are.
"""
import math
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


def test_prompt_and_steps():
    import prompted_decoder as ex
    from vla_simd_b200 import ops

    shapes = [(2, 4, 6, 13), (0, 0, 0, 3), (1, 3, 5, 30)]
    dec = ex.PromptedDecoder(layers=2, hidden=320, n_q=6, n_kv=2, ffn=640, vocab=300, batch=3, max_tokens=128, page=16)
    pos = [ex.prompt_positions(*s) for s in shapes]
    lens = [p.shape[1] for p in pos]
    frames = torch.tensor([f * r * c for f, r, c, _ in shapes], dtype=torch.int32, device="cuda")
    x = torch.randn(sum(lens), dec.hidden, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    all_pos = torch.cat(pos, 1).int().cuda()
    G, d = dec.n_q // dec.n_kv, dec.d

    def attend(q, k, v, lim):
        s = torch.einsum("ihd,jhd->hij", q.double(), k.double().repeat_interleave(G, 1)) / math.sqrt(d)
        s = s.masked_fill(torch.arange(k.shape[0], device="cuda")[None, None] >= lim[None, :, None], -math.inf)
        return torch.einsum("hij,jhd->ihd", s.softmax(-1), v.double().repeat_interleave(G, 1))

    def plain_prompt_attention(q, k, v, cu, prefix):
        out = torch.empty_like(q)
        for b in range(3):
            lo, hi = int(cu[b]), int(cu[b + 1])
            lim = torch.maximum(torch.arange(1, hi - lo + 1, device="cuda"), prefix[b].long())
            out[lo:hi] = attend(q[lo:hi], k[lo:hi], v[lo:hi], lim).to(q.dtype)
        return out

    def plain_cache_attention(q, cache, table, n):
        out = torch.empty_like(q)
        for b in range(3):
            at = torch.arange(int(n[b]), device="cuda")
            k, v = ops.kv4_read(cache, dec.slots(torch.full_like(at, b), at))
            out[b] = attend(q[b:b + 1], k, v, torch.tensor([len(at)], device="cuda"))[0].to(q.dtype)
        return out

    def run(prompt_attention, kv4_attention):
        dec.lens.zero_()
        for c in dec.caches:
            c.zero_()
        real = ops.prompt_attention, ops.kv4_attention
        ops.prompt_attention, ops.kv4_attention = prompt_attention, kv4_attention
        try:
            out = [dec.prompt(x, lens, all_pos, frames)]
            for i in range(3):
                out.append(dec.step(torch.tensor([5 + i, 17, 200 - i], device="cuda")))
        finally:
            ops.prompt_attention, ops.kv4_attention = real
        return out

    got = run(ops.prompt_attention, ops.kv4_attention)
    want = run(plain_prompt_attention, plain_cache_attention)
    assert dec.lens.tolist() == [n + 3 for n in lens]
    for g, w in zip(got, want):
        assert g.shape == (3, 300) and (g - w).norm() <= 0.05 * w.norm()
    assert ops.device_status() == 0
