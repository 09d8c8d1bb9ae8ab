"""The serving operators of a prompted policy, as measured cases.

Four operators that a prompt of frames and text goes through, in their order:

  rope     norms of the query and key heads with the multi-axis rotary positions
  prompt   attention over packed prompts of different lengths, grouped heads
  append   keys and values into the paged 4-bit cache (read back as values)
  decode   attention of new tokens (one, or a chunk) over that cache

`run` computes them either in a plain form (elementary torch operations in 32
bits) or, where `own` is set, by the framework's calls. Head counts and widths
are SmolVLA's (15 query heads over 5 key heads of 64) and a generic 32 over 8
of 128.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS, BASE = 1e-6, 10000.0
GROUP = 32        # channels that share a scale in the cache
INV15 = 1.0 / 15.0


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one new token of one robot: SmolVLA's heads in the framework's own fp32; latency alone
        dict(name="rope one token", op="rope", tokens=1, nq=15, nkv=5, d=64, sections="32", norm=False, restart=False,
             packed=True, dtype="f32", out="f32"),
        # a video prompt: time, height and width axes, norms, q and k views of one packed projection; odd length
        dict(name="rope video prompt", op="rope", tokens=4099, nq=32, nkv=8, d=128, sections="16,24,24", norm=True,
             restart=False, packed=True, dtype="bf16", out="bf16"),
        # image patches with a restarted frequency range for each axis, from the framework's fp32 activations to fp16
        dict(name="rope image patches", op="rope", tokens=16384, nq=16, nkv=16, d=64, sections="16,16", norm=True,
             restart=True, packed=False, dtype="f32", out="f16"),
        # a few prompts of one instruction and two frames each, frames seen in both directions (prefix), SmolVLA's heads
        dict(name="prompt short batch", op="prompt", lens="177,1,241,33", past=0, nq=15, nkv=5, d=64, causal=True,
             prefix=128, dtype="f16"),
        # a ragged batch of ordinary prompts, one of them a single token
        dict(name="prompt ragged batch", op="prompt", lens="2048,1,777,1531,64,129,1000,300", past=0, nq=32, nkv=8,
             d=128, causal=True, prefix=0, dtype="bf16"),
        # one long history
        dict(name="prompt long", op="prompt", lens="16384", past=0, nq=32, nkv=8, d=128, causal=True, prefix=0,
             dtype="bf16"),
        # one decoding step of 33 sequences
        dict(name="append step", op="append", tokens=33, nkv=8, d=128, page=64, dtype="bf16", order="scattered"),
        # a prompt's keys and values
        dict(name="append prompt", op="append", tokens=16384, nkv=8, d=128, page=64, dtype="bf16", order="pages"),
        # one robot, one token, a cached prefix of ordinary length
        dict(name="decode one", op="decode", lens="1021", queries=1, nq=15, nkv=5, d=64, page=16, causal=True,
             dtype="f16"),
        # action chunks of 50 queries, SmolVLA's, over cached prefixes, all queries seeing all of the prefix, in fp32
        dict(name="decode action chunk", op="decode", lens="241,177,305,33,241,192,256,113", queries=50, nq=15, nkv=5,
             d=64, page=64, causal=False, dtype="f32"),
        # a ragged serving batch
        dict(name="decode ragged batch", op="decode", lens="8192,1,4097,333,6000,17,2048,1500,64,7777,900,3001,120,5000,250,1024",
             queries=1, nq=32, nkv=8, d=128, page=64, causal=True, dtype="bf16"),
        # a full serving batch of long histories
        dict(name="decode long batch", op="decode", lens=",".join(["16384"] * 48), queries=1, nq=32, nkv=8, d=128,
             page=128, causal=True, dtype="bf16"),
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "prompt", "append", "decode"])
    nq, nkv, d = rng.choice([(15, 5, 64), (32, 8, 128), (16, 16, 64), (12, 4, 128), (8, 1, 64), (28, 4, 128)])
    half = rng.choice(["bf16", "f16"])
    if op == "rope":
        axes, pairs = rng.choice([1, 2, 3]), d // 2
        if rng.random() < 0.25:
            pairs //= 2                      # half of the channels rotated
        cut = [pairs] if axes == 1 else [pairs // 2] * 2 if axes == 2 else [pairs // 4, pairs * 3 // 8, pairs * 3 // 8]
        return dict(op=op, tokens=log_int(rng, 1, 16384), nq=nq, nkv=nkv, d=d, sections=",".join(map(str, cut)),
                    norm=rng.random() < 0.7, restart=axes > 1 and rng.random() < 0.3, packed=rng.random() < 0.5,
                    dtype=rng.choice(["f32", half]), out=rng.choice(["f32", half]))
    if op == "prompt":
        n = rng.choice([1, 1, 2, 3, 5, 8])
        causal, past = rng.random() < 0.8, rng.choice([0, 0, log_int(rng, 1, 512)])
        top = int((15800 if causal else 11000) / math.sqrt(n))   # the scores stay within the longest listed prompt's
        return dict(op=op, lens=",".join(str(log_int(rng, 1, top)) for _ in range(n)), past=past, nq=nq, nkv=nkv, d=d,
                    causal=causal,
                    prefix=rng.choice([0, 0, log_int(rng, 1, 512)]), dtype=half)
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        return dict(op=op, tokens=log_int(rng, 1, 16384), nkv=nkv, d=d, page=page, dtype=rng.choice(["f32", half]),
                    order=rng.choice(["scattered", "pages"]))
    n = log_int(rng, 1, 48)
    queries = rng.choice([1, 1, 1, log_int(rng, 2, 50)])
    return dict(op=op, lens=",".join(str(log_int(rng, 1, 16384)) for _ in range(n)) if queries == 1 else
                ",".join(str(log_int(rng, 1, 2048)) for _ in range(n)), queries=queries, nq=nq, nkv=nkv, d=d, page=page,
                causal=rng.random() < 0.7, dtype=rng.choice(["f32", half, half]))


def ints(text):
    return [int(x) for x in text.split(",")]


# ---------------------------------------------------------------- the inputs

def frame_positions(tokens, axes):
    """Positions of a prompt: text counts on all axes together, frames of 16 x 24 patches step in time, row and column."""
    t = torch.arange(tokens)
    if axes == 1:
        return t[None].int()
    frame, y, x = t // 384, t % 384 // 24, t % 24
    return torch.stack([frame, y, x] if axes == 3 else [y, x]).int()


def pack_codes(k, v):
    """Quantized keys and values of whole blocks, in the cache's layout: k, v = (codes [..., 16, d], s and m
    [..., 16, d / 32]) -> bytes [..., 20 * d]. The layout is the one include/vla_simd_cuda.h states."""
    lead = k[0].shape[:-2]
    ng = k[1].shape[-1]
    nib = torch.arange(8, device=k[0].device, dtype=torch.int32) * 4

    def words(c):                            # [..., words, 8] -> int32 words, the nibbles lowest first
        return (c.to(torch.int32) << nib).sum(-1, dtype=torch.int32)

    n = len(lead)
    # k codes: token (j, n), channel (g, kq, i) -> [j, n, kq, g] words of the nibbles i
    kc = k[0].reshape(*lead, 2, 8, ng, 4, 8).permute(*range(n), n, n + 1, n + 3, n + 2, n + 4)
    # v codes: token (j, kq, e), channel (g, n, i) -> [j, n, kq, g] words of the nibbles (e, i)
    vc = v[0].reshape(*lead, 2, 4, 2, ng, 8, 4).permute(*range(n), n, n + 4, n + 1, n + 3, n + 2, n + 5)
    vc = vc.reshape(*lead, 2, 8, 4, ng, 8)

    def by_quad(x):                          # token (j, kq, e) -> [kq, g, j, e]
        return x.reshape(*lead, 2, 4, 2, ng).permute(*range(n), n + 1, n + 3, n, n + 2)

    def as_bytes(x):
        return x.contiguous().reshape(*lead, -1).view(torch.uint8)

    km = k[2].reshape(*lead, 2, 8, ng).transpose(n, n + 1)   # token (j, n) -> [n, j, g]
    return torch.cat([as_bytes(words(kc)), as_bytes(by_quad(k[1])), as_bytes(km),
                      as_bytes(words(vc)), as_bytes(by_quad(v[1])), as_bytes(by_quad(v[2]))], -1)


def quantize(x):
    """x [..., d] -> codes [..., d] (int32), s and m [..., d / 32] (fp16): the cache's rounding, in 32 bits."""
    g = x.float().reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.amin(-1).clamp(-65504.0, 65504.0), g.amax(-1).clamp(-65504.0, 65504.0)
    s, m = ((hi - lo) * INV15).half(), lo.half()
    s32, m32 = s.float()[..., None], m.float()[..., None]
    codes = torch.where(s32 > 0, (g - m32) / torch.where(s32 > 0, s32, torch.ones_like(s32)), torch.zeros_like(g))
    return codes.round().clamp(0, 15).to(torch.int32).reshape(x.shape), s, m


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    st = dict(case)
    op, nkv, d = case["op"], case["nkv"], case["d"]
    dt = DT[case["dtype"]]

    def normal(*shape, spread=1.0):
        return torch.randn(*shape, generator=gen, device="cuda") * spread

    offset = normal(nkv, d, spread=0.5)      # keys have channels with a mean of their own
    if op == "rope":
        t, nq = case["tokens"], case["nq"]
        sections = ints(case["sections"])
        st["sections"] = tuple(sections)
        if case["packed"]:                   # q, k (and v) of one projection: strided views
            qkv = normal(t, nq + 2 * nkv, d).to(dt)
            st["q"], st["k"] = qkv[:, :nq], qkv[:, nq:nq + nkv]
        else:
            st["q"], st["k"] = normal(t, nq, d).to(dt), normal(t, nkv, d).to(dt)
        at = int(torch.randint(0, 4096, (1,), generator=gen, device="cuda"))   # a session that has gone on for a while
        st["pos"] = (frame_positions(t, len(sections)) + at).cuda()
        st["qw"] = 1.0 + 0.2 * normal(d) if case["norm"] else None
        st["kw"] = 1.0 + 0.2 * normal(d) if case["norm"] else None
        return st
    if op == "prompt":
        lq = ints(case["lens"])
        lk = [n + case["past"] for n in lq]
        tq, tk, nq = sum(lq), sum(lk), case["nq"]
        st["q"] = normal(tq, nq, d).to(dt)
        kv = normal(tk, 2 * nkv, d).to(dt)   # keys and values of one projection
        st["k"], st["v"] = kv[:, :nkv] + offset.to(dt), kv[:, nkv:]
        st["cu_q"] = torch.tensor([0] + lq).cumsum(0).int().cuda()
        st["cu_k"] = torch.tensor([0] + lk).cumsum(0).int().cuda()
        st["max_q"], st["max_k"] = max(lq), max(lk)
        st["prefix"] = torch.full((len(lq),), case["prefix"], dtype=torch.int32, device="cuda") if case["prefix"] else None
        return st
    page = case["page"]
    if op == "append":
        t = case["tokens"]
        n_pages = -(-t // page) + 3
        st["k"], st["v"] = (normal(t, nkv, d) + offset).to(dt), normal(t, nkv, d).to(dt)
        order = torch.randperm(n_pages, generator=gen, device="cuda")
        if case["order"] == "pages":         # a prompt fills its pages in order, the pages lie anywhere
            at = torch.arange(t, device="cuda")
            st["slots"] = order[at // page] * page + at % page
        else:                                # the next slot of many sequences
            st["slots"] = torch.randperm(n_pages * page, generator=gen, device="cuda")[:t]
        st["cache"] = torch.zeros(n_pages, nkv, page // 16, 20 * d, dtype=torch.uint8, device="cuda")
        return st
    lens = ints(case["lens"])
    pages = [-(-n // page) for n in lens]
    n_pages = sum(pages) + 2
    k = quantize(normal(n_pages, nkv, page // 16, 16, d) + offset[:, None, None])
    v = quantize(normal(n_pages, nkv, page // 16, 16, d))
    st["cache"] = pack_codes(k, v)
    order = torch.randperm(n_pages, generator=gen, device="cuda").int()
    table = torch.zeros(len(lens), max(pages), dtype=torch.int32, device="cuda")
    used = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[used:used + n]
        used += n
    st["table"], st["lens"] = table, torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["max_len"] = max(lens)
    st["q"] = normal(len(lens), case["queries"], case["nq"], d).to(dt)
    return st


# ------------------------------------------------------------ the plain forms

def rope_plain(st):
    def one(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        half = sum(st["sections"])
        a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1).to(DT[st["out"]])

    sections = torch.tensor(st["sections"], device="cuda")
    half = sum(st["sections"])
    i = torch.arange(half, device="cuda")
    axis = (i[:, None] >= sections.cumsum(0)[None]).sum(-1)
    # a position times a frequency loses the position in 32 bits: the angle alone is formed in 64
    if st["restart"]:
        start = sections.cumsum(0) - sections
        freq = BASE ** -((i - start[axis]).double() / sections[axis].double())
    else:
        freq = BASE ** -(i.double() / half)
    angle = st["pos"][axis].double().T * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    return one(st["q"], st["qw"]), one(st["k"], st["kw"])


def softmax_values(s, v):
    """softmax(s) @ v over the last axis in 32 bits, s overwritten; a row of -inf gives zeros."""
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top > -math.inf, top, torch.zeros_like(top))).exp_()
    total = s.sum(-1, keepdim=True)
    return (s @ v) / torch.where(total > 0, total, torch.ones_like(total))


def prompt_plain(st):
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    nq, nkv, d = st["nq"], st["nkv"], st["d"]
    cq, ck = st["cu_q"].long(), st["cu_k"].long()
    lq, lk = cq.diff(), ck.diff()
    i, j = torch.arange(st["max_q"], device="cuda"), torch.arange(st["max_k"], device="cuda")
    # padded to [sequences, longest]: rows past a sequence's end are clamped here and left out below
    qp = q[(cq[:-1, None] + i).clamp(max=q.shape[0] - 1)].reshape(-1, i.numel(), nkv, nq // nkv, d)
    at = (ck[:-1, None] + j).clamp(max=k.shape[0] - 1)
    kp, vp = k[at].transpose(1, 2), v[at].transpose(1, 2)                       # [n, nkv, Lk, d]
    qp = qp.permute(0, 2, 3, 1, 4).reshape(-1, nkv, nq // nkv * i.numel(), d)   # [n, nkv, G * Lq, d]
    lim = lk[:, None].expand(-1, i.numel())
    if st["causal"]:
        lim = torch.minimum((i[None] + 1 + (lk - lq)[:, None]).clamp(min=0), lim)
    if st["prefix"] is not None:
        lim = torch.maximum(lim, torch.minimum(st["prefix"].long(), lk)[:, None])
    s = qp @ kp.transpose(-1, -2)
    s = s.mul_(1.0 / math.sqrt(d)).view(-1, nkv, nq // nkv, i.numel(), j.numel())
    s.masked_fill_((j >= lim[..., None])[:, None, None], -math.inf)
    o = softmax_values(s.view(qp.shape[0], nkv, -1, j.numel()), vp)
    o = o.view(-1, nkv, nq // nkv, i.numel(), d).permute(0, 3, 1, 2, 4).reshape(-1, i.numel(), nq, d)
    return o[i[None] < lq[:, None]].to(DT[st["dtype"]])


def append_plain(st):
    def values(x):
        codes, s, m = quantize(x)
        g = codes.float().reshape(*s.shape, GROUP)
        return (g * s.float()[..., None] + m.float()[..., None]).reshape(x.shape)

    return values(st["k"]), values(st["v"])


def unpack(blocks):
    """Bytes [..., 20 * d] of the cache's blocks -> keys and values [..., 16, d] in 32 bits."""
    lead, d = blocks.shape[:-1], blocks.shape[-1] // 20
    ng, n = d // GROUP, len(blocks.shape) - 1
    nib = torch.arange(8, device=blocks.device, dtype=torch.int32) * 4
    kc, ks, km, vc, vs, vm = blocks.split([8 * d, d, d, 8 * d, d, d], -1)

    def codes(b, *shape):
        return ((b.contiguous().view(torch.int32).reshape(*lead, 2, 8, 4, ng, 1) >> nib) & 15).reshape(*lead, *shape)

    def by_quad(b):
        x = b.contiguous().view(torch.float16).reshape(*lead, 4, ng, 2, 2)
        return x.permute(*range(n), n + 2, n, n + 3, n + 1).reshape(*lead, 16, ng, 1).float()

    k = codes(kc, 2, 8, 4, ng, 8).permute(*range(n), n, n + 1, n + 3, n + 2, n + 4).reshape(*lead, 16, ng, GROUP)
    v = codes(vc, 2, 8, 4, ng, 2, 4).permute(*range(n), n, n + 2, n + 4, n + 3, n + 1, n + 5).reshape(*lead, 16, ng, GROUP)
    km = km.contiguous().view(torch.float16).reshape(*lead, 8, 2, ng).transpose(n, n + 1).reshape(*lead, 16, ng, 1)
    k = k.float().mul_(by_quad(ks)).add_(km.float())
    v = v.float().mul_(by_quad(vs)).add_(by_quad(vm))
    return k.reshape(*lead, 16, d), v.reshape(*lead, 16, d)


def decode_plain(st):
    q = st["q"].float()
    B, lq, nq, d = q.shape
    nkv = st["nkv"]
    k, v = unpack(st["cache"][st["table"].long()].transpose(1, 2))      # [B, nkv, pages, blocks, 16, d]
    k, v = k.reshape(B, nkv, -1, d), v.reshape(B, nkv, -1, d)
    j = torch.arange(k.shape[2], device="cuda")
    lim = st["lens"].long()[:, None].expand(-1, lq)
    if st["causal"]:
        lim = (lim - lq + 1 + torch.arange(lq, device="cuda")).clamp(min=0)
    qp = q.reshape(B, lq, nkv, nq // nkv, d).permute(0, 2, 3, 1, 4).reshape(B, nkv, -1, d)
    s = (qp @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).view(B, nkv, nq // nkv, lq, -1)
    s.masked_fill_((j >= lim[..., None])[:, None, None], -math.inf)
    o = softmax_values(s.view(B, nkv, nq // nkv * lq, -1), v)
    return o.view(B, nkv, nq // nkv, lq, d).permute(0, 3, 1, 2, 4).reshape(B, lq, nq, d).to(DT[st["dtype"]])


PLAIN = {"rope": rope_plain, "prompt": prompt_plain, "append": append_plain, "decode": decode_plain}


def run(st):
    if not own:
        return PLAIN[st["op"]](st)
    from vla_simd_b200 import ops
    if st["op"] == "rope":
        return ops.qk_norm_rope(st["q"], st["k"], st["pos"], st["sections"], st["qw"], st["kw"], eps=EPS, base=BASE,
                                restart=st["restart"], out_dtype=DT[st["out"]])
    if st["op"] == "prompt":
        return ops.prompt_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], causal=st["causal"],
                                    prefix=st["prefix"])
    if st["op"] == "append":
        ops.kv4_append(st["cache"], st["k"], st["v"], st["slots"])
        return ops.kv4_read(st["cache"], st["slots"])
    return ops.kv4_attention(st["q"], st["cache"], st["table"], st["lens"], causal=st["causal"])


def work(case):
    op, nkv, d = case["op"], case["nkv"], case["d"]
    size = SIZE[case["dtype"]]
    if op == "rope":
        values = case["tokens"] * (case["nq"] + nkv) * d
        return {"bytes": values * (size + SIZE[case["out"]]) + 4 * case["tokens"] * len(ints(case["sections"])),
                "flops": values * (6.0 + (4.0 if case["norm"] else 0.0))}
    if op == "append":                       # read, 5 bits a value written and read back, the values written
        values = 2 * case["tokens"] * nkv * d
        return {"bytes": values * (size + 2 * 0.625 + 4), "flops": values * 8.0}
    lens, nq = ints(case["lens"]), case["nq"]
    if op == "prompt":
        pairs = 0
        for n in lens:
            lk = n + case["past"]
            pre = min(case["prefix"], lk)
            if case["causal"]:               # sum of max(i + 1 + past, prefix) over the queries
                first = max(0, min(n, pre - case["past"]))
                pairs += first * pre + (n - first) * case["past"] + (n * (n + 1) - first * (first + 1)) // 2
            else:
                pairs += n * lk
        tq, tk = sum(lens), sum(lens) + case["past"] * len(lens)
        return {"bytes": size * d * (2.0 * tq * nq + 2.0 * tk * nkv), "flops": 4.0 * d * nq * pairs}
    lq = case["queries"]
    pairs = sum(max(0, n - lq + 1 + i) if case["causal"] else n for n in lens for i in range(lq))
    return {"bytes": sum(lens) * nkv * 2 * d * 0.625 + 2.0 * size * len(lens) * lq * nq * d, "flops": 4.0 * d * nq * pairs}


# ------------------------------------------------- the definitions, in 64 bits

def exact_rope(st):
    f, half = [], sum(st["sections"])
    for n in st["sections"]:
        f += [BASE ** (-j / n) if st["restart"] else BASE ** (-(len(f) + j) / half) for j in range(n)]
    axis = [a for a, n in enumerate(st["sections"]) for _ in range(n)]
    pos = st["pos"].double()
    turn = torch.stack([torch.polar(torch.ones_like(pos[a]), pos[a] * w) for a, w in zip(axis, f)], -1)
    out = []
    for x, w in ((st["q"], st["qw"]), (st["k"], st["kw"])):
        y = x.double().clone()
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + EPS).sqrt() * w.double()
        z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn[:, None]
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
        out.append(y)
    return tuple(out)


def exact_rows(q, k, v, lim):
    """q [rows, d] over k, v [keys, d], row r seeing lim[r] keys, in pieces of the rows."""
    out = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64, device=q.device)
    at = torch.arange(k.shape[0], device=q.device)
    for r in range(0, q.shape[0], 4096):
        s = (q[r:r + 4096] @ k.T) / math.sqrt(q.shape[1])
        seen = at[None] < lim[r:r + 4096, None]
        p = torch.softmax(s.masked_fill(~seen, -1e300), -1) * seen
        out[r:r + 4096] = p @ v
    return out


def exact_prompt(st):
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    cq, ck = st["cu_q"].tolist(), st["cu_k"].tolist()
    for n in range(len(cq) - 1):
        lq, lk = cq[n + 1] - cq[n], ck[n + 1] - ck[n]
        lim = [min(lk, max(0, i + 1 + lk - lq)) if st["causal"] else lk for i in range(lq)]
        if st["prefix"] is not None:
            lim = [max(x, min(int(st["prefix"][n]), lk)) for x in lim]
        lim = torch.tensor(lim, device="cuda")
        for h in range(st["nq"]):
            g = h // (st["nq"] // st["nkv"])
            out[cq[n]:cq[n + 1], h] = exact_rows(st["q"][cq[n]:cq[n + 1], h].double(), st["k"][ck[n]:ck[n + 1], g].double(),
                                                 st["v"][ck[n]:ck[n + 1], g].double(), lim)
    return out


def exact_append(st):
    out = []
    for x in (st["k"], st["v"]):
        y = x.double().unflatten(-1, (-1, GROUP))
        lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
        s, m = ((hi - lo) / 15).float().half().double(), lo.float().half().double()
        c = ((y - m) / s.clamp(min=1e-12)).round().clamp(0, 15) * (s > 0)
        out.append((c * s + m).flatten(-2))
    return tuple(out)


def exact_decode(st):
    d, lq, nq, nkv, page = st["d"], st["queries"], st["nq"], st["nkv"], st["page"]
    ng = d // GROUP
    t, c = torch.arange(16, device="cuda")[:, None], torch.arange(d, device="cuda")[None]
    g = c // 32
    quad = 2 * ((((t % 8) // 2 * ng + g) * 2 + t // 8) * 2 + t % 2)             # byte of a scale, by token and group
    k_at = ((t * 4 + c % 32 // 8) * ng + g) * 4 + c % 8 // 2                    # byte of a key's code
    v_at = ((t // 8 * 32 + c % 32 // 4 * 4 + t % 8 // 2) * ng + g) * 4 + t % 2 * 2 + c % 4 // 2
    km_at = 2 * ((t % 8 * 2 + t // 8) * ng + g)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")

    def number(block, at):                   # the fp16 number at a byte
        two = torch.stack([block[..., at], block[..., at + 1]], -1)
        return two.view(torch.float16)[..., 0].double()

    for b, n in enumerate(st["lens"].tolist()):
        blocks = st["cache"][st["table"][b, :-(-n // page)].long()]             # [pages, nkv, blocks, 20 d]
        lim = torch.tensor([max(0, n - lq + 1 + i) if st["causal"] else n for i in range(lq)], device="cuda")
        for h in range(nkv):
            x = blocks[:, h].reshape(-1, 20 * d)
            k = (x[:, k_at] >> (c % 2 * 4)) & 15
            k = k.double() * number(x, 8 * d + quad) + number(x, 9 * d + km_at)
            v = (x[:, 10 * d + v_at] >> (c % 2 * 4)) & 15
            v = v.double() * number(x, 18 * d + quad) + number(x, 19 * d + quad)
            k, v = k.reshape(-1, d)[:n], v.reshape(-1, d)[:n]
            for r in range(nq // nkv):
                out[b, :, h * (nq // nkv) + r] = exact_rows(st["q"][b, :, h * (nq // nkv) + r].double(), k, v, lim)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return {"rope": exact_rope, "prompt": exact_prompt, "append": exact_append, "decode": exact_decode}[case["op"]](st)
