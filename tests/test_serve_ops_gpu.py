"""The prompt and 4-bit cache operators against their definitions in 64 bits.

Tolerances, per element. u is the unit roundoff of the output type (2^-8 bf16,
2^-11 fp16, 2^-24 fp32):
* rope: one output rounding, and in 32 bits the norm's sum of at most 256
  squares (16 sequential adds and a tree: 2^-20), rsqrt, three products and a sine and
  a cosine of an angle known to 2^-25 turns (2^-22 each): 2^-19 of the pair.
* prompt attention: one output rounding of o, weights rounded to the type (u of
  A = sum p |v|), and 2^-12 of A for scores (at most 128 products summed in 32
  bits, |score| <= 2^6: 2^-15 absolute), exponentials and sums.
* cache attention: one output rounding, for bf16 weights rounded at 2^-11, and
  the same 2^-12 of A; fp32 also holds 5e-6 in the 2-norm, where the errors of a
  sum of 128 in 32 bits are independent (sqrt(128) 2^-24 on scores below 2^3).
"""
import math

import numpy as np
import pytest
import torch

from vla_simd_b200 import VLA_ERR_ARG, VLA_ERR_SHAPE, VlaError, lib, ops

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def assert_within(got, want, tol):
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / tol).nan_to_num(9e9).max()} times the bound"


# ---------------------------------------------------------------- rope

def rope_reference(x, pos, sections, w, eps, base, restart):
    x = x.double()
    y = x if w is None else x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    half = sum(sections)
    a, b = y[..., :half], y[..., half:2 * half]
    cols = []
    i = 0
    for axis, n in enumerate(sections):
        for j in range(n):
            f = base ** (-j / n) if restart else base ** (-i / half)
            cols.append(pos[axis].double() * f)
            i += 1
    ang = torch.stack(cols, -1)[:, None]
    out = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), y[..., 2 * half:]], -1)
    size = torch.cat([a.abs() + b.abs(), a.abs() + b.abs(), y[..., 2 * half:].abs()], -1)
    return out, size


def check_rope(q, k, pos, sections, qw, kw, restart=False, out=None, base=10000.0, eps=1e-6):
    got = ops.qk_norm_rope(q, k, pos, sections, qw, kw, eps=eps, base=base, restart=restart, out_dtype=out)
    for g, x, w in zip(got, (q, k), (qw, kw)):
        if x is None:
            assert g is None
            continue
        want, size = rope_reference(x, pos, sections, w, eps, base, restart)
        assert g.dtype == (out or x.dtype) and g.shape == x.shape
        assert_within(g, want, U[g.dtype] * want.abs() + 2.0 ** -19 * size + 2.0 ** -24 * (g.dtype == F16) + 1e-30)


@pytest.mark.parametrize("T,nq,nkv,d,sections,norm,restart", [
    (1, 15, 5, 64, (32,), True, False),
    (1, 1, 1, 2, (1,), True, False),
    (3, 4, 2, 128, (16, 24, 24), True, False),
    (37, 16, 16, 64, (16, 16), True, True),
    (5, 3, 1, 96, (8, 16, 16, 8), True, False),
    (7, 8, 8, 128, (32,), False, False),          # half of the channels pass through
    (9, 2, 1, 80, (3, 7), True, True),            # pairs that do not come in fours
    (6, 5, 5, 10, (2, 1), True, False),
    (2, 2, 2, 256, (64, 64), True, False),
    (2, 1, 3, 32, (16,), False, False),
    (2051, 4, 2, 64, (8, 12, 12), True, False),   # the many-token form, odd
    (4, 40, 8, 136, (20, 20, 24), True, False),
])
@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16), (BF16, F32), (F16, BF16)])
def test_rope(T, nq, nkv, d, sections, norm, restart, types):
    g = gen(T * 1000 + d)
    q, k = randn(g, T, nq, d, dtype=types[0]), randn(g, T, nkv, d, dtype=types[0])
    pos = torch.randint(0, 5000, (len(sections), T), generator=g, device="cuda", dtype=torch.int32)
    w = [1 + 0.3 * randn(g, d) if norm else None for _ in range(2)]
    check_rope(q, k, pos, sections, *w, restart=restart, out=types[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rope_strides_positions_and_values(dtype):
    g = gen(5)
    T, nq, nkv, d = 19, 6, 3, 64
    qkv = randn(g, T, nq + 2 * nkv, d, dtype=dtype)
    pos = torch.tensor([[0, -1, 1, 7, 2 ** 20, 2 ** 24, 2 ** 31 - 1, -2 ** 31] + [5] * 11], dtype=torch.int32, device="cuda")
    w = 1 + 0.3 * randn(g, d)
    check_rope(qkv[:, :nq], qkv[:, nq:nq + nkv], pos, (32,), w, None)          # a norm on q alone, views
    wide = randn(g, T, nq, 2 * d + 1, dtype=dtype)                             # odd strides and addresses
    check_rope(wide[:, :, 1:1 + d], wide[:, ::2, d:2 * d], pos, (32,), w, w)
    by_head = randn(g, nq, T, d, dtype=dtype).transpose(0, 1)                  # heads outermost
    check_rope(by_head, by_head[:, :2], pos, (16,), w, w, base=1e6)
    every_other = randn(g, T, nq, 2 * d, dtype=dtype)[..., ::2]                # channels apart: copied
    check_rope(every_other, None, pos, (32,), w, None)
    zero = torch.zeros(T, nq, d, dtype=dtype, device="cuda")                   # a row of zeros stays zeros
    out, _ = ops.qk_norm_rope(zero, None, pos, (32,), w)
    assert (out == 0).all()
    out, none = ops.qk_norm_rope(zero[:0], zero[:0, :2], pos[:, :0].contiguous(), (32,), w)
    assert out.shape == (0, nq, d) and none.shape == (0, 2, d)


def test_rope_keeps_other_rows_from_a_nan():
    g = gen(6)
    q, k = randn(g, 4, 4, 64), randn(g, 4, 2, 64)
    q[1, 2, 5], k[3, 0, 9] = math.nan, math.inf
    pos = torch.arange(4, dtype=torch.int32, device="cuda")[None].contiguous()
    w = torch.ones(64, device="cuda")
    a, b = ops.qk_norm_rope(q, k, pos, (32,), w, w)
    assert a[1, 2].isnan().all() and a.isnan().sum() == 64
    bad = torch.zeros_like(b, dtype=torch.bool)
    bad[3, 0] = True
    assert b[~bad].isfinite().all()


# ---------------------------------------------------------------- prompts

def limits(lq, lk, causal, prefix):
    lim = np.full(lq, lk)
    if causal:
        lim = np.clip(np.arange(lq) + 1 + lk - lq, 0, lk)
    return np.maximum(lim, min(prefix, lk))


def attend(q, k, v, lim, scale):
    """q [rows, d] over k, v [keys, d]; returns softmax.v and sum p |v| (64 bits), unseen keys never touched."""
    o = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    for n in sorted(set(lim)):
        rows = torch.tensor([i for i, x in enumerate(lim) if x == n], device=q.device)
        if n > 0:
            p = torch.softmax(scale * (q[rows].double() @ k[:n].double().T), -1)
            o[rows], a[rows] = p @ v[:n].double(), p @ v[:n].double().abs()
    return o, a


def check_prompt(q, k, v, lq, lk, causal=True, prefix=None, scale=None, cu_k=True, start=0):
    n_q, n_kv, d = q.shape[1], k.shape[1], q.shape[2]
    cq = torch.tensor([start] + lq).cumsum(0).int().cuda()
    ck = torch.tensor([start] + lk).cumsum(0).int().cuda()
    pre = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda")
    got = ops.prompt_attention(q, k, v, cq, ck if cu_k else None, scale=scale, causal=causal, prefix=pre)
    assert got.shape == q.shape and got.dtype == q.dtype
    sc = 1 / math.sqrt(d) if scale is None else scale
    for s in range(len(lq)):
        lim = limits(lq[s], lk[s], causal, 0 if prefix is None else prefix[s])
        for h in range(n_q):
            kh = h // (n_q // n_kv)
            kk, vv = k[ck[s]:ck[s + 1], kh], v[ck[s]:ck[s + 1], kh]
            o, a = attend(q[cq[s]:cq[s + 1], h], kk, vv, lim, sc)
            assert_within(got[cq[s]:cq[s + 1], h], o, U[q.dtype] * (o.abs() + a) + 2.0 ** -12 * a + 1e-30)
    assert ops.device_status() == 0
    return got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lens,nq,nkv,d", [
    ([1], 1, 1, 64), ([1, 1, 1], 15, 5, 64), ([2, 0, 3], 4, 4, 128), ([127, 128, 129], 2, 1, 64),
    ([255, 1, 257], 4, 2, 128), ([300], 15, 5, 64), ([33, 0, 0, 70], 32, 8, 128), ([200], 7, 1, 96),
    ([65], 5, 5, 8), ([130], 12, 4, 72), ([90, 40], 28, 4, 128), ([64], 32, 1, 64), ([40], 66, 2, 64),
    ([50], 131, 1, 24), ([700], 3, 3, 128), ([1025, 511], 8, 2, 64), ([17] * 40, 2, 1, 64),
])
def test_prompt_causal(dtype, lens, nq, nkv, d):
    g = gen(sum(lens) + d)
    T = sum(lens)
    check_prompt(randn(g, T, nq, d, dtype=dtype), randn(g, T, nkv, d, dtype=dtype), randn(g, T, nkv, d, dtype=dtype),
                 lens, lens, cu_k=False)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("prefix", [None, [0, 50, 400]])
@pytest.mark.parametrize("lq,lk", [([5, 64, 130], [5, 300, 131]), ([1, 1, 1], [1, 128, 257]),
                                   ([40, 9, 200], [3, 9, 0]), ([0, 3, 129], [7, 0, 128])])
def test_prompt_past_prefix_and_empty_rows(lq, lk, causal, prefix):
    g = gen(3)
    q = randn(g, sum(lq), 6, 64, dtype=BF16)
    k, v = randn(g, sum(lk), 2, 64, dtype=BF16), randn(g, sum(lk), 2, 64, dtype=BF16)
    got = check_prompt(q, k, v, lq, lk, causal, prefix)
    at = 0
    for s in range(3):
        lim = limits(lq[s], lk[s], causal, 0 if prefix is None else prefix[s])
        empty = torch.from_numpy(lim == 0).cuda()
        assert (got[at:at + lq[s]][empty] == 0).all()
        at += lq[s]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_large_scores(dtype, d):
    """Maxima that keep growing along the keys (every rescaling of the sums), and rows of one dominant key."""
    g = gen(8)
    T, nq, nkv = 520, 4, 2
    q = randn(g, T, nq, d, dtype=dtype).abs()
    k = (randn(g, T, nkv, d).abs() * torch.linspace(0, 4, T, device="cuda")[:, None, None] / d).to(dtype)
    v = randn(g, T, nkv, d, dtype=dtype)
    check_prompt(q, k, v, [T], [T], scale=4.0)
    check_prompt(q, -k, v, [T], [T], scale=4.0)
    check_prompt(q, k, v, [T], [T], causal=False, scale=-3.0)
    check_prompt(q, k, v, [T], [T], scale=0.0)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("nq,nkv,d", [(2, 1, 128), (3, 1, 64)])
def test_prompt_of_many_ring_rounds(dtype, nq, nkv, d):
    g = gen(17)
    T = 3001
    q, k, v = randn(g, T, nq, d, dtype=dtype), randn(g, T, nkv, d, dtype=dtype), randn(g, T, nkv, d, dtype=dtype)
    check_prompt(q[:300], k, v, [300], [T])
    check_prompt(q, k, v, [T], [T], causal=False)
    check_prompt(q, k, v, [T - 64, 64], [T - 64, 64], prefix=[1500, 10])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prompt_strides(dtype):
    g = gen(9)
    T, nq, nkv, d = 150, 6, 2, 64
    qkv = randn(g, T, nq + 2 * nkv, d, dtype=dtype)
    check_prompt(qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:], [100, 50], [100, 50])
    by_head = randn(g, nq, T, d, dtype=dtype).transpose(0, 1)
    kv_by_head = randn(g, 2 * nkv, T, d, dtype=dtype).transpose(0, 1)
    check_prompt(by_head, kv_by_head[:, :nkv], kv_by_head[:, nkv:], [150], [150])
    odd = randn(g, T, nq + 2 * nkv, d + 3, dtype=dtype)[..., 1:1 + d]          # copied: no tensor map describes it
    check_prompt(odd[:, :nq], odd[:, nq:nq + nkv], odd[:, nq + nkv:], [150], [150])
    one = randn(g, T, 1, d, dtype=dtype).expand(T, nkv, d)                     # one head for all, stride 0
    check_prompt(qkv[:, :nq], one, one, [150], [150])


@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_masked_places_do_not_reach_a_row(fill, d):
    g = gen(10)
    lens = [70, 133, 5, 260]
    T, nq, nkv = sum(lens) + 40, 4, 2
    q, k, v = randn(g, T, nq, d, dtype=BF16), randn(g, T, nkv, d, dtype=BF16), randn(g, T, nkv, d, dtype=BF16)
    for x in (k, v):           # before the first sequence, in one sequence, past the last
        x[:20], x[20 + 70 + 133:20 + 70 + 133 + 5], x[-20:] = fill, fill, fill
    k, v = k.contiguous(), v.contiguous()
    cu = torch.tensor([20] + lens).cumsum(0).int().cuda()
    got = ops.prompt_attention(q, k, v, cu)
    for s in (0, 1, 3):
        lo, hi = int(cu[s]), int(cu[s + 1])
        for h in range(nq):
            o, a = attend(q[lo:hi, h], k[lo:hi, h // 2], v[lo:hi, h // 2], limits(hi - lo, hi - lo, True, 0), d ** -0.5)
            assert_within(got[lo:hi, h], o, U[BF16] * (o.abs() + a) + 2.0 ** -12 * a)
    # a value that the causal mask hides from the earlier rows of its own sequence
    lo, hi, at = int(cu[3]), int(cu[4]), 200
    k2, v2 = k.clone(), v.clone()
    k2[lo + at, 0], v2[lo + at, 1] = fill, fill
    got = ops.prompt_attention(q, k2, v2, cu)
    want = ops.prompt_attention(q, k, v, cu)
    assert torch.equal(got[lo:lo + at].isfinite(), torch.ones_like(got[lo:lo + at], dtype=torch.bool))
    assert_within(got[lo:lo + at], want[lo:lo + at].double(), 2 * U[BF16] * want[lo:lo + at].double().abs() + 2.0 ** -7)
    assert not got[lo + at:hi, 2:].isfinite().any()      # and the rows that see it show it


def test_prompt_on_another_stream_and_in_a_graph():
    g = gen(11)
    q, k, v = (randn(g, 200, n, 64, dtype=BF16) for n in (4, 2, 2))
    cu = torch.tensor([0, 200], dtype=torch.int32, device="cuda")
    want = ops.prompt_attention(q, k, v, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.prompt_attention(q, k, v, cu)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.prompt_attention(q, k, v, cu)
    q.mul_(0.5)
    graph.replay()
    assert torch.equal(out, ops.prompt_attention(q, k, v, cu))


# ---------------------------------------------------------------- 4-bit cache

def quantized(x):
    """The definition in 32-bit IEEE operations on the CPU: codes, s, m."""
    x = x.float().cpu().unflatten(-1, (-1, 32))
    bad = ~x.isfinite().all(-1)
    x = torch.where(bad[..., None], torch.zeros(()), x)
    lo, hi = x.amin(-1).clamp(-65504, 65504), x.amax(-1).clamp(-65504, 65504)
    s, m = ((hi - lo) * np.float32(1 / 15)).half(), lo.half()
    sf = s.float()[..., None]
    c = torch.where(sf > 0, (x - m.float()[..., None]) / torch.where(sf > 0, sf, torch.ones(())), torch.zeros(()))
    c = c.round().clamp(0, 15)
    s[bad] = m[bad] = math.nan
    return c, s, m


def values(x):
    c, s, m = quantized(x)
    return (c * s.float()[..., None] + m.float()[..., None]).flatten(-2)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,nkv,d,page", [(1, 1, 64, 16), (1, 8, 128, 64), (33, 5, 64, 32), (130, 3, 128, 16), (257, 2, 64, 256)])
def test_kv4_append_and_read(dtype, T, nkv, d, page):
    g = gen(T + d)
    n_pages = T // page + 3
    k, v = randn(g, T, nkv, d, dtype=dtype), (randn(g, T, nkv, d) * 3 + 1).to(dtype)
    k[0, 0, :32] = 0.25                         # a group of one value
    k[-1, -1, :32], v[0, 0, -32:] = 1e-6, 0.0
    slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:T]
    cache = ops.kv4_cache(n_pages, nkv, d, page)
    before = cache.clone()
    ops.kv4_append(cache, k, v, slots)
    rk, rv = ops.kv4_read(cache, slots)
    assert torch.equal(rk.cpu(), values(k)) and torch.equal(rv.cpu(), values(v))
    for x, y in ((k, rk), (v, rv)):             # half a step, the rounding of m and of a step of 15 ends
        c, s, m = quantized(x)
        step = s.float()[..., None].expand(c.shape).flatten(-2)
        slack = (x.float().cpu().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True) * 2.0 ** -9).expand(c.shape).flatten(-2)
        assert ((x.float().cpu() - y.cpu()).abs() <= 0.5 * step + slack + 1e-7).all()
    other = torch.ones(n_pages * page, dtype=torch.bool, device="cuda")
    other[slots] = False                        # nothing else was written
    rest = other.nonzero().flatten()
    zk, zv = ops.kv4_read(cache, rest)
    assert (zk == 0).all() and (zv == 0).all() and (before == 0).all()
    for out in (BF16, F16):
        rk2, rv2 = ops.kv4_read(cache, slots, dtype=out)
        assert torch.equal(rk2, rk.to(out)) and torch.equal(rv2, rv.to(out))
    assert ops.device_status() == 0


def test_kv4_block_layout():
    """The bytes are the ones the header states."""
    g = gen(2)
    d, ng = 128, 4
    k, v = randn(g, 16, 1, d), randn(g, 16, 1, d)
    cache = ops.kv4_cache(1, 1, d, 16)
    ops.kv4_append(cache, k, v, torch.arange(16, device="cuda"))
    b = cache.cpu().numpy().reshape(-1)
    words = lambda at: b[at:at + 8 * d].view(np.uint32).reshape(2, 8, 4, ng)  # noqa: E731
    quad = lambda at: b[at:at + d].view(np.float16).reshape(4, ng, 2, 2)      # noqa: E731
    kc, ks, km, vc, vs, vm = words(0), quad(8 * d), b[9 * d:10 * d].view(np.float16).reshape(8, 2, ng), words(10 * d), \
        quad(18 * d), quad(19 * d)
    for x, name in ((k, "k"), (v, "v")):
        c, s, m = (y[:, 0].numpy() for y in quantized(x))
        for t in range(16):
            j, n, q, e = t // 8, t % 8, t % 8 // 2, t % 2
            for ch in range(d):
                g_, r = ch // 32, ch % 32
                code = kc[j, n, r // 8, g_] >> (4 * (r % 8)) if name == "k" else vc[j, r // 4, q, g_] >> (4 * (4 * e + r % 4))
                assert code & 15 == c[t, g_, r]
            for g_ in range(ng):
                assert (ks if name == "k" else vs)[q, g_, j, e] == s[t, g_]
                assert (km[n, j, g_] if name == "k" else vm[q, g_, j, e]) == m[t, g_]


def test_kv4_special_values_and_slots():
    cache = ops.kv4_cache(2, 1, 64, 16)
    k, v = torch.zeros(6, 1, 64, device="cuda"), torch.zeros(6, 1, 64, device="cuda")
    k[0, 0, 3], k[1, 0, 40], v[2, 0, 0] = math.nan, math.inf, -math.inf
    k[3, 0, :32] = 3e38 * torch.linspace(-1, 1, 32, device="cuda")          # past fp16: clamped, finite
    k[4], v[5] = 1.5, -2.0
    slots = torch.tensor([0, 31, 7, 8, -1, 20], device="cuda")
    ops.kv4_append(cache, k, v, slots)
    assert ops.device_status() == 0
    rk, rv = ops.kv4_read(cache, slots)
    assert rk[0, 0, :32].isnan().all() and (rk[0, 0, 32:] == 0).all() and rk[1, 0, 32:].isnan().all()
    assert rv[2, 0, :32].isnan().all() and (rv[2, 0, 32:] == 0).all()
    assert rk[3].isfinite().all() and rk[3, 0, 0] == -65504 and abs(float(rk[3, 0, 31]) - 65504) <= 64
    assert (rk[4] == 0).all() and (rv[4] == 0).all() and (rv[5] == -2).all()
    ops.kv4_append(cache, k[:1], v[:1], torch.tensor([32], device="cuda"))  # past the cache: skipped, reported
    assert ops.device_status() == 2 and ops.device_status() == 0
    zk, _ = ops.kv4_read(cache, torch.tensor([32], device="cuda"))
    assert (zk == 0).all() and ops.device_status() == 2
    ops.kv4_append(cache, k[:0], v[:0], slots[:0])


def test_kv4_append_strides():
    g = gen(4)
    T, nkv, d = 21, 3, 64
    qkv = randn(g, T, 9 + 2 * nkv, d, dtype=BF16)
    odd = randn(g, T, 2 * nkv, d + 1, dtype=BF16)
    slots = torch.arange(T, device="cuda") + 5
    for k, v in ((qkv[:, 9:9 + nkv], qkv[:, 9 + nkv:]), (odd[:, :nkv, 1:], odd[:, nkv:, :d])):
        cache = ops.kv4_cache(3, nkv, d, 16)
        ops.kv4_append(cache, k, v, slots)
        rk, rv = ops.kv4_read(cache, slots)
        assert torch.equal(rk.cpu(), values(k)) and torch.equal(rv.cpu(), values(v))


def make_cache(g, lens, nkv, d, page, spread=1.0, extra=2):
    """A cache whose pages lie anywhere, holding random keys and values; the unused bytes are garbage."""
    pages = [-(-n // page) for n in lens]
    n_pages = sum(pages) + extra
    cache = ops.kv4_cache(n_pages, nkv, d, page)
    cache.random_(0, 256, generator=g)
    cache[..., 8 * d:10 * d] = 0xFF          # NaN scales and minima where nothing is written
    cache[..., 18 * d:] = 0xFF
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    table = torch.full((len(lens), max(max(pages), 1)), -7, dtype=torch.int32, device="cuda")
    kv, used = [], 0
    for b, n in enumerate(lens):
        table[b, :pages[b]] = order[used:used + pages[b]]
        used += pages[b]
        k = randn(g, n, nkv, d) + 0.5 * randn(g, 1, nkv, d)
        v = randn(g, n, nkv, d) * spread
        at = torch.arange(n, device="cuda")
        ops.kv4_append(cache, k, v, table[b].long()[at // page] * page + at % page)
        kv.append((k, v))
    return cache, table, kv


def check_decode(q, cache, table, kv, causal, scale=None):
    B, lq, nq, d = q.shape
    nkv = cache.shape[1]
    lens = torch.tensor([k.shape[0] for k, _ in kv], dtype=torch.int32, device="cuda")
    got = ops.kv4_attention(q, cache, table, lens, scale=scale, causal=causal)
    assert got.shape == q.shape and got.dtype == q.dtype and ops.device_status() == 0
    sc = 1 / math.sqrt(d) if scale is None else scale
    off = size = 0.0
    for b, (k, v) in enumerate(kv):
        k, v = values(k).cuda(), values(v).cuda()
        lim = limits(lq, k.shape[0], causal, 0)
        for h in range(nq):
            kh = h // (nq // nkv)
            o, a = attend(q[b, :, h], k[:, kh], v[:, kh], lim, sc)
            w = 2.0 ** -11 if q.dtype == BF16 else 0.0
            # a code times its scale is at most |v| + |m|, and |m| is below 5 sigma here: twice A and a little
            assert_within(got[b, :, h], o, U[q.dtype] * o.abs() + (2.0 ** -12 + w) * (2 * a + a.amax(-1, keepdim=True)) + 1e-30)
            off += float((got[b, :, h].double() - o).square().sum())
            size += float(o.square().sum())
    if q.dtype == F32 and size:
        assert math.sqrt(off / size) <= 5e-6
    return got


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("lens,nq,nkv,d,page", [
    ([1], 1, 1, 64, 16), ([1, 0, 2], 15, 5, 64, 16), ([15, 16, 17], 8, 1, 128, 32), ([63, 64, 65, 255], 32, 8, 128, 64),
    ([256, 257, 1000], 12, 4, 128, 16), ([4097], 5, 5, 64, 128), ([300, 20], 28, 4, 128, 256), ([777], 33, 1, 64, 64),
    ([9000], 4, 1, 128, 64),
])
def test_kv4_attention_single_token(dtype, lens, nq, nkv, d, page):
    g = gen(sum(lens) + d)
    cache, table, kv = make_cache(g, lens, nkv, d, page)
    q = randn(g, len(lens), 1, nq, d, dtype=dtype)
    got = check_decode(q, cache, table, kv, True)
    assert torch.equal(ops.kv4_attention(q[:, 0], cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda")), got[:, 0])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,lq,nq,nkv,d", [([241, 33, 3, 0], 50, 15, 5, 64), ([130, 70], 3, 8, 2, 128), ([600], 17, 4, 4, 64)])
def test_kv4_attention_chunk(dtype, causal, lens, lq, nq, nkv, d):
    g = gen(lq)
    cache, table, kv = make_cache(g, lens, nkv, d, 32)
    wide = randn(g, len(lens), lq, nq + 3, d, dtype=dtype)
    got = check_decode(wide[:, :, :nq], cache, table, kv, causal)
    for b, n in enumerate(lens):
        empty = torch.from_numpy(limits(lq, n, causal, 0) == 0).cuda()
        assert (got[b][empty] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("spread", [1e-4, 300.0])
def test_kv4_attention_value_ranges(dtype, spread):
    """Values whose scales lie near fp16's ends, queries of any size, scores of any sign."""
    g = gen(12)
    cache, table, kv = make_cache(g, [500], 2, 64, 64, spread=spread)
    q = randn(g, 1, 1, 8, 64, dtype=dtype)
    check_decode(q, cache, table, kv, True)
    check_decode(q, cache, table, kv, True, scale=-0.5)
    if dtype != F16:
        check_decode(q * 1e-12, cache, table, kv, True, scale=1e11)
        check_decode(q * 1e12, cache, table, kv, True, scale=1e-13)


def test_kv4_attention_values_grow_along_the_sequence():
    g = gen(13)
    cache, table, kv = make_cache(g, [900], 1, 64, 64)
    k, v = kv[0]
    v = v * torch.logspace(-5, 4, 900, device="cuda")[:, None, None]
    at = torch.arange(900, device="cuda")
    ops.kv4_append(cache, k, v, table[0].long()[at // 64] * 64 + at % 64)
    check_decode(randn(g, 1, 1, 4, 64), cache, table, [(k, v)], True)


def test_kv4_attention_nan_stays_where_it_is():
    g = gen(14)
    cache, table, kv = make_cache(g, [100, 100], 2, 64, 16)
    q = randn(g, 2, 8, 4, 64)
    clean = check_decode(q, cache, table, kv, True)
    k, v = kv[0][0].clone(), kv[0][1].clone()
    v[96, 0, 5], k[97, 1, 60] = math.nan, math.inf
    at = torch.arange(100, device="cuda")
    ops.kv4_append(cache, k, v, table[0].long()[at // 16] * 16 + at % 16)
    lens = torch.tensor([100, 100], dtype=torch.int32, device="cuda")
    got = ops.kv4_attention(q, cache, table, lens)
    assert torch.equal(got[1], clean[1])
    assert torch.equal(got[0, :3], clean[0, :3])              # tokens 92 .. 94 see neither
    assert got[0, 4:, :2, :32].isnan().all() and got[0, 4:, :2, 32:].isfinite().all()
    assert got[0, 5:, 2:].isnan().all() and got[0, :5, 2:].isfinite().all()


def test_kv4_attention_bad_page_is_left_out():
    g = gen(15)
    cache, table, kv = make_cache(g, [40], 1, 64, 16)
    q = randn(g, 1, 1, 2, 64)
    lens = torch.tensor([40], dtype=torch.int32, device="cuda")
    bad = table.clone()
    bad[0, 1] = 10 ** 6
    got = ops.kv4_attention(q, cache, bad, lens)
    assert ops.device_status() == 2 and got.isfinite().all()
    more = torch.tensor([4000], dtype=torch.int32, device="cuda")   # a length past the table is the table's end
    full = torch.cat([table[:, :2], table[:, :1]], 1).contiguous()
    assert torch.equal(ops.kv4_attention(q, cache, full, more, causal=False),
                       ops.kv4_attention(q, cache, full, torch.tensor([48], dtype=torch.int32, device="cuda"), causal=False))


def test_kv4_attention_repeats_bit_for_bit():
    g = gen(16)
    cache, table, kv = make_cache(g, [5000, 300, 1200], 4, 128, 64)
    q = randn(g, 3, 1, 16, 128, dtype=BF16)
    lens = torch.tensor([5000, 300, 1200], dtype=torch.int32, device="cuda")
    first = ops.kv4_attention(q, cache, table, lens)
    for _ in range(5):
        assert torch.equal(ops.kv4_attention(q, cache, table, lens), first)


# ---------------------------------------------------------------- refusals

def test_refusals():
    x = torch.zeros(2, 4, 64, device="cuda")
    pos = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    for bad in (dict(sections=(33,)), dict(sections=()), dict(sections=(0,)), dict(sections=(8,) * 2), dict(pos=pos.long()),
                dict(k=x[:1]), dict(k=x.half()), dict(q_weight=torch.ones(63, device="cuda")), dict(eps=-1.0),
                dict(base=0.0), dict(out_dtype=torch.float64), dict(q=x.double(), k=x.double()), dict(q=x[0])):
        with pytest.raises((ValueError, VlaError)):
            ops.qk_norm_rope(**{**dict(q=x, k=x, pos=pos, sections=(32,)), **bad})
    with pytest.raises((ValueError, VlaError)):
        ops.qk_norm_rope(x[..., :63], None, pos, (8,))
    h = x.to(BF16)
    cu = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    for bad in (dict(q=x, k=x, v=x), dict(k=h[..., :32].contiguous()), dict(v=h.half()), dict(k=h[:, :3], v=h[:, :3]),
                dict(cu_q=cu.long()), dict(cu_k=cu[:1]), dict(prefix=cu), dict(scale=math.inf), dict(cu_q=cu[:0]),
                dict(q=h.cpu())):
        with pytest.raises((ValueError, VlaError)):
            ops.prompt_attention(**{**dict(q=h, k=h, v=h, cu_q=cu), **bad})
    for d in (12, 136):
        y = torch.zeros(2, 1, d, dtype=BF16, device="cuda")
        with pytest.raises(VlaError) as e:
            ops.prompt_attention(y, y, y, cu)
        assert e.value.code == VLA_ERR_ARG
    for n in ((2, 1, 96), (2, 1, 64, 24), (2, 1, 64, 8)):
        with pytest.raises(ValueError):
            ops.kv4_cache(*n)
    cache = ops.kv4_cache(2, 4, 64, 16)
    slots = torch.arange(2, device="cuda")
    for bad in (dict(k=x[:, :3]), dict(v=x.half()), dict(slots=slots.int()), dict(slots=slots[:1]), dict(cache=cache.float()),
                dict(cache=cache[..., ::2]), dict(k=x.double(), v=x.double()), dict(k=x.cpu())):
        with pytest.raises((ValueError, VlaError)):
            ops.kv4_append(**{**dict(cache=cache, k=x, v=x, slots=slots), **bad})
    with pytest.raises(ValueError):
        ops.kv4_read(cache, slots, dtype=torch.int32)
    table, lens = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    for bad in (dict(q=x[..., :32]), dict(q=x[:, :3]), dict(q=x.double()), dict(table=table.long()), dict(table=table[:1]),
                dict(lens=lens.long()), dict(lens=lens[:1]), dict(scale=math.nan), dict(q=x.cpu())):
        with pytest.raises((ValueError, VlaError)):
            ops.kv4_attention(**{**dict(q=x, cache=cache, table=table, lens=lens), **bad})
    big = torch.zeros(1, 70000, 32, 64, device="cuda", dtype=BF16)
    with pytest.raises(VlaError) as e:
        ops.kv4_attention(big, ops.kv4_cache(2, 4, 64, 16), table[:1], lens[:1])
    assert e.value.code == VLA_ERR_SHAPE


def test_c_refusals():
    """The C entries refuse without launching: null pointers, addresses and strides that do not fit, short workspaces."""
    L = lib()
    h = torch.zeros(4, 2, 64, dtype=BF16, device="cuda")
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    p, c = h.data_ptr(), cu.data_ptr()

    def prompt(out=p, q=p, qt=128, qh=64, k=p, typ=2, cq=c, n_seq=1, tq=4, d=64, nq=2, nkv=2):
        return L.vla_cuda_prompt_attention(out, q, qt, qh, k, 128, 64, p, 128, 64, typ, cq, c, None, n_seq, tq, 4, nq, nkv,
                                           d, 0.125, 1, None)

    for bad in (dict(out=None), dict(q=None), dict(q=p + 2), dict(qt=130), dict(qh=-64), dict(k=None), dict(typ=0), dict(typ=3),
                dict(cq=None), dict(n_seq=-1), dict(tq=-1), dict(d=0), dict(nq=3), dict(nkv=0), dict(out=p + 8)):
        assert prompt(**bad) == VLA_ERR_ARG, bad
    assert prompt(tq=0, q=None) == 0 and prompt(n_seq=0, cq=None) == 0
    cache = ops.kv4_cache(64, 2, 64, 128)
    table = torch.zeros(1, 64, dtype=torch.int32, device="cuda")
    lens = torch.tensor([8192], dtype=torch.int32, device="cuda")
    need = L.vla_cuda_kv4_attention_workspace_bytes(1, 1, 2, 2, 64, 64, 128)
    assert need > 0
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")

    def decode(page=128, cache=cache.data_ptr(), ld=64, ws=ws.data_ptr(), size=need, table=table.data_ptr()):
        return L.vla_cuda_kv4_attention(p, p, 128, 0, 64, 2, cache, 64, page, table, ld, 64, lens.data_ptr(), 1, 1, 2, 2, 64,
                                        0.125, 1, ws, size, None)

    for bad in (dict(page=48), dict(page=8), dict(cache=None), dict(cache=cache.data_ptr() + 4), dict(ld=63), dict(ws=None),
                dict(size=need - 1), dict(ws=ws.data_ptr() + 4), dict(table=None)):
        assert decode(**bad) == VLA_ERR_ARG, bad
    assert decode() == 0
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("power", [-121, -117, -110, 105, 110, 120, 122])
def test_kv4_attention_queries_of_any_size(dtype, power):
    """Queries near the ends of their type, the scale as far the other way: scores of ordinary size."""
    g = gen(18)
    cache, table, kv = make_cache(g, [300], 2, 64, 64)
    q = randn(g, 1, 1, 4, 64, dtype=dtype).clamp(-7.9, 7.9).double() * 2.0 ** power
    check_decode(q.to(dtype), cache, table, kv, True, scale=2.0 ** (-power - 3))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T", [1000, 4096, 16384])
@pytest.mark.parametrize("rest", [1 / 8, 1 / 90, 1 / 400])
def test_prompt_many_small_weights_beside_a_large_one(dtype, T, rest):
    """A first key of nearly all the weight, and the others, which share `rest` of it: down to 2^-22 each, in channels
    that the first key's value may leave to them alone."""
    g = gen(19)
    d = 64
    q, k = torch.zeros(3, 1, d, device="cuda", dtype=dtype), torch.zeros(T, 1, d, device="cuda", dtype=dtype)
    q[:, 0, 0], q[:, 0, 1] = 1.0, 0.03125
    score = -math.log(rest / T)
    k[0, 0, 0] = math.floor(score)                                  # the score in two parts that bf16 holds
    k[0, 0, 1] = 32 * (score - math.floor(score))
    v = (1.0 + randn(g, T, 1, d)).to(dtype)
    check_prompt(q, k, v, [3], [T], causal=False, scale=1.0)
    check_prompt(q, k, torch.ones_like(v), [3], [T], causal=False, scale=1.0)
