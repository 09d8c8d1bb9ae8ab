"""Attention over prompts and over the 4-bit cache where keys or queries are not finite.

A row that sees a score of NaN or +infinity is NaN; a score of -infinity beside finite ones weighs nothing; a row
that sees nothing is zeros, and what a row does not see does not change it. That is what a softmax in 64 bits gives,
and the finite rows hold the tolerances of the finite tests.
"""
import math

import pytest
import torch

from test_serve_ops_gpu import BF16, F16, F32, U, assert_within, attend, gen, limits, randn
from vla_simd_b200 import ops

pytestmark = pytest.mark.gpu


def check_prompt_rows(q, k, v, lq, causal=True, prefix=0):
    """One sequence whose last query sees the last key; returns how many rows are NaN."""
    lk, d = k.shape[0], q.shape[2]
    cq, ck = (torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (lq, lk))
    pre = torch.tensor([prefix], dtype=torch.int32, device="cuda") if prefix else None
    got = ops.prompt_attention(q, k, v, cq, ck, causal=causal, prefix=pre)
    lim, group, nan = limits(lq, lk, causal, prefix), q.shape[1] // k.shape[1], 0
    for h in range(q.shape[1]):
        o, a = attend(q[:, h], k[:, h // group], v[:, h // group], lim, d ** -0.5)
        assert torch.equal(got[:, h].isnan(), o.isnan())
        tol = U[q.dtype] * (o.abs() + a) + 2.0 ** -12 * a + 1e-30
        assert_within(got[:, h].double().nan_to_num(0.0), o.nan_to_num(0.0), tol.nan_to_num(0.0))
        nan += int(o.isnan().any(-1).sum())
    assert ops.device_status() == 0
    return nan


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("fill", [math.nan, math.inf, -math.inf])
def test_prompt_bad_key_at_each_position(dtype, d, fill):
    """A bad key alone at each of 16 positions in a row, in steps that rows see in full and in masked ones."""
    g = gen(21)
    T, nq, nkv = 200, 4, 2
    q, k, v = randn(g, T, nq, d, dtype=dtype), randn(g, T, nkv, d, dtype=dtype), randn(g, T, nkv, d, dtype=dtype)
    for at in [*range(16), *range(48, 64), *range(64, 80), 127, 128, 199]:
        bad = k.clone()
        bad[at, 0, at % d] = fill
        nan = check_prompt_rows(q, bad, v, T)
        if math.isnan(fill):
            assert nan == 2 * (T - at)
        assert check_prompt_rows(q[:1], bad, v, 1) == (2 if math.isnan(fill) else int((q[0, :2, at % d] * fill > 0).sum()))
    bad = k.clone()
    bad[70:80, 1] = fill                     # a run of keys, every channel, dense and behind a prefix
    check_prompt_rows(q, bad, v, T, causal=False)
    check_prompt_rows(q, bad, v, T, prefix=90)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prompt_bad_query(dtype):
    g = gen(22)
    T, d = 300, 64
    q, k, v = (randn(g, T, n, d, dtype=dtype) for n in (3, 3, 3))
    bad = q.clone()
    bad[7, 0, 3], bad[0, 1, 0] = math.nan, math.nan
    bad[299, 2, 63], bad[150, 1, 9] = math.inf, -math.inf      # an infinity meets keys of both signs
    assert check_prompt_rows(bad, k, v, T) == 4
    assert check_prompt_rows(bad, k, v, T, causal=False) == 4


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prompt_scores_of_minus_infinity(dtype):
    """Rows that score -infinity throughout are NaN, with finite keys in front or behind they are those keys' rows."""
    g = gen(23)
    T, d = 330, 64
    q, k, v = (randn(g, T, 1, d, dtype=dtype) for _ in range(3))
    q[:, 0, 5] = q[:, 0, 5].abs() + 0.5
    first = k.clone()
    first[:129, 0, 5] = -math.inf
    assert check_prompt_rows(q, first, v, T) == 129
    last = k.clone()
    last[100:, 0, 5] = -math.inf
    assert check_prompt_rows(q, last, v, T) == 0
    # the same where a hidden NaN in a value sends a tile's rows the other way
    hidden = v.clone()
    hidden[250] = math.nan
    assert check_prompt_rows(q, first, hidden, T) == 129 + T - 250
    assert check_prompt_rows(q, last, hidden, T) == T - 250


# ---------------------------------------------------------------- 4-bit cache

def cache_of(k, v, page=32):
    """One sequence's keys and values [T, n_kv, d] in a cache, its pages backwards."""
    T, nkv, d = k.shape
    pages = -(-T // page)
    cache = ops.kv4_cache(pages, nkv, d, page)
    table = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device="cuda")[None].contiguous()
    at = torch.arange(T, device="cuda")
    slots = table[0].long()[at // page] * page + at % page
    ops.kv4_append(cache, k, v, slots)
    return cache, table, *ops.kv4_read(cache, slots)


def check_cache_rows(q, k, v, causal=True):
    """q [queries, n_q, d] over one sequence; returns how many rows are NaN in every channel."""
    cache, table, k, v = cache_of(k, v)
    lq, nq, d = q.shape
    got = ops.kv4_attention(q[None], cache, table, torch.tensor([k.shape[0]], dtype=torch.int32, device="cuda"), causal=causal)[0]
    group, lim, nan = nq // k.shape[1], limits(lq, k.shape[0], causal, 0), 0
    for h in range(nq):
        o, a = attend(q[:, h], k[:, h // group], v[:, h // group], lim, d ** -0.5)
        assert torch.equal(got[:, h].isnan(), o.isnan())
        w = 2.0 ** -11 if q.dtype == BF16 else 0.0
        a = a.nan_to_num(0.0)
        tol = U[q.dtype] * o.abs().nan_to_num(0.0) + (2.0 ** -12 + w) * (2 * a + a.amax(-1, keepdim=True)) + 1e-30
        assert_within(got[:, h].double().nan_to_num(0.0), o.nan_to_num(0.0), tol)
        nan += int(o.isnan().all(-1).sum())
    assert ops.device_status() == 0
    return nan


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T", [1, 33, 300, 4000])
def test_cache_bad_query(dtype, d, T):
    g = gen(31)
    k, v = randn(g, T, 2, d), randn(g, T, 2, d)
    for fill in (math.nan, math.inf, -math.inf):
        q = randn(g, 3, 6, d, dtype=dtype)
        q[2, 1, 5], q[1, 4, d - 1] = fill, fill
        # an infinity times keys of one sign is no NaN by itself, but its row has no finite maximum
        assert check_cache_rows(q, k, v) == (2 if T > 1 else 1) and check_cache_rows(q, k, v, causal=False) == 2


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T,bad", [
    (1, slice(0, 1)),            # the only key
    (16, slice(0, 16)),          # all of them
    (300, slice(32, 64)),        # a tile of a warp
    (300, slice(288, 300)),      # the last few
    (300, slice(7, 8)),          # one among others
    (4000, slice(0, 1024)),      # whole chunks of a split call
    (4000, slice(2048, 4000)),
    (4000, slice(3999, 4000)),
])
def test_cache_bad_keys(dtype, d, T, bad):
    g = gen(32)
    k, v, q = randn(g, T, 2, d), randn(g, T, 2, d), randn(g, 4, 4, d, dtype=dtype)
    k[bad, 0, 3] = math.nan
    seen = sum(n > bad.start for n in limits(4, T, True, 0))
    assert check_cache_rows(q, k, v) == 2 * seen and check_cache_rows(q, k, v, causal=False) == 8


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_cache_bad_keys_and_values_that_weigh_next_to_nothing(dtype):
    """Warps and chunks whose finite scores are hundreds below another's still bring their NaN along."""
    g = gen(33)
    T, d = 4000, 64
    q = randn(g, 1, 2, d, dtype=dtype).abs() + 0.5
    k, v = randn(g, T, 2, d), randn(g, T, 2, d)
    k[70] += 60.0
    bad = k.clone()
    bad[[10, 3000], 0, 9] = math.nan
    assert check_cache_rows(q, bad, v) == 1
    assert check_cache_rows(q, bad[:200], v[:200]) == 1
    bad = v.clone()
    bad[[10, 3000], 0, 9] = math.nan         # 32 channels of a value, not the row
    assert check_cache_rows(q, k, bad) == 0


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_rows_before_a_hidden_value_keep_their_bits(dtype, d):
    """A NaN in a value that a whole tile of rows does not multiply changes none of its bits, in any run."""
    g = gen(24)
    T = 512
    q, k, v = (randn(g, T, 8, d, dtype=dtype) for _ in range(3))
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    clean = ops.prompt_attention(q, k, v, cu)
    bad = v.clone()
    bad[200], bad[T - 1] = math.nan, math.inf
    first = ops.prompt_attention(q, k, bad, cu)
    assert torch.equal(first[:128], clean[:128]) and first[200:].isnan().any(-1).all()
    for _ in range(20):
        assert torch.equal(ops.prompt_attention(q, k, bad, cu).nan_to_num(9.0), first.nan_to_num(9.0))
