"""Attention over prompts and over the 4-bit cache where keys or queries are not finite.

A row that sees a score of NaN or +infinity is NaN; a score of -infinity beside finite ones weighs nothing; a row
that sees nothing is zeros, and what a row does not see does not change it. That is what a softmax in 64 bits gives,
and the finite rows hold the tolerances of the finite tests.
"""
import math

import pytest
import torch

from test_serve_ops_gpu import BF16, F16, U, assert_within, attend, gen, limits, randn
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
