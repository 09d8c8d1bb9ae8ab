"""examples/prompted_decoder.py: what does not fit its cache is refused on the host, before anything is launched."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

import prompted_decoder as ex  # noqa: E402


@pytest.fixture
def dec(monkeypatch):
    """A decoder of 2 sequences of at most 48 tokens whose layers stay on the host."""
    monkeypatch.setattr(ex.ops, "pack_weights_i8", lambda w: (w, w))
    monkeypatch.setattr(ex.ops, "kv4_cache", lambda *a: None)
    monkeypatch.setattr(ex.ops, "dense_linear_i8", lambda h, w, s: h)
    for name in ("ones", "zeros", "randn", "arange", "tensor", "Generator"):
        real = getattr(torch, name)
        monkeypatch.setattr(torch, name, lambda *a, _real=real, **kw: _real(*a, **{**kw, **({"device": "cpu"} if "device" in kw else {})}))
    d = ex.PromptedDecoder(layers=1, hidden=32, n_q=2, n_kv=1, ffn=8, vocab=8, batch=2, max_tokens=40, page=16)
    d._layers = lambda x, pos, slots, attend: x
    return d


def prompt(dec, lens, rows=None, axes=3):
    n = sum(lens) if rows is None else rows
    return dec.prompt(torch.zeros(n, 32), lens, torch.zeros(axes, n, dtype=torch.int32), None)


def test_lengths_that_fit(dec):
    prompt(dec, [46, 3])
    step = torch.zeros(2, dtype=torch.long)
    dec.step(step)
    dec.step(step)
    assert dec.lens.tolist() == [48, 5]
    with pytest.raises(ValueError, match="does not fit"):
        dec.step(step)
    assert dec.lens.tolist() == [48, 5]
    prompt(dec, [1, 1])                      # a new batch starts over
    dec.step(step)


@pytest.mark.parametrize("lens,rows,axes", [([49, 3], None, 3), ([3, 1000], None, 3), ([3], None, 3), ([1, 2, 3], None, 3),
                                            ([4, 0], None, 3), ([], 0, 3), ([4, 4], 7, 3), ([4, 4], None, 2)])
def test_prompts_that_do_not_fit(dec, lens, rows, axes):
    with pytest.raises(ValueError):
        prompt(dec, lens, rows, axes)


def test_steps_of_another_batch(dec):
    prompt(dec, [4, 4])
    for n in (1, 3):
        with pytest.raises(ValueError):
            dec.step(torch.zeros(n, dtype=torch.long))
