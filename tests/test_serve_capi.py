"""The prompt and 4-bit cache entries of the C ABI, as far as they go without a GPU: sizes and refusals."""
import ctypes

import pytest

from vla_simd_b200 import VLA_ERR_ARG, VLA_ERR_SHAPE, lib

P = 4096   # an aligned address that a refused call never reads


def rope(L, tokens=1, n_q=1, n_kv=1, d=64, sections=(32,), in_type=0, out_type=0, q=P, pos=P, eps=1e-6, base=1e4, axes=None):
    s = (ctypes.c_int32 * max(len(sections), 1))(*sections)
    return L.vla_cuda_qk_norm_rope(P, P, out_type, q, 64, 64, P, 64, 64, in_type, pos, s, len(sections) if axes is None else axes,
                                   0, None, None, eps, base, tokens, n_q, n_kv, d, None)


@pytest.mark.parametrize("bad", [
    dict(tokens=-1), dict(n_q=-1), dict(n_kv=70000), dict(d=0), dict(d=63), dict(d=258), dict(sections=(33,)),
    dict(sections=(16, 17)), dict(sections=(0,)), dict(sections=(32, -1)), dict(sections=(), axes=0), dict(sections=(1,) * 5),
    dict(in_type=3), dict(out_type=-1), dict(q=None), dict(pos=None), dict(eps=-1.0), dict(eps=float("nan")), dict(base=0.0),
    dict(base=float("inf")),
])
def test_rope_refuses(bad):
    assert rope(lib(), **bad) == VLA_ERR_ARG


def prompt(L, out=P, q=P, qt=128, qh=64, k=P, kt=128, typ=2, cu=P, n_seq=1, tq=4, tk=4, n_q=2, n_kv=2, d=64, scale=0.125):
    return L.vla_cuda_prompt_attention(out, q, qt, qh, k, kt, 64, P, 128, 64, typ, cu, P, None, n_seq, tq, tk, n_q, n_kv, d,
                                       scale, 1, None)


@pytest.mark.parametrize("bad", [
    dict(out=None), dict(out=P + 8), dict(q=None), dict(q=P + 2), dict(qt=0), dict(qt=132), dict(qh=-64), dict(k=None), dict(kt=4),
    dict(typ=0), dict(typ=3), dict(cu=None), dict(n_seq=-1), dict(tq=-1), dict(tk=-1), dict(n_q=3), dict(n_kv=0), dict(n_q=0),
    dict(d=0), dict(d=12), dict(d=136), dict(scale=float("inf")), dict(scale=float("nan")),
])
def test_prompt_refuses(bad):
    assert prompt(lib(), **bad) == VLA_ERR_ARG


def test_nothing_to_do_is_no_error():
    assert rope(lib(), tokens=0, q=None, pos=None) == 0
    assert prompt(lib(), tq=0, q=None) == 0 and prompt(lib(), n_seq=0, cu=None) == 0
    assert decode(lib(), batch=0, q=None) == 0 and decode(lib(), queries=0, q=None) == 0
    assert append(lib(), tokens=0, k=None, slots=None) == 0


def append(L, cache=P, n_pages=4, page=16, k=P, typ=0, slots=P, tokens=1, n_kv=1, d=64):
    return L.vla_cuda_kv4_append(cache, n_pages, page, k, 64, 64, P, 64, 64, typ, slots, tokens, n_kv, d, None)


@pytest.mark.parametrize("bad", [
    dict(cache=None), dict(cache=P + 4), dict(n_pages=0), dict(page=8), dict(page=48), dict(page=512), dict(k=None), dict(typ=3),
    dict(slots=None), dict(tokens=-1), dict(n_kv=0), dict(d=32), dict(d=96), dict(n_pages=2 ** 31 // 16),
])
def test_append_refuses(bad):
    assert append(lib(), **bad) == VLA_ERR_ARG


def decode(L, q=P, cache=P, page=16, table=P, ld=4, pages=4, lens=P, batch=1, queries=1, n_q=2, n_kv=2, d=64, scale=0.1, ws=None):
    return L.vla_cuda_kv4_attention(P, q, 128, 128, 64, 0, cache, 64, page, table, ld, pages, lens, batch, queries, n_q, n_kv, d,
                                    scale, 1, ws, 0, None)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(cache=None), dict(page=17), dict(table=None), dict(ld=3), dict(pages=-1), dict(lens=None), dict(batch=-1),
    dict(batch=70000), dict(queries=-1), dict(n_q=3), dict(d=80), dict(scale=float("nan")), dict(ws=P + 8),
    dict(pages=64, ld=64),   # more than one chunk: a workspace is needed
])
def test_decode_refuses(bad):
    assert decode(lib(), **bad) == VLA_ERR_ARG


def test_decode_refuses_too_many_rows():
    assert decode(lib(), queries=600000) == VLA_ERR_SHAPE


def test_sizes():
    L = lib()
    assert [L.vla_cuda_kv4_block_bytes(d) for d in (64, 128, 32, 96)] == [1280, 2560, 0, 0]
    size = L.vla_cuda_kv4_attention_workspace_bytes
    assert size(1, 1, 32, 8, 128, 1, 128) == 0 and size(1, 1, 32, 8, 128, 0, 64) == 0 and size(1, 1, 3, 2, 64, 8, 64) == 0
    # (head_dim + 2) fp32 for each row and chunk
    assert size(1, 1, 32, 8, 128, 64, 128) % (4 * 130 * 32) == 0 and size(1, 1, 32, 8, 128, 64, 128) > 0


@pytest.mark.parametrize("page", [16, 256])
def test_decode_refuses_tables_whose_keys_pass_32_bits(page):
    """A chunk past the last key of 2^31 would have no 32-bit number: at most 2^30 tokens a sequence."""
    L = lib()
    most = 2 ** 30 // page
    size = L.vla_cuda_kv4_attention_workspace_bytes
    assert size(1, 1, 2, 2, 64, most, page) > 0 and size(1, 1, 2, 2, 64, most + 1, page) == 0

    def call(pages):   # batch 0: nothing is launched
        return L.vla_cuda_kv4_attention(P, P, 128, 128, 64, 0, P, 64, page, P, pages, pages, P, 0, 1, 2, 2, 64, 0.1, 1, P, 0, None)

    assert call(most) == 0
    for pages in (most + 1, (2 ** 31 - 1) // page):
        assert call(pages) == VLA_ERR_ARG


def test_prompt_refuses_totals_past_32_bits():
    """Rounded up to whole tiles, a total near 2^31 would be negative."""
    for n in (2 ** 30 + 1, 2 ** 31 - 1):
        assert prompt(lib(), tq=n, n_seq=0) == VLA_ERR_ARG and prompt(lib(), tk=n, n_seq=0) == VLA_ERR_ARG
    assert prompt(lib(), tq=2 ** 30, tk=2 ** 30, n_seq=0) == 0   # no sequence: nothing is launched


@pytest.mark.parametrize("batch,queries,n_q,n_kv,d,pages,page,chunks", [
    (1, 1, 15, 5, 64, 64, 16, 8), (8, 50, 15, 5, 64, 5, 64, 1), (16, 1, 32, 8, 128, 128, 64, 8), (48, 1, 32, 8, 128, 128, 128, 4),
])
def test_chunks_that_the_stated_times_speak_of(batch, queries, n_q, n_kv, d, pages, page, chunks):
    size = lib().vla_cuda_kv4_attention_workspace_bytes(batch, queries, n_q, n_kv, d, pages, page)
    assert size == (0 if chunks == 1 else batch * queries * n_q * chunks * (d + 2) * 4)
