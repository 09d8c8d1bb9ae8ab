"""Op-level wrappers over include/vla_simd_cuda.h for torch CUDA tensors.

Each function mirrors one reference op (src/ops/quant_ops.h, lm_ops.h,
conv_ops.h) - same argument meaning, the outputs allocated here for
convenience - and launches on torch's current stream. torch supplies device
memory and the stream handle only; the compute is the library's kernels.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import EPI_ACC, check, lib


def _p(t):
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def i8_ld(K: int) -> int:
    return int(lib().vla_cuda_i8_ld(K))


def quantize_act_i8(x: torch.Tensor, ld: int | None = None):
    """x [seq, K] fp32 -> (xq [seq, ld] int8, ascale [seq] fp32)."""
    seq, K = x.shape
    ld = ld or i8_ld(K)
    xq = torch.empty((seq, ld), dtype=torch.int8, device=x.device)
    s = torch.empty(seq, dtype=torch.float32, device=x.device)
    check(lib().vla_cuda_quantize_act_i8(_p(x.contiguous()), _p(xq), _p(s), seq, K, ld, _stream()),
          "vla_cuda_quantize_act_i8")
    return xq, s


def pack_weights_i8(W: torch.Tensor, ld: int | None = None):
    """W [N, K] fp32 -> (Wq [N, ld] int8, wscale [N])."""
    N, K = W.shape
    ld = ld or i8_ld(K)
    q = torch.empty((N, ld), dtype=torch.int8, device=W.device)
    s = torch.empty(N, dtype=torch.float32, device=W.device)
    check(lib().vla_cuda_pack_weights_i8(_p(W.contiguous()), _p(q), _p(s), N, K, ld, _stream()),
          "vla_cuda_pack_weights_i8")
    return q, s


def gemm_i8(xq, ascale, Wq, wscale, K, bias=None, mode=0, res=None, out=None, amax=None, amax_rows=1,
            force_simt=False, ascale_per_row=True):
    """The W8A8 GEMM with its fused epilogue (vla_cuda_gemm_i8)."""
    M, N = xq.shape[0], Wq.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=torch.int32 if mode & EPI_ACC else torch.float32, device=xq.device)
    ldr = res.stride(0) if res is not None else 0
    check(lib().vla_cuda_gemm_i8(_p(out), out.stride(0), _p(xq), xq.stride(0), _p(ascale), 1 if ascale_per_row else 0,
                                 _p(Wq), Wq.stride(0), _p(wscale), _p(bias), _p(res), ldr, M, N, K, mode, _p(amax),
                                 amax_rows, 1 if force_simt else 0, _stream()), "vla_cuda_gemm_i8")
    return out


def gemm_i8_rowq_supported(M, N, K):
    return bool(lib().vla_cuda_gemm_i8_rowq_supported(int(M), int(N), int(K)))


def gemm_i8_rowq(xq, ascale, Wq, wscale, K, qamax, qsync, bias=None, relu=False):
    """The W8A8 GEMM (+ ReLU) with its output quantized per row for the next
    W8A8 GEMM (vla_cuda_gemm_i8_rowq): returns (q int8 [M, N], scale [M]).
    qamax [M] and qsync [2 * ceil(M / 128)] int32 (zeroed) are the caller's."""
    M, N = xq.shape[0], Wq.shape[0]
    q = torch.empty((M, N), dtype=torch.int8, device=xq.device)
    s = torch.empty(M, dtype=torch.float32, device=xq.device)
    check(lib().vla_cuda_gemm_i8_rowq(_p(q), N, _p(s), _p(xq), xq.stride(0), _p(ascale), _p(Wq), Wq.stride(0),
                                      _p(wscale), _p(bias), M, N, K, 1 if relu else 0, _p(qamax), _p(qsync),
                                      _stream()), "vla_cuda_gemm_i8_rowq")
    return q, s


def gemm_i8_splitk(xq, ascale, Wq, wscale, K, ws, counters, bias=None, mode=0, res=None, out=None):
    """The W8A8 GEMM with K split over independent CTAs (vla_cuda_gemm_i8_splitk):
    M <= 128 rows; ws int32 and counters int32 (zeroed) are the caller's workspace."""
    M, N = xq.shape[0], Wq.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=torch.int32 if mode & EPI_ACC else torch.float32, device=xq.device)
    ldr = res.stride(0) if res is not None else 0
    check(lib().vla_cuda_gemm_i8_splitk(_p(out), out.stride(0), _p(xq), xq.stride(0), _p(ascale), _p(Wq), Wq.stride(0),
                                        _p(wscale), _p(bias), _p(res), ldr, M, N, K, mode, _p(ws), ws.numel(),
                                        _p(counters), counters.numel(), _stream()), "vla_cuda_gemm_i8_splitk")
    return out


def dense_linear_i8(x, Wq, wscale, bias=None):
    """tcpu::dense_linear_i8: fp32 x [seq, K] -> fp32 [seq, N], x quantized per token."""
    seq, K = x.shape
    N = Wq.shape[0]
    out = torch.empty((seq, N), dtype=torch.float32, device=x.device)
    xq = torch.empty((seq, i8_ld(K)), dtype=torch.int8, device=x.device)
    s = torch.empty(seq, dtype=torch.float32, device=x.device)
    check(lib().vla_cuda_dense_linear_i8(_p(out), _p(x.contiguous()), _p(Wq), _p(wscale), _p(bias), seq, N, K,
                                         Wq.stride(0), _p(xq), _p(s), _stream()), "vla_cuda_dense_linear_i8")
    return out


def conv2d_i8(x, Wq, wscale, bias, Cout, k, stride, pad, clip=1.0, mode=0, res=None):
    """tcpu::conv2d_i8 over F NHWC frames: x [F, H, W, Cin] -> [F, Ho, Wo, Cout]."""
    F, H, W, Cin = x.shape
    Ho, Wo = (H + 2 * pad - k) // stride + 1, (W + 2 * pad - k) // stride + 1
    ldw = Wq.stride(0)
    out = torch.empty((F, Ho, Wo, Cout), dtype=torch.float32, device=x.device)
    col = torch.empty((F * Ho * Wo, ldw), dtype=torch.int8, device=x.device)
    rs = torch.empty(F * Ho * Wo, dtype=torch.float32, device=x.device)
    am = torch.zeros(F, dtype=torch.int32, device=x.device)
    check(lib().vla_cuda_conv2d_i8(_p(out), _p(x.contiguous()), F, H, W, Cin, _p(Wq), ldw, _p(wscale), _p(bias), Cout,
                                   k, stride, pad, clip, mode, _p(res), _p(col), _p(rs), _p(am), _stream()),
          "vla_cuda_conv2d_i8")
    return out


def layernorm(x, w, b, eps=1e-5):
    seq, H = x.shape
    out = torch.empty_like(x)
    check(lib().vla_cuda_layernorm(_p(out), _p(x.contiguous()), _p(w), _p(b), seq, H, eps, _stream()),
          "vla_cuda_layernorm")
    return out


def gqa_attention(Q, K, V, n_q, n_kv, scale, mask=None, head_dim=64):
    seq_q, seq_k = Q.shape[0], K.shape[0]
    out = torch.empty((seq_q, n_q * head_dim), dtype=torch.float32, device=Q.device)
    check(lib().vla_cuda_gqa_attention(_p(out), _p(Q.contiguous()), _p(K.contiguous()), _p(V.contiguous()), seq_q,
                                       seq_k, n_q, n_kv, head_dim, scale, _p(mask), _stream()),
          "vla_cuda_gqa_attention")
    return out


def gqa_attention_tc(Q, K, V, n_q, n_kv, scale, mask=None, head_dim=64):
    """The tensor-core (3xTF32 tcgen05) attention: same contract, not bit-identical."""
    seq_q, seq_k = Q.shape[0], K.shape[0]
    out = torch.empty((seq_q, n_q * head_dim), dtype=torch.float32, device=Q.device)
    check(lib().vla_cuda_gqa_attention_tc(_p(out), _p(Q.contiguous()), _p(K.contiguous()), _p(V.contiguous()),
                                          seq_q, seq_k, n_q, n_kv, head_dim, scale, _p(mask), _stream()),
          "vla_cuda_gqa_attention_tc")
    return out


def maxpool2d_relu(x, k=3, stride=2, pad=1):
    F, H, W, C = x.shape
    Ho, Wo = (H + 2 * pad - k) // stride + 1, (W + 2 * pad - k) // stride + 1
    out = torch.empty((F, Ho, Wo, C), dtype=torch.float32, device=x.device)
    check(lib().vla_cuda_maxpool2d_relu(_p(out), _p(x.contiguous()), F, H, W, C, k, stride, pad, _stream()),
          "vla_cuda_maxpool2d_relu")
    return out


def dense_linear_f32(x, W, bias=None):
    """tcpu::dense_linear (fp32), the reference's summation order."""
    seq, K = x.shape
    N = W.shape[0]
    out = torch.empty((seq, N), dtype=torch.float32, device=x.device)
    check(lib().vla_cuda_dense_linear_f32(_p(out), _p(x.contiguous()), _p(W.contiguous()), _p(bias), seq, N, K,
                                          _stream()), "vla_cuda_dense_linear_f32")
    return out


# ---- lm / conv ops of the other policy families (src/ops/lm_ops.h, conv_ops.h)

def rmsnorm(x, w, eps=1e-6):
    """tcpu::rmsnorm: sequential double sum of squares per row."""
    seq, hidden = x.shape
    out = torch.empty_like(x)
    check(lib().vla_cuda_rmsnorm(_p(out), _p(x.contiguous()), _p(w.contiguous()), seq, hidden, eps, _stream()),
          "vla_cuda_rmsnorm")
    return out


def rope_neox(x, pos, n_heads, head_dim, base=10000.0):
    """tcpu::rope_neox on a copy of x [seq, n_heads*head_dim]; pos int32 [seq]."""
    y = x.contiguous().clone()
    check(lib().vla_cuda_rope_neox(_p(y), _p(pos.to(torch.int32).contiguous()), y.shape[0], n_heads, head_dim, base,
                                   _stream()), "vla_cuda_rope_neox")
    return y


def activation(name, x, u=None):
    """tcpu::{silu_gate, silu, gelu_tanh, gelu_erf, relu, mish}; returns a new tensor."""
    x = x.contiguous()
    out = torch.empty_like(x)
    fn = getattr(lib(), f"vla_cuda_{name}")
    if name == "silu_gate":
        rc = fn(_p(out), _p(x), _p(u.contiguous()), x.numel(), _stream())
    else:
        rc = fn(_p(out), _p(x), x.numel(), _stream())
    check(rc, f"vla_cuda_{name}")
    return out


def groupnorm(x, scale, bias, groups, eps=1e-5, fuse_relu=False):
    """tcpu::groupnorm over x [n_pixels, C] (channels last)."""
    P, C = x.shape
    out = torch.empty_like(x)
    scratch = torch.empty(int(lib().vla_cuda_groupnorm_scratch_bytes(C)), dtype=torch.uint8, device=x.device)
    check(lib().vla_cuda_groupnorm(_p(out), _p(x.contiguous()), _p(scale.contiguous()), _p(bias.contiguous()), P, C,
                                   groups, eps, 1 if fuse_relu else 0, _p(scratch), _stream()), "vla_cuda_groupnorm")
    return out


def spatial_softmax(x, grid):
    """tcpu::spatial_softmax: x [n_pixels, C], grid [n_pixels, 2] -> [C, 2]."""
    P, C = x.shape
    out = torch.empty((C, 2), dtype=torch.float32, device=x.device)
    check(lib().vla_cuda_spatial_softmax(_p(out), _p(x.contiguous()), _p(grid.contiguous()), P, C, _stream()),
          "vla_cuda_spatial_softmax")
    return out


def im2col1d(x, k, stride, pad):
    """tcpu::im2col1d: x [T, Cin] -> [Tout, k*Cin]."""
    T, Cin = x.shape
    Tout = (T + 2 * pad - k) // stride + 1
    col = torch.empty((Tout, k * Cin), dtype=torch.float32, device=x.device)
    check(lib().vla_cuda_im2col1d(_p(col), _p(x.contiguous()), T, Cin, k, stride, pad, Tout, _stream()),
          "vla_cuda_im2col1d")
    return col


def conv_transpose1d(x, W, bias, k, stride, pad):
    """tcpu::conv_transpose1d: x [T, Cin], W [Cin, k, Cout] -> [(T-1)*stride-2*pad+k, Cout]."""
    T, Cin = x.shape
    Cout = W.shape[-1]
    Tout = (T - 1) * stride - 2 * pad + k
    out = torch.empty((Tout, Cout), dtype=torch.float32, device=x.device)
    check(lib().vla_cuda_conv_transpose1d(_p(out), _p(x.contiguous()), _p(W.contiguous()), _p(bias), T, Cin, Cout, k,
                                          stride, pad, _stream()), "vla_cuda_conv_transpose1d")
    return out


# ---- prompts and the 4-bit cache (no counterpart in the reference)

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _on_device(*tensors):
    dev = torch.cuda.current_device()
    for t in tensors:
        _need(t is None or (t.is_cuda and t.device.index == dev), "tensors have to be on the current CUDA device")


def _typed(x, name):
    _need(x.dtype in _TYPES, f"{name} has to be float32, float16 or bfloat16")
    return _TYPES[x.dtype]


def _heads(x, name):
    """[tokens, heads, d] with contiguous channels; other strides stay as they are."""
    _need(x.dim() == 3, f"{name} has to be [tokens, heads, head_dim]")
    return x if x.stride(2) == 1 or x.shape[2] == 1 else x.contiguous()


def _int32(x, name):
    _need(x.dtype == torch.int32, f"{name} has to be int32")
    return x.contiguous()


def qk_norm_rope(q, k, pos, sections, q_weight=None, k_weight=None, eps=1e-6, base=10000.0, restart=False,
                 out_dtype=None):
    """Norms of the query and key heads and their multi-axis rotary positions in one pass.

    q [T, n_q, d], k [T, n_kv, d] (or None); pos int32 [axes, T]; sections: rotated pairs of each axis; weights
    fp32 [d] or None (no norm). Returns (q_out, k_out) in out_dtype (default: q's)."""
    q = _heads(q, "q")
    T, n_q, d = q.shape
    in_type, out_dtype = _typed(q, "q"), out_dtype or q.dtype
    _need(out_dtype in _TYPES, "out_dtype has to be float32, float16 or bfloat16")
    n_kv, k_out = 0, None
    if k is not None:
        k = _heads(k, "k")
        _need(k.dtype == q.dtype and k.shape[0] == T and k.shape[2] == d, "k has to match q in type, tokens and width")
        n_kv = k.shape[1]
        k_out = torch.empty((T, n_kv, d), dtype=out_dtype, device=q.device)
    pos = _int32(pos, "pos")
    _need(tuple(pos.shape) == (len(sections), T), "pos has to be [axes, tokens], one axis for each of sections")
    for w in (q_weight, k_weight):
        _need(w is None or (w.dtype == torch.float32 and tuple(w.shape) == (d,) and w.is_contiguous()),
              "weights have to be contiguous float32 [head_dim]")
    _on_device(q, k, pos, q_weight, k_weight)
    q_out = torch.empty((T, n_q, d), dtype=out_dtype, device=q.device)
    ks = (0, 0) if k is None else (k.stride(0), k.stride(1))
    check(lib().vla_cuda_qk_norm_rope(_p(q_out), _p(k_out), _TYPES[out_dtype], _p(q), q.stride(0), q.stride(1), _p(k),
                                      *ks, in_type, _p(pos), (ctypes.c_int32 * len(sections))(*sections),
                                      len(sections), 1 if restart else 0, _p(q_weight), _p(k_weight), eps, base, T, n_q,
                                      n_kv, d, _stream()), "vla_cuda_qk_norm_rope")
    return q_out, k_out


def _tma_heads(x, name):
    """_heads whose address and strides are (nonzero) multiples of 16 bytes; a copy where they are not."""
    x = _heads(x, name)
    if x.data_ptr() % 16 or x.stride(0) % 8 or x.stride(1) % 8 or not x.stride(0) or not x.stride(1):
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def prompt_attention(q, k, v, cu_q, cu_k=None, scale=None, causal=True, prefix=None):
    """Attention over packed prompts: q [Tq, n_q, d], k / v [Tk, n_kv, d] (fp16 or bf16), cu_q / cu_k int32
    [n_seq + 1] (cu_k defaults to cu_q), prefix int32 [n_seq] or None. Returns [Tq, n_q, d]."""
    q, k, v = _tma_heads(q, "q"), _tma_heads(k, "k"), _tma_heads(v, "v")
    Tq, n_q, d = q.shape
    Tk, n_kv = k.shape[:2]
    _need(q.dtype in (torch.float16, torch.bfloat16) and k.dtype == q.dtype and v.dtype == q.dtype,
          "q, k and v have to be float16, or bfloat16")
    _need(k.shape == v.shape and k.shape[2] == d, "k and v have to match in shape, and q in width")
    cu_q = _int32(cu_q, "cu_q")
    cu_k = cu_q if cu_k is None else _int32(cu_k, "cu_k")
    _need(cu_q.dim() == 1 and cu_q.shape == cu_k.shape and cu_q.numel() > 0, "cu_q and cu_k have to be [n_seq + 1]")
    n_seq = cu_q.numel() - 1
    if prefix is not None:
        prefix = _int32(prefix, "prefix")
        _need(tuple(prefix.shape) == (n_seq,), "prefix has to be [n_seq]")
    _on_device(q, k, v, cu_q, cu_k, prefix)
    out = torch.empty((Tq, n_q, d), dtype=q.dtype, device=q.device)
    check(lib().vla_cuda_prompt_attention(_p(out), _p(q), q.stride(0), q.stride(1), _p(k), k.stride(0), k.stride(1),
                                          _p(v), v.stride(0), v.stride(1), _TYPES[q.dtype], _p(cu_q), _p(cu_k),
                                          _p(prefix), n_seq, Tq, Tk, n_q, n_kv, d,
                                          1.0 / math.sqrt(d) if scale is None else scale, 1 if causal else 0,
                                          _stream()), "vla_cuda_prompt_attention")
    return out


def kv4_cache(n_pages, n_kv, head_dim, page=64, device="cuda"):
    """An empty paged 4-bit cache: uint8 [n_pages, n_kv, page // 16, 20 * head_dim]."""
    size = int(lib().vla_cuda_kv4_block_bytes(head_dim))
    _need(size > 0 and page in (16, 32, 64, 128, 256), "head_dim has to be 64 or 128, page 16, 32, 64, 128 or 256")
    return torch.zeros((n_pages, n_kv, page // 16, size), dtype=torch.uint8, device=device)


def _cache(cache):
    _need(cache.dtype == torch.uint8 and cache.dim() == 4 and cache.is_contiguous() and cache.shape[3] % 20 == 0,
          "cache has to be kv4_cache's")
    n_pages, n_kv, blocks, size = cache.shape
    return n_pages, n_kv, 16 * blocks, size // 20


def kv4_append(cache, k, v, slots):
    """Quantizes k and v [T, n_kv, d] into the cache's slots (int64 [T], negative: skipped)."""
    n_pages, n_kv, page, d = _cache(cache)
    k, v = _heads(k, "k"), _heads(v, "v")
    T = k.shape[0]
    _need(tuple(k.shape) == (T, n_kv, d) and k.shape == v.shape and k.dtype == v.dtype,
          "k and v have to be [tokens, n_kv, head_dim] of the cache, of one type")
    _need(slots.dtype == torch.int64 and tuple(slots.shape) == (T,), "slots has to be int64 [tokens]")
    slots = slots.contiguous()
    _on_device(cache, k, v, slots)
    check(lib().vla_cuda_kv4_append(_p(cache), n_pages, page, _p(k), k.stride(0), k.stride(1), _p(v), v.stride(0),
                                    v.stride(1), _typed(k, "k"), _p(slots), T, n_kv, d, _stream()),
          "vla_cuda_kv4_append")


def kv4_read(cache, slots, dtype=torch.float32):
    """The values of the cache's slots: (k, v) [T, n_kv, d]; zeros for a negative slot."""
    n_pages, n_kv, page, d = _cache(cache)
    _need(dtype in _TYPES, "dtype has to be float32, float16 or bfloat16")
    _need(slots.dtype == torch.int64 and slots.dim() == 1, "slots has to be int64 [tokens]")
    slots = slots.contiguous()
    _on_device(cache, slots)
    k = torch.empty((slots.numel(), n_kv, d), dtype=dtype, device=cache.device)
    v = torch.empty_like(k)
    check(lib().vla_cuda_kv4_read(_p(cache), n_pages, page, _p(k), _p(v), _TYPES[dtype], _p(slots), slots.numel(), n_kv,
                                  d, _stream()), "vla_cuda_kv4_read")
    return k, v


def kv4_attention(q, cache, table, lens, scale=None, causal=True):
    """Attention of new tokens over the 4-bit cache: q [B, n_q, d] or [B, queries, n_q, d], table int32 [B, pages],
    lens int32 [B] (tokens in the cache, the new ones among them). Returns q's shape and type."""
    n_pages, n_kv, page, d = _cache(cache)
    _need(q.dim() in (3, 4) and q.shape[-1] == d, "q has to be [batch, (queries,) n_q, head_dim] of the cache's width")
    x = q if q.stride(-1) == 1 else q.contiguous()
    B, n_q = x.shape[0], x.shape[-2]
    queries, q_tok = (1, 0) if x.dim() == 3 else (x.shape[1], x.stride(1))
    typ = _typed(x, "q")
    _need(table.dtype == torch.int32 and table.dim() == 2 and table.shape[0] == B, "table has to be int32 [batch, pages]")
    if table.stride(1) != 1 or (B > 1 and table.stride(0) < table.shape[1]):
        table = table.contiguous()
    lens = _int32(lens, "lens")
    _need(tuple(lens.shape) == (B,), "lens has to be [batch]")
    _on_device(x, cache, table, lens)
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    pages = table.shape[1]
    size = int(lib().vla_cuda_kv4_attention_workspace_bytes(B, queries, n_q, n_kv, d, pages, page))
    ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
    check(lib().vla_cuda_kv4_attention(_p(out), _p(x), x.stride(0), q_tok, x.stride(-2), typ, _p(cache), n_pages, page,
                                       _p(table), max(table.stride(0), pages), pages, _p(lens), B, queries, n_q, n_kv, d,
                                       1.0 / math.sqrt(d) if scale is None else scale, 1 if causal else 0, _p(ws),
                                       size, _stream()), "vla_cuda_kv4_attention")
    return out


def device_status() -> int:
    return int(lib().vla_cuda_device_status())
