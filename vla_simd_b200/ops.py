"""Op-level wrappers over include/vla_simd_cuda.h for torch CUDA tensors.

Each function mirrors one reference op (src/ops/quant_ops.h, lm_ops.h,
conv_ops.h) - same argument meaning, the outputs allocated here for
convenience - and launches on torch's current stream. torch supplies device
memory and the stream handle only; the compute is the library's kernels.
"""
from __future__ import annotations

import ctypes

import torch

from . import EPI_ACC, check, lib


def _p(t):
    return None if t is None else t.data_ptr()


# the current stream's handle alone: current_stream() builds a Stream object, 3 us a call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream() -> int:
    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(torch.cuda.current_device())


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


# A call of these takes a few microseconds on the device at single tokens, so the
# wrappers look at each argument once.

def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _on_device(*tensors):
    dev = torch.cuda.current_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError("tensors have to be on the current CUDA device")


def _typed(x):
    t = _TYPES.get(x.dtype)
    if t is None:
        raise ValueError("q, k and v have to be float32, float16 or bfloat16")
    return t


def _new(like, shape, dtype):
    """A contiguous tensor for an output."""
    if like.dtype is dtype and like.shape == shape and like.is_contiguous():
        return torch.empty_like(like)
    return like.new_empty(shape, dtype=dtype)


def _heads(x):
    """[tokens, heads, d] with contiguous channels; other strides stay as they are. Returns it and its strides."""
    if x.dim() != 3:
        raise ValueError("q, k and v have to be [tokens, heads, head_dim]")
    st = x.stride()
    if st[2] != 1 and x.shape[2] != 1:
        x = x.contiguous()
        st = x.stride()
    return x, st


def _int32(x, what):
    if x.dtype is not torch.int32:
        raise ValueError(f"{what} has to be int32")
    return x if x.is_contiguous() else x.contiguous()


def qk_norm_rope(q, k, pos, sections, q_weight=None, k_weight=None, eps=1e-6, base=10000.0, restart=False,
                 out_dtype=None):
    """Norms of the query and key heads and their multi-axis rotary positions in one pass.

    q [T, n_q, d], k [T, n_kv, d] (or None); pos int32 [axes, T]; sections: rotated pairs of each axis; weights
    fp32 [d] or None (no norm). Returns (q_out, k_out) in out_dtype (default: q's)."""
    q, qs = _heads(q)
    T, n_q, d = q.shape
    in_type = _typed(q)
    if out_dtype is None:
        out_dtype = q.dtype
    _need(out_dtype in _TYPES, "out_dtype has to be float32, float16 or bfloat16")
    n_kv, k_out, ks = 0, None, (0, 0)
    if k is not None:
        k, ks = _heads(k)
        n_kv = k.shape[1]
        _need(k.dtype is q.dtype and k.shape[0] == T and k.shape[2] == d, "k has to match q in type, tokens and width")
        k_out = _new(k, (T, n_kv, d), out_dtype)
    axes = len(sections)
    pos = _int32(pos, "pos")
    _need(pos.shape == (axes, T), "pos has to be [axes, tokens], one axis for each of sections")
    for w in (q_weight, k_weight):
        if w is not None:
            _need(w.dtype is torch.float32 and w.shape == (d,) and w.is_contiguous(),
                  "weights have to be contiguous float32 [head_dim]")
    _on_device(q, k, pos, q_weight, k_weight)
    q_out = _new(q, (T, n_q, d), out_dtype)
    check(lib().vla_cuda_qk_norm_rope(q_out.data_ptr(), _p(k_out), _TYPES[out_dtype], q.data_ptr(), qs[0], qs[1], _p(k),
                                      ks[0], ks[1], in_type, pos.data_ptr(), (ctypes.c_int32 * axes)(*sections), axes,
                                      restart, _p(q_weight), _p(k_weight), eps, base, T, n_q, n_kv, d, _stream()),
          "vla_cuda_qk_norm_rope")
    return q_out, k_out


def _tma_heads(x):
    """_heads whose address and strides are (nonzero) multiples of 16 bytes; a copy where they are not."""
    x, st = _heads(x)
    if x.data_ptr() % 16 or st[0] % 8 or st[1] % 8 or not st[0] or not st[1]:
        x = x.clone(memory_format=torch.contiguous_format)
        st = x.stride()
    return x, st


def prompt_attention(q, k, v, cu_q, cu_k=None, scale=None, causal=True, prefix=None):
    """Attention over packed prompts: q [Tq, n_q, d], k / v [Tk, n_kv, d] (fp16 or bf16), cu_q / cu_k int32
    [n_seq + 1] (cu_k defaults to cu_q), prefix int32 [n_seq] or None. Returns [Tq, n_q, d]; its rows outside every
    sequence (before cu_q[0], from cu_q[-1] on) are not written and hold anything."""
    (q, qs), (k, ks), (v, vs) = _tma_heads(q), _tma_heads(k), _tma_heads(v)
    Tq, n_q, d = q.shape
    Tk, n_kv, dk = k.shape
    typ = _typed(q)
    _need(typ and k.dtype is q.dtype and v.dtype is q.dtype, "q, k and v have to be float16, or bfloat16")
    _need(k.shape == v.shape and dk == d, "k and v have to match in shape, and q in width")
    cu_q = _int32(cu_q, "cu_q")
    cu_k = cu_q if cu_k is None else _int32(cu_k, "cu_k")
    n_seq = cu_q.numel() - 1
    _need(cu_q.dim() == 1 and cu_q.shape == cu_k.shape and n_seq >= 0, "cu_q and cu_k have to be [n_seq + 1]")
    if prefix is not None:
        prefix = _int32(prefix, "prefix")
        _need(prefix.shape == (n_seq,), "prefix has to be [n_seq]")
    _on_device(q, k, v, cu_q, cu_k, prefix)
    out = _new(q, (Tq, n_q, d), q.dtype)
    check(lib().vla_cuda_prompt_attention(out.data_ptr(), q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1],
                                          v.data_ptr(), vs[0], vs[1], typ, cu_q.data_ptr(), cu_k.data_ptr(), _p(prefix),
                                          n_seq, Tq, Tk, n_q, n_kv, d, d ** -0.5 if scale is None else scale, causal,
                                          _stream()), "vla_cuda_prompt_attention")
    return out


def kv4_cache(n_pages, n_kv, head_dim, page=64, device="cuda"):
    """An empty paged 4-bit cache: uint8 [n_pages, n_kv, page // 16, 20 * head_dim]."""
    size = int(lib().vla_cuda_kv4_block_bytes(head_dim))
    _need(size > 0 and page in (16, 32, 64, 128, 256), "head_dim has to be 64 or 128, page 16, 32, 64, 128 or 256")
    return torch.zeros((n_pages, n_kv, page // 16, size), dtype=torch.uint8, device=device)


def _cache(cache):
    if cache.dtype is not torch.uint8 or cache.dim() != 4 or not cache.is_contiguous() or cache.shape[3] % 20:
        raise ValueError("cache has to be kv4_cache's")
    n_pages, n_kv, blocks, size = cache.shape
    return n_pages, n_kv, 16 * blocks, size // 20


def _slots(slots, T):
    if slots.dtype is not torch.int64 or slots.dim() != 1 or (T is not None and slots.shape[0] != T):
        raise ValueError("slots has to be int64 [tokens]")
    return slots if slots.is_contiguous() else slots.contiguous()


def kv4_append(cache, k, v, slots):
    """Quantizes k and v [T, n_kv, d] into the cache's slots (int64 [T], negative: skipped)."""
    n_pages, n_kv, page, d = _cache(cache)
    (k, ks), (v, vs) = _heads(k), _heads(v)
    T = k.shape[0]
    _need(k.shape == (T, n_kv, d) and k.shape == v.shape and k.dtype is v.dtype,
          "k and v have to be [tokens, n_kv, head_dim] of the cache, of one type")
    slots = _slots(slots, T)
    _on_device(cache, k, v, slots)
    check(lib().vla_cuda_kv4_append(cache.data_ptr(), n_pages, page, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0],
                                    vs[1], _typed(k), slots.data_ptr(), T, n_kv, d, _stream()), "vla_cuda_kv4_append")


def kv4_read(cache, slots, dtype=torch.float32):
    """The values of the cache's slots: (k, v) [T, n_kv, d]; zeros for a negative slot."""
    n_pages, n_kv, page, d = _cache(cache)
    typ = _TYPES.get(dtype)
    _need(typ is not None, "dtype has to be float32, float16 or bfloat16")
    slots = _slots(slots, None)
    _on_device(cache, slots)
    T = slots.shape[0]
    k = cache.new_empty((T, n_kv, d), dtype=dtype)
    v = torch.empty_like(k)
    check(lib().vla_cuda_kv4_read(cache.data_ptr(), n_pages, page, k.data_ptr(), v.data_ptr(), typ, slots.data_ptr(), T,
                                  n_kv, d, _stream()), "vla_cuda_kv4_read")
    return k, v


def kv4_attention(q, cache, table, lens, scale=None, causal=True):
    """Attention of new tokens over the 4-bit cache: q [B, n_q, d] or [B, queries, n_q, d], table int32 [B, pages],
    lens int32 [B] (tokens in the cache, the new ones among them). Returns q's shape and type. The work is planned by
    the table's width: hand over the columns in use (table[:, :n], no copy) of one made for much longer sequences."""
    n_pages, n_kv, page, d = _cache(cache)
    shape = q.shape
    _need(len(shape) in (3, 4) and shape[-1] == d, "q has to be [batch, (queries,) n_q, head_dim] of the cache's width")
    st = q.stride()
    if st[-1] != 1:
        q = q.contiguous()
        st = q.stride()
    B, n_q = shape[0], shape[-2]
    queries, q_tok = (1, 0) if len(shape) == 3 else (shape[1], st[1])
    typ = _typed(q)
    _need(table.dtype is torch.int32 and table.dim() == 2 and table.shape[0] == B, "table has to be int32 [batch, pages]")
    pages = table.shape[1]
    ld, step = table.stride()
    if step != 1 or ld < pages:
        table = table.contiguous()
        ld = pages
    lens = _int32(lens, "lens")
    _need(lens.shape == (B,), "lens has to be [batch]")
    _on_device(q, cache, table, lens)
    L = lib()
    out = _new(q, shape, q.dtype)
    size = L.vla_cuda_kv4_attention_workspace_bytes(B, queries, n_q, n_kv, d, pages, page)
    ws = cache.new_empty(size) if size else None
    check(L.vla_cuda_kv4_attention(out.data_ptr(), q.data_ptr(), st[0], q_tok, st[-2], typ, cache.data_ptr(), n_pages,
                                   page, table.data_ptr(), ld, pages, lens.data_ptr(), B, queries, n_q, n_kv, d,
                                   d ** -0.5 if scale is None else scale, causal, _p(ws), size, _stream()),
          "vla_cuda_kv4_attention")
    return out


def device_status() -> int:
    return int(lib().vla_cuda_device_status())
