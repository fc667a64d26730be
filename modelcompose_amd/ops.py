"""Thin torch-tensor wrappers over the C ABI (include/mc_hip.h).  PyTorch provides device memory and
the current HIP stream; all arithmetic happens in libmc_hip.so.  No CPU fallback."""
from __future__ import annotations

import contextlib
import ctypes as C
import math
import operator
import threading
from typing import Optional, Sequence

import torch

from . import _lib

ACT = {None: 0, "none": 0, "gelu": 1, "quick_gelu": 2, "silu": 3, "relu": 4}
# mc_gemm_args.family (include/mc_hip.h): which kernel family runs a linear.  Each family adds a row's products in ONE fp32 order whatever
# the number of rows; "auto" picks by M (strip for M <= 64, tile above), so a caller whose rows must not depend on how many other rows share
# the launch - the inference towers and projectors, whose row count is B x tokens - pins "tile" with `with ops.gemm_family("tile"):`.
FAMILY = {None: 0, "auto": 0, "strip": 1, "tile": 2}
_family_tls = threading.local()


def _fam(family=None) -> int:
    return FAMILY[family] if family is not None else getattr(_family_tls, "v", 0)


@contextlib.contextmanager
def gemm_family(name):
    """Default kernel family of every linear() / linear_ex() / linear_grouped() call of this thread inside the block."""
    old = getattr(_family_tls, "v", 0)
    _family_tls.v = FAMILY[name]
    try:
        yield
    finally:
        _family_tls.v = old

BF16 = _lib.storage_dtype()      # the library's 16-bit storage element: bf16, or fp16 with MC_STORAGE_DTYPE=fp16 (_lib.set_storage_dtype)


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _p(t: Optional[torch.Tensor]):
    return C.c_void_p(0 if t is None else t.data_ptr())


def _req(t: torch.Tensor, dtype="storage", name="tensor"):
    if isinstance(dtype, str):
        dtype = BF16                                       # the library's storage element (rebound by _lib.set_storage_dtype)
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device (HIP) tensor; this path has no CPU fallback")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    return t


def ceil_to(x: int, m: int) -> int:
    return (x + m - 1) // m * m


class PackedWeight:
    """A linear weight in the MFMA-fragment layout of csrc/gemm.hip (+ optional bf16 bias)."""
    __slots__ = ("data", "N", "K", "Kp", "bias")

    def __init__(self, data, N, K, bias=None):
        self.data, self.N, self.K, self.Kp, self.bias = data, N, K, ceil_to(K, 64), bias

    @property
    def nbytes(self):
        return self.data.numel() * 2


def packed_elems(N: int, K: int) -> int:
    return ceil_to(N, 16) * ceil_to(K, 64)


def pack_weight(w: torch.Tensor, bias: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> PackedWeight:
    """[N, K] row-major (any float dtype, device) -> PackedWeight."""
    w = _req(w.to(BF16), BF16, "weight")
    if w.dim() != 2:
        raise ValueError("weight must be 2-D [N, K]")
    if w.stride(1) != 1:
        w = w.contiguous()
    N, K = w.shape
    if out is None:
        out = torch.empty(packed_elems(N, K), dtype=BF16, device=w.device)
    _lib.check(_lib.lib().mc_pack_weight_bf16(_p(w), w.stride(0), _p(out), N, K, _stream()), "mc_pack_weight_bf16")
    b = None if bias is None else _req(bias.to(BF16).contiguous(), BF16, "bias")
    return PackedWeight(out, N, K, b)


def unpack_weight(pw: PackedWeight) -> torch.Tensor:
    out = torch.empty(pw.N, pw.K, dtype=BF16, device=pw.data.device)
    _lib.check(_lib.lib().mc_unpack_weight_bf16(_p(pw.data), _p(out), pw.N, pw.K, _stream()), "mc_unpack_weight_bf16")
    return out


def compose_weight(w: Optional[torch.Tensor], terms: Sequence, N: int, K: int, rowmajor_out: bool = False):
    """W' = W + Σ scale·B·A  ->  PackedWeight.  terms = [(A [r,K], B [N,r], scale), ...] (device tensors)."""
    dev = (w if w is not None else terms[0][0]).device
    n = len(terms)
    r = 0
    ats, bs = [], []
    for (a, b, s) in terms:
        r0 = a.shape[0]
        rp = ceil_to(r0, 32)
        at = a.to(BF16).t().contiguous()                 # [K, r]
        bb = b.to(BF16).contiguous()                     # [N, r]
        if rp != r0:
            at = torch.nn.functional.pad(at, (0, rp - r0))
            bb = torch.nn.functional.pad(bb, (0, rp - r0))
        if r and rp != r:
            raise ValueError("all LoRA terms of one linear must share the rank")
        r = rp
        ats.append(at)
        bs.append(bb)
    out = torch.empty(packed_elems(N, K), dtype=BF16, device=dev)
    rm = torch.empty(N, K, dtype=BF16, device=dev) if rowmajor_out else None
    if w is not None:
        w = _req(w.to(BF16), BF16, "w")
        if w.stride(1) != 1:
            w = w.contiguous()
    at_arr = (C.c_void_p * max(n, 1))(*[t.data_ptr() for t in ats])
    b_arr = (C.c_void_p * max(n, 1))(*[t.data_ptr() for t in bs])
    sc = (C.c_float * max(n, 1))(*[float(t[2]) for t in terms])
    _lib.check(_lib.lib().mc_compose_weight_bf16(_p(w), 0 if w is None else w.stride(0), at_arr, b_arr, sc, n, r, _p(out),
                                                 _p(rm), K, N, K, _stream()), "mc_compose_weight_bf16")
    pw = PackedWeight(out, N, K)
    return (pw, rm) if rowmajor_out else pw


def linear(x: torch.Tensor, w: PackedWeight, act=None, residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
           out_f32: bool = False, alpha: float = 1.0, bias: bool = True, beta: float = 1.0, auto_split: bool = False, family=None) -> torch.Tensor:
    """out[M,N] = act(alpha * x W^T + b) + beta * residual.  x: [M, Kp] bf16 (Kp = K padded to 64, pad columns zero).
    auto_split: let the library split K when the launch would under-fill the GPU (training-time rank projections; the choice depends
    on M, so inference leaves it off to stay batch-invariant).  family: "auto" / "strip" / "tile" (default: the thread's gemm_family)."""
    _req(x, BF16, "x")
    if x.dim() != 2 or x.stride(1) != 1:
        raise ValueError("x must be 2-D with contiguous rows")
    M, Kx = x.shape
    if Kx != w.Kp:
        raise ValueError(f"x has {Kx} columns, weight expects K padded to {w.Kp}")
    if out is None:
        out = torch.empty(M, w.N, dtype=torch.float32 if out_f32 else BF16, device=x.device)
    b = w.bias if bias else None
    a = _lib.GemmArgsC(x.data_ptr(), x.stride(0), w.data.data_ptr(), 0 if b is None else b.data_ptr(), 0 if residual is None else residual.data_ptr(),
                       0 if residual is None else residual.stride(0), out.data_ptr(), out.stride(0), M, w.N, w.Kp, ACT[act],
                       1 if out_f32 else 0, alpha, beta, 0, 0, -1 if auto_split else 1, 0.0, 0, 0, 0.0, 0 if auto_split else _fam(family))
    _lib.check(_lib.lib().mc_gemm_ex_bf16(C.byref(a), _stream()), "mc_gemm_ex_bf16")
    return out


def linear_ex(x: torch.Tensor, w: PackedWeight, row_scale: Optional[torch.Tensor] = None, swiglu: bool = False,
              residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, out_f32: bool = False, rms_eps: float = 0.0,
              rope=None, rms_out: Optional[torch.Tensor] = None, rms_out_eps: float = 0.0, family=None) -> torch.Tensor:
    """mc_gemm_ex_bf16: row_scale fp32 [M] (1/rms of a folded RMSNorm), swiglu (gate/up interleaved per 16 rows -> [M, N/2]),
    rms_eps > 0 (strip family): the RMSNorm factor computed inside the launch; rope = rope_scatter(...): the launch is a prefill's q|k|v
    projection, RoPE and the q / KV-cache scatter happen in its epilogue (the returned buffer is scratch then)."""
    _req(x, BF16, "x")
    M, Kx = x.shape
    if Kx != w.Kp:
        raise ValueError(f"x has {Kx} columns, weight expects K padded to {w.Kp}")
    n_out = w.N // 2 if swiglu else w.N
    if out is None:
        out = torch.empty(M, n_out, dtype=torch.float32 if out_f32 else BF16, device=x.device)
    a = _lib.GemmArgsC(x.data_ptr(), x.stride(0), w.data.data_ptr(), 0, 0 if residual is None else residual.data_ptr(),
                       0 if residual is None else residual.stride(0), out.data_ptr(), out.stride(-2), M, w.N, w.Kp, 0,
                       1 if out_f32 else 0, 1.0, 1.0, 0 if row_scale is None else row_scale.data_ptr(),
                       1 if swiglu else 0, 1, float(rms_eps), 0 if rope is None else C.addressof(rope[0]),
                       0 if rms_out is None else rms_out.data_ptr(), float(rms_out_eps), _fam(family))
    _lib.check(_lib.lib().mc_gemm_ex_bf16(C.byref(a), _stream()), "mc_gemm_ex_bf16")
    return out


def rope_scatter(row_b, row_pos, row_t, cos, sin, q_out, k_cache, v_cache, H, Hkv, D, Lq, Smax):
    """struct mc_rope_scatter for linear_ex / linear_grouped (returns (struct, tensors kept alive))."""
    r = _lib.RopeScatterC(*[t.data_ptr() for t in (row_b, row_pos, row_t, cos, sin, q_out, k_cache, v_cache)], H, Hkv, D, Lq, Smax)
    return (r, (row_b, row_pos, row_t, cos, sin, q_out, k_cache, v_cache))


def linear_grouped(x: torch.Tensor, weights: Sequence[PackedWeight], group_start: Sequence[int], row_scale: Optional[torch.Tensor] = None,
                   swiglu: bool = False, residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, rope=None,
                   rms_out: Optional[torch.Tensor] = None, rms_out_eps: float = 0.0, family=None) -> torch.Tensor:
    """mc_gemm_grouped_bf16: rows [group_start[g], group_start[g+1]) of x use weights[g] (routed LocalLoRA linear)."""
    _req(x, BF16, "x")
    w0 = weights[0]
    M = x.shape[0]
    n_out = w0.N // 2 if swiglu else w0.N
    if out is None:
        out = torch.empty(M, n_out, dtype=BF16, device=x.device)
    a = _lib.GemmArgsC(x.data_ptr(), x.stride(0), 0, 0, 0 if residual is None else residual.data_ptr(),
                       0 if residual is None else residual.stride(0), out.data_ptr(), out.stride(0), 0, w0.N, w0.Kp, 0, 0, 1.0, 1.0,
                       0 if row_scale is None else row_scale.data_ptr(), 1 if swiglu else 0, 1, 0.0, 0 if rope is None else C.addressof(rope[0]),
                       0 if rms_out is None else rms_out.data_ptr(), float(rms_out_eps), _fam(family))
    gs = (C.c_int32 * len(group_start))(*group_start)
    wp = (C.c_void_p * len(weights))(*[w.data.data_ptr() for w in weights])
    _lib.check(_lib.lib().mc_gemm_grouped_bf16(C.byref(a), len(weights), gs, wp, _stream()), "mc_gemm_grouped_bf16")
    return out


def rms_scale(x, eps):
    _req(x, BF16, "x")
    M, D = x.shape
    rs = torch.empty(M, dtype=torch.float32, device=x.device)
    _lib.check(_lib.lib().mc_rms_scale_bf16(_p(x), x.stride(0), _p(rs), M, D, eps, _stream()), "mc_rms_scale_bf16")
    return rs


def rmsnorm(x, w, eps, out=None):
    _req(x, BF16, "x")
    M, D = x.shape
    out = torch.empty_like(x) if out is None else out
    _lib.check(_lib.lib().mc_rmsnorm_bf16(_p(x), x.stride(0), _p(w), _p(out), out.stride(0), M, D, eps, _stream()), "mc_rmsnorm_bf16")
    return out


def layernorm(x, w, b, eps, out=None):
    _req(x, BF16, "x")
    M, D = x.shape
    out = torch.empty_like(x) if out is None else out
    _lib.check(_lib.lib().mc_layernorm_bf16(_p(x), x.stride(0), _p(w), _p(b), _p(out), out.stride(0), M, D, eps, _stream()), "mc_layernorm_bf16")
    return out


def add_layernorm(x, table, idx, w, b, eps, sum_out=None, out=None):
    """(sum, LayerNorm(sum)) with sum[r] = bf16(x[r] + table[idx[r]]) in one pass (mc_add_layernorm_bf16); sum_out may alias x."""
    _req(x, BF16, "x")
    M, D = x.shape
    sum_out = torch.empty_like(x) if sum_out is None else sum_out
    out = torch.empty_like(x) if out is None else out
    _lib.check(_lib.lib().mc_add_layernorm_bf16(_p(x), x.stride(0), _p(table), table.stride(0), _p(idx), _p(sum_out), sum_out.stride(0), _p(w), _p(b),
                                                _p(out), out.stride(0), M, D, eps, _stream()), "mc_add_layernorm_bf16")
    return sum_out, out


def attn_mask(key_valid: Optional[torch.Tensor] = None, batch_split=None):
    """struct mc_attn_mask or None: key_valid uint8 [B, >= S] (0 = masked key), batch_split = (b_inner, inner_stride) - the two-level batch
    index of the Lq, S <= 8 kernel.  The returned struct holds raw pointers: keep key_valid alive until the launch has been issued."""
    if key_valid is None and batch_split is None:
        return None
    bi, st = (0, 0) if batch_split is None else (int(batch_split[0]), int(batch_split[1]))
    return _lib.AttnMaskC(0 if key_valid is None else key_valid.data_ptr(), 0 if key_valid is None else key_valid.stride(0), bi, st)


def _mask_ref(m):
    return None if m is None else C.byref(m)


def rope_kv(qkv, row_b, row_pos, row_t, cos, sin, q_out, k_cache, v_cache, H, Hkv, D, Lq, Smax):
    M = qkv.shape[0]
    _lib.check(_lib.lib().mc_rope_kv_bf16(_p(qkv), qkv.stride(0), _p(row_b), _p(row_pos), _p(row_t), _p(cos), _p(sin), _p(q_out),
                                          _p(k_cache), _p(v_cache), M, H, Hkv, D, Lq, Smax, _stream()), "mc_rope_kv_bf16")


def attn_prefill(q, k, v, out, B, H, Hkv, Lq, S, D, q_strides, k_strides, v_strides, o_row_stride, causal, q_offset=0,
                 scale=None, out_map=None, kv_lens=None, rel_table=None, rel_off=0, q_gate=None, key_valid=None, batch_split=None):
    scale = (1.0 / math.sqrt(D)) if scale is None else scale
    mk = attn_mask(key_valid, batch_split)
    _lib.check(_lib.lib().mc_attn_prefill_bf16(_p(q), *q_strides, _p(k), *k_strides, _p(v), *v_strides, _p(out), o_row_stride,
                                               _p(out_map), _p(kv_lens), B, H, Hkv, Lq, S, D, 1 if causal else 0, q_offset,
                                               scale, _p(rel_table), 0 if rel_table is None else rel_table.stride(0), rel_off,
                                               _p(q_gate), _mask_ref(mk), _stream()), "mc_attn_prefill_bf16")
    return out


def attn_probs(q, k, B, H, Hkv, Lq, S, D, q_strides, k_strides, causal=True, q_offset=0, scale=None, kv_lens=None, key_valid=None, out=None):
    """softmax(scale q k^T + mask) itself, (B, H, Lq, S) in the storage dtype (mc_attn_probs_bf16: output_attentions)."""
    scale = (1.0 / math.sqrt(D)) if scale is None else scale
    if out is None:
        out = torch.empty(B, H, Lq, S, dtype=q.dtype, device=q.device)
    _lib.check(_lib.lib().mc_attn_probs_bf16(_p(q), *q_strides, _p(k), *k_strides, _p(kv_lens), _p(key_valid),
                                             0 if key_valid is None else key_valid.stride(0), _p(out), B, H, Hkv, Lq, S, D,
                                             1 if causal else 0, q_offset, scale, _stream()), "mc_attn_probs_bf16")
    return out


def decode_workspace(B, H, D, S, device):
    """fp32 scratch of the decode attention: one partial per (b, h) and 512-key chunk of a cache of S positions (+ the new token's)."""
    n = C.c_int64(0)
    _lib.check(_lib.lib().mc_attn_decode_workspace_bytes(B, H, D, S, C.byref(n)), "mc_attn_decode_workspace_bytes")
    return torch.empty(n.value // 4, dtype=torch.float32, device=device)


def attn_decode(q, k, v, out, B, H, Hkv, S, D, q_strides, k_strides, v_strides, o_sb, nsplit=1, workspace=None, scale=None,
                kv_lens=None, key_valid=None):
    scale = (1.0 / math.sqrt(D)) if scale is None else scale
    if workspace is None and (nsplit > 1 or S > 19968):
        workspace = decode_workspace(B, H, D, S, q.device)
    _lib.check(_lib.lib().mc_attn_decode_bf16(_p(q), *q_strides, _p(k), *k_strides, _p(v), *v_strides, _p(out), o_sb,
                                              _p(workspace), _p(kv_lens), B, H, Hkv, S, D, nsplit, scale, _mask_ref(attn_mask(key_valid)), _stream()),
               "mc_attn_decode_bf16")
    return out


def silu_mul(gate_up, I, out=None):
    M = gate_up.shape[0]
    out = torch.empty(M, I, dtype=BF16, device=gate_up.device) if out is None else out
    _lib.check(_lib.lib().mc_silu_mul_bf16(_p(gate_up), gate_up.stride(0), _p(out), out.stride(0), M, I, _stream()), "mc_silu_mul_bf16")
    return out


def copy_rows(src, dst, n_rows, src_idx=None, dst_idx=None):
    D = src.shape[-1]
    _lib.check(_lib.lib().mc_copy_rows_bf16(_p(src), src.stride(-2), _p(src_idx), _p(dst), dst.stride(-2), _p(dst_idx), n_rows, D,
                                            _stream()), "mc_copy_rows_bf16")
    return dst


def embed_rows(table, ids, dst, dst_idx=None):
    n = ids.numel()
    _lib.check(_lib.lib().mc_embed_rows_bf16(_p(table), table.stride(0), _p(ids), _p(dst), dst.stride(-2), _p(dst_idx), n,
                                             table.shape[1], _stream()), "mc_embed_rows_bf16")
    return dst


def argmax(logits_f32, out=None):
    M, N = logits_f32.shape
    out = torch.empty(M, dtype=torch.int64, device=logits_f32.device) if out is None else out
    _lib.check(_lib.lib().mc_argmax_f32(_p(logits_f32), logits_f32.stride(0), _p(out), M, N, _stream()), "mc_argmax_f32")
    return out


def log_softmax(logits_f32, out=None):
    """mc_log_softmax_f32: rows of fp32 logits -> log-probabilities (beam search scoring)."""
    M, N = logits_f32.shape
    out = torch.empty(M, N, dtype=torch.float32, device=logits_f32.device) if out is None else out
    _lib.check(_lib.lib().mc_log_softmax_f32(_p(logits_f32), logits_f32.stride(0), _p(out), out.stride(0), M, N, _stream()), "mc_log_softmax_f32")
    return out


def sample_step(logits_f32, temperature=1.0, top_k=0, top_p=1.0, seed=0, step=0, uniform=None, want_probs=False):
    """One sampled token per row of logits [M, V] fp32 (HF warper order: temperature, top-k, top-p, multinomial).  Returns ids int64 [M]
    (and the final probabilities [M, V] when want_probs)."""
    M, V = logits_f32.shape
    ids = torch.empty(M, dtype=torch.int64, device=logits_f32.device)
    probs = torch.empty(M, V, dtype=torch.float32, device=logits_f32.device) if want_probs else None
    _lib.check(_lib.lib().mc_sample_step_f32(_p(logits_f32), logits_f32.stride(0), _p(ids), None, 0, None, int(step), None, int(seed) & (2 ** 64 - 1),
                                             M, V, float(temperature), int(top_k), float(top_p), _p(uniform), _p(probs), V, _stream()),
               "mc_sample_step_f32")
    return (ids, probs) if want_probs else ids


def im2col(x, kh, kw, sh, sw, Kp=None):
    _req(x, BF16, "x")
    x = x.contiguous()
    B, Cc, Hh, Ww = x.shape
    K = Cc * kh * kw
    Kp = ceil_to(K, 64) if Kp is None else Kp
    oh, ow = (Hh - kh) // sh + 1, (Ww - kw) // sw + 1
    out = torch.empty(B * oh * ow, Kp, dtype=BF16, device=x.device)
    _lib.check(_lib.lib().mc_im2col_bf16(_p(x), _p(out), B, Cc, Hh, Ww, kh, kw, sh, sw, Kp, _stream()), "mc_im2col_bf16")
    return out, oh, ow


def vit_assemble(patches, cls, pos, B, T, D):
    out = torch.empty(B, T + (1 if cls is not None else 0), D, dtype=BF16, device=patches.device)
    _lib.check(_lib.lib().mc_vit_assemble_bf16(_p(patches), _p(cls), _p(pos), _p(out), B, T, D, _stream()), "mc_vit_assemble_bf16")
    return out


def add(a, b, out=None):
    out = torch.empty_like(a) if out is None else out
    _lib.check(_lib.lib().mc_add_bf16(_p(a), _p(b), _p(out), a.numel(), _stream()), "mc_add_bf16")
    return out


# ---- encoder-specific kernels ---------------------------------------------------------------------------
def add_rows(x, table, idx=None, out=None):
    """out[r] = x[r] + table[idx[r]] (idx None -> r)."""
    out = torch.empty_like(x) if out is None else out
    _lib.check(_lib.lib().mc_add_rows_bf16(_p(x), x.stride(0), _p(table), table.stride(0), _p(idx), _p(out), out.stride(0), x.shape[0],
                                           x.shape[1], _stream()), "mc_add_rows_bf16")
    return out


def zero_rows(x, rows):
    if rows.numel():
        _lib.check(_lib.lib().mc_zero_rows_bf16(_p(x), x.stride(0), _p(rows), rows.numel(), x.shape[1], _stream()), "mc_zero_rows_bf16")
    return x


def beats_padding(frame_mask_u8, B, T, span, x, kv_lens, bad_flag):
    """Device-side forward_padding_mask + x[padding_mask] = 0 of BEATs (mc_beats_padding_bf16): fills kv_lens [B] int32, zeroes the padded
    token rows of x [B * T, D], ORs 1 into bad_flag[0] when some clip's padding is not a suffix."""
    _lib.check(_lib.lib().mc_beats_padding_bf16(_p(frame_mask_u8), frame_mask_u8.stride(0), B, T, span, _p(x), x.stride(0), x.shape[1], _p(kv_lens),
                                                _p(bad_flag), _stream()), "mc_beats_padding_bf16")


def im2col_ex(x, strides, B, Cc, Hin, Win, c0, Cg, kh, kw, sh, sw, ph, pw, oh, ow, Kp=None):
    """x: bf16 device tensor addressed as x[b*s_b + c*s_c + y*s_h + x*s_w]."""
    K = Cg * kh * kw
    Kp = ceil_to(K, 64) if Kp is None else Kp
    out = torch.empty(B * oh * ow, Kp, dtype=BF16, device=x.device)
    _lib.check(_lib.lib().mc_im2col_ex_bf16(_p(x), *strides, _p(out), B, Cc, Hin, Win, c0, Cg, kh, kw, sh, sw, ph, pw, oh, ow, Kp,
                                            _stream()), "mc_im2col_ex_bf16")
    return out


def beats_gate(g8, grep_a, B, L, H):
    gate = torch.empty(B, H, L, dtype=torch.float32, device=g8.device)
    _lib.check(_lib.lib().mc_beats_gate_f32(_p(g8), _p(grep_a), _p(gate), B, L, H, _stream()), "mc_beats_gate_f32")
    return gate


def group_max(x, G, n, out=None, bcast=None):
    C_ = x.shape[1]
    if out is None and bcast is None:
        out = torch.empty(G, C_, dtype=BF16, device=x.device)
    _lib.check(_lib.lib().mc_group_max_bf16(_p(x), x.stride(0), _p(out), 0 if out is None else out.stride(0), _p(bcast),
                                            0 if bcast is None else bcast.stride(0), G, n, C_, _stream()), "mc_group_max_bf16")
    return out


def fps(pts, npoint, start_idx=None):
    B, N, Cc = pts.shape
    idx = torch.empty(B, npoint, dtype=torch.int32, device=pts.device)
    centers = torch.empty(B, npoint, 3, dtype=torch.float32, device=pts.device)
    _lib.check(_lib.lib().mc_fps_bf16(_p(pts), B, N, Cc, _p(start_idx), npoint, _p(idx), _p(centers), _stream()), "mc_fps_bf16")
    return idx, centers


def knn_group(pts, centers, k, Kp=64):
    B, N, Cc = pts.shape
    G = centers.shape[1]
    out = torch.empty(B * G * k, Kp, dtype=BF16, device=pts.device)
    idx = torch.empty(B, G, k, dtype=torch.int32, device=pts.device)
    _lib.check(_lib.lib().mc_knn_group_bf16(_p(pts), B, N, Cc, _p(centers), G, k, _p(out), Kp, _p(idx), _stream()), "mc_knn_group_bf16")
    return out, idx


def f32_rows_to_bf16(x, Kp=64):
    rows, Cc = x.shape
    out = torch.empty(rows, Kp, dtype=BF16, device=x.device)
    _lib.check(_lib.lib().mc_f32_rows_to_bf16(_p(x), Cc, _p(out), Kp, rows, _stream()), "mc_f32_rows_to_bf16")
    return out


# ---- training step (csrc/train.hip, csrc/attention_bwd.hip) ---------------------------------------------
def transpose(x, Rp=None, out=None):
    """[R, C] bf16 (row stride free) -> [C, Rp] with zero padded columns R..Rp-1."""
    R, Cc = x.shape
    Rp = R if Rp is None else Rp
    out = torch.empty(Cc, Rp, dtype=BF16, device=x.device) if out is None else out
    _lib.check(_lib.lib().mc_transpose_bf16(_p(x), x.stride(0), _p(out), out.stride(0), R, Cc, Rp, _stream()), "mc_transpose_bf16")
    return out


_tn_ws = {}


def gemm_tn(a_list, b_list, out_list, alpha=1.0):
    """out_i[P, Q] (fp32) = alpha * a_i^T b_i for up to 3 same-shape problems; a_i [M, P], b_i [M, Q] bf16 with contiguous rows."""
    a0, b0 = a_list[0], b_list[0]
    M, P = a0.shape
    Q = b0.shape[1]
    n = len(a_list)
    L = _lib.lib()
    need = C.c_int64(0)
    _lib.check(L.mc_gemm_tn_workspace_floats(M, P, Q, n, C.byref(need)), "mc_gemm_tn_workspace_floats")
    ws = None
    if need.value:
        ws = _tn_ws.get(a0.device)
        if ws is None or ws.numel() < need.value:
            ws = torch.empty(need.value, dtype=torch.float32, device=a0.device)
            _tn_ws[a0.device] = ws
    for t in list(a_list) + list(b_list):
        if t.stride(1) != 1 or t.dtype != BF16:
            raise ValueError("gemm_tn operands must be bf16 with contiguous rows")
    if any(t.stride(0) != a0.stride(0) for t in a_list) or any(t.stride(0) != b0.stride(0) for t in b_list) or \
            any(o.stride(0) != out_list[0].stride(0) or o.dtype != torch.float32 for o in out_list):
        raise ValueError("gemm_tn: the problems of one launch must share strides; outputs are fp32")
    pa = (C.c_void_p * n)(*[t.data_ptr() for t in a_list])
    pb = (C.c_void_p * n)(*[t.data_ptr() for t in b_list])
    po = (C.c_void_p * n)(*[t.data_ptr() for t in out_list])
    _lib.check(L.mc_gemm_tn_bf16(pa, a0.stride(0), pb, b0.stride(0), po, out_list[0].stride(0), n, M, P, Q, float(alpha), _p(ws), _stream()),
               "mc_gemm_tn_bf16")
    return out_list


def pack_weight_t(w_t: torch.Tensor, out: Optional[torch.Tensor] = None) -> PackedWeight:
    """Packed form of W = w_t^T for a row-major w_t [K, N] (no transposed copy in HBM)."""
    _req(w_t, BF16, "w_t")
    K, N = w_t.shape
    if w_t.stride(1) != 1:
        raise ValueError("w_t must have contiguous rows")
    data = torch.empty(packed_elems(N, K), dtype=BF16, device=w_t.device) if out is None else out
    _lib.check(_lib.lib().mc_pack_weight_strided_bf16(_p(w_t), 1, w_t.stride(0), _p(data), N, K, _stream()), "mc_pack_weight_strided_bf16")
    return PackedWeight(data, N, K)


def lora_mask_rows(t, row_adapter, r, n_adapters):
    """t [M, n_linears * n_adapters * r]: zero every r-wide block that does not belong to the row's adapter."""
    _lib.check(_lib.lib().mc_lora_mask_rows_bf16(_p(t), t.stride(0), _p(row_adapter), t.shape[0], r, n_adapters, t.shape[1], _stream()),
               "mc_lora_mask_rows_bf16")
    return t


def rmsnorm_bwd(x, g, dy, eps, dres=None, out=None):
    M, D = x.shape
    out = torch.empty(M, D, dtype=BF16, device=x.device) if out is None else out
    _lib.check(_lib.lib().mc_rmsnorm_bwd_bf16(_p(x), x.stride(0), _p(g), _p(dy), dy.stride(0), _p(dres), 0 if dres is None else dres.stride(0),
                                              _p(out), out.stride(0), M, D, eps, _stream()), "mc_rmsnorm_bwd_bf16")
    return out


def swiglu_bwd(gu, dinter, out=None):
    M, I2 = gu.shape
    out = torch.empty(M, I2, dtype=BF16, device=gu.device) if out is None else out
    _lib.check(_lib.lib().mc_swiglu_bwd_bf16(_p(gu), gu.stride(0), _p(dinter), dinter.stride(0), _p(out), out.stride(0), M, I2 // 2, _stream()),
               "mc_swiglu_bwd_bf16")
    return out


def act(pre, kind, dy=None):
    """dy None: act(pre); else dy * act'(pre).  Contiguous tensors."""
    out = torch.empty_like(pre)
    _lib.check(_lib.lib().mc_act_bf16(_p(pre), _p(dy), _p(out), pre.numel(), ACT[kind], _stream()), "mc_act_bf16")
    return out


def ce_loss(logits_f32, labels, inv_n, want_grad=True):
    """labels int64 [M] (already shifted, < 0 ignored) -> (loss_rows fp32 [M], dlogits bf16 [M, V] = (softmax - onehot) * inv_n);
    want_grad=False skips the gradient (dlogits is None)."""
    M, V = logits_f32.shape
    loss_rows = torch.empty(M, dtype=torch.float32, device=logits_f32.device)
    dl = torch.empty(M, V, dtype=BF16, device=logits_f32.device) if want_grad else None
    _lib.check(_lib.lib().mc_ce_loss_f32(_p(logits_f32), logits_f32.stride(0), _p(labels), _p(loss_rows), _p(dl), dl.stride(0) if want_grad else 0,
                                         M, V, inv_n, _stream()), "mc_ce_loss_f32")
    return loss_rows, dl


def colsum(x, out=None):
    M, Cc = x.shape
    out = torch.empty(Cc, dtype=torch.float32, device=x.device) if out is None else out
    _lib.check(_lib.lib().mc_colsum_bf16(_p(x), x.stride(0), _p(out), M, Cc, _stream()), "mc_colsum_bf16")
    return out


def rope_inplace(x, row_pos, cos, sin, n_heads, D, sign):
    _lib.check(_lib.lib().mc_rope_inplace_bf16(_p(x), x.stride(0), _p(row_pos), _p(cos), _p(sin), x.shape[0], n_heads, D, sign, _stream()),
               "mc_rope_inplace_bf16")
    return x


def attn_prefill_lse(q, k, v, out, lse, B, H, Lq, S, D, q_strides, k_strides, v_strides, o_row_stride, causal, scale=None, kv_lens=None,
                     dropout=None):
    """dropout = (p, seed, stream_id): dropout on the attention probabilities (mc_attn_prefill_dropout_bf16); pass the same triple to attn_bwd."""
    sc = (1.0 / math.sqrt(D)) if scale is None else scale
    if dropout is not None and dropout[0] > 0:
        _lib.check(_lib.lib().mc_attn_prefill_dropout_bf16(_p(q), *q_strides, _p(k), *k_strides, _p(v), *v_strides, _p(out), o_row_stride,
                                                           _p(kv_lens), B, H, H, Lq, S, D, 1 if causal else 0, 0, sc, _p(lse), float(dropout[0]),
                                                           int(dropout[1]) & (2 ** 64 - 1), int(dropout[2]), None, _stream()), "mc_attn_prefill_dropout_bf16")
        return out
    _lib.check(_lib.lib().mc_attn_prefill_lse_bf16(_p(q), *q_strides, _p(k), *k_strides, _p(v), *v_strides, _p(out), o_row_stride, None,
                                                   _p(kv_lens), B, H, H, Lq, S, D, 1 if causal else 0, 0, sc, None, 0, 0, None, _p(lse),
                                                   None, _stream()), "mc_attn_prefill_lse_bf16")
    return out


def attn_bwd(q, k, v, o, d_o, lse, dq, dk, dv, B, H, Lq, S, D, q_strides, k_strides, v_strides, o_strides, dq_strides, dk_strides, dv_strides,
             causal, scale=None, kv_lens=None, dropout=None):
    delta = torch.empty(B * H * Lq, dtype=torch.float32, device=q.device)
    dp, dseed, dstream = (float(dropout[0]), int(dropout[1]) & (2 ** 64 - 1), int(dropout[2])) if dropout is not None else (0.0, 0, 0)
    a = _lib.AttnBwdArgsC(q.data_ptr(), *q_strides, k.data_ptr(), *k_strides, v.data_ptr(), *v_strides, o.data_ptr(), d_o.data_ptr(), *o_strides,
                          lse.data_ptr(), delta.data_ptr(), dq.data_ptr(), *dq_strides, dk.data_ptr(), *dk_strides, dv.data_ptr(), *dv_strides,
                          0 if kv_lens is None else kv_lens.data_ptr(), B, H, Lq, S, D, 1 if causal else 0, 0,
                          (1.0 / math.sqrt(D)) if scale is None else scale, dp, dseed, dstream)
    _lib.check(_lib.lib().mc_attn_bwd_bf16(C.byref(a), _stream()), "mc_attn_bwd_bf16")


def adamw(p32, g32, m, v, p16, lr, beta1, beta2, eps, wd, step, grad_scale=1.0):
    _lib.check(_lib.lib().mc_adamw_f32(_p(p32), _p(g32), _p(m), _p(v), _p(p16), p32.numel(), lr, beta1, beta2, eps, wd, step, grad_scale, _stream()),
               "mc_adamw_f32")


def adamw_segments(p32, g32, m, v, p16, segs_dev, n_segs, lr, lr_alt, beta1, beta2, eps, wd, step, grad_scale=1.0):
    """AdamW with two learning-rate groups chosen per element (mc_adamw_segments_f32; segs_dev: uint8 tensor of mc_adamw_seg records)."""
    _lib.check(_lib.lib().mc_adamw_segments_f32(_p(p32), _p(g32), _p(m), _p(v), _p(p16), _p(segs_dev), n_segs, lr, lr_alt, beta1, beta2, eps, wd,
                                                step, grad_scale, _stream()), "mc_adamw_segments_f32")


def axpy_f32(y, x, alpha=1.0):
    """y += alpha * x (flat fp32)."""
    assert y.dtype == torch.float32 and x.dtype == torch.float32 and y.numel() == x.numel()
    _lib.check(_lib.lib().mc_axpy_f32(_p(y), _p(x), y.numel(), float(alpha), _stream()), "mc_axpy_f32")


def layernorm_bwd(x, g, dy, eps, want_t=True):
    """-> (dx, t = dy * xhat or None): LayerNorm backward w.r.t. the input; dgamma = colsum(t), dbeta = colsum(dy)."""
    M, D = x.shape
    dx = torch.empty(M, D, dtype=BF16, device=x.device)
    t = torch.empty(M, D, dtype=BF16, device=x.device) if want_t else None
    _lib.check(_lib.lib().mc_layernorm_bwd_bf16(_p(x), x.stride(0), _p(g), _p(dy), dy.stride(0), _p(dx), dx.stride(0), _p(t),
                                                0 if t is None else t.stride(0), M, D, float(eps), _stream()), "mc_layernorm_bwd_bf16")
    return dx, t


def dropout(x, p: float, seed: int, stream_id: int, out=None, accumulate: bool = False, alpha: float = 1.0):
    """out = (accumulate ? out : 0) + alpha * x * keep / (1 - p); keep from Philox4x32-10 keyed by (seed, stream_id, element index)."""
    M, K = x.shape
    out = torch.empty(M, K, dtype=BF16, device=x.device) if out is None else out
    _lib.check(_lib.lib().mc_dropout_bf16(_p(x), x.stride(0), _p(out), out.stride(0), M, K, float(p), int(seed) & (2 ** 64 - 1), int(stream_id),
                                          int(accumulate), float(alpha), _stream()), "mc_dropout_bf16")
    return out


def cast_bf16(x32, out=None):
    out = torch.empty(x32.shape, dtype=BF16, device=x32.device) if out is None else out
    _lib.check(_lib.lib().mc_cast_f32_bf16(_p(x32), _p(out), x32.numel(), _stream()), "mc_cast_f32_bf16")
    return out


def attn_decode_rope(qkv, cos, sin, k_cache, v_cache, out, kv_lens, B, H, Hkv, Smax, D, nsplit=1, workspace=None, scale=None, key_valid=None):
    """Decode attention with RoPE + KV append fused (caches [B, Hkv, Smax, D]); kv_lens counts the token being decoded.
    qkv: the [B, (H + 2 Hkv) D] bf16 rows.  nsplit is a launch shape, not part of the result."""
    sc = (1.0 / math.sqrt(D)) if scale is None else scale
    st = (Hkv * Smax * D, D, Smax * D)
    if workspace is None and (nsplit > 1 or Smax > 19968):
        workspace = decode_workspace(B, H, D, Smax, out.device)
    _lib.check(_lib.lib().mc_attn_decode_rope_bf16(_p(qkv), qkv.stride(0), _p(cos), _p(sin), _p(k_cache), *st, _p(v_cache), *st, _p(out),
                                                   out.stride(0), _p(workspace), _p(kv_lens), B, H, Hkv, Smax, D, nsplit, sc,
                                                   _mask_ref(attn_mask(key_valid)), _stream()),
               "mc_attn_decode_rope_bf16")
    return out


# ---- low-precision serving: 4-bit weights, the 8-bit KV cache, logits processing (csrc/gemm_q4.hip, csrc/kv8.hip, csrc/logits.hip) -------
# A decode step's launches last a few microseconds, so the wrappers are kept short: one test of everything a tensor has to be, and a look at what was wrong only
# when it fails.  They launch on the current stream of their tensors' device, whichever device is current.
_fns: dict = {}
_F32, _I32, _I64, _U8 = torch.float32, torch.int32, torch.int64, torch.uint8


def _call(name, index, *args):
    fn = _fns.get(name)
    if fn is None:                                          # (one library per process: _lib.set_storage_dtype)
        fn = _fns[name] = getattr(_lib.lib(), name)
    if index == torch._C._cuda_getDevice():                 # (a tensor of the device exists: HIP is initialised)
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, name)


def _device(t, name):
    """Index of a tensor's device."""
    i = t.get_device()
    if i < 0:
        raise ValueError(f"{name} must be a device (HIP) tensor; this path has no CPU fallback")
    return i


def _arg(t, name, index, dtype, shape):
    """Address of a tensor that has to be of this device, type and shape, with the elements of its last dimension adjacent."""
    if t.get_device() != index or t.dtype != dtype or t.shape != shape or (t.stride(-1) != 1 and shape[-1] > 1):
        if t.get_device() != index:
            raise ValueError(f"{name} must be on device {index}, got {t.device}")
        if t.dtype != dtype:
            raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
        if t.shape != shape:
            raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
        raise ValueError(f"{name}: elements of the last dimension must be adjacent")
    return t.data_ptr()


def _fixed(*names):
    """Class decorator: the public fields are read-only views of the private slots.  The C structs hold the addresses, strides and sizes of construction, so a
    field that could be replaced would be ignored by the next call, and the memory it held would be freed under it."""
    def wrap(cls):
        for n in names:
            setattr(cls, n, property(operator.attrgetter("_" + n)))
        return cls
    return wrap


@_fixed("codes", "scales", "zeros", "N", "K", "group", "index")
class Q4Weight:
    """A linear weight in 4 bits: W[n, k] = scales[n, k // group] * (code[n, k] - zeros[n, k // group]).
    codes uint8 [N, K / 2] (two codes to a byte, even k in the low half), scales [N, K / group] in the storage dtype, zeros uint8 [N, K / group] or None (8);
    group = K // scales.shape[1]: 32, 64 or 128.  bias (storage dtype [N]) as in PackedWeight; it may be set, the other fields are those of construction."""
    __slots__ = ("_codes", "_scales", "_zeros", "_bias", "_N", "_K", "_group", "_index", "_c")

    def __init__(self, codes, scales, zeros=None, bias=None):
        index = _device(codes, "codes")
        if codes.dim() != 2 or scales.dim() != 2:
            raise ValueError("codes must be 2-D [N, K / 2] and scales 2-D [N, K / group]")
        N, half = codes.shape
        G = scales.shape[1]
        K = 2 * half
        group = K // G if G else 0
        if group not in (32, 64, 128) or group * G != K:
            raise ValueError(f"scales give groups of {K}/{G} columns: 32, 64 or 128 are supported")
        pc = _arg(codes, "codes", index, _U8, (N, half))
        ps = _arg(scales, "scales", index, BF16, (N, G))
        pz = 0 if zeros is None else _arg(zeros, "zeros", index, _U8, (N, G))
        # (a single row has no row stride: torch may report anything there)
        one = N < 2
        self._codes, self._scales, self._zeros, self._N, self._K, self._group, self._index = codes, scales, zeros, N, K, group, index
        self.bias = bias
        self._c = _lib.Q4WeightC(pc, half if one else codes.stride(0), ps, G if one else scales.stride(0), pz,
                                 0 if zeros is None else G if one else zeros.stride(0), N, K, group)

    @property
    def bias(self):
        return self._bias

    @bias.setter
    def bias(self, bias):
        if bias is not None:
            _arg(bias, "bias", self._index, BF16, (self._N,))
        self._bias = bias

    @property
    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in (self._codes, self._scales, self._zeros) if t is not None)


def quantize_q4(w: torch.Tensor, group: int = 128, symmetric: bool = True, bias: Optional[torch.Tensor] = None) -> Q4Weight:
    """[N, K] storage dtype -> Q4Weight: symmetric - scale = amax / 7 around code 8; else scale = range / 15 with a zero point per group."""
    _req(w, BF16, "weight")
    if w.dim() != 2 or group not in (32, 64, 128) or w.shape[0] == 0 or w.shape[1] == 0 or w.shape[1] % group:
        raise ValueError(f"weight must be 2-D [N, K] with K a multiple of the group (32, 64 or 128), got {tuple(w.shape)} and {group}")
    if w.stride(1) != 1 or w.stride(0) % 8 or w.stride(0) < w.shape[1] or w.data_ptr() % 16:
        w = w.clone(memory_format=torch.contiguous_format)      # (contiguous() keeps a contiguous weight at its odd address)
    N, K = w.shape
    codes = torch.empty(N, K // 2, dtype=_U8, device=w.device)
    scales = torch.empty(N, K // group, dtype=BF16, device=w.device)
    zeros = None if symmetric else torch.empty(N, K // group, dtype=_U8, device=w.device)
    _call("mc_quantize_q4_bf16", w.get_device(), w.data_ptr(), w.stride(0) if N > 1 else K, codes.data_ptr(), scales.data_ptr(),
          0 if zeros is None else zeros.data_ptr(), N, K, group)
    return Q4Weight(codes, scales, zeros, bias)


def dequantize_q4(w: Q4Weight) -> PackedWeight:
    """The 16-bit PackedWeight of a 4-bit weight (each element rounded once): linear() with more than 64 rows."""
    out = torch.empty(packed_elems(w._N, w._K), dtype=BF16, device=w._codes.device)
    _call("mc_dequantize_q4_bf16", w._index, C.byref(w._c), out.data_ptr())
    return PackedWeight(out, w._N, w._K, w._bias)


def linear_q4(x: torch.Tensor, w: Q4Weight, residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, out_f32: bool = False,
              bias: bool = True) -> torch.Tensor:
    """out[M, N] = x W^T (+ bias) (+ residual) for at most 64 rows x [M, K] (the decode step's form of linear(); larger launches: linear(x,
    dequantize_q4(w)), with x padded to its Kp).  fp32 sums; the codes enter as exact integers, the zero point as zero * sum(x); an infinity in x gives the
    infinities and NaN of linear().  A row's bits do not depend on M.  out may be the residual, but may not overlap x."""
    index = _device(x, "x")
    if x.dim() != 2:
        raise ValueError("x must be 2-D [M, K]")
    M, N, dt = x.shape[0], w._N, _F32 if out_f32 else BF16
    px = _arg(x, "x", index, BF16, (M, w._K))
    if M > 64:
        raise ValueError(f"linear_q4 takes at most 64 rows, got {M}: use linear(x, dequantize_q4(w))")
    if w._index != index:
        raise ValueError(f"the weight is on device {w._index}, x on device {index}")
    if out is None:
        out = torch.empty((M, N), dtype=_F32, device=x.device) if out_f32 else x.new_empty((M, N))
        po, ldo = out.data_ptr(), N
    else:
        po, ldo = _arg(out, "out", index, dt, (M, N)), out.stride(0)
    pr, ldr = (0, 0) if residual is None else (_arg(residual, "residual", index, BF16, (M, N)), residual.stride(0))
    if M:
        # (mc_linear_q4_workspace_bytes)
        ws = torch.empty((M + 15) // 16 * 16 * w._K, dtype=BF16, device=x.device) if M > 16 else None
        _call("mc_linear_q4_bf16", index, px, x.stride(0) if M > 1 else w._K, w._c, w._bias.data_ptr() if bias and w._bias is not None else 0, pr, ldr, po, ldo, M,
              1 if out_f32 else 0, 0 if ws is None else ws.data_ptr())
    return out


@_fixed("k", "k_scale", "v", "v_scale", "B", "Hkv", "S", "D", "index")
class Kv8Cache:
    """An 8-bit KV cache of one layer: codes k, v [B, Hkv, S, D] (torch.float8_e4m3fn or torch.int8, equal strides, head_dim contiguous) and their fp32
    scales k_scale, v_scale [B, Hkv, S], one per vector.  kv8_cache() makes one; slices over the batch of an existing one are caches too.
    The fields are those of construction: a grown cache is a new one."""
    __slots__ = ("_k", "_k_scale", "_v", "_v_scale", "_B", "_Hkv", "_S", "_D", "_index", "_c")
    _formats = {torch.float8_e4m3fn: 1, torch.int8: 2}

    def __init__(self, k, k_scale, v, v_scale):
        index = _device(k, "the cache")
        fmt = self._formats.get(k.dtype)
        if fmt is None or k.dim() != 4:
            raise ValueError(f"codes must be float8_e4m3fn or int8 [B, Hkv, S, D], got {k.dtype} {tuple(k.shape)}")
        B, Hkv, S, D = shape = k.shape
        pk, pv = _arg(k, "k", index, k.dtype, shape), _arg(v, "v", index, k.dtype, shape)
        pks, pvs = _arg(k_scale, "k_scale", index, _F32, shape[:3]), _arg(v_scale, "v_scale", index, _F32, shape[:3])
        st, ss = k.stride(), k_scale.stride()
        if st != v.stride() or ss != v_scale.stride():
            raise ValueError("k and v (and their scales) must have the same strides")
        # (a dimension of size 1 has no stride: torch may report anything there)
        sb, sh, sp = st[0] if B > 1 else D, st[1] if Hkv > 1 else D, st[2] if S > 1 else D
        zb, zh = ss[0] if B > 1 else 1, ss[1] if Hkv > 1 else 1
        if not (sb > 0 and sh > 0 and sp > 0 and zb > 0 and zh > 0):
            raise ValueError("a cache has no broadcast dimensions")
        self._k, self._k_scale, self._v, self._v_scale, self._B, self._Hkv, self._S, self._D, self._index = k, k_scale, v, v_scale, B, Hkv, S, D, index
        self._c = _lib.Kv8CacheC(pk, pks, pv, pvs, sb, sh, sp, zb, zh, B, Hkv, S, D, fmt)

    @property
    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in (self._k, self._k_scale, self._v, self._v_scale))


def kv8_cache(B, Hkv, S, D, device="cuda", dtype=torch.float8_e4m3fn) -> Kv8Cache:
    """An empty (all zero) cache of S positions."""
    z = lambda dt, *s: torch.zeros(s, dtype=dt, device=device)
    k, v = (z(_U8, B, Hkv, S, D).view(dtype) for _ in range(2))
    return Kv8Cache(k, z(_F32, B, Hkv, S), v, z(_F32, B, Hkv, S))


def _rope_args(qkv, cos, sin, cache, H, rows):
    index, width = _device(qkv, "qkv"), (H + 2 * cache._Hkv) * cache._D
    p = _arg(qkv, "qkv", index, BF16, (rows, width))
    if cache._index != index:
        raise ValueError(f"the cache is on device {cache._index}, qkv on device {index}")
    n_pos = cos.shape[0]
    pc, ps = _arg(cos, "cos", index, _F32, (n_pos, cache._D // 2)), _arg(sin, "sin", index, _F32, (n_pos, cache._D // 2))
    if not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("cos and sin must be contiguous")
    return index, p, qkv.stride(0) if rows > 1 else width, pc, ps, n_pos


def rope_kv8(qkv, row_b, row_pos, row_t, cos, sin, q_out, cache: Kv8Cache, H, Lq):
    """rope_kv() for an 8-bit cache: rows [M, (H + 2 Hkv) D] of a q|k|v projection -> rotated queries in q_out [B * Lq, H * D] (row row_b * Lq + row_t), rotated keys and the
    values quantised to position row_pos of sequence row_b.  Rows with row_b < 0, or outside the cache, the tables or q_out, are skipped; a position is
    written by at most one row of a call."""
    M = qkv.shape[0]
    index, p, ld, pc, ps, n_pos = _rope_args(qkv, cos, sin, cache, H, M)
    rb, rp, rt = _arg(row_b, "row_b", index, _I32, (M,)), _arg(row_pos, "row_pos", index, _I32, (M,)), _arg(row_t, "row_t", index, _I32, (M,))
    pq = _arg(q_out, "q_out", index, BF16, q_out.shape)
    if not q_out.is_contiguous() or q_out.numel() != cache._B * Lq * H * cache._D:
        raise ValueError(f"q_out must hold {cache._B} x {Lq} contiguous rows of {H * cache._D}")
    if M:
        _call("mc_rope_kv8", index, p, ld, rb, rp, rt, pc, ps, n_pos, pq, cache._c, M, H, Lq)
    return q_out


def kv8_read(cache: Kv8Cache, n=None, kv_lens=None):
    """The first n (default: all) positions in the storage dtype: (k, v) [B, Hkv, n, D]; positions from kv_lens[b] on are zeros.  What attn_prefill reads when a
    later chunk of a prompt attends to keys that are in the cache already."""
    n = cache._S if n is None else int(n)
    pl = 0 if kv_lens is None else _arg(kv_lens, "kv_lens", cache._index, _I32, (cache._B,))
    if n < 0 or n > cache._S:
        raise ValueError(f"{n} positions of a cache of {cache._S}")
    k = torch.empty((cache._B, cache._Hkv, n, cache._D), dtype=BF16, device=cache._k.device)
    v = torch.empty_like(k)
    if n:
        _call("mc_kv8_read", cache._index, cache._c, pl, n, k.data_ptr(), v.data_ptr())
    return k, v


_decode8_ws: dict = {}          # (B, H, D, S) -> bytes of scratch


def _decode8_scratch(B, H, D, S):
    n = C.c_int64(0)
    _lib.check(_lib.lib().mc_attn_decode8_workspace_bytes(B, H, D, S, C.byref(n)), "mc_attn_decode8_workspace_bytes")
    if len(_decode8_ws) >= 4096:
        _decode8_ws.clear()
    _decode8_ws[(B, H, D, S)] = n.value
    return n.value


def _decode8(name, head, x, cache, H, kv_lens, out, scale, key_valid):
    """The arguments that attn_decode8 and attn_decode8_rope share, and the call.  The scratch is the caching allocator's: calls in flight on other streams, and
    captured graphs, have their own."""
    B, D, S, index = cache._B, cache._D, cache._S, cache._index
    pl = 0 if kv_lens is None else _arg(kv_lens, "kv_lens", index, _I32, (B,))
    pm = ms = 0
    if key_valid is not None:
        if key_valid.dtype == torch.bool:
            key_valid = key_valid.view(_U8)
        if key_valid.dim() != 2 or key_valid.shape[1] < S:
            raise ValueError(f"key_valid must be [B, >= {S}], got {tuple(key_valid.shape)}")
        pm, ms = _arg(key_valid, "key_valid", index, _U8, (B, key_valid.shape[1])), key_valid.stride(0)
    if out is None:
        out = x.new_empty((B, H * D))
        po, so = out.data_ptr(), H * D
    else:
        po, so = _arg(out, "out", index, BF16, (B, H * D)), out.stride(0)
    ws = torch.empty(_decode8_ws.get((B, H, D, S)) or _decode8_scratch(B, H, D, S), dtype=_U8, device=x.device)
    _call(name, index, *head, cache._c, pl, pm, ms, po, so, ws.data_ptr(), H, D ** -0.5 if scale is None else scale)
    return out


def attn_decode8(q, cache: Kv8Cache, kv_lens=None, out=None, scale=None, key_valid=None):
    """Decode attention over an 8-bit cache: q [B, H, D] (one rotated query per sequence; H a multiple of Hkv), kv_lens int32 [B] (None: every position) ->
    out [B, H * D].  key_valid uint8 / bool [B, >= S]: 0 = masked.  A sequence without a key gives zeros.  out may not overlap q."""
    index = _device(q, "q")
    if q.dim() != 3:
        raise ValueError("q must be [B, H, D]")
    H = q.shape[1]
    pq = _arg(q, "q", index, BF16, (cache._B, H, cache._D))
    if cache._index != index:
        raise ValueError(f"the cache is on device {cache._index}, q on device {index}")
    return _decode8("mc_attn_decode8", (pq, q.stride(0) if cache._B > 1 else cache._D, q.stride(1) if H > 1 else cache._D), q, cache, H, kv_lens, out, scale, key_valid)


def attn_decode8_rope(qkv, cos, sin, cache: Kv8Cache, kv_lens, H, out=None, scale=None, key_valid=None):
    """attn_decode_rope() over an 8-bit cache: the pre-rotary rows qkv [B, (H + 2 Hkv) D] of the tokens at positions kv_lens[b] - 1 (kv_lens int32 [B] counts them)
    are rotated, appended to the cache and attended.  A sequence with kv_lens[b] outside 1 .. min(S, rows of cos) is left alone: zeros, nothing written."""
    if kv_lens is None:
        raise ValueError("kv_lens is needed: it places the new token")
    index, p, ld, pc, ps, n_pos = _rope_args(qkv, cos, sin, cache, H, cache._B)
    return _decode8("mc_attn_decode8_rope", (p, ld, pc, ps, n_pos), qkv, cache, H, kv_lens, out, scale, key_valid)


def logits_process(logits, prompt_ids=None, prompt_lens=None, output_ids=None, output_lens=None, repetition_penalty=None, presence_penalty=None,
                   frequency_penalty=None, bias_ids=None, bias=None, allowed=None, out=None):
    """Penalties, biases and a token mask on logits [M, V] fp32, before argmax() / sample_step() (out=logits: in place).
    prompt_ids / output_ids int64 [M, n] with optional int32 lengths [M]: the repetition penalty (l / r or l * r) reads both, frequency * count + presence
    only the output ids.  The penalties are fp32 tensors [M]; bias_ids int32 [M, n] with bias fp32 [M, n] (a token may be listed twice: the biases add up);
    allowed int32 [M, ceil(V / 32)]: bit t & 31 of word t >> 5 clear = -inf.  Ids outside [0, V) are ignored:
    ragged lists are padded with -1.
    out is logits itself or does not overlap it."""
    index = _device(logits, "logits")
    if logits.dim() != 2:
        raise ValueError("logits must be 2-D [M, V]")
    M, V = logits.shape
    pl = _arg(logits, "logits", index, _F32, (M, V))
    if out is None:
        out = logits.new_empty((M, V))
        po, ldo = out.data_ptr(), V
    else:
        po, ldo = _arg(out, "out", index, _F32, (M, V)), out.stride(0)
    pp = ldp = ppl = np_ = pq = ldq = pql = nq = p1 = p2 = p3 = 0
    if prompt_ids is not None:
        if prompt_ids.dim() != 2:
            raise ValueError("prompt_ids must be 2-D [M, n]")
        np_, ldp = prompt_ids.shape[1], prompt_ids.stride(0)
        pp = _arg(prompt_ids, "prompt_ids", index, _I64, (M, np_))
        if prompt_lens is not None:
            ppl = _arg(prompt_lens, "prompt_lens", index, _I32, (M,))
    elif prompt_lens is not None:
        raise ValueError("prompt_lens without prompt_ids")
    if output_ids is not None:
        if output_ids.dim() != 2:
            raise ValueError("output_ids must be 2-D [M, n]")
        nq, ldq = output_ids.shape[1], output_ids.stride(0)
        pq = _arg(output_ids, "output_ids", index, _I64, (M, nq))
        if output_lens is not None:
            pql = _arg(output_lens, "output_lens", index, _I32, (M,))
    elif output_lens is not None:
        raise ValueError("output_lens without output_ids")
    if repetition_penalty is not None:
        p1 = _arg(repetition_penalty, "repetition_penalty", index, _F32, (M,))
    if presence_penalty is not None:
        p2 = _arg(presence_penalty, "presence_penalty", index, _F32, (M,))
    if frequency_penalty is not None:
        p3 = _arg(frequency_penalty, "frequency_penalty", index, _F32, (M,))
    pb = pv = ldb = nb = pa = lda = 0
    if (bias_ids is None) != (bias is None):
        raise ValueError("bias_ids and bias go together")
    if bias is not None:
        if bias.dim() != 2:
            raise ValueError("bias must be 2-D [M, n]")
        nb, ldb = bias.shape[1], bias.stride(0)
        pb, pv = _arg(bias_ids, "bias_ids", index, _I32, (M, nb)), _arg(bias, "bias", index, _F32, (M, nb))
        if M > 1 and bias_ids.stride(0) != ldb:
            raise ValueError("bias_ids and bias must have the same row stride")
    if allowed is not None:
        pa, lda = _arg(allowed, "allowed", index, _I32, (M, (V + 31) // 32)), allowed.stride(0)
    if M and V:
        _call("mc_logits_process_f32", index, _lib.LogitsArgsC(pl, logits.stride(0), po, ldo, M, V, pp, ldp, ppl, np_, pq, ldq, pql, nq, p1, p2, p3, pb, pv, ldb, nb, pa, lda))
    return out
