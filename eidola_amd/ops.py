"""Operator-level host API over the C ABI: tensors in, status-checked launches out.

Every function takes torch tensors that already live on the GPU, checks dtype/shape/
contiguity on the host, and passes raw device pointers plus the current HIP stream to the
library.  Nothing here computes attention: if the HIP library is absent the call raises.
"""
import ctypes as C
import math
from array import array
from dataclasses import dataclass

import numpy as np
import torch

from . import _lib
from ._lib import AttnArgs, AttnDesc, KV_BF16, KV_FP8_E4M3, check, load_library


@dataclass
class AttnGeometry:
    """Static shape of one attention layer and its paged KV cache."""
    num_q_heads: int = 64
    num_kv_heads: int = 8
    head_dim: int = 64
    block_size: int = 16
    softmax_scale: float = 0.125
    window: int = 0          # 0 = full causal
    kv_dtype: int = KV_BF16
    partition_size: int = 0  # 0 = library picks


def make_desc(geom, *, num_seqs, num_q_tokens, max_q_len, max_kv_len, max_blocks_per_seq,
              num_blocks, sum_kv_len=0):
    d = AttnDesc()
    d.struct_size = C.sizeof(AttnDesc)
    d.num_seqs = num_seqs
    d.num_q_tokens = num_q_tokens
    d.max_q_len = max_q_len
    d.max_kv_len = max_kv_len
    d.num_q_heads = geom.num_q_heads
    d.num_kv_heads = geom.num_kv_heads
    d.head_dim = geom.head_dim
    d.block_size = geom.block_size
    d.max_blocks_per_seq = max_blocks_per_seq
    d.num_blocks = num_blocks
    d.softmax_scale = geom.softmax_scale
    d.window = geom.window
    d.kv_dtype = geom.kv_dtype
    d.partition_size = geom.partition_size
    d.sum_kv_len = sum_kv_len  # host-side sum of seq_lens (or an upper bound), 0 = unknown
    return d


def workspace_bytes(desc):
    return load_library().eid_workspace_bytes(C.byref(desc))


def partition_size(desc):
    return load_library().eid_partition_size(C.byref(desc))


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _kv_torch_dtype(kv_dtype):
    return torch.bfloat16 if kv_dtype == KV_BF16 else torch.uint8


def _require(t, name, dtype, ndim=None):
    if t is None:
        raise ValueError(f"{name} is None")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dims, got {t.dim()}")


def _cache_view(t, geom, name):
    """Accept fp8 caches as uint8 or torch.float8_e4m3fn storage."""
    if geom.kv_dtype == KV_FP8_E4M3 and t.dtype == torch.float8_e4m3fn:
        t = t.view(torch.uint8)
    _require(t, name, _kv_torch_dtype(geom.kv_dtype), 4)
    if tuple(t.shape[1:]) != (geom.block_size, geom.num_kv_heads, geom.head_dim):
        raise ValueError(f"{name} must be [num_blocks, {geom.block_size}, {geom.num_kv_heads}, "
                         f"{geom.head_dim}], got {tuple(t.shape)}")
    return t


def kv_write(geom, k_new, v_new, k_cache, v_cache, slot_mapping, k_scale=None, v_scale=None):
    """Stage K1: cache_flat[slot_mapping[t]] = k_new[t] (bit copy, or fp8 quantise)."""
    _require(k_new, "k_new", torch.bfloat16, 3)
    _require(v_new, "v_new", torch.bfloat16, 3)
    k_cache = _cache_view(k_cache, geom, "k_cache")
    v_cache = _cache_view(v_cache, geom, "v_cache")
    _require(slot_mapping, "slot_mapping", torch.int64, 1)
    T = k_new.shape[0]
    if tuple(k_new.shape) != (T, geom.num_kv_heads, geom.head_dim) or k_new.shape != v_new.shape:
        raise ValueError("k_new / v_new must be [T, num_kv_heads, head_dim]")
    if slot_mapping.shape[0] != T:
        raise ValueError("slot_mapping must have one entry per new token")
    if k_cache.shape != v_cache.shape:
        raise ValueError("k_cache and v_cache shapes differ")
    if geom.kv_dtype == KV_FP8_E4M3:
        _require(k_scale, "k_scale", torch.float32, 1)
        _require(v_scale, "v_scale", torch.float32, 1)
    desc = make_desc(geom, num_seqs=1, num_q_tokens=1, max_q_len=1, max_kv_len=1,
                     max_blocks_per_seq=1, num_blocks=k_cache.shape[0])
    check(load_library().eid_kv_write(C.byref(desc), _ptr(k_new), _ptr(v_new), _ptr(k_cache),
                                      _ptr(v_cache), _ptr(slot_mapping), T, _ptr(k_scale),
                                      _ptr(v_scale), _stream()))


def rope_kv_write(geom, qkv, positions, cos_sin, k_cache, v_cache, slot_mapping, k_scale=None,
                  v_scale=None, q_out=None):
    """Fused RoPE + QKV split + slot-mapped KV write.  qkv is [T, (Hq + 2 Hkv) * D] bf16,
    cos_sin [max_pos, D] fp32 (per position D/2 cosines then D/2 sines); returns q_out
    [T, Hq, D] bf16."""
    _require(qkv, "qkv", torch.bfloat16, 2)
    _require(positions, "positions", torch.int32, 1)
    _require(cos_sin, "cos_sin", torch.float32, 2)
    k_cache = _cache_view(k_cache, geom, "k_cache")
    v_cache = _cache_view(v_cache, geom, "v_cache")
    _require(slot_mapping, "slot_mapping", torch.int64, 1)
    T = qkv.shape[0]
    if qkv.shape[1] != (geom.num_q_heads + 2 * geom.num_kv_heads) * geom.head_dim:
        raise ValueError("qkv must be [T, (num_q_heads + 2 num_kv_heads) * head_dim]")
    if positions.shape[0] != T or slot_mapping.shape[0] != T:
        raise ValueError("positions and slot_mapping must have one entry per token")
    if cos_sin.shape[1] != geom.head_dim:
        raise ValueError("cos_sin must be [max_pos, head_dim]")
    if geom.kv_dtype == KV_FP8_E4M3:
        _require(k_scale, "k_scale", torch.float32, 1)
        _require(v_scale, "v_scale", torch.float32, 1)
    if q_out is None:
        q_out = torch.empty((T, geom.num_q_heads, geom.head_dim), dtype=torch.bfloat16,
                            device=qkv.device)
    else:
        _require(q_out, "q_out", torch.bfloat16, 3)
    desc = make_desc(geom, num_seqs=1, num_q_tokens=1, max_q_len=1, max_kv_len=1,
                     max_blocks_per_seq=1, num_blocks=k_cache.shape[0])
    check(load_library().eid_rope_kv_write(
        C.byref(desc), _ptr(qkv), _ptr(positions), _ptr(cos_sin), cos_sin.shape[0], _ptr(q_out),
        _ptr(k_cache), _ptr(v_cache), _ptr(slot_mapping), T, _ptr(k_scale), _ptr(v_scale),
        _stream()))
    return q_out


def qkv_rope_kv_write(geom, hidden, weight, bias, positions, cos_sin, k_cache, v_cache,
                      slot_mapping, k_scale=None, v_scale=None, q_out=None):
    """QKV projection + rope_kv_write in one launch (at most 64 tokens): hidden [T, K] bf16,
    weight [(Hq + 2 Hkv) * D, K] bf16, bias [(Hq + 2 Hkv) * D] bf16 or None; the rest as
    rope_kv_write.  Returns q_out [T, Hq, D] bf16; bit-identical to o_proj + rope_kv_write."""
    _require(hidden, "hidden", torch.bfloat16, 2)
    _require(weight, "weight", torch.bfloat16, 2)
    _require(positions, "positions", torch.int32, 1)
    _require(cos_sin, "cos_sin", torch.float32, 2)
    k_cache = _cache_view(k_cache, geom, "k_cache")
    v_cache = _cache_view(v_cache, geom, "v_cache")
    _require(slot_mapping, "slot_mapping", torch.int64, 1)
    T, K = hidden.shape
    N = (geom.num_q_heads + 2 * geom.num_kv_heads) * geom.head_dim
    if tuple(weight.shape) != (N, K):
        raise ValueError(f"weight must be [{N}, {K}]")
    if bias is not None:
        _require(bias, "bias", torch.bfloat16, 1)
        if bias.shape[0] != N:
            raise ValueError(f"bias must be [{N}]")
    if positions.shape[0] != T or slot_mapping.shape[0] != T:
        raise ValueError("positions and slot_mapping must have one entry per token")
    if cos_sin.shape[1] != geom.head_dim:
        raise ValueError("cos_sin must be [max_pos, head_dim]")
    if geom.kv_dtype == KV_FP8_E4M3:
        _require(k_scale, "k_scale", torch.float32, 1)
        _require(v_scale, "v_scale", torch.float32, 1)
    if q_out is None:
        q_out = torch.empty((T, geom.num_q_heads, geom.head_dim), dtype=torch.bfloat16,
                            device=hidden.device)
    else:
        _require(q_out, "q_out", torch.bfloat16, 3)
    desc = make_desc(geom, num_seqs=1, num_q_tokens=1, max_q_len=1, max_kv_len=1,
                     max_blocks_per_seq=1, num_blocks=k_cache.shape[0])
    check(load_library().eid_qkv_rope_kv_write(
        C.byref(desc), _ptr(hidden), _ptr(weight), _ptr(bias), K, _ptr(positions), _ptr(cos_sin),
        cos_sin.shape[0], _ptr(q_out), _ptr(k_cache), _ptr(v_cache), _ptr(slot_mapping), T,
        _ptr(k_scale), _ptr(v_scale), _stream()))
    return q_out


def o_proj(attn_out, weight, bias=None, residual=None, out=None):
    """Output projection after attention: attn_out [T, Hq, D] (or [T, K]) bf16, weight [N, K]
    bf16 (out_features x in_features), optional bias [N] and residual [T, N] bf16; returns
    out [T, N] bf16 = attn_out @ weight^T + bias + residual (fp32 sums, one bf16 rounding).
    `out` may be the residual buffer itself."""
    if attn_out.dim() == 3:
        attn_out = attn_out.reshape(attn_out.shape[0], -1)
    _require(attn_out, "attn_out", torch.bfloat16, 2)
    _require(weight, "weight", torch.bfloat16, 2)
    T, K = attn_out.shape
    N = weight.shape[0]
    if weight.shape[1] != K:
        raise ValueError("weight must be [out_features, in_features] with in_features = %d" % K)
    if bias is not None:
        _require(bias, "bias", torch.bfloat16, 1)
        if bias.shape[0] != N:
            raise ValueError("bias must be [out_features]")
    if residual is not None:
        _require(residual, "residual", torch.bfloat16, 2)
        if tuple(residual.shape) != (T, N):
            raise ValueError("residual must be [T, out_features]")
    if out is None:
        out = torch.empty((T, N), dtype=torch.bfloat16, device=attn_out.device)
    else:
        _require(out, "out", torch.bfloat16, 2)
        if tuple(out.shape) != (T, N):
            raise ValueError("out must be [T, out_features]")
    check(load_library().eid_o_proj(_ptr(attn_out), _ptr(weight), _ptr(bias), _ptr(residual),
                                    _ptr(out), T, N, K, _stream()))
    return out


def yarn_cos_sin(max_pos, head_dim=64, base=150000.0, scaling_factor=32.0,
                 initial_context=4096.0, ntk_alpha=1.0, ntk_beta=32.0):
    """[max_pos, head_dim] fp32 table for eid_rope_kv_write (numpy): per position head_dim/2
    cosines then head_dim/2 sines with YaRN "NTK-by-parts" frequency blending and the
    attention-temperature factor 0.1 ln(scaling_factor) + 1 folded in, as the published
    gpt-oss model definition describes its rotary embedding (defaults are that model's
    configuration).  scaling_factor <= 1 gives plain RoPE."""
    half = head_dim // 2
    freq = base ** (np.arange(0, head_dim, 2, dtype=np.float64) / head_dim)
    if scaling_factor > 1.0:
        concentration = 0.1 * np.log(scaling_factor) + 1.0
        low = half * np.log(initial_context / (ntk_beta * 2 * np.pi)) / np.log(base)
        high = half * np.log(initial_context / (ntk_alpha * 2 * np.pi)) / np.log(base)
        ramp = (np.arange(half, dtype=np.float64) - low) / (high - low)
        mask = 1.0 - np.clip(ramp, 0.0, 1.0)
        inv_freq = (1.0 / (scaling_factor * freq)) * (1.0 - mask) + (1.0 / freq) * mask
    else:
        concentration = 1.0
        inv_freq = 1.0 / freq
    ang = np.arange(max_pos, dtype=np.float64)[:, None] * inv_freq[None, :]
    return np.concatenate([np.cos(ang) * concentration, np.sin(ang) * concentration],
                          axis=1).astype(np.float32)


def _host_i32(a, name, n):
    """A host copy of a length array as contiguous int32 numpy (the library reads it during
    the call); accepts numpy arrays and CPU tensors."""
    if a is None:
        return None
    if isinstance(a, torch.Tensor):
        if a.is_cuda:
            raise ValueError(f"{name} must live in host memory")
        a = a.numpy()
    a = np.ascontiguousarray(a, dtype=np.int32)
    if a.shape != (n,):
        raise ValueError(f"{name} must have {n} entries")
    return a


def _host_bt(a, block_table):
    """A host copy of the block table as contiguous int32 numpy of the device table's shape."""
    if a is None:
        return None
    if isinstance(a, torch.Tensor):
        if a.is_cuda:
            raise ValueError("block_table_host must live in host memory")
        a = a.numpy()
    a = np.ascontiguousarray(a, dtype=np.int32)
    if a.shape != tuple(block_table.shape):
        raise ValueError("block_table_host must have the shape of block_table")
    return a


def _attn_call(fn_name, geom, q, k_cache, v_cache, block_table, seq_lens, cu_seqlens_q,
               max_q_len, max_kv_len, sinks, k_scale, v_scale, out, lse, workspace,
               return_lse, sum_kv_len=0, k_new=None, v_new=None, seq_lens_host=None,
               cu_seqlens_q_host=None, block_table_host=None):
    _require(q, "q", torch.bfloat16, 3)
    k_cache = _cache_view(k_cache, geom, "k_cache")
    v_cache = _cache_view(v_cache, geom, "v_cache")
    _require(block_table, "block_table", torch.int32, 2)
    _require(seq_lens, "seq_lens", torch.int32, 1)
    S = seq_lens.shape[0]
    T = q.shape[0]
    if tuple(q.shape[1:]) != (geom.num_q_heads, geom.head_dim):
        raise ValueError("q must be [T, num_q_heads, head_dim]")
    if block_table.shape[0] != S:
        raise ValueError("block_table must have one row per sequence")
    if cu_seqlens_q is not None:
        _require(cu_seqlens_q, "cu_seqlens_q", torch.int32, 1)
        if cu_seqlens_q.shape[0] != S + 1:
            raise ValueError("cu_seqlens_q must have num_seqs + 1 entries")
    if sinks is not None:
        _require(sinks, "sinks", torch.float32, 1)
    if geom.kv_dtype == KV_FP8_E4M3:
        _require(k_scale, "k_scale", torch.float32, 1)
        _require(v_scale, "v_scale", torch.float32, 1)
    desc = make_desc(geom, num_seqs=S, num_q_tokens=T, max_q_len=max_q_len,
                     max_kv_len=max_kv_len, max_blocks_per_seq=block_table.shape[1],
                     num_blocks=k_cache.shape[0], sum_kv_len=sum_kv_len)
    if out is None:
        out = torch.empty_like(q)
    else:
        _require(out, "out", torch.bfloat16, 3)
    if return_lse and lse is None:
        lse = torch.empty((T, geom.num_q_heads), dtype=torch.float32, device=q.device)
    lib = load_library()
    need = lib.eid_workspace_bytes(C.byref(desc))
    if need == 0:
        check(getattr(lib, fn_name)(C.byref(desc), C.byref(AttnArgs()), None))
    own_ws = fn_name == "eid_attn_decode_noalloc"   # the library's static array serves it
    if workspace is None and not own_ws:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    args = AttnArgs()
    args.q = q.data_ptr()
    args.out = out.data_ptr()
    args.lse = lse.data_ptr() if lse is not None else None
    args.k_cache = k_cache.data_ptr()
    args.v_cache = v_cache.data_ptr()
    args.block_table = block_table.data_ptr()
    args.cu_seqlens_q = cu_seqlens_q.data_ptr() if cu_seqlens_q is not None else None
    args.seq_lens = seq_lens.data_ptr()
    args.sinks = sinks.data_ptr() if sinks is not None else None
    args.k_scale = k_scale.data_ptr() if k_scale is not None else None
    args.v_scale = v_scale.data_ptr() if v_scale is not None else None
    if not own_ws:
        args.workspace = workspace.data_ptr()
        args.workspace_bytes = workspace.numel() * workspace.element_size()
    for name, t in (("k_new", k_new), ("v_new", v_new)):
        if t is not None:
            _require(t, name, torch.bfloat16, 3)
            if tuple(t.shape) != (S, geom.num_kv_heads, geom.head_dim):
                raise ValueError(f"{name} must be [num_seqs, num_kv_heads, head_dim]")
            setattr(args, name, t.data_ptr())
    sl_h = _host_i32(seq_lens_host, "seq_lens_host", S)
    cu_h = _host_i32(cu_seqlens_q_host, "cu_seqlens_q_host", S + 1)
    args.seq_lens_host = sl_h.ctypes.data if sl_h is not None else None
    args.cu_seqlens_q_host = cu_h.ctypes.data if cu_h is not None else None
    bt_h = _host_bt(block_table_host, block_table)
    args.block_table_host = bt_h.ctypes.data if bt_h is not None else None
    check(getattr(lib, fn_name)(C.byref(desc), C.byref(args), _stream()))
    return (out, lse) if return_lse else out


class PreparedCall:
    """A validated (desc, args) pair bound to one entry point: calling it only crosses the
    C ABI (no tensor checks, no allocation), for launch-rate-sensitive loops.  The tensors
    are kept alive by the object."""

    def __init__(self, fn_name, desc, args, keep, out, lse):
        self._fn = getattr(load_library(), fn_name)
        self.desc, self.args, self._keep, self.out, self.lse = desc, args, keep, out, lse
        self._d, self._a = C.byref(desc), C.byref(args)

    def __call__(self, stream=None):
        st = _stream() if stream is None else C.c_void_p(stream)
        rc = self._fn(self._d, self._a, st)
        if rc:
            check(rc)
        return self.out

    def bound_to(self, lib):
        """The same call through another build of the library (the measurement build)."""
        other = PreparedCall.__new__(PreparedCall)
        other.__dict__.update(self.__dict__)
        other._fn = getattr(lib, self._fn.__name__)
        return other


def prepare(fn_name, geom, q, k_cache, v_cache, block_table, seq_lens, cu_seqlens_q=None, *,
            max_q_len=1, max_kv_len, sinks=None, k_scale=None, v_scale=None, out=None, lse=None,
            workspace=None, sum_kv_len=0, k_new=None, v_new=None, seq_lens_host=None,
            cu_seqlens_q_host=None, block_table_host=None):
    """Build a PreparedCall for "eid_attn_decode" / "eid_attn_varlen" / "eid_lse_merge".
    `seq_lens_host` / `cu_seqlens_q_host` (host copies of the two length arrays) are copied
    and kept by the object."""
    k_cache = _cache_view(k_cache, geom, "k_cache")
    v_cache = _cache_view(v_cache, geom, "v_cache")
    _require(q, "q", torch.bfloat16, 3)
    _require(block_table, "block_table", torch.int32, 2)
    _require(seq_lens, "seq_lens", torch.int32, 1)
    desc = make_desc(geom, num_seqs=seq_lens.shape[0], num_q_tokens=q.shape[0],
                     max_q_len=max_q_len, max_kv_len=max_kv_len,
                     max_blocks_per_seq=block_table.shape[1], num_blocks=k_cache.shape[0],
                     sum_kv_len=sum_kv_len)
    need = load_library().eid_workspace_bytes(C.byref(desc))
    if need == 0:
        check(getattr(load_library(), fn_name)(C.byref(desc), C.byref(AttnArgs()), None))
    if out is None:
        out = torch.empty_like(q)
    own_ws = fn_name == "eid_attn_decode_noalloc"   # the library's static array serves it
    if workspace is None and not own_ws:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    args = AttnArgs()
    args.q, args.out = q.data_ptr(), out.data_ptr()
    args.lse = lse.data_ptr() if lse is not None else None
    args.k_cache, args.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
    args.block_table, args.seq_lens = block_table.data_ptr(), seq_lens.data_ptr()
    args.cu_seqlens_q = cu_seqlens_q.data_ptr() if cu_seqlens_q is not None else None
    args.sinks = sinks.data_ptr() if sinks is not None else None
    args.k_scale = k_scale.data_ptr() if k_scale is not None else None
    args.v_scale = v_scale.data_ptr() if v_scale is not None else None
    if not own_ws:
        args.workspace = workspace.data_ptr()
        args.workspace_bytes = workspace.numel()
    args.k_new = k_new.data_ptr() if k_new is not None else None
    args.v_new = v_new.data_ptr() if v_new is not None else None
    S = seq_lens.shape[0]
    sl_h = _host_i32(seq_lens_host, "seq_lens_host", S)
    cu_h = _host_i32(cu_seqlens_q_host, "cu_seqlens_q_host", S + 1)
    sl_h = sl_h.copy() if sl_h is not None else None
    cu_h = cu_h.copy() if cu_h is not None else None
    args.seq_lens_host = sl_h.ctypes.data if sl_h is not None else None
    args.cu_seqlens_q_host = cu_h.ctypes.data if cu_h is not None else None
    bt_h = _host_bt(block_table_host, block_table)
    bt_h = bt_h.copy() if bt_h is not None else None
    args.block_table_host = bt_h.ctypes.data if bt_h is not None else None
    keep = (q, k_cache, v_cache, block_table, seq_lens, cu_seqlens_q, sinks, k_scale, v_scale,
            k_new, v_new, sl_h, cu_h, bt_h,
            workspace)  # workspace stays last: callers share it via _keep[-1]
    return PreparedCall(fn_name, desc, args, keep, out, lse)


def attn_decode(geom, q, k_cache, v_cache, block_table, seq_lens, *, max_kv_len, sinks=None,
                k_scale=None, v_scale=None, out=None, lse=None, workspace=None,
                return_lse=False, sum_kv_len=0, k_new=None, v_new=None, seq_lens_host=None,
                block_table_host=None):
    """Stages K2+K4: one query row per sequence (q is [num_seqs, Hq, D]).  `sum_kv_len` is the
    optional host-side sum of seq_lens (any upper bound): it sizes the launch to the work;
    `seq_lens_host`, a host copy of seq_lens, lets the library plan the launch exactly.
    With `k_new` / `v_new` ([num_seqs, Hkv, D] bf16: the newest token of every sequence, not
    yet in the cache) the call writes those rows into the caches itself (stage K1 fused)."""
    return _attn_call("eid_attn_decode", geom, q, k_cache, v_cache, block_table, seq_lens, None,
                      1, max_kv_len, sinks, k_scale, v_scale, out, lse, workspace, return_lse,
                      sum_kv_len, k_new, v_new, seq_lens_host, None, block_table_host)


def attn_decode_noalloc(geom, q, k_cache, v_cache, block_table, seq_lens, *, max_kv_len, out,
                        sinks=None, k_scale=None, v_scale=None, lse=None, sum_kv_len=0,
                        k_new=None, v_new=None, seq_lens_host=None, block_table_host=None):
    """attn_decode through the entry point that allocates nothing: the split-KV partials go
    to the library's static device array (batches whose workspace would exceed
    STATIC_WORKSPACE_BYTES raise EID_ERR_WORKSPACE), and `out` must be given.  Calls on one
    GPU share that array and must not overlap in time."""
    if out is None:
        raise ValueError("out must be given: this call allocates nothing")
    return _attn_call("eid_attn_decode_noalloc", geom, q, k_cache, v_cache, block_table,
                      seq_lens, None, 1, max_kv_len, sinks, k_scale, v_scale, out, lse, None,
                      False, sum_kv_len, k_new, v_new, seq_lens_host, None, block_table_host)


def attn_varlen(geom, q, k_cache, v_cache, block_table, seq_lens, cu_seqlens_q, *, max_q_len,
                max_kv_len, sinks=None, k_scale=None, v_scale=None, out=None, lse=None,
                workspace=None, return_lse=False, sum_kv_len=0, seq_lens_host=None,
                cu_seqlens_q_host=None):
    """Stages K2/K3+K4 on a ragged cu_seqlens batch (prefill chunks, verify rows, decodes).
    With host copies of both length arrays the library plans the launches exactly."""
    return _attn_call("eid_attn_varlen", geom, q, k_cache, v_cache, block_table, seq_lens,
                      cu_seqlens_q, max_q_len, max_kv_len, sinks, k_scale, v_scale, out, lse,
                      workspace, return_lse, sum_kv_len, None, None, seq_lens_host,
                      cu_seqlens_q_host)


def lse_merge(geom, workspace, seq_lens, cu_seqlens_q, *, num_q_tokens, max_q_len, max_kv_len,
              max_blocks_per_seq, num_blocks, sinks=None, out=None, lse=None):
    """Stage K4 alone over partials already present in `workspace` (see workspace_layout)."""
    S = seq_lens.shape[0]
    desc = make_desc(geom, num_seqs=S, num_q_tokens=num_q_tokens, max_q_len=max_q_len,
                     max_kv_len=max_kv_len, max_blocks_per_seq=max_blocks_per_seq,
                     num_blocks=num_blocks)
    if out is None:
        out = torch.zeros((num_q_tokens, geom.num_q_heads, geom.head_dim), dtype=torch.bfloat16,
                          device=workspace.device)
    args = AttnArgs()
    args.out = out.data_ptr()
    args.lse = lse.data_ptr() if lse is not None else None
    args.cu_seqlens_q = cu_seqlens_q.data_ptr() if cu_seqlens_q is not None else None
    args.seq_lens = seq_lens.data_ptr()
    args.sinks = sinks.data_ptr() if sinks is not None else None
    args.workspace = workspace.data_ptr()
    args.workspace_bytes = workspace.numel() * workspace.element_size()
    check(load_library().eid_lse_merge(C.byref(desc), C.byref(args), _stream()))
    return out


# The operators below check their tensors in one expression each (a Python check of its own for every
# property of every tensor would cost more than the kernels of a small batch); what fails there is looked
# at property by property to name it.

def _fits(t, dtype, device, shape):
    return t.dtype is dtype and t.get_device() == device and t.shape == shape and t.is_contiguous()


def _need(t, name, dtype, device, shape):
    """Raises unless `t` is a contiguous tensor of that type and shape on that GPU."""
    if t is not None and _fits(t, dtype, device, shape):
        return
    _require(t, name, dtype, len(shape))
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, not on GPU {device}")
    raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")


def _device_of(t, name):
    """Index of the GPU that holds `t`: every other tensor of the call has to be there."""
    if t is None or not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor")
    return t.get_device()


def _cache_shape(t, geom, name):
    """(type, shape) that the caches of a call must have, from the first of them."""
    if t is None or t.dim() != 4 or t.shape[1:] != (geom.block_size, geom.num_kv_heads, geom.head_dim):
        _cache_view(t, geom, name)
    dtype = torch.float8_e4m3fn if geom.kv_dtype == KV_FP8_E4M3 and t.dtype == torch.float8_e4m3fn \
        else _kv_torch_dtype(geom.kv_dtype)
    return dtype, t.shape


def _launch(device, call):
    """call(stream) on the device's current stream, with the device made current."""
    # (the handle itself: a torch.cuda.Stream object around it costs 1 us, a tenth of a small call)
    stream = torch._C._cuda_getCurrentRawStream(device)
    if torch.cuda.current_device() == device:
        check(call(stream))
    else:
        with torch.cuda.device(device):
            check(call(stream))


def _workspace(t, need, device):
    """The caller's workspace, checked, or one from the allocator; None where none is needed."""
    if t is None:
        return torch.empty(need, dtype=torch.uint8, device=f"cuda:{device}") if need else None
    if t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"workspace must be a contiguous tensor on GPU {device}")
    return t


def _rows_desc(geom, S, max_blocks, num_blocks, max_kv_len=1):
    """Descriptor for the operators over cached rows."""
    return make_desc(geom, num_seqs=S, num_q_tokens=max(S, 1), max_q_len=1, max_kv_len=max_kv_len,
                     max_blocks_per_seq=max_blocks, num_blocks=num_blocks)


def attn_tree_workspace_bytes(desc):
    return load_library().eid_attn_tree_workspace_bytes(C.byref(desc))


def attn_tree(geom, q, k_cache, v_cache, block_table, seq_lens, cu_seqlens_q, tree_mask, *, max_q_len,
              max_kv_len, sinks=None, k_scale=None, v_scale=None, out=None, lse=None, workspace=None,
              return_lse=False, sum_kv_len=0):
    """Attention for trees of drafted tokens: row i of a sequence sees its context and the tokens
    whose bits are set in tree_mask[i] ([T, words] int64, bit j % 64 of word j / 64 = token j of
    the same sequence, at most 256 tokens).  The tokens' K/V rows stand in the cache behind the
    context (seq_lens counts them).  geom.window is measured in depths.  `workspace`: a uint8
    tensor of attn_tree_workspace_bytes, for callers that keep one (one call at a time)."""
    dev = _device_of(q, "q")
    kv, cache_shape = _cache_shape(k_cache, geom, "k_cache")
    if seq_lens is None or block_table is None or block_table.dim() != 2 or tree_mask is None or tree_mask.dim() != 2:
        raise ValueError("seq_lens must be [S], block_table [S, max_blocks], tree_mask [T, words]")
    T, S, f32, i32 = q.shape[0], seq_lens.shape[0], torch.float32, torch.int32
    blocks, words = block_table.shape[1], tree_mask.shape[1]
    Hq, Hkv = geom.num_q_heads, geom.num_kv_heads
    q_shape = (T, Hq, geom.head_dim)
    _need(q, "q", torch.bfloat16, dev, q_shape)
    _need(k_cache, "k_cache", kv, dev, cache_shape)
    _need(v_cache, "v_cache", kv, dev, cache_shape)
    _need(block_table, "block_table", i32, dev, (S, blocks))
    _need(seq_lens, "seq_lens", i32, dev, (S,))
    _need(cu_seqlens_q, "cu_seqlens_q", i32, dev, (S + 1,))
    _need(tree_mask, "tree_mask", torch.int64, dev, (T, words))
    if sinks is not None:
        _need(sinks, "sinks", f32, dev, (Hq,))
    fp8 = geom.kv_dtype == KV_FP8_E4M3
    if fp8:
        _need(k_scale, "k_scale", f32, dev, (Hkv,))
        _need(v_scale, "v_scale", f32, dev, (Hkv,))
    if out is None:
        out = torch.empty_like(q)
    else:
        _need(out, "out", torch.bfloat16, dev, q_shape)
    if lse is not None:
        _need(lse, "lse", f32, dev, (T, Hq))
    elif return_lse:
        lse = torch.empty((T, Hq), dtype=f32, device=q.device)
    desc = make_desc(geom, num_seqs=S, num_q_tokens=T, max_q_len=max_q_len, max_kv_len=max_kv_len,
                     max_blocks_per_seq=blocks, num_blocks=cache_shape[0], sum_kv_len=sum_kv_len)
    lib, ref = load_library(), C.byref(desc)
    workspace = _workspace(workspace, lib.eid_attn_tree_workspace_bytes(ref), dev)
    args = AttnArgs(q=q.data_ptr(), out=out.data_ptr(), k_cache=k_cache.data_ptr(), v_cache=v_cache.data_ptr(),
                    block_table=block_table.data_ptr(), cu_seqlens_q=cu_seqlens_q.data_ptr(),
                    seq_lens=seq_lens.data_ptr())
    if lse is not None:
        args.lse = lse.data_ptr()
    if sinks is not None:
        args.sinks = sinks.data_ptr()
    if fp8:
        args.k_scale, args.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
    if workspace is not None:
        args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.nbytes
    _launch(dev, lambda stream: lib.eid_attn_tree(ref, C.byref(args), tree_mask.data_ptr(), words, stream))
    return (out, lse) if return_lse else out


def kv_score(geom, q, lse, k_cache, block_table, seq_lens, cu_seqlens_q, scores, *, max_q_len, max_kv_len,
             k_scale=None, sum_kv_len=0, workspace=None):
    """Adds the attention weight that every cached key receives from this step's rows to `scores`
    ([num_blocks, num_kv_heads, 16] fp32, paged like the caches; the step's own keys start from 0).
    `lse` is what the step's attention call returned (rows in a line: there is no form for a tree's).
    Returns `scores`.  `workspace`: a uint8 tensor of kv_score_workspace_bytes, for callers that keep one
    (one call at a time)."""
    dev = _device_of(q, "q")
    kv, cache_shape = _cache_shape(k_cache, geom, "k_cache")
    if seq_lens is None or block_table is None or block_table.dim() != 2:
        raise ValueError("seq_lens must be [S], block_table [S, max_blocks]")
    T, S, f32, i32 = q.shape[0], seq_lens.shape[0], torch.float32, torch.int32
    blocks = block_table.shape[1]
    _need(q, "q", torch.bfloat16, dev, (T, geom.num_q_heads, geom.head_dim))
    _need(lse, "lse", f32, dev, (T, geom.num_q_heads))
    _need(k_cache, "k_cache", kv, dev, cache_shape)
    _need(block_table, "block_table", i32, dev, (S, blocks))
    _need(seq_lens, "seq_lens", i32, dev, (S,))
    _need(cu_seqlens_q, "cu_seqlens_q", i32, dev, (S + 1,))
    _need(scores, "scores", f32, dev, (cache_shape[0], geom.num_kv_heads, geom.block_size))
    scale = None
    if geom.kv_dtype == KV_FP8_E4M3:
        _need(k_scale, "k_scale", f32, dev, (geom.num_kv_heads,))
        scale = k_scale.data_ptr()
    desc = make_desc(geom, num_seqs=S, num_q_tokens=T, max_q_len=max_q_len, max_kv_len=max_kv_len,
                     max_blocks_per_seq=blocks, num_blocks=cache_shape[0], sum_kv_len=sum_kv_len)
    lib, ref = load_library(), C.byref(desc)
    workspace = _workspace(workspace, lib.eid_kv_score_workspace_bytes(ref), dev)
    ws, n = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.nbytes)
    _launch(dev, lambda stream: lib.eid_kv_score(
        ref, q.data_ptr(), lse.data_ptr(), k_cache.data_ptr(), block_table.data_ptr(), cu_seqlens_q.data_ptr(),
        seq_lens.data_ptr(), scale, scores.data_ptr(), ws, n, stream))
    return scores


def kv_score_workspace_bytes(desc):
    """Bytes of workspace kv_score needs (0: none)."""
    return load_library().eid_kv_score_workspace_bytes(C.byref(desc))


def kv_select(geom, scores, block_table, seq_lens, *, budget, keep_first=0, keep_last=0, max_kv_len, keep=None,
              counts=None):
    """The rows of every sequence that stay when its cache is cut to `budget` rows, per KV head: the
    first keep_first, the last keep_last and the highest scores between them (ties: the lower
    row).  Returns (keep [S, num_kv_heads, budget] int32, ascending, -1 behind the count; counts
    [S] int32)."""
    dev = _device_of(scores, "scores")
    if seq_lens is None or block_table is None or block_table.dim() != 2 or scores.dim() != 3:
        raise ValueError("seq_lens must be [S], block_table [S, max_blocks], scores [num_blocks, num_kv_heads, 16]")
    S, f32, i32 = seq_lens.shape[0], torch.float32, torch.int32
    blocks, num_blocks = block_table.shape[1], scores.shape[0]
    if max_kv_len > blocks * geom.block_size:
        raise ValueError(f"block_table cannot hold max_kv_len {max_kv_len}")
    if budget <= 0:
        raise ValueError("budget must be positive")
    _need(scores, "scores", f32, dev, (num_blocks, geom.num_kv_heads, geom.block_size))
    _need(block_table, "block_table", i32, dev, (S, blocks))
    _need(seq_lens, "seq_lens", i32, dev, (S,))
    if keep is None:
        keep = torch.empty((S, geom.num_kv_heads, budget), dtype=i32, device=scores.device)
    else:
        _need(keep, "keep", i32, dev, (S, geom.num_kv_heads, budget))
    if counts is None:
        counts = torch.empty((S,), dtype=i32, device=scores.device)
    else:
        _need(counts, "counts", i32, dev, (S,))
    desc = _rows_desc(geom, S, blocks, num_blocks, max_kv_len)
    lib = load_library()
    _launch(dev, lambda stream: lib.eid_kv_select(
        C.byref(desc), scores.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), budget, keep_first, keep_last,
        keep.data_ptr(), counts.data_ptr(), stream))
    return keep, counts


def _layers(tensors, name, dtype, device, shape):
    """Addresses of one tensor per layer, all of them of that type and shape."""
    T = torch.Tensor
    if not (set(map(T.get_device, tensors)) == {device} and all([t.shape == shape for t in tensors])
            and all([t.dtype is dtype for t in tensors]) and all(map(T.is_contiguous, tensors))):
        for i, t in enumerate(tensors):
            _need(t, f"{name}[{i}]", dtype, device, shape)
    return list(map(T.data_ptr, tensors))


def kv_compact(geom, k_caches, v_caches, block_table, seq_lens, keep, counts, *, starts=None, scores=None):
    """Moves row keep[..., i] of every sequence to row starts[s] + i (i < counts[s]), in place, in the
    caches of all layers (lists of [num_blocks, 16, Hkv, D] tensors) and in their `scores`
    (list, optional).  keep is int32 and ascending, keep[..., i] >= starts[s] + i: [S, N] (the same
    rows in every layer and head), [S, Hkv, N] (in every layer) or [layers, S, Hkv, N]; seq_lens is
    the length before the move.  The sequence's length afterwards is starts[s] + counts[s]; Scheduler.truncate,
    called first, refuses sequences that share the pages."""
    n = len(k_caches)
    if n == 0 or len(v_caches) != n or (scores is not None and len(scores) != n):
        raise ValueError("k_caches, v_caches (and scores) must be lists with one tensor per layer")
    dev = _device_of(keep, "keep")
    kv, cache_shape = _cache_shape(k_caches[0], geom, "k_caches[0]")
    if seq_lens is None or block_table is None or block_table.dim() != 2 or not 2 <= keep.dim() <= 4:
        raise ValueError("keep must be [S, N], [S, num_kv_heads, N] or [layers, S, num_kv_heads, N]; seq_lens [S]; "
                         "block_table [S, max_blocks]")
    S, i32, H = seq_lens.shape[0], torch.int32, geom.num_kv_heads
    blocks, N, dims = block_table.shape[1], keep.shape[-1], keep.dim()
    at = _layers(k_caches, "k_caches", kv, dev, cache_shape) + _layers(v_caches, "v_caches", kv, dev, cache_shape)
    if scores is not None:
        at += _layers(scores, "scores", torch.float32, dev, (cache_shape[0], H, geom.block_size))
    if len(set(at)) != len(at):
        raise ValueError("a tensor is given twice")
    _need(block_table, "block_table", i32, dev, (S, blocks))
    _need(seq_lens, "seq_lens", i32, dev, (S,))
    _need(counts, "counts", i32, dev, (S,))
    _need(keep, "keep", i32, dev, (S, N) if dims == 2 else (S, H, N) if dims == 3 else (n, S, H, N))
    first = None
    if starts is not None:
        _need(starts, "starts", i32, dev, (S,))
        first = starts.data_ptr()
    desc = _rows_desc(geom, S, blocks, cache_shape[0])
    host = array("q", at)   # (a ctypes array of 72 takes 4 us more to fill)
    base = host.buffer_info()[0]
    lib = load_library()
    _launch(dev, lambda stream: lib.eid_kv_compact(
        C.byref(desc), n, base, base + 8 * n, base + 16 * n if scores is not None else None, block_table.data_ptr(),
        seq_lens.data_ptr(), keep.data_ptr(), S * H * N if dims == 4 else 0, N if dims == 2 else H * N,
        0 if dims == 2 else N, N, counts.data_ptr(), first, stream))


def workspace_layout(desc):
    """(partition, nparts_max, ws_rows, ml_offset, acc_offset): after a 256-byte plan header
    (and, when a sequence can have more than one partition, one int32 per sequence: its number
    of pieces) the split-KV workspace holds
    ml  float32 [num_seqs*ws_rows, nparts_max, Hq, 2]  (m in natural-log units, l) and
    o   float16 [num_seqs*ws_rows, nparts_max, Hq, 64] (partition output sum e^(s-m) v / l) at
    the byte offsets returned."""
    P = partition_size(desc)
    if (16 < desc.max_q_len <= 32 and desc.num_kv_heads % 8 == 0
            and desc.num_seqs * desc.num_kv_heads <= 64):
        qmax = 32
    elif (8 < desc.max_q_len <= 16 and desc.num_kv_heads % 8 == 0
            and desc.num_seqs * desc.num_kv_heads <= 448):
        qmax = 16   # rows of a split-KV sequence (see short_q_max in eid_api.cpp)
    else:
        qmax = 8 if 6 < desc.max_q_len <= 8 else 6
    if desc.window > 0:
        span = min(desc.max_kv_len, desc.window + qmax + desc.block_size - 1)
    else:
        span = desc.max_kv_len
    nparts = (span + P - 1) // P
    head = 256
    if nparts > 1:
        # (see make_plan in eid_api.cpp) the per-sequence piece counts of an even split sit behind
        # the plan header; with a run-time partition the ranges are cut anywhere in a sequence:
        # one more piece than whole partitions
        if desc.partition_size == 0 and P == 256:
            nparts += 1
        head += (desc.num_seqs * 4 + 255) // 256 * 256
    ws_rows = min(desc.max_q_len, qmax)
    cells = desc.num_seqs * ws_rows * desc.num_q_heads * nparts
    ml_bytes = (cells * 8 + 255) // 256 * 256
    return P, nparts, ws_rows, head, head + ml_bytes
