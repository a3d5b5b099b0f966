"""Operators for a batch of requests that continue one prompt, over torch CUDA tensors.

Mirrors dfl_qk_norm_rope, dfl_prefix_attention and dfl_verify_drafts (include/dflash_b200.h): shapes, dtypes and strides are
read off the tensors, outputs and workspaces come from torch's allocator on the call's stream, nothing waits for the GPU.
torch is imported with the first call only; the rest of the package does not need it.
"""
import contextlib
import ctypes as C
import struct

F32, F16, BF16 = 0, 1, 30
MAX_ROPE_AXES = 3


class QkNormRopeArgs(C.Structure):
    _fields_ = [("src_dtype", C.c_int32), ("dst_dtype", C.c_int32), ("n_tokens", C.c_uint32), ("n_q_heads", C.c_uint32), ("n_kv_heads", C.c_uint32),
                ("head_dim", C.c_uint32), ("rotary_dim", C.c_uint32), ("n_axes", C.c_uint32), ("sections", C.c_uint32 * MAX_ROPE_AXES),
                ("interleaved", C.c_int32), ("theta", C.c_double), ("eps", C.c_float), ("_pad", C.c_uint32), ("q", C.c_void_p), ("k", C.c_void_p),
                ("v", C.c_void_p)] + [(n, C.c_int64) for n in ("q_token_stride", "q_head_stride", "k_token_stride", "k_head_stride", "v_token_stride",
                                                               "v_head_stride")] + \
               [("q_weight", C.c_void_p), ("k_weight", C.c_void_p), ("positions", C.c_void_p), ("position_axis_stride", C.c_int64), ("kv_rows", C.c_void_p),
                ("n_kv_out_rows", C.c_uint64), ("q_out", C.c_void_p), ("k_out", C.c_void_p), ("v_out", C.c_void_p)] + \
               [(n, C.c_int64) for n in ("q_out_token_stride", "q_out_head_stride", "k_out_row_stride", "k_out_head_stride", "v_out_row_stride",
                                         "v_out_head_stride")]


class PrefixAttentionArgs(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("batch", C.c_uint32), ("n_tokens", C.c_uint32), ("n_q_heads", C.c_uint32), ("n_kv_heads", C.c_uint32),
                ("head_dim", C.c_uint32), ("scale", C.c_float), ("_pad", C.c_uint32), ("prefix_len", C.c_uint64), ("own_capacity", C.c_uint64),
                ("q", C.c_void_p), ("q_batch_stride", C.c_int64), ("q_token_stride", C.c_int64), ("q_head_stride", C.c_int64),
                ("prefix_k", C.c_void_p), ("prefix_v", C.c_void_p), ("prefix_k_row_stride", C.c_int64), ("prefix_k_head_stride", C.c_int64),
                ("prefix_v_row_stride", C.c_int64), ("prefix_v_head_stride", C.c_int64), ("own_k", C.c_void_p), ("own_v", C.c_void_p),
                ("own_k_batch_stride", C.c_int64), ("own_k_row_stride", C.c_int64), ("own_k_head_stride", C.c_int64),
                ("own_v_batch_stride", C.c_int64), ("own_v_row_stride", C.c_int64), ("own_v_head_stride", C.c_int64),
                ("own_len", C.c_void_p), ("q_len", C.c_void_p), ("out", C.c_void_p), ("out_batch_stride", C.c_int64),
                ("out_token_stride", C.c_int64), ("out_head_stride", C.c_int64), ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64)]


class VerifyDraftsArgs(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("batch", C.c_uint32), ("n_drafts", C.c_uint32), ("_pad", C.c_uint32), ("vocab", C.c_uint64), ("logits", C.c_void_p),
                ("logits_batch_stride", C.c_int64), ("logits_row_stride", C.c_int64), ("draft_probs", C.c_void_p), ("probs_batch_stride", C.c_int64),
                ("probs_row_stride", C.c_int64)] + \
               [(n, C.c_void_p) for n in ("drafts", "n_draft", "temperature", "u_accept", "u_sample", "n_accepted_out", "tokens_out", "workspace")] + \
               [("workspace_bytes", C.c_uint64)]


def _packer(cls):
    """struct.Struct of a C structure's fields in their order: filling one this way takes a tenth of the time of ctypes' attributes."""
    code = {C.c_int32: "i", C.c_uint32: "I", C.c_int64: "q", C.c_uint64: "Q", C.c_double: "d", C.c_float: "f", C.c_void_p: "P"}
    fmt = "@" + "".join(code[f] if f in code else code[f._type_] * f._length_ for _, f in cls._fields_)
    s = struct.Struct(fmt)
    assert s.size == C.sizeof(cls), cls
    return s


_ROPE, _ATTN, _VERIFY = _packer(QkNormRopeArgs), _packer(PrefixAttentionArgs), _packer(VerifyDraftsArgs)
_FNS = None


def _fns():
    """The library's entry points with their argument types, and torch."""
    global _FNS
    if _FNS is None:
        import torch
        from . import check, lib
        L = lib()
        for name in ("qk_norm_rope", "prefix_attention", "verify_drafts"):
            f = getattr(L, "dfl_" + name)
            f.argtypes, f.restype = [C.c_int32, C.c_char_p, C.c_void_p], C.c_int32
        for name in ("prefix_attention_workspace", "verify_drafts_workspace"):
            f = getattr(L, "dfl_" + name)
            f.argtypes, f.restype = [C.c_int32, C.c_char_p, C.POINTER(C.c_uint64)], C.c_int32
        dtypes = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
        _FNS = (L, torch, check, dtypes)
    return _FNS


def _dtype(dtypes, x, name):
    d = dtypes.get(x.dtype)
    if d is None:
        raise TypeError(f"{name}: dtype {x.dtype} is not float32, float16 or bfloat16")
    return d


def _need(x, name, shape, like, dtype=None):
    """x has this shape (None: any extent) and dtype, lies on like's device, with a contiguous last dimension."""
    if x.shape != shape and (x.dim() != len(shape) or any(want is not None and got != want for got, want in zip(x.shape, shape))):
        raise ValueError(f"{name}: shape {tuple(x.shape)}, expected {tuple('any' if s is None else s for s in shape)}")
    if x.device != like.device or not x.is_cuda:
        raise ValueError(f"{name}: on {x.device}, expected {like.device} (a CUDA device)" if like.is_cuda else f"{name}: on {x.device}, expected a CUDA device")
    if dtype is not None and x.dtype != dtype:
        raise TypeError(f"{name}: dtype {x.dtype}, expected {dtype}")
    if shape and shape[-1] != 1 and x.stride(-1) != 1 and x.shape[-1] > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return x


def _dense(x, name, shape, like, dtype):
    _need(x, name, shape, like, dtype)
    if not x.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    return x.data_ptr()


def _output(x, name, shape, like, dtype=None):
    _need(x, name, shape, like, dtype)
    if any(s == 0 and n > 1 for s, n in zip(x.stride(), x.shape)):
        raise ValueError(f"{name}: an expanded dimension cannot be written")
    return x


def _no_grad(torch, *tensors):
    """The operators have no backward pass: a result that autograd would take for a constant is refused."""
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in tensors):
        raise RuntimeError("no backward pass: call it under torch.no_grad() or on detached tensors")


@contextlib.contextmanager
def _elsewhere(torch, x, stream):
    with torch.cuda.device(x.device):
        s = torch.cuda.current_stream(x.device) if stream is None else stream
        if s.device != x.device:
            raise ValueError(f"stream on {s.device}, tensors on {x.device}")
        with torch.cuda.stream(s):
            yield s.cuda_stream


def _on(torch, x, stream):
    """The call's device and stream as torch's current ones (what is allocated inside belongs to that stream), and the stream's handle."""
    if stream is None and torch.cuda.current_device() == x.device.index:
        return contextlib.nullcontext(torch.cuda.current_stream(x.device).cuda_stream)
    return _elsewhere(torch, x, stream)


def qk_norm_rope(q, k, positions, *, theta, rotary_dim=None, sections=None, interleaved=False, q_weight=None, k_weight=None, eps=1e-6,
                 q_out=None, k_out=None, k_rows=None, v=None, v_out=None, stream=None):
    """Per-head RMS norm of q [T, Hq, D] and k [T, Hkv, D], rotation by `positions` (int32 [T], or [axes, T] with `sections` frequencies to
    an axis), and the store of the K (and V) rows: at row t, or at k_rows[t] (int64) of k_out / v_out [rows, Hkv, D], rows outside of which
    are dropped.  Weights are f32 [D].  Outputs that are not given are new tensors of q's dtype.  Returns (q_out, k_out) or, with v, (q_out,
    k_out, v_out)."""
    L, torch, check, dtypes = _fns()
    if q.dim() != 3:
        raise ValueError(f"q: shape {tuple(q.shape)}, expected [tokens, heads, dim]")
    T, hq, D = q.shape
    _need(q, "q", (T, hq, D), q)
    hk = k.shape[1] if k.dim() == 3 else 0
    _need(k, "k", (T, hk, D), q, q.dtype)
    if positions.dim() == 1:
        positions = positions[None]
    axes = positions.shape[0]
    _need(positions, "positions", (axes, T), q, torch.int32)
    if not 1 <= axes <= MAX_ROPE_AXES:
        raise ValueError("positions: one to three axes")
    rotary_dim = D if rotary_dim is None else rotary_dim
    sections = [rotary_dim // 2] if sections is None and axes == 1 else sections
    if sections is None or len(sections) != axes:
        raise ValueError("sections: one number of frequencies for each axis")
    wq = 0 if q_weight is None else _dense(q_weight, "q_weight", (D,), q, torch.float32)
    wk = 0 if k_weight is None else _dense(k_weight, "k_weight", (D,), q, torch.float32)
    rows = 0
    if k_rows is not None:
        rows = _dense(k_rows, "k_rows", (T,), q, torch.int64)
        if k_out is None or (v is not None and v_out is None):
            raise ValueError("k_rows: needs k_out (and v_out)")
    if v is not None:
        _need(v, "v", (T, hk, D), q, q.dtype)
    _no_grad(torch, q, k, v, q_weight, k_weight)
    with _on(torch, q, stream) as handle:
        q_out = torch.empty((T, hq, D), dtype=q.dtype, device=q.device) if q_out is None else _output(q_out, "q_out", (T, hq, D), q)
        k_out = torch.empty((T, hk, D), dtype=q_out.dtype, device=q.device) if k_out is None else _output(k_out, "k_out", (None, hk, D), q, q_out.dtype)
        v_in, v_s, vo, vo_s = 0, (0, 0), 0, (0, 0)
        if v is not None:
            v_out = torch.empty((T, hk, D), dtype=q_out.dtype, device=q.device) if v_out is None else _output(v_out, "v_out", (k_out.shape[0], hk, D), q, q_out.dtype)
            v_in, v_s, vo, vo_s = v.data_ptr(), v.stride(), v_out.data_ptr(), v_out.stride()
        q_s, k_s, qo_s, ko_s = q.stride(), k.stride(), q_out.stride(), k_out.stride()
        a = _ROPE.pack(_dtype(dtypes, q, "q"), _dtype(dtypes, q_out, "q_out"), T, hq, hk, D, rotary_dim, axes, *sections, *(0,) * (MAX_ROPE_AXES - axes),
                       1 if interleaved else 0, theta, eps, 0, q.data_ptr(), k.data_ptr(), v_in, q_s[0], q_s[1], k_s[0], k_s[1], v_s[0], v_s[1], wq, wk,
                       positions.data_ptr(), positions.stride(0), rows, k_out.shape[0], q_out.data_ptr(), k_out.data_ptr(), vo,
                       qo_s[0], qo_s[1], ko_s[0], ko_s[1], vo_s[0], vo_s[1])
        check(L.dfl_qk_norm_rope(q.device.index, a, handle))
    return (q_out, k_out) if v is None else (q_out, k_out, v_out)


def prefix_attention(q, prefix_k, prefix_v, own_k=None, own_v=None, own_len=None, *, q_len=None, scale=None, out=None, stream=None):
    """Attention of a batch over one shared prefix and each request's own rows: q [B, n, Hq, D], prefix_k / prefix_v [P, Hkv, D], own_k / own_v
    [B, cap, Hkv, D] of which own_len[b] (int32) are in use, the block's own rows the last of them.  q_len (int32 [B]): how many of a request's n
    queries exist (all when None); output rows behind them are left as they were (zero in a new tensor).  scale: 1 / sqrt(D) when None."""
    L, torch, check, dtypes = _fns()
    if q.dim() != 4:
        raise ValueError(f"q: shape {tuple(q.shape)}, expected [batch, tokens, heads, dim]")
    B, n, hq, D = q.shape
    _need(q, "q", (B, n, hq, D), q)
    _need(prefix_k, "prefix_k", (None, None, D), q, q.dtype)
    P, hk = prefix_k.shape[:2]
    _need(prefix_v, "prefix_v", (P, hk, D), q, q.dtype)
    cap, ok, ok_s, ov, ov_s, lens = 0, 0, (0, 0, 0), 0, (0, 0, 0), 0
    if own_k is not None:
        if own_v is None or own_len is None:
            raise ValueError("own_k: needs own_v and own_len")
        _need(own_k, "own_k", (B, None, hk, D), q, q.dtype)
        cap = own_k.shape[1]
        _need(own_v, "own_v", (B, cap, hk, D), q, q.dtype)
        lens = _dense(own_len, "own_len", (B,), q, torch.int32)
        ok, ok_s, ov, ov_s = own_k.data_ptr(), own_k.stride(), own_v.data_ptr(), own_v.stride()
    q_lens = 0 if q_len is None else _dense(q_len, "q_len", (B,), q, torch.int32)
    _no_grad(torch, q, prefix_k, prefix_v, own_k, own_v)
    with _on(torch, q, stream) as handle:
        if out is None:
            out = (torch.empty if q_len is None else torch.zeros)((B, n, hq, D), dtype=q.dtype, device=q.device)
        _output(out, "out", (B, n, hq, D), q, q.dtype)
        q_s, pk_s, pv_s, o_s = q.stride(), prefix_k.stride(), prefix_v.stride(), out.stride()
        fields = (_dtype(dtypes, q, "q"), B, n, hq, hk, D, D ** -0.5 if scale is None else scale, 0, P, cap, q.data_ptr(), q_s[0], q_s[1], q_s[2],
                  prefix_k.data_ptr(), prefix_v.data_ptr(), pk_s[0], pk_s[1], pv_s[0], pv_s[1], ok, ov, ok_s[0], ok_s[1], ok_s[2], ov_s[0], ov_s[1], ov_s[2],
                  lens, q_lens, out.data_ptr(), o_s[0], o_s[1], o_s[2])
        dev, need = q.device.index, C.c_uint64()
        check(L.dfl_prefix_attention_workspace(dev, _ATTN.pack(*fields, 0, 0), need))
        work = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
        check(L.dfl_prefix_attention(dev, _ATTN.pack(*fields, work.data_ptr() if need.value else 0, need.value), handle))
    return out


def verify_drafts(logits, drafts, u_accept, u_sample, *, draft_probs=None, n_draft=None, temperature=None, stream=None):
    """How many of each request's drafts (int32 [B, K]) stand against the target's logits [B, K + 1, V], and the token behind them: returns
    (n_accepted int32 [B], tokens int32 [B, K + 1], -1 behind the drawn token).  u_accept [B, K] and u_sample [B] are f32 in [0, 1).
    draft_probs f32 [B, K, V]: the distributions the drafts were drawn from (None: each draft had all the mass); n_draft int32 [B]: drafts that
    exist; temperature f32 [B]: 0 is greedy.  n_accepted[b] = -1 - row where that row is no distribution."""
    L, torch, check, dtypes = _fns()
    if logits.dim() != 3:
        raise ValueError(f"logits: shape {tuple(logits.shape)}, expected [batch, drafts + 1, vocab]")
    B, R, V = logits.shape
    K = R - 1
    if K < 0:
        raise ValueError("logits: one row at least")
    _need(logits, "logits", (B, R, V), logits)
    d = _dense(drafts, "drafts", (B, K), logits, torch.int32)
    ua = _dense(u_accept, "u_accept", (B, K), logits, torch.float32)
    us = _dense(u_sample, "u_sample", (B,), logits, torch.float32)
    probs, p_s = 0, (0, 0)
    if draft_probs is not None:
        _need(draft_probs, "draft_probs", (B, K, V), logits, torch.float32)
        probs, p_s = draft_probs.data_ptr(), draft_probs.stride()
    nd = 0 if n_draft is None else _dense(n_draft, "n_draft", (B,), logits, torch.int32)
    temp = 0 if temperature is None else _dense(temperature, "temperature", (B,), logits, torch.float32)
    _no_grad(torch, logits, draft_probs)
    with _on(torch, logits, stream) as handle:
        n_accepted = torch.empty(B, dtype=torch.int32, device=logits.device)
        tokens = torch.empty((B, R), dtype=torch.int32, device=logits.device)
        fields = (_dtype(dtypes, logits, "logits"), B, K, 0, V, logits.data_ptr(), logits.stride(0), logits.stride(1), probs, p_s[0], p_s[1], d, nd, temp, ua, us,
                  n_accepted.data_ptr(), tokens.data_ptr())
        dev, need = logits.device.index, C.c_uint64()
        check(L.dfl_verify_drafts_workspace(dev, _VERIFY.pack(*fields, 0, 0), need))
        work = torch.empty(need.value, dtype=torch.uint8, device=logits.device) if need.value else None
        check(L.dfl_verify_drafts(dev, _VERIFY.pack(*fields, work.data_ptr() if need.value else 0, need.value), handle))
    return n_accepted, tokens
