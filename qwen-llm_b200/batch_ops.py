"""Operators for a batch of requests that continue one prompt, over torch CUDA tensors.

Mirrors dfl_qk_norm_rope, dfl_prefix_attention and dfl_verify_drafts (include/dflash_b200.h): shapes, dtypes and strides are
read off the tensors, outputs and workspaces come from torch's allocator on the call's stream, nothing waits for the GPU.
torch is imported with the first call only; the rest of the package does not need it.
"""
import contextlib
import ctypes as C

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


def _lib():
    from . import lib
    return lib()


def _check(status):
    from . import check
    check(status)


def _dtype(x, name):
    d = {"torch.float32": F32, "torch.float16": F16, "torch.bfloat16": BF16}.get(str(x.dtype))
    if d is None:
        raise TypeError(f"{name}: dtype {x.dtype} is not float32, float16 or bfloat16")
    return d


def _need(x, name, shape, like, dtype=None, dense=False):
    """x has this shape (None: any extent) and dtype, lies on like's device, with a contiguous last dimension (dense: altogether)."""
    if x.dim() != len(shape) or any(want is not None and got != want for got, want in zip(x.shape, shape)):
        raise ValueError(f"{name}: shape {tuple(x.shape)}, expected {tuple('any' if s is None else s for s in shape)}")
    if x.device != like.device or not x.is_cuda:
        raise ValueError(f"{name}: on {x.device}, expected {like.device} (a CUDA device)")
    if dtype is not None and x.dtype != dtype:
        raise TypeError(f"{name}: dtype {x.dtype}, expected {dtype}")
    if dense and not x.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    if x.dim() and x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return x


@contextlib.contextmanager
def _on(x, stream):
    """The call's device and stream as torch's current ones (what is allocated inside belongs to that stream), and the stream's handle."""
    import torch
    with torch.cuda.device(x.device):
        s = torch.cuda.current_stream(x.device) if stream is None else stream
        if s.device != x.device:
            raise ValueError(f"stream on {s.device}, tensors on {x.device}")
        with torch.cuda.stream(s):
            yield C.c_void_p(s.cuda_stream)


def _p(x):
    return None if x is None else x.data_ptr()


def qk_norm_rope(q, k, positions, *, theta, rotary_dim=None, sections=None, interleaved=False, q_weight=None, k_weight=None, eps=1e-6,
                 q_out=None, k_out=None, k_rows=None, v=None, v_out=None, stream=None):
    """Per-head RMS norm of q [T, Hq, D] and k [T, Hkv, D], rotation by `positions` (int32 [T], or [axes, T] with `sections` frequencies to
    an axis), and the store of the K (and V) rows: at row t, or at k_rows[t] (int64) of k_out / v_out [rows, Hkv, D], rows outside of which
    are dropped.  Weights are f32 [D].  Outputs that are not given are new tensors of q's dtype.  Returns (q_out, k_out) or, with v, (q_out,
    k_out, v_out)."""
    import torch
    T, hq, D = q.shape if q.dim() == 3 else _need(q, "q", (None, None, None), q)
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
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            _need(w, name, (D,), q, torch.float32, dense=True)
    if k_rows is not None:
        _need(k_rows, "k_rows", (T,), q, torch.int64, dense=True)
        if k_out is None or (v is not None and v_out is None):
            raise ValueError("k_rows: needs k_out (and v_out)")
    if v is not None:
        _need(v, "v", (T, hk, D), q, q.dtype)
    with _on(q, stream) as handle:
        q_out = torch.empty((T, hq, D), dtype=q.dtype, device=q.device) if q_out is None else _need(q_out, "q_out", (T, hq, D), q)
        k_out = torch.empty((T, hk, D), dtype=q_out.dtype, device=q.device) if k_out is None else _need(k_out, "k_out", (None, hk, D), q, q_out.dtype)
        if v is not None:
            v_out = torch.empty((T, hk, D), dtype=q_out.dtype, device=q.device) if v_out is None else _need(v_out, "v_out", (k_out.shape[0], hk, D), q, q_out.dtype)
        a = QkNormRopeArgs(src_dtype=_dtype(q, "q"), dst_dtype=_dtype(q_out, "q_out"), n_tokens=T, n_q_heads=hq, n_kv_heads=hk, head_dim=D, rotary_dim=rotary_dim,
                           n_axes=axes, interleaved=1 if interleaved else 0, theta=theta, eps=eps, q=_p(q), k=_p(k), v=_p(v),
                           q_token_stride=q.stride(0), q_head_stride=q.stride(1), k_token_stride=k.stride(0), k_head_stride=k.stride(1),
                           q_weight=_p(q_weight), k_weight=_p(k_weight), positions=_p(positions), position_axis_stride=positions.stride(0),
                           kv_rows=_p(k_rows), n_kv_out_rows=k_out.shape[0], q_out=_p(q_out), k_out=_p(k_out), v_out=_p(v_out) if v is not None else None,
                           q_out_token_stride=q_out.stride(0), q_out_head_stride=q_out.stride(1), k_out_row_stride=k_out.stride(0), k_out_head_stride=k_out.stride(1))
        for i, n in enumerate(sections):
            a.sections[i] = n
        if v is not None:
            a.v_token_stride, a.v_head_stride, a.v_out_row_stride, a.v_out_head_stride = v.stride(0), v.stride(1), v_out.stride(0), v_out.stride(1)
        _check(_lib().dfl_qk_norm_rope(C.c_int32(q.device.index), C.byref(a), handle))
    return (q_out, k_out) if v is None else (q_out, k_out, v_out)


def prefix_attention(q, prefix_k, prefix_v, own_k=None, own_v=None, own_len=None, *, q_len=None, scale=None, out=None, stream=None):
    """Attention of a batch over one shared prefix and each request's own rows: q [B, n, Hq, D], prefix_k / prefix_v [P, Hkv, D], own_k / own_v
    [B, cap, Hkv, D] of which own_len[b] (int32) are in use, the block's own rows the last of them.  q_len (int32 [B]): how many of a request's n
    queries exist (all when None); output rows behind them are left as they were (zero in a new tensor).  scale: 1 / sqrt(D) when None."""
    import torch
    if q.dim() != 4:
        raise ValueError(f"q: shape {tuple(q.shape)}, expected [batch, tokens, heads, dim]")
    B, n, hq, D = q.shape
    _need(q, "q", (B, n, hq, D), q)
    _need(prefix_k, "prefix_k", (None, None, D), q, q.dtype)
    P, hk = prefix_k.shape[:2]
    _need(prefix_v, "prefix_v", (P, hk, D), q, q.dtype)
    cap = 0
    if own_k is not None:
        if own_v is None or own_len is None:
            raise ValueError("own_k: needs own_v and own_len")
        _need(own_k, "own_k", (B, None, hk, D), q, q.dtype)
        cap = own_k.shape[1]
        _need(own_v, "own_v", (B, cap, hk, D), q, q.dtype)
        _need(own_len, "own_len", (B,), q, torch.int32, dense=True)
    if q_len is not None:
        _need(q_len, "q_len", (B,), q, torch.int32, dense=True)
    with _on(q, stream) as handle:
        if out is None:
            out = (torch.empty if q_len is None else torch.zeros)((B, n, hq, D), dtype=q.dtype, device=q.device)
        _need(out, "out", (B, n, hq, D), q, q.dtype)
        a = PrefixAttentionArgs(dtype=_dtype(q, "q"), batch=B, n_tokens=n, n_q_heads=hq, n_kv_heads=hk, head_dim=D, scale=D ** -0.5 if scale is None else scale,
                                prefix_len=P, own_capacity=cap, q=_p(q), q_batch_stride=q.stride(0), q_token_stride=q.stride(1), q_head_stride=q.stride(2),
                                prefix_k=_p(prefix_k), prefix_v=_p(prefix_v), prefix_k_row_stride=prefix_k.stride(0), prefix_k_head_stride=prefix_k.stride(1),
                                prefix_v_row_stride=prefix_v.stride(0), prefix_v_head_stride=prefix_v.stride(1), q_len=_p(q_len),
                                out=_p(out), out_batch_stride=out.stride(0), out_token_stride=out.stride(1), out_head_stride=out.stride(2))
        if own_k is not None:
            a.own_k, a.own_v, a.own_len = _p(own_k), _p(own_v), _p(own_len)
            a.own_k_batch_stride, a.own_k_row_stride, a.own_k_head_stride = own_k.stride()[:3]
            a.own_v_batch_stride, a.own_v_row_stride, a.own_v_head_stride = own_v.stride()[:3]
        L, dev, need = _lib(), C.c_int32(q.device.index), C.c_uint64()
        _check(L.dfl_prefix_attention_workspace(dev, C.byref(a), C.byref(need)))
        work = torch.empty(need.value, dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = _p(work) if need.value else None, need.value
        _check(L.dfl_prefix_attention(dev, C.byref(a), handle))
    return out


def verify_drafts(logits, drafts, u_accept, u_sample, *, draft_probs=None, n_draft=None, temperature=None, stream=None):
    """How many of each request's drafts (int32 [B, K]) stand against the target's logits [B, K + 1, V], and the token behind them: returns
    (n_accepted int32 [B], tokens int32 [B, K + 1], -1 behind the drawn token).  u_accept [B, K] and u_sample [B] are f32 in [0, 1).
    draft_probs f32 [B, K, V]: the distributions the drafts were drawn from (None: each draft had all the mass); n_draft int32 [B]: drafts that
    exist; temperature f32 [B]: 0 is greedy.  n_accepted[b] = -1 - row where that row is no distribution."""
    import torch
    if logits.dim() != 3:
        raise ValueError(f"logits: shape {tuple(logits.shape)}, expected [batch, drafts + 1, vocab]")
    B, R, V = logits.shape
    K = R - 1
    if K < 0:
        raise ValueError("logits: one row at least")
    _need(logits, "logits", (B, R, V), logits)
    _need(drafts, "drafts", (B, K), logits, torch.int32, dense=True)
    _need(u_accept, "u_accept", (B, K), logits, torch.float32, dense=True)
    _need(u_sample, "u_sample", (B,), logits, torch.float32, dense=True)
    if draft_probs is not None:
        _need(draft_probs, "draft_probs", (B, K, V), logits, torch.float32)
    if n_draft is not None:
        _need(n_draft, "n_draft", (B,), logits, torch.int32, dense=True)
    if temperature is not None:
        _need(temperature, "temperature", (B,), logits, torch.float32, dense=True)
    with _on(logits, stream) as handle:
        n_accepted = torch.empty(B, dtype=torch.int32, device=logits.device)
        tokens = torch.empty((B, R), dtype=torch.int32, device=logits.device)
        a = VerifyDraftsArgs(dtype=_dtype(logits, "logits"), batch=B, n_drafts=K, vocab=V, logits=_p(logits), logits_batch_stride=logits.stride(0),
                             logits_row_stride=logits.stride(1), drafts=_p(drafts), n_draft=_p(n_draft), temperature=_p(temperature),
                             u_accept=_p(u_accept), u_sample=_p(u_sample), n_accepted_out=_p(n_accepted), tokens_out=_p(tokens))
        if draft_probs is not None:
            a.draft_probs, a.probs_batch_stride, a.probs_row_stride = _p(draft_probs), draft_probs.stride(0), draft_probs.stride(1)
        L, dev, need = _lib(), C.c_int32(logits.device.index), C.c_uint64()
        _check(L.dfl_verify_drafts_workspace(dev, C.byref(a), C.byref(need)))
        work = torch.empty(need.value, dtype=torch.uint8, device=logits.device)
        a.workspace, a.workspace_bytes = _p(work) if need.value else None, need.value
        _check(L.dfl_verify_drafts(dev, C.byref(a), handle))
    return n_accepted, tokens
