"""Operators for a batch of requests that continue one prompt, over torch CUDA tensors.

Mirrors dfl_qk_norm_rope, dfl_prefix_attention and dfl_verify_drafts (include/dflash_b200.h): shapes, dtypes and strides are
read off the tensors, outputs and workspaces come from torch's allocator on the call's stream, nothing waits for the GPU.  With `stream` the work goes to
that stream: it has to be ordered behind what the inputs come from, and whoever reads the outputs behind it, as with torch.cuda.stream().
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
_WORK = struct.Struct("@PQ")   # the last two fields of the structures with a workspace
_FNS = None


def _fns():
    """The library's entry points with their argument types, torch, the status check, dtype codes, the handle of a device's current stream, and autograd's notice."""
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
        # the handle without a Stream object around it, where torch has that: 0.1 us instead of 2.3
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda dev: torch.cuda.current_stream(dev).cuda_stream)
        # says to autograd that a caller's tensors have changed, so that a graph that saved one of them does not take it for what it was
        written = getattr(torch._C, "_increment_version", None) or torch.autograd.graph.increment_version
        _FNS = (L, torch, check, dtypes, raw, written)
    return _FNS


def _dtype(dtypes, x, name):
    d = dtypes.get(x.dtype)
    if d is None:
        raise TypeError(f"{name}: dtype {x.dtype} is not float32, float16 or bfloat16")
    return d


def _device(x, name, dims, what):
    """The device number of the tensor that the others are measured by."""
    if x.dim() != dims:
        raise ValueError(f"{name}: shape {tuple(x.shape)}, expected {what}")
    if not x.is_cuda:
        raise ValueError(f"{name}: on {x.device}, expected a CUDA device")
    return x.get_device()


def _extents(x, name, dims, what):
    if x.dim() != dims:
        raise ValueError(f"{name}: shape {tuple(x.shape)}, expected {what}")
    return x.shape


# Calls of a few microseconds on the device are bounded by the checks here, so a tensor is asked for each of its properties once and looked at closely
# only when it is out of line: norm and rotation of one token take the host 13 us a call, 10 of them here.
def _take(x, name, shape, dtype, dev):
    """(address, strides) of a tensor that has this shape and dtype, lies on device number `dev` and is contiguous in its last dimension."""
    s = x.stride()
    if x.shape != shape or x.dtype is not dtype or x.get_device() != dev or s[-1] != 1:
        if x.shape != shape:
            raise ValueError(f"{name}: shape {tuple(x.shape)}, expected {tuple(shape)}")
        if x.get_device() != dev:
            raise ValueError(f"{name}: on {x.device}, expected cuda:{dev}")
        if x.dtype is not dtype:
            raise TypeError(f"{name}: dtype {x.dtype}, expected {dtype}")
        if x.shape[-1] > 1:
            raise ValueError(f"{name}: the last dimension must be contiguous")
    return x.data_ptr(), s


def _take_out(x, name, shape, dtype, dev):
    p, s = _take(x, name, shape, dtype, dev)
    if 0 in s and any(i == 0 and n > 1 for i, n in zip(s, x.shape)):
        raise ValueError(f"{name}: an expanded dimension cannot be written")
    return p, s


def _dense(x, name, shape, dtype, dev):
    p, _ = _take(x, name, shape, dtype, dev)
    if not x.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    return p


def _no_grad(torch, *tensors):
    """The operators have no derivatives: a result that autograd would take for a constant is refused, and an output that it tracks."""
    if torch.is_grad_enabled():
        for x in tensors:
            if x is not None and x.requires_grad:
                raise RuntimeError("no backward pass: call it under torch.no_grad() or on detached tensors")
    fw = torch.autograd.forward_ad
    if fw._current_level >= 0:   # inside a dual_level(); no_grad() does not reach that
        for x in tensors:
            if x is not None and fw.unpack_dual(x).tangent is not None:
                raise RuntimeError("no forward-mode derivative: a tensor has a tangent")


@contextlib.contextmanager
def _current(torch, dev, stream, tensors):
    """The device, and the stream where one is given, as torch's current ones: what is allocated inside belongs to that stream, and the memory of the
    tensors that the call was given goes to no other one before the stream has passed the call."""
    with torch.cuda.device(dev):
        if stream is not None and stream.device.index != dev:
            raise ValueError(f"stream on {stream.device}, tensors on cuda:{dev}")
        with torch.cuda.stream(stream):
            yield
        if stream is not None:
            for x in tensors:
                if x is not None:
                    x.record_stream(stream)


def qk_norm_rope(q, k, positions, *, theta, rotary_dim=None, sections=None, interleaved=False, q_weight=None, k_weight=None, eps=1e-6,
                 q_out=None, k_out=None, k_rows=None, v=None, v_out=None, stream=None):
    """Per-head RMS norm of q [T, Hq, D] and k [T, Hkv, D], rotation by `positions` (int32 [T], or [axes, T] with `sections` frequencies to
    an axis), and the store of the K (and V) rows: at row t of k_out / v_out, which have as many at least, or at k_rows[t] (int64) of k_out / v_out
    [rows, Hkv, D], rows outside of which are dropped.  Weights are f32 [D].  Outputs that are not given are new tensors of q_out's dtype, and that one of
    q's.  Returns (q_out, k_out) or, with v, (q_out, k_out, v_out)."""
    L, torch, check, dtypes, raw, written = _fns()
    dev = _device(q, "q", 3, "[tokens, heads, dim]")
    if stream is not None or torch.cuda.current_device() != dev:
        with _current(torch, dev, stream, (q, k, positions, q_weight, k_weight, q_out, k_out, k_rows, v, v_out)):
            return qk_norm_rope(q, k, positions, theta=theta, rotary_dim=rotary_dim, sections=sections, interleaved=interleaved, q_weight=q_weight,
                                k_weight=k_weight, eps=eps, q_out=q_out, k_out=k_out, k_rows=k_rows, v=v, v_out=v_out)
    shape, dt, f32 = q.shape, q.dtype, torch.float32
    T, hq, D = shape
    hk = _extents(k, "k", 3, "[tokens, heads, dim]")[1]
    kv_shape = (T, hk, D)
    q_p, q_s = _take(q, "q", shape, dt, dev)
    k_p, k_s = _take(k, "k", kv_shape, dt, dev)
    if positions.dim() == 1:
        axes, axis_stride = 1, 0
        pos_p, _ = _take(positions, "positions", (T,), torch.int32, dev)
    else:
        axes = _extents(positions, "positions", 2, "[tokens] or [axes, tokens]")[0]
        pos_p, pos_s = _take(positions, "positions", (axes, T), torch.int32, dev)
        axis_stride = pos_s[0]
    if not 1 <= axes <= MAX_ROPE_AXES:
        raise ValueError("positions: one to three axes")
    rotary_dim = D if rotary_dim is None else rotary_dim
    sections = [rotary_dim // 2] if sections is None and axes == 1 else sections
    if sections is None or len(sections) != axes:
        raise ValueError("sections: one number of frequencies for each axis")
    wq = 0 if q_weight is None else _take(q_weight, "q_weight", (D,), f32, dev)[0]
    wk = 0 if k_weight is None else _take(k_weight, "k_weight", (D,), f32, dev)[0]
    rows = 0
    if k_rows is not None:
        rows, _ = _take(k_rows, "k_rows", (T,), torch.int64, dev)
        if k_out is None or (v is not None and v_out is None):
            raise ValueError("k_rows: needs k_out (and v_out)")
    _no_grad(torch, q, k, v, q_weight, k_weight, q_out, k_out, v_out)
    if q_out is None:
        q_out = torch.empty(shape, dtype=dt, device=q.device)
    out_dt = q_out.dtype
    qo_p, qo_s = _take_out(q_out, "q_out", shape, out_dt, dev)
    if k_out is None:
        k_out = torch.empty(kv_shape, dtype=out_dt, device=q.device)
    n_rows = _extents(k_out, "k_out", 3, "[rows, heads, dim]")[0]
    ko_p, ko_s = _take_out(k_out, "k_out", (n_rows, hk, D), out_dt, dev)
    v_p, v_s, vo_p, vo_s = 0, (0, 0), 0, (0, 0)
    if v is not None:
        v_p, v_s = _take(v, "v", kv_shape, dt, dev)
        if v_out is None:
            v_out = torch.empty(kv_shape, dtype=out_dt, device=q.device)
        v_rows = n_rows if k_rows is not None else _extents(v_out, "v_out", 3, "[rows, heads, dim]")[0]
        vo_p, vo_s = _take_out(v_out, "v_out", (v_rows, hk, D), out_dt, dev)
        n_rows = min(n_rows, v_rows)
    elif v_out is not None:
        raise ValueError("v_out: without v")
    a = _ROPE.pack(_dtype(dtypes, q, "q"), _dtype(dtypes, q_out, "q_out"), T, hq, hk, D, rotary_dim, axes, *sections, *(0,) * (MAX_ROPE_AXES - axes),
                   1 if interleaved else 0, theta, eps, 0, q_p, k_p, v_p, q_s[0], q_s[1], k_s[0], k_s[1], v_s[0], v_s[1], wq, wk, pos_p, axis_stride, rows,
                   n_rows, qo_p, ko_p, vo_p, qo_s[0], qo_s[1], ko_s[0], ko_s[1], vo_s[0], vo_s[1])
    check(L.dfl_qk_norm_rope(dev, a, raw(dev)))
    outs = (q_out, k_out) if v is None else (q_out, k_out, v_out)
    written(outs)
    return outs


def prefix_attention(q, prefix_k, prefix_v, own_k=None, own_v=None, own_len=None, *, q_len=None, scale=None, out=None, stream=None):
    """Attention of a batch over one shared prefix and each request's own rows: q [B, n, Hq, D], prefix_k / prefix_v [P, Hkv, D], own_k / own_v
    [B, cap, Hkv, D] of which own_len[b] (int32) are in use, the block's own rows the last of them.  q_len (int32 [B]): how many of a request's n
    queries exist (all when None); output rows behind them are left as they were (zero in a new tensor).  scale: 1 / sqrt(D) when None."""
    L, torch, check, dtypes, raw, written = _fns()
    dev = _device(q, "q", 4, "[batch, tokens, heads, dim]")
    if stream is not None or torch.cuda.current_device() != dev:
        with _current(torch, dev, stream, (q, prefix_k, prefix_v, own_k, own_v, own_len, q_len, out)):
            return prefix_attention(q, prefix_k, prefix_v, own_k, own_v, own_len, q_len=q_len, scale=scale, out=out)
    shape, dt = q.shape, q.dtype
    B, n, hq, D = shape
    q_p, q_s = _take(q, "q", shape, dt, dev)
    P, hk, _ = _extents(prefix_k, "prefix_k", 3, "[keys, heads, dim]")
    pk_p, pk_s = _take(prefix_k, "prefix_k", (P, hk, D), dt, dev)
    pv_p, pv_s = _take(prefix_v, "prefix_v", (P, hk, D), dt, dev)
    cap, ok_p, ok_s, ov_p, ov_s, lens = 0, 0, (0, 0, 0), 0, (0, 0, 0), 0
    if own_k is not None:
        if own_v is None or own_len is None:
            raise ValueError("own_k: needs own_v and own_len")
        cap = _extents(own_k, "own_k", 4, "[batch, rows, heads, dim]")[1]
        ok_p, ok_s = _take(own_k, "own_k", (B, cap, hk, D), dt, dev)
        ov_p, ov_s = _take(own_v, "own_v", (B, cap, hk, D), dt, dev)
        lens, _ = _take(own_len, "own_len", (B,), torch.int32, dev)
    elif own_v is not None:   # (own_len alone is clamped to the rows there are: none)
        raise ValueError("own_v: without own_k")
    q_lens = 0 if q_len is None else _take(q_len, "q_len", (B,), torch.int32, dev)[0]
    _no_grad(torch, q, prefix_k, prefix_v, own_k, own_v, out)
    if out is None:
        out = (torch.empty if q_len is None else torch.zeros)(shape, dtype=dt, device=q.device)
    o_p, o_s = _take_out(out, "out", shape, dt, dev)
    a = _ATTN.pack(_dtype(dtypes, q, "q"), B, n, hq, hk, D, D ** -0.5 if scale is None else scale, 0, P, cap, q_p, q_s[0], q_s[1], q_s[2], pk_p, pv_p, pk_s[0], pk_s[1],
                   pv_s[0], pv_s[1], ok_p, ov_p, ok_s[0], ok_s[1], ok_s[2], ov_s[0], ov_s[1], ov_s[2], lens, q_lens, o_p, o_s[0], o_s[1], o_s[2], 0, 0)
    need = C.c_uint64()
    check(L.dfl_prefix_attention_workspace(dev, a, need))
    size = need.value
    if size:
        work = q.new_empty(size // 2)   # of 16-bit elements
        a = a[:-_WORK.size] + _WORK.pack(work.data_ptr(), size)
    check(L.dfl_prefix_attention(dev, a, raw(dev)))
    written((out,))
    return out


def verify_drafts(logits, drafts, u_accept, u_sample, *, draft_probs=None, n_draft=None, temperature=None, stream=None):
    """How many of each request's drafts (int32 [B, K]) stand against the target's logits [B, K + 1, V], and the token behind them: returns
    (n_accepted int32 [B], tokens int32 [B, K + 1], -1 behind the drawn token).  u_accept [B, K] and u_sample [B] are f32 in [0, 1).
    draft_probs f32 [B, K, V]: the distributions the drafts were drawn from (None: each draft had all the mass); n_draft int32 [B]: drafts that
    exist; temperature f32 [B]: 0 is greedy.  n_accepted[b] = -1 - row where that row is no distribution."""
    L, torch, check, dtypes, raw, _ = _fns()
    dev = _device(logits, "logits", 3, "[batch, drafts + 1, vocab]")
    if stream is not None or torch.cuda.current_device() != dev:
        with _current(torch, dev, stream, (logits, drafts, u_accept, u_sample, draft_probs, n_draft, temperature)):
            return verify_drafts(logits, drafts, u_accept, u_sample, draft_probs=draft_probs, n_draft=n_draft, temperature=temperature)
    shape, f32, i32 = logits.shape, torch.float32, torch.int32
    B, R, V = shape
    K = R - 1
    if K < 0:
        raise ValueError("logits: one row at least")
    x_p, x_s = _take(logits, "logits", shape, logits.dtype, dev)
    d = _dense(drafts, "drafts", (B, K), i32, dev)
    ua = _dense(u_accept, "u_accept", (B, K), f32, dev)
    us, _ = _take(u_sample, "u_sample", (B,), f32, dev)
    probs, p_s = (0, (0, 0)) if draft_probs is None else _take(draft_probs, "draft_probs", (B, K, V), f32, dev)
    nd = 0 if n_draft is None else _take(n_draft, "n_draft", (B,), i32, dev)[0]
    temp = 0 if temperature is None else _take(temperature, "temperature", (B,), f32, dev)[0]
    _no_grad(torch, logits, draft_probs)
    n_accepted, tokens = drafts.new_empty(B), drafts.new_empty((B, R))
    a = _VERIFY.pack(_dtype(dtypes, logits, "logits"), B, K, 0, V, x_p, x_s[0], x_s[1], probs, p_s[0], p_s[1], d, nd, temp, ua, us, n_accepted.data_ptr(),
                     tokens.data_ptr(), 0, 0)
    need = C.c_uint64()
    check(L.dfl_verify_drafts_workspace(dev, a, need))
    size = need.value
    if size:
        work = drafts.new_empty(size // 4)   # of 32-bit elements
        a = a[:-_WORK.size] + _WORK.pack(work.data_ptr(), size)
    check(L.dfl_verify_drafts(dev, a, raw(dev)))
    return n_accepted, tokens
