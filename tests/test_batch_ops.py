"""Operators for a batch over one prompt, without a GPU: the ctypes mirror against the header, and what the entry points refuse.

Refusals are decided on the host before anything is enqueued; the addresses here are never followed."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest

from dflb import ROOT, pkg
import importlib

ops = importlib.import_module("qwen-llm_b200.batch_ops")
HEADER = os.path.join(ROOT, "include", "dflash_b200.h")
STRUCTS = {"dfl_qk_norm_rope_args": ops.QkNormRopeArgs, "dfl_prefix_attention_args": ops.PrefixAttentionArgs, "dfl_verify_drafts_args": ops.VerifyDraftsArgs}
PTR = 0x10000000   # 16-byte aligned, never read


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_mirror_has_the_header_s_layout(name, tmp_path):
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("no C compiler")
    fields = [f[0] for f in STRUCTS[name]._fields_]
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"%s\"\nint main(void) {\n" % HEADER
    src += "".join('    printf("%%zu\\n", offsetof(%s, %s));\n' % (name, f) for f in fields) + '    printf("%%zu\\n", sizeof(%s));\n    return 0;\n}\n' % name
    (tmp_path / "a.c").write_text(src)
    subprocess.check_call([gcc, "-o", str(tmp_path / "a"), str(tmp_path / "a.c")])
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "a")]).split()]
    assert got == [getattr(STRUCTS[name], f).offset for f in fields] + [C.sizeof(STRUCTS[name])]
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), open(HEADER).read(), re.S).group(1)
    assert set(re.findall(r"(\w+)(?:\[\w+\])?(?=[,;])", re.sub(r"/\*.*?\*/", "", body, flags=re.S))) == set(fields)


def rope_args(**kw):
    a = ops.QkNormRopeArgs(src_dtype=ops.F32, dst_dtype=ops.F16, n_tokens=3, n_q_heads=4, n_kv_heads=2, head_dim=64, rotary_dim=32, n_axes=1, theta=1e4, eps=1e-6,
                           q=PTR, k=PTR, v=PTR, positions=PTR, q_out=PTR, k_out=PTR, v_out=PTR, n_kv_out_rows=3, q_token_stride=256, q_head_stride=64)
    a.sections[0] = 16
    for k, v in kw.items():
        if k == "sections":
            for i, n in enumerate(v):
                a.sections[i] = n
        else:
            setattr(a, k, v)
    return a


def attn_args(**kw):
    a = ops.PrefixAttentionArgs(dtype=ops.F16, batch=2, n_tokens=3, n_q_heads=4, n_kv_heads=2, head_dim=64, scale=0.125, prefix_len=10, own_capacity=8, q=PTR, prefix_k=PTR,
                                prefix_v=PTR, own_k=PTR, own_v=PTR, own_len=PTR, out=PTR, workspace=PTR, workspace_bytes=1 << 40)
    for f, _ in ops.PrefixAttentionArgs._fields_:
        if f.endswith("_stride"):
            setattr(a, f, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def verify_args(**kw):
    a = ops.VerifyDraftsArgs(dtype=ops.F32, batch=2, n_drafts=3, vocab=100, logits=PTR, logits_batch_stride=400, logits_row_stride=100, drafts=PTR, u_accept=PTR,
                             u_sample=PTR, n_accepted_out=PTR, tokens_out=PTR, workspace=PTR, workspace_bytes=1 << 40)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


REFUSED = [
    (rope_args, "dfl_qk_norm_rope", dict(src_dtype=12), "UNSUPPORTED"),
    (rope_args, "dfl_qk_norm_rope", dict(dst_dtype=8), "UNSUPPORTED"),
    (rope_args, "dfl_qk_norm_rope", dict(head_dim=1), "BAD_SHAPE"),
    (rope_args, "dfl_qk_norm_rope", dict(head_dim=513), "BAD_SHAPE"),
    (rope_args, "dfl_qk_norm_rope", dict(rotary_dim=33), "BAD_SHAPE"),
    (rope_args, "dfl_qk_norm_rope", dict(rotary_dim=66), "BAD_SHAPE"),
    (rope_args, "dfl_qk_norm_rope", dict(sections=[15]), "BAD_SHAPE"),
    (rope_args, "dfl_qk_norm_rope", dict(n_axes=0), "BAD_ARG"),
    (rope_args, "dfl_qk_norm_rope", dict(n_axes=4), "BAD_ARG"),
    (rope_args, "dfl_qk_norm_rope", dict(n_axes=2, sections=[4, 12], interleaved=1), "BAD_SHAPE"),   # frequency 23 of 16
    (rope_args, "dfl_qk_norm_rope", dict(theta=0.5), "BAD_ARG"),
    (rope_args, "dfl_qk_norm_rope", dict(theta=float("nan")), "BAD_ARG"),
    (rope_args, "dfl_qk_norm_rope", dict(eps=-1.0), "BAD_ARG"),
    (rope_args, "dfl_qk_norm_rope", dict(q=None), "BAD_ARG"),
    (rope_args, "dfl_qk_norm_rope", dict(k_out=None), "BAD_ARG"),
    (rope_args, "dfl_qk_norm_rope", dict(v_out=None), "BAD_ARG"),
    (rope_args, "dfl_qk_norm_rope", dict(positions=None), "BAD_ARG"),
    (rope_args, "dfl_qk_norm_rope", dict(n_kv_out_rows=2), "BAD_SHAPE"),
    (rope_args, "dfl_qk_norm_rope", dict(q_token_stride=-1), "BAD_SHAPE"),
    (attn_args, "dfl_prefix_attention", dict(dtype=ops.F32), "UNSUPPORTED"),
    (attn_args, "dfl_prefix_attention", dict(head_dim=80), "UNSUPPORTED"),
    (attn_args, "dfl_prefix_attention", dict(n_q_heads=5), "BAD_SHAPE"),
    (attn_args, "dfl_prefix_attention", dict(n_q_heads=130), "BAD_SHAPE"),
    (attn_args, "dfl_prefix_attention", dict(n_kv_heads=0), "BAD_SHAPE"),
    (attn_args, "dfl_prefix_attention", dict(scale=0.0), "BAD_ARG"),
    (attn_args, "dfl_prefix_attention", dict(scale=float("inf")), "BAD_ARG"),
    (attn_args, "dfl_prefix_attention", dict(prefix_len=1 << 30), "BAD_SHAPE"),
    (attn_args, "dfl_prefix_attention", dict(q_token_stride=12), "BAD_SHAPE"),
    (attn_args, "dfl_prefix_attention", dict(own_v_row_stride=-64), "BAD_SHAPE"),
    (attn_args, "dfl_prefix_attention", dict(prefix_v=PTR + 8), "BAD_ARG"),
    (attn_args, "dfl_prefix_attention", dict(own_len=None), "BAD_ARG"),
    (attn_args, "dfl_prefix_attention", dict(prefix_k=None), "BAD_ARG"),
    (attn_args, "dfl_prefix_attention", dict(out=None), "BAD_ARG"),
    (attn_args, "dfl_prefix_attention", dict(batch=1 << 30), "BAD_SHAPE"),
    (verify_args, "dfl_verify_drafts", dict(dtype=12), "UNSUPPORTED"),
    (verify_args, "dfl_verify_drafts", dict(vocab=0), "BAD_SHAPE"),
    (verify_args, "dfl_verify_drafts", dict(vocab=1 << 31), "BAD_SHAPE"),
    (verify_args, "dfl_verify_drafts", dict(n_drafts=256), "BAD_SHAPE"),
    (verify_args, "dfl_verify_drafts", dict(drafts=None), "BAD_ARG"),
    (verify_args, "dfl_verify_drafts", dict(u_accept=None), "BAD_ARG"),
    (verify_args, "dfl_verify_drafts", dict(tokens_out=None), "BAD_ARG"),
    (verify_args, "dfl_verify_drafts", dict(logits_row_stride=-1), "BAD_SHAPE"),
    (verify_args, "dfl_verify_drafts", dict(workspace=PTR + 16), "BAD_ARG"),
    (verify_args, "dfl_verify_drafts", dict(workspace_bytes=8), "BAD_SHAPE"),
]


def entry_point(name):
    f = C.CFUNCTYPE(C.c_int32, C.c_int32, C.c_void_p, C.c_void_p)
    return f((name, pkg.lib()))


@pytest.mark.parametrize("make,entry,change,status", REFUSED, ids=["%s-%s" % (e[4:], "-".join(c)) for _, e, c, _ in REFUSED])
def test_refused_before_anything_runs(make, entry, change, status):
    with pytest.raises(pkg.DflError) as e:
        pkg.check(entry_point(entry)(0, C.byref(make(**change)), None))
    assert e.value.name == status and entry[4:] in str(e.value)


@pytest.mark.parametrize("make,entry", [(rope_args, "dfl_qk_norm_rope"), (attn_args, "dfl_prefix_attention"), (verify_args, "dfl_verify_drafts")])
def test_null_arguments_and_no_device(make, entry):
    with pytest.raises(pkg.DflError) as e:
        pkg.check(entry_point(entry)(0, None, None))
    assert e.value.name == "BAD_ARG"
    if pkg.device_count() == 0:
        with pytest.raises(pkg.DflError) as e:
            pkg.check(entry_point(entry)(0, C.byref(make()), None))
        assert e.value.name == "NO_DEVICE"


def test_wrappers_refuse_what_they_can_see():
    torch = pytest.importorskip("torch")
    q = torch.zeros(2, 4, 64)
    with pytest.raises(ValueError, match="q: on cpu, expected a CUDA device"):
        pkg.qk_norm_rope(q, q, torch.zeros(2, dtype=torch.int32), theta=1e4)
    with pytest.raises(ValueError, match="q: shape"):
        pkg.prefix_attention(q, q, q)
    with pytest.raises(ValueError, match="logits: shape"):
        pkg.verify_drafts(q[0], None, None, None)


# addresses that their type does not allow, and K or V rows that lie one upon another
MORE_REFUSED = [
    (rope_args, "dfl_qk_norm_rope", dict(q=PTR + 2), "BAD_ARG"),
    (rope_args, "dfl_qk_norm_rope", dict(k_out=PTR + 1), "BAD_ARG"),
    (rope_args, "dfl_qk_norm_rope", dict(q_weight=PTR + 2), "BAD_ARG"),
    (rope_args, "dfl_qk_norm_rope", dict(positions=PTR + 2), "BAD_ARG"),
    (rope_args, "dfl_qk_norm_rope", dict(kv_rows=PTR + 4), "BAD_ARG"),
    (attn_args, "dfl_prefix_attention", dict(own_len=PTR + 2), "BAD_ARG"),
    (attn_args, "dfl_prefix_attention", dict(q_len=PTR + 1), "BAD_ARG"),
    (attn_args, "dfl_prefix_attention", dict(own_k_batch_stride=0), "BAD_SHAPE"),
    (attn_args, "dfl_prefix_attention", dict(prefix_v_head_stride=0), "BAD_SHAPE"),
    (attn_args, "dfl_prefix_attention", dict(prefix_k_row_stride=0), "BAD_SHAPE"),
    (attn_args, "dfl_prefix_attention", dict(out_token_stride=0), "BAD_SHAPE"),
    (verify_args, "dfl_verify_drafts", dict(logits=PTR + 2), "BAD_ARG"),
    (verify_args, "dfl_verify_drafts", dict(draft_probs=PTR + 2), "BAD_ARG"),
    (verify_args, "dfl_verify_drafts", dict(tokens_out=PTR + 2), "BAD_ARG"),
    (verify_args, "dfl_verify_drafts", dict(workspace=None), "BAD_ARG"),
]


@pytest.mark.parametrize("make,entry,change,status", MORE_REFUSED, ids=["%s-%s" % (e[4:], "-".join(c)) for _, e, c, _ in MORE_REFUSED])
def test_refused_addresses_and_strides(make, entry, change, status):
    test_refused_before_anything_runs(make, entry, change, status)


def test_verify_workspace_has_room_for_its_counters_whatever_the_machine():
    # whether rows are counted depends on how many SMs there are; the size, asked for without a device, does not
    f = C.CFUNCTYPE(C.c_int32, C.c_int32, C.c_void_p, C.c_void_p)(("dfl_verify_drafts_workspace", pkg.lib()))
    for batch, drafts, vocab in ((1, 0, 1000), (1, 1, 10), (3, 15, 151936), (30, 7, 32000), (128, 7, 151936), (500, 0, 151936)):
        need = C.c_uint64()
        pkg.check(f(0, C.byref(verify_args(batch=batch, n_drafts=drafts, vocab=vocab)), C.byref(need)))
        rows, pieces = batch * (drafts + 1), -(-vocab // 8192)
        assert need.value == -(-rows * pieces * 16 // 256) * 256 + (4 * (rows + batch) if drafts else 0)
