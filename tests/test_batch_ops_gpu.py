"""Operators for a batch over one prompt against their definitions in 64 bits."""
import math

import pytest

from dflb import pkg

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- norm, rotation, store ------------------------------------------------------------------------------------------
def axis_of(half, axes, sections, interleaved):
    if not interleaved:
        return [a for a in range(axes) for _ in range(sections[a])]
    return [j % axes if j < axes * sections[j % axes] else 0 for j in range(half)]


def rope_ref(x, w, pos, theta, rot, sections, interleaved, eps=1e-6):
    """(result, |y_j| + |y_partner|) in 64 bits"""
    x = x.double()
    half = rot // 2
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    y = y if w is None else y * w.double()
    size = y.abs()
    if half:
        ax = torch.tensor(axis_of(half, pos.shape[0], sections, interleaved), device=x.device)
        freq = torch.tensor([theta ** (-j / half) for j in range(half)], dtype=torch.float64, device=x.device)
        ang = (pos[ax].t().double() * freq)[:, None]
        a, b = y[..., :half], y[..., half:rot]
        size = torch.cat([a.abs() + b.abs()] * 2 + [size[..., rot:]], -1)
        y = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), y[..., rot:]], -1)
    return y, size


def rope_close(got, want, size, dim):
    # the sum of squares: at most dim / 32 + 5 roundings, halved by the root; root, two products, cos and sin, the two-term sum: 16 more.  The
    # reference's own angle: 2^31 radians in 64 bits are off by 2^-22 (freq within 2^-53 of itself, twice).
    tol = size * ((dim / 64 + 20) * 2.0 ** -24 + 2.0 ** -21) + want.abs() * torch.finfo(got.dtype).eps / 2 + 2.0 ** -25
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), ((got.double() - want).abs() / tol).max()


ROPE = [
    # tokens, q heads, kv heads, dim, rot, axes, interleaved, src, dst
    (1, 32, 8, 128, 32, 1, False, "bf16", "bf16"),
    (1, 1, 1, 64, 64, 1, False, "f32", "f32"),
    (5, 16, 2, 256, 64, 1, True, "f32", "f16"),
    (17, 4, 4, 128, 128, 3, True, "f16", "f16"),
    (33, 6, 3, 64, 64, 3, False, "bf16", "f32"),
    (700, 8, 2, 256, 256, 2, True, "bf16", "f16"),
    (3, 5, 1, 80, 80, 2, False, "f16", "bf16"),
    (4, 3, 1, 96, 10, 1, False, "f32", "bf16"),
    (2, 2, 2, 2, 2, 1, False, "f32", "f32"),
    (2, 2, 1, 7, 6, 1, False, "f16", "f16"),
    (9, 2, 1, 512, 300, 3, True, "bf16", "bf16"),
    (6, 2, 2, 128, 0, 1, False, "f16", "f16"),
    (3000, 3, 1, 128, 64, 1, False, "bf16", "bf16"),
]


def rope_case(tokens, hq, hk, dim, rot, axes, interleaved, src, seed=0):
    g = rng(seed + tokens * 7 + dim)
    heads = torch.randn(tokens, hq + 2 * hk, dim, device="cuda", generator=g).mul_(torch.rand(tokens, 1, 1, device="cuda", generator=g) * 30 + 0.01).to(DT[src])
    pos = torch.randint(-2 ** 31, 2 ** 31 - 1, (axes, tokens), device="cuda", generator=g).to(torch.int32)
    if tokens > 2:
        pos[:, 1:] //= 20000
        heads[1] = 0     # a row of zeros stays one
    half = rot // 2
    rest = min(half // 3, max(0, (half - 1) // axes)) if axes > 1 else 0
    sections = [half - rest * (axes - 1)] + [rest] * (axes - 1)
    w = [torch.rand(dim, device="cuda", generator=g) + 0.5 for _ in "qk"]
    return heads[:, :hq], heads[:, hq:hq + hk], heads[:, hq + hk:], pos, sections, w


@pytest.mark.parametrize("case", ROPE, ids=str)
def test_rope_against_the_definition(case):
    tokens, hq, hk, dim, rot, axes, interleaved, src, dst = case
    q, k, v, pos, sections, (wq, wk) = rope_case(*case[:-1])
    rows = torch.randperm(tokens + 5, device="cuda", generator=rng(1))[:tokens] if tokens > 1 else torch.tensor([3], device="cuda")
    if tokens > 4:
        rows[2], rows[3] = -1, tokens + 5    # two tokens without a place
    k_out = torch.full((tokens + 5, hk, dim), 7.0, device="cuda", dtype=DT[dst])
    v_out = k_out.clone()
    q_out = torch.empty(tokens, hq, dim, device="cuda", dtype=DT[dst])
    got = pkg.qk_norm_rope(q, k, pos, theta=1e6, rotary_dim=rot, sections=sections, interleaved=interleaved, q_weight=wq, k_weight=wk, q_out=q_out, k_out=k_out, k_rows=rows,
                           v=v, v_out=v_out)
    want, size = rope_ref(q, wq, pos, 1e6, rot, sections, interleaved)
    rope_close(got[0], want, size, dim)
    kept = (rows >= 0) & (rows < tokens + 5)
    want, size = rope_ref(k, wk, pos, 1e6, rot, sections, interleaved)
    rope_close(k_out[rows[kept]], want[kept], size[kept], dim)
    assert torch.equal(v_out[rows[kept]], v[kept].to(DT[dst]))
    free = torch.ones(tokens + 5, dtype=torch.bool, device="cuda")
    free[rows[kept]] = False
    assert (k_out[free] == 7).all() and (v_out[free] == 7).all()


def test_rope_without_weights_rows_or_v_and_in_place():
    q, k, _, pos, sections, _ = rope_case(40, 4, 2, 128, 64, 1, False, "bf16")
    a = pkg.qk_norm_rope(q, k, pos[0], theta=1e4, rotary_dim=64)
    for got, x in zip(a, (q, k)):
        want, size = rope_ref(x, None, pos, 1e4, 64, sections, False)
        rope_close(got, want, size, 128)
    q2, k2 = q.clone(), k.clone()
    b = pkg.qk_norm_rope(q2, k2, pos[0], theta=1e4, rotary_dim=64, q_out=q2, k_out=k2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_rope_strides_and_alignment_change_no_bits():
    q, k, v, pos, sections, (wq, wk) = rope_case(50, 4, 2, 128, 128, 1, False, "bf16")
    a = pkg.qk_norm_rope(q, k, pos, theta=1e4, sections=sections, q_weight=wq, k_weight=wk, v=v)
    # an odd start, odd strides and transposed heads
    def odd(x):
        buf = torch.zeros(x.shape[1], x.shape[0], 131, device="cuda", dtype=x.dtype)
        view = buf[..., 1:129].transpose(0, 1)
        view.copy_(x)
        return view
    out = [odd(torch.zeros_like(x)) for x in (q, k, v)]
    b = pkg.qk_norm_rope(odd(q), odd(k), pos, theta=1e4, sections=sections, q_weight=wq, k_weight=wk, v=odd(v), q_out=out[0], k_out=out[1], v_out=out[2])
    for x, y, like in zip(a, b, (q, k, v)):
        if like is v:
            assert torch.equal(x, y)
        else:   # the sums of another kernel: a last place of f32 ahead of the rounding
            assert (x.float() - y.float()).abs().le(x.float().abs() * 2.0 ** -7 + 1e-6).all()


def test_rope_of_nothing_and_of_no_heads():
    e = torch.empty(0, 4, 64, device="cuda")
    a = pkg.qk_norm_rope(e, e[:, :2], torch.empty(0, device="cuda", dtype=torch.int32), theta=1e4)
    assert a[0].shape == (0, 4, 64)
    q, k, _, pos, sections, _ = rope_case(5, 4, 2, 64, 64, 1, False, "f16")
    full = pkg.qk_norm_rope(q, k, pos, theta=1e4, sections=sections)
    alone = pkg.qk_norm_rope(q, k[:, :0], pos, theta=1e4, sections=sections)
    assert torch.equal(full[0], alone[0])


# ---- attention ------------------------------------------------------------------------------------------------------
def attn_ref(q, pk, pv, ok, ov, own_len, q_len, scale):
    """(result, bound on the error) in 64 bits, requests and heads one by one"""
    B, n, hq, D = q.shape
    hk, P = pk.shape[1], pk.shape[0]
    G = hq // hk
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    eps = torch.finfo(q.dtype).eps / 2
    for b in range(B):
        own = 0 if ok is None else min(max(int(own_len[b]), 0), ok.shape[1])
        rows = n if q_len is None else min(max(int(q_len[b]), 0), n)
        for h in range(hk):
            K, V = pk[:, h].double(), pv[:, h].double()
            if own:
                K, V = torch.cat([K, ok[b, :own, h].double()]), torch.cat([V, ov[b, :own, h].double()])
            Q = q[b, :rows, h * G:(h + 1) * G].double()
            S = torch.einsum("igd,kd->igk", Q, K) * scale
            last = P + (own - rows + torch.arange(rows, device=q.device)).clamp(min=-1)    # the prefix is seen by all
            seen = (torch.arange(P + own, device=q.device) <= last[:, None])[:, None]
            S = S.masked_fill(~seen, -math.inf)
            top = S.amax(-1, keepdim=True) if P + own else torch.zeros(rows, G, 1, dtype=torch.float64, device=q.device)
            top = torch.where(top == -math.inf, 0.0, top)
            W = torch.exp(S - top)
            W = torch.where(seen, W, 0.0) if P + own else W
            L = W.sum(-1, keepdim=True)
            o = torch.where(L > 0, torch.einsum("igk,kd->igd", W, V) / L.clamp(min=1e-300), 0.0)
            out[b, :rows, h * G:(h + 1) * G] = o
            if P + own and rows:
                # A score is a sum of D products in at most D / 16 + 4 steps that drop what is below 2^-23 of the largest sum on the way; exp
                # and the scaling add 2^-22 of the score and of the weight; all of it acts on a weight and on the sum of weights.
                reach = (Q.norm(dim=-1).amax() * K.norm(dim=-1).amax() * scale).item()   # no partial sum is larger
                err = 2 * ((D / 16 + 4) * 2.0 ** -23 * reach + 2.0 ** -20)
                A = torch.where(L > 0, torch.einsum("igk,kd->igd", W, V.abs()) / L.clamp(min=1e-300), 0.0)
                # a weight's rounding is half a step of itself, in f16 at least half of the smallest number's step (weights are at least
                # 2^-25 exact beside a largest one of 1 or more)
                low = 2.0 ** -25 * V.abs().sum(0) if q.dtype == torch.float16 else 0.0
                tol[b, :rows, h * G:(h + 1) * G] = A * (eps * 1.01 + err) + low + o.abs() * eps + 2.0 ** -25
    return out, tol


def attn_case(B, n, hq, hk, D, P, cap, dt, layout="rows", seed=0, sharp=1.0):
    g = rng(seed * 1000 + B * 17 + n * 3 + P + cap + D)
    dev = {"device": "cuda", "generator": g}
    q = (torch.randn(B, n, hq, D, **dev) * sharp).to(DT[dt])
    if layout == "rows":
        kv = [torch.randn(P, hk, D, **dev).to(DT[dt]) for _ in "kv"] + [torch.randn(B, cap, hk, D, **dev).to(DT[dt]) for _ in "kv"]
    else:
        kv = [torch.randn(hk, P, D, **dev).to(DT[dt]).transpose(0, 1) for _ in "kv"] + [torch.randn(B, hk, cap, D, **dev).to(DT[dt]).transpose(1, 2) for _ in "kv"]
    return [q] + kv


def attn_check(got, q, pk, pv, ok, ov, own_len, q_len=None, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want, tol = attn_ref(q, pk, pv, ok, ov, own_len, q_len, scale)
    rows = torch.full((q.shape[0],), q.shape[1], device="cuda") if q_len is None else q_len.clamp(0, q.shape[1])
    there = (torch.arange(q.shape[1], device="cuda") < rows[:, None])[..., None, None].expand_as(want)
    off = (got.double() - want).abs()[there] - tol[there]
    assert torch.isfinite(got[there]).all() and (off <= 0).all(), off.max()


ATTN = [
    # batch, n, q heads, kv heads, dim, prefix, capacity, dtype, layout
    (1, 1, 1, 1, 128, 1, 1, "f16", "rows"),
    (1, 1, 4, 1, 128, 0, 1, "bf16", "rows"),
    (2, 1, 8, 2, 64, 127, 130, "bf16", "rows"),
    (3, 1, 8, 2, 128, 128, 128, "f16", "heads"),
    (3, 5, 6, 2, 128, 129, 40, "bf16", "rows"),
    (2, 16, 32, 8, 128, 1000, 300, "f16", "rows"),
    (5, 16, 14, 2, 128, 511, 257, "bf16", "heads"),
    (2, 8, 16, 2, 256, 700, 129, "bf16", "rows"),
    (2, 3, 5, 1, 256, 4097, 64, "f16", "heads"),
    (1, 300, 4, 2, 64, 50, 333, "f16", "rows"),
    (2, 515, 8, 2, 128, 1029, 700, "bf16", "rows"),
    (1, 130, 8, 1, 256, 130, 260, "f16", "rows"),
    (40, 1, 8, 4, 128, 3000, 200, "f16", "rows"),
    (64, 4, 4, 1, 64, 2049, 20, "bf16", "rows"),
    (2, 1, 64, 1, 128, 5000, 9, "bf16", "rows"),
    (1, 1, 8, 8, 128, 20000, 1000, "f16", "rows"),
    (3, 257, 3, 1, 128, 0, 300, "bf16", "rows"),
    (7, 9, 7, 7, 64, 65, 10, "f16", "heads"),
    # several items to a CTA, row blocks with both halves and with one in turn
    (40, 150, 16, 8, 64, 200, 170, "bf16", "rows"),
    (30, 77, 16, 8, 128, 300, 200, "f16", "rows"),
    (50, 20, 32, 4, 256, 257, 150, "bf16", "rows"),
]


@pytest.mark.parametrize("case", ATTN, ids=str)
def test_attention_against_the_definition(case):
    B, n, hq, hk, D, P, cap, dt, layout = case
    q, pk, pv, ok, ov = attn_case(*case[:8], layout=layout)
    g = rng(5)
    own_len = torch.randint(min(n, cap), cap + 1, (B,), device="cuda", generator=g).to(torch.int32)
    attn_check(pkg.prefix_attention(q, pk, pv, ok, ov, own_len), q, pk, pv, ok, ov, own_len)
    # a padded batch, its lengths from nothing to all; what lies behind them may hold anything
    q_len = torch.randint(0, n + 1, (B,), device="cuda", generator=g).to(torch.int32)
    own_len = (q_len + torch.randint(0, cap + 1, (B,), device="cuda", generator=g)).clamp(max=cap).to(torch.int32)
    out = torch.full_like(q, 3.0)
    clean = pkg.prefix_attention(q, pk, pv, ok, ov, own_len, q_len=q_len, out=out)
    assert clean is out
    attn_check(out, q, pk, pv, ok, ov, own_len, q_len)
    gone = torch.arange(n, device="cuda") >= q_len[:, None]
    assert (out[gone] == 3).all()
    behind = torch.arange(cap, device="cuda") >= own_len[:, None]
    q[gone] = math.nan
    ok[behind], ov[behind] = math.nan, math.inf
    again = torch.full_like(q, 3.0)
    pkg.prefix_attention(q, pk, pv, ok, ov, own_len, q_len=q_len, out=again)
    assert torch.equal(out, again)


def test_attention_without_own_rows_and_of_rows_that_see_nothing():
    q, pk, pv, ok, ov = attn_case(3, 4, 8, 2, 128, 300, 16, "bf16")
    attn_check(pkg.prefix_attention(q, pk, pv), q, pk, pv, None, None, None)
    # own rows fewer than queries: the first queries see none of them
    own_len = torch.tensor([0, 2, 16], device="cuda", dtype=torch.int32)
    attn_check(pkg.prefix_attention(q, pk, pv, ok, ov, own_len), q, pk, pv, ok, ov, own_len)
    got = pkg.prefix_attention(q, pk[:0], pv[:0], ok, ov, own_len)
    attn_check(got, q, pk[:0], pv[:0], ok, ov, own_len)
    assert (got[0] == 0).all() and (got[1, :2] == 0).all() and (got[1, 2:] != 0).any()
    assert (pkg.prefix_attention(q, pk[:0], pv[:0]) == 0).all()
    # lengths out of range are taken as the nearest in it
    wild = torch.tensor([-5, 1000, 7], device="cuda", dtype=torch.int32)
    near = torch.tensor([0, 16, 7], device="cuda", dtype=torch.int32)
    assert torch.equal(pkg.prefix_attention(q, pk, pv, ok, ov, wild), pkg.prefix_attention(q, pk, pv, ok, ov, near))
    assert pkg.prefix_attention(q[:0], pk, pv).shape == (0, 4, 8, 128)


@pytest.mark.parametrize("dim,dt", [(64, "f16"), (128, "bf16"), (128, "f16"), (256, "bf16")])
def test_attention_with_scores_that_grow_and_with_far_ones(dim, dt):
    # maxima that rise from tile to tile, by little and by a lot, and fall again; scores of some hundreds
    q, pk, pv, ok, ov = attn_case(2, 3, 4, 1, dim, 1500, 200, dt, seed=3)
    ramp = torch.cat([torch.linspace(0.02, 3, 700), torch.linspace(3, 0.1, 500), torch.full((300,), 2.0)])
    pk = (torch.sign(q[0, 0, 0].float())[None, None] * ramp.cuda()[:, None, None] + 0.05 * pk.float()).to(DT[dt])
    q = (q.float().abs() * torch.sign(q[0, 0, 0].float())).to(DT[dt])
    q[1, 2] = -q[1, 2]
    own_len = torch.tensor([200, 77], device="cuda", dtype=torch.int32)
    for scale in (None, 1.0, 1e-3):
        attn_check(pkg.prefix_attention(q, pk, pv, ok, ov, own_len, scale=scale), q, pk, pv, ok, ov, own_len, scale=scale)


def test_attention_scores_of_minus_infinity():
    q, pk, pv, ok, ov = attn_case(2, 2, 2, 1, 64, 200, 8, "f16")
    q = q.abs() + 0.1
    pk[:150] = -math.inf
    own_len = torch.tensor([8, 4], device="cuda", dtype=torch.int32)
    attn_check(pkg.prefix_attention(q, pk, pv, ok, ov, own_len), q, pk[150:], pv[150:], ok, ov, own_len)
    pk[:] = -math.inf
    assert (pkg.prefix_attention(q, pk, pv) == 0).all()


def test_attention_of_a_request_does_not_depend_on_its_batch():
    q, pk, pv, ok, ov = attn_case(6, 4, 8, 2, 128, 2000, 64, "f16")
    own_len = torch.tensor([4, 64, 10, 33, 5, 20], device="cuda", dtype=torch.int32)
    full = pkg.prefix_attention(q, pk, pv, ok, ov, own_len)
    attn_check(full, q, pk, pv, ok, ov, own_len)
    poisoned = q.clone()
    poisoned[2] = math.nan
    got = pkg.prefix_attention(poisoned, pk, pv, ok, ov, own_len)
    rest = torch.tensor([0, 1, 3, 4, 5], device="cuda")
    assert torch.equal(got[rest], full[rest]) and torch.isnan(got[2]).all()
    assert torch.equal(full, pkg.prefix_attention(q, pk, pv, ok, ov, own_len))    # the same bits every time


def test_attention_strided_tensors_and_a_cache_beyond_32_bits():
    q, pk, pv, ok, ov = attn_case(2, 3, 4, 2, 128, 100, 50, "bf16")
    own_len = torch.tensor([50, 9], device="cuda", dtype=torch.int32)
    want = pkg.prefix_attention(q, pk, pv, ok, ov, own_len)
    wide = torch.zeros(2, 3, 12, 128, device="cuda", dtype=torch.bfloat16)
    wide[:, :, 4:8] = q
    big = torch.zeros(2, 1200000, 2, 1024, device="cuda", dtype=torch.bfloat16)   # 9.8 GB, request 1 from byte 4.9e9 on
    big[:, :50, :, 512:640], big[:, :50, :, 640:768] = ok, ov
    out = torch.zeros(3, 4, 2, 128, device="cuda", dtype=torch.bfloat16).permute(2, 0, 1, 3)
    got = pkg.prefix_attention(wide[:, :, 4:8], pk, pv, big[:, :, :, 512:640], big[:, :, :, 640:768], own_len, out=out)
    attn_check(got, q, pk, pv, ok, ov, own_len)
    far = torch.zeros(2, 1200000, 2, 1024, device="cuda", dtype=torch.bfloat16)
    far[1, 1199000:1199050, :, :128], far[1, 1199000:1199050, :, 128:256] = ok[0], ov[0]
    got = pkg.prefix_attention(q[:1], far[1, 1199000:1199050, :, :128], far[1, 1199000:1199050, :, 128:256])
    attn_check(got, q[:1], ok[0], ov[0], None, None, None)


# ---- verification ---------------------------------------------------------------------------------------------------
def verify_ref(logits, drafts, ua, us, probs, n_draft, temperature):
    B, R, V = logits.shape
    counts, tokens = [], torch.full((B, R), -1, dtype=torch.int32)
    for b in range(B):
        t = 1.0 if temperature is None else float(temperature[b])
        n = R - 1 if n_draft is None else min(max(int(n_draft[b]), 0), R - 1)
        r = 0
        while True:
            x = logits[b, r].double()
            if not (t >= 0 and t < math.inf) or torch.isnan(x).any() or (x == math.inf).any() or (x == -math.inf).all():
                tokens[b] = -1
                counts.append(-1 - r)
                break
            if t > 0:
                p = torch.exp((x - x.max()) / t)
                p = p / p.sum()
            else:
                p = torch.zeros_like(x)
                p[int((x == x.max()).nonzero()[0])] = 1
            if r < n:
                d = int(drafts[b, r])
                q = torch.zeros_like(p)
                if probs is not None:
                    q = probs[b, r].double()
                elif 0 <= d < V:
                    q[d] = 1
                if 0 <= d < V and float(ua[b, r]) * float(q[d]) < float(p[d]):
                    tokens[b, r] = d
                    r += 1
                    continue
                rest = (p - q).clamp(min=0)
                p = rest if float(rest.sum()) > 0 else p
            upto = p.cumsum(0)
            tokens[b, r] = int((upto > float(us[b]) * float(upto[-1])).nonzero()[0])
            counts.append(r)
            break
    return torch.tensor(counts, dtype=torch.int32), tokens


def verify_case(B, K, V, dt, probs, seed=0, lead=True):
    g = rng(seed * 100 + B + K * 31 + V)
    dev = {"device": "cuda", "generator": g}
    x = torch.randn(B, K + 1, V, **dev) * 2
    best = torch.randint(0, V, (B, K + 1, 1), **dev)
    if lead:
        x.scatter_(2, best, 3 + math.log(V))
    q = torch.softmax(x[:, :K] * 0.8 + 0.4 * torch.randn(B, K, V, **dev), -1) if probs else None
    drafts = torch.multinomial(q.view(B * K, V), 1, generator=g).view(B, K) if probs and K else torch.where(torch.rand(B, K, **dev) < 0.9, best[:, :K, 0], torch.randint(0, V, (B, K), **dev))
    return x.to(DT[dt]), drafts.to(torch.int32), torch.rand(B, K, **dev), torch.rand(B, **dev), q


def verify_check(x, d, ua, us, q=None, n_draft=None, temperature=None):
    got = pkg.verify_drafts(x, d, ua, us, draft_probs=q, n_draft=n_draft, temperature=temperature)
    want = verify_ref(x, d, ua, us, q, n_draft, temperature)
    assert torch.equal(got[0].cpu(), want[0]), (got[0], want[0])
    assert torch.equal(got[1].cpu(), want[1]), (got[1], want[1])
    return got


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("B,K,V", [(1, 0, 1), (1, 1, 2), (3, 2, 33), (2, 15, 151936), (40, 5, 1000), (5, 7, 32001), (2, 3, 4097), (1, 255, 50)])
def test_verify_against_the_definition(B, K, V, probs, dt):
    for seed in range(3):
        x, d, ua, us, q = verify_case(B, K, V, dt, probs, seed)
        verify_check(x, d, ua, us, q)
        g = rng(seed)
        n = torch.randint(-1, K + 2, (B,), device="cuda", generator=g).to(torch.int32)
        t = torch.rand(B, device="cuda", generator=g) * 2
        t[::3] = 0
        verify_check(x, d, ua, us, q, n, t)


def test_verify_flat_rows_and_the_ends_of_the_unit_interval():
    V = 4096
    x = torch.zeros(5, 2, V, device="cuda")
    d = torch.tensor([[0], [V - 1], [7], [7], [7]], device="cuda", dtype=torch.int32)
    below = float(torch.nextafter(torch.tensor(1.0), torch.tensor(0.0)))
    ua = torch.tensor([[0.0], [1 / V], [below], [1 / V * (1 - 2 ** -20)], [0.5]], device="cuda")   # at, below and beside p = 1 / V, all exact
    us = torch.tensor([0.0, 0.0, below, 0.5, 1 / V], device="cuda")
    n, tok = verify_check(x, d, ua, us)
    assert n.tolist() == [1, 0, 0, 1, 0] and tok[0].tolist() == [0, 0] and tok[1, 0] == 0 and tok[2, 0] == V - 1


def test_verify_masked_tokens_refused_rows_and_drafts_outside():
    x, d, ua, us, q = verify_case(8, 3, 500, "f32", False, 4)
    x[0, :, 100:] = -math.inf
    d[0, 0] = 200                              # a draft whose probability is zero
    x[1, 0, 3] = math.nan
    x[2, 1, 3] = math.inf
    d[2, 0] = int(x[2, 0].argmax())
    ua[2, 0] = 0.0
    x[3, 0] = -math.inf
    x[4, 3, 0] = math.nan                      # a row that counts only if all drafts stand
    d[5, 0] = -1
    d[6, 1] = 500
    x[7] = x[7].clamp(max=torch.finfo(torch.float32).min)   # the type's lowest value everywhere
    n, _ = verify_check(x, d, ua, us)
    assert n[1] == -1 and n[2] == -2 and n[3] == -1 and n[5] == 0
    t = torch.tensor([-1.0, math.nan, math.inf, 1e-30, 1e30, 1e-45, 0.0, 1.0], device="cuda")
    verify_check(x, d, ua, us, temperature=t)


def test_verify_residual_that_is_empty_draws_from_the_target():
    # q equals p in 64 bits: a draft cannot be refused there; and with more than p everywhere it is, with nothing left over
    x = torch.zeros(2, 2, 8, device="cuda")
    q = torch.full((2, 1, 8), 0.125, device="cuda")
    q[1] = 0.5
    n, tok = verify_check(x, torch.zeros(2, 1, device="cuda", dtype=torch.int32), torch.full((2, 1), 0.999, device="cuda"), torch.full((2,), 0.5, device="cuda"), q)
    assert n.tolist() == [1, 0] and tok[1].tolist() == [4, -1]


def test_verify_strided_logits():
    x, d, ua, us, q = verify_case(3, 4, 700, "bf16", True, 9)
    big = torch.full((3, 7, 801), math.nan, device="cuda", dtype=torch.bfloat16)
    big[:, 1:6, 3:703] = x
    wide = torch.full((4, 3, 705), math.nan, device="cuda").permute(1, 0, 2)
    wide[:, :, 1:701] = q
    a = pkg.verify_drafts(x, d, ua, us, draft_probs=q)
    b = pkg.verify_drafts(big[:, 1:6, 3:703], d, ua, us, draft_probs=wide[:, :, 1:701])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert pkg.verify_drafts(x[:0], d[:0], ua[:0], us[:0])[1].shape == (0, 5)


# ---- together -------------------------------------------------------------------------------------------------------
class Step:
    """One layer's attention and a head over a batch of drafted blocks: norm, rotate and store, attend, decide."""

    def __init__(self, seed, B=5, n=4, hq=8, hk=2, D=128, P=333, cap=64, V=1000):
        g = rng(seed)
        dev = {"device": "cuda", "generator": g}
        self.B, self.n, self.hq, self.hk, self.D, self.cap = B, n, hq, hk, D, cap
        self.pk, self.pv = (torch.randn(P, hk, D, **dev).half() for _ in "kv")
        self.kc, self.vc = (torch.full((B, cap, hk, D), math.nan, device="cuda", dtype=torch.half) for _ in "kv")
        self.P, self.head, self.w = P, torch.randn(hq * D, V, **dev) * 0.3, [torch.rand(D, **dev) + 0.5 for _ in "qk"]
        self.own = torch.randint(0, 20, (B,), **dev).to(torch.int32)
        for b in range(B):
            self.kc[b, :int(self.own[b])], self.vc[b, :int(self.own[b])] = (torch.randn(int(self.own[b]), hk, D, **dev).half() for _ in "kv")
        self.x = torch.randn(B * n, (hq + 2 * hk) * D, **dev)
        self.d, self.ua, self.us = torch.randint(0, V, (B, n - 1), **dev).to(torch.int32), torch.rand(B, n - 1, **dev) * 0.02, torch.rand(B, **dev)

    def inputs(self):
        i = torch.arange(self.n, device="cuda")
        rows = (torch.arange(self.B, device="cuda")[:, None] * self.cap + self.own[:, None] + i).reshape(-1)
        pos = (self.P + self.own[:, None] + i).reshape(-1).to(torch.int32)
        heads = self.x.view(self.B * self.n, self.hq + 2 * self.hk, self.D)
        return rows, pos, heads[:, :self.hq], heads[:, self.hq:self.hq + self.hk], heads[:, self.hq + self.hk:]

    def run(self, stream=None):
        rows, pos, q, k, v = self.inputs()
        qo = torch.empty(q.shape, device="cuda", dtype=torch.half)
        pkg.qk_norm_rope(q, k, pos, theta=1e6, rotary_dim=32, q_weight=self.w[0], k_weight=self.w[1], q_out=qo, k_out=self.kc.view(-1, self.hk, self.D), k_rows=rows, v=v,
                         v_out=self.vc.view(-1, self.hk, self.D), stream=stream)
        o = pkg.prefix_attention(qo.view(self.B, self.n, self.hq, self.D), self.pk, self.pv, self.kc, self.vc, self.own + self.n, stream=stream)
        self.logits = o.reshape(self.B, self.n, -1).float() @ self.head
        return o, *pkg.verify_drafts(self.logits, self.d, self.ua, self.us, stream=stream)


def test_a_step_of_a_batch():
    s = Step(0)
    o, n, tok = s.run()
    rows, pos, q, k, v = s.inputs()
    want, size = rope_ref(k, s.w[1], pos[None], 1e6, 32, [16], False)
    rope_close(s.kc.view(-1, s.hk, s.D)[rows], want, size, s.D)
    qr, size = rope_ref(q, s.w[0], pos[None], 1e6, 32, [16], False)
    attn_check(o, qr.half().view(s.B, s.n, s.hq, s.D), s.pk, s.pv, s.kc, s.vc, s.own + s.n)
    want = verify_ref(s.logits, s.d, s.ua, s.us, None, None, None)
    assert torch.equal(n.cpu(), want[0]) and torch.equal(tok.cpu(), want[1])
    # a drafter that agrees on some tokens
    d = torch.where(torch.rand(s.d.shape, device="cuda", generator=rng(2)) < 0.7, s.logits[:, :-1].argmax(-1).to(torch.int32), s.d)
    verify_check(s.logits, d, s.ua, s.us)


def test_a_captured_step_follows_its_inputs_and_other_streams_work():
    s, side = Step(1), torch.cuda.Stream()
    want = [x.clone() for x in s.run()]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a, b in zip(s.run(), want):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = s.run()
    for seed in (1, 2, 3):
        t = Step(seed)
        for name in ("pk", "pv", "kc", "vc", "head", "own", "x", "d", "ua", "us"):
            getattr(s, name).copy_(getattr(t, name))
        t.w, s.w[0][:], s.w[1][:] = t.w, t.w[0], t.w[1]
        graph.replay()
        for a, b in zip(got, t.run()):
            assert torch.equal(a, b)


def test_two_calls_at_once_on_two_streams():
    steps = [Step(s, B=20, n=8, P=4000) for s in (4, 5)]
    want = [[x.clone() for x in s.run()] for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    got = [[], []]
    for _ in range(5):
        for i, (s, st) in enumerate(zip(steps, streams)):
            with torch.cuda.stream(st):
                got[i].append(s.run())
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(r, w))


# ---- what is refused only where there is a device ------------------------------------------------------------------
def test_workspaces_that_are_too_small_or_lie_askew():
    import ctypes as C
    import importlib
    ops = importlib.import_module("qwen-llm_b200.batch_ops")
    q, pk, pv, ok, ov = attn_case(3, 1, 8, 2, 128, 5000, 64, "bf16")
    own_len = torch.tensor([1, 64, 9], device="cuda", dtype=torch.int32)
    out = torch.full_like(q, 7)
    a = ops.PrefixAttentionArgs(dtype=ops.BF16, batch=3, n_tokens=1, n_q_heads=8, n_kv_heads=2, head_dim=128, scale=0.1, prefix_len=5000, own_capacity=64)
    for name, x in (("q", q), ("prefix_k", pk), ("prefix_v", pv), ("own_k", ok), ("own_v", ov), ("own_len", own_len), ("out", out)):
        setattr(a, name, x.data_ptr())
    for name, x in (("q", q), ("out", out)):
        for i, n in enumerate(("batch", "token", "head")):
            setattr(a, f"{name}_{n}_stride", x.stride(i))
    for name, x in (("prefix_k", pk), ("prefix_v", pv)):
        for i, n in enumerate(("row", "head")):
            setattr(a, f"{name}_{n}_stride", x.stride(i))
    for name, x in (("own_k", ok), ("own_v", ov)):
        for i, n in enumerate(("batch", "row", "head")):
            setattr(a, f"{name}_{n}_stride", x.stride(i))
    L = pkg.lib()
    I, V = C.c_int32, C.c_void_p
    query, call = C.CFUNCTYPE(I, I, V, V)(("dfl_prefix_attention_workspace", L)), C.CFUNCTYPE(I, I, V, V)(("dfl_prefix_attention", L))
    need = C.c_uint64()
    pkg.check(query(0, C.byref(a), C.byref(need)))
    assert need.value > 0
    work = torch.empty(need.value + 512, device="cuda", dtype=torch.uint8)
    a.workspace, a.workspace_bytes = work.data_ptr(), need.value - 1
    for change, name in ((dict(), "BAD_SHAPE"), (dict(workspace=work.data_ptr() + 128, workspace_bytes=need.value), "BAD_ARG"), (dict(workspace=None), "BAD_ARG")):
        for k, v in change.items():
            setattr(a, k, v)
        with pytest.raises(pkg.DflError) as e:
            pkg.check(call(0, C.byref(a), None))
        assert e.value.name == name
    torch.cuda.synchronize()
    assert (out == 7).all()
    a.workspace = work.data_ptr()
    pkg.check(call(0, C.byref(a), None))
    torch.cuda.synchronize()
    attn_check(out, q, pk, pv, ok, ov, own_len, scale=a.scale)


def test_wrappers_refuse_gradients_and_outputs_that_overlap_themselves():
    q, pk, pv, ok, ov = attn_case(2, 3, 4, 2, 64, 100, 8, "f16")
    pos = torch.arange(6, device="cuda", dtype=torch.int32)
    flat, keys = q.reshape(6, 4, 64), pk[:6]
    for x in (q.clone().requires_grad_(), q):
        if x.requires_grad:
            with pytest.raises(RuntimeError, match="no backward pass"):
                pkg.prefix_attention(x, pk, pv)
            with pytest.raises(RuntimeError, match="no backward pass"):
                pkg.qk_norm_rope(x.reshape(6, 4, 64), keys, pos, theta=1e4)
            with torch.no_grad():
                a = pkg.prefix_attention(x, pk, pv)
        else:
            assert torch.equal(pkg.prefix_attention(x, pk, pv), a)
    logits = torch.zeros(2, 2, 10, device="cuda", requires_grad=True)
    u = torch.zeros(2, 1, device="cuda")
    with pytest.raises(RuntimeError, match="no backward pass"):
        pkg.verify_drafts(logits, u.to(torch.int32), u, u[:, 0].contiguous())
    with pytest.raises(ValueError, match="out: an expanded dimension"):
        pkg.prefix_attention(q, pk, pv, out=torch.empty(1, 3, 4, 64, device="cuda", dtype=torch.half).expand(2, 3, 4, 64))
    with pytest.raises(ValueError, match="k_out: an expanded dimension"):
        pkg.qk_norm_rope(flat, keys, pos, theta=1e4, k_out=torch.empty(6, 1, 64, device="cuda", dtype=torch.half).expand(6, 2, 64))
    with pytest.raises(pkg.DflError, match="a stride of K or V is zero"):
        pkg.prefix_attention(q, pk[:, :1].expand(100, 2, 64), pv)


# ---- sizes that spread otherwise -----------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens,hq,hk,dim", [(300, 32, 8, 128), (40, 5, 3, 64), (1500, 2, 2, 256)])
def test_rope_heads_shared_out_over_warps(tokens, hq, hk, dim):
    q, k, v, pos, sections, w = rope_case(tokens, hq, hk, dim, dim // 2, 1, False, "bf16")
    rows = torch.randperm(2 * tokens, device="cuda", generator=rng(1))[:tokens]
    rows[::5] = -1
    cache = [torch.full((2 * tokens, hk, dim), 3.0, device="cuda", dtype=torch.bfloat16) for _ in "kv"]
    qo, ko, vo = pkg.qk_norm_rope(q, k, pos, theta=1e4, rotary_dim=dim // 2, sections=sections, q_weight=w[0], k_weight=w[1], v=v, k_out=cache[0], v_out=cache[1], k_rows=rows)
    rope_close(qo, *rope_ref(q, w[0], pos, 1e4, dim // 2, sections, False), dim)
    kept = rows >= 0
    want, size = rope_ref(k, w[1], pos, 1e4, dim // 2, sections, False)
    rope_close(ko[rows[kept]], want[kept], size[kept], dim)
    assert torch.equal(vo[rows[kept]], v[kept])
    left = torch.ones(2 * tokens, device="cuda", dtype=torch.bool)
    left[rows[kept]] = False
    assert (ko[left] == 3).all() and (vo[left] == 3).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("probs", [False, True])
def test_verify_more_pieces_than_are_under_way_at_once(probs, dt):
    B, K, V = 70, 15, 20001      # some rows are never needed, and which becomes known on the way
    x, d, ua, us, q = verify_case(B, K, V, dt, probs, 7)
    g = rng(5)
    n = torch.randint(0, K + 1, (B,), device="cuda", generator=g).to(torch.int32)
    t = torch.rand(B, device="cuda", generator=g) * 1.5
    t[::4] = 0
    a, _ = verify_check(x, d, ua, us, q)
    b, _ = verify_check(x, d, ua, us, q, n, t)
    assert (a < K).any() and (a > 0).any() and not torch.equal(a, b)
    x[3, 2, 5] = math.nan
    verify_check(x, d, ua, us, q, n, t)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = pkg.verify_drafts(x, d, ua, us, draft_probs=q, n_draft=n, temperature=t)
    for seed in (8, 9):
        new = verify_case(B, K, V, dt, probs, seed)
        for old, y in zip((x, d, ua, us) + ((q,) if probs else ()), new):
            old.copy_(y)
        graph.replay()
        want = pkg.verify_drafts(x, d, ua, us, draft_probs=q, n_draft=n, temperature=t)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_verify_a_refused_draft_with_all_the_mass():
    # u = 1 lies outside [0, 1): such a draft falls, nothing is left beside it, and it is drawn from the target itself
    x = torch.full((2, 2, 300), -math.inf, device="cuda")
    x[:, :, 17] = 2.0
    d = torch.full((2, 1), 17, device="cuda", dtype=torch.int32)
    n, tok = pkg.verify_drafts(x, d, torch.ones(2, 1, device="cuda"), torch.tensor([0.0, 0.9], device="cuda"))
    assert n.tolist() == [0, 0] and tok.tolist() == [[17, -1]] * 2


@pytest.mark.parametrize("case", [(333, 1, 3, 1, 128, 64, 260, "f16", "rows"), (301, 2, 4, 1, 64, 0, 500, "bf16", "rows"), (151, 1, 5, 5, 128, 700, 1030, "bf16", "heads")], ids=str)
def test_attention_of_many_requests_with_few_rows(case):
    # an odd number of them, of lengths from nothing to all
    test_attention_against_the_definition(case)


@pytest.mark.parametrize("case", [(300, 8, 4, 64, 60, 1, True, "bf16", "f16"), (33, 6, 2, 64, 2, 1, False, "f32", "f32"), (257, 4, 3, 128, 102, 3, True, "bf16", "bf16"),
                                  (40, 5, 1, 128, 126, 1, False, "f16", "f32"), (65, 3, 2, 256, 250, 2, False, "f32", "bf16"), (7, 1, 1, 256, 6, 3, True, "f16", "f16"),
                                  (90, 4, 2, 80, 78, 2, True, "bf16", "bf16"), (129, 2, 2, 96, 96, 1, False, "f32", "f16")], ids=str)
def test_rope_rotary_widths_of_all_kinds(case):
    test_rope_against_the_definition(case)


@pytest.mark.parametrize("case", [(100, 1, 16, 4, 64, 3000, 130, "bf16", "rows"), (50, 4, 8, 2, 256, 900, 40, "f16", "rows"), (50, 2, 16, 4, 128, 2500, 140, "f16", "heads")], ids=str)
def test_attention_of_some_hundred_rows_a_head(case):
    test_attention_against_the_definition(case)


@pytest.mark.parametrize("case", [(56, 7, 56, 8, 128, 1300, 246, "f16", "rows"), (42, 100, 8, 8, 128, 853, 100, "bf16", "rows"), (30, 8, 16, 2, 256, 6001, 515, "bf16", "heads"),
                                  (60, 12, 12, 2, 64, 5000, 300, "f16", "rows"), (30, 8, 16, 2, 256, 12001, 515, "f16", "heads"),
                                  (56, 7, 56, 8, 64, 1300, 246, "bf16", "rows"), (42, 60, 8, 8, 64, 1853, 300, "f16", "heads")], ids=str)
def test_attention_of_prefix_and_own_items_that_fill_up_each_other(case):
    test_attention_against_the_definition(case)


# ---- draws at the ends of what has mass -----------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("B,V", [(300, 20000), (100, 32001), (20, 40000), (2, 151936), (30, 300)])
def test_verify_u_of_one_draws_the_last_token_with_mass(B, V, dt):
    # Rows that end in tokens without mass, as a masked vocabulary does: some of them inside one warp's run, some over many.  The last token's weight
    # is some 1e-9 of the row's at least, a sum's roundings 1e-13, so u = 1 (and more) can only mean that token.
    for seed in range(4):
        g = rng(seed * 10 + V)
        x = torch.randn(B, 2, V, device="cuda", generator=g).mul_(2).to(DT[dt])
        last = (torch.rand(B, device="cuda", generator=g) * V).long().clamp(min=3)
        last[::5] = V - 1 - torch.arange(len(last[::5]), device="cuda") % 5
        last.clamp_(min=3, max=V - 1)
        x.masked_fill_((torch.arange(V, device="cuda") > last[:, None])[:, None], -math.inf)
        us = torch.ones(B, device="cuda")
        us[::7] = 1.5
        us[1] = math.inf
        none = torch.empty(B, 0, device="cuda")
        n, tok = pkg.verify_drafts(x[:, :1], none.to(torch.int32), none, us)
        assert (n == 0).all() and torch.equal(tok[:, 0].long(), last)
        # behind a refused draft without distributions, and from what is left beside one: q holds all of p from `last` on, token `before` is the last with a rest
        d = torch.zeros(B, 1, device="cuda", dtype=torch.int32)
        never = torch.full((B, 1), 1.0, device="cuda")
        n, tok = pkg.verify_drafts(x, d, never, us)
        assert (n == 0).all() and torch.equal(tok[:, 0].long(), last)
        p = torch.softmax(x[:, :1].double(), -1)
        before = (last // 2).clamp(min=1)
        q = torch.where(torch.arange(V, device="cuda") > before[:, None, None], p * 2, p * 0.5).float()
        q[:, 0, 0] = 1.0
        n, tok = pkg.verify_drafts(x, d, never, us, draft_probs=q)
        assert (n == 0).all() and torch.equal(tok[:, 0].long(), before)


# ---- drafts beside the border of standing and falling ---------------------------------------------------------------
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("B,K,V,sharp", [(64, 3, 151936, 2.0), (6, 3, 151936, 1.0), (40, 15, 32001, 0.3), (12, 7, 1000, 3.0), (5, 255, 777, 1.0)])
def test_verify_drafts_a_step_of_f32_beside_the_border(B, K, V, sharp, probs, dt):
    # u q(d) is one of the f32 numbers around p(d), within 2^-23 of it: far from it for a sum in 64 bits (1e-13), nothing for one in 32 (some 1e-7)
    g = rng(V + B)
    dev = {"device": "cuda", "generator": g}
    x = (torch.randn(B, K + 1, V, **dev) * sharp).to(DT[dt])
    t = torch.rand(B, **dev) + 0.5
    d = torch.randint(0, V, (B, K), **dev).to(torch.int32)
    p = torch.softmax(x.double() / t.double()[:, None, None], -1)[:, :K].gather(2, d.long()[..., None])[..., 0]
    ua = torch.rand(B, K, **dev) * 0.6 + 0.3
    goal = p / ua.double() if probs else p
    near = goal.float()
    steps = torch.randint(0, 4, (B, K), **dev)
    near = torch.where(steps == 0, torch.nextafter(near, torch.ones_like(near)), torch.where(steps > 1, torch.nextafter(near, torch.zeros_like(near)), near))
    q = None
    if probs:
        q = torch.softmax(torch.randn(B, K, V, **dev), -1)
        q.scatter_(2, d.long()[..., None], near[..., None])
    else:
        ua = near
    n, _ = verify_check(x, d, ua, torch.rand(B, **dev), q, None, t)
    assert n.max() > 1 and n.min() < K     # some stand, some fall


# ---- temperatures at the ends of f32 --------------------------------------------------------------------------------
@pytest.mark.parametrize("probs", [False, True])
def test_verify_temperatures_at_the_ends_of_f32_count_as_the_nearest_usable(probs):
    # logits of the temperature's own size, so that the weights are neither equal nor zero: subnormal ones under the smallest, huge ones under the largest
    B, K, V = 8, 2, 3001
    low, high = 2.0 ** -122, 2.0 ** 122
    t = torch.tensor([1e-45, 1e-40, 1.1e-38, low, high, 2e37, 3.4e38, 1.0], device="cuda")
    for seed in range(3):
        x, d, ua, us, q = verify_case(B, K, V, "f32", probs, seed)
        x = (x * t.clamp(low, high)[:, None, None].double()).float()
        x[6, :, 5:9] = torch.finfo(torch.float32).min
        got = pkg.verify_drafts(x, d, ua, us, draft_probs=q, temperature=t)
        want = verify_ref(x, d, ua, us, q, None, t.clamp(low, high))
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
        # logits far apart: a row's largest alone, and all alike
        x = x / t.clamp(low, high)[:, None, None]
        verify_check(x, d, ua, us, q, None, t)


# ---- memory on other streams ----------------------------------------------------------------------------------------
def test_tensors_given_with_a_stream_stay_theirs_until_it_has_passed():
    # made on the current stream, used on another, dropped at once: their memory may not go to the next tensor before the other stream has read it
    side = torch.cuda.Stream()
    q, pk, pv, ok, ov = attn_case(4, 8, 16, 2, 128, 3000, 64, "bf16")
    own_len = torch.tensor([8, 64, 33, 20], device="cuda", dtype=torch.int32)
    pos = torch.arange(32, device="cuda", dtype=torch.int32)
    x, d, ua, us, p = verify_case(4, 3, 60000, "f32", True)
    calls = [
        (lambda a, **kw: pkg.prefix_attention(*a, **kw), (q, pk, pv, ok, ov, own_len)),
        (lambda a, **kw: pkg.qk_norm_rope(a[0], a[1], a[2], theta=1e4, v=a[3], **kw), (q.reshape(32, 16, 128), pk[:32].clone(), pos, pv[:32].clone())),
        (lambda a, **kw: pkg.verify_drafts(*a[:4], draft_probs=a[4], **kw), (x, d, ua, us, p)),
    ]
    for call, tensors in calls:
        as_tuple = lambda r: r if isinstance(r, tuple) else (r,)
        want = [y.clone() for y in as_tuple(call(tensors))]
        torch.cuda.synchronize()
        given = [y.clone() for y in tensors]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)      # some 10 ms
        got = as_tuple(call(given, stream=side))
        sizes = [(y.shape, y.dtype) for y in given]
        del given
        over = [torch.zeros(s, dtype=t, device="cuda") for s, t in sizes]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        del over


# ---- torch's bookkeeping ---------------------------------------------------------------------------------------------
def wrapper_inputs(dt="f16"):
    q, pk, pv, ok, ov = attn_case(2, 3, 4, 2, 64, 100, 8, dt)
    pos = torch.arange(6, device="cuda", dtype=torch.int32)
    return q, pk, pv, ok, ov, torch.tensor([8, 5], device="cuda", dtype=torch.int32), q.reshape(6, 4, 64), pk[:6], pv[:6], pos


def test_wrappers_refuse_outputs_that_require_gradients():
    q, pk, pv, ok, ov, own_len, flat, k, v, pos = wrapper_inputs()
    leaf = lambda x: torch.zeros_like(x).requires_grad_()
    for call in (lambda: pkg.prefix_attention(q, pk, pv, out=leaf(q)), lambda: pkg.qk_norm_rope(flat, k, pos, theta=1e4, q_out=leaf(flat)),
                 lambda: pkg.qk_norm_rope(flat, k, pos, theta=1e4, k_out=leaf(k)), lambda: pkg.qk_norm_rope(flat, k, pos, theta=1e4, v=v, v_out=leaf(v))):
        with pytest.raises(RuntimeError, match="no backward pass"):
            call()
        with torch.no_grad():
            call()


def test_wrappers_refuse_tangents():
    import torch.autograd.forward_ad as fw
    q, pk, pv, ok, ov, own_len, flat, k, v, pos = wrapper_inputs()
    logits, u = torch.zeros(2, 2, 10, device="cuda"), torch.zeros(2, 1, device="cuda")
    with fw.dual_level(), torch.no_grad():     # forward mode is not what no_grad() turns off
        dual = lambda x: fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: pkg.prefix_attention(dual(q), pk, pv), lambda: pkg.prefix_attention(q, pk, dual(pv)), lambda: pkg.prefix_attention(q, pk, pv, ok, dual(ov), own_len),
                     lambda: pkg.prefix_attention(q, pk, pv, out=dual(torch.empty_like(q))), lambda: pkg.qk_norm_rope(dual(flat), k, pos, theta=1e4),
                     lambda: pkg.qk_norm_rope(flat, k, pos, theta=1e4, k_weight=dual(torch.ones(64, device="cuda"))), lambda: pkg.qk_norm_rope(flat, k, pos, theta=1e4, v=dual(v)),
                     lambda: pkg.qk_norm_rope(flat, k, pos, theta=1e4, q_out=dual(torch.empty_like(flat))), lambda: pkg.verify_drafts(dual(logits), u.int(), u, u[:, 0].contiguous())):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
        pkg.prefix_attention(q, pk, pv)        # without tangents as ever
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: pkg.prefix_attention(x, pk, pv), (q,), (torch.ones_like(q),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: pkg.prefix_attention(x, pk, pv))(q[None])


def test_a_saved_tensor_that_is_written_over_is_noticed():
    q, pk, pv, ok, ov, own_len, flat, k, v, pos = wrapper_inputs("bf16")
    for name, call in (("out", lambda x: pkg.prefix_attention(q, pk, pv, out=x)), ("q_out", lambda x: pkg.qk_norm_rope(flat, k, pos, theta=1e4, q_out=x)),
                       ("k_out", lambda x: pkg.qk_norm_rope(flat, k, pos, theta=1e4, k_out=x)), ("v_out", lambda x: pkg.qk_norm_rope(flat, k, pos, theta=1e4, v=v, v_out=x))):
        x = torch.ones_like({"out": q, "q_out": flat, "k_out": k, "v_out": v}[name])
        w = torch.ones_like(x).requires_grad_()
        y = (x * w).sum()                      # saves x
        before = x._version
        with torch.no_grad():
            call(x)
        assert x._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


# ---- which arguments go together ------------------------------------------------------------------------------------
def test_rope_new_v_rows_beside_a_longer_k_out():
    q, k, v, pos, sections, (wq, wk) = rope_case(9, 4, 2, 64, 64, 1, False, "bf16")
    want = pkg.qk_norm_rope(q, k, pos, theta=1e4, sections=sections, q_weight=wq, k_weight=wk, v=v)
    k_out, v_out = (torch.full((12, 2, 64), 5.0, device="cuda", dtype=torch.bfloat16) for _ in "kv")
    got = pkg.qk_norm_rope(q, k, pos, theta=1e4, sections=sections, q_weight=wq, k_weight=wk, v=v, k_out=k_out)
    assert got[1] is k_out and got[2].shape == (9, 2, 64) and torch.equal(got[2], want[2]) and torch.equal(k_out[:9], want[1]) and (k_out[9:] == 5).all()
    got = pkg.qk_norm_rope(q, k, pos, theta=1e4, sections=sections, q_weight=wq, k_weight=wk, v=v, v_out=v_out)
    assert got[2] is v_out and torch.equal(v_out[:9], want[2]) and torch.equal(got[1], want[1]) and (v_out[9:] == 5).all()
    # rows by number: both outputs are one cache
    rows = torch.arange(9, device="cuda")
    with pytest.raises(ValueError, match="v_out: shape"):
        pkg.qk_norm_rope(q, k, pos, theta=1e4, sections=sections, v=v, k_out=k_out, v_out=v_out[:11], k_rows=rows)
    with pytest.raises(pkg.DflError, match="fewer output rows than tokens"):
        pkg.qk_norm_rope(q, k, pos, theta=1e4, sections=sections, v=v, v_out=v_out[:8])


def test_wrappers_refuse_arguments_that_nothing_would_read():
    q, pk, pv, ok, ov, own_len, flat, k, v, pos = wrapper_inputs()
    for extra in (dict(own_v=ov), dict(own_v=ov, own_len=own_len)):
        with pytest.raises(ValueError, match="own_v: without own_k"):
            pkg.prefix_attention(q, pk, pv, **extra)
    assert torch.equal(pkg.prefix_attention(q, pk, pv, own_len=own_len), pkg.prefix_attention(q, pk, pv))   # clamped to the rows there are: none
    with pytest.raises(ValueError, match="own_k: needs own_v and own_len"):
        pkg.prefix_attention(q, pk, pv, ok, ov)
    with pytest.raises(ValueError, match="v_out: without v"):
        pkg.qk_norm_rope(flat, k, pos, theta=1e4, v_out=torch.empty_like(v))


def test_a_call_with_a_stream_inside_a_capture():
    q, pk, pv, ok, ov = attn_case(3, 4, 8, 2, 128, 900, 32, "f16")
    own_len = torch.tensor([4, 32, 11], device="cuda", dtype=torch.int32)
    x, d, ua, us, _ = verify_case(3, 3, 5000, "f32", False)
    want = pkg.prefix_attention(q, pk, pv, ok, ov, own_len), *pkg.verify_drafts(x, d, ua, us)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        got = pkg.prefix_attention(q * 1, pk, pv, ok, ov, own_len, stream=side), *pkg.verify_drafts(x * 1, d, ua, us, stream=side)   # inputs made inside and dropped
        torch.cuda.current_stream().wait_stream(side)
    for y in got:
        y.zero_()
    for _ in range(3):
        graph.replay()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_wrappers_under_inference_mode():
    q, pk, pv, ok, ov, own_len, flat, k, v, pos = wrapper_inputs()
    want = pkg.prefix_attention(q, pk, pv, ok, ov, own_len), *pkg.qk_norm_rope(flat, k, pos, theta=1e4, v=v)
    outs = torch.empty_like(q), torch.empty_like(flat), torch.empty_like(k), torch.empty_like(v)     # made outside, as a cache is
    with torch.inference_mode():
        for kept in (outs, [torch.empty_like(x) for x in outs]):
            got = pkg.prefix_attention(q, pk, pv, ok, ov, own_len, out=kept[0]), *pkg.qk_norm_rope(flat, k, pos, theta=1e4, v=v, q_out=kept[1], k_out=kept[2], v_out=kept[3])
            for a, b in zip(got, want):
                assert torch.equal(a, b)
