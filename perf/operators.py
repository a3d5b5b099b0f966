"""Performance cases of the operators for a batch of requests that continue one prompt.

A step of such a batch norms and rotates the queries and keys of the block and stores its K / V rows, attends over the
shared prompt and each request's own rows, and, behind the head, decides which drafted tokens stand.  Geometries are those of
`qwen-llm_b200/synthetic.py` (32 / 8 heads of 128, 16 / 2 heads of 256, vocabulary 151 936) and relatives of them.
"""
import importlib
import math

import torch

own = False
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    rope = {"op": "rope", "theta": 1e7}
    attn = {"op": "attn", "layout": "rows"}
    verify = {"op": "verify", "vocab": 151936, "dtype": "f32"}
    return [
        # one decoded token of one request: latency
        {"name": "rope_token", **rope, "tokens": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 32, "axes": 1, "interleaved": False, "src": "bf16", "dst": "bf16", "cache": 4096},
        # a drafted block of 64 requests, f32 activations into an fp16 cache, a quarter of a wide head rotated
        {"name": "rope_block", **rope, "tokens": 1024, "q_heads": 16, "kv_heads": 2, "dim": 256, "rot": 64, "axes": 1, "interleaved": False, "src": "f32", "dst": "f16", "cache": 16384},
        # an ordinary long prompt
        {"name": "rope_prompt", **rope, "tokens": 8191, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "axes": 1, "interleaved": False, "src": "bf16", "dst": "bf16", "cache": 8192},
        # a video prompt: time, height and width dealt out over the frequencies in turn
        {"name": "rope_video", **rope, "tokens": 32768, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "axes": 3, "interleaved": True, "src": "bf16", "dst": "bf16", "cache": 40000},
        # a few requests, one token each, a short prompt: latency
        {"name": "attn_token_small", **attn, "batch": 4, "n": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "prefix": 1000, "cap": 256, "dtype": "bf16", "ragged": False},
        # many requests decoding over a long shared prompt, each with an answer of its own
        {"name": "attn_token_64", **attn, "batch": 64, "n": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "prefix": 32768, "cap": 1024, "dtype": "f16", "ragged": False},
        # drafted blocks of 48 requests, some of them shorter
        {"name": "attn_block_48", **attn, "batch": 48, "n": 16, "q_heads": 32, "kv_heads": 8, "dim": 128, "prefix": 16385, "cap": 700, "dtype": "f16", "ragged": True},
        # wide heads, eight queries to a key, cache rows head by head
        {"name": "attn_block_wide", **attn, "layout": "heads", "batch": 30, "n": 8, "q_heads": 16, "kv_heads": 2, "dim": 256, "prefix": 12001, "cap": 515, "dtype": "bf16", "ragged": False},
        # the requests' own prompts of different lengths behind the shared one
        {"name": "attn_prompts", **attn, "batch": 4, "n": 2048, "q_heads": 32, "kv_heads": 8, "dim": 128, "prefix": 8192, "cap": 2048, "dtype": "bf16", "ragged": True},
        # one request's block, proposals of a drafter that names one token: latency
        {"name": "verify_one", **verify, "batch": 1, "drafts": 15, "probs": False, "greedy": False, "ragged": False},
        # sixteen requests with the drafter's distributions
        {"name": "verify_16", **verify, "batch": 16, "drafts": 15, "probs": True, "greedy": False, "ragged": True},
        # a large batch
        {"name": "verify_128", **verify, "batch": 128, "drafts": 7, "probs": False, "greedy": False, "ragged": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attn", "attn", "attn", "verify", "verify"])
    if op == "rope":
        dim = rng.choice([64, 128, 256])
        axes = rng.choice([1, 1, 2, 3])
        kv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 5, 8])
        rot = rng.choice([dim, dim // 2, dim // 4, 2 * rng.randint(3, dim // 2)])
        tokens = _log_int(rng, 1, max(2, 32768 * 48 * 128 // (kv * (group + 2) * dim) // 2))
        return {"op": op, "theta": rng.choice([1e4, 1e6, 1e7]), "tokens": min(tokens, 32768), "q_heads": kv * group, "kv_heads": kv, "dim": dim, "rot": rot, "axes": axes,
                "interleaved": rng.random() < 0.5, "src": rng.choice(["f32", "f16", "bf16", "bf16"]), "dst": rng.choice(["f32", "f16", "bf16"]),
                "cache": min(tokens, 32768) + rng.randint(0, 4096)}
    if op == "attn":
        while True:
            dim, kv, group = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.randint(1, 8)
            n = rng.choice([1, 1, rng.randint(2, 16), rng.randint(2, 16), _log_int(rng, 17, 2048)])
            batch = _log_int(rng, 1, 64)
            prefix = rng.choice([0, _log_int(rng, 1, 65536), _log_int(rng, 256, 65536), _log_int(rng, 1024, 65536)])
            cap = max(n, _log_int(rng, 1, 4096))
            rows = batch * n * kv * group
            # no dearer than attn_prompts: its products, and its matrix of scores in the plain form
            if rows * dim * (prefix + cap) <= 4 * 2048 * 32 * 128 * 10240 and rows * (prefix + cap) <= 4 * 2048 * 32 * 10240 and batch * cap * kv * dim <= 1 << 28:
                break
        return {"op": op, "layout": rng.choice(["rows", "heads"]), "batch": batch, "n": n, "q_heads": kv * group, "kv_heads": kv, "dim": dim, "prefix": prefix, "cap": cap,
                "dtype": rng.choice(["f16", "bf16"]), "ragged": rng.random() < 0.5}
    while True:
        batch, drafts, vocab = _log_int(rng, 1, 128), rng.randint(0, 15), rng.choice([151936, 32000, _log_int(rng, 2, 200000)])
        probs = rng.random() < 0.5
        if batch * ((drafts + 1) + (drafts if probs else 0)) * vocab <= 128 * 8 * 151936:
            break
    return {"op": op, "vocab": vocab, "dtype": rng.choice(["f32", "f32", "f16", "bf16"]), "batch": batch, "drafts": drafts, "probs": probs,
            "greedy": rng.random() < 0.2, "ragged": rng.random() < 0.5}


def _sections(case):
    """How many of the rot / 2 frequencies each axis has: the first axis takes what the others leave."""
    half, axes = case["rot"] // 2, case["axes"]
    rest = half * 5 // 16 if axes == 3 else half // 2 if axes == 2 else 0
    rest = min(rest, (half - 1) // axes)
    return [half - rest * (axes - 1)] + [rest] * (axes - 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = {"device": "cuda", "generator": g}
    if case["op"] == "rope":
        T, hq, hk, D = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"]
        qkv = torch.randn(T, (hq + 2 * hk) * D, **dev).mul_(torch.rand(T, 1, **dev) * 3 + 0.1).to(DTYPES[case["src"]])   # one row of the fused projection
        heads = qkv.view(T, hq + 2 * hk, D)
        start = int(torch.randint(0, 100000, (1,), generator=torch.Generator().manual_seed(seed)))
        t = torch.arange(T, device="cuda")
        pos = torch.stack([start + t // 64 if case["axes"] > 1 else start + t, start + t // 8 % 8, start + t % 8][: case["axes"]]).to(torch.int32)
        s = {"q": heads[:, :hq], "k": heads[:, hq:hq + hk], "v": heads[:, hq + hk:], "pos": pos, "sections": _sections(case),
             "wq": torch.rand(D, **dev) + 0.5, "wk": torch.rand(D, **dev) + 0.5,
             "q_out": torch.empty(T, hq, D, device="cuda", dtype=DTYPES[case["dst"]]),
             "rows": torch.randperm(case["cache"], **dev)[:T],
             "k_cache": torch.zeros(case["cache"], hk, D, device="cuda", dtype=DTYPES[case["dst"]]),
             "v_cache": torch.zeros(case["cache"], hk, D, device="cuda", dtype=DTYPES[case["dst"]])}
    elif case["op"] == "attn":
        B, n, hq, hk, D, P, cap = (case[k] for k in ("batch", "n", "q_heads", "kv_heads", "dim", "prefix", "cap"))
        dt = DTYPES[case["dtype"]]
        s = {"q": torch.randn(B, n, hq, D, **dev).mul_(1.5).to(dt)}
        if case["layout"] == "rows":
            kv = [torch.randn(P, hk, D, **dev).to(dt) for _ in "kv"] + [torch.randn(B, cap, hk, D, **dev).to(dt) for _ in "kv"]
        else:
            kv = [torch.randn(hk, P, D, **dev).to(dt).transpose(0, 1) for _ in "kv"] + [torch.randn(B, hk, cap, D, **dev).to(dt).transpose(1, 2) for _ in "kv"]
        s["pk"], s["pv"], s["ok"], s["ov"] = kv
        q_len = torch.randint(max(1, n // 2), n + 1, (B,), **dev) if case["ragged"] else torch.full((B,), n, device="cuda")
        own_len = q_len + (torch.rand(B, **dev) * (cap - q_len + 1)).long().clamp(max=cap - n) if cap > n else q_len
        s["own_len"] = own_len.to(torch.int32)
        s["q_len"] = q_len.to(torch.int32) if case["ragged"] else None
        s["out"] = torch.zeros(B, n, hq, D, device="cuda", dtype=dt)
    else:
        B, K, V = case["batch"], case["drafts"], case["vocab"]
        logits = torch.randn(B, K + 1, V, **dev).mul_(2.0)
        # most of a row's mass sits on one token, as in text: 50 to 97 % of it
        share = torch.rand(B, K + 1, 1, **dev) * 0.47 + 0.5
        lead = torch.randint(0, V, (B, K + 1, 1), **dev)
        logits.scatter_(2, lead, 2.0 + math.log(V) + torch.log(share / (1 - share)))
        s = {"u_accept": torch.rand(B, K, **dev), "u_sample": torch.rand(B, **dev), "probs": None, "n_draft": None}
        s["logits"] = logits.to(DTYPES[case["dtype"]])
        if case["probs"] and K:
            near = logits[:, :K] * 0.9
            near.add_(torch.randn(B, K, V, **dev), alpha=0.3)
            s["probs"] = torch.softmax(near, -1)
            s["drafts"] = torch.multinomial(s["probs"].view(B * K, V), 1, generator=g).view(B, K).to(torch.int32)
        else:
            other = torch.randint(0, V, (B, K), **dev)
            s["drafts"] = torch.where(torch.rand(B, K, **dev) < 0.95, lead[:, :K, 0], other).to(torch.int32)
        if case["ragged"]:
            s["n_draft"] = torch.randint(0, K + 1, (B,), **dev).to(torch.int32)
        s["temperature"] = torch.rand(B, **dev) * 0.6 + 0.7
        if case["greedy"]:
            s["temperature"] = s["temperature"] * (torch.rand(B, **dev) < 0.5)
    s["case"] = dict(case)
    return s


def _axis_of(case, sections):
    """Which axis turns frequency j: blocks of frequencies one behind the other, or dealt out in turn."""
    j = torch.arange(case["rot"] // 2)
    if not case["interleaved"]:
        return torch.repeat_interleave(torch.arange(case["axes"]), torch.tensor(sections))
    a = j % case["axes"]
    return torch.where(j < case["axes"] * torch.tensor(sections)[a], a, torch.zeros_like(a))


def _rope_plain(s):
    case, half, rot = s["case"], s["case"]["rot"] // 2, s["case"]["rot"]
    freq = torch.pow(torch.tensor(case["theta"], dtype=torch.float64, device="cuda"), -torch.arange(half, device="cuda", dtype=torch.float64) / half)
    axis = _axis_of(case, s["sections"]).cuda()
    angle = s["pos"][axis].t().double() * freq    # [T][half]; far positions lose their place on the circle in 32 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, w):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        a, b = x[..., :half], x[..., half:rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)

    dt = s["q_out"].dtype
    s["q_out"].copy_(turned(s["q"], s["wq"]).to(dt))
    s["k_cache"].index_copy_(0, s["rows"], turned(s["k"], s["wk"]).to(dt))
    s["v_cache"].index_copy_(0, s["rows"], s["v"].to(dt))
    return s["q_out"], s["k_cache"], s["v_cache"]


def _attn_plain(s):
    q = s["q"].float()
    B, n, hq, D = q.shape
    cap, hk = s["ok"].shape[1:3]
    G, P = hq // hk, s["pk"].shape[0]
    scale = 1 / math.sqrt(D)
    q = q.view(B, n, hk, G, D) * scale
    own_len, i = s["own_len"].long(), torch.arange(n, device="cuda")
    q_len = torch.full_like(own_len, n) if s["q_len"] is None else s["q_len"].long()
    j = torch.arange(cap, device="cuda")
    seen = j < (own_len - q_len)[:, None, None] + i[:, None] + 1                                     # [B][n][cap]
    mine = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(B, hk, n * G, D), s["ok"].float().permute(0, 2, 3, 1)).view(B, hk, n, G, cap)
    mine.masked_fill_(~seen[:, None, :, None], -math.inf)
    shared = torch.matmul(q.permute(2, 0, 1, 3, 4).reshape(hk, B * n * G, D), s["pk"].float().permute(1, 2, 0))   # [hk][B n G][P]
    top = mine.amax(-1) if cap else torch.full((B, hk, n, G), -math.inf, device="cuda")
    if P:
        top = torch.maximum(top, shared.amax(-1).view(hk, B, n, G).permute(1, 0, 2, 3))
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    mine.sub_(top[..., None]).exp_()
    shared.sub_(top.permute(1, 0, 2, 3).reshape(hk, B * n * G, 1)).exp_()
    total = mine.sum(-1) + shared.sum(-1).view(hk, B, n, G).permute(1, 0, 2, 3)
    ov = s["ov"].float().masked_fill((j >= own_len[:, None])[..., None, None], 0.0)
    o = torch.matmul(mine.view(B, hk, n * G, cap), ov.permute(0, 2, 1, 3)).view(B, hk, n, G, D)
    o += torch.matmul(shared, s["pv"].float().permute(1, 0, 2)).view(hk, B, n, G, D).permute(1, 0, 2, 3, 4)
    o = torch.where(total[..., None] > 0, o / total[..., None], torch.zeros_like(o))
    o = o.permute(0, 2, 1, 3, 4).reshape(B, n, hq, D).to(s["out"].dtype)
    s["out"].copy_(torch.where((i < q_len[:, None])[..., None, None], o, s["out"]))   # rows behind a request's last token stay as they were
    return s["out"]


def _verify_plain(s):
    x = s["logits"].double()     # the sum of a row decides at a border: 64 bits
    B, R, V = x.shape
    K = R - 1
    t = s["temperature"].double()[:, None, None]
    w = torch.exp((x - x.amax(-1, keepdim=True)) / torch.where(t > 0, t, torch.ones_like(t)))
    best = torch.where(x == x.amax(-1, keepdim=True), torch.arange(V, device="cuda"), V).amin(-1, keepdim=True)   # ties: the lowest index
    w = torch.where(t > 0, w, torch.zeros_like(w).scatter_(2, best, 1.0))
    p = w / w.sum(-1, keepdim=True)
    n = torch.full((B,), K, device="cuda") if s["n_draft"] is None else s["n_draft"].long()
    d = s["drafts"].long()
    p_d = p[:, :K].gather(2, d[..., None])[..., 0]
    q_d = torch.ones_like(p_d) if s["probs"] is None else s["probs"].gather(2, d[..., None])[..., 0].double()
    i = torch.arange(K, device="cuda")
    stands = (s["u_accept"].double() * q_d < p_d) & (i < n[:, None])
    taken = stands.long().cumprod(1).sum(1)
    row = p.gather(1, taken[:, None, None].expand(B, 1, V))[:, 0]
    refused = taken < n
    at = taken.clamp(max=max(K - 1, 0))
    if K and s["probs"] is not None:
        q = s["probs"].gather(1, at[:, None, None].expand(B, 1, V))[:, 0].double()
        rest = (row - q).clamp(min=0.0)
    elif K:
        rest = row.scatter(1, d.gather(1, at[:, None]), 0.0)
    else:
        rest = row
    rest = torch.where((refused & (rest.sum(1) > 0))[:, None], rest, row)
    total = rest.cumsum(1)
    token = (total <= (s["u_sample"].double() * total[:, -1])[:, None]).sum(1)
    slot = torch.arange(R, device="cuda")
    tokens = torch.cat([d, torch.full((B, 1), -1, device="cuda")], 1)
    tokens = torch.where(slot < taken[:, None], tokens, torch.where(slot == taken[:, None], token[:, None], torch.full_like(tokens, -1)))
    return taken.to(torch.int32), tokens.to(torch.int32)


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"rope": _rope_plain, "attn": _attn_plain, "verify": _verify_plain}[op](s)
    pkg = importlib.import_module("qwen-llm_b200")
    if op == "rope":
        c = s["case"]
        return pkg.qk_norm_rope(s["q"], s["k"], s["pos"], theta=c["theta"], rotary_dim=c["rot"], sections=s["sections"], interleaved=c["interleaved"],
                                q_weight=s["wq"], k_weight=s["wk"], eps=EPS, q_out=s["q_out"], k_out=s["k_cache"], k_rows=s["rows"], v=s["v"], v_out=s["v_cache"])
    if op == "attn":
        return pkg.prefix_attention(s["q"], s["pk"], s["pv"], s["ok"], s["ov"], s["own_len"], q_len=s["q_len"], out=s["out"])
    return pkg.verify_drafts(s["logits"], s["drafts"], s["u_accept"], s["u_sample"], draft_probs=s["probs"], n_draft=s["n_draft"], temperature=s["temperature"])


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "rope":
        n = case["tokens"] * (case["q_heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": n * (size[case["src"]] + size[case["dst"]]) + case["tokens"] * (4 * case["axes"] + 8), "flops": 8.0 * n}
    if case["op"] == "attn":
        B, n, hq, hk, D, P, cap = (case[k] for k in ("batch", "n", "q_heads", "kv_heads", "dim", "prefix", "cap"))
        q_len = (max(1, n // 2) + n) / 2 if case["ragged"] else n     # the mean of what prepare() deals out
        before = (cap - n) / 2                                        # own rows ahead of the block
        rows = B * q_len
        keys = P + before + (q_len + 1) / 2
        return {"bytes": 2.0 * (2 * rows * hq * D + 2 * (P + B * (before + q_len)) * hk * D), "flops": 4.0 * rows * hq * D * keys}
    # a row is needed when every draft ahead of it stands: some seven in ten do, whether the drafter names a token or a distribution
    B, K, V = case["batch"], case["drafts"], case["vocab"]
    drafts = K / 2 if case["ragged"] else K
    rows = min(drafts + 1, (1 - 0.7 ** (drafts + 1)) / 0.3)
    return {"bytes": B * V * (rows * size[case["dtype"]] + (4.0 if case["probs"] else 0.0)), "flops": 6.0 * B * rows * V}


def exact(case, seed):
    s = prepare(case, seed)

    def rope():
        rot, half = case["rot"], case["rot"] // 2
        owner = [-1] * half
        if case["interleaved"]:
            for a in range(case["axes"] - 1, -1, -1):
                for m in range(s["sections"][a]):
                    if a and m * case["axes"] + a < half:
                        owner[m * case["axes"] + a] = a
            owner = [max(a, 0) for a in owner]
        else:
            owner = [a for a, count in enumerate(s["sections"]) for _ in range(count)]
        turn = torch.empty(case["tokens"], half, dtype=torch.float64, device="cuda")
        for j in range(half):
            turn[:, j] = s["pos"][owner[j]].double() * case["theta"] ** (-2.0 * j / rot)
        z = torch.polar(torch.ones_like(turn), turn)[:, None]
        results = []
        for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
            x = x.double()
            x = x / (x.pow(2).sum(-1, keepdim=True) / case["dim"] + EPS).sqrt() * w.double()
            y = torch.complex(x[..., :half].contiguous(), x[..., half:rot].contiguous()) * z
            x[..., :half], x[..., half:rot] = y.real, y.imag
            results.append(x)
        k = torch.zeros(s["k_cache"].shape, dtype=torch.float64, device="cuda")
        v = torch.zeros_like(k)
        k[s["rows"]], v[s["rows"]] = results[1], s["v"].double()
        return results[0], k, v

    def attn():
        q, out = s["q"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        B, n, hq, D = q.shape
        group, P = hq // s["ok"].shape[2], s["pk"].shape[0]
        for b in range(B):
            mine = int(s["own_len"][b])
            rows = n if s["q_len"] is None else int(s["q_len"][b])
            for h in range(hq // group):
                keys = torch.cat([s["pk"][:, h], s["ok"][b, :mine, h]]).double()
                values = torch.cat([s["pv"][:, h], s["ov"][b, :mine, h]]).double()
                for lo in range(0, rows, 256):
                    hi = min(rows, lo + 256)
                    x = torch.einsum("igd,kd->igk", q[b, lo:hi, h * group:(h + 1) * group].double(), keys) / math.sqrt(D)
                    last = P + mine - rows + torch.arange(lo, hi, device="cuda")
                    x = x.masked_fill((torch.arange(P + mine, device="cuda") > last[:, None])[:, None], -math.inf)
                    out[b, lo:hi, h * group:(h + 1) * group] = torch.einsum("igk,kd->igd", torch.softmax(x, -1), values)
        return out

    def verify():
        B, R, V = s["logits"].shape
        counts, tokens = [], torch.full((B, R), -1, dtype=torch.int32)
        for b in range(B):
            temperature, limit = float(s["temperature"][b]), R - 1 if s["n_draft"] is None else int(s["n_draft"][b])

            def distribution(r):
                x = s["logits"][b, r].double()
                if temperature > 0:
                    return torch.softmax(x / temperature, 0)
                p = torch.zeros_like(x)
                p[int((x == x.max()).nonzero()[0])] = 1.0
                return p

            r = 0
            while True:
                p = distribution(r)
                if r == limit:
                    break
                d = int(s["drafts"][b, r])
                q = torch.zeros_like(p)
                if s["probs"] is None:
                    q[d] = 1.0
                else:
                    q = s["probs"][b, r].double()
                if not float(s["u_accept"][b, r]) * float(q[d]) < float(p[d]):
                    rest = torch.relu(p - q)
                    p = rest if float(rest.sum()) > 0 else p
                    break
                tokens[b, r] = d
                r += 1
            upto = torch.cumsum(p, 0)
            tokens[b, r] = int((upto > float(s["u_sample"][b]) * float(upto[-1])).nonzero()[0])
            counts.append(r)
        return torch.tensor(counts, dtype=torch.int32, device="cuda"), tokens.cuda()

    return {"rope": rope, "attn": attn, "verify": verify}[case["op"]]()
