"""Operators that take prompts, not only single new tokens, through a Qwen3 dense model over paged KV caches: the plan of a
step (page tables and slots from request lengths), the linear layers with their epilogues, head norm with rotary
positions of one or several axes and the write into the page pools, and causal attention of ragged rows over the pools.

A case is a dict of plain values; ``op`` picks the operator, the rest are its sizes:

``plan``    ``PagedPlanOp``        B requests, T token slots, ``fill``: share of T that the step uses
``rope``    ``PagedQkNormRopeOp``  T tokens (``pad`` of them behind the last one), A axes, chunked or interleaved sections
``linear``  ``LinearOp``           act(X[M, K] W[N, K]^T + bias) + residual
``attn``    ``AttnPromptOp``       B rows with q_lo..q_hi new tokens on c_lo..c_hi cached ones

Where ``own`` is true, ``run`` calls the framework; otherwise it computes the same in elementary torch operations in
32 bits, rounded once at the end.
"""

from __future__ import annotations

import torch

own = False

BF16 = torch.bfloat16
EPS = 1e-6
MOST_FLOPS, MOST_BYTES, MOST_SCORES = 8.2e11, 6.1e8, 2.2e9  # drawn cases stay inside what the largest listed ones need


def listed():
    return [
        # Every decode step of a batch of 32: one new token each, a page now and then. Launch latency.
        dict(name="plan_decode_b32", op="plan", B=32, T=32, fill=1.0, max_pages=128, page=64, c_lo=0, c_hi=8100),
        # A full server's step: 512 requests, prompts in pieces between single tokens, 16384 token slots.
        dict(name="plan_mixed_b512", op="plan", B=512, T=16384, fill=0.9, max_pages=128, page=64, c_lo=0, c_hi=6000),
        # A step of 32 single tokens at 32 different positions, 8B heads. Launch latency.
        dict(name="rope_tokens_32", op="rope", T=32, pad=0, H=32, NKV=8, D=128, S=8192, page=256, axes=1, interleaved=False),
        # A prompt with images: time, height and width positions in the interleaved order, 2B heads, a padded tail.
        dict(name="rope_images_8189", op="rope", T=8189, pad=61, H=16, NKV=8, D=128, S=8192, page=128, axes=3, interleaved=True),
        # The q/k/v projection of an odd handful of tokens, with a bias: one pass over the weight.
        dict(name="linear_qkv_17", op="linear", M=17, N=6144, K=4096, act=None, bias=True, residual=False, out="bf16"),
        # Scores over the vocabulary for a batch, kept in 32 bits.
        dict(name="linear_vocab_64", op="linear", M=64, N=151936, K=1024, act=None, bias=False, residual=False, out="fp32"),
        # The down projection of a short prompt with the residual stream added.
        dict(name="linear_down_777", op="linear", M=777, N=4096, K=12288, act=None, bias=False, residual=True, out="bf16"),
        # Gate and up projections of a long prompt with SwiGLU: the largest product of a layer.
        dict(name="linear_gate_up_4096", op="linear", M=4096, N=12288, K=4096, act="swiglu", bias=False, residual=False, out="bf16"),
        # A whole prompt of one user, 8B heads.
        dict(name="attn_prompt_8192", op="attn", B=1, H=32, NKV=8, D=128, q_lo=8192, q_hi=8192, c_lo=0, c_hi=0, page=256),
        # Prompts worked off in pieces: new tokens behind contexts of different lengths.
        dict(name="attn_pieces_b8", op="attn", B=8, H=32, NKV=8, D=128, q_lo=65, q_hi=600, c_lo=300, c_hi=7400, page=128),
        # Single tokens of 32 users over long caches, the form that serving takes between prompts.
        dict(name="attn_tokens_b32", op="attn", B=32, H=32, NKV=8, D=128, q_lo=1, q_hi=1, c_lo=1000, c_hi=8100, page=64),
        # Short prompts with small heads and an odd group of query heads per kv head.
        dict(name="attn_short_d64", op="attn", B=5, H=14, NKV=2, D=64, q_lo=33, q_hi=300, c_lo=0, c_hi=0, page=64),
    ]


def _log_int(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    while True:
        case = _draw_any(rng)
        w = work(case)
        if w["flops"] > MOST_FLOPS or w["bytes"] > MOST_BYTES:
            continue
        if case["op"] == "attn" and case["B"] * case["H"] * case["q_hi"] * (case["q_hi"] + case["c_hi"]) > MOST_SCORES:
            continue
        return case


def _draw_any(rng):
    op = rng.choice(["plan", "rope", "linear", "linear", "attn", "attn"])
    H, NKV = rng.choice([(32, 8), (16, 8), (64, 8), (14, 2), (8, 8), (6, 2), (32, 1)])
    page = rng.choice([64, 128, 256])
    D = rng.choice([64, 128])
    if op == "plan":
        B = _log_int(rng, 1, 1024)
        c_hi = _log_int(rng, 1, 8192)
        T = _log_int(rng, B, 32768)
        room = c_hi + T  # a row may take the whole step
        return dict(op=op, B=B, T=T, fill=rng.choice([0.5, 0.9, 1.0]), max_pages=-(-room // page), page=page, c_lo=0, c_hi=c_hi)
    if op == "rope":
        T = _log_int(rng, 1, 12000)
        return dict(op=op, T=T, pad=rng.choice([0, T // 7]), H=H, NKV=NKV, D=D, S=_log_int(rng, 64, 16384), page=page,
                    axes=rng.choice([1, 2, 3]), interleaved=rng.random() < 0.5)
    if op == "linear":
        act = rng.choice([None, None, "swiglu", "silu", "gelu", "relu"])
        return dict(op=op, M=_log_int(rng, 1, 8192), N=_log_int(rng, 32, 26000), K=8 * _log_int(rng, 8, 1600), act=act,
                    bias=rng.random() < 0.4, residual=rng.random() < 0.4, out=rng.choice(["bf16", "bf16", "fp32"]))
    q_hi, c_hi = _log_int(rng, 1, 8192), rng.choice([0, _log_int(rng, 1, 16384)])
    return dict(op=op, B=_log_int(rng, 1, 48), H=H, NKV=NKV, D=D, q_lo=max(1, q_hi // rng.choice([1, 3, 40])), q_hi=q_hi,
                c_lo=c_hi // rng.choice([1, 7]), c_hi=c_hi, page=page)


# ------------------------------------------------------------------- inputs ---
def _spread(lo, hi, n):
    """n lengths between lo and hi, in no order: a property of the case, not of the seed."""
    return [lo + int((hi - lo) * ((i * 0.6180339887 + 0.999) % 1.0) + 0.5) for i in range(n)]


def _normal(g, *shape, std=1.0, mean=0.0, dtype=BF16):
    t = torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
    if std != 1.0:
        t.mul_(std)
    if mean:
        t.add_(mean)
    return t


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sections(case):
    """Rotary frequencies per axis: all of them, halves, or 3/8, 5/16 and 5/16."""
    half = case["D"] // 2
    return {1: (half,), 2: (half // 2, half // 2), 3: (half - 2 * (half * 5 // 16), half * 5 // 16, half * 5 // 16)}[case["axes"]]


def _axis_of_frequency(case):
    sections, half, axes = _sections(case), case["D"] // 2, case["axes"]
    if case["interleaved"]:
        return [i % axes if i // axes < sections[i % axes] else 0 for i in range(half)]
    return [a for a, n in enumerate(sections) for _ in range(n)]


def _tables(S, D):
    inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D))
    ang = torch.arange(S, dtype=torch.float64, device="cuda")[:, None] * inv
    return (torch.cat([f(ang)] * 2, -1).to(BF16) for f in (torch.cos, torch.sin))


def _plan_lengths(case, seed):
    """Cached and new tokens of each request; the step's tokens are dealt out at random, one each at least where they suffice."""
    B, used = case["B"], max(1, int(case["T"] * case["fill"]))
    g = torch.Generator().manual_seed(seed)
    cached = torch.randint(case["c_lo"], case["c_hi"] + 1, (B,), generator=g)
    new = torch.bincount(torch.randint(0, B, (max(0, used - B),), generator=g), minlength=B) + (torch.arange(B) < used).long()
    return cached, new


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    op = case["op"]
    s = dict(case=case, op=op)
    if op == "plan":
        B, page, wide = case["B"], case["page"], case["max_pages"]
        cached, new = _plan_lengths(case, seed)
        held = (cached + page - 1) // page
        spare = int(((cached + new + page - 1) // page - held).sum()) + 17
        pages = int(held.sum()) + spare
        order = torch.randperm(pages, generator=cpu).to(torch.int32)
        table = torch.full((B, wide), -1, dtype=torch.int32)
        table[torch.arange(wide) < held[:, None]] = order[: pages - spare]
        free = torch.full((pages,), -1, dtype=torch.int32)
        free[:spare] = order[pages - spare :]
        s.update(ctx=cached.to(torch.int32).cuda(), new=new.to(torch.int32).cuda(), table=table.cuda(), free=free.cuda(),
                 count=_ints([spare]), pages=pages)
        if own:
            import ezops_b200 as ez

            s["fn"] = ez.PagedPlanOp(B, case["T"], wide, page, pages, backend="cuda")
            s["plan"] = s["fn"].new_plan("cuda")
    elif op == "rope":
        T, H, NKV, D, S, page = (case[k] for k in ("T", "H", "NKV", "D", "S", "page"))
        n = T - case["pad"]
        pages = -(-n // page) + 2
        positions = torch.full((case["axes"], T), -1, dtype=torch.int32)
        positions[:, :n] = torch.randint(0, S, (case["axes"], n), generator=cpu)
        slots = torch.full((T,), -1, dtype=torch.int32)
        slots[:n] = torch.randperm(pages * page, generator=cpu)[:n]
        cos, sin = _tables(S, D)
        s.update(n=n, axis=torch.tensor(_axis_of_frequency(case), device="cuda"), positions=positions.cuda(), slots=slots.cuda(),
                 qkv=_normal(g, T, (H + 2 * NKV) * D), qw=_normal(g, D, std=0.1, mean=1.0), kw=_normal(g, D, std=0.1, mean=1.0),
                 cos=cos, sin=sin, K=_normal(g, pages, NKV, page, D), V=_normal(g, pages, NKV, page, D),
                 out=torch.zeros(T, H, D, device="cuda", dtype=BF16))
        if own:
            import ezops_b200 as ez

            s["fn"] = ez.PagedQkNormRopeOp(T, H, D, S, page, pages, backend="cuda", num_kv_heads=NKV, sections=_sections(case),
                                           interleaved=case["interleaved"])
    elif op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        s.update(x=_normal(g, M, K), w=_normal(g, N * (2 if case["act"] == "swiglu" else 1), K, std=0.02),
                 bias=_normal(g, N * (2 if case["act"] == "swiglu" else 1), std=0.5) if case["bias"] else None,
                 residual=_normal(g, M, N) if case["residual"] else None,
                 out=torch.empty(M, N, device="cuda", dtype=BF16 if case["out"] == "bf16" else torch.float32))
        if own:
            import ezops_b200 as ez

            s["fn"] = ez.LinearOp(M, N, K, backend="cuda", bias=case["bias"], activation=case["act"], residual=case["residual"],
                                  out_dtype=s["out"].dtype)
    else:
        B, H, NKV, D, page = (case[k] for k in ("B", "H", "NKV", "D", "page"))
        q, c = _spread(case["q_lo"], case["q_hi"], B), _spread(case["c_lo"], case["c_hi"], B)
        wide = max(-(-(a + b) // page) for a, b in zip(q, c))
        used = [-(-(a + b) // page) for a, b in zip(q, c)]
        pages = sum(used) + 1
        order = torch.randperm(pages, generator=cpu)
        table = torch.full((B, wide), -1, dtype=torch.int32)
        table[torch.arange(wide) < torch.tensor(used)[:, None]] = order[: pages - 1].to(torch.int32)
        T = sum(q)
        s.update(q=_normal(g, T, H, D), K=_normal(g, pages, NKV, page, D), V=_normal(g, pages, NKV, page, D), table=table.cuda(),
                 lens=_ints([a + b for a, b in zip(q, c)]), cu=_ints([sum(q[:i]) for i in range(B + 1)]), q_max=max(q),
                 out=torch.empty(T, H, D, device="cuda", dtype=BF16))
        if own:
            import ezops_b200 as ez

            s["fn"] = ez.AttnPromptOp(B, T, H, D, wide, page, backend="cuda", num_kv_heads=NKV)
    return s


# --------------------------------------------------------------------- pass ---
def run(state):
    if state["op"] == "plan":
        return _run_plan(state)
    if state["op"] == "rope":
        return _run_rope(state)
    if state["op"] == "linear":
        return _run_linear(state)
    return _run_attn(state)


def _run_plan(s):
    if own:
        p = s["fn"](s["ctx"], s["new"], s["table"], s["free"], s["count"], out=s["plan"])
        return p.seq_lens, p.cu_tokens, p.positions, p.slots, p.free_count, s["table"]
    c = s["case"]
    T, page, table = c["T"], c["page"], s["table"]
    cap = c["max_pages"] * page
    ctx = s["ctx"].long().clamp(0, cap)
    cu = torch.nn.functional.pad(s["new"].long().clamp(min=0).cumsum(0).clamp(max=T), (1, 0))
    lens = (ctx + cu.diff()).clamp(max=cap)
    held, need = (ctx + page - 1) // page, (lens + page - 1) // page
    taken = (need - held).cumsum(0)
    j = torch.arange(c["max_pages"], device="cuda")
    at = s["count"].long() - 1 - ((taken - need)[:, None] + j)  # the k-th new page of the step is free[count - 1 - k]
    ids = torch.where(at >= 0, s["free"][at.clamp(0, s["free"].numel() - 1)], -1)
    ids = torch.where((ids >= 0) & (ids < s["pages"]), ids, -1)
    table.copy_(torch.where((j >= held[:, None]) & (j < need[:, None]), ids, table))
    t = torch.arange(T, device="cuda")
    real = t < cu[-1]
    row = torch.searchsorted(cu[1:], t, right=True).clamp(max=c["B"] - 1)
    pos = ctx[row] + t - cu[row]
    ids = table[row, (pos // page).clamp(0, c["max_pages"] - 1)].long()
    slots = torch.where(real & (pos < cap) & (ids >= 0) & (ids < s["pages"]), ids * page + pos % page, -1)
    positions = torch.where(real, pos, -1)
    return lens.int(), cu.int(), positions.int(), slots.int(), (s["count"] - taken[-1]).int(), table


def _run_rope(s):
    if own:
        return s["fn"](s["qkv"], s["qw"], s["kw"], s["cos"], s["sin"], s["positions"], s["slots"], s["K"], s["V"], out=s["out"]), s["K"], s["V"]
    c, n = s["case"], s["n"]
    H, NKV, D, page = c["H"], c["NKV"], c["D"], c["page"]
    x = s["qkv"][:n].float().view(n, H + 2 * NKV, D)
    i = torch.arange(D // 2, device="cuda")
    at = s["positions"][s["axis"], :n].T.long()
    cos, sin = s["cos"][at, i].float()[:, None], s["sin"][at, i].float()[:, None]

    def head(x, w):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = x[..., : D // 2], x[..., D // 2 :]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(BF16)

    s["out"][:n] = head(x[:, :H], s["qw"])
    slot = s["slots"][:n].long()
    s["K"][slot // page, :, slot % page] = head(x[:, H : H + NKV], s["kw"])
    s["V"][slot // page, :, slot % page] = x[:, H + NKV :].to(BF16)
    return s["out"], s["K"], s["V"]


def _run_linear(s):
    if own:
        return s["fn"](s["x"], s["w"], bias=s["bias"], residual=s["residual"], out=s["out"])
    act = s["case"]["act"]
    z = s["x"].float() @ s["w"].float().T
    if s["bias"] is not None:
        z = z + s["bias"].float()
    if act == "swiglu":
        gate, up = z[:, : s["case"]["N"]], z[:, s["case"]["N"] :]
        z = gate / (1 + torch.exp(-gate)) * up
    elif act == "silu":
        z = z / (1 + torch.exp(-z))
    elif act == "gelu":
        z = 0.5 * z * torch.erfc(z * -(0.5**0.5))
    elif act == "relu":
        z = torch.where(z > 0, z, 0)
    if s["residual"] is not None:
        z = z + s["residual"].float()
    return z.to(s["out"].dtype)


def _run_attn(s):
    if own:
        return s["fn"](s["q"], s["K"], s["V"], s["table"], s["lens"], s["cu"], out=s["out"])
    c = s["case"]
    B, H, NKV, D = (c[k] for k in ("B", "H", "NKV", "D"))
    T, G, most = s["q"].shape[0], H // NKV, s["q_max"]
    # rows of queries [B, most, ...], rows of keys [B, pages, NKV, page, D] -> [B, NKV, keys, D]
    cu, lens = s["cu"].long(), s["lens"].long()
    i = torch.arange(most, device="cuda")
    token = (cu[:-1, None] + i).clamp(max=T - 1)
    q = s["q"][token].float().view(B, most, NKV, G, D).permute(0, 2, 3, 1, 4).reshape(B, NKV, G * most, D)
    pages = s["table"].long().clamp(min=0)
    k, v = (t[pages].float().transpose(1, 2).reshape(B, NKV, -1, D) for t in (s["K"], s["V"]))
    j = torch.arange(k.shape[2], device="cuda")
    v = torch.where((j < lens[:, None])[:, None, :, None], v, 0)
    scores = (q @ k.transpose(-1, -2)).mul_(D**-0.5).view(B, NKV, G, most, -1)
    seen = j <= (lens - cu.diff())[:, None, None] + i[:, None]  # [B, most, keys]
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, NKV, G * most, -1) @ v).view(B, NKV, G, most, D) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(B, most, H, D)
    t = torch.arange(T, device="cuda")
    row = torch.searchsorted(cu[1:], t, right=True)
    return o[row, t - cu[row]].to(BF16)


# --------------------------------------------------------------------- cost ---
def work(case):
    """Every input read once, every output written once: two bytes an element, four for indices and 32-bit results."""
    op = case["op"]
    if op == "plan":
        B, T = case["B"], case["T"]
        fresh = max(1, int(T * case["fill"])) // case["page"]
        # lengths in; lengths, offsets, positions and slots out; new pages from the free list into the table
        return dict(bytes=4 * (4 * B + 2 * T + 2 * fresh), flops=4 * T)
    if op == "rope":
        n, H, NKV, D = case["T"] - case["pad"], case["H"], case["NKV"], case["D"]
        rows = min(case["S"], n)
        return dict(bytes=2 * n * D * 2 * (H + 2 * NKV) + 4 * rows * D + 4 * D + 4 * n * (1 + case["axes"]), flops=10 * n * (H + NKV) * D)
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        rows = N * (2 if case["act"] == "swiglu" else 1)
        extra = (rows if case["bias"] else 0) + (M * N if case["residual"] else 0)
        return dict(bytes=2 * (M * K + rows * K + extra) + M * N * (2 if case["out"] == "bf16" else 4), flops=2 * M * rows * K)
    B, H, NKV, D = (case[k] for k in ("B", "H", "NKV", "D"))
    q, c = _spread(case["q_lo"], case["q_hi"], B), _spread(case["c_lo"], case["c_hi"], B)
    pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(q, c))
    return dict(bytes=2 * D * (2 * H * sum(q) + 2 * NKV * (sum(q) + sum(c))), flops=4 * H * D * pairs)


# -------------------------------------------------------------------- exact ---
def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits; the plan's whole numbers request by request."""
    s = prepare(case, seed)
    if case["op"] == "plan":
        return _exact_plan(case, s)
    if case["op"] == "rope":
        return _exact_rope(case, s)
    if case["op"] == "linear":
        z = s["x"].double() @ s["w"].double().T
        if case["bias"]:
            z += s["bias"].double()
        F = torch.nn.functional
        acts = {None: lambda z: z, "silu": F.silu, "gelu": F.gelu, "relu": F.relu,
                "swiglu": lambda z: F.silu(z[:, : case["N"]]) * z[:, case["N"] :]}
        y = acts[case["act"]](z)
        return y + s["residual"].double() if case["residual"] else y
    return _exact_attn(case, s)


def _exact_plan(case, s):
    page, T = case["page"], case["T"]
    ctx, new, table = s["ctx"].tolist(), s["new"].tolist(), s["table"].cpu()
    free = s["free"].tolist()[: int(s["count"])]
    lens, cu, positions, slots = [], [0], [], []
    for b, (a, n) in enumerate(zip(ctx, new)):
        n = min(n, T - cu[-1])
        cu.append(cu[-1] + n)
        lens.append(a + n)
        for j in range(-(-a // page), -(-(a + n) // page)):
            table[b, j] = free.pop()
        at = torch.arange(a, a + n)
        positions.append(at)
        slots.append(table[b, at // page].long() * page + at % page)
    tail = [torch.full((T - cu[-1],), -1)]
    out = (_ints(lens), _ints(cu), torch.cat(positions + tail), torch.cat(slots + tail), _ints([len(free)]), table)
    return tuple(t.to(torch.int32).cuda() for t in out)


def _exact_rope(case, s):
    n, H, NKV, D, page = s["n"], case["H"], case["NKV"], case["D"], case["page"]
    parts = s["qkv"][:n].double().split([H * D, NKV * D, NKV * D], 1)
    q, k, v = (t.reshape(n, -1, D) for t in parts)
    cos, sin = torch.empty(n, D, device="cuda", dtype=torch.float64), torch.empty(n, D, device="cuda", dtype=torch.float64)
    for i, axis in enumerate(_axis_of_frequency(case) * 2):  # both halves of a head have the same frequencies
        at = s["positions"][axis, :n].long()
        cos[:, i], sin[:, i] = s["cos"][at, i].double(), s["sin"][at, i].double()

    def turned(x, w):
        x = w.double() * x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
        a, b = x.chunk(2, -1)
        return x * cos[:, None] + torch.cat([-b, a], -1) * sin[:, None]

    out, K, V = s["out"].double(), s["K"].double(), s["V"].double()
    out[:n] = turned(q, s["qw"])
    slot = s["slots"][:n].long()
    at = (slot // page, slice(None), slot % page)
    K[at], V[at] = turned(k, s["kw"]), v
    return out, K, V


def _exact_attn(case, s):
    NKV, D, page = case["NKV"], case["D"], case["page"]
    cu, lens = s["cu"].tolist(), s["lens"].tolist()
    rows = []
    for b, n in enumerate(lens):
        m = cu[b + 1] - cu[b]
        at = s["table"][b, : -(-n // page)].long()
        k, v = (t[at].double().transpose(0, 1).reshape(NKV, -1, D)[:, :n] for t in (s["K"], s["V"]))
        q = s["q"][cu[b] : cu[b + 1]].double().view(m, NKV, -1, D)
        later = torch.ones(m, n, dtype=torch.bool, device="cuda").triu(n - m + 1)
        heads = []
        for h in range(NKV):
            group = []
            for x in q[:, h].unbind(1):
                group.append((x @ k[h].T / D**0.5).masked_fill_(later, float("-inf")).softmax(-1) @ v[h])
            heads.append(torch.stack(group, 1))
        rows.append(torch.stack(heads, 1).reshape(m, -1, D))
    return torch.cat(rows)
