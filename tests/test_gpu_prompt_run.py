"""The prompt operators as a program uses them: prompts go through a small model layer by layer, each step planned on the
GPU, and single tokens follow - through the prompt operators again, and through the decode stack on the same pools."""

import math

import pytest
import torch

import ezops_b200 as ez
from ezops_b200 import _lib
from ezops_b200 import workloads as wl

pytestmark = pytest.mark.gpu
I32 = torch.int32
B, PAGE, MAX_PAGES, PAGES, LAYERS, T_MAX = 3, 64, 8, 20, 2, 320
SH = wl.LayerShape("small", 512, 1024, 8, 2, 64)


class Model:
    def __init__(self, seed=3):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s, std=1.0, mean=0.0: (torch.randn(*s, generator=g) * std + mean).to(torch.bfloat16).cuda()  # noqa: E731
        H, I, D, NKV = SH.hidden, SH.inter, SH.head_dim, SH.num_kv_heads
        self.layers = [dict(K_cache=r(PAGES, NKV, PAGE, D), V_cache=r(PAGES, NKV, PAGE, D), Wqkv=r(SH.q_rows + 2 * SH.kv_rows, H, std=H**-0.5),
                            Wo=r(H, SH.q_rows, std=SH.q_rows**-0.5), Wgu=r(2 * I, H, std=H**-0.5), Wd=r(H, I, std=I**-0.5),
                            input_norm_w=r(H, std=0.1, mean=1.0), post_norm_w=r(H, std=0.1, mean=1.0), q_norm_w=r(D, std=0.1, mean=1.0),
                            k_norm_w=r(D, std=0.1, mean=1.0)) for _ in range(LAYERS)]
        self.cos, self.sin = (t.cuda() for t in wl.rope_tables(MAX_PAGES * PAGE, D))
        kw = dict(backend="cuda")
        self.plan_op = ez.PagedPlanOp(B, T_MAX, MAX_PAGES, PAGE, PAGES, **kw)
        self.norm = ez.RmsNormOp(T_MAX, H, dtype=torch.bfloat16, with_weight=True, **kw)
        self.qkv = ez.LinearOp(T_MAX, SH.q_rows + 2 * SH.kv_rows, H, **kw)
        self.rope = ez.PagedQkNormRopeOp(T_MAX, SH.num_heads, D, MAX_PAGES * PAGE, PAGE, PAGES, num_kv_heads=NKV, **kw)
        self.attn = ez.AttnPromptOp(B, T_MAX, SH.num_heads, D, MAX_PAGES, PAGE, num_kv_heads=NKV, **kw)
        self.o = ez.LinearOp(T_MAX, H, SH.q_rows, residual=True, **kw)
        self.gate_up = ez.LinearOp(T_MAX, I, H, activation="swiglu", **kw)
        self.down = ez.LinearOp(T_MAX, H, I, residual=True, **kw)
        self.table = torch.full((B, MAX_PAGES), -1, dtype=I32, device="cuda")
        self.free = torch.randperm(PAGES, generator=g).to(I32).cuda()
        self.count = torch.tensor([PAGES], dtype=I32, device="cuda")
        self.ctx = torch.zeros(B, dtype=I32, device="cuda")
        self.new = torch.zeros(B, dtype=I32, device="cuda")
        self.plan = self.plan_op.new_plan("cuda")
        self.heads = torch.zeros(T_MAX, SH.num_heads, D, dtype=torch.bfloat16, device="cuda")

    def step(self, x):
        """One step of T_MAX token slots; ``new`` says how many of them each request uses."""
        p = self.plan_op(self.ctx, self.new, self.table, self.free, self.count, out=self.plan)
        xn = torch.empty_like(x)
        x = x.clone()
        for L in self.layers:
            self.norm(x, L["input_norm_w"], xn)
            q = self.rope(self.qkv(xn, L["Wqkv"]), L["q_norm_w"], L["k_norm_w"], self.cos, self.sin, p.positions, p.slots, L["K_cache"],
                          L["V_cache"], out=self.heads)
            a = self.attn(q, L["K_cache"], L["V_cache"], self.table, p.seq_lens, p.cu_tokens, out=torch.zeros_like(q))
            self.o(a.view(T_MAX, -1), L["Wo"], residual=x, out=x)
            self.norm(x, L["post_norm_w"], xn)
            self.down(self.gate_up(xn, L["Wgu"]), L["Wd"], residual=x, out=x)
        self.ctx.copy_(p.seq_lens)
        self.count.copy_(p.free_count)
        return x


def whole_sequences64(model, sequences):
    """The model over whole sequences in 64 bits, no caches."""
    D, NKV, I = SH.head_dim, SH.num_kv_heads, SH.inter
    norm = lambda x, w: x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()  # noqa: E731
    out = []
    for x in sequences:
        x = x.double()
        n = x.shape[0]
        c, s = model.cos[:n].double()[:, None], model.sin[:n].double()[:, None]
        turn = lambda h: h * c + torch.cat([-h[..., D // 2 :], h[..., : D // 2]], -1) * s  # noqa: E731
        for L in model.layers:
            q, k, v = (norm(x, L["input_norm_w"]) @ L["Wqkv"].double().T).split([SH.q_rows, SH.kv_rows, SH.kv_rows], -1)
            q, k = turn(norm(q.reshape(n, -1, D), L["q_norm_w"])), turn(norm(k.reshape(n, -1, D), L["k_norm_w"]))
            k, v = (t.reshape(n, NKV, D).repeat_interleave(SH.num_heads // NKV, 1) for t in (k, v))
            scores = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(D)
            scores = scores.masked_fill(torch.ones(n, n, device="cuda", dtype=torch.bool).triu(1), float("-inf"))
            x = x + torch.einsum("hij,jhd->ihd", scores.softmax(-1), v).reshape(n, -1) @ L["Wo"].double().T
            g = norm(x, L["post_norm_w"]) @ L["Wgu"].double().T
            x = x + (torch.nn.functional.silu(g[:, :I]) * g[:, I:]) @ L["Wd"].double().T
        out.append(x)
    return out


def rel(a, e):
    return ((a.double() - e).norm() / e.norm()).item()


def test_prompts_in_pieces_then_single_tokens(cuda_device):
    _lib.device_status()
    model = Model()
    torch.manual_seed(0)
    lengths = [200, 70, 131]
    sequences = [torch.randn(n, SH.hidden, device="cuda").to(torch.bfloat16) for n in lengths]
    expected = whole_sequences64(model, sequences)
    got = [[] for _ in range(B)]
    done = [0] * B

    def feed(new, run):
        x = torch.full((T_MAX, SH.hidden), 0.5, device="cuda", dtype=torch.bfloat16)
        at = 0
        for b, n in enumerate(new):
            x[at : at + n] = sequences[b][done[b] : done[b] + n]
            at += n
        model.new.copy_(torch.tensor(new, dtype=I32))
        y, at = run(x), 0
        for b, n in enumerate(new):
            got[b].append(y[at : at + n])
            at += n
            done[b] += n

    for new in ([150, 0, 129], [1, 65, 1], [47, 1, 0]):
        feed(new, model.step)

    # single tokens from a captured graph: the plan, the pools and the lengths move on by themselves
    static = torch.zeros(T_MAX, SH.hidden, device="cuda", dtype=torch.bfloat16)
    model.new.zero_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        model.step(static)  # warm-up: a step without tokens changes nothing
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = model.step(static)

    def replay(x):
        static.copy_(x)
        graph.replay()
        return result.clone()

    for new in ([1, 1, 0], [1, 0, 1]):
        feed(new, replay)
    assert done == [200, 67, 131]

    # and the decode stack takes over on the same pools and table
    stack = ez.get_kernel("qwen3_decode_stack", "cuda")(B, MAX_PAGES * PAGE, SH.hidden, SH.inter, SH.num_heads, SH.head_dim, LAYERS,
                                                        num_kv_heads=SH.num_kv_heads)
    sequences[0] = torch.cat([sequences[0], torch.randn(3, SH.hidden, device="cuda").to(torch.bfloat16)])
    sequences[2] = torch.cat([sequences[2], torch.randn(3, SH.hidden, device="cuda").to(torch.bfloat16)])
    expected = whole_sequences64(model, sequences)
    for _ in range(3):
        model.new.fill_(1)
        p = model.plan_op(model.ctx, model.new, model.table, model.free, model.count, out=model.plan)
        x = torch.stack([sequences[b][done[b]] for b in range(B)])
        y = stack(x, model.layers, model.cos, model.sin, seq_lens=p.seq_lens, page_table=model.table, page_size=PAGE)
        model.ctx.copy_(p.seq_lens)
        model.count.copy_(p.free_count)
        for b in range(B):
            got[b].append(y[b : b + 1])
            done[b] += 1
    assert _lib.device_status() == 0
    used = sum(-(-n // PAGE) for n in done)
    assert int(model.count) == PAGES - used
    taken = model.table[model.table >= 0]
    assert taken.numel() == used == taken.unique().numel()
    for b in range(B):
        # the layer operators' own bound: 1e-2 relative error per layer, growing with the square root of their number
        y = torch.cat(got[b])
        assert rel(y, expected[b]) < 1e-2 * math.sqrt(LAYERS)
        worst = ((y.double() - expected[b]).norm(dim=-1) / expected[b].norm(dim=-1)).max().item()
        assert worst < 2e-2 * math.sqrt(LAYERS)


def test_images_in_pieces_then_single_tokens(cuda_device):
    """Requests with an image in them: positions of three axes, which the program brings and which run behind the place in the cache
    from the image on, first in pieces, then token by token through the same operators."""
    _lib.device_status()
    sections = (12, 10, 10)
    model = Model()
    model.rope = ez.PagedQkNormRopeOp(T_MAX, SH.num_heads, SH.head_dim, MAX_PAGES * PAGE, PAGE, PAGES, num_kv_heads=SH.num_kv_heads,
                                      sections=sections, interleaved=True, backend="cuda")
    torch.manual_seed(1)
    lengths, positions = [180, 70, 131], []
    for n, (at, rows, columns) in zip(lengths, ((20, 6, 8), (0, 4, 4), (50, 2, 30))):  # text, an image of so many patches, text
        text = torch.arange(at).expand(3, -1)
        image = at + torch.stack([torch.zeros(rows * columns, dtype=torch.int64), torch.arange(rows).repeat_interleave(columns),
                                  torch.arange(columns).repeat(rows)])
        rest = at + max(rows, columns) + torch.arange(n - at - rows * columns)
        positions.append(torch.cat([text, image, rest.expand(3, -1)], 1))
        assert positions[-1].shape == (3, n) and int(positions[-1][:, -1].max()) < n - 1
    sequences = [torch.randn(n, SH.hidden, device="cuda").to(torch.bfloat16) for n in lengths]
    got, done = [[] for _ in range(B)], [0] * B
    for new in ([100, 0, 60], [79, 66, 68], [1, 1, 1], [0, 2, 1], [0, 1, 1]):
        x = torch.zeros(T_MAX, SH.hidden, device="cuda", dtype=torch.bfloat16)
        where = torch.full((3, T_MAX), -1, dtype=I32)
        at = 0
        for b, n in enumerate(new):
            x[at : at + n], where[:, at : at + n] = sequences[b][done[b] : done[b] + n], positions[b][:, done[b] : done[b] + n]
            at += n
        where = where.cuda()
        model.new.copy_(torch.tensor(new, dtype=I32))
        rope = model.rope
        model.rope = lambda qkv, qw, kw, cos, sin, _, *rest, where=where, **kw2: rope(qkv, qw, kw, cos, sin, where, *rest, **kw2)
        y, at = model.step(x), 0
        model.rope = rope
        for b, n in enumerate(new):
            got[b].append(y[at : at + n])
            at += n
            done[b] += n
    assert done == lengths and _lib.device_status() == 0
    axis = torch.tensor([i % 3 if i // 3 < sections[i % 3] else 0 for i in range(SH.head_dim // 2)] * 2)
    for b in range(B):
        at = positions[b][axis].T.cuda()  # [tokens, D]
        column = torch.arange(SH.head_dim, device="cuda")
        tables = Model.__new__(Model)
        tables.layers, tables.cos, tables.sin = model.layers, model.cos[at, column], model.sin[at, column]
        (expected,) = whole_sequences64(tables, sequences[b : b + 1])
        assert rel(torch.cat(got[b]), expected) < 1e-2 * math.sqrt(LAYERS)
