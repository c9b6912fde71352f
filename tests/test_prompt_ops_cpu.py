"""Host-side behaviour of the prompt operators: registry, constructors, the torch references against plain 64-bit loops, and
the refusals of the C entries (which come before anything touches CUDA)."""

import ctypes

import pytest
import torch

import ezops_b200 as ez
from ezops_b200 import _lib
from ezops_b200.ops.paged_qk_norm_rope import axis_of_frequency

I32 = torch.int32


def test_registry_family():
    assert ez.list_ops("prompt") == ["attn_prompt", "linear", "paged_plan", "paged_qk_norm_rope"]
    assert "linear" not in ez.list_ops()
    for op in ez.list_ops("prompt"):
        assert ez.list_backends(op) == ["cuda"]
        assert ez.get_kernel(op, "cuda").op_name == op


@pytest.mark.parametrize("make,match", [
    (lambda: ez.PagedPlanOp(0, 1, 1, 64, 1), "batch"),
    (lambda: ez.PagedPlanOp(1, 1, 1, 96, 1), "page_size"),
    (lambda: ez.PagedPlanOp(9000, 1, 1, 64, 1, backend="cuda"), "8192"),
    (lambda: ez.PagedQkNormRopeOp(1, 8, 96, 10, 64, 1), "head_dim"),
    (lambda: ez.PagedQkNormRopeOp(1, 8, 128, 10, 64, 1, num_kv_heads=3), "divisible"),
    (lambda: ez.PagedQkNormRopeOp(1, 8, 128, 10, 64, 1, sections=(24, 20)), "sections"),
    (lambda: ez.PagedQkNormRopeOp(1, 8, 128, 10, 64, 1, sections=(16, 16, 16, 16)), "sections"),
    (lambda: ez.PagedQkNormRopeOp(1, 8, 128, 10, 64, 1, sections=(4, 30, 30), interleaved=True), "interleaved"),
    (lambda: ez.LinearOp(4, 8, 12), "divisible by 8"),
    (lambda: ez.LinearOp(4, 8, 16, activation="tanh"), "activation"),
    (lambda: ez.LinearOp(4, 8, 16, out_dtype=torch.float16), "out_dtype"),
    (lambda: ez.AttnPromptOp(1, 1, 8, 80, 1, 64), "head_dim"),
    (lambda: ez.AttnPromptOp(1, 1, 8, 64, 1, 32), "page_size"),
    (lambda: ez.AttnPromptOp(1, 1, 129, 64, 1, 64, num_kv_heads=1), "128 query heads"),
])
def test_constructors_refuse(make, match):
    with pytest.raises(ValueError, match=match):
        make()


def test_linear_wants_what_it_was_made_for():
    op = ez.LinearOp(2, 8, 16, bias=True)
    X, W, b, _ = op.gen_data("cpu")
    with pytest.raises(ValueError, match="with a bias"):
        op(X, W)
    with pytest.raises(ValueError, match="without a residual"):
        op(X, W, bias=b, residual=X)


def test_cuda_backends_refuse_host_tensors():
    for op in (ez.LinearOp(2, 8, 16, backend="cuda"), ez.AttnPromptOp(2, 5, 8, 64, 3, 64, backend="cuda"),
               ez.PagedQkNormRopeOp(5, 8, 64, 10, 64, 2, backend="cuda"), ez.PagedPlanOp(2, 8, 4, 64, 8, backend="cuda")):
        data = op.gen_data("cpu")
        with pytest.raises(ValueError, match="CUDA"):
            op(*(t for t in data if t is not None))


def test_axis_of_frequency():
    assert axis_of_frequency((4,), False) == [0] * 4
    assert axis_of_frequency((2, 1, 1), False) == [0, 0, 1, 2]
    assert axis_of_frequency((4, 2, 2), True) == [0, 1, 2, 0, 1, 2, 0, 0]
    assert axis_of_frequency((2, 2), True) == [0, 1, 0, 1]


def test_plan_reference():
    op = ez.PagedPlanOp(3, 10, 3, 64, 6)
    ctx, new, table = torch.tensor([63, 0, 64]), torch.tensor([3, 0, 2]), torch.tensor([[4, -1, -1], [-1] * 3, [2, -1, -1]])
    free, count = torch.tensor([5, 0, 1, -1, -1, -1]), torch.tensor([3])
    args = [t.to(I32) for t in (ctx, new, table, free, count)]
    p = op(*args)
    assert args[2].tolist() == [[4, 1, -1], [-1, -1, -1], [2, 0, -1]]
    assert p.seq_lens.tolist() == [66, 0, 66] and p.cu_tokens.tolist() == [0, 3, 3, 5]
    assert p.positions.tolist() == [63, 64, 65, 64, 65] + [-1] * 5
    assert p.slots.tolist() == [4 * 64 + 63, 64, 65, 0, 1] + [-1] * 5
    assert p.free_count.tolist() == [1]
    # one page short: its entry and slots are -1
    args[2] = torch.tensor([[4, -1, -1], [-1] * 3, [2, -1, -1]], dtype=I32)
    args[4] = torch.tensor([1], dtype=I32)
    p = op(*args)
    assert p.free_count.tolist() == [-1] and args[2].tolist() == [[4, 5, -1], [-1] * 3, [2, -1, -1]]
    assert p.slots.tolist()[3:5] == [-1, -1]


def test_rope_reference_token_by_token():
    op = ez.PagedQkNormRopeOp(6, 4, 64, 50, 64, 2, num_kv_heads=2, sections=(12, 10, 10), interleaved=True)
    qkv, qw, kw, cos, sin, positions, slots, K, V = op.gen_data("cpu")
    positions[:, 2] = -1
    slots[3] = -1
    K0 = K.clone()
    out = op(qkv, qw, kw, cos, sin, positions, slots, K, V, out=torch.zeros(6, 4, 64, dtype=torch.bfloat16))
    axes = axis_of_frequency(op.sections, True)
    for t in range(6):
        x = qkv[t].double().view(8, 64)
        for h in range(6):
            n = x[h] / (x[h].square().mean() + 1e-6).sqrt() * (qw if h < 4 else kw).double()
            y = torch.empty(64, dtype=torch.float64)
            for i in range(32):
                at = int(positions[axes[i], t])
                c, s = float(cos[at, i]), float(sin[at, i])
                y[i], y[i + 32] = n[i] * c - n[i + 32] * s, n[i + 32] * c + n[i] * s
            got = out[t, h] if h < 4 else K[int(slots[t]) // 64, h - 4, int(slots[t]) % 64]
            if t == 2:
                assert h >= 4 or (got == 0).all()
            elif not (t == 3 and h >= 4):
                assert torch.allclose(got.double(), y, rtol=2**-8, atol=1e-5)
    assert torch.equal(K[int(slots[2]) // 64, :, int(slots[2]) % 64], K0[int(slots[2]) // 64, :, int(slots[2]) % 64])


def test_attention_reference_query_by_query():
    op = ez.AttnPromptOp(3, 9, 4, 64, 3, 64, num_kv_heads=2)
    Q, K, V, table, lens, cu = op.gen_data("cpu")
    cu = torch.tensor([0, 5, 5, 9], dtype=I32)
    lens = torch.tensor([3, 7, 70], dtype=I32)  # fewer keys than tokens in the first row
    table = torch.tensor([[0, -1, -1], [1, -1, -1], [1, 0, -1]], dtype=I32)
    out = op(Q, K, V, table, lens, cu)
    for b in (0, 2):
        m, n = int(cu[b + 1] - cu[b]), int(lens[b])
        for i in range(m):
            seen = n - m + i + 1
            for h in range(4):
                if seen <= 0:
                    assert (out[cu[b] + i, h] == 0).all()
                    continue
                keys = torch.stack([K[int(table[b, j // 64]), h // 2, j % 64] for j in range(seen)]).double()
                vals = torch.stack([V[int(table[b, j // 64]), h // 2, j % 64] for j in range(seen)]).double()
                p = torch.softmax(keys @ Q[cu[b] + i, h].double() / 8, 0)
                assert torch.allclose(out[cu[b] + i, h].double(), p @ vals, rtol=2**-8, atol=2**-8)


def test_c_entries_refuse_without_a_gpu():
    lib, P = _lib.load(), ctypes.c_void_p
    a, b, c, odd = P(0x100000), P(0x2000000), P(0x4000000), P(0x4000002)
    bad, shape, none = _lib.EZB_ERR_INVALID_ARGUMENT, _lib.EZB_ERR_UNSUPPORTED_SHAPE, _lib.EZB_ERR_WORKSPACE

    def plan(*sizes, out=c, ctx=a):
        outs = [P(out.value + 0x100000 * i) for i in range(5)]
        return lib.ezb_paged_plan(ctx, b, P(0x3000000), P(0x3800000), P(0x3900000), *outs, *sizes, None)

    assert plan(0, 8, 4, 64, 8, 8) == bad
    assert plan(2, 8, 4, 48, 8, 8) == shape and b"power of two" in lib.ezb_last_error_message()
    assert plan(8193, 8, 4, 64, 8, 8) == shape
    assert plan(2, 8, 1 << 20, 2048, 8, 8) == shape
    assert plan(2, 8, 4, 64, 8, 8, out=a) == bad and b"overlaps" in lib.ezb_last_error_message()
    assert lib.ezb_paged_plan(*[None] * 10, 2, 8, 4, 64, 8, 8, None) == bad

    def rope(T=4, H=4, NKV=2, D=64, rows=10, sections=(32,), interleaved=0, page=64, pages=4, ld=None, qkv=a, out=c):
        arr = (ctypes.c_int * len(sections))(*sections)
        return lib.ezb_paged_qk_norm_rope(qkv, (H + 2 * NKV) * D if ld is None else ld, None, None, b, b, b, b, b, b, out, T, H, NKV, D,
                                          rows, len(sections), arr, interleaved, page, pages, 1e-6, None)

    assert rope(T=0) == bad and rope(D=96) == shape and rope(NKV=3) == shape and rope(page=65) == shape
    assert rope(sections=(16, 8)) == shape and rope(sections=(40, -8)) == shape and rope(sections=(8, 8, 8, 8)) == shape
    assert rope(sections=(0, 16, 16), interleaved=1) == shape
    assert rope(ld=500) == bad and rope(ld=516) == bad and rope(qkv=odd) == bad and rope(out=a) == bad
    assert rope(pages=1 << 25) == shape

    def linear(M=4, N=8, K=16, X=a, ldx=None, W=b, bias=None, res=None, ldres=None, out=c, ldout=None, act=0, f32=0):
        return lib.ezb_linear_bf16(X, K if ldx is None else ldx, W, bias, res, N if ldres is None else ldres, out,
                                   N if ldout is None else ldout, M, N, K, act, f32, None)

    assert linear(M=0) == bad and linear(K=12) == shape and linear(act=5) == bad and linear(act=-1) == bad
    assert linear(X=odd) == bad and linear(W=odd) == bad and linear(ldx=8) == bad and linear(ldx=20) == bad and linear(ldout=7) == bad
    assert linear(out=P(0x4000001)) == bad and linear(out=odd, f32=1) == bad
    assert linear(out=a) == bad and linear(out=b) == bad and linear(bias=c) == bad
    assert linear(res=P(0x4000010)) == bad and linear(res=c, ldres=9) == bad and linear(res=c, f32=1) == bad
    assert b"overlaps residual" in lib.ezb_last_error_message()
    assert linear(M=1 << 30, N=1 << 30) == shape

    def attn(B=2, T=8, H=4, NKV=2, D=64, max_pages=4, page=64, pages=9, Q=a, ldq=256, out=c, ldo=256, w=b, size=1 << 30):
        return lib.ezb_attn_prompt(Q, ldq, b, b, b, b, b, out, ldo, w, size, B, T, H, NKV, D, max_pages, page, pages, None)

    assert attn(B=0) == bad and attn(T=0) == bad and attn(D=32) == shape and attn(NKV=3) == shape and attn(page=32) == shape
    assert attn(H=258, ldq=1 << 15, ldo=1 << 15, NKV=2) == shape
    assert attn(ldq=255) == bad and attn(ldq=260) == bad and attn(ldo=128) == bad and attn(Q=odd) == bad and attn(out=odd) == bad
    assert attn(out=a) == bad and attn(w=None) == none and attn(size=100) == none
    assert attn(max_pages=1 << 25) == shape
    assert lib.ezb_attn_prompt_workspace_bytes(96) == 0


def test_packed_entries_are_the_same_calls():
    """Words in the order of the arguments: pointers, negative sizes and a float arrive as they are."""
    lib = _lib.load()
    import struct

    def same(name, *args):
        words = [struct.unpack("i", struct.pack("f", a))[0] if isinstance(a, float) else 0 if a is None else a for a in args]
        code = getattr(lib, name)(*args)
        message = lib.ezb_last_error_message()
        assert code < 0 and getattr(lib, name + "_packed")(struct.pack(f"{len(words)}q", *words)) == code
        assert lib.ezb_last_error_message() == message
        return message

    p = 0x7F0012345600
    assert b"null" in same("ezb_paged_plan", *[None] * 10, 2, 8, 4, 64, 8, 8, None)
    assert b"8192" in same("ezb_paged_plan", *[p] * 10, 9000, 8, 4, 64, 8, 8, None)
    assert b"positive" in same("ezb_linear_bf16", p, 64, p, None, None, 8, p, 8, -3, 8, 64, 0, 0, None)
    assert b"128 query" in same("ezb_attn_prompt", p, 1 << 40, p, p, p, p, p, p, 1 << 41, p, 1 << 33, 1, 1, 129, 1, 64, 1, 64, 1, None)
    assert b"apart" in same("ezb_paged_qk_norm_rope", p, 8, None, None, *[p] * 7, 1, 8, 8, 64, 16, 1, p, 0, 64, 1, 1e-6, None)
    assert lib.ezb_attn_prompt_packed(None) == lib.ezb_paged_plan(*[None] * 10, 2, 8, 4, 64, 8, 8, None)


@pytest.mark.parametrize("name", ["ezb_paged_plan", "ezb_paged_qk_norm_rope", "ezb_linear_bf16", "ezb_attn_prompt"])
def test_packed_sizes_beyond_32_bits_are_refused(name):
    """A size that a 32-bit argument cannot hold is refused; cut off, 2**32 + 8 would be a call for 8."""
    import struct

    lib, kinds = _lib.load(), _lib.SIGNATURES[name][1]
    sizes = [i for i, kind in enumerate(kinds) if kind is ctypes.c_int]
    assert len(sizes) >= 5
    for at in sizes:
        for size in (1 << 31, (1 << 32) + 8, (1 << 62) + 64, -(1 << 31) - 1):
            words = [8 if kind is ctypes.c_int else 0 for kind in kinds]
            words[at] = size
            assert getattr(lib, name + "_packed")(struct.pack(f"{len(words)}q", *words)) == _lib.EZB_ERR_UNSUPPORTED_SHAPE
            assert b"32 bits" in lib.ezb_last_error_message()


class _FaultyLib:
    """A library whose status word reads ``word`` once (cleared by the read)."""

    def __init__(self, word):
        self.word = word

    def ezb_device_status(self, out, clear):
        out._obj.value, word = self.word, self.word
        self.word = 0 if clear else self.word
        return _lib.EZB_ERR_DEVICE_FAULT if word else _lib.EZB_OK

    def ezb_stream_capture_id(self, stream):
        return 0


@pytest.fixture
def host_workspaces(monkeypatch):
    """``_Workspaces`` on the host: its tensors come from there, and nothing is being captured."""
    from ezops_b200.kernels import sm100_prompt

    empty = torch.empty
    monkeypatch.setattr(sm100_prompt, "_capturing", lambda: False)
    monkeypatch.setattr(sm100_prompt.torch, "empty", lambda n, dtype, device: empty(n, dtype=dtype).fill_(9))
    return sm100_prompt._Workspaces


@pytest.mark.parametrize("word", [0x105, 0x302])
def test_workspaces_are_renewed_after_a_recorded_fault(monkeypatch, host_workspaces, word):
    """A call that gave up leaves its counters half counted; reading the fault has every operator start from cleared ones.  Any
    fault does: the word keeps the first one only."""
    lib = _FaultyLib(0)
    monkeypatch.setattr(_lib, "_lib", lib)
    spaces = [host_workspaces(lib) for _ in range(2)]
    before = [s.get(8192, 0, stream) for s in spaces for stream in (1, 2)]
    for ws in before:
        assert (ws[:4096] == 0).all()
        ws[:4096] = 3  # what a call that gave up leaves
    assert _lib.device_status() == 0
    assert all(s.get(8192, 0, stream) is before[2 * i + stream - 1] for i, s in enumerate(spaces) for stream in (1, 2))
    lib.word = word
    assert _lib.device_status() == word
    for s in spaces:
        for stream in (1, 2):
            ws = s.get(8192, 0, stream)
            assert (ws[:4096] == 0).all() and ws is s.get(8192, 0, stream)


def test_workspaces_of_many_streams_do_not_pile_up(host_workspaces):
    spaces = host_workspaces(_FaultyLib(0))
    kept = spaces.get(8192, 0, 0)
    for stream in range(1, 8):
        spaces.get(8192, 0, stream)
    assert spaces.get(8192, 0, 0) is kept
    for stream in range(8, 500):
        ws = spaces.get(8192, stream % 2, stream)
        assert ws is spaces.get(8192, stream % 2, stream) and (ws[:4096] == 0).all()
        assert len(spaces._eager) <= 8


def _spans(**at):
    """Addresses of a call's arrays, far apart, but for those given."""
    names = ("ctx", "new", "table", "free", "count", "lens", "cu", "positions", "slots", "left", "qkv", "qw", "kw", "cos", "sin", "K", "V",
             "Q", "out", "ws")
    return {name: at.get(name, 0x1000000 * (i + 1)) for i, name in enumerate(names)}


def test_results_that_overlap_are_refused():
    """Whatever a call writes has to lie apart from all else that it reads or writes."""
    lib, bad = _lib.load(), _lib.EZB_ERR_INVALID_ARGUMENT

    def refused(code, what):
        assert code == bad, what
        assert b"overlap" in lib.ezb_last_error_message(), (what, lib.ezb_last_error_message())

    def plan(**at):
        a = _spans(**at)
        return lib.ezb_paged_plan(*[a[n] for n in ("ctx", "new", "table", "free", "count", "lens", "cu", "positions", "slots", "left")],
                                  4, 100, 8, 64, 32, 40, None)

    base = _spans()
    writes, reads = ("table", "lens", "cu", "positions", "slots", "left"), ("ctx", "new", "free", "count")
    for w in writes:
        for other in (*writes, *reads):
            if w != other:
                refused(plan(**{w: base[other]}), (w, other))
    refused(plan(lens=base["cu"] + 16), "last entry of cu")
    refused(plan(free=base["table"] + 4 * 31), "last entry of the table")

    def rope(**at):
        a, sections = _spans(**at), (ctypes.c_int * 1)(32)
        return lib.ezb_paged_qk_norm_rope(a["qkv"], 520, a["qw"], a["kw"], a["cos"], a["sin"], a["positions"], a["slots"], a["K"], a["V"],
                                          a["out"], 4, 4, 2, 64, 10, 1, sections, 0, 64, 3, 1e-6, None)

    for w in ("K", "V", "out"):
        for other in ("qkv", "qw", "kw", "cos", "sin", "positions", "slots", "K", "V", "out"):
            if w != other:
                refused(rope(**{w: base[other]}), (w, other))
    refused(rope(V=base["K"] + 2 * (3 * 2 * 64 * 64 - 8)), "end of K")

    def attn(**at):
        a = _spans(**at)
        return lib.ezb_attn_prompt(a["Q"], 256, a["K"], a["V"], a["table"], a["lens"], a["cu"], a["out"], 256, a["ws"], 1 << 25, 2, 8, 4, 2,
                                   64, 4, 64, 9, None)

    for other in ("Q", "K", "V", "table", "lens", "cu", "ws"):
        refused(attn(out=base[other]), ("out", other))
        if other != "ws":
            refused(attn(ws=base[other]), ("ws", other))
    refused(attn(out=base["ws"] + 512), "inside the workspace")
