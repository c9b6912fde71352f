"""The prompt operators on the GPU against plain 64-bit implementations: sizes, lengths, masks and strides where they can
go wrong.  Tolerances count roundings: bf16 rounds by at most 2^-8 of the value, fp32 by 2^-24; a tensor-core product adds
its K terms 16 at a time into an fp32 sum, one rounding (2^-23, it may truncate) of at most the sum of absolute values each."""

import pytest
import torch

import ezops_b200 as ez
from ezops_b200 import _lib

pytestmark = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32
DEV = "cuda"


@pytest.fixture(autouse=True)
def _healthy(cuda_device):
    _lib.device_status()
    yield
    assert _lib.device_status() == 0


def ints(*values):
    return torch.tensor(values, dtype=I32, device=DEV)


def close(actual, expected, tol):
    """|actual - expected| <= tol everywhere (NaN nowhere)."""
    excess = (actual.double() - expected).abs() - tol
    assert not torch.isnan(actual).any()
    assert (excess <= 0).all(), f"{(excess > 0).sum().item()} of {excess.numel()} outside, worst {excess.max().item():.3e}"


# ------------------------------------------------------------------- plan ---
def plan_case(B, T, max_pages, page, ctx, new, spare, seed=0, bad=False):
    g = torch.Generator().manual_seed(seed)
    ctx, new = torch.as_tensor(ctx), torch.as_tensor(new)
    held = (ctx.clamp(0, max_pages * page) + page - 1) // page
    pages = int(held.sum()) + max(spare, 1)
    order = torch.randperm(pages, generator=g)
    table = torch.full((B, max_pages), -7)
    table[torch.arange(max_pages) < held[:, None]] = order[: int(held.sum())]
    free = torch.full((pages + 3,), -9)
    free[:spare] = order[int(held.sum()) : int(held.sum()) + spare]
    if bad:  # ids outside the pools, in the table and in the list
        table[0, 0], free[spare - 1] = pages, -2
    args = [t.to(I32) for t in (ctx, new, table, free, torch.tensor([spare]))]
    ref = ez.PagedPlanOp(B, T, max_pages, page, pages)
    op = ez.PagedPlanOp(B, T, max_pages, page, pages, backend="cuda")
    expected_table = args[2].clone()
    expected = ref(args[0], args[1], expected_table, *args[3:])
    dev = [t.to(DEV) for t in args]
    out = op(*dev)
    for name, a, e in zip(out._fields, out, expected):
        assert torch.equal(a.cpu(), e), name
    assert torch.equal(dev[2].cpu(), expected_table)
    return op, dev, out


@pytest.mark.parametrize("B,T", [(1, 1), (1, 5000), (3, 64), (32, 32), (33, 1025), (257, 2048), (1000, 1024), (1000, 9000), (8192, 8192)])
@pytest.mark.parametrize("page", [64, 256])
def test_plan_matches_the_definition(B, T, page):
    g = torch.Generator().manual_seed(B + T)
    max_pages = 4096 // page + -(-T // page)
    ctx = torch.randint(0, 4096, (B,), generator=g) if B < 2000 else torch.randint(0, 200, (B,), generator=g)
    share = torch.bincount(torch.randint(0, B, (T,), generator=g), minlength=B)
    need = ((ctx + share + page - 1) // page - (ctx + page - 1) // page).sum()
    plan_case(B, T, max_pages, page, ctx, share, int(need) + 5)


def test_plan_lengths_of_zero_negative_and_too_many():
    page = 64
    # nothing new anywhere; a row without anything; negative lengths; a full page; more than the row holds
    plan_case(4, 16, 4, page, [0, 64, 70, 0], [0, 0, 0, 0], 4)
    plan_case(5, 40, 4, page, [0, 64, -3, 255, 200], [3, 1, 2, 1, -5], 9)
    plan_case(2, 300, 4, page, [200, 300], [100, 50], 9)  # 256 positions a row
    plan_case(3, 10, 4, page, [0, 1, 2], [6, 6, 6], 9)  # 18 tokens into 10
    plan_case(2, 10, 4, page, [0, 0], [2**30, 2**30], 9)


def test_plan_with_too_few_pages_and_bad_ids():
    _, _, out = plan_case(3, 400, 8, 64, [10, 64, 0], [100, 130, 100], 3)
    assert int(out.free_count) < 0
    plan_case(2, 200, 8, 64, [64, 0], [90, 90], 6, bad=True)
    plan_case(2, 200, 8, 64, [64, 0], [90, 90], 0)


def test_plan_in_a_graph_follows_its_inputs():
    op, dev, _ = plan_case(3, 64, 8, 64, [10, 64, 0], [1, 20, 5], 6)
    plan = op.new_plan(DEV)
    table0 = dev[2].clone()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        op(*dev, out=plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(*dev, out=plan)
    ref = ez.PagedPlanOp(3, 64, 8, 64, op.num_pages)
    for new in ([1, 1, 1], [0, 63, 0], [30, 0, 34]):
        dev[1].copy_(torch.tensor(new, dtype=I32))
        dev[2].copy_(table0)
        graph.replay()
        host = [t.cpu() for t in (dev[0], dev[1], table0, dev[3], dev[4])]
        expected = ref(*host)
        assert all(torch.equal(a.cpu(), e) for a, e in zip(plan, expected)) and torch.equal(dev[2].cpu(), host[2])


# ------------------------------------------------------------------- rope ---
SECTIONS = {64: [((32,), False), ((16, 16), True), ((12, 10, 10), True), ((8, 12, 12), False), ((32, 0, 0), True)],
            128: [((64,), False), ((32, 32), False), ((24, 20, 20), True), ((24, 20, 20), False), ((0, 64), False)]}


def rope64(op, qkv, qw, kw, cos, sin, positions):
    """q and k after norm and rotation in 64 bits, and the size of what is added there."""
    from ezops_b200.ops.paged_qk_norm_rope import axis_of_frequency

    T, D, H, NKV = qkv.shape[0], op.head_dim, op.num_heads, op.num_kv_heads
    x = qkv.double().reshape(T, H + 2 * NKV, D)
    w = torch.ones(H + NKV, D, device=DEV, dtype=torch.float64)
    if qw is not None:
        w[:H] = qw.double()
    if kw is not None:
        w[H:] = kw.double()
    n = x[:, : H + NKV] / (x[:, : H + NKV].square().mean(-1, keepdim=True) + op.rms_eps).sqrt() * w
    axis = torch.tensor(axis_of_frequency(op.sections, op.interleaved) * 2, device=DEV)
    at = positions.reshape(len(op.sections), T).long().clamp(min=0)[axis].T
    c, s = (t[at, torch.arange(D, device=DEV)].double()[:, None] for t in (cos, sin))
    r = torch.cat([-n[..., D // 2 :], n[..., : D // 2]], -1)
    return n * c + r * s, (n * c).abs() + (r * s).abs(), x[:, H + NKV :]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", range(5))
@pytest.mark.parametrize("T,H,NKV,page", [(1, 8, 8, 64), (7, 14, 2, 128), (33, 32, 8, 256), (1201, 6, 2, 64), (3000, 32, 1, 128)])
def test_rope_matches_the_formula(T, H, NKV, page, D, kind):
    sections, interleaved = SECTIONS[D][kind]
    torch.manual_seed(T + kind)
    pages = -(-T // page) + 2
    op = ez.PagedQkNormRopeOp(T, H, D, 517, page, pages, backend="cuda", num_kv_heads=NKV, sections=sections, interleaved=interleaved)
    qkv, qw, kw, cos, sin, positions, slots, K, V = op.gen_data()
    if kind == 1:
        qw = kw = None
    if T > 5:
        positions[..., T - 2 :] = -1  # padding
        slots[T - 2 :] = -1
        slots[1] = -1  # a real token that is not cached
        positions[0, 3], slots[3] = -5, 0  # padding in the middle, with a slot that must stay untouched
        slots[:T][(slots == 0) & (torch.arange(T, device=DEV) != 3)] = -1
    if T == 33:  # rows further apart, a slice of a wider tensor
        wide = torch.randn(T, qkv.shape[1] + 24, device=DEV).to(BF16)
        wide[:, 8 : 8 + qkv.shape[1]] = qkv
        qkv = wide[:, 8 : 8 + qkv.shape[1]]
    K0, V0 = K.clone(), V.clone()
    out = torch.full((T, H, D), 7.0, device=DEV, dtype=BF16)
    got = op(qkv, qw, kw, cos, sin, positions, slots, K, V, out=out)
    assert got is out
    y, size, v = rope64(op, qkv, qw, kw, cos, sin, positions)
    # one bf16 rounding; about a dozen fp32 roundings of the two products in front of it
    tol = 2**-8 * y.abs() + 2**-20 * size
    real = (positions.reshape(len(sections), T) >= 0).all(0)
    close(out[real], y[real][:, :H], tol[real][:, :H])
    assert (out[~real] == 7.0).all()
    keep = real & (slots >= 0)
    slot = slots[keep].long()
    at = (slot // page, slice(None), slot % page)
    close(K[at], y[keep][:, H:], tol[keep][:, H:])
    assert torch.equal(V[at], v[keep].to(BF16))
    K[at], V[at] = K0[at], V0[at]
    assert torch.equal(K, K0) and torch.equal(V, V0)  # nothing else was written


def test_rope_agrees_with_the_decode_operator():
    """One axis, one token per row: the operator of a decode step on contiguous caches (the same arithmetic, another order
    of the sum of squares: at most one bf16 step apart)."""
    B, H, NKV, D, S = 5, 16, 8, 128, 256
    dec = ez.FusedQkNormRopeOp(B, H, D, S, [0, 255, 17, 64, 100], backend="cuda", num_kv_heads=NKV)
    q, k, v, qw, kw, cos, sin, Kc, Vc = dec.gen_data()
    op = ez.PagedQkNormRopeOp(B, H, D, S, S, B, backend="cuda", num_kv_heads=NKV)
    positions = ints(0, 255, 17, 64, 100)
    slots = positions + S * torch.arange(B, device=DEV, dtype=I32)
    Kp, Vp = Kc.clone(), Vc.clone()
    q_out, _ = dec(q, k, v, qw, kw, cos, sin, Kc, Vc)
    got = op(torch.cat([q.reshape(B, -1), k.reshape(B, -1), v.reshape(B, -1)], 1), qw, kw, cos, sin, positions, slots, Kp, Vp)
    for a, e in ((got, q_out), (Kp, Kc)):
        assert ((a.float() - e.float()).abs() <= 2**-7 * e.float().abs() + 2**-18).all()
    assert torch.equal(Vp, Vc)


def test_rope_records_positions_and_slots_out_of_range():
    op = ez.PagedQkNormRopeOp(3, 4, 64, 100, 64, 2, backend="cuda", num_kv_heads=2)
    data = list(op.gen_data())
    data[5], data[6] = ints(5, 6, 7), ints(0, 128, 3)
    K0, out = data[7].clone(), torch.zeros(3, 4, 64, device=DEV, dtype=BF16)
    op(*data, out=out)
    assert _lib.device_status() == 0x303
    assert out[1].abs().sum() > 0 and torch.equal(data[7][1], K0[1])  # q is there, no page touched
    data[5], data[6] = ints(5, 100, 7), ints(0, 1, 3)
    K0 = data[7].clone()
    out.zero_()
    op(*data, out=out)
    assert _lib.device_status() == 0x301
    assert out[1].abs().sum() == 0 and torch.equal(data[7][0, :, 1], K0[0, :, 1])


# ----------------------------------------------------------------- linear ---
def linear64(op, X, W, bias, residual):
    """The result in 64 bits and how far fp32 arithmetic and the final rounding may be from it."""
    z = X.double() @ W.double().T
    err = (X.shape[1] / 16 + 4) * 2**-23 * (X.double().abs() @ W.double().abs().T)
    if bias is not None:
        z = z + bias.double()
        err = err + 2**-23 * z.abs()
    N, F = op.out_features, torch.nn.functional
    if op.activation == "swiglu":
        g, u = z[:, :N], z[:, N:]
        y = F.silu(g) * u
        err = 1.1 * err[:, :N] * u.abs() + F.silu(g).abs() * err[:, N:] + 2**-20 * y.abs()  # |silu'| < 1.1
    else:
        y = z if op.activation is None else getattr(F, op.activation)(z)
        if op.activation is not None:
            err = 1.13 * err + 2**-20 * z.abs()  # |gelu'| < 1.13; a handful of fp32 roundings of the argument and the result
    if residual is not None:
        y = y + residual.double()
        err = err + 2**-23 * (y.abs() + residual.double().abs())
    return y, err + (2**-8 if op.out_dtype == BF16 else 2**-24) * y.abs() + 1e-30


def linear_case(M, N, K, act=None, bias=False, residual=False, out_dtype=BF16, seed=0):
    torch.manual_seed(seed + M + N + K)
    op = ez.LinearOp(M, N, K, backend="cuda", bias=bias, activation=act, residual=residual, out_dtype=out_dtype)
    X, W, b, r = op.gen_data()
    out = op(X, W, bias=b, residual=r)
    assert out.dtype == out_dtype and out.shape == (M, N)
    y, tol = linear64(op, X, W, b, r)
    close(out, y, tol)


@pytest.mark.parametrize("M", [1, 2, 17, 64, 65, 127, 128, 129, 256, 300, 777])
@pytest.mark.parametrize("N,K", [(1, 8), (40, 64), (129, 200), (512, 1024), (1000, 72)])
def test_linear_sizes(M, N, K):
    linear_case(M, N, K)
    linear_case(M, N, K, act="swiglu", bias=True, residual=True)


@pytest.mark.parametrize("act", [None, "silu", "gelu", "relu", "swiglu"])
@pytest.mark.parametrize("out_dtype", [BF16, torch.float32])
@pytest.mark.parametrize("bias,residual", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("M", [5, 200])
def test_linear_epilogues(M, act, out_dtype, bias, residual):
    linear_case(M, 264, 320, act, bias, residual, out_dtype)


@pytest.mark.parametrize("M,N,K", [(2048, 4096, 1024), (1111, 2600, 2048), (4096, 256, 4096), (513, 20000, 512)])
@pytest.mark.parametrize("act", [None, "swiglu"])
def test_linear_many_tiles(M, N, K, act):
    linear_case(M, N, K, act, residual=act is None)


@pytest.mark.parametrize("M", [1, 17, 64])
@pytest.mark.parametrize("out_dtype", [BF16, torch.float32])
def test_linear_few_rows_many_tiles(M, out_dtype):
    """Several rounds of tiles per CTA, tiles cut along K and not, results that are no multiple of a tile."""
    linear_case(M, 60001, 64, bias=True, residual=True, out_dtype=out_dtype)
    linear_case(M, 30000, 200, act="silu", out_dtype=out_dtype)
    linear_case(M, 20008, 136, act="swiglu", bias=True, out_dtype=out_dtype)
    linear_case(M, 520, 8192, bias=True, out_dtype=out_dtype)


@pytest.mark.parametrize("M", [3, 500])
def test_linear_strides_and_in_place_residual(M):
    N, K = 200, 136
    torch.manual_seed(M)
    op = ez.LinearOp(M, N, K, backend="cuda", residual=True)
    X, W, _, r = op.gen_data()
    wide = torch.randn(M, K + 40, device=DEV).to(BF16)
    wide[:, 16 : 16 + K] = X
    y, tol = linear64(op, X, W, None, r)
    stream = torch.full((M, N + 7), 3.0, device=DEV, dtype=BF16)  # rows an odd number of elements apart
    stream[:, 2 : 2 + N] = r
    view = stream[:, 2 : 2 + N]
    got = op(wide[:, 16 : 16 + K], W, residual=view, out=view)
    assert got.data_ptr() == view.data_ptr()
    close(view, y, tol)
    assert (stream[:, :2] == 3.0).all() and (stream[:, 2 + N :] == 3.0).all()
    # input and output as columns of one tensor
    both = torch.zeros(M, K + N, device=DEV, dtype=BF16)
    both[:, :K] = X
    op(both[:, :K], W, residual=r, out=both[:, K:])
    close(both[:, K:], y, tol)
    assert torch.equal(both[:, :K], X)


def test_linear_rows_do_not_mix():
    """A row of infinities or NaN stays in its row."""
    for M in (20, 300):
        op = ez.LinearOp(M, 96, 64, backend="cuda", activation="relu")
        X, W, _, _ = op.gen_data()
        clean = op(X, W)
        X[4], X[7] = float("inf"), float("nan")
        out = op(X, W)
        keep = torch.ones(M, dtype=torch.bool, device=DEV)
        keep[[4, 7]] = False
        assert torch.equal(out[keep], clean[keep]) and torch.isnan(out[7]).all()


@pytest.mark.parametrize("M", [9, 300])
def test_linear_other_stream_and_graph(M):
    op = ez.LinearOp(M, 512, 256, backend="cuda", bias=True)
    X, W, b, _ = op.gen_data()
    plain = op(X, W, bias=b)
    out = torch.empty_like(plain)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        op(X, W, bias=b, out=out)
    s.synchronize()
    assert torch.equal(out, plain)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(X, W, bias=b, out=out)
    X.mul_(2)
    graph.replay()
    assert torch.equal(out, op(X, W, bias=b))


# -------------------------------------------------------------- attention ---
def attn64(Q, K, V, table, lens, cu, NKV, page):
    """The result in 64 bits, and the weighted sum of |v| that the rounding of the weights is relative to."""
    D = Q.shape[2]
    out = torch.zeros(Q.shape, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(out)
    for b, n in enumerate(lens):
        m = cu[b + 1] - cu[b]
        if m == 0 or n == 0:
            continue
        at = table[b, : -(-n // page)].long()
        k, v = (t[at].double().transpose(0, 1).reshape(NKV, -1, D)[:, :n] for t in (K, V))
        q = Q[cu[b] : cu[b + 1]].double().view(m, NKV, -1, D)
        s = torch.einsum("mhgd,hnd->hgmn", q, k) / D**0.5
        i = torch.arange(m, device=DEV)[:, None] + (n - m)
        s = s.masked_fill(torch.arange(n, device=DEV) > i, float("-inf"))
        p = torch.softmax(s, -1).nan_to_num(0.0)
        for dst, x in ((out, v), (size, v.abs())):
            dst[cu[b] : cu[b + 1]] = torch.einsum("hgmn,hnd->mhgd", p, x).reshape(m, -1, D)
    return out, size


def attn_data(new, ctx, H, NKV, D, page, seed=0, extra_pages=2, behind=0):
    """Pools whose unused part is NaN; tokens behind the last row when asked for."""
    torch.manual_seed(seed)
    lens = [max(0, a + b) for a, b in zip(new, ctx)]
    used = [-(-n // page) for n in lens]
    wide = max(1, max(used)) + 1
    pages = sum(used) + extra_pages
    order = torch.randperm(pages)
    table = torch.full((len(new), wide), -1)
    K, V = (torch.full((pages, NKV, page, D), float("nan"), device=DEV, dtype=BF16) for _ in range(2))
    at = 0
    for b, (n, u) in enumerate(zip(lens, used)):
        table[b, :u] = order[at : at + u]
        at += u
        for pool in (K, V):
            rows = torch.randn(NKV, n, D, device=DEV).to(BF16)
            for j in range(u):
                part = rows[:, j * page : (j + 1) * page]
                pool[int(table[b, j]), :, : part.shape[1]] = part
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    Q = torch.randn(max(1, cu[-1] + behind), H, D, device=DEV).to(BF16)
    return Q, K, V, table.to(I32).to(DEV), lens, cu


def attn_check(op, Q, K, V, table, lens, cu, NKV, page, out=None):
    got = op(Q, K, V, table, ints(*lens), ints(*cu), out=out)
    e, size = attn64(Q, K, V, table, lens, cu, NKV, page)
    # bf16 weights (2^-8 of each) and a bf16 result; scores and exponentials in fp32 (arguments below 64, 2^-14 in all)
    tol = 2**-8 * e.abs() + (2**-8 + 2**-14) * size + 1e-30
    close(got[: cu[-1]], e[: cu[-1]], tol[: cu[-1]])
    return got


def attn_case(new, ctx, H, NKV, D, page, **kw):
    Q, K, V, table, lens, cu = attn_data(new, ctx, H, NKV, D, page, **kw)
    op = ez.AttnPromptOp(len(new), Q.shape[0], H, D, table.shape[1], page, backend="cuda", num_kv_heads=NKV)
    return op, (Q, K, V, table, lens, cu), attn_check(op, Q, K, V, table, lens, cu, NKV, page)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 500])
@pytest.mark.parametrize("D", [64, 128])
def test_attn_one_prompt(n, D):
    attn_case([n], [0], 8, 2, D, 64)


@pytest.mark.parametrize("H,NKV", [(4, 4), (6, 3), (6, 2), (10, 2), (14, 2), (16, 2), (32, 1), (43, 1), (100, 1), (128, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_attn_groups(H, NKV, D):
    attn_case([70, 1, 150], [0, 333, 200], H, NKV, D, 128)


@pytest.mark.parametrize("page", [64, 128, 256, 1024])
def test_attn_pages_and_contexts(page):
    attn_case([1, 64, 7, 200, 1], [63, 64, 1000, 57, 0], 16, 4, 128, page)
    attn_case([1, 1, 1, 1], [1500, 2047, 128, 127], 32, 8, 128, page)


def test_attn_rows_without_tokens_or_keys():
    op, data, got = attn_case([0, 5, 0, 40, 0], [0, 10, 300, 0, 7], 8, 2, 128, 64)
    # fewer keys than tokens: the first queries see nothing
    for D in (64, 128):
        Q, K, V, table, lens, cu = attn_data([70, 300, 3], [0, 0, 0], 8, 2, D, 64)
        lens = [20, 130, 0]
        op = ez.AttnPromptOp(3, Q.shape[0], 8, D, table.shape[1], 64, backend="cuda", num_kv_heads=2)
        got = attn_check(op, Q, K, V, table, lens, cu, 2, 64)
        assert (got[:50] == 0).all() and (got[70:240] == 0).all() and (got[370:] == 0).all()


def test_attn_all_rows_empty_leaves_the_output():
    op = ez.AttnPromptOp(3, 4, 8, 128, 1, 64, backend="cuda", num_kv_heads=2)
    Q, K, V, table, _, _ = attn_data([4], [0], 8, 2, 128, 64)
    out = torch.full_like(Q, 5.0)
    op(Q, K, V, table.repeat(3, 1)[:, :1].contiguous(), ints(0, 9, 3), ints(0, 0, 0, 0), out=out)
    assert (out == 5.0).all()


def test_attn_tokens_behind_the_last_row_stay():
    Q, K, V, table, lens, cu = attn_data([33, 20], [5, 100], 8, 4, 128, 64, behind=9)
    op = ez.AttnPromptOp(2, Q.shape[0], 8, 128, table.shape[1], 64, backend="cuda", num_kv_heads=4)
    out = torch.full_like(Q, 5.0)
    attn_check(op, Q, K, V, table, lens, cu, 4, 64, out=out)
    assert (out[53:] == 5.0).all()


def test_attn_strided_rows():
    Q, K, V, table, lens, cu = attn_data([50, 1], [5, 300], 8, 4, 64, 64)
    op = ez.AttnPromptOp(2, Q.shape[0], 8, 64, table.shape[1], 64, backend="cuda", num_kv_heads=4)
    T = Q.shape[0]
    wide = torch.randn(T, 8 * 64 + 64, device=DEV).to(BF16)
    wide[:, 32 : 32 + 512] = Q.view(T, -1)
    out = torch.full((T, 600), 2.0, device=DEV, dtype=BF16)
    view = out[:, 8 : 8 + 512].unflatten(1, (8, 64))
    got = op(wide[:, 32 : 32 + 512].unflatten(1, (8, 64)), K, V, table, ints(*lens), ints(*cu), out=view)
    assert torch.equal(got, op(Q, K, V, table, ints(*lens), ints(*cu)))
    assert (out[:, :8] == 2.0).all() and (out[:, 520:] == 2.0).all()


def test_attn_large_scores():
    """One key far above the rest, growing along the row: the running maximum moves at every tile, and weights vanish."""
    Q, K, V, table, lens, cu = attn_data([3, 260], [1000, 0], 8, 2, 128, 64)
    for b in range(2):
        for j in range(-(-lens[b] // 64)):
            K[int(table[b, j])] *= 1 + j
    Q = (Q * 4).to(BF16)
    op = ez.AttnPromptOp(2, Q.shape[0], 8, 128, table.shape[1], 64, backend="cuda", num_kv_heads=2)
    got = op(Q, K, V, table, ints(*lens), ints(*cu))
    e, size = attn64(Q, K, V, table, lens, cu, 2, 64)
    # scores up to 4 * 17 * sqrt(128) * 5, in units of log2 below 2^12: an fp32 rounding of that is 2^-12, twice, and so is the
    # product's own (8 roundings of at most 2^-23 * 2^14): weights may be off by 2^-8
    close(got, e, 2**-8 * e.abs() + 2**-6 * size)


@pytest.mark.parametrize("B,low,high", [(400, 1, 3), (1000, 0, 2), (37, 1, 90)])
def test_attn_many_rows(B, low, high):
    g = torch.Generator().manual_seed(B)
    new = torch.randint(low, high + 1, (B,), generator=g).tolist()
    ctx = torch.randint(0, 200, (B,), generator=g).tolist()
    attn_case(new, ctx, 4, 2, 64, 64)


def test_attn_few_tokens_among_many_empty_rows():
    B = 5000
    new, ctx = [0] * B, [0] * B
    for b, (n, c) in {3: (40, 0), 4: (1, 500), 777: (200, 100), 4095: (1, 0), 4999: (70, 64)}.items():
        new[b], ctx[b] = n, c
    attn_case(new, ctx, 8, 2, 128, 64)


@pytest.mark.parametrize("D", [64, 128])
def test_attn_one_long_row_for_many_ctas(D):
    """A few queries behind a long context: every CTA has a part of the same unit, odd counts of blocks in each."""
    for new, ctx in ([2], [30000]), ([33], [9999]), ([1, 1], [12800, 128 * 37 - 1]), ([40, 1], [5000, 63]):
        attn_case(new, ctx, 8, 1, D, 128)


def test_attn_long_rows_are_cut_and_joined():
    op, (Q, K, V, table, lens, cu), got = attn_case([1, 1500, 129], [9000, 3000, 0], 8, 1, 128, 256)
    for _ in range(3):
        assert torch.equal(op(Q, K, V, table, ints(*lens), ints(*cu)), got)  # equal calls, equal bits
    attn_case([2048], [0], 4, 4, 128, 128)
    attn_case([1], [20000], 8, 2, 64, 64)


def test_attn_agrees_with_the_decode_operator():
    B, H, NKV, D, page = 6, 16, 8, 128, 64
    Q, K, V, table, lens, cu = attn_data([1] * B, [900, 0, 63, 64, 500, 777], H, NKV, D, page)
    op = ez.AttnPromptOp(B, B, H, D, table.shape[1], page, backend="cuda", num_kv_heads=NKV)
    dec = ez.get_kernel("attn_decode", "cuda")(B, H, table.shape[1] * page, D, num_kv_heads=NKV)
    got = op(Q, K, V, table, ints(*lens), ints(*cu))
    want = dec.call_paged(Q[:, :, None], K, V, table, ints(*lens), page)[:, :, 0]
    _, size = attn64(Q, K, V, table, lens, cu, NKV, page)
    assert ((got.double() - want.double()).abs() <= 2 * (2**-8 * want.double().abs() + (2**-8 + 2**-14) * size)).all()


def test_attn_bad_table_entries_read_as_zeros():
    Q, K, V, table, lens, cu = attn_data([40, 1], [200, 300], 8, 2, 128, 64)
    table[0, 1], table[1, 2] = -1, K.shape[0]
    op = ez.AttnPromptOp(2, Q.shape[0], 8, 128, table.shape[1], 64, backend="cuda", num_kv_heads=2)
    got = op(Q, K, V, table, ints(*lens), ints(*cu))
    assert _lib.device_status() == 0x302
    zero = torch.zeros_like(K[:1])
    Kz, Vz = torch.cat([K, zero]), torch.cat([V, zero])
    fixed = table.clone()
    fixed[0, 1] = fixed[1, 2] = K.shape[0]
    assert torch.equal(got, op(Q, Kz, Vz, fixed, ints(*lens), ints(*cu)))


def test_attn_offsets_beyond_its_arrays_are_cut():
    Q, K, V, table, lens, cu = attn_data([40, 30], [0, 0], 8, 2, 128, 64)
    op = ez.AttnPromptOp(2, Q.shape[0], 8, 128, table.shape[1], 64, backend="cuda", num_kv_heads=2)
    want = op(Q, K, V, table, ints(*lens), ints(*cu))
    assert torch.equal(op(Q, K, V, table, ints(*lens), ints(-3, 40, 10**6)), want)


def test_attn_graph_follows_lengths():
    Q, K, V, table, lens, cu = attn_data([100, 60, 1], [300, 0, 500], 8, 2, 128, 64)
    op = ez.AttnPromptOp(3, Q.shape[0], 8, 128, table.shape[1], 64, backend="cuda", num_kv_heads=2)
    d_lens, d_cu, out = ints(*lens), ints(*cu), torch.zeros_like(Q)
    op(Q, K, V, table, d_lens, d_cu, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(Q, K, V, table, d_lens, d_cu, out=out)
    for new in ([100, 60, 1], [1, 1, 1], [161, 0, 0], [0, 3, 400 - 400]):
        c = [0, new[0], new[0] + new[1], sum(new)]
        n = [min(a, b) for a, b in zip([new[0] + 200, 60, 501], lens)]
        d_cu.copy_(torch.tensor(c, dtype=I32)), d_lens.copy_(torch.tensor(n, dtype=I32))
        graph.replay()
        e, size = attn64(Q, K, V, table, n, c, 2, 64)
        close(out[: c[-1]], e[: c[-1]], (2**-8 * e.abs() + (2**-8 + 2**-14) * size + 1e-30)[: c[-1]])


@pytest.mark.parametrize("M,N,K,act", [(100, 8, 8192, None), (300, 64, 4984, None), (555, 44, 5544, "silu"), (279, 1, 4096, "gelu"),
                                       (1500, 60, 5000, None), (70, 20, 6000, "swiglu"), (257, 250, 12000, None), (700, 60, 4200, "swiglu")])
@pytest.mark.parametrize("out_dtype", [BF16, torch.float32])
def test_linear_tiles_cut_along_k(M, N, K, act, out_dtype):
    """Few results behind a long K: parts meet in shared memory; equal calls give equal bits."""
    op = ez.LinearOp(M, N, K, backend="cuda", bias=True, activation=act, residual=True, out_dtype=out_dtype)
    torch.manual_seed(M)
    X, W, b, r = op.gen_data()
    out = op(X, W, bias=b, residual=r)
    y, tol = linear64(op, X, W, b, r)
    close(out, y, tol)
    for _ in range(3):
        assert torch.equal(op(X, W, bias=b, residual=r), out)


@pytest.mark.parametrize("M,N,K,act", [(700, 1043, 200, "gelu"), (2500, 9001, 72, None), (190, 19494, 136, "relu"), (100, 5000, 520, "silu"),
                                       (128, 640, 1000, None), (129, 6402, 264, "swiglu"), (1030, 5005, 80, "swiglu"), (66, 33, 64, "swiglu"),
                                       (5000, 31, 72, "silu")])
@pytest.mark.parametrize("out_dtype", [BF16, torch.float32])
def test_linear_rows_that_start_anywhere(M, N, K, act, out_dtype):
    """A lane per output column: one and several rounds of tiles of every width, last tiles of both kinds, pitches of any size."""
    linear_case(M, N, K, act, True, True, out_dtype)
    op = ez.LinearOp(M, N, K, backend="cuda", activation=act, residual=True, out_dtype=out_dtype)
    torch.manual_seed(N)
    X, W, _, r = op.gen_data()
    y, tol = linear64(op, X, W, None, r)
    wide_r = torch.full((M, N + 5), 9.0, device=DEV, dtype=BF16)
    wide_r[:, 3 : 3 + N] = r
    wide = torch.full((M, N + 9), 3.0, device=DEV, dtype=out_dtype)
    out = wide[:, 4 : 4 + N]
    op(X, W, residual=wide_r[:, 3 : 3 + N], out=out)
    close(out, y, tol)
    assert (wide[:, :4] == 3.0).all() and (wide[:, 4 + N :] == 3.0).all()


def attn_rows(B, D, seed):
    """An operator, its arguments and the result of a call that cuts units between CTAs."""
    op = ez.AttnPromptOp(B, B, 8, D, 64, 64, num_kv_heads=2, backend="cuda")
    g = torch.Generator(device=DEV).manual_seed(seed)
    Q = torch.randn(B, 8, D, generator=g, device=DEV).to(BF16)
    K, V = (torch.randn(B * 64, 2, 64, D, generator=g, device=DEV).to(BF16) for _ in range(2))
    table = torch.arange(B * 64, device=DEV, dtype=torch.int32).view(B, 64)
    lens = torch.randint(2000, 4096, (B,), generator=g, device=DEV, dtype=torch.int32)
    return op, [Q, K, V, table, lens, torch.arange(B + 1, device=DEV, dtype=torch.int32)]


def test_attn_first_call_in_a_capture():
    """A first call that is captured leaves nothing behind that a call outside of the graph would use, before or after a replay."""
    op, args = attn_rows(3, 128, 1)
    want = attn_rows(3, 128, 1)[0](*args)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(*args, out=out)
    assert torch.equal(op(*args), want)
    for _ in range(2):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    assert torch.equal(op(*args), want)


def test_attn_streams_and_graphs_side_by_side():
    """One operator on two streams at once, and two graphs of it replayed at once: each has a workspace of its own."""
    op, args = attn_rows(2, 128, 2)
    other = [a.clone() for a in args]
    other[0] = -other[0]
    want, want2 = op(*args), op(*other)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for a in (args, other):
        out, graph = torch.zeros_like(want), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(8):
                op(*a, out=out)
        graphs.append(graph)
        outs.append(out)
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want2)
    results = [[], []]
    for _ in range(50):
        for i, a in enumerate((args, other)):
            with torch.cuda.stream(streams[i]):
                results[i].append(op(*a))
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results[0]) and all(torch.equal(r, want2) for r in results[1])


def test_pools_of_more_than_two_to_the_31_elements():
    """The last pages of large pools give what the same pages of small ones give, bit for bit."""
    NKV, page, D, pages = 8, 256, 128, 8300
    K, V = (torch.zeros(pages, NKV, page, D, device=DEV, dtype=BF16) for _ in range(2))
    assert K.numel() > 2**31
    op, (Q, k, v, table, lens, cu), want = attn_case([40, 1], [300, 500], 32, NKV, D, page)
    few = k.shape[0]
    K[-few:], V[-few:] = k, v
    far = torch.where(table >= 0, table + (pages - few), table)
    assert torch.equal(op(Q, K, V, far, ints(*lens), ints(*cu)), want)
    T = 50
    small, large = (ez.PagedQkNormRopeOp(T, 32, D, 512, page, n, backend="cuda", num_kv_heads=NKV) for n in (few, pages))
    qkv, qw, kw, cos, sin, positions, slots, k, v = small.gen_data()
    K[-few:], V[-few:] = k, v
    q = small(qkv, qw, kw, cos, sin, positions, slots, k, v)
    far = torch.where(slots >= 0, slots + (pages - few) * page, slots)
    assert torch.equal(large(qkv, qw, kw, cos, sin, positions, far, K, V), q)
    assert torch.equal(K[-few:], k) and torch.equal(V[-few:], v)


@pytest.mark.parametrize("N", [60000, 60001])
def test_linear_results_of_more_than_two_to_the_31_elements(N):
    M, K = 36000, 64
    op = ez.LinearOp(M, N, K, backend="cuda", residual=True)
    torch.manual_seed(N)
    X, W = torch.randn(M, K, device=DEV).to(BF16), torch.randn(N, K, device=DEV).to(BF16)
    r = torch.randn(M, N, device=DEV, dtype=BF16)
    out = op(X, W, residual=r)
    at = torch.tensor([0, 127, 128, 17000, 35791, 35792, 35999], device=DEV)  # 35791 * N is just below 2^31
    y, tol = linear64(op, X[at], W, None, r[at])
    close(out[at], y, tol)


@pytest.mark.parametrize("M", [5, 30, 64, 100, 129, 700])
@pytest.mark.parametrize("N,K", [(600, 520), (600, 4096), (2000, 12800), (40, 12800), (20001, 2056)])
def test_linear_fp32_results_keep_their_precision(M, N, K):
    """Each of the 32 steps of a segment may cut 2^-23 of the sum so far (2^-24 on average), which grows like the root of the steps:
    2/3 * 32 * 2^-24 of the segment, and segments err independently; plus a rounding per segment.  Sums that stay in the tensor
    cores for all of K = 12800 are 1.4e-5 off."""
    op = ez.LinearOp(M, N, K, backend="cuda", out_dtype=torch.float32)
    torch.manual_seed(M + N + K)
    X, W, _, _ = op.gen_data()
    y = X.double() @ W.double().T
    assert (op(X, W).double() - y).norm() <= (64 / 3 * 2**-24 + (K / 512) ** 0.5 * 2**-24) * y.norm()
    for act in ("swiglu", "gelu"):
        linear_case(M, min(N, 900) // 2, K, act, True, True, torch.float32)


@pytest.mark.parametrize("M,N,K", [(65, 33, 2048), (127, 515, 4600), (129, 200, 4096), (321, 77, 1000), (1000, 60, 4096), (4096, 100, 4096),
                                   (4001, 128, 3848)])
@pytest.mark.parametrize("act", [None, "gelu", "swiglu"])
@pytest.mark.parametrize("out_dtype", [BF16, torch.float32])
def test_linear_groups_of_rows(M, N, K, act, out_dtype):
    """Few results behind a long K: the last group of rows is shorter, and nothing behind the result is written."""
    linear_case(M, N, K, act, True, True, out_dtype)
    op = ez.LinearOp(M, N, K, backend="cuda", activation=act, out_dtype=out_dtype)
    X, W, _, _ = op.gen_data()
    wide = torch.full((M + 70, N + 3), 3.0, device=DEV, dtype=out_dtype)
    op(X, W, out=wide[:M, 1 : 1 + N])
    close(wide[:M, 1 : 1 + N], *linear64(op, X, W, None, None))
    assert (wide[M:] == 3.0).all() and (wide[:, 0] == 3.0).all() and (wide[:, 1 + N :] == 3.0).all()


def test_attn_goes_on_after_a_recorded_fault():
    """A wait that runs out leaves counters of cut rows half counted, so that nobody would join their parts any more.  Put there
    by hand; once a fault (here a bad page) has been read, calls give what a fresh operator gives."""
    op, args = attn_rows(2, 128, 3)
    want = op(*args)
    for ws in op._kernel._spaces._eager.values():
        ws[:640].view(torch.int32).fill_(1)
    bad = args[3].clone()
    bad[0, 0] = -1
    other = attn_rows(2, 128, 3)[0]
    other(*args[:3], bad, *args[4:])
    assert _lib.device_status() == 0x302
    assert torch.equal(op(*args), want) and torch.equal(op(*args), want)


def test_attn_on_more_streams_than_workspaces():
    op, args = attn_rows(2, 128, 4)
    want = op(*args)
    streams = [torch.cuda.Stream() for _ in range(12)]
    torch.cuda.synchronize()
    results = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(op(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results) and len(op._kernel._spaces._eager) <= 8


@pytest.mark.parametrize("ctx,new,cu,lens", [([0, 0], [2**30, 2**30], [0, 2**30, 2**30], [2**30, 0]),
                                             ([2**30, 5], [2**30, 7], [0, 2**30, 2**30], [2**30, 5]),
                                             ([2**29, 0], [2**29, 2**30], [0, 2**29, 2**30], [2**30, 2**29])])
def test_plan_of_the_largest_sizes(ctx, new, cu, lens):
    """2^30 token slots, rows of 2^30 positions: sums of two such numbers do not fit in 32 bits."""
    page, pages, T = 1 << 20, 1024, 1 << 30
    op = ez.PagedPlanOp(2, T, pages, page, pages, backend="cuda")
    table = (torch.arange(2 * pages, dtype=I32, device=DEV) % pages).view(2, pages)  # (the rows share pages)
    free = (torch.arange(2 * pages, dtype=I32, device=DEV) % pages).flip(0).contiguous()  # taken in the order of their numbers
    held = [-(-c // page) for c in ctx]
    first = free.numel()
    plan = op(ints(*ctx), ints(*new), table, free, ints(first))
    assert plan.cu_tokens.tolist() == cu and plan.seq_lens.tolist() == lens
    need = [-(-n // page) for n in lens]
    assert int(plan.free_count) == first - sum(need) + sum(held)
    taken = 0
    for b in range(2):
        for j in (held[b], need[b] - 1):
            if held[b] <= j < need[b]:
                assert int(table[b, j]) == (taken + j - held[b]) % pages
        taken += need[b] - held[b]
        lo, hi = cu[b], cu[b + 1]
        for at in range(lo, hi, 1 << 28):
            pos = torch.arange(ctx[b] + at - lo, ctx[b] + min(at + (1 << 28), hi) - lo, device=DEV)
            part = slice(at, at + pos.numel())
            assert torch.equal(plan.positions[part].long(), pos)
            slot = table[b].long()[(pos // page).clamp(max=pages - 1)] * page + pos % page
            assert torch.equal(plan.slots[part].long(), torch.where(pos < pages * page, slot, -1))
    assert (plan.positions[cu[2] :] == -1).all() and (plan.slots[cu[2] :] == -1).all()


def test_steps_without_tokens():
    """No rows in, no rows out; nothing is written, and what would be refused otherwise still is."""
    op = ez.LinearOp(4, 24, 64, backend="cuda", bias=True, residual=True, activation="swiglu")
    X, W, b, r = op.gen_data()
    out = op(X[:0], W, bias=b, residual=r[:0])
    assert out.shape == (0, 24) and out.dtype == BF16 and out.is_cuda
    given = torch.empty(0, 24, device=DEV, dtype=BF16)
    assert op(X[:0], W, bias=b, residual=r[:0], out=given) is given
    with pytest.raises(ValueError, match="W must have shape"):
        op(X[:0], W[:5], bias=b, residual=r[:0])
    with pytest.raises(ValueError, match="residual must have shape"):
        op(X[:0], W, bias=b, residual=r)

    for sections in (None, (12, 10, 10)):
        op = ez.PagedQkNormRopeOp(4, 8, 64, 50, 64, 3, backend="cuda", num_kv_heads=2, sections=sections)
        qkv, qw, kw, cos, sin, positions, slots, K, V = op.gen_data()
        K0, V0 = K.clone(), V.clone()
        out = op(qkv[:0], qw, kw, cos, sin, positions[:, :0].contiguous(), slots[:0], K, V)
        assert out.shape == (0, 8, 64) and torch.equal(K, K0) and torch.equal(V, V0)
        with pytest.raises(ValueError, match="slots must have shape"):
            op(qkv[:0], qw, kw, cos, sin, positions[:, :0].contiguous(), slots, K, V)

    Q, K, V, table, _, _ = attn_data([4], [0], 8, 2, 128, 64)
    op = ez.AttnPromptOp(1, 4, 8, 128, table.shape[1], 64, backend="cuda", num_kv_heads=2)
    out = op(Q[:0], K, V, table, ints(4), ints(0, 0))
    assert out.shape == (0, 8, 128) and out.dtype == BF16
    with pytest.raises(ValueError, match="page_table must have shape"):
        op(Q[:0], K, V, table[:, :1].contiguous(), ints(4), ints(0, 0))
    with pytest.raises(ValueError):
        op(Q, K[:0], V[:0], table, ints(4), ints(0, 4))
    with pytest.raises(ValueError, match="free_pages is empty"):
        plan = ez.PagedPlanOp(1, 4, 2, 64, 4, backend="cuda")
        plan(ints(0), ints(1), torch.zeros(1, 2, dtype=I32, device=DEV), ints(), ints(0))


@pytest.mark.parametrize("M,N", [(5, 4000), (40, 1999), (100, 1999), (700, 2048), (700, 2001)])
@pytest.mark.parametrize("act", ["silu", "gelu", "swiglu"])
def test_linear_activations_in_their_tails(M, N, act):
    """Relative bounds down to where the results vanish; the arguments are exact (a bf16 value times a power of two).  In units of
    2^-23: silu's exponent x log2(e) is off by two roundings, |x| log2(e), which makes |x| of e^-x; ex2 2, rcp 1, sum and product 1
    (times one more product in swiglu, half a unit).  gelu's exponent has three roundings of x^2 log2(e) / 2, which make 3/4 x^2;
    the fit 3.3, t = rcp(..) 2 times the condition of t P(t) (below 2.5), its seven fma 4, ex2 2, products 2.  Behind that: flushed."""
    low = -87.0 if act != "gelu" else -12.5
    op = ez.LinearOp(M, N, 8, backend="cuda", activation=act, out_dtype=torch.float32)
    X, W = torch.zeros(M, 8, device=DEV, dtype=BF16), torch.zeros(op.weight_rows, 8, device=DEV, dtype=BF16)
    X[:, 0] = 2.0 ** -(torch.arange(M, device=DEV) % 5)
    W[:N, 0] = torch.linspace(-100.0 if act != "gelu" else -16.0, 30.0, N, device=DEV)
    if act == "swiglu":
        W[N:, 0] = torch.linspace(1.0, 2.0, N, device=DEV)
    out = op(X, W)
    z = X[:, :1].double() @ W[:, 0].double()[None]
    x = z[:, :N]
    if act == "gelu":
        y, units = 0.5 * x * torch.special.erfc(-x * 0.5**0.5), 0.75 * x * x + 17
    else:
        y, units = x / (1 + torch.exp(-x)), x.abs() + 5
        if act == "swiglu":
            y = y * z[:, N:]
    # below `low` the results are smaller than 2^-118 (87 e^-87 times a factor of up to 2) and 2^-114 (12.5 erfc(12.5 / sqrt 2) / 2)
    tol = torch.where(x < low, 2.0**-117 if act != "gelu" else 2.0**-113, units * 2**-23 * y.abs() + 2.0**-149)
    close(out, y, tol)


@pytest.mark.parametrize("new,ctx,H,NKV,D", [([4096], [0], 32, 8, 128), ([8191], [0], 8, 2, 128), ([4097], [0], 32, 8, 64),
                                             ([8192], [0], 4, 4, 64), ([700, 2500, 1], [5000, 3001, 9000], 16, 4, 128),
                                             ([1100, 1, 2300], [6000, 4000, 77], 14, 2, 64), ([939, 313, 626], [0, 0, 0], 8, 8, 64)])
def test_attn_long_prompts(new, ctx, H, NKV, D):
    """Thousands of tokens per row: many units per CTA, cut at both ends of a share, of both head sizes."""
    attn_case(new, ctx, H, NKV, D, 256)
