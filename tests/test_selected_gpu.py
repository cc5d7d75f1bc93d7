"""Block means, block selection and attention over selected blocks (GPU) against float64
loops on the CPU (tests/selected_oracle.py, which derives the tolerances)."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests import selected_oracle as so

pytestmark = pytest.mark.gpu


def _normal(gen, *shape, dtype="float32", f=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * f).to(getattr(torch, dtype))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- means -----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("L,bs,H,d", [(1, 16, 1, 8), (130, 64, 3, 64), (257, 32, 2, 128), (100, 128, 5, 96), (63, 16, 2, 20),
                                      (33, 16, 1, 5), (2049, 1024, 1, 64)])
def test_block_means(dtype, L, bs, H, d):
    import jaxmodules_amd as jm

    k = _normal(_gen(L), 3, L, H, d, dtype=dtype)
    lengths = _ints(L, max(L // 2, 1), 0)
    for n in (None, lengths, _ints(L + 5, -3, 1)):
        got = jm.block_means(k, bs, n)
        want = so.means(k, bs, n)
        assert got.dtype == torch.float32
        # one rounding of a float64 sum (whose own error is far below a float32 step)
        assert ((got.cpu().double() - want).abs() <= 2.0 ** -24 * (1 + 1e-6) * want.abs() + 1e-12 * k.double().abs().max().item()).all()


def test_block_means_of_views():
    import jaxmodules_amd as jm

    x = _normal(_gen(1), 2, 3, 100, 64)
    flat = _normal(_gen(2), 2 * 100 * 3 * 64 + 1)
    for k in (x.transpose(1, 2), flat[1:].view(2, 100, 3, 64), x.transpose(1, 2)[..., ::2]):
        assert torch.equal(jm.block_means(k, 16), jm.block_means(k.contiguous(), 16))


@pytest.mark.parametrize("new", [1, 4, 16, 40])
def test_block_means_update_writes_the_touched_blocks_alone(new):
    import jaxmodules_amd as jm

    k = _normal(_gen(3), 5, 100, 2, 64, dtype="bfloat16")
    lengths = _ints(100, 48, 49, 3, 0)
    full = jm.block_means(k, 16, lengths)
    out = torch.full_like(full, 7.0)
    assert jm.block_means(k, 16, lengths, out=out, new=new) is out
    for b, n in enumerate((100, 48, 49, 3, 0)):
        for j in range(full.shape[1]):
            touched = j * 16 < n and (j + 1) * 16 > n - new
            assert torch.equal(out[b, j], full[b, j] if touched else torch.full_like(full[b, j], 7.0)), (b, j)


# ---- selection -------------------------------------------------------------------------


SELECTIONS = [
    # B, N, Hq, Hkv, d, L, bs, count, first, last
    (1, 1, 1, 1, 8, 16, 16, 1, 0, 1), (2, 130, 4, 2, 64, 130, 16, 4, 1, 1), (1, 300, 8, 1, 128, 300, 16, 7, 0, 0),
    (2, 70, 2, 2, 96, 70, 16, 16, 1, 2), (1, 500, 3, 3, 40, 500, 16, 5, 2, 3), (1, 2100, 2, 1, 64, 2100, 16, 9, 1, 1),
    (1, 9, 4, 2, 20, 2500, 16, 33, 1, 1),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("case", SELECTIONS)
@pytest.mark.parametrize("causal", [True, False])
def test_select_blocks(case, causal, dtype):
    import jaxmodules_amd as jm

    B, N, Hq, Hkv, d, L, bs, count, first, last = case
    gen = _gen(N + d)
    q, k = _normal(gen, B, N, Hq, d, dtype=dtype), _normal(gen, B, L, Hkv, d, dtype=dtype)
    m = jm.block_means(k, bs)
    got = jm.select_blocks(q, m, bs, count, is_causal=causal, first=first, last=last)
    assert torch.equal(got.cpu(), so.select(q, m, bs, count, causal, first, last)[0])


@pytest.mark.parametrize("N", [1, 3, 8, 20])
def test_select_for_served_tokens(N):
    import jaxmodules_amd as jm

    gen = _gen(N)
    q, m = _normal(gen, 5, N, 4, 64, dtype="bfloat16"), _normal(gen, 5, 70, 2, 64)
    lengths = _ints(70 * 16, 500, 17, 16, 0)
    starts = lengths - N
    for kw in (dict(starts=starts, lengths=lengths), dict(starts=starts), dict(lengths=lengths),
               dict(lengths=lengths, is_causal=False), dict(starts=_ints(-5, 5000, 0, 1, 2))):
        got = jm.select_blocks(q, m, 16, 6, **kw)
        want = so.select(q, m, 16, 6, kw.get("is_causal", True), 1, 1, kw.get("starts"), kw.get("lengths"))[0]
        assert torch.equal(got.cpu(), want), kw


@pytest.mark.parametrize("nblk", [100, 500, 1900, 5000])
@pytest.mark.parametrize("N", [2, 40])
def test_select_many_blocks_ties_and_odd_values(nblk, N):
    """Every form of the choice; equal means (ties to the lower index), zeros of both
    signs, infinities and NaN."""
    import jaxmodules_amd as jm

    gen = _gen(nblk)
    m = torch.randint(-1, 2, (1, nblk, 1, 8), generator=gen, device="cuda").float()  # few distinct scores
    q = torch.randint(-1, 2, (1, N, 2, 8), generator=gen, device="cuda").float()
    m[0, 7] = -0.0
    for count in (3, 64, nblk // 2 if nblk < 2000 else 999):
        got = jm.select_blocks(q, m, 16, count, is_causal=False)
        assert torch.equal(got.cpu(), so.select(q, m, 16, count, False)[0])
    m[0, 11, 0, 0] = float("nan")
    m[0, 12, 0, 1], m[0, 13, 0, 2] = float("inf"), -float("inf")
    got = jm.select_blocks(q, m, 16, 20, is_causal=False)
    assert torch.equal(got.cpu(), so.select(q, m, 16, 20, False)[0])


def test_select_close_scores():
    """Scores a float32 sum cannot tell apart: means that differ in their last place."""
    import jaxmodules_amd as jm

    gen = _gen(5)
    base = _normal(gen, 1, 1, 1, 64)
    m = base.expand(1, 200, 1, 64).clone()
    step = torch.randint(-3, 4, m.shape, generator=gen, device="cuda")
    m = (m.view(torch.int32) + step.int()).view(torch.float32)
    q = _normal(gen, 1, 50, 2, 64)
    got = jm.select_blocks(q, m, 16, 11, is_causal=False)
    assert torch.equal(got.cpu(), so.select(q, m, 16, 11, False)[0])


def test_select_views():
    import jaxmodules_amd as jm

    gen = _gen(6)
    q, m = _normal(gen, 2, 4, 50, 64, dtype="bfloat16").transpose(1, 2), _normal(gen, 2, 2, 40, 64).transpose(1, 2)
    odd = _normal(gen, 2 * 50 * 4 * 64 + 1, dtype="bfloat16")[1:].view(2, 50, 4, 64)
    for x in (q, odd):
        assert torch.equal(jm.select_blocks(x, m, 16, 5), jm.select_blocks(x.contiguous().clone(), m.contiguous(), 16, 5))


# ---- attention -------------------------------------------------------------------------


def _blocks(gen, B, N, Hkv, count, nblk):
    """Any order, some of them past the query, repeated or -1."""
    return torch.randint(-1, nblk + 1, (B, N, Hkv, count), generator=gen, device="cuda", dtype=torch.int32)


def _check(got, want, dt, top, d, terms, what):
    value, mag = want
    tol = so.tolerance(value, mag, dt, top, d, terms)
    err = (got.detach().cpu().double() - value).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((err / tol)[bad].max()))


SHAPES = [
    # B, N, L, Hq, Hkv, d, bs, count
    (1, 1, 1, 1, 1, 8, 16, 1), (2, 40, 40, 4, 2, 64, 16, 3), (1, 300, 300, 8, 2, 64, 64, 3), (2, 129, 260, 6, 6, 128, 32, 5),
    (1, 700, 700, 4, 1, 128, 64, 6), (1, 200, 500, 3, 1, 80, 128, 3), (1, 150, 600, 2, 2, 64, 256, 2),
    (2, 60, 100, 40, 2, 64, 16, 4), (1, 400, 400, 2, 1, 40, 48, 40), (1, 90, 333, 4, 2, 20, 80, 3), (1, 2300, 260, 2, 1, 64, 64, 2),
    # few of many blocks for many queries of one head: by blocks, not by tiles of queries
    (1, 700, 700, 2, 2, 64, 16, 1), (2, 400, 900, 1, 1, 128, 16, 2), (1, 500, 2000, 2, 1, 96, 16, 1), (1, 300, 4096, 1, 1, 128, 256, 1),
    (1, 300, 2048, 2, 2, 64, 128, 1),
    # more blocks than a workgroup holds the selections of at a time
    (1, 130, 9000, 2, 2, 64, 16, 30), (1, 40, 20000, 1, 1, 64, 16, 200),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(shape, causal, dtype):
    import jaxmodules_amd as jm

    B, N, L, Hq, Hkv, d, bs, count = shape
    gen = _gen(N + L + d)
    f = d ** -0.25
    q, k, v = (_normal(gen, B, n, h, d, dtype=dtype, f=f).requires_grad_() for n, h in ((N, Hq), (L, Hkv), (L, Hkv)))
    do = _normal(gen, B, N, Hq, d, dtype=dtype)
    blocks = _blocks(gen, B, N, Hkv, count, -(-L // bs))
    o = jm.selected_attention(q, k, v, blocks, bs, is_causal=causal)
    assert o.dtype == q.dtype and o.shape == q.shape
    with torch.no_grad():
        assert torch.equal(o, jm.selected_attention(q, k, v, blocks, bs, is_causal=causal))
    ok = so.visible(blocks, N, L, bs, causal, None, None)
    want, top = so.attend(q, k, v, ok, do=do)
    _check(o, want["o"], o.dtype, top, d, count * bs, "o")
    grads = torch.autograd.grad(o, (q, k, v), do)
    for n, g in zip(("dq", "dk", "dv"), grads):
        _check(g, want[n], o.dtype, top, d, max(count * bs, N * Hq // Hkv), n)
    unseen = ~ok.any(2).permute(0, 2, 1)  # [B, L, Hkv]
    assert not grads[1].cpu()[unseen].any() and not grads[2].cpu()[unseen].any()
    empty = ~ok.any(3).permute(0, 2, 1).repeat_interleave(Hq // Hkv, 2)
    assert not o.detach().cpu()[empty].any() and not grads[0].cpu()[empty].any()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("N,Hq,bs,count", [(1, 8, 64, 9), (1, 2, 16, 70), (4, 6, 32, 20), (17, 4, 64, 5), (1, 34, 128, 3)])
def test_served_tokens(N, Hq, bs, count, dtype):
    """The last tokens of ragged sequences in a cache whose unused rest holds NaN."""
    import jaxmodules_amd as jm

    gen = _gen(N + Hq)
    B, L, Hkv, d = 6, 1500, 2, 64
    lengths = _ints(1500, 777, 64, max(N, 17), 1, 0)
    starts = lengths - N
    q = _normal(gen, B, N, Hq, d, dtype=dtype)
    k, v = (_normal(gen, B, L, Hkv, d, dtype=dtype) for _ in range(2))
    for b, n in enumerate(lengths.tolist()):
        k[b, n:], v[b, n:] = float("nan"), float("nan")
    blocks = _blocks(gen, B, N, Hkv, count, -(-L // bs))
    for st in (starts, None):
        causal = st is not None
        o = jm.selected_attention(q, k, v, blocks, bs, starts=st, lengths=lengths, is_causal=causal)
        want, top = so.attend(q, k, v, so.visible(blocks, N, L, bs, causal, st, lengths))
        _check(o, want["o"], o.dtype, top, d, count * bs, "o")


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("bs,N", [(32, 200), (128, 200), (16, 1200)])
def test_odd_values_stay_with_the_queries_that_see_them(dtype, bs, N):
    """NaN and infinities in a token reach no query before it, in any output.  (1200
    queries with their own block alone run by blocks.)"""
    import jaxmodules_amd as jm

    gen = _gen(8)
    own = N > 1000
    hq = 2 if own else 4
    q, k, v, do = (_normal(gen, 1, N, h, 64, dtype=dtype) for h in (hq, 2, 2, hq))
    if own:
        blocks = (torch.arange(N, device="cuda", dtype=torch.int32) // bs)[None, :, None, None].expand(1, N, 2, 1).contiguous()
    else:
        blocks = torch.arange(-(-N // bs), device="cuda", dtype=torch.int32).expand(1, N, 2, -1).contiguous()

    def grads(q, k, v, do):
        x = [t.clone().requires_grad_() for t in (q, k, v)]
        o = jm.selected_attention(*x, blocks, bs)
        return [o.detach(), *torch.autograd.grad(o, x, do)]

    clean = grads(q, k, v, do)
    at = 150
    for which in range(4):
        x = [t.clone() for t in (q, k, v, do)]
        x[which][0, at, 0, 3], x[which][0, at, 0, 5] = float("nan"), float("inf")
        got = grads(*x)
        assert torch.equal(got[0][0, :at], clean[0][0, :at]) and torch.equal(got[1][0, :at], clean[1][0, :at]), which
        # keys behind the token are not seen by it: an odd query or gradient does not reach them
        if which in (0, 3):
            for g, c in zip(got[2:], clean[2:]):
                assert g[0, at + 1:].isfinite().all()
                torch.testing.assert_close(g[0, at + 1:], c[0, at + 1:], rtol=2e-2, atol=1e-5)
        assert not got[0 if which < 3 else 1][0, at].isfinite().all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("d", [64, 128])
def test_odd_values_reach_their_own_columns_alone(dtype, d):
    """NaN and infinities in columns of one value (or key, query, gradient) leave the other
    columns of every output that adds it as they are, and are seen in their own."""
    import jaxmodules_amd as jm

    gen = _gen(15)
    N, at, bs = 130, 70, 64
    q, k, v, do = (_normal(gen, 1, N, 2, d, dtype=dtype) for _ in range(4))
    blocks = torch.arange(3, device="cuda", dtype=torch.int32).expand(1, N, 2, -1).contiguous()
    odd, cols = [3, d - 9], [c for c in range(d) if c not in (3, d - 9)]

    def outputs(v, do):
        x = [t.clone().requires_grad_() for t in (q, k, v)]
        o = jm.selected_attention(*x, blocks, bs)
        return o.detach(), *torch.autograd.grad(o, x, do)

    clean = outputs(v, do)
    w = v.clone()
    w[0, at, 0, odd[0]], w[0, at, 0, odd[1]] = float("nan"), float("inf")
    o = outputs(w, do)[0]
    assert torch.equal(o[..., cols], clean[0][..., cols]) and torch.equal(o[:, :at], clean[0][:, :at])
    assert o[0, at:, 0, odd[0]].isnan().all() and (o[0, at:, 0, odd[1]] == float("inf")).all()
    assert torch.equal(o[:, :, 1], clean[0][:, :, 1])
    w = do.clone()
    w[0, at, 0, odd[0]] = float("nan")
    dv = outputs(v, w)[3]
    assert torch.equal(dv[..., cols], clean[3][..., cols]) and torch.equal(dv[:, at + 1:], clean[3][:, at + 1:])
    assert dv[0, : at + 1, 0, odd[0]].isnan().all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_strides_scale_and_order(dtype):
    import jaxmodules_amd as jm

    gen = _gen(9)
    B, N, H, d, bs = 2, 100, 2, 64, 32
    heads_major = [_normal(gen, B, H, N, d, dtype=dtype).transpose(1, 2) for _ in range(3)]
    flat = _normal(gen, B * N * H * d + 1, dtype=dtype)
    odd = [flat[1:].view(B, N, H, d)] * 3
    one = [_normal(gen, B, N, 1, d, dtype=dtype).expand(B, N, H, d)] * 3
    blocks = _blocks(gen, B, N, H, 3, 4)
    for views in (heads_major, odd, one):
        for scale in (None, -0.3, 0.0):
            res = []
            for fit in (lambda t: t.detach(), lambda t: t.detach().clone(memory_format=torch.contiguous_format)):
                x = [fit(t).requires_grad_() for t in views]
                o = jm.selected_attention(*x, blocks if len(res) == 0 else blocks.flip(3).contiguous(), bs, scale=scale)
                up = torch.ones(1, 1, 1, 1, dtype=o.dtype, device="cuda").expand_as(o)
                res.append([o.detach(), *torch.autograd.grad(o, x, up)])
            for a, b in zip(*res):  # (the order of the slots is the order of the sums)
                torch.testing.assert_close(a, b, rtol=2 ** -6 if dtype == "bfloat16" else 1e-4, atol=2e-2 if dtype == "bfloat16" else 1e-5)
            want, top = so.attend(*views, so.visible(blocks, N, N, bs, True, None, None), scale=0.125 if scale is None else scale)
            _check(res[0][0], want["o"], res[0][0].dtype, top, d, 96, "o")


def test_nothing_to_attend_to():
    import jaxmodules_amd as jm

    for shape_q, shape_k, count in (((0, 4, 2, 64), (0, 4, 2, 64), 1), ((1, 0, 2, 64), (1, 4, 2, 64), 1), ((1, 4, 2, 64), (1, 0, 2, 64), 1),
                                    ((1, 4, 2, 64), (1, 4, 2, 64), 0)):
        q, k, v = (torch.randn(s, device="cuda", requires_grad=True) for s in (shape_q, shape_k, shape_k))
        blocks = torch.zeros((*shape_q[:2], shape_k[2], count), dtype=torch.int32, device="cuda")
        o = jm.selected_attention(q, k, v, blocks, 16)
        assert o.shape == q.shape and not o.any()
        assert all(not g.any() and g.shape == x.shape for g, x in zip(torch.autograd.grad(o, (q, k, v), torch.ones_like(o)), (q, k, v)))
    q, k, v = (torch.randn(1, 20, 2, 64, device="cuda", requires_grad=True) for _ in range(3))
    o = jm.selected_attention(q, k, v, torch.full((1, 20, 2, 3), -1, dtype=torch.int32, device="cuda"), 16)
    assert not o.any() and all(not g.any() for g in torch.autograd.grad(o, (q, k, v), torch.ones_like(o)))


def test_gradients_of_some_inputs():
    import jaxmodules_amd as jm

    gen = _gen(11)
    q, k, v = (_normal(gen, 1, 50, 2, 64) for _ in range(3))
    blocks = _blocks(gen, 1, 50, 2, 2, 4)
    full = [x.clone().requires_grad_() for x in (q, k, v)]
    want = torch.autograd.grad(jm.selected_attention(*full, blocks, 16).sum(), full)
    for i in range(3):
        x = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        assert torch.equal(torch.autograd.grad(jm.selected_attention(*x, blocks, 16).sum(), x[i])[0], want[i])


def test_gradient_against_differences():
    """Central differences of the entry point in float32: the third derivative's h^2 and
    the values' u / h are both below 1e-2 of the gradient here."""
    import jaxmodules_amd as jm

    gen = _gen(12)
    x = [_normal(gen, 1, 48, h, 64, f=0.35).requires_grad_() for h in (4, 2, 2)]
    blocks = _blocks(gen, 1, 48, 2, 2, 3)
    u = _normal(gen, 1, 48, 4, 64)
    loss = lambda *t: (jm.selected_attention(*t, blocks, 16).double() * u).sum()  # noqa: E731
    g = torch.autograd.grad(loss(*x), x)
    with torch.no_grad():
        for _ in range(6):
            a = [_normal(gen, *t.shape) for t in x]
            h = 2.0 ** -6
            num = (loss(*(t + h * b for t, b in zip(x, a))) - loss(*(t - h * b for t, b in zip(x, a)))) / (2 * h)
            terms = [(y.double() * b) for y, b in zip(g, a)]
            assert abs(num - sum(t.sum() for t in terms)) <= 1e-2 * math.sqrt(sum(t.square().sum().item() for t in terms))


def test_run_together_on_a_side_stream_and_captured():
    """norm_rotary -> block_means -> select_blocks -> selected_attention and its backward,
    as a model's layer runs them; every replay of the captured step equals the eager one."""
    import jaxmodules_amd as jm

    gen = _gen(13)
    B, N, Hq, Hkv, d = 1, 300, 4, 2, 64
    q, k, v, do = (_normal(gen, B, N, h, d, dtype="bfloat16") for h in (Hq, Hkv, Hkv, Hq))
    w = torch.ones(d, device="cuda")
    f, scale = jm.rotary_frequencies(d, device="cuda")

    def step():
        x = [t.detach().requires_grad_() for t in (q, k, v, w)]
        a, c = jm.norm_rotary(x[0], x[1], x[3], x[3], inv_freq=f, scale=scale)
        blocks = jm.select_blocks(a, jm.block_means(c, 32), 32, 4)
        o = jm.selected_attention(a, c, x[2], blocks, 32)
        return [blocks, o.detach(), *torch.autograd.grad(o, x, do)]

    want = step()
    ok = so.visible(want[0], N, N, 32, True, None, None)
    a, c = jm.norm_rotary(q, k, w, w, inv_freq=f, scale=scale)
    ref, top = so.attend(a, c, v, ok)
    _check(want[1], ref["o"], torch.bfloat16, top, d, 128, "o")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(side, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        for t in (q, k, v):
            t.copy_(torch.randn_like(t))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, eager)), i


def test_a_token_served_equals_the_prompt():
    """Each token of a sequence from a cache (means kept up, one query) gives what the
    whole prompt gave for it."""
    import jaxmodules_amd as jm

    gen = _gen(14)
    L, bs, d = 150, 16, 64
    q, k, v = (_normal(gen, 2, L, h, d) for h in (4, 2, 2))
    blocks = jm.select_blocks(q, jm.block_means(k, bs), bs, 4)
    prompt = jm.selected_attention(q, k, v, blocks, bs)
    cache_k, cache_v = (torch.full_like(x, float("nan")) for x in (k, v))
    means = torch.zeros((2, -(-L // bs), 2, d), device="cuda")
    for t in range(L):
        cache_k[:, t], cache_v[:, t] = k[:, t], v[:, t]
        lengths = torch.full((2,), t + 1, dtype=torch.int32, device="cuda")
        jm.block_means(cache_k, bs, lengths, out=means, new=1)
        b = jm.select_blocks(q[:, t:t + 1], means, bs, 4, starts=lengths - 1, lengths=lengths)
        assert torch.equal(b[:, 0], blocks[:, t]), t
        o = jm.selected_attention(q[:, t:t + 1], cache_k, cache_v, b, bs, starts=lengths - 1, lengths=lengths)
        torch.testing.assert_close(o[:, 0], prompt[:, t], rtol=1e-4, atol=1e-5)


def test_blocks_changed_before_the_backward_are_an_error():
    import jaxmodules_amd as jm

    x = [torch.randn(1, 40, 2, 64, device="cuda", requires_grad=True) for _ in range(3)]
    blocks = torch.zeros((1, 40, 2, 1), dtype=torch.int32, device="cuda")
    o = jm.selected_attention(*x, blocks, 16)
    blocks.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


# ---- calls at the edges ------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("N,L,H,bs,count", [(150, 200, 2, 32, 3), (150, 700, 1, 16, 1), (20, 300, 4, 64, 2), (5, 200, 2, 16, 4)])
def test_padded_batches_with_gradients(N, L, H, bs, count, dtype):
    """The last N tokens of ragged sequences, some shorter than N or empty: queries before a
    sequence's start see nothing, and NaN behind its end reaches no gradient."""
    import jaxmodules_amd as jm

    gen = _gen(N + L)
    lengths = _ints(L, 77, 16, 0, -5)
    starts = lengths - N
    B, d = len(lengths), 64
    q, do = (_normal(gen, B, N, H, d, dtype=dtype) for _ in range(2))
    k, v = (_normal(gen, B, L, 1, d, dtype=dtype) for _ in range(2))
    for b, n in enumerate(lengths.tolist()):
        k[b, max(n, 0):], v[b, max(n, 0):] = float("nan"), float("nan")
    x = [t.requires_grad_() for t in (q, k, v)]
    blocks = _blocks(gen, B, N, 1, count, -(-L // bs))
    o = jm.selected_attention(*x, blocks, bs, starts=starts, lengths=lengths)
    grads = torch.autograd.grad(o, x, do)
    want, top = so.attend(*x, so.visible(blocks, N, L, bs, True, starts, lengths), do=do)
    _check(o, want["o"], o.dtype, top, d, count * bs, "o")
    for n, g in zip(("dq", "dk", "dv"), grads):
        _check(g, want[n], o.dtype, top, d, max(count * bs, N * H), n)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("N", [4, 100])
@pytest.mark.parametrize("Hq", [3, 5, 33, 40, 64])
def test_groups_of_any_size(Hq, N, dtype):
    import jaxmodules_amd as jm

    gen = _gen(Hq)
    d, bs, L = 64, 16, 120
    x = [_normal(gen, 1, n, h, d, dtype=dtype).requires_grad_() for n, h in ((N, Hq), (L, 1), (L, 1))]
    do = _normal(gen, 1, N, Hq, d, dtype=dtype)
    blocks = _blocks(gen, 1, N, 1, 3, 8)
    starts = _ints(L - N)
    o = jm.selected_attention(*x, blocks, bs, starts=starts)
    want, top = so.attend(*x, so.visible(blocks, N, L, bs, True, starts, None), do=do)
    _check(o, want["o"], o.dtype, top, d, 48, "o")
    for n, g in zip(("dq", "dk", "dv"), torch.autograd.grad(o, x, do)):
        _check(g, want[n], o.dtype, top, d, N * Hq, n)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("bs,count,L", [(1040, 2, 2100), (4096, 1, 300), (1024, 3, 2048), (16, 1024, 500)])
def test_wide_blocks_and_long_selections(bs, count, L, dtype):
    import jaxmodules_amd as jm

    gen = _gen(bs + count)
    N, d = 70, 64
    x = [_normal(gen, 1, n, h, d, dtype=dtype).requires_grad_() for n, h in ((N, 2), (L, 1), (L, 1))]
    do = _normal(gen, 1, N, 2, d, dtype=dtype)
    nblk = -(-L // bs)
    blocks = _blocks(gen, 1, N, 1, count, nblk)
    blocks[0, ::7, 0, 0], blocks[0, 1::7, 0, 0] = -2 ** 31, 2 ** 31 - 1
    for causal in (True, False):
        starts = _ints(L - N) if causal else None
        o = jm.selected_attention(*x, blocks, bs, starts=starts, is_causal=causal)
        want, top = so.attend(*x, so.visible(blocks.clamp(-1, nblk), N, L, bs, causal, starts, None), do=do)
        _check(o, want["o"], o.dtype, top, d, L, "o")
        for n, g in zip(("dq", "dk", "dv"), torch.autograd.grad(o, x, do)):
            _check(g, want[n], o.dtype, top, d, L, n)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("N,bs,count", [(8, 16, 4), (120, 32, 2), (400, 16, 1)])
def test_keys_expanded_over_the_sequence_or_overlapping(N, bs, count, dtype):
    """K one row for all keys (stride 0), V rows of 64 that start 8 apart."""
    import jaxmodules_amd as jm

    gen = _gen(N)
    L, d = 500, 64
    q, do = _normal(gen, 1, N, 2, d, dtype=dtype).requires_grad_(), _normal(gen, 1, N, 2, d, dtype=dtype)
    row = _normal(gen, 1, 1, 2, d, dtype=dtype).requires_grad_()
    flat = _normal(gen, 2 * (8 * L + d), dtype=dtype)
    blocks = _blocks(gen, 1, N, 2, count, -(-L // bs))
    starts = _ints(L - N)
    res = []
    for dense in (False, True):
        k = row.expand(1, L, 2, d)
        v = flat.as_strided((1, L, 2, d), (0, 8, 8 * L + d, 1)).detach()
        if dense:
            k, v = k.clone(memory_format=torch.contiguous_format), v.clone(memory_format=torch.contiguous_format)
        v.requires_grad_()
        o = jm.selected_attention(q, k, v, blocks, bs, starts=starts)
        res.append([o, *torch.autograd.grad(o, (q, row, v), do)])
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_positions_at_the_end_of_int32():
    import jaxmodules_amd as jm

    gen = _gen(3)
    q, k, v = (_normal(gen, 1, n, 2, 64, dtype="bfloat16") for n in (30, 200, 200))
    m = jm.block_means(k, 16)
    far = _ints(2 ** 31 - 1)
    sel = jm.select_blocks(q, m, 16, 3, starts=far)
    assert torch.equal(sel, jm.select_blocks(q, m, 16, 3, is_causal=False))
    assert torch.equal(jm.selected_attention(q, k, v, sel, 16, starts=far), jm.selected_attention(q, k, v, sel, 16, is_causal=False))
    none = jm.select_blocks(q, m, 16, 3, starts=-far)
    assert (none == -1).all()
    assert not jm.selected_attention(q, k, v, sel, 16, starts=-far).any()


@pytest.mark.parametrize("N", [1, 20])
def test_a_cache_of_more_than_2_31_elements(N):
    """The newest keys of one long cache: offsets pass 32 bits in means, scores and attention."""
    import jaxmodules_amd as jm

    gen = _gen(N)
    H, d, bs, L = 8, 128, 16, 1_100_000
    cache = torch.empty((1, L, 2, H, d), dtype=torch.bfloat16, device="cuda")  # K and V of a token side by side
    assert cache.numel() > 2 ** 31
    tail = 40 * bs  # the keys that are filled
    cache[:, L - tail - bs:] = 0.0
    cache[:, L - tail:] = _normal(gen, 1, tail, 2, H, d, dtype="bfloat16")
    k, v = cache[:, :, 0], cache[:, :, 1]
    q = _normal(gen, 1, N, 2 * H, d, dtype="bfloat16")
    lengths, starts = _ints(L), _ints(L - N)
    nblk = L // bs
    means = torch.full((1, nblk, H, d), -1.0, device="cuda")
    jm.block_means(k, bs, lengths, out=means, new=tail)
    torch.testing.assert_close(means[:, nblk - 40:].double().cpu(), so.means(k[:, L - tail:], bs), rtol=2 ** -23, atol=1e-30)
    assert (means[:, : nblk - 40] == -1).all()
    means[:, : nblk - 40] = 0.0  # (scores 0: the best few of the filled ones are above)
    sel = jm.select_blocks(q, means, bs, 6, starts=starts, lengths=lengths, first=0)
    want, score = so.select(q, means[:, nblk - 40:], bs, 6, starts=starts - (L - tail), lengths=lengths - (L - tail), first=0)
    assert (np.sort(score[..., :-2], -1)[..., -5] > 0).all()
    assert torch.equal((sel - (nblk - 40)).cpu(), want)
    sel = nblk - 40 + _blocks(gen, 1, N, H, 6, 40)
    o = jm.selected_attention(q, k, v, sel, bs, starts=starts, lengths=lengths)
    # (-1 of the draw is the block before the filled ones: the oracle's tail holds it too)
    own, more = (sel - (nblk - 41)).clamp(-1, 41), tail + bs
    ref, top = so.attend(q, k[:, L - more:], v[:, L - more:], so.visible(own, N, more, bs, True, starts - (L - more), None))
    _check(o, ref["o"], o.dtype, top, d, 6 * bs, "o")


def test_means_and_choice_of_many_blocks():
    import jaxmodules_amd as jm

    gen = _gen(8)
    L, d = 1_100_000, 8
    k = _normal(gen, 1, L, 1, d, dtype="bfloat16")
    m = jm.block_means(k, 16)
    torch.testing.assert_close(m, k.view(1, L // 16, 16, 1, d).double().mean(2).float(), rtol=2 ** -22, atol=1e-30)
    q = _normal(gen, 1, 3, 2, d, dtype="bfloat16")
    sel = jm.select_blocks(q, m, 16, 5, is_causal=False, first=0, last=0)
    score = torch.einsum("bnd,bjd->bnj", q.double().sum(2), m[:, :, 0].double())
    assert torch.equal(sel[0, :, 0].long(), score[0].topk(5).indices.sort().values)


def test_two_streams_at_once():
    """Calls in flight together on two streams have workspaces of their own."""
    import jaxmodules_amd as jm

    gen = _gen(21)
    sets = []
    for i, (n, bs, count) in enumerate(((2000, 64, 8), (1500, 32, 6))):
        x = [_normal(gen, 1, n, h, 128, dtype="bfloat16").requires_grad_() for h in (8, 2, 2)]
        sets.append((x, _normal(gen, 1, n, 8, 128, dtype="bfloat16"), bs, count, torch.cuda.Stream()))

    def step(x, do, bs, count, _):
        sel = jm.select_blocks(x[0], jm.block_means(x[1], bs), bs, count)
        o = jm.selected_attention(*x, sel, bs)
        return [sel, o.detach(), *torch.autograd.grad(o, x, do)]

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(sets):
            with torch.cuda.stream(s[-1]):
                got[i].append(step(*s))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


def test_two_captured_graphs_replayed_in_turn():
    import jaxmodules_amd as jm

    gen = _gen(22)
    cases = []
    for n, lengths in ((1, _ints(700, 90)), (64, _ints(700, 300))):
        q = _normal(gen, 2, n, 8, 64, dtype="bfloat16")
        k, v = (_normal(gen, 2, 704, 2, 64, dtype="bfloat16") for _ in range(2))
        means = jm.block_means(k, 32, lengths)

        def run(q=q, k=k, v=v, means=means, lengths=lengths, n=n):
            jm.block_means(k, 32, lengths, out=means, new=n)
            sel = jm.select_blocks(q, means, 32, 6, starts=lengths - n, lengths=lengths)
            return sel, jm.selected_attention(q, k, v, sel, 32, starts=lengths - n, lengths=lengths)

        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        cases.append((graph, out, run, (q, k, v), lengths))
    for i in range(3):
        for graph, _, _, x, lengths in cases:
            for t in x:
                t.copy_(torch.randn_like(t))
            lengths.add_(1)
            graph.replay()
        for _, out, run, _, _ in cases:
            assert all(torch.equal(a, b) for a, b in zip(out, run())), i
