"""GPU tests of the attention operators against the float64 oracle.  Tolerances are the oracle's elementwise bounds (half a step of
the element type for each rounding, 2^-24 per float32 operation: oracle/attention_oracle.py)."""
import math

import pytest
import torch

from oracle import attention_oracle as ao

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _library():
    assert torch.cuda.is_available(), "the gpu-marked tests need a GPU"
    from pstl_diffusion_policy_amd import ffi
    ffi.lib()


@pytest.fixture(autouse=True)
def _poisoned_empty(monkeypatch):
    """conftest's fixture of this name for tensors of all three element types: its fill, 2.66e36, is no half-precision number."""
    real_empty, real_empty_like = torch.empty, torch.empty_like

    def poisoned(t):
        if t.is_cuda and t.is_floating_point() and t.numel() > 0:
            t.fill_(6e4 if t.dtype == torch.float16 else 2.66e36)
        return t

    monkeypatch.setattr(torch, "empty", lambda *a, **k: poisoned(real_empty(*a, **k)))
    monkeypatch.setattr(torch, "empty_like", lambda *a, **k: poisoned(real_empty_like(*a, **k)))
    yield


def within(name, got, want, tol):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    got = got.detach().cpu().double()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    err = torch.where(same, torch.zeros_like(want), (got - want).abs())
    bad = ~(err <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %g against a bound of %g" % (
        name, int(bad.sum()), bad.numel(), float(torch.nan_to_num(err, nan=math.inf)[bad].max()), float(tol[bad].min()))


def make(B, Lq, Lk, Hq, Hk, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, n, h, D, generator=g).to(dtype) for n, h in ((Lq, Hq), (Lk, Hk), (Lk, Hk), (Lq, Hq))]


def check_attention(q, k, v, do, gpu=None, train=True, **kw):
    """Forward and backward on the GPU (operands `gpu` if given: views, other layouts) against the oracle."""
    from pstl_diffusion_policy_amd import attention as A
    dtype = q.dtype
    res = ao.attention(q, k, v, dout=do if train else None, bounds_for=dtype, **kw)
    opts = {n: (x.to(DEV) if isinstance(x, torch.Tensor) else x) for n, x in kw.items()}
    qg, kg, vg = gpu or [t.to(DEV) for t in (q, k, v)]
    if train:
        qg, kg, vg = (t.detach().requires_grad_() for t in (qg, kg, vg))
    out, lse = A.attention(qg, kg, vg, return_lse=True, **opts)
    assert out.dtype == dtype
    within("out", out, res["out"], res["tol_out"])
    within("lse", lse, res["lse"], res["tol_lse"])
    if train:
        grads = torch.autograd.grad(out, (qg, kg, vg), do.to(DEV))
        for n, got in zip(("dq", "dk", "dv"), grads):
            assert got.dtype == dtype
            within(n, got, res[n], res["tol_" + n])
    return out


SHAPES = [  # B, Lq, Lk, Hq, Hk, D
    (1, 1, 1, 1, 1, 8), (3, 5, 5, 2, 2, 16), (2, 12, 12, 8, 8, 32), (2, 20, 20, 4, 2, 40), (1, 32, 32, 3, 1, 64), (2, 33, 31, 4, 4, 72),
    (1, 1, 33, 8, 2, 128), (2, 1, 300, 4, 4, 64), (1, 3, 1000, 16, 2, 96), (2, 64, 65, 2, 1, 24), (1, 127, 129, 3, 3, 80),
    (2, 130, 200, 6, 2, 128), (1, 257, 140, 5, 1, 56), (1, 40, 700, 9, 3, 112), (1, 300, 20, 4, 2, 64), (1, 100, 1100, 2, 2, 104),
]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_attention(shape, dtype):
    check_attention(*make(*shape, dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_attention_masked_ragged_causal_dropout(shape, dtype):
    """Everything at once; lengths from zero to full, masks that leave rows empty."""
    B, Lq, Lk = shape[:3]
    g = torch.Generator().manual_seed(1)
    for B in (B, B + 3):
        q, k, v, do = make(B, *shape[1:], dtype, seed=2)
        ql = torch.randint(0, Lq + 1, (B,), generator=g, dtype=torch.int32)
        kl = torch.randint(0, Lk + 1, (B,), generator=g, dtype=torch.int32)
        ql[-1], kl[-1] = Lq, Lk
        mask = torch.rand(B, Lk, generator=g) < 0.6
        check_attention(q, k, v, do, causal=True, key_mask=mask, q_lens=ql, k_lens=kl, dropout_p=0.25, seed=2 ** 63 + 12345)
        check_attention(q, k, v, do, causal=False, key_mask=mask.to(torch.uint8), dropout_p=0.125, seed=7, scale=0.3)
        check_attention(q, k, v, do, causal=True, train=False)


@pytest.mark.parametrize("Lq, Lk", [(50, 50), (64, 64), (65, 65), (128, 128), (129, 129), (10, 90), (90, 10), (200, 333), (333, 200), (1, 77), (2, 2)])
def test_causal_borders(Lq, Lk):
    for Hq, Hk in ((1, 1), (3, 1), (4, 2)):
        check_attention(*make(1, Lq, Lk, Hq, Hk, 32, torch.bfloat16, seed=Lq), causal=True)
        check_attention(*make(1, Lq, Lk, Hq, Hk, 32, torch.float32, seed=Lq), causal=True)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(33, 12, 300, 8, 4, 32), (33, 50, 70, 4, 4, 64), (17, 130, 290, 8, 4, 80), (33, 40, 270, 4, 4, 128)],
                         ids=lambda s: "x".join(map(str, s)))
def test_batches_that_fill_the_chip(shape, dtype):
    """Many sequences: 128-row workgroups, however short; small ones of the same length take 32-row tiles.  With and without masks."""
    B, Lq, Lk = shape[:3]
    g = torch.Generator().manual_seed(Lq * 7 + Lk)
    q, k, v, do = make(B, *shape[1:], dtype, seed=4)
    check_attention(q, k, v, do)
    ql = torch.randint(0, Lq + 1, (B,), generator=g, dtype=torch.int32)
    kl = torch.randint(0, Lk + 1, (B,), generator=g, dtype=torch.int32)
    mask = torch.rand(B, Lk, generator=g) < 0.6
    check_attention(q, k, v, do, causal=True, key_mask=mask, q_lens=ql, k_lens=kl, dropout_p=0.25, seed=77)


def test_long_sequences():
    check_attention(*make(1, 1500, 1500, 2, 1, 64, torch.bfloat16), causal=True)
    check_attention(*make(2, 1, 20000, 8, 2, 128, torch.float16), train=False, k_lens=torch.tensor([20000, 4097], dtype=torch.int32))


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("Lq, Lk", [(0, 5), (5, 0), (0, 0)])
def test_empty_lengths(Lq, Lk, dtype):
    q, k, v, do = make(2, Lq, Lk, 4, 2, 16, dtype)
    out = check_attention(q, k, v, do)
    assert not out.any()
    q, k, v, do = make(0, 3, 4, 4, 2, 16, dtype)
    check_attention(q, k, v, do)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("B, Lq, Lk, D", [(3, 9, 11, 24), (3, 70, 90, 24), (3, 1, 500, 24), (3, 70, 90, 104), (66, 40, 140, 40)])
def test_hidden_places_may_hold_anything(B, Lq, Lk, D, dtype):
    """NaN and infinities in masked keys, behind the lengths, and in the gradients of rows behind them."""
    q, k, v, do = make(B, Lq, Lk, 4, 2, D, dtype)
    g = torch.Generator().manual_seed(5)
    mask = torch.rand(B, Lk, generator=g) < 0.7
    ql = torch.tensor([Lq, max(Lq // 2, 1), 0] * (B // 3), dtype=torch.int32)
    kl = torch.tensor([Lk, Lk // 3, Lk] * (B // 3), dtype=torch.int32)
    bad = [math.nan, math.inf, -math.inf]
    for b in range(B):
        for i in range(Lq):
            if i >= ql[b]:
                q[b, i], do[b, i] = bad[i % 3], bad[(i + 1) % 3]
        for j in range(Lk):
            if j >= kl[b] or not mask[b, j]:
                k[b, j], v[b, j] = bad[j % 3], bad[(j + 1) % 3]
    check_attention(q, k, v, do, key_mask=mask, q_lens=ql, k_lens=kl)
    check_attention(q, k, v, do, key_mask=mask, q_lens=ql, k_lens=kl, causal=True, dropout_p=0.25, seed=3)


def test_all_keys_masked():
    for Lq, Lk in ((4, 6), (100, 140), (1, 400)):
        q, k, v, do = make(2, Lq, Lk, 2, 2, 32, torch.float32)
        mask = torch.ones(2, Lk, dtype=torch.bool)
        mask[1] = False
        out = check_attention(q, k, v, do, key_mask=mask)
        assert not out[1].any()


def test_nan_and_infinity_in_seen_places_show():
    from pstl_diffusion_policy_amd import attention as A
    for Lq, Lk in ((4, 6), (100, 140), (1, 400)):
        q, k, v, _ = (t.to(DEV) for t in make(1, Lq, Lk, 1, 1, 32, torch.float32))
        k[0, 3] = math.nan
        assert A.attention(q, k, v).isnan().all()
        k[0, 3], v[0, 2, 0, 5] = 0.0, math.inf
        out = A.attention(q, k, v)
        assert (out[..., 5] == math.inf).all() and out[..., :5].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
def test_strided_views(dtype):
    """A fused projection, (B, H, L, D) tensors, a cache with more slots than keys, a batch that shares one set of keys."""
    for B, Lq, Lk, Hq, Hk, D in ((2, 9, 9, 4, 2, 32), (2, 100, 100, 4, 2, 32), (3, 1, 150, 8, 2, 64)):
        q, k, v, do = make(B, Lq, Lk, Hq, Hk, D, dtype, seed=8)
        if Lq == Lk:
            fused = torch.cat([t for t in (q, k, v)], 2).to(DEV)
            views = [fused[:, :, :Hq], fused[:, :, Hq:Hq + Hk], fused[:, :, Hq + Hk:]]
            check_attention(q, k, v, do, gpu=views)
        check_attention(q, k, v, do, gpu=[t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for t in (q, k, v)])
        wide = torch.full((B, Lk + 7, Hk, 2 * D), math.nan, dtype=dtype, device=DEV)
        wide[:, :Lk, :, :D], wide[:, :Lk, :, D:] = k.to(DEV), v.to(DEV)
        check_attention(q, k, v, do, gpu=[q.to(DEV), wide[:, :Lk, :, :D], wide[:, :Lk, :, D:]])
        check_attention(q, k[:1].expand_as(k), v[:1].expand_as(v), do, gpu=[q.to(DEV), k[:1].to(DEV).expand_as(k), v[:1].to(DEV).expand_as(v)])


def test_gradient_layouts():
    """What autograd hands over: an expanded gradient (sum), a transposed one, a gradient of a slice."""
    q, k, v, _ = make(2, 40, 50, 4, 2, 24, torch.bfloat16)
    from pstl_diffusion_policy_amd import attention as A

    def grads(f):
        t = [x.to(DEV).requires_grad_() for x in (q, k, v)]
        return torch.autograd.grad(f(A.attention(*t)), t)

    w = torch.randn(2, 4, 40, 24, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    for f, do in ((lambda o: o.sum(), torch.ones_like(q)), (lambda o: (o.transpose(1, 2) * w.to(DEV)).sum(), w.transpose(1, 2)),
                  (lambda o: o[:, 3:5].sum(), torch.nn.functional.pad(torch.ones(2, 2, 4, 24), (0, 0, 0, 0, 3, 35)).to(torch.bfloat16))):
        res = ao.attention(q, k, v, dout=do, bounds_for=torch.bfloat16)
        for n, got in zip(("dq", "dk", "dv"), grads(f)):
            within(n, got, res[n], res["tol_" + n])


def test_gradient_against_differences():
    """Directional differences of the kernel's own forward pass in float32.  With h = 2^-6 the central difference's third-order term
    is below h^2 |d|^3 ~ 1e-3 of the value for directions of unit length; the forward's rounding enters as bound / h."""
    from pstl_diffusion_policy_amd import attention as A
    q, k, v, do = make(1, 70, 90, 4, 2, 32, torch.float32, seed=11)
    t = [x.to(DEV) for x in (q, k, v)]
    W = do.to(DEV).double()
    out, lse = A.attention_forward(*t, causal=True, dropout_p=0.25, seed=5)
    grads = A.attention_backward(do.to(DEV), *t, out, lse, causal=True, dropout_p=0.25, seed=5)
    res = ao.attention(q, k, v, causal=True, dropout_p=0.25, seed=5, bounds_for=torch.float32)
    h, noise = 2.0 ** -6, float((res["tol_out"] * do.abs().double()).sum())
    for i in range(3):
        d = torch.randn(t[i].shape, generator=torch.Generator().manual_seed(i)).to(DEV)
        d /= d.norm()
        hi, lo = ([x + (s * h * d if j == i else 0) for j, x in enumerate(t)] for s in (1, -1))
        val = lambda a: float((A.attention(*a, causal=True, dropout_p=0.25, seed=5).double() * W).sum())
        diff, want = (val(hi) - val(lo)) / (2 * h), float((grads[i].double() * d).sum())
        assert abs(diff - want) <= noise / h + h * h * float(W.norm()), (i, diff, want)


def test_offsets_past_32_bits():
    """A cache whose last keys lie more than 2^31 elements (4 GiB) behind its first."""
    q, k, v, do = make(1, 4, 70, 2, 1, 64, torch.bfloat16, seed=12)
    for Lq in (4, 130):
        q, _, _, do = make(1, Lq, 70, 2, 1, 64, torch.bfloat16, seed=13)
        stride = (1 << 31) // 60 // 8 * 8
        base = torch.empty(70 * stride, dtype=torch.bfloat16, device=DEV)
        gk, gv = base.as_strided((1, 70, 1, 64), (0, stride, 64, 1)), base.as_strided((1, 70, 1, 64), (0, stride, 64, 1), 128)
        gk.copy_(k), gv.copy_(v)
        check_attention(q, k, v, do, gpu=[q.to(DEV), gk, gv])
        del base, gk, gv


def test_more_than_2_31_packed_rows_of_keys_behind_the_length():
    """Causal, 16 heads to a key head, a cache whose slots x heads pass 2^31 with five keys in it: the rest gets zeros."""
    from pstl_diffusion_policy_amd import attention as A
    Lk, G, D = 2 ** 27 + 4096, 16, 8
    g = torch.Generator().manual_seed(5)
    q, do = (torch.randn(1, 2, G, D, generator=g, dtype=torch.float32).to(DEV, torch.bfloat16) for _ in range(2))
    k = torch.zeros(1, 1, 1, D, device=DEV, dtype=torch.bfloat16).expand(1, Lk, 1, D)      # (every slot the same memory)
    kw = dict(causal=True, k_lens=torch.tensor([5], dtype=torch.int32, device=DEV))
    out, lse = A.attention_forward(q, k, k, **kw)
    dq, dk, dv = A.attention_backward(do, q, k, k, out, lse, **kw)
    assert not dk[:, 5:].any() and not dv[:, 5:].any() and not out.any()
    # equal keys: P = 1 / 4 for the first query and 1 / 5 for the second
    want = (do[0, 0].double() / 4 + do[0, 1].double() / 5).sum(0)
    mag = (do[0].double().abs() / 4).sum((0, 1))
    # (P rounded to bfloat16, lse and exp in float32, the result rounded)
    assert ((dv[0, 0, 0].double() - want).abs() <= 3 * 2.0 ** -8 * mag).all()


def test_results_repeat_bit_for_bit():
    from pstl_diffusion_policy_amd import attention as A
    for shape in ((2, 300, 500, 4, 2, 64), (2, 300, 500, 4, 2, 128), (3, 20, 20, 4, 2, 32), (1, 2, 3000, 8, 2, 128)):
        q, k, v, do = (t.to(DEV) for t in make(*shape, torch.bfloat16))
        runs = []
        for _ in range(3):
            out, lse = A.attention_forward(q, k, v, dropout_p=0.25, seed=9)
            runs.append((out, lse) + A.attention_backward(do, q, k, v, out, lse, dropout_p=0.25, seed=9))
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_other_streams_and_two_calls_at_once():
    from pstl_diffusion_policy_amd import attention as A
    q, k, v, do = (t.to(DEV) for t in make(1, 2, 4000, 8, 2, 128, torch.bfloat16))
    want = A.attention(q, k, v)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(A.attention(q, k, v))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    q, k, v, do = (t.to(DEV) for t in make(4, 300, 400, 8, 2, 128, torch.bfloat16))
    out, lse = A.attention_forward(q, k, v, causal=True)
    want = A.attention_backward(do, q, k, v, out, lse, causal=True)
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(A.attention_backward(do, q, k, v, out, lse, causal=True))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


@pytest.mark.parametrize("shape", [(2, 20, 20, 4, 2, 32), (2, 150, 200, 4, 2, 64), (2, 150, 200, 4, 2, 128), (1, 1, 5000, 8, 2, 64)])
def test_captured_step_replays_with_other_seeds(shape):
    """Forward and backward captured in a graph; the seed lives in device memory.  Every replay against the eager result, with eager
    work between the replays; a second graph beside the first."""
    from pstl_diffusion_policy_amd import attention as A
    from pstl_diffusion_policy_amd.engine import DynBlock, GraphCapture
    q, k, v, do = (t.to(DEV) for t in make(*shape, torch.bfloat16))
    seed = torch.zeros(1, dtype=torch.int64, device=DEV)
    dyn = DynBlock(torch.device(DEV, 0))

    def body(s):
        def step():
            out, lse = A.attention_forward(q, k, v, dropout_p=0.25, seed=s)
            return (out,) + A.attention_backward(do, q, k, v, out, lse, dropout_p=0.25, seed=s) + (
                A.dropout_add(out, 0.5, seed=s, residual=q), A.attention(q, k, v))
        return step

    def eager(value):
        return body(value)()

    graphs = [GraphCapture(body(seed)), GraphCapture(body(dyn.dev))]
    x = do.clone()
    for n, value in enumerate((1, 2 ** 40 + 3, 5, -7)):
        seed.fill_(value)
        dyn.set(value)
        want = eager(value)
        x = x * 1.5 + want[0]
        for gr in graphs if n % 2 else graphs[::-1]:
            got = gr.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b), value


def test_captured_backward_while_an_eager_graph_lives():
    """An eager autograd graph of the same leaves is alive while the explicit forward and backward are captured."""
    from pstl_diffusion_policy_amd import attention as A
    from pstl_diffusion_policy_amd.engine import GraphCapture
    leaves = [t.to(DEV).requires_grad_() for t in make(2, 40, 50, 4, 2, 32, torch.float32)[:3]]
    do = make(2, 40, 50, 4, 2, 32, torch.float32)[3].to(DEV)
    alive = A.attention(*leaves, dropout_p=0.25, seed=4)

    def step():
        t = [x.detach() for x in leaves]
        out, lse = A.attention_forward(*t, dropout_p=0.25, seed=4)
        return A.attention_backward(do, *t, out, lse, dropout_p=0.25, seed=4)

    graph = GraphCapture(step)
    alive.backward(do)
    for _ in range(3):
        got = graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b.grad) for a, b in zip(got, leaves))


def test_autograd_refuses_overwritten_masks_and_second_derivatives():
    from pstl_diffusion_policy_amd import attention as A
    q, k, v = (t.to(DEV).requires_grad_() for t in make(2, 4, 6, 2, 2, 16, torch.float32)[:3])
    mask = torch.ones(2, 6, dtype=torch.bool, device=DEV)
    out = A.attention(q, k, v, key_mask=mask)
    mask[0, 0] = False
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()
    seed = torch.ones(1, dtype=torch.int64, device=DEV)
    x = torch.ones(8, device=DEV, requires_grad=True)
    y = A.dropout_add(x, 0.5, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    g, = torch.autograd.grad(A.attention(q, k, v).square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---------------------------------------------------------------------------------------------------------------
ROPE_SHAPES = [(1, 1, 1, 1, 16, 16), (2, 3, 4, 2, 32, 32), (3, 20, 8, 8, 32, 16), (2, 7, 3, 1, 40, 32), (1, 50, 16, 4, 128, 128), (2, 9, 5, 5, 80, 64),
               (4, 1, 16, 2, 128, 64), (1, 3, 2, 2, 256, 256), (1, 2, 2, 1, 248, 16), (3, 700, 3, 3, 64, 64), (1, 9000, 2, 1, 24, 16)]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", ROPE_SHAPES, ids=["x".join(map(str, s)) for s in ROPE_SHAPES])
def test_qk_norm_rope(shape, dtype):
    """Bounds: every output is a float32 value of relative error (D + 16) 2^-24 in the magnitudes it is made of (the sum of squares,
    the reciprocal root, weight, cosine and sine to 2^-23), rounded once to the element type; a weight's gradient adds B L H terms."""
    from pstl_diffusion_policy_amd import attention as A
    B, L, Hq, Hk, D, rot = shape
    u = ao.half_step(dtype)
    g = torch.Generator().manual_seed(D + L)
    for interleaved, far, eps in ((False, 0, 1e-6), (True, 3_000_000_000, 1e-3)):
        fused, dfused = (torch.randn(B, L, Hq + Hk, D, generator=g).to(dtype) for _ in range(2))
        wq, wk = (1 + 0.2 * torch.randn(D, generator=g) for _ in range(2))
        pos = torch.arange(L) + far if interleaved else torch.randint(-5, 200000, (B, L), generator=g)
        f = A.rope_frequencies(rot)
        x = fused.to(DEV).requires_grad_()
        w = [t.to(DEV).requires_grad_() for t in (wq, wk)]
        y = A.qk_norm_rope(x[:, :, :Hq], x[:, :, Hq:], *w, pos.to(DEV), f.to(DEV), eps=eps, interleaved=interleaved)
        d = dfused.to(DEV)
        dx, dwq, dwk = torch.autograd.grad(y, (x, *w), (d[:, :, :Hq], d[:, :, Hq:]))
        for name, sl, yy, ww, dw in (("q", slice(0, Hq), y[0], wq, dwq), ("k", slice(Hq, None), y[1], wk, dwk)):
            res = ao.qk_norm_rope(fused[:, :, sl], ww, pos, f, eps, interleaved, dy=dfused[:, :, sl])
            rel = (D + 16) * ao.E32
            sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
            within("y" + name, yy, res["y"], u * res["y"].abs() + rel * res["mag"] + sub)
            within("dx" + name, dx[:, :, sl], res["dx"], u * res["dx"].abs() + 2 * rel * res["dx_mag"] + sub)
            n = B * L * (Hq if name == "q" else Hk)
            within("dw" + name, dw, res["dw"], (rel + n * ao.E32) * res["dw_mag"])


def test_qk_norm_rope_positions_and_views():
    """Positions as an expanded row, as a column of a wider table, alone; (B, H, L, D) operands; one token of each sequence."""
    from pstl_diffusion_policy_amd import attention as A
    g = torch.Generator().manual_seed(3)
    B, D = 3, 32
    f, w = A.rope_frequencies(D), 1 + 0.1 * torch.randn(D, generator=g)
    table = torch.randint(0, 90000, (B, 40), generator=g)
    views = [(6, lambda t: t[:, 3:9]), (6, lambda t: t[:1, :6].expand(B, 6)), (6, lambda t: t[0, 1:7]), (1, lambda t: t[:, 7:8]),
             (1, lambda t: t[0, :1])]
    for L, view in views:
        x = torch.randn(B, 4, L, D, generator=g)
        q, xg = x.transpose(1, 2), x.to(DEV).transpose(1, 2)
        yq, yk = A.qk_norm_rope(xg, xg[:, :, 1:3], w.to(DEV), w.to(DEV), view(table.to(DEV)), f.to(DEV))
        res = ao.qk_norm_rope(q, w, view(table), f)
        tol = ao.half_step(torch.float32) * res["y"].abs() + (D + 16) * ao.E32 * res["mag"]
        within("yq", yq, res["y"], tol)
        within("yk", yk, res["y"][:, :, 1:3], tol[:, :, 1:3])


def test_strides_of_dimensions_of_size_one():
    from pstl_diffusion_policy_amd import attention as A
    q, k, v, do = make(1, 5, 40, 1, 1, 16, torch.bfloat16, seed=2)
    odd = []
    for t in (q, k, v):
        base = torch.zeros(t.numel() + 64, dtype=t.dtype, device=DEV)
        view = base.as_strided(t.shape, (3, 16, 5, 1))
        view.copy_(t)
        odd.append(view)
    check_attention(q, k, v, do, gpu=odd)


def test_qk_norm_rope_zero_rows_empty_batches_and_repeats():
    from pstl_diffusion_policy_amd import attention as A
    f = A.rope_frequencies(16).to(DEV)
    w = torch.ones(24, device=DEV)
    pos = torch.arange(5, device=DEV)
    z = torch.zeros(2, 5, 3, 24, device=DEV, dtype=torch.bfloat16)
    yq, yk = A.qk_norm_rope(z, z[:, :, :1], w, w, pos, f)
    assert not yq.any() and not yk.any()
    e = torch.zeros(0, 5, 3, 24, device=DEV)
    yq, yk = A.qk_norm_rope(e, e, w, w, pos, f)
    assert yq.shape == (0, 5, 3, 24)
    dq, dk, dwq, dwk = A.qk_norm_rope_backward(e, e, e, e, w, w, pos, f)
    assert dq.shape == e.shape and not dwq.any() and not dwk.any()
    g = torch.Generator().manual_seed(0)
    q, k, dq, dk = (torch.randn(3, 800, 4, 24, generator=g).to(DEV) for _ in range(4))
    runs = [A.qk_norm_rope_backward(dq, dk, q, k, w, w, torch.arange(800, device=DEV), f) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 255, 2048, 2049, 100003])
@pytest.mark.parametrize("offset", [0, 3, 2 ** 35 - 5])
def test_dropout_add(n, offset, dtype):
    """The mask exactly; a value is one product and one sum in float32 and one rounding."""
    from pstl_diffusion_policy_amd import attention as A
    g = torch.Generator().manual_seed(n)
    x, res, dy = (torch.randn(n, generator=g).to(dtype) for _ in range(3))
    u = ao.half_step(dtype)
    for p, seed in ((0.1, 5), (0.5, -1), (0.0, 1), (1.0, 1)):
        keep, gain = ao.dropout_keep(n, p, seed, offset)
        xg, rg = x.to(DEV).requires_grad_(), res.to(DEV).requires_grad_()
        want = torch.where(keep, x.double() * gain, torch.zeros(())) + res.double()
        y = A.dropout_add(xg, p, seed=seed, offset=offset, residual=rg)
        mag = x.double().abs() * gain + res.double().abs()
        within("y", y, want, u * want.abs() + 3 * ao.E32 * mag + 2.0 ** -25)
        dx, dr = torch.autograd.grad(y, (xg, rg), dy.to(DEV))
        assert torch.equal(dr.cpu(), dy) and not dx.cpu()[~keep].any()
        within("dx", dx, torch.where(keep, dy.double() * gain, torch.zeros(())), u * dy.double().abs() * gain + 2 * ao.E32 * dy.double().abs() * gain + 2.0 ** -25)
        plain = A.dropout_add(x.to(DEV), p, seed=seed, offset=offset)
        within("no residual", plain, torch.where(keep, x.double() * gain, torch.zeros(())), u * x.double().abs() * gain + 2 * ao.E32 * mag + 2.0 ** -25)


def test_dropout_odd_views_and_dropped_infinities():
    from pstl_diffusion_policy_amd import attention as A
    base = torch.randn(5000, generator=torch.Generator().manual_seed(1)).to(DEV)
    for view in (base[1:4001], base[3:3003].view(30, 100).t(), base[:0], base.to(torch.bfloat16)[5:2005]):
        keep, gain = ao.dropout_keep(view.numel(), 0.25, 9)
        y = A.dropout_add(view, 0.25, seed=9, residual=view)
        want = torch.where(keep.reshape(view.shape), view.cpu().double() * (gain + 1), view.cpu().double())
        within("y", y, want, (ao.half_step(view.dtype) + 4 * ao.E32) * want.abs())
    x = torch.full((1000,), math.inf, device=DEV)
    keep, _ = ao.dropout_keep(1000, 0.5, 3)
    y = A.dropout_add(x, 0.5, seed=3).cpu()
    assert (y[keep] == math.inf).all() and (y[~keep] == 0).all()


# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
def test_the_operators_together(dtype):
    """An attention sub-layer as a token model trains it: projection -> per-head norm and rotation -> attention with dropout ->
    dropout into the residual stream; outputs and all gradients against the same layer in float64 on the same masks.  Bounds: the
    layer's intermediate values are rounded to the element type at seven places; a relative perturbation of 8 u of every
    intermediate, in the norm of the whole tensor, is what the float64 layer is perturbed by to see how far its own gradients move."""
    from pstl_diffusion_policy_amd import attention as A
    B, L, Hq, Hk, D = 3, 12, 4, 2, 32
    g = torch.Generator().manual_seed(21)
    x0 = torch.randn(B, L, Hq * D, generator=g).to(dtype)
    wp = (torch.randn(Hq * D, (Hq + 2 * Hk) * D, generator=g) / math.sqrt(Hq * D)).to(dtype)
    wo = (torch.randn(Hq * D, Hq * D, generator=g) / math.sqrt(Hq * D)).to(dtype)
    gq, gk = (1 + 0.1 * torch.randn(D, generator=g) for _ in range(2))
    mask = torch.rand(B, L, generator=g) < 0.8
    dy = torch.randn(B, L, Hq * D, generator=g).to(dtype)
    pos = torch.arange(L)
    f = A.rope_frequencies(D)

    def layer_gpu():
        leaves = [t.to(DEV).requires_grad_() for t in (x0, wp, wo, gq, gk)]
        x, w1, w2, a, b = leaves
        h = (x @ w1).view(B, L, Hq + 2 * Hk, D)
        q, k = A.qk_norm_rope(h[:, :, :Hq], h[:, :, Hq:Hq + Hk], a, b, pos.to(DEV), f.to(DEV))
        o = A.attention(q, k, h[:, :, Hq + Hk:], key_mask=mask.to(DEV), dropout_p=0.125, seed=31)
        y = A.dropout_add(o.reshape(B, L, Hq * D) @ w2, 0.25, seed=32, residual=x)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy.to(DEV)))

    def layer_64(noise=0.0, s=0):
        gen = torch.Generator().manual_seed(s)
        wob = lambda t: t * (1 + noise * (2 * torch.rand(t.shape, generator=gen, dtype=torch.float64) - 1)) if noise else t
        leaves = [t.double().requires_grad_() for t in (x0, wp, wo, gq, gk)]
        x, w1, w2, a, b = leaves
        h = wob((x @ w1).view(B, L, Hq + 2 * Hk, D))
        ang = pos.double()[None, :, None, None] * f
        turned = []
        for t, w in ((h[:, :, :Hq], a), (h[:, :, Hq:Hq + Hk], b)):
            z = t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w
            z1, z2 = z[..., :D // 2], z[..., D // 2:]
            turned.append(wob(torch.cat((z1 * ang.cos() - z2 * ang.sin(), z2 * ang.cos() + z1 * ang.sin()), -1)))
        q, k = turned
        k, v = (t.repeat_interleave(Hq // Hk, 2) for t in (k, h[:, :, Hq + Hk:]))
        s_ = torch.einsum("bihd,bjhd->bhij", q, k) / math.sqrt(D)
        p = torch.softmax(s_.masked_fill(~mask[:, None, None], -math.inf), -1)
        keep, gain = ao.attention_keep(B, Hk, L * Hq // Hk, L, 0.125, 31)
        keep = keep.reshape(B, Hk, L, Hq // Hk, L).permute(0, 1, 3, 2, 4).reshape(B, Hq, L, L)
        p = wob(torch.where(keep, p * gain, torch.zeros((), dtype=torch.float64)))
        o = wob(torch.einsum("bhij,bjhd->bihd", p, v))
        z = wob(o.reshape(B, L, Hq * D) @ w2)
        keep, gain = ao.dropout_keep(z.numel(), 0.25, 32)
        y = torch.where(keep.reshape(z.shape), z * gain, torch.zeros((), dtype=torch.float64)) + x
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy.double()))

    got, want = layer_gpu(), layer_64()
    u = ao.half_step(dtype)
    moved = [layer_64(8 * u, s) for s in range(4)]
    for i, name in enumerate(("y", "dx", "dwp", "dwo", "dgq", "dgk")):
        err = float((got[i].cpu().double() - want[i]).norm())
        bound = max(float((m[i] - want[i]).norm()) for m in moved) + 4 * u * float(want[i].norm())
        assert err <= bound, (name, err, bound)


# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("Lk", [33, 100, 300])
@pytest.mark.parametrize("B, Lq", [(0, 3), (2, 0), (0, 0), (0, 200)])
def test_empty_batches_and_queries_with_many_keys(B, Lq, Lk, dtype):
    """No sequence or no query where the keys pass one tile: empty results, and zeros as the gradients of keys nobody asked."""
    for D in (16, 104):
        q, k, v, do = make(B, Lq, Lk, 4, 2, D, dtype)
        check_attention(q, k, v, do)
        check_attention(q, k, v, do, causal=True, key_mask=torch.ones(B, Lk, dtype=torch.bool), dropout_p=0.25, seed=5)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("B, Lq, Lk, Hq, Hk, D", [
    (3, 9, 11, 2, 2, 24), (3, 20, 30, 4, 2, 40), (3, 70, 20, 4, 2, 64),      # up to 32 keys: in pairs, alone, several row tiles
    (3, 2, 500, 4, 2, 24), (3, 5, 2000, 4, 2, 104), (3, 8, 600, 4, 4, 64),   # few rows: one part, and divided keys
    (3, 70, 90, 4, 2, 24), (66, 40, 140, 4, 2, 40), (3, 300, 450, 4, 2, 128)])
@pytest.mark.parametrize("bad", [math.inf, math.nan], ids=["inf", "nan"])
def test_rows_that_see_nothing_are_zeros_beside_visible_infinities(B, Lq, Lk, Hq, Hk, D, bad, dtype):
    """A key or a value that the sequence's other rows see is infinite or NaN: queries behind q_lens, and queries whose causal limit
    leaves them no key, still give exact zeros, lse = -inf and no gradient."""
    from pstl_diffusion_policy_amd import attention as A
    q, k, v, do = make(B, Lq, Lk, Hq, Hk, D, dtype, seed=6)
    ql = torch.tensor([Lq // 2 + 1, Lq, 1] * (B // 3), dtype=torch.int32)
    kl = torch.tensor([Lk, max(Lq // 2, 1), Lk] * (B // 3), dtype=torch.int32).clamp(max=Lk)
    row = torch.arange(Lq)[None]
    behind = row >= ql[:, None]
    assert behind.any()
    for which in (0, 1):
        bk, bv = k.clone(), v.clone()
        (bk, bv)[which][:, 0, :, ::3] = bad
        args = [t.to(DEV) for t in (q, bk, bv)]
        for causal, p in ((False, 0.0), (True, 0.0), (True, 0.25)):
            empty = behind | (row < (ql - kl)[:, None]) if causal else behind
            kw = dict(causal=causal, q_lens=ql.to(DEV), k_lens=kl.to(DEV), dropout_p=p, seed=8)
            out, lse = A.attention_forward(*args, **kw)
            dq, dk, dv = A.attention_backward(do.to(DEV), *args, out, lse, **kw)
            for name, t in (("out", out), ("dq", dq)):
                t = t.cpu()[empty]
                assert (t == 0).all(), (name, which, causal, p, int((t != 0).sum()))
            assert (lse.cpu().permute(0, 2, 1, 3)[empty] == -math.inf).all()
            assert not out.cpu()[~empty].isfinite().all()                                    # (the others show it)
            hidden = torch.arange(Lk)[None] >= kl[:, None]
            assert not dk.cpu()[hidden].any() and not dv.cpu()[hidden].any()


def test_forward_mode_raises_instead_of_dropping_the_tangent():
    from torch.autograd import forward_ad
    from pstl_diffusion_policy_amd import attention as A
    q, k, v, _ = (t.to(DEV) for t in make(2, 4, 6, 2, 2, 16, torch.float32))
    w, pos, f = torch.ones(16, device=DEV), torch.arange(4, device=DEV), A.rope_frequencies(16).to(DEV)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: A.attention(dual(q), k, v), lambda: A.attention(q, k, dual(v), return_lse=True),
                 lambda: A.qk_norm_rope(q, dual(q), w, w, pos, f), lambda: A.qk_norm_rope(q, q, dual(w), w, pos, f),
                 lambda: A.dropout_add(dual(q), 0.5, seed=1), lambda: A.dropout_add(q, 0.5, seed=1, residual=dual(q))]
        for call in calls:
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
                call()
        with torch.no_grad(), pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
            A.attention(dual(q), k, v)
        assert forward_ad.unpack_dual(A.attention(q, k, v)).tangent is None      # (nothing dual goes in)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_weight_gradients_lose_nothing_between_workgroups(dtype):
    """2048 tokens of one head of ones at position 0 (norm 1, no rotation): every workgroup's part of a weight's gradient is one
    gradient, exactly.  Their sum, 2^24 and 2047 small whole numbers, is the float64 sum rounded once; sums in 32 bits lose the ones
    that meet 2^24."""
    from pstl_diffusion_policy_amd import attention as A
    g = torch.Generator().manual_seed(2)
    x = torch.ones(2, 1024, 1, 32).to(DEV, dtype)
    dy = torch.randint(1, 4, (2, 1024, 1, 32), generator=g).float()
    dy[0, 0] = 2.0 ** 24
    w, f = torch.ones(32, device=DEV), A.rope_frequencies(16).to(DEV)
    _, _, dwq, dwk = A.qk_norm_rope_backward(dy.to(DEV, dtype), -dy.to(DEV, dtype), x, x, w, w, torch.zeros(1024, dtype=torch.int64, device=DEV), f, eps=0.0)
    want = dy.double().sum((0, 1, 2)).float()
    assert torch.equal(dwq.cpu(), want) and torch.equal(dwk.cpu(), -want)
