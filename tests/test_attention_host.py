"""CPU tests of the attention operators: what the entry points refuse (Python and C), the binding's structures, the oracle's
gradients against differences, the dropout masks' statistics."""
import ctypes
import math
import os
import re
import subprocess
import sys

import numpy as np
import pytest
import torch

from conftest import ROOT
from oracle import attention_oracle as ao


def qkv(B=2, Lq=3, Lk=5, Hq=4, Hk=2, D=16, dtype=torch.float32):
    return torch.zeros(B, Lq, Hq, D, dtype=dtype), torch.zeros(B, Lk, Hk, D, dtype=dtype), torch.zeros(B, Lk, Hk, D, dtype=dtype)


def test_structures_match_the_header():
    from pstl_diffusion_policy_amd import ffi
    header = re.sub(r"/\*.*?\*/", " ", open(os.path.join(ROOT, "include", "pstl_hip.h")).read(), flags=re.S)
    for name, cls in (("pstl_attn_mat", ffi.AttnMat), ("pstl_qk_rope", ffi.QkRope), ("pstl_attn", ffi.Attn)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), header, flags=re.S).group(1)
        fields, want = [], []
        for decl in [d.strip() for d in body.split(";") if d.strip()]:
            decl = decl.replace("const ", "")
            ctype = re.match(r"\w+", decl).group(0)
            for var in decl[len(ctype):].split(","):
                var = var.strip()
                fields.append(var.lstrip("* "))
                want.append(ctypes.c_void_p if "*" in var else {"int32_t": ctypes.c_int32, "float": ctypes.c_float,
                            "uint64_t": ctypes.c_uint64, "int64_t": ctypes.c_int64, "pstl_attn_mat": ffi.AttnMat}[ctype])
        assert [(n, t) for n, t in cls._fields_] == list(zip(fields, want)), name
    from pstl_diffusion_policy_amd import attention as A
    for packed, cls in ((A._ATTN, ffi.Attn), (A._ROPE, ffi.QkRope)):      # the bytes attention.py hands over
        flat = [t for f in cls._fields_ for t in (f[1]._fields_ if f[1] is ffi.AttnMat else [f])]
        assert packed.size == ctypes.sizeof(cls) and len(packed.unpack(bytes(packed.size))) == len(flat)
        values = list(range(1, len(flat) + 1))
        a = cls.from_buffer_copy(packed.pack(*values))
        got = []
        for n, t in cls._fields_:
            x = getattr(a, n)
            got += [getattr(x, m) for m, _ in x._fields_] if t is ffi.AttnMat else [x]
        assert got == values


@pytest.mark.parametrize("change, error, text", [
    (dict(q=torch.zeros(2, 3, 4, 16, dtype=torch.float64)), TypeError, "float32, bfloat16 or float16"),
    (dict(q=[1]), TypeError, "must be a tensor"),
    (dict(q=torch.zeros(2, 3, 64)), ValueError, "must be \\(B, L, H, D\\)"),
    (dict(k=torch.zeros(2, 5, 2, 16, dtype=torch.float16)), TypeError, "the queries are"),
    (dict(k=torch.zeros(2, 5, 3, 16)), ValueError, "k and v must be"),
    (dict(k=torch.zeros(2, 5, 3, 16), v=torch.zeros(2, 5, 3, 16)), ValueError, "must divide"),
    (dict(v=torch.zeros(2, 4, 2, 16)), ValueError, "k and v must be"),
    (dict(k=torch.zeros(3, 5, 2, 16)), ValueError, "k and v must be"),
    (dict(q=torch.zeros(2, 3, 4, 12), k=torch.zeros(2, 5, 2, 12), v=torch.zeros(2, 5, 2, 12)), ValueError, "multiple of 8"),
    (dict(q=torch.zeros(2, 3, 4, 136), k=torch.zeros(2, 5, 2, 136), v=torch.zeros(2, 5, 2, 136)), ValueError, "up to 128"),
    (dict(key_mask=torch.zeros(2, 5)), TypeError, "bool or uint8"),
    (dict(key_mask=torch.zeros(2, 4, dtype=torch.bool)), ValueError, "key_mask must be"),
    (dict(key_mask=torch.zeros(5, 2, dtype=torch.bool).t()), ValueError, "consecutive"),
    (dict(q_lens=torch.zeros(2, dtype=torch.int64)), TypeError, "int32"),
    (dict(k_lens=torch.zeros(3, dtype=torch.int32)), ValueError, "k_lens must be"),
    (dict(dropout_p=1.0), ValueError, "\\[0, 1\\)"),
    (dict(dropout_p=-0.1), ValueError, "\\[0, 1\\)"),
    (dict(dropout_p=float("nan")), ValueError, "\\[0, 1\\)"),
    (dict(dropout_p=0.001), ValueError, "1/256"),
    (dict(dropout_p=0.9999), ValueError, "1/256"),
    (dict(), RuntimeError, "on the GPU"),
])
def test_attention_refuses(change, error, text):
    from pstl_diffusion_policy_amd import attention as A
    q, k, v = qkv()
    kw = dict(q=q, k=k, v=v)
    kw.update(change)
    with pytest.raises(error, match=text):
        A.attention(kw.pop("q"), kw.pop("k"), kw.pop("v"), **kw)


def test_scale_seed_and_layout_checks():
    from pstl_diffusion_policy_amd import attention as A
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            A._attn_scale(bad, 16)
    dev = torch.device("cpu")
    assert A._seed(-1, dev) == (2 ** 64 - 1, None) and A._seed(2 ** 64 + 5, dev) == (5, None)
    for bad in (1.5, None, True, "1"):
        with pytest.raises(TypeError, match="seed"):
            A._seed(bad, dev)
    for bad in (torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int64), torch.zeros(3)):
        with pytest.raises(TypeError, match="seed tensor"):
            A._seed(bad, dev)
    with pytest.raises(ValueError, match="device"):
        A._seed(torch.zeros(1, dtype=torch.int64), torch.device("meta"))
    assert A._seed(torch.zeros(4), dev)[1] is not None
    base = torch.zeros(2, 3, 4, 24, dtype=torch.bfloat16)
    assert A._aligned(base) and A._aligned(base.transpose(1, 2)) and A._aligned(base[:, :, 1:]) and A._aligned(base[..., 8:16])
    assert not A._aligned(base[..., 4:12])                # rows start 8 bytes past a 16-byte border
    assert not A._aligned(base.transpose(2, 3))           # elements of a row are apart
    assert not A._aligned(torch.zeros(2, 3, 4, 12, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="contiguous"):
        A._check_aligned("q", base[..., 4:12])
    one = torch.zeros(200).as_strided((1, 4, 1, 16), (3, 16, 5, 1))      # strides of dimensions of size 1 mean nothing
    assert one.is_contiguous() and A._aligned(one) and A._mat(one)[1:] == (0, 16, 0)
    g = torch.ones((), dtype=torch.bfloat16).expand(2, 3, 4, 24)     # what sum().backward() hands over
    assert A._aligned(A._gradient(g, base))
    assert A._aligned(A._gradient(base.flatten()[4:52].view(1, 1, 6, 8), base))


@pytest.mark.parametrize("change, error, text", [
    (dict(k=torch.zeros(2, 4, 2, 32)), ValueError, "share B, L and D"),
    (dict(q=torch.zeros(2, 3, 4, 20), k=torch.zeros(2, 3, 2, 20)), ValueError, "multiple of 8"),
    (dict(q_weight=torch.ones(32, dtype=torch.bfloat16)), TypeError, "float32"),
    (dict(k_weight=torch.ones(16)), ValueError, "k_weight must be"),
    (dict(positions=torch.zeros(3, dtype=torch.int32)), TypeError, "int64"),
    (dict(positions=torch.zeros(2, dtype=torch.int64)), ValueError, "positions must be"),
    (dict(inv_freq=torch.ones(16)), TypeError, "float64"),
    (dict(inv_freq=torch.ones(4, dtype=torch.float64)), ValueError, "multiple of 16"),
    (dict(inv_freq=torch.ones(24, dtype=torch.float64)), ValueError, "multiple of 16"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(), RuntimeError, "on the GPU"),
])
def test_qk_norm_rope_refuses(change, error, text):
    from pstl_diffusion_policy_amd import attention as A
    kw = dict(q=torch.zeros(2, 3, 4, 32), k=torch.zeros(2, 3, 2, 32), q_weight=torch.ones(32), k_weight=torch.ones(32),
              positions=torch.arange(3), inv_freq=A.rope_frequencies(32))
    kw.update(change)
    with pytest.raises(error, match=text):
        A.qk_norm_rope(**kw)
    with pytest.raises(ValueError, match="multiple of 16"):
        A.rope_frequencies(24)


def test_dropout_refuses():
    from pstl_diffusion_policy_amd import attention as A
    x = torch.zeros(3, 4)
    for kw, error, text in ((dict(p=1.5), ValueError, "p must be"), (dict(p=float("nan")), ValueError, "p must be"),
                            (dict(offset=-1), ValueError, "offset"), (dict(offset=1.0), ValueError, "offset"),
                            (dict(residual=torch.zeros(3, 4, dtype=torch.float16)), TypeError, "residual is"),
                            (dict(residual=torch.zeros(4)), ValueError, "residual must be"),
                            (dict(seed=1.0), TypeError, "seed"), (dict(), RuntimeError, "on the GPU")):
        args = dict(p=0.5, seed=1)
        args.update(kw)
        with pytest.raises(error, match=text):
            A.dropout_add(x, **args)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        A.dropout_add(x.double(), 0.5, seed=1)


def c_attn(**kw):
    """A pstl_attn that passes every check (its addresses are never read on the host)."""
    from pstl_diffusion_policy_amd import ffi
    m = (1 << 20, 640, 64, 16)
    d = dict(dtype=0, B=2, Lq=10, Lk=10, Hq=4, Hk=2, D=16, causal=0, scale=0.25, dropout_256=0, q=m, k=m, v=m, o=m, dout=m, dq=m, dk=m,
             dv=m, lse=1 << 20, work=1 << 20)
    d.update(kw)
    return ffi.Attn(**d)


@pytest.mark.parametrize("kw, code", [
    (dict(dtype=3), -2), (dict(B=-1), -1), (dict(Lq=-1), -1), (dict(Hk=0), -1), (dict(Hq=3), -2), (dict(D=12), -2), (dict(D=136), -2),
    (dict(D=0), -2), (dict(scale=0.0), -1), (dict(scale=float("nan")), -1), (dict(dropout_256=256), -1), (dict(dropout_256=-1), -1),
    (dict(q=(0, 640, 64, 16)), -1), (dict(q=((1 << 20) + 8, 640, 64, 16)), -1), (dict(k=(1 << 20, 640, 66, 16)), -1),
    (dict(dtype=1, v=(1 << 20, 640, 64, 12)), -1), (dict(o=(0, 0, 0, 0)), -1), (dict(Lk=1 << 30), -2), (dict(Lq=1 << 30), -2),
    (dict(Lq=1 << 25, Hq=64, Hk=1), -2),
])
def test_c_entry_points_refuse_bad_attention_calls(kw, code):
    from pstl_diffusion_policy_amd import ffi
    L = ffi.lib()
    a = c_attn(**kw)
    assert L.pstl_attention(ctypes.byref(a), None) == code
    assert L.pstl_attention_backward(ctypes.byref(a), None) == code


def test_c_entry_points_refuse_missing_buffers_and_accept_empty_calls():
    from pstl_diffusion_policy_amd import ffi
    L = ffi.lib()
    assert L.pstl_attention(None, None) == -1 and L.pstl_attention_backward(None, None) == -1
    for name in ("dout", "dq", "dk", "dv"):
        assert L.pstl_attention_backward(ctypes.byref(c_attn(**{name: (0, 0, 0, 0)})), None) == -1
    assert L.pstl_attention_backward(ctypes.byref(c_attn(lse=None)), None) == -1
    assert L.pstl_attention_backward(ctypes.byref(c_attn(work=None)), None) == -1
    split = c_attn(B=1, Lq=1, Lk=100000, work=None)
    assert L.pstl_attention_work_floats(ctypes.byref(split)) > 0 and L.pstl_attention(ctypes.byref(split), None) == -1
    none = (0, 0, 0, 0)
    empty = c_attn(B=0, q=none, k=none, v=none, o=none, dout=none, dq=none, dk=none, dv=none, lse=None, work=None)
    assert L.pstl_attention(ctypes.byref(empty), None) == 0 and L.pstl_attention_backward(ctypes.byref(empty), None) == 0
    assert L.pstl_attention_work_floats(ctypes.byref(c_attn(D=12))) == 0
    m = (1 << 20, 640, 64, 16)
    rope = dict(dtype=0, B=2, L=10, Hq=4, Hk=4, D=16, rot=16, eps=1e-6, q=m, k=m, yq=m, yk=m, dyq=m, dyk=m, dq=m, dk=m, wq=1 << 20,
                wk=1 << 20, positions=1 << 20, inv_freq=1 << 20, dwq=1 << 20, dwk=1 << 20, work=1 << 20)
    for kw, code in ((dict(D=20), -2), (dict(rot=8), -2), (dict(rot=32), -2), (dict(D=264), -2), (dict(dtype=-1), -2), (dict(eps=-1.0), -1),
                     (dict(wq=None), -1), (dict(wk=(1 << 20) + 4), -1), (dict(positions=None), -1), (dict(q=none), -1), (dict(Hq=0), -1)):
        a = ffi.QkRope(**dict(rope, **kw))
        assert L.pstl_qk_norm_rope(ctypes.byref(a), None) == code, kw
        assert L.pstl_qk_norm_rope_backward(ctypes.byref(a), None) == code, kw
    assert L.pstl_qk_norm_rope_backward(ctypes.byref(ffi.QkRope(**dict(rope, dwq=None))), None) == -1
    assert L.pstl_qk_norm_rope(None, None) == -1
    one = 1 << 20
    for args in ((3, 8, one, None, one, 0, 0, None, 0), (0, -1, one, None, one, 0, 0, None, 0), (0, 8, one, None, one, 65537, 0, None, 0),
                 (0, 8, None, None, one, 0, 0, None, 0), (0, 8, one, None, one, 0, 0, None, -1), (0, 8, one + 2, None, one, 0, 0, None, 0)):
        assert L.pstl_dropout_add(*args, None) in (-1, -2), args
    assert L.pstl_dropout_add(0, 0, None, None, None, 0, 0, None, 0, None) == 0


def test_workspace_sizes_the_binding_takes_for_granted():
    """attention.py asks for the backward workspace, and for none with few keys, without calling the library."""
    from pstl_diffusion_policy_amd import attention as A
    from pstl_diffusion_policy_amd import ffi
    L = ffi.lib()
    for B, Lq, Lk, Hq, Hk in ((1, 1, 1, 1, 1), (3, 17, 900, 12, 4), (2, 0, 5, 2, 2), (70000, 2, 32, 8, 2), (1, 5000, 32, 1, 1)):
        a = c_attn(B=B, Lq=Lq, Lk=Lk, Hq=Hq, Hk=Hk, D=32)
        assert L.pstl_attention_backward_work_floats(ctypes.byref(a)) == B * Hq * Lq + 1
        if Lk <= A.SHORT_KEYS:
            assert L.pstl_attention_work_floats(ctypes.byref(a)) == 0


@pytest.mark.parametrize("B, Lq, Lk, Hq, Hk, D", [(1, 1, 1, 1, 1, 8), (4096, 12, 12, 8, 8, 32), (4, 1, 32768, 16, 2, 128), (1, 5, 1 << 29, 8, 1, 64),
                                                  (1, 1 << 20, 1 << 20, 8, 8, 128), (65536, 1, 33, 64, 8, 64), (3, 100, 65, 6, 3, 80)])
def test_split_calls_cover_every_key_with_bounded_work(B, Lq, Lk, Hq, Hk, D):
    """The workspace of a call that divides its keys: at most a few results per compute unit, however long the keys are."""
    from pstl_diffusion_policy_amd import ffi
    L = ffi.lib()
    a = c_attn(B=B, Lq=Lq, Lk=Lk, Hq=Hq, Hk=Hk, D=D)
    n, R = L.pstl_attention_work_floats(ctypes.byref(a)), Lq * Hq // Hk
    assert n % (B * Hk * R * (D + 2)) == 0
    splits = n // (B * Hk * R * (D + 2))
    assert splits != 1 and splits * B * Hk * ((R + 31) // 32) <= 4 * 256 + B * Hk * ((R + 31) // 32)


@pytest.mark.parametrize("causal, masked, lens, p", [(False, False, False, 0.0), (True, False, True, 0.0), (False, True, True, 0.25)])
def test_oracle_gradients_against_differences(causal, masked, lens, p):
    g = torch.Generator().manual_seed(3)
    B, Lq, Lk, Hq, Hk, D = 2, 4, 6, 4, 2, 8
    t = [torch.randn(B, n, h, D, generator=g, dtype=torch.float64) for n, h in ((Lq, Hq), (Lk, Hk), (Lk, Hk), (Lq, Hq))]
    kw = dict(causal=causal, key_mask=torch.rand(B, Lk, generator=g) < 0.6 if masked else None,
              q_lens=torch.tensor([4, 3], dtype=torch.int32) if lens else None,
              k_lens=torch.tensor([6, 2], dtype=torch.int32) if lens else None, dropout_p=p, seed=77)
    res = ao.attention(*t[:3], dout=t[3], **kw)
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn(t[i].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        hi, lo = ([x + (s * h * d if j == i else 0) for j, x in enumerate(t[:3])] for s in (1, -1))
        diff = ((ao.attention(*hi, **kw)["out"] - ao.attention(*lo, **kw)["out"]) * t[3]).sum() / (2 * h)
        assert abs(float((res[name] * d).sum() - diff)) < 1e-8 * (1 + abs(float(diff))), name


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_norm_rope_gradients_against_differences(interleaved):
    g = torch.Generator().manual_seed(4)
    x, dy = (torch.randn(2, 3, 2, 40, generator=g, dtype=torch.float64) for _ in range(2))
    w = 1 + 0.1 * torch.randn(40, generator=g, dtype=torch.float64)
    pos, f = torch.tensor([[0, 5, 1000000], [7, -3, 2]]), 10000.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    kw = dict(interleaved=interleaved)
    res = ao.qk_norm_rope(x, w, pos, f, dy=dy, **kw)
    assert torch.allclose(res["y"].square().sum(-1), (ao.qk_norm_rope(x, w, pos * 0, f, **kw)["y"]).square().sum(-1))     # a rotation
    dx, dw = torch.randn(x.shape, generator=g, dtype=torch.float64), torch.randn(40, generator=g, dtype=torch.float64)
    h = 1e-6
    val = lambda xx, ww: float((ao.qk_norm_rope(xx, ww, pos, f, **kw)["y"] * dy).sum())
    assert abs((val(x + h * dx, w) - val(x - h * dx, w)) / (2 * h) - float((res["dx"] * dx).sum())) < 1e-6
    assert abs((val(x, w + h * dw) - val(x, w - h * dw)) / (2 * h) - float((res["dw"] * dw).sum())) < 1e-6


def test_dropout_masks_have_the_rate_and_no_structure():
    """Kept fractions within 5 standard deviations, rows and columns too, and neighbours uncorrelated."""
    n = 1 << 18
    for p in (0.1, 0.5):
        keep, gain = ao.dropout_keep(n, p, seed=12345, offset=8 * 1000)
        q = 1 - round(65536 * p) / 65536
        assert abs(gain * q - 1) < 1e-12
        x = keep.double() - q
        sd = math.sqrt(q * (1 - q))
        assert abs(float(x.mean())) < 5 * sd / math.sqrt(n)
        for lag in (1, 2, 7, 8, 9, 64):
            assert abs(float((x[:-lag] * x[lag:]).mean())) < 5 * sd * sd / math.sqrt(n - lag), lag
    keep, gain = ao.attention_keep(4, 2, 64, 64, 0.25, seed=99)
    x = keep.double() - 0.75
    sd, m = math.sqrt(0.75 * 0.25), x.numel()
    assert gain == 4 / 3 and abs(float(x.mean())) < 5 * sd / math.sqrt(m)
    for dim in (1, 2, 3):
        a, b = x.narrow(dim, 0, x.shape[dim] - 1), x.narrow(dim, 1, x.shape[dim] - 1)
        assert abs(float((a * b).mean())) < 5 * sd * sd / math.sqrt(a.numel()), dim
    other, _ = ao.attention_keep(4, 2, 64, 64, 0.25, seed=100)
    assert abs(float((x * (other.double() - 0.75)).mean())) < 5 * sd * sd / math.sqrt(m)
    # shards of one tensor draw what the whole draws
    whole, _ = ao.dropout_keep(1000, 0.3, seed=5)
    part, _ = ao.dropout_keep(400, 0.3, seed=5, offset=600)
    np.testing.assert_array_equal(whole[600:].numpy(), part.numpy())


def test_forward_plans_cover_every_key_and_row(tmp_path):
    """The choice of the forward kernel, compiled by itself and swept over sizes: every key in one part, every row in one tile, and
    empty calls divide by nothing."""
    exe = str(tmp_path / "attn_plan")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                           os.path.join(ROOT, "tests", "hostsim", "attn_plan_main.cpp"), "-o", exe])
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, (run.returncode, run.stdout, run.stderr)
    assert " 0 failures" in run.stdout


def test_empty_calls_need_no_workspace():
    """No sequence or no query, with more keys than one tile holds.  In a process of its own: a division by zero would end it."""
    code = """
import ctypes, sys
sys.path[:0] = %r
from test_attention_host import c_attn
from pstl_diffusion_policy_amd import ffi
L = ffi.lib()
for dtype in range(3):
    for B, Lq in ((0, 3), (2, 0), (0, 0), (0, 200)):
        for Lk in (0, 5, 32, 33, 100, 128, 256, 300, 100000):
            none = (0, 0, 0, 0)
            a = c_attn(dtype=dtype, B=B, Lq=Lq, Lk=Lk, q=none, o=none, work=None, **({"k": none, "v": none} if B == 0 else {}))
            print(dtype, B, Lq, Lk, flush=True)
            assert L.pstl_attention_work_floats(ctypes.byref(a)) == 0
            assert L.pstl_attention(ctypes.byref(a), None) == 0
print("whole")
""" % [ROOT, os.path.join(ROOT, "tests")]
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.endswith("whole\n"), (run.returncode, run.stdout[-200:], run.stderr[-2000:])


def test_a_tangent_asks_for_a_derivative():
    """Forward mode: a dual tensor has requires_grad False, and the operators, which have no forward-mode formula, must not take it
    for a constant.  (What they then do needs the GPU.)"""
    from torch.autograd import forward_ad
    from pstl_diffusion_policy_amd import attention as A
    x, plain = torch.ones(4), torch.ones(4)
    assert not A._needs_grad(x, None, plain)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.full((4,), 2.0))
        assert not dual.requires_grad
        assert not A._needs_grad(plain, None)
        assert A._needs_grad(plain, None, dual) and A._needs_grad(dual)
        with torch.no_grad():
            assert A._needs_grad(dual)      # (no_grad stops the backward mode only)
    assert not A._needs_grad(x, None, plain)
    assert A._needs_grad(plain.clone().requires_grad_(), None)


@pytest.mark.parametrize("kw", [
    dict(dtype=1, B=1 << 24, Lq=1, Lk=33, Hq=1, Hk=1),             # few rows: a workgroup of 256 per sequence
    dict(dtype=1, B=1 << 23, Lq=64, Lk=33, Hq=2, Hk=2),            # 128-row workgroups
    dict(dtype=1, B=1 << 26, Lq=1, Lk=20, Hq=1, Hk=1),             # up to 32 keys: a wavefront per sequence
    dict(dtype=0, B=1 << 27, Lq=2, Lk=3, Hq=1, Hk=1),              # in pairs
])
def test_calls_past_the_largest_grid_are_refused_before_a_launch(kw):
    """A grid holds fewer than 2^32 threads: such a call is refused by its sizes, whole, and not by a launch that fails half way."""
    from pstl_diffusion_policy_amd import ffi
    L = ffi.lib()
    a = c_attn(D=8, **kw)
    assert L.pstl_attention(ctypes.byref(a), None) == -2
    assert L.pstl_attention_backward(ctypes.byref(a), None) == -2


def test_dropout_past_the_largest_grid_and_backward_by_keys_alone_are_refused():
    from pstl_diffusion_policy_amd import ffi
    L = ffi.lib()
    one = 1 << 20
    assert L.pstl_dropout_add(1, 1 << 35, one, None, one, 0, 0, None, 0, None) == -2
    # few queries, long keys: the queries' grid is small, the keys' is not (16-bit heads over 64 wide: 512 threads a workgroup)
    for dtype, D, Lk in ((1, 8, (1 << 30) - 64), (0, 8, (1 << 30) - 64), (2, 72, (1 << 29) + 64)):
        rc = L.pstl_attention_backward(ctypes.byref(c_attn(dtype=dtype, B=1, Lq=1, Lk=Lk, Hq=8, Hk=8, D=D)), None)
        assert (Lk + 63) // 64 * 8 * (512 if D > 64 else 256) >= 1 << 32 and rc == -2, (dtype, D, rc)


def test_launches_happen_on_the_operands_device(monkeypatch):
    """The guard around every launch: the operand's device is the current one inside, and the caller's again afterwards, also when the
    launch raises."""
    from pstl_diffusion_policy_amd import attention as A
    state = {"device": 0, "switches": 0}

    class Switch:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, state["device"] = state["device"], self.index
            state["switches"] += 1

        def __exit__(self, *exc):
            state["device"] = self.before

    class Operand:
        def __init__(self, index):
            self.get_device = lambda: index

    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["device"])
    monkeypatch.setattr(torch.cuda, "device", Switch)

    @A._device_guard
    def launch(q, extra):
        if extra == "raise":
            raise RuntimeError("refused")
        return state["device"], extra

    assert launch(Operand(0), 5) == (0, 5) and state["switches"] == 0      # (already there: nothing is switched)
    assert launch(Operand(3), 6) == (3, 6) and state == {"device": 0, "switches": 1}
    with pytest.raises(RuntimeError, match="refused"):
        launch(Operand(2), "raise")
    assert state == {"device": 0, "switches": 2}
    for name in ("_rope_launch", "_attn_forward", "_attn_backward", "_dropout_launch"):
        assert getattr(A, name).__qualname__.startswith("_device_guard"), name
