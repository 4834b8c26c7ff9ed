"""Attention over tokens on MI355X: per-head norm with position rotation, softmax attention, dropout -- each with its gradient.

Operators for models of tokens (a scene's ego / neighbour / lane tokens, the time steps of a trajectory, long sequences), beside
the token encoders of engine.Sampler / engine.RectTrainer.  All arithmetic runs in libpstl_hip.so (csrc/attention_kernels.hip,
attention_bwd_kernels.hip, token_kernels.hip); tensors are float32, bfloat16 or float16, sums have 32 bits or more.

  qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq)      rotate(w o x / rms(x)) for queries and keys, one launch
  attention(q, k, v, ...)                                          softmax(scale q k^T) v over padded, ragged, grouped-head batches
  dropout_add(x, p, seed=...)                                      residual + dropout(x); the mask is a function of (seed, element)

The three work under torch.autograd in reverse mode (forward mode raises).  `attention_forward` / `attention_backward`,
`qk_norm_rope_forward` / `qk_norm_rope_backward` and `dropout_backward` are the same calls without autograd, for hosts that
sequence launches themselves (a training step captured in a HIP graph: engine.GraphCapture).  Every call only enqueues launches on
the current stream of the tensors' device -- no synchronisation, no host copy -- and can be captured; call it once before
capturing.

A seed is an int, or a tensor in device memory that the kernels read when they RUN (int64, one element, or the block of an
engine.DynBlock): a captured step draws another mask at each replay.  It must keep its value until the backward pass has run.

There is no CPU path: tensors must live on the GPU and the library must be built (ffi.lib() raises otherwise).
"""
import math
import struct

import torch
from torch.autograd import forward_ad as _forward_ad

from . import ffi

_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
SHORT_KEYS = 32               # up to here one wavefront holds all keys: never a workspace
MAX_HEAD_DIM = 128            # attention (include/pstl_hip.h, PSTL_ATTN_MAX_D)
MAX_ROPE_HEAD_DIM = 256       # qk_norm_rope (PSTL_ROPE_MAX_D)
_MASKS = (torch.bool, torch.uint8)
# pstl_attn and pstl_qk_rope as bytes (ffi.Attn, ffi.QkRope; a ctypes.Structure takes longer to fill than a small call runs)
_ATTN = struct.Struct("@8ifiQQ32q6q")
_ROPE = struct.Struct("@8ifi32q8q")
_raw_stream = torch._C._cuda_getCurrentRawStream      # current_stream().cuda_stream without the two objects around it


# ---------------------------------------------------------------------------------------------------------------
# arguments
# ---------------------------------------------------------------------------------------------------------------
def _rows(name, t, like=None):
    """Checks a (B, L, H, D) operand."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor, got %s" % (name, type(t).__name__))
    if t.dtype not in _CODES:
        raise TypeError("%s must be float32, bfloat16 or float16, got %s" % (name, t.dtype))
    if t.dim() != 4:
        raise ValueError("%s must be (B, L, H, D), got %s" % (name, tuple(t.shape)))
    if like is not None:
        if t.dtype is not like.dtype:
            raise TypeError("%s is %s, the queries are %s" % (name, t.dtype, like.dtype))
        if t.device != like.device:
            raise ValueError("%s is on %s, the queries are on %s" % (name, t.device, like.device))


def _strides(t):
    """Strides of sequence, position and head; that of a dimension of size 1 means nothing and is left out."""
    return [0 if n == 1 else st for n, st in zip(t.shape[:3], t.stride())]


def _aligned(t):
    """Can the kernels read t's rows 16 bytes at a time?"""
    el = t.element_size()
    return t.stride(3) == 1 and t.data_ptr() % 16 == 0 and not any(st * el % 16 for st in _strides(t))


def _on_gpu(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("attention operators run in libpstl_hip.so on the GPU; got a %s tensor" % t.device)


def _check_aligned(name, t):
    if t.numel() and not _aligned(t):
        raise ValueError("%s: the elements of a row must be consecutive and every row 16-byte aligned (shape %s, strides %s, "
                         "address mod 16 = %d); pass %s.contiguous()" % (name, tuple(t.shape), t.stride(), t.data_ptr() % 16, name))


def _mat(t):
    sb, sl, sh, _ = t.stride()
    if (sb | sl | sh) & 7:
        sb, sl, sh = _strides(t)
    return t.data_ptr(), sb, sl, sh


def _good(t, like, el16):
    """Is t (B, L, H, D) of `like`'s type and device, with rows the kernels can read 16 bytes at a time?"""
    sb, sl, sh, sd = t.stride()
    return (t.dtype is like.dtype and t.get_device() == like.get_device() and sd == 1 and not (sb | sl | sh) % el16
            and not t.data_ptr() % 16)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _gradient(t, like):
    """An incoming gradient in a layout the kernels read (autograd hands over expanded and transposed ones)."""
    if t.dtype != like.dtype:
        t = t.to(like.dtype)
    return t if not t.numel() or _aligned(t) else t.contiguous() if not t.is_contiguous() else t.clone()


def _seed(seed, device):
    """(value, device tensor or None)"""
    if isinstance(seed, torch.Tensor):
        dyn = seed.dtype == torch.float32 and seed.numel() == 4
        if not dyn and not (seed.dtype == torch.int64 and seed.numel() == 1):
            raise TypeError("a seed tensor holds one int64 (or is the four float32 words of an engine.DynBlock), got %s %s"
                            % (seed.dtype, tuple(seed.shape)))
        if seed.device != device or not seed.is_contiguous() or seed.data_ptr() % 8:
            raise ValueError("a seed tensor lives on the operands' device (%s), contiguous and 8-byte aligned" % device)
        return 0, seed
    if isinstance(seed, bool) or not isinstance(seed, int):
        raise TypeError("seed must be an int or a device tensor, got %s" % type(seed).__name__)
    return seed & (2 ** 64 - 1), None


def _once(backward):
    """torch.autograd.function.once_differentiable (a second derivative raises), entered only when a graph of the backward pass is
    asked for."""
    guarded = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def _needs_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if getattr(t, "requires_grad", False):
                return True
    if _forward_ad._current_level >= 0:      # inside a dual_level: a tangent goes through the Function as well, which raises
        return any(isinstance(t, torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None for t in tensors)
    return False


def _device_guard(launch):
    """launch(q, ...) with q's device as the current one, if it is not already."""
    def run(q, *args):
        index = q.get_device()
        if index == torch.cuda.current_device():
            return launch(q, *args)
        with torch.cuda.device(index):
            return launch(q, *args)
    return run


# ---------------------------------------------------------------------------------------------------------------
# per-head norm + rotation
# ---------------------------------------------------------------------------------------------------------------
def rope_frequencies(rot_dim, base=10000.0, device=None):
    """The usual table base^(-2 i / rot_dim), i < rot_dim / 2, in float64 (the angles are formed in 64 bits)."""
    if rot_dim < 16 or rot_dim % 16:
        raise ValueError("rot_dim must be a positive multiple of 16, got %d" % rot_dim)
    return float(base) ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)


def _rope_checks(q, k, q_weight, k_weight, positions, inv_freq, eps):
    try:      # everything at once; what is wrong, and how to say it, below
        B, L, Hq, D = q.shape
        dev, el16 = q.get_device(), 4 if q.dtype is torch.float32 else 8
        if (q.dtype in _CODES and dev >= 0 and k.shape[0] == B and k.shape[1] == L and k.shape[2] > 0 and Hq > 0 and k.shape[3] == D
                and not D % 8 and 8 <= D <= MAX_ROPE_HEAD_DIM and _good(q, q, el16) and _good(k, q, el16)
                and q_weight.dtype is torch.float32 and k_weight.dtype is torch.float32 and q_weight.shape == (D,) == k_weight.shape
                and q_weight.get_device() == dev == k_weight.get_device() and q_weight.is_contiguous() and k_weight.is_contiguous()
                and not (q_weight.data_ptr() | k_weight.data_ptr()) % 16
                and positions.dtype is torch.int64 and positions.get_device() == dev and positions.is_contiguous()
                and (positions.shape == (B, L) or positions.shape == (L,))
                and inv_freq.dtype is torch.float64 and inv_freq.get_device() == dev and inv_freq.is_contiguous() and inv_freq.dim() == 1
                and not inv_freq.numel() % 8 and 16 <= 2 * inv_freq.numel() <= D and eps >= 0.0):
            return
    except (AttributeError, TypeError, ValueError, IndexError):
        pass
    _rope_diagnose(q, k, q_weight, k_weight, positions, inv_freq, eps)


def _rope_diagnose(q, k, q_weight, k_weight, positions, inv_freq, eps):
    if not eps >= 0.0:
        raise ValueError("eps must not be negative, got %r" % (eps,))
    _rows("q", q)
    _rows("k", k, q)
    B, L, Hq, D = q.shape
    if k.shape[0] != B or k.shape[1] != L or k.shape[3] != D:
        raise ValueError("q and k must share B, L and D: %s against %s" % (tuple(q.shape), tuple(k.shape)))
    if Hq < 1 or k.shape[2] < 1:
        raise ValueError("q and k need at least one head")
    if D % 8 or not 8 <= D <= MAX_ROPE_HEAD_DIM:
        raise ValueError("the head dimension must be a multiple of 8 up to %d, got %d" % (MAX_ROPE_HEAD_DIM, D))
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w.dtype != torch.float32:
            raise TypeError("%s must be float32 (the framework's parameters are), got %s" % (name, w.dtype))
        if tuple(w.shape) != (D,) or w.stride(0) != 1 or w.device != q.device:
            raise ValueError("%s must be (%d,), contiguous, on %s" % (name, D, q.device))
    if positions.dtype != torch.int64:
        raise TypeError("positions must be int64, got %s" % positions.dtype)
    if tuple(positions.shape) not in ((L,), (B, L)) or positions.device != q.device or (L > 1 and positions.stride(-1) != 1):
        raise ValueError("positions must be (L,) or (B, L) = (%d, %d) with consecutive elements, on %s" % (B, L, q.device))
    if inv_freq.dtype != torch.float64:
        raise TypeError("inv_freq must be float64, got %s" % inv_freq.dtype)
    rot = 2 * inv_freq.numel()
    if inv_freq.dim() != 1 or rot < 16 or rot % 16 or rot > D or not inv_freq.is_contiguous() or inv_freq.device != q.device:
        raise ValueError("inv_freq must be (rot/2,), rot a multiple of 16 up to D = %d, contiguous, on %s" % (D, q.device))
    _on_gpu(q, q_weight, positions, inv_freq)
    for name, t in (("q", q), ("k", k)):
        _check_aligned(name, t)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w.data_ptr() % 16:
            raise ValueError("%s must be 16-byte aligned" % name)


_rope_work = {}      # head dimension -> floats of workspace


@_device_guard
def _rope_launch(q, k, wq, wk, positions, inv_freq, eps, interleaved, dyq=None, dyk=None):
    """The call on checked operands; with the gradients of its outputs: the backward pass."""
    B, L, Hq, D = q.shape
    Hk = k.shape[2]
    dev = q.device
    out_q = torch.empty(q.shape, dtype=q.dtype, device=dev)      # forward's results, or the gradients of q and k
    out_k = torch.empty(k.shape, dtype=q.dtype, device=dev)
    oq, ok = (out_q.data_ptr(), L * Hq * D, Hq * D, D), (out_k.data_ptr(), L * Hk * D, Hk * D, D)
    pos_stride = positions.stride(0) if positions.dim() == 2 else 0
    lib, stream = ffi.lib(), _raw_stream(dev.index)
    if dyq is None:
        rc = lib.pstl_qk_norm_rope(_ROPE.pack(
            _CODES[q.dtype], B, L, Hq, Hk, D, 2 * inv_freq.numel(), 1 if interleaved else 0, eps, 0, *_mat(q), *_mat(k), *oq, *ok,
            0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, wq.data_ptr(), wk.data_ptr(), positions.data_ptr(), pos_stride,
            inv_freq.data_ptr(), 0, 0, 0), stream)
        if rc:
            ffi.check(rc, "qk_norm_rope")
        return out_q, out_k
    dyq, dyk = _gradient(dyq, q), _gradient(dyk, k)
    dwq = torch.empty(D, dtype=torch.float32, device=dev)
    dwk = torch.empty(D, dtype=torch.float32, device=dev)
    if D not in _rope_work:
        _rope_work[D] = lib.pstl_qk_norm_rope_work_floats(bytes(ffi.QkRope(D=D)))
    work = torch.empty(_rope_work[D], dtype=torch.float32, device=dev)
    rc = lib.pstl_qk_norm_rope_backward(_ROPE.pack(
        _CODES[q.dtype], B, L, Hq, Hk, D, 2 * inv_freq.numel(), 1 if interleaved else 0, eps, 0, *_mat(q), *_mat(k),
        0, 0, 0, 0, 0, 0, 0, 0, *_mat(dyq), *_mat(dyk), *oq, *ok, wq.data_ptr(), wk.data_ptr(), positions.data_ptr(), pos_stride,
        inv_freq.data_ptr(), dwq.data_ptr(), dwk.data_ptr(), work.data_ptr()), stream)
    if rc:
        ffi.check(rc, "qk_norm_rope_backward")
    return out_q, out_k, dwq, dwk


def qk_norm_rope_forward(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, interleaved=False):
    """qk_norm_rope without autograd."""
    _rope_checks(q, k, q_weight, k_weight, positions, inv_freq, eps)
    return _rope_launch(q, k, q_weight, k_weight, positions, inv_freq, eps, interleaved)


def qk_norm_rope_backward(dyq, dyk, q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, interleaved=False):
    """(dq, dk, dq_weight, dk_weight) of qk_norm_rope, from its ORIGINAL inputs and the gradients of its outputs."""
    _rope_checks(q, k, q_weight, k_weight, positions, inv_freq, eps)
    for name, t, x in (("dyq", dyq, q), ("dyk", dyk, k)):
        if t.shape != x.shape or t.device != x.device:
            raise ValueError("%s must be %s on %s" % (name, tuple(x.shape), x.device))
    return _rope_launch(q, k, q_weight, k_weight, positions, inv_freq, eps, interleaved, dyq, dyk)


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, positions, inv_freq, eps, interleaved):
        _rope_checks(q, k, wq, wk, positions, inv_freq, eps)
        ctx.save_for_backward(q, k, wq, wk, positions, inv_freq)
        ctx.opts = (eps, interleaved)
        return _rope_launch(q, k, wq, wk, positions, inv_freq, eps, interleaved)

    @staticmethod
    @_once
    def backward(ctx, dyq, dyk):
        return _rope_launch(*ctx.saved_tensors, *ctx.opts, dyq, dyk) + (None,) * 4


def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, interleaved=False):
    """Queries and keys, each normalised per head and rotated by position: rotate(w o x / sqrt(mean(x^2) + eps)) -> (yq, yk).

    q (B, L, Hq, D), k (B, L, Hk, D), D a multiple of 8 up to 256; views of a fused projection are read in place.  q_weight,
    k_weight (D,) float32.  positions (L,) or (B, L) int64.  inv_freq (rot/2,) float64 (rope_frequencies): the first rot elements
    of a head are rotated, pair i = (i, i + rot/2) or, interleaved, (2i, 2i + 1), by positions * inv_freq[i]; the others are only
    normalised.  Differentiable in q, k and the weights."""
    if _needs_grad(q, k, q_weight, k_weight):
        return _QkNormRope.apply(q, k, q_weight, k_weight, positions, inv_freq, eps, interleaved)
    return qk_norm_rope_forward(q, k, q_weight, k_weight, positions, inv_freq, eps, interleaved)


# ---------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------
def _attn_checks(q, k, v, key_mask, q_lens, k_lens, dropout_p):
    """Checks the operands; returns the dropout probability in 256ths."""
    try:      # everything at once; what is wrong, and how to say it, below
        B, Lq, Hq, D = q.shape
        Bk, Lk, Hk, _ = shape = k.shape
        dev, el16 = q.get_device(), 4 if q.dtype is torch.float32 else 8
        n256 = int(round(256 * dropout_p))
        if (q.dtype in _CODES and dev >= 0 and Bk == B and shape[3] == D and v.shape == shape and Hk > 0 and Hq > 0 and not Hq % Hk
                and not D % 8 and 8 <= D <= MAX_HEAD_DIM and _good(q, q, el16) and _good(k, q, el16) and _good(v, q, el16)
                and (dropout_p == 0.0 or 1 <= n256 <= 255)
                and (key_mask is None or (key_mask.dtype in _MASKS and key_mask.get_device() == dev and key_mask.shape == (B, Lk)
                                          and key_mask.is_contiguous()))
                and (q_lens is None or (q_lens.dtype is torch.int32 and q_lens.shape == (B,) and q_lens.get_device() == dev
                                        and q_lens.is_contiguous()))
                and (k_lens is None or (k_lens.dtype is torch.int32 and k_lens.shape == (B,) and k_lens.get_device() == dev
                                        and k_lens.is_contiguous()))):
            return n256
    except (AttributeError, TypeError, ValueError, IndexError):
        pass
    return _attn_diagnose(q, k, v, key_mask, q_lens, k_lens, dropout_p)


def _attn_diagnose(q, k, v, key_mask, q_lens, k_lens, dropout_p):
    _rows("q", q)
    _rows("k", k, q)
    _rows("v", v, q)
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    if tuple(k.shape) != (B, Lk, Hk, D) or v.shape != k.shape:
        raise ValueError("k and v must be (B, Lk, Hk, D) with the queries' B and D: q %s, k %s, v %s"
                         % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if Hk < 1 or Hq < 1 or Hq % Hk:
        raise ValueError("the key heads (%d) must divide the query heads (%d)" % (Hk, Hq))
    if D % 8 or not 8 <= D <= MAX_HEAD_DIM:
        raise ValueError("the head dimension must be a multiple of 8 up to %d, got %d" % (MAX_HEAD_DIM, D))
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8):
            raise TypeError("key_mask must be bool or uint8 (true = visible), got %s" % key_mask.dtype)
        if tuple(key_mask.shape) != (B, Lk) or key_mask.device != q.device or (Lk > 1 and key_mask.stride(1) != 1):
            raise ValueError("key_mask must be (B, Lk) = (%d, %d) with consecutive elements, on %s" % (B, Lk, q.device))
    for name, t in (("q_lens", q_lens), ("k_lens", k_lens)):
        if t is None:
            continue
        if t.dtype != torch.int32:
            raise TypeError("%s must be int32, got %s" % (name, t.dtype))
        if tuple(t.shape) != (B,) or t.device != q.device or not t.is_contiguous():
            raise ValueError("%s must be (B,) = (%d,), contiguous, on %s" % (name, B, q.device))
    if not 0.0 <= dropout_p < 1.0:
        raise ValueError("dropout_p must be in [0, 1), got %r" % (dropout_p,))
    n256 = int(round(256 * dropout_p))
    if dropout_p > 0.0 and not 1 <= n256 <= 255:
        raise ValueError("dropout_p is realised in steps of 1/256, from 1/256 to 255/256; got %r" % (dropout_p,))
    _on_gpu(q)
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check_aligned(name, t)
    return n256


def _attn_scale(scale, D):
    if scale is None:
        return 1.0 / math.sqrt(D)
    scale = float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite, got %r" % (scale,))
    return scale


@_device_guard
def _attn_forward(q, k, v, causal, key_mask, q_lens, k_lens, scale, n256, seed, seed_dev, need_lse):
    """The call on checked operands: (out, lse or None)."""
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    dev = q.device
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    lse = torch.empty((B, Hk, Lq, Hq // Hk), dtype=torch.float32, device=dev) if need_lse else None
    head = (_CODES[q.dtype], B, Lq, Lk, Hq, Hk, D, 1 if causal else 0, scale, n256, seed, _ptr(seed_dev), *_mat(q), *_mat(k), *_mat(v),
            out.data_ptr(), Lq * Hq * D, Hq * D, D, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, _ptr(lse), _ptr(key_mask),
            0 if key_mask is None else key_mask.stride(0), _ptr(q_lens), _ptr(k_lens))
    lib = ffi.lib()
    a = _ATTN.pack(*head, 0)
    if Lk > SHORT_KEYS:      # (few rows against many keys: the call may be split)
        n = lib.pstl_attention_work_floats(a)
        if n:
            work = torch.empty(n, dtype=torch.float32, device=dev)
            a = _ATTN.pack(*head, work.data_ptr())
    rc = lib.pstl_attention(a, _raw_stream(dev.index))
    if rc:
        ffi.check(rc, "attention")
    return out, lse


@_device_guard
def _attn_backward(q, k, v, dout, out, lse, causal, key_mask, q_lens, k_lens, scale, n256, seed, seed_dev):
    """The call on checked operands: (dq, dk, dv)."""
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    dev, dtype = q.device, q.dtype
    dout = _gradient(dout, q)
    dq = torch.empty(q.shape, dtype=dtype, device=dev)
    dk = torch.empty(k.shape, dtype=dtype, device=dev)
    dv = torch.empty(k.shape, dtype=dtype, device=dev)
    work = torch.empty(B * Hq * Lq + 1, dtype=torch.float32, device=dev)      # pstl_attention_backward_work_floats
    rc = ffi.lib().pstl_attention_backward(_ATTN.pack(
        _CODES[dtype], B, Lq, Lk, Hq, Hk, D, 1 if causal else 0, scale, n256, seed, _ptr(seed_dev), *_mat(q), *_mat(k), *_mat(v),
        *_mat(out), *_mat(dout), dq.data_ptr(), Lq * Hq * D, Hq * D, D, dk.data_ptr(), Lk * Hk * D, Hk * D, D, dv.data_ptr(),
        Lk * Hk * D, Hk * D, D, lse.data_ptr(), _ptr(key_mask), 0 if key_mask is None else key_mask.stride(0), _ptr(q_lens),
        _ptr(k_lens), work.data_ptr()), _raw_stream(dev.index))
    if rc:
        ffi.check(rc, "attention_backward")
    return dq, dk, dv


def attention_forward(q, k, v, causal=False, key_mask=None, q_lens=None, k_lens=None, scale=None, dropout_p=0.0, seed=0,
                      need_lse=True):
    """attention without autograd: (out, lse).  lse (B, Hk, Lq, Hq/Hk) float32 is what attention_backward takes (None with
    need_lse=False)."""
    n256 = _attn_checks(q, k, v, key_mask, q_lens, k_lens, dropout_p)
    return _attn_forward(q, k, v, causal, key_mask, q_lens, k_lens, _attn_scale(scale, q.shape[3]), n256, *_seed(seed, q.device),
                         need_lse)


def attention_backward(dout, q, k, v, out, lse, causal=False, key_mask=None, q_lens=None, k_lens=None, scale=None,
                       dropout_p=0.0, seed=0):
    """(dq, dk, dv) of attention, from its inputs, its results and the gradient of `out`.  Deterministic: no atomics."""
    n256 = _attn_checks(q, k, v, key_mask, q_lens, k_lens, dropout_p)
    B, Lq, Hq, _ = q.shape
    Hk = k.shape[2]
    for name, t in (("dout", dout), ("out", out)):
        if t.shape != q.shape or t.device != q.device:
            raise ValueError("%s must be %s on %s" % (name, tuple(q.shape), q.device))
    if (out.dtype != q.dtype or lse.dtype != torch.float32 or tuple(lse.shape) != (B, Hk, Lq, Hq // Hk) or not lse.is_contiguous()
            or lse.device != q.device):
        raise ValueError("out (%s) and lse (float32, %s) are what attention_forward returned" % (q.dtype, (B, Hk, Lq, Hq // Hk)))
    _check_aligned("out", out)
    return _attn_backward(q, k, v, dout, out, lse, causal, key_mask, q_lens, k_lens, _attn_scale(scale, q.shape[3]), n256,
                          *_seed(seed, q.device))


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, key_mask, q_lens, k_lens, scale, dropout_p, seed, want_lse):
        n256 = _attn_checks(q, k, v, key_mask, q_lens, k_lens, dropout_p)
        scale = _attn_scale(scale, q.shape[3])
        seed, seed_dev = _seed(seed, q.device)
        out, lse = _attn_forward(q, k, v, causal, key_mask, q_lens, k_lens, scale, n256, seed, seed_dev, True)
        # (saved, so that autograd refuses a backward pass whose masks, lengths or seed were overwritten in between)
        ctx.save_for_backward(q, k, v, out, lse, key_mask, q_lens, k_lens, seed_dev)
        ctx.opts = (causal, scale, n256, seed)
        if not want_lse:
            return out
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @_once
    def backward(ctx, dout, *_):
        q, k, v, out, lse, key_mask, q_lens, k_lens, seed_dev = ctx.saved_tensors
        causal, scale, n256, seed = ctx.opts
        return _attn_backward(q, k, v, dout, out, lse, causal, key_mask, q_lens, k_lens, scale, n256, seed, seed_dev) + (None,) * 8


def attention(q, k, v, causal=False, key_mask=None, q_lens=None, k_lens=None, scale=None, dropout_p=0.0, seed=0,
              return_lse=False):
    """softmax(scale q k^T over the visible keys) v -> (B, Lq, Hq, D).

    q (B, Lq, Hq, D), k and v (B, Lk, Hk, D): Hk divides Hq (query head h reads key head h // (Hq/Hk)), D a multiple of 8 up to
    128.  Strided views are read in place (rows 16-byte aligned): a cache of Lk slots, a fused projection, (B, H, L, D) tensors
    transposed.  scale: 1/sqrt(D) by default.
    A query sees the keys j < k_lens[b] ((B,) int32; Lk) that key_mask ((B, Lk) bool / uint8, true = visible) shows it and, with
    causal, j <= i + k_lens[b] - q_lens[b]: the ends of the sequences are aligned, so a single new query sees its whole cache.
    Queries i >= q_lens[b] and queries that see nothing give zeros, and no gradient.  What is hidden by the mask or lies behind the
    lengths may hold anything; what only the causal order hides from a query that sees other keys must be finite.
    dropout_p drops probabilities: it is rounded to the nearest 1/256 (0.1 is 26/256 = 0.1016, 0.01 is 3/256 = 0.0117; what would
    round to 0 or 1 raises) and kept ones are scaled by the inverse of the realised keep probability; seed draws the mask.  return_lse: also the log of the softmax's sums, (B, Hq, Lq) float32, without a gradient.
    Differentiable in q, k and v; the backward pass forms the probabilities again and is deterministic."""
    if _needs_grad(q, k, v):
        res = _Attention.apply(q, k, v, causal, key_mask, q_lens, k_lens, scale, dropout_p, seed, return_lse)
        if not return_lse:
            return res
        out, lse = res
    else:
        out, lse = attention_forward(q, k, v, causal, key_mask, q_lens, k_lens, scale, dropout_p, seed, need_lse=return_lse)
        if not return_lse:
            return out
    B, Lq, Hq, _ = q.shape
    return out, lse.permute(0, 1, 3, 2).reshape(B, Hq, Lq)


# ---------------------------------------------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------------------------------------------
@_device_guard
def _dropout_launch(x, residual, p, value, seed_dev, offset):
    if not x.is_contiguous():
        x = x.contiguous()
    if residual is not None and not residual.is_contiguous():
        residual = residual.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    rc = ffi.lib().pstl_dropout_add(_CODES[x.dtype], x.numel(), x.data_ptr(), _ptr(residual), y.data_ptr(), int(round(65536 * p)),
                                    value - 2 ** 64 if value >= 2 ** 63 else value, _ptr(seed_dev), offset,
                                    _raw_stream(x.get_device()))
    if rc:
        ffi.check(rc, "dropout_add")
    return y


def _dropout_checks(x, p, offset, residual):
    if x.dtype not in _CODES:
        raise TypeError("x must be float32, bfloat16 or float16, got %s" % x.dtype)
    if not 0.0 <= p <= 1.0:
        raise ValueError("p must be in [0, 1], got %r" % (p,))
    if isinstance(offset, bool) or not isinstance(offset, int) or not 0 <= offset < 2 ** 62:
        raise ValueError("offset must be an int in [0, 2^62), got %r" % (offset,))
    if residual is not None:
        if residual.dtype != x.dtype:
            raise TypeError("residual is %s, x is %s" % (residual.dtype, x.dtype))
        if residual.shape != x.shape or residual.device != x.device:
            raise ValueError("residual must be %s on %s" % (tuple(x.shape), x.device))


def dropout_backward(dy, p, seed, offset=0):
    """The gradient of dropout_add in x: the same mask on dy (its gradient in the residual is dy itself)."""
    _dropout_checks(dy, p, offset, None)
    seed = _seed(seed, dy.device)
    _on_gpu(dy)
    return _dropout_launch(dy, None, p, *seed, offset)


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, seed_dev, offset):
        ctx.save_for_backward(seed_dev)
        ctx.opts = (p, seed, offset)
        return _dropout_launch(x, residual, p, seed, seed_dev, offset)

    @staticmethod
    @_once
    def backward(ctx, dy):
        p, seed, offset = ctx.opts
        need_x, need_residual = ctx.needs_input_grad[:2]
        dx = _dropout_launch(dy, None, p, seed, ctx.saved_tensors[0], offset) if need_x else None
        return dx, dy if need_residual else None, None, None, None, None


def dropout_add(x, p, seed, offset=0, residual=None):
    """residual + dropout(x): every element of x is dropped with probability p (to 1/65536), the kept ones are scaled by the
    inverse of the realised keep probability.  The mask is a function of (seed, offset + index of the element in x's order) and is
    drawn again by the backward pass.  offset lets several tensors (or the shards of one) share a seed.  residual: x's shape
    and type, or None.  Differentiable in x and residual."""
    _dropout_checks(x, p, offset, residual)
    seed, seed_dev = _seed(seed, x.device)
    _on_gpu(x)
    if _needs_grad(x, residual):
        return _DropoutAdd.apply(x, residual, p, seed, seed_dev, offset)
    return _dropout_launch(x, residual, p, seed, seed_dev, offset)
