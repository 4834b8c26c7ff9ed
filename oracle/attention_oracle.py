"""CPU restatement, in float64, of the attention operators: per-head norm with rotation, attention, dropout -- results, gradients
by the formulas, and elementwise bounds on what a kernel that rounds its operands once may be off by.

Bounds.  u = half a step of the element type, e = 2^-24.  A sum of n products in float32 is off by at most n e times the sum of
their magnitudes, whatever the order.
"""
import math

import numpy as np
import torch

E32 = 2.0 ** -24
M32 = 0xFFFFFFFF


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def philox(c0, c1, c2, c3, seed):
    """Philox4x32-7 on numpy uint64 arrays of 32-bit words -> four arrays."""
    c = [np.asarray(x, dtype=np.uint64) for x in np.broadcast_arrays(c0, c1, c2, c3)]
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(7):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & np.uint64(M32), (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1),
             p0 & np.uint64(M32)]
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    return c


def dropout_keep(n, p, seed, offset=0):
    """(keep (n,) bool, gain)"""
    t = np.arange(n, dtype=np.uint64) + np.uint64(offset)
    g = t // np.uint64(8)
    w = np.stack(philox(g & np.uint64(M32), g >> np.uint64(32), 0, 0x44524F50, seed & (2 ** 64 - 1)))
    word = np.take_along_axis(w, ((t % np.uint64(8)) // np.uint64(2)).astype(np.int64)[None], 0)[0]
    bits = (word >> (np.uint64(16) * (t % np.uint64(2)))) & np.uint64(0xFFFF)
    thr = int(round(65536 * p))
    return torch.from_numpy(bits >= np.uint64(thr)), (65536.0 / (65536 - thr) if thr < 65536 else 0.0)


def attention_keep(B, Hk, R, Lk, p, seed):
    """(keep (B, Hk, R, Lk) bool, gain) for packed rows r = i G + g"""
    u, r, j = np.arange(B * Hk)[:, None, None], np.arange(R)[None, :, None], np.arange(Lk)[None, None, :]
    w = np.stack(philox(j // 4, r // 4, u, 0x41545444, seed & (2 ** 64 - 1)))
    word = np.take_along_axis(w, np.broadcast_to(r % 4, w.shape[1:])[None], 0)[0]
    byte = (word >> np.broadcast_to(8 * (j % 4), word.shape).astype(np.uint64)) & np.uint64(255)
    thr = int(round(256 * p))
    return torch.from_numpy(byte >= np.uint64(thr)).reshape(B, Hk, R, Lk), 256.0 / (256 - thr)


def visible(B, Lq, Lk, causal, key_mask, q_lens, k_lens):
    """(B, Lq, Lk) bool"""
    ql = torch.full((B,), Lq) if q_lens is None else q_lens.long().clamp(0, Lq)
    kl = torch.full((B,), Lk) if k_lens is None else k_lens.long().clamp(0, Lk)
    i, j = torch.arange(Lq)[None, :, None], torch.arange(Lk)[None, None, :]
    see = (i < ql[:, None, None]) & (j < kl[:, None, None])
    if causal:
        see = see & (j <= i + (kl - ql)[:, None, None])
    if key_mask is not None:
        see = see & key_mask.bool()[:, None, :]
    return see


def attention(q, k, v, causal=False, key_mask=None, q_lens=None, k_lens=None, scale=None, dropout_p=0.0, seed=0, dout=None,
              bounds_for=None):
    """dict with out, lse (B, Hq, Lq) and, given dout, dq, dk, dv; with bounds_for = a dtype also tol_<name> for each.  Inputs are
    converted to float64; hidden operands are replaced by zeros first (they may hold anything)."""
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G, R = Hq // Hk, Lq * (Hq // Hk)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    see_b = visible(B, Lq, Lk, causal, key_mask, q_lens, k_lens)
    row_on = torch.ones(B, Lq, dtype=torch.bool) if q_lens is None else torch.arange(Lq)[None] < q_lens[:, None]
    key_on = torch.ones(B, Lk, dtype=torch.bool) if k_lens is None else torch.arange(Lk)[None] < k_lens[:, None]
    if key_mask is not None:
        key_on = key_on & key_mask.bool()
    rows = lambda t: t.reshape(B, Lq, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, R, D)
    back = lambda t: t.reshape(B, Hk, Lq, G, D).permute(0, 2, 1, 3, 4).reshape(B, Lq, Hq, D)
    on = lambda t, m: torch.where(m[..., None, None], t.double(), torch.zeros((), dtype=torch.float64))
    qd = rows(on(q, row_on))
    kd, vd = (on(t, key_on).permute(0, 2, 1, 3) for t in (k, v))
    see = see_b[:, None, :, None, :].expand(B, 1, Lq, G, Lk).reshape(B, 1, R, Lk)
    s = scale * qd @ kd.transpose(2, 3)
    s = s.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(s, -1) if Lk else torch.full((B, Hk, R), -math.inf, dtype=torch.float64)
    p = torch.exp(s - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[..., None])
    keep, gain = attention_keep(B, Hk, R, Lk, dropout_p, seed) if dropout_p > 0 else (torch.ones_like(p, dtype=torch.bool), 1.0)
    pd = torch.where(keep, p * gain, torch.zeros_like(p))
    o = pd @ vd
    res = dict(out=back(o), lse=lse.reshape(B, Hk, Lq, G).permute(0, 1, 3, 2).reshape(B, Hq, Lq))
    if dout is not None:
        do = rows(on(dout, row_on))
        dp = do @ vd.transpose(2, 3)
        delta = (do * o).sum(-1, keepdim=True)
        ds = p * (torch.where(keep, dp * gain, torch.zeros_like(dp)) - delta)
        res["dq"] = back(scale * ds @ kd)
        res["dk"] = (scale * ds.transpose(2, 3) @ qd).permute(0, 2, 1, 3)
        res["dv"] = (pd.transpose(2, 3) @ do).permute(0, 2, 1, 3)
    if bounds_for is not None:
        u = half_step(bounds_for)
        up = 0.0 if bounds_for == torch.float32 else u       # the probabilities and dS are operands in the inputs' type
        sub = 2.0 ** -25 if bounds_for == torch.float16 else 0.0      # half a step of half precision's smallest numbers
        # a score: D products, the scaling by log2(e) and the subtraction of the maximum (whose own error cancels in P: the
        # same number divides); exp2 and the division: 8 steps; the sum over the keys
        s_abs = (scale * qd.abs() @ kd.abs().transpose(2, 3)).masked_fill(~see, 0.0)
        es = (D + 4) * E32 * s_abs.amax(-1, keepdim=True) if Lk else torch.zeros(B, Hk, R, 1, dtype=torch.float64)
        lse_abs = torch.where(lse == -math.inf, torch.zeros_like(lse), lse.abs())[..., None]
        rel = 2 * es + (Lk + 16) * E32 + 4 * E32 * lse_abs
        res["tol_lse"] = ((es + (Lk + 8) * E32 + 4 * E32 * lse_abs)[..., 0]).reshape(B, Hk, Lq, G).permute(0, 1, 3, 2).reshape(B, Hq, Lq)
        w = pd @ vd.abs()
        to = (up + rel + Lk * E32) * w + u * o.abs() + sub * gain * (1 + vd.abs().sum(2, keepdim=True))
        res["tol_out"] = back(to)
        if dout is not None:
            edp = (D + 2) * E32 * gain * (do.abs() @ vd.abs().transpose(2, 3))
            edelta = (do.abs() * to).sum(-1, keepdim=True) + (D + 2) * E32 * (do * o).abs().sum(-1, keepdim=True) \
                + Lk * E32 * (pd * dp.abs()).sum(-1, keepdim=True)
            eds = (up + rel + 4 * E32) * ds.abs() + (1 + rel) * p * (edp + edelta) + sub * see
            res["tol_dq"] = back(scale * (eds @ kd.abs() + Lk * E32 * ds.abs() @ kd.abs())) + u * res["dq"].abs() + sub
            res["tol_dk"] = (scale * (eds + R * E32 * ds.abs()).transpose(2, 3) @ qd.abs()).permute(0, 2, 1, 3) + u * res["dk"].abs() + sub
            res["tol_dv"] = (((up + rel + R * E32) * pd + sub * gain * see).transpose(2, 3) @ do.abs()).permute(0, 2, 1, 3) \
                + u * res["dv"].abs() + sub
    return res


def qk_norm_rope(x, w, positions, inv_freq, eps=1e-6, interleaved=False, dy=None):
    """One of the two tensors: dict with y and, given dy, dx, dw; `mag` = the magnitude that rounding errors of y scale with."""
    B, L, H, D = x.shape
    x, w = x.double(), w.double()
    pos = positions.double() if positions.dim() == 2 else positions.double()[None].expand(B, L)
    ang = pos[:, :, None, None] * inv_freq.double()
    rot = 2 * inv_freq.numel()
    i = torch.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)

    def turn(z, sign):
        y = z.clone()
        y[..., a] = z[..., a] * ang.cos() - sign * z[..., b] * ang.sin()
        y[..., b] = z[..., b] * ang.cos() + sign * z[..., a] * ang.sin()
        return y

    def mags(z):
        m = z.abs()
        m[..., a], m[..., b] = (z[..., a].abs() + z[..., b].abs(),) * 2
        return m

    r = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    xh = x * r
    res = dict(y=turn(xh * w, 1.0), mag=mags(xh * w))
    if dy is not None:
        dz, mz = turn(dy.double(), -1.0), mags(dy.double())
        res["dw"] = (dz * xh).sum((0, 1, 2))
        res["dw_mag"] = (mz * xh.abs()).sum((0, 1, 2))
        mean = (w * dz * xh).mean(-1, keepdim=True)
        res["dx"] = r * (w * dz - xh * mean)
        res["dx_mag"] = r * ((w * mz).abs() + xh.abs() * (w * mz * xh).abs().mean(-1, keepdim=True))
    return res
