"""The operators around a block in 64 bits, with bounds on what fp32 kernels may be off by
(not collected by pytest).

U = 2^-24 is the rounding of one fp32 operation.  A sum over a row is a chain of at
most 8 additions and 10 levels over the threads, so its result is off by at most 18 U
times the sum of magnitudes; a mean over a row is off by at most 20 U times the largest
magnitude.  The bounds below carry such terms to first order with constants rounded up,
and add half a step of the output's type."""
import numpy as np
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the step between the smallest values of a type (fp16 has them in reach)."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps


def assert_within(got, ref, bound, what):
    got = got.detach().double().cpu()
    ref, bound = ref.cpu(), bound.cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = (got - ref).abs() - bound
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 0, f"{what}: over its bound by {worst:.3e} (bound {bound.flatten()[off.argmax()].item():.3e})"


def keep_mask(count, threshold, seed, offset):
    """Truth values of the first elements that stay."""
    return keep_mask_at(0, count, threshold, seed, offset)


def keep_mask_at(first, count, threshold, seed, offset):
    """Truth values of the elements from `first` (a multiple of 8) on that stay: Philox4x32-10 in unsigned 64-bit
    numpy arithmetic."""
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    group = first // 8 + np.arange(-(-count // 8), dtype=np.uint64)
    c = [group & low, group >> shift, np.full_like(group, offset & 0xFFFFFFFF), np.full_like(group, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> shift) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> shift) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    words = np.stack(c, -1)
    halves = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], -1).reshape(-1)[:count]
    return torch.from_numpy((halves >= np.uint64(threshold)).copy())


class NormRef:
    """norm(v) * w + b of rows v [rows, dim] in 64 bits, its gradient, and bounds."""

    def __init__(self, v, dv, kind, w, b, eps):
        """dv: how far the kernel's v may be off."""
        self.kind, dim = kind, v.shape[1]
        w = torch.ones(dim, dtype=torch.float64) if w is None else w
        b = torch.zeros(dim, dtype=torch.float64) if b is None else b
        mean = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros(len(v), 1, dtype=torch.float64)
        c = v - mean
        self.rstd = 1 / torch.sqrt(c.square().mean(1, keepdim=True) + eps)
        self.hat, self.w = c * self.rstd, w
        self.out = self.hat * w + b
        top = v.abs().amax(1, keepdim=True)
        # c off by the error of v, of the mean and a rounding; rstd by that of the root
        # mean square, at most the largest error of c times rstd, and its own sums.
        dc = dv + dv.amax(1, keepdim=True) + 24 * U * top
        rel = dc.amax(1, keepdim=True) * self.rstd + 24 * U
        self.dhat = dc * self.rstd + self.hat.abs() * rel + 2 * U * self.hat.abs()
        self.bound = self.dhat * w.abs() + 4 * U * (self.out.abs() + b.abs())
        self.rel = rel

    def back(self, dn, ddn):
        """(gradient of v, its bound) for the gradient dn, off by ddn."""
        g, dg = dn * self.w, ddn * self.w.abs() + U * (dn * self.w).abs()
        m1 = (g * self.hat).mean(1, keepdim=True)
        m0 = g.mean(1, keepdim=True) if self.kind == "layer" else torch.zeros_like(m1)
        d = g - m0 - self.hat * m1
        mag = g.abs().mean(1, keepdim=True)
        mag1 = (g * self.hat).abs().mean(1, keepdim=True)
        dm0 = dg.mean(1, keepdim=True) + 24 * U * mag
        dm1 = (dg * self.hat.abs() + g.abs() * self.dhat).mean(1, keepdim=True) + 24 * U * mag1
        dd = dg + dm0 + self.hat.abs() * dm1 + self.dhat * m1.abs() + 4 * U * (g.abs() + m0.abs() + (self.hat * m1).abs())
        return d * self.rstd, dd * self.rstd + d.abs() * self.rstd * (self.rel + 4 * U)


def sum_bound(terms, dterms, rows, dim_axis=0):
    """Bound of a sum over rows: the terms' own errors and a chain of at most rows + 64 additions."""
    return dterms.sum(dim_axis) + (rows + 64) * U * terms.abs().sum(dim_axis)


def block_reference(x, y, post, gate, scale, alpha, keep, rate, after, dout, dn):
    """Everything block_residual computes, as {name: (value, bound in fp32)} in 64 bits.  x, y [rows,
    dim]; gate None or broadcast to [rows, dim]; post, after: (kind, w, b, eps) or None; keep
    truth values or None; rate the share dropped; dout / dn may be None."""
    zero = torch.zeros_like(x)
    made = {}
    if y is None:
        k = k0 = z = dz = zero
        out, dout_f = x, zero
    else:
        n1 = None if post is None else NormRef(y, zero, *post)
        b, db_ = (y, zero) if post is None else (n1.out, n1.bound)
        inv = 1.0 if keep is None else 1 / (1 - rate)
        kf = torch.ones_like(x) if keep is None else keep.double()
        z = torch.where(kf > 0, b * inv, zero)
        dz = torch.where(kf > 0, db_ * inv + 3 * U * (b * inv).abs(), zero)
        g = torch.ones_like(x) if gate is None else gate
        s = torch.ones(x.shape[1], dtype=torch.float64) if scale is None else scale
        k0 = g * s
        out = alpha * x + k0 * z
        # the kernel forms gate * scale, alpha * x and their product and sum with a rounding each
        dout_f = k0.abs() * dz + 4 * U * (k0 * z).abs() + 3 * U * ((alpha * x).abs() + out.abs())
        made["out"] = (out, dout_f)
    n2 = None
    if after is not None:
        n2 = NormRef(out, dout_f, *after)
        made["n"] = (n2.out, n2.bound)
    if dout is None and dn is None:
        return made
    rows = len(x)
    go = zero if dout is None else dout
    dgo = zero
    if dn is not None:
        back, dback = n2.back(dn, zero)
        go, dgo = go + back, dback + U * (go + back).abs()
        made["d_next_weight"] = ((dn * n2.hat).sum(0), sum_bound(dn * n2.hat, dn.abs() * (n2.dhat + U * n2.hat.abs()), rows))
        made["d_next_bias"] = (dn.sum(0), sum_bound(dn, zero, rows))
    made["d_x"] = (alpha * go, abs(alpha) * dgo + U * (alpha * go).abs())
    if y is None:
        return made
    zg, dzg = z * go, dz * go.abs() + z.abs() * dgo + 2 * U * (z * go).abs()
    made["d_scale"] = ((g * zg).sum(0), sum_bound(g * zg, g.abs() * dzg + 2 * U * (g * zg).abs(), rows))
    made["d_gate_terms"] = (s * zg, s.abs() * dzg + 2 * U * (s * zg).abs())
    d = kf * inv * k0 * go
    dd = kf * inv * k0.abs() * dgo + 5 * U * d.abs()
    if post is not None:
        made["d_weight"] = ((d * n1.hat).sum(0), sum_bound(d * n1.hat, dd * n1.hat.abs() + d.abs() * (n1.dhat + U * n1.hat.abs()), rows))
        made["d_bias"] = (d.sum(0), sum_bound(d, dd, rows))
        d, dd = n1.back(d, dd)
    made["d_y"] = (d, dd)
    return made


def rotary_reference(x, positions, freqs, pairs, layout, magnitude, inverse=False):
    """x [B, H, N, d] turned in 64 bits; positions [B or 1, N, axes]; pairs per axis."""
    axis = torch.repeat_interleave(torch.arange(len(pairs)), torch.tensor(pairs))
    angle = (positions[..., axis].double() * freqs).unsqueeze(1)
    cos, sin = angle.cos() * magnitude, angle.sin() * magnitude * (-1 if inverse else 1)
    p = sum(pairs)
    first = torch.arange(p) if layout == "half" else 2 * torch.arange(p)
    second = first + (p if layout == "half" else 1)
    out = x.double().clone()
    a, b = x.double()[..., first], x.double()[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, a * sin + b * cos
    return out
