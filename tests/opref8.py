"""Plain 64-bit forms of the root-mean-square norm and of e4m3 with a scale for 128, and the error bounds they go with
(counting roundings as in opref.py)."""

import torch

from opref import U, half_step, smallest

# ---------------------------------------------------------------- e4m3
# the 127 finite magnitudes, in the order of their codes
GRID = torch.tensor([m * 2.0 ** -9 for m in range(8)] +
                    [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)], dtype=torch.float64)[:127]


def blocks(x, tall):
    """x [rows, k] padded with zeros as [row blocks, tall, steps, 128]."""
    rows, k = x.shape
    v = torch.zeros(rows + -rows % tall, k + -k % 128, dtype=torch.float64)
    v[:rows, :k] = x
    return v.reshape(v.shape[0] // tall, tall, v.shape[1] // 128, 128)


def quantize(x, tall):
    """(codes [rows, Kp], scales [row blocks, steps]) of x by search: the smallest scale that fits, then the nearest grid
    point, the even code where two are equally near."""
    x = x.double().cpu()
    rows, k = x.shape
    v = blocks(x, tall)
    fine = torch.isfinite(v).all(3).all(1)
    top = torch.where(torch.isfinite(v), v, torch.zeros_like(v)).abs().amax((1, 3))
    fits = top.unsqueeze(-1) <= 448.0 * torch.exp2(torch.arange(255, dtype=torch.float64) - 127)
    s = fits.long().argmax(-1)
    s[~fine] = 255
    a = torch.where(fine[:, None, :, None], v, torch.zeros_like(v)) / torch.exp2(s.double() - 127)[:, None, :, None]
    a = a.reshape(v.shape[0] * tall, -1)[:rows]
    m = a.abs().contiguous()
    hi = torch.searchsorted(GRID, m).clamp(max=126)  # the first grid point at or above
    lo = (hi - 1).clamp(min=0)
    up, down = GRID[hi] - m, m - GRID[lo]
    codes = torch.where(up < down, hi, torch.where(up > down, lo, torch.where(hi % 2 == 0, hi, lo)))
    return codes + 128 * torch.signbit(a).long(), s


def values(codes, scales, k, tall):
    """The values [rows, k] of codes and scales, as bytes or as numbers."""
    c, s = (t.cpu() if t.dtype == torch.int64 else t.cpu().view(torch.uint8).long() for t in (codes, scales))
    mag = torch.cat([GRID, torch.tensor([float("nan")], dtype=torch.float64)])
    v = torch.where(c >= 128, -mag[c % 128], mag[c % 128])
    f = torch.where(s == 255, torch.full((), float("nan"), dtype=torch.float64), torch.exp2(s.double() - 127))
    f = f.repeat_interleave(tall, 0)[:c.shape[0]].repeat_interleave(128, 1)
    return v[:, :k] * f[:, :k]


def tensor_values(q):
    return values(q.codes, q.scales, q.shape[-1], q.block)


def product(a, b, dtype, order=8):
    """a [M, K] times b [K, N] (values as held) and a bound for the kernels' output.

    The scaled instructions take 8 consecutive products at a time, aligned to the one with the largest exponent: of the others
    what lies below 2^-13 of that power of two is cut off, less than 2^-13 of the largest product each (its power of two is
    at most itself).  The groups' sums then add up in fp32, K / 8 of them in any order."""
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    a, b = a.to(dev), b.contiguous().to(dev)
    k = a.shape[1]
    pad = -k % order
    ag = torch.nn.functional.pad(a.abs(), (0, pad)).reshape(a.shape[0], -1, order)
    bg = torch.nn.functional.pad(b.abs(), (0, 0, 0, pad)).reshape(-1, order, b.shape[1])
    cut = torch.zeros(a.shape[0], b.shape[1], dtype=torch.float64, device=dev)
    for g in range(ag.shape[1]):
        cut += (ag[:, g, :, None] * bg[None, g]).amax(1)
    e = (order - 1) * 2.0 ** -13 * cut + (k // order + 2) * U * (a.abs() @ b.abs())
    ref = a @ b
    bound = half_step(dtype) * (ref.abs() + e) + e + smallest(dtype)
    return ref.cpu(), bound.cpu()


# ---------------------------------------------------------------- root-mean-square norm
class Rms64:
    """The norm of h [rows, n] and its gradients in 64 bits, with bounds for the fp32 kernels' outputs."""

    def __init__(self, h, w, eps):
        self.h = h.double().cpu().reshape(-1, h.shape[-1])
        n = self.h.shape[1]
        self.w = torch.ones(n, dtype=torch.float64) if w is None else w.double().cpu()
        self.rstd = 1.0 / torch.sqrt((self.h ** 2).mean(-1, keepdim=True) + eps)
        self.z = self.h * self.rstd
        self.y = self.z * self.w
        # additions in sequence within a row: a thread's elements (32 at most in registers, n / 1024 + 8 in the wide
        # kernels), 6 lane steps, 16 waves' parts
        self.adds = 56 if n <= 16384 else 56 + n // 1024 + 8
        # rstd: half the relative error of the mean of squares (its sum, 1 / n, the product, eps), the root and the quotient
        self.r_rstd = (self.adds / 2 + 5) * U
        self.r_z = self.r_rstd + U

    def e_y(self):
        return (self.r_z + U) * self.y.abs()

    def bound_y(self, dtype):
        e = self.e_y()
        return half_step(dtype) * (self.y.abs() + e) + e + smallest(dtype)

    def grads(self, dy, dtype, wdtype, dh=None):
        """(dx, dw) and their bounds."""
        dy = dy.double().cpu().reshape(self.h.shape)
        rows, n = self.h.shape
        g = dy * self.w
        s = (g * self.z).mean(-1, keepdim=True)
        dx = self.rstd * (g - self.z * s)
        # the mean: its sum's roundings, those of g, z and 1 / n
        e_s = (self.adds + 4) * U * (g * self.z).abs().mean(-1, keepdim=True) + self.r_z * (g * self.z).abs().mean(-1, keepdim=True)
        e = self.rstd * (3 * U * (g.abs() + (self.z * s).abs()) + self.r_z * (self.z * s).abs() + self.z.abs() * e_s)
        e = e + (self.r_rstd + U) * dx.abs()
        if dh is not None:
            d = dh.double().cpu().reshape(self.h.shape)
            e = e + U * (d.abs() + dx.abs())
            dx = dx + d
        # rows in sequence: a thread's rows, its workgroup's groups, the parts of a wave (of 16) and the waves
        adds = rows // 256 + 64 + 64 + 16
        dw = (dy * self.z).sum(0)
        e_w = (adds * U + self.r_z) * (dy * self.z).abs().sum(0)

        def bound(v, e, t):
            return half_step(t) * (v.abs() + e) + e + smallest(t)
        return (dx, dw), (bound(dx, e, dtype), bound(dw, e_w, wdtype))
