"""Plain 64-bit forms of layer norm, dropout and MXFP4 for the tests, and the error bounds they go with.

Bounds count roundings.  U = 2^-24 is half a step of fp32; a sum of m terms taken in fp32 by `adds` additions
in sequence on any path is within adds * U * sum|terms| of exact (first order); an output rounded to type t is
within eps(t) / 2 of its value.
"""

import numpy as np
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the spacing of the type's subnormal numbers (an absolute rounding error near zero)."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------- dropout
def philox(counter, key):
    """Philox4x32-10 (Salmon et al., SC 2011) of uint64 arrays holding 32-bit words: counter (4 arrays), key (2 ints)."""
    c = [np.asarray(w, dtype=np.uint64) for w in counter]
    k0, k1 = int(key[0]), int(key[1])
    m = np.uint64(0xFFFFFFFF)
    s = np.uint64(32)
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> s) ^ c[1] ^ np.uint64(k0), b & m, (a >> s) ^ c[3] ^ np.uint64(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def kept(rows, n, keep, seed, offset, first_row=0):
    """bool [rows, n]: element (row, col) draws number col % 8 of the block (row ceil(n / 8) + col // 8, offset)."""
    nc = -(-n // 8)
    q = np.arange(first_row * nc, (first_row + rows) * nc, dtype=np.uint64)
    lo, hi = np.uint64(0xFFFFFFFF), np.uint64(32)
    z = np.zeros_like(q)
    w = philox([q & lo, q >> hi, z + np.uint64(offset & 0xFFFFFFFF), z + np.uint64(offset >> 32 & 0xFFFFFFFF)],
               (seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF))
    u = np.stack([h for word in w for h in (word & np.uint64(0xFFFF), word >> np.uint64(16))], axis=-1)
    return torch.from_numpy((u.reshape(rows, 8 * nc)[:, :n] < keep))


def drop64(x, p, seed, offset=0):
    """x as [rows, n] doubles with dropout applied, and the scaled mask."""
    keep = 65536 - round(65536 * p)
    x = x.double().cpu()
    x2 = x.reshape(-1, x.shape[-1])
    k = kept(*x2.shape, keep, seed, offset).reshape(x.shape)
    scale = 65536.0 / keep if keep else 0.0
    return torch.where(k, x * scale, torch.zeros_like(x)), k.double() * scale


# ---------------------------------------------------------------- layer norm
class Norm64:
    """Layer norm of h [rows, n] and its gradients in 64 bits, with bounds for the fp32 kernels' outputs."""

    def __init__(self, h, w, b, eps):
        self.h = h.double().cpu().reshape(-1, h.shape[-1])
        rows, n = self.h.shape
        self.w = torch.ones(n, dtype=torch.float64) if w is None else w.double().cpu()
        self.b = torch.zeros(n, dtype=torch.float64) if b is None else b.double().cpu()
        self.mean = self.h.mean(-1, keepdim=True)
        self.rstd = 1.0 / torch.sqrt(((self.h - self.mean) ** 2).mean(-1, keepdim=True) + eps)
        self.z = (self.h - self.mean) * self.rstd
        self.y = self.z * self.w + self.b
        # additions in sequence within a row: a thread's elements (32 at most in registers, n / 1024 + 8 in the wide
        # kernels), 6 lane steps, 16 waves' parts, and the merge's own operations
        self.adds = 64 if n <= 16384 else 64 + n // 1024 + 8
        a = self.adds
        # the mean is off by a U mean|h|; z then by that, its own two roundings, and half the variance's relative
        # error: its sum's a roundings, the deviations' (2 U and the wave means' a U, to second order in their share) and
        # those of the quotient and the root
        self.e_mean = a * U * self.h.abs().mean(-1, keepdim=True)
        self.e_z = self.rstd * (self.e_mean + 2 * U * self.h.abs()) + (a + 8) * U * self.z.abs() + \
            self.z.abs() * self.rstd * self.e_mean
        self.e_rstd = self.rstd * ((a + 8) * U + self.rstd * self.e_mean)

    def bound_y(self, dtype):
        exact = self.e_z * self.w.abs() + 2 * U * ((self.z * self.w).abs() + self.b.abs())
        return half_step(dtype) * (self.y.abs() + exact) + exact + smallest(dtype)

    def grads(self, dy, dtype, wdtype, dh=None):
        """dn (or dh + dn), dw, db and their bounds."""
        dy = dy.double().cpu().reshape(self.h.shape)
        rows, n = self.h.shape
        g = dy * self.w
        s1, s2 = g.mean(-1, keepdim=True), (g * self.z).mean(-1, keepdim=True)
        dn = self.rstd * (g - s1 - self.z * s2)
        a = self.adds
        e1 = (a + 2) * U * g.abs().mean(-1, keepdim=True)
        e2 = (a + 3) * U * (g * self.z).abs().mean(-1, keepdim=True) + (g.abs() * self.e_z).mean(-1, keepdim=True)
        inner = g.abs() + s1.abs() + (self.z * s2).abs()
        e_dn = self.rstd * (4 * U * inner + e1 + self.z.abs() * e2 + self.e_z * s2.abs()) + \
            (self.e_rstd / self.rstd) * dn.abs()
        if dh is not None:
            d2 = dh.double().cpu().reshape(self.h.shape)
            e_dn = e_dn + U * (d2.abs() + dn.abs())
            dn = dn + d2
        # rows in sequence: a thread's rows, its workgroup's groups, the parts of a wave (of 16) and the waves
        adds = rows // 256 + 64 + 64 + 16
        dw, db = (dy * self.z).sum(0), dy.sum(0)
        e_dw = adds * U * (dy * self.z).abs().sum(0) + (dy.abs() * self.e_z).sum(0)
        e_db = adds * U * dy.abs().sum(0)

        def bound(v, e, t):
            return half_step(t) * (v.abs() + e) + e + smallest(t)
        return (dn, dw, db), (bound(dn, e_dn, dtype), bound(dw, e_dw, wdtype), bound(db, e_db, wdtype)), e_dn


def assert_within(got, ref, bound, what):
    got = got.detach().double().cpu().reshape(ref.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - ref).abs() - bound
    worst = int(off.argmax()) if off.numel() else 0
    assert off.numel() == 0 or off.max() <= 0, (
        f"{what}: {float(got.reshape(-1)[worst])} for {float(ref.reshape(-1)[worst])}, bound "
        f"{float(bound.expand_as(ref).reshape(-1)[worst])} at {worst} of {tuple(ref.shape)}; "
        f"{float((off > 0).double().mean()):.2e} of the elements outside")


# ---------------------------------------------------------------- MXFP4
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def mx_quantize(x):
    """(codes [rows, Kp] as numbers 0 .. 15, scales [rows, Kp / 32]) of x by search: the nearest grid point of
    x / scale, the even code where two are equally near."""
    x = x.double().cpu()
    rows, k = x.shape
    kp = -(-k // 128) * 128
    v = torch.zeros(rows, kp, dtype=torch.float64)
    v[:, :k] = x
    v = v.reshape(rows, -1, 32)
    top = v.abs().amax(-1)
    s = torch.zeros(top.shape, dtype=torch.int64)
    fine = torch.isfinite(v).all(-1)
    some = fine & (top > 0)
    s[some] = (torch.floor(torch.log2(top[some])).long() - 2 + 127).clamp(min=0)
    # log2 of a power of two's neighbours is safe in doubles for values that fp32 holds, checked here
    e = s[some] - 127 + 2
    assert ((top[some] >= torch.exp2(e.double())) | (s[some] == 0)).all() and (top[some] < torch.exp2(e.double() + 1)).all()
    a = torch.where(fine.unsqueeze(-1), v, torch.zeros_like(v)) / torch.exp2(s.double() - 127).unsqueeze(-1)
    d = (a.abs().unsqueeze(-1) - torch.tensor(GRID, dtype=torch.float64)).abs()
    best = d.amin(-1, keepdim=True)
    near = d == best
    # among equally near neighbours the even code
    pick = torch.where(near, torch.arange(8) % 2 * 8 + torch.arange(8), torch.full((8,), 99)).argmin(-1)
    codes = pick + 8 * torch.signbit(a).long()
    codes = torch.where(fine.unsqueeze(-1), codes, torch.zeros_like(codes))
    s[~fine] = 255
    return codes.reshape(rows, kp), s


def mx_values(codes, scales, k):
    mag = torch.tensor(GRID + [-g for g in GRID], dtype=torch.float64)[codes]
    return (mag * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1))[:, :k]


def mx_nibbles(packed):
    p = packed.cpu().long()
    return torch.stack([p & 15, p >> 4], -1).reshape(p.shape[0], -1)


def product_bound(a, b, dtype, extra=0):
    """a [M, K] times b [K, N] in fp32 in any order: K roundings of sums at most, and the output's."""
    if torch.cuda.is_available():
        a, b = a.cuda(), b.contiguous().cuda()
    mag = (a.abs() @ b.abs()).cpu()
    e = (a.shape[1] + extra) * U * mag
    ref = (a @ b).cpu()
    return ref, half_step(dtype) * (ref.abs() + e) + e + smallest(dtype)
