"""float64 restatements of the operators on 8-bit kept rows and of the gated residual norm, on the
CPU, written from their definitions."""
import numpy as np
import torch

GROUP, BIAS = 32, 133


def exponents(mag, most=254):
    """Exponent byte of every group of 32 columns of the float32 magnitudes [rows, C]."""
    rows, C = mag.shape
    G = -(-C // GROUP)
    wide = np.zeros((rows, G * GROUP))
    wide[:, :C] = np.where(np.isfinite(mag), np.abs(mag), 0).astype(np.float32)
    amax = wide.reshape(rows, G, GROUP).max(2)
    e = np.zeros((rows, G), np.int64)
    need = amax > np.ldexp(127.5, -BIAS)
    m, x = np.frexp(np.where(need, amax, 1.0) / 127.5)      # amax = m 2^x 127.5, m in [0.5, 1)
    e[need] = (np.where(m > 0.5, x, x - 1) + BIAS)[need]
    return np.clip(e, 0, most)


def spread(e, C):
    return np.repeat(e, GROUP, axis=1)[:, :C]


def codes_of(v, e):
    """Whole numbers (float64), not clamped: v in float64."""
    with np.errstate(invalid="ignore", over="ignore"):
        return np.rint(np.ldexp(v, BIAS - spread(e, v.shape[1])))


def finish(q, v):
    q = np.clip(np.where(np.isfinite(v), q, 0), -127, 127)
    return np.where(np.isfinite(v), q, -128).astype(np.int8)


def pack(x, most=254):
    """(codes, exps) of float32 rows (16-bit rows: widened)."""
    x = np.asarray(x, np.float32)
    e = exponents(x, most)
    return finish(codes_of(x.astype(np.float64), e), x), e.astype(np.uint8)


def unpack(codes, exps):
    v = np.ldexp(codes.astype(np.float64), spread(exps.astype(np.int64), codes.shape[1]) - BIAS)
    return np.where(codes == -128, np.nan, v)


def bn_pack(z, mean, invstd, gamma, beta, act):
    """(codes, exps) of the normalised rows, float64 statistics, on the kink's side."""
    with np.errstate(invalid="ignore"):
        zh = (z - mean) * invstd
    with np.errstate(over="ignore"):
        zf = zh.astype(np.float32)
    e = exponents(zf)
    q = codes_of(zh, e)
    if act:
        with np.errstate(divide="ignore", invalid="ignore"):
            t = (-beta.astype(np.float32) / gamma.astype(np.float32)).astype(np.float64)
            on = zh * gamma + beta > 0
            at = np.ldexp(np.broadcast_to(t, zh.shape), BIAS - spread(e, zh.shape[1]))
        pos, neg = gamma > 0, gamma < 0
        q = np.where(pos & on, np.fmax(q, np.floor(at) + 1), q)
        q = np.where(pos & ~on, np.fmin(q, np.floor(at)), q)
        q = np.where(neg & on, np.fmin(q, np.ceil(at) - 1), q)
        q = np.where(neg & ~on, np.fmax(q, np.ceil(at)), q)
    return finish(q, zf.astype(np.float64)), e.astype(np.uint8)


def bn_on(zq, gamma, beta):
    """Side of the kink of values read back."""
    with np.errstate(divide="ignore", invalid="ignore"):
        t = (-beta.astype(np.float32) / gamma.astype(np.float32)).astype(np.float64)
        return np.where(gamma > 0, zq > t, np.where(gamma < 0, zq < t, (beta > 0) & np.isfinite(zq)))


def bn_stats(z, eps):
    mean = z.mean(0)
    var = ((z - mean) ** 2).mean(0)
    return mean, 1 / np.sqrt(var + np.float64(np.float32(eps)))


def norm(v, kind, eps):
    mu = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    r = 1 / torch.sqrt(((v - mu) ** 2).mean(1, keepdim=True) + eps)
    return mu, r


class Residual:
    """The gated residual norm on float64 CPU tensors, forward and backward, and for every result
    the sum of the magnitudes that make it up (what rounding errors scale with).  xq, fq: x and f as
    the backward sees them."""

    def __init__(self, x, f, xq=None, fq=None, post=None, pre=None, gate=None, scale=None, seen=None):
        """post, pre: (kind, weight or None, bias or None, eps) or None."""
        C = x.shape[1]
        one = torch.ones(C, dtype=torch.float64)
        self.C, self.post, self.pre = C, post, pre
        self.s = one if scale is None else scale
        g = torch.ones(x.shape[0], 1, dtype=torch.float64) if gate is None else gate
        self.G = g.shape[1]
        seen = torch.ones(x.shape[0], dtype=torch.bool) if seen is None else seen
        self.seen = seen.double().unsqueeze(1)
        self.g = g.repeat_interleave(C // self.G, dim=1) * self.seen
        self.wf, self.bf = self._affine(post)
        self.wo, self.bo = self._affine(pre)
        f = torch.where(seen.unsqueeze(1), f, torch.zeros_like(f))
        fq = f if fq is None else torch.where(seen.unsqueeze(1), fq, torch.zeros_like(f))
        xq = x if xq is None else xq
        if post is None:
            self.muf, self.rf = torch.zeros_like(x[:, :1]), torch.ones_like(x[:, :1])
        else:
            self.muf, self.rf = norm(f, post[0], post[3])
        n = (f - self.muf) * self.rf
        self.out = x + self.g * self.s * (n * self.wf + self.bf)
        Mn = (f.abs() + self.muf.abs()) * self.rf
        self.M_out = x.abs() + (self.g * self.s).abs() * (Mn * self.wf.abs() + self.bf.abs())
        if pre is not None:
            self.muo, self.ro = norm(self.out, pre[0], pre[3])
            o = (self.out - self.muo) * self.ro
            self.h = o * self.wo + self.bo
            Mo = (self.M_out + self.M_out.mean(1, keepdim=True)) * self.ro
            Mo = Mo + o.abs() * (Mo * o.abs()).mean(1, keepdim=True)
            self.M_h = Mo * self.wo.abs() + self.bo.abs()
        # as the backward sees the rows
        self.n = (fq - self.muf) * self.rf
        self.Mn = (fq.abs() + self.muf.abs()) * self.rf
        self.v = self.n * self.wf + self.bf
        self.Mv = self.Mn * self.wf.abs() + self.bf.abs()
        if pre is not None:
            u = xq + self.g * self.s * self.v
            self.o = (u - self.muo) * self.ro
            self.Mo = (xq.abs() + (self.g * self.s).abs() * self.Mv + self.muo.abs()) * self.ro

    def _affine(self, p):
        one = torch.ones(self.C, dtype=torch.float64)
        w = one if p is None or p[1] is None else p[1]
        b = 0 * one if p is None or p[2] is None else p[2]
        return w, b

    def backward(self, d_out, d_h):
        def mean(t):
            return t.mean(1, keepdim=True)
        zero = torch.zeros_like(self.out)
        d = zero if d_out is None else d_out
        M = d.abs()
        got, mag = {}, {}
        dh = zero if d_h is None or self.pre is None else d_h
        if self.pre is not None:
            q = dh * self.wo
            layer = 1.0 if self.pre[0] == "layer" else 0.0
            d = d + self.ro * (q - self.o * mean(q * self.o) - layer * mean(q))
            M = M + self.ro * (q.abs() + layer * mean(q.abs()) + self.Mo * mean(q.abs() * self.o.abs())
                               + self.o.abs() * mean(q.abs() * self.Mo))
            got["w_pre"], mag["w_pre"] = (dh * self.o).sum(0), (dh.abs() * self.Mo).sum(0)
            got["b_pre"], mag["b_pre"] = dh.sum(0), dh.abs().sum(0)
        got["x"], mag["x"] = d, M
        e, Me = d * self.g, M * self.g.abs()
        got["w_post"], mag["w_post"] = self.s * (e * self.n).sum(0), self.s.abs() * (Me * self.Mn).sum(0)
        got["b_post"], mag["b_post"] = self.s * e.sum(0), self.s.abs() * Me.sum(0)
        got["scale"], mag["scale"] = (e * self.v).sum(0), (Me * self.Mv).sum(0)
        k, Mk = e * self.s * self.wf, Me * (self.s * self.wf).abs()
        if self.post is None:
            got["f"], mag["f"] = k, Mk
        else:
            layer = 1.0 if self.post[0] == "layer" else 0.0
            got["f"] = self.seen * self.rf * (k - self.n * mean(k * self.n) - layer * mean(k))
            mag["f"] = self.rf * (Mk + layer * mean(Mk) + self.Mn * mean(Mk * self.Mn))
        shape = (d.shape[0], self.G, -1)
        got["gate"] = (d * self.s * self.v * self.seen).view(shape).sum(2)
        mag["gate"] = (M * self.s.abs() * self.Mv).view(shape).sum(2)
        return got, mag
