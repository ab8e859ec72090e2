"""AdamW with moments in 8 bits, from its definition on real numbers held in 64 bits (the tests' oracle; CPU)."""
import math

import torch

MASK = 0xFFFFFFFF
PHI, SQ2, SQ3 = 0x9E3779B1, 0x6A09E667, 0xBB67AE85


def mix(x: int) -> int:
    x = ((x ^ (x >> 16)) * SQ2) & MASK
    x = ((x ^ (x >> 15)) * SQ3) & MASK
    return x ^ (x >> 16)


def hashes(n, seed, place, step):
    """32 bits for every element of the optimizer's ``place``-th parameter in its ``step``-th step."""
    key = mix((mix((seed + place * PHI) & MASK) + step) & MASK)
    x = (torch.arange(n) * PHI + key) & MASK
    x = ((x ^ (x >> 16)) * SQ2) & MASK
    x = ((x ^ (x >> 15)) * SQ3) & MASK
    return x ^ (x >> 16)


def to_grid(x, rnd, emin, keep):
    """Non-negative x in blocks of 256 to 3 mantissa bits, normal from 2^emin of the block's scale; up where the part that
    would be cut off and the dither (16 bits, at the middle of its step) reach one. ``keep``: what is not 0 stays so."""
    n = x.numel()
    pad = -n % 256
    x, rnd = (torch.nn.functional.pad(t, (0, pad)).view(-1, 256) for t in (x, rnd))
    # the largest magnitude is the 32-bit value's: 37.5 * 0.05 is 1.875 there and lies above it in 64 bits
    top = x.amax(1).float().double()
    mant, ex = torch.frexp(top)                    # top = mant * 2^ex, mant in [1/2, 1)
    ex = torch.where(torch.ceil(mant * 16) >= 16, ex, ex - 1)     # rounded up to 3 bits it still is under 2 * 2^ex
    scale = torch.ldexp(torch.ones(()).double(), ex.clamp(min=-126)).double()[:, None]
    y = x / scale
    unit = torch.ldexp(torch.ones(()).double(), (torch.frexp(y)[1] - 1).clamp(min=emin) - 3)
    cut = y / unit
    up = (cut - torch.floor(cut)) + (rnd.double() + 0.5) / 65536 >= 1
    out = (torch.floor(cut) + up) * unit
    if keep:
        out = torch.where((x > 0) & (out == 0), unit, out)
    return (out * scale).view(-1)[:n]


def spacing(x, emin):
    """How far apart a value's two neighbours in the code are at most: an eighth of it, or the step of gradual underflow,
    2^(emin - 3) of a scale that is at most twice the block's largest magnitude."""
    flat = x.abs().reshape(-1)
    pad = torch.nn.functional.pad(flat, (0, -flat.numel() % 256)).view(-1, 256)
    step = pad.amax(1, keepdim=True) * 2.0 ** (emin - 2)
    return torch.maximum(flat / 8, step.expand_as(pad).reshape(-1)[:flat.numel()]).view(x.shape) * (1 + 2.0 ** -20)


class Oracle:
    """``p``, ``m``, ``v``: lists of flat-shaped float64 tensors, the state before and after :meth:`step`."""

    def __init__(self, p, m, v, t, bits, low):
        self.p, self.m, self.v, self.t, self.bits, self.low = p, m, v, t, bits, low
        self.norm = None

    @classmethod
    def of(cls, opt, params, bits):
        from raydp_amd.ops.fused_optim import decode_moments
        m, v, t = [], [], []
        for p in params:
            st = opt.state.get(p)
            if not st:
                a = b = torch.zeros(p.shape, dtype=torch.float64)
                t.append(0)
            elif bits == 8:
                a, b = (x.double().cpu() for x in decode_moments(st["exp_avg"], st["exp_avg_sq"], st["scales"]))
                t.append(int(st["step"]))
            else:
                a, b = st["exp_avg"].double().cpu(), st["exp_avg_sq"].double().cpu()
                t.append(int(st["step"]))
            m.append(a.clone())
            v.append(b.clone())
        return cls([p.detach().double().cpu().clone() for p in params], m, v, t, bits,
                   [p.dtype == torch.bfloat16 for p in params])

    def step(self, grads, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, maximize=False, max_grad_norm=None,
             seed=0):
        b1, b2 = betas
        f = 1.0
        if max_grad_norm is not None:
            self.norm = math.sqrt(sum(float(g.square().sum()) for g in grads))
            f = min(1.0, max_grad_norm / (self.norm + 1e-6))
        self.m_terms, self.upd_terms = [], []     # the larger term of m, and the update if nothing cancelled in it
        for i, g in enumerate(grads):
            g = g * (-f if maximize else f)
            self.t[i] += 1
            t = self.t[i]
            self.m_terms.append(torch.maximum((b1 * self.m[i]).abs(), ((1 - b1) * g).abs()))
            m = b1 * self.m[i] + (1 - b1) * g
            v = b2 * self.v[i] + (1 - b2) * g * g
            p = self.p[i] * (1 - lr * weight_decay)
            den = torch.sqrt(v / (1 - b2 ** t)) + eps
            self.upd_terms.append(lr * self.m_terms[i] / (1 - b1 ** t) / den)
            p = p - lr * (m / (1 - b1 ** t)) / den
            h = hashes(g.numel(), seed, i, t)
            if self.bits == 8:
                s = m.shape
                m = (to_grid(m.abs().view(-1), h & 0xFFFF, -14, False) * torch.sign(m.view(-1))).view(s)
                v = to_grid(v.view(-1), h >> 16, -30, True).view(s)
            if self.low[i]:
                unit = torch.ldexp(torch.ones(()).double(), torch.frexp(p)[1] - 8)
                cut = p.abs() / unit
                up = (cut - torch.floor(cut)) + ((((h * SQ2) & MASK) >> 16).double() / 65536).view(p.shape) >= 1
                p = (torch.floor(cut) + up) * unit * torch.sign(p)
            self.p[i], self.m[i], self.v[i] = p, m, v
