"""AdamW over many tensors with the moments in 8 or 32 bits, and clipping by the global gradient norm
(``csrc/hip/adamw.hip``; public names in :mod:`raydp_amd.ops.fused_optim`).

* :class:`FusedAdamW` -- ``torch.optim.AdamW``'s update (decoupled weight decay) as one launch per 64 tensors.
  Parameters are contiguous fp32 or bf16. ``state_bits=8`` keeps each moment in one byte plus two scale bytes per 256
  elements (2.01 bytes per parameter where fp32 moments take 8); ``state_bits=32`` keeps them in fp32. fp32 weights
  that a fused Linear tower reads get their bf16 image in the same pass; bf16 parameters have no master copy and are
  rounded stochastically. Step counts live on the device, so a step can be captured into a HIP graph once an eager step
  has made the state.
* :func:`clip_grad_norm_` -- ``torch.nn.utils.clip_grad_norm_`` (2-norm) in two launches per 256 tensors, without a host
  read. ``FusedAdamW(max_grad_norm=...)`` applies the same factor inside the step instead, without the pass that
  rewrites the gradients.
* :func:`decode_moments` -- the values that 8-bit moments stand for.

On the CPU the same operators are computed by torch expressions with the same codes.
"""
import math
from typing import Iterable, Optional, Tuple, Union

import torch

BLOCK = 256                  # elements of a tensor that share a scale
_M_EMIN, _V_EMIN = -14, -30
_MASK, _PHI, _SQ2, _SQ3 = 0xFFFFFFFF, 0x9E3779B1, 0x6A09E667, 0xBB67AE85


_module = None


def _ext():
    global _module
    if _module is None:
        from raydp_amd.native import loader
        _module = loader.load_torch()
    return _module


# --------------------------------------------------------------------------------------- moments in 8 bits
def _mix(x):
    x = ((x ^ (x >> 16)) * _SQ2) & _MASK
    x = ((x ^ (x >> 15)) * _SQ3) & _MASK
    return x ^ (x >> 16)


def _dither(n: int, seed: int, ordinal: int, step: int, device):
    """32 random bits for each of ``n`` elements, as csrc/hip/adamw.hip makes them (in int64)."""
    key = _mix((_mix((seed + ordinal * _PHI) & _MASK) + step) & _MASK)
    i = torch.arange(n, device=device)
    return _mix(((i & _MASK) * _PHI + (i >> 32) * _SQ2 + key) & _MASK)


def _pow2(e):
    return ((e + 1023) << 52).view(torch.float64)


def _blocks(x):
    """[blocks, 256] of a flat tensor, the last block filled up with zeros."""
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _encode(x, rnd16, emin):
    """(codes, biased scale exponents) of blocks of non-negative fp32 values: 3 mantissa bits, normal from 2^emin. A scale of
    255 marks a block with a NaN (of any sign and payload) or an infinity."""
    s = (((x.view(torch.int32) & 0x7FFFFFFF).long().amax(1) + 0xFFFFF) >> 23).clamp(max=255)
    y = x.double() * _pow2(127 - s.clamp(min=1))[:, None]
    f = ((y.view(torch.int64) >> 52) - 1023).clamp(min=emin)
    code = ((torch.round(y * _pow2(3 - f) * 2.0 ** 20).long() + rnd16 * 16 + 8) >> 20) + 8 * (f - emin)
    return torch.where((s == 255)[:, None], 0, code), s


def _decode(code, s, emin):
    e, man = code >> 3, code & 7
    y = torch.where(e > 0, (8 + man).double() * _pow2(e.clamp(min=1) - 1 + emin - 3), man.double() * 2.0 ** (emin - 3))
    return (y * torch.where(s == 255, math.nan, _pow2(s.clamp(min=1) - 127))[:, None]).float()


def _encode_moments(m, v, h):
    """(exp_avg, exp_avg_sq, scales) in 8 bits from fp32 moments and 32 dither bits per element."""
    h = _blocks(h)
    mb, vb = _blocks(m.reshape(-1)), _blocks(v.reshape(-1))
    mc, ms = _encode(mb.abs(), h & 0xFFFF, _M_EMIN)
    mc = mc | ((mb.view(torch.int32) < 0) & (ms != 255)[:, None]).long() * 128
    vc, vs = _encode(vb, h >> 16, _V_EMIN)
    vc = torch.where((vb > 0) & (vs != 255)[:, None], vc.clamp(min=1), vc)    # it is divided by
    n, scales = m.numel(), torch.stack([ms, vs], 1).to(torch.uint8)
    return (mc.to(torch.uint8).view(-1)[:n].view(m.shape), vc.to(torch.uint8).view(-1)[:n].view(v.shape), scales)


def _scale_rows(n: int) -> int:
    return -(-n // BLOCK)


def decode_moments(exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor, scales: torch.Tensor,
                   dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values of one parameter's 8-bit moments (``state[p]["exp_avg"]``, ``["exp_avg_sq"]``, ``["scales"]``) in
    ``dtype`` (fp32 or bf16: a code has 4 significant bits, so both hold it exactly). A block that held a value which
    was not finite decodes to NaN."""
    n = exp_avg.numel()
    for t, name in ((exp_avg, "exp_avg"), (exp_avg_sq, "exp_avg_sq"), (scales, "scales")):
        if t.dtype != torch.uint8 or not t.is_contiguous():
            raise ValueError(f"decode_moments: {name} must be contiguous uint8 (8-bit moments)")
        if t.device != exp_avg.device:
            raise ValueError("decode_moments: moments and scales are on different devices")
    if exp_avg_sq.shape != exp_avg.shape or scales.numel() != 2 * _scale_rows(n):
        raise ValueError(f"decode_moments: {n} elements need moments of one shape and {2 * _scale_rows(n)} scale bytes, "
                         f"got {tuple(exp_avg_sq.shape)} and {scales.numel()}")
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"decode_moments: dtype {dtype} (fp32 or bf16)")
    if not exp_avg.is_cuda:
        mc, vc, s = (t.long() for t in (_blocks(exp_avg.view(-1)), _blocks(exp_avg_sq.view(-1)), scales.view(-1, 2)))
        m = _decode(mc & 127, s[:, 0], _M_EMIN) * (1 - (mc >> 7) * 2)
        v = _decode(vc, s[:, 1], _V_EMIN)
        return tuple(t.view(-1)[:n].view(exp_avg.shape).to(dtype) for t in (m, v))
    if (exp_avg.data_ptr() | exp_avg_sq.data_ptr()) & 3 or scales.data_ptr() & 1:
        raise ValueError("decode_moments: moments must start at a multiple of 4 bytes, scales at an even address")
    return tuple(_ext().decode_moments(exp_avg, exp_avg_sq, scales, dtype == torch.bfloat16))


# --------------------------------------------------------------------------------------- norm and clipping
@torch.no_grad()
def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float) -> torch.Tensor:
    """Scale the gradients of ``parameters`` in place by ``min(1, max_norm / (norm + 1e-6))``, ``norm`` their global
    2-norm (summed in 64 bits), and return the norm (0-dim fp32, on the gradients' device, without a host
    synchronisation). Gradients are dense (in any dimension order) fp32 or bf16; a gradient that is listed twice
    counts once, and gradients that share memory otherwise raise. A norm that is not finite is not kept from the gradients
    (a NaN makes all of them NaN, an infinity 0 and NaN), as in ``torch.nn.utils.clip_grad_norm_``."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grad_norm_: max_norm must not be negative, got {max_norm}")
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = list({id(g): g for g in (p.grad for p in parameters) if g is not None}.values())
    if not grads:
        return torch.zeros(())
    if grads[0].is_cuda:
        return _ext().clip_grad_norm(grads, max_norm)
    for g in grads:
        if g.layout != torch.strided:
            raise ValueError("clip_grad_norm_: sparse gradients are not supported")
        if g.device != grads[0].device:
            raise ValueError(f"clip_grad_norm_: gradients on {grads[0].device} and {g.device}")
        if g.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError(f"clip_grad_norm_: gradient dtype {g.dtype} (fp32 or bf16)")
        if not _dense(g):
            raise ValueError("clip_grad_norm_: gradients must be dense (no gaps, no broadcast dimensions)")
    _check_overlap(grads, "clip_grad_norm_: gradients")
    norm = torch.sqrt(sum(g.double().square().sum() for g in grads))
    f = (max_norm / (norm + 1e-6)).clamp(max=1.0).float()
    for g in grads:
        g.copy_(g.float() * f)
    return norm.float()


def _check_overlap(tensors, what):
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors if t.numel())
    if any(b[0] < a[1] for a, b in zip(spans, spans[1:])):
        raise ValueError(f"{what} share memory")


def _dense(t: torch.Tensor) -> bool:
    """Every element once, without gaps, in whatever order."""
    need = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda v: v[1]):
        if stride != need:
            return False
        need *= size
    return True


# --------------------------------------------------------------------------------------- the optimizer
class FusedAdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` on the multi-tensor kernels, with the moments in 8 or 32 bits.

    ``state_bits``      8: one byte per moment and two scale bytes per 256 elements, rounded stochastically (the hash of
                        ``seed``, the parameter's place, the step and the element's index: the same run gives the same
                        bits); 32: fp32.
    ``max_grad_norm``   clip by the global 2-norm of all gradients inside the step (``.grad`` is left as it is; the norm
                        is ``self.grad_norm``, on the device). A step whose norm is not finite is left out: parameters,
                        moments and step counts stay as they are. None: no clipping, nothing is left out.
    ``lr``              a number, or a 0-dim fp32 tensor on the parameters' device (read by the kernel: a captured step
                        sees what a scheduler fills in). A tensor on the host is read at every step and cannot be captured;
                        ``load_state_dict`` moves one to the parameters' device.

    State per parameter: ``step`` (0-dim fp32 on the parameter's device), ``exp_avg``, ``exp_avg_sq`` (uint8 codes or
    fp32) and, for 8 bits, ``scales`` (uint8 ``[ceil(n / 256), 2]``); :func:`decode_moments` gives their values.
    ``load_state_dict`` also takes the state of a ``torch.optim.AdamW`` and codes its moments; one with ``amsgrad``, or of a
    ``torch.optim.Adam`` whose ``weight_decay`` meant another thing, raises before anything is changed.

    ``eps`` is 0 or at least 2^-126. Parameters are contiguous fp32 or bf16; gradients are dense and of the parameter's
    type. Sparse gradients, parameters that share memory, a first step inside a graph capture raise."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 8, max_grad_norm: Optional[float] = None, maximize: bool = False, seed: int = 0):
        self._check_options(dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                 max_grad_norm=max_grad_norm, seed=seed))
        super().__init__(params, dict(lr=lr, betas=tuple(float(b) for b in betas), eps=float(eps),
                                      weight_decay=float(weight_decay), state_bits=int(state_bits),
                                      max_grad_norm=None if max_grad_norm is None else float(max_grad_norm),
                                      maximize=bool(maximize), seed=int(seed)))
        self.grad_norm: Optional[torch.Tensor] = None

    @staticmethod
    def _check_options(o):
        lr, eps, betas, clip = o["lr"], o["eps"], o["betas"], o["max_grad_norm"]
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1:
                raise ValueError("FusedAdamW: a tensor lr must have one element")
        elif not 0.0 <= lr:
            raise ValueError(f"FusedAdamW: invalid learning rate {lr}")
        if eps != 0.0 and not eps >= 2.0 ** -126:
            raise ValueError(f"FusedAdamW: eps must be 0 or a normal fp32 number (at least 2^-126), got {eps}")
        if len(betas) != 2 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"FusedAdamW: invalid betas {betas}")
        if not o["weight_decay"] >= 0.0:
            raise ValueError(f"FusedAdamW: invalid weight_decay {o['weight_decay']}")
        if o["state_bits"] not in (8, 32):
            raise ValueError(f"FusedAdamW: state_bits is 8 or 32, got {o['state_bits']}")
        if clip is not None and not clip >= 0.0:
            raise ValueError(f"FusedAdamW: invalid max_grad_norm {clip}")
        if not 0 <= int(o["seed"]) <= _MASK:
            raise ValueError(f"FusedAdamW: seed must fit 32 bits, got {o['seed']}")

    def __setstate__(self, state):
        super().__setstate__(state)
        self._fill_groups()
        self.__dict__.setdefault("grad_norm", None)

    def _fill_groups(self):
        for g in self.param_groups:      # (a state dict of torch.optim.AdamW has fewer options)
            for k, v in self.defaults.items():
                g.setdefault(k, v)

    def add_param_group(self, group):
        super().add_param_group(group)
        params = self.param_groups[-1]["params"]
        try:
            self._check_options(self.param_groups[-1])
            for p in params:
                if p.dtype not in (torch.float32, torch.bfloat16):
                    raise TypeError(f"FusedAdamW: parameter dtype {p.dtype} (fp32 or bf16)")
            if len({id(p) for p in params}) < len(params):
                raise ValueError("FusedAdamW: a parameter is listed twice")
        except (TypeError, ValueError):
            self.param_groups.pop()
            raise

    def load_state_dict(self, state_dict):
        saved = state_dict["state"]
        # torch casts floating state to the parameter's type and codes with it: the saved bits are put back below
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        mine = [p for g in self.param_groups for p in g["params"]]
        for k, (i, p) in enumerate(zip(ids, mine)):
            if saved.get(i):
                self._check_saved(saved[i], k, p)
        for g in state_dict["param_groups"]:
            self._check_options({**self.defaults, **g})
            if g.get("amsgrad"):
                raise ValueError("FusedAdamW: the state is of an amsgrad optimizer, whose largest second moments it does not keep")
            if g.get("weight_decay") and g.get("decoupled_weight_decay") is False:
                raise ValueError("FusedAdamW: the state is of an Adam whose weight_decay was added to the gradients; here "
                                 "it shrinks the parameters (for that, set decoupled_weight_decay in the state's group)")
        super().load_state_dict(state_dict)
        self._fill_groups()
        for g in self.param_groups:      # a checkpoint's rate is read where the step is: a captured one sees what is filled in
            if isinstance(g["lr"], torch.Tensor) and not g["lr"].is_cuda and g["params"] and g["params"][0].is_cuda:
                g["lr"] = g["lr"].detach().to(g["params"][0].device, torch.float32)
        params = [(g, p) for g in self.param_groups for p in g["params"]]
        for i, (g, p) in zip(ids, params):
            src = saved.get(i)
            if not src:
                continue
            st = {"step": torch.as_tensor(src["step"], dtype=torch.float32).detach().clone().to(p.device)}
            m, v = (src[n].detach().to(p.device) for n in ("exp_avg", "exp_avg_sq"))
            coded = m.dtype == torch.uint8
            if coded:
                sc = src["scales"].detach().to(p.device, copy=True).contiguous()
            m, v = (t.clone(memory_format=torch.contiguous_format) for t in (m, v))
            if g["state_bits"] == 8:
                if not coded:
                    half = torch.full((p.numel(),), (1 << 31) | (1 << 15), dtype=torch.int64, device=p.device)
                    m, v, sc = _encode_moments(m.float(), v.float(), half)
                st.update(exp_avg=m, exp_avg_sq=v, scales=sc)
            else:
                m, v = decode_moments(m, v, sc) if coded else (m.float(), v.float())
                st.update(exp_avg=m, exp_avg_sq=v)
            self.state[p] = st

    @staticmethod
    def _check_saved(src, k, p):
        if any(n not in src for n in ("step", "exp_avg", "exp_avg_sq")):
            raise ValueError(f"FusedAdamW: state of parameter {k} lacks step, exp_avg or exp_avg_sq")
        m, v = src["exp_avg"], src["exp_avg_sq"]
        if m.shape != p.shape or v.shape != p.shape:
            raise ValueError(f"FusedAdamW: moments of parameter {k} are {tuple(m.shape)}, the parameter is {tuple(p.shape)}")
        if torch.uint8 in (m.dtype, v.dtype):
            sc = src.get("scales")
            if sc is None or m.dtype != v.dtype or sc.dtype != torch.uint8 or sc.numel() != 2 * _scale_rows(p.numel()):
                raise ValueError(f"FusedAdamW: 8-bit state of parameter {k} is incomplete")

    def _new_state(self, p, bits):
        """The parameter's state, made with its first gradient."""
        if p.grad.layout != torch.strided:
            raise RuntimeError("FusedAdamW does not support sparse gradients")
        if not p.is_contiguous():
            raise ValueError("FusedAdamW: parameters must be contiguous")
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedAdamW: the first step of a parameter cannot be captured into a graph (its state "
                               "would be zeroed by every replay): run one eager step first")
        st = self.state[p]
        st["step"] = torch.zeros((), dtype=torch.float32, device=p.device)
        kind = torch.uint8 if bits == 8 else torch.float32
        for n in ("exp_avg", "exp_avg_sq"):
            st[n] = torch.zeros(p.shape, dtype=kind, device=p.device)
        if bits == 8:
            st["scales"] = torch.zeros(_scale_rows(p.numel()), 2, dtype=torch.uint8, device=p.device)
        return st

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        state, steps, owners, place, clip, seed = self.state, [], [], 0, None, None
        for group in self.param_groups:
            params, grads, places, images = [], [], [], {}
            for o, p in enumerate(group["params"], place):
                g = p.grad
                if g is not None:
                    if getattr(p, "_raydp_image_owner", None) is not None and p.is_cuda:
                        self._image(p, len(params), images, owners)
                    params.append(p)
                    grads.append(g)
                    places.append(o)
            place += len(group["params"])
            if not params:
                continue
            if seed is None:
                clip, seed = group["max_grad_norm"], group["seed"]
            elif group["max_grad_norm"] != clip or group["seed"] != seed:
                raise ValueError("FusedAdamW: max_grad_norm and seed are the optimizer's, not a group's")
            bits = group["state_bits"]
            if bits not in (8, 32):
                raise ValueError(f"FusedAdamW: state_bits is 8 or 32, got {bits}")
            states = [state[p] or self._new_state(p, bits) for p in params]
            steps.append((params, grads, states, places, images, group))
        if not steps:
            if self.param_groups[0]["max_grad_norm"] is not None:
                self.grad_norm = torch.zeros((), device=next(p for g in self.param_groups for p in g["params"]).device)
            return loss
        if steps[0][0][0].is_cuda:
            norm = _ext().adamw_step(steps, -1.0 if clip is None else clip, seed)
            if clip is not None:          # (None: nothing but empty tensors)
                self.grad_norm = norm if norm is not None else torch.zeros((), device=steps[0][0][0].device)
            for tower, li in owners:
                tower.image_updated(li)
        else:
            with torch.no_grad():
                self._cpu_step(steps, clip)
        return loss

    @staticmethod
    def _image(p, index, images, owners):
        from raydp_amd.ops.fused_optim import _image_of
        tower, li, img = _image_of(p)
        if img is not None:
            # (a step that is left out writes no image: it has to be the weight's before)
            if tower._versions[li] != (p.data_ptr(), p._version):
                tower._refresh_images()
            images[index] = img
            owners.append((tower, li))

    # ------------------------------------------------------------------ CPU
    def _cpu_step(self, groups, clip):
        scale, dev = 1.0, groups[0][0][0].device
        for params, grads, states, _, _, group in groups:
            for p, g, st in zip(params, grads, states):
                if g.layout != torch.strided:
                    raise RuntimeError("FusedAdamW does not support sparse gradients")
                if p.device != dev or g.device != dev:
                    raise ValueError(f"FusedAdamW: parameters with gradients on {dev} and {p.device}")
                if p.dtype not in (torch.float32, torch.bfloat16) or g.dtype != p.dtype:
                    raise TypeError(f"FusedAdamW: parameter {p.dtype} with gradient {g.dtype} (both fp32 or both bf16)")
                if not p.is_contiguous():
                    raise ValueError("FusedAdamW: parameters must be contiguous")
                if (st["exp_avg"].dtype == torch.uint8) != (group["state_bits"] == 8):
                    raise ValueError(f"FusedAdamW: state_bits is {group['state_bits']}, the moments of a parameter are "
                                     f"{st['exp_avg'].dtype}")
        _check_overlap([p for params, *_ in groups for p in params], "FusedAdamW: parameters")
        if clip is not None:
            norm = torch.sqrt(sum(g.double().square().sum() for _, grads, _, _, _, _ in groups for g in grads))
            self.grad_norm = norm.float()
            if not bool(torch.isfinite(norm)):
                return
            scale = (clip / (norm + 1e-6)).clamp(max=1.0).float()
        for params, grads, states, places, _, group in groups:
            b1, b2 = group["betas"]
            bits, lr = group["state_bits"], float(group["lr"])
            for p, g, st, place in zip(params, grads, states, places):
                if not p.numel():
                    continue
                st["step"] += 1
                t = int(st["step"])
                g = g.float() * (-scale if group["maximize"] else scale)
                m, v = (st["exp_avg"], st["exp_avg_sq"]) if bits == 32 else \
                    decode_moments(st["exp_avg"], st["exp_avg_sq"], st["scales"])
                m = m * b1 + g * (1 - b1)
                v = v * b2 + (g * g) * (1 - b2)
                den = torch.sqrt(v) * (1.0 / math.sqrt(1.0 - b2 ** t)) + group["eps"]
                new = p.float() * (1.0 - lr * group["weight_decay"]) + m / den * (-lr / (1.0 - b1 ** t))
                low = p.dtype == torch.bfloat16
                h = _dither(p.numel(), group["seed"], place, t, p.device) if bits == 8 or low else None
                if bits == 8:
                    codes = _encode_moments(m, v, h)
                    for n, c in zip(("exp_avg", "exp_avg_sq", "scales"), codes):
                        st[n].copy_(c)
                else:
                    st["exp_avg"].copy_(m)
                    st["exp_avg_sq"].copy_(v)
                if low:
                    b = new.view(torch.int32).long() & _MASK
                    r = (((h * _SQ2) & _MASK) >> 16).view(p.shape)
                    b = torch.where(torch.isnan(new), b, b + r) >> 16 << 16
                    new = torch.where(b > 0x7FFFFFFF, b - (1 << 32), b).int().view(torch.float32)
                p.copy_(new)
