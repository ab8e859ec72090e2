"""Routed experts (``csrc/hip/experts.hip``): a router's top-k softmax, samples sorted by expert, and back with weights.

    weights, experts = route(logits, k)                 # [T, k] fp32, [T, k] int32 (-1: none)
    plan = expert_plan(experts, num_experts, capacity)  # a stable counting sort; capacity None: no sample is dropped
    rows = dispatch(x, plan)                            # [R, D]: expert e owns rows offsets[e] .. offsets[e] + load[e]
    y = combine(f(rows), plan, weights)                 # [T, D]: sum over a sample's experts

Nothing is read back to the host, so a step with them can be captured into a HIP graph; with a ``capacity`` every expert's
rows are a slice of fixed size (``rows.view(num_experts, capacity, D)``) that a ``FusedLinearTower`` takes as it is.

``route``, ``dispatch`` and ``combine`` are differentiable (once). On the GPU all run on the HIP kernels and fail loudly if
the library is missing; on the CPU they are the equivalent PyTorch expressions (any floating type, for tests and CPU-only
hosts).
"""
import contextlib
import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from raydp_amd.ops import _hip

MAX_EXPERTS, MAX_TOPK = 1024, 32
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_VEC = {0: 4, 1: 8, 2: 8}          # elements of a 16-byte vector
_INT32 = 0x7FFFFFFF
LAST_LEVEL = 256 << 20          # bytes of the last-level cache


class PlanArgs(ctypes.Structure):
    _fields_ = [("ids", ctypes.c_void_p), ("wide", ctypes.c_int), ("n", ctypes.c_int), ("E", ctypes.c_int),
                ("chunk", ctypes.c_int), ("blocks", ctypes.c_int), ("capacity", ctypes.c_int), ("rows", ctypes.c_int),
                ("pad_", ctypes.c_int), ("counts", ctypes.c_void_p), ("position", ctypes.c_void_p),
                ("source", ctypes.c_void_p), ("load", ctypes.c_void_p), ("offsets", ctypes.c_void_p)]


class RowArgs(ctypes.Structure):
    _fields_ = [("T", ctypes.c_longlong), ("rows", ctypes.c_longlong), ("ldx", ctypes.c_longlong), ("k", ctypes.c_int),
                ("D", ctypes.c_int), ("lg", ctypes.c_int), ("stream", ctypes.c_int), ("position", ctypes.c_void_p),
                ("source", ctypes.c_void_p), ("x", ctypes.c_void_p), ("w", ctypes.c_void_p), ("h", ctypes.c_void_p),
                ("out", ctypes.c_void_p), ("dw", ctypes.c_void_p)]


_bound = None


def _lib():
    global _bound
    L = _hip.lib()
    if _bound is not L:
        vp, i, ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
        L.rx_route_fwd.argtypes = [vp, ll, i, ll, i, i, i, vp, vp, vp, vp]
        L.rx_route_bwd.argtypes = [vp, ll, i, vp, vp, vp, vp, ll, i, i, vp, vp]
        L.rx_expert_plan.argtypes = [vp, vp, vp]
        L.rx_rows_scatter.argtypes = [vp, i, vp]
        L.rx_rows_gather.argtypes = [vp, i, vp]
        for n in ("rx_route_fwd", "rx_route_bwd", "rx_expert_plan", "rx_rows_scatter", "rx_rows_gather"):
            getattr(L, n).restype = i
        L.rx_expert_sizes.argtypes = [vp]
        L.rx_expert_sizes.restype = None
        got = (ctypes.c_int * 4)()
        L.rx_expert_sizes(got)
        want = [ctypes.sizeof(PlanArgs), ctypes.sizeof(RowArgs), MAX_EXPERTS, MAX_TOPK]
        if list(got) != want:
            raise RuntimeError(f"layout mismatch between Python and csrc/hip/experts.hip: C {list(got)} vs {want}")
        _bound = L
    return L


def _on(device):
    return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """``t`` with contiguous rows (any distance between them)."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


# ------------------------------------------------------------------------------------------------ router
def _route_gpu(z, k, renormalize, keep):
    T, E = z.shape
    w = torch.empty(T, k, dtype=torch.float32, device=z.device)
    ids = torch.empty(T, k, dtype=torch.int32, device=z.device)
    norm = torch.empty(T, 2, dtype=torch.float32, device=z.device) if keep else None
    with _on(z.device):
        _hip.check(_lib().rx_route_fwd(z.data_ptr(), z.stride(0), _DTYPES[z.dtype], T, E, k, int(renormalize),
                                       w.data_ptr(), ids.data_ptr(), norm.data_ptr() if keep else None,
                                       _hip.stream_ptr(z.device)), "rx_route_fwd")
    return w, ids, norm


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, renormalize):
        z = _rows_of(logits)
        w, ids, norm = _route_gpu(z, k, renormalize, not renormalize)
        # the gradient of the renormalised weights needs no logits
        ctx.save_for_backward(*((w, ids) if renormalize else (w, ids, norm, z)))
        ctx.meta = (tuple(logits.shape), logits.dtype)
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        return w, ids

    @staticmethod
    @once_differentiable
    def backward(ctx, dw, _):
        if dw is None:
            return None, None, None
        w, ids = ctx.saved_tensors[:2]
        norm, z = ctx.saved_tensors[2:] if len(ctx.saved_tensors) == 4 else (None, None)
        (T, E), dtype = ctx.meta
        dw = dw.contiguous()
        dz = torch.empty(T, E, dtype=dtype, device=w.device)
        with _on(w.device):
            _hip.check(_lib().rx_route_bwd(z.data_ptr() if z is not None else None, z.stride(0) if z is not None else 0,
                                           _DTYPES[dtype], norm.data_ptr() if norm is not None else None, w.data_ptr(),
                                           ids.data_ptr(), dw.data_ptr(), T, E, w.shape[1], dz.data_ptr(),
                                           _hip.stream_ptr(w.device)), "rx_route_bwd")
        return dz, None, None


def route(logits: torch.Tensor, k: int, renormalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """The ``k`` experts of every sample and their weights: ``[T, k]`` fp32 weights (differentiable) and int32 experts, in
    the order of the logits (ties: the lowest expert first).

    ``logits``       ``[T, E]``, fp32, bf16 or fp16; at most 1024 experts, ``k`` at most 32
    ``renormalize``  True: weights of a sample are the softmax over its chosen experts (they sum to 1); False: the chosen
                     entries of the softmax over all experts

    An expert whose logit is ``-inf`` is never chosen; a sample with fewer than ``k`` others gets expert -1 with weight 0
    in the places that are left (all of them, for a padding row of ``-inf``). A NaN is not chosen and makes the weights of
    its row NaN."""
    if logits.dim() != 2 or not logits.is_floating_point():
        raise ValueError(f"route: logits must be floating [T, E], got {logits.dtype} {tuple(logits.shape)}")
    T, E = logits.shape
    k = int(k)
    if not 1 <= k <= min(E, MAX_TOPK):
        raise ValueError(f"route: k must be between 1 and min(E, {MAX_TOPK}), got k={k} with E={E}")
    if E > MAX_EXPERTS:
        raise ValueError(f"route: at most {MAX_EXPERTS} experts, got {E}")
    if not logits.is_cuda:
        return _route_cpu(logits, k, renormalize)
    if logits.dtype not in _DTYPES:
        raise TypeError(f"route: logits dtype {logits.dtype} (fp32, bf16 or fp16)")
    if logits.requires_grad and torch.is_grad_enabled():
        return _Route.apply(logits, k, bool(renormalize))
    return _route_gpu(_rows_of(logits), k, renormalize, False)[:2]


def _route_cpu(logits, k, renormalize):
    z = logits.float() if logits.dtype in (torch.bfloat16, torch.float16) else logits
    bad = torch.isnan(z)
    order = torch.sort(z.detach().masked_fill(bad, -torch.inf), dim=1, descending=True, stable=True)
    top, ids = order.values[:, :k], order.indices[:, :k]
    there = top > -torch.inf
    peak = torch.where(there[:, :1], top[:, :1], 0.0)
    part = torch.where(there, torch.exp(z.gather(1, ids).masked_fill(~there, 0.0) - peak), 0.0)
    total = part.sum(1, keepdim=True) if renormalize else torch.exp(z - peak).sum(1, keepdim=True)
    w = part / torch.where(total == 0, 1.0, total)
    w = torch.where(bad.any(1, keepdim=True), torch.nan, w)
    return (w.float() if z.dtype == torch.float32 else w), torch.where(there, ids, -1).int()


# ------------------------------------------------------------------------------------------------ plan
class ExpertPlan:
    """Where every choice of expert goes (all tensors int32, on the experts' device).

    ``position``  ``[T, k]``: the row of sample t's j-th choice, -1 where it has none or its expert is full
    ``source``    ``[rows]``: the choice ``t * k + j`` that fills a row, -1 for a row that stays empty
    ``load``      ``[E]``: how many choices asked for an expert (with a capacity: also those that were dropped)
    ``offsets``   ``[E + 1]``: an expert's first row
    ``rows``      ``E * capacity``, or ``T * k`` without a capacity"""
    __slots__ = ("position", "source", "load", "offsets", "tokens", "k", "num_experts", "capacity", "rows")

    def __init__(self, position, source, load, offsets, num_experts, capacity):
        self.position, self.source, self.load, self.offsets = position, source, load, offsets
        self.tokens, self.k = position.shape
        self.num_experts, self.capacity, self.rows = num_experts, capacity, source.shape[0]


def expert_plan(experts: torch.Tensor, num_experts: int, capacity: Optional[int] = None) -> ExpertPlan:
    """Sort the choices ``experts`` (``[T, k]`` int32 or int64) by expert, stably: an expert's rows are in the order of
    ``t * k + j``. -1, and any other number that is no expert, is no choice. ``capacity`` (None: unlimited): rows of every
    expert; later choices of a full expert are dropped."""
    if experts.dim() != 2 or experts.shape[1] < 1 or experts.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"expert_plan: experts must be int32 or int64 [T, k], got {experts.dtype} {tuple(experts.shape)}")
    E = int(num_experts)
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"expert_plan: num_experts must be between 1 and {MAX_EXPERTS}, got {E}")
    if capacity is not None and int(capacity) < 1:
        raise ValueError(f"expert_plan: capacity must be positive, got {capacity}")
    T, k = experts.shape
    n, C = T * k, int(capacity) if capacity is not None else 0
    rows = E * C if C else n
    if max(n, rows) > _INT32:
        raise ValueError(f"expert_plan: {max(n, rows)} choices or rows do not fit 32 bits")
    if not experts.is_cuda:
        return _plan_cpu(experts, E, C, rows)
    dev = experts.device
    ids = experts if experts.is_contiguous() else experts.contiguous()
    chunk, blocks = _plan_grid(n)
    # one allocation: position, source, load, offsets, scratch
    buf = torch.empty(n + rows + 2 * E + 1 + (blocks * E if blocks > 1 else 0), dtype=torch.int32, device=dev)
    at = buf.data_ptr()
    a = PlanArgs(ids.data_ptr(), int(ids.dtype == torch.int64), n, E, chunk, blocks, C, rows, 0, None, at, at + 4 * n,
                 at + 4 * (n + rows), at + 4 * (n + rows + E))
    with _on(dev):
        _hip.check(_lib().rx_expert_plan(ctypes.byref(a), at + 4 * (n + rows + 2 * E + 1) if blocks > 1 else None,
                                         _hip.stream_ptr(dev)), "rx_expert_plan")
    return ExpertPlan(buf[:n].view(T, k), buf[n:n + rows], buf[n + rows:n + rows + E],
                      buf[n + rows + E:n + rows + 2 * E + 1], E, C or None)


def _plan_grid(n: int) -> Tuple[int, int]:
    """(choices per workgroup, workgroups): one workgroup up to 4096 choices, which needs one launch and not two; at most
    256 workgroups beyond, as each sums the counts of all."""
    if n <= 4096:
        return max(1024, -(-n // 1024) * 1024), 1
    chunk = max(1024, -(-n // (256 * 1024)) * 1024)
    return chunk, -(-n // chunk)


def _plan_cpu(experts, E, C, rows):
    T, k = experts.shape
    flat = experts.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.sort(key, stable=True).indices
    load = torch.bincount(key, minlength=E + 1)
    start = torch.cumsum(load, 0) - load
    rank = torch.empty_like(order)
    rank[order] = torch.arange(key.numel()) - start[key[order]]
    base = torch.arange(E + 1) * C if C else start
    keep = (key < E) & ((rank < C) if C else True)
    position = torch.where(keep, base[key] + rank, -1)
    source = torch.full((rows,), -1, dtype=torch.int64)
    source[position[keep]] = torch.nonzero(keep).flatten()
    return ExpertPlan(position.view(T, k).int(), source.int(), load[:E].int(), base.int(), E, C or None)


# ------------------------------------------------------------------------------------------------ rows
def _row_args(plan, D, dtype, x=None, ldx=0, w=None, h=None, out=None, dw=None):
    code = _DTYPES[dtype]
    units = -(-D // _VEC[code])
    # samples' rows and expert rows, these twice where products are taken: more than the last-level cache is streamed past it
    touched = (plan.tokens + plan.rows * (2 if dw is not None else 1)) * D * dtype.itemsize
    a = RowArgs(plan.tokens, plan.rows, ldx, plan.k, D, min(6, (units - 1).bit_length()), int(touched > LAST_LEVEL),
                plan.position.data_ptr(), plan.source.data_ptr())
    a.x, a.w, a.h, a.out, a.dw = (t.data_ptr() if t is not None else None for t in (x, w, h, out, dw))
    return a, code


def _scatter(plan, x, w=None, h=None):
    """(expert rows with ``x`` (times ``w``) in them, inner products with ``h`` or None)."""
    D = x.shape[1]
    x = _rows_of(x)
    out = torch.empty(plan.rows, D, dtype=x.dtype, device=x.device)
    dw = torch.empty(plan.tokens, plan.k, dtype=torch.float32, device=x.device) if h is not None else None
    a, code = _row_args(plan, D, x.dtype, x, x.stride(0), w, h, out, dw)
    with _on(x.device):
        _hip.check(_lib().rx_rows_scatter(ctypes.byref(a), code, _hip.stream_ptr(x.device)), "rx_rows_scatter")
    return out, dw


def _gather(plan, h, w=None):
    D = h.shape[1]
    out = torch.empty(plan.tokens, D, dtype=h.dtype, device=h.device)
    a, code = _row_args(plan, D, h.dtype, w=w, h=h, out=out)
    with _on(h.device):
        _hip.check(_lib().rx_rows_gather(ctypes.byref(a), code, _hip.stream_ptr(h.device)), "rx_rows_gather")
    return out


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.plan = plan
        return _scatter(plan, x)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        return _gather(ctx.plan, g.contiguous()), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, plan):
        ctx.plan = plan
        ctx.weighted = weights is not None
        if weights is not None:
            ctx.save_for_backward(weights, *((rows,) if ctx.needs_input_grad[1] else ()))
        return _gather(plan, rows, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        if not ctx.weighted:
            return _scatter(ctx.plan, g)[0], None, None
        w, rows = ctx.saved_tensors if len(ctx.saved_tensors) == 2 else (ctx.saved_tensors[0], None)
        drows, dw = _scatter(ctx.plan, g, w, rows)
        return drows, dw, None


def _check_rows(t, plan, want, what):
    if t.dim() != 2 or t.shape[0] != want or t.shape[1] < 1 or not t.is_floating_point():
        raise ValueError(f"{what}: expected floating [{want}, D] for this plan, got {t.dtype} {tuple(t.shape)}")
    if t.device != plan.position.device:
        raise ValueError(f"{what}: rows on {t.device}, plan on {plan.position.device}")
    if t.is_cuda and t.dtype not in _DTYPES:
        raise TypeError(f"{what}: dtype {t.dtype} (fp32, bf16 or fp16)")
    if t.shape[1] > _INT32 - 1024:
        raise ValueError(f"{what}: rows of {t.shape[1]} elements")


def dispatch(x: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """Expert rows ``[plan.rows, D]``: row ``plan.position[t, j]`` is ``x[t]``, rows that no sample fills are 0. The
    gradient of ``x`` is summed over a sample's rows in fp32."""
    _check_rows(x, plan, plan.tokens, "dispatch")
    if not x.is_cuda:
        rows = x[(plan.source.long().clamp(min=0) // plan.k)] if plan.tokens else x.new_zeros(plan.rows, x.shape[1])
        return torch.where((plan.source >= 0)[:, None], rows, 0.0)
    return _Dispatch.apply(x, plan) if x.requires_grad and torch.is_grad_enabled() else _scatter(plan, x)[0]


def combine(rows: torch.Tensor, plan: ExpertPlan, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Back in sample order: ``y[t] = sum_j weights[t, j] * rows[plan.position[t, j]]`` (``weights`` None: 1), summed in
    fp32 and rounded to the type of ``rows`` once; a sample without rows gives 0. Gradients reach ``rows`` and
    ``weights`` (a choice without a row has gradient 0)."""
    _check_rows(rows, plan, plan.rows, "combine")
    if weights is not None:
        if tuple(weights.shape) != (plan.tokens, plan.k) or not weights.is_floating_point():
            raise ValueError(f"combine: weights must be floating [{plan.tokens}, {plan.k}], got {weights.dtype} "
                             f"{tuple(weights.shape)}")
        if weights.device != rows.device:
            raise ValueError(f"combine: weights on {weights.device}, rows on {rows.device}")
    if not rows.is_cuda:
        return _combine_cpu(rows, plan, weights)
    rows = rows.contiguous()
    if weights is not None:
        weights = weights.float().contiguous()
    if torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad)):
        return _Combine.apply(rows, weights, plan)
    return _gather(plan, rows, weights)


def _combine_cpu(rows, plan, weights):
    wide = torch.float64 if rows.dtype == torch.float64 else torch.float32
    if plan.rows == 0:
        return rows.new_zeros(plan.tokens, rows.shape[1])
    there = (plan.position >= 0)[:, :, None]
    part = torch.where(there, rows.to(wide)[plan.position.long().clamp(min=0)], 0.0)
    if weights is not None:
        part = part * torch.where(there, weights.to(wide)[:, :, None], 0.0)
    return part.sum(1).to(rows.dtype)
