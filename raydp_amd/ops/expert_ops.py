"""Routed experts (``csrc/hip/experts.hip``): a router's top-k softmax, samples sorted by expert, and back with weights.

    weights, experts = route(logits, k)                 # [T, k] fp32, [T, k] int32 (-1: none)
    plan = expert_plan(experts, num_experts, capacity)  # a stable counting sort; capacity None: no sample is dropped
    rows = dispatch(x, plan)                            # [R, D]: expert e owns rows offsets[e] .. offsets[e] + load[e]
    y = combine(f(rows), plan, weights)                 # [T, D]: sum over a sample's experts

Nothing is read back to the host, so a step with them can be captured into a HIP graph; with a ``capacity`` every expert's
rows are a slice of fixed size (``rows.view(num_experts, capacity, D)``) that a ``FusedLinearTower`` takes as it is.

``route``, ``dispatch`` and ``combine`` are differentiable (once, in reverse; a forward-mode tangent raises on the GPU).
Capturing a backward pass through them is refused when it would reach what an eager call on the default stream made:
intermediate results, or leaves that something the call returned still holds.

On the GPU all run on the HIP kernels (through ``csrc/torch/raydp_torch.cc``) and fail loudly if these are missing; on the
CPU they are the equivalent PyTorch expressions (any floating type, for tests and CPU-only hosts).
"""
from typing import Optional, Tuple

import torch

MAX_EXPERTS, MAX_TOPK = 1024, 32
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_INT32 = 0x7FFFFFFF


_module = None


def _ext():
    global _module
    if _module is None:
        from raydp_amd.native import loader
        _module = loader.load_torch()
    return _module


# ------------------------------------------------------------------------------------------------ router
def route(logits: torch.Tensor, k: int, renormalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """The ``k`` experts of every sample and their weights: ``[T, k]`` fp32 weights (differentiable) and int32 experts, in
    the order of the logits (ties: the lowest expert first).

    ``logits``       ``[T, E]``, fp32, bf16 or fp16; at most 1024 experts, ``k`` at most 32
    ``renormalize``  True: weights of a sample are the softmax over its chosen experts (they sum to 1); False: the chosen
                     entries of the softmax over all experts

    An expert whose logit is ``-inf`` is never chosen; a sample with fewer than ``k`` others gets expert -1 with weight 0
    in the places that are left (all of them, for a padding row of ``-inf``). A NaN is not chosen and makes the weights of
    its row, and what reaches its logits from them, NaN."""
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
    return _ext().route(logits, k, bool(renormalize))


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
    w = w * torch.where(bad.any(1, keepdim=True), torch.nan, 1.0)      # (a product: the gradient shows the NaN too)
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
    return ExpertPlan(*_ext().expert_plan(experts, E, C), E, C or None)


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
    return _ext().dispatch(x, plan.position, plan.source)


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
    return _ext().combine(rows, weights, plan.position, plan.source)


def _combine_cpu(rows, plan, weights):
    wide = torch.float64 if rows.dtype == torch.float64 else torch.float32
    if plan.rows == 0:
        return rows.new_zeros(plan.tokens, rows.shape[1])
    there = (plan.position >= 0)[:, :, None]
    part = torch.where(there, rows.to(wide)[plan.position.long().clamp(min=0)], 0.0)
    if weights is not None:
        part = part * torch.where(there, weights.to(wide)[:, :, None], 0.0)
    return part.sum(1).to(rows.dtype)
