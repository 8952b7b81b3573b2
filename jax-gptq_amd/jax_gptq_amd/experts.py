"""Mixture of experts on packed weights: tokens sorted by expert and back, and the experts' products.

The reference's packed product takes one matrix (``op.py:19-69``); a layer of experts has E of them and a router that
picks ``top_k`` for every token.  The pieces, in the order a layer uses them::

    plan = sort_tokens(expert_ids, n_experts)                 # [T, top_k] ids -> rows by expert
    up   = quantized_expert_matmul(x, W_up, plan)             # [T * top_k, N], rows by expert
    gate = quantized_expert_matmul(x, W_gate, plan)
    down = quantized_expert_matmul(silu(gate) * up, W_down, plan, sorted_rows=True)
    y    = combine_tokens(down, plan, weights)                # [T, K], weighted and added up

``W_*`` are :class:`QuantizedExperts`, from :func:`stack_experts` (packed matrices, e.g. of separate ``gptq`` calls)
or :func:`gptq_experts` (all experts of a layer against the tokens that reach them).  An id outside
``0 .. n_experts - 1`` marks a (token, choice) pair that goes nowhere, e.g. padding: its rows stand behind the last
expert's, are zero, and add nothing.  Differentiable with respect to activations and router weights, in reverse mode
(forward mode raises); the packed matrices are frozen, as in ``quantized_matmul``.  Nothing here waits for the GPU, so everything but
``gptq_experts`` can be captured into a HIP graph.  As with any torch operator, capture a backward pass with leaves
that no eager graph still refers to.
"""
from __future__ import annotations

import torch

from . import _native as N
from .gptq import _DT, QuantizedMatrix, _dev, _float_dev, _ptr, _stream, gptq, pack_matrix

__all__ = ["QuantizedExperts", "TokenPlan", "stack_experts", "gptq_experts", "sort_tokens", "gather_tokens",
           "combine_tokens", "quantized_expert_matmul"]

MAX_EXPERTS = 1024


def _on_device(t, like, what):
    """``t`` contiguous; operands of one call live on one GPU."""
    if t.get_device() != like.get_device():
        raise ValueError(f"{what} is on {t.device}, expected {like.device}")
    return t if t.is_contiguous() else t.contiguous()


def _float_tensor(x):
    """Float tensor on a GPU, contiguous, in a type the kernels take.  A tensor that is on a GPU stays there."""
    if isinstance(x, torch.Tensor) and x.is_cuda:
        if x.dtype not in _DT:
            x = x.to(torch.float32)
        return x if x.is_contiguous() else x.contiguous()
    return _float_dev(x)


class QuantizedExperts:
    """The packed matrices of ``E`` experts: ``int_weight`` ``[E, R, N]`` uint8 with ``R`` packed rows of ``W[e]``
    ``[K, N]`` (``bits`` 4: two rows a byte, ``K = 2 R``; 8: one), ``zero`` / ``scale`` ``[E, N]`` or, with
    ``group_size``, ``[E, K / group_size, N]``.  ``stack[e]`` is expert ``e`` as a :class:`QuantizedMatrix` (a view)."""

    def __init__(self, int_weight, zero, scale, bits=4, group_size=0):
        if bits not in (4, 8):
            raise ValueError("bits must be 4 or 8")
        group_size = int(group_size or 0)
        if int_weight.dim() != 3 or int_weight.dtype != torch.uint8:
            raise ValueError("int_weight must be a uint8 tensor [n_experts, packed rows, N]")
        E, R, C = int_weight.shape
        K = R * (8 // bits)
        if not 1 <= E <= MAX_EXPERTS:
            raise ValueError(f"between 1 and {MAX_EXPERTS} experts")
        if group_size < 0 or (group_size and (K % group_size or (bits == 4 and group_size % 2))):
            raise ValueError("group_size must divide K (and be even for 4-bit codes)")
        tables = (E, K // group_size, C) if group_size else (E, C)
        if tuple(zero.shape) != tables or tuple(scale.shape) != tables:
            raise ValueError(f"zero and scale must be {list(tables)}")
        if zero.device != int_weight.device or scale.device != int_weight.device:
            raise ValueError("int_weight, zero and scale must be on one device")
        self.int_weight = int_weight
        self.zero = zero
        self.scale = scale
        self.bits = bits
        self.group_size = group_size

    @property
    def shape(self):
        E, R, C = self.int_weight.shape
        return (E, R * (8 // self.bits), C)

    @property
    def dtype(self):
        return self.zero.dtype

    def __len__(self):
        return self.int_weight.shape[0]

    def __getitem__(self, e):
        e = range(len(self))[e]         # IndexError past the end, so that iteration stops
        return QuantizedMatrix(self.int_weight[e], self.zero[e], self.scale[e], contraction_axis=0, bits=self.bits,
                               group_size=self.group_size)

    def tree_flatten(self):
        return (self.int_weight, self.zero, self.scale), (self.bits, self.group_size)

    @classmethod
    def tree_unflatten(cls, aux, children):
        return cls(*children, bits=aux[0], group_size=aux[1])

    def to(self, device):
        return QuantizedExperts(self.int_weight.to(device), self.zero.to(device), self.scale.to(device), self.bits,
                                self.group_size)


def stack_experts(matrices):
    """One :class:`QuantizedExperts` of packed matrices ``[K, N]`` of one shape, width and group size."""
    matrices = list(matrices)
    if not matrices:
        raise ValueError("at least one expert")
    first = matrices[0]
    for m in matrices:
        if m.contraction_axis != 0 or m.int_weight.dim() != 2:
            raise ValueError("experts are 2-D matrices packed along axis 0")
        if (tuple(m.int_weight.shape), m.bits, m.group_size, m.zero.dtype, m.scale.dtype, tuple(m.zero.shape)) != \
                (tuple(first.int_weight.shape), first.bits, first.group_size, first.zero.dtype, first.scale.dtype,
                 tuple(first.zero.shape)):
            raise ValueError("all experts must have the same shape, code width, groups and parameter type")
    return QuantizedExperts(torch.stack([_dev(m.int_weight, torch.uint8) for m in matrices]),
                            torch.stack([_dev(m.zero) for m in matrices]),
                            torch.stack([_dev(m.scale) for m in matrices]),
                            bits=first.bits, group_size=first.group_size)


class TokenPlan:
    """What :func:`sort_tokens` found.  ``T`` tokens of ``top_k`` choices; pair ``i = token * top_k + choice``.

    ``order`` int32 ``[T * top_k]``: the pairs by expert, ties in order of the pair; ``position``: its inverse;
    ``offsets`` int32 ``[n_experts + 1]``: expert ``e`` owns rows ``offsets[e]`` to ``offsets[e + 1]``, rows from
    ``offsets[n_experts]`` on go nowhere.  ``token_shape``: the shape of the ids without their last axis."""

    def __init__(self, order, position, offsets, token_shape, top_k, n_experts):
        self.order = order
        self.position = position
        self.offsets = offsets
        self.token_shape = tuple(token_shape)
        self.top_k = top_k
        self.n_experts = n_experts
        self.n_rows = order.numel()
        self.n_tokens = self.n_rows // top_k


def sort_tokens(expert_ids, n_experts):
    """The :class:`TokenPlan` of integer ``expert_ids`` ``[..., top_k]`` (``[T]``: one choice per token)."""
    ids = expert_ids if isinstance(expert_ids, torch.Tensor) and expert_ids.is_cuda else _dev(expert_ids)
    if ids.dtype not in (torch.int32, torch.int64):
        if ids.is_floating_point() or ids.is_complex() or ids.dtype == torch.bool:
            raise TypeError("expert_ids must be integers")
        ids = ids.to(torch.int64)
    n_experts = int(n_experts)
    if not 1 <= n_experts <= MAX_EXPERTS:
        raise ValueError(f"n_experts must be between 1 and {MAX_EXPERTS}")
    if ids.dim() == 0:
        raise ValueError("expert_ids must have at least one dimension")
    if ids.dim() == 1:
        ids = ids.reshape(-1, 1)
    top_k = ids.shape[-1]
    if top_k == 0:
        raise ValueError("at least one choice per token")
    ids = ids.contiguous()
    order, position, offsets = N.load_torch().sort(ids, n_experts)
    return TokenPlan(order, position, offsets, ids.shape[:-1], top_k, n_experts)


def _rows_of(x, rows, plan, what):
    """``x`` as ``[rows, width]`` on the plan's GPU."""
    dims = x.dim()
    if dims < 2:
        raise ValueError(f"{what} must have at least 2 dimensions")
    x = _on_device(x, plan.order, what)
    width = x.size(-1)
    if width == 0 or x.numel() != rows * width:
        raise ValueError(f"{what} has {x.numel() // max(width, 1)} rows of {width}, expected {rows}")
    return x if dims == 2 else x.reshape(rows, width)


def gather_tokens(x, plan):
    """The tokens' rows in sorted order: ``x`` ``[T, K]`` (or ``[..., K]``) -> ``[T * top_k, K]``; rows of pairs that
    go nowhere are zero.  The gradient adds up a token's copies in fp32 and rounds once."""
    x = _rows_of(_float_tensor(x), plan.n_tokens, plan, "x")
    return N.load_torch().gather(x, plan.position, plan.offsets, plan.top_k)


def combine_tokens(y, plan, weights=None):
    """The sorted rows back at their tokens: ``y`` ``[T * top_k, N]`` -> ``[T, N]`` (leading axes as the ids had),
    ``out[t] = sum_j weights[t, j] * y[row of (t, j)]`` in fp32 in order of ``j``, rounded once to ``y``'s type.
    ``weights``: ``[..., top_k]`` of any float type, one each without them.  Differentiable in both."""
    y = _rows_of(_float_tensor(y), plan.n_rows, plan, "y")
    if weights is not None:
        weights = _on_device(_float_tensor(weights), plan.order, "weights")
        if weights.numel() != plan.n_rows or (weights.shape[-1] != plan.top_k if weights.dim() > 1 else plan.top_k > 1):
            raise ValueError(f"weights must be [..., {plan.top_k}] with one row per token")
    out = N.load_torch().combine(y, weights, plan.position, plan.offsets, plan.top_k)
    return out if len(plan.token_shape) == 1 else out.reshape(plan.token_shape + (y.size(1),))


def quantized_expert_matmul(x, experts, plan, sorted_rows=False, transpose_b=False):
    """Every expert's rows times its packed matrix: ``[T * top_k, N]`` in sorted order, ``x_row @ W[e]``
    (``transpose_b``: ``x_row @ W[e].T``), zero for rows that go nowhere.

    ``x`` holds the tokens ``[T, K]`` (``[..., K]``), whose rows the kernels fetch through the plan, or, with
    ``sorted_rows``, the rows in sorted order ``[T * top_k, K]``.  The codes enter the matrix cores exactly (fp32
    activations as three bfloat16 parts), sums and scales are fp32, and the result is rounded once to ``x``'s type
    (``quantized_matmul`` rounds to fp16 on the way, as the reference does).  ``transpose_b``, and with it the gradient,
    applies the scale to ``x``: 16-bit rows times scale enter as two bfloat16 parts, which leave out up to 2^-18 of each
    term.  A row of ``x`` with an infinity or a NaN may become NaN throughout, other rows do not see it; so may one whose
    sums of ``x`` times codes over a group, which come before the scale, or, transposed, of ``x`` times scale times codes
    leave fp32's range.  Equal calls give equal bits; which kernel runs, and with it the order of a row's sums, follows
    from the number of pairs for each expert on average, those that go nowhere included, and from the rows that every
    expert has.  Differentiable with respect to ``x``."""
    if not isinstance(experts, QuantizedExperts):
        raise TypeError("experts must be QuantizedExperts")
    if len(experts) != plan.n_experts:
        raise ValueError(f"{len(experts)} matrices for a plan of {plan.n_experts} experts")
    x = _rows_of(_float_tensor(x), plan.n_rows if sorted_rows else plan.n_tokens, plan, "x")
    inner = experts.shape[2 if transpose_b else 1]
    assert x.shape[1] == inner, f"Inner dim mismatch: {x.shape[1]} != {inner}"
    packed = _on_device(experts.int_weight, x, "int_weight")
    zero = _float_tensor(_on_device(experts.zero, x, "zero"))
    scale = _on_device(experts.scale, x, "scale")
    if scale.dtype != zero.dtype:           # the kernels read both in one type: fp32 holds either
        zero, scale = zero.float(), scale.float()
    return N.load_torch().matmul(x, packed, zero, scale, plan.order, plan.position, plan.offsets, plan.top_k, experts.bits,
                                 experts.group_size, bool(sorted_rows), bool(transpose_b))


def _rows_at(x, rows):
    """Copies of some rows of ``x``."""
    out = x.new_empty((rows.numel(), x.shape[1]))
    rows = rows.long()
    with torch.cuda.device(x.device):
        N.check(N.load().gptq_hip_gather_rows(_stream(), _ptr(x), _ptr(out), x.element_size(), out.shape[0], x.shape[1],
                                              _ptr(rows)), "gather_rows")
    return out


def gptq_experts(W, xs, expert_ids, bits=4, **options):
    """The solve for all experts of a layer: ``W`` ``[E, K, N]``, calibration batches ``xs`` ``[..., K]`` and for each
    the router's ids ``[..., top_k]`` -> :class:`QuantizedExperts`.

    Each expert is solved by :func:`gptq` against the rows that reach it, copied when its turn comes: one expert's rows are
    held beside the batches, not ``top_k`` copies of them.
    An expert that no row reaches has no Hessian; it is rounded to its own grid, which is the solve with the identity
    as its Hessian.  ``options`` are those of :func:`gptq` (``block_size``, ``damping``, ``group_size``, ...) but ``H``
    and ``shared``, which are one Hessian for several matrices."""
    for name in ("H", "shared"):
        if options.get(name) is not None:
            raise ValueError(f"{name} is one Hessian for several matrices; every expert has its own")
    if not isinstance(W, torch.Tensor):
        W = _dev(W)
    if W.dim() != 3:
        raise ValueError("W must be [n_experts, K, N]")
    E, K, _ = W.shape
    xs, expert_ids = list(xs), list(expert_ids)
    if len(xs) != len(expert_ids):
        raise ValueError("one tensor of expert ids per calibration batch")
    routed = []
    for x, ids in zip(xs, expert_ids):
        plan = sort_tokens(ids, E)
        x = _rows_of(_float_tensor(x), plan.n_tokens, plan, "x")
        if x.shape[1] != K:
            raise ValueError(f"calibration feature dim {x.shape[1]} != K={K}")
        routed.append((x, plan, plan.offsets.tolist()))
    out = []
    for e in range(E):
        batches = [_rows_at(x, plan.order[at[e]:at[e + 1]] // plan.top_k) for x, plan, at in routed if at[e + 1] > at[e]]
        if not batches:
            batches = [torch.eye(K, dtype=torch.float32, device=_dev(W[e]).device)]
        Q, params = gptq(W[e], batches, bits=bits, **options)
        out.append(pack_matrix(Q, params))
    return stack_experts(out)
