"""Argument checks of the mixture-of-experts operators that need no GPU: the C entry points refuse before they touch the
device, and the containers refuse tensors that do not fit together."""
import ctypes

import pytest
import torch

from jax_gptq_amd import _native as N
from jax_gptq_amd.experts import (QuantizedExperts, TokenPlan, gptq_experts, quantized_expert_matmul, sort_tokens,
                                  stack_experts)
from jax_gptq_amd.gptq import QuantizedMatrix

NULL = ctypes.c_void_p(0)
SOME = ctypes.c_void_p(1 << 20)          # never dereferenced: every call below is refused or empty


@pytest.fixture(scope="module")
def lib():
    return N.load()


def test_sort_refusals(lib):
    def call(ids=SOME, id_bytes=8, pairs=8, experts=4, order=SOME, position=SOME, offsets=SOME, ws=NULL, nb=0):
        return lib.gptq_hip_expert_sort(NULL, ids, id_bytes, pairs, experts, order, position, offsets, ws, nb)
    assert call(pairs=-1) == N.EINVAL
    assert call(pairs=(1 << 30) + 1) == N.EINVAL
    assert call(experts=0) == N.EINVAL and call(experts=1025) == N.EINVAL
    assert call(id_bytes=2) == N.EDTYPE
    assert call(ids=NULL) == N.EINVAL and call(order=NULL) == N.EINVAL
    assert call(position=NULL) == N.EINVAL and call(offsets=NULL) == N.EINVAL
    big = 1 << 20
    need = lib.gptq_hip_expert_sort_workspace_bytes(big, 64)
    assert need > 0 and lib.gptq_hip_expert_sort_workspace_bytes(100, 64) == 0
    assert call(pairs=big, experts=64, ws=SOME, nb=need - 1) == N.EWORKSPACE
    assert call(pairs=big, experts=64, ws=NULL, nb=need) == N.EWORKSPACE


def test_sort_workspace_stays_small(lib):
    # at most 256 workgroups, whose counts are all that the workspace holds
    for pairs in (1 << 14, 1 << 20, (1 << 30) - 5, 1 << 30):
        assert lib.gptq_hip_expert_sort_workspace_bytes(pairs, 1024) <= 256 * 1025 * 4


def test_row_operator_refusals(lib):
    def gather(dt=N.F16, tokens=4, k=2, width=8, experts=4, x=SOME, pos=SOME, off=SOME, out=SOME):
        return lib.gptq_hip_expert_gather(NULL, x, dt, tokens, k, width, pos, off, experts, out)
    for bad in (dict(tokens=-1), dict(k=0), dict(width=-1), dict(experts=0), dict(experts=1025), dict(tokens=1 << 24),
                dict(tokens=1 << 23, k=1 << 10), dict(width=1 << 26), dict(x=NULL), dict(pos=NULL), dict(off=NULL),
                dict(out=NULL)):
        assert gather(**bad) == N.EINVAL, bad
    assert gather(dt=N.F64) == N.EDTYPE
    assert gather(tokens=0, x=NULL) == N.OK and gather(width=0, x=NULL) == N.OK

    def combine(dt=N.F16, tokens=4, k=2, width=8, w=NULL, wdt=N.F32, out_dt=N.F16, y=SOME):
        return lib.gptq_hip_expert_combine(NULL, y, dt, tokens, k, width, SOME, SOME, 4, w, wdt, SOME, out_dt)
    assert combine(dt=7) == N.EDTYPE and combine(w=SOME, wdt=N.F64) == N.EDTYPE
    assert combine(out_dt=N.BF16) == N.EDTYPE and combine(out_dt=N.F32) == N.EDTYPE
    assert combine(y=NULL) == N.EINVAL and combine(k=0) == N.EINVAL
    assert combine(tokens=0) == N.OK

    def grad(dt=N.F16, tokens=4, y=SOME, g=SOME, dy=SOME, dw=SOME, wdt=N.F32):
        return lib.gptq_hip_expert_combine_grad(NULL, y, g, dt, tokens, 2, 8, SOME, SOME, 4, SOME, wdt, dy, dw)
    assert grad(dt=N.F64) == N.EDTYPE and grad(wdt=9) == N.EDTYPE
    assert grad(g=NULL) == N.EINVAL and grad(y=NULL) == N.EINVAL
    assert grad(tokens=0) == N.OK and grad(dy=NULL, dw=NULL, g=NULL, y=NULL) == N.OK


def test_product_refusals(lib):
    def call(x=SOME, dt=N.F16, x_rows=4, order=SOME, k=2, rows=8, off=SOME, experts=4, packed=SOME, R=32, C=64,
             zero=SOME, scale=SOME, zdt=N.F32, group=32, bits=4, tr=0, out=SOME, odt=N.F16):
        return lib.gptq_hip_expert_qmatmul(NULL, x, dt, x_rows, order, k, rows, off, experts, packed, R, C, zero, scale,
                                           zdt, group, bits, tr, out, odt, NULL, 0)
    for bad in (dict(bits=3), dict(experts=0), dict(experts=1025), dict(k=0), dict(x_rows=-1), dict(rows=9),
                dict(order=NULL), dict(R=0), dict(C=0), dict(group=-32), dict(group=24), dict(R=33, group=3),
                dict(x=NULL), dict(off=NULL), dict(packed=NULL), dict(zero=NULL), dict(scale=NULL), dict(out=NULL),
                dict(x_rows=1 << 23, rows=1 << 24), dict(R=1 << 20, group=0), dict(C=(1 << 20) + 1)):
        assert call(**bad) == N.EINVAL, bad
    for bad in (dict(dt=N.F64), dict(zdt=N.F64), dict(odt=N.BF16), dict(dt=N.F32, odt=N.F16)):
        assert call(**bad) == N.EDTYPE, bad
    assert call(x_rows=0, rows=0, x=NULL) == N.OK


def _stack(E=3, R=16, C=8, group=0, bits=4):
    K = R * (8 // bits)
    t = (E, K // group, C) if group else (E, C)
    return torch.zeros(E, R, C, dtype=torch.uint8), torch.zeros(t), torch.ones(t)


def test_container():
    iw, z, s = _stack(group=8)
    q = QuantizedExperts(iw, z, s, group_size=8)
    assert q.shape == (3, 32, 8) and len(q) == 3 and q.dtype == torch.float32
    one = q[-1]
    assert isinstance(one, QuantizedMatrix) and one.shape == (32, 8) and one.group_size == 8
    assert len(list(q)) == 3
    with pytest.raises(IndexError):
        q[3]
    children, aux = q.tree_flatten()
    assert QuantizedExperts.tree_unflatten(aux, children).group_size == 8
    assert QuantizedExperts(*_stack(bits=8), bits=8).shape == (3, 16, 8)


def test_container_refusals():
    iw, z, s = _stack()
    for args, kw in (((iw, z, s), dict(bits=5)), ((iw[0], z, s), {}), ((iw.int(), z, s), {}), ((iw, z[:, :4], s), {}),
                     ((iw, z, s[:2]), {}), ((iw, z, s), dict(group_size=8)), ((iw, z, s), dict(group_size=5)),
                     ((iw, z, s), dict(group_size=-8)), ((iw[:0], z[:0], s[:0]), {}),
                     ((torch.zeros(1025, 1, 1, dtype=torch.uint8), torch.zeros(1025, 1), torch.zeros(1025, 1)), {})):
        with pytest.raises(ValueError):
            QuantizedExperts(*args, **kw)
    with pytest.raises(ValueError):
        stack_experts([])
    a = QuantizedMatrix(torch.zeros(4, 8, dtype=torch.uint8), torch.zeros(8), torch.ones(8))
    b = QuantizedMatrix(torch.zeros(4, 6, dtype=torch.uint8), torch.zeros(6), torch.ones(6))
    with pytest.raises(ValueError):
        stack_experts([a, b])
    with pytest.raises(ValueError):
        stack_experts([QuantizedMatrix(torch.zeros(4, 8, dtype=torch.uint8), torch.zeros(4), torch.ones(4), 1)])


def test_product_wants_a_stack_that_fits_the_plan():
    plan = TokenPlan(torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32),
                     torch.zeros(5, dtype=torch.int32), (2,), 2, 4)
    assert plan.n_tokens == 2 and plan.n_rows == 4
    with pytest.raises(TypeError):
        quantized_expert_matmul(torch.zeros(2, 32), torch.zeros(4, 32, 8), plan)
    with pytest.raises(ValueError):
        quantized_expert_matmul(torch.zeros(2, 32), QuantizedExperts(*_stack()), plan)


def test_solve_refuses_one_hessian_for_all_experts():
    # H and shared belong to matrices applied to the same activations; every expert has its own
    W, xs, ids = torch.zeros(2, 128, 16), [torch.zeros(4, 128)], [torch.zeros(4, 1, dtype=torch.int64)]
    with pytest.raises(ValueError, match="H"):
        gptq_experts(W, xs, ids, H=torch.eye(128))
    with pytest.raises(ValueError, match="shared"):
        gptq_experts(W, xs, ids, shared={})


def test_workspace_query_of_what_the_product_refuses(lib):
    def need(x_rows=600, rows=1200, R=512, C=1024, bits=4, group=64, experts=4, dt=N.F16, zdt=N.F32, tr=0):
        return lib.gptq_hip_expert_qmatmul_workspace_bytes(x_rows, rows, R, C, bits, group, experts, dt, zdt, tr)
    assert need() > 0 and need(tr=1) > 0
    for bad in (dict(group=1 << 32), dict(group=-64), dict(group=1 << 40, R=1 << 50), dict(group=96), dict(bits=3),
                dict(rows=1 << 24), dict(x_rows=1 << 40), dict(R=1 << 40), dict(C=1 << 40), dict(experts=0),
                dict(experts=1 << 20), dict(rows=0), dict(x_rows=-1), dict(dt=9), dict(zdt=N.F64)):
        for tr in (0, 1):
            assert need(**bad, tr=tr) == 0, (bad, tr)
