"""What autograd may ask of the experts' operators besides a plain backward pass."""
import pytest
import torch

from test_gpu_experts import Layer, ids_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def X():
    from jax_gptq_amd import experts
    return experts


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


E, TOP_K, K, N, T = 4, 2, 128, 96, 12


def operators(X):
    """name -> (function of a differentiable tensor and a plan, that tensor, a stack or None)"""
    stack = Layer(X, 1, E, K, N, 4, 64).stack
    w = torch.rand(T, TOP_K).cuda()
    y = torch.randn(T * TOP_K, N).cuda()
    return {
        "gather": (lambda x, p: X.gather_tokens(x, p), torch.randn(T, K).cuda(), None),
        "combine": (lambda y, p: X.combine_tokens(y, p, w), y, None),
        "combine_plain": (lambda y, p: X.combine_tokens(y, p), y, None),
        "combine_weights": (lambda w, p: X.combine_tokens(y, p, w), w, None),
        "matmul": (lambda x, p: X.quantized_expert_matmul(x, stack, p), torch.randn(T, K).cuda(), stack),
        "matmul_rows": (lambda x, p: X.quantized_expert_matmul(x, stack, p, sorted_rows=True),
                        torch.randn(T * TOP_K, K).cuda(), stack),
        "matmul_back": (lambda x, p: X.quantized_expert_matmul(x, stack, p, transpose_b=True), torch.randn(T, N).cuda(),
                        stack),
    }


NAMES = ["gather", "combine", "combine_plain", "combine_weights", "matmul", "matmul_rows", "matmul_back"]


# ------------------------------------------------------------------------------------ what a backward pass reads
@pytest.mark.parametrize("buffer", ["position", "offsets"])
@pytest.mark.parametrize("name", NAMES)
def test_plan_written_to_before_the_backward_pass(X, name, buffer):
    f, x, _ = operators(X)[name]
    plan = X.sort_tokens(ids_of(0, T, TOP_K, E).cuda(), E)
    out = f(x.requires_grad_(), plan)
    getattr(plan, buffer).zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), x)


@pytest.mark.parametrize("buffer", ["int_weight", "zero", "scale"])
@pytest.mark.parametrize("name", ["matmul", "matmul_rows", "matmul_back"])
def test_weights_written_to_before_the_backward_pass(X, name, buffer):
    f, x, stack = operators(X)[name]
    plan = X.sort_tokens(ids_of(0, T, TOP_K, E).cuda(), E)
    out = f(x.requires_grad_(), plan)
    getattr(stack, buffer).mul_(2)          # one buffer used for several layers
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), x)


@pytest.mark.parametrize("name", ["matmul", "matmul_rows", "matmul_back"])
def test_weights_replaced_before_the_backward_pass(X, name):
    """The gradient is that of the weights and the plan that the product read, a graph of the gradient included."""
    f, x, stack = operators(X)[name]
    ids = ids_of(0, T, TOP_K, E).cuda()
    x.requires_grad_()
    want = torch.autograd.grad(f(x, X.sort_tokens(ids, E)).sum(), x)[0]
    plan = X.sort_tokens(ids, E)
    out = f(x, plan)
    other, routed = Layer(X, 9, E, K, N, 4, 64).stack, X.sort_tokens(ids.flip(0), E)
    stack.int_weight, stack.zero, stack.scale = other.int_weight, other.zero, other.scale
    plan.order, plan.position, plan.offsets = routed.order, routed.position, routed.offsets
    for graph in (False, True):
        assert torch.equal(torch.autograd.grad(out.sum(), x, create_graph=graph, retain_graph=True)[0], want)
