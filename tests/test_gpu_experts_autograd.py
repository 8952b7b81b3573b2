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


# ------------------------------------------------------------------------------------ a graph of the gradient
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", ["gather", "combine", "combine_plain", "matmul", "matmul_rows", "matmul_back"])
def test_gradient_is_the_same_with_a_graph_of_it(X, name, dt):
    """create_graph says what may be asked later, not what the gradient is."""
    f, x, _ = operators(X)[name]
    plan = X.sort_tokens(ids_of(0, T, TOP_K, E, 0.1).cuda(), E)
    x = x.to(dt).requires_grad_()
    out = f(x, plan)
    g = torch.randn_like(out)
    plain = torch.autograd.grad(out, x, g, retain_graph=True)[0]
    graph = torch.autograd.grad(out, x, g, create_graph=True)[0]
    assert graph.dtype == dt and torch.equal(plain, graph)


def test_weights_gradient_is_the_same_with_a_graph_of_it(X):
    plan = X.sort_tokens(ids_of(0, T, TOP_K, E, 0.1).cuda(), E)
    for dt, wt in ((torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16)):
        y, w = torch.randn(T * TOP_K, N).to(dt).cuda().requires_grad_(), torch.rand(T, TOP_K).to(wt).cuda().requires_grad_()
        out = X.combine_tokens(y, plan, w)
        plain = torch.autograd.grad(out, (y, w), torch.ones_like(out), retain_graph=True)
        graph = torch.autograd.grad(out, (y, w), torch.ones_like(out), create_graph=True)
        for a, b in zip(plain, graph):
            assert torch.equal(a, b)


@pytest.mark.parametrize("name", NAMES)
def test_graph_of_the_gradient_of_an_empty_batch(X, name):
    f, x, _ = operators(X)[name]
    if name == "combine" or name == "combine_weights":
        y, w = torch.zeros(0, N).cuda(), torch.zeros(0, TOP_K).cuda()
        f, x = (lambda a, p: X.combine_tokens(a, p, w), y) if name == "combine" else (lambda a, p: X.combine_tokens(y, p, a), w)
    x = x[:0].clone().requires_grad_()
    out = f(x, X.sort_tokens(torch.zeros(0, TOP_K, dtype=torch.int64).cuda(), E))
    (dx,) = torch.autograd.grad(out.square().sum(), x, create_graph=True)
    assert dx.shape == x.shape
    if dx.requires_grad:
        (ddx,) = torch.autograd.grad(dx.square().sum(), x)
        assert ddx.shape == x.shape


def _dense(layer):
    w = [(c - z) * s for c, z, s in (layer.parts(e) for e in range(layer.E))]
    return torch.stack(w)


@pytest.mark.parametrize("name", ["gather", "combine", "matmul", "matmul_back"])
@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
def test_second_and_third_derivatives(X, name, dt):
    """grad(sum(grad(sum(f^2 h)) ^ 2)) and once more, against the same in 64 bits with index operations.  A derivative of
    order n is a chain of n + 1 operators, each rounded once to dt (a half step of the largest value, and sums of two of
    those where copies meet): 4 (n + 1) half steps cover it.  (Half a step is eps / 2 of the smallest normal number at
    least: of fp16 results of 1e-6, 2^-25 = 3e-8.)"""
    layer = Layer(X, 1, E, K, N, 4, 64)
    w64 = _dense(layer)
    ids = ids_of(0, T, TOP_K, E, 0.1)
    plan = X.sort_tokens(ids.cuda(), E)
    order, position, live = plan.order.cpu().long(), plan.position.cpu().long(), int(plan.offsets[-1])
    expert = torch.bucketize(torch.arange(T * TOP_K), plan.offsets.cpu()[1:].long(), right=True).clamp_max(E - 1)
    alive = (torch.arange(T * TOP_K) < live).double()[:, None]
    weights = torch.rand(T, TOP_K)

    def reference(x, w):
        if name == "gather":
            return x[order // TOP_K] * alive
        if name == "combine":
            return ((x * alive)[position].reshape(T, TOP_K, -1) * w[:, :, None]).sum(1)
        m = w64 if name == "matmul" else w64.transpose(1, 2)
        return (x[order // TOP_K][:, None] @ m[expert])[:, 0] * alive

    def ours(x, w):
        if name == "gather":
            return X.gather_tokens(x, plan)
        if name == "combine":
            return X.combine_tokens(x, plan, w)
        return X.quantized_expert_matmul(x, layer.stack, plan, transpose_b=name == "matmul_back")

    x = torch.randn(T * TOP_K if name == "combine" else T, N if name == "matmul_back" else K).to(dt)
    results = []
    for f, a, w in ((ours, x.cuda(), weights.cuda()), (reference, x.double(), weights.double())):
        a.requires_grad_()
        w.requires_grad_()
        wrt = (a, w) if name == "combine" else (a,)
        out = f(a, w)
        found, value = [], 0.5 * (out.double() if dt == torch.float32 else out.float()).square().mean()
        for _ in range(3):
            grads = torch.autograd.grad(value, wrt, create_graph=True, allow_unused=True)
            found += [g.detach().cpu().double() for g in grads if g is not None]
            value = sum(g.float().square().sum() if f is ours else g.square().sum() for g in grads if g is not None)
            if not value.requires_grad:
                break
        results.append(found)
    half = torch.finfo(dt).eps / 2
    for n, (got, want) in enumerate(zip(*results)):
        order_of = n // (2 if name == "combine" else 1) + 1
        largest = want.abs().max()
        step = half * largest.clamp_min(torch.finfo(dt).smallest_normal)
        assert (got - want).abs().max() <= 4 * (order_of + 1) * step + 2.0 ** -14 * largest, n


# ------------------------------------------------------------------------------------ forward mode
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(X, name):
    """A tangent is not lost without a word."""
    import torch.autograd.forward_ad as forward
    f, x, _ = operators(X)[name]
    plan = X.sort_tokens(ids_of(0, T, TOP_K, E).cuda(), E)
    want = f(x, plan)
    with forward.dual_level():
        with pytest.raises((NotImplementedError, RuntimeError)):
            f(forward.make_dual(x, torch.ones_like(x)), plan)
        assert torch.equal(f(x, plan), want)        # without a tangent: as ever


# ------------------------------------------------------------------------------------ the nodes' own duties
@pytest.mark.parametrize("name", NAMES)
def test_backward_twice_and_unused_gradients(X, name):
    f, x, _ = operators(X)[name]
    plan = X.sort_tokens(ids_of(0, T, TOP_K, E).cuda(), E)
    x.requires_grad_()
    out = f(x, plan)
    want = torch.autograd.grad(out.sum(), x)[0]
    with pytest.raises(RuntimeError):                       # what it saved is gone, or it saved nothing and agrees
        again = torch.autograd.grad(out.sum(), x)[0]
        assert torch.equal(again, want)
        raise RuntimeError
    with torch.no_grad():
        assert not f(x, plan).requires_grad
    assert not f(x.detach(), plan).requires_grad
    out = f(x * 1, plan)                                    # an input that is not a leaf
    out.sum().backward()
    assert torch.equal(x.grad, want)


@pytest.mark.parametrize("name", NAMES)
def test_function_transforms_are_right_or_refused(X, name):
    f, x, _ = operators(X)[name]
    plan = X.sort_tokens(ids_of(0, T, TOP_K, E).cuda(), E)
    leaf = x.clone().requires_grad_()
    want = torch.autograd.grad(f(leaf, plan).sum(), leaf)[0]
    both = torch.stack([x, 2 * x])
    for call, right in ((lambda: torch.func.grad(lambda a: f(a, plan).sum())(x), want),
                        (lambda: torch.func.jvp(lambda a: f(a, plan), (x,), (x,))[1], f(x, plan)),
                        (lambda: torch.func.vmap(lambda a: f(a, plan))(both), torch.stack([f(x, plan), f(2 * x, plan)]))):
        try:
            got = call()
        except (RuntimeError, NotImplementedError):
            continue
        assert torch.equal(got, right)


def test_only_the_gradients_that_are_wanted(X):
    plan = X.sort_tokens(ids_of(0, T, TOP_K, E).cuda(), E)
    y, w = torch.randn(T * TOP_K, N).cuda(), torch.rand(T, TOP_K).cuda()
    want = None
    for need_y, need_w in ((True, True), (True, False), (False, True)):
        a, b = y.clone().requires_grad_(need_y), w.clone().requires_grad_(need_w)
        X.combine_tokens(a, plan, b).sum().backward()
        want = want or (a.grad, b.grad)
        assert (torch.equal(a.grad, want[0]) if need_y else a.grad is None)
        assert (torch.equal(b.grad, want[1]) if need_w else b.grad is None)


def test_a_plan_and_a_stack_made_in_inference_mode(X):
    """They can be trained through: the gradient is that of a plan and a stack made outside of it."""
    ids, g = ids_of(0, T, TOP_K, E).cuda(), torch.randn(T * TOP_K, N).cuda()
    made = []
    for mode in (False, True):
        with torch.inference_mode(mode):
            stack, plan = Layer(X, 1, E, K, N, 4, 64).stack, X.sort_tokens(ids, E)
        torch.manual_seed(5)
        x, w = torch.randn(T, K).cuda().requires_grad_(), torch.rand(T, TOP_K).cuda().requires_grad_()
        rows = X.quantized_expert_matmul(x, stack, plan) + X.gather_tokens(x, plan)[:, :N]
        out = X.combine_tokens(rows * g, plan, w)
        made.append(torch.autograd.grad(out.sum(), (x, w), retain_graph=True))
        for a, b in zip(made[-1], torch.autograd.grad(out.sum(), (x, w))):
            assert torch.equal(a, b)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out.sum(), (x, w))
    for a, b in zip(*made):
        assert torch.equal(a, b)
