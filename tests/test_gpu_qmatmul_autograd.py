"""What autograd may ask of ``quantized_matmul`` besides a plain backward pass."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _matrix(bits=4):
    from jax_gptq_amd.gptq import QuantizedMatrix
    gen = torch.Generator().manual_seed(1)
    packed = torch.randint(0, 256, (64 if bits == 4 else 128, 96), generator=gen, dtype=torch.uint8)
    zero, scale = torch.full((96,), 8.0), torch.rand(96, generator=gen) * 0.01 + 0.005
    return QuantizedMatrix(packed.cuda(), zero.cuda(), scale.cuda(), bits=bits)


@pytest.mark.parametrize("transpose", [False, True])
def test_forward_mode_is_refused(transpose):
    """A tangent is not lost without a word."""
    import torch.autograd.forward_ad as forward
    from jax_gptq_amd.op import quantized_matmul
    w, x = _matrix(), torch.randn(5, 96 if transpose else 128).half().cuda()
    want = quantized_matmul(x, w, transpose_b=transpose)
    with forward.dual_level():
        with pytest.raises((NotImplementedError, RuntimeError)):
            quantized_matmul(forward.make_dual(x, torch.ones_like(x)), w, transpose_b=transpose)
        assert torch.equal(quantized_matmul(x, w, transpose_b=transpose), want)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("transpose", [False, True])
def test_a_graph_of_the_gradient_is_recorded(bits, transpose):
    """grad(sum(grad(sum(y^2) / 2) . v)) = W W^T v, which was missing without a word beside other terms."""
    from jax_gptq_amd.gptq import unpack_matrix
    from jax_gptq_amd.op import quantized_matmul
    torch.manual_seed(0)
    w = _matrix(bits)
    if bits == 8:
        w.zero.fill_(128)
        w.scale /= 16
    dense = unpack_matrix(w).double()
    dense = dense.t() if transpose else dense
    x = torch.randn(5, dense.shape[0]).half().cuda().requires_grad_()
    v = torch.randn_like(x)
    y = quantized_matmul(x, w, transpose_b=transpose)
    plain = torch.autograd.grad(y, x, y.detach(), retain_graph=True)[0]
    dx = torch.autograd.grad((y.float().square() / 2).sum(), x, create_graph=True)[0]
    assert torch.equal(plain, dx)
    second = torch.autograd.grad((dx.float() * v.float()).sum() + x.float().sum(), x)[0]
    want = v.double() @ dense @ dense.t() + 1
    # two products and a sum, each rounded once to fp16 (a half step of the largest value), and what the kernels' operands
    # leave out (2^-11 of a term): 2^-8 of the largest value covers them
    assert (second.double() - want).abs().max() <= 2.0 ** -8 * want.abs().max()


@pytest.mark.parametrize("remat", [False, True])
def test_a_graph_of_the_gradient_is_recorded_by_unpacked_products(remat):
    """The same where a model function's product unpacks the matrix, and drops it until the backward pass."""
    from jax_gptq_amd import use_quantized
    from jax_gptq_amd.gptq import unpack_matrix
    torch.manual_seed(0)
    w = _matrix()
    dense = unpack_matrix(w).double()
    x = torch.randn(5, dense.shape[0]).cuda().requires_grad_()
    v = torch.randn_like(x)
    y = use_quantized(lambda p, a: a @ p, use_kernel=False, remat_unpack=remat)(w, x)
    plain = torch.autograd.grad(y, x, y.detach(), retain_graph=True)[0]
    dx = torch.autograd.grad((y.square() / 2).sum(), x, create_graph=True)[0]
    assert torch.equal(plain, dx)
    second = torch.autograd.grad((dx * v).sum() + x.sum(), x)[0]
    want = v.double() @ dense @ dense.t() + 1
    # two fp32 products of 128 and 96 terms: (128 + 96) 2^-24 of the terms' sizes, well under 2^-14 of the largest value
    assert (second.double() - want).abs().max() <= 2.0 ** -14 * want.abs().max()
