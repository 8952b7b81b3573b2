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
