"""Experts' products where rounding could hide: rows and gradients of one sign, long sums, what is cut off an operand.

The kernels add up x (o + c) with codes that enter under an offset o (0, 64 or 128) and take x (o + z) from it, piece by
piece of the contraction.  Every fp32 rounding within a piece is at most 2^-24 of S, the sum of |x| (128 + c + |z|) s
over the piece; r of them, independent, come to sqrt(r) 2^-24 S, and pieces add up as the root of the sum of squares.
Four times that covers the largest of some thousand outputs.  Rows of random sign would not see it: their sums are small
themselves.
"""
import pytest
import torch

from test_gpu_experts import TYPES, Layer, half_step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def X():
    from jax_gptq_amd import experts
    return experts


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


def one_expert(X, rows):
    return X.sort_tokens(torch.zeros(rows, 1, dtype=torch.int64).cuda(), 1)


def check_pieces(y, rows, layer, piece, roundings, cut=0.0, transpose=False):
    """``y`` against ``rows @ W`` in 64 bits, pieces of ``piece`` terms with ``roundings`` fp32 roundings each; ``cut``:
    relative error of one multiplied operand."""
    rows, y = rows.double().cpu(), y.cpu()
    c, z, s = layer.parts(0)
    w, big = (c - z) * s, (c + 128 + z.abs()) * s
    if transpose:
        w, big = w.t(), big.t()
    ref = rows @ w
    squares = torch.zeros_like(ref)
    for at in range(0, w.shape[0], piece):
        squares += (rows[:, at:at + piece].abs() @ big[at:at + piece].abs()).square()
    tol = half_step(ref, y.dtype) + 4 * roundings ** 0.5 * 2.0 ** -24 * squares.sqrt()
    tol = tol + 4 * cut * (rows.square() @ w.square()).sqrt()
    err = (y.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float((err / tol).max()), float(err.square().mean().sqrt() / ref.square().mean().sqrt()))


# rows: tiles of 32, 64 and 128 rows
@pytest.mark.parametrize("rows", [8, 100, 300])
@pytest.mark.parametrize("N,bits,group", [(11008, 4, 128), (11008, 8, 0), (11008, 4, 32), (65552, 4, 0), (65536, 8, 64),
                                          (33, 4, 64)])
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
def test_transposed_product_of_one_sign(X, rows, N, bits, group, dt):
    """The gradient of a sum, and gradients after a function that leaves one sign."""
    layer = Layer(X, N, 1, 128, N, bits, group)
    plan = one_expert(X, rows)
    g = torch.randn(rows, N).abs()
    g[:rows // 2] = 1
    g = g.to(TYPES[dt])
    y = X.quantized_expert_matmul(g.cuda(), layer.stack, plan, sorted_rows=True, transpose_b=True)
    # pieces of 128 channels: up to 24 products into one sum, 64 terms in the other, the six parts that join them
    check_pieces(y, g, layer, 128, 24 + 64 + 6, cut=2.0 ** -25 if dt == "fp32" else 2.0 ** -15, transpose=True)
