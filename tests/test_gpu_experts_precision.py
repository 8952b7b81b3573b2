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


def wide_product(x, stack, plan, transpose):
    """The sorted rows' product in fp32 whatever the rows' type, through the C entry point."""
    from jax_gptq_amd import _native as N
    lib, code = N.load(), {torch.float16: N.F16, torch.bfloat16: N.BF16, torch.float32: N.F32}
    E, R, C = stack.int_weight.shape
    out = torch.empty(x.shape[0], stack.shape[1 if transpose else 2], device=x.device)
    sizes = (stack.group_size, E, code[x.dtype], code[stack.zero.dtype], transpose)
    ws = torch.empty(lib.gptq_hip_expert_qmatmul_workspace_bytes(x.shape[0], x.shape[0], R, C, stack.bits, *sizes) + 16,
                     dtype=torch.uint8, device=x.device)
    N.check(lib.gptq_hip_expert_qmatmul(
        torch.cuda.current_stream().cuda_stream, x.data_ptr(), code[x.dtype], x.shape[0], None, plan.top_k, x.shape[0],
        plan.offsets.data_ptr(), E, stack.int_weight.data_ptr(), R, C, stack.zero.data_ptr(), stack.scale.data_ptr(),
        code[stack.zero.dtype], stack.group_size, stack.bits, transpose, out.data_ptr(), N.F32, ws.data_ptr(), ws.numel()),
        "expert_qmatmul")
    return out


@pytest.mark.parametrize("rows", [3, 60, 300])
@pytest.mark.parametrize("bits,group", [(8, 0), (8, 32), (4, 64)])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_transposed_product_cuts_operands_by_2_to_the_minus_18(X, rows, bits, group, dt):
    """Two bf16 parts rounded to nearest leave out 2^-9 2^-9 of x s; fp32 results show it.  All terms are positive (zeros
    of 0), so the error is at most that much of the sum, and r 2^-24 of it for the roundings of 64 channels."""
    N = 64
    layer = Layer(X, rows, 1, 128, N, bits, group)
    layer.zero.zero_()
    # products with a row of ones whose last bits are all set, in the first half of the channels
    layer.scale[..., :N // 2] = 1 + 2.0 ** -15 - 2.0 ** -23
    layer.scale[..., 1:N // 2:2] = 1 + 2.0 ** -9 - 2.0 ** -17
    layer.stack = X.QuantizedExperts(layer.packed.cuda(), layer.zero.cuda(), layer.scale.cuda(), bits, group)
    plan = one_expert(X, rows)
    g = torch.randn(rows, N).abs()
    g[:(rows + 1) // 2] = 1
    g = g.to(TYPES[dt])
    c, _, s = layer.parts(0)
    ref = g.double() @ (c * s).t()
    # bits 4: the codes come with an offset of at most 128, whose sum is taken off again: 2 (128 + 15) / mean code more
    size = ref if bits == 8 else g.double() @ ((c + 256) * s).t()
    err = (wide_product(g.cuda(), layer.stack, plan, 1).cpu().double() - ref).abs()
    tol = 2.0 ** -18 * ref + (2 * N // 16 + 3) * 2.0 ** -24 * size
    assert (err <= tol).all(), float((err / ref).max())


# rows: strips, tiles of 32 and 64 rows
@pytest.mark.parametrize("rows", [4, 28, 100, 200])
@pytest.mark.parametrize("K,bits,group", [(8192, 4, 8192), (8192, 4, 0), (6144, 4, 1024), (8448, 8, 4224), (4928, 4, 704),
                                          (65536, 4, 65536), (4096, 4, 128)])
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
def test_product_of_one_sign(X, rows, K, bits, group, dt):
    """Rows behind a function that leaves one sign; sums without groups and groups of many hundred features."""
    layer = Layer(X, K, 1, K, 144, bits, group)
    x = torch.randn(rows, K).abs()
    x[:rows // 2] = 1
    x = x.to(TYPES[dt])
    y = X.quantized_expert_matmul(x.cuda(), layer.stack, one_expert(X, rows))
    # pieces of 512 features: up to 96 products, 8 + 8 + 8 additions for the rows' sum, what joins them
    check_pieces(y, x, layer, 512, 96 + 24 + 8)
