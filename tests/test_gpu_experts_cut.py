"""Products whose tiles fill whole rounds of workgroups and a bit of another: the tiles of the last round are cut along the
contraction and joined by a second kernel, the others are not."""
import pytest
import torch

from test_gpu_experts import test_product_and_gradient as check_product_and_gradient

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def X():
    from jax_gptq_amd import experts
    return experts


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


CUT = [  # T, top_k, E, K, N, bits, group, dropped
    (600, 2, 2, 1024, 6800, 4, 128, 0),       # 540 tiles of 64 x 256 (fp32: 1026 of 32 x 256), 512 (1024) at a time
    (600, 2, 2, 1024, 6800, 8, 32, 0.02),
    (900, 1, 9, 1024, 4096, 4, 64, 0),        # 288 tiles in two halves of K, 256 at a time
    (600, 2, 2, 13600, 1040, 4, 32, 0),       # transposed, 540 tiles of 128 x 256, 512 (fp32: 256) at a time
    (600, 2, 2, 13600, 1040, 8, 0, 0.02),
    (1200, 2, 16, 5632, 1040, 4, 128, 0),     # transposed, 1056 tiles of 64 x 256, 1024 (512) at a time
    (640, 2, 64, 4352, 1040, 4, 64, 0),       # transposed, about 1088 tiles of 32 x 256, the same
]


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("shape", CUT, ids=lambda s: "x".join(map(str, s)))
def test_whole_rounds_and_a_cut_one(X, shape, dt):
    check_product_and_gradient(X, shape, dt)
