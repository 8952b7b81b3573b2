"""The solve for a layer of experts: what it holds while it runs, and rows in every form that a batch may have."""
import pytest
import torch

from test_gpu_experts import ids_of

pytestmark = pytest.mark.gpu


def _peak(call):
    """Bytes that a call holds at most beyond what was there before."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    call()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before


def test_one_experts_rows_are_held_at_a_time():
    from jax_gptq_amd.experts import gptq_experts
    from jax_gptq_amd.gptq import gptq
    E, K, N, T = 16, 256, 64, 2048
    W = (0.05 * torch.randn(E, K, N)).cuda()
    xs = [torch.randn(T, K).cuda() for _ in range(2)]
    ids = [torch.arange(E).repeat(T, 1).cuda() for _ in range(2)]             # every token to every expert
    one = _peak(lambda: gptq(W[0], xs))
    # beside one solve: one expert's rows (as many bytes as the batches), the plans (2 E T + E + 1 numbers of 4 bytes each,
    # twice while they are made), the packed stack twice, and 4 MiB for what allocations are rounded up to
    batches = sum(x.numel() * 4 for x in xs)
    plans = 2 * (2 * E * T + E + 1) * 4
    stack = E * (K // 2 * N + 8 * N)
    assert _peak(lambda: gptq_experts(W, xs, ids)) <= one + batches + 2 * plans + 2 * stack + (4 << 20) < one + E * batches


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float32])
def test_batches_of_every_form(dt):
    """Leading axes, strides, host tensors, an empty batch, a batch that reaches one expert only, padded ids: the codes are
    those of gptq() on the rows themselves."""
    from jax_gptq_amd.experts import gptq_experts
    from jax_gptq_amd.gptq import gptq, pack_matrix
    torch.manual_seed(0)
    E, K, N = 3, 128, 48
    W = (0.05 * torch.randn(E, K, N)).cuda()
    xs = [torch.randn(4, 50, K).to(dt).cuda(), torch.randn(150, 2 * K).to(dt).cuda()[:, ::2], torch.randn(170, K).to(dt),
          torch.zeros(0, K).to(dt).cuda(), torch.randn(140, K).to(dt).cuda()]
    ids = [ids_of(1, 200, 2, E, 0.1).reshape(4, 50, 2), ids_of(2, 150, 1, E), ids_of(3, 170, 2, E, 0.2),
           torch.zeros(0, 2, dtype=torch.int64), torch.full((140, 1), 1)]
    stack = gptq_experts(W, xs, [i.cuda() for i in ids])
    for e in range(E):
        rows = []
        for x, i in zip(xs, ids):
            token, _ = (i.reshape(-1, i.shape[-1]) == e).nonzero(as_tuple=True)
            if token.numel():
                rows.append(x.reshape(-1, K).cpu()[token].cuda())
        Q, p = gptq(W[e], rows)
        assert torch.equal(stack[e].int_weight, pack_matrix(Q, p).int_weight)
