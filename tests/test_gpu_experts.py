"""Mixture-of-experts operators against plain 64-bit implementations: sizes and masks where they can go wrong.

Tolerances.  A result is rounded once: half a step, eps / 2 of its type, relative to its value; below the smallest
normal number the steps no longer shrink, so half a step is at least eps / 2 of that number (fp16: 2^-11 2^-14).  The products add up
to K + 3 K / g fp32 roundings, each at most 2^-24 of a partial sum; for terms of independent signs a partial sum has
the size of the root of the sum of squares `norm` of the terms as the kernels add them (x (128 + c + |z|) s: codes may
enter with an offset of 128), so K 2^-24 norm covers them.  The transposed product multiplies g s in parts of together
16 bits (24 for fp32): independent relative errors of at most 2^-17 (2^-25), eight times which covers their sum
over all terms, whose size is the norm of g s (c - z).
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def X():
    from jax_gptq_amd import experts
    return experts


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(0)


def half_step(ref, dtype):
    info = torch.finfo(dtype)
    return info.eps / 2 * ref.abs().clamp_min(info.smallest_normal)


def within(got, ref, tol):
    """Largest error in units of its tolerance is at most one."""
    err = (got.detach().cpu().double() - ref).abs()
    worst = float((err / tol.clamp_min(1e-300)).nan_to_num(nan=float("inf")).max()) if err.numel() else 0.0
    assert worst <= 1.0, worst


# ------------------------------------------------------------------------------------ oracle
def ref_sort(ids, E):
    flat = ids.reshape(-1).tolist()
    buckets = [[] for _ in range(E + 1)]
    for i, e in enumerate(flat):
        buckets[e if 0 <= e < E else E].append(i)
    order = [i for b in buckets for i in b]
    position = [0] * len(order)
    for p, i in enumerate(order):
        position[i] = p
    offsets = [0]
    for b in buckets[:E]:
        offsets.append(offsets[-1] + len(b))
    return order, position, offsets


def codes_of(packed, bits):
    p = packed.long()
    if bits == 8:
        return p
    E, R, C = p.shape
    return torch.stack((p & 15, p >> 4), dim=2).reshape(E, 2 * R, C)


class Layer:
    """A random stack on the CPU and on the GPU."""

    def __init__(self, X, seed, E, K, N, bits=4, group=0, tables="fp32", fraction=False):
        gen = torch.Generator().manual_seed(seed)
        self.E, self.K, self.N, self.bits, self.group = E, K, N, bits, group
        R = K // 2 if bits == 4 else K
        self.packed = torch.randint(0, 256, (E, R, N), generator=gen, dtype=torch.uint8)
        shape = (E, K // group, N) if group else (E, N)
        top = 15 if bits == 4 else 255
        zero = torch.rand(shape, generator=gen) * top
        self.zero = (zero if fraction else zero.round()).to(TYPES[tables])
        self.scale = ((0.3 + torch.rand(shape, generator=gen)) * 0.1 / top).to(TYPES[tables])
        self.stack = X.QuantizedExperts(self.packed.cuda(), self.zero.cuda(), self.scale.cuda(), bits, group)

    def parts(self, e):
        """codes, zero, scale of expert e in 64 bits, [K, N] each"""
        c = codes_of(self.packed[e:e + 1], self.bits)[0].double()
        z, s = self.zero[e].double(), self.scale[e].double()
        if self.group:
            return c, z.repeat_interleave(self.group, 0), s.repeat_interleave(self.group, 0)
        return c, z[None].expand_as(c), s[None].expand_as(c)


def ids_of(seed, T, k, E, dropped=0.0, dtype=torch.int64):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.rand(T, E, generator=gen).argsort(dim=1)[:, :k] if k <= E else torch.randint(0, E, (T, k), generator=gen)
    if dropped:
        ids[torch.rand(T, k, generator=gen) < dropped] = -1
    return ids.to(dtype)


def check_product(y, rows, layer, offsets, transpose=False, x_type=None):
    """y [P, N] on the GPU against rows [P, K] (the exact 16- or 32-bit values)."""
    rows, y = rows.double().cpu(), y.detach().cpu()
    x_type = x_type or y.dtype
    for e in range(layer.E):
        a, b = offsets[e], offsets[e + 1]
        if a == b:
            continue
        c, z, s = layer.parts(e)
        w, big = (c - z) * s, (c + 128 + z.abs()) * s
        if transpose:
            w, big = w.t(), big.t()
        ref = rows[a:b] @ w
        norm = (rows[a:b].square() @ big.square()).sqrt()
        tol = half_step(ref, y.dtype) + rows.shape[1] * 2.0 ** -24 * norm
        if transpose:
            part = 2.0 ** -25 if x_type == torch.float32 else 2.0 ** -17
            tol = tol + 8 * part * (rows[a:b].square() @ w.square()).sqrt()
        err = (y[a:b].double() - ref).abs()
        bad = ~(err <= tol)
        assert not bad.any(), (e, int(bad.sum()), float((err / tol).max()), bad.nonzero()[:3].tolist())
    assert (y[offsets[-1]:] == 0).all()


# ------------------------------------------------------------------------------------ sort
@pytest.mark.parametrize("T,k,E,dropped,dtype", [
    (0, 2, 8, 0, torch.int64), (1, 1, 1, 0, torch.int64), (1, 2, 8, 0, torch.int32), (5, 3, 4, 0.5, torch.int64),
    (33, 2, 8, 0.1, torch.int32), (64, 1, 64, 0, torch.int64), (127, 8, 128, 0.05, torch.int32),
    (1025, 2, 60, 0, torch.int64), (8192, 1, 3, 0.02, torch.int32), (8193, 1, 1024, 0, torch.int64),
    (20011, 3, 255, 0.01, torch.int32), (70000, 4, 17, 0, torch.int64), (9, 1, 1024, 0, torch.int64)])
def test_sort(X, T, k, E, dropped, dtype):
    ids = ids_of(T + k, T, k, E, dropped, dtype)
    plan = X.sort_tokens(ids.cuda(), E)
    order, position, offsets = ref_sort(ids, E)
    assert plan.offsets.tolist() == offsets
    assert plan.order.tolist() == order and plan.position.tolist() == position
    assert plan.n_tokens == T and plan.top_k == k and plan.n_rows == T * k


def test_sort_ids_of_nowhere_and_one_busy_expert(X):
    ids = torch.tensor([[0, 1 << 32], [7, 8], [-1, -(1 << 40)], [(1 << 32) + 3, 3], [3, 3], [2 ** 63 - 1, 0]])
    plan = X.sort_tokens(ids.cuda(), 8)
    order, position, offsets = ref_sort(ids, 8)
    assert (plan.order.tolist(), plan.position.tolist(), plan.offsets.tolist()) == (order, position, offsets)
    for value in (5, -1, 8):
        ids = torch.full((3000, 4), value, dtype=torch.int32)
        plan = X.sort_tokens(ids.cuda(), 8)
        assert plan.order.tolist() == list(range(12000))
        assert plan.offsets.tolist() == ref_sort(ids, 8)[2]


def test_sort_other_integer_types_shapes_and_refusals(X):
    ids = torch.randint(0, 6, (2, 5, 3), dtype=torch.int16)
    plan = X.sort_tokens(ids.cuda(), 6)
    assert plan.token_shape == (2, 5) and plan.order.tolist() == ref_sort(ids, 6)[0]
    assert X.sort_tokens(ids[0, :, 0].cuda(), 6).top_k == 1
    t = torch.randint(0, 6, (4, 10)).cuda().t()                       # strided
    assert X.sort_tokens(t, 6).order.tolist() == ref_sort(t.cpu(), 6)[0]
    assert X.sort_tokens(ids.numpy(), 6).order.tolist() == ref_sort(ids, 6)[0]
    with pytest.raises(TypeError):
        X.sort_tokens(torch.zeros(4, 2).cuda(), 6)
    for bad in (0, 1025):
        with pytest.raises(ValueError):
            X.sort_tokens(ids.cuda(), bad)
    with pytest.raises(ValueError):
        X.sort_tokens(torch.zeros(4, 0, dtype=torch.int64).cuda(), 4)
    with pytest.raises(ValueError):
        X.sort_tokens(torch.tensor(3).cuda(), 4)


# ------------------------------------------------------------------------------------ rows
@pytest.mark.parametrize("T,k,E,K,dropped", [(1, 1, 1, 1, 0), (3, 2, 4, 7, 0.3), (17, 2, 8, 64, 0), (29, 4, 16, 909, 0.2),
                                             (130, 1, 5, 2051, 0), (40, 8, 8, 4096, 0.1), (6, 2, 8, 4104, 0)])
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
def test_gather(X, T, k, E, K, dropped, dt):
    ids = ids_of(T, T, k, E, dropped)
    order, position, offsets = ref_sort(ids, E)
    live = offsets[-1]
    x = torch.randn(T, K).to(TYPES[dt])
    g = torch.randn(T * k, K).to(TYPES[dt])
    g[live:] = float("nan")                                           # rows of nowhere: never looked at
    plan = X.sort_tokens(ids.cuda(), E)
    xg = x.cuda().requires_grad_()
    rows = X.gather_tokens(xg, plan)
    want = torch.zeros(T * k, K, dtype=x.dtype)
    want[:live] = x[torch.tensor(order[:live], dtype=torch.long) // k]
    assert torch.equal(rows.detach().cpu(), want)
    assert torch.equal(X.gather_tokens(x.cuda(), plan).cpu(), want)
    (dx,) = torch.autograd.grad(rows, xg, g.cuda())
    ref, size = torch.zeros(T, K, dtype=torch.float64), torch.zeros(T, K, dtype=torch.float64)
    for p, i in enumerate(order[:live]):
        ref[i // k] += g[p].double()
        size[i // k] += g[p].double().abs()
    # k - 1 fp32 additions, one rounding
    within(dx, ref, half_step(ref, x.dtype) + k * 2.0 ** -24 * size)


@pytest.mark.parametrize("T,k,E,K,dropped", [(1, 1, 1, 1, 0), (3, 2, 4, 7, 0.3), (29, 4, 16, 909, 0.2), (6, 2, 8, 4096, 0),
                                             (130, 1, 5, 2051, 0.1), (40, 8, 8, 2304, 0.1)])
@pytest.mark.parametrize("dt,wt", [("fp16", "fp32"), ("bf16", "bf16"), ("fp32", "fp32"), ("bf16", "fp16"),
                                   ("fp16", None)])
def test_combine(X, T, k, E, K, dropped, dt, wt):
    ids = ids_of(T + 1, T, k, E, dropped)
    order, position, offsets = ref_sort(ids, E)
    live = offsets[-1]
    y = torch.randn(T * k, K).to(TYPES[dt])
    y[live:] = float("nan")
    w = torch.rand(T, k).to(TYPES[wt]) if wt else None
    g = torch.randn(T, K).to(TYPES[dt])
    plan = X.sort_tokens(ids.cuda(), E)
    yg = y.cuda().requires_grad_()
    wg = w.cuda().requires_grad_() if wt else None
    out = X.combine_tokens(yg, plan, wg)
    assert out.shape == (T, K) and out.dtype == y.dtype
    wd = w.double() if wt else torch.ones(T, k, dtype=torch.float64)
    ref, size = torch.zeros(T, K, dtype=torch.float64), torch.zeros(T, K, dtype=torch.float64)
    rdy, rdw = torch.zeros(T * k, K, dtype=torch.float64), torch.zeros(T, k, dtype=torch.float64)
    dw_size = torch.zeros(T, k, dtype=torch.float64)
    for p, i in enumerate(order[:live]):
        t, j = divmod(i, k)
        term = wd[t, j] * y[p].double()
        ref[t] += term
        size[t] += term.abs()
        rdy[p] = wd[t, j] * g[t].double()
        rdw[t, j] = (g[t].double() * y[p].double()).sum()
        dw_size[t, j] = (g[t].double() * y[p].double()).abs().sum()
    # k fused multiply-adds of at most 2^-24 of the sum of magnitudes each, one rounding
    within(out, ref, half_step(ref, y.dtype) + k * 2.0 ** -24 * size)
    grads = torch.autograd.grad(out, (yg, wg) if wt else (yg,), g.cuda())
    # one product in fp32, one rounding
    within(grads[0], rdy, half_step(rdy, y.dtype) + 2.0 ** -24 * rdy.abs())
    if wt:
        # K products in chains of at most ceil(K / 256) + 16 additions
        within(grads[1], rdw, half_step(rdw, w.dtype) + (K / 256 + 24) * 2.0 ** -24 * dw_size)
        assert (grads[1].cpu()[torch.tensor(position).reshape(T, k) >= live] == 0).all()


def test_rows_leading_axes_strides_and_refusals(X):
    ids = ids_of(3, 12, 2, 4).reshape(3, 4, 2)
    plan = X.sort_tokens(ids.cuda(), 4)
    x = torch.randn(3, 4, 24).half()
    want = x.reshape(12, 24)[torch.tensor(ref_sort(ids, 4)[0]) // 2]
    assert torch.equal(X.gather_tokens(x.cuda(), plan).cpu(), want)
    wide = torch.randn(3, 4, 48).half().cuda()
    assert torch.equal(X.gather_tokens(wide[..., ::2], plan), X.gather_tokens(wide[..., ::2].contiguous(), plan))
    odd = torch.randn(12 * 24 + 1).half().cuda()[1:].reshape(12, 24)            # starts between two 4-byte words
    assert torch.equal(X.gather_tokens(odd, plan).cpu(), odd.cpu()[torch.tensor(ref_sort(ids, 4)[0]) // 2])
    y = torch.randn(24, 16).cuda()
    assert X.combine_tokens(y, plan).shape == (3, 4, 16)
    assert X.combine_tokens(y, plan, torch.ones(3, 4, 2).cuda()).shape == (3, 4, 16)
    for bad in (torch.zeros(11, 24), torch.zeros(24), torch.zeros(12, 0)):
        with pytest.raises(ValueError):
            X.gather_tokens(bad.cuda(), plan)
    with pytest.raises(ValueError):
        X.combine_tokens(y[:23], plan)
    for bad in (torch.ones(3, 4), torch.ones(4, 3, 4)):
        with pytest.raises(ValueError):
            X.combine_tokens(y, plan, bad.cuda())
    with pytest.raises(ValueError):
        X.combine_tokens(y, plan, torch.ones(24).cuda())


def test_combine_reads_no_row_of_nowhere(X):
    ids = torch.full((5, 2), -1)
    plan = X.sort_tokens(ids.cuda(), 4)
    y = torch.full((10, 33), float("nan")).cuda().requires_grad_()
    w = torch.ones(5, 2).cuda().requires_grad_()
    out = X.combine_tokens(y, plan, w)
    assert (out == 0).all()
    dy, dw = torch.autograd.grad(out, (y, w), torch.ones_like(out))
    assert (dy == 0).all() and (dw == 0).all()
    assert (X.gather_tokens(torch.randn(5, 7).cuda(), plan) == 0).all()


# ------------------------------------------------------------------------------------ products
SHAPES = [  # T, k, E, K, N, bits, group, dropped
    (1, 2, 8, 256, 128, 4, 128, 0),           # one token
    (1, 1, 1, 64, 16, 4, 0, 0),
    (7, 2, 4, 512, 320, 4, 64, 0.2),
    (5, 4, 32, 1024, 200, 4, 32, 0),          # hardly any expert has two rows
    (40, 1, 2, 384, 136, 4, 128, 0),          # more than 16 rows each
    (75, 2, 3, 256, 272, 4, 256, 0.1),
    (150, 2, 2, 320, 528, 4, 64, 0),          # more than 64 rows each
    (300, 2, 4, 512, 640, 4, 128, 0.05),
    (700, 1, 2, 256, 512, 4, 0, 0),           # many rows each
    (19, 2, 4, 250, 909, 4, 0, 0),            # K no multiple of 32, an odd number of channels
    (9, 2, 4, 96, 17, 4, 6, 0),               # groups that are no multiple of 32
    (6, 2, 3, 70, 5, 4, 14, 0.3),
    (3, 2, 4, 2, 1, 4, 0, 0),
    (4, 1, 2, 1056, 33, 4, 96, 0),
    (11, 2, 4, 768, 909, 8, 0, 0),            # 8-bit codes
    (90, 2, 2, 256, 144, 8, 128, 0.1),
    (200, 2, 3, 288, 260, 8, 32, 0),
    (5, 1, 2, 33, 40, 8, 0, 0),               # an odd number of input features
    (5, 1, 2, 35, 40, 8, 7, 0),
]


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_product_and_gradient(X, shape, dt):
    T, k, E, K, N, bits, group, dropped = shape
    layer = Layer(X, sum(shape[:6]), E, K, N, bits, group, tables="fp16" if N % 2 else "fp32")
    ids = ids_of(T, T, k, E, dropped)
    order, _, offsets = ref_sort(ids, E)
    live = offsets[-1]
    token = torch.tensor(order, dtype=torch.long) // k
    plan = X.sort_tokens(ids.cuda(), E)
    x = torch.randn(T, K).to(TYPES[dt])
    xg = x.cuda().requires_grad_()
    y = X.quantized_expert_matmul(xg, layer.stack, plan)
    assert y.shape == (T * k, N) and y.dtype == x.dtype
    check_product(y, x[token], layer, offsets)
    # the same rows in sorted order: the same bits
    rows = X.gather_tokens(x.cuda(), plan).requires_grad_()
    ys = X.quantized_expert_matmul(rows, layer.stack, plan, sorted_rows=True)
    assert torch.equal(ys, y)
    g = torch.randn(T * k, N).to(TYPES[dt])
    g[live:] = float("nan")
    (dr,) = torch.autograd.grad(ys, rows, g.cuda())
    check_product(dr, g, layer, offsets, transpose=True)
    (dx,) = torch.autograd.grad(y, xg, g.cuda())
    ref, tol = torch.zeros(T, K, dtype=torch.float64), torch.zeros(T, K, dtype=torch.float64)
    for e in range(E):
        a, b = offsets[e], offsets[e + 1]
        if a == b:
            continue
        c, z, s = layer.parts(e)
        w, big = ((c - z) * s).t(), ((c + 128 + z.abs()) * s).t()
        part = 2.0 ** -25 if dt == "fp32" else 2.0 ** -17
        gd = g[a:b].double()
        ref.index_add_(0, token[a:b], gd @ w)
        one = (N * 2.0 ** -24 * (gd.square() @ big.square()).sqrt() + 8 * part * (gd.square() @ w.square()).sqrt()
               + 2.0 ** -23 * (gd @ w).abs())
        tol.index_add_(0, token[a:b], one)
    within(dx, ref, tol + half_step(ref, x.dtype))


# More of what decides how a product is computed: many experts (more than a wavefront counts at once), rows per expert
# on either side of each change, both code widths, groups of 32, channels that are no multiple of 16.
MORE_SHAPES = [
    (700, 8, 128, 128, 272, 4, 64, 0.02),     # 128 experts, 43 rows each
    (300, 8, 128, 96, 272, 8, 32, 0.02),      # 18 rows each
    (1100, 1, 1024, 64, 33, 8, 0, 0),         # hardly any columns
    (40, 4, 256, 64, 144, 4, 32, 0.1),        # 160 rows over 256 experts
    (500, 1, 1023, 128, 200, 4, 64, 0.3),
    (60, 1, 2, 384, 136, 4, 128, 0),          # 30 rows each
    (90, 1, 3, 320, 256, 8, 32, 0.1),
    (33, 2, 2, 640, 400, 4, 32, 0),
    (70, 2, 2, 448, 512, 4, 64, 0),           # 70 rows each, K in seven stages
    (90, 2, 2, 512, 255, 8, 0, 0),
    (30, 4, 64, 256, 1040, 4, 256, 0),        # about two rows each, strips that share their last channels
    (17, 1, 1, 8192, 128, 4, 0, 0),           # a long sum without groups
    (200, 1, 1, 4160, 64, 8, 0, 0),
    (260, 2, 64, 64, 1100, 4, 32, 0.05),      # 8 rows each, tiles of 256 channels
    (64, 1, 1, 64, 16, 4, 32, 0),
    (300, 2, 4, 576, 2064, 4, 64, 0.1),       # contractions that are cut, also where rows go nowhere
    (90, 1, 2, 288, 4096, 8, 32, 0.1),
    (20, 2, 4, 260, 1100, 4, 0, 0),
    (600, 2, 2, 512, 1040, 4, 128, 0.05),
    (1200, 2, 600, 128, 1024, 4, 0, 0),       # more tiles than run at a time: the last ones are cut
    (620, 1, 1, 512, 1040, 8, 64, 0),
]


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("shape", MORE_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_product_more_shapes(X, shape, dt):
    test_product_and_gradient(X, shape, dt)


@pytest.mark.parametrize("T", [1, 40, 130, 700])
def test_product_of_subnormal_rows(X, T):
    """Rows of which most values are below fp16's smallest normal number, and a scale that brings the results back."""
    layer = Layer(X, T, 2, 256, 144, 4, 64)
    layer.scale *= 2.0 ** 14
    layer.stack = X.QuantizedExperts(layer.packed.cuda(), layer.zero.cuda(), layer.scale.cuda(), 4, 64)
    ids = ids_of(T, T, 1, 2)
    order, _, offsets = ref_sort(ids, 2)
    plan = X.sort_tokens(ids.cuda(), 2)
    x = (torch.randn(T, 256) * 2e-5).half()
    check_product(X.quantized_expert_matmul(x.cuda(), layer.stack, plan), x[torch.tensor(order)], layer, offsets)
    g = (torch.randn(T, 144) * 2e-5).half()
    y = X.quantized_expert_matmul(g.cuda(), layer.stack, plan, sorted_rows=True, transpose_b=True)
    check_product(y, g, layer, offsets, transpose=True)


@pytest.mark.parametrize("T", [1, 60, 700])
def test_product_where_nothing_goes_anywhere(X, T):
    layer = Layer(X, T, 3, 1024, 1040, 4, 64)
    plan = X.sort_tokens(torch.full((T, 2), -1).cuda(), 3)
    for dt in ("fp16", "fp32"):
        x = torch.full((T, 1024), float("nan")).to(TYPES[dt]).cuda().requires_grad_()
        y = X.quantized_expert_matmul(x, layer.stack, plan)
        assert (y == 0).all()
        (dx,) = torch.autograd.grad(y, x, torch.full_like(y, float("nan")))
        assert (dx == 0).all()


@pytest.mark.parametrize("T,bits,group", [(2, 4, 0), (2, 8, 32), (40, 4, 32), (200, 8, 0), (200, 4, 65536)])
def test_product_of_long_rows(X, T, bits, group):
    E, K, N = 1, 131072, 144
    layer = Layer(X, T, E, K, N, bits, group)
    plan = X.sort_tokens(torch.zeros(T, 1, dtype=torch.int64).cuda(), E)
    x = torch.randn(T, K).bfloat16()
    check_product(X.quantized_expert_matmul(x.cuda(), layer.stack, plan), x, layer, [0, T])
    g = torch.randn(T, N).bfloat16()
    check_product(X.quantized_expert_matmul(g.cuda(), layer.stack, plan, sorted_rows=True, transpose_b=True), g, layer,
                  [0, T], transpose=True)


def test_tables_of_two_types(X):
    layer = Layer(X, 3, 2, 128, 64, 4, 64)
    plan = X.sort_tokens(ids_of(1, 9, 1, 2).cuda(), 2)
    x = torch.randn(9, 128).half().cuda()
    mixed = X.QuantizedExperts(layer.packed.cuda(), layer.zero.half().cuda(), layer.scale.cuda(), 4, 64)
    want = X.quantized_expert_matmul(x, layer.stack, plan)        # the zeros are whole numbers: the same in fp16
    assert torch.equal(X.quantized_expert_matmul(x, mixed, plan), want)
    again = X.stack_experts(list(mixed))
    assert again.scale.dtype == torch.float32 and torch.equal(X.quantized_expert_matmul(x, again, plan), want)


@pytest.mark.parametrize("T", [2, 200])
def test_product_offsets_past_32_bits(X, T):
    """A stack of more than 2^32 bytes whose last expert lies behind that, and an expert wider than most."""
    E, R, N = 10, 512, 1 << 20
    K = 2 * R
    packed = torch.zeros(E, R, N, dtype=torch.uint8, device="cuda")
    packed[-1] = torch.randint(0, 256, (R, N), dtype=torch.uint8, device="cuda")
    assert packed.numel() > 1 << 32
    zero, scale = torch.full((E, N), 8.0, device="cuda"), torch.full((E, N), 0.01, device="cuda")
    stack = X.QuantizedExperts(packed, zero, scale, 4)
    ids = torch.full((T, 1), E - 1)
    ids[0] = 0
    plan = X.sort_tokens(ids.cuda(), E)
    x = torch.randn(T, K).half()
    y = X.quantized_expert_matmul(x.cuda(), stack, plan)
    at = torch.cat([torch.arange(40), torch.arange(N - 40, N), torch.randint(0, N, (40,))])
    codes = codes_of(packed[-1:, :, at.cuda()].cpu(), 4)[0].double()
    w, big = (codes - 8) * 0.01, (codes + 136) * 0.01
    xd = x.double()
    ref, norm = xd @ w, (xd.square() @ big.square()).sqrt()
    ref[0], norm[0] = xd[0].sum() * -0.08, xd[0].norm() * 1.36
    order = torch.tensor(ref_sort(ids, E)[0])
    # (0.01 in fp32 is off by up to 2^-24 of itself, on top of the sum)
    tol = half_step(ref, torch.float16) + (K + 1) * 2.0 ** -24 * norm
    within(y[:, at.cuda()], ref[order], tol[order])
    # and back, where only the columns above hold a gradient
    g = torch.zeros(T, N, dtype=torch.float16)
    at = at.unique()
    g[:, at] = torch.randn(T, at.numel()).half()
    codes = codes_of(packed[-1:, :, at.cuda()].cpu(), 4)[0].double()
    gd = g[:, at].double()
    got = X.quantized_expert_matmul(g.cuda(), stack, plan, sorted_rows=True, transpose_b=True)
    ref, norm = gd @ ((codes - 8) * 0.01).t(), (gd.square() @ ((codes + 136) * 0.01).square().t()).sqrt()
    ref[0], norm[0] = gd[0].sum() * -0.08, gd[0].norm() * 1.36
    part = (gd.square() @ ((codes - 8) * 0.01).square().t()).sqrt()
    part[0] = gd[0].norm() * 0.08
    within(got, ref, half_step(ref, torch.float16) + (N * 2.0 ** -24 + 2.0 ** -24) * norm + 8 * 2.0 ** -17 * part)


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("T,k,E,K,N,bits,group", [(6, 2, 4, 256, 192, 4, 64), (50, 2, 2, 128, 384, 8, 0),
                                                  (260, 1, 2, 384, 256, 4, 128), (5, 2, 3, 36, 21, 4, 12)])
def test_transposed_product_of_tokens(X, T, k, E, K, N, bits, group, dt):
    layer = Layer(X, T, E, K, N, bits, group, tables="bf16")
    ids = ids_of(T, T, k, E)
    order, _, offsets = ref_sort(ids, E)
    x = torch.randn(T, N).to(TYPES[dt])
    xg = x.cuda().requires_grad_()
    plan = X.sort_tokens(ids.cuda(), E)
    y = X.quantized_expert_matmul(xg, layer.stack, plan, transpose_b=True)
    check_product(y, x[torch.tensor(order) // k], layer, offsets, transpose=True)
    g = torch.randn(T * k, K).to(TYPES[dt])
    (dx,) = torch.autograd.grad(y, xg, g.cuda())
    # the gradient is the untransposed product summed over a token's copies: every copy brings K 2^-24 of the norm of
    # its terms (an error relative to the terms, not to their sum: a sum near zero keeps it) and 2^-23 of itself for
    # its fp32 value and the addition
    token = torch.tensor(order) // k
    ref, tol = torch.zeros(T, N, dtype=torch.float64), torch.zeros(T, N, dtype=torch.float64)
    for e in range(E):
        a, b = offsets[e], offsets[e + 1]
        if a == b:
            continue
        c, z, s = layer.parts(e)
        gd = g[a:b].double()
        one = gd @ ((c - z) * s)
        ref.index_add_(0, token[a:b], one)
        tol.index_add_(0, token[a:b], K * 2.0 ** -24 * (gd.square() @ ((c + 128 + z.abs()) * s).square()).sqrt()
                       + 2.0 ** -23 * one.abs())
    within(dx, ref, tol + half_step(ref, x.dtype))


@pytest.mark.parametrize("T", [1, 9, 60, 200])
@pytest.mark.parametrize("tables", ["fp16", "bf16", "fp32"])
def test_product_tables_and_fractional_zeros(X, T, tables):
    layer = Layer(X, T, 3, 256, 144, 4, 64, tables=tables, fraction=True)
    ids = ids_of(T, T, 2, 3)
    order, _, offsets = ref_sort(ids, 3)
    plan = X.sort_tokens(ids.cuda(), 3)
    for dt in ("fp16", "bf16"):
        x = torch.randn(T, 256).to(TYPES[dt])
        check_product(X.quantized_expert_matmul(x.cuda(), layer.stack, plan), x[torch.tensor(order) // 2], layer, offsets)
        g = torch.randn(2 * T, 144).to(TYPES[dt])
        check_product(X.quantized_expert_matmul(g.cuda(), layer.stack, plan, sorted_rows=True, transpose_b=True), g,
                      layer, offsets, transpose=True)


@pytest.mark.parametrize("T,dt", [(4, "fp16"), (40, "bf16"), (40, "fp32"), (300, "fp16"), (300, "bf16")])
def test_product_rows_do_not_see_each_other(X, T, dt):
    """A row of NaN or infinities spoils itself only; one expert takes nearly all rows; an expert stays empty."""
    layer = Layer(X, T, 3, 192, 160, 4, 64)
    ids = torch.zeros(T, 1, dtype=torch.int64)
    ids[0], ids[-1] = 2, -1
    order, _, offsets = ref_sort(ids, 3)
    plan = X.sort_tokens(ids.cuda(), 3)
    x = torch.randn(T, 192).to(TYPES[dt])
    clean = X.quantized_expert_matmul(x.cuda(), layer.stack, plan)
    check_product(clean, x[torch.tensor(order)], layer, offsets)
    bad = x.clone()
    bad[1, 5], bad[2, 7], bad[-1] = float("nan"), float("inf"), float("nan")
    y = X.quantized_expert_matmul(bad.cuda(), layer.stack, plan)
    row = torch.tensor(order)
    keep = ((row != 1) & (row != 2)).cuda()
    assert torch.equal(y[keep], clean[keep])
    assert y[(row == 1).cuda()].isnan().all() and not y[(row == 2).cuda()].isfinite().any()
    g = torch.randn(T, 160).to(TYPES[dt])
    cg = X.quantized_expert_matmul(g.cuda(), layer.stack, plan, sorted_rows=True, transpose_b=True)
    g2 = g.clone()
    g2[0, 3] = float("nan")
    bg = X.quantized_expert_matmul(g2.cuda(), layer.stack, plan, sorted_rows=True, transpose_b=True)
    assert torch.equal(bg[1:], cg[1:]) and bg[0].isnan().all()


def test_product_same_expert_twice_and_repeatable(X):
    layer = Layer(X, 5, 4, 256, 256, 4, 128)
    ids = torch.tensor([[2, 2], [2, 0], [0, 0], [2, 2]])
    order, _, offsets = ref_sort(ids, 4)
    plan = X.sort_tokens(ids.cuda(), 4)
    x = torch.randn(4, 256).half()
    y = X.quantized_expert_matmul(x.cuda(), layer.stack, plan)
    check_product(y, x[torch.tensor(order) // 2], layer, offsets)
    for _ in range(5):
        assert torch.equal(X.quantized_expert_matmul(x.cuda(), layer.stack, plan), y)


def test_product_unaligned_and_strided_operands(X):
    E, K, N = 3, 128, 64
    base = Layer(X, 9, E, K, N, 4, 64)
    ids = ids_of(9, 30, 2, E)
    order, _, offsets = ref_sort(ids, E)
    plan = X.sort_tokens(ids.cuda(), E)
    x = torch.randn(30, K).half()
    want = X.quantized_expert_matmul(x.cuda(), base.stack, plan)
    check_product(want, x[torch.tensor(order) // 2], base, offsets)
    # weights, tables and activations that begin one element past an allocation
    def shifted(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        buf[1:] = t.cuda().reshape(-1)
        return buf[1:].reshape(t.shape)
    odd = X.QuantizedExperts(shifted(base.packed), shifted(base.zero), shifted(base.scale), 4, 64)
    assert torch.equal(X.quantized_expert_matmul(shifted(x), odd, plan), want)
    g = torch.randn(60, N).half()
    back = X.quantized_expert_matmul(g.cuda(), base.stack, plan, sorted_rows=True, transpose_b=True)
    assert torch.equal(X.quantized_expert_matmul(shifted(g), odd, plan, sorted_rows=True, transpose_b=True), back)
    # a stack and activations that are strided views
    wide = torch.randn(30, 2 * K).half()
    assert torch.equal(X.quantized_expert_matmul(wide.cuda()[:, ::2], base.stack, plan),
                       X.quantized_expert_matmul(wide[:, ::2].contiguous().cuda(), base.stack, plan))
    big = torch.zeros(2 * E, K // 2, N, dtype=torch.uint8)
    big[::2] = base.packed
    view = X.QuantizedExperts(big.cuda()[::2], base.zero.cuda(), base.scale.cuda(), 4, 64)
    assert torch.equal(X.quantized_expert_matmul(x.cuda(), view, plan), want)


def test_product_refusals(X):
    layer = Layer(X, 1, 4, 64, 32, 4, 32)
    plan = X.sort_tokens(ids_of(1, 6, 2, 4).cuda(), 4)
    x = torch.randn(6, 64).half().cuda()
    with pytest.raises(TypeError):
        X.quantized_expert_matmul(x, layer.stack[0], plan)
    with pytest.raises(ValueError):
        X.quantized_expert_matmul(x, layer.stack, X.sort_tokens(ids_of(1, 6, 2, 5).cuda(), 5))
    with pytest.raises(ValueError):
        X.quantized_expert_matmul(x, layer.stack, plan, sorted_rows=True)        # 6 rows, not 12
    with pytest.raises(AssertionError):
        X.quantized_expert_matmul(x[:, :32], layer.stack, plan)
    with pytest.raises(ValueError):
        X.quantized_expert_matmul(x, layer.stack.to("cpu"), plan)


def test_empty_batch(X):
    layer = Layer(X, 1, 4, 64, 32, 4, 32)
    plan = X.sort_tokens(torch.zeros(0, 2, dtype=torch.int64).cuda(), 4)
    x = torch.zeros(0, 64).half().cuda().requires_grad_()
    y = X.quantized_expert_matmul(x, layer.stack, plan)
    out = X.combine_tokens(y, plan, torch.zeros(0, 2).cuda())
    assert y.shape == (0, 32) and out.shape == (0, 32) and X.gather_tokens(x, plan).shape == (0, 64)
    (dx,) = torch.autograd.grad(out, x, torch.zeros_like(out))
    assert dx.shape == x.shape


# ------------------------------------------------------------------------------------ as they are used
def _block(X, x, up, gate, down, ids, w):
    plan = X.sort_tokens(ids, len(up))
    h = torch.nn.functional.silu(X.quantized_expert_matmul(x, gate.stack, plan)) * \
        X.quantized_expert_matmul(x, up.stack, plan)
    return X.combine_tokens(X.quantized_expert_matmul(h, down.stack, plan, sorted_rows=True), plan, w)


def _block_ref(x, up, gate, down, ids, w):
    T, k = ids.shape
    rows = []
    for t in range(T):
        acc = torch.zeros(down.N, dtype=torch.float64)
        for j in range(k):
            e = int(ids[t, j])
            if not 0 <= e < up.E:
                continue
            wu, wg, wd = (((c - z) * s) for c, z, s in (up.parts(e), gate.parts(e), down.parts(e)))
            acc = acc + w[t, j] * ((torch.nn.functional.silu(x[t] @ wg) * (x[t] @ wu)) @ wd)
        rows.append(acc)
    return torch.stack(rows)


Layer.__len__ = lambda self: self.E


@pytest.mark.parametrize("T", [1, 6, 70])
def test_block_and_its_gradients(X, T):
    """The pieces as a layer uses them, fp32, against 64 bits and against differences of the 64-bit block."""
    E, k, K, H = 4, 2, 128, 192
    up, gate, down = Layer(X, 1, E, K, H, 4, 64), Layer(X, 2, E, K, H, 4, 64), Layer(X, 3, E, H, K, 4, 0)
    ids = ids_of(T, T, k, E, 0.2 if T > 1 else 0)
    x, w, g = torch.randn(T, K), torch.rand(T, k), torch.randn(T, K)
    xg, wg = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    out = _block(X, xg, up, gate, down, ids.cuda(), wg)
    xd, wd = x.double().requires_grad_(), w.double().requires_grad_()
    ref = _block_ref(xd, up, gate, down, ids, wd)
    # three products of about 2^-17 relative to their size, each: 2^-14 of the largest value
    assert (out.detach().cpu().double() - ref.detach()).abs().max() <= 2.0 ** -14 * ref.abs().max()
    dx, dw = torch.autograd.grad(out, (xg, wg), g.cuda())
    rdx, rdw = torch.autograd.grad(ref, (xd, wd), g.double())
    assert (dx.cpu().double() - rdx).abs().max() <= 2.0 ** -13 * rdx.abs().max()
    assert (dw.cpu().double() - rdw).abs().max() <= 2.0 ** -13 * rdw.abs().max()
    # the formula's gradient itself, by central differences of the 64-bit block along one direction
    d, h = torch.randn(T, K, dtype=torch.float64), 1e-5
    with torch.no_grad():
        plus = (_block_ref(xd + h * d, up, gate, down, ids, wd) * g.double()).sum()
        minus = (_block_ref(xd - h * d, up, gate, down, ids, wd) * g.double()).sum()
    slope, scale = (plus - minus) / (2 * h), (rdx * d).norm()
    assert abs(float(slope - (dx.cpu().double() * d).sum())) <= 1e-3 * float(scale) + 1e-9


@pytest.mark.parametrize("T,dt", [(1, "fp16"), (24, "bf16"), (200, "fp16")])
def test_block_in_a_graph_on_another_stream(X, T, dt):
    """Captured and replayed with new inputs, eager work between the replays."""
    E, k, K, H = 8, 2, 256, 320
    up, gate, down = Layer(X, 1, E, K, H, 4, 64), Layer(X, 2, E, K, H, 4, 64), Layer(X, 3, E, H, K, 4, 32)
    x = torch.randn(T, K).to(TYPES[dt]).cuda()
    w = torch.rand(T, k).cuda()
    ids = ids_of(0, T, k, E).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _block(X, x, up, gate, down, ids, w)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _block(X, x, up, gate, down, ids, w)
    for i in range(4):
        x.copy_(torch.randn(T, K))
        w.copy_(torch.rand(T, k))
        ids.copy_(ids_of(i + 1, T, k, E, 0.1 if i == 2 else 0))
        graph.replay()
        torch.cuda.synchronize()
        want = _block(X, x, up, gate, down, ids, w)
        assert torch.equal(out, want)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = _block(X, x, up, gate, down, ids, w)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, want)


def test_two_streams_at_once(X):
    """Calls on two streams, neither waiting for the other, each with its own workspaces."""
    E, k, K, H, T = 4, 2, 512, 768, 300
    layers = [(Layer(X, i, E, K, H, 4, 64), Layer(X, i + 5, E, K, H, 4, 64), Layer(X, i + 9, E, H, K, 4, 64))
              for i in range(2)]
    xs = [torch.randn(T, K).half().cuda() for _ in range(2)]
    ids = [ids_of(i, T, k, E).cuda() for i in range(2)]
    w = torch.rand(T, k).cuda()
    want = [_block(X, xs[i], *layers[i], ids[i], w) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(6):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(_block(X, xs[i], *layers[i], ids[i], w))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert torch.equal(y, want[i])


def test_two_graphs_replayed_in_turn(X):
    E, k, K, H = 4, 2, 256, 384
    up, gate, down = Layer(X, 1, E, K, H, 4, 64), Layer(X, 2, E, K, H, 4, 64), Layer(X, 3, E, H, K, 4, 64)
    graphs = []
    for T in (3, 260):
        x, w, ids = torch.randn(T, K).half().cuda(), torch.rand(T, k).cuda(), ids_of(T, T, k, E).cuda()
        _block(X, x, up, gate, down, ids, w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _block(X, x, up, gate, down, ids, w)
        graphs.append((graph, x, w, ids, out))
    for _ in range(3):
        for _, x, _, _, _ in graphs:
            x.copy_(torch.randn(x.shape))
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, x, w, ids, out in graphs:
            assert torch.equal(out, _block(X, x, up, gate, down, ids, w))


def test_gradient_in_a_graph(X):
    E, k, K, H, T = 4, 2, 128, 192, 50
    layer = Layer(X, 1, E, K, H, 4, 64)
    ids = ids_of(0, T, k, E).cuda()
    x, g, w = torch.randn(T, K).half().cuda(), torch.randn(T, H).half().cuda(), torch.rand(T, k).cuda()

    def step():
        xi, wi = x.detach().requires_grad_(), w.detach().requires_grad_()
        plan = X.sort_tokens(ids, E)
        out = X.combine_tokens(X.quantized_expert_matmul(xi, layer.stack, plan), plan, wi)
        return (out.detach(),) + torch.autograd.grad(out, (xi, wi), g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        x.copy_(torch.randn(T, K))
        g.copy_(torch.randn(T, H))
        ids.copy_(ids_of(i + 5, T, k, E, 0.1))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_gradient_of_the_gradient(X):
    """A graph of the gradient (create_graph) goes through the operators again; fp32 against the 64-bit block."""
    E, k, K, H, T = 3, 2, 64, 96, 9
    up, gate, down = Layer(X, 1, E, K, H, 4, 32), Layer(X, 2, E, K, H, 4, 32), Layer(X, 3, E, H, K, 4, 32)
    ids = ids_of(4, T, k, E, 0.2)
    x, w, g = torch.randn(T, K), torch.rand(T, k), torch.randn(T, K)

    def second(block, x, w, g, ids):
        out = block(x, ids, w)
        dx, dw = torch.autograd.grad(out, (x, w), g, create_graph=True)
        return torch.autograd.grad(dx.square().sum() + dw.square().sum(), (x, w))
    got = second(lambda a, i, b: _block(X, a, up, gate, down, i, b), x.cuda().requires_grad_(),
                 w.cuda().requires_grad_(), g.cuda(), ids.cuda())
    ref = second(lambda a, i, b: _block_ref(a, up, gate, down, i, b), x.double().requires_grad_(),
                 w.double().requires_grad_(), g.double(), ids)
    for a, b in zip(got, ref):
        assert (a.cpu().double() - b).abs().max() <= 2.0 ** -12 * b.abs().max()
    # and the rows' own operators
    plan = X.sort_tokens(ids.cuda(), E)
    r = torch.randn(T, K).cuda().requires_grad_()
    rows = X.gather_tokens(r, plan)
    (d,) = torch.autograd.grad(rows.square().sum(), r, create_graph=True)
    (dd,) = torch.autograd.grad(d.sum(), r)
    live = torch.tensor([[float(0 <= int(i) < E) for i in row] for row in ids]).sum(1).cuda()
    assert torch.allclose(dd, 2 * live[:, None].expand_as(dd))


# ------------------------------------------------------------------------------------ the solve for a layer of experts
@pytest.mark.parametrize("group", [None, 128])
def test_gptq_experts(X, group):
    """Each expert's codes are those of gptq() on the rows that reach it; an expert without rows is rounded to its own
    grid."""
    from jax_gptq_amd.gptq import gptq, pack_matrix, unpack_matrix
    E, K, N, T = 3, 128, 96, 400
    W = (0.05 * torch.randn(E, K, N)).cuda()
    xs = [torch.randn(T, K).cuda() for _ in range(2)]
    ids = [torch.randint(0, 2, (T, 1)).cuda() * 2 for _ in range(2)]              # experts 0 and 2
    stack = X.gptq_experts(W, xs, ids, group_size=group)
    assert stack.shape == (E, K, N) and stack.group_size == (group or 0)
    for e in (0, 2):
        Q, p = gptq(W[e], [x[i[:, 0] == e] for x, i in zip(xs, ids)], group_size=group)
        assert torch.equal(stack[e].int_weight, pack_matrix(Q, p).int_weight)
    step = stack.scale[1].max()
    assert (unpack_matrix(stack[1]) - W[1]).abs().max() <= 0.5001 * step
    plan = X.sort_tokens(ids[0], E)
    y = X.quantized_expert_matmul(xs[0], stack, plan)
    rows = X.gather_tokens(xs[0], plan)
    at = plan.offsets.tolist()
    for e in (0, 2):
        want = rows[at[e]:at[e + 1]].double() @ unpack_matrix(stack[e]).double()
        assert (y[at[e]:at[e + 1]].double() - want).abs().max() <= 1e-5 * want.abs().max()
    with pytest.raises(ValueError):
        X.gptq_experts(W[0], xs, ids)
    with pytest.raises(ValueError):
        X.gptq_experts(W, xs, ids[:1])
    with pytest.raises(ValueError):
        X.gptq_experts(W, [x[:, :64] for x in xs], ids)


def test_stack_experts_is_the_matrices(X):
    from jax_gptq_amd.gptq import get_col_quantize_params, pack_matrix, unpack_matrix
    qs = []
    for e in range(3):
        W = torch.randn(64, 24).cuda()
        p = get_col_quantize_params(W)
        codes = (W / p["scale"] + p["zero"]).round().clamp(0, 15)
        qs.append(pack_matrix((codes - p["zero"]) * p["scale"], p))
    stack = X.stack_experts(qs)
    for q, s in zip(qs, stack):
        assert torch.equal(unpack_matrix(q), unpack_matrix(s))
