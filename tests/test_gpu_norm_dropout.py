"""Group norm with an activation (csrc/group_norm.hip) and seeded dropout (csrc/dropout.hip) against 64-bit definitions.

Tolerances.  u = 2^-24.  The statistics are sums of at most 64 terms a thread joined in wider steps, so mean and 1 / std
carry at most 64 u of the mean absolute deviation, which is below one standard deviation: 64 u (1 + |xhat|) |w| in z.
The adds of z and the native exponential cost a few u of the terms.  Outputs are rounded once: half a step of their type.
"""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _map(shape, dtype, seed, layout="channels_last", mean=0.0):
    n, c, h, w = shape
    g = torch.Generator().manual_seed(seed)
    t = (torch.randn(shape, generator=g) + mean).to(dtype)
    if layout == "slice":                          # a channel slice of a wider channels-last buffer
        buf = torch.randn(n, c + 16, h, w, generator=g).to(dtype).cuda().contiguous(memory_format=torch.channels_last)
        buf[:, 8:8 + c] = t.cuda()
        return buf[:, 8:8 + c]
    if layout == "odd slice":                      # rows that start off 16 bytes
        buf = torch.randn(n, c + 3, h, w, generator=g).to(dtype).cuda().contiguous(memory_format=torch.channels_last)
        buf[:, 1:1 + c] = t.cuda()
        return buf[:, 1:1 + c]
    t = t.cuda()
    return t.contiguous(memory_format=torch.channels_last) if layout == "channels_last" else t.contiguous()


def _definition(x, groups, w, b, eps, act, res, dy):
    """(y, dx, dw, db, dres, z, xhat, dz, rstd) in 64 bits."""
    n, c, h, wd = x.shape
    x, w, b, dy = x.double(), w.double().view(1, c, 1, 1), b.double().view(1, c, 1, 1), dy.double()
    g = x.reshape(n, groups, -1)
    var, mean = torch.var_mean(g, dim=2, keepdim=True, unbiased=False)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = ((g - mean) * rstd).reshape(x.shape)
    z = xhat * w + b + (res.double() if res is not None else 0)
    s = torch.sigmoid(z)
    y = {None: z, "relu": z.clamp_min(0), "silu": z * s}[act]
    dz = {None: dy, "relu": dy * (z > 0), "silu": dy * s * (1 + z * (1 - s))}[act]
    t = (dz * w).reshape(n, groups, -1)
    xg = xhat.reshape(n, groups, -1)
    dx = rstd * (t - t.mean(2, keepdim=True) - xg * (t * xg).mean(2, keepdim=True))
    return (y, dx.reshape(x.shape), (dz * xhat).sum((0, 2, 3)), dz.sum((0, 2, 3)), dz, z, xhat, dz,
            rstd.expand_as(g).reshape(x.shape))


def _within(name, got, want, tol):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (name, int(bad.sum()), float((err / tol.clamp_min(1e-300)).max()))


def _check_norm(shape, groups, dtype, act, residual, layout="channels_last", mean=0.0, seed=0):
    from distributedpytorch_amd import ops
    n, c, h, w = shape
    x = _map(shape, dtype, seed, layout, mean)
    res = _map(shape, dtype, seed + 1, layout) if residual else None
    dy = _map(shape, dtype, seed + 2, layout)
    g = torch.Generator().manual_seed(seed + 3)
    wt, bs = (1 + 0.3 * torch.randn(c, generator=g)).cuda(), (0.3 * torch.randn(c, generator=g)).cuda()
    y64, dx64, dw64, db64, dr64, z, xhat, dz, rstd = _definition(x, groups, wt, bs, 1e-5, act, res, dy)
    if act == "relu":      # (the oracle's inputs hold no value on the border itself)
        zn = (z - res.double()).abs() if residual else 0.0
        assert (z.abs() > 8 * U * zn).all()
    leaves = [t.detach().requires_grad_(True) for t in ([x, wt, bs] + ([res] if residual else []))]
    y = ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], 1e-5, act=act,
                           residual=leaves[3] if residual else None)
    assert y.is_contiguous(memory_format=torch.channels_last) and y.dtype == dtype
    with torch.no_grad():
        again = ops.group_norm_act(x, groups, wt, bs, 1e-5, act=act, residual=res)
    assert torch.equal(again, y)
    grads = torch.autograd.grad(y, leaves, dy)
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps      # half a step of the subnormal range and more
    wv = wt.double().abs().view(1, c, 1, 1)
    dz_err = 64 * U * (1 + xhat.abs()) * wv + 8 * U * (z.abs() + xhat.abs() * wv + 1)
    _within("y", y, y64, half * y64.abs() + 1.2 * dz_err + 16 * U * y64.abs() * (1 + z.abs()) + tiny)
    # silu'' and the cost of its native exponential: |silu'| <= 1.1, |silu''| <= 0.5
    e_dz = (0.5 * dz_err + 32 * U) * dy.double().abs() if act == "silu" else 0.0 * dy.double()
    t = (dz * wv).abs()
    gmean = lambda a: a.reshape(n, groups, -1).mean(2, keepdim=True).expand(n, groups, c // groups * h * w).reshape(a.shape)  # noqa: E731,E501
    scale = rstd * (t + gmean(t) + xhat.abs() * gmean(t * (1 + xhat.abs())))
    tol = half * dx64.abs() + 160 * U * scale * (1 + xhat.abs()) + rstd * (e_dz * wv + gmean(e_dz * wv) * (1 + xhat.abs())) + tiny
    _within("dx", grads[0], dx64, tol)
    tot = (dz.abs() * (1 + xhat.abs())).sum((0, 2, 3))
    extra = (e_dz * (1 + xhat.abs())).sum((0, 2, 3))
    _within("dw", grads[1], dw64, 160 * U * tot + extra + 1e-30)
    _within("db", grads[2], db64, 160 * U * tot + extra + 1e-30)
    if residual:
        _within("dres", grads[3], dr64, half * dr64.abs() + e_dz + 4 * U * dr64.abs() + tiny)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act,residual", [(None, False), (None, True), ("relu", False), ("relu", True), ("silu", True)])
def test_group_norm_types_and_activations(dtype, act, residual):
    _check_norm((3, 48, 17, 13), 16, dtype, act, residual)


@pytest.mark.parametrize("shape,groups", [
    ((1, 1, 1, 1), 1), ((2, 8, 1, 1), 8), ((2, 8, 1, 1), 1), ((1, 3, 2, 12), 1), ((2, 21, 9, 7), 7), ((5, 3, 77, 7), 3),
    ((1, 256, 33, 33), 32), ((2, 304, 31, 29), 16), ((2, 728, 5, 9), 8), ((1, 2048, 10, 5), 4), ((1, 2056, 3, 3), 257),
    ((1, 64, 129, 129), 1), ((40, 64, 2, 2), 32), ((1, 4, 257, 255), 2),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_group_norm_shapes(shape, groups, dtype):
    _check_norm(shape, groups, dtype, "silu", False, seed=sum(shape))


@pytest.mark.parametrize("shape,groups", [
    # on both sides of what one block holds: single elements, packs, and more blocks than two a CU
    ((3, 48, 51, 53), 16), ((3, 48, 55, 51), 16), ((2, 64, 61, 33), 8), ((2, 64, 65, 67), 8), ((16, 96, 9, 7), 32),
    ((17, 96, 9, 7), 32), ((17, 192, 9, 7), 32),
])
@pytest.mark.parametrize("act,residual", [("relu", False), ("silu", True), (None, True)])
@pytest.mark.parametrize("dtype", TYPES)
def test_group_norm_groups_in_one_block_and_in_passes(shape, groups, act, residual, dtype):
    _check_norm(shape, groups, dtype, act, residual, seed=sum(shape))


@pytest.mark.parametrize("layout", ["contiguous", "slice", "odd slice"])
@pytest.mark.parametrize("dtype", TYPES)
def test_group_norm_layouts(layout, dtype):
    _check_norm((2, 64, 9, 11), 8, dtype, "relu", True, layout, seed=5)


@pytest.mark.parametrize("mean", [100.0, 3000.0])
def test_group_norm_mean_far_above_the_spread(mean):
    _check_norm((2, 32, 40, 40), 4, torch.float32, None, False, mean=mean, seed=9)


def test_group_norm_without_weights_and_empty():
    from distributedpytorch_amd import ops
    x = _map((2, 16, 6, 6), torch.float32, 3).requires_grad_(True)
    y = ops.group_norm_act(x, 4)
    want = torch.nn.functional.group_norm(x.double(), 4)
    assert (y.double() - want).abs().max() < 64 * U * 8
    y.sum().backward()
    assert x.grad.abs().max() < 160 * U * 8
    e = torch.zeros(0, 16, 6, 6, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    ops.group_norm_act(e, 4, w, act="relu").sum().backward()
    assert e.grad.shape == e.shape and torch.equal(w.grad, torch.zeros_like(w))


def test_group_norm_keeps_nan_to_its_group():
    from distributedpytorch_amd import ops
    x = _map((2, 16, 6, 6), torch.bfloat16, 4)
    x[1, 5, 2, 3] = float("nan")
    x[0, 12, 0, 0] = float("inf")
    y = ops.group_norm_act(x, 4, act="relu")
    bad = torch.isnan(y).flatten(2).any(2).cpu()
    want = torch.zeros(2, 16, dtype=torch.bool)
    want[1, 4:8] = True
    want[0, 12:16] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("shape", [(2, 64, 17, 17), (1, 64, 129, 129)])
def test_group_norm_repeats_bit_for_bit_and_replays(shape):
    from distributedpytorch_amd import ops
    x, dy = _map(shape, torch.bfloat16, 1).requires_grad_(True), _map(shape, torch.bfloat16, 2)
    w, b = torch.randn(64, device="cuda").requires_grad_(True), torch.randn(64, device="cuda").requires_grad_(True)

    def step():
        y = ops.group_norm_act(x, 8, w, b, act="silu")
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)

    first, second = step(), step()
    assert all(torch.equal(a, c) for a, c in zip(first, second))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(_map(shape, torch.bfloat16, 10 + k))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want)), k


def test_group_norm_refuses_other_types_on_the_gpu():
    from distributedpytorch_amd import ops
    with pytest.raises(TypeError):
        ops.group_norm_act(torch.zeros(1, 8, 2, 2, device="cuda", dtype=torch.float64), 2)
    with pytest.raises(ValueError):
        ops.group_norm_act(torch.zeros(1, 8, 2, 2, device="cuda"), 2, torch.ones(8))


# ------------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count", [1, 7, 8, 9, 2047, 2048, 2049, 100003])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_equals_the_definition(dtype, count, residual):
    from distributedpytorch_amd import ops
    from distributedpytorch_amd.ops.dropout import dropout_keep, dropout_threshold
    g = torch.Generator().manual_seed(count)
    x = torch.randn(count, generator=g).to(dtype).cuda().requires_grad_(True)
    r = torch.randn(count, generator=g).to(dtype).cuda().requires_grad_(True) if residual else None
    dy = torch.randn(count, generator=g).to(dtype).cuda()
    seed = 0x9E3779B97F4A7C15 + count
    y = ops.dropout(x, 0.3, seed=seed, residual=r)
    keep = dropout_keep(count, seed, 0.3).cuda()
    s = 65536.0 / (65536.0 - dropout_threshold(0.3))
    want = torch.where(keep, x.detach().double() * s, 0.0)
    if residual:
        want = want + r.detach().double()
    half = torch.finfo(dtype).eps / 2
    # the factor, its product and the sum are rounded to 32 bits before the type's own rounding
    # below the smallest normal value 2^e the type's step no longer shrinks: it is 2^e eps there (fp16 2^-14 2^-10 = 2^-24)
    # and a rounding is off by up to half of it, which half a step relative to the value does not cover
    sub = torch.finfo(dtype).smallest_normal * half
    tol = half * want.abs() + 3 * U * (want.abs() + 2 * x.detach().double().abs()) + sub
    assert ((y.double() - want).abs() <= tol).all()
    if not residual:
        assert torch.equal(y != 0, keep & (x != 0))
    grads = torch.autograd.grad(y, [x] + ([r] if residual else []), dy)
    want = torch.where(keep, dy.double() * s, 0.0)
    assert ((grads[0].double() - want).abs() <= (half + 3 * U) * want.abs() + sub).all()
    if residual:
        assert torch.equal(grads[1], dy)


@pytest.mark.parametrize("offset", [0, 1, 4])
@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_any_alignment_gives_one_mask(offset, dtype):
    from distributedpytorch_amd import ops
    base = torch.randn(5000, device="cuda").to(dtype)
    part = base[offset:offset + 4321]
    assert torch.equal(ops.dropout(part, 0.5, seed=5), ops.dropout(part.clone(), 0.5, seed=5))
    with ops.backend("torch"):
        plain = ops.dropout(part, 0.5, seed=5)
    assert torch.equal(ops.dropout(part, 0.5, seed=5), plain)


def test_dropout_layouts_follow_memory_order():
    from distributedpytorch_amd import ops
    x = torch.randn(2, 5, 7, 3, device="cuda")
    cl = x.contiguous(memory_format=torch.channels_last).requires_grad_(True)
    y = ops.dropout(cl, 0.5, seed=9)
    assert y.stride() == cl.stride()
    flat = ops.dropout(cl.detach().permute(0, 2, 3, 1).contiguous().view(-1), 0.5, seed=9)
    assert torch.equal(y.detach().permute(0, 2, 3, 1).reshape(-1), flat)
    (dx,) = torch.autograd.grad(y, cl, torch.ones_like(x))              # a gradient in the other layout
    assert torch.equal(dx != 0, y != 0)
    odd = torch.randn(2, 5, 7, 6, device="cuda")[..., ::2]
    assert torch.equal(ops.dropout(odd, 0.5, seed=9), ops.dropout(odd.contiguous(), 0.5, seed=9))


def test_dropout_device_seed_and_replay():
    from distributedpytorch_amd import ops
    seed = torch.tensor([12345], device="cuda")
    x = torch.randn(3, 1001, device="cuda").requires_grad_(True)
    dy = torch.randn(3, 1001, device="cuda")

    def step():
        y = ops.dropout(x, 0.25, seed=seed)
        return (y.detach(),) + torch.autograd.grad(y, (x,), dy)

    assert torch.equal(step()[0], ops.dropout(x.detach(), 0.25, seed=12345))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    seen = []
    for value in (1, -1, 1 << 40):
        seed.fill_(value)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), value
        assert torch.equal(want[0], ops.dropout(x.detach(), 0.25, seed=value))
        seen.append(want[0].clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_dropout_drops_infinities():
    from distributedpytorch_amd import ops
    x = torch.full((4096,), float("inf"), device="cuda", dtype=torch.bfloat16)
    y = ops.dropout(x, 0.5, seed=4)
    assert ((y == 0) | torch.isinf(y)).all() and (y == 0).any()
    assert torch.equal(ops.dropout(x, 1.0, seed=4), torch.zeros_like(x))
    assert ops.dropout(x[:0], 0.5, seed=4).numel() == 0


def test_dropout_refuses_other_types_on_the_gpu():
    from distributedpytorch_amd import ops
    with pytest.raises(TypeError):
        ops.dropout(torch.zeros(8, device="cuda", dtype=torch.float64), 0.5)
    with pytest.raises(ValueError):
        ops.dropout(torch.zeros(8, device="cuda"), 0.5, seed=torch.zeros(1, dtype=torch.int64))
