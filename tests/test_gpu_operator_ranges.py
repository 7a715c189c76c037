"""Group norm, cross attention and dropout at the ends of what they accept: buffers past 2^31 elements, strides past what
32-bit offsets reach, other streams, rows of NaN, seeds that change, second derivatives, lengths that are refused."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from test_gpu_cross_attention import _check, _inputs  # noqa: E402
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = 2.0 ** -8                  # bf16


def _rand(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def test_group_norm_past_31_bits_of_elements():
    """33 images of 64 x 1024 x 1024: 2^31 + 2^26 elements; the first and the last image against 64 bits.

    A thread sums 1,024 of its channel's positions, and joins come after: N = 1,100 roundings u.  Statistics: xhat is off by
    N u (1 + |xhat|).  Gradient: dx = rstd (w dz - m1 - xhat m2) with means off by N u of their magnitudes' means, all of it
    twice for rstd.  Where z lies within its error of ReLU's border either side is right, and moves the means by as much."""
    from distributedpytorch_amd import ops
    n, c, h, groups, N = 33, 64, 1024, 8, 1100
    x = torch.empty((n, c, h, h), dtype=torch.bfloat16, device="cuda", memory_format=torch.channels_last)
    for i in range(n):
        x[i] = _rand(c, h, h, seed=i)
    w, b = _rand(c, seed=100, dtype=torch.float32), _rand(c, seed=101, dtype=torch.float32)
    leaf = x.requires_grad_(True)
    y = ops.group_norm_act(leaf, groups, w, b, act="relu")
    (dx,) = torch.autograd.grad(y, leaf, x.detach())                  # (x again as the gradient: no third buffer)
    for i in (0, n - 1):
        xi = x.detach()[i:i + 1].double()
        by_group = lambda t: t.reshape(groups, -1).mean(1, keepdim=True).expand(groups, t.numel() // groups).reshape(t.shape)  # noqa: E731
        mean = by_group(xi)
        rstd = 1 / torch.sqrt(by_group((xi - mean) ** 2) + 1e-5)
        xhat = (xi - mean) * rstd
        ww = w.double().view(1, c, 1, 1)
        z = xhat * ww + b.double().view(1, c, 1, 1)
        ez = N * U * (1 + xhat.abs()) * ww.abs() + 8 * U * (1 + z.abs())
        want = z.clamp_min(0)
        assert ((y.detach()[i:i + 1].double() - want).abs() <= ez + HALF * want).all(), i
        t = xi * ww * (z > 0)
        m1, m2 = by_group(t), by_group(t * xhat)
        want = rstd * (t - m1 - xhat * m2)
        unsure = z.abs() <= ez
        flip = unsure * (xi * ww).abs()
        tol = 2 * N * U * rstd * (t.abs() + by_group(t.abs()) + xhat.abs() * by_group((t * xhat).abs())
                                  + (1 + xhat.abs()) * m2.abs())
        tol += rstd * (by_group(flip) + xhat.abs() * by_group(flip * xhat.abs())) + HALF * want.abs()
        assert (((dx[i:i + 1].double() - want).abs() <= tol) | unsure).all(), i


def test_dropout_past_31_bits_of_elements():
    from distributedpytorch_amd import ops
    from distributedpytorch_amd.ops.dropout import dropout_keep
    count, p = (1 << 31) + 4093, 0.25
    x = torch.ones(count, dtype=torch.float16, device="cuda")
    y = ops.dropout(x, p, seed=77)
    keep = y != 0
    del x, y
    first = dropout_keep(4096, 77, p, "cuda")
    assert torch.equal(keep[:4096], first)
    # the tail's blocks, from the generator's definition at their own counters
    blocks = (count + 7) // 8
    want = dropout_keep(count, 77, p, "cuda")[(blocks - 600) * 8:]
    assert torch.equal(keep[(blocks - 600) * 8:], want)
    # binomial: six standard deviations of 2^31 draws
    assert abs(float(keep.sum(dtype=torch.int64)) / count - (1 - p)) < 6 * (p * (1 - p) / count) ** 0.5


def _attention(q, k, v, dout, **kw):
    from distributedpytorch_amd import ops
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = ops.cross_attention(*leaves, **kw)
    return (out.detach(), *torch.autograd.grad(out, leaves, dout))


def test_cross_attention_over_keys_past_31_bits_of_elements():
    """2^24 + 70 keys of 128: a query that points at one key finds that key's value, wherever it lies."""
    lk, d = (1 << 24) + 70, 128
    k, v = (torch.empty(1, lk, 1, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for t, seed in ((k, 0), (v, 1)):
        for a in range(0, lk, 1 << 22):
            t[:, a:a + (1 << 22)] = _rand(1, min(1 << 22, lk - a), 1, d, seed=seed + a)
    at = torch.tensor([0, 63, 1 << 20, (1 << 24) - 1, 1 << 24, lk - 1], device="cuda")
    q = k[:, at].contiguous()
    dout = _rand(1, len(at), 1, d, seed=9)
    # scores: scale |k|^2 ~ 4 x 128 at its own key, normal of spread 4 sqrt(128) = 45 elsewhere (the largest of 1.7e7 lies
    # near 5.5 spreads): nothing else has a probability above exp(-150)
    got = _attention(q, k, v, dout, scale=4.0)
    assert torch.equal(got[0], v[:, at])
    assert torch.equal(got[3][:, at], dout)                            # dv = dout where P = 1, and zeros elsewhere
    assert int((got[3] != 0).any(dim=-1).sum()) == len(at)
    assert not got[2].isnan().any() and not got[1].isnan().any()


@pytest.mark.parametrize("beyond", [False, True])
@pytest.mark.parametrize("axis", ["keys", "rows"])
def test_cross_attention_strides_around_32_bit_offsets(axis, beyond):
    """Positions 2^23 - 8 elements apart are the last that 32-bit offsets inside a tile serve, 2^23 go another way: both
    must compute what dense tensors of the same values give, bit for bit."""
    step = (1 << 23) if beyond else (1 << 23) - 8
    lq, lk, d = (5, 70, 64) if axis == "keys" else (70, 5, 64)
    n = max(lq, lk)
    buf = torch.zeros((n - 1) * step + 3 * d, dtype=torch.bfloat16, device="cuda")
    far = buf.as_strided((1, n, 2, d), (0, step, d, 1))
    far.copy_(_rand(1, n, 2, d, seed=1))
    q = far if axis == "rows" else _rand(1, lq, 2, d, seed=2)
    k = far if axis == "keys" else _rand(1, lk, 2, d, seed=3)
    v, dout = _rand(1, lk, 2, d, seed=4), _rand(1, lq, 2, d, seed=5)
    for got, want in zip(_attention(q, k, v, dout), _attention(q.contiguous(), k.contiguous(), v, dout)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("share,heads", [(3, 2), (7, 1), (64, 1), (128, 1)])
def test_cross_attention_any_share_of_a_head(share, heads):
    q, k, v, dout = _inputs(2, 37, 90, heads * share, heads, 32, torch.bfloat16, seed=share)
    _check(q, k, v, dout)


def test_cross_attention_nan_row_reaches_every_gradient_it_is_part_of():
    q, k, v, dout = (_rand(2, n, 2, 64, seed=i) for i, n in enumerate((40, 90, 90, 40)))
    q[1, 7, 1, 3] = float("nan")
    out, dq, dk, dv = _attention(q, k, v, dout)
    assert out[1, 7, 1].isnan().all() and dq[1, 7, 1].isnan().all()
    assert dk[1, :, 1].isnan().all() and dv[1, :, 1].isnan().all()
    for t in (out, dq, dk, dv):
        keep = torch.ones_like(t, dtype=torch.bool)
        keep[1, :, 1] = False
        assert not t[keep].isnan().any()
    keep = torch.arange(40, device="cuda") != 7
    assert not out[1, keep, 1].isnan().any() and not dq[1, keep, 1].isnan().any()


def _all_three(x, w, b, q, k, v):
    from distributedpytorch_amd import ops
    y = ops.group_norm_act(x, 4, w, b, act="silu")
    y = ops.dropout(y, 0.3, seed=5)
    o = ops.cross_attention(q, k, v)
    return y, o


def test_two_streams_at_once_compute_what_one_does():
    sets = []
    for s in range(2):
        x = _rand(2, 32, 70, 50, seed=s).contiguous(memory_format=torch.channels_last).requires_grad_(True)
        w, b = _rand(32, seed=s + 2, dtype=torch.float32), _rand(32, seed=s + 4, dtype=torch.float32)
        q, k, v = (_rand(2, n, 2, 64, seed=s + n).requires_grad_(True) for n in (300, 2000, 2000))
        sets.append((x, w, b, q, k, v))
    def run(a):
        y, o = _all_three(*a)
        return [y, o, *torch.autograd.grad((y, o), (a[0], *a[3:]), (y.detach(), o.detach()))]
    want = [run(a) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for again in got[i]:
            for a, b in zip(again, want[i]):
                assert torch.equal(a, b)


def test_second_derivatives_are_refused():
    from distributedpytorch_amd import ops
    x = _rand(1, 8, 4, 4).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    q = _rand(1, 5, 1, 16).requires_grad_(True)
    for y, leaf in ((ops.group_norm_act(x, 2), x), (ops.dropout(x, 0.5, seed=1), x), (ops.cross_attention(q, q, q), q)):
        with pytest.raises(NotImplementedError, match="gradients of gradients"):
            torch.autograd.grad(y.float().sum(), leaf, create_graph=True)
        torch.cuda.synchronize()


def test_a_seed_that_changed_before_backward_is_refused():
    from distributedpytorch_amd import ops
    x = _rand(64).requires_grad_(True)
    seed = torch.tensor([3], device="cuda")
    y = ops.dropout(x, 0.5, seed=seed)
    seed.fill_(4)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, torch.ones_like(y))


def test_lengths_past_the_kernels_are_refused():
    from distributedpytorch_amd import ops
    one = torch.zeros(1, 1, 1, 8, dtype=torch.bfloat16, device="cuda")
    far = one.expand(1, (1 << 32) + 64, 1, 8)                          # (no memory behind it)
    with pytest.raises(NotImplementedError, match="up to"):
        ops.cross_attention(one, far, far)
    with pytest.raises(NotImplementedError, match="up to"):
        ops.cross_attention(far, one, one)


def test_one_tensor_as_every_operand():
    from distributedpytorch_amd import ops
    q = _rand(2, 70, 2, 64, seed=1).requires_grad_(True)
    out = ops.cross_attention(q, q, q)
    (together,) = torch.autograd.grad(out, q, q.detach())
    apart = _attention(q.detach(), q.detach(), q.detach(), q.detach())
    assert torch.equal(out, apart[0])
    # three bf16 gradients added in an order of autograd's: two roundings of partial sums
    want = sum(t.double() for t in apart[1:])
    tol = 2 * HALF * sum(t.double().abs() for t in apart[1:])
    assert ((together.double() - want).abs() <= tol).all()
    x = _rand(2, 32, 9, 9, seed=2).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    y = ops.group_norm_act(x, 4, act="relu", residual=x)
    a, r = x.detach().requires_grad_(True), x.detach().clone().requires_grad_(True)
    ya = ops.group_norm_act(a, 4, act="relu", residual=r)
    assert torch.equal(y, ya)
    (gx,) = torch.autograd.grad(y, x, x.detach())
    ga, gr = torch.autograd.grad(ya, (a, r), x.detach())
    assert torch.equal(gx, ga + gr)


def _calls():
    """(inputs by name, call) of each operator, every input wanting a gradient."""
    from distributedpytorch_amd import ops
    x, r = (_rand(2, 24, 9, 11, seed=s).contiguous(memory_format=torch.channels_last) for s in (1, 2))
    w, b = _rand(24, seed=3, dtype=torch.float32), _rand(24, seed=4, dtype=torch.bfloat16)
    q, k, v = _rand(2, 70, 4, 40, seed=5), _rand(2, 90, 2, 40, seed=6), _rand(2, 90, 2, 40, seed=7)
    return {
        "norm": (dict(x=x, weight=w, bias=b, residual=r), lambda x, weight, bias, residual:
                 ops.group_norm_act(x, 6, weight, bias, act="silu", residual=residual)),
        "norm without act": (dict(x=x, weight=w, bias=b, residual=r), lambda x, weight, bias, residual:
                             ops.group_norm_act(x, 6, weight, bias, residual=residual)),
        "dropout": (dict(x=x, residual=r), lambda x, residual: ops.dropout(x, 0.4, seed=9, residual=residual)),
        "attention": (dict(q=q, k=k, v=v), ops.cross_attention),
    }


@pytest.mark.parametrize("name", ["norm", "norm without act", "dropout", "attention"])
def test_each_input_alone_gets_the_gradient_it_gets_among_all(name):
    inputs, call = _calls()[name]
    leaves = {n: t.clone().requires_grad_(True) for n, t in inputs.items()}
    y = call(**leaves)
    dy = _rand(*y.shape, seed=11)
    want = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy, retain_graph=True)))
    again = torch.autograd.grad(y, list(leaves.values()), dy)               # the same graph a second time
    for n, g in zip(leaves, again):
        assert torch.equal(g, want[n]) and g.dtype == leaves[n].dtype and g.shape == leaves[n].shape
    for n in inputs:
        one = {m: t.clone().requires_grad_(m == n) for m, t in inputs.items()}
        out = call(**one)
        assert torch.equal(out, y)
        (g,) = torch.autograd.grad(out, one[n], dy)
        assert torch.equal(g, want[n])
    with torch.inference_mode():
        assert torch.equal(call(**inputs), y)


@pytest.mark.parametrize("name", ["norm", "dropout", "attention"])
def test_checkpointed_calls_give_the_same_gradients(name):
    from torch.utils.checkpoint import checkpoint
    inputs, call = _calls()[name]
    leaves = {n: t.clone().requires_grad_(True) for n, t in inputs.items()}
    y = call(**leaves)
    dy = _rand(*y.shape, seed=11)
    want = torch.autograd.grad(y, list(leaves.values()), dy)
    again = checkpoint(lambda *a: call(*a), *leaves.values(), use_reentrant=False)
    assert torch.equal(again, y)
    for g, w in zip(torch.autograd.grad(again, list(leaves.values()), dy), want):
        assert torch.equal(g, w)


@pytest.mark.parametrize("shape", [(1, 3, 20001, 1, 1, 64), (1, 1, 16641, 4, 1, 128), (2, 5, 2500, 2, 2, 40)])
@pytest.mark.parametrize("ragged", [False, True])
def test_cross_attention_of_few_rows_in_many_parts(shape, ragged):
    """Up to 157 parts, joined by four waves; ragged: most parts hold no key."""
    b, lk = shape[0], shape[2]
    lens = torch.tensor([lk // 3, 0][:b], dtype=torch.int64, device="cuda") if ragged else None
    mask = torch.arange(lk, device="cuda").remainder(130).ge(65).expand(b, lk) if ragged else None
    _check(*_inputs(*shape, torch.bfloat16, seed=lk), lens=lens, mask=mask)
