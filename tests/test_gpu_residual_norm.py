"""Norm behind a block, gate, residual sum and norm in front of the next against 64 bits. GPU only (-m gpu).

Bounds: a sum of squares over n elements is a chain of at most 16 (past 16384 elements: n / 1024) additions a thread and ten over the CTA, of terms that do not cancel: with the division,
the root and the products by factor and gain a norm is off by 2^-24 (chain + 16) of itself, where the sum's own share counts half. The gate is one rounding, scale and sum one each."""
import pytest

pytestmark = pytest.mark.gpu
STEP = 2.0**-24


def normed(x, gain, epsilon):
    f = (x.square().mean(1, keepdim=True) + epsilon).rsqrt()
    return x * f * (1.0 if gain is None else gain.double()), f


def check(ctx, tokens, n, behind=True, gate="none", gain=True, scale=1.0, epsilon=1e-6, offset=0, pad=0, in_place=False, seed=0, size=1.0):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(seed)

    def plane():
        return torch.randn(tokens * (n + pad) + offset, generator=gen, device="cuda")[offset:].view(tokens, n + pad)[:, :n]

    x, delta = plane() * 3 * size, plane() * size
    if offset or pad:
        x, delta = (plane().copy_(a) for a in (x, delta))
    delta_gain, last_gain = 1.0 + 0.2 * torch.randn((2, n), generator=gen, device="cuda")
    delta_gain, last_gain = delta_gain if behind else None, last_gain if gain else None
    shape = {"none": None, "channels": (n,), "tokens": (tokens, 1), "elements": (tokens, n)}[gate]
    g = None if shape is None else torch.randn(shape, generator=gen, device="cuda")
    x0, d0 = x.double(), delta.double()
    y = plane()
    x_out = None if in_place else plane()
    got = ctx.residual_norm(x, delta, last_gain, delta_gain=delta_gain, gate=g, residual_scale=scale, epsilon=epsilon, x_out=x_out, y=y)
    ctx.check()
    assert got is y
    out = x if in_place else x_out
    chain = 26 if n <= 16384 else n / 1024 + 10
    d = d0
    if behind:
        d = normed(d0, delta_gain, epsilon)[0]
    step = d.abs() * STEP * ((chain / 2 + 8) if behind else 0)
    if g is not None:
        d, step = d * g.double(), (step + d.abs() * STEP) * g.double().abs()
    scale = float(torch.tensor(scale))  # (as fp32)
    want = x0 + scale * d
    off_x = abs(scale) * step + STEP * (want.abs() + abs(scale) * d.abs()) + 2.0**-149
    assert ((out.double() - want).abs() <= 1.01 * off_x).all()
    want_y, f = normed(want, last_gain, epsilon)
    weight = f * (1.0 if last_gain is None else last_gain.double().abs())
    # the factor depends on every element of x': sum |x'| off_x / sum x'^2 of it at most
    through = (want.abs() * off_x).sum(1, keepdim=True) / (want.square().sum(1, keepdim=True) + n * epsilon).clamp(min=1e-300)
    assert ((y.double() - want_y).abs() <= 1.01 * (weight * off_x + want_y.abs() * (STEP * (chain / 2 + 8) + through)) + 2.0**-149).all()
    if offset == 0 and pad == 0 and not in_place:
        assert torch.equal(x, x0.float())


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 31, 64, 127, 1000, 1023, 2560, 4096, 5000, 8192, 8193, 11008, 16384, 16385, 40000, 100003])
@pytest.mark.parametrize("behind", [False, True])
def test_widths(rq_ctx, n, behind):
    check(rq_ctx, 3, n, behind, "elements", seed=n)


@pytest.mark.parametrize("gate", ["none", "channels", "tokens", "elements"])
@pytest.mark.parametrize("behind", [False, True])
@pytest.mark.parametrize("gain", [False, True])
@pytest.mark.parametrize("n", [96, 4100])
def test_gates_and_gains(rq_ctx, gate, behind, gain, n):
    check(rq_ctx, 5, n, behind, gate, gain, scale=0.22)


@pytest.mark.parametrize("tokens", [1, 2, 149, 2039])
def test_tokens(rq_ctx, tokens):
    check(rq_ctx, tokens, 2560, True, "channels")


@pytest.mark.parametrize("offset,pad", [(1, 0), (0, 1), (2, 3), (4, 4), (3, 5)])
@pytest.mark.parametrize("n", [63, 4096])
def test_alignment_and_strides(rq_ctx, offset, pad, n):
    check(rq_ctx, 7, n, True, "elements", offset=offset, pad=pad)


@pytest.mark.parametrize("n", [700, 4096, 12000, 20000])
def test_in_place(rq_ctx, n):
    check(rq_ctx, 6, n, True, "tokens", in_place=True)


@pytest.mark.parametrize("scale", [0.0, -1.5, 1e-3, 40.0])
def test_scales(rq_ctx, scale):
    check(rq_ctx, 4, 1024, True, "none", scale=scale)


@pytest.mark.parametrize("size,epsilon", [(1e-12, 1e-6), (1e-12, 0.0), (1e12, 1e-5)])
def test_sizes(rq_ctx, size, epsilon):
    check(rq_ctx, 4, 1024, False, "none", size=size, epsilon=epsilon)


def test_y_may_be_delta_and_zeros_stay(rq_ctx):
    import torch

    for n in (1024, 30000):
        x, delta = torch.randn((3, n), device="cuda"), torch.randn((3, n), device="cuda")
        gain = torch.ones(n, device="cuda")
        want_x = torch.empty_like(x)
        want = rq_ctx.residual_norm(x, delta, gain, delta_gain=gain, x_out=want_x)
        assert torch.equal(rq_ctx.residual_norm(x, delta, gain, delta_gain=gain, y=delta), want) and torch.equal(x, want_x)
    zero = torch.zeros((2, 256), device="cuda")
    assert rq_ctx.residual_norm(zero, zero, torch.ones(256, device="cuda"), delta_gain=torch.ones(256, device="cuda")).eq(0).all()


def test_a_token_by_itself_has_the_same_bits(rq_ctx):
    import torch

    for n in (2560, 2561, 9000):
        x, delta, gain = torch.randn((40, n), device="cuda"), torch.randn((40, n), device="cuda"), torch.randn(n, device="cuda")
        out = torch.empty_like(x)
        y = rq_ctx.residual_norm(x, delta, gain, delta_gain=gain, x_out=out)
        for t in (0, 7, 39):
            one = torch.empty((1, n), device="cuda")
            assert torch.equal(rq_ctx.residual_norm(x[t : t + 1].clone(), delta[t : t + 1].clone(), gain, delta_gain=gain, x_out=one), y[t : t + 1]) and torch.equal(one, out[t : t + 1])


def test_recorded(rq_ctx):
    import torch

    x, delta, gain = torch.randn((4, 2048), device="cuda"), torch.randn((4, 2048), device="cuda"), torch.ones(2048, device="cuda")
    out, y = torch.empty_like(x), torch.empty_like(x)
    rq_ctx.residual_norm(x, delta, gain, x_out=out, y=y)
    torch.cuda.synchronize()
    rq_ctx.residual_norm(x, delta, gain, x_out=out, y=y, stream=rq_ctx.sequence_begin())
    sequence = rq_ctx.sequence_end()
    for _ in range(3):
        x.normal_()
        sequence.run()
        torch.cuda.synchronize()
        want_x = torch.empty_like(x)
        assert torch.equal(rq_ctx.residual_norm(x, delta, gain, x_out=want_x), y) and torch.equal(want_x, out)
    sequence.free()


def test_refusals(rq_ctx):
    import torch

    x, n = torch.zeros((4, 64), device="cuda"), torch.zeros(64, device="cuda")
    for wrong in (dict(delta=x[:, :32]), dict(delta=x.double()), dict(delta=x.cpu()), dict(delta=x.T.contiguous().T), dict(gain=n[:32]), dict(delta_gain=n.double()), dict(gate=torch.zeros(4, device="cuda")),
                  dict(gate=torch.zeros((4, 32), device="cuda")), dict(gate=torch.zeros((64, 4), device="cuda").T), dict(y=x[:2]), dict(x_out=x[:, :32])):
        with pytest.raises(ValueError):
            rq_ctx.residual_norm(**dict(x=x, delta=x, gain=n) | wrong)
    rq_ctx.check()


def test_gates_by_broadcast_and_by_stride(rq_ctx):
    import torch

    x, delta = torch.randn((5, 96), device="cuda"), torch.randn((5, 96), device="cuda")
    gate = torch.randn((5, 200), device="cuda")
    for g in (gate[:, 3:99], gate[:, 7:8], gate[:1, :96].expand(5, 96)):
        out = torch.empty_like(x)
        rq_ctx.residual_norm(x, delta, gate=g, x_out=out)
        want = x.double() + g.double() * delta.double()
        assert ((out.double() - want).abs() <= STEP * (2 * (g.double() * delta.double()).abs() + want.abs())).all()
