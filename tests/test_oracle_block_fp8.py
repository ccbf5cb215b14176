"""CPU: the 64-bit oracle of the 8-bit blocks against torch's own e4m3 and e8m0 types, autograd and differences."""
import pytest
import torch

from oracle import block_fp8 as ref


def test_e4m3_rounding_is_the_types():
    g = torch.Generator().manual_seed(0)
    v = torch.cat([torch.randn(4000, generator=g) * 2.0 ** torch.randint(-12, 9, (4000,), generator=g),
                   torch.arange(-448, 449).float() / 2, torch.arange(-64, 65).float() * 2.0 ** -11]).clamp(-448, 448)
    assert torch.equal(ref.round_e4m3(v.double()).float(), v.to(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("rows", [1, 128])
def test_scale_is_the_least_power_of_two_that_fits(rows):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(200, 300, generator=g) * torch.exp2(torch.randint(-20, 20, (200, 1), generator=g).float())
    x[3], x[5, 128:256] = 0.0, 448.0 * 2.0 ** -3
    x[6, 128:256] = 448.0 * 2.0 ** -3 * (1 + 2.0 ** -23)
    q, each, scale = ref.quantize(x, rows)
    assert q.abs().max() <= 448 and scale.shape == (-(-200 // rows), 3)
    full = torch.nn.functional.pad(x.double(), (0, 84, 0, -200 % rows)).reshape(-1, rows, 3, 128).abs().amax((1, 3))
    some = full > 0
    assert bool((full <= 448 * scale).all()) and bool((full > 448 * scale / 2)[some].all())
    assert bool((scale == 1)[~some].all())
    if rows == 1:
        assert scale[5, 1] == 2.0 ** -3 and scale[6, 1] == 2.0 ** -2
    # half a step of each value
    assert bool(((q * each - x.double()).abs() <= ref.half_step(x.double() / each) * each).all())
    assert torch.equal(scale.float().to(torch.float8_e8m0fnu).double(), scale)


def test_what_is_not_finite():
    x = torch.ones(2, 256)
    x[0, 3], x[0, 7], x[1, 200] = float("inf"), float("nan"), float("-inf")
    q, each, scale = ref.quantize(x, 1)
    assert q.isnan().sum() == 3 and bool((scale == 2.0 ** -8).all())  # 1 = 256 * 2^-8
    assert bool((torch.where(q.isnan(), torch.ones_like(q), q * each) == 1).all())


def test_gradients_against_autograd_and_differences():
    g = torch.Generator().manual_seed(2)
    s, b, dy, ds = (torch.randn(3, 24, generator=g, dtype=torch.float64) for _ in range(4))
    s.requires_grad_(True), b.requires_grad_(True)
    y, r = ref.rms_norm(s, 1e-6)
    want, = torch.autograd.grad((y * dy).sum() + (s * ds).sum(), s)
    got = ref.norm_backward(dy, ds, y.detach(), r.detach())
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-12)
    wa, wb = torch.autograd.grad((ref.gate(s, b) * dy).sum(), (s, b))
    ga, gb = ref.gate_backward(dy, s.detach(), b.detach())
    assert torch.allclose(ga, wa, rtol=1e-12, atol=1e-12) and torch.allclose(gb, wb, rtol=1e-12, atol=1e-12)
    h, s0, b0 = 1e-6, s.detach(), b.detach()
    for i in range(0, 24, 5):  # central differences
        e = torch.zeros(24, dtype=torch.float64)
        e[i] = h
        d = ((ref.rms_norm(s0 + e, 1e-6)[0] - ref.rms_norm(s0 - e, 1e-6)[0]) * dy).sum(1) / (2 * h) + ds[:, i]
        assert torch.allclose(d, got[:, i], rtol=1e-6, atol=1e-7)
        d = ((ref.gate(s0 + e, b0) - ref.gate(s0 - e, b0)) * dy).sum(1) / (2 * h)
        assert torch.allclose(d, ga[:, i], rtol=1e-6, atol=1e-7)


def test_embedding_gradient_against_autograd():
    g = torch.Generator().manual_seed(3)
    w = torch.randn(11, 6, generator=g, dtype=torch.float64).requires_grad_(True)
    tokens = torch.randint(0, 11, (4, 9), generator=g)
    dy = torch.randn(4, 9, 6, generator=g, dtype=torch.float64)
    want, = torch.autograd.grad((torch.nn.functional.embedding(tokens, w, padding_idx=2) * 1.5 * dy).sum(), w)
    got, size = ref.embedding_grad(tokens, dy, 11, 1.5, padding_idx=2)
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-12) and bool((size >= got.abs() - 1e-12).all())
    tokens[0, 0], tokens[1, 1] = -1, 11  # outside: no part
    out, _ = ref.embedding_grad(tokens, dy, 11, 1.5, padding_idx=2)
    assert out.shape == (11, 6) and not torch.equal(out, got)
