"""GPU: the embedding and its gradient by sorted tokens against the 64-bit oracle.

A lookup is one fp32 product, rounded once: the same bits as torch's.  A gradient's row
is a sum of n fp32 values (bf16 and fp16 are exact in fp32), off by at most n 2^-24 of the sum of their
sizes, times the scale (2^-24), rounded once (2^-8, 2^-11 or 2^-24 of the value, fp16's subnormal spacing 2^-24)."""
import pytest
import torch

import kerneldev_amd as kd
from oracle.block_fp8 import embedding_grad

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = list(U)


@pytest.fixture(params=["native", "python"])
def route(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(kd._lib, "eager", lambda *_: False)
    return request.param


def _case(tokens, vocab, dim, dtype, dev, seed=0):
    g = torch.Generator("cpu").manual_seed(seed)
    w = torch.randn(vocab, dim, generator=g).to(dtype).to(dev).requires_grad_(True)
    dy = torch.randn(*tokens.shape, dim, generator=g).to(dtype).to(dev)
    return tokens.to(dev), w, dy


def _check(tokens, w, dy, scale=1.0, padding_idx=None):
    y = kd.embedding(tokens, w, scale, padding_idx)
    dw, = torch.autograd.grad(y, w, dy)
    inside = (tokens >= 0) & (tokens < w.shape[0])
    want = (w.detach()[tokens.clamp(0, w.shape[0] - 1).long()].float() * torch.tensor(scale, dtype=torch.float32)).to(w.dtype)
    assert torch.equal(y.detach()[inside], want[inside]) and bool(y.detach()[~inside].isnan().all())
    ref, size = embedding_grad(tokens, dy, w.shape[0], scale, padding_idx)
    n = torch.bincount(tokens[inside].reshape(-1), minlength=w.shape[0]).double()[:, None]
    u = U[w.dtype]
    off = (n + 2) * 2.0 ** -24 * size
    err = (dw.double() - ref).abs()
    assert bool((err <= u * (ref.abs() + off) * (1 + 2.0 ** -20) + off + (2.0 ** -25 if w.dtype == torch.float16 else 0)).all())
    return dw


# chunks of 32 positions, sorting workgroups of 4096, passes of up to 11 bits, columns by 256 and by 64
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (1, 5, 8), (31, 2, 7), (32, 2, 4), (33, 3, 256), (64, 1, 260), (65, 262, 768),
                                         (1000, 262, 65), (4096, 2047, 64), (4097, 2048, 12), (5000, 50021, 36),
                                         (70000, 300, 20), (66000, 5000, 9), (300, 1 << 22, 4)])
def test_embedding(dev, n, vocab, dim, dtype):
    g = torch.Generator("cpu").manual_seed(n)
    tokens = (torch.rand(n, generator=g, dtype=torch.float64).pow(3) * vocab).long().clamp(max=vocab - 1)
    tokens, w, dy = _case(tokens, vocab, dim, dtype, dev, n)
    _check(tokens, w, dy, 1.0)
    _check(tokens.int(), w, dy, 27.7, padding_idx=0)


@pytest.mark.parametrize("dtype", TYPES)
def test_runs_of_equal_tokens(dev, dtype):
    """One token throughout (its run takes every chunk), runs that end on a chunk's edge and one place off it, the last token."""
    for tokens in (torch.full((5000,), 3), torch.arange(4096) // 32, (torch.arange(4100) + 1) // 32, (torch.arange(4100) + 31) // 64,
                   torch.cat([torch.full((40,), 261), torch.zeros(33, dtype=torch.int64)]), torch.arange(262).flip(0)):
        t, w, dy = _case(tokens, 262, 300, dtype, dev)
        _check(t, w, dy, 0.5)


def test_shapes_strides_and_the_outside(dev, route):
    g = torch.Generator("cpu").manual_seed(1)
    tokens = torch.randint(0, 50, (6, 37, 2), generator=g)
    t, w, dy = _case(tokens, 50, 24, torch.bfloat16, dev)
    _check(t, w, dy)
    _check(t[..., 1], w, dy[..., 1, :])  # strided tokens and gradient
    _check(t.transpose(0, 1), w, dy.transpose(0, 1))
    bad = t.clone()
    bad[0, 0, 0], bad[1, 2, 1], bad[3, 3, 0] = -1, 50, 1 << 40  # outside: NaN, and no part in the gradient
    _check(bad, w, dy, padding_idx=7)
    neg = kd.embedding(t, w, padding_idx=-1)
    dw, = torch.autograd.grad(neg, w, dy)
    assert not dw[49].any() and dw[48].any()
    empty = kd.embedding(t[:0], w)
    assert empty.shape == (0, 37, 2, 24) and not torch.autograd.grad(empty.sum(), w)[0].any()
    one = kd.embedding(t[0, 0, 0], w)  # a token without dimensions
    assert torch.equal(one, w[t[0, 0, 0]])
    odd = torch.randn(51 * 24 + 1, device=dev).bfloat16()[1:].view(51, 24).requires_grad_(True)  # a base of 2 bytes
    _check(t, odd, dy)
    y = kd.embedding(t, w)
    assert ("CppFunction" in type(y.grad_fn).__name__) == (route == "native")
    g, = torch.autograd.grad((y * w[0]).float().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|no autograd formula"):
        g.float().sum().backward()
    s, = torch.autograd.grad(y.sum(), w)  # an expanded gradient
    assert torch.equal(s, torch.autograd.grad(kd.embedding(t, w), w, torch.ones_like(y))[0])


def test_not_a_number_stays_in_its_row(dev):
    tokens = torch.arange(300) % 10
    t, w, dy = _case(tokens, 12, 40, torch.bfloat16, dev)
    dy[13, 5] = float("nan")
    dw, = torch.autograd.grad(kd.embedding(t, w), w, dy)
    bad = torch.zeros(12, 40, dtype=torch.bool, device=dev)
    bad[3, 5] = True
    assert torch.equal(dw.isnan(), bad)


def test_same_bits_every_time_captured_and_on_another_stream(dev):
    g = torch.Generator("cpu").manual_seed(2)
    t, w, dy = _case(torch.randint(0, 262, (8, 2048), generator=g), 262, 768, torch.bfloat16, dev)

    def step():
        y = kd.embedding(t, w, 2.0)
        return y.detach(), torch.autograd.grad(y, w, dy)[0]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        t.copy_((t * 7 + k) % 262)
        dy.mul_(0.5 + k)
        graph.replay()
        got = [x.clone() for x in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step(), got)), k


def test_compiled(dev):
    t, w, dy = _case(torch.arange(500) % 262, 262, 64, torch.bfloat16, dev)
    y = torch.compile(lambda t, w: kd.embedding(t, w, 3.0), fullgraph=True)(t, w)
    z = kd.embedding(t, w, 3.0)
    assert torch.equal(y, z) and torch.equal(torch.autograd.grad(y, w, dy)[0], torch.autograd.grad(z, w, dy)[0])
    torch.library.opcheck(torch.ops.kdattn.embed, (t, w.detach(), 2.0), test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.kdattn.embed_grad, (t, dy, 262, 2.0, -1), test_utils=("test_schema", "test_faketensor"))


def test_offsets_past_32_bits(dev):
    """A table of 2^32 values and a gradient alike: the last rows of both."""
    vocab, dim, n = (1 << 22) + 5, 1032, 300
    w = torch.zeros(vocab, dim, device=dev, dtype=torch.bfloat16)
    tokens = torch.cat([torch.arange(vocab - 150, vocab), torch.arange(100), torch.full((50,), vocab - 1)]).to(dev)
    w[tokens] = torch.randn(n, dim, device=dev).bfloat16()
    w.requires_grad_(True)
    dy = torch.randn(n, dim, device=dev).bfloat16()
    y = kd.embedding(tokens, w)
    assert torch.equal(y.detach(), w.detach()[tokens])
    dw, = torch.autograd.grad(y, w, dy)
    ref = torch.zeros(150, dim, device=dev, dtype=torch.float64).index_add_(0, torch.cat([torch.arange(150), torch.full((50,), 149)]).to(dev),
                                                                            torch.cat([dy[:150], dy[250:]]).double())
    assert bool(((dw[-150:].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -16).all())
    assert torch.equal(dw[:100], dy[150:250]) and not dw[100:-150].any()


def test_more_chunks_than_one_launch_takes(dev):
    """Some 2^22 chunks of sorted positions; whole numbers, whose sums fp32 holds."""
    n, vocab = (1 << 26) + (1 << 22) + 5, 300
    g = torch.Generator(dev).manual_seed(1)
    tokens = torch.randint(0, vocab, (n,), device=dev, generator=g, dtype=torch.int32)
    dy = torch.randint(0, 3, (n, 1), device=dev, generator=g).float()
    w = torch.zeros(vocab, 1, device=dev, requires_grad=True)
    dw, = torch.autograd.grad(kd.embedding(tokens, w), w, dy)
    assert torch.equal(dw[:, 0].double(), torch.bincount(tokens, weights=dy[:, 0].double(), minlength=vocab))
