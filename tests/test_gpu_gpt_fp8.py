"""GPU: GPTModel with its projections on 8-bit blocks: the operators together, as a training step uses them."""
import copy

import pytest
import torch

from kerneldev_amd.gpt import VOCAB, GPTModel, config5_batch
from kerneldev_amd.span_head import max_spans

pytestmark = pytest.mark.gpu


def _model(dev, projections, dtype=torch.bfloat16, **size):
    torch.manual_seed(3)
    return GPTModel(projections=projections, **size).to(dev).to(dtype)


def _step(model, batch, cotangent):
    tokens, in_span, span_id, is_prefix, correct = batch
    scores, loss = model(tokens, correct_idx=correct, in_span=in_span, span_id=span_id, is_prefix=is_prefix)
    params = dict(model.named_parameters())
    grads = torch.autograd.grad((scores.float() * cotangent).sum(), list(params.values()))
    return scores.detach(), loss.detach(), dict(zip(params, grads))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_step_against_16_bit_projections(dev, dtype):
    """One layer on the same weights.  A value's rounding to e4m3 is off by 2^-4 of it at most and by 2^-4 / sqrt(3) =
    0.036 in root mean square if spread evenly over a step, less over a binade (0.026 on normal values); a product of two such
    operands is off by about 0.037 of itself, the scores and gradients by the root of the sum of the squares of the some
    ten roundings on their way: 0.12.  Twice that is allowed."""
    size = dict(dim=256, n_layers=1, n_heads=4, max_seq_len=1024, mlp_hidden=512)
    batch = [t.to(dev) for t in config5_batch(B=2, L=1024, seed=1)]
    a, b = _model(dev, None, dtype, **size), _model(dev, "fp8_e4m3", dtype, **size)
    assert set(a.state_dict()) == set(b.state_dict())
    cot = torch.randn(2, max_spans(batch[0]), generator=torch.Generator().manual_seed(2)).to(dev) * 1e-2
    sa, _, ga = _step(a, batch, cot)
    sb, _, gb = _step(b, batch, cot)
    assert (sa - sb).norm() <= 0.24 * sa.norm()
    for name, g in ga.items():
        assert gb[name].isfinite().all() and (g.float() - gb[name].float()).norm() <= 0.24 * g.float().norm() + 1e-6, name


def test_training_steps_are_the_same_bits_and_capture(dev):
    """The specified size for one layer: a step twice, and replayed from a graph after the weights moved."""
    size = dict(n_layers=1)
    batch = [t.to(dev) for t in config5_batch(B=2, L=512, seed=4)]
    m = _model(dev, "fp8_e4m3", **size)
    tokens, in_span, span_id, is_prefix, _ = batch
    plan = m.plan(tokens, in_span, span_id, is_prefix)
    params = list(m.parameters())
    cot = torch.randn(2, 512, 768, device=dev).bfloat16()

    def step():
        h = m.hidden(tokens, None, None, None, plan)
        return [h.detach(), *torch.autograd.grad(h, params, cot)]

    def step_without_library_sums():
        """(the positions' gradient is a library sum over the batch, whose capture is not this test's)"""
        h, delta = m.token_emb.weight[:1].detach().expand(2 * 512, 768).reshape(2, 512, 768).contiguous() + cot, None
        for blk in m.blocks:
            h, delta = blk.forward_fp8(h, delta, None, None, None, plan)
        return [h.detach(), delta.detach(), *torch.autograd.grad([h, delta], weights, [cot, cot])]

    weights = [p for n, p in m.named_parameters() if "blocks" in n]
    first, again = step(), step()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    step_without_library_sums()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step_without_library_sums()
    for k in range(3):
        with torch.no_grad():
            for p in params:
                p.mul_(1.1)
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step_without_library_sums(), got)), k


def test_language_model_loss_and_inference(dev):
    m = _model(dev, "fp8_e4m3", dim=128, n_layers=2, n_heads=2, max_seq_len=64, mlp_hidden=256)
    tokens = torch.randint(6, VOCAB, (3, 37), device=dev, generator=torch.Generator(dev).manual_seed(1))
    logits, loss = m(tokens, targets=tokens)
    loss.backward()
    assert logits.shape == (3, 37, VOCAB) and all(p.grad is not None and p.grad.isfinite().all() for p in m.parameters())
    with torch.no_grad():
        assert torch.equal(m(tokens)[0], logits)
        one = m(tokens[:1, :1])[0]  # one token
    assert one.shape == (1, 1, VOCAB) and one.isfinite().all()
    c = copy.deepcopy(m)  # (the default's parameters, under either form)
    d = GPTModel(dim=128, n_layers=2, n_heads=2, max_seq_len=64, mlp_hidden=256).to(dev).bfloat16()
    d.load_state_dict(c.state_dict())
    with pytest.raises(ValueError, match="projections"):
        GPTModel(projections="int8")
