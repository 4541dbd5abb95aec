"""Muon on 16-bit parameters, its state across a checkpoint, and steps that
refuse before they change anything."""

import copy

import pytest
import torch

from chunkedgreedy_amd import nn

pytestmark = pytest.mark.gpu

R = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def grads(shape, dtype, size, seed, count):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [(size * torch.randn(shape, device="cuda", generator=gen)).to(dtype)
            for _ in range(count)]


def weight(shape, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=gen).to(dtype).requires_grad_()


# The momentum is a sum of n gradients in 32 bits, each rounded once and
# multiplied by a factor below 1 (n + 1 roundings of at most the sum of
# magnitudes); the parameter is rounded to its type once a step, of a value
# that 32-bit sums of three terms give (off by 2^-22 of them).
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [1e-3, 6000.0])
def test_momentum_is_held_in_32_bits(sporder, dtype, size):
    w = weight((60, 40), dtype)
    opt = nn.Muon([w], lr=0.05, momentum=0.95)
    m = torch.zeros(60, 40, device="cuda", dtype=torch.float64)
    total = torch.zeros_like(m)
    # Small steps beside a large first one: 2^-8 of it would be lost in 16 bits.
    for k, g in enumerate(grads((60, 40), dtype, size, 1, 40)):
        w.grad = g if k == 0 or size > 1.0 else g * 2.0**-7
        before = w.detach().float().clone()
        m = 0.95 * m + w.grad.double()
        total = 0.95 * total + w.grad.double().abs()
        opt.step()
        held = opt.state[w]["momentum"]
        assert held.dtype == torch.float32
        assert ((held.double() - m).abs() <= (k + 2) * 2.0**-23 * total).all()
        update = sporder.newton_schulz(w.grad.float() + 0.95 * held)
        want = before - 0.05 * (60 / 40) ** 0.5 * update
        off = (w.detach().float() - want).abs()
        # newton_schulz of a lookahead rounded differently: 1e-4 of the step at most.
        assert (off <= R[dtype] * want.abs() + 1e-4 * 0.05).all()
    assert w.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_checkpoint_keeps_the_momentum(sporder, dtype):
    first, second = weight((30, 50), dtype, 2), weight((4, 20, 20), dtype, 3)
    opt = nn.Muon([{"params": [first], "lr": 0.1}, {"params": [second]}])
    for g, h in zip(grads((30, 50), dtype, 1.0, 4, 3), grads((4, 20, 20), dtype, 1.0, 5, 3)):
        first.grad, second.grad = g, h
        opt.step()
    saved = copy.deepcopy(opt.state_dict())
    a, b = first.detach().clone().requires_grad_(), second.detach().clone().requires_grad_()
    again = nn.Muon([{"params": [a]}, {"params": [b]}])
    again.load_state_dict(saved)
    for p, q in ((first, a), (second, b)):
        assert again.state[q]["momentum"].dtype == torch.float32
        assert torch.equal(again.state[q]["momentum"], opt.state[p]["momentum"])
        p.grad = grads(p.shape, dtype, 1.0, 6, 1)[0]
        q.grad = p.grad.clone()
    opt.step()
    again.step()
    assert torch.equal(first, a) and torch.equal(second, b)


def bad_parameters():
    sparse = torch.zeros(4, 4, device="cuda").requires_grad_()
    sparse.grad = torch.sparse_coo_tensor([[0], [1]], [1.0], (4, 4)).cuda()
    plain = [torch.zeros(4, 4), torch.zeros(4, 4, device="cuda", dtype=torch.float64),
             torch.zeros(65537, 1, device="cuda"), torch.zeros(32769, 1, 1, device="cuda")]
    for p in plain:
        p.requires_grad_().grad = torch.zeros_like(p)
    return plain + [sparse]


def test_a_step_that_refuses_changes_nothing(sporder):
    for bad in bad_parameters():
        w = weight((5, 6), torch.float32)
        w.grad = torch.ones_like(w)
        before, rest = w.detach().clone(), bad.detach().clone()
        opt = nn.Muon([w, bad])
        with pytest.raises((TypeError, ValueError)):
            opt.step()
        assert torch.equal(w, before) and torch.equal(bad, rest) and not opt.state
        bad.grad = None
        opt.step()
        assert not torch.equal(w, before)
    w = weight((5, 6), torch.float32)
    w.grad = torch.ones_like(w)
    other = weight((6, 5), torch.float32)
    other.grad = torch.ones_like(other)
    before = w.detach().clone()
    opt = nn.Muon([{"params": [w]}, {"params": [other]}])
    opt.param_groups[1]["steps"] = 0
    with pytest.raises(ValueError):
        opt.step()
    opt.param_groups[1]["steps"] = 5
    opt.add_param_group({"params": [weight((3,), torch.float32)]})
    opt.param_groups[2]["params"][0].grad = torch.ones(3, device="cuda")
    with pytest.raises(ValueError):
        opt.step()
    assert torch.equal(w, before) and not opt.state


def test_parameters_without_elements_are_passed_over(sporder):
    w = weight((5, 6), torch.float32)
    empty = [torch.zeros(s, device="cuda", requires_grad=True) for s in ((0, 5), (3, 0), (0, 2, 2))]
    for p in [w, *empty]:
        p.grad = torch.ones_like(p)
    before = w.detach().clone()
    nn.Muon([empty[0], w, *empty[1:]]).step()
    assert not torch.equal(w, before)

