"""The training operators in a model (chunkedgreedy_amd.nn and the GCN's
options), against the same model of torch operations.

- Gradients through autograd equal torch's: within 1e-5 of the sum of
  magnitudes, 32-bit sums of a few hundred terms on both sides.
- Training with every option follows the torch model's losses: both differ
  from exact training by 32-bit rounding only, some 1e-6 per epoch, over 6
  epochs; 1e-4 relative.
- With learned node vectors the loss does not depend on the row order.
"""

import numpy as np
import pytest
import torch

from chunkedgreedy_amd import e2e_gcn, nn, synth

pytestmark = pytest.mark.gpu


def close(got, want, scale):
    assert got.shape == want.shape and got.dtype == want.dtype
    assert ((got - want).abs() <= 1e-5 * scale + 1e-12).all()


def test_embedding_autograd(sporder):
    g = torch.Generator(device="cuda").manual_seed(1)
    table = torch.randn(50, 24, device="cuda", generator=g, requires_grad=True)
    tok = torch.randint(0, 50, (6, 40), device="cuda", generator=g)
    up = torch.randn(6, 40, 24, device="cuda", generator=g)
    (nn.embedding(table, tok, scale=2.0, padding_idx=3) * up).sum().backward()
    mine, table.grad = table.grad, None
    (table[tok] * 2.0 * up * (tok != 3)[..., None]).sum().backward()
    close(mine, table.grad, table.grad.abs().max())


@pytest.mark.parametrize("given", ["both", "weight", "bias", "none"])
def test_layer_norm_autograd(sporder, given):
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(5, 60, 36, device="cuda", generator=g, requires_grad=True)
    up = torch.randn(5, 60, 36, device="cuda", generator=g)
    w = torch.randn(36, device="cuda", generator=g, requires_grad=True)
    b = torch.randn(36, device="cuda", generator=g, requires_grad=True)
    w_in = w if given in ("both", "weight") else None
    b_in = b if given in ("both", "bias") else None
    (nn.layer_norm(x, w_in, b_in, eps=1e-3) * up).sum().backward()
    leaves = [t for t in (x, w_in, b_in) if t is not None]
    mine = [t.grad for t in leaves]
    for t in leaves:
        t.grad = None
    c = x - x.mean(-1, keepdim=True)
    h = c * ((c * c).mean(-1, keepdim=True) + 1e-3).rsqrt()
    ((h * (1.0 if w_in is None else w_in) + (0.0 if b_in is None else b_in)) * up).sum().backward()
    for got, t in zip(mine, leaves):
        close(got, t.grad, up.abs().sum((0, 1)).max() if t is not x else t.grad.abs().max() * 10)


def test_muon_step(sporder):
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randn(70, 30, device="cuda", generator=g, requires_grad=True)
    start = w.detach().clone()
    opt = nn.Muon([w], lr=0.1, momentum=0.9)
    m, want = torch.zeros_like(start), start.clone()
    for _ in range(3):
        w.grad = torch.randn(70, 30, device="cuda", generator=g)
        m = 0.9 * m + w.grad
        want -= 0.1 * (70 / 30) ** 0.5 * sporder.newton_schulz(w.grad + 0.9 * m)
        opt.step()
    assert (w.detach() - want).abs().max() < 1e-5 and not torch.equal(w.detach(), start)
    with pytest.raises(ValueError):
        nn.Muon([torch.zeros(3, device="cuda", requires_grad=True)])


def torch_training(ptr, ind, features, hidden, classes, epochs, seed):
    """The model of e2e_gcn with --embed --layer-norm --muon in plain torch."""
    dev = "cuda"
    n = ptr.shape[0] - 1
    g = torch.Generator(device=dev).manual_seed(seed)
    X = torch.randn(n, features, device=dev, generator=g)
    y = torch.randint(0, classes, (n,), device=dev, generator=g)
    deg = torch.from_numpy(np.diff(ptr).astype(np.float32)).to(dev).clamp_min(1.0)
    rows = torch.repeat_interleave(torch.arange(n), torch.from_numpy(np.diff(ptr).astype(np.int64)))
    A = torch.zeros(n, n).index_put_((rows, torch.from_numpy(ind).long()), torch.ones(ind.shape[0]),
                                     accumulate=True).to(dev)
    A = deg.rsqrt()[:, None] * A * deg.rsqrt()[None, :]
    torch.manual_seed(seed)
    W1 = torch.nn.Linear(features, hidden).to(dev)
    W2 = torch.nn.Linear(hidden, classes).to(dev)
    table = X.clone().requires_grad_()
    scale = torch.ones(hidden, device=dev, requires_grad=True)
    shift = torch.zeros(hidden, device=dev, requires_grad=True)
    adam = torch.optim.Adam([W1.bias, W2.bias, scale, shift, table], lr=0.01)
    momenta = [torch.zeros_like(W1.weight), torch.zeros_like(W2.weight)]
    losses = []
    for _ in range(epochs):
        for p in (W1.weight, W2.weight):
            p.grad = None
        adam.zero_grad()
        h = torch.nn.functional.layer_norm(A @ W1(table), (hidden,), scale, shift)
        z = W2(A @ torch.relu(h))
        loss = torch.nn.functional.cross_entropy(z, y)
        loss.backward()
        adam.step()
        with torch.no_grad():
            for p, m in zip((W1.weight, W2.weight), momenta):
                m.mul_(0.95).add_(p.grad)
                x = (p.grad + 0.95 * m).double()
                tall = x.shape[0] > x.shape[1]
                x = x.t().contiguous() if tall else x
                x = x / (x.norm() + 1e-7)
                for _ in range(5):
                    a = x @ x.t().contiguous()
                    x = 3.4445 * x + (-4.7750 * a + 2.0315 * (a @ a)) @ x
                x = (x.t() if tall else x).float()
                p.add_(x, alpha=-0.02 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5)
        losses.append(float(loss.detach()))
    return losses


def test_gcn_with_every_option_follows_torch(sporder):
    ptr, ind, _ = synth.chung_lu(1500, 2.1, 12, 61)
    print("[nn] n=1500 epochs=6", flush=True)
    dev = torch.device("cuda")
    n = ptr.shape[0] - 1
    g = torch.Generator(device=dev).manual_seed(7)
    X = torch.randn(n, 20, device=dev, generator=g)
    y = torch.randint(0, 9, (n,), device=dev, generator=g)
    r = e2e_gcn.train(torch.from_numpy(ptr).to(dev), torch.from_numpy(ind).to(dev), X, y, hidden=24,
                      classes=9, epochs=4, warmup=2, seed=7, norm=True, muon=True,
                      tokens=torch.arange(n, dtype=torch.int32, device=dev))
    want = torch_training(ptr, ind, 20, 24, 9, 6, 7)
    assert r["losses"] == pytest.approx(want, rel=1e-4)
    assert r["losses"][-1] < r["losses"][0]


def test_gcn_options_do_not_depend_on_the_order(sporder):
    ptr, ind, _ = synth.chung_lu(3000, 2.1, 12, 62)
    print("[nn] n=3000 epochs=4", flush=True)
    rows = e2e_gcn.run(ptr, ind, features=24, hidden=32, classes=7, epochs=4,
                       orders=("ORIGIN", "sporder-csg"), seed=3, embed=True, norm=True, muon=True)
    assert all(r["embed"] and r["layer_norm"] and r["muon"] for r in rows)
    assert rows[1]["final_loss"] == pytest.approx(rows[0]["final_loss"], rel=1e-4)
