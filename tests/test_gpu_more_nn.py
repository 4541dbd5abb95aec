"""Dropout, the norms around a block and the linear cross entropy together, in
the GCN's options and in a small stack of blocks, against the same model of
torch operations.

- The stack's gradients equal the formulas' in 64 bits.  Its 32-bit values pass
  through some ten operations of 2^-24 each and sums of at most a few hundred
  terms (2^-24 times the sum of magnitudes per partial sum); the products of the
  loss have operands of 22 bits (2^-21 a term).  Norms divide by values near 1.
  1e-4 of the largest gradient holds ten times what that adds up to.
- Bfloat16 rounds each element by at most 2^-8 of itself.  Some 24 roundings lie
  between the inputs and the first parameter's gradient, of independent signs and
  sizes: 24^1/2 2^-8 / 3^1/2 = 0.011 in norm; a single row has few terms to
  average, so half of the worst case, 12 2^-8 = 0.047, is allowed.
- A captured step's replays equal the eager steps bit for bit: the same kernels
  in the same order, with the masks of the next call each.
- Training with every option follows the torch model's losses: both differ from
  exact training by 32-bit rounding only, some 1e-6 per epoch, over 6 epochs;
  1e-4 relative.
"""

import numpy as np
import pytest
import torch

from chunkedgreedy_amd import e2e_gcn, nn, synth

pytestmark = pytest.mark.gpu


def make(kind, rows, dim, classes, blocks, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, dim, generator=g)
    y = torch.randint(0, classes, (rows,), generator=g)
    y[1::5] = -100
    params = []
    for _ in range(blocks):
        params.append(torch.randn(dim, dim, generator=g) / dim**0.5)
        params += [1.0 + 0.1 * torch.randn(dim, generator=g) for _ in range(2)]
    params.append(torch.randn(classes, dim, generator=g) / dim**0.5)
    params.append(0.1 * torch.randn(classes, generator=g))
    cuda = [p.to(kind).cuda().requires_grad_() for p in params]
    return x.to(kind).cuda(), y.cuda(), cuda


def forward(x, y, params, drop):
    """Blocks of a product, dropout and the norms, and the loss."""
    stream = h = x
    *layers, head, bias = params
    for k in range(0, len(layers), 3):
        out = drop(h @ layers[k])
        stream, h = nn.residual_norm(out, stream, post_weight=layers[k + 1], weight=layers[k + 2],
                                     scale=0.5)
    return nn.linear_cross_entropy(h, head, y, bias)


def exact(x, y, params, masks, p):
    """The same in 64 bits on the CPU, with the masks given."""
    leaves = [q.detach().double().cpu().requires_grad_() for q in params]
    stream = h = x.double().cpu()
    *layers, head, bias = leaves
    rms = lambda v: v * (v.square().mean(-1, keepdim=True) + 1e-5).rsqrt()  # noqa: E731
    for k in range(0, len(layers), 3):
        out = (h @ layers[k]) * masks[k // 3] / (1.0 - p)
        stream = stream + 0.5 * layers[k + 1] * rms(out)
        h = layers[k + 2] * rms(stream)
    loss = torch.nn.functional.cross_entropy(h @ head.t() + bias, y.cpu())
    loss.backward()
    return loss.item(), [q.grad for q in leaves]


def masks_of(drop, shape, count):
    state = drop.state.clone()
    out = []
    for _ in range(count):
        out.append((nn.dropout(torch.ones(shape, device="cuda"), drop.p, state) != 0).double().cpu())
        state[1] += 1
    return out


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, dim, classes", [(1, 8, 3), (37, 33, 200), (300, 64, 50)])
def test_stack_matches_the_formulas(sporder, kind, rows, dim, classes):
    print(f"[stack] {kind} {rows} {dim} {classes}", flush=True)
    x, y, params = make(kind, rows, dim, classes, 3)
    drop = nn.Dropout(0.3, seed=5).cuda()
    masks = masks_of(drop, x.shape, 3)
    loss = forward(x, y, params, drop)
    loss.backward()
    want, grads = exact(x, y, params, masks, 0.3)
    limit = 1e-4 if kind == torch.float32 else 12 * 2.0**-8
    assert abs(loss.item() - want) <= limit * max(1.0, abs(want))
    for p, grad in zip(params, grads):
        got = p.grad.double().cpu()
        if kind == torch.float32:
            assert (got - grad).abs().max() <= limit * grad.abs().max()
        else:
            assert (got - grad).norm() <= limit * grad.norm()


def test_captured_steps_drop_anew_and_equal_eager_ones(sporder):
    print("[stack] captured", flush=True)
    x, y, params = make(torch.bfloat16, 96, 64, 500, 2)

    def step(drop):
        for p in params:
            p.grad = None
        loss = forward(x, y, params, drop)
        grads = torch.autograd.grad(loss, params)
        return [loss.detach(), *grads]

    drop = nn.Dropout(0.25, seed=9).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(drop)
    torch.cuda.current_stream().wait_stream(side)
    drop.state.copy_(torch.tensor([9, 0]))
    eager = [[t.clone() for t in step(drop)] for _ in range(3)]
    assert drop.state.tolist() == [9, 6]  # two calls a step
    drop.state.copy_(torch.tensor([9, 0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(drop)
    drop.state.copy_(torch.tensor([9, 0]))
    for want in eager:
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        step(nn.Dropout(0.25, seed=1).cuda())  # eager work between the replays
    assert not torch.equal(eager[0][0], eager[1][0])


def torch_training(ptr, ind, X, y, hidden, classes, epochs, seed, blocks, p):
    """e2e_gcn's model with --blocks and --dropout in plain torch, with the same
    masks."""
    dev = "cuda"
    n = ptr.shape[0] - 1
    deg = torch.from_numpy(np.diff(ptr).astype(np.float32)).to(dev).clamp_min(1.0)
    rows = torch.repeat_interleave(torch.arange(n), torch.from_numpy(np.diff(ptr).astype(np.int64)))
    A = torch.zeros(n, n).index_put_((rows, torch.from_numpy(ind).long()), torch.ones(ind.shape[0]),
                                     accumulate=True).to(dev)
    A = deg.rsqrt()[:, None] * A * deg.rsqrt()[None, :]
    torch.manual_seed(seed)
    W1 = torch.nn.Linear(X.shape[1], hidden).to(dev)
    W2 = torch.nn.Linear(hidden, classes).to(dev)
    params = list(W1.parameters()) + list(W2.parameters())
    layers = []
    for _ in range(blocks):
        linear = torch.nn.Linear(hidden, hidden).to(dev)
        norms = [torch.ones(hidden, device=dev, requires_grad=True) for _ in range(2)]
        layers.append((linear, *norms))
        params += list(linear.parameters()) + norms
    opt = torch.optim.Adam(params, lr=0.01)
    rms = lambda v: v * (v.square().mean(-1, keepdim=True) + 1e-5).rsqrt()  # noqa: E731
    losses = []
    for epoch in range(epochs):
        def drop(v, k):
            ones = torch.ones(n, hidden, device=dev)
            return v * nn.dropout(ones, p, seed + k, offset=epoch) if p else v
        opt.zero_grad()
        h = drop(torch.relu(A @ W1(X)), 0)
        stream = h
        for k, (linear, post, pre) in enumerate(layers):
            stream = stream + post * rms(drop(A @ linear(h), k + 1))
            h = pre * rms(stream)
        loss = torch.nn.functional.cross_entropy(W2(A @ h), y)
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    return losses


@pytest.mark.parametrize("blocks, p, fused", [(0, 0.0, True), (0, 0.2, False), (2, 0.0, False),
                                              (2, 0.3, True)])
def test_gcn_options_follow_torch(sporder, blocks, p, fused):
    ptr, ind, _ = synth.chung_lu(1500, 2.1, 12, 71)
    print(f"[gcn] n=1500 epochs=6 {blocks} {p} {fused}", flush=True)
    dev = torch.device("cuda")
    n = ptr.shape[0] - 1
    g = torch.Generator(device=dev).manual_seed(8)
    X = torch.randn(n, 20, device=dev, generator=g)
    y = torch.randint(0, 9, (n,), device=dev, generator=g)
    r = e2e_gcn.train(torch.from_numpy(ptr).to(dev), torch.from_numpy(ind).to(dev), X, y, hidden=24,
                      classes=9, epochs=4, warmup=2, seed=8, blocks=blocks, dropout=p,
                      fused_loss=fused)
    want = torch_training(ptr, ind, X, y, 24, 9, 6, 8, blocks, p)
    assert r["losses"] == pytest.approx(want, rel=1e-4)


def test_gcn_with_all_options_runs(sporder):
    ptr, ind, _ = synth.chung_lu(2000, 2.1, 12, 72)
    print("[gcn] n=2000 every option", flush=True)
    rows = e2e_gcn.run(ptr, ind, features=24, hidden=32, classes=7, epochs=3,
                       orders=("ORIGIN", "sporder-csg"), seed=3, fused=True, embed=True, norm=True,
                       muon=True, blocks=2, dropout=0.1, fused_loss=True)
    for r in rows:
        assert r["blocks"] == 2 and r["dropout"] == 0.1 and r["fused_loss"]
        assert np.isfinite(r["final_loss"])
    # without dropout the loss does not depend on the order
    rows = e2e_gcn.run(ptr, ind, features=24, hidden=32, classes=7, epochs=3,
                       orders=("ORIGIN", "sporder-csg"), seed=3, blocks=2, fused_loss=True)
    assert rows[1]["final_loss"] == pytest.approx(rows[0]["final_loss"], rel=1e-4)
