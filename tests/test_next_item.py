"""examples/next_item.py: the operators and the row update together as one model uses them, against the same model written
with torch's autograd in 64 bits, and a short training run.  No counterpart in the reference."""
import importlib.util
import math
from pathlib import Path

import pytest
import torch


def _example():
    path = Path(__file__).resolve().parents[1] / 'examples' / 'next_item.py'
    spec = importlib.util.spec_from_file_location('next_item', path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _autograd(model, ids, targets, eps):
    """Loss and gradients of the same weights by autograd, in float64 on the CPU."""
    leaf = lambda r: r[:, 0].double().cpu().requires_grad_()  # noqa: E731
    table, head = leaf(model.table), leaf(model.head)
    blocks = [(leaf(a), leaf(b)) for a, b in model.blocks]
    gains = [leaf(g) for g in model.gains]
    ids, targets = ids.cpu(), targets.cpu()

    def norm(h, g):
        return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * g[0]
    h = table[ids]
    for (a, b), g in zip(blocks, gains):
        h = h + torch.relu(norm(h, g) @ a) @ b
    logp = torch.log_softmax(norm(h, gains[-1]) @ head.t(), -1)
    has = targets >= 0
    own = logp[torch.arange(len(ids)), targets.clamp(min=0)]
    ent = -(logp.exp() * logp).sum(-1)
    loss = -((own + model.beta * ent) * has).sum() / has.sum()
    loss.backward()
    return loss.detach(), table.grad, [w.grad for pair in blocks for w in pair] + [head.grad] + [g.grad for g in gains]


@pytest.mark.gpu
def test_gradients_equal_autograd(dev):
    """Every gradient of one step in float32.  The products' sums are of at most 301 fp32 terms (u = 2^-24 each), there are
    about ten products and norms in a row, and errors are taken against each gradient's largest entry: 1e-4 is 1,700 u."""
    ex = _example()
    model = ex.NextItem(items=301, width=48, hidden=80, layers=2, dtype=torch.float32, device=dev)
    g = torch.Generator().manual_seed(1)
    x = ex.sessions(g, 301, 9, 7).to(dev)
    ids, targets = x[:, :-1].reshape(-1), x[:, 1:].reshape(-1).clone()
    targets[5] = -1
    loss, rows, d_rows, grads = model.gradients(ids, targets)
    ref_loss, ref_table, ref = _autograd(model, ids, targets, ex.EPS)
    assert abs(float(loss) - float(ref_loss)) < 1e-4 * float(ref_loss)
    got = torch.zeros_like(ref_table)
    got[rows.cpu()] = d_rows.double().cpu()
    for a, b in [(got, ref_table)] + [(a.double().cpu().reshape(b.shape), b) for a, b in zip(grads, ref)]:
        assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max())


@pytest.mark.gpu
def test_training_and_serving(dev):
    """The loss falls well below the uniform one, clipping holds the norm, and the rule's successors lead the list."""
    ex = _example()
    model = ex.NextItem(items=500, width=64, layers=1, lr=5e-3, device=dev)
    g = torch.Generator().manual_seed(2)
    first = last = None
    for _ in range(150):
        x = ex.sessions(g, 500, 32, 16).to(dev)
        loss, norm = model.train(x[:, :-1].reshape(-1), x[:, 1:].reshape(-1))
        last = float(loss)
        first = last if first is None else first
        assert math.isfinite(last) and math.isfinite(float(norm))
    assert abs(first - math.log(500)) < 1.0 and last < 0.5 * math.log(500)
    ids = torch.arange(0, 500, 7, device=dev)
    top, lp = model.likeliest(ids)
    assert float((top[:, 0] == (ids * 3 + 7) % 500).float().mean()) > 0.9
    assert bool((lp[:, :-1] >= lp[:, 1:]).all())
