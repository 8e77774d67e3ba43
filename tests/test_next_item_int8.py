"""examples/next_item.py with activations kept in 8 bits, and its draws: the operators of elara_amd.int8, sampling and norms as one model
uses them.  No counterpart in the reference."""
import importlib.util
from pathlib import Path

import pytest
import torch

U = 2.0 ** -24


def _example():
    path = Path(__file__).resolve().parents[1] / 'examples' / 'next_item.py'
    spec = importlib.util.spec_from_file_location('next_item', path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _batch(ex, dev, items):
    x = ex.sessions(torch.Generator().manual_seed(1), items, 16, 12).to(dev)
    targets = x[:, 1:].reshape(-1).clone()
    targets[5] = -1
    return x[:, :-1].reshape(-1), targets


@pytest.mark.gpu
def test_gradients_from_kept_activations(dev):
    """The forward pass and what does not read a kept value are bitwise those of the model that keeps nothing in 8 bits.  The last
    block's first weight meets its kept input alone: each entry is within sum |du| s / 2 of the other model's (s a value's scale: half
    a step of rounding), and both sums' fp32 errors.  Further down everything is within what rounding leaves: a value's error has the
    standard deviation s / sqrt(12), s at most max / 63.5 of its group of 80 or so roughly normal values (max below 4 deviations), so
    1.8 % of their deviation, once for each of two blocks: 5 % of each gradient's norm."""
    ex = _example()
    a, b = (ex.NextItem(items=301, width=80, hidden=96, layers=2, dtype=torch.float32, device=dev, keep8=k) for k in (False, True))
    ids, targets = _batch(ex, dev, 301)
    la, rows_a, da, ga = a.gradients(ids, targets)
    lb, rows_b, db, gb = b.gradients(ids, targets)
    assert torch.equal(la, lb) and torch.equal(rows_a, rows_b)
    # dense(): (w1, w2) of each block, the head, the gains
    for i in (3, 4, 7):                            # the last block's second weight, the head, the last gain
        assert torch.equal(ga[i], gb[i])
    add, h, kept = b.forward(ids)
    nrm, w1, w2, u = kept[-1]
    full, _, _, _ = a.forward(ids)[2][-1]
    assert torch.equal(full.rstd, nrm.rstd)
    # du of the last block, as both models compute it, from its own gradient: da = y^T du
    step = nrm.y.scale.repeat_interleave(ex.GROUP, 1)[:, :80].double()
    last = a.forward(ids)
    du = _last_du(ex, a, last, targets).double()
    size = full.y.double().abs().t() @ du.abs()
    bound = step.t() @ du.abs() / 2 + 2 * (len(ids) + 64) * U * size * 2
    diff = (ga[2].double() - gb[2].double()).abs()
    assert bool((diff <= bound).all()), float((diff - bound).max())
    assert float(diff.max()) > 0
    for x, y in [(da, db)] + list(zip(ga, gb)):
        assert float((x.double() - y.double()).norm()) <= 0.05 * float(x.double().norm())


def _last_du(ex, model, forward, targets):
    from elara_amd import logprobs, norms
    add, h, kept = forward
    last = norms.rms_norm(add, model._gain(-1), ex.EPS, residual=h)
    head = model._weight(model.head)
    logits = last.y @ head.t()
    r = logprobs.token_logprobs(logits, targets)
    has = (targets >= 0).float()
    n = has.sum().clamp(min=1)
    d = logprobs.token_logprobs_backward(logits, targets, r.lse, r.entropy, -(has / n), -model.beta * has / n)
    dh, _ = norms.rms_norm_backward(d @ head, last.h, model._gain(-1), last.rstd)
    _, _, b, u = kept[-1]
    return (dh @ b.t()) * (u > 0)


@pytest.mark.gpu
def test_training_step_and_draws(dev):
    """A few steps run with kept activations in bf16; draws come from the product's own logits."""
    from elara_amd import int8, norms, sampling
    ex = _example()
    model = ex.NextItem(items=500, width=64, layers=2, lr=5e-3, device=dev, keep8=True)
    ids, targets = _batch(ex, dev, 500)
    for _ in range(3):
        loss, norm = model.train(ids, targets)
        assert torch.isfinite(loss) and torch.isfinite(norm)
    head = model.head8()
    assert head.q.shape == (500, 64) and head.scale.shape == (500, 1)
    u = torch.rand(len(ids), generator=torch.Generator().manual_seed(3)).to(dev)
    r = model.draw(ids, u, head, temperature=0.9, top_k=30, top_p=0.9)
    assert r.token.shape == ids.shape and bool(((r.token >= 0) & (r.token < 500)).all()) and bool((r.logprob <= 0).all())
    add, h, _ = model.forward(ids)
    y = norms.rms_norm(add, model._gain(-1), ex.EPS, residual=h).y
    logits = int8.linear(int8.quantize(y), head, dtype=torch.float32)
    exact = y.double() @ model._weight(model.head).double().t()
    # each operand within half a step, 1 / 254 of its row's largest: the product within the sum of both shares of |y| |w|
    ya, wa = y.double().abs(), model._weight(model.head).double().abs()
    bound = (ya.amax(1, keepdim=True) / 254) @ wa.sum(1)[None] + ya.sum(1, keepdim=True) @ (wa.amax(1) / 254)[None] + \
        64 * (ya.amax(1, keepdim=True) / 254) @ (wa.amax(1) / 254)[None] + 1e-6
    assert bool(((logits.double() - exact).abs() <= bound).all())
    assert torch.equal(model.draw(ids, u, head, temperature=0.0).token,
                       sampling.sample_tokens(int8.linear(int8.quantize(y), head, dtype=torch.bfloat16), u, top_k=1).token)
    again = model.draw(ids, u, head, temperature=0.9, top_k=30, top_p=0.9)
    assert torch.equal(r.token, again.token) and torch.equal(r.logprob, again.logprob)
