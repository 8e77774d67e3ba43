"""A next-item model trained and served with this library: an item table in ELARA records looked up row by row, a small
residual trunk, a softmax over all items.

One training step, and what runs it:
  rows of the batch's unique items     dedup.unique
  residual blocks h += relu(norm(h) W1) W2   norms.rms_norm, with the block's output added inside the next norm
  loss over all items                  logprobs.token_logprobs (log probability of the next item, entropy bonus)
  its gradient to the logits           logprobs.token_logprobs_backward, written over the logits
  back through the blocks              norms.rms_norm_backward (the residual stream's gradient added inside)
  sums per unique item                 dedup.embedding_dense_backward
  clipping over all gradients          gradnorm.clip_grad_norm, 16-bit gradients into the fp32 that Adam reads
  update                               ops.gpu_adam (the batch's rows), ops.adam_rows_dense (the dense weights)

With keep8 the norms' inputs and outputs are kept for the backward pass in 8 bits (int8.quantize with power-of-two scales), and the
backward pass reads them so: norms.rms_norm_backward_int8 and int8.weight_grad.  (The inner activation stays as it is: where it is
positive has to be known exactly.)

Serving scores one session: rms_norm_fp8 before the output product and token_logprobs for the likeliest items; or draws its next item:
the output product in 8-bit integers (int8.linear) and sampling.sample_tokens.

    python examples/next_item.py [--items 20000 --width 256 --batch 64 --length 32 --steps 100 --keep8]

The data is synthetic: sessions that walk the items by a fixed rule and jump at random now and then.
"""
import argparse
import math
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from elara_amd import dedup, gradnorm, int8, logprobs, norms, ops, sampling, synth  # noqa: E402
from elara_amd.gpu_ops import init_rows  # noqa: E402

EPS = 1e-6
GROUP = 128      # columns of a scale of what is kept in 8 bits


class NextItem:
    """Weights are the w of (w, m, v) records, [rows, 3, width] fp32; activations and products have `dtype`."""

    def __init__(self, items, width, hidden=None, layers=2, dtype=torch.bfloat16, lr=1e-3, max_norm=1.0, entropy=1e-3,
                 device='cuda:0', seed=0, keep8=False):
        hidden = hidden or 2 * width
        self.items, self.dtype, self.hp, self.max_norm, self.beta = items, dtype, (lr, 0.9, 0.999, 1e-8), max_norm, entropy
        self.keep8 = keep8
        dev = torch.device(device)

        def records(rows, cols, bound, first):
            ids = torch.arange(first, first + rows, dtype=torch.int64, device=dev)
            return init_rows(ids, cols, seed, bound)
        self.table = records(items, width, synth.bound_for(width), 0)
        self.head = records(items, width, synth.bound_for(width), items)
        self.blocks, at = [], 2 * items
        for _ in range(layers):
            self.blocks.append((records(width, hidden, synth.bound_for(width), at),
                                records(hidden, width, synth.bound_for(hidden), at + width)))
            at += width + hidden
        self.gains = [torch.zeros(1, 3, width, device=dev) for _ in range(layers + 1)]
        for g in self.gains:
            g[:, 0] = 1.0
        self.step = 0

    def dense(self):
        """The records that every step updates, in the order of their gradients."""
        return [w for pair in self.blocks for w in pair] + [self.head] + self.gains

    def _weight(self, rec):
        return rec[:, 0].to(self.dtype)

    def _gain(self, i):
        return self.gains[i][0, 0]

    def forward(self, ids):
        """The last norm's input and what the backward needs, for ids [n]."""
        h = self.table[ids, 0].to(self.dtype)
        add, kept = None, []
        for i, (w1, w2) in enumerate(self.blocks):
            n = norms.rms_norm(add if add is not None else h, self._gain(i), EPS, residual=h if add is not None else None)
            h = n.h
            a, b = self._weight(w1), self._weight(w2)
            u = torch.relu(n.y @ a)
            add = u @ b
            if self.keep8:
                n = norms.Norm(int8.quantize(n.y, GROUP, pow2=True), int8.quantize(h, GROUP, pow2=True), n.rstd)
            kept.append((n, a, b, u))
        return add, h, kept

    def gradients(self, ids, targets):
        """(loss, unique item ids, their summed gradients, gradients of dense()): a step without its update."""
        add, h, kept = self.forward(ids)
        last = norms.rms_norm(add, self._gain(-1), EPS, residual=h)
        head = self._weight(self.head)
        logits = last.y @ head.t()
        r = logprobs.token_logprobs(logits, targets)
        n = (targets >= 0).sum().clamp(min=1)
        has = (targets >= 0).float()
        loss = -(r.logprob + self.beta * r.entropy * has).sum() / n
        d = logprobs.token_logprobs_backward(logits, targets, r.lse, r.entropy, -(has / n), -self.beta * has / n, out=logits)
        d_head = d.t() @ last.y
        dh, d_gain = norms.rms_norm_backward(d @ head, last.h, self._gain(-1), last.rstd)
        pairs, gains = [], [d_gain]
        for i in range(len(kept) - 1, -1, -1):
            nrm, a, b, u = kept[i]
            db = u.t() @ dh
            du = (dh @ b.t()) * (u > 0)
            if self.keep8:
                da = int8.weight_grad(du, nrm.y, transposed=True)
                dh, d_gain = norms.rms_norm_backward_int8(du @ a.t(), nrm.h, self._gain(i), nrm.rstd, dh=dh)
            else:
                da = nrm.y.t() @ du
                dh, d_gain = norms.rms_norm_backward(du @ a.t(), nrm.h, self._gain(i), nrm.rstd, dh=dh)
            pairs = [da, db] + pairs
            gains = [d_gain] + gains
        rows, inverse = dedup.unique(ids, bound=self.items)
        d_rows = dedup.embedding_dense_backward(dh.float(), inverse, rows.numel())
        return loss, rows, d_rows, pairs + [d_head] + gains

    def train(self, ids, targets):
        """One step on ids [n] and the items that followed them [n] (negative: none); returns (loss, gradient norm)."""
        loss, rows, d_rows, grads = self.gradients(ids, targets)
        out = [torch.empty(g.shape, dtype=torch.float32, device=g.device) for g in grads]
        norm = gradnorm.clip_grad_norm([d_rows] + grads, self.max_norm, out=[d_rows] + out)
        self.step += 1
        ops.gpu_adam(self.table, rows, d_rows, *self.hp, self.step)
        for rec, g in zip(self.dense(), out):
            ops.adam_rows_dense(rec, g, *self.hp, self.step)
        return loss, norm

    def likeliest(self, ids, k=5):
        """The k likeliest next items of each id and their log probabilities, the output product's input in fp8.  (This library
        has no fp8 product, so the bytes are widened for torch's; a program with one passes q.y and q.scale to it.)"""
        add, h, _ = self.forward(ids)
        q = norms.rms_norm_fp8(add, self._gain(-1), EPS, residual=h)
        logits = (q.y.to(self.dtype) @ self._weight(self.head).t()) * q.scale.to(self.dtype)
        r = logprobs.token_logprobs(logits, torch.full_like(ids, -1), k=k)
        return r.top_id, r.top_logprob


    def head8(self):
        """The output weight in 8-bit integers with a scale for each item: made once for many draws."""
        return int8.quantize(self._weight(self.head))

    def draw(self, ids, u, head8, **settings):
        """An item after each id, drawn with the numbers u [n] in [0, 1) and sampling.sample_tokens' settings, and its log
        probability."""
        add, h, _ = self.forward(ids)
        x = int8.quantize(norms.rms_norm(add, self._gain(-1), EPS, residual=h).y)
        return sampling.sample_tokens(int8.linear(x, head8, dtype=self.dtype), u, **settings)


def sessions(gen, items, batch, length, jump=0.1):
    """[batch, length + 1] items: each follows from the one before by a fixed rule, or is a jump anywhere."""
    x = torch.empty(batch, length + 1, dtype=torch.int64)
    x[:, 0] = torch.randint(0, items, (batch,), generator=gen)
    for t in range(length):
        follow = (x[:, t] * 3 + 7) % items
        leap = torch.rand(batch, generator=gen) < jump
        x[:, t + 1] = torch.where(leap, torch.randint(0, items, (batch,), generator=gen), follow)
    return x


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument('--items', type=int, default=20_000)
    ap.add_argument('--width', type=int, default=256)
    ap.add_argument('--batch', type=int, default=64)
    ap.add_argument('--length', type=int, default=32)
    ap.add_argument('--steps', type=int, default=100)
    ap.add_argument('--lr', type=float, default=2e-3)
    ap.add_argument('--keep8', action='store_true', help='keep the norms\' inputs and outputs in 8 bits for the backward pass')
    a = ap.parse_args(argv)
    gen = torch.Generator().manual_seed(0)
    model = NextItem(a.items, a.width, lr=a.lr, keep8=a.keep8)
    losses, began = [], None
    for s in range(a.steps):
        x = sessions(gen, a.items, a.batch, a.length).cuda()
        loss, norm = model.train(x[:, :-1].reshape(-1), x[:, 1:].reshape(-1))
        losses.append(loss)
        if s == 4:
            torch.cuda.synchronize()
            began = time.perf_counter()
        if s % 20 == 0 or s == a.steps - 1:
            print(f'step {s:4d}  loss {float(loss):7.4f} (uniform {math.log(a.items):.4f})  gradient norm {float(norm):.4f}',
                  flush=True)
    torch.cuda.synchronize()
    if began is not None and a.steps > 5:
        print(f'{(a.steps - 5) * a.batch * a.length / (time.perf_counter() - began):.0f} tokens/s')
    ids = torch.arange(3, device='cuda:0') * 11
    top, lp = model.likeliest(ids)
    for i, t, p in zip(ids.tolist(), top.tolist(), lp.tolist()):
        print(f'after item {i} (by the rule {(3 * i + 7) % a.items}): {t}  log probabilities {[round(v, 3) for v in p]}')
    drawn = model.draw(ids.repeat(4), torch.rand(12, generator=gen).cuda(), model.head8(), temperature=0.8, top_k=50, top_p=0.95)
    print(f'four draws after each: {drawn.token.view(4, 3).t().tolist()}')
    return [float(v) for v in losses]


if __name__ == '__main__':
    main()
