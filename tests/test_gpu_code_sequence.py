"""The losses, dropout, lookup and optimizer together, as examples/train_code_sequence.py has them: that it runs in every type, and its gradients against the same
model in 64 bits on the CPU, the masks from the oracle's generator.

Bar: a gradient goes through some thousand float32 additions in a row (sums over 97 codes, 24 columns, 290 rows, and their products), each off by at
most 2^-24 of the magnitudes that it adds, so 2,000 x 2^-24 of the gradient's own norm, which is of their size here."""
import os
import sys

import numpy as np
import pytest
import torch

import training_ref as R

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'examples'))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_it_runs(dtype):
    from train_code_sequence import train
    losses = train(codes=300, count=8, length=40, width=72, experts=4, steps=3, dtype=dtype)
    assert len(losses) == 3 and np.all(np.isfinite(losses))


@pytest.mark.parametrize('width', [24, 80])
def test_gradients(width):
    import train_code_sequence as S
    codes, experts, drop, seed, balance = 97, 5, 0.25, 11, 0.3
    numbers = S.sequences(codes, 10, 30, 3)
    dev = torch.device('cuda:0')
    p = {k: t.requires_grad_() for k, t in S.parameters(codes, width, experts, 4, torch.float32, dev).items()}
    loss, counts = S.step_loss(p, numbers.to(dev), drop, seed, balance)
    loss.backward()

    q = {k: t.detach().cpu().double().requires_grad_() for k, t in p.items()}
    before, after = numbers[:, :-1].reshape(-1), numbers[:, 1:].reshape(-1)
    n, threshold = len(before), round(drop * 65536)
    kept = [torch.tensor(R.philox_bits(n * width, seed, offset) >= threshold).view(n, width) / (1 - threshold / 65536) for offset in (0, 1)]
    h = q['codebook'][before.clamp(min=0)] * (before >= 0)[:, None] * kept[0]
    logits = h @ q['router']
    chosen = logits.topk(2, dim=1).indices
    gates = torch.zeros_like(logits).scatter(1, chosen, torch.softmax(logits.gather(1, chosen), 1))
    out = ((h @ q['experts']).view(-1, experts, width) * gates[:, :, None]).sum(1) * kept[1] + h
    z = out @ q['codebook'].t() * width ** -0.5
    want = torch.nn.functional.cross_entropy(z, after, ignore_index=-1)
    there = before >= 0
    number = torch.bincount(chosen[there].flatten(), minlength=experts)
    even = experts * ((number / number.sum()) * torch.softmax(logits[there], 1).mean(0)).sum()
    (want + balance * even).backward()
    assert torch.equal(counts.cpu(), number)
    assert abs(float(loss.detach()) - float((want + balance * even).detach())) <= 2000 * 2.0 ** -24 * float(want.detach())
    for k in p:
        off = (p[k].grad.cpu().double() - q[k].grad).norm() / q[k].grad.norm()
        assert float(off) <= 2000 * 2.0 ** -24, (k, float(off))
