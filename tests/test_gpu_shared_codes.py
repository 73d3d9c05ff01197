"""The operators together, as examples/train_shared_codes.py has them: lookup, render, sorted gradient, clipped AdamW step. Training
lowers the loss, and 8-bit states end within 10 % of what 32-bit ones reach. The step's gradients of codebook rows equal those
of per-primitive features summed by row."""
import os
import sys

import numpy as np
import pytest
import torch

import training_ref as R

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'examples'))


def test_training_with_shared_codes():
    from train_shared_codes import train
    ends = {}
    for bits in (32, 8):
        losses = train(primitives=20_000, codes=512, steps=60, state_bits=bits, width=320, height=180)
        assert np.all(np.isfinite(losses))
        ends[bits] = np.mean(losses[-5:])
        print(f'shared codes, {bits}-bit states: loss {losses[0]:.4f} -> {ends[bits]:.4f}', flush=True)
        assert ends[bits] < 0.7 * losses[0]
    assert ends[8] < 1.1 * ends[32]


def test_codebook_gradient_is_the_sum_of_feature_gradients():
    import efgs
    import train_shared_codes as T
    dev = torch.device('cuda:0')
    T.train(primitives=200, codes=8, steps=1, width=64, height=48)   # (selects the appearance)
    n, codes, scale = 3000, 37, 0.5
    p = T.scene_tensors(n, codes, 96, 64, 4, dev)
    cam = T.make_scene('c3', n=1, width=96, height=64)['camera']
    settings = efgs.RasterizerSettings(
        w2c=torch.tensor(cam['w2c'], device=dev), cam_position=torch.tensor(cam['position'], device=dev), bg_color=torch.zeros(3, device=dev),
        appearance_degree=1, width=96, height=64, focal_x=cam['focal_x'], focal_y=cam['focal_y'], center_x=48.0, center_y=32.0, near_plane=0.2,
        far_plane=1e4, proper_antialiasing=False, render_base=True, render_residual=True)
    numbers = torch.randint(-1, codes, (n,), device=dev)
    p['codebook'].requires_grad_()
    upstream = torch.randn(3, 64, 96, device=dev)
    image = T.render(p, numbers, settings, scale)
    got = torch.autograd.grad(image, p['codebook'], upstream)[0]
    features = efgs.embedding(numbers, p['codebook'].detach(), scale).requires_grad_()
    same = efgs.diff_rasterize(p['means'], p['scales'], p['rotations'], p['opacities'], torch.empty(0, device=dev), settings,
                               base_colors=p['base_colors'], residual_params=features, mlp_weights=p['mlp_weights'])
    assert torch.equal(image, same)
    by_primitive = torch.autograd.grad(same, features, upstream)[0]
    want, size, entries = R.embedding_gradient(numbers.cpu().numpy(), by_primitive.double().cpu().numpy(), codes, scale)
    # (a float32 sum of k values: (k + 1) e of their magnitudes, and e for the last rounding)
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= (entries[:, None] + 2) * 2.0 ** -24 * size)
