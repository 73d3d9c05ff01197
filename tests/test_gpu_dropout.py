"""efgs.dropout on the GPU: masks against Philox4x32-10 in Python's whole numbers (oracle/training_ref.py), values bit for bit, one float32 product and sum
rounded once to the type."""
import numpy as np
import pytest
import torch

import training_ref as R

pytestmark = pytest.mark.gpu

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
DEVICE = 'cuda:0'


def expected(x, bits, p, residual=None):
    threshold = round(p * 65536)
    kept = torch.tensor(bits >= threshold, device=DEVICE).view(x.shape)
    scale = torch.tensor(65536.0 / (65536 - threshold) if threshold < 65536 else 0.0, dtype=torch.float32, device=DEVICE)
    out = torch.where(kept, x.float() * scale, torch.zeros((), device=DEVICE))
    return (out if residual is None else out + residual.float()).to(x.dtype)


@pytest.mark.parametrize('n', [1, 7, 8, 9, 63, 2047, 2048, 2049, 5000])
@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('with_residual', [False, True])
def test_lengths(n, dtype, with_residual):
    import efgs
    rng = torch.Generator(DEVICE).manual_seed(n)
    x, residual, up = (torch.randn(n, generator=rng, device=DEVICE).to(TYPES[dtype]) for _ in range(3))
    residual = residual.requires_grad_() if with_residual else None
    x.requires_grad_()
    for p, seed, offset in ((0.1, 7, 0), (0.5, (1 << 64) - 3, (1 << 62) + 12), (0.0, 1, 1), (1.0, 1, 1)):
        bits = R.philox_bits(n, seed, offset)
        out = efgs.dropout(x, p, seed=seed, offset=offset, residual=residual)
        assert out.dtype == x.dtype and torch.equal(out, expected(x.detach(), bits, p, None if residual is None else residual.detach()))
        grads = torch.autograd.grad(out, (x,) if residual is None else (x, residual), up)
        assert torch.equal(grads[0], expected(up, bits, p))
        assert residual is None or torch.equal(grads[1], up)


def test_seeds_that_are_negative_or_on_the_device():
    import efgs
    x = torch.randn(1000, device=DEVICE, requires_grad=True)
    for seed in (-5, 12345678901234567):
        at = torch.tensor([seed], device=DEVICE)
        out = efgs.dropout(x, 0.3, seed=at, offset=4)
        assert torch.equal(out, expected(x.detach(), R.philox_bits(1000, seed & (1 << 64) - 1, 4), 0.3))
        assert torch.equal(out, efgs.dropout(x, 0.3, seed=seed, offset=4))
        g = torch.randn_like(x)
        assert torch.equal(torch.autograd.grad(out, x, g, retain_graph=True)[0], expected(g, R.philox_bits(1000, seed & (1 << 64) - 1, 4), 0.3))
        at += 1
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            torch.autograd.grad(out, x, g)


def test_the_default_generator_is_drawn_from_and_advanced():
    import efgs
    x = torch.ones(4096, device=DEVICE)
    torch.cuda.manual_seed(11)
    a, b = efgs.dropout(x, 0.5), efgs.dropout(x, 0.5)
    torch.cuda.manual_seed(11)
    c, d = efgs.dropout(x, 0.5), efgs.dropout(x, 0.5)
    assert torch.equal(a, c) and torch.equal(b, d) and not torch.equal(a, b)


def test_shares_and_independence():
    """Of n elements a share of 1 - p is kept, within six deviations, also of those whose neighbour is, and of both halves of every word."""
    import efgs
    n = 1 << 22
    x = torch.ones(n, device=DEVICE)
    for p in (0.05, 0.5, 0.9):
        kept = (efgs.dropout(x, p, seed=3) != 0).double()
        deviation = np.sqrt(p * (1 - p) / (n // 8))
        assert abs(float(kept.mean()) - (1 - p)) < 6 * np.sqrt(p * (1 - p) / n) + 2.0 ** -17
        assert torch.all((kept.view(-1, 8).mean(0) - (1 - p)).abs() < 6 * deviation + 2.0 ** -17)
        for shift in (1, 2, 8, 64):
            both = float((kept[shift:] * kept[:-shift]).mean())
            assert abs(both - (1 - p) ** 2) < 6 * np.sqrt(1.0 / n)
        other = (efgs.dropout(x, p, seed=3, offset=1) != 0).double()
        assert abs(float((kept * other).mean()) - (1 - p) ** 2) < 6 * np.sqrt(1.0 / n)


def test_what_stands_in_dropped_places_is_gone():
    import efgs
    bits = R.philox_bits(64, 9, 0)
    x = torch.full((64,), float('nan'), device=DEVICE)
    out = efgs.dropout(x, 0.5, seed=9)
    assert np.array_equal(torch.isnan(out).cpu().numpy(), bits >= 32768)
    assert torch.all(out[torch.tensor(bits < 32768, device=DEVICE)] == 0)


@pytest.mark.parametrize('dtype', list(TYPES))
def test_strides_shapes_and_alignment(dtype):
    import efgs
    base = torch.randn(37, 53, device=DEVICE).to(TYPES[dtype])
    for x in (base.t(), base[1:, 1:], base.view(-1)[1:], base.view(-1)[3:4], base[:, None, ::2]):
        want = efgs.dropout(x.contiguous(), 0.25, seed=5)
        got = efgs.dropout(x, 0.25, seed=5)
        assert torch.equal(got, want) and got.is_contiguous()
        y = x.detach().requires_grad_()
        up = torch.randn(1, device=DEVICE).to(TYPES[dtype]).expand(x.shape)
        grad = torch.autograd.grad(efgs.dropout(y, 0.25, seed=5, residual=x), y, up)[0]
        assert torch.equal(grad, efgs.dropout(up.contiguous(), 0.25, seed=5))
    empty = torch.empty(0, 5, device=DEVICE, requires_grad=True)
    out = efgs.dropout(empty, 0.5, seed=1)
    assert out.shape == (0, 5) and torch.autograd.grad(out.sum(), empty)[0].shape == (0, 5)


def test_a_long_tensor():
    """Elements past 2^31: more than a launch's threads take once."""
    import efgs
    n, first = (1 << 31) + 4099, (1 << 31) - 8
    x = torch.ones(n, dtype=torch.bfloat16, device=DEVICE)
    out = efgs.dropout(x, 0.5, seed=21)
    bits = R.philox_bits(4099 + 8, 21, 0, first)
    assert torch.equal(out[first:], expected(x[first:], bits, 0.5))
    assert torch.equal(out[:4096], expected(x[:4096], R.philox_bits(4096, 21, 0), 0.5))


def test_a_captured_step_replays_with_a_seed_that_counts():
    import efgs
    x = torch.randn(5000, device=DEVICE, requires_grad=True)
    seed = torch.tensor([100], device=DEVICE)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = efgs.dropout(x, 0.5, seed=seed)
        grad = torch.autograd.grad(out, x, torch.ones_like(out))[0]
        seed += 1
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        bits = R.philox_bits(5000, 100 + k, 0)
        assert torch.equal(out, expected(x.detach(), bits, 0.5)) and torch.equal(grad, expected(torch.ones_like(x), bits, 0.5))
    assert int(seed) == 104


def test_a_capture_without_a_seed_is_refused():
    import efgs
    x = torch.randn(50, device=DEVICE)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match='needs its seed'):
            efgs.dropout(x, 0.5)
        y = x + 1
    graph.replay()
    assert torch.equal(y, x + 1)


def test_on_another_stream():
    import efgs
    x = torch.randn(100_000, device=DEVICE)
    want = efgs.dropout(x, 0.5, seed=2)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = efgs.dropout(x * 1.0, 0.5, seed=2)
    stream.synchronize()
    assert torch.equal(got, want)


def test_the_residuals_gradient_is_its_own():
    """Leaves that gather their gradients: none of them shares memory with the upstream gradient or with another's."""
    import efgs
    x, residual, other = (torch.randn(4096, device=DEVICE, requires_grad=True) for _ in range(3))
    up = torch.ones(4096, device=DEVICE)
    for k in range(1, 4):
        efgs.dropout(x, 0.5, seed=k, residual=residual).backward(up)
        assert torch.all(up == 1) and torch.all(residual.grad == k) and residual.grad.data_ptr() != up.data_ptr()
    residual.grad = None
    for k in range(1, 4):
        ((efgs.dropout(x, 0.5, seed=k, residual=residual) + other) * 1.0).backward(up)
        assert torch.all(residual.grad == k) and torch.all(other.grad == k)
        assert len({t.data_ptr() for t in (x.grad, residual.grad, other.grad, up)}) == 4


def test_threads_draw_different_masks():
    """Draws from the default generator by several threads at once: no two the same, and the generator advanced by all of them."""
    import sys
    import threading

    import efgs
    threads, calls = 8, 150
    torch.cuda.manual_seed(5)
    generator = torch.cuda.default_generators[0]
    before, x = generator.get_offset(), torch.ones(256, device=DEVICE)
    masks = [[] for _ in range(threads)]
    start = threading.Barrier(threads)

    def draw(out):
        start.wait()
        for _ in range(calls):
            out.append(efgs.dropout(x, 0.5))

    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        workers = [threading.Thread(target=draw, args=(out,)) for out in masks]
        for w in workers:
            w.start()
        for w in workers:
            w.join()
    finally:
        sys.setswitchinterval(interval)
    kept = (torch.stack([m for out in masks for m in out]) != 0).cpu().numpy()
    assert len({row.tobytes() for row in kept}) == threads * calls
    assert generator.get_offset() == before + 4 * threads * calls


def test_where_a_launchs_threads_begin_again():
    """A launch has 2^31 threads at most, eight elements each: both sides of element 2^34, and a tail of three."""
    import efgs
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip('takes 70 GB of GPU memory')
    n = (1 << 34) + 4099
    x = torch.ones(n, dtype=torch.bfloat16, device=DEVICE)
    out = efgs.dropout(x, 0.25, seed=33, offset=5)
    for first, last in ((0, 4096), ((1 << 31) - 4096, (1 << 31) + 4096), ((1 << 34) - 4096, n)):
        assert torch.equal(out[first:last], expected(x[first:last], R.philox_bits(last - first, 33, 5, first), 0.25))
    del x, out
    torch.cuda.empty_cache()
