"""What programs may hand the training operators beside ordinary tensors: nodes called directly, hooks, dual numbers, copies and
saved states of optimizers, values at the ends of their types. Refused before any device work, or computed by the formulas."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEVICE = 'cuda:0'


def test_embedding_node_checks_its_upstream():
    """A node called directly passes autograd's own checks by: shapes and devices that the kernels would read past are refused."""
    import efgs
    indices = torch.randint(0, 9, (5, 3), device=DEVICE)
    table = torch.randn(9, 4, device=DEVICE, requires_grad=True)
    out = efgs.embedding(indices, table)
    for upstream in (torch.ones(5, 2, 4, device=DEVICE), torch.ones(15, 4, device=DEVICE), torch.ones(1, device=DEVICE), torch.ones(5, 3, 5, device=DEVICE)):
        with pytest.raises(ValueError, match="the output's shape"):
            out.grad_fn(upstream)
    with pytest.raises(ValueError, match="on the gradient's device"):
        out.grad_fn(torch.ones(5, 3, 4))
    with pytest.raises(ValueError, match='float32, bfloat16 or float16'):
        out.grad_fn(torch.ones(5, 3, 4, device=DEVICE, dtype=torch.float64))
    got = out.grad_fn(torch.ones(5, 3, 4, device=DEVICE))
    got = got[0] if isinstance(got, tuple) else got
    assert torch.equal(got, torch.bincount(indices.reshape(-1), minlength=9).float()[:, None].expand(9, 4))


def test_embedding_node_checks_what_hooks_give_back():
    """Hooks on saved tensors that return the indices on the host, or as floats, are refused; in other strides they are read right."""
    import efgs
    indices = torch.randint(0, 9, (6, 5), device=DEVICE)
    table = torch.randn(9, 4, device=DEVICE, requires_grad=True)
    upstream = torch.randn(6, 5, 4, device=DEVICE)
    want = torch.autograd.grad(efgs.embedding(indices, table), table, upstream)[0]
    for unpack in (lambda x: x.cpu(), lambda x: x.float(), lambda x: x.short()):
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, unpack):
            out = efgs.embedding(indices, table)
        with pytest.raises(ValueError, match='indices'):
            out.backward(upstream)
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x.t().contiguous().t()):
        out = efgs.embedding(indices, table)
    assert torch.equal(torch.autograd.grad(out, table, upstream)[0], want)


@pytest.mark.parametrize('requires_grad', [False, True])
@pytest.mark.parametrize('grad_mode', [False, True])
def test_embedding_of_a_dual_number_is_refused(requires_grad, grad_mode):
    """There is no forward-mode derivative: an error, as the rasterizer's, and no result without a tangent."""
    import efgs
    from torch.autograd import forward_ad
    indices = torch.randint(0, 9, (5,), device=DEVICE)
    table = torch.randn(9, 4, device=DEVICE, requires_grad=requires_grad)
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            efgs.embedding(indices, forward_ad.make_dual(table, torch.ones_like(table)))
        assert efgs.embedding(indices, table).shape == (5, 4)


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('eps', [1e-38, 2e-39, 1e-42, 2.0 ** -149, 1e-60])
def test_eps_below_the_least_reciprocal(bits, eps):
    """The reciprocal of an eps below 2^-128 is no float, yet the formula is: a parameter whose moments are zero keeps to its decay, one whose
    m is not zero and whose v underflows moves by lr m / eps (an eps below float32's least number counts as that), and to
    ordinary gradients the eps is nothing. Bars: e = 2^-24; 4 e of p and of the update for the ordinary ones, 16 e for m / eps."""
    import efgs
    e, n, lr, decay = 2.0 ** -24, 700, 1e-3, 0.05
    kept = {}
    for value in (eps, 1e-33):
        p = torch.linspace(-2.0, 2.0, n, device=DEVICE).requires_grad_()
        p0 = p.detach().clone()
        generator = torch.Generator(DEVICE).manual_seed(3)
        p.grad = torch.randn(n, generator=generator, device=DEVICE) * 0.1
        p.grad[256:512] = 0.0
        p.grad[520] = 1e-24
        opt = efgs.AdamW([p], lr=lr, weight_decay=decay, eps=value, state_bits=bits)
        opt.step()
        kept[value] = p.detach().double()
    now, other, p0 = kept[eps], kept[1e-33], p0.double()
    assert bool(((now - p0 * (1 - lr * decay)).abs() <= 3 * e * p0.abs())[256:512].all())
    ordinary = torch.arange(n, device=DEVICE) != 520
    assert bool(((now - other).abs() <= 4 * e * (p0.abs() + lr))[ordinary].all())
    want = float(p0[520]) * (1 - lr * decay) - lr * float(torch.tensor(1e-24)) / max(eps, 2.0 ** -149)
    assert float(now[520]) == pytest.approx(want, rel=16 * e)


@pytest.mark.parametrize('bits', [32, 8])
def test_a_copied_optimizer_goes_on_bit_for_bit(bits):
    """A model and its optimizer copied together, and pickled together."""
    import copy
    import pickle
    import efgs
    p = torch.randn(1500, device=DEVICE).requires_grad_()
    p.grad = torch.randn(1500, device=DEVICE)
    opt = efgs.AdamW([p], state_bits=bits, max_grad_norm=0.5, seed=3)
    opt.step()
    copies = [copy.deepcopy((p, opt)), pickle.loads(pickle.dumps((p, opt)))]
    opt.step()
    for q, other in copies:
        q.grad = p.grad.clone()
        other.step()
        assert torch.equal(q, p) and float(other.grad_norm) == float(opt.grad_norm)
        assert all(torch.equal(x, y) for x, y in zip(other.moments(q), opt.moments(p)))


def test_a_resumed_run_of_8_bit_states_is_the_same_run():
    """The dither of a resumed optimizer is the saved one's, whatever seed it was made with."""
    import copy
    import efgs
    p = torch.randn(1500, device=DEVICE).requires_grad_()
    p.grad = torch.randn(1500, device=DEVICE)
    opt = efgs.AdamW([p], state_bits=8, max_grad_norm=0.5, seed=3)
    opt.step()
    q = p.detach().clone().requires_grad_()
    q.grad = p.grad.clone()
    other = efgs.AdamW([q], state_bits=8)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    opt.step()
    other.step()
    assert torch.equal(q, p) and all(torch.equal(x, y) for x, y in zip(other.moments(q), opt.moments(p)))


@pytest.mark.parametrize('change', [dict(betas=(0.95, 0.9)), dict(betas=(0.9, 0.81)), dict(state_bits=16), dict(lr=float('nan')), dict(eps=-1.0)])
def test_a_refused_group_leaves_no_state_behind(change):
    """Values that a program set between steps: the refused step makes no states that a later one could not read."""
    import efgs
    p, q = (torch.ones(300, device=DEVICE).requires_grad_() for _ in range(2))
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    opt = efgs.AdamW([{'params': [p]}, {'params': [q], 'state_bits': 8}], seed=5)
    group = opt.param_groups[1]
    kept = dict(group)
    group.update(change)
    with pytest.raises((RuntimeError, ValueError), match='efgs'):
        opt.step()
    assert torch.equal(p, torch.ones_like(p)) and len(opt.state) == 0
    group.update(kept)
    opt.step()
    other = torch.ones(300, device=DEVICE).requires_grad_()
    other.grad = torch.ones_like(other)
    efgs.AdamW([other], state_bits=8, seed=5).step()
    assert torch.equal(q, other) and opt.state[q]['step'] == 1


@pytest.mark.parametrize('bits', [32, 8])
def test_a_step_that_runs_out_of_memory_can_be_taken_again(bits):
    """The second of a state's tensors does not fit (a limit on the process's memory): nothing half made stays."""
    import efgs
    torch.cuda.empty_cache()
    p = torch.ones(96 << 20, dtype=torch.bfloat16, device=DEVICE).requires_grad_()
    p.grad = torch.ones_like(p)
    opt = efgs.AdamW([p], lr=0.1, state_bits=bits)
    one = p.numel() * (4 if bits == 32 else 1)
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + 1.5 * one) / total)
    try:
        with pytest.raises(torch.cuda.OutOfMemoryError):
            opt.step()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    opt.step()
    assert opt.state[p]['step'] == 1 and bool((p[:: 1 << 20] < 1.0).all())
    del opt, p
    torch.cuda.empty_cache()


def test_parameters_made_in_inference_mode():
    """They have no version to count; a step updates them once, and counts."""
    import efgs
    with torch.inference_mode():
        p = torch.ones(300, device=DEVICE)
        p.grad = torch.ones_like(p)
        opt = efgs.AdamW([p], lr=0.1)
        opt.step()
    q = torch.ones(300, device=DEVICE).requires_grad_()
    q.grad = torch.ones_like(q)
    efgs.AdamW([q], lr=0.1).step()
    assert opt.state[p]['step'] == 1 and torch.equal(p, q)


def test_scratch_follows_the_call():
    """A gradient of a few rows takes no more scratch after one of many has run: 12,288 indices into 5,000 rows of 8 floats need two lists of
    8 bytes a key, a table of 512 KB and a few KB of open rows; 2 MB are allowed beside the gradient itself."""
    import efgs

    def peak(n, rows, columns):
        table = torch.zeros(rows, columns, device=DEVICE, requires_grad=True)
        indices = torch.randint(0, rows, (n,), device=DEVICE)
        out = efgs.embedding(indices, table)
        upstream = torch.ones_like(out)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        torch.autograd.grad(out, table, upstream)
        return torch.cuda.max_memory_allocated() - before - table.numel() * 4

    assert peak(400_000, 50_000, 1024) > 40 << 20
    assert peak(12_288, 5_000, 8) < 2 << 20
    assert peak(500, 100, 8) < 2 << 20
