"""What programs may hand the training operators beside ordinary values, as far as it shows without a GPU: states on the host,
copies and saved states of optimizers, groups that no step could take."""
import pytest
import torch


def _coded_state(n):
    return dict(step=1, exp_avg_ratio=torch.zeros(n, dtype=torch.uint8), exp_avg_sq_root=torch.zeros(n, dtype=torch.uint8),
                root_scale=torch.zeros((n + 255) // 256), ratio_bound=7.0)


def test_moments_of_coded_states_on_the_host_are_refused():
    """8-bit states loaded for a parameter on the host: no kernel is given their addresses."""
    import efgs
    p = torch.nn.Parameter(torch.zeros(5))
    opt = efgs.AdamW([p], state_bits=8)
    opt.state[p] = _coded_state(5)
    for params in (p, [p]):
        with pytest.raises(ValueError, match='GPU'):
            opt.moments(params)


def test_a_parameter_twice_in_a_group_is_refused():
    """Blocks of one launch would update the same elements at once."""
    import efgs
    p, q = (torch.nn.Parameter(torch.zeros(3)) for _ in range(2))
    with pytest.raises(ValueError, match='more than once'):
        efgs.AdamW([p, q, p])
    opt = efgs.AdamW([p])
    with pytest.raises(ValueError, match='more than once'):
        opt.add_param_group({'params': [q, q]})
    assert len(opt.param_groups) == 1
    opt.add_param_group({'params': [q]})


def test_copies_and_pickles_of_an_optimizer_keep_its_settings():
    import copy
    import io
    import pickle
    import efgs
    p = torch.nn.Parameter(torch.zeros(3))
    opt = efgs.AdamW([p], state_bits=8, max_grad_norm=0.5, seed=11)
    opt.grad_norm = torch.tensor(2.0)
    saved = io.BytesIO()
    torch.save(opt, saved)
    saved.seek(0)
    for other in (copy.deepcopy(opt), copy.copy(opt), pickle.loads(pickle.dumps(opt)), torch.load(saved, weights_only=False)):
        assert other.max_grad_norm == 0.5 and other.seed == 11 and float(other.grad_norm) == 2.0
        assert other.param_groups[0]['state_bits'] == 8
        other.step()                # no gradients: nothing to do
        assert other.grad_norm is None


def test_a_saved_state_holds_the_seed_and_the_clipping_bound():
    """As a learning rate they are taken from what is loaded; saved states without them leave the optimizer's own."""
    import efgs
    p = torch.nn.Parameter(torch.zeros(3))
    saved = efgs.AdamW([p], max_grad_norm=0.5, seed=11).state_dict()
    assert saved['seed'] == 11 and saved['max_grad_norm'] == 0.5
    other = efgs.AdamW([p], max_grad_norm=2.0, seed=12)
    other.load_state_dict({k: saved[k] for k in ('state', 'param_groups')})
    assert other.seed == 12 and other.max_grad_norm == 2.0
    other.load_state_dict(saved)
    assert other.seed == 11 and other.max_grad_norm == 0.5
    other.load_state_dict(efgs.AdamW([p]).state_dict())
    assert other.seed == 0 and other.max_grad_norm is None
    with pytest.raises(ValueError, match='max_grad_norm'):
        other.load_state_dict({**saved, 'max_grad_norm': -1.0})
    assert other.seed == 0 and other.max_grad_norm is None


def test_saved_states_of_torch_optimizers():
    """torch.optim.AdamW's are taken as they are, whose groups know no state_bits: 32, which their states have. Those of another formula
    (amsgrad, maximize, weight decay through the gradient) or without what a group needs are refused, and change nothing."""
    import efgs
    p = torch.nn.Parameter(torch.randn(4, 3))
    theirs = torch.optim.AdamW([p], lr=0.25, betas=(0.8, 0.9), eps=1e-5, weight_decay=0.125)
    p.grad = torch.randn(4, 3)
    theirs.step()
    q = torch.nn.Parameter(torch.zeros(4, 3))
    for bits in (32, 8):
        ours = efgs.AdamW([q], state_bits=bits)
        ours.load_state_dict(theirs.state_dict())
        group, state = ours.param_groups[0], ours.state[q]
        assert (group['lr'], tuple(group['betas']), group['eps'], group['weight_decay'], group['state_bits']) == (0.25, (0.8, 0.9), 1e-5, 0.125, 32)
        assert state['step'] == 1 and isinstance(state['step'], int)
        assert torch.equal(state['exp_avg'], theirs.state[p]['exp_avg']) and torch.equal(state['exp_avg_sq'], theirs.state[p]['exp_avg_sq'])
    ours = efgs.AdamW([q], lr=0.5)
    ours.load_state_dict(torch.optim.Adam([p], weight_decay=0.0).state_dict())
    ours = efgs.AdamW([q], lr=0.5)
    for other in (torch.optim.AdamW([p], amsgrad=True), torch.optim.AdamW([p], maximize=True), torch.optim.Adam([p], weight_decay=0.1),
                  torch.optim.SGD([p], lr=0.1)):
        with pytest.raises(ValueError, match='efgs'):
            ours.load_state_dict(other.state_dict())
        assert ours.param_groups[0]['lr'] == 0.5 and len(ours.state) == 0
    with pytest.raises(ValueError, match='amsgrad'):
        efgs.AdamW([{'params': [q], 'amsgrad': True}])


def test_saved_states_of_other_strides_are_laid_out_anew():
    import efgs
    p = torch.nn.Parameter(torch.zeros(4, 3))
    saved = efgs.AdamW([p]).state_dict()
    moments = torch.arange(12.0).view(3, 4).t()
    saved['state'] = {0: dict(step=torch.tensor(5.0), exp_avg=moments, exp_avg_sq=moments + 1)}
    opt = efgs.AdamW([p])
    opt.load_state_dict(saved)
    for key, want in (('exp_avg', moments), ('exp_avg_sq', moments + 1)):
        assert opt.state[p][key].is_contiguous() and torch.equal(opt.state[p][key], want)
    assert opt.state[p]['step'] == 5


def test_hooks_on_loading_see_and_give_what_is_loaded():
    """A hook before loading may give another saved state; one behind it sees the states as they stay."""
    import efgs
    p = torch.nn.Parameter(torch.zeros(4, dtype=torch.bfloat16))
    saved = efgs.AdamW([p], seed=4).state_dict()
    saved['state'] = {0: dict(step=2, exp_avg=torch.ones(4), exp_avg_sq=torch.ones(4))}
    opt, seen = efgs.AdamW([p]), []
    before = opt.register_load_state_dict_pre_hook(
        lambda _, given: {**given, 'seed': 9, 'state': {0: dict(given['state'][0], step=7, exp_avg=torch.full((4,), 3.0))}})
    behind = opt.register_load_state_dict_post_hook(lambda o: seen.append((o.state[p]['exp_avg'].dtype, o.state[p]['step'])))
    opt.load_state_dict(saved)
    assert opt.state[p]['step'] == 7 and torch.equal(opt.state[p]['exp_avg'], torch.full((4,), 3.0)) and opt.seed == 9
    assert seen == [(torch.float32, 7)]
    before.remove()
    opt.load_state_dict(saved)
    assert opt.state[p]['step'] == 2 and opt.seed == 4 and len(seen) == 2
    behind.remove()
    opt.load_state_dict(saved)
    assert len(seen) == 2


@pytest.mark.parametrize('bad', [dict(lr=float('nan')), dict(lr=float('inf')), dict(lr=[1e-3, float('nan')]), dict(lr=torch.tensor([1e-3, 1e-3])), dict(lr='0.1'),
                                 dict(lr=None), dict(weight_decay=float('nan')), dict(weight_decay=float('-inf')), dict(eps=float('inf')), dict(eps=None),
                                 dict(betas=(0.9,)), dict(betas=0.9), dict(state_bits='8')])
def test_values_that_no_step_could_take_are_refused_at_once(bad):
    import efgs
    p = torch.nn.Parameter(torch.zeros(3))
    with pytest.raises(ValueError):
        efgs.AdamW([p], **bad)
    with pytest.raises(ValueError):
        efgs.AdamW([{'params': [p], **bad}])
    opt = efgs.AdamW([torch.nn.Parameter(torch.zeros(2))])
    with pytest.raises(ValueError):
        opt.add_param_group({'params': [p], **bad})
    assert len(opt.param_groups) == 1


def test_values_that_turn_into_numbers_are_taken():
    import efgs
    opt = efgs.AdamW([torch.nn.Parameter(torch.zeros(3))], lr=torch.tensor(0.5), betas=[0.5, 0.75], eps=0, weight_decay=1)
    assert float(opt.param_groups[0]['lr']) == 0.5
    efgs.AdamW([torch.nn.Parameter(torch.zeros(3))], lr=(1, 2.0, torch.tensor(3.0)))
