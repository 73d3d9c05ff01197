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
