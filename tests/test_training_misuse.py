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
