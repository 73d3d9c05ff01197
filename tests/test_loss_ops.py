"""The losses and dropout as far as they show without a GPU: the oracle's formulas against differences and known values, and what the entry points refuse
before they touch a device."""
import ctypes

import numpy as np
import pytest
import torch

import training_ref as R


def test_cross_entropy_gradients_against_differences():
    rng = np.random.default_rng(1)
    x, w, y = rng.normal(size=(5, 8)), rng.normal(size=(9, 8)), np.array([0, 3, -1, 8, 3])
    weights = rng.normal(size=5)
    losses, _, _, dx, dw = R.cross_entropy(x, w, y, 0.7, weights)
    assert losses[2] == 0 and np.all(dx[2] == 0)

    def f(x, w):
        return (R.cross_entropy(x, w, y, 0.7, weights)[0] * weights).sum()
    h = 1e-5
    for _ in range(6):
        a, b = rng.normal(size=x.shape), rng.normal(size=w.shape)
        slope = (f(x + h * a, w + h * b) - f(x - h * a, w - h * b)) / (2 * h)
        assert abs(slope - (dx * a).sum() - (dw * b).sum()) < 1e-8 * (1 + abs(slope))


def test_cross_entropy_oracle_against_torch():
    rng = np.random.default_rng(2)
    x, w, y = rng.normal(size=(6, 4)), rng.normal(size=(7, 4)), np.array([0, -100, 6, 2, 2, 1])
    want = torch.nn.functional.cross_entropy(torch.tensor(1.3 * x @ w.T), torch.tensor(y), reduction='none', ignore_index=-100)
    assert np.allclose(R.cross_entropy(x, w, y, 1.3, np.ones(6))[0], want.numpy(), rtol=1e-12, atol=1e-12)


def test_balance_gradients_against_differences():
    rng = np.random.default_rng(3)
    z, indices = rng.normal(size=(7, 5)), rng.integers(-1, 6, (7, 2))
    indices[3] = -1
    loss, counts, gradient = R.balance(z, indices)
    assert np.all(gradient[3] == 0) and counts.sum() == ((indices >= 0) & (indices < 5)).sum()
    for _ in range(6):
        a, h = rng.normal(size=z.shape), 1e-5
        slope = (R.balance(z + h * a, indices)[0] - R.balance(z - h * a, indices)[0]) / (2 * h)
        assert abs(slope - (gradient * a).sum()) < 1e-8
    assert abs(R.balance(np.zeros((8, 4)), (np.arange(8) % 4)[:, None])[0] - 1.0) < 1e-12


def test_philox_known_answers():
    """Known answers of Philox4x32-10, from the generator's published test vectors."""
    def words(seed, counter_low, offset):
        bits = R.philox_bits(8, seed, offset, counter_low * 8)
        return [int(bits[2 * k]) | int(bits[2 * k + 1]) << 16 for k in range(4)]
    assert words(0, 0, 0) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    ones = (1 << 64) - 1
    assert words(ones, ones, ones) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]


def test_refusals_of_the_python_entry_points():
    import efgs
    x, w, y = torch.zeros(4, 8), torch.zeros(9, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match='GPU device'):
        efgs.linear_cross_entropy(x, w, y)
    with pytest.raises(ValueError, match='two dimensions'):
        efgs.linear_cross_entropy(x, w[0], y)
    with pytest.raises(ValueError, match='columns'):
        efgs.linear_cross_entropy(x[:, :7], w, y)
    with pytest.raises(ValueError, match='shape without its columns'):
        efgs.linear_cross_entropy(x, w, y[:3])
    with pytest.raises(ValueError, match='int32 or int64'):
        efgs.linear_cross_entropy(x, w, y.float())
    with pytest.raises(ValueError, match="table's type"):
        efgs.linear_cross_entropy(x.half(), w, y)
    with pytest.raises(ValueError, match='float32, bfloat16 or float16'):
        efgs.linear_cross_entropy(x.double(), w.double(), y)
    with pytest.raises(ValueError, match='GPU device'):
        efgs.dropout(x, 0.5)
    with pytest.raises(ValueError, match='GPU device'):
        efgs.dropout(x, 0.5, seed=1)
    with pytest.raises(ValueError, match='needs a seed'):
        efgs.dropout(x, 0.5, offset=1)
    with pytest.raises(ValueError, match='offset must lie'):
        efgs.dropout(x, 0.5, seed=1, offset=-1)
    with pytest.raises(ValueError, match='GPU device'):
        efgs.balance_loss(x, y)
    with pytest.raises(ValueError, match='int32 or int64'):
        efgs.balance_loss(x, y.float())
    with pytest.raises(ValueError, match='shape without its experts'):
        efgs.balance_loss(x, y[:3])
    with pytest.raises(ValueError, match='last dimension'):
        efgs.balance_loss(torch.zeros(4, 0), y)


def _entropy(**how):
    from efgs import _lib
    e = _lib.Entropy(None, None, None, 4, 9, 8, 8, 8, 8, 0, 2, 1.0)
    for k, v in how.items():
        setattr(e, k, v)
    return e


@pytest.mark.parametrize('how', [dict(n=-1), dict(rows=1 << 31), dict(columns=-2), dict(columns=(1 << 22) + 1), dict(target_bytes=2), dict(type=3), dict(reduction=3), dict(scale=float('inf')),
                                 dict(scale=float('nan')), dict(table_stride=-1), dict(n=1 << 30, columns=1 << 30), dict(rows=1 << 30, columns=1 << 30)])
def test_refusals_of_the_c_cross_entropy(how):
    from efgs import _lib
    e = _entropy(**how)
    alloc = _lib.ALLOC_FN(lambda ctx, n: None)
    assert _lib.lib.efgs_linear_cross_entropy_saved_bytes(ctypes.byref(e)) == -1
    assert _lib.lib.efgs_linear_cross_entropy_forward(ctypes.byref(e), None, None, alloc, None, None) != 0
    assert _lib.lib.efgs_linear_cross_entropy_backward(ctypes.byref(e), None, None, None, None, alloc, None, None) != 0
    assert _lib.lib.efgs_last_error()


def test_null_pointers_and_failed_allocations_of_the_c_entry_points():
    from efgs import _lib
    lib, alloc, one = _lib.lib, _lib.ALLOC_FN(lambda ctx, n: None), ctypes.c_void_p(256)
    assert lib.efgs_linear_cross_entropy_saved_bytes(None) == -1
    assert lib.efgs_linear_cross_entropy_forward(None, one, None, alloc, None, None) != 0
    assert lib.efgs_linear_cross_entropy_forward(ctypes.byref(_entropy()), one, None, alloc, None, None) != 0
    full = _entropy(features=one, table=one, targets=one)
    assert lib.efgs_linear_cross_entropy_forward(ctypes.byref(full), None, None, alloc, None, None) != 0
    assert lib.efgs_linear_cross_entropy_forward(ctypes.byref(full), one, None, alloc, None, None) != 0 and b'allocation' in lib.efgs_last_error()
    assert lib.efgs_linear_cross_entropy_backward(ctypes.byref(full), one, one, one, one, alloc, None, None) != 0 and b'allocation' in lib.efgs_last_error()
    assert lib.efgs_linear_cross_entropy_backward(ctypes.byref(full), None, one, one, one, alloc, None, None) != 0
    assert lib.efgs_dropout(None, None, None, 4, 0, 0.5, 0, None, 0, None) != 0
    assert lib.efgs_dropout(one, None, one, -1, 0, 0.5, 0, None, 0, None) != 0
    for p in (-0.1, 1.1, float('nan')):
        assert lib.efgs_dropout(one, None, one, 4, 0, p, 0, None, 0, None) != 0
    assert lib.efgs_dropout(one, None, one, 4, 7, 0.5, 0, None, 0, None) != 0
    assert lib.efgs_dropout(None, None, None, 0, 0, 0.5, 0, None, 0, None) == 0
    for experts in (0, 8193):
        assert lib.efgs_balance_loss_forward(one, one, 8, 4, experts, 1, 0, one, one, one, alloc, None, None) != 0
    assert lib.efgs_balance_loss_forward(one, one, 8, 4, 8, 1, 0, one, one, one, alloc, None, None) != 0 and b'allocation' in lib.efgs_last_error()
    assert lib.efgs_balance_loss_forward(one, one, 3, 4, 8, 1, 0, one, one, one, alloc, None, None) != 0
    for chosen in (-1, 65537):
        assert lib.efgs_balance_loss_forward(one, one, 8, 4, 8, chosen, 0, one, one, one, alloc, None, None) != 0
        assert lib.efgs_balance_loss_backward(one, one, 8, 4, 8, chosen, 0, one, one, one, None) != 0
    assert lib.efgs_balance_loss_forward(one, None, 8, 4, 8, 1, 0, one, one, one, alloc, None, None) != 0
    assert lib.efgs_balance_loss_backward(one, one, 8, 4, 8, 1, 0, None, one, one, None) != 0
