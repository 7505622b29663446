"""CPU: construction, names and flat layout of a policy with the gated core."""
import pickle

import pytest
import torch


class Discrete(object):
    n = 6


class Box(object):
    shape = (3,)


@pytest.mark.parametrize('shape,space,hidden', [((11,), Box(), 64), ((4, 84, 84), Discrete(), 512)])
def test_gated_policy_layout(shape, space, hidden):
    from a2c_ppo_acktr.model import Policy
    pol = Policy(shape, space, base_kwargs={'recurrent': 'gated'})
    assert pol.is_recurrent and pol.recurrent_hidden_state_size == hidden
    names = [n for n, _ in pol.named_parameters()]
    core = ['base.core.in_proj.weight', 'base.core.in_proj.bias', 'base.core.out_proj.weight', 'base.core.out_proj.bias']
    assert names[:4] == core and not any('gru' in n for n in names)
    lo, hi = pol.flat_params.data_ptr(), pol.flat_params.data_ptr() + 4 * pol.flat_params.numel()
    assert all(lo <= p.data_ptr() < hi for p in pol.parameters())
    gates = pol.base.core.in_proj.bias.detach()[:hidden]
    assert abs(float(torch.sigmoid(gates[0])) - 0.5) < 1e-6 and abs(float(torch.sigmoid(gates[-1])) - 127 / 128) < 1e-6
    again = pickle.loads(pickle.dumps(pol))
    assert torch.equal(again.flat_params, pol.flat_params)
    with pytest.raises(RuntimeError):                     # no CPU path
        pol.get_value(torch.zeros((2,) + shape), torch.zeros(2, hidden), torch.ones(2, 1))


def test_other_values_are_refused():
    from a2c_ppo_acktr import algo
    from a2c_ppo_acktr.model import Policy
    with pytest.raises(ValueError):
        Policy((11,), Box(), base_kwargs={'recurrent': 'lstm'})
    pol = Policy((11,), Box())
    with pytest.raises(ValueError):
        algo.PPO(pol, 0.2, 1, 1, 0.5, 0.0, lr=1e-3, eps=1e-5, state_bits=8)
    with pytest.raises(ValueError):
        algo.PPO(pol, 0.2, 1, 1, 0.5, 0.0, lr=1e-3, eps=1e-5, weight_decay=-1.0)


def test_what_was_falsy_or_truthy_still_is():
    from a2c_ppo_acktr.model import Policy
    assert not Policy((11,), Box(), base_kwargs={'recurrent': None}).is_recurrent
    assert not Policy((11,), Box(), base_kwargs={'recurrent': 0}).is_recurrent
    assert hasattr(Policy((11,), Box(), base_kwargs={'recurrent': 1}).base, 'gru')


@pytest.mark.parametrize('value', ['gru', 'yes', 'True', '1'])
def test_strings_are_taken_by_their_truth(value):
    from a2c_ppo_acktr.model import Policy
    torch.manual_seed(3)
    a = Policy((11,), Box(), base_kwargs={'recurrent': value})
    torch.manual_seed(3)
    b = Policy((11,), Box(), base_kwargs={'recurrent': True})
    assert hasattr(a.base, 'gru') and torch.equal(a.flat_params, b.flat_params)
    assert not Policy((11,), Box(), base_kwargs={'recurrent': ''}).is_recurrent


def test_the_gru_is_what_it_was():
    """same initialiser calls in the same order: a seed gives the same GRU policy with and without the new core in the package"""
    from a2c_ppo_acktr.model import Policy
    torch.manual_seed(7)
    a = Policy((11,), Box(), base_kwargs={'recurrent': True})
    assert [n for n, _ in a.named_parameters()][0] == 'base.gru.weight_ih_l0' and a.base.rnn is a.base.gru
