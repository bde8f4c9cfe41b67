"""Learning rates and weight decays of AdamW that change between steps."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def values(n, seed):
    return torch.randn(n, generator=torch.Generator().manual_seed(seed)).cuda()


def make(st, lr=1e-3, wd=0.0):
    return st.AdamW([values(50, 1), values(300, 2)], [values(50, 3), values(300, 4)], lr=lr, weight_decay=wd)


@pytest.mark.parametrize("value", [1e-4, 1, 0, np.float32(0.5), np.float64(1e-2), [1e-4, 1e-2], (1e-4, 0), np.array([0.1, 0.2])])
@pytest.mark.parametrize("name", ["lr", "weight_decay"])
def test_rates_are_set_as_they_are_given_to_begin_with(pkg, name, value):
    """One value or one per tensor, at any time: the steps that follow are those of an optimizer that had it from there on."""
    st = pkg.strategy
    a = make(st, 0.1, 0.2)
    a.step()
    b = st.AdamW([p.clone() for p in a.params], a.grads, lr=value if name == "lr" else 0.1, weight_decay=0.2 if name == "lr" else value,
                 moments=[st.Moments(m.exp_avg.clone(), m.exp_avg_sq.clone()) for m in a.moments])
    b.step_count = 1
    setattr(a, name, value)
    assert getattr(a, name) == getattr(b, name) and len(getattr(a, name)) == 2
    a.step(), b.step()
    assert all(torch.equal(x, y) for x, y in zip(a.params, b.params))
    assert not torch.equal(a.params[0], make(st).params[0])


def test_rates_of_another_length_are_refused(pkg):
    st = pkg.strategy
    opt = make(st)
    before = [p.clone() for p in opt.params]
    for name in ("lr", "weight_decay"):
        for bad in ([0.1], [0.1] * 3, []):
            with pytest.raises(RuntimeError, match="values for 2 tensors"):
                setattr(opt, name, bad)
        for change in (lambda x: x.append(0.1), lambda x: (x.pop(), x.pop())):
            change(getattr(opt, name))
            with pytest.raises(RuntimeError, match="values for 2 tensors"):
                opt.step()
        setattr(opt, name, 0.1)
    assert opt.step_count == 0 and all(torch.equal(a, b) for a, b in zip(before, opt.params))


def test_a_scheduler_changes_one_entry(pkg):
    st = pkg.strategy
    opt = make(st, [0.1, 0.2])
    st.ExponentialLR(opt, 0.5, 1).step()
    assert opt.lr == [0.1, 0.1]
    st.ExponentialLR(opt, 0.5).step()
    assert opt.lr == [0.05, 0.05]
    start = [p.clone() for p in opt.params]
    opt.step()
    # the first step is lr times the gradient's sign (and eps): the change of parameters of up to 4 is rounded by 2^-23, so 1e-5 of lr = 0.05
    assert all(((a - b).abs() - 0.05).abs().median() < 1e-5 * 0.05 + 2.0 ** -22 for a, b in zip(start, opt.params))
