"""stack_expert_modules on modules whose weights one stack cannot hold as they are: refused, with the modules left as
they were."""
import pytest
import torch

from nano_ktrans_b200 import stack_expert_modules


class Expert(torch.nn.Module):
    def __init__(self, dtype=torch.bfloat16, hidden=4, inter=3, device="cpu"):
        super().__init__()
        for n, (o, i) in (("w1", (inter, hidden)), ("w3", (inter, hidden)), ("w2", (hidden, inter))):
            setattr(self, n, torch.nn.Linear(i, o, bias=False, dtype=dtype, device=device))


def state(mods):
    return [(p, p.data_ptr(), p.dtype) for m in mods for p in m.parameters()]


@pytest.mark.parametrize("odd", [dict(dtype=torch.float32), dict(dtype=torch.float16), dict(hidden=6), dict(inter=5),
                                 dict(device="meta")])
def test_experts_that_differ(odd):
    mods = [Expert(), Expert(**odd), Expert()]
    before = state(mods)
    with pytest.raises(ValueError, match="differ"):
        stack_expert_modules(mods)
    assert state(mods) == before


def test_one_projection_that_differs():
    mods = [Expert(), Expert()]
    mods[1].w2.double()
    with pytest.raises(ValueError, match="differ"):
        stack_expert_modules(mods)


def test_an_expert_given_twice():
    """Its one parameter cannot be a view of two places: an update would reach only one of them."""
    a, b = Expert(), Expert()
    with pytest.raises(ValueError, match="share"):
        stack_expert_modules([a, b, a])
    b.w3.weight = a.w3.weight
    with pytest.raises(ValueError, match="share"):
        stack_expert_modules([a, b])
    c = Expert()
    c.w1.weight = c.w3.weight
    with pytest.raises(ValueError, match="share"):
        stack_expert_modules([c])


def test_weights_that_are_not_parameters():
    """A weight worked out from others (a parametrisation, a wrapper's property) cannot be a view of the stack."""
    m = Expert(torch.float32)
    torch.nn.utils.parametrizations.weight_norm(m.w1)
    with pytest.raises(ValueError, match="linear layers"):
        stack_expert_modules([m])

    class Wrapped(torch.nn.Module):
        def __init__(self, base):
            super().__init__()
            self.base = base

        @property
        def weight(self):
            return self.base.weight

    m = Expert()
    m.w2 = Wrapped(m.w2)
    with pytest.raises(ValueError, match="linear layers"):
        stack_expert_modules([m])
