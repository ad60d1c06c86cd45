"""checkpoint_linears' handle, on the CPU."""
import types

import torch

from sandmuon_amd import act8


def test_close_leaves_a_forward_that_was_put_over_its_own():
    model = torch.nn.Sequential(torch.nn.Linear(4, 4), torch.nn.Linear(4, 4))
    handle = act8.checkpoint_linears(model)
    mine = types.MethodType(lambda module, x: x + 1, model[0])
    model[0].forward = mine
    handle.close()
    assert model[0].__dict__["forward"] is mine and "forward" not in model[1].__dict__
    assert torch.equal(model[0](torch.zeros(2, 4)), torch.ones(2, 4))
    handle.close()
    # and one taken away already
    handle = act8.checkpoint_linears(model)
    assert list(handle.modules) == ["1"]
    del model[1].forward
    handle.close()
