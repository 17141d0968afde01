"""CPU: host-side rules of the transformer-layer operators and modules at their edges (no launch)."""
import copy

import torch

from mo_yolo_amd import modules


# ---------------------------------------------------------------------------------------------------------------- prepared weights
def _weights(layer):
    return layer._prepared(torch.device("cpu"), torch.float32, layer._build)["w"][:, :layer.cin]      # (the padded copy: "wf" is the parameter itself here)


def test_prepared_weights_follow_the_parameters():
    lin = modules._Linear(8, 12)
    first = _weights(lin)
    assert torch.equal(first, lin.weight) and lin._prepared(torch.device("cpu"), torch.float32, lin._build) is lin._prep.data
    with torch.no_grad():
        lin.weight.add_(1.0)                                                   # in place: the version
    assert torch.equal(_weights(lin), lin.weight)
    old = lin.weight.data
    for _ in range(4):                                                         # other memory, twice between two calls: never the address of what was prepared
        lin.weight.data = lin.weight.data.clone() + 1.0
        lin.weight.data = lin.weight.data.clone() + 1.0
        assert torch.equal(_weights(lin), lin.weight)
    lin.weight.data = old
    assert torch.equal(_weights(lin), old)
    lin.weight.data.mul_(2.0)                                                  # through .data nothing counts it
    modules.forget_prepared(torch.nn.Sequential(lin))
    assert torch.equal(_weights(lin), lin.weight)


def test_a_module_in_training_prepares_its_weights_in_every_call():
    lin = modules._Linear(8, 12)
    with torch.no_grad():
        lin._trains()                                                          # (the differentiable form without a gradient: not training)
    keeps = lambda: lin._prepared(torch.device("cpu"), torch.float32, lin._build) is lin._prepared(torch.device("cpu"), torch.float32, lin._build)  # noqa: E731
    assert keeps()
    lin._trains()
    for _ in range(3):
        lin.weight.data.add_(1.0)                                              # as a replayed graph does: no version
        lin.bias.data.add_(1.0)
        got = lin._prepared(torch.device("cpu"), torch.float32, lin._build)
        assert torch.equal(got["w"][:, :8], lin.weight) and torch.equal(got["b"], lin.bias) and not keeps()
    lin.weight.requires_grad_(False)
    assert not keeps()                                                         # (its bias still trains)
    lin.requires_grad_(False)
    assert keeps() and torch.equal(_weights(lin), lin.weight)
    lin.load_state_dict({"weight": torch.ones(12, 8), "bias": torch.zeros(12)})
    assert torch.equal(_weights(lin), torch.ones(12, 8))


def test_copies_of_a_module_prepare_their_own_weights():
    lin = modules._Linear(8, 12)
    _weights(lin)
    lin._trains()
    twin = copy.deepcopy(lin)
    assert twin._prep is not lin._prep and twin._prep.data is None and not twin._prep.trained
    with torch.no_grad():
        twin.weight.add_(1.0)
    assert torch.equal(_weights(twin), twin.weight) and torch.equal(_weights(lin), lin.weight)


def test_the_differentiable_forms_say_that_they_train():
    """Every holder of parameters that the differentiable forms of the layer and of QIM use."""
    import inspect
    for cls in (modules._Linear, modules._MHA):
        assert "self._trains()" in inspect.getsource(cls.forward_train)
    held = [m for top in (modules.MOTRDecoderLayer(), modules.QueryInteractionModule(None, 256, 256)) for m in top.modules() if isinstance(m, modules._ParamModule)]
    assert held and all(isinstance(m, (modules._Linear, modules._MHA)) for m in held)
