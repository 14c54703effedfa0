"""CPU: the helper that says to autograd that a list of tensors has been written (neat_host_written)."""
import torch

from neat_amd import lib


def test_versions_rise_and_what_has_none_is_passed_over():
    with torch.inference_mode():
        frozen = torch.zeros(3)
    ps = [torch.nn.Parameter(torch.zeros(2)), torch.zeros(4), frozen]
    view = ps[1][1:]
    before = [ps[0]._version, ps[1]._version]
    lib.written()(ps)
    assert [ps[0]._version, ps[1]._version] == [b + 1 for b in before] and view._version == ps[1]._version
    lib.written()([])
    lib.written()([None, 3.0])
    lib.written()(tuple(ps))                        # no list: nothing is touched
    assert ps[0]._version == before[0] + 1
