"""The table of cosines and sines through a model's conversions."""
import copy

import pytest
import torch

import tokenweave_amd as tw


class Model(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.rotary = tw.RotaryPositions(64, 32, 3000)
        self.proj = torch.nn.Linear(4, 4)


@pytest.mark.parametrize("convert", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(),
                                     lambda m: m.to("cpu", torch.float16), lambda m: copy.deepcopy(m).half().float(),
                                     lambda m: m.half().bfloat16().half()])
def test_a_models_type_leaves_the_table_in_fp32(convert):
    """The ops take a table of fp32, and 16 bits hold no position past some hundreds apart."""
    model = Model()
    want = model.rotary.cos_sin.clone()
    model = convert(model)
    assert model.rotary.cos_sin.dtype == torch.float32 and torch.equal(model.rotary.cos_sin, want)
    assert dict(model.rotary.named_buffers())["cos_sin"] is model.rotary.cos_sin and not model.rotary.state_dict()


def test_other_conversions_reach_the_table():
    model = Model().to("meta").bfloat16()
    assert model.rotary.cos_sin.device.type == "meta" and model.rotary.cos_sin.dtype == torch.float32
    model = Model()
    model._apply(lambda t: t + 1)
    assert model.proj.weight.dtype == torch.float32 and float(model.rotary.cos_sin[0, 0].detach()) == 2.0
