"""The status calls for what never was on a GPU: no finding, and no need of a device."""
import torch

import ascend_kernel_b200 as ak
from ascend_kernel_b200.moe_layer import MoELayer
from tests.test_moe_layer import TorchRowOps, small_case


def test_a_host_device_has_no_findings():
    for clear in (False, True):
        assert ak.last_status(torch.device("cpu"), clear=clear) == (0, 0)
        assert ak.last_status("cpu", clear=clear) == (0, 0)
    ak.check_status("cpu")


def test_a_layer_on_host_tensors_reports_none():
    c = small_case()
    layer = MoELayer(c["w13"], c["s13"], c["o13"], c["w2"], c["s2"], c["o2"], c["E"], c["top_k"], None, TorchRowOps)
    layer.forward(c["x"], c["logits"])
    assert layer.read_status() == (0, 0)
