"""The example layer: router, routed experts and shared expert together, and the router's gradient in a step of the gate.

Its bf16 roundings (both shared products, their SwiGLU, the routed sum, the final sum) are each half a unit of 2^-7,
0.17% of a value on average; six of them side by side stay below 1%."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "w4_moe_layer.py")


@pytest.mark.parametrize("tokens", [1, 16, 200])
def test_example(pkg, tokens):
    spec = importlib.util.spec_from_file_location("w4_moe_layer", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.main(tokens) < 0.01
    assert pkg.device_status(reset=True) == 0
