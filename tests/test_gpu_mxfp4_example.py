"""examples/mxfp4_mlp.py runs, and its errors are those of the formats."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", ["1", "40"])
def test_mlp(rows):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "mxfp4_mlp.py")
    spec = importlib.util.spec_from_file_location("mxfp4_mlp", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    off = module.main(["--rows", rows, "--hidden", "1024", "--inner", "1376"])
    # E4M3 keeps 3 mantissa bits (about 0.03 a value), E2M1 one (about 0.12), through two projections and a product
    assert off["e4m3"][1] < 0.08 and off["mxfp4"][1] < 0.35
    assert off["e4m3"][1] < off["mxfp4"][1]
