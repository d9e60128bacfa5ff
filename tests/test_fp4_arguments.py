"""CPU: arguments of the microscaled operators that contradict one another."""
import pytest
import torch

import int4linear_b200 as L
from int4linear_b200 import fp4


def test_quantize_refuses_a_format_that_is_not_its_outputs():
    cpu = torch.device("cpu")
    outs = {fmt: fp4.Fp4Matrix._new(4, 64, fmt, None, cpu) for fmt in fp4.FORMATS}
    for fmt, out in outs.items():
        assert fp4._wanted_format(None, out) == fmt and fp4._wanted_format(fmt, out) == fmt
        for other in [f for f in fp4.FORMATS if f != fmt] + ["fp4"]:
            with pytest.raises(ValueError):
                fp4._wanted_format(other, out)
    assert fp4._wanted_format(None, None) == "mxfp4" and fp4._wanted_format("nvfp4", None) == "nvfp4"


@pytest.mark.gpu
def test_quantize_into_an_output_of_another_format(cuda):
    x = torch.randn((4, 64), device=cuda)
    for fmt, other in (("mxfp4", "nvfp4"), ("nvfp4", "mxfp4")):
        out = L.quantize_fp4(x, fmt)
        codes = out.codes.clone()
        with pytest.raises(ValueError):
            L.quantize_fp4(-x, other, out=out)
        assert torch.equal(out.codes, codes)
        assert L.quantize_fp4(x, fmt, out=out) is out and L.quantize_fp4(x, out=out) is out
    assert L.quantize_fp4(x).format == "mxfp4"
