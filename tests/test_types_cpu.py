"""Tensor types that the library does not know are refused with its own error, before anything is called."""
import pytest
import torch

KNOWN = {torch.float32: "DT_F32", torch.float16: "DT_F16", torch.bfloat16: "DT_BF16", torch.int32: "DT_S32"}


@pytest.mark.parametrize("dtype", [torch.float64, torch.int64, torch.int16, torch.uint8, torch.int8, torch.bool,
                                   torch.float8_e4m3fn, torch.complex64])
def test_unknown_types_raise_the_librarys_error(pkg, dtype):
    with pytest.raises(pkg.W8A8Error, match=str(dtype)):
        pkg._dt(torch.zeros(1, dtype=dtype))


@pytest.mark.parametrize("dtype", KNOWN)
def test_known_types_have_the_headers_codes(pkg, dtype):
    assert pkg._dt(torch.zeros(1, dtype=dtype)) == getattr(pkg, KNOWN[dtype])
