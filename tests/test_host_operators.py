"""GPU: the paged-cache operators through the C++ host side, by the C++ test program of that name."""
import pytest

from test_host_cpp import _run


@pytest.mark.gpu
def test_host_operators():
    _run("host_operators_test", 120)
