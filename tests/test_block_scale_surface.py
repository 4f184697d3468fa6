"""The block-scaled launchers through the C++ host surface (tests/cpp/test_block_scale.cpp)."""
import pytest

from test_cpp_surface import _run


@pytest.mark.gpu
def test_block_scale_launchers_of_the_cpp_surface():
    assert _run("test_block_scale").count("PASS ") == 2
