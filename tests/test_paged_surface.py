"""The paged cache's launchers and adjusted logits through the C++ host surface (tests/cpp/test_paged_cache.cpp)."""
import pytest

from test_cpp_surface import _run


@pytest.mark.gpu
def test_paged_launchers_of_the_cpp_surface():
    assert _run("test_paged_cache").count("PASS ") == 2
