"""What the serving operators' host code refuses at the ends of its arguments' range (on the CPU)."""
import pytest

from test_serving_host import INVALID, OK, Host, call, lib  # noqa: F401


@pytest.mark.parametrize("op", ["decode", "prefill"])
def test_scales_at_the_ends_of_f32(lib, op):  # noqa: F811
    """Scores are taken in units of log2(e): a scale that passes f32 with it is refused, others run."""
    host = Host(lib)
    for scale in (3.4e38, 2.4e38, 2.36e38):
        for into in (True, False):
            assert call(host, op, into, scale=scale) == INVALID and b"log2" in lib.host_message()
    assert not host.launches()
    for scale in (2.0 ** 127, 2.35e38, 1e-30, 1e-38, 1e-45, 0.0, -0.0, -1.0, -3.4e38):
        assert call(host, op, scale=scale) == OK and host.launches()
