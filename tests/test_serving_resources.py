"""No kernel of the operators over caller-held caches keeps registers in scratch memory."""
from test_kernel_resources import scratch  # noqa: F401 (a fixture)


def test_serving_kernels_keep_no_registers_in_scratch(scratch):  # noqa: F811
    names = ("cache_write", "cache_read", "shared_attend", "alone_attend", "shared_join", "verify_")
    kernels = {n: b for n, b in scratch.items() if any(x in n for x in names)}
    for x in names:
        assert any(x in n for n in kernels), x
    assert not {n: b for n, b in kernels.items() if b}
