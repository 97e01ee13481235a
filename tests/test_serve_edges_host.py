"""What the operators of voxtral_b200_serve.h refuse at the edges of their sizes and arrays. No GPU."""
import sys

import pytest


@pytest.fixture(scope="module")
def serve(pkg):
    return sys.modules[pkg.__name__ + ".serve"]


@pytest.mark.parametrize("sizes", [(60973, 16381, 128, 135800960), (65535, 16384, 256, 1 << 30), (32768, 16384, 64, 1 << 30), (1024, 1024, 128, 8192)])
def test_open_refuses_rows_whose_bytes_pass_64_bits(serve, sizes):
    """Each size within its own limit; the first one's product wraps to 105 MB."""
    with pytest.raises(RuntimeError, match="2\\^40 bytes"):
        serve.KV4Cache(*sizes)
