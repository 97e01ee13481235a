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


def test_evict_takes_masses_as_long_as_either_cache(serve):
    """The layout that attention over `into` wants for its masses is [seqs, kv_heads, into.capacity]."""
    def cache(capacity):
        c = serve.KV4Cache.__new__(serve.KV4Cache)
        c.L, c.seqs, c.kv_heads, c.head_dim, c.capacity, c.h = serve.serve_lib(), 2, 3, 64, capacity, 1
        c.close = lambda: None
        return c
    a = lambda *shape, dtype="float32": serve.DeviceArray(4096, shape, dtype)  # noqa: E731
    c, into, at, kept = cache(64), cache(100), a(2, dtype="int32"), a(2, 3, 32, dtype="int32")
    for n in (32, 64, 100):
        assert c.evict_call(into, at, at, a(2, 3, 64), a(2, 3, n), kept, keep=32)._keep[0].new_mass_ld == n
    for bad in (a(2, 3, 31), a(2, 3, 33), a(3, 2, 100), a(2, 3, 99), a(600)):
        with pytest.raises(ValueError):
            c.evict_call(into, at, at, a(2, 3, 64), bad, kept, keep=32)
    small = cache(16)
    with pytest.raises(ValueError):
        c.evict_call(small, at, at, a(2, 3, 64), a(2, 3, 16), kept, keep=32)
