"""The long-context serving example: its parts run together, the bookkeeping
ends where it should, and the 4-bit steps stay as near to attention over
unquantised keys and values as 4 bits allow (a step of a 16-level quantiser
over a Gaussian's range of about 5 deviations is off by 0.1 deviations rms,
the value's share of the result's norm, and the keys' errors move the
probabilities by about as much again: 0.15 together)."""
import pytest

pytestmark = pytest.mark.gpu


def test_serve_packed_example():
    from decode import Shape
    from serve_packed import serve
    r = serve(Shape(layers=1), seqs=3, prompt=150, chunk=40, steps=12, limit=196, keep=160, recent=32)
    assert r["evictions"] == 1 and r["finite"]
    assert r["rel_distance"] < 0.15
    assert r["lengths"][0] == 160 + 12 - 6 and r["seen"] == [n + 40 + 12 for n in r["lens"]]
