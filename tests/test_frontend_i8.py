"""The front end's own refusals of the 8-bit layers (no device needed: they come
before the library is called)."""
import pytest

import zkml_amd as z


class Buffer:
    ptr, nbytes = 1 << 20, 4096


@pytest.mark.parametrize("slots", [2, 4])
def test_an_order_of_several_slots_needs_the_number_of_tokens(monkeypatch, slots):
    """x's rows follow from nothing else that is given then: the default of one row
    for each of y's would let a bad order read slots times past x."""
    def called():
        raise AssertionError("the library was called")

    monkeypatch.setattr(z, "lib", called)
    ctx, d = object.__new__(z.Context), Buffer()
    ctx.h = None
    with pytest.raises(z.ZkError, match="tokens"):
        ctx.i8_matmul_experts(d, d, d, 8, 2, 3, 16, d, order=d, slots=slots)
