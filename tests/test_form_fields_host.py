"""A form's numbers as the C structure takes them."""

from __future__ import annotations

from types import SimpleNamespace

import pytest


@pytest.mark.parametrize("name", ["softcap", "scale"])
def test_numbers_that_float32_takes_for_zero_are_refused(name) -> None:
    """0 stands for no cap and for the default scale, which a tiny number does not mean."""
    from microserve_b200.attention import _PACK_FORM, AttentionForm

    batch = SimpleNamespace(n_tokens=1, max_q=1, batch_size=1)
    for value in (1e-46, 5e-324):
        with pytest.raises(ValueError, match="float32"):
            AttentionForm(**{name: value}).fields(0, 4, batch)
    fields = AttentionForm(**{name: 1e-45}).fields(0, 4, batch)
    zero = AttentionForm().fields(0, 4, batch)
    assert _PACK_FORM(*fields) != _PACK_FORM(*zero)
