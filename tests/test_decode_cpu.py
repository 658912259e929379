"""The host side of generation over the paged cache: what it refuses before anything reaches a GPU."""
from types import SimpleNamespace

import pytest
import torch


def _decoder(**kw):
    """A decoder without buffers; whatever comes after the checks fails for want of an attribute."""
    from distrain_b200.models.decode import PagedDecoder
    dec = PagedDecoder.__new__(PagedDecoder)
    dec.eng, dec.dev = SimpleNamespace(V=100), torch.device("cpu")
    dec.max_prompt, dec.max_new, dec.max_batch, dec.n, dec.length = 8, 4, 2, 2, 0
    dec.__dict__.update(kw)
    return dec


@pytest.mark.parametrize("bad", [100, -1, 2 ** 31 - 1, 10 ** 12])
def test_ids_outside_the_vocabulary_are_refused(bad):
    """An id past the embedding's rows would be read out of range on the GPU."""
    dec = _decoder()
    with pytest.raises(ValueError, match="vocabulary"):
        dec.prefill([1, 2, bad])
    with pytest.raises(ValueError, match="vocabulary"):
        dec.step([99, bad])
    with pytest.raises(AttributeError):  # ids of the vocabulary pass
        dec.prefill([0, 99])
