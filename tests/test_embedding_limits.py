"""What the embedding's backward cannot launch is refused with its other arguments,
before any device work: the refusal comes first, whatever else is missing."""
import pytest

from spilltune_amd import _lib


@pytest.mark.parametrize("dtype,H,accumulate", [(1, 1 << 20, 0), (1, 1 << 20, 1), (0, 1 << 20, 0),
                                                (1, 1 << 12, 0)])
def test_too_many_threads_are_refused_first(dtype, H, accumulate):
    with pytest.raises(ValueError, match="launch"):
        _lib.call("st_embedding_bwd", None, None, 0, (1 << 31) - 1, 8, H, 1.0, -1, 16, dtype, accumulate,
                  None, 0, None)
