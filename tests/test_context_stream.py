"""The stream that a context is given (no GPU: what is refused before the device is reached)."""
import pytest

import arf_amd


def test_the_default_stream_is_refused():
    # (an address of 0 would make a stream of the context's own, which the caller's work is not ordered with)
    with pytest.raises(ValueError, match="stream 0"):
        arf_amd.Context(0, stream=0)
