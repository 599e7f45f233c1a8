"""What the serving example refuses before it runs anything."""
import pytest

from flash_attention_factory_amd import serving_example as E


@pytest.mark.parametrize("prompts,answer,piece,what", [
    ([[3, 4], []], 2, 256, "at least one token"), ([[1] * 60], 6, 256, "at most 64"), ([[1]], 2, 0, "a piece one"),
    ([[1] * 40, [2] * 40, [3] * 40], 2, 256, "more blocks"),
])
def test_requests_that_cannot_be_served(prompts, answer, piece, what):
    server = E.Server(2, 64, layers=1, device="cpu")
    with pytest.raises(ValueError, match=what):
        server.serve(prompts, answer, piece)
    assert len(server.free) == 8


def test_nothing_to_serve():
    server = E.Server(1, 32, layers=1, device="cpu")
    assert server.serve([], 3) == [] and server.serve([[1, 2]], 0) == [[]]
