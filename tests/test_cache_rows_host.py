"""Which rows the caches take for a chunk's packed ones (no GPU is needed)."""
import pytest
import torch

from libero_hip.episodes import Chunk, Layers
from libero_hip.room import DeviceChunk


def ragged(counts):
    import numpy as np
    counts = np.asarray(counts)
    start = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
    return Chunk(counts, start)


def test_even_rows_of_a_device_chunk_are_packed():
    chunk = DeviceChunk(torch.zeros(3, dtype=torch.int32), 6, 3, (2, 3))
    x = torch.randn((2, 3, 4, 8))
    assert Layers._packed(chunk, x).shape == (6, 4, 8) and Layers._packed(chunk, x).data_ptr() == x.data_ptr()
    packed = x.flatten(0, 1)
    assert Layers._packed(chunk, packed) is packed
    lse = torch.zeros((2, 3, 4))
    assert Layers._packed(chunk, lse, 1).shape == (6, 4)


@pytest.mark.parametrize('chunk', [ragged([1, 3]), DeviceChunk(torch.zeros(3, dtype=torch.int32), 6, 3, (6,))])
def test_padded_rows_are_refused(chunk):
    """A chunk of one and three tokens in rows of two times three: the padding is no world's."""
    with pytest.raises(ValueError, match='packed'):
        Layers._packed(chunk, torch.zeros((2, 3, 4, 8)))
    packed = torch.zeros((chunk.tokens, 4, 8))
    assert Layers._packed(chunk, packed) is packed


def test_rows_of_other_shapes_are_refused():
    chunk = DeviceChunk(torch.zeros(3, dtype=torch.int32), 6, 3, (2, 3))
    for shape in ((3, 2, 4, 8), (1, 6, 4, 8), (6, 1, 4, 8), (2, 4, 4, 8)):
        with pytest.raises(ValueError, match=r'\(2, 3, '):
            Layers._packed(chunk, torch.zeros(shape))


def test_even_chunks_keep_their_rows():
    import numpy as np
    x = torch.zeros((2, 3, 4, 8))
    assert Layers._packed(Chunk(np.array([3, 3]), None), x) is x
