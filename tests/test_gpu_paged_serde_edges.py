"""Chunks from a paged cache: what must not be stored."""
import pytest
import torch

from test_gpu_paged_serde import D, H, L, PAGE, blob, codec, new_pages  # noqa: F401 (codec: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_tokens_without_a_slot_are_not_stored(codec, index):  # noqa: F811
    """Padding and slots outside the cache leave rows of a blob as they are, with whatever its memory had: another request's keys, say."""
    from cachegen_b200 import paged
    ser, de, fmt = codec
    pages = new_pages(fmt, 4)
    pages.copy_(torch.randn(pages.shape, generator=torch.Generator().manual_seed(1)).half())
    good = torch.arange(40, device="cuda", dtype=index)
    for bad in (-1, -2, 4 * PAGE, 2 ** 31 - 1):
        slots = good.clone()
        slots[17] = bad
        for call in (ser.encode_paged, ser.to_bytes_paged):
            with pytest.raises(RuntimeError, match="slots"):
                call(pages, slots)
    last = torch.arange(4 * PAGE - 40, 4 * PAGE, device="cuda", dtype=index)
    assert de.from_bytes(ser.to_bytes_paged(pages, last)).numel() == 2 * L * 40 * H * D
    paged.check_status()
