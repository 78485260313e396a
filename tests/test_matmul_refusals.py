"""Products with packed weights: further calls that the Python layer refuses before a device is touched."""
import pytest


@pytest.mark.parametrize("name", ["float32", "int8", "int32", "float16", "bfloat16"])
def test_packed_weights_are_bytes(name):
    """A tensor of the right size in bytes whose elements are something else is not read as blocks."""
    import torch
    import gguf_amd as g
    dt = getattr(torch, name)
    w = torch.zeros(4 * 144, dtype=torch.uint8).view(dt)
    x, y = torch.zeros(2, 256), torch.zeros(2, 4)
    with pytest.raises(TypeError):
        g.matvec(12, y, w, x)
    with pytest.raises(TypeError):
        g.get_rows(12, torch.zeros(2, 256), w, torch.zeros(2, dtype=torch.int64))
    blocks = torch.zeros(2 * 256 * 144, dtype=torch.uint8)
    for at in range(3):
        packed = [(12, blocks.view(dt) if i == at else blocks) for i in range(3)]
        with pytest.raises(TypeError):
            g.MoeLayer(torch.zeros(2, 256), *packed, hidden=256, ff=256, top_k=1)


def test_float_weights_may_be_float_tensors():
    """F16 and BF16 weights as tensors of that type, and of no other: the next check is the device's."""
    import torch
    import gguf_amd as g
    x, y = torch.zeros(1, 16), torch.zeros(1, 4)
    for ty, own, other in ((1, torch.float16, torch.bfloat16), (30, torch.bfloat16, torch.float16)):
        for w in (torch.zeros(4, 16, dtype=own), torch.zeros(4 * 32, dtype=torch.uint8)):
            with pytest.raises(ValueError, match="device"):
                g.matvec(ty, y, w, x)
        with pytest.raises(TypeError):
            g.matvec(ty, y, torch.zeros(4, 16, dtype=other), x)
