"""What RotaryTable.check and check_layers report, from any stream and for any list of modules; tables that are views."""

import pytest
import torch

import ress_amd as ress
from ress_amd.aggregator import Block, RoPE2D


@pytest.mark.gpu
def test_a_position_turned_on_another_stream(dev):
    """check waits for the device, not for the current stream alone, and a second one finds nothing."""
    rope = ress.RotaryTable(64, 8, axes=1, device=dev)
    x, a = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16, device=dev), torch.randn(4096, 4096, device=dev)
    pos = torch.arange(6, 10, device=dev)
    ress.rotate(x, pos - 6, rope)
    rope.check()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(40):  # some 40 ms in front of it
            b = torch.matmul(a, a)
        ress.rotate(x, pos, rope)
    with pytest.raises(RuntimeError, match="outside the rotation table"):
        rope.check()
    rope.check()
    torch.cuda.synchronize()
    rope.check()
    assert b.shape == a.shape


@pytest.mark.gpu
@pytest.mark.parametrize("given", ["model", "blocks", "attentions"])
def test_a_list_of_modules(dev, given):
    """The rotary modules below the given ones are looked at, too."""
    block = ress.enable_gradients(Block(128, 2, 2.0, RoPE2D()).to(dev, torch.bfloat16))
    model = torch.nn.Sequential(block)
    modules = {"model": model, "blocks": [block], "attentions": [block.attn]}[given]
    x = torch.zeros(1, 4, 128, dtype=torch.bfloat16, device=dev)
    block(x, torch.full((1, 4, 2), 7, device=dev))
    ress.check_layers(modules)
    block(x, torch.full((1, 4, 2), 1 << 20, device=dev))
    with pytest.raises(RuntimeError, match="outside the rotation table"):
        ress.check_layers(modules)
    ress.check_layers(modules)


def test_check_on_the_host():
    rope = ress.RotaryTable(64, 8, axes=1, device="cpu")
    rope.check()
    rope.status.fill_(1)
    with pytest.raises(RuntimeError, match="outside the rotation table"):
        rope.check()
    rope.check()


@pytest.mark.gpu
@pytest.mark.parametrize("at", [0, 1, 2, 3])
def test_a_table_anywhere_in_memory(dev, at):
    """from_table takes a contiguous view that starts at any element."""
    angles = torch.arange(16, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    values = torch.stack([angles.cos(), angles.sin()], 1).float()
    memory = torch.empty(values.numel() + 4, device=dev)
    view = memory[at:at + values.numel()].view(values.shape)
    view.copy_(values)
    x, pos = torch.randn(1, 2, 16, 64, generator=torch.Generator().manual_seed(0)).to(dev, torch.bfloat16), torch.arange(16, device=dev)
    got = ress.rotate(x, pos, ress.RotaryTable.from_table(view, 64, 1))
    assert torch.equal(got, ress.rotate(x, pos, ress.RotaryTable.from_table(values.to(dev), 64, 1)))
