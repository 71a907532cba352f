"""A block table that is converted once serves the calls of one stream only."""
import pytest
import torch

from miniserve_amd.attention import block_table_i32

pytestmark = pytest.mark.gpu


def test_a_conversion_is_not_shared_between_streams(device):
    table = torch.arange(300, device=device).view(3, 100)  # int64
    a, b = (torch.cuda.Stream(device) for _ in range(2))
    a.wait_stream(torch.cuda.current_stream(device))
    b.wait_stream(torch.cuda.current_stream(device))
    print("[case] two streams", flush=True)
    with torch.cuda.stream(a):
        torch.cuda._sleep(20_000_000)  # (about 10 ms: the conversion on this stream waits)
        first = block_table_i32(table, device)
        assert block_table_i32(table, device) is first
    with torch.cuda.stream(b):
        second = block_table_i32(table, device)
        assert second is not first
        assert torch.equal(second.cpu(), torch.arange(300, dtype=torch.int32).view(3, 100))
    a.synchronize()
    assert torch.equal(first, second)
    with torch.cuda.stream(a):
        table += 1  # in place: converted anew
        third = block_table_i32(table, device)
        assert third is not first and torch.equal(third, first + 1)
