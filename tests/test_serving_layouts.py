"""What the paged structures tell the kernels of a tensor's layout, without a GPU."""
import struct

import pytest
import torch

import q4kb200 as q


class OnDevice:
    """A CPU tensor that says it is on device 0."""

    def __init__(self, t):
        self.t = t

    def get_device(self):
        return 0

    def __getattr__(self, name):
        return getattr(self.t, name)


def batch_of(table):
    n = table.shape[0]
    return q.PagedBatch(OnDevice(torch.arange(n + 1, dtype=torch.int32)), OnDevice(torch.ones(n, dtype=torch.int32)), OnDevice(table))


def stride_and_width(batch):
    return q._PagedBatch.from_buffer_copy(batch.packed.ljust(struct.calcsize("@iiPPPqi0q"), b"\0"))


@pytest.mark.parametrize("table,stride", [
    (torch.zeros(4, 3, dtype=torch.int32), 3),
    (torch.zeros(1, 3, dtype=torch.int32).expand(4, 3), 0),  # samples of one prompt
    (torch.zeros(1, 1, dtype=torch.int32).expand(4, 1), 0),
    (torch.zeros(4, 9, dtype=torch.int32)[:, :3], 9),
    (torch.zeros(1, 9, dtype=torch.int32)[:, :3], 3),
    (torch.zeros(12, 3, dtype=torch.int32)[::4], 12),
    (torch.zeros(9, dtype=torch.int32).as_strided((4, 3), (2, 1)), 2),  # refused by the calls
])
def test_page_table_rows(table, stride):
    packed = stride_and_width(batch_of(table))
    assert (packed.table_stride, packed.table_width) == (stride, table.shape[1])
