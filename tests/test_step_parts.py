"""What a decoder step's book-keeping does on the host: requests with few new rows apart from the others."""
import torch

from ane_fieldfare_b200.decoder import Step


def step(rows, sharing=((), ()), maxRows=99):
    total, requests = sum(rows or []), len(rows or [0])
    start = torch.tensor([0, *torch.tensor(rows or [0]).cumsum(0).tolist()], dtype=torch.int32)
    s = Step(start, torch.zeros(total), torch.zeros(total), torch.arange(requests) + 100, torch.arange(requests)[:, None] * 10 + torch.arange(3), maxRows, rows=rows)
    s.sharing = sharing
    s.groupStart, s.prefixLengths = (torch.tensor(x, dtype=torch.int32) for x in sharing)
    return s


def test_all_of_one_kind_are_the_step_itself():
    for rows, few in (([1, 0, 4], True), ([5, 0, 9], False), ([0, 0], True)):
        s = step(rows)
        part, other = s.parts(4) if few else s.parts(4)[::-1]
        assert part == (None, s) and other is None


def test_a_bound_decides_for_all_where_the_rows_are_not_known():
    s = step(None, maxRows=4)
    assert s.parts(4) == ((None, s), None) and s.parts(3) == (None, (None, s))


def test_rows_lengths_and_tables_of_the_parts():
    s = step([1, 7, 0, 2, 5, 3])
    (i, few), (j, many) = s.parts(3)
    assert i.tolist() == [0, 8, 9, 15, 16, 17] and j.tolist() == [1, 2, 3, 4, 5, 6, 7, 10, 11, 12, 13, 14]
    assert few.rowStart.tolist() == [0, 1, 3, 6] and many.rowStart.tolist() == [0, 7, 12]
    assert few.lengths.tolist() == [100, 103, 105] and many.lengths.tolist() == [101, 104]
    assert few.blockTable.tolist() == [[0, 1, 2], [30, 31, 32], [50, 51, 52]] and many.blockTable[:, 0].tolist() == [10, 40]
    assert few.maxRows == 3 and many.maxRows == 7 and many.groupStart is None
    s.lengths += 1  # (the device's: taken again)
    assert s.parts(3)[1][1].lengths.tolist() == [102, 105]


def test_groups_of_the_parts():
    s = step([20, 1, 20, 20, 1, 20, 1, 20, 20], sharing=([0, 3, 4, 6, 9], [128, 0, 64, 256]))
    (_, few), (_, many) = s.parts(4)
    assert many.groupStart.tolist() == [0, 2, 3, 4, 6] and many.prefixLengths.tolist() == [128, 0, 0, 256] and many.maxPrefix == 256
    assert few.groupStart is None  # (one of each group)
    s = step([1, 20, 1, 1, 20, 20], sharing=([2, 4, 6], [32, 48]))
    (_, few), (_, many) = s.parts(4)
    assert few.groupStart.tolist() == [1, 3] and few.prefixLengths.tolist() == [32] and few.maxPrefix == 32
    assert many.groupStart.tolist() == [1, 3] and many.prefixLengths.tolist() == [48]
