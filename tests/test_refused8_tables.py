"""What the entry points that are given a table's size refuse before anything is launched. The addresses are made up, so this runs without a device only."""
import pytest
import torch

from tileinfer_b200.kernels import library

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: not for a machine with a device")
AT = 0x7F0000001000


def refused(rc, *words, code=1):
    assert rc == code, rc
    said = library.lib().ti_last_error().decode()
    assert all(w in said for w in words), said


def attention(slots=8, columns=16, table_stride=16, seqs=4, max_new=1):
    return library.lib().ti_attention8_table(AT, AT, AT, AT, AT, AT, AT, table_stride, AT, AT, AT, AT, 1 << 40, None, 0.1, seqs, 4, 8, 2, 64, 64, max_new, 1000, 100, 0, slots, columns, None)


def test_attention8():
    refused(attention(), "16-byte")                          # the status word is missing: all else was taken
    for change in (dict(slots=-1), dict(columns=-1), dict(table_stride=-1)):
        refused(attention(**change), "table")
    refused(attention(columns=2 ** 30, seqs=8), "2^31 tiles", code=2)
    refused(attention(table_stride=2 ** 30, seqs=8), "16-byte")            # a row's pitch is no length
    assert attention(seqs=0) == 0 and attention(max_new=0) == 0


def write(columns=16, table_stride=16, slots=8, codes=AT + 8):
    return library.lib().ti_cache_write8_table(codes, AT, AT, AT, AT, 1024, 128, AT, 1024, 128, AT, table_stride, slots, AT, AT, AT, 4, 4, 8, 128, 64, 100, 1, 1, columns, None)


def test_cache_write8():
    refused(write(), "16-byte")
    refused(write(table_stride=0), "16-byte")                # rows that are one
    for change in (dict(columns=0), dict(columns=-1), dict(table_stride=-1), dict(slots=0)):
        refused(write(**change), "sequences")
