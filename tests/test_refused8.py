"""What the entry points of the 8-bit operators refuse before anything is launched. The addresses are made up, so this runs without a device only."""
import pytest
import torch

from tileinfer_b200.kernels import library

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: not for a machine with a device")
AT = 0x7F0000001000


def refused(rc, *words, code=1):
    assert rc == code, rc
    said = library.lib().ti_last_error().decode()
    assert all(w in said for w in words), said


def quantize(codes=AT, scales=AT, x=AT, ldx=64, dtype=1, n=4, k=64, rows=1):
    return library.lib().ti_quantize8(codes, scales, x, ldx, dtype, n, k, rows, None)


@pytest.mark.parametrize("change,word", [(dict(codes=AT + 8), "16-byte"), (dict(x=AT + 1), "misaligned"), (dict(x=AT + 2, dtype=0), "misaligned"), (dict(scales=AT + 2), "misaligned"),
                                         (dict(k=24), "blocks"), (dict(rows=2), "blocks"), (dict(n=-1), "blocks"), (dict(dtype=5), "element type"),
                                         (dict(n=16 * 65536), "too many"), (dict(n=128 * 65536, rows=128), "too many")])
def test_quantize8(change, word):
    refused(quantize(**change), word)


def linear(y=AT, x=AT, ldx=4096, x_scales=None, codes=AT, n=20, out=4096, k=4096, epilogue=0, ws=AT, ws_bytes=1 << 30, status=AT):
    return library.lib().ti_linear8(y, out, x, ldx, x_scales, codes, AT, n, out, k, epilogue, 0.0, 0.0, 0.0, 0.0, ws, ws_bytes, status, None)


@pytest.mark.parametrize("change,word", [(dict(codes=AT + 8), "16-byte"), (dict(x=AT + 8, x_scales=AT), "16-byte"), (dict(ldx=4104, x_scales=AT), "16-byte"), (dict(ws=None), "work space"),
                                         (dict(ws=AT + 8), "work space"), (dict(ws_bytes=100), "work space"), (dict(status=None), "status"), (dict(epilogue=3), "epilogue"),
                                         (dict(epilogue=9), "epilogue"), (dict(k=4104), "tokens"), (dict(n=-1), "tokens"), (dict(x=AT + 1), "misaligned")])
def test_linear8(change, word):
    refused(linear(**change), word)


@pytest.mark.parametrize("n", [1, 8, 9, 64, 300, 3000])
def test_linear8_work_space(n):
    """Nothing for tokens that come as codes, or that are few; else what their codes and scales take."""
    need = library.lib().ti_linear8_workspace
    assert need(n, 4096, 4096, 1) == 0
    assert need(n, 4096, 4096, 0) == (0 if n <= 8 else n * 4096 + n * 32 * 4)
    assert need(n, 4096, 400, 0) == (0 if n <= 8 else -(-n * 400 // 16) * 16 + -(-n * 16 // 16) * 16)
    assert need(n, 21504, 4096, 0) == (0 if n <= 4 else n * 4096 + n * 32 * 4)


def write(k_codes=AT, v_codes=AT, k=AT, v=AT, page_size=64, dim=128, max_new=1, seqs=4, dtype=1, pages=100):
    return library.lib().ti_cache_write8(k_codes, v_codes, AT, AT, k, 1024, 128, v, 1024, 128, AT, 16, 8, AT, AT, AT, seqs, 4, 8, dim, page_size, pages, max_new, dtype, None)


@pytest.mark.parametrize("change,word,code", [(dict(k_codes=AT + 8), "16-byte", 1), (dict(v_codes=AT + 4), "16-byte", 1), (dict(k=AT + 1), "misaligned", 1), (dict(v=AT + 2, dtype=0), "misaligned", 1),
                                              (dict(page_size=32), "pages of 64", 2), (dict(dim=24), "multiple of 16", 2), (dict(dim=272), "multiple of 16", 2), (dict(seqs=-1), "sequences", 1),
                                              (dict(max_new=2 ** 31 - 1, seqs=2 ** 20), "too many", 1), (dict(dtype=7), "element type", 1), (dict(pages=0), "sequences", 1)])
def test_cache_write8(change, word, code):
    refused(write(**change), word, code=code)


def attention(out=AT, q=AT, k=AT, v=AT, ws=AT, ws_bytes=1 << 40, status=AT, scale=0.1, seqs=4, n=4, nq=8, nkv=2, dim=64, page_size=64, max_new=1, max_len=1000, pages=100,
              window=0, table_stride=16):
    return library.lib().ti_attention8(out, q, k, v, AT, AT, AT, table_stride, AT, AT, AT, ws, ws_bytes, status, scale, seqs, n, nq, nkv, dim, page_size, max_new, max_len, pages,
                                       window, None)


@pytest.mark.parametrize("change,word,code", [(dict(k=AT + 8), "16-byte", 1), (dict(v=AT + 8), "16-byte", 1), (dict(q=AT + 2), "4-byte", 1), (dict(out=AT + 2), "4-byte", 1),
                                              (dict(ws=None), "work space", 1), (dict(ws=AT + 8), "work space", 1), (dict(status=None), "16-byte", 1), (dict(scale=0.0), "scale", 1),
                                              (dict(scale=-1.0), "scale", 1), (dict(seqs=-1), "sequences", 1), (dict(window=-1), "sequences", 1), (dict(pages=0), "sequences", 1),
                                              (dict(page_size=32), "pages of 64", 2), (dict(dim=24), "multiple of 16", 2), (dict(dim=272), "multiple of 16", 2),
                                              (dict(nq=9), "heads", 2), (dict(pages=2 ** 26, nkv=2), "2^31 rows", 2), (dict(table_stride=2 ** 30, seqs=8), "2^31 tiles", 2)])
def test_attention8(change, word, code):
    refused(attention(**change), word, code=code)


def test_attention8_without_work():
    assert attention(seqs=0) == 0 and attention(n=0) == 0 and attention(max_new=0) == 0
