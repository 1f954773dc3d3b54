"""What the C entry points refuse by an address alone, before anything is launched. The addresses are made up, so this runs without a device only."""
import pytest
import torch

from tileinfer_b200.kernels import library

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: not for a machine with a device")
AT = 0x7F0000001000


def refused(rc):
    assert rc == 1, rc
    return library.lib().ti_last_error().decode()


def attention_few(out=AT, q=AT, k=AT, v=AT, ws=AT):
    return library.lib().ti_attention_few(out, q, k, v, AT, 4, AT, AT, AT, ws, 1 << 30, AT, 0.1, 1, 4, 2, 64, 64, 2, 4, 0, None)


@pytest.mark.parametrize("change", [dict(q=AT + 2), dict(out=AT + 2), dict(q=AT + 1), dict(out=AT + 6)])
def test_attention_few_queries_and_outputs(change):
    assert "4-byte aligned" in refused(attention_few(**change))


@pytest.mark.parametrize("change", [dict(k=AT + 8), dict(v=AT + 2), dict(ws=AT + 4)])
def test_attention_few_pages_and_work_space(change):
    assert "aligned" in refused(attention_few(**change)) or "work space" in refused(attention_few(**change))


@pytest.mark.parametrize("n,out,k", [(20, 4096, 4096), (8, 2048, 9216)])
@pytest.mark.parametrize("shift", [1, 4, 8])
def test_linear4_work_space(n, out, k, shift):
    lib = library.lib()
    assert lib.ti_linear4_parts(n, out, k) > 0                # such a product takes one
    rc = lib.ti_linear4(AT, out, AT, k, AT, AT, None, n, out, k, 128, 0, 0.0, 0.0, 0.0, 0.0, 1, AT + shift, AT, None)
    assert "work space must be 16-byte aligned" in refused(rc)
