"""Argument errors and empty sizes of the training operators' C entry points, without a device."""

import pytest

from xfold_cpu_b200 import _capi
from xfold_cpu_b200.build import LIB_PATH


@pytest.mark.skipif(not LIB_PATH.exists(), reason="library not built")
def test_number_documents_arguments():
    lib = _capi.load()
    bad = _capi.ERR_INVALID

    def call(q=256, nq=4, k=256, nk=8, batch=2, q_out=256, k_out=256, ws=256, size=1 << 20):
        return lib.xfb_number_documents(q, nq, nq, k, nk, nk, batch, q_out, k_out, ws, size, None)

    assert call(nq=-1) == call(nk=-1) == call(batch=-1) == bad
    assert call(nk=1 << 30) == call(nq=1 << 30) == call(batch=65536) == bad
    assert call(q=None) == call(q_out=None) == bad
    assert call(k=None) == call(k_out=None) == bad
    need = lib.xfb_number_documents_workspace(2, 4, 8)
    assert need >= 2 * 2 * 12 * 12
    assert call(size=need - 1) == bad
    assert "workspace" in _capi.last_error()
    assert call(ws=8) == bad
    assert call(batch=0) == call(nq=0, nk=0) == _capi.OK
    assert lib.xfb_number_documents_workspace(2, -1, 8) == 0
    assert lib.xfb_number_documents_workspace(0, 4, 8) == 0


@pytest.mark.skipif(not LIB_PATH.exists(), reason="library not built")
def test_linear_of_no_rows():
    lib = _capi.load()
    assert lib.xfb_linear(None, 0, 24, 16, 16, None, None, _capi.BF16, 0, None) == _capi.OK
    assert lib.xfb_linear(None, 0, 20, 16, 16, None, None, _capi.BF16, 0, None) == \
        _capi.ERR_INVALID
