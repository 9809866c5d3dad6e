"""Calls of the 4-bit cache's and draft verification's entry points that have nothing
to do: empty arrays may have no address, and none is needed."""
import pytest


@pytest.fixture(scope="module")
def lib():
    from overfit_b200 import _lib, build
    build.build()
    return _lib.load()


@pytest.mark.parametrize("n,rows", [(0, 1), (1, 0), (0, 0)])
def test_calls_without_rows_need_no_buffers(lib, n, rows):
    from overfit_b200 import _lib
    assert lib.ovf_kv_q4_append(None, None, None, None, None, None, n, rows, 8, 128, 64, None, None, 0, None) == _lib.OVF_OK
    assert lib.ovf_kv_q4_read(None, None, None, None, n, rows, 8, 128, 64, None, None, None) == _lib.OVF_OK
    assert lib.ovf_attention_q4(None, None, None, None, None, None, None, None, n, rows, 32, 8, 128, 64, None, None, 0, 0.1,
                                None, None) == _lib.OVF_OK
    # shapes are checked all the same
    assert lib.ovf_kv_q4_append(None, None, None, None, None, None, n, rows, 8, 96, 64, None, None, 0, None) == _lib.OVF_EINVAL
    assert lib.ovf_attention_q4(None, None, None, None, None, None, None, None, n, rows, 30, 8, 128, 64, None, None, 0, 0.1,
                                None, None) == _lib.OVF_EINVAL


def test_verification_of_no_sequences(lib):
    from overfit_b200 import _lib
    assert lib.ovf_verify_drafts(None, None, None, None, None, None, 0, 3, 100, None, None, None) == _lib.OVF_OK
    assert lib.ovf_verify_drafts(None, None, None, None, None, None, 0, 3, 0, None, None, None) == _lib.OVF_EINVAL
