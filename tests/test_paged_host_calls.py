"""The paged cache's further entry points without a GPU: null handles are refused
before any device work."""
import pytest

from pesti_b200 import build, kq, paged


@pytest.fixture(scope="module")
def lib():
    build.build()
    return paged._bind(kq.load_library())


def test_a_tracked_append_without_a_handle_is_refused(lib):
    assert lib.kq_kv_append_tracked(None, None, 0, 0, 1, None, None, None, None, 0, 0, 1.0, None, 0, None, None,
                                    0) == kq.KQ_ERR_INVALID_ARG


def test_a_table_width_without_a_handle_is_refused(lib):
    assert lib.kq_kv_set_table_cols(None, 4) == kq.KQ_ERR_INVALID_ARG
