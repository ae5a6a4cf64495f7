"""Where a workspace's calls report expired waits (pcb_set_status_word), without a GPU."""
import pytest

from phoenix_core_b200 import _lib


@pytest.fixture(scope="module")
def library():
    from phoenix_core_b200.csrc import build
    build.build()
    return _lib.lib()


def test_refusals(library):
    ws, word = 1 << 20, 1 << 21                                    # (addresses are only kept)
    assert library.pcb_set_status_word(None, word) == _lib.PCB_ERR_INVALID_ARGUMENT
    assert library.pcb_set_status_word(ws, word + 2) == _lib.PCB_ERR_INVALID_ARGUMENT
    assert library.pcb_set_status_word(ws, word) == _lib.PCB_OK
    assert library.pcb_set_status_word(ws, word + 4) == _lib.PCB_OK
    assert library.pcb_set_status_word(ws, None) == _lib.PCB_OK
    assert library.pcb_set_status_word(ws, None) == _lib.PCB_OK     # none to take back
