"""qfg_row_quant_set_option without a GPU."""
import pytest

from qwen38_flash_ops_b200 import _lib


@pytest.mark.parametrize("key,value,message", [(b"give_ups", b"1", "unknown option give_ups"), (None, b"1", "null argument"), (b"give_up", None, "null argument")])
def test_options_that_are_refused(key, value, message):
    lib = _lib.load()
    assert lib.qfg_row_quant_set_option(key, value) == _lib.QFG_INVALID_ARGUMENT
    assert lib.qfg_last_error().decode() == "RowQuant: " + message


def test_an_option_that_is_taken():
    assert _lib.load().qfg_row_quant_set_option(b"give_up", b"0") == _lib.QFG_OK
