"""Calls go to the library that ``_lib.load`` gives at that moment."""
import pytest

from td_benchmark_b200 import _lib


class Fake:
    """Stands for the library: every entry returns ``code``."""

    def __init__(self, code):
        self.code, self.called = code, []

    def __getattr__(self, name):
        return lambda *args: self.called.append((name, args)) or self.code

    def b2m_last_error(self):
        return b"made up"


def _refused_by_the_real_library():
    with pytest.raises(_lib.B2MError, match="below 1 ms"):
        _lib.call("b2m_set_timeout_ns", 10)


def test_a_library_put_in_place_is_called_and_goes_with_its_place(monkeypatch):
    """Also for an entry that was called before, and not beyond the replacement."""
    if not _lib.LIB_PATH.exists():
        pytest.skip("libb2m.so not built")
    _refused_by_the_real_library()
    for where in ("_lib", "load"):
        for code in (0, 2):
            fake = Fake(code)
            with monkeypatch.context() as m:
                m.setattr(_lib, where, fake if where == "_lib" else lambda: fake)
                if code:
                    with pytest.raises(_lib.B2MError, match="B2M_ERR_CUDA: made up"):
                        _lib.call("b2m_set_timeout_ns", 10)
                else:
                    _lib.call("b2m_set_timeout_ns", 10)
            assert fake.called == [("b2m_set_timeout_ns", (10,))]
            _refused_by_the_real_library()
