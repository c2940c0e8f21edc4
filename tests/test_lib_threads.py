"""The first calls of several threads at once load the autograd module once, and none of them gets half of it."""
import importlib.util
import threading
import time

from cbm4gnn_amd import _lib


def test_one_load_for_all_threads(monkeypatch):
    made, got, errors = [], [], []
    real = importlib.util.module_from_spec

    def slowly(spec):
        made.append(spec)
        module = real(spec)
        time.sleep(0.05)                                    # where another thread may take over
        return module
    monkeypatch.setattr(_lib.importlib.util, "module_from_spec", slowly)
    monkeypatch.setattr(_lib, "_autograd", None)
    together = threading.Barrier(8)

    def first_call():
        together.wait()
        try:
            got.append(_lib.autograd_lib().NormBatch)
        except Exception as e:                              # noqa: BLE001  (told to the test's own thread)
            errors.append(e)
    threads = [threading.Thread(target=first_call) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and len(made) == 1 and len(got) == 8 and len(set(got)) == 1


def test_a_load_that_fails_can_be_tried_again(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "_autograd", None)
    with monkeypatch.context() as m:
        m.setattr(_lib, "AUTOGRAD_LIB", str(tmp_path / "nope.so"))
        for _ in range(2):
            try:
                _lib.autograd_lib()
                raise AssertionError("loaded")
            except _lib.CbmLibraryError:
                pass
    assert _lib.autograd_lib().NormBatch
