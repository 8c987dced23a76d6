"""Which tests run where: calls with made-up addresses never on a machine with a device, GPU tests only there."""
import pathlib
import types

import conftest
import pytest


class Item:
    def __init__(self, file, *keywords):
        self.path, self.keywords, self.skipped = pathlib.Path("tests") / file, set(keywords), False

    def add_marker(self, mark):
        assert mark.name == "skip"
        self.skipped = True


@pytest.mark.parametrize("device,skipped", [(True, [False, True, False]), (False, [True, False, False])])
def test_what_is_skipped(monkeypatch, device, skipped):
    items = [Item("test_gpu_attn.py", "gpu"), Item("test_gpu_attn.py"), Item("test_abi.py")]
    monkeypatch.setattr(conftest, "_has_gpu", lambda: device)
    conftest.pytest_collection_modifyitems(types.SimpleNamespace(), items)
    assert [i.skipped for i in items] == skipped
