"""``build()`` compiles every source each time: objects of other flags or of a moved clock are not taken for current."""
import __graft_entry__ as entry
from dllm import _build


def test_build_compiles_again(monkeypatch):
    calls = []

    def build(**kw):
        calls.append(kw)
        return _build.LIB_PATH

    monkeypatch.setattr(_build, "build", build)
    entry.build()
    assert len(calls) == 1 and calls[0].get("force") is True
