"""The first serving operators of a process called by two threads at once. No GPU needed."""
import pytest

import nunchi_b200 as nb

pytest.importorskip("torch")


def test_the_types_are_filled_in_last(monkeypatch):
    """Whoever finds the table of types filled goes on without asking again: all else has to be there by then."""
    seen = []

    class Table(dict):
        def update(self, *a, **k):
            seen.append([getattr(nb, x) for x in ("_F32", "_F16", "_BF16", "_I32", "_stream_of")])
            super().update(*a, **k)

    for x in ("_F32", "_F16", "_BF16", "_I32", "_stream_of"):
        monkeypatch.setattr(nb, x, None)
    monkeypatch.setattr(nb, "_TYPE", Table())
    nb._types()
    assert len(seen) == 1 and None not in seen[0]
    assert sorted(nb._TYPE.values()) == [0, 1, 2]
