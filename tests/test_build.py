"""When the torch extension is built again."""

import os

from sabrecoder_b200 import build as B


def test_the_extension_follows_torch_and_its_sources(monkeypatch, tmp_path):
    """Built once, kept while nothing changes, built again for another torch or python
    (whose ABI it holds), a newer source, or when it is not known what it was for."""
    import torch
    built = []

    def run(cmd, tmp, out, verbose):
        built.append(out)
        with open(out, "w") as f:
            f.write("so")

    source, header = tmp_path / "call.cpp", tmp_path / "sabre.h"
    source.write_text(""), header.write_text("")
    for name, value in (("CALL", str(tmp_path / "_call.so")), ("CALL_SOURCE", str(source)), ("HEADER", str(header)),
                        ("nvcc", lambda: "/usr/local/cuda/bin/nvcc"), ("_run", run)):
        monkeypatch.setattr(B, name, value)

    def count():
        built.clear()
        assert B.build_call() == B.CALL
        return len(built)

    assert [count(), count()] == [1, 0]
    with monkeypatch.context() as other:
        other.setattr(torch, "__version__", "99.0.0")
        assert [count(), count()] == [1, 0]
    assert [count(), count()] == [1, 0]
    os.utime(B.CALL, (1, 1))  # older than its sources
    assert [count(), count()] == [1, 0]
    for f in tmp_path.glob("_call.so.*"):
        f.unlink()
    assert [count(), count()] == [1, 0]
