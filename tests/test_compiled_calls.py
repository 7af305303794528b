"""The compiled plain-case calls (gncde/_calls.so): what they do not know is an error or the Python code's, never the end of
the process (no GPU)."""
import os
import subprocess
import sys
import textwrap
import types

import pytest

from gncde import _lib, engine

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perm-equiv-graph-neural-cdes_amd")
CALLS = ["engine.linear_cross_entropy(odd, W, None, t)",
         "engine.linear_cross_entropy(x, odd, None, t)",
         "engine.linear_cross_entropy(x, W, odd, t)",
         "engine.linear_cross_entropy(x, W, None, odd)",
         "engine.linear_cross_entropy(x, W, None, t, odd)",
         "engine.linear_cross_entropy_grad(odd, W, None, t, x, x)",
         "engine.linear_cross_entropy_grad(x, W, None, t, odd, odd)",
         "engine.linear_cross_entropy_grad(x, W, None, t, x, odd)",
         "engine.global_norm([odd])",
         "engine.global_norm([x, odd])",
         "engine.clip_by_global_norm([odd], 1.0, out=[odd])"]


@pytest.mark.parametrize("odd", ["torch.nested.nested_tensor([torch.zeros(2, 4), torch.zeros(3, 4)])",
                                 "torch.nested.nested_tensor([torch.zeros(2, 4), torch.zeros(3, 4)], layout=torch.jagged)",
                                 "torch.zeros(3, 4).to_sparse()", "torch.zeros(3, 4, device='meta')", "3"],
                         ids=["nested", "jagged", "sparse", "meta", "number"])
def test_odd_arguments_are_errors(odd):
    """In a process of its own, whose exit status says whether every call came back."""
    code = textwrap.dedent(f"""
        import torch
        from gncde import engine
        x, W, t = torch.zeros(3, 4), torch.zeros(5, 4), torch.zeros(3, dtype=torch.int64)
        odd = {odd}
        for call in {CALLS!r}:
            try:
                eval(call)
                print("no error:", call, flush=True)
            except Exception:
                print("error:", call, flush=True)
    """)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env={**os.environ, "PYTHONPATH": PKG})
    assert r.stdout.splitlines() == [f"error: {c}" for c in CALLS] and r.returncode == 0, (r.stdout, r.stderr[-300:])


def test_calls_of_other_sources_are_refused(monkeypatch):
    """The module in the tree is the tree's; one of other sources, or of none that it names, is turned down."""
    assert engine._calls().source_sha256 == _lib.source_sha256(_lib.calls_source_files())
    monkeypatch.setattr(engine, "_fast", None)
    real = _lib.source_sha256
    monkeypatch.setattr(_lib, "source_sha256", lambda files=None: "0" * 64 if files else real())
    with pytest.raises(_lib.GncdeError, match="_calls.so was built from sources .* rebuild"):
        engine._calls()
    assert engine._fast is None
    monkeypatch.undo()
    with pytest.raises(_lib.GncdeError, match="rebuild"):
        _lib.verify_calls(types.SimpleNamespace())


def test_calls_sha_covers_the_signatures(tmp_path):
    names = [os.path.basename(f) for f in _lib.calls_source_files()]
    assert names == ["gncde_calls.cpp", "gncde.h"]
    copies = [tmp_path / n for n in names]
    for c, f in zip(copies, _lib.calls_source_files()):
        c.write_bytes(open(f, "rb").read())
    base = _lib.source_sha256([str(c) for c in copies])
    assert base == engine._calls().source_sha256
    copies[1].write_bytes(copies[1].read_bytes() + b"\n")
    assert _lib.source_sha256([str(c) for c in copies]) != base
