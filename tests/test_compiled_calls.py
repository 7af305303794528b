"""The compiled plain-case calls (gncde/_calls.so): what they do not know is an error or the Python code's, never the end of
the process (no GPU)."""
import os
import subprocess
import sys
import textwrap

import pytest

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
