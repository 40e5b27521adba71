"""Importing the package asks nothing of CUDA: who looks for devices fixes which of them are visible, and keeps children that are forked
later from using any."""
import subprocess
import sys
import textwrap


def test_import_does_not_look_for_devices():
    code = textwrap.dedent("""
        import torch
        asked = []
        for name in ("is_available", "device_count", "init", "current_device"):
            setattr(torch.cuda, name, lambda *a, name=name, **k: asked.append(name))
        torch._C._cuda_getDeviceCount = lambda *a: asked.append("_cuda_getDeviceCount")
        import dart_pytorch_b200, dart_pytorch_b200.ops, dart_pytorch_b200.nn, dart_pytorch_b200.models
        print(asked)
    """)
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "[]", run.stdout + run.stderr
