"""What the build makes where torch is not installed: all but the module that is built on its headers."""
import subprocess
import sys
from pathlib import Path

import llm_capi

PKG = Path(llm_capi.__file__).resolve().parent


def targets(python):
    run = subprocess.run(["make", "-n", "-B", "-C", str(PKG), "all", f"PY={python}"], capture_output=True, text=True,
                         timeout=120)
    return run.returncode, run.stdout


def test_all_without_torch(tmp_path):
    python = tmp_path / "python"
    python.write_text("#!/bin/sh\n"
                      f"exec {sys.executable} -c 'import sys; sys.modules[\"torch\"] = None; import importlib.util as u\n"
                      "find = u.find_spec\n"
                      "u.find_spec = lambda name, *a: None if name == \"torch\" else find(name, *a)\n"
                      "code = sys.argv[2]; sys.argv = sys.argv[2:]; exec(code)' \"$@\"\n")
    python.chmod(0o755)
    code, out = targets(python)
    assert code == 0 and "libllm_decoder_hip.so" in out and "llm_decoder" in out
    assert "torch_calls.cpp" not in out
    code, out = targets(sys.executable)
    assert code == 0 and "torch_calls.cpp" in out
