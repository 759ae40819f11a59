"""The build without torch: the library and the host module do not need it."""
import importlib.util
import sys
from pathlib import Path

BUILD = Path(__file__).resolve().parent.parent / "qwen3asr.rs_b200" / "build.py"


def test_without_torch_the_extension_module_is_left_out(monkeypatch, capsys):
    spec = importlib.util.spec_from_file_location("vasr_build_under_test", BUILD)
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    ran = []
    monkeypatch.setattr(build, "_run", lambda cmd: ran.append(cmd))
    monkeypatch.setattr(build, "build_cuda", lambda verbose=False: ran.append("cuda"))
    monkeypatch.setattr(build, "build_host", lambda: ran.append("host"))
    monkeypatch.setitem(sys.modules, "torch", None)  # an import raises ImportError
    build.build()
    assert ran == ["cuda", "host"]
    assert "_vasr_calls" in capsys.readouterr().err
