"""The native torch module serves the paged and likelihood operators alone: the
rest of the package works where it is missing or does not load."""
import shutil
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parent.parent / "rdna4-quant_b200"


def package_without(tmp_path, module):
    """A copy of the Python files with libr4q.so; `module`: None, or what _r4q_torch.so holds."""
    root = tmp_path / PKG.name
    shutil.copytree(PKG / "r4q", root / "r4q", ignore=shutil.ignore_patterns("__pycache__"))
    for f in PKG.glob("*.py"):
        shutil.copy(f, root)
    (root / "libr4q.so").symlink_to(PKG / "libr4q.so")
    if module is not None:
        (root / "_r4q_torch.so").write_bytes(module)
    return root


@pytest.mark.parametrize("module", [None, b"of another build"])
def test_the_rest_of_the_package_does_without_it(tmp_path, module):
    code = f"""
        import sys; sys.path.insert(0, {str(package_without(tmp_path, module))!r})
        import int4_hip, fused_ops
        from r4q import decode, moe, ops, paged, prefill, serve
        import torch
        assert ops.L._PKG.parent == __import__('pathlib').Path({str(tmp_path)!r}).resolve()
        paged.PageAllocator(4, 16, 1, 4).extend({{0: 3}})
        try:
            ops.rmsnorm(torch.zeros(1, 64), torch.zeros(64))
        except ValueError as e:
            assert "CUDA" in str(e)
        for _ in range(2):
            try:
                ops.token_logprobs(torch.zeros(1, 4))
                raise SystemExit("no error")
            except ImportError as e:
                assert "_r4q_torch.so" in str(e), e
        print("served")
    """
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "served" in r.stdout, r.stderr[-2000:]


def test_threads_that_use_it_first_at_once():
    code = f"""
        import sys; sys.path.insert(0, {str(PKG)!r})
        import threading
        from r4q import ops
        import torch
        start, errors = threading.Barrier(8), []
        def first():
            start.wait()
            try:
                ops.token_logprobs(torch.zeros(1, 4))
            except ValueError as e:
                errors.append(str(e))
        ts = [threading.Thread(target=first) for _ in range(8)]
        [t.start() for t in ts]; [t.join() for t in ts]
        assert len(errors) == 8 and all("CUDA" in e for e in errors), errors
        print("served")
    """
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(code)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "served" in r.stdout, r.stderr[-2000:]


def test_build_remakes_it_for_another_torch(monkeypatch, tmp_path):
    """build() with every compiler run recorded instead: nothing to do twice, the module alone after a torch upgrade."""
    import torch
    from r4q import build as b
    src, out = tmp_path / "csrc", tmp_path / "out"
    src.mkdir(), out.mkdir()
    (src / "torch_ops.cpp").write_text("")
    (src / "a.cu").write_text("")
    for name, value in dict(CSRC=src, TORCH_SRC=src / "torch_ops.cpp", OUT=out / "libr4q.so",
                            TORCH_OUT=out / "_r4q_torch.so", BUILD=out / "build").items():
        monkeypatch.setattr(b, name, value)
    runs = []

    def record(cmd, **kw):
        made = Path(cmd[cmd.index("-o") + 1])
        made.write_text("")
        runs.append(made.name)
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(b.subprocess, "run", record)
    b.build()
    assert sorted(runs) == ["_r4q_torch.so.tmp", "a.o", "libr4q.so.tmp"] and (out / "_r4q_torch.so").exists()
    runs.clear()
    b.build()
    assert runs == []
    monkeypatch.setattr(torch, "__version__", "99.0")
    b.build()
    assert runs == ["_r4q_torch.so.tmp"]
    runs.clear()
    b.build()
    assert runs == []
