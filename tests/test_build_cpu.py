"""The build without PyTorch, and the binding that it then lacks."""
import os
import subprocess
import sys
import textwrap

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def build_copy(tmp_path, prepare, old=True):
    """build.build(force) in a process of its own, over one small source and with
    its outputs in tmp_path, after `prepare`; (libhq4.so there, binding there, stderr)."""
    src = tmp_path / "csrc"
    src.mkdir()
    (src / "one.cu").write_text('extern "C" int one() { return 1; }\n')
    if old:
        (tmp_path / "_hq4_torch.so").write_text("of other sources")
    code = textwrap.dedent("""
        import importlib.util, os, sys
        spec = importlib.util.spec_from_file_location("hq4_build", sys.argv[1])
        b = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(b)
        b.sources = lambda: [os.path.join(sys.argv[2], "csrc", "one.cu")]
        b.LIB, b.TORCH_LIB = (os.path.join(sys.argv[2], n) for n in ("libhq4.so", "_hq4_torch.so"))
    """) + textwrap.dedent(prepare) + "\nb.build(force=True)\n"
    out = subprocess.run([sys.executable, "-c", code, os.path.join(ROOT, "hetero_infer_b200", "build.py"), str(tmp_path)],
                         capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr
    return (tmp_path / "libhq4.so").exists(), (tmp_path / "_hq4_torch.so").exists(), out.stderr


@pytest.mark.parametrize("prepare", ["sys.modules['torch'] = None",                                  # not installed
                                     "os.environ['CXX'] = '/nonexistent/g++'",                       # no host compiler
                                     "b.TORCH_SRC = os.path.join(sys.argv[2], 'missing.cpp')"])      # it does not compile
def test_library_without_the_binding(tmp_path, prepare):
    lib, binding, said = build_copy(tmp_path, prepare)
    assert lib and not binding
    assert "_hq4_torch.so was not built" in said


def test_a_missing_binding_is_named(tmp_path, monkeypatch):
    from hetero_infer_b200 import _lib, build
    monkeypatch.setattr(build, "TORCH_LIB", str(tmp_path / "_hq4_torch.so"))
    monkeypatch.setattr(_lib, "_torch_calls", None)
    with pytest.raises(RuntimeError, match="_hq4_torch.so is missing"):
        _lib.torch_calls()


def test_a_binding_for_another_torch(tmp_path, monkeypatch):
    """It is neither taken for up to date nor loaded."""
    import shutil
    from hetero_infer_b200 import _lib, build
    path = str(tmp_path / "_hq4_torch.so")
    shutil.copy(build.TORCH_LIB, path)
    monkeypatch.setattr(build, "TORCH_LIB", path)
    monkeypatch.setattr(_lib, "_torch_calls", None)
    (tmp_path / "_hq4_torch.so.torch").write_text(build.torch_version() + "\n")
    assert build.up_to_date(path) and build.torch_version()
    (tmp_path / "_hq4_torch.so.torch").write_text("1.0.0\n")
    assert not build.up_to_date(path)
    with pytest.raises(RuntimeError, match="built for torch 1.0.0"):
        _lib.torch_calls()
